"""`ops.scaled_embedding` (`tv_scaled_embedding_*`) against its definition in 64 bits.

u = 2^-24 is half a step of fp32, e half a step of the result's type.  Bounds, counting roundings:
  out = scale * w: scale to fp32 (u), the product (u), the type (e)           -> (2 u + e) |out|
  dW of a token with n rows: n - 1 additions in any order, scale to fp32, the product, the type
                                  -> (n + 1) u sum |scale dout| + e |dW|
(fp16 results below its normal range are off by up to 2^-25 as well)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.float32, torch.bfloat16), (torch.float32, torch.float16)]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0


def _ids(kind, rows, vocab, gen):
    if kind == 'same':
        return torch.full((rows,), vocab - 1)
    if kind == 'padding':
        return torch.full((rows,), -1)
    if kind == 'backwards':
        return (vocab - 1 - torch.arange(rows)) % vocab
    if kind == 'wild':              # far outside the table on both sides, and inside
        pool = torch.tensor([-1, -5, vocab, vocab + 1, 2 ** 40, -2 ** 63, 2 ** 63 - 1, 2 ** 32, 0, vocab - 1])
        return pool[torch.randint(len(pool), (rows,), generator=gen)]
    if kind == 'runs':              # few tokens, each in long runs that cross every border
        return (torch.arange(rows) // 700) % min(vocab, 3)
    u = torch.rand(rows, generator=gen, dtype=torch.float64)
    return ((float(vocab) ** u).long() - 1).clamp(0, vocab - 1)


def _reference(weight, ids, scale, padding, dout):
    """(out, dW, sum |scale dout| per element of dW, rows per token) in float64 on the CPU."""
    v = weight.shape[0]
    named = (ids >= 0) & (ids < v)
    if padding is not None:
        named &= ids != padding
    at = torch.where(named, ids, v)
    table = torch.cat([weight.double().cpu(), torch.zeros(1, weight.shape[1], dtype=torch.float64)])
    out = table[at] * scale
    d = dout.double().cpu() * scale
    dw = torch.zeros_like(table).index_add_(0, at, d)[:v]
    size = torch.zeros_like(table).index_add_(0, at, d.abs())[:v]
    count = torch.bincount(at, minlength=v + 1)[:v].double()[:, None]
    return out, dw, size, count


def _check(weight, ids, scale, padding, out_dtype, dout, device):
    from tracevae_amd import ops
    w = weight.to(device).requires_grad_(True)
    out = ops.scaled_embedding(w, ids.to(device), scale, padding, out_dtype)
    assert out.dtype == out_dtype and out.shape == ids.shape + (weight.shape[1],)
    # memory that held NaN before: rows of dW that no token names have to be written
    junk = torch.full(tuple(weight.shape), math.nan, dtype=weight.dtype, device=device)
    del junk
    (dw,) = torch.autograd.grad(out, w, dout.to(device) if dout.device != device else dout)
    assert dw.dtype == weight.dtype and dw.shape == weight.shape and dw.is_contiguous()
    ref, rdw, size, count = _reference(weight, ids.reshape(-1), scale, padding, dout.reshape(-1, weight.shape[1]))
    tiny = 2.0 ** -25 if torch.float16 in (out_dtype, weight.dtype) else 0.0
    got = out.detach().cpu().double().reshape(ref.shape)
    assert ((got - ref).abs() <= (2 * U + _half_step(out_dtype)) * ref.abs() + tiny).all()
    got = dw.cpu().double()
    assert ((got - rdw).abs() <= (count + 1) * U * size + _half_step(weight.dtype) * rdw.abs() * (1 + 1e-3) + tiny).all()
    assert (got[count[:, 0] == 0] == 0).all()
    return out, dw


@pytest.mark.parametrize('rows,vocab,dim', [(1, 1, 1), (2, 5, 3), (31, 1000, 40), (33, 7, 64), (257, 1023, 250),
                                           (1021, 997, 251), (5000, 1024, 40), (4097, 1025, 8), (300, 70001, 130),
                                           (20000, 1000, 16), (9000, 5, 1027), (2049, 300000, 33),
                                           (64, 50, 5), (65, 17, 600), (128, 300, 72), (129, 300, 72), (100, 90000, 9),
                                           (8192, 300, 20), (8193, 300, 20)])
@pytest.mark.parametrize('kind', ['zipf', 'same', 'wild', 'runs'])
def test_rows_and_gradient(device, rows, vocab, dim, kind):
    for k, (table, out_dtype) in enumerate(TYPES):
        if dim * vocab > 2_000_000 and k not in (0, 3):
            continue
        g = torch.Generator().manual_seed(rows + vocab + dim + k)
        ids = _ids(kind, rows, vocab, g)
        w = (torch.randn(vocab, dim, generator=g)).to(table)
        dout = (torch.randn(rows, dim, generator=g) * 0.1).to(out_dtype)
        padding = [None, vocab // 2, 0][k % 3]
        a = _check(w, ids, math.sqrt(dim), padding, out_dtype, dout, device)
        b = _check(w, ids, math.sqrt(dim), padding, out_dtype, dout, device)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])        # bit-stable


@pytest.mark.parametrize('rows,vocab,dim', [(70000, 1000, 40), (140000, 3, 72), (70000, 200001, 24)])
@pytest.mark.parametrize('kind', ['zipf', 'same', 'runs', 'backwards'])
def test_long_batches(device, rows, vocab, dim, kind):
    g = torch.Generator().manual_seed(rows + vocab)
    ids = _ids(kind, rows, vocab, g)
    w = torch.randn(vocab, dim, generator=g)
    _check(w, ids, 0.5, None, torch.float32, torch.randn(rows, dim, generator=g), device)
    _check(w.bfloat16(), ids, 0.5, None, torch.bfloat16, torch.randn(rows, dim, generator=g).bfloat16(), device)


@pytest.mark.parametrize('rows,vocab,dim', [(700, 1501, 513), (700, 1499, 1030), (5000, 401, 2051), (3000, 33, 1280)])
@pytest.mark.parametrize('kind', ['zipf', 'same', 'runs'])
def test_wide_rows(device, rows, vocab, dim, kind):
    """Absent rows of 1 to 8 KB, tokens of many tiles in several slabs of columns."""
    g = torch.Generator().manual_seed(rows + vocab + dim)
    ids = _ids(kind, rows, vocab, g)
    w = torch.randn(vocab, dim, generator=g)
    d = torch.randn(rows, dim, generator=g)
    for table, out_dtype in ((torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                             (torch.float16, torch.float16)):
        _check(w.to(table), ids, 0.5, vocab // 2, out_dtype, d.to(out_dtype), device)


def test_no_rows_and_nothing_but_padding(device):
    for table, out_dtype in TYPES:
        w = torch.randn(70, 24).to(table)
        _check(w, torch.zeros(0, dtype=torch.int64), 2.0, None, out_dtype, torch.zeros(0, 24, dtype=out_dtype), device)
        _check(w, _ids('padding', 500, 70, None), 2.0, None, out_dtype, torch.randn(500, 24).to(out_dtype), device)
        _check(w, torch.full((500,), 3), 2.0, 3, out_dtype, torch.randn(500, 24).to(out_dtype), device)


@pytest.mark.parametrize('rows,vocab,dim', [(0, 70, 24), (5, 300, 3), (128, 300, 72), (129, 300, 72),
                                           (700, 1501, 513), (300, 70001, 130), (2049, 300000, 33),
                                           (70000, 200001, 24), (20000, 5, 8)])
@pytest.mark.parametrize('kind', ['zipf', 'same', 'padding'])
def test_every_row_of_the_table_gradient_is_written(device, rows, vocab, dim, kind):
    """Into memory full of NaN, with a row before and a row behind that stay as they are, and so does what lies
    behind the workspace."""
    from tracevae_amd import hip
    codes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    g = torch.Generator().manual_seed(rows + vocab)
    ids = _ids(kind, rows, vocab, g)
    for table, rt in TYPES[:4]:
        d = torch.randn(rows, dim, generator=g).to(rt)
        need = hip.query('tv_scaled_embedding_bwd_workspace_bytes', rows, dim, vocab)
        ws = torch.full((need + 256,), 255, dtype=torch.uint8, device=device)
        around = torch.full((vocab + 2, dim), math.nan, dtype=table, device=device)
        ids_d, d_d = ids.to(device), d.to(device)
        hip.call('tv_scaled_embedding_bwd', rows, dim, vocab, codes[table], codes[rt], hip.ptr(ids_d), -1, 0.5,
                 hip.ptr(d_d), dim, around[1:].data_ptr(), hip.ptr(ws), need)
        _, dw, size, count = _reference(torch.zeros(vocab, dim), ids, 0.5, None, d)
        got = around.cpu().double()
        assert torch.isnan(got[0]).all() and torch.isnan(got[-1]).all() and (ws[need:] == 255).all()
        assert ((got[1:-1] - dw).abs() <= (count + 1) * U * size + _half_step(table) * dw.abs() * (1 + 1e-3)
                + (2.0 ** -25 if torch.float16 in (table, rt) else 0.0)).all()


def test_infinities_and_nan_stay_in_their_rows(device):
    """inf / NaN in rows of the table that no token names, and in the gradient of padded rows."""
    from tracevae_amd import ops
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 40, (3000,), generator=g)
    ids[::7] = -1
    w = torch.randn(50, 48, generator=g)
    w[40:] = math.nan
    d = torch.randn(3000, 48, generator=g)
    d[::7] = math.inf
    x = w.to(device).requires_grad_(True)
    out = ops.scaled_embedding(x, ids.to(device), 3.0)
    assert torch.isfinite(out).all()
    (dw,) = torch.autograd.grad(out, x, d.to(device))
    assert torch.isfinite(dw).all() and (dw[40:] == 0).all()
    d[1, 5] = math.inf                                    # one named row: one element of one token
    (dw,) = torch.autograd.grad(ops.scaled_embedding(x, ids.to(device), 3.0), x, d.to(device))
    bad = ~torch.isfinite(dw.cpu())
    assert bad.sum() == 1 and bad[ids[1], 5]


@pytest.mark.parametrize('table,out_dtype', TYPES)
@pytest.mark.parametrize('dim', [40, 41, 256])
def test_strides_and_alignment(device, table, out_dtype, dim):
    """Rows of a wider table, columns of a wider gradient, ids of two dimensions; every address at an
    odd element."""
    g = torch.Generator().manual_seed(dim)
    wide = torch.randn(200 * (dim + 7) + 1, generator=g).to(table).to(device)[1:].view(200, dim + 7)
    ids = _ids('zipf', 1500, 200, g).view(30, 50)
    dwide = torch.randn(1500 * (dim + 5) + 3, generator=g).to(out_dtype).to(device)[3:].view(30, 50, dim + 5)
    from tracevae_amd import ops
    w = wide[:, 3:3 + dim].detach().requires_grad_(True)
    out = ops.scaled_embedding(w, ids.to(device), 1.5, 7, out_dtype)
    for dout in (dwide[:, :, 2:2 + dim], dwide[:, :, 2:2 + dim].transpose(0, 1).contiguous().transpose(0, 1),
                 dwide[:1, :1, :1].expand(30, 50, dim)):
        (dw,) = torch.autograd.grad(out, w, dout, retain_graph=True)
        _, want = _check(wide[:, 3:3 + dim].cpu().contiguous(), ids, 1.5, 7, out_dtype,
                         dout.contiguous().cpu(), device)
        assert torch.equal(dw, want)
    assert torch.equal(out.detach(), ops.scaled_embedding(w.detach().contiguous(), ids.to(device), 1.5, 7, out_dtype))


def test_difference_quotient_and_two_uses(device):
    """Whole numbers, so every sum is exact: <out(w + h) - out(w), d> = <h, dW>, and a table that is
    looked up twice gets both gradients."""
    from tracevae_amd import ops
    g = torch.Generator().manual_seed(4)
    w = torch.randint(-8, 9, (300, 36), generator=g).float().to(device).requires_grad_(True)
    h = torch.randint(-8, 9, (300, 36), generator=g).float().to(device)
    d = torch.randint(-8, 9, (4000, 36), generator=g).float().to(device)
    ids = torch.randint(-1, 300, (4000,), generator=g).to(device)
    out = ops.scaled_embedding(w, ids, 2.0, 17)
    (dw,) = torch.autograd.grad(out, w, d)
    with torch.no_grad():
        moved = ops.scaled_embedding(w + h, ids, 2.0, 17)
    assert float(((moved - out).double() * d.double()).sum()) == float((h.double() * dw.double()).sum())
    (ops.scaled_embedding(w, ids, 2.0, 17) * d).sum().backward(retain_graph=True)
    (ops.scaled_embedding(w, ids.flip(0), 2.0, 17) * d.flip(0)).sum().backward()
    assert torch.equal(w.grad, 2 * dw)


def test_one_id_without_a_dimension(device):
    from tracevae_amd import ops
    w = torch.randn(9, 20, device=device, requires_grad=True)
    out = ops.scaled_embedding(w, torch.tensor(4, device=device), 2.0)
    assert out.shape == (20,) and torch.equal(out, 2 * w[4])
    (dw,) = torch.autograd.grad(out, w, torch.ones(1, device=device).expand(20))
    want = torch.zeros(9, 20, device=device)
    want[4] = 2.0
    assert torch.equal(dw, want)


def test_no_second_derivative_and_no_changed_ids(device):
    from tracevae_amd import ops
    w = torch.randn(50, 16, device=device, requires_grad=True)
    ids = torch.randint(0, 50, (100,), device=device)
    d = torch.randn(100, 16, device=device, requires_grad=True)
    (dw,) = torch.autograd.grad(ops.scaled_embedding(w, ids, 2.0), w, d, create_graph=True)
    want = torch.autograd.grad(ops.scaled_embedding(w, ids, 2.0), w, d.detach())[0]
    assert torch.equal(dw.detach(), want)
    with pytest.raises(RuntimeError, match='twice'):
        dw.sum().backward()
    out = ops.scaled_embedding(w, ids, 2.0)
    ids.fill_(3)                                          # as with torch's own lookup
    with pytest.raises(RuntimeError, match='modified'):
        out.sum().backward()
    with torch.no_grad():
        assert not ops.scaled_embedding(w, ids, 2.0).requires_grad
    assert not ops.scaled_embedding(w.detach(), ids, 2.0).requires_grad


@pytest.mark.parametrize('requires', [False, True])
@pytest.mark.parametrize('grad', [False, True])
def test_a_tangent_of_the_table_is_refused(device, requires, grad):
    import torch.autograd.forward_ad as forward
    from tracevae_amd import ops
    ids = torch.arange(60, device=device) % 30
    w = torch.randn(30, 8, device=device).requires_grad_(requires)
    with forward.dual_level(), torch.set_grad_enabled(grad):
        dual = forward.make_dual(w, torch.ones_like(w))
        with pytest.raises(NotImplementedError, match='forward'):
            ops.scaled_embedding(dual, ids, 2.0)


def test_a_tangent_of_the_gradient_is_refused(device):
    import torch.autograd.forward_ad as forward
    from tracevae_amd import ops
    w = torch.randn(30, 8, device=device, requires_grad=True)
    out = ops.scaled_embedding(w, torch.arange(60, device=device) % 30, 2.0)
    ones = torch.ones(60, 8, device=device)
    with forward.dual_level():
        with pytest.raises(NotImplementedError, match='forward'):
            torch.autograd.grad(out, w, forward.make_dual(ones, ones))


def test_function_transforms_are_refused(device):
    from tracevae_amd import ops
    w = torch.randn(30, 8, device=device)
    ids = torch.arange(60, device=device) % 30

    def look(x):
        return ops.scaled_embedding(x, ids, 2.0)

    for call in (lambda: torch.func.vmap(lambda i: ops.scaled_embedding(w, i))(ids.view(2, 30)),
                 lambda: torch.func.vmap(look)(torch.stack([w, w])),
                 lambda: torch.func.grad(lambda x: look(x).sum())(w),
                 lambda: torch.func.jvp(look, (w,), (w,))):
        with pytest.raises(RuntimeError):
            call()
    x = w.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(look(x), x, torch.ones(2, 60, 8, device=device), is_grads_batched=True)


@pytest.mark.parametrize('dim', [1, 6])
def test_views_with_the_opposite_sign(device, dim):
    """The imaginary part of a conjugate is a view of the values with the sign pending."""
    from tracevae_amd import ops
    w = torch.randn(30, dim, device=device)
    ids = torch.arange(60, device=device) % 30
    assert torch.equal(ops.scaled_embedding(torch._neg_view(w), ids, 2.0), -2 * w[ids])
    x = w.clone().requires_grad_(True)
    d = torch.randn(60, dim, dtype=torch.complex64, device=device)
    (want,) = torch.autograd.grad(ops.scaled_embedding(x, ids, 2.0), x, -d.imag.clone())
    for dout in (d.conj().imag, torch._neg_view(d.imag.contiguous())):
        assert dout.is_neg()
        (dw,) = torch.autograd.grad(ops.scaled_embedding(x, ids, 2.0), x, dout)
        assert torch.equal(dw, want)


def test_zeros_without_memory(device):
    from tracevae_amd import ops
    x = torch.randn(30, 6, device=device, requires_grad=True)
    ids = torch.arange(600, device=device) % 30
    for rows in (60, 600):
        zeros = torch._efficientzerotensor((rows, 6), device=device)
        assert zeros.data_ptr() == 0
        (dw,) = torch.autograd.grad(ops.scaled_embedding(x, ids[:rows], 2.0), x, zeros)
        assert torch.equal(dw, torch.zeros_like(x))
    out = ops.scaled_embedding(torch._efficientzerotensor((30, 6), device=device), ids, 2.0)
    assert torch.equal(out, torch.zeros(600, 6, device=device))


def test_more_than_2_to_the_31_elements(device):
    """bf16 rows of 2^21 + 5 tokens by 1030 columns: positions beyond 32 bits in the rows and in their
    gradient (4.3 GB each)."""
    from tracevae_amd import ops
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip('needs 48 GiB of free GPU memory')
    rows, dim, v = 2 ** 21 + 5, 1030, 4096
    g = torch.Generator(device=device).manual_seed(3)
    ids = torch.randint(0, v, (rows,), generator=g, device=device)
    ids[:100] = 7
    ids[-100:] = 7
    w = torch.randn(v, dim, generator=g, device=device).bfloat16().requires_grad_(True)
    out = ops.scaled_embedding(w, ids, 1.0)
    for r in (0, 1, rows // 2, rows - 2, rows - 1):
        assert torch.equal(out[r], w[ids[r]])
    dout = torch.randn(rows, dim, generator=g, device=device, dtype=torch.bfloat16)
    (dw,) = torch.autograd.grad(out, w, dout)
    for token in (0, 7, 2048, v - 1):
        x = dout[ids == token].double()
        want, n = x.sum(0), x.shape[0]
        assert ((dw[token].double() - want).abs() <= (n + 1) * U * x.abs().sum(0) + 2.0 ** -8 * want.abs()).all()
    del out, dout, dw
    torch.cuda.empty_cache()


def test_a_lookup_of_more_rows_than_one_launch_takes(device):
    """2^23 + 5 rows of 1028 fp32 (34.5 GB): one workgroup for every two rows, 2^22 in a launch."""
    from tracevae_amd import ops
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip('needs 48 GiB of free GPU memory')
    rows, dim, v = 2 ** 23 + 5, 1028, 1000
    w = torch.randn(v, dim, device=device)
    ids = torch.arange(rows, device=device) * 7 % v
    out = ops.scaled_embedding(w, ids, 1.0)
    for r0 in (0, rows // 2, 2 ** 23 - 1000, rows - 1000):
        assert torch.equal(out[r0:r0 + 1000], w[ids[r0:r0 + 1000]])
    assert torch.equal(out[:, 5], w[:, 5][ids]) and torch.equal(out[:, -1], w[:, -1][ids])
    del out
    torch.cuda.empty_cache()


def test_captured_and_replayed(device):
    """Forward and gradient in one captured graph, replayed on new ids with eager calls of another size
    between the replays: equal to the eager result every time."""
    from tracevae_amd import ops
    g = torch.Generator().manual_seed(6)
    rows, v, dim = 3000, 5000, 48
    ids = torch.zeros(rows, dtype=torch.int64, device=device)
    w = torch.randn(v, dim, generator=g).to(device).requires_grad_(True)
    dout = torch.randn(rows, dim, generator=g).to(device)

    def both():
        out = ops.scaled_embedding(w, ids, 2.0)
        return out, torch.autograd.grad(out, w, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dw = both()
    out, dw = out.detach(), dw.detach()
    for k, kind in enumerate(['zipf', 'same', 'runs', 'padding', 'wild']):
        ids.copy_(_ids(kind, rows, v, g))
        w.data.add_(1.0)
        graph.replay()
        other = torch.randint(0, 50, (rows * (k + 1),), device=device)
        small = torch.randn(50, 32, device=device, requires_grad=True)
        torch.autograd.grad(ops.scaled_embedding(small, other, 1.0).sum(), small)
        torch.cuda.synchronize()
        want_out, want_dw = both()
        assert torch.equal(out, want_out.detach()) and torch.equal(dw, want_dw), kind


@pytest.mark.parametrize('cast', [False, True])
def test_a_capture_beside_a_living_eager_graph_is_refused(device, cast):
    """A captured backward pass that leads to a leaf whose accumulator an eager graph holds is refused while
    the capture is still sound; without that graph, or up to a tensor made in the capture, it is taken."""
    from tracevae_amd import ops
    ids = torch.arange(600, device=device) % 37
    w = torch.randn(40, 16, device=device, requires_grad=True)
    dout = torch.randn(600, 16, device=device, dtype=torch.bfloat16 if cast else torch.float32)

    def both(backward):
        table = w.bfloat16() if cast else w
        out = ops.scaled_embedding(table, ids, 2.0)
        return out, backward(out, table)

    want = both(lambda out, table: torch.autograd.grad(out, w, dout)[0])[1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(lambda out, table: torch.autograd.grad(out, w, dout)[0])
    torch.cuda.synchronize()
    kept = w * 1.0                                        # the eager graph
    refused = []

    def expect_refusal(backward):
        def run(out, table):
            try:
                backward(out, table)
            except RuntimeError as e:
                refused.append('eager graph' in str(e))
        return run

    for backward in (lambda out, table: torch.autograd.grad(out, w, dout), lambda out, table: out.backward(dout)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(expect_refusal(backward))[0].detach()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, 2 * (w.detach().bfloat16() if cast else w.detach())[ids])
    assert refused == [True, True] and w.grad is None
    if cast:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            dw = both(lambda out, table: torch.autograd.grad(out, table, dout)[0])[1].detach()
        graph.replay()
        assert torch.equal(dw.float(), want)
    assert torch.equal(torch.autograd.grad(kept.sum(), w)[0], torch.ones_like(w))
    del kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw = both(lambda out, table: torch.autograd.grad(out, w, dout)[0])[1].detach()
    for _ in range(3):
        dw.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, want)


def test_the_node_called_by_hand_refuses_other_gradients(device):
    from tracevae_amd import ops
    w = torch.randn(10, 4, device=device, requires_grad=True)
    node = ops.scaled_embedding(w, torch.arange(10, device=device)).grad_fn
    ones = torch.ones(10, 4, device=device)
    for bad in (ones.cpu(), ones.half(), ones.double(), ones.to_sparse()):
        with pytest.raises(RuntimeError, match='must be a dense tensor'):
            node(bad)
    with pytest.raises(RuntimeError):
        node(ones[:5])
    assert torch.equal(node(ones)[0], ones)


def test_two_streams_at_once(device):
    from tracevae_amd import ops
    g = torch.Generator().manual_seed(8)
    jobs, want = [], []
    for k in range(2):
        w = torch.randn(3000, 64, generator=g).to(device).requires_grad_(True)
        ids = torch.randint(0, 3000, (50000,), generator=g).to(device)
        d = torch.randn(50000, 64, generator=g).to(device)
        jobs.append((w, ids, d, torch.cuda.Stream()))
        want.append(torch.autograd.grad(ops.scaled_embedding(w, ids, 1.0), w, d)[0])
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, (w, ids, d, s) in enumerate(jobs):
            with torch.cuda.stream(s):
                got[k].append(torch.autograd.grad(ops.scaled_embedding(w, ids, 1.0), w, d)[0])
    torch.cuda.synchronize()
    for k in range(2):
        for x in got[k]:
            assert torch.equal(x, want[k])


def test_refusals(device):
    from tracevae_amd import hip, ops
    w, ids = torch.zeros(10, 4, device=device), torch.zeros(3, dtype=torch.int64, device=device)
    with pytest.raises(hip.HipLibraryError):
        ops.scaled_embedding(w, ids.cpu())
    with pytest.raises(hip.HipLibraryError):
        ops.scaled_embedding(w.cpu(), ids)
    with pytest.raises(TypeError):
        ops.scaled_embedding(w, ids.int())
    with pytest.raises(TypeError):
        ops.scaled_embedding(w.double(), ids)
    with pytest.raises(TypeError):
        ops.scaled_embedding(w.bfloat16(), ids, out_dtype=torch.float32)
    with pytest.raises(TypeError):
        ops.scaled_embedding(w.bfloat16(), ids, out_dtype=torch.float16)
    for bad in (w[0], w[:0], w[:, :0]):
        with pytest.raises(ValueError):
            ops.scaled_embedding(bad, ids)


@pytest.mark.parametrize('bits,capture', [(32, False), (8, False), (32, True), (8, True)])
def test_table_trained_by_lookup_gradient_and_adamw(device, bits, capture):
    """The operators as they are used together: rows of a table, a loss, the table's gradient by sorted
    tokens, clipping and the AdamW step - eager or captured into one graph and replayed with new ids -
    against the same steps in float64 on the CPU.  With 32-bit moments the weights stay within the
    roundings of the steps (the gradient's relative error is at most (n + 2) u, Adam's change is lr
    times a ratio of which it is the error, times sqrt(t) for the steps before); with 8-bit moments
    gradient, moments and codes of each step are checked against the step's own inputs."""
    import adamw_reference as ref
    from tracevae_amd import ops
    from tracevae_amd.optim import AdamW
    g = torch.Generator().manual_seed(9)
    v, dim, rows = 512, 24, 700
    table = (torch.randn(v, dim, generator=g) * 0.1).to(device).requires_grad_(True)
    opt = AdamW([table], lr=1e-2, weight_decay=0.1, state_bits=bits, seed=11)
    ids = torch.zeros(rows, dtype=torch.int64, device=device)
    target = torch.randn(rows, dim, generator=g).to(device)

    def step():
        out = ops.scaled_embedding(table, ids, 4.0, padding_idx=0)
        dout = 2.0 * (out - target)                       # of the squared error
        (grad,) = torch.autograd.grad(out, table, dout)
        opt.step([grad], global_clip_norm=5.0)
        return dout.detach(), grad

    batches = [_ids('zipf', rows, v, g) for _ in range(5)]
    ids.copy_(batches[0])
    torch.cuda.synchronize()
    if capture:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            dout, grad = step()
    for batch in batches:
        ids.copy_(batch)
        w0 = table.detach().cpu().double().reshape(-1)
        s0 = {k: x.cpu().clone() for k, x in opt.state.items()}
        t = opt.steps + 1
        if capture:
            graph.replay()
        else:
            dout, grad = step()
        torch.cuda.synchronize()
        _, dw, size, count = _reference(w0.view(v, dim), batch, 4.0, 0, dout)
        assert ((grad.cpu().double() - dw).abs() <= (count + 1) * U * size).all()
        gx = grad.cpu().double().reshape(-1)
        norm = float(gx.square().sum().sqrt())
        assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -40 * norm
        if bits == 32:
            m0, v0 = s0['exp_avg'].double(), s0['exp_avg_sq'].double()
        else:
            m0 = s0['exp_avg8'].double() * s0['exp_avg_scale'].double().repeat_interleave(256)
            v0 = (s0['exp_rms8'].double() * s0['exp_rms_scale'].double().repeat_interleave(256)) ** 2
        coef = min(1.0, 5.0 / (norm + 1e-6))
        p1, m1, v1, change = ref.step(w0, gx, m0, v0, t, 1e-2, 0.9, 0.999, 1e-8, 0.1, coef)
        size = 1e-2 / (1 - 0.9 ** t) / (v1.sqrt() / math.sqrt(1 - 0.999 ** t) + 1e-8)
        big = (0.9 * m0).abs() + (0.1 * gx * coef).abs()
        bound = 3 * U * (w0.abs() + change.abs()) + 11 * U * change.abs() + 5 * U * big * size
        assert ((table.detach().cpu().double().reshape(-1) - p1).abs() <= bound).all()
        if bits == 8:
            words = ref.random_words(torch.arange(v * dim), 11, t).view(-1, 256)
            for name, x, u in (('exp_avg', m1, words & 0xffff), ('exp_rms', v1.sqrt(), words >> 16)):
                q, scale = ref.to_codes(x.view(-1, 256), u, name == 'exp_rms')
                assert torch.equal(opt.state[name + '_scale'].cpu(), scale.view(-1))
                assert torch.equal(opt.state[name + '8'].cpu().double().view(-1, 256), q)


def test_backward_accumulates_and_the_optimizer_reads_grad(device):
    """The loop of a user's program: .backward() twice into .grad, step(), zero_grad(); tensors of three
    types in one optimizer, gradients by autograd."""
    from tracevae_amd import AdamW, ops
    gen = torch.Generator().manual_seed(12)
    table = torch.nn.Parameter((torch.randn(300, 32, generator=gen) * 0.1).to(device))
    half = torch.nn.Parameter((torch.randn(300, 32, generator=gen) * 0.1).half().to(device))
    head = torch.nn.Linear(32, 5).to(device).bfloat16()
    unused = torch.nn.Parameter(torch.ones(7, device=device))
    opt = AdamW([table, half, *head.parameters(), unused], lr=1e-2, weight_decay=0.0, state_bits=8)
    ids = torch.randint(-1, 300, (6, 50), generator=gen).to(device)
    grads = []
    for _ in range(2):
        a = ops.scaled_embedding(table, ids, 2.0, out_dtype=torch.bfloat16)
        b = ops.scaled_embedding(half, ids, 2.0)
        (head(a).float().square().mean() + b.float().square().sum()).backward()
        grads.append([p.grad.clone() for p in (table, half, *head.parameters())])
    for first, both in zip(*grads):                       # (twice a number is exact)
        assert torch.equal(both, 2 * first)
    before = [p.detach().clone() for p in opt.params]
    version = table._version
    norm = opt.step(global_clip_norm=1.0)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads[1]))
    assert abs(float(norm) - want) <= 2.0 ** -40 * want
    assert table._version > version                       # autograd knows that it was written
    for p, q in zip(opt.params, before):
        assert torch.equal(p, q) == (p is unused)
        assert torch.isfinite(p).all()
    named = torch.zeros(300, dtype=torch.bool)
    named[ids.cpu().reshape(-1)[ids.cpu().reshape(-1) >= 0]] = True
    assert torch.equal(table.detach().cpu()[~named], before[0].cpu()[~named])     # rows nobody named
    opt.zero_grad()
    assert all(p.grad is None for p in opt.params)
