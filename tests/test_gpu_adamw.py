"""`optim.AdamW` (`tv_adamw_*`) against the formula in 64 bits (`adamw_reference.py`).

Every step is compared on its own: the reference starts from the state the kernel left.  u = 2^-24
is half a step of fp32.  Bounds with 32-bit moments, counting roundings:
  m   b1 (1), its product is fused; 1 - b1, coef, g coef, (1 - b1) g (4); the sum (1)
      -> 5 u (|b1 m| + |(1 - b1) g|), which M below stands for
  v   1 - b2, coef and g coef twice each, two products, the sum: 8 u v
  p   keep, p keep, the sum: 3 u |p|; the change: v 8 / 2, sqrt, bias correction, its fma, eps,
      division, step size, 1 for what is of second order: 11 u |change|, and 5 u of it by m with
      M in place of m.
With 8-bit moments m and v are float64 up to their conversion, and codes and scales are EQUAL.
A 16-bit parameter is its master rounded: equal."""
import copy
import math

import numpy as np
import pytest
import torch

import adamw_reference as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8)
ODD = [(7, 37), (1,), (256,), (255,), (257,), (0,), (3, 5, 11), (4096,), (4097,), (64, 150), (2, 4100)]


def _flat(tensors, offsets, total):
    out = torch.zeros(total, dtype=torch.float64)
    for t, at in zip(tensors, offsets):
        out[at:at + t.numel()] = t.detach().double().cpu().reshape(-1)
    return out


def _params(shapes, dtype, device, seed, shift=0):
    """Tensors of one buffer with `shift` elements between them (so that they are misaligned)."""
    g = torch.Generator().manual_seed(seed)
    total = sum(math.prod(s) for s in shapes) + shift * len(shapes) + shift
    buf = (torch.randn(total, generator=g) * 0.1).to(dtype).to(device)
    out, at = [], shift
    for s in shapes:
        n = math.prod(s)
        out.append(buf[at:at + n].view(s))
        at += n + shift
    return out


def _grads(params, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(p.shape, generator=g) * 10.0 ** (spread * torch.randn(1, generator=g)) * 1e-2)
            .to(p.dtype).to(p.device) for p in params]


class Twin(object):
    """Checks the steps of one optimizer against the reference."""

    def __init__(self, opt, decay):
        self.opt = opt
        self.decay = decay
        self.total = sum((p.numel() + 255) // 256 * 256 for p in opt.params)
        self.t = opt.steps
        self.dec = torch.zeros(self.total, dtype=torch.float64)
        self.inside = torch.zeros(self.total, dtype=torch.bool)
        for p, at, d in zip(opt.params, opt.offsets, decay):
            self.dec[at:at + p.numel()] = d
            self.inside[at:at + p.numel()] = True

    def moments(self):
        s = {k: v.cpu() for k, v in self.opt.state.items()}
        if self.opt.state_bits == 32:
            return s['exp_avg'].double(), s['exp_avg_sq'].double()
        m = s['exp_avg8'].double() * s['exp_avg_scale'].double().repeat_interleave(256)
        r = s['exp_rms8'].double() * s['exp_rms_scale'].double().repeat_interleave(256)
        return m, r * r

    def weights(self):
        p = _flat(self.opt.params, self.opt.offsets, self.total)
        return self.opt.state['master'].cpu().double() if 'master' in self.opt.state else p

    def step(self, grads, clip=None, given=None):
        """One step with `grads` (default: handed to step() as they are), checked."""
        opt = self.opt
        m0, v0 = self.moments()
        p0 = self.weights()
        g = _flat([torch.zeros_like(p) if x is None else x for p, x in zip(opt.params, grads)],
                  opt.offsets, self.total)
        has = torch.zeros(self.total, dtype=torch.bool)
        for p, x, at in zip(opt.params, grads, opt.offsets):
            has[at:at + p.numel()] = x is not None
        before = {k: v.clone().cpu() for k, v in opt.state.items()}
        norm = opt.step(grads if given is None else given, global_clip_norm=clip)
        self.t += 1
        assert opt.steps == self.t
        coef = 1.0
        if clip:
            want = float(g.square().sum().sqrt())
            # at most 2^13 additions in 64 bits, in another order
            assert abs(float(norm) - want) <= 2.0 ** -40 * want
            coef = min(1.0, clip / (want + 1e-6))
        b1, b2 = opt.betas
        p1, m1, v1, change = ref.step(p0, g, m0, v0, self.t, opt.lr, b1, b2, opt.eps, self.dec, coef)
        size = opt.lr / (1 - b1 ** self.t) / (v1.sqrt() / math.sqrt(1 - b2 ** self.t) + opt.eps)
        big = (b1 * m0).abs() + ((1 - b1) * g * coef).abs()
        got_m, got_v = self.moments()
        got_p = self.weights()
        s = {k: v.cpu() for k, v in opt.state.items()}
        if opt.state_bits == 32:
            assert ((got_m - m1).abs() <= 5 * U * big)[has].all()
            assert ((got_v - v1).abs() <= 8 * U * v1)[has].all()
            bound = 3 * U * (p0.abs() + change.abs()) + 11 * U * change.abs() + 5 * U * big * size
        else:
            words = ref.random_words(torch.arange(self.total), opt.seed, self.t).view(-1, 256)
            hb = has.view(-1, 256).any(1)
            for name, x, u in (('exp_avg', m1, words & 0xffff), ('exp_rms', v1.sqrt(), words >> 16)):
                q, scale = ref.to_codes(x.view(-1, 256), u, name == 'exp_rms')
                assert torch.equal(s[name + '_scale'][hb], scale.view(-1)[hb])
                assert torch.equal(s[name + '8'].double().view(-1, 256)[hb], q[hb])
            bound = 3 * U * (p0.abs() + change.abs()) + 8 * U * change.abs()
        # below 2^-126 fp32 has steps of 2^-149 whatever the value: in m, times what it is multiplied by,
        # in the quotient, times the step size, and in the result
        bound = bound + 2.0 ** -149 * (size + opt.lr / (1 - b1 ** self.t) + 1)
        assert ((got_p - p1).abs() <= bound)[has].all()
        # what has no gradient, and what lies between tensors, is as it was
        for k, v in s.items():
            keep = ~has if v.numel() == self.total else ~has.view(-1, 256).any(1)
            inside = (self.inside if v.numel() == self.total else self.inside.view(-1, 256).any(1))
            assert torch.equal(v.view(torch.uint8).view(v.numel(), -1)[keep & inside],
                               before[k].view(torch.uint8).view(v.numel(), -1)[keep & inside]), k
            assert (v.float()[~inside] == 0).all(), k
        if 'master' in s:
            for p, at in zip(opt.params, opt.offsets):
                w = s['master'][at:at + p.numel()].to(p.dtype)
                assert torch.equal(p.cpu().reshape(-1), w)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('shift,clip', [(0, None), (1, 0.5), (3, 1e6)])
def test_steps_against_the_formula(device, bits, dtype, shift, clip):
    from tracevae_amd.optim import AdamW
    params = _params(ODD, dtype, device, 1, shift)
    decay = [0.1 * (i % 3) for i in range(len(params))]
    opt = AdamW(params, weight_decay=decay, state_bits=bits, seed=12345, **HYPER)
    twin = Twin(opt, decay)
    around = [p.clone() for p in params]
    for k in range(3):
        twin.step(_grads(params, 10 + k), clip)
    assert any(not torch.equal(a, b) for a, b in zip(around, params))


@pytest.mark.parametrize('bits', [32, 8])
def test_steps_with_and_without_clipping_in_turn(device, bits):
    """A step without norm and guard over few tensors is one launch that counts by itself; others count in
    a launch of their own: in turn, and with a tensor list too long for the first kind."""
    from tracevae_amd.optim import AdamW
    for shapes in (ODD, ODD + [(1024 * 4096 + 5,)]):
        params = _params(shapes, torch.float32, device, 41)
        opt = AdamW(params, weight_decay=0.01, state_bits=bits, **HYPER)
        twin = Twin(opt, [0.01] * len(shapes))
        guard = torch.zeros(1, device=device)
        for k, clip in enumerate([None, 0.5, None, None, 2.0, None]):
            twin.step(_grads(params, 42 + k), clip)
            if k == 2:
                opt.step([None] * len(shapes), None, guard, 1)
                opt.step([None] * len(shapes))
                twin.t += 2


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('chunks', [64, 65, 127, 128, 129])
def test_around_the_one_launch_limit(device, bits, chunks):
    """Up to 128 chunks an unclipped step is one launch whose last workgroup counts it: against the formula, and
    captured and replayed against eager steps."""
    from tracevae_amd.optim import AdamW
    shapes = [(4096 * (chunks - 3) - 5,), (100,), (4097,)]
    params = _params(shapes, torch.float32, device, 71)
    opt = AdamW(params, weight_decay=0.01, state_bits=bits, **HYPER)
    twin = Twin(opt, [0.01] * 3)
    for k in range(3):
        twin.step(_grads(params, 72 + k))
    copies = [p.clone() for p in params]
    other = AdamW(copies, weight_decay=0.01, state_bits=bits, **HYPER)
    other.load_state_dict(opt.state_dict())
    g = _grads(params, 75)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(g)
    for k in range(3):
        for x, y in zip(g, _grads(params, 76 + k)):
            x.copy_(y)
        graph.replay()
        other.step(g)
        assert opt.steps == other.steps == 4 + k
        for a, b in zip([*params, *opt.state.values()], [*copies, *other.state.values()]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize('bits', [32, 8])
def test_eps_of_zero_leaves_the_padding_zero(device, bits):
    from tracevae_amd.optim import AdamW
    params = _params([(255,), (3, 5), (1,), (4097,)], torch.bfloat16, device, 31)
    opt = AdamW(params, weight_decay=0.0, state_bits=bits, lr=1e-2, eps=0.0)
    twin = Twin(opt, [0.0] * 4)
    for k in range(2):
        twin.step([torch.where(x.abs() < 1e-6, torch.full_like(x, 1e-3), x) for x in _grads(params, 32 + k)])
    assert all(torch.isfinite(p).all() for p in params)


@pytest.mark.parametrize('bits', [32, 8])
def test_tensors_without_gradient_and_strided_gradients(device, bits):
    from tracevae_amd.optim import AdamW
    params = _params([(30, 40), (5,), (300,), (17, 2)], torch.float32, device, 2)
    opt = AdamW(params, weight_decay=0.1, state_bits=bits, **HYPER)
    twin = Twin(opt, [0.1] * 4)
    g = _grads(params, 3)
    twin.step([g[0], None, g[2], g[3]], 1.0)
    # a transposed gradient, a broadcast one, a column of a wider buffer
    g = _grads(params, 4)
    wide = torch.zeros(300, 3, device=device)
    wide[:, 1] = g[2]
    given = [g[0].t().contiguous().t(), torch.full((1,), 0.25, device=device).expand(5), wide[:, 1], g[3]]
    twin.step([given[0], given[1], given[2], None], 1.0)
    twin.step([None] * 4)
    twin.step([None] * 4, 1.0)


@pytest.mark.parametrize('bits', [32, 8])
def test_gradients_with_the_sign_pending(device, bits):
    from tracevae_amd.optim import AdamW
    params = _params([(300,), (1,)], torch.float32, device, 61)
    opt = AdamW(params, weight_decay=0.01, state_bits=bits, **HYPER)
    twin = Twin(opt, [0.01] * 2)
    g = _grads(params, 62)
    given = [torch._neg_view(-g[0]), torch.complex(torch.zeros_like(g[1]), -g[1]).conj().imag]
    assert all(x.is_neg() for x in given)
    twin.step(g, 1.0, given)
    with pytest.raises(ValueError):
        AdamW([torch._neg_view(torch.ones(5, device=device))])
    params[0].data = torch._neg_view(torch.ones(300, device=device))
    if params[0].is_neg():
        with pytest.raises(TypeError):
            opt.step(g)


@pytest.mark.parametrize('bits', [32, 8])
def test_zero_gradients_without_memory(device, bits):
    """autograd's zeros, whose address is null, are a gradient of zeros and not the absence of one."""
    from tracevae_amd.optim import AdamW
    params = _params([(300,), (17, 3)], torch.bfloat16, device, 67)
    opt = AdamW(params, weight_decay=0.01, state_bits=bits, **HYPER)
    twin = Twin(opt, [0.01] * 2)
    twin.step(_grads(params, 68))
    for k, clip in enumerate((None, 1.0)):
        g = [torch.zeros_like(params[0]), _grads(params, 69 + k)[1]]
        twin.step(g, clip, [torch._efficientzerotensor((300,), dtype=torch.bfloat16, device=device), g[1]])


@pytest.mark.parametrize('bits', [32, 8])
def test_more_tensors_than_one_launch_takes(device, bits):
    from tracevae_amd.optim import AdamW
    shapes = [(1 + (i * 37) % 300,) for i in range(900)] + [(5000,)]
    params = _params(shapes, torch.float32, device, 5, 1)
    opt = AdamW(params, weight_decay=0.0, state_bits=bits, **HYPER)
    twin = Twin(opt, [0.0] * len(shapes))
    for k in range(2):
        twin.step(_grads(params, 6 + k), 0.3)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
def test_infinite_and_nan_gradients_stay_where_they_are(device, bits, bad):
    from tracevae_amd.optim import AdamW
    params = _params([(1000,)], torch.float32, device, 7)
    clean = [p.clone() for p in params]
    opt = AdamW(params, state_bits=bits, **HYPER)
    other = AdamW(clean, state_bits=bits, **HYPER)
    g = _grads(params, 8)
    h = [x.clone() for x in g]
    for i in (0, 300, 999):
        g[0][i] = bad
        h[0][i] = 0.0
    for _ in range(2):
        opt.step(g)
        other.step(h)
    p, q = params[0].cpu(), clean[0].cpu()
    hit = torch.zeros(1000, dtype=torch.bool)
    hit[[0, 300, 999]] = True
    assert torch.isnan(p[hit]).all()
    assert torch.equal(p[~hit], q[~hit])
    # a NaN norm makes everything NaN, as the formula says; an infinite one leaves NaN where the
    # infinite gradient was and no gradient elsewhere
    opt.step(g, global_clip_norm=1.0)
    if math.isnan(bad):
        assert torch.isnan(params[0]).all()
    else:
        assert torch.isfinite(params[0].cpu()[~hit]).all()


@pytest.mark.parametrize('bits', [32, 8])
def test_extreme_gradients(device, bits):
    """All zero, the smallest and large fp32 magnitudes in one block or each in its own."""
    from tracevae_amd.optim import AdamW
    params = _params([(256,), (256,), (256,), (512,)], torch.float32, device, 9)
    opt = AdamW(params, weight_decay=0.01, state_bits=bits, **HYPER)
    g = [torch.zeros(256, device=device), torch.full((256,), 1e-42, device=device),
         torch.full((256,), 1e15, device=device), torch.randn(512, device=device)]
    g[3][0], g[3][1], g[3][2] = 1e15, 1e-30, 0.0
    before = [p.clone() for p in params]
    for _ in range(3):
        opt.step(g)
        for p in params:
            assert torch.isfinite(p).all()
    # |change| <= lr (1 + u..) / keeps its sign: Adam's first steps move by lr whatever the size
    assert torch.allclose(params[0], before[0] * (1 - 1e-2 * 0.01) ** 3, rtol=1e-6, atol=0)
    moved = (params[2] - before[2] * (1 - 1e-2 * 0.01) ** 3)
    assert ((moved + 3e-2).abs() < 3e-2 * 0.15).all()       # 8 bits: m and r are within 1/8 of theirs


@pytest.mark.parametrize('dtype,size', [(torch.float32, 1e38), (torch.float32, 3e38), (torch.bfloat16, 2e38)])
def test_the_largest_gradients(device, dtype, size):
    """A first step moves every parameter by lr, whatever the gradient is: 8 u of it (1 / v_rcp), m, r and the
    constants 4 u more, less than 16 u."""
    from tracevae_amd.optim import AdamW
    p = torch.zeros(600, dtype=dtype, device=device)
    g = torch.full((600,), size, device=device).to(dtype)
    g[::2] *= -1
    g[100:300] *= 1e-3
    opt = AdamW([p], weight_decay=0.0, state_bits=8, **HYPER)
    opt.step([g])
    w = opt.state['master'][:600] if 'master' in opt.state else p
    want = -1e-2 * torch.sign(g).double()
    assert ((w.double() - want).abs() <= 16 * U * 1e-2).all()


def test_the_smallest_gradients_without_eps(device):
    """m = 1e-39 and r = 3.2e-40 lie among fp32's numbers with steps of 2^-149: half a step is 2^-150 / 3.2e-40,
    2.3e-6, of r, and 7e-7 of m, 7e-8 of their quotient's divisor."""
    from tracevae_amd.optim import AdamW
    p = torch.zeros(600, device=device)
    g = torch.full((600,), 1e-38, device=device)
    g[::2] *= -1
    g[100:300] = 1e-3
    opt = AdamW([p], lr=1e-2, weight_decay=0.0, eps=0.0, state_bits=8)
    opt.step([g])
    assert ((p.double() + 1e-2 * torch.sign(g).double()).abs() <= 1e-2 * 4e-6).all()


def test_codes_of_tiny_and_mixed_magnitudes(device):
    """Blocks from 1e-36 to 1e15 in size, each with elements over 12 decades, zeros among them, and blocks
    of nothing but zeros: codes and scales equal to the definition's."""
    from tracevae_amd.optim import AdamW
    gen = torch.Generator().manual_seed(3)
    params = [torch.zeros(200, 256, device=device), torch.zeros(300, device=device)]
    opt = AdamW(params, weight_decay=0.0, state_bits=8, seed=9, **HYPER)
    twin = Twin(opt, [0.0, 0.0])
    for k in range(3):
        size = 10.0 ** torch.linspace(-36, 15, 200).view(-1, 1)
        g = torch.randn(200, 256, generator=gen) * size * 10.0 ** (-12 * torch.rand(200, 256, generator=gen))
        g[torch.rand(200, 256, generator=gen) < 0.2] = 0.0
        g[::7] = 0.0
        twin.step([g.to(device), torch.zeros(300, device=device)])


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('kind,value,skipped', [(1, math.nan, True), (1, 3.0, False), (2, 1.0, True),
                                                (2, 0.0, False)])
def test_guarded_step(device, bits, kind, value, skipped):
    from tracevae_amd.optim import AdamW
    params = _params([(700,)], torch.bfloat16, device, 11)
    opt = AdamW(params, state_bits=bits, **HYPER)
    opt.step(_grads(params, 12))
    before = dict(opt.state_dict(), p=params[0].clone())
    guard = torch.tensor([value], device=device)
    host = torch.zeros(1, pin_memory=True)
    opt.step(_grads(params, 13), 1.0, guard, kind, host)
    torch.cuda.synchronize()
    assert np.array_equal(host.numpy(), np.float32([value]), equal_nan=True)
    after = dict(opt.state_dict(), p=params[0].clone())
    assert after['step'] == (1 if skipped else 2)
    assert torch.equal(before['p'], after['p']) == skipped
    for k in before:
        # (a step that is taken may leave all codes of sqrt(v) where they were: without a gradient it
        # falls by 0.05 %, a code is up to 12 % wide)
        if skipped and k != 'step':
            assert torch.equal(before[k].view(torch.uint8), after[k].view(torch.uint8)), k


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('clip', [1.0, None])
def test_captured_step_counts_on(device, bits, clip):
    """One captured step, replayed with eager work of its own between the replays and another
    learning rate for the last ones, against an eager twin: equal bits after every replay."""
    from tracevae_amd.optim import AdamW
    params = _params(ODD, torch.bfloat16, device, 14, 1)
    twins = [p.clone() for p in params]
    opt = AdamW(params, state_bits=bits, **HYPER)
    eager = AdamW(twins, state_bits=bits, **HYPER)
    g = _grads(params, 15)
    opt.step(g, clip)
    eager.step(g, clip)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(g, clip)
    assert opt.steps == 1                                 # capturing runs nothing
    for k in range(5):
        for x, y in zip(g, _grads(params, 20 + k)):
            x.copy_(y)
        if k == 3:
            opt.set_lr(3e-3)
            eager.set_lr(3e-3)
        graph.replay()
        junk = torch.randn(1000, device=device).sum().item()
        assert math.isfinite(junk)
        eager.step(g, clip)
        assert opt.steps == eager.steps == k + 2
        for a, b in zip(params, twins):
            assert torch.equal(a, b)
        for name in opt.state:
            assert torch.equal(opt.state[name].view(torch.uint8), eager.state[name].view(torch.uint8))


def test_state_dict_continues_bit_for_bit(device):
    from tracevae_amd.hip import HipLibraryError
    from tracevae_amd.optim import AdamW
    for bits in (32, 8):
        params = _params(ODD, torch.float16, device, 16)
        opt = AdamW(params, state_bits=bits, seed=3, **HYPER)
        opt.step(_grads(params, 17))
        saved = copy.deepcopy({k: (v.cpu() if torch.is_tensor(v) else v) for k, v in opt.state_dict().items()})
        copies = [p.clone() for p in params]
        again = AdamW(copies, state_bits=bits, seed=3, **HYPER)
        again.load_state_dict(saved)
        for k in range(2):
            opt.step(_grads(params, 18 + k), 1.0)
            again.step(_grads(params, 18 + k), 1.0)
        for a, b in zip(params, copies):
            assert torch.equal(a, b)
        with pytest.raises(ValueError):
            AdamW(copies, state_bits=40 - bits, **HYPER).load_state_dict(saved)
        with pytest.raises(ValueError):
            AdamW(copies[:3], state_bits=bits, **HYPER).load_state_dict(saved)
        with pytest.raises(HipLibraryError):
            again.load_state_dict(dict(saved, step=-1))
        assert again.steps == 3
        for k in opt.state:
            assert torch.equal(opt.state[k].view(torch.uint8), again.state[k].view(torch.uint8))


def test_a_state_of_another_seed_is_refused(device):
    from tracevae_amd.optim import AdamW

    def make(seed, bits=8):
        return AdamW([torch.ones(300, device=device)], state_bits=bits, seed=seed, **HYPER)

    a = make(2 ** 40 + 5)
    a.step([torch.randn(300, device=device)])
    state = a.state_dict()
    for seed in (5, 2 ** 32 + 5):                         # (the low 32 bits are the seed)
        b = make(seed)
        b.load_state_dict(state)
        assert b.steps == 1
    b = make(6)
    before = b.state_dict()
    with pytest.raises(ValueError, match='seed'):
        b.load_state_dict(state)
    for k, v in b.state_dict().items():
        assert v == 0 if k == 'step' else torch.equal(v.view(torch.uint8), before[k].view(torch.uint8))
    del state['seed']                                     # one that names none is taken
    b.load_state_dict(state)
    assert b.steps == 1 and set(make(1, 32).state_dict()) == {'exp_avg', 'exp_avg_sq', 'step'}


def test_a_captured_learning_rate(device):
    """A rate whose store was captured is set by every replay; set_lr to the rate before is a store again."""
    from tracevae_amd.optim import AdamW
    params = _params([(600,)], torch.float32, device, 63)
    opt = AdamW(params, weight_decay=0.01, **HYPER)
    twin = Twin(opt, [0.01])
    twin.step(_grads(params, 64))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.set_lr(1e-3)
    for lr in (1e-2, 1e-3):
        opt.set_lr(lr)
        twin.step(_grads(params, 65))
        graph.replay()
        opt.set_lr(lr)
        twin.step(_grads(params, 66))


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('how', ['deepcopy', 'save'])
def test_a_copy_of_an_optimizer_stands_alone(device, bits, how):
    """The copy has parameters, state and addresses of its own: it steps on when the original is gone, and
    leaves the original as it was."""
    import gc
    import io
    from tracevae_amd.optim import AdamW
    params = _params(ODD, torch.bfloat16, device, 85)
    opt = AdamW(params, weight_decay=0.1, state_bits=bits, seed=3, **HYPER)
    opt.step(_grads(params, 86), 1.0)
    opt.set_lr(5e-3)
    if how == 'deepcopy':
        twin = copy.deepcopy(opt)
    else:                                         # (plain pickle does not take torch's 8-bit tensors back)
        file = io.BytesIO()
        torch.save(opt, file)
        file.seek(0)
        twin = torch.load(file, weights_only=False)
    at = {x.data_ptr() for x in [*params, *opt.state.values(), opt._plan, opt.grad_norm] if x.numel()}
    mine = [x for x in [*twin.params, *twin.state.values(), twin._plan, twin.grad_norm] if x.numel()]
    assert not at & {x.data_ptr() for x in mine}
    kept = [x.clone() for x in [*params, *opt.state.values()]]
    twin.step(_grads(params, 87))
    for a, b in zip([*params, *opt.state.values()], kept):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert opt.steps == 1 and twin.steps == 2
    for k, clip in enumerate((None, 1.0, None)):
        opt.step(_grads(params, 87 + k), clip)
    want = [x.clone() for x in [*params, *opt.state.values()]]
    del opt, params, kept
    gc.collect()
    for k, clip in ((1, 1.0), (2, None)):
        twin.set_lr(5e-3)
        twin.step(_grads(twin.params, 87 + k), clip)
    for a, b in zip([*twin.params, *twin.state.values()], want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert twin.steps == 4


def test_the_master_follows_a_weight_that_was_written(device):
    from tracevae_amd.optim import AdamW
    for bits in (32, 8):
        params = _params([(600,), (40,)], torch.bfloat16, device, 21)
        opt = AdamW(params, weight_decay=0.0, state_bits=bits, **HYPER)
        opt.step(_grads(params, 22))
        params[0].data.copy_(torch.linspace(-3, 3, 600).to(torch.bfloat16))     # a loaded checkpoint
        want = params[0].clone()
        g = [torch.zeros_like(p) for p in params]
        opt.state['exp_avg' if bits == 32 else 'exp_avg_scale'].zero_()
        opt.step(g)
        assert torch.equal(params[0], want)
        assert torch.equal(opt.state['master'][:600].cpu(), want.float().cpu())


def test_a_moved_parameter_is_found(device):
    from tracevae_amd.optim import AdamW
    params = _params([(600,)], torch.float32, device, 23)
    twins = [p.clone() for p in params]
    opt, other = AdamW(params, **HYPER), AdamW(twins, **HYPER)
    for k in range(2):
        opt.step(_grads(params, 24 + k))
        other.step(_grads(params, 24 + k))
        old = params[0].data
        params[0].set_(params[0].clone())
        assert params[0].data_ptr() != old.data_ptr()
        assert torch.equal(params[0], twins[0])


@pytest.mark.parametrize('bits', [32, 8])
def test_the_plan_of_a_captured_step_outlives_a_move(device, bits):
    """An eager step over a parameter that has moved makes a new plan; a captured one goes on with the plan that
    it was captured with, over the tensor that was there."""
    import weakref
    from tracevae_amd.optim import AdamW
    params = _params(ODD, torch.float32, device, 81)
    opt = AdamW(params, state_bits=bits, **HYPER)
    g = _grads(params, 82)
    opt.step(g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(g)
    plan, image = weakref.ref(opt._plan), opt._plan.clone()
    first = params[0].data
    for _ in range(3):
        params[0].set_(params[0].clone())
        opt.step(g)
        junk = [torch.full_like(image, -1) for _ in range(4)]       # takes what was freed
    assert plan() is not None and torch.equal(plan(), image)
    assert opt._plan is not plan() and all(x.data_ptr() != plan().data_ptr() for x in junk)
    for k in range(2):
        here, there = params[0].clone(), first.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(params[0], here) and not torch.equal(first, there)
        assert opt.steps == 5 + k
    assert torch.isfinite(first).all() and len(opt._captured_plans) == 1


def test_a_changed_list_of_parameters_is_refused(device):
    from tracevae_amd.optim import AdamW
    params = _params([(600,), (5,)], torch.float32, device, 83)
    opt = AdamW(params, **HYPER)
    for change in (lambda: opt.params.append(params[0]), lambda: opt.params.clear()):
        keep = list(opt.params)
        change()
        with pytest.raises(ValueError, match='made for 2'):
            opt.step([None] * len(opt.params))
        opt.params[:] = keep
    opt.step(_grads(params, 84))
    assert opt.steps == 1


def test_on_a_stream_of_its_own(device):
    from tracevae_amd.optim import AdamW
    params = _params([(100000,)], torch.float32, device, 26)
    twins = [p.clone() for p in params]
    opt, other = AdamW(params, state_bits=8, **HYPER), AdamW(twins, state_bits=8, **HYPER)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for k in range(3):
            opt.step([x for x in _grads(params, 27 + k)], 1.0)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        other.step(_grads(twins, 27 + k), 1.0)
    assert torch.equal(params[0], twins[0])


def test_codes_keep_the_value_on_average(device):
    """4096 blocks of the same 256 values: the mean code of each value lies within 6 standard errors
    of the value (a code is one of two neighbours, `gap` apart, so its deviation is at most gap / 2;
    6 sigma over 512 checks fails once in 10^6 even for an unlucky seed, and the seed is fixed)."""
    from tracevae_amd.optim import AdamW
    blocks = 4096
    g = torch.Generator().manual_seed(1)
    row = torch.randn(256, generator=g) * torch.exp(2 * torch.randn(256, generator=g))
    params = [torch.zeros(blocks, 256, device=device)]
    opt = AdamW(params, state_bits=8, seed=7, **HYPER)
    opt.step([row.to(device).expand(blocks, 256)])
    for name, want in (('exp_avg', 0.1 * row.double()), ('exp_rms', math.sqrt(0.001) * row.double().abs())):
        scale = opt.state[name + '_scale'].cpu().double()
        assert (scale == scale[0]).all()
        q = opt.state[name + '8'].cpu().double().view(blocks, 256)
        y = want / scale[0]
        at = (torch.searchsorted(ref.GRID, y.abs().clamp(max=448.0), right=True) - 1).clamp(max=125)
        gap = ref.GRID[at + 1] - ref.GRID[at]
        off = (q.mean(0) - y).abs()
        if name == 'exp_rms':                 # (a positive rms below the least code is held at it)
            off = off[y >= 2.0 ** -9]
            gap = gap[y >= 2.0 ** -9]
        assert off.numel() > 200
        assert (off <= 6 * gap / 2 / math.sqrt(blocks) + gap * 2.0 ** -16).all()


def test_elements_beyond_32_bits(device):
    """A tensor of 2^32 + 5000 elements (8-bit moments): its last elements, and the first ones, step
    as a small tensor's with the same random words do."""
    from tracevae_amd.optim import AdamW
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip('needs 64 GiB of free GPU memory')
    n = 2 ** 32 + 5000
    p = torch.zeros(n, device=device)
    g = torch.zeros(n, device=device)
    gen = torch.Generator().manual_seed(2)
    ends = [(0, 1000), (2 ** 32 - 1024, 2 ** 32 + 1024), (n - 1000, n)]
    for a, b in ends:
        p[a:b] = torch.randn(b - a, generator=gen).to(device)
        g[a:b] = torch.randn(b - a, generator=gen).to(device)
    opt = AdamW([p], weight_decay=0.1, state_bits=8, seed=5, **HYPER)
    before = [p[a:b].clone() for a, b in ends]
    opt.step([g])
    for (a, b), p0 in zip(ends, before):
        b0, b1 = a // 256, -(-b // 256)
        gx = torch.zeros((b1 - b0) * 256, dtype=torch.float64)
        gx[a - b0 * 256:b - b0 * 256] = g[a:b].cpu().double()
        p1, m1, v1, change = ref.step(p0.cpu().double(), g[a:b].cpu().double(), 0.0,
                                      torch.zeros(b - a).double(), 1, 1e-2, 0.9, 0.999, 1e-8, 0.1, 1.0)
        assert ((p[a:b].cpu().double() - p1).abs()
                <= 3 * U * (p0.cpu().double().abs() + change.abs()) + 8 * U * change.abs()).all()
        words = ref.random_words(torch.arange(b0 * 256, b1 * 256), 5, 1).view(-1, 256)
        q, scale = ref.to_codes((1 - 0.9) * gx.view(-1, 256), words & 0xffff, False)
        got = opt.state['exp_avg8'][b0 * 256:min(b1 * 256, opt.state['exp_avg8'].numel())].cpu().double()
        assert torch.equal(got, q.view(-1)[:got.numel()])
    del p, g, opt
    torch.cuda.empty_cache()


def test_more_chunks_than_one_launch_takes(device):
    """2^33 + 5000 elements (8-bit moments): the elements on both sides of the second launch's beginning."""
    from tracevae_amd.optim import AdamW
    if torch.cuda.mem_get_info()[0] < 112 << 30:
        pytest.skip('needs 112 GiB of free GPU memory')
    n, a, b = 2 ** 33 + 5000, 2 ** 33 - 1024, 2 ** 33 + 1024
    p = torch.zeros(n, device=device)
    g = torch.zeros(n, device=device)
    gen = torch.Generator().manual_seed(4)
    p[a:b] = torch.randn(b - a, generator=gen).to(device)
    g[a:b] = torch.randn(b - a, generator=gen).to(device)
    p[-1] = g[-1] = 1.0
    p0, g0 = p[a:b].cpu().double(), g[a:b].cpu().double()
    opt = AdamW([p], weight_decay=0.1, state_bits=8, seed=5, **HYPER)
    opt.step([g])
    p1, m1, v1, change = ref.step(p0, g0, 0.0, torch.zeros(b - a).double(), 1, 1e-2, 0.9, 0.999, 1e-8, 0.1, 1.0)
    assert ((p[a:b].cpu().double() - p1).abs() <= 3 * U * (p0.abs() + change.abs()) + 8 * U * change.abs()).all()
    words = ref.random_words(torch.arange(a, b), 5, 1).view(-1, 256)
    q, scale = ref.to_codes((1 - 0.9) * g0.view(-1, 256), words & 0xffff, False)
    assert torch.equal(opt.state['exp_avg8'][a:b].cpu().double(), q.view(-1))
    assert float(p[-1]) < 1.0 and opt.steps == 1
    del p, g, opt
    torch.cuda.empty_cache()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_a_large_model_with_32_bit_moments(device, dtype):
    """More than 4096 chunks, where fewer workgroups share a CU, with and without clipping."""
    from tracevae_amd.optim import AdamW
    shapes = [(300,), (4096 * 4096 + 777,), (3, 5)]
    params = _params(shapes, dtype, device, 51)
    opt = AdamW(params, weight_decay=0.1, **HYPER)
    twin = Twin(opt, [0.1] * 3)
    for k, clip in enumerate((1.0, None)):
        twin.step(_grads(params, 52 + k), clip)


def test_refusals(device):
    from tracevae_amd import hip
    from tracevae_amd.optim import AdamW
    p = torch.zeros(10, device=device)
    for bad in (torch.zeros(10), ):
        with pytest.raises(hip.HipLibraryError):
            AdamW([bad])
    with pytest.raises(TypeError):
        AdamW([p.double()])
    with pytest.raises(ValueError):
        AdamW([torch.zeros(4, 6, device=device).t()])
    with pytest.raises(ValueError):
        AdamW([])
    with pytest.raises(ValueError):
        AdamW([p], state_bits=16)
    with pytest.raises(ValueError):
        AdamW([p], weight_decay=[0.1, 0.1])
    with pytest.raises(hip.HipLibraryError, match='overlap'):
        AdamW([p, p])
    buf = torch.zeros(20, device=device)
    with pytest.raises(hip.HipLibraryError, match='overlap'):
        AdamW([buf[:11], buf[10:]])
    for kw in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(lr=-1.0),
               dict(weight_decay=-0.1), dict(lr=math.nan)):
        with pytest.raises(hip.HipLibraryError):
            AdamW([p], **kw)
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.step([])
    for g in (torch.zeros(10, device=device, dtype=torch.bfloat16), torch.zeros(9, device=device),
              torch.zeros(10)):
        with pytest.raises(TypeError):
            opt.step([g])
    with pytest.raises(hip.HipLibraryError):
        opt.step([p.clone()], -1.0)
    for lr in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            opt.set_lr(lr)
    for guard in (torch.zeros(1), torch.zeros(1, device=device, dtype=torch.float64), torch.zeros(2, device=device)):
        with pytest.raises(TypeError):
            opt.step([p.clone()], None, guard, 1)
    for host in (torch.zeros(1, dtype=torch.float64, pin_memory=True), torch.zeros(1, device=device)):
        with pytest.raises(TypeError):
            opt.step([p.clone()], None, torch.zeros(1, device=device), 1, host)
    opt.state['exp_avg'] = torch.zeros(1, device=device)              # (a copy of the dict)
    assert opt.state['exp_avg'].numel() == 256
    q = torch.zeros(10, device=device, requires_grad=True)
    other = AdamW([q])
    q.grad = torch.ones(10, device=device)
    for data in (torch.zeros(10), torch.zeros(11, device=device)):
        keep = q.data
        q.grad = None
        q.data = data
        with pytest.raises(TypeError):
            other.step()
        q.data = keep
    sparse = torch.zeros(10, device=device).to_sparse()
    with pytest.raises(TypeError):
        opt.step([sparse])
    assert other.steps == 0
    with pytest.raises(hip.HipLibraryError):
        opt.step([p.clone()], 1.0, torch.zeros(1, device=device), 1, torch.zeros(1))   # not pinned
    assert opt.steps == 0


@pytest.mark.parametrize('kind', ['adamw', 'adamw8'])
def test_flat_optimizer_takes_adamw(device, kind):
    """`FlatOptimizer(kind=...)` and the same steps of `torch.optim.AdamW` on the CPU: 32-bit moments
    to the fp32 error of three steps, 8-bit ones to the size of their codes (a moment is off by at
    most 1/8, the change then by at most 1/3 of lr in each step)."""
    from helpers import rel_err
    from tracevae_amd.train import FlatOptimizer, FlatParameters
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(30, 50), torch.nn.Linear(50, 7))
    other = copy.deepcopy(net)
    net.to(device)
    flat = FlatParameters(net, tail_prefix='1.')
    opt = FlatOptimizer(flat, kind, weight_decay=0.1)
    opt.set_lr(1e-2)
    ropt = torch.optim.AdamW([{'params': [p for n, p in other.named_parameters() if 'bias' not in n],
                               'weight_decay': 0.1},
                              {'params': [p for n, p in other.named_parameters() if 'bias' in n],
                               'weight_decay': 0.0}], lr=1e-2)
    for step in range(3):
        x = torch.randn(16, 30)
        flat.zero_grad()
        (net(x.to(device)) ** 2).sum().backward()
        opt.step(10.0)
        ropt.zero_grad()
        (other(x) ** 2).sum().backward()
        torch.nn.utils.clip_grad_norm_(other.parameters(), 10.0)
        ropt.step()
    for (n, p), (_, q) in zip(net.named_parameters(), other.named_parameters()):
        if kind == 'adamw':
            assert rel_err(p, q) < 1e-4, n
        else:
            assert float((p.cpu() - q).abs().max()) < 1e-2, n


@pytest.mark.parametrize('kind', ['adamw', 'adamw8'])
def test_trainer_runs_both_phases_with_adamw(device, kind):
    """`--train.optimizer=adamw` / `adamw8` through `Trainer.step`: finite losses, parameters of the
    phase move, the others do not, a NaN step changes nothing."""
    from helpers import make_config, make_flat
    from tracevae_amd.batch import DeviceTraceStore, TraceGraphBatch
    from tracevae_amd.config import parse_flags
    from tracevae_amd.model import TraceVAE
    from tracevae_amd.train import NANLossError, Trainer
    flat, lr = make_flat(16, 30, 12)
    cfg = make_config()
    parse_flags(cfg, [f'--train.optimizer={kind}', '--train.weight_decay=0.05'])
    torch.manual_seed(0)
    vae = TraceVAE(cfg.model, 30, max_node_count=12).to(device)
    trainer = Trainer(vae, cfg, world_size=1)
    store = DeviceTraceStore(flat, lr, 30)
    G = TraceGraphBatch.from_store(store, np.arange(16), 12)
    for latency_only in (False, True):
        trainer.set_phase(latency_only)
        before = trainer.flat.flat.clone()
        for _ in range(2):
            assert math.isfinite(float(trainer.step(G)['loss']))
        trainer.finish()
        tail = trainer.flat.tail_start
        assert not torch.equal(before[tail:], trainer.flat.flat[tail:])
        assert torch.equal(before[:tail], trainer.flat.flat[:tail]) == latency_only
    before = trainer.flat.flat.clone()
    steps = trainer.optimizer.adamw.steps
    bad = trainer.flat.params[next(n for n in trainer.flat.names if n.startswith('latency_vae.'))]
    keep = bad.data.clone()
    with torch.no_grad():
        bad.fill_(math.nan)
    trainer.step(G)
    with pytest.raises(NANLossError):
        trainer.finish()
    with torch.no_grad():
        bad.copy_(keep)
    assert torch.equal(before, trainer.flat.flat) and trainer.optimizer.adamw.steps == steps


def _trainer(flags):
    from helpers import make_config, make_flat
    from tracevae_amd.batch import DeviceTraceStore, TraceGraphBatch
    from tracevae_amd.config import parse_flags
    from tracevae_amd.model import TraceVAE
    from tracevae_amd.train import Trainer
    flat, lr = make_flat(16, 30, 12)
    cfg = make_config()
    parse_flags(cfg, flags)
    torch.manual_seed(0)
    vae = TraceVAE(cfg.model, 30, max_node_count=12).to('cuda')
    trainer = Trainer(vae, cfg, world_size=1)
    return trainer, TraceGraphBatch.from_store(DeviceTraceStore(flat, lr, 30), np.arange(16), 12)


@pytest.mark.parametrize('latency_only', [False, True])
@pytest.mark.parametrize('kind', ['adamw', 'adamw8'])
def test_trainer_decays_in_place_of_the_l2_term(device, kind, latency_only):
    """Loss and gradients are those of a model without the L2 term, and one update is AdamW's on them: clipped
    to 10, biases not decayed."""
    a, G = _trainer([f'--train.optimizer={kind}'])
    b, _ = _trainer(['--train.l2_reg=0'])
    got = []
    for trainer in (a, b):
        trainer.set_phase(latency_only)
        torch.manual_seed(1)
        got.append(trainer.local_gradients(G)['loss'].detach())
    assert torch.equal(got[0], got[1])
    start = a.optimizer.start
    assert torch.equal(a.flat.grad[start:], b.flat.grad[start:])
    assert torch.equal(a.flat.flat, b.flat.flat)
    grad, before = a.flat.grad.cpu().double(), a.flat.flat.cpu().double()
    a.update()
    used = torch.zeros_like(grad)
    decay = torch.zeros_like(grad)
    for n in a.flat.names:
        at, end = a.flat.slices[n][0], a.flat.slices[n][0] + a.flat.params[n].numel()
        if at >= start:
            used[at:end] = 1
            decay[at:end] = 0.0 if 'bias' in n else 0.01
    coef = min(1.0, 10.0 / (float((grad * used).square().sum().sqrt()) + 1e-6))
    p1, m1, v1, change = ref.step(before, grad, torch.zeros_like(grad), torch.zeros_like(grad), 1, a.optimizer.lr,
                                  0.9, 0.999, 1e-8, decay, coef)
    # the bound at the top, with M = |m| in a first step, and the steps of 2^-149 as in Twin.step
    size = a.optimizer.lr / (1 - 0.9) / (v1.sqrt() / math.sqrt(1 - 0.999) + 1e-8)
    bound = 3 * U * (before.abs() + change.abs()) + 16 * U * change.abs() + 2.0 ** -149 * (size + a.optimizer.lr * 10 + 1)
    after = a.flat.flat.cpu().double()
    assert ((after - p1).abs() <= bound)[used > 0].all()
    assert torch.equal(after[used == 0], before[used == 0])
    assert float(change[used > 0].abs().max()) > 0


def test_trainer_refuses_a_regulariser_that_its_optimizer_does_not_use(device):
    from tracevae_amd.train import FlatOptimizer
    for flags, name in ((['--train.optimizer=adamw', '--train.l2_reg=0.001'], 'l2_reg'),
                        (['--train.optimizer=adam', '--train.weight_decay=0.1'], 'weight_decay'),
                        (['--train.weight_decay=0.1'], 'weight_decay')):
        with pytest.raises(ValueError, match=f'does not use train.{name}'):
            _trainer(flags)
    trainer, _ = _trainer(['--train.weight_decay=0', '--train.l2_reg=0.001'])
    assert trainer.l2_reg == 0.001
    with pytest.raises(ValueError, match='no weight decay'):
        FlatOptimizer(trainer.flat, 'adam', weight_decay=0.1)
    assert _trainer(['--train.optimizer=adamw8', '--train.l2_reg=0'])[0].l2_reg is None
