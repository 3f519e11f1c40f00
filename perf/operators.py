"""What the token-table and parameter-update operators are measured on.

Two families of passes:

* `lookup` / `lookup_grad`: rows of an embedding table by token id, times a scale, padding ids giving
  zero rows - and the gradient of the table from the gradient of those rows;
* `adamw`: one AdamW step (decoupled weight decay, optional clipping by the global norm) over many
  tensors at once, the moments in 32 bits or in 8 bits with one scale per block of 256.

`own` false: elementary torch operations.  `own` true: `tracevae_amd.ops.scaled_embedding` and
`tracevae_amd.optim.AdamW`.
"""
import math

import torch

own = False

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
WIDTH = {'f32': 4, 'bf16': 2, 'f16': 2}
BLOCK = 256                       # elements of a tensor that share the scale of their 8-bit moments
F8 = torch.float8_e4m3fn
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
U32 = 0xffffffff


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def listed():
    def lookup(name, op, tokens, vocab, dim, table, out, ids, pad):
        return {'name': name, 'op': op, 'tokens': tokens, 'vocab': vocab, 'dim': dim,
                'table': table, 'out': out, 'ids': ids, 'pad': pad}

    def adamw(name, tensors, size, depth, model, bits, clip, step):
        return {'name': name, 'op': 'adamw', 'tensors': tensors, 'size': size, 'depth': depth,
                'model': model, 'bits': bits, 'clip': clip, 'step': step}

    return [
        # one new token for each of 64 sequences: latency
        lookup('lookup_step', 'lookup', 64, 50001, 1024, 'bf16', 'bf16', 'zipf', 0.0),
        # a batch of prompts padded to one length
        lookup('lookup_prompts', 'lookup', 65536, 100003, 4096, 'bf16', 'bf16', 'zipf', 0.1),
        # the operation embedding of a training batch of 512 traces: 1000 operations, 40 wide
        lookup('grad_operations', 'lookup_grad', 25600, 1000, 40, 'f32', 'f32', 'zipf', 0.0),
        # a ragged batch, odd sizes everywhere
        lookup('grad_odd', 'lookup_grad', 1021, 997, 251, 'f16', 'f16', 'uniform', 0.05),
        # a text batch: an fp32 table that feeds bf16 activations, some tokens far more frequent
        lookup('grad_text', 'lookup_grad', 32768, 50001, 1024, 'f32', 'bf16', 'zipf', 0.1),
        # long batches over few operations: a few rows take most of the sums
        lookup('grad_heavy', 'lookup_grad', 262144, 1000, 512, 'bf16', 'bf16', 'heavy', 0.0),
        # the small heads of the model alone (fine-tuning a head): latency, first step
        adamw('adamw_heads', 'heads', 500, 4, 'f32', 32, 0.0, 0),
        # every parameter of the default model (177 tensors, 14 million values), clipped
        adamw('adamw_model', 'model', 500, 4, 'f32', 32, 10.0, 1000),
        adamw('adamw8_model', 'model', 500, 4, 'f32', 8, 10.0, 1000),
        # a deep network with 16-bit weights and their 32-bit masters
        adamw('adamw_deep', 'blocks', 2048, 6, 'bf16', 32, 1.0, 1000),
        # the same depth with moments in 8 bits, 32-bit weights
        adamw('adamw8_deep', 'blocks', 2048, 6, 'f32', 8, 0.0, 1000),
        # odd sizes: rows of the state that end inside a block, unaligned tensors
        adamw('adamw8_odd', 'odd', 331, 5, 'f16', 8, 1.0, 7),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.random()
    if kind < 0.2:
        dim = log(16, 4096)
        model = rng.choice(['f32', 'bf16', 'f16'])
        return {'op': 'lookup', 'tokens': log(1, 65536), 'vocab': log(100, 100003), 'dim': dim,
                'table': model, 'out': model, 'ids': rng.choice(['zipf', 'uniform']),
                'pad': rng.choice([0.0, 0.1, 0.3])}
    if kind < 0.55:
        tokens, dim = log(16, 262144), log(16, 2048)
        dim = max(8, min(dim, 100_000_000 // tokens))
        table, out = rng.choice([('f32', 'f32'), ('bf16', 'bf16'), ('f16', 'f16'), ('f32', 'bf16')])
        vocab = min(log(50, 100003), 100_000_000 // dim)
        return {'op': 'lookup_grad', 'tokens': tokens, 'vocab': vocab, 'dim': dim, 'table': table,
                'out': out, 'ids': rng.choice(['zipf', 'uniform', 'heavy']),
                'pad': rng.choice([0.0, 0.05, 0.2])}
    tensors = rng.choice(['heads', 'model', 'blocks', 'odd'])
    size = {'heads': log(32, 2000), 'model': log(32, 1000), 'blocks': log(64, 1500),
            'odd': log(33, 900)}[tensors]
    return {'op': 'adamw', 'tensors': tensors, 'size': size, 'depth': rng.randint(1, 6),
            'model': rng.choice(['f32', 'f32', 'bf16', 'f16']), 'bits': rng.choice([8, 32]),
            'clip': rng.choice([0.0, 1.0, 10.0]), 'step': rng.choice([0, 1, 7, 1000, 50000])}


def shapes(case):
    """The tensors of one model, in registration order: (shape, takes weight decay)."""
    n, depth, kind = case['size'], case['depth'], case['tensors']
    if kind == 'heads':           # mean / log-std heads and the small dense layers around z
        one = [((10, 2 * n), True), ((10,), False), ((n, 10), True), ((n,), False)]
        return one * depth
    if kind == 'model':           # GAT stacks, heads, flow and dense layers of the default model
        w = 2 * n
        out = [((1000, 40), True)]
        for _ in range(depth):
            for _ in range(3):
                out += [((w, w), True), ((1, 2, n), True), ((1, 2, n), True), ((w,), False),
                        ((w,), True), ((w,), False)]
            out += [((w, 40), True), ((1, 2, n), True), ((1, 2, n), True), ((w,), False),
                    ((10, w), True), ((10,), False)]
        for _ in range(5):
            out += [((5,), False), ((5,), True), ((64, 5), True), ((64,), False), ((5, 64), True),
                    ((5,), False), ((5, 64), True), ((5,), False), ((10, 10), True)]
        out += [((n, 10), True), ((n,), False), ((n, n), True), ((n,), False),
                ((1280, n), True), ((1280,), False), ((1000, w), True), ((1000,), False),
                ((33, n), True), ((33,), False)]
        return out
    if kind == 'blocks':          # a table and square / wide layers with their norms
        out = [((20011, n), True)]
        for _ in range(depth):
            out += [((n,), False)] + [((n, n), True)] * 4 + [((n,), False), ((4 * n, n), True),
                                                           ((4 * n,), False), ((n, 4 * n), True)]
        return out
    out = []                      # 'odd'
    for i in range(depth):
        out += [((n, n + 2 * i), True), ((n + 2 * i,), False), ((3, n - 2), True), ((1,), False),
                ((2 * n + 1, 17), True), ((255,), False), ((257,), False), ((n, 3 * n), True)]
    return out


def layout(case):
    """[(offset, size, shape, decayed)] of the tensors in buffers where each begins a new block."""
    got, at = [], 0
    for shape, decayed in shapes(case):
        size = math.prod(shape)
        got.append((at, size, shape, decayed))
        at += -(-size // BLOCK) * BLOCK
    return got, at


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _token_inputs(case, seed):
    g = _generator(seed)
    n, v, d = case['tokens'], case['vocab'], case['dim']
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    if case['ids'] == 'uniform':
        rank = (u * v).long()
    elif case['ids'] == 'zipf':                      # frequency falls as 1 / rank
        rank = (float(v) ** u).long() - 1
    else:                                            # half of all tokens are the same three
        rank = torch.where(u < 0.5, (u * 6).long(), ((u - 0.5) * 2 * v).long())
    ids = rank.clamp(0, v - 1) * 7919 % v            # frequent tokens lie apart in the table
    if case['pad']:
        ids = torch.where(torch.rand(n, generator=g, device=DEV) < case['pad'], -1, ids)
    s = {'ids': ids, 'scale': math.sqrt(d),
         'weight': (torch.randn(v, d, generator=g, device=DEV) * 0.02).to(TYPES[case['table']])}
    if case['op'] == 'lookup_grad':
        s['dout'] = (torch.randn(n, d, generator=g, device=DEV) * 1e-2).to(TYPES[case['out']])
    return s


def _adamw_inputs(case, seed):
    g = _generator(seed)
    tensors, total = layout(case)
    blocks = total // BLOCK
    model = TYPES[case['model']]
    inside = torch.zeros(total, dtype=torch.bool, device=DEV)
    decay = torch.zeros(blocks, 1, device=DEV)
    for at, size, _, decayed in tensors:
        inside[at:at + size] = True
        if decayed:
            decay[at // BLOCK:-(-(at + size) // BLOCK)] = DECAY
    inside = inside.view(blocks, BLOCK)

    def normal(spread):           # magnitudes differ from block to block, as layers and rows do
        x = torch.randn(blocks, BLOCK, generator=g, device=DEV)
        return x * torch.exp(spread * torch.randn(blocks, 1, generator=g, device=DEV)) * inside

    # rows of a table that no token of this batch named: no gradient, and some never had one
    touched = (torch.rand(blocks, 1, generator=g, device=DEV) < 0.9).float()
    ever = torch.maximum(touched, (torch.rand(blocks, 1, generator=g, device=DEV) < 0.5).float())
    w = normal(0.3) * 0.02
    s = {'tensors': tensors, 'step': case['step'], 'decay': decay,
         'seed': seed % 65521, 'param': w.to(model).view(-1),
         'grad': (normal(1.0) * 1e-3 * touched).to(model).view(-1)}
    if case['model'] != 'f32':    # the 32-bit master rounds to the weight
        fine = w * (1 + 1e-3 * torch.randn(blocks, BLOCK, generator=g, device=DEV))
        s['master'] = torch.where(fine.to(model) == w.to(model), fine, w.to(model).float()).view(-1)
    if case['step'] == 0:
        m = torch.zeros(blocks, BLOCK, device=DEV)
        r = torch.zeros(blocks, BLOCK, device=DEV)
    else:
        m = normal(1.0) * 3e-4 * ever
        r = (normal(1.0).abs() * 3e-4 + 1.1 * m.abs()) * ever
    if case['bits'] == 32:
        s['exp_avg'], s['exp_avg_sq'] = m.view(-1), (r * r).view(-1)
    else:
        for name, x in (('exp_avg', m), ('exp_rms', r)):
            scale = x.abs().amax(1, keepdim=True) / 448
            s[name + '8'] = torch.where(scale > 0, x / scale, x).clamp(-448, 448).to(F8).view(-1)
            s[name + '_scale'] = scale.view(-1)
    return s


def prepare(case, seed):
    if case['op'] != 'adamw':
        s = _token_inputs(case, seed)
        s['case'] = case
        if case['op'] == 'lookup_grad' and own:
            s['weight'].requires_grad_(True)
        return s
    s = _adamw_inputs(case, seed)
    s['case'] = case
    if own:
        from tracevae_amd.optim import AdamW
        params = []
        for at, size, shape, _ in s['tensors']:
            p = torch.nn.Parameter(s['param'][at:at + size].view(shape))
            p.grad = s['grad'][at:at + size].view(shape)
            params.append(p)
        opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS,
                    weight_decay=[DECAY if d else 0.0 for _, _, _, d in s['tensors']],
                    state_bits=case['bits'], seed=s['seed'])
        names = ('exp_avg', 'exp_avg_sq') if case['bits'] == 32 else \
            ('exp_avg8', 'exp_avg_scale', 'exp_rms8', 'exp_rms_scale')
        if case['model'] != 'f32':
            names += ('master',)
        opt.load_state_dict(dict({k: s.pop(k) for k in names}, step=case['step']))
        return {'case': case, 'opt': opt, 'param': s['param'], 'grad': s['grad']}
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(s):
    case = s['case']
    if case['op'] == 'adamw':
        return _run_adamw(s)
    out_type = TYPES[case['out']]
    if own:
        from tracevae_amd import ops
        out = ops.scaled_embedding(s['weight'], s['ids'], s['scale'], padding_idx=-1,
                                   out_dtype=out_type)
        if case['op'] == 'lookup':
            return out
        return [out.detach(), torch.autograd.grad(out, s['weight'], s['dout'])[0]]
    w, ids = s['weight'], s['ids']
    named = (ids >= 0) & (ids < case['vocab'])
    rows = w[ids.clamp(0, case['vocab'] - 1)].float() * s['scale']
    out = torch.where(named[:, None], rows, 0.0).to(out_type)
    if case['op'] == 'lookup':
        return out
    # rows in the order of their tokens; running sums over them are long: 64 bits
    place, order = torch.where(named, ids, case['vocab']).sort(stable=True)
    bounds = torch.searchsorted(place, torch.arange(case['vocab'] + 1, device=DEV))
    sums = torch.zeros(case['dim'], ids.numel() + 1, dtype=torch.float64, device=DEV)
    torch.cumsum(s['dout'][order].t().double(), 1, out=sums[:, 1:])
    dw = (sums[:, bounds[1:]] - sums[:, bounds[:-1]]).t() * s['scale']
    return [out, dw.to(w.dtype)]


def _run_adamw(s):
    case = s['case']
    if own:
        opt = s['opt']
        norm = opt.step(global_clip_norm=case['clip'] or None)
        out = {'param': s['param'], **{k: v for k, v in opt.state.items() if k != 'step'}}
        if case['clip']:
            out['norm'] = norm
        return out
    out = {'param': s['param']}
    s['step'] += 1
    t, bits = s['step'], case['bits']
    wide = torch.float64 if bits == 8 else torch.float32
    g = s['grad'].view(-1, BLOCK).to(wide)
    if case['clip']:
        out['norm'] = s['grad'].double().square().sum().sqrt()
        g = g * (case['clip'] / (out['norm'] + 1e-6)).clamp(max=1.0).to(wide)
    w = s['param'] if case['model'] == 'f32' else s['master']
    if bits == 32:
        m, v = s['exp_avg'].view(-1, BLOCK), s['exp_avg_sq'].view(-1, BLOCK)
    else:
        # a value next to a border between two codes: 64 bits
        m = s['exp_avg8'].view(-1, BLOCK).double() * s['exp_avg_scale'].view(-1, 1).double()
        r = s['exp_rms8'].view(-1, BLOCK).double() * s['exp_rms_scale'].view(-1, 1).double()
        v = r * r
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    r = v.sqrt()
    step = (m * (LR / (1 - BETA1 ** t)) / (r / math.sqrt(1 - BETA2 ** t) + EPS)).float()
    w.copy_((w.view(-1, BLOCK) * (1 - LR * s['decay']) - step).view(-1))
    if case['model'] != 'f32':
        s['param'].copy_(w)
        out['master'] = w
    if bits == 32:
        s['exp_avg'].copy_(m.view(-1))
        s['exp_avg_sq'].copy_(v.view(-1))
        out.update(exp_avg=s['exp_avg'], exp_avg_sq=s['exp_avg_sq'])
        return out
    bits16 = _random_words(m.numel(), s['seed'], t)
    for name, x, u in (('exp_avg', m, bits16 & 0xffff), ('exp_rms', r, bits16 >> 16)):
        scale = x.abs().amax(1, keepdim=True).float() / 448
        y = x.abs() / torch.where(scale > 0, scale, 1.0).double()
        # the distance between codes around y, then up with the probability of what is left over
        ulp = torch.ldexp(torch.ones_like(y), torch.frexp(y.clamp(min=2.0 ** -6))[1] - 4)
        q = torch.floor(y / ulp + (u.view_as(y).double() + 0.5) / 65536) * ulp
        if name == 'exp_rms':
            q = torch.where(x > 0, q.clamp(min=2.0 ** -9), q)     # a positive rms stays positive
        q = torch.copysign(q.clamp(max=448.0), x).float().to(F8)
        s[name + '8'].copy_(q.view(-1))
        s[name + '_scale'].copy_(scale.view(-1))
        out[name + '8'], out[name + '_scale'] = s[name + '8'], s[name + '_scale']
    return out


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x6a09e667) & U32
    x = x ^ (x >> 15)
    x = (x * 0xbb67ae85) & U32
    return x ^ (x >> 16)


def _random_words(n, seed, step):
    """32 random bits of each element: a hash of (seed, step, index)."""
    i = torch.arange(n, dtype=torch.int64, device=DEV)
    key = _mix((_mix(seed & U32) + step) & U32)
    return _mix(_mix((key + (i >> 32)) & U32) ^ (i & U32))


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    if case['op'] == 'adamw':
        n = sum(math.prod(shape) for shape, _ in shapes(case))
        wide = WIDTH[case['model']]
        weights = 8 if wide == 4 else 8 + wide            # read and written; 16-bit copies written
        moments = 16 if case['bits'] == 32 else 4 + 16 / BLOCK
        return {'bytes': n * (wide + weights + moments), 'flops': n * 14}
    n, v, d = case['tokens'], case['vocab'], case['dim']
    table, out = WIDTH[case['table']], WIDTH[case['out']]
    bytes_ = 8 * n + min(n, v) * d * table + n * d * out
    flops = n * d
    if case['op'] == 'lookup_grad':
        bytes_ += 8 * n + n * d * out + v * d * table
        flops += n * d
    return {'bytes': bytes_, 'flops': flops}


# ---------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    if case['op'] != 'adamw':
        s = _token_inputs(case, seed)
        ids, v = s['ids'], case['vocab']
        # a zero row stands behind the table for every id that names none
        table = torch.cat([s['weight'].double(), torch.zeros(1, case['dim'], device=DEV).double()])
        place = torch.where((ids < 0) | (ids >= v), v, ids)
        out = table.index_select(0, place).mul_(s['scale'])
        if case['op'] == 'lookup':
            return out
        del table
        dw = torch.zeros(v + 1, case['dim'], dtype=torch.float64, device=DEV)
        dw = dw.index_add_(0, place, s['dout'].double())[:v].mul_(s['scale'])
        return [out, dw]
    s = _adamw_inputs(case, seed)
    t = case['step'] + 1
    n = s['param'].numel()
    g = s['grad'].double()
    out = {}
    if case['clip']:
        norm = torch.linalg.vector_norm(g)
        out['norm'] = norm
        if float(norm) + 1e-6 > case['clip']:
            g = g * (case['clip'] / (float(norm) + 1e-6))
    if case['bits'] == 32:
        m, v = s['exp_avg'].double(), s['exp_avg_sq'].double()
    else:
        m = s['exp_avg8'].double() * s['exp_avg_scale'].double().repeat_interleave(BLOCK)
        v = (s['exp_rms8'].double() * s['exp_rms_scale'].double().repeat_interleave(BLOCK)) ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    del g
    w = (s['param'] if case['model'] == 'f32' else s['master']).double()
    w = w - LR * s['decay'].double().view(-1).repeat_interleave(BLOCK) * w
    w = w - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    out['param'] = w
    if case['model'] != 'f32':
        out['master'] = w
    if case['bits'] == 32:
        return {**out, 'exp_avg': m, 'exp_avg_sq': v}
    # every value of the 8-bit type, and the one above it
    grid = torch.arange(127, dtype=torch.uint8, device=DEV).view(F8).double()
    above = torch.cat([grid[1:], grid[-1:]])
    place = torch.arange(n, dtype=torch.int64, device=DEV)
    key = _scramble((_scramble(torch.tensor(s['seed'], device=DEV)) + t) % (1 << 32))
    word = _scramble(_scramble((key + place // (1 << 32)) % (1 << 32)) ^ (place % (1 << 32)))
    for name, x, u in (('exp_avg', m, word % 65536), ('exp_rms', v.sqrt(), word // 65536)):
        scale = x.abs().view(-1, BLOCK).amax(1).float().div(448)
        y = x.abs() / scale.double().repeat_interleave(BLOCK)
        y = torch.nan_to_num(y, nan=0.0).clamp(max=448.0)
        at = torch.searchsorted(grid, y, right=True) - 1
        gap = (above[at] - grid[at]).clamp(min=1e-300)
        up = (y - grid[at]) / gap + (u.double() + 0.5) / 65536 >= 1
        q = torch.where(up, above[at], grid[at])
        if name == 'exp_rms':
            q = torch.where((x > 0) & (q == 0), grid[1], q)
        out[name + '8'] = q * torch.sign(x)
        out[name + '_scale'] = scale.double()
    return out


def _scramble(x):
    """Two rounds of shift and multiply, by the fractional bits of the square roots of 2 and 3."""
    for shift, factor in ((16, 0x6a09e667), (15, 0xbb67ae85)):
        x = ((x ^ (x >> shift)) * factor) % (1 << 32)
    return x ^ (x >> 16)
