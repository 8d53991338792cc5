"""The layer norm and the AdamW step as a user calls them, at sizes of real use, with their plain forms.

``listed()`` names the cases, ``draw(rng)`` makes more of the same ranges, ``prepare`` makes a case's data on the GPU, ``run``
does one pass, ``exact`` says in 64 bits what a pass returns.  ``own`` False: the plain forms, in elementary torch operations;
``own`` True: the framework's calls.

Layer norm over C channels: y = (x - mean) / sqrt(var + eps) * gamma + beta for every token (the last dimension) or every pixel
of an NCHW map in channels_last memory; a training pass returns y and the gradients of x, gamma and beta.

AdamW over the tensors of a model, laid out one after the other with every start rounded up to 4 elements:
  g' = g * min(1, max_norm / (|g| + 1e-6));  m' = b1 m + (1 - b1) g';  v' = b2 v + (1 - b2) g'^2;
  p' = p - lr wd p - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps).
With 8-bit states a tensor's moments are held as e4m3 numbers, 256 to a block, each block with a power of two as its scale (an
exponent byte E, the scale is 2^(E - 127)): m itself, and r = sqrt(v).  E puts the block's largest finite magnitude into
[128, 256).  A magnitude between two e4m3 numbers goes to the upper one if its fraction of the way plus u is 1 or more, u in
[0, 1) from a hash of the element's place, the step and a seed, so that what an average gains in small steps is not lost; r > 0
is held as no less than the smallest code."""
import math

import torch

own = False

A, B, M32 = 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF       # 2^32 / golden ratio, 2^32 * frac(sqrt 3): both odd
TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
GROUPS = ({'lr': 1e-3, 'betas': (0.9, 0.999), 'eps': 1e-8, 'weight_decay': 0.05},       # weights
          {'lr': 2e-3, 'betas': (0.9, 0.99), 'eps': 1e-8, 'weight_decay': 0.0})         # norms and biases
T0 = 200                                                                                # steps taken before the first pass


def listed():
    ln, adam = {'op': 'layer_norm'}, {'op': 'adamw'}
    return [
        # one token through an already trained layer: nothing but latency
        {'name': 'ln 1 token', **ln, 'rows': 1, 'C': 256, 'type': 'float32', 'train': False, 'gap': 0},
        # the 64x48 maps of the first branch of the 32-channel pose net, batch 32: many short rows
        {'name': 'ln map c32', **ln, 'B': 32, 'C': 32, 'H': 64, 'W': 48, 'type': 'float32', 'train': True},
        # the first branch of the 48-channel net at 384x288: a channel count that is no power of two
        {'name': 'ln map c48 bf16', **ln, 'B': 16, 'C': 48, 'H': 96, 'W': 72, 'type': 'bfloat16', 'train': True},
        # 192 patches of 16x16 per 256x192 image, batch 32, as tokens
        {'name': 'ln tokens bf16', **ln, 'rows': 6144, 'C': 768, 'type': 'bfloat16', 'train': True, 'gap': 0},
        # odd everything: a ragged set of tokens, an odd width, rows cut out of a wider tensor
        {'name': 'ln ragged fp16', **ln, 'rows': 1537, 'C': 771, 'type': 'float16', 'train': True, 'gap': 5},
        # evaluation of a wide layer in fp32
        {'name': 'ln eval c2048', **ln, 'rows': 12289, 'C': 2048, 'type': 'float32', 'train': False, 'gap': 0},
        # the widest rows over many tokens
        {'name': 'ln wide bf16', **ln, 'rows': 16384, 'C': 4096, 'type': 'bfloat16', 'train': True, 'gap': 0},
        # a head that is tuned alone
        {'name': 'adamw head', **adam, 'tensors': 6, 'elements': 20011, 'bits': 32, 'clip': False},
        # all of the 32-channel pose net
        {'name': 'adamw w32', **adam, 'tensors': 300, 'elements': 28500000, 'bits': 32, 'clip': False},
        {'name': 'adamw8 w32', **adam, 'tensors': 300, 'elements': 28500000, 'bits': 8, 'clip': False},
        # a small net of odd tensors, clipped
        {'name': 'adamw8 clip odd', **adam, 'tensors': 61, 'elements': 3300007, 'bits': 8, 'clip': True},
        # all of the 48-channel pose net, clipped
        {'name': 'adamw clip w48', **adam, 'tensors': 200, 'elements': 63600000, 'bits': 32, 'clip': True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        kind, train = rng.choice(sorted(TYPES)), rng.random() < 0.7
        room = (1 << 25 if kind == 'float32' else 1 << 26) // (1 if train else 2)      # elements
        if rng.random() < 0.4:
            C, H, W = _log(rng, 16, 512), rng.randint(1, 96), rng.randint(1, 72)
            return {'op': 'layer_norm', 'B': _log(rng, 1, max(1, min(64, room // (C * H * W)))), 'C': C, 'H': H, 'W': W,
                    'type': kind, 'train': train}
        C = _log(rng, 1, 16384)
        return {'op': 'layer_norm', 'rows': _log(rng, 1, max(1, min(100000, room // C))), 'C': C, 'type': kind, 'train': train,
                'gap': rng.choice((0, 0, 1, 8))}
    tensors = _log(rng, 1, 300)
    return {'op': 'adamw', 'tensors': tensors, 'elements': _log(rng, 1000, 60000000), 'bits': rng.choice((32, 8)),
            'clip': rng.random() < 0.5}


def _sizes(case):
    """Elements of every tensor, three decades apart, the large ones (group 0) first; the rest are group 1."""
    T, N = case['tensors'], case['elements']
    w = [2.0 ** (-10.0 * ((i * 0.6180339887) % 1.0)) for i in range(T)]
    n = [max(1, int(N * x / sum(w))) for x in w]
    big = [s for s in n if s * 8 * T >= N]
    return big, [s for s in n if s * 8 * T < N]


def _ends(sizes):
    """(first element of each tensor, elements of the whole layout)"""
    at, total = [], 0
    for s in sizes:
        at.append(total)
        total += (s + 3) // 4 * 4
    return at, total


def _norm_inputs(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    kind, C = TYPES[case['type']], case['C']
    rand = lambda *shape: torch.randn(*shape, device='cuda', generator=g)          # noqa: E731
    if 'H' in case:
        shape = (case['B'], case['H'], case['W'], C)
        x = ((rand(*shape) + 0.5) * (0.5 + rand(C).abs())).to(kind).permute(0, 3, 1, 2)
        dy = rand(*shape).to(kind).permute(0, 3, 1, 2)
    else:
        x = ((rand(case['rows'], C + case['gap']) + 0.5) * (0.5 + rand(C + case['gap']).abs())).to(kind)[:, :C]
        dy = rand(case['rows'], C).to(kind)
    return {'case': case, 'x': x, 'dy': dy, 'gamma': 1 + 0.1 * rand(C), 'beta': 0.1 * rand(C)}


def _adam_inputs(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    big, small = _sizes(case)
    sizes = big + small
    at, total = _ends(sizes)
    split = _ends(big)[1]
    starts = torch.tensor(at, device='cuda')
    spans = torch.tensor([b - a for a, b in zip(at, at[1:] + [total])], device='cuda')
    real = torch.tensor(sizes, device='cuda')
    of = torch.repeat_interleave(torch.arange(len(sizes), device='cuda'), spans, output_size=total)      # an element's tensor
    inside = torch.arange(total, device='cuda') - starts[of] < real[of]
    rand = lambda: torch.randn(total, device='cuda', generator=g) * inside          # noqa: E731
    scale = torch.exp(torch.randn(len(sizes), device='cuda', generator=g))[of] * 1e-3
    s = {'case': case, 'sizes': sizes, 'at': at, 'split': split, 'big': len(big), 'seed': seed % 1000, 't': T0,
         'p': 0.05 * rand(), 'g': rand() * scale, 'max_norm': 1e-3 * math.sqrt(case['elements']) if case['clip'] else None}
    m, v = 0.3 * rand() * scale, (rand() * scale) ** 2 + 0.1 * scale ** 2 * inside
    if case['bits'] == 32:
        s['m'], s['v'] = m, v
    else:
        blocks = [(a + k, min(256, n - k)) for a, n in zip(at, sizes) for k in range(0, n, 256)]
        s['first'] = torch.tensor([b[0] for b in blocks], device='cuda')
        s['count'] = torch.tensor([(b[1] + 3) // 4 * 4 for b in blocks], device='cuda')
        u = torch.full((total,), 0.5, device='cuda')
        (s['m'], s['m_scale']), (s['r'], s['r_scale']) = _hold(m, s, u, 0.0), _hold(v.sqrt(), s, u, 2.0 ** -9)
    return s


def prepare(case, seed):
    if case['op'] == 'layer_norm':
        s = _norm_inputs(case, seed)
        if own:
            from advmix_amd import ops
            s['layer_norm'] = ops.layer_norm
            if case['train']:
                s['x'].requires_grad_()
                s['gamma'], s['beta'] = torch.nn.Parameter(s['gamma']), torch.nn.Parameter(s['beta'])
        return s
    s = _adam_inputs(case, seed)
    if own:
        from advmix_amd.utils.utils import FlatAdamW
        parts = lambda t: [t[a:a + n] for a, n in zip(s['at'], s['sizes'])]          # noqa: E731
        params = [torch.nn.Parameter(t) for t in parts(s['p'])]
        for p, g in zip(params, parts(s['g'])):
            p.grad = g
        groups = [dict(GROUPS[0], params=params[:s['big']]), dict(GROUPS[1], params=params[s['big']:])]
        opt = FlatAdamW([g for g in groups if g['params']], state_bits=case['bits'], max_norm=s['max_norm'], seed=s['seed'])
        keys = ('exp_avg', 'exp_avg_sq') if case['bits'] == 32 else ('exp_avg_codes', 'exp_avg_root_codes')
        state = {i: {'step': float(T0), keys[0]: m, keys[1]: v} for i, (m, v) in
                 enumerate(zip(parts(s['m']), parts(s['v' if case['bits'] == 32 else 'r'])))}
        if case['bits'] == 8:
            blocks = [(n + 255) // 256 for n in s['sizes']]
            for i, (m, r) in enumerate(zip(s['m_scale'].split(blocks), s['r_scale'].split(blocks))):
                state[i].update(exp_avg_scale=m, exp_avg_root_scale=r)
        opt.load_state_dict({'state': state, 'param_groups': opt.state_dict()['param_groups']})
        s = {'case': case, 'opt': opt}
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------------
def _norm(s):
    case, dim = s['case'], 1 if 'H' in s['case'] else -1
    x, g, b = s['x'].float(), s['gamma'], s['beta']
    if dim == 1:
        g, b = g.view(-1, 1, 1), b.view(-1, 1, 1)
    d = x - x.mean(dim, keepdim=True)
    inv = 1 / torch.sqrt((d * d).mean(dim, keepdim=True) + 1e-5)
    h = d * inv
    y = (h * g + b).to(s['x'].dtype)
    if not case['train']:
        return y
    dy, rows = s['dy'].float(), (0, 2, 3) if dim == 1 else (0,)
    gh = dy * g
    dx = inv * (gh - gh.mean(dim, keepdim=True) - h * (gh * h).mean(dim, keepdim=True))
    return {'y': y, 'dx': dx.to(s['x'].dtype), 'dgamma': (dy * h).sum(rows), 'dbeta': dy.sum(rows)}


def _mix(x):
    x = x ^ (x >> 15)
    x = (x * B) & M32
    return x ^ (x >> 13)


def _dither(s, n):
    """(u for m, u for r) in [0, 1), 16 bits each, from the place, the step and the seed."""
    key = _mix((s['t'] + _mix((s['seed'] * A) & M32)) & M32)
    x = _mix((torch.arange(n, device='cuda') * A + key) & M32)
    return (x >> 16).float() / 65536, (x & 0xFFFF).float() / 65536


def _block_of(s, n):
    return torch.repeat_interleave(torch.arange(s['first'].numel(), device='cuda'), s['count'], output_size=n)


def _held(codes, scale, s):
    """What the codes stand for, in 32 bits."""
    return codes.float() * torch.exp2(scale.view(torch.uint8).float() - 127)[_block_of(s, codes.numel())]


def _hold(x, s, u, least):
    """(codes, scales) of x."""
    n, a = x.numel(), x.abs()
    at = s['first'][:, None] + torch.arange(256, device='cuda')
    inside = torch.arange(256, device='cuda') < s['count'][:, None]
    top = (a[at.clamp(max=n - 1)] * inside).amax(1)
    E = ((torch.frexp(top)[1] - 1 - 7 + 127).clamp(0, 254) * (top > 0)).to(torch.int32)
    z = a * torch.exp2(127 - E.float())[_block_of(s, n)]
    q = torch.exp2((torch.frexp(z)[1] - 1 - 3).clamp(min=-9).float())
    z = torch.floor(z / q + u) * q
    z = torch.where(a > 0, z.clamp(min=least), z) if least else z
    return torch.copysign(z, x).to(torch.float8_e4m3fn), E.to(torch.uint8).view(torch.float8_e8m0fnu)


def _step(s):
    case, p, g, split = s['case'], s['p'], s['g'], s['split']
    s['t'] += 1
    if s['max_norm'] is not None:
        norm = g.double().square().sum().sqrt()
        g = g * (s['max_norm'] / (norm + 1e-6)).clamp(max=1.0).float()
    if case['bits'] == 32:
        m, v = s['m'], s['v']
    else:
        m, v = _held(s['m'], s['m_scale'], s), _held(s['r'], s['r_scale'], s).square()
    new = [_group(GROUPS[k], s['t'], *(t[cut] for t in (p, g, m, v))) for k, cut in enumerate((slice(0, split), slice(split, None)))]
    p.copy_(torch.cat([x[0] for x in new]))
    m, v = (torch.cat([x[k] for x in new]) for k in (1, 2))
    if case['bits'] == 32:
        s['m'].copy_(m)
        s['v'].copy_(v)
        return {'p': p, 'm': s['m'], 'v': s['v']}
    um, ur = _dither(s, p.numel())
    (s['m'], s['m_scale']), (s['r'], s['r_scale']) = _hold(m, s, um, 0.0), _hold(v.sqrt(), s, ur, 2.0 ** -9)
    return {'p': p, 'm': s['m'], 'm_scale': s['m_scale'], 'r': s['r'], 'r_scale': s['r_scale']}


def _group(h, t, p, g, m, v):
    b1, b2 = h['betas']
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    upd = m / (v.sqrt() * (1 / math.sqrt(1 - b2 ** t)) + h['eps'])
    return p - p * (h['lr'] * h['weight_decay']) - upd * (h['lr'] / (1 - b1 ** t)), m, v


def run(s):
    case = s['case']
    if not own:
        return _norm(s) if case['op'] == 'layer_norm' else _step(s)
    if case['op'] == 'layer_norm':
        if not case['train']:
            return s['layer_norm'](s['x'], s['gamma'], s['beta'], eps=1e-5)
        x, gamma, beta = s['x'], s['gamma'], s['beta']
        x.grad = gamma.grad = beta.grad = None
        y = s['layer_norm'](x, gamma, beta, eps=1e-5)
        y.backward(s['dy'])
        return {'y': y, 'dx': x.grad, 'dgamma': gamma.grad, 'dbeta': beta.grad}
    opt = s['opt']
    opt.step()
    if case['bits'] == 32:
        p, m, v = opt.flat_state()[:3]
        return {'p': p, 'm': m, 'v': v}
    p, m, r, _, m_scale, r_scale = opt.flat_state()
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    return {'p': p, 'm': m.view(f8), 'm_scale': m_scale.view(e8), 'r': r.view(f8), 'r_scale': r_scale.view(e8)}


def work(case):
    if case['op'] == 'layer_norm':
        C = case['C']
        n = case['B'] * C * case['H'] * case['W'] if 'H' in case else case['rows'] * C
        size = 4 if case['type'] == 'float32' else 2
        if case['train']:                                 # x and dy in, y and dx out; gamma, beta and their gradients
            return {'bytes': 4 * n * size + 4 * C * 4, 'flops': 22 * n}
        return {'bytes': 2 * n * size + 2 * C * 4, 'flops': 8 * n}
    n = sum(sum(x) for x in _sizes(case))
    each = 28 if case['bits'] == 32 else 16 + 4 / 256     # p, m, v in and out, g in
    return {'bytes': each * n, 'flops': (15 if case['bits'] == 32 else 30) * n + (2 * n if case['clip'] else 0)}


# ---- in 64 bits -----------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case['op'] == 'layer_norm':
        s = _norm_inputs(case, seed)
        C = case['C']
        rows = lambda t: (t.permute(0, 2, 3, 1) if 'H' in case else t).double().reshape(-1, C)          # noqa: E731
        back = lambda t: t.view(case['B'], case['H'], case['W'], C).permute(0, 3, 1, 2) if 'H' in case else t          # noqa: E731
        x, dy, w, b = rows(s['x']), rows(s['dy']), s['gamma'].double(), s['beta'].double()
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        sd = torch.sqrt(var + 1e-5)
        xh = (x - mean) / sd
        y = torch.addcmul(b, xh, w)
        if not case['train']:
            return back(y)
        t = dy * w
        dots = (torch.einsum('ij,ij->i', t, xh) / C)[:, None]
        return {'y': back(y), 'dx': back((t - t.sum(1, keepdim=True) / C - xh * dots) / sd), 'dgamma': (dy * xh).sum(0), 'dbeta': dy.sum(0)}
    s = _adam_inputs(case, seed)
    n, t = s['p'].numel(), T0 + 1
    second = torch.arange(n, device='cuda') >= s['split']
    pick = lambda f: torch.where(second, torch.tensor(f(GROUPS[1]), device='cuda', dtype=torch.float64), f(GROUPS[0]))          # noqa: E731
    g = s['g'].double()
    if case['clip']:
        g = g * min(1.0, s['max_norm'] / (float(torch.linalg.vector_norm(g)) + 1e-6))
    if case['bits'] == 32:
        m, v = s['m'].double(), s['v'].double()
    else:
        block = torch.zeros(n, dtype=torch.int64, device='cuda')
        block[s['first'][1:]] = 1
        block = block.cumsum(0)
        power = lambda e: torch.ldexp(torch.ones((), dtype=torch.float64, device='cuda'), e)          # noqa: E731
        m, r = (s[k].double() * power(s[k + '_scale'].view(torch.uint8).to(torch.int32) - 127)[block] for k in ('m', 'r'))
        v = r ** 2
    m = torch.lerp(g, m, pick(lambda h: h['betas'][0]))
    v = torch.lerp(g ** 2, v, pick(lambda h: h['betas'][1]))
    mh, vh = m / pick(lambda h: 1 - h['betas'][0] ** t), v / pick(lambda h: 1 - h['betas'][1] ** t)
    p = s['p'].double() * pick(lambda h: 1 - h['lr'] * h['weight_decay']) - pick(lambda h: h['lr']) * mh / (vh.sqrt() + pick(lambda h: h['eps']))
    if case['bits'] == 32:
        return {'p': p, 'm': m, 'v': v}
    import numpy as np

    def spread(x):
        with np.errstate(over='ignore'):
            x = x ^ (x >> np.uint32(15))
            x = x * np.uint32(B)
            return x ^ (x >> np.uint32(13))
    one = lambda x: np.array([x & M32], dtype=np.uint32)          # noqa: E731
    key = spread(one(t + int(spread(one(s['seed'] * A))[0])))
    with np.errstate(over='ignore'):
        bits = spread(np.arange(n, dtype=np.uint32) * np.uint32(A) + key)
    out = {'p': p}
    for name, x, u, least in (('m', m, bits >> np.uint32(16), 0.0), ('r', v.sqrt(), bits & np.uint32(0xFFFF), 2.0 ** -9)):
        u = torch.from_numpy(u.astype(np.float64) / 65536).cuda()
        top = torch.zeros(s['first'].numel(), dtype=torch.float64, device='cuda').scatter_reduce(0, block, x.abs(), 'amax')
        low = torch.where(top > 0, torch.floor(torch.log2(top)), -120.0) - 7      # the scale's exponent
        low = low.clamp(min=-127.0)
        z = x.abs() / power(low.to(torch.int32))[block]
        grid = power(torch.where(z >= 2.0 ** -6, torch.floor(torch.log2(z.clamp(min=2.0 ** -6))), -6.0).to(torch.int32) - 3)
        down = torch.floor(z / grid)
        z = grid * (down + (z / grid - down + u >= 1))
        z = torch.where(x != 0, z.clamp(min=least), z)
        out[name], out[name + '_scale'] = torch.sign(x) * z, power(low.to(torch.int32))
    return out
