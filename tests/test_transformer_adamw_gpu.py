"""utils.FlatAdamW on a GPU against torch.optim.AdamW and the formulas in 64 bits.

Tolerances.  u = 2^-24.  m and v take three and four roundings a step and carry (1 + b) of the last step's error on: after k
steps they are off by at most 4 k u of the sum of their terms' magnitudes.  p takes two roundings a step plus an update whose
factors (m, sqrt v, quotient, the coefficients in fp32) carry at most 4 k + 12 u: |error| <= k (2 u |p| + (8 k + 12) u lr-ish update).
8-bit codes are equal: m' and sqrt(v') are defined in fp32, every operation rounded, and from there on everything is exact."""
import copy

import numpy as np
import pytest
import torch

import adamw_plain as plain

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def dev():
    assert torch.cuda.is_available(), 'GPU tests need a GPU'
    return torch.device('cuda:0')


def AdamW(*a, **k):
    from advmix_amd.utils.utils import FlatAdamW
    return FlatAdamW(*a, **k)


SHAPES = [(6, 4, 3, 3), (6,), (1,), (257,), (256,), (33, 31), (3, 1025), (1024,), (5,), (2, 2048), (0,), (1023,)]


def make(shapes=SHAPES, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(*s, generator=g)) for s in shapes]


def on_device(ps):
    return [torch.nn.Parameter(p.detach().clone().to(dev())) for p in ps]


def grads(ps, it, scale=1e-2):
    g = torch.Generator().manual_seed(1000 + it)
    return [torch.randn(*p.shape, generator=g) * scale * (1 + k) for k, p in enumerate(ps)]


def close(name, got, want, tol):
    err = (got.detach().double().cpu() - want).abs()
    assert bool((err <= tol).all()), '%s: worst %.3g of allowed %.3g' % (name, float(err.max()), float((tol + 0 * err).min()))


@pytest.mark.parametrize('clip', [None, 0.05, 1e6])
@pytest.mark.parametrize('wd', [0.0, 0.1])
def test_32_bit_step_matches_torch(clip, wd):
    """Six steps over tensors of odd sizes in two groups, a scheduler's change of the learning rate between; fp64 torch.optim."""
    ref = [torch.nn.Parameter(p.detach().double()) for p in make()]
    mine = on_device(make())
    two = lambda ps: [dict(params=ps[:5], weight_decay=wd, lr=2e-3, betas=(0.8, 0.99)), dict(params=ps[5:], weight_decay=0.0, eps=1e-6)]          # noqa: E731
    o_ref, o = torch.optim.AdamW(two(ref), lr=1e-3), AdamW(two(mine), lr=1e-3, max_norm=clip)
    biggest = [p.detach().abs() for p in ref]
    moved = [torch.zeros_like(p) for p in ref]
    for it in range(6):
        o.zero_grad()
        for a, b, g in zip(ref, mine, grads(ref, it)):
            a.grad = g.double()
            b.grad.copy_(g.to(dev()))
        if clip is not None:
            norm = torch.nn.utils.clip_grad_norm_(ref, clip, foreach=False)
        old = [p.detach().clone() for p in ref]
        o_ref.step()
        o.step()
        moved = [m + (p.detach() - q).abs() for m, p, q in zip(moved, ref, old)]
        if clip is not None:
            assert abs(float(o.grad_norm) - float(norm)) <= 4 * U * float(norm)
            assert torch.equal(mine[0].grad, grads(ref, it)[0].to(dev()))      # .grad keeps what the backward pass left
        if it == 2:
            for opt in (o_ref, o):
                opt.param_groups[0]['lr'] = 5e-4
    k = 6
    for p, q, b, mv in zip(ref, mine, biggest, moved):
        close('p', q, p.detach(), k * (2 * U * (b + mv) + (8 * k + 12) * U * mv) + 1e-30)
    sd = o.state_dict()
    for i, p in enumerate(ref):
        if p.numel():
            st = o_ref.state[p]
            assert float(sd['state'][i]['step']) == 6
            close('m', sd['state'][i]['exp_avg'], st['exp_avg'], 4 * k * U * (st['exp_avg'].abs() + st['exp_avg_sq'].sqrt() * 8))
            close('v', sd['state'][i]['exp_avg_sq'], st['exp_avg_sq'], 5 * k * U * st['exp_avg_sq'] + 1e-40)


def held(o, i):
    """(m values, m E, r values, r E) of parameter i, values in memory order as the e4m3 numbers they are held as."""
    st = o.state_dict()['state'][i]
    flat = lambda t: (t.permute(0, 2, 3, 1) if t.dim() == 4 else t).reshape(-1)          # noqa: E731
    out = []
    for k in ('exp_avg', 'exp_avg_root'):
        out += [flat(st[k + '_codes'].float().cpu()).double().numpy(), st[k + '_scale'].view(torch.uint8).cpu().long().numpy()]
    return out


@pytest.mark.parametrize('clip', [None, 0.05])
@pytest.mark.parametrize('seed', [0, 77])
def test_8_bit_step_matches_the_formula(seed, clip):
    """Every step from the state the device itself holds: codes and exponents as the formula says, weights in fp32."""
    ps = make()
    mine = on_device(ps)
    hy = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    o = AdamW(mine, state_bits=8, max_norm=clip, seed=seed, **hy)
    flat = lambda t: (t.detach().cpu().permute(0, 2, 3, 1) if t.dim() == 4 else t.detach().cpu()).double().reshape(-1).numpy()          # noqa: E731
    for t in range(1, 5):
        o.zero_grad()
        gs = grads(ps, t)
        if t == 3:
            gs[9][1, 5:300] = 0.0
            gs[9][0] *= 1e-7                                # a block of one tensor with far smaller gradients
        for p, g in zip(mine, gs):
            p.grad.copy_(g.to(dev()))
        c = 1.0
        if clip is not None:
            c = float(np.float32(min(1.0, clip / (np.sqrt(sum(float((g.double() ** 2).sum()) for g in gs)) + 1e-6))))
        before = [(flat(p), *held(o, i)) for i, p in enumerate(mine)]
        o.step()
        for i, (p, g) in enumerate(zip(mine, gs)):
            if p.numel() == 0:
                continue
            p0, m0, Em0, r0, Er0 = before[i]
            spread = lambda E: np.repeat(2.0 ** (E - 127.0), 256)[:p0.size]          # noqa: E731
            m0, v0 = m0 * spread(Em0), (r0 * spread(Er0)) ** 2
            gg = (flat(g).astype(np.float32) * np.float32(c)).astype(np.float64)
            m1, v1, m, v = plain.moments(m0, v0, gg, *hy['betas'])
            um, ur = plain.dither(np.arange(p0.size) + p._flat_off, t, seed)
            got = held(o, i)
            for k, (x, u, least) in enumerate(((m1, um, 0.0), (np.sqrt(v1), ur, 2.0 ** -9))):
                want, E = plain.hold(x, u, least)
                assert np.array_equal(got[2 * k + 1], E) and np.array_equal(got[2 * k], want), (t, i, k)
            want = plain.weights(p0, m, v, t, hy['lr'], *hy['betas'], hy['eps'], hy['weight_decay'])
            step = np.abs(want - p0)
            # m may cancel: its error is 3 u of |m0| + |g|, which the quotient by sqrt(v) >= sqrt(1 - b2) |g| keeps below 40 u lr
            tol = 2 * U * np.abs(p0) + 20 * U * step + 200 * U * hy['lr'] * (1 + np.abs(m0) / np.maximum(np.sqrt(v), 1e-30))
            assert (np.abs(flat(p) - want) <= tol).all(), (t, i, float((np.abs(flat(p) - want) / tol).max()))


@pytest.mark.parametrize('sizes', [(100001, 7), (130000, 77), (300001, 1025), (17000001, 3000)], ids=str)
@pytest.mark.parametrize('bits', [32, 8])
def test_larger_steps(bits, sizes):
    """Small steps (no launch before theirs), larger ones, and ones past the caches: two clipped steps, all elements."""
    g = torch.Generator(device=dev()).manual_seed(2)
    ps = [torch.nn.Parameter(torch.randn(n, device=dev(), generator=g)) for n in sizes]
    o = AdamW([dict(params=[ps[0]], weight_decay=0.1), dict(params=[ps[1]], lr=3e-3, weight_decay=0.0)], betas=(0.9, 0.99),
              state_bits=bits, max_norm=1.0, seed=5)
    for t in (1, 2):
        for p in ps:
            p.grad.copy_(torch.randn(p.shape, device=dev(), generator=g) * 1e-2)
        norm = float(sum((p.grad.double() ** 2).sum() for p in ps).sqrt())
        c = float(np.float32(min(1.0, 1.0 / (norm + 1e-6))))
        before = [(p.detach().double().cpu().numpy(), p.grad.cpu().numpy()) for p in ps]
        states = [t_.clone() for t_ in o.flat_state()]
        o.step()
        assert abs(float(o.grad_norm) - norm) <= 4 * U * norm and int(o.flat_state()[3]) == t
        for k, p in enumerate(ps):
            n, off, (lo, hi) = p.numel(), p._flat_off, o._blocks[k]
            p0, gr = before[k]
            gr = gr * np.float32(c)
            cut = lambda x: x[off:off + n].cpu()          # noqa: E731
            if bits == 32:
                m0, v0 = (cut(x).double().numpy() for x in states[1:3])
            else:
                val = lambda x, e: cut(x).view(torch.float8_e4m3fn).double().numpy() * np.repeat(2.0 ** (e[lo:hi].cpu().double().numpy() - 127), 256)[:n]          # noqa: E731
                m0, v0 = val(states[1], states[4]), val(states[2], states[5]) ** 2
            m1, v1, m, v = plain.moments(m0, v0, gr.astype(np.float64), 0.9, 0.99)
            now = o.flat_state()
            if bits == 32:                                  # (the same operations, each rounded)
                assert np.array_equal(cut(now[1]).numpy(), m1) and np.array_equal(cut(now[2]).numpy(), v1)
            else:
                um, ur = plain.dither(np.arange(n) + off, t, 5)
                for x, u, least, codes, scale in ((m1, um, 0.0, now[1], now[4]), (np.sqrt(v1), ur, 2.0 ** -9, now[2], now[5])):
                    want, E = plain.hold(x, u, least)
                    assert np.array_equal(scale[lo:hi].cpu().numpy(), E)
                    assert np.array_equal(cut(codes).view(torch.float8_e4m3fn).double().numpy(), want)
            lr, wd = (1e-3, 0.1) if k == 0 else (3e-3, 0.0)
            want = plain.weights(p0, m, v, t, lr, 0.9, 0.99, 1e-8, wd)
            tol = 2 * U * np.abs(p0) + 20 * U * np.abs(want - p0) + 200 * U * lr * (1 + np.abs(m0) / np.maximum(np.sqrt(v), 1e-30))
            assert (np.abs(p.detach().double().cpu().numpy() - want) <= tol).all()


def test_8_bit_moments_follow_the_32_bit_ones():
    """600 steps of random gradients that shrink on the way.  The formulas in 64 bits give: the average of r^2 over 4096 elements is
    1.036 of v's, one element's ratio spreads by 0.36 (so the average by 0.006; five times that is allowed), and the weights are
    0.136 off (half as much again allowed); with nearest rounding it would be 0.64 and 0.33."""
    a, b = (torch.nn.Parameter(torch.zeros(4096, device=dev())) for _ in range(2))
    o32, o8 = AdamW([a], weight_decay=0.0), AdamW([b], weight_decay=0.0, state_bits=8)
    g = torch.Generator(device=dev()).manual_seed(0)
    for t in range(600):
        x = torch.randn(4096, device=dev(), generator=g) * (3.0 if t < 150 else 0.5)      # the gradients shrink: v has to fall
        a.grad.copy_(x)
        b.grad.copy_(x)
        o32.step()
        o8.step()
    v = o32.state_dict()['state'][0]['exp_avg_sq'].double().mean()
    o = AdamW([torch.nn.Parameter(torch.zeros(4096, device=dev()))], weight_decay=0.0)
    o.load_state_dict(o8.state_dict())                      # 8-bit state into a 32-bit optimizer
    v8 = o.state_dict()['state'][0]['exp_avg_sq'].double().mean()
    assert abs(float(v8 / v) - 1.036) < 0.03, float(v8 / v)
    assert float((a.detach() - b.detach()).norm() / a.detach().norm()) < 0.2


@pytest.mark.parametrize('bits', [32, 8])
def test_state_dict_round_trip_continues_bit_for_bit(bits, tmp_path):
    mine = on_device(make())
    o = AdamW(mine, state_bits=bits, max_norm=0.5, seed=3)

    def step(opt, ps, it):
        opt.zero_grad()
        for p, g in zip(ps, grads(ps, it)):
            p.grad.copy_(g.to(dev()))
        opt.step()
    for it in range(3):
        step(o, mine, it)
    torch.save({'o': o.state_dict(), 'p': [p.detach().clone() for p in mine]}, str(tmp_path / 's.pth'))
    back = torch.load(str(tmp_path / 's.pth'), weights_only=True)
    other = [torch.nn.Parameter(p.clone()) for p in back['p']]
    o2 = AdamW(other, state_bits=bits, max_norm=0.5, seed=3)
    o2.load_state_dict(back['o'])
    for it in range(3, 6):
        step(o, mine, it)
        step(o2, other, it)
    assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(mine, other))
    assert all(torch.equal(a, b) for a, b in zip(o.flat_state(), o2.flat_state()))


@pytest.mark.parametrize('bits', [32, 8])
def test_a_state_without_moments_starts_from_zero(bits):
    def run(opt, ps, its):
        for it in its:
            opt.zero_grad()
            for p, g in zip(ps, grads(ps, it)):
                p.grad.copy_(g.to(dev()))
            opt.step()
    fresh, used = on_device(make()), on_device(make())
    o1, o2 = AdamW(fresh, state_bits=bits), AdamW(used, state_bits=bits)
    run(o2, used, range(3))
    with torch.no_grad():
        for a, b in zip(used, fresh):
            a.copy_(b)
    sd = torch.optim.AdamW(make()).state_dict()              # saved before its first step: no state at all
    sd['param_groups'] = [{k: v for k, v in g.items() if k in ('lr', 'betas', 'eps', 'weight_decay', 'params')} for g in sd['param_groups']]
    o2.load_state_dict(sd)
    run(o1, fresh, range(3, 5))
    run(o2, used, range(3, 5))
    assert all(torch.equal(a, b) for a, b in zip(o1.flat_state(), o2.flat_state()))


def test_state_of_the_other_width_and_of_torch():
    ref = [torch.nn.Parameter(p.detach().clone()) for p in make()]
    o_ref = torch.optim.AdamW(ref)
    for it in range(2):
        for p, g in zip(ref, grads(ref, it)):
            p.grad = g
        o_ref.step()
    sd = o_ref.state_dict()
    sd['param_groups'] = [{k: v for k, v in g.items() if k in ('lr', 'betas', 'eps', 'weight_decay', 'params')} for g in sd['param_groups']]
    o32, o8 = AdamW(on_device(ref)), AdamW(on_device(ref), state_bits=8)
    o32.load_state_dict(copy.deepcopy(sd))
    o8.load_state_dict(copy.deepcopy(sd))
    o = AdamW(on_device(ref))
    o.load_state_dict(o8.state_dict())
    for i, p in enumerate(ref):
        if not p.numel():
            continue
        st = o_ref.state[p]
        got = o32.state_dict()['state'][i]
        assert torch.equal(got['exp_avg'].cpu(), st['exp_avg']) and torch.equal(got['exp_avg_sq'].cpu(), st['exp_avg_sq'])
        got = o.state_dict()['state'][i]
        top = float(st['exp_avg'].abs().max())
        # nearest e4m3: 2^-4 relative, 2^-10 * 2^-7 of the block's largest below the normal range
        close('m', got['exp_avg'], st['exp_avg'].double(), 2.0 ** -4 * st['exp_avg'].double().abs() + 2.0 ** -16 * top)
        r, rt = got['exp_avg_sq'].double().sqrt().cpu(), st['exp_avg_sq'].double().sqrt()
        close('r', r, rt, 2.0 ** -4 * rt * 1.001 + 2.0 ** -16 * float(rt.max()))
        assert int(o.flat_state()[3]) == 2


@pytest.mark.parametrize('bits', [32, 8])
def test_gradients_that_are_not_finite_stay_where_they_are(bits):
    """One element's NaN or infinity poisons that element alone, moments included; so does a zero gradient leave zeros alone."""
    p = torch.nn.Parameter(torch.ones(600, device=dev()))
    o = AdamW([p], state_bits=bits)
    for _ in range(3):
        p.grad.fill_(1e-3)
        p.grad[7], p.grad[300] = float('nan'), float('inf')
        p.grad[20] = 0.0
        o.step()
    bad = ~torch.isfinite(p.detach()).cpu()
    assert bad[7] and bool((bad.nonzero().view(-1) == torch.tensor([7, 300])).all()) and int(bad.sum()) == 2
    q = torch.nn.Parameter(torch.ones(600, device=dev()))
    o2 = AdamW([q], state_bits=bits)
    for _ in range(3):
        q.grad.fill_(1e-3)
        q.grad[20] = 0.0
        o2.step()
    keep = ~bad.to(dev())
    assert torch.equal(p.detach()[keep], q.detach()[keep])


def test_extreme_magnitudes_in_8_bits():
    """Blocks near the ends of fp32's exponents, subnormal gradients, a single large element among small ones."""
    n = 256 * 5
    g = torch.full((n,), 1e-3)
    g[:256] = 1e-19
    g[256:512] = 3e18
    g[512:768] = 1e-41
    g[768] = 1e4
    g[1024:] = 0.0
    p = torch.nn.Parameter(torch.zeros(n, device=dev()))
    o = AdamW([p], state_bits=8, weight_decay=0.0, eps=1e-30)
    for t in range(1, 4):
        p.grad.copy_(g)
        m0, Em, r0, Er = held(o, 0)
        o.step()
        m1, Em1, r1, Er1 = held(o, 0)
        assert np.isfinite(m1).all() and np.isfinite(r1).all() and torch.isfinite(p).all()
        assert Em1[4] == 0 and Er1[4] == 0 and not m1[1024:].any() and not r1[1024:].any()
        assert (r1[768:1024] > 0).all()                     # r > 0 never becomes 0
        with np.errstate(under='ignore'):
            spread = lambda E: np.repeat(2.0 ** (E - 127.0), 256)          # noqa: E731
            mf, vf, _, _ = plain.moments(m0 * spread(Em), (r0 * spread(Er)) ** 2, g.double().numpy(), 0.9, 0.999)
        um, ur = plain.dither(np.arange(n), t, 0)
        for x, u, least, got, E in ((mf, um, 0.0, m1, Em1), (np.sqrt(vf), ur, 2.0 ** -9, r1, Er1)):
            want, Ew = plain.hold(x, u, least)
            assert np.array_equal(E, Ew) and np.array_equal(got, want), t


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('clip', [None, 0.1])
def test_captured_step_replays(bits, clip):
    """A captured step replayed with new gradients and a changed learning rate is the eager step."""
    a, b = on_device(make()), on_device(make())
    oa, ob = AdamW(a, state_bits=bits, max_norm=clip), AdamW(b, state_bits=bits, max_norm=clip)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
    for it in range(5):
        for x, y, g in zip(a, b, grads(a, it)):
            x.grad.copy_(g.to(dev()))
            y.grad.copy_(g.to(dev()))
        if it == 3:
            oa.param_groups[0]['lr'] = ob.param_groups[0]['lr'] = 1e-4
        oa.step()
        ob.sync_hyper()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(oa.flat_state(), ob.flat_state())), it
    assert int(ob.flat_state()[3]) == 5


def test_clipping_with_a_norm_that_is_not_finite():
    """As torch.nn.utils.clip_grad_norm_: an infinite norm scales everything to 0 (and infinity to NaN), NaN makes all NaN."""
    for bad, rest in ((float('inf'), 'zero'), (float('nan'), 'nan')):
        p = torch.nn.Parameter(torch.ones(64, device=dev()))
        o = AdamW([p], weight_decay=0.0, max_norm=1.0)
        p.grad.fill_(1e-3)
        p.grad[5] = bad
        o.step()
        q = p.detach().cpu()
        assert torch.isnan(q[5])
        keep = torch.arange(64) != 5
        assert bool(torch.isnan(q[keep]).all()) if rest == 'nan' else torch.equal(q[keep], torch.ones(63))
        assert not torch.isfinite(o.grad_norm)


def test_norm_of_large_and_small_gradients():
    """fp32 squares would overflow at 1e20 and vanish at 1e-25: the sum is taken in fp64."""
    for scale in (1e25, 1e-25):
        p = torch.nn.Parameter(torch.ones(100003, device=dev()))
        o = AdamW([p], max_norm=1.0)
        p.grad.fill_(scale)
        o.step()
        want = scale * 100003 ** 0.5
        assert abs(float(o.grad_norm) - want) <= 1e-6 * want


def test_on_another_stream_and_detached_gradients():
    p, q = on_device(make()), on_device(make())
    o, o2 = AdamW(p), AdamW(q)
    for x, y, g in zip(p, q, grads(p, 0)):
        x.grad.copy_(g.to(dev()))
        y.grad.copy_(g.to(dev()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o.step()
    torch.cuda.current_stream().wait_stream(side)
    o2.step()
    assert all(torch.equal(a, b) for a, b in zip(o.flat_state(), o2.flat_state()))
    p[0].grad = torch.zeros_like(p[0])
    with pytest.raises(RuntimeError):
        o.step()


def test_gaps_between_tensors_stay_zero():
    mine = on_device(make([(5,), (1,), (1027,), (3, 3)]))
    for bits in (32, 8):
        o = AdamW([torch.nn.Parameter(p.detach().clone()) for p in mine], state_bits=bits, max_norm=1.0)
        for it in range(3):
            o.flat_grads.zero_()
            for p, g in zip(o.param_groups[0]['params'], grads(mine, it)):
                p.grad.copy_(g.to(dev()))
            o.step()
        own = torch.zeros_like(o.flat_params, dtype=torch.bool)
        for p in o.param_groups[0]['params']:
            own[p._flat_off:p._flat_off + p.numel()] = True
        for t in o.flat_state()[:3]:
            assert not t[~own].any()


def test_refusals_on_the_device():
    p = torch.nn.Parameter(torch.ones(8, device=dev()))
    o = AdamW([p], max_norm=1.0)
    with pytest.raises(RuntimeError):
        o.add_param_group({'params': [torch.nn.Parameter(torch.ones(3, device=dev()))]})
    for bad in (0.0, -1.0, float('nan'), None):
        o.max_norm = bad
        with pytest.raises(ValueError):
            o.step()
    o.max_norm = 1.0
    o.param_groups[0]['lr'] = -1.0
    with pytest.raises(ValueError):
        o.step()
    o.param_groups[0]['lr'] = 1e-3
    sd = o.state_dict()
    codes = dict(step=1.0, exp_avg_codes=torch.zeros(8, dtype=torch.uint8), exp_avg_scale=torch.zeros(1, dtype=torch.uint8),
                 exp_avg_root_codes=torch.zeros(8, dtype=torch.uint8), exp_avg_root_scale=torch.zeros(1, dtype=torch.uint8))
    for spoil in (lambda s: s['state'].update({0: dict(codes, exp_avg_codes=torch.zeros(8))}),
                  lambda s: s['state'].update({0: dict(codes, exp_avg_scale=torch.zeros(2, dtype=torch.uint8))}),
                  lambda s: s['state'].update({0: dict(codes, exp_avg_root_codes=torch.zeros(9, dtype=torch.uint8))}),
                  lambda s: s['state'][0].pop('exp_avg'), lambda s: s['state'][0].update(exp_avg=torch.zeros(9)),
                  lambda s: s.update(param_groups=s['param_groups'] * 2), lambda s: s['param_groups'][0].update(eps=0.0)):
        s = copy.deepcopy(sd)
        spoil(s)
        with pytest.raises(ValueError):
            o.load_state_dict(s)
    assert o.param_groups[0]['eps'] == 1e-8
    o.step()


def test_closure_and_scheduler():
    """step(closure) computes the gradients and hands the loss back; a torch scheduler drives the learning rate."""
    w = torch.nn.Parameter(torch.ones(4, 8, device=dev()))
    o = AdamW([w], lr=0.1, weight_decay=0.0, eps=1e-8)
    sched = torch.optim.lr_scheduler.MultiStepLR(o, [1], 0.1)
    x = rand_like(w)

    def closure():
        o.zero_grad()
        loss = (w * x).sum()
        loss.backward()
        return loss
    for lr in (0.1, 0.01):
        before = w.detach().clone()
        loss = o.step(closure)
        assert abs(float(loss.detach()) - float((before.double() * x.double()).sum())) <= 1e-4
        # a constant gradient: m / sqrt(v) is its sign after bias correction
        assert float((w.detach() - (before - lr * x.sign())).abs().max()) <= 1e-5
        sched.step()


def rand_like(t):
    return torch.randn(*t.shape, generator=torch.Generator().manual_seed(5)).to(t.device)


@pytest.mark.parametrize('bits', [32, 8])
def test_layer_norms_trained_with_adamw(bits):
    """conv -> layer norm -> ReLU -> conv, two groups, clipped, the gradients accumulated into the flat buffer: three steps
    against the same net in 64 bits on the CPU (32-bit moments) / the first step (8-bit moments: the same by construction)."""
    from advmix_amd import ops
    torch.manual_seed(0)
    cl = lambda t: t.contiguous(memory_format=torch.channels_last)          # noqa: E731
    w1, w2 = 0.2 * torch.randn(32, 16, 1, 1), 0.2 * torch.randn(16, 32, 1, 1)
    gamma, beta = 1 + 0.1 * torch.randn(32), 0.1 * torch.randn(32)
    mine = [torch.nn.Parameter(cl(t.to(dev())) if t.dim() == 4 else t.to(dev())) for t in (w1, w2, gamma, beta)]
    ref = [torch.nn.Parameter(t.double()) for t in (w1, w2, gamma, beta)]
    groups = lambda ps: [dict(params=ps[:2], weight_decay=0.1), dict(params=ps[2:], weight_decay=0.0)]          # noqa: E731
    o, o_ref = AdamW(groups(mine), lr=1e-2, eps=1e-4, state_bits=bits, max_norm=0.5), torch.optim.AdamW(groups(ref), lr=1e-2, eps=1e-4)
    for it in range(3 if bits == 32 else 1):
        x, dy = torch.randn(4, 16, 8, 6), torch.randn(4, 16, 8, 6)
        o.zero_grad()
        a, b, g, be = mine
        h = ops.activation(ops.layer_norm(ops.conv2d(cl(x.to(dev())), a), g, be), ops.ACT_RELU)
        ops.conv2d(h, b).backward(cl(dy.to(dev())))
        o_ref.zero_grad()
        a, b, g, be = ref
        c = torch.nn.functional.conv2d(x.double(), a).permute(0, 2, 3, 1)
        d = c - c.mean(-1, keepdim=True)
        h = (d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * g + be).permute(0, 3, 1, 2).relu()
        torch.nn.functional.conv2d(h, b).backward(dy.double())
        for p, q in zip(mine, ref):
            assert float((p.grad.double().cpu() - q.grad).abs().max()) <= 1e-4 * float(q.grad.abs().max())
        torch.nn.utils.clip_grad_norm_(ref, 0.5)
        o.step()
        o_ref.step()
        for p, q in zip(mine, ref):                         # gradients to 1e-4 of their largest, updates bounded by lr / eps
            assert float((p.detach().double().cpu() - q.detach()).abs().max()) <= 1e-4 * (it + 1)


@pytest.mark.parametrize('bits,clip', [(32, None), (8, 1.0)])
def test_advmix_step_as_graphs_and_eager(bits, clip, monkeypatch):
    """The AdvMix step with FlatAdamW for both networks, deterministic mode, one launch lane: three batches through
    AdvMixGraphRunner (warm-up, snapshot, restore, replays) leave the bits that the eager step leaves."""
    import types
    from advmix_amd import ops
    from advmix_amd.core.function import advmix_step
    from advmix_amd.graph import AdvMixGraphRunner
    from advmix_amd.utils.utils import adamw_groups
    from oracle.synth import synth_batch
    from test_models_gpu import _tiny_setup
    monkeypatch.setattr(ops, 'MAX_LANES', 1)
    args = types.SimpleNamespace(alpha=0.1, adv_loss_weight=1.0)
    data = []
    for it in range(3):
        v, t, w = synth_batch('hrnet_tiny.it%d' % (it % 2), 2, 5, 64, 64)
        data.append(([x.cuda().contiguous() for x in v], t.cuda(), w.cuda()))

    def nets():
        _, D, G, T, crit, _, _, _ = _tiny_setup(lr=1e-3)
        return (D, G, T, crit) + tuple(AdamW(adamw_groups(m, 0.05), lr=1e-3, state_bits=bits, max_norm=clip, seed=k) for k, m in enumerate((D, G)))
    try:
        ops.set_deterministic(True)
        D, G, T, crit, oD, oG = nets()
        runner = AdvMixGraphRunner(args, D, G, T, crit, oD, oG, *data[0], warmup=2)
        losses = []
        for batch in data:
            runner.load_batch(*batch)
            loss, _ = runner.step()
            losses.append(float(loss))
        torch.cuda.synchronize()
        D2, G2, T2, crit2, oD2, oG2 = nets()
        for batch, loss in zip(data, losses):
            l2, _ = advmix_step(args, D2, G2, T2, crit2, oD2, oG2, *batch)
            assert float(l2) == loss
    finally:
        ops.set_deterministic(False)
    for a, b in ((oD, oD2), (oG, oG2)):
        assert int(a.flat_state()[3]) == 3
        assert all(torch.equal(x, y) for x, y in zip(a.flat_state(), b.flat_state()))


def test_get_optimizer_trains_a_pose_net():
    """TRAIN.OPTIMIZER adamw through get_optimizer: groups, and one plain_step of a small pose net moves every tensor."""
    import types
    from advmix_amd.core.loss import JointsMSELoss
    from advmix_amd.config import CfgNode
    from advmix_amd.core.function import plain_step
    from advmix_amd.utils.utils import get_optimizer
    from advmix_amd import models
    from oracle import configs
    cfg = CfgNode({'MODEL': {'NAME': 'pose_resnet', 'EXTRA': configs.RES18_TINY, 'NUM_JOINTS': 5, 'INIT_WEIGHTS': True, 'PRETRAINED': ''},
                   'TRAIN': {'OPTIMIZER': 'adamw', 'LR': 1e-3, 'WD': 0.05, 'STATE_BITS': 8, 'CLIP_NORM': 1.0}})
    net = models.pose_resnet.get_pose_net(cfg, is_train=True).to(dev()).train()
    o = get_optimizer(cfg, net)
    assert o.state_bits == 8 and [g['weight_decay'] for g in o.param_groups] == [0.05, 0.0]
    assert all(p.dim() >= 2 for p in o.param_groups[0]['params']) and all(p.dim() < 2 for p in o.param_groups[1]['params'])
    assert sum(len(g['params']) for g in o.param_groups) == len(list(net.parameters()))
    before = o.flat_params.clone()
    x = torch.randn(2, 3, 64, 64, generator=torch.Generator().manual_seed(3)).to(dev())
    with torch.no_grad():
        hm = net(x)
    target, tw = torch.rand_like(hm), torch.ones(hm.shape[0], 5, 1, device=dev())
    loss, _ = plain_step(net, JointsMSELoss(use_target_weight=True).cuda(), o, x, target, tw)
    assert torch.isfinite(loss) and torch.isfinite(o.flat_params).all()
    for p in net.parameters():
        lo = p._flat_off
        if bool(p.grad.abs().max() > 0):
            assert not torch.equal(o.flat_params[lo:lo + p.numel()], before[lo:lo + p.numel()])

