"""What layer_norm and FlatAdamW refuse without a GPU, the C entries' argument checks (nothing is launched), and the plain form
of the 8-bit moments: what the device's codes are checked against."""
import ctypes
import types

import numpy as np
import pytest
import torch

import adamw_plain as plain


def test_layer_norm_refuses_the_cpu_and_other_types():
    from advmix_amd import ops
    for t in (torch.zeros(4, 8), torch.zeros(1, 8, 2, 2), torch.zeros(4, 8, dtype=torch.float64)):
        with pytest.raises(TypeError):
            ops.layer_norm(t)
    x = torch.zeros(4, 8)
    for bad in (('x',), (None,), (x, 1.0), (x, x, 'b'), (x, None, None, 'eps')):
        with pytest.raises(TypeError):
            ops.layer_norm(*bad)
    with pytest.raises(TypeError):
        ops._node.layer_norm(x)


def test_row_stride_of_layouts():
    from advmix_amd.ops import _row_stride
    x = torch.zeros(6, 10)
    assert _row_stride(x) == 10 and _row_stride(x[:, 2:7]) == 10 and _row_stride(x[::2]) == 20
    assert _row_stride(x.t()) is None and _row_stride(x[:, ::2]) is None
    assert _row_stride(x[:1].expand(6, 10)) == 0 and _row_stride(x[0]) == 10
    assert _row_stride(torch.zeros(2, 3, 10)) == 10 and _row_stride(torch.zeros(2, 5, 10)[:, 1:4]) is None
    assert _row_stride(torch.zeros(1, 5, 10)[:, 1:4]) == 10 and _row_stride(torch.zeros(2, 1, 10)) == 10
    nchw = torch.zeros(2, 8, 3, 4)
    assert _row_stride(nchw) is None and _row_stride(nchw.contiguous(memory_format=torch.channels_last)) == 8
    assert _row_stride(torch.zeros(2, 1, 3, 4)) == 1 and _row_stride(torch.zeros(5, 1)[:, :1]) == 1


def test_c_entries_refuse_bad_arguments():
    """Every check comes before a launch: no GPU is needed, and none may be touched."""
    from advmix_amd._lib import lib
    p = ctypes.c_void_p(4096)                               # never read
    ok = dict(x=p, ldx=8, gamma=p, beta=p, y=p, mean=p, rstd=p, rows=4, C=8, dtype=0, eps=1e-5)
    for bad in (dict(x=None), dict(y=None), dict(ldx=-1), dict(mean=None), dict(rstd=None), dict(rows=0), dict(rows=-1), dict(C=0),
                dict(C=-5), dict(dtype=3), dict(dtype=-1), dict(eps=-1.0), dict(eps=float('nan')), dict(rows=2 ** 62)):
        a = dict(ok, **bad)
        assert lib.advmix_layer_norm_fwd(*[a[k] for k in ok], None) == 1, bad
    ok = dict(dy=p, lddy=8, x=p, ldx=8, gamma=p, mean=p, rstd=p, dx=p, dg=p, db=p, part=p, add=1, rows=4, C=8, dtype=0)
    for bad in (dict(dy=None), dict(lddy=-1), dict(x=None), dict(ldx=-1), dict(mean=None), dict(rstd=None), dict(part=None), dict(rows=0),
                dict(C=0), dict(dtype=7)):
        a = dict(ok, **bad)
        assert lib.advmix_layer_norm_bwd(*[a[k] for k in ok], None) == 1, bad
    assert lib.advmix_layer_norm_parts(0, 8, 0) == 0 and lib.advmix_layer_norm_parts(4, 0, 0) == 0
    for rows, C in ((1, 1), (5, 70000), (10 ** 7, 32), (2 ** 40, 1024)):
        assert 1 <= lib.advmix_layer_norm_parts(rows, C, 1) <= min(rows, 4096)
    ok = dict(p=p, g=p, m=p, v=p, table=p, chunks=1, hyper=p, groups=1, step=p, part=None, nparts=0, norm=None, coef=p)
    for bad in (dict(p=None), dict(g=None), dict(m=None), dict(v=None), dict(table=None), dict(chunks=0), dict(hyper=None), dict(groups=0),
                dict(step=None), dict(nparts=3), dict(part=p), dict(part=p, nparts=3), dict(coef=None)):
        a = dict(ok, **bad)
        assert lib.advmix_adamw(*[a[k] for k in ok], None) == 1, bad
    ok = dict(p=p, g=p, m=p, r=p, ms=p, rs=p, table=p, chunks=1, hyper=p, groups=1, step=p, part=None, nparts=0, norm=None, seed=0, coef=p)
    for bad in (dict(m=None), dict(r=None), dict(ms=None), dict(rs=None), dict(chunks=-1), dict(part=p, nparts=1)):
        a = dict(ok, **bad)
        assert lib.advmix_adamw8(*[a[k] for k in ok], None) == 1, bad
    assert lib.advmix_grad_sumsq(None, 4, p, 1, None) == 1 and lib.advmix_grad_sumsq(p, 0, p, 1, None) == 1
    assert lib.advmix_grad_sumsq(p, 4, None, 1, None) == 1 and lib.advmix_grad_sumsq(p, 4, p, 0, None) == 1
    assert lib.advmix_moments_pack(None, p, p, p, 1, 0, None) == 1 and lib.advmix_moments_unpack(p, p, p, p, 0, 0, None) == 1


def test_adamw_refuses():
    from advmix_amd.utils.utils import FlatAdamW
    P = lambda *s: torch.nn.Parameter(torch.zeros(*s))          # noqa: E731
    a = P(3)
    for bad in (dict(lr=-1.0), dict(lr=float('nan')), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=0.0), dict(eps=1e-40),
                dict(weight_decay=-0.1), dict(state_bits=16), dict(max_norm=0.0), dict(max_norm=float('inf')), dict(seed=-1), dict(seed=2 ** 31)):
        with pytest.raises(ValueError):
            FlatAdamW([P(3)], **bad)
    with pytest.raises(ValueError):
        FlatAdamW([dict(params=[P(3)], amsgrad=True)])
    with pytest.raises(ValueError):
        FlatAdamW([dict(params=[P(3)]), dict(params=[P(2)], eps=-1.0)])
    with pytest.raises(ValueError), pytest.warns(UserWarning):
        FlatAdamW([a, a])
    with pytest.raises(ValueError):
        FlatAdamW([dict(params=[a]), dict(params=[a])])
    with pytest.raises(ValueError):
        FlatAdamW([torch.nn.Parameter(torch.zeros(3), requires_grad=False)])
    with pytest.raises(ValueError):
        FlatAdamW([P(0)])
    with pytest.raises(TypeError):
        FlatAdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.bfloat16))])
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        FlatAdamW([P(3)]).step()


def test_get_optimizer_groups_and_config():
    from advmix_amd.config import cfg as default
    from advmix_amd.utils.utils import FlatAdamW, adamw_groups, get_optimizer
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 4, 3), torch.nn.BatchNorm2d(4), torch.nn.Linear(4, 2))
    net[2].bias.requires_grad = False
    g = adamw_groups(net, 0.05)
    assert [len(x['params']) for x in g] == [2, 3] and [x['weight_decay'] for x in g] == [0.05, 0.0]
    assert [len(x['params']) for x in adamw_groups(torch.nn.BatchNorm2d(4), 0.1)] == [2]
    c = default.clone()
    assert c.TRAIN.STATE_BITS == 32 and c.TRAIN.CLIP_NORM == 0.0 and c.TRAIN.OPTIMIZER == 'adam'
    c.defrost()
    c.merge_from_list(['TRAIN.OPTIMIZER', 'adamw', 'TRAIN.STATE_BITS', '8', 'TRAIN.CLIP_NORM', '1.5', 'TRAIN.WD', '0.02'])
    o = get_optimizer(c, net)
    assert type(o) is FlatAdamW and o.state_bits == 8 and o.max_norm == 1.5 and o.param_groups[0]['weight_decay'] == 0.02
    short = types.SimpleNamespace(TRAIN=type(c.TRAIN)({'OPTIMIZER': 'adamw', 'LR': 1e-3, 'WD': 0.0}))
    o = get_optimizer(short, net)
    assert o.state_bits == 32 and o.max_norm is None


def test_plain_8_bit_numbers_are_e4m3():
    """What hold() puts down is an e4m3 number of its block's scale, a neighbour of the value, and exact where the value is one."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal(1000) * np.exp(rng.standard_normal(1000) * 4)).astype(np.float32)
    x[[3, 500]] = 0.0
    u = rng.integers(0, 65536, 1000) / 65536
    h, E = plain.hold(x, u, 0.0)
    t = torch.from_numpy(h).float()
    assert torch.equal(t.to(torch.float8_e4m3fn).float(), t)
    z = x.astype(np.float64) / np.repeat(2.0 ** (E - 127.0), 256)[:1000]
    assert (np.abs(h - z) < plain.step_size(np.abs(z))).all()
    for k in range(0, 1000, 256):
        assert 128 <= np.abs(z[k:k + 256]).max() < 256
    again, E2 = plain.hold(z, u, 0.0)
    fixed, E3 = plain.hold(h, rng.integers(0, 65536, 1000) / 65536, 0.0)
    assert np.array_equal(fixed * np.repeat(2.0 ** (E3 - 127.0), 256)[:1000], h)      # on the grid stays on the grid
    assert (plain.hold(np.full(256, 1e-30), np.zeros(256), 2.0 ** -9)[0] > 0).all()


def test_plain_dither_is_uniform_and_uncorrelated():
    """256 steps x 4096 places: mean, variance and neighbours' correlation, each within five standard deviations."""
    for k in (0, 1):
        x = np.stack([plain.dither(np.arange(4096), t, 0)[k] for t in range(1, 257)])
        n = x.size
        assert abs(x.mean() - 0.5 + 2.0 ** -17) < 5 * (1 / 12) ** 0.5 / n ** 0.5
        assert abs(12 * x.var() - 1) < 5 * (0.8 / n) ** 0.5
        for a, b in ((x[:-1], x[1:]), (x[:-4], x[4:]), (x[:, :-1], x[:, 1:]), (x[:, :-4], x[:, 4:]), (x[:, :-256], x[:, 256:])):
            assert abs(np.corrcoef(a.ravel(), b.ravel())[0, 1]) < 5 / a.size ** 0.5
