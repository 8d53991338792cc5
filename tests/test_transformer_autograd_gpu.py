"""ops.layer_norm as a part of torch's autograd: saved-tensor hooks, shared gradients, streams, what it has to refuse.  Formulas and
tolerances are those of the layer norm's own tests."""
import pytest
import torch

from test_transformer_layer_norm_gpu import U, check, check_grads, check_y, dev, formula, inputs, ops

pytestmark = pytest.mark.gpu


def norm(form, x, gamma, beta):
    """The layer norm by itself, or as the member of a launch group."""
    o = ops()
    return o.layer_norm(x, gamma, beta) if form == 'single' else o.run_group([(o.LayerNorm, (x, gamma, beta), 1e-5)])[0]


def check_all(x, gamma, beta, f):
    assert all(t.grad is not None for t in (x, gamma, beta))
    check_grads(x.grad, gamma.grad, beta.grad, f)


def dense(t):
    return t.clone(memory_format=torch.contiguous_format)


@pytest.mark.parametrize('form', ['single', 'group'])
@pytest.mark.parametrize('kind', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('what', ['rows that lay apart, dense', 'rows that lay apart, transposed', 'map, dense NCHW', 'tokens, apart'])
def test_saved_x_in_another_layout(what, kind, form):
    """Saved-tensor hooks hand x back in a layout of their own: the backward pass reads it as it lies."""
    x, dy, gamma, beta = inputs((2, 24, 6, 5) if 'map' in what else (40, 100), kind)
    if 'lay apart' in what:
        x = torch.cat([x, x[:, :8]], 1)[:, :100]
    back = {'rows that lay apart, dense': dense, 'rows that lay apart, transposed': lambda t: t.t().contiguous().t(),
            'map, dense NCHW': dense, 'tokens, apart': lambda t: torch.cat([t, t], 1)[:, 100:]}[what]
    mine = tuple(x.shape)
    x = x.detach().requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: back(t) if tuple(t.shape) == mine else t):
        y = norm(form, x, gamma, beta)
    y.backward(dy)
    f = formula(x, gamma, beta, dy, 1e-5)
    check_y(y, f)
    check_grads(x.grad, *((gamma.grad, beta.grad) if form == 'single' else (None, None)), f)


@pytest.mark.parametrize('form', ['single', 'group'])
@pytest.mark.parametrize('pin', [False, True])
@pytest.mark.parametrize('shape', [(30, 72), (2, 24, 6, 5)], ids=str)
def test_saved_on_the_host(shape, pin, form):
    x, dy, gamma, beta = inputs(shape, torch.float16)
    if x.dim() == 2:
        x = torch.cat([x, x], 1)[:, 1:73]
    x = x.detach().requires_grad_()
    with torch.autograd.graph.save_on_cpu(pin_memory=pin):
        y = norm(form, x, gamma, beta)
    y.backward(dy)
    f = formula(x, gamma, beta, dy, 1e-5)
    check_y(y, f)
    check_grads(x.grad, *((gamma.grad, beta.grad) if form == 'single' else (None, None)), f)


@pytest.mark.parametrize('form', ['single', 'group'])
@pytest.mark.parametrize('how', ['fewer rows', 'other type', 'on the host'])
def test_saved_x_that_is_not_x_is_refused(how, form):
    """Checked on the host, before any launch."""
    x, dy, gamma, beta = inputs((40, 100), torch.float32)
    spoil = {'fewer rows': lambda t: t[:10], 'other type': lambda t: t.bfloat16(), 'on the host': lambda t: t.cpu()}[how]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: spoil(t) if tuple(t.shape) == (40, 100) else t):
        y = norm(form, x.requires_grad_(), gamma, beta)
    with pytest.raises((RuntimeError, TypeError)):
        y.backward(dy)
    norm(form, x, gamma, beta).backward(dy)
    check_grads(x.grad, None, None, formula(x, gamma, beta, dy, 1e-5))


def check_sum(got, parts, what):
    """A gradient that several sums meet in: (sum, its terms' magnitudes, rows, e of the formula's tolerance) each, and a rounding of
    the total for every addition."""
    want = sum(f[what] for f in parts)
    tol = 0
    for f in parts:
        (rows, C), n = f['xh'].shape, f['xh'].shape[1] / 64 + 16
        e = (n * (f['R'] + 2) + 8) * U * (1 + f['xh'].abs())
        terms = f['dy'] * f['xh'] if what == 'dg' else f['dy']
        tol = tol + (rows / 256 + 512 + len(parts)) * U * terms.abs().sum(0) + ((e * f['dy'].abs()).sum(0) if what == 'dg' else 0)
    check(what, got, want, tol)


@pytest.mark.parametrize('form', ['single', 'group'])
@pytest.mark.parametrize('shape', [(0, 16), (1, 16), (3, 2), (16, 768), (700, 100), (900, 3), (3, 16384), (2, 20000), (2, 24, 6, 5)], ids=str)
def test_one_parameter_as_gamma_and_beta(shape, form):
    """Its gradient is the sum of both, whether it has one yet or not."""
    x, dy, p, _ = inputs(shape, torch.float32)
    f = formula(x, p, p, dy, 1e-5)
    both = dict(f, both=f['dg'] + f['db'])
    for times in (1, 2):
        y = norm(form, x, p, p)
        y.backward(dy)
        if not f['dy'].numel():
            assert not p.grad.any()
            continue
        check_y(y, f)
        rows, C = f['xh'].shape
        e = (C / 64 + 16) * (f['R'] + 2) + 8
        tol = (rows / 256 + 512 + 4) * U * ((f['dy'] * f['xh']).abs().sum(0) + f['dy'].abs().sum(0)) + (e * U * (1 + f['xh'].abs()) * f['dy'].abs()).sum(0)
        check('dgamma + dbeta', p.grad, times * both['both'], times * tol)


def two_streams(forms, wait):
    """Two layer norms with the same gamma and beta, none of them with a gradient yet, forward on two streams, backward in one pass;
    the stream of the node that runs first is busy, so its first write comes last if nothing waits for it."""
    one = inputs((400, 72), torch.float32)
    two = inputs((300, 72), torch.float32, seed=9)
    gamma, beta = one[2:]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ys = []
    for (x, dy, _, _), s, form in zip((one, two), streams, forms):
        x.requires_grad_()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ys.append(norm(form, x, gamma, beta))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.stream(streams[1]):                     # (the later node runs first)
        torch.cuda._sleep(wait)
    torch.autograd.backward(ys, [one[1], two[1]])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    fs = [formula(x, gamma, beta, dy, 1e-5) for x, dy, _, _ in (one, two)]
    for (x, _, _, _), f in zip((one, two), fs):
        check_grads(x.grad, None, None, f)
    check_sum(gamma.grad, fs, 'dg')
    check_sum(beta.grad, fs, 'db')


@pytest.mark.parametrize('forms', [('single', 'single'), ('group', 'single'), ('single', 'group')], ids=str)
def test_shared_parameters_on_two_streams(forms):
    two_streams(forms, 20000000)


def test_shared_parameters_on_two_streams_of_a_capture():
    """The same inside one captured graph: every replay leaves the eager sum."""
    o = ops()
    one, two = inputs((400, 72), torch.float32), inputs((300, 72), torch.float32, seed=9)
    gamma, beta = one[2:]
    leaves = [t[0].clone().requires_grad_() for t in (one, two)]
    other = torch.cuda.Stream()

    def both():
        cur = torch.cuda.current_stream()
        other.wait_stream(cur)
        y1 = o.layer_norm(leaves[0], gamma, beta)
        with torch.cuda.stream(other):
            y2 = o.layer_norm(leaves[1], gamma, beta)
        cur.wait_stream(other)
        torch.autograd.backward([y1, y2], [one[1], two[1]])
        cur.wait_stream(other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want = [p.grad.clone() for p in (gamma, beta)]
    fs = [formula(t[0], gamma, beta, t[1], 1e-5) for t in (one, two)]
    check_sum(want[0], fs, 'dg')
    check_sum(want[1], fs, 'db')
    for t in (*leaves, gamma, beta):
        t.grad = None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        both()
    made = [gamma.grad, beta.grad]
    for _ in range(4):
        for t in made:
            t.fill_(float('nan'))                           # (made in the capture: the first pass stores)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(made, want))
    o.layer_norm(leaves[0], gamma, beta).backward(one[1])   # an eager pass on another stream than the capture's adds to them
    check_sum(gamma.grad, fs + fs[:1], 'dg')
    check_sum(beta.grad, fs + fs[:1], 'db')


def test_forward_mode_through_the_backward_pass_is_refused():
    """A gradient with a tangent: its derivative would be dropped.  The graph stays as it is."""
    import torch.autograd.forward_ad as fwd_ad
    x, dy, gamma, beta = inputs((20, 24), torch.float32)
    y = ops().layer_norm(x.requires_grad_(), gamma, beta)
    with fwd_ad.dual_level():
        with pytest.raises(NotImplementedError, match='tangent'):
            torch.autograd.grad(y, x, fwd_ad.make_dual(dy, torch.ones_like(dy)))
    assert gamma.grad is None
    y.backward(dy)
    check_all(x, gamma, beta, formula(x, gamma, beta, dy, 1e-5))


@pytest.mark.parametrize('how', ['jit.trace', 'make_fx'])
def test_recording_is_refused(how):
    """A recorded graph would hold the allocation of y (of dx) and none of the kernels."""
    from torch.fx.experimental.proxy_tensor import make_fx
    record = (lambda f, t: torch.jit.trace(f, (t,), check_trace=False)) if how == 'jit.trace' else lambda f, t: make_fx(f)(t)
    x, dy, gamma, beta = inputs((20, 24), torch.float32)
    with pytest.raises(NotImplementedError, match='record'):
        record(lambda t: ops().layer_norm(t, gamma, beta) * 1, x)
    y = ops().layer_norm(x.requires_grad_(), gamma, beta)
    if how == 'make_fx':                                    # (a trace runs the backward pass as a whole)
        with pytest.raises(NotImplementedError, match='record'):
            record(lambda g: torch.autograd.grad(y, x, g, retain_graph=True)[0], dy)
        assert gamma.grad is None
    y.backward(dy)
    check_all(x, gamma, beta, formula(x, gamma, beta, dy, 1e-5))


def test_checkpointed_compiled_and_counted():
    """What runs the layer norm as it is keeps running it: checkpoints of both kinds, a compiled function around it, a counting mode."""
    from torch.utils.checkpoint import checkpoint
    from torch.utils.flop_counter import FlopCounterMode
    x, dy, gamma, beta = inputs((20, 24), torch.float32)
    f = formula(x, gamma, beta, dy, 1e-5)
    x.requires_grad_()
    plain = lambda t: ops().layer_norm(t, gamma, beta)          # noqa: E731
    for run in (lambda t: checkpoint(plain, t, use_reentrant=True), lambda t: checkpoint(plain, t, use_reentrant=False),
                torch.compile(plain, backend='eager')):
        x.grad = gamma.grad = beta.grad = None
        y = run(x)
        check_y(y, f)
        y.backward(dy)
        check_all(x, gamma, beta, f)
    with FlopCounterMode(display=False), torch.no_grad():
        check_y(plain(x), f)


@pytest.mark.parametrize('form', ['single', 'group'])
def test_views_of_the_other_sign_and_zeros_without_memory(form):
    """x and dy as lazy negatives, dy as torch's zeros that own no memory: what they stand for counts."""
    x, dy, gamma, beta = inputs((20, 24), torch.float32)
    xn = x.clone().requires_grad_()
    y = norm(form, xn._neg_view(), gamma, beta)
    f = formula(-x, gamma, beta, -dy, 1e-5)
    check_y(y, f)
    y.backward(dy._neg_view(), retain_graph=True)
    check_grads(-xn.grad, gamma.grad, beta.grad, f)
    xn.grad = gamma.grad = beta.grad = None
    y.backward(torch._efficientzerotensor(20, 24, device=dev()))
    assert not xn.grad.any() and not gamma.grad.any() and not beta.grad.any()
    x, dy, gamma, beta = inputs((20, 1), torch.float32)      # (one channel: any stride would do)
    norm(form, x.requires_grad_(), gamma, beta).backward(torch._efficientzerotensor(20, 1, device=dev()))
    assert not x.grad.any() and not gamma.grad.any() and not beta.grad.any()


class Wrapped(torch.Tensor):
    """A tensor whose operations are Python's, without memory of its own."""
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, f, types, a=(), k=None):
        raise AssertionError('no operation of this tensor is to run')


def test_what_is_no_plain_tensor_is_refused():
    """Checked on the host, before any launch."""
    o = ops()
    x, dy, gamma, beta = inputs((20, 24), torch.float32)
    for bad in (x.to_sparse(), Wrapped(x), torch._efficientzerotensor(20, 24, device=dev())):
        with pytest.raises(TypeError):
            o.layer_norm(bad, gamma, beta)
    for bad in (gamma.detach()._neg_view(), Wrapped(gamma), torch._efficientzerotensor(24, device=dev()), gamma.detach().to_sparse()):
        for form in ('single', 'group') if type(bad) is torch.Tensor else ('single',):
            with pytest.raises(TypeError):
                norm(form, x, bad, beta)
            with pytest.raises(TypeError):
                norm(form, x, gamma, bad)
    y = o.layer_norm(x.requires_grad_(), gamma, beta)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.autograd.grad(y, x, torch.stack([dy, dy]), is_grads_batched=True, retain_graph=True)
    y.backward(dy)
    check_all(x, gamma, beta, formula(x, gamma, beta, dy, 1e-5))


def test_parameters_behind_saved_tensor_hooks():
    """The member's gamma and beta are not copies of the hooks': their gradients arrive, and a change of gamma is refused as ever."""
    x, dy, gamma, beta = inputs((30, 72), torch.float32)
    f = formula(x, gamma, beta, dy, 1e-5)
    x.requires_grad_()
    for form in ('single', 'group'):
        x.grad = gamma.grad = beta.grad = None
        with torch.autograd.graph.save_on_cpu():
            y = norm(form, x, gamma, beta)
        y.backward(dy)
        check_all(x, gamma, beta, f)
        y = norm(form, x, gamma, beta)
        with torch.no_grad():
            gamma.mul_(1.0)
        with pytest.raises(RuntimeError):
            y.backward(dy)


def chain(o, subs, tensors, n_out):
    return o.run_group([(o.Chain, tensors, (subs, (0,), n_out))])[0]


def test_two_readers_of_one_map_in_a_chain():
    """One map read by two layer norms of a chain: its gradient is the sum of theirs."""
    o = ops()
    x, dy, g1, b1 = inputs((2, 24, 6, 5), torch.float32)
    _, dy2, _, _ = inputs((2, 24, 6, 5), torch.float32, seed=4)
    g2, b2 = (torch.nn.Parameter(p.detach().flip(0).clone()) for p in (g1, b1))
    subs = ((o.LayerNorm, (('s', 0), ('i', 1), ('i', 2)), 1e-5, 1), (o.LayerNorm, (('s', 0), ('i', 3), ('i', 4)), 1e-5, 2))
    y1, y2 = chain(o, subs, (x.requires_grad_(), g1, b1, g2, b2), (1, 2))
    torch.autograd.backward([y1, y2], [dy, dy2])
    f1, f2 = formula(x, g1, b1, dy, 1e-5), formula(x, g2, b2, dy2, 1e-5)
    check_y(y1, f1)
    check_y(y2, f2)
    check_grads(None, g1.grad, b1.grad, f1)
    check_grads(None, g2.grad, b2.grad, f2)
    n = 24 / 64 + 16                                        # both terms' own tolerances and a rounding of their sum
    want, tol = f1['dx'] + f2['dx'], U * (f1['dx'] + f2['dx']).abs()
    for f in (f1, f2):
        top = f['h'].abs().amax(1, keepdim=True) * (1 + f['xh'].abs().amax(1, keepdim=True)) ** 2
        tol = tol + (n * (f['R'] + 4) + 16) * U * f['rstd'] * top + U * f['dx'].abs()
    check('dx', x.grad.permute(0, 2, 3, 1).reshape(-1, 24), want, tol)


def test_two_readers_of_a_16_bit_tensor_in_a_chain_are_refused():
    """Refused on the host when the second gradient would be added."""
    o = ops()
    x, dy, g, b = inputs((2, 24, 6, 5), torch.float32)
    t = inputs((40, 24), torch.bfloat16)[0].requires_grad_()
    subs = ((o.LayerNorm, (('i', 1), ('i', 2), ('i', 3)), 1e-5, 1), (o.LayerNorm, (('i', 1), ('i', 2), ('i', 3)), 1e-5, 2))
    y1, y2 = chain(o, subs, (x, t, g, b), (1, 2))
    with pytest.raises(TypeError, match='fan-in'):
        torch.autograd.backward([y1, y2], [torch.ones_like(y1), torch.ones_like(y2)])
    for bad in (x.bfloat16(), x.reshape(48, 30)):
        with pytest.raises((TypeError, ValueError)):        # what a chain's slots are
            chain(o, ((o.LayerNorm, (('s', 0), None, None), 1e-5, 1),), (bad,), (1,))


def test_chains_of_one_group_that_share_parameters():
    """Two chains, two lanes, the second one's input far longer on its way: one gradient for gamma and beta, both parts in it."""
    o = ops()
    sets = [inputs((2, 24, 6, 5), torch.float32), inputs((4, 24, 48, 40), torch.float32, seed=3)]
    gamma, beta = sets[0][2:]
    for _ in range(3):
        gamma.grad = beta.grad = None
        sub = ((o.LayerNorm, (('s', 0), ('i', 1), ('i', 2)), 1e-5, 1),)
        ys = o.run_group([(o.Chain, (x.requires_grad_(), gamma, beta), (sub, (0,), (1,))) for x, _, _, _ in sets])
        for x, _, _, _ in sets:
            x.grad = None
        torch.autograd.backward([y for (y,) in ys], [dy for _, dy, _, _ in sets])
        fs = [formula(x, gamma, beta, dy, 1e-5) for x, dy, _, _ in sets]
        for (x, _, _, _), f in zip(sets, fs):
            check_grads(x.grad, None, None, f)
        check_sum(gamma.grad, fs, 'dg')
        check_sum(beta.grad, fs, 'db')


@pytest.mark.parametrize('kind', [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('shape', [(1, 1), (4096, 1), (3, 1, 8, 6)], ids=str)
def test_one_channel(shape, kind):
    """The norm of one number is 0 whatever it is: y is beta, and x and gamma have a gradient of 0, to the bit."""
    x, dy, gamma, beta = inputs(shape, kind)
    y = ops().layer_norm(x.requires_grad_(), gamma, beta)
    y.backward(dy)
    assert torch.equal(y, beta.detach().to(kind).expand_as(y))
    assert not x.grad.any() and not gamma.grad.any()
    f = formula(x, gamma, beta, dy, 1e-5)
    check_grads(None, None, beta.grad, f)


def test_gradients_are_ordinary_tensors(tmp_path):
    """Gradients that a pass has made carry a note of their stream: they save, copy and step like any other."""
    import copy
    x, dy, gamma, beta = inputs((30, 72), torch.float32)
    ops().layer_norm(x, gamma, beta).backward(dy)
    f = formula(x, gamma, beta, dy, 1e-5)
    torch.save([gamma.grad, beta.grad], str(tmp_path / 'g.pth'))
    for dg, db in ([gamma.grad, beta.grad], torch.load(str(tmp_path / 'g.pth'), weights_only=True), copy.deepcopy([gamma.grad, beta.grad]),
                   [t.clone() for t in (gamma.grad, beta.grad)], [t.detach() for t in (gamma.grad, beta.grad)],
                   [torch.compile(lambda t: t * 1, backend='eager')(t) for t in (gamma.grad, beta.grad)]):
        check_grads(None, dg, db, f)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in (gamma, beta)]
    for p, q in zip((gamma, beta), twin):
        q.grad = p.grad.clone()
    norms = [torch.nn.utils.clip_grad_norm_(ps, 0.5) for ps in ((gamma, beta), twin)]
    assert torch.equal(*norms)
    for ps in ((gamma, beta), twin):
        torch.optim.AdamW(ps, foreach=True).step()
    assert all(torch.equal(p, q) and torch.equal(p.grad, q.grad) for p, q in zip((gamma, beta), twin))
