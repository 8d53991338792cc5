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
