"""What ops.layer_norm refuses before it looks at the device: results that would be silently wrong.  Nothing is launched."""
import pytest
import torch

from advmix_amd import ops


def args(which=None, change=None):
    a = [torch.randn(5, 8, generator=torch.Generator().manual_seed(k)) if k == 0 else torch.ones(8) for k in range(3)]
    if which is not None:
        a[which] = change(a[which])
    return a


@pytest.mark.parametrize('which', [0, 1, 2])
def test_forward_mode(which):
    """A tangent would be dropped; the members of launch groups refuse it likewise."""
    import torch.autograd.forward_ad as fwd_ad
    with fwd_ad.dual_level():
        a = args(which, lambda t: fwd_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(NotImplementedError, match='tangent'):
            ops.layer_norm(*a)
        with pytest.raises(TypeError):                      # (no tangent: the device is what is wrong)
            ops.layer_norm(*args())
    with pytest.raises(TypeError):
        ops.layer_norm(*a)                                  # the level is closed


def traced(f, x):
    torch.jit.trace(f, (x,), check_trace=False)


def symbolic(**how):
    from torch.fx.experimental.proxy_tensor import make_fx
    return lambda f, x: make_fx(f, **how)(x)


def fake(f, x):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        f(torch.randn(5, 8))


RECORDERS = {'jit.trace': traced, 'make_fx': symbolic(), 'make_fx, pre-dispatch': symbolic(pre_dispatch=True),
             'make_fx, fake': symbolic(tracing_mode='fake'), 'make_fx, symbolic': symbolic(tracing_mode='symbolic'), 'fake tensors': fake,
             'functionalize': lambda f, x: torch.func.functionalize(f)(x), 'func.grad': lambda f, x: torch.func.grad(lambda v: f(v).sum())(x),
             'func.vjp': lambda f, x: torch.func.vjp(f, x), 'vmap': lambda f, x: torch.func.vmap(f)(x)}


@pytest.mark.parametrize('of', ['its input', 'another input'])
@pytest.mark.parametrize('how', list(RECORDERS))
def test_recording(how, of):
    """A recorded graph would hold the output's allocation and none of the kernels."""
    c = torch.randn(5, 8)
    f = (lambda v: ops.layer_norm(v) * 1) if of == 'its input' else (lambda v: v * ops.layer_norm(c))
    with pytest.raises(NotImplementedError, match='record'):
        RECORDERS[how](f, torch.randn(5, 8))
    with pytest.raises(TypeError):                          # none is active any more: the device is what is wrong
        f(torch.randn(5, 8))


def test_what_only_watches_operations_is_not_refused():
    """Modes that count or hand on what runs do not make the result wrong: the device is what is wrong here."""
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False), torch.device('cpu'):
        with pytest.raises(TypeError):
            ops.layer_norm(torch.randn(5, 8))


def test_fan_in_of_16_bit_gradients():
    """A Chain adds up the gradients of a tensor with several readers in fp32 only: anything else would be read past its end."""
    for a, b in ((torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.bfloat16)):
        with pytest.raises(TypeError, match='fan-in'):
            ops._add(None, torch.zeros(2, 8, dtype=a), torch.zeros(2, 8, dtype=b))


@pytest.mark.parametrize('node', ['None', 'types.SimpleNamespace(torch_version="0.1")'])
def test_without_the_torch_side_module(node):
    """_node.so absent, or built for another torch: every other op stays importable, layer_norm says what is missing."""
    import os
    import subprocess
    import sys
    code = ('import sys, types, torch\nimport advmix_amd\nnode = %s\nsys.modules["advmix_amd._node"] = node\n'
            'if node: advmix_amd._node = node\n'
            'from advmix_amd import ops, models\n'
            'assert ops._node is None and callable(ops.conv2d) and ops.LayerNorm\n'
            'try: ops.layer_norm(torch.zeros(2, 3))\n'
            'except ImportError as e: print("said:", e)\n' % node)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and 'said:' in r.stdout and 'advmix_amd.build' in r.stdout, (r.stdout, r.stderr)
    assert ('torch 0.1' in r.stdout) == (node != 'None')


def test_one_gradient_buffer_as_both_is_only_added_to():
    """The C entry: a launch that stores two sums to one place is refused before anything is launched."""
    import ctypes
    from advmix_amd._lib import lib
    p = ctypes.c_void_p(4096)                               # never read
    for add in (0, 1, 2, 4):
        assert lib.advmix_layer_norm_bwd(p, 8, p, 8, p, p, p, p, p, p, p, add, 4, 8, 0, None) == 1, add
