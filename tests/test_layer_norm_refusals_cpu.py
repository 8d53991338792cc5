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
