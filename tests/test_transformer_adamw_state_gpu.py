"""utils.FlatAdamW.load_state_dict: a state that is refused leaves the optimizer as it was."""
import copy

import pytest
import torch

from test_transformer_adamw_gpu import SHAPES, AdamW, dev, grads, make, on_device

pytestmark = pytest.mark.gpu


SPOILED = {
    'maximize': lambda sd: sd['param_groups'][1].update(maximize=True),          # (a key that the optimizer's groups do not have)
    'amsgrad': lambda sd: sd['param_groups'][1].update(amsgrad=True, foreach=None),
    'lr': lambda sd: sd['param_groups'][0].update(lr=float('nan'), fused=True),
    'betas': lambda sd: sd['param_groups'][0].update(betas=None, fused=True),
    'one beta': lambda sd: sd['param_groups'][1].update(betas=(0.9,)),
    'eps': lambda sd: sd['param_groups'][0].update(eps='x', capturable=False),
    'step': lambda sd: sd['state'][3].update(step=float('nan')),
    'step before the first': lambda sd: sd['state'][3].update(step=-1.0),
    'no step': lambda sd: sd['state'][3].pop('step'),
    'last shape': lambda sd: sd['state'][len(SHAPES) - 1].update({k: v[:1] for k, v in sd['state'][len(SHAPES) - 1].items() if k != 'step'}),
    'last scale': lambda sd: sd['state'][len(SHAPES) - 1].update({k: v.view(-1, 1) for k, v in sd['state'][len(SHAPES) - 1].items()
                                                                  if k.endswith('scale')} or {'exp_avg': torch.zeros(5, 1)}),
}


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('what', list(SPOILED))
def test_refused_states_change_nothing(what, bits):
    def take(o, ps, it):
        for p, g in zip(ps, grads(ps, it)):
            p.grad.copy_(g.to(dev()))
        o.step()
    two = lambda ps: [dict(params=ps[:5], weight_decay=0.1), dict(params=ps[5:], weight_decay=0.0)]          # noqa: E731
    mine, twin = on_device(make()), on_device(make())
    o, o2 = AdamW(two(mine), state_bits=bits), AdamW(two(twin), state_bits=bits)
    for opt, ps in ((o, mine), (o2, twin)):
        take(opt, ps, 0)
    sd = copy.deepcopy(o.state_dict())
    take(o, mine, 1)
    take(o2, twin, 1)
    SPOILED[what](sd)
    groups = [{k: v for k, v in g.items() if k != 'params'} for g in o.param_groups]
    with pytest.raises((ValueError, TypeError, KeyError)):
        o.load_state_dict(sd)
    assert [{k: v for k, v in g.items() if k != 'params'} for g in o.param_groups] == groups
    take(o, mine, 2)
    take(o2, twin, 2)
    assert all(torch.equal(a, b) for a, b in zip(o.flat_state(), o2.flat_state()))
