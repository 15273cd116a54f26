"""The operators around a recurrence at their edges: derivatives that they do not have, extreme values, gradients of views and of single
outputs.  Tolerances as derived in test_gpu_layers.py."""
import pytest
import torch
from torch.autograd import forward_ad

import rewy_b200
from test_gpu_layers import NAMES, _calls, _gen, _leaves

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", NAMES)
def test_a_forward_mode_derivative_is_refused(name):
    """Of an input, and of a gradient that comes back (forward over reverse)."""
    call, xs = _calls(_gen(30))[name]
    mine = _leaves(xs)
    out = call(**mine)
    with forward_ad.dual_level():
        for n, x in xs.items():
            with pytest.raises(RuntimeError, match="has no forward-mode derivative"):
                call(**{**xs, n: forward_ad.make_dual(x, torch.ones_like(x))})
        for o in out:
            seed = forward_ad.make_dual(torch.ones_like(o), torch.ones_like(o))
            with pytest.raises(RuntimeError, match="has no forward-mode derivative"):
                torch.autograd.grad(o, list(mine.values()), seed, retain_graph=True, allow_unused=True)
