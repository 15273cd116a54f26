"""What the operators around a recurrence refuse at their edges.  No GPU is needed: each check stands in front of the one for CUDA
tensors."""
import pytest
import torch
from torch.autograd import forward_ad

import rewy_b200
from test_layers import _conv, _conv_step, _gated, _kda, _residual, _scan, _scan_step, z


def _gdn(**kw):
    a = dict(q=z(2, 2, 8), k=z(2, 2, 8), v=z(2, 4, 6), g=z(2, 4), beta=z(2, 4), state=z(5, 4, 8, 6))
    a.update(kw)
    return rewy_b200.step_gated_delta_rule(**a)


def _gdn2(**kw):
    a = dict(q=z(2, 2, 8), k=z(2, 2, 8), v=z(2, 4, 6), g=z(2, 4, 8), b=z(2, 4, 8), w=z(2, 4, 6), state=z(5, 4, 8, 6))
    a.update(kw)
    return rewy_b200.step_gdn2(**a)


def _delta(**kw):
    a = dict(q=z(2, 2, 8), k=z(2, 2, 8), v=z(2, 4, 6), beta=z(2, 4), state=z(5, 4, 8, 6))
    a.update(kw)
    return rewy_b200.step_delta_rule(**a)


OPERANDS = [(_conv, dict(x=z(2, 9, 16), weight=z(16, 4), bias=z(16), initial_state=z(2, 3, 16))),
            (_scan, dict(u=z(1, 9, 12), dt=z(1, 9, 12), A=z(12, 16), B=z(1, 9, 16), C=z(1, 9, 16), D=z(12), z=z(1, 9, 12), dt_bias=z(12),
                         initial_state=z(1, 12, 16))),
            (_gated, dict(x=z(3, 8), gate=z(3, 8), weight=z(8))),
            (_residual, dict(x=z(3, 8), residual=z(3, 8), weight=z(8), scale=z(8))),
            (_conv_step, dict(x=z(2, 16), state=z(5, 3, 16), weight=z(16, 4), bias=z(16))),
            (_scan_step, dict(u=z(2, 12), dt=z(2, 12), A=z(12, 16), B=z(2, 16), C=z(2, 16), state=z(5, 12, 16), D=z(12), z=z(2, 12), dt_bias=z(12))),
            (_kda, dict(q=z(2, 2, 8), k=z(2, 2, 8), v=z(2, 4, 6), g=z(2, 4, 8), beta=z(2, 4), state=z(5, 4, 8, 6), A_log=z(4), dt_bias=z(32),
                        use_gate_in_kernel=True)),
            (_gdn, dict(g=z(2, 4), beta=z(2, 4))), (_gdn2, dict(b=z(2, 4, 8), w=z(2, 4, 6))), (_delta, dict(k=z(2, 2, 8), beta=z(2, 4)))]
ONE_EACH = [(call, kw, n) for call, kw in OPERANDS for n, t in kw.items() if isinstance(t, torch.Tensor)]
NAMES = [f"{call.__name__[1:]}-{n}" for call, _, n in ONE_EACH]


@pytest.mark.parametrize("call,kw,name", ONE_EACH, ids=NAMES)
def test_an_operand_with_a_forward_mode_derivative_is_refused(call, kw, name):
    """The kernels would return a value without its tangent, which reads as a derivative of zero.  Under no_grad too: it does not
    switch forward mode off."""
    with forward_ad.dual_level():
        dual = {**kw, name: forward_ad.make_dual(kw[name], torch.ones_like(kw[name]))}
        with pytest.raises(RuntimeError, match="has no forward-mode derivative"):
            call(**dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="has no forward-mode derivative"):
            call(**dual)
        plain = {**kw, name: forward_ad.unpack_dual(dual[name]).primal}
        with pytest.raises(RuntimeError, match="needs CUDA tensors"):
            call(**plain)


@pytest.mark.parametrize("call,kw,name", ONE_EACH, ids=NAMES)
def test_jvp_is_refused(call, kw, name):
    with pytest.raises(RuntimeError, match="has no forward-mode derivative"):
        torch.func.jvp(lambda t: call(**{**kw, name: t}), (kw[name],), (torch.ones_like(kw[name]),))
