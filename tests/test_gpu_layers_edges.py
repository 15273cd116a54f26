"""The operators around a recurrence at their edges: derivatives that they do not have, extreme values, gradients of views and of single
outputs.  Tolerances as derived in test_gpu_layers.py."""
import pytest
import torch
from torch.autograd import forward_ad

import rewy_b200
from test_gpu_layers import BF16, FP32, NAMES, _calls, _compare, _gen, _leaves, oracle

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


@pytest.mark.parametrize("dtype", (BF16, FP32))
@pytest.mark.parametrize("D", (64, 1000, 9001))
@pytest.mark.parametrize("size", (1e-12, 1e-14, 1e-18))
def test_norms_of_very_small_rows_without_eps(dtype, D, size):
    """eps = 0: r is 1 / size, beyond 10^12, and its cube leaves FP32, but every gradient is finite.  Squares down to 10^-36 are
    ordinary FP32 numbers, so the tolerance is that of other rows."""
    rn = _gen(31)
    x, gate, weight = (size * rn(6, D)).to(dtype), rn(6, D).to(dtype), 1 + 0.2 * rn(D)
    for gate_first in (False, True):
        kw = dict(eps=0.0, gate_first=gate_first)
        _compare(lambda **x: (rewy_b200.gated_rms_norm(**x, **kw),), lambda **x: (oracle.gated_rms_norm(**x, **kw),),
                 dict(x=x, gate=gate, weight=weight), (dtype,))
    for scale in (0.5, 0.5 + rn(D)):
        _compare(lambda **x: rewy_b200.residual_rms_norm(**x, eps=0.0), lambda **x: oracle.residual_rms_norm(**x, eps=0.0),
                 dict(x=x, residual=(size * rn(6, D)).to(dtype), weight=weight, scale=scale), (dtype, dtype))


def test_an_optional_operand_without_memory_is_refused():
    """A bias that is a wrapper beside an input that is none: refused, not left out."""
    from test_layers_edges import Wrapper
    rn = _gen(32)
    x, weight = rn(2, 9, 16), rn(16, 4)
    with pytest.raises(RuntimeError, match="needs tensors with memory of their own"):
        rewy_b200.causal_conv(x, weight, Wrapper(rn(16)))
    with pytest.raises(RuntimeError, match="needs tensors with memory of their own"):
        rewy_b200.causal_conv_step(x[:, 0], rn(5, 3, 16), weight, slots=Wrapper(torch.zeros(2, dtype=torch.int32)))


def test_transforms_give_slices_or_raise():
    """vmap runs an operator slice by slice; grad of torch.func, which wraps its tensors, raises."""
    rn = _gen(33)
    x, gate, weight = rn(3, 4, 64), rn(4, 64), rn(64)
    got = torch.func.vmap(lambda v: rewy_b200.gated_rms_norm(v, gate, weight))(x)
    assert torch.equal(got, torch.stack([rewy_b200.gated_rms_norm(v, gate, weight) for v in x]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: rewy_b200.gated_rms_norm(v, gate, weight).sum())(x[0])


@pytest.mark.parametrize("name", NAMES)
def test_backwards_are_counted(name):
    """``assert_used`` as after any training step: both directions; a forward alone does not pass it."""
    call, xs = _calls(_gen(34))[name]
    rewy_b200.stats(reset=True)
    mine = _leaves(xs)
    out = call(**mine)
    with pytest.raises(RuntimeError, match="No optimized_backward calls"):
        rewy_b200.assert_used((name,))
    for _ in range(2):
        torch.autograd.grad(out[0].sum(), list(mine.values()), retain_graph=True, allow_unused=True)
    rewy_b200.assert_used((name,))
    assert rewy_b200.stats() == {f"{name}.optimized_backward": 2, f"{name}.optimized_forward": 1}
    assert rewy_b200.stats(reset=True) and rewy_b200.stats() == {}
    torch.autograd.grad(out[0].sum(), list(mine.values()), allow_unused=True)
    assert rewy_b200.stats(reset=True) == {f"{name}.optimized_backward": 1}
