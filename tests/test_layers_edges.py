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


def _wide(*s):
    """A tensor of these sizes over one element: no memory."""
    return z(1).expand(*s)


BIG, N32 = 1 << 32, torch.int32
LARGE = [
    (_conv, dict(x=_wide(1, BIG + 64, 4), weight=z(4, 4)), "up to 1073741824 tokens per sequence, got 4294967360"),
    (_conv, dict(x=_wide(BIG + 2, 64, 4), weight=z(4, 4)), "up to 1073741824 sequences, got 4294967298"),
    (_conv, dict(x=_wide(1 << 20, 1 << 11, 4), weight=z(4, 4)), "up to 1073741824 tokens, got 2147483648"),
    (_conv, dict(x=_wide(1, 9, BIG + 8), weight=_wide(BIG + 8, 4)), "up to 16777216 channels, got 4294967304"),
    (_scan, dict(u=_wide(1, BIG + 9, 12), dt=_wide(1, BIG + 9, 12), B=_wide(1, BIG + 9, 16), C=_wide(1, BIG + 9, 16)),
     "up to 1073741824 tokens per sequence, got 4294967305"),
    (_scan, dict(u=_wide(BIG + 1, 9, 12), dt=_wide(BIG + 1, 9, 12), B=_wide(BIG + 1, 9, 16), C=_wide(BIG + 1, 9, 16)), "up to 1073741824 sequences"),
    (_scan, dict(u=_wide(1, 9, BIG + 8), dt=_wide(1, 9, BIG + 8), A=_wide(BIG + 8, 16)), "up to 16777216 channels"),
    (_conv_step, dict(x=_wide(BIG + 1, 1), state=z(5, 3, 1), weight=z(1, 4), slots=z(1, dtype=N32).expand(BIG + 1)), "up to 2147483647 rows, got 4294967297"),
    (_conv_step, dict(x=_wide(2, BIG + 1), state=_wide(5, 3, BIG + 1), weight=_wide(BIG + 1, 4)), "up to 16777216 channels"),
    (_scan_step, dict(u=_wide(BIG + 1, 12), dt=_wide(BIG + 1, 12), B=_wide(BIG + 1, 16), C=_wide(BIG + 1, 16), slots=z(1, dtype=N32).expand(BIG + 1)),
     "up to 2147483647 rows"),
    (_scan_step, dict(u=_wide(2, BIG + 4), dt=_wide(2, BIG + 4), A=_wide(BIG + 4, 16), state=_wide(5, BIG + 4, 16)), "up to 16777216 channels"),
    (_kda, dict(q=_wide(BIG + 2, 2, 8), k=_wide(BIG + 2, 2, 8), v=_wide(BIG + 2, 4, 6), g=_wide(BIG + 2, 4, 8), beta=_wide(BIG + 2, 4),
                slots=z(1, dtype=N32).expand(BIG + 2)), "up to 2147483647 rows"),
    (_kda, dict(v=_wide(2, BIG + 4, 6), g=_wide(2, BIG + 4, 8), beta=_wide(2, BIG + 4), state=_wide(5, BIG + 4, 8, 6)), "up to 2147483647 heads"),
    (_kda, dict(q=_wide(2, BIG + 2, 8), k=_wide(2, BIG + 2, 8), v=_wide(2, BIG + 2, 6)), "up to 2147483647 heads"),
]


@pytest.mark.parametrize("call,kw,words", LARGE, ids=[f"{c.__name__[1:]}-{i}" for i, (c, _, _) in enumerate(LARGE)])
def test_sizes_that_32_bits_do_not_hold_are_refused(call, kw, words):
    """Narrowed before they were asked, 2^32 + 64 tokens would be 64: the rest of the output would never be written."""
    with pytest.raises(RuntimeError, match=words):
        call(**kw)


def test_workspaces_of_refused_sizes_are_none():
    import ctypes
    from rewy_b200 import _capi
    lib, most = _capi.load(), (1 << 31) - 1
    for name in ("rewy_conv_bwd_workspace_bytes", "rewy_scan_checkpoint_bytes", "rewy_scan_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_size_t
    for B, T, D in ((1, most, 64), (most, most, 64), (1, 64, most), (1 << 16, (1 << 14) + 1, 64)):
        assert lib.rewy_conv_bwd_workspace_bytes(B, T, D, 4) == 0
        assert lib.rewy_scan_checkpoint_bytes(B, T, D, 16) == 0
        assert lib.rewy_scan_workspace_bytes(B, T, D, 16, 1, 0) == lib.rewy_scan_workspace_bytes(B, T, D, 16, 1, 1) == 0
    assert lib.rewy_scan_checkpoint_bytes(1, 64, 64, 65) == 0
    assert lib.rewy_conv_bwd_workspace_bytes(1 << 16, 1 << 14, 64, 4) > 0 and lib.rewy_scan_workspace_bytes(1 << 16, 1 << 14, 64, 16, 1, 1) > 0


@pytest.mark.parametrize("family", (-1, 4, 7, 1 << 40))
def test_the_step_operator_itself_refuses_an_unknown_family(family):
    from rewy_b200 import _capi
    _capi.load_torch()
    step = torch.ops.rewy_b200.delta_step
    operands = (z(2, 2, 8), z(2, 2, 8), z(2, 4, 6), z(2, 4, 8), z(2, 4), None, None, z(5, 4, 8, 6), None, None, False, 0.0, None, None, False)
    with pytest.raises(RuntimeError, match=f"family must be 0 to 3, got {family}"):
        step(family, *operands)
    with pytest.raises(RuntimeError, match="step_kda: needs CUDA tensors"):
        step(_capi.KDA, *operands)


class Wrapper(torch.Tensor):
    """A tensor of the GPU by its device, without memory: what distributed and quantised subclasses are."""
    @staticmethod
    def __new__(cls, like):
        return torch.Tensor._make_wrapper_subclass(cls, like.shape, dtype=like.dtype, device="cuda")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} is not asked for")


def test_tensors_without_memory_are_refused():
    """Their address reads as NULL, which an entry takes for an operand that is not there."""
    x, gate, weight = Wrapper(z(3, 8)), Wrapper(z(3, 8)), Wrapper(z(8))
    assert x.is_cuda and x.data_ptr() == 0
    with pytest.raises(RuntimeError, match="needs tensors with memory of their own"):
        rewy_b200.gated_rms_norm(x, gate, weight)
    with pytest.raises(RuntimeError, match="needs tensors with memory of their own"):
        rewy_b200.causal_conv(Wrapper(z(2, 9, 16)), Wrapper(z(16, 4)), Wrapper(z(16)))
    with pytest.raises(RuntimeError, match="needs tensors with memory of their own"):
        rewy_b200.step_delta_rule(*(Wrapper(z(2, 4, 8)) for _ in range(3)), Wrapper(z(2, 4)), Wrapper(z(5, 4, 8, 8)))
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        fake = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        with pytest.raises(RuntimeError, match="needs tensors with memory of their own|Cannot access data pointer"):
            rewy_b200.residual_rms_norm(fake(3, 8), fake(3, 8), fake(8))


def test_counts_kept_elsewhere_join_the_report(monkeypatch):
    from rewy_b200 import layers, runtime
    rewy_b200.stats(reset=True)
    given = [{"causal_conv.optimized_backward": 2}, {}, {"causal_conv.optimized_backward": 1}]
    monkeypatch.setattr(runtime, "_elsewhere", [lambda: given.pop(0) if given else {}])
    rewy_b200.assert_used(("causal_conv",))
    assert rewy_b200.stats() == {"causal_conv.optimized_backward": 2}
    assert rewy_b200.stats(reset=True) == {"causal_conv.optimized_backward": 3} and rewy_b200.stats() == {}
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        _conv()
    assert layers._backwards() == {}     # the library is loaded and has nothing to add
