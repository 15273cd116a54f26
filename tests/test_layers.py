"""Host side of the operators around a recurrence: what they refuse, with which words, and that the package stays importable
without torch or the library.  No GPU is needed: every check stands in front of the one for CUDA tensors."""
import subprocess
import sys

import pytest
import torch

import rewy_b200
from conftest import ROOT

z = torch.zeros
F16 = torch.float16


def test_the_operators_load_on_first_use():
    code = "import sys, rewy_b200; assert 'torch' not in sys.modules; assert 'causal_conv' in dir(rewy_b200); print(rewy_b200.step_kda.__name__)"
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip() == "step_kda", run.stderr
    with pytest.raises(AttributeError, match="no attribute 'step_nothing'"):
        rewy_b200.step_nothing


def _conv(x=z(2, 9, 16), weight=z(16, 4), **kw):
    return rewy_b200.causal_conv(x, weight, **kw)


def _scan(**kw):
    a = dict(u=z(1, 9, 12), dt=z(1, 9, 12), A=z(12, 16), B=z(1, 9, 16), C=z(1, 9, 16))
    a.update(kw)
    return rewy_b200.selective_scan(**a)


def _conv_step(**kw):
    a = dict(x=z(2, 16), state=z(5, 3, 16), weight=z(16, 4))
    a.update(kw)
    return rewy_b200.causal_conv_step(**a)


def _scan_step(**kw):
    a = dict(u=z(2, 12), dt=z(2, 12), A=z(12, 16), B=z(2, 16), C=z(2, 16), state=z(5, 12, 16))
    a.update(kw)
    return rewy_b200.selective_scan_step(**a)


def _kda(**kw):
    a = dict(q=z(2, 2, 8), k=z(2, 2, 8), v=z(2, 4, 6), g=z(2, 4, 8), beta=z(2, 4), state=z(5, 4, 8, 6))
    a.update(kw)
    return rewy_b200.step_kda(**a)


def _gated(x=z(3, 8), gate=z(3, 8), weight=z(8), **kw):
    return rewy_b200.gated_rms_norm(x, gate, weight, **kw)


def _residual(x=z(3, 8), residual=z(3, 8), weight=z(8), **kw):
    return rewy_b200.residual_rms_norm(x, residual, weight, **kw)


CU = torch.tensor([0, 4, 9])
REFUSED = [
    (_conv, dict(x=z(2, 16)), r"x must have the shape \[B, T, D\]"),
    (_conv, dict(x=z(2, 0, 16)), "x must not be empty"),
    (_conv, dict(x=z(0, 9, 16)), "x must not be empty"),
    (_conv, dict(x=z(2, 9, 16, dtype=torch.float64)), "x must be BF16, FP16 or FP32"),
    (_conv, dict(x=z(2, 9, 16, dtype=torch.int32)), "x must be BF16, FP16 or FP32"),
    (_conv, dict(weight=z(16, 5)), "takes 2 to 4 taps, got 5"),
    (_conv, dict(weight=z(16, 1)), "takes 2 to 4 taps, got 1"),
    (_conv, dict(weight=z(15, 4)), r"weight must have the shape \[16, W\]"),
    (_conv, dict(weight=z(16, 4, dtype=torch.float64)), "weight must be BF16, FP16 or FP32"),
    (_conv, dict(bias=z(15)), r"bias must have the shape \[16\]"),
    (_conv, dict(bias=z(16, dtype=F16)), "bias must be Float, got Half"),
    (_conv, dict(initial_state=z(2, 4, 16)), r"initial_state must have the shape \[2, 3, 16\]"),
    (_conv, dict(initial_state=z(2, 3, 16, dtype=F16)), "initial_state must be Float"),
    (_conv, dict(cu_seqlens=CU), "packed sequences need a batch of 1"),
    (_conv, dict(x=z(1, 9, 16), cu_seqlens=torch.tensor([0, 4, 4, 9])), "positive lengths that add up to the token count"),
    (_conv, dict(x=z(1, 9, 16), cu_seqlens=torch.tensor([0, 4, 8])), "positive lengths that add up to the token count"),
    (_conv, dict(x=z(1, 9, 16), cu_seqlens=torch.tensor([1, 4, 9])), "positive lengths that add up to the token count"),
    (_conv, dict(x=z(1, 9, 16), cu_seqlens=torch.tensor([0, 5, 4, 9])), "positive lengths that add up to the token count"),
    (_conv, dict(x=z(1, 9, 16), cu_seqlens=CU.float()), "int32 or int64 offsets"),
    (_conv, dict(x=z(1, 9, 16), cu_seqlens=torch.tensor([0])), "offsets of one sequence or more"),
    (_conv, dict(x=z(1, 9, 16), cu_seqlens=CU, cu_seqlens_cpu=torch.tensor([0, 9])), "differ in length"),
    (_conv, dict(x=z(1, 9, 16), cu_seqlens_cpu=CU), "cu_seqlens_cpu goes with cu_seqlens"),
    (_conv, dict(x=z(1, 9, 16), cu_seqlens=CU, initial_state=z(1, 3, 16)), r"initial_state must have the shape \[2, 3, 16\]"),
    (_conv, dict(activation="gelu"), "activation must be None or 'silu', got 'gelu'"),
    (_conv, {}, "needs CUDA tensors"),
    (_scan, dict(u=z(9, 12)), r"u must have the shape \[B, T, M\]"),
    (_scan, dict(u=z(1, 0, 12)), "u must not be empty"),
    (_scan, dict(dt=z(1, 9, 1)), r"dt must have the shape \[1, 9, 12\]"),
    (_scan, dict(z=z(1, 8, 12)), r"z must have the shape"),
    (_scan, dict(A=z(12)), r"A must have the shape \[12, N\]"),
    (_scan, dict(A=z(12, 65)), "takes 1 to 64 states per channel, got 65"),
    (_scan, dict(A=z(12, 16, dtype=F16)), "A must be Float, got Half"),
    (_scan, dict(B=z(1, 9, 15)), "B must have the shape"),
    (_scan, dict(B=z(1, 9, 5, 16)), "G a divisor of the channels"),
    (_scan, dict(C=z(1, 9, 2, 16)), "B and C must have the same groups"),
    (_scan, dict(C=z(1, 9, 16, dtype=F16)), "C must be Float, got Half"),
    (_scan, dict(D=z(11)), r"D must have the shape \[12\]"),
    (_scan, dict(dt_bias=z(12, dtype=F16)), "dt_bias must be Float"),
    (_scan, dict(initial_state=z(1, 16, 12)), r"initial_state must have the shape \[1, 12, 16\]"),
    (_scan, {}, "needs CUDA tensors"),
    (_conv_step, dict(x=z(2, 1, 16)), r"x must have the shape \[B, D\]"),
    (_conv_step, dict(state=z(5, 4, 16)), r"state must have the shape \[pool, 3, 16\]"),
    (_conv_step, dict(state=z(5, 3, 16, dtype=F16)), "state must be Float"),
    (_conv_step, dict(state=z(5, 16, 3).transpose(1, 2)), "updated in place and must be contiguous"),
    (_conv_step, dict(state=z(1, 3, 16)), "1 states for 2 rows"),
    (_conv_step, dict(slots=torch.tensor([0.0, 1.0])), "slots must be int32 or int64"),
    (_conv_step, dict(slots=torch.tensor([0])), r"slots must have the shape \[2\]"),
    (_conv_step, dict(x=z(2, 16, requires_grad=True)), "a step has no gradient"),
    (_conv_step, {}, "needs CUDA tensors"),
    (_scan_step, dict(u=z(2, 1, 12)), r"u must have the shape \[B, M\]"),
    (_scan_step, dict(state=z(5, 16, 12)), r"state must have the shape \[pool, 12, 16\]"),
    (_scan_step, dict(state=z(5, 12, 16, dtype=F16)), "state must be Float"),
    (_scan_step, dict(state=z(1, 12, 16)), "1 states for 2 rows"),
    (_scan_step, dict(A=z(12, 16, requires_grad=True)), "a step has no gradient"),
    (_scan_step, {}, "needs CUDA tensors"),
    (_kda, dict(k=z(2, 2, 7)), r"k must have the shape \[2, 2, 8\]"),
    (_kda, dict(v=z(2, 3, 6)), "must be a multiple of the query/key heads"),
    (_kda, dict(q=z(2, 2, 129), k=z(2, 2, 129)), "head dimensions above 128"),
    (_kda, dict(g=z(2, 4)), r"g must have the shape \[2, 4, 8\]"),
    (_kda, dict(g=None), "g must be given"),
    (_kda, dict(beta=z(2, 2)), r"beta must have the shape \[2, 4\]"),
    (_kda, dict(state=z(5, 4, 6, 8)), r"state must have the shape \[pool, 4, 8, 6\]"),
    (_kda, dict(state=z(5, 4, 8, 6), state_v_first=True), r"state must have the shape \[pool, 4, 6, 8\]"),
    (_kda, dict(state=z(5, 4, 8, 6, dtype=F16)), "state must be Float"),
    (_kda, dict(use_gate_in_kernel=True), "A_log must be provided"),
    (_kda, dict(use_gate_in_kernel=True, A_log=z(3)), r"A_log must have the shape \[4\]"),
    (_kda, dict(allow_neg_eigval=True), "requires `use_beta_sigmoid_in_kernel=True`"),
    (_kda, dict(v=z(2, 4, 6, dtype=F16)), "v must be Float"),
    (_kda, {}, "needs CUDA tensors"),
    (_gated, dict(gate=z(3, 7)), r"gate must have the shape \[3, 8\]"),
    (_gated, dict(gate=z(3, 8, dtype=F16)), "gate must be Float"),
    (_gated, dict(weight=z(7)), r"weight must have the shape \[8\]"),
    (_gated, dict(x=z(0, 8), gate=z(0, 8)), "x must have rows of values"),
    (_gated, dict(x=z(1, 16385), gate=z(1, 16385), weight=z(16385)), "rows of up to 16384 values"),
    (_gated, dict(activation="tanh"), "activation must be 'silu' or 'sigmoid'"),
    (_gated, {}, "needs CUDA tensors"),
    (_residual, dict(residual=z(8)), r"residual must have the shape \[3, 8\]"),
    (_residual, dict(residual=z(3, 8, dtype=F16)), "residual must have the type of x or FP32"),
    (_residual, dict(scale=z(3)), r"scale must have the shape \[8\]"),
    (_residual, {}, "needs CUDA tensors"),
]


@pytest.mark.parametrize("call,kw,words", REFUSED, ids=[f"{c.__name__[1:]}-{i}" for i, (c, _, _) in enumerate(REFUSED)])
def test_refusals(call, kw, words):
    before = rewy_b200.stats()
    with pytest.raises((RuntimeError, ValueError), match=words):
        call(**kw)
    assert rewy_b200.stats() == before


def test_workspace_sizes():
    """What the C entries ask for: nothing for shapes that they refuse, the sums' and segments' room otherwise."""
    import ctypes
    from rewy_b200 import _capi
    lib = _capi.load()
    for name in ("rewy_conv_bwd_workspace_bytes", "rewy_scan_checkpoint_bytes", "rewy_scan_workspace_bytes", "rewy_norm_bwd_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_size_t
    assert lib.rewy_conv_bwd_workspace_bytes(1, 100, 0, 4) == lib.rewy_conv_bwd_workspace_bytes(1, 100, 64, 5) == 0
    assert lib.rewy_scan_workspace_bytes(1, 100, 64, 65, 1, 1) == lib.rewy_scan_workspace_bytes(1, 100, 64, 16, 3, 1) == 0
    assert lib.rewy_scan_checkpoint_bytes(2, 33, 64, 16) == 2 * 3 * 64 * 16 * 4
    assert lib.rewy_scan_workspace_bytes(8, 4096, 4096, 16, 1, 0) == 0                      # one segment: no joining
    assert lib.rewy_scan_workspace_bytes(1, 4096, 64, 16, 1, 0) > 0
    assert lib.rewy_norm_bwd_workspace_bytes(ctypes.c_int64(0), 64) == 0
    assert lib.rewy_norm_bwd_workspace_bytes(ctypes.c_int64(5), 16384) == 5 * 2 * 16384 * 4


def test_c_entries_refuse_what_they_do_not_take():
    import ctypes
    from rewy_b200 import _capi
    lib = _capi.load()
    for name in ("rewy_conv_fwd", "rewy_conv_bwd", "rewy_conv_step", "rewy_scan_fwd", "rewy_scan_bwd", "rewy_scan_step", "rewy_gated_norm_fwd",
                 "rewy_gated_norm_bwd", "rewy_residual_norm_fwd", "rewy_residual_norm_bwd", "rewy_delta_step"):
        fn = getattr(lib, name)
        assert fn(None, None) == 1, name                                                    # REWY_ERR_NULL
        blank = (ctypes.c_char * 1024)()
        assert fn(ctypes.byref(blank), None) not in (0, 5), name                            # zeros: refused before any launch
        assert lib.rewy_last_error()
