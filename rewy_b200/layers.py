"""Operators around a recurrence in a layer, for training, prompts and single tokens.

    causal_conv, causal_conv_step          the short causal convolution in front of a recurrence, with its activation and state
    selective_scan, selective_scan_step    the selective state space scan, with its time step, skip and gate
    gated_rms_norm                         the norm behind a recurrence with the layer's gate
    residual_rms_norm                      the residual sum with the block's scale and the norm in front of the next block
    step_kda, step_gated_delta_rule,       one token of the delta rules whose chunked operators are in ``functions``: the
    step_gdn2, step_delta_rule             form in which a model answers

All of them are CUDA kernels behind torch operators (csrc/layers.cpp); there is no CPU or PyTorch fallback.  Activations are
BF16, FP16 or FP32, one type per call; parameters of the norms and the convolution have any of the three; recurrent states, A,
D and dt_bias are FP32.  Layouts are token-major; tensors may be views with any strides (rows whose elements are not
neighbours are copied first).  Every sum is FP32 and every output is rounded once; results repeat bit for bit.  Packed
sequences work as in the chunked operators (``cu_seqlens``, batch 1, positive lengths; ``cu_seqlens_cpu`` avoids a copy to the
host, which a captured call must avoid).  Gradients are first order and reverse mode: forward mode raises.

The steps update ``state``, which must be contiguous, in place.  With ``slots`` (int32 or int64, one per row) row b works on ``state[slots[b]]`` of a
pool; a row whose index lies outside the pool (-1: a padded row), or is that of a row before it, is skipped: its output is
zero and no state changes.
"""
import torch

from . import _capi
from .runtime import count_elsewhere, record


def _backwards():
    """Backwards since the last call, which autograd runs without passing through Python (csrc/layers.cpp)."""
    if not _loaded:
        return {}
    counts = torch.ops.rewy_b200.layer_backwards()
    return {f"{name}.optimized_backward": n for name, n in zip(_TRAINED, counts) if n}


_TRAINED = ("causal_conv", "selective_scan", "gated_rms_norm", "residual_rms_norm")   # in the library's order
_loaded = False
count_elsewhere(_backwards)


def _operator(op, kind=None):
    """The torch operator ``op``, loaded with its first call; calls count as ``kind``."""
    fn, kind = None, kind or op

    def call(*args):
        global _loaded
        nonlocal fn
        if fn is None:
            _capi.load_torch()
            _loaded = True
            fn = getattr(torch.ops.rewy_b200, op).default
        out = fn(*args)
        record(kind, "optimized_forward")
        return out

    return call


_causal_conv = _operator("causal_conv")
_causal_conv_step = _operator("causal_conv_step")
_selective_scan = _operator("selective_scan")
_selective_scan_step = _operator("selective_scan_step")
_gated_rms_norm = _operator("gated_rms_norm")
_residual_rms_norm = _operator("residual_rms_norm")
_delta_step = {name: _operator("delta_step", name) for name in ("step_kda", "step_gated_delta_rule", "step_gdn2", "step_delta_rule")}


def _silu(op, activation):
    if activation not in (None, "silu", "swish"):
        raise ValueError(f"rewy_b200 {op}: activation must be None or 'silu', got {activation!r}")
    return activation is not None


@torch.compiler.disable
def causal_conv(x, weight, bias=None, *, activation=None, initial_state=None, output_final_state=False, cu_seqlens=None,
                cu_seqlens_cpu=None):
    """Causal convolution per channel: y_t = act(bias + sum_w weight[:, w] x_(t-W+1+w)).  x [B,T,D]; weight [D,W] (or
    [D,1,W]) with 2 <= W <= 4; bias [D]; activation None or "silu".  ``initial_state`` [B,W-1,D] (packed: [sequences,W-1,D]) in the
    type of x holds the inputs before each sequence, the oldest first (default zeros).  Returns (y, final_state or None)."""
    return _causal_conv(x, weight, bias, _silu("causal_conv", activation), initial_state, output_final_state,
                 cu_seqlens, cu_seqlens_cpu)


@torch.compiler.disable
def causal_conv_step(x, state, weight, bias=None, *, activation=None, slots=None):
    """One token of ``causal_conv`` per row: x [B,D], state [pool,W-1,D] updated in place.  Returns y [B,D]."""
    return _causal_conv_step(x, state, weight, bias, _silu("causal_conv_step", activation), slots)


@torch.compiler.disable
def selective_scan(u, dt, A, B, C, D=None, *, z=None, dt_bias=None, dt_softplus=False, initial_state=None,
                   output_final_state=False, cu_seqlens=None, cu_seqlens_cpu=None):
    """Selective state space scan.  With dt = softplus(dt + dt_bias) (``dt_softplus``) or dt + dt_bias:

        h_t = exp(dt_t A) h_(t-1) + dt_t u_t B_t,    y_t = (C_t h_t + D u_t) silu(z_t)

    u, dt, z [B,T,M]; A [M,N]; B, C [B,T,G,N] or [B,T,N] (channel m reads group m // (M // G)); D, dt_bias [M]; N up to 64;
    ``initial_state`` [B,M,N] (packed: [sequences,M,N]).  Returns (y, final_state or None)."""
    return _selective_scan(u, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, output_final_state,
                 cu_seqlens, cu_seqlens_cpu)


@torch.compiler.disable
def selective_scan_step(u, dt, A, B, C, state, D=None, *, z=None, dt_bias=None, dt_softplus=False, slots=None):
    """One token of ``selective_scan`` per row: u, dt, z [B,M], B, C [B,G,N] or [B,N], state [pool,M,N] updated in place.
    Returns y [B,M]."""
    return _selective_scan_step(u, dt, A, B, C, state, D, z, dt_bias, dt_softplus, slots)


@torch.compiler.disable
def gated_rms_norm(x, gate, weight, *, eps=1e-6, activation="silu", gate_first=False):
    """n(x) * weight * act(gate) over the last dimension (up to 16384), or with ``gate_first`` n(x * act(gate)) * weight;
    n(v) = v / sqrt(mean(v^2) + eps), squares in FP32: with eps = 0 rows down to an rms of 1e-18.  x, gate [..., D]; weight [D];
    activation "silu" or "sigmoid"."""
    if activation not in ("silu", "swish", "sigmoid"):
        raise ValueError(f"rewy_b200 gated_rms_norm: activation must be 'silu' or 'sigmoid', got {activation!r}")
    return _gated_rms_norm(x, gate, weight, eps, int(activation == "sigmoid"), gate_first)


@torch.compiler.disable
def residual_rms_norm(x, residual, weight, *, scale=None, eps=1e-6):
    """residual_out = residual + scale * x, y = n(residual_out) * weight over the last dimension (up to 16384).  x [..., D];
    residual of the same shape, in the type of x or FP32, or None; scale a number or a tensor [D] with a gradient.  The norm
    is that of the sum before it is rounded to the residual's type.  Returns (y, residual_out)."""
    vector = scale if isinstance(scale, torch.Tensor) else None
    number = 1.0 if scale is None or vector is not None else float(scale)
    return _residual_rms_norm(x, residual, weight, vector, number, eps)


def _step(name, family, q, k, v, state, *, g=None, beta=None, b=None, w=None, scale=None, slots=None, qk_norm=False, beta_scale=0.0,
          A_log=None, dt_bias=None, state_v_first=False):
    return _delta_step[name](_capi.FAMILY_ID[family], q, k, v, g, beta, b, w, state, scale, slots, qk_norm, beta_scale,
                 A_log, dt_bias, state_v_first)


def _beta_scale(use_sigmoid, allow_neg_eigval):
    if allow_neg_eigval and not use_sigmoid:
        raise ValueError("`allow_neg_eigval=True` requires `use_beta_sigmoid_in_kernel=True`.")
    return (2.0 if allow_neg_eigval else 1.0) if use_sigmoid else 0.0


def _need(name, **tensors):
    for n, t in tensors.items():
        if t is None:
            raise ValueError(f"rewy_b200 {name}: {n} must be given")


@torch.compiler.disable
def step_kda(q, k, v, g, beta, state, *, scale=None, slots=None, use_qk_l2norm_in_kernel=False, use_gate_in_kernel=False,
             use_beta_sigmoid_in_kernel=False, allow_neg_eigval=False, A_log=None, dt_bias=None, state_v_first=False):
    """One token of ``chunk_kda`` per row.  q, k [B,H,K]; v [B,HV,V]; g [B,HV,K] natural-log decay, or the raw gate input with
    ``use_gate_in_kernel`` (then ``A_log`` with HV values and optionally ``dt_bias`` with HV*K); beta [B,HV]; state [pool,HV,K,V] FP32 ([pool,HV,V,K]
    with ``state_v_first``) updated in place; HV a multiple of H, K and V up to 128.  Returns o [B,HV,V]."""
    _need("step_kda", g=g, beta=beta)
    if use_gate_in_kernel and A_log is None:
        raise ValueError("A_log must be provided when use_gate_in_kernel=True.")
    flat = lambda t: None if t is None else t.float().reshape(-1)  # noqa: E731  (as the chunked operator takes them)
    gate = dict(A_log=flat(A_log), dt_bias=flat(dt_bias)) if use_gate_in_kernel else {}
    return _step("step_kda", "kda", q, k, v, state, g=g, beta=beta, scale=scale, slots=slots, qk_norm=use_qk_l2norm_in_kernel,
                 beta_scale=_beta_scale(use_beta_sigmoid_in_kernel, allow_neg_eigval), state_v_first=state_v_first, **gate)


@torch.compiler.disable
def step_gated_delta_rule(q, k, v, g, beta, state, *, scale=None, slots=None, use_qk_l2norm_in_kernel=False,
                          use_beta_sigmoid_in_kernel=False, allow_neg_eigval=False, state_v_first=False):
    """One token of ``chunk_gated_delta_rule`` per row: as ``step_kda`` with one decay per head, g [B,HV]."""
    _need("step_gated_delta_rule", g=g, beta=beta)
    return _step("step_gated_delta_rule", "gdn", q, k, v, state, g=g, beta=beta, scale=scale, slots=slots,
                 qk_norm=use_qk_l2norm_in_kernel, beta_scale=_beta_scale(use_beta_sigmoid_in_kernel, allow_neg_eigval),
                 state_v_first=state_v_first)


@torch.compiler.disable
def step_gdn2(q, k, v, g, b, w, state, *, scale=None, slots=None, use_qk_l2norm_in_kernel=False, state_v_first=False):
    """One token of ``chunk_gdn2`` per row: as ``step_kda`` with the erase gate b [B,HV,K] and the write gate w [B,HV,V] in the
    type of q instead of beta."""
    _need("step_gdn2", g=g, b=b, w=w)
    return _step("step_gdn2", "gdn2", q, k, v, state, g=g, b=b, w=w, scale=scale, slots=slots, qk_norm=use_qk_l2norm_in_kernel,
                 state_v_first=state_v_first)


@torch.compiler.disable
def step_delta_rule(q, k, v, beta, state, *, scale=None, slots=None, use_qk_l2norm_in_kernel=False, state_v_first=False):
    """One token of ``chunk_delta_rule`` per row: as ``step_kda`` without a decay."""
    _need("step_delta_rule", beta=beta)
    return _step("step_delta_rule", "delta", q, k, v, state, beta=beta, scale=scale, slots=slots, qk_norm=use_qk_l2norm_in_kernel,
                 state_v_first=state_v_first)
