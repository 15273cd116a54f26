"""Operators around a recurrence against their FP64 definitions: types, odd sizes, strides, packed sequences, states, gradients,
single tokens, streams, graphs.

Tolerances.  An output is rounded once: at most half a step of its type relative to the value (bf16 2^-8, fp16 2^-11, fp32
2^-24).  In front of that stands FP32 arithmetic: a sum of n terms in which each is off by a few 2^-24 is off by about
sqrt(n) 2^-23 of its norm (n <= 1000 here: 4e-6), a decay by 3 2^-23 per step of the state's memory; 2e-5 of the norm covers
both.  Element by element a sum may cancel, so the bound there is half a step of the value plus 1e-4 of the output's rms."""
import pytest
import torch

import rewy_b200
from oracle import layers as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=gen, device=DEV)


def _close(got, want, name, cancels=0.0):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    half = torch.finfo(got.dtype).eps / 2
    got, want = got.detach().double(), want.detach().double()
    off, rms = (got - want).abs(), want.square().mean().sqrt()
    assert torch.isfinite(got).all(), name
    assert off.norm() <= (half + 2e-5) * want.norm() + cancels * want.numel() ** 0.5 + 1e-12, (name, (off.norm() / want.norm()).item())
    assert (off <= half * want.abs() * 1.001 + 1e-4 * rms + cancels + 1e-12).all(), (name, (off / rms).max().item())


def _leaves(xs):
    return {n: (x.detach().clone().requires_grad_() if isinstance(x, torch.Tensor) else x) for n, x in xs.items()}


def _compare(call, reference, xs, out_dtypes, cancels=lambda seeds: {}):
    """Outputs and all gradients of ``call`` against those of ``reference`` on the same values in FP64.  ``cancels`` gives what
    a gradient may be off by beside its own size, where it is a difference of larger numbers."""
    mine, exact = _leaves(xs), _leaves({n: x.double() if isinstance(x, torch.Tensor) else x for n, x in xs.items()})
    got, want = call(**mine), reference(**exact)
    rn = _gen(99)
    seeds = [rn(*w.shape).to(t) for w, t in zip(want, out_dtypes)]
    names = [n for n, x in xs.items() if isinstance(x, torch.Tensor)]
    for i, (g, w, t) in enumerate(zip(got, want, out_dtypes)):
        assert g.dtype == t
        _close(g, w, f"output {i}")
    grads = torch.autograd.grad(got, [mine[n] for n in names], seeds)
    exacts = torch.autograd.grad(want, [exact[n] for n in names], [s.double() for s in seeds])
    extra = cancels(seeds)
    for n, g, w in zip(names, grads, exacts):
        assert g.dtype == xs[n].dtype, n
        _close(g, w, f"d{n}", extra.get(n, 0.0))
    with torch.no_grad():
        for g, again in zip(got, call(**mine)):
            assert torch.equal(g, again)
    return got, grads


def _cu(lengths):
    if lengths is None:
        return {}, None
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(lengths).cumsum(0)])
    return dict(cu_seqlens=cu.to(DEV, torch.int32), cu_seqlens_cpu=cu), cu.tolist()


# ---- causal convolution ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("B,T,D,lengths", [(1, 1, 8, None), (2, 3, 13, None), (3, 77, 264, None), (1, 600, 40, (1, 2, 3, 250, 8, 336)), (2, 520, 1000, None)])
@pytest.mark.parametrize("W,bias,activation,state", [(4, True, "silu", True), (3, False, None, True), (2, True, "silu", False), (4, False, "silu", True)])
def test_causal_conv(dtype, B, T, D, lengths, W, bias, activation, state):
    rn = _gen(1)
    kw, cu = _cu(lengths)
    sequences = len(lengths) if lengths else B
    xs = dict(x=rn(B, T, D).to(dtype), weight=rn(D, W) / 2)
    if bias:
        xs["bias"] = rn(D)
    if state:
        xs["initial_state"] = rn(sequences, W - 1, D).to(dtype)

    def call(**x):
        y, fin = rewy_b200.causal_conv(**x, activation=activation, output_final_state=state, **kw)
        assert (fin is not None) == state
        return (y, fin) if state else (y,)

    def reference(**x):
        return oracle.causal_conv(**x, activation=activation, cu=cu)[:2 if state else 1]

    _compare(call, reference, xs, (dtype, dtype) if state else (dtype,))


@pytest.mark.parametrize("dtype", (BF16, FP32))
def test_causal_conv_takes_views_and_module_weights(dtype):
    """A slice of a wider projection (aligned and not), a transposed input, a [D, 1, W] weight in the activations' type."""
    rn = _gen(2)
    wide = rn(2, 50, 200).to(dtype)
    weight = (rn(96, 1, 4) / 2).to(dtype)
    for x in (wide[..., 8:104], wide[..., 3:99], rn(2, 96, 50).to(dtype).transpose(1, 2), wide[:1, :, :96].expand(2, -1, -1)):
        w = weight.detach().clone().requires_grad_()
        x = x.detach().requires_grad_()
        y, fin = rewy_b200.causal_conv(x, w, activation="silu", output_final_state=True)
        x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
        want, state = oracle.causal_conv(x64, w64[:, 0], activation="silu")
        _close(y, want, "y")
        assert torch.equal(fin.double(), state)
        dy = rn(2, 50, 96).to(dtype)
        for g, e in zip(torch.autograd.grad(y, (x, w), dy), torch.autograd.grad(want, (x64, w64), dy.double())):
            _close(g, e, "gradient")


# ---- selective scan --------------------------------------------------------------------------------------------------

def _scan_inputs(rn, B, T, M, N, G, dtype, sequences, options):
    xs = dict(u=rn(B, T, M).to(dtype), dt=rn(B, T, M).to(dtype) if "softplus" in options else (0.3 * rn(B, T, M).abs()).to(dtype),
              A=-torch.rand(M, N, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)) * 2 - 0.05, B=rn(B, T, G, N).to(dtype), C=rn(B, T, G, N).to(dtype))
    if "skip" in options:
        xs["D"] = rn(M)
    if "gate" in options:
        xs["z"] = rn(B, T, M).to(dtype)
    if "softplus" in options:
        xs["dt_bias"] = rn(M) - 2
    if "state" in options:
        xs["initial_state"] = rn(sequences, M, N)
    return xs


def _scan_pair(options, kw, cu):
    state, flags = "state" in options, dict(dt_softplus="softplus" in options)

    def call(**x):
        return rewy_b200.selective_scan(**x, **flags, output_final_state=state, **kw)[:2 if state else 1]

    def reference(**x):
        return oracle.selective_scan(**x, **flags, cu=cu)[:2 if state else 1]

    return call, reference


ALL = ("skip", "gate", "softplus", "state")


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("B,T,M,N,G,lengths,options", [
    (1, 1, 8, 16, 1, None, ALL),                                        # one token
    (2, 17, 13, 5, 1, None, ALL),                                       # nothing divides anything
    (1, 33, 40, 1, 2, None, ("gate", "softplus")),                      # one state
    (2, 100, 64, 16, 2, None, ()),                                      # the bare recurrence
    (1, 70, 24, 64, 3, None, ("skip", "state")),                        # most states
    (3, 48, 36, 20, 1, None, ALL),                                      # 20 states on 8 lanes
    (1, 150, 72, 16, 1, (1, 15, 16, 17, 32, 1, 1, 67), ALL),            # sequences that begin inside tiles and at their ends
    (1, 64, 2400, 16, 1, (20, 44), ("softplus", "gate")),               # enough channels for one segment
])
def test_selective_scan(dtype, B, T, M, N, G, lengths, options):
    kw, cu = _cu(lengths)
    xs = _scan_inputs(_gen(4), B, T, M, N, G, dtype, len(lengths) if lengths else B, options)
    _compare(*_scan_pair(options, kw, cu), xs, (dtype, FP32) if "state" in options else (dtype,))


@pytest.mark.parametrize("N", (3, 8, 16, 32, 64))
@pytest.mark.parametrize("B,T,lengths", [(1, 1000, None), (2, 641, None), (1, 1000, (1, 127, 128, 300, 84, 320, 40)), (1, 1000, (999, 1)), (1, 768, (256, 128, 384))])
def test_selective_scan_in_segments(B, T, lengths, N):
    """Few channels: the token axis is cut; sequences begin inside segments, at their ends, and span several."""
    kw, cu = _cu(lengths)
    xs = _scan_inputs(_gen(5), B, T, 24, N, 1, FP32, len(lengths) if lengths else B, ALL)
    _compare(*_scan_pair(ALL, kw, cu), xs, (FP32, FP32))


def test_selective_scan_takes_views():
    """u and z halves of one projection, B and C slices of another with a common odd offset, a transposed dt, [B,T,N] factors."""
    rn = _gen(6)
    for dtype in (BF16, FP32):
        for shift in (0, 3):
            wide, proj = rn(2, 60, 97 * 2).to(dtype), rn(2, 60, 40 + 8).to(dtype)
            M = 96 if shift == 0 else 95
            u, z = wide[..., :M], wide[..., 96:96 + M]
            Bm, C = proj[..., shift:shift + 16], proj[..., 16 + shift:32 + shift]
            dt = (0.2 * rn(2, M, 60).abs()).to(dtype).transpose(1, 2)
            A = -rn(M, 16).abs()
            y, fin = rewy_b200.selective_scan(u, dt, A, Bm, C, z=z, output_final_state=True)
            want, state = oracle.selective_scan(u.double(), dt.double(), A.double(), Bm.double()[:, :, None], C.double()[:, :, None], z=z.double())
            _close(y, want, "y")
            _close(fin, state, "state")


def test_selective_scan_keeps_to_extreme_steps():
    """A step of zero leaves the state alone, a very long one forgets it, in both directions of the time axis."""
    rn, T = _gen(7), 40
    dt = torch.zeros(1, T, 32, device=DEV)
    dt[:, ::5] = 1e4
    dt[:, 1::7] = 0.5
    xs = dict(u=rn(1, T, 32), dt=dt, A=-rn(32, 16).abs() - 0.1, B=rn(1, T, 1, 16), C=rn(1, T, 1, 16), initial_state=rn(1, 32, 16))
    call, reference = _scan_pair(("state",), {}, None)
    _compare(call, reference, xs, (FP32, FP32))


# ---- norms -----------------------------------------------------------------------------------------------------------

def _norm_cancels(v, dn, factors):
    """The gradient of a norm is r dn - v r^3 mean(dn v): with one value in a row the two are equal but for eps, and what is left is
    eps / v^2 of either.  Each is at most r max|dn| (the mean of dn n, |n| <= sqrt(D), n / sqrt(D) a unit vector: r |n| |mean dn n|
    <= r sqrt(D) max|dn|) and off by its roundings, fewer than 16 of 2^-24: the square sum, the division, r three times, the
    products.  So the difference is off by at most 2^-20 r sqrt(D) max|dn| however small it is itself; ``factors`` is what
    multiplies it on the way to each input.  At D >= 64 in these tests that is below 1e-5 of the gradients' own size."""
    v = v.double()
    D = v.shape[-1]
    r = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6)
    off = 2.0 ** -20 * D ** 0.5 * (r * dn.double().abs()).max().item()
    return {n: off * f for n, f in factors.items()}


WIDTHS = [(5, 1), (1, 64), (300, 128), (37, 96), (70, 130), (33, 256), (9, 1000), (21, 1024), (5, 1030), (40, 4096), (3, 8192), (2, 9001), (2, 16384)]


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("rows,D", WIDTHS)
@pytest.mark.parametrize("activation,gate_first", [("silu", False), ("sigmoid", True), ("silu", True)])
def test_gated_rms_norm(dtype, rows, D, activation, gate_first):
    rn = _gen(8)
    xs = dict(x=(2 * rn(rows, D)).to(dtype), gate=rn(rows, D).to(dtype), weight=1 + 0.2 * rn(D))
    kw = dict(activation=activation, gate_first=gate_first, eps=1e-5)
    s, top = oracle.act(activation, xs["gate"].double()), lambda v: v.double().abs().max().item()
    dn = lambda seeds: seeds[0].double() * xs["weight"].double() * (1 if gate_first else s)  # noqa: E731
    cancels = lambda seeds: _norm_cancels(xs["x"].double() * (s if gate_first else 1), dn(seeds),  # noqa: E731
                                          {"x": top(s), "gate": 1.1 * top(xs["x"])} if gate_first else {"x": 1.0})
    _compare(lambda **x: (rewy_b200.gated_rms_norm(**x, **kw),), lambda **x: (oracle.gated_rms_norm(**x, **kw),), xs, (dtype,), cancels)


@pytest.mark.parametrize("dtype,residual_dtype", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP16, FP32), (FP32, FP32), (BF16, None)])
@pytest.mark.parametrize("rows,D", WIDTHS)
@pytest.mark.parametrize("scale", (None, 0.3, "channel"))
def test_residual_rms_norm(dtype, residual_dtype, rows, D, scale):
    rn = _gen(9)
    xs = dict(x=rn(rows, D).to(dtype), residual=None if residual_dtype is None else (2 * rn(rows, D)).to(residual_dtype), weight=1 + 0.2 * rn(D),
              scale=0.5 + rn(D) if scale == "channel" else scale)
    number = 1.0 if scale is None else xs["scale"]
    total, top = number * xs["x"].double() + (0 if xs["residual"] is None else xs["residual"].double()), lambda v: v.double().abs().max().item()
    cancels = lambda seeds: _norm_cancels(total, seeds[0].double() * xs["weight"].double(),  # noqa: E731
                                          {"x": top(torch.as_tensor(number)), "residual": 1.0, "scale": rows * top(xs["x"])})
    _compare(lambda **x: rewy_b200.residual_rms_norm(**x), lambda **x: oracle.residual_rms_norm(**{**x, "scale": 1.0 if x["scale"] is None else x["scale"]}),
             xs, (dtype, residual_dtype or dtype), cancels)


def test_norms_take_views_and_many_rows():
    """Heads of a projection's slice, a transposed batch, an expanded gate; more rows than one grid takes at once."""
    rn = _gen(10)
    proj, weight = rn(3, 50, 6 * 128 + 8).to(BF16), 1 + 0.1 * rn(128)
    x = rn(3, 50, 6, 128).to(BF16)
    for gate in (proj[..., :768].unflatten(-1, (6, 128)), proj[..., 5:773].unflatten(-1, (6, 128)), x.transpose(0, 1).contiguous().transpose(0, 1),
                 proj[..., None, :128].expand(-1, -1, 6, -1), rn(3, 50, 128, 6).to(BF16).transpose(-1, -2)):
        _close(rewy_b200.gated_rms_norm(x, gate, weight), oracle.gated_rms_norm(x.double(), gate.double(), weight.double()), "gated")
        y, r = rewy_b200.residual_rms_norm(gate, x, weight, scale=0.5)
        want = oracle.residual_rms_norm(gate.double(), x.double(), weight.double(), 0.5)
        _close(y, want[0], "residual norm")
        _close(r, want[1], "residual")
    big = [rn(70001, 64).to(BF16) for _ in range(2)]
    weight = (1 + 0.1 * rn(64)).to(BF16)
    xs = dict(x=big[0], gate=big[1], weight=weight)
    mine, exact = _leaves(xs), _leaves({n: v.double() for n, v in xs.items()})
    y, want = rewy_b200.gated_rms_norm(**mine), oracle.gated_rms_norm(**exact)
    for n, g, e in zip(xs, torch.autograd.grad(y, list(mine.values()), big[0]), torch.autograd.grad(want, list(exact.values()), big[0].double())):
        _close(g, e, n)


# ---- single tokens ---------------------------------------------------------------------------------------------------

def _slots(B, pool, kind):
    """Rows with slots in no order, one padded (-1), one beyond the pool and one that repeats an earlier row's."""
    slots = torch.randperm(pool, generator=torch.Generator().manual_seed(B))[:B]
    live = torch.ones(B, dtype=torch.bool)
    if B >= 6:
        slots[1], slots[3], slots[5] = -1, pool, slots[0]
        live[[1, 3, 5]] = False
    return slots.to(DEV, kind), slots.clamp(0, pool - 1).to(DEV), live.to(DEV)


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("B,D,W,kind", [(1, 8, 4, torch.int32), (7, 13, 3, torch.int64), (70, 1000, 4, torch.int32), (300, 40, 2, torch.int32)])
def test_causal_conv_step(dtype, B, D, W, kind):
    rn = _gen(11)
    x, state, weight, bias = rn(B, D).to(dtype), rn(B + 3, W - 1, D).to(dtype), rn(D, W) / 2, rn(D)
    slots, at, live = _slots(B, B + 3, kind)
    before = state.clone()
    y = rewy_b200.causal_conv_step(x, state, weight, bias, activation="silu", slots=slots)
    want, new = oracle.causal_conv(x[:, None].double(), weight.double(), bias.double(), "silu", before[at].double())
    _close(y, want[:, 0] * live[:, None], "y")
    expected = before.clone()
    expected[at[live]] = new[live].to(dtype)
    assert torch.equal(state, expected)
    old = before.clone()
    y = rewy_b200.causal_conv_step(x, before, weight)       # without slots: row b has state b
    _close(y, oracle.causal_conv(x[:, None].double(), weight.double(), initial_state=old[:B].double())[0][:, 0], "y")
    assert torch.equal(before[:B, -1], x) and torch.equal(before[:B, :-1], old[:B, 1:]) and torch.equal(before[B:], old[B:])


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("B,M,N,G,kind", [(1, 8, 16, 1, torch.int32), (7, 26, 5, 2, torch.int64), (70, 1000, 16, 1, torch.int32), (9, 36, 64, 3, torch.int32),
                                          (300, 40, 20, 1, torch.int32)])
def test_selective_scan_step(dtype, B, M, N, G, kind):
    rn = _gen(12)
    xs = _scan_inputs(rn, B, 1, M, N, G, dtype, B + 3, ALL)
    state = xs.pop("initial_state")
    slots, at, live = _slots(B, B + 3, kind)
    before = state.clone()
    one = {n: x[:, 0] if x.dim() > 2 else x for n, x in xs.items()}
    y = rewy_b200.selective_scan_step(**one, state=state, dt_softplus=True, slots=slots)
    want, new = oracle.selective_scan(**{n: x.double() for n, x in xs.items()}, dt_softplus=True, initial_state=before[at].double())
    _close(y, want[:, 0] * live[:, None], "y")
    _close(state[at[live]], new[live], "state")
    rest = torch.ones(B + 3, dtype=torch.bool, device=DEV)
    rest[at[live]] = False
    assert torch.equal(state[rest], before[rest])


def _delta_reference(family, xs, state, groups, options):
    """One token by the recurrence of the chunked operators' oracle."""
    from oracle import recurrence
    x = {n: v.double().cpu() for n, v in xs.items()}
    if options:
        x["q"], x["k"] = (x[n] / torch.sqrt(x[n].square().sum(-1, keepdim=True) + 1e-6) for n in ("q", "k"))
        if "beta" in x:
            x["beta"] = torch.sigmoid(x["beta"])
        if family == "kda":
            HV, K = x["g"].shape[1:]
            x["g"] = -torch.exp(x.pop("A_log"))[:, None] * torch.nn.functional.softplus(x["g"] + x.pop("dt_bias").view(HV, K), threshold=700.0)
    x["q"], x["k"] = (x[n].repeat_interleave(groups, 1) for n in ("q", "k"))
    x = {n: v[:, None] for n, v in x.items()}
    return recurrence(family, {**x, "initial_state": state.double().cpu()}, scale=xs["q"].shape[-1] ** -0.5)


STEPS = {"kda": "step_kda", "gdn": "step_gated_delta_rule", "gdn2": "step_gdn2", "delta": "step_delta_rule"}


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("family", STEPS)
@pytest.mark.parametrize("v_first", (False, True))
@pytest.mark.parametrize("B,H,groups,K,V,options", [(1, 1, 1, 128, 128, True), (7, 2, 2, 128, 128, True), (6, 3, 1, 64, 100, False), (2, 2, 3, 33, 7, False),
                                                    (40, 4, 1, 128, 128, False)])
def test_delta_steps(dtype, family, v_first, B, H, groups, K, V, options):
    rn, HV = _gen(13), H * groups
    unit = (lambda x: x) if options else (lambda x: torch.nn.functional.normalize(x, dim=-1))
    xs = dict(q=unit(rn(B, H, K)).to(dtype), k=unit(rn(B, H, K)).to(dtype), v=rn(B, HV, V).to(dtype))
    kw = dict(use_qk_l2norm_in_kernel=True) if options else {}
    if family == "gdn":
        xs["g"] = -rn(B, HV).abs()
    elif family == "kda" and options:
        xs.update(g=rn(B, HV, K).to(dtype), A_log=rn(HV), dt_bias=rn(HV, K))
        kw["use_gate_in_kernel"] = True
    elif family != "delta":
        xs["g"] = -0.2 * rn(B, HV, K).abs()
    if family == "gdn2":
        xs.update(b=torch.sigmoid(rn(B, HV, K)).to(dtype), w=torch.sigmoid(rn(B, HV, V)).to(dtype))
        sigmoid = False
    else:
        sigmoid = options and family != "delta"
        xs["beta"] = (rn(B, HV) if sigmoid else torch.sigmoid(rn(B, HV))).to(dtype)
        if sigmoid:
            kw["use_beta_sigmoid_in_kernel"] = True
    slots, at, live = _slots(B, B + 2, torch.int32)
    state = 0.3 * rn(B + 2, HV, K, V)
    mine = state.transpose(-1, -2).contiguous() if v_first else state.clone()
    o = getattr(rewy_b200, STEPS[family])(**xs, state=mine, slots=slots, state_v_first=v_first, **kw)
    if options and not sigmoid:
        xs = {n: (torch.logit(x.double()) if n == "beta" else x) for n, x in xs.items()}   # the reference takes logits there
    want, new = _delta_reference(family, xs, state[at], groups, options)
    _close(o, want[:, 0].to(DEV) * live[:, None, None], "o")
    mine = mine.transpose(-1, -2) if v_first else mine
    _close(mine[at[live]], new.to(DEV)[live], "state")
    rest = torch.ones(B + 2, dtype=torch.bool, device=DEV)
    rest[at[live]] = False
    assert torch.equal(mine[rest], state[rest])


# ---- runs of them together -------------------------------------------------------------------------------------------

def test_a_state_space_layer_answers_token_by_token_what_it_gives_for_the_prompt():
    """conv, scan, gated norm, residual norm over 40 tokens at once, and the last 8 of them one by one from the states in between."""
    rn, B, T, M, N, cut = _gen(14), 3, 40, 64, 16, 32
    x, z, dt, Bm, C = rn(B, T, M), rn(B, T, M), rn(B, T, M), rn(B, T, N), rn(B, T, N)
    weight, A, D, bias, norm = rn(M, 4) / 2, -rn(M, N).abs(), rn(M), rn(M) - 2, 1 + 0.1 * rn(M)
    residual = rn(B, T, M)

    def prompt(sl, conv0=None, scan0=None):
        u, conv1 = rewy_b200.causal_conv(x[:, sl], weight, activation="silu", initial_state=conv0, output_final_state=True)
        y, scan1 = rewy_b200.selective_scan(u, dt[:, sl], A, Bm[:, sl], C[:, sl], D, dt_bias=bias, dt_softplus=True, initial_state=scan0, output_final_state=True)
        y = rewy_b200.gated_rms_norm(y, z[:, sl], norm)
        return rewy_b200.residual_rms_norm(y, residual[:, sl], norm, scale=0.5), conv1, scan1

    (want, want_r), conv, scan = prompt(slice(0, T))
    _, conv_state, scan_state = prompt(slice(0, cut))
    for t in range(cut, T):
        u = rewy_b200.causal_conv_step(x[:, t], conv_state, weight, activation="silu")
        y = rewy_b200.selective_scan_step(u, dt[:, t], A, Bm[:, t], C[:, t], scan_state, D, dt_bias=bias, dt_softplus=True)
        y = rewy_b200.gated_rms_norm(y, z[:, t], norm)
        y, r = rewy_b200.residual_rms_norm(y, residual[:, t], norm, scale=0.5)
        _close(y, want[:, t], f"token {t}")
        _close(r, want_r[:, t], f"residual of token {t}")
    assert torch.equal(conv_state, conv)
    _close(scan_state, scan, "scan state")


@pytest.mark.parametrize("family,name", [("kda", "chunk_kda"), ("gdn", "chunk_gated_delta_rule"), ("delta", "chunk_delta_rule"), ("gdn2", "chunk_gdn2")])
def test_a_delta_layer_answers_token_by_token_what_it_gives_for_the_prompt(family, name):
    """The short convolution of q, k and v, the chunked operator, the gated norm; then the last tokens by steps.  The chunked
    operator's products take BF16 operands: its outputs are held to 8e-3 of the norm elsewhere, and so are the steps to them."""
    rn, B, T, H, cut = _gen(15), 2, 80, 2, 72
    bf = lambda *s: rn(*s).to(BF16)  # noqa: E731
    x, weight, norm, gate = bf(B, T, 3 * H * 128), rn(3 * H * 128, 4) / 2, 1 + 0.1 * rn(128), bf(B, T, H, 128)
    extra = {}
    if family in ("kda", "gdn2"):
        extra["g"] = -0.1 * rn(B, T, H, 128).abs()
    if family == "gdn":
        extra["g"] = -0.3 * rn(B, T, H).abs()
    if family == "gdn2":
        extra.update(b=torch.sigmoid(rn(B, T, H, 128)).to(BF16), w=torch.sigmoid(rn(B, T, H, 128)).to(BF16))
    else:
        extra["beta"] = torch.sigmoid(rn(B, T, H)).to(BF16)
    heads = lambda y: y.unflatten(-1, (3, H, 128)).unbind(-3)  # noqa: E731

    def prompt(sl):
        y, conv = rewy_b200.causal_conv(x[:, sl], weight, activation="silu", output_final_state=True)
        q, k, v = (t.contiguous() for t in heads(y))
        with rewy_b200.use_backend("optimized"):
            o, state = getattr(rewy_b200, name)(q, k, v, **{n: e[:, sl].contiguous() for n, e in extra.items()}, use_qk_l2norm_in_kernel=True,
                                                output_final_state=True)
        return rewy_b200.gated_rms_norm(o, gate[:, sl], norm), conv, state

    want, conv, state = prompt(slice(0, T))
    _, conv_state, delta_state = prompt(slice(0, cut))
    delta_state = delta_state.contiguous()
    for t in range(cut, T):
        q, k, v = heads(rewy_b200.causal_conv_step(x[:, t], conv_state, weight, activation="silu"))
        o = getattr(rewy_b200, STEPS[family])(q, k, v, **{n: e[:, t] for n, e in extra.items()}, state=delta_state, use_qk_l2norm_in_kernel=True)
        y = rewy_b200.gated_rms_norm(o, gate[:, t], norm)
        off = (y.double() - want[:, t].double()).norm() / want[:, t].double().norm()
        assert off <= 1.6e-2, (t, off.item())       # both sides round q, k, v, o to BF16: twice 8e-3
    assert torch.equal(conv_state, conv)
    assert (delta_state - state).norm() <= 8e-3 * state.norm()


# ---- gradients, streams, graphs --------------------------------------------------------------------------------------

def _calls(rn, dtype=FP32):
    """Each trainable operator on small leaves: name -> (function, leaves)."""
    conv = dict(x=rn(1, 20, 16).to(dtype), weight=rn(16, 4), bias=rn(16), initial_state=rn(1, 3, 16).to(dtype))
    scan = _scan_inputs(rn, 1, 500, 24, 16, 1, dtype, 1, ALL)
    gated = dict(x=rn(9, 40).to(dtype), gate=rn(9, 40).to(dtype), weight=rn(40))
    residual = dict(x=rn(9, 40).to(dtype), residual=rn(9, 40).to(dtype), weight=rn(40), scale=rn(40))
    return {"causal_conv": (lambda **x: rewy_b200.causal_conv(**x, activation="silu", output_final_state=True), conv),
            "selective_scan": (lambda **x: rewy_b200.selective_scan(**x, dt_softplus=True, output_final_state=True), scan),
            "gated_rms_norm": (lambda **x: (rewy_b200.gated_rms_norm(**x),), gated),
            "residual_rms_norm": (lambda **x: rewy_b200.residual_rms_norm(**x), residual)}


NAMES = ("causal_conv", "selective_scan", "gated_rms_norm", "residual_rms_norm")


@pytest.mark.parametrize("name", NAMES)
def test_gradients_against_differences(name):
    """Central differences of the FP64 definition along a random direction, step 1e-6: their own error is about 1e-9 of the value,
    the FP32 gradients' along a direction 2e-5 of its norm."""
    call, xs = _calls(_gen(16))[name]
    mine = _leaves(xs)
    out = call(**mine)
    rn = _gen(17)
    seeds = [rn(*o.shape) for o in out]
    grads = torch.autograd.grad(out, list(mine.values()), seeds)
    definition = {"causal_conv": lambda **x: oracle.causal_conv(**x, activation="silu"), "selective_scan": lambda **x: oracle.selective_scan(**x, dt_softplus=True),
                  "gated_rms_norm": lambda **x: (oracle.gated_rms_norm(**x),), "residual_rms_norm": oracle.residual_rms_norm}[name]
    value = lambda x: sum((o * s.double()).sum() for o, s in zip(definition(**x), seeds)).item()  # noqa: E731
    for (n, x), g in zip(xs.items(), grads):
        direction = rn(*x.shape).double()
        base = {k: v.double() for k, v in xs.items()}
        up, down = ({**base, n: base[n] + s * 1e-6 * direction} for s in (1, -1))
        slope = (value(up) - value(down)) / 2e-6
        assert abs(slope - (g.double() * direction).sum().item()) <= 4e-5 * (g.double().norm() * direction.norm()).item() + 1e-6, n


@pytest.mark.parametrize("name", NAMES)
def test_only_some_gradients_are_wanted(name):
    """One leaf at a time, an output whose gradient never comes, an expanded gradient: the same values as all together."""
    call, xs = _calls(_gen(18))[name]
    everything = _leaves(xs)
    out = call(**everything)
    want = dict(zip(xs, torch.autograd.grad(out[0].sum(), list(everything.values()), allow_unused=True)))
    for n in xs:
        mine = {k: v.detach().clone().requires_grad_(k == n) for k, v in xs.items()}
        got, = torch.autograd.grad(call(**mine)[0].sum(), [mine[n]])
        assert torch.equal(got, want[n]), n
    last = call(**everything)[-1]
    for g in torch.autograd.grad(last.sum(), list(everything.values()), allow_unused=True):
        assert g is None or torch.isfinite(g).all()


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_raise(name):
    call, xs = _calls(_gen(19))[name]
    mine = _leaves(xs)
    grads = torch.autograd.grad(call(**mine)[0].sum(), list(mine.values()), create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(sum(g.sum() for g in grads), list(mine.values()), allow_unused=True)


@pytest.mark.parametrize("name", NAMES)
def test_saved_inputs_changed_in_place_are_noticed(name):
    call, xs = _calls(_gen(20))[name]
    mine = _leaves(xs)
    out = call(**mine)
    with torch.no_grad():
        next(iter(mine.values())).add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out[0].sum(), list(mine.values()), allow_unused=True)


@pytest.mark.parametrize("name", NAMES)
def test_another_stream_gives_the_same(name):
    call, xs = _calls(_gen(21), BF16)[name]

    def step():
        mine = _leaves(xs)
        out = call(**mine)
        return (*out, *torch.autograd.grad(out[0].float().sum(), list(mine.values()), allow_unused=True))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert a is b is None or torch.equal(a, b)


@pytest.mark.parametrize("name", NAMES)
def test_a_captured_training_step_replays_on_new_values(name):
    """Forward and backward in one graph, replayed after the inputs have changed; two graphs of one call share nothing."""
    call, xs = _calls(_gen(22), BF16)[name]
    mine = _leaves(xs)

    def step():
        out = call(**mine)
        return [*out, *torch.autograd.grad(out[0], list(mine.values()), torch.ones_like(out[0]), allow_unused=True)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    other = _calls(_gen(23), BF16)[name][1]
    with torch.no_grad():
        for n, v in mine.items():
            v.copy_(other[n])
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = step()
    for _, out in graphs:
        for a, b in zip(out, want):
            assert a is b is None or torch.equal(a, b)


def test_captured_steps_replay():
    """The single-token form of a layer in a graph: replays advance the states as eager calls do."""
    rn, B, M = _gen(24), 5, 256
    x, weight, A = rn(B, M).to(BF16), rn(M, 4), -rn(M, 16).abs()
    dt, Bm, C = 0.1 * rn(B, M).abs().to(BF16), rn(B, 16).to(BF16), rn(B, 16).to(BF16)
    q, v, g, beta = rn(B, 2, 128).to(BF16), rn(B, 2, 128).to(BF16), -rn(B, 2).abs(), torch.sigmoid(rn(B, 2))
    slots = torch.tensor([4, 0, -1, 2, 3], device=DEV, dtype=torch.int32)
    states = [rn(6, 3, M).to(BF16), rn(6, M, 16), rn(6, 2, 128, 128)]

    def step(s):
        u = rewy_b200.causal_conv_step(x, s[0], weight, activation="silu", slots=slots)
        y = rewy_b200.selective_scan_step(u, dt, A, Bm, C, s[1], slots=slots)
        return y, rewy_b200.step_gated_delta_rule(q, q, v, g, beta, s[2], slots=slots, use_qk_l2norm_in_kernel=True)

    eager, held = [s.clone() for s in states], [s.clone() for s in states]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([s.clone() for s in states])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for _ in range(3):
        graph.replay()
        want = step(eager)
    torch.cuda.synchronize()
    for a, b in zip([*out, *held], [*want, *eager]):
        assert torch.equal(a, b)


def test_steps_refuse_gradients_and_count_as_writes():
    rn = _gen(25)
    x, state, weight = rn(2, 16), rn(2, 3, 16), rn(16, 4).requires_grad_()
    with pytest.raises(RuntimeError, match="a step has no gradient"):
        rewy_b200.causal_conv_step(x, state, weight)
    version = state._version
    with torch.no_grad():
        rewy_b200.causal_conv_step(x, state, weight)
    assert state._version > version


# ---- long tensors and the kernels behind the calls -------------------------------------------------------------------

def test_offsets_beyond_32_bits():
    """More than 2^31 elements in a tensor: its last rows give what they give alone."""
    gen = torch.Generator(device=DEV).manual_seed(26)
    rn = lambda *s, t=BF16: torch.empty(*s, device=DEV, dtype=t).normal_(generator=gen)  # noqa: E731
    D, tail = 4096, 9
    rows = (1 << 31) // D + 100
    x, weight = rn(1, rows, D), rn(D, 4, t=FP32) / 2
    y, fin = rewy_b200.causal_conv(x, weight, activation="silu", output_final_state=True)
    alone, _ = rewy_b200.causal_conv(x[:, -tail:], weight, activation="silu", initial_state=x[:, -tail - 3:-tail].contiguous())
    assert torch.equal(y[:, -tail:], alone) and torch.equal(fin, x[:, -3:])
    del y
    norm = rn(D, t=FP32)
    whole = rewy_b200.gated_rms_norm(x, x, norm)
    assert torch.equal(whole[:, -tail:], rewy_b200.gated_rms_norm(x[:, -tail:], x[:, -tail:], norm))
    del whole
    y, r = rewy_b200.residual_rms_norm(x, x, norm, scale=0.5)
    for a, b in zip((y, r), rewy_b200.residual_rms_norm(x[:, -tail:], x[:, -tail:], norm, scale=0.5)):
        assert torch.equal(a[:, -tail:], b)
    del y, r
    M = 256                                                    # the scan: as many tokens as make 2^31 elements of u
    u = x.view(1, -1, M)
    A, Bm = -torch.rand(M, 16, device=DEV) - 0.5, rn(1, u.shape[1], 16)
    y, _ = rewy_b200.selective_scan(u, u, A, Bm, Bm, dt_softplus=True)
    short, _ = rewy_b200.selective_scan(u[:, -2000:], u[:, -2000:], A, Bm[:, -2000:], Bm[:, -2000:], dt_softplus=True)
    _close(y[:, -1000:], short[:, -1000:].float(), "scan")     # 1000 tokens of steps around 0.7 forget where they began
    del x, u, y
    pool, one = (1 << 31) // (M * 16) + 3, torch.tensor([-1], device=DEV, dtype=torch.int32)
    state = torch.zeros(pool, M, 16, device=DEV)
    state[-1] = 1.0
    v, b = rn(1, M), rn(1, 16)
    first, last = (rewy_b200.selective_scan_step(v, v.abs(), A, b, b, s, slots=one + i) for s, i in ((state, pool), (state[-1:].clone(), 1)))
    assert torch.equal(first, last) and not torch.equal(state[-1], torch.ones_like(state[-1])) and not state[0].any()


def test_kernels_are_launched_and_calls_counted():
    from rewy_b200 import _capi
    rn = _gen(27)
    rewy_b200.stats(reset=True)
    before = _capi.launch_count()
    x, w = rn(4, 64), rn(64)
    rewy_b200.gated_rms_norm(x, x, w)
    rewy_b200.residual_rms_norm(x, None, w)
    rewy_b200.causal_conv(x[None], rn(64, 4))
    assert _capi.launch_count() == before + 3
    assert rewy_b200.stats(reset=True) == {f"{n}.optimized_forward": 1 for n in ("causal_conv", "gated_rms_norm", "residual_rms_norm")}
