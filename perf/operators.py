"""What stands around a recurrence in a layer, as measurable cases: the short causal convolution in front of it, the
selective state space scan beside the delta rules, the norms before and after a block with its gate and residual scale, and
the single-token step of the delta rules with which a model answers.

  conv           ``causal_conv`` over a prompt or a training batch (forward and backward)
  conv_step      ``causal_conv_step``, one token for every sequence of a decoding batch, state updated in place
  scan           ``selective_scan`` over a prompt or a training batch (forward and backward)
  scan_step      ``selective_scan_step``
  gated_norm     ``gated_rms_norm``: the norm behind a recurrence with the layer's gate
  residual_norm  ``residual_rms_norm``: the residual sum with the block's scale, and the norm in front of the next block
  delta_step     ``step_kda``, ``step_gated_delta_rule``, ``step_gdn2``, ``step_delta_rule``

Where ``own`` is false the operators are computed in their plain form, elementary tensor operations in 32 bits.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
K = 128  # key and value channels of a delta rule's head


def listed():
    cases = {
        # the q, k, v convolution of a layer in training: 16 q/k heads and 32 value heads of 128 channels
        "conv_train": dict(op="conv", B=2, T=4096, M=8192, W=4, type="bf16", train=True, bias=False, act=True, sequences=0, state=False),
        # documents of arbitrary lengths behind one another, each from its own state to its own state
        "conv_prefill_packed": dict(op="conv", B=1, T=16001, M=2048, W=4, type="bf16", train=False, bias=True, act=True, sequences=12, state=True),
        # one token for each of 64 sequences, states in a pool of 96
        "conv_step": dict(op="conv_step", B=64, M=8192, W=4, type="bf16", bias=True, act=True, pool=96),
        # a state space layer's training step with everything fused into the scan
        "scan_train": dict(op="scan", B=2, T=4096, M=4096, N=16, G=1, type="bf16", train=True, gate=True, skip=True, softplus=True, sequences=0, state=False),
        # a narrow layer on one odd length in 32 bits, states in and out: a test, a tiny model, a small shard
        "scan_train_narrow": dict(op="scan", B=1, T=2000, M=1024, N=16, G=2, type="fp32", train=True, gate=False, skip=True, softplus=False, sequences=0, state=True),
        # packed prompts, each continued from its own state
        "scan_prefill_packed": dict(op="scan", B=1, T=16001, M=2048, N=16, G=1, type="bf16", train=False, gate=True, skip=True, softplus=True, sequences=12, state=True),
        # one token for each of 64 sequences
        "scan_step": dict(op="scan_step", B=64, M=4096, N=16, G=1, type="bf16", gate=True, skip=True, softplus=True, pool=96),
        # the norm behind a gated delta rule: rows of one head, the gate from the layer's own projection
        "gated_norm_train": dict(op="gated_norm", rows=131072, M=128, type="bf16", train=True, act="silu", gate_first=False),
        # residual sum with a scale per channel and the next block's norm, in training
        "residual_norm_train": dict(op="residual_norm", rows=8192, M=4096, type="bf16", train=True, scale="channel"),
        # the same for a few decoding sequences
        "residual_norm_decode": dict(op="residual_norm", rows=16, M=2048, type="bf16", train=False, scale="number"),
        # decoding with KDA, gate, normalisation and sigmoid fused: 64 sequences of 32 heads
        "delta_step_kda": dict(op="delta_step", family="kda", B=64, H=32, groups=1, type="bf16", options=True, pool=64),
        # one conversation, two value heads to each key head: latency counts
        "delta_step_gdn": dict(op="delta_step", family="gdn", B=1, H=8, groups=2, type="bf16", options=True, pool=1),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _spread(rng, lo, hi):
    """Whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("conv", "scan", "conv", "scan", "gated_norm", "residual_norm", "conv_step", "scan_step", "delta_step"))
    kind = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32"))
    yes = lambda p=0.5: rng.random() < p  # noqa: E731
    if op in ("conv", "scan"):
        M, T, B, train = 8 * _spread(rng, 8, 512), _spread(rng, 1, 16384), _spread(rng, 1, 16), yes()
        if yes(0.2):
            M -= rng.randint(1, 7)
        most = 1 << 24
        while B * T * M > most:
            B, T = (B // 2, T) if B > 1 else (1, max(1, T // 2))
        packed = rng.randint(2, min(9, T)) if yes(0.4) and T >= 2 else 0
        c = dict(op=op, B=1 if packed else B, T=T, M=M, type=kind, train=train, sequences=packed, state=yes())
        if op == "conv":
            return dict(c, W=rng.choice((2, 3, 4, 4)), bias=yes(), act=yes(0.8))
        G = rng.choice((1, 1, 2))
        return dict(c, M=M + M % G, N=rng.choice((4, 8, 16, 16, 16, 32)), G=G, gate=yes(), skip=yes(0.8), softplus=yes(0.7))
    if op == "conv_step":
        B = _spread(rng, 1, 128)
        return dict(op=op, B=B, M=_spread(rng, 64, 8192), W=rng.choice((2, 3, 4)), type=kind, bias=yes(), act=yes(0.8), pool=B + rng.randint(0, 40))
    if op == "scan_step":
        B = _spread(rng, 1, 128)
        return dict(op=op, B=B, M=2 * _spread(rng, 32, 2048), N=rng.choice((8, 16, 16, 32)), G=rng.choice((1, 2)), type=kind, gate=yes(), skip=yes(0.8),
                    softplus=yes(0.7), pool=B + rng.randint(0, 40))
    if op == "delta_step":
        B = _spread(rng, 1, 64)
        return dict(op=op, family=rng.choice(("kda", "gdn", "gdn2", "delta")), B=B, H=_spread(rng, 1, 16), groups=rng.choice((1, 1, 2)), type=kind,
                    options=yes(), pool=B + rng.randint(0, 20))
    if op == "gated_norm":
        M = rng.choice((64, 128, 128, 256, 1000, 2048, 4096))
        return dict(op=op, rows=_spread(rng, 1, max(2, (1 << 23) // M)), M=M, type=kind, train=yes(), act=rng.choice(("silu", "silu", "sigmoid")), gate_first=yes(0.3))
    M = _spread(rng, 64, 8192)
    return dict(op=op, rows=_spread(rng, 1, max(2, (1 << 23) // M)), M=M, type=kind, train=yes(), scale=rng.choice(("none", "number", "channel")))


class _Make:
    """Tensors from one seed."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.host = torch.Generator()
        self.host.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device="cuda")

    def slots(self, B, pool):
        return torch.randperm(pool, generator=self.host)[:B].to(device="cuda", dtype=torch.int32)

    def steps(self, *shape):
        """What softplus makes a time step between 0.001 and 0.1 of."""
        step = torch.exp(self.uniform(*shape) * math.log(100.0) + math.log(0.001))
        return step + torch.log(-torch.expm1(-step))

    def offsets(self, T, sequences):
        """Offsets of documents of uneven lengths, one token at least each."""
        cut = torch.randperm(T - 1, generator=self.host)[:sequences - 1].sort().values + 1
        return torch.cat([torch.zeros(1, dtype=torch.int64), cut, torch.tensor([T])])


def _sequences(case):
    return case["sequences"] or case["B"]


def prepare(case, seed):
    """Inputs as the layers hand them over.  Names are those of the operators' arguments; ``wrt`` lists what a training
    step wants gradients of, ``out_grads`` the gradients that come from behind."""
    m, op, t = _Make(seed), case["op"], TYPES[case["type"]]
    x, s = {}, {"case": case}
    if op in ("conv", "conv_step"):
        M, W = case["M"], case["W"]
        x["weight"] = (2 * m.uniform(M, W) - 1) / math.sqrt(W)
        x["bias"] = (2 * m.uniform(M) - 1) / math.sqrt(W) if case["bias"] else None
    if op in ("scan", "scan_step"):
        M, N, G = case["M"], case["N"], case["G"]
        x["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * (0.8 + 0.4 * m.uniform(M, N))
        x["D"] = 1 + 0.1 * m.normal(M) if case["skip"] else None
        x["dt_bias"] = m.steps(M) if case["softplus"] else None
    if op == "conv":
        B, T = case["B"], case["T"]
        x["x"] = m.normal(B, T, M).to(t)
        x["initial_state"] = m.normal(_sequences(case), W - 1, M).to(t) if case["state"] else None
        out = [m.normal(B, T, M).to(t)] + ([m.normal(_sequences(case), W - 1, M).to(t)] if case["state"] else [])
    elif op == "scan":
        B, T = case["B"], case["T"]
        x["u"] = m.normal(B, T, M).to(t)
        x["dt"] = (0.5 * m.normal(B, T, M) if case["softplus"] else torch.exp(m.uniform(B, T, M) * math.log(100.0) + math.log(0.001))).to(t)
        x["B"], x["C"] = m.normal(B, T, G, N).to(t), m.normal(B, T, G, N).to(t)
        x["z"] = m.normal(B, T, M).to(t) if case["gate"] else None
        x["initial_state"] = 0.3 * m.normal(_sequences(case), M, N) if case["state"] else None
        out = [m.normal(B, T, M).to(t)] + ([0.3 * m.normal(_sequences(case), M, N)] if case["state"] else [])
    elif op == "conv_step":
        x["x"], x["state"], x["slots"] = m.normal(case["B"], M).to(t), m.normal(case["pool"], W - 1, M).to(t), m.slots(case["B"], case["pool"])
    elif op == "scan_step":
        B = case["B"]
        x["u"] = m.normal(B, M).to(t)
        x["dt"] = (0.5 * m.normal(B, M) if case["softplus"] else torch.exp(m.uniform(B, M) * math.log(100.0) + math.log(0.001))).to(t)
        x["B"], x["C"] = m.normal(B, G, N).to(t), m.normal(B, G, N).to(t)
        x["z"] = m.normal(B, M).to(t) if case["gate"] else None
        x["state"], x["slots"] = 0.3 * m.normal(case["pool"], M, N), m.slots(B, case["pool"])
    elif op == "gated_norm":
        R, M = case["rows"], case["M"]
        x["x"], x["gate"], x["weight"] = m.normal(R, M).to(t), m.normal(R, M).to(t), 1 + 0.1 * m.normal(M)
        out = [m.normal(R, M).to(t)]
    elif op == "residual_norm":
        R, M = case["rows"], case["M"]
        x["x"], x["residual"], x["weight"] = m.normal(R, M).to(t), (3 * m.normal(R, M)).to(t), 1 + 0.1 * m.normal(M)
        x["scale"] = {"none": None, "number": 0.7, "channel": 0.5 + 0.1 * m.normal(M)}[case["scale"]]
        out = [m.normal(R, M).to(t), m.normal(R, M).to(t)]
    else:
        B, H, f = case["B"], case["H"], case["family"]
        HV = H * case["groups"]
        unit = (lambda v: v) if case["options"] else (lambda v: torch.nn.functional.normalize(v, dim=-1))
        x["q"], x["k"], x["v"] = unit(m.normal(B, H, K)).to(t), unit(m.normal(B, H, K)).to(t), m.normal(B, HV, K).to(t)
        if f == "gdn":
            x["g"] = -torch.exp(m.uniform(HV)) * torch.nn.functional.softplus(m.normal(B, HV))
        elif f == "kda" and case["options"]:
            x["g"], x["A_log"], x["dt_bias"] = (0.5 * m.normal(B, HV, K)).to(t), torch.log(1 + 15 * m.uniform(HV)), m.steps(HV * K)
        elif f != "delta":
            x["g"] = -0.1 * torch.nn.functional.softplus(m.normal(B, HV, K))
        if f == "gdn2":
            x["b"], x["w"] = torch.sigmoid(m.normal(B, HV, K)).to(t), torch.sigmoid(m.normal(B, HV, K)).to(t)
        else:
            logits = m.normal(B, HV)
            x["beta"] = (logits if case["options"] and f != "delta" else torch.sigmoid(logits)).to(t)
        x["state"], x["slots"] = 0.1 * m.normal(case["pool"], HV, K, K), m.slots(B, case["pool"])
    if case.get("train"):
        s["wrt"] = [n for n, v in x.items() if isinstance(v, torch.Tensor)]
        s["out_grads"] = out
        for n in s["wrt"]:
            x[n].requires_grad_()
    if case.get("sequences"):
        s["cu"] = m.offsets(case["T"], case["sequences"])
        s["cu_device"] = s["cu"].to(device="cuda", dtype=torch.int32)
    s["x"] = x
    return s


# ---------------------------------------------------------------------------------------------------------------------
# what a user's program calls


def _own(s):
    import rewy_b200
    case, x = s["case"], s["x"]
    op = case["op"]
    kw = {}
    if case.get("sequences"):
        kw = dict(cu_seqlens=s["cu_device"], cu_seqlens_cpu=s["cu"])
    if op == "conv":
        out = rewy_b200.causal_conv(x["x"], x["weight"], x["bias"], activation="silu" if case["act"] else None,
                                    initial_state=x["initial_state"], output_final_state=case["state"], **kw)
    elif op == "scan":
        out = rewy_b200.selective_scan(x["u"], x["dt"], x["A"], x["B"], x["C"], x["D"], z=x["z"], dt_bias=x["dt_bias"],
                                       dt_softplus=case["softplus"], initial_state=x["initial_state"],
                                       output_final_state=case["state"], **kw)
    elif op == "conv_step":
        y = rewy_b200.causal_conv_step(x["x"], x["state"], x["weight"], x["bias"], activation="silu" if case["act"] else None, slots=x["slots"])
        return y, x["state"]
    elif op == "scan_step":
        y = rewy_b200.selective_scan_step(x["u"], x["dt"], x["A"], x["B"], x["C"], x["state"], x["D"], z=x["z"], dt_bias=x["dt_bias"],
                                          dt_softplus=case["softplus"], slots=x["slots"])
        return y, x["state"]
    elif op == "gated_norm":
        out = (rewy_b200.gated_rms_norm(x["x"], x["gate"], x["weight"], activation=case["act"], gate_first=case["gate_first"]),)
    elif op == "residual_norm":
        out = rewy_b200.residual_rms_norm(x["x"], x["residual"], x["weight"], scale=x["scale"])
    else:
        step = {"kda": rewy_b200.step_kda, "gdn": rewy_b200.step_gated_delta_rule, "gdn2": rewy_b200.step_gdn2, "delta": rewy_b200.step_delta_rule}
        if case["options"]:
            kw["use_qk_l2norm_in_kernel"] = True
            if case["family"] in ("kda", "gdn"):
                kw["use_beta_sigmoid_in_kernel"] = True
            if case["family"] == "kda":
                kw["use_gate_in_kernel"] = True
        return step[case["family"]](**x, **kw), x["state"]
    out = tuple(o for o in out if o is not None)
    if not case["train"]:
        return out
    return out, torch.autograd.grad(out, [x[n] for n in s["wrt"]], s["out_grads"])


# ---------------------------------------------------------------------------------------------------------------------
# plain forms


def _places(case, cu, device):
    """(offsets, sequence of each token, place of each token in its sequence) of the flat token axis."""
    if cu is None:
        cu = torch.arange(case["B"] + 1) * case["T"]
    cu = cu.to(device)
    sequence = torch.repeat_interleave(torch.arange(cu.numel() - 1, device=device), cu[1:] - cu[:-1])
    return cu, sequence, torch.arange(sequence.numel(), device=device) - cu[sequence]


def _act(name, v):
    return v * torch.sigmoid(v) if name == "silu" else torch.sigmoid(v)


def _plain_conv(case, x, cu):
    W, M = case["W"], case["M"]
    cu, sequence, place = _places(case, cu, x["x"].device)
    S = cu.numel() - 1
    state = x["initial_state"] if x["initial_state"] is not None else x["x"].new_zeros(S, W - 1, M)
    rows = torch.cat([x["x"].reshape(-1, M), state.reshape(-1, M)])
    at = lambda seq, p: torch.where(p >= 0, cu[seq] + p, sequence.numel() + seq * (W - 1) + W - 1 + p)  # noqa: E731
    y = sum(x["weight"][:, W - 1 - o] * rows[at(sequence, place - o)] for o in range(W))
    if x["bias"] is not None:
        y = y + x["bias"]
    if case["act"]:
        y = _act("silu", y)
    seq = torch.arange(S, device=cu.device)[:, None]
    last = (cu[1:] - cu[:-1])[:, None] - (W - 1) + torch.arange(W - 1, device=cu.device)
    return (y.view(x["x"].shape),) + ((rows[at(seq, last)],) if case["state"] else ())


def _running(a, b):
    """h_t = a_t h_(t-1) + b_t along the first axis from h = 0, by doubling."""
    a, b, o = a.clone(), b.clone(), 1
    while o < a.shape[0]:
        b = torch.cat([b[:o], b[o:] + a[o:] * b[:-o]])
        a = torch.cat([a[:o], a[o:] * a[:-o]])
        o *= 2
    return b


def _grouped(v, M):
    """[T, G, N] -> [T, M, N]"""
    return v.repeat_interleave(M // v.shape[1], 1)


def _plain_scan(case, x, cu, grads, types):
    """Forward and, with the outputs' gradients, the backward by the adjoint recurrence."""
    B, T, M, N, G = case["B"], case["T"], case["M"], case["N"], case["G"]
    cu, sequence, place = _places(case, cu, x["u"].device)
    flat = {n: x[n].reshape(B * T, *x[n].shape[2:]) for n in ("u", "dt", "B", "C", "z") if x[n] is not None}
    raw = flat["dt"] + (x["dt_bias"] if x["dt_bias"] is not None else 0)
    dt = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs())) if case["softplus"] else raw
    Bm, Cm = _grouped(flat["B"], M), _grouped(flat["C"], M)
    decay = torch.exp(dt[..., None] * x["A"])
    first = (place == 0)[:, None, None]
    gain = (dt * flat["u"])[..., None] * Bm
    if x["initial_state"] is not None:
        gain[cu[:-1]] += decay[cu[:-1]] * x["initial_state"]
    h = _running(torch.where(first, 0, decay), gain)
    y = (h * Cm).sum(-1)
    if x["D"] is not None:
        y = y + x["D"] * flat["u"]
    z = flat.get("z")
    out = (y if z is None else y * _act("silu", z)).view(x["u"].shape)
    out = (out, h[cu[1:] - 1]) if case["state"] else (out,)
    if grads is None:
        return out
    d, dy = {}, grads[0].reshape(B * T, M)
    if z is not None:
        sig = torch.sigmoid(z)
        d["z"] = (dy * y * sig * (1 + z * (1 - sig))).view(x["z"].shape)
        dy = dy * z * sig
    back = dy[..., None] * Cm
    if case["state"]:
        back[cu[1:] - 1] += grads[1]
    after = torch.cat([torch.where(first, 0, decay)[1:], torch.zeros_like(decay[:1])])
    gh = _running(after.flip(0), back.flip(0)).flip(0)
    del back, after
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[cu[:-1]] = x["initial_state"] if x["initial_state"] is not None else 0
    through = gh * before * decay
    if x["initial_state"] is not None:
        d["initial_state"] = (gh * decay)[cu[:-1]]
    drive = (gh * Bm).sum(-1)
    ddt = (through * x["A"]).sum(-1) + drive * flat["u"]
    d["A"] = (through * dt[..., None]).sum(0)
    del through, before
    d["u"] = drive * dt + (x["D"] * dy if x["D"] is not None else 0)
    shared = lambda v: v.view(B, T, G, M // G, N).sum(3)  # noqa: E731
    d["C"], d["B"] = shared(dy[..., None] * h), shared(gh * (dt * flat["u"])[..., None])
    if x["D"] is not None:
        d["D"] = (dy * flat["u"]).sum(0)
    if case["softplus"]:
        ddt = ddt * torch.sigmoid(raw)
        d["dt_bias"] = ddt.sum(0)
    d["dt"] = ddt
    return out, [d[n].view(x[n].shape) for n in types]


def _rms(v, eps=1e-6):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)


def _plain_gated_norm(case, x):
    gate = _act(case["act"], x["gate"])
    return ((_rms(x["x"] * gate) if case["gate_first"] else _rms(x["x"]) * gate) * x["weight"],)


def _plain_residual_norm(case, x):
    r = x["residual"] + (x["x"] if x["scale"] is None else x["scale"] * x["x"])
    return _rms(r) * x["weight"], r


def _plain_delta_step(case, x, state):
    f, G = case["family"], case["groups"]
    q, k = (x[n].repeat_interleave(G, 1) for n in ("q", "k"))
    if case["options"]:
        q, k = (v * torch.rsqrt((v * v).sum(-1, keepdim=True) + 1e-6) for v in (q, k))
    if f != "delta":
        g = x["g"]
        if f == "kda" and case["options"]:
            raw = g + x["dt_bias"].view(1, -1, K)
            g = -torch.exp(x["A_log"])[:, None] * (torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs())))
        state = state * torch.exp(g if f != "gdn" else g[..., None])[..., None]
    if f == "gdn2":
        write = x["w"] * x["v"] - ((x["b"] * k)[..., None] * state).sum(-2)
    else:
        beta = torch.sigmoid(x["beta"]) if case["options"] and f != "delta" else x["beta"]
        write = beta[..., None] * (x["v"] - (k[..., None] * state).sum(-2))
    state = state + k[..., None] * write[..., None, :]
    return (q[..., None] * state).sum(-2) * K ** -0.5, state


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    t = TYPES[case["type"]]
    x = {n: v.detach().float() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for n, v in s["x"].items()}
    if op.endswith("step"):
        at = x["slots"].long()
        old = x["state"][at]
        if op == "conv_step":
            rows = torch.cat([old, x["x"][:, None]], 1)
            y = (rows * x["weight"].t()).sum(1) + (x["bias"] if x["bias"] is not None else 0)
            y, new = _act("silu", y) if case["act"] else y, rows[:, 1:]
        elif op == "scan_step":
            one = dict(case, T=1, state=True, sequences=0)
            v = {n: (x[n][:, None] if x[n] is not None else None) for n in ("u", "dt", "B", "C", "z")}
            y, new = _plain_scan(one, {**v, "A": x["A"], "D": x["D"], "dt_bias": x["dt_bias"], "initial_state": old}, None, None, None)
            y = y[:, 0]
        else:
            y, new = _plain_delta_step(case, x, old)
        s["x"]["state"][at] = new.to(s["x"]["state"].dtype)
        return y.to(t), s["x"]["state"]
    grads = [g.float() for g in s["out_grads"]] if case["train"] else None
    cu = s.get("cu")
    if op == "scan":
        out = _plain_scan(case, x, cu, grads, s.get("wrt"))
        out, d = out if case["train"] else (out, None)
        kinds = (t, torch.float32)
    else:
        form = {"conv": lambda c, v: _plain_conv(c, v, cu), "gated_norm": _plain_gated_norm, "residual_norm": _plain_residual_norm}[op]
        if case["train"]:
            x = {n: v.requires_grad_() if n in s["wrt"] else v for n, v in x.items()}
        out = form(case, x)
        d = torch.autograd.grad(out, [x[n] for n in s["wrt"]], grads) if case["train"] else None
        kinds = (t, t)
    out = tuple(o.detach().to(k) for o, k in zip(out, kinds))
    return out if d is None else (out, tuple(g.to(s["x"][n].dtype) for g, n in zip(d, s["wrt"])))


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, token by token and sequence by sequence


def _exact_conv(case, x, cu, grads):
    W = case["W"]
    X = x["x"].reshape(-1, case["M"])
    Y, DX, finals, dinit = torch.empty_like(X), torch.zeros_like(X), [], []
    dW = torch.zeros_like(x["weight"])
    db = torch.zeros_like(x["weight"][:, 0])
    for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        L = b - a
        head = x["initial_state"][i] if x["initial_state"] is not None else X.new_zeros(W - 1, case["M"])
        line = torch.cat([head, X[a:b]])
        pre = torch.zeros_like(X[a:b])
        for w in range(W):
            pre += x["weight"][:, w] * line[w:w + L]
        if x["bias"] is not None:
            pre += x["bias"]
        sig = 1 / (1 + torch.exp(-pre))
        Y[a:b] = pre * sig if case["act"] else pre
        if case["state"]:
            finals.append(line[L:])
        if grads is not None:
            g = grads[0].reshape(X.shape)[a:b]
            if case["act"]:
                g = g * (sig + pre * sig * (1 - sig))
            dline = torch.zeros_like(line)
            for w in range(W):
                dline[w:w + L] += x["weight"][:, w] * g
                dW[:, w] += (g * line[w:w + L]).sum(0)
            db += g.sum(0)
            if case["state"]:
                dline[L:] += grads[1][i]
            DX[a:b] = dline[W - 1:]
            dinit.append(dline[:W - 1])
    out = (Y.view(x["x"].shape),) + ((torch.stack(finals),) if case["state"] else ())
    return out, {"x": DX.view(x["x"].shape), "weight": dW, "bias": db, "initial_state": torch.stack(dinit) if dinit else None}


def _exact_scan(case, x, cu, grads):
    """One token after the other, the sequences of a batch side by side."""
    M, N, G, T = case["M"], case["N"], case["G"], case["T"]
    packed = len(cu) - 1 > 1 and case["sequences"]
    spans = [(a, b, 0, i) for i, (a, b) in enumerate(zip(cu[:-1], cu[1:]))] if packed else [(0, T, slice(None), slice(None))]
    wide = lambda v: torch.stack([v[..., m * G // M, :] for m in range(0, M, max(1, M // G))], -2).repeat_interleave(max(1, M // G), -2)  # noqa: E731
    lead = (case["B"],) if not packed else ()
    sq = lambda v, t: v[0, t] if packed else v[:, t]  # noqa: E731
    raw = x["dt"] + (x["dt_bias"] if x["dt_bias"] is not None else 0)
    dt = torch.nn.functional.softplus(raw, threshold=700) if case["softplus"] else raw
    Y = torch.empty_like(x["u"])
    keep = x["u"].new_empty((case["T"],) + lead + (M, N)) if grads is not None else None
    d = {n: torch.zeros_like(v) for n, v in x.items() if isinstance(v, torch.Tensor)} if grads is not None else {}
    finals = []
    sig = 1 / (1 + torch.exp(-x["z"])) if x["z"] is not None else None
    dY = grads[0] * (x["z"] * sig if sig is not None else 1) if grads is not None else None
    for a, b, row, seq in spans:
        start = x["initial_state"][seq] if x["initial_state"] is not None else x["u"].new_zeros(lead + (M, N))
        h = start
        for t in range(a, b):
            h = torch.exp(sq(dt, t)[..., None] * x["A"]) * h + (sq(dt, t) * sq(x["u"], t))[..., None] * wide(sq(x["B"], t))
            y = (h * wide(sq(x["C"], t))).sum(-1)
            if packed:
                Y[0, t] = y
            else:
                Y[:, t] = y
            if keep is not None:
                keep[t] = h
        finals.append(h)
        if grads is None:
            continue
        gh = (grads[1][seq] if case["state"] else torch.zeros_like(h)).clone()
        for t in range(b - 1, a - 1, -1):
            old, now = keep[t - 1] if t > a else start, sq(dt, t)
            gh = gh + sq(dY, t)[..., None] * wide(sq(x["C"], t))
            decay = torch.exp(now[..., None] * x["A"])
            q = gh * old * decay
            drive = (gh * wide(sq(x["B"], t))).sum(-1)
            share = lambda v: v.reshape(lead + (G, M // G, N)).sum(-2)  # noqa: E731
            for n, v in (("dt", (q * x["A"]).sum(-1) + drive * sq(x["u"], t)), ("u", drive * now),
                         ("C", share(sq(dY, t)[..., None] * keep[t])), ("B", share(gh * (now * sq(x["u"], t))[..., None]))):
                if packed:
                    d[n][0, t] = v
                else:
                    d[n][:, t] = v
            q = q * now[..., None]
            d["A"] += q if packed else q.sum(0)
            gh = gh * decay
        if x["initial_state"] is not None:
            d["initial_state"][seq] = gh
    if x["D"] is not None:
        Y += x["D"] * x["u"]
    out = Y * x["z"] * sig if sig is not None else Y
    if grads is not None:
        if sig is not None:
            d["z"] = grads[0] * Y * (sig + x["z"] * sig * (1 - sig))
        if x["D"] is not None:
            d["u"] += x["D"] * dY
            d["D"] = (dY * x["u"]).sum((0, 1))
        if case["softplus"]:
            d["dt"] = d["dt"] / (1 + torch.exp(-raw))
            d["dt_bias"] = d["dt"].sum((0, 1))
    return (out,) + (((torch.stack(finals) if packed else finals[0]),) if case["state"] else ()), d


def _exact_gated_norm(case, x, grads):
    X, g, w = x["x"], x["gate"], x["weight"]
    sig = 1 / (1 + torch.exp(-g))
    s, ds = (g * sig, sig + g * sig * (1 - sig)) if case["act"] == "silu" else (sig, sig * (1 - sig))
    v = X * s if case["gate_first"] else X
    r = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6)
    n = v * r
    y = n * w if case["gate_first"] else n * w * s
    if grads is None:
        return (y,), {}
    dy = grads[0]
    dn = dy * w if case["gate_first"] else dy * w * s
    dv = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    if case["gate_first"]:
        return (y,), {"x": dv * s, "gate": dv * X * ds, "weight": (dy * n).sum(0)}
    return (y,), {"x": dv, "gate": dy * n * w * ds, "weight": (dy * n * s).sum(0)}


def _exact_residual_norm(case, x, grads):
    a = 1.0 if x["scale"] is None else x["scale"]
    r = x["residual"] + a * x["x"]
    inv = 1 / torch.sqrt(r.square().mean(-1, keepdim=True) + 1e-6)
    n = r * inv
    if grads is None:
        return (n * x["weight"], r), {}
    dn = grads[0] * x["weight"]
    dr = grads[1] + inv * (dn - n * (dn * n).mean(-1, keepdim=True))
    return (n * x["weight"], r), {"x": a * dr, "residual": dr, "weight": (grads[0] * n).sum(0), "scale": (dr * x["x"]).sum(0)}


def _exact_step(case, x, op):
    at = x["slots"].long()
    state = x["state"].clone()
    old = state[at]
    if op == "conv_step":
        y = x["x"] * x["weight"][:, -1]
        for w in range(case["W"] - 1):
            y = y + old[:, w] * x["weight"][:, w]
        y = y + x["bias"] if x["bias"] is not None else y
        y = y / (1 + torch.exp(-y)) if case["act"] else y
        new = torch.cat([old[:, 1:], x["x"][:, None]], 1)
    elif op == "scan_step":
        raw = x["dt"] + (x["dt_bias"] if x["dt_bias"] is not None else 0)
        dt = torch.nn.functional.softplus(raw, threshold=700) if case["softplus"] else raw
        per = case["M"] // case["G"]
        new = old * torch.exp(dt[..., None] * x["A"]) + (dt * x["u"])[..., None] * x["B"].repeat_interleave(per, 1)
        y = torch.einsum("bmn,bmn->bm", new, x["C"].repeat_interleave(per, 1))
        y = y + x["D"] * x["u"] if x["D"] is not None else y
        y = y * x["z"] / (1 + torch.exp(-x["z"])) if x["z"] is not None else y
    else:
        f, G = case["family"], case["groups"]
        q, k = x["q"], x["k"]
        if case["options"]:
            q, k = q / torch.sqrt(q.square().sum(-1, keepdim=True) + 1e-6), k / torch.sqrt(k.square().sum(-1, keepdim=True) + 1e-6)
        q, k = q.repeat_interleave(G, 1), k.repeat_interleave(G, 1)
        new = old
        if f == "gdn":
            new = new * torch.exp(x["g"])[..., None, None]
        elif f == "kda" and case["options"]:
            step = torch.nn.functional.softplus(x["g"] + x["dt_bias"].view(-1, K), threshold=700)
            new = new * torch.exp(-torch.exp(x["A_log"])[:, None] * step)[..., None]
        elif f != "delta":
            new = new * torch.exp(x["g"])[..., None]
        if f == "gdn2":
            r = x["w"] * x["v"] - torch.einsum("bhk,bhkv->bhv", x["b"] * k, new)
        else:
            beta = 1 / (1 + torch.exp(-x["beta"])) if case["options"] and f != "delta" else x["beta"]
            r = beta[..., None] * (x["v"] - torch.einsum("bhk,bhkv->bhv", k, new))
        new = new + torch.einsum("bhk,bhv->bhkv", k, r)
        y = torch.einsum("bhk,bhkv->bhv", q, new) / math.sqrt(K)
    state[at] = new
    return y, state


def exact(case, seed):
    s = prepare(case, seed)
    x = {n: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for n, v in s["x"].items()}
    op = case["op"]
    if op.endswith("step"):
        return _exact_step(case, x, op)
    grads = [g.double() for g in s["out_grads"]] if case["train"] else None
    if op in ("conv", "scan"):
        cu = s["cu"].tolist() if case["sequences"] else [i * case["T"] for i in range(case["B"] + 1)]
        out, d = (_exact_conv if op == "conv" else _exact_scan)(case, x, cu, grads)
    else:
        out, d = (_exact_gated_norm if op == "gated_norm" else _exact_residual_norm)(case, x, grads)
    return out if grads is None else (out, tuple(d[n] for n in s["wrt"]))


def work(case):
    """Inputs read once and outputs written once, and the operations of the formulas (an exponential counted as one)."""
    op, e = case["op"], BYTES[case["type"]]
    if op == "conv":
        n, M, W = case["B"] * case["T"] * case["M"], case["M"], case["W"]
        state = _sequences(case) * (W - 1) * M * e if case["state"] else 0
        params = M * (W + case["bias"]) * 4
        act = 4 if case["act"] else 0
        forward = {"bytes": 2 * n * e + 2 * state + params, "flops": n * (2 * W + act)}
        if not case["train"]:
            return forward
        # x and dy read, y, dx and the parameters' gradients written; the pre-activation, dx and dweight summed
        return {"bytes": forward["bytes"] + 2 * n * e + 2 * state + params, "flops": forward["flops"] + n * (6 * W + 2 * act)}
    if op == "scan":
        tokens, M, N, G = case["B"] * case["T"], case["M"], case["N"], case["G"]
        per_channel = tokens * M * e * (2 + case["gate"])
        shared = tokens * 2 * G * N * e
        params = (M * N + M * (case["skip"] + case["softplus"])) * 4
        state = _sequences(case) * M * N * 4 if case["state"] else 0
        inputs = per_channel + shared + params + state
        y = tokens * M * e + state
        forward = tokens * M * (7 * N + 4 + 4 * case["gate"] + 4 * case["softplus"])
        if not case["train"]:
            return {"bytes": inputs + y, "flops": forward}
        return {"bytes": 2 * inputs + 2 * y, "flops": forward + tokens * M * (22 * N + 8 + 8 * case["gate"] + 4 * case["softplus"])}
    if op == "conv_step":
        n, W = case["B"] * case["M"], case["W"]
        return {"bytes": n * e * (2 + 2 * (W - 1)) + case["M"] * (W + case["bias"]) * 4, "flops": n * (2 * W + 4 * case["act"])}
    if op == "scan_step":
        n, M, N = case["B"] * case["M"], case["M"], case["N"]
        return {"bytes": n * (8 * N + e * (3 + case["gate"])) + M * (N + 2) * 4 + case["B"] * 2 * case["G"] * N * e, "flops": n * (7 * N + 12)}
    if op in ("gated_norm", "residual_norm"):
        n, M = case["rows"] * case["M"], case["M"]
        params = M * 4 * (2 if case.get("scale") == "channel" else 1)
        moved = 3 * n * e if op == "gated_norm" else 4 * n * e           # two inputs, one or two outputs
        forward = {"bytes": moved + params, "flops": n * 9}
        if not case["train"]:
            return forward
        # the outputs' gradients read, the inputs' written; what the forward read counts once for both
        return {"bytes": 2 * moved + 2 * params, "flops": n * 30}
    f, HV = case["family"], case["H"] * case["groups"]
    heads = case["B"] * HV
    gates = {"kda": K * (e if case["options"] else 4) + e, "gdn": 4 + e, "gdn2": K * 4 + 2 * K * e, "delta": e}[f]
    return {"bytes": heads * (2 * K * K * 4 + 2 * K * e + gates) + case["B"] * case["H"] * 2 * K * e, "flops": heads * K * K * 7}
