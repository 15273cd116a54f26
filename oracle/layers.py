"""FP64 definitions of the operators around a recurrence, token by token, differentiable by autograd.

Test infrastructure: never imported by the product package.  Inputs are FP64 tensors; ``cu`` is a list of offsets of packed
sequences (batch 1) or None.
"""
import torch


def _spans(x, cu):
    if cu is None:
        return [(slice(b, b + 1), 0, x.shape[1]) for b in range(x.shape[0])]
    return [(slice(0, 1), a, b) for a, b in zip(cu[:-1], cu[1:])]


def act(name, v):
    return v * torch.sigmoid(v) if name == "silu" else torch.sigmoid(v) if name == "sigmoid" else v


def causal_conv(x, weight, bias=None, activation=None, initial_state=None, cu=None):
    """Returns (y, states after the last token [sequences, W-1, D])."""
    W, ys, states = weight.shape[1], [], []
    for i, (b, t0, t1) in enumerate(_spans(x, cu)):
        head = initial_state[i] if initial_state is not None else x.new_zeros(W - 1, x.shape[2])
        line = torch.cat([head, x[b, t0:t1][0]])
        pre = sum(line[w:w + t1 - t0] * weight[:, w] for w in range(W))
        ys.append(act(activation, pre if bias is None else pre + bias))
        states.append(line[t1 - t0:])
    return torch.cat(ys).view(x.shape), torch.stack(states)


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None, cu=None):
    """B, C [B,T,G,N].  Returns (y, states after the last token [sequences, M, N])."""
    M = u.shape[2]
    dt = dt if dt_bias is None else dt + dt_bias
    if dt_softplus:
        dt = torch.nn.functional.softplus(dt, threshold=700.0)
    B, C = (v.repeat_interleave(M // v.shape[2], 2) for v in (B, C))
    ys, states = [], []
    for i, (b, t0, t1) in enumerate(_spans(u, cu)):
        h = initial_state[i] if initial_state is not None else u.new_zeros(M, A.shape[1])
        for t in range(t0, t1):
            h = torch.exp(dt[b, t][0][:, None] * A) * h + (dt[b, t] * u[b, t])[0][:, None] * B[b, t][0]
            ys.append((h * C[b, t][0]).sum(-1))
        states.append(h)
    y = torch.stack(ys).view(u.shape)
    if D is not None:
        y = y + D * u
    return (y if z is None else y * act("silu", z)), torch.stack(states)


def gated_rms_norm(x, gate, weight, eps=1e-6, activation="silu", gate_first=False):
    s = act(activation, gate)
    v = x * s if gate_first else x
    n = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    return n * weight if gate_first else n * weight * s


def residual_rms_norm(x, residual, weight, scale=1.0, eps=1e-6):
    r = scale * x if residual is None else residual + scale * x
    return r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps) * weight, r
