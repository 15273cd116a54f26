"""The operators around a recurrence at their edges: derivatives that they do not have, extreme values, gradients of views and of single
outputs.  Tolerances as derived in test_gpu_layers.py."""
import pytest
import torch
from torch.autograd import forward_ad

import rewy_b200
from test_gpu_layers import BF16, DEV, FP16, FP32, NAMES, _calls, _close, _compare, _gen, _leaves, oracle

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


def test_decays_over_the_range_of_arguments():
    """Through a step on a state of ones without input: exp(dt A) for arguments a from -1e-9 to -80.  A log2 e and its constant, the
    product with dt and the multiply-add each round by 2^-24 of the argument at most, the offset that the multiply-add adds is below
    2e-8, the exponential is within 2 ulp (2^-22).  Errors of one sign would gather up over a state's memory, token by token: on
    average they stay below half a step of values under 1, 2^-24, as correctly rounded values' own errors do, plus the argument's."""
    gen = torch.Generator(device=DEV).manual_seed(41)
    edges = (1e-9, 1e-8, 1e-7, 1e-6, 1e-5, 1e-4, 1e-3, 5e-3, 0.02, 0.1, 0.5, 1.0, 4.0, 16.0, 64.0)
    for lo, hi in zip(edges, edges[1:]):
        M, N, B = 1024, 64, 8
        A = -(lo * (hi / lo) ** torch.rand(M, N, device=DEV, generator=gen, dtype=torch.float64)).float()
        dt, state, none = 0.75 + 0.5 * torch.rand(B, M, device=DEV, generator=gen), torch.ones(B, M, N, device=DEV), torch.zeros(B, N, device=DEV)
        rewy_b200.selective_scan_step(torch.zeros_like(dt), dt, A, none, none, state)
        a = dt.double()[:, :, None] * A.double()
        off = state.double() / a.exp() - 1
        assert (off.abs() <= 2 ** -22 + 2e-8 - a * 4 * 2 ** -24).all(), (lo, off.abs().max().item())
        assert off.mean().abs() <= 2 ** -24 - (a.mean() * 4 * 2 ** -24), (lo, off.mean().item())


# ---- gradients of views, of single outputs and of long tensors -------------------------------------------------------

@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("shift", (0, 3))
@pytest.mark.parametrize("T", (60, 700))
def test_selective_scan_gradients_of_views(dtype, shift, T):
    """u and z halves of one projection, B and C slices of another (aligned and at an odd offset), a transposed dt; in one segment of
    tokens and in several."""
    rn, M = _gen(35), 96 - (shift > 0)
    xs = dict(wide=rn(2, T, 194).to(dtype), proj=rn(2, T, 48).to(dtype), steps=(0.2 * rn(2, M, T).abs()).to(dtype), A=-rn(M, 16).abs() - 0.05, D=rn(M))

    def apply(scan, wide, proj, steps, A, D):
        u, z, Bm, C = wide[..., :M], wide[..., 96:96 + M], proj[..., shift:shift + 16], proj[..., 16 + shift:32 + shift]
        return scan(u, steps.transpose(1, 2), A, Bm, C, D, z)

    _compare(lambda **x: apply(lambda u, dt, A, B, C, D, z: rewy_b200.selective_scan(u, dt, A, B, C, D, z=z, output_final_state=True), **x),
             lambda **x: apply(lambda u, dt, A, B, C, D, z: oracle.selective_scan(u, dt, A, B[:, :, None], C[:, :, None], D, z), **x), xs, (dtype, FP32))


def test_selective_scan_gradients_of_broadcast_inputs():
    """One B for all groups, one C and one dt for all sequences: their gradients are the sums over what they were spread to."""
    rn = _gen(36)
    xs = dict(u=rn(3, 40, 24), dt=0.3 * rn(1, 40, 24).abs(), A=-rn(24, 16).abs() - 0.05, B=rn(3, 40, 1, 16), C=rn(1, 40, 2, 16))
    spread = lambda u, dt, A, B, C: (u, dt.expand(3, -1, -1), A, B.expand(-1, -1, 2, -1), C.expand(3, -1, -1, -1))  # noqa: E731
    _compare(lambda **x: rewy_b200.selective_scan(*spread(**x))[:1], lambda **x: oracle.selective_scan(*spread(**x))[:1], xs, (FP32,))


VIEWS = {"heads of a slice": (BF16, (3, 50, 776), lambda g: g[..., :768].unflatten(-1, (6, 128))),
         "at an odd offset": (BF16, (3, 50, 776), lambda g: g[..., 5:773].unflatten(-1, (6, 128))),
         "transposed batch": (FP16, (50, 3, 6, 128), lambda g: g.transpose(0, 1)),
         "rows apart": (FP32, (3, 50, 128, 6), lambda g: g.transpose(-1, -2)),
         "three strides": (BF16, (3, 100, 12, 128), lambda g: g[:, ::2, ::2]),
         "one for all heads": (FP32, (3, 50, 1, 128), lambda g: g.expand(-1, -1, 6, -1))}


@pytest.mark.parametrize("view", VIEWS)
def test_norm_gradients_of_views(view):
    rn = _gen(37)
    dtype, size, of = VIEWS[view]
    xs = dict(x=rn(3, 50, 6, 128).to(dtype), base=rn(*size).to(dtype), weight=1 + 0.1 * rn(128))
    for first in (False, True):
        _compare(lambda x, base, weight: (rewy_b200.gated_rms_norm(x, of(base), weight, gate_first=first),),
                 lambda x, base, weight: (oracle.gated_rms_norm(x, of(base), weight, gate_first=first),), xs, (dtype,))
        _compare(lambda x, base, weight: (rewy_b200.gated_rms_norm(of(base), x, weight, gate_first=first),),
                 lambda x, base, weight: (oracle.gated_rms_norm(of(base), x, weight, gate_first=first),), xs, (dtype,))
    _compare(lambda x, base, weight: rewy_b200.residual_rms_norm(x, of(base), weight, scale=0.5),
             lambda x, base, weight: oracle.residual_rms_norm(x, of(base), weight, 0.5), xs, (dtype, dtype))
    _compare(lambda x, base, weight: rewy_b200.residual_rms_norm(of(base), x, weight, scale=0.5),
             lambda x, base, weight: oracle.residual_rms_norm(of(base), x, weight, 0.5), xs, (dtype, dtype))


@pytest.mark.parametrize("name", ("causal_conv", "selective_scan", "residual_rms_norm"))
def test_gradients_of_the_last_output_alone(name):
    """The final state or the residual without the output beside it, whose gradient then never comes."""
    call, xs = _calls(_gen(38))[name]
    definition = {"causal_conv": lambda **x: oracle.causal_conv(**x, activation="silu"), "selective_scan": lambda **x: oracle.selective_scan(**x, dt_softplus=True),
                  "residual_rms_norm": oracle.residual_rms_norm}[name]
    mine, exact = _leaves(xs), _leaves({n: x.double() for n, x in xs.items()})
    got, want = call(**mine)[-1], definition(**exact)[-1]
    seed = _gen(39)(*got.shape)
    grads = torch.autograd.grad(got, list(mine.values()), seed, allow_unused=True)
    exacts = torch.autograd.grad(want, list(exact.values()), seed.double(), allow_unused=True)
    for (n, x), g, e in zip(xs.items(), grads, exacts):
        _close(torch.zeros_like(x) if g is None else g, torch.zeros_like(x) if e is None else e, n)


def test_gradients_beyond_32_bits():
    """More than 2^31 elements in a tensor: the gradients of its last rows are what they are alone, bit for bit where a row's arithmetic
    does not depend on the others, and the convolution's weight gradient is that of the definition over all rows."""
    gen = torch.Generator(device=DEV).manual_seed(40)
    rn = lambda *s, t=BF16: torch.empty(*s, device=DEV, dtype=t).normal_(generator=gen)  # noqa: E731
    D, tail = 4096, 9
    rows = (1 << 31) // D + 100
    x, dy, weight = rn(1, rows, D), rn(1, rows, D), (rn(D, 4, t=FP32) / 2).requires_grad_()

    def conv(x, dy, state=None):
        x = x.detach().requires_grad_()
        y, _ = rewy_b200.causal_conv(x, weight, activation="silu", initial_state=state)
        return torch.autograd.grad(y, (x, weight), dy)

    dx, dw = conv(x, dy)
    alone, _ = conv(x[:, -tail:], dy[:, -tail:], x[:, -tail - 3:-tail].contiguous())
    assert torch.equal(dx[:, -tail:], alone)
    del dx
    last = [v[..., -8:].double().detach().requires_grad_() for v in (x, weight.t())]
    y, _ = oracle.causal_conv(last[0], last[1].t(), activation="silu")
    _close(dw[-8:], torch.autograd.grad(y, last[1], dy[..., -8:].double())[0].t(), "dweight")
    del y, last
    norm = rn(D, t=FP32)

    def gated(x, dy):
        x, gate = x.detach().requires_grad_(), dy.detach().requires_grad_()
        return torch.autograd.grad(rewy_b200.gated_rms_norm(x, gate, norm), (x, gate), dy)

    whole = gated(x, dy)
    for a, b in zip(whole, gated(x[:, -tail:], dy[:, -tail:])):
        assert torch.equal(a[:, -tail:], b)
    del whole

    def residual(x, dy):
        x, r = x.detach().requires_grad_(), dy.detach().requires_grad_()
        return torch.autograd.grad(rewy_b200.residual_rms_norm(x, r, norm, scale=0.5), (x, r), (dy, x.detach()))

    whole = residual(x, dy)
    for a, b in zip(whole, residual(x[:, -tail:], dy[:, -tail:])):
        assert torch.equal(a[:, -tail:], b)
    del whole
    M = 256
    x, dy = x.view(1, -1, M), dy.view(1, -1, M)
    A, Bm = -torch.rand(M, 16, device=DEV) - 0.5, rn(1, x.shape[1], 16)

    def scan(u, dy, Bm):
        u, dt, Bm = (v.detach().requires_grad_() for v in (u, u, Bm))
        y, _ = rewy_b200.selective_scan(u, dt, A, Bm, Bm.detach(), dt_softplus=True)
        return torch.autograd.grad(y, (u, dt, Bm), dy)

    whole, short = scan(x, dy, Bm), scan(x[:, -2000:], dy[:, -2000:], Bm[:, -2000:])
    for a, b in zip(whole, short):                          # 1000 tokens forget where they began; both sides are rounded to BF16
        a, b = a[:, -1000:].double(), b[:, -1000:].double()
        assert ((a - b).abs() <= 2 ** -7 * 1.01 * b.abs() + 1e-4 * b.square().mean().sqrt()).all()
