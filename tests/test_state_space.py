"""The layers of a state space block (norm_residual, causal_conv, selective_scan in pysiglib_amd/sequence.py) against their formulas in 64
bits, and their gradients also against differences of those.

Tolerances.  u = 2^-24, 2^-8, 2^-11 is the largest relative rounding error of float32, bfloat16 and float16; an output rounded once is off by u
times its size.  What 32-bit steps add on the way is bounded by evaluating the formula on absolute values twice, once with every factor
enlarged by the roundings that it goes through: the difference bounds the error, however the terms are ordered."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

DEV = "cuda:0"
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SMALL = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


@pytest.fixture(scope="module")
def P():
    import pysiglib_amd
    return pysiglib_amd


def f64(t):
    return t.detach().double().cpu().numpy()


def within(got, want, bound, what):
    """Every value within the bound; infinities and NaN in the same places."""
    got = f64(got)
    assert got.shape == want.shape, what
    fine = np.isfinite(want)
    assert (np.isnan(got) == np.isnan(want)).all(), what
    assert (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all(), what
    off = np.abs(got[fine] - want[fine])
    over = off - np.broadcast_to(bound, want.shape)[fine]
    assert over.size == 0 or over.max() <= 0, (what, float(over.max()), float(off.max()))


def rounded(want, bound, dtype):
    """The bound of a result in `dtype` whose 32-bit value is within `bound`."""
    return bound + ROUND[dtype] * (np.abs(want) + bound) + SMALL[dtype]


def numbers(rng, *shape, dtype=torch.float32, size=1.0):
    return torch.tensor(size * rng.standard_normal(shape)).to(dtype).to(DEV)


def whole_numbers(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts_of(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-v))


def slope(v):
    s = sigmoid(v)
    return s * (1 + v * (1 - s))


def same_bits(a, b):
    for x, y in zip(a, b):
        if x is not None and x.numel():
            assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)), "the same inputs give the same bits"


# ---- the norm of the residual stream ----

def norm_oracle(total, w, eps, grad=None, grad_total=None):
    """Values and what 32-bit steps may add: a sum of `channels` squares and a dozen roundings, of values no larger than the row's largest."""
    channels = total.shape[-1]
    r = 1 / np.sqrt((total * total).mean(-1, keepdims=True) + eps)
    y = total * r * w
    f32 = (channels + 16) * U32
    if grad is None:
        return y, f32 * np.abs(y)
    u = grad * w
    mean = (u * total).mean(-1, keepdims=True)
    ds = r * (u - total * r * r * mean)
    more = f32 * 2 * r * (np.abs(u) + np.abs(total) * r * r * np.abs(u * total).mean(-1, keepdims=True))
    if grad_total is not None:
        ds, more = ds + grad_total, more + U32 * (np.abs(ds) + np.abs(grad_total))
    axes = tuple(range(total.ndim - 1))
    terms = np.abs(grad * total * r).sum(axes)
    rows = total.size // channels
    return y, f32 * np.abs(y), ds, more, (grad * total * r).sum(axes), (f32 + (rows + 8) * U32) * terms


NORM_SHAPES = [(1, 1), (3, 7), (2, 64), (5, 127), (3, 512), (1500, 513), (33, 1000), (7, 4096), (3, 5000), (2, 16384), (1100, 24), (4, 8200), (2, 3, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stream", ["none", "same", "float32"])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norm_residual(P, dtype, stream, shape):
    rng = np.random.default_rng(shape[-1])
    kind = torch.float32 if stream == "float32" else dtype
    x, w = numbers(rng, *shape, dtype=dtype), numbers(rng, shape[-1]) * 0.3 + 1
    residual = None if stream == "none" else numbers(rng, *shape, dtype=kind, size=3.0)
    out, total = P.norm_residual(x, residual, w, eps=1e-5)
    if residual is None:
        assert total is x
    else:
        want = f64(x) + f64(residual)
        within(total, want, rounded(want, U32 * np.abs(want), kind), "total")
        assert torch.equal(total, (x.float() + residual.float()).to(kind))
    grad, after = numbers(rng, *shape, dtype=dtype), numbers(rng, *shape, dtype=kind)
    want = norm_oracle(f64(total), f64(w), 1e-5, f64(grad), f64(after))
    within(out, want[0], rounded(want[0], want[1], dtype), "out")
    back = P.norm_residual_backprop(grad, total, w, grad_total=after, eps=1e-5)
    same_bits(back, P.norm_residual_backprop(grad, total, w, grad_total=after, eps=1e-5))
    within(back[0], want[2], rounded(want[2], want[3], dtype), "grad_x")
    within(back[1], want[2], rounded(want[2], want[3], kind), "grad_residual")
    assert (back[0] is back[1]) == (kind == dtype)
    within(back[2], want[4], rounded(want[4], want[5], torch.float32), "grad_weight")
    want = norm_oracle(f64(total), f64(w), 1e-5, f64(grad))
    within(P.norm_residual_backprop(grad, total, w, eps=1e-5)[0], want[2], rounded(want[2], want[3], dtype), "without the gradient of the sum")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stream", ["none", "same", "float32"])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norm_residual_in_8_bits(P, dtype, stream, shape):
    """q is the nearest of the format's values to out / scale, which is off by the roundings of out and of the division: half a step is 2^-4
    of the value, or 2^-10 among the smallest."""
    rng = np.random.default_rng(shape[-1])
    kind = torch.float32 if stream == "float32" else dtype
    x, w = numbers(rng, *shape, dtype=dtype), numbers(rng, shape[-1]) * 0.3 + 1
    x[..., 0] *= 50.0
    residual = None if stream == "none" else numbers(rng, *shape, dtype=kind, size=3.0)
    q, scales, total = P.norm_residual_float8(x, residual, w, eps=1e-5)
    assert q.dtype == torch.float8_e4m3fn and scales.shape == (*shape[:-1], 1)
    if residual is not None:
        assert torch.equal(total, (x.float() + residual.float()).to(kind))
    y, more = norm_oracle(f64(total), f64(w), 1e-5)
    want = np.abs(y).max(-1, keepdims=True) / 448
    within(scales, want, more.max(-1, keepdims=True) / 448 + 2 * U32 * want + 1e-45, "scales")
    v = y / f64(scales)
    off = more / f64(scales) + 4 * U32 * np.abs(v)
    within(q.float(), v, np.maximum(2.0 ** -4 * (np.abs(v) + off), 2.0 ** -10) + off, "q")
    assert (f64(q.float().abs().amax(-1)) == 448).all()
    within(q.float(), f64((total.float() * 0 + torch.tensor(v, device=DEV).float()).clamp(-448, 448).to(torch.float8_e4m3fn).float()),
           np.maximum(2.0 ** -3 * np.abs(v), 2.0 ** -9) * (1 + 2.0 ** -3), "q and torch's own conversion are at most a step apart")


@pytest.mark.gpu
def test_norm_residual_in_8_bits_rounds_to_nearest_and_ties_to_even(P):
    """A row whose norm, weight and scale are exact: r = 1 for entries of one size, weights do the rest."""
    v = torch.cat([torch.tensor([448.0, 17.0, 19.0, 18.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 2.0 ** -6, 1.0625, 1.1875, -1.0625, 432.0, 0.0, 465.0 / 464 * 440])])
    x = torch.ones((2, len(v)), device=DEV)
    q, scales, _ = P.norm_residual_float8(x, None, v.to(DEV), eps=0.0)
    assert (scales == 1.0).all()
    assert torch.equal(q[0].float().cpu(), v.to(torch.float8_e4m3fn).float()) and torch.equal(q[0].float(), q[1].float())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [40, 3000, 9000])
def test_norm_residual_of_zeros_and_of_what_is_not_finite(P, dtype, channels):
    """A row's values stay in it."""
    x = torch.ones((6, channels), dtype=dtype, device=DEV)
    x[1] = 0.0
    x[2, 5], x[3, channels - 1] = float("nan"), float("inf")
    w = torch.ones(channels, device=DEV)
    out, _ = P.norm_residual(x, None, w, eps=1e-6)
    assert (out[1] == 0).all() and torch.isnan(out[2]).all() and torch.isnan(out[3, -1]) and (out[3, :-1] == 0).all()
    assert torch.isfinite(out[[0, 4, 5]]).all()
    q, scales, _ = P.norm_residual_float8(x, None, w, eps=1e-6)
    assert (q[1].float() == 0).all() and scales[1] == 1 and scales[2] == 1 and scales[3] == 1
    assert torch.isnan(q[2].float()).all() and torch.isnan(q[3, -1].float()) and (q[0].float() == 448).all()
    dx, _, dw = P.norm_residual_backprop(torch.ones_like(x), x, w)
    assert torch.isfinite(dx[[0, 1, 4, 5]]).all() and torch.isnan(dx[2]).all() and torch.isnan(dw[5])
    tiny = torch.full((1, channels), 1e-30, device=DEV)
    q, scales, _ = P.norm_residual_float8(tiny.to(torch.float32), None, w * 1e-9, eps=1.0)
    assert torch.isfinite(scales).all() and ((q.float().abs() <= 448) | (scales < 1e-37)).all()


@pytest.mark.gpu
def test_norm_residual_gradients_are_differences(P):
    rng = np.random.default_rng(5)
    t, w, g, after = numbers(rng, 4, 30), numbers(rng, 30) + 1, numbers(rng, 4, 30), numbers(rng, 4, 30)
    dx, _, dw = P.norm_residual_backprop(g, t, w, grad_total=after, eps=1e-3)
    loss = lambda t, w: (norm_oracle(t, w, 1e-3)[0] * f64(g)).sum() + (t * f64(after)).sum()       # noqa: E731
    for _ in range(4):
        v, z = rng.standard_normal(t.shape), rng.standard_normal(30)
        d = (loss(f64(t) + 1e-4 * v, f64(w)) - loss(f64(t) - 1e-4 * v, f64(w))) / 2e-4
        assert abs((f64(dx) * v).sum() - d) <= 1e-5 * np.abs(f64(dx) * v).sum()
        d = (loss(f64(t), f64(w) + 1e-4 * z) - loss(f64(t), f64(w) - 1e-4 * z)) / 2e-4
        assert abs((f64(dw) * z).sum() - d) <= 1e-5 * np.abs(f64(dw) * z).sum()


# ---- the convolution ----

def conv_oracle(x, state, w, bias, starts, silu, grad=None, grad_final=None):
    """Over packed rows; the outputs and their bounds."""
    rows, channels = x.shape
    width = w.shape[1]
    kept = width - 1
    y, ey = np.zeros_like(x), np.zeros_like(x)
    final = np.zeros_like(state)
    dx, ex = np.zeros_like(x), np.zeros_like(x)
    d0, e0 = np.zeros_like(state), np.zeros_like(state)
    dw, ew, db, eb = np.zeros_like(w), np.zeros_like(w), np.zeros(channels), np.zeros(channels)
    for i in range(len(starts) - 1):
        s, t = starts[i], starts[i + 1]
        n = t - s
        ext = np.concatenate((state[i], x[s:t]))
        final[i] = ext[n:]
        v, size = np.tile(bias, (n, 1)), np.tile(np.abs(bias), (n, 1))
        for k in range(width):
            v, size = v + w[:, k] * ext[k:k + n], size + np.abs(w[:, k] * ext[k:k + n])
        ev = (width + 2) * U32 * size
        # the activation: its slope is at most 1.1, and the exponential of v is off by 2 |v| roundings and a few
        y[s:t] = v * sigmoid(v) if silu else v
        ey[s:t] = 1.1 * ev + (8 + 2 * np.abs(v)) * U32 * np.abs(y[s:t]) if silu else ev
        if grad is None:
            continue
        g = grad[s:t]
        e = g * slope(v) if silu else g
        # its second derivative is at most 0.5; the slope's two terms are at most 1 + |v| times the exponential's error
        ee = np.abs(g) * (0.5 * ev + (1 + np.abs(v)) * (12 + 2 * np.abs(v)) * U32) if silu else 0 * g
        back, eback, bsize = np.zeros_like(ext), np.zeros_like(ext), np.zeros_like(ext)
        for k in range(width):
            back[k:k + n] += e * w[:, k]
            eback[k:k + n] += ee * np.abs(w[:, k])
            bsize[k:k + n] += np.abs(e * w[:, k])
            dw[:, k] += (e * ext[k:k + n]).sum(0)
            ew[:, k] += (ee * np.abs(ext[k:k + n]) + (rows + 8) * U32 * np.abs(e * ext[k:k + n])).sum(0)
        db += e.sum(0)
        eb += (ee + (rows + 8) * U32 * np.abs(e)).sum(0)
        back[n:] += grad_final[i]
        bsize[n:] += np.abs(grad_final[i])
        eback += (width + 2) * U32 * bsize
        dx[s:t], ex[s:t] = back[kept:], eback[kept:]
        d0[i], e0[i] = back[:kept], eback[:kept]
    return (y, final, dx, dw, db, d0), (ey, 0 * final, ex, ew, eb, e0)


CONV_SEQUENCES = [[1], [2], [3], [7] * 30, [0, 5, 0, 0, 1, 130, 0], [400, 1, 1, 1, 126, 2, 128, 129], [0, 0], [2500], [16, 16, 32, 15, 17, 48]]


def check_conv(P, dtype, lengths, channels, width, silu, packed, with_bias=True, with_states=True, seed=0):
    rng = np.random.default_rng(seed + channels + width)
    starts, n = starts_of(lengths), len(lengths)
    rows = starts[-1]
    both = numbers(rng, rows, 2 * channels, dtype=dtype)            # a part of a projection
    x, grad = both[:, :channels], numbers(rng, rows, channels, dtype=dtype)
    w, bias = numbers(rng, channels, width), numbers(rng, channels)
    state, gf = numbers(rng, n, width - 1, channels, dtype=dtype), numbers(rng, n, width - 1, channels, dtype=dtype)
    shape = lambda t: t if packed else t.reshape(n, -1, channels)    # noqa: E731
    options = dict(silu=silu, offsets=whole_numbers(starts) if packed else None, initial_state=state if with_states else None)
    b = bias if with_bias else None
    y, final = P.causal_conv(shape(x), w, b, **options)
    back = P.causal_conv_backprop(shape(grad), shape(x), w, b, grad_final=gf if with_states else None, **options)
    same_bits((y, *back), (P.causal_conv(shape(x), w, b, **options)[0],
                           *P.causal_conv_backprop(shape(grad), shape(x), w, b, grad_final=gf if with_states else None, **options)))
    zero = np.zeros((n, width - 1, channels))
    want, bound = conv_oracle(f64(x), f64(state) if with_states else zero, f64(w), f64(bias) if with_bias else np.zeros(channels), starts, silu,
                              f64(grad), f64(gf) if with_states else zero)
    assert (f64(final) == want[1]).all(), "the last rows are copies"
    assert (back[2] is None) == (not with_bias)
    for name, got, v, e, kind in zip(("y", "dx", "dw", "db", "d0"), (y, *back), (want[0], *want[2:]), (bound[0], *bound[2:]),
                                     (dtype, dtype, torch.float32, torch.float32, dtype)):
        if got is not None:
            within(got.reshape(v.shape), v, rounded(v, e, kind), name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", CONV_SEQUENCES)
@pytest.mark.parametrize("channels,width,silu", [(1, 4, True), (5, 2, True), (40, 4, True), (133, 3, False), (3, 8, True), (600, 4, True)])
def test_causal_conv_packed(P, dtype, lengths, channels, width, silu):
    check_conv(P, dtype, lengths, channels, width, silu, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("batch,length,channels", [(3, 50, 70), (2, 5, 9), (1, 1, 3), (4, 64, 2)])
def test_causal_conv_batched(P, dtype, width, batch, length, channels):
    check_conv(P, dtype, [length] * batch, channels, width, width % 2 == 0, False)
    check_conv(P, dtype, [length] * batch, channels, width, width % 2 == 1, False, with_bias=False, with_states=False, seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 4, 8])
@pytest.mark.parametrize("rows,channels", [(1, 1), (5, 37), (64, 256)])
def test_causal_conv_step_follows_the_sequence(P, dtype, width, rows, channels):
    rng = np.random.default_rng(rows)
    x, w, bias = numbers(rng, rows, 12, channels, dtype=dtype), numbers(rng, channels, width), numbers(rng, channels)
    state = numbers(rng, rows, width - 1, channels, dtype=dtype)
    want, final = P.causal_conv(x, w, bias, initial_state=state)
    before = state._version
    for t in range(12):
        assert torch.equal(P.causal_conv_step(x[:, t], state, w, bias), want[:, t])
    assert torch.equal(state, final) and state._version > before
    want = P.causal_conv_step(x[0, 0], state[0].clone(), w, None, silu=False)
    assert torch.equal(P.causal_conv(x[:1, :1], w, None, initial_state=state[:1], silu=False)[0][0, 0], want)


@pytest.mark.gpu
def test_causal_conv_gradients_are_differences(P):
    rng = np.random.default_rng(3)
    rows, channels, width, starts = 60, 5, 4, [0, 2, 2, 33, 60]
    x, state, w, bias = numbers(rng, rows, channels), numbers(rng, 4, width - 1, channels), numbers(rng, channels, width), numbers(rng, channels)
    g, gf = numbers(rng, rows, channels), numbers(rng, 4, width - 1, channels)
    grads = P.causal_conv_backprop(g, x, w, bias, grad_final=gf, initial_state=state, offsets=whole_numbers(starts))

    def loss(x, w, bias, state):
        (y, final, *_), _ = conv_oracle(x, state, w, bias, starts, True)
        return (y * f64(g)).sum() + (final * f64(gf)).sum()

    at = [f64(t) for t in (x, w, bias, state)]
    for k in range(4):
        for _ in range(3):
            v = rng.standard_normal(at[k].shape)
            up, down = list(at), list(at)
            up[k], down[k] = at[k] + 1e-4 * v, at[k] - 1e-4 * v
            d = (loss(*up) - loss(*down)) / 2e-4
            assert abs((f64(grads[k]) * v).sum() - d) <= 1e-5 * np.abs(f64(grads[k]) * v).sum(), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_causal_conv_of_what_is_not_finite(P, dtype, bad):
    """It reaches the rows and weights that the formula sums it into, not a neighbouring sequence or channel."""
    x = torch.ones((90, 24), dtype=dtype, device=DEV)
    x[29, 3] = bad
    w = torch.ones((24, 4), device=DEV)
    offsets = whole_numbers([0, 30, 30, 90])
    y, final = P.causal_conv(x, w, offsets=offsets, silu=False)
    at = ~torch.isfinite(y)
    assert at.sum() == 1 and at[29, 3] and not torch.isfinite(final[0, 2, 3])
    dx, dw, _, d0 = P.causal_conv_backprop(torch.ones_like(x), x, w, offsets=offsets, silu=True)
    at = ~torch.isfinite(dx)
    assert at[:, [c for c in range(24) if c != 3]].sum() == 0 and at[30:].sum() == 0 and at[:26].sum() == 0
    assert torch.isfinite(d0).all() and torch.isfinite(dw[[c for c in range(24) if c != 3]]).all()


# ---- the scan ----

def scan_terms(k, dt, x, b, c, d, a, gate, h0, starts, of, gy=None, g=None, gf=None, gate_slope=None, chain=None, n_sum=0, widen=0.0):
    """Outputs over packed rows, from the factors of the formula: k (rows, channels, states) the decays, gate = z sigmoid(z), chain = the
    derivative of dt.  Sums of n terms are enlarged by widen * n."""
    rows, channels = x.shape
    states = a.shape[1]
    y, h_all, before = np.zeros_like(x), np.zeros((rows, channels, states)), np.zeros((rows, channels, states))
    final = np.array(h0, dtype=np.float64)
    du = (dt * x)[..., None]
    for i in range(len(starts) - 1):
        h = h0[i]
        for t in range(starts[i], starts[i + 1]):
            before[t] = h
            h = (k[t] * h + du[t] * b[t][of]) * (1 + widen)
            h_all[t] = h
        final[i] = h
    over = lambda v, n: v * (1 + widen * n)          # noqa: E731
    y = over((h_all * c[:, of]).sum(-1) + d * x, states + 6)
    out = [y * gate, final]
    if gy is None:
        return out
    G_all, into = np.zeros_like(h_all), np.zeros_like(h_all)
    d0 = np.array(gf, dtype=np.float64)
    for i in range(len(starts) - 1):
        back = gf[i]
        for t in range(starts[i + 1] - 1, starts[i] - 1, -1):
            G = (back + gy[t][:, None] * c[t][of]) * (1 + widen)
            G_all[t] = G
            back = G * k[t]
            into[t] = back
        d0[i] = back
    groups = b.shape[1]
    grouped = lambda v: over(v.reshape(rows, groups, channels // groups, states).sum(2), channels + 8)         # noqa: E731
    rate = into * before
    through = over((G_all * b[:, of]).sum(-1), states + 6)
    ddt = over((rate * a).sum(-1), states + 8) + through * x
    ddelta = ddt * (1 + 2 * widen) * chain
    out += [through * dt + d * gy, ddelta, over((rate * dt[..., None]).sum(0), rows + 16), grouped(G_all * du), grouped(h_all * gy[..., None]),
            over((gy * x).sum(0), rows + 8), g * y * gate_slope, over(ddelta.sum(0), rows + 8), d0]
    return out


NAMES = ("y", "final", "dx", "ddelta", "da", "db", "dc", "dd", "dz", "dbias", "d0")


def scan_oracle(x, delta, a, b, c, d, z, bias, h0, starts, softplus, g=None, gf=None):
    """Values and bounds.  Roundings: dt 10 + 4 |raw| (softplus: the argument's sum and product, the exponential, five of the polynomial), a
    decay 8 + |m| (16 + depth) with m = dt a its exponent: those of dt, of a log2(e), of the product, and of sums of dt over up to `depth` rows
    where a segment's decay is taken at once; the gate 8 + 2 |z|."""
    channels = x.shape[1]
    of = np.arange(channels) // (channels // b.shape[1])
    raw = delta + bias
    dt = np.logaddexp(raw, 0) if softplus else raw
    chain = sigmoid(raw) if softplus else np.ones_like(raw)
    gate = z * sigmoid(z) if z is not None else np.ones_like(x)
    gs = slope(z) if z is not None else np.zeros_like(x)
    m = dt[..., None] * a
    gy = None if g is None else g * gate
    want = scan_terms(np.exp(m), dt, x, b, c, d, a, gate, h0, starts, of, gy, g, gf, gs, chain)
    depth = 24
    ab = np.abs
    edt, ez = (10 + 4 * ab(raw)) * U32, (8 + 2 * ab(z)) * U32 if z is not None else 2 * U32
    gsa = sigmoid(z) * (1 + ab(z) * (1 - sigmoid(z))) if z is not None else gs
    args = lambda s: (np.exp(m) * (1 + s * (8 + ab(m) * (16 + depth + 4 * ab(raw[..., None]))) * U32), ab(dt) * (1 + s * edt), ab(x), ab(b), ab(c) * (1 + s * U32),  # noqa: E731
                      ab(d), ab(a) * (1 + 2 * s * U32), ab(gate) * (1 + s * ez), ab(h0), starts, of,
                      None if g is None else ab(gy) * (1 + s * ez), None if g is None else ab(g), None if gf is None else ab(gf), ab(gsa) * (1 + s * 2 * ez),
                      chain * (1 + s * (8 + 2 * ab(raw)) * U32))
    plain, wide = scan_terms(*args(0)), scan_terms(*args(1), widen=2 * U32)
    return want, [p - q + 2 * U32 * p for p, q in zip(wide, plain)]


def scan_inputs(dtype, rows, n, channels, states, groups, seed, decays=1.0):
    rng = np.random.default_rng(seed)
    both = numbers(rng, rows, groups, 2 * states, dtype=dtype)
    t = dict(x=numbers(rng, rows, channels, dtype=dtype), delta=numbers(rng, rows, channels, dtype=dtype), b=both[..., :states], c=both[..., states:],
             z=numbers(rng, rows, channels, dtype=dtype), g=numbers(rng, rows, channels, dtype=dtype),
             a=-decays * torch.tensor(np.exp(rng.uniform(-2, 1, (channels, states))), dtype=torch.float32, device=DEV),
             d=numbers(rng, channels), bias=numbers(rng, channels) - 2.0, h0=numbers(rng, n, channels, states), gf=numbers(rng, n, channels, states))
    return t


def check_scan(P, t, starts, packed, gate=True, softplus=True, d=True, bias=True, states=True, skip=()):
    n, (rows, channels), dtype = len(starts) - 1, t["x"].shape, t["x"].dtype
    shape = lambda v: v if packed or v is None else v.reshape(n, -1, *v.shape[1:])          # noqa: E731
    z = t["z"] if gate else None
    options = dict(d=t["d"] if d else None, z=shape(z), delta_bias=t["bias"] if bias else None, softplus=softplus,
                   initial_state=t["h0"] if states else None, offsets=whole_numbers(starts) if packed else None)
    args = [shape(t["x"]), shape(t["delta"]), t["a"], shape(t["b"]), shape(t["c"])]
    out = P.selective_scan(*args, **options)
    back = P.selective_scan_backprop(shape(t["g"]), *args, grad_final=t["gf"] if states else None, **options)
    same_bits((*out, *back), (*P.selective_scan(*args, **options),
                              *P.selective_scan_backprop(shape(t["g"]), *args, grad_final=t["gf"] if states else None, **options)))
    none = np.zeros((n, channels, t["a"].shape[1]))
    want, bound = scan_oracle(f64(t["x"]), f64(t["delta"]), f64(t["a"]), f64(t["b"]), f64(t["c"]), f64(t["d"]) if d else np.zeros(channels),
                              f64(z) if gate else None, f64(t["bias"]) if bias else np.zeros(channels), f64(t["h0"]) if states else none, starts, softplus,
                              f64(t["g"]), f64(t["gf"]) if states else none)
    kinds = (dtype, torch.float32, dtype, dtype, torch.float32, dtype, dtype, torch.float32, dtype, torch.float32, torch.float32)
    assert (back[5] is None, back[6] is None, back[7] is None) == (not d, not gate, not bias)
    for name, got, w, e, kind in zip(NAMES, (*out, *back), want, bound, kinds):
        if got is not None and name not in skip:
            within(got.reshape(w.shape), w, rounded(w, e, kind), name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,channels,states,groups", [
    ([1], 1, 1, 1), ([1], 70, 16, 1), ([5, 5], 3, 4, 1), ([17] * 3, 64, 16, 1), ([16, 16], 256, 8, 2), ([300] * 2, 40, 16, 2), ([130], 33, 64, 1),
    ([100] * 2, 36, 33, 3), ([700], 66, 13, 1), ([65] * 4, 20, 5, 5), ([64], 130, 32, 1), ([8] * 5, 300, 3, 1)])
def test_selective_scan_batched(P, dtype, lengths, channels, states, groups):
    starts = starts_of(lengths)
    t = scan_inputs(dtype, starts[-1], len(lengths), channels, states, groups, seed=channels + states)
    check_scan(P, t, starts, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,channels,states,groups", [
    ([1], 5, 16, 1), ([0, 5, 0, 0, 1, 130, 0], 40, 16, 1), ([400, 1, 1, 1, 126, 2, 128, 129], 30, 16, 3), ([7] * 60, 6, 2, 1), ([0, 0], 8, 16, 1),
    ([33, 64, 63, 65, 1], 20, 40, 2), ([500, 0, 300], 9, 7, 1)])
def test_selective_scan_packed(P, dtype, lengths, channels, states, groups):
    starts = starts_of(lengths)
    t = scan_inputs(dtype, starts[-1], len(lengths), channels, states, groups, seed=len(lengths) + states)
    check_scan(P, t, starts, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate,softplus,d,bias,states", [(False, True, True, True, True), (True, False, True, True, True), (True, True, False, False, False),
                                                         (False, True, False, True, False)])
def test_selective_scan_without_some_of_its_inputs(P, dtype, gate, softplus, d, bias, states):
    t = scan_inputs(dtype, 300, 2, 24, 16, 1, seed=4)
    if not softplus:
        t["delta"], t["bias"] = t["delta"].abs() * 0.3, t["bias"].abs() * 0.1
    check_scan(P, t, [0, 150, 300], False, gate=gate, softplus=softplus, d=d, bias=bias, states=states)
    check_scan(P, t, [0, 70, 300], True, gate=gate, softplus=softplus, d=d, bias=bias, states=states)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("decays", [0.0, 1e-3, 30.0, 3000.0])
def test_selective_scan_with_slow_and_fast_decays(P, dtype, decays):
    """Memory of all the rows, and of none."""
    t = scan_inputs(dtype, 400, 1, 20, 16, 1, seed=7, decays=decays)
    check_scan(P, t, [0, 400], False)


@pytest.mark.gpu
def test_selective_scan_where_the_chip_is_full(P):
    """More sequences than there are pieces for the sums over rows: a block goes through several."""
    t = scan_inputs(torch.float32, 3 * 300, 300, 250, 64, 1, seed=1)
    check_scan(P, t, [3 * i for i in range(301)], True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,states,groups", [(1, 1, 1, 1), (3, 40, 16, 2), (64, 130, 64, 1), (5, 12, 7, 3), (7, 33, 2, 1)])
@pytest.mark.parametrize("full", [True, False])
def test_selective_scan_step_follows_the_formula(P, dtype, rows, channels, states, groups, full):
    t = scan_inputs(dtype, rows * 3, rows, channels, states, groups, seed=rows)
    state = t["h0"].clone()
    wanted = f64(state)
    options = dict(d=t["d"], delta_bias=t["bias"]) if full else {}
    for i in range(3):
        part = slice(i * rows, (i + 1) * rows)
        was, before = f64(state), state._version
        got = P.selective_scan_step(t["x"][part], t["delta"][part], t["a"], t["b"][part], t["c"][part], state, z=t["z"][part] if full else None, **options)
        assert state._version > before
        want, bound = scan_oracle(f64(t["x"][part]), f64(t["delta"][part]), f64(t["a"]), f64(t["b"][part]), f64(t["c"][part]),
                                  f64(t["d"]) if full else np.zeros(channels), f64(t["z"][part]) if full else None,
                                  f64(t["bias"]) if full else np.zeros(channels), was, list(range(rows + 1)), True)
        within(got, want[0], rounded(want[0], bound[0], dtype), "y")
        within(state, want[1], rounded(want[1], bound[1], torch.float32), "state")
    one = P.selective_scan_step(t["x"][0], t["delta"][0], t["a"], t["b"][0], t["c"][0], state[0].clone())
    assert torch.equal(one, P.selective_scan_step(t["x"][:1], t["delta"][:1], t["a"], t["b"][:1], t["c"][:1], state[:1].clone())[0])
    assert wanted.shape == state.shape


@pytest.mark.gpu
def test_selective_scan_gradients_are_differences(P):
    starts = [0, 40, 41, 41, 150]
    t = scan_inputs(torch.float32, 150, 4, 6, 5, 2, seed=11)
    args = [t[k] for k in ("x", "delta", "a", "b", "c")]
    grads = P.selective_scan_backprop(t["g"], *args, d=t["d"], z=t["z"], delta_bias=t["bias"], grad_final=t["gf"], initial_state=t["h0"], offsets=whole_numbers(starts))
    names = ("x", "delta", "a", "b", "c", "d", "z", "bias", "h0")
    at = {k: f64(t[k]) for k in names}

    def loss(v):
        channels = v["x"].shape[1]
        of = np.arange(channels) // (channels // v["b"].shape[1])
        dt = np.logaddexp(v["delta"] + v["bias"], 0)
        y, final = scan_terms(np.exp(dt[..., None] * v["a"]), dt, v["x"], v["b"], v["c"], v["d"], v["a"], v["z"] * sigmoid(v["z"]), v["h0"], starts, of)
        return (y * f64(t["g"])).sum() + (final * f64(t["gf"])).sum()

    rng = np.random.default_rng(0)
    for name, grad in zip(names, grads):
        for _ in range(3):
            v = rng.standard_normal(at[name].shape)
            d = (loss({**at, name: at[name] + 1e-4 * v}) - loss({**at, name: at[name] - 1e-4 * v})) / 2e-4
            assert abs((f64(grad) * v).sum() - d) <= 2e-5 * np.abs(f64(grad) * v).sum(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [24, 30, 64])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["x", "z", "g", "b", "c"])
def test_selective_scan_of_what_is_not_finite(P, dtype, channels, bad, which):
    """It reaches what the formula sums it into: not other sequences, other channels' own values, or rows on the other side."""
    t = scan_inputs(dtype, 300, 3, channels, 16, 1, seed=2)
    t[which][120].view(-1)[3] = bad
    starts = [0, 100, 200, 300]
    args, options = [t[k] for k in ("x", "delta", "a", "b", "c")], dict(d=t["d"], z=t["z"], delta_bias=t["bias"], initial_state=t["h0"], offsets=whole_numbers(starts))
    y, final = P.selective_scan(*args, **options)
    dx, ddelta, da, db, dc, dd, dz, dbias, d0 = P.selective_scan_backprop(t["g"], *args, grad_final=t["gf"], **options)
    fine = torch.isfinite
    mine = [c for c in range(channels) if c == 3] if which in ("x", "z", "g") else list(range(channels))
    others = [c for c in range(channels) if c not in mine]
    for v in (y, dx, ddelta, dz):
        assert fine(v[:100]).all() and fine(v[200:]).all() and fine(v[:, others]).all()
    assert fine(final[[0, 2]]).all() and fine(d0[[0, 2]]).all()
    assert fine(y[100:120]).all()
    for v in (db, dc):
        assert fine(v[:100]).all() and fine(v[200:]).all()
    assert fine(da[others]).all() and fine(dd[others]).all() and fine(dbias[others]).all()
    # where they are, against the same formulas in 64 bits
    with np.errstate(all="ignore"):
        want, _ = scan_oracle(f64(t["x"]), f64(t["delta"]), f64(t["a"]), f64(t["b"]), f64(t["c"]), f64(t["d"]), f64(t["z"]), f64(t["bias"]), f64(t["h0"]), starts,
                              True, f64(t["g"]), f64(t["gf"]))
    for name, got, w in zip(NAMES, (y, final, dx, ddelta, da, db, dc, dd, dz, dbias, d0), want):
        assert (np.isfinite(f64(got)) == np.isfinite(w)).all(), name


# ---- all of them ----

@pytest.mark.gpu
def test_layers_of_nothing(P):
    for shape in [(0, 5, 3), (2, 0, 3)]:
        n = shape[0]
        x, w = torch.zeros(shape, device=DEV), torch.ones((3, 4), device=DEV)
        start = torch.ones((n, 3, 3), device=DEV)
        y, final = P.causal_conv(x, w, initial_state=start)
        assert y.shape == shape and (shape[1] or torch.equal(final, start))
        dx, dw, _, d0 = P.causal_conv_backprop(x, x, w, grad_final=start, initial_state=start)
        assert dx.shape == shape and (dw == 0).all() and (shape[1] or torch.equal(d0, start))
        a, b, h = -torch.ones((3, 2), device=DEV), torch.zeros((*shape[:2], 1, 2), device=DEV), torch.ones((n, 3, 2), device=DEV)
        y, final = P.selective_scan(x, x, a, b, b, initial_state=h)
        assert y.shape == shape and (shape[1] or torch.equal(final, h))
        back = P.selective_scan_backprop(x, x, x, a, b, b, d=w[:, 0].contiguous(), grad_final=h, initial_state=h)
        assert (back[2] == 0).all() and (back[5] == 0).all() and (shape[1] or torch.equal(back[8], h))
    none, at = torch.zeros((0, 4), device=DEV), whole_numbers([0])
    w = torch.ones((4, 2), device=DEV)
    assert P.causal_conv(none, w, offsets=at)[1].shape == (0, 1, 4)
    assert (P.causal_conv_backprop(none, none, w, offsets=at)[1] == 0).all()
    b = torch.zeros((0, 1, 2), device=DEV)
    assert P.selective_scan(none, none, -w, b, b, offsets=at)[1].shape == (0, 4, 2)
    assert (P.selective_scan_backprop(none, none, none, -w, b, b, offsets=at)[2] == 0).all()
    five, b = torch.ones((5, 4), device=DEV), torch.ones((5, 1, 2), device=DEV)          # rows of no sequence
    assert (P.selective_scan_backprop(five, five, five, -w, b, b, offsets=at)[2] == 0).all()
    assert (P.causal_conv_backprop(five, five, w, offsets=at)[1] == 0).all()
    assert P.norm_residual(none, none, w[:, 0].contiguous())[0].shape == (0, 4)
    assert (P.norm_residual_backprop(none, none, w[:, 0].contiguous())[2] == 0).all()
    q, s, _ = P.norm_residual_float8(none, None, w[:, 0].contiguous())
    assert q.shape == (0, 4) and s.shape == (0, 1)
    assert P.causal_conv_step(none, torch.zeros((0, 1, 4), device=DEV), w).shape == (0, 4)
    assert P.selective_scan_step(none, none, -w, torch.zeros((0, 1, 2), device=DEV), torch.zeros((0, 1, 2), device=DEV), torch.zeros((0, 4, 2), device=DEV)).shape == (0, 4)


def raw(fn, *args):
    """A C entry point on the current stream, tensors as their addresses."""
    assert fn(*(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args), torch.cuda.current_stream().cuda_stream) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(300, 24), (3000, 9)])
@pytest.mark.parametrize("offsets,cut", [([7, 100, 100, 290], None), ([-5, 100, 290], [0, 100, 290]), ([20, 100, 1 << 30], [20, 100, -1]),
                                         ([-9, -7, 60, 1 << 30, (1 << 30) + 5], [0, 0, 60, -1, -1])])
def test_layers_leave_other_rows_alone(P, dtype, rows, channels, offsets, cut):
    """Straight calls on buffers that hold a mark: rows of no sequence keep it, sequences are cut to the rows there are, and every sequence has a
    state behind it."""
    from pysiglib_amd import _loader as L
    offsets, n = ([x if x > 1 << 20 or x < 0 else x * rows // 300 for x in offsets]), len(offsets) - 1
    cut = [rows if x == -1 else x * rows // 300 for x in cut] if cut else offsets
    first, past, at = cut[0], cut[-1], whole_numbers(offsets)
    code, inside, part = L.SEQUENCE_DTYPES[str(dtype).split(".")[1]], [c - cut[0] for c in cut], slice(cut[0], cut[-1])
    marked = lambda like: torch.full_like(like, 77.0, memory_format=torch.contiguous_format)          # noqa: E731

    def alone(*tensors):
        for t in tensors:
            assert (t[:first] == 77.0).all() and (t[past:] == 77.0).all()

    rng = np.random.default_rng(rows)
    x, g, w, bias = numbers(rng, rows, channels, dtype=dtype), numbers(rng, rows, channels, dtype=dtype), numbers(rng, channels, 4), numbers(rng, channels)
    state, gf = numbers(rng, n, 3, channels, dtype=dtype), numbers(rng, n, 3, channels, dtype=dtype)
    y, final, dx, d0, dw, db = marked(x), marked(state), marked(x), marked(state), marked(w), marked(bias)
    raw(L.CUSIG_CAUSAL_CONV, code, x, w, bias, state, y, final, at, n, 0, rows, channels, 4, channels, True)
    size = L.CUSIG_CAUSAL_CONV_BACKPROP_WORKSPACE(rows, channels, 4)
    space = torch.zeros(size, dtype=torch.uint8, device=DEV)
    raw(L.CUSIG_CAUSAL_CONV_BACKPROP, code, g, x, w, bias, state, gf, dx, dw, db, d0, at, n, 0, rows, channels, 4, channels, channels, True, space, size)
    want, bound = conv_oracle(f64(x)[part], f64(state), f64(w), f64(bias), inside, True, f64(g)[part], f64(gf))
    for name, got, v, e, kind in zip(("y", "final", "dx", "dw", "db", "d0"), (y[part], final, dx[part], dw, db, d0), want, bound,
                                     (dtype, dtype, dtype, torch.float32, torch.float32, dtype)):
        within(got, v, rounded(v, e, kind), name)
    alone(y, dx)

    t = scan_inputs(dtype, rows, n, channels, 16, 1, seed=rows)
    y, final, grads = marked(t["x"]), marked(t["h0"]), [marked(t[k]) for k in ("x", "delta", "a", "b", "c", "d", "z", "bias", "h0")]
    strides = (channels, channels, channels, 32, 32, 32, 32)
    inputs = [t[k] for k in ("x", "delta", "a", "b", "c", "d", "z", "bias")]
    size = L.CUSIG_SELECTIVE_SCAN_WORKSPACE(True, n, 0, rows, channels, 16, 1)
    space = torch.zeros(max(size, 1), dtype=torch.uint8, device=DEV)
    raw(L.CUSIG_SELECTIVE_SCAN, code, *inputs, t["h0"], y, final, at, n, 0, rows, channels, 16, 1, *strides, True, space, size)
    size = L.CUSIG_SELECTIVE_SCAN_BACKPROP_WORKSPACE(True, n, 0, rows, channels, 16, 1)
    space = torch.zeros(size, dtype=torch.uint8, device=DEV)
    raw(L.CUSIG_SELECTIVE_SCAN_BACKPROP, code, t["g"], *inputs, t["gf"], t["h0"], *grads, at, n, 0, rows, channels, 16, 1, channels, *strides, True, space, size)
    if rows == 300:
        of = {k: f64(t[k])[part] for k in ("x", "delta", "b", "c", "z", "g")}
        want, bound = scan_oracle(of["x"], of["delta"], f64(t["a"]), of["b"], of["c"], f64(t["d"]), of["z"], f64(t["bias"]), f64(t["h0"]), inside, True, of["g"], f64(t["gf"]))
        kinds = (dtype, torch.float32, dtype, dtype, torch.float32, dtype, dtype, torch.float32, dtype, torch.float32, torch.float32)
        for name, got, v, e, kind in zip(NAMES, (y, final, *grads), want, bound, kinds):
            within(got[part] if len(got) == rows else got, v, rounded(v, e, kind), name)
    else:
        inside = whole_numbers(inside)
        args = [t[k][part] if len(t[k]) == rows else t[k] for k in ("x", "delta", "a", "b", "c")]
        one = P.selective_scan(*args, d=t["d"], z=t["z"][part], delta_bias=t["bias"], initial_state=t["h0"], offsets=inside)
        assert torch.isfinite(y[part].float()).all() and (y[part].float() - one[0].float()).abs().max() <= 4 * ROUND[dtype] * one[0].float().abs().max() + 1e-4
    alone(y, grads[0], grads[1], grads[3], grads[4], grads[6])


@pytest.mark.gpu
def test_offsets_that_do_not_ascend_stay_inside(P):
    """They make no sense, and nothing outside the tensors is touched."""
    rng = np.random.default_rng(0)
    x, w = numbers(rng, 500, 20), numbers(rng, 20, 4)
    b = numbers(rng, 500, 1, 16)
    a = -numbers(rng, 20, 16).abs()
    for offsets in ([300, 100, 500, 0], [0, 500, 0, 500], [500, 0, 0, 0], [1 << 30, -1 << 30, 7, 1 << 30], [0, 500, 100, 200, 300, 50, 500, -7]):
        at = whole_numbers(offsets)
        P.causal_conv(x, w, offsets=at)
        P.causal_conv_backprop(x, x, w, offsets=at)
        P.selective_scan(x, x, a, b, b, z=x, offsets=at)
        P.selective_scan_backprop(x, x, x, a, b, b, z=x, offsets=at)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_layers_take_parts_of_projections_and_other_streams(P):
    rng = np.random.default_rng(1)
    t = scan_inputs(torch.bfloat16, 2 * 90, 2, 24, 16, 2, seed=5)
    whole = torch.cat([t["x"], t["z"], t["delta"], t["b"].flatten(1), t["c"].flatten(1), t["g"]], 1).reshape(2, 90, -1)
    x, z, delta, b, c, g = whole.split([24, 24, 24, 32, 32, 24], -1)
    b, c = b.unflatten(-1, (2, 16)), c.unflatten(-1, (2, 16))
    w, weight = numbers(rng, 24, 4), numbers(rng, 24)
    call = lambda x, z, delta, b, c, g: (*P.selective_scan(x, delta, t["a"], b, c, z=z), *P.selective_scan_backprop(g, x, delta, t["a"], b, c, z=z),   # noqa: E731
                                         *P.causal_conv(x, w), *P.causal_conv_backprop(g, x, w), *P.norm_residual(x, z, weight),
                                         *P.norm_residual_backprop(g, x, weight, grad_total=z))
    want = call(*(v.contiguous() for v in (x, z, delta, b, c, g)))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call(x, z, delta, b, c, g)
        turned = [v.transpose(0, 1).contiguous().transpose(0, 1) for v in (x, z, delta, b, c, g)]
        again = call(*turned)
        strided = [torch.stack((v, v), -1)[..., 0] for v in (x, z, delta, b, c, g)]
        last = call(*strided)
    side.synchronize()
    for other in (got, again, last):
        same_bits(want, other)


@pytest.mark.gpu
def test_two_streams_at_once(P):
    """Nothing is shared between calls."""
    t = scan_inputs(torch.bfloat16, 600, 1, 100, 16, 1, seed=6)
    args = [t[k] for k in ("x", "delta", "a", "b", "c")]
    w = torch.ones((100, 4), device=DEV)
    call = lambda: (*P.selective_scan(*args, z=t["z"], offsets=whole), *P.selective_scan_backprop(t["g"], *args, z=t["z"], offsets=whole),        # noqa: E731
                    *P.causal_conv_backprop(t["g"], t["x"], w, offsets=whole), *P.norm_residual_backprop(t["g"], t["x"], w[:, 0].contiguous()))
    whole = whole_numbers([0, 200, 600])
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for s, kept in zip(streams, got):
            with torch.cuda.stream(s):
                kept.append(call())
    torch.cuda.synchronize()
    for kept in got:
        for one in kept:
            same_bits(want, one)


@pytest.mark.gpu
def test_autograd_gives_the_gradients(P):
    A = P.torch_api
    t = scan_inputs(torch.float16, 177, 4, 20, 16, 2, seed=1)
    starts = [0, 40, 47, 47, 177]
    at = whole_numbers(starts)
    names = ("x", "delta", "a", "b", "c", "d", "z", "bias", "h0")
    leaf = {k: t[k].clone().requires_grad_(True) for k in names}
    y, final = A.selective_scan(leaf["x"], leaf["delta"], leaf["a"], leaf["b"], leaf["c"], d=leaf["d"], z=leaf["z"], delta_bias=leaf["bias"],
                                initial_state=leaf["h0"], offsets=at)
    torch.autograd.backward([y, final], [t["g"], t["gf"]])
    args, options = [t[k] for k in ("x", "delta", "a", "b", "c")], dict(d=t["d"], z=t["z"], delta_bias=t["bias"], initial_state=t["h0"], offsets=at)
    want = P.selective_scan_backprop(t["g"], *args, grad_final=t["gf"], **options)
    for k, g in zip(names, want):
        assert torch.equal(leaf[k].grad, g), k
    # the last states alone, and few of the inputs
    one = t["x"].clone().requires_grad_(True)
    A.selective_scan(one, *args[1:], offsets=at)[1].sum().backward()
    assert torch.equal(one.grad, P.selective_scan_backprop(torch.zeros_like(t["x"]), *args, grad_final=torch.ones_like(t["h0"]), offsets=at)[0])
    rng = np.random.default_rng(0)
    w, bias, state, gs = numbers(rng, 20, 4), numbers(rng, 20), numbers(rng, 4, 3, 20, dtype=torch.float16), numbers(rng, 4, 3, 20, dtype=torch.float16)
    leaves = [v.clone().requires_grad_(True) for v in (t["x"], w, bias, state)]
    out = A.causal_conv(*leaves[:3], initial_state=leaves[3], offsets=at, silu=False)
    torch.autograd.backward(out, [t["g"], gs])
    for v, g in zip(leaves, P.causal_conv_backprop(t["g"], t["x"], w, bias, grad_final=gs, initial_state=state, offsets=at, silu=False)):
        assert torch.equal(v.grad, g)
    weight = numbers(rng, 20)
    for kind in (torch.float16, torch.float32):
        r, gt = t["z"].to(kind), t["delta"].to(kind)
        leaves = [v.clone().requires_grad_(True) for v in (t["x"], r, weight)]
        out, total = A.norm_residual(*leaves, eps=1e-3)
        torch.autograd.backward([out, total], [t["g"], gt])
        for v, g in zip(leaves, P.norm_residual_backprop(t["g"], total.detach(), weight, grad_total=gt, eps=1e-3)):
            assert torch.equal(v.grad, g)
        leaves = [v.clone().requires_grad_(True) for v in (t["x"], r, weight)]
        A.norm_residual(*leaves)[1].sum().backward()
        assert (leaves[0].grad == 1).all() and (leaves[1].grad == 1).all() and (leaves[2].grad == 0).all()
    leaves = [v.clone().requires_grad_(True) for v in (t["x"], weight)]
    out, total = A.norm_residual(leaves[0], None, leaves[1])
    assert total is leaves[0]
    torch.autograd.backward([out, total], [t["g"], t["z"]])
    dx, _, dw = P.norm_residual_backprop(t["g"], t["x"], weight)
    assert torch.equal(leaves[1].grad, dw) and torch.equal(leaves[0].grad, dx + t["z"])


@pytest.mark.gpu
def test_second_derivatives_are_refused(P):
    A = P.torch_api
    x, w = torch.randn((2, 6, 8), device=DEV, requires_grad=True), torch.randn((8, 4), device=DEV)
    b = torch.randn((2, 6, 1, 4), device=DEV)
    for out in (A.causal_conv(x, w)[0], A.selective_scan(x, x, -w.abs(), b, b)[0], A.norm_residual(x, x.detach(), w[:, 0].contiguous())[0]):
        grad, = torch.autograd.grad(out.square().sum(), x, create_graph=True, retain_graph=True)
        with pytest.raises(RuntimeError):
            (grad.sum() + x.sum()).backward()


@pytest.mark.gpu
def test_a_captured_graph_replays(P):
    """A training pass and a serving step: every replay gives what the same calls give outside the graph."""
    t = scan_inputs(torch.bfloat16, 400, 2, 64, 16, 1, seed=3)
    offsets, w, weight = whole_numbers([0, 130, 400]), torch.randn((64, 4), device=DEV), torch.randn(64, device=DEV)
    state, rows = torch.zeros((2, 64, 16), device=DEV), torch.zeros((2, 3, 64), dtype=torch.bfloat16, device=DEV)

    def step():
        out, total = P.norm_residual(t["x"], t["z"], weight)
        v, _ = P.causal_conv(out, w, offsets=offsets)
        y, final = P.selective_scan(v, t["delta"], t["a"], t["b"], t["c"], z=t["z"], initial_state=t["h0"], offsets=offsets)
        back = P.selective_scan_backprop(t["g"], v, t["delta"], t["a"], t["b"], t["c"], z=t["z"], initial_state=t["h0"], offsets=offsets)
        dv = P.causal_conv_backprop(back[0], out, w, offsets=offsets)
        dn = P.norm_residual_backprop(dv[0], total, weight)
        q = P.norm_residual_float8(t["x"], t["z"], weight)
        one = P.causal_conv_step(t["x"][:2], rows, w)
        two = P.selective_scan_step(one, t["delta"][:2], t["a"], t["b"][:2], t["c"][:2], state)
        return [v for v in (out, total, v, y, final, *back, *dv, *dn, *q, one, two, rows.clone(), state.clone()) if v is not None]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for turn in range(4):
        t["x"].copy_(torch.randn_like(t["x"]))
        offsets.copy_(whole_numbers([0, 100 + 70 * turn, 400 - turn]))
        for v in captured:
            v.view(torch.uint8).zero_()
        state.fill_(0.5)
        rows.fill_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in captured]
        state.fill_(0.5)
        rows.fill_(0.25)
        want = step()
        inside = 400 - turn
        for a, b in zip(got, want):
            if a.dim() and a.shape[0] == 400:
                a, b = a[:inside], b[:inside]
            # rows behind the last sequence are not written: what the norm makes of them is left out
            if a.shape != (64,):
                same_bits([a], [b])


@pytest.mark.gpu
def test_a_block_run_together(P):
    """A residual block of norm, projection, convolution, scan and projection: trained a step through autograd against the same block of plain
    64-bit operations, then run a token at a time with its states."""
    A, gen = P.torch_api, torch.Generator().manual_seed(0)
    width, inner, states, lengths = 48, 96, 16, [70, 1, 129]
    starts = starts_of(lengths)
    make = lambda *s, size=1.0: (size * torch.randn(s, generator=gen, dtype=torch.float64)).float().double()           # noqa: E731
    p = dict(norm=1 + make(width, size=0.1), enter=make(2 * inner, width, size=width ** -0.5), taps=make(inner, 4, size=0.5), bias=make(inner, size=0.1),
             mix=make(inner + 2 * states, inner, size=inner ** -0.5), delta_bias=make(inner, size=0.5) - 3, d=1 + make(inner, size=0.1),
             a=-torch.exp(make(inner, states, size=0.5)), leave=make(width, inner, size=inner ** -0.5))
    x, residual, g = make(200, width), make(200, width), make(200, width)

    def block(p, x, residual, norm, conv, scan):
        out, total = norm(x, residual, p["norm"])
        v, z = torch.nn.functional.linear(out, p["enter"]).chunk(2, -1)
        v = conv(v, p["taps"], p["bias"])
        delta, b, c = torch.nn.functional.linear(v, p["mix"]).split([inner, states, states], -1)
        return total + torch.nn.functional.linear(scan(v, delta, p["a"], b[:, None], c[:, None], p["d"], z, p["delta_bias"]), p["leave"])

    def plain_norm(x, r, w):
        t = x + r
        return t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w, t

    def plain_conv(v, w, bias):
        out = []
        for s, e in zip(starts, starts[1:]):
            rows = torch.cat((v.new_zeros(3, inner), v[s:e]))
            out.append((rows.unfold(0, 4, 1) * w).sum(-1) + bias)
        return torch.nn.functional.silu(torch.cat(out))

    def plain_scan(x, delta, a, b, c, d, z, bias):
        dt, ys = torch.nn.functional.softplus(delta + bias), []
        for s, e in zip(starts, starts[1:]):
            h = 0
            for t in range(s, e):
                h = torch.exp(dt[t][:, None] * a) * h + (dt[t] * x[t])[:, None] * b[t]
                ys.append((h * c[t]).sum(-1) + d * x[t])
        return torch.stack(ys) * torch.nn.functional.silu(z)

    leaves = {k: v.clone().requires_grad_(True) for k, v in p.items()}
    inputs = [x.clone().requires_grad_(True), residual.clone().requires_grad_(True)]
    want = block(leaves, *inputs, plain_norm, plain_conv, plain_scan)
    want.backward(g)
    at = whole_numbers(starts)
    mine = {k: v.float().to(DEV).requires_grad_(True) for k, v in p.items()}
    own = [v.float().to(DEV).requires_grad_(True) for v in (x, residual)]
    got = block(mine, *own, lambda x, r, w: A.norm_residual(x, r, w), lambda v, w, bias: A.causal_conv(v, w, bias, offsets=at)[0],
                lambda x, delta, a, b, c, d, z, bias: A.selective_scan(x, delta, a, b, c, d=d, z=z, delta_bias=bias, offsets=at)[0])
    got.backward(g.float().to(DEV))
    # products of up to 128 terms one behind the other, some 40 roundings in each layer: well below 2^-24 times a thousand of the largest
    near = lambda u, v: float((u.double().cpu() - v).abs().max()) <= 1024 * U32 * float(v.abs().max())          # noqa: E731
    assert near(got.detach(), want.detach())
    for k in p:
        assert near(mine[k].grad, leaves[k].grad), k
    for u, v in zip(own, inputs):
        assert near(u.grad, v.grad)
    # one token after the other, the three sequences side by side
    with torch.no_grad():
        w = {k: v.detach() for k, v in mine.items()}
        rows, state = torch.zeros((3, 3, inner), device=DEV), torch.zeros((3, inner, states), device=DEV)
        for t in range(max(lengths)):
            now = torch.tensor([s + min(t, n - 1) for s, n in zip(starts, lengths)], device=DEV)
            y = block(w, own[0][now], own[1][now], lambda x, r, w: P.norm_residual(x, r, w), lambda v, w, bias: P.causal_conv_step(v, rows, w, bias),
                      lambda x, delta, a, b, c, d, z, bias: P.selective_scan_step(x, delta, a, b, c, state, d=d, z=z, delta_bias=bias))
            for i, n in enumerate(lengths):
                if t < n:
                    assert float((y[i].double().cpu() - want[starts[i] + t].detach()).abs().max()) <= 1024 * U32 * float(want.detach().abs().max())


@pytest.mark.gpu
def test_gradients_of_shared_inputs_where_there_are_no_channels(P):
    at = whole_numbers([1, 4])
    for dtype in TYPES:
        x, b = torch.zeros((5, 0), dtype=dtype, device=DEV), torch.ones((5, 2, 3), dtype=dtype, device=DEV)
        a = torch.zeros((0, 3), device=DEV)
        for offsets, first, past in ((None, 0, 5), (at, 1, 4)):
            back = P.selective_scan_backprop(x, x, x, a, b, b, offsets=offsets)
            assert (back[3][first:past] == 0).all() and (back[4][first:past] == 0).all()
    b = torch.full((5, 2, 3), 7.0, device=DEV)
    from pysiglib_amd import _loader as L
    raw(L.CUSIG_SELECTIVE_SCAN_BACKPROP, 0, x, x, x, a, b, b, 0, 0, 0, 0, 0, x, x, a, b, b, 0, 0, 0, x, at, 1, 0, 5, 0, 3, 2, 0, 0, 0, 0, 6, 3, 6, 3, True, 0, 0)
    assert (b[1:4] == 0).all() and (b[0] == 7).all() and (b[4] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [40, 2000])
def test_norm_residual_in_8_bits_of_outputs_whose_scale_is_zero(P, channels):
    """max |out| / 448 of less than half of 2^-149 is zero in 32 bits: the scale is 1, and the outputs, far below 2^-10, are zero."""
    x = torch.ones((2, channels), device=DEV)
    q, scales, _ = P.norm_residual_float8(x, None, torch.full((channels,), 2.0 ** -142, device=DEV), eps=0.0)
    assert (scales == 1).all() and (q.float() == 0).all()


@pytest.mark.gpu
def test_weights_of_very_many_channels(P):
    """Sums over the rows for more columns than one launch has threads for."""
    channels = 1 << 25
    x = torch.ones((2, channels), dtype=torch.bfloat16, device=DEV)
    dw = P.causal_conv_backprop(x, x, torch.zeros((channels, 4), device=DEV), torch.zeros(channels, device=DEV), silu=False)[1:3]
    # two rows: the last tap saw both, the one before it the first
    assert (dw[0] == torch.tensor([0.0, 0.0, 1.0, 2.0], device=DEV)).all() and (dw[1] == 2).all()
    del dw, x
    channels, states = 1 << 22, 32
    x = torch.ones((1, channels), dtype=torch.bfloat16, device=DEV)
    one = torch.ones((1, 1, states), dtype=torch.bfloat16, device=DEV)
    h = torch.ones((channels, states), device=DEV)
    # one row, a = 0, dt = 1: da = h c dt, the gradient of d is x's product with g
    back = P.selective_scan_backprop(x, x, x, torch.zeros_like(h), one, one, d=torch.zeros(channels, device=DEV), softplus=False, initial_state=h)
    assert (back[2] == 1).all() and (back[5] == 1).all()


@pytest.mark.gpu
def test_tensors_of_more_than_32_bits_of_elements(P):
    """A long sequence of zeros, and behind it a short one that starts beyond 2^31 elements: as alone."""
    channels, rows, last = 8192, 270000, 50
    assert (rows - last) * channels > 1 << 31
    kind = torch.bfloat16
    rng = np.random.default_rng(0)
    small = {k: numbers(rng, last, channels, dtype=kind) for k in ("x", "delta", "z", "g")}
    big = {}
    for k, v in small.items():
        big[k] = torch.zeros((rows, channels), dtype=kind, device=DEV)
        big[k][-last:] = v
    at, alone = whole_numbers([0, rows - last, rows]), whole_numbers([0, last])
    w, bias = numbers(rng, channels, 4), numbers(rng, channels)
    y, final = P.causal_conv(big["x"], w, bias, offsets=at)
    want, end = P.causal_conv(small["x"], w, bias, offsets=alone)
    assert torch.equal(y[-last:], want) and torch.equal(final[1:], end)
    dx = P.causal_conv_backprop(big["g"], big["x"], w, bias, offsets=at)[0]
    assert torch.equal(dx[-last:], P.causal_conv_backprop(small["g"], small["x"], w, bias, offsets=alone)[0])
    del y, dx
    out, total = P.norm_residual(big["x"], big["z"], bias)
    want, sums = P.norm_residual(small["x"], small["z"], bias)
    assert torch.equal(total[-last:], sums)
    assert (out[-last:].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()         # another split of a row: a step of the output
    del out
    dx = P.norm_residual_backprop(big["g"], total, bias)[0]
    want = P.norm_residual_backprop(small["g"], sums, bias)[0]
    assert (dx[-last:].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
    del dx, total
    states = 4
    a, d = -numbers(rng, channels, states).abs(), numbers(rng, channels)
    b = torch.zeros((rows, 1, states), dtype=kind, device=DEV)
    b[-last:] = numbers(rng, last, 1, states, dtype=kind)
    some = b[-last:].clone()
    y, final = P.selective_scan(big["x"], big["delta"], a, b, b, d=d, z=big["z"], offsets=at)
    want, end = P.selective_scan(small["x"], small["delta"], a, some, some, d=d, z=small["z"], offsets=alone)
    # the segments may be others: a state is then a sum in another order, far below a step of bfloat16
    assert (y[-last:].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
    assert (final[1] - end[0]).abs().max() <= 2.0 ** -16 * end.abs().max() and (final[0] == 0).all()
    del y
    back = P.selective_scan_backprop(big["g"], big["x"], big["delta"], a, b, b, d=d, z=big["z"], offsets=at)
    want = P.selective_scan_backprop(small["g"], small["x"], small["delta"], a, some, some, d=d, z=small["z"], offsets=alone)
    for i in (0, 1, 3, 4, 6):
        assert (back[i][-last:].float() - want[i].float()).abs().max() <= 2.0 ** -7 * want[i].float().abs().max(), i
    for i in (2, 5):            # the zeros add nothing
        assert (back[i] - want[i]).abs().max() <= 2.0 ** -14 * want[i].abs().max(), i


@pytest.mark.gpu
def test_gradients_of_two_inputs_are_two_tensors(P):
    x, r = (torch.randn((3, 40), device=DEV, requires_grad=True) for _ in range(2))
    w = torch.ones(40, device=DEV)
    for _ in range(2):
        P.torch_api.norm_residual(x, r, w)[0].square().sum().backward()
    want = r.grad.clone()
    assert torch.equal(x.grad, want)
    x.grad.add_(1.0)
    assert torch.equal(r.grad, want)


# ---- refusals ----

@pytest.mark.gpu
def test_refusals(P):
    x, w = torch.zeros((2, 3, 4), device=DEV), torch.ones((4, 2), device=DEV)
    v = torch.ones(4, device=DEV)
    state = torch.zeros((2, 1, 4), device=DEV)
    at = whole_numbers([0, 3])
    for args, options in [((x, w[:3]), {}), ((x, w, v[:3]), {}), ((x[0, 0], w), {}), ((x, torch.ones((4, 9), device=DEV)), {}), ((x, torch.ones((4, 0), device=DEV)), {}),
                          ((x, w), dict(initial_state=state[:1])), ((x, w), dict(offsets=at)), ((x, v), {}), ((x, w.cpu()), {})]:
        with pytest.raises(ValueError):
            P.causal_conv(*args, **options)
    for args, options in [((x.double(), w), {}), ((x, w.half()), {}), ((x, w, v.half()), {}), ((x, w), dict(initial_state=state.half())), ((x, w), dict(silu=1)),
                          ((x[0], w), dict(offsets=at.long()))]:
        with pytest.raises(TypeError):
            P.causal_conv(*args, **options)
    with pytest.raises(ValueError):
        P.causal_conv_backprop(x[:1], x, w)
    with pytest.raises(TypeError):
        P.causal_conv_backprop(x.half(), x, w)
    with pytest.raises(ValueError):
        P.causal_conv_step(x[:, 0], torch.zeros((2, 1, 8), device=DEV)[..., ::2], w)
    with pytest.raises(ValueError):
        P.causal_conv_step(x[:, 0], state[:1], w)
    with pytest.raises(TypeError):
        P.causal_conv_step(x[:, 0], state.half(), w)
    a, b, h = -torch.ones((4, 5), device=DEV), torch.zeros((2, 3, 2, 5), device=DEV), torch.zeros((2, 4, 5), device=DEV)
    assert P.selective_scan(x, x, a, b, b)[0].shape == x.shape
    for args, options in [((x, x[:1], a, b, b), {}), ((x, x, a[:3], b, b), {}), ((x, x, a, b[:1], b), {}), ((x, x, a, b, b[..., :4]), {}), ((x, x, a, b[:, :, 0], b), {}),
                          ((x, x, torch.ones((4, 65), device=DEV), b, b), {}), ((x, x, torch.ones((4, 0), device=DEV), b[..., :0], b[..., :0]), {}),
                          ((x[..., :3], x[..., :3], a[:3], b, b), {}), ((x, x, a, b, b), dict(z=x[:1])), ((x, x, a, b, b), dict(d=v[:3])),
                          ((x, x, a, b, b), dict(delta_bias=v[:3])), ((x, x, a, b, b), dict(initial_state=h[:1])), ((x, x, a, b, b), dict(offsets=at)),
                          ((x[0, 0], x[0, 0], a, b[0, 0], b[0, 0]), {}), ((x, x, a, b[:, :, :0], b[:, :, :0]), {}), ((x, x, a.cpu(), b, b), {})]:
        with pytest.raises(ValueError):
            P.selective_scan(*args, **options)
    for args, options in [((x, x.half(), a, b, b), {}), ((x, x, a.half(), b, b), {}), ((x, x, a, b.half(), b), {}), ((x, x, a, b, b), dict(z=x.half())),
                          ((x, x, a, b, b), dict(softplus=1)), ((x, x, a, b, b), dict(initial_state=h.half())), ((x.double(), x, a, b, b), {})]:
        with pytest.raises(TypeError):
            P.selective_scan(*args, **options)
    with pytest.raises(ValueError):
        P.selective_scan_backprop(x[:1], x, x, a, b, b)
    with pytest.raises(ValueError):
        P.selective_scan_backprop(x, x, x, a, b, b, grad_final=h[:1])
    with pytest.raises(ValueError):
        P.selective_scan_step(x[:, 0], x[:, 0], a, b[:, 0], b[:, 0], torch.zeros((2, 5, 4), device=DEV).transpose(1, 2))
    with pytest.raises(TypeError):
        P.selective_scan_step(x[:, 0], x[:, 0], a, b[:, 0], b[:, 0], h.half())
    for args in [(x, x[:1], v), (x, None, v[:3]), (torch.zeros((1, 16385), device=DEV), None, torch.ones(16385, device=DEV)), (x[..., :0], None, v[:0])]:
        with pytest.raises(ValueError):
            P.norm_residual(*args)
        with pytest.raises(ValueError):
            P.norm_residual_float8(*args)
    for args in [(x, x.half(), v), (x.half(), x.bfloat16(), v), (x, None, v.half()), (x, np.zeros((2, 3, 4)), v), (x.double(), None, v)]:
        with pytest.raises(TypeError):
            P.norm_residual(*args)
    with pytest.raises(ValueError):
        P.norm_residual_backprop(x, x, v, grad_total=x[:1])
    with pytest.raises(TypeError):
        P.norm_residual_backprop(x.half(), x, v, grad_total=x.half())
    with pytest.raises(ValueError):
        P.norm_residual_backprop(x, x[:1], v)
    with pytest.raises(TypeError):
        P.norm_residual_backprop(x, None, v)


def test_refuses_host_tensors(P):
    x, w = torch.zeros((2, 3, 4)), torch.ones((4, 2))
    with pytest.raises(RuntimeError):
        P.causal_conv(x, w)
    with pytest.raises(RuntimeError):
        P.selective_scan(x, x, w, x[..., None, :2], x[..., None, :2])
    with pytest.raises(RuntimeError):
        P.norm_residual(x, None, w[:, 0].contiguous())
    with pytest.raises(TypeError):
        P.norm_residual(None, None, w)
    with pytest.raises(TypeError):
        P.causal_conv(None, w)
    with pytest.raises(TypeError):
        P.selective_scan(None, x, w, x, x)


def test_the_entry_points_report_what_is_wrong(P):
    """Sizes that do not fit are refused on the host, before any launch."""
    from pysiglib_amd import _loader as L
    at, s7 = 256, (4,) * 7
    forward = lambda dtype=1, n=2, length=3, rows=6, channels=4, states=2, groups=1, y=at, a=at: L.CUSIG_SELECTIVE_SCAN(         # noqa: E731
        dtype, at, at, a, at, at, 0, 0, 0, 0, y, at, 0, n, length, rows, channels, states, groups, *s7, True, 0, 0, 0)
    for bad in (dict(rows=7), dict(states=65), dict(states=0), dict(groups=3), dict(groups=0), dict(dtype=3), dict(y=0), dict(a=0), dict(rows=1 << 31, length=1 << 30),
                dict(channels=1 << 24)):
        assert forward(**bad) == 2 and L.last_error_message(), bad
    # one sequence of 4000 rows is cut: scratch of the right size and alignment
    size = L.CUSIG_SELECTIVE_SCAN_WORKSPACE(False, 1, 4000, 4000, 4, 2, 1)
    assert size > 0
    for space, bytes_ in ((0, size), (256, size - 1), (8, size)):
        assert L.CUSIG_SELECTIVE_SCAN(1, at, at, at, at, at, 0, 0, 0, 0, at, at, 0, 1, 4000, 4000, 4, 2, 1, *s7, True, space, bytes_, 0) == 2
    size = L.CUSIG_SELECTIVE_SCAN_BACKPROP_WORKSPACE(False, 1, 40, 40, 4, 2, 1)
    back = lambda z=0, dz=0, d=0, dd=0, space=256, bytes_=size, dx=at: L.CUSIG_SELECTIVE_SCAN_BACKPROP(       # noqa: E731
        1, at, at, at, at, at, at, d, z, 0, 0, 0, dx, at, at, at, at, dd, dz, 0, at, 0, 1, 40, 40, 4, 2, 1, 4, *s7, True, space, bytes_, 0)
    for bad in (dict(z=at), dict(d=at), dict(space=0), dict(bytes_=size - 1), dict(space=8), dict(dx=0)):
        assert back(**bad) == 2, bad
    assert L.CUSIG_SELECTIVE_SCAN_STEP(1, at, at, at, at, at, 0, 0, 0, 0, at, 2, 4, 2, 1, *s7, True, 0) == 2
    conv = lambda width=4, rows=6, w=at, final=at, dtype=1: L.CUSIG_CAUSAL_CONV(dtype, at, w, 0, 0, at, final, 0, 2, 3, rows, 4, width, 4, True, 0)        # noqa: E731
    for bad in (dict(width=0), dict(width=9), dict(rows=5), dict(w=0), dict(final=0), dict(dtype=7)):
        assert conv(**bad) == 2, bad
    size = L.CUSIG_CAUSAL_CONV_BACKPROP_WORKSPACE(6, 4, 4)
    for space, bytes_ in ((0, size), (256, size - 1), (8, size)):
        assert L.CUSIG_CAUSAL_CONV_BACKPROP(1, at, at, at, 0, 0, 0, at, at, 0, at, 0, 2, 3, 6, 4, 4, 4, 4, True, space, bytes_, 0) == 2
    assert L.CUSIG_CAUSAL_CONV_BACKPROP(1, at, at, at, 0, 0, 0, at, 0, 0, at, 0, 2, 3, 6, 4, 4, 4, 4, True, 256, size, 0) == 2
    assert L.CUSIG_CAUSAL_CONV_STEP(1, at, 0, at, 0, at, 2, 4, 4, 4, True, 0) == 2
    norm = lambda dtype=1, other=1, channels=8, residual=0, total=0, w=at: L.CUSIG_NORM_RESIDUAL(dtype, other, at, residual, w, at, total, 0, 2, channels, 8, 8, 1e-6, 0)  # noqa: E731
    for bad in (dict(other=2), dict(dtype=0, other=1), dict(channels=16385), dict(channels=0), dict(residual=at), dict(w=0), dict(dtype=9, other=9)):
        assert norm(**bad) == 2, bad
    size = L.CUSIG_NORM_RESIDUAL_BACKPROP_WORKSPACE(8)
    for space, bytes_, dw, other, dr in ((0, size, at, 1, 0), (256, size - 1, at, 1, 0), (8, size, at, 1, 0), (256, size, 0, 1, 0), (256, size, at, 0, 0)):
        assert L.CUSIG_NORM_RESIDUAL_BACKPROP(1, other, at, 0, at, at, at, dr, dw, 2, 8, 8, 8, 8, 1e-6, space, bytes_, 0) == 2


def test_the_entry_points_refuse_sizes_beyond_their_numbers(P):
    from pysiglib_amd import _loader as L
    at = 256
    assert L.CUSIG_SELECTIVE_SCAN_WORKSPACE(False, 1, 5, 5, 0, 2, 1 << 32) == 0
    assert L.CUSIG_SELECTIVE_SCAN_BACKPROP_WORKSPACE(False, 1, 5, 5, 0, 2, 1 << 32) == 0
    # 2^30 sequences of 2^34 rows: the product is zero in 64 bits
    n, length = 1 << 30, 1 << 34
    assert L.CUSIG_SELECTIVE_SCAN(1, at, at, at, at, at, 0, 0, 0, 0, at, at, 0, n, length, 0, 4, 2, 1, *(4,) * 7, True, at, 1 << 62, 0) == 2
    assert L.CUSIG_SELECTIVE_SCAN_BACKPROP(1, at, at, at, at, at, at, 0, 0, 0, 0, 0, at, at, at, at, at, 0, 0, 0, at, 0, n, length, 0, 4, 2, 1, 4, *(4,) * 7, True, at,
                                           1 << 62, 0) == 2
    assert L.CUSIG_CAUSAL_CONV(1, at, at, 0, 0, at, at, 0, n, length, 0, 4, 4, 4, True, 0) == 2
    # distances of rows that 32 bits do not hold 16 times
    for i in range(3):
        for stride in (-4, (1 << 24) + 1):
            strides = [4] * 7
            strides[i] = stride
            assert L.CUSIG_SELECTIVE_SCAN(1, at, at, at, at, at, 0, at, 0, 0, at, at, 0, 2, 3, 6, 4, 2, 1, *strides, True, at, 1 << 40, 0) == 2
            assert L.CUSIG_SELECTIVE_SCAN_BACKPROP(1, at, at, at, at, at, at, 0, at, 0, 0, 0, at, at, at, at, at, 0, at, 0, at, 0, 2, 3, 6, 4, 2, 1, 4, *strides, True, at,
                                                   1 << 40, 0) == 2
    for stride in (-4, (1 << 24) + 1):
        assert L.CUSIG_SELECTIVE_SCAN_BACKPROP(1, at, at, at, at, at, at, 0, 0, 0, 0, 0, at, at, at, at, at, 0, 0, 0, at, 0, 2, 3, 6, 4, 2, 1, stride, *(4,) * 7, True, at,
                                               1 << 40, 0) == 2
