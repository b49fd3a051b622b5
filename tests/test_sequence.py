"""The layers of a sequence model (pysiglib_amd/sequence.py) against their formulas in 64 bits, written out step by step in
NumPy, and their gradients also against differences of those.

Tolerances follow from the number formats.  u = 2^-24, 2^-8, 2^-11 is the largest relative rounding error of float32,
bfloat16 and float16; an output rounded once is off by u times its size.  What 32-bit sums add is bounded for each operator
where it is used."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

DEV = "cuda:0"
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# float16 values below the normal numbers are spaced evenly
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


# ---- the recurrence ----

def recurrence_oracle(x, g, h0, starts, grad=None, grad_final=None, h=None):
    """Step by step in 64 bits over packed rows.  Returns the outputs and, for each, a bound of what 32-bit steps may add:
    a step rounds the decay (relative error (4 + |2 g|) u: the argument's product and the exponential) and the sum, so
    E_t = a_t E_{t-1} + (8 + 2 |g_t|) u M_t, with M the recurrence of the sizes; composing runs of steps adds roundings of
    the same products, at most as many again."""
    rows, channels = x.shape
    a = np.exp(g)
    out, err = np.zeros_like(x), np.zeros_like(x)
    final = h0.copy()
    final_err = np.zeros_like(h0)
    for i in range(len(starts) - 1):
        s, m, e = h0[i].copy(), np.abs(h0[i]), np.zeros(channels)
        for t in range(starts[i], starts[i + 1]):
            s = a[t] * s + x[t]
            m = a[t] * m + np.abs(x[t])
            step = 2 * U32 * (8 + 2 * np.abs(np.where(np.isfinite(g[t]), g[t], 0.0))) * m
            e = a[t] * e + step
            out[t], err[t] = s, e
        final[i], final_err[i] = s, e
    if grad is None:
        return (out, final), (err, final_err)
    prev = np.concatenate((np.zeros((1, channels)), h[:-1])) if rows else h
    dx, dg, d0 = np.zeros_like(x), np.zeros_like(x), grad_final.copy()
    ex, eg, e0 = np.zeros_like(x), np.zeros_like(x), np.zeros_like(h0)
    for i in range(len(starts) - 1):
        c, m, e = grad_final[i].copy(), np.abs(grad_final[i]), np.zeros(channels)
        for t in range(starts[i + 1] - 1, starts[i] - 1, -1):
            before = h0[i] if t == starts[i] else prev[t]
            dx[t], ex[t] = grad[t] + c, e + U32 * (m + np.abs(grad[t]))
            m = a[t] * (m + np.abs(grad[t]))
            c = a[t] * (c + grad[t])
            e = a[t] * e + 2 * U32 * (8 + 2 * np.abs(np.where(np.isfinite(g[t]), g[t], 0.0))) * m
            dg[t], eg[t] = c * before, (e + 2 * U32 * np.abs(c)) * np.abs(before)
        d0[i], e0[i] = c, e
    return (out, final, dx, dg, d0), (err, final_err, ex, eg, e0)


def recurrence_inputs(dtype, rows, channels, n, seed, low=-2.0):
    rng = np.random.default_rng(seed)
    rate = np.exp(rng.uniform(-6, 1, channels))
    g = np.maximum(-rate * rng.exponential(size=(rows, 1)), low * 10)
    x, grad = rng.standard_normal((rows, channels)), rng.standard_normal((rows, channels))
    make = lambda v: torch.tensor(v, dtype=torch.float64).to(dtype)                      # noqa: E731
    single = lambda: torch.tensor(rng.standard_normal((n, channels)), dtype=torch.float32)   # noqa: E731
    return make(x), make(g), single(), make(grad), single()


def check_recurrence(P, x, g, h0, grad, grad_final, starts, shape=None, offsets=None, with_states=True):
    """shape: of the batched call, or None with offsets."""
    dtype = x.dtype
    put = lambda t: t.to(DEV).reshape(shape) if shape else t.to(DEV)                     # noqa: E731
    state = lambda t: t.to(DEV).reshape(*shape[:-2], shape[-1]) if shape else t.to(DEV)  # noqa: E731
    options = dict(offsets=None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=DEV))
    if with_states:
        options["initial_state"] = state(h0)
    else:
        h0, grad_final = torch.zeros_like(h0), torch.zeros_like(grad_final)
    h, final = P.linear_recurrence(put(x), put(g), **options)
    back = P.linear_recurrence_backprop(h, put(g), put(grad), grad_final=state(grad_final) if with_states else None, **options)
    again = P.linear_recurrence(put(x), put(g), **options), P.linear_recurrence_backprop(
        h, put(g), put(grad), grad_final=state(grad_final) if with_states else None, **options)
    for one, two in zip((h, final, *back), (*again[0], *again[1])):
        assert torch.equal(one.nan_to_num(), two.nan_to_num()), "the same inputs give the same bits"
    want, bound = recurrence_oracle(f64(x), f64(g), f64(h0), starts, f64(grad), f64(grad_final), f64(h).reshape(x.shape))
    u = ROUND[dtype]
    for name, got, w, b in zip(("h", "final", "dx", "dg", "d0"), (h, final, *back), want, bound):
        rounded = (u if name in ("h", "dx", "dg") else U32) * (np.abs(w) + b) + SMALL[dtype if name in ("h", "dx", "dg") else torch.float32]
        within(got.reshape(w.shape), w, b + rounded, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,length,channels", [(1, 1, 1), (3, 1, 5), (2, 129, 33), (1, 700, 130), (5, 17, 16), (2, 300, 67),
                                                   (1, 9000, 9), (1, 6000, 70)])
def test_recurrence_batched(P, dtype, batch, length, channels):
    inputs = recurrence_inputs(dtype, batch * length, channels, batch, seed=length)
    check_recurrence(P, *inputs, [i * length for i in range(batch + 1)], shape=(batch, length, channels))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,channels", [([1], 3), ([0, 5, 0, 0, 1, 130, 0], 40), ([400, 1, 1, 1, 126, 2, 128, 129], 133),
                                              ([7] * 300, 5), ([1] * 1500, 3), ([0, 0], 4),
                                              ([3000, 0, 2500, 0], 40), ([5000], 2)])
@pytest.mark.parametrize("with_states", [True, False])
def test_recurrence_packed(P, dtype, lengths, channels, with_states):
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    inputs = recurrence_inputs(dtype, starts[-1], channels, len(lengths), seed=len(lengths))
    check_recurrence(P, *inputs, starts, offsets=starts, with_states=with_states)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_recurrence_decays_at_the_ends_of_their_range(P, dtype):
    """-inf forgets the state (also one that is infinite, in the chunks behind it), 0 keeps it, growth keeps a zero state."""
    rows, channels = 700, 20
    x, g, h0, grad, gf = recurrence_inputs(dtype, rows, channels, 1, seed=3)
    g[:, 0] = 0.0
    g[::7, 1] = -float("inf")
    g[:, 2] = -float("inf")
    g[:, 3], x[:, 3], h0[:, 3] = 1.0, 0.0, 0.0
    x[650:, 3] = 1e-3
    g[650:, 3] = 0.0
    grad[:, 3], gf[:, 3] = 0.0, 0.0
    g[:, 4] = -60.0
    check_recurrence(P, x, g, h0, grad, gf, [0, rows], shape=(1, rows, channels))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(1, 1), (3, 7), (64, 256), (5, 1030)])
def test_recurrence_step_follows_the_scan(P, dtype, rows, channels):
    x, g, h0, _, _ = recurrence_inputs(dtype, rows * 3, channels, rows, seed=rows)
    both = torch.cat((x, g), 1).to(DEV).reshape(3, rows, 2 * channels)         # parts of one projection
    state = h0.to(DEV)
    want, e = f64(h0), 0.0
    for t in range(3):
        got = P.linear_recurrence_step(both[t, :, :channels], both[t, :, channels:], state)
        gt, xt = f64(both[t, :, channels:]), f64(both[t, :, :channels])
        size = np.exp(gt) * np.abs(want) + np.abs(xt)
        want = np.exp(gt) * want + xt
        e = np.exp(gt) * e + (8 + 2 * np.abs(gt)) * U32 * size
        within(state, want, e + SMALL[torch.float32], "state")
        within(got, want, e + ROUND[dtype] * (np.abs(want) + e) + SMALL[dtype], "h")


@pytest.mark.gpu
def test_recurrence_gradients_are_differences(P):
    """Along random directions: <gradient, v> is the central difference of the loss in 64 bits, whose error is the third
    derivative's, below 1e-6 of the terms at a step of 1e-4."""
    rows, channels, starts = 90, 6, [0, 40, 41, 90]
    x, g, h0, grad, gf = recurrence_inputs(torch.float32, rows, channels, 3, seed=8)
    offsets = torch.tensor(starts, dtype=torch.int32, device=DEV)
    h, _ = P.linear_recurrence(x.to(DEV), g.to(DEV), initial_state=h0.to(DEV), offsets=offsets)
    dx, dg, d0 = P.linear_recurrence_backprop(h, g.to(DEV), grad.to(DEV), grad_final=gf.to(DEV), initial_state=h0.to(DEV), offsets=offsets)

    def loss(x, g, h0):
        (h, final), _ = recurrence_oracle(x, g, h0, starts)
        return (h * f64(grad)).sum() + (final * f64(gf)).sum()

    rng = np.random.default_rng(0)
    at, grads = [f64(x), f64(g), f64(h0)], [f64(dx), f64(dg), f64(d0)]
    for k in range(3):
        for _ in range(3):
            v = rng.standard_normal(at[k].shape)
            up, down = list(at), list(at)
            up[k], down[k] = at[k] + 1e-4 * v, at[k] - 1e-4 * v
            want = (loss(*up) - loss(*down)) / 2e-4
            size = np.abs(grads[k] * v).sum()
            assert abs((grads[k] * v).sum() - want) <= 1e-5 * size, k


@pytest.mark.gpu
def test_recurrence_takes_rows_apart_and_other_streams(P):
    x, g, h0, grad, gf = recurrence_inputs(torch.bfloat16, 2 * 150, 24, 2, seed=5)
    dense = P.linear_recurrence(x.to(DEV).reshape(2, 150, 24), g.to(DEV).reshape(2, 150, 24))
    both = torch.cat((g, x, grad), 1).to(DEV).reshape(2, 150, 72)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        parts = P.linear_recurrence(both[..., 24:48], both[..., :24])
        back = P.linear_recurrence_backprop(parts[0], both[..., :24], both[..., 48:])
    side.synchronize()
    want = P.linear_recurrence_backprop(dense[0], g.to(DEV).reshape(2, 150, 24), grad.to(DEV).reshape(2, 150, 24))
    turned = P.linear_recurrence(both[..., 24:48].transpose(0, 1).contiguous().transpose(0, 1), both[..., :24])
    for a, b in zip((*parts, *back, *turned), (*dense, *want, *dense)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_recurrence_of_nothing(P):
    for shape in [(0, 5, 3), (2, 0, 3), (2, 5, 0)]:
        x = torch.zeros(shape, device=DEV)
        start = torch.ones((shape[0], shape[2]), device=DEV)
        h, final = P.linear_recurrence(x, x, initial_state=start)
        assert h.shape == x.shape
        if shape[1] == 0:
            assert torch.equal(final, start)
        dx, dg, d0 = P.linear_recurrence_backprop(h, x, x, grad_final=start)
        assert d0.shape == start.shape
        if shape[1] == 0:
            assert torch.equal(d0, start)
    assert P.linear_recurrence_step(torch.zeros((0, 4), device=DEV), torch.zeros((0, 4), device=DEV), torch.zeros((0, 4), device=DEV)).shape == (0, 4)


# ---- norms and rotation ----

def rotary_oracle(x, w, cos, sin, positions, interleaved, eps, grad=None):
    rows, heads, dim = x.shape
    half = cos.shape[1]
    one = 2 * np.arange(half) if interleaved else np.arange(half)
    two = one + 1 if interleaved else one + half
    c, s = cos[positions][:, None], sin[positions][:, None]

    def turn(y, s):
        z = y.copy()
        z[..., one], z[..., two] = y[..., one] * c - y[..., two] * s, y[..., two] * c + y[..., one] * s
        return z

    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = turn(x * r * w, s)
    if grad is None:
        return y
    g = turn(grad, -s)
    u = g * w
    dx = r * (u - x * r * r * (u * x).mean(-1, keepdims=True))
    return y, dx, (g * x * r).sum((0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,kv,dim,rotary,interleaved", [
    (1, 1, 1, 2, 2, False), (1, 1, 1, 2, 0, True), (5, 3, 1, 64, 64, False), (33, 8, 2, 128, 128, True), (7, 5, 5, 96, 48, False),
    (7, 6, 3, 90, 34, True), (4, 2, 2, 90, 34, False), (3, 40, 8, 128, 128, False), (700, 4, 4, 32, 20, False), (3, 2, 1, 256, 256, False),
    (2, 0, 3, 72, 72, True), (3, 2, 0, 40, 8, False), (2100, 2, 1, 16, 6, True)])
def test_norm_rotary(P, dtype, tokens, heads, kv, dim, rotary, interleaved):
    rng = np.random.default_rng(dim + tokens)
    rows = torch.tensor(rng.standard_normal((tokens, heads + 2 * kv, dim))).to(dtype).to(DEV)
    q, k = rows[:, :heads], rows[:, heads:heads + kv]
    if heads:
        q[0, 0] = 0.0                   # a head of zeros: the norm is eps alone
    if heads > 1:
        q[-1, 1] *= 100.0
    grads = [torch.tensor(rng.standard_normal((tokens, n, dim))).to(dtype).to(DEV) for n in (heads, kv)]
    weights = [torch.tensor(1 + 0.3 * rng.standard_normal(dim), dtype=torch.float32, device=DEV) for _ in range(2)]
    cos, sin = P.rotary_tables(50, rotary, base=1000., device=DEV)
    positions = torch.tensor(rng.integers(0, 50, tokens), dtype=torch.int32, device=DEV)
    args = (q, k, *weights, cos, sin, positions)
    out = P.norm_rotary(*args, eps=1e-5, interleaved=interleaved)
    back = P.norm_rotary_backprop(*grads, *args, eps=1e-5, interleaved=interleaved)
    again = P.norm_rotary_backprop(*grads, *args, eps=1e-5, interleaved=interleaved)
    for a, b in zip(back, again):
        assert torch.equal(a, b)
    u = ROUND[dtype]
    for i, (x, w, g) in enumerate(zip((q, k), weights, grads)):
        want = rotary_oracle(f64(x), f64(w), f64(cos), f64(sin), f64(positions).astype(int), interleaved, 1e-5, f64(g))
        # sums of dim terms in 32 bits and a dozen roundings on the way, of values no larger than the row's largest
        f32 = (dim + 16) * U32
        size = np.abs(want[0]).max(-1, keepdims=True) if dim else 0.0
        within(out[i], want[0], u * np.abs(want[0]) + f32 * size + SMALL[dtype], "out")
        # the second term cancels the first where the gradient is along x: their sizes count, not the difference's
        r = 1 / np.sqrt((f64(x) ** 2).mean(-1, keepdims=True) + 1e-5)
        terms = 2 * r * (np.abs(f64(g)).max(-1, keepdims=True) * 2 * np.abs(f64(w)).max()) * (1 + (np.abs(f64(x)) * r).max(-1, keepdims=True) ** 2)
        within(back[i], want[1], u * np.abs(want[1]) + f32 * terms + SMALL[dtype], "dx")
        # tokens * heads terms added in pieces: at most 64 roundings deep in a lane, 64 slots, 512 / 16 + 16 pieces
        n = max(tokens * max(heads, kv), 1)
        each = np.abs(f64(x) * r).max() * np.abs(f64(g)).max() * 2 if x.numel() else 0.0
        within(back[2 + i], want[2], (f32 + min(n, 512) * U32) * n * each, "dw")


@pytest.mark.gpu
def test_norm_rotary_gradients_are_differences(P):
    rng = np.random.default_rng(2)
    tokens, heads, dim = 3, 2, 12
    x = torch.tensor(rng.standard_normal((tokens, heads, dim)), dtype=torch.float32, device=DEV)
    w = torch.tensor(1 + 0.3 * rng.standard_normal(dim), dtype=torch.float32, device=DEV)
    g = torch.tensor(rng.standard_normal((tokens, heads, dim)), dtype=torch.float32, device=DEV)
    cos, sin = P.rotary_tables(9, 8, device=DEV)
    positions = torch.tensor([8, 0, 3], dtype=torch.int32, device=DEV)
    dx, _, dw, _ = P.norm_rotary_backprop(g, g, x, x, w, w, cos, sin, positions)
    loss = lambda x, w: (rotary_oracle(x, w, f64(cos), f64(sin), np.array([8, 0, 3]), False, 1e-6) * f64(g)).sum()   # noqa: E731
    for _ in range(4):
        v, z = rng.standard_normal(x.shape), rng.standard_normal(dim)
        d = (loss(f64(x) + 1e-4 * v, f64(w)) - loss(f64(x) - 1e-4 * v, f64(w))) / 2e-4
        assert abs((f64(dx) * v).sum() - d) <= 1e-5 * np.abs(f64(dx) * v).sum()
        d = (loss(f64(x), f64(w) + 1e-4 * z) - loss(f64(x), f64(w) - 1e-4 * z)) / 2e-4
        assert abs((f64(dw) * z).sum() - d) <= 1e-5 * np.abs(f64(dw) * z).sum()


@pytest.mark.gpu
def test_norm_rotary_outside_the_tables_and_of_nothing(P):
    q, w = torch.ones((3, 2, 8), device=DEV), torch.ones(8, device=DEV)
    cos, sin = P.rotary_tables(4, 4, device=DEV)
    out, _ = P.norm_rotary(q, q, w, w, cos, sin, torch.tensor([0, 4, -1], dtype=torch.int32, device=DEV))
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:]).all()
    none = torch.ones((0, 2, 8), device=DEV)
    at = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert P.norm_rotary(none, none, w, w, cos, sin, at)[0].shape == (0, 2, 8)
    assert (P.norm_rotary_backprop(none, none, none, none, w, w, cos, sin, at)[2] == 0).all()


# ---- attention ----

def starts_of(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def attention_oracle(q, k, v, q_lengths, k_places, k_lengths, causal, scale, grad=None, u=0.0):
    """One sequence and head after the other.  Returns (out, lse[, dq, dk, dv]) and a bound for each of them.

    A score is a sum of dim products in 32 bits: off by e = (dim + 8) u32 scale |q||k|, so its weight by 2 e of its size; a
    weight is rounded to the inputs' type (u) before the second product, and weights far below the largest by 2^-24 of that
    (float16 has no smaller numbers); sums of n terms in 32 bits add (n + 16) u32 of their terms' sizes.  Backward, ds =
    p (dp - delta) is rounded likewise, and delta comes from the rounded output: off by u times |grad||out|."""
    heads, dim = q.shape[1:]
    group = heads // k.shape[1]
    out, lse = np.zeros_like(q), np.full(q.shape[:2], -np.inf)
    b_out, b_lse = np.zeros_like(q), np.zeros(q.shape[:2])
    grads = [np.zeros_like(t) for t in (q, k, v)]
    bounds = [np.zeros_like(t) for t in (q, k, v)]
    first = 0
    for n, a in enumerate(q_lengths):
        rows, cols = slice(first, first + a), slice(k_places[n], k_places[n] + k_lengths[n])
        first += a
        m = k_lengths[n]
        if not m or not a:
            continue
        hidden = np.arange(m)[None] > np.arange(a)[:, None] + m - a if causal else np.zeros((a, m), bool)
        for h in range(heads):
            Q, K, V = q[rows, h], k[cols, h // group], v[cols, h // group]
            score = np.where(hidden, -np.inf, Q @ K.T * scale)
            e = (dim + 8) * U32 * scale * (np.abs(Q) @ np.abs(K).T)
            top = score.max(1, keepdims=True)
            top[top == -np.inf] = 0.0
            w = np.exp(score - top)
            total = w.sum(1, keepdims=True)
            seen = total > 0
            total[~seen] = 1.0
            w = w / total
            e = np.where(hidden, 0.0, e)
            off = 2 * e.max(1, keepdims=True) + u + (m + 16) * U32
            tiny = m * 2.0 ** -24 * np.abs(V).max()
            out[rows, h] = w @ V
            b_out[rows, h] = np.where(seen, 2 * off * (w @ np.abs(V)) + tiny, 0.0)
            with np.errstate(divide="ignore"):
                lse[rows, h] = np.where(seen, top + np.log(total), -np.inf)[:, 0]
            b_lse[rows, h] = (off - u)[:, 0] + 4 * U32 * (np.abs(top[:, 0]) + 16)
            if grad is None:
                continue
            G = grad[rows, h]
            dp = G @ V.T
            delta = (G * out[rows, h]).sum(1, keepdims=True)
            ds = w * (dp - delta)
            # |dp - delta| at its largest, and its own error: delta's, and 32-bit sums of dim terms
            wrong = (u + (dim + 16) * U32) * (np.abs(G) * (np.abs(out[rows, h]) + b_out[rows, h])).sum(1, keepdims=True) + (
                dim + 8) * U32 * (np.abs(G) @ np.abs(V).T) + (np.abs(G) * b_out[rows, h]).sum(1, keepdims=True)
            b_ds = w * ((off + u) * (np.abs(dp) + np.abs(delta)) + wrong) + 2.0 ** -24 * (np.abs(dp) + np.abs(delta))
            b_ds = np.where(hidden, 0.0, b_ds)
            b_w = np.where(hidden, 0.0, w * (off + u) + 2.0 ** -24)
            grads[0][rows, h] = ds @ K * scale
            bounds[0][rows, h] = (b_ds + (m + 16) * U32 * np.abs(ds)) @ np.abs(K) * scale
            grads[1][cols, h // group] += ds.T @ Q * scale
            bounds[1][cols, h // group] += (b_ds + (a * group + 16) * U32 * np.abs(ds)).T @ np.abs(Q) * scale
            grads[2][cols, h // group] += w.T @ G
            bounds[2][cols, h // group] += (b_w + (a * group + 16) * U32 * w).T @ np.abs(G)
    if grad is None:
        return (out, lse), (b_out, b_lse)
    return (out, lse, *grads), (b_out, b_lse, *bounds)


def attention_inputs(dtype, q_rows, k_rows, heads, kv, dim, seed):
    rng = np.random.default_rng(seed)
    make = lambda rows, h, std: torch.tensor(std * rng.standard_normal((rows, h, dim))).to(dtype).to(DEV)      # noqa: E731
    return make(q_rows, heads, 1.4), make(k_rows, kv, 1.4), make(k_rows, kv, 1.0), make(q_rows, heads, 1.0)


HALVES = [torch.bfloat16, torch.float16]
SEQUENCES = [([1], [1]), ([0, 3, 0], [0, 3, 0]), ([64], [64]), ([65, 1, 255, 256, 257, 31], None), ([700], None), ([2] * 70, None),
             ([5, 1, 0, 7, 40], [130, 0, 9, 3, 33]), ([300], [290]), ([90], [500]), ([1, 1, 2], [900, 65, 64]), ([33, 0, 1] * 100, None),
             ([600, 530], None), ([2200], None)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("queries,keys", SEQUENCES)
@pytest.mark.parametrize("heads,kv,dim,causal", [(1, 1, 64, True), (4, 2, 128, True), (6, 1, 40, False), (3, 3, 96, True), (2, 2, 8, True),
                                                 (8, 1, 128, False)])
def test_attention(P, dtype, queries, keys, heads, kv, dim, causal):
    keys = keys or queries
    qs, ks = starts_of(queries), starts_of(keys)
    q, k, v, _ = attention_inputs(dtype, qs[-1], ks[-1], heads, kv, dim, seed=dim + qs[-1])
    offsets = [torch.tensor(s, dtype=torch.int32, device=DEV) for s in (qs, ks)]
    out, lse = P.attention(q, k, v, *offsets, causal=causal)
    u = ROUND[dtype]
    want, bound = attention_oracle(f64(q), f64(k), f64(v), queries, ks, keys, causal, dim ** -0.5, u=u)
    within(out, want[0], bound[0] + u * (np.abs(want[0]) + bound[0]) + SMALL[dtype], "out")
    within(lse, want[1], bound[1], "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("queries,keys", SEQUENCES)
@pytest.mark.parametrize("heads,kv,dim,causal", [(1, 1, 64, True), (4, 2, 128, True), (6, 1, 40, False), (3, 3, 96, True), (2, 1, 128, False)])
def test_attention_gradients(P, dtype, queries, keys, heads, kv, dim, causal):
    keys = keys or queries
    qs, ks = starts_of(queries), starts_of(keys)
    q, k, v, g = attention_inputs(dtype, qs[-1], ks[-1], heads, kv, dim, seed=dim + ks[-1])
    offsets = [torch.tensor(s, dtype=torch.int32, device=DEV) for s in (qs, ks)]
    out, lse = P.attention(q, k, v, *offsets, causal=causal)
    got = P.attention_backprop(g, q, k, v, out, lse, *offsets, causal=causal)
    again = P.attention_backprop(g, q, k, v, out, lse, *offsets, causal=causal)
    u = ROUND[dtype]
    want, bound = attention_oracle(f64(q), f64(k), f64(v), queries, ks, keys, causal, dim ** -0.5, grad=f64(g), u=u)
    for name, x, y, w, b in zip(("dq", "dk", "dv"), got, again, want[2:], bound[2:]):
        assert torch.equal(x, y), "the same inputs give the same bits"
        within(x, w, b + u * (np.abs(w) + b) + SMALL[dtype], name)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 2.0 ** -12])
def test_attention_gradients_are_differences(P, size):
    """Along random directions against central differences of the loss in 64 bits; small gradients as well, whose products
    float16 does not hold.  Terms of a direction are off by a few roundings each, so their sum by 8 u of their 2-norm times
    four standard deviations."""
    lengths, heads, kv, dim = [40, 3, 70], 4, 2, 64
    starts = starts_of(lengths)
    q, k, v, g = attention_inputs(torch.float16, 113, 113, heads, kv, dim, seed=6)
    g = g * size
    offsets = torch.tensor(starts, dtype=torch.int32, device=DEV)
    out, lse = P.attention(q, k, v, offsets, offsets)
    grads = [f64(t) for t in P.attention_backprop(g, q, k, v, out, lse, offsets, offsets)]
    at = [f64(t) for t in (q, k, v)]
    rng = np.random.default_rng(1)
    loss = lambda x: (attention_oracle(*x, lengths, starts, lengths, True, dim ** -0.5)[0][0] * f64(g)).sum()       # noqa: E731
    for i in range(3):
        for _ in range(2):
            z = rng.standard_normal(at[i].shape)
            up, down = list(at), list(at)
            up[i], down[i] = at[i] + 1e-4 * z, at[i] - 1e-4 * z
            want = (loss(up) - loss(down)) / 2e-4
            assert abs((grads[i] * z).sum() - want) <= 32 * ROUND[torch.float16] * np.sqrt(((grads[i] * z) ** 2).sum()), i


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lengths,heads,kv,dim,causal", [([40] * 8, 4, 4, 64, True), ([600], 2, 1, 40, False), ([640], 2, 1, 80, False),
                                                         ([900], 2, 1, 128, False), ([1300], 2, 1, 128, True)])
def test_attention_gradients_are_off_by_few_roundings(P, dtype, lengths, heads, kv, dim, causal):
    """The error's size as a whole, in that of the exact gradient rounded once to the type.  dV is a product of rounded
    weights, rounded: 2 of these squared.  dQ and dK are products of rounded dS, rounded, where dS, whose sum is zero, meets
    keys with a mean of their own: 0.2 more at these scores.  What else goes into dS may add half a rounding's: 2.7, 1.65."""
    starts = starts_of(lengths)
    q, k, v, g = attention_inputs(dtype, starts[-1], starts[-1], heads, kv, dim, seed=17)
    offsets = torch.tensor(starts, dtype=torch.int32, device=DEV)
    out, lse = P.attention(q, k, v, offsets, offsets, causal=causal)
    got = P.attention_backprop(g, q, k, v, out, lse, offsets, offsets, causal=causal)
    want = attention_oracle(f64(q), f64(k), f64(v), lengths, starts, lengths, causal, dim ** -0.5, grad=f64(g))[0][2:]
    for name, x, w in zip(("dq", "dk", "dv"), got, want):
        once = f64(torch.tensor(w).to(dtype)) - w
        assert np.linalg.norm(f64(x) - w) <= 1.65 * np.linalg.norm(once), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lengths,heads,kv,dim", [([1], 1, 1, 64), ([0, 5, 64, 65, 700, 33], 8, 2, 128), ([2500, 1, 3000], 12, 1, 40),
                                                  ([129] * 40, 4, 4, 64), ([4100], 5, 1, 128), ([300, 0, 17], 48, 1, 64)])
@pytest.mark.parametrize("queries", [1, 2, 5])
def test_attention_against_a_cache(P, dtype, lengths, heads, kv, dim, queries):
    """A few new tokens of each sequence, keys and values in a cache with room for more: what lies behind the lengths is
    never looked at, here it is not a number."""
    room, n = max(lengths) + 3, len(lengths)
    q, k, v, _ = attention_inputs(dtype, n * queries, n * room, heads, kv, dim, seed=room)
    for i, m in enumerate(lengths):
        k[i * room + m:(i + 1) * room] = float("nan")
        v[i * room + m:(i + 1) * room] = float("inf")
    places = [i * room for i in range(n + 1)]
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)         # noqa: E731
    out, lse = P.attention(q, k, v, whole([i * queries for i in range(n + 1)]), whole(places), k_lengths=whole(lengths), scale=0.11)
    again = P.attention(q, k, v, whole([i * queries for i in range(n + 1)]), whole(places), k_lengths=whole(lengths), scale=0.11)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    u = ROUND[dtype]
    want, bound = attention_oracle(f64(q), f64(k), f64(v), [queries] * n, places, lengths, True, 0.11, u=u)
    within(out, want[0], bound[0] + u * (np.abs(want[0]) + bound[0]) + SMALL[dtype], "out")
    within(lse, want[1], bound[1], "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
def test_attention_of_parts_of_a_projection_with_large_scores(P, dtype):
    """Rows with gaps; scores in the hundreds, so that weights run from 1 to nothing and the maximum moves late."""
    lengths, heads, kv, dim = [200, 77], 4, 2, 64
    starts = starts_of(lengths)
    rng = np.random.default_rng(4)
    rows = torch.tensor(rng.standard_normal((277, heads + 2 * kv, dim))).to(dtype).to(DEV)
    rows[:, :heads] *= 20.0
    rows[150, heads:heads + kv] *= 30.0
    offsets = torch.tensor(starts, dtype=torch.int32, device=DEV)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
    out, lse = P.attention(q, k, v, offsets, offsets, causal=True)
    u = ROUND[dtype]
    want, bound = attention_oracle(f64(q), f64(k), f64(v), lengths, starts, lengths, True, dim ** -0.5, u=u)
    within(out, want[0], bound[0] + u * (np.abs(want[0]) + bound[0]) + SMALL[dtype], "out")
    within(lse, want[1], bound[1], "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lengths,past,heads,kv,dim", [([300, 70, 5], 0, 4, 2, 64), ([700], 0, 2, 1, 128), ([900], 0, 2, 2, 40), ([5, 3], 400, 4, 2, 128),
                                                       ([1, 12], 300, 2, 1, 64)])
def test_attention_with_values_that_are_not_finite(P, dtype, lengths, past, heads, kv, dim):
    """A value that is infinite or not a number reaches the queries that see its key, and no others; so does a key."""
    keys = [n + past for n in lengths]
    qs, ks = starts_of(lengths), starts_of(keys)
    q, k, v, _ = attention_inputs(dtype, qs[-1], ks[-1], heads, kv, dim, seed=qs[-1])
    offsets = [torch.tensor(s, dtype=torch.int32, device=DEV) for s in (qs, ks)]
    clean, _ = P.attention(q, k, v, *offsets)
    for n in range(len(lengths)):
        for back, ch, x in [(1, 0, float("nan")), (2, dim - 1, float("inf")), (lengths[n] // 2 + 1, 5, -float("inf"))]:
            if back <= keys[n]:
                v[ks[n + 1] - back, 0, ch] = x
    out, lse = P.attention(q, k, v, *offsets)
    assert torch.isfinite(lse).all()
    values, group = f64(v), heads // kv
    want, touched = f64(clean).copy(), np.zeros(out.shape, bool)
    for n, a in enumerate(lengths):
        for j in range(a):
            row, seen = qs[n] + j, slice(ks[n], ks[n + 1] - a + j + 1)
            bad = np.where(np.isfinite(values[seen, 0]), 0.0, values[seen, 0])
            with np.errstate(invalid="ignore"):
                total = bad.sum(0)
            touched[row, :group] = total != 0
            want[row, :group] = np.where(total != 0, total, want[row, :group])
    got = f64(out)
    assert (np.isnan(got) == np.isnan(want)).all() and (got[touched & ~np.isnan(want)] == want[touched & ~np.isnan(want)]).all()
    assert (got[~touched] == want[~touched]).all()
    k[ks[-1] - 1] = float("nan")
    out, _ = P.attention(q, k, torch.nan_to_num(v, 0.0, 0.0, 0.0), *offsets)
    assert torch.isfinite(out[:-1]).all() and torch.isnan(out[-1]).all()


@pytest.mark.gpu
def test_offsets_that_do_not_ascend_stay_inside(P):
    """Offsets are not read on the host: whatever they hold, nothing is read or written outside the tensors."""
    rng = np.random.default_rng(3)
    rows = 300
    q, k, v, g = attention_inputs(torch.float16, rows, rows, 2, 1, 64, seed=3)
    x = torch.zeros((rows, 40), dtype=torch.bfloat16, device=DEV)
    for n in (1, 5, 64, 65, 400):
        offsets = torch.tensor(rng.integers(-1000, 1000, n + 1), dtype=torch.int32, device=DEV)
        offsets[n // 2] = 0
        offsets[n // 2 + 1] = rows
        out, lse = P.attention(q, k, v, offsets, offsets)
        P.attention(q, k, v, offsets, offsets, k_lengths=offsets[:-1].contiguous())
        P.attention_backprop(g, q, k, v, out, torch.zeros_like(lse), offsets, offsets)
        P.linear_recurrence(x, x, offsets=offsets)
        P.linear_recurrence_backprop(x, x, x, offsets=offsets)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_attention_of_nothing(P):
    q, k = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device=DEV), torch.zeros((3, 1, 64), dtype=torch.bfloat16, device=DEV)
    zero, at = torch.tensor([0, 0], dtype=torch.int32, device=DEV), torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    assert P.attention(q, k, k, zero, at)[0].shape == (0, 2, 64)
    out, lse = P.attention(torch.ones((3, 2, 64), dtype=torch.bfloat16, device=DEV), k[:0], k[:0], at, zero)
    assert (out == 0).all() and (lse == -float("inf")).all()


# ---- through autograd, and all together ----

@pytest.mark.gpu
def test_autograd_gives_the_gradients(P):
    lengths, heads, kv, dim = [40, 7, 0, 130], 4, 2, 64
    starts = starts_of(lengths)
    offsets = torch.tensor(starts, dtype=torch.int32, device=DEV)
    q, k, v, g = attention_inputs(torch.bfloat16, 177, 177, heads, kv, dim, seed=1)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = P.torch_api.attention(*leaves, offsets, offsets, scale=0.2)
    out.backward(g)
    same, lse = P.attention(q, k, v, offsets, offsets, scale=0.2)
    assert torch.equal(out, same)
    for x, y in zip(leaves, P.attention_backprop(g, q, k, v, same, lse, offsets, offsets, scale=0.2)):
        assert torch.equal(x.grad, y)
    w = [torch.rand(dim, device=DEV).requires_grad_(True) for _ in range(2)]
    cos, sin = P.rotary_tables(200, dim, device=DEV)
    at = torch.arange(177, dtype=torch.int32, device=DEV)
    leaves = [q.clone().requires_grad_(True), k.clone().requires_grad_(True), *w]
    a, b = P.torch_api.norm_rotary(*leaves, cos, sin, at, interleaved=True)
    (a.float().sum() + 2 * b.float().sum()).backward()
    want = P.norm_rotary_backprop(torch.ones_like(q), torch.full_like(k, 2.0), q, k, w[0].detach(), w[1].detach(), cos, sin, at, interleaved=True)
    for x, y in zip(leaves, want):
        assert torch.equal(x.grad, y)
    x, gate, h0, grad, gf = (t.to(DEV) for t in recurrence_inputs(torch.float16, 177, 20, 4, seed=2))
    leaves = [t.clone().requires_grad_(True) for t in (x, gate, h0)]
    h, final = P.torch_api.linear_recurrence(leaves[0], leaves[1], initial_state=leaves[2], offsets=offsets)
    torch.autograd.backward([h, final], [grad, gf])
    for t, y in zip(leaves, P.linear_recurrence_backprop(h.detach(), gate, grad, grad_final=gf, initial_state=h0, offsets=offsets)):
        assert torch.equal(t.grad, y)
    leaf = x.clone().requires_grad_(True)
    _, final = P.torch_api.linear_recurrence(leaf, gate, offsets=offsets)
    final.sum().backward()
    want = P.linear_recurrence_backprop(P.linear_recurrence(x, gate, offsets=offsets)[0], gate, torch.zeros_like(x),
                                        grad_final=torch.ones_like(final), offsets=offsets)[0]
    assert torch.equal(leaf.grad, want)


@pytest.mark.gpu
def test_the_example_learns_and_serves(P):
    import importlib.util
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("stream_model", os.path.join(root, "examples", "stream_model.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(0)
    model = example.StreamModel()
    losses = example.train(model, 30, gen, say=lambda line: None)
    assert sum(losses[-5:]) < 0.8 * sum(losses[:5]) and model.mix.weight.grad.abs().max() > 0
    worst, size = example.serve(model, gen)
    # both ways round to bfloat16 in a dozen places, at different ones inside the attention
    assert worst <= 32 * ROUND[torch.bfloat16] * max(size, 1.0)


@pytest.mark.gpu
def test_a_captured_graph_replays(P):
    """Serving captures its step: every replay gives what the same calls give outside the graph."""
    n, heads, kv, dim, room = 4, 8, 2, 128, 700
    q, k, v, _ = attention_inputs(torch.bfloat16, n, n * room, heads, kv, dim, seed=9)
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)         # noqa: E731
    queries, places, lengths = whole(range(n + 1)), whole([i * room for i in range(n + 1)]), whole([700, 1, 333, 64])
    w = torch.ones(dim, device=DEV)
    cos, sin = P.rotary_tables(room, dim, device=DEV)
    state, decay = torch.zeros((n, heads * dim), device=DEV), torch.full((n, heads * dim), -0.1, dtype=torch.bfloat16, device=DEV)

    def step():
        a, _ = P.norm_rotary(q, q[:, :kv], w, w, cos, sin, lengths - 1)
        out, lse = P.attention(a, k, v, queries, places, k_lengths=lengths)
        scan = P.linear_recurrence(out.flatten(1)[None].expand(3, n, heads * dim).reshape(1, 3 * n, heads * dim), decay.repeat(3, 1)[None])[0]
        return out, lse, scan, P.linear_recurrence_step(out.flatten(1), decay, state)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for turn in range(4):
        q.copy_(torch.randn_like(q))
        lengths.copy_(whole([700 - 100 * turn, 1 + turn, 333, 64]))
        state.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        state.zero_()
        for a, b in zip(got, step()):
            assert torch.equal(a, b), turn


# ---- refusals ----

@pytest.mark.gpu
def test_refusals(P):
    x, s = torch.zeros((2, 3, 4), device=DEV), torch.zeros((2, 4), device=DEV)
    with pytest.raises(TypeError):
        P.linear_recurrence(x.double(), x.double())
    with pytest.raises(TypeError):
        P.linear_recurrence(x, x.half())
    with pytest.raises(ValueError):
        P.linear_recurrence(x, x[:, :2])
    with pytest.raises(ValueError):
        P.linear_recurrence(x[0, 0], x[0, 0])
    with pytest.raises(ValueError):
        P.linear_recurrence(x, x, initial_state=s[:1])
    with pytest.raises(TypeError):
        P.linear_recurrence(x, x, initial_state=s.half())
    with pytest.raises(ValueError):
        P.linear_recurrence(x, x, offsets=torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(TypeError):
        P.linear_recurrence(x[0], x[0], offsets=torch.zeros(3, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):
        P.linear_recurrence(x[0], x[0], offsets=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        P.linear_recurrence_backprop(x, x, x[:1])
    with pytest.raises(ValueError):
        P.linear_recurrence_step(s, s, torch.zeros((4, 2), device=DEV).t())
    with pytest.raises(TypeError):
        P.linear_recurrence_step(s, s, s.half())
    q, w = torch.zeros((2, 3, 8), device=DEV), torch.ones(8, device=DEV)
    cos, sin = P.rotary_tables(4, 8, device=DEV)
    at = torch.zeros(2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        P.norm_rotary(q, q[:1], w, w, cos, sin, at)
    with pytest.raises(ValueError):
        P.norm_rotary(q, q, w[:4], w, cos, sin, at)
    with pytest.raises(TypeError):
        P.norm_rotary(q, q, w.half(), w, cos, sin, at)
    with pytest.raises(ValueError):
        P.norm_rotary(q[..., :6], q[..., :6], w[:6], w[:6], cos, sin, at)
    with pytest.raises(ValueError):
        P.norm_rotary(q[..., :7], q[..., :7], w[:7], w[:7], cos, sin, at)
    with pytest.raises(TypeError):
        P.norm_rotary(q, q, w, w, cos, sin, at.long())
    with pytest.raises(TypeError):
        P.norm_rotary(q, q, w, w, cos, sin, at, interleaved=1)
    with pytest.raises(ValueError):
        P.norm_rotary_backprop(q[:, :2], q, q, q, w, w, cos, sin, at)
    q = torch.zeros((4, 4, 64), dtype=torch.float16, device=DEV)
    k, at = q[:, :2], torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    assert P.attention(q, k, k, at, at)[0].shape == q.shape
    for args in [(q.float(), k.float(), k.float(), at, at), (q, k.bfloat16(), k, at, at), (q, k, k, at.long(), at)]:
        with pytest.raises(TypeError):
            P.attention(*args)
    for args in [(q, k, k[:, :1], at, at), (q, q[:, :3], q[:, :3], at, at), (q[..., :60], k[..., :60], k[..., :60], at, at), (q, k, k, at, at[:1]),
                 (q, k, k[:2], at, at), (q[:, :0], k, k, at, at), (q.repeat(1, 1, 3), k.repeat(1, 1, 3), k.repeat(1, 1, 3), at, at)]:
        with pytest.raises(ValueError):
            P.attention(*args)
    out, lse = P.attention(q, k, k, at, at)
    for args in [(q[:2], q, k, k, out, lse), (k, q, k, k, out, lse), (q, q, k, k, out[:2], lse), (q, q, k, k, out, lse[:, :2])]:
        with pytest.raises(ValueError):
            P.attention_backprop(*args, at, at)
    with pytest.raises(TypeError):
        P.attention_backprop(q, q, k, k, out, lse.half(), at, at)
    for options in [dict(scale=0.0), dict(scale=float("inf")), dict(k_lengths=at)]:
        with pytest.raises(ValueError):
            P.attention(q, k, k, at, at, **options)


def test_refuses_host_tensors(P):
    x = torch.zeros((2, 3))
    with pytest.raises(RuntimeError):
        P.linear_recurrence(x, x)
    with pytest.raises(TypeError):
        P.linear_recurrence(np.zeros((2, 3)), x)
    with pytest.raises(ValueError):
        P.rotary_tables(4, 3, device="cpu")
    cos, sin = P.rotary_tables(4, 6, base=100., scale=2., device="cpu")
    want = np.arange(4)[:, None] / 2 * 100.0 ** (-np.arange(3) / 3)
    assert np.abs(f64(cos) - np.cos(want)).max() <= U32 and np.abs(f64(sin) - np.sin(want)).max() <= U32


def test_the_entry_points_report_what_is_wrong(P):
    """Straight calls of the C entry points that never reach the GPU: status 2 and a message, nothing thrown."""
    from pysiglib_amd import _loader as L
    assert L.CUSIG_LINEAR_RECURRENCE(7, 0, 0, 0, 0, 0, 0, 1, 1, 1, 1, 1, 1, 0, 0, 0) == 2
    assert L.CUSIG_LINEAR_RECURRENCE(0, 0, 0, 0, 0, 0, 0, 1, 1, 1, 1, 1, 1, 0, 0, 0) == 2 and "missing" in L.last_error_message()
    assert L.CUSIG_LINEAR_RECURRENCE(0, 8, 8, 0, 8, 8, 0, 3, 1, 1, 1, 1, 1, 0, 0, 0) == 2
    assert L.CUSIG_LINEAR_RECURRENCE(0, 8, 8, 0, 8, 8, 0, 1, 100000, 100000, 8, 8, 8, 0, 0, 0) == 2 and "workspace" in L.last_error_message()
    assert L.CUSIG_LINEAR_RECURRENCE(0, 8, 8, 0, 8, 8, 0, 1, 5000, 5000, 8, 1 << 21, 8, 8, 1 << 40, 0) == 2 and "2^20" in L.last_error_message()
    assert L.CUSIG_LINEAR_RECURRENCE_STEP(0, 0, 0, 0, 0, 1, 1, 1, 1, 0) == 2
    assert L.CUSIG_LINEAR_RECURRENCE(0, 0, 0, 0, 0, 0, 0, 0, 5, 0, 8, 8, 8, 0, 0, 0) == 0
    rotary = [0, 8, 8, 8, 8, 8, 8, 8, 8, 8, 2, 2, 2, 8, 8, 4, 16, 8, 16, 8, 1e-6, False, 0]
    for at, value, text in [(13, 300, "too many"), (13, 9, "even"), (14, 3, "even"), (14, 16, "too many"), (5, 0, "missing"), (1, 0, "missing")]:
        args = list(rotary)
        args[at] = value
        assert L.CUSIG_NORM_ROTARY(*args) == 2 and text in L.last_error_message(), (at, value)
    attention = [1, 8, 8, 8, 8, 8, 0, 8, 8, 4, 4, 1, 2, 1, 64, 128, 64, 64, 64, 64, 64, 0.1, True, 0, 0, 0]
    for at, value, text in [(0, 0, "bfloat16"), (14, 60, "multiple of 8"), (14, 136, "multiple of 8"), (13, 0, "heads"), (12, 3, None), (21, 0.0, "scale"),
                            (15, 1 << 23, "apart"), (7, 0, "missing"), (1, 0, "missing")]:
        args = list(attention)
        args[at] = value
        if at == 12:
            args[13] = 2
        assert L.CUSIG_ATTENTION(*args) == 2 and (text is None or text in L.last_error_message()), (at, value)
    many = list(attention)
    many[11], many[9], many[10] = 100, 100000, 100000        # the list of the sequences' tiles needs room
    assert L.CUSIG_ATTENTION_WORKSPACE(100000, 100000, 100, 2, 1, 64) > 0
    assert L.CUSIG_ATTENTION(*many) == 2 and "workspace" in L.last_error_message()
    assert L.CUSIG_ATTENTION_WORKSPACE(4, 4, 0, 2, 1, 64) == 0 and L.CUSIG_ATTENTION_BACKPROP_WORKSPACE(4, 4, 0, 2, 64) > 0


# ---- gradients of very different sizes in one call ----

def gradients_of(P, q, k, v, g, lengths, causal):
    starts = starts_of(lengths)
    offsets = torch.tensor(starts, dtype=torch.int32, device=DEV)
    out, lse = P.attention(q, k, v, offsets, offsets, causal=causal)
    got = P.attention_backprop(g, q, k, v, out, lse, offsets, offsets, causal=causal)
    dim = q.shape[2]
    want = attention_oracle(f64(q), f64(k), f64(v), lengths, starts, lengths, causal, dim ** -0.5, grad=f64(g))[0][2:]
    return got, want


def few_roundings(got, want, dtype, what):
    """As in test_attention_gradients_are_off_by_few_roundings, of a part of the rows: their error in that of one rounding."""
    once = f64(torch.tensor(want).to(dtype)) - want
    off = f64(got) - want
    assert np.linalg.norm(off) <= 1.65 * np.linalg.norm(once), (what, float(np.linalg.norm(off) / np.linalg.norm(once)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("small,large", [(0.1, 4000.0), (0.01, 400.0), (0.1, 8.0)])
def test_attention_gradients_beside_much_larger_ones(P, dtype, dim, small, large):
    """A sequence's gradients have the same error whatever the other sequences' are, and a key's whatever those of queries
    that do not see it are."""
    lengths, heads, kv = [300, 200, 300], 2, 1
    starts = starts_of(lengths)
    q, k, v, g = attention_inputs(dtype, 800, 800, heads, kv, dim, seed=dim)
    g[:starts[1]] *= small
    g[starts[1]:starts[2]] *= large
    g[starts[2]:starts[2] + 40] *= large        # keys from 40 on are seen by queries of small gradients alone
    g[starts[2] + 40:] *= small
    got, want = gradients_of(P, q, k, v, g, lengths, True)
    for name, x, w in zip(("dq", "dk", "dv"), got, want):
        for rows in (slice(0, starts[1]), slice(starts[1], starts[2]), slice(starts[2] + 40, starts[3])):
            few_roundings(x[rows], w[rows], dtype, (name, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("v_size,g_size", [(30000.0, 1e-4), (1e-3, 1000.0)])
def test_attention_gradients_where_values_are_large_or_small(P, dtype, dim, v_size, g_size):
    """What float16 has to hold between the products is as large as gradients times values, not as the gradients."""
    lengths, heads, kv = [300, 37], 2, 1
    q, k, v, g = attention_inputs(dtype, 337, 337, heads, kv, dim, seed=dim + 1)
    v = v.sign() * v_size if v_size > 1 else v * v_size
    got, want = gradients_of(P, q, k, v, g * g_size, lengths, True)
    for name, x, w in zip(("dq", "dk"), got, want):
        few_roundings(x, w, dtype, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim,causal", [(64, True), (64, False), (128, False)])
@pytest.mark.parametrize("ahead", [8.0, 16.0, 24.0, 40.0])
@pytest.mark.parametrize("name", ["dk", "dv"])
def test_attention_gradients_of_keys_with_little_weight(P, dtype, dim, causal, ahead, name):
    """One key takes nearly all the weight of each query: the others' gradients are small, and as exact as the type holds
    them."""
    q, k, v, g = attention_inputs(dtype, 600, 600, 2, 1, dim, seed=int(ahead))
    q *= 0.3
    k *= 0.3
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[0, :, 0] = ahead * dim ** 0.5 / 8.0
    got, want = gradients_of(P, q, k, v, g * 256.0, [600], causal)
    which = ("dq", "dk", "dv").index(name)
    few_roundings(got[which][1:], want[which][1:], dtype, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lengths,heads,kv,dim", [([100, 40], 4, 2, 64), ([150], 2, 1, 128), ([90, 5, 33], 2, 2, 40), ([33] * 70, 1, 1, 64),
                                                  ([1500, 40], 1, 1, 96)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["q", "k", "v", "grad"])
@pytest.mark.parametrize("first", [False, True])
def test_attention_gradients_of_what_is_not_finite(P, dtype, lengths, heads, kv, dim, bad, which, first):
    """One element that is not finite reaches what the formula sums it into, over the visible pairs, and nothing else."""
    starts = starts_of(lengths)
    offsets = torch.tensor(starts, dtype=torch.int32, device=DEV)
    tensors = dict(zip(("q", "k", "v", "grad"), attention_inputs(dtype, starts[-1], starts[-1], heads, kv, dim, seed=dim)))

    def gradients():
        q, k, v, g = (tensors[n] for n in ("q", "k", "v", "grad"))
        out, lse = P.attention(q, k, v, offsets, offsets)
        return P.attention_backprop(g, q, k, v, out, lse, offsets, offsets)

    clean = [f64(t) for t in gradients()]
    n = 0
    t, ch = 0 if first else lengths[0] // 2, 3
    row = starts[n] + t
    tensors[which][row, 0, ch] = bad
    got = [f64(x) for x in gradients()]
    q, k, v, g = (f64(tensors[x])[starts[n]:starts[n + 1]] for x in ("q", "k", "v", "grad"))
    # sums over visible pairs alone, of the head that has it
    m, scale = lengths[n], dim ** -0.5
    want = [np.zeros((m, dim)) for _ in range(3)]
    K, V, Q, G = k[:, 0], v[:, 0], q[:, 0], g[:, 0]
    with np.errstate(all="ignore"):
        for i in range(m):
            s = K[:i + 1] @ Q[i] * scale
            # scores of -infinity alone are those of a query that sees nothing: no weights
            p = np.zeros(i + 1) if (s == -np.inf).all() else np.exp(s - s.max()) / np.exp(s - s.max()).sum()
            out = (p[:, None] * V[:i + 1]).sum(0)
            ds = p * ((V[:i + 1] * G[i]).sum(1) - (G[i] * out).sum())
            want[0][i] = (ds[:, None] * K[:i + 1]).sum(0)
            want[1][:i + 1] += ds[:, None] * Q[i]
            want[2][:i + 1] += p[:, None] * G[i]
    group = heads // kv
    for name, x, c, w in zip(("dq", "dk", "dv"), got, clean, want):
        fine = np.isfinite(w)
        here = x[starts[n]:starts[n + 1], 0]
        assert (np.isfinite(here) == fine).all(), (name, np.argwhere(np.isfinite(here) != fine)[:5])
        # what lies before (queries) or behind (keys) the element's token has nothing to do with it
        apart = slice(0, t) if name == "dq" else slice(t + 1, m)
        if which in ("q", "grad") or name == "dq":
            assert (here[apart] == c[starts[n]:starts[n + 1], 0][apart]).all(), name
        assert (x[starts[1]:] == c[starts[1]:]).all(), name
        others = slice(group if name == "dq" and which in ("k", "v") else 1, None)
        assert (x[:, others] == c[:, others]).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rotary", [(256, 100), (256, 250), (254, 4), (252, 2), (254, 254)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rotary_of_the_widest_heads(P, dtype, dim, rotary, interleaved):
    test_norm_rotary(P, dtype, 5, 3, 2, dim, rotary, interleaved)


# ---- rows that belong to no sequence, offsets that leave the tensors ----

def whole_numbers(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def raw(fn, *args):
    """A C entry point on the current stream, tensors as their addresses."""
    code = fn(*(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args), torch.cuda.current_stream().cuda_stream)
    assert code == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(300, 24), (5000, 24), (5000, 3), (9000, 70)])
@pytest.mark.parametrize("offsets,cut", [([7, 100, 100, 290], None), ([-5, 100, 290], [0, 100, 290]), ([20, 100, 1 << 30], [20, 100, -1]),
                                         ([-9, -7, 60, 1 << 30, (1 << 30) + 5], [0, 0, 60, -1, -1])])
def test_recurrence_leaves_other_rows_alone(P, dtype, rows, channels, offsets, cut):
    """Straight calls on buffers that hold a mark: rows of no sequence keep it, sequences are cut to the rows there are, and
    every sequence has a state behind it.  Short calls walk sequences, long ones publish: both alike."""
    from pysiglib_amd import _loader as L
    offsets, n = ([x if x > 1 << 20 or x < 0 else x * rows // 300 for x in offsets]), len(offsets) - 1
    cut = [rows if x == -1 else x * rows // 300 for x in cut] if cut else offsets
    x, g, h0, grad, gf = (t.to(DEV) for t in recurrence_inputs(dtype, rows, channels, n, seed=rows))
    code = L.SEQUENCE_DTYPES[str(dtype).split(".")[1]]
    size = L.CUSIG_LINEAR_RECURRENCE_WORKSPACE(code, rows, n, channels)
    space = torch.zeros(max(size, 1), dtype=torch.uint8, device=DEV)
    marked = lambda shape, t=dtype: torch.full(shape, 77.0, dtype=t, device=DEV)       # noqa: E731
    h, final = marked(x.shape), marked(h0.shape, torch.float32)
    at = whole_numbers(offsets)
    raw(L.CUSIG_LINEAR_RECURRENCE, code, x, g, h0, h, final, at, n, 0, rows, channels, channels, channels, space, size)
    dx, dg, d0 = marked(x.shape), marked(x.shape), marked(h0.shape, torch.float32)
    raw(L.CUSIG_LINEAR_RECURRENCE_BACKPROP, code, h, g, grad, gf, h0, dx, dg, d0, at, n, 0, rows, channels, channels, channels, space, size)
    first, past = cut[0], cut[-1]
    part = slice(first, past)
    inside = [c - first for c in cut]
    want, bound = recurrence_oracle(f64(x)[part], f64(g)[part], f64(h0), inside, f64(grad)[part], f64(gf), f64(h)[part])
    for name, got, w, b in zip(("h", "final", "dx", "dg", "d0"), (h, final, dx, dg, d0), want, bound):
        mine = got[part] if name in ("h", "dx", "dg") else got
        u, tiny = (ROUND[dtype], SMALL[dtype]) if name in ("h", "dx", "dg") else (U32, SMALL[torch.float32])
        within(mine, w, b + u * (np.abs(w) + b) + tiny, name)
        if name in ("h", "dx", "dg"):
            assert (got[:first] == 77.0).all() and (got[past:] == 77.0).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("room", [40, 3000])
@pytest.mark.parametrize("n", [2, 70])
def test_attention_leaves_other_rows_alone(P, dtype, room, n):
    """Rows of queries before the first sequence and behind the last keep what they held, with the keys in one piece and
    in several."""
    from pysiglib_amd import _loader as L
    heads, kv, dim, before, behind = 4, 2, 64, 3, 6
    q_rows, k_rows = before + n + behind, n * room
    q, k, v, _ = attention_inputs(dtype, q_rows, k_rows, heads, kv, dim, seed=room)
    out = torch.full(q.shape, 77.0, dtype=dtype, device=DEV)
    lse = torch.full(q.shape[:2], 77.0, dtype=torch.float32, device=DEV)
    sizes = (q_rows, k_rows, n, heads, kv, dim)
    size = L.CUSIG_ATTENTION_WORKSPACE(*sizes)
    space = torch.full((max(size, 4),), 255, dtype=torch.uint8, device=DEV)          # no number anywhere
    at, places = whole_numbers(range(before, before + n + 1)), whole_numbers([i * room for i in range(n + 1)])
    raw(L.CUSIG_ATTENTION, L.SEQUENCE_DTYPES[str(dtype).split(".")[1]], q, k, v, at, places, 0, out, lse, *sizes, heads * dim, dim, kv * dim, dim,
        kv * dim, dim, dim ** -0.5, True, space, size)
    mine = slice(before, before + n)
    want, _ = P.attention(q[mine], k, v, at - before, places)
    bound = 4 * ROUND[dtype] * f64(v).max()         # cut in ranges differently: weights rounded at other maxima
    assert np.abs(f64(out[mine]) - f64(want)).max() <= bound
    for t in (out, lse):
        assert (t[:before] == 77.0).all() and (t[before + n:] == 77.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("keys", [700, 2560, 3000, 6000])
def test_an_infinite_value_stays_infinite_over_ranges_of_keys(P, dtype, keys):
    """Keys cut in any number of ranges: an infinite value in the last one gives infinity, as in one piece."""
    q, k, v, _ = attention_inputs(dtype, 1, keys, 1, 1, 64, seed=keys)
    clean, _ = P.attention(q, k, v, whole_numbers([0, 1]), whole_numbers([0, keys]))
    v[keys - 1, 0, 5], v[keys - 1, 0, 6], v[0, 0, 7] = float("inf"), -float("inf"), float("inf")
    out, lse = P.attention(q, k, v, whole_numbers([0, 1]), whole_numbers([0, keys]))
    got = f64(out)[0, 0]
    assert got[5] == np.inf and got[6] == -np.inf and got[7] == np.inf
    same = [c for c in range(64) if c not in (5, 6, 7)]
    assert (got[same] == f64(clean)[0, 0, same]).all()


# ---- rows far apart, many blocks ----

@pytest.mark.gpu
def test_attention_of_tokens_far_apart(P):
    """The last tokens of long sequences side by side: tokens 2^24 elements apart."""
    n, length, heads, dim = 3, 4096, 32, 128
    rows = torch.randn((n, length, heads, dim), device=DEV).to(torch.bfloat16)
    last = rows[:, -1]
    at = whole_numbers(range(n + 1))
    dense = last.contiguous()
    assert last.stride(0) == 1 << 24
    for args in [(last, dense, dense), (dense, last, last), (last, last, last)]:
        for got, want in zip(P.attention(*args, at, at), P.attention(dense, dense, dense, at, at)):
            assert torch.equal(got, want)
    out, lse = P.attention(dense, dense, dense, at, at)
    for got, want in zip(P.attention_backprop(last, last, last, last, out, lse, at, at), P.attention_backprop(dense, dense, dense, dense, out, lse, at, at)):
        assert torch.equal(got, want)
    one = whole_numbers([0, 1])
    single = rows[1:2, -1]                 # a single token: the distance to the next has no meaning
    assert torch.equal(P.attention(single, single, single, one, one)[0], single)
    out, lse = P.attention(single, single, single, one, one)
    assert P.attention_backprop(single, single, single, single, out, lse, one, one)[0].shape == single.shape


@pytest.mark.gpu
def test_recurrence_of_rows_far_apart(P):
    """A few channels of very long rows."""
    wide = torch.randn((12, (1 << 20) + 8), device=DEV).to(torch.bfloat16)
    x, g, grad = wide[:, :16], -wide[:, 16:32].abs(), wide[:, 32:48]
    far = torch.empty_like(wide)
    far[:, :16] = g
    g = far[:, :16]
    assert min(t.stride(0) for t in (x, g, grad)) > 1 << 20
    dense = [t.contiguous() for t in (x, g, grad)]
    at = whole_numbers([0, 5, 12])
    got, want = P.linear_recurrence(x, g, offsets=at), P.linear_recurrence(*dense[:2], offsets=at)
    back, same = P.linear_recurrence_backprop(want[0], g, grad, offsets=at), P.linear_recurrence_backprop(want[0], *dense[1:], offsets=at)
    for a, b in zip((*got, *back), (*want, *same)):
        assert torch.equal(a, b)
    state = torch.zeros((12, 16), device=DEV)
    assert torch.equal(P.linear_recurrence_step(x, g, state), dense[0])


@pytest.mark.gpu
def test_more_threads_than_a_launch_has(P):
    """A launch numbers its threads with 32 bits: these calls have more, and go in several."""
    from pysiglib_amd import _loader as L
    # 2^24 + 3 sequences of one step, a block of 256 threads to each
    n = (1 << 24) + 3
    x = torch.randn((n, 1, 4), device=DEV).to(torch.bfloat16)
    g, start = torch.zeros_like(x), torch.randn((n, 4), device=DEV)
    assert L.CUSIG_LINEAR_RECURRENCE_WORKSPACE(1, n, n, 4) == 0
    h, final = P.linear_recurrence(x, g, initial_state=start)
    want = start + x[:, 0].float()
    assert torch.equal(final, want) and torch.equal(h[:, 0], want.to(torch.bfloat16))
    dx, dg, d0 = P.linear_recurrence_backprop(h, g, x, grad_final=start, initial_state=start)
    assert torch.equal(d0, want) and torch.equal(dx[:, 0], want.to(torch.bfloat16)) and torch.equal(dg[:, 0], (want * start).to(torch.bfloat16))
    del x, g, start, h, final, want, dx, dg, d0
    # 2^26 + 5 tokens, a wave to each
    tokens = (1 << 26) + 5
    q = torch.ones((tokens, 1, 2), dtype=torch.bfloat16, device=DEV)
    q[-3:, 0, 1] = -1.0
    w = torch.tensor([2.0, 3.0], device=DEV)
    cos, sin = P.rotary_tables(1, 0, device=DEV)
    out, _ = P.norm_rotary(q, q[:, :0], w, w, cos, sin, torch.zeros(tokens, dtype=torch.int32, device=DEV), eps=0.0)
    assert (out[..., 0] == 2.0).all() and (out[:-3, 0, 1] == 3.0).all() and (out[-3:, 0, 1] == -3.0).all()
    del q, out
    # 65 sequences of one token, 2^19 heads: a block to each
    heads, n = 1 << 19, 65
    q, k, v, g = (torch.randn((n, heads, 8), device=DEV).to(torch.bfloat16) for _ in range(4))
    at = whole_numbers(range(n + 1))
    out, lse = P.attention(q, k, v, at, at, scale=0.5)
    assert torch.equal(out, v)
    score = (q.double() * k.double()).sum(-1) * 0.5
    size = (q.double() * k.double()).abs().sum(-1) * 0.5
    assert ((lse - score).abs() <= 16 * U32 * (size + 1)).all()
    dq, dk, dv = P.attention_backprop(g, q, k, v, out, lse, at, at, scale=0.5)
    assert torch.equal(dv, g)
    # dp - delta, 8 terms each, is nothing but their roundings
    most = 32 * U32 * (g.double() * v.double()).abs().sum(-1, keepdim=True) * 0.5
    assert (dq.double().abs() <= most * k.double().abs() * 1.01).all() and (dk.double().abs() <= most * q.double().abs() * 1.01).all()


# ---- decays of -inf, states that are not finite ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(700, 24), (6000, 24), (6000, 2), (9000, 70)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_recurrence_forgets_at_minus_infinity_and_nowhere_else(P, dtype, rows, channels, bad):
    """A state that is not finite goes on through any number of decays, and ends at one whose exponential is zero in 32 bits,
    -inf or not; backwards alike.  Wherever in a block's rows that is."""
    rng = np.random.default_rng(rows)
    x, g, h0, grad, gf = recurrence_inputs(dtype, rows, channels, 1, seed=rows)
    g = torch.minimum(g, torch.tensor(-0.25, dtype=dtype))
    ends = np.full(channels, rows)
    for c in range(channels):
        begin = int(rng.integers(0, rows // 3))
        x[begin, c] = bad
        if c % 3:
            ends[c] = int(rng.integers(begin + 1, rows))
            g[ends[c], c] = -float("inf") if c % 3 == 1 else -300.0
    put = lambda t: t.to(DEV)[None]              # noqa: E731
    h, final = P.linear_recurrence(put(x), put(g), initial_state=put(h0)[0])
    got, last = f64(h)[0], f64(final)[0]
    for c in range(channels):
        begin = int(np.flatnonzero(~np.isfinite(f64(x[:, c])))[0])
        end = ends[c]
        assert np.isfinite(got[:begin, c]).all() and np.isfinite(got[end:, c]).all(), c
        assert (np.isinf if bad == bad else np.isnan)(got[begin:end, c]).all(), c
        assert np.isfinite(last[c]) == (end < rows), c
        if end < rows:
            assert got[end, c] == f64(x[end, c]), c
    # backwards from a gradient that is not finite
    x, g, h0, grad, gf = recurrence_inputs(dtype, rows, channels, 1, seed=rows)
    g = torch.minimum(g, torch.tensor(-0.25, dtype=dtype))
    stops = np.full(channels, -1)
    at = np.zeros(channels, int)
    for c in range(channels):
        at[c] = int(rng.integers(2 * rows // 3, rows))
        grad[at[c], c] = bad
        if c % 3:
            stops[c] = int(rng.integers(0, at[c]))
            g[stops[c], c] = -float("inf") if c % 3 == 1 else -300.0
    h, _ = P.linear_recurrence(put(x), put(g), initial_state=put(h0)[0])
    dx, dg, d0 = (f64(t)[0] for t in P.linear_recurrence_backprop(h, put(g), put(grad), grad_final=put(gf)[0], initial_state=put(h0)[0]))
    for c in range(channels):
        s = stops[c]
        assert np.isfinite(dx[at[c] + 1:, c]).all() and np.isfinite(dx[:max(s, 0), c]).all(), c
        assert not np.isfinite(dx[max(s, 0):at[c] + 1, c]).any(), c
        assert not np.isfinite(dg[s + 1:at[c] + 1, c]).any() and np.isfinite(dg[at[c] + 1:, c]).all() and np.isfinite(dg[:s + 1, c]).all(), c
        assert np.isfinite(d0[c]) == (s >= 0), c
    # an infinite state meets a decay of -inf: neither gradient of that step depends on it
    x, g, h0, grad, gf = recurrence_inputs(dtype, rows, channels, 1, seed=rows)
    h, _ = P.linear_recurrence(put(x), put(g))
    g[rows // 2] = -float("inf")
    h[0, rows // 2 - 1] = float("inf")
    _, dg, _ = P.linear_recurrence_backprop(h, put(g), put(grad))
    assert (dg[0, rows // 2] == 0).all()


# ---- with autograd around them ----

@pytest.mark.gpu
def test_a_state_that_is_replaced_is_known_to_autograd(P):
    """An operation that kept the state for its gradient finds out that it has changed."""
    x, state = torch.randn((3, 8), device=DEV), torch.randn((3, 8), device=DEV)
    w = torch.ones((3, 8), device=DEV, requires_grad=True)
    kept = (w * state).sum()
    before = state._version
    P.linear_recurrence_step(x, x, state)
    assert state._version > before
    with pytest.raises(RuntimeError):
        kept.backward()
    with torch.inference_mode():
        P.linear_recurrence_step(x, x, torch.zeros((3, 8), device=DEV))


@pytest.mark.gpu
def test_second_derivatives_are_refused(P):
    """The gradients are not differentiable: they say so, rather than leave a part of a second derivative out."""
    A = P.torch_api
    at = whole_numbers([0, 6])
    q, k = (torch.randn((6, n, 64), device=DEV).half().requires_grad_(True) for n in (2, 1))
    w = torch.ones(64, device=DEV, requires_grad=True)
    cos, sin = P.rotary_tables(8, 64, device=DEV)
    x = torch.randn((2, 6, 8), device=DEV, requires_grad=True)
    positions = torch.arange(6, dtype=torch.int32, device=DEV)
    for out, leaf in [(A.attention(q, k, k, at, at), q), (A.norm_rotary(q, k, w, w, cos, sin, positions)[0], q),
                      (A.linear_recurrence(x, -x.detach().abs())[0], x)]:
        for loss in (out.float().sum(), out.float().square().sum()):
            grad, = torch.autograd.grad(loss, leaf, create_graph=True, retain_graph=True)
            assert torch.isfinite(grad).all()
            with pytest.raises(RuntimeError):
                (grad.float().sum() + leaf.float().sum()).backward()
        grad, = torch.autograd.grad(out.float().sum(), leaf)
        assert not grad.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("keys", [False, True])
def test_lists_of_tiles_hold_what_offsets_that_do_not_ascend_name(P, keys):
    """Offsets to and fro name more tiles than 32 bits count: the list keeps to its room, and nothing around it changes."""
    from pysiglib_amd import _loader as L
    rows, n, dim = 1 << 22, 140000, 8
    at, none = torch.zeros(n + 1, dtype=torch.int32, device=DEV), torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    at[1::2] = rows
    wide, small = torch.zeros((rows, 1, dim), dtype=torch.bfloat16, device=DEV), torch.zeros((4, 1, dim), dtype=torch.bfloat16, device=DEV)
    out, one = torch.zeros_like(wide), torch.zeros_like(small)
    if keys:
        sizes, size = (4, rows, n, 1, 1, dim), L.CUSIG_ATTENTION_BACKPROP_WORKSPACE(4, rows, n, 1, dim)
    else:
        sizes, size = (rows, 4, n, 1, 1, dim), L.CUSIG_ATTENTION_WORKSPACE(rows, 4, n, 1, 1, dim)
    space = torch.full((size + 2 * 4096,), 91, dtype=torch.uint8, device=DEV)
    inner = space[4096:4096 + size]
    lse = torch.zeros((rows, 1), device=DEV)
    if keys:
        raw(L.CUSIG_ATTENTION_BACKPROP, 1, small, small, wide, wide, small, lse, none, at, one, out, out, *sizes, dim, dim, dim, dim, dim, dim, dim, dim,
            0.5, True, inner, size)
    else:
        raw(L.CUSIG_ATTENTION, 1, wide, small, small, at, none, 0, out, lse, *sizes, dim, dim, dim, dim, dim, dim, 0.5, True, inner, size)
    assert (space[:4096] == 91).all() and (space[4096 + size:] == 91).all() and (out == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim", [8, 40, 64, 96, 128])
@pytest.mark.parametrize("queries,keys", [(300, 300), (1, 700), (2, 40)])
def test_keys_of_minus_infinity_have_no_weight(P, dtype, dim, queries, keys):
    """A key that is infinite in one channel, against queries that make its score -infinity: as if it were not there, in any
    channel of heads of any width."""
    q, k, v, _ = attention_inputs(dtype, queries, keys, 2, 1, dim, seed=dim)
    at = [whole_numbers([0, n]) for n in (queries, keys)]
    for channel in sorted({0, dim - 8, dim - 1}):
        key, query = k.clone(), q.clone()
        query[..., channel] = query[..., channel].abs() + 0.5
        key[3:keys - 1:5, 0, channel] = -float("inf")
        without = f64(key)
        without[3:keys - 1:5] = 0.0
        without[3:keys - 1:5, 0, channel] = -1e30
        out, lse = P.attention(query, key, v, *at, causal=False)
        u = ROUND[dtype]
        with np.errstate(over="ignore"):
            want, bound = attention_oracle(f64(query), without, f64(v), [queries], [0, keys], [keys], False, dim ** -0.5, u=u)
        sizes = f64(key)
        sizes[~np.isfinite(sizes)] = 0.0
        _, bound = attention_oracle(f64(query), sizes, f64(v), [queries], [0, keys], [keys], False, dim ** -0.5, u=u)
        # the weights are those of the other keys: at most 5 / 4 of what the bound takes them to be
        within(out, want[0], 2 * (bound[0] + u * (np.abs(want[0]) + bound[0])) + SMALL[dtype], "out")
        within(lse, want[1], 2 * bound[1], "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim,queries,keys,causal", [(64, 600, 600, True), (64, 600, 600, False), (128, 300, 600, False), (128, 1, 8000, True), (40, 3, 3000, True)])
@pytest.mark.parametrize("ahead", [8.0, 12.0, 16.0])
def test_attention_beside_a_key_that_takes_the_weight(P, dtype, dim, queries, keys, causal, ahead):
    """One key takes nearly all of each query's weight and has no value: the output is that of the others, as exact as the
    type holds it."""
    q, k, v, _ = attention_inputs(dtype, queries, keys, 2, 1, dim, seed=int(ahead))
    q *= 0.3
    k *= 0.3
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[0, :, 0] = ahead * dim ** 0.5 / 8.0
    v[0] = 0.0
    v *= 256.0
    at = [whole_numbers([0, n]) for n in (queries, keys)]
    out, _ = P.attention(q, k, v, *at, causal=causal)
    want = attention_oracle(f64(q), f64(k), f64(v), [queries], [0, keys], [keys], causal, dim ** -0.5)[0][0]
    few_roundings(out, want, dtype, "out")


def test_weights_without_a_place_for_their_gradients_are_refused(P):
    """Before anything reaches the GPU, also where there are no tokens and the gradients are zero."""
    from pysiglib_amd import _loader as L
    size = L.CUSIG_NORM_ROTARY_BACKPROP_WORKSPACE(8)
    for tokens in (2, 0):
        for at in (12, 13):
            args = [0] + [256] * 13 + [tokens, 2, 2, 8, 8, 4, 16, 8, 16, 8, 16, 8, 16, 8, 1e-6, False, 256, size, 0]
            args[at] = 0
            assert L.CUSIG_NORM_ROTARY_BACKPROP(*args) == 2 and "missing" in L.last_error_message(), (tokens, at)


def test_a_workspace_that_is_not_aligned_is_refused(P):
    """Words of it are 64-bit and accessed at once; before anything reaches the GPU."""
    from pysiglib_amd import _loader as L
    far = 1 << 40
    calls = [(L.CUSIG_LINEAR_RECURRENCE, [0, 256, 256, 0, 256, 256, 0, 1, 100000, 100000, 8, 8, 8]),
             (L.CUSIG_LINEAR_RECURRENCE_BACKPROP, [0, 256, 256, 256, 0, 0, 256, 256, 256, 0, 1, 100000, 100000, 8, 8, 8]),
             (L.CUSIG_NORM_ROTARY_BACKPROP, [0] + [256] * 13 + [2, 2, 2, 8, 8, 4, 16, 8, 16, 8, 16, 8, 16, 8, 1e-6, False]),
             (L.CUSIG_ATTENTION, [1] + [256] * 5 + [0, 256, 256, 100000, 100000, 100, 2, 1, 64, 128, 64, 64, 64, 64, 64, 0.1, True]),
             (L.CUSIG_ATTENTION_BACKPROP, [1] + [256] * 11 + [4, 4, 1, 2, 1, 64, 128, 64, 64, 64, 64, 64, 128, 64, 0.1, True])]
    for fn, args in calls:
        assert fn(*args, 260, far, 0) == 2 and "aligned" in L.last_error_message(), fn
        assert fn(*args, 256, 0, 0) == 2 and "too small" in L.last_error_message(), fn
