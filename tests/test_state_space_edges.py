"""Values at the ends of the number formats, and places of the state space layers that only some sizes reach (see test_state_space.py,
whose formulas, bounds and helpers these are)."""
import os
import re

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_state_space import (DEV, NAMES, P, TYPES, U32, check_scan, f64, numbers, raw, rounded, same_bits, scan_inputs, scan_oracle,  # noqa: E402,F401
                                    starts_of, whole_numbers)


# ---- the norm in 8 bits ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [5, 40, 2000, 9000])
def test_norm_in_8_bits_of_infinite_outputs(P, dtype, channels):
    """Their scale is infinite: the quotient by it is zero for finite outputs, of either sign, and NaN for infinite ones.  A row whose infinite
    weight meets a zero holds NaN instead."""
    rng = np.random.default_rng(channels)
    x = numbers(rng, 6, channels, dtype=dtype)
    x[:, 1] = 1.0
    x[4, 1] = 0.0
    x[5, 1] = -1.0
    for top in (float("inf"), float("-inf"), 3.4e38):
        w = numbers(rng, channels)
        w[1] = top
        if top == 3.4e38:       # finite, and its product with a value above the row's mean is not
            x[:, 1] = torch.tensor([40.0, 40.0, 40.0, 40.0, 0.0, -40.0], device=DEV)
        q, scales, _ = P.norm_residual_float8(x, None, w, eps=1e-6)
        q, held = q.float(), [0, 1, 2, 3, 5]
        if top == 3.4e38:
            assert torch.isfinite(scales[4]).all() and torch.isfinite(q[4]).all()
        else:
            assert scales[4] == 1 and torch.isnan(q[4, 1]) and torch.isfinite(q[4, [c for c in range(channels) if c != 1]]).all()
        assert torch.isposinf(scales[held]).all(), "the largest size of the row divided by 448"
        assert torch.isnan(q[held, 1]).all() and (q[held][:, [c for c in range(channels) if c != 1]] == 0).all()
        out = P.norm_residual(x.float(), None, w, eps=1e-6)[0]
        want = (out / scales).clamp(-448, 448)[held]
        assert np.array_equal(f64(q[held]), f64(want), equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [64, 2048, 16384])
@pytest.mark.parametrize("scale", [2.0 ** -60, 1.1 * 2.0 ** -64, 2.0 ** -64, 0.9 * 2.0 ** -64, 1.3 * 2.0 ** -126, 2.0 ** -126, 0.7 * 2.0 ** -126, 2.0 ** -140, 5 * 2.0 ** -149,
                                   2.0 ** -149, 1e30])
def test_norm_in_8_bits_with_scales_at_the_ends_of_float32(P, dtype, channels, scale):
    """Entries of one size in a row whose length is a power of two: the norm is 1, and the outputs are the weights.  The scale is off by its rounding,
    half a step, which is all of a subnormal one's; the quotient by it is off by a correction's few roundings and by half a step of the format,
    2^-4 of the value, or 2^-10 among the smallest."""
    rng = np.random.default_rng(channels)
    x = torch.tensor(rng.choice([-1.0, 1.0], (3, channels))).to(dtype).to(DEV)
    w = np.float32(448 * scale * np.exp2(-12 * rng.random(channels)) * rng.choice([-1.0, 1.0], channels))
    w[5] = np.float32(448 * scale)
    q, scales, _ = P.norm_residual_float8(x, None, torch.tensor(w, device=DEV), eps=0.0)
    out, top = f64(x) * w.astype(np.float64), float(np.abs(w).max())
    assert (np.abs(f64(scales) - top / 448) <= np.maximum(U32 * top / 448, 2.0 ** -150)).all() and (f64(scales) > 0).all()
    v = np.clip(out / f64(scales), -448, 448)
    assert (np.abs(f64(q.float()) - v) <= np.maximum(2.0 ** -4 * np.abs(v), 2.0 ** -10) * (1 + 8 * U32) + 4 * U32 * np.abs(v)).all()
    assert (np.sign(f64(q.float())) * np.sign(out) >= 0).all() and (np.abs(f64(q.float())).max(-1) >= 448 * 2 / 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,stream", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
def test_norm_of_results_that_go_past_the_caches(P, dtype, stream):
    """Large results are stored in another way: the bits are those of the same rows in small calls."""
    rows, channels, part = 40000, 1024, 5000
    assert rows * channels * 2 * (2 if stream == torch.float32 else 1) * 2 > 144 << 20 > part * channels * 8
    gen = torch.Generator(DEV).manual_seed(1)
    make = lambda kind: torch.randn((rows, channels), generator=gen, device=DEV).to(kind)          # noqa: E731
    x, r, g, after, w = make(dtype), make(stream), make(dtype), make(stream), torch.randn(channels, generator=gen, device=DEV)
    out, total = P.norm_residual(x, r, w)
    dx, dr, _ = P.norm_residual_backprop(g, total, w, grad_total=after)
    wide = torch.cat((x, x), 1), torch.cat((r, r), 1), torch.cat((w, w))
    q, scales, sums = P.norm_residual_float8(*wide)
    for i in range(0, rows, part):
        at = slice(i, i + part)
        same_bits((out[at], total[at]), P.norm_residual(x[at], r[at], w))
        same_bits((dx[at], dr[at]), P.norm_residual_backprop(g[at], total[at], w, grad_total=after[at])[:2])
        same_bits((q[at], scales[at], sums[at]), P.norm_residual_float8(wide[0][at], wide[1][at], wide[2]))


# ---- the scan ----

def test_a_waves_accesses_to_shared_memory_are_kept_in_order():
    """The scan's waves exchange values through shared memory without a barrier.  The compiler may move a lane's reads across what other lanes
    write, to addresses that it can tell apart from the lane's own: between the phases of a tile (its values are put there; rows are gone through;
    pairs of channels are read), and before the next tile's, the sources have to hold it back."""
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pysiglib_amd", "csrc")
    phases = re.compile(r"(?P<put>col\.put(?:_shared)?\()|(?P<rows>col\.read_shared\()|(?P<pairs>const auto& row = in\[|\]\[col\.channel_of\(i\) \+ k\])"
                        r"|(?P<sync>wave_sync\(\);|__syncthreads\(\);)")
    seen = 0
    for name in ("seq_selective.hip", "seq_selective_backward.hip"):
        with open(os.path.join(here, name)) as fh:
            kernels = re.split(r"__global__ void", fh.read())[1:]
        for text in kernels:
            found = [m.lastgroup for m in phases.finditer(text)]
            if "put" not in found:
                continue
            seen += 1
            found = found[found.index("put"):]
            last = None
            for phase in found + ["put"]:           # the next tile's
                assert last in (None, "sync", phase) or phase == "sync", (name, text.split("(")[1].split()[-1], last, phase)
                last = phase
    assert seen == 3


def like_the_formula(got, want, bound, dtype, name):
    """The same infinities and NaN, and what is finite within its bound (where what it is bounded by is)."""
    got = f64(got).reshape(want.shape)
    assert (np.isnan(got) == np.isnan(want)).all() and (np.isposinf(got) == np.isposinf(want)).all() and (np.isneginf(got) == np.isneginf(want)).all(), name
    at = np.isfinite(want) & np.isfinite(bound)
    bound = rounded(np.where(at, want, 0.0), np.where(at, bound, 0.0), dtype)
    assert (np.abs(got[at] - want[at]) <= bound[at]).all(), name


def infinite_scan(P, t, starts, packed=True):
    """Outputs and gradients beside those of the formula: [(name, got, want, bound, type)]."""
    dtype, n = t["x"].dtype, len(starts) - 1
    shape = lambda v: v if packed else v.reshape(n, -1, *v.shape[1:])          # noqa: E731
    args = [shape(t["x"]), shape(t["delta"]), t["a"], shape(t["b"]), shape(t["c"])]
    options = dict(d=t["d"], z=shape(t["z"]), delta_bias=t["bias"], initial_state=t["h0"], offsets=whole_numbers(starts) if packed else None)
    got = (*P.selective_scan(*args, **options), *P.selective_scan_backprop(shape(t["g"]), *args, grad_final=t["gf"], **options))
    with np.errstate(all="ignore"):
        want, bound = scan_oracle(*(f64(t[k]) for k in ("x", "delta", "a", "b", "c", "d", "z", "bias", "h0")), starts, True, f64(t["g"]), f64(t["gf"]))
    kinds = (dtype, torch.float32, dtype, dtype, torch.float32, dtype, dtype, torch.float32, dtype, torch.float32, torch.float32)
    return list(zip(NAMES, got, want, bound, kinds))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("states", [1, 2, 3, 4, 5, 7, 8, 13, 16, 20, 33, 63, 64])
@pytest.mark.parametrize("which", ["x", "g", "h0", "gf", "delta"])
def test_selective_scan_of_infinities_with_any_number_of_states(P, dtype, states, which):
    """A channel's room may be for more states than it has: an infinity meets nothing there that the formula does not have."""
    starts = starts_of([20, 0, 33, 7])
    t = scan_inputs(dtype, 60, 4, 6, states, 2, seed=states, decays=0.3)
    at = (40, 3) if which in ("x", "g", "delta") else (2, 3, 0)
    t[which][at] = float("inf")
    for name, got, want, bound, kind in infinite_scan(P, t, starts):
        if which != "delta" or name not in ("ddelta", "dbias"):
            like_the_formula(got, want, bound, kind, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("states", [1, 2, 3, 4, 5, 7, 13, 16, 20, 33, 63])
@pytest.mark.parametrize("which", ["x", "h0", "delta"])
def test_selective_scan_step_of_infinities_with_any_number_of_states(P, dtype, states, which):
    t = scan_inputs(dtype, 5, 5, 6, states, 2, seed=states, decays=0.3)
    t[which][(2, 3) if which != "h0" else (2, 3, 0)] = float("inf")
    state = t["h0"].clone()
    y = P.selective_scan_step(t["x"], t["delta"], t["a"], t["b"], t["c"], state, d=t["d"], z=t["z"], delta_bias=t["bias"])
    with np.errstate(all="ignore"):
        want, bound = scan_oracle(*(f64(t[k]) for k in ("x", "delta", "a", "b", "c", "d", "z", "bias", "h0")), list(range(6)), True)
    like_the_formula(y, want[0], bound[0], dtype, "y")
    like_the_formula(state, want[1], bound[1], torch.float32, "state")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("states", [1, 4, 7, 16, 40])
@pytest.mark.parametrize("row", [0, 19, 40, 59])
def test_selective_scan_gradient_of_an_infinite_step(P, dtype, states, row):
    """softplus has the slope 1 there, and everything before the step is forgotten: the gradient is that of x's product alone."""
    t = scan_inputs(dtype, 60, 2, 6, states, 2, seed=states, decays=0.3)
    t["delta"][row, 3] = float("inf")
    for name, got, want, bound, kind in infinite_scan(P, t, [0, 20, 60]):
        like_the_formula(got, want, bound, kind, name)
        if name == "ddelta":
            assert np.isfinite(want[row, 3])
    t["delta"][row, 3] = float("nan")
    _, got, want, _, _ = infinite_scan(P, t, [0, 20, 60])[3]
    assert torch.isnan(got[row, 3]) and np.isnan(want[row, 3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels,states,groups", [(1024, 4, 1), (512, 8, 1), (256, 16, 1), (512, 16, 2), (128, 32, 1), (64, 64, 1), (256, 13, 1), (1024, 3, 1)])
def test_selective_scan_with_four_full_waves_to_a_block(P, dtype, channels, states, groups):
    """Channels of a group that fill four waves: their gradients come from blocks of four waves, which add up their sums over channels."""
    t = scan_inputs(dtype, 100, 2, channels, states, groups, seed=channels + states)
    check_scan(P, t, [0, 50, 100], False)
    check_scan(P, t, [0, 37, 100], True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,channels,states", [([1200], 6, 16), ([1043], 5, 20), ([300], 9, 4), ([330], 7, 3), ([700], 300, 8), ([1500, 0, 1500, 1600], 4, 16),
                                                     ([301, 2, 500], 3, 2)])
def test_selective_scan_of_many_segments(P, dtype, lengths, channels, states):
    """More than 64 segments to a sequence: several threads to a state join them."""
    starts = starts_of(lengths)
    t = scan_inputs(dtype, starts[-1], len(lengths), channels, states, 1, seed=channels)
    if len(lengths) == 1:
        check_scan(P, t, starts, False)
    check_scan(P, t, starts, True)


# ---- offsets that make no sense ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("states", [3, 16])
def test_offsets_that_do_not_ascend_write_only_into_the_outputs(P, dtype, states):
    """Every output and the workspace lies in a buffer that holds a mark before and behind it."""
    from pysiglib_amd import _loader as L
    rows, channels, code, margin = 500, 20, L.SEQUENCE_DTYPES[str(dtype).split(".")[1]], 65536
    rng = np.random.default_rng(states)
    buffers = []

    def inside(like=None, size=0):
        size = like.numel() * like.element_size() if like is not None else size
        whole = torch.full((size + 2 * margin,), 0x5A, dtype=torch.uint8, device=DEV)
        buffers.append((whole, size))
        part = whole[margin:margin + size]
        return part if like is None else part.view(like.dtype)

    def untouched(what):
        for whole, size in buffers:
            assert (whole[:margin] == 0x5A).all() and (whole[margin + size:] == 0x5A).all(), what
        buffers.clear()

    w, bias = numbers(rng, channels, 4), numbers(rng, channels)
    strides = (channels, channels, channels, 2 * states, 2 * states, 2 * states, 2 * states)
    for offsets in ([300, 100, 500, 0], [0, 500, 0, 500], [500, 0, 0, 0], [1 << 30, -1 << 30, 7, 1 << 30], [0, 500, 100, 200, 300, 50, 500, -7], [499, 1, 498, 2, 497, 3],
                    [7, 7, 7, 1, 1, 1, 500, 500, 9]):
        at, n = whole_numbers(offsets), len(offsets) - 1
        t = scan_inputs(dtype, rows, n, channels, states, 1, seed=1)
        state = numbers(rng, n, 3, channels, dtype=dtype)
        raw(L.CUSIG_CAUSAL_CONV, code, t["x"], w, bias, state, inside(t["x"]), inside(state), at, n, 0, rows, channels, 4, channels, True)
        untouched(("conv", offsets))
        size = L.CUSIG_CAUSAL_CONV_BACKPROP_WORKSPACE(rows, channels, 4)
        raw(L.CUSIG_CAUSAL_CONV_BACKPROP, code, t["g"], t["x"], w, bias, state, state, inside(t["x"]), inside(w), inside(bias), inside(state), at, n, 0, rows, channels, 4,
            channels, channels, True, inside(size=size), size)
        untouched(("conv gradients", offsets))
        inputs = [t[k] for k in ("x", "delta", "a", "b", "c", "d", "z", "bias")]
        size = L.CUSIG_SELECTIVE_SCAN_WORKSPACE(True, n, 0, rows, channels, states, 1)
        raw(L.CUSIG_SELECTIVE_SCAN, code, *inputs, t["h0"], inside(t["x"]), inside(t["h0"]), at, n, 0, rows, channels, states, 1, *strides, True, inside(size=size), size)
        untouched(("scan", offsets))
        size = L.CUSIG_SELECTIVE_SCAN_BACKPROP_WORKSPACE(True, n, 0, rows, channels, states, 1)
        grads = [inside(t[k]) for k in ("x", "delta", "a")] + [inside(t["b"].contiguous()) for _ in range(2)] + [inside(t[k]) for k in ("d", "z", "bias", "h0")]
        raw(L.CUSIG_SELECTIVE_SCAN_BACKPROP, code, t["g"], *inputs, t["gf"], t["h0"], *grads, at, n, 0, rows, channels, states, 1, channels, *strides, True,
            inside(size=size), size)
        untouched(("scan gradients", offsets))
