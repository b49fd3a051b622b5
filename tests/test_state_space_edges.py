"""Values at the ends of the number formats, and places of the state space layers that only some sizes reach (see test_state_space.py,
whose formulas, bounds and helpers these are)."""
import os
import re

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_state_space import DEV, NAMES, P, TYPES, f64, numbers, rounded, scan_inputs, scan_oracle, starts_of, whole_numbers  # noqa: E402,F401


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
