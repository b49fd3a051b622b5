"""Values at the ends of the number formats, and places of the state space layers that only some sizes reach (see test_state_space.py,
whose formulas, bounds and helpers these are)."""
import os
import re

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_state_space import DEV, P, TYPES, f64, numbers  # noqa: E402,F401


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
