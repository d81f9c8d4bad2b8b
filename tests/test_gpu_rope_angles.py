"""What rq_rope_rows makes of an angle, by rows of (1, 0): its cosine and sine themselves.

Tolerance, u = 2^-24: the functions within one step (u for values up to 1), the remainder of the angle past f32 added
with one rounding (u / 2): 1.5 u; the angle itself, of three roundings in 64 bits, 2^-51 of it."""
import numpy as np
import pytest

from rusty_amd import Rope
from test_gpu_rope import pairs, run_rows

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("theta,most", [(10000.0, 1000), (10000.0, 200000), (500000.0, 2 ** 31 - 1)])
@pytest.mark.parametrize("backward", [False, True])
def test_sine_and_cosine(ctx, engine, layout, theta, most, backward):
    rot, tokens = 128, 4000
    positions = np.random.default_rng(1).integers(-most, most, tokens, endpoint=True)
    f, _ = Rope.frequencies_of(rot, theta)
    angle = np.asarray(positions, np.longdouble)[:, None] * np.asarray(f, np.longdouble)
    a, b = pairs(rot, layout)
    x = np.zeros((tokens, 1, rot), np.float32)
    x[..., a] = 1.0
    got = run_rows(ctx, engine, x, positions, Rope(ctx, rot, layout=layout, theta=theta), "f32", backward=backward)[:, 0]
    tol = 1.5 * U + np.abs(np.asarray(angle, np.float64)) * 2.0 ** -51
    for part, want in ((got[:, a], np.cos(angle)), (got[:, b], -np.sin(angle) if backward else np.sin(angle))):
        off = np.abs(part.astype(np.float64) - np.asarray(want, np.float64))
        print(f"worst {(off / U).max():.3f} u, of the tolerance {(off / tol).max():.3f}", flush=True)
        assert (off <= tol).all()
