"""rq_qmatmul_loras: the types that test_gpu_loras.py does not combine; the tolerances are those derived there."""
import numpy as np
import pytest

from test_gpu_loras import KIND, U, adapters, case, check, run, truth, weight

pytestmark = pytest.mark.gpu

OTHER_TYPES = [("f16", "f16", "f32"), ("f32", "f16", "f32"), ("f32", "f32", "f16"), ("f16", "f32", "f16")]


@pytest.mark.parametrize("x_t,y_t,a_t", OTHER_TYPES)
@pytest.mark.parametrize("form", ["rowwise8", "affine8"])
@pytest.mark.parametrize("m,n,k,rank", [(1, 256, 512, 16), (2, 136, 1024, 70), (5, 256, 512, 40), (33, 264, 512, 21), (256, 131, 512, 9),
                                        (257, 131, 512, 33), (300, 256, 512, 16), (300, 264, 1024, 100)])
def test_types(ctx, engine, x_t, y_t, a_t, form, m, n, k, rank):
    """fp16 rows of 3 and more take affine weights u s + b rounded to fp16, half a step of each: 2^-11 P, within the
    2^-10 P of `rounded`."""
    if form == "rowwise8" or m <= 2 or m > 16 or x_t == "f32":
        return case(ctx, engine, m + rank, m, n, k, 4, rank, form, x_t, y_t, a_t, some_ranks=rank == 40)
    g = np.random.default_rng(m + rank)
    w, w64 = weight(ctx, g, n, k, form)
    a, b = adapters(g, 4, rank, k, n, a_t)
    x, f, ids = g.standard_normal((m, k)).astype(np.float16), (g.random(4) + 0.5).astype(np.float32), g.integers(-1, 4, m)
    want, tol = truth(x, w64, a, b, f, ids, [rank] * 4, y_t, True)
    check(run(ctx, engine, x, w, a, b, f, ids, None, x_t, y_t, a_t), want, tol, f"{m}x{n}x{k} {x_t}/{y_t}/{a_t}")


@pytest.mark.parametrize("x_t,y_t,a_t", OTHER_TYPES)
@pytest.mark.parametrize("m,n,k,rank", [(1, 256, 512, 16), (2, 136, 1024, 70), (5, 256, 512, 40), (33, 264, 512, 21), (300, 256, 512, 16)])
def test_types_of_4_bit_codes(ctx, engine, x_t, y_t, a_t, m, n, k, rank):
    """Up to 48 rows the products are formed with codes + 16 and sums of x (test_gpu_linear4.py):
    (k / 32 + 64) u + 2^-21 of sum |x| s (u + 40), s (u + 40) below 55 of the
    largest scale; past 16 each product loses half an fp16 step of the weight, and of an f32 row."""
    g = np.random.default_rng(m + rank)
    w, w64 = weight(ctx, g, n, k, "affine4")
    a, b = adapters(g, 4, rank, k, n, a_t)
    x = g.standard_normal((m, k)).astype(KIND[x_t][0])
    f, ids = (g.random(4) + 0.5).astype(np.float32), g.integers(-1, 4, m)
    want, tol = truth(x, w64, a, b, f, ids, [rank] * 4, y_t, m > 16)
    tol += (((k / 32 + 64) * U + 2.0 ** -21) * 55 * 0.15 / 16 + 2.0 ** -25) * np.abs(x.astype(np.float64)).sum(1, keepdims=True)
    check(run(ctx, engine, x, w, a, b, f, ids, None, x_t, y_t, a_t), want, tol, f"{m}x{n}x{k} {x_t}/{y_t}/{a_t}")


@pytest.mark.parametrize("x_t,y_t,a_t", OTHER_TYPES)
@pytest.mark.parametrize("form,m,n,k", [("rowwise8", 1100, 5640, 192), ("affine8", 700, 3712, 128)])
def test_types_of_large_products(ctx, engine, x_t, y_t, a_t, form, m, n, k):
    g = np.random.default_rng(m)
    case(ctx, engine, m, m, n, k, 5, 24, form, x_t, y_t, a_t, ids=np.repeat(g.integers(-1, 5, m // 90 + 1), 90)[:m])
