"""The attention over the 4-bit cache within its rigorous bound (attend_bound), on inputs that make the
bound narrow; test_attend_bound.py shows on the CPU what the bound rejects."""
import numpy as np
import pytest

import attend_bound as ab
from test_gpu_serving import BF16, F32, SHAPES, Batch

pytestmark = pytest.mark.gpu


def held(B, got, q, scale, ot, exact):
    """Every request's result within the bound; the largest share of it that was used."""
    used = 0.0
    for b, (k, n) in enumerate(B.reqs):
        if n == 0:
            continue
        s0 = int(B.start[b])
        want, tol = ab.bound(q[s0:s0 + n], B.values[b], B.exps[b], B.kv, scale, n, "f32" if ot == F32 else "bf16", exact)
        err = np.abs(got[s0:s0 + n] - want)
        assert (err <= tol).all(), (b, float((err / np.maximum(tol, 1e-300)).max()))
        used = max(used, float((err / np.maximum(tol, 1e-300)).max()))
    return used


def grid_batch(k3, kv, rope, page, reqs, seed, lift=None):
    g = np.random.default_rng(seed)

    def edit(b, x):
        x[:] = ab.grid_rows(g, len(x), kv, rope, lift)
    B = Batch(k3, kv, rope, page, reqs, seed=seed, edit=edit)
    for b in range(len(reqs)):
        assert len(B.exps[b]) == 0 or ((B.exps[b] >= -16).all() and (B.exps[b] <= -2).all())
    return B, g


@pytest.mark.parametrize("qt,ot", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("case", SHAPES)
def test_attend_exact_products(k3, case, qt, ot):
    """Scores without a rounding, so that every position counts against the weights' half steps alone."""
    kv, rope, page, H, reqs = case
    B, g = grid_batch(k3, kv, rope, page, reqs, kv + H)
    n = int(B.start[-1])
    q = ab.grid_queries(g, n, H, kv, rope, 1.0)
    held(B, B.call(q, H, n, qt, ot, 2.0 ** -6), q, 2.0 ** -6, ot, True)


@pytest.mark.parametrize("case", SHAPES)
def test_attend_fp32_queries(k3, case):
    """fp32 queries against the definition for the queries as they are taken: fp16 in units of the row."""
    kv, rope, page, H, reqs = case
    B = Batch(k3, kv, rope, page, reqs, seed=kv + H)
    n = int(B.start[-1])
    q = B.queries(H, n, 1.0, F32)
    scale = float(np.float32(0.07))
    held(B, B.call(q, H, n, F32, F32, 0.07), q, scale, F32, False)


@pytest.mark.parametrize("gain", [1.0, 8.0, 64.0])
@pytest.mark.parametrize("kv,rope,H,n", [(512, 64, 64, 2), (512, 64, 16, 1), (256, 32, 24, 3), (128, 16, 100, 1)])
def test_attend_moving_maximum(k3, kv, rope, H, n, gain):
    """Tiles whose maxima jump and fall back, with exact scores: each rescaling of the accumulator counts."""
    reqs = [(64 * len(ab.LIFT) - 9, n), (64 * len(ab.LIFT) * 3 + 5, n), (200, 1)]
    B, g = grid_batch(k3, kv, rope, 64, reqs, kv + H, ab.LIFT)
    N = int(B.start[-1])
    q = ab.grid_queries(g, N, H, kv, rope, gain, True)
    held(B, B.call(q, H, N, BF16, F32, 2.0 ** -4), q, 2.0 ** -4, F32, True)
