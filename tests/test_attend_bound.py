"""The bound that the attention is held to (attend_bound) tells right from wrong: results with a
mistake, made here from the definition, are outside it, and the definition itself, with the kernel's
roundings, is inside."""
import numpy as np
import pytest

import attend_bound as ab
import serving_ref as ref


def outside(got, want, tol):
    return bool((np.abs(got - want) > tol).any())


def values(x, kv):
    fields, value = ref.quantise(x, kv)
    return value, fields[3].astype(int) - 127


def as_the_kernel_rounds(q, v, kv, scale, n):
    """fp32 scores, fp16 weights over an unrounded sum."""
    q = ab.rounded(q)
    out = np.zeros((n, q.shape[1], kv))
    for j in range(n):
        seen = max(0, len(v) - n + j + 1)
        if seen:
            s = (q[j].astype(np.float32) @ v[:seen].T.astype(np.float32) * np.float32(scale)).astype(np.float64)
            p = np.exp(s - s.max(1, keepdims=True)) * 128
            out[j] = (p.astype(np.float16).astype(np.float64) @ v[:seen, :kv]) / p.sum(1, keepdims=True)
    return out


def test_grid_rows_are_held_as_they_are():
    g = np.random.default_rng(0)
    for kv, rope in ((512, 64), (128, 16), (256, 0)):
        x = ab.grid_rows(g, 300, kv, rope, ab.LIFT if rope else None)
        v, e = values(x, kv)
        assert np.array_equal(v, x) and (e >= -16).all() and (e <= -2).all()
        q = ab.grid_queries(g, 2, 3, kv, rope, 4.0, True) if rope else ab.grid_queries(g, 2, 3, kv, rope, 4.0)
        assert np.array_equal(ab.rounded(q), q)


@pytest.mark.parametrize("kv,rope,L,n,gain", [(512, 64, 200, 1, 1.0), (512, 64, 130, 4, 1.0), (256, 32, 65, 3, 1.0),
                                              (128, 0, 33, 2, 2.0)])
def test_lost_and_shifted_positions_are_outside(kv, rope, L, n, gain):
    g = np.random.default_rng(L)
    x, q = ab.grid_rows(g, L, kv, rope), ab.grid_queries(g, n, 8, kv, rope, gain)
    v, e = values(x, kv)
    want, tol = ab.bound(q, v, e, kv, 2.0 ** -6, n, "bf16", True)
    assert not outside(as_the_kernel_rounds(q, v, kv, 2.0 ** -6, n), want, tol)
    for wrong in (0 * want, -want, 5 * want):
        assert outside(wrong, want, tol)
    for t in range(L - n + 1):
        assert outside(ab.without(q, v, kv, 2.0 ** -6, n, t), want, tol), t
    for by in (-1, 1):
        if n > 1 or by < 0:
            assert outside(ab.shifted(q, v, kv, 2.0 ** -6, n, by), want, tol)


@pytest.mark.parametrize("fp32", [False, True])
def test_lost_positions_are_outside_for_any_numbers(fp32):
    """Rows and queries as they come: the sums' own roundings take most of the bound."""
    g = np.random.default_rng(5)
    for kv, rope, L, n in ((512, 64, 129, 2), (512, 64, 64, 1), (128, 16, 70, 3)):
        x = (g.standard_normal((L, kv + rope)) * np.exp(0.5 * g.standard_normal((L, 1)))).astype(np.float32)
        q = g.standard_normal((n, 8, kv + rope)).astype(np.float32)
        if not fp32:
            q = ((q.view(np.uint32) + 0x8000) & 0xffff0000).view(np.float32)
        v, e = values(x, kv)
        want, tol = ab.bound(q, v, e, kv, 0.07, n)
        assert not outside(as_the_kernel_rounds(q, v, kv, 0.07, n), want, tol)
        for t in range(L - n + 1):
            assert outside(ab.without(ab.rounded(q), v, kv, 0.07, n, t), want, tol), t
        for wrong in (0 * want, -want, 5 * want):
            assert outside(wrong, want, tol)


@pytest.mark.parametrize("gain", [1.0, 8.0])
def test_a_skipped_rescale_is_outside(gain):
    g = np.random.default_rng(6)
    kv, rope, L, n = 512, 64, 64 * len(ab.LIFT) - 9, 2
    x, q = ab.grid_rows(g, L, kv, rope, ab.LIFT), ab.grid_queries(g, n, 4, kv, rope, gain, True)
    v, e = values(x, kv)
    want, tol = ab.bound(q, v, e, kv, 2.0 ** -4, n, "f32", True)
    assert not outside(as_the_kernel_rounds(q, v, kv, 2.0 ** -4, n), want, tol)
    for wrong in (0 * want, -want, 5 * want, ab.no_rescale(q, v, kv, 2.0 ** -4, n)):
        assert (np.abs(wrong - want) > tol).reshape(n * 4, kv).any(1).all(), "in every row"
    # one move alone that is left out is seen where what came before it still counts
    if gain == 1.0:
        assert all(outside(ab.no_rescale(q, v, kv, 2.0 ** -4, n, k), want, tol) for k in range(3))
    s = q.astype(np.float64) @ v.T * 2.0 ** -4
    top = s[0].argmax(1)
    for h in range(4):
        assert outside(ab.without(q, v, kv, 2.0 ** -4, n, int(top[h])), want, tol)


def test_small_rotated_keys_under_large_latents():
    """Their rounding is in the bound: without the term, keys that the kernel loses would be outside,
    and with it a result that drops the rotated part altogether still is."""
    g = np.random.default_rng(7)
    kv, rope, L, n = 128, 64, 40, 1
    x = (g.standard_normal((L, kv + rope)) * 2.0 ** -7).astype(np.float32)
    x[:, kv:] *= np.float32(2.0 ** -8)
    q = np.zeros((n, 4, kv + rope), np.float32)
    q[:, :, kv:] = g.integers(-4, 5, (n, 4, rope)) * 1024.0
    v, e = values(x, kv)
    want, tol = ab.bound(q, v, e, kv, 1.0, n)
    res = e - np.clip(e, -16, -2)
    assert (e < -2).all()
    # the rotated keys as the kernel has them, in units of 2^(res - 2)
    up = np.ldexp(v[:, kv:], -e[:, None]).astype(np.float64)
    k16 = np.ldexp(up, np.clip(e + 2, -14, 0)[:, None]).astype(np.float16).astype(np.float64)
    w = v.copy()
    w[:, kv:] = np.ldexp(k16, (res - 2)[:, None])
    assert (np.abs(w[:, kv:] - v[:, kv:]) <= np.ldexp(1.0, -27 + res)[:, None]).all() and (w != v).any()
    s = q[0].astype(np.float64) @ w.T
    p = np.exp(s - s.max(1, keepdims=True))
    got = (p / p.sum(1, keepdims=True)) @ v[:, :kv]
    assert not outside(got[None], want, tol)
    w[:, kv:] = 0
    s = q[0].astype(np.float64) @ w.T
    p = np.exp(s - s.max(1, keepdims=True))
    assert outside(((p / p.sum(1, keepdims=True)) @ v[:, :kv])[None], want, tol)
