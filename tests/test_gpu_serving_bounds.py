"""The attention over the 4-bit cache within its rigorous bound (attend_bound), on inputs that make the
bound narrow; test_attend_bound.py shows on the CPU what the bound rejects."""
import numpy as np
import pytest

import attend_bound as ab
import serving_ref as ref
from k3cuda import DevBuf, check
from test_gpu_serving import BF16, F32, SHAPES, Batch, Loop, same_pages, to_bf16

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


@pytest.mark.parametrize("H", [64, 16])
def test_attend_small_rotated_keys_under_large_latents(k3, H):
    """Queries on the rotated part alone, of keys so small that their way to fp16 rounds them."""
    kv, rope = 128, 64

    def edit(b, x):
        x *= np.float32(2.0 ** -7)
        x[:, kv:] *= np.float32(2.0 ** -8)
    B = Batch(k3, kv, rope, 64, [(40, 1), (300, 2)], seed=13, spread=0.0, edit=edit)
    q = np.zeros((3, H, kv + rope), np.float32)
    q[:, :, kv:] = np.random.default_rng(13).integers(-4, 5, (3, H, rope)) * 1024.0
    held(B, B.call(q, H, 3, BF16, F32, 1.0), q, 1.0, F32, False)


@pytest.mark.parametrize("qt", [BF16, F32])
@pytest.mark.parametrize("H", [16, 64])
def test_attend_queries_with_nan_and_infinity_are_nan(k3, H, qt):
    """They are NaN wherever they see a position, a single one too, whichever sign the products have, and
    in items that several CTAs share; the other rows are as without them."""
    kv, rope = 256, 32
    reqs = [(1, 1), (1, 1), (2, 1), (130, 2), (3000, 1), (1, 2)]
    B, g = grid_batch(k3, kv, rope, 64, reqs, 17)
    N = int(B.start[-1])
    q = ab.grid_queries(g, N, H, kv, rope, 1.0)
    clean = B.call(q, H, N, qt, F32, 2.0 ** -6)
    held(B, clean, q, 2.0 ** -6, F32, True)
    bad = np.zeros((N, H), bool)
    for n in range(N):
        for h, v in ((1, np.inf), (2, -np.inf), (5, np.nan), (7, np.inf)):
            q[n, h] = np.abs(q[n, h]) if h == 7 else q[n, h]
            q[n, h, (37 * n + 11 * h) % (kv + rope)] = v
            bad[n, h] = True
    q[:, 9], bad[:, 9] = -np.inf, True
    got = B.call(q, H, N, qt, F32, 2.0 ** -6)
    none = N - 2                                   # the last request's first row sees nothing
    assert (got[none] == 0).all()
    bad[none] = False
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("H", [8, 64])
def test_attend_columns_of_small_weights_alone(k3, H):
    """The last position has nearly all the weight and zeros in half of its columns, where what is left are
    weights of 2^-20 to 2^-34, which fp16 holds to 2^-32."""
    kv, rope = 128, 16
    g = np.random.default_rng(19)

    def edit(b, x):
        x[:] = ab.grid_rows(g, len(x), kv, rope)
        x[:, kv:] = 0
        x[:, kv] = -14 - np.arange(len(x)) / 2.0
        x[-1, kv] = 0
        x[-1, :kv:2] = 0
    B = Batch(k3, kv, rope, 16, [(20, 1)], seed=19, edit=edit)
    q = np.zeros((1, H, kv + rope), np.float32)
    q[:, :, kv] = 1.0
    got = B.call(q, H, 1, BF16, F32, 1.0)
    held(B, got, q, 1.0, F32, True)
    assert (got[0, :, :kv:2] != 0).any()


class Bf16Loop(Loop):
    """The serving step with bf16 queries, which the kernel takes as they are."""

    def __init__(self, lib, g, **kw):
        super().__init__(lib, g, **kw)
        self.q16 = DevBuf(self.N * self.H * self.w * 2)

    def calls(self):
        lib, d = self.lib, {k: b.ptr for k, b in self.dev.items()}
        check(lib.k3d_page_plan(self.pages.p, d["len"], d["new"], self.B, self.N, d["start"], d["kvl"], d["pos"],
                                d["slots"], d["status"]))
        check(lib.k3d_cache4_store(self.shape, self.pool.ptr, d["x"], F32, self.w, d["slots"], self.N))
        check(lib.k3d_mla_attend4(d["o"], F32, self.q16.ptr, BF16, self.shape, self.pool.ptr, self.pages.t.ptr, 12, d["start"],
                                  d["kvl"], self.B, self.N, self.H, 0.07, self.ws.ptr, self.nws))


@pytest.mark.parametrize("H,kv,rope", [(16, 256, 32), (64, 512, 64)])
def test_serving_steps_position_by_position(k3, H, kv, rope):
    """plan -> store -> attend over steps that keep some of their drafts, ragged and with a request that
    brings nothing: every element within the bound, which a position too many or too few leaves."""
    g = np.random.default_rng(61)
    L = Bf16Loop(k3, g, B=5, K=3, H=H, kv=kv, rope=rope)
    lens = np.zeros(L.B, int)
    known = [(np.zeros((0, L.w)), np.zeros(0, int)) for _ in range(L.B)]
    for step in range(7):
        new = [4, 1, 3, 0 if step == 2 else 2, 4]
        h = L.inputs(lens, new)
        L.q16.upload(to_bf16(h["q"]))
        L.calls()
        check(k3.k3d_sync())
        code, start, kvl, _, slots = L.host.plan(lens.tolist(), new, L.N)
        assert code == 0
        same_pages(L.pages, L.host)
        o = L.dev["o"].download(np.float32, (L.N, H, kv))
        fields, value = ref.quantise(h["x"], kv)
        e = fields[3].astype(int) - 127
        for b in range(L.B):
            r = slice(start[b], start[b + 1])
            v = np.concatenate([known[b][0][:lens[b]], value[r]])
            x = np.concatenate([known[b][1][:lens[b]], e[r]])
            known[b] = (v, x)
            if new[b]:
                want, tol = ab.bound(h["q"][r], v, x, kv, float(np.float32(0.07)), new[b])
                assert (np.abs(o[r] - want) <= tol).all(), (step, b)
                if lens[b] + new[b] > 1:
                    lost = ab.without(h["q"][r], v, kv, 0.07, new[b], 0)
                    assert (np.abs(lost - want) > tol).any(), "the bound sees the first position"
        lens = lens + np.minimum(new, g.integers(1, 4, L.B))          # some of the drafts are kept
        if step == 4:
            lens[1] = 0                                               # a request ended, another in its place
