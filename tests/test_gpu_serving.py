"""Serving operators on the GPU against their definitions in 64 bits (serving_ref)."""
import ctypes

import numpy as np
import pytest

import k3cuda
import serving_ref as ref
from k3cuda import DevBuf, check

pytestmark = pytest.mark.gpu

F32, BF16 = k3cuda.K3D_DT_F32, k3cuda.K3D_DT_BF16


def to_bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def i32(v):
    return DevBuf.from_array(np.ascontiguousarray(v, np.int32).reshape(-1))


# -------------------------------------------------------------------- store and load ----
def store(lib, shape, pool, x, slots, dtype=F32, ld=None):
    n, w = x.shape
    ld = ld or w
    host = np.full((n, ld), 7, np.float32 if dtype == F32 else np.uint16)
    host[:, :w] = x if dtype == F32 else to_bf16(x)
    X, S = DevBuf.from_array(host), i32(slots)
    check(lib.k3d_cache4_store(shape, pool.ptr, X.ptr, dtype, ld, S.ptr, n))
    check(lib.k3d_sync())


def load(lib, shape, pool, slots, w, dtype=F32, ld=None, fill=5.0):
    n = len(slots)
    ld = ld or w
    host = np.full((n, ld), fill, np.float32)
    O, S = DevBuf.from_array(host if dtype == F32 else to_bf16(host)), i32(slots)
    check(lib.k3d_cache4_load(shape, pool.ptr, O.ptr, dtype, ld, S.ptr, n))
    check(lib.k3d_sync())
    out = O.download(np.float32 if dtype == F32 else np.uint16, (n, ld))
    return (out if dtype == F32 else from_bf16(out))


def rows(g, n, w, spread=2.0):
    return (g.standard_normal((n, w)) * np.exp(spread * g.standard_normal((n, 1)))).astype(np.float32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kv,rope,page,n,pad", [(512, 64, 64, 1, 0), (512, 64, 64, 130, 0), (512, 48, 16, 33, 3),
                                                (256, 16, 32, 70, 1), (128, 0, 1024, 257, 0), (384, 32, 48, 9, 8)])
def test_rows_round_trip(k3, kv, rope, page, n, pad, dtype):
    g = np.random.default_rng(kv + n)
    w = kv + rope
    n_pages = -(-n // page) + 3
    shape = k3cuda.K3dCache4(kv, rope, page, n_pages)
    pool = DevBuf(k3.k3d_cache4_bytes(shape))
    x = rows(g, n, w)
    x[0] = 0.0
    if n > 8:
        x[1, :kv] = 0.0                                    # only the rope part
        x[2, kv:] = 0.0
        x[3] *= np.float32(1e-30)
        x[4] *= np.float32(1e30)
        x[5, 16:32] *= np.float32(1e-9)                    # a block far below its row
        x[6, ::16] = 2688.0                                # the largest value of the unit
        x[7] = np.float32(2.0) ** -149                     # the smallest fp32 there is
    if dtype == BF16:
        x = from_bf16(to_bf16(x))
    slots = g.permutation(n_pages * page)[:n].astype(np.int32)
    if n > 20:
        slots[10::7] = -1
    check(k3.k3d_memset(pool.ptr, 0xff, pool.nbytes))
    store(k3, shape, pool, x, slots, dtype, w + pad)
    fields, value = ref.quantise(x, kv)
    want = np.full((n_pages, ref.page_bytes(kv, rope, page)), 0xff, np.uint8)
    ref.put_rows(want, kv, rope, page, slots, fields)
    got = pool.download(np.uint8, want.shape)
    assert np.array_equal(got, want), "bytes of the pool, and nothing outside the slots"
    out = load(k3, shape, pool, slots, w, F32, w + pad)
    keep = slots >= 0
    assert np.array_equal(out[keep, :w], value[keep].astype(np.float32))
    assert (out[~keep] == 5.0).all() and (out[:, w:] == 5.0).all(), "rows and columns outside are left as they were"
    # bf16 holds the latent part exactly and rounds the fp16 rope part
    b = load(k3, shape, pool, slots, w, BF16, w + pad)
    assert np.array_equal(b[keep, :w], from_bf16(to_bf16(value[keep])))


def test_rows_with_nan_and_infinity_are_nan(k3):
    kv, rope, page = 512, 64, 64
    shape = k3cuda.K3dCache4(kv, rope, page, 1)
    pool = DevBuf(k3.k3d_cache4_bytes(shape))
    g = np.random.default_rng(1)
    x = rows(g, 6, 576)
    x[1, 3], x[2, 575], x[3, 511], x[4, 512] = np.nan, np.inf, -np.inf, np.nan
    store(k3, shape, pool, x, np.arange(6))
    out = load(k3, shape, pool, np.arange(6), 576)
    bad = np.isnan(out)
    assert bad[1:5].all() and not bad[0].any() and not bad[5].any()


def test_slots_outside_the_pool_are_refused(k3):
    shape = k3cuda.K3dCache4(512, 64, 16, 2)
    pool = DevBuf(k3.k3d_cache4_bytes(shape))
    check(k3.k3d_memset(pool.ptr, 0, pool.nbytes))
    X, S = DevBuf.from_array(np.ones((3, 576), np.float32)), i32([0, 32, -2])
    check(k3.k3d_cache4_store(shape, pool.ptr, X.ptr, F32, 576, S.ptr, 3))
    assert k3.k3d_sync() == k3cuda.K3D_EDEVICE
    code, site = ctypes.c_int(), ctypes.c_int()
    k3.k3d_device_error(ctypes.byref(code), ctypes.byref(site))
    assert code.value == k3cuda.K3D_EBOUND
    k3.k3d_clear_status()
    got = load(k3, shape, pool, [0, 1], 576)
    want = ref.quantise(np.ones((1, 576), np.float32), 512)[1]
    assert np.array_equal(got[:1], want.astype(np.float32)) and (got[1] == 0.0).all()


# -------------------------------------------------------------------------- attention ----
class Batch:
    """Requests (kv_len, n_new) with their rows stored, and the oracle's values."""

    def __init__(self, lib, kv, rope, page, reqs, seed, spread=0.5, n_extra=3, first_page=0, edit=None):
        g = np.random.default_rng(seed)
        self.lib, self.kv, self.w, self.page, self.reqs = lib, kv, kv + rope, page, reqs
        need = [-(-k // page) for k, _ in reqs]
        n_pages = sum(need) + n_extra + first_page
        self.shape = k3cuda.K3dCache4(kv, rope, page, n_pages)
        self.pool = DevBuf(lib.k3d_cache4_bytes(self.shape))
        check(lib.k3d_memset(self.pool.ptr, 0xff, self.pool.nbytes))     # NaN wherever nothing is stored
        ids = first_page + g.permutation(n_pages - first_page)
        self.max_pages = max(need + [1]) + 1
        self.table = np.full((len(reqs), self.max_pages), -1, np.int32)
        self.values, self.exps, at = [], [], 0
        for b, (k, _) in enumerate(reqs):
            self.table[b, :need[b]] = ids[at:at + need[b]]
            at += need[b]
            x = rows(g, k, self.w, spread)
            if edit:
                edit(b, x)
            t = np.arange(k)
            slots = (self.table[b, t // page] * page + t % page).astype(np.int32)
            if k:
                store(lib, self.shape, self.pool, x, slots)
            fields, value = ref.quantise(x, kv)
            self.values.append(value)
            self.exps.append(fields[3].astype(int) - 127)
        self.start = np.concatenate([[0], np.cumsum([n for _, n in reqs])]).astype(np.int32)
        self.bufs = [i32(self.table), i32(self.start), i32([k for k, _ in reqs])]
        self.g = g

    def queries(self, H, N, gain, qt):
        q = (self.g.standard_normal((N, H, self.w)) * gain).astype(np.float32)
        return from_bf16(to_bf16(q)) if qt == BF16 else q

    def call(self, q, H, N, qt, ot, scale, out=None, sync=True):
        lib = self.lib
        Q = DevBuf.from_array(to_bf16(q) if qt == BF16 else q)
        O = out or DevBuf.from_array(np.full((N, H, self.kv), 9, np.float32) if ot == F32 else
                                     to_bf16(np.full((N, H, self.kv), 9, np.float32)))
        n = lib.k3d_mla_attend4_ws_bytes(self.shape, len(self.reqs), N, H)
        WS = DevBuf(n)
        check(lib.k3d_memset(WS.ptr, 0xff, n))
        T, R, K = self.bufs
        check(lib.k3d_mla_attend4(O.ptr, ot, Q.ptr, qt, self.shape, self.pool.ptr, T.ptr, self.max_pages, R.ptr, K.ptr,
                                  len(self.reqs), N, H, scale, WS.ptr, n))
        if sync:
            check(lib.k3d_sync())
        got = O.download(np.float32 if ot == F32 else np.uint16, (N, H, self.kv))
        return got if ot == F32 else from_bf16(got)

    def compare(self, got, q, H, qt, ot, scale):
        """Elementwise: half a step of the result's type, the weights' rounding to fp16 (2^-11 of
        sum p|v|), q's rounding to fp16 where it is fp32 and the fp32 sums of 576 products
        (both as a change of the scores), and 2^-16 of sum p|v| for exp2 and the running sums.
        Small weights: the kernel rounds P = 2^(a - m + 7), a = s + e (base 2), m <= max a, to
        fp16, whose steps stop at 2^-24, so P is off by up to 2^-25 however small it is. With
        L = sum 2^(s - m + 7) >= 2^(7 - e*), e* the unit of the position of max a, the result
        sum P (v 2^-e) / L moves by at most 2^-32 sum |v| 2^(e* - e)."""
        eps = 2.0 ** -8 if ot == BF16 else 2.0 ** -24
        for b, (k, n) in enumerate(self.reqs):
            v = self.values[b]
            s0 = int(self.start[b])
            want = ref.attend(q[s0:s0 + n], v, self.kv, scale, n)
            for j in range(n):
                seen = max(0, k - n + j + 1)
                if seen == 0:
                    assert (got[s0 + j] == 0).all()
                    continue
                x = q[s0 + j].astype(np.float64)
                s = x @ v[:seen].T * scale
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                mag = p @ np.abs(v[:seen, :self.kv])
                ds = scale * (np.abs(x) @ np.abs(v[:seen]).T).max(1) * ((2.0 ** -11 if qt == F32 else 0.0) + 576 * 2.0 ** -24)
                top = self.exps[b][(s * np.log2(np.e) + self.exps[b][:seen]).argmax(1)]
                low = 2.0 ** -32 * np.exp2(top[:, None]) * (np.abs(v[:seen, :self.kv]) * np.exp2(-1.0 * self.exps[b][:seen, None])).sum(0)
                tol = eps * np.abs(want[j]) + (2.0 ** -11 + 2.0 ** -16 + np.expm1(2 * ds))[:, None] * mag + low
                err = np.abs(got[s0 + j] - want[j])
                assert (err <= tol).all(), (b, j, float((err / tol).max()))


SHAPES = [
    # kv, rope, page, heads, (kv_len, n_new)
    (512, 64, 64, 64, [(1, 1)]),
    (512, 64, 64, 64, [(63, 1), (64, 1), (65, 1)]),
    (512, 64, 16, 8, [(17, 1), (0, 0), (5, 5), (100, 3)]),
    (512, 64, 128, 16, [(3000, 1), (129, 2), (1, 1)]),
    (512, 64, 48, 64, [(200, 4), (49, 1)]),
    (256, 32, 32, 24, [(33, 2), (1, 1), (200, 7)]),
    (128, 0, 16, 5, [(70, 3), (16, 1)]),
    (384, 48, 64, 33, [(130, 1), (64, 2)]),
    (512, 64, 64, 128, [(300, 2)]),
    (512, 16, 64, 96, [(100, 1), (7, 3)]),
    (256, 64, 64, 1, [(500, 1), (20, 20)]),
    (512, 64, 64, 64, [(2, 4), (1, 3)]),                    # rows that see nothing
    (512, 64, 1024, 12, [(2500, 70)]),
]


@pytest.mark.parametrize("qt,ot", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("case", SHAPES)
def test_attend(k3, case, qt, ot):
    kv, rope, page, H, reqs = case
    B = Batch(k3, kv, rope, page, reqs, seed=kv + H)
    n = int(B.start[-1])
    scale = 0.07
    q = B.queries(H, n + 2, 1.0, qt)
    got = B.call(q, H, n + 2, qt, ot, scale)
    B.compare(got, q, H, qt, ot, scale)
    assert (got[n:] == 9.0).all(), "rows behind the last request are left as they were"


@pytest.mark.parametrize("gain", [0.0, 25.0, 300.0])
def test_attend_flat_and_steep_scores(k3, gain):
    """Scores that are all equal, and scores hundreds apart whose maximum keeps moving."""
    B = Batch(k3, 512, 64, 64, [(700, 2), (130, 1)], seed=3, spread=1.5)
    q = B.queries(64, 3, gain, BF16)
    got = B.call(q, 64, 3, BF16, F32, 0.07)
    B.compare(got, q, 64, BF16, F32, 0.07)


def test_attend_rising_scores(k3):
    """Every position scores above the last one, so each tile moves the maximum."""
    def edit(b, x):
        x[:] = np.abs(x) * (np.arange(1, len(x) + 1)[:, None] / len(x)).astype(np.float32)
    B = Batch(k3, 512, 64, 64, [(1500, 1)], seed=4, spread=0.0, edit=edit)
    q = np.abs(B.queries(16, 1, 3.0, BF16))
    got = B.call(q, 16, 1, BF16, F32, 0.07)
    B.compare(got, q, 16, BF16, F32, 0.07)


def test_attend_rows_of_far_units(k3):
    """Neighbouring positions whose rows differ by 2^60 in size."""
    def edit(b, x):
        x[1::3] *= np.float32(2.0 ** -30)
        x[2::3] *= np.float32(2.0 ** 30)
    B = Batch(k3, 256, 32, 16, [(90, 1)], seed=5, spread=0.0, edit=edit)
    q = B.queries(8, 1, 2.0 ** -30, F32)
    got = B.call(q, 8, 1, F32, F32, 0.07)
    B.compare(got, q, 8, F32, F32, 0.07)


def test_attend_nan_in_a_later_draft_stays_there(k3):
    def edit(b, x):
        x[-1, 5] = np.nan
    B = Batch(k3, 512, 64, 64, [(100, 3)], seed=6, edit=edit)
    q = B.queries(64, 3, 1.0, BF16)
    got = B.call(q, 64, 3, BF16, F32, 0.07)
    assert not np.isnan(got[:2]).any() and np.isnan(got[2]).all()


def test_attend_past_32_bit_offsets(k3):
    """Pages above 4 GiB of the pool."""
    page = 128
    first = (1 << 32) // ref.page_bytes(512, 64, page) + 5
    B = Batch(k3, 512, 64, page, [(300, 1), (40, 2)], seed=7, first_page=first)
    q = B.queries(16, 3, 1.0, BF16)
    got = B.call(q, 16, 3, BF16, F32, 0.07)
    B.compare(got, q, 16, BF16, F32, 0.07)


def test_attend_many_ragged_requests(k3):
    g = np.random.default_rng(8)
    reqs = [(int(g.integers(1, 400)), 1) for _ in range(90)] + [(0, 0)] * 3 + [(40, 5)]
    B = Batch(k3, 256, 32, 16, reqs, seed=8)
    n = int(B.start[-1])
    q = B.queries(16, n, 1.0, BF16)
    got = B.call(q, 16, n, BF16, BF16, 0.07)
    B.compare(got, q, 16, BF16, BF16, 0.07)


@pytest.mark.parametrize("kv,rope,H,reqs", [
    (512, 64, 64, [(2000, 1)]), (512, 64, 64, [(3000, 1)]), (512, 64, 64, [(9000, 2), (300, 1)]),   # 16, 32, 64 rows to an item
    (512, 64, 24, [(1200, 3), (65, 1)]), (512, 64, 24, [(2600, 3), (0, 0), (65, 1)]), (512, 64, 24, [(8000, 5), (65, 1)]),
    (128, 16, 100, [(600, 1), (1, 1)]), (256, 0, 100, [(1800, 1), (64, 1)]), (128, 16, 100, [(5000, 2), (64, 1)]),
    (384, 64, 17, [(900, 4)]), (512, 64, 8, [(400, 9), (3, 3)]), (512, 64, 64, [(64, 2)] * 9 + [(1500, 1)]),
    (512, 64, 32, [(64, 2)] * 9 + [(1500, 2)]), (512, 64, 32, [(640, 2)] * 9 + [(1500, 2)]),
])
def test_attend_few_items(k3, kv, rope, H, reqs):
    """Small batches, whose items have fewer rows while that finds idle SMs."""
    b = Batch(k3, kv, rope, 64, reqs, seed=H + len(reqs))
    n = int(b.start[-1])
    q = b.queries(H, n, 1.0, BF16)
    got = b.call(q, H, n, BF16, F32, 0.07)
    b.compare(got, q, H, BF16, F32, 0.07)


@pytest.mark.parametrize("B", [2, 31, 32, 33, 63, 64, 65, 449, 900])
def test_attend_batch_sizes(k3, B):
    """Some requests without rows, some without positions, one far longer than the others."""
    g = np.random.default_rng(B)
    reqs = [(int(g.integers(0, 90)), int(g.integers(0, 3))) for _ in range(B)]
    reqs = [(max(k, n), n) for k, n in reqs]
    reqs[B // 2] = (4000, 1)
    reqs[-1] = (70, 2)
    b = Batch(k3, 128, 16, 16, reqs, seed=B)
    n = int(b.start[-1])
    q = b.queries(24, n, 1.0, BF16)
    got = b.call(q, 24, n, BF16, F32, 0.07)
    b.compare(got, q, 24, BF16, F32, 0.07)


def test_attend_pages_outside_the_pool(k3):
    """They raise the device error and count as not there."""
    B = Batch(k3, 512, 64, 64, [(200, 1)], seed=9)
    bad = B.table.copy()
    bad[0, 1] = B.shape.n_pages + 4
    B.bufs[0] = i32(bad)
    q = B.queries(64, 1, 1.0, BF16)
    got = B.call(q, 64, 1, BF16, F32, 0.07, sync=False)
    assert k3.k3d_sync() == k3cuda.K3D_EDEVICE
    k3.k3d_clear_status()
    B.values[0] = np.concatenate([B.values[0][:64], B.values[0][128:]])
    B.exps[0] = np.concatenate([B.exps[0][:64], B.exps[0][128:]])
    B.reqs = [(136, 1)]
    B.compare(got, q, 64, BF16, F32, 0.07)


# -------------------------------------------------------------------------- page plans ----
class DevPages:
    def __init__(self, lib, page, n_pages, max_pages, B, free):
        self.lib, self.B, self.n_pages, self.max_pages = lib, B, n_pages, max_pages
        fl = np.full(n_pages, -1, np.int32)
        fl[:len(free)] = free
        self.t, self.h, self.f, self.n = (i32(np.full((B, max_pages), -1)), i32(np.zeros(B)), i32(fl), i32([len(free)]))
        self.p = k3cuda.K3dPages(page, n_pages, max_pages, self.t.ptr, self.h.ptr, self.f.ptr, self.n.ptr)

    def plan(self, lens, new, N):
        L, W = i32(lens), i32(new)
        o = [i32(np.full(self.B + 1, 99)), i32(np.full(self.B, 99)), i32(np.full(max(N, 1), 99)),
             i32(np.full(max(N, 1), 99)), i32([99])]
        check(self.lib.k3d_page_plan(self.p, L.ptr, W.ptr, self.B, N, *(b.ptr for b in o)))
        check(self.lib.k3d_sync())
        return (int(o[4].download(np.int32, 1)[0]), o[0].download(np.int32, self.B + 1).tolist(),
                o[1].download(np.int32, self.B).tolist(), o[2].download(np.int32, N).tolist(),
                o[3].download(np.int32, N).tolist())

    def state(self):
        return (self.t.download(np.int32, (self.B, self.max_pages)), self.h.download(np.int32, self.B),
                self.f.download(np.int32, self.n_pages), int(self.n.download(np.int32, 1)[0]))


def same_pages(dev, host):
    table, held, free, n = dev.state()
    assert held.tolist() == [len(t) for t in host.table]
    for b, t in enumerate(host.table):
        assert table[b].tolist() == t + [-1] * (host.max_pages - len(t))
    assert free[:n].tolist() == host.free


@pytest.mark.parametrize("B,page,top,N", [(1, 64, 300, 400), (7, 16, 90, 200), (64, 64, 500, 9000), (1500, 32, 60, 20000),
                                          (8192, 16, 3, 30000)])
def test_plan_follows_the_requests(k3, B, page, top, N):
    g = np.random.default_rng(B)
    max_pages = -(-2 * top // page) + 1
    n_pages = int(B * max_pages * 0.6) + 4
    free = g.permutation(n_pages).tolist()
    dev, host = DevPages(k3, page, n_pages, max_pages, B, free), ref.Pages(page, n_pages, max_pages, B, free)
    lens = np.zeros(B, int)
    for step in range(6):
        if step == 0:
            new = g.integers(0, top, B)                            # prompts, some requests not there yet
        elif step == 3:
            lens, new = np.where(g.random(B) < 0.4, 0, lens), np.zeros(B, int)   # requests that ended
        else:
            lens = np.maximum(0, lens - g.integers(0, 3, B))        # drafts that were rejected
            new = g.integers(0, 6, B)
        got, want = dev.plan(lens, new, N), host.plan(lens.tolist(), new.tolist(), N)
        assert got == want, step
        same_pages(dev, host)
        if want[0] == 0:
            lens = lens + new


def test_plan_taking_and_giving_back_is_the_identity(k3):
    dev = DevPages(k3, 16, 40, 12, 3, list(range(39, -1, -1)))
    dev.plan([0, 0, 0], [20, 5, 0], 64)
    before = dev.state()
    dev.plan([20, 5, 0], [40, 60, 33], 200)
    assert dev.plan([20, 5, 0], [0, 0, 0], 0)[0] == k3cuda.K3D_PLAN_OK
    after = dev.state()
    assert all(np.array_equal(a, b) for a, b in zip(before, after))


@pytest.mark.parametrize("N", [1024, 1025, 2047, 2048, 2049])
@pytest.mark.parametrize("B", [64, 256, 257, 1500])
def test_plan_around_its_row_limits(k3, B, N):
    """Rows written by the planning CTA (of 256 threads up to 256 requests and 1024 rows, else of 1024) and
    by the second launch above 2048; several requests to a thread; steps that fill N to the last row."""
    g = np.random.default_rng(B + N)
    page, max_pages = 16, 12
    n_pages = B * 6 + 40
    free = g.permutation(n_pages).tolist()
    dev, host = DevPages(k3, page, n_pages, max_pages, B, free), ref.Pages(page, n_pages, max_pages, B, free)
    lens = np.zeros(B, int)
    for step in range(4):
        top = max(1, N // B)
        new = g.integers(0, min(top, 31) + 1, B)
        if step == 2:                                              # exactly N rows
            new[:] = N // B
            new[:N - new.sum()] += 1
        assert new.sum() <= N
        got, want = dev.plan(lens, new, N), host.plan(lens.tolist(), new.tolist(), N)
        assert want[0] == 0 and got == want, step
        same_pages(dev, host)
        lens = np.where(g.random(B) < 0.2, 0, lens + g.integers(0, new + 1))


@pytest.mark.parametrize("off", [(1, 1), (0, 2), (3, 0)])
@pytest.mark.parametrize("N", [2051, 5000])
def test_plan_rows_at_any_alignment(k3, N, off):
    """pos and slots need no more than an int's alignment; nothing is written outside them."""
    g = np.random.default_rng(N)
    B, page = 50, 16
    free = g.permutation(700).tolist()
    dev, host = DevPages(k3, page, 700, 40, B, free), ref.Pages(page, 700, 40, B, free)
    lens, new = np.zeros(B, int), g.integers(0, N // B + 1, B)
    L, W = i32(lens), i32(new)
    rs, kl, st = i32(np.zeros(B + 1)), i32(np.zeros(B)), i32([9])
    pos, slots = (i32(np.full(N + 8, 77)) for _ in range(2))
    check(k3.k3d_page_plan(dev.p, L.ptr, W.ptr, B, N, rs.ptr, kl.ptr, pos.ptr + 4 * off[0], slots.ptr + 4 * off[1], st.ptr))
    check(k3.k3d_sync())
    want = host.plan(lens.tolist(), new.tolist(), N)
    for buf, o, w in ((pos, off[0], want[3]), (slots, off[1], want[4])):
        v = buf.download(np.int32, N + 8)
        assert v[o:o + N].tolist() == w and (v[:o] == 77).all() and (v[o + N:] == 77).all()


@pytest.mark.parametrize("lens,new,N,code", [
    ([10, 20], [200, 200], 1000, k3cuda.K3D_PLAN_PAGES), ([10, 20], [8, 8], 15, k3cuda.K3D_PLAN_ROWS),
    ([10, 20], [1, 400], 1000, k3cuda.K3D_PLAN_TABLE), ([-1, 20], [8, 8], 100, k3cuda.K3D_PLAN_BAD),
    ([10, 20], [8, -8], 100, k3cuda.K3D_PLAN_BAD), ([2 ** 31 - 1, 0], [1, 0], 100, k3cuda.K3D_PLAN_BAD)])
def test_plan_that_cannot_be_met_changes_nothing(k3, lens, new, N, code):
    dev = DevPages(k3, 16, 20, 20, 2, list(range(20)))
    assert dev.plan([10, 20], [0, 0], 4)[0] == k3cuda.K3D_PLAN_OK
    before = dev.state()
    got = dev.plan(lens, new, N)
    assert got == (code, [0, 0, 0], [0, 0], [-1] * N, [-1] * N)
    assert all(np.array_equal(a, b) for a, b in zip(before, dev.state()))


# ----------------------------------------------------------------------- probabilities ----
def softmax(lib, x, temp, in_place=False, off=0):
    rows, V = x.shape
    X = DevBuf.from_array(np.concatenate([np.zeros(off, np.float32), x.reshape(-1)]))
    P = X if in_place else DevBuf((x.size + off) * 4)
    T = DevBuf.from_array(np.asarray(temp, np.float32)) if temp is not None else None
    check(lib.k3d_logits_softmax(P.ptr + 4 * off, X.ptr + 4 * off, T.ptr if T else None, rows, V))
    check(lib.k3d_sync())
    return P.download(np.float32, x.size + off)[off:].reshape(x.shape)


def softmax_close(got, x, temp):
    """Relative: the argument (x - max) / T (four roundings), exp2 (two steps), the sums of a
    thread's, a block's and a cluster's terms in order, the reciprocal and the product."""
    want = ref.softmax(x, temp)
    V = x.shape[1]
    for r in range(x.shape[0]):
        t = 1.0 if temp is None else float(temp[r])
        m = np.nanmax(x[r]) if np.isfinite(np.nanmax(x[r])) else 0.0
        with np.errstate(invalid="ignore"):
            d = np.nan_to_num(np.abs(x[r].astype(np.float64) - m) * 1.4427 / (t if t > 0 else 1.0), nan=0.0, posinf=0.0)
        tol = want[r] * 2.0 ** -24 * (4 * np.minimum(d, 200) + 8 + V / 512 + 40) + 2.0 ** -126
        assert (np.abs(got[r] - want[r]) <= tol).all(), r


@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 31), (5, 1000), (4, 1001), (3, 4096), (2, 32003), (2, 163840),
                                    (1, 500001)])
def test_softmax(k3, rows, V):
    g = np.random.default_rng(V)
    x = (g.standard_normal((rows, V)) * 4).astype(np.float32)
    temp = g.uniform(0.2, 2.0, rows).astype(np.float32)
    softmax_close(softmax(k3, x, None), x, None)
    softmax_close(softmax(k3, x, temp), x, temp)
    softmax_close(softmax(k3, x, temp, in_place=True), x, temp)
    softmax_close(softmax(k3, x, temp, off=1), x, temp)


@pytest.mark.parametrize("rows,V", [(36, 33000), (38, 33000), (75, 33001), (160, 17000), (300, 2500), (5, 70000)])
def test_softmax_row_counts(k3, rows, V):
    """Sixteen, eight, four or one CTA to a row, greedy rows among them."""
    g = np.random.default_rng(rows)
    x = (g.standard_normal((rows, V)) * 4).astype(np.float32)
    temp = np.where(np.arange(rows) % 3 == 0, 0.0, 0.7).astype(np.float32)
    softmax_close(softmax(k3, x, temp), x, temp)


def test_softmax_greedy_takes_the_first_maximum(k3):
    x = np.zeros((4, 20000), np.float32)
    x[0, [777, 15000]] = 3.0
    x[1] = -np.inf
    x[1, 19999] = -5.0
    x[2, 4] = np.nan
    got = softmax(k3, x, np.array([0.0, -1.0, np.nan, 0.0], np.float32))
    assert [int(r.argmax()) for r in got] == [777, 19999, 0, 0] and (got.sum(1) == 1.0).all()


def test_softmax_masked_rows(k3):
    g = np.random.default_rng(2)
    low = np.finfo(np.float32).min
    x = g.standard_normal((7, 9000)).astype(np.float32)
    x[0, ::2] = -np.inf
    x[1] = -np.inf                                   # nothing left: zeros
    x[2] = low                                       # the type's lowest value everywhere: uniform
    x[3, 5], x[3, 8000] = np.inf, np.inf             # the whole on two places
    x[4, 1::2] = np.nan
    x[5] = np.nan
    x[6, 100:] = low
    got = softmax(k3, x, None)
    softmax_close(got, x, None)
    assert (got[1] == 0).all() and (got[5] == 0).all() and got[3, 5] == 0.5
    hot = softmax(k3, x[:1], np.array([np.inf], np.float32))
    assert (hot[0, ::2] == 0).all() and np.allclose(hot[0, 1::2], 1 / 4500, rtol=1e-6)


def test_softmax_at_the_ends_of_the_temperatures(k3):
    """1 / T leaves fp32 below 2^-128: the maxima share the whole, as they do at any T so small."""
    g = np.random.default_rng(5)
    x = g.standard_normal((5, 5000)).astype(np.float32)
    x[:, [3, 4001]] = 6.0
    temp = np.array([1e-45, 1e-40, 1e-30, 1e30, 3e38], np.float32)
    got = softmax(k3, x, temp)
    softmax_close(got, x, temp)
    assert (got[:3, 3] == 0.5).all() and (got[:3, 4001] == 0.5).all()


@pytest.mark.parametrize("rows,V", [(4, 70000), (2, 65537), (1, 300000)])
def test_softmax_sixteen_ctas_to_a_row(k3, rows, V):
    """Up to four rows of 65536 and more, greedy rows among them."""
    g = np.random.default_rng(V)
    x = (g.standard_normal((rows, V)) * 4).astype(np.float32)
    temp = np.where(np.arange(rows) % 2 == 1, 0.0, 0.7).astype(np.float32)
    softmax_close(softmax(k3, x, temp), x, temp)


@pytest.mark.parametrize("V", [9000, 9001])
def test_softmax_of_logits_further_apart_than_fp32(k3, V):
    """x - max passes fp32's largest number where (x - max) / T does not."""
    g = np.random.default_rng(V)
    x = (g.standard_normal((5, V)) * 1e38).clip(-3.4e38, 3.4e38).astype(np.float32)
    x[:, 3], x[:, 700], x[4] = 3.4e38, -3.4e38, np.tile(np.float32([3.4e38, -3.4e38]), V)[:V]
    x[1, 5::7] = -np.inf
    temp = np.array([1e38, 3e38, np.inf, 5e37, np.inf], np.float32)
    got = softmax(k3, x, temp)
    softmax_close(got, x, temp)
    assert (np.abs(got[[2, 4]] * V - 1) <= 1e-5).all() and got[0, 700] > 0


# ------------------------------------------------------------------------ verification ----
def verify(lib, target, draft, ids, nd, u, us):
    B, K1, V = target.shape
    bufs = [DevBuf.from_array(np.ascontiguousarray(a)) if a is not None else None
            for a in (target.astype(np.float32), None if draft is None else draft.astype(np.float32),
                      ids.astype(np.int32), None if nd is None else np.asarray(nd, np.int32), u.astype(np.float32),
                      us.astype(np.float32))]
    tok, acc = i32(np.full((B, K1), 99)), i32(np.full(B, 99))
    check(lib.k3d_spec_verify(tok.ptr, acc.ptr, *(b.ptr if b is not None else None for b in bufs), B, K1 - 1, V))
    check(lib.k3d_sync())
    return tok.download(np.int32, (B, K1)), acc.download(np.int32, B)


def chances(g, shape, gain=2.0):
    x = g.standard_normal(shape) * gain
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 2, 7), (40, 3, 1000), (33, 4, 4099), (5, 32, 257), (2, 4, 163840), (9, 0, 300),
                                   (2, 1, 16384)])
def test_verify(k3, B, K, V, probs):
    g = np.random.default_rng(B * 7 + K + V)
    z = g.standard_normal((B, K + 1, V)) * 2.0
    e = np.exp(z - z.max(-1, keepdims=True))
    target = (e / e.sum(-1, keepdims=True)).astype(np.float32)
    draft = None
    if K:
        z = z[:, :K] + g.standard_normal((B, K, V)) * 0.5
        e = np.exp(z - z.max(-1, keepdims=True))
        draft = (e / e.sum(-1, keepdims=True)).astype(np.float32)
    ids = np.zeros((B, K), np.int32)
    for b in range(B):
        for i in range(K):
            c = np.cumsum(draft[b, i].astype(np.float64))
            ids[b, i] = min(V - 1, np.searchsorted(c, g.random() * c[-1]))
    u, us = g.random((B, K)).astype(np.float32), g.random(B).astype(np.float32)
    us[0] = 0.0
    if B > 2:
        us[1] = np.float32(1.0) - np.float32(2.0 ** -24)
    nd = g.integers(0, K + 1, B) if B > 3 else None
    q = draft if probs else None
    if not probs:
        u *= np.float32(0.02)                       # certain drafts are kept with p(d) alone
    want = ref.verify(target, q, ids, nd, u, us)
    got = verify(k3, target, q, ids, nd, u, us)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


def test_verify_edges(k3):
    g = np.random.default_rng(11)
    V, K, B = 50, 2, 9
    target, draft = chances(g, (B, K + 1, V)), chances(g, (B, K, V))
    ids = g.integers(0, V, (B, K)).astype(np.int32)
    u, us = np.full((B, K), 0.999, np.float32), g.random(B).astype(np.float32)
    draft[0] = target[0, :K]                         # the same distribution: u q < p holds for u < 1
    draft[1] = np.float32(1.0)                       # p <= q everywhere: nothing left, so p itself
    target[2] = 0.0                                  # no token can be drawn
    target[3, 0] = np.nan
    target[4, 0] = 0.0
    target[4, 0, 49] = 1.0                           # all on the last token
    ids[5] = V                                       # not in the vocabulary
    ids[6, 0] = -3
    u[7] = 1.0                                       # u q < p fails at equality
    draft[7] = target[7, :K]
    us[8] = 1.0                                      # above the range: the last weight
    want = ref.verify(target, draft, ids, None, u, us)
    got = verify(k3, target, draft, ids, None, u, us)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert want[1][0] == 2 and want[1][7] == 0 and want[0][2, 0] == -1


def test_verify_largest_sums(k3):
    """A row of ones over the largest vocabulary: the running sum ends just below 2^63."""
    V = (1 << 19) - 1
    target = np.ones((2, 1, V), np.float32)
    ids, u, us = np.zeros((2, 0)), np.zeros((2, 0)), np.array([0.5, 1.0 - 2.0 ** -24])
    want = ref.verify(target, None, ids, None, u, us)
    got = verify(k3, target, None, np.zeros((2, 1)), None, np.zeros((2, 1)), us)
    assert (got[0] == want[0]).all() and (got[1] == want[1]).all()


def test_verify_draws_the_distribution(k3):
    """Drafts from q, verified against p, come out distributed as p: 4096 requests over six
    tokens. The count of a token is binomial, so five standard deviations bound it but for one
    run in a million and a half; the seed is fixed."""
    g = np.random.default_rng(12)
    B, V = 4096, 6
    p = np.array([0.4, 0.25, 0.2, 0.1, 0.05, 0.0], np.float32)
    q = np.array([0.1, 0.2, 0.2, 0.2, 0.2, 0.1], np.float32)
    ids = g.choice(V, (B, 1), p=q / q.sum()).astype(np.int32)
    got, _ = verify(k3, np.broadcast_to(p, (B, 2, V)), np.broadcast_to(q, (B, 1, V)), ids, None,
                    g.random((B, 1)).astype(np.float32), g.random(B).astype(np.float32))
    count = np.bincount(got[:, 0], minlength=V)
    assert (np.abs(count - B * p) <= 5 * np.sqrt(B * p * (1 - p))).all(), count


# ------------------------------------------------------------------------ a serving step ----
class Loop:
    """One step of a serving loop as one run of calls on fixed buffers: plan the pages, store the
    new rows, attend, probabilities of the rows' logits, verify the drafts."""

    def __init__(self, lib, g, B=5, K=3, H=16, kv=256, rope=32, page=16, n_pages=90, V=700):
        self.lib, self.g, self.B, self.K, self.H, self.kv, self.w, self.page, self.V = lib, g, B, K, H, kv, kv + rope, page, V
        self.N = B * (K + 1)
        self.shape = k3cuda.K3dCache4(kv, rope, page, n_pages)
        self.pool = DevBuf(lib.k3d_cache4_bytes(self.shape))
        check(lib.k3d_memset(self.pool.ptr, 0xff, self.pool.nbytes))
        self.free = g.permutation(n_pages).tolist()
        self.pages = DevPages(lib, page, n_pages, 12, B, self.free)
        self.host = ref.Pages(page, n_pages, 12, B, self.free)
        f = np.float32
        self.dev = {k: DevBuf.from_array(np.zeros(s, t)) for k, s, t in (
            ("len", B, np.int32), ("new", B, np.int32), ("start", B + 1, np.int32), ("kvl", B, np.int32),
            ("pos", self.N, np.int32), ("slots", self.N, np.int32), ("status", 1, np.int32),
            ("x", (self.N, self.w), f), ("q", (self.N, H, self.w), f), ("o", (self.N, H, kv), f),
            ("logits", (self.N, V), f), ("p", (self.N, V), f), ("temp", self.N, f), ("draft", (B, K, V), f),
            ("ids", (B, K), np.int32), ("nd", B, np.int32), ("u", (B, K), f), ("us", B, f),
            ("tok", (B, K + 1), np.int32), ("acc", B, np.int32))}
        self.nws = lib.k3d_mla_attend4_ws_bytes(self.shape, B, self.N, H)
        self.ws = DevBuf(self.nws)

    def inputs(self, lens, new):
        g, B, K, V = self.g, self.B, self.K, self.V
        h = {"len": np.int32(lens), "new": np.int32(new), "x": rows(g, self.N, self.w, 0.5),
             "q": from_bf16(to_bf16(g.standard_normal((self.N, self.H, self.w)))), "nd": np.int32([n - 1 for n in new]),
             "logits": (g.standard_normal((self.N, V)) * 3).astype(np.float32),
             "temp": np.where(g.random(self.N) < 0.3, 0, 0.8).astype(np.float32), "draft": chances(g, (B, K, V)),
             "ids": g.integers(0, V, (B, K)).astype(np.int32), "u": (g.random((B, K)) * 0.3).astype(np.float32),
             "us": g.random(B).astype(np.float32)}
        for k, v in h.items():
            self.dev[k].upload(v)
        return h

    def calls(self):
        lib, d = self.lib, {k: b.ptr for k, b in self.dev.items()}
        check(lib.k3d_page_plan(self.pages.p, d["len"], d["new"], self.B, self.N, d["start"], d["kvl"], d["pos"],
                                d["slots"], d["status"]))
        check(lib.k3d_cache4_store(self.shape, self.pool.ptr, d["x"], F32, self.w, d["slots"], self.N))
        check(lib.k3d_mla_attend4(d["o"], F32, d["q"], F32, self.shape, self.pool.ptr, self.pages.t.ptr, 12, d["start"],
                                  d["kvl"], self.B, self.N, self.H, 0.07, self.ws.ptr, self.nws))
        check(lib.k3d_logits_softmax(d["p"], d["logits"], d["temp"], self.N, self.V))
        # a request's target rows lie K + 1 apart: here every request brings K + 1 rows
        check(lib.k3d_spec_verify(d["tok"], d["acc"], d["p"], d["draft"], d["ids"], d["nd"], d["u"], d["us"], self.B,
                                  self.K, self.V))

    def results(self):
        shapes = {"start": (np.int32, self.B + 1), "kvl": (np.int32, self.B), "slots": (np.int32, self.N),
                  "o": (np.float32, (self.N, self.H, self.kv)), "p": (np.float32, (self.N, self.V)),
                  "tok": (np.int32, (self.B, self.K + 1)), "acc": (np.int32, self.B), "status": (np.int32, 1)}
        return {k: self.dev[k].download(*v) for k, v in shapes.items()}


def run_steps(k3, graph):
    g = np.random.default_rng(21)
    L = Loop(k3, g)
    B, K = L.B, L.K
    lens = np.zeros(B, int)
    known = [np.zeros((0, L.w)) for _ in range(B)]            # what the oracle's cache holds
    out, ex = [], None
    for step in range(6):
        new = [K + 1] * B
        h = L.inputs(lens, new)
        if graph and ex is None:
            check(k3.k3d_graph_begin())
            L.calls()
            ex = k3.k3d_graph_end()
            assert ex
        if graph:
            check(k3.k3d_graph_launch(ex))
        else:
            L.calls()
        check(k3.k3d_sync())
        r = L.results()
        code, start, kvl, _, slots = L.host.plan(lens.tolist(), new, L.N)
        assert code == 0 and r["status"][0] == 0
        assert r["start"].tolist() == start and r["kvl"].tolist() == kvl and r["slots"].tolist() == slots
        same_pages(L.pages, L.host)
        values = ref.quantise(h["x"], L.kv)[1]
        for b in range(B):
            known[b] = np.concatenate([known[b][:lens[b]], values[start[b]:start[b + 1]]])
            want = ref.attend(h["q"][start[b]:start[b + 1]], known[b], L.kv, 0.07, new[b])
            # fp32 results: the weights' and the scores' rounding as in Batch.compare, for values
            # of up to about 10 and scores' sums of magnitudes of up to 0.07 x 300 x 4
            assert np.abs(r["o"][start[b]:start[b + 1]] - want).max() <= 10 * (2.0 ** -11 + np.expm1(2 * 84 * (2.0 ** -11 + 288 * 2.0 ** -24)))
        softmax_close(r["p"], h["logits"], h["temp"])
        tok, acc = ref.verify(r["p"].reshape(B, K + 1, L.V), h["draft"], h["ids"], h["nd"], h["u"], h["us"])
        assert np.array_equal(r["tok"], tok) and np.array_equal(r["acc"], acc)
        lens = lens + acc + 1                                  # the rejected drafts' rows are given up
        if step == 3:
            lens[1] = 0                                        # a request that ended, another in its place
            known[1] = known[1][:0]
        out.append({k: v.copy() for k, v in r.items()})
    if ex:
        k3.k3d_graph_destroy(ex)
    return out


def test_serving_steps_and_their_graph(k3):
    """Six steps against the definitions, called one by one and as a graph that is replayed with
    new contents of the same buffers: the same bits."""
    eager, graph = run_steps(k3, False), run_steps(k3, True)
    for a, b in zip(eager, graph):
        for k in a:
            assert np.array_equal(a[k], b[k]), k


def test_serving_step_on_another_stream(k3):
    """The calls run on the stream that k3d_set_stream names."""
    rt = ctypes.CDLL("libcudart.so.12")
    s = ctypes.c_void_p()
    assert rt.cudaStreamCreateWithFlags(ctypes.byref(s), 1) == 0
    own = k3.k3d_stream()
    try:
        check(k3.k3d_sync())
        check(k3.k3d_set_stream(s))
        got = run_steps(k3, False)
    finally:
        check(k3.k3d_sync())
        check(k3.k3d_set_stream(own))
        rt.cudaStreamDestroy(s)
    want = run_steps(k3, False)
    for a, b in zip(got, want):
        for k in a:
            assert np.array_equal(a[k], b[k]), k


@pytest.mark.parametrize("kv,rope", [(128, 16), (512, 64)])
def test_attend_on_two_streams_at_once(k3, kv, rope):
    """Two calls with a workspace each, on two streams that do not wait for one another: the same
    bits as one after the other."""
    rt = ctypes.CDLL("libcudart.so.12")
    s = ctypes.c_void_p()
    batches = [Batch(k3, kv, rope, 64, [(3000, 2), (700, 1)], seed=41), Batch(k3, kv, rope, 64, [(1500, 3)] * 6, seed=42)]
    sets = []
    for b in batches:
        n = int(b.start[-1])
        q = b.queries(64, n, 1.0, BF16)
        want = b.call(q, 64, n, BF16, F32, 0.07)
        nb = k3.k3d_mla_attend4_ws_bytes(b.shape, len(b.reqs), n, 64)
        sets.append((b, n, DevBuf.from_array(to_bf16(q)), DevBuf(want.nbytes), DevBuf(nb), nb, want))
    own = k3.k3d_stream()
    assert rt.cudaStreamCreateWithFlags(ctypes.byref(s), 1) == 0
    try:
        for _ in range(8):
            for (b, n, Q, O, W, nb, _), stream in zip(sets, (own, s)):
                check(k3.k3d_set_stream(stream))
                T, R, K = b.bufs
                check(k3.k3d_mla_attend4(O.ptr, F32, Q.ptr, BF16, b.shape, b.pool.ptr, T.ptr, b.max_pages, R.ptr, K.ptr,
                                         len(b.reqs), n, 64, 0.07, W.ptr, nb))
        check(k3.k3d_sync())
    finally:
        check(k3.k3d_set_stream(own))
        check(k3.k3d_sync())
        rt.cudaStreamDestroy(s)
    for b, n, Q, O, W, nb, want in sets:
        assert np.array_equal(O.download(np.float32, want.shape), want)


def test_attend_bits_do_not_depend_on_the_run(k3):
    """Splits, merges and launches in one order: the same bits every time."""
    B = Batch(k3, 512, 64, 64, [(5000, 2), (700, 1), (64, 3)], seed=31)
    q = B.queries(64, 6, 1.0, BF16)
    first = B.call(q, 64, 6, BF16, F32, 0.07)
    for _ in range(5):
        assert np.array_equal(first, B.call(q, 64, 6, BF16, F32, 0.07))


def test_attend_lengths_that_do_not_fit(k3):
    """A kv_len above max_pages * page, or row_starts that run past N, raise the device error; the
    rows of the other requests are right."""
    B = Batch(k3, 256, 32, 16, [(40, 1), (30, 1)], seed=32)
    B.bufs[2] = i32([10 ** 6, 30])
    q = B.queries(16, 2, 1.0, BF16)
    got = B.call(q, 16, 2, BF16, F32, 0.07, sync=False)
    assert k3.k3d_sync() == k3cuda.K3D_EDEVICE
    k3.k3d_clear_status()
    want = ref.attend(q[1:2], B.values[1], 256, 0.07, 1)
    assert np.abs(got[1:2] - want).max() <= 2.0 ** -6
    B.bufs[1], B.bufs[2] = i32([0, 1, 9]), i32([40, 30])
    got = B.call(q, 16, 2, BF16, F32, 0.07, sync=False)
    assert k3.k3d_sync() == k3cuda.K3D_EDEVICE
    k3.k3d_clear_status()
    assert np.abs(got[:1] - ref.attend(q[:1], B.values[0], 256, 0.07, 1)).max() <= 2.0 ** -6


@pytest.mark.parametrize("kv,rope,H", [(128, 0, 16), (512, 64, 16), (256, 32, 32)])
def test_attend_of_few_rows_beside_other_work(k3, kv, rope, H):
    """Items of up to 32 rows, whose P is held for two tiles, many tiles each, beside another call on
    a second stream that takes the memory and the issue slots: the same bits as alone."""
    rt = ctypes.CDLL("libcudart.so.12")
    s = ctypes.c_void_p()
    b = Batch(k3, kv, rope, 64, [(4000, 1)] * 6 + [(900, 1), (3001, 1)], seed=51)
    n = int(b.start[-1])
    q = b.queries(H, n, 1.0, BF16)
    want = b.call(q, H, n, BF16, F32, 0.07)
    b.compare(want, q, H, BF16, F32, 0.07)
    nb = k3.k3d_mla_attend4_ws_bytes(b.shape, len(b.reqs), n, H)
    Q, O, W = DevBuf.from_array(to_bf16(q)), DevBuf(want.nbytes), DevBuf(nb)
    x = np.zeros((64, 100000), np.float32)
    X, P = DevBuf.from_array(x), DevBuf(x.nbytes)
    own = k3.k3d_stream()
    assert rt.cudaStreamCreateWithFlags(ctypes.byref(s), 1) == 0
    try:
        for _ in range(20):
            check(k3.k3d_set_stream(s))
            check(k3.k3d_logits_softmax(P.ptr, X.ptr, None, *x.shape))
            check(k3.k3d_set_stream(own))
            T, R, K = b.bufs
            check(k3.k3d_mla_attend4(O.ptr, F32, Q.ptr, BF16, b.shape, b.pool.ptr, T.ptr, b.max_pages, R.ptr, K.ptr,
                                     len(b.reqs), n, H, 0.07, W.ptr, nb))
        check(k3.k3d_sync())
    finally:
        check(k3.k3d_set_stream(s))
        check(k3.k3d_sync())
        check(k3.k3d_set_stream(own))
        rt.cudaStreamDestroy(s)
    assert np.array_equal(O.download(np.float32, want.shape), want)


def test_attend_workspace_asked_for_before_the_device(k3):
    """A program may size its buffers before its first library call: the size is the same then, and
    attention takes it."""
    import os
    import subprocess
    import sys
    code = ("import k3cuda; lib = k3cuda.load(); c = k3cuda.K3dCache4(512, 64, 64, 9)\n"
            "a = [lib.k3d_mla_attend4_ws_bytes(c, 3, 5, h) for h in (1, 64, 128)]\n"
            "k3cuda.check(lib.k3d_init(0))\n"
            "assert a == [lib.k3d_mla_attend4_ws_bytes(c, 3, 5, h) for h in (1, 64, 128)], a\nprint(*a)")
    env = dict(os.environ, PYTHONPATH=os.path.dirname(k3cuda.__file__))
    out = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    c = k3cuda.K3dCache4(512, 64, 64, 9)
    assert [int(v) for v in out.stdout.split()] == [k3.k3d_mla_attend4_ws_bytes(c, 3, 5, h) for h in (1, 64, 128)]
