"""Refusals of the serving operators. Arguments are checked before the device is touched, so a
wrong call is answered without a GPU (the addresses here are never read)."""
import ctypes

import pytest

import k3cuda
import serving_ref as ref

A = 1 << 20                    # an aligned address that nothing reads
EINVAL, EUNSUP, OK = k3cuda.K3D_EINVAL, k3cuda.K3D_EUNSUPPORTED, k3cuda.K3D_OK
F32, BF16 = k3cuda.K3D_DT_F32, k3cuda.K3D_DT_BF16


@pytest.fixture
def lib():
    lib = k3cuda.load()
    lib.k3d_clear_status()
    yield lib
    lib.k3d_clear_status()


def shape(kv=512, rope=64, page=64, n=8):
    return k3cuda.K3dCache4(kv, rope, page, n)


BAD_SHAPES = [shape(kv=0), shape(kv=96), shape(kv=640), shape(rope=8), shape(rope=80), shape(rope=-16), shape(page=8),
              shape(page=24), shape(page=2048), shape(n=0), shape(n=1 << 26)]


@pytest.mark.parametrize("bad", BAD_SHAPES)
def test_cache_shapes(lib, bad):
    assert lib.k3d_cache4_bytes(bad) == 0
    assert lib.k3d_cache4_store(bad, A, A, F32, 1024, A, 1) == EINVAL
    assert lib.k3d_cache4_load(bad, A, A, F32, 1024, A, 1) == EINVAL
    assert lib.k3d_mla_attend4_ws_bytes(bad, 1, 1, 8) == 0
    assert lib.k3d_mla_attend4(A, BF16, A, BF16, bad, A, A, 1, A, A, 1, 1, 8, 1.0, A, 1 << 40) == EINVAL


@pytest.mark.parametrize("kv,rope,page", [(512, 64, 64), (128, 0, 16), (384, 48, 1024)])
def test_pool_bytes(lib, kv, rope, page):
    assert lib.k3d_cache4_bytes(shape(kv, rope, page, 5)) == 5 * ref.page_bytes(kv, rope, page)


@pytest.mark.parametrize("f", ["k3d_cache4_store", "k3d_cache4_load"])
def test_rows(lib, f):
    f, s = getattr(lib, f), shape()
    assert f(s, A, A, F32, 576, A, -1) == EINVAL
    assert f(s, A, A, F32, 575, A, 1) == EINVAL
    assert f(s, A, A, k3cuda.K3D_DT_F16, 576, A, 1) == EUNSUP
    assert f(None, A, A, F32, 576, A, 1) == EINVAL
    for bad in ((None, A, A), (A, None, A), (A, A, None), (A + 8, A, A), (A, A + 2, A), (A, A, A + 2)):
        assert f(s, bad[0], bad[1], F32, 576, bad[2], 1) == EINVAL
    assert f(s, A, A + 1, BF16, 576, A, 1) == EINVAL
    assert f(s, None, None, F32, 576, None, 0) == OK


def test_attend(lib):
    s = shape()
    n = lib.k3d_mla_attend4_ws_bytes(s, 2, 3, 64)
    assert n > 0
    assert lib.k3d_mla_attend4_ws_bytes(s, 0, 3, 64) == 0 and lib.k3d_mla_attend4_ws_bytes(s, 2, 3, 0) == 0

    def call(out=A, ot=BF16, q=A, qt=BF16, c=s, pool=A, table=A, mp=4, rs=A, kl=A, B=2, N=3, H=64, ws=A, nb=n):
        return lib.k3d_mla_attend4(out, ot, q, qt, c, pool, table, mp, rs, kl, B, N, H, 0.1, ws, nb)

    for name in ("out", "q", "pool", "table", "rs", "kl", "ws"):
        assert call(**{name: None}) == EINVAL, name
        assert call(**{name: A + 2}) == EINVAL, name
    for name in ("out", "q", "pool", "ws"):
        assert call(**{name: A + 8}) == EINVAL, name
    assert call(ot=k3cuda.K3D_DT_F16) == EUNSUP and call(qt=7) == EUNSUP
    for kw in (dict(B=0), dict(N=-1), dict(H=0), dict(H=1025), dict(mp=0), dict(mp=1 << 26), dict(nb=n - 1), dict(c=None)):
        assert call(**kw) == EINVAL, kw
    assert call(N=0, out=None, q=None) == OK


def test_plan(lib):
    def pages(**kw):
        d = dict(page=64, n_pages=100, max_pages=10, table=A, held=A, free_list=A, n_free=A)
        d.update(kw)
        return k3cuda.K3dPages(*(d[k] for k in ("page", "n_pages", "max_pages", "table", "held", "free_list", "n_free")))

    def call(p=None, ln=A, nw=A, B=4, N=8, rs=A, kl=A, pos=A, sl=A, st=A):
        return lib.k3d_page_plan(p if p is not None else pages(), ln, nw, B, N, rs, kl, pos, sl, st)

    for k in ("page", "n_pages", "max_pages"):
        assert call(pages(**{k: 0})) == EINVAL
    for k in ("table", "held", "free_list", "n_free"):
        assert call(pages(**{k: None})) == EINVAL
    assert call(pages(page=1 << 16, n_pages=1 << 16)) == EINVAL
    for kw in (dict(ln=None), dict(nw=None), dict(B=0), dict(B=8193), dict(N=-1), dict(rs=None), dict(kl=None),
               dict(pos=None), dict(sl=None), dict(st=None)):
        assert call(**kw) == EINVAL, kw
    assert lib.k3d_page_plan(None, A, A, 4, 8, A, A, A, A, A) == EINVAL


def test_softmax_and_verify(lib):
    assert lib.k3d_logits_softmax(A, A, None, -1, 10) == EINVAL
    assert lib.k3d_logits_softmax(A, A, None, 1, 0) == EINVAL
    assert lib.k3d_logits_softmax(None, A, None, 1, 10) == EINVAL
    assert lib.k3d_logits_softmax(A, None, None, 1, 10) == EINVAL
    assert lib.k3d_logits_softmax(A + 2, A, None, 1, 10) == EINVAL
    assert lib.k3d_logits_softmax(A, A, None, 1 << 29, 10) == EINVAL
    assert lib.k3d_logits_softmax(None, None, None, 0, 10) == OK

    def call(tok=A, na=A, p=A, q=A, ids=A, nd=A, u=A, us=A, B=2, K=4, V=100):
        return lib.k3d_spec_verify(tok, na, p, q, ids, nd, u, us, B, K, V)

    for kw in (dict(B=-1), dict(K=-1), dict(K=33), dict(V=0), dict(tok=None), dict(na=None), dict(p=None),
               dict(ids=None), dict(u=None), dict(us=None), dict(p=A + 1), dict(q=A + 2)):
        assert call(**kw) == EINVAL, kw
    assert call(B=0, tok=None) == OK


def test_verify_vocabularies_whose_sums_overflow(lib):
    for v in (1 << 19, (1 << 31) - 1):
        assert lib.k3d_spec_verify(A, A, A, A, A, A, A, A, 2, 4, v) == EINVAL


def test_counts_beyond_31_bits(lib):
    s, big = shape(), (1 << 30) + 1
    n = lib.k3d_mla_attend4_ws_bytes(s, 2, 3, 64)

    def attend(max_pages=4, B=2, N=3, H=64):
        return lib.k3d_mla_attend4(A, BF16, A, BF16, s, A, A, max_pages, A, A, B, N, H, 0.1, A, n)

    for kw in (dict(max_pages=(1 << 24) + 1), dict(B=big), dict(N=big, H=1), dict(N=(1 << 24) + 1)):
        assert attend(**kw) == EINVAL, kw
    assert lib.k3d_cache4_store(s, A, A, F32, 576, A, big) == EINVAL
    assert lib.k3d_cache4_load(s, A, A, F32, 576, A, big) == EINVAL
    assert lib.k3d_logits_softmax(A, A, None, 1, big) == EINVAL
    p = k3cuda.K3dPages(64, 100, 10, A, A, A, A)
    assert lib.k3d_page_plan(p, A, A, 4, big, A, A, A, A, A) == EINVAL
    p = k3cuda.K3dPages(1, big, 10, A, A, A, A)
    assert lib.k3d_page_plan(p, A, A, 4, 8, A, A, A, A, A) == EINVAL


def test_plan_arrays_are_whole_ints(lib):
    for i in range(7):
        args = [A + 2 if i == k else A for k in range(7)]
        p = k3cuda.K3dPages(64, 100, 10, A, A, A, A)
        assert lib.k3d_page_plan(p, args[0], args[1], 4, 8, *args[2:]) == EINVAL
    for i in range(4):
        p = k3cuda.K3dPages(64, 100, 10, *(A + 1 if i == k else A for k in range(4)))
        assert lib.k3d_page_plan(p, A, A, 4, 8, A, A, A, A, A) == EINVAL


def test_without_a_gpu_valid_calls_fail_loudly(lib):
    import glob
    if glob.glob("/dev/nvidia[0-9]*"):
        pytest.skip("checks the no-GPU failure path")
    assert lib.k3d_logits_softmax(A, A, None, 1, 10) == k3cuda.K3D_ENODEV
    assert lib.k3d_cache4_store(shape(), A, A, F32, 576, A, 1) == k3cuda.K3D_ENODEV
