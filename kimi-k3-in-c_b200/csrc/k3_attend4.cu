// k3_attend4.cu -- absorbed MLA attention over the paged 4-bit latent cache, for any number
// of new tokens per request (k3_mla_cached, k3_ops.c:321-410, in the absorbed form of
// k3_mla.cu; the row format is in k3_cache4.cuh).
//
//   s[r][t] = scale q[r] . row[t],  t < the keys that row r sees
//   o[r]    = sum_t softmax(s[r])[t] row[t][0 .. kv)
// Row r = (new token j of request b, head): it sees the first kv_len[b] - new_b + j + 1
// positions (none: zeros).
#include "k3_cache4.cuh"
#include "k3_ops.cuh"

namespace k3 {
namespace {

struct Attend {
    Pool4 d;
    const void *q;
    void *out;
    const int *table, *row_start, *kv_len;
    int max_pages, B, N, H;
    int q_f32, out_f32;
    float scale;
};

// The request of token n, or -1 behind the last row.
__device__ __forceinline__ int request_of_row(const int *start, int B, int n)
{
    if (n >= start[B]) return -1;
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= n) lo = mid; else hi = mid;
    }
    return lo;
}

// grid (N, ceil(H / 8)), one warp per head, tiles of 16 positions as fp32 in shared memory.
__global__ void __launch_bounds__(256) k_attend4_plain(Attend a)
{
    pdl_wait();
    pdl_trigger();
    __shared__ float tile[16][576 + 4];
    const int n = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y * 8 + warp;
    const int W = a.d.kv + a.d.rope;
    const int b = request_of_row(a.row_start, a.B, n);
    if (b < 0) return;
    const int j = n - a.row_start[b], nw = a.row_start[b + 1] - a.row_start[b];
    int kvl = a.kv_len[b];
    if (kvl > a.max_pages * a.d.page) {
        if (threadIdx.x == 0) k3_raise_at(K3D_EBOUND, K3_SITE_CACHE4, b, kvl, 2);
        kvl = a.max_pages * a.d.page;
    }
    const int seen = max(0, kvl - nw + j + 1);
    float q[18], acc[18];
#pragma unroll
    for (int i = 0; i < 18; i++) {
        q[i] = acc[i] = 0.f;
        const int c = lane + 32 * i;
        if (h < a.H && c < W) {
            const size_t at = ((size_t)n * a.H + h) * W + c;
            q[i] = a.q_f32 ? ((const float *)a.q)[at] : bf16_to_f32(((const uint16_t *)a.q)[at]);
        }
    }
    float m = -INFINITY, l = 0.f;
    for (int t0 = 0; t0 < seen; t0 += 16) {
        __syncthreads();
        // a tile never crosses a page (page % 16 == 0)
        const int pg = a.table[(size_t)b * a.max_pages + t0 / a.d.page];
        const bool ok = pg >= 0 && pg < a.d.n_pages;
        if (!ok && threadIdx.x == 0) k3_raise_at(K3D_EBOUND, K3_SITE_CACHE4, b, pg, 3);
        const int tn = ok ? min(16, seen - t0) : 0;
        const uint8_t *base = a.d.p + (size_t)(ok ? pg : 0) * a.d.page_bytes;
        const int in0 = t0 % a.d.page;
        for (int i = threadIdx.x; i < tn * W; i += blockDim.x) {
            const int r = i / W, c = i % W, in = in0 + r;
            const uint32_t eb = base[a.d.o_exp + in];
            const float unit = eb == 255u ? __uint_as_float(0x7fc00000u) : e8m0_to_f32(eb);
            float v;
            if (c < a.d.kv) {
                const uint32_t byte = base[(size_t)in * (a.d.kv / 2) + c / 2];
                const float2 f = f16x2_to_f32x2(e2m1x2_to_f16x2(byte));
                v = (c & 1 ? f.y : f.x) * e4m3_to_f32(base[a.d.o_scale + in * (a.d.kv / 16) + c / 16]);
            } else {
                v = __half2float(reinterpret_cast<const __half *>(base + a.d.o_rope)[in * a.d.rope + c - a.d.kv]);
            }
            tile[r][c] = v * unit;
        }
        __syncthreads();
        for (int r = 0; r < tn; r++) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 18; i++)
                if (lane + 32 * i < W) s = fmaf(q[i], tile[r][lane + 32 * i], s);
            s = warp_sum(s) * a.scale;
            const float mn = fmaxf(m, s);
            const float f = m == -INFINITY ? 0.f : expf(m - mn);
            const float p = s == -INFINITY ? 0.f : expf(s - mn);
            l = l * f + p;
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (lane + 32 * i < a.d.kv) acc[i] = fmaf(p, tile[r][lane + 32 * i], acc[i] * f);
            m = mn;
        }
    }
    if (h >= a.H) return;
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int c = lane + 32 * i;
        if (c < a.d.kv) {
            const size_t at = ((size_t)n * a.H + h) * a.d.kv + c;
            if (a.out_f32) ((float *)a.out)[at] = acc[i] * inv;
            else ((uint16_t *)a.out)[at] = f32_to_bf16_bits(acc[i] * inv);
        }
    }
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" {

size_t k3d_mla_attend4_ws_bytes(const K3dCache4 *c, int B, int N, int H)
{
    if (cache4_check(c, "k3d_mla_attend4_ws_bytes") || B < 1 || N < 0 || H < 1) return 0;
    return 256;
}

int k3d_mla_attend4(void *out, int out_dtype, const void *q, int q_dtype, const K3dCache4 *c, const void *pool,
                    const int *table, int max_pages, const int *row_start, const int *kv_len, int B, int N, int H,
                    float scale, void *ws, size_t ws_bytes)
{
    K3_TRY(cache4_check(c, "k3d_mla_attend4"));
    if (B < 1 || N < 0 || H < 1 || H > 1024 || max_pages < 1 || (long long)max_pages * c->page > 0x7fffffffLL)
        return fail(K3D_EINVAL, "k3d_mla_attend4: B %d, N %d, H %d (1 to 1024), max_pages %d", B, N, H, max_pages);
    for (int t : {out_dtype, q_dtype})
        if (t != K3D_DT_F32 && t != K3D_DT_BF16)
            return fail(K3D_EUNSUPPORTED, "k3d_mla_attend4: q and out are K3D_DT_F32 or K3D_DT_BF16, not %d", t);
    if (N == 0) return K3D_OK;
    if (!out || !q || !pool || !table || !row_start || !kv_len || !ws)
        return fail(K3D_EINVAL, "k3d_mla_attend4 null pointer");
    if (((uintptr_t)out | (uintptr_t)q | (uintptr_t)pool | (uintptr_t)ws) & 15u)
        return fail(K3D_EINVAL, "k3d_mla_attend4: out, q, pool and ws are 16-byte aligned");
    if (((uintptr_t)table | (uintptr_t)row_start | (uintptr_t)kv_len) & 3u)
        return fail(K3D_EINVAL, "k3d_mla_attend4: unaligned table, row_start or kv_len");
    if (ws_bytes < k3d_mla_attend4_ws_bytes(c, B, N, H)) return fail(K3D_EINVAL, "k3d_mla_attend4 workspace");
    K3_TRY(ensure_ctx());
    const Attend a{pool4(c, pool), q, out, table, row_start, kv_len, max_pages, B, N, H,
                   q_dtype == K3D_DT_F32, out_dtype == K3D_DT_F32, scale};
    launch_pdl(k_attend4_plain, dim3(N, (H + 7) / 8), dim3(256), 0, stream(), a);
    note_launch();
    return check_launch("mla attend4");
}

}  // extern "C"
