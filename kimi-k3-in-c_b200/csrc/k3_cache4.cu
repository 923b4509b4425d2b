// k3_cache4.cu -- rows of the paged 4-bit latent cache: quantise into slots, and read back.
// The counterpart for the bf16 cache is the row that k_mla_prep writes at the position
// (k3_mla.cu); the CPU engine's cache holds expanded fp32 keys (k3_ops.c:321-410).
#include "k3_cache4.cuh"
#include "k3_ops.cuh"

namespace k3 {

int cache4_check(const K3dCache4 *c, const char *who)
{
    if (!c) return fail(K3D_EINVAL, "%s: null cache shape", who);
    if (c->kv_lora < 128 || c->kv_lora > 512 || c->kv_lora % 128)
        return fail(K3D_EINVAL, "%s: kv_lora %d (a multiple of 128 up to 512)", who, c->kv_lora);
    if (c->qk_rope < 0 || c->qk_rope > 64 || c->qk_rope % 16)
        return fail(K3D_EINVAL, "%s: qk_rope %d (a multiple of 16 up to 64)", who, c->qk_rope);
    if (c->page < 16 || c->page > 1024 || c->page % 16)
        return fail(K3D_EINVAL, "%s: page %d (a multiple of 16 up to 1024)", who, c->page);
    if (c->n_pages < 1 || (long long)c->n_pages * c->page > 0x7fffffffLL)
        return fail(K3D_EINVAL, "%s: %d pages of %d rows (slots are 31-bit)", who, c->n_pages, c->page);
    return K3D_OK;
}

namespace {

constexpr int kRowWarps = 4;      // rows per CTA, one warp each

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(uint16_t v) { return bf16_to_f32(v); }

// n consecutive elements (8 or 16) starting at src, 16-byte loads when VEC.
template <bool VEC, int N>
__device__ __forceinline__ void load_n(float *v, const float *src)
{
    if (VEC) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const float4 t = reinterpret_cast<const float4 *>(src)[i];
            v[4 * i] = t.x; v[4 * i + 1] = t.y; v[4 * i + 2] = t.z; v[4 * i + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = src[i];
    }
}

template <bool VEC, int N>
__device__ __forceinline__ void load_n(float *v, const uint16_t *src)
{
    if (VEC) {
#pragma unroll
        for (int i = 0; i < N / 8; i++) {
            const uint4 t = reinterpret_cast<const uint4 *>(src)[i];
            const uint32_t u[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[8 * i + 2 * k] = __uint_as_float(u[k] << 16);
                v[8 * i + 2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = bf16_to_f32(src[i]);
    }
}

__device__ __forceinline__ float pow2f(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

// The smallest k with a <= m 2^k for m = lim x 2^-1 in [0.5, 1) and its binary exponent le
// (lim = m 2^le); -100 for a = 0.
__device__ __forceinline__ int unit_exp(float a, float m, int le)
{
    if (!(a > 0.f)) return -100;
    int e;
    const float f = frexpf(a, &e);
    return e - le + (f > m ? 1 : 0);
}

// One warp per row, lane l the 16-value block l of the latent and rope elements 2l, 2l + 1.
// All loads are issued before the row's maximum is formed; the code's three
// bits are exact comparisons of |y| with t s (t a midpoint of two codes, s four significant
// bits), so no quotient is rounded onto a tie. Traffic (2304 or 1152 bytes in, 417
// out per row at 512 + 64) and the arithmetic take about as long for prompts, one memory round
// trip is a decode step's time. 8191 bf16 rows stored and read back as fp32: 14.6 us (ten CTAs an
// SM; 15.0 without the bound, 17.5 with sixteen, which spill), 64 rows 3.8.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kRowWarps, 10) k_cache4_store(Pool4 d, const T *x, size_t ldx,
                                                                const int *slots, int N)
{
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int r = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    if (r >= N) return;
    const int slot = slots[r];                       // on its way together with the row
    const T *src = x + (size_t)r * ldx;
    const bool own = lane * 16 < d.kv, ropes = 2 * lane < d.rope;
    float v[16], rv[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = 0.f;
    if (own) load_n<VEC, 16>(v, src + lane * 16);
    if (ropes) {
        rv[0] = to_f(src[d.kv + 2 * lane]);
        rv[1] = to_f(src[d.kv + 2 * lane + 1]);
    }
    if (slot < 0 || slot >= d.n_pages * d.page) {
        if (slot != -1 && lane == 0) k3_raise_at(K3D_EBOUND, K3_SITE_CACHE4, r, slot, 0);
        return;
    }
    float amax = 0.f, rmax = fmaxf(fabsf(rv[0]), fabsf(rv[1]));
    bool fine = fabsf(rv[0]) <= 3.4028234e38f && fabsf(rv[1]) <= 3.4028234e38f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        amax = fmaxf(amax, fabsf(v[i]));
        fine = fine && fabsf(v[i]) <= 3.4028234e38f;      // false for a NaN or an infinity
    }
    fine = __all_sync(0xffffffffu, fine);
    const float lmax = warp_max(amax);
    rmax = warp_max(rmax);
    int k = max(-100, max(unit_exp(lmax, 0.65625f, 12), unit_exp(rmax, 0.5f, 16)));
    if (!fine) k = 0;
    // 2^-k in two factors: alone it leaves the range of fp32 at the smallest k
    const int half = (-k) >> 1;
    const float up = pow2f(half), up2 = pow2f(-k - half);
    const int pg = slot / d.page, in = slot - pg * d.page;
    uint8_t *base = d.p + (size_t)pg * d.page_bytes;
    if (own) {
        const float ay = fine ? amax * up * up2 : 0.f;
        const __nv_fp8_storage_t sb = __nv_cvt_float_to_fp8(__fdiv_rn(ay, 6.0f), __NV_SATFINITE, __NV_E4M3);
        // a scale of 0: nothing is above its midpoints
        const float s0 = e4m3_to_f32(sb), s = s0 > 0.f ? s0 : __int_as_float(0x7f800000);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float y = fine ? v[i] * up * up2 : 0.f;
            const float a = fabsf(y);
            const bool b2 = a >= 1.75f * s;
            const bool b1 = a >= (b2 ? 3.5f * s : 0.75f * s);
            const bool b0 = a > (b2 ? (b1 ? 5.0f * s : 2.5f * s) : (b1 ? 1.25f * s : 0.25f * s));
            const uint32_t c = ((__float_as_uint(y) >> 28) & 8u) | (b2 ? 4u : 0u) | (b1 ? 2u : 0u) | (b0 ? 1u : 0u);
            w[i >> 3] |= c << (4 * (i & 7));
        }
        *reinterpret_cast<uint2 *>(base + (size_t)in * (d.kv / 2) + lane * 8) = make_uint2(w[0], w[1]);
        base[d.o_scale + in * (d.kv / 16) + lane] = sb;
    }
    if (ropes) {
        const __half2 h = fine ? __floats2half2_rn(rv[0] * up * up2, rv[1] * up * up2) : __floats2half2_rn(0.f, 0.f);
        *reinterpret_cast<__half2 *>(base + d.o_rope + ((size_t)in * d.rope + 2 * lane) * 2) = h;
    }
    if (lane == 0) base[d.o_exp + in] = fine ? (uint8_t)(k + 127) : (uint8_t)255;
}

__device__ __forceinline__ void put_n(float *dst, const float *v, bool vec)
{
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            reinterpret_cast<float4 *>(dst)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) dst[i] = v[i];
    }
}

__device__ __forceinline__ void put_n(uint16_t *dst, const float *v, bool vec)
{
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        u[i] = (uint32_t)f32_to_bf16_bits(v[2 * i]) | ((uint32_t)f32_to_bf16_bits(v[2 * i + 1]) << 16);
    if (vec) {
        reinterpret_cast<uint4 *>(dst)[0] = make_uint4(u[0], u[1], u[2], u[3]);
        reinterpret_cast<uint4 *>(dst)[1] = make_uint4(u[4], u[5], u[6], u[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) dst[i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
    }
}

__device__ __forceinline__ void put_1(float *dst, float v) { *dst = v; }
__device__ __forceinline__ void put_1(uint16_t *dst, float v) { *dst = f32_to_bf16_bits(v); }

// The rows of `slots` as fp32 or bf16 (bf16 holds every latent value exactly; the fp16 rope
// part is rounded to it). One warp per row, the lanes as in the store.
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) k_cache4_load(Pool4 d, T *out, size_t ldo, const int *slots, int N,
                                                               int vec)
{
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int r = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    if (r >= N) return;
    const int slot = slots[r];
    if (slot < 0 || slot >= d.n_pages * d.page) {
        if (slot != -1 && lane == 0) k3_raise_at(K3D_EBOUND, K3_SITE_CACHE4, r, slot, 1);
        return;
    }
    const int pg = slot / d.page, in = slot - pg * d.page;
    const uint8_t *base = d.p + (size_t)pg * d.page_bytes;
    const bool own = lane * 16 < d.kv, ropes = 2 * lane < d.rope;
    uint2 w = make_uint2(0u, 0u);
    uint8_t sb = 0;
    __half2 h = __floats2half2_rn(0.f, 0.f);
    if (own) {
        w = *reinterpret_cast<const uint2 *>(base + (size_t)in * (d.kv / 2) + lane * 8);
        sb = base[d.o_scale + in * (d.kv / 16) + lane];
    }
    if (ropes) h = *reinterpret_cast<const __half2 *>(base + d.o_rope + ((size_t)in * d.rope + 2 * lane) * 2);
    const uint32_t eb = base[d.o_exp + in];
    const float unit = eb == 255u ? __uint_as_float(0x7fc00000u) : e8m0_to_f32(eb);
    T *dst = out + (size_t)r * ldo;
    if (own) {
        const float s = e4m3_to_f32(sb);
        uint32_t q[8];
        e2m1x8_to_f16x8(w.x, q);
        e2m1x8_to_f16x8(w.y, q + 4);
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float2 f = f16x2_to_f32x2(q[i]);
            v[2 * i] = f.x * s * unit;
            v[2 * i + 1] = f.y * s * unit;
        }
        put_n(dst + lane * 16, v, vec);
    }
    if (ropes) {
        const float2 f = __half22float2(h);
        put_1(dst + d.kv + 2 * lane, f.x * unit);
        put_1(dst + d.kv + 2 * lane + 1, f.y * unit);
    }
}

bool rows_vec(const void *p, size_t ld, size_t elem) { return !((uintptr_t)p & 15u) && !((ld * elem) & 15u); }

int rows_check(const K3dCache4 *c, const void *pool, const void *x, int dtype, size_t ld, const int *slots, int N,
               const char *who)
{
    K3_TRY(cache4_check(c, who));
    if (N < 0 || N > 1 << 30) return fail(K3D_EINVAL, "%s: %d rows (up to 2^30)", who, N);
    if (dtype != K3D_DT_F32 && dtype != K3D_DT_BF16)
        return fail(K3D_EUNSUPPORTED, "%s: rows are K3D_DT_F32 or K3D_DT_BF16, not %d", who, dtype);
    if (ld < (size_t)(c->kv_lora + c->qk_rope))
        return fail(K3D_EINVAL, "%s: %zu elements between rows of %d", who, ld, c->kv_lora + c->qk_rope);
    if (N == 0) return K3D_OK;
    if (!pool || !x || !slots) return fail(K3D_EINVAL, "%s: null pointer", who);
    if (((uintptr_t)pool & 15u) || ((uintptr_t)x & (dtype == K3D_DT_F32 ? 3u : 1u)) || ((uintptr_t)slots & 3u))
        return fail(K3D_EINVAL, "%s: the pool is 16-byte aligned, rows and slots by their element", who);
    return K3D_OK;
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" {

size_t k3d_cache4_bytes(const K3dCache4 *c)
{
    if (cache4_check(c, "k3d_cache4_bytes")) return 0;
    return pool4(c, nullptr).page_bytes * (size_t)c->n_pages;
}

int k3d_cache4_store(const K3dCache4 *c, void *pool, const void *x, int dtype, size_t ldx, const int *slots, int N)
{
    K3_TRY(rows_check(c, pool, x, dtype, ldx, slots, N, "k3d_cache4_store"));
    if (N == 0) return K3D_OK;
    K3_TRY(ensure_ctx());
    const Pool4 d = pool4(c, pool);
    const dim3 grid((N + kRowWarps - 1) / kRowWarps), block(32 * kRowWarps);
    const bool vec = rows_vec(x, ldx, dtype == K3D_DT_F32 ? 4 : 2);
    if (dtype == K3D_DT_F32)
        launch_pdl(vec ? k_cache4_store<float, true> : k_cache4_store<float, false>, grid, block, 0, stream(), d,
                   (const float *)x, ldx, slots, N);
    else
        launch_pdl(vec ? k_cache4_store<uint16_t, true> : k_cache4_store<uint16_t, false>, grid, block, 0, stream(), d,
                   (const uint16_t *)x, ldx, slots, N);
    note_launch();
    return check_launch("cache4 store");
}

int k3d_cache4_load(const K3dCache4 *c, const void *pool, void *out, int dtype, size_t ldo, const int *slots, int N)
{
    K3_TRY(rows_check(c, pool, out, dtype, ldo, slots, N, "k3d_cache4_load"));
    if (N == 0) return K3D_OK;
    K3_TRY(ensure_ctx());
    const Pool4 d = pool4(c, pool);
    const dim3 grid((N + kRowWarps - 1) / kRowWarps), block(32 * kRowWarps);
    const int vec = rows_vec(out, ldo, dtype == K3D_DT_F32 ? 4 : 2) ? 1 : 0;
    if (dtype == K3D_DT_F32)
        launch_pdl(k_cache4_load<float>, grid, block, 0, stream(), d, (float *)out, ldo, slots, N, vec);
    else
        launch_pdl(k_cache4_load<uint16_t>, grid, block, 0, stream(), d, (uint16_t *)out, ldo, slots, N, vec);
    note_launch();
    return check_launch("cache4 load");
}

}  // extern "C"
