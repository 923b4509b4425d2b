// k3_sample.cu -- from logits to tokens beyond the greedy argmax of k3d_lm_head_argmax
// (argmax_, k3_run.c:134-135): the sampling probabilities of logits rows, and the
// verification of drafted tokens against them.
//
// Both give a row of the vocabulary to one cluster of CTAs, so that the row is read from
// memory once and the CTAs' partial results meet in distributed shared memory.
#include "k3_common.cuh"
#include "k3_ops.cuh"

namespace k3 {
namespace {

bool vec4(const void *p) { return !((uintptr_t)p & 15u); }

__device__ __forceinline__ uint32_t sm_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ float ex2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ int cl_rank()
{
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return (int)r;
}

__device__ __forceinline__ void cl_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t cl_map(uint32_t a, int rank)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}

__device__ __forceinline__ float cl_ld_f32(const void *p, int rank)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cl_map(sm_addr(p), rank)) : "memory");
    return v;
}

__device__ __forceinline__ unsigned long long cl_ld_u64(const void *p, int rank)
{
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cl_map(sm_addr(p), rank)) : "memory");
    return v;
}

// ------------------------------------------------------------------ probabilities ----
// p = exp((x - max) / T) / sum over a row of V. A NaN counts as minus infinity; with +inf
// in the row its places share the whole; a row without any finite or +inf value is zeros.
// T <= 0: 1 on the first maximum.
//
// A CTA owns the contiguous elements [c0, c1) of its row and passes over them twice: a running
// maximum and sum per thread (32 values at a time, one factor to a new maximum), one exchange
// over the cluster, then the probabilities, read again from L1 or L2 (the rows in work, two to
// four CTAs an SM, are below 100 MB) and written. Memory is read once and written once. Sums
// are fp32 per thread, then over the block and the cluster in a fixed order.
//
// Measured and left: the row kept in shared memory (82 KB a CTA) or in registers between the
// passes, 158 and 166 us for 320 rows of 163840: a cluster barrier waits for the loads in
// flight of the row behind it, and of the clusters of eight such CTAs only 15 lie on the card.
constexpr int kSmThreads = 512;

template <bool VEC>
__global__ void __launch_bounds__(kSmThreads, 2) k_logits_softmax(float *p, const float *x, const float *temp, int V,
                                                                 int chunk, int csize)
{
    __shared__ float red_m[kSmThreads / 32], red_s[kSmThreads / 32];
    __shared__ int red_i[kSmThreads / 32];
    __shared__ float x_m, x_s, x_n;                    // this CTA's maximum, its sum or first index, its +inf
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = cl_rank();
    const size_t r = blockIdx.x / csize;
    const int c0 = min(V, rank * chunk), n = min(V, c0 + chunk) - c0;
    const float *xr = x + r * (size_t)V + c0;
    float *pr = p + r * (size_t)V + c0;
    const float T = temp ? temp[r] : 1.0f;
    const float NEG = __int_as_float(0xff800000), POS = __int_as_float(0x7f800000);
    const bool greedy = !(T > 0.f);
    // 2 log2(e) / T, for differences that are taken in halves, since t - m alone may leave fp32 where
    // (t - m) / T does not; finite at a subnormal T: 0 c stays 0
    const float c = fminf(2.885390081777927f / T, 3.4028234e38f);
    constexpr int W = VEC ? 4 : 1, U = VEC ? 10 : 20, nw = kSmThreads / 32;   // values of a load, loads of a step
    // e^((t - 2 h) / T), h half of the largest; minus infinity is 0 at any temperature, an infinite one too
    auto weigh = [&](float t, float h) { return t > NEG ? ex2(fmaf(t, 0.5f, -h) * c) : 0.f; };
    auto load = [&](float v[U][W], int i0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * kSmThreads * W;
            if constexpr (VEC) {
                float4 t = make_float4(NEG, NEG, NEG, NEG);
                if (i < n) t = *reinterpret_cast<const float4 *>(xr + i);
                v[u][0] = t.x; v[u][1] = t.y; v[u][2] = t.z; v[u][3] = t.w;
            } else {
                v[u][0] = i < n ? xr[i] : NEG;
            }
        }
    };
    constexpr int step = U * kSmThreads * W;

    float m = NEG, s = 0.f;
    int first = 0x7fffffff;
    for (int i0 = tid * W; i0 < n; i0 += step) {
        float v[U][W];
        load(v, i0);
        float top = m;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int k = 0; k < W; k++) {
                v[u][k] = v[u][k] != v[u][k] ? NEG : v[u][k];
                top = fmaxf(top, v[u][k]);
            }
        if (greedy) {
            if (top > m) {
#pragma unroll
                for (int u = U - 1; u >= 0; u--)
#pragma unroll
                    for (int k = W - 1; k >= 0; k--)
                        if (v[u][k] == top) first = c0 + i0 + u * kSmThreads * W + k;
            }
        } else if (top < POS) {
            const float ref = top > NEG ? 0.5f * top : 0.f;
            s *= weigh(m, ref);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int k = 0; k < W; k++) s += weigh(v[u][k], ref);
        }
        m = top;
    }
    // the block's, then the cluster's
    const float mw = warp_max(m);
    if (lane == 0) red_m[warp] = mw;
    __syncthreads();
    float mc = red_m[0];
    for (int i = 1; i < nw; i++) mc = fmaxf(mc, red_m[i]);
    if (greedy) {
        first = __reduce_min_sync(0xffffffffu, m == mc ? first : 0x7fffffff);
        if (lane == 0) red_i[warp] = first;
    } else {
        s = warp_sum(m > NEG && mc < POS ? s * exp2f((0.5f * m - 0.5f * mc) * c) : 0.f);
        if (lane == 0) red_s[warp] = s;
    }
    __syncthreads();
    if (tid == 0) {
        float sc = 0.f;
        int fc = 0x7fffffff;
        for (int i = 0; i < nw; i++) {
            if (greedy) fc = min(fc, red_i[i]);
            else sc += red_s[i];
        }
        x_m = mc;
        x_s = greedy ? __int_as_float(fc) : sc;
    }
    cl_sync();
    // lane k has CTA k's (a loop over the CTAs in every thread took longer than a pass)
    const float mk = lane < csize ? cl_ld_f32(&x_m, lane) : NEG;
    const float sk = lane < csize ? cl_ld_f32(&x_s, lane) : 0.f;
    const float M = warp_max(mk);
    if (greedy) {
        const int best = __reduce_min_sync(0xffffffffu, lane < csize && M > NEG && mk == M ? __float_as_int(sk) : 0x7fffffff);
        for (int i = tid * W; i < n; i += kSmThreads * W) {
            if constexpr (VEC)
                *reinterpret_cast<float4 *>(pr + i) = make_float4(c0 + i == best, c0 + i + 1 == best, c0 + i + 2 == best, c0 + i + 3 == best);
            else
                pr[i] = c0 + i == best ? 1.f : 0.f;
        }
        cl_sync();                                     // nobody leaves while x_m and x_s are read
        return;
    }
    float S;
    if (M < POS) {
        S = warp_sum(lane < csize && mk > NEG ? sk * exp2f((0.5f * mk - 0.5f * M) * c) : 0.f);
    } else {
        // +inf in the row: its places are counted
        float k = 0.f;
        for (int i = tid; i < n; i += kSmThreads) k += xr[i] == POS ? 1.f : 0.f;
        k = warp_sum(k);
        __syncthreads();
        if (lane == 0) red_s[warp] = k;
        __syncthreads();
        if (tid == 0) {
            k = 0.f;
            for (int i = 0; i < nw; i++) k += red_s[i];
            x_n = k;
        }
        cl_sync();
        S = warp_sum(lane < csize ? cl_ld_f32(&x_n, lane) : 0.f);
    }
    const float inv = S > 0.f ? 1.0f / S : 0.f, ref = M > NEG ? 0.5f * M : 0.f;
    for (int i0 = tid * W; i0 < n; i0 += step) {
        float v[U][W];
        load(v, i0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * kSmThreads * W;
#pragma unroll
            for (int k = 0; k < W; k++) v[u][k] = (M < POS ? weigh(v[u][k], ref) : v[u][k] == POS ? 1.f : 0.f) * inv;
            if (i < n) {
                if constexpr (VEC)
                    __stcs(reinterpret_cast<float4 *>(pr + i), make_float4(v[u][0], v[u][1], v[u][2], v[u][3]));
                else
                    __stcs(pr + i, v[u][0]);
            }
        }
    }
    cl_sync();                                         // nobody leaves while its words are read
}

// ------------------------------------------------------------------- verification ----
// Draft i of a request is kept while u_i q_i(d_i) < p_i(d_i) (products of fp32 numbers,
// exact in 64 bits); with n of them kept the next token is drawn from max(p_n - q_n, 0), or
// from p_n where every draft was kept, at the place u of the weights' running sum. Each
// weight is taken as a whole number of 2^-44, so the sums are exact in 64 bits and the token
// does not depend on how the row is split or in which order it is added.
//
// One cluster per request: each CTA adds its contiguous share of the row, the CTAs' totals
// meet in distributed shared memory, and the CTA, then the warp, then the quarter of its share
// that the threshold falls into is walked once more. Bytes: one row of p and one of q per
// request. 64 registers (4 bytes spilled), and 512 threads while all CTAs are resident at once (two
// to an SM), else 256: with 512 threads of 100 registers, one CTA to an SM, 64 requests took 49 us.
constexpr int kVMax = 512;                // threads
constexpr int kVParts = 4;
constexpr int kMaxDraft = 32;
constexpr int kMaxVocab = 1 << 19;        // as many weights of 2^44 add up to 2^63: no row of p overflows the sums

struct Verify {
    int *tokens, *n_accept;
    const float *p, *q;
    const int *ids, *n_draft;
    const float *u, *us;
    int B, K, V, chunk, csize;
};

// r in whole 2^-44, truncated; NaN is 0, and a value above 1 is no probability. By the number's
// fields: mantissa x 2^21 shifted down by 127 - exponent (a conversion to 64 bits is slow).
__device__ __forceinline__ unsigned long long weight(float r)
{
    const uint32_t b = __float_as_uint(fminf(fmaxf(r, 0.f), 1.0f));
    const uint32_t e = b >> 23;
    const unsigned long long m = (unsigned long long)((b & 0x7fffffu) | 0x800000u) << 21;
    return m >> min(127u - e, 63u);                    // below 2^-63, subnormal numbers and 0: nothing is left
}

template <bool VEC>
__global__ void __launch_bounds__(kVMax, 2) k_spec_verify(Verify a)
{
    __shared__ unsigned long long wsum[kVMax / 32];
    __shared__ unsigned long long x_total;
    __shared__ int s_n;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = blockDim.x >> 5, rank = cl_rank();
    const int b = blockIdx.x / a.csize;
    const int K = a.K, V = a.V;
    // what does not depend on another load is sent for together
    const float us = a.us[b];
    const int nd0 = a.n_draft ? a.n_draft[b] : K;
    int id = -1;
    float ua = 0.f;
    if (warp == 0 && lane < K) {
        id = a.ids[(size_t)b * K + lane];
        ua = a.u[(size_t)b * K + lane];
    }
    const int nd = max(0, min(K, nd0));
    if (warp == 0) {
        bool kept = false;
        if (lane < nd) {
            if (id >= 0 && id < V) {
                const float pd = a.p[((size_t)b * (K + 1) + lane) * V + id];
                const float qd = a.q ? a.q[((size_t)b * K + lane) * V + id] : 1.0f;
                kept = (double)ua * (double)qd < (double)pd;
            }
        }
        const unsigned lost = __ballot_sync(0xffffffffu, !kept);
        const int n = lost ? min(nd, __ffs(lost) - 1) : nd;
        if (lane == 0) s_n = n;
    }
    __syncthreads();
    const int n = s_n;
    const bool cut0 = n < nd;                          // a draft was rejected
    const float *p = a.p + ((size_t)b * (K + 1) + n) * V;
    const float *q = cut0 && a.q ? a.q + ((size_t)b * K + n) * V : nullptr;
    const int one = cut0 && !a.q ? a.ids[(size_t)b * K + n] : -1;    // a draft without probabilities: all on one
    constexpr int W = VEC ? 4 : 1;

    // this warp's contiguous share [w0, w1), in quarters
    const int c0 = min(V, rank * a.chunk), c1 = min(V, c0 + a.chunk);
    const int quarter = (((c1 - c0) + nwarps * kVParts - 1) / (nwarps * kVParts) + 3) & ~3;
    const int w0 = min(c1, c0 + warp * quarter * kVParts), w1 = min(c1, w0 + quarter * kVParts);

    auto weights = [&](int i, bool cut, unsigned long long w[W]) {
        float v[W];
        if constexpr (VEC) {
            const float4 t = *reinterpret_cast<const float4 *>(p + i);
            v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        } else {
            v[0] = p[i];
        }
        if (cut) {
            if (q) {
                float z[W];
                if constexpr (VEC) {
                    const float4 t = *reinterpret_cast<const float4 *>(q + i);
                    z[0] = t.x; z[1] = t.y; z[2] = t.z; z[3] = t.w;
                } else {
                    z[0] = q[i];
                }
#pragma unroll
                for (int k = 0; k < W; k++) v[k] = v[k] - z[k];
            } else {
#pragma unroll
                for (int k = 0; k < W; k++)
                    if (i + k == one) v[k] = v[k] - 1.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < W; k++) w[k] = weight(v[k]);
    };

    bool cut = cut0;
    unsigned long long total = 0, before = 0, mine = 0, part[kVParts];
    for (int pass = 0; pass < 2; pass++) {
        unsigned long long s = 0;
#pragma unroll
        for (int z = 0; z < kVParts; z++) {
            const int z0 = min(w1, w0 + z * quarter), z1 = min(w1, z0 + quarter);
            part[z] = 0;
#pragma unroll 5
            for (int i = z0 + lane * W; i < z1; i += 32 * W) {
                unsigned long long w[W];
                weights(i, cut, w);
#pragma unroll
                for (int k = 0; k < W; k++) part[z] += w[k];
            }
            s += part[z];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) wsum[warp] = s;
        __syncthreads();
        mine = 0;
        for (int i = 0; i < nwarps; i++) mine += wsum[i];
        if (tid == 0) x_total = mine;
        cl_sync();
        // lane k has CTA k's total
        const unsigned long long xt = lane < a.csize ? cl_ld_u64(&x_total, lane) : 0;
        total = xt;
        before = lane < rank ? xt : 0;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            total += __shfl_xor_sync(0xffffffffu, total, o);
            before += __shfl_xor_sync(0xffffffffu, before, o);
        }
        total = __shfl_sync(0xffffffffu, total, 0);
        before = __shfl_sync(0xffffffffu, before, 0);
        cl_sync();                                     // every CTA has read the totals
        // p <= q everywhere leaves nothing: the draw is then from p itself
        if (total > 0 || !cut) break;
        cut = false;
    }
    // warp 0 still holds the drafts
    if (rank == 0 && warp == 0) {
        int *out = a.tokens + (size_t)b * (K + 1);
        if (lane < n) out[lane] = id;
        for (int i = lane; i <= K; i += 32)
            if (i > n || (i == n && total == 0)) out[i] = -1;
        if (lane == 0) a.n_accept[b] = n;
    }
    if (total == 0) return;
    // t = floor(u total): the token is the first whose running sum passes t
    unsigned long long t = 0;
    if (us > 0.f) {
        const double f = floor((double)us * (double)(long long)total);
        t = f >= (double)(long long)total ? total - 1 : (unsigned long long)f;
    }
    if (t < before || t >= before + mine) return;
    unsigned long long lead = before;
    for (int i = 0; i < warp; i++) lead += wsum[i];
    if (t < lead || t >= lead + wsum[warp]) return;
    int z0 = w0;
#pragma unroll
    for (int z = 0; z < kVParts; z++) {
        unsigned long long s = part[z];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (t >= lead + s && z < kVParts - 1) {
            lead += s;
            z0 = min(w1, z0 + quarter);
        } else {
            break;
        }
    }
    const int z1 = min(w1, z0 + quarter);
#pragma unroll 5
    for (int i0 = z0; i0 < z1; i0 += 32 * W) {
        const int i = i0 + lane * W;
        unsigned long long w[W];
#pragma unroll
        for (int k = 0; k < W; k++) w[k] = 0;
        if (i < z1) weights(i, cut, w);
        unsigned long long s = 0;
#pragma unroll
        for (int k = 0; k < W; k++) s += w[k];
        unsigned long long run = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, lead + run > t);
        if (hit) {
            if (lane == __ffs(hit) - 1) {
                unsigned long long c = lead + run - s;
                int at = i;
#pragma unroll
                for (int k = 0; k < W; k++) {
                    if (c > t) break;
                    c += w[k];
                    at = i + k;
                }
                a.tokens[(size_t)b * (K + 1) + n] = at;
            }
            return;
        }
        lead += __shfl_sync(0xffffffffu, run, 31);
    }
}

// CTAs to a row: sixteen (more than the portable eight) while the rows take no more than half of
// the SMs so, else eight or four while all of them lie on the card at once (two to an SM), else
// `many`. Each has 4096 elements at least, and 16384 where the rows fill the card anyway, since a
// CTA's start and exchanges then cost more than its share (300 rows of 10001: 27 us with a least
// share of 2048, 12 so; of 40000: 36 and 25; 64 rows of 163840: 24.5 us with eight CTAs, 19.3 with
// four). Verification takes its CTAs by the same rule: 64 requests are 24.2 us with eight and 24.5
// with four.
int cluster_of(int rows, int V, int many)
{
    const long long room = 2LL * sm_count();
    int cs = rows * 64LL <= room ? 16 : rows * 8LL <= room ? 8 : rows * 4LL <= room ? 4 : many;
    const int least = rows * 4LL > room ? 16384 : 4096;
    while (cs > 1 && V < (long long)cs * least) cs >>= 1;
    return cs;
}

// Lets a kernel run in clusters of sixteen; set once per kernel and device.
int wide_clusters(const void *f)
{
    static const void *done[64][8];
    int d = 0;
    cudaGetDevice(&d);
    for (const void *&e : done[d & 63]) {
        if (e == f) return K3D_OK;
        if (e) continue;
        if (cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
            cudaGetLastError();
            return fail(K3D_ECUDA, "clusters of sixteen CTAs");
        }
        e = f;
        return K3D_OK;
    }
    return K3D_OK;
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" {

int k3d_logits_softmax(float *p, const float *logits, const float *temp, int rows, int vocab)
{
    if (rows < 0 || vocab < 1 || vocab > 1 << 30) return fail(K3D_EINVAL, "k3d_logits_softmax: %d rows of %d", rows, vocab);
    if (rows == 0) return K3D_OK;
    if (!p || !logits) return fail(K3D_EINVAL, "k3d_logits_softmax null pointer");
    if (((uintptr_t)p | (uintptr_t)logits | (uintptr_t)temp) & 3u)
        return fail(K3D_EINVAL, "k3d_logits_softmax: unaligned pointer");
    if ((long long)rows * 8 > 0x7fffffffLL) return fail(K3D_EINVAL, "k3d_logits_softmax: %d rows", rows);
    K3_TRY(ensure_ctx());
    // four CTAs to a row where the rows fill the card (320 rows of 163840: 81 us with four, 93
    // with two, 99 with eight)
    const int cs = cluster_of(rows, vocab, 4);
    K3_TRY(wide_clusters(vec4(p) && vec4(logits) && vocab % 4 == 0 ? (const void *)k_logits_softmax<true>
                                                                    : (const void *)k_logits_softmax<false>));
    const int chunk = ((vocab + cs - 1) / cs + 3) & ~3;
    const bool vec = vec4(p) && vec4(logits) && vocab % 4 == 0;
    launch_pdl_cluster(vec ? k_logits_softmax<true> : k_logits_softmax<false>, dim3(rows * cs), dim3(kSmThreads), 0, stream(),
                       cs, p, logits, temp, vocab, chunk, cs);
    note_launch();
    return check_launch("logits softmax");
}

int k3d_spec_verify(int *tokens, int *n_accept, const float *target, const float *draft, const int *ids,
                    const int *n_draft, const float *u_accept, const float *u_sample, int B, int K, int vocab)
{
    if (B < 0 || K < 0 || K > kMaxDraft || vocab < 1 || vocab >= kMaxVocab)
        return fail(K3D_EINVAL, "k3d_spec_verify: B %d, K %d (0 to %d), vocab %d (below %d)", B, K, kMaxDraft, vocab, kMaxVocab);
    if (B == 0) return K3D_OK;
    if (!tokens || !n_accept || !target || !u_sample || (K > 0 && (!ids || !u_accept)))
        return fail(K3D_EINVAL, "k3d_spec_verify null pointer");
    if (((uintptr_t)tokens | (uintptr_t)n_accept | (uintptr_t)target | (uintptr_t)draft | (uintptr_t)ids |
         (uintptr_t)n_draft | (uintptr_t)u_accept | (uintptr_t)u_sample) & 3u)
        return fail(K3D_EINVAL, "k3d_spec_verify: unaligned pointer");
    if ((long long)B * 8 > 0x7fffffffLL) return fail(K3D_EINVAL, "k3d_spec_verify: B %d", B);
    K3_TRY(ensure_ctx());
    const int cs = cluster_of(B, vocab, 8);
    K3_TRY(wide_clusters(vec4(target) && vec4(draft) && vocab % 4 == 0 ? (const void *)k_spec_verify<true>
                                                                        : (const void *)k_spec_verify<false>));
    Verify a{tokens, n_accept, target, K > 0 ? draft : nullptr, ids, n_draft, u_accept, u_sample, B, K, vocab,
             ((vocab + cs - 1) / cs + 3) & ~3, cs};
    const bool vec = vec4(target) && vec4(draft) && vocab % 4 == 0;
    launch_pdl_cluster(vec ? k_spec_verify<true> : k_spec_verify<false>, dim3(B * cs), dim3(B * cs <= 2 * sm_count() ? kVMax : kVMax / 2), 0, stream(),
                       cs, a);
    note_launch();
    return check_launch("spec verify");
}

}  // extern "C"
