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
// A CTA owns the contiguous elements [c0, c1) of its row: it keeps up to `keep` of them in
// shared memory while it reads them (the rest is read again), so a row of 163840 costs one
// read and one write of memory. Sums are fp32 per thread, then over the block and the
// cluster in a fixed order.
constexpr int kSmThreads = 512;

__device__ __forceinline__ float block_max(float v, float *red)
{
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < (int)(blockDim.x >> 5); i++) v = fmaxf(v, red[i]);
    return v;
}

__device__ __forceinline__ float block_sum(float v, float *red)
{
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < (int)(blockDim.x >> 5); i++) v += red[i];
    return v;
}

template <bool VEC>
__global__ void __launch_bounds__(kSmThreads) k_logits_softmax(float *p, const float *x, const float *temp, int V,
                                                              int chunk, int keep, int csize)
{
    extern __shared__ __align__(16) float row[];       // [keep]
    __shared__ float red[32];
    __shared__ float x_f[2];                           // this CTA's maximum, then sum
    __shared__ int x_i;                                // index of its first maximum
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, rank = cl_rank();
    const size_t r = blockIdx.x / csize;
    const float *xr = x + r * (size_t)V;
    float *pr = p + r * (size_t)V;
    const int c0 = min(V, rank * chunk), n = min(V, c0 + chunk) - c0;
    const float NEG = __int_as_float(0xff800000);
    xr += c0;
    pr += c0;
    constexpr int W = VEC ? 4 : 1;

    auto load = [&](int i, float v[W]) {
        if constexpr (VEC) {
            const float4 t = *reinterpret_cast<const float4 *>(xr + i);
            v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        } else {
            v[0] = xr[i];
        }
#pragma unroll
        for (int k = 0; k < W; k++)
            if (v[k] != v[k]) v[k] = NEG;
    };

    float m = NEG;
#pragma unroll 8
    for (int i = tid * W; i < n; i += kSmThreads * W) {
        float v[W];
        load(i, v);
#pragma unroll
        for (int k = 0; k < W; k++) {
            m = fmaxf(m, v[k]);
            if (i + k < keep) row[i + k] = v[k];
        }
    }
    m = block_max(m, red);
    if (tid == 0) x_f[0] = m;
    cl_sync();
    const int lane = tid & 31;                         // lane k looks at CTA k
    const float M = warp_max(lane < csize ? cl_ld_f32(&x_f[0], lane) : NEG);
    const float T = temp ? temp[r] : 1.0f;

    auto value = [&](int i, float v[W]) {
        if (i + W <= keep) {
#pragma unroll
            for (int k = 0; k < W; k++) v[k] = row[i + k];
        } else {
            load(i, v);
        }
    };
    // e^((x - max) / T); minus infinity is 0 at any temperature, an infinite one too
    auto weigh = [&](float x, float ref, float c, bool inf) {
        if (inf) return x == M ? 1.f : 0.f;
        return x > NEG ? exp2f((x - ref) * c) : 0.f;
    };
    auto put = [&](int i, const float v[W]) {
        if constexpr (VEC) {
            *reinterpret_cast<float4 *>(pr + i) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            pr[i] = v[0];
        }
    };

    if (!(T > 0.f)) {
        // greedy: the lowest index that holds the maximum (none in a row of minus infinities)
        int first = 0x7fffffff;
        if (M > NEG)
            for (int i = tid * W; i < n; i += kSmThreads * W) {
                float v[W];
                value(i, v);
#pragma unroll
                for (int k = 0; k < W; k++)
                    if (v[k] == M) first = min(first, c0 + i + k);
            }
        first = __reduce_min_sync(0xffffffffu, first);
        if (tid == 0) x_i = 0x7fffffff;
        __syncthreads();
        if ((tid & 31) == 0) atomicMin(&x_i, first);
        cl_sync();
        const int at = __reduce_min_sync(0xffffffffu, lane < csize ? __float_as_int(cl_ld_f32(&x_i, lane)) : 0x7fffffff);
        for (int i = tid * W; i < n; i += kSmThreads * W) {
            float v[W];
#pragma unroll
            for (int k = 0; k < W; k++) v[k] = c0 + i + k == at ? 1.0f : 0.0f;
            put(i, v);
        }
        cl_sync();                                     // nobody leaves while x_i is read
        return;
    }
    const float c = 1.4426950408889634f / T;
    const bool inf = M == __int_as_float(0x7f800000);
    const float ref = M > NEG ? M : 0.f;
    float s = 0.f;
#pragma unroll 4
    for (int i = tid * W; i < n; i += kSmThreads * W) {
        float v[W];
        value(i, v);
#pragma unroll
        for (int k = 0; k < W; k++) {
            v[k] = weigh(v[k], ref, c, inf);
            s += v[k];
            if (i + k < keep) row[i + k] = v[k];
        }
    }
    s = block_sum(s, red);
    if (tid == 0) x_f[1] = s;
    cl_sync();
    const float S = warp_sum(lane < csize ? cl_ld_f32(&x_f[1], lane) : 0.f);
    const float inv = S > 0.f ? 1.0f / S : 0.f;
#pragma unroll 4
    for (int i = tid * W; i < n; i += kSmThreads * W) {
        float v[W];
        if (i + W <= keep) {
#pragma unroll
            for (int k = 0; k < W; k++) v[k] = row[i + k];
        } else {
            load(i, v);
#pragma unroll
            for (int k = 0; k < W; k++) v[k] = weigh(v[k], ref, c, inf);
        }
#pragma unroll
        for (int k = 0; k < W; k++) v[k] *= inv;
        put(i, v);
    }
    cl_sync();                                         // nobody leaves while x_f is read
}

// The same for rows that fit a cluster's registers (163840 in eight CTAs): a thread has 4 PER
// values of its CTA's share, and the next row's loads are on their way while this one's sums
// meet, so that a card full of clusters reads and writes without a pause. A CTA takes e^((x -
// m_c) / T) against its own maximum m_c, so that one exchange (m_c, sum) over the cluster
// serves both reductions. With a block of shared memory per row and CTA instead (the kernel
// above, which stays for longer rows) 320 rows of 163840 took 158 us.
template <bool VEC, int PER>
__global__ void __launch_bounds__(kSmThreads, 1) k_logits_softmax_reg(float *p, const float *x, const float *temp, int rows,
                                                                     int V, int chunk, int csize)
{
    __shared__ float red[2][kSmThreads / 32];
    __shared__ int red_i[kSmThreads / 32];
    __shared__ float x_m[2], x_s[2];                   // this CTA's maximum, and its sum or first index
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = cl_rank();
    const int c0 = min(V, rank * chunk), n = min(V, c0 + chunk) - c0;
    const int step = gridDim.x / csize;
    const float NEG = __int_as_float(0xff800000), POS = __int_as_float(0x7f800000);
    constexpr int nw = kSmThreads / 32;
    auto at = [&](int k, int j) { return VEC ? (k * kSmThreads + tid) * 4 + j : (k * 4 + j) * kSmThreads + tid; };
    auto load = [&](float v[PER][4], int r) {
        const float *xr = x + (size_t)r * V + c0;
#pragma unroll
        for (int k = 0; k < PER; k++) {
            if constexpr (VEC) {
                float4 t = make_float4(NEG, NEG, NEG, NEG);
                if (at(k, 0) < n) t = *reinterpret_cast<const float4 *>(xr + at(k, 0));
                v[k][0] = t.x; v[k][1] = t.y; v[k][2] = t.z; v[k][3] = t.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) v[k][j] = at(k, j) < n ? xr[at(k, j)] : NEG;
            }
        }
    };
    float v[PER][4];
    int r = blockIdx.x / csize, turn = 0;
    load(v, r);
    for (; r < rows; r += step, turn ^= 1) {
        float nx[PER][4];
        if (r + step < rows) load(nx, r + step);
        const float T = temp ? temp[r] : 1.0f;
        float m = NEG;
#pragma unroll
        for (int k = 0; k < PER; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (v[k][j] != v[k][j]) v[k][j] = NEG;
                m = fmaxf(m, v[k][j]);
            }
        m = warp_max(m);
        if (lane == 0) red[0][warp] = m;
        __syncthreads();
        m = red[0][0];
        for (int i = 1; i < nw; i++) m = fmaxf(m, red[0][i]);
        const bool greedy = !(T > 0.f);
        const float c = 1.4426950408889634f / T;
        if (greedy) {
            int first = 0x7fffffff;
            if (m > NEG) {
#pragma unroll
                for (int k = 0; k < PER; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (v[k][j] == m) first = min(first, c0 + at(k, j));
            }
            first = __reduce_min_sync(0xffffffffu, first);
            if (lane == 0) red_i[warp] = first;
            __syncthreads();
            if (tid == 0) {
                for (int i = 0; i < nw; i++) first = min(first, red_i[i]);
                x_m[turn] = m;
                x_s[turn] = __int_as_float(first);
            }
        } else {
            const float ref = m > NEG ? m : 0.f;
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < PER; k++) {
                float part = 0.f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float t = v[k][j];
                    // minus infinity is 0 at any temperature, an infinite one too
                    v[k][j] = m == POS ? (t == POS ? 1.f : 0.f) : t > NEG ? exp2f((t - ref) * c) : 0.f;
                    part += v[k][j];
                }
                s += part;
            }
            s = warp_sum(s);
            if (lane == 0) red[1][warp] = s;
            __syncthreads();
            if (tid == 0) {
                s = 0.f;
                for (int i = 0; i < nw; i++) s += red[1][i];
                x_m[turn] = m;
                x_s[turn] = s;
            }
        }
        cl_sync();
        // lane k has CTA k's (a loop over the CTAs in every thread cost more than the row's sums)
        const float mk = lane < csize ? cl_ld_f32(&x_m[turn], lane) : NEG;
        const float sk = lane < csize ? cl_ld_f32(&x_s[turn], lane) : 0.f;
        const float M = warp_max(mk);
        float *pr = p + (size_t)r * V + c0;
        float f = 0.f;
        int best = 0x7fffffff;
        if (greedy) {
            best = __reduce_min_sync(0xffffffffu, lane < csize && M > NEG && mk == M ? __float_as_int(sk) : 0x7fffffff);
        } else {
            // a CTA's share of the whole: e^((m_c - M) / T) over the sum
            auto scale = [&](float mc) { return mc == M ? 1.f : M == POS || mc == NEG ? 0.f : exp2f((mc - M) * c); };
            const float S = warp_sum(lane < csize ? sk * scale(mk) : 0.f);
            f = S > 0.f ? scale(m) / S : 0.f;
        }
#pragma unroll
        for (int k = 0; k < PER; k++) {
            float o[4];
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = greedy ? (c0 + at(k, j) == best ? 1.f : 0.f) : v[k][j] * f;
            if constexpr (VEC) {
                if (at(k, 0) < n) *reinterpret_cast<float4 *>(pr + at(k, 0)) = make_float4(o[0], o[1], o[2], o[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (at(k, j) < n) pr[at(k, j)] = o[j];
            }
        }
#pragma unroll
        for (int k = 0; k < PER; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) v[k][j] = nx[k][j];
    }
    cl_sync();                                         // nobody leaves while x_m and x_s are read
}

template <bool VEC, int PER>
int softmax_reg(float *p, const float *x, const float *temp, int rows, int V, int chunk, int cs)
{
    // clusters that lie on the card at once, by device and cluster size
    static int fit[64][9];
    int d = 0;
    cudaGetDevice(&d);
    int &n = fit[d & 63][cs];
    if (n == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(cs);
        cfg.blockDim = dim3(kSmThreads);
        cudaLaunchAttribute a;
        a.id = cudaLaunchAttributeClusterDimension;
        a.val.clusterDim.x = (unsigned)cs;
        a.val.clusterDim.y = a.val.clusterDim.z = 1;
        cfg.attrs = &a;
        cfg.numAttrs = 1;
        int got = 0;
        if (cudaOccupancyMaxActiveClusters(&got, k_logits_softmax_reg<VEC, PER>, &cfg) != cudaSuccess || got < 1) {
            cudaGetLastError();
            got = 1;
        }
        n = got;
    }
    launch_pdl_cluster(k_logits_softmax_reg<VEC, PER>, dim3((rows < n ? rows : n) * cs), dim3(kSmThreads), 0, stream(), cs, p, x,
                       temp, rows, V, chunk, cs);
    note_launch();
    return check_launch("logits softmax");
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
// request. 256 threads and 64 registers, so that four CTAs lie on an SM: with 512 threads of
// 100 registers 64 requests took 49 us.
constexpr int kVThreads = 256;
constexpr int kVWarps = kVThreads / 32;
constexpr int kVParts = 4;
constexpr int kMaxDraft = 32;

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
__global__ void __launch_bounds__(kVThreads, 4) k_spec_verify(Verify a)
{
    __shared__ unsigned long long wsum[kVWarps];
    __shared__ unsigned long long x_total;
    __shared__ int s_n;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = cl_rank();
    const int b = blockIdx.x / a.csize;
    const int K = a.K, V = a.V;
    const int nd = a.n_draft ? max(0, min(K, a.n_draft[b])) : K;
    int id = -1;
    if (warp == 0) {
        bool kept = false;
        if (lane < nd) {
            id = a.ids[(size_t)b * K + lane];
            if (id >= 0 && id < V) {
                const float pd = a.p[((size_t)b * (K + 1) + lane) * V + id];
                const float qd = a.q ? a.q[((size_t)b * K + lane) * V + id] : 1.0f;
                kept = (double)a.u[(size_t)b * K + lane] * (double)qd < (double)pd;
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
    const float us = a.us[b];
    constexpr int W = VEC ? 4 : 1;

    // this warp's contiguous share [w0, w1), in quarters
    const int c0 = min(V, rank * a.chunk), c1 = min(V, c0 + a.chunk);
    const int quarter = (((c1 - c0) + kVWarps * kVParts - 1) / (kVWarps * kVParts) + 3) & ~3;
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
        for (int i = 0; i < kVWarps; i++) mine += wsum[i];
        if (tid == 0) x_total = mine;
        cl_sync();
        // lane k has CTA k's total
        const unsigned long long xt = lane < a.csize ? cl_ld_u64(&x_total, lane) : 0;
        total = xt;
        before = lane < rank ? xt : 0;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
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

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" {

int k3d_logits_softmax(float *p, const float *logits, const float *temp, int rows, int vocab)
{
    if (rows < 0 || vocab < 1) return fail(K3D_EINVAL, "k3d_logits_softmax: %d rows of %d", rows, vocab);
    if (rows == 0) return K3D_OK;
    if (!p || !logits) return fail(K3D_EINVAL, "k3d_logits_softmax null pointer");
    if (((uintptr_t)p | (uintptr_t)logits | (uintptr_t)temp) & 3u)
        return fail(K3D_EINVAL, "k3d_logits_softmax: unaligned pointer");
    if ((long long)rows * 8 > 0x7fffffffLL) return fail(K3D_EINVAL, "k3d_logits_softmax: %d rows", rows);
    K3_TRY(ensure_ctx());
    // the largest cluster whose CTAs still have a few thousand elements each
    int cs = 8;
    while (cs > 1 && vocab < cs * 2048) cs >>= 1;
    const int chunk = ((vocab + cs - 1) / cs + 3) & ~3;
    const bool vec = vec4(p) && vec4(logits) && vocab % 4 == 0;
    const int per = (chunk + 4 * kSmThreads - 1) / (4 * kSmThreads);
    if (per <= 2)
        return vec ? softmax_reg<true, 2>(p, logits, temp, rows, vocab, chunk, cs)
                   : softmax_reg<false, 2>(p, logits, temp, rows, vocab, chunk, cs);
    if (per <= 5)
        return vec ? softmax_reg<true, 5>(p, logits, temp, rows, vocab, chunk, cs)
                   : softmax_reg<false, 5>(p, logits, temp, rows, vocab, chunk, cs);
    if (per <= 10)
        return vec ? softmax_reg<true, 10>(p, logits, temp, rows, vocab, chunk, cs)
                   : softmax_reg<false, 10>(p, logits, temp, rows, vocab, chunk, cs);
    const int cap = 50 * 1024;                         // floats that fit beside the static arrays
    const int keep = chunk < cap ? chunk : cap;
    static unsigned long long init = 0;                // one bit per device
    if (!(init & dev_bit())) {
        allow_smem_max(k_logits_softmax<true>);
        allow_smem_max(k_logits_softmax<false>);
        init |= dev_bit();
    }
    launch_pdl_cluster(vec ? k_logits_softmax<true> : k_logits_softmax<false>, dim3(rows * cs), dim3(kSmThreads),
                       (size_t)keep * 4, stream(), cs, p, logits, temp, vocab, chunk, keep, cs);
    note_launch();
    return check_launch("logits softmax");
}

int k3d_spec_verify(int *tokens, int *n_accept, const float *target, const float *draft, const int *ids,
                    const int *n_draft, const float *u_accept, const float *u_sample, int B, int K, int vocab)
{
    if (B < 0 || K < 0 || K > kMaxDraft || vocab < 1)
        return fail(K3D_EINVAL, "k3d_spec_verify: B %d, K %d (0 to %d), vocab %d", B, K, kMaxDraft, vocab);
    if (B == 0) return K3D_OK;
    if (!tokens || !n_accept || !target || !u_sample || (K > 0 && (!ids || !u_accept)))
        return fail(K3D_EINVAL, "k3d_spec_verify null pointer");
    if (((uintptr_t)tokens | (uintptr_t)n_accept | (uintptr_t)target | (uintptr_t)draft | (uintptr_t)ids |
         (uintptr_t)n_draft | (uintptr_t)u_accept | (uintptr_t)u_sample) & 3u)
        return fail(K3D_EINVAL, "k3d_spec_verify: unaligned pointer");
    if ((long long)B * 8 > 0x7fffffffLL) return fail(K3D_EINVAL, "k3d_spec_verify: B %d", B);
    K3_TRY(ensure_ctx());
    int cs = 8;
    while (cs > 1 && vocab < cs * 2048) cs >>= 1;
    Verify a{tokens, n_accept, target, K > 0 ? draft : nullptr, ids, n_draft, u_accept, u_sample, B, K, vocab,
             ((vocab + cs - 1) / cs + 3) & ~3, cs};
    const bool vec = vec4(target) && vec4(draft) && vocab % 4 == 0;
    launch_pdl_cluster(vec ? k_spec_verify<true> : k_spec_verify<false>, dim3(B * cs), dim3(kVThreads), 0, stream(), cs, a);
    note_launch();
    return check_launch("spec verify");
}

}  // extern "C"
