// k3_pages.cu -- page tables and slot maps of a batch of requests, planned on the device.
// The CPU engine keeps one sequence in one contiguous cache (its position is a host
// counter, k3_run.c:158-300); the device-side plan of the expert exchange (k3_moe.cu) is the
// sibling: nothing is read back to the host, so a step with it captures into a graph.
//
// With need_b = ceil((len_b + new_b) / page) and held_b the pages that request b holds:
//   given back  pages need_b .. held_b - 1 go onto the free stack, the last page of the last
//               request first, so that what an earlier call took last lies deepest
//   taken       max(need_b - held_b, 0) pages come off the stack, requests in order
//   row_start   the exclusive prefix sum of new_b; pos and slot of each new row follow
// Taking n pages and giving the same n back leaves the stack as it was, entry for entry.
#include <limits.h>

#include "k3_common.cuh"
#include "k3_ops.cuh"

namespace k3 {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxReq = 8192;            // requests per call: 32 KB of row starts in shared memory
constexpr int kPer = kMaxReq / kPlanThreads;

struct Plan {
    K3dPages p;
    const int *len, *nnew;
    int *row_start, *kv_len, *pos, *slots, *status;
    int B, N;
};

// exclusive prefix and total of one value per thread over the block
__device__ __forceinline__ long long block_scan(long long v, long long *total, long long *part)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 31) part[warp] = s;
    __syncthreads();
    long long before = 0, all = 0;
    const int nw = blockDim.x >> 5;
    for (int i = 0; i < nw; i++) {
        const long long t = part[i];
        if (i < warp) before += t;
        all += t;
    }
    *total = all;
    return before + s - v;
}

// The request of row t: the last b with row_start[b] <= t (empty requests are passed over).
__device__ __forceinline__ int request_of(const int *start, int B, int t)
{
    int lo = 0, hi = B;                  // start[lo] <= t < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void fill_row(const Plan &a, const int *start, int t, int rows)
{
    int pos = -1, slot = -1;
    if (t < rows) {
        const int b = request_of(start, a.B, t);
        pos = a.len[b] + (t - start[b]);
        const int pg = pos / a.p.page;
        slot = a.p.table[(size_t)b * a.p.max_pages + pg] * a.p.page + (pos - pg * a.p.page);
    }
    a.pos[t] = pos;
    a.slots[t] = slot;
}

// One CTA: the scan over the requests, the stack, the tables, and, up to a.N rows given by
// `fill`, the rows too.
__global__ void __launch_bounds__(kPlanThreads) k_page_plan(Plan a, int fill)
{
    pdl_wait();
    pdl_trigger();
    extern __shared__ int start[];                  // [B + 1] row starts
    __shared__ long long part[32];
    __shared__ int s_bad;
    const int tid = threadIdx.x;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    // a contiguous run of requests per thread
    const int per = (a.B + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    int need[kPer], held[kPer];
    long long grow = 0, drop = 0, rows = 0;
    int bad = 0;
    for (int k = 0; k < per && b0 + k < b1; k++) {
        const int ln = a.len[b0 + k], nw = a.nnew[b0 + k], h = a.p.held[b0 + k];
        const long long total = (long long)ln + nw;
        if (ln < 0 || nw < 0 || h < 0 || h > a.p.max_pages || total > INT_MAX) {
            bad = max(bad, K3D_PLAN_BAD);
            need[k] = held[k] = 0;
            continue;
        }
        const int nd = (int)((total + a.p.page - 1) / a.p.page);
        if (nd > a.p.max_pages) bad = max(bad, K3D_PLAN_TABLE);
        need[k] = nd;
        held[k] = h;
        if (nd > h) grow += nd - h; else drop += h - nd;
        rows += nw;
    }
    if (bad) atomicMax(&s_bad, bad);
    long long all_grow, all_drop, all_rows;
    const long long g0 = block_scan(grow, &all_grow, part);
    const long long d0 = block_scan(drop, &all_drop, part);
    const long long r0 = block_scan(rows, &all_rows, part);
    const int nf = *a.p.n_free;
    __syncthreads();                                // s_bad is complete
    int code = s_bad;
    if (code == K3D_PLAN_OK) {
        if (nf < 0 || nf + all_drop > a.p.n_pages) code = K3D_PLAN_BAD;
        else if (all_rows > a.N) code = K3D_PLAN_ROWS;
        else if (all_grow > nf + all_drop) code = K3D_PLAN_PAGES;
    }
    const bool ok = code == K3D_PLAN_OK;
    if (tid == 0) {
        *a.status = code;
        a.row_start[a.B] = start[a.B] = ok ? (int)all_rows : 0;
    }
    // row starts and lengths; on a failure no request has rows
    {
        long long r = r0;
        for (int k = 0; k < per && b0 + k < b1; k++) {
            const int b = b0 + k;
            a.row_start[b] = start[b] = ok ? (int)r : 0;
            a.kv_len[b] = ok ? a.len[b] + a.nnew[b] : 0;
            if (ok) r += a.nnew[b];
        }
    }
    if (ok) {
        // given back: rank i of the releases in (request, page) order lies at nf + all_drop - 1 - i
        long long d = d0;
        for (int k = 0; k < per && b0 + k < b1; k++)
            for (int j = need[k]; j < held[k]; j++, d++) {
                int *e = a.p.table + (size_t)(b0 + k) * a.p.max_pages + j;
                a.p.free_list[nf + all_drop - 1 - d] = *e;
                *e = -1;
            }
        __syncthreads();
        const long long have = nf + all_drop;
        long long g = g0;
        for (int k = 0; k < per && b0 + k < b1; k++) {
            for (int j = held[k]; j < need[k]; j++, g++)
                a.p.table[(size_t)(b0 + k) * a.p.max_pages + j] = a.p.free_list[have - 1 - g];
            a.p.held[b0 + k] = need[k];
        }
        if (tid == 0) *a.p.n_free = (int)(have - all_grow);
    }
    __syncthreads();                                // tables and row starts of the whole block
    if (fill)
        for (int t = tid; t < a.N; t += kPlanThreads) fill_row(a, start, t, start[a.B]);
}

__global__ void __launch_bounds__(256) k_page_rows(Plan a)
{
    pdl_wait();
    pdl_trigger();
    extern __shared__ int start[];
    for (int i = threadIdx.x; i <= a.B; i += blockDim.x) start[i] = a.row_start[i];
    __syncthreads();
    for (int t = blockIdx.x * blockDim.x + threadIdx.x; t < a.N; t += gridDim.x * blockDim.x)
        fill_row(a, start, t, start[a.B]);
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" int k3d_page_plan(const K3dPages *p, const int *len, const int *n_new, int B, int N, int *row_start,
                             int *kv_len, int *pos, int *slots, int *status)
{
    if (!p || !p->table || !p->held || !p->free_list || !p->n_free || !len || !n_new || !row_start || !kv_len || !status)
        return fail(K3D_EINVAL, "k3d_page_plan null pointer");
    if (p->page < 1 || p->n_pages < 1 || p->max_pages < 1 || (long long)p->page * p->n_pages > INT_MAX)
        return fail(K3D_EINVAL, "k3d_page_plan: page %d, n_pages %d, max_pages %d (slots are 31-bit)", p->page,
                    p->n_pages, p->max_pages);
    if (B < 1 || B > kMaxReq) return fail(K3D_EINVAL, "k3d_page_plan: %d requests (1 to %d)", B, kMaxReq);
    if (N < 0 || (N > 0 && (!pos || !slots))) return fail(K3D_EINVAL, "k3d_page_plan: %d rows", N);
    K3_TRY(ensure_ctx());
    const Plan a{*p, len, n_new, row_start, kv_len, pos, slots, status, B, N};
    const size_t smem = (size_t)(B + 1) * sizeof(int);
    // Up to 4096 rows the one CTA writes them itself; above, a second launch spreads them.
    const int fill = N <= 4096 ? 1 : 0;
    launch_pdl(k_page_plan, dim3(1), dim3(kPlanThreads), smem, stream(), a, fill);
    note_launch();
    K3_TRY(check_launch("page plan"));
    if (!fill) {
        const int most = 8 * sm_count();
        const int grid = (N + 255) / 256;
        launch_pdl(k_page_rows, dim3(grid < most ? grid : most), dim3(256), smem, stream(), a);
        note_launch();
        K3_TRY(check_launch("page rows"));
    }
    return K3D_OK;
}
