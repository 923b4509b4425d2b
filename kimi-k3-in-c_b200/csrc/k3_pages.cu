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

constexpr int kMaxReq = 8192;            // requests per call: four arrays of 32 KB in shared memory
constexpr int kMaxPer = 8;               // requests per thread at most (1024 threads)

struct Plan {
    K3dPages p;
    const int *len, *nnew;
    int *row_start, *kv_len, *pos, *slots, *status;
    int B, N;
};

// exclusive prefixes and totals of three values per thread over the block, one barrier
struct Three { long long a, b, c; };

__device__ __forceinline__ Three block_scan(Three v, Three *total, Three *part)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    Three s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, s.a, o), y = __shfl_up_sync(0xffffffffu, s.b, o),
                        z = __shfl_up_sync(0xffffffffu, s.c, o);
        if (lane >= o) { s.a += x; s.b += y; s.c += z; }
    }
    if (lane == 31) part[warp] = s;
    __syncthreads();
    Three before = {0, 0, 0}, all = {0, 0, 0};
    for (int i = 0; i < nw; i++) {
        const Three t = part[i];
        if (i < warp) { before.a += t.a; before.b += t.b; before.c += t.c; }
        all.a += t.a; all.b += t.b; all.c += t.c;
    }
    *total = all;
    return Three{before.a + s.a - v.a, before.b + s.b - v.b, before.c + s.c - v.c};
}

// The request of row (or moved page) t: the last b with start[b] <= t (empty requests are passed over).
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

// One CTA: the scan over the requests, the stack, the tables, and, with `fill`, the rows too.
// The pages that move are dealt out over the threads whichever request they belong to (a
// thread for each request took 37 us with 100 prompts of up to 128 pages). What a call needs
// is three round trips to memory, so a small batch gets a small block. 64 requests of four tokens:
// 3 us, 100 prompts of up to 8192 tokens and their return, with the rows: 23 us.
__global__ void __launch_bounds__(1024) k_page_plan(Plan a, int fill)
{
    pdl_wait();
    pdl_trigger();
    extern __shared__ int start[];                  // [4][B + 1]: row starts, first page taken, first given back, need
    __shared__ Three part[32];
    __shared__ int s_bad;
    const int tid = threadIdx.x, nt = blockDim.x;
    int *s_grow = start + a.B + 1, *s_drop = s_grow + a.B + 1, *s_need = s_drop + a.B + 1;
    if (tid == 0) s_bad = 0;
    const int nf = *a.p.n_free;
    // a contiguous run of requests per thread
    const int per = (a.B + nt - 1) / nt;
    const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    int ln[kMaxPer], nw[kMaxPer], held[kMaxPer];
#pragma unroll
    for (int k = 0; k < kMaxPer; k++) {
        const bool on = b0 + k < b1;
        ln[k] = on ? a.len[b0 + k] : 0;
        nw[k] = on ? a.nnew[b0 + k] : 0;
        held[k] = on ? a.p.held[b0 + k] : 0;
    }
    __syncthreads();                                // s_bad is set
    Three mine = {0, 0, 0};                         // pages taken, pages given back, rows
    int bad = 0;
    // of lengths that add up to 31 bits; 32-bit unsigned, so the rounding up does not overflow
    auto need_of = [&](int k) { return (int)(((uint32_t)ln[k] + (uint32_t)nw[k] + (uint32_t)a.p.page - 1u) / (uint32_t)a.p.page); };
#pragma unroll
    for (int k = 0; k < kMaxPer; k++) {
        if (b0 + k >= b1) continue;
        if (ln[k] < 0 || nw[k] < 0 || held[k] < 0 || held[k] > a.p.max_pages || (long long)ln[k] + nw[k] > INT_MAX) {
            bad = K3D_PLAN_BAD;
            continue;
        }
        const int need = need_of(k);
        if (need > a.p.max_pages) bad = max(bad, K3D_PLAN_TABLE);
        mine.a += max(0, need - held[k]);
        mine.b += max(0, held[k] - need);
        mine.c += nw[k];
    }
    if (bad) atomicMax(&s_bad, bad);
    Three all;
    Three at = block_scan(mine, &all, part);        // its barrier also completes s_bad
    int code = s_bad;
    if (code == K3D_PLAN_OK) {
        if (nf < 0 || nf + all.b > a.p.n_pages) code = K3D_PLAN_BAD;
        else if (all.c > a.N) code = K3D_PLAN_ROWS;
        else if (all.a > nf + all.b) code = K3D_PLAN_PAGES;
    }
    const bool ok = code == K3D_PLAN_OK;
    if (tid == 0) {
        *a.status = code;
        a.row_start[a.B] = start[a.B] = ok ? (int)all.c : 0;
        s_grow[a.B] = ok ? (int)all.a : 0;
        s_drop[a.B] = ok ? (int)all.b : 0;
        if (ok) *a.p.n_free = (int)(nf + all.b - all.a);
    }
    // row starts and lengths; on a failure no request has rows
#pragma unroll
    for (int k = 0; k < kMaxPer; k++) {
        const int b = b0 + k;
        if (b >= b1) continue;
        a.row_start[b] = start[b] = ok ? (int)at.c : 0;
        a.kv_len[b] = ok ? ln[k] + nw[k] : 0;
        s_grow[b] = ok ? (int)at.a : 0;
        s_drop[b] = ok ? (int)at.b : 0;
        if (ok) {
            const int need = need_of(k);
            a.p.held[b] = s_need[b] = need;
            at.a += max(0, need - held[k]);
            at.b += max(0, held[k] - need);
            at.c += nw[k];
        }
    }
    __syncthreads();
    if (ok) {
        // pages after the call: the first of request b's that moved is its need (given back) or
        // its need less what was taken
        const int taken = (int)all.a, back = (int)all.b;
        // eight at a time: all the reads, then the writes (the compiler cannot tell that they do
        // not meet, and would wait for each read)
        for (int i0 = tid; i0 < back; i0 += 8 * nt) {
            int *e[8], page[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int i = i0 + k * nt;
                e[k] = nullptr;
                if (i < back) {
                    const int b = request_of(s_drop, a.B, i);
                    e[k] = a.p.table + (size_t)b * a.p.max_pages + s_need[b] + (i - s_drop[b]);
                    page[k] = *e[k];
                }
            }
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (e[k]) {
                    a.p.free_list[nf + back - 1 - (i0 + k * nt)] = page[k];
                    *e[k] = -1;
                }
        }
        if (back > 0) __syncthreads();              // what was given back may be taken
        for (int i0 = tid; i0 < taken; i0 += 8 * nt) {
            int page[8];
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (i0 + k * nt < taken) page[k] = a.p.free_list[nf + back - 1 - (i0 + k * nt)];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int i = i0 + k * nt;
                if (i < taken) {
                    const int b = request_of(s_grow, a.B, i);
                    a.p.table[(size_t)b * a.p.max_pages + s_need[b] - (s_grow[b + 1] - i)] = page[k];
                }
            }
        }
    }
    if (fill) {
        if (ok && all.a > 0) __syncthreads();       // the tables of the whole block
        for (int t = tid; t < a.N; t += nt) fill_row(a, start, t, start[a.B]);
    }
}

// Four consecutive rows to a thread: they share a search for their request most of the time,
// and go out as 16 bytes where the arrays allow it.
__global__ void __launch_bounds__(256) k_page_rows(Plan a, int vec)
{
    pdl_wait();
    pdl_trigger();
    extern __shared__ int start[];
    for (int i = threadIdx.x; i <= a.B; i += blockDim.x) start[i] = a.row_start[i];
    __syncthreads();
    const int rows = start[a.B];
    for (int t0 = (blockIdx.x * blockDim.x + threadIdx.x) * 4; t0 < a.N; t0 += gridDim.x * blockDim.x * 4) {
        int pos[4], slot[4], b = -1, end = 0, p = 0, q = 0, in = 0, base = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int t = t0 + k;
            pos[k] = slot[k] = -1;
            if (t >= rows) continue;
            bool turn = false;                      // another page
            if (b < 0 || t >= end) {
                b = request_of(start, a.B, t);
                end = start[b + 1];
                p = a.len[b] + t - start[b];
                q = (int)((uint32_t)p / (uint32_t)a.p.page);
                in = p - q * a.p.page;
                turn = true;
            } else {
                p++;
                if (++in == a.p.page) { in = 0; q++; turn = true; }
            }
            if (turn) base = a.p.table[(size_t)b * a.p.max_pages + q] * a.p.page;
            pos[k] = p;
            slot[k] = base + in;
        }
        if (vec && t0 + 4 <= a.N) {
            *reinterpret_cast<int4 *>(a.pos + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
            *reinterpret_cast<int4 *>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        } else {
            for (int k = 0; k < 4 && t0 + k < a.N; k++) {
                a.pos[t0 + k] = pos[k];
                a.slots[t0 + k] = slot[k];
            }
        }
    }
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" int k3d_page_plan(const K3dPages *p, const int *len, const int *n_new, int B, int N, int *row_start,
                             int *kv_len, int *pos, int *slots, int *status)
{
    if (!p || !p->table || !p->held || !p->free_list || !p->n_free || !len || !n_new || !row_start || !kv_len || !status)
        return fail(K3D_EINVAL, "k3d_page_plan null pointer");
    if (p->page < 1 || p->n_pages < 1 || p->n_pages > 1 << 30 || p->max_pages < 1 || (long long)p->page * p->n_pages > INT_MAX)
        return fail(K3D_EINVAL, "k3d_page_plan: page %d, n_pages %d, max_pages %d (slots are 31-bit)", p->page,
                    p->n_pages, p->max_pages);
    if (B < 1 || B > kMaxReq) return fail(K3D_EINVAL, "k3d_page_plan: %d requests (1 to %d)", B, kMaxReq);
    if (N < 0 || N > 1 << 30 || (N > 0 && (!pos || !slots))) return fail(K3D_EINVAL, "k3d_page_plan: %d rows", N);
    if (((uintptr_t)p->table | (uintptr_t)p->held | (uintptr_t)p->free_list | (uintptr_t)p->n_free | (uintptr_t)len |
         (uintptr_t)n_new | (uintptr_t)row_start | (uintptr_t)kv_len | (uintptr_t)pos | (uintptr_t)slots |
         (uintptr_t)status) & 3u)
        return fail(K3D_EINVAL, "k3d_page_plan: unaligned pointer");
    K3_TRY(ensure_ctx());
    const Plan a{*p, len, n_new, row_start, kv_len, pos, slots, status, B, N};
    const size_t smem = (size_t)(B + 1) * sizeof(int);
    static unsigned long long init = 0;                // one bit per device
    if (!(init & dev_bit())) {
        allow_smem_max(k_page_plan);
        init |= dev_bit();
    }
    // Up to 2048 rows the one CTA writes them itself; above, a second launch spreads them (us, by
    // the CTA and by a launch: 64 requests of 32 tokens 6.5 and 6.9, of 64 tokens 8.0 and 6.8).
    const int fill = N <= 2048 ? 1 : 0;
    // A small batch's time is the block's barriers and scans, a large one's the rows to a thread (us
    // with 256 and 1024 threads: 64 requests of one token 3.2 and 5.5, of four 3.3 and 5.5, 256 of four
    // 5.8 and 6.0, 64 of 32 tokens 7.8 and 6.7, 1024 of two 10.6 and 7.9; 300 of one token 4.7 and 5.9).
    const int threads = B <= 256 && N <= 1024 ? 256 : 1024;
    launch_pdl(k_page_plan, dim3(1), dim3(threads), 4 * smem, stream(), a, fill);
    note_launch();
    K3_TRY(check_launch("page plan"));
    if (!fill) {
        const int most = 8 * sm_count();
        const int grid = (N + 1023) / 1024;
        const int vec = !(((uintptr_t)pos | (uintptr_t)slots) & 15u) ? 1 : 0;
        launch_pdl(k_page_rows, dim3(grid < most ? grid : most), dim3(256), smem, stream(), a, vec);
        note_launch();
        K3_TRY(check_launch("page rows"));
    }
    return K3D_OK;
}
