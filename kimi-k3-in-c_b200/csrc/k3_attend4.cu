// k3_attend4.cu -- absorbed MLA attention over the paged 4-bit latent cache, for any number
// of new tokens per request (k3_mla_cached, k3_ops.c:321-410, in the absorbed form of
// k3_mla.cu; the row format is in k3_cache4.cuh).
//
//   s[r][t] = scale q[r] . row[t],  t < the keys that row r sees
//   o[r]    = sum_t softmax(s[r])[t] row[t][0 .. kv)
// Row r = (new token j of request b, head): it sees the first kv_len[b] - new_b + j + 1
// positions (none: zeros).
//
// WORK. The rows of a request are contiguous in q ([N][H] flattened); an item is up to 64 of
// them (whole tokens when H <= 64, else 64 heads of one token), or up to 32 or 16 where few items
// would leave SMs idle: Q, the result and the merge are then spread. An item counts one unit for
// each tile of 64 positions and five for its start (Q, the first tile's way through the
// pipeline and the result take about as long as five tiles, 10 us), the units of all items,
// item-major, are cut into one contiguous range per CTA, and a cut that falls into an item's
// start moves to its beginning. So ragged lengths balance themselves: 142 -> 114 us for 16
// ragged requests of four tokens, 64 heads, up to 8192 positions, against ranges of tiles
// alone, where a CTA that met four items took half as long again as the average one. An item
// that one CTA covers is written directly; the parts of a cut item (at most two per CTA) go to
// the workspace as (unnormalised o, max, sum) and a second kernel adds them in CTA order.
// Units are numbered in 31 bits: a call of more than 2^30 raises K3D_EBOUND.
//
// PRODUCTS (tcgen05, fp16 x fp16, fp32 accumulators in tensor memory). A tile's rows are
// widened once to fp16, 64 values to a 128-byte swizzled panel row, and serve both products
// from the same bytes:
//   S [64 rows][64 keys]     = Q K^T      M = 64, K-major A = Q and B = the tile
//   O^T [kv][rows] (4 x 128) += V^T P^T   M = 128 latents, A = the tile read MN-major,
//                                         B = P, K-major, N = the rows rounded up to 16
// O^T rather than O keeps the accumulator of 64 rows in 256 of the 512 columns, which leaves
// room for two S; O of 64 rows and 512 latents would fill all of them.
//
// UNITS. The fp16 operand holds values in units of 2^-2. A stored row's latents are multiples of
// 2^-10 of its own 2^e, so for -16 <= e <= -2 (largest latent between 0.02 and 672) their step to
// 2^-2 is exact in fp16. A row outside keeps a residual 2^r in fp32: its scores are multiplied by
// it, and its weight P carries it into the second product, so that latents of any size stay exact.
// The rotated key is any fp16 number of 2^e: for e < -2 its step rounds by at most 2^-25 of the unit
// 2^(-2 + r), 2^-11 of 2^e at most, where the row's largest value is at least 1344 of them. q is
// fp16 in units of its row (exact for bf16 within 2^-29 of the row's largest value).
//
// SOFTMAX. With a = s log2(e) + r: P = 2^(a - m + 7), rounded to fp16 (half a step is 2^-12
// on average, an eighth of a bf16 result's), and the sum takes 2^(a - r - m + 7) in fp32. m
// moves only when a tile's maximum passes it by 2^8, so the accumulator is rescaled rarely;
// P stays below 2^15 and weights down to 2^-21 of the largest keep all their bits.
//
// ROLES (448 threads): warps 0-7 load a tile ahead into registers, widen and store it;
// warps 8-11 do the softmax and the rescaling; these 12 load Q and write the results; warp
// 12 issues S, warp 13 O^T. A tile is handed over in pieces of 256 latents: O(t) frees a piece
// of the buffer, the widening of tile t + 2 fills it while O(t) goes on, and S(t + 2) follows
// it, so that the softmax of tile t + 1 has the length of O(t) and S(t + 2) to run in. Up to 32
// rows P is held for two tiles in turn, so that it is written while O(t - 1) runs (16 heads: 70 ->
// 68 us). What is held for two tiles has a barrier for each (k3_attend4_order.h); every wait is
// bounded (k3_bulk.cuh).
//
// BOUND. A tile of 64 positions x 576 values takes about 3600 cycles: its chain (widening 1500, S
// 2000, softmax 2300, half of O^T 900) goes round two buffers, which with Q fill the shared
// memory. The tensor pipe needs 1920 of them (32 for an MMA of S, 48 for one of O^T, both bound
// by what they read from shared memory), the widening's stores 580. 512 + 64, one call:
//   64 requests, one token, 16 heads, up to 8192 positions    67 us
//   16 requests, four tokens, 64 heads, up to 8192 positions  92 us
//   one request, one token, 64 heads: 1000 positions 16.8 us, 32768 positions 30.5 us
//   one request, 2048 tokens behind 2048 positions, 64 heads  1.8 ms (486 TFLOP/s)
// One request is bound by what surrounds its tiles: Q, the first loads, the result, the merge. The
// constants (units of an item's start, the merge's shares) were measured at 512 + 64 and serve every
// shape: 128 + 64 takes 44, 57, 14.6 and 22.5 us for the first four. 128 registers: 8 bytes are
// spilled at 256 and 512 latents, 24 in the merge of few pieces.
// Measured and left: 18 warps (96 registers, spills), the widening by two groups of four warps
// that take tiles in turn, pieces of 128 or of 512 latents, two raw buffers ahead (registers
// again), Q by all 14 warps in one batch (103 -> 121 us), and Q through a bulk copy into the free
// tile buffer (68 -> 69.5 us: its conversion takes the time, not its way).
#include "k3_attend4_order.h"
#include "k3_bulk.cuh"
#include "k3_cache4.cuh"
#include "k3_ops.cuh"

namespace k3 {
namespace at4 {

using namespace bulk;

constexpr int kT = 64;                    // positions per tile
constexpr int kR = 64;                    // rows per item
constexpr int kHalf = kR / 2;             // rows of which P is held for two tiles in turn
constexpr int kPanel = kT * 128;          // bytes of a panel: 64 rows x 64 fp16
constexpr int kThreads = 448;
constexpr int kMaxUnits = 1 << 30;
constexpr int kStart = 5;                 // units that an item counts beside its tiles
constexpr float kLift = 7.f;              // P = 2^(a - m + 7)
constexpr float kStep = 8.f;              // m moves when a tile passes it by this
constexpr int kUnit = -2;                 // the fp16 operand is in units of 2^kUnit
constexpr int kDown = 14;                 // a row's 2^e is taken into fp16 for kUnit - 14 <= e <= kUnit
constexpr float kUnitF = 0.25f;

// How requests are cut into items: up to `rows` rows of whole tokens, or of the heads of one.
struct Split {
    int rows;
    int per, hc;                          // tokens of an item (H <= rows), chunks of `rows` heads of a token
};

struct Args {
    Pool4 d;
    const void *q;
    void *out;
    const int *table, *row_start, *kv_len;
    int max_pages, B, N, H;
    int q_f32, out_f32;
    Split split[3];                       // 64, 32 and 16 rows
    int splits;                           // how many of them the kernel may choose from
    float inv_h;                          // 1 / H
    float scale;
    float *part;                          // [grid][2][kv / 32][16][32][4]: latent block, row / 4, latent, row % 4
    float2 *ml;                           // [grid][2][64] (max, sum), base 2
    int4 *info;                           // [grid][2]: {u0, item begin, item end, split}, {row0, rows, 0, 0}
};

// Pieces of 256 latents in which a tile is handed over.
template <int NB>
__host__ __device__ constexpr int pieces() { return (NB + 1) / 2; }

struct Smem {                             // offsets from the 1024-byte aligned base
    uint32_t q, k, p, kinfo, row, bars, total;
};

__host__ __device__ inline Smem smem_layout(int kv, int rope)
{
    Smem s;
    const uint32_t panels = kv / 64 + (rope ? 1 : 0);
    s.q = 0;
    s.k = s.q + panels * kPanel;
    s.p = s.k + 2 * panels * kPanel;
    s.kinfo = s.p + kR * 128;             // float [2][64]: residual of each position
    s.row = s.kinfo + 2 * kT * 4;         // int [64] exponents of Q's rows, float [64] factors, int [2][4] flags
    s.bars = s.row + 2 * kR * 4 + 32;
    s.total = s.bars + 208 + 64;          // barriers, then int [2][8]: a warp's rows have no residual
    return s;
}

// One request as the scheduler sees it.
struct Req {
    int first, n, kvl, items, tiles;
};

__device__ __forceinline__ int items_of(const Split &sp, int n)
{
    return sp.hc > 1 ? n * sp.hc : (int)((uint32_t)(n + sp.per - 1) / (uint32_t)sp.per);
}

__device__ __forceinline__ Req request(const Args &a, const Split &sp, int b, int r0, int r1, int kvl)
{
    Req r;
    int n = r1 - r0;
    const int cap = a.max_pages * a.d.page;
    if (r0 < 0 || n < 0 || r1 > a.N || kvl < 0 || kvl > cap) {
        k3_raise_at(K3D_EBOUND, K3_SITE_CACHE4, b, r1, kvl);
        if (r0 < 0 || n < 0 || r1 > a.N) n = 0;
        kvl = max(0, min(kvl, cap));
    }
    r.first = r0;
    r.n = n;
    r.kvl = kvl;
    r.items = items_of(sp, n);
    r.tiles = max(1, (kvl + kT - 1) / kT);
    return r;
}

__device__ __forceinline__ Req request(const Args &a, const Split &sp, int b)
{
    return request(a, sp, b, a.row_start[b], a.row_start[b + 1], a.kv_len[b]);
}

// The piece of an item that a CTA works on, and the rows of it.
struct Seg {
    int b, n, kvl;
    int row0, rows;                       // flattened rows of q
    int j0;                               // new token of the first row
    int t0, t1;                           // tiles [t0, t1), cut to what the item sees
    int begin, end;                       // units of the whole item
    bool whole;
};

struct Cursor {
    int u, u1, b, pre;
    Req r;
    int si;                               // which split
};

__device__ __forceinline__ bool next_seg(const Args &a, Cursor &c, Seg &s)
{
    if (c.u >= c.u1) return false;
    while (c.u >= c.pre + c.r.items * (c.r.tiles + kStart)) {
        c.pre += c.r.items * (c.r.tiles + kStart);
        c.b++;
        c.r = request(a, a.split[c.si], c.b);
    }
    const int item = (int)((uint32_t)(c.u - c.pre) / (uint32_t)(c.r.tiles + kStart));
    s.b = c.b;
    s.n = c.r.n;
    s.kvl = c.r.kvl;
    s.begin = c.pre + item * (c.r.tiles + kStart);
    s.end = s.begin + c.r.tiles + kStart;
    const int first = c.r.first;
    int last;
    const Split &sp = a.split[c.si];
    if (sp.hc == 1) {
        s.j0 = item * sp.per;
        const int tok = min(sp.per, c.r.n - s.j0);
        s.row0 = (first + s.j0) * a.H;
        s.rows = tok * a.H;
        last = s.j0 + tok - 1;
    } else {
        s.j0 = last = (int)((uint32_t)item / (uint32_t)sp.hc);
        const int h0 = (item - s.j0 * sp.hc) * sp.rows;
        s.row0 = (first + s.j0) * a.H + h0;
        s.rows = min(sp.rows, a.H - h0);
    }
    const int stop = min(c.u1, s.end);
    const int seen = max(0, c.r.kvl - c.r.n + last + 1);
    s.t0 = max(0, c.u - s.begin - kStart);
    s.t1 = min(stop - s.begin - kStart, (seen + kT - 1) / kT);
    s.whole = c.u == s.begin && stop == s.end;
    c.u = stop;
    return true;
}

// ------------------------------------------------------------------- tcgen05 wrappers ----
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void named_sync(int id, int n) { asm volatile("bar.sync %0, %1;" :: "r"(id), "r"(n) : "memory"); }

// SWIZZLE_128B descriptors, in two words: the low one has the address (16-byte units) and the
// lead stride, the high one is a constant (groups of 8 rows, or of 8 k, 1024 B apart). K-major:
// the lead is not used. MN-major: 64-element blocks lie `lead` bytes apart.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);

__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | (1u << 16); }

__device__ __forceinline__ uint32_t desc_mn(uint32_t addr, uint32_t lead)
{
    return ((addr >> 4) & 0x3FFFu) | ((lead >> 4) << 16);
}

// kind::f16, fp32 D, fp16 A and B
__device__ __forceinline__ uint32_t idesc(int M, int N, int a_mn)
{
    return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// The whole warp runs the issue loop and one lane's predicate is on the instruction. Only the
// descriptors' low words change between MMAs: with 64-bit arithmetic on whole descriptors every
// MMA took nine moves to uniform registers, and unrolled loops more instruction fetches than
// MMAs' time.
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accum, uint32_t lead)
{
    asm volatile("{\n\t.reg .pred p, l;\n\t.reg .b64 da, db;\n\t"
                 "mov.b64 da, {%1, %6};\n\t"
                 "mov.b64 db, {%2, %6};\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 l, %5, 0;\n\t"
                 "@l tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "r"(b), "r"(id), "r"(accum), "r"(lead), "n"(kDescHi) : "memory");
}

__device__ __forceinline__ void commit(uint32_t bar, uint32_t lead)
{
    asm volatile("{\n\t.reg .pred l;\n\t"
                 "setp.ne.b32 l, %1, 0;\n\t"
                 "@l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                 :: "r"(bar), "r"(lead) : "memory");
}

__device__ __forceinline__ uint32_t elect()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}

// A whole warp's bounded wait: the lanes leave together, with the same answer.
__device__ __forceinline__ bool wait_all(uint32_t b, uint32_t parity, volatile int *abort, int site, int who, int where)
{
    // the limit and the other roles' give-up are looked at every 32 tries only
    bool ok = mbar_try(b, parity);
    if (!__all_sync(0xffffffffu, ok)) {
        for (int i = 0; i < 32 && !ok; i++) ok = mbar_try(b, parity);
        if (!ok) ok = mbar_wait(b, parity, abort, site, who, where);
    }
    return __all_sync(0xffffffffu, ok);
}

#define K3_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), \
                    "=r"(r[i + 6]), "=r"(r[i + 7])

// 16 lanes x 64 columns: element 4 i + 2 h + e is row lane / 4 + 8 h, column 8 i + 2 (lane % 4) + e
__device__ __forceinline__ void ld_s(uint32_t taddr, float v[32])
{
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
                 "%26,%27,%28,%29,%30,%31}, [%32];"
                 : K3_R8(r, 0), K3_R8(r, 8), K3_R8(r, 16), K3_R8(r, 24) : "r"(taddr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void ld16(uint32_t taddr, float v[16])
{
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : K3_R8(r, 0), K3_R8(r, 8) : "r"(taddr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void st16(uint32_t taddr, const float v[16])
{
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 16; i++) r[i] = __float_as_uint(v[i]);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
                    "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
                    "r"(r[15]) : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ float ex2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// the larger of a >= 0 and |b|, of two bf16 values each (a NaN gives way)
__device__ __forceinline__ uint32_t absmax_bf16x2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("{\n\t.reg .b32 t;\n\tabs.bf16x2 t, %2;\n\tmax.bf16x2 %0, %1, t;\n\t}" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// two values rounded to bf16, x in the low half
__device__ __forceinline__ uint32_t bf16x2(float x, float y)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}

__device__ __forceinline__ void sts16(uint32_t addr, uint4 v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// 2^x of a whole x in [-126, 127] kept as a float: x + 127 lands in the low mantissa bits
__device__ __forceinline__ float unit(float e)
{
    return __uint_as_float(__float_as_uint(e + 12583039.0f) << 23);
}

// Byte `at` of row `row` in a panel of 128-byte rows, 16-byte units swizzled by the row.
__device__ __forceinline__ uint32_t swz(int row, int unit) { return (uint32_t)(row * 128 + ((unit ^ (row & 7)) << 4)); }

__device__ __forceinline__ uint2 ld_v2(const void *p)
{
    uint2 r;
    asm volatile("ld.global.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p) : "memory");
    return r;
}

// 16 bytes that no other thread reads, past L1 (a plain load: earlier work of the stream may
// still have been writing the pool when this kernel was launched)
__device__ __forceinline__ uint4 ld_v4(const void *p)
{
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
    return r;
}

// ------------------------------------------------------------------------ the widening ----
// Thread (position, part) of a tile, four parts to a position: of every 128 latents the 16
// from 16 part and the 16 from 64 + 16 part on (8 bytes of codes and a scale each), and up to
// two 16-byte units of the rope key. The eight lanes of a store phase (two positions x four
// parts) then hit eight different 16-byte banks.
template <int NB>
struct Raw {
    uint2 lo[NB], hi[NB], scale[NB];      // scale: the E4M3 bytes of the 128 latents
    uint4 rope[2];
    int e;                                // exponent byte, or -1: not there
};

// A thread's place in the page table, a tile at a time: the entry of the next tile is on its
// way while this one's rows are loaded, and is checked only when it is used.
struct Place {
    int pos, page, in;                    // position, its page of the request, its row there
    int entry;                            // the table's entry, -1 past the length
};

__device__ __forceinline__ void look_up(Place &p, const int *table, int kvl)
{
    p.entry = p.pos < kvl ? table[p.page] : -1;
}

__device__ __forceinline__ void advance(Place &p, int page)
{
    p.pos += kT;
    p.in += kT;
    while (p.in >= page) { p.in -= page; p.page++; }
}

// What is not there gets scales of 0: its latents become zeros whatever the codes are, and
// its scores are not looked at.
template <int NB>
__device__ __forceinline__ void load_raw(Raw<NB> &r, const Args &a, const Place &p, int kvl, int part)
{
    r.e = -1;
#pragma unroll
    for (int i = 0; i < NB; i++) r.scale[i] = make_uint2(0u, 0u);
    if (p.pos >= kvl) return;
    if (p.entry < 0 || p.entry >= a.d.n_pages) {          // no page of the pool: not there
        k3_raise_at(K3D_EBOUND, K3_SITE_CACHE4, p.page, p.entry, p.pos);
        return;
    }
    const uint8_t *base = a.d.p + (size_t)p.entry * a.d.page_bytes;
    const uint8_t *c = base + p.in * (NB * 64) + part * 8;
    const uint8_t *s = base + a.d.o_scale + p.in * (NB * 8);
#pragma unroll
    for (int i = 0; i < NB; i++) {
        r.lo[i] = ld_v2(c + i * 64);
        r.hi[i] = ld_v2(c + i * 64 + 32);
        r.scale[i] = ld_v2(s + i * 8);
    }
    const uint8_t *rp = base + a.d.o_rope + p.in * 2 * a.d.rope;
    if (part < a.d.rope / 8) r.rope[0] = ld_v4(rp + part * 16);
    if (part + 4 < a.d.rope / 8) r.rope[1] = ld_v4(rp + (part + 4) * 16);
    r.e = base[a.d.o_exp + p.in];
}

__device__ __forceinline__ uint32_t unit_step(int e)
{
    // 2^(e - kUnit), from 2^-14 to 1, as f16x2
    return (uint32_t)(min(max(e - 127 - kUnit, -kDown), 0) + 15) * 0x04000400u;
}

// This thread's 32 of 128 latents: two 16-byte units of each of two panels. at0 and at1: the
// units' places in a panel.
__device__ __forceinline__ void widen(uint2 lo, uint2 hi, uint2 scale, uint32_t up, uint32_t panels2, uint32_t at0,
                                      uint32_t at1, uint32_t sel)
{
    uint32_t s2;                          // the two scales as f16x2
    asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
        : "=r"(s2) : "r"(__byte_perm(scale.x, scale.y, sel)));
    s2 = hmul2(s2, up);
    const uint32_t f[2] = {__byte_perm(s2, s2, 0x1010), __byte_perm(s2, s2, 0x3232)};
    const uint32_t w[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t h[4];
        e2m1x8_to_f16x8(w[j], h);
        const uint32_t k = f[j >> 1];
        sts16(panels2 + (uint32_t)(j >> 1) * kPanel + ((j & 1) ? at1 : at0),
              make_uint4(hmul2(h[0], k), hmul2(h[1], k), hmul2(h[2], k), hmul2(h[3], k)));
    }
}

// ------------------------------------------------------------------------------- Q ----
// Rows warp, warp + 12, ... of the item: fp16 in units of 2^(e - 14), e the row's exponent (its
// largest value in [2^13, 2^14)), which the softmax takes into its factor. Rows behind the last
// up to a multiple of 16 are zeros that see everything: they cost no case of their own. What lies
// behind them reaches rows of S only that nobody reads.
template <bool F32>
__device__ __forceinline__ void load_q_rows(const Args &a, const Seg &s, uint32_t sq, int *rexp, int warp, int lane)
{
    constexpr int RB = F32 ? 1 : 3;                       // rows in flight (36 registers or 24)
    const int W = a.d.kv + a.d.rope, chunks = W / 8, nr = (s.rows + 15) & ~15;
    for (int r0 = warp; r0 < nr; r0 += 12 * RB) {
        uint4 raw[RB][3][F32 ? 2 : 1];
#pragma unroll
        for (int i = 0; i < RB; i++) {
            const int r = r0 + 12 * i;
            const size_t at = (size_t)(s.row0 + r) * W;
#pragma unroll
            for (int c = 0; c < 3; c++) {
                const int ch = lane + 32 * c;
                const uint4 *p = reinterpret_cast<const uint4 *>((const char *)a.q + (at + ch * 8) * (F32 ? 4 : 2));
#pragma unroll
                for (int k = 0; k < (F32 ? 2 : 1); k++)
                    raw[i][c][k] = ch < chunks && r < s.rows ? p[k] : make_uint4(0u, 0u, 0u, 0u);
            }
        }
#pragma unroll
        for (int i = 0; i < RB; i++) {
            const int r = r0 + 12 * i;
            if (r >= nr) break;
            auto value = [&](int c, float v[8]) {
                const uint4 x = raw[i][c][0], y = raw[i][c][F32 ? 1 : 0];
                const uint32_t u[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                if (F32) {
#pragma unroll
                    for (int k = 0; k < 8; k++) v[k] = __uint_as_float(u[k]);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        v[2 * k] = __uint_as_float(u[k] << 16);
                        v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
                    }
                }
            };
            float m = 0.f;
            if (F32) {
#pragma unroll
                for (int c = 0; c < 3; c++) {
                    float v[8];
                    value(c, v);
#pragma unroll
                    for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(v[k]));
                }
            } else {
                uint32_t t = 0u;                          // two at a time
#pragma unroll
                for (int c = 0; c < 3; c++) {
                    const uint4 x = raw[i][c][0];
                    t = absmax_bf16x2(absmax_bf16x2(absmax_bf16x2(absmax_bf16x2(t, x.x), x.y), x.z), x.w);
                }
                m = fmaxf(__uint_as_float(t << 16), __uint_as_float(t & 0xffff0000u));
            }
            m = warp_max(m);
            // m < 2^e. A row with an infinity is NaN throughout, as one with a NaN makes its scores: scores
            // of minus infinity alone would read as positions that are not seen
            const bool finite = m <= 3.4028234e38f;
            const int e = finite ? max((int)(__float_as_uint(m) >> 23) - 126, -110) : 0;
            // the sign of the scale goes into q, so that a larger product is a larger score
            const float up = finite ? copysignf(__uint_as_float((uint32_t)(127 + 14 - e) << 23), a.scale)
                                    : __int_as_float(0x7fc00000);
#pragma unroll
            for (int c = 0; c < 3; c++) {
                const int ch = lane + 32 * c;
                if (ch < chunks) {
                    float v[8];
                    value(c, v);
                    uint32_t h[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const __half2 t = __floats2half2_rn(v[2 * k] * up, v[2 * k + 1] * up);
                        h[k] = *reinterpret_cast<const uint32_t *>(&t);
                    }
                    sts16(sq + (uint32_t)(ch >> 3) * kPanel + swz(r, ch & 7), make_uint4(h[0], h[1], h[2], h[3]));
                }
            }
            if (lane == 0) rexp[r] = e;
        }
    }
}

__device__ __forceinline__ void load_q(const Args &a, const Seg &s, uint32_t sq, int *rexp, int warp, int lane)
{
    if (a.q_f32) load_q_rows<true>(a, s, sq, rexp, warp, lane);
    else load_q_rows<false>(a, s, sq, rexp, warp, lane);
}

// |scale| log2(e) 2^(e - 14 + kUnit), the power in two factors (it may be below -126)
__device__ __forceinline__ float score_factor(const Args &a, int e)
{
    const int k = e - 14 + kUnit, k1 = k >> 1;
    return fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(k1 + 127) << 23) *
           __uint_as_float((uint32_t)(k - k1 + 127) << 23);
}

// the positions that row r of the item sees
__device__ __forceinline__ int sees(const Args &a, const Seg &s, bool tokens, int r)
{
    const int j = s.j0 + (tokens ? (int)(((float)r + 0.5f) * a.inv_h) : 0);
    return r < s.rows ? max(0, s.kvl - s.n + j + 1) : 0x7fffffff;
}

// This warp's third of an item's result: the 16-row groups sub, sub + 3, ... of its quarter of
// the lanes (latents). A whole item: neighbouring lanes trade halves, so that each writes a
// pair of latents of eight rows. A piece: as it lies, four rows to a 16-byte store.
template <int NB>
__device__ __forceinline__ void write_out(const Args &a, const Seg &s, size_t slot, uint32_t t_o, int NR, bool any,
                                          const float *rowf, int warp, int lane)
{
    const int q = warp & 3, sub = warp >> 2, ng = NR / 16;
    const uint32_t lanes = (uint32_t)(32 * q) << 16;
    constexpr int kv = NB * 128;
    for (int i = sub; i < NB * ng; i += 3) {
        const int blk = i / ng, c0 = (i - blk * ng) * 16;
        float o[16];
        if (any) {
            ld16(t_o + lanes + (uint32_t)(blk * kR + c0), o);
        } else {
#pragma unroll
            for (int k = 0; k < 16; k++) o[k] = 0.f;
        }
        if (s.whole) {
            const int col = blk * 128 + 32 * q + (lane & ~1), up = (lane & 1) * 8;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float give = (lane & 1) ? o[k] : o[k + 8];
                const float got = __shfl_xor_sync(0xffffffffu, give, 1);
                const int r = c0 + k + up;
                if (r < s.rows) {
                    const float f = rowf[r];
                    const float x = ((lane & 1) ? got : o[k]) * f, y = ((lane & 1) ? o[k + 8] : got) * f;
                    const size_t at = (size_t)(s.row0 + r) * kv + col;
                    if (a.out_f32) {
                        *reinterpret_cast<float2 *>((float *)a.out + at) = make_float2(x, y);
                    } else {
                        *reinterpret_cast<uint32_t *>((uint16_t *)a.out + at) = bf16x2(x, y);
                    }
                }
            }
        } else {
            float4 *dst = reinterpret_cast<float4 *>(a.part) + ((slot * (NB * 4) + blk * 4 + q) * 16 + c0 / 4) * 32 + lane;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (c0 + 4 * k < s.rows) dst[k * 32] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        }
    }
}

// Tensor memory columns: the CTA holds all 512, so they begin at 0. S of the two buffers, then
// O^T, 64 columns for every 128 latents.
constexpr uint32_t kColO = 2 * kT;

// S of tile k (the k-th of this CTA) into its buffer's columns.
template <int NB>
__device__ __forceinline__ bool issue_s(int rope, uint32_t sq, uint32_t sk, uint32_t b_kfull, uint32_t b_sfull,
                                        uint32_t b_sfree, volatile int *abort, int k, uint32_t lead)
{
    const int buf = at4_buf(k);
    if (k >= 2 && !wait_all(b_sfree + 8 * buf, at4_phase(k - 2), abort, K3_SITE_CACHE4, 13, k)) return false;
    uint32_t da = desc_k(sq), db = desc_k(sk + (uint32_t)buf * (NB * 2 + (rope ? 1 : 0)) * kPanel);
    const uint32_t id = idesc(64, kT, 0), d = (uint32_t)(buf * kT);
#pragma unroll 1
    for (int i = 0; i < NB; i++) {
        if (!(i & 1) && !wait_all(b_kfull + 8 * (buf * 2 + (i >> 1)), at4_phase(k), abort, K3_SITE_CACHE4, 4, k)) return false;
        tc_after();
#pragma unroll
        for (int p = 0; p < 2; p++) {
#pragma unroll
            for (int k4 = 0; k4 < 4; k4++) mma(d, da + 2 * k4, db + 2 * k4, id, p | k4 ? 1u : (i ? 1u : 0u), lead);
            da += kPanel / 16;
            db += kPanel / 16;
        }
    }
#pragma unroll
    for (int k4 = 0; k4 < 4; k4++)
        if (k4 < rope / 16) mma(d, da + 2 * k4, db + 2 * k4, id, 1u, lead);
    commit(b_sfull + 8 * buf, lead);
    return true;
}

// O^T += V^T P^T of tile k; every 256 latents that have been used are given back.
template <int NB>
__device__ __forceinline__ void issue_o(int rope, uint32_t sk, uint32_t sp, uint32_t b_pv, uint32_t id, int k, uint32_t accum,
                                        uint32_t lead)
{
    const int buf = at4_buf(k);
    uint32_t da = desc_mn(sk + (uint32_t)buf * (NB * 2 + (rope ? 1 : 0)) * kPanel, kPanel), d = kColO, bar = b_pv + 16 * buf;
    const uint32_t db = desc_k(sp);
#pragma unroll 1
    for (int blk = 0; blk < NB; blk++) {
#pragma unroll
        for (int k4 = 0; k4 < kT / 16; k4++) mma(d, da + 128 * k4, db + 2 * k4, id, k4 ? 1u : accum, lead);
        if ((blk & 1) || blk == NB - 1) {
            commit(bar, lead);
            bar += 8;
        }
        da += 2 * kPanel / 16;
        d += kR;
    }
}

// SPLIT: the kernel chooses how many rows an item has (else 64; with the choice in one kernel the
// large batches took 1 us more).
template <int NB, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) k_attend4(const __grid_constant__ Args a)
{
    extern __shared__ unsigned char smem_raw[];
    __shared__ long long red[kThreads / 32];
    __shared__ int s_cur[10];
    const uint32_t raw = saddr(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char *gb = smem_raw + (base - raw);
    const Smem L = smem_layout(NB * 128, a.d.rope);
    const uint32_t panels = NB * 2 + (a.d.rope ? 1 : 0);
    float *kinfo = reinterpret_cast<float *>(gb + L.kinfo);
    int *rexp = reinterpret_cast<int *>(gb + L.row);                    // exponents of Q's rows
    float *rowf = reinterpret_cast<float *>(gb + L.row + kR * 4);       // rescale factors, then 1 / sum
    int *flags = reinterpret_cast<int *>(gb + L.row + 2 * kR * 4);      // [2][4]
    const uint32_t b_qfull = base + L.bars, b_qempty = b_qfull + 8;
    // of each tile buffer and 256 latents: widened (kfull), and O^T added (pv, the last of a tile
    // standing for the tile); S, P and "S is read" (sfree) of each buffer
    const uint32_t b_kfull = b_qfull + 16, b_pv = b_kfull + 64, b_sfull = b_pv + 64, b_pfull = b_sfull + 16;
    const uint32_t b_drain = b_pfull + 16, b_sfree = b_drain + 8;
    volatile int *abort = reinterpret_cast<volatile int *>(gb + L.bars + 200);
    uint32_t *tslot = reinterpret_cast<uint32_t *>(gb + L.bars + 204);
    int *kplain = reinterpret_cast<int *>(gb + L.bars + 208);           // [2][8]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        mbar_init(b_qfull, 12);
        mbar_init(b_qempty, 1);
        for (int i = 0; i < 8; i++) {
            mbar_init(b_kfull + 8 * i, 8);
            mbar_init(b_pv + 8 * i, 1);
        }
        mbar_init(b_sfull, 1);
        mbar_init(b_sfull + 8, 1);
        mbar_init(b_pfull, 4);
        mbar_init(b_pfull + 8, 4);
        mbar_init(b_drain, 2);
        mbar_init(b_sfree, 4);
        mbar_init(b_sfree + 8, 4);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(saddr(tslot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before();
    }
    __syncthreads();
    tc_after();
    const uint32_t tmem = *tslot;
    pdl_wait();
    pdl_trigger();

    // ---- this CTA's units: the requests' totals, then the request that holds the first unit. Up
    // to 64 requests every warp does it for itself, two requests to a lane; more are dealt out over
    // the block, which meets three times (1 us more with one request, of a call's 20).
    Cursor cur;
    cur.b = 0; cur.pre = 0;
    const Req none = {0, 0, 0, 0, 1};
    cur.r = none;
    cur.si = 0;
    const int c = blockIdx.x;
    const bool few = a.B <= 64;
    const int per = few ? 2 : (a.B + kThreads - 1) / kThreads, me = few ? lane : tid;
    const int rb0 = min(a.B, me * per), rb1 = min(a.B, rb0 + per);
    long long mine = 0;
    Req lo = none, hi = none;
    if (few) {
        if (rb0 < rb1) {
            const int2 k = make_int2(a.kv_len[rb0], a.kv_len[rb1 - 1]);
            const int x = a.row_start[rb0], y = a.row_start[rb0 + 1], z = a.row_start[rb1];
            lo = request(a, a.split[0], rb0, x, y, k.x);
            if (rb1 - rb0 > 1) hi = request(a, a.split[0], rb0 + 1, y, z, k.y);
        }
        // fewer rows make no fewer tiles
        const bool idle = SPLIT && __reduce_add_sync(0xffffffffu, lo.items * lo.tiles + hi.items * hi.tiles) <= (int)gridDim.x;
        for (int i = idle ? a.splits - 1 : 0; i > 0; i--) {
            const Split sp = a.split[i];
            const int x = items_of(sp, lo.n), y = items_of(sp, hi.n);
            if (__reduce_add_sync(0xffffffffu, x * lo.tiles + y * hi.tiles) <= (int)gridDim.x) {
                cur.si = i;
                lo.items = x;
                hi.items = y;
                break;
            }
        }
        mine = (long long)lo.items * (lo.tiles + kStart) + (long long)hi.items * (hi.tiles + kStart);
    } else {
        for (int b = rb0; b < rb1; b++) {
            const Req r = request(a, a.split[0], b);
            mine += (long long)r.items * (r.tiles + kStart);
        }
    }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
    }
    long long lead = incl - mine, total = __shfl_sync(0xffffffffu, incl, 31);
    if (!few) {
        if (lane == 31) red[warp] = incl;
        __syncthreads();
        total = 0;
        for (int i = 0; i < kThreads / 32; i++) {
            if (i < warp) lead += red[i];
            total += red[i];
        }
    }
    if (total > kMaxUnits) {                              // unit numbers are 31-bit
        if (tid == 0) k3_raise_at(K3D_EBOUND, K3_SITE_CACHE4, a.N, a.H, 4);
        total = 0;
    }
    const int U = (int)total, before = (int)min(lead, (long long)kMaxUnits);
    const int G = min((int)gridDim.x, U);
    // the first U % G CTAs take one unit more than the others
    const int each = G > 0 ? (int)((uint32_t)U / (uint32_t)G) : 0, more = U - each * G;
    const int cut0 = c < G ? c * each + min(c, more) : 0, cut1 = c < G ? cut0 + each + (c < more ? 1 : 0) : 0;
    cur.u = cut0;
    cur.u1 = cut1;
    // a cut in the request of `r` whose units begin at `pre`, moved out of an item's start
    auto moved_cut = [&](int cut, int pre, int tiles) {
        const int len = tiles + kStart, begin = pre + (int)((uint32_t)(cut - pre) / (uint32_t)len) * len;
        return cut - begin <= kStart ? begin : cut;
    };
    if (few) {
        if (cut0 < cut1) {
            auto holds = [&](int cut, int &b, int &pre, Req &r) {
                const unsigned m = __ballot_sync(0xffffffffu, incl > cut);
                const int l = m ? __ffs(m) - 1 : 0, units = lo.items * (lo.tiles + kStart);
                const bool second = cut >= before + units;
                const Req &mine = second ? hi : lo;
                b = 2 * l + __shfl_sync(0xffffffffu, second ? 1 : 0, l);
                pre = __shfl_sync(0xffffffffu, before + (second ? units : 0), l);
                r.first = __shfl_sync(0xffffffffu, mine.first, l);
                r.n = __shfl_sync(0xffffffffu, mine.n, l);
                r.kvl = __shfl_sync(0xffffffffu, mine.kvl, l);
                r.items = __shfl_sync(0xffffffffu, mine.items, l);
                r.tiles = __shfl_sync(0xffffffffu, mine.tiles, l);
                return m != 0;
            };
            int b1, pre1;
            Req r1;
            holds(cut0, cur.b, cur.pre, cur.r);
            cur.u = moved_cut(cut0, cur.pre, cur.r.tiles);
            if (holds(cut1, b1, pre1, r1)) cur.u1 = moved_cut(cut1, pre1, r1.tiles);
        }
    } else {
        if (tid == 0) s_cur[7] = cut0, s_cur[8] = cut1;
        __syncthreads();
        // the thread whose requests hold a cut: the request, and where the cut moves
        for (int k = 0; k < 2; k++) {
            const int cut = k ? cut1 : cut0;
            if (cut0 < cut1 && cut >= before && cut < before + mine) {
                int pre = before;
                for (int b = rb0; b < rb1; b++) {
                    const Req r = request(a, a.split[0], b);
                    const int len = r.tiles + kStart;
                    if (cut < pre + r.items * len) {
                        s_cur[7 + k] = moved_cut(cut, pre, r.tiles);
                        if (k == 0) {
                            s_cur[0] = b; s_cur[1] = pre; s_cur[2] = r.first; s_cur[3] = r.n;
                            s_cur[4] = r.kvl; s_cur[5] = r.items; s_cur[6] = r.tiles;
                        }
                        break;
                    }
                    pre += r.items * len;
                }
            }
        }
        __syncthreads();
        cur.u = s_cur[7];
        cur.u1 = s_cur[8];
        if (cut0 < cut1) {
            cur.b = s_cur[0];
            cur.pre = s_cur[1];
            cur.r.first = s_cur[2]; cur.r.n = s_cur[3]; cur.r.kvl = s_cur[4];
            cur.r.items = s_cur[5]; cur.r.tiles = s_cur[6];
        }
    }
    const int u0 = cur.u;
    if (tid == 12 * 32) {
        // an empty range (its cuts moved together) keeps its place in the order
        int4 i0 = make_int4(c < G ? u0 : 0x7fffffff, -1, -1, cur.si), i1 = make_int4(0, 0, 0, 0);
        Cursor t = cur;
        Seg s;
        if (next_seg(a, t, s)) {
            i0.y = s.begin;
            i0.z = s.end;
            i1 = make_int4(s.row0, s.rows, 0, 0);
        }
        a.info[2 * c] = i0;
        a.info[2 * c + 1] = i1;
    }
    const uint32_t sq = base + L.q, sk = base + L.k, sp = base + L.p;
    constexpr uint32_t t_o = kColO;
    Seg s;
    int item = 0, g = 0;                                  // items and tiles so far (barrier phases)

    if (warp < 8) {
        // ------------------------------------------------------------------- widening
        const int row = tid >> 2, part = tid & 3;
        const uint32_t at0 = swz(row, 2 * part), at1 = swz(row, 2 * part + 1);
        const uint32_t rope0 = swz(row, part), rope1 = swz(row, part + 4);
        const uint32_t sel = (uint32_t)(part | ((4 + part) << 4));
        bool dead = false;
        while (next_seg(a, cur, s)) {
            const bool slot1 = item > 0;                  // a later piece of this CTA
            const bool any = s.t0 < s.t1;
            Raw<NB> nx;
            Place at;
            const int *table = a.table + (size_t)s.b * a.max_pages;
            at.pos = s.t0 * kT + row;
            at.page = (int)((uint32_t)at.pos / (uint32_t)a.d.page);
            at.in = at.pos - at.page * a.d.page;
            if (any) {
                look_up(at, table, s.kvl);
                load_raw<NB>(nx, a, at, s.kvl, part);
                advance(at, a.d.page);
                look_up(at, table, s.kvl);
            }
            if (item > 0 && !dead && !wait_all(b_qempty, (item - 1) & 1, abort, K3_SITE_CACHE4, 1, item)) dead = true;
            if (!dead) load_q(a, s, sq, rexp, warp, lane);
            async_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_qfull);
            item++;
            for (int t = s.t0; t < s.t1 && !dead; t++, g++) {
                const Raw<NB> r = nx;
                if (t + 1 < s.t1) {
                    load_raw<NB>(nx, a, at, s.kvl, part);
                    advance(at, a.d.page);
                    look_up(at, table, s.kvl);
                }
                const int buf = at4_buf(g);
                const uint32_t tile = sk + (uint32_t)buf * panels * kPanel, up = unit_step(r.e);
                // the residual; NaN for a row of NaN, minus infinity where there is none
                const int e = r.e - 127;
                const float res = r.e < 0 ? __int_as_float(0xff800000)
                                : r.e == 255 ? __int_as_float(0x7fc00000) : (float)(e - min(max(e, kUnit - kDown), kUnit));
                const int plain = __all_sync(0xffffffffu, res == 0.f);
                // as soon as O(g - 2) has used 256 latents of the buffer, this tile's take their place
#pragma unroll
                for (int h = 0; h < pieces<NB>(); h++) {
                    if (g >= 2 && !wait_all(b_pv + 8 * (buf * 2 + h), at4_phase(g - 2), abort, K3_SITE_CACHE4, 2, g)) { dead = true; break; }
#pragma unroll
                    for (int i = 2 * h; i < 2 * h + 2 && i < NB; i++)
                        widen(r.lo[i], r.hi[i], r.scale[i], up, tile + 2 * i * kPanel, at0, at1, sel);
                    if (h == pieces<NB>() - 1) {
                        const uint32_t pan = tile + 2 * NB * kPanel;
                        if (part < a.d.rope / 8)
                            sts16(pan + rope0, make_uint4(hmul2(r.rope[0].x, up), hmul2(r.rope[0].y, up), hmul2(r.rope[0].z, up), hmul2(r.rope[0].w, up)));
                        if (part + 4 < a.d.rope / 8)
                            sts16(pan + rope1, make_uint4(hmul2(r.rope[1].x, up), hmul2(r.rope[1].y, up), hmul2(r.rope[1].z, up), hmul2(r.rope[1].w, up)));
                        if (part == 0) kinfo[buf * kT + row] = res;
                        if (lane == 0) kplain[buf * 8 + warp] = plain;
                    }
                    async_fence();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(b_kfull + 8 * (buf * 2 + h));
                }
            }
            named_sync(2, 384);                           // the item's sums are written, O^T is complete
            tc_after();
            if (!dead)
                write_out<NB>(a, s, (size_t)c * 2 + (slot1 ? 1 : 0), t_o, (s.rows + 15) & ~15, any, rowf, warp, lane);
            tc_before();
        }
    } else if (warp >= 12) {
        // ----------------------------------------------- MMA issue: S (warp 12), O^T (warp 13)
        const uint32_t lead = elect();
        for (;;) {
            const bool have = next_seg(a, cur, s);
            if (!__any_sync(0xffffffffu, have)) break;
            const int nt = __reduce_max_sync(0xffffffffu, max(0, s.t1 - s.t0));
            bool stop = false;
            if (warp == 12) {
                if (!wait_all(b_qfull, item & 1, abort, K3_SITE_CACHE4, 3, item)) break;
                tc_after();
                item++;
                for (int i = 0; i < nt; i++) {
                    stop = !issue_s<NB>(a.d.rope, sq, sk, b_kfull, b_sfull, b_sfree, abort, g + i, lead);
                    if (stop) break;
                }
                if (stop) break;
                commit(b_qempty, lead);
            } else {
                const bool two = __any_sync(0xffffffffu, s.rows <= kHalf);
                const uint32_t id_o = idesc(128, __reduce_max_sync(0xffffffffu, (s.rows + 15) & ~15), 1);
                for (int i = 0; i < nt; i++) {
                    stop = !wait_all(b_pfull + 8 * at4_buf(g + i), at4_phase(g + i), abort, K3_SITE_CACHE4, 5, g + i);
                    if (stop) break;
                    tc_after();
                    issue_o<NB>(a.d.rope, sk, sp + (two ? (uint32_t)at4_buf(g + i) * (kHalf * 128) : 0u), b_pv, id_o, g + i, i ? 1u : 0u, lead);
                }
                if (stop) break;
            }
            g += nt;
        }
        __syncwarp();
        // every MMA of this warp has completed once this barrier flips
        if (elect()) commit(b_drain, 1u);
        __syncwarp();
    } else {
        // --------------------------------------------------- softmax, rescale, results
        const int w = warp - 8, gr = lane >> 2, t4 = lane & 3;
        const int ra = 16 * w + gr, rb = ra + 8;          // this thread's rows
        const float NEG = __int_as_float(0xff800000);
        const uint32_t lanes = (uint32_t)(32 * w) << 16;
        bool dead = false;
        while (next_seg(a, cur, s)) {
            const bool slot1 = item > 0;
            if (item > 0 && !dead && !wait_all(b_qempty, (item - 1) & 1, abort, K3_SITE_CACHE4, 6, item)) dead = true;
            if (!dead) load_q(a, s, sq, rexp, warp, lane);
            async_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_qfull);
            if (!dead && !wait_all(b_qfull, item & 1, abort, K3_SITE_CACHE4, 7, item)) dead = true;
            item++;
            const int NR = (s.rows + 15) & ~15;
            const bool busy = 16 * w < s.rows;            // a warp without rows only keeps in step
            const bool two = s.rows <= kHalf;             // P has room for two tiles
            const float fa = score_factor(a, rexp[ra]), fb = score_factor(a, rexp[rb]);
            const bool tokens = a.split[cur.si].hc == 1;
            const int la = sees(a, s, tokens, ra), lb = sees(a, s, tokens, rb);
            const int low = __reduce_min_sync(0xffffffffu, min(la, lb));   // what every row of the warp sees
            float ma = NEG, mb = NEG, suma = 0.f, sumb = 0.f;
            for (int t = s.t0; t < s.t1; t++, g++) {
                const int buf = at4_buf(g);
                float ca = 1.f, cb = 1.f;
                uint32_t pa[8], pb[8];
                if (busy) {
                    if (!dead && !(wait_all(b_kfull + 8 * (buf * 2 + pieces<NB>() - 1), at4_phase(g), abort, K3_SITE_CACHE4, 8, g) &&
                                   wait_all(b_sfull + 8 * buf, at4_phase(g), abort, K3_SITE_CACHE4, 9, g)))
                        dead = true;
                    tc_after();
                    float v[32];
                    ld_s(lanes + (uint32_t)(buf * kT), v);
                    tc_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(b_sfree + 8 * buf);
                    const int4 k0 = *reinterpret_cast<const int4 *>(kplain + buf * 8);
                    const int4 k1 = *reinterpret_cast<const int4 *>(kplain + buf * 8 + 4);
                    const bool plain = (k0.x & k0.y & k0.z & k0.w & k1.x & k1.y & k1.z & k1.w) && t * kT + kT <= low;
                    // moves the references to a tile's maxima; a row's accumulator changes only if
                    // it held something
                    auto move = [&](float xa, float xb) {
                        xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, 1));
                        xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, 1));
                        xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, 2));
                        xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, 2));
                        if (ma == NEG) ma = xa;
                        else if (xa > ma + kStep) { ca = ex2(ma - xa); suma *= ca; ma = xa; }
                        if (mb == NEG) mb = xb;
                        else if (xb > mb + kStep) { cb = ex2(mb - xb); sumb *= cb; mb = xb; }
                    };
                    if (plain) {
                        // every row sees the whole tile, no residuals: the product's maximum is the
                        // score's, and the sum adds what P is rounded from
                        float xa = fmaxf(v[0], v[1]), xb = fmaxf(v[2], v[3]);
#pragma unroll
                        for (int i = 1; i < 8; i++) {
                            xa = fmaxf(xa, fmaxf(v[4 * i], v[4 * i + 1]));
                            xb = fmaxf(xb, fmaxf(v[4 * i + 2], v[4 * i + 3]));
                        }
                        move(xa * fa, xb * fb);
                        const float na = kLift - (ma == NEG ? 0.f : ma), nb = kLift - (mb == NEG ? 0.f : mb);
                        float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float p0 = ex2(fmaf(v[4 * i], fa, na)), p1 = ex2(fmaf(v[4 * i + 1], fa, na));
                            const float p2 = ex2(fmaf(v[4 * i + 2], fb, nb)), p3 = ex2(fmaf(v[4 * i + 3], fb, nb));
                            s0 += p0; s1 += p1; s2 += p2; s3 += p3;
                            const __half2 h0 = __floats2half2_rn(p0, p1), h1 = __floats2half2_rn(p2, p3);
                            pa[i] = *reinterpret_cast<const uint32_t *>(&h0);
                            pb[i] = *reinterpret_cast<const uint32_t *>(&h1);
                        }
                        suma += s0 + s1;
                        sumb += s2 + s3;
                    } else {
                        const float2 *ki = reinterpret_cast<const float2 *>(kinfo + buf * kT);
                        float xa = NEG, xb = NEG;
                        float kr[16];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float2 k = ki[4 * i + t4];  // residuals of two neighbouring positions
                            const float u0 = unit(k.x), u1 = unit(k.y);
                            const int pos = t * kT + 8 * i + 2 * t4;
                            kr[2 * i] = k.x;
                            kr[2 * i + 1] = k.y;
                            const bool h0 = k.x != NEG, h1 = k.y != NEG;
                            v[4 * i] = h0 && pos < la ? v[4 * i] * fa * u0 : NEG;
                            v[4 * i + 1] = h1 && pos + 1 < la ? v[4 * i + 1] * fa * u1 : NEG;
                            v[4 * i + 2] = h0 && pos < lb ? v[4 * i + 2] * fb * u0 : NEG;
                            v[4 * i + 3] = h1 && pos + 1 < lb ? v[4 * i + 3] * fb * u1 : NEG;
                            xa = fmaxf(xa, fmaxf(v[4 * i] + k.x, v[4 * i + 1] + k.y));
                            xb = fmaxf(xb, fmaxf(v[4 * i + 2] + k.x, v[4 * i + 3] + k.y));
                        }
                        move(xa, xb);
                        const float na = (ma == NEG ? 0.f : ma) - kLift, nb = (mb == NEG ? 0.f : mb) - kLift;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float r0 = kr[2 * i], r1 = kr[2 * i + 1];
                            suma += ex2(v[4 * i] - na) + ex2(v[4 * i + 1] - na);
                            sumb += ex2(v[4 * i + 2] - nb) + ex2(v[4 * i + 3] - nb);
                            // a masked position is minus infinity whatever its residual is
                            const float p0 = v[4 * i] == NEG ? 0.f : ex2(v[4 * i] + r0 - na);
                            const float p1 = v[4 * i + 1] == NEG ? 0.f : ex2(v[4 * i + 1] + r1 - na);
                            const float p2 = v[4 * i + 2] == NEG ? 0.f : ex2(v[4 * i + 2] + r0 - nb);
                            const float p3 = v[4 * i + 3] == NEG ? 0.f : ex2(v[4 * i + 3] + r1 - nb);
                            const __half2 h0 = __floats2half2_rn(p0, p1), h1 = __floats2half2_rn(p2, p3);
                            pa[i] = *reinterpret_cast<const uint32_t *>(&h0);
                            pb[i] = *reinterpret_cast<const uint32_t *>(&h1);
                        }
                    }
                } else if (lane == 0) {
                    mbar_arrive(b_sfree + 8 * buf);
                }
                const bool moved = __any_sync(0xffffffffu, ca != 1.f || cb != 1.f);
                if (lane == 0) flags[buf * 4 + w] = (moved ? 1 : 0) | (dead ? 2 : 0);
                // O(t - 1) has been added: P may be written, and the accumulator rescaled. Of two P
                // this tile's was read by O(t - 2), which the widening of this tile has waited for.
                auto added = [&] {
                    if (t > s.t0 && !dead && !wait_all(b_pv + 8 * (at4_buf(g - 1) * 2 + pieces<NB>() - 1), at4_phase(g - 1), abort, K3_SITE_CACHE4, 10, g)) dead = true;
                    tc_after();
                };
                if (!two) added();
                const uint32_t sp_t = sp + (two ? (uint32_t)buf * (kHalf * 128) : 0u);
                if (busy) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        asm volatile("st.shared.b32 [%0], %1;" :: "r"(sp_t + swz(ra, i) + 4 * t4), "r"(pa[i]) : "memory");
                        asm volatile("st.shared.b32 [%0], %1;" :: "r"(sp_t + swz(rb, i) + 4 * t4), "r"(pb[i]) : "memory");
                    }
                }
                if (moved && t4 == 0) { rowf[ra] = ca; rowf[rb] = cb; }
                if (!moved && t4 == 0) { rowf[ra] = 1.f; rowf[rb] = 1.f; }
                named_sync(1, 128);
                const int4 fl = *reinterpret_cast<const int4 *>(flags + buf * 4);
                const int f = fl.x | fl.y | fl.z | fl.w;
                if (f & 2) { dead = true; break; }        // the same for all four warps
                if ((f & 1) && t > s.t0) {
                    if (two) added();
                    for (int blk = 0; blk < NB; blk++)
                        for (int c0 = 0; c0 < NR; c0 += 16) {
                            float o[16];
                            ld16(t_o + lanes + (uint32_t)(blk * kR + c0), o);
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] *= rowf[c0 + i];
                            st16(t_o + lanes + (uint32_t)(blk * kR + c0), o);
                        }
                }
                if (f & 1) named_sync(1, 128);            // rowf is rewritten by the next tile
                async_fence();
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b_pfull + 8 * buf);
            }
            // ---- the item's sums
            suma += __shfl_xor_sync(0xffffffffu, suma, 1);
            sumb += __shfl_xor_sync(0xffffffffu, sumb, 1);
            suma += __shfl_xor_sync(0xffffffffu, suma, 2);
            sumb += __shfl_xor_sync(0xffffffffu, sumb, 2);
            const bool any = s.t0 < s.t1;
            const size_t slot = (size_t)c * 2 + (slot1 ? 1 : 0);
            if (t4 == 0) {
                if (s.whole) {
                    rowf[ra] = suma == 0.f ? 0.f : kUnitF / suma;
                    rowf[rb] = sumb == 0.f ? 0.f : kUnitF / sumb;
                } else {
                    a.ml[slot * kR + ra] = make_float2(ma, suma);
                    a.ml[slot * kR + rb] = make_float2(mb, sumb);
                }
            }
            if (any && !dead && !wait_all(b_pv + 8 * (at4_buf(g - 1) * 2 + pieces<NB>() - 1), at4_phase(g - 1), abort, K3_SITE_CACHE4, 11, g)) dead = true;
            tc_after();
            tc_before();
            named_sync(2, 384);
            tc_after();
            if (!dead) write_out<NB>(a, s, slot, t_o, NR, any, rowf, warp, lane);
            tc_before();
        }
    }
    __syncthreads();
    if (tid == 0) {
        const long long t0 = clock64();
        while (!mbar_try(b_drain, 0)) {
            if (clock64() - t0 > kSpinLimit) { k3_raise_at(K3D_ETIMEOUT, K3_SITE_CACHE4, 12, 0, (int)blockIdx.x); break; }
        }
    }
    __syncthreads();
    if (warp == 12) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
    }
}

// The pieces of each cut item, added in CTA order. Block (k, y, z): the k-th cut item of 64 rows (an
// item is led by the first CTA boundary inside it), its row groups of four y, y + gridDim.y, ...,
// and the z-th share of the latents. Two round trips to memory: the CTAs' info side by side,
// then the pieces with their maxima and sums. blockDim / share threads take a latent's pieces
// in turn and meet in shared memory: few cut items (one long request) get many shares and
// threads, so that the pieces, 131 KB each, are read by the whole card; many get blocks of 256
// threads that lie beside each other on an SM.
constexpr int kMergeMax = 512;            // threads
constexpr int kFew = 8;                   // pieces of an item whose weights are held for all rows
constexpr int kMaxGrid = 148;             // CTAs of k_attend4 (one per SM of a B200)
static_assert(kMaxGrid <= 256, "a thread of the merge for each");
static_assert((kMaxGrid + 1) * 4 >= kFew * kR, "the weights of a few pieces lie in a piece's four each");

// a piece that saw nothing has no weight
__device__ __forceinline__ float weigh(float x, float top, float sum)
{
    return x == __int_as_float(0xff800000) && sum == 0.f ? 0.f : exp2f(x - top);
}

struct Few {
    int2 rows;                            // the item's first row and how many
    size_t first;                         // the first piece's slot
    int c, np, lat;
    int rg_end, rg0, hop;                 // this thread's row groups
};

// Up to kFew pieces: the weights of all rows at once, a row to a thread; then a row group after
// the other, with nothing to wait for but its pieces.
__device__ __forceinline__ void merge_few(const Args &a, const Few &f, float *w, float4 *s_inv4)   // w: [kFew][64]
{
    const int tid = threadIdx.x, odd = tid & 1, kv = a.d.kv;
    auto slot = [&](int k) { return k == 0 ? f.first : (size_t)(f.c - 1 + k) * 2; };
    if (tid < f.rows.y) {
        float2 v[kFew];
        float M = __int_as_float(0xff800000), l = 0.f;
#pragma unroll
        for (int k = 0; k < kFew; k++)
            if (k < f.np) v[k] = a.ml[slot(k) * kR + tid];
#pragma unroll
        for (int k = 0; k < kFew; k++)
            if (k < f.np) M = fmaxf(M, v[k].x);
#pragma unroll
        for (int k = 0; k < kFew; k++)
            if (k < f.np) {
                const float x = weigh(v[k].x, M, v[k].y);
                w[k * kR + tid] = x;
                l = fmaf(x, v[k].y, l);
            }
        reinterpret_cast<float *>(s_inv4)[tid] = l == 0.f ? 0.f : kUnitF / l;
    }
    __syncthreads();
    const float4 *src = reinterpret_cast<const float4 *>(a.part) + (size_t)(f.lat >> 5) * 512 + (f.lat & 31);
    const size_t step = (size_t)(kv / 32) * 512;
    for (int g = f.rg0; g < f.rg_end; g += f.hop) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < f.np; k0 += 4) {
            float4 o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = k0 + k < f.np ? src[slot(k0 + k) * step + g * 32] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (k0 + k >= f.np) break;
                const float4 x = *reinterpret_cast<const float4 *>(w + (k0 + k) * kR + g * 4);
                // without weight nothing is added, whatever the piece holds
                acc[0] = x.x != 0.f ? fmaf(o[k].x, x.x, acc[0]) : acc[0];
                acc[1] = x.y != 0.f ? fmaf(o[k].y, x.y, acc[1]) : acc[1];
                acc[2] = x.z != 0.f ? fmaf(o[k].z, x.z, acc[2]) : acc[2];
                acc[3] = x.w != 0.f ? fmaf(o[k].w, x.w, acc[3]) : acc[3];
            }
        }
        const float4 inv = s_inv4[g];
        const float u[4] = {inv.x, inv.y, inv.z, inv.w};
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = u[i] == 0.f ? 0.f : acc[i] * u[i];
        // neighbouring lanes trade, so that each writes a pair of latents of two rows
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float got = __shfl_xor_sync(0xffffffffu, odd ? acc[i] : acc[i + 2], 1);
            const float x = odd ? got : acc[i], y = odd ? acc[i + 2] : got;
            const int r = g * 4 + i + 2 * odd;
            if (r < f.rows.y) {
                const size_t at = (size_t)(f.rows.x + r) * kv + (f.lat & ~1);
                if (a.out_f32) *reinterpret_cast<float2 *>((float *)a.out + at) = make_float2(x, y);
                else *reinterpret_cast<uint32_t *>((uint16_t *)a.out + at) = bf16x2(x, y);
            }
        }
    }
}

template <bool FEW, bool SPLIT>
__global__ void __launch_bounds__(FEW ? 256 : kMergeMax, FEW ? 4 : 2) k_attend4_merge(const Args a, int grid, int nrg)
{
    __shared__ int s_u0[kMaxGrid + 1], s_begin[kMaxGrid + 1], s_end[kMaxGrid + 1];
    __shared__ int2 s_rows[kMaxGrid + 1];
    __shared__ int s_cnt[kMergeMax / 32], s_c, s_m;        // s_m: the split
    __shared__ float4 s_w[kMaxGrid + 1];               // a piece's weight for four rows
    __shared__ float4 s_red[2][kMergeMax / 32], s_acc[kMergeMax];
    __shared__ float4 s_inv4[kR / 4];                 // 1 / sum of a row
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    if (tid == 0) s_c = -1;
    if (tid < grid) {
        const int4 x = a.info[2 * tid], y = a.info[2 * tid + 1];
        s_u0[tid] = x.x;
        s_begin[tid] = x.y;
        s_end[tid] = x.z;
        s_rows[tid] = make_int2(y.x, y.y);
        if (SPLIT && tid == 0) s_m = x.w;
    }
    __syncthreads();
    // items of fewer rows: m of them share the blocks that one of 64 rows has
    const int sh = SPLIT ? s_m : 0, m = 1 << sh, part = blockIdx.y & (m - 1), which = (blockIdx.x << sh) + part;
    const int y0 = blockIdx.y >> sh, ny = (gridDim.y - part + m - 1) >> sh;
    const bool leads = tid >= 1 && tid < grid && s_begin[tid] >= 0 && s_begin[tid] < s_u0[tid] && s_u0[tid - 1] <= s_begin[tid];
    const unsigned m32 = __ballot_sync(0xffffffffu, leads);
    if (lane == 0) s_cnt[warp] = __popc(m32);
    __syncthreads();
    int rank = __popc(m32 & ((1u << lane) - 1u));
    for (int k = 0; k < warp; k++) rank += s_cnt[k];
    if (leads && rank == which) s_c = tid;
    __syncthreads();
    const int c = s_c;
    if (c < 0) return;
    // pieces: CTA c - 1 (its second slot unless the item begins its range), then c, c + 1, ...
    const int2 rw = s_rows[c];
    const int end = s_end[c];
    const int np = 1 + __syncthreads_count(tid >= c && tid < grid && s_u0[tid] < end);
    const size_t first = (size_t)(c - 1) * 2 + (s_u0[c - 1] == s_begin[c] ? 0 : 1);
    auto slot = [&](int k) { return k == 0 ? first : (size_t)(c - 1 + k) * 2; };
    const float NEG = __int_as_float(0xff800000);
    const int kv = a.d.kv, share = kv / gridDim.z, ways = blockDim.x / share;
    const int lat = blockIdx.z * share + tid % share, way = tid / share;
    if (FEW && np <= kFew) {
        merge_few(a, Few{rw, first, c, np, lat, way < ways ? (rw.y + 3) / 4 : 0, y0 * ways + way, ny * ways},
                  reinterpret_cast<float *>(s_w), s_inv4);
        return;
    }
    for (int rg = y0; rg < nrg && rg * 4 < rw.y; rg += ny) {
        const float4 *src = reinterpret_cast<const float4 *>(a.part) + ((size_t)(lat >> 5) * 16 + rg) * 32 + (lat & 31);
        const size_t step = (size_t)(kv / 32) * 512;
        // the first pieces are on their way before their weights are known
        float4 ahead[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int k = way + i * ways;
            ahead[i] = way < ways && k < np ? src[slot(k) * step] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float4 M = make_float4(NEG, NEG, NEG, NEG), l = make_float4(0.f, 0.f, 0.f, 0.f);
        auto ml4 = [&](int k, float4 &m, float4 &s) {
            const float4 *p = reinterpret_cast<const float4 *>(a.ml + slot(k) * kR + rg * 4);
            const float4 x = p[0], y = p[1];
            m = make_float4(x.x, x.z, y.x, y.z);
            s = make_float4(x.y, x.w, y.y, y.w);
        };
        for (int k = tid; k < np; k += blockDim.x) {
            float4 m, s;
            ml4(k, m, s);
            M = make_float4(fmaxf(M.x, m.x), fmaxf(M.y, m.y), fmaxf(M.z, m.z), fmaxf(M.w, m.w));
        }
        M = make_float4(warp_max(M.x), warp_max(M.y), warp_max(M.z), warp_max(M.w));
        if (lane == 0) s_red[0][warp] = M;
        __syncthreads();
        for (int i = 0; i < nw; i++) {
            const float4 t = s_red[0][i];
            M = make_float4(fmaxf(M.x, t.x), fmaxf(M.y, t.y), fmaxf(M.z, t.z), fmaxf(M.w, t.w));
        }
        for (int k = tid; k < np; k += blockDim.x) {
            float4 m, s;
            ml4(k, m, s);
            const float4 f = make_float4(weigh(m.x, M.x, s.x), weigh(m.y, M.y, s.y), weigh(m.z, M.z, s.z), weigh(m.w, M.w, s.w));
            s_w[k] = f;
            l = make_float4(fmaf(f.x, s.x, l.x), fmaf(f.y, s.y, l.y), fmaf(f.z, s.z, l.z), fmaf(f.w, s.w, l.w));
        }
        l = make_float4(warp_sum(l.x), warp_sum(l.y), warp_sum(l.z), warp_sum(l.w));
        if (lane == 0) s_red[1][warp] = l;
        __syncthreads();
        l = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < nw; i++) {
            const float4 t = s_red[1][i];
            l.x += t.x; l.y += t.y; l.z += t.z; l.w += t.w;
        }
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](int k, const float4 &o) {
            const float4 w = s_w[k];
            // without weight nothing is added, whatever the piece holds
            acc.x = w.x != 0.f ? fmaf(o.x, w.x, acc.x) : acc.x;
            acc.y = w.y != 0.f ? fmaf(o.y, w.y, acc.y) : acc.y;
            acc.z = w.z != 0.f ? fmaf(o.z, w.z, acc.z) : acc.z;
            acc.w = w.w != 0.f ? fmaf(o.w, w.w, acc.w) : acc.w;
        };
        if (way < ways) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (way + i * ways < np) add(way + i * ways, ahead[i]);
#pragma unroll 1
            for (int k = way + 4 * ways; k < np; k += 4 * ways) {
                float4 o[4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    o[i] = k + i * ways < np ? src[slot(k + i * ways) * step] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (k + i * ways < np) add(k + i * ways, o[i]);
            }
        }
        if (way > 0 && way < ways) s_acc[tid] = acc;
        __syncthreads();
        if (way == 0) {
            for (int i = 1; i < ways; i++) {
                const float4 t = s_acc[i * share + tid];
                acc.x += t.x; acc.y += t.y; acc.z += t.z; acc.w += t.w;
            }
            const float v[4] = {acc.x, acc.y, acc.z, acc.w}, s[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (rg * 4 + i < rw.y) {
                    const float r = s[i] == 0.f ? 0.f : v[i] * (kUnitF / s[i]);
                    const size_t at = (size_t)(rw.x + rg * 4 + i) * kv + lat;
                    if (a.out_f32) ((float *)a.out)[at] = r;
                    else ((uint16_t *)a.out)[at] = f32_to_bf16_bits(r);
                }
        }
        __syncthreads();
    }
}

static int grid_size() { return sm_count() < kMaxGrid ? sm_count() : kMaxGrid; }

static Split split(int H, int rows) { return {rows, H <= rows ? rows / H : 1, (H + rows - 1) / rows}; }

static long long most_items(int N, int H, int rows) { return (long long)N * ((H + rows - 1) / rows); }

static size_t al256(size_t b) { return (b + 255) & ~(size_t)255; }

struct Ws {
    size_t part, ml, info, total;
};

// For the whole of kMaxGrid, so that the size does not depend on when it is asked for.
static Ws ws_layout(int kv)
{
    const size_t g = kMaxGrid;
    Ws w;
    w.part = 0;
    w.ml = al256(g * 2 * kR * kv * sizeof(float));
    w.info = w.ml + al256(g * 2 * kR * sizeof(float2));
    w.total = w.info + al256(g * 2 * sizeof(int4));
    return w;
}

template <int NB, bool SPLIT>
static cudaError_t launch_as(const Args &a, int grid, size_t smem, cudaStream_t st)
{
    static unsigned long long init = 0;   // one bit per device
    if (!(init & dev_bit())) {
        allow_smem_max(k_attend4<NB, SPLIT>);
        init |= dev_bit();
    }
    return launch_pdl(k_attend4<NB, SPLIT>, dim3(grid), dim3(kThreads), smem, st, a);
}

template <int NB>
static cudaError_t launch(const Args &a, int grid, size_t smem, cudaStream_t st)
{
    return a.splits > 1 ? launch_as<NB, true>(a, grid, smem, st) : launch_as<NB, false>(a, grid, smem, st);
}

}  // namespace at4
}  // namespace k3

using namespace k3;

extern "C" {

size_t k3d_mla_attend4_ws_bytes(const K3dCache4 *c, int B, int N, int H)
{
    if (cache4_check(c, "k3d_mla_attend4_ws_bytes") || B < 1 || N < 0 || H < 1) return 0;
    return at4::ws_layout(c->kv_lora).total;
}

int k3d_mla_attend4(void *out, int out_dtype, const void *q, int q_dtype, const K3dCache4 *c, const void *pool,
                    const int *table, int max_pages, const int *row_start, const int *kv_len, int B, int N, int H,
                    float scale, void *ws, size_t ws_bytes)
{
    K3_TRY(cache4_check(c, "k3d_mla_attend4"));
    // positions, rows and requests are counted in 31 bits, with a tile to spare
    constexpr long long kMost = 1LL << 30;
    if (B < 1 || B > kMost || N < 0 || H < 1 || H > 1024 || max_pages < 1 || (long long)max_pages * c->page > kMost ||
        (long long)N * H > kMost)
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
    const at4::Ws w = at4::ws_layout(c->kv_lora);
    char *wb = (char *)ws;
    const int grid = at4::grid_size();
    // at most one cut item per CTA boundary, and no more than there are items
    const long long items = at4::most_items(N, H, at4::kR);
    const int cuts = (int)(items < grid - 1 ? items : grid - 1);
    // row groups by the average rows of a request (more are looped over)
    const long long rows = ((long long)N + B - 1) / B * H;
    const int most = (H < at4::kR ? at4::kR / H * H : at4::kR) + 3;
    const int nrg = most / 4;
    int y = (int)(rows < 4LL * nrg ? (rows + 3) / 4 : nrg);
    // Fewer rows to an item where the items are so few that the kernel may find idle SMs: the
    // smallest split whose tiles have a CTA each is taken there (64 heads, 1000 positions: 19.4 us
    // with items of 64 rows, 17.5 with 16).
    int splits = 1;
    while (splits < 3 && B <= 64 && y >= 1 << splits && at4::most_items(N, H, at4::kR >> splits) * 4 <= grid) splits++;
    const at4::Args a{pool4(c, pool), q, out, table, row_start, kv_len, max_pages, B, N, H,
                      q_dtype == K3D_DT_F32, out_dtype == K3D_DT_F32, {at4::split(H, 64), at4::split(H, 32), at4::split(H, 16)},
                      splits, 1.0f / (float)H, scale,
                      (float *)(wb + w.part), (float2 *)(wb + w.ml), (int4 *)(wb + w.info)};
    const size_t smem = 1024 + at4::smem_layout(c->kv_lora, c->qk_rope).total;
    switch (c->kv_lora / 128) {
    case 1: at4::launch<1>(a, grid, smem, stream()); break;
    case 2: at4::launch<2>(a, grid, smem, stream()); break;
    case 3: at4::launch<3>(a, grid, smem, stream()); break;
    default: at4::launch<4>(a, grid, smem, stream()); break;
    }
    note_launch();
    K3_TRY(check_launch("mla attend4"));
    if (cuts > 0) {
        int z = (c->kv_lora + 255) / 256, threads = 256;
        // Items that are cut in a few pieces on average: one wave of blocks that go through their
        // row groups without meeting (64 items: 21 us with a block for each group, 11 so).
        const bool few = cuts * at4::kFew >= grid;
        if (few) {
            const int wave = 4 * grid / (cuts * z);
            y = y < wave ? y : wave > 1 ? wave : 1;
        } else {
            // shares of 32 latents where an item may have more than 32 pieces (32768 positions:
            // 32 us with shares of 64, 30.3 with 32), else of 64 (1000 positions: 19.2 and 19.7)
            const int least = grid > 32 && (long long)max_pages * c->page > 32 * at4::kT ? 32 : 64;
            while (c->kv_lora % (z * 2) == 0 && c->kv_lora / (z * 2) >= least && (long long)cuts * y * z * 2 <= 2 * grid) z *= 2;
            if ((long long)cuts * y * z <= 2 * grid) threads = 512;
        }
        launch_pdl(few ? splits > 1 ? at4::k_attend4_merge<true, true> : at4::k_attend4_merge<true, false>
                       : splits > 1 ? at4::k_attend4_merge<false, true> : at4::k_attend4_merge<false, false>,
                   dim3(cuts, y, z), dim3(threads), 0, stream(), a, grid, nrg);
        note_launch();
        K3_TRY(check_launch("mla attend4 merge"));
    }
    return K3D_OK;
}

}  // extern "C"
