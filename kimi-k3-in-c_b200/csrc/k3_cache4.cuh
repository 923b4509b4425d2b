// k3_cache4.cuh -- the 4-bit latent row and the paged pool that holds it, shared by the
// store / load kernels (k3_cache4.cu) and the attention over the pool (k3_attend4.cu).
//
// A row of kv latent values and rope rotated key values is held in units of 2^e:
//   e       smallest integer >= -100 with max|latent| <= 2688 2^e and max|rope| <= 32768 2^e
//           (2688 = 6 x 448, the largest E2M1 code times the largest E4M3 scale); one byte
//           e + 127, or 255 for a row that held a NaN or an infinity (all its values are NaN)
//   latent  blocks of 16: s = e4m3(max|x| 2^-e / 6), codes e2m1(x 2^-e / s), ties to even
//   rope    fp16 of x 2^-e
// Within a row every value is therefore an fp16 number times 2^e: code x scale has at most
// six significant bits and lies in [2^-10, 2688], so the attention multiplies fp16 latents
// without a rounding and applies 2^e per key. (Rotated keys far below their row's
// latents are rounded on the way, k3_attend4.cu.)
// A page holds `page` rows as four arrays, each 16-byte aligned (page is a multiple of 16):
//   codes [page][kv/2] | scales [page][kv/16] | rope [page][rope] fp16 | exponents [page]
#pragma once
#include <cuda_fp8.h>

#include "k3_common.cuh"

namespace k3 {

struct Pool4 {
    uint8_t *p;
    int kv, rope, page, n_pages;
    size_t page_bytes;
    uint32_t o_scale, o_rope, o_exp;      // offsets of the arrays in a page
};

inline Pool4 pool4(const K3dCache4 *c, const void *pool)
{
    Pool4 d;
    d.p = (uint8_t *)const_cast<void *>(pool);
    d.kv = c->kv_lora; d.rope = c->qk_rope; d.page = c->page; d.n_pages = c->n_pages;
    d.o_scale = (uint32_t)c->page * (c->kv_lora / 2);
    d.o_rope = d.o_scale + (uint32_t)c->page * (c->kv_lora / 16);
    d.o_exp = d.o_rope + (uint32_t)c->page * 2 * c->qk_rope;
    d.page_bytes = (size_t)d.o_exp + c->page;
    return d;
}

// K3D_OK, or K3D_EINVAL recorded with the entry point's name.
int cache4_check(const K3dCache4 *c, const char *who);

// E4M3 byte -> fp32 (exact; 0x7f and 0xff, which the store never writes, are NaN).
__device__ __forceinline__ float e4m3_to_f32(uint8_t b)
{
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

}  // namespace k3
