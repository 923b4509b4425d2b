/* k3_attend4_order.h -- which barrier and which phase of it announce a step of tile g in
 * k_attend4 (k3_attend4.cu), g counting a CTA's tiles from 0. Two tiles are on their way at a
 * time, and everything that is held for both (the widened tile, S, P, the end of O^T) has a
 * barrier for each, which flips once for every second tile.
 *
 * A wait by parity cannot tell a phase from the one two further on, so a barrier may only flip
 * again once everyone who waits for its last phase has seen it. With a barrier for each of the
 * two that follows from the chain: whatever tile g + 2 announces comes behind its widening,
 * which waits for O(g), which comes behind all that tile g announced. One barrier for both P
 * would not do: with up to 32 rows P(g + 1) does not wait for O(g), and would flip the barrier
 * under a wait for P(g). A CPU test walks through every order of the roles with these two
 * functions. */
#ifndef K3_ATTEND4_ORDER_H
#define K3_ATTEND4_ORDER_H

#ifdef __CUDACC__
#define K3_AT4_HD __host__ __device__ __forceinline__
#else
#define K3_AT4_HD static inline
#endif

/* The buffer of tile g, and its barrier. */
K3_AT4_HD int at4_buf(int g) { return g & 1; }

/* The parity to wait with for tile g's phase of that barrier. */
K3_AT4_HD unsigned at4_phase(int g) { return (unsigned)(g >> 1) & 1u; }

#endif
