"""How far the attention over the 4-bit cache may be from its definition, element by element, and
inputs that make the bound narrow.

With exact scores s_t, weights p_t and result o = sum p_t v_t, the kernel has scores off by at most d_t,
so its weights are p_t e^(+-d_t) over their sum, and since sum p_t (v_t - o) = 0 its result is off by at
most  sum p_t expm1(d_t) |v_t - o| / sum p_t e^(-d_t).  d_t, in natural units:
  * the fp32 sum of W products, each addition off by at most a step (the tensor core truncates) of a
    running sum of at most scale sum|q v|: W 2^-23 of that; nothing where `exact`, that is where all
    products and their sums are multiples of a power of two below 2^24 of it;
  * the way from the product to the exponent: the factor (three roundings), the product, the reference
    m, its difference and the residual: eight roundings of numbers of at most |s_t| + max|s| + 15 ln 2 +
    |r| ln 2, r the largest residual exponent, each 2^-24 of it;
  * the rotated key, fp16 in units of 2^e, is taken to units of 2^-2 2^res, res = e - clamp(e, -16, -2), and
    rounds by at most 2^-25 of that unit where e < -2: scale sum_rope |q| 2^(-27 + res).
q is fp16 in units of its row (exact for bf16 within 2^-29 of its largest); the definition is given it so.
Then, of sum p_t |v_t|: 2^-11 for the fp16 weights, n 2^-22 for the fp32 sums over n positions (weights
and values, a step each) and 2^-20 for exp2 and the merge. And half a step of the result's type.

Weights below 2^-14 / 2^7 of the running maximum: the kernel rounds P_t = 2^(a_t - m + 7), a_t = s_t log2(e) +
r_t, r_t the position's residual exponent, to fp16, whose steps stop at 2^-24, so P_t is off by up to 2^-25
however small it is. The result is sum P_t (v_t 2^-r_t) / L with L = sum 2^(a_t - r_t - m + 7). m is never
above the largest a, which position * has, so its term alone gives L >= 2^(7 - r_*): the result moves by at
most 2^-25 sum |v_t| 2^-r_t / 2^(7 - r_*) = 2^-32 sum |v_t| 2^(r_* - r_t). (In a column where the
positions of weight hold zeros that is all there is.)"""
import numpy as np

import serving_ref as ref

EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def rounded(q):
    """Query rows as the kernel takes them: fp16 of q 2^(14 - e), the row's largest value in
    [2^(e - 1), 2^e)."""
    q = np.asarray(q, np.float64)
    e = np.frexp(np.abs(q).max(-1, keepdims=True))[1]
    return np.ldexp(np.ldexp(q, 14 - e).astype(np.float16).astype(np.float64), e - 14)


def bound(q, v, exps, kv, scale, n, out="f32", exact=False):
    """One request: (want, tol), both [n][H][kv]. q [n][H][W], v [kv_len][W] and exps [kv_len] as
    serving_ref.quantise gives them (exps: the exponent e)."""
    L, H = len(v), q.shape[1]
    want, tol = np.zeros((n, H, kv)), np.zeros((n, H, kv))
    q = rounded(q)
    W = q.shape[-1]
    for j in range(n):
        seen = max(0, L - n + j + 1)
        if seen == 0:
            continue
        x, w, e = q[j], v[:seen], exps[:seen]
        res = e - np.clip(e, -16, -2)
        s = x @ w.T * scale
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        o = p @ w[:, :kv]
        mag = scale * (np.abs(x) @ np.abs(w).T)
        d = (0.0 if exact else W * 2.0 ** -23) * mag
        d += 8 * 2.0 ** -24 * (np.abs(s) + np.abs(s).max(1, keepdims=True) + np.log(2) * (15 + np.abs(res).max()))
        d += scale * np.abs(x[:, kv:]).sum(1)[:, None] * np.where(e < -2, 2.0 ** (-27.0 + res), 0.0)
        t = np.einsum("ht,htk->hk", p * np.expm1(d), np.abs(w[None, :, :kv] - o[:, None]))
        t /= (p * np.exp(-d)).sum(1)[:, None]
        t += (2.0 ** -11 + seen * 2.0 ** -22 + 2.0 ** -20) * (p @ np.abs(w[:, :kv]))
        top = res[(s * np.log2(np.e) + res).argmax(1)]
        t += 2.0 ** -32 * np.exp2(1.0 * top[:, None]) * (np.abs(w[:, :kv]) * np.exp2(-1.0 * res[:, None])).sum(0)
        want[j], tol[j] = o, t + EPS[out] * (np.abs(o) + t)
    return want, tol


# ------------------------------------------------------------------------------ inputs ----
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def grid_rows(g, k, kv, rope, lift=None):
    """Rows that the cache holds as they are: latents of the E2M1 values (a 6 in each block, so that its
    scale is a power of two), whole rotated keys; lift[t // 64] is the first rotated key of position t."""
    x = np.zeros((k, kv + rope), np.float32)
    x[:, :kv] = g.choice(GRID, (k, kv)) * g.choice([-1.0, 1.0], (k, kv))
    blocks = x[:, :kv].reshape(k, kv // 16, 16)
    at = g.integers(0, 16, blocks.shape[:2])
    np.put_along_axis(blocks, at[:, :, None], 6.0 * g.choice([-1.0, 1.0], at.shape)[:, :, None], 2)
    x[:, :kv] = blocks.reshape(k, kv)
    if rope:
        x[:, kv:] = g.integers(-2, 3, (k, rope))
        if lift is not None:
            x[:, kv] = np.asarray(lift)[(np.arange(k) // 64) % len(lift)]
    return x


def grid_queries(g, N, H, kv, rope, gain, lifted=False):
    """Queries of -1, 0 and 1, a third each, times a power of two."""
    q = g.integers(-1, 2, (N, H, kv + rope)).astype(np.float32)
    if lifted:
        q[:, :, kv] = 1.0
    return q * np.float32(gain)


# the first rotated key by tiles: with a scale of 2^-4 and gain 1, 11 is one power of two; the running
# maximum jumps by up to 12 powers of two, falls back, and the tiles at the end still share the weight
LIFT = [0, 100, 30, 120, 240, 180, 300, 330, 320, 340, 335]


# ---------------------------------------------------------------- mistakes, made on the CPU ----
def without(q, v, kv, scale, n, t):
    """The result that leaves position t out."""
    L = len(v)
    out = np.zeros((n, q.shape[1], kv))
    for j in range(n):
        keep = [i for i in range(max(0, L - n + j + 1)) if i != t]
        if keep:
            out[j] = ref.attend(q[j:j + 1], v[keep], kv, scale, 1)[0]
    return out


def shifted(q, v, kv, scale, n, by):
    """The result whose causal limit is off by `by`."""
    L = len(v)
    out = np.zeros((n, q.shape[1], kv))
    for j in range(n):
        seen = min(L, max(0, L - n + j + 1 + by))
        if seen:
            out[j] = ref.attend(q[j:j + 1], v[:seen], kv, scale, 1)[0]
    return out


def no_rescale(q, v, kv, scale, n, which=None):
    """Tiles of 64 with a running maximum that moves, whose sum follows it and whose accumulator does not,
    at all moves or at the which-th alone."""
    L = len(v)
    out = np.zeros((n, q.shape[1], kv))
    for j in range(n):
        seen = max(0, L - n + j + 1)
        if not seen:
            continue
        s = q[j].astype(np.float64) @ v[:seen].T * scale
        for h in range(q.shape[1]):
            m, l, o, moves = -np.inf, 0.0, np.zeros(kv), 0
            for t in range(0, seen, 64):
                top = s[h, t:t + 64].max()
                if m == -np.inf:
                    m = top
                elif top > m + 8 * np.log(2):
                    f = np.exp(m - top)
                    l *= f
                    if which is not None and moves != which:
                        o *= f
                    moves += 1
                    m = top
                p = np.exp(s[h, t:t + 64] - m)
                l += p.sum()
                o += p @ v[t:min(t + 64, seen), :kv]
            out[j, h] = o / l
    return out
