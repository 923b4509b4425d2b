"""Plain definitions, in 64 bits or whole numbers, of the serving operators: the 4-bit latent
row, the attention over it, page plans, probabilities and the verification of drafts."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _e4m3_table():
    v = []
    for b in range(127):
        e, m = b >> 3, b & 7
        v.append((1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6)
    return np.array(v)


E4M3 = _e4m3_table()


def _nearest(x, table):
    """Index of the nearest table entry, the even one of two as near."""
    hi = np.clip(np.searchsorted(table, x), 1, len(table) - 1)
    lo = hi - 1
    a, b = x - table[lo], table[hi] - x
    up = (b < a) | ((a == b) & (hi % 2 == 0))
    return np.where(up, hi, lo)


def quantise(x, kv):
    """Rows [N][kv + rope] as (codes, scale bytes, rope fp16, exponent bytes) and their values."""
    x = np.asarray(x, np.float64)
    n = x.shape[0]
    bad = ~np.isfinite(x).all(1)
    x = np.where(bad[:, None], 0.0, x)

    def unit(a, m, le):
        f, e = np.frexp(a)
        return np.where(a > 0, e - le + (f > m), -100)

    k = np.maximum(unit(np.abs(x[:, :kv]).max(1), 0.65625, 12),
                   unit(np.abs(x[:, kv:]).max(1) if x.shape[1] > kv else np.zeros(n), 0.5, 16))
    k = np.where(bad, 0, np.maximum(k, -100)).astype(np.int64)
    y = np.ldexp(x, -k[:, None])
    blk = y[:, :kv].reshape(n, kv // 16, 16)
    sb = _nearest((np.abs(blk).max(2) / 6).astype(np.float32).astype(np.float64), E4M3)
    s = E4M3[sb][:, :, None]
    code = _nearest(np.divide(np.abs(blk), s, out=np.zeros_like(blk), where=s > 0), E2M1)
    lat = E2M1[code] * np.where(np.signbit(blk), -1.0, 1.0) * s
    rope = y[:, kv:].astype(np.float16)
    value = np.concatenate([lat.reshape(n, kv), rope.astype(np.float64)], 1)
    value = np.ldexp(value, k[:, None])
    value[bad] = np.nan
    code = (code | (np.signbit(blk) << 3)).reshape(n, kv // 2, 2).astype(np.uint8)
    return ((code[:, :, 0] | (code[:, :, 1] << 4)).astype(np.uint8), sb.astype(np.uint8), rope,
            np.where(bad, 255, k + 127).astype(np.uint8)), value


def page_bytes(kv, rope, page):
    return page * (kv // 2 + kv // 16 + 2 * rope + 1)


def put_rows(pool, kv, rope, page, slots, fields):
    """Writes quantised rows into a pool (uint8 [n_pages][page bytes]) at their slots."""
    codes, scales, rp, exps = fields
    o1 = page * (kv // 2)
    o2 = o1 + page * (kv // 16)
    o3 = o2 + page * 2 * rope
    for r, s in enumerate(slots):
        if s < 0:
            continue
        p, i = divmod(int(s), page)
        pool[p, i * (kv // 2):(i + 1) * (kv // 2)] = codes[r]
        pool[p, o1 + i * (kv // 16):o1 + (i + 1) * (kv // 16)] = scales[r]
        if rope:
            pool[p, o2 + i * 2 * rope:o2 + (i + 1) * 2 * rope] = rp[r].view(np.uint8)
        pool[p, o3 + i] = exps[r]


def attend(q, values, kv, scale, n_new):
    """One request: q [n_new][H][W], values [kv_len][W]; rows without a position are zeros."""
    L = len(values)
    out = np.zeros((n_new, q.shape[1], kv))
    for j in range(n_new):
        seen = max(0, L - n_new + j + 1)
        if seen == 0:
            continue
        v = values[:seen]
        s = q[j].astype(np.float64) @ v.T * scale
        with np.errstate(invalid="ignore"):
            p = np.exp(s - s.max(1, keepdims=True))
            out[j] = (p / p.sum(1, keepdims=True)) @ v[:, :kv]
    return out


class Pages:
    """The page plan in Python lists."""

    def __init__(self, page, n_pages, max_pages, B, free):
        self.page, self.n_pages, self.max_pages = page, n_pages, max_pages
        self.table = [[] for _ in range(B)]
        self.free = list(free)

    def plan(self, lens, new, N):
        need = [-(-(a + b) // self.page) for a, b in zip(lens, new)]
        back = [(b, j) for b in range(len(lens)) for j in range(need[b], len(self.table[b]))]
        free = self.free + [self.table[b][j] for b, j in reversed(back)]
        more = sum(max(0, n - len(t)) for n, t in zip(need, self.table))
        code = 0
        if max(need) > self.max_pages:
            code = 3
        elif sum(new) > N:
            code = 2
        elif more > len(free):
            code = 1
        if code:
            return code, [0] * (len(lens) + 1), [0] * len(lens), [-1] * N, [-1] * N
        for b, n in enumerate(need):
            del self.table[b][n:]
            while len(self.table[b]) < n:
                self.table[b].append(free.pop())
        self.free = free
        start = [0]
        pos, slots = [], []
        for b, n in enumerate(new):
            start.append(start[-1] + n)
            for t in range(lens[b], lens[b] + n):
                pos.append(t)
                slots.append(self.table[b][t // self.page] * self.page + t % self.page)
        pad = N - len(pos)
        return 0, start, [a + b for a, b in zip(lens, new)], pos + [-1] * pad, slots + [-1] * pad


def softmax(x, temp):
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    out = np.zeros_like(x)
    for r in range(x.shape[0]):
        t = 1.0 if temp is None else float(temp[r])
        m = x[r].max()
        if m == -np.inf:
            continue
        if not t > 0:
            out[r, int(x[r].argmax())] = 1.0
        elif m == np.inf:
            out[r] = (x[r] == np.inf) / (x[r] == np.inf).sum()
        else:
            with np.errstate(invalid="ignore"):
                e = np.where(x[r] == -np.inf, 0.0, np.exp((x[r] - m) / t))
            out[r] = e / e.sum()
    return out


def verify(target, draft, ids, n_draft, u, us):
    """Python whole numbers: weights in 2^-44."""
    B, K1, V = target.shape
    K = K1 - 1
    tokens, acc = [], []

    def weights(r):
        r = np.clip(np.nan_to_num(np.asarray(r, np.float32), nan=0.0), 0.0, 1.0)
        return np.floor(r.astype(np.float64) * 2.0 ** 44).astype(np.int64)

    for b in range(B):
        nd = K if n_draft is None else max(0, min(K, int(n_draft[b])))
        n = 0
        while n < nd:
            d = int(ids[b, n])
            if not 0 <= d < V:
                break
            qd = 1.0 if draft is None else float(draft[b, n, d])
            if not float(u[b, n]) * qd < float(target[b, n, d]):
                break
            n += 1
        p = target[b, n].astype(np.float32)
        w = weights(p)
        if n < nd:
            if draft is not None:
                cut = p - draft[b, n].astype(np.float32)
            else:
                cut = p.copy()
                if 0 <= ids[b, n] < V:
                    cut[ids[b, n]] -= np.float32(1)
            if weights(cut).sum() > 0:
                w = weights(cut)
        total = int(w.sum())
        if total == 0:
            tok = -1
        else:
            x = float(us[b])
            t = min(int(np.floor(x * float(total))), total - 1) if x > 0 else 0
            tok = int(np.searchsorted(np.cumsum(w), t, side="right"))
        tokens.append([int(i) for i in ids[b, :n]] + [tok] + [-1] * (K - n))
        acc.append(n)
    return np.array(tokens, np.int32), np.array(acc, np.int32)
