"""The serving operators around the latent cache: what one pass of each is, in plain torch
and through the library.

Five operators, as a serving loop with drafted tokens runs them:
  plan     page tables and slot maps from the requests' lengths (k3d_page_plan)
  store    latent rows quantised to 4 bits into their slots, and read back
           (k3d_cache4_store, k3d_cache4_load)
  attend   absorbed MLA attention over the paged 4-bit cache (k3d_mla_attend4)
  softmax  sampling probabilities of logits rows, a temperature each (k3d_logits_softmax)
  verify   drafted tokens against the target's probabilities (k3d_spec_verify)

THE 4-BIT ROW. A row of kv_lora latent values and qk_rope rotated key values is held in
units of 2^e, e the row's own exponent (one byte, e + 127): every 16 latent values share an
E4M3 scale s = e4m3(max|x| 2^-e / 6) and are E2M1 codes of x 2^-e / s, two to a byte, the
even element in the low nibble; the rotated key is fp16 of x 2^-e. e is the smallest integer
>= -100 with max|latent| <= 2688 2^e (6 x 448) and max|rope| <= 32768 2^e. A row with a NaN
or an infinity is stored as NaN (exponent byte 255). A page holds `page` rows as four arrays
one after the other: codes [page][kv_lora / 2], scales [page][kv_lora / 16], rope
[page][qk_rope] fp16, exponent bytes [page].
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

VOCAB = 163840
HEAD = 192          # qk_nope + qk_rope: the softmax scale is 1 / sqrt(192)

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


# --------------------------------------------------------------------------- the cases ----
def listed():
    return [
        # one chat request, a short context, one token a step: launch latency
        {"name": "attend 1 x 1000, 64 heads", "op": "attend", "B": 1, "L": 1000, "ragged": 0, "n": 1,
         "H": 64, "kv": 512, "rope": 64, "page": 64},
        # one long document, one token a step: the cached positions are split over the card
        {"name": "attend 1 x 32768, 64 heads", "op": "attend", "B": 1, "L": 32768, "ragged": 0, "n": 1,
         "H": 64, "kv": 512, "rope": 64, "page": 64},
        # a batch of ragged contexts on one of four ranks that share the heads: bytes bound
        {"name": "attend 64 ragged, 16 heads", "op": "attend", "B": 64, "L": 8192, "ragged": 7, "n": 1,
         "H": 16, "kv": 512, "rope": 64, "page": 64},
        # three drafted tokens and the last accepted one verified together: arithmetic bound
        {"name": "attend 16 ragged x 4, 64 heads", "op": "attend", "B": 16, "L": 8192, "ragged": 3, "n": 4,
         "H": 64, "kv": 512, "rope": 64, "page": 64},
        # the new rows of a decode step of 64 sequences
        {"name": "store 64 rows", "op": "store", "N": 64, "x": "f32", "kv": 512, "rope": 64, "page": 64},
        # a prompt's rows of 8191 tokens
        {"name": "store 8191 rows", "op": "store", "N": 8191, "x": "bf16", "kv": 512, "rope": 64, "page": 64},
        # a decode step of 64 requests with four tokens each, and the drafts rolled back
        {"name": "plan 64 x 4", "op": "plan", "B": 64, "L": 8192, "n": 4, "prompt": False, "page": 64},
        # 100 prompts of up to 8192 tokens admitted and given back
        {"name": "plan 100 prompts", "op": "plan", "B": 100, "L": 8192, "n": 0, "prompt": True, "page": 64},
        # the rows of one request's verification: the last token and four drafts
        {"name": "softmax 5 rows", "op": "softmax", "rows": 5, "V": VOCAB, "greedy": False},
        # the same of a batch of 64, some of its requests greedy
        {"name": "softmax 320 rows", "op": "softmax", "rows": 320, "V": VOCAB, "greedy": True},
        # one request, four drafts that carry their probabilities
        {"name": "verify 1 x 4", "op": "verify", "B": 1, "K": 4, "V": VOCAB, "probs": True},
        # a batch of 64 with up to four drafts each
        {"name": "verify 64 x 4", "op": "verify", "B": 64, "K": 4, "V": VOCAB, "probs": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "store", "plan", "softmax", "verify"])
    if op == "attend":
        H = rng.choice([8, 16, 24, 32, 64, 96, 128])
        n = rng.choice([1, 1, 2, 3, 5, 8])
        B = _log(rng, 1, 64)
        # as much as the largest listed case at most: rows x positions, and cached rows
        most = min(16 * 4096 * 256 // (B * n * H), 64 * 4096 // B, 32768)
        L = _log(rng, 1, max(2, most))
        return {"op": op, "B": B, "L": max(L, n), "ragged": rng.randrange(1 << 16), "n": n, "H": H,
                "kv": rng.choice([512, 512, 512, 256, 128]), "rope": rng.choice([64, 64, 64, 32, 16]),
                "page": rng.choice([16, 32, 64, 128])}
    if op == "store":
        return {"op": op, "N": _log(rng, 1, 8191), "x": rng.choice(["f32", "bf16"]),
                "kv": rng.choice([512, 512, 256, 128]), "rope": rng.choice([64, 64, 32, 16]),
                "page": rng.choice([16, 32, 64, 128])}
    if op == "plan":
        prompt = rng.random() < 0.5
        return {"op": op, "B": _log(rng, 1, 100 if prompt else 700), "L": _log(rng, 8, 8192),
                "n": 0 if prompt else rng.randint(1, 8), "prompt": prompt, "page": rng.choice([16, 32, 64, 128])}
    V = _log(rng, 1000, VOCAB)
    if op == "softmax":
        return {"op": op, "rows": _log(rng, 1, 320), "V": V, "greedy": rng.random() < 0.5}
    return {"op": op, "B": _log(rng, 1, 64), "K": rng.randint(1, 4), "V": V, "probs": rng.random() < 0.7}


def _lengths(case):
    """The requests' lengths of a case: kv lengths with the new rows, and the new rows."""
    B, L, n = case["B"], case["L"], case["n"]
    r = random.Random(case["ragged"])
    if not case["ragged"]:
        return [L] * B, [n] * B
    new = [n] * B
    kv = [max(new[b], r.randint(max(1, L // 16), L)) for b in range(B)]
    return kv, new


def _plan_lengths(case):
    r = random.Random(case["B"] * 131 + case["L"])
    lens = [r.randint(1, case["L"]) for _ in range(case["B"])]
    return ([0] * len(lens), lens) if case["prompt"] else (lens, [case["n"]] * len(lens))


def work(case):
    op = case["op"]
    if op == "attend":
        kv, new = _lengths(case)
        row = case["kv"] // 2 + case["kv"] // 16 + 2 * case["rope"] + 1
        w = case["kv"] + case["rope"]
        rows = sum(new) * case["H"]
        keys = sum(sum(k - m + j + 1 for j in range(m)) for k, m in zip(kv, new)) * case["H"]
        return {"bytes": sum(kv) * row + rows * 2 * (w + case["kv"]) + 4 * sum(-(-k // case["page"]) for k in kv),
                "flops": 2 * keys * (w + case["kv"])}
    if op == "store":
        row = case["kv"] // 2 + case["kv"] // 16 + 2 * case["rope"] + 1
        w = case["kv"] + case["rope"]
        return {"bytes": case["N"] * (w * (4 if case["x"] == "f32" else 2) + 2 * row + 4 * w + 8),
                "flops": case["N"] * w * 4}
    if op == "plan":
        ln, new = _plan_lengths(case)
        pages = sum(-(-(a + b) // case["page"]) - -(-a // case["page"]) for a, b in zip(ln, new))
        return {"bytes": 8 * sum(new) + 4 * 4 * pages + 4 * 10 * case["B"], "flops": 0}
    if op == "softmax":
        return {"bytes": 8 * case["rows"] * case["V"], "flops": 4 * case["rows"] * case["V"]}
    rows = 2 if case["probs"] else 1
    return {"bytes": case["B"] * case["V"] * 4 * rows, "flops": 3 * case["B"] * case["V"]}


# --------------------------------------------------------------------- the 4-bit row ----
def _sections(kv, rope, page):
    a = page * (kv // 2)
    b = a + page * (kv // 16)
    c = b + page * 2 * rope
    return a, b, c, c + page


def _views(pool, kv, rope, page):
    a, b, c, d = _sections(kv, rope, page)
    n = pool.shape[0]
    return (pool[:, :a].view(n, page, kv // 2), pool[:, a:b].view(n, page, kv // 16),
            pool[:, b:c].view(torch.float16).view(n, page, rope), pool[:, c:d])


def _pow2(k):
    """2^k in fp32 for -126 <= k <= 127, by its bits (a pow() may be an ulp off)."""
    return ((k.int() + 127) << 23).view(torch.float32)


def _quantise(x, kv):
    """Rows of fp32 as (codes, scales, rope, exponent byte); every step is exact in fp32 but the
    two roundings that define the format."""
    lat, rope = x[:, :kv], x[:, kv:]
    ml, el = torch.frexp(lat.abs().amax(1))
    mr, er = torch.frexp(rope.abs().amax(1))
    kl = torch.where(ml > 0, el - 12 + (ml > 0.65625).int(), -100)
    kr = torch.where(mr > 0, er - 16 + (mr > 0.5).int(), -100)
    k = torch.maximum(kl, kr).clamp(min=-100)
    bad = ~torch.isfinite(x).all(1)
    k = torch.where(bad, 0, k)
    x = torch.where(bad[:, None], 0.0, x)
    # two factors: 2^-k alone leaves the range of fp32 for the smallest k
    half = torch.div(-k, 2, rounding_mode="floor")
    y = x * _pow2(half)[:, None] * _pow2(-k - half)[:, None]
    blk = y[:, :kv].reshape(-1, kv // 16, 16)
    scale = (blk.abs().amax(2) / 6.0).to(torch.float8_e4m3fn)
    s = scale.float()[:, :, None]
    a = blk.abs()
    code = ((a > 0.25 * s).int() + (a >= 0.75 * s).int() + (a > 1.25 * s).int() + (a >= 1.75 * s).int()
            + (a > 2.5 * s).int() + (a >= 3.5 * s).int() + (a > 5.0 * s).int())
    code = torch.where(s > 0, code, 0) | (torch.signbit(blk).int() << 3)
    code = code.reshape(-1, kv // 2, 2)
    packed = (code[:, :, 0] | (code[:, :, 1] << 4)).to(torch.uint8)
    return packed, scale.view(torch.uint8), y[:, kv:].to(torch.float16), torch.where(bad, 255, k + 127).to(torch.uint8)


def _values(codes, scales, rope, exps, lut):
    """What stored rows stand for, fp32 [rows][kv + rope]; lut: the two values of every byte."""
    n = codes.shape[0]
    lat = lut[codes.int()].reshape(n, -1, 16) * scales.view(torch.float8_e4m3fn).float()[:, :, None]
    unit = torch.where(exps == 255, float("nan"), _pow2(exps.clamp(1, 254).int() - 127))
    return torch.cat([lat.reshape(n, -1), rope.float()], 1) * unit[:, None]


def _lut(dev):
    t = torch.tensor(E2M1, device=dev)
    b = torch.arange(256, device=dev)
    return torch.stack([t[b & 15], t[b >> 4]], 1)


# ------------------------------------------------------------------------- the inputs ----
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 2654435761 % (1 << 31) + 17)
    op = case["op"]
    st = {"case": dict(case), "op": op}

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    if op == "attend":
        kv, new = _lengths(case)
        B, H, W, page = case["B"], case["H"], case["kv"] + case["rope"], case["page"]
        need = [-(-k // page) for k in kv]
        max_pages = max(need) + 1
        n_pages = sum(need) + 8
        pages = torch.randperm(n_pages, generator=g, device=dev).int()
        table = torch.full((B, max_pages), -1, dtype=torch.int32, device=dev)
        at = 0
        for b in range(B):
            table[b, :need[b]] = pages[at:at + need[b]]
            at += need[b]
        size = _sections(case["kv"], case["rope"], page)[3]
        pool = torch.empty(n_pages, size, dtype=torch.uint8, device=dev)
        views = _views(pool, case["kv"], case["rope"], page)
        step = max(1, (1 << 16) // page)
        for p in range(0, n_pages, step):         # normalised latents and rotated keys: N(0, 1)
            m = min(step, n_pages - p)
            x = torch.randn(m * page, W, generator=g, device=dev)
            for v, t in zip(views, _quantise(x, case["kv"])):
                v[p:p + m] = t.reshape(v[p:p + m].shape)
        N = sum(new)
        st.update(pool=pool, table=table, N=N, q=torch.randn(N, H, W, generator=g, device=dev).bfloat16(),
                  row_start=ints(np.concatenate([[0], np.cumsum(new)]).tolist()), kv_len=ints(kv),
                  out=torch.empty(N, H, case["kv"], dtype=torch.bfloat16, device=dev), max_kv=max(kv),
                  max_new=max(new), lut=_lut(dev), scale=1.0 / math.sqrt(HEAD))
    elif op == "store":
        N, W, page = case["N"], case["kv"] + case["rope"], case["page"]
        n_pages = -(-N // page) + 8
        x = torch.randn(N, W, generator=g, device=dev) * torch.exp(
            torch.randn(N, 1, generator=g, device=dev))
        # the slots of a plan: whole pages in any order, and a padded row in sixteen of a batch
        slots = (torch.randperm(n_pages, generator=g, device=dev)[:, None] * page
                 + torch.arange(page, device=dev)).reshape(-1)[:N].int()
        slots[15::16] = -1
        size = _sections(case["kv"], case["rope"], page)[3]
        st.update(x=x if case["x"] == "f32" else x.bfloat16(), slots=slots, lut=_lut(dev),
                  pool=torch.zeros(n_pages, size, dtype=torch.uint8, device=dev),
                  out=torch.zeros(N, W, dtype=torch.float32, device=dev))
    elif op == "plan":
        ln, new = _plan_lengths(case)
        B, page = case["B"], case["page"]
        held = [-(-a // page) for a in ln]
        most = [-(-(a + b) // page) for a, b in zip(ln, new)]
        n_pages = sum(most) + 16
        perm = torch.randperm(n_pages, generator=g, device=dev).int()
        table = torch.full((B, max(most) + 1), -1, dtype=torch.int32, device=dev)
        at = 0
        for b in range(B):
            table[b, :held[b]] = perm[at:at + held[b]]
            at += held[b]
        free = torch.full((n_pages,), -1, dtype=torch.int32, device=dev)
        free[:n_pages - at] = perm[at:]
        N = sum(new) + 5                                # a step's slots are padded to a capacity
        out = [[torch.zeros(B + 1, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev),
                torch.zeros(N, dtype=torch.int32, device=dev), torch.zeros(N, dtype=torch.int32, device=dev),
                torch.zeros(1, dtype=torch.int32, device=dev)] for _ in range(2)]
        st.update(table=table, held=ints(held), free=free, n_free=ints([n_pages - at]), len=ints(ln),
                  new=ints(new), none=ints([0] * B), n_pages=n_pages, N=N, out=out)
    else:
        V = case["V"]
        if op == "softmax":
            rows = case["rows"]
            # peaked logits, a few of them masked by the type's lowest value or minus infinity
            x = torch.randn(rows, V, generator=g, device=dev) * 3.0
            x[:, 5::1009] = float("-inf")
            x[:, 6::1013] = torch.finfo(torch.float32).min
            temp = torch.rand(rows, generator=g, device=dev) * 1.2 + 0.3
            if case["greedy"]:
                temp[::3] = 0.0
            st.update(x=x, temp=temp, out=torch.empty_like(x))
        else:
            B, K = case["B"], case["K"]
            zt = torch.randn(B, K + 1, V, generator=g, device=dev) * 3.0
            zq = zt[:, :K] + torch.randn(B, K, V, generator=g, device=dev) * 0.7
            target = _softmax(zt, None)
            draft = _softmax(zq, None)
            u = torch.rand(B, K, generator=g, device=dev)
            # a draft is drawn from its own probabilities
            ids = torch.multinomial(draft.reshape(B * K, V), 1, generator=g).reshape(B, K).int()
            nd = torch.full((B,), K, dtype=torch.int32, device=dev)
            nd[2::5] = max(K - 1, 0)
            st.update(target=target, draft=draft if case["probs"] else None, ids=ids, u=u, n_draft=nd,
                      us=torch.rand(B, generator=g, device=dev),
                      tokens=torch.empty(B, K + 1, dtype=torch.int32, device=dev),
                      n_accept=torch.empty(B, dtype=torch.int32, device=dev))
    return st


# -------------------------------------------------------------------- the plain forms ----
def _attend(st):
    """softmax(scale q . row + causal mask) times the rows' latent parts, over padded sequences."""
    c = st["case"]
    kv, page, H, B = c["kv"], c["page"], c["H"], c["B"]
    n_tab = -(-st["max_kv"] // page)
    P = n_tab * page
    pages = st["table"][:, :n_tab].long().clamp(min=0).reshape(-1)
    rows = [v[pages].reshape(B * P, *v.shape[2:]) for v in _views(st["pool"], kv, c["rope"], page)]
    row = _values(*rows, st["lut"]).reshape(B, P, -1)
    at = torch.arange(P, device=row.device)
    here = at[None] < st["kv_len"][:, None]
    row = torch.where(here[:, :, None], row, 0.0)
    start, M = st["row_start"].long(), st["max_new"]
    j = torch.arange(M, device=row.device)
    new = start[1:] - start[:-1]
    src = (start[:-1, None] + j).clamp(max=st["N"] - 1)
    q = st["q"][src].float()                                        # [B][M][H][W]
    s = torch.matmul(q.reshape(B, M * H, -1), row.transpose(1, 2)).reshape(B, M, H, P) * st["scale"]
    last = st["kv_len"][:, None] - new[:, None] + j                 # the last position a row sees
    s = torch.where((at <= last[:, :, None])[:, :, None], s, float("-inf"))
    top = s.amax(3, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(3, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    o = torch.matmul(p.reshape(B, M * H, P), row[:, :, :kv]).reshape(B, M, H, kv)
    t = torch.arange(st["N"], device=row.device)
    b = torch.searchsorted(start[1:].contiguous(), t, right=True)
    return o[b, t - start[b]].bfloat16()


def _store(st):
    c = st["case"]
    kv, rope, page = c["kv"], c["rope"], c["page"]
    slots = st["slots"].long()
    keep = slots >= 0
    # a padded row goes to its own spare place behind the pool's rows
    n = st["pool"].shape[0] * page
    views = _views(st["pool"], kv, rope, page)
    got = []
    for v, t in zip(views, _quantise(st["x"].float(), kv)):
        flat = v.reshape(n, -1)
        old = flat[slots.clamp(min=0)]
        t = torch.where(keep[:, None], t.reshape(len(slots), -1), old)
        spare = torch.cat([flat, flat.new_zeros(1, flat.shape[1])])
        spare[torch.where(keep, slots, n)] = t
        v.copy_(spare[:n].reshape(v.shape))
        got.append(v.reshape(n, -1)[slots.clamp(min=0)].reshape(len(slots), *v.shape[2:]))
    return torch.where(keep[:, None], _values(*got, st["lut"]), 0.0)


def _plan(st, ln, new):
    c = st["case"]
    page, dev = c["page"], ln.device
    table, held, free, n_free = st["table"], st["held"].long(), st["free"], st["n_free"].long()
    N, n_pages = st["N"], st["n_pages"]
    total = (ln + new).long()
    need = (total + page - 1) // page
    grow, drop = (need - held).clamp(min=0), (held - need).clamp(min=0)
    ok = (need.max() <= table.shape[1]) & (grow.sum() <= n_free[0] + drop.sum()) & (new.long().sum() <= N)
    col = torch.arange(table.shape[1], device=dev)[None]
    # given back: from the last page of the last request on, so that what was taken last lies
    # deepest and the stack is as it was before it was taken
    out = ok & (col >= need[:, None]) & (col < held[:, None])
    rank = (drop.cumsum(0) - drop)[:, None] + col - need[:, None]
    spare = torch.cat([free, free.new_zeros(1)])
    spare[torch.where(out, n_free + drop.sum() - 1 - rank, n_pages)] = table
    have = n_free + drop.sum()
    into = ok & (col >= held[:, None]) & (col < need[:, None])
    rank = (grow.cumsum(0) - grow)[:, None] + col - held[:, None]
    took = spare[torch.where(into, have - 1 - rank, 0)]
    table.copy_(torch.where(into, took, torch.where(out, -1, table)))
    free.copy_(spare[:n_pages])
    st["held"].copy_(torch.where(ok, need, held))
    st["n_free"].copy_(torch.where(ok, have - grow.sum(), n_free))
    start = torch.cat([new.new_zeros(1), new.cumsum(0)]).long() * ok
    t = torch.arange(N, device=dev)
    b = torch.searchsorted(start[1:].contiguous(), t, right=True).clamp(max=len(ln) - 1)
    inside = t < start[-1]
    pos = ln.long()[b] + t - start[b]
    slot = table[b, (pos // page).clamp(0, table.shape[1] - 1)].long() * page + pos % page
    return [start.int(), (total * ok).int(), torch.where(inside, pos, -1).int(), torch.where(inside, slot, -1).int(),
            torch.where(ok, 0, 1).int().reshape(1)]


def _softmax(x, temp):
    """exp((x - max) / temp) over its sum; a temperature of 0 is all on the first maximum."""
    top = x.amax(-1, keepdim=True)
    t = 1.0 if temp is None else torch.where(temp > 0, temp, 1.0)[:, None]
    e = torch.exp((x - top) / t)
    p = e / e.sum(-1, keepdim=True)
    if temp is None:
        return p
    at = torch.arange(x.shape[-1], device=x.device)
    first = torch.where(x == top, at, x.shape[-1]).amin(-1, keepdim=True)
    return torch.where(temp[:, None] > 0, p, (at == first).float())


def _verify(st):
    """Draft i is kept while u_i q_i(d_i) < p_i(d_i); behind the last one kept, a token is drawn
    from max(p - q, 0) (from p where all were kept) in 2^-44 steps, so that sums are exact."""
    p, q, ids, nd = st["target"], st["draft"], st["ids"].long(), st["n_draft"].long()
    B, K, V = p.shape[0], p.shape[1] - 1, p.shape[2]
    pd = p[:, :K].gather(2, ids[:, :, None])[:, :, 0].double()
    qd = q.gather(2, ids[:, :, None])[:, :, 0].double() if q is not None else torch.ones_like(pd)
    i = torch.arange(K + 1, device=p.device)
    kept = (st["u"].double() * qd < pd) & (i[None, :K] < nd[:, None])
    n = kept.long().cumprod(1).sum(1)
    b = torch.arange(B, device=p.device)
    r = p[b, n]
    row = n.clamp(max=K - 1)
    if q is not None:
        less = q[b, row]
    else:
        less = (torch.arange(V, device=p.device) == ids[b, row][:, None]).float()
    cut = (r - less).clamp(min=0.0)
    w = (torch.where((n < nd)[:, None], cut, r).double() * 2.0 ** 44).floor().long()
    whole = (r.double() * 2.0 ** 44).floor().long()
    w = torch.where(w.sum(1, keepdim=True) > 0, w, whole)
    run = w.cumsum(1)
    total = run[:, -1:]
    t = torch.minimum((st["us"].double()[:, None] * total.double()).floor().long(), total - 1)
    token = torch.searchsorted(run, t, right=True)[:, 0]
    token = torch.where(total[:, 0] > 0, token, -1)
    wide = torch.cat([ids, ids[:, :1]], 1)
    tokens = torch.where(i[None] < n[:, None], wide, torch.where(i[None] == n[:, None], token[:, None], -1))
    return [tokens.int(), n.int()]


# ------------------------------------------------------------------------ the library ----
_k3 = None


def _lib():
    global _k3
    if _k3 is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kimi-k3-in-c_b200"))
        import k3cuda
        lib = k3cuda.init(torch.cuda.current_device())
        k3cuda.check(lib.k3d_set_stream(torch.cuda.current_stream().cuda_stream), "k3d_set_stream")
        _k3 = k3cuda
    return _k3


def _calls(k3, st):
    """The library calls of one pass with their arguments: the addresses, sizes and workspace that a
    serving program fixes when it sets its buffers up, and what the pass returns."""
    lib, op, c = k3.load(), st["op"], st["case"]

    def at(t):
        return None if t is None else t.data_ptr()

    if op in ("attend", "store"):
        shape = k3.K3dCache4(c["kv"], c["rope"], c["page"], st["pool"].shape[0])
    if op == "attend":
        n = lib.k3d_mla_attend4_ws_bytes(shape, c["B"], st["N"], c["H"])
        st["ws"] = torch.empty(n, dtype=torch.uint8, device=st["q"].device)
        return [(lib.k3d_mla_attend4, (
            at(st["out"]), k3.K3D_DT_BF16, at(st["q"]), k3.K3D_DT_BF16, shape, at(st["pool"]), at(st["table"]),
            st["table"].shape[1], at(st["row_start"]), at(st["kv_len"]), c["B"], st["N"], c["H"], st["scale"],
            at(st["ws"]), n))], st["out"]
    if op == "store":
        W, x = c["kv"] + c["rope"], k3.K3D_DT_F32 if c["x"] == "f32" else k3.K3D_DT_BF16
        return [(lib.k3d_cache4_store, (shape, at(st["pool"]), at(st["x"]), x, W, at(st["slots"]), c["N"])),
                (lib.k3d_cache4_load, (shape, at(st["pool"]), at(st["out"]), k3.K3D_DT_F32, W, at(st["slots"]),
                                       c["N"]))], st["out"]
    if op == "plan":
        pages = k3.K3dPages(c["page"], st["n_pages"], st["table"].shape[1], at(st["table"]), at(st["held"]),
                            at(st["free"]), at(st["n_free"]))
        return [(lib.k3d_page_plan, (pages, at(st["len"]), at(new), c["B"], st["N"], *(at(t) for t in out)))
                for new, out in ((st["new"], st["out"][0]), (st["none"], st["out"][1]))], [
                    *st["out"], st["table"], st["held"], st["free"], st["n_free"]]
    if op == "softmax":
        return [(lib.k3d_logits_softmax, (at(st["out"]), at(st["x"]), at(st["temp"]), c["rows"], c["V"]))], st["out"]
    return [(lib.k3d_spec_verify, (
        at(st["tokens"]), at(st["n_accept"]), at(st["target"]), at(st["draft"]), at(st["ids"]), at(st["n_draft"]),
        at(st["u"]), at(st["us"]), c["B"], c["K"], c["V"]))], [st["tokens"], st["n_accept"]]


def _run_own(st):
    k3 = _lib()
    if "calls" not in st:
        st["calls"] = _calls(k3, st)
    calls, out = st["calls"]
    for f, a in calls:
        k3.check(f(*a), f.__name__)
    return out


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "attend":
        return _attend(state)
    if op == "store":
        return _store(state)
    if op == "plan":
        first = _plan(state, state["len"], state["new"])
        second = _plan(state, state["len"], state["none"])
        return [first, second, state["table"], state["held"], state["free"], state["n_free"]]
    if op == "softmax":
        return _softmax(state["x"], state["temp"])
    return _verify(state)


# ------------------------------------------------------------------- in 64 bits, apart ----
def _two(e):
    """2^e in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _bits(codes, scales, rope, exps):
    """The rows' values in 64 bits, from the fields of each number."""
    def small(v, man, bias):                     # a float of `man` mantissa bits, sign left out
        e, m = v >> man, v & ((1 << man) - 1)
        e, m = e.double(), m.double() / (1 << man)
        return torch.where(e > 0, (1 + m) * _two(e - bias), m * 2.0 ** (1.0 - bias))
    c = codes.long()
    c = torch.stack([c & 15, c >> 4], -1).reshape(c.shape[0], -1)
    v = small(c & 7, 1, 1) * (1.0 - 2.0 * (c >> 3).double())
    s = small(scales.long() & 127, 3, 7)
    v = v * s.repeat_interleave(16, 1)
    unit = _two(exps.long() - 127)
    unit[exps == 255] = float("nan")
    return torch.cat([v, rope.double()], 1) * unit[:, None]


def exact(case, seed):
    op = case["op"]
    if op not in ("attend", "store", "softmax"):
        return None                              # whole numbers
    st = prepare(case, seed)
    if op == "softmax":
        rows = []
        for x, t in zip(st["x"], st["temp"].tolist()):
            x = x.double()
            if t > 0:
                rows.append(torch.softmax(x / t, 0))
            else:
                rows.append(torch.zeros_like(x).index_fill_(0, x.argmax(), 1.0))
        return torch.stack(rows)
    kv, page = case["kv"], case["page"]
    if op == "store":
        x = st["x"].double()
        al, ar = x[:, :kv].abs().amax(1), x[:, kv:].abs().amax(1)
        e = torch.maximum(torch.ceil(torch.log2(al / 2688)), torch.ceil(torch.log2(ar / 32768)))
        y = x / _two(e)[:, None]
        b = y[:, :kv].reshape(len(x), -1, 16)
        s = (b.abs().amax(2, keepdim=True) / 6).float().to(torch.float8_e4m3fn).double()
        grid = torch.tensor(E2M1[:8], device=x.device, dtype=torch.float64)
        far = (b.abs()[..., None] / s[..., None] - grid).abs()
        # the nearest of the eight; of two as near, the even code
        near = far.amin(-1, keepdim=True)
        odd = torch.arange(8, device=x.device) % 2
        pick = torch.where(far == near, odd, 2).argmin(-1)
        lat = grid[pick] * torch.sign(b) * s
        out = torch.cat([lat.reshape(len(x), -1), y[:, kv:].half().double()], 1) * _two(e)[:, None]
        out[st["slots"] < 0] = 0.0
        return out
    out = torch.zeros(st["N"], case["H"], kv, dtype=torch.float64, device=st["q"].device)
    views = _views(st["pool"], kv, case["rope"], page)
    start, lens = st["row_start"].tolist(), st["kv_len"].tolist()
    for b, L in enumerate(lens):
        n_tab = -(-L // page)
        pages = st["table"][b, :n_tab].long()
        rows = _bits(*(v[pages].reshape(n_tab * page, *v.shape[2:])[:L] for v in views))
        n = start[b + 1] - start[b]
        for j in range(n):
            seen = rows[:L - n + j + 1]
            p = torch.softmax(st["q"][start[b] + j].double() @ seen.T * st["scale"], 1)
            out[start[b] + j] = p @ seen[:, :kv]
    return out
