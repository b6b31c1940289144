"""Plain 64-bit forms of the paged KV-cache operators, on CPU or GPU tensors,
and the inputs of their tests (imported, not collected)."""
import math

import torch


def pages_for(n, ps):
    return -(-n // ps)


def make_table(lens, ps, gen, width=None, device="cuda", junk=None):
    """Block table over randomly ordered pages; unused entries hold `junk` (default
    a page number far outside any pool).  Returns (table, unused pages, pool)."""
    need = [pages_for(n, ps) for n in lens]
    pool = sum(need) + 3
    perm = torch.randperm(pool, generator=gen).to(torch.int32)
    width = width or max(1, max(need, default=1))
    table = torch.full((len(lens), width), 10 ** 8 if junk is None else junk, dtype=torch.int32)
    at = 0
    for r, k in enumerate(need):
        table[r, :k] = perm[at:at + k]
        at += k
    return table.to(device), perm[at:].to(device), pool


def make_pool(pool, hkv, ps, d, dtype, gen, layout="hnd", device="cuda"):
    """k and v pages [P, Hkv, ps, D]: dense ("hnd"), rows before heads ("nhd"),
    or k and v interleaved page by page in one buffer ("joint")."""
    def rnd(*shape):
        return torch.randn(*shape, generator=gen).to(dtype).to(device)
    if layout == "hnd":
        return rnd(pool, hkv, ps, d), rnd(pool, hkv, ps, d)
    if layout == "nhd":
        return (rnd(pool, ps, hkv, d).permute(0, 2, 1, 3),
                rnd(pool, ps, hkv, d).permute(0, 2, 1, 3))
    both = rnd(pool, 2, hkv, ps, d)
    return both[:, 0], both[:, 1]


def rows_of(cache, table_row, n, g):
    """Rows 0..n-1 of head g of a page list, in 64 bits."""
    ps = cache.shape[2]
    k = pages_for(n, ps)
    if n == 0:
        return torch.zeros(0, cache.shape[3], dtype=torch.float64, device=cache.device)
    return torch.cat([cache[int(p), g] for p in table_row[:k].tolist()], 0)[:n].double()


def prefill_reference(q, kp, vp, table, new, lens, scale, cap, slopes, bidir,
                      prefix_pages=None, P=0):
    u = torch.finfo(q.dtype).eps / 2
    T, hq, d = q.shape
    hkv = kp.shape[1]
    o = torch.zeros(T, hq, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    t = 0
    for r, n in enumerate(new):
        L = lens[r]
        for g in range(hkv):
            k, v = rows_of(kp, table[r], L, g), rows_of(vp, table[r], L, g)
            if P:
                k = torch.cat([rows_of(kp, prefix_pages, P, g), k])
                v = torch.cat([rows_of(vp, prefix_pages, P, g), v])
            for h in range(g * hq // hkv, (g + 1) * hq // hkv):
                sl = slopes[h].double() if slopes is not None else None
                oh, th = attend_many(q[t:t + n, h].double(), k, v,
                                     torch.arange(P + L - n, P + L, device=q.device),
                                     P + min(bidir[r], L) if bidir is not None else 0,
                                     scale, cap, sl, u)
                o[t:t + n, h], tol[t:t + n, h] = oh, th
        t += n
    return o, tol


def attend_many(q, k, v, pos, least, scale, cap, slope, u):
    """Rows q [n, D] at positions pos, attending the keys j < max(pos + 1, least),
    in 64 bits: the results and how far a kernel with weights of unit roundoff u
    may be off.

    o = sum w_j v_j / sum w_j.  With A = sum w_j |v_j| / sum w_j:
      rounding o once               u |o|
      rounding each weight once     u A   (the sum in the denominator is of unrounded ones)
      a weight below 2^-14 in fp16 is off by at most 2^-25:  n 2^-25 max|v| (the largest
      weight is at least 1, so the denominator is too)
      a score off by e gives a weight off by a factor exp(e), twice (above and below):
      2 e A.  The fp32 dot product is off by at most (D + 2) 2^-23 sum|q k| scale, the cap
      and the bias by 2^-20 max(|z|, cap) (a few roundings and the library's tanh, exp)
      fp32 sums over n keys in steps of 16:  (n / 16 + 8) 2^-22 A
    """
    n, d = q.shape
    L = k.shape[0]
    if n == 0 or L == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    end = (pos + 1).clamp(min=least)[:, None]
    z = (q @ k.T) * scale
    mag = (q.abs() @ k.abs().T).amax(1, keepdim=True) * abs(scale)
    if cap:
        z = cap * torch.tanh(z / cap)
    j = torch.arange(L, device=q.device)[None, :]
    if slope is not None:
        z = z - slope * (pos[:, None] - j).abs().double()
    keep = j < end
    some = keep.any(1, keepdim=True)
    zk = torch.where(keep, z, torch.full_like(z, -math.inf))
    top = torch.where(some, zk.amax(1, keepdim=True), torch.zeros_like(mag))
    w = torch.where(keep, torch.exp(zk - top), torch.zeros_like(z))
    w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    o, A = w @ v, w @ v.abs()
    zmax = torch.where(keep, z.abs(), torch.zeros_like(z)).amax(1, keepdim=True) \
        if slope is not None else torch.zeros_like(mag)
    spread = (top - torch.where(keep, z, top.expand_as(z)).amin(1, keepdim=True)).clamp(max=60.)
    e = (d + 2) * 2.0 ** -23 * mag + 2.0 ** -20 * torch.maximum(zmax, spread).clamp(min=max(1.0, cap))
    cnt = keep.sum(1, keepdim=True).double()
    tol = u * o.abs() + (u + 2 * e + (cnt / 16 + 8) * 2.0 ** -22) * A + \
        cnt * 2.0 ** -25 * v.abs().max()
    # the last rounding also rounds what the others left: (1 + u)
    return o, torch.where(some, (1 + u) * tol, torch.zeros_like(tol))


def decode_reference(q, kp, vp, table, lens, scale, prefix_pages, prefix_len, cap, slopes):
    u = torch.finfo(q.dtype).eps / 2
    B, hq, d = q.shape
    hkv = kp.shape[1]
    o = torch.zeros(B, hq, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for g in range(hkv):
        if prefix_len:
            k0, v0 = rows_of(kp, prefix_pages, prefix_len, g), rows_of(vp, prefix_pages, prefix_len, g)
        for b in range(B):
            k, v = rows_of(kp, table[b], lens[b], g), rows_of(vp, table[b], lens[b], g)
            if prefix_len:
                k, v = torch.cat([k0, k]), torch.cat([v0, v])
            p = prefix_len + lens[b] - 1
            for h in range(g * hq // hkv, (g + 1) * hq // hkv):
                sl = slopes[h].double() if slopes is not None else None
                oh, th = attend_many(q[b:b + 1, h].double(), k, v,
                                     torch.tensor([p], device=q.device), 0, scale, cap, sl, u)
                o[b, h], tol[b, h] = oh[0], th[0]
    return o, tol


def plan_reference(cached, new, table, free, ps, T, head, prefix):
    """The step plan, one token at a time (lists in, lists out; table in place)."""
    R, width = len(cached), len(table[0])
    cu, lens = [0], []
    slots, positions, seqs = [-1] * T, [0] * T, [-1] * T
    before = [list(row) for row in table]
    at = head
    for r in range(R):
        c, n = max(cached[r], 0), max(new[r], 0)
        have, want = pages_for(c, ps), pages_for(c + n, ps)
        row = list(before[r])
        for col in range(have, want):
            page = free[at] if 0 <= at < len(free) and free[at] >= 0 else -1
            at += 1
            if col < width:
                row[col] = page
        table[r] = row
        for i in range(n):
            t, p = cu[-1] + i, c + i
            if t >= T:
                break
            page = row[p // ps] if p // ps < width else -1
            slots[t] = page * ps + p % ps if page >= 0 else -1
            positions[t] = prefix + p
            seqs[t] = r
        cu.append(cu[-1] + n)
        lens.append(c + n)
    return table, cu, lens, slots, positions, seqs, at


def rope_reference(x, cos, sin):
    """x [T, H, D]; fp32 products and sum, rounded once to x's type."""
    h = x.shape[-1] // 2
    xf = x.float()
    rot = torch.cat([-xf[..., h:], xf[..., :h]], dim=-1)
    return (xf * cos[:, None] + rot * sin[:, None]).to(x.dtype)


def rope_tables(n, d, device="cuda"):
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    emb = torch.cat([ang, ang], dim=-1)
    return emb.cos().float().to(device), emb.sin().float().to(device)
