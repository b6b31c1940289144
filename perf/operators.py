"""The paged KV-cache operators, case by case, for timing and comparison.

Each case is one call of one operator of ``ddq_b200.paged``.  ``run`` computes
it in plain torch operations (``own`` false) or through the library (``own``
true) on what ``prepare`` made; ``exact`` gives the definition in 64 bits.

  plan     block table, slots and positions of a step from the request lengths
  write    rotary embedding of q and k, k and v into their pages
  prefill  attention of the new tokens of ragged requests over their pages
           (causal, optional tanh cap, distance bias, bidirectional prefix)
  decode   attention of one token per sequence over a shared prefix and the
           sequence's own pages
"""
import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 64 running sequences: one new token each
        {"name": "plan_step_64", "op": "plan", "requests": 64, "new_lo": 1, "new_hi": 1,
         "cached_hi": 4096, "page": 16, "prefix": 0, "pad": 0},
        # a step of a busy server: decodes and prompt chunks mixed, a padded token count
        {"name": "plan_mixed_512", "op": "plan", "requests": 512, "new_lo": 1, "new_hi": 255,
         "cached_hi": 2048, "page": 16, "prefix": 512, "pad": 317},
        # the cache write of one decode step of 64 sequences
        {"name": "write_step_64", "op": "write", "tokens": 64, "hq": 14, "hkv": 2, "d": 64,
         "page": 16, "dtype": "fp16", "max_pos": 32768},
        # the cache write of a large batch of prompts
        {"name": "write_prompts_32k", "op": "write", "tokens": 32768, "hq": 32, "hkv": 8,
         "d": 128, "page": 64, "dtype": "bf16", "max_pos": 32768},
        # three short prompts, one of them a single token: latency
        {"name": "prefill_short", "op": "prefill", "new": "1 37 200", "cached": "0 0 0",
         "hq": 14, "hkv": 2, "d": 64, "page": 16, "dtype": "fp16", "cap": 0.0, "bias": False,
         "bidir": ""},
        # eight prompts of 512 tokens, the sizes of the batch prefill here
        {"name": "prefill_8x512", "op": "prefill", "new": "512 512 512 512 512 512 512 512",
         "cached": "0 0 0 0 0 0 0 0",
         "hq": 14, "hkv": 2, "d": 64, "page": 64, "dtype": "fp16", "cap": 0.0, "bias": False,
         "bidir": ""},
        # packed documents of very different lengths, capped scores, a distance
        # bias and a bidirectional prefix
        {"name": "prefill_docs_masks", "op": "prefill",
         "new": "1 2500 17 640 129 1023 333 64 1800 5 911 256",
         "cached": "700 0 33 128 1 0 950 4000 77 2047 0 512",
         "hq": 16, "hkv": 2, "d": 128, "page": 32, "dtype": "bf16", "cap": 30.0, "bias": True,
         "bidir": "8 500 50 0 130 1023 1000 4010 0 1 911 300"},
        # the last chunk of a long prompt: few rows, a long axis
        {"name": "prefill_chunk_32k", "op": "prefill", "new": "509", "cached": "32259",
         "hq": 14, "hkv": 2, "d": 64, "page": 64, "dtype": "fp16", "cap": 0.0, "bias": False,
         "bidir": ""},
        # four prompts of 4096 tokens, wide heads: the largest
        {"name": "prefill_4x4096", "op": "prefill", "new": "4096 4096 4096 4096",
         "cached": "0 0 0 0",
         "hq": 32, "hkv": 8, "d": 128, "page": 64, "dtype": "fp16", "cap": 0.0, "bias": False,
         "bidir": ""},
        # a decode step of 64 sequences behind one 512-token prompt, up to 256 tokens each
        {"name": "decode_64_prefix512", "op": "decode", "batch": 64, "prefix": 512, "own_lo": 1,
         "own_hi": 256, "hq": 14, "hkv": 2, "d": 64, "page": 16, "dtype": "fp16", "cap": 0.0,
         "bias": False},
        # a decode step of ragged sequences with nothing in common, capped and biased
        {"name": "decode_40_ragged", "op": "decode", "batch": 40, "prefix": 0, "own_lo": 1,
         "own_hi": 32768, "hq": 32, "hkv": 8, "d": 128, "page": 16, "dtype": "bf16",
         "cap": 50.0, "bias": True},
        # a large batch behind a long shared document that ends inside a page
        {"name": "decode_256_prefix32k", "op": "decode", "batch": 256, "prefix": 32001,
         "own_lo": 0, "own_hi": 511, "hq": 32, "hkv": 8, "d": 128, "page": 64, "dtype": "fp16",
         "cap": 0.0, "bias": False},
    ]


def _text(xs):
    return " ".join(str(x) for x in xs)


def _ints(case, key):
    return [int(x) for x in case[key].split()]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "prefill", "decode"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        return {"op": op, "requests": _log_int(rng, 1, 512), "new_lo": rng.choice([0, 1]),
                "new_hi": _log_int(rng, 1, 255), "cached_hi": _log_int(rng, 1, 4096),
                "page": page, "prefix": rng.choice([0, _log_int(rng, 1, 4096)]),
                "pad": rng.randrange(0, 400)}
    hkv = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 7, 8])
    d = rng.choice([64, 128])
    if g * hkv > 32:
        g = 4
    base = {"op": op, "hq": g * hkv, "hkv": hkv, "d": d, "page": page,
            "dtype": rng.choice(["fp16", "bf16"])}
    if op == "write":
        base.update(tokens=_log_int(rng, 1, 32768), max_pos=32768)
        return base
    base.update(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.4)
    if op == "decode":
        base.update(batch=_log_int(rng, 1, 256), own_lo=rng.choice([0, 1]))
        prefix = rng.choice([0, _log_int(rng, 1, 32001)])
        base.update(prefix=prefix,
                    own_hi=_log_int(rng, 1, 4096 if base["batch"] <= 64 else 512))
        return base
    n = _log_int(rng, 1, 16)
    left = 16384
    new, cached, bidir = [], [], []
    masked = rng.random() < 0.3
    for _ in range(n):
        m = _log_int(rng, 1, max(1, min(4096, left // n)))
        c = rng.choice([0, 0, _log_int(rng, 1, 4096)])
        new.append(m)
        cached.append(c)
        bidir.append(rng.randrange(0, m + c + 1))
    base.update(new=_text(new), cached=_text(cached), bidir=_text(bidir) if masked else "")
    return base


# ---------------------------------------------------------------- the lengths
def _plan_lens(case):
    rng = random.Random(case["requests"] * 7919 + case["cached_hi"])
    cached = [rng.randint(0, case["cached_hi"]) for _ in range(case["requests"])]
    new = [rng.randint(case["new_lo"], max(case["new_lo"], case["new_hi"]))
           for _ in range(case["requests"])]
    return cached, new


def _own_lens(case):
    """The sequences' own tokens: most of them short, a few long."""
    rng = random.Random(case["batch"] * 104729 + case["own_hi"])
    lo, hi = case["own_lo"], max(case["own_lo"], case["own_hi"])
    lens = [lo + int((hi - lo) * rng.random() ** 2) for _ in range(case["batch"])]
    lens[0] = hi
    return lens


def _pages(n, page):
    return -(-n // page)


# ------------------------------------------------------------------- prepare
def _table(lens, page, gen, extra, device):
    """Block table of the requests over randomly ordered pages; unused entries
    hold -1.  Returns it with the number of pages of the pool."""
    need = [_pages(n, page) for n in lens]
    pool = sum(need) + extra
    perm = torch.randperm(max(pool, 1), generator=gen, device=device).to(torch.int32)
    width = max(1, max(need) if need else 1)
    rows = torch.full((len(lens), width), -1, dtype=torch.int32, device=device)
    at = 0
    for r, k in enumerate(need):
        rows[r, :k] = perm[at:at + k]
        at += k
    return rows, perm[at:], max(pool, 1)


def _cache(pool, case, gen, device):
    dt = _DTYPES[case["dtype"]]
    shape = (pool, case["hkv"], case["page"], case["d"])
    k = torch.randn(shape, generator=gen, device=device, dtype=torch.float32).to(dt)
    v = torch.randn(shape, generator=gen, device=device, dtype=torch.float32).to(dt)
    return k, v


def _slopes(hq, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32,
                        device=device)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    st = {"case": case}
    page = case["page"]
    if case["op"] == "plan":
        cached, new = _plan_lens(case)
        need = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        held, free, _ = _table(cached, page, gen, need + 64, dev)
        width = max(1, max(_pages(c + n, page) for c, n in zip(cached, new)))
        table = torch.full((len(cached), width), -1, dtype=torch.int32, device=dev)
        w = min(width, held.shape[1])
        table[:, :w] = held[:, :w]
        st.update(cached=torch.tensor(cached, dtype=torch.int32, device=dev),
                  new=torch.tensor(new, dtype=torch.int32, device=dev), table=table, free=free,
                  head=torch.tensor([seed % 50], dtype=torch.int32, device=dev),
                  tokens=sum(new) + case["pad"])
        return st
    hq, hkv, d, dt = case["hq"], case["hkv"], case["d"], _DTYPES[case["dtype"]]
    if case["op"] == "write":
        T = case["tokens"]
        pool = _pages(T, page) + 3
        k, v = _cache(pool, case, gen, dev)
        slots = torch.randperm(pool * page, generator=gen, device=dev)[:T].to(torch.int64)
        slots[torch.rand(T, generator=gen, device=dev) < 0.01] = -1     # padded rows
        pos = torch.randint(0, case["max_pos"], (T,), generator=gen, device=dev)
        inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, dtype=torch.float64, device=dev) / d))
        ang = torch.arange(case["max_pos"], dtype=torch.float64, device=dev)[:, None] * inv
        emb = torch.cat([ang, ang], dim=-1)
        qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=gen, device=dev).to(dt)
        st.update(k=k, v=v, slots=slots, pos=pos, cos=emb.cos().float(), sin=emb.sin().float(),
                  qkv=qkv)
        return st
    slopes = _slopes(hq, dev) if case["bias"] else None
    if case["op"] == "prefill":
        new, bidir = _ints(case, "new"), _ints(case, "bidir")
        lens = [c + n for c, n in zip(_ints(case, "cached"), new)]
        table, _, pool = _table(lens, page, gen, 1, dev)
        k, v = _cache(pool, case, gen, dev)
        T = sum(new)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        st.update(k=k, v=v, table=table, slopes=slopes, cu_host=cu, lens_host=lens,
                  q=torch.randn(T, hq, d, generator=gen, device=dev).to(dt),
                  cu=torch.tensor(cu, dtype=torch.int32, device=dev),
                  lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                  bidir=torch.tensor(bidir, dtype=torch.int32, device=dev) if bidir else None)
        return st
    lens = _own_lens(case)
    prefix = case["prefix"]
    rows, _, pool = _table(lens + [prefix], page, gen, 1, dev)
    width = max(1, _pages(max(lens), page))
    k, v = _cache(pool, case, gen, dev)
    st.update(k=k, v=v, table=rows[:-1, :width].contiguous(), slopes=slopes, lens_host=lens,
              prefix_pages=rows[-1, :_pages(prefix, page)].contiguous() if prefix else None,
              q=torch.randn(len(lens), hq, d, generator=gen, device=dev).to(dt),
              lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    return st


# ----------------------------------------------------------------- plain form
def _plain_plan(st):
    page, T = st["case"]["page"], st["tokens"]
    cached, new, table, free = st["cached"].long(), st["new"].long(), st["table"], st["free"]
    R, width = table.shape
    lens = cached + new
    have = (cached + page - 1) // page
    need = (lens + page - 1) // page - have
    first = st["head"].long() + torch.cumsum(need, 0) - need
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=new.device), torch.cumsum(new, 0)])
    col = torch.arange(width, device=new.device)[None, :]
    idx = first[:, None] + col - have[:, None]
    taken = (col >= have[:, None]) & (col < (have + need)[:, None])
    fresh = torch.where(idx < free.numel(), free[idx.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(taken, fresh, table))
    t = torch.arange(T, device=new.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    real = t < cu[-1]
    s = seq.clamp(max=R - 1)
    p = cached[s] + t - cu[s]
    pg = table[s, (p // page).clamp(max=width - 1)].long()
    slots = torch.where(real & (pg >= 0), pg * page + p % page, -1)
    pos = torch.where(real, p + st["case"]["prefix"], 0)
    return (table, cu.to(torch.int32), lens.to(torch.int32), slots, pos,
            torch.where(real, seq, -1).to(torch.int32),
            (st["head"].long() + need.sum()).to(torch.int32))


def _plain_write(st):
    c = st["case"]
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    k, v, qkv = st["k"], st["v"], st["qkv"]
    T = qkv.shape[0]
    x = qkv[:, :(hq + hkv) * d].reshape(T, hq + hkv, d).float()
    cos, sin = st["cos"][st["pos"]][:, None], st["sin"][st["pos"]][:, None]
    rot = torch.cat([-x[..., d // 2:], x[..., :d // 2]], dim=-1)
    y = (x * cos + rot * sin).to(qkv.dtype)
    ok = st["slots"] >= 0
    pg, row = st["slots"][ok] // page, st["slots"][ok] % page
    k[pg, :, row] = y[ok, hq:]
    v[pg, :, row] = qkv[ok, (hq + hkv) * d:].reshape(-1, hkv, d)
    return y[:, :hq].contiguous(), k, v


def _gather(cache, pages, n):
    """The first n rows of a page list, [Hkv, n, D] in 32 bits."""
    x = cache[pages.long()].float()
    return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n]


def _plain_prefill(st):
    c = st["case"]
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    g, scale, cap = hq // hkv, d ** -0.5, c["cap"]
    out = torch.empty_like(st["q"])
    for r, n in enumerate(_ints(c, "new")):
        L, a = st["lens_host"][r], st["cu_host"][r]
        pages = st["table"][r, :_pages(L, page)]
        k, v = _gather(st["k"], pages, L), _gather(st["v"], pages, L)
        q = st["q"][a:a + n].float().reshape(n, hkv, g, d).permute(1, 2, 0, 3)
        s = torch.matmul(q.reshape(hkv, g * n, d), k.transpose(1, 2)).mul_(scale)
        s = s.reshape(hkv, g, n, L)
        if cap:
            s = cap * torch.tanh(s / cap)
        p = torch.arange(L - n, L, device=s.device)[:, None]
        j = torch.arange(L, device=s.device)[None, :]
        if st["slopes"] is not None:
            s = s - st["slopes"].reshape(hkv, g, 1, 1) * (p - j).abs().float()
        end = p + 1
        if st["bidir"] is not None:
            end = torch.maximum(end, st["bidir"][r].long())
        s.masked_fill_(j >= end, float("-inf"))
        s.sub_(s.amax(-1, keepdim=True)).exp_()
        l = s.sum(-1, keepdim=True)
        o = torch.matmul(s.reshape(hkv, g * n, L), v).reshape(hkv, g, n, d) / l
        out[a:a + n] = o.permute(2, 0, 1, 3).reshape(n, hq, d).to(out.dtype)
    return out


def _plain_decode(st):
    c = st["case"]
    hq, hkv, d, page, P = c["hq"], c["hkv"], c["d"], c["page"], c["prefix"]
    g, scale, cap = hq // hkv, d ** -0.5, c["cap"]
    B = st["q"].shape[0]
    q = st["q"].float().reshape(B, hkv, g, d)
    out = torch.empty_like(st["q"])

    def scores(x, pos, j):
        x = x * scale
        if cap:
            x = cap * torch.tanh(x / cap)
        if st["slopes"] is not None:
            x = x - st["slopes"].reshape(hkv, g, 1) * (pos - j).abs().float()
        return x
    if P:
        kp, vp = _gather(st["k"], st["prefix_pages"], P), _gather(st["v"], st["prefix_pages"], P)
        sp = torch.matmul(q.permute(1, 0, 2, 3).reshape(hkv, B * g, d), kp.transpose(1, 2))
        sp = sp.reshape(hkv, B, g, P)
        jp = torch.arange(P, device=q.device)
    acc, m, l = [], [], []
    for b, L in enumerate(st["lens_host"]):
        parts, vals = [], []
        pos = P + L - 1
        if P:
            parts.append(scores(sp[:, b], pos, jp))
            vals.append(vp)
        if L:
            pages = st["table"][b, :_pages(L, page)]
            k = _gather(st["k"], pages, L)
            j = P + torch.arange(L, device=q.device)
            parts.append(scores(torch.matmul(q[b], k.transpose(1, 2)), pos, j))
            vals.append(_gather(st["v"], pages, L))
        if not parts:
            out[b] = 0
            continue
        top = torch.stack([x.amax(-1) for x in parts]).amax(0)[..., None]
        es = [(x - top).exp() for x in parts]
        den = sum(e.sum(-1, keepdim=True) for e in es)
        num = sum(torch.matmul(e, v) for e, v in zip(es, vals))
        out[b] = (num / den).reshape(hq, d).to(out.dtype)
    return out


# ------------------------------------------------------------------------ run
def run(state):
    c = state["case"]
    op = c["op"]
    if not own:
        return {"plan": _plain_plan, "write": _plain_write, "prefill": _plain_prefill,
                "decode": _plain_decode}[op](state)
    from ddq_b200 import paged
    if op == "plan":
        p = paged.plan_step(state["cached"], state["new"], state["table"], state["free"],
                            c["page"], state["tokens"], free_head=state["head"],
                            prefix_len=c["prefix"])
        return (state["table"], p.cu_new, p.lens, p.slots, p.positions, p.seq_ids, p.free_head)
    if op == "write":
        q = paged.rope_kv_write(state["qkv"], state["k"], state["v"], state["cos"], state["sin"],
                                state["slots"], state["pos"], c["hq"], c["hkv"], c["d"])
        return q, state["k"], state["v"]
    if op == "prefill":
        return paged.prefill_attention(state["q"], state["k"], state["v"], state["table"],
                                       state["cu"], state["lens"], c["d"] ** -0.5,
                                       softcap=c["cap"], slopes=state["slopes"],
                                       bidir=state["bidir"])
    return paged.decode_attention(state["q"], state["k"], state["v"], state["table"],
                                  state["lens"], c["d"] ** -0.5,
                                  prefix_pages=state["prefix_pages"], prefix_len=c["prefix"],
                                  softcap=c["cap"], slopes=state["slopes"])


# ----------------------------------------------------------------------- work
def work(case):
    page = case["page"]
    if case["op"] == "plan":
        cached, new = _plan_lens(case)
        fresh = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        R, T = case["requests"], sum(new) + case["pad"]
        # lengths in, sums and lengths out; the fresh pages read and entered,
        # the partly filled page of each request looked up; three words a token
        return {"bytes": R * 8 + (R + 1) * 4 + R * 4 + fresh * 8 + R * 4 + T * 20, "flops": 0}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "write":
        T = case["tokens"]
        rows = min(T, case["max_pos"])
        return {"bytes": T * (hq + 2 * hkv) * d * 2 * 2 + rows * d * 8 + T * 16,
                "flops": T * (hq + hkv) * d * 3}
    if case["op"] == "prefill":
        pairs = keys = 0
        new, bidir = _ints(case, "new"), _ints(case, "bidir")
        for r, (n, c) in enumerate(zip(new, _ints(case, "cached"))):
            b = bidir[r] if bidir else 0
            L = n + c
            keys += L
            # row i attends max(c + i + 1, min(b, L)) keys
            b = min(b, L)
            low = max(0, min(n, b - c))            # rows whose end is b
            pairs += low * b + sum(range(c + low + 1, L + 1))
        T = sum(new)
        return {"bytes": T * hq * d * 4 + keys * hkv * d * 4, "flops": 4 * pairs * hq * d}
    lens = _own_lens(case)
    B, P = case["batch"], case["prefix"]
    return {"bytes": B * hq * d * 4 + (P + sum(lens)) * hkv * d * 4,
            "flops": 4 * (B * P + sum(lens)) * hq * d}


# ---------------------------------------------------------------------- exact
def _rows64(cache, pages, n, head):
    """Rows 0..n-1 of one key/value head, read page by page."""
    if n == 0:
        return torch.zeros(0, cache.shape[3], dtype=torch.float64, device=cache.device)
    sel = torch.index_select(cache[:, head], 0, pages.long())
    return sel.flatten(0, 1)[:n].double()


def _softmax64(q, k, v, pos, j, end, scale, cap, slope):
    """q [n, d]; k, v [m, d]; pos, end [n, 1]; j [m]: the definition, row by row."""
    z = (q @ k.T) * scale
    if cap:
        z = torch.tanh(z / cap) * cap
    if slope is not None:
        z = z - slope * (pos - j).abs().double()
    keep = j[None, :] < end
    z = torch.where(keep, z, torch.full_like(z, -math.inf))
    w = torch.softmax(z, dim=1) if z.shape[1] else z
    w = torch.where(keep.any(1, keepdim=True), w, torch.zeros_like(w))
    return w @ v


def exact(case, seed):
    st = prepare(case, seed)
    page = case["page"]
    if case["op"] == "plan":
        return None         # whole numbers
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "write":
        k, v = st["k"].double(), st["v"].double()
        qkv = st["qkv"].double()
        c, s = st["cos"].double()[st["pos"]], st["sin"].double()[st["pos"]]
        h = d // 2

        def turn(x):
            lo, hi = x[:, :h], x[:, h:]
            return torch.cat([lo * c[:, :h] - hi * s[:, :h], hi * c[:, h:] + lo * s[:, h:]], 1)
        q = torch.stack([turn(qkv[:, i * d:(i + 1) * d]) for i in range(hq)], 1)
        ok = (st["slots"] >= 0).nonzero()[:, 0]
        at = st["slots"][ok]
        for i in range(hkv):
            kr = turn(qkv[:, (hq + i) * d:(hq + i + 1) * d])
            vr = qkv[:, (hq + hkv + i) * d:(hq + hkv + i + 1) * d]
            k[at // page, i, at % page] = kr[ok]
            v[at // page, i, at % page] = vr[ok]
        return q, k, v
    scale, cap = 1.0 / math.sqrt(d), case["cap"]
    dev = st["q"].device
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=dev)
    if case["op"] == "prefill":
        bidir = _ints(case, "bidir")
        for r, n in enumerate(_ints(case, "new")):
            a, L = st["cu_host"][r], st["lens_host"][r]
            pages = st["table"][r, :_pages(L, page)]
            pos = (torch.arange(n, device=dev) + (L - n))[:, None]
            end = (pos + 1).clamp(min=min(bidir[r], L) if bidir else 0)
            j = torch.arange(L, device=dev)
            for h in range(hq):
                kk = _rows64(st["k"], pages, L, h * hkv // hq)
                vv = _rows64(st["v"], pages, L, h * hkv // hq)
                sl = st["slopes"][h].double() if st["slopes"] is not None else None
                out[a:a + n, h] = _softmax64(st["q"][a:a + n, h].double(), kk, vv, pos, j, end,
                                             scale, cap, sl)
        return out
    P = case["prefix"]
    g = hq // hkv
    for h in range(hkv):
        kp = vp = None
        if P:
            kp = _rows64(st["k"], st["prefix_pages"], P, h)
            vp = _rows64(st["v"], st["prefix_pages"], P, h)
        for b, L in enumerate(st["lens_host"]):
            if P + L == 0:
                continue
            pages = st["table"][b, :_pages(L, page)]
            kk, vv = _rows64(st["k"], pages, L, h), _rows64(st["v"], pages, L, h)
            if P:
                kk, vv = torch.cat([kp, kk]), torch.cat([vp, vv])
            j = torch.arange(P + L, device=dev)
            pos = torch.full((g, 1), P + L - 1, device=dev)
            sl = st["slopes"][h * g:(h + 1) * g].double()[:, None] \
                if st["slopes"] is not None else None
            out[b, h * g:(h + 1) * g] = _softmax64(
                st["q"][b, h * g:(h + 1) * g].double(), kk, vv, pos, j, pos + 1, scale, cap, sl)
    return out
