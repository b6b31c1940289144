"""The paged KV-cache operators on the GPU: the step plan (whole numbers, exact),
the rotary embedding with the page write (bit for bit the fp32 form), prompt and
decode attention against 64-bit forms with derived tolerances, their masks,
lengths, layouts, bad pages, streams and graphs, and a run of them together."""
import math
import os
import random
import subprocess
import sys

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
ERR_PAGE = 8


@pytest.fixture(autouse=True)
def no_device_error(cuda_device):
    """Every test starts and ends without a device error; the ones that cause
    one read it themselves."""
    device_error()
    yield
    assert device_error() == 0


def device_error():
    import ctypes
    from ddq_b200 import _lib
    code = ctypes.c_int(-1)
    assert _lib.load().ddq_device_error(ctypes.byref(code),
                                        torch.cuda.current_stream().cuda_stream) == 0
    return code.value


def ints(xs, dtype=torch.int32):
    return torch.tensor(list(xs), dtype=dtype, device="cuda")


def close(o, want, tol):
    if o.numel() == 0:
        return
    bad = (o.double() - want).abs() - tol
    assert torch.isfinite(o.float()).all()
    assert bad.max().item() <= 0, (bad.max().item(), tol.max().item(),
                                   (bad > 0).sum().item(), bad.numel())


# ------------------------------------------------------------------ step plan
@pytest.mark.parametrize("R,new_lo,new_hi,cached_hi,ps,prefix,pad,short,narrow", [
    (1, 1, 1, 0, 16, 0, 0, 0, 0), (1, 0, 0, 40, 16, 0, 3, 0, 0), (64, 1, 1, 900, 16, 0, 0, 0, 0),
    (7, 0, 50, 100, 32, 37, 11, 0, 0), (33, 1, 300, 700, 128, 512, 0, 0, 0),
    (513, 0, 9, 260, 16, 0, 700, 0, 0), (1025, 0, 40, 600, 64, 5, 1, 0, 0),
    (8192, 0, 3, 64, 256, 0, 9, 0, 0),
    (20, 1, 64, 100, 16, 0, 5, 9, 0),     # the free list runs out
    (20, 1, 64, 100, 16, 0, 0, 0, 4),     # table rows too short
])
def test_step_plan(R, new_lo, new_hi, cached_hi, ps, prefix, pad, short, narrow):
    from ddq_b200 import paged
    rng = random.Random(R * 31 + ps)
    cached = [rng.randint(0, cached_hi) for _ in range(R)]
    new = [rng.randint(new_lo, new_hi) for _ in range(R)]
    need = [ref.pages_for(c + n, ps) for c, n in zip(cached, new)]
    width = max(1, max(need) - narrow)
    ids = list(range(sum(need) + 50))
    rng.shuffle(ids)
    table = [[-7] * width for _ in range(R)]
    for r in range(R):
        for col in range(min(width, ref.pages_for(cached[r], ps))):
            table[r][col] = ids.pop()
    head = rng.randint(0, 20)
    taken = sum(need) - sum(ref.pages_for(c, ps) for c in cached)
    free = ids[:head + taken - short] if short else ids
    T = sum(new) + pad
    big = torch.full((R, width + 5), -9, dtype=torch.int32, device="cuda")  # strided rows
    big[:, :width] = torch.tensor(table, dtype=torch.int32)
    p = paged.plan_step(ints(cached), ints(new), big[:, :width], ints(free), ps, T,
                        free_head=ints([head]), prefix_len=prefix)
    torch.cuda.synchronize()
    table, cu, lens, slots, pos, seqs, at = ref.plan_reference(cached, new, table, free, ps, T,
                                                               head, prefix)
    assert big[:, :width].cpu().tolist() == table
    assert (big[:, width:] == -9).all()
    assert p.cu_new.tolist() == cu and p.lens.tolist() == lens
    assert p.slots.tolist() == slots and p.positions.tolist() == pos
    assert p.seq_ids.tolist() == seqs and p.free_head.tolist() == [at]


def test_step_plan_counts_more_tokens_than_rows_and_negative_lengths():
    from ddq_b200 import paged
    cached, new, ps, T = [5, -3, 0], [4, 30, -2], 16, 20   # 34 tokens, 20 rows
    table = [[2, -1, -1]] + [[-1] * 3] * 2
    t = torch.tensor(table, dtype=torch.int32, device="cuda")
    p = paged.plan_step(ints(cached), ints(new), t, ints([9, 4, 1]), ps, T)
    table, cu, lens, slots, pos, seqs, at = ref.plan_reference(cached, new, table, [9, 4, 1], ps,
                                                               T, 0, 0)
    assert t.cpu().tolist() == table and p.cu_new.tolist() == cu and p.lens.tolist() == lens
    assert p.slots.tolist() == slots and p.positions.tolist() == pos
    assert p.seq_ids.tolist() == seqs and p.free_head.tolist() == [at]


def test_step_plan_lengths_at_the_ends_of_int32_stay_in_bounds():
    from ddq_b200 import paged
    big = 2 ** 31 - 1
    t = torch.full((4, 2), -1, dtype=torch.int32, device="cuda")
    p = paged.plan_step(ints([big, 0, -big - 1, 3]), ints([big, big, big, 1]), t,
                        ints([5, 6]), 256, 64)
    torch.cuda.synchronize()
    assert p.slots.numel() == 64 and int(p.slots.max()) < 7 * 256


# ----------------------------------------------------------- RoPE + page write
@pytest.mark.parametrize("T,hq,hkv,d,ps,dtype,layout", [
    (1, 14, 2, 64, 16, F16, "hnd"), (64, 14, 2, 64, 16, F16, "nhd"), (37, 8, 8, 128, 64, BF16, "hnd"),
    (300, 16, 2, 128, 32, F16, "joint"), (129, 3, 1, 64, 128, BF16, "nhd"),
    (1000, 5, 5, 64, 256, F16, "hnd"), (0, 14, 2, 64, 16, F16, "hnd")])
def test_rope_and_page_write_bitwise(T, hq, hkv, d, ps, dtype, layout):
    from ddq_b200 import paged
    gen = torch.Generator().manual_seed(T + d)
    pool = ref.pages_for(max(T, 1), ps) + 2
    kp, vp = ref.make_pool(pool, hkv, ps, d, dtype, gen, layout)
    cos, sin = ref.rope_tables(500, d)
    slots = torch.randperm(pool * ps, generator=gen)[:T].cuda()
    slots[::7] = -1
    pos = torch.randint(0, 500, (T,), generator=gen).cuda()
    wide = torch.randn(T, (hq + 2 * hkv) * d + 8, generator=gen).to(dtype).cuda()
    qkv = wide[:, :(hq + 2 * hkv) * d]           # strided rows
    k0, v0 = kp.clone(), vp.clone()
    q = paged.rope_kv_write(qkv, kp, vp, cos, sin, slots, pos, hq, hkv, d)
    torch.cuda.synchronize()
    y = ref.rope_reference(qkv[:, :(hq + hkv) * d].reshape(T, hq + hkv, d), cos[pos], sin[pos])
    assert torch.equal(q, y[:, :hq])
    ok = slots >= 0
    k0[slots[ok] // ps, :, slots[ok] % ps] = y[ok, hq:]
    v0[slots[ok] // ps, :, slots[ok] % ps] = qkv[ok, (hq + hkv) * d:].reshape(-1, hkv, d)
    assert torch.equal(kp, k0) and torch.equal(vp, v0)   # every other row untouched


def test_rope_write_leaves_out_slots_and_positions_outside():
    from ddq_b200 import paged
    gen = torch.Generator().manual_seed(3)
    kp, vp = ref.make_pool(2, 2, 16, 64, F16, gen)
    cos, sin = ref.rope_tables(10, 64)
    qkv = torch.randn(4, 18 * 64, generator=gen).half().cuda()
    k0, v0 = kp.clone(), vp.clone()
    out = torch.full((4, 14, 64), 7.0, dtype=F16, device="cuda")
    paged.rope_kv_write(qkv, kp, vp, cos, sin, ints([32, 5, 2 ** 40, -2 ** 62], torch.int64),
                        ints([1, 10, -1, 2 ** 40], torch.int64), 14, 2, 64, out=out)
    assert device_error() == ERR_PAGE
    k0[0, :, 5] = kp[0, :, 5]       # position 10 of 10: no key (value written)
    assert torch.equal(kp, k0)
    v0[0, :, 5] = qkv[1, 16 * 64:].reshape(2, 64)
    assert torch.equal(vp, v0)
    y = ref.rope_reference(qkv[:1, :14 * 64].reshape(1, 14, 64), cos[1:2], sin[1:2])
    assert torch.equal(out[:1], y) and (out[1:] == 7.0).all()


# ------------------------------------------------------------ prompt attention
def prefill_case(new, cached, hq, hkv, d, ps, dtype, layout="hnd", cap=0.0, bias=False,
                 bidir=None, seed=0, qscale=1.0, tail=0, prefix=0):
    gen = torch.Generator().manual_seed(seed + sum(new) + d)
    lens = [n + c for n, c in zip(new, cached)]
    table, _, pool = ref.make_table(lens + [prefix], ps, gen)
    kp, vp = ref.make_pool(pool, hkv, ps, d, dtype, gen, layout)
    q = (torch.randn(sum(new) + tail, hq, d, generator=gen) * qscale).to(dtype).cuda()
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / hq) for h in range(hq)]).cuda() if bias else None
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return dict(q=q, kp=kp, vp=vp, table=table[:-1], cu=ints(cu), lens=ints(lens), slopes=slopes,
                prefix=table[-1, :max(1, ref.pages_for(prefix, ps))].contiguous(),
                bidir=ints(bidir) if bidir is not None else None), lens


def run_prefill(c, new, lens, d, cap=0.0, bidir=None, out=None, prefix=0, scale=None):
    from ddq_b200 import paged
    scale = d ** -0.5 if scale is None else scale
    o = paged.prefill_attention(c["q"], c["kp"], c["vp"], c["table"], c["cu"], c["lens"], scale,
                                softcap=cap, slopes=c["slopes"], bidir=c["bidir"], out=out,
                                prefix_pages=c["prefix"], prefix_len=prefix)
    torch.cuda.synchronize()
    T = sum(new)
    want, tol = ref.prefill_reference(c["q"][:T], c["kp"], c["vp"], c["table"], new, lens, scale,
                                      cap, c["slopes"], bidir, c["prefix"], prefix)
    close(o[:T], want, tol)
    return o


@pytest.mark.parametrize("new,cached,hq,hkv,d,ps,dtype,layout", [
    ([1], [0], 14, 2, 64, 16, F16, "hnd"), ([1], [16], 14, 2, 64, 16, F16, "hnd"),
    ([5], [127], 4, 4, 64, 16, F16, "hnd"), ([128], [0], 2, 2, 64, 64, F16, "hnd"),
    ([1, 37, 200], [0, 0, 0], 14, 2, 64, 16, F16, "nhd"),
    ([129, 0, 255, 3], [1, 50, 0, 700], 14, 2, 64, 32, BF16, "joint"),
    ([64, 1, 513], [100, 1000, 0], 16, 2, 128, 128, F16, "hnd"),
    ([300], [1111], 3, 1, 128, 256, BF16, "nhd"), ([77, 130], [0, 64], 32, 1, 64, 64, F16, "hnd"),
    ([600], [0], 8, 8, 128, 16, F16, "hnd"), ([17], [3000], 14, 2, 64, 16, F16, "hnd"),
    ([1], [5000], 8, 1, 128, 64, BF16, "hnd"), ([40] * 30, [0] * 30, 6, 2, 64, 16, F16, "hnd"),
    ([1] * 70, list(range(70)), 14, 2, 64, 16, F16, "hnd")])
def test_prefill_attention(new, cached, hq, hkv, d, ps, dtype, layout):
    c, lens = prefill_case(new, cached, hq, hkv, d, ps, dtype, layout)
    run_prefill(c, new, lens, d)


@pytest.mark.parametrize("d,hq,hkv,dtype,ps", [
    (128, 32, 4, BF16, 64), (64, 14, 2, F16, 16), (128, 8, 8, F16, 32), (64, 32, 32, BF16, 64),
    (128, 16, 1, F16, 128)])
def test_prefill_attention_many_requests(d, hq, hkv, dtype, ps):
    """More tiles than the GPU has SMs, whole and half-filled ones in turn, and
    requests without new tokens among them."""
    rng = random.Random(d + hq)
    R = 60 * 8 // hkv if hkv < 8 else 60
    new = [rng.choice([1, 5, 16, 17, 40, 64, 100, 129, 0]) for _ in range(R)]
    cached = [rng.choice([0, 0, 3, 127, 300]) for _ in range(R)]
    c, lens = prefill_case(new, cached, hq, hkv, d, ps, dtype)
    o = run_prefill(c, new, lens, d)
    for _ in range(3):
        assert torch.equal(run_prefill(c, new, lens, d), o)


@pytest.mark.parametrize("cap,bias,bidir", [
    (30.0, False, None), (5.0, False, None), (0.0, True, None), (0.0, False, "mixed"),
    (50.0, True, None), (0.0, True, "mixed"), (20.0, True, "mixed")])
@pytest.mark.parametrize("d,dtype,hq,hkv", [(64, F16, 14, 2), (128, BF16, 8, 2)])
def test_prefill_attention_masks_and_scores(cap, bias, bidir, d, dtype, hq, hkv):
    new, cached = [130, 1, 260, 19, 64], [0, 300, 45, 7, 0]
    bd = [100, 301, 9999, 0, -5] if bidir else None
    c, lens = prefill_case(new, cached, hq, hkv, d, 32, dtype, "hnd", cap, bias, bd, qscale=2.0)
    run_prefill(c, new, lens, d, cap, bd)


@pytest.mark.parametrize("qscale", [0.5, 2.5, 8.0])
@pytest.mark.parametrize("cap,bias,bidir", [(30.0, True, True), (30.0, False, False),
                                            (0.0, True, True)])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_prefill_attention_capped_scores_of_every_size(qscale, cap, bias, bidir, d, dtype):
    """Key tiles wholly before, around and wholly behind the rows, with scores below
    a sixth of the cap, below half of it, and above."""
    new, cached = [100, 300], [900, 100]
    bd = [1000, 390] if bidir else None
    c, lens = prefill_case(new, cached, 8, 2, d, 64, dtype, "hnd", cap, bias, bd, qscale=qscale)
    run_prefill(c, new, lens, d, cap, bd)


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_prefill_attention_capped_rows_before_position_zero(d, dtype):
    """A bidirectional prefix shows keys to rows that stand before them and have no
    key of their own, under a bias of hundreds; long rows with a steep bias."""
    new, cached = [600, 40, 130], [0, 0, 2000]
    bd = [1, 3, 0]
    c, lens = prefill_case(new, cached, 8, 2, d, 32, dtype, "hnd", 20.0, True, bd)
    lens = [1, 30, lens[2]]
    c["lens"] = ints(lens)
    o = run_prefill(c, new, lens, d, 20.0, bd)
    v0 = c["vp"][int(c["table"][0, 0]), :, 0].repeat_interleave(4, 0)
    assert torch.equal(o[:600], v0.expand(600, 8, d))


@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-12])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (0.0, True), (20.0, True)])
def test_prefill_attention_scales(scale, cap, bias):
    new, cached = [70, 150], [300, 20]
    c, lens = prefill_case(new, cached, 4, 2, 64, 16, F16, "hnd", cap, bias)
    run_prefill(c, new, lens, 64, cap, scale=scale)


@pytest.mark.parametrize("R", [31, 32, 33])
def test_prefill_attention_batches_of_unequal_requests(R):
    rng = random.Random(R)
    new = [rng.choice([0, 1, 7, 64, 130]) for _ in range(R)]
    cached = [rng.choice([0, 5, 128, 400, 900]) for _ in range(R)]
    c, lens = prefill_case(new, cached, 7, 1, 64, 16, F16)
    run_prefill(c, new, lens, 64)


@pytest.mark.parametrize("d,dtype,ps,prefix,cap,bias,bidir", [
    (64, F16, 16, 37, 0.0, False, None), (64, F16, 16, 128, 0.0, False, [100, 0, 999, 3]),
    (128, BF16, 64, 1, 30.0, True, None), (128, F16, 32, 700, 0.0, True, [100, 0, 999, 3]),
    (64, BF16, 128, 2000, 0.0, False, None)])
def test_prefill_attention_behind_a_shared_prefix(d, dtype, ps, prefix, cap, bias, bidir):
    new, cached = [130, 1, 260, 0], [0, 300, 45, 9]
    c, lens = prefill_case(new, cached, 14, 2, d, ps, dtype, "hnd", cap, bias, bidir,
                           prefix=prefix)
    run_prefill(c, new, lens, d, cap, bidir, prefix=prefix)


def test_prefill_attention_rows_without_keys_are_zero_and_rows_behind_stay():
    """Lengths below the number of new tokens (a row before position 0 has no
    key), a length of zero, and padded rows behind the last request."""
    new, cached = [5, 3, 2], [0, 0, 0]
    c, lens = prefill_case(new, cached, 14, 2, 64, 16, F16, tail=9)
    lens = [3, 0, 2]
    c["lens"] = ints(lens)
    out = torch.full_like(c["q"], 3.0)
    o = run_prefill(c, new, lens, 64, out=out)
    assert (o[:2] == 0).all() and (o[5:8] == 0).all() and (o[10:] == 3.0).all()


@pytest.mark.parametrize("d,ps", [(64, 16), (128, 64)])
def test_prefill_attention_never_looks_behind_a_request(d, ps):
    """NaN and infinity in the unused rows of the last page, in unused pages and
    in padded query rows; table entries behind the length name no page."""
    new, cached = [37, 130, 1], [3, 130, 0]
    c, lens = prefill_case(new, cached, 14, 2, d, ps, F16, tail=5)
    used = torch.zeros(c["kp"].shape[0], ps, dtype=torch.bool, device="cuda")
    for r, L in enumerate(lens):
        for j in range(L):
            used[int(c["table"][r, j // ps]), j % ps] = True
    for x, bad in ((c["kp"], float("nan")), (c["vp"], float("inf"))):
        x.masked_fill_(~used[:, None, :, None], bad)
    c["vp"][..., ::2].masked_fill_(~used[:, None, :, None], float("nan"))
    c["q"][sum(new):] = float("nan")
    run_prefill(c, new, lens, d)


def test_prefill_attention_large_scores_and_equal_scores():
    """Scores of hundreds (one weight takes all), rising along the keys so that
    the running maximum moves in every tile, and all-equal scores."""
    new, cached = [200], [500]
    c, lens = prefill_case(new, cached, 4, 2, 64, 16, F16, qscale=40.0)
    run_prefill(c, new, lens, 64)
    c["q"].fill_(1.0)
    ramp = torch.arange(700, dtype=torch.float32, device="cuda") / 100
    for j in range(700):
        c["kp"][int(c["table"][0, j // 16]), :, j % 16] = ramp[j].half()
    run_prefill(c, new, lens, 64)
    c["q"].zero_()
    run_prefill(c, new, lens, 64)


def test_prefill_attention_strided_queries_and_output():
    """q a slice of a wider projection row, out head-major."""
    new, cached = [70, 3], [10, 200]
    c, lens = prefill_case(new, cached, 14, 2, 64, 16, F16)
    wide = torch.zeros(73, 18 * 64, dtype=F16, device="cuda")
    wide[:, 64:15 * 64] = c["q"].reshape(73, -1)
    c["q"] = wide[:, 64:15 * 64].view(73, 14, 64)
    out = torch.zeros(14, 73, 64, dtype=F16, device="cuda").transpose(0, 1)
    run_prefill(c, new, lens, 64, out=out)


# ------------------------------------------------------------ decode attention
def decode_case(lens, prefix, hq, hkv, d, ps, dtype, layout="hnd", bias=False, seed=0,
                qscale=1.0, width=None):
    gen = torch.Generator().manual_seed(seed + sum(lens) + prefix + d)
    table, _, pool = ref.make_table(list(lens) + [prefix], ps, gen, width)
    kp, vp = ref.make_pool(pool, hkv, ps, d, dtype, gen, layout)
    q = (torch.randn(len(lens), hq, d, generator=gen) * qscale).to(dtype).cuda()
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / hq) for h in range(hq)]).cuda() if bias else None
    w = width or max(1, ref.pages_for(max(lens), ps))
    return dict(q=q, kp=kp, vp=vp, table=table[:-1, :w],
                prefix=table[-1, :max(1, ref.pages_for(prefix, ps))].contiguous(),
                lens=ints(lens), slopes=slopes)


def run_decode(c, lens, prefix, d, cap=0.0, out=None):
    from ddq_b200 import paged
    scale = d ** -0.5
    o = paged.decode_attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], scale,
                               prefix_pages=c["prefix"], prefix_len=prefix, softcap=cap,
                               slopes=c["slopes"], out=out)
    torch.cuda.synchronize()
    want, tol = ref.decode_reference(c["q"], c["kp"], c["vp"], c["table"], lens, scale,
                                     c["prefix"], prefix, cap, c["slopes"])
    close(o, want, tol)
    return o


@pytest.mark.parametrize("lens,prefix,hq,hkv,d,ps,dtype,layout", [
    ([1], 0, 14, 2, 64, 16, F16, "hnd"), ([0], 0, 14, 2, 64, 16, F16, "hnd"),
    ([33], 0, 14, 2, 64, 16, F16, "nhd"), ([1, 0, 700, 31, 32, 33], 0, 14, 2, 64, 16, F16, "hnd"),
    ([5, 0, 100], 1, 14, 2, 64, 16, F16, "hnd"), ([1, 40, 7], 130, 14, 2, 64, 32, BF16, "joint"),
    ([3000, 1, 2], 0, 8, 8, 64, 64, F16, "hnd"), ([500, 20], 1000, 16, 2, 128, 16, F16, "nhd"),
    ([257] * 9, 511, 4, 1, 128, 256, BF16, "hnd"), ([0, 0, 0], 77, 6, 2, 64, 16, F16, "hnd"),
    (list(range(64)), 512, 14, 2, 64, 16, F16, "hnd"), ([60], 5000, 32, 2, 128, 128, F16, "hnd"),
    ([900, 3], 200, 24, 1, 64, 64, BF16, "hnd"), ([10, 20], 300, 40, 1, 128, 16, F16, "hnd"),
    ([9000], 0, 14, 2, 64, 16, F16, "hnd"), ([2, 300] * 50, 129, 3, 3, 64, 64, F16, "hnd")])
def test_decode_attention(lens, prefix, hq, hkv, d, ps, dtype, layout):
    c = decode_case(lens, prefix, hq, hkv, d, ps, dtype, layout)
    o = run_decode(c, lens, prefix, d)
    if prefix == 0:
        for b, n in enumerate(lens):
            assert n > 0 or (o[b] == 0).all()


@pytest.mark.parametrize("cap,bias", [(30.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("d,dtype,hq,hkv", [(64, F16, 14, 2), (128, BF16, 16, 1)])
def test_decode_attention_scores(cap, bias, d, dtype, hq, hkv):
    lens, prefix = [1, 77, 0, 600, 32], 150
    c = decode_case(lens, prefix, hq, hkv, d, 16, dtype, bias=bias, qscale=3.0)
    run_decode(c, lens, prefix, d, cap)


def test_decode_attention_wide_table_and_short_lengths():
    """Table rows for thousands of pages, most of them unused."""
    lens = [3, 17, 0, 250]
    c = decode_case(lens, 0, 14, 2, 64, 16, F16, width=2048)
    run_decode(c, lens, 0, 64)


@pytest.mark.parametrize("d,ps,prefix", [(64, 16, 21), (128, 64, 200)])
def test_decode_attention_never_looks_behind_the_lengths(d, ps, prefix):
    lens = [1, 37, 0, 130]
    c = decode_case(lens, prefix, 14, 2, d, ps, F16)
    used = torch.zeros(c["kp"].shape[0], ps, dtype=torch.bool, device="cuda")
    for row, L in list(zip(c["table"], lens)) + [(c["prefix"], prefix)]:
        for j in range(L):
            used[int(row[j // ps]), j % ps] = True
    c["kp"].masked_fill_(~used[:, None, :, None], float("nan"))
    c["vp"].masked_fill_(~used[:, None, :, None], float("inf"))
    c["vp"][..., ::2].masked_fill_(~used[:, None, :, None], float("nan"))
    run_decode(c, lens, prefix, d)


def test_decode_attention_large_scores():
    lens, prefix = [300, 5, 1000], 260
    c = decode_case(lens, prefix, 14, 2, 64, 16, F16, qscale=60.0)
    run_decode(c, lens, prefix, 64)


def test_decode_equals_the_prefix_copied_into_every_sequence():
    """The shared prefix gives what the same keys in each sequence's own pages give."""
    from ddq_b200 import paged
    lens, prefix, ps = [1, 16, 40], 48, 16
    c = decode_case(lens, prefix, 14, 2, 64, ps, F16)
    a = run_decode(c, lens, prefix, 64)
    own = torch.zeros(3, 3 + c["table"].shape[1], dtype=torch.int32, device="cuda")
    own[:, :3], own[:, 3:] = c["prefix"], c["table"]
    b = paged.decode_attention(c["q"], c["kp"], c["vp"], own, ints([n + prefix for n in lens]),
                               0.125)
    # both are within the tolerance of the same value
    want, tol = ref.decode_reference(c["q"], c["kp"], c["vp"], c["table"], lens, 0.125,
                                     c["prefix"], prefix, 0.0, None)
    close(b, want, tol)
    assert (a.float() - b.float()).abs().max() <= 2 * tol.max()


# ------------------------------------------------- bad tables, streams, graphs
def test_pages_outside_the_pool_touch_no_other_request():
    from ddq_b200 import paged
    lens, prefix = [40, 100, 7], 0
    c = decode_case(lens, prefix, 14, 2, 64, 16, F16)
    good = run_decode(c, lens, prefix, 64)
    want, tol = ref.decode_reference(c["q"], c["kp"], c["vp"], c["table"], lens, 0.125,
                                     c["prefix"], 0, 0.0, None)
    pool = c["kp"].shape[0]
    for bad in (-1, pool, 2 ** 31 - 1, -2 ** 31):
        t = c["table"].clone()
        t[1, 3] = bad
        o = paged.decode_attention(c["q"], c["kp"], c["vp"], t, c["lens"], 0.125)
        assert device_error() == ERR_PAGE
        assert torch.equal(o[0], good[0]) and torch.equal(o[2], good[2])
        p = paged.prefill_attention(c["q"], c["kp"], c["vp"], t, ints([0, 1, 2, 3]), c["lens"],
                                    0.125)
        assert device_error() == ERR_PAGE
        close(p[::2], want[::2], tol[::2])


def test_a_length_beyond_the_table_is_reported():
    from ddq_b200 import paged
    c = decode_case([30, 20], 0, 14, 2, 64, 16, F16)
    c["lens"] = ints([10 ** 6, 20])
    good = run_decode(decode_case([30, 20], 0, 14, 2, 64, 16, F16), [30, 20], 0, 64)
    o = paged.decode_attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], 0.125)
    assert device_error() == ERR_PAGE
    assert torch.equal(o[1], good[1])
    paged.prefill_attention(c["q"], c["kp"], c["vp"], c["table"], ints([0, 1, 2]), c["lens"],
                            0.125)
    assert device_error() == ERR_PAGE


@pytest.mark.parametrize("d", [64, 128])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(d):
    """The scores-ready signal left out (a test hook): the bounded waits give up, the
    kernel winds down, and the device error word says so."""
    from ddq_b200 import _lib, paged
    new, cached = [300, 20], [100, 0]
    c, lens = prefill_case(new, cached, 8, 2, d, 16, F16)
    lib = _lib.load()
    assert lib.ddq_set_debug(1, 2_000_000) == 0          # 2 ms
    try:
        paged.prefill_attention(c["q"], c["kp"], c["vp"], c["table"], c["cu"], c["lens"],
                                d ** -0.5)
        torch.cuda.synchronize()
    finally:
        lib.ddq_set_debug(0, 0)
    assert device_error() == 7                            # DDQ_ERR_TIMEOUT
    run_prefill(c, new, lens, d)


def test_pages_far_into_a_large_pool():
    """Offsets of the pool beyond 2^32 bytes and 2^31 elements."""
    from ddq_b200 import paged
    hq, hkv, d, ps, P = 16, 8, 128, 64, 36000            # 2.4 G elements each
    kp = torch.empty(P, hkv, ps, d, dtype=F16, device="cuda")
    vp = torch.empty_like(kp)
    gen = torch.Generator().manual_seed(2)
    pages = torch.tensor([P - 1, 1, P - 7, P - 2, 33000, 5], dtype=torch.int32)
    n = 300
    slots = (pages.long()[torch.arange(n) // ps] * ps + torch.arange(n) % ps).cuda()
    cos, sin = ref.rope_tables(n, d)
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=gen).half().cuda()
    pos = torch.arange(n, device="cuda")
    q = paged.rope_kv_write(qkv, kp, vp, cos, sin, slots, pos, hq, hkv, d)
    y = ref.rope_reference(qkv[:, :(hq + hkv) * d].reshape(n, -1, d), cos, sin)
    k, v = y[:, hq:], qkv[:, (hq + hkv) * d:].reshape(n, hkv, d)
    assert torch.equal(kp[slots // ps, :, slots % ps], k)
    assert torch.equal(vp[slots // ps, :, slots % ps], v)
    table = pages[None].cuda()
    o = paged.prefill_attention(q, kp, vp, table, ints([0, n]), ints([n]), d ** -0.5)
    want, tol = ref.prefill_reference(q, kp, vp, table, [n], [n], d ** -0.5, 0.0, None, None)
    close(o, want, tol)
    o = paged.decode_attention(q[-1:], kp, vp, table[:, 2:], ints([n - 2 * ps]), d ** -0.5,
                               prefix_pages=table[0, :2].contiguous(), prefix_len=2 * ps)
    close(o[0], want[-1], tol[-1])


def test_results_do_not_change_from_call_to_call():
    lens, prefix = [700, 3, 64, 2000], 900
    c = decode_case(lens, prefix, 14, 2, 64, 16, F16)
    first = run_decode(c, lens, prefix, 64)
    p, plens = prefill_case([300, 9], [40, 2000], 14, 2, 64, 16, F16)
    pf = run_prefill(p, [300, 9], plens, 64)
    for _ in range(5):
        assert torch.equal(run_decode(c, lens, prefix, 64), first)
        assert torch.equal(run_prefill(p, [300, 9], plens, 64), pf)


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing is initialised by a call in a way that a capture forbids."""
    code = """
import torch
from ddq_b200 import paged
i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
kp, vp = (torch.zeros(8, 2, 16, 64, dtype=torch.float16, device="cuda") for _ in range(2))
cos, sin = torch.ones(64, 64, device="cuda"), torch.zeros(64, 64, device="cuda")
qkv = torch.ones(5, 18 * 64, dtype=torch.float16, device="cuda")
table, free, old, new, pre = i([-1] * 2, [-1] * 2), i(5, 2, 3), i(0, 0), i(4, 1), i(7)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    p = paged.plan_step(old, new, table, free, 16, 5, prefix_len=9)
    q = paged.rope_kv_write(qkv, kp, vp, cos, sin, p.slots, p.positions, 14, 2, 64)
    o = paged.prefill_attention(q, kp, vp, table, p.cu_new, p.lens, 0.125)
    d = paged.decode_attention(q[3:], kp, vp, table, p.lens, 0.125, pre, 9)
g.replay()
torch.cuda.synchronize()
assert table[:, 0].tolist() == [5, 2] and (o == 1).all() and (q == 1).all()
# keys of ones (weight e^8) behind a prefix of zeros
want = torch.tensor([n / (n + 9 * 2.718281828 ** -8) for n in (4, 1)], device="cuda")
assert ((d.float() - want[:, None, None]).abs() < 2.0 ** -10).all()
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_graphs_and_two_streams_share_nothing():
    """Two captured decode steps replayed at once on two streams, lengths moved
    on the device in between, while eager calls run on a third."""
    from ddq_b200 import paged
    lens = [[900, 4, 2], [10, 1200, 77]]
    cs = [decode_case(x, 600, 14, 2, 64, 16, F16, seed=i) for i, x in enumerate(lens)]

    def call(c):
        return paged.decode_attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], 0.125,
                                      prefix_pages=c["prefix"], prefix_len=600)
    for c in cs:
        call(c)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(3):
        now = [[max(0, n - step) for n in x] for x in lens]
        for c, x in zip(cs, now):
            c["lens"].copy_(ints(x))
        torch.cuda.synchronize()
        for _ in range(20):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            call(cs[0])
        torch.cuda.synchronize()
        for c, x, o in zip(cs, now, outs):
            want, tol = ref.decode_reference(c["q"], c["kp"], c["vp"], c["table"], x, 0.125,
                                             c["prefix"], 600, 0.0, None)
            close(o, want, tol)


# -------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype,hq,hkv,d,ps,prefix,cap,bias", [
    (F16, 14, 2, 64, 16, 37, 0.0, False), (BF16, 8, 2, 128, 32, 0, 25.0, True)])
def test_a_serving_run(dtype, hq, hkv, d, ps, prefix, cap, bias):
    """Prompts of different lengths behind a shared prefix, in two chunks, then
    decode steps in a captured graph: plan, RoPE + page write and attention of
    each step, against dense 64-bit attention over all keys so far."""
    from ddq_b200 import paged
    gen = torch.Generator().manual_seed(11)
    R, width, scale = 5, 12, d ** -0.5
    u = torch.finfo(dtype).eps / 2
    pool = R * width + ref.pages_for(prefix, ps) + 4
    kp, vp = ref.make_pool(pool, hkv, ps, d, dtype, gen)
    kp.fill_(float("nan")), vp.fill_(float("nan"))
    perm = torch.randperm(pool, generator=gen).to(torch.int32).cuda()
    npre = ref.pages_for(prefix, ps)
    prefix_pages, free = perm[:npre].contiguous(), perm[npre:].contiguous()
    cos, sin = ref.rope_tables(2000, d)
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / hq) for h in range(hq)]).cuda() if bias else None
    W = (hq + 2 * hkv) * d

    def project(T):
        return torch.randn(T, W, generator=gen).to(dtype).cuda()
    hist_k = [torch.zeros(0, hkv, d, dtype=dtype, device="cuda") for _ in range(R)]
    hist_v = [x.clone() for x in hist_k]
    pre_k = pre_v = None
    if prefix:          # the prefix itself: one request's pages
        x = project(prefix)
        i = torch.arange(prefix, device="cuda")
        slots = prefix_pages[i // ps].long() * ps + i % ps
        paged.rope_kv_write(x, kp, vp, cos, sin, slots, i, hq, hkv, d)
        y = ref.rope_reference(x[:, :(hq + hkv) * d].reshape(prefix, -1, d), cos[i], sin[i])
        pre_k, pre_v = y[:, hq:], x[:, (hq + hkv) * d:].reshape(prefix, hkv, d)

    table = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    cached, head = ints([0] * R), ints([0])

    def expect(qs, ks, vs, pos):
        k = torch.cat([pre_k, ks]) if prefix else ks
        v = torch.cat([pre_v, vs]) if prefix else vs
        os_, ts = [], []
        for h in range(hq):
            g = h * hkv // hq
            o, t = ref.attend_many(qs[:, h].double(), k[:, g].double(), v[:, g].double(), pos, 0,
                                   scale, cap, slopes[h].double() if bias else None, u)
            os_.append(o)
            ts.append(t)
        return torch.stack(os_, 1), torch.stack(ts, 1)

    def note(x, p, new):
        """Rotate the step's tokens on the side and add them to the histories."""
        T = sum(new)
        y = ref.rope_reference(x[:T, :(hq + hkv) * d].reshape(T, -1, d), cos[p.positions[:T]],
                               sin[p.positions[:T]])
        v = x[:T, (hq + hkv) * d:].reshape(T, hkv, d)
        at = 0
        for r, n in enumerate(new):
            hist_k[r] = torch.cat([hist_k[r], y[at:at + n, hq:]])
            hist_v[r] = torch.cat([hist_v[r], v[at:at + n]])
            at += n
        return y[:, :hq]
    # prompts, two chunks, in padded steps
    for new in ([9, 40, 1, 0, 63], [30, 0, 5, 17, 2]):
        T = sum(new) + 3
        p = paged.plan_step(cached, ints(new), table, free, ps, T, free_head=head,
                            prefix_len=prefix)
        x = project(T)
        q = paged.rope_kv_write(x, kp, vp, cos, sin, p.slots, p.positions, hq, hkv, d)
        o = paged.prefill_attention(q, kp, vp, table, p.cu_new, p.lens, scale, softcap=cap,
                                    slopes=slopes, prefix_pages=prefix_pages, prefix_len=prefix)
        qr = note(x, p, new)
        assert torch.equal(q[:sum(new)], qr)
        at = 0
        for r, n in enumerate(new):
            L = prefix + hist_k[r].shape[0]
            want, tol = expect(qr[at:at + n], hist_k[r], hist_v[r],
                               torch.arange(L - n, L, device="cuda"))
            close(o[at:at + n], want, tol)
            at += n
        cached, head = p.lens, p.free_head
    # decode steps: the graph reads and advances its own lengths and free head
    cached, head, one = cached.clone(), head.clone(), ints([1] * R)
    x = project(R)

    def step():
        p = paged.plan_step(cached, one, table, free, ps, R, free_head=head, prefix_len=prefix)
        q = paged.rope_kv_write(x, kp, vp, cos, sin, p.slots, p.positions, hq, hkv, d)
        o = paged.decode_attention(q, kp, vp, table, p.lens, scale, prefix_pages=prefix_pages,
                                   prefix_len=prefix, softcap=cap, slopes=slopes)
        cached.copy_(p.lens)
        head.copy_(p.free_head)
        return p, o
    p, o = step()                                   # eager
    graph = None
    for s in range(6):
        if s:
            if graph is None:
                c0, h0 = cached.clone(), head.clone()
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    p, o = step()
                cached.copy_(c0), head.copy_(h0)
            x.copy_(project(R))
            graph.replay()
        torch.cuda.synchronize()
        qr = note(x, p, [1] * R)
        for r in range(R):
            L = prefix + hist_k[r].shape[0]
            assert int(p.positions[r]) == L - 1
            want, tol = expect(qr[r:r + 1], hist_k[r], hist_v[r],
                               torch.tensor([L - 1], device="cuda"))
            close(o[r:r + 1], want, tol)


# --------------------------------------------- what scores and weights may be off
def strict(q, k, v, pos, least, scale, cap, slope, w):
    """As ``paged_reference.attend_many``, with a bound that does not grow with the cap.

    softcap * tanh(s / softcap) is a function of s whose relative error, evaluated in
    32 bits, is a few 2^-23 whatever the cap, so a score z is off by at most 2^-20 |z|
    (and by the dot product's (D + 2) 2^-23 sum|q k| scale; 2^-20 also for the exponential).
    w: how far a weight is off, relative to it, on its way to the weighted sum."""
    n, d = q.shape
    L = k.shape[0]
    z = (q @ k.T) * scale
    mag = (q.abs() @ k.abs().T).amax(1, keepdim=True) * abs(scale)
    if cap:
        z = cap * torch.tanh(z / cap)
    j = torch.arange(L, device=q.device)[None, :]
    if slope is not None:
        z = z - slope * (pos[:, None] - j).abs().double()
    keep = j < (pos + 1).clamp(min=least)[:, None]
    z = torch.where(keep, z, torch.full_like(z, -math.inf))
    p = torch.softmax(z, 1)
    o, A = p @ v, p @ v.abs()
    zmax = torch.where(keep, z.abs(), torch.zeros_like(z)).amax(1, keepdim=True)
    e = (d + 2) * 2.0 ** -23 * mag + 2.0 ** -20 * zmax.clamp(min=1.0)
    cnt = keep.sum(1, keepdim=True).double()
    return o, (w + 2 * e + (cnt / 16 + 8) * 2.0 ** -22) * A + cnt * 2.0 ** -25 * v.abs().max()


def strict_decode(c, lens, prefix, scale, cap, w):
    """Every row of a decode case: the 64-bit results and their bounds."""
    q, u = c["q"], torch.finfo(c["q"].dtype).eps / 2
    B, hq, d = q.shape
    hkv = c["kp"].shape[1]
    o = torch.zeros(B, hq, d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    for b, n in enumerate(lens):
        if prefix + n == 0:
            continue
        for h in range(hq):
            g = h * hkv // hq
            k = torch.cat([ref.rows_of(c["kp"], c["prefix"], prefix, g),
                           ref.rows_of(c["kp"], c["table"][b], n, g)])
            v = torch.cat([ref.rows_of(c["vp"], c["prefix"], prefix, g),
                           ref.rows_of(c["vp"], c["table"][b], n, g)])
            sl = c["slopes"][h].double() if c["slopes"] is not None else None
            x, t = strict(q[b:b + 1, h].double(), k, v,
                          torch.tensor([prefix + n - 1], device="cuda"), 0, scale, cap, sl, w)
            o[b, h], tol[b, h] = x[0], (1 + u) * (t + u * x.abs())[0]
    return o, tol


@pytest.mark.parametrize("cap", [50.0, 1e3, 1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("d,dtype,hq,hkv,prefix,bias", [
    (64, F16, 14, 2, 0, False), (128, BF16, 16, 1, 0, True), (64, F16, 8, 2, 40, True)])
def test_decode_attention_keeps_small_scores_under_a_large_cap(cap, d, dtype, hq, hkv, prefix,
                                                               bias):
    """Scores of a few units, far below the cap: the cap leaves them as they are."""
    from ddq_b200 import paged
    lens = [3, 9, 1, 40]
    c = decode_case(lens, prefix, hq, hkv, d, 16, dtype, bias=bias, qscale=2.0)
    o = paged.decode_attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], d ** -0.5,
                               prefix_pages=c["prefix"], prefix_len=prefix, softcap=cap,
                               slopes=c["slopes"])
    want, tol = strict_decode(c, lens, prefix, d ** -0.5, cap, torch.finfo(dtype).eps / 2)
    close(o, want, tol)


def test_decode_attention_small_scores_beside_some_above_a_large_cap():
    """A sequence, a head and single keys whose scores exceed half the cap, next to small ones."""
    from ddq_b200 import paged
    lens, cap = [30, 40, 35], 1e6
    c = decode_case(lens, 0, 8, 1, 64, 16, BF16)
    c["q"][0, 3] *= 1e6
    c["kp"][int(c["table"][1, 0]), 0, 5] *= -1e7
    o = paged.decode_attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], 0.125,
                               softcap=cap)
    want, tol = strict_decode(c, lens, 0, 0.125, cap, torch.finfo(BF16).eps / 2)
    tol[1] = 1e30       # (sums of 1e7 in that sequence's scores)
    close(o, want, tol)


@pytest.mark.parametrize("cap", [50.0, 1e3, 1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("bias", [False, True])
def test_prefill_attention_small_scores_beside_some_above_a_large_cap(cap, bias):
    """Rows whose scores exceed half the cap among rows of small scores."""
    from ddq_b200 import paged
    new, cached = [40], [10]
    c, lens = prefill_case(new, cached, 8, 1, 64, 16, BF16, "hnd", cap, bias)
    c["q"][5, 2] *= 1e6
    o = paged.prefill_attention(c["q"], c["kp"], c["vp"], c["table"], c["cu"], c["lens"], 0.125,
                                softcap=cap, slopes=c["slopes"])
    u = torch.finfo(BF16).eps / 2
    k, v = ref.rows_of(c["kp"], c["table"][0], 50, 0), ref.rows_of(c["vp"], c["table"][0], 50, 0)
    for h in range(8):
        sl = c["slopes"][h].double() if bias else None
        want, tol = strict(c["q"][:, h].double(), k, v, torch.arange(10, 50, device="cuda"), 0,
                           0.125, cap, sl, u)
        close(o[:, h], want, (1 + u) * (tol + u * want.abs()))


@pytest.mark.parametrize("cap", [1e-3, 1e-30, 1e-39])
def test_attention_under_a_tiny_cap(cap):
    """Every score is the cap or nearly so, a score of 0 stays 0: all weights are equal."""
    from ddq_b200 import paged
    new, cached = [5, 40], [0, 100]
    c, lens = prefill_case(new, cached, 8, 2, 64, 16, F16)
    c["q"][3] = 0
    o = paged.prefill_attention(c["q"], c["kp"], c["vp"], c["table"], c["cu"], c["lens"], 0.125,
                                softcap=cap)
    want, tol = ref.prefill_reference(c["q"], c["kp"], c["vp"], c["table"], new, lens, 0.125, cap,
                                      None, None)
    close(o, want, tol)
    last = [4, 44]
    o = paged.decode_attention(c["q"][last], c["kp"], c["vp"], c["table"], c["lens"], 0.125,
                               softcap=cap)
    close(o, want[last], tol[last])


def test_step_plan_with_its_inputs_between_the_rows_of_the_table():
    """One buffer a request row: pages, then other state; nothing of it is in the way."""
    from ddq_b200 import paged
    state = torch.full((2, 10), -1, dtype=torch.int32, device="cuda")
    table, cached, new = state[:, :8], state[0, 8:], state[1, 8:]
    cached.copy_(ints([3, 16])), new.copy_(ints([20, 1]))
    table[0, 0], table[1, 0] = 5, 7
    want = [row[:] for row in table.tolist()]
    p = paged.plan_step(cached, new, table, ints([9, 8, 2]), 16, 21)
    want, cu, lens, slots, pos, seqs, at = ref.plan_reference([3, 16], [20, 1], want, [9, 8, 2],
                                                              16, 21, 0, 0)
    assert table.tolist() == want and cached.tolist() == [3, 16] and new.tolist() == [20, 1]
    assert p.cu_new.tolist() == cu and p.lens.tolist() == lens and p.slots.tolist() == slots
    assert p.positions.tolist() == pos and p.free_head.tolist() == [at]


@pytest.mark.parametrize("extra", [0, 40])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (20.0, True)])
def test_prefill_attention_of_a_request_cut_by_the_rows_of_q(extra, cap, bias):
    """A step whose last request has more new tokens than q has rows (plan_step gives such
    sums where num_tokens is too small): the rows that exist keep their positions."""
    from ddq_b200 import paged
    new, cached = [0] * extra + [4, 300], [0] * extra + [30, 100]
    c, lens = prefill_case(new, cached, 8, 2, 64, 16, F16, "hnd", cap, bias)
    want, tol = ref.prefill_reference(c["q"], c["kp"], c["vp"], c["table"], new, lens, 0.125, cap,
                                      c["slopes"], None)
    for T in (5, 104, 303):
        o = paged.prefill_attention(c["q"][:T], c["kp"], c["vp"], c["table"], c["cu"], c["lens"],
                                    0.125, softcap=cap, slopes=c["slopes"])
        close(o, want[:T], tol[:T])


@pytest.mark.parametrize("new,cached", [([20], [11]), ([3, 300], [0, 7])])
def test_capped_scores_do_not_depend_on_what_lies_behind_a_request(new, cached):
    """The same bits whatever the unused rows of the last page hold."""
    from ddq_b200 import paged
    c, lens = prefill_case(new, cached, 14, 2, 64, 16, F16, "hnd", 30.0, True)
    outs = []
    for fill in (0.0, 1e4, float("nan"), -60000.0):
        for r, n in enumerate(lens):
            if n % 16:
                c["kp"][int(c["table"][r, n // 16]), :, n % 16:] = fill
        outs.append(paged.prefill_attention(c["q"], c["kp"], c["vp"], c["table"], c["cu"],
                                            c["lens"], 0.125, softcap=30.0, slopes=c["slopes"]))
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


@pytest.mark.parametrize("dtype,d,hq,hkv", [(F16, 64, 14, 2), (BF16, 128, 8, 2), (F16, 128, 16, 1),
                                            (BF16, 64, 24, 2)])
def test_decode_attention_weights_reach_the_sum_in_two_parts(dtype, d, hq, hkv):
    """Values that cancel show a weight's rounding: two parts leave (u / 2)^2 or so of it."""
    from ddq_b200 import paged
    lens = [2, 4, 6, 30, 64, 33] * 4
    c = decode_case(lens, 0, hq, hkv, d, 16, dtype)
    c["q"][..., 4:] = 0                       # dot products of four exact products
    c["vp"].fill_(1.0)
    c["vp"][:, :, 1::2] = -1.0
    o = paged.decode_attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], 0.125)
    u = torch.finfo(dtype).eps / 2
    want, tol = strict_decode(c, lens, 0, 0.125, 0.0, u * u)
    close(o, want, tol)


@pytest.mark.parametrize("hq,hkv,dtype,ps,prefix", [(14, 2, F16, 64, 0), (16, 2, BF16, 32, 100),
                                                    (9, 3, F16, 256, 0)])
def test_decode_attention_64_wide_with_units_for_two_blocks_an_sm(hq, hkv, dtype, ps, prefix):
    """More units of 32 keys than one block on each SM has warps for, ranges that cut most
    sequences, heads in groups of 3, 7 and 8."""
    rng = random.Random(hq)
    lens = [rng.choice([0, 1, 40, 1200, 2500, 1999]) for _ in range(48)]
    c = decode_case(lens, prefix, hq, hkv, 64, ps, dtype)
    o = run_decode(c, lens, prefix, 64)
    assert torch.equal(run_decode(c, lens, prefix, 64), o)


# ------------------------------------------- calls that the documentation allows
@pytest.mark.parametrize("d,hq,hkv,prefix", [(64, 14, 2, 0), (128, 16, 1, 0), (64, 8, 2, 300)])
def test_a_wait_of_the_decode_kernel_that_runs_out_is_reported(d, hq, hkv, prefix):
    """A copy announced larger than it is (a test hook): the warps' bounded waits give up, the
    kernel winds down, the device error word says so, and the next call is right."""
    from ddq_b200 import _lib, paged
    lens = [300, 0, 20, 700]
    c = decode_case(lens, prefix, hq, hkv, d, 16, F16)
    lib = _lib.load()
    assert lib.ddq_set_debug(1, 2_000_000) == 0          # 2 ms
    try:
        paged.decode_attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], d ** -0.5,
                               prefix_pages=c["prefix"], prefix_len=prefix)
        torch.cuda.synchronize()
    finally:
        lib.ddq_set_debug(0, 0)
    assert device_error() == 7                            # DDQ_ERR_TIMEOUT
    run_decode(c, lens, prefix, d)


@pytest.mark.parametrize("prefix,cap", [(0, 0.0), (70, 20.0)])
def test_prefill_attention_bidirectional_beyond_32_requests(prefix, cap):
    rng = random.Random(5)
    R = 70
    new = [rng.choice([0, 1, 7, 30, 130]) for _ in range(R)]
    cached = [rng.choice([0, 5, 128, 300]) for _ in range(R)]
    bd = [rng.choice([0, 3, n + c, 10 ** 6]) for n, c in zip(new, cached)]
    c, lens = prefill_case(new, cached, 8, 2, 64, 16, F16, "hnd", cap, bool(cap), bd,
                           prefix=prefix)
    run_prefill(c, new, lens, 64, cap, bd, prefix=prefix)


@pytest.mark.parametrize("new,cached", [([200], [0]), ([512] * 4, [0] * 4), ([3, 90], [700, 40])])
@pytest.mark.parametrize("width", [512, 8192])
def test_prefill_attention_with_a_table_wider_than_the_requests(new, cached, width):
    """A table for the longest context there may be: most parts of the key axis are empty."""
    c, lens = prefill_case(new, cached, 14, 2, 64, 16, F16)
    table = torch.full((len(new), width), -1, dtype=torch.int32, device="cuda")
    table[:, :c["table"].shape[1]] = c["table"]
    c["table"] = table
    o = run_prefill(c, new, lens, 64)
    assert torch.equal(run_prefill(c, new, lens, 64), o)


@pytest.mark.parametrize("prefix", [0, 150])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_attention_into_its_own_queries(prefix, cap):
    """out = q, for one part of the key axis and for several."""
    for new, cached in (([300, 5], [0, 40]), ([20], [3000])):
        c, lens = prefill_case(new, cached, 14, 2, 64, 16, F16, prefix=prefix, cap=cap)
        want = run_prefill(c, new, lens, 64, cap, prefix=prefix)
        from ddq_b200 import paged
        paged.prefill_attention(c["q"], c["kp"], c["vp"], c["table"], c["cu"], c["lens"], 0.125,
                                softcap=cap, prefix_pages=c["prefix"], prefix_len=prefix,
                                out=c["q"])
        assert torch.equal(c["q"], want)
    lens = [3000, 1, 0, 40, 700]
    c = decode_case(lens, prefix, 14, 2, 64, 16, F16)
    want = run_decode(c, lens, prefix, 64, cap)
    paged.decode_attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], 0.125,
                           prefix_pages=c["prefix"], prefix_len=prefix, softcap=cap, out=c["q"])
    assert torch.equal(c["q"], want)
