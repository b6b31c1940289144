"""CPU tests of the paged KV-cache operators: what the C ABI and the Python
entry points refuse before they touch a GPU (pointers are placeholders that are
never dereferenced), and the plain reference of the plan against itself."""
import ctypes

import pytest
import torch

import paged_reference as ref
from ddq_b200 import _lib, paged
from ddq_b200.build import build

A, U = 256, 264            # 16-byte aligned, misaligned
OK, INVALID, SHAPE, ALIGN = 0, 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def cache(k=A, v=A, P=10, ps=16, hkv=2, d=64, strides=None, dtype=1):
    st = strides or (hkv * ps * d, ps * d, d)
    return ctypes.byref(_lib.PagedCache(k, v, P, ps, hkv, d, *st, dtype))


def test_plan_step_refusals(lib):
    def plan(cached=A, table=A, stride=8, width=8, free=A, nfree=4, head=A, ps=16, prefix=0,
             slots=A, head_out=A + 16, R=2, T=5):
        return lib.ddq_plan_step(cached, A, table, stride, width, free, nfree, head, ps, prefix,
                                 A, A, slots, A, A, head_out, R, T, None)
    assert plan(R=0) == SHAPE and plan(T=-1) == SHAPE and plan(R=8193) == SHAPE
    assert plan(width=0) == SHAPE and plan(stride=7) == SHAPE
    assert plan(ps=8) == SHAPE and plan(ps=48) == SHAPE and plan(ps=512) == SHAPE
    assert plan(prefix=-1) == SHAPE and plan(nfree=-1) == SHAPE and plan(T=2 ** 31) == SHAPE
    assert plan(cached=None) == INVALID and plan(table=None) == INVALID
    assert plan(slots=None) == INVALID and plan(free=None) == INVALID
    assert plan(head_out=None) == INVALID
    assert plan(head=A, head_out=A) == INVALID      # read by every CTA, written by one


def test_rope_kv_refusals(lib):
    def rope(qkv=A, stride=18 * 64, c=None, cos=A, q=A, T=3, hq=14, max_pos=10):
        return lib.ddq_paged_rope_kv(qkv, stride, c or cache(), cos, A, max_pos, A, A, q, T, hq,
                                     None)
    assert rope(T=0) == OK
    assert rope(T=-1) == SHAPE and rope(hq=0) == SHAPE and rope(max_pos=-1) == SHAPE
    assert rope(stride=18 * 64 - 8) == SHAPE
    assert rope(qkv=None) == INVALID and rope(cos=None) == INVALID and rope(q=None) == INVALID
    assert rope(qkv=U) == ALIGN and rope(q=U) == ALIGN and rope(cos=U) == ALIGN
    assert rope(stride=18 * 64 + 4) == ALIGN
    assert rope(c=cache(k=None)) == INVALID and rope(c=cache(dtype=2)) == INVALID
    assert rope(c=cache(ps=24)) == SHAPE and rope(c=cache(d=96)) == SHAPE
    assert rope(c=cache(P=0)) == SHAPE and rope(c=cache(hkv=0)) == SHAPE
    assert rope(c=cache(k=U)) == ALIGN and rope(c=cache(strides=(2052, 1024, 64))) == ALIGN
    # pages that share rows must not be written
    assert rope(c=cache(strides=(0, 16 * 64, 64))) == SHAPE
    assert rope(c=cache(strides=(16 * 64, 16 * 64, 64))) == SHAPE


def test_attention_refusals(lib):
    def pre(q=A, ts=14 * 64, hs=64, c=None, table=A, stride=8, width=8, cu=A, lens=A, scale=0.1,
            cap=0.0, out=A, ots=14 * 64, ohs=64, T=3, R=2, hq=14, prefix=None, plen=0):
        return lib.ddq_paged_prefill_attention(q, ts, hs, c or cache(), table, stride, width, cu,
                                               lens, None, prefix, plen, None, scale, cap, out, ots, ohs, T, R,
                                               hq, None, 0, None)

    def dec(q=A, ts=14 * 64, hs=64, c=None, table=A, stride=8, width=8, prefix=None, plen=0,
            lens=A, scale=0.1, cap=0.0, out=A, ots=14 * 64, ohs=64, T=3, hq=14):
        return lib.ddq_paged_decode_attention(q, ts, hs, c or cache(), table, stride, width, lens,
                                              prefix, plen, None, scale, cap, out, ots, ohs, T,
                                              hq, None, 0, None)
    for f in (pre, dec):
        assert f(T=0) == OK and f(T=-1) == SHAPE
        assert f(hq=15) == SHAPE and f(hq=0) == SHAPE and f(width=0) == SHAPE
        assert f(stride=7) == SHAPE
        assert f(q=None) == INVALID and f(out=None) == INVALID and f(lens=None) == INVALID
        assert f(table=None) == INVALID
        assert f(scale=float("nan")) == INVALID and f(scale=float("inf")) == INVALID
        assert f(cap=-1.0) == INVALID and f(cap=float("inf")) == INVALID
        assert f(q=U) == ALIGN and f(out=U) == ALIGN and f(ts=900) == ALIGN
        assert f(ohs=68, ots=2000) == ALIGN
        assert f(ots=64) == SHAPE and f(ohs=0) == SHAPE     # rows of out that overlap
        assert f(c=cache(ps=8)) == SHAPE and f(c=cache(d=80)) == SHAPE
        assert f(c=cache(dtype=0)) == INVALID
        assert f(plen=-1) == SHAPE and f(plen=5) == INVALID     # no prefix pages
        # positions that 32 bits cannot hold
        assert f(width=2 ** 27, stride=2 ** 27) == SHAPE
        assert f(width=2 ** 26, stride=2 ** 26, prefix=A, plen=2 ** 30) == SHAPE
    assert pre(R=0) == OK and pre(R=-1) == SHAPE and pre(cu=None) == INVALID


def test_python_entry_points_want_cuda_tensors():
    """On CPU tensors every entry point raises before it reaches the library."""
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 4, dtype=torch.int32)
    kv = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    q = torch.zeros(2, 14, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="plan_step: cached"):
        paged.plan_step(i, i, t, i, 16, 4)
    with pytest.raises(RuntimeError, match="rope_kv_write: k_pages"):
        paged.rope_kv_write(q.reshape(2, -1), kv, kv, q, q, i, i, 14, 2, 64)
    with pytest.raises(RuntimeError, match="prefill_attention: k_pages"):
        paged.prefill_attention(q, kv, kv, t, i, i, 0.1)
    with pytest.raises(RuntimeError, match="decode_attention: k_pages"):
        paged.decode_attention(q, kv, kv, t, i, 0.1)


def test_plan_reference_by_hand():
    table, cu, lens, slots, pos, seqs, at = ref.plan_reference(
        [3, 16, 0], [2, 1, 0], [[5, -1], [7, -1], [-1, -1]], [9, 8], 16, 5, 0, 100)
    assert table == [[5, -1], [7, 9], [-1, -1]] and cu == [0, 2, 3, 3] and lens == [5, 17, 0]
    assert slots == [83, 84, 144, -1, -1] and pos == [103, 104, 116, 0, 0]
    assert seqs == [0, 0, 1, -1, -1] and at == 1


def test_plan_step_refuses_outputs_over_what_other_blocks_read(lib):
    """Every block reads all lengths while the first writes: lens in the place of cached
    (or of new_tokens) gave slots and positions too large by the new tokens."""
    R, T, width, stride, nfree = 3, 5, 8, 16, 4
    size = dict(cached=4 * R, new=4 * R, free=4 * nfree, head=4, cu=4 * R + 4, lens=4 * R,
                slots=8 * T, pos=8 * T, seq=4 * T, head_out=4)
    home = {name: (1 << 20) + 0x1000 * i for i, name in enumerate([*size, "table"])}

    def plan(**moved):
        p = {**home, **moved}
        return lib.ddq_plan_step(p["cached"], p["new"], p["table"], stride, width, p["free"],
                                 nfree, p["head"], 16, 0, p["cu"], p["lens"], p["slots"],
                                 p["pos"], p["seq"], p["head_out"], R, T, None)
    written = ("cu", "lens", "slots", "pos", "seq", "head_out")
    for name in written:
        for other in size:
            if other != name:   # at the same place; the ends overlapping by a word
                assert plan(**{name: home[other]}) == INVALID
                assert plan(**{name: home[other] + size[other] - 4}) == INVALID
                assert plan(**{name: home[other] - size[name] + 4}) == INVALID
    for name in size:           # a table row; its last word; the row before its first word
        for row in range(R):
            at = home["table"] + 4 * stride * row
            assert plan(**{name: at}) == INVALID
            assert plan(**{name: at + 4 * width - 4}) == INVALID
            assert plan(**{name: at - size[name] + 4}) == INVALID


def test_index_arrays_off_their_natural_alignment_are_refused(lib):
    """An int64 read at a multiple of 4 (an int32 at one of 2) would fault on the device."""
    four, two = (1 << 20) + 4, (1 << 20) + 2
    names = ("cached", "new", "table", "free", "head", "cu", "lens", "slots", "pos", "seq",
             "head_out")
    home = {name: (2 << 20) + 0x1000 * i for i, name in enumerate(names)}

    def plan(**moved):
        p = {**home, **moved}
        return lib.ddq_plan_step(p["cached"], p["new"], p["table"], 8, 8, p["free"], 4, p["head"],
                                 16, 0, p["cu"], p["lens"], p["slots"], p["pos"], p["seq"],
                                 p["head_out"], 3, 5, None)
    for name in names:
        assert plan(**{name: two}) == ALIGN
    assert plan(slots=four) == ALIGN and plan(pos=four) == ALIGN

    def rope(slots=A, pos=A):
        return lib.ddq_paged_rope_kv(A, 18 * 64, cache(), A, A, 10, slots, pos, A, 3, 14, None)
    assert rope(slots=four) == ALIGN and rope(pos=four) == ALIGN

    def pre(table=A, cu=A, lens=A, bidir=None, prefix=None, plen=0, slopes=None):
        return lib.ddq_paged_prefill_attention(A, 14 * 64, 64, cache(), table, 8, 8, cu, lens,
                                               bidir, prefix, plen, slopes, 0.1, 0.0, A, 14 * 64,
                                               64, 3, 2, 14, None, 0, None)

    def dec(table=A, lens=A, prefix=None, plen=0, slopes=None):
        return lib.ddq_paged_decode_attention(A, 14 * 64, 64, cache(), table, 8, 8, lens, prefix,
                                              plen, slopes, 0.1, 0.0, A, 14 * 64, 64, 3, 14,
                                              None, 0, None)
    for f in (pre, dec):
        assert f(table=two) == ALIGN and f(lens=two) == ALIGN and f(slopes=two) == ALIGN
        assert f(prefix=two, plen=5) == ALIGN
    assert pre(cu=two) == ALIGN and pre(bidir=two) == ALIGN
