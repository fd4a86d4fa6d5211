"""CPU: what the operators between the products refuse before any launch, the cache's
geometry, the oracle's own consistency, and the C entry points' argument checks.  Device
tensors are stood in for by CPU ones (refused: there is no CPU fallback) and, for the C entry
points, by aligned addresses that are never read, since every call here is refused."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import awq_b200
from awq_b200 import _lib
from oracle import layer as L

INV, UNSUP, WS = _lib.AWQ_ERR_INVALID_ARG, _lib.AWQ_ERR_UNSUPPORTED, _lib.AWQ_ERR_WORKSPACE
P = 4096                                     # an aligned address


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(head_dim=256), dict(group_size=16),
                                dict(head_dim=64, group_size=128), dict(page_size=8),
                                dict(page_size=48), dict(page_size=2048)])
def test_cache_refuses_geometry(kw):
    args = dict(head_dim=128, page_size=64, group_size=64)
    args.update(kw)
    with pytest.raises(ValueError):
        awq_b200.KV4Cache.allocate(4, 2, device="cpu", **args)
    c = awq_b200.KV4Cache.allocate(4, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        awq_b200.KV4Cache(c.data[:, :, :2], 128, 64, 128)
    with pytest.raises(TypeError):
        awq_b200.KV4Cache(c.data.float(), 128, 64, 128)
    with pytest.raises(ValueError):
        awq_b200.KV4Cache.allocate(0, 2, 128, device="cpu")


def test_cache_geometry():
    lib = _lib.load()
    for D, g in ((64, 32), (64, 64), (128, 32), (128, 64), (128, 128)):
        for page in (16, 64, 1024):
            c = awq_b200.KV4Cache.allocate(3, 5, D, page, g, device="cpu")
            assert c.data.shape[3] == L.block_bytes(D, g)
            assert c.data[0].numel() == lib.awq_kv4_page_bytes(5, D, g, page) \
                == 5 * page * (D + 8 * D // g)
    assert lib.awq_kv4_page_bytes(1, 96, 32, 16) == 0


def test_cpu_tensors_are_refused():
    c = awq_b200.KV4Cache.allocate(4, 2, 64, device="cpu")
    x = torch.zeros((3, 2, 64), dtype=torch.float16)
    slots = torch.zeros(3, dtype=torch.int64)
    i32 = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: awq_b200.kv4_append(x, x, slots, c), lambda: awq_b200.kv4_gather(c, slots),
                 lambda: awq_b200.kv4_attention(x, c, torch.zeros((3, 2), dtype=torch.int32), i32),
                 lambda: awq_b200.rope_axes(x, x, slots, torch.zeros(32), (32,)),
                 lambda: awq_b200.kv4_pages_step(torch.zeros((3, 2), dtype=torch.int32), i32, i32,
                                                 i32[:1], i32, i32, 16, 4)):
        with pytest.raises(ValueError, match="CUDA only"):
            call()
    w = (torch.zeros((64, 8), dtype=torch.int32), torch.zeros((1, 8), dtype=torch.int32),
         torch.zeros((1, 64), dtype=torch.float16))
    with pytest.raises(ValueError, match="CUDA only"):
        awq_b200.gemm_epilogue(torch.zeros((1, 64), dtype=torch.float16), *w, 64)
    with pytest.raises(TypeError):
        awq_b200.rope_axes([1], x, slots, torch.zeros(32), (32,))


def _append(k=P, v=P, slots=P, T=4, cache=P, pages=4, H=2, D=64, g=64, page=16):
    return _lib.load().awq_kv4_append(k, 128, 64, v, 128, 64, slots, T, cache, pages, H, D, g, page, None)


def test_append_entry_refusals():
    assert _append(D=80) == UNSUP and _append(g=16) == UNSUP and _append(page=24) == UNSUP
    assert _append(g=128) == UNSUP and _append(page=8) == UNSUP and _append(page=2048) == UNSUP
    assert _append(pages=0) == INV and _append(H=0) == INV and _append(T=-1) == INV
    assert _append(k=None) == INV and _append(slots=None) == INV and _append(cache=None) == INV
    assert _append(k=P + 1) == INV and _append(slots=P + 4) == INV and _append(cache=P + 8) == INV
    assert _append(T=0, k=None, v=None, slots=None, cache=None) == 0
    assert "power of two" in (_append(page=24), _lib.load().awq_last_error().decode())[1]


def _gather(cache=P, T=4, slots=P, k=P, v=P, D=64):
    return _lib.load().awq_kv4_gather(cache, 4, 2, D, 64, 16, slots, T, k, v, None)


def test_gather_entry_refusals():
    assert _gather(D=32) == UNSUP and _gather(T=-2) == INV and _gather(cache=None) == INV
    assert _gather(k=P + 4) == INV and _gather(v=None) == INV and _gather(T=0, k=None, v=None) == 0


def test_gather_entry_refuses_outputs_its_stores_do_not_fit():
    """The kernel stores 16 bytes at a time."""
    for off in (2, 8):
        assert _gather(k=P + off) == INV and _gather(v=P + off) == INV
    assert "16-byte" in (_gather(k=P + 8), _lib.load().awq_last_error().decode())[1]


def _attention(q=P, q_ts=128, T=4, H=4, cache=P, Hk=2, D=64, table=P, stride=8, width=8, lens=P,
               cu=None, R=4, max_q=1, scale=0.1, out=P, o_ts=256, ws=P, nb=1 << 40, page=16):
    return _lib.load().awq_kv4_attention(q, q_ts, 64, T, H, cache, 4, Hk, D, 64, page, table, stride,
                                         width, lens, cu, R, max_q, scale, out, o_ts, 64, ws, nb, None)


def test_attention_entry_refusals():
    assert _attention(D=72) == UNSUP and _attention(H=3) == INV and _attention(H=0) == INV
    assert _attention(R=8193, T=8193) == UNSUP and _attention(max_q=0) == INV
    assert _attention(T=5) == INV and _attention(max_q=2) == INV          # no cu_q: one row each
    assert _attention(scale=float("inf")) == INV and _attention(scale=float("nan")) == INV
    assert _attention(stride=7) == INV and _attention(T=-1, R=-1) == UNSUP
    assert _attention(q=None) == INV and _attention(out=None) == INV and _attention(lens=None) == INV
    assert _attention(q=P + 8) == INV and _attention(q_ts=132) == INV and _attention(out=P + 4) == INV
    assert _attention(o_ts=130) == INV and _attention(cache=P + 8) == INV and _attention(table=None) == INV
    big = 1 << 26                                                          # tiles past 32 bits
    assert _attention(width=big, stride=big, R=64, T=64) == UNSUP
    assert _attention(R=0, T=0, q=None, out=None) == 0


def _pages(table=P, stride=8, width=8, held=P, free=P, cap=9, count=P, lens=P, new=P, R=3, page=16,
           slots=P, pos=P, T=5, cu=P, nl=P, st=P):
    return _lib.load().awq_kv4_pages_step(table, stride, width, held, free, cap, count, lens, new,
                                          None, R, page, slots, pos, T, cu, nl, st, None)


def test_pages_entry_refusals():
    assert _pages(R=8193) == UNSUP and _pages(R=-1) == UNSUP and _pages(stride=7) == INV
    assert _pages(page=0) == INV and _pages(T=-1) == INV and _pages(cap=-1) == INV
    for name in ("table", "held", "free", "count", "lens", "new", "slots", "pos", "cu", "nl", "st"):
        assert _pages(**{name: None}) == INV, name


def test_pages_and_attention_entries_refuse_misaligned_integers():
    for name in ("table", "held", "free", "count", "lens", "new", "pos", "cu", "nl", "st"):
        assert _pages(**{name: P + 2}) == INV, name
    assert _pages(slots=P + 4) == INV
    assert _attention(table=P + 2) == INV and _attention(lens=P + 1) == INV
    assert _attention(cu=P + 2) == INV
    assert "4-byte" in _lib.load().awq_last_error().decode()


def _rope(q=P, H=2, k=P, Hk=1, T=3, D=64, pos=P, is64=1, inv=P, sections=(32,), out_q=P, out_k=P):
    import ctypes
    sec = (ctypes.c_int32 * max(1, len(sections)))(*sections)
    return _lib.load().awq_rope_axes(q, 128, 64, H, k, 64, 64, Hk, T, D, pos, is64, 3, inv, sec,
                                     len(sections), 0, out_q, 128, 64, out_k, 64, 64, None)


def test_rope_entry_refusals():
    assert _rope(sections=()) == INV and _rope(sections=(1,) * 5) == INV and _rope(sections=(33,)) == INV
    assert _rope(sections=(0,)) == INV and _rope(sections=(-1, 5)) == INV and _rope(D=1024) == INV
    assert _rope(q=None) == INV and _rope(out_k=None) == INV and _rope(pos=None) == INV
    assert _rope(pos=P + 4) == INV and _rope(inv=P + 2) == INV and _rope(q=P + 1) == INV
    assert _rope(T=0) == 0 and _rope(H=0, Hk=0, q=None, k=None) == 0


def test_rows_of_one_tensor_apart():
    """What rope_axes asks of two views: their ranges meet, but they are different columns."""
    from awq_b200 import layer
    buf = torch.zeros((7, 5, 64), dtype=torch.float16)
    for a, b, apart in ((buf[:6, :4], buf[:6, 4:], True), (buf[:6, 4:], buf[:6, :4], True),
                        (buf[:6, :4], buf[1:, 4:], True), (buf[:6, :4], buf[:6, 3:4], False),
                        (buf[:6, :4], buf[1:, :1], False), (buf[:6, 1:], buf[:6, 1:2], False)):
        assert awq_b200._overlap(a, b) and layer._apart(a, b) is apart


def test_rows_that_share_no_element():
    """What rope_axes and kv4_attention ask of a given output."""
    from awq_b200 import layer
    buf = torch.zeros((6, 4, 64), dtype=torch.float16)
    for t in (buf, buf[:, 1:3], buf[::2], buf[:, ::2], buf[..., :32], buf[:1], buf[:, :1], buf[:0],
              buf.view(4, 6, 64).transpose(0, 1), buf[:1].expand(1, 4, 64)):
        assert layer._distinct(t), t.stride()
    for t in (buf[:1].expand(6, 4, 64), buf[:, :1].expand(6, 4, 64),
              buf.as_strided((6, 4, 64), (128, 64, 1)), buf.as_strided((6, 4, 64), (256, 32, 1))):
        assert not layer._distinct(t), t.stride()


def _epilogue(act=0, res=P, ldr=64, bias=P, out=P, N=64):
    return _lib.load().awq_gemm_f16_epilogue(P, 64, P, P, P, bias, act, res, ldr, out, N, 2, N, 64, 64,
                                             None, 0, None)


def test_epilogue_entry_refusals():
    assert _epilogue(act=-1) == INV and _epilogue(act=5) == INV and _epilogue(ldr=63) == INV
    assert _epilogue(res=P + 1) == INV and _epilogue(bias=P + 1) == INV and _epilogue(out=None) == INV
    assert _epilogue(N=60) == INV


# ---- the oracle --------------------------------------------------------------------------
@pytest.mark.parametrize("D,group", [(64, 32), (128, 32), (128, 128)])
def test_oracle_layout_round_trip(D, group):
    rng = np.random.default_rng(D + group)
    H, page, pages = 2, 32, 3
    k, v = (rng.standard_normal((7, H, D)).astype(np.float16) for _ in range(2))
    data = rng.integers(0, 256, (pages, H, page // 16, L.block_bytes(D, group)), dtype=np.uint8)
    slots = rng.permutation(pages * page)[:7]
    for t in range(7):
        L.write_slot(data, int(slots[t]), k[t], v[t], page, group)
    gk, gv = L.read_slots(data, slots, D, page, group)
    for got, x in ((gk, k), (gv, v)):
        assert np.array_equal(got, L.values(*L.quantize(x, group)))
        step = np.repeat(L.quantize(x, group)[1].astype(np.float64), group, -1)
        # half a step, plus what rounding the step to fp16 moves the fifteenth one
        assert (np.abs(got - x) <= step * (0.5 + 15 * 2.0 ** -11) + 2.0 ** -25).all()


def test_oracle_words_cover_every_channel():
    for D in (64, 128):
        k = {(o, s) for o, s in (L._k_at(D, c) for c in range(D))}
        v = {(o, s) for odd in (0, 1) for o, s in (L._v_at(D, c, odd) for c in range(D))}
        assert len(k) == D and max(o for o, _ in k) == D // 2 - 1
        assert len(v) == 2 * D and max(o for o, _ in v) == D - 1


def test_oracle_pages_give_and_take_back():
    table, held = np.full((2, 3), -1), np.zeros(2, int)
    st = L.pages_step(table, held, np.arange(6), 6, [0, 0], [17, 16], 16, 40)
    assert st[0].tolist() == [[5, 4, -1], [3, -1, -1]] and st[3] == 3 and st[-1] == 0
    assert st[4][:18].tolist() == [*range(80, 96), 64, 48] and st[4][33] == -1
    again = L.pages_step(st[0], st[1], st[2], st[3], [0, 16], [17, 0], 16, 40, [True, False])
    assert again[0].tolist() == st[0].tolist() and again[3] == 3 and again[2].tolist() == st[2].tolist()
