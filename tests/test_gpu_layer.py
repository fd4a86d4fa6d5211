"""GPU: rotary positions, the paged 4-bit cache, page bookkeeping and attention over the
cache, each against its 64-bit restatement (oracle/layer.py).

Tolerances.  u16 = 2^-11 is half a step of fp16, u32 = 2^-24 of fp32.
* cache codes, scales, minima, slots, tables: equal.
* gather: fp16(c s + m) of an fp32 fma: |err| <= (u16 + u32) |x| + 2^-25 (half the least
  fp16 step).
* rope: fp32 sine / cosine within 4 u32 + the reduced angle's 2^-24 of a half turn (pi u32),
  two products and a sum: |err| <= 12 u32 (|a| + |b|), then u16 |y| + 2^-25.
* attention: let A = |scale| sum |q| (15 s + |m|) bound the terms of a score.  The fp32 score
  sums D products and folds s and m in, each rounded at the size of A: off by e = (D + 8) u32
  A, plus the hardware exponential's 2 ulp (2^-22).  A softmax weight p_t is then off by
  d_t = e_t + sum_t p_t e_t (its own error and the sum's), relative.  The weights p s are
  rounded to fp16: u16 relative, or, below fp16's normal range, half a subnormal step 2^-25
  of the softmax reference, which is at most the largest p s.  The weights meet c - 8, and
  p meets m + 8 s, in fp32 (rounded once, u32).  Hence
  |err| <= sum_t (p_t ((u16 + d_t) s |c - 8| + (d_t + u32) |m + 8 s|) + 2^-25 max(p s) 15)
           + u16 |o| + 2^-25.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import awq_b200
from oracle import layer as L

pytestmark = pytest.mark.gpu
U16, U32, TINY = 2.0 ** -11, 2.0 ** -24, 2.0 ** -25


@pytest.fixture(autouse=True)
def _status(cuda):
    awq_b200.device_status()
    yield


@pytest.fixture(params=["extension", "ctypes"])
def glue(request, monkeypatch):
    """The C++ host glue, and the Python path that stands in for it where it is not built."""
    if request.param == "ctypes":
        monkeypatch.setattr(awq_b200, "_ext", None)
    else:
        assert awq_b200._ext is not None


def dev(x, dtype=None):
    t = torch.as_tensor(np.asarray(x), device="cuda")
    return t if dtype is None else t.to(dtype)


# ---- rope ---------------------------------------------------------------------------------
ROPE = [  # T, q heads, k heads, D, sections, interleaved
    (1, 28, 4, 128, (64,), False), (5, 28, 4, 128, (16, 24, 24), False),
    (3, 7, 1, 128, (16, 24, 24), True), (2, 4, 2, 64, (5, 7, 3), True),
    (7, 3, 1, 80, (8, 16, 8), False), (4, 1, 0, 16, (1,), False), (2, 2, 2, 512, (100, 156), False),
]


@pytest.mark.parametrize("T,H,Hk,D,sections,inter", ROPE)
@pytest.mark.parametrize("pos_type", [torch.int64, torch.int32])
def test_rope(cuda, T, H, Hk, D, sections, inter, pos_type):
    rng = np.random.default_rng(T * 100 + D)
    half = sum(sections)
    x = rng.standard_normal((T, H + Hk, D)).astype(np.float16)
    pos = rng.integers(0, 2_000_000, (len(sections), T))
    pos[:, 0] = [0, -5, 2 ** 31 - 1, 1][:len(sections)]
    inv = (1e6 ** (-np.arange(half) / half)).astype(np.float32)
    fused = dev(x)
    q, k = fused[:, :H], fused[:, H:]
    oq, ok = awq_b200.rope_axes(q, k, dev(pos).to(pos_type), dev(inv), sections, inter)
    ref = L.rope(x, pos, inv, sections, inter)
    size = np.abs(x.astype(np.float64))
    size[..., :2 * half] += np.roll(size[..., :2 * half], half, -1)
    got = torch.cat([oq, ok], 1).double().cpu().numpy()
    assert (np.abs(got - ref) <= 12 * U32 * size + U16 * np.abs(ref) + TINY).all()
    assert torch.equal(fused, dev(x))
    # in place, on the views
    awq_b200.rope_axes(q, k, dev(pos).to(pos_type), dev(inv), sections, inter, out_q=q, out_k=k)
    assert torch.equal(q, oq) and torch.equal(k, ok)


def test_rope_unaligned_and_transposed(cuda):
    """An odd start and a head-major layout take the scalar path, with the same values."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 4, 64)).astype(np.float16)
    pos = dev(rng.integers(0, 5000, (1, 6)))
    inv = dev((1e4 ** (-np.arange(32) / 32)).astype(np.float32))
    want = awq_b200.rope_axes(dev(x), dev(x[:, :2]), pos, inv, (32,))
    buf = torch.zeros(6 * 4 * 64 + 1, dtype=torch.float16, device="cuda")
    odd = buf[1:].view(6, 4, 64)
    odd.copy_(dev(x))
    heads = dev(x).transpose(0, 1).contiguous().transpose(0, 1)
    for q in (odd, heads):
        got = awq_b200.rope_axes(q, q[:, :2], pos[0], inv, (32,))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rope_refuses_outputs_that_share_memory(cuda, glue):
    """out_q and out_k may be columns of the same rows, and nothing else in common."""
    x = torch.randn((6, 5, 64), device="cuda").half()
    q, k = x[:, :4], x[:, 4:]
    pos, inv = torch.arange(6, device="cuda"), torch.ones(32, device="cuda")
    buf = torch.zeros((7, 5, 64), dtype=torch.float16, device="cuda")
    want = awq_b200.rope_axes(q, k, pos, inv, (32,))
    got = awq_b200.rope_axes(q, k, pos, inv, (32,), out_q=buf[:6, :4], out_k=buf[:6, 4:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = awq_b200.rope_axes(q, k, pos, inv, (32,), out_q=buf[:6, 1:], out_k=buf[:6, :1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for oq, ok in ((buf[:6, :4], buf[:6, 3:4]), (buf[:6, :4], buf[1:, :1]), (buf[:6, 1:], buf[:6, 1:2])):
        with pytest.raises(ValueError, match="out_q overlaps out_k"):
            awq_b200.rope_axes(q, k, pos, inv, (32,), out_q=oq, out_k=ok)


def test_outputs_whose_rows_share_memory_are_refused(cuda, glue):
    """An expanded output has one row for many; any order of tokens and heads is fine."""
    x = torch.randn((6, 4, 64), device="cuda").half()
    pos, inv = torch.arange(6, device="cuda"), torch.ones(32, device="cuda")
    want = awq_b200.rope_axes(x, x, pos, inv, (32,))[0]
    heads = torch.zeros((4, 6, 64), dtype=torch.float16, device="cuda").transpose(0, 1)
    assert torch.equal(awq_b200.rope_axes(x, x, pos, inv, (32,), out_k=heads)[1], want)
    cache = awq_b200.KV4Cache.allocate(6, 2, 64, 16)
    awq_b200.kv4_append(x[:, :2], x[:, 2:], torch.arange(6, device="cuda") * 16, cache)
    table = torch.arange(6, dtype=torch.int32, device="cuda")[:, None]
    lens = torch.ones(6, dtype=torch.int32, device="cuda")
    want = awq_b200.kv4_attention(x, cache, table, lens)
    assert torch.equal(awq_b200.kv4_attention(x, cache, table, lens, out=heads), want)
    for o in (heads[:1].expand(6, 4, 64), heads[:, :1].expand(6, 4, 64)):
        with pytest.raises(ValueError, match="share no element"):
            awq_b200.rope_axes(x, x, pos, inv, (32,), out_q=o)
        with pytest.raises(ValueError, match="share no element"):
            awq_b200.kv4_attention(x, cache, table, lens, out=o)


# ---- append and gather --------------------------------------------------------------------
def sample(rng, T, H, D):
    """Rows with wide, narrow, constant, subnormal and large groups."""
    x = rng.standard_normal((T, H, D)) * np.exp(rng.uniform(-3, 3, (T, H, 1)))
    x[rng.random((T, H)) < 0.1] = 0.25
    x[rng.random((T, H)) < 0.1] *= 2.0 ** -22
    x[rng.random((T, H)) < 0.1] *= 1000
    tie = rng.random((T, H)) < 0.2                    # quotients that fall on ties
    x[tie] = rng.integers(0, 31, (int(tie.sum()), D)) / 2.0 - 3
    return x.clip(-65504, 65504).astype(np.float16)


CACHES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.mark.parametrize("D,group", CACHES)
@pytest.mark.parametrize("page,H,T", [(16, 1, 1), (16, 4, 37), (64, 3, 50), (1024, 2, 9)])
def test_append_bytes_and_gather(cuda, D, group, page, H, T):
    rng = np.random.default_rng(D + group + T)
    k, v = sample(rng, T, H, D), sample(rng, T, H, D)
    pages = T // page + 3
    slots = rng.permutation(pages * page)[:T]
    cache = awq_b200.KV4Cache.allocate(pages, H, D, page, group)
    cache.data.random_(0, 256)
    before = cache.data.cpu().numpy()
    want = before.copy()
    for t in range(T):
        L.write_slot(want, int(slots[t]), k[t], v[t], page, group)
    fused = dev(np.concatenate([k, v], 1))            # strided views
    awq_b200.kv4_append(fused[:, :H], fused[:, H:], dev(slots), cache)
    bad = np.argwhere(cache.data.cpu().numpy() != want)     # and nothing else changed
    assert len(bad) == 0, bad[:8].tolist()
    ask = np.concatenate([slots, [-1]])
    gk, gv = (x.double().cpu().numpy() for x in awq_b200.kv4_gather(cache, dev(ask)))
    rk, rv = L.read_slots(want, slots, D, page, group)
    for got, ref in ((gk, rk), (gv, rv)):
        assert (np.abs(got[:T] - ref) <= (U16 + U32) * np.abs(ref) + TINY).all()
        assert (got[T] == 0).all()
    assert awq_b200.device_status() == 0


def test_append_skips_and_non_finite(cuda):
    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((4, 2, 64)).astype(np.float16) for _ in range(2))
    k[0, 0, 3], v[0, 1, 40], k[3, 1, 0] = np.nan, np.inf, -np.inf
    cache = awq_b200.KV4Cache.allocate(2, 2, 64, 16, 32)
    awq_b200.kv4_append(dev(k), dev(v), dev(np.array([31, -1, -7, 0])), cache)
    want = np.zeros(tuple(cache.data.shape), np.uint8)
    for t, s in ((0, 31), (3, 0)):
        L.write_slot(want, s, k[t], v[t], 16, 32)
    gk, gv = awq_b200.kv4_gather(cache, dev(np.array([31, 0])))
    rk, rv = L.read_slots(want, [31, 0], 64, 16, 32)
    for got, ref in ((gk, rk), (gv, rv)):
        got = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        ok = ~np.isnan(ref)
        assert (np.abs(got - ref)[ok] <= (U16 + U32) * np.abs(ref)[ok] + TINY).all()
    assert np.isnan(gk[0, 0, :32].cpu().numpy()).all() and not np.isnan(gk[0, 0, 32:].cpu().numpy()).any()
    assert awq_b200.device_status() == 0
    awq_b200.kv4_append(dev(k), dev(v), dev(np.array([-1, 32, -1, 10 ** 12])), cache)
    again = awq_b200.kv4_gather(cache, dev(np.array([31, 0])))
    assert torch.equal(again[0].view(torch.int16), gk.view(torch.int16))
    assert awq_b200.device_status() == 2             # slots past the cache are reported


# ---- pages --------------------------------------------------------------------------------
def pages_state(rng, R, width, page, spare, max_new, refill=0.3):
    lens = rng.integers(0, width * page // 2, R)
    held = -(-lens // page)
    reset = rng.random(R) < refill
    new = rng.integers(0, max_new + 1, R)
    total = int(held.sum()) + spare
    ids = rng.permutation(total)
    table = np.full((R, width), -1)
    at = 0
    for r in range(R):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    free = np.full(total, -1)
    free[:spare] = ids[at:]
    lens = np.where(reset, 0, lens)
    return table, held, free, spare, lens, new, reset


def run_pages(table, held, free, count, lens, new, reset, page, max_tokens):
    st = [dev(x).int() for x in (table, held, free, [count], lens, new)]
    out = awq_b200.kv4_pages_step(*st, page_size=page, max_tokens=max_tokens,
                                  reset=None if reset is None else dev(reset))
    ref = L.pages_step(table, held, free, count, lens, new, page, max_tokens, reset)
    got = [st[0], st[1], st[2], st[3], *out]
    for name, g, w in zip(("table", "held", "free", "count", "slots", "positions", "cu_q",
                           "lens", "status"), got, ref):
        assert np.array_equal(g.cpu().numpy().reshape(np.shape(w)), w), name
    return ref


@pytest.mark.parametrize("R,width,page,max_new", [
    (1, 1, 16, 1), (1, 40, 16, 300), (7, 12, 16, 40), (64, 16, 64, 1), (511, 9, 32, 3),
    (513, 9, 32, 3), (2048, 6, 16, 20), (8192, 2, 16, 2), (3, 700, 1, 200)])
def test_pages_step(cuda, R, width, page, max_new):
    rng = np.random.default_rng(R)
    table, held, free, count, lens, new, reset = pages_state(
        rng, R, width, page, R * (max_new // page + 2) + 5, max_new)
    new = np.minimum(new, width * page - lens)
    ref = run_pages(table, held, free, count, lens, new, reset, page, int(new.sum()) + 3)
    assert ref[-1] == 0
    # the step after it, without replaced rows, exactly as many tokens as fit
    table, held, free, count, _, _, _, lens, _ = ref
    new = np.minimum(1, width * page - lens)
    assert run_pages(table, held, free, count, lens, new, None, page, int(new.sum()))[-1] == 0


def test_pages_step_refusals_change_nothing(cuda):
    rng = np.random.default_rng(2)
    table, held, free, count, lens, new, reset = pages_state(rng, 20, 8, 16, 3, 30, refill=0.0)
    lens, new = np.full(20, 17), np.full(20, 16)
    held[:] = 2
    short = run_pages(table, held, free, count, lens, new, None, 16, 400)[-1]
    assert short == 17
    assert run_pages(table, held, free, count, lens, new, None, 16, 319)[-1] == -1   # tokens
    new[3] = 8 * 16
    assert run_pages(table, held, free, count, lens, new, None, 16, 4000)[-1] == -1  # width
    new[3] = -1
    assert run_pages(table, held, free, count, lens, new, None, 16, 4000)[-1] == -1
    new[3], lens[5] = 1, -1
    assert run_pages(table, held, free, count, lens, new, None, 16, 4000)[-1] == -1
    lens[5], held[7] = 1, 9
    assert run_pages(table, held, free, count, lens, new, None, 16, 4000)[-1] == -1
    held[7] = 2
    assert run_pages(table, held, free, -1, lens, new, None, 16, 4000)[-1] == -1
    assert run_pages(table, held, free, len(free) + 1, lens, new, None, 16, 4000)[-1] == -1


# ---- attention ----------------------------------------------------------------------------
def make_cache(rng, lens, Hk, D, group, page, small=False):
    """A cache filled by the library's append; returns it, its table and the float64 K, V."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    cache = awq_b200.KV4Cache.allocate(pages, Hk, D, page, group)
    cache.data.fill_(0xFF)                             # unwritten params are NaN
    ids = rng.permutation(pages)
    table = np.full((len(lens), max(need + [1]) + 1), -1)
    kv, at = [], 0
    for r, n in enumerate(lens):
        table[r, :need[r]] = ids[at:at + need[r]]
        at += need[r]
        k = rng.standard_normal((n, Hk, D)) + 4 * (rng.random((1, Hk, D)) < 0.05)
        v = rng.standard_normal((n, Hk, D)) * np.exp(rng.uniform(-6, 1, (n, Hk, 1)))
        if small:
            v *= 2.0 ** -12
        slots = table[r, np.arange(n) // page] * page + np.arange(n) % page
        awq_b200.kv4_append(dev(k.astype(np.float16)), dev(v.astype(np.float16)), dev(slots), cache)
        kv.append((k, v, slots))
    data = cache.data.cpu().numpy()
    return cache, dev(table).int(), [L.read_slots(data, s, D, page, group) for _, _, s in kv], data, kv


def bound(q, K, V, ref, scale, data, slots, D, page, group):
    """The module docstring's bound for one request, [n, H, D]."""
    n, H, _ = q.shape
    Lk, Hk = K.shape[:2]
    out = np.zeros(ref.shape)
    G = D // group
    par = np.zeros((Lk, Hk, 2, G, 2))
    for t, slot in enumerate(slots):
        pg, at = divmod(int(slot), page)
        p = np.ascontiguousarray(data[pg, :, at // 16, 16 * D:]).view(np.float16)
        par[t] = p.reshape(Hk, 2, 16, G, 2)[:, :, at % 16].astype(np.float64)
    rep = lambda x: np.repeat(x, group, -1)
    ks, km, vs, vm = (rep(par[:, :, a, :, b]) for a in (0, 1) for b in (0, 1))
    for i in range(n):
        seen = Lk - n + i + 1
        if seen <= 0:
            continue
        for h in range(H):
            hk = h // (H // Hk)
            s = scale * (K[:seen, hk] @ q[i, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            size = abs(scale) * ((15 * ks[:seen, hk] + np.abs(km[:seen, hk])) @ np.abs(q[i, h]))
            e = (D + 8) * U32 * size + 2.0 ** -22
            d = e + (p @ e)                             # of a weight, and of the sum
            sc = vs[:seen, hk]
            mid = vm[:seen, hk] + 8 * sc
            c8 = np.abs(V[:seen, hk] - mid)             # s |c - 8|
            w = p[:, None] * sc
            sub = (2.0 ** -25) * w.max() * np.where(sc > 0, 15.0, 0).max(-1, keepdims=True)
            out[i, h] = (p[:, None] * ((U16 + d[:, None]) * c8 + (d[:, None] + U32) * np.abs(mid))
                         + sub).sum(0)
    return out + U16 * np.abs(ref) + TINY


def check_attention(rng, lens, qs, H, Hk, D, group, page, scale=None, small=False, pad=0):
    cache, table, KV, data, kv = make_cache(rng, lens, Hk, D, group, page, small)
    scale = D ** -0.5 if scale is None else scale
    cu = np.concatenate([[0], np.cumsum(qs)])
    q = rng.standard_normal((cu[-1] + pad, H, D)).astype(np.float16)
    out = torch.full((cu[-1] + pad, H, D), 7.5, dtype=torch.float16, device="cuda")
    decode = all(n == 1 for n in qs) and not pad
    got = awq_b200.kv4_attention(dev(q), cache, table, dev(lens).int(),
                                 None if decode else dev(cu).int(), 1 if decode else max(qs),
                                 scale, out)
    assert got is out
    assert awq_b200.device_status() == 0
    got = got.double().cpu().numpy()
    assert (got[cu[-1]:] == 7.5).all()                  # rows behind the last request
    for r in range(len(lens)):
        K, V = KV[r]
        rows = slice(cu[r], cu[r + 1])
        ref = L.attention(q[rows], K, V, scale)
        tol = bound(q[rows].astype(np.float64), K, V, ref, scale, data, kv[r][2], D, page, group)
        err = np.abs(got[rows] - ref)
        assert (err <= tol).all(), (r, float((err / tol).max()))
    if not decode:                                      # one at a time gives the same bits
        again = awq_b200.kv4_attention(dev(q), cache, table, dev(lens).int(), dev(cu).int(),
                                       max(qs), scale)
        assert torch.equal(again[:cu[-1]].cpu(), out[:cu[-1]].cpu())
        assert (again[cu[-1]:] == 0).all()


@pytest.mark.parametrize("D,group", CACHES)
@pytest.mark.parametrize("H,Hk", [(1, 1), (7, 1), (28, 4), (6, 2), (16, 1), (20, 2)])
def test_attention_decode_heads(cuda, D, group, H, Hk):
    check_attention(np.random.default_rng(H), [1, 33, 100], [1, 1, 1], H, Hk, D, group, 16)


@pytest.mark.parametrize("page", [16, 32, 64, 1024])
@pytest.mark.parametrize("lens", [[0], [1], [15, 16, 17, 31, 32, 33], [0, 1000, 0, 5], [2500]])
def test_attention_decode_lengths(cuda, page, lens):
    check_attention(np.random.default_rng(page), lens, [1] * len(lens), 14, 2, 128, 64, page)


@pytest.mark.parametrize("D,group", [(64, 32), (128, 128)])
def test_attention_small_values_and_scale(cuda, D, group):
    rng = np.random.default_rng(9)
    check_attention(rng, [300, 40], [1, 1], 4, 2, D, group, 32, small=True)
    check_attention(rng, [300, 40], [1, 1], 4, 2, D, group, 32, scale=2.0)
    check_attention(rng, [300, 40], [1, 1], 4, 2, D, group, 32, scale=-0.3)


@pytest.mark.parametrize("D,group,H,Hk", [(128, 128, 28, 4), (64, 32, 6, 2), (128, 32, 3, 3)])
@pytest.mark.parametrize("lens,qs", [([5], [5]), ([70, 33], [3, 17]), ([9, 4, 130], [0, 6, 65]),
                                     ([40, 40, 40], [1, 2, 40])])
def test_attention_chunks(cuda, D, group, H, Hk, lens, qs):
    check_attention(np.random.default_rng(len(lens)), lens, qs, H, Hk, D, group, 16, pad=3)


def test_attention_many_requests(cuda):
    """More requests than prefix entries, most of them short: items end inside warps."""
    rng = np.random.default_rng(11)
    R = 1500
    lens = rng.integers(0, 3, R) * rng.integers(0, 40, R)
    check_attention(rng, [int(x) for x in lens], [1] * R, 2, 1, 64, 64, 16)


def test_attention_skips_bad_pages_and_lengths(cuda):
    rng = np.random.default_rng(12)
    cache, table, KV, _, _ = make_cache(rng, [64, 64], 1, 64, 64, 16)
    q = rng.standard_normal((2, 4, 64)).astype(np.float16)
    lens = dev(np.array([64, 64])).int()
    table[0, 1] = -1                                    # tokens 16..31 are not there
    table[1, 3] = cache.num_pages
    got = awq_b200.kv4_attention(dev(q), cache, table, lens).double().cpu().numpy()
    assert awq_b200.device_status() == 2
    for r, keep in ((0, [*range(16), *range(32, 64)]), (1, list(range(48)))):
        K, V = (x[keep] for x in KV[r])
        ref = L.attention(q[r:r + 1], K, V, 0.125)
        assert np.abs(got[r:r + 1] - ref).max() <= 2e-3 * np.abs(V).max()
    table[0, 1] = 0
    got = awq_b200.kv4_attention(dev(q), cache, table, dev(np.array([10 ** 6, -3])).int())
    assert awq_b200.device_status() == 2
    assert (got[1] == 0).all()


def test_attention_nan_stays_in_seen_rows(cuda):
    """A NaN key or value makes the rows that see it NaN, and no other."""
    rng = np.random.default_rng(13)
    cache, table, _, _, kv = make_cache(rng, [40], 1, 64, 64, 16)
    k = torch.full((1, 1, 64), float("nan"), dtype=torch.float16, device="cuda")
    awq_b200.kv4_append(k, k, dev(kv[0][2][37:38]), cache)
    q = dev(rng.standard_normal((6, 2, 64)).astype(np.float16))
    got = awq_b200.kv4_attention(q, cache, table, dev(np.array([40])).int(),
                                 dev(np.array([0, 6])).int(), 6)
    bad = torch.isnan(got).flatten(1)
    assert bad[3:].all() and not bad[:3].any()


def test_attention_graph_and_streams(cuda):
    """Captured once, replayed with other lengths, and two graphs replayed at the same time."""
    rng = np.random.default_rng(14)
    lens = [200, 333]
    cache, table, KV, _, _ = make_cache(rng, lens, 2, 128, 128, 32)
    q = dev(rng.standard_normal((2, 14, 128)).astype(np.float16))
    kv_lens = dev(np.array(lens)).int()
    want = awq_b200.kv4_attention(q, cache, table, kv_lens)
    part = dev(np.array([57, 1])).int()
    want2 = awq_b200.kv4_attention(q, cache, table, part)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        for _ in range(2):
            live = kv_lens.clone()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                out = awq_b200.kv4_attention(q, cache, table, live)
            graphs.append((g, live, out))
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for lens_now, ref in ((kv_lens, want), (part, want2), (kv_lens, want)):
        for _, live, _ in graphs:
            live.copy_(lens_now)
        torch.cuda.synchronize()
        for _ in range(20):
            for st, (g, _, _) in zip((a, b), graphs):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, ref) for _, _, out in graphs)


@pytest.mark.parametrize("D,group,H,Hk", [(128, 128, 7, 1), (128, 64, 8, 2), (128, 32, 4, 4),
                                          (64, 64, 14, 2), (64, 32, 2, 1)])
@pytest.mark.parametrize("lens,qs,page", [([300], [300], 64), ([700, 90], [37, 90], 16),
                                          ([1030], [65], 32), ([64, 1500, 10], [64, 3, 10], 128),
                                          ([50, 129], [70, 129], 16)])
def test_attention_prompt_chunks(cuda, D, group, H, Hk, lens, qs, page):
    """Many query rows (tcgen05 kernel) beside few, steps that end inside blocks, more query
    tokens than cached ones."""
    check_attention(np.random.default_rng(sum(lens)), lens, qs, H, Hk, D, group, page, pad=2)


@pytest.mark.parametrize("D,group,H,Hk", [(128, 128, 7, 1), (128, 32, 4, 4), (64, 64, 16, 2),
                                          (64, 32, 1, 1)])
@pytest.mark.parametrize("rows", [255, 256, 257, 512, 513])
def test_attention_prompt_row_tiles(cuda, D, group, H, Hk, rows):
    """Chunks whose query rows end at, before and behind an item of 256 rows, beside a chunk
    and a token that take the other kernel."""
    G = H // Hk
    n = -(-rows // G)
    check_attention(np.random.default_rng(rows), [n + 45, 40, 9], [n, 3, 1], H, Hk, D, group, 32, pad=1)


@pytest.mark.parametrize("D,group", CACHES)
def test_attention_prompt_nan_and_lost_page(cuda, D, group):
    """300 query rows of a request: a page the table does not name, and a NaN key and value."""
    rng = np.random.default_rng(24)
    cache, table, KV, _, kv = make_cache(rng, [200], 1, D, group, 16)
    q = rng.standard_normal((150, 2, D)).astype(np.float16)
    lens, cu = dev(np.array([200])).int(), dev(np.array([0, 150])).int()
    page1 = int(table[0, 1])
    table[0, 1] = -1
    got = awq_b200.kv4_attention(dev(q), cache, table, lens, cu, 150).double().cpu().numpy()
    assert awq_b200.device_status() == 2
    keep = [*range(16), *range(32, 200)]
    K, V = (x[keep] for x in KV[0])
    # row i sees the tokens up to 50 + i
    ref = np.stack([L.attention(q[i:i + 1], K[:35 + i], V[:35 + i], D ** -0.5)[0] for i in range(150)])
    assert np.abs(got - ref).max() <= 2e-3 * np.abs(V).max()
    table[0, 1] = page1
    k = torch.full((1, 1, D), float("nan"), dtype=torch.float16, device="cuda")
    awq_b200.kv4_append(k, k, dev(kv[0][2][150:151]), cache)
    got = awq_b200.kv4_attention(dev(q), cache, table, lens, cu, 150)
    bad = torch.isnan(got).flatten(1)
    assert bad[100:].all() and not bad[:100].any()


def test_attention_requests_that_share_rows(cuda):
    """cu_q that goes back and forth lists more work than the call admits: the kernels count
    it, compute nothing and say so.  R requests of n rows and 2^19 tokens each."""
    R, n, width, page = 8192, 800, 512, 1024
    cache = awq_b200.KV4Cache.allocate(1, 1, 64, page, 64)
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda").expand(R, width)
    lens = torch.full((R,), width * page, dtype=torch.int32, device="cuda")
    cu = (torch.arange(R + 1, device="cuda") % 2 * n).int()
    q = torch.zeros((n, 1, 64), dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    awq_b200.kv4_attention(q, cache, table.contiguous(), lens, cu, 4, out=out)
    assert awq_b200.device_status() == 2
    assert (out == 7.0).all()


def test_attention_prompt_scale_and_small_values(cuda):
    rng = np.random.default_rng(21)
    for kw in (dict(small=True), dict(scale=2.0), dict(scale=-0.3), dict(scale=0.0)):
        check_attention(rng, [200], [100], 4, 2, 128, 64, 32, **kw)


def test_attention_prompt_bad_pages_and_nan(cuda):
    rng = np.random.default_rng(22)
    cache, table, KV, _, kv = make_cache(rng, [200], 1, 128, 64, 16)
    q = rng.standard_normal((90, 2, 128)).astype(np.float16)
    lens, cu = dev(np.array([200])).int(), dev(np.array([0, 90])).int()
    page1 = int(table[0, 1])
    table[0, 1] = -1
    got = awq_b200.kv4_attention(dev(q), cache, table, lens, cu, 90).double().cpu().numpy()
    assert awq_b200.device_status() == 2
    keep = [*range(16), *range(32, 200)]
    K, V = (x[keep] for x in KV[0])
    ref = L.attention(q, K, V, 128 ** -0.5)
    assert np.abs(got - ref).max() <= 2e-3 * np.abs(V).max()
    table[0, 1] = page1                                 # rows 40.. see token 150, others do not
    k = torch.full((1, 1, 128), float("nan"), dtype=torch.float16, device="cuda")
    awq_b200.kv4_append(k, k, dev(kv[0][2][150:151]), cache)
    got = awq_b200.kv4_attention(dev(q), cache, table, lens, cu, 90)
    bad = torch.isnan(got).flatten(1)
    assert bad[40:].all() and not bad[:40].any()


def test_attention_prompt_graph_with_other_lengths(cuda):
    rng = np.random.default_rng(23)
    lens = [300, 260]
    cache, table, KV, _, _ = make_cache(rng, lens, 2, 128, 128, 32)
    q = dev(rng.standard_normal((220, 4, 128)).astype(np.float16))
    live, cu = dev(np.array(lens)).int(), dev(np.array([0, 100, 220])).int()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = awq_b200.kv4_attention(q, cache, table, live, cu, 220)
    for new_lens, new_cu in (([300, 260], [0, 100, 220]), ([31, 260], [0, 1, 180]), ([0, 0], [0, 0, 220])):
        live.copy_(dev(np.array(new_lens)))
        cu.copy_(dev(np.array(new_cu)))
        want = awq_b200.kv4_attention(q, cache, table, live, cu, 220)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:new_cu[-1]], want[:new_cu[-1]])
    assert awq_b200.device_status() == 0


# ---- attention: value scales close together and far apart, and tokens of little weight -------
class Tokens:
    """One request's keys and values as the cache holds them, in float64, from its definition."""

    def __init__(self, k, v, group):
        self.group = group
        (kc, ks, km), (vc, vs, vm) = L.quantize(k, group), L.quantize(v, group)
        self.K, self.V = L.values(kc, ks, km), L.values(vc, vs, vm)
        rep = lambda x: np.repeat(x.astype(np.float64), group, -1)
        self.ks, self.km, self.vs, self.vm = rep(ks), rep(km), rep(vs), rep(vm)
        self.top = vs.astype(np.float64).max(-1).T      # [kv heads][tokens] largest value scale

    def cached(self, k, v, rng, page):
        """A cache with these tokens in shuffled pages, and its table."""
        n, Hk, D = k.shape
        need = -(-n // page)
        cache = awq_b200.KV4Cache.allocate(need + 1, Hk, D, page, self.group)
        table = rng.permutation(need + 1)[:need]
        slots = table[np.arange(n) // page] * page + np.arange(n) % page
        awq_b200.kv4_append(dev(k), dev(v), dev(slots), cache)
        return cache, dev(table[None]).int()

    def check(self, q, got, seen, lost, scale):
        """A token's rows q, got [H, D] that see `seen` tokens, against the docstring's bound,
        `lost` (of the largest p s) in the place of 2^-25."""
        H, D = q.shape
        q = q.astype(np.float64)
        ref = L.attention(q[None], self.K[:seen], self.V[:seen], scale)[0]
        for h in range(H):
            hk = h // (H // self.K.shape[1])
            K, ks, km, vs, vm = (x[:seen, hk] for x in (self.K, self.ks, self.km, self.vs, self.vm))
            s = scale * (K @ q[h])
            p = np.exp(s - s.max())
            p /= p.sum()
            e = (D + 8) * U32 * abs(scale) * ((15 * ks + np.abs(km)) @ np.abs(q[h])) + 2.0 ** -22
            d = (e + p @ e)[:, None]
            mid = vm + 8 * vs
            sub = lost * (p[:, None] * vs).max() * np.where(vs > 0, 15.0, 0).max(-1, keepdims=True)
            tol = (p[:, None] * ((U16 + d) * np.abs(self.V[:seen, hk] - mid) + (d + U32) * np.abs(mid))
                   + sub).sum(0) + U16 * np.abs(ref[h]) + TINY
            err = np.abs(got[h] - ref[h])
            assert (err <= tol).all(), (seen, h, float((err / tol).max()))


@pytest.mark.parametrize("D,group,H,Hk", [(128, 128, 7, 1), (128, 64, 8, 2), (128, 32, 4, 4),
                                          (64, 64, 14, 2), (64, 32, 2, 1)])
@pytest.mark.parametrize("spread", [0, 4])
def test_attention_prompt_values_of_one_size(cuda, D, group, H, Hk, spread):
    """Values whose scales lie within 2^7 of one another in every step of 128 / groups tokens,
    over 3000 cached tokens, so that most steps are all seen and take the tcgen05 kernel's
    shorter form."""
    rng = np.random.default_rng(D + group + spread)
    n = -(-300 * Hk // H)
    Lk = 3000 + n
    k = (rng.standard_normal((Lk, Hk, D)) + 4 * (rng.random((1, Hk, D)) < 0.05)).astype(np.float16)
    v = (rng.standard_normal((Lk, Hk, D)) * np.exp2(rng.uniform(0, spread, (Lk, Hk, 1)))).astype(np.float16)
    tok = Tokens(k, v, group)
    step = 128 * group // D
    steps = tok.top[:, :Lk // step * step].reshape(Hk, -1, step)
    assert (steps.max(-1) <= 128 * steps.min(-1)).all()
    cache, table = tok.cached(k, v, rng, 64)
    q = rng.standard_normal((n, H, D)).astype(np.float16)
    got = awq_b200.kv4_attention(dev(q), cache, table, dev([Lk]).int(), dev([0, n]).int(), n)
    assert awq_b200.device_status() == 0
    got = got.double().cpu().numpy()
    for i in (0, n // 2, n - 1):
        tok.check(q[i], got[i], Lk - n + i + 1, 2.0 ** -25, D ** -0.5)


def ladder(rng, n, Hk, D, group, q0, drop, sizes):
    """Keys whose scores against q = q0 in channel 0 fall below token 0's by `drop` [n] bits, and
    values with codes 0 (a group's first channel) and 15, at the scales `sizes` [n]."""
    bits = D ** -0.5 * np.log2(np.e) * q0
    k, v = np.zeros((n, Hk, D)), np.zeros((n, Hk, D))
    k[:, :, 0] = ((drop.max() + 1 - drop) / bits)[:, None]
    v[:] = 15 * sizes[:, None, None]
    v[:, :, ::group] = 0
    return k.astype(np.float16), v.astype(np.float16)


@pytest.mark.parametrize("D,group,H", [(128, 128, 7), (128, 32, 4), (64, 64, 8)])
@pytest.mark.parametrize("ratio", [100, 250])
def test_attention_prompt_one_token_weighs_most(cuda, D, group, H, ratio):
    """One token that takes nearly all the weight, one beside it without weight whose value
    scale is `ratio` times as large, and 4000 tokens 17 to 18 bits below the first: their sum
    counts 0.1 of its scale, and none may be lost against the large scale.  160 requests over
    the same pages, so that one CTA works through all tokens of the first."""
    rng = np.random.default_rng(ratio + D)
    R, n, Lk = 160, -(-256 // H), 4100
    drop = rng.uniform(17.2, 18.2, Lk)
    drop[0] = 0
    sizes = np.full(Lk, 2.0 ** -6)
    sizes[5] *= ratio
    k, v = ladder(rng, Lk, 1, D, group, 8.0, drop, sizes)
    tok = Tokens(k, v, group)
    assert tok.top[0].max() == ratio * tok.top[0].min()
    cache, table = tok.cached(k, v, rng, 64)
    q = np.zeros((R * n, H, D), np.float16)
    q[:, :, 0] = 8
    got = awq_b200.kv4_attention(dev(q), cache, table.expand(R, -1).contiguous(), dev([Lk] * R).int(),
                                 dev(n * np.arange(R + 1)).int(), n)
    got = got.double().cpu().numpy()
    for r, i in ((0, 0), (0, n - 1), (R - 1, n // 2)):
        tok.check(q[0], got[r * n + i], Lk - n + i + 1, 2.0 ** -25, D ** -0.5)


@pytest.mark.parametrize("D,group", [(64, 32), (128, 64), (128, 32)])
@pytest.mark.parametrize("n,H", [(1, 1), (3, 4), (37, 7)])
def test_attention_groups_of_unequal_scale(cuda, D, group, n, H):
    """The first group's value scales are 2^22 times the others', and every eighth token weighs
    2^0.55 times the rest, so that a weight rounded to the fourth of itself would show.  Where
    all tokens have one scale the softmax reference lies 2^7 below the largest p s: a weight is
    off by 2^-32 of that at most."""
    rng = np.random.default_rng(D + n)
    Lk = 300
    drop = np.where(np.arange(Lk) % 8 == 0, 0, 0.55)
    k, v = ladder(rng, Lk, 1, D, group, 8.0, drop, np.full(Lk, 2.0 ** -12))
    v[:, :, :group] = (v[:, :, :group].astype(np.float64) * 2.0 ** 22).astype(np.float16)
    tok = Tokens(k, v, group)
    assert (tok.vs[:, 0, :group] == 2.0 ** 10).all() and (tok.vs[:, 0, group:] == 2.0 ** -12).all()
    cache, table = tok.cached(k, v, rng, 64)
    q = np.zeros((n, H, D), np.float16)
    q[:, :, 0] = 8
    got = awq_b200.kv4_attention(dev(q), cache, table, dev([Lk]).int(), dev([0, n]).int(), n)
    got = got.double().cpu().numpy()
    for i in {0, n - 1}:
        tok.check(q[i], got[i], Lk - n + i + 1, 2.0 ** -32, D ** -0.5)


@pytest.mark.parametrize("n", [1, 3, 200])
@pytest.mark.parametrize("at", [3, 290])
def test_attention_nan_value_of_no_weight(cuda, n, at):
    """A seen token whose value is NaN makes its group NaN even where its weight is below
    fp32's range (0 * NaN), in full tiles and in the last one."""
    rng = np.random.default_rng(at)
    Lk, D, group = 300 + n, 128, 64
    k = np.zeros((Lk, 1, D), np.float16)
    k[:, :, 0] = 8
    k[at, :, 0] = -8                                     # 64 x 16 x 128^-0.5 = 90 nats: 130 bits
    v = rng.standard_normal((Lk, 1, D)).astype(np.float16)
    v[at, 0, 5] = np.nan
    tok = Tokens(k, v, group)
    cache, table = tok.cached(k, v, rng, 64)
    q = np.zeros((n, 1, D), np.float16)
    q[:, :, 0] = 64
    got = awq_b200.kv4_attention(dev(q), cache, table, dev([Lk]).int(), dev([0, n]).int(), n)
    got = torch.isnan(got).cpu().numpy()
    assert got[:, 0, :64].all() and not got[:, 0, 64:].any()


@pytest.mark.parametrize("width,pages,want", [(1 << 18, 7, (1 << 31) - 7), (1 << 18, 0, (1 << 31) - 1),
                                              ((1 << 18) + 1, 7, (1 << 31) - 1), (1 << 19, 0, (1 << 31) - 1)])
def test_pages_step_shortage_beyond_32_bits(cuda, width, pages, want):
    """8192 requests that need 2^18 pages or more each, which the table has room for: the
    shortage is reported as 2^31 - 1 at most, 2^32 of it included."""
    R = 8192
    table = torch.empty((R, width), dtype=torch.int32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    held, new = torch.zeros(R, **i32), torch.zeros(R, **i32)
    lens = torch.full((R,), width, **i32)
    free, count = torch.arange(7, **i32), torch.full((1,), pages, **i32)
    slots, pos, cu, new_lens, status = awq_b200.kv4_pages_step(table, held, free, count, lens, new, 1, 4)
    assert int(status) == want
    assert int(count) == pages and (held == 0).all() and torch.equal(free, torch.arange(7, **i32))
    assert (slots == -1).all() and (cu == 0).all() and torch.equal(new_lens, lens)


@pytest.mark.parametrize("D,group,H,Hk", [(128, 128, 7, 1), (128, 32, 7, 1), (64, 64, 2, 1)])
@pytest.mark.parametrize("n", [1, 5, 150])
def test_attention_long_context(cuda, D, group, H, Hk, n):
    """20000 cached tokens, values of one size: sums of many small weights, on both kernels."""
    rng = np.random.default_rng(n + D)
    Lk = 20000
    k = (rng.standard_normal((Lk, Hk, D)) + 4 * (rng.random((1, Hk, D)) < 0.05)).astype(np.float16)
    v = (0.7 * rng.standard_normal((Lk, Hk, D))).astype(np.float16)
    tok = Tokens(k, v, group)
    cache, table = tok.cached(k, v, rng, 64)
    q = rng.standard_normal((n, H, D)).astype(np.float16)
    got = awq_b200.kv4_attention(dev(q), cache, table, dev([Lk]).int(), dev([0, n]).int(), n)
    assert awq_b200.device_status() == 0
    got = got.double().cpu().numpy()
    for i in {0, n - 1}:
        tok.check(q[i], got[i], Lk - n + i + 1, 2.0 ** -25, D ** -0.5)


@pytest.mark.parametrize("n", [2, 60])
def test_cache_beyond_32_bits(cuda, n):
    """A cache of 9.7 GB whose requests lie on both sides of 2^32 bytes and at its end."""
    rng = np.random.default_rng(n)
    D, group, Hk, H, page, Lk = 128, 128, 2, 8, 64, 130
    pages = 9_700_000_000 // (Hk * page * (D + 8))
    cache = awq_b200.KV4Cache.allocate(pages, Hk, D, page, group)
    cache.data.fill_(0xFF)
    half = 2 ** 32 // (Hk * page * (D + 8))
    table = np.array([[half - 1, half, half + 1], [pages - 1, 0, pages - 2]])
    k, v = (rng.standard_normal((2, Lk, Hk, D)).astype(np.float16) for _ in range(2))
    slots = table[:, np.arange(Lk) // page] * page + np.arange(Lk) % page
    awq_b200.kv4_append(dev(k).flatten(0, 1), dev(v).flatten(0, 1), dev(slots).flatten(), cache)
    q = rng.standard_normal((2 * n, H, D)).astype(np.float16)
    got = awq_b200.kv4_attention(dev(q), cache, dev(table).int(), dev([Lk, Lk]).int(),
                                 dev([0, n, 2 * n]).int(), n).double().cpu().numpy()
    gk, gv = (x.double().cpu().numpy() for x in awq_b200.kv4_gather(cache, dev(slots[1])))
    for r in range(2):
        tok = Tokens(k[r], v[r], group)
        for i in {0, n - 1}:
            tok.check(q[r * n + i], got[r * n + i], Lk - n + i + 1, 2.0 ** -25, D ** -0.5)
    for a, ref in ((gk, tok.K), (gv, tok.V)):
        assert (np.abs(a - ref) <= (U16 + U32) * np.abs(ref) + TINY).all()
    assert awq_b200.device_status() == 0
