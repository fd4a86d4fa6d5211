"""64-bit restatement of the operators between the products -- TEST INFRASTRUCTURE ONLY.

numpy, from the definitions in include/awq_b200.h: rotary positions with several axes, the
4-bit cache (quantization, byte layout, page bookkeeping), causal attention over it, and the
product's bias / activation / residual epilogue.
"""
from __future__ import annotations

import math

import numpy as np


# ---- rotary positions -------------------------------------------------------------------
def axis_of(i: int, sections, interleaved: bool) -> int:
    if interleaved:
        a = i % len(sections)
        return a if i // len(sections) < sections[a] else 0
    a = 0
    while i >= sections[a]:
        i -= sections[a]
        a += 1
    return a


def rope(x, positions, inv_freq, sections, interleaved=False):
    """x [T, H, D] -> float64; positions [axes, T]."""
    x = np.asarray(x, dtype=np.float64)
    y = x.copy()
    half = sum(sections)
    for i in range(half):
        th = np.asarray(positions[axis_of(i, sections, interleaved)], np.float64) * float(inv_freq[i])
        c, s = np.cos(th)[:, None], np.sin(th)[:, None]
        y[..., i] = x[..., i] * c - x[..., i + half] * s
        y[..., i + half] = x[..., i + half] * c + x[..., i] * s
    return y


# ---- the 4-bit cache --------------------------------------------------------------------
def quantize(x, group: int):
    """fp16 [..., D] -> codes uint8 [..., D], scale and minimum fp16 [..., D / group]."""
    x = np.asarray(x, np.float16)
    g = x.astype(np.float64).reshape(*x.shape[:-1], -1, group)
    finite = np.isfinite(g).all(-1)
    gz = np.where(np.isfinite(g), g, 0.0)
    lo, hi = gz.min(-1) + 0.0, gz.max(-1) + 0.0     # -0 is stored as +0
    s = ((hi - lo) / 15).astype(np.float16)
    sd = s.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(sd > 0, np.rint((gz - lo[..., None]) / sd), 0.0)
    c = np.where(finite[..., None], np.clip(c, 0, 15), 0).astype(np.uint8)
    s = np.where(finite, s, np.float16(np.nan)).astype(np.float16)
    m = np.where(finite, lo, np.nan).astype(np.float16)
    return c.reshape(x.shape), s, m


def values(codes, s, m):
    """float64 code * scale + minimum."""
    g = codes.shape[-1] // s.shape[-1]
    return (codes.astype(np.float64) * np.repeat(s.astype(np.float64), g, -1)
            + np.repeat(m.astype(np.float64), g, -1))


def block_bytes(D: int, group: int) -> int:
    return 16 * D + 128 * (D // group)


def _k_at(D: int, ch: int):
    """(byte in a token's K row, shift) of a channel."""
    w, j, t = min(D // 32, 4), ch // 32, ch // 8 % 4
    word = (j // w) * 4 * w + t * w + j % w
    return 4 * word + (ch % 8) // 2, 4 * (ch % 2)


def _v_at(D: int, ch: int, odd: int):
    """(byte in a token pair's V row, shift) of a channel of its even or odd token."""
    w, i, h = min(D // 32, 4), ch // 32, ch // 4 % 8
    word = (i // w) * 8 * w + h * w + i % w
    return 4 * word + 2 * odd + (ch % 4) // 2, 4 * (ch % 2)


def write_slot(data, slot: int, k, v, page: int, group: int) -> None:
    """Quantize one token's k, v [H, D] into data uint8 [pages, H, page / 16, block]."""
    H, D = k.shape
    G = D // group
    pg, at = divmod(slot, page)
    blk, b = divmod(at, 16)
    kc, ks, km = quantize(k, group)
    vc, vs, vm = quantize(v, group)
    for h in range(H):
        row = data[pg, h, blk]
        for ch in range(D):
            o, sh = _k_at(D, ch)
            o += b * (D // 2)
            row[o] = (int(row[o]) & (0xF0 >> sh)) | int(kc[h, ch]) << sh
            o, sh = _v_at(D, ch, b % 2)
            o += 8 * D + b // 2 * D
            row[o] = (int(row[o]) & (0xF0 >> sh)) | int(vc[h, ch]) << sh
        for off, s, m in ((16 * D, ks, km), (16 * D + 64 * G, vs, vm)):
            par = np.stack([s[h], m[h]], -1).astype(np.float16).reshape(-1).view(np.uint8)
            row[off + b * 4 * G:off + (b + 1) * 4 * G] = par


def read_slots(data, slots, D: int, page: int, group: int):
    """float64 K and V [T, H, D] of the slots."""
    G = D // group
    kb, ksh = map(np.array, zip(*[_k_at(D, c) for c in range(D)]))
    vb, vsh = map(np.array, zip(*[_v_at(D, c, 0) for c in range(D)]))
    K, V = [], []
    for slot in slots:
        pg, at = divmod(int(slot), page)
        row, b = data[pg, :, at // 16], at % 16
        kc = (row[:, b * (D // 2) + kb] >> ksh) & 15
        vc = (row[:, 8 * D + b // 2 * D + 2 * (b % 2) + vb] >> vsh) & 15
        par = np.ascontiguousarray(row[:, 16 * D:]).view(np.float16).reshape(-1, 2, 16, G, 2)
        K.append(values(kc, par[:, 0, b, :, 0], par[:, 0, b, :, 1]))
        V.append(values(vc, par[:, 1, b, :, 0], par[:, 1, b, :, 1]))
    shape = (0, data.shape[1], D)
    return (np.stack(K) if K else np.zeros(shape)), (np.stack(V) if V else np.zeros(shape))


def pages_step(table, held, free, count, lens, new, page, max_tokens, reset=None):
    """One step of page bookkeeping on int lists / arrays; returns new copies of the state and
    the outputs (table, held, free, count, slots, positions, cu_q, new_lens, status)."""
    table, held, free = (np.array(x, np.int64).copy() for x in (table, held, free))
    R, width = table.shape
    reset = [False] * R if reset is None else [bool(x) for x in reset]
    slots, pos = np.full(max_tokens, -1, np.int64), np.zeros(max_tokens, np.int64)

    def refuse(status):
        return table, held, free, count, slots, pos, np.zeros(R + 1, np.int64), np.array(lens), status

    gone = sum(int(held[r]) for r in range(R) if reset[r] and held[r] >= 0)
    kept = [0 if reset[r] else int(held[r]) for r in range(R)]
    need = [-(-(int(lens[r]) + int(new[r])) // page) for r in range(R)]
    if any(held[r] < 0 or held[r] > width or lens[r] < 0 or new[r] < 0 or need[r] > width
           or lens[r] + new[r] > 2 ** 31 - 1 for r in range(R)) \
            or count < 0 or count + gone > len(free) or sum(int(n) for n in new) > max_tokens:
        return refuse(-1)
    fresh = sum(max(0, need[r] - kept[r]) for r in range(R))
    if fresh > count + gone:
        return refuse(fresh - count - gone)
    released = [int(table[r, c]) for r in range(R) if reset[r] for c in range(held[r])]
    for r in range(R):
        if reset[r]:
            table[r, :held[r]] = -1
    stack = [int(p) for p in free[:count]] + released[::-1]
    for r in range(R):
        for c in range(kept[r], need[r]):
            table[r, c] = stack.pop()
        held[r] = max(kept[r], need[r])
    out = np.array(free)
    out[:len(stack)] = stack
    out[len(stack):count + gone] = -1
    cu, t = [0], 0
    for r in range(R):
        for p in range(int(lens[r]), int(lens[r]) + int(new[r])):
            pg = table[r, p // page]
            slots[t], pos[t] = (-1 if pg < 0 else pg * page + p % page), p
            t += 1
        cu.append(t)
    return (table, held, out, len(stack), slots, pos, np.array(cu),
            np.array(lens) + np.array(new), 0)


# ---- attention --------------------------------------------------------------------------
def attention(q, K, V, scale):
    """q [n, H, D], K and V [L, Hk, D] -> float64 [n, H, D]; row i sees tokens 0..L - n + i."""
    q = np.asarray(q, np.float64)
    n, H, D = q.shape
    L, Hk = K.shape[:2]
    out = np.zeros((n, H, D))
    for i in range(n):
        seen = L - n + i + 1
        if seen <= 0:
            continue
        for h in range(H):
            hk = h // (H // Hk)
            s = scale * (K[:seen, hk] @ q[i, h])
            p = np.exp(s - s.max())
            out[i, h] = p @ V[:seen, hk] / p.sum()
    return out


# ---- the product's epilogue -------------------------------------------------------------
def activate(y, name: str):
    if name == "none":
        return y
    if name == "relu":
        return np.where(y > 0, y, 0.0 * y)
    if name == "silu":
        return y / (1 + np.exp(-y))
    if name == "gelu":
        return 0.5 * y * (1 + np.vectorize(math.erf)(y / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * y * (1 + np.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    raise ValueError(name)


def epilogue(y, bias=None, activation="none", residual=None):
    y = np.asarray(y, np.float64)
    if bias is not None:
        y = y + np.asarray(bias, np.float64)
    y = activate(y, activation)
    return y if residual is None else y + np.asarray(residual, np.float64)
