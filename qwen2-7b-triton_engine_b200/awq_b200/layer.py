"""The operators between a decoder layer's packed products: rotary positions, a paged
key/value cache held in 4 bits, and attention over it.

  rope_axes(q, k, positions, inv_freq, sections)          rotary positions, 1 to 4 axes
  KV4Cache.allocate(num_pages, kv_heads, head_dim)        the cache
  kv4_pages_step(block_table, held, free_pages, ...)      block tables and slot maps of a step
  kv4_append(k, v, slots, cache)                          quantize new tokens into the cache
  kv4_gather(cache, slots)                                read tokens back as fp16
  kv4_attention(q, cache, block_table, kv_lens)           causal attention over the pages

A step of a layer: q/k/v product (bias in its epilogue) -> ``rope_axes`` -> ``kv4_append``
-> ``kv4_attention`` -> o product (residual in its epilogue, ``gemm_epilogue``).
``tp.AttentionLinearsTP.attend`` runs it.  ``kv4_pages_step`` runs once per step, for all
layers.  All of them take fp16 data, run on the current stream of the tensors' device, do
not synchronise and can be captured in a CUDA graph; there is no CPU fallback.  Formulas,
formats and refusals: include/awq_b200.h.
"""
from __future__ import annotations

import ctypes
import sys
from dataclasses import dataclass

import torch

from . import _lib

__all__ = ["KV4Cache", "rope_axes", "kv4_pages_step", "kv4_append", "kv4_gather",
           "kv4_attention"]


def _core():
    return sys.modules[__package__]


def _ext():
    """The C++ host glue (the same steps as the functions below), or None."""
    return _core()._ext


def _tensors(*args) -> bool:
    """Whether all arguments are tensors (or None): what the C++ signatures take.  Others go
    through the Python path, which names them."""
    return all(a is None or isinstance(a, torch.Tensor) for a in args)


def _need(t, name: str, dtype, ndim: int, device=None) -> None:
    _core()._require_cuda(t, name)
    dtypes = dtype if isinstance(dtype, tuple) else (dtype,)
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).split('.')[-1] for d in dtypes)}, "
                        f"got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D, got shape {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def _need_dense(t, name: str, dtype, shape, device) -> None:
    """A contiguous tensor of exactly this shape (state and outputs, never copied)."""
    _need(t, name, dtype, len(shape), device)
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(shape)} tensor, got "
                         f"{tuple(t.shape)}")


def _last_dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


@dataclass(frozen=True)
class KV4Cache:
    """A paged key/value cache in 4 bits: ``data`` uint8 [num_pages, kv_heads,
    page_size / 16, block bytes], contiguous, one block holding 16 tokens' codes, scales and
    minima of keys and values (csrc/awq_kv4.cuh).  head_dim 64 or 128; page_size a power of
    two from 16 to 1024; group_size (channels that share a scale) 32, 64 or 128, at most
    head_dim.  A token of a kv head takes head_dim + 8 * head_dim / group_size bytes.  Whole
    pages may be copied (``data[dst] = data[src]``) to fork a request."""
    data: torch.Tensor
    head_dim: int
    page_size: int
    group_size: int

    def __post_init__(self):
        D, g, P = self.head_dim, self.group_size, self.page_size
        if D not in (64, 128):
            raise ValueError(f"head_dim={D} must be 64 or 128")
        if g not in (32, 64, 128) or g > D:
            raise ValueError(f"group_size={g} must be 32, 64 or 128 and at most head_dim={D}")
        if P < 16 or P > 1024 or P & (P - 1):
            raise ValueError(f"page_size={P} must be a power of two from 16 to 1024")
        d = self.data
        if not isinstance(d, torch.Tensor) or d.dtype != torch.uint8:
            raise TypeError("data must be a uint8 torch.Tensor")
        block = 16 * D + 128 * (D // g)
        if d.dim() != 4 or d.shape[0] < 1 or d.shape[1] < 1 or d.shape[2] != P // 16 \
                or d.shape[3] != block or not d.is_contiguous():
            raise ValueError(f"data must be a contiguous [num_pages, kv_heads, {P // 16}, {block}] "
                             f"tensor, got {tuple(d.shape)}")

    @classmethod
    def allocate(cls, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 group_size: int | None = None, device=None) -> "KV4Cache":
        """A zeroed cache on ``device`` (default: the current CUDA device); group_size
        defaults to the head dimension."""
        g = head_dim if group_size is None else group_size
        if num_pages < 1 or kv_heads < 1 or g < 1:
            raise ValueError("num_pages, kv_heads and group_size must be positive")
        dev = torch.device("cuda") if device is None else torch.device(device)
        return cls(torch.zeros((num_pages, kv_heads, page_size // 16,
                                16 * head_dim + 128 * (head_dim // g)),
                               dtype=torch.uint8, device=dev), head_dim, page_size, g)

    @property
    def num_pages(self) -> int:
        return self.data.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.data.shape[1]

    def _shape_args(self):
        return self.num_pages, self.kv_heads, self.head_dim, self.group_size, self.page_size

    def _check(self) -> torch.device:
        _core()._require_cuda(self.data, "cache.data")
        return self.data.device


def rope_axes(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
              sections, interleaved: bool = False, out_q: torch.Tensor | None = None,
              out_k: torch.Tensor | None = None):
    """Rotary positions on q [T, q_heads, D] and k [T, k_heads, D] (fp16; strided views, e.g.
    of the fused q/k/v rows, are read in place).  positions int64 or int32 [axes, T], or [T]
    for one axis; inv_freq fp32 [half]; sections: frequencies per axis, half in all, 2 * half
    <= D (the channels behind pass through).  ``interleaved`` deals frequency i to axis
    i % axes while that axis has sections left, else to axis 0.  Angles keep full accuracy at
    any position.  Returns (out_q, out_k): new dense tensors, or those given, which may be q
    and k themselves (in place)."""
    ext = _ext()
    if ext is not None and _tensors(q, k, positions, inv_freq, out_q, out_k):
        return ext.rope_axes(q, k, positions, inv_freq, [int(x) for x in sections],
                             bool(interleaved), out_q, out_k)
    _need(q, "q", torch.float16, 3)
    dev = q.device
    _need(k, "k", torch.float16, 3, dev)
    T, H, D = q.shape
    if k.shape[0] != T or k.shape[2] != D:
        raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    sections = tuple(int(s) for s in sections)
    half = sum(sections)
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or half < 1 or 2 * half > D:
        raise ValueError(f"sections={sections} must be 1 to 4 counts that rotate 2 to {D} channels")
    if positions.dim() == 1:
        positions = positions[None]
    _need(positions, "positions", (torch.int64, torch.int32), 2, dev)
    if tuple(positions.shape) != (len(sections), T):
        raise ValueError(f"positions must be [{len(sections)}, {T}], got {tuple(positions.shape)}")
    _need_dense(inv_freq, "inv_freq", torch.float32, (half,), dev)
    positions = _last_dense(positions)
    q, k = _last_dense(q), _last_dense(k)
    outs = []
    for x, o, name in ((q, out_q, "out_q"), (k, out_k, "out_k")):
        if o is None:
            o = torch.empty(x.shape, dtype=torch.float16, device=dev)
        else:
            _need(o, name, torch.float16, 3, dev)
            if o.shape != x.shape or (D > 1 and o.stride(2) != 1) or not _distinct(o):
                raise ValueError(f"{name} must be {tuple(x.shape)} with a dense last dimension "
                                 "and rows that share no element")
            same = o.data_ptr() == x.data_ptr() and o.stride() == x.stride()
            for y in (q, k):
                if _core()._overlap(o, y) and not (same and y is x) and not _apart(o, y):
                    raise ValueError(f"{name} overlaps an input other than as that input itself")
        outs.append(o)
    oq, ok = outs
    if _core()._overlap(oq, ok) and not _apart(oq, ok):
        raise ValueError("out_q overlaps out_k")
    if T == 0:
        return oq, ok
    lib = _lib.load()
    sec = (ctypes.c_int32 * len(sections))(*sections)
    with _core()._DeviceGuard(dev):
        _lib.check(lib.awq_rope_axes(
            q.data_ptr(), q.stride(0), q.stride(1), H, k.data_ptr(), k.stride(0), k.stride(1),
            k.shape[1], T, D, positions.data_ptr(), int(positions.dtype == torch.int64),
            positions.stride(0), inv_freq.data_ptr(), sec, len(sections), int(bool(interleaved)),
            oq.data_ptr(), oq.stride(0), oq.stride(1), ok.data_ptr(), ok.stride(0), ok.stride(1),
            _core()._stream_handle(dev)))
    return oq, ok


def _distinct(t: torch.Tensor) -> bool:
    """Whether no two rows of t [T, H, D] (last dimension dense) share an element: heads within
    tokens or tokens within heads, not expanded ones."""
    (T, H, D), (ts, hs) = t.shape, t.stride()[:2]
    return t.numel() == 0 or (H == 1 or hs >= D) and (T == 1 or ts >= (H - 1) * hs + D) \
        or (T == 1 or ts >= D) and (H == 1 or hs >= (T - 1) * ts + D)


def _apart(o: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether o and y are different columns of the same rows (views of one fused q/k/v
    tensor), so that their address ranges interleave without sharing an element."""
    if o.stride(0) != y.stride(0) or o.stride(0) <= 0:
        return False
    row = o.stride(0) * o.element_size()

    def cols(t):
        return (t.shape[1] - 1) * t.stride(1) * 2 + t.shape[2] * 2 if t.stride(1) >= 0 else row + 1
    d = (y.data_ptr() - o.data_ptr()) % row
    return cols(o) <= d and d + cols(y) <= row


def kv4_pages_step(block_table: torch.Tensor, held: torch.Tensor, free_pages: torch.Tensor,
                   free_count: torch.Tensor, kv_lens: torch.Tensor, new_tokens: torch.Tensor,
                   page_size: int, max_tokens: int, reset: torch.Tensor | None = None):
    """The page bookkeeping of one step, on the GPU from the requests' lengths.

    State, updated in place (int32): block_table [R, max_blocks] (-1 where unused), held [R],
    the stack free_pages [capacity] with free_count [1] entries.  Input: kv_lens [R] tokens
    cached so far, new_tokens [R], reset (bool [R]): such a row's pages go back to the stack
    first (a finished request; give kv_lens 0 there).  Returns (slots int64 [max_tokens],
    positions int32 [max_tokens], cu_q int32 [R + 1], new_lens int32 [R], status int32 [1]):
    where each new token goes and its position, request after request, -1 and 0 behind the
    last one.  status 0; n > 0: n pages short; -1: a length out of range.  A refused step
    (status not 0) changes nothing and has no tokens.  At most 8192 requests."""
    ext = _ext()
    if ext is not None and _tensors(block_table, held, free_pages, free_count, kv_lens,
                                    new_tokens, reset):
        return ext.kv4_pages_step(block_table, held, free_pages, free_count, kv_lens, new_tokens,
                                  int(page_size), int(max_tokens), reset)
    _need(block_table, "block_table", torch.int32, 2)
    dev = block_table.device
    R, width = block_table.shape
    if width and block_table.stride(1) != 1 or (R > 1 and block_table.stride(0) < width):
        raise ValueError("block_table must have dense, non-overlapping rows")
    _need_dense(held, "held", torch.int32, (R,), dev)
    _need(free_pages, "free_pages", torch.int32, 1, dev)
    _need_dense(free_pages, "free_pages", torch.int32, tuple(free_pages.shape), dev)
    _need_dense(free_count, "free_count", torch.int32, (1,), dev)
    _need_dense(kv_lens, "kv_lens", torch.int32, (R,), dev)
    _need_dense(new_tokens, "new_tokens", torch.int32, (R,), dev)
    if reset is not None:
        _need_dense(reset, "reset", (torch.bool, torch.uint8), (R,), dev)
    page_size, max_tokens = int(page_size), int(max_tokens)
    if page_size < 1 or max_tokens < 0:
        raise ValueError("page_size must be positive and max_tokens not negative")
    slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    ints = torch.empty(max_tokens + 2 * R + 2, dtype=torch.int32, device=dev)
    positions, cu_q, lens, status = ints.split([max_tokens, R + 1, R, 1])
    lib = _lib.load()
    with _core()._DeviceGuard(dev):
        _lib.check(lib.awq_kv4_pages_step(
            block_table.data_ptr(), block_table.stride(0) if R > 1 else width, width,
            held.data_ptr(), free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(),
            kv_lens.data_ptr(), new_tokens.data_ptr(),
            reset.data_ptr() if reset is not None else None, R, page_size, slots.data_ptr(),
            positions.data_ptr(), max_tokens, cu_q.data_ptr(), lens.data_ptr(),
            status.data_ptr(), _core()._stream_handle(dev)))
    return slots, positions, cu_q, lens, status


def kv4_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: KV4Cache) -> None:
    """Quantize k and v [T, kv_heads, head_dim] (fp16, strided views are read in place) into
    the cache's slots (int64 [T], page * page_size + offset; negative: skipped).  The slots of
    a call must differ, as those of ``kv4_pages_step`` do."""
    ext = _ext()
    if ext is not None and _tensors(k, v, slots):
        return ext.kv4_append(k, v, slots, cache.data, cache.head_dim, cache.page_size,
                              cache.group_size)
    dev = cache._check()
    _need(k, "k", torch.float16, 3, dev)
    _need(v, "v", torch.float16, 3, dev)
    _need(slots, "slots", torch.int64, 1, dev)
    T = slots.shape[0]
    want = (T, cache.kv_heads, cache.head_dim)
    if tuple(k.shape) != want or tuple(v.shape) != want:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be {want}")
    if T == 0:
        return
    k, v, slots = _last_dense(k), _last_dense(v), slots.contiguous()
    lib = _lib.load()
    with _core()._DeviceGuard(dev):
        _lib.check(lib.awq_kv4_append(
            k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
            slots.data_ptr(), T, cache.data.data_ptr(), *cache._shape_args(),
            _core()._stream_handle(dev)))


def kv4_gather(cache: KV4Cache, slots: torch.Tensor):
    """(k, v) fp16 [T, kv_heads, head_dim] of the cache's slots (int64 [T]; zeros where a slot
    is negative): what attention reads, rounded to fp16."""
    ext = _ext()
    if ext is not None and _tensors(slots):
        return ext.kv4_gather(cache.data, cache.head_dim, cache.page_size, cache.group_size, slots)
    dev = cache._check()
    _need(slots, "slots", torch.int64, 1, dev)
    T = slots.shape[0]
    k = torch.empty((T, cache.kv_heads, cache.head_dim), dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    if T == 0:
        return k, v
    slots = slots.contiguous()
    lib = _lib.load()
    with _core()._DeviceGuard(dev):
        _lib.check(lib.awq_kv4_gather(cache.data.data_ptr(), *cache._shape_args(),
                                      slots.data_ptr(), T, k.data_ptr(), v.data_ptr(),
                                      _core()._stream_handle(dev)))
    return k, v


def kv4_attention(q: torch.Tensor, cache: KV4Cache, block_table: torch.Tensor,
                  kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, max_q: int = 1,
                  scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of q [T, q_heads, head_dim] (fp16) over the cache: fp16, same shape.

    block_table int32 [R, max_blocks], kv_lens int32 [R]: the tokens of each request in the
    cache, its new ones included.  Without cu_q, T = R and row r is request r's last token.
    With cu_q (int32 [R + 1]) request r has the rows cu_q[r] to cu_q[r + 1], its last tokens;
    max_q says how many rows a request has at most (it chooses the kernel; a wrong one costs
    time and may move roundings).  Query head h reads kv head h // (q_heads / kv_heads).
    scale defaults to head_dim ** -0.5.  Rows that see no token are zeros.  Rows behind cu_q[R]
    are left as they are in ``out`` and are zeros in a new tensor."""
    ext = _ext()
    if ext is not None and _tensors(q, block_table, kv_lens, cu_q, out):
        return ext.kv4_attention(q, cache.data, cache.head_dim, cache.page_size, cache.group_size,
                                 block_table, kv_lens, cu_q, int(max_q), scale, out)
    dev = cache._check()
    _need(q, "q", torch.float16, 3, dev)
    T, H, D = q.shape
    if D != cache.head_dim:
        raise ValueError(f"q has head_dim {D}, the cache {cache.head_dim}")
    if H < 1 or H % cache.kv_heads:
        raise ValueError(f"{H} query heads do not group over {cache.kv_heads} kv heads")
    _need(block_table, "block_table", torch.int32, 2, dev)
    R, width = block_table.shape
    if (width > 1 and block_table.stride(1) != 1) or (R > 1 and block_table.stride(0) < width):
        block_table = block_table.contiguous()
    _need_dense(kv_lens, "kv_lens", torch.int32, (R,), dev)
    max_q = int(max_q)
    if cu_q is None:
        if T != R or max_q != 1:
            raise ValueError(f"without cu_q every request has one query row: {T} rows, {R} "
                             f"requests, max_q={max_q}")
    else:
        _need_dense(cu_q, "cu_q", torch.int32, (R + 1,), dev)
        if max_q < 1:
            raise ValueError("max_q must be positive")
    if q.stride(2) != 1 or q.data_ptr() % 16 or q.stride(0) % 8 or q.stride(1) % 8:
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
    if out is None:
        new = torch.empty if cu_q is None else torch.zeros
        out = new((T, H, D), dtype=torch.float16, device=dev)
    else:
        _need(out, "out", torch.float16, 3, dev)
        if tuple(out.shape) != (T, H, D) or out.stride(2) != 1 or out.data_ptr() % 8 \
                or out.stride(0) % 4 or out.stride(1) % 4 or not _distinct(out):
            raise ValueError(f"out must be {(T, H, D)} with a dense last dimension, 8-byte "
                             "aligned rows that share no element")
        if _core()._overlap(out, q):
            raise ValueError("out overlaps q")
    if T == 0 or R == 0:
        return out
    lib = _lib.load()
    with _core()._DeviceGuard(dev):
        need = _attention_workspace(lib, dev, D, min(max_q, T) * (H // cache.kv_heads))
        # a workspace of this call alone: graphs that replay at once must not share one
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(lib.awq_kv4_attention(
            q.data_ptr(), q.stride(0), q.stride(1), T, H, cache.data.data_ptr(),
            *cache._shape_args(), block_table.data_ptr(),
            block_table.stride(0) if R > 1 else width, width, kv_lens.data_ptr(),
            cu_q.data_ptr() if cu_q is not None else None, R, max_q,
            float(D ** -0.5 if scale is None else scale), out.data_ptr(), out.stride(0),
            out.stride(1), ws.data_ptr(), need, _core()._stream_handle(dev)))
    return out


_attn_ws: dict = {}


def _attention_workspace(lib, dev: torch.device, head_dim: int, max_rows: int) -> int:
    key = (dev.index, head_dim, max_rows)
    need = _attn_ws.get(key)
    if need is None:
        need = int(lib.awq_kv4_attention_workspace_bytes(head_dim, max_rows))
        if need and len(_attn_ws) < 65536:
            _attn_ws[key] = need
    return need
