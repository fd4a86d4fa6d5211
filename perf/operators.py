"""Workloads of the operators around a layer's packed 4-bit products, at this library's shapes.

Five operators that run between and behind the AWQ projections of a decoder layer:

  gemm       the packed product with bias, activation and residual in its epilogue
  rope       rotary positions with several axes on the heads of a fused q/k/v row
  pages      block tables and slot maps of a paged cache, built from request lengths
  append     keys and values quantized to 4 bits into their cache slots, and read back
  attention  attention over the 4-bit pages, from single tokens to prompt chunks

``listed`` names the workloads, ``draw`` makes one more of the same ranges, ``prepare``
makes a workload's inputs on the GPU, ``run`` makes one pass (elementary torch operations
when ``own`` is false, this library's entry points when it is true), ``exact`` is the same
result in 64 bits and ``work`` the bytes and operations a pass cannot do without.
"""
from __future__ import annotations

import math
import random
import sys

import torch

own = False

DEV = "cuda"


def _library():
    """This repository's package (its folder name is not a module name)."""
    path = "qwen2-7b-triton_engine_b200"
    if path not in sys.path:
        sys.path.insert(1, path)
    import awq_b200
    return awq_b200


# ---------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------
def listed():
    return [
        # the down projection of one decoded token, added to the residual stream
        dict(name="gemm_token_down", op="gemm", M=1, K=18944, N=3584, group=128,
             activation="none", bias=False, residual=True),
        # a biased, activated layer for the tokens of a dozen requests
        dict(name="gemm_batch_gelu", op="gemm", M=12, K=3584, N=4608, group=128,
             activation="gelu_tanh", bias=True, residual=True),
        # the down projection of a long prompt, added to the residual stream
        dict(name="gemm_prompt_down", op="gemm", M=2048, K=18944, N=3584, group=128,
             activation="none", bias=False, residual=True),
        # the rotary step of a decode batch far into its contexts
        dict(name="rope_tokens", op="rope", T=8, q_heads=28, kv_heads=4, dim=128, axes="64",
             interleaved=False, far=1000000),
        # a long prompt of text and image patches: time, height and width positions
        dict(name="rope_prompt", op="rope", T=8191, q_heads=28, kv_heads=4, dim=128,
             axes="16,24,24", interleaved=False, far=32768),
        # a decode step of 64 requests, a few of them replaced by new prompts
        dict(name="pages_step", op="pages", R=64, page=16, max_len=2048, replaced=3, prompt=100),
        # a full server: 2048 requests, a hundred replaced by prompts
        dict(name="pages_server", op="pages", R=2048, page=64, max_len=16384, replaced=101,
             prompt=301),
        # the keys and values of a decode batch
        dict(name="append_tokens", op="append", T=64, kv_heads=4, dim=128, group=128, page=64,
             pages=256),
        # the keys and values of a long prompt in small groups and small pages
        dict(name="append_prompt", op="append", T=8191, kv_heads=4, dim=128, group=32, page=16,
             pages=1024),
        # one request, one token
        dict(name="attention_token", op="attention", R=1, q_heads=28, kv_heads=4, dim=128,
             group=128, page=64, min_q=1, max_q=1, min_len=1000, max_len=1000),
        # a decode batch of ragged, long contexts
        dict(name="attention_batch", op="attention", R=48, q_heads=28, kv_heads=4, dim=128,
             group=64, page=64, min_q=1, max_q=1, min_len=1, max_len=16384),
        # prompt chunks behind cached contexts, as a scheduler mixes them
        dict(name="attention_chunks", op="attention", R=4, q_heads=28, kv_heads=4, dim=128,
             group=128, page=64, min_q=1, max_q=1024, min_len=777, max_len=8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemm", "rope", "pages", "append", "attention"])
    if op == "gemm":
        group = rng.choice([64, 128])
        K = group * _log_int(rng, 512 // group, 18944 // group)
        N = 8 * _log_int(rng, 32, 4736)
        if rng.random() < 0.6:            # whole TMA boxes; the rest takes any multiple of 8
            N = (N + 31) // 32 * 32
        M = min(_log_int(rng, 1, 2048), max(1, (2048 * 18944 * 3584) // (K * N)))
        return dict(op=op, M=M, K=K, N=N, group=group,
                    activation=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    bias=rng.random() < 0.5, residual=rng.random() < 0.7)
    if op == "rope":
        dim = rng.choice([64, 128])
        half = dim // 2
        axes = rng.choice([f"{half}", f"{half // 4},{half * 3 // 8},{half * 3 // 8}",
                           f"{half // 8},{half // 4},{half // 4}"])   # the last: partly rotated
        kv = rng.choice([1, 2, 4])
        return dict(op=op, T=_log_int(rng, 1, 8191), q_heads=kv * rng.choice([1, 4, 7]),
                    kv_heads=kv, dim=dim, axes=axes, interleaved=rng.random() < 0.4,
                    far=_log_int(rng, 100, 1000000))
    if op == "pages":
        R = _log_int(rng, 1, 2048)
        replaced = rng.randint(0, max(0, min(R // 8, 101)))
        return dict(op=op, R=R, page=rng.choice([16, 32, 64]), max_len=_log_int(rng, 64, 4096),
                    replaced=replaced, prompt=_log_int(rng, 1, 301))
    if op == "append":
        dim = rng.choice([64, 128])
        group = rng.choice([g for g in (32, 64, 128) if g <= dim])
        T, page = _log_int(rng, 1, 8191), rng.choice([16, 32, 64])
        return dict(op=op, T=T, kv_heads=rng.choice([1, 2, 4]), dim=dim, group=group, page=page,
                    pages=(T + page - 1) // page + rng.randint(1, 64))
    dim = rng.choice([64, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= dim])
    kv = rng.choice([1, 2, 4])
    heads = kv * rng.choice([1, 4, 7])
    case = dict(op=op, R=1, q_heads=heads, kv_heads=kv, dim=dim, group=group,
                page=rng.choice([16, 32, 64]), min_q=1, max_q=1, min_len=1, max_len=1)
    if rng.random() < 0.6:
        case["R"] = _log_int(rng, 1, 48)
        case["max_len"] = _log_int(rng, 1, 16384)
    else:
        case["R"] = rng.randint(1, 4)
        case["max_q"] = _log_int(rng, 2, 1024)
        case["max_len"] = case["max_q"] + _log_int(rng, 1, 7168)
        case["min_len"] = case["max_q"]
    return case


def _spread(case, what, lo, hi, n):
    """n lengths of a case, the same for every seed: the ends first, the rest over the
    logarithm of the range."""
    rng = random.Random(f"{what}:{n}:{lo}:{hi}")
    vals = [hi, lo] + [_log_int(rng, lo, hi) if hi > 64 * lo and rng.random() < 0.3
                       else rng.randint(lo, hi) for _ in range(n)]
    return vals[:n]


def _lengths(case):
    """(cached tokens, query tokens) of each request of an attention case."""
    q = _spread(case, "q", case["min_q"], case["max_q"], case["R"])
    kv = _spread(case, "kv", case["min_len"], case["max_len"], case["R"])
    return [max(a, b) for a, b in zip(kv, q)], q


# ---------------------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "gemm":
        M, K, N, g = case["M"], case["K"], case["N"], case["group"]
        b = K * N // 2 + (K // g) * N * 5 // 2 + 2 * M * K + 2 * M * N
        b += 2 * M * N * case["residual"] + 2 * N * case["bias"]
        return {"bytes": b, "flops": 2 * M * N * K}
    if op == "rope":
        sections = [int(s) for s in case["axes"].split(",")]
        rot = 2 * sum(sections)
        heads = case["q_heads"] + case["kv_heads"]
        return {"bytes": case["T"] * (4 * heads * case["dim"] + 8 * len(sections)) + 2 * rot,
                "flops": case["T"] * heads * rot * 3}
    if op == "pages":
        lens, new, reset, _ = _requests(case)
        tokens = sum(new)
        moved = sum(-(-n // case["page"]) for n, r in zip(new, reset) if r)
        return {"bytes": 21 * case["R"] + 12 * tokens + 8 * moved, "flops": 0}
    if op == "append":
        T, H, D, g = case["T"], case["kv_heads"], case["dim"], case["group"]
        packed = H * (D + 8 * D // g)
        # fp16 keys and values in, the packed rows out and in again, fp16 out
        return {"bytes": T * (8 * H * D + 2 * packed + 16), "flops": T * H * D * 10}
    kv, q = _lengths(case)
    H, Hk, D, g = case["q_heads"], case["kv_heads"], case["dim"], case["group"]
    rows = sum(q)
    pairs = sum(n * (L - n) + n * (n + 1) // 2 for L, n in zip(kv, q))
    return {"bytes": sum(kv) * Hk * (D + 8 * D // g) + 4 * rows * H * D,
            "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    return {"gemm": _prepare_gemm, "rope": _prepare_rope, "pages": _prepare_pages,
            "append": _prepare_append, "attention": _prepare_attention}[case["op"]](case, gen)


def _randn(gen, *shape):
    return torch.randn(shape, device=DEV, generator=gen)


def _randint(gen, lo, hi, shape, dtype=torch.int32):
    return torch.randint(lo, hi, shape, device=DEV, generator=gen, dtype=torch.int64).to(dtype)


def _prepare_gemm(case, gen):
    M, K, N, g = case["M"], case["K"], case["N"], case["group"]
    G = K // g
    qweight = _randint(gen, -2 ** 31, 2 ** 31, (K, N // 8))
    # zeros around the middle of the code range, scales that keep the outputs near 1
    zeros = _randint(gen, 6, 10, (G, N // 8, 8), torch.int64)
    qzeros = (zeros << (4 * torch.arange(8, device=DEV))).sum(-1)
    qzeros = torch.where(qzeros >= 2 ** 31, qzeros - 2 ** 32, qzeros).to(torch.int32)
    scales = (0.5 + torch.rand((G, N), device=DEV, generator=gen)) * (0.2 / math.sqrt(K))
    st = dict(case=case, x=_randn(gen, M, K).half(), qweight=qweight, qzeros=qzeros,
              scales=scales.half(), bias=None, residual=None)
    if case["bias"]:
        st["bias"] = (0.5 * _randn(gen, N)).half()
    if case["residual"]:
        st["residual"] = (2 * _randn(gen, M, N)).half()
    return st


def _prepare_rope(case, gen):
    T, H, Hk, D = case["T"], case["q_heads"], case["kv_heads"], case["dim"]
    sections = tuple(int(s) for s in case["axes"].split(","))
    half = sum(sections)
    qkv = _randn(gen, T, (H + 2 * Hk) * D).half()       # the fused product's rows
    pos = _randint(gen, 0, case["far"], (len(sections), T), torch.int64)
    inv_freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    return dict(case=case, q=qkv[:, :H * D].view(T, H, D),
                k=qkv[:, H * D:(H + Hk) * D].view(T, Hk, D), positions=pos,
                inv_freq=inv_freq.float(), sections=sections)


def _requests(case):
    """Lengths before the step, new tokens, which rows are replaced, pages held."""
    R, P = case["R"], case["page"]
    lens = _spread(case, "pages", 1, case["max_len"], R)
    reset = [0] * R
    for r in random.Random(f"replaced:{R}").sample(range(R), case["replaced"]):
        reset[r] = 1
    held = [-(-n // P) for n in lens]
    new = [case["prompt"] if x else 1 for x in reset]
    lens = [0 if x else n for n, x in zip(lens, reset)]
    return lens, new, reset, held


def _prepare_pages(case, gen):
    lens, new, reset, held = _requests(case)
    R, P = case["R"], case["page"]
    width = max(-(-(case["max_len"] + 1) // P), -(-case["prompt"] // P))
    total = sum(held) + R + case["replaced"] * -(-case["prompt"] // P) + 7
    ids = torch.randperm(total, device=DEV, generator=gen).to(torch.int32)
    held_t = torch.tensor(held, dtype=torch.int32, device=DEV)
    taken = torch.arange(width, device=DEV)[None] < held_t[:, None]
    table = torch.full((R, width), -1, dtype=torch.int32, device=DEV)
    table[taken] = ids[:sum(held)]
    free = torch.full((total,), -1, dtype=torch.int32, device=DEV)
    free[:total - sum(held)] = ids[sum(held):]
    return dict(case=case, table=table, held=held_t, free=free,
                count=torch.tensor([total - sum(held)], dtype=torch.int32, device=DEV),
                lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                new=torch.tensor(new, dtype=torch.int32, device=DEV),
                reset=torch.tensor(reset, dtype=torch.bool, device=DEV),
                max_tokens=sum(new) + 5)


def _key_values(gen, T, H, D):
    """Keys with a few channels far from zero, as biased key projections have, and values."""
    shift = torch.where(torch.rand((H, D), device=DEV, generator=gen) < 0.04, 6.0, 0.0)
    shift = shift * _randn(gen, H, D)
    return (_randn(gen, T, H, D) + shift).half(), (0.7 * _randn(gen, T, H, D)).half()


def _prepare_append(case, gen):
    T, H, D, P = case["T"], case["kv_heads"], case["dim"], case["page"]
    k, v = _key_values(gen, T, H, D)
    slots = torch.randperm(case["pages"], device=DEV, generator=gen)
    slots = (slots[:, None] * P + torch.arange(P, device=DEV)).flatten()
    if T <= 256:            # single tokens of T requests; otherwise the pages of one prompt
        slots = slots[torch.randperm(slots.numel(), device=DEV, generator=gen)]
    cache = torch.zeros((case["pages"], H, P // 16, _block_bytes(D, case["group"])),
                        dtype=torch.uint8, device=DEV)
    return dict(case=case, k=k, v=v, slots=slots[:T].contiguous(), cache=cache)


def _prepare_attention(case, gen):
    H, Hk, D, P, g = (case[n] for n in ("q_heads", "kv_heads", "dim", "page", "group"))
    kv, q = _lengths(case)
    need = [-(-n // P) for n in kv]
    pages = sum(need) + 3
    cache = torch.empty((pages, Hk, P // 16, _block_bytes(D, g)), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 24) // (P * Hk * D))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        k, v = _key_values(gen, (b - a) * P, Hk, D)
        k, v = (x.view(b - a, P, Hk, D).transpose(1, 2) for x in (k, v))
        cache[a:b] = _pack(*_quantize(k, g), *_quantize(v, g))
    ids = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.full((case["R"], max(need) + 2), -1, dtype=torch.int32, device=DEV)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = ids[at:at + n]
        at += n
    cu = [0]
    for n in q:
        cu.append(cu[-1] + n)
    return dict(case=case, q=_randn(gen, cu[-1], H, D).half(), cache=cache, table=table,
                lens=torch.tensor(kv, dtype=torch.int32, device=DEV),
                cu_q=torch.tensor(cu, dtype=torch.int32, device=DEV), cu_host=cu, kv_host=kv,
                scale=D ** -0.5)


# ---------------------------------------------------------------------------------------
# the packed cache in torch
#
# A page holds, for each kv head, blocks of 16 tokens:
#   K codes   [16 tokens][D/8 words]    word (j // w) * 4 w + w t + j % w holds the channels
#                                       8 (4 j + t) + p at bits 4 p, t < 4, w = min(D/32, 4)
#   V codes   [8 token pairs][D/4 words] word (i // w) * 8 w + w h + i % w holds the channels
#                                       4 (8 i + h) + p, h < 8: even token in the low half
#   K params  [16 tokens][D/g]          fp16 scale, fp16 minimum
#   V params  [16 tokens][D/g]
# ---------------------------------------------------------------------------------------
def _block_bytes(D, g):
    return 16 * D + 128 * (D // g)


def _k_words(D):
    w = min(D // 32, 4)
    return [4 * j + t for b in range(D // 32 // w) for t in range(4)
            for j in range(b * w, (b + 1) * w)]          # octet of each word, in word order


def _v_words(D):
    w = min(D // 32, 4)
    return [8 * i + h for b in range(D // 32 // w) for h in range(8)
            for i in range(b * w, (b + 1) * w)]          # quad of each word, in word order


def _half_grid(x):
    """float64 values rounded once to fp16's grid (ties to even); x >= 0."""
    e = torch.frexp(x)[1].clamp(min=-13)
    step = torch.ldexp(torch.ones_like(x), e - 11)
    return (torch.round(x / step) * step).half()


def _quantize(x, g):
    """fp16 [..., D] -> codes uint8 [..., D], scale and minimum fp16 [..., D/g]."""
    x = x.double().unflatten(-1, (-1, g))
    lo = x.amin(-1, keepdim=True)
    s = _half_grid((x.amax(-1, keepdim=True) - lo) / 15)
    sd = s.double()
    c = torch.where(sd > 0, torch.round((x - lo) / torch.where(sd > 0, sd, 1.0)), 0.0)
    return c.clamp(0, 15).to(torch.uint8).flatten(-2), s.squeeze(-1), lo.half().squeeze(-1)


def _pack(kc, ks, km, vc, vs, vm):
    """Codes [n, H, P, D] and params [n, H, P, D/g] -> bytes [n, H, P/16, block]."""
    n, H, P, D = kc.shape
    kw = kc.view(n, H, P // 16, 16, D // 8, 8)[..., _k_words(D), :]
    kb = (kw[..., 0::2] | (kw[..., 1::2] << 4)).flatten(-3)
    vw = vc.view(n, H, P // 16, 8, 2, D // 4, 4)[..., _v_words(D), :].transpose(-3, -2)
    vb = (vw[..., 0::2] | (vw[..., 1::2] << 4)).flatten(-4)
    kp = torch.stack([ks, km], -1).view(n, H, P // 16, -1).contiguous().view(torch.uint8)
    vp = torch.stack([vs, vm], -1).view(n, H, P // 16, -1).contiguous().view(torch.uint8)
    return torch.cat([kb, vb, kp, vp], -1)


def _unpack(blocks, D):
    """bytes [..., block] -> K and V codes [..., 16, D], params [..., 16, D/g, 2]."""
    lead, a = blocks.shape[:-1], 8 * D
    kb = blocks[..., :a].reshape(*lead, 16, D // 8, 4)
    kn = torch.stack([kb & 15, kb >> 4], -1).flatten(-2)
    k = torch.empty_like(kn)
    k[..., _k_words(D), :] = kn
    vb = blocks[..., a:2 * a].reshape(*lead, 8, D // 4, 2, 2)
    vn = torch.stack([vb & 15, vb >> 4], -1).flatten(-2)
    v = torch.empty_like(vn)
    v[..., _v_words(D), :, :] = vn
    p = blocks[..., 2 * a:].contiguous().view(torch.float16).reshape(*lead, 2, 16, -1, 2)
    return (k.flatten(-2), v.transpose(-3, -2).flatten(-2).flatten(-3, -2),
            p[..., 0, :, :, :], p[..., 1, :, :, :])


def _values(codes, params):
    """Codes [..., D] and params [..., D/g, 2] -> fp32 values."""
    G = params.shape[-2]
    x = codes.float().unflatten(-1, (G, -1))
    return (x * params[..., :1].float() + params[..., 1:].float()).flatten(-2)


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    return {"gemm": _run_gemm, "rope": _run_rope, "pages": _run_pages, "append": _run_append,
            "attention": _run_attention}[state["case"]["op"]](state)


_SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)                 # bit of element n % 8 in its word


def _weights(st):
    """fp16 [K, N]: (code - zero) * scale, rounded once, as the packed format defines it."""
    sh = torch.tensor(_SHIFTS, dtype=torch.int32, device=DEV)
    w = ((st["qweight"][..., None] >> sh) & 15).flatten(1)
    z = ((st["qzeros"][..., None] >> sh) & 15).flatten(1)
    g = st["case"]["group"]
    d = (w.unflatten(0, (-1, g)) - z[:, None]).half() * st["scales"][:, None]
    return d.flatten(0, 1)


def _activate(y, name):
    if name == "relu":
        return torch.where(y > 0, y, 0.0)
    if name == "silu":
        return y / (1 + torch.exp(-y))
    if name == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _run_gemm(st):
    case = st["case"]
    if own:
        return _library().gemm_epilogue(st["x"], st["qweight"], st["qzeros"], st["scales"],
                                        case["group"], bias=st["bias"],
                                        activation=case["activation"], residual=st["residual"])
    y = st["x"].float() @ _weights(st).float()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    y = _activate(y, case["activation"])
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.half()


def _axis_of(sections, interleaved):
    """The position axis of each frequency."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    A = len(sections)
    return [i % A if i // A < sections[i % A] else 0 for i in range(sum(sections))]


def _run_rope(st):
    case = st["case"]
    if own:
        return _library().rope_axes(st["q"], st["k"], st["positions"], st["inv_freq"],
                                    st["sections"], interleaved=case["interleaved"])
    axis = torch.tensor(_axis_of(st["sections"], case["interleaved"]), device=DEV)
    angle = st["positions"][axis].T.double() * st["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    h = sum(st["sections"])
    out = []
    for x in (st["q"], st["k"]):
        a, b, rest = x[..., :h].float(), x[..., h:2 * h].float(), x[..., 2 * h:].float()
        out.append(torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).half())
    return tuple(out)


def _run_pages(st):
    case = st["case"]
    P, R = case["page"], case["R"]
    if own:
        slots, positions, cu, lens, status = _library().kv4_pages_step(
            st["table"], st["held"], st["free"], st["count"], st["lens"], st["new"],
            page_size=P, max_tokens=st["max_tokens"], reset=st["reset"])
        return dict(slots=slots, positions=positions, cu=cu, lens=lens, status=status,
                    table=st["table"], held=st["held"], free=st["free"], count=st["count"])
    table, held, free, count = (st[n].long() for n in ("table", "held", "free", "count"))
    lens0, new, reset = st["lens"].long(), st["new"].long(), st["reset"]
    col = torch.arange(table.shape[1], device=DEV)[None]
    # pages of replaced rows go onto the stack, the first of them on top
    gone = reset[:, None] & (col < held[:, None])
    rank = (gone.flatten().long().cumsum(0) - 1).view_as(gone)
    n_gone = gone.sum()
    at = torch.where(gone, count + n_gone - 1 - rank, free.numel())
    stack = torch.cat([free, free.new_zeros(1)]).scatter(0, at.flatten(), table.flatten())
    kept = torch.where(reset, 0, held)
    table = torch.where(gone, -1, table)
    lens = lens0 + new
    need = torch.maximum(kept, (lens + P - 1) // P)
    fresh = (col >= kept[:, None]) & (col < need[:, None])
    rank = (fresh.flatten().long().cumsum(0) - 1).view_as(fresh)
    top = count + n_gone
    table = torch.where(fresh, stack[(top - 1 - rank).clamp(0, free.numel())], table)
    count = top - fresh.sum()
    ids = torch.arange(free.numel(), device=DEV)
    free = torch.where(ids < count, stack[:-1], -1)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(st["max_tokens"], device=DEV)
    row = torch.searchsorted(cu[1:], t, right=True).clamp(max=R - 1)
    pos = lens0[row] + t - cu[row]
    live = t < cu[-1]
    page = table[row, torch.where(live, pos // P, 0)]
    st["table"].copy_(table)
    st["held"].copy_(need)
    st["free"].copy_(free)
    st["count"].copy_(count)
    return dict(slots=torch.where(live, page * P + pos % P, -1),
                positions=torch.where(live, pos, 0).int(), cu=cu.int(), lens=lens.int(),
                status=torch.zeros(1, dtype=torch.int32, device=DEV), table=st["table"],
                held=st["held"], free=st["free"], count=st["count"])


def _run_append(st):
    case = st["case"]
    D, g, P = case["dim"], case["group"], case["page"]
    if own:
        lib = _library()
        cache = lib.KV4Cache(st["cache"], head_dim=D, page_size=P, group_size=g)
        lib.kv4_append(st["k"], st["v"], st["slots"], cache)
        return lib.kv4_gather(cache, st["slots"])
    slots = st["slots"]
    page, block, at = slots // P, slots % P // 16, slots % 16
    cache, T, H, a = st["cache"], case["T"], case["kv_heads"], 8 * D
    kc, ks, km = _quantize(st["k"], g)
    vc, vs, vm = _quantize(st["v"], g)
    kw = kc.view(T, H, D // 8, 8)[..., _k_words(D), :]
    kb = (kw[..., 0::2] | (kw[..., 1::2] << 4)).flatten(-2)
    vw = vc.view(T, H, D // 4, 4)[..., _v_words(D), :]
    vb = vw[..., 0::2] | (vw[..., 1::2] << 4)                            # [T, H, D/4, 2]
    kp = torch.stack([ks, km], -1).flatten(-2).view(torch.uint8)
    vp = torch.stack([vs, vm], -1).flatten(-2).view(torch.uint8)
    where = (page[:, None, None], torch.arange(H, device=DEV)[:, None], block[:, None, None])
    n = kp.shape[-1]
    row = torch.arange(D // 2, device=DEV)
    cache[(*where, at[:, None, None] * (D // 2) + row)] = kb
    word = torch.arange(D // 4, device=DEV)
    byte = a + (at // 2)[:, None] * D + word * 4 + (at % 2)[:, None] * 2
    byte = torch.stack([byte, byte + 1], -1).flatten(1)
    cache[(*where, byte[:, None])] = vb.flatten(-2)
    par = 2 * a + at[:, None, None] * n + torch.arange(n, device=DEV)
    cache[(*where, par)] = kp
    cache[(*where, par + 16 * n)] = vp
    k, v, kq, vq = _unpack(cache[page, :, block], D)                     # [T, H, 16, D]
    i = torch.arange(T, device=DEV)
    return _values(k[i, :, at], kq[i, :, at]).half(), _values(v[i, :, at], vq[i, :, at]).half()


def _sequence(st, r):
    """K and V of request r in fp32, [Hk, L, D]."""
    case, L = st["case"], st["kv_host"][r]
    P, D = case["page"], case["dim"]
    ids = st["table"][r, :-(-L // P)].long()
    k, v, kq, vq = _unpack(st["cache"][ids].transpose(0, 1), D)          # [Hk, n, P/16, 16, D]
    return (_values(c, p).flatten(1, 3)[:, :L] for c, p in ((k, kq), (v, vq)))


def _run_attention(st):
    case = st["case"]
    if own:
        lib = _library()
        cache = lib.KV4Cache(st["cache"], head_dim=case["dim"], page_size=case["page"],
                             group_size=case["group"])
        if case["max_q"] == 1:
            return lib.kv4_attention(st["q"], cache, st["table"], st["lens"], scale=st["scale"])
        return lib.kv4_attention(st["q"], cache, st["table"], st["lens"], cu_q=st["cu_q"],
                                 max_q=case["max_q"], scale=st["scale"])
    H, Hk, D = case["q_heads"], case["kv_heads"], case["dim"]
    out = torch.empty_like(st["q"])
    for r, L in enumerate(st["kv_host"]):
        a, b = st["cu_host"][r], st["cu_host"][r + 1]
        n = b - a
        k, v = _sequence(st, r)
        q = st["q"][a:b].float().view(n, Hk, H // Hk, D).permute(1, 2, 0, 3)
        s = (q @ k[:, None].transpose(-1, -2)) * st["scale"]             # [Hk, G, n, L]
        hidden = torch.arange(L, device=DEV) > torch.arange(L - n, L, device=DEV)[:, None]
        s = s.masked_fill_(hidden, float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = (p @ v[:, None]) / p.sum(-1, keepdim=True)
        out[a:b] = o.permute(2, 0, 1, 3).reshape(n, H, D).half()
    return out


# ---------------------------------------------------------------------------------------
# the same results in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    return {"gemm": _exact_gemm, "rope": _exact_rope, "pages": lambda c, s: None,
            "append": _exact_append, "attention": _exact_attention}[case["op"]](case, seed)


def _exact_gemm(case, seed):
    st = prepare(case, seed)
    K, N, g = case["K"], case["N"], case["group"]
    W = torch.empty((K, N), dtype=torch.float64, device=DEV)
    zero = torch.empty((K // g, N), dtype=torch.float64, device=DEV)
    for e, slot in enumerate((0, 4, 1, 5, 2, 6, 3, 7)):
        W[:, e::8] = (st["qweight"] >> (4 * slot)).bitwise_and(15).double()
        zero[:, e::8] = (st["qzeros"] >> (4 * slot)).bitwise_and(15).double()
    W -= zero.repeat_interleave(g, 0)
    W *= st["scales"].double().repeat_interleave(g, 0)
    W = W.half().double()         # the product of 5 and 11 bits is exact before this rounding
    y = st["x"].double() @ W
    if st["bias"] is not None:
        y += st["bias"].double()
    name = case["activation"]
    if name == "relu":
        y = y.clamp(min=0)
    elif name == "silu":
        y = y * torch.reciprocal(1 + (-y).exp())
    elif name == "gelu":
        y = y * torch.special.erfc(-y * 0.5 ** 0.5) / 2
    elif name == "gelu_tanh":
        z = (2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)
        y = y * torch.reciprocal(1 + (-2 * z).exp())
    if st["residual"] is not None:
        y += st["residual"].double()
    return y


def _exact_rope(case, seed):
    st = prepare(case, seed)
    sections = st["sections"]
    h, A = sum(sections), len(sections)
    out = [x.double() for x in (st["q"], st["k"])]
    turned = [x.clone() for x in out]
    ends = [sum(sections[:a + 1]) for a in range(A)]
    for i in range(h):
        if case["interleaved"]:
            a = i % A if i // A < sections[i % A] else 0
        else:
            a = sum(1 for e in ends if e <= i)
        th = st["positions"][a].double() * float(st["inv_freq"][i])
        rot = torch.polar(torch.ones_like(th), th)[:, None]
        for x, y in zip(out, turned):
            z = torch.complex(x[..., i], x[..., i + h]) * rot
            y[..., i], y[..., i + h] = z.real, z.imag
    return tuple(turned)


def _nearest_half(x):
    """float64 -> the nearest fp16 value (ties to even), by comparing neighbours."""
    import numpy as np
    return torch.from_numpy(x.cpu().numpy().astype(np.float16).astype(np.float64)).to(x.device)


def _exact_append(case, seed):
    st = prepare(case, seed)
    g = case["group"]
    out = []
    for x in (st["k"], st["v"]):
        y = torch.empty(x.shape, dtype=torch.float64, device=DEV)
        for a in range(0, case["dim"], g):
            part = x[..., a:a + g].double()
            low, high = part.min(-1, keepdim=True)[0], part.max(-1, keepdim=True)[0]
            step = _nearest_half((high - low) / 15)
            code = ((part - low) / step).nan_to_num(0.0).round().clamp(0, 15)
            y[..., a:a + g] = low + code * step
        out.append(y)
    return tuple(out)


def _exact_attention(case, seed):
    st = prepare(case, seed)
    kv, q = _lengths(case)
    H, Hk, D, P, g = (case[n] for n in ("q_heads", "kv_heads", "dim", "page", "group"))
    w = min(D // 32, 4)
    c = torch.arange(D, device=DEV)
    j, t = c // 32, c // 8 % 4                       # key channel -> its word, then its nibble
    k_nib = ((j // w * 4 * w + w * t + j % w) * 8 + c % 8).tolist()
    i, h8 = c // 32, c // 4 % 8                      # value channel -> its word, nibble of 4
    v_nib = ((i // w * 8 * w + w * h8 + i % w) * 8 + c % 4).tolist()
    out = torch.empty((sum(q), H, D), dtype=torch.float64, device=DEV)
    at = 0
    for r, (L, n) in enumerate(zip(kv, q)):
        pages = st["table"][r, :-(-L // P)].long()
        for hk in range(Hk):
            blocks = st["cache"][pages, hk].flatten(0, 1)                # [blocks, bytes]
            nib = torch.empty((blocks.shape[0], 32 * D), dtype=torch.uint8, device=DEV)
            nib[:, 0::2], nib[:, 1::2] = blocks[:, :16 * D] % 16, blocks[:, :16 * D] // 16
            kc = nib[:, :16 * D].reshape(-1, D)[:, k_nib]
            pair = nib[:, 16 * D:].reshape(-1, 2 * D)
            even, odd = pair[:, v_nib], pair[:, [x + 4 for x in v_nib]]
            vc = torch.stack([even, odd], 1).view(-1, D)
            par = blocks[:, 16 * D:].contiguous().view(torch.float16).double()
            par = par.view(-1, 2, 16, D // g, 2).transpose(0, 1).flatten(1, 2)   # [2, tokens, G, 2]
            k, v = (x.double() * p[..., 0].repeat_interleave(g, 1) + p[..., 1].repeat_interleave(g, 1)
                    for x, p in ((kc, par[0]), (vc, par[1])))
            k, v = k[:L], v[:L]
            for h in range(hk * (H // Hk), (hk + 1) * (H // Hk)):
                s = st["scale"] * (st["q"][at:at + n, h].double() @ k.T)
                s = s + torch.full((n, L), float("-inf"), dtype=torch.float64,
                                   device=DEV).triu(L - n + 1)
                out[at:at + n, h] = torch.softmax(s, -1) @ v
        at += n
    return out
