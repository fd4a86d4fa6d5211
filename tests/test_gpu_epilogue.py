"""GPU: awq_b200.gemm_epilogue (act(x @ W + bias) + residual) on every kernel family against
the 64-bit form.

Tolerance.  S = sum |x| |W|.  The product is off by at most e = K 2^-23 S (fp32 sums, counted
as truncated) + u16 S up to 4 tokens, where the decode kernel keeps (w - z) s unrounded while
the oracle's W is the fp16 one (u16 = 2^-11).  Every activation's slope is at most 1.13, and
its own fp32 arithmetic (hardware exponential, approximate divide, erfc) is within 2^-20 of
|y|.  Then one fp16 rounding: |err| <= 1.13 e + 2^-20 |y| + u16 |out| + 2^-25.
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import awq_b200
from kernels import awq_gemm
from oracle import layer as L
from oracle import oracle as O

pytestmark = pytest.mark.gpu
U16 = 2.0 ** -11


def make(M, K, N, gs, seed):
    rng = np.random.default_rng(seed)
    qw, qz, s = O.make_awq_layer(K, N, gs, seed=seed)
    x = O.make_x(M, K, seed=seed + 1)
    bias = (0.5 * rng.standard_normal(N)).astype(np.float16)
    res = (2 * rng.standard_normal((M, N))).astype(np.float16)
    return x, qw, qz, s, bias, res


def dev(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


def product(x, qw, qz, s, gs):
    """y and S in float64, on the GPU (the shapes here reach 2048 x 3584 x 4096)."""
    W = torch.from_numpy(O.awq_dequant(qw, qz, s, gs)).cuda().double()
    x = torch.from_numpy(x).cuda().double()
    return (x @ W).cpu().numpy(), (x.abs() @ W.abs()).cpu().numpy()


def check(got, y, S, M, K, bias, act, res):
    e = K * 2.0 ** -23 * S + (U16 * S if M <= 4 else 0)
    pre = y if bias is None else y + bias.astype(np.float64)
    ref = L.epilogue(y, bias, act, res)
    tol = 1.13 * e + 2.0 ** -20 * np.abs(pre) + U16 * np.abs(ref) + 2.0 ** -25
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= tol).all(), float((err / tol).max())


# decode (4 and 8 token sets, split and not), small-M, prefill (split-K, grid, stream-K,
# persistent), 16-token launches, and N % 32 != 0 (generic kernel)
SHAPES = [(1, 512, 256, 128), (4, 1024, 3584, 128), (8, 512, 4608, 64), (7, 256, 64, 64),
          (12, 512, 512, 128), (16, 1024, 37888, 128), (40, 512, 256, 128), (33, 256, 72, 128),
          (3, 256, 40, 64), (300, 1024, 768, 128), (100, 512, 512, 64), (2048, 256, 3584, 128),
          (2048, 4096, 3584, 128), (2047, 256, 5120, 128), (1500, 18944, 3584, 128)]


@pytest.mark.parametrize("M,K,N,gs", SHAPES)
def test_epilogue_every_kernel(cuda, M, K, N, gs):
    x, qw, qz, s, bias, res = make(M, K, N, gs, seed=M + N)
    y, S = product(x, qw, qz, s, gs)
    xd, qwd, qzd, sd, bd, rd = dev(x, qw, qz, s, bias, res)
    acts = ["none", "relu", "silu", "gelu", "gelu_tanh"] if M * N < 200000 else ["none", "gelu_tanh"]
    for act in acts:
        out = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, bias=bd, activation=act, residual=rd)
        check(out, y, S, M, K, bias, act, res)
    out = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, activation="silu")
    check(out, y, S, M, K, None, "silu", None)
    # nothing but the product: the product's own bits
    out = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, bias=bd)
    assert torch.equal(out, awq_b200.gemm(xd, qwd, qzd, sd, gs, bias=bd))
    assert torch.equal(awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs), awq_b200.gemm(xd, qwd, qzd, sd, gs))
    # the residual stream in place, and with strided rows (odd strides read element by element)
    want = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, residual=rd)
    check(want, y, S, M, K, None, "none", res)
    for pad in (8, 3):
        wide = torch.zeros((M, N + pad), dtype=torch.float16, device="cuda")
        wide[:, :N] = rd
        assert torch.equal(awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, residual=wide[:, :N]), want)
    stream = rd.clone()
    assert awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, residual=stream, out=stream) is stream
    assert torch.equal(stream, want)
    assert awq_b200.device_status() == 0


def test_shapes_reach_every_prefill_schedule(cuda):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    lib, kinds = awq_b200._lib.load(), set()
    for M, K, N, _ in SHAPES:
        if M > 64:
            k, p = ctypes.c_int(), ctypes.c_int()
            lib.awq_tc_schedule(M, N, K, sms, ctypes.byref(k), ctypes.byref(p))
            kinds.add(k.value)
    assert kinds == {0, 1, 2, 3}


def test_drop_in_shape_and_empty(cuda):
    x, qw, qz, s, bias, res = make(6, 512, 256, 128, seed=1)
    xd, qwd, qzd, sd, bd, rd = dev(x, qw, qz, s, bias, res)
    out = awq_gemm.awq_gemm_epilogue_forward(xd.view(2, 3, 512), qwd, qzd, sd, 128, bias=bd,
                                             activation="relu", residual=rd.view(2, 3, 256))
    assert out.shape == (2, 3, 256)
    assert torch.equal(out.view(6, 256), awq_b200.gemm_epilogue(xd, qwd, qzd, sd, 128, bias=bd,
                                                                activation="relu", residual=rd))
    assert awq_b200.gemm_epilogue(xd[:0], qwd, qzd, sd, 128, residual=rd[:0]).shape == (0, 256)


def test_activation_extremes(cuda):
    """Saturated, huge, infinite and NaN sums through every activation, on each kernel."""
    K, N = 64, 64
    qw, qz, s = O.make_awq_layer(K, N, 64, seed=4)
    vals = np.array([0.0, -0.0, 30.0, -30.0, 100.0, -100.0, 60000.0, -60000.0, 1e-7, np.nan],
                    np.float16)
    bias = np.resize(vals, N)
    for M in (1, 12, 100):
        x = np.zeros((M, K), np.float16)
        xd, qwd, qzd, sd, bd = dev(x, qw, qz, s, bias)
        for act in ("none", "relu", "silu", "gelu", "gelu_tanh"):
            got = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, 64, bias=bd, activation=act)
            got = got.double().cpu().numpy()
            with np.errstate(over="ignore"):
                ref = L.activate(bias.astype(np.float64), act)
            assert np.array_equal(np.isnan(got), np.broadcast_to(np.isnan(ref), got.shape))
            ok = ~np.isnan(ref)
            assert (np.abs(got - ref)[:, ok] <= (U16 + 2.0 ** -20) * np.abs(ref[ok]) + 2.0 ** -25
                    + 2.0 ** -20 * np.abs(bias[ok].astype(np.float64)) * (np.abs(ref[ok]) > 0)).all()


def test_graphs_replay_at_the_same_time(cuda):
    """Two captured split-K calls of one stream, replayed on two streams: own workspaces."""
    x, qw, qz, s, bias, res = make(1, 18944, 3584, 128, seed=6)
    xd, qwd, qzd, sd, rd = dev(x, qw, qz, s, res)
    want = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, 128, residual=rd)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(st):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                out = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, 128, residual=rd)
            graphs.append((g, out))
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(50):
        for stream, (g, _) in zip((a, b), graphs):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out, want)


def test_residual_where_the_generic_kernel_takes_several_launches(cuda):
    """N % 32 != 0 and more 16-token chunks than one launch has counters for: 148 column strips,
    so 110 chunks a launch, and the last 40 rows in a second one."""
    M, K, N, gs = 1800, 64, 37880, 64
    first = 16384 // -(-N // 256) * 16
    assert first == 1760
    x, qw, qz, s, bias, _ = make(M, K, N, gs, seed=8)
    rd = (2 * torch.randn((M, N), device="cuda", generator=torch.Generator("cuda").manual_seed(9))).half()
    xd, qwd, qzd, sd, bd = dev(x, qw, qz, s, bias)
    rows = [*range(8), *range(first - 8, M)]
    y, S = product(x[rows], qw, qz, s, gs)
    res = rd[rows].cpu().numpy()
    out = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, bias=bd, activation="relu", residual=rd)
    check(out[rows], y, S, M, K, bias, "relu", res)
    # a residual of wider rows, and the residual stream in place
    want = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, residual=rd)
    check(want[rows], y, S, M, K, None, "none", res)
    wide = torch.zeros((M, N + 8), dtype=torch.float16, device="cuda")
    wide[:, :N] = rd
    assert torch.equal(awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, residual=wide[:, :N]), want)
    awq_b200.gemm_epilogue(xd, qwd, qzd, sd, gs, residual=rd, out=rd)
    assert torch.equal(rd, want)
    assert awq_b200.device_status() == 0


def test_activation_of_infinite_sums(cuda):
    """+-inf through every activation as its formula gives them: y / (1 + exp(-y)) and the gelu
    forms are inf at inf and -inf / inf or -inf * 0 = NaN at -inf."""
    inf, nan = np.inf, np.nan
    want = {"none": (inf, -inf), "relu": (inf, 0.0), "silu": (inf, nan), "gelu": (inf, nan),
            "gelu_tanh": (inf, nan)}
    for M, K, N in ((1, 64, 64), (12, 64, 64), (100, 64, 64), (300, 64, 512), (20, 64, 40)):
        qw, qz, s = O.make_awq_layer(K, N, 64, seed=4)
        x = np.zeros((M, K), np.float16)
        bias = np.resize(np.array([inf, -inf, 1.0], np.float16), N)
        xd, qwd, qzd, sd, bd = dev(x, qw, qz, s, bias)
        for act, (plus, minus) in want.items():
            got = awq_b200.gemm_epilogue(xd, qwd, qzd, sd, 64, bias=bd, activation=act).float().cpu().numpy()
            for at, ref in ((bias == inf, plus), (bias == -inf, minus)):
                assert np.array_equal(got[:, at], np.full((M, at.sum()), ref, np.float32), equal_nan=True), act
            assert np.isfinite(got[:, bias == 1]).all()
