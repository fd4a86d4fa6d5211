"""GPU: products captured into CUDA graphs -- each graph has a workspace of its own, so that
graphs captured on one stream replay beside one another, beside eager calls on that stream, and
after a larger call has replaced the stream's own workspace.  The shapes split along K, so that
every call uses arrival counters and partial sums."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import awq_b200
from awq_b200 import tp
from kernels import awq_gemm
from oracle import oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "ctypes"])
def glue(request, monkeypatch):
    """The C++ host glue, and the Python path that stands in for it where it is not built."""
    if request.param == "ctypes":
        monkeypatch.setattr(awq_b200, "_ext", None)
    else:
        assert awq_b200._ext is not None


def layer(K, N, seed):
    w = [torch.from_numpy(a).cuda() for a in O.make_awq_layer(K, N, 128, seed=seed)]
    b = torch.from_numpy((0.1 * np.random.default_rng(seed).standard_normal(N)).astype(np.float16)).cuda()
    return w, b


CALLS = {
    "gemm": lambda x, w, b: awq_gemm.awq_gemm_forward(x, *w, 128),
    "bias": lambda x, w, b: awq_gemm.awq_gemm_bias_forward(x, *w, b, 128),
    "silu_mul": lambda x, w, b: awq_gemm.awq_gemm_silu_mul_forward(x, *w, 128),
    "epilogue": lambda x, w, b: awq_gemm.awq_gemm_epilogue_forward(x, *w, 128, bias=b, activation="gelu"),
}


def capture(stream, fn):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = fn()
    return g, out


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("M,K,N", [(1, 18944, 3584), (12, 3584, 4608), (300, 1024, 1024)])
def test_graphs_beside_one_another_and_eager_calls(cuda, glue, call, M, K, N):
    w, b = layer(K, N, M)
    fn = CALLS[call]
    xs = [torch.from_numpy(O.make_x(M, K, seed=i)).cuda() for i in range(3)]
    want = [fn(x, w, b) for x in xs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):                        # nothing ran on this stream before
        # two calls a graph, the second on the first one's counters
        graphs = [capture(s, lambda: (fn(x, w, b), fn(x, w, b))) for x in xs[:2]]
    torch.cuda.synchronize()
    a, c = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        for st, (g, _) in zip((a, c), reversed(graphs)):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(s):
            out = fn(xs[2], w, b)
    torch.cuda.synchronize()
    assert torch.equal(out, want[2])
    for (_, outs), ref in zip(graphs, want):
        assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)
    assert awq_b200.device_status() == 0


def test_graph_after_a_larger_call_on_its_stream(cuda, glue):
    """The stream's workspace is replaced by a larger one, and its memory taken by others: the
    graph neither reads nor writes it."""
    w, _ = layer(18944, 3584, 1)
    x = torch.from_numpy(O.make_x(1, 18944, seed=1)).cuda()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        want = awq_b200.gemm(x, *w, 128)
        g, out = capture(s, lambda: awq_b200.gemm(x, *w, 128))
        big = torch.from_numpy(O.make_x(300, 18944, seed=2)).cuda()
        awq_b200.gemm(big, *w, 128)
        # of every size that the first workspace's block could serve
        taken = [torch.full((n,), 77, dtype=torch.uint8, device="cuda")
                 for n in (1 << 20, 1 << 19, 1 << 20, 2 << 20, 4 << 20, 8 << 20, 20 << 20)]
        for _ in range(3):
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all((t == 77).all() for t in taken)


def test_captured_attention_blocks_beside_one_another(cuda):
    """Two graphs of AttentionLinearsTP.attend and an MLP, each with its cache, captured on one
    stream and replayed on two: the q/k/v and gate+up products as well have their own workspaces."""
    HID, H, HK, D, INTER, PAGE, R = 3584, 28, 4, 128, 2048, 16, 2

    def wt(K, N, seed, bias=None):                    # outputs near the inputs' size
        (qw, qz, sc), _ = layer(K, N, seed)
        return tp.AWQWeights(qw, qz, (sc / 64).contiguous(), 128, bias)
    attn = tp.AttentionLinearsTP(wt(HID, (H + 2 * HK) * D, 1, layer(HID, (H + 2 * HK) * D, 1)[1]),
                                 wt(H * D, HID, 2), H, HK, D, 1, 0)
    mlp = tp.TensorParallelMLP(wt(HID, 2 * INTER, 3), wt(INTER, HID, 4), INTER, 1, 0)
    i32 = dict(dtype=torch.int32, device="cuda")
    inv = (1e4 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().cuda()
    table = torch.arange(R, **i32)[:, None].contiguous()
    lens, pos = torch.full((R,), 1, **i32), torch.zeros(R, **i32)
    slots = torch.arange(R, device="cuda") * PAGE
    s = torch.cuda.Stream()

    def block(x, cache):
        y = attn.attend(x, cache, slots, table, lens, pos, inv, (D // 2,), residual=x)
        return mlp(y, residual=y)
    xs = [torch.from_numpy(O.make_x(R, HID, seed=i)).cuda() for i in range(2)]
    caches = [awq_b200.KV4Cache.allocate(R, HK, D, PAGE) for _ in xs]
    want = [block(x, c) for x, c in zip(xs, caches)]
    assert all(torch.isfinite(w).all() for w in want)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graphs = [capture(s, lambda: block(x, c)) for x, c in zip(xs, caches)]
    torch.cuda.synchronize()
    for _ in range(30):
        for st, (g, _) in zip((torch.cuda.Stream(), torch.cuda.Stream()), reversed(graphs)):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
    for (_, out), ref in zip(graphs, want):
        assert torch.equal(out, ref)
    assert awq_b200.device_status() == 0
