"""GPU: the operators between the products run together, as a decoder layer uses them:
kv4_pages_step -> AttentionLinearsTP.attend (q/k/v product, rotary positions, append,
attention, o product with residual) -> MLP with residual, over prompts, captured decode steps,
a replaced request and a padded batch."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import awq_b200
from awq_b200 import tp
from oracle import layer as L
from oracle import oracle as O

pytestmark = pytest.mark.gpu
HID, H, HK, D, INTER, GS, PAGE = 256, 4, 2, 64, 512, 64, 16
U16 = 2.0 ** -11


def weights(K, N, seed, bias=False):
    qw, qz, s = (torch.from_numpy(a).cuda() for a in O.make_awq_layer(K, N, GS, seed=seed))
    b = torch.from_numpy((0.1 * np.random.default_rng(seed).standard_normal(N)).astype(np.float16)).cuda()
    return tp.AWQWeights(qw, qz, s, GS, b if bias else None)


class State:
    def __init__(self, R, blocks, pages):
        i32 = dict(dtype=torch.int32, device="cuda")
        self.cache = awq_b200.KV4Cache.allocate(pages, HK, D, PAGE, 32)
        self.cache.data.fill_(0xFF)                      # unwritten scales are NaN
        self.table = torch.full((R, blocks), -1, **i32)
        self.held, self.lens = torch.zeros(R, **i32), torch.zeros(R, **i32)
        self.free = torch.arange(pages, **i32)
        self.count = torch.full((1,), pages, **i32)
        self.new = torch.zeros(R, **i32)
        self.reset = torch.zeros(R, dtype=torch.bool, device="cuda")

    def pages(self, max_tokens):
        return awq_b200.kv4_pages_step(self.table, self.held, self.free, self.count, self.lens,
                                       self.new, PAGE, max_tokens, self.reset)


@pytest.fixture(scope="module")
def layer(request):
    attn = tp.AttentionLinearsTP(weights(HID, (H + 2 * HK) * D, 1, bias=True),
                                 weights(H * D, HID, 2, bias=True), H, HK, D, 1, 0)
    mlp = tp.TensorParallelMLP(weights(HID, 2 * INTER, 3), weights(INTER, HID, 4), INTER, 1, 0)
    inv = (1e4 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().cuda()
    return attn, mlp, inv


def run(layer, st, x, max_tokens, max_q, ragged=True):
    attn, mlp, inv = layer
    slots, pos, cu, lens, status = st.pages(max_tokens)
    y = attn.attend(x, st.cache, slots, st.table, lens, pos, inv, (D // 2,),
                    cu_q=cu if ragged else None, max_q=max_q, residual=x)
    z = mlp(y, residual=y)
    return y, z, slots, pos, cu, lens, status


def check(layer, st, x, out, ragged, max_q):
    """Each stage again on its own inputs: the composition's bits, and the cached values and
    the attention against 64 bits."""
    attn, mlp, inv = layer
    y, z, slots, pos, cu, lens, status = out
    assert int(status) == 0
    T = x.shape[0]
    q, k, v = (t.unflatten(-1, (-1, D)) for t in attn.project_qkv(x))
    rq, rk = awq_b200.rope_axes(q, k, pos, inv, (D // 2,))
    live = slots >= 0
    gk, gv = awq_b200.kv4_gather(st.cache, slots)
    for got, src in ((gk, rk), (gv, v)):
        vals = L.values(*L.quantize(src.cpu().numpy(), 32))
        err = np.abs(got.double().cpu().numpy() - vals)[live.cpu().numpy()]
        assert (err <= (U16 + 2.0 ** -24) * np.abs(vals)[live.cpu().numpy()] + 2.0 ** -25).all()
    a = awq_b200.kv4_attention(rq, st.cache, st.table, lens, cu if ragged else None, max_q)
    want = tp._default_epilogue()(a.view(T, -1), attn.o.w.qweight, attn.o.w.qzeros, attn.o.w.scales,
                                  GS, bias=attn.o.w.bias, residual=x)
    assert torch.equal(y, want)
    assert torch.equal(z, mlp(y, residual=y))
    # attention of the last request's last row, from the cache's bytes
    cu_h, lens_h = cu.tolist(), lens.tolist()
    data, table = st.cache.data.cpu().numpy(), st.table.cpu().numpy()
    for r in range(len(lens_h)):
        n, Lr = cu_h[r + 1] - cu_h[r], lens_h[r]
        if n == 0:
            continue
        at = table[r, np.arange(Lr) // PAGE] * PAGE + np.arange(Lr) % PAGE
        K, V = L.read_slots(data, at, D, PAGE, 32)
        ref = L.attention(rq[cu_h[r]:cu_h[r + 1]].cpu().numpy(), K, V, D ** -0.5)
        got = a[cu_h[r]:cu_h[r + 1]].double().cpu().numpy()
        # weights in fp16 (u16 of sums of |values|) and the output's rounding; the scores are
        # small here, so their fp32 errors stay below a tenth of that
        assert (np.abs(got - ref) <= 2.2 * U16 * np.abs(V).max() + U16 * np.abs(ref)).all()


def test_prompts_then_captured_steps_then_replacement(cuda, layer):
    R, rng = 3, torch.Generator(device="cuda").manual_seed(5)
    st = State(R, 12, 40)
    make = lambda n: (torch.randn((n, HID), device="cuda", generator=rng) * 0.5).half()
    # prompts of 40, 0 and 75 tokens in a batch padded to 120 rows
    st.new.copy_(torch.tensor([40, 0, 75]))
    x = make(120)
    out = run(layer, st, x, 120, 75)
    check(layer, st, x, out, True, 75)
    assert out[4].tolist() == [0, 40, 40, 115] and (out[2][115:] == -1).all()
    pad = layer[0].o.w.bias + x[115:]                    # rows behind the last token
    assert torch.allclose(out[0][115:].float(), pad.float(), atol=0, rtol=2.0 ** -10)
    st.lens.copy_(out[5])
    # a captured decode step for all rows, the empty one included
    st.new.fill_(1)
    xs = make(R)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            cap = run(layer, st, xs, R, 1, ragged=False)
    for step in range(20):
        xs.copy_(make(R))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        if step in (0, 8, 19):
            check(layer, st, xs, cap, False, 1)
        assert cap[5].tolist() == [41 + step, 1 + step, 76 + step]
        st.lens.copy_(cap[5])
    # the first request gives its pages to a new prompt while the others step on
    before = int(st.count)
    st.reset.copy_(torch.tensor([True, False, False]))
    st.lens[0] = 0
    st.new.copy_(torch.tensor([90, 1, 1]))
    x = make(92)
    out = run(layer, st, x, 92, 90)
    check(layer, st, x, out, True, 90)
    assert int(st.count) == before + 4 - 6 - sum(int(n) % PAGE == 1 for n in out[5][1:])
    assert awq_b200.device_status() == 0


def test_refused_step_runs_through_harmlessly(cuda, layer):
    """A step that is short of pages has no tokens: nothing is written, the rows give the
    residual and o's bias."""
    st = State(2, 4, 2)
    st.new.copy_(torch.tensor([20, 20]))
    x = torch.randn((40, HID), device="cuda").half()
    before = st.cache.data.clone()
    y, z, slots, pos, cu, lens, status = run(layer, st, x, 40, 20)
    assert int(status) == 2 and (slots == -1).all() and cu.tolist() == [0, 0, 0]
    assert torch.equal(st.cache.data, before) and int(st.count) == 2
    want = (x.float() + layer[0].o.w.bias.float()).half()
    assert torch.equal(y, want)
    assert awq_b200.device_status() == 0


def test_attend_refusals(cuda, layer):
    attn = layer[0]
    st = State(1, 4, 4)
    x = torch.zeros((1, HID), dtype=torch.float16, device="cuda")
    slots, pos, cu, lens, _ = st.pages(1)
    other = awq_b200.KV4Cache.allocate(4, 1, D, PAGE, 32)
    with pytest.raises(ValueError, match="cache holds"):
        attn.attend(x, other, slots, st.table, lens, pos, layer[2], (D // 2,))
    odd = tp.AttentionLinearsTP(weights(HID, (H + 2 * HK) * D, 1), weights(H * D, HID, 2), H, HK, D, 3, 1)
    with pytest.raises(ValueError, match="whole groups"):
        odd.attend(x, st.cache, slots, st.table, lens, pos, layer[2], (D // 2,))


def test_step_without_tokens(cuda, layer):
    """A step of requests that all pause: no rows, no pages, no change."""
    st = State(2, 4, 4)
    before = st.cache.data.clone()
    y, z, slots, pos, cu, lens, status = run(layer, st, torch.zeros((0, HID), dtype=torch.float16,
                                                                    device="cuda"), 0, 1)
    assert y.shape == z.shape == (0, HID) and slots.shape == pos.shape == (0,)
    assert int(status) == 0 and cu.tolist() == [0, 0, 0] and lens.tolist() == [0, 0]
    assert torch.equal(st.cache.data, before) and int(st.count) == 4
    assert awq_b200.device_status() == 0
