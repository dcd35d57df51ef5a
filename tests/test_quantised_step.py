"""A decoder step on 4-bit weights and 8-bit KV pages, ended by a drawn token: int4_linear,
qk_norm_rope_append_q8, paged_decode_attention_q8 and sample behind each other, as a serving
loop runs them.  Each operator is held to its definition at the inputs that the operators
ahead of it gave (tolerances as their own tests derive them); whole steps are compared bit
for bit between eager runs, replayed graphs, streams and batch paddings."""
import math

import numpy as np
import pytest
import torch

from helm_amd import kernels as hk
from helm_amd.kernels import attention as ka
from helm_amd.kernels import fused
from test_int4_linear import check as check_int4
from test_kv_q8 import EPS, check_attention, held, quantised, random_pool, rope_reference
from test_sample import definition

HQ, HKV, D, P, H, VOCAB = 8, 2, 64, 16, 320, 1500
QKV = (HQ + 2 * HKV) * D


class Step:
    """Weights, pages and the step over them; every buffer is made once."""

    def __init__(self, b, pages=12, seed=0):
        g = torch.Generator().manual_seed(seed)

        def weight(n, k, gs):
            c, s = hk.quantize_int4(torch.randn(n, k, generator=g) * k ** -0.5, gs)
            return (c, s, gs), hk.Int4Weight.pack(c, s).to("cuda")
        self.plain_qkv, self.w_qkv = weight(QKV, H, 64)
        self.plain_o, self.w_o = weight(H, HQ * D, 128)
        self.plain_head, self.w_head = weight(VOCAB, H, 32)
        self.qn, self.kn = ((1 + 0.1 * torch.randn(D, generator=g)).half().cuda() for _ in range(2))
        self.inv = (1e6 ** (-torch.arange(0, D, 2).double() / D)).float().cuda()
        self.pool = random_pool(b * pages, HKV, P, D, seed + 1)
        self.table = torch.randperm(b * pages, generator=g).int().view(b, pages).cuda()
        self.x = torch.empty(b, H, dtype=torch.float16, device="cuda")
        self.u = torch.empty(b, device="cuda")
        self.pos = torch.zeros(b, dtype=torch.int32, device="cuda")
        self.lens, self.slots, self.offs = (torch.zeros_like(self.pos) for _ in range(3))
        self.workspace = ka.AttnWorkspace(torch.device("cuda", 0))
        self.drawn = fused.sample_workspace(b, VOCAB, "cuda")

    def place(self, x, u, pos):
        """Inputs of a step at positions `pos` (below 0: the item is padding)."""
        self.x.copy_(x)
        self.u.copy_(u)
        pos = torch.tensor(pos, dtype=torch.int32)
        live = pos >= 0
        at = pos.clamp(min=0)
        page = self.table.cpu()[torch.arange(len(pos)), (at // P).long()]
        self.pos.copy_(at)
        self.lens.copy_(torch.where(live, pos + 1, 0))
        self.slots.copy_(torch.where(live, page, -1))
        self.offs.copy_(at % P)

    def run(self, splits=0):
        qkv = hk.int4_linear(self.x, self.w_qkv)
        q = fused.qk_norm_rope_append_q8(qkv, self.qn, self.kn, EPS, self.pos, self.inv, None, self.pool, self.slots,
                                         self.offs, HQ, HKV, D, P)
        o = ka.paged_decode_attention_q8(q, self.pool, self.table, self.lens, P, num_splits=splits, workspace=self.workspace)
        y = hk.int4_linear(o.view(-1, HQ * D), self.w_o)
        logits = hk.int4_linear(y, self.w_head)
        return qkv, q, o, y, logits, fused.sample(logits, self.u, 0.8, 40, 0.95, 0.0, workspace=self.drawn)


def inputs(b, n, seed):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(b, H, generator=g).half().cuda(), torch.rand(b, generator=g).cuda()) for _ in range(n)]


def bytes_of(pool):
    return [t.clone() for t in (pool.k, pool.v, pool.k_scale, pool.v_scale)]


@pytest.mark.gpu
@pytest.mark.parametrize("pos", [[0], [150], [0, 15, 16, 17, 100, 191], [3 * i for i in range(20)]])
def test_every_operator_at_the_step_s_own_values(cuda, pos):
    b = len(pos)
    s = Step(b, seed=b)
    s.place(*inputs(b, 1, 5)[0], pos)
    qkv, q, o, y, logits, token = s.run()
    for out, x, (c, sc, gs) in ((qkv, s.x, s.plain_qkv), (y, o.view(b, -1), s.plain_o), (logits, y, s.plain_head)):
        check_int4(out, x, c, sc, None, gs)
    eq, ek, ev = rope_reference(qkv.cpu(), s.qn.cpu(), s.kn.cpu(), s.pos.cpu(), s.inv.cpu(), HQ, HKV, D)
    top = eq.abs().amax(-1, keepdim=True)
    assert ((q.cpu().double() - eq).abs() <= 2.0 ** -11 * eq.abs() + 2.0 ** -20 * top + 2.0 ** -25).all()
    at = (s.slots.cpu().long(), slice(None), s.offs.cpu().long())
    c, sc = quantised(ev.half())
    assert torch.equal(s.pool.v.cpu()[at], c) and torch.equal(s.pool.v_scale.cpu()[at], sc)
    ks = s.pool.k_scale.cpu()[at].double()[..., None]
    top = ek.abs().amax(-1, keepdim=True)
    assert ((held(s.pool)[0][at] - ek).abs() <= ks * (0.5 + 127 * 2.0 ** -11) + 2.0 ** -20 * top).all()
    check_attention(o, q, s.pool, s.table, s.lens, 1 / math.sqrt(D))
    rows, u = logits.cpu().numpy(), s.u.cpu().numpy()
    for i in range(b):
        want, near = definition(rows[i], u[i], 0.8, 40, 0.95, 0.0)
        assert near > 1e-12 and int(token[i]) == want


@pytest.mark.gpu
def test_replayed_graph_equals_eager_steps(cuda):
    """Twelve tokens, each by an eager step on one pool and by a replay on another, eager work of
    the other pool and a synchronization in between."""
    b = 5
    eager, held_by_graph = Step(b, seed=3), Step(b, seed=3)
    held_by_graph.place(*inputs(b, 1, 9)[0], [-1] * b)      # nothing is written by the first runs
    held_by_graph.run(3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = held_by_graph.run(3)
    for n, (x, u) in enumerate(inputs(b, 12, 4)):
        pos = [n + 13, n, 80 + n, -1 if n % 3 else n, 31 + n]
        eager.place(x, u, pos)
        want = [t.clone() for t in eager.run(3)]
        held_by_graph.place(x, u, pos)
        graph.replay()
        torch.cuda.synchronize()
        for w, g in zip(want, out):
            assert torch.equal(w, g)
        for w, g in zip(bytes_of(eager.pool), bytes_of(held_by_graph.pool)):
            assert torch.equal(w, g)


@pytest.mark.gpu
def test_two_graphs_with_their_own_workspaces_in_turn(cuda):
    steps = [Step(3, seed=7), Step(3, seed=8)]
    twins = [Step(3, seed=7), Step(3, seed=8)]
    graphs, outs = [], []
    for s in steps:
        s.place(*inputs(3, 1, 1)[0], [-1] * 3)
        s.run(4)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(s.run(4))
    streams = [torch.cuda.Stream() for _ in steps]
    for n, (x, u) in enumerate(inputs(3, 4, 2)):
        want = []
        for s, t in zip(steps, twins):
            s.place(x, u, [n, 40 + n, 150])
            t.place(x, u, [n, 40 + n, 150])
            want.append([o.clone() for o in t.run(4)])
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert all(torch.equal(a, c) for a, c in zip(w, o))


@pytest.mark.gpu
def test_on_another_stream_than_the_tensors_own(cuda):
    a, c = Step(4, seed=2), Step(4, seed=2)
    x, u = inputs(4, 1, 3)[0]
    for s in (a, c):
        s.place(x, u, [5, 70, 16, 0])
    want = a.run(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run(2)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    assert all(torch.equal(x, y) for x, y in zip(bytes_of(a.pool), bytes_of(c.pool)))


@pytest.mark.gpu
def test_padding_items_leave_the_others_and_the_pages_alone(cuda):
    """Items of a padded batch (no slot, no tokens) write nothing and answer zeros."""
    whole, part = Step(6, seed=4), Step(6, seed=4)
    x, u = inputs(6, 1, 6)[0]
    whole.place(x, u, [9, 33, 64, 100, 15, 16])
    part.place(x, u, [9, -1, 64, 100, -1, -1])
    before = bytes_of(part.pool)
    want, got = whole.run(2), part.run(2)
    keep, pad = [0, 2, 3], [1, 4, 5]
    for w, g in zip(want, got):
        assert torch.equal(w[keep], g[keep])
    assert not got[2][pad].any() and not got[4][pad].any()
    written = {(int(part.slots[i]), int(part.offs[i])) for i in keep}
    for old, new in zip(before, bytes_of(part.pool)):
        same = (old == new).cpu()
        assert {(s, t) for s, _, t, *_ in np.argwhere(~same.numpy()).tolist()} <= written


@pytest.mark.gpu
def test_a_prompt_then_steps_agree_with_steps_alone(cuda):
    """Pages written by a prompt of 700 tokens hold what one step per token would have left."""
    n, p = 700, 16
    g = torch.Generator().manual_seed(12)
    heads, kv = 16, 8
    qkv = torch.randn(n, (heads + 2 * kv) * D, generator=g).half().cuda()
    inv = (1e6 ** (-torch.arange(0, D, 2).double() / D)).float().cuda()
    pos = torch.arange(n, dtype=torch.int32, device=cuda)
    table = torch.randperm(44, generator=g).int().cuda()
    slots, offs = table[(pos // p).long()], pos % p
    pools = [ka.alloc_q8_pool(44, kv, p, D, cuda) for _ in range(2)]
    q = fused.qk_norm_rope_append_q8(qkv, None, None, EPS, pos, inv, None, pools[0], slots, offs, heads, kv, D)
    for i in range(n):
        one = fused.qk_norm_rope_append_q8(qkv[i:i + 1], None, None, EPS, pos[i:i + 1], inv, None, pools[1], slots[i:i + 1],
                                           offs[i:i + 1], heads, kv, D)
    assert torch.equal(one, q[-1:])
    assert all(torch.equal(a, c) for a, c in zip(bytes_of(pools[0]), bytes_of(pools[1])))
    # and the prompt's own attention over the pages as fp16
    view = ka.dequantize_pages(pools[0], table)
    last = ka.prefill_attention(q, view, torch.arange(44, dtype=torch.int32, device=cuda), p)[-1:]
    o = ka.paged_decode_attention_q8(q[-1:], pools[0], table[None], torch.tensor([n], dtype=torch.int32, device=cuda))
    check_attention(o, q[-1:], pools[0], table[None], torch.tensor([n]), 1 / math.sqrt(D))
    # the fp16 copy rounds each value by 2^-11: a score by delta = 2^-11 scale sum |q k|, the weights by a
    # factor e^(2 delta) at most and so their mean of V by 4 delta max |V|; the prompt kernel's weights in fp16
    # 2^-10 max |V|, the copy of V and the two results 2^-11 each
    k, v = (t[table.cpu().long()].transpose(0, 1).reshape(kv, -1, D)[:, :n] for t in held(pools[0]))
    delta = 2.0 ** -11 * D ** -0.5 * float((q[-1].cpu().double().abs().view(kv, -1, D) @ k.abs().transpose(1, 2)).max())
    assert float((last.double() - o.double()).abs().max()) <= (4 * delta + 2.0 ** -10 + 3 * 2.0 ** -11) * float(v.abs().max())
