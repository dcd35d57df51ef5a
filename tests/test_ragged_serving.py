"""The operators of ragged batches together, as a server runs them: prompts in chunks beside
decoding sequences, forks that share pages, windows that free them, compaction, captured steps.

Each sequence's projections are kept on the side; what a step attends is checked against fp64
from them, q and k turned in fp64 and rounded to fp16 as the cache holds them.  A value within the
kernel's 2^-19 of a border between two fp16 numbers may be rounded to the other one, a step of 2^-10 of
it, in one of 2^8 dims: that moves a score by 2^-10 |q_d k_d| D^-0.5, at most 1.4e-3 for |q_d k_d| <= 16, and
the output by p (1 - p) 2 max |v| times as much, 0.7e-3 max |v|.  With the probabilities' rounding (2^-11
of sum p |v - o|, at most 2^-10 max |v|) and the output's (2^-11 |o|) that is below 2^-9 max |v| + 2^-11 |o|;
2^-9 max |v| is asked for.
"""
import math

import pytest
import torch

from helm_amd.kernels import attention as ka
from helm_amd.kernels import fused

HQ, HKV, D, P = 8, 2, 128, 16
SLOTS = 96


class Server:
    """Sequences as lists of projected tokens, their pages, and the device tensors of a step."""

    def __init__(self, window=0, sinks=0, rot=D, inter=False, seed=0, batch=4, rows=96):
        self.window, self.sinks, self.rot, self.inter = window, sinks, rot, inter
        self.g = torch.Generator().manual_seed(seed)
        self.inv, self.scale = fused.rope_scaled_inv_freq(rot, 1e4, "yarn", 4.0, 64)
        self.k = torch.full((SLOTS, HKV, P, D), math.nan, dtype=torch.float16, device="cuda")
        self.v = torch.full((SLOTS, HKV, D, P), math.nan, dtype=torch.float16, device="cuda")
        self.pool = ka.PoolView.of_pool(self.k, self.v.transpose(2, 3))
        self.free = list(range(SLOTS))
        self.tokens = [[] for _ in range(batch)]          # rows of qkv
        self.pages = [[] for _ in range(batch)]
        self.users = {}                                   # slot -> sequences that hold it
        self.batch, self.rows, self.cols = batch, rows, 24
        dev = dict(device="cuda")
        self.qkv = torch.zeros(rows, (HQ + 2 * HKV) * D, dtype=torch.float16, **dev)
        self.table = torch.full((batch, self.cols), -1, dtype=torch.int32, **dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, **dev)
        self.starts = torch.zeros(batch + 1, dtype=torch.int32, **dev)
        self.q = torch.empty(rows, HQ, D, dtype=torch.float16, **dev)
        self.out = torch.empty(rows, HQ, D, dtype=torch.float16, **dev)
        self.ws = ka.AttnWorkspace(torch.device("cuda", 0))
        self.d_inv = self.inv.cuda()

    def take(self):
        s = self.free.pop(torch.randint(0, len(self.free), (1,), generator=self.g).item())
        self.users[s] = 1
        return s

    def drop(self, s):
        self.users[s] -= 1
        if not self.users[s]:
            del self.users[s]
            self.free.append(s)
            self.k[s], self.v[s] = math.nan, math.nan     # whoever still reads it shows

    def load(self, new):
        """Host side of a step: `new[b]` tokens for each sequence."""
        starts = [0]
        for b, n in enumerate(new):
            rows = torch.randn(n, (HQ + 2 * HKV) * D, generator=self.g).half()
            self.tokens[b] += list(rows)
            while len(self.pages[b]) * P < len(self.tokens[b]):
                self.pages[b].append(self.take())
            first = len(self.tokens[b]) - n
            if self.window:                               # pages that no token to come sees
                for j, s in enumerate(self.pages[b]):
                    if s >= 0 and j * P >= self.sinks and (j + 1) * P <= first - self.window + 1:
                        self.drop(s)
                        self.pages[b][j] = -1
            starts.append(starts[-1] + n)
        self.new = new
        for b in range(self.batch):
            row = self.pages[b] + [-1] * (self.cols - len(self.pages[b]))
            self.table[b] = torch.tensor(row, dtype=torch.int32)
        self.lens.copy_(torch.tensor([len(t) for t in self.tokens]))
        self.starts.copy_(torch.tensor(starts))
        live = [self.tokens[b][i] for b, n in enumerate(new) for i in range(len(self.tokens[b]) - n, len(self.tokens[b]))]
        self.qkv.zero_()
        if live:
            self.qkv[:len(live)] = torch.stack(live).cuda()
        self.out.fill_(7.0)

    def step(self, **kw):
        fused.rope_append(self.qkv, self.pool, self.table, self.lens, self.starts, P, self.d_inv, HQ, HKV, D, self.inter,
                          self.scale, q_out=self.q)
        ka.chunk_attention(self.q, self.pool, self.table, self.lens, self.starts, P, self.window, self.sinks,
                           workspace=self.ws, out=self.out, **kw)

    def turned(self, b):
        """q [n, HQ, D], k, v [n, HKV, D] of a sequence's tokens in fp64, rounded as the cache rounds."""
        x = torch.stack(self.tokens[b]).double().view(len(self.tokens[b]), -1, D)
        ang = torch.arange(len(x)).double()[:, None, None] * self.inv.double()
        c, s = torch.cos(ang) * self.scale, torch.sin(ang) * self.scale
        at = torch.arange(self.rot)
        re, im = (at[0::2], at[1::2]) if self.inter else (at[:self.rot // 2], at[self.rot // 2:])
        y = x[:, :HQ + HKV].clone()
        y[..., re], y[..., im] = x[:, :HQ + HKV, re] * c - x[:, :HQ + HKV, im] * s, x[:, :HQ + HKV, im] * c + x[:, :HQ + HKV, re] * s
        y = y.half().double()
        return y[:, :HQ], y[:, HQ:], x[:, HQ + HKV:]

    def check(self):
        row = 0
        out = self.out.cpu().double()
        for b, n in enumerate(self.new):
            if not n:
                continue
            q, k, v = self.turned(b)
            for p in range(len(q) - n, len(q)):
                j = torch.arange(p + 1)
                if self.window:
                    j = j[(j > p - self.window) | (j < self.sinks)]
                s = torch.einsum("hgd,khd->hgk", q[p].view(HKV, -1, D), k[j]) * D ** -0.5
                want = torch.einsum("hgk,khd->hgd", torch.softmax(s, -1), v[j]).reshape(HQ, D)
                err = (out[row] - want).abs().max().item()
                assert err <= 2.0 ** -9 * v.abs().max().item(), (b, p, err)
                row += 1
        assert (out[row:] == 7.0).all()                   # padding

    def fork(self, parents):
        """All sequences become children: the first of a parent goes on in its last page."""
        seen, fresh, tokens, pages = set(), [], [], []
        for p in parents:
            own = p in seen
            seen.add(p)
            fresh.append(self.take() if own else -1)
        lens = [len(self.tokens[p]) for p in parents]
        table, n = ka.fork_pages(self.pool, self.table, self.lens, torch.tensor(parents, dtype=torch.int32, device="cuda"),
                                 torch.tensor(fresh, dtype=torch.int32, device="cuda"), P)
        assert n.tolist() == lens
        old = self.pages
        for i, p in enumerate(parents):
            pages.append(table[i].tolist()[:max(len(old[p]), lens[i] // P + 1 if fresh[i] >= 0 else 0)])
            for s in pages[i]:
                if s >= 0 and s != fresh[i]:
                    self.users[s] += 1
            tokens.append(list(self.tokens[p]))
        for b in range(self.batch):
            for s in old[b]:
                if s >= 0:
                    self.drop(s)
        self.pages, self.tokens = pages, tokens

    def compact(self):
        """Pages at the pool's end move to its first free slots."""
        used = sorted(self.users)
        holes = [s for s in range(len(used)) if s not in self.users]
        moves = {s: h for s, h in zip([s for s in used if s >= len(used)], holes)}
        if not moves:
            return
        ka.copy_pages(self.pool, torch.tensor(list(moves), dtype=torch.int32, device="cuda"),
                      torch.tensor(list(moves.values()), dtype=torch.int32, device="cuda"), P)
        self.pages = [[moves.get(s, s) for s in row] for row in self.pages]
        self.users = {moves.get(s, s): n for s, n in self.users.items()}
        self.free = [s for s in range(SLOTS) if s not in self.users]
        for s in self.free:
            self.k[s], self.v[s] = math.nan, math.nan


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks,rot,inter", [(0, 0, D, False), (40, 3, 32, True), (17, 0, D // 2, False), (64, 16, D, True)])
def test_a_served_batch(window, sinks, rot, inter):
    s = Server(window, sinks, rot, inter)
    for new in ([70, 1, 0, 20], [26, 1, 64, 1], [0, 1, 1, 1], [1, 1, 1, 1]):
        s.load(new)
        s.step()
        s.check()
    s.fork([2, 2, 0, 2])
    for new in ([1, 1, 1, 1], [5, 1, 0, 3]):
        s.load(new)
        s.step(max_new=5)
        s.check()
    s.compact()
    s.load([1, 1, 1, 1])
    s.step(max_new=1)
    s.check()
    # the single-token form
    s.fork([1, 1, 1, 3])
    s.load([1, 1, 1, 1])
    s.step()
    one = ka.window_decode_attention(s.q[:4], s.pool, s.table, s.lens, P, s.window, s.sinks)
    s.out[:4] = one
    s.check()


@pytest.mark.gpu
def test_a_captured_step_serves_every_batch():
    """One graph of append and attention, replayed for prompts, mixed batches and decode; eager work
    between the replays."""
    s, e = Server(50, 4, 64, False, seed=3), Server(50, 4, 64, False, seed=3)
    s.load([3, 2, 1, 0]), e.load([3, 2, 1, 0])
    s.step(), e.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.step()
    graph.replay()
    for new in ([60, 20, 1, 9], [1, 1, 1, 1], [0, 0, 0, 90], [1, 1, 1, 1], [2, 40, 1, 30]):
        s.load(new), e.load(new)
        graph.replay()
        e.step()
        torch.cuda.synchronize()
        assert torch.equal(s.out, e.out)
        s.check()
        if new == [1, 1, 1, 1]:
            s.fork([3, 3, 0, 1]), e.fork([3, 3, 0, 1])
