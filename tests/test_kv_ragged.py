"""Rotary positions of a ragged batch into pages, and pages moved inside a pool: refusals on the
CPU; on the GPU against the definition in fp64, moved bytes bit for bit.

Tolerance of a rotated value: one rounding to fp16 (2^-11 of it), and in fp32 the norm's factor
(D products and sums in order-free 8 + log2 steps, rsqrt, two products: 2^-20 of a value with
room), cos and sin (2^-22 each), two products and a sum of values up to sqrt 2 of the pair's
length: 2^-19 of the pair's length in all.
"""
import ctypes
import math
import re

import pytest
import torch

from helm_amd import _native
from helm_amd.kernels import attention as ka
from helm_amd.kernels import fused

FAKE = ctypes.c_void_p(16)             # never dereferenced: the checks fail first


def c_pool(hkv=2, p=16, d=64, slots=8, **kw):
    f = dict(k=16, v=16, k_slot_stride=hkv * p * d, k_head_stride=p * d, v_slot_stride=hkv * d * p, v_head_stride=d * p,
             v_dim_stride=p, num_slots=slots)
    f.update(kw)
    return ka.KvPoolStruct(*f.values())


def last_error():
    return _native.lib().helm_last_error().decode()


# ── refusals ─────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("change, code, text", [
    (dict(qkv=None), -1, "null"), (dict(pt=None), -1, "null"), (dict(lens=None), -1, "null"), (dict(q=None), -1, "null"),
    (dict(inv=None), -1, "null"), (dict(kw=None), -1, "both"), (dict(N=0), -1, "positive"), (dict(B=0), -1, "positive"),
    (dict(starts=None), -1, "one row"), (dict(rot=66), -1, "rotary_dim"), (dict(rot=7), -1, "rotary_dim"),
    (dict(rot=-2), -1, "rotary_dim"), (dict(pts=3), -1, "stride"), (dict(st=500), -1, "overlap"),
    (dict(st=516), -2, "aligned"), (dict(qkv=ctypes.c_void_p(24)), -2, "aligned"), (dict(q=ctypes.c_void_p(24)), -2, "aligned"),
    (dict(qw=ctypes.c_void_p(24)), -2, "aligned"), (dict(d=96), -2, "head_dim"), (dict(p=8), -2, "page size"),
    (dict(pool=c_pool(slots=0)), -1, "too small"), (dict(pool=c_pool(v_dim_stride=8)), -1, "too small"),
    (dict(pool=c_pool(k_head_stride=1028)), -2, "multiples of 8"), (dict(pool=c_pool(k=24)), -2, "aligned"),
    (dict(pool=c_pool(v=None)), -1, "null"), (dict(N=1 << 28), -2, "too many")])
def test_rope_c_refusals(change, code, text):
    a = dict(qkv=FAKE, st=512, qw=FAKE, kw=FAKE, pt=FAKE, pts=4, cols=4, lens=FAKE, starts=FAKE, inv=FAKE, rot=64, q=FAKE,
             pool=None, N=4, B=2, hq=4, hkv=2, d=64, p=16)
    a.update(change)
    pool = a["pool"] or c_pool(a["hkv"], a["p"], a["d"])
    rc = _native.lib().helm_rope_append(a["qkv"], a["st"], a["qw"], a["kw"], 1e-6, a["pt"], a["pts"], a["cols"], a["lens"],
                                        a["starts"], None, a["inv"], a["rot"], 0, 1.0, a["q"], ctypes.byref(pool), a["N"],
                                        a["B"], a["hq"], a["hkv"], a["d"], a["p"], None)
    assert rc == code and re.search(text, last_error()), (rc, last_error())


def test_copy_and_fork_c_refusals():
    lib = _native.lib()
    pool = c_pool()
    p = ctypes.byref(pool)
    assert lib.helm_copy_pages(p, None, FAKE, 1, 2, 64, 16, None) == -1
    assert lib.helm_copy_pages(p, FAKE, FAKE, 0, 2, 64, 16, None) == -1
    assert lib.helm_copy_pages(p, FAKE, FAKE, 1, 0, 64, 16, None) == -1
    assert lib.helm_copy_pages(p, FAKE, FAKE, 1, 2, 80, 16, None) == -2
    assert lib.helm_copy_pages(p, FAKE, FAKE, 1, 2, 64, 24, None) == -2
    assert lib.helm_copy_pages(None, FAKE, FAKE, 1, 2, 64, 16, None) == -1
    assert lib.helm_copy_pages(p, FAKE, FAKE, 2**31 - 1, 2, 64, 16, None) == -2 and "too many" in last_error()

    def fork(table=FAKE, ts=4, lens=FAKE, B=2, parents=FAKE, fresh=FAKE, out=FAKE, os=4, lo=FAKE, n=2, cols=4):
        return lib.helm_fork_pages(p, table, ts, lens, B, parents, fresh, out, os, lo, n, cols, 2, 64, 16, None)
    for bad in (dict(table=None), dict(lens=None), dict(parents=None), dict(fresh=None), dict(out=None), dict(lo=None),
                dict(B=0), dict(n=0), dict(cols=0), dict(ts=3), dict(os=3)):
        assert fork(**bad) == -1, bad
    assert fork(cols=1 << 27, ts=1 << 27, os=1 << 27) == -2
    q8 = ka.KvPoolQ8Struct(16, 16, 16, 16, 2 * 16 * 64, 2 * 16, 8)
    assert lib.helm_copy_pages_q8(ctypes.byref(q8), None, FAKE, 1, 2, 64, 16, None) == -1
    assert lib.helm_copy_pages_q8(ctypes.byref(q8), FAKE, FAKE, 1, 4, 64, 16, None) == -1
    assert lib.helm_fork_pages_q8(ctypes.byref(q8), FAKE, 4, FAKE, 2, FAKE, None, FAKE, 4, FAKE, 2, 4, 2, 64, 16, None) == -1


def test_cpu_tensors_are_refused():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    pool = ka.PoolView.of_pool(k, ka.alloc_v((4, 2, 16, 64), zero=True))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ka.copy_pages(pool, i, i, 16)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ka.fork_pages(pool, i.view(2, 1), i, i, i, 16)
    with pytest.raises(RuntimeError, match="on the GPU"):
        fused.rope_append(torch.zeros(2, 256).half(), pool, i.view(2, 1), i, None, 16, torch.zeros(32), 2, 2, 64)
    with pytest.raises(RuntimeError, match="page size"):
        ka.copy_pages(pool, i, i)


# ── frequencies ──────────────────────────────────────────────────────────────

@pytest.mark.parametrize("rot", [2, 32, 64, 128])
def test_scaled_frequencies(rot):
    theta, factor, ctx = 1e6, 4.0, 32768
    base = [theta ** (-2 * i / rot) for i in range(rot // 2)]
    for kind in ("linear", "theta", "bands", "yarn"):
        inv, scale = fused.rope_scaled_inv_freq(rot, theta, kind, factor, ctx)
        assert inv.dtype == torch.float32 and inv.shape == (rot // 2,)
        assert scale == (0.1 * math.log(4.0) + 1.0 if kind == "yarn" else 1.0)
        one, _ = fused.rope_scaled_inv_freq(rot, theta, kind, 1.0, ctx)
        assert torch.allclose(one, fused.rope_inv_freq(rot, theta), rtol=1e-5)
        for x, b in zip(inv.tolist(), base):             # between the base and its factor-th part
            assert b / factor * (1 - 1e-6) <= x <= b * (1 + 1e-6)
            turns = ctx * b / (2 * math.pi)
            if kind == "linear":
                assert x == pytest.approx(b / factor, rel=1e-6)
            if kind == "bands":
                share = min(max((turns - 1) / 31, 0), 1)
                assert x == pytest.approx(b * share + b / factor * (1 - share), rel=1e-6)
    if rot == 128:
        inv, _ = fused.rope_scaled_inv_freq(rot, theta, "theta", factor)
        assert inv[0] == 1.0 and inv[-1].item() == pytest.approx(base[-1] / factor, rel=1e-6)
        inv, _ = fused.rope_scaled_inv_freq(rot, theta, "yarn", factor, ctx)
        # 32 turns at dim 23.6, one at 39.6: dims to 23 stay, dims from 40 on are divided
        assert inv[23].item() == pytest.approx(base[23], rel=1e-6) and inv[24] < base[24]
        assert inv[40].item() == pytest.approx(base[40] / 4, rel=1e-6) and inv[39] > base[39] / 4 * 1.01


def test_scaled_frequencies_refusals():
    for bad in ((0, 1e4, "linear", 2.0), (7, 1e4, "linear", 2.0), (64, 1e4, "linear", 0.5), (64, 1e4, "linear", math.nan),
                (64, 1e4, "bands", 2.0), (64, 1e4, "yarn", 2.0), (64, 1e4, "other", 2.0)):
        with pytest.raises(RuntimeError, match="rope_scaled_inv_freq"):
            fused.rope_scaled_inv_freq(*bad)
    with pytest.raises(RuntimeError, match="beta"):
        fused.rope_scaled_inv_freq(64, 1e4, "bands", 2.0, 4096, beta_fast=1.0, beta_slow=1.0)


# ── rotary append ────────────────────────────────────────────────────────────

class Rope:
    def __init__(self, heads, page, seqs, rot, inter, norm=False, scale=1.0, first=0, pad=0, seed=0, start=True):
        hq, hkv, d = self.heads = heads
        g = torch.Generator().manual_seed(seed)
        self.page, self.seqs, self.rot, self.inter, self.scale, self.first = page, seqs, rot, inter, scale, first
        n = sum(k for _, k in seqs)
        self.rows = first + n + pad
        self.qkv = torch.randn(self.rows, (hq + 2 * hkv) * d, generator=g).half()
        self.inv = (1.0 / 1e4 ** (torch.arange(rot // 2, dtype=torch.float64) * 2 / max(rot, 1))).float()
        self.norms = [(1 + 0.1 * torch.randn(d, generator=g)).half() if norm else None for _ in range(2)]
        cols = max(-(-(c + k) // page) for c, k in seqs) + 1
        need = [(i, j) for i, (c, k) in enumerate(seqs) for j in range(c // page, -(-(c + k) // page)) if k]
        slots = len(need) + 2
        order = torch.randperm(slots, generator=g)
        self.table = torch.full((len(seqs), cols), -1, dtype=torch.int32)
        for (i, j), s in zip(need, order):
            self.table[i, j] = s
        self.lens = torch.tensor([c + k for c, k in seqs], dtype=torch.int32)
        self.starts = torch.tensor([first + sum(k for _, k in seqs[:i]) for i in range(len(seqs) + 1)], dtype=torch.int32)
        self.k0, self.v0 = torch.randn(slots, hkv, page, d, generator=g).half(), torch.randn(slots, hkv, d, page, generator=g).half()

    def run(self, positions=None, starts=True):
        self.d_k, self.d_v = self.k0.cuda(), self.v0.cuda()
        self.pool = ka.PoolView.of_pool(self.d_k, self.d_v.transpose(2, 3))
        hq, hkv, d = self.heads
        q = torch.full((self.rows, hq, d), 7.0, dtype=torch.float16, device="cuda")
        got = fused.rope_append(self.qkv.cuda(), self.pool, self.table.cuda(), self.lens.cuda(),
                                self.starts.cuda() if starts else None, self.page, self.inv.cuda(), hq, hkv, d, self.inter,
                                self.scale, *(w if w is None else w.cuda() for w in self.norms), eps=1e-5,
                                positions=None if positions is None else positions.cuda(), q_out=q)
        assert got is q
        return q.cpu(), self.d_k.cpu(), self.d_v.cpu()

    def check(self, got, positions=None):
        hq, hkv, d = self.heads
        q = torch.full((self.rows, hq, d), 7.0, dtype=torch.float64)
        k, v = self.k0.double(), self.v0.clone()
        tq, tk = torch.zeros(self.rows, hq, d), torch.zeros_like(k)
        at = torch.arange(self.rot)
        re_, im = (at[0::2], at[1::2]) if self.inter else (at[:self.rot // 2], at[self.rot // 2:])
        x = self.qkv.double().view(self.rows, -1, d)
        for i, (c, n) in enumerate(self.seqs):
            for t in range(n):
                r, p = int(self.starts[i]) + t, c + t
                y = x[r, :hq + hkv].clone()
                for part, w in ((slice(0, hq), self.norms[0]), (slice(hq, None), self.norms[1])):
                    if w is not None:
                        y[part] = y[part] / torch.sqrt((y[part] ** 2).mean(-1, keepdim=True) + 1e-5) * w.double()
                ang = float(p if positions is None else positions[r]) * self.inv.double()
                cs, sn = torch.cos(ang) * self.scale, torch.sin(ang) * self.scale
                a, b = y[:, re_].clone(), y[:, im].clone()
                length = y.abs()
                length[:, re_] = length[:, im] = torch.sqrt(a * a + b * b) * abs(self.scale)
                y[:, re_], y[:, im] = a * cs - b * sn, b * cs + a * sn
                tol = 2.0 ** -11 * y.abs() + 2.0 ** -19 * length + 2.0 ** -25
                q[r], tq[r] = y[:hq], tol[:hq].float()
                s, o = int(self.table[i, p // self.page]), p % self.page
                if s >= 0:
                    k[s, :, o], tk[s, :, o] = y[hq:], tol[hq:].float()
                    v[s, :, :, o] = self.qkv[r].view(-1, d)[hq + hkv:]
        assert torch.equal(got[2], v)                    # v's bits, and nothing beside them
        assert ((got[0].double() - q).abs() <= tq).all()
        assert ((got[1].double() - k).abs() <= tk).all()  # (0 where nothing was written)


HEADS = [(4, 2, 128), (7, 1, 64), (6, 6, 64), (5, 5, 128)]
LONG = [(3, 450), (0, 1), (0, 0), (100, 333), (15, 17), (16, 16), (7, 900)]     # the form for many rows


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("inter", [False, True])
def test_rope_few_rows(heads, inter):
    d = heads[2]
    for i, rot in enumerate([d, d // 2, d // 4, 2, 0, 26, d - 2]):
        r = Rope(heads, (16, 32, 64)[i % 3], [(0, 1), (99, 3), (5, 0), (15, 2), (31, 1), (200, 20)], rot, inter,
                 norm=bool(i & 1), scale=1.0 if i < 3 else 1.14, first=i % 2, pad=i % 3, seed=i)
        r.check(r.run())


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS[:3])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_many_rows(heads, inter):
    d = heads[2]
    for i, rot in enumerate([d, d // 2, 16, 0, 26]):
        r = Rope(heads, (16, 32, 64)[i % 3], LONG, rot, inter, norm=bool(i & 1), scale=1.0 if i else 1.14, first=i % 2,
                 pad=i % 3, seed=i)
        assert r.rows * (heads[0] + 2 * heads[1]) >= 9000
        r.check(r.run())


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(40, 8, 128), (72, 8, 128), (61, 9, 64), (150, 10, 64)])
def test_rope_heads_of_a_workgroup(heads):
    """Enough rows for 8 and for 16 heads a workgroup, and heads that fill no last one."""
    for inter in (False, True):
        r = Rope(heads, 16, LONG, heads[2] // 2 if inter else heads[2], inter, norm=not inter, seed=int(inter))
        r.check(r.run())


@pytest.mark.gpu
def test_rope_far_positions_and_positions_of_their_own():
    r = Rope((2, 1, 64), 64, [(1000003, 2), (130000, 1)], 64, False)
    r.check(r.run())
    p = torch.tensor([2**31 - 1, 0, 77777], dtype=torch.int32)
    r.check(r.run(positions=p), positions=p)
    r = Rope((4, 2, 128), 16, [(3, 1500)], 128, False, seed=2)
    p = torch.randint(0, 10**6, (1500,), dtype=torch.int32)
    r.check(r.run(positions=p), positions=p)


@pytest.mark.gpu
def test_rope_one_row_each_without_starts():
    for n in (1, 5, 1400):
        r = Rope((4, 2, 128), 16, [((7 * i) % 90, 1) for i in range(n)], 64, True, seed=n)
        r.check(r.run(starts=False))


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])
def test_rope_places_outside(many):
    """Slots outside the pool, positions past the table and before 0: nothing is written there,
    q is."""
    seqs = [(20, 30), (40, 1200 if many else 12)]
    r = Rope((4, 2, 128), 16, seqs, 128, False)
    q, k, v = r.run()
    cut = r.table.clone()
    cut[0, 2] = -1                                       # tokens 32 .. 47 of the first sequence
    cut[1, 3] = 10**6                                    # 48 .. 63 of the second
    r.table = cut
    r.run()
    r.table = torch.where(cut == 10**6, torch.full_like(cut, -1), cut)
    r.check((q, r.d_k.cpu(), r.d_v.cpu()))
    r.table = r.table[:, :3].contiguous()                # the table ends at token 48
    q2, k2, v2 = r.run()
    assert torch.equal(q2, q)
    r.lens[0] = 10                                       # 20 rows stand before the sequence
    r.run()
    assert torch.equal(r.d_k[r.table[0, 1].item()].cpu(), r.k0[r.table[0, 1].item()])


@pytest.mark.gpu
def test_rope_strides_streams_and_graph():
    r = Rope((4, 2, 128), 16, [(20, 3), (3, 2)], 128, True, norm=True)
    want = r.run()
    r.check(want)
    wide = torch.zeros(5, 8 * 128 + 4, dtype=torch.float16, device="cuda")[:, 4:]
    wide.copy_(r.qkv)
    k, v = r.k0.cuda(), r.v0.cuda()
    pool = ka.PoolView.of_pool(k, v.transpose(2, 3))
    args = (wide, pool, r.table.cuda(), r.lens.cuda(), r.starts.cuda(), 16, r.inv.cuda(), 4, 2, 128, True, 1.0,
            r.norms[0].cuda(), r.norms[1].cuda(), 1e-5)
    q = torch.empty(5, 4, 128, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fused.rope_append(*args, q_out=q)
    side.synchronize()
    assert torch.equal(q.cpu(), want[0]) and torch.equal(k.cpu(), want[1]) and torch.equal(v.cpu(), want[2])
    dense = wide.contiguous()
    args = (dense,) + args[1:]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fused.rope_append(*args, q_out=q)
    for _ in range(3):
        k.copy_(r.k0), v.copy_(r.v0), q.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q.cpu(), want[0]) and torch.equal(k.cpu(), want[1]) and torch.equal(v.cpu(), want[2])


@pytest.mark.gpu
def test_rope_python_refusals():
    r = Rope((4, 2, 64), 16, [(20, 3), (3, 2)], 64, False)
    pool = ka.PoolView.of_pool(r.k0.cuda(), r.v0.cuda().transpose(2, 3))
    base = dict(qkv=r.qkv.cuda(), pool=pool, page_table=r.table.cuda(), seq_lens=r.lens.cuda(), q_starts=r.starts.cuda(),
                page_size=16, inv_freq=r.inv.cuda(), num_q_heads=4, num_kv_heads=2, head_dim=64)
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    for change in (dict(qkv=base["qkv"].float()), dict(qkv=base["qkv"][:, 1:]), dict(num_kv_heads=1), dict(num_q_heads=5),
                   dict(page_size=8), dict(page_size=32), dict(page_table=base["page_table"].long()),
                   dict(seq_lens=base["seq_lens"][:1]), dict(q_starts=base["q_starts"][:2]), dict(q_starts=None),
                   dict(inv_freq=base["inv_freq"].double()), dict(inv_freq=torch.ones(33, device="cuda")),
                   dict(positions=torch.zeros(4, dtype=torch.int32, device="cuda")), dict(q_norm_w=w),
                   dict(q_norm_w=w, k_norm_w=w[:32]), dict(q_out=base["qkv"]), dict(inv_freq=r.inv)):
        with pytest.raises(RuntimeError, match="rope_append|fp16"):
            fused.rope_append(**{**base, **change})


# ── pages moved ──────────────────────────────────────────────────────────────

def pools(hkv, p, d, slots, seed=0):
    """(view, tensors, page of each tensor) of an fp16 pool and of one of codes."""
    g = torch.Generator().manual_seed(seed)

    def bits(*shape, dtype):
        n = torch.empty(shape, dtype=dtype).element_size()
        return torch.randint(-128, 128, (*shape[:-1], shape[-1] * n), generator=g, dtype=torch.int8).view(dtype).cuda()
    k, v = bits(slots, hkv, p, d, dtype=torch.float16), bits(slots, hkv, d, p, dtype=torch.float16)
    yield ka.PoolView.of_pool(k, v.transpose(2, 3)), [k, v]
    k, v = bits(slots, hkv, p, d, dtype=torch.int8), bits(slots, hkv, d, p, dtype=torch.int8)
    ks, vs = bits(slots, hkv, p, dtype=torch.float16), bits(slots, hkv, p, dtype=torch.float16)
    yield ka.Q8PoolView(k, v.transpose(2, 3), ks, vs), [k, v, ks, vs]


def raw(t):
    return t.contiguous().view(torch.int8).cpu().clone()


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,p,d", [(8, 16, 128), (1, 64, 64), (3, 32, 128), (5, 16, 64)])
@pytest.mark.parametrize("n", [1, 7, 200])
def test_copy_pages(hkv, p, d, n):
    for view, ts in pools(hkv, p, d, 2 * n + 4):
        order = torch.randperm(2 * n + 4, generator=torch.Generator().manual_seed(n)).int()
        src, dst = order[:n].clone(), order[n:2 * n].clone()
        want = [raw(t) for t in ts]
        if n > 5:
            src[0], dst[1], src[2], dst[3] = -1, 2 * n + 4, 10**9, -5          # skipped
            dst[4] = src[4]
        for i in range(n):
            if 0 <= src[i] < 2 * n + 4 and 0 <= dst[i] < 2 * n + 4:
                for w in want:
                    w[dst[i]] = w[src[i]]
        ka.copy_pages(view, src.cuda(), dst.cuda(), p)
        for w, t in zip(want, ts):
            assert torch.equal(raw(t), w)
    ka.copy_pages(view, src[:0].cuda(), dst[:0].cuda(), p)


@pytest.mark.gpu
def test_copy_pages_of_strided_pools():
    hkv, d, cap = 2, 64, 128
    ks, vs = ka.alloc_sequences(2, hkv, cap, d, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    ks.copy_(torch.randn(ks.shape, generator=g, device="cuda")), vs.copy_(torch.randn(vs.shape, generator=g, device="cuda"))
    k0, v0 = ks.clone(), vs.clone()
    view = ka.PoolView.of_sequences(ks, vs, 32)          # slot 4 b + i: page i of sequence b
    ka.copy_pages(view, torch.tensor([1, 6], dtype=torch.int32, device="cuda"),
                  torch.tensor([5, 0], dtype=torch.int32, device="cuda"), 32)
    for a, b in ((ks, k0), (vs, v0)):
        b[1, :, 32:64], b[0, :, 0:32] = b[0, :, 32:64].clone(), b[1, :, 64:96].clone()
        assert torch.equal(a, b)
    kb, vb = ka.alloc_blocked_sequences(2, hkv, cap, d, 32, device="cuda")
    kb.copy_(k0), vb.copy_(torch.randn(vb.shape, generator=g, device="cuda"))
    v1 = vb.clone()
    ka.copy_pages(ka.PoolView.of_blocked_sequences(kb, vb, 32), torch.tensor([2], dtype=torch.int32, device="cuda"),
                  torch.tensor([7], dtype=torch.int32, device="cuda"), 32)
    k0[1, :, 96:128], v1[:, 1, 3] = k0[0, :, 64:96].clone(), v1[:, 0, 2].clone()
    assert torch.equal(kb, k0) and torch.equal(vb, v1)


def forked(table, lens, parents, fresh, p):
    """Rows, lengths and copied pages by the definition."""
    rows, out, moves = [], [], []
    cols = table.shape[1]
    for q, f in zip(parents.tolist(), fresh.tolist()):
        if not 0 <= q < table.shape[0]:
            rows.append([-1] * cols)
            out.append(0)
            continue
        n = min(max(int(lens[q]), 0), cols * p)
        row, full = table[q].tolist(), n // p
        if f >= 0 and full < cols:
            if n % p:
                moves.append((row[full], f))
            row[full:] = [f] + [-1] * (cols - full - 1)
        rows.append(row)
        out.append(n)
    return torch.tensor(rows, dtype=torch.int32), torch.tensor(out, dtype=torch.int32), moves


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,p,d,n", [(8, 16, 128, 6), (1, 64, 64, 16), (3, 32, 128, 100), (2, 16, 64, 700)])
def test_fork_pages(hkv, p, d, n):
    g = torch.Generator().manual_seed(n)
    B, cols = 9, 300
    for view, ts in pools(hkv, p, d, B * 8 + n + 2):
        slots = B * 8 + n + 2
        lens = torch.tensor([0, 1, p - 1, p, p + 1, 5 * p, 7 * p + 3, cols * p + 9, -4], dtype=torch.int32)
        table = torch.randint(0, B * 8, (B, cols), generator=g).int()
        table[6, 7] = slots                              # a last page outside the pool
        parents = torch.randint(-1, B + 1, (n,), generator=g).int()
        fresh = (torch.randperm(n, generator=g) + B * 8).int()
        fresh[torch.rand(n, generator=g) < 0.3] = -1
        fresh[n // 2] = slots + 5                        # (in the table, but not copied to)
        want = [raw(t) for t in ts]
        rows, out, moves = forked(table, lens, parents, fresh, p)
        for s, f in moves:
            if s < slots and f < slots:
                for w in want:
                    w[f] = w[s]
        got = ka.fork_pages(view, table.cuda(), lens.cuda(), parents.cuda(), fresh.cuda(), p)
        assert torch.equal(got[0].cpu(), rows) and torch.equal(got[1].cpu(), out)
        for w, t in zip(want, ts):
            assert torch.equal(raw(t), w)


@pytest.mark.gpu
def test_fork_into_given_rows_and_refusals():
    view, ts = next(pools(2, 16, 64, 40))
    table = torch.arange(24, dtype=torch.int32, device="cuda").view(4, 6)
    lens = torch.tensor([20, 33, 96, 7], dtype=torch.int32, device="cuda")
    parents = torch.tensor([1, 1, 2], dtype=torch.int32, device="cuda")
    fresh = torch.tensor([-1, 30, 31], dtype=torch.int32, device="cuda")
    wide = torch.full((3, 10), 99, dtype=torch.int32, device="cuda")
    lo = torch.empty(3, dtype=torch.int32, device="cuda")
    got = ka.fork_pages(view, table, lens, parents, fresh, 16, table_out=wide[:, 2:8], lens_out=lo)
    assert got[1] is lo and lo.tolist() == [33, 33, 96]
    assert wide[:, 2:8].tolist() == [list(range(6, 12)), [6, 7, 30, -1, -1, -1], list(range(12, 18))]
    assert (wide[:, :2] == 99).all() and (wide[:, 8:] == 99).all()
    assert torch.equal(raw(ts[0][30]), raw(ts[0][8])) and not torch.equal(raw(ts[0][31]), raw(ts[0][17]))
    for bad in (dict(table_out=table[:3]), dict(lens_out=lens[:3]), dict(table_out=wide), dict(fresh=fresh[:2]),
                dict(parents=parents.long()), dict(page_table=table.long()), dict(seq_lens=lens[:2]),
                dict(page_size=8), dict(lens_out=parents), dict(parents=parents.cpu())):
        with pytest.raises(RuntimeError):
            ka.fork_pages(**{**dict(pool=view, page_table=table, seq_lens=lens, parents=parents, fresh=fresh, page_size=16), **bad})
    for bad in ((parents.long(), fresh), (parents, fresh[:2]), (parents.cpu(), fresh)):
        with pytest.raises(RuntimeError):
            ka.copy_pages(view, *bad, 16)
    assert ka.fork_pages(view, table, lens, parents[:0], fresh[:0], 16)[0].shape == (0, 6)


@pytest.mark.gpu
def test_moves_replayed_from_a_graph():
    view, ts = next(pools(2, 16, 64, 64))
    k0 = [t.clone() for t in ts]
    src = torch.arange(8, dtype=torch.int32, device="cuda")
    dst = src + 8
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8)
    lens = torch.tensor([20, 33], dtype=torch.int32, device="cuda")
    parents = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    fresh = torch.tensor([40, 41], dtype=torch.int32, device="cuda")
    to, lo = torch.empty_like(table), torch.empty_like(lens)

    def step():
        ka.copy_pages(view, src, dst, 16)
        ka.fork_pages(view, table, lens, parents, fresh, 16, table_out=to, lens_out=lo)
    step()
    torch.cuda.synchronize()
    want = [raw(t) for t in ts]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in (20, 5, 33):
        for t, z in zip(ts, k0):
            t.copy_(z)
        lens.copy_(torch.tensor([n, 33]))
        to.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert to[0, n // 16] == 40 and lo.tolist() == [n, 33]
        if n == 20:
            assert all(torch.equal(raw(t), w) for t, w in zip(ts, want))


@pytest.mark.gpu
def test_pools_past_32_bits():
    """Pages whose first element lies behind 2^32 of the pool: written, read, copied, forked."""
    hkv, p, d = 8, 64, 128
    slots = (1 << 32) // (hkv * p * d) + 40              # 65576 pages of 128 KiB each for K and V
    k = torch.empty(slots, hkv, p, d, dtype=torch.float16, device="cuda")
    v = torch.empty(slots, hkv, d, p, dtype=torch.float16, device="cuda")
    pool = ka.PoolView.of_pool(k, v.transpose(2, 3))
    hi = slots - 40
    r = Rope((8, hkv, d), p, [(0, 150), (0, 40)], d, False, seed=5)
    low = torch.where(r.table >= 0, r.table, -1)
    small = r.run()
    r.check(small)
    table = torch.where(low >= 0, low + hi, -1).cuda()
    for i in range(len(r.k0)):                           # the same bits before, behind the border
        k[hi + i].copy_(r.k0[i]), v[hi + i].copy_(r.v0[i])
    q = torch.empty(190, 8, d, dtype=torch.float16, device="cuda")
    lens, starts = r.lens.cuda(), r.starts.cuda()
    fused.rope_append(r.qkv.cuda(), pool, table, lens, starts, p, r.inv.cuda(), 8, hkv, d, q_out=q)
    n = len(r.k0)
    assert torch.equal(q.cpu(), small[0]) and torch.equal(k[hi:hi + n].cpu(), small[1]) and torch.equal(v[hi:hi + n].cpu(), small[2])
    near = ka.PoolView.of_pool(small[1].cuda(), small[2].cuda().transpose(2, 3))
    for kw in ({}, {"window": 30, "sinks": 2}):
        far = ka.chunk_attention(q, pool, table, lens, starts, p, **kw)
        assert torch.equal(far, ka.chunk_attention(q, near, low.int().cuda(), lens, starts, p, **kw))
    last = q[torch.tensor([149, 189])].contiguous()
    assert torch.equal(ka.window_decode_attention(last, pool, table, lens, p, 70),
                       ka.window_decode_attention(last, near, low.int().cuda(), lens, p, 70))
    one = torch.tensor([hi + 20], dtype=torch.int32, device="cuda")
    ka.copy_pages(pool, table[0, :1].contiguous(), one, p)
    assert torch.equal(k[hi + 20], k[table[0, 0]]) and torch.equal(v[hi + 20], v[table[0, 0]])
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows, _ = ka.fork_pages(pool, table, lens, zero, one + 1, p)
    assert rows[0, 2] == hi + 21 and torch.equal(k[hi + 21], k[table[0, 2]]) and torch.equal(v[hi + 21], v[table[0, 2]])
