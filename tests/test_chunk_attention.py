"""Attention of ragged batches over a paged cache, windows and sinks: refusals on the CPU; on
the GPU against the definition in fp64.

Every place of the pool that no row sees holds NaN, and every table entry that none needs is
outside the pool: the output is finite only if none of them counts.

Tolerances.  Few rows: probabilities enter the product to 2^-22, so an output is off by its own
rounding, 2^-11 |o|, and by the exponent of scores up to 64 (64 * 2^-23 and a few ulps): 2^-16 of the
largest |v|.  Many rows: a probability is rounded to fp16, off by 2^-11 of itself, in numerator
and denominator alike, so the output moves by at most 2^-11 of sum p |v - o| <= 2 max |v|; below
2^-14 of the largest one it is off by 2^-25 at most, with n keys by n 2^-24 max |v| in all.  With
equal scores (k = 0) all probabilities are 1 and sums of small whole numbers exact: the output is off
by its rounding and that of one division, which tells every key that is left out or too many.
"""
import ctypes
import math

import pytest
import torch

from helm_amd import _native
from helm_amd.kernels import attention as ka


# ── refusals ─────────────────────────────────────────────────────────────────

def cpu_pool(hkv=2, p=16, d=64, slots=4):
    k = torch.zeros(slots, hkv, p, d, dtype=torch.float16)
    return ka.PoolView.of_pool(k, ka.alloc_v((slots, hkv, p, d), zero=True))


def test_cpu_tensors_are_refused():
    q, pt, n = torch.zeros(2, 4, 64).half(), torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    qs = torch.tensor([0, 1, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ka.chunk_attention(q, cpu_pool(), pt, n, qs, 16)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ka.window_decode_attention(q, cpu_pool(), pt, n, 16, 8)
    with pytest.raises(RuntimeError, match="q_starts"):
        ka.chunk_attention(q, cpu_pool(), pt, n, None, 16)


FAKE = ctypes.c_void_p(16)             # never dereferenced: the checks fail first


def c_call(q=FAKE, st=256, sh=64, pool=None, pt=FAKE, pts=8, lens=FAKE, starts=FAKE, N=4, B=2, hq=4, hkv=2, d=64, p=16,
           pages=8, new=4, window=0, sinks=0, scale=0.1, out=FAKE, ot=256, oh=64, ws=FAKE, nws=1 << 40):
    s = pool or ka.KvPoolStruct(16, 16, hkv * p * d, p * d, hkv * d * p, d * p, p, 8)
    rc = _native.lib().helm_chunk_attn(q, st, sh, ctypes.byref(s), pt, pts, lens, starts, N, B, hq, hkv, d, p, pages, new,
                                       window, sinks, scale, out, ot, oh, ws, nws, None)
    return rc, _native.lib().helm_last_error().decode()


@pytest.mark.parametrize("change, code, text", [
    (dict(q=None), -1, "null"), (dict(pt=None), -1, "null"), (dict(lens=None), -1, "null"), (dict(out=None), -1, "null"),
    (dict(N=0), -1, "positive"), (dict(B=0), -1, "positive"), (dict(pages=0), -1, "positive"), (dict(new=0), -1, "positive"),
    (dict(window=-1), -1, "negative"), (dict(sinks=-1), -1, "negative"),
    (dict(starts=None), -1, "one row per sequence"), (dict(hq=5, sh=64), -1, "multiple"),
    (dict(scale=0.0), -1, "scale"), (dict(scale=-1.0), -1, "scale"), (dict(scale=math.nan), -1, "scale"),
    (dict(scale=math.inf), -1, "scale"), (dict(d=96), -2, "head_dim"), (dict(p=8), -2, "page size"),
    (dict(pts=7), -1, "stride"), (dict(sh=60), -2, "multiples of 8"), (dict(oh=66), -2, "multiples"),
    (dict(q=ctypes.c_void_p(24)), -2, "aligned"), (dict(out=ctypes.c_void_p(20)), -2, "aligned"),
    (dict(N=1 << 30), -2, "too many rows"), (dict(pages=1 << 27, pts=1 << 27), -2, "2\\^30 keys"),
    (dict(ws=None, nws=0), -1, "workspace"), (dict(ws=ctypes.c_void_p(24)), -1, "workspace"),
    (dict(nws=8), -1, "workspace"),
    (dict(pool=ka.KvPoolStruct(16, 16, 2048, 1000, 2048, 1024, 16, 8)), -1, "too small"),
    (dict(pool=ka.KvPoolStruct(16, 16, 2048, 1024, 2048, 1024, 8, 8)), -1, "too small"),
    (dict(pool=ka.KvPoolStruct(16, 16, 2048, 1028, 2048, 1024, 16, 8)), -2, "multiples of 8"),
    (dict(pool=ka.KvPoolStruct(16, 16, 2048, 1024, 1 << 40, 1 << 38, 1 << 24, 8)), -2, "32-bit"),
    (dict(pool=ka.KvPoolStruct(24, 16, 2048, 1024, 2048, 1024, 16, 8)), -2, "aligned"),
    (dict(pool=ka.KvPoolStruct(16, 16, 2048, 1024, 2048, 1024, 16, 0)), -1, "too small"),
])
def test_c_refusals(change, code, text):
    import re
    args = dict(pages=64, pts=64)
    args.update(change)
    rc, msg = c_call(**args)
    assert rc == code and re.search(text, msg), (rc, msg)


@pytest.mark.parametrize("N,B,hq,hkv,pages,new,window,sinks", [
    (1, 1, 8, 8, 1, 1, 0, 0), (4, 4, 32, 8, 1024, 1, 4096, 4), (20, 4, 32, 8, 200, 5, 0, 0), (4096, 1, 40, 8, 1024, 4096, 0, 0),
    (700, 25, 40, 8, 512, 700, 0, 0), (300, 300, 16, 1, 9, 1, 0, 0), (64, 2, 64, 1, 100, 60, 0, 0), (9000, 3, 32, 32, 99, 9000, 100, 0)])
def test_workspace_is_bounded(N, B, hq, hkv, pages, new, window, sinks):
    """Never more than 4/3 * 512 pieces of 128 rows, whatever the lengths (and none where no
    sequence can have two pieces)."""
    f = _native.lib().helm_chunk_attn_workspace_bytes
    need = f(N, B, hq, hkv, 128, 16, pages, new, window, sinks)
    assert 0 <= need <= 2 * (4 * max(512, hkv) + 2 * hkv) // 3 * 128 * 130 * 4
    assert need % 8 == 0
    if pages * 16 <= 128:
        assert need == 0
    assert f(0, B, hq, hkv, 128, 16, pages, new, window, sinks) == 0


# ── the definition ───────────────────────────────────────────────────────────

class Batch:
    """seqs: (cached, new) of each sequence."""

    def __init__(self, heads, page, seqs, window=0, sinks=0, pad=0, seed=0, flat=False, first=0, holes=(), spare=3,
                 layout="pool"):
        hq, hkv, d = self.heads = heads
        self.page, self.seqs, self.window, self.sinks, self.flat = page, seqs, window, sinks, flat
        g = torch.Generator().manual_seed(seed)
        n = sum(k for _, k in seqs)
        self.rows, self.first = n + pad + first, first
        cols = max(1, max(-(-(c + k) // page) for c, k in seqs)) + spare
        self.q = torch.randn(self.rows, hq, d, generator=g).half()
        lens = [c + k for c, k in seqs]
        self.starts = torch.tensor([first] + [first + sum(k for _, k in seqs[:i + 1]) for i in range(len(seqs))])
        # K, V of each sequence and the keys that some row sees
        self.k, self.v, self.live = [], [], []
        need = []
        for i, (c, k) in enumerate(seqs):
            L = c + k
            kk = torch.randn(hkv, L, d, generator=g).half()
            vv = torch.randn(hkv, L, d, generator=g).half()
            if flat:
                kk.zero_()
                vv = torch.where(vv > 0, 1.0, -1.0).half()
            key = torch.arange(L)
            live = (key >= c - window + 1) | (key < sinks) if window else torch.ones(L, dtype=torch.bool)
            if k == 0:
                live &= False
            for h in holes:                              # pages without a slot
                if h[0] == i:
                    live &= key // page != h[1]
            self.k.append(kk)
            self.v.append(vv)
            self.live.append(live)
            need.append([j for j in range(-(-L // page)) if live[j * page:(j + 1) * page].any()])
        total = sum(len(x) for x in need)
        slots = total + 3
        order = torch.randperm(slots, generator=g)[:total].tolist()
        table = torch.full((len(seqs), cols), -1)
        table[:, 1::2] = slots + 7                       # entries outside the pool, either way
        kp = torch.full((slots, hkv, page, d), math.nan).half()
        vp = torch.full((slots, hkv, d, page), math.nan).half()
        at = 0
        for i, js in enumerate(need):
            for j in js:
                s = order[at]
                at += 1
                table[i, j] = s
                for t in range(page):
                    key = j * page + t
                    if key < lens[i] and self.live[i][key]:
                        kp[s, :, t] = self.k[i][:, key]
                        vp[s, :, :, t] = self.v[i][:, key]
        self.table, self.lens = table.int(), torch.tensor(lens).int()
        self.kp, self.vp, self.slots = kp, vp, slots

    def cuda(self):
        self.d_q, self.d_table, self.d_lens = self.q.cuda(), self.table.cuda(), self.lens.cuda()
        self.d_starts = self.starts.int().cuda()
        self.pool = ka.PoolView.of_pool(self.kp.cuda(), self.vp.cuda().transpose(2, 3))
        return self

    def exact(self, scale=None, coverage=None):
        hq, hkv, d = self.heads
        out = torch.full((self.rows, hq, d), 7.0, dtype=torch.float64)
        for i, (c, k) in enumerate(self.seqs):
            key = torch.arange(c + k)
            for t in range(k):
                p = c + t
                seen = self.live[i] & (key <= p)
                if self.window:
                    seen &= (key > p - self.window) | (key < self.sinks)
                if coverage is not None:
                    seen &= key < coverage
                r = int(self.starts[i]) + t
                if not seen.any():
                    out[r] = 0.0
                    continue
                q = self.q[r].double().view(hkv, hq // hkv, d)
                s = torch.einsum("hgd,hkd->hgk", q, self.k[i][:, seen].double()) * (d ** -0.5 if scale is None else scale)
                out[r] = torch.einsum("hgk,hkd->hgd", torch.softmax(s, -1), self.v[i][:, seen].double()).reshape(hq, d)
        return out

    def run(self, **kw):
        out = torch.full((self.rows, self.heads[0], self.heads[2]), 7.0, dtype=torch.float16, device="cuda")
        r = ka.chunk_attention(self.d_q, self.pool, self.d_table, self.d_lens, self.d_starts, self.page, self.window,
                               self.sinks, out=out, **kw)
        assert r is out
        return out.cpu()

    def check(self, got, want, few=False):
        n = max(c + k for c, k in self.seqs)
        top = max(float(v.abs().max()) for v in self.v if v.numel()) if any(v.numel() for v in self.v) else 0.0
        if self.flat:
            tol = 2.0 ** -11 * want.abs() + 2.0 ** -22
        elif few:
            tol = 2.0 ** -11 * want.abs() + 2.0 ** -16 * top
        else:
            tol = 2.0 ** -11 * want.abs() + top * (2.0 ** -10 + 2.0 ** -16 + n * 2.0 ** -24)
        err = (got.double() - want).abs()
        assert torch.isfinite(got).all()
        worst = (err - tol).max().item()
        assert worst <= 0, f"off by up to {err.max().item():.2e}, {worst:.2e} too much at {(err - tol).argmax().item()}"


HEADS = [(8, 2, 128), (10, 2, 64), (5, 1, 128), (6, 6, 64), (16, 1, 64), (40, 1, 128), (34, 2, 64)]
FEW = [   # one row tile per sequence: decode, drafts
    [(0, 1)], [(1, 1)], [(15, 1)], [(16, 1)], [(31, 1), (32, 1), (63, 1)], [(500, 1), (0, 1), (77, 1), (130, 1)],
    [(200, 3), (0, 2), (17, 1)], [(0, 0), (40, 2), (9, 0), (700, 3)],
]
MANY = [
    [(0, 17)], [(0, 64), (5, 33)], [(100, 129)], [(0, 200), (60, 1), (300, 40)], [(63, 65), (64, 64), (65, 1)],
    [(0, 1), (0, 300), (0, 0), (31, 2)],
]
WINDOWS = [(0, 0), (1, 0), (1, 1), (16, 4), (33, 0), (64, 17), (100, 40), (5, 200), (1000, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("seqs", range(len(FEW)))
@pytest.mark.parametrize("heads", HEADS)
def test_few_rows(heads, seqs, flat):
    for i, (window, sinks) in enumerate(WINDOWS[::2] if flat else WINDOWS[1::3]):
        b = Batch(heads, (16, 32, 64)[(i + seqs) % 3], FEW[seqs], window, sinks, pad=2, seed=i, flat=flat).cuda()
        b.check(b.run(max_new=3), b.exact())


@pytest.mark.gpu
@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("seqs", range(len(MANY)))
@pytest.mark.parametrize("heads", HEADS)
def test_many_rows(heads, seqs, flat):
    for i, (window, sinks) in enumerate(WINDOWS[::3] if flat else WINDOWS[1::4]):
        b = Batch(heads, (16, 32, 64)[(i + seqs) % 3], MANY[seqs], window, sinks, pad=i, seed=i, flat=flat, first=i % 2).cuda()
        b.check(b.run(), b.exact())


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("heads", HEADS[:3])
def test_decode(heads, window, sinks):
    seqs = [(c, 1) for c in (0, 1, 15, 16, 17, 63, 64, 100, 333, 900)]
    for flat in (True, False):
        b = Batch(heads, 16, seqs, window, sinks, flat=flat).cuda()
        got = ka.window_decode_attention(b.d_q, b.pool, b.d_table, b.d_lens, 16, window, sinks)
        b.check(got.cpu(), b.exact(), few=heads[0] // heads[1] <= 32)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 3)])
def test_pieces(window, sinks):
    """Few sequences over many keys: keys cut into pieces and joined again."""
    for heads, seqs in (((4, 2, 128), [(5000, 1)]), ((8, 2, 64), [(3001, 7), (40, 1)]), ((8, 1, 128), [(4000, 60)]),
                        ((6, 2, 128), [(2500, 150), (1, 1), (3000, 2)])):
        for flat in (True, False):
            b = Batch(heads, 16, seqs, window, sinks, flat=flat).cuda()
            b.check(b.run(), b.exact())


@pytest.mark.gpu
def test_pages_without_a_slot():
    b = Batch((8, 2, 128), 16, [(300, 40), (90, 2), (16, 0)], holes=[(0, 0), (0, 7), (0, 20), (1, 5), (1, 2)], flat=True).cuda()
    b.check(b.run(), b.exact())
    b = Batch((8, 2, 128), 32, [(20, 30), (0, 1)], holes=[(0, 0), (0, 1), (1, 0)], flat=True).cuda()   # nothing left
    want = b.exact()
    assert (want[30] == 0).all() and (want[:30] == 0).any()
    b.check(b.run(), want)


@pytest.mark.gpu
def test_lengths_past_the_table_and_below_the_rows():
    b = Batch((8, 2, 64), 16, [(100, 20), (100, 1)], flat=True, spare=0).cuda()
    cols = 5                                             # the table ends at token 80
    table = b.d_table[:, :cols].contiguous()
    out = torch.full_like(b.d_q, 7.0)
    ka.chunk_attention(b.d_q, b.pool, table, b.d_lens, b.d_starts, 16, out=out)
    b.check(out.cpu(), b.exact(coverage=80))
    # 3 tokens in all, 5 rows: the first two stand before the sequence and see nothing
    b = Batch((4, 2, 64), 16, [(0, 3)], flat=True)
    b.rows, b.q = 5, torch.cat([b.q, b.q[:2]])
    b.starts[1] = 5
    b.cuda()
    got = b.run()
    assert (got[:2] == 0).all()
    b.starts = b.starts.clone()
    b.starts[0] = 2
    want = b.exact()
    want[:2] = 0
    b.check(got, want)


@pytest.mark.gpu
def test_rows_past_max_new_stay():
    b = Batch((8, 2, 128), 16, [(50, 9), (20, 1)], flat=True).cuda()
    for most in (1, 3, 4, 8):
        want = b.exact()
        want[most:9] = 7.0
        b.check(b.run(max_new=most), want)


@pytest.mark.gpu
def test_infinite_and_nan_keys_behind_the_mask():
    """A key that a row does not see may hold anything, also where another row sees it."""
    b = Batch((4, 2, 128), 16, [(40, 30)], window=20, sinks=2).cuda()
    want = b.exact()
    late = b.pool.k.clone()
    key = 40 + 29                                        # seen by the last row only
    late[b.table[0, key // 16], :, key % 16] = math.nan
    pool = ka.PoolView.of_pool(late, b.pool.v)
    out = torch.empty_like(b.d_q)
    ka.chunk_attention(b.d_q, pool, b.d_table, b.d_lens, b.d_starts, 16, 20, 2, out=out)
    assert torch.isnan(out[29]).all()
    got = out.cpu()
    got[29] = want[29].half()
    b.check(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("few", [True, False])
def test_strides_and_scale(few):
    b = Batch((8, 2, 128), 16, [(70, 2), (20, 3)] if few else [(70, 60), (20, 30)], seed=3).cuda()
    want = b.exact(scale=0.05)
    wide = torch.full((b.rows, 12, 136), math.nan, dtype=torch.float16, device="cuda")
    q = wide[:, 2:10, 4:132]                             # rows that start 8 bytes off an aligned place
    q.copy_(b.d_q)
    out = torch.full((b.rows, 9, 132), 7.0, dtype=torch.float16, device="cuda")[:, 1:, :128]
    kw = {"max_new": 4} if few else {}
    ka.chunk_attention(q, b.pool, b.d_table, b.d_lens, b.d_starts, 16, scale=0.05, out=out, **kw)
    b.check(out.cpu(), want)
    # heads-first q, a table that is a slice of a wider one
    hq = b.d_q.transpose(0, 1).contiguous().transpose(0, 1)
    table = torch.full((2, 40), -5, dtype=torch.int32, device="cuda")
    table[:, 3:3 + b.table.shape[1]] = b.d_table
    got = ka.chunk_attention(hq, b.pool, table[:, 3:3 + b.table.shape[1]], b.d_lens, b.d_starts, 16, scale=0.05, **kw)
    b.check(got.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["sequences", "blocked"])
def test_contiguous_sequences(layout):
    hq, hkv, d, cap = 8, 2, 128, 320
    g = torch.Generator().manual_seed(1)
    k, v = torch.zeros(2, hkv, 300, d), torch.randn(2, hkv, 300, d, generator=g).sign().half()
    if layout == "sequences":
        ks, vs = ka.alloc_sequences(2, hkv, cap, d, device="cuda")
        ks[:, :, :300], vs[:, :, :300] = k.half().cuda(), v.cuda()
        view = ka.PoolView.of_sequences(ks, vs, 16)
    else:
        ks, vb = ka.alloc_blocked_sequences(2, hkv, cap, d, 16, device="cuda")
        ks[:, :, :300] = k.half().cuda()
        full = torch.zeros(2, hkv, cap, d)
        full[:, :, :300] = v
        vb.copy_(full.view(2, hkv, cap // 16, 16, d).permute(1, 0, 2, 4, 3).half())
        view = ka.PoolView.of_blocked_sequences(ks, vb, 16)
    table = torch.arange(2 * cap // 16, dtype=torch.int32, device="cuda").view(2, -1)
    q = torch.randn(102, hq, d, generator=g).half().cuda()
    got = ka.chunk_attention(q, view, table, torch.tensor([300, 211], dtype=torch.int32, device="cuda"),
                             torch.tensor([0, 100, 102], dtype=torch.int32, device="cuda"), 16, window=50)
    for r, b, p in [(0, 0, 200), (57, 0, 257), (99, 0, 299), (100, 1, 209), (101, 1, 210)]:
        want = v[b, :, p - 49:p + 1].double().mean(1).repeat_interleave(hq // hkv, 0)
        assert ((got[r].cpu().double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -22).all()


@pytest.mark.gpu
def test_many_sequences():
    """More sequences than a workgroup has threads."""
    seqs = [((7 * i) % 40, (1, 0, 2, 1, 5)[i % 5]) for i in range(700)]
    seqs[300] = (10, 90)
    for kw in ({}, {"max_new": 90}):
        b = Batch((4, 2, 64), 16, seqs, flat=True).cuda()
        b.check(b.run(**kw), b.exact())
    b = Batch((4, 2, 64), 16, [(c, 1) for c, _ in seqs], flat=True).cuda()
    b.check(ka.window_decode_attention(b.d_q, b.pool, b.d_table, b.d_lens, 16, 0).cpu(), b.exact())


@pytest.mark.gpu
def test_runs_alike_and_on_other_streams():
    b = Batch((8, 2, 128), 16, [(2000, 100), (900, 1), (0, 40)]).cuda()
    first = b.run()
    for _ in range(3):
        assert torch.equal(b.run(), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ws = [ka.AttnWorkspace(torch.device("cuda", 0)) for _ in range(2)]
    outs = [torch.empty_like(b.d_q) for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(4):                                   # two calls at once
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            ka.chunk_attention(b.d_q, b.pool, b.d_table, b.d_lens, b.d_starts, 16, workspace=ws[i % 2], out=outs[i % 2])
    torch.cuda.synchronize()
    assert torch.equal(outs[0].cpu(), first) and torch.equal(outs[1].cpu(), first)


@pytest.mark.gpu
def test_captured_call_takes_other_lengths():
    """One graph, replayed with other lengths, tables and starts of the same tensors."""
    shapes = [[(700, 60), (30, 1), (5, 20)], [(10, 1), (1, 79), (0, 1)], [(0, 0), (0, 0), (3000, 2)], [(40, 27), (40, 27), (40, 27)]]
    cols, slots, rows = 200, 240, 81
    heads = (8, 2, 128)
    q = torch.empty(rows, 8, 128, dtype=torch.float16, device="cuda")
    table = torch.full((3, cols), -1, dtype=torch.int32, device="cuda")
    lens, starts = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    k = torch.zeros(slots, 2, 16, 128, dtype=torch.float16, device="cuda")
    v = ka.alloc_v((slots, 2, 16, 128), device="cuda", zero=True)
    pool, ws, out = ka.PoolView.of_pool(k, v), ka.AttnWorkspace(q.device), torch.empty_like(q)

    def call():
        ka.chunk_attention(q, pool, table, lens, starts, 16, workspace=ws, out=out)

    def load(i):
        b = Batch(heads, 16, shapes[i], seed=i)
        table.fill_(-1)
        table[:, :b.table.shape[1]] = torch.where(b.table < b.slots, b.table, -1).cuda()
        lens.copy_(b.lens), starts.copy_(b.starts)
        k[:b.slots], v.transpose(2, 3)[:b.slots] = b.kp.cuda(), b.vp.cuda()
        q.zero_()
        q[:b.rows] = b.q.cuda()
        out.fill_(7.0)
        return b
    load(0)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in (1, 0, 3, 2, 1):
        b = load(i)
        graph.replay()
        got = out.clone()
        out.fill_(7.0)
        call()
        torch.cuda.synchronize()
        assert torch.equal(got, out)
        b.check(got[:b.rows].cpu(), b.exact())
        assert (got[b.rows:] == 7.0).all()


@pytest.mark.gpu
def test_python_refusals():
    b = Batch((4, 2, 64), 16, [(5, 2), (0, 1)]).cuda()
    args = dict(q=b.d_q, pool=b.pool, page_table=b.d_table, seq_lens=b.d_lens, q_starts=b.d_starts, page_size=16)
    bad = [dict(q=b.d_q.float()), dict(q=b.d_q[:, :3]), dict(q=b.d_q[..., :32]), dict(page_size=8), dict(page_size=32),
           dict(page_table=b.d_table.long()), dict(page_table=b.d_table.t()), dict(page_table=b.d_table[:, :0]),
           dict(seq_lens=b.d_lens.long()),
           dict(seq_lens=b.d_lens[:1]), dict(q_starts=b.d_starts[:2]), dict(q_starts=b.d_starts.long()), dict(window=-1),
           dict(sinks=-1), dict(max_new=0), dict(scale=0.0), dict(scale=math.inf), dict(out=b.d_q.float()),
           dict(out=b.d_q[:2]), dict(q_starts=b.d_starts.cpu()), dict(workspace=ka.AttnWorkspace(torch.device("cpu")))]
    for change in bad:
        with pytest.raises(RuntimeError):
            if "workspace" in change:
                big = Batch((4, 2, 64), 16, [(600, 2)]).cuda()
                ka.chunk_attention(big.d_q, big.pool, big.d_table, big.d_lens, big.d_starts, 16, **change)
            else:
                ka.chunk_attention(**{**args, **change})
    with pytest.raises(RuntimeError):
        ka.window_decode_attention(b.d_q, b.pool, b.d_table, b.d_lens, 16, 4)      # three rows, two sequences
    empty = ka.chunk_attention(b.d_q[:0], b.pool, b.d_table, b.d_lens, b.d_starts, 16)
    assert empty.shape == (0, 4, 64)


def flat_pool(L, hkv, d, page, seed):
    """Keys of zeros and values of +-1 of one sequence of L tokens in shuffled pages, its table, and the
    sums of values up to each token [L + 1, hkv, d]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = -(-L // page)
    v = torch.randint(0, 2, (n * page, hkv, d), generator=g, device="cuda", dtype=torch.int8) * 2 - 1
    order = torch.randperm(n, generator=g, device="cuda")
    vp = torch.empty(n, hkv, d, page, dtype=torch.float16, device="cuda")
    vp[order] = v.view(n, page, hkv, d).permute(0, 2, 3, 1).half()
    kp = torch.zeros(n, hkv, page, d, dtype=torch.float16, device="cuda")
    sums = torch.cat([torch.zeros(1, hkv, d, dtype=torch.int32, device="cuda"), v.int().cumsum(0, dtype=torch.int32)])
    return ka.PoolView.of_pool(kp, vp.transpose(2, 3)), order.int()[None].contiguous(), sums


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 1, 64, 16), (8, 2, 128, 64)])
@pytest.mark.parametrize("window", [0, 100, 20000])
def test_long_prompts(hq, hkv, d, page, window):
    """Tens of thousands of rows after tens of thousands of keys, every row against exact sums."""
    n, L = 30000, 41003
    pool, table, sums = flat_pool(L, hkv, d, page, 1)
    q = torch.randn(n, hq, d, dtype=torch.float16, device="cuda")
    out = ka.chunk_attention(q, pool, table, torch.tensor([L], dtype=torch.int32, device="cuda"),
                             torch.tensor([0, n], dtype=torch.int32, device="cuda"), page, window, 3 if window else 0)
    p = torch.arange(L - n, L, device="cuda")
    lo = (p - window + 1).clamp(min=0) if window else torch.zeros_like(p)
    total, count = sums[p + 1] - sums[lo], p + 1 - lo
    if window:
        more = lo.clamp(max=3)                           # sinks before the window
        total, count = total + sums[more], count + more
    want = (total.double() / count.double()[:, None, None]).repeat_interleave(hq // hkv, 1)
    assert ((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -22).all()


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 1000, 200000])
def test_decode_after_hundreds_of_thousands_of_tokens(window):
    L = 300017
    pool, table, sums = flat_pool(L, 2, 64, 16, 2)
    q = torch.randn(1, 8, 64, dtype=torch.float16, device="cuda")
    out = ka.window_decode_attention(q, pool, table, torch.tensor([L], dtype=torch.int32, device="cuda"), 16, window, 7)
    lo = L - window if window else 0
    more = 7 if window else 0
    want = ((sums[L] - sums[lo] + sums[more]).double() / (L - lo + more)).repeat_interleave(4, 0)
    assert ((out[0].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -22).all()
