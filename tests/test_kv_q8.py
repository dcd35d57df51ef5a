"""KV pages of 8-bit codes: refusals on the CPU; the writes, the way back and the decode
attention on the GPU against fp64 and against torch's own quantisation.

Codes.  x and s are fp16 numbers with 11-bit mantissas, so x / s lies exactly on or at
least 2^-12 away from a border n + 1/2 of the codes, and an fp32 quotient below 128 is off by
at most 2^-17: codes and scales of fp16 values are equal to torch's, bit for bit.  Keys are
quantised from fp32 after norm and RoPE: at most half a step plus what the fp32 chain is off
(about ten roundings of 2^-24 of the row's largest, 2^-20 with room).

Attention.  The output's rounding is off by 2^-11 |o|; scores up to 64 in the exponent are off
by 64 * 2^-23 plus a few ulps, so a probability by 2^-17 relative and a weighted mean of values
by 2^-16 of the largest |v|.
"""
import ctypes
import math

import pytest
import torch

from helm_amd import _native
from helm_amd.kernels import attention as ka
from helm_amd.kernels import fused

EPS = 1e-6


def random_pool(slots, hkv, p, d, seed, junk=False):
    g = torch.Generator().manual_seed(seed)
    pool = ka.alloc_q8_pool(slots, hkv, p, d, "cuda")
    pool.k.copy_(torch.randint(-127, 128, pool.k.shape, generator=g, dtype=torch.int8))
    pool.v.copy_(torch.randint(-127, 128, pool.v.shape, generator=g, dtype=torch.int8))
    for s in (pool.k_scale, pool.v_scale):
        s.copy_(((0.3 + torch.rand(s.shape, generator=g)) * 0.02).half())
        if junk:
            s.fill_(float("nan"))
    return pool


def held(pool):
    """fp64 K and V [slots, Hkv, P, D] on the CPU."""
    return ((pool.k.cpu().double() * pool.k_scale.cpu().double()[..., None]),
            (pool.v.cpu().double() * pool.v_scale.cpu().double()[..., None]))


def quantised(x):
    """Codes and scales of fp16 rows, by torch."""
    s = (x.float().abs().amax(-1) / 127.0).half()
    ok = (s > 0)[..., None]
    c = torch.where(ok, torch.round(x.float() / torch.where(ok, s[..., None].float(), 1.0)), 0.0).clamp(-127, 127)
    return c.to(torch.int8), s


# ── refusals ─────────────────────────────────────────────────────────────────

def test_pool_view_refusals():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    v = ka.alloc_v((4, 2, 16, 64), dtype=torch.int8, zero=True)
    s = torch.zeros(4, 2, 16).half()
    ka.Q8PoolView(k, v, s, s)
    for bad in ((k.half(), v, s, s), (k, k, s, s), (k, v, s.float(), s), (k, v, s[:, :1], s), (k[:, :, :8], v[:, :, :8], s[:, :, :8], s[:, :, :8]),
                (k.transpose(1, 2).contiguous().transpose(1, 2), v, s, s), (k[:0], v[:0], s[:0], s[:0]),
                (k, v, s, s.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(RuntimeError, match="Q8PoolView"):
            ka.Q8PoolView(*bad)
    pool = ka.Q8PoolView(k, v, s, s)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ka.paged_decode_attention_q8(torch.zeros(1, 2, 64).half(), pool, i[None], i)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ka.kv_append_q8(torch.zeros(1, 2, 1, 64).half(), torch.zeros(1, 2, 1, 64).half(), pool, i, i)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ka.dequantize_pages(pool, i)
    with pytest.raises(RuntimeError, match="on the GPU"):
        fused.qk_norm_rope_append_q8(torch.zeros(1, 384).half(), None, None, EPS, i, torch.zeros(32), None, pool, i, i, 2, 2, 64)


def test_c_entry_refusals():
    lib = _native.lib()
    fake = ctypes.c_void_p(16)
    P, D, H = 16, 128, 8

    def pool(k=16, ss=H * P * D, sss=H * P, n=4):
        return ctypes.byref(ka.KvPoolQ8Struct(k, 16, 16, 16, ss, sss, n))

    def attn(pool=pool(), d=D, p=P, hq=32, hkv=H, pages=4, splits=0, ws=None, nbytes=0, pts=4, qs=128, b=1, out=fake):
        return lib.helm_paged_decode_attn_q8(fake, qs, qs, pool, fake, pts, fake, out, b, hq, hkv, d, p, pages, 0.1,
                                             splits, ws, nbytes, None)
    assert attn(pool=None) == -1 and attn(pool=pool(k=0)) == -1 and attn(pool=pool(n=0)) == -1 and attn(out=None) == -1
    assert attn(pool=pool(k=8)) == -2 and attn(pool=pool(ss=H * P * D - 16)) == -1
    assert attn(pool=pool(ss=H * P * D + 8)) == -2 and attn(pool=pool(sss=H * P + 4)) == -2
    assert attn(d=96) == -2 and attn(p=8) == -2 and attn(hq=31) == -1 and attn(hq=8 * 17) == -2
    assert attn(splits=-1) == -1 and attn(pts=3) == -1 and attn(qs=4) == -2 and attn(b=0) == -1
    assert attn(pages=64, pts=64) == -1 and b"workspace" in lib.helm_last_error()
    need = lib.helm_paged_attn_q8_workspace_bytes(1, 32, H, D, P, 64, 0)
    assert need > 0 and attn(pages=64, pts=64, ws=ctypes.c_void_p(8), nbytes=need) == -1
    assert attn(pages=64, pts=64, ws=fake, nbytes=need - 1) == -1
    assert lib.helm_kv_append_q8(fake, None, pool(), fake, fake, 1, H, 1, D, P, None) == -1
    assert lib.helm_kv_append_q8(fake, fake, pool(), fake, fake, 1, H, 17, D, P, None) == -1
    assert lib.helm_dequantize_pages(pool(), None, 1, fake, fake, H, D, P, None) == -1
    assert lib.helm_dequantize_pages(pool(), fake, 1, ctypes.c_void_p(24), fake, H, D, P, None) == -2

    def app(stride=(32 + 16) * D, qn=None, kn=None, inv=fake):
        return lib.helm_qk_norm_rope_append_q8(fake, stride, qn, kn, EPS, fake, inv, fake, pool(), fake, fake, 1, 32, H,
                                               D, P, None)
    assert app(inv=None) == -1 and app(qn=fake) == -1 and app(stride=D) == -1 and app(stride=48 * D + 4) == -2


@pytest.mark.parametrize("pages,p", [(1, 16), (44, 32), (1024, 16), (100000, 16), (60000, 64)])
def test_splits_fit_their_staged_pages(pages, p):
    for b in (1, 4, 16, 100):
        for want in (0, 1, 7):
            n = ka.q8_workspace_bytes(b, 16, 8, 64, p, pages, want) // (b * 16 * 66 * 4) or 1
            assert n >= want and -(-(-(-pages * p // 64)) // n) * (64 // p) <= ka.MAX_SPLIT_PAGES


# ── writes and the way back ──────────────────────────────────────────────────

@pytest.mark.gpu
@pytest.mark.parametrize("hkv,p,d", [(8, 16, 128), (3, 32, 64), (1, 64, 128)])
@pytest.mark.parametrize("n_tok", [1, 5])
def test_kv_append_equals_torch_and_leaves_the_rest(cuda, hkv, p, d, n_tok):
    pool = random_pool(6, hkv, p, d, 1)
    before = [t.clone() for t in (pool.k, pool.v, pool.k_scale, pool.v_scale)]
    g = torch.Generator().manual_seed(2)
    k = (torch.randn(4, hkv, n_tok, d, generator=g) * torch.tensor([1.0, 1e-3, 300.0, 1.0]).view(4, 1, 1, 1)).half()
    v = torch.randn(4, hkv, n_tok, d, generator=g).half()
    v[0, 0, 0] = 0
    v[1] = 6e-8                                          # the smallest fp16 numbers: a scale of 0
    slots = torch.tensor([5, 0, 2, 9], dtype=torch.int32)
    offs = torch.tensor([0, p - n_tok, 7, 1], dtype=torch.int32)
    ka.kv_append_q8(k.cuda(), v.cuda(), pool, slots.cuda(), offs.cuda(), p)
    want = [t.cpu().clone() for t in before]
    for b in range(3):                                   # (the fourth item's slot is outside the pool)
        at = slice(int(offs[b]), int(offs[b]) + n_tok)
        for i, x in ((0, k), (1, v)):
            c, s = quantised(x[b])
            want[i][slots[b], :, at] = c
            want[2 + i][slots[b], :, at] = s
    for got, w in zip((pool.k, pool.v, pool.k_scale, pool.v_scale), want):
        assert torch.equal(got.cpu(), w)


@pytest.mark.gpu
def test_append_of_values_that_are_not_finite_and_past_the_page(cuda):
    pool = random_pool(2, 2, 16, 64, 3)
    old = pool.k[1, :, :14].clone(), pool.v[1, :, :14].clone()
    k = torch.randn(1, 2, 4, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    v = k.clone()
    k[0, 0, 0, 5], v[0, 1, 1, 7] = float("nan"), float("inf")
    ka.kv_append_q8(k, v, pool, torch.tensor([1], dtype=torch.int32, device=cuda),
                    torch.tensor([14], dtype=torch.int32, device=cuda))   # tokens 2 and 3 lie past the page
    view = ka.dequantize_pages(pool, torch.tensor([1], dtype=torch.int32, device=cuda))
    assert view.k[0, 0, 14].isnan().all() and view.k[0, 1, 14].isfinite().all()
    assert view.v[0, 1, 15].isnan().all() and view.v[0, 0, 15].isfinite().all()
    assert torch.equal(pool.k[1, :, :14], old[0]) and torch.equal(pool.v[1, :, :14], old[1])


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,p,d", [(8, 16, 128), (2, 32, 64), (1, 64, 128)])
def test_dequantize_pages(cuda, hkv, p, d):
    pool = random_pool(7, hkv, p, d, 4)
    pages = torch.tensor([3, 3, 0, 7, -1, 6], dtype=torch.int32)
    view = ka.dequantize_pages(pool, pages.cuda())
    k, v = held(pool)
    for i, s in enumerate(pages.tolist()):
        inside = 0 <= s < 7
        assert torch.equal(view.k[i].cpu(), k[s].half() if inside else torch.zeros(hkv, p, d).half())
        assert torch.equal(view.v[i].cpu(), v[s].half() if inside else torch.zeros(hkv, p, d).half())
    assert ka.dequantize_pages(pool, pages[:0].cuda()).k.shape == (0, hkv, p, d)


def rope_reference(qkv, qw, kw, pos, inv, hq, hkv, d):
    n = qkv.shape[0]
    x = qkv.double().view(n, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if qw is not None:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + EPS) * qw.double()
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * kw.double()
    a = pos.double().view(n, 1, 1) * inv.double()
    c, s = torch.cat([a.cos(), a.cos()], -1), torch.cat([a.sin(), a.sin()], -1)

    def turn(t):
        return t * c + torch.cat([-t[..., d // 2:], t[..., :d // 2]], -1) * s
    return turn(q), turn(k), v


@pytest.mark.gpu
@pytest.mark.parametrize("n,hq,hkv,p,d,first", [(1, 32, 8, 16, 128, 0), (5, 16, 8, 32, 64, 131071), (3, 8, 1, 64, 128, 77),
                                                (300, 32, 8, 16, 128, 5), (600, 16, 8, 16, 64, 1000), (1000, 8, 1, 32, 128, 3),
                                                (257, 40, 8, 64, 128, 60000), (400, 5, 5, 16, 64, 15)])
@pytest.mark.parametrize("norm", [True, False])
def test_norm_rope_append(cuda, n, hq, hkv, p, d, first, norm):
    g = torch.Generator().manual_seed(n)
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g).half()
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).half() for _ in range(2))
    if not norm:
        qw = kw = None
    pos = torch.arange(first, first + n, dtype=torch.int32)
    inv = (1e6 ** (-torch.arange(0, d, 2).double() / d)).float()
    pages = (first + n - 1) // p - first // p + 1
    order = torch.randperm(pages + 2, generator=g)[:pages].int()
    slots = order[(pos // p - first // p).long()]
    if n > 4:
        slots[n // 2] = -1                               # a token that is not to be kept
    pool = random_pool(pages + 2, hkv, p, d, 5)
    before = [t.cpu().clone() for t in (pool.k, pool.v, pool.k_scale, pool.v_scale)]
    dev = [None if t is None else t.cuda() for t in (qkv, qw, kw, pos, inv, slots, pos % p)]
    out = fused.qk_norm_rope_append_q8(dev[0], dev[1], dev[2], EPS, dev[3], dev[4], None, pool, dev[5], dev[6], hq, hkv,
                                       d, p)
    q, k, v = rope_reference(qkv, qw, kw, pos, inv, hq, hkv, d)
    top = q.abs().amax(-1, keepdim=True)
    assert ((out.cpu().double() - q).abs() <= 2.0 ** -11 * q.abs() + 2.0 ** -20 * top + 2.0 ** -25).all()
    live = torch.arange(n)[slots >= 0]
    at = (slots[live].long(), slice(None), (pos[live] % p).long())
    c, s = quantised(v.half())
    assert torch.equal(pool.v.cpu()[at], c[live]) and torch.equal(pool.v_scale.cpu()[at], s[live])
    ks = pool.k_scale.cpu()[at].double()[..., None]
    top = k[live].abs().amax(-1, keepdim=True)
    assert ((ks - top / 127).abs() <= (2.0 ** -11 + 2.0 ** -20) * top / 127 + 2.0 ** -25).all()
    # half a step, a largest code that a scale 2^-11 short clips, and the chain
    err = (pool.k.cpu()[at].double() * ks - k[live]).abs()
    assert (err <= ks * (0.5 + 127 * 2.0 ** -11) + 2.0 ** -20 * top).all()
    for t, old in zip((pool.k, pool.v, pool.k_scale, pool.v_scale), before):
        t = t.cpu().clone()
        t[at] = old[at]
        assert torch.equal(t, old)                       # no other place written


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,p,d,n", [(32, 8, 16, 128, 500), (20, 5, 32, 64, 500)])
def test_append_does_not_depend_on_the_batch(cuda, hq, hkv, p, d, n):
    """A token's bits are the same written alone, in a small batch and in a prompt."""
    g = torch.Generator().manual_seed(8)
    wide = torch.randn(n, (hq + 2 * hkv) * d + 8, generator=g).half().cuda()
    qkv = wide[:, :-8]
    w = (1 + 0.1 * torch.randn(d, generator=g)).half().cuda()
    pos = torch.arange(40, 40 + n, dtype=torch.int32, device=cuda)
    inv = (1e6 ** (-torch.arange(0, d, 2).double() / d)).float().cuda()
    slots, offs = (pos // p).int(), (pos % p).int()
    pools = [ka.alloc_q8_pool(40, hkv, p, d, cuda) for _ in range(2)]
    q0 = fused.qk_norm_rope_append_q8(qkv, w, w, EPS, pos, inv, None, pools[0], slots, offs, hq, hkv, d)
    q1 = torch.cat([fused.qk_norm_rope_append_q8(qkv[i:i + s], w, w, EPS, pos[i:i + s], inv, None, pools[1], slots[i:i + s],
                                                 offs[i:i + s], hq, hkv, d) for i, s in ((0, 1), (1, 16), (17, 90), (107, 393))])
    assert torch.equal(q0, q1)
    for a, b in zip((pools[0].k, pools[0].v, pools[0].k_scale, pools[0].v_scale),
                    (pools[1].k, pools[1].v, pools[1].k_scale, pools[1].v_scale)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,p,d", [(32, 8, 16, 128), (20, 5, 32, 64)])
@pytest.mark.parametrize("places", ["any", "runs"])
def test_append_to_any_places(cuda, hq, hkv, p, d, places):
    """Tokens of a prompt in any order of places, some outside the pool, some not finite."""
    n = 509
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g).half()
    qkv[77, 5], qkv[78, hq * d + 3], qkv[79, -1], qkv[80] = float("nan"), float("inf"), float("nan"), 0
    at = torch.randperm(40 * p, generator=g)[:n]
    if places == "runs":                                 # starts and lengths of every kind, in pages in any order
        at, page = [], iter(torch.randperm(40 * p // 16, generator=g).tolist())
        for i in range(n):
            first, length = i % 5, 1 + i % 11
            base = next(page, None)
            at += [] if base is None else [base * 16 + j for j in range(first, min(first + length, 16))]
        at = torch.tensor((at + [-p] * n)[:n])
    slots, offs = (at // p).int(), (at % p).int()
    slots[100], slots[101], offs[102], offs[103] = -1, 40, p, -1
    w = (1 + 0.1 * torch.randn(d, generator=g)).half().cuda()
    pos = torch.arange(n, dtype=torch.int32, device=cuda)
    inv = (1e6 ** (-torch.arange(0, d, 2).double() / d)).float().cuda()
    pools = [random_pool(40, hkv, p, d, 11) for _ in range(2)]
    qkv, slots, offs = qkv.cuda(), slots.cuda(), offs.cuda()
    q0 = fused.qk_norm_rope_append_q8(qkv, w, w, EPS, pos, inv, None, pools[0], slots, offs, hq, hkv, d)
    q1 = torch.cat([fused.qk_norm_rope_append_q8(qkv[i:i + 100], w, w, EPS, pos[i:i + 100], inv, None, pools[1], slots[i:i + 100],
                                                 offs[i:i + 100], hq, hkv, d) for i in range(0, n, 100)])
    assert torch.equal(q0.nan_to_num(77.0), q1.nan_to_num(77.0))
    for name in ("k", "v", "k_scale", "v_scale"):
        a, b = (getattr(x, name) for x in pools)
        assert torch.equal(a.view(torch.int8), b.view(torch.int8))


# ── attention ────────────────────────────────────────────────────────────────

def attention_reference(q, pool, table, lens, scale):
    k, v = held(pool)
    b, hq, d = q.shape
    hkv, p = pool.num_kv_heads, pool.page_size
    out = torch.zeros(b, hq, d, dtype=torch.float64)
    top = torch.zeros(b, hq, 1, dtype=torch.float64)
    for i in range(b):
        rows = [(s, t) for j, s in enumerate(table[i].tolist()) for t in range(p)
                if j * p + t < int(lens[i]) and 0 <= s < pool.num_slots]
        if not rows:
            continue
        s, t = (torch.tensor(x) for x in zip(*rows))
        for h in range(hq):
            kk, vv = k[s, h // (hq // hkv), t], v[s, h // (hq // hkv), t]
            out[i, h] = torch.softmax(kk @ q[i, h].double() * scale, 0) @ vv
            top[i, h] = vv.abs().max()
    return out, top


def check_attention(o, q, pool, table, lens, scale):
    e, top = attention_reference(q.cpu(), pool, table.cpu(), lens.cpu(), scale)
    err = (o.cpu().double() - e).abs()
    tol = 2.0 ** -11 * e.abs() + 2.0 ** -16 * top + 2.0 ** -25
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,p,d", [(32, 8, 16, 128), (5, 5, 32, 64), (16, 1, 64, 128), (40, 8, 16, 64), (12, 2, 32, 128),
                                        (8, 8, 64, 64)])
@pytest.mark.parametrize("splits", [0, 1, 3, 40])
def test_attention_against_fp64(cuda, hq, hkv, p, d, splits):
    lens = torch.tensor([0, 1, 63, 64, 65, 200, 777], dtype=torch.int32)
    cols = -(-777 // p)
    pool = random_pool(7 * cols, hkv, p, d, hq)
    g = torch.Generator().manual_seed(d)
    table = torch.randperm(7 * cols, generator=g).int().view(7, cols)
    q = torch.randn(7, hq, d, generator=g).half()
    # places behind an item's last token hold what an unwritten page may hold
    for i, n in enumerate(lens.tolist()):
        for j in range(cols):
            keep = min(max(n - j * p, 0), p)
            pool.k_scale[int(table[i, j]), :, keep:] = float("nan")
            pool.v_scale[int(table[i, j]), :, keep:] = float("inf")
    o = ka.paged_decode_attention_q8(q.cuda(), pool, table.cuda(), lens.cuda(), p, num_splits=splits)
    assert not o[0].any()
    for s in (pool.k_scale, pool.v_scale):
        s.nan_to_num_(nan=0.0, posinf=0.0)
    check_attention(o, q, pool, table, lens, 1 / math.sqrt(d))


@pytest.mark.gpu
def test_attention_large_scores_small_values_and_bad_pages(cuda):
    hq, hkv, p, d = 16, 4, 16, 128
    pool = random_pool(64, hkv, p, d, 2)
    pool.v_scale *= 1e-4
    table = torch.randperm(64, generator=torch.Generator().manual_seed(0)).int().view(2, 32)
    table[0, 3], table[1, 0], table[1, 31] = -1, 64, 1 << 30           # entries outside the pool
    lens = torch.tensor([500, 512], dtype=torch.int32)
    q = (torch.randn(2, hq, d, generator=torch.Generator().manual_seed(1)) * 1.5).half()
    o = ka.paged_decode_attention_q8(q.cuda(), pool, table.cuda(), lens.cuda(), p, scale=0.1)
    check_attention(o, q, pool, table, lens, 0.1)
    table[:] = -1
    assert not ka.paged_decode_attention_q8(q.cuda(), pool, table.cuda(), lens.cuda(), p).any()


@pytest.mark.gpu
def test_attention_lengths_past_the_table_end_with_it(cuda):
    pool = random_pool(8, 2, 16, 64, 2)
    table = torch.arange(8, dtype=torch.int32, device=cuda).view(2, 4)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    full = torch.tensor([64, 64], dtype=torch.int32, device=cuda)
    o = ka.paged_decode_attention_q8(q, pool, table, full)
    assert torch.equal(ka.paged_decode_attention_q8(q, pool, table, full + 1000), o)
    assert not ka.paged_decode_attention_q8(q, pool, table, -full).any()
    assert not ka.paged_decode_attention_q8(q, pool, table[:, :0], full).any()
    assert ka.paged_decode_attention_q8(q[:0], pool, table[:0], full[:0]).shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("splits,n", [(1, 256), (8, 2000)])
def test_a_nan_in_a_live_token_reaches_its_item_alone(cuda, splits, n):
    pool = random_pool(2 * n // 16, 2, 16, 128, 2)
    table = torch.arange(2 * n // 16, dtype=torch.int32, device=cuda).view(2, -1)
    lens = torch.tensor([n, n], dtype=torch.int32, device=cuda)
    q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(1)).half().cuda()
    clean = ka.paged_decode_attention_q8(q, pool, table, lens, num_splits=splits)
    for t in (pool.k_scale, pool.v_scale):
        old = t[3, 1, 5].clone()
        t[3, 1, 5] = float("nan")
        o = ka.paged_decode_attention_q8(q, pool, table, lens, num_splits=splits)
        assert o[0, 2:].isnan().all() and torch.equal(o[0, :2], clean[0, :2]) and torch.equal(o[1], clean[1])
        t[3, 1, 5] = old
    q[1, 0, 7] = float("inf")                            # and one in q its head alone
    o = ka.paged_decode_attention_q8(q, pool, table, lens, num_splits=splits)
    assert o[1, 0].isnan().all() and torch.equal(o[1, 1:], clean[1, 1:]) and torch.equal(o[0], clean[0])


@pytest.mark.gpu
def test_attention_of_many_items_follows_their_lengths(cuda):
    """150 items (three waves of lengths), most of them empty or short, one long; the same bits
    whatever the other items hold."""
    b, hq, hkv, p, d = 150, 4, 2, 16, 64
    lens = torch.zeros(b, dtype=torch.int32)
    lens[::7], lens[77], lens[149] = 33, 3000, 129
    cols = -(-3000 // p)
    pool = random_pool(400, hkv, p, d, 3)
    table = torch.randint(0, 400, (b, cols), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    q = torch.randn(b, hq, d, generator=torch.Generator().manual_seed(1)).half()
    o = ka.paged_decode_attention_q8(q.cuda(), pool, table.cuda(), lens.cuda(), p)
    some = torch.tensor([0, 1, 7, 70, 76, 77, 78, 147, 149])
    check_attention(o[some.cuda()], q[some], pool, table[some], lens[some], d ** -0.5)
    assert not o[lens.cuda() == 0].any()


@pytest.mark.gpu
def test_captured_attention_follows_new_lengths(cuda):
    b, hq, hkv, p, d = 3, 8, 2, 16, 128
    pool = random_pool(3 * 128, hkv, p, d, 3)
    table = torch.arange(3 * 128, dtype=torch.int32, device=cuda).view(3, 128)
    q = torch.randn(b, hq, d, generator=torch.Generator().manual_seed(1)).half().cuda()
    lens = torch.tensor([5, 2000, 900], dtype=torch.int32, device=cuda)
    ws = ka.AttnWorkspace(cuda)
    ka.paged_decode_attention_q8(q, pool, table, lens, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ka.paged_decode_attention_q8(q, pool, table, lens, workspace=ws)
    for n in ([2048, 1, 0], [64, 64, 65], [0, 0, 0], [700, 2048, 2048]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, ka.paged_decode_attention_q8(q, pool, table, lens))


@pytest.mark.gpu
def test_attention_strides_views_and_refusals(cuda):
    hq, hkv, p, d = 8, 2, 16, 128
    # slots of one layer of a pool that interleaves layers
    k = torch.randint(-127, 128, (6, 3, hkv, p, d), dtype=torch.int8, device=cuda)
    v = torch.randint(-127, 128, (6, 3, hkv, d, p), dtype=torch.int8, device=cuda)
    s = (torch.rand(2, 6, 3, hkv, p, device=cuda) * 0.02).half()
    pool = ka.Q8PoolView(k[:, 1], v[:, 1].transpose(-1, -2), s[0][:, 1], s[1][:, 1])
    table = torch.tensor([[4, 0, 9], [2, 5, 9]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([30, 17], dtype=torch.int32, device=cuda)
    wide = torch.randn(2, 20, d, device=cuda).half()
    q = wide[:, 3:11]
    o = ka.paged_decode_attention_q8(q, pool, table[:, :2], lens, p)
    check_attention(o, q, pool, table[:, :2], lens, 1 / math.sqrt(d))
    flat = torch.randn(2 * hq * d + 1, device=cuda).half()[1:].view(2, hq, d)      # not 16-byte aligned
    assert torch.equal(ka.paged_decode_attention_q8(flat, pool, table, lens),
                       ka.paged_decode_attention_q8(flat.clone(), pool, table, lens))
    for bad in (lambda: ka.paged_decode_attention_q8(q.float(), pool, table, lens),
                lambda: ka.paged_decode_attention_q8(q[..., :64], pool, table, lens),
                lambda: ka.paged_decode_attention_q8(q, pool, table.long(), lens),
                lambda: ka.paged_decode_attention_q8(q, pool, table[:1], lens),
                lambda: ka.paged_decode_attention_q8(q, pool, table, lens[:1]),
                lambda: ka.paged_decode_attention_q8(q, pool, table, lens, 32),
                lambda: ka.paged_decode_attention_q8(wide[:, :7], pool, table, lens),
                lambda: ka.paged_decode_attention_q8(q, pool, table, lens, out=o.float()),
                lambda: ka.kv_append_q8(q[:, :3, None], q[:, :3, None], pool, lens, lens),
                lambda: ka.kv_append_q8(q[:, :2, None], q[:, :2, None], pool, lens[:1], lens),
                lambda: ka.dequantize_pages(pool, table),
                lambda: fused.qk_norm_rope_append_q8(wide.view(2, -1), None, None, EPS, lens, torch.zeros(64, device=cuda), None,
                                                     pool, lens, lens, 8, 2, 128),
                lambda: fused.qk_norm_rope_append_q8(wide[:, :12].reshape(2, -1), wide[0, 0], None, EPS, lens,
                                                     torch.zeros(64, device=cuda), None, pool, lens, lens, 8, 2, 128)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.gpu
def test_prompt_attends_dequantised_pages(cuda):
    """A prompt's chunk over 8-bit history: fp16 copies of the pages through prefill_attention.
    K, V, the probabilities and the output are each rounded to fp16 (2^-11): a score q.k moves by
    2^-11 |q||k|, the weighted mean by twice what its largest score moves plus two roundings of v."""
    hq, hkv, p, d, past, t = 8, 2, 16, 64, 70, 20
    pool = random_pool(8, hkv, p, d, 6)
    pages = torch.tensor([5, 1, 7, 0, 3, 2], dtype=torch.int32, device=cuda)
    q = torch.randn(t, hq, d, generator=torch.Generator().manual_seed(1)).half()
    view = ka.dequantize_pages(pool, pages)
    o = ka.prefill_attention(q.cuda(), view, torch.arange(6, dtype=torch.int32, device=cuda), p, q_start=past)
    for i in range(t):
        e, top = attention_reference(q[i:i + 1], pool, pages.cpu()[None], torch.tensor([past + i + 1]), 1 / math.sqrt(d))
        k, _ = held(pool)
        move = 2.0 ** -11 * float(q[i].double().norm(dim=-1).max() * k.norm(dim=-1).max()) / math.sqrt(d)
        assert ((o[i].cpu().double() - e[0]).abs() <= (2 * move + 3 * 2.0 ** -11) * top[0] + 2.0 ** -11 * e[0].abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,p,d", [(3, 16, 128), (2, 64, 64)])
@pytest.mark.parametrize("n_tok", [1, 2, 3, 4, 6, 9, 16])
def test_kv_append_at_every_place_of_a_word(cuda, hkv, p, d, n_tok):
    """n_tok tokens from every offset, before and past the page too."""
    offs = torch.arange(-5, p + 2, dtype=torch.int32)
    n = len(offs)
    g = torch.Generator().manual_seed(n_tok)
    k, v = (torch.randn(n, hkv, n_tok, d, generator=g).half() for _ in range(2))
    pool = random_pool(n, hkv, p, d, 6)
    want = [t.cpu().clone() for t in (pool.k, pool.v, pool.k_scale, pool.v_scale)]
    slots = torch.randperm(n, generator=g).int()
    ka.kv_append_q8(k.cuda(), v.cuda(), pool, slots.cuda(), offs.cuda(), p)
    for b in range(n):
        for t in range(n_tok):
            at = int(offs[b]) + t
            if 0 <= at < p:
                for i, x in ((0, k), (1, v)):
                    c, s = quantised(x[b, :, t])
                    want[i][slots[b], :, at] = c
                    want[2 + i][slots[b], :, at] = s
    for got, w in zip((pool.k, pool.v, pool.k_scale, pool.v_scale), want):
        assert torch.equal(got.cpu(), w)


def test_a_workspace_keeps_what_it_has_outgrown():
    ws = ka.AttnWorkspace(torch.device("cpu"))
    first = ws.reserve(-1, 1000)
    ws.buf.fill_(5.0)
    assert ws.reserve(-1, 900) == first
    sizes = []
    for n in (1004, 1100, 5000):
        ws.reserve(-1, n)
        assert ws.buf.nbytes >= n
        sizes.append(ws.buf.nbytes)
    assert sizes == [2000, 2000, 5000]
    assert [t.data_ptr() for t in ws._outgrown if t.numel()][0] == first and (ws._outgrown[1] == 5.0).all()


@pytest.mark.gpu
def test_a_captured_call_outlives_its_workspace_s_growth(cuda):
    g = torch.Generator().manual_seed(14)
    pool = random_pool(64, 8, 16, 128, 15)
    ws = ka.AttnWorkspace(torch.device("cuda", 0))
    q = torch.randn(1, 32, 128, generator=g).half().cuda()
    table = torch.randperm(64, generator=g).int().view(1, 64).cuda()
    lens = torch.tensor([1000], dtype=torch.int32, device=cuda)
    want = ka.paged_decode_attention_q8(q, pool, table, lens, num_splits=8, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ka.paged_decode_attention_q8(q, pool, table, lens, num_splits=8, workspace=ws)
    many = q.expand(9, 32, 128).contiguous()
    for n in (3, 9):                                     # the workspace grows; others take what is free
        ka.paged_decode_attention_q8(many[:n], pool, table.expand(n, 64).contiguous(), lens.expand(n).contiguous(),
                                     num_splits=16, workspace=ws)
        others = [torch.full((1 << 18,), float(n), device=cuda) for _ in range(8)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all((t == float(n)).all() for t in others)


@pytest.mark.gpu
def test_a_pool_past_32_bits_of_elements(cuda):
    """Pages whose first element lies past 2^32: writes, attention and the way back, as in a small pool."""
    n, hkv, p, d = 270000, 8, 16, 128
    big, small = ka.alloc_q8_pool(n, hkv, p, d, cuda), ka.alloc_q8_pool(30, hkv, p, d, cuda)
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(400, (32 + 2 * hkv) * d, generator=g).half().cuda()
    inv = (1e6 ** (-torch.arange(0, d, 2).double() / d)).float().cuda()
    pos = torch.arange(400, dtype=torch.int32, device=cuda)
    order = torch.randperm(25, generator=g).int().cuda()
    outs = []
    for pool, base in ((big, n - 25), (small, 3)):
        slots = order[(pos // p).long()] + base
        q = torch.cat([fused.qk_norm_rope_append_q8(qkv[a:b], None, None, EPS, pos[a:b], inv, None, pool, slots[a:b],
                                                    pos[a:b] % p, 32, hkv, d) for a, b in ((0, 10), (10, 390))])
        kv = qkv[390:].view(10, 48, d)[:, 32:].unsqueeze(2)
        ka.kv_append_q8(kv[:, :hkv], kv[:, hkv:], pool, slots[390:], pos[390:] % p)
        o = ka.paged_decode_attention_q8(q[-1:], pool, (order + base)[None], torch.tensor([400], dtype=torch.int32, device=cuda))
        view = ka.dequantize_pages(pool, order + base)
        outs.append((q, o, view.k, view.v))
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and outs[0][1].any()
    assert not big.k[:n - 25].any() and not big.v[:1000].any()
