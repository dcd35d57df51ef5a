"""Linears with 4-bit weights: layout and refusals on the CPU, products on the GPU
against fp64.

Tolerance of one output.  The last rounding is off by at most 2^-11 |y|.  Up to 16 tokens
a group's sum runs over (b + u) x with b + u < 272 for half of the inputs and < 32 for the
others, and a start of sum((b + 8) x), in at most 32 fp32 additions of partial sums no larger
than 300 sum|x|, each off by at most 2^-24 of that: 32 * 2^-24 * 300 * s sum|x|, summed over
the groups.  Above 16 tokens every weight is
rounded to fp16 (2^-11 |w|) and the sum has K / 8 additions of partial sums no larger than
sum|w x|.  These are worst cases; as a whole, rounding errors are independent: the norm of
the error is at most 2^-11 / sqrt(3) of the norm of y for the last rounding and as much for
the weights', 4.0e-4 together.
"""
import numpy as np
import pytest
import torch

from helm_amd import _native
from helm_amd import kernels as hk

SHAPES = [(1, 32, 32), (16, 128, 128), (40, 160, 32), (250, 1056, 32), (4096, 4096, 128), (130, 17408, 128),
          (1024, 12288, 64), (4100, 2560, 64), (72, 8192, 32)]


def make(n, k, gs, seed, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    scale = ((0.5 + torch.rand(n, k // gs, generator=g)) * 0.006).half()
    return codes.to(device), scale.to(device)


def test_pack_places_every_code_as_documented():
    for n, k, gs in ((1, 32, 32), (17, 160, 32), (40, 256, 64), (33, 384, 128)):
        codes, scale = make(n, k, gs, n)
        w = hk.Int4Weight.pack(codes, scale)
        kt = -(-k // 128)
        words = w.qweight.numpy().view(np.uint32).reshape(-1)
        for i in range(n):
            for j in range(0, k, 7):
                lane = (j % 32) // 8 * 16 + i % 16
                word = int(words[((i // 16 * kt + j // 128) * 64 + lane) * 4 + j % 128 // 32])
                assert ((word >> (4 * (j % 8 // 2) + 16 * (j % 2))) & 15) - 8 == int(codes[i, j])
        s = w.scale
        assert s.shape == (-(-n // 16), kt, 128 // gs, 16)
        for i in range(n):
            for g in range(k // gs):
                assert s[i // 16, g * gs // 128, g % (128 // gs), i % 16] == scale[i, g]


def test_pack_pads_with_zero_weights_and_unpacks():
    codes, scale = make(5, 160, 32, 3)
    w = hk.Int4Weight.pack(codes, scale)
    c, s = w.unpack()
    assert torch.equal(c, codes) and torch.equal(s, scale)
    full = hk.Int4Weight(w.qweight, w.scale, 16, 256, 32).dequantize()
    assert not full[5:].any() and not full[:, 160:].any()
    assert torch.equal(w.dequantize(), codes.float() * scale.float().repeat_interleave(32, 1))


@pytest.mark.parametrize("gs", [32, 64, 128])
def test_quantize_is_within_half_a_step(gs):
    w = torch.randn(20, 512, generator=torch.Generator().manual_seed(gs)).half().float()
    w[3] = 0
    codes, scale = hk.quantize_int4(w, gs)
    s = scale.float().repeat_interleave(gs, 1)
    # fp16(amax / 7) may be 2^-11 short of amax / 7: the largest code is then off by 7 * 2^-11 steps more
    assert ((codes.float() * s - w).abs() <= s * (0.5 + 7 * 2.0 ** -11)).all()
    assert codes.abs().max() <= 7 and not codes[3].any()


def test_refusals():
    codes, scale = make(16, 128, 64, 0)
    for bad in (codes.float(), codes[0]):
        with pytest.raises(RuntimeError, match="codes must be int8"):
            hk.Int4Weight.pack(bad, scale)
    with pytest.raises(RuntimeError, match="does not fit"):
        hk.Int4Weight.pack(codes, scale[:8])
    with pytest.raises(RuntimeError, match="group size"):
        hk.Int4Weight.pack(codes, torch.ones(16, 8).half())
    with pytest.raises(RuntimeError, match=r"\[-8, 7\]"):
        hk.Int4Weight.pack(codes + 8, scale)
    with pytest.raises(ValueError):
        hk.quantize_int4(torch.zeros(4, 100), 32)
    w = hk.Int4Weight.pack(codes, scale)
    with pytest.raises(RuntimeError, match="on the GPU"):
        hk.int4_linear(torch.zeros(1, 128).half(), w)
    import ctypes
    fake = ctypes.c_void_p(16)
    lib = _native.lib()

    def call(x=fake, ldx=128, gs=64, ldy=16, m=1, n=16, k=128, ws=None, ws_bytes=0, q=fake):
        return lib.helm_int4_linear(x, ldx, q, fake, gs, None, fake, ldy, m, n, k, ws, ws_bytes, None)
    assert call(x=None) == -1 and call(ldx=64) == -1 and call(ldy=8) == -1 and call(m=0) == -1
    assert call(gs=48) == -2 and call(k=96) == -2 and call(ldx=132) == -2 and call(q=ctypes.c_void_p(8)) == -2
    assert lib.helm_int4_linear_workspace_bytes(1, 4096, 17408, 64) > 0
    assert call(n=4096, ldy=4096, k=17408, ldx=17408) == -1
    assert b"workspace" in lib.helm_last_error()


def test_patch_swaps_linears_and_leaves_odd_ones():
    import torch.nn as nn
    m = nn.Sequential(nn.Linear(128, 40), nn.Sequential(nn.Linear(96, 8), nn.Linear(256, 5, bias=False)))
    m.lm_head = nn.Linear(128, 4)
    assert hk.patch_int4_linears(m, 128, exclude=("lm_head",)) == 2
    assert isinstance(m[0], hk.Int4Linear) and isinstance(m[1][0], nn.Linear) and isinstance(m[1][1], hk.Int4Linear)
    assert m[0].weight.shape == (40, 128) and m[0].bias.dtype == torch.float16 and "int4=True" in repr(m[0])
    assert set(m.state_dict()) >= {"0.qweight", "0.scale", "0.bias"}


# ── on the GPU ───────────────────────────────────────────────────────────────

def check(y, x, codes, scale, bias, gs):
    x64, m = x.double().cpu(), x.shape[0]
    s = scale.double().cpu().repeat_interleave(gs, 1)
    w = codes.double().cpu() * s
    e = x64 @ w.t() + (0 if bias is None else bias.double().cpu())
    tol = 2.0 ** -11 * e.abs() + 2.0 ** -25
    if m <= 16:
        tol += 32 * 2.0 ** -24 * 300 * (x64.abs() @ s.t())
    else:
        tol += (2.0 ** -11 + w.shape[1] / 8 * 2.0 ** -23) * (x64.abs() @ w.abs().t())
    err = (y.double().cpu() - e).abs()
    assert (err <= tol).all(), float((err / tol).max())
    if e.numel() >= 1000 and bias is None:
        assert float(err.norm() / e.norm()) <= 4.0e-4


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,gs", SHAPES)
@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 33, 70, 90, 200])
def test_against_fp64(cuda, m, n, k, gs):
    codes, scale = make(n, k, gs, 7 * m + n)
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, k, generator=g).half().cuda()
    bias = torch.randn(n, generator=g).half().cuda() if m % 2 else None
    w = hk.Int4Weight.pack(codes.cuda(), scale.cuda())
    y = hk.int4_linear(x, w, bias)
    assert y.shape == (m, n) and y.dtype == torch.float16
    check(y, x, codes, scale, bias, gs)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40])
def test_strides_shapes_and_out(cuda, m):
    codes, scale = make(72, 256, 64, 1)
    w = hk.Int4Weight.pack(codes, scale).to(cuda)
    wide = torch.randn(m, 400, generator=torch.Generator().manual_seed(2)).half().cuda()
    x = wide[:, 8:264]
    whole = hk.int4_linear(x.contiguous(), w)
    check(whole, x, codes, scale, None, 64)
    assert torch.equal(hk.int4_linear(x, w), whole)                       # strided rows
    assert torch.equal(hk.int4_linear(wide[:, 3:259], w), hk.int4_linear(wide[:, 3:259].contiguous(), w))
    assert torch.equal(hk.int4_linear(x.unsqueeze(0), w), whole.unsqueeze(0))
    askew = torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].view(m, 256)  # contiguous, not 16-byte aligned
    assert torch.equal(hk.int4_linear(askew, w), whole)
    out = torch.full((m, 72), 7.0, dtype=torch.float16, device=cuda)
    assert hk.int4_linear(x, w, out=out) is out and torch.equal(out, whole)
    assert hk.int4_linear(x[:0], w).shape == (0, 72)
    one = x[:1].expand(m, 256)
    assert torch.equal(hk.int4_linear(one, w), hk.int4_linear(one.contiguous(), w))
    assert torch.equal(hk.int4_linear(x[0], w), hk.int4_linear(x[:1], w)[0])
    mod = hk.Int4Linear(w)
    assert torch.equal(mod(x), whole) and mod.weight.shape == (72, 256)
    for bad in (dict(out=out[:, :8]), dict(bias=torch.zeros(71, device=cuda).half()), dict(bias=torch.zeros(72, device=cuda))):
        with pytest.raises(RuntimeError):
            hk.int4_linear(x, w, **bad)
    with pytest.raises(RuntimeError, match="fp16"):
        hk.int4_linear(x.float(), w)
    with pytest.raises(RuntimeError, match="laid out"):
        hk.Int4Weight(w.qweight, w.scale, 90, 256, 64)


@pytest.mark.gpu
def test_rows_do_not_depend_on_their_neighbours(cuda):
    codes, scale = make(200, 640, 128, 4)
    w = hk.Int4Weight.pack(codes, scale).to(cuda)
    x = torch.randn(16, 640, generator=torch.Generator().manual_seed(1)).half().cuda()
    whole = hk.int4_linear(x, w)
    for m in (1, 2, 9):
        assert torch.equal(hk.int4_linear(x[:m], w), whole[:m])
    x[3] = float("nan")
    bad = hk.int4_linear(x, w)
    keep = [i for i in range(16) if i != 3]
    assert bad[3].isnan().all() and torch.equal(bad[keep], whole[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 30])
def test_captured_and_on_another_stream(cuda, m):
    codes, scale = make(512, 17408, 128, 9)
    w = hk.Int4Weight.pack(codes, scale).to(cuda)
    g = torch.Generator().manual_seed(3)
    xs = [torch.randn(m, 17408, generator=g).half().cuda() for _ in range(3)]
    eager = [hk.int4_linear(x, w) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = hk.int4_linear(xs[0], w)
    side.synchronize()
    assert torch.equal(y, eager[0])
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hk.int4_linear(x, w)
    for i in (1, 2, 0, 1):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[i])


def test_rows_too_far_apart_for_the_c_entry():
    import ctypes
    fake = ctypes.c_void_p(16)
    far = _native.lib().helm_int4_linear
    assert far(fake, (1 << 23) + 8, fake, fake, 64, None, fake, 16, 2, 16, 128, None, 0, None) == -2
    assert b"2^23" in _native.lib().helm_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 20])
def test_rows_far_apart(cuda, m):
    codes, scale = make(40, 256, 64, 6)
    w = hk.Int4Weight.pack(codes, scale).to(cuda)
    for ldx in (1 << 23, (1 << 23) + 8):
        x = torch.empty((m - 1) * ldx + 256, dtype=torch.float16, device=cuda).as_strided((m, 256), (ldx, 1))
        x.copy_(torch.randn(m, 256, generator=torch.Generator().manual_seed(m)).half())
        check(hk.int4_linear(x, w), x, codes, scale, None, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(20, 4096, 4096), (60, 900, 2176), (95, 2000, 1152), (127, 4100, 1408), (260, 1300, 640),
                                   (500, 2064, 896), (129, 300, 128), (33, 130, 384)])
def test_prompts_of_every_tile_height_and_slicing(cuda, m, n, k, gs):
    codes, scale = make(n, k, gs, m)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(n)).half().cuda()
    check(hk.int4_linear(x, hk.Int4Weight.pack(codes.cuda(), scale.cuda())), x, codes, scale, None, gs)


@pytest.mark.gpu
@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 128), (40, 640), (250, 1152), (4100, 2560), (4096, 12288), (17408, 5120)])
def test_two_blocks_of_tokens(cuda, n, k, gs):
    """17 to 32 tokens: the decode form's bound, and rows that do not depend on their neighbours."""
    codes, scale = make(n, k, gs, n)
    w = hk.Int4Weight.pack(codes.cuda(), scale.cuda())
    x = torch.randn(32, k, generator=torch.Generator().manual_seed(k)).half().cuda()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(5)).half().cuda()
    s = scale.double().repeat_interleave(gs, 1)
    for m in (17, 24, 31, 32):
        y = hk.int4_linear(x[:m], w, bias)
        e = x[:m].double().cpu() @ (codes.double() * s).t() + bias.double().cpu()
        err = (y.double().cpu() - e).abs()
        assert (err <= 2.0 ** -11 * e.abs() + 2.0 ** -25 + 32 * 2.0 ** -24 * 300 * (x[:m].double().cpu().abs() @ s.t())).all()
    x[20] = float("nan")
    bad = hk.int4_linear(x, w, bias)
    keep = [i for i in range(32) if i != 20]
    assert bad[20].isnan().all() and torch.equal(bad[keep], y[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 20, 40])
def test_weights_past_32_bits_of_bytes(cuda, m):
    """4.3 GB of codes: the last outputs against the product with their own tiles."""
    nt, kt = 16384, 256
    q = torch.randint(-2 ** 31, 2 ** 31 - 1, (nt, kt, 64, 4), dtype=torch.int32, device=cuda)
    s = ((0.5 + torch.rand(nt, kt, 1, 16, device=cuda)) * 0.006).half()
    w = hk.Int4Weight(q, s, nt * 16, kt * 128, 128)
    x = torch.randn(m, kt * 128, generator=torch.Generator().manual_seed(m)).half().cuda()
    y = hk.int4_linear(x, w)
    for first in (0, nt // 2, nt - 2):
        codes, scale = hk.Int4Weight(q[first:first + 2].clone(), s[first:first + 2].clone(), 32, kt * 128, 128).unpack()
        check(y[:, first * 16:first * 16 + 32], x, codes, scale, None, 128)
