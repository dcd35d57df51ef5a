"""int4_linear against its definition in fp64 where the kernels' forms could part from it: one rounding
whatever the number of tokens, scales of any size, infinite inputs, inputs of one sign, and every form that
the shapes can take.

Tolerance.  y = fp16(e + d) with e exact, so |y - e| <= |fp16(e) - e| + 2 |d| (the distance to the nearest
fp16 number changes by no more than its argument does).  d sums fp32 errors, each at most 2^-23 (a matrix
instruction may cut off instead of rounding) of a partial sum:
  * sums over the codes themselves (17 tokens and more): up to 128 inputs of a group one after another, partial
    sums no larger than sum |c x| of the group, then K / 32 groups, 16 waves or slices and the bias;
  * up to 16 tokens: 32 additions of partial sums no larger than 300 sum |x| of the group (codes plus 8 behind an
    offset of up to 256), the rest as above.
As a whole d is far smaller: its signs are independent, and its norm below 2^-18 of e's norm.
"""
import numpy as np
import pytest
import torch

from helm_amd import kernels as hk


def make(n, k, gs, seed, big=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8, device="cuda")
    scale = ((0.5 + torch.rand(n, k // gs, generator=g, device="cuda")) * 0.006 * big).half()
    return codes, scale


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").half()


def exact(x, codes, scale, bias=None):
    """fp64 products, and the bounds' sums: sum |w x| and sum s |x|."""
    gs = codes.shape[1] // scale.shape[1]
    s = scale.double().repeat_interleave(gs, 1)
    w, x64 = codes.double() * s, x.double()
    e = x64 @ w.t().contiguous()
    if bias is not None:
        e += bias.double()
    return e, x64.abs() @ w.abs().t().contiguous(), x64.abs() @ s.t().contiguous()


def check(y, x, codes, scale, bias=None):
    e, wx, sx = exact(x, codes, scale, bias)
    k, m = codes.shape[1], x.shape[0]
    d = (k / 32 + 16 + 20 + (0 if m <= 16 else 128)) * 2.0 ** -23 * wx + (32 * 2.0 ** -23 * 300 * sx if m <= 16 else 0)
    if bias is not None:
        d += 2.0 ** -23 * bias.double().abs()
    nearest = (e.half().double() - e).abs()
    err = (y.double() - e).abs()
    assert (err <= nearest + 2 * d).all(), float((err - nearest - 2 * d).max())
    if e.numel() >= 4000:
        assert float(err.norm()) <= float(nearest.norm()) + 2.0 ** -17 * float(e.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 16, 17, 32, 33, 64, 65, 100, 250])
@pytest.mark.parametrize("n,k", [(200, 256), (1000, 4096)])
def test_one_rounding_at_any_number_of_tokens(cuda, m, gs, n, k):
    codes, scale = make(n, k, gs, m)
    x = normal(n + m, m, k)
    bias = normal(5, n)
    w = hk.Int4Weight.pack(codes, scale)
    check(hk.int4_linear(x, w), x, codes, scale)
    check(hk.int4_linear(x, w, bias), x, codes, scale, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 20, 33, 100])
def test_scales_whose_products_fp16_does_not_hold(cuda, m, gs):
    """Scales up to 60000 and down to the smallest: code * scale is beyond fp16 or below its steps, y is not."""
    n, k = 150, 384
    codes, _ = make(n, k, gs, m)
    scale = torch.full((n, k // gs), 60000.0, device=cuda).half()
    scale[::2] = 2.0 ** -24
    scale[::3] = 3 * 2.0 ** -24
    x = normal(3, m, k) * 2.0 ** -6
    x[:, ::5] = 0
    for factor in (2.0 ** -3, 1.0):
        xs = (x.float() * factor).half()
        check(hk.int4_linear(xs, hk.Int4Weight.pack(codes, scale)), xs, codes, scale)


def with_infinities(m, n, k, gs):
    """x with infinities in three rows, and weights of which half of the outputs have no code of 0."""
    codes, scale = make(n, k, gs, m + n)
    half = codes[:(n + 1) // 2]
    half[half == 0] = 3
    x = normal(k, m, k)
    clean = x.clone()
    x[0, k // 3] = float("inf")
    x[m // 2, k - 1] = float("-inf")                      # the last one: next to where K may end inside a tile
    x[m - 1, 1] = float("inf")
    x[m - 1, k - 9] = float("inf")
    return x, clean, codes, scale


def check_infinities(x, clean, codes, scale):
    w = hk.Int4Weight.pack(codes, scale)
    y, finite = hk.int4_linear(x, w).cpu(), hk.int4_linear(clean, w).cpu()
    gs = codes.shape[1] // scale.shape[1]
    e = x.cpu().double() @ (codes.cpu().double() * scale.cpu().double().repeat_interleave(gs, 1)).t()
    rows = ~x.isfinite().all(-1).cpu()
    assert torch.equal(y[~rows], finite[~rows])           # the other tokens keep their bits
    got, want = y[rows].double(), e[rows]
    assert not want.isfinite().any() and want.isinf().any()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0.0, 1.0, -1.0), want.nan_to_num(0.0, 1.0, -1.0))


INFINITE = [(40, 128, 128), (72, 160, 32), (100, 192, 64), (250, 1056, 32), (130, 17408, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,gs", INFINITE)
@pytest.mark.parametrize("m", [33, 70, 90, 200])
def test_infinite_inputs_of_a_prompt(cuda, m, n, k, gs):
    check_infinities(*with_infinities(m, n, k, gs))


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,gs", INFINITE + [(1000, 4096, 64), (300, 5120, 128), (600, 2048, 128), (16400, 512, 32)])
@pytest.mark.parametrize("m", [1, 5, 16, 17, 32])
def test_infinite_inputs_of_a_few_tokens(cuda, m, n, k, gs):
    check_infinities(*with_infinities(m, n, k, gs))


@pytest.mark.gpu
@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 16, 17, 32, 33, 100])
def test_inputs_of_one_sign(cuda, m, gs):
    """Sums of codes plus an offset are far larger than the sums of codes that they stand for."""
    n, k = 500, 4096
    codes, scale = make(n, k, gs, m)
    x = (2.0 + normal(m, m, k).float().abs()).half()
    for signed in (x, -x):
        check(hk.int4_linear(signed, hk.Int4Weight.pack(codes, scale)), signed, codes, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(33, 40), (130, 6144)])
def test_rows_of_a_prompt_far_apart(cuda, m, n):
    """The largest row stride that the tiled product takes (its offsets have 32 bits), and one beyond."""
    k = 160
    codes, scale = make(n, k, 32, m)
    w = hk.Int4Weight.pack(codes, scale)
    for ldx in (1 << 23, (1 << 23) + 8):
        x = torch.empty((m - 1) * ldx + k, dtype=torch.float16, device=cuda).as_strided((m, k), (ldx, 1))
        x.copy_(normal(m, m, k))
        check(hk.int4_linear(x, w), x.contiguous(), codes, scale)
