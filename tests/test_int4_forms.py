"""Every kernel of int4_linear at shapes that pick it (helm_int4_linear_form), against fp64 at a sample of
outputs; and the longest walks over row tiles.  A shape list that a refitted choice no longer covers fails."""
import ctypes

import pytest
import torch

from helm_amd import _native
from helm_amd import kernels as hk
from test_int4_rounding import check, normal

# rows a tile of the tiled product, sliced or not; tiles a wave of the GEMV by blocks of 16 tokens, sliced or not
FORMS = ({(0, rows, s, gs) for rows in (32, 64, 96, 128) for s in (False, True) for gs in (32, 64, 128)}
         | {(1, uw, s, gs) for gs, most in ((32, 2), (64, 3), (128, 4)) for uw in range(1, most + 1) for s in (False, True)}
         | {(2, uw, s, gs) for gs, most in ((32, 1), (64, 2), (128, 2)) for uw in range(1, most + 1) for s in (False, True)})
PROMPTS = ([(m, n, k, gs) for gs in (32, 64, 128) for m, n, k in ((33, 256, 128), (777, 4096, 128), (1500, 4096, 6144))]
           + [(150, 2000, 640, 32), (77, 2560, 1536, 32), (1500, 2560, 1280, 32), (199, 6144, 4096, 32), (777, 7168, 1536, 32),
              (777, 912, 17408, 32), (199, 25600, 128, 32), (777, 3008, 4096, 32), (100, 12288, 12800, 32)]
           + [(m, n, k, gs) for gs in (64, 128) for m, n, k in (
               (33, 6144, 384), (77, 1504, 2560), (333, 25600, 512), (777, 272, 6656), (100, 2000, 19968), (777, 6144, 1024),
               (2000, 272, 4096), (150, 5120, 10752), (2000, 6144, 1536), (1500, 1504, 4608))])
TOKENS = ([(m, n, k, gs) for gs in (32, 64, 128) for m, n, k in ((1, 256, 128), (5, 512, 2048), (1, 256, 4608), (16, 512, 12800),
                                                                 (17, 256, 128), (24, 2560, 384), (17, 256, 4608), (31, 912, 12288))]
          + [(1, 2560, 2176, 32), (16, 2000, 2176, 32), (1, 8192, 4608, 32), (5, 8192, 10752, 32), (31, 912, 10752, 32)]
          + [(m, n, k, gs) for gs in (64, 128) for m, n, k in (
              (5, 256, 4608), (16, 2000, 2176), (1, 3008, 12800), (5, 6144, 12800), (1, 4096, 10752), (16, 4096, 4608),
              (31, 2000, 2560), (17, 7168, 14848), (24, 10240, 14848))]
          + [(16, 10240, 6656, 64), (1, 1024, 25600, 64), (1, 2560, 6656, 128), (5, 8192, 6656, 128), (1, 10240, 12800, 128),
             (5, 12288, 12800, 128), (5, 6144, 17408, 128), (16, 5120, 17408, 128)])
# row tiles of a workgroup: 9 (three tiles a wave), 38, 64, and 64 from 257 workgroups
WALKS = [(1, 34816, 5120, 128), (16, 34816, 5120, 64), (1, 151936, 4736, 128), (16, 151936, 4096, 128), (1, 151936, 2048, 32),
         (32, 151936, 1024, 128), (1, 262144, 256, 128), (16, 262160, 256, 64), (24, 262160, 128, 32)]


def form(m, n, k, gs):
    f = (ctypes.c_int32 * 3)()
    _native.call("helm_int4_linear_form", m, n, k, gs, f)
    return f[0], f[1], f[2] > 1, gs


def test_the_shapes_cover_every_kernel():
    assert {form(*s) for s in PROMPTS} == {f for f in FORMS if f[0] == 0}
    assert {form(*s) for s in TOKENS} == {f for f in FORMS if f[0] > 0}


def test_form_agrees_with_the_workspace_and_refuses():
    f = (ctypes.c_int32 * 3)()
    for m, n, k, gs in PROMPTS + TOKENS + WALKS:
        _native.call("helm_int4_linear_form", m, n, k, gs, f)
        need = f[2] * m * -(-n // 16) * 16 * 4 if f[2] > 1 else 0
        assert _native.lib().helm_int4_linear_workspace_bytes(m, n, k, gs) == need
    lib = _native.lib()
    assert lib.helm_int4_linear_form(0, 16, 128, 64, f) == -1 and lib.helm_int4_linear_form(1, 16, 128, 64, None) == -1
    assert lib.helm_int4_linear_form(1, 16, 96, 64, f) == -2 and lib.helm_int4_linear_form(1, 16, 128, 48, f) == -2
    assert lib.helm_int4_linear_form(1, 1 << 28, 128, 64, f) == -2


def run(m, n, k, gs, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    nt, kt = n // 16, k // 128
    q = torch.randint(-2 ** 31, 2 ** 31 - 1, (nt, kt, 64, 4), generator=g, dtype=torch.int32, device="cuda")
    s = ((0.5 + torch.rand(nt, kt, 128 // gs, 16, generator=g, device="cuda")) * 0.006).half()
    x, bias = normal(seed + 1, m, k), normal(seed + 2, n) if m % 2 else None
    y = hk.int4_linear(x, hk.Int4Weight(q, s, n, k, gs), bias)
    # the first and last outputs and some between
    some = torch.randint(0, nt, (10,), generator=torch.Generator().manual_seed(seed))
    at = torch.unique(torch.cat([torch.arange(min(nt, 2)), torch.arange(max(nt - 2, 0), nt), some])).cuda()
    codes, scale = hk.Int4Weight(q[at], s[at], 16 * len(at), k, gs).unpack()
    cols = (at[:, None] * 16 + torch.arange(16, device="cuda")).flatten()
    check(y[:, cols], x, codes, scale, None if bias is None else bias[cols])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gs", PROMPTS)
def test_prompts(cuda, m, n, k, gs):
    run(m, n, k, gs, m + n + k)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gs", TOKENS)
def test_tokens(cuda, m, n, k, gs):
    run(m, n, k, gs, m + n + k)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gs", WALKS)
def test_long_walks(cuda, m, n, k, gs):
    run(m, n, k, gs, m + n + k)
