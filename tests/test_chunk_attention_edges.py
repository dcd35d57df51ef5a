"""chunk_attention where its definition is easy to miss: windows of sequences that are longer than
their table, one key far above very many others, the bound of the workspace."""
import math

import pytest
import torch

from helm_amd import _native
from helm_amd.kernels import attention as ka
from test_chunk_attention import Batch


# ── windows and tables ───────────────────────────────────────────────────────

@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(79, 0), (80, 0), (81, 3), (100, 0), (119, 1), (120, 0), (10 ** 9, 5),
                                          (2 ** 31 - 1, 0), (2 ** 40, 0)])
@pytest.mark.parametrize("seqs", [[(100, 20), (100, 1)], [(120, 1), (70, 1), (79, 1), (85, 1)]])
def test_a_window_as_long_as_the_table_hides_keys_of_longer_sequences(seqs, window, sinks):
    """The table ends at token 80, the rows stand behind it: a row at p sees the keys from p - window + 1
    to 79 (equal scores and values of +-1: every key too many or too few shows)."""
    b = Batch((8, 2, 64), 16, seqs, window, sinks, flat=True, spare=0).cuda()
    table = b.d_table[:, :5].contiguous()
    out = torch.full_like(b.d_q, 7.0)
    ka.chunk_attention(b.d_q, b.pool, table, b.d_lens, b.d_starts, 16, window, sinks, out=out)
    b.check(out.cpu(), b.exact(coverage=80))
    if all(k == 1 for _, k in seqs):
        out = ka.window_decode_attention(b.d_q, b.pool, table, b.d_lens, 16, window, sinks)
        b.check(out.cpu(), b.exact(coverage=80))


@pytest.mark.gpu
def test_windows_past_2_to_the_30():
    """No position passes 2^31 - 2: from 2^31 - 1 on a window is none.  Below, up to 2^30 are supported."""
    b = Batch((4, 2, 64), 16, [(5, 2), (0, 1)], flat=True).cuda()
    for window in (2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 63):
        b.window = window
        b.check(b.run(), b.exact())
    for window in (2 ** 30 + 1, 2 ** 31 - 2):
        b.window = window
        with pytest.raises(RuntimeError, match="2\\^30"):
            b.run()


# ── one key far above very many others ───────────────────────────────────────

def peaked(heads, batch, new, n, nats, at, page=64):
    """`batch` sequences of n + 1 tokens over two slots: the key at `at` scores `nats` (a whole number of
    2^-6) and has values of -1, all others score 0 and have values of +1.  The calls' arguments, and
    what each of the `new` rows gives."""
    hq, hkv, d = heads
    k = torch.zeros(2, hkv, page, d, dtype=torch.float16, device="cuda")
    v = ka.alloc_v((2, hkv, page, d), device="cuda")
    v.fill_(1.0)
    k[0, :, at % page, 0] = nats
    v[0, :, at % page] = -1.0
    table = torch.ones(batch, -(-(n + 1) // page), dtype=torch.int32, device="cuda")
    table[:, at // page] = 0
    q = torch.randn(batch * new, hq, d, generator=torch.Generator().manual_seed(0)).half().cuda()
    q[..., 0] = 1.0
    lens = torch.full((batch,), n + 1, dtype=torch.int32, device="cuda")
    starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * new
    p = torch.arange(n + 1 - new, n + 1, dtype=torch.float64)          # others that a row sees
    tail = p * math.exp(-nats)
    return (q, ka.PoolView.of_pool(k, v), table, lens, starts, page), (tail - 1) / (tail + 1), tail / (tail + 1)


# (n, nats): the others' share of the weight, their single weights from 2^-21 to 2^-25.2
PEAKS = [(16384, 14.5), (131072, 15.0), (131072, 17.5), (262144, 16.265625)]


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(8, 8, 64), (8, 8, 128)])
@pytest.mark.parametrize("n,nats", PEAKS)
def test_many_rows_with_one_key_far_above_the_others(heads, n, nats):
    """A weight w of the largest is off by 2^-11 w or, where it is small, by 2^-32 (fp16 at 2^7 of it), in
    numerator and denominator alike: the output by 2^-11 sum w |v - o| <= 2^-11 4 tail, by 2 n 2^-32, by its
    own rounding and by 2^-16 of the exponents'.  And the sums are fp32: a matrix instruction adds eight products
    to a sum with one rounding to nearest, n keys are n / 8 of them, which one weight above all others
    makes alike.  With that weight as 1 a numerator within (-1, 0) is off by 2^-25 each time, a denominator
    within [1, 2) by 2^-24, the quotient by n (2^-28 + 2^-27) in all."""
    for batch, at in ((64, 0), (64, 20000), (64, n // 2 + 5), (1, 0)):   # whole, and in pieces
        at = min(at, n // 3)
        args, want, tail = peaked(heads, batch, 40, n, nats, at)
        got = ka.chunk_attention(*args, scale=1.0, max_new=40).cpu().double().view(batch, 40, -1)
        want, tail = want.view(1, 40, 1), tail.view(1, 40, 1)
        err = (got - want).abs()
        tol = 2.0 ** -11 * want.abs() + 2.0 ** -9 * tail + n * (2.0 ** -31 + 2.0 ** -28 + 2.0 ** -27) + 2.0 ** -16
        assert (err <= tol).all(), f"{batch} sequences, at {at}: off by {err.max().item():.2e}, {tol.min().item():.2e} allowed"


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(8, 8, 64), (8, 8, 128), (160, 8, 64)])
@pytest.mark.parametrize("n,nats", PEAKS)
def test_few_rows_with_one_key_far_above_the_others(heads, n, nats):
    """In the product a weight w of the largest is off by 2^-22 w or, where it is small, by 2^-32 (two
    fp16 parts at 2^7 of it), in the sum of the weights by nothing: the output by n 2^-32, by 2^-22, by its own
    rounding and by 2^-16 of the exponents'.  And the sums are fp32: a wave adds a quarter of the keys, eight at a
    time in two parts, n / 16 roundings of 2^-25 of the largest weight as above; its denominators, a lane's 8
    keys of 32 at a time, n / 128 of 2^-24."""
    for batch, at in ((64, 0), (64, 20000), (1, 0)):
        at = min(at, n // 3)
        args, want, _ = peaked(heads, batch, 1, n, nats, at)
        got = ka.window_decode_attention(*args[:4], args[5], 0, scale=1.0).cpu().double().view(batch, -1)
        err = (got - want).abs()
        tol = 2.0 ** -11 * want.abs() + n * (2.0 ** -32 + 2.0 ** -29 + 2.0 ** -31) + 2.0 ** -22 + 2.0 ** -16
        assert (err <= tol).all(), f"{batch} sequences, at {at}: off by {err.max().item():.2e}, {tol.min().item():.2e} allowed"


# ── workspace ────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,N,B,hq,hkv,pages,new,window,sinks", [
    # (rows of a partial in each form that the call can run)
    ((16,), 1, 1, 32, 8, 1024, 1, 4096, 4), ((16,), 300, 300, 16, 1, 900, 1, 0, 0), ((16,), 64, 64, 8, 8, 4096, 1, 0, 0),
    ((16,), 9, 3, 5, 1, 77, 3, 0, 0), ((32,), 20, 4, 32, 8, 200, 5, 0, 0), ((32,), 40, 40, 40, 2, 333, 1, 2000, 0),
    ((128,), 4096, 1, 40, 8, 1024, 4096, 0, 0), ((128,), 64, 2, 64, 1, 100, 60, 0, 0), ((128,), 7, 7, 34, 1, 640, 1, 0, 0),
    ((16, 128), 700, 25, 40, 8, 512, 700, 0, 0), ((32, 128), 600, 9, 40, 2, 512, 300, 0, 0),
    ((16, 128), 9000, 3, 32, 32, 990, 9000, 3000, 9), ((16, 128), 800, 3, 2048, 1024, 100, 700, 0, 0)])
def test_workspace_of_each_form(rows, N, B, hq, hkv, pages, new, window, sinks, d):
    """Partials of at most 512 / Hkv pieces a kv head and two more, of as many rows as the form's tiles,
    D values and two numbers each, whatever the lengths; nothing where no sequence can have two pieces."""
    f = _native.lib().helm_chunk_attn_workspace_bytes
    pieces = hkv * (max(512 // hkv, 1) + 2)
    bound = sum(pieces * r * (d + 2) * 4 for r in rows)
    assert 0 < f(N, B, hq, hkv, d, 16, pages, new, window, sinks) <= bound
    assert f(N, B, hq, hkv, d, 16, 8, new, window, sinks) == 0              # 128 tokens
