"""Sampling: refusals on the CPU, drawn tokens on the GPU against the definition in extended
precision.  Tokens are whole numbers and have to be equal; the inputs are drawn so that no
border lies within 1e-9 of a random number (checked)."""
import ctypes

import numpy as np
import pytest
import torch

from helm_amd import _native
from helm_amd.kernels import fused


def definition(row, u, t, k, p, lo):
    """(token, distance of the nearest border that decides it, relative to the mass)"""
    x = row.astype(np.longdouble)
    n = len(x)
    if not t > 0:
        return int(np.argmax(np.where(np.isnan(row), np.inf, row))) if not np.isnan(row).any() else int(
            np.flatnonzero(np.isnan(row))[0]), 1.0
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return 0, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, np.longdouble(1), np.exp((x - top) / np.longdouble(np.float32(t))))
    order = np.lexsort((np.arange(n), -x))
    order = order[x[order] > -np.inf]
    near = 1.0
    if k > 0:
        order = order[:k]
    if np.float32(p) < 1:
        mass = np.cumsum(w[order])
        target = np.longdouble(np.float32(p)) * mass[-1]
        order = order[:max(1, 1 + int(np.count_nonzero(mass[:-1] < target)))]
        d = np.abs(mass[:-1] - target) / mass[-1]
        near = min(near, float(d[d > 0].min()) if (d > 0).any() else 1.0)
    keep = order[(w[order] >= np.longdouble(np.float32(lo))) | (order == order[0])]
    keep = np.sort(keep)
    mass = np.cumsum(w[keep])
    target = np.longdouble(np.float32(u)) * mass[-1]
    i = int(np.searchsorted(mass, target, side="right"))
    i = min(i, len(keep) - 1)
    while w[keep[i]] == 0:
        i -= 1
    return int(keep[i]), min(near, float(np.abs(mass - target).min() / mass[-1]))


def run(x, u, t, k, p, lo, **kw):
    def dev(v, dtype):
        return torch.tensor(np.asarray(v), dtype=dtype, device="cuda") if np.ndim(v) else v
    y = fused.sample(x, torch.tensor(u, dtype=torch.float32, device="cuda"), dev(t, torch.float32), dev(k, torch.int32),
                     dev(p, torch.float32), dev(lo, torch.float32), **kw)
    return y.cpu().numpy()


def check(x, u, t, k, p, lo, exact_ties=False):
    got = run(x, u, t, k, p, lo)
    rows = x.cpu().numpy()
    for i in range(len(rows)):
        pick = [v[i] if np.ndim(v) else v for v in (t, k, p, lo)]
        want, near = definition(rows[i], u[i], *pick)
        assert near > 1e-12 or exact_ties, "a border next to the random number: take another seed"
        assert got[i] == want, (i, int(got[i]), want, near, pick, u[i])


def logits(m, n, seed, std=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, n, generator=g) * std).half().cuda()


def test_refusals():
    assert fused.sample_workspace(3, 5000, "cpu").numel() == _native.lib().helm_sample_workspace_bytes(3, 5000) > 0
    with pytest.raises(RuntimeError, match="on the GPU"):
        fused.sample(torch.zeros(1, 8).half(), torch.zeros(1))
    lib = _native.lib()
    fake = ctypes.c_void_p(16)

    def call(x=fake, ldx=8, m=1, n=8, ws=fake, ws_bytes=1 << 20, u=fake):
        return lib.helm_sample(x, ldx, m, n, u, None, None, None, None, 1.0, 0, 1.0, 0.0, fake, ws, ws_bytes, None)
    assert call(x=None) == -1 and call(u=None) == -1 and call(m=0) == -1 and call(ldx=7) == -1
    assert call(ws=None) == -1 and call(ws_bytes=100) == -1 and call(ws=ctypes.c_void_p(24)) == -1
    assert call(n=1 << 23, ldx=1 << 23) == -2 and call(m=70000) == -2
    assert lib.helm_sample_workspace_bytes(0, 5) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 7, 63, 1000, 4096, 4097, 32000, 50257, 151936])
def test_against_the_definition(cuda, n):
    m = 12
    x = logits(m, n, n)
    r = np.random.default_rng(n)
    t = r.choice(np.float32([0.0, 0.2, 0.7, 1.0, 1.7]), m)
    k = r.choice([0, 0, 1, 3, 20, 500, n, 10 * n], m)
    p = r.choice(np.float32([1.0, 1.0, 0.05, 0.5, 0.9, 0.99]), m)
    lo = r.choice(np.float32([0.0, 0.0, 0.01, 0.2]), m)
    check(x, r.random(m, dtype=np.float32), t, k, p, lo)


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,p,lo", [(1.0, 0, 1.0, 0.0), (0.6, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05),
                                      (0.9, 40, 0.7, 0.02), (5.0, 100000, 0.999, 0.0), (0.01, 0, 1.0, 0.0)])
def test_numbers_for_all_rows(cuda, t, k, p, lo):
    x = logits(20, 50000, 5)
    check(x, np.random.default_rng(1).random(20, dtype=np.float32), t, k, p, lo)


@pytest.mark.gpu
def test_ties_go_to_the_lowest_index(cuda):
    n = 20000
    x = torch.zeros(6, n, dtype=torch.float16, device=cuda)
    x[3:, ::3] = 2.0
    u = np.float32([0.0, 0.5, 0.999, 0.0, 0.5, 0.999])
    for k, p in ((0, 1.0), (100, 1.0), (7000, 1.0), (0, 0.25), (5000, 0.5), (1, 0.5)):
        check(x, u, 1.0, k, p, 0.0, exact_ties=True)
    x[:, 5] = -0.0                                       # equals 0
    check(x, u, 1.0, 6, 1.0, 0.0, exact_ties=True)


@pytest.mark.gpu
def test_masked_infinite_and_nan_logits(cuda):
    x = logits(9, 9000, 3)
    x[0] = float("-inf")
    x[1] = float("-inf")
    x[1, 8999] = -5.0
    x[2, 100:] = float("-inf")
    x[3, ::2] = float("nan")
    x[4, 70], x[4, 4500], x[4, 8999] = float("inf"), float("inf"), float("inf")
    x[5] = float("nan")
    x[6, 4096:8192] = float("-inf")                      # a slice with nothing in it
    x[7] = -65504.0
    x[8] = 65504.0
    u = np.random.default_rng(4).random(9, dtype=np.float32)
    for k, p, lo in ((0, 1.0, 0.0), (50, 0.9, 0.0), (0, 0.8, 0.1), (0, 1.0, 1.0), (0, 0.0, 0.0), (0, 1.0, 3.0)):
        check(x, u, 1.0, k, p, lo, exact_ties=True)
    assert run(x, u, 0.0, 0, 1.0, 0.0).tolist() == fused.argmax(x).tolist()


@pytest.mark.gpu
def test_random_numbers_at_and_past_their_ends(cuda):
    x = logits(5, 6000, 8)
    last = run(x, [1.0 - 2.0 ** -24] * 5, 1.0, 40, 1.0, 0.0)
    assert (run(x, [1.0, 2.0, float("inf"), 1.0, 1.0], 1.0, 40, 1.0, 0.0) == last).all()
    first = run(x, [0.0] * 5, 1.0, 40, 1.0, 0.0)
    assert (run(x, [-1.0, 0.0, float("nan"), -0.0, -float("inf")], 1.0, 40, 1.0, 0.0) == first).all()
    top = torch.topk(x.float(), 40, -1).indices.cpu().numpy()
    assert (first == top.min(-1)).all() and (last == top.max(-1)).all()


@pytest.mark.gpu
def test_frequencies_follow_the_weights(cuda):
    """20000 evenly spread random numbers for one row: a token is drawn as often as its share says,
    off by at most one at either end of its interval."""
    m, n = 20000, 300
    row = logits(1, n, 11, 1.5)
    u = (np.arange(m) + 0.5).astype(np.float32) / m
    got = np.bincount(run(row.expand(m, n), u, 0.8, 100, 0.95, 0.0), minlength=n)
    w = np.exp((row[0].cpu().numpy().astype(np.float64) - float(row.max())) / np.float32(0.8))
    order = np.argsort(-w, kind="stable")[:100]
    mass = np.cumsum(w[order])
    order = order[:1 + np.count_nonzero(mass[:-1] < np.float32(0.95) * mass[-1])]
    share = np.zeros(n)
    share[order] = w[order] / w[order].sum()
    assert (np.abs(got - m * share) <= 1.001).all()


@pytest.mark.gpu
def test_strides_shapes_and_refusals(cuda):
    wide = logits(6, 5011, 9)
    x = wide[:, 3:5003]
    u = torch.rand(6, generator=torch.Generator().manual_seed(0)).cuda()
    want = fused.sample(x.contiguous(), u, 0.8, 50, 0.9)
    assert torch.equal(fused.sample(x, u, 0.8, 50, 0.9), want)
    assert torch.equal(fused.sample(x.contiguous().view(2, 3, 5000), u.view(2, 3), 0.8, 50, 0.9), want.view(2, 3))
    assert torch.equal(fused.sample(x.t().contiguous().t(), u, 0.8, 50, 0.9), want)
    out = torch.empty(6, dtype=torch.int64, device=cuda)
    ws = fused.sample_workspace(6, 5000, cuda)
    ws.fill_(255)
    assert fused.sample(x, u, 0.8, 50, 0.9, out=out, workspace=ws) is out and torch.equal(out, want)
    assert fused.sample(x[:0], u[:0]).shape == (0,)
    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=float("nan")), dict(min_p=-0.1), dict(out=u),
                dict(workspace=ws[:100]), dict(top_k=torch.zeros(6, device=cuda)), dict(temperature=torch.ones(5, device=cuda))):
        with pytest.raises(RuntimeError):
            fused.sample(x, u, **bad)
    with pytest.raises(RuntimeError, match="u must be"):
        fused.sample(x, u[:5])
    with pytest.raises(RuntimeError, match="fp16"):
        fused.sample(x.float(), u)


@pytest.mark.gpu
def test_captured_graph_replays(cuda):
    xs = [logits(4, 32000, s) for s in range(3)]
    us = [torch.rand(4, generator=torch.Generator().manual_seed(s)).cuda() for s in range(3)]
    eager = [fused.sample(x, u, 0.9, 100, 0.95, 0.01) for x, u in zip(xs, us)]
    x, u = xs[0].clone(), us[0].clone()
    ws = fused.sample_workspace(4, 32000, cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fused.sample(x, u, 0.9, 100, 0.95, 0.01, workspace=ws)
    for i in (1, 2, 0, 1, 1):
        x.copy_(xs[i])
        u.copy_(us[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[i])


@pytest.mark.gpu
@pytest.mark.parametrize("k,p,lo", [(0, 0.999, 0.0), (40000, 1.0, 0.0), (50000, 0.99, 0.001)])
def test_a_full_slice_without_the_border_s_chunk(cuda, k, p, lo):
    """Slices of 4096 logits of which the last holds only numbers above the border's range."""
    n = 17 * 4096
    x = logits(3, n, 21).clamp_(-7.5, 7.5)
    x[:, 16 * 4096:] = (8.0 + torch.rand(4096, generator=torch.Generator().manual_seed(3)) * 0.5).half().cuda()
    check(x, np.array([0.1, 0.9, 0.9995], np.float32), 2.0, k, p, lo)


@pytest.mark.gpu
def test_the_largest_rows(cuda):
    n = 64 * 4096
    x = logits(4, n, 31)
    x[3] = 0.5                                           # ties alone
    check(x, np.float32([0.3, 0.999, 0.5, 0.25]), np.float32([1.0, 0.7, 1.5, 1.0]), [0, 64, 70000, 5000],
          np.float32([0.95, 1.0, 0.999, 1.0]), np.float32([0.0, 0.0, 0.001, 0.5]), exact_ties=True)
    with pytest.raises(RuntimeError, match="262144"):
        fused.sample(logits(1, n + 1, 3), torch.zeros(1, device=cuda))
