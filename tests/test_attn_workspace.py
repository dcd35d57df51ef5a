"""One AttnWorkspace for fp16 and 8-bit decode attention: captured calls of either kind go on using the
buffer that they were captured with, whichever kind of call makes it grow."""
import gc
import weakref

import pytest
import torch

from helm_amd.kernels import attention as ka


@pytest.mark.parametrize("grow", [lambda ws: ws.get(4, 32, 128, 8), lambda ws: ws.reserve(-1, 1 << 20)])
@pytest.mark.parametrize("first", [lambda ws: ws.get(1, 8, 64, 2), lambda ws: ws.reserve(-1, 1000)])
def test_what_either_call_outgrows_stays(first, grow):
    ws = ka.AttnWorkspace(torch.device("cpu"))
    first(ws)
    held, address = weakref.ref(ws.buf), ws.buf.data_ptr()
    ws.buf.fill_(3.0)
    grow(ws)
    gc.collect()
    assert ws.buf.data_ptr() != address
    assert held() is not None and held().data_ptr() == address and (held() == 3.0).all()


def test_growth_is_twofold_at_least_and_get_splits_the_buffer():
    ws = ka.AttnWorkspace(torch.device("cpu"))
    o, ml = ws.get(2, 3, 64, 5)
    assert (o.numel(), ml.numel(), ws.buf.numel()) == (2 * 3 * 5 * 64, 2 * 3 * 5 * 2, 2 * 3 * 5 * 66)
    assert o.data_ptr() == ws.buf.data_ptr() and ml.data_ptr() == o.data_ptr() + 4 * o.numel()
    size = ws.buf.numel()
    ws.get(2, 3, 64, 6)
    assert ws.buf.numel() == 2 * size
    ws.reserve(-1, 8)
    ws.get(1, 1, 64, 1)
    assert ws.buf.numel() == 2 * size and len(ws._outgrown) == 2


def pools(seed):
    """An fp16 and an 8-bit pool of 64 pages, a table over all of them and q of one item."""
    g = torch.Generator().manual_seed(seed)
    k16 = torch.randn(64, 8, 16, 128, generator=g).half().cuda()
    v16 = ka.alloc_v((64, 8, 16, 128), dtype=torch.float16, device="cuda")
    v16.copy_(torch.randn(64, 8, 16, 128, generator=g).half())
    q8 = ka.alloc_q8_pool(64, 8, 16, 128, "cuda")
    table = torch.randperm(64, generator=g).int().view(1, 64).cuda()
    lens = torch.tensor([1000], dtype=torch.int32, device="cuda")
    slots = table.view(64, 1).expand(64, 16).reshape(-1).contiguous()
    ka.kv_append_q8(k16[table[0].long()].transpose(1, 2).reshape(-1, 8, 1, 128),
                    v16[table[0].long()].transpose(1, 2).reshape(-1, 8, 1, 128), q8, slots,
                    torch.arange(16, dtype=torch.int32, device="cuda").repeat(64))
    q = torch.randn(1, 32, 128, generator=g).half().cuda()
    return ka.PoolView.of_pool(k16, v16), q8, table, lens, q


@pytest.mark.gpu
@pytest.mark.parametrize("captured,growing", [(8, 16), (16, 8), (16, 16)])
def test_a_captured_call_outlives_growth_by_the_other_kind(cuda, captured, growing):
    p16, p8, table, lens, q = pools(3)
    ws = ka.AttnWorkspace(torch.device("cuda", 0))

    def call(bits, n, splits):
        args = (q.expand(n, 32, 128).contiguous(),), (table.expand(n, 64).contiguous(), lens.expand(n).contiguous())
        if bits == 8:
            return ka.paged_decode_attention_q8(*args[0], p8, *args[1], 16, num_splits=splits, workspace=ws)
        return ka.paged_decode_attention(*args[0], p16, *args[1], 16, num_splits=splits, workspace=ws)
    want = call(captured, 1, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(captured, 1, 8)
    for n in (3, 9):                                     # the workspace grows; others take what is free
        call(growing, n, 16)
        others = [torch.full((1 << 18,), float(n), device=cuda) for _ in range(8)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all((t == float(n)).all() for t in others)
