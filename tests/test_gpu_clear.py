"""dg_clear and the cleared state that the loss head's counters start from, in recorded steps too."""
import os
import re

import pytest
import torch

from diffgraph_amd import _lib, ops

gpu = pytest.mark.gpu
DEV = "cuda"
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "diffgraph_amd", "csrc")


def test_no_entry_point_records_a_memset_node():
    """A memset on a caller's stream becomes a memset node where the caller records; counters that are not cleared on a
    replay are indexes that nothing bounds.  The kernels' sources clear by kernels alone."""
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".hip", ".h")):
            text = open(os.path.join(CSRC, name)).read()
            assert not re.search(r"hipMemset\w*Async\s*\(", text), name


def _clear(t, begin, count):
    _lib.check(_lib.load().dg_clear(t.data_ptr() + begin, count, _lib.stream_ptr(t.device)), "dg_clear")


@gpu
@pytest.mark.parametrize("begin", [0, 1, 15, 16, 37])
@pytest.mark.parametrize("count", [0, 1, 3, 15, 16, 17, 63, 4096, 100003, 40000001])
def test_clear_takes_its_bytes_and_no_others(begin, count):
    t = torch.full((begin + count + 64,), 7, dtype=torch.uint8, device=DEV)
    _clear(t, begin, count)
    assert not bool(t[begin: begin + count].any())
    assert bool((t[:begin] == 7).all()) and bool((t[begin + count:] == 7).all())


@gpu
def test_every_replay_clears_and_lists_the_rows_anew():
    """Recorded: the clear of a buffer and the rows a batch names.  Between the replays the memory is filled with what the
    words must not keep (negative numbers among them), the batch changes, and other work runs eagerly."""
    nu, ni, B = 500, 700, 300
    g = torch.Generator().manual_seed(3)
    draw = lambda hi: torch.randint(0, hi, (B,), generator=g)  # noqa: E731
    ancs, poss, negs = draw(nu).to(DEV), draw(ni).to(DEV), draw(ni).to(DEV)
    buf = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    act = ops.active_rows_buffers(B, nu + ni, DEV)

    def step():
        _clear(buf, 0, buf.numel())
        ops.active_rows(ancs, poss, negs, nu, ni, out=act)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(6):
        a, p, n = draw(nu), draw(ni), draw(ni)
        ancs.copy_(a), poss.copy_(p), negs.copy_(n)
        buf.fill_(0xF0 + k)
        act[0].fill_(-5 - k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert not bool(buf.any())
        users, items = torch.unique(a), torch.unique(torch.cat([p, n]))
        assert act[3].tolist() == [users.numel(), items.numel()]
        assert torch.equal(act[1][: users.numel()].cpu().long(), users) and torch.equal(act[2][: items.numel()].cpu().long(), items)
        assert torch.equal(act[0].cpu() != 0, torch.zeros(nu + ni, dtype=torch.bool).index_fill_(0, torch.cat([users, nu + items]), True))
