"""Captured blocks over packed rows with packed texts, replayed with other lengths of rows and texts."""

import pytest
import torch

from test_gpu_packed_block import DIM, _setup

pytestmark = pytest.mark.gpu


def test_replays_with_other_rows_and_texts(pkg, dev):
    """In the form with one self-attention launch for all requests every length is read on the GPU: ids, positions, offsets and texts' offsets
    that are changed together give what an eager call with those lengths gives."""
    ws, packed, pos, h, temb, _ = _setup(pkg, dev)
    h = torch.nan_to_num(h)  # (rows of no request become a request's)
    g = torch.Generator(device=dev).manual_seed(8)
    ctx = torch.randn(200, DIM, device=dev, generator=g).to(torch.bfloat16)
    text = pkg.PackedRequests.from_lengths([20, 33, 7, 59], 200, dev)

    def call(packed, pos, text):
        return pkg.packed_dit_forward(ws, h, temb, packed, pos, [pkg.project_packed_cross_kv(w, ctx, text) for w in ws])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(packed, pos, text)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(packed, pos, text)
    rows = packed.rows
    for lens, texts in (([48, 70, 1, 300], [20, 33, 7, 59]), ([1, 2, 3, 4], [0, 200, 0, 0]), ([rows, 0, 0, 0], [50, 50, 50, 50]), ([0, 100, 250, 60], [1, 0, 150, 3])):
        assert sum(lens) <= rows
        other = pkg.PackedRequests.from_lengths(lens, rows, dev)
        other_text = pkg.PackedRequests.from_lengths(texts, 200, dev)
        other_pos = torch.randint(0, 40, (rows, 3), generator=torch.Generator().manual_seed(lens[0])).to(torch.int32).to(dev)
        for mine, theirs in ((packed.request_ids, other.request_ids), (packed.offsets, other.offsets), (text.offsets, other_text.offsets), (pos, other_pos)):
            mine.copy_(theirs)
        graph.replay()
        torch.cuda.synchronize()
        want = call(other, other_pos, other_text)
        torch.cuda.synchronize()
        assert torch.isfinite(want).all() and torch.equal(got, want), lens
        assert not want[sum(lens):].any()
