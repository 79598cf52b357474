"""PackedRequests as a value: three fields as ever for callers that take it apart by position, the offsets beside them."""

import copy
import pickle

import torch


def test_three_fields_by_position(pkg):
    p = pkg.PackedRequests.from_lengths([2, 0, 3], 7, "cpu")
    lengths, rows, ids = p
    assert lengths == (2, 0, 3) and rows == 7 and ids is p.request_ids and len(p) == 3
    assert p[2] is p.request_ids and p[-1] is p.request_ids and tuple(p)[:2] == ((2, 0, 3), 7)
    assert p._fields == ("lengths", "rows", "request_ids") and list(p._asdict()) == list(p._fields)
    again = pkg.PackedRequests(*p)
    assert again.offsets is None and again.rows == 7 and list(again.spans()) == [(0, 2), (2, 2), (2, 5)]
    match p:
        case (_, n, _):
            assert n == 7


def test_offsets_go_along(pkg):
    p = pkg.PackedRequests.from_lengths([2, 0, 3], 7, "cpu")
    assert p.offsets.tolist() == [0, 2, 2, 5] and p.offsets.dtype == torch.int32
    for other in (copy.copy(p), copy.deepcopy(p), pickle.loads(pickle.dumps(p))):
        assert type(other) is pkg.PackedRequests and other.offsets.tolist() == [0, 2, 2, 5] and other.request_ids.tolist() == p.request_ids.tolist()
    assert p._replace(rows=9).offsets is p.offsets and p._replace(rows=9).rows == 9
    mine = torch.zeros(4, dtype=torch.int32)
    assert p._replace(offsets=mine).offsets is mine and p._replace(offsets=None).offsets is None and p.offsets.tolist() == [0, 2, 2, 5]
    # other lengths have other offsets: those of before would be wrong for them
    assert p._replace(lengths=(1, 1, 3)).offsets is None and p._replace(lengths=(1, 1, 3), offsets=mine).offsets is mine
    given = pkg.PackedRequests((2, 3), 5, p.request_ids[:5], mine)
    assert given.offsets is mine and pkg.PackedRequests((2, 3), 5, p.request_ids[:5], offsets=mine).offsets is mine
    assert pkg.PackedRequests._make([(2, 3), 5, p.request_ids]).offsets is None
