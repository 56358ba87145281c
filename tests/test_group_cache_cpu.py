"""The remembered groupings of pair-id tensors: a full memory gives up its oldest
entry, not the one the same call has just made."""

from __future__ import annotations

import torch

from maxsim_b200 import _ops


def test_a_full_memory_keeps_the_newest_groupings(monkeypatch):
    made = []
    monkeypatch.setattr(_ops, "group_pairs", lambda ids, n: made.append(ids) or object())
    monkeypatch.setattr(_ops, "_GROUP_CACHE", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ids = [torch.zeros(_ops.GROUP_MIN_PAIRS, dtype=torch.int32) for _ in range(3 * _ops._GROUP_CACHE_LIMIT)]
    alone = torch.zeros(_ops.GROUP_MIN_PAIRS, dtype=torch.int32)
    _ops._groups(alone, alone, 5)  # a forward pass groups by document only: the pairs below start at odd places
    for by_document, by_query in zip(ids[::2], ids[1::2]):
        first = _ops._groups(by_document, by_document, 5), _ops._groups(by_query, by_query, 5)
        # the second call of a pair finds both, whatever the memory held before
        assert (_ops._groups(by_document, by_document, 5), _ops._groups(by_query, by_query, 5)) == first
    assert len(made) == len(ids) + 1 and len(_ops._GROUP_CACHE) <= _ops._GROUP_CACHE_LIMIT
    by_query.add_(1)  # written: grouped again
    assert _ops._groups(by_query, by_query, 5) is not first[1]
