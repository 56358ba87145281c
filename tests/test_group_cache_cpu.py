"""The remembered groupings of pair-id tensors: a full memory gives up its oldest
entry, not the one the same call has just made."""

from __future__ import annotations

import threading

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


def test_two_threads_that_find_the_memory_full(monkeypatch):
    """Another thread's call arrives between the look for the oldest entry and its removal: neither
    call fails, both groupings are remembered."""
    other = []

    class Memory(dict):
        def __iter__(self):
            oldest = next(super().__iter__())
            if not other:  # once: the first thread has looked, the second comes in
                other.append(threading.Thread(target=group, args=(ids[-1],)))
                other[0].start()
                other[0].join(0.5)  # it may have to wait for this one
            return iter([oldest])

    failed = []

    def group(t):
        try:
            _ops._groups(t, t, 5)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    monkeypatch.setattr(_ops, "group_pairs", lambda ids, n: object())
    monkeypatch.setattr(_ops, "_GROUP_CACHE", Memory())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    limit = _ops._GROUP_CACHE_LIMIT
    ids = [torch.zeros(_ops.GROUP_MIN_PAIRS, dtype=torch.int32) for _ in range(limit + 2)]
    for t in ids[:limit]:
        group(t)
    assert not other
    group(ids[limit])
    other[0].join()
    assert not failed, failed
    assert len(_ops._GROUP_CACHE) == limit
    assert all(_ops._groups(t, t, 5, build=False) is not None for t in ids[limit:])
    _ops.forget_pair_groups()
    assert len(_ops._GROUP_CACHE) == 0


def test_many_threads_share_the_memory(monkeypatch):
    monkeypatch.setattr(_ops, "group_pairs", lambda ids, n: object())
    monkeypatch.setattr(_ops, "_GROUP_CACHE", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    failed = []

    def work():
        try:
            mine = [torch.zeros(_ops.GROUP_MIN_PAIRS, dtype=torch.int32) for _ in range(300)]
            for t in mine:
                first = _ops._groups(t, t, 5)
                again = _ops._groups(t, t, 5, build=False)  # forgotten, or the same
                assert again is None or again is first
            _ops.forget_pair_groups()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert len(_ops._GROUP_CACHE) <= _ops._GROUP_CACHE_LIMIT
