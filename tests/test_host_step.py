"""The host's part of a step of many requests and of forks, with the launches left out: no GPU is touched."""

import time

import pytest
import torch

from falcon_perception_amd import ops
from falcon_perception_amd.paged_attention import PagedKVCache


@pytest.fixture
def launches(monkeypatch):
    """The calls that would be launches, with their arguments."""
    seen = []
    monkeypatch.setattr(ops.N, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    class Made:
        copy_src = copy_dst = copy_rows = None

    def step_tables(*args, **kw):
        seen.append(("step_tables", args, kw))
        return Made

    monkeypatch.setattr(ops, "step_tables", step_tables)
    monkeypatch.setattr(ops, "copy_pages", lambda *args: seen.append(("copy_pages", args, {})))
    return seen


def cache_of(slots, n_pages, P=16, columns=None, **kw):
    return PagedKVCache(n_pages, P, slots, 1, 64, 1, torch.bfloat16, device="cpu", max_blocks_per_seq=columns, **kw)


def test_pages_lie_where_the_kernel_looks_for_them(launches):
    """Request b's block have + i is entry count - off_b - need_b + i of the list, off_b the pages of the requests before; pages that were
    reserved ahead of the step are among them."""
    cache = cache_of(6, 60, columns=30)
    slots = [cache.allocate() for _ in range(4)]
    cache.reserve(slots[2], None, 70)
    old = [0, 0, 0, 0]
    for new in ([40, 0, 20, 33], [48, 1, 100, 33], [49, 90, 101, 90]):
        cache.step_tables(slots, old, new)
        (ids, before, after, free, count, table, P, rows), kw = launches[-1][1:]
        assert ids.tolist() == slots and before.tolist() == old and after.tolist() == new and rows == sum(new) - sum(old)
        assert count.tolist() == [len(free)]
        off = 0
        for s, o, n in zip(slots, old, new):
            have, need = -(-o // P), -(-n // P) - -(-o // P)
            assert free[len(free) - off - need:len(free) - off].tolist() == cache.page_table_cpu[s][have:have + need]
            off += need
        assert off == len(free)
        old = new


def test_the_time_of_a_step_grows_with_its_requests(launches):
    """Eight times the requests take no more than 24 times as long: 8 where the time is linear, 64 where it grows with the square."""

    def seconds(B):
        best = 1e9
        for _ in range(3):
            cache = cache_of(B + 1, 16 * B + 1, P=1, columns=16)
            slots = [cache.allocate() for _ in range(B)]
            t = time.perf_counter()
            cache.step_tables(slots, [0] * B, [16] * B)
            best = min(best, time.perf_counter() - t)
        return best

    seconds(64)
    assert seconds(4096) < 24 * seconds(512)


def test_a_step_inside_a_capture_changes_nothing(launches, monkeypatch):
    cache = cache_of(8, 60, columns=30, prefix_sharing=True)
    slot = cache.allocate()
    cache.reserve(slot, None, 40)
    state = lambda: ([list(x) for x in cache.page_table_cpu], list(cache.free_pages), list(cache.free_batch_idx), list(cache.capacity),
                     dict(cache._prefixes), dict(cache._page_slots), cache.page_table.tolist())
    before = state()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: cache.fork(slot, 40, 2), lambda: cache.fork(slot, 32), lambda: cache.step_tables([slot], [40], [50])):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            call()
        assert state() == before and not launches
