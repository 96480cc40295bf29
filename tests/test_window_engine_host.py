"""Host side of the engine's attention window (no GPU): what a request reserves, and the pages it gives back."""
import random

import pytest

from redline_llm_b200.engine import DUMMY_BLOCK, KV_BLOCK, BlockAllocator, Request, Scheduler, blocks_for_tokens


def drive(s, steps=100000):
    """Runs the scheduler as the engine does - prompt chunks, decode steps, trim after each - and checks at every query that
    the pages it sees are held."""
    most, done = 0, 0
    for _ in range(steps):
        plan = s.plan_step()
        if plan[0] == "idle":
            return most, done
        if plan[0] == "flush":
            for r in plan[1]:
                s.release(r)
            continue
        rows = []
        if plan[0] == "prefill":
            _, r, a, b = plan
            rows = [(r, p) for p in (a, b - 1)]
            r.prefilled = b
        else:
            rows = [(r, r.cached) for r in plan[1]]
        for r, p in rows:                        # a query at position p sees the sinks and the window up to p
            for t in list(range(min(s.sinks, p + 1))) + list(range(max(0, p - s.window + 1), p + 1)):
                assert r.blocks[t // KV_BLOCK] != DUMMY_BLOCK, (p, t)
        most = max(most, sum(1 for r in s.running for b in r.blocks if b != DUMMY_BLOCK))
        held = [b for r in s.running for b in r.blocks if b != DUMMY_BLOCK]
        assert len(held) == len(set(held)), "a page belongs to two requests"
        assert s.alloc.reserved <= s.alloc.free_blocks
        if plan[0] == "prefill":
            s.trim(r, b)
            if b == len(r.prompt):
                r.cached = b
                done += s.complete(r, 1)[2]
        else:
            for r in list(plan[1]):
                r.cached += 1
                done += s.complete(r, 1)[2]
                if not r.finished:
                    s.trim(r, r.cached)
    raise AssertionError("did not finish")


@pytest.mark.parametrize("window,sinks,chunk", [(1, 0, 16), (16, 4, 32), (40, 17, 7), (100, 0, 64), (64, 64, 100), (5000, 3, 128)])
def test_a_request_holds_what_its_window_needs_and_returns_everything(window, sinks, chunk):
    rnd = random.Random(window)
    total = 400
    a = BlockAllocator(total)
    s = Scheduler(a, max_batch=4, max_seq_len=4096, prefill_chunk=chunk, window=window, sinks=sinks)
    for i in range(12):
        s.enqueue(Request(i, [1] * rnd.randint(1, 900), rnd.randint(1, 300), ignore_eos=True))
    most, done = drive(s)
    assert done == 12 and s.aborts == 0
    assert a.free_blocks == total - 1 and a.reserved == 0
    assert most <= 4 * s.held_blocks()


def test_a_long_request_fits_a_small_pool_only_with_a_window():
    for window, aborted in ((0, 1), (64, 0)):
        a = BlockAllocator(20)
        s = Scheduler(a, max_batch=1, max_seq_len=4096, prefill_chunk=32, window=window, sinks=4 if window else 0)
        s.enqueue(Request(0, [1] * 600, 500, ignore_eos=True))
        if window:
            assert s.held_blocks() < blocks_for_tokens(1100)
            assert drive(s)[1] == 1
        else:
            assert s.plan_step()[0] == "flush"
            s.release(s.running[0])
        assert s.aborts == aborted and a.free_blocks == 19 and a.reserved == 0


def test_without_a_window_nothing_is_trimmed():
    a = BlockAllocator(20)
    s = Scheduler(a, 1, 4096, 32)
    r = Request(0, [1] * 100, 10)
    s.enqueue(r)
    s.plan_step()
    before = list(r.blocks)
    s.trim(r, 1000)
    assert r.blocks == before and s.held_blocks() > 1 << 20


def test_the_host_work_of_a_decode_step_does_not_grow_with_the_context():
    """trim() runs after every decode step of every request: over a whole request it looks at each page a fixed number of
    times, however long the list of pages has become."""
    class Counted(list):
        looks = 0

        def __iter__(self):
            for x in list.__iter__(self):
                Counted.looks += 1
                yield x

        def __getitem__(self, k):
            Counted.looks += 1
            return list.__getitem__(self, k)

    a = BlockAllocator(60)
    s = Scheduler(a, 1, 1 << 20, 32, window=64, sinks=20)
    r = Request(0, [1] * 32, 8000, ignore_eos=True)
    s.enqueue(r)
    s.plan_step()
    r.blocks = Counted(r.blocks)
    r.prefilled = r.cached = 32
    s.trim(r, 32)
    for _ in range(6000):
        assert s.plan_step()[0] == "decode"
        r.cached += 1
        s.trim(r, r.cached)
        held = [b for b in list.__iter__(r.blocks) if b != DUMMY_BLOCK]
        assert len(held) <= s.held_blocks()
        assert r.reserved_left + len(held) <= r.need
    assert Counted.looks <= 4 * len(r.blocks), f"{Counted.looks} looks at {len(r.blocks)} pages"
    s.release(r)
    assert a.free_blocks == 59 and a.reserved == 0
