"""Blocks with several owners, forked sequences and compacted pools: the host side."""
import numpy as np
import pytest

from aicomp_amd.block_manager import BlockAllocator, OutOfBlocks, PlanError, StepPlanner, check_plan


def test_a_shared_block_is_free_when_its_last_owner_frees_it():
    a = BlockAllocator(6, 16)
    b = a.allocate(3)
    a.share(b[:2])
    a.share(b[:1])
    assert a.num_used == 3 and a.shared.tolist() == [True, True, False, False, False, False]
    a.free(b)
    assert a.num_used == 2 and a.shared.tolist() == [True, False, False, False, False, False]
    a.free(b[:2])
    assert a.num_used == 1 and not a.shared.any()
    a.free(b[:1])
    assert a.num_used == 0
    with pytest.raises(ValueError, match="double free"):
        a.free(b[:1])
    with pytest.raises(ValueError, match="not allocated"):
        a.share([0])
    with pytest.raises(ValueError, match="out of range"):
        a.share([6])
    a.share([])
    c = a.allocate(6)
    assert sorted(c.tolist()) == list(range(6))


def test_compaction_moves_to_the_low_end():
    a = BlockAllocator(10, 16)
    blocks = a.allocate(9)
    a.share([7])
    a.free([0, 2, 3, 5])
    pairs = a.compact()
    assert a.num_used == 5 and pairs.tolist() == [[6, 0], [7, 2], [8, 3]]
    assert np.flatnonzero(a._owned).tolist() == [0, 1, 2, 3, 4] and np.flatnonzero(a.shared).tolist() == [2]
    assert a.allocate(5).tolist() == [5, 6, 7, 8, 9]
    assert a.compact().shape == (0, 2)
    a.free([2])
    assert not a.shared.any() and a.num_used == 10
    assert blocks.size == 9


def planner(**kw):
    return StepPlanner(**{**dict(num_blocks=20, block_size=16, max_seqs=4, max_seq_len=256, max_num_batched_tokens=128,
                                 prefill_chunk=64, device="cpu", check_plans=True), **kw})


def test_forked_sequences_share_full_blocks_and_part_at_the_last():
    p = planner()
    p.add_request("a", 40, max_new_tokens=30)
    p.schedule()
    pairs = p.fork("a", "b")
    a, b = p.blocks_of("a"), p.blocks_of("b")
    assert a[:2] == b[:2] and a[2] != b[2] and pairs.tolist() == [[a[2], b[2]]] and pairs.dtype == np.int64
    assert p.context_len("b") == 40 and p.alloc.num_used == 4
    plan = p.schedule()                                   # both decode; the plan is checked with the shared blocks allowed
    assert sorted(plan.seq_ids) == ["a", "b"] and len(set(plan.host_slot_mapping.tolist())) == 2
    with pytest.raises(PlanError, match="share a block"):
        check_plan(plan, 20, 16)                          # nothing says that they may
    for _ in range(10):
        p.schedule()
    assert p.blocks_of("a")[:2] == p.blocks_of("b")[:2] and not set(p.blocks_of("a")[2:]) & set(p.blocks_of("b")[2:])
    p.finish("a")
    assert not p.alloc.shared.any() and p.alloc.num_used == len(p.blocks_of("b"))
    p.finish("b")
    assert p.alloc.num_used == 0


def test_a_fork_at_a_block_border_copies_nothing():
    p = planner()
    p.add_request("a", 32)
    p.schedule()
    assert p.fork("a", "b").shape == (0, 2) and p.alloc.num_used == 2
    plan = p.schedule()
    assert len(set((plan.host_slot_mapping // 16).tolist())) == 2       # each opened a block of its own


def test_a_fork_that_cannot_be_had_changes_nothing():
    p = planner(num_blocks=3)
    p.add_request("a", 40)
    with pytest.raises(ValueError, match="not running"):
        p.fork("a", "b")
    p.schedule()
    with pytest.raises(OutOfBlocks):
        p.fork("a", "b")
    assert p.num_running == 1 and not p.alloc.shared.any() and p.alloc.num_used == 3
    with pytest.raises(ValueError, match="already known"):
        p.fork("a", "a")
    q = planner(max_seqs=1)
    q.add_request("a", 40)
    q.schedule()
    with pytest.raises(ValueError, match="in use"):
        q.fork("a", "b")


def test_a_write_into_a_shared_block_is_found():
    p = planner(check_plans=False)
    p.add_request("a", 40)
    plan = p.schedule()
    mask = np.zeros(20, dtype=bool)
    mask[plan.host_slot_mapping[0] // 16] = True
    with pytest.raises(PlanError, match="other sequences share"):
        check_plan(plan, 20, 16, mask)


def test_compacted_tables_follow_their_blocks():
    p = planner()
    for s, n in (("a", 40), ("b", 60), ("c", 20)):
        p.add_request(s, n)
    p.schedule()
    p.fork("b", "d")
    p.finish("a")
    before = {s: p.blocks_of(s) for s in "bcd"}
    pairs = p.compact()
    move = dict(pairs.tolist())
    assert pairs.shape[0] > 0 and not set(move) & set(move.values())
    for s in "bcd":
        assert p.blocks_of(s) == [move.get(x, x) for x in before[s]]
    assert max(max(p.blocks_of(s)) for s in "bcd") == p.alloc.num_used - 1
    while p.schedule() is not None and p.context_len("b") < 100:       # plans are checked
        pass
    for s in "bcd":
        p.finish(s)
    assert p.alloc.num_used == 0


def test_preemption_leaves_shared_blocks_with_the_others():
    p = planner(num_blocks=5, check_plans=True)
    p.add_request("a", 40)
    p.schedule()
    p.fork("a", "b")                                       # 2 shared, 2 of their own, one free
    seen = []
    for _ in range(40):
        plan = p.schedule()
        seen += plan.preempted
        if seen:
            break
    assert seen == ["b"] and not p.alloc.shared.any()
    assert p.alloc.num_used == len(p.blocks_of("a"))
