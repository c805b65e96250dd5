"""Prefixes whose rows all see each other, in steps of a planner: one chunk ingests them, and a step that has a part of one is refused
(the host side, without a GPU)."""
import numpy as np
import pytest
import torch

from aicomp_amd.block_manager import StepPlanner
from aicomp_amd.generation import PagedAttentionBackend


def planner(**kw):
    return StepPlanner(**{**dict(num_blocks=40, block_size=16, max_seqs=4, max_seq_len=256, max_num_batched_tokens=128,
                                 prefill_chunk=32, device="cpu", check_plans=True), **kw})


def backend():
    return PagedAttentionBackend(1, 40, 1, 16, dtype=torch.float32, device="cpu")


FORMS = [lambda x: x, lambda x: np.asarray(x, dtype=np.int32), lambda x: torch.tensor(x, dtype=torch.int32), lambda x: torch.tensor(x)]


@pytest.mark.parametrize("form", FORMS, ids=["list", "array", "int32", "int64"])
def test_a_step_with_a_part_of_a_prefix_is_refused(form):
    p, b = planner(), backend()
    p.add_request("a", 20)
    p.add_request("b", 100)
    plan = p.schedule()                                         # 20 and 32 tokens
    with pytest.raises(ValueError, match="'b'.*prefix of 33.*ends at 32"):
        b.begin_step(plan, prefix_lens=form([20, 33]))
    assert b.plan is None and b.prefix_lens is None             # nothing of the refused step stays
    b.begin_step(plan, prefix_lens=form([20, 32]))
    assert b.prefix_lens.dtype == torch.int32 and b.prefix_lens.tolist() == [20, 32]
    plan = p.schedule()                                         # the second chunk; "a" decodes
    assert sorted(zip(plan.seq_ids, plan.host_context_lens.tolist())) == [("a", 21), ("b", 64)]
    b.begin_step(plan, prefix_lens=form([32 if s == "b" else 20 for s in plan.seq_ids]))
    with pytest.raises(ValueError, match="prefix of 22"):       # a row of one token too
        b.begin_step(plan, prefix_lens=form([0 if s == "b" else 22 for s in plan.seq_ids]))
    b.begin_step(plan)
    assert b.prefix_lens is None


def test_prefix_lens_of_another_step_are_refused():
    p, b = planner(), backend()
    p.add_request("a", 20)
    plan = p.schedule()
    for bad in ([1, 2], [], [[3]], [0.5]):
        with pytest.raises(ValueError, match="one per sequence"):
            b.begin_step(plan, prefix_lens=bad)


def first_chunks(p, steps=40):
    """Tokens of each sequence's first chunk, over steps in which every sequence is seen."""
    first, contexts = {}, {}
    for _ in range(steps):
        plan = p.schedule()
        if plan is None:
            break
        for s, n, c in zip(plan.seq_ids, plan.new_lens.tolist(), plan.host_context_lens.tolist()):
            if c == n:
                first.setdefault(s, []).append(n)
            contexts[s] = c
        for s in p.completed():
            p.finish(s)
    return first, contexts


def test_a_first_chunk_holds_the_prefix():
    p = planner()
    p.add_request("a", 100, 5, prefix_len=70)                    # longer than prefill_chunk
    p.add_request("b", 100, 5, prefix_len=60)                    # 58 tokens are left of the step: waits for the next one
    p.add_request("c", 40, 5, prefix_len=10)                     # (behind b; its chunk is that of every prompt)
    first, contexts = first_chunks(p)
    assert first == {"a": [70], "b": [60], "c": [32]} and contexts == {"a": 104, "b": 104, "c": 44}


def test_a_prefix_survives_preemption_and_forks():
    p = planner(num_blocks=12)
    p.add_request("a", 60, 60, prefix_len=50)
    p.add_request("b", 60, 60, prefix_len=55)
    first, _ = first_chunks(p, 200)
    assert p.num_preemptions > 0 and len(first["b"]) > 1         # ingested again, by one chunk again
    assert set(first["a"]) == {50} and set(first["b"]) == {55}
    p = planner(num_blocks=9)
    p.add_request("a", 60, prefix_len=50)
    p.schedule()
    p.schedule()
    p.fork("a", "b")
    seen = []
    while not seen:
        seen = p.schedule().preempted
    assert seen == ["b"]
    p.finish("a")
    plan = p.schedule()
    assert plan.seq_ids == ["b"] and plan.new_lens.tolist() == [50]


def test_prefixes_that_no_step_can_hold_are_refused():
    p = planner()
    for prefix in (-1, 101):
        with pytest.raises(ValueError, match="prefix_len"):
            p.add_request("a", 100, prefix_len=prefix)
    with pytest.raises(ValueError, match="prefix_len"):
        p.add_request("a", 200, prefix_len=129)                  # max_num_batched_tokens is 128
    p.add_request("a", 200, prefix_len=128)
    plan = p.schedule()
    assert plan.new_lens.tolist() == [128]
