"""A step of drafted tokens whose model fails: the driver and its planner go on as if it had not been begun (runs without a GPU)."""
import pytest
import torch

from aicomp_amd.block_manager import StepPlanner
from aicomp_amd.generation import ScheduleGeneration


class Backend:
    """Takes the steps and moves nothing."""
    device = torch.device("cpu")

    def __init__(self):
        self.plans, self.fails = [], False

    def begin_step(self, plan):
        if self.fails:
            raise MemoryError("no room")
        self.plans.append(plan)

    def keep_drafts(self, kept):
        self.kept = kept


def driver():
    backend, state = Backend(), {"fails": False}

    def model(ids, positions):
        if state["fails"]:
            raise RuntimeError("layer 1 refuses")
        return torch.nn.functional.one_hot(ids % 11, 11).float()

    planner = StepPlanner(num_blocks=8, max_seqs=2, max_seq_len=64, max_num_batched_tokens=64, device="cpu", check_plans=True)
    gen = ScheduleGeneration(model, backend, planner)
    gen.prefill(torch.arange(30).view(2, 15))
    return gen, planner, backend, state


TREES = ([[3, 4, 5], [6]], [[-1, 0, 0], [-1]])


@pytest.mark.parametrize("where", ["model", "begin_step", "tokens"])
def test_a_failed_draft_step_leaves_nothing_open(where):
    gen, planner, backend, state = driver()
    used = planner.alloc.num_used
    state["fails"], backend.fails = where == "model", where == "begin_step"
    tokens = [[3, 4, 2 ** 70], [6]] if where == "tokens" else TREES[0]
    with pytest.raises((RuntimeError, MemoryError, ValueError, OverflowError)):
        gen.draft_step(tokens, TREES[1])
    state["fails"] = backend.fails = False
    with pytest.raises(ValueError, match="follows draft_step"):
        gen.keep_drafts([[0], [0]])
    assert [planner.context_len(b) for b in (0, 1)] == [15, 15] and planner.alloc.num_used == used
    # every way on: a plain step, another tree, a fork, another batch
    assert gen.decode_step(torch.tensor([3, 6])).argmax(-1).tolist() == [3, 6]
    got = gen.draft_step(*TREES)
    assert [x.argmax(-1).tolist() for x in got] == [[3, 4, 5], [6]]
    gen.keep_drafts([[0, 2], [0]])
    assert [planner.context_len(b) for b in (0, 1)] == [18, 17] and backend.kept.keep.tolist() == [0, 2, 0]
    gen.clear_cache()
    assert planner.alloc.num_used == 0
    gen.prefill(torch.arange(12).view(1, 12))
    assert planner.context_len(0) == 12


def test_a_failed_draft_step_then_another_batch():
    gen, planner, backend, state = driver()
    state["fails"] = True
    with pytest.raises(RuntimeError, match="refuses"):
        gen.draft_step(*TREES)
    state["fails"] = False
    gen.clear_cache()
    assert planner.alloc.num_used == 0 and gen.prefill(torch.arange(20).view(2, 10)).shape == (2, 11)
