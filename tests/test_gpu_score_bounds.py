"""The bound of the contexts that a chunk call by a score rule may be given: both host routes, right, small and large ones."""
import pytest
import torch

from aicomp_amd import ops
from aicomp_amd.block_manager import StepPlanner
from helpers import kernels_of
from test_gpu_score_attn import BF16, F16, F32, FP8, Case, check, expect, run_prefill, slopes_of
from test_gpu_score_steps import RuledModel, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype,pool", [(BF16, None), (F16, FP8), (F32, None)])
@pytest.mark.parametrize("bound", [0, 1, 200, 4000])
def test_a_bound_sizes_the_call_and_cuts_nothing(monkeypatch, dtype, pool, bound, native):
    if not native:
        monkeypatch.setattr(ops, "_FAST", None)
    c = Case([200, 33, 5], [70, 33, 1], 8, 2, 128, dtype=dtype, pool=pool, seed=13, rows_behind=2, width=250)
    want, mean_abs, size = expect(c, 20.0, slopes_of(8), 0, None, None)
    got = []
    names = kernels_of(lambda: got.append(run_prefill(c, 20.0, slopes_of(8), longest_context=bound)))
    # 4000 tokens are worth dividing among workgroups, 200 are not
    assert any("score_prefill_join" in n for n in names) == (bound in (0, 4000)), names
    assert bool((got[0][-2:] == 7.0).all())
    check(got[0][:-2], c, want, mean_abs, size)


@pytest.mark.parametrize("native", [True, False])
def test_a_bound_beyond_the_table_or_32_bits(monkeypatch, native):
    if not native:
        monkeypatch.setattr(ops, "_FAST", None)
    c = Case([200], [70], 8, 2, 128, seed=13)
    assert torch.equal(run_prefill(c, 20.0, longest_context=2 ** 31 - 1), run_prefill(c, 20.0))
    for bad in (-1, 2 ** 31, -2 ** 40):
        with pytest.raises(RuntimeError, match="longest.context"):
            run_prefill(c, 20.0, longest_context=bad)


def test_the_backends_first_chunks_are_one_kernel(device):
    """A short prompt in a planner's wide tables: no layer joins parts; recorded steps are sized for the table."""
    m = RuledModel(device, BF16)
    b = m.backend(600, BF16, device, max_positions=8192)
    planner = StepPlanner(600, 16, max_seqs=2, max_seq_len=8192, device=device)
    planner.add_request("a", 60)
    plan = planner.schedule()
    ids = torch.randint(0, 97, (60,), generator=torch.Generator().manual_seed(2)).to(device)
    b.begin_step(plan)
    out = []
    names = kernels_of(lambda: out.append(m.paged(b)(ids, plan.positions)))
    assert sum("score_prefill" in n for n in names) == 2 and not any("score_prefill_join" in n for n in names), names
    close(out[0][-1], m.naive(ids), BF16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        recorded = m.paged(b)(ids, plan.positions)
    names = kernels_of(g.replay)
    assert any("score_prefill_join" in n for n in names), names
    for _ in range(2):
        recorded.zero_()
        g.replay()
        close(recorded[-1], m.naive(ids), BF16)
