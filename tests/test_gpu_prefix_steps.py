"""A prefix longer than the planner's chunks, through a decoder's layers: every row of it sees all of it, as in the whole sequence at once."""
import pytest
import torch

from aicomp_amd.block_manager import StepPlanner
from test_gpu_score_steps import RuledModel, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("on_device", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefix_longer_than_a_chunk(device, dtype, on_device):
    m = RuledModel(device, dtype)
    g = torch.Generator().manual_seed(4)
    ids = {s: torch.randint(0, 97, (n,), generator=g).to(device) for s, n in (("a", 75), ("b", 66))}
    prefix = {"a": 60, "b": 50}
    b = m.backend(20, dtype, device)
    planner = StepPlanner(20, 16, max_seqs=2, max_seq_len=100, prefill_chunk=24, max_num_batched_tokens=96, device=device)
    for s in ids:
        planner.add_request(s, ids[s].numel(), 1, prefix_len=prefix[s])
    model, last = m.paged(b), {}
    while len(last) < 2:
        plan = planner.schedule()
        lens = [prefix[s] for s in plan.seq_ids]
        b.begin_step(plan, prefix_lens=torch.tensor(lens, dtype=torch.int32, device=device) if on_device else lens)
        cu = plan.host_cu_q_lens
        tok = torch.cat([ids[s][torch.from_numpy(plan.host_positions[cu[r]:cu[r + 1]]).to(device)] for r, s in enumerate(plan.seq_ids)])
        out = model(tok, plan.positions)
        for r, s in enumerate(plan.seq_ids):
            if plan.host_context_lens[r] == ids[s].numel():
                last[s] = out[cu[r + 1] - 1]
    for s in ids:
        close(last[s], m.naive(ids[s], prefix=prefix[s]), dtype)


def test_prefixes_are_not_read_while_a_step_is_recorded(device):
    m = RuledModel(device, torch.bfloat16)
    b = m.backend(20, torch.bfloat16, device)
    planner = StepPlanner(20, 16, max_seqs=2, max_seq_len=100, prefill_chunk=24, device=device)
    planner.add_request("a", 20)
    plan = planner.schedule()
    g = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=device)
    with torch.cuda.graph(g):
        x.add_(1)
        with pytest.raises(RuntimeError, match="before the recording"):
            b.begin_step(plan, prefix_lens=[20])
    g.replay()
    assert b.plan is None and bool((x == 1).all())
