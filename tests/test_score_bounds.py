"""Chunks by a score rule are laid out for the contexts that they have, not for the table's width (without a GPU: the sizes that the
library plans, and what the backend hands over)."""
import numpy as np
import pytest
import torch

from aicomp_amd import _lib, generation
from aicomp_amd.block_manager import StepPlanner
from aicomp_amd.generation import PagedAttentionBackend


@pytest.mark.parametrize("new", [16, 64, 128, 256, 512])
def test_short_prompts_in_a_wide_table_are_one_part(new):
    """32 / 8 heads of 128, a table of 8192 tokens: no scratch, so no second kernel, once the bound is known."""
    size = lambda bound: _lib.load().aicomp_paged_score_workspace_bytes(1, new, new, 32, 8, 128, 16, 512, _lib.BF16, _lib.BF16, 0, bound)
    assert size(0) > 0 and size(new) == 0
    assert size(8192) == size(0) and size(7000) > 0             # contexts that long are divided


def test_the_backend_hands_over_the_bound(monkeypatch):
    seen = []
    monkeypatch.setattr(generation.ops, "paged_score_prefill_attn", lambda *a, **kw: seen.append(("chunks", kw["longest_context"])))
    monkeypatch.setattr(generation.ops, "paged_score_decode_attn", lambda *a, **kw: seen.append(("rows", kw["longest_context"])))
    monkeypatch.setattr(generation.ops, "kv_append", lambda *a, **kw: None)
    b = PagedAttentionBackend(1, 40, 1, 16, dtype=torch.float32, device="cpu")
    b.set_score_rule(0, softcap=30.0)
    p = StepPlanner(40, 16, max_seqs=4, max_seq_len=256, max_num_batched_tokens=64, prefill_chunk=32, device="cpu")
    for s, n in (("a", 20), ("b", 70), ("c", 9)):
        p.add_request(s, n)
    steps = []
    for _ in range(4):
        plan = p.schedule()
        b.begin_step(plan)
        T = plan.total_new_tokens
        b.attend(0, torch.zeros(T, 2, 16), torch.zeros(T, 1, 16), torch.zeros(T, 1, 16))
        lens, npre = plan.host_context_lens, plan.num_prefill_seqs
        steps += [("chunks", int(lens[:npre].max()))] if npre else []
        steps += [("rows", int(lens[npre:].max()))] if len(lens) > npre else []
    assert seen == steps and {k for k, _ in seen} == {"chunks", "rows"}
    assert all(isinstance(v, int) for _, v in seen) and max(v for _, v in seen) < 256
