"""Chunks by a score rule where a wrong border would be small in the result: every row of calls that take 128 rows to a workgroup against
float64, rows beside keys that are not finite among them, and block sizes other than 16.  Cases, oracle and tolerances are those of
test_gpu_score_attn.py: a row's bound is made of its own weighted mean of |v| and its own largest score."""
import math

import pytest
import torch

from helpers import kernels_of
from oracle.score_oracle import score_attention_rows
from test_gpu_score_attn import BF16, CHUNKS, F16, F32, FP8, Case, check, expect, large_case, rule, run_prefill, slopes_of, visible

pytestmark = pytest.mark.gpu


def expect_rows(c, cap, slopes, window, first, prefix):
    parts, t = [], 0
    for s, n in enumerate(c.new):
        k, v = c.rows(s)
        parts.append(score_attention_rows(c.q[t:t + n], k, v, c.ctx[s] - n, c.scale, cap, slopes, window,
                                          None if first is None else first[t:t + n], 0 if prefix is None else int(prefix[s])))
        t += n
    return [torch.cat(x) for x in zip(*parts)]


@pytest.mark.parametrize("dtype,pool,name", [(BF16, None, "cap"), (BF16, None, "window"), (BF16, None, "all"), (F16, None, "slopes"),
                                             (BF16, FP8, "all"), (F32, None, "all")])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_every_row_of_large_chunks(dtype, pool, name, d):
    c = large_case(d, dtype, pool, 61)
    r = rule(name, c, torch.Generator().manual_seed(9))
    if name == "all":
        r["prefix"] = torch.full((len(c.new),), 90, dtype=torch.int32)
    want, mean_abs, size = expect_rows(c, r.get("cap", 0.0), r.get("slopes"), r.get("window", 0), r.get("first"), r.get("prefix"))
    total = sum(c.new)
    check(run_prefill(c, **r)[:total], c, want, mean_abs, size)


@pytest.mark.parametrize("dtype,pool", [(BF16, None), (F16, FP8)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_of_large_chunks_beside_values_that_are_not_finite(dtype, pool, d):
    """Keys whose values are not finite: every row that sees none of them is what it is without them."""
    c, clean = large_case(d, dtype, pool, 63), large_case(d, dtype, pool, 63)
    bad = [set() for _ in c.new]
    for s in range(0, len(c.new) - 3, 3):
        for j in (c.ctx[s] - 1, 50 + s, c.ctx[s] // 2):
            bad[s].add(j)
            at = c.v[int(c.table[s, j // 16]), :, j % 16]
            if pool == FP8:
                at.view(torch.uint8).fill_(0x7f)                          # (the code that is not a number)
            else:
                at.fill_(math.inf)
    window = 40
    sees = torch.cat([torch.tensor([any(p - window < j <= p for j in bad[s]) for p in range(c.ctx[s] - n, c.ctx[s])])
                      for s, n in enumerate(c.new)])
    assert bool(sees.any()) and not bool(sees.all())
    got = run_prefill(c, 5.0, window=window)[:sum(c.new)]
    assert not bool(torch.isfinite(got[sees]).any())
    want, mean_abs, size = expect_rows(clean, 5.0, None, window, None, None)
    check(got[~sees], c, want[~sees], mean_abs[~sees], size[~sees])


RULES_BY_BLOCK = ["cap", "all", "prefix_window"]


@pytest.mark.parametrize("name", RULES_BY_BLOCK)
@pytest.mark.parametrize("bs", [1, 8, 24, 32, 64])
@pytest.mark.parametrize("dtype,pool,hq,hkv,d", [(BF16, None, 4, 1, 128), (F16, FP8, 4, 2, 64), (F32, None, 3, 1, 64), (BF16, None, 8, 1, 256)])
def test_chunks_of_other_block_sizes(dtype, pool, hq, hkv, d, bs, name):
    g = torch.Generator().manual_seed(6)
    for i, (ctx, new) in enumerate(CHUNKS[k] for k in ("one", "ragged", "short_context", "empty_chunk")):
        c = Case(ctx, new, hq, hkv, d, bs=bs, dtype=dtype, pool=pool, seed=i, rows_behind=3)
        if name == "prefix_window":
            r = {"prefix": torch.tensor([50, 7, 1000, 0, 33][:len(ctx)], dtype=torch.int32), "window": 40, "slopes": slopes_of(hq)}
        else:
            r = rule(name, c, g)
        want, mean_abs, size = expect(c, r.get("cap", 0.0), r.get("slopes"), r.get("window", 0), r.get("first"), r.get("prefix"))
        got = run_prefill(c, **r)
        assert bool((got[-3:] == 7.0).all()), "rows behind the last sequence were written"
        check(got[:-3], c, want, mean_abs, size)


@pytest.mark.parametrize("bs", [8, 32])
@pytest.mark.parametrize("dtype,pool", [(BF16, None), (F16, FP8), (F32, None)])
def test_chunks_of_other_block_sizes_never_look_at_masked_keys(dtype, pool, bs):
    c = Case([300, 47, 260], [70, 13, 33], 8, 4, 128, bs=bs, dtype=dtype, pool=pool, seed=9)
    first = torch.cat([torch.full((n,), f, dtype=torch.int32) for n, f in zip(c.new, (190, 20, 0))])
    c.poison(visible(c, 50, first))
    want, mean_abs, size = expect(c, 10.0, None, 50, first, None)
    got = []
    names = kernels_of(lambda: got.append(run_prefill(c, cap=10.0, window=50, first=first)))
    assert any("score_generic" in n for n in names), names
    check(got[0], c, want, mean_abs, size)
