"""The larger tiles of prompts and trees, which calls of many workgroups take: 128 queries or rows to a workgroup, several tiles to a
sequence, ragged, behind cached keys, beside values that are not finite; and the largest rows of the kernels that take every size.  Against
float64, with the tolerances of test_gpu_latent.py."""
import math

import pytest
import torch

from helpers import kernels_of
from test_gpu_latent import Case as Latent
from test_gpu_latent import attention_bound, check, expect_prompt, prompt_case, run_prompt
from test_gpu_tree import Case as Tree

pytestmark = pytest.mark.gpu
BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def tile_of(name, kernel):
    """The numbers among the template's arguments."""
    return [int(x) for x in name.split(kernel + "<", 1)[1].split(">")[0].replace(" ", "").split(",") if x.lstrip("-").isdigit()]


RAGGED = ([1, 127, 128, 129, 255, 256, 257, 400, 2, 64, 383, 384, 385, 33, 300, 190],
          [0, 300, 1, 0, 65, 64, 0, 13, 290, 128, 0, 127, 129, 200, 63, 0])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("name", ["whole", "behind", "ragged", "ragged_17", "many_queries_few_keys"])
def test_prompts_of_large_tiles(device, dtype, name):
    """448 workgroups of 128 queries or more.  Up to 16 sequences are taken by cost, 17 in the order of the grid."""
    new, prior, H = {"whole": ([1000], [0], 64), "behind": ([520, 129], [200, 77], 80), "ragged": (*RAGGED, 12),
                     "ragged_17": (RAGGED[0] + [130], RAGGED[1] + [5], 12),
                     "many_queries_few_keys": ([300, 400, 129], [-20, 0, -129], 80)}[name]
    keys = [n + p for n, p in zip(new, prior)]
    q, expanded, latent = prompt_case(keys, new, H, dtype=dtype, seed=41, rows_behind=2)
    got = []
    ran = kernels_of(lambda: got.append(run_prompt(q, expanded, latent, keys, new, 128, 64, 0.07, max_q_len=max(new))))
    assert any("prompt_attn_kernel" in k and tile_of(k, "prompt_attn_kernel") == [2] for k in ran), ran
    want, mean_abs, size = expect_prompt(q, expanded, latent, keys, new, 128, 64, 0.07)
    check(got[0][:-2], want, attention_bound(want, mean_abs, size, 192, dtype))
    assert bool((got[0][-2:] == 7.0).all())


@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_tiles_of_prompts_beside_tokens_that_are_not_finite(dtype, value):
    keys, new, H = [200, 390, 260], [200, 300, 257], 64
    q, expanded, latent = prompt_case(keys, new, H, dtype=dtype, seed=42)
    want, mean_abs, size = expect_prompt(q, expanded, latent, keys, new, 128, 64, 0.07)
    tol = attention_bound(want, mean_abs, size, 192, dtype)
    at = [(0, 130), (1, 389), (2, 3 + 128)]                    # (sequence, key): of a value; the last one of the context; the second tile
    bad, worse, sees = expanded.clone(), expanded.clone(), []
    starts = [0, 200, 590]
    for s, j in at:
        bad[starts[s] + j, :, 128 + 5 * s:128 + 5 * s + 2] = value
        worse[starts[s] + j, :, 40 + s] = value
    sees = torch.cat([torch.arange(keys[s] - new[s], keys[s]) >= j for s, j in at])
    got = run_prompt(q, bad, latent, keys, new, 128, 64, 0.07)
    assert not bool(torch.isfinite(got[sees]).all(-1).any())
    check(got[~sees], want[~sees], tol[~sees])
    got = run_prompt(q, worse, latent, keys, new, 128, 64, 0.07)
    check(got[~sees], want[~sees], tol[~sees])


TREES = ([1040 + 37 * i % 500 for i in range(20)], [40, 33, 1, 64, 17, 39, 2, 48, 31, 32, 63, 20, 5, 55, 36, 16, 47, 60, 7, 34])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,pool", [(BF16, None), (F16, None), (BF16, FP8), (F16, FP8)])
def test_trees_of_large_tiles_divided(device, d, dtype, pool):
    """More than 64 rows to a KV head in more than 128 items over contexts that no workgroup has whole."""
    ctx, new = TREES
    c = Tree(ctx, new, 32, 8, d, dtype=dtype, pool=pool, seed=43, rows_behind=2)
    c.poison()
    got = []
    ran = kernels_of(lambda: got.append(c.run(max_q_len=max(new))))
    assert any("row_attn_shared_kernel" in k and tile_of(k, "row_attn_shared_kernel")[:2] == [d, 2] for k in ran), ran
    assert any("row_join_kernel" in k for k in ran), ran
    c.check(got[0])


@pytest.mark.parametrize("hq,hkv", [(1, 1), (12, 4), (16, 1)])
@pytest.mark.parametrize("dtype,pool", [(BF16, None), (F16, None), (F32, None), (BF16, FP8), (F16, FP8)])
def test_long_trees_of_other_heads(hq, hkv, dtype, pool):
    for d in (64, 128, 256):
        c = Tree([4100, 700], [9, 64], hq, hkv, d, dtype=dtype, pool=pool, seed=47, rows_behind=3)
        c.poison()
        c.check(c.run(max_q_len=64, longest_context=4100))


def test_large_tiles_of_trees_beside_drafts_that_are_not_finite():
    ctx, new = TREES
    for dtype, pool, which in ((BF16, None, "v"), (F16, None, "v"), (F16, FP8, "v"), (BF16, None, "k")):
        clean, c = (Tree(ctx, new, 32, 8, 128, dtype=dtype, pool=pool, seed=44) for _ in range(2))
        where = torch.zeros(c.k.shape[0], 16, dtype=torch.bool)
        bad = {s: ctx[s] - new[s] + new[s] // 2 for s in range(0, 20, 3)}
        for s, j in bad.items():
            where[c.table[s, j // 16].long(), j % 16] = True
        c.bad(where, which == "k", which == "v")
        got = c.run()
        want, mean_abs, size = clean.expect()
        sees = torch.cat([clean.visible(s)[:, bad[s]] if s in bad else torch.zeros(new[s], dtype=torch.bool) for s in range(20)])
        assert bool(sees.any()) and not bool(sees.all()) and not bool(torch.isfinite(got[sees]).all(-1).any())
        tol = attention_bound(want, mean_abs, size, 128, dtype)
        check(got[~sees], want[~sees], tol[~sees])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_largest_rows(dtype):
    """1024 + 256 elements of a latent row; prompts of 1216 + 64 and 1024."""
    c = Latent([90, 33, 300], [20, 33, 7], 2, 1024, 256, dtype=dtype, seed=45)
    c.poison()
    c.check(c.run())
    keys, new = [70, 300], [70, 9]
    q, expanded, latent = prompt_case(keys, new, 2, 1216, 64, 1024, dtype, seed=46)
    got = run_prompt(q, expanded, latent, keys, new, 1216, 64, 0.03)
    want, mean_abs, size = expect_prompt(q, expanded, latent, keys, new, 1216, 64, 0.03)
    check(got, want, attention_bound(want, mean_abs, size, 1280, dtype))
