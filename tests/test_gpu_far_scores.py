"""Scores far from zero, where a float32 score is rounded by more than a weight spans: rows over latent rows, trees, prompts, every
kernel of them, against float64.

A row's scores, in base 2, are float32 sums of dk products times a factor, so off by at most e = (dk + 44) 2^-24 of their size.  Where the
largest of them leads by more than 2 e + 64, the others weigh less than 2^-64 and the result is the value there: in 16 bits that value
itself, whose weight and sum are alike, in float32 within 2^-20.  Where it does not, the result is a mean of the values seen, whatever its
weights: between the smallest and the largest of them, up to the roundings of the weights and of the result, three of at most eps / 2.
Keys that are all alike weigh alike whatever their score: the result is the plain mean.
"""
import math

import pytest
import torch

import test_gpu_latent as latent
import test_gpu_tree as tree
from oracle.rows_oracle import tree_visible

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def far(dk, exponent, scale):
    """Elements 1 to 3 times their size, all products of a query's and a key's positive: their scores, in base 2, are about 2^exponent.
    Returns the factors of the key's and of the query's elements."""
    size = exponent - math.log2(4 * dk * scale / math.log(2))
    of_key = min(size / 2, 13.0)
    return 2.0 ** of_key, 2.0 ** (size - of_key)


def spread(g, *shape):
    return 1 + 2 * torch.rand(*shape, generator=g)


def check_rows(got, q, k, v, visible, scale):
    """One sequence: ``got [n, H, dv]``, ``q [n, H, dk]``, ``k [c, Hkv, dk]``, ``v [c, Hkv, dv]``, ``visible [n, c]``.  Returns how many
    rows have one key that leads."""
    n, H, dk = q.shape
    group, u, lead = H // k.shape[1], torch.finfo(got.dtype).eps / 2, 0
    assert bool(torch.isfinite(got).all())
    for h in range(H):
        x = q[:, h].double() @ k[:, h // group].double().T * (scale / math.log(2))
        size = q[:, h].double().abs() @ k[:, h // group].double().abs().T * abs(scale / math.log(2))
        x, size = x.masked_fill(~visible, -math.inf), size.masked_fill(~visible, 0)
        vh, have = v[:, h // group].double(), got[:, h].double()
        top = x.topk(min(2, x.shape[1]), dim=-1)
        gap = top.values[:, 0] - top.values[:, 1] if x.shape[1] > 1 else torch.full((n,), math.inf)
        clear = gap > 2 * (dk + 44) * 2.0 ** -24 * size.amax(-1) + 64
        want = vh[top.indices[:, 0]]
        tol = want.abs() * (2.0 ** -20 if got.dtype == F32 else 0.0)
        assert bool(((have - want).abs() <= tol)[clear].all()), f"head {h}: {(have - want)[clear].abs().max()}"
        low = torch.stack([vh[s].amin(0) for s in visible])
        high = torch.stack([vh[s].amax(0) for s in visible])
        slack = 4 * u * torch.maximum(low.abs(), high.abs())
        assert bool(((have >= low - slack) & (have <= high + slack)).all()), f"head {h}"
        lead += int(clear.sum())
    return lead


EXPONENTS = [(F16, 20), (F16, 27), (F16, 30), (F16, 32), (BF16, 20), (BF16, 27), (BF16, 34), (BF16, 60), (BF16, 90), (F32, 34), (F32, 90)]


LATENT = {"one": ([90, 1, 700, 33], [1] * 4, 16), "one_divided": ([1500, 40], [1] * 2, 16), "one_many_heads": ([90, 1, 700, 33], [1] * 4, 40),
          "many_heads_divided": ([1500, 40], [1] * 2, 40), "chunk": ([150, 40, 300], [20, 40, 7], 6), "tree": ([150, 40, 300], [20, 40, 7], 6)}


def latent_case(name, dtype, exponent, sign):
    ctx, new, H = LATENT[name]
    c = latent.Case(ctx, new, H, dtype=dtype, seed=31)
    if name == "tree":
        c.tree()
    g = torch.Generator().manual_seed(32)
    key, query = far(576, exponent, c.scale)
    side = torch.randint(0, 2, (576,), generator=g) * 2 - 1
    c.pool = (spread(g, *c.pool.shape) * side * key).to(dtype)
    c.q = (spread(g, *c.q.shape) * side * (sign * query)).to(dtype)
    return c


def run_latent(name, dtype, exponent, sign):
    c = latent_case(name, dtype, exponent, sign)
    got, t, lead = c.run(longest_context=0 if "divided" in name else max(c.ctx)), 0, 0
    for s, n in enumerate(c.new):
        k = c.rows(s)[:, None]
        lead += check_rows(got[t:t + n], c.q[t:t + n], k, k[..., :c.C], c.visible(s), c.scale)
        t += n
    assert exponent < 27 or lead > t * c.H // 2


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,exponent", EXPONENTS)
@pytest.mark.parametrize("name", LATENT)
def test_latent_rows(name, dtype, exponent, sign):
    run_latent(name, dtype, exponent, sign)


TREE = {"few_rows": ([150, 40, 300], [7, 4, 8], 8, 2), "few_rows_divided": ([1500, 40], [7, 4], 8, 2),
        "many_rows": ([150, 40, 300], [20, 40, 7], 8, 2), "many_rows_divided": ([1500, 90], [70, 30], 8, 2)}


def run_tree(name, dtype, exponent, sign, alike=False):
    ctx, new, hq, hkv = TREE[name]
    c = tree.Case(ctx, new, hq, hkv, 128, dtype=dtype, seed=34)
    g = torch.Generator().manual_seed(35)
    key, query = far(128, exponent, c.scale)
    side = torch.randint(0, 2, (128,), generator=g) * 2 - 1
    c.k = (spread(g, *((1, 1, 1, 128) if alike else c.k.shape)) * side * key).to(dtype).expand(c.k.shape).contiguous()
    c.q = (spread(g, *c.q.shape) * side * (sign * query)).to(dtype)
    got, t, lead = c.run(longest_context=0 if "divided" in name else max(c.ctx)), 0, 0
    if alike:
        for s, n in enumerate(c.new):
            see, v = c.visible(s).double(), c.rows(s)[1].repeat_interleave(hq // hkv, 1).flatten(1)
            mean, size = [(see @ x / see.sum(1, keepdim=True)).view(n, hq, 128) for x in (v, v.abs())]
            latent.check(got[t:t + n], mean, latent.attention_bound(mean, size, torch.zeros(n, hq).double(), 128, dtype))
            t += n
        return
    for s, n in enumerate(c.new):
        lead += check_rows(got[t:t + n], c.q[t:t + n], *c.rows(s), c.visible(s), c.scale)
        t += n
    assert exponent < 27 or lead > t * hq // 2


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,exponent", EXPONENTS)
@pytest.mark.parametrize("name", TREE)
def test_trees(name, dtype, exponent, sign):
    run_tree(name, dtype, exponent, sign)
    run_tree(name, dtype, exponent, sign, alike=True)


# (448 workgroups of 128 queries or more: the larger tile)
PROMPT = {"small": ([200, 90, 1], [200, 30, 1], 3), "large": ([140, 200], [140, 129], 112)}


def run_prompt(name, dtype, exponent, sign, alike=False):
    keys, new, H = PROMPT[name]
    g = torch.Generator().manual_seed(37)
    key, query = far(192, exponent, 0.07)
    side = torch.randint(0, 2, (192,), generator=g) * 2 - 1
    Tq, Tk = sum(new), sum(keys)
    q = (spread(g, Tq, H, 192) * side * (sign * query)).to(dtype)
    k = spread(g, *((1, 1, 192) if alike else (Tk, H, 192))) * side * key
    k[..., 128:] = k[:, :1, 128:]                                  # shared by the heads
    k = k.to(dtype).expand(Tk, H, 192).contiguous()
    v = torch.randn(Tk, H, 128, generator=g).to(dtype)
    rows = torch.cat((torch.zeros(Tk, 512, dtype=dtype), k[:, 0, 128:]), dim=-1)
    expanded = torch.cat((k[..., :128], v), dim=-1)
    got = latent.run_prompt(q, expanded, rows, keys, new, 128, 64, 0.07, max_q_len=max(new))
    t = u = lead = 0
    for c, n in zip(keys, new):
        if alike:
            mean, size = [x.cumsum(0)[c - n:] / torch.arange(c - n + 1, c + 1)[:, None, None] for x in
                          (v[u:u + c].double(), v[u:u + c].double().abs())]
            latent.check(got[t:t + n], mean, latent.attention_bound(mean, size, torch.zeros(n, H).double(), 192, dtype))
        else:
            lead += check_rows(got[t:t + n], q[t:t + n], k[u:u + c], v[u:u + c], tree_visible(c, n), 0.07)
        t, u = t + n, u + c
    assert alike or exponent < 27 or lead > t * H // 2


# (float32 prompts have one kernel, whatever their number of heads)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("name,dtype,exponent", [(name, *x) for name in PROMPT for x in EXPONENTS if name == "small" or x[0] != F32])
def test_prompts(name, dtype, exponent, sign):
    run_prompt(name, dtype, exponent, sign)
    run_prompt(name, dtype, exponent, sign, alike=True)


# Nothing a row sees is within 1e30 = 2^99.7 of zero.  The sums of products that a score is made of are larger than it, by up to ln 2 / 0.07
# = 2^3.3 here, and by 9 / 4 = 2^1.2 where all elements are the largest: of scores of 2^122 they stay below 2^126.5, inside float32; of
# 2^125 they would not, and a sum that is infinite tells nothing of its keys.
LAST = [(dtype, exponent, sign) for dtype in (BF16, F32) for exponent in (110, 122) for sign in (1, -1)]


@pytest.mark.parametrize("dtype,exponent,sign", LAST)
@pytest.mark.parametrize("name", LATENT)
def test_latent_rows_to_the_end_of_float32(name, dtype, exponent, sign):
    run_latent(name, dtype, exponent, sign)


@pytest.mark.parametrize("dtype,exponent,sign", LAST)
@pytest.mark.parametrize("name", TREE)
def test_trees_to_the_end_of_float32(name, dtype, exponent, sign):
    run_tree(name, dtype, exponent, sign)
    run_tree(name, dtype, exponent, sign, alike=True)


@pytest.mark.parametrize("name,dtype,exponent,sign", [(name, *x) for name in PROMPT for x in LAST if name == "small" or x[0] != F32])
def test_prompts_to_the_end_of_float32(name, dtype, exponent, sign):
    run_prompt(name, dtype, exponent, sign)
    run_prompt(name, dtype, exponent, sign, alike=True)
