"""Attention of trees of drafted tokens over the paged K and V pools, and the accepted rows moved together, against plain forms.

Tolerances of the attention: those of test_gpu_latent.py with scores of D products; an fp8 pool's codes are exact in the 16-bit formats
and its scales are float32 factors.  Moved rows are copies: equal.
"""
import math

import pytest
import torch

from aicomp_amd import ops
from oracle.rows_oracle import kept, masked_attention, tree_visible
from test_gpu_latent import attention_bound, check, parents_of

pytestmark = pytest.mark.gpu
BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
TYPES = [(BF16, None), (F16, None), (F32, None), (BF16, FP8), (F16, FP8)]


class Case:
    def __init__(self, ctx, new, hq, hkv, d, bs=16, dtype=BF16, pool=None, seed=0, rows_behind=0, spread=1.5):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.new, self.hq, self.hkv, self.d, self.bs, self.dtype = ctx, new, hq, hkv, d, bs, dtype
        self.pool = pool or dtype
        need = [-(-max(c, 0) // bs) for c in ctx]
        nb = sum(need) + 3
        order = torch.randperm(nb, generator=g)
        self.table = torch.randint(-5, nb + 5, (len(ctx), max(max(need), 1) + 2), generator=g, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.k, self.v = torch.randn(2, nb, hkv, bs, d, generator=g)
        self.ks = self.vs = None
        if self.pool == FP8:
            self.ks, self.vs = torch.rand(2, hkv, generator=g) * 0.01 + 0.005
            self.k = (self.k / self.ks[:, None, None]).clamp(-448, 448)
            self.v = (self.v / self.vs[:, None, None]).clamp(-448, 448)
        self.k, self.v = self.k.to(self.pool), self.v.to(self.pool)
        self.q = (torch.randn(sum(new) + rows_behind, hq, d, generator=g) * spread).to(dtype)
        self.parents = [parents_of(n, s + seed) for s, n in enumerate(new)]
        self.scale = 1 / math.sqrt(d)

    def rows(self, s):
        j = torch.arange(max(self.ctx[s], 0))
        blk, off = self.table[s].long()[j // self.bs], j % self.bs
        k, v = self.k[blk, :, off].double(), self.v[blk, :, off].double()
        return (k, v) if self.ks is None else (k * self.ks.double()[:, None], v * self.vs.double()[:, None])

    def bad(self, where, k=True, v=True):
        """Not a number into these rows [num_blocks, bs] of the pools."""
        for t in [x for x, on in ((self.k, k), (self.v, v)) if on]:
            if self.pool == FP8:
                t.view(torch.uint8).transpose(1, 2)[where] = 0x7f
            else:
                t.transpose(1, 2)[where] = torch.inf if self.dtype == F16 else torch.nan

    def poison(self):
        free = torch.ones(self.k.shape[0], self.bs, dtype=torch.bool)
        for s, c in enumerate(self.ctx):
            j = torch.arange(max(c, 0))
            free[self.table[s].long()[j // self.bs], j % self.bs] = False
        self.bad(free)

    def run(self, masks=None, **kw):
        cuda = lambda x: None if x is None else x.cuda()
        out = torch.full_like(self.q, 7.0).cuda()
        masks = torch.from_numpy(ops.tree_masks(self.parents)) if masks is None else masks
        if masks.shape[0] < self.q.shape[0]:
            masks = torch.cat((masks, masks.new_zeros(self.q.shape[0] - masks.shape[0], masks.shape[1])))
        cu = torch.tensor([0] + torch.tensor(self.new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        lens = torch.tensor(self.ctx, dtype=torch.int32, device="cuda")
        ops.paged_tree_attn(out, self.q.cuda(), self.k.cuda(), self.v.cuda(), self.table.cuda(), lens, cu, masks.cuda(), self.scale,
                            k_scale=cuda(self.ks), v_scale=cuda(self.vs), **kw)
        return out.cpu()

    def visible(self, s):
        return tree_visible(self.ctx[s], self.new[s], self.parents[s])

    def expect(self):
        parts, t = [], 0
        for s, (c, n) in enumerate(zip(self.ctx, self.new)):
            if n > c:
                z = torch.zeros(n, self.hq, self.d, dtype=torch.float64)
                parts.append((z, z, z[..., 0]))
            elif n:
                parts.append(masked_attention(self.q[t:t + n], *self.rows(s), self.visible(s), self.scale))
            t += n
        return [torch.cat(x) for x in zip(*parts)]

    def check(self, got):
        want, mean_abs, size = self.expect()
        t = sum(self.new)
        check(got[:t], want, attention_bound(want, mean_abs, size, self.d, self.dtype))
        assert bool((got[t:] == 7.0).all()), "rows behind the last sequence were written"


TREES = {"one": ([40], [1]), "fresh": ([30], [30]), "ragged": ([300, 47, 260, 64, 31], [70, 13, 1, 32, 31]),
         "short_context": ([5, 90, 0], [9, 20, 3]), "empty": ([33, 20, 500], [3, 0, 17]),
         "many": ([60 + 9 * i for i in range(40)], [1 + i % 9 for i in range(40)]), "long": ([4100, 700], [9, 64])}


@pytest.mark.parametrize("name", TREES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 2), (12, 4), (16, 1)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,pool", TYPES)
def test_trees(dtype, pool, d, hq, hkv, name):
    if name == "long" and (hq, hkv) != (8, 2):
        pytest.skip("one head layout is enough for the long contexts")
    c = Case(*TREES[name], hq, hkv, d, dtype=dtype, pool=pool, seed=1, rows_behind=3)
    c.poison()
    c.check(c.run(max_q_len=max(c.new), longest_context=max(c.ctx)))


@pytest.mark.parametrize("bs", [1, 8, 24, 32])
@pytest.mark.parametrize("dtype,pool,d", [(BF16, None, 128), (F16, FP8, 64), (F32, None, 64)])
def test_other_block_sizes(dtype, pool, d, bs):
    c = Case(*TREES["ragged"], 4, 2, d, bs=bs, dtype=dtype, pool=pool, seed=2)
    c.poison()
    c.check(c.run())


@pytest.mark.parametrize("n", [63, 64, 65, 130, 200])
@pytest.mark.parametrize("dtype,pool", [(BF16, None), (F16, FP8)])
def test_trees_of_several_words(dtype, pool, n):
    c = Case([n + 70, n, n + 5], [n, n, 7], 4, 2, 128, dtype=dtype, pool=pool, seed=3)
    c.check(c.run())


@pytest.mark.parametrize("dtype,pool,d", [(BF16, None, 128), (F16, FP8, 64), (F32, None, 128)])
def test_masks_that_are_no_trees(dtype, pool, d):
    """Rows that see nothing, not themselves, later drafts, and bits of drafts that are not there."""
    c = Case([21, 150, 80], [21, 30, 17], 4, 1, d, dtype=dtype, pool=pool, seed=4)
    g = torch.Generator().manual_seed(5)
    masks = torch.randint(-2 ** 62, 2 ** 62, (68, 1), generator=g) * 2 + torch.randint(0, 2, (68, 1), generator=g)
    masks[5], masks[25], masks[67] = 0, 0, -1
    got, t = c.run(masks), 0
    for s, n in enumerate(c.new):
        see = torch.ones(n, c.ctx[s], dtype=torch.bool)
        for i in range(n):
            see[i, c.ctx[s] - n:] = torch.tensor([(int(masks[t + i, 0]) >> b) & 1 == 1 for b in range(n)])
        want, mean_abs, size = masked_attention(c.q[t:t + n], *c.rows(s), see, c.scale)
        check(got[t:t + n], want, attention_bound(want, mean_abs, size, d, dtype))
        t += n
    assert bool((got[5] == 0).all())


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dtype,pool", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_rows_beside_drafts_that_are_not_finite(d, dtype, pool, which):
    clean = Case([200, 75, 40], [40, 40, 40], 8, 2, d, dtype=dtype, pool=pool, seed=6)
    c = Case([200, 75, 40], [40, 40, 40], 8, 2, d, dtype=dtype, pool=pool, seed=6)
    bad, where = {0: 160 + 21, 1: 35 + 39, 2: 3}, torch.zeros(c.k.shape[0], 16, dtype=torch.bool)
    for s, j in bad.items():
        where[c.table[s, j // 16].long(), j % 16] = True
    c.bad(where, which == "k", which == "v")
    got = c.run()
    want, mean_abs, size = clean.expect()
    sees = torch.cat([clean.visible(s)[:, j] for s, j in bad.items()])
    assert bool(sees.any()) and not bool(sees.all())
    if which == "v" or dtype != F16 or pool == FP8:                  # (an infinite key can be of weight 0)
        assert not bool(torch.isfinite(got[sees]).all(-1).any())
    tol = attention_bound(want, mean_abs, size, d, dtype)
    check(got[~sees], want[~sees], tol[~sees])


def test_chain_is_causal_attention():
    """A tree without branches gives what the chunk kernels give, to the rounding of the formats."""
    c = Case([300, 90], [33, 20], 8, 2, 128, seed=7)
    c.parents = [list(range(-1, n - 1)) for n in c.new]
    got = c.run()
    q, out = c.q.cuda(), torch.empty_like(c.q).cuda()
    ops.paged_prefill_attn(out, q, c.k.cuda(), c.v.cuda(), c.table.clamp(0, c.k.shape[0] - 1).cuda(),
                           torch.tensor(c.ctx, dtype=torch.int32, device="cuda"),
                           torch.tensor([0, 33, 53], dtype=torch.int32, device="cuda"), c.scale, max_q_len=33)
    want, mean_abs, size = c.expect()
    tol = attention_bound(want, mean_abs, size, 128, BF16)
    check(got, want, tol)
    assert bool(((got.double() - out.cpu().double()).abs() <= 4 * tol).all())


# ------------------------------------------------------------------------------------------ accepted rows
def keep_case(firsts, keep, bs, width, nb, seed):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(nb, generator=g)
    table, at = torch.full((len(firsts), width), -1, dtype=torch.int32), 0
    for s, (f, k) in enumerate(zip(firsts, keep)):
        n = min(width, -(-(f + (k[-1] if k else 0) + 1) // bs))
        table[s, :n] = order[at:at + n]
        at += n
    flat = torch.tensor([x for row in keep for x in row], dtype=torch.int32)
    cu = torch.tensor([0] + torch.tensor([len(k) for k in keep]).cumsum(0).tolist(), dtype=torch.int32)
    return table, torch.tensor(firsts, dtype=torch.int32), flat, cu


KEEPS = {"one": ([37], [[0, 2, 3, 7]]), "in_place": ([5, 0], [[0, 1, 2], [0]]), "shift": ([14, 30], [[1, 2, 3, 4, 5, 6, 7, 8, 9, 10], [3]]),
         "none": ([3, 9, 40], [[0, 9], [], [5, 6, 7, 8, 20]]), "wide": ([100], [list(range(1, 90, 2))])}


@pytest.mark.parametrize("where", ["host", "device"])
@pytest.mark.parametrize("name", KEEPS)
@pytest.mark.parametrize("shape,dtype", [((2, 16, 64), BF16), ((3, 1, 16), F32), ((1, 16, 3), FP8), ((8, 16, 128), F16), ((2, 5, 7), BF16),
                                         ((16, 576), BF16)])
def test_keep_rows(shape, dtype, name, where):
    firsts, keep = KEEPS[name]
    bs = shape[-2]
    table, first, flat, cu = keep_case(firsts, keep, bs, 200 // bs + 2, 500 // bs + 10, 8)
    g = torch.Generator().manual_seed(9)
    pools = [torch.randint(0, 120, (500 // bs + 10, *shape), generator=g, dtype=torch.uint8).to(dtype) for _ in range(5)]
    dev = [p.cuda() for p in pools]
    args = (first, flat, cu) if where == "host" else (first.cuda(), flat.cuda(), cu.cuda())
    ops.keep_rows(dev, table.cuda(), *args)
    for p, d in zip(pools, dev):
        four = (lambda x: x[:, None] if x.dim() == 3 else x)(p.view(torch.uint8) if dtype == FP8 else p)
        want = kept(four, table, firsts, keep)
        got = d.cpu().view(torch.uint8) if dtype == FP8 else d.cpu()
        assert torch.equal(got.view(want.shape), want)


def test_keep_rows_of_more_pools_than_one_launch_and_tokens_beyond_the_table():
    keep = [[0, 3, 5], [2, 40]]
    table, first, flat, cu = keep_case([10, 30], keep, 16, 4, 20, 10)
    pools = [torch.randn(20, 2, 16, 8, generator=torch.Generator().manual_seed(i)) for i in range(131)]
    dev = [p.cuda() for p in pools]
    ops.keep_rows(dev, table.cuda(), first, flat, cu)              # (token 70 of sequence 1 is beyond its 64)
    for p, d in zip(pools, dev):
        assert torch.equal(d.cpu(), kept(p, table, [10, 30], keep))
