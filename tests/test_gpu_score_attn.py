"""Attention by a score rule against the float64 oracle: one token per sequence and chunks, every type pair and head_dim, masks
that leave rows empty, non-finite values where nothing may look, rows behind the last sequence.

Tolerance, per output element and derived from the formats: the result is rounded once (half a step of the output type, u = eps / 2
relative).  The matrix-core kernels round the weights to the 16-bit type, u each, so that the mean moves by at most 2 u times the
weighted mean of |v| and of the result.  A score is a float32 sum of up to 256 products: off by at most ds = 300 * 2^-24 * max_j scale
sum_d |q_d k_jd| (a cap only shrinks it; cap - 2 cap / (1 + e^y) itself adds up to 4 half steps of float32 at cap), which moves a weight by e^(2 ds) - 1 relative to the others.  Float32 sums of up to 2000
weights and exponents of up to 2^7 add less than 1e-5 of that; a float32 call rounds no weight.
"""
import math

import pytest
import torch

from aicomp_amd import _lib, ops
from helpers import kernels_of
from oracle.score_oracle import score_attention

pytestmark = pytest.mark.gpu
BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


class Case:
    """Pools, tables and queries of sequences with ``ctx`` tokens, the last ``new`` of them rows of the call."""

    def __init__(self, ctx, new, hq, hkv, d, bs=16, dtype=BF16, pool=None, seed=0, rows_behind=0, width=None, poison=False):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.new, self.hq, self.hkv, self.d, self.bs = ctx, new, hq, hkv, d, bs
        self.dtype, self.pool_dtype = dtype, pool or dtype
        need = [-(-max(c, 0) // bs) for c in ctx]
        nb = sum(need) + 3
        order = torch.randperm(nb, generator=g)
        width = width or max(max(need), 1) + 2
        self.table = torch.randint(0, nb, (len(ctx), width), generator=g, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.k = torch.randn(nb, hkv, bs, d, generator=g)
        self.v = torch.randn(nb, hkv, bs, d, generator=g)
        self.ks = self.vs = None
        if self.pool_dtype == FP8:
            self.ks, self.vs = torch.rand(hkv, generator=g) * 0.01 + 0.005, torch.rand(hkv, generator=g) * 0.01 + 0.005
            # (cut to +-448 like the append does: a code beyond that is not a number)
            self.k = (self.k / self.ks[:, None, None]).clamp(-448, 448).to(FP8)
            self.v = (self.v / self.vs[:, None, None]).clamp(-448, 448).to(FP8)
        else:
            self.k, self.v = self.k.to(self.pool_dtype), self.v.to(self.pool_dtype)
        self.total = sum(new) + rows_behind
        self.q = torch.randn(self.total, hq, d, generator=g).mul_(1.5).to(dtype)
        self.scale = 1 / math.sqrt(d)

    def rows(self, s):
        """K and V of a sequence's context, as the values they stand for."""
        c = max(self.ctx[s], 0)
        j = torch.arange(c)
        blk, off = self.table[s].long()[j // self.bs], j % self.bs
        k, v = self.k[blk, :, off].double(), self.v[blk, :, off].double()
        if self.ks is not None:
            k, v = k * self.ks.double()[:, None], v * self.vs.double()[:, None]
        return k, v

    def poison(self, visible):
        """Not a number into every pool row that no row of the call sees."""
        nb = self.k.shape[0]
        keep = torch.zeros(nb, self.bs, dtype=torch.bool)
        for s, seen in enumerate(visible):
            j = torch.nonzero(seen).flatten()
            keep[self.table[s].long()[j // self.bs], j % self.bs] = True
        bad = ~keep
        for t, x in ((self.k, math.nan), (self.v, math.inf if self.pool_dtype != FP8 else math.nan)):
            hit = torch.tensor(x).to(self.pool_dtype)
            t.transpose(1, 2)[bad] = hit.expand(self.hkv, self.d) if self.pool_dtype != FP8 else hit.view(torch.uint8).expand(
                self.hkv, self.d).contiguous().view(FP8)


def expect(c, cap, slopes, window, first, prefix):
    outs, means, sizes, t = [], [], [], 0
    for s, (ctx, n) in enumerate(zip(c.ctx, c.new)):
        if n > ctx:
            outs.append(torch.zeros(n, c.hq, c.d, dtype=torch.float64))
            means.append(outs[-1])
            sizes.append(torch.zeros(n, c.hq, dtype=torch.float64))
        elif n:
            k, v = c.rows(s)
            o, m, z = score_attention(c.q[t:t + n], k, v, ctx - n, c.scale, cap, slopes, window,
                                      None if first is None else first[t:t + n], 0 if prefix is None else int(prefix[s]))
            outs.append(o), means.append(m), sizes.append(z)
        t += n
    return torch.cat(outs), torch.cat(means), torch.cat(sizes)


def check(got, c, want, mean_abs, size, cap=0.0):
    assert bool(torch.isfinite(want).all()) and bool(torch.isfinite(got).all())
    u = torch.finfo(c.dtype).eps / 2
    uq = 0.0 if c.dtype == F32 else u
    ds = 300 * 2.0 ** -24 * size[..., None] + 4 * 2.0 ** -24 * cap
    tol = u * want.abs() + (2 * uq + torch.expm1(2 * ds) + 1e-5) * (mean_abs + want.abs()) + 1e-30
    if c.dtype == F16:
        tol = tol + 2.0 ** -24                              # (results and weights below the normal numbers)
    bad = (got.double() - want).abs() > tol
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} out of tolerance, first at {i}: {got[tuple(i)]} for {want[tuple(i)]}, "
                             f"tolerance {tol[tuple(i)]}")


def cuda(x):
    return None if x is None else x.cuda()


def run_decode(c, cap=0.0, slopes=None, window=0, first=None, **kw):
    q = c.q.cuda()
    out = torch.full_like(q, 7.0)
    lens = torch.tensor(c.ctx, dtype=torch.int32, device="cuda")
    ops.paged_score_decode_attn(out, q, c.k.cuda(), c.v.cuda(), c.table.cuda(), lens, c.scale, cap, cuda(slopes), window, cuda(first),
                                cuda(c.ks), cuda(c.vs), **kw)
    return out.cpu()


def run_prefill(c, cap=0.0, slopes=None, window=0, first=None, prefix=None, **kw):
    q = c.q.cuda()
    out = torch.full_like(q, 7.0)
    lens = torch.tensor(c.ctx, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0] + list(torch.tensor(c.new).cumsum(0)), dtype=torch.int32, device="cuda")
    ops.paged_score_prefill_attn(out, q, c.k.cuda(), c.v.cuda(), c.table.cuda(), lens, cu, c.scale, max(c.new), cap, cuda(slopes),
                                 window, cuda(first), cuda(prefix), cuda(c.ks), cuda(c.vs), **kw)
    return out.cpu()


def slopes_of(hq):
    return torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq)


RULES = {"none": {}, "cap": {"cap": 5.0}, "slopes": {"slopes": True}, "window": {"window": 70}, "window1": {"window": 1},
         "all": {"cap": 30.0, "slopes": True, "window": 100, "first": True}}
BOTH = pytest.mark.routing("balanced", "library")       # decode calls on either schedule
TYPES = [(BF16, None), (F16, None), (F32, None), (BF16, FP8), (F16, FP8)]


def rule(name, c, g):
    r = dict(RULES[name])
    if r.get("slopes"):
        r["slopes"] = slopes_of(c.hq)
    if r.get("first"):
        # some rows begin inside the last window, one row sees nothing
        r["first"] = torch.randint(-3, 60, (c.total,), generator=g, dtype=torch.int32)
        r["first"][-1] = 100000
    return r


DECODE_LENS = [[1], [0, 5, 300, 17], [33, 64, 65, 1000, 16, 15]]


@BOTH
@pytest.mark.parametrize("name", list(RULES))
@pytest.mark.parametrize("dtype,pool", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (6, 1, 256), (28, 4, 128)])
def test_decode(dtype, pool, hq, hkv, d, name):
    g = torch.Generator().manual_seed(5)
    for i, lens in enumerate(DECODE_LENS):
        c = Case(lens, [1] * len(lens), hq, hkv, d, dtype=dtype, pool=pool, seed=i)
        r = rule(name, c, g)
        want, mean_abs, size = expect(c, r.get("cap", 0.0), r.get("slopes"), r.get("window", 0), r.get("first"), None)
        check(run_decode(c, **r), c, want, mean_abs, size)


@BOTH
@pytest.mark.parametrize("bs", [8, 16, 32])
@pytest.mark.parametrize("longest", [0, 100, 4000])
def test_decode_blocks_and_hints(bs, longest):
    """Other block sizes; a hint that is too small cuts nothing."""
    c = Case([700, 3, 250], [1, 1, 1], 8, 2, 64, bs=bs, seed=3)
    want, mean_abs, size = expect(c, 20.0, None, 0, None, None)
    check(run_decode(c, cap=20.0, longest_context=longest), c, want, mean_abs, size)


@BOTH
@pytest.mark.parametrize("dtype,pool", [(BF16, None), (F16, FP8)])
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 128), (16, 2, 64)])
def test_decode_of_many_rows(dtype, pool, hq, hkv, d):
    """Rows that several waves of the balanced schedule share, and waves that cross rows; empty ones among them."""
    lens = [int(x) for x in torch.randint(0, 700, (70,), generator=torch.Generator().manual_seed(1))]
    lens[3] = lens[69] = 0
    c = Case(lens, [1] * 70, hq, hkv, d, dtype=dtype, pool=pool, seed=1)
    first = torch.randint(-5, 400, (70,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    for r in ({"cap": 20.0}, {"window": 129, "slopes": slopes_of(hq)}, {"first": first, "cap": 8.0}):
        want, mean_abs, size = expect(c, r.get("cap", 0.0), r.get("slopes"), r.get("window", 0), r.get("first"), None)
        check(run_decode(c, **r), c, want, mean_abs, size)


def test_decode_of_more_rows_than_the_balanced_schedule_holds():
    lens = [1 + i % 50 for i in range(1100)]
    c = Case(lens, [1] * 1100, 2, 1, 64, seed=1)
    want, mean_abs, size = expect(c, 20.0, None, 30, None, None)
    check(run_decode(c, cap=20.0, window=30), c, want, mean_abs, size)


def visible(c, window=0, first=None, prefix=None):
    out, t = [], 0
    for s, (ctx, n) in enumerate(zip(c.ctx, c.new)):
        seen = torch.zeros(max(ctx, 0), dtype=torch.bool)
        j = torch.arange(max(ctx, 0))
        for i in range(n):
            p = ctx - n + i
            m = (j <= p) | (j < (0 if prefix is None else int(prefix[s])))
            if window:
                m &= p - j < window
            if first is not None:
                m &= j >= int(first[t])
            seen |= m
            t += 1
        out.append(seen)
    return out


@BOTH
@pytest.mark.parametrize("dtype,pool", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_never_looks_at_masked_keys(dtype, pool, d):
    c = Case([300, 47, 129, 64], [1] * 4, 8, 4, d, dtype=dtype, pool=pool, seed=9)
    first = torch.tensor([13, 46, 0, 61], dtype=torch.int32)
    c.poison(visible(c, 75, first))
    want, mean_abs, size = expect(c, 10.0, None, 75, first, None)
    check(run_decode(c, cap=10.0, window=75, first=first), c, want, mean_abs, size)


CHUNKS = {"one": ([1], [1]), "ragged": ([5, 40, 200, 1, 90], [5, 33, 70, 1, 90]), "short_context": ([3, 100, 0], [9, 20, 4]),
          "empty_chunk": ([70, 30, 64], [64, 0, 17]), "long": ([600, 513], [300, 513])}


@pytest.mark.parametrize("name", list(RULES) + ["prefix", "prefix_window_documents"])
@pytest.mark.parametrize("dtype,pool", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (4, 2, 64), (3, 1, 64), (2, 1, 256)])
def test_prefill(dtype, pool, hq, hkv, d, name):
    g = torch.Generator().manual_seed(6)
    for i, (shape, (ctx, new)) in enumerate(CHUNKS.items()):
        if shape == "long" and (dtype != BF16 or hq != 4):
            continue
        c = Case(ctx, new, hq, hkv, d, dtype=dtype, pool=pool, seed=i, rows_behind=3)
        if name.startswith("prefix"):
            r = {"prefix": torch.tensor([50, 7, 1000, 0, 33][:len(ctx)], dtype=torch.int32)}
            if name == "prefix_window_documents":
                r.update(window=40, first=torch.randint(0, 80, (c.total,), generator=g, dtype=torch.int32), slopes=slopes_of(hq))
        else:
            r = rule(name, c, g)
        want, mean_abs, size = expect(c, r.get("cap", 0.0), r.get("slopes"), r.get("window", 0), r.get("first"), r.get("prefix"))
        got = run_prefill(c, **r)
        assert (got[-3:] == 7.0).all(), "rows behind the last sequence were written"
        check(got[:-3], c, want, mean_abs, size)


@pytest.mark.parametrize("dtype,pool", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prefill_never_looks_at_masked_keys(dtype, pool, d):
    """A window behind long priors: keys before every row's window, and beyond the contexts, are not numbers."""
    c = Case([300, 47, 260], [70, 13, 33], 8, 4, d, dtype=dtype, pool=pool, seed=9)
    first = torch.cat([torch.full((n,), f, dtype=torch.int32) for n, f in zip(c.new, (190, 20, 0))])
    c.poison(visible(c, 50, first))
    want, mean_abs, size = expect(c, 10.0, None, 50, first, None)
    check(run_prefill(c, cap=10.0, window=50, first=first), c, want, mean_abs, size)


@pytest.mark.parametrize("d", [64, 128])
def test_masked_keys_of_a_row_that_others_see(d):
    """Keys that one row of a chunk sees and its neighbours do not (the causal edge, the window's edge), infinite: the other rows
    stay finite."""
    c = Case([90], [60], 4, 1, d, dtype=BF16, seed=2)
    blk, off = int(c.table[0, 89 // 16]), 89 % 16
    c.v[blk, :, off] = math.inf                              # the last key: row 59 alone
    first_blk, first_off = int(c.table[0, 0]), 11
    c.v[first_blk, :, first_off] = math.inf                  # key 11: rows at positions up to 30, the first alone
    got = run_prefill(c, window=20)
    assert not torch.isfinite(got[0]).any() and not torch.isfinite(got[59]).any()
    inner = Case([90], [60], 4, 1, d, dtype=BF16, seed=2)
    want, mean_abs, size = expect(inner, 0.0, None, 20, None, None)
    check(got[1:59], inner, want[1:59], mean_abs[1:59], size[1:59])


@BOTH
def test_cut_to_the_table():
    """A context beyond the table is cut to it (as in the plain decode call)."""
    c = Case([200, 64], [1, 1], 4, 2, 128, seed=4, width=13)
    c.table = c.table[:, :10].contiguous()
    want_case = Case([160, 64], [1, 1], 4, 2, 128, seed=4, width=13)
    want_case.q, want_case.table, want_case.k, want_case.v = c.q, c.table, c.k, c.v
    want, mean_abs, size = expect(want_case, 20.0, None, 0, None, None)
    check(run_decode(c, cap=20.0), c, want, mean_abs, size)


@BOTH
def test_bad_table_entries_stay_in_the_pool():
    c = Case([100, 40], [1, 1], 4, 2, 128, seed=4)
    fixed = Case([100, 40], [1, 1], 4, 2, 128, seed=4)
    nb = c.k.shape[0]
    c.table[0, 2], c.table[1, 0] = 10 ** 6, -5
    fixed.table[0, 2], fixed.table[1, 0] = nb - 1, 0
    assert torch.equal(run_decode(c, cap=20.0), run_decode(fixed, cap=20.0))
    c.new = fixed.new = [7, 3]
    c.total = 10
    c.q = fixed.q = torch.randn(10, 4, 128).bfloat16()
    assert torch.equal(run_prefill(c, cap=20.0), run_prefill(fixed, cap=20.0))


@BOTH
def test_saturated_caps():
    """Scores far beyond the cap on both sides, and a cap so small that all weights are alike."""
    c = Case([500], [1], 8, 2, 128, seed=8)
    c.q = c.q * 40
    for cap in (50.0, 1e-3, 200.0):
        want, mean_abs, size = expect(c, cap, None, 0, None, None)
        # (the products' rounding moves a score by no more than twice the cap)
        check(run_decode(c, cap=cap), c, want, mean_abs, size.clamp(max=2 * cap))
        p = Case([500], [37], 8, 2, 128, seed=8)
        p.q = p.q * 40
        want, mean_abs, size = expect(p, cap, None, 0, None, None)
        check(run_prefill(p, cap=cap), p, want, mean_abs, size.clamp(max=2 * cap))


@BOTH
def test_plain_rule_agrees_with_the_plain_operator():
    """No rule at all is causal attention, decode and chunks."""
    c = Case([700, 90, 33], [1, 1, 1], 8, 2, 128, seed=11)
    q, k, v, t = c.q.cuda(), c.k.cuda(), c.v.cuda(), c.table.cuda()
    lens = torch.tensor(c.ctx, dtype=torch.int32, device="cuda")
    plain = torch.empty_like(q)
    ops.paged_decode_attn(plain, q, k, v, t, lens, c.scale)
    want, mean_abs, size = expect(c, 0.0, None, 0, None, None)
    check(plain.cpu(), c, want, mean_abs, size)
    check(run_decode(c), c, want, mean_abs, size)


def test_ops_refusals():
    c = Case([40], [1], 4, 2, 128)
    q, k, v, t = c.q.cuda(), c.k.cuda(), c.v.cuda(), c.table.cuda()
    lens = torch.tensor([40], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    call = lambda **kw: ops.paged_score_decode_attn(out, q, k, v, t, lens, 0.1, **kw)
    with pytest.raises(RuntimeError, match="slopes must be"):
        call(slopes=torch.ones(3, device="cuda"))
    with pytest.raises(RuntimeError, match="slopes is on"):
        call(slopes=torch.ones(4))
    with pytest.raises(RuntimeError, match="first_keys"):
        call(first_keys=torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="window"):
        call(window=-1)
    with pytest.raises(RuntimeError, match="softcap"):
        call(softcap=-2.0)
    with pytest.raises(RuntimeError, match="workspace"):
        big = torch.zeros(1, 256, dtype=torch.int32, device="cuda")
        ops.paged_score_decode_attn(out, q, k, v, big, lens, 0.1, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="prefix_lens"):
        ops.paged_score_prefill_attn(out, q, k, v, t, lens, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 0.1,
                                     prefix_lens=torch.zeros(2, dtype=torch.int32, device="cuda"))


def wide(c, g):
    """Every term of the rule, and a window that is worth dividing."""
    return {**rule("all", c, g), "window": 900}


FEW = [([700, 40, 0, 1333], [33, 40, 0, 2], 8, 2, 128, 16), ([2100], [17], 8, 8, 64, 16), ([900, 1800], [5, 70], 6, 2, 256, 16)]


@pytest.mark.parametrize("shape", FEW, ids=["ragged", "one", "d256"])
@pytest.mark.parametrize("types", [(BF16, None), (F16, FP8), (F32, None)], ids=["bf16", "f16-fp8", "f32"])
@pytest.mark.parametrize("name", list(RULES) + ["wide"])
def test_prefill_few_rows_divides_their_keys(shape, types, name):
    """With a workspace the keys of few rows are divided among workgroups, without one they are not: both are right, and what the
    keys that no row sees hold changes neither."""
    ctx, new, hq, hkv, d, bs = shape
    c = Case(ctx, new, hq, hkv, d, bs, *types, seed=11, rows_behind=3)
    g = torch.Generator().manual_seed(5)
    r = wide(c, g) if name == "wide" else rule(name, c, g)
    full = {"cap": 0.0, "slopes": None, "window": 0, "first": None, **r}
    prefix = torch.tensor([300] * len(ctx), dtype=torch.int32) if name in ("all", "wide") else None
    want, mean, size = expect(c, full["cap"], full["slopes"], full["window"], full["first"], prefix)
    n = sum(new)
    lib = _lib.load()
    q, lens = c.q.cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device="cuda")
    k, v, table = c.k.cuda(), c.v.cuda(), c.table.cuda()
    t = [cuda(x) for x in (c.ks, c.vs, full["slopes"], full["first"], prefix)]
    ptr = lambda x: None if x is None else x.data_ptr()
    qd, kd = ops._DT[c.dtype], ops._DT[c.pool_dtype]
    need = lib.aicomp_paged_score_workspace_bytes(len(ctx), c.total, max(new), hq, hkv, d, bs, table.shape[1], qd, kd, full["window"], 0)
    assert need > 0 or full["window"]                                       # (a short window is one part)
    for own in (need, 0):
        ws = torch.full((max(own, 16),), 0xff, dtype=torch.uint8, device="cuda")              # (not a number, read as float)
        out = torch.full_like(q, 7.0)
        rc = lib.aicomp_paged_score_attn(
            out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), table.stride(0), lens.data_ptr(), cu.data_ptr(),
            len(ctx), c.total, max(new), hq, hkv, d, bs, table.shape[1], k.shape[0], c.scale, qd, kd, ptr(t[0]), ptr(t[1]),
            full["cap"], ptr(t[2]), full["window"], ptr(t[3]), ptr(t[4]), 0, ws.data_ptr() if own else None, own,
            torch.cuda.current_stream().cuda_stream)
        _lib.check(rc, lib)
        got = out.cpu()
        assert bool((got[n:] == 7.0).all())
        check(got[:n], c, want, mean, size)


def test_divided_keys_that_are_not_finite():
    """Infinite values of keys that only neighbours see: in the last rows' parts, every row of the call has its own keys."""
    c = Case([2000], [40], 8, 2, 128, seed=3)
    for j in (5, 700, 1970, 1999):                                          # (visible to some of the 40 rows)
        blk = int(c.table[0, j // 16])
        c.v[blk, :, j % 16] = math.inf
    first = torch.full((40,), 6, dtype=torch.int32)                         # key 5: to no row
    first[7:20] = 701                                                       # key 700: not to these
    first[20:30] = 1971                                                     # key 1970: not to these
    got = run_prefill(c, 5.0, first=first)[:40].double()
    clean = Case([2000], [40], 8, 2, 128, seed=3)
    want, mean, size = expect(clean, 5.0, None, 0, first, None)
    sees = torch.zeros(40, dtype=torch.bool)
    for j in (5, 700, 1970, 1999):
        pos = torch.arange(1960, 2000)
        sees |= (first <= j) & (j <= pos)
    assert bool(sees.any()) and not bool(sees.all())
    assert bool((got[sees] == math.inf).all())
    check(got[~sees], c, want[~sees], mean[~sees], size[~sees])


def test_divided_chunks_in_two_graphs():
    """Two captured calls of divided keys, replayed side by side on two streams: each has scratch of its own."""
    cases = [Case([1500, 900], [30, 9], 8, 2, 128, seed=s) for s in (21, 22)]
    want, graphs, outs, keep = [], [], [], []
    stream = torch.cuda.Stream()
    for c in cases:
        want.append(run_prefill(c, 5.0))
        q, k, v, table = c.q.cuda(), c.k.cuda(), c.v.cuda(), c.table.cuda()
        lens = torch.tensor(c.ctx, dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, 30, 39], dtype=torch.int32, device="cuda")
        out = torch.full_like(q, 7.0)
        keep.append((q, k, v, table, lens, cu))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            ops.paged_score_prefill_attn(out, q, k, v, table, lens, cu, c.scale, 30, 5.0)
        graphs.append(g), outs.append(out)
    for _ in range(3):
        for out in outs:
            out.fill_(7.0)
        torch.cuda.synchronize()
        side = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(10):
            for g, s in zip(graphs, side):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out.cpu(), w)


@pytest.mark.parametrize("types", TYPES, ids=["bf16", "f16", "f32", "bf16-fp8", "f16-fp8"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cap", [1024.0, 0.01])
def test_largest_and_small_caps(types, d, cap):
    """A cap so large that it changes little, and one so small that nearly all scores are at it."""
    c = Case([300, 65, 1], [1, 1, 1], 8, 2, d, 16, *types, seed=31)
    want, mean, size = expect(c, cap, None, 0, None, None)
    check(run_decode(c, cap), c, want, mean, size, cap)
    c = Case([300, 65, 40], [70, 65, 1], 8, 2, d, 16, *types, seed=32)
    want, mean, size = expect(c, cap, None, 0, None, None)
    check(run_prefill(c, cap), c, want, mean, size, cap)


# calls that take 128 rows to a workgroup: (query heads, KV heads, sequences' new tokens, tokens before them)
LARGE = {64: (16, 4, [300] * 27 + [37, 1, 129], 70), 128: (16, 4, [300] * 14 + [37, 1, 129], 100), 256: (8, 2, [300] * 17 + [37, 1, 65], 40)}


def large_case(d, dtype, pool, seed):
    hq, hkv, new, before = LARGE[d]
    return Case([n + before for n in new], new, hq, hkv, d, dtype=dtype, pool=pool, seed=seed, rows_behind=2)


def one_by_one(c, **r):
    """The same rows, a call for each sequence: few workgroups, 64 rows to each."""
    outs, t = [], 0
    for s, n in enumerate(c.new):
        one = Case.__new__(Case)
        one.__dict__.update(c.__dict__)
        one.ctx, one.new, one.table, one.q, one.total = [c.ctx[s]], [n], c.table[s:s + 1].contiguous(), c.q[t:t + n], n
        part = {**r}
        for name in ("first", "prefix"):
            if part.get(name) is not None:
                part[name] = part[name][t:t + n] if name == "first" else part[name][s:s + 1]
        outs.append(run_prefill(one, **part))
        t += n
    return torch.cat(outs)


@pytest.mark.parametrize("name", ["none", "cap", "slopes", "window", "all"])
@pytest.mark.parametrize("dtype,pool", [(BF16, None), (F16, None), (BF16, FP8), (F32, None)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_large_chunks(dtype, pool, d, name):
    """Every row against the calls of single sequences, rows here and there against float64."""
    c = large_case(d, dtype, pool, 41)
    g = torch.Generator().manual_seed(8)
    r = rule(name, c, g)
    if name == "all":
        r["prefix"] = torch.full((len(c.new),), 90, dtype=torch.int32)
    got = []
    names = [n for n in kernels_of(lambda: got.append(run_prefill(c, **r))) if "score_prefill" in n]
    wide = dtype != F32 and not (d == 64 and (pool is not None or "slopes" in r))
    assert len(names) == 1 and (f", 2, {d}," in names[0]) == wide, names
    got = got[0]
    total = sum(c.new)
    assert bool((got[total:] == 7.0).all())
    other = one_by_one(c, **r)
    starts = [sum(c.new[:s]) for s in range(len(c.new))]
    picks = sorted({t for s, n in enumerate(c.new[-4:], len(c.new) - 4) for t in (starts[s], starts[s] + n // 2, starts[s] + n - 1)} |
                   set(torch.randint(0, total, (40,), generator=g).tolist()))
    wants, means, sizes = [], [], []
    for t in picks:
        s = max(i for i, b in enumerate(starts) if b <= t)
        k, v = c.rows(s)
        w, m, z = score_attention(c.q[t:t + 1], k, v, c.ctx[s] - c.new[s] + t - starts[s], c.scale, r.get("cap", 0.0), r.get("slopes"),
                                  r.get("window", 0), None if r.get("first") is None else r["first"][t:t + 1],
                                  0 if r.get("prefix") is None else int(r["prefix"][s]))
        wants.append(w), means.append(m), sizes.append(z)
    want, mean, size = torch.cat(wants), torch.cat(means), torch.cat(sizes)
    check(got[picks], c, want, mean, size)
    check(other[picks], c, want, mean, size)
    # (two right results differ by two tolerances at most: of |v| up to 6 the mean is at most 6 and so is the result, 9 for both; sizes
    # up to 30 give e^(2 ds) - 1 = 1.08e-3)
    u = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    tol = 2 * (u * other.double().abs() + (2 * u + 1.1e-3) * 9.0)
    assert bool(((got[:total].double() - other.double()).abs() <= tol).all())


@pytest.mark.parametrize("d", [64, 128])
def test_large_chunks_with_values_that_are_not_finite(d):
    """Keys of some rows alone, infinite, in a call of 128 rows to a workgroup: as in the calls of single sequences."""
    c = large_case(d, BF16, None, 43)
    for s in range(0, len(c.new) - 3, 3):
        for j in (c.ctx[s] - 1, 50 + s, c.ctx[s] // 2):
            c.v[int(c.table[s, j // 16]), :, j % 16] = math.inf
    r = {"cap": 5.0, "window": 40}
    got, other = run_prefill(c, **r)[:sum(c.new)], one_by_one(c, **r)
    finite = torch.isfinite(got)
    assert torch.equal(finite, torch.isfinite(other)) and not bool(finite.all()) and bool(finite.any())
    u = 2.0 ** -8
    tol = 2 * (u * other.double().abs() + (2 * u + 1.1e-3) * 9.0)
    assert bool(((got.double() - other.double()).abs() <= tol)[finite].all())


@pytest.mark.routing("library")
@pytest.mark.parametrize("name", ["cap", "slopes", "all"])
@pytest.mark.parametrize("dtype,pool,hq,hkv,d,longest", [
    (BF16, None, 8, 2, 128, 600), (F16, None, 4, 4, 128, 513), (F16, FP8, 16, 2, 128, 640), (BF16, None, 8, 2, 64, 1100),
    (F32, None, 8, 2, 64, 640), (F32, None, 16, 2, 64, 600), (F32, None, 8, 2, 128, 400), (F32, None, 16, 2, 128, 448)])
def test_decode_rows_of_eight_waves(decode_routing, dtype, pool, hq, hkv, d, longest, name):
    """Rows that are whole and long in few workgroups."""
    c = Case([longest, 1, longest - 17, 65, 255, 256, 257], [1] * 7, hq, hkv, d, dtype=dtype, pool=pool, seed=51)
    g = torch.Generator().manual_seed(9)
    r = rule(name, c, g)
    if name == "all":
        r["window"] = longest - 40
    tile = (64 if d == 64 else 32) // (2 if dtype == F32 else 1)    # a window reaches into a tile more; eight waves beyond 16 tiles
    waves = 8 if min(longest, r.get("window", longest) + tile - 1) > 16 * tile else 4
    assert waves == 8 or (longest, name) == (513, "all")
    got = []
    names = [n for n in kernels_of(lambda: got.append(run_decode(c, longest_context=longest, **r))) if "paged_decode" in n]
    assert len(names) == 1 and f"{waves}, false>" in names[0] and "Ruled" in names[0], names
    want, mean, size = expect(c, r.get("cap", 0.0), r.get("slopes"), r.get("window", 0), r.get("first"), None)
    check(got[0], c, want, mean, size)
