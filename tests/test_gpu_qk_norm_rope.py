"""Normed and rotated heads appended to the pools, and block copies, against float64 and exact copies.

Tolerance of a normed, rotated element: the result is rounded once to its type (eps / 2 relative); before that float32 sums of D
squares, a reciprocal root, two products per element and the rotation's two products and a sum, less than D + 8 roundings of 2^-24
relative to |a| + |b| of the pair (a sum of D positive terms in any order is off by at most D half steps).
"""
import pytest
import torch

from aicomp_amd import ops
from oracle.score_oracle import norm_rope

pytestmark = pytest.mark.gpu
BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def inputs(T, hq, hkv, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, (hq + 2 * hkv) * d, generator=g) * 3).to(dtype).cuda()        # slices of one projection
    q, k, v = x[:, :hq * d].view(T, hq, d), x[:, hq * d:(hq + hkv) * d].view(T, hkv, d), x[:, (hq + hkv) * d:].view(T, hkv, d)
    w = 1 + 0.3 * torch.randn(2, d, generator=g)
    return g, q, k, v, w[0].contiguous().cuda(), w[1].contiguous().cuda()


def close(got, want, d, dtype, rotated, interleaved):
    """``want`` float64 of the norm and rotation; the partner's size enters the tolerance."""
    u = torch.finfo(dtype).eps / 2
    pair = want.abs().clone()
    if rotated:
        r = want[..., :rotated]
        if interleaved:
            both = r.reshape(*r.shape[:-1], rotated // 2, 2).abs().sum(-1, keepdim=True).expand(*r.shape[:-1], rotated // 2, 2)
            pair[..., :rotated] = both.reshape(r.shape)
        else:
            both = r[..., :rotated // 2].abs() + r[..., rotated // 2:].abs()
            pair[..., :rotated] = torch.cat((both, both), -1)
    # a pair's turned values are at most sqrt(2) times smaller in sum than what they came from
    tol = u * want.abs() + (d + 8) * 2.0 ** -24 * 1.5 * pair + (2.0 ** -25 if dtype == F16 else 0)
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), (got.double() - want).abs().max())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d,rotary", [(128, 128), (128, 32), (64, 64), (64, 0), (256, 256), (96, 48), (80, 32), (16, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_append(dtype, d, rotary, interleaved):
    for T, hq, hkv in ((1, 4, 1), (7, 6, 2), (300, 9, 3)):
        g, q, k, v, qw, kw = inputs(T, hq, hkv, d, dtype, seed=T)
        inv = 1.0 / (10000.0 ** (torch.arange(0, rotary, 2).float() / max(rotary, 1)))
        cos, sin = ops.rotary_pair_tables(inv, 500, device="cuda") if rotary else (None, None)
        pos = torch.randint(0, 500, (T,), generator=g)
        nb = -(-T // 16) + 2
        slots = torch.randperm(nb * 16, generator=g)[:T]
        kp, vp = torch.full((nb, hkv, 16, d), 3.0, dtype=dtype, device="cuda"), torch.full((nb, hkv, 16, d), 3.0, dtype=dtype, device="cuda")
        out = torch.empty(T, hq, d, dtype=dtype, device="cuda")
        before = q.clone()
        got = ops.qk_norm_rope_kv_append(q, k, v, qw, kw, cos, sin, pos.cuda() if rotary else None, kp, vp, slots.cuda(), eps=1e-5,
                                         interleaved=interleaved, query_out=out)
        assert got is out and torch.equal(q, before)
        angles = pos[:, None].double() * inv.double() if rotary else None
        close(out.cpu(), norm_rope(q.cpu(), qw.cpu(), 1e-5, angles, interleaved), d, dtype, rotary, interleaved)
        rows = lambda pool: pool.cpu().transpose(1, 2).reshape(nb * 16, hkv, d)
        close(rows(kp)[slots], norm_rope(k.cpu(), kw.cpu(), 1e-5, angles, interleaved), d, dtype, rotary, interleaved)
        assert torch.equal(rows(vp)[slots], v.cpu())
        rest = torch.ones(nb * 16, dtype=torch.bool)
        rest[slots] = False
        assert (rows(kp)[rest] == 3).all() and (rows(vp)[rest] == 3).all()
        # in place
        ops.qk_norm_rope_kv_append(q, k, v, qw, kw, cos, sin, pos.cuda() if rotary else None, kp, vp, slots.cuda(), eps=1e-5,
                                   interleaved=interleaved)
        assert torch.equal(q, out)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_fp8_pools(dtype):
    """The codes are those of the float32 result: within half a step of e4m3 (2^-4 relative, 2^-10 below the normal numbers)."""
    T, hq, hkv, d = 50, 8, 2, 128
    g, q, k, v, qw, kw = inputs(T, hq, hkv, d, dtype)
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2).float() / d))
    cos, sin = ops.rotary_pair_tables(inv, 100, device="cuda")
    pos, slots = torch.arange(T), torch.randperm(80, generator=g)[:T]
    ks, vs = torch.tensor([0.01, 0.02]), torch.tensor([0.03, 0.02])
    kp, vp = torch.zeros(5, hkv, 16, d, dtype=FP8, device="cuda"), torch.zeros(5, hkv, 16, d, dtype=FP8, device="cuda")
    ops.qk_norm_rope_kv_append(q, k, v, qw, kw, cos, sin, pos.cuda(), kp, vp, slots.cuda(), k_scale=ks.cuda(), v_scale=vs.cuda())
    want_k = norm_rope(k.cpu(), kw.cpu(), 1e-6, pos[:, None].double() * inv.double(), False) / ks.double()[:, None]
    want_v = v.cpu().double() / vs.double()[:, None]
    for pool, want in ((kp, want_k), (vp, want_v)):
        got = pool.cpu().float().double().transpose(1, 2).reshape(80, hkv, d)[slots]
        want = want.clamp(-448, 448)
        assert ((got - want).abs() <= 2.0 ** -4 * want.abs() * (1 + 1e-3) + 2.0 ** -10 * (1 + 1e-3)).all()


def test_padding_rows_and_far_positions():
    T, hq, hkv, d = 6, 4, 2, 64
    g, q, k, v, qw, kw = inputs(T, hq, hkv, d, BF16)
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2).float() / d))
    cos, sin = ops.rotary_pair_tables(inv, 40, device="cuda")
    pos = torch.tensor([0, 39, 40, -1, 5, 6])                       # 40 and -1 have no row: left alone
    slots = torch.tensor([3, 47, 5, 6, -1, 48])                     # -1 and 48 are outside: the query alone
    kp, vp = (torch.full((3, hkv, 16, d), 3.0, dtype=BF16, device="cuda") for _ in range(2))
    out = torch.full((T, hq, d), 7.0, dtype=BF16, device="cuda")
    ops.qk_norm_rope_kv_append(q, k, v, qw, kw, cos, sin, pos.cuda(), kp, vp, slots.cuda(), query_out=out)
    want = norm_rope(q.cpu(), qw.cpu(), 1e-6, pos[:, None].double() * inv.double(), False)
    keep = torch.tensor([0, 1, 4, 5])
    close(out.cpu()[keep], want[keep], d, BF16, d, False)
    assert (out[2:4] == 7).all()
    written = (kp.cpu().transpose(1, 2).reshape(48, -1) != 3).any(1)
    assert torch.nonzero(written).flatten().tolist() == [3, 47]


def test_rotation_or_norm_alone():
    T, hq, hkv, d = 9, 4, 2, 128
    g, q, k, v, qw, kw = inputs(T, hq, hkv, d, BF16)
    inv = 1.0 / (10000.0 ** (torch.arange(0, 64, 2).float() / 64))
    cos, sin = ops.rotary_pair_tables(inv, T, device="cuda")
    slots = torch.arange(T).cuda()
    kp, vp = (torch.zeros(1, hkv, 16, d, dtype=BF16, device="cuda") for _ in range(2))
    out = torch.empty_like(q)
    ops.qk_norm_rope_kv_append(q, k, v, None, kw, cos, sin, None, kp, vp, slots, query_out=out)      # (no positions: row t)
    angles = torch.arange(T)[:, None].double() * inv.double()
    close(out.cpu(), norm_rope(q.cpu(), None, 0, angles, False), d, BF16, 64, False)
    close(kp.cpu()[0].transpose(0, 1)[:T], norm_rope(k.cpu(), kw.cpu(), 1e-6, angles, False), d, BF16, 64, False)


def test_refusals():
    g, q, k, v, qw, kw = inputs(3, 4, 2, 64, BF16)
    kp = torch.zeros(1, 2, 16, 64, dtype=BF16, device="cuda")
    slots = torch.arange(3).cuda()
    call = lambda **kw_: ops.qk_norm_rope_kv_append(**{**dict(
        query=q, key=k, value=v, q_weight=qw, k_weight=kw, cos=None, sin=None, positions=None, k_pool=kp, v_pool=kp,
        slot_mapping=slots), **kw_})
    table = torch.zeros(10, 32, device="cuda")
    with pytest.raises(RuntimeError, match="q_weight"):
        call(q_weight=qw.bfloat16())
    with pytest.raises(RuntimeError, match="come together"):
        call(cos=table)
    with pytest.raises(RuntimeError, match="float32"):
        call(cos=table.bfloat16(), sin=table.bfloat16())
    with pytest.raises(RuntimeError, match="rotate 128"):
        call(cos=torch.zeros(10, 64, device="cuda"), sin=torch.zeros(10, 64, device="cuda"))
    with pytest.raises(RuntimeError, match="one row per token"):
        call(cos=table[:2], sin=table[:2])
    with pytest.raises(RuntimeError, match="positions"):
        call(cos=table, sin=table, positions=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="eps"):
        call(eps=-1.0)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        call(cos=torch.zeros(10, 4, device="cuda"), sin=torch.zeros(10, 4, device="cuda"))
    with pytest.raises(RuntimeError, match="slot_mapping"):
        call(slot_mapping=slots[:2])


@pytest.mark.parametrize("dtype,hkv,bs,d", [(BF16, 8, 16, 128), (F32, 1, 16, 64), (FP8, 3, 16, 64), (BF16, 1, 1, 10), (FP8, 1, 3, 7)])
def test_copy_blocks(dtype, hkv, bs, d):
    g = torch.Generator().manual_seed(1)
    nb = 37
    for pools_n, n in ((1, 1), (6, 18), (130, 3)):
        pools = [torch.randint(0, 255, (nb, hkv, bs, d * torch.empty((), dtype=dtype).element_size()), generator=g,
                               dtype=torch.uint8).cuda().view(dtype) for _ in range(pools_n)]
        order = torch.randperm(nb, generator=g)[:2 * n]
        pairs = order.view(n, 2).contiguous()
        raw = lambda t: t.view(torch.uint8).cpu()
        want = [raw(t).clone() for t in pools]
        for t in want:
            for a, b in pairs.tolist():
                t[b] = t[a]
        copies = [t.clone() for t in pools]
        ops.copy_blocks(pools, pairs.cuda())
        assert all(torch.equal(raw(t), w) for t, w in zip(pools, want))
        ops.copy_blocks(copies, pairs)                               # pairs on the host
        assert all(torch.equal(raw(t), w) for t, w in zip(copies, want))


def test_copy_blocks_beyond_the_pool_are_skipped_and_host_pairs_checked():
    pool = torch.arange(4 * 16, dtype=F32, device="cuda").view(4, 1, 16, 1)
    before = pool.clone()
    ops.copy_blocks([pool], torch.tensor([[0, 4], [-1, 1], [2, 2], [1 << 40, 3]], device="cuda"))
    assert torch.equal(pool, before)
    for pairs, match in (([[0, 4]], "outside"), ([[0, 2], [1, 2]], "same target"), ([[0, 1], [1, 2]], "target of one")):
        with pytest.raises(RuntimeError, match=match):
            ops.copy_blocks([pool], torch.tensor(pairs))
    with pytest.raises(RuntimeError, match="alike"):
        ops.copy_blocks([pool, pool[:2]], torch.tensor([[0, 1]]))
    ops.copy_blocks([pool], torch.empty(0, 2, dtype=torch.int64))
    assert torch.equal(pool, before)
