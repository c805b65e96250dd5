"""Blocks whose bytes lie beyond 2^32 of a pool, and calls whose rows all see nothing: attention by a score rule, the append of normed
heads and block copies do there what they do with the same blocks at a pool's start."""
import pytest
import torch

from aicomp_amd import ops
from test_gpu_score_attn import BF16, F16, F32, FP8, Case, run_decode, run_prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,pool,hq,hkv,d", [(BF16, None, 8, 8, 128), (F16, FP8, 16, 8, 128), (F32, None, 8, 8, 128), (BF16, None, 8, 8, 256)])
def test_blocks_beyond_32_bits(device, dtype, pool, hq, hkv, d):
    pool = pool or dtype
    block = hkv * 16 * d * torch.empty((), dtype=pool).element_size()
    nb = 2 ** 32 // block + 300
    far = nb - 130                                          # 130 blocks there, of a sequence of 1500 tokens and one of 520
    g = torch.Generator(device=device).manual_seed(3)
    mk = lambda *s: torch.randn(*s, generator=g, device=device)
    near = [(mk(nb - far, hkv, 16, d) * (40 if pool == FP8 else 1)).clamp(-448, 448).to(pool) for _ in range(2)]
    pools = [torch.empty(nb, hkv, 16, d, dtype=pool, device=device) for _ in range(2)]
    for p, x in zip(pools, near):
        p.view(torch.uint8)[far:] = x.view(torch.uint8)
    scale = torch.full((hkv,), 0.025, device=device)
    table = torch.full((2, 94), -1, dtype=torch.int32, device=device)
    order = torch.randperm(nb - far, generator=g, device=device).to(torch.int32)
    table[0, :94], table[1, :33] = order[:94], order[94:127]
    lens = torch.tensor([1500, 520], dtype=torch.int32, device=device)
    cu = torch.tensor([0, 40, 57], dtype=torch.int32, device=device)
    q, slopes = mk(57, hq, d).to(dtype), torch.rand(hq, generator=g, device=device)
    key, value = (mk(2, hkv, d).to(dtype) for _ in range(2))
    w, (cos, sin) = 1 + 0.1 * mk(2, d), ops.rotary_pair_tables(torch.rand(d // 2, generator=g, device=device), 2000)
    pos = lens.long() - 1
    results = []
    for kp, vp, shift in ((near[0].clone(), near[1].clone(), 0), (*pools, far)):
        t = torch.where(table >= 0, table + shift, table)
        slots = t[torch.arange(2, device=device), pos // 16].long() * 16 + pos % 16
        rows = ops.qk_norm_rope_kv_append(q[:2], key, value, w[0], w[1], cos, sin, pos, kp, vp, slots, k_scale=scale, v_scale=scale,
                                          query_out=torch.empty_like(q[:2]))
        ops.copy_blocks([kp, vp], torch.tensor([[shift, shift + 127], [shift + 1, shift + 129]], device=device))
        a, b = torch.empty_like(rows), torch.empty_like(q)
        ops.paged_score_decode_attn(a, rows, kp, vp, t, lens, d ** -0.5, 30.0, slopes, k_scale=scale, v_scale=scale)
        ops.paged_score_prefill_attn(b, q, kp, vp, t, lens, cu, d ** -0.5, 40, 30.0, slopes, k_scale=scale, v_scale=scale)
        assert bool(torch.isfinite(a).all()) and bool(torch.isfinite(b).all())
        results.append((rows, a, b, kp[shift:].view(torch.uint8), vp[shift:].view(torch.uint8)))
    for x, y in zip(*results):
        assert torch.equal(x, y)
    assert torch.equal(results[0][3][127], results[0][3][0]) and torch.equal(results[1][3][129], results[1][3][1])


@pytest.mark.routing("balanced", "library")
@pytest.mark.parametrize("dtype,pool,hq,hkv,d,bs", [(BF16, None, 8, 2, 128, 16), (F16, FP8, 4, 4, 64, 16), (F32, None, 4, 1, 64, 16),
                                                   (F32, None, 16, 2, 128, 16), (BF16, None, 4, 2, 256, 16), (BF16, None, 8, 2, 128, 32)])
def test_calls_whose_rows_all_see_nothing(decode_routing, dtype, pool, hq, hkv, d, bs):
    for ctx, first in (([2000, 70, 1], 5000), ([0, 0, 0], 0), ([0, -3, 0], 0)):
        c = Case(ctx, [1] * 3, hq, hkv, d, bs=bs, dtype=dtype, pool=pool, seed=1)
        starts = torch.full((3,), first, dtype=torch.int32)
        assert not bool(run_decode(c, cap=20.0, first=starts).any())
        if min(ctx) >= 0:
            new = [min(x, 40) if first else 5 for x in ctx]                      # (no context: chunks that are longer than it)
            c = Case(ctx, new, hq, hkv, d, bs=bs, dtype=dtype, pool=pool, seed=1)
            assert not bool(run_prefill(c, cap=20.0, first=torch.full((sum(new),), first, dtype=torch.int32)).any())
