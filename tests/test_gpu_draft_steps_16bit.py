"""Steps of drafted tokens in the types that models are served in: prompts, trees, kept rows and plain steps after them, through the
planner, the backends and the step call, one layer against float64 over the text that should be cached."""
import math

import pytest
import torch

from aicomp_amd import ops
from aicomp_amd.block_manager import StepPlanner, paged_attention_step
from aicomp_amd.generation import LatentAttentionBackend, PagedAttentionBackend
from oracle.rows_oracle import masked_attention, tree_visible
from test_gpu_latent import attention_bound, check

pytestmark = pytest.mark.gpu
BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn

# a step: prompts and plain tokens (None), or trees of drafts and which of them stay
PLAY = [None, None,
        ({"a": [-1, 0, 0, 2, 1, 3, 3], "b": [-1], "c": [-1, 0, 0, 0]}, {"a": [0, 2, 3, 6], "b": [0], "c": [0, 3]}),
        None,
        ({"c": [-1] + [i // 2 for i in range(39)], "a": [-1, 0, 1, 2, 3]}, {"c": [0, 2, 5, 12, 25], "a": [0, 1, 2]}),
        ({"b": [-1, 0, 0]}, {}),
        None, None]


def planner_of(device):
    p = StepPlanner(num_blocks=40, max_seqs=4, max_seq_len=256, max_num_batched_tokens=128, prefill_chunk=64, device=device, check_plans=True)
    for sid, n in (("a", 40), ("b", 90), ("c", 13)):
        p.add_request(sid, n)
    return p


def play(planner, step, keep):
    """``step(plan, trees)`` and ``keep(moved, kept)`` through the whole of it."""
    for what in PLAY:
        if what is None:
            step(planner.schedule(), {})
            continue
        plan = planner.schedule_drafts(what[0])
        step(plan, what[0])
        keep(planner.keep_drafts(plan, what[1]), what[0], what[1])


def plain_bound(want, dtype):
    """Of the calls beside the trees, as their own tests hold them: 1e-2 or 2e-2 of the value in 16 bits, 1e-5 of either in float32."""
    return torch.full_like(want, 1e-5) if dtype == F32 else (2e-2 * want.abs()).clamp(min=1e-2)


def fed(text, rows):
    """The cached text of a sequence with these rows behind it."""
    return rows if text is None else torch.cat((text, rows))


TYPES = [(BF16, None), (F16, None), (BF16, FP8), (F16, FP8), (F32, None)]


@pytest.mark.parametrize("via", ["backend", "step"])
@pytest.mark.parametrize("dtype,pool", TYPES)
def test_drafts_over_pools(device, dtype, pool, via):
    hq, hkv, d, g = 8, 2, 64, torch.Generator().manual_seed(51)
    planner, backend = planner_of(device), PagedAttentionBackend(1, 40, hkv, d, dtype, device, kv_dtype=pool)
    ks, vs = [torch.rand(hkv, generator=g) * 0.01 + 0.01 for _ in range(2)] if pool else (None, None)
    if pool:
        backend.set_scales(0, ks, vs)
    kp, vp = backend.k_pools[0], backend.v_pools[0]
    texts = {}

    def step(plan, trees):
        T = plan.total_new_tokens
        q, k, v = [torch.randn(T, h, d, generator=g).to(dtype) for h in (hq, hkv, hkv)]
        dev = [x.to(device) for x in (q, k, v)]
        if via == "backend":
            backend.begin_step(plan)
            out = backend.attend(0, *dev)
        else:
            out = paged_attention_step(plan, torch.empty_like(dev[0]), *dev, kp, vp, backend.scale, backend.k_scales[0], backend.v_scales[0])
        out, slot = out.cpu(), torch.from_numpy(plan.host_slot_mapping.copy())
        cached = []
        for p, x, s in ((kp, k, ks), (vp, v, vs)):
            have = p[slot.to(device) // 16, :, slot.to(device) % 16].cpu().double()
            if s is None:
                assert torch.equal(have, x.double())
            else:
                have = have * s.double()[:, None]                  # (half a step of a code, 2^-4, or of the smallest ones)
                assert bool(((have - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * s.double()[:, None]).all())
            cached.append(have)
        cu = plan.host_cu_q_lens
        for r, sid in enumerate(plan.seq_ids):
            mine, n = slice(int(cu[r]), int(cu[r + 1])), int(cu[r + 1] - cu[r])
            texts[sid] = [fed(t, x[mine]) for t, x in zip(texts.get(sid, (None, None)), cached)]
            c = len(texts[sid][0])
            assert c == int(plan.host_context_lens[r])
            want, mean_abs, size = masked_attention(q[mine], *texts[sid], tree_visible(c, n, trees.get(sid)), backend.scale)
            check(out[mine], want, attention_bound(want, mean_abs, size, d, dtype) if trees else plain_bound(want, dtype))

    def keep(moved, trees, kept):
        for sid, tree in trees.items():
            n, stay = len(tree), kept.get(sid, [])
            texts[sid] = [torch.cat((t[:-n], t[-n:][stay])) for t in texts[sid]]
        backend.keep_drafts(moved)

    play(planner, step, keep)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rotated_drafts(device, dtype, interleaved):
    """Rotated by their places in the text: the rows and queries that the rotation alone gives at those places, then as above."""
    hq, hkv, d, g = 8, 2, 128, torch.Generator().manual_seed(52)
    inv = 1.0 / 10000.0 ** (torch.arange(0, d, 2, dtype=torch.float32) / d)
    planner = planner_of(device)
    backend = PagedAttentionBackend(1, 40, hkv, d, dtype, device, inv_freq=inv, max_positions=256, interleaved=interleaved)
    scratch = [torch.zeros_like(p) for p in (backend.k_pools[0], backend.v_pools[0])]
    texts = {}

    def step(plan, trees):
        T = plan.total_new_tokens
        q, k, v = [torch.randn(T, h, d, generator=g).to(dtype).to(device) for h in (hq, hkv, hkv)]
        cu, where = plan.host_cu_q_lens, []
        for r, sid in enumerate(plan.seq_ids):
            n, done = int(cu[r + 1] - cu[r]), len(texts[sid][0]) if sid in texts else 0
            depth = list(range(n))
            for b, parent in enumerate(trees.get(sid, ())):
                depth[b] = 0 if parent < 0 else depth[parent] + 1
            where += [done + x for x in depth]
        where, rotated = torch.tensor(where, device=device), torch.empty_like(q)
        if interleaved:
            cos, sin = ops.rotary_pair_tables(inv, 256, device=device)
            ops.qk_norm_rope_kv_append(q, k, v, None, None, cos, sin, where, *scratch, plan.slot_mapping, 0.0, True, query_out=rotated)
        else:
            cos, sin = ops.rotary_tables(inv, 256, dtype, device=device)
            ops.rope_kv_append(q, k, v, cos, sin, where, *scratch, plan.slot_mapping, query_out=rotated)
        backend.begin_step(plan)
        out, slot, rotated = backend.attend(0, q, k, v).cpu(), plan.slot_mapping, rotated.cpu()
        cached = [p[slot // 16, :, slot % 16].cpu().double() for p in (backend.k_pools[0], backend.v_pools[0])]
        for have, p in zip(cached, scratch):
            assert torch.equal(have, p[slot // 16, :, slot % 16].cpu().double())
        for r, sid in enumerate(plan.seq_ids):
            mine, n = slice(int(cu[r]), int(cu[r + 1])), int(cu[r + 1] - cu[r])
            texts[sid] = [fed(t, x[mine]) for t, x in zip(texts.get(sid, (None, None)), cached)]
            see = tree_visible(len(texts[sid][0]), n, trees.get(sid))
            want, mean_abs, size = masked_attention(rotated[mine], *texts[sid], see, backend.scale)
            check(out[mine], want, attention_bound(want, mean_abs, size, d, dtype) if trees else plain_bound(want, dtype))

    def keep(moved, trees, kept):
        for sid, tree in trees.items():
            n, stay = len(tree), kept.get(sid, [])
            texts[sid] = [torch.cat((t[:-n], t[-n:][stay])) for t in texts[sid]]
        backend.keep_drafts(moved)

    play(planner, step, keep)


@pytest.mark.parametrize("H", [6, 40])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_drafts_over_latent_rows(device, dtype, H):
    """Rows of 512 + 64, heads of 128 + 64 and 128: append, expanded prompts, absorbed chunks, trees, kept rows, tokens.

    Bound, from roundings of u = eps / 2 relative each, independent of one another: a sum of errors within +-c_i passes 7 sqrt(sum c_i^2)
    with a chance of 2 e^-24.5 (Hoeffding).  A score: of the row and the multiplied query (absorbed), of the row and the key made of it
    (expanded), of the rotated parts, ds = 7 u scale sqrt(2 sum_c q'_c^2 r_c^2 + sum_n q_n^2 k_n^2 + 2 sum_d ..); the mean moves by
    (e^(2 ds) - 1) sum_j p_j |v_j - out|.  The value: the rows', the rounded mean's, the weights' and the expanded values' own; the
    result's, u.  In float16 a product's terms may be below the normal numbers: 2^-24 on the result.
    """
    N, D, C, V, g = 128, 64, 512, 128, torch.Generator().manual_seed(53)
    w_k, w_v = [(torch.randn(H, n, C, generator=g) / math.sqrt(C)).to(dtype) for n in (N, V)]
    weight = 1 + 0.2 * torch.randn(C, generator=g)
    inv = 1.0 / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
    scale, u = 0.1 / math.sqrt(N + D), torch.finfo(dtype).eps / 2
    planner = planner_of(device)
    backend = LatentAttentionBackend(1, 40, C, D, inv, scale, dtype, device, 256)
    backend.set_layer(0, w_k, w_v, weight)
    texts, forms = {}, []

    def turn(x, at):
        angle = at.double()[:, None] * inv
        c, s = [t[:, None] if x.dim() == 3 else t for t in (angle.cos(), angle.sin())]
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    def step(plan, trees):
        T = plan.total_new_tokens
        q, x = torch.randn(T, H, N + D, generator=g).to(dtype), torch.randn(T, C + D, generator=g).to(dtype)
        backend.begin_step(plan)
        out = backend.attend(0, q.to(device), x.to(device)).double().cpu()
        cu = plan.host_cu_q_lens
        forms.append((bool(trees), plan.num_prefill_seqs, plan.num_seqs))
        for r, sid in enumerate(plan.seq_ids):
            mine, n = slice(int(cu[r]), int(cu[r + 1])), int(cu[r + 1] - cu[r])
            done = len(texts[sid][0]) if sid in texts else 0
            at = torch.arange(done, done + n)
            for b, parent in enumerate(trees.get(sid, ())):
                at[b] = done if parent < 0 else at[parent] + 1
            texts[sid] = [fed(t, y) for t, y in zip(texts.get(sid, (None, None)), (x[mine], at))]
            xs, places = texts[sid][0].double(), texts[sid][1]
            row = xs[:, :C] * torch.rsqrt(xs[:, :C].pow(2).mean(-1, keepdim=True) + 1e-6) * weight.double()
            rk, qs = turn(xs[:, C:], places), q[mine].double()
            qr = turn(qs[..., N:], at)
            k, v = [torch.einsum("hnc,sc->shn", w.double(), row) for w in (w_k, w_v)]
            see = tree_visible(done + n, n, trees.get(sid))
            score = scale * (torch.einsum("qhn,shn->hqs", qs[..., :N], k) + torch.einsum("qhd,sd->hqs", qr, rk))
            p = score.masked_fill(~see, -math.inf).softmax(-1)
            want = torch.einsum("hqs,shv->qhv", p, v)
            qa = torch.einsum("qhn,hnc->qhc", qs[..., :N], w_k.double())
            ds = (2 * torch.einsum("qhc,sc->qhs", qa ** 2, row ** 2) + torch.einsum("qhn,shn->qhs", qs[..., :N] ** 2, k ** 2)
                  + 2 * torch.einsum("qhd,sd->qhs", qr ** 2, rk ** 2))
            ds = 7 * u * scale * ds.masked_fill(~see[:, None], 0).amax(-1, keepdim=True).sqrt()
            spread = torch.stack([torch.einsum("hs,shv->hv", p[:, i], (v - want[i]).abs()) for i in range(n)])
            w2, o = w_v.double() ** 2, torch.einsum("hqs,sc->qhc", p, row)
            of_rows = torch.einsum("hvc,qhc->qhv", w2, torch.einsum("hqs,sc->qhc", p ** 2, row ** 2))
            of_mean = torch.einsum("hvc,qhc->qhv", w2, o ** 2)
            of_values = torch.einsum("hqs,shv->qhv", p ** 2, v ** 2)
            tol = 7 * u * (of_rows + of_mean + 2 * of_values).sqrt() + torch.expm1(2 * ds) * spread + u * want.abs() + 2.0 ** -24
            err = (out[mine] - want).abs()
            assert bool((err <= tol).all()), (sid, float((err / tol).max()))
            assert float(tol.mean()) < 0.3 * float(v.pow(2).mean().sqrt())             # (no idle bound)

    def keep(moved, trees, kept):
        for sid, tree in trees.items():
            n, stay = len(tree), kept.get(sid, [])
            texts[sid] = [torch.cat((t[:-n], t[-n:][stay])) for t in texts[sid]]
        backend.keep_drafts(moved)

    play(planner, step, keep)
    assert [f[0] for f in forms] == [what is not None for what in PLAY] and forms[0][1] >= 2 and forms[1][1] == 1 < forms[1][2]
