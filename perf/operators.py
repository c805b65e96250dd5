"""Cases of the operators around a decoder layer whose queries and keys are normed per head and whose attention scores follow
a rule (a cap by tanh, a bias by distance, a window, documents, a prefix), and of moving pages of the cache:

  norm_rope  RMS norm of every query and key head, rotary positions, append to the paged pools
  decode     one new token per sequence over the paged pools, scores by the rule
  prefill    the rows of prompt chunks over the paged pools, scores by the rule
  copy       blocks of every layer's pools copied (a fork's last block, a compaction)

``run`` is one call: with ``own`` the framework's operator, else the same mathematics in elementary torch operations.
"""
from __future__ import annotations

import math
from statistics import NormalDist

import torch

own = False
BS = 16                                   # tokens per block of the pools
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "f32": 4, "fp8": 1}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def _norm_rope(name, tokens, hq, hkv, d, rotary, interleaved, dtype):
    c = {"op": "norm_rope", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "rotary": rotary, "interleaved": interleaved,
         "dtype": dtype}
    return {**c, "name": name} if name else c


def _attn(name, op, seqs, lo, hi, spread, q_lo, q_hi, hq, hkv, d, dtype, pool, cap, slopes, window, document, prefix):
    c = {"op": op, "seqs": seqs, "lo": lo, "hi": hi, "spread": spread, "q_lo": q_lo, "q_hi": q_hi, "hq": hq, "hkv": hkv, "d": d,
         "dtype": dtype, "pool": pool, "cap": cap, "slopes": slopes, "window": window, "document": document, "prefix": prefix}
    return {**c, "name": name} if name else c


def _copy(name, layers, pairs, hkv, d, dtype):
    c = {"op": "copy", "layers": layers, "pairs": pairs, "hkv": hkv, "d": d, "dtype": dtype}
    return {**c, "name": name} if name else c


def listed():
    return [
        # the step of a single sequence, where the launch is all there is
        _norm_rope("norm_rope_one_token", 1, 32, 8, 128, 128, False, "bf16"),
        # a long prompt; neighbours are pairs, half of each head is rotated
        _norm_rope("norm_rope_prompt_part", 8192, 32, 8, 128, 64, True, "fp16"),
        # a single chat over a short context
        _attn("decode_cap_one_row", "decode", 1, 700, 700, "even", 1, 1, 32, 8, 64, "bf16", "bf16", 50.0, False, 0, 0, 0),
        # float32 models, a small batch
        _attn("decode_cap_f32", "decode", 4, 64, 512, "even", 1, 1, 32, 8, 64, "f32", "f32", 30.0, False, 0, 0, 0),
        # a serving batch over contexts of all ages
        _attn("decode_cap_batch", "decode", 64, 512, 4096, "even", 1, 1, 32, 8, 128, "bf16", "bf16", 50.0, False, 0, 0, 0),
        # a layer that looks back over a window, in a large batch over an 8-bit cache
        _attn("decode_window_fp8", "decode", 128, 1024, 8192, "even", 1, 1, 64, 8, 128, "bf16", "fp8", 0.0, False, 1024, 0, 0),
        # few long contexts of unlike length, scores that fall with distance
        _attn("decode_slopes_long", "decode", 16, 256, 32768, "skewed", 1, 1, 32, 8, 128, "fp16", "fp16", 0.0, True, 0, 0, 0),
        # one long prompt, all of it in one call: the most work
        _attn("prefill_cap_prompt", "prefill", 1, 0, 0, "even", 8192, 8192, 32, 8, 128, "bf16", "bf16", 50.0, False, 0, 0, 0),
        # chunks of prompts over what is cached already, in a layer with a window
        _attn("prefill_cap_window_chunks", "prefill", 4, 0, 2048, "even", 512, 512, 32, 8, 128, "bf16", "bf16", 50.0, False, 1024,
              0, 0),
        # ragged prompts packed from documents that do not see each other; each begins with a part whose rows see all of it
        _attn("prefill_documents", "prefill", 12, 0, 0, "even", 37, 1500, 16, 4, 64, "fp16", "fp16", 0.0, True, 0, 300, 64),
        # a sequence is forked: its last block, in every layer
        _copy("copy_fork", 32, 1, 8, 128, "bf16"),
        # the pool is compacted
        _copy("copy_compact", 16, 500, 8, 128, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "decode", "decode", "decode", "prefill", "prefill", "prefill", "copy"])
    d = rng.choice([64, 128])
    if op == "norm_rope":
        hkv = rng.choice([1, 2, 4, 8])
        return _norm_rope(None, _log(rng, 1, 8192), hkv * rng.choice([1, 2, 4]), hkv, d, d // rng.choice([1, 1, 2, 4]),
                          rng.random() < 0.5, rng.choice(["bf16", "fp16", "f32"]))
    if op == "copy":
        return _copy(None, rng.randint(1, 32), _log(rng, 1, 250), rng.choice([1, 2, 4, 8]), d, rng.choice(["bf16", "f32"]))
    hkv, group = rng.choice([2, 4, 8]), rng.choice([1, 2, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    pool = rng.choice([dtype, dtype, "fp8"])
    cap = rng.choice([0.0, 20.0, 30.0, 50.0])
    slopes = rng.random() < 0.3
    window = rng.choice([0, 0, _log(rng, 100, 4096)])
    if cap == 0.0 and not slopes and window == 0:
        cap = 50.0
    if op == "decode":
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 33, max(34, min(32768, 262144 // seqs)))
        return _attn(None, op, seqs, rng.randint(1, hi), hi, rng.choice(["even", "skewed"]), 1, 1, hkv * group, hkv, d, dtype, pool,
                     cap, slopes, window, rng.choice([0, 0, 200]), 0)
    seqs = _log(rng, 1, 16)
    q_hi = _log(rng, 17, max(18, min(4096, 8192 // seqs)))
    return _attn(None, op, seqs, 0, rng.choice([0, _log(rng, 20, 2048)]), "even", rng.randint(2, q_hi), q_hi, hkv * group, hkv, d,
                 dtype, pool, cap, slopes, window, rng.choice([0, 0, 200]), rng.choice([0, 0, 50]))


# ---------------------------------------------------------------------------------------------- lengths
def _spread(n, lo, hi, how="even"):
    """n lengths of lo .. hi: in turns through the range, or most of them short (lognormal around an eighth of hi)."""
    if how == "skewed":
        z = [NormalDist().inv_cdf((((i * 7) % n if n % 7 else i) + 0.5) / n) for i in range(n)]
        return [max(lo, min(hi, int(hi / 8 * math.exp(x)))) for x in z]
    return [lo + int((hi - lo) * ((0.5 + 0.6180339887498949 * i) % 1.0) + 0.5) for i in range(n)]


def _lengths(case):
    """New tokens and contexts (with them) of every sequence."""
    if case["op"] == "decode":
        return [1] * case["seqs"], _spread(case["seqs"], case["lo"], case["hi"], case["spread"])
    new = _spread(case["seqs"], case["q_lo"], case["q_hi"])
    return new, [a + b for a, b in zip(_spread(case["seqs"], case["lo"], case["hi"]), new)]


def _first_keys(case):
    """The first key of each row's document: documents of every other length around the case's, one after the other."""
    if not case["document"]:
        return None
    n = case["document"]
    return [(p // n) * n if (p // n) % 2 else max(0, (p // n) * n - n // 3) for q, c in zip(*_lengths(case)) for p in range(c - q, c)]


def _ranges(case):
    """(first visible key, end of the visible keys) of every row."""
    first = _first_keys(case)
    got, t = [], 0
    for q, c in zip(*_lengths(case)):
        for p in range(c - q, c):
            lo = max(first[t] if first else 0, p - case["window"] + 1 if case["window"] else 0)
            got.append((lo, max(p + 1, min(case["prefix"], c))))
            t += 1
    return got


# ---------------------------------------------------------------------------------------------- inputs
class State:
    pass


def _pool(shape, dtype, g):
    """A pool's blocks and, where it holds 8 bits, the scale of each head."""
    x = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32)
    if dtype != "fp8":
        return x.to(DTYPES[dtype]), None
    scale = x.abs().amax(dim=(0, 2, 3)) / 448.0
    return (x / scale[None, :, None, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = State()
    s.case, s.op = case, case["op"]
    d, hkv = case["d"], case["hkv"]
    if s.op == "copy":
        blocks = 2 * case["pairs"] + 8
        s.pools = torch.randn((2 * case["layers"], blocks, hkv, BS, d), device="cuda", generator=g, dtype=torch.float32).to(
            DTYPES[case["dtype"]])
        s.each = list(s.pools.unbind(0))
        order = torch.randperm(blocks, device="cuda", generator=g)[:2 * case["pairs"]]
        s.pairs = order.view(-1, 2).contiguous()
        return s
    dt, hq = DTYPES[case["dtype"]], case["hq"]
    if s.op == "norm_rope":
        T, r = case["tokens"], case["rotary"]
        x = torch.randn((T, (hq + 2 * hkv) * d), device="cuda", generator=g, dtype=torch.float32).to(dt)
        s.query = x[:, :hq * d].view(T, hq, d)                    # slices of one projection
        s.key = x[:, hq * d:(hq + hkv) * d].view(T, hkv, d)
        s.value = x[:, (hq + hkv) * d:].view(T, hkv, d)
        s.q_weight, s.k_weight = (1 + 0.1 * torch.randn((2, d), device="cuda", generator=g)).unbind(0)
        angles = torch.arange(8192, device="cuda", dtype=torch.float64)[:, None] * (
            500000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r))[None, :]
        s.cos, s.sin = angles.cos().float(), angles.sin().float()
        s.positions = torch.randint(0, 8192, (1,), device="cuda", generator=g) if T == 1 else torch.arange(T, device="cuda") % 8192
        blocks = -(-T // BS) + 1
        s.slots = (torch.randperm(blocks, device="cuda", generator=g)[:, None] * BS + torch.arange(BS, device="cuda")).view(-1)[:T].clone()
        s.k_pool = torch.zeros((blocks, hkv, BS, d), device="cuda", dtype=dt)
        s.v_pool = torch.zeros_like(s.k_pool)
        s.q_out = torch.empty((T, hq, d), device="cuda", dtype=dt)
        s.interleaved = case["interleaved"]
        return s
    new, ctx = _lengths(case)
    T, width = sum(new), -(-max(ctx) // BS)
    need = [-(-c // BS) for c in ctx]
    blocks = sum(need) + sum(need) // 10 + 1
    s.k_pool, s.k_scale = _pool((blocks, hkv, BS, d), case["pool"], g)
    s.v_pool, s.v_scale = _pool((blocks, hkv, BS, d), case["pool"], g)
    order = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    starts = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    at = starts[:, None] + torch.arange(width, device="cuda")
    s.table = order[at.clamp(max=blocks - 1)].contiguous()
    s.lens = torch.tensor(ctx, device="cuda", dtype=torch.int32)
    s.cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], device="cuda", dtype=torch.int32)
    s.longest, s.max_q = max(ctx), max(new)
    s.query = torch.randn((T, hq, d), device="cuda", generator=g, dtype=torch.float32).mul_(1.5).to(dt)
    s.out = torch.empty_like(s.query)
    s.scale = 1 / math.sqrt(d)
    s.cap, s.window = case["cap"], case["window"]
    s.slopes = torch.exp2(-8.0 * torch.arange(1, hq + 1, device="cuda", dtype=torch.float32) / hq) if case["slopes"] else None
    first = _first_keys(case)
    s.first = torch.tensor(first, device="cuda", dtype=torch.int32) if first else None
    s.prefix = torch.full((len(ctx),), case["prefix"], device="cuda", dtype=torch.int32) if case["prefix"] else None
    return s


# --------------------------------------------------------------------------------------------- the call
def run(s):
    if own:
        return _own(s)
    if s.op == "copy":
        s.pools[:, s.pairs[:, 1]] = s.pools[:, s.pairs[:, 0]]
        return s.pools
    return _plain_norm_rope(s) if s.op == "norm_rope" else _plain_attn(s)


def _own(s):
    from aicomp_amd import ops
    if s.op == "copy":
        ops.copy_blocks(s.each, s.pairs)
        return s.pools
    if s.op == "norm_rope":
        ops.qk_norm_rope_kv_append(s.query, s.key, s.value, s.q_weight, s.k_weight, s.cos, s.sin, s.positions, s.k_pool, s.v_pool,
                                   s.slots, eps=EPS, interleaved=s.interleaved, query_out=s.q_out)
        return s.q_out, s.k_pool, s.v_pool
    if s.op == "decode":
        return ops.paged_score_decode_attn(s.out, s.query, s.k_pool, s.v_pool, s.table, s.lens, s.scale, softcap=s.cap,
                                           slopes=s.slopes, window=s.window, first_keys=s.first, k_scale=s.k_scale,
                                           v_scale=s.v_scale, longest_context=s.longest)
    return ops.paged_score_prefill_attn(s.out, s.query, s.k_pool, s.v_pool, s.table, s.lens, s.cu, s.scale, max_q_len=s.max_q,
                                        softcap=s.cap, slopes=s.slopes, window=s.window, first_keys=s.first,
                                        prefix_lens=s.prefix, k_scale=s.k_scale, v_scale=s.v_scale)


def _plain_rows(x, weight, cos, sin, interleaved):
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    half = cos.shape[-1]
    c, n = cos[:, None], sin[:, None]
    if interleaved:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack((a * c - b * n, b * c + a * n), dim=-1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat((a * c - b * n, b * c + a * n), dim=-1)
    return torch.cat((turned, y[..., 2 * half:]), dim=-1)


def _plain_norm_rope(s):
    cos, sin = s.cos[s.positions], s.sin[s.positions]
    s.q_out.copy_(_plain_rows(s.query, s.q_weight, cos, sin, s.interleaved))
    block, at = s.slots // BS, s.slots % BS
    s.k_pool[block, :, at] = _plain_rows(s.key, s.k_weight, cos, sin, s.interleaved).to(s.k_pool.dtype)
    s.v_pool[block, :, at] = s.value
    return s.q_out, s.k_pool, s.v_pool


def _gathered(pool, scale, table):
    """[S, Hkv, keys, D] in 32 bits."""
    x = pool[table.long()].float()                                # [S, blocks, Hkv, BS, D]
    if scale is not None:
        x = x * scale[None, None, :, None, None]
    S, nb, hkv, bs, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(S, hkv, nb * bs, d)


def _plain_attn(s):
    T, hq, d = s.query.shape
    S, hkv, M = s.table.shape[0], s.k_pool.shape[1], s.max_q
    k, v = _gathered(s.k_pool, s.k_scale, s.table), _gathered(s.v_pool, s.v_scale, s.table)
    L, G = k.shape[2], hq // hkv
    new = (s.cu[1:] - s.cu[:-1]).long()
    i = torch.arange(M, device=k.device)
    row = (s.cu[:-1].long()[:, None] + i).clamp(max=T - 1)         # [S, M] rows of the padded grid
    real = i < new[:, None]
    p = (s.lens.long() - new)[:, None] + i                         # positions
    q = s.query.float()[row].view(S, M, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(S, hkv, G * M, d)
    x = torch.matmul(q, k.transpose(2, 3)).view(S, hkv, G, M, L)
    x *= s.scale
    if s.cap:
        x = torch.tanh(x.div_(s.cap)).mul_(s.cap)
    j = torch.arange(L, device=k.device)
    if s.slopes is not None:
        x -= s.slopes.view(1, hkv, G, 1, 1) * (p[:, :, None] - j).abs().view(S, 1, 1, M, L)
    seen = j <= p[:, :, None]
    if s.prefix is not None:
        seen |= j < s.prefix.long()[:, None, None]
    seen &= j < s.lens.long()[:, None, None]
    if s.window:
        seen &= p[:, :, None] - j < s.window
    if s.first is not None:
        seen &= j >= s.first.long()[row][:, :, None]
    x.masked_fill_(~seen.view(S, 1, 1, M, L), -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(S, hkv, G * M, L), v).view(S, hkv, G, M, d) / total.clamp(min=1e-30)
    s.out[row[real]] = o.permute(0, 3, 1, 2, 4).reshape(S, M, hq, d)[real].to(s.out.dtype)
    return s.out


# ------------------------------------------------------------------------------------------------ work
def work(case):
    d, hkv = case["d"], case["hkv"]
    if case["op"] == "copy":
        return {"bytes": 2 * 2 * case["layers"] * case["pairs"] * hkv * BS * d * SIZE[case["dtype"]], "flops": 0}
    hq, e = case["hq"], SIZE[case["dtype"]]
    if case["op"] == "norm_rope":
        T, r = case["tokens"], case["rotary"]
        rows = T * (hq + 2 * hkv) * d
        return {"bytes": 2 * rows * e + min(T, 8192) * r * 4 + 16 * T + 8 * d, "flops": T * (hq + hkv) * (5 * d + 3 * r)}
    pairs = keys = t = 0
    new, ctx = _lengths(case)
    rows = _ranges(case)
    for q in new:
        mine = rows[t:t + q]
        pairs += sum(max(0, b - a) for a, b in mine)
        keys += max(0, max(b for _, b in mine) - min(a for a, _ in mine))
        t += q
    return {"bytes": 2 * keys * hkv * d * SIZE[case["pool"]] + 2 * t * hq * d * e + 4 * sum(-(-c // BS) for c in ctx),
            "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "copy":
        want = s.pools.clone()
        for a, b in s.pairs.tolist():
            want[:, b] = s.pools[:, a]
        return want
    if s.op == "norm_rope":
        T = case["tokens"]
        turn = torch.complex(s.cos.double(), s.sin.double())[s.positions][:, None]
        half, got = case["rotary"] // 2, []
        for x, w in ((s.query, s.q_weight), (s.key, s.k_weight)):
            y = x.double() * w.double() / ((x.double() ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
            r = y[..., :2 * half]
            pairs = r.reshape(T, -1, half, 2) if s.interleaved else r.reshape(T, -1, 2, half).transpose(2, 3)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            r = z.reshape(r.shape) if s.interleaved else z.transpose(2, 3).reshape(r.shape)
            got.append(torch.cat((r, y[..., 2 * half:]), dim=-1))
        pools = []
        for x in (got[1], s.value.double()):
            flat = torch.zeros((s.k_pool.shape[0] * BS, case["hkv"], case["d"]), device="cuda", dtype=torch.float64)
            flat[s.slots] = x
            pools.append(flat.view(-1, BS, case["hkv"], case["d"]).transpose(1, 2).contiguous())
        return got[0], pools[0], pools[1]
    new, ctx = _lengths(case)
    group = case["hq"] // case["hkv"]
    want = torch.zeros(s.query.shape, device="cuda", dtype=torch.float64)
    limits = torch.tensor(_ranges(case), device="cuda")
    t = 0
    for n, (q, c) in enumerate(zip(new, ctx)):
        at = torch.arange(c, device="cuda")
        block, slot = s.table[n].long()[at // BS], at % BS
        lo, hi = limits[t:t + q, 0], limits[t:t + q, 1]
        seen = (at >= lo[:, None]) & (at < hi[:, None])
        for h in range(case["hkv"]):
            k, v = s.k_pool[block, h, slot].double(), s.v_pool[block, h, slot].double()
            if s.k_scale is not None:
                k, v = k * s.k_scale[h].double(), v * s.v_scale[h].double()
            for e in range(h * group, (h + 1) * group):
                x = s.query[t:t + q, e].double() @ k.T * s.scale
                if s.cap:
                    x = s.cap * torch.tanh(x / s.cap)
                if s.slopes is not None:
                    x = x - s.slopes[e].double() * (torch.arange(c - q, c, device="cuda")[:, None] - at).abs()
                x = torch.where(seen, x, -math.inf)
                full = seen.any(1)
                want[t:t + q, e][full] = torch.softmax(x[full], dim=-1) @ v
        t += q
    return want
