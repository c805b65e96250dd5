"""Cases of the operators around a cache of latent rows (one shared row of a token for all heads, its last elements rotated) and around
trees of drafted tokens:

  latent_append  RMS norm of the latent part, rotation of the shared key and of the queries' rotated part, append to the paged pool
  latent_attn    attention over the paged latent rows, queries absorbed: one token per sequence, chunks, trees of drafts
  prompt_attn    attention of prompts over keys and values expanded from the latent rows
  tree_attn      attention of trees of drafted tokens over the paged K and V pools
  keep_rows      the cache rows of the accepted drafts moved to their final positions, in every layer's pools

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
R, ROPE = 512, 64                         # latent and rotated elements of a row
NOPE, DV = 128, 128                       # expanded: elements of a head's key (without the rotated ones) and value
SCALE = 1 / math.sqrt(NOPE + ROPE)        # of both forms


# ------------------------------------------------------------------------------------------------ cases
def _append(name, tokens, heads, interleaved, dtype):
    c = {"op": "latent_append", "tokens": tokens, "heads": heads, "interleaved": interleaved, "dtype": dtype}
    return {**c, "name": name} if name else c


def _latent(name, rows, seqs, lo, hi, spread, q_lo, q_hi, heads, dtype):
    """rows: "one" token per sequence, causal "chunk"s, or "tree"s of drafts; lo .. hi: tokens cached before."""
    c = {"op": "latent_attn", "rows": rows, "seqs": seqs, "lo": lo, "hi": hi, "spread": spread, "q_lo": q_lo, "q_hi": q_hi,
         "heads": heads, "dtype": dtype}
    return {**c, "name": name} if name else c


def _prompt(name, seqs, lo, hi, q_lo, q_hi, heads, dtype):
    c = {"op": "prompt_attn", "seqs": seqs, "lo": lo, "hi": hi, "spread": "even", "q_lo": q_lo, "q_hi": q_hi, "heads": heads,
         "dtype": dtype}
    return {**c, "name": name} if name else c


def _tree(name, seqs, lo, hi, spread, q_lo, q_hi, hq, hkv, d, dtype, pool):
    c = {"op": "tree_attn", "rows": "tree", "seqs": seqs, "lo": lo, "hi": hi, "spread": spread, "q_lo": q_lo, "q_hi": q_hi, "hq": hq,
         "hkv": hkv, "d": d, "dtype": dtype, "pool": pool}
    return {**c, "name": name} if name else c


def _keep(name, layers, seqs, drafts, kept, hkv, d, dtype):
    c = {"op": "keep_rows", "layers": layers, "seqs": seqs, "drafts": drafts, "kept": kept, "hkv": hkv, "d": d, "dtype": dtype}
    return {**c, "name": name} if name else c


def listed():
    return [
        # the step of a single sequence, where the launch is all there is
        _append("latent_append_one_token", 1, 16, True, "bf16"),
        # a long prompt
        _append("latent_append_prompt", 8192, 16, False, "fp16"),
        # a single chat over a short context
        _latent("latent_one_row", "one", 1, 700, 700, "even", 1, 1, 16, "bf16"),
        # a serving batch over contexts of all ages; a rank's share of the heads
        _latent("latent_batch", "one", 64, 512, 4096, "even", 1, 1, 16, "bf16"),
        # all heads on one GPU
        _latent("latent_all_heads", "one", 32, 512, 4096, "even", 1, 1, 128, "fp16"),
        # drafted tokens over contexts of unlike length, some of them long
        _latent("latent_drafts", "tree", 16, 256, 16384, "skewed", 5, 24, 16, "bf16"),
        # one long prompt, all of it in one call
        _prompt("prompt_whole", 1, 0, 0, 8192, 8192, 16, "bf16"),
        # ragged prompts, parts of them behind what is cached already
        _prompt("prompt_ragged", 12, 0, 2048, 37, 1500, 16, "fp16"),
        # a single chat with a small tree of drafts
        _tree("tree_one_sequence", 1, 700, 700, "even", 9, 9, 32, 8, 64, "bf16", "bf16"),
        # a serving batch, trees up to the size of one word of the mask
        _tree("tree_batch", 32, 512, 4096, "even", 16, 64, 32, 8, 128, "bf16", "bf16"),
        # a single chat accepts a few drafts
        _keep("keep_one_sequence", 32, 1, 9, 4, 8, 128, "bf16"),
        # a serving batch does
        _keep("keep_batch", 16, 64, 32, 8, 8, 128, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["latent_append", "latent_attn", "latent_attn", "latent_attn", "prompt_attn", "prompt_attn", "tree_attn", "tree_attn",
                     "keep_rows"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "latent_append":
        return _append(None, _log(rng, 1, 8192), rng.choice([4, 8, 16, 32]), rng.random() < 0.5, rng.choice(["bf16", "fp16", "f32"]))
    if op == "keep_rows":
        drafts = _log(rng, 2, 100)
        seqs = _log(rng, 1, 64)
        return _keep(None, rng.randint(1, min(32, 1024 // seqs)), seqs, drafts, rng.randint(1, min(drafts, 12)),
                     rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), rng.choice(["bf16", "f32"]))
    if op == "prompt_attn":
        seqs = _log(rng, 1, 16)
        q_hi = _log(rng, 17, min(4096, 8192 // seqs))
        return _prompt(None, seqs, 0, rng.choice([0, _log(rng, 20, 2048)]), rng.randint(1, q_hi), q_hi, rng.choice([2, 4, 8, 16]), dtype)
    rows = "tree" if op == "tree_attn" else rng.choice(["one", "one", "chunk", "tree"])
    seqs = _log(rng, 1, 64)
    hi = _log(rng, 33, max(34, min(32768, 98304 // seqs)))
    lo, spread = rng.randint(0, hi), rng.choice(["even", "skewed"])
    q_hi = 1 if rows == "one" else _log(rng, 2, min(100, 1024 // seqs))
    q_lo = rng.randint(1, q_hi)
    if op == "latent_attn":
        heads = rng.choice([8, 16, 16, 32, 64, 128])
        if q_hi > 1:
            heads = min(heads, 32)
        return _latent(None, rows, seqs, lo, hi, spread, q_lo, q_hi, heads, dtype)
    hkv = rng.choice([2, 4, 8])
    return _tree(None, seqs, lo, hi, spread, q_lo, q_hi, hkv * rng.choice([1, 2, 4, 8]), hkv, rng.choice([64, 128]), dtype,
                 rng.choice([dtype, dtype, "fp8"]))


# ---------------------------------------------------------------------------------------------- lengths
def _spread(n, lo, hi, how="even"):
    """n lengths of lo .. hi: in turns through the range, or most of them short (lognormal around an eighth of hi)."""
    if how == "skewed":
        z = [NormalDist().inv_cdf((((i * 7) % n if n % 7 else i) + 0.5) / n) for i in range(n)]
        return [max(lo, min(hi, int(hi / 8 * math.exp(x)))) for x in z]
    return [lo + int((hi - lo) * ((0.5 + 0.6180339887498949 * i) % 1.0) + 0.5) for i in range(n)]


def _lengths(case):
    """New tokens and contexts (with them) of every sequence."""
    new = _spread(case["seqs"], case["q_lo"], case["q_hi"])
    return new, [a + b for a, b in zip(_spread(case["seqs"], case["lo"], case["hi"], case["spread"]), new)]


def _parents(n, seq):
    """A tree of n drafts: each hangs on one of the few before it."""
    got, x = [-1], 12345 + 7919 * seq
    for i in range(1, n):
        x = (x * 1103515245 + 12345) % 2 ** 31
        got.append(i - 1 - (x >> 16) % min(i, 5))
    return got


def _ancestors(n, seq):
    """For each draft the drafts that it sees, itself among them, as the bits of a whole number."""
    got = []
    for i, p in enumerate(_parents(n, seq)):
        got.append((1 << i) | (got[p] if p >= 0 else 0))
    return got


def _words(case):
    """Those bits in 64-bit words, as many as the longest tree takes: [rows][words]."""
    new, _ = _lengths(case)
    width = -(-max(new) // 64)
    rows = [b for s, n in enumerate(new) for b in _ancestors(n, s)]
    return [[w - 2 ** 64 if w >= 2 ** 63 else w for w in ((b >> (64 * k)) % 2 ** 64 for k in range(width))] for b in rows]


def _kept(case):
    """The drafts that each sequence keeps: the first one, and later ones whose rows are no row's new place (so that a second pass
    leaves what the first one made)."""
    got, n = [], case["kept"]
    for s in range(case["seqs"]):
        step = max(1, (case["drafts"] - n) // n)
        got.append([0] + [k for k in (n + (i - 1) * step + (s + i) % step for i in range(1, n)) if k < case["drafts"]])
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


def _table(s, ctx, g):
    """Block tables of sequences of these lengths, their blocks strewn over the pool."""
    need = [-(-c // BS) for c in ctx]
    blocks = sum(need) + sum(need) // 10 + 1
    order = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    starts = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    at = starts[:, None] + torch.arange(max(need), device="cuda")
    s.table = order[at.clamp(max=blocks - 1)].contiguous()
    return blocks


def _cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], device="cuda", dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = State()
    s.case, s.op = case, case["op"]
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32)

    if s.op == "latent_append":
        T, H = case["tokens"], case["heads"]
        s.latent = (0.7 * randn(T, R + ROPE)).to(dt)               # a projection's output
        s.query = randn(T, H, NOPE + ROPE).to(dt)[:, :, NOPE:]     # the rotated part of every head
        s.weight = 1 + 0.1 * randn(R)
        angles = torch.arange(8192, device="cuda", dtype=torch.float64)[:, None] * (
            500000.0 ** (-torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float64) / ROPE))[None, :]
        s.cos, s.sin = angles.cos().float(), angles.sin().float()
        s.positions = torch.randint(0, 8192, (1,), device="cuda", generator=g) if T == 1 else torch.arange(T, device="cuda") % 8192
        blocks = -(-T // BS) + 1
        s.slots = (torch.randperm(blocks, device="cuda", generator=g)[:, None] * BS + torch.arange(BS, device="cuda")).view(-1)[:T].clone()
        s.pool = torch.zeros((blocks, BS, R + ROPE), device="cuda", dtype=dt)
        s.absorbed = torch.zeros((T, H, R + ROPE), device="cuda", dtype=dt)
        s.q_out = s.absorbed[:, :, R:]                             # beside the absorbed part
        s.interleaved = case["interleaved"]
        return s
    if s.op == "keep_rows":
        keep = _kept(case)
        first = [int(x) for x in torch.randint(100, 200, (case["seqs"],), generator=torch.Generator().manual_seed(seed))]
        blocks = _table(s, [200 + case["drafts"]] * case["seqs"], g)
        s.pools = randn(2 * case["layers"], blocks, case["hkv"], BS, case["d"]).to(dt)
        s.each = list(s.pools.unbind(0))
        s.first = torch.tensor(first, device="cuda", dtype=torch.int32)
        s.keep = torch.tensor([k for row in keep for k in row], device="cuda", dtype=torch.int32)
        s.cu = _cu([len(row) for row in keep])
        return s
    new, ctx = _lengths(case)
    T = sum(new)
    s.max_q, s.longest = max(new), max(ctx)
    s.cu, s.lens = _cu(new), torch.tensor(ctx, device="cuda", dtype=torch.int32)
    if s.op == "prompt_attn":
        H = case["heads"]
        s.query = (1.2 * randn(T, H, NOPE + ROPE)).to(dt)
        expanded = randn(sum(ctx), H, NOPE + DV).to(dt)            # one projection of the latent rows
        s.key, s.value = expanded[:, :, :NOPE], expanded[:, :, NOPE:]
        s.rope_key = randn(sum(ctx), R + ROPE).to(dt)[:, R:]       # beside the latent part
        s.cu_k = _cu(ctx)
        s.out = torch.empty((T, H, DV), device="cuda", dtype=dt)
        return s
    blocks = _table(s, ctx, g)
    s.masks = torch.tensor(_words(case), device="cuda", dtype=torch.int64) if case["rows"] == "tree" else None
    if s.op == "latent_attn":
        H = case["heads"]
        s.pool = randn(blocks, BS, R + ROPE).to(dt)
        s.query = torch.cat((0.6 * randn(T, H, R), 1.2 * randn(T, H, ROPE)), dim=-1).to(dt)
        s.out = torch.empty((T, H, R), device="cuda", dtype=dt)
        return s
    d, hkv = case["d"], case["hkv"]
    s.k_pool, s.k_scale = _pool((blocks, hkv, BS, d), case["pool"], g)
    s.v_pool, s.v_scale = _pool((blocks, hkv, BS, d), case["pool"], g)
    s.query = (1.5 * randn(T, case["hq"], d)).to(dt)
    s.out = torch.empty_like(s.query)
    return s


# --------------------------------------------------------------------------------------------- the call
def run(s):
    if own:
        return _own(s)
    return {"latent_append": _plain_append, "latent_attn": _plain_latent, "prompt_attn": _plain_prompt, "tree_attn": _plain_tree,
            "keep_rows": _plain_keep}[s.op](s)


def _own(s):
    from aicomp_amd import ops
    if s.op == "latent_append":
        ops.latent_kv_append(s.latent, s.weight, s.cos, s.sin, s.positions, s.pool, s.slots, eps=EPS, interleaved=s.interleaved,
                             query=s.query, query_out=s.q_out)
        return s.q_out, s.pool
    if s.op == "keep_rows":
        ops.keep_rows(s.each, s.table, s.first, s.keep, s.cu)
        return s.pools
    if s.op == "prompt_attn":
        return ops.latent_prompt_attn(s.out, s.query, s.key, s.rope_key, s.value, s.cu, s.cu_k, SCALE, max_q_len=s.max_q)
    if s.op == "latent_attn":
        if s.case["rows"] == "one":
            return ops.paged_latent_attn(s.out, s.query, s.pool, s.table, s.lens, SCALE, longest_context=s.longest)
        return ops.paged_latent_attn(s.out, s.query, s.pool, s.table, s.lens, SCALE, cu_q_lens=s.cu, max_q_len=s.max_q,
                                     tree_masks=s.masks, longest_context=s.longest)
    return ops.paged_tree_attn(s.out, s.query, s.k_pool, s.v_pool, s.table, s.lens, s.cu, s.masks, 1 / math.sqrt(s.case["d"]),
                               max_q_len=s.max_q, k_scale=s.k_scale, v_scale=s.v_scale, longest_context=s.longest)


def _turned(x, cos, sin, interleaved):
    """Pairs of the last elements rotated, in 32 bits; cos and sin have one column per pair."""
    x, half = x.float(), cos.shape[-1]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_append(s):
    cos, sin = s.cos[s.positions], s.sin[s.positions]
    x = s.latent[:, :R].float()
    normed = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s.weight
    row = torch.cat((normed, _turned(s.latent[:, R:], cos, sin, s.interleaved)), dim=-1)
    s.pool.view(-1, R + ROPE)[s.slots] = row.to(s.pool.dtype)
    s.q_out.copy_(_turned(s.query, cos[:, None], sin[:, None], s.interleaved))
    return s.q_out, s.pool


def _softmax(x, seen):
    """Softmax over the last axis where seen; rows that see nothing are zero.  In place on x."""
    x.masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = x.sub_(top).exp_()
    return x.div_(x.sum(-1, keepdim=True).clamp(min=1e-30))


def _grid(s, L):
    """Rows of the padded grid [S, M], which of them are real, and the keys [S, M, L] that they see."""
    T, M, S = s.query.shape[0], s.max_q, s.lens.shape[0]
    i, j = torch.arange(M, device="cuda"), torch.arange(L, device="cuda")
    new = (s.cu[1:] - s.cu[:-1]).long()
    row = (s.cu[:-1].long()[:, None] + i).clamp(max=T - 1)
    prior = (s.lens.long() - new)[:, None, None]
    at = j - prior                                                 # which draft or chunk token a key is
    masks = getattr(s, "masks", None)
    if masks is None:
        seen = at <= i[:, None]
    else:
        words = masks[row]                                         # [S, M, W]
        bit = torch.gather(words, 2, (at // 64).clamp(0, words.shape[2] - 1).expand(S, M, L)) >> (at % 64) & 1
        seen = (at < 0) | (bit == 1)
    return row, i < new[:, None], seen & (j < s.lens.long()[:, None, None])


def _plain_latent(s):
    S, bw = s.table.shape
    T, H, D = s.query.shape
    c = s.pool[s.table.long()].float().view(S, bw * BS, D)         # [S, L, R + ROPE]
    row, real, seen = _grid(s, bw * BS)
    M = row.shape[1]
    q = s.query.float()[row].view(S, M * H, D)
    x = torch.matmul(q, c.transpose(1, 2)).view(S, M, H, bw * BS).mul_(SCALE)
    x = _softmax(x, seen[:, :, None])
    o = torch.matmul(x.view(S, M * H, bw * BS), c[:, :, :R].contiguous()).view(S, M, H, R)
    s.out[row[real]] = o[real].to(s.out.dtype)
    return s.out


def _plain_prompt(s):
    new, ctx = _lengths(s.case)
    t = u = 0
    for n, c in zip(new, ctx):
        key = torch.cat((s.key[u:u + c].float(), s.rope_key[u:u + c].float()[:, None].expand(c, s.key.shape[1], ROPE)), dim=-1)
        x = torch.matmul(s.query[t:t + n].float().transpose(0, 1), key.permute(1, 2, 0)).mul_(SCALE)
        seen = torch.arange(c, device="cuda") <= torch.arange(c - n, c, device="cuda")[:, None]
        s.out[t:t + n] = torch.matmul(_softmax(x, seen), s.value[u:u + c].float().transpose(0, 1)).transpose(0, 1).to(s.out.dtype)
        t, u = t + n, u + c
    return s.out


def _gathered(pool, scale, table):
    """[S, Hkv, keys, D] in 32 bits."""
    x = pool[table.long()].float()                                # [S, blocks, Hkv, BS, D]
    if scale is not None:
        x = x * scale[None, None, :, None, None]
    S, nb, hkv, bs, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(S, hkv, nb * bs, d)


def _plain_tree(s):
    T, hq, d = s.query.shape
    S, hkv = s.table.shape[0], s.k_pool.shape[1]
    k, v = _gathered(s.k_pool, s.k_scale, s.table), _gathered(s.v_pool, s.v_scale, s.table)
    L, G = k.shape[2], hq // hkv
    row, real, seen = _grid(s, L)
    M = row.shape[1]
    q = s.query.float()[row].view(S, M, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(S, hkv, G * M, d)
    x = torch.matmul(q, k.transpose(2, 3)).view(S, hkv, G, M, L).mul_(1 / math.sqrt(d))
    x = _softmax(x, seen.view(S, 1, 1, M, L))
    o = torch.matmul(x.view(S, hkv, G * M, L), v).view(S, hkv, G, M, d)
    s.out[row[real]] = o.permute(0, 3, 1, 2, 4).reshape(S, M, hq, d)[real].to(s.out.dtype)
    return s.out


def _plain_keep(s):
    seq = torch.repeat_interleave(torch.arange(s.first.shape[0], device="cuda"), (s.cu[1:] - s.cu[:-1]).long(),
                                  output_size=s.keep.shape[0])
    start = s.first.long()[seq]
    src, dst = start + s.keep.long(), start + torch.arange(s.keep.shape[0], device="cuda") - s.cu.long()[seq]
    a, b = s.table[seq, src // BS].long(), s.table[seq, dst // BS].long()
    s.pools[:, b, :, dst % BS] = s.pools[:, a, :, src % BS]
    return s.pools


# ------------------------------------------------------------------------------------------------ work
def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "latent_append":
        T, H = case["tokens"], case["heads"]
        return {"bytes": 2 * T * (R + ROPE + H * ROPE) * e + min(T, 8192) * ROPE * 4 + 16 * T + 4 * R,
                "flops": T * (5 * R + 3 * ROPE * (H + 1))}
    if case["op"] == "keep_rows":
        moved = sum(k != i for row in _kept(case) for i, k in enumerate(row))
        return {"bytes": 2 * 2 * case["layers"] * moved * case["hkv"] * case["d"] * e, "flops": 0}
    new, ctx = _lengths(case)
    T, table = sum(new), 4 * sum(-(-c // BS) for c in ctx)
    if case.get("rows") == "tree":
        pairs = sum((c - n) * n + sum(bin(b).count("1") for b in _ancestors(n, s)) for s, (n, c) in enumerate(zip(new, ctx)))
    else:
        pairs = sum((c - n) * n + n * (n + 1) // 2 for n, c in zip(new, ctx))
    if case["op"] == "latent_attn":
        H = case["heads"]
        return {"bytes": sum(ctx) * (R + ROPE) * e + T * H * (2 * R + ROPE) * e + table, "flops": 2 * pairs * H * (2 * R + ROPE)}
    if case["op"] == "prompt_attn":
        H = case["heads"]
        return {"bytes": sum(ctx) * (H * (NOPE + DV) + ROPE) * e + T * H * (NOPE + ROPE + DV) * e,
                "flops": 2 * pairs * H * (NOPE + ROPE + DV)}
    return {"bytes": 2 * sum(ctx) * case["hkv"] * case["d"] * SIZE[case["pool"]] + 2 * T * case["hq"] * case["d"] * e + table,
            "flops": 4 * pairs * case["hq"] * case["d"]}


# ------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "latent_append":
        turn = torch.complex(s.cos.double(), s.sin.double())[s.positions][:, None]

        def rotated(x):
            pairs = x.double().unflatten(-1, (ROPE // 2, 2) if s.interleaved else (2, ROPE // 2))
            pairs = pairs if s.interleaved else pairs.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            return (z if s.interleaved else z.transpose(-1, -2)).flatten(-2)

        x = s.latent[:, :R].double()
        flat = torch.zeros((s.pool.shape[0] * BS, R + ROPE), device="cuda", dtype=torch.float64)
        flat[s.slots, :R] = x * s.weight.double() / ((x ** 2).sum(-1, keepdim=True) / R + EPS).sqrt()
        flat[s.slots, R:] = rotated(s.latent[:, None, R:])[:, 0]
        return rotated(s.query), flat.view(s.pool.shape)
    if s.op == "keep_rows":
        want = s.pools.clone()
        for n, row in enumerate(_kept(case)):
            p = int(s.first[n])
            for i, k in enumerate(row):
                a, b = p + k, p + i
                want[:, int(s.table[n, b // BS]), :, b % BS] = s.pools[:, int(s.table[n, a // BS]), :, a % BS]
        return want
    new, ctx = _lengths(case)
    want = torch.zeros(s.out.shape, device="cuda", dtype=torch.float64)
    t = u = 0
    for n, (q, c) in enumerate(zip(new, ctx)):
        at = torch.arange(c, device="cuda")
        seen = at <= torch.arange(c - q, c, device="cuda")[:, None]
        if case.get("rows") == "tree":
            bits = _ancestors(q, n)
            seen[:, c - q:] = torch.tensor([[(b >> i) & 1 == 1 for i in range(q)] for b in bits], device="cuda")
        if s.op != "prompt_attn":
            block, slot = s.table[n].long()[at // BS], at % BS
        for h in range(s.query.shape[1]):
            if s.op == "latent_attn":
                if h == 0:
                    k = s.pool[block, slot].double()
                    v = k[:, :R]
                scale = SCALE
            elif s.op == "prompt_attn":
                k = torch.cat((s.key[u:u + c, h], s.rope_key[u:u + c]), dim=-1).double()
                v, scale = s.value[u:u + c, h].double(), SCALE
            else:
                g = h // (case["hq"] // case["hkv"])
                k, v, scale = s.k_pool[block, g, slot].double(), s.v_pool[block, g, slot].double(), 1 / math.sqrt(case["d"])
                if s.k_scale is not None:
                    k, v = k * s.k_scale[g].double(), v * s.v_scale[g].double()
            x = torch.where(seen, s.query[t:t + q, h].double() @ k.T * scale, -math.inf)
            want[t:t + q, h] = torch.softmax(x, dim=-1) @ v
        t, u = t + q, u + c
    return want
