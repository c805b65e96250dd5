"""Plain float64 forms of the latent cache rows, of attention by an explicit mask and of the accepted rows (test infrastructure)."""
import torch


def latent_rows(latent, weight, eps, turn):
    """``latent [T, C + D]`` -> rows: the latent part normed by RMS, the last D elements passed through ``turn``."""
    C = weight.numel() if weight is not None else latent.shape[1] - turn.width
    x = latent.double()
    c = x[:, :C]
    if weight is not None:
        c = c * weight.double() / (c.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    return torch.cat((c, turn(x[:, None, C:])[:, 0]), dim=-1)


class Turn:
    """Rotation of ``[T, H, D]`` by tables ``[P, D/2]`` at ``positions [T]``; pairs are halves, or neighbours."""

    def __init__(self, cos, sin, positions, interleaved):
        self.cos, self.sin = cos.double()[positions][:, None], sin.double()[positions][:, None]
        self.interleaved, self.width = interleaved, 2 * cos.shape[1]

    def __call__(self, x):
        x = x.double()
        a, b = (x[..., 0::2], x[..., 1::2]) if self.interleaved else x.chunk(2, dim=-1)
        u, v = a * self.cos - b * self.sin, b * self.cos + a * self.sin
        return torch.stack((u, v), -1).flatten(-2) if self.interleaved else torch.cat((u, v), -1)


def masked_attention(q, k, v, visible, scale):
    """``q [n, H, dk]``, ``k [c, Hkv, dk]``, ``v [c, Hkv, dv]``, ``visible [n, c]`` -> the output ``[n, H, dv]``, the weighted mean of
    |v| there, and of each row the largest ``scale * sum |q_d k_d|`` among the keys that it sees (what errors are measured by)."""
    n, H, _ = q.shape
    q, k, v = q.double(), k.double(), v.double()
    group = H // k.shape[1]
    out, mean = (torch.zeros(n, H, v.shape[2], dtype=torch.float64) for _ in range(2))
    size = torch.zeros(n, H, dtype=torch.float64)
    some = visible.any(1)
    for h in range(H):
        kh, vh = k[:, h // group], v[:, h // group]
        seen = visible[some]
        x = torch.where(seen, q[some, h] @ kh.nan_to_num(0, 0, 0).T * scale, torch.tensor(-torch.inf, dtype=torch.float64))
        w = torch.softmax(x, dim=-1)
        clean = vh.nan_to_num(0, 0, 0)
        out[some, h], mean[some, h] = w @ clean, w @ clean.abs()
        big = q[some, h].abs() @ kh.nan_to_num(0, 0, 0).abs().T * abs(scale)
        size[some, h] = torch.where(seen, big, torch.zeros(())).amax(-1) if seen.numel() else 0
    return out, mean, size


def tree_visible(ctx, n, parents=None):
    """``[n, ctx]``: what the last n tokens see, causally, or as drafts of a tree (``parents``: -1 or an earlier draft)."""
    see = torch.arange(ctx) < torch.full((n, 1), ctx - n)
    for i in range(n):
        if parents is None:
            see[i, ctx - n:ctx - n + i + 1] = True
        else:
            b = i
            while b >= 0:
                see[i, ctx - n + b] = True
                b = parents[b]
    return see


def kept(pool, table, first, keep):
    """``pool [num_blocks, Hkv, bs, D]`` after the kept rows of every sequence moved; ``keep``: a list per sequence."""
    want, bs = pool.clone(), pool.shape[2]
    for s, row in enumerate(keep):
        for i, k in enumerate(row):
            a, b = first[s] + k, first[s] + i
            if a >= table.shape[1] * bs:
                continue
            want[table[s, b // bs], :, b % bs] = pool[table[s, a // bs], :, a % bs]
    return want
