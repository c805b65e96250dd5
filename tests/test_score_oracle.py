"""The two forms of the float64 oracle of attention by a score rule agree: key by key, and all rows of a head at once."""
import pytest
import torch

from oracle.score_oracle import score_attention, score_attention_rows


@pytest.mark.parametrize("rule", [{}, {"cap": 5.0}, {"slopes": True, "window": 7}, {"prefix": 20, "cap": 2.0}, {"first": True, "prefix": 9},
                                  {"cap": 3.0, "slopes": True, "window": 11, "first": True, "prefix": 30}])
@pytest.mark.parametrize("n,ctx", [(1, 1), (13, 40), (40, 40)])
def test_all_rows_at_once(rule, n, ctx):
    g = torch.Generator().manual_seed(n)
    q, k, v = torch.randn(n, 4, 16, generator=g), torch.randn(ctx, 2, 16, generator=g), torch.randn(ctx, 2, 16, generator=g)
    kw = dict(cap=rule.get("cap", 0.0), slopes=torch.rand(4, generator=g) if rule.get("slopes") else None, window=rule.get("window", 0),
              first_keys=torch.randint(-2, ctx + 2, (n,), generator=g) if rule.get("first") else None, prefix=rule.get("prefix", 0))
    for a, b in zip(score_attention(q, k, v, ctx - n, 0.25, **kw), score_attention_rows(q, k, v, ctx - n, 0.25, **kw)):
        assert (a - b).abs().max() <= 1e-13 * max(1.0, float(a.abs().max()))
