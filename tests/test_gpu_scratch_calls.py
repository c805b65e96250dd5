"""Two threads on one stream, each of whose calls needs the stream's scratch for partials that a second kernel joins: every result is
that of the thread's calls alone."""
import threading

import pytest
import torch

from aicomp_amd import _lib, ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def cases(device):
    """Divided decode rows through a prepared call, plain and by a rule; divided chunks in their default form."""
    g = torch.Generator(device=device).manual_seed(7)
    mk = lambda *s: torch.randn(*s, generator=g, device=device).to(BF)
    pools, q = (mk(400, 2, 16, 128), mk(400, 2, 16, 128)), mk(40, 8, 128)
    steps = [p.clone() for p in pools]
    table = torch.randperm(400, device=device, generator=g).to(torch.int32).view(2, 200)
    lens = torch.tensor([3000, 1700], dtype=torch.int32, device=device)
    cu = torch.tensor([0, 30, 40], dtype=torch.int32, device=device)
    prepared = ops.PreparedDecode(*pools, table, lens, 8, BF, 0.09)
    assert prepared.need > 0
    registered, out = _lib.torch_ops(), lambda: torch.empty_like(q[:2])
    # the operator's step: row 3000 of its lengths, both sequences in tables of their own
    rows = torch.arange(3002, dtype=torch.int32, device=device)[:, None].expand(-1, 2).contiguous()
    wide, kv = torch.randperm(400, device=device, generator=g).to(torch.int32).view(2, 200), mk(2, 2, 1, 128)

    def by_operator():
        o = out()
        registered.paged_decode_attn(o, q[:2], *pools, table, lens, 0.09)
        return o
    return {"operator": by_operator,
            "step": lambda: registered.decode_step(q[:2, :, None], kv, kv, *steps, wide, rows, 2999, 4, 0.09),
            "prepared": lambda: prepared(torch.empty_like(q[:2]), q[:2]),
            "plain": lambda: ops.paged_decode_attn(torch.empty_like(q[:2]), q[:2], *pools, table, lens, 0.09),
            "rows": lambda: ops.paged_score_decode_attn(torch.empty_like(q[:2]), q[:2], *pools, table, lens, 0.09, 30.0),
            "chunks": lambda: ops.paged_score_prefill_attn(torch.empty_like(q), q, *pools, table, lens, cu, 0.09, softcap=30.0)}


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("pair", [("prepared", "chunks"), ("prepared", "rows"), ("plain", "chunks"), ("prepared", "plain"),
                                  ("operator", "operator"), ("operator", "step")], ids="-".join)
def test_two_threads_on_one_stream(device, monkeypatch, pair, native):
    if not native:
        monkeypatch.setattr(ops, "_FAST", None)
    calls = [cases(device)[name] for name in pair]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            for _ in range(60):
                got[i].append(calls[i]())
        except Exception as e:                                          # (reported by the test, not by the thread)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
