"""Normed heads, scores by a rule and forked sequences as a decoder uses them: through the backend and the planner, against a plain
float32 model without a cache; recorded into graphs; by the native and the ctypes host routes; on other streams."""
import math
import threading

import pytest
import torch
import torch.nn.functional as F

from aicomp_amd import ops
from aicomp_amd.block_manager import StepPlanner
from aicomp_amd.generation import PagedAttentionBackend, ScheduleGeneration

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.routing("balanced", "library")


class RuledModel:
    """Three layers of a decoder whose heads are normed and partly rotated: a cap, a window with slopes, neither."""

    RULES = [dict(softcap=20.0), dict(window=24, slopes=True), {}]

    def __init__(self, device, dtype, hq=4, hkv=2, d=64, rotary=32, interleaved=False, vocab=97, hidden=128, norm=True, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d, self.interleaved, self.norm = hq, hkv, d, interleaved, norm
        w = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(device, dtype)
        self.embed = torch.randn(vocab, hidden, generator=g).to(device, dtype)
        self.qkv = [w((hq + 2 * hkv) * d, hidden) for _ in self.RULES]
        self.o = [w(hidden, hq * d) for _ in self.RULES]
        self.head = w(vocab, hidden)
        self.weights = [(1 + 0.2 * torch.randn(2, d, generator=g)).to(device) for _ in self.RULES]
        self.inv_freq = (1.0 / (10000.0 ** (torch.arange(0, rotary, 2).float() / rotary))).to(device)
        self.slopes = torch.exp2(-2.0 * torch.arange(1, hq + 1)).to(device)

    def backend(self, blocks, dtype, device, max_positions=512, kv_dtype=None):
        b = PagedAttentionBackend(len(self.RULES), blocks, self.hkv, self.d, dtype=dtype, device=device, inv_freq=self.inv_freq,
                                  max_positions=max_positions, interleaved=self.interleaved, kv_dtype=kv_dtype)
        for i, r in enumerate(self.RULES):
            if self.norm:
                b.set_head_norm(i, self.weights[i][0], self.weights[i][1], eps=1e-5)
            if r:
                b.set_score_rule(i, r.get("softcap", 0.0), self.slopes if r.get("slopes") else None, r.get("window", 0))
        return b

    @staticmethod
    def rms(x):
        return (x.float() * torch.rsqrt(x.float().pow(2).mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def paged(self, backend):
        def model(ids, positions):
            x, T = self.embed[ids], ids.numel()
            for i in range(len(self.RULES)):
                qkv = F.linear(self.rms(x), self.qkv[i]).view(T, self.hq + 2 * self.hkv, self.d)
                a = backend.attend(i, qkv[:, :self.hq], qkv[:, self.hq:self.hq + self.hkv], qkv[:, self.hq + self.hkv:])
                x = x + F.linear(a.reshape(T, -1), self.o[i])
            return F.linear(self.rms(x), self.head)
        return model

    def rotate(self, x, weight):
        """[S, H, D] float64: norm and rotation."""
        if self.norm:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * weight.double()
        r = 2 * self.inv_freq.numel()
        a = torch.arange(x.shape[0], device=x.device)[:, None, None].double() * self.inv_freq.double()
        if self.interleaved:
            u, v = x[..., 0:r:2], x[..., 1:r:2]
            t = torch.stack((u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()), -1).flatten(-2)
        else:
            u, v = x[..., :r // 2], x[..., r // 2:r]
            t = torch.cat((u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()), -1)
        return torch.cat((t, x[..., r:]), -1)

    def naive(self, ids, first=None, prefix=0):
        """ids [S] -> logits of the last token, the whole sequence at once, in float64 from the weights as they are."""
        x, S = self.embed[ids].double(), ids.numel()
        rms = lambda t: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6)
        at = torch.arange(S, device=ids.device)
        for i, rule in enumerate(self.RULES):
            qkv = F.linear(rms(x), self.qkv[i].double()).view(S, self.hq + 2 * self.hkv, self.d)
            q = self.rotate(qkv[:, :self.hq], self.weights[i][0])
            k = self.rotate(qkv[:, self.hq:self.hq + self.hkv], self.weights[i][1]).repeat_interleave(self.hq // self.hkv, 1)
            v = qkv[:, self.hq + self.hkv:].repeat_interleave(self.hq // self.hkv, 1)
            s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(self.d)
            if rule.get("softcap"):
                s = rule["softcap"] * torch.tanh(s / rule["softcap"])
            if rule.get("slopes"):
                s = s - self.slopes.double()[:, None, None] * (at[:, None] - at).abs()
            seen = (at <= at[:, None]) | (at < prefix)
            if rule.get("window"):
                seen &= at[:, None] - at < rule["window"]
            if first is not None:
                seen &= at >= first[:, None]
            a = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, -math.inf), -1), v)
            x = x + F.linear(a.reshape(S, -1), self.o[i].double())
        return F.linear(rms(x), self.head.double())[-1]


def close(got, want, dtype):
    """Logits of three layers: about ten roundings each of the residual stream and the projections, which add up like a random
    walk of relative steps eps / 2 over sums of 64 to 256 terms; 40 steps of the largest logit bound them."""
    tol = 40 * torch.finfo(dtype).eps / 2 * want.abs().max() + 1e-4
    assert (got.double() - want).abs().max() <= tol, ((got.double() - want).abs().max(), tol)


@BOTH
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved,d,rotary,norm", [(False, 64, 32, True), (True, 128, 128, True), (False, 64, 64, False),
                                                       (True, 64, 16, False)])
def test_generation_with_forks_and_compaction(device, dtype, interleaved, d, rotary, norm):
    m = RuledModel(device, dtype, d=d, rotary=rotary, interleaved=interleaved, norm=norm)
    b = m.backend(40, dtype, device)
    planner = StepPlanner(40, 16, max_seqs=6, max_seq_len=256, prefill_chunk=32, max_num_batched_tokens=64, device=device,
                          check_plans=True)
    gen = ScheduleGeneration(m.paged(b), b, planner)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 97, (n,), generator=g).to(device) for n in (70, 33, 48)]
    ids = torch.zeros(3, 70, dtype=torch.int64, device=device)
    for i, p in enumerate(prompts):
        ids[i, :p.numel()] = p
    logits = gen.prefill(ids, prompt_lens=[70, 33, 48])
    for i, p in enumerate(prompts):
        close(logits[i], m.naive(p), dtype)
    assert gen.fork(0) == 3 and gen.fork(2) == 4            # a partly filled last block, and none
    prompts += [prompts[0], prompts[2]]
    for step in range(20):
        tok = torch.randint(0, 97, (5,), generator=g).to(device)
        prompts = [torch.cat((p, tok[i:i + 1])) for i, p in enumerate(prompts)]
        logits = gen.decode_step(tok)
        if step in (0, 1, 19):
            for i, p in enumerate(prompts):
                close(logits[i], m.naive(p), dtype)
        if step == 5:                                      # the parent of a fork leaves, the pool is compacted
            planner.finish(gen._batch.pop(0))
            prompts.pop(0)
            pairs = planner.compact()
            assert pairs.shape[0] > 0
            b.copy_blocks(pairs)
            prompts.append(prompts[0])
            assert gen.fork(0) == 4
    gen.clear_cache()
    assert planner.alloc.num_used == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_documents_and_prefixes(device, dtype):
    """A chunked prompt of packed documents, and one whose first part sees itself as a whole."""
    m = RuledModel(device, dtype)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 97, (75,), generator=g).to(device)
    first = (torch.arange(75, device=device, dtype=torch.int32) // 20) * 20
    for kw, want in (({"first_keys": first}, m.naive(ids, first=first)),
                     ({"prefix_lens": torch.tensor([20], dtype=torch.int32, device=device)}, m.naive(ids, prefix=20))):
        b = m.backend(10, dtype, device)
        planner = StepPlanner(10, 16, max_seqs=2, max_seq_len=100, prefill_chunk=40, device=device)
        planner.add_request("s", 75)
        model, out = m.paged(b), None
        for _ in range(2):
            plan = planner.schedule()
            at = plan.positions
            b.begin_step(plan, **{k: (v[at].contiguous() if k == "first_keys" else v) for k, v in kw.items()})
            out = model(ids[at], at)
        close(out[-1], want, dtype)


def _calls(device, seed=0):
    """Arguments of every call, small."""
    g = torch.Generator(device=device).manual_seed(seed)
    BF = torch.bfloat16
    mk = lambda *s: torch.randn(*s, generator=g, device=device).to(BF)
    S, hq, hkv, d, nb = 3, 8, 2, 128, 200
    a = dict(kp=mk(nb, hkv, 16, d), vp=mk(nb, hkv, 16, d), q=mk(S, hq, d), k=mk(S, hkv, d), v=mk(S, hkv, d),
             table=torch.randperm(nb, generator=g, device=device)[:S * 60].view(S, 60).to(torch.int32),
             lens=torch.tensor([900, 17, 300], dtype=torch.int32, device=device), pos=torch.tensor([899, 16, 299], device=device),
             w=1 + 0.1 * torch.randn(2, d, generator=g, device=device), slopes=torch.rand(hq, generator=g, device=device),
             cq=mk(50, hq, d), ccu=torch.tensor([0, 33, 50], dtype=torch.int32, device=device),
             clens=torch.tensor([600, 40], dtype=torch.int32, device=device),
             pairs=torch.tensor([[190, 191], [192, 193]], device=device))
    a["cos"], a["sin"] = ops.rotary_pair_tables(torch.rand(32, generator=g, device=device), 1000)
    a["slots"] = a["table"][torch.arange(S, device=device), a["pos"] // 16].long() * 16 + a["pos"] % 16
    a["out"], a["cout"], a["qr"] = torch.empty_like(a["q"]), torch.empty_like(a["cq"]), torch.empty_like(a["q"])
    return a


def _step(a):
    ops.qk_norm_rope_kv_append(a["q"], a["k"], a["v"], a["w"][0], a["w"][1], a["cos"], a["sin"], a["pos"], a["kp"], a["vp"],
                               a["slots"], query_out=a["qr"])
    ops.paged_score_decode_attn(a["out"], a["qr"], a["kp"], a["vp"], a["table"], a["lens"], 0.09, 30.0, a["slopes"])
    ops.paged_score_prefill_attn(a["cout"], a["cq"], a["kp"], a["vp"], a["table"][:2], a["clens"], a["ccu"], 0.09, 33, 30.0,
                                 a["slopes"], window=100)
    ops.copy_blocks([a["kp"], a["vp"]], a["pairs"])


def _results(a):
    return [a[n].clone() for n in ("qr", "out", "cout", "kp", "vp")]


@BOTH
def test_native_and_ctypes_routes_agree(device, monkeypatch):
    a = _calls(device)
    _step(a)
    native = _results(a)
    monkeypatch.setattr(ops, "_FAST", None)
    a = _calls(device)
    _step(a)
    for x, y in zip(native, _results(a)):
        assert torch.equal(x, y)


@BOTH
def test_two_graphs_side_by_side(device):
    """Two recorded steps replayed at once on two streams, with eager steps between: each as its eager step is."""
    cases, graphs, want = [_calls(device, 1), _calls(device, 2)], [], []
    eager = _calls(device, 3)
    for a in cases:
        _step(a)
        _step(a)                                            # (the first copied blocks that the second reads: from here on steps repeat)
        want.append(_results(a))
    torch.cuda.synchronize()
    for a in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _step(a)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for a in cases:
            for n in ("qr", "out", "cout"):
                a[n].zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        _step(eager)
        torch.cuda.synchronize()
        for a, w in zip(cases, want):
            for x, y in zip(_results(a), w):
                assert torch.equal(x, y)


def test_replays_follow_the_lengths(device):
    """A recorded decode step whose context grows past what the table's use was when it was recorded."""
    a = _calls(device)
    call = lambda out: ops.paged_score_decode_attn(out, a["q"], a["kp"], a["vp"], a["table"], a["lens"], 0.09, 30.0, None, 200)
    a["lens"].fill_(5)
    call(a["out"])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(a["out"])
    for lens in ([5, 6, 7], [960, 100, 0], [33, 950, 512]):
        a["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        assert torch.equal(a["out"], call(torch.empty_like(a["out"])))


def test_another_stream(device):
    a, b = _calls(device), _calls(device)
    _step(a)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        _step(b)
    torch.cuda.synchronize()
    for x, y in zip(_results(a), _results(b)):
        assert torch.equal(x, y)


def test_repeatable(device):
    a = _calls(device)
    _step(a)
    _step(a)                                                # (reads blocks that the first one copied)
    first = _results(a)
    for _ in range(3):
        _step(a)
        for x, y in zip(first, _results(a)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("change", [
    dict(slots=lambda t: t.int()), dict(w=lambda t: t.bfloat16()), dict(cos=lambda t: t[:, ::2]), dict(k=lambda t: t.float()),
    dict(slopes=lambda t: t[:3]), dict(lens=lambda t: t.long()), dict(table=lambda t: t[:2]), dict(ccu=lambda t: t[:-1].long()),
    dict(pairs=lambda t: t.int()), dict(kp=lambda t: t.transpose(0, 1)), dict(lens=lambda t: t.cpu()),
    dict(pairs=lambda t: t.t().contiguous().t())])
def test_what_the_native_route_declines_is_refused_by_name(device, change):
    a = _calls(device)
    for n, f in change.items():
        a[n] = f(a[n])
    with pytest.raises(RuntimeError):
        _step(a)


@pytest.mark.parametrize("native", [True, False])
@BOTH
def test_two_threads_on_one_stream(device, monkeypatch, native):
    """Divided decode rows and divided chunks of two threads: each thread's results are those of its calls alone."""
    if not native:
        monkeypatch.setattr(ops, "_FAST", None)
    cases = []
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        pools = [torch.randn(400, 2, 16, 128, device=device, generator=g).bfloat16() for _ in range(2)]
        q = torch.randn(40, 8, 128, device=device, generator=g).bfloat16()
        table = torch.randperm(400, device=device, generator=g).to(torch.int32).view(2, 200)
        lens = torch.tensor([3000, 1700], dtype=torch.int32, device=device)
        cu = torch.tensor([0, 30, 40], dtype=torch.int32, device=device)

        def call(q=q, pools=pools, table=table, lens=lens, cu=cu):
            a, b = torch.empty_like(q[:2]), torch.empty_like(q)
            ops.paged_score_decode_attn(a, q[:2], *pools, table, lens, 0.09, 30.0)
            ops.paged_score_prefill_attn(b, q, *pools, table, lens, cu, 0.09, 30, 30.0)
            return a, b
        cases.append(call)
    want = [c() for c in cases]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            for _ in range(50):
                got[i].append(cases[i]())
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
        for a, b in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])
