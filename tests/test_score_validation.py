"""Refusals of the C ABI of normed heads, scores by a rule and block copies: every one happens on the host, before any device work,
so the pointers are placeholders that are never followed (runs without a GPU)."""
import ctypes

import pytest
import torch

from aicomp_amd import _lib, ops

P = 0x10000          # a non-null, 16-byte aligned placeholder
EINVAL, EUNSUPPORTED, EWORKSPACE = 1, 2, 4
F32, BF16, FP8, F16 = _lib.F32, _lib.BF16, _lib.FP8_E4M3, _lib.F16
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def err(lib):
    return lib.aicomp_kv_last_error().decode()


def norm(lib, **kw):
    a = dict(q=P, qo=P, qts=1024, qhs=128, qots=1024, qohs=128, k=P, v=P, kts=256, khs=128, qw=P, kw=P, eps=1e-6, cos=P, sin=P,
             ts=64, rows=100, rotary=128, inter=0, pos=P, kp=P, vp=P, slots=P, n=5, hq=8, hkv=2, d=128, bs=16, nb=64, dt=BF16,
             pdt=BF16, ks=None, vs=None, stream=None)
    a.update(kw)
    return lib.aicomp_qk_norm_rope_kv_append(*a.values())


def test_norm_rope_refusals(lib):
    assert norm(lib, n=0) == 0
    assert norm(lib, n=-1) == EINVAL and "negative" in err(lib)
    assert norm(lib, slots=None) == EINVAL and "null pointer" in err(lib)
    assert norm(lib, hkv=0) == EINVAL and "bad sizes" in err(lib)
    assert norm(lib, dt=FP8) == EUNSUPPORTED and norm(lib, pdt=F32) == EUNSUPPORTED
    assert norm(lib, pdt=FP8) == EINVAL and "k_scale" in err(lib)
    assert norm(lib, d=72, rotary=16) == EUNSUPPORTED and norm(lib, d=272, qhs=272, qohs=272, khs=272) == EUNSUPPORTED
    assert norm(lib, rotary=24) == EUNSUPPORTED and "rotary_dim" in err(lib)
    assert norm(lib, rotary=144) == EUNSUPPORTED and norm(lib, rotary=-16) == EUNSUPPORTED
    assert norm(lib, sin=None) == EINVAL and "tables" in err(lib)
    assert norm(lib, rows=0) == EINVAL and norm(lib, ts=60) == EINVAL
    assert norm(lib, ts=66) == EUNSUPPORTED and "16 bytes" in err(lib)
    assert norm(lib, eps=-1e-6) == EINVAL and norm(lib, eps=NAN) == EINVAL and norm(lib, eps=INF) == EINVAL
    assert norm(lib, qhs=64) == EINVAL and "overlap" in err(lib)
    assert norm(lib, kts=-8) == EINVAL
    assert norm(lib, qts=1028) == EUNSUPPORTED
    assert norm(lib, qw=P + 4) == EUNSUPPORTED and "aligned" in err(lib)


def attn(lib, **kw):
    a = dict(out=P, q=P, kp=P, vp=P, table=P, stride=8, lens=P, cu=None, seqs=4, total=4, max_q=1, hq=8, hkv=2, d=128, bs=16, mb=8,
             nb=64, scale=0.1, qd=BF16, kd=BF16, ks=None, vs=None, cap=0.0, slopes=None, window=0, first=None, prefix=None,
             longest=0, ws=None, wsb=0, stream=None)
    a.update(kw)
    return lib.aicomp_paged_score_attn(*a.values())


def test_score_refusals(lib):
    assert attn(lib, seqs=0) == 0 and attn(lib, total=0) == 0
    assert attn(lib, seqs=-1) == EINVAL and "negative" in err(lib)
    assert attn(lib, lens=None) == EINVAL and "null pointer" in err(lib)
    assert attn(lib, hq=7) == EINVAL and "not a multiple" in err(lib)
    assert attn(lib, d=80) == EUNSUPPORTED and "head_dim" in err(lib)
    assert attn(lib, qd=F32) == EUNSUPPORTED and "type pair" in err(lib)
    assert attn(lib, qd=F32, kd=FP8, ks=P, vs=P) == EUNSUPPORTED
    assert attn(lib, kd=FP8) == EINVAL and "k_scale" in err(lib)
    assert attn(lib, qd=9) == EINVAL
    assert attn(lib, mb=1 << 28, stride=1 << 28) == EINVAL and "table" in err(lib)
    assert attn(lib, stride=7) == EINVAL and "stride" in err(lib)
    assert attn(lib, window=-1) == EINVAL and "window" in err(lib)
    assert attn(lib, cap=-1.0) == EINVAL and "softcap" in err(lib)
    assert attn(lib, cap=NAN) == EINVAL and attn(lib, scale=INF) == EINVAL
    assert attn(lib, longest=-1) == EINVAL
    assert attn(lib, q=P + 2) == EUNSUPPORTED and "aligned" in err(lib)
    assert attn(lib, total=5) == EINVAL and "one row per sequence" in err(lib)
    assert attn(lib, prefix=P) == EINVAL
    assert attn(lib, cu=P, max_q=0) == EINVAL and "max_q_len" in err(lib)
    assert attn(lib, cu=P, max_q=5) == EINVAL


def test_score_caps(lib):
    for cu in (None, P):
        assert attn(lib, cu=cu, total=4, cap=1025.0) == EUNSUPPORTED and "softcap" in err(lib)
        assert attn(lib, cu=cu, total=4, cap=1e-40) == EUNSUPPORTED and "overflows" in err(lib)      # 3 * 0.1 / 1e-40 = 3e39
        assert attn(lib, cu=cu, total=4, scale=3e38) == EINVAL
    assert attn(lib, cap=INF) == EINVAL and attn(lib, cap=-1.0) == EINVAL and attn(lib, cap=NAN) == EINVAL


def test_numbers_beyond_32_bits_are_refused():
    """A window of 2^32 + 5 is not one of 5."""
    for name in ("window", "longest_context"):
        for bad in (2 ** 32 + 5, 2 ** 31, -2 ** 33):
            with pytest.raises(RuntimeError, match=name):
                ops._int32(bad, name)
    assert ops._int32(2 ** 31 - 1, "window") == 2 ** 31 - 1 and ops._int32(0, "window") == 0


@pytest.mark.routing("balanced", "library")
def test_score_workspace(lib, decode_routing):
    size = lambda rows, mb, window=0, longest=0: lib.aicomp_paged_score_workspace_bytes(rows, rows, 0, 8, 2, 128, 16, mb, BF16, BF16, window,
                                                                                        longest)
    need = size(4, 256)
    assert need > 0
    assert attn(lib, mb=256, stride=256) == EWORKSPACE and str(need) in err(lib)
    assert attn(lib, mb=256, stride=256, ws=P, wsb=need - 1) == EWORKSPACE
    assert attn(lib, mb=256, stride=256, ws=P + 4, wsb=need) == EINVAL and "aligned" in err(lib)
    if decode_routing == "library":                             # whole rows of a small call
        assert size(4, 2) == 0
        assert size(4, 256, window=32) == 0 and size(4, 256, longest=32) == 0
    assert size(0, 256) == 0 and size(4, 256, window=-1) == 0


def test_score_chunk_workspace(lib):
    size = lambda seqs, total, longest, mb, window=0, bound=0, dt=BF16, bs=16: lib.aicomp_paged_score_workspace_bytes(
        seqs, total, longest, 8, 2, 128, bs, mb, dt, dt, window, bound)
    need = size(1, 4, 4, 256)
    assert need > 0 and need % (4 * 8 * 130 * 4) == 0                       # sums, reference and weight of every part
    assert size(1, 4, 4, 2) == 0 and size(1, 4, 4, 256, window=32) == 0 and size(1, 4, 4, 256, bound=32) == 0      # short rows
    assert size(16, 65536, 4096, 256) == 0                                  # many rows
    assert size(1, 4, 4, 256, dt=F32) > 0 and size(1, 4, 4, 256, bs=32) == 0
    assert size(1, 0, 4, 256) == 0 and size(1, 4, -1, 256) == 0
    assert attn(lib, cu=P, mb=256, stride=256, total=4, max_q=4, ws=P, wsb=need - 1) == EWORKSPACE and str(need) in err(lib)
    assert attn(lib, cu=P, mb=256, stride=256, total=4, max_q=4, ws=P + 4, wsb=need) == EINVAL and "aligned" in err(lib)


def test_copy_refusals(lib):
    def call(pools=(P, P), bytes_=64, nb=8, pairs=P, n=2):
        return lib.aicomp_kv_copy_blocks((ctypes.c_void_p * max(1, len(pools)))(*pools), len(pools), bytes_, nb, pairs, n, None)
    assert call(pools=()) == 0 and call(n=0) == 0
    assert call(n=-1) == EINVAL and "negative" in err(lib)
    assert call(pools=(P, None)) == EINVAL and "pool 1" in err(lib)
    assert call(pairs=None) == EINVAL and "null pointer" in err(lib)
    assert call(bytes_=0) == EINVAL and call(nb=0) == EINVAL
    assert lib.aicomp_kv_copy_blocks(None, 2, 64, 8, P, 2, None) == EINVAL


def test_cpu_tensors_are_refused():
    pool = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    one32, one64 = torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.qk_norm_rope_kv_append(x, x, x, None, None, None, None, None, pool, pool, one64)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.paged_score_decode_attn(x, x, pool, pool, one32[None], one32, 1.0)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.paged_score_prefill_attn(x, x, pool, pool, one32[None], one32, torch.zeros(2, dtype=torch.int32), 1.0)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.copy_blocks([pool], torch.zeros(1, 2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="at least one pool"):
        ops.copy_blocks([], torch.zeros(1, 2, dtype=torch.int64))


def test_pair_tables_are_exact_far_out():
    inv = 1.0 / (10000.0 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64))
    cos, sin = ops.rotary_pair_tables(inv.float(), 70001, attention_scaling=1.25)
    want = 70000.0 * inv.float().double()
    assert cos.dtype == torch.float32 and cos.shape == (70001, 32)
    # one rounding of float64 values, the scaling's product among them
    assert (cos[70000].double() - want.cos() * 1.25).abs().max() <= 1.25 * 2.0 ** -24 + 1e-15
    assert (sin[70000].double() - want.sin() * 1.25).abs().max() <= 1.25 * 2.0 ** -24 + 1e-15
