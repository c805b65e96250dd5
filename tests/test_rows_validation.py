"""Refusals of the C ABI of latent rows, trees of drafts and accepted rows, and of their tensor-level calls: every one happens on the
host, before any device work, so the pointers are placeholders that are never followed (runs without a GPU)."""
import ctypes

import numpy as np
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


def append(lib, **kw):
    a = dict(latent=P, ls=576, weight=P, eps=1e-6, cos=P, sin=P, ts=32, rows=100, inter=0, pos=P, q=P, qo=P, qts=192 * 16, qhs=192,
             qots=576 * 16, qohs=576, out=None, os=0, pool=P, slots=P, n=5, heads=16, c=512, d=64, bs=16, nb=64, dt=BF16, stream=None)
    a.update(kw)
    return lib.aicomp_latent_kv_append(*a.values())


def test_append_refusals(lib):
    assert append(lib, n=0) == 0
    assert append(lib, n=-1) == EINVAL and "negative" in err(lib)
    for name in ("latent", "cos", "sin", "pool", "slots", "q", "qo"):
        assert append(lib, **{name: None}) == EINVAL and "null pointer" in err(lib)
    assert append(lib, heads=0) == EINVAL and append(lib, bs=0) == EINVAL and append(lib, nb=0) == EINVAL and append(lib, heads=-1) == EINVAL
    assert append(lib, nb=2 ** 62) == EINVAL
    assert append(lib, dt=FP8) == EUNSUPPORTED and append(lib, dt=9) == EUNSUPPORTED
    assert append(lib, c=520) == EUNSUPPORTED and append(lib, d=24) == EUNSUPPORTED and append(lib, d=0) == EUNSUPPORTED
    assert append(lib, c=1040, ls=1104) == EUNSUPPORTED
    assert append(lib, rows=0) == EINVAL and append(lib, ts=28) == EINVAL and append(lib, ts=34) == EUNSUPPORTED
    assert append(lib, eps=NAN) == EINVAL and append(lib, eps=-1.0) == EINVAL and append(lib, eps=INF) == EINVAL
    assert append(lib, ls=570) == EINVAL and append(lib, qhs=32) == EINVAL and append(lib, qots=-8) == EINVAL
    assert append(lib, out=P, os=570) == EINVAL and append(lib, out=P, os=580) == EUNSUPPORTED
    assert append(lib, ls=580) == EUNSUPPORTED and append(lib, qhs=196) == EUNSUPPORTED
    assert append(lib, pool=P + 8) == EUNSUPPORTED and "aligned" in err(lib)
    assert append(lib, n=2 ** 31) == EINVAL and "one launch" in err(lib)


def latent(lib, **kw):
    a = dict(out=P, q=P, pool=P, table=P, stride=8, lens=P, cu=P, masks=P, words=1, seqs=4, total=20, max_q=9, heads=16, c=512, d=64, bs=16,
             mb=8, nb=64, scale=0.1, dt=BF16, longest=0, ws=None, wsb=0, stream=None)
    a.update(kw)
    return lib.aicomp_paged_latent_attn(*a.values())


def tree(lib, **kw):
    a = dict(out=P, q=P, kp=P, vp=P, table=P, stride=8, lens=P, cu=P, masks=P, words=1, seqs=4, total=20, max_q=9, hq=8, hkv=2, d=128,
             bs=16, mb=8, nb=64, scale=0.1, qd=BF16, kd=BF16, ks=None, vs=None, longest=0, ws=None, wsb=0, stream=None)
    a.update(kw)
    return lib.aicomp_paged_tree_attn(*a.values())


@pytest.mark.parametrize("call", [latent, tree])
def test_refusals_of_both_paged_calls(lib, call):
    assert call(lib, seqs=0) == 0 and call(lib, total=0) == 0
    assert call(lib, seqs=-1) == EINVAL and call(lib, total=-1) == EINVAL
    for name in ("out", "q", "table", "lens"):
        assert call(lib, **{name: None}) == EINVAL and "null pointer" in err(lib)
    assert call(lib, bs=0) == EINVAL and call(lib, mb=0) == EINVAL and call(lib, nb=0) == EINVAL
    assert call(lib, mb=2 ** 30, stride=2 ** 30) == EINVAL
    assert call(lib, stride=7) == EINVAL and "stride" in err(lib)
    assert call(lib, scale=NAN) == EINVAL and call(lib, scale=INF) == EINVAL and call(lib, scale=3e38) == EINVAL
    assert call(lib, longest=-1) == EINVAL
    assert call(lib, max_q=0) == EINVAL and call(lib, max_q=21) == EINVAL and "max_q_len" in err(lib)
    assert call(lib, words=0) == EINVAL and call(lib, words=-1) == EINVAL and "masks" in err(lib)
    assert call(lib, masks=P + 4) == EINVAL
    assert call(lib, q=P + 8) == EUNSUPPORTED and "aligned" in err(lib)


def test_latent_refusals(lib):
    assert latent(lib, heads=0) == EINVAL and latent(lib, heads=70000) == EINVAL
    assert latent(lib, c=0) == EUNSUPPORTED and latent(lib, c=500) == EUNSUPPORTED and latent(lib, d=24) == EUNSUPPORTED
    assert latent(lib, d=-16) == EUNSUPPORTED and latent(lib, c=1040) == EUNSUPPORTED
    assert latent(lib, dt=FP8) == EUNSUPPORTED
    assert latent(lib, cu=None) == EINVAL and latent(lib, cu=None, masks=None, words=0) == EINVAL and "one row per sequence" in err(lib)
    assert latent(lib, cu=None, total=4) == EINVAL and "need cu_q_lens" in err(lib)
    assert latent(lib, masks=None) == EINVAL


def test_tree_refusals(lib):
    assert tree(lib, cu=None) == EINVAL and tree(lib, masks=None) == EINVAL
    assert tree(lib, hq=7) == EINVAL and "not a multiple" in err(lib)
    assert tree(lib, d=80) == EUNSUPPORTED and tree(lib, qd=F32) == EUNSUPPORTED and tree(lib, kd=F16) == EUNSUPPORTED
    assert tree(lib, kd=FP8) == EINVAL and "k_scale" in err(lib)


def prompt(lib, **kw):
    a = dict(out=P, q=P, k=P, kts=4096, khs=256, r=P, rts=576, v=P, vts=4096, vhs=256, cu=P, cuk=P, seqs=3, total=30, keys=50, max_q=20,
             heads=16, n=128, d=64, dv=128, scale=0.1, dt=BF16, stream=None)
    a.update(kw)
    return lib.aicomp_latent_prompt_attn(*a.values())


def test_prompt_refusals(lib):
    assert prompt(lib, seqs=0) == 0 and prompt(lib, total=0) == 0
    assert prompt(lib, seqs=-1) == EINVAL and prompt(lib, keys=-1) == EINVAL
    for name in ("out", "q", "k", "r", "v", "cu", "cuk"):
        assert prompt(lib, **{name: None}) == EINVAL and "null pointer" in err(lib)
    assert prompt(lib, heads=0) == EINVAL and prompt(lib, heads=70000) == EINVAL
    assert prompt(lib, n=120) == EUNSUPPORTED and prompt(lib, d=0) == EUNSUPPORTED and prompt(lib, dv=8) == EUNSUPPORTED
    assert prompt(lib, dt=FP8) == EUNSUPPORTED
    assert prompt(lib, max_q=0) == EINVAL and prompt(lib, max_q=31) == EINVAL
    assert prompt(lib, scale=NAN) == EINVAL
    assert prompt(lib, kts=-8) == EINVAL and prompt(lib, rts=577) == EUNSUPPORTED and prompt(lib, vhs=4) == EUNSUPPORTED
    assert prompt(lib, v=P + 2) == EUNSUPPORTED and "aligned" in err(lib)


def keep(lib, **kw):
    a = dict(pools=(ctypes.c_void_p * 2)(P, P), n=2, row=256, hkv=2, bs=16, nb=64, table=P, stride=8, mb=8, first=P, keep=P, cu=P, seqs=3,
             total=5, stream=None)
    a.update(kw)
    return lib.aicomp_kv_keep_rows(*a.values())


def test_keep_refusals(lib):
    assert keep(lib, n=0) == 0 and keep(lib, seqs=0) == 0 and keep(lib, total=0) == 0
    assert keep(lib, n=-1) == EINVAL and keep(lib, total=-1) == EINVAL
    assert keep(lib, table=None) == EINVAL and keep(lib, pools=None) == EINVAL and keep(lib, keep=None) == EINVAL
    assert keep(lib, pools=(ctypes.c_void_p * 2)(P, None)) == EINVAL and "pool 1" in err(lib)
    assert keep(lib, row=0) == EINVAL and keep(lib, hkv=0) == EINVAL and keep(lib, mb=9) == EINVAL and keep(lib, nb=0) == EINVAL
    assert keep(lib, row=2 ** 31 - 1) == EINVAL and keep(lib, seqs=2 ** 24) == EINVAL and "one launch" in err(lib)


def test_calls_refuse_tensors_of_the_host():
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    pool, i32 = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.paged_tree_attn(x, x, pool, pool, i32[None], i32[:1], i32, torch.zeros(1, 1, dtype=torch.int64), 1.0)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.paged_latent_attn(x, x, pool[:, 0], i32[None], i32[:1], 1.0)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.latent_kv_append(x[0], None, torch.zeros(4, 8), torch.zeros(4, 8), None, pool[:, 0], torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.latent_prompt_attn(x, x, x, x[0], x, i32, i32, 1.0)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.keep_rows([pool], i32[None], i32[:1], i32[:1], i32)


def test_tree_masks():
    got = ops.tree_masks([[-1, 0, 0, 2], [], [-1, -1]])
    assert got.dtype == np.int64 and got.tolist() == [[1], [3], [5], [13], [1], [2]]
    chain = ops.tree_masks([list(range(-1, 129))])
    assert chain.shape == (130, 3) and chain[129].tolist() == [-1, -1, 3] and chain[63].tolist() == [-1, 0, 0]
    assert ops.tree_masks([]).shape == (0, 1)
    for bad in ([0], [-1, 1], [-1, -2], [-1, 5]):
        with pytest.raises(ValueError, match="parent"):
            ops.tree_masks([bad])


def test_a_pool_is_moved_once(lib):
    """The second of two moves of one pool would start from what the first has moved already."""
    bytes_ = 64 * 2 * 16 * 256
    for pools in ((P, P), (P, P + bytes_ - 256), (P + bytes_ - 16, P)):
        assert keep(lib, pools=(ctypes.c_void_p * 2)(*pools)) == EINVAL and "overlap" in err(lib)
    assert keep(lib, pools=(ctypes.c_void_p * 4)(P, P + 2 * bytes_, P + bytes_, P + 2 * bytes_ - 1), n=4) == EINVAL and "overlap" in err(lib)
    assert keep(lib, nb=2 ** 60) == EINVAL and "bytes" in err(lib)


def test_sizes_that_pass_32_bits_are_refused(lib):
    """A kernel's loop over the entries, and a token's place in its table, are 32 bits."""
    pools = (ctypes.c_void_p * 2)(P, P + 2 ** 30)
    assert keep(lib, pools=pools, total=2 ** 31 - 1) == EINVAL and keep(lib, pools=pools, total=2 ** 31 - 8) == EINVAL
    assert keep(lib, pools=pools, mb=2 ** 27, stride=2 ** 27) == EINVAL and "sizes" in err(lib)
    for call in (latent, tree):
        assert call(lib, mb=2 ** 27 - 1, stride=2 ** 27) == EINVAL and "sizes" in err(lib)
        assert call(lib, total=2 ** 31 - 9) == EINVAL and "max_q_len" in err(lib)
    assert prompt(lib, keys=2 ** 31 - 1) == EINVAL and prompt(lib, total=2 ** 31 - 500) == EINVAL and "sizes" in err(lib)
