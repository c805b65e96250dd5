"""The largest rows of latent caches that the C ABI takes, as the header states them, and sizes whose sums and products pass the integers
they are held in: refused on the host, before any device work (runs without a GPU; the pointers are never followed)."""
import os
import re

import pytest

from test_rows_validation import BF16, EINVAL, EUNSUPPORTED, F16, F32, append, err, latent, lib, prompt, tree  # noqa: F401

BIG = 2 ** 31 - 16                      # the largest multiple of 16 in 32 bits


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_rows_of_latent_attention(lib, dt):
    for c, d in ((1024, 272), (1040, 16), (16, 1280), (1024, BIG), (BIG, 16), (BIG, BIG), (BIG, 1040)):
        assert latent(lib, c=c, d=d, dt=dt) == EUNSUPPORTED and "1280" in err(lib), (c, d)
        assert lib.aicomp_paged_latent_workspace_bytes(4, 20, 9, 16, c, d, 16, 8, dt, 0) == 0


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_heads_of_prompts(lib, dt):
    for n, d, dv in ((1264, 32, 128), (1280, 16, 16), (128, 64, 1040), (BIG, BIG, 128), (BIG, 64, 128), (64, BIG, 128), (BIG, 32, 16),
                     (128, 64, BIG)):
        assert prompt(lib, n=n, d=d, dv=dv, dt=dt) == EUNSUPPORTED and "1280" in err(lib), (n, d, dv)


def test_appended_rows(lib):
    assert append(lib, c=1040, ls=1104) == EUNSUPPORTED and "1024" in err(lib)
    for d in (65552, 2 ** 20, BIG):
        assert append(lib, d=d, ls=2 ** 40, ts=2 ** 40, qhs=2 ** 40, qohs=2 ** 40, qts=2 ** 44, qots=2 ** 44) == EUNSUPPORTED and \
            "65536" in err(lib)


def test_tokens_and_heads_of_an_append(lib):
    for n in (2 ** 32, 2 ** 60, 2 ** 62, 2 ** 63 - 1, 2 ** 63 - 8):
        assert append(lib, n=n) == EINVAL and "one launch" in err(lib), n
        assert append(lib, n=n, q=None, qo=None, heads=0) == EINVAL and "one launch" in err(lib), n
    for heads in (2 ** 31 - 1, 2 ** 31 - 2):
        for n in (2, 5, 2 ** 33):
            assert append(lib, heads=heads, n=n) == EINVAL and "one launch" in err(lib), (heads, n)

def test_the_header_states_them():
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "aicomp_kv.h")).read()
    text = re.sub(r"\s+\*?\s*", " ", text)
    assert "latent_dim + rope_dim at most 1280" in text and "nope_dim + rope_dim at most 1280, value_dim at most 1024" in text
    assert "rope_dim at most 65536" in text
