"""Calls of two threads that share a stream's scratch: between taking the buffer and the end of its launches a call is alone, whichever
pair of entry points it is (the library is a stand-in that says which calls are inside it; runs without a GPU)."""
import itertools
import threading
import time
from contextlib import nullcontext

import pytest
import torch

from aicomp_amd import _lib, ops

BF = torch.bfloat16
ENTRIES = ("aicomp_paged_decode_attn", "aicomp_paged_decode_attn_append", "aicomp_paged_score_attn")


class Library:
    """Entry points that take a while, as one does that waits for room in the stream's queue."""

    def __init__(self):
        self.inside, self.most, self.calls = 0, 0, []
        for name in ENTRIES:
            setattr(self, name, self._entry(name))

    def _entry(self, name):
        def call(*args):
            self.inside += 1
            self.most = max(self.most, self.inside)
            time.sleep(0.02)
            self.inside -= 1
            self.calls.append(name)
            return 0
        return call

    def aicomp_paged_decode_workspace_bytes(self, *args):
        return 256

    def aicomp_paged_score_workspace_bytes(self, *args):
        return 256


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    monkeypatch.setattr(ops, "_FAST", None)
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_req", lambda ok, msg: None)              # (the tensors are the host's)
    monkeypatch.setattr(ops, "_stream", lambda t: 0)
    monkeypatch.setattr(ops, "_current_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_guard", lambda t: nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    return lib


def users(lib):
    pool = torch.zeros(4, 2, 16, 64, dtype=BF)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([40], dtype=torch.int32)
    q, kv = torch.zeros(1, 4, 64, dtype=BF), torch.zeros(1, 2, 64, dtype=BF)
    cu = torch.tensor([0, 1], dtype=torch.int32)
    prepared = ops.PreparedDecode(pool, pool, table, lens, 4, BF, 0.1)
    return {
        "decode": lambda: ops.paged_decode_attn(torch.empty_like(q), q, pool, pool, table, lens, 0.1),
        "decode_append": lambda: ops.paged_decode_attn(torch.empty_like(q), q, pool, pool, table, lens, 0.1, new_key=kv, new_value=kv),
        "prepared": lambda: prepared(torch.empty_like(q), q),
        "prepared_append": lambda: prepared(torch.empty_like(q), q, kv, kv),
        "step4d": lambda: prepared.step4d(torch.empty(1, 4, 1, 64, dtype=BF), q[:, :, None], kv[:, :, None], kv[:, :, None], 2, lens,
                                          ready=lambda: None),
        "score_decode": lambda: ops.paged_score_decode_attn(torch.empty_like(q), q, pool, pool, table, lens, 0.1),
        "score_prefill": lambda: ops.paged_score_prefill_attn(torch.empty_like(q), q, pool, pool, table, lens, cu, 0.1),
    }


NAMES = ("decode", "decode_append", "prepared", "prepared_append", "step4d", "score_decode", "score_prefill")


@pytest.mark.parametrize("pair", list(itertools.combinations_with_replacement(NAMES, 2)), ids="-".join)
def test_one_call_at_a_time(lib, pair):
    calls = users(lib)
    start, errors = threading.Barrier(2), []

    def work(name):
        try:
            start.wait()
            for _ in range(3):
                calls[name]()
        except Exception as e:                                          # (reported by the test, not by the thread)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(name,)) for name in pair]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert len(lib.calls) == 6 and lib.most == 1, lib.most


def test_a_call_made_in_ready_does_not_wait_for_itself(lib):
    """``step4d`` calls ``ready`` right before its launch; what it does may be a call with scratch."""
    calls = users(lib)
    pool = torch.zeros(4, 2, 16, 64, dtype=BF)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([40], dtype=torch.int32)
    q, kv = torch.zeros(1, 4, 1, 64, dtype=BF), torch.zeros(1, 2, 1, 64, dtype=BF)
    ops.PreparedDecode(pool, pool, table, lens, 4, BF, 0.1).step4d(torch.empty_like(q), q, kv, kv, 2, lens, ready=calls["decode"])
    assert lib.calls == ["aicomp_paged_decode_attn", "aicomp_paged_decode_attn_append"]
