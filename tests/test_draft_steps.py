"""Steps of drafted tokens on the host: what the planner plans for a tree, what it leaves when some of its drafts are kept, and which
drafts a model's picks accept."""
import numpy as np
import pytest
import torch

from aicomp_amd.block_manager import OutOfBlocks, StepPlanner
from aicomp_amd.generation import accept_drafts
from oracle.rows_oracle import tree_visible


def planner(num_blocks=32, **kw):
    kw = {"max_seqs": 6, "max_seq_len": 128, "max_num_batched_tokens": 64, "prefill_chunk": 64, "block_size": 16, "check_plans": True,
          "device": "cpu", **kw}
    return StepPlanner(num_blocks=num_blocks, **kw)


def started(lens, **kw):
    p = planner(**kw)
    for i, n in enumerate(lens):
        p.add_request(f"s{i}", n)
    while p.schedule(decode=()) is not None:
        pass
    return p


def test_a_step_of_drafts():
    p = started([15, 30])
    tree, line = [-1, 0, 0, 1, 2, -1], [-1, 0]
    plan = p.schedule_drafts({"s1": tree, "s0": line})
    assert plan.seq_ids == ["s1", "s0"] and plan.num_prefill_seqs == 2 and plan.max_q_len == 6 and plan.total_new_tokens == 8
    assert plan.context_lens.tolist() == [36, 17] and plan.cu_q_lens.tolist() == [0, 6, 8]
    assert plan.positions.tolist() == [30, 31, 31, 32, 32, 30, 15, 16]
    assert plan.host_positions.tolist() == plan.positions.tolist()
    places = [30, 31, 32, 33, 34, 35, 15, 16]
    rows = [0] * 6 + [1] * 2
    assert plan.slot_mapping.tolist() == [int(plan.block_table[r, x // 16]) * 16 + x % 16 for r, x in zip(rows, places)]
    want = tree_visible(36, 6, tree)[:, 30:].tolist()
    got = [[bool(int(m) >> a & 1) for a in range(6)] for m in plan.tree_masks[:6, 0].tolist()]
    assert got == want and plan.tree_masks[6:, 0].tolist() == [1, 3]
    # the lengths stay until some drafts are kept, and nothing else is planned
    assert p.context_len("s0") == 15 and p.context_len("s1") == 30
    for call in (p.schedule, p.compact, lambda: p.fork("s0", "x"), lambda: p.schedule_drafts({"s0": [-1]})):
        with pytest.raises(ValueError, match="still open"):
            call()
    kept = p.keep_drafts(plan, {"s1": [0, 2, 4]})
    assert kept.first.tolist() == [30, 15] and kept.keep.tolist() == [0, 2, 4] and kept.cu_keep.tolist() == [0, 3, 3]
    assert kept.block_table is plan.block_table and kept.moves
    assert p.context_len("s1") == 33 and p.context_len("s0") == 15
    assert p.alloc.num_used == 3 + 1                           # s0's second block, opened for its drafts, is free again
    nxt = p.schedule()
    assert dict(zip(nxt.seq_ids, nxt.positions.tolist())) == {"s0": 15, "s1": 33}
    with pytest.raises(ValueError, match="open step"):
        p.keep_drafts(plan, {})


def test_first_drafts_move_nothing():
    p = started([15, 30])
    plan = p.schedule_drafts({"s0": [-1, 0, 1], "s1": [-1, 0, 0]})
    kept = p.keep_drafts(plan, {"s0": [0, 1, 2], "s1": [0, 1]})
    assert not kept.moves and p.context_len("s0") == 18 and p.context_len("s1") == 32 and p.alloc.num_used == 2 + 2
    plan = p.schedule_drafts({"s1": [-1, 0, 0]})
    assert p.keep_drafts(plan, {"s1": [0, 2]}).moves and p.alloc.num_used == 2 + 3
    plan = p.schedule_drafts({"s1": [-1, 0, 0]})
    kept = p.keep_drafts(plan, {})
    assert not kept.moves and kept.keep.numel() == 0 and p.context_len("s1") == 34


def test_refusals_leave_the_planner_as_it_was():
    p = started([15, 30], num_blocks=4)
    p.add_request("waits", 40)
    used, table = p.alloc.num_used, p._tab.copy()
    for parents, match in (({}, "no sequences"), ({"s0": []}, "no drafts"), ({"x": [-1]}, "not running"), ({"waits": [-1]}, "not running"),
                           ({"s0": [0]}, "comes before"), ({"s0": [-1, 2, 0]}, "comes before"), ({"s0": [-2]}, "comes before"),
                           ({"s0": [-1] * 114}, "max_seq_len"), ({"s0": [-1] * 40, "s1": [-1] * 40}, "a step's 64")):
        with pytest.raises(ValueError, match=match):
            p.schedule_drafts(parents)
    with pytest.raises(OutOfBlocks):
        p.schedule_drafts({"s0": [-1, 0], "s1": [-1] * 20})
    assert p.alloc.num_used == used and (p._tab == table).all() and p._drafts is None
    plan = p.schedule_drafts({"s0": [-1, 0, 0, 2]})
    for kept, match in (({"s1": [0]}, "has no drafts"), ({"s0": [1]}, "not a path"), ({"s0": [0, 3]}, "not a path"),
                        ({"s0": [0, 2, 2]}, "not a path"), ({"s0": [0, 4]}, "not a path"), ({"s0": [-1]}, "not a path")):
        with pytest.raises(ValueError, match=match):
            p.keep_drafts(plan, kept)
    assert p.keep_drafts(plan, {"s0": [0, 2, 3]}).moves and p.context_len("s0") == 18


def test_inside_a_prompt_there_are_no_drafts():
    p = planner(prefill_chunk=16)
    p.add_request("a", 40)
    p.schedule()
    with pytest.raises(ValueError, match="inside its prompt"):
        p.schedule_drafts({"a": [-1]})


def test_a_sequence_that_ends_while_its_drafts_are_open():
    p = started([15, 30])
    plan = p.schedule_drafts({"s0": [-1, 0, 0], "s1": [-1, 0, 0]})
    p.finish("s0")
    kept = p.keep_drafts(plan, {"s0": [0, 2], "s1": [0, 2]})
    assert kept.keep.tolist() == [0, 2] and kept.cu_keep.tolist() == [0, 0, 2] and p.alloc.num_used == 2


def test_drafts_of_a_fork_stay_out_of_shared_blocks():
    p = started([32])
    assert p.fork("s0", "f").shape[0] == 0                     # both blocks are full: shared
    plan = p.schedule_drafts({"s0": [-1, 0, 0], "f": [-1, 0, 0]})          # (check_plans looks at the slots)
    assert p.alloc.num_used == 4
    p.keep_drafts(plan, {"s0": [0, 2]})
    assert p.alloc.num_used == 3 and p.context_len("f") == 32 and p.context_len("s0") == 34
    p.finish("s0")
    p.finish("f")
    assert p.alloc.num_used == 0


def test_random_runs_keep_the_tokens_in_their_places():
    """A cache on the host, written by slot, moved as the kept drafts say: every sequence reads its own text."""
    rng = np.random.default_rng(3)
    p = planner(num_blocks=64, max_seqs=4, block_size=8, max_num_batched_tokens=48, prefill_chunk=48)
    cache = np.full(64 * 8, -1, dtype=np.int64)
    text = {}
    for i in range(4):
        text[i] = rng.integers(0, 1000, int(rng.integers(1, 30))).tolist()
        p.add_request(i, len(text[i]))
    done = {i: 0 for i in text}
    def store(plan, toks):
        cache[plan.host_slot_mapping] = toks
    def check(plan):
        for r, sid in enumerate(plan.seq_ids):
            j = np.arange(p.context_len(sid))
            assert cache[plan.host_block_table[r][j // 8].astype(np.int64) * 8 + j % 8].tolist() == text[sid][:j.size]
    while (plan := p.schedule(decode=())) is not None:
        news = np.diff(plan.host_cu_q_lens)
        store(plan, [x for sid, n in zip(plan.seq_ids, news) for x in text[sid][p.context_len(sid) - n:p.context_len(sid)]])
    for _ in range(60):
        who = [i for i in text if rng.random() < 0.8 and len(text[i]) < 100]
        if not who:
            continue
        trees = {i: [-1] + [int(rng.integers(-1 if b > 3 else 0, b)) for b in range(1, int(rng.integers(1, 12)))] for i in who}
        guess = {i: rng.integers(0, 1000, len(trees[i])).tolist() for i in who}
        plan = p.schedule_drafts(trees)
        store(plan, [x for i in who for x in guess[i]])
        for r, i in enumerate(who):
            at = plan.host_positions[plan.host_cu_q_lens[r]:plan.host_cu_q_lens[r + 1]]
            depth = [0] * len(trees[i])
            for b, q in enumerate(trees[i]):
                depth[b] = 0 if q < 0 else depth[q] + 1
            assert (at == len(text[i]) + np.asarray(depth)).all()
        kept = {}
        for i in who:
            b = int(rng.integers(-1, len(trees[i])))
            path = []
            while b >= 0:
                path.insert(0, b)
                b = trees[i][b]
            kept[i] = path
        moved = p.keep_drafts(plan, kept)
        for r, i in enumerate(who):
            text[i] += [guess[i][b] for b in kept[i]]
            for to, b in enumerate(moved.keep[moved.cu_keep[r]:moved.cu_keep[r + 1]].tolist()):
                f, t = int(moved.first[r]) + b, int(moved.first[r]) + to
                tab = plan.host_block_table[r].astype(np.int64)
                cache[tab[t // 8] * 8 + t % 8] = cache[tab[f // 8] * 8 + f % 8]
        check(plan)
        assert p.alloc.num_used == sum(-(-len(t) // 8) for t in text.values())
    assert sum(map(len, text.values())) > 200


def test_accepted_drafts():
    # the text's next tokens are 7 (draft 0), then what the model picks: 5, 9, 4
    assert accept_drafts([7], [-1], [5]) == ([0], 5)
    assert accept_drafts([7, 6, 5, 9, 9], [-1, 0, 0, 1, 2], [5, 9, 9, 1, 4]) == ([0, 2, 4], 4)
    assert accept_drafts([7, 5, 5, 9], [-1, 0, 0, 2], [5, 8, 9, 4]) == ([0, 1], 8)            # the first of two alike
    assert accept_drafts(torch.tensor([7, 5]), [-1, 0], torch.tensor([5, 3])) == ([0, 1], 3)
    assert accept_drafts([7, 5], [-1, -1], [5, 3]) == ([0], 5)                               # (draft 1 follows the text, not draft 0)
    for args in (([], [], []), ([7], [0], [1]), ([7, 5], [-1], [1, 2]), ([7], [-1], [1, 2])):
        with pytest.raises(ValueError):
            accept_drafts(*args)
