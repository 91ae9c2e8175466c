"""Host rules of sessions that share pages and verify drafts (CPU): the uniforms of a verified step, arguments that are
refused, which sessions read their prefixes together."""
import random
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from mesh_b200 import ops
from mesh_b200.engine import serving
from mesh_b200.oracle.tensor_ops import deterministic_sample_threshold


def _draw(weights, u):
    c = np.cumsum(weights)
    return int(np.nonzero(c > u * c[-1])[0][0])


@pytest.mark.parametrize("kv_len", [0, 11, 4096])
@pytest.mark.parametrize("drafted_by", ["prefill or decode", "a verified step"])
def test_verified_tokens_follow_the_target_when_drafts_have_the_sessions_seed(kv_len, drafted_by):
    """One draft over three tokens, drawn with the number this framework's own sampler uses at that position for the same
    seed; accepting and drawing as the verification does. Over 60000 seeds each frequency's standard deviation is
    sqrt(1/3 2/3 / 60000) = 0.0019; five of them bound every token."""
    n = 60000
    p, q = np.full(3, 1 / 3), np.array([0.8, 0.1, 0.1])
    count = np.zeros(3)
    for seed in range(n):
        if drafted_by == "prefill or decode":
            u = deterministic_sample_threshold(seed ^ (kv_len + 1))
        else:  # a step without drafts in the draft model's engine
            u = serving._verify_thresholds(seed, kv_len, 0)[1]
        x = _draw(q, u)
        (accept,), draw = serving._verify_thresholds(seed, kv_len, 1)
        count[x if accept * q[x] < p[x] else _draw(np.maximum(p - q, 0), draw)] += 1
    assert np.abs(count / n - p).max() <= 5 * np.sqrt(1 / 3 * 2 / 3 / n), count / n


def test_thresholds_of_a_session_are_all_different():
    """Every uniform that one seed gives: those of ordinary steps, of accepting, and of drawing behind drafts."""
    seen = set()
    for kv_len in range(300):
        accept, draw = serving._verify_thresholds(77, kv_len, 1)
        seen |= {serving._verify_thresholds(77, kv_len, 0)[1], accept[0], draw}
    assert len(seen) >= 898  # 24-bit numbers: 900 of them coincide 0.02 times on average
    # a draft's own number does not depend on how many stand before it
    assert serving._verify_thresholds(77, 40, 5)[0][3] == serving._verify_thresholds(77, 43, 1)[0][0]
    # without drafts the token is decode_step's
    assert serving._verify_thresholds(77, 40, 0) == ([], deterministic_sample_threshold(77 ^ 41))


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf"), 1e-40])
def test_attention_over_shared_prefixes_refuses_a_scale_that_is_not_positive(scale):
    plan = ops.PrefixGroups(2, 4, 2, 64, device="cpu")
    q, cache = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.ones(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="scale"):
        ops.attn_shared_prefix(q, cache, cache, table, lens, plan, torch.empty_like(q), scale)


# ------------------------------------------------------------------------------------ which sessions share
def _forest(r, sessions, roots, step):
    """Page lists as forks leave them: a child has the full pages of its parent at that moment, both go on with new ones."""
    page = iter(range(1, 1 << 30))
    paths = [[next(page) for _ in range(r.randint(0, step))] for _ in range(roots)]
    while len(paths) < sessions:
        for p in paths:
            if r.random() < 0.5:
                p.extend(next(page) for _ in range(r.randint(0, step)))
        paths.append(list(r.choice(paths)))
    for p in paths:
        p.extend(next(page) for _ in range(r.randint(0, 2)))
    r.shuffle(paths)
    return paths


def _common(paths):
    return next((i for i, x in enumerate(zip(*paths)) if len(set(x)) > 1), min(len(p) for p in paths))


def _partitions(items):
    if not items:
        yield []
        return
    for rest in _partitions(items[1:]):
        yield [[items[0]]] + rest
        for i in range(len(rest)):
            yield rest[:i] + [[items[0]] + rest[i]] + rest[i + 1:]


@pytest.mark.parametrize("seed", range(120))
def test_prefix_groups_save_the_most(seed):
    """Against every partition of up to seven sequences."""
    r = random.Random(seed)
    paths = _forest(r, r.randint(1, 7), r.randint(1, 2), r.choice((1, 3, 9)))
    best = max(sum((len(b) - 1) * _common([paths[i] for i in b]) for b in part) for part in _partitions(list(range(len(paths)))))
    got = serving._shared_prefixes(paths)
    flat = [i for m, _ in got for i in m]
    assert len(flat) == len(set(flat)) and all(len(m) > 1 and 0 < n <= _common([paths[i] for i in m]) for m, n in got)
    assert sum((len(m) - 1) * n for m, n in got) == best


def test_prefix_groups_of_a_long_chain_of_forks():
    """Every session forked from the one before, a page later: deeper than the interpreter's stack."""
    paths = [list(range(1, i + 2)) + [10 ** 6 + i] for i in range(1500)]
    got = serving._shared_prefixes(paths)
    # halves above halves: groups of the deeper sequences leave the rest to a group further up
    assert sum((len(m) - 1) * n for m, n in got) >= 1499 * 1500 // 4
    assert all(paths[i][:n] == paths[m[0]][:n] for m, n in got for i in m)


def _engine_of(sessions, window=0, hkv=8, D=128, ps=16):
    eng = SimpleNamespace(runner=SimpleNamespace(hq=4 * hkv, hkv=hkv, D=D, window=window), page_size=ps, max_batch=128, _prefixes={})
    return lambda **kw: serving.Engine._prefix_groups(eng, sessions, **kw)


def _session(sid, pages, kv_len, forked=True):
    return serving.Session(sid, [1], 10, pages=pages, kv_len=kv_len, slot=sid, status="decoding", forked=forked)


def test_an_early_branch_leaves_the_others_together():
    """64 sessions share 8192 keys, one more parted from them after two pages."""
    shared = list(range(1, 513))
    many = [_session(i, shared + [1000 + i], 8192 + 5) for i in range(64)]
    early = _session(64, shared[:2] + [2000, 2001], 50)
    alone = _session(65, [3000, 3001], 20, forked=False)
    for order in (many + [early, alone], [early] + many, [alone, early] + many[::-1]):
        ((slots, keys),) = _engine_of(order)()
        assert sorted(slots) == list(range(64)) and keys == 8192
    # two that share too little by themselves still count where there is no least saving
    other = [_session(70 + i, [4000, 4001 + i], 20) for i in range(2)]
    assert sorted((len(s), k) for s, k in _engine_of(many + other)(min_bytes=0)) == [(2, 16), (64, 8192)]
    assert _engine_of(other)() == [] and _engine_of([early, alone])(min_bytes=0) == []


def test_a_window_counts_only_what_it_covers():
    """Ordinary decoding reads the keys inside the window alone, a shared prefix is read whole."""
    shared = list(range(1, 513))
    many = [_session(i, shared + [1000 + i], 8192 + 5) for i in range(16)]
    assert len(_engine_of(many)()) == 1
    assert len(_engine_of(many, window=8192)()) == 1
    assert _engine_of(many, window=512)(min_bytes=0) == []       # 16 x 506 keys against 8192
    assert len(_engine_of(many, window=1024)(min_bytes=0)) == 1  # 16 x 1018
    assert _engine_of(many, window=4)(min_bytes=0) == []


@pytest.mark.parametrize("seed", range(12))
def test_groups_that_stand_are_those_of_a_fresh_look(seed):
    """Decoding, forks, departures and compactions in any order, with the allocator's own pages."""
    from mesh_b200.engine.pages import _PyPageAllocator
    r, ps = random.Random(seed), 16
    alloc = _PyPageAllocator(600, 1)
    live = []
    eng = SimpleNamespace(runner=SimpleNamespace(hq=32, hkv=8, D=128, window=0), page_size=ps, max_batch=128, _prefixes={})

    def grow(s, n):
        s.kv_len += n
        while len(s.pages) * ps < s.kv_len:
            s.pages += alloc.alloc(1)

    for sid in range(2):
        live.append(_session(sid, [], 0, forked=False))
        grow(live[-1], r.randint(20, 120))
    sid = 2
    for _ in range(120):
        for s in live:
            grow(s, 1)
        op = r.random()
        if op < 0.15 and len(live) < 9:
            a = r.choice(live)
            full = a.kv_len // ps
            alloc.share(a.pages[:full])
            a.forked = True
            live.append(_session(sid, a.pages[:full] + (alloc.alloc(1) if a.kv_len % ps else []), a.kv_len))
            sid += 1
        elif op < 0.22 and len(live) > 2:
            alloc.free(live.pop(r.randrange(len(live))).pages)
        elif op < 0.3:
            used = sorted({p for s in live for p in s.pages})
            n = 1 + len(used)
            remap = [-1] * 600
            for p in used:
                remap[p] = p if p < n else remap[p]
            for p, q in zip([p for p in used if p >= n], [q for q in range(1, n) if q not in used]):
                remap[p] = q
            alloc.remap(remap)
            for s in live:
                s.pages = [remap[p] for p in s.pages]
        act = [s for s in live if r.random() < 0.9]
        got = serving.Engine._prefix_groups(eng, act, min_bytes=0)
        assert got == serving.Engine._prefix_groups(SimpleNamespace(**{**vars(eng), "_prefixes": {}}), act, min_bytes=0)
        for slots, keys in got:
            by = {s.slot: s for s in act}
            assert all(by[x].pages[:keys // ps] == by[slots[0]].pages[:keys // ps] and keys <= by[x].kv_len for x in slots)


def test_groups_are_worked_out_once_for_a_set_of_sessions(monkeypatch):
    looks, real = [], serving._shared_prefixes
    monkeypatch.setattr(serving, "_shared_prefixes", lambda paths: looks.append(len(paths)) or real(paths))
    sessions = [_session(i, list(range(1, 41)) + [100 + i], 645) for i in range(4)]
    groups = _engine_of(sessions)
    for step in range(20):
        assert groups(min_bytes=0) == [([0, 1, 2, 3], 640)]
        for s in sessions:
            s.kv_len += 1
            if s.kv_len > 16 * len(s.pages):
                s.pages.append(200 + 4 * step + s.sid)
    sessions.append(_session(4, sessions[0].pages[:41] + [900], 660))
    assert groups(min_bytes=0) == [([0, 1, 2, 3, 4], 640)]
    del sessions[1]
    assert groups(min_bytes=0) == [([0, 2, 3, 4], 640)] and looks == [4, 5, 4]


def test_prefixes_are_shared_where_that_is_faster():
    """The measured sides of the threshold, 8 KV heads of 128."""
    for n, keys, shared in ((2, 4096, False), (8, 1024, False), (4, 4096, True), (8, 2048, True), (16, 4096, True)):
        pages = list(range(1, keys // 16 + 1))
        sessions = [_session(i, pages + [9000 + i], keys + 7) for i in range(n)]
        assert bool(_engine_of(sessions)()) == shared, (n, keys)
