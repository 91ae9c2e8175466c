"""Sessions that share pages and verify drafts, at their edges: drafts that another engine drew with the same seeds, compactions
that are refused, probabilities that do not fit their drafts, and NaN in queries and keys of the attention over shared prefixes
or in pages that nobody attends."""
import math

import numpy as np
import pytest
import torch

from mesh_b200 import ops
from mesh_b200.engine.serving import _verify_thresholds
from test_fork_verify_gpu import _check_greedy, _engine, _prompt, _start
from test_sharing_gpu import _attn_64, _check_attn, _gen, _i32, _run_shared, _shared_case, _verify_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _check_err():
    yield
    ops.scratch(torch.device("cuda", torch.cuda.current_device())).check("kernel")


def _draft(eng, prompts, counts, temps, seeds):
    """Tokens that a draft model's engine gives behind each prompt, and the probabilities they were drawn from."""
    eng.runner.keep_logits = True
    sids = [eng.submit(p, c, temperature=t, seed_base=z) for p, c, t, z in zip(prompts, counts, temps, seeds)]
    eng.prefill_step(token_budget=1 << 20)
    assert not eng.waiting
    rows = {i: [eng.runner.last_logits[i].clone()] for i in range(len(sids))}
    for k in range(1, max(counts)):
        at = {i: eng.sessions[sid].slot for i, sid in enumerate(sids) if counts[i] > k}
        eng.decode_step()
        for i, slot in at.items():
            rows[i].append(eng.runner.last_logits[slot].clone())
    eng.flush_history()
    return [eng.sessions[sid].generated for sid in sids], [torch.softmax(torch.stack(rows[i]) / t, -1) for i, t in enumerate(temps)]


def test_sampled_verification_is_the_rule_on_the_targets_logits():
    """Sessions with a draft model's tokens and probabilities, with guesses, and with none, in one step: what each keeps and
    draws is what the rejection rule gives for the logits of that step and the session's uniforms. The draft model has the
    target's weights, seeds and temperature, so nearly all of its tokens are accepted; one guess in many thousands is."""
    eng, cfg = _engine()
    draft, _ = _engine(graphs=False)
    V, n_new = cfg.vocab_size, 26
    prompts = [_prompt(cfg, n, seed=n) for n in (5, 33, 16, 47, 20)]
    temps, seeds = [1.0, 0.7, 1.3, 1.0, 1.0], [0, 0, 9, 9, 12345]
    sids = [eng.submit(p, n_new, temperature=t, seed_base=z) for p, t, z in zip(prompts, temps, seeds)]
    eng.prefill_step(token_budget=1 << 20)
    eng.flush_history()
    accepted = refused = 0
    for turn in range(n_new):
        act = [i for i, s in enumerate(sids) if eng.sessions[s].status == "decoding"]
        if not act:
            break
        state = {i: (list(eng.sessions[sids[i]].generated), eng.sessions[sids[i]].kv_len) for i in act}
        modelled = [i for i in act if (i + turn) % 4 < 2]
        drafts, probs = {sids[i]: [] for i in act}, {}
        if modelled:
            counts = [1 + (i + turn) % 5 for i in modelled]
            got, q = _draft(draft, [prompts[i] + state[i][0] for i in modelled], counts, [temps[i] for i in modelled],
                            [seeds[i] for i in modelled])
            for i, d, x in zip(modelled, got, q):
                drafts[sids[i]], probs[sids[i]] = d, x
        for i in act:
            if i not in modelled and (i + turn) % 4 == 2:
                drafts[sids[i]] = [(17 * turn + k) % V for k in range(1 + turn % 3)]
        new = eng.verify_step(drafts, probs)
        T = eng.runner.last_logits.shape[0] // len(act)
        logits = eng.runner.last_logits.view(len(act), T, V)
        for j, i in enumerate(act):
            d = drafts[sids[i]][:n_new - len(state[i][0]) - 1]
            n = len(d)
            acc, draw = _verify_thresholds(seeds[i], state[i][1], n)
            q = probs[sids[i]][None, :n] if sids[i] in probs and n else None
            tokens, a, _, near = _verify_plain(logits[j:j + 1, :n + 1], _i32([d]).view(1, n), torch.tensor([acc + [draw]], dtype=torch.float32),
                                               torch.tensor([1.0 / temps[i]], dtype=torch.float32), q, None)
            assert near > 1e-11  # no decision within the rounding of 64-bit sums
            assert new[sids[i]] == tokens[0][:a[0] + 1], (turn, i)
            assert eng.sessions[sids[i]].generated == state[i][0] + new[sids[i]]
            accepted += a[0]
            refused += n > a[0]
    assert accepted >= 20 and refused >= 10
    assert all(len(eng.sessions[s].generated) == n_new for s in sids) and eng.alloc.num_used == 0
    eng.close()
    draft.close()


@pytest.mark.parametrize("why", ["an earlier error", "a page of its own", "a second holder"])
def test_a_refused_compaction_moves_nothing(why):
    """The engine goes on with the tokens it gives without, and compacts once the reason is gone."""
    eng, cfg = _engine(pages=60)
    prompts, news = [_prompt(cfg, n, seed=n) for n in (50, 20, 33, 40, 9)], [6, 30, 4, 30, 30]

    def run(refuse):
        sids = _start(eng, prompts, 30)
        for sid, n in zip(sids, news):
            eng.sessions[sid].max_new_tokens = n
        for _ in range(8):  # the first and the third are through: holes
            eng.decode_step()
        if refuse:
            eng.flush_history()
            torch.cuda.synchronize()
            pages = {s.sid: list(s.pages) for s in eng.running if s}
            kept = eng.runner.kv.k.clone(), eng.runner.kv.v.clone()
            tables = eng.bt_host.copy()
            if why == "an earlier error":
                ops.scratch(eng.device).err.fill_(5)
            elif why == "a page of its own":
                extra = eng.alloc.alloc(eng.alloc.num_free)[-1:]  # the last one stays taken
                eng.alloc.free([p for p in range(1, 60) if eng.alloc.refs(p) and p not in extra + sum(pages.values(), [])])
            else:
                extra = eng.running[1].pages[:1]
                eng.alloc.share(extra)
            used = eng.alloc.num_used
            with pytest.raises(RuntimeError, match="bad argument" if why == "an earlier error" else "holders"):
                eng.compact()
            assert torch.equal(eng.runner.kv.k, kept[0]) and torch.equal(eng.runner.kv.v, kept[1])
            assert pages == {s.sid: s.pages for s in eng.running if s} and (eng.bt_host == tables).all() and eng.alloc.num_used == used
            for _ in range(3):
                eng.decode_step()
            if why != "an earlier error":
                eng.alloc.free(extra)
            live = eng.compact()
            assert live == 1 + eng.alloc.num_used and max(p for s in eng.running if s for p in s.pages) < live
        eng.run()
        return [eng.sessions[s].generated for s in sids]

    want = run(False)
    assert run(True) == want
    assert eng.alloc.num_used == 0
    eng.close()


def test_probabilities_that_do_not_fit_their_drafts_are_refused():
    """One row would be spread over all drafts. A refused step leaves the sessions as they were."""
    eng, cfg = _engine()
    V = cfg.vocab_size
    a, b = _start(eng, [_prompt(cfg, 12), _prompt(cfg, 20)], 30, temperature=1.0)
    eng.flush_history()
    before = [(list(eng.sessions[s].generated), eng.sessions[s].kv_len) for s in (a, b)]
    good = torch.full((3, V), 1.0 / V, device=DEV)
    for bad in (good[:1], good[:2], good[0], good[:, :V - 1], good[:, :1], good[None], good.long()):
        with pytest.raises(ValueError, match="probabilities"):
            eng.verify_step({b: [1], a: [1, 2, 3]}, {a: bad})
    assert before == [(eng.sessions[s].generated, eng.sessions[s].kv_len) for s in (a, b)]
    got = eng.verify_step({a: [1, 2, 3], b: [4]}, {a: good, b: None})
    assert all(1 <= len(g) <= 4 for g in got.values())
    assert eng.verify_step({a: [1], b: []}, {a: good.cpu()})[b]  # rows behind the drafts are not looked at
    eng.close()


@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (4, 2, 64), (8, 8, 128)])
@pytest.mark.parametrize("T", [1, 2])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("where", ["query", "shared key", "own key", "last key"])
def test_nan_makes_the_rows_that_meet_it_nan(hq, hkv, D, T, shared, where):
    """Whether their keys are one worker's, cut over several, or behind a prefix, and whatever an earlier call left in the
    workspace; the other rows keep their values."""
    groups = [([3, 0, 1], 300), ([4, 2], 1000)]
    own = [T + 5, T, 1500, 70, 2500, T + 1, 90, 3000, 0]
    q, kc, vc, table, lens = _shared_case(9, T, hq, hkv, D, 16, groups, own, seed=61)
    G, scale = hq // hkv, 1.0 / math.sqrt(D)
    clean, mag = _attn_64(q, kc, vc, table, lens, T, scale)
    plan = ops.PrefixGroups(9, hq, hkv, D, q_len=T).set(groups if shared else [])
    out = torch.empty_like(q)
    ops.attn_shared_prefix(q, kc, vc, table, lens, plan, out, scale)  # leaves finite partials behind
    _check_attn(out, clean, mag)
    hit = torch.zeros(9, T, hq, dtype=torch.bool)
    pos = lens.cpu()[:, None] - T + torch.arange(T)
    if where == "query":
        for b, t, h in ((0, 0, 1), (2, T - 1, hq - 1), (5, 0, 0), (7, T - 1, 2), (8, 0, 0)):
            q.view(9, T, hq, D)[b, t, h] = math.nan
            hit[b, t, h] = pos[b, t] >= 0  # the empty slot has no key, so it stays zero
    else:
        h = hkv - 1
        spots = {"shared key": [(3, 131), (4, 990)], "own key": [(2, 1700), (3, 310), (7, 40), (6, 33)],
                 "last key": [(b, int(lens[b]) - 1) for b in (0, 2, 5, 7)]}[where]
        for b, key in spots:
            kc[table[b, key // 16].long(), h, key % 16, 3] = math.nan
            members = next((g for g, n in groups if b in g and key < n), [b])
            for m in members:
                for t in range(T):
                    if pos[m, t] >= key:
                        hit[m, t, h * G:(h + 1) * G] = True
    assert hit.any() and not hit.all()
    for _ in range(2):
        ops.attn_shared_prefix(q, kc, vc, table, lens, plan, out, scale)
        bad = out.view(9 * T, hq, D).isnan()
        assert torch.equal(bad.all(-1).cpu().view(9, T, hq), hit) and torch.equal(bad.any(-1), bad.all(-1))
        keep = ~bad.view(9 * T, hq * D)
        _check_attn(torch.where(keep, out, 0), torch.where(keep, clean, 0), mag)


@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (4, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("window", [0, 45])
@pytest.mark.parametrize("prefix", [1, 15, 31, 200, 333])
def test_what_nobody_attends_may_hold_anything(hq, hkv, D, T, window, prefix):
    """The members' own copies of a prefix that ends inside a page (it is read through the first sequence), the keys that every
    row's window has left behind, and the tails of pages hold NaN and infinity."""
    groups = [([2, 0, 4, 1], prefix)]
    own = [T + 60, T, T + 7, 900, T + 200, 77, T + 1]
    q, kc, vc, table, lens = _shared_case(7, T, hq, hkv, D, 16, groups, own, seed=71, junk=True)
    want, mag = _attn_64(q, kc, vc, table, lens, T, 1.0 / math.sqrt(D), window)
    full = prefix // 16
    for b in (0, 4, 1):
        page = int(table[b, full])
        kc[page, :, :prefix % 16] = math.nan
        vc[page, :, :prefix % 16] = math.inf
        table[b, :full] = 0  # as if they had never been told of the shared pages
    kc[0], vc[0] = math.nan, math.inf
    if window:
        for b in (3, 5):
            for key in range(max(0, int(lens[b]) - T + 1 - window)):
                page = int(table[b, key // 16])
                kc[page, :, key % 16], vc[page, :, key % 16] = math.nan, -math.inf
    plan = ops.PrefixGroups(7, hq, hkv, D, q_len=T).set(groups)
    out = torch.full_like(q, math.nan)
    ops.attn_shared_prefix(q, kc, vc, table, lens, plan, out, 1.0 / math.sqrt(D), window=window)
    _check_attn(out, want, mag)


@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 40])
def test_a_window_beyond_every_key_is_none(window):
    groups = [([1, 2], 100)]
    case = _shared_case(5, 8, 8, 2, 64, 16, groups, [5, 8, 30, 40, 0], seed=81)
    plain, _ = _run_shared(case, 8, 8, 2, 64, groups)
    out, _ = _run_shared(case, 8, 8, 2, 64, groups, window=window)
    assert torch.equal(out, plain)
    _check_attn(out, *_attn_64(*case, 8, 1.0 / math.sqrt(64)))


@pytest.mark.parametrize("kind", [list, tuple, np.array, torch.tensor])
def test_page_lists_of_any_kind(kind):
    """Counts beside a list of pages may be an array or a tensor, with zeros among them."""
    pool = torch.randn(2, 9, 2, 16, 64, device=DEV, generator=_gen(91)).to(torch.bfloat16)
    k, v = pool.clone(), -pool
    for src, dst, tokens in (([1, 1, 2], [3, 4, 5], [0, 7, 16]), ([1], [6], [0]), ([8], [7], [1])):
        want = k.clone()
        for a, b, t in zip(src, dst, tokens):
            want[:, b, :, :t] = k[:, a, :, :t]
        ops.kv_pages_copy(k, v, src, dst, kind(tokens))
        assert torch.equal(k, want) and torch.equal(v, -want)


@pytest.mark.parametrize("graphs", [True, False])
def test_two_families_and_an_early_branch_decode_together(graphs, monkeypatch):
    """Sessions of two prompts, forked at several lengths: groups of different prefixes in one step, which change as branches fork
    and finish. Every token is the greedy one after those before it."""
    from mesh_b200.engine import serving
    monkeypatch.setattr(serving, "SHARED_PREFIX_MIN_BYTES", 0)
    eng, cfg = _engine(pages=120, max_batch=16, graphs=graphs)
    ref, _ = _engine(pages=200, graphs=False, max_tokens=2048)
    prompts = [_prompt(cfg, 20, seed=1), _prompt(cfg, 70, seed=2), _prompt(cfg, 33, seed=3)]
    a, b, alone = _start(eng, prompts, 60)
    early = eng.fork_session(a, 1)                    # one page in common with what follows
    for _ in range(30):
        eng.decode_step()
    kids = eng.fork_session(a, 3) + eng.fork_session(b, 2)
    eng.decode_step()
    groups = sorted((len(s), n) for s, n in eng._prefix_groups([s for s in eng.running if s]))
    assert groups == [(3, 96), (4, 48)]
    eng.sessions[kids[0]].max_new_tokens = 36         # one leaves while the others go on
    for _ in range(8):
        eng.decode_step()
    more = eng.fork_session(kids[3], 1)
    eng.compact()
    eng.run()
    done = {a: 0, b: 1, alone: 2, early[0]: 0, **{k: 0 for k in kids[:3]}, **{k: 1 for k in kids[3:] + more}}
    assert all(len(eng.sessions[s].generated) == (36 if s == kids[0] else 60) for s in done)
    _check_greedy(ref, [(prompts[i], eng.sessions[s].generated) for s, i in done.items()])
    assert eng.alloc.num_used == 0
    eng.close()
    ref.close()
