"""Sessions forked from one another, pools compacted between steps and drafted tokens verified, in the serving engine.

Page placement does not enter the arithmetic, so compaction is compared bitwise. Forked and verifying sessions run on other
kernels, batch shapes and splits than a session alone, whose logits differ by bf16 rounding (about 1 % of their root mean
square; tests/test_model_gpu.py allows 3 % between decode and prefill), and random weights give near ties. So every
greedy token is held against a prefill of the tokens before it: its logit may be below the largest by what two
logits 3 % off each can make, taken five times to cover the largest of thousands (0.3 of the root mean square, where
the largest of 4096 lies about 3.5 above the mean).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _engine(preset="small", pages=96, max_batch=8, graphs=True, seed=7, max_tokens=512):
    from mesh_b200.config import EngineConfig, get_preset
    from mesh_b200.engine.serving import Engine
    from mesh_b200.models.llama import KVPool, LlamaRunner
    from mesh_b200.models.weights import synthetic_device_weights
    cfg = get_preset(preset)
    ecfg = EngineConfig(max_seq_len=256, use_cuda_graphs=graphs)
    w = synthetic_device_weights(cfg, 0, 1, seed=seed, device=DEV)
    kv = KVPool(cfg, w.layout.local_kv_heads, pages, 16, DEV)
    return Engine(LlamaRunner(w, ecfg, kv, DEV, max_tokens=max_tokens), ecfg, max_batch=max_batch), cfg


def _prompt(cfg, n, seed=21):
    return torch.randint(0, cfg.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _start(eng, prompts, n_new, **kw):
    sids = [eng.submit(p, n_new, **kw) for p in prompts]
    while eng.waiting:
        eng.prefill_step()
    return sids


def _check_greedy(ref, sequences):
    """sequences: (prompt, generated). Every generated token is the greedy one after those before it."""
    todo = [(p + g[:k], g[k]) for p, g in sequences for k in range(len(g))]
    ref.runner.keep_logits = True
    for i in range(0, len(todo), 8):
        part = todo[i:i + 8]
        for tokens, _ in part:
            ref.submit(tokens, 1)
        ref.prefill_step(token_budget=1 << 20)
        assert not ref.waiting
        logits = ref.runner.last_logits
        picked = logits.gather(1, torch.tensor([[t] for _, t in part], device=DEV))[:, 0]
        rms = logits.pow(2).mean(1).sqrt()
        assert (picked >= logits.amax(1) - 0.3 * rms).all(), (i, ((logits.amax(1) - picked) / rms).tolist())
    ref.flush_history()


@pytest.fixture(scope="module")
def ref():
    eng, _ = _engine(pages=200, graphs=False, max_tokens=2048)
    yield eng
    eng.close()


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("length", [32, 41, 7, 16, 100])
def test_forks_continue_like_their_parent(length, shared, monkeypatch, ref):
    from mesh_b200.engine import serving
    monkeypatch.setattr(serving, "SHARED_PREFIX_MIN_BYTES", 0 if shared else 1 << 60)
    eng, cfg = _engine()
    (a,) = _start(eng, [_prompt(cfg, length)], 20)
    for _ in range(3):
        eng.decode_step()
    used = eng.alloc.num_used
    kids = eng.fork_session(a, 3)
    tail = eng.sessions[a].kv_len % 16
    assert eng.alloc.num_used == used + (3 if tail else 0)  # full pages are shared, not copied
    grand = eng.fork_session(kids[1], 1)
    eng.run()
    gen = [eng.sessions[sid].generated for sid in [a] + kids + grand]
    assert all(len(g) == 20 and g[:4] == gen[0][:4] for g in gen)
    if not shared:
        assert all(g == gen[0] for g in gen)  # the same kernel on equal rows
    _check_greedy(ref, [(_prompt(cfg, length), g) for g in gen[::2]])
    assert eng.alloc.num_used == 0
    assert any(len(k) == 3 for k in eng.dec.graphs if isinstance(k, tuple)) == (shared and length > 16 - 3)
    eng.close()


def test_sampled_forks_part_and_leave_each_other_alone():
    eng, cfg = _engine()
    (a,) = _start(eng, [_prompt(cfg, 30)], 24, temperature=1.0, seed_base=5)
    eng.decode_step()
    kids = eng.fork_session(a, 3, seeds=[5, 6, 7])
    eng.run()
    gen = {sid: eng.sessions[sid].generated for sid in [a] + kids}
    assert gen[kids[0]] == gen[a]  # the parent's seed repeats it
    assert gen[kids[1]] != gen[a] and gen[kids[1]] != gen[kids[2]]
    assert all(g[:2] == gen[a][:2] and len(g) == 24 for g in gen.values())
    eng.close()


def test_fork_refusals():
    eng, cfg = _engine(max_batch=2, pages=6)
    sid = eng.submit(_prompt(cfg, 20), 8)
    with pytest.raises(ValueError):
        eng.fork_session(sid)
    eng.prefill_step()
    with pytest.raises(ValueError):
        eng.fork_session(sid, 0)
    with pytest.raises(ValueError):
        eng.fork_session(sid, 1, seeds=[1, 2])
    with pytest.raises(RuntimeError):
        eng.fork_session(sid, 2)
    held = eng.alloc.alloc(eng.alloc.num_free)
    with pytest.raises(RuntimeError):
        eng.fork_session(sid, 1)
    eng.alloc.free(held)
    assert eng.fork_session(sid, 1)
    eng.close()


def test_compaction_between_steps_changes_no_token():
    eng, cfg = _engine(pages=60)
    prompts = [_prompt(cfg, n, seed=n) for n in (50, 20, 33, 40, 9)]
    news = [6, 30, 4, 30, 30]

    def run(compact):
        sids = [eng.submit(p, n) for p, n in zip(prompts, news)]
        while eng.waiting:
            eng.prefill_step()
        step = 0
        while eng.has_work():
            eng.decode_step()
            step += 1
            if compact and step in (5, 7, 20):
                live = eng.compact()
                assert live == 1 + eng.alloc.num_used
                assert max(p for s in eng.running if s for p in s.pages) < live
                assert eng.alloc.refs(live) == 0
        eng.flush_history()
        return [eng.sessions[s].generated for s in sids]

    want = run(False)
    assert run(True) == want
    assert eng.alloc.num_used == 0
    eng.close()


@pytest.mark.parametrize("preset", ["small", "tiny"])
def test_verified_drafts_are_what_greedy_decoding_gives(preset):
    eng, cfg = _engine(preset)
    ref, _ = _engine(preset, pages=200, graphs=False, max_tokens=2048)
    prompts = [_prompt(cfg, n, seed=n) for n in (1, 25, 47, 30)]
    guess = eng.generate(prompts, 25)
    sids = _start(eng, prompts, 25)
    eng.flush_history()
    turn = accepted = refused = 0
    while any(eng.sessions[s].status == "decoding" for s in sids):
        act = [s for s in sids if eng.sessions[s].status == "decoding"]
        drafts, before = {}, {}
        for s in act:
            i = sids.index(s)
            before[s] = list(eng.sessions[s].generated)
            d = guess[i][len(before[s]):][:(turn + i) % 6]  # none to five drafts, right as far as the runs agree
            if len(d) > 2 and turn % 2:                     # the third is wrong
                d = d[:2] + [(d[2] + 1) % cfg.vocab_size] + d[3:]
            drafts[s] = d
        got = eng.verify_step(drafts)
        best = eng.runner.last_logits.view(len(act), -1, cfg.vocab_size).argmax(-1).tolist()
        for i, s in enumerate(act):
            n = len(drafts[s][:24 - len(before[s])])
            a = 0
            while a < n and drafts[s][a] == best[i][a]:
                a += 1
            assert got[s] == drafts[s][:a] + [best[i][a]] and eng.sessions[s].generated == before[s] + got[s]
            accepted += a
            refused += n - a
        turn += 1
        if turn == 2:
            eng.decode_step()               # ordinary steps mix with verified ones
            eng.flush_history()
    assert accepted > 10 and refused > 5
    assert all(len(eng.sessions[s].generated) == 25 for s in sids) and eng.alloc.num_used == 0
    _check_greedy(ref, [(p, eng.sessions[s].generated) for p, s in zip(prompts, sids)])
    eng.close()
    ref.close()


def test_verified_sampled_drafts_follow_the_seed():
    """A draft model that proposes the target's own distribution: tokens are drawn, repeatably, and most are accepted."""
    eng, cfg = _engine()
    V = cfg.vocab_size

    def run():
        (a,) = _start(eng, [_prompt(cfg, 12)], 30, temperature=1.0, seed_base=11)
        eng.flush_history()
        g = torch.Generator(device=DEV).manual_seed(3)
        steps = 0
        while eng.sessions[a].status == "decoding":
            q = torch.full((4, V), 1.0 / V, device=DEV)
            d = torch.multinomial(q, 1, generator=g)[:, 0].tolist()
            eng.verify_step({a: d}, {a: q})
            steps += 1
        return eng.sessions[a].generated, steps

    first, steps = run()
    again, _ = run()
    assert first == again and len(first) == 30 and steps <= 29
    eng.close()


@pytest.mark.parametrize("tokens", [257, 320, 511])
def test_product_reads_what_the_kernel_before_it_wrote(tokens):
    """Between 257 and 511 rows (a verified batch, a short prefill) a product takes its rows as the first operand; it must
    not fetch them before the kernel that writes them has finished."""
    from mesh_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(tokens, 1024, device=DEV, generator=g).to(torch.bfloat16)
    w = (torch.randn(1536, 1024, device=DEV, generator=g) * 0.05).to(torch.bfloat16)
    one = torch.ones(1024, dtype=torch.bfloat16, device=DEV)
    normed, out = torch.empty_like(x), torch.empty(tokens, 1536, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    ops.add_rmsnorm(x, one, normed, 1e-5)
    torch.cuda.synchronize()
    want = normed.float() @ w.float().T
    for _ in range(30):
        normed.fill_(float("nan"))
        ops.add_rmsnorm(x, one, normed, 1e-5)
        ops.linear(normed, w, out=out)
        # fp32 sums, rounded once to bf16 (2^-8), against fp32 sums in another order (1024 terms, far below it)
        assert torch.allclose(out.float(), want, rtol=2 ** -7, atol=2 ** -8)


def test_verify_refusals():
    eng, cfg = _engine(max_batch=4)
    waiting = eng.submit(_prompt(cfg, 9), 8)
    with pytest.raises(ValueError):
        eng.verify_step({waiting: [1]})
    eng.prefill_step()
    with pytest.raises(ValueError):
        eng.verify_step({waiting: [cfg.vocab_size]})
    (nucleus,) = _start(eng, [_prompt(cfg, 9)], 8, temperature=0.7, top_p=0.9)
    with pytest.raises(ValueError):
        eng.verify_step({nucleus: [1]})
    (long,) = _start(eng, [_prompt(cfg, 9)], 60)
    with pytest.raises(ValueError):
        eng.verify_step({long: list(range(40))})
    assert eng.verify_step({}) == {}
    assert len(eng.sessions[long].generated) <= 1
    assert eng.verify_step({long: []})[long]  # no drafts: one token, as a decode step
    eng.close()


@pytest.mark.parametrize("graphs", [True, False])
def test_forks_drafts_and_compaction_together(graphs, monkeypatch, ref):
    """A search as a server would run it: one long prompt forked, its branches decoded over the shared pages, drafts verified,
    branches dropped, the pool compacted, one branch forked again, and the rest finished beside another session."""
    from mesh_b200.engine import serving
    monkeypatch.setattr(serving, "SHARED_PREFIX_MIN_BYTES", 0)
    eng, cfg = _engine(pages=80, graphs=graphs)
    prompt, other = _prompt(cfg, 90), _prompt(cfg, 25, seed=3)
    a, b = _start(eng, [prompt, other], 30)
    eng.decode_step()
    kids = eng.fork_session(a, 3)
    for _ in range(4):
        eng.decode_step()
    eng.flush_history()
    wrong = [0, 1]
    got = eng.verify_step({a: wrong, kids[0]: wrong[:1], kids[1]: [], b: wrong[1:]})
    assert all(len(g) >= 1 for g in got.values()) and len(got[kids[1]]) == 1
    first = got[kids[1]][0]  # what the shared history goes on with
    got = eng.verify_step({kids[2]: [first]})
    assert got[kids[2]][0] == first or len(got[kids[2]]) == 1
    for s in (a, kids[2]):  # two branches are dropped, the parent among them
        eng._free_session(eng.sessions[s])
        eng.sessions[s].status = "finished"
    live = eng.compact()
    assert live == 1 + eng.alloc.num_used
    more = eng.fork_session(kids[0], 2)
    assert eng.alloc.refs(eng.sessions[kids[0]].pages[0]) == 4
    eng.run()
    done = [kids[0], kids[1]] + more
    assert all(len(eng.sessions[s].generated) == 30 for s in done + [b])
    _check_greedy(ref, [(prompt, eng.sessions[s].generated) for s in done] + [(other, eng.sessions[b].generated)])
    assert eng.alloc.num_used == 0
    eng.close()
