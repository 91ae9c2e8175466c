"""Measured cases of the serving operators around sessions that fork one another and propose tokens ahead:

* ``attention``  paged decode attention of a batch in which groups of sessions share a long prefix (``ops.attn_shared_prefix``);
* ``copy``       pages of the KV pool copied inside it, whole or only their first tokens, as a fork does (``ops.kv_pages_copy``);
* ``compact``    live pages moved to the front of the pool and the block tables rewritten (``ops.kv_pages_compact``);
* ``verify``     drafted tokens accepted or replaced against the target's probabilities (``ops.verify_drafts``).

``run`` computes the plain form from elementary torch operations where ``own`` is false, and calls the framework where it is true.
Head layouts, layer counts and vocabularies are those of the model presets (8B: 32/8 heads of 128, 32 layers, 128256 tokens; a rank of the
70B split eight ways: 8/1 heads; 1.1B: 32/4 heads of 64, 22 layers, 32000 tokens) and pages hold 16 tokens, the engine's default.
"""
import math

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # four answers to one short prompt, a few tokens in: the smallest step, bound by latency
        dict(name="attention forks of 4", op="attention", batch=4, groups=1, alone=0, prefix=512, most=40, tokens=1, hq=32, hkv=8, dim=128, page=16),
        # a full decode batch behind one system prompt of 8k tokens
        dict(name="attention 64 behind 8k", op="attention", batch=64, groups=1, alone=0, prefix=8192, most=512, tokens=1, hq=32, hkv=8, dim=128, page=16),
        # several prompts at once, some sessions without any; odd counts, prefixes that end inside a page
        dict(name="attention ragged groups", op="attention", batch=61, groups=5, alone=7, prefix=2011, most=777, tokens=1, hq=32, hkv=4, dim=64, page=16),
        # the target's pass over four drafted tokens and the last one of each session, on one rank of eight
        dict(name="attention drafts of 4", op="attention", batch=32, groups=2, alone=0, prefix=4096, most=300, tokens=5, hq=8, hkv=1, dim=128, page=16),
        # the largest: 128 sessions behind a document of 16k tokens
        dict(name="attention 128 behind 16k", op="attention", batch=128, groups=1, alone=0, prefix=16384, most=1024, tokens=1, hq=32, hkv=8, dim=128, page=16),
        # a session forked into three: the tokens of its last, half-filled page
        dict(name="copy a fork of 3", op="copy", heads=8, dim=128, layers=32, page=16, pages=64, pairs=3, tokens=9),
        # whole pages of a long session (duplicated before a branch rewrites it)
        dict(name="copy 200 pages", op="copy", heads=8, dim=128, layers=32, page=16, pages=600, pairs=200, tokens=16),
        # a small pool with few holes, and a large one after most sessions have gone
        dict(name="compact 1.1B pool", op="compact", heads=4, dim=64, layers=22, page=16, pages=512, seqs=11, per=13, shared=5, moves=40),
        dict(name="compact 8B pool", op="compact", heads=8, dim=128, layers=32, page=16, pages=900, seqs=24, per=14, shared=32, moves=210),
        # one session, four drafts
        dict(name="verify 1 session", op="verify", batch=1, drafts=4, vocab=128256, probs=True, greedy=0, half=False),
        # no draft model (tokens guessed from the prompt), a third of the sessions greedy, half-width logits, ragged draft counts
        dict(name="verify guesses", op="verify", batch=33, drafts=7, vocab=32000, probs=False, greedy=3, half=True),
        # a full batch with the draft model's probabilities
        dict(name="verify 64 sessions", op="verify", batch=64, drafts=4, vocab=128256, probs=True, greedy=0, half=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "copy", "compact", "verify"))
    if op == "attention":
        hq, hkv, dim = rng.choice(((32, 8, 128), (8, 1, 128), (32, 4, 64), (4, 1, 128), (16, 4, 128), (8, 8, 64)))
        tokens = rng.choice((1, 1, 1, 2, 3, 5, 8))
        batch = _log(rng, 1, 128)
        groups = min(rng.choice((1, 1, 2, 3, 7)), batch)
        alone = rng.randint(0, max(0, min(9, batch - groups)))
        most = max(tokens, _log(rng, 8, 1024))
        # at most the largest listed case's keys and products
        room = min(128 * 16384 * 8 * 128 // (batch * hkv * dim), 128 * 16384 * 32 * 128 // (batch * hq * dim * tokens))
        prefix = min(_log(rng, 16, 16384), room)
        return dict(op=op, batch=batch, groups=groups, alone=alone, prefix=prefix, most=most, tokens=tokens, hq=hq, hkv=hkv, dim=dim, page=rng.choice((16, 16, 32)))
    if op == "copy":
        heads, dim, layers = rng.choice(((8, 128, 32), (1, 128, 80), (4, 64, 22)))
        pages = rng.randint(100, 600)
        return dict(op=op, heads=heads, dim=dim, layers=layers, page=16, pages=pages, pairs=_log(rng, 1, pages // 3), tokens=rng.choice((16, rng.randint(1, 16))))
    if op == "compact":
        heads, dim, layers = rng.choice(((8, 128, 32), (1, 128, 80), (4, 64, 22)))
        pages, seqs, shared = rng.randint(200, 900), rng.randint(1, 40), rng.randint(0, 32)
        per = rng.randint(1, max(1, min(14, (pages // 2 - 33) // seqs)))
        live = 1 + shared + seqs * per
        return dict(op=op, heads=heads, dim=dim, layers=layers, page=16, pages=pages, seqs=seqs, per=per, shared=shared, moves=rng.randint(0, min(live - 1, pages - live, 210)))
    vocab = rng.choice((32000, 128256, 4096, rng.randint(1000, 128256)))
    drafts = rng.randint(1, 8)
    batch = min(_log(rng, 1, 64), 64 * 5 * 128256 // ((drafts + 1) * vocab))
    return dict(op=op, batch=batch, drafts=drafts, vocab=vocab, probs=rng.random() < 0.6, greedy=rng.choice((0, 0, 2, 3)), half=rng.random() < 0.4)


# ------------------------------------------------------------------------------------------------ what a user's program has in hand
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    return {"attention": _prepare_attention, "copy": _prepare_copy, "compact": _prepare_compact, "verify": _prepare_verify}[case["op"]](case, g, h)


def _int(x):
    return torch.as_tensor(x).to(torch.int32).to(DEV)


def _prepare_attention(c, g, h):
    B, T, ps, hkv, dim = c["batch"], c["tokens"], c["page"], c["hkv"], c["dim"]
    n, in_groups = c["groups"], c["batch"] - c["alone"]
    seqs = torch.randperm(B, generator=h)[:in_groups].tolist()  # sessions sit in any slot
    members = [sorted(seqs[i::n]) for i in range(n)]
    shared = [max(1, c["prefix"] - 37 * i) for i in range(n)]  # prefixes of other lengths, that end inside a page
    lens = torch.randint(T, max(T, c["most"]) + 1, (B,), generator=h)
    for m, p in zip(members, shared):
        lens[m] += p
    need = (lens + ps - 1) // ps
    table = torch.zeros(B, int(need.max()), dtype=torch.int64)
    own_pages = [int(x) for x in need]
    for m, p in zip(members, shared):
        for b in m:
            own_pages[b] -= p // ps
    total = sum(own_pages) + sum(p // ps for p in shared)
    ids = (torch.randperm(total, generator=h) + 1)  # page 0 stays free, as in the engine's pools
    at = 0
    for m, p in zip(members, shared):
        k = p // ps
        table[m, :k] = ids[at:at + k]
        at += k
    for b in range(B):
        k = own_pages[b]
        table[b, int(need[b]) - k:int(need[b])] = ids[at:at + k]
        at += k
    shape = (total + 1, hkv, ps, dim)
    kc = torch.randn(shape, device=DEV, generator=g).to(torch.bfloat16)
    vc = torch.randn(shape, device=DEV, generator=g).to(torch.bfloat16)
    for m, p in zip(members, shared):  # the page that the prefix ends in was copied when the sessions forked
        if p % ps:
            to, frm = table[m, p // ps].to(DEV), int(table[m[0], p // ps])
            kc[to, :, :p % ps] = kc[frm, :, :p % ps]
            vc[to, :, :p % ps] = vc[frm, :, :p % ps]
    q = (torch.randn(B * T, c["hq"] * dim, device=DEV, generator=g) * 1.5).to(torch.bfloat16)
    s = dict(op="attention", q=q, kc=kc, vc=vc, table=_int(table), lens=_int(lens), scale=1.0 / math.sqrt(dim), tokens=T)
    if own:
        from mesh_b200 import ops
        s["groups"] = ops.PrefixGroups(B, c["hq"], hkv, dim, q_len=T, device=DEV)
        s["groups"].set(list(zip(members, shared)))
    return s


def _pools(c, g):
    shape = (c["layers"], c["pages"], c["heads"], c["page"], c["dim"])
    return torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16), torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16)


def _prepare_copy(c, g, h):
    k, v = _pools(c, g)
    ids = torch.randperm(c["pages"] - 1, generator=h) + 1
    n = c["pairs"]
    src, dst = ids[:n].clone(), ids[n:2 * n]
    if c["tokens"] < c["page"]:
        src[:] = src[0]  # a fork: every child's last page from the one parent's
    return dict(op="copy", k=k, v=v, src=_int(src), dst=_int(dst), tokens=_int(torch.full((n,), c["tokens"])))


def _prepare_compact(c, g, h):
    k, v = _pools(c, g)
    live = 1 + c["shared"] + c["seqs"] * c["per"]
    low = torch.randperm(live - 1, generator=h)[:live - 1 - c["moves"]] + 1
    high = torch.randperm(c["pages"] - live, generator=h)[:c["moves"]] + live
    ids = torch.cat([low, high])[torch.randperm(live - 1, generator=h)]
    table = torch.zeros(c["seqs"], c["shared"] + c["per"] + 3, dtype=torch.int64)
    table[:, :c["shared"]] = ids[:c["shared"]]
    table[:, c["shared"]:c["shared"] + c["per"]] = ids[c["shared"]:].view(c["seqs"], c["per"])
    return dict(op="compact", k=k, v=v, table=_int(table), counts=_int(torch.full((c["seqs"],), c["shared"] + c["per"])))


def _prepare_verify(c, g, h):
    B, K, V = c["batch"], c["drafts"], c["vocab"]
    base = torch.randn(B, K + 1, V, device=DEV, generator=g) * 2.5
    logits = base + 0.6 * torch.randn(B, K + 1, V, device=DEV, generator=g)  # the target: near the draft model, not it
    u = torch.rand(B, K, V, device=DEV, generator=g).clamp_(1e-9, 1.0 - 1e-7)
    ids = (base[:, :K] - torch.log(-torch.log(u))).argmax(-1)  # drafted from the draft model's probabilities
    probs = torch.softmax(base[:, :K], -1) if c["probs"] else None
    if not c["probs"]:
        best = logits[:, :K].argmax(-1)
        ids = torch.where(torch.rand(B, K, device=DEV, generator=g) < 0.6, best, ids)
    inv_t = 1.0 / (0.5 + torch.rand(B, device=DEV, generator=g))
    if c["greedy"]:
        inv_t[::c["greedy"]] = 0.0
    lens = torch.full((B,), K) if c["probs"] else torch.randint(0, K + 1, (B,), generator=h)
    if c["half"]:
        logits = logits.to(torch.bfloat16)
    return dict(op="verify", logits=logits, ids=_int(ids), probs=probs, uniforms=torch.rand(B, K + 1, device=DEV, generator=g), inv_t=inv_t, lens=_int(lens))


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        from mesh_b200 import ops
        if s["op"] == "attention":
            out = torch.empty_like(s["q"])
            return ops.attn_shared_prefix(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["groups"], out, s["scale"])
        if s["op"] == "copy":
            ops.kv_pages_copy(s["k"], s["v"], s["src"], s["dst"], s["tokens"])
            return dict(k=s["k"], v=s["v"])
        if s["op"] == "compact":
            table, remap, live = ops.kv_pages_compact(s["k"], s["v"], s["table"], s["counts"])
            return dict(k=s["k"], v=s["v"], table=table, remap=remap, live=live)
        tokens, accepted, probs = ops.verify_drafts(s["logits"], s["ids"], s["uniforms"], inv_t=s["inv_t"], draft_probs=s["probs"], draft_lens=s["lens"])
        return dict(tokens=tokens, accepted=accepted, probs=probs)
    return {"attention": _attention, "copy": _copy, "compact": _compact, "verify": _verify}[s["op"]](s)


def _attention(s):
    """Softmax attention of every session's new tokens over its own pages, in fp32."""
    q, kc, T = s["q"], s["kc"], s["tokens"]
    hkv, ps, dim = kc.shape[1:]
    B, P = s["table"].shape
    G = q.shape[1] // dim // hkv
    pages = s["table"].long()
    k = kc[pages].permute(0, 2, 1, 3, 4).reshape(B, hkv, P * ps, dim).float()
    v = s["vc"][pages].permute(0, 2, 1, 3, 4).reshape(B, hkv, P * ps, dim).float()
    x = q.view(B, T, hkv, G, dim).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * T, dim).float()
    score = torch.matmul(x, k.transpose(2, 3)).view(B, hkv, G, T, P * ps) * s["scale"]
    last = s["lens"].long()[:, None] - T + torch.arange(T, device=q.device)  # the key that each new token sits at
    seen = torch.arange(P * ps, device=q.device) <= last[:, :, None]
    score = torch.where(seen[:, None, None], score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(B, hkv, G * T, P * ps), v).view(B, hkv, G, T, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(B * T, -1).to(torch.bfloat16)


def _copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    k, v = s["k"], s["v"]
    took = (torch.arange(k.shape[3], device=k.device) < s["tokens"][:, None])[None, :, None, :, None]
    k[:, dst] = torch.where(took, k[:, src], k[:, dst])
    v[:, dst] = torch.where(took, v[:, src], v[:, dst])
    return dict(k=k, v=v)


def _compact(s):
    """The pages from the live count up go, in order, into the holes below it; entries of a table past its count stay."""
    k, v, table = s["k"], s["v"], s["table"].long()
    n = k.shape[1]
    valid = torch.arange(table.shape[1], device=k.device) < s["counts"][:, None]
    used = torch.zeros(n, dtype=torch.bool, device=k.device)
    used[torch.where(valid, table, torch.zeros_like(table)).reshape(-1)] = True
    used[0] = True  # the reserved page
    ids = torch.arange(n, device=k.device)
    live = used.sum()
    src, dst = (used & (ids >= live)).nonzero()[:, 0], (~used & (ids < live)).nonzero()[:, 0]
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    remap = torch.where(used, ids, torch.full_like(ids, -1))
    remap[src] = dst
    return dict(k=k, v=v, table=torch.where(valid, remap[table], table).to(torch.int32), remap=remap.to(torch.int32), live=live.to(torch.int32).reshape(1))


def _verify(s):
    """Draft k of a session is accepted while u_k q(x_k) < p(x_k); the token after the last accepted one is drawn from max(p - q, 0) (from p after
    the last draft) at the point u of its mass. Greedy sessions (inv_t 0) accept the target's first maximum. In 64 bits: the draw compares sums
    over the vocabulary with a point that may lie between two near ones."""
    B, K1, V = s["logits"].shape
    K = K1 - 1
    dev = s["logits"].device
    x, ids = s["logits"].double(), s["ids"].long()
    greedy = s["inv_t"] <= 0
    best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device=dev), V).amin(-1)
    y = (x - x.amax(-1, keepdim=True)) * torch.where(greedy, torch.ones_like(s["inv_t"]), s["inv_t"]).double()[:, None, None]
    p = torch.exp(y)
    p = p / p.sum(-1, keepdim=True)
    at = torch.arange(V, device=dev)
    px = torch.where(greedy[:, None], (best[:, :K] == ids).double(), p[:, :K].gather(2, ids[..., None])[..., 0])
    if s["probs"] is not None:
        qx = s["probs"].gather(2, ids[..., None])[..., 0].double()
    else:
        qx = torch.ones_like(px)
    passed = torch.where(greedy[:, None], px > 0, s["uniforms"][:, :K].double() * qx < px) & (torch.arange(K, device=dev) < s["lens"][:, None])
    n = torch.cumprod(passed.to(torch.int64), 1).sum(1)
    rows = torch.arange(B, device=dev)
    rest = p[rows, n]
    k = torch.clamp(n, max=K - 1)
    if s["probs"] is not None:
        less = torch.clamp(rest - s["probs"][rows, k].double(), min=0)
    else:
        less = torch.where(at == ids[rows, k][:, None], torch.zeros_like(rest), rest)
    rejected = (n < s["lens"])[:, None] & (less.sum(1, keepdim=True) > 0)
    rest = torch.where(rejected, less, rest)
    mass = torch.cumsum(rest, 1)
    drawn = (mass > s["uniforms"][:, K:].double() * mass[:, -1:]).to(torch.int64)
    new = torch.where(greedy, best[rows, n], drawn.argmax(1))
    col = torch.arange(K1, device=dev)
    padded = torch.cat([ids, ids[:, :1]], 1)
    tokens = torch.where(col < n[:, None], padded, torch.where(col == n[:, None], new[:, None], torch.full_like(padded, -1)))
    given = torch.arange(K, device=dev) < s["lens"][:, None]
    return dict(tokens=tokens.to(torch.int32), accepted=n.to(torch.int32), probs=torch.where(given, px, torch.zeros_like(px)).float())


# ------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    if case["op"] in ("copy", "compact"):
        return None  # moves alone: nothing is computed
    s = prepare(case, seed)
    if case["op"] == "attention":
        T, dim, hkv, ps = case["tokens"], case["dim"], case["hkv"], case["page"]
        G = case["hq"] // hkv
        outs = []
        for b, n in enumerate(s["lens"].tolist()):
            pages = s["table"][b, :(n + ps - 1) // ps].long()
            k = s["kc"][pages].double().transpose(1, 2).reshape(-1, hkv, dim)[:n]
            v = s["vc"][pages].double().transpose(1, 2).reshape(-1, hkv, dim)[:n]
            x = s["q"][b * T:(b + 1) * T].double().view(T, hkv, G, dim)
            a = torch.einsum("thgd,nhd->hgtn", x, k) / math.sqrt(dim)
            late = torch.arange(n, device=DEV)[None] > (n - T + torch.arange(T, device=DEV))[:, None]
            a = torch.softmax(a.masked_fill(late, -math.inf), -1)
            outs.append(torch.einsum("hgtn,nhd->thgd", a, v).reshape(T, -1))
        return torch.cat(outs)
    x, ids, lens = s["logits"].double(), s["ids"].long(), s["lens"].tolist()
    probs = torch.zeros(ids.shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        for k in range(n):
            t = float(s["inv_t"][b])
            if t > 0:
                z = x[b, k] * t
                probs[b, k] = torch.exp(z[ids[b, k]] - torch.logsumexp(z, 0))
            else:
                probs[b, k] = float(int(torch.nonzero(x[b, k] == x[b, k].max())[0]) == int(ids[b, k]))
    return dict(tokens=None, accepted=None, probs=probs)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "attention":
        # the mean length of a session's own part; a shared prefix is read once for its group
        rest = (c["tokens"] + max(c["tokens"], c["most"])) / 2
        shared = [max(1, c["prefix"] - 37 * i) for i in range(c["groups"])]
        keys = sum(shared) + c["batch"] * rest
        seen = c["batch"] * rest + (c["batch"] - c["alone"]) * sum(shared) / c["groups"]
        row = c["hq"] * c["dim"] * c["tokens"]
        return {"bytes": keys * c["hkv"] * c["dim"] * 4 + c["batch"] * row * 4, "flops": 4 * seen * row}
    page = c["layers"] * c["heads"] * c["dim"] * 4 if c["op"] in ("copy", "compact") else 0  # K and V of one token
    if c["op"] == "copy":
        read = c["tokens"] * (1 if c["tokens"] < c["page"] else c["pairs"])
        return {"bytes": page * (read + c["tokens"] * c["pairs"]), "flops": 0}
    if c["op"] == "compact":
        return {"bytes": 2 * page * c["page"] * c["moves"] + 8 * c["seqs"] * (c["shared"] + c["per"]) + 4 * c["pages"], "flops": 0}
    rows = c["batch"] * (c["drafts"] + 1)
    # every row of logits once (each draft's target probability is an answer), and the draft's row where one is rejected
    return {"bytes": rows * c["vocab"] * (2 if c["half"] else 4) + (c["batch"] * c["vocab"] * 4 if c["probs"] else 0), "flops": 4 * rows * c["vocab"]}
