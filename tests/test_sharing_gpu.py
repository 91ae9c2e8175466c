"""Sessions that share pages and propose tokens ahead: page copies, compaction, attention over shared prefixes and
draft verification, each against a plain implementation in 64 bits (moves: exactly), at the sizes and masks
where they can go wrong, and run together as a serving step uses them.

Tolerances. Attention rounds its weights to bf16 for the product with V (each off by at most eps/2 = 2^-8
relative) and its output once more: |error| <= 2^-8 (sum w |v| + |o|) elementwise, plus fp32 sums over at
most a few thousand keys (each addition 2^-24 of values whose magnitudes sum to sum w |v|; 2^-11 bounds 8192
of them) and scores whose fp32 error (a 128-term product, |s| <= 64: 128 * 2^-24 * 64 < 2^-10) scales a weight by as
much. The bound used is (2^-8 + 2^-9) (sum w |v| + |o|).
"""
import math

import pytest
import torch

from mesh_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _check_err():
    yield
    ops.scratch(torch.device("cuda", torch.cuda.current_device())).check("kernel")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _pools(L=3, P=40, hkv=2, ps=16, D=64, seed=0):
    g = _gen(seed)
    return [torch.randn(L, P, hkv, ps, D, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------ page copies
@pytest.mark.parametrize("hkv,ps,D", [(2, 16, 64), (1, 16, 128), (8, 16, 128), (3, 8, 24), (5, 7, 8), (8, 32, 128)])
@pytest.mark.parametrize("as_list", [True, False])
def test_kv_pages_copy(hkv, ps, D, as_list):
    k, v = _pools(hkv=hkv, ps=ps, D=D)
    src, dst = [7, 7, 2, 39, 0], [1, 30, 38, 12, 11]
    tokens = [ps, 1, 0, ps // 2, ps - 1]
    wk, wv = k.clone(), v.clone()
    for a, b, t in zip(src, dst, tokens):
        wk[:, b, :, :t] = k[:, a, :, :t]
        wv[:, b, :, :t] = v[:, a, :, :t]
    if as_list:
        ops.kv_pages_copy(k, v, src, dst, tokens)
    else:
        ops.kv_pages_copy(k, v, _i32(src), _i32(dst), _i32(tokens))
    assert torch.equal(k, wk) and torch.equal(v, wv)
    ops.kv_pages_copy(k, v, [], [])  # nothing to copy
    ops.kv_pages_copy(k, v, [3], [4])
    assert torch.equal(k[:, 4], wk[:, 3]) and torch.equal(v[:, 4], wv[:, 3])


def test_kv_pages_copy_padding_is_left_out():
    k, v = _pools()
    wk = k.clone()
    wk[:, 9] = k[:, 4]
    ops.kv_pages_copy(k, v, _i32([4, -1, 5]), _i32([9, 6, -1]))
    assert torch.equal(k, wk)


def test_kv_pages_copy_many_pairs():
    k, v = _pools(L=2, P=3000, hkv=1, D=64)
    perm = torch.randperm(3000, generator=torch.Generator().manual_seed(3))
    src, dst = perm[:1500], perm[1500:]
    wk, wv = k.clone(), v.clone()
    wk[:, dst.to(DEV)] = k[:, src.to(DEV)]
    wv[:, dst.to(DEV)] = v[:, src.to(DEV)]
    ops.kv_pages_copy(k, v, src.to(torch.int32).to(DEV), dst.to(torch.int32).to(DEV))
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_kv_pages_copy_refusals():
    k, v = _pools()
    for bad in (([40], [1]), ([1], [-1]), ([1, 2], [3]), ([1, 2], [3, 3]), ([1, 2], [2, 3]), ([5], [5])):
        with pytest.raises(ValueError):
            ops.kv_pages_copy(k, v, *bad)
    with pytest.raises(ValueError):
        ops.kv_pages_copy(k, v, [1], [2], [17])
    with pytest.raises(RuntimeError):
        ops.kv_pages_copy(k, v.float(), _i32([1]), _i32([2]))
    with pytest.raises(RuntimeError):
        ops.kv_pages_copy(k, v, _i32([1]), _i32([2, 3]))
    with pytest.raises(RuntimeError):
        ops.kv_pages_copy(k, v, _i32([1]).long(), _i32([2]).long())
    with pytest.raises(RuntimeError):
        ops.kv_pages_copy(k[:, :, :, :, :60], v[:, :, :, :, :60], _i32([1]), _i32([2]))
    before = k.clone()
    for src, dst in (([40], [1]), ([1], [40]), ([1, 2], [3, 3]), ([1, 2], [2, 3])):
        ops.kv_pages_copy(k, v, _i32(src), _i32(dst))
        with pytest.raises(RuntimeError, match="5 bad argument"):
            ops.scratch(DEV).check("copy")
    assert torch.equal(k[:, 1], before[:, 1])  # ids outside the pool moved nothing


# ------------------------------------------------------------------------------------ compaction
def _compact_plain(pages, reserved, table, counts):
    live = set(range(reserved))
    for row, c in zip(table, counts):
        live |= set(row[:c])
    n = len(live)
    high = sorted(p for p in live if p >= n)
    holes = sorted(p for p in range(n) if p not in live)
    remap = [p if p in live else -1 for p in range(pages)]
    for a, b in zip(high, holes):
        remap[a] = b
    new = [[remap[p] if i < c else p for i, p in enumerate(row)] for row, c in zip(table, counts)]
    return new, remap, n, high, holes


@pytest.mark.parametrize("pages,rows,width,reserved,seed", [(40, 4, 6, 1, 0), (40, 4, 6, 0, 1), (40, 1, 1, 1, 2),
                                                            (33, 8, 4, 1, 3), (1000, 30, 20, 1, 4), (64, 3, 9, 5, 5),
                                                            (5000, 64, 70, 1, 6), (32, 1, 31, 1, 7)])
@pytest.mark.parametrize("in_place", [True, False])
def test_kv_pages_compact(pages, rows, width, reserved, seed, in_place):
    import random
    r = random.Random(seed)
    k, v = _pools(L=2, P=pages, hkv=1, D=64, seed=seed)
    counts = [r.randint(0, width) for _ in range(rows)]
    pool = r.sample(range(reserved, pages), min(pages - reserved, sum(counts)))
    table = [[r.choice(pool) if pool else 0 for _ in range(width)] for _ in range(rows)]  # pages shared between rows
    new, remap, live, high, holes = _compact_plain(pages, reserved, table, counts)
    wk, wv = k.clone(), v.clone()
    if high:
        wk[:, holes], wv[:, holes] = k[:, high], v[:, high]
    t = _i32(table)
    kept = t.clone()
    got, gmap, glive = ops.kv_pages_compact(k, v, t, _i32(counts), reserved=reserved, out_tables=t if in_place else None)
    assert got.tolist() == new and gmap.tolist() == remap and glive.tolist() == [live]
    assert torch.equal(k, wk) and torch.equal(v, wv)
    assert in_place or torch.equal(t, kept)
    # what is compact already does not move
    again, amap, alive = ops.kv_pages_compact(k, v, got.clone(), _i32(counts), reserved=reserved)
    assert again.tolist() == new and alive.tolist() == [live]
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_kv_pages_compact_full_and_empty():
    k, v = _pools(P=9)
    kept = k.clone()
    t = _i32([[8, 7, 6, 5, 4, 3, 2, 1]])
    got, remap, live = ops.kv_pages_compact(k, v, t, _i32([8]))
    assert torch.equal(got, t) and live.tolist() == [9] and remap.tolist() == list(range(9))
    got, remap, live = ops.kv_pages_compact(k, v, t, _i32([0]))
    assert torch.equal(got, t) and live.tolist() == [1] and remap.tolist() == [0] + [-1] * 8
    assert torch.equal(k, kept)


def test_kv_pages_compact_refusals():
    k, v = _pools()
    t, c = _i32([[1, 2]]), _i32([2])
    with pytest.raises(RuntimeError):
        ops.kv_pages_compact(k, v, t, _i32([1, 2]))
    with pytest.raises(RuntimeError):
        ops.kv_pages_compact(k, v, t, c, reserved=41)
    with pytest.raises(RuntimeError):
        ops.kv_pages_compact(k, v, t.long(), c)
    with pytest.raises(RuntimeError):
        ops.kv_pages_compact(k, v, t.cpu(), c.cpu())
    kept = k.clone()
    got, _, live = ops.kv_pages_compact(k, v, _i32([[1, 40, -3, 2]]), _i32([4]))
    with pytest.raises(RuntimeError, match="5 bad argument"):
        ops.scratch(DEV).check("compact")
    assert got.tolist() == [[1, 40, -3, 2]] and live.tolist() == [3] and torch.equal(k, kept)


# ------------------------------------------------------------------------------------ attention over shared prefixes
def _shared_case(B, T, hq, hkv, D, ps, groups, own, seed, junk=False):
    """groups: (sequences, prefix length); own: each sequence's keys after its prefix (0: an empty slot if
    it is in no group). junk: NaN and infinity in every page position past a sequence's end."""
    g, h = _gen(seed), torch.Generator().manual_seed(seed)
    prefix = [0] * B
    for seqs, n in groups:
        for b in seqs:
            prefix[b] = n
    lens = [p + o for p, o in zip(prefix, own)]
    need = [-(-n // ps) for n in lens]
    total = sum(need) + 1
    ids = (torch.randperm(total - 1, generator=h) + 1).tolist()
    width = max(need) + 1
    table = torch.zeros(B, width, dtype=torch.int64)
    for b in range(B):
        for i in range(need[b]):
            table[b, i] = ids.pop()
    for seqs, n in groups:
        for b in seqs[1:]:
            k = min(n // ps, need[b])
            table[b, :k] = table[seqs[0], :k]
    kc = torch.randn(total, hkv, ps, D, device=DEV, generator=g).to(torch.bfloat16)
    vc = torch.randn(total, hkv, ps, D, device=DEV, generator=g).to(torch.bfloat16)
    for seqs, n in groups:
        if n % ps:
            for b in seqs[1:]:
                if need[b] > n // ps:
                    for c in (kc, vc):
                        c[table[b, n // ps], :, :n % ps] = c[table[seqs[0], n // ps], :, :n % ps]
    if junk:
        used = torch.zeros(total, ps, dtype=torch.bool)
        for b in range(B):
            for i in range(need[b]):
                used[table[b, i], :min(ps, lens[b] - i * ps)] = True
        bad = (~used).to(DEV)[:, None, :, None]
        kc = torch.where(bad, torch.full_like(kc, math.nan), kc)
        vc = torch.where(bad, torch.full_like(vc, math.inf), vc)
    q = torch.randn(B * T, hq * D, device=DEV, generator=g).to(torch.bfloat16)
    return q, kc, vc, table.to(torch.int32).to(DEV), _i32(lens)


def _attn_64(q, kc, vc, table, lens, T, scale, window=0):
    """(o, sum w |v|) in 64 bits, one sequence after another."""
    hkv, ps, D = kc.shape[1:]
    B = lens.shape[0]
    hq = q.shape[1] // D
    o = torch.zeros(B * T, hq, D, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(o)
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            continue
        pages = table[b, :-(-n // ps)].long()
        k = kc[pages].transpose(1, 2).reshape(-1, hkv, D)[:n].double().repeat_interleave(hq // hkv, 1)
        v = vc[pages].transpose(1, 2).reshape(-1, hkv, D)[:n].double().repeat_interleave(hq // hkv, 1)
        x = q[b * T:(b + 1) * T].double().view(T, hq, D)
        s = torch.einsum("thd,nhd->htn", x, k) * scale
        pos = n - T + torch.arange(T, device=DEV)[:, None]
        key = torch.arange(n, device=DEV)[None]
        hide = key > pos
        if window:
            hide = hide | (key <= pos - window)
        w = torch.softmax(s.masked_fill(hide, -math.inf), -1).nan_to_num(0.0)
        o[b * T:(b + 1) * T] = torch.einsum("htn,nhd->thd", w, v)
        mag[b * T:(b + 1) * T] = torch.einsum("htn,nhd->thd", w, v.abs())
    return o.reshape(B * T, -1), mag.reshape(B * T, -1)


def _check_attn(out, want, mag):
    bound = (2 ** -8 + 2 ** -9) * (mag + want.abs()) + 1e-30
    worst = ((out.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst


def _run_shared(case, T, hq, hkv, D, groups, window=0, **kw):
    q, kc, vc, table, lens = case
    plan = ops.PrefixGroups(lens.shape[0], hq, hkv, D, q_len=T).set(groups)
    out = torch.full_like(q, math.nan)
    ops.attn_shared_prefix(q, kc, vc, table, lens, plan, out, 1.0 / math.sqrt(D), window=window, **kw)
    return out, plan


HEADS = [(32, 8, 128), (8, 1, 128), (8, 1, 64), (4, 4, 64), (4, 2, 128)]


@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("T", [1, 2, 5, 8])
@pytest.mark.parametrize("window", [0, 90])
def test_attn_shared_prefix_groups(hq, hkv, D, T, window):
    groups = [([5, 0, 2], 300), ([1, 6, 7, 8, 9, 10], 77), ([3], 130)]
    own = [T, T + 1, T + 40, T + 3, T + 200, T + 64, T + 15, T + 16, T, T + 129, T + 2, T + 33]
    case = _shared_case(12, T, hq, hkv, D, 16, groups, own, seed=T + hq, junk=True)
    out, _ = _run_shared(case, T, hq, hkv, D, groups, window)
    want, mag = _attn_64(*case, T, 1.0 / math.sqrt(D), window)
    _check_attn(out, want, mag)


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000, 4097])
def test_attn_shared_prefix_lengths(prefix):
    hq, hkv, D, T = 32, 8, 128, 1
    groups = [([0, 1, 2, 3, 4], prefix)]
    case = _shared_case(5, T, hq, hkv, D, 16, groups, [1, 2, 17, 64, 31], seed=prefix, junk=True)
    out, _ = _run_shared(case, T, hq, hkv, D, groups)
    _check_attn(out, *_attn_64(*case, T, 1.0 / math.sqrt(D)))


@pytest.mark.parametrize("B", [1, 2, 17, 33, 64, 130, 256])
@pytest.mark.parametrize("hq,hkv,D,T", [(32, 8, 128, 1), (32, 4, 64, 1), (8, 1, 128, 3)])
def test_attn_shared_prefix_batches(B, hq, hkv, D, T):
    groups = [(list(range(B))[::-1], 513)]
    own = [T + (7 * i) % 50 for i in range(B)]
    case = _shared_case(B, T, hq, hkv, D, 16, groups, own, seed=B)
    out, _ = _run_shared(case, T, hq, hkv, D, groups)
    _check_attn(out, *_attn_64(*case, T, 1.0 / math.sqrt(D)))


@pytest.mark.parametrize("ps", [16, 32, 48, 128])
def test_attn_shared_prefix_page_sizes(ps):
    hq, hkv, D, T = 8, 2, 64, 2
    groups = [([0, 2, 3], 200), ([1, 4], 96)]
    case = _shared_case(6, T, hq, hkv, D, ps, groups, [5, 9, 60, 130, 2, 300], seed=ps, junk=True)
    out, _ = _run_shared(case, T, hq, hkv, D, groups)
    _check_attn(out, *_attn_64(*case, T, 1.0 / math.sqrt(D)))


def test_attn_shared_prefix_without_groups_and_empty_slots():
    """Lengths of zero, of one, and shorter than the new tokens: rows without a key give zeros."""
    hq, hkv, D, T = 32, 8, 128, 4
    case = _shared_case(6, T, hq, hkv, D, 16, [], [0, 1, 4, 700, 0, 2], seed=1)
    out, _ = _run_shared(case, T, hq, hkv, D, [])
    want, mag = _attn_64(*case, T, 1.0 / math.sqrt(D))
    _check_attn(out, want, mag)
    assert out.view(6, T, -1)[0].abs().sum() == 0 and out.view(6, T, -1)[1, :3].abs().sum() == 0


def test_attn_shared_prefix_member_shorter_than_the_prefix():
    """A slot of a group that holds less than the shared prefix sees its own length only."""
    hq, hkv, D, T = 8, 2, 128, 1
    groups = [([0, 1, 2], 256)]
    q, kc, vc, table, lens = _shared_case(3, T, hq, hkv, D, 16, groups, [10, 10, 10], seed=4)
    lens = _i32([266, 100, 0])
    out, _ = _run_shared((q, kc, vc, table, lens), T, hq, hkv, D, groups)
    want, mag = _attn_64(q, kc, vc, table, lens, T, 1.0 / math.sqrt(D))
    _check_attn(out, want, mag)


def test_attn_shared_prefix_large_scores():
    """Scores in the hundreds: the running maximum carries the sums."""
    hq, hkv, D, T = 8, 2, 128, 1
    groups = [(list(range(9)), 700)]
    q, kc, vc, table, lens = _shared_case(9, T, hq, hkv, D, 16, groups, list(range(1, 10)), seed=5)
    kc *= 4
    out, _ = _run_shared((q, kc, vc, table, lens), T, hq, hkv, D, groups)
    want, mag = _attn_64(q, kc, vc, table, lens, T, 1.0 / math.sqrt(D))
    _check_attn(out, want, mag)


def test_attn_shared_prefix_equals_itself_and_follows_the_graph():
    """The same call twice gives the same bits; a captured call follows new groups, tables and lengths."""
    hq, hkv, D, T = 32, 8, 128, 1
    groups = [([0, 1, 4, 5], 600), ([2, 6], 200)]
    q, kc, vc, table, lens = _shared_case(8, T, hq, hkv, D, 16, groups, [3, 9, 70, 200, 1, 33, 64, 5], seed=6)
    scale = 1.0 / math.sqrt(D)
    plan = ops.PrefixGroups(8, hq, hkv, D).set(groups)
    out = torch.empty_like(q)
    ops.attn_shared_prefix(q, kc, vc, table, lens, plan, out, scale)
    first = out.clone()
    ops.attn_shared_prefix(q, kc, vc, table, lens, plan, out, scale)
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attn_shared_prefix(q, kc, vc, table, lens, plan, out, scale)
    out.zero_()
    graph.replay()
    want, mag = _attn_64(q, kc, vc, table, lens, T, scale)
    _check_attn(out, want, mag)
    plan.set([])  # the sessions part: same tables, nothing shared
    graph.replay()
    _check_attn(out, want, mag)
    lens.copy_(_i32([603, 300, 10, 1, 0, 630, 264, 5]))
    plan.set([([5, 0], 512), ([1, 4], 64)])
    graph.replay()
    want, mag = _attn_64(q, kc, vc, table, lens, T, scale)
    _check_attn(out, want, mag)


def test_attn_shared_prefix_two_streams():
    """Two plans on two streams do not share a workspace."""
    hq, hkv, D, T = 32, 8, 128, 1
    groups = [(list(range(16)), 1024)]
    cases = [_shared_case(16, T, hq, hkv, D, 16, groups, [20] * 16, seed=s) for s in (7, 8)]
    plans = [ops.PrefixGroups(16, hq, hkv, D).set(groups) for _ in cases]
    outs = [torch.empty_like(c[0]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, p, o, s in zip(cases, plans, outs, streams):
            with torch.cuda.stream(s):
                ops.attn_shared_prefix(*c, p, o, 1.0 / math.sqrt(D))
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        _check_attn(o, *_attn_64(*c, T, 1.0 / math.sqrt(D)))


def test_attn_shared_prefix_refusals():
    with pytest.raises(ValueError):
        ops.PrefixGroups(4, 8, 3, 128)
    with pytest.raises(ValueError):
        ops.PrefixGroups(4, 8, 2, 96)
    with pytest.raises(ValueError):
        ops.PrefixGroups(4, 64, 1, 128, q_len=2)
    with pytest.raises(ValueError):
        ops.PrefixGroups(0, 8, 2, 128)
    plan = ops.PrefixGroups(4, 8, 2, 64)
    for bad in ([([0, 4], 16)], [([0, 1], 16), ([1, 2], 16)], [([0, 0], 16)], [([0], -1)]):
        with pytest.raises(ValueError):
            plan.set(bad)
    q, kc, vc, table, lens = _shared_case(4, 1, 8, 2, 64, 16, [], [5, 6, 7, 8], seed=9)
    out = torch.empty_like(q)
    with pytest.raises(ValueError):
        ops.attn_shared_prefix(q[:3], kc, vc, table[:3], lens[:3], plan, out[:3], 1.0)
    with pytest.raises(ValueError):
        ops.attn_shared_prefix(q, kc[:, :1], vc[:, :1], table, lens, plan, out, 1.0)
    with pytest.raises(RuntimeError):
        ops.attn_shared_prefix(q.float(), kc, vc, table, lens, plan, out, 1.0)
    with pytest.raises(RuntimeError):
        ops.attn_shared_prefix(q, kc, vc, table.long(), lens, plan, out, 1.0)
    with pytest.raises(RuntimeError):
        ops.attn_shared_prefix(q, kc[:, :, :8].contiguous(), vc[:, :, :8].contiguous(), table, lens, plan, out, 1.0)
    with pytest.raises(RuntimeError):
        ops.attn_shared_prefix(q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, table, lens, plan, out, 1.0)


# ------------------------------------------------------------------------------------ draft verification
def _verify_plain(logits, ids, u, inv_t, probs, lens):
    """The rule in 64 bits, token by token, on the CPU. Also how near the decisions came to another outcome."""
    x, ids, u = logits.double().cpu(), ids.cpu(), u.double().cpu()
    B, K1, V = x.shape
    K = K1 - 1
    tokens, accepted, near = [], [], 1.0
    prob = torch.zeros(B, K, dtype=torch.float64)
    for b in range(B):
        t = 1.0 if inv_t is None else float(inv_t[b])
        n = K if lens is None else max(0, min(K, int(lens[b])))
        rows = []
        for k in range(n + 1):
            z = torch.where(torch.isnan(x[b, k]), -math.inf, x[b, k])
            m = z.max()
            best = int((z == m).nonzero()[0]) if m > -math.inf else -1
            if t <= 0:
                rows.append((None, best))
                continue
            e = torch.where(z == m, torch.ones_like(z), torch.exp((z - m) * t)) if m > -math.inf else torch.zeros_like(z)
            rows.append((e / e.sum() if m > -math.inf else e, best))
        a = n
        for k in range(n):
            i = int(ids[b, k])
            inside = 0 <= i < V
            p = (float(rows[k][1] == i) if t <= 0 else float(rows[k][0][i])) if inside else 0.0
            prob[b, k] = p
            if a == n:
                qx = 1.0 if probs is None or not inside else float(torch.nan_to_num(probs[b, k, i].double(), nan=0.0).clamp(min=0))
                if not (p > 0 if t <= 0 else float(u[b, k]) * qx < p and p > 0):
                    a = k
                if t > 0 and p > 0:
                    near = min(near, abs(float(u[b, k]) * qx - p) / p)
        p, best = rows[a]
        new = best
        if t > 0 and best >= 0:
            w = p
            if a < n:
                if probs is not None:
                    w = (p - torch.nan_to_num(probs[b, a].double().cpu(), nan=0.0).clamp(min=0)).clamp(min=0)
                else:
                    w = p.clone()
                    if 0 <= int(ids[b, a]) < V:
                        w[int(ids[b, a])] = 0
                if not w.sum() > 0:
                    w = p
            c = torch.cumsum(w, 0)
            point = float(u[b, K]) * float(c[-1])
            new = int((c > point).nonzero()[0])
            gap = torch.cat([c - point, torch.tensor([1.0], dtype=torch.float64)]).abs()
            near = min(near, float(gap[gap > 0].min() / c[-1])) if float(u[b, K]) > 0 else near
        tokens.append([int(ids[b, k]) for k in range(a)] + [new] + [-1] * (K - a))
        accepted.append(a)
    return tokens, accepted, prob, near


def _verify_case(B, K, V, seed, half=False, qhalf=False, probs=True, scale=2.5, noise=0.6):
    g = _gen(seed)
    base = torch.randn(B, K + 1, V, device=DEV, generator=g) * scale
    logits = base + noise * torch.randn(B, K + 1, V, device=DEV, generator=g)
    gum = -torch.log(-torch.log(torch.rand(B, K, V, device=DEV, generator=g).clamp(1e-9, 1 - 1e-7)))
    ids = (base[:, :K] + gum).argmax(-1).to(torch.int32)
    q = torch.softmax(base[:, :K], -1) if probs else None
    u = torch.rand(B, K + 1, device=DEV, generator=g)
    inv_t = (0.5 + torch.rand(B, device=DEV, generator=g)).float()
    if half:
        logits = logits.to(torch.bfloat16)
    if qhalf and q is not None:
        q = q.to(torch.bfloat16)
    return logits, ids, u, inv_t, q


def _check_verify(logits, ids, u, inv_t, q, lens=None, tol=1e-11):
    got = ops.verify_drafts(logits, ids, u, inv_t=inv_t, draft_probs=q, draft_lens=lens)
    tokens, accepted, prob, near = _verify_plain(logits, ids, u, inv_t, q, lens)
    assert near > tol  # the inputs do not put a decision within the 64-bit sums' own rounding
    assert got[1].tolist() == accepted
    assert got[0].tolist() == tokens
    # probabilities are rounded once to fp32 (2^-24 relative), from 64-bit sums
    assert torch.allclose(got[2].double().cpu(), prob, rtol=2 ** -23, atol=1e-37)
    return accepted


@pytest.mark.parametrize("B,K,V", [(1, 4, 128256), (7, 3, 32000), (5, 1, 1), (5, 2, 2), (9, 8, 1001), (3, 31, 300),
                                   (4, 0, 777), (33, 4, 4097), (2, 5, 8192), (2, 5, 8193), (3, 2, 40961)])
@pytest.mark.parametrize("half,qhalf,probs", [(False, False, True), (True, True, True), (True, False, False),
                                              (False, True, True), (False, False, False)])
def test_verify_drafts(B, K, V, half, qhalf, probs):
    logits, ids, u, inv_t, q = _verify_case(B, K, V, seed=B * 100 + K, half=half, qhalf=qhalf, probs=probs)
    acc = _check_verify(logits, ids, u, inv_t, q)
    if probs and V > 1000 and B * K > 20:
        assert 0 < sum(acc) < B * K  # some are accepted, some refused


def test_verify_drafts_greedy_ragged_and_defaults():
    logits, ids, u, inv_t, q = _verify_case(24, 5, 3001, seed=1, half=True)  # bf16: ties between maxima
    best = logits.float().argmax(-1).to(torch.int32)[:, :5]
    ids = torch.where(torch.rand(24, 5, device=DEV, generator=_gen(2)) < 0.8, best, ids)
    inv_t[::2] = 0.0
    lens = _i32([i % 6 for i in range(22)] + [9, -2])
    _check_verify(logits, ids, u, inv_t, q, lens)
    _check_verify(logits, ids, u, inv_t, None, lens)
    _check_verify(logits, ids, u, None, q, None)


def test_verify_drafts_equal_distributions():
    """p = q: everything is accepted for u < 1, and with u = 1 nothing is left over, so p itself is drawn from."""
    B, K, V = 6, 3, 2000
    logits = torch.zeros(B, K + 1, V, device=DEV)  # p = 1 / V exactly
    logits[:, :, 1024:] = -math.inf                # 1024 tokens: q = 2^-10 without rounding
    q = torch.where(torch.arange(V, device=DEV) < 1024, 2.0 ** -10, 0.0).expand(B, K, V).contiguous()
    ids = torch.randint(0, 1024, (B, K), device=DEV, generator=_gen(3)).to(torch.int32)
    u = torch.rand(B, K + 1, device=DEV, generator=_gen(4))
    tokens, accepted, probs = ops.verify_drafts(logits, ids, u, draft_probs=q)
    assert accepted.tolist() == [K] * B and torch.equal(tokens[:, :K], ids)
    assert tokens[:, K].tolist() == (u[:, K].double() * 1024).long().tolist()
    assert torch.equal(probs, torch.full_like(probs, 2.0 ** -10))
    u[:, 1] = 1.0
    tokens, accepted, _ = ops.verify_drafts(logits, ids, u, draft_probs=q)
    assert accepted.tolist() == [1] * B
    assert tokens[:, 1].tolist() == (u[:, K].double() * 1024).long().tolist()
    assert (tokens[:, 2:] == -1).all()


def test_verify_drafts_masked_rows():
    """-inf, NaN and +inf logits, the type's lowest value, rows with nothing to choose, drafts outside the vocabulary."""
    V, K = 9000, 2
    logits, ids, u, inv_t, q = _verify_case(12, K, V, seed=5)
    ids[:] = ids.clamp(min=10)
    logits[0, 0] = -math.inf                      # nothing to choose in the first row
    logits[1, 0, 5:] = -math.inf                  # the draft is masked
    logits[2, :, ::2] = math.nan
    logits[3, 0, 17] = math.inf
    logits[3, 0, 8999] = math.inf
    ids[3, 0] = 8999
    logits[4, :] = torch.finfo(torch.float32).min  # masked with the lowest value throughout: uniform
    logits[5, :, 1:] = torch.finfo(torch.float32).min
    ids[6, 0], ids[7, 1] = V, -1
    q[8, 0, ::3] = math.nan
    q[8, 1, 1::3] = -1.0
    q[9] = 1.0                                    # more than p everywhere: nothing is left of p
    logits[10, :] = -math.inf
    logits[10, :, 8191] = 3.0
    ids[10] = 8191
    q[10, :, 8191] = 1.0
    logits[11] = math.nan
    _check_verify(logits, ids, u, inv_t, q)
    _check_verify(logits, ids, u, inv_t, None)
    _check_verify(logits, ids, u, torch.zeros_like(inv_t), q)


def test_verify_drafts_uniform_ends():
    """u = 0 draws the first token with mass; a u that reaches 1 draws the last."""
    V = 5000
    logits = torch.full((2, 1, V), -math.inf, device=DEV)
    logits[:, 0, [100, 4500]] = 0.0
    ids = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    tokens, accepted, probs = ops.verify_drafts(logits, ids, torch.tensor([[0.0], [1.0]], device=DEV))
    assert tokens.tolist() == [[100], [4500]] and accepted.tolist() == [0, 0] and probs.shape == (2, 0)


def test_verify_drafts_strided_rows():
    """Rows of a wider buffer, starting at odd elements; probabilities likewise."""
    for half in (False, True):
        logits, ids, u, inv_t, q = _verify_case(5, 3, 2999, seed=6, half=half, qhalf=half)
        wide = torch.full((5, 4, 3011), 50.0, device=DEV, dtype=logits.dtype)
        wide[:, :, 3:3002] = logits
        qwide = torch.full((5, 3, 3001), 9.0, device=DEV, dtype=q.dtype)
        qwide[:, :, 1:3000] = q
        _check_verify(wide[:, :, 3:3002], ids, u, inv_t, qwide[:, :, 1:3000])


def test_verify_drafts_distribution():
    """Accepted and drawn tokens follow the target: 30000 sessions of one draft over 8 tokens. Each frequency's
    standard deviation is sqrt(p (1 - p) / n) < 0.003; five of them bound every token."""
    n, V = 30000, 8
    g = _gen(7)
    base = torch.randn(V, device=DEV, generator=g)
    target = torch.randn(V, device=DEV, generator=g)
    p, q = torch.softmax(target, 0), torch.softmax(base, 0)
    ids = torch.multinomial(q.expand(n, V), 1, generator=g).to(torch.int32)
    u = torch.rand(n, 2, device=DEV, generator=g)
    tokens, _, _ = ops.verify_drafts(target.expand(n, 2, V), ids, u, draft_probs=q.expand(n, 1, V))
    freq = torch.bincount(tokens[:, 0].long(), minlength=V).double() / n
    sd = (p.double() * (1 - p.double()) / n).sqrt()
    assert ((freq - p.double()).abs() <= 5 * sd).all()


def test_verify_drafts_captured():
    logits, ids, u, inv_t, q = _verify_case(6, 4, 10007, seed=8)
    ops.verify_drafts(logits, ids, u, inv_t=inv_t, draft_probs=q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, accepted, _ = ops.verify_drafts(logits, ids, u, inv_t=inv_t, draft_probs=q)
    other = _verify_case(6, 4, 10007, seed=9)
    for to, frm in zip((logits, ids, u, inv_t, q), other):
        to.copy_(frm)
    graph.replay()
    want, acc, _, near = _verify_plain(*other, None)
    assert near > 1e-11 and tokens.tolist() == want and accepted.tolist() == acc


def test_verify_drafts_refusals():
    logits, ids, u, inv_t, q = _verify_case(2, 3, 50, seed=10)
    with pytest.raises(ValueError):
        ops.verify_drafts(logits[0], ids, u)
    for bad in (dict(draft_ids=ids.long()), dict(uniforms=u[:, :3]), dict(uniforms=u.double()), dict(draft_ids=ids[:, :2]),
                dict(inv_t=inv_t[:1]), dict(draft_probs=q[:, :, :49]), dict(draft_probs=q.double()),
                dict(draft_lens=_i32([1])), dict(logits=logits.double()), dict(logits=logits.transpose(1, 2)),
                dict(inv_t=inv_t.cpu()), dict(logits=logits.cpu())):
        args = dict(logits=logits, draft_ids=ids, uniforms=u, inv_t=inv_t, draft_probs=q, draft_lens=None)
        args.update(bad)
        with pytest.raises(RuntimeError):
            ops.verify_drafts(**args)
    big = torch.zeros(1, 33, 4, device=DEV)
    with pytest.raises(RuntimeError):
        ops.verify_drafts(big, torch.zeros(1, 32, dtype=torch.int32, device=DEV), torch.zeros(1, 33, device=DEV))


def test_attn_shared_prefix_counts_its_keys_in_32_bits():
    """1024 sequences x 8 KV heads x 8 tiles of rows x 16384 slices of 16 keys: 2^30 pieces of work."""
    plan = ops.PrefixGroups(1024, 64, 8, 64, q_len=8)
    q = torch.zeros(8192, 4096, dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros(2, 8, 256, 64, dtype=torch.bfloat16, device="cuda")
    lens = torch.full((1024,), 8, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="more keys than one call"):
        ops.attn_shared_prefix(q, pool, pool, torch.zeros(1024, 1024, dtype=torch.int32, device="cuda"), lens, plan,
                               torch.empty_like(q), 1.0)
    out = torch.full_like(q, 7)
    ops.attn_shared_prefix(q, pool, pool, torch.ones(1024, 1020, dtype=torch.int32, device="cuda"), lens, plan, out, 1.0)
    assert bool((out == 0).all())  # every value is zero


@pytest.mark.parametrize("own", [700, 40, 3])
def test_attn_shared_prefix_own_keys_of_either_amount(own):
    """Much to read behind the prefix (all workers take part) and little (those of one CTA per SM)."""
    B, hq, hkv, D = 96, 32, 8, 128
    groups = [(list(range(B)), 256)]
    case = _shared_case(B, 1, hq, hkv, D, 16, groups, [own] * B, seed=31)
    out, _ = _run_shared(case, 1, hq, hkv, D, groups)
    _check_attn(out, *_attn_64(*case, 1, 1 / math.sqrt(D)))


def test_host_lists_are_refused_inside_a_capture():
    """Their copy would read the same, by then reused, host memory at every replay."""
    plan = ops.PrefixGroups(2, 8, 2, 64)
    pool = torch.zeros(1, 4, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="host"):
            plan.set([([0, 1], 16)])
        with pytest.raises(RuntimeError, match="host"):
            ops.kv_pages_copy(pool, pool.clone(), [1], [2])
        pool.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((pool == 1).all()) and plan.n_items == 0


def test_attention_and_verification_on_two_streams_at_once():
    """Calls with groups of their own on two streams give what they give alone."""
    hq, hkv, D = 32, 8, 128
    groups = [(list(range(24)), 700)]
    cases = [_shared_case(24, 1, hq, hkv, D, 16, groups, [30 + 9 * i for i in range(24)], seed=s) for s in (41, 42)]
    plans = [ops.PrefixGroups(24, hq, hkv, D).set(groups) for _ in cases]
    logits = [torch.randn(3, 5, 32000, device=DEV, generator=_gen(s)) for s in (43, 44)]
    ids = torch.randint(0, 32000, (3, 4), dtype=torch.int32, device=DEV, generator=_gen(45))
    u = torch.rand(3, 5, device=DEV, generator=_gen(46))

    def run(i, out):
        q, kc, vc, table, lens = cases[i]
        ops.attn_shared_prefix(q, kc, vc, table, lens, plans[i], out, 1 / math.sqrt(D))
        return ops.verify_drafts(logits[i], ids, u)

    alone = []
    for i in range(2):
        out = torch.empty_like(cases[i][0])
        alone.append((out, *run(i, out)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[torch.empty_like(cases[i][0]) for _ in range(8)] for i in range(2)]
    got = [[], []]
    for k in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append((outs[i][k], *run(i, outs[i][k])))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(one, alone[i]))


def test_unaligned_views_and_empty_pools_are_refused():
    """The kernels read 16 bytes at a time."""
    q, kc, vc, table, lens = _shared_case(2, 1, 8, 2, 64, 16, [], [5, 6], seed=51)
    plan = ops.PrefixGroups(2, 8, 2, 64)
    off = torch.zeros(q.numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view_as(q)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.attn_shared_prefix(off, kc, vc, table, lens, plan, torch.empty_like(q), 1.0)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.attn_shared_prefix(q, kc, vc, table, lens, plan, off, 1.0)
    off_kv = torch.zeros(kc.numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view_as(kc)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.attn_shared_prefix(q, off_kv, vc, table, lens, plan, torch.empty_like(q), 1.0)
    none = torch.zeros(0, 4, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="empty pools"):
        ops.kv_pages_copy(none, none.clone(), [1], [2])
    torch.cuda.synchronize()
