"""The operators of drafted decoding over a bounded fp16 cache, measured.

A serving program that drafts several continuations of each sequence as a tree
checks all of them in one pass, keeps the path that the model agrees with, and
holds each sequence to a budget of cached tokens by letting go of those that
little attention went to:

tree     attention of a tree of drafted tokens over the paged cache: a node sees
         the context, its ancestors and itself
accept   the path of drafted tokens that the model's own choices confirm, and its
         K and V moved together behind the context, all layers
weigh    one decode step's attention that also adds up, per cached token and KV
         head, the attention weight the token got
path     the same sums for the tokens of an accepted path, after the pass
evict    the tokens with the largest sums chosen, per layer and KV head, and their
         K and V moved to the front, all layers

The pools are [nb, 16, H, 128] fp16 pages, a sequence's token t in row t % 16 of
page tables[b, t // 16].  A tree's N nodes are the sequence's last N tokens; its
mask words say which nodes a node sees (bit j % 64 of word j // 64: node j).
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE, D = 16, 128
DEV = "cuda"


def listed():
    return [
        # one chat at a short context, a small tree: launch and latency count
        dict(name="tree b1 2k x 8", kind="tree", batch=1, ctx=2048, ragged=False, heads=2, n_rep=6,
             nodes=8, pruned=False),
        # the repository's headline batch and context, 16 drafted tokens each
        dict(name="tree b16 16k x 16", kind="tree", batch=16, ctx=16384, ragged=False, heads=2,
             n_rep=6, nodes=16, pruned=False),
        # a busy server: large trees of different sizes over contexts of all lengths, wider KV
        dict(name="tree b8 ragged 8k x 64", kind="tree", batch=8, ctx=8191, ragged=True, heads=8,
             n_rep=4, nodes=64, pruned=True),
        # one long document, an odd tree: few rows, a long axis to split
        dict(name="tree b1 100k x 33", kind="tree", batch=1, ctx=100003, ragged=False, heads=2,
             n_rep=6, nodes=33, pruned=False),
        # one sequence's tree of 16 accepted, all layers' K and V
        dict(name="accept b1 x 16", kind="accept", batch=1, nodes=16, start=2045, layers=28,
             heads=2),
        # sixteen sequences' trees of 64
        dict(name="accept b16 x 64", kind="accept", batch=16, nodes=64, start=1019, layers=28,
             heads=2),
        # one chat's decode step, its sums kept
        dict(name="weigh b1 2k", kind="weigh", batch=1, ctx=2048, ragged=False, heads=2, n_rep=6),
        # the headline batch's
        dict(name="weigh b16 16k", kind="weigh", batch=16, ctx=16384, ragged=False, heads=2,
             n_rep=6),
        # accepted paths of the headline batch: up to 5 of 16 nodes
        dict(name="path b16 16k", kind="path", batch=16, ctx=16384, ragged=False, heads=2, n_rep=6,
             nodes=16, most=5),
        # many short chats of all lengths, wider KV
        dict(name="path b48 ragged 1.5k", kind="path", batch=48, ctx=1531, ragged=True, heads=8,
             n_rep=4, nodes=8, most=4),
        # one conversation brought back to half its tokens
        dict(name="evict b1 4k to 2k", kind="evict", batch=1, ctx=4096, ragged=False, heads=2,
             layers=28, budget=2048, sinks=4, recent=512),
        # sequences of several lengths to one budget
        dict(name="evict b4 ragged 12k", kind="evict", batch=4, ctx=12289, ragged=True, heads=2,
             layers=28, budget=4001, sinks=4, recent=1000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "accept", "weigh", "path", "evict"])
    heads = rng.choice([1, 2, 3, 4, 8])
    if kind == "accept":
        return dict(kind=kind, batch=_log(rng, 1, 24), nodes=_log(rng, 1, 128),
                    start=rng.randrange(0, 1200), layers=_log(rng, 1, 28), heads=heads)
    if kind == "evict":
        heads, batch, layers = rng.choice([1, 2, 3]), _log(rng, 1, 8), _log(rng, 1, 28)
        ctx = _log(rng, 16, max(17, min(100003, 600000 // (heads * batch * layers))))
        budget = 1 + rng.randrange(ctx)
        recent = rng.randrange(budget + 1)
        return dict(kind=kind, batch=batch, ctx=ctx, ragged=rng.random() < 0.5, heads=heads,
                    layers=layers, budget=budget, sinks=rng.randrange(min(8, budget - recent) + 1),
                    recent=recent)
    batch, n_rep = _log(rng, 1, 96), rng.choice([1, 2, 4, 6, 7, 8, 16])
    nodes = _log(rng, 1, 128) if kind == "tree" else _log(rng, 1, 24)
    most = 16 * 16384 * 2 // (heads * batch)
    if kind != "weigh":
        most = min(most, 16 * 16384 * 2 * 96 // (heads * batch * nodes * n_rep))
    ctx = _log(rng, nodes, max(nodes + 1, min(100003, most)))
    got = dict(kind=kind, batch=batch, ctx=ctx, ragged=rng.random() < 0.6, heads=heads, n_rep=n_rep)
    if kind == "tree":
        got.update(nodes=nodes, pruned=rng.random() < 0.4)
    if kind == "path":
        got.update(nodes=nodes, most=1 + rng.randrange(min(nodes, 8)))
    return got


def _spread(lo, hi, n, step):
    """n whole numbers over lo..hi in mixed order (a case's own, of no seed)."""
    if n == 1:
        return [hi]
    while math.gcd(step, n) != 1:
        step += 1
    return [lo + (hi - lo) * ((step * i + 3) % n) // (n - 1) for i in range(n)]


def _lengths(case):
    """Tokens of each sequence, drafted ones among them."""
    b, ctx = case["batch"], case["ctx"]
    return _spread(min(ctx, case.get("nodes", 1)), ctx, b, 5) if case["ragged"] else [ctx] * b


def _counts(case):
    """Nodes of each sequence's tree, or accepted tokens of each path."""
    b = case["batch"]
    if case["kind"] == "path":
        return _spread(1, case["most"], b, 7)
    return _spread(1, case["nodes"], b, 7) if case.get("pruned") else [case["nodes"]] * b


def work(case):
    kind = case["kind"]
    if kind == "accept":
        rows = case["batch"] * case["layers"] * 2 * case["heads"] * min(case["nodes"], 4)
        return {"bytes": rows * D * 2 * 2 + case["batch"] * case["nodes"] * 20, "flops": 0}
    lens = _lengths(case)
    h = case["heads"]
    if kind == "evict":
        kept = sum(min(n, case["budget"]) for n in lens) * case["layers"] * h
        return {"bytes": sum(lens) * case["layers"] * h * 4 + kept * (8 + 2 * 2 * D * 2), "flops": 0}
    if kind == "weigh":
        rows = case["batch"] * h * case["n_rep"]
        return {"bytes": sum(lens) * h * (2 * D * 2 + 8) + rows * D * 2 * 2,
                "flops": sum(lens) * h * case["n_rep"] * (4 * D + 4)}
    counts = _counts(case)
    rows = sum(counts) * h * case["n_rep"]
    pairs = sum(c * n for c, n in zip(counts, lens)) * h * case["n_rep"]
    if kind == "path":
        return {"bytes": sum(lens) * h * (D * 2 + 8) + rows * (D * 2 + 4), "flops": pairs * 2 * D}
    return {"bytes": sum(lens) * h * 2 * D * 2 + rows * (D * 2 * 2 + 4), "flops": pairs * 4 * D}


def _trees(batch, nodes, seed):
    """Parents [batch, nodes] int32 of random trees whose node 0 is the root."""
    rng = np.random.default_rng(seed)
    i = np.arange(nodes)
    parents = np.floor(i * rng.random((batch, nodes)) ** 0.6).astype(np.int32)
    parents = np.minimum(parents, np.maximum(i - 1, 0)).astype(np.int32)
    parents[:, 0] = -1
    return parents


def _mask_words(parents):
    """int64 [batch, nodes, words]: each node's ancestors and itself."""
    b, n = parents.shape
    words = np.zeros((b, n, -(-n // 64)), np.uint64)
    for i in range(n):
        if i:
            words[:, i] = words[np.arange(b), parents[:, i]]
        words[:, i, i // 64] |= np.uint64(1 << (i % 64))
    return torch.from_numpy(words.view(np.int64)).to(DEV)


def _cache(case, gen):
    """One layer's pools, tables and lengths, with pages in any order."""
    b, h, lens = case["batch"], case["heads"], _lengths(case)
    width = -(-max(lens) // PAGE)
    nb = b * width + 7
    k = torch.randn(nb, PAGE, h, D, generator=gen, device=DEV, dtype=torch.float16)
    v = torch.randn(nb, PAGE, h, D, generator=gen, device=DEV, dtype=torch.float16)
    tables = torch.randperm(nb, generator=gen, device=DEV)[:b * width].view(b, width)
    return dict(k=k, v=v, tables=tables.to(torch.int32), longest=max(lens),
                lens=torch.tensor(lens, dtype=torch.int32, device=DEV))


def _sums(case, width, gen):
    """Weight sums as some time of serving leaves them, and each sequence's row."""
    b, slots = case["batch"], case["batch"] + 3
    sums = torch.exp(2 * torch.randn(slots, case["heads"], width, generator=gen, device=DEV)) * 0.01
    return sums, torch.randperm(slots, generator=gen, device=DEV)[:b].to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, st = case["kind"], {"case": case}
    if own:
        from latentserve_amd.kernels.hip import cache_eviction, tree_attention
        st.update(trees=tree_attention, eviction=cache_eviction)
    b, h = case["batch"], case["heads"]
    if kind in ("tree", "weigh", "path"):
        st.update(_cache(case, gen))
        r = case["n_rep"]
    if kind in ("tree", "path"):
        # q as a view of one projection's output, q, k and v of a token together
        n = case["nodes"]
        x = torch.randn(b, n, h * (r + 2), D, generator=gen, device=DEV).half()
        st["q"] = x[:, :, :h * r].unflatten(2, (h, r))
        st["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEV)
    if kind == "tree":
        st["masks"] = _mask_words(_trees(b, n, seed))
    elif kind == "weigh":
        st["q"] = torch.randn(b, h, r, D, generator=gen, device=DEV).half()
        st["sums"], st["rows"] = _sums(case, st["tables"].shape[1] * PAGE, gen)
    elif kind == "path":
        st["sums"], st["rows"] = _sums(case, st["tables"].shape[1] * PAGE, gen)
        most = case["most"]
        pick = torch.rand(b, n, generator=gen, device=DEV).argsort(1)[:, :most].sort(1).values
        st["path"] = pick.to(torch.int32)
        # the attention's own statistics, as the tree's pass left them
        x, live = _path_scores(st)
        lse = torch.logsumexp(torch.where(live, x, -math.inf), -1)           # [B, H, most, r]
        lse = torch.where(live.any(-1), lse, torch.zeros_like(lse))
        st["lse"] = torch.zeros(b, n, h, r, device=DEV)
        st["lse"][torch.arange(b, device=DEV)[:, None], pick] = lse.transpose(1, 2)
    elif kind == "accept":
        n, start, layers = case["nodes"], case["start"], case["layers"]
        width = -(-(start + n) // PAGE)
        nb = b * width + 5
        st["all"] = torch.randn(layers, 2, nb, PAGE, h, D, generator=gen, device=DEV,
                                dtype=torch.float16)
        st["k_pools"], st["v_pools"] = ([x[z] for x in st["all"]] for z in (0, 1))
        st["tables"] = torch.randperm(nb, generator=gen, device=DEV)[:b * width].view(b, width) \
            .to(torch.int32)
        st["lens"] = torch.full((b,), start + n, dtype=torch.int32, device=DEV)
        # a model that agrees with one child of about four nodes in five
        rng = np.random.default_rng(seed)
        parents = _trees(b, n, seed)
        tokens = rng.integers(0, 1000, (b, n))
        choices = rng.integers(1000, 2000, (b, n))
        for i in range(n - 1, 0, -1):
            at = np.arange(b)[rng.random(b) < 0.8]
            choices[at, parents[at, i]] = tokens[at, i]
        st["parents"], st["tokens"], st["choices"] = (
            torch.from_numpy(np.ascontiguousarray(a)).to(DEV) for a in (parents, tokens, choices))
    elif kind == "evict":
        lens, layers = _lengths(case), case["layers"]
        width = -(-max(lens) // PAGE)
        nb = b * width + 5
        st["all"] = torch.randn(layers, 2, nb, PAGE, h, D, generator=gen, device=DEV,
                                dtype=torch.float16)
        st["k_pools"], st["v_pools"] = ([x[z] for x in st["all"]] for z in (0, 1))
        st["tables"] = torch.randperm(nb, generator=gen, device=DEV)[:b * width].view(b, width) \
            .to(torch.int32)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        # sums of some time's steps: few large, many small, some equal
        w = torch.exp(2 * torch.randn(layers, b, h, width * PAGE, generator=gen, device=DEV)) * 0.01
        few = torch.rand(w.shape, generator=gen, device=DEV)
        st["sums"] = torch.where(few < 0.03, torch.zeros_like(w), w)
    return st


def run(state):
    return _RUN[state["case"]["kind"]](state)


# ---- tree ----------------------------------------------------------------------


def _rows_of(pool, tables):
    """[B, H, T, D] of a pool's pages in their sequences' order, fp32."""
    x = pool[tables.long()]                                                # [B, P, 16, H, D]
    return x.flatten(1, 2).transpose(1, 2).float().contiguous()


def _tree(st):
    if own:
        lse = torch.empty(st["q"].shape[:4], device=DEV)
        out = st["trees"].tree_attention(st["q"], st["k"], st["v"], st["tables"], st["lens"],
                                         st["masks"], st["counts"], max_seq_len=st["longest"],
                                         lse=lse)
        return out, lse
    q, n = st["q"], st["q"].shape[1]
    b, h, r = q.shape[0], q.shape[2], q.shape[3]
    k = _rows_of(st["k"], st["tables"])
    x = torch.matmul(q.float().permute(0, 2, 1, 3, 4).flatten(2, 3),
                     k.transpose(2, 3).contiguous()) / math.sqrt(D)       # [B, H, N r, T]
    del k
    t = torch.arange(x.shape[-1], device=x.device)
    node = t - (st["lens"] - n)[:, None]                                  # [B, T]: context < 0
    j = node.clamp(0, n - 1)
    word = st["masks"].gather(2, (j // 64)[:, None].expand(b, n, -1))     # [B, N, T]
    seen = ((word >> (j % 64)[:, None]) & 1).bool()
    count = st["counts"][:, None]
    live = (node < 0)[:, None] | (seen & (node < count)[:, None])
    live = live & (torch.arange(n, device=x.device) < count)[:, :, None]
    live = live[:, None, :, None].expand(b, h, n, r, -1).flatten(2, 3)
    x = torch.where(live, x, torch.full_like(x, -math.inf))
    best = x.amax(-1, keepdim=True)
    best = torch.where(best == -math.inf, torch.zeros_like(best), best)
    p = torch.exp(x - best)
    del x, live
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p, _rows_of(st["v"], st["tables"])) / total.clamp_min(1e-30)
    lse = (best + torch.log(total))[..., 0].unflatten(2, (n, r)).transpose(1, 2).contiguous()
    return y.unflatten(2, (n, r)).transpose(1, 2).contiguous().half(), lse


# ---- weigh and path --------------------------------------------------------------


def _weigh(st):
    if own:
        out = st["eviction"].paged_decode_weights(st["q"], st["k"], st["v"], st["tables"],
                                                  st["lens"], st["sums"], st["rows"],
                                                  max_seq_len=st["longest"])
        return out, st["sums"]
    k = _rows_of(st["k"], st["tables"])
    x = torch.matmul(st["q"].float(), k.transpose(2, 3).contiguous()) / math.sqrt(D)
    del k
    live = (torch.arange(x.shape[-1], device=x.device) < st["lens"][:, None])[:, None, None]
    x = torch.where(live, x, torch.full_like(x, -math.inf))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    st["sums"][st["rows"].long()] += p.sum(2)
    return torch.matmul(p, _rows_of(st["v"], st["tables"])).half(), st["sums"]


def _path_scores(st):
    """Scores [B, H, P, r, T] of the path's rows, and which of them count."""
    q, path = st["q"], st["path"].long()
    b, _, h, r, _ = q.shape
    most = path.shape[1]
    rows = q[torch.arange(b, device=DEV)[:, None], path].float()           # [B, P, H, r, D]
    k = _rows_of(st["k"], st["tables"])
    x = torch.matmul(rows.permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous(),
                     k.transpose(2, 3).contiguous()) / math.sqrt(D)
    t, i = torch.arange(x.shape[-1], device=DEV), torch.arange(most, device=DEV)
    end = (st["lens"] - st["counts"])[:, None] + i + 1                     # [B, P]
    live = (t < end[..., None]) & (i < st["counts"][:, None])[..., None]
    return x.unflatten(2, (most, r)), live[:, None, :, None].expand(b, h, most, r, -1)


def _path(st):
    if own:
        st["eviction"].add_weights(st["q"], st["lse"], st["k"], st["tables"], st["lens"],
                                   st["sums"], st["rows"], path=st["path"], lengths=st["counts"],
                                   max_seq_len=st["longest"])
        return st["sums"]
    x, live = _path_scores(st)
    b = x.shape[0]
    lse = st["lse"][torch.arange(b, device=DEV)[:, None], st["path"].long()]   # [B, P, H, r]
    p = torch.exp(x - lse.transpose(1, 2)[..., None])
    st["sums"][st["rows"].long()] += torch.where(live, p, torch.zeros_like(p)).sum((2, 3))
    return st["sums"]


# ---- accept and evict --------------------------------------------------------------


def _slots(tables, pos):
    """Flat token slots of positions pos [..., B, H, K] (any leading dimensions)."""
    b = torch.arange(tables.shape[0], device=DEV)[:, None, None]
    return tables[b, pos // PAGE].long() * PAGE + pos % PAGE


def _move(st, src, dst):
    """Rows at positions src [L or 1, B, H, K] of all layers' pools to dst [B, 1, K]."""
    rows = st["all"].flatten(2, 3)                                         # [L, 2, slots, H, D]
    l = torch.arange(rows.shape[0], device=DEV)[:, None, None, None, None]
    z = torch.arange(2, device=DEV)[:, None, None, None]
    head = torch.arange(rows.shape[3], device=DEV)[:, None]
    rows[l, z, _slots(st["tables"], dst), head] = \
        rows[l, z, _slots(st["tables"], src)[:, None], head]


def _accept(st):
    if own:
        got = st["trees"].accept_tokens(st["tokens"], st["parents"], st["choices"], st["k_pools"],
                                        st["v_pools"], st["tables"], st["lens"])
        return (*got, st["all"])
    tokens, choices = st["tokens"], st["choices"]
    b, n = tokens.shape
    i = torch.arange(n, device=DEV)
    par = st["parents"].long().clamp_min(0)
    # the child that each node is followed by: the first whose token its choice is
    fits = (par[:, None] == i[:, None]) & (i > 0) & (tokens[:, None] == choices[..., None])
    then = torch.where(fits, i, n).amin(-1)                                # [B, N], n: none
    then = torch.cat((then, torch.full((b, 1), n, device=DEV)), 1)
    # the nodes that the root leads to, by doubling
    on = torch.zeros(b, n + 1, dtype=torch.bool, device=DEV)
    on[:, 0] = True
    hop = then
    for _ in range(n.bit_length()):
        on = on | (torch.zeros_like(hop).scatter_add_(1, hop, on.long()) > 0)
        hop = hop.gather(1, hop)
    on = on[:, :n]
    length = on.sum(1)
    at = torch.where(on, on.cumsum(1) - 1, n)
    path = torch.full((b, n + 1), -1, device=DEV).scatter_(1, at, i.expand(b, n))[:, :n]
    last = path.gather(1, length[:, None] - 1)
    start = st["lens"].long() - n
    src = start[:, None] + torch.where(path >= 0, path, i)
    heads = st["all"].shape[4]
    _move(st, src[None, :, None].expand(1, b, heads, n), (start[:, None] + i)[:, None])
    return path.int(), length.int(), choices.gather(1, last)[:, 0], st["all"]


def _evict(st):
    case = st["case"]
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    if own:
        got = st["eviction"].evict_tokens(st["sums"], st["k_pools"], st["v_pools"], st["tables"],
                                          st["lens"], budget, sinks=sinks, recent=recent)
        return (*got, st["all"])
    w = st["sums"]
    width = w.shape[-1]
    lens = st["lens"].long()[:, None, None]
    t = torch.arange(width, device=DEV)
    # sums are not negative: their bits are in their order; the lower position first
    order = w.view(torch.int32).long()
    order = torch.where((t < sinks) | (t >= lens - recent), 1 << 32, order)
    order = torch.where(t < lens, order, -1)
    key = torch.topk(order * (1 << 24) + (width - 1 - t), min(budget, width), dim=-1).values
    pos = (width - 1 - (key & ((1 << 24) - 1))).sort(-1).values
    pos = torch.nn.functional.pad(pos, (0, budget - pos.shape[-1]))
    j = torch.arange(budget, device=DEV)
    has = j < lens
    kept = torch.where(has, w.gather(-1, pos), torch.zeros_like(w[..., :1]))
    in_table = j.clamp_max(width - 1)
    _move(st, torch.where(has, pos, in_table), in_table.expand(w.shape[1], 1, -1))
    return torch.where(has, pos, -1).int(), kept, st["all"]


_RUN = {"tree": _tree, "weigh": _weigh, "path": _path, "accept": _accept, "evict": _evict}


# ---- 64 bits, from the definitions ------------------------------------------------


def _sequence(st, which, b, length):
    """Rows of sequence b in 64 bits: [H, length, D]."""
    pos = torch.arange(length, device=DEV)
    page = st["tables"][b].long()[pos // PAGE]
    return st[which][page, pos % PAGE].double().transpose(0, 1).contiguous()


def _attend64(q, k, v, seen):
    """q [H, R, D], seen [R, T] -> out [H, R, D], lse [H, R]; rows that see nothing: 0, -inf."""
    x = q @ k.transpose(1, 2).contiguous() / math.sqrt(D)
    x = x.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(torch.isfinite(lse), lse, 0.0)[..., None])
    return p, p @ v if v is not None else None, lse


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind in ("accept", "evict"):
        return _moved(st, kind)
    q, lens = st["q"], _lengths(case)
    if kind == "tree":
        b, n, h, r, _ = q.shape
        parents, counts = _trees(b, n, seed), _counts(case)
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        lse = torch.full((b, n, h, r), -math.inf, dtype=torch.float64, device=DEV)
        for i, (length, count) in enumerate(zip(lens, counts)):
            seen = np.zeros((n, length), bool)
            for node in range(count):
                up = node
                while up >= 0:
                    seen[node, length - n + up] = True
                    up = parents[i, up]
                seen[node, :length - n] = True
            seen = torch.from_numpy(seen[:count]).to(DEV).repeat_interleave(r, 0)
            rows = q[i, :count].double().permute(1, 0, 2, 3).reshape(h, count * r, D)
            _, y, s = _attend64(rows, _sequence(st, "k", i, length), _sequence(st, "v", i, length),
                                seen)
            out[i, :count] = y.reshape(h, count, r, D).permute(1, 0, 2, 3)
            lse[i, :count] = s.reshape(h, count, r).transpose(0, 1)
        return out, lse
    sums = st["sums"].double()
    if kind == "weigh":
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        for i, length in enumerate(lens):
            seen = torch.ones(q.shape[2], length, dtype=torch.bool, device=DEV)
            p, out[i], _ = _attend64(q[i].double(), _sequence(st, "k", i, length),
                                     _sequence(st, "v", i, length), seen)
            sums[st["rows"][i], :, :length] += p.sum(1)
        return out, sums
    for i, (length, count) in enumerate(zip(lens, _counts(case))):
        k = _sequence(st, "k", i, length).transpose(1, 2).contiguous()
        for at in range(count):
            node, end = int(st["path"][i, at]), length - count + at + 1
            x = q[i, node].double() @ k / math.sqrt(D)                     # [H, r, length]
            p = torch.exp(x - st["lse"][i, node].double()[..., None])[..., :end]
            sums[st["rows"][i], :, :end] += p.sum(1)
    return sums


def _moved(st, kind):
    """What accept and evict return: they move and choose, and compute no values."""
    case, tables = st["case"], st["tables"].long()
    rows = st["all"].flatten(2, 3)
    b = case["batch"]
    if kind == "accept":
        n = case["nodes"]
        tokens, parents, choices = (st[x].tolist() for x in ("tokens", "parents", "choices"))
        path = torch.full((b, n), -1, dtype=torch.int32)
        lengths, then = [], []
        for i in range(b):
            at, found = 0, [0]
            while True:
                child = [j for j in range(1, n) if parents[i][j] == at
                         and tokens[i][j] == choices[i][at]]
                if not child:
                    break
                at = child[0]
                found.append(at)
            path[i, :len(found)] = torch.tensor(found)
            lengths.append(len(found))
            then.append(choices[i][at])
            for j, node in enumerate(found):
                to, come = case["start"] + j, case["start"] + node
                rows[:, :, tables[i, to // PAGE] * PAGE + to % PAGE] = \
                    rows[:, :, tables[i, come // PAGE] * PAGE + come % PAGE]
        return path.to(DEV), torch.tensor(lengths, dtype=torch.int32), torch.tensor(then), st["all"]
    layers, budget, h = case["layers"], case["budget"], case["heads"]
    keep = torch.full((layers, b, h, budget), -1, dtype=torch.int32, device=DEV)
    kept = torch.zeros(layers, b, h, budget, dtype=torch.float64, device=DEV)
    for i, length in enumerate(_lengths(case)):
        pos = torch.arange(length, device=DEV)
        slot = tables[i, pos // PAGE] * PAGE + pos % PAGE
        w = st["sums"][:, i, :, :length].double()
        rank = w.clone()
        rank[..., :case["sinks"]] = math.inf
        rank[..., max(0, length - case["recent"]):] = math.inf
        got = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
        got = got.sort(-1).values                                          # [L, H, K]
        keep[:, i, :, :got.shape[-1]] = got
        kept[:, i, :, :got.shape[-1]] = w.gather(-1, got)
        for z in (0, 1):
            for head in range(h):
                of = slot[got[:, head]]                                    # [L, K]
                new = rows[:, z, :, head].gather(1, of[..., None].expand(-1, -1, D))
                rows[:, z, slot[:got.shape[-1]], head] = new
    return keep, kept, st["all"]
