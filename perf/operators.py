"""The operators of branching generation over a 4-bit cache, measured.

A serving program that samples several continuations of one long prompt keeps
the prompt's K and V in 4 bits, branches a sequence by copying the page it
ends in, and ranks the branches by their tokens' log probabilities:

store    K and V of new tokens quantized into the 4-bit pools at their slots,
         and rows of the pools read back as values
attend   one decode step's attention over 4-bit pools
copy     pages copied to other pages of the same pools, all layers together
score    log probability of a given token a row, the row's entropy, its most
         likely tokens

The 4-bit entry of a token: per KV head, each group of 32 adjacent channels has
a minimum m and a step s = fp16((max - m) / 15) (difference and quotient in
fp32; the values here are far from fp16's largest, where the next smaller s is
taken if m + 15 s would pass it), both fp16; a channel's code is the whole number
nearest to (x - m) / s (ties to even), kept in 0..15 (0 where s is 0), and it
stands for fp16(m + s * code).  The pools (nb pages of 16 tokens, H heads, 128 channels):

k_codes   uint8 [nb, H, 16, 64]     a token's row: 16 words of 8 codes, word
                                    4 g + j the channels 32 j + 8 g + (0..7)
k_affine  fp16  [nb, H, 16, 4, 2]   (s, m) of each token and group
v_codes   uint8 [nb, H, 16, 16, 4]  word (o, t): channels 8 o + (0..7) of token t
v_affine  fp16  [nb, H, 4, 4, 2, 4] s, then m, of tokens 4 a + (0..3), by
                                    group and a

Code i of a word is its bits 4 i .. 4 i + 3 (little endian).
"""

from __future__ import annotations

import math

import torch

own = False

PAGE, D, GROUP = 16, 128, 32
DEV = "cuda"


def listed():
    return [
        # one chat at a short context: launch and latency count
        dict(name="attend b1 2k", kind="attend", batch=1, ctx=2048, ragged=False, heads=2, n_rep=6),
        # the repository's headline batch and context
        dict(name="attend b16 16k", kind="attend", batch=16, ctx=16384, ragged=False, heads=2,
             n_rep=6),
        # a busy server: many short chats of all lengths, wider KV
        dict(name="attend b48 ragged 1.5k", kind="attend", batch=48, ctx=1531, ragged=True, heads=8,
             n_rep=4),
        # two long documents: few rows, a long axis to split
        dict(name="attend b2 100k", kind="attend", batch=2, ctx=100003, ragged=False, heads=2,
             n_rep=6),
        # a decode step's token of each of 16 sequences, in the middle of their pages
        dict(name="store b16 tokens", kind="store", batch=16, tokens=1, start=8197, heads=2,
             back=16),
        # four prompts of 2048 tokens, read back for the next chunk's attention
        dict(name="store b4 x 2048", kind="store", batch=4, tokens=2048, start=0, heads=2,
             back=2048),
        # the odd last chunk of one prompt, wider KV, behind 1003 tokens that are there
        dict(name="store b1 x 1021 at 1003", kind="store", batch=1, tokens=1021, start=1003,
             heads=8, back=2024),
        # one sequence branched into eight: the page it ends in, all layers' K and V
        dict(name="copy 8 branches", kind="copy", pages=8, branch=True, layers=28, heads=2,
             blocks=512),
        # pages moved down together after many sequences ended
        dict(name="copy 160 pages", kind="copy", pages=160, branch=False, layers=28, heads=2,
             blocks=512),
        # a decode step's chosen tokens with their alternatives
        dict(name="score b16 top 20", kind="score", rows=16, vocab=151936, top=20, dtype="float16"),
        # a prompt's tokens scored, no alternatives
        dict(name="score 1021 rows", kind="score", rows=1021, vocab=151936, top=0, dtype="float16"),
        # one row of processed logits in fp32, an odd vocabulary
        dict(name="score 1 row fp32", kind="score", rows=1, vocab=32003, top=5, dtype="float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "store", "copy", "score", "score"])
    if kind == "attend":
        heads, batch = rng.choice([1, 2, 3, 4, 8]), _log(rng, 1, 96)
        ctx = _log(rng, 1, max(1, min(100003, 16 * 16384 * 2 // (heads * batch))))
        return dict(kind=kind, batch=batch, ctx=ctx, ragged=rng.random() < 0.6, heads=heads,
                    n_rep=rng.choice([1, 2, 4, 6, 7, 8, 16]))
    if kind == "store":
        heads, batch = rng.choice([1, 2, 3, 8]), _log(rng, 1, 48)
        tokens = _log(rng, 1, max(1, 16384 // (heads * batch)))
        start = rng.randrange(0, 1200)
        back = PAGE if tokens == 1 else start + tokens
        return dict(kind=kind, batch=batch, tokens=tokens, start=start, heads=heads, back=back)
    if kind == "copy":
        pages = _log(rng, 1, 160)
        return dict(kind=kind, pages=pages, branch=rng.random() < 0.4, layers=_log(rng, 1, 28),
                    heads=rng.choice([1, 2]), blocks=2 * pages + rng.randrange(0, 100))
    top = rng.choice([0, 1, 5, 20, 32])
    return dict(kind=kind, rows=_log(rng, 1, 1021 if top == 0 else 128), vocab=_log(rng, 1000, 151936),
                top=top, dtype=rng.choice(["float16", "float16", "float32"]) if top else "float16")


def _lengths(case):
    """Lengths of an attend case's sequences: all ctx, or spread over 1..ctx
    (deterministic: they are the case's)."""
    b, ctx = case["batch"], case["ctx"]
    if not case["ragged"] or b == 1:
        return [ctx] * b
    return [1 + (ctx - 1) * ((5 * i + 3) % b) // (b - 1) for i in range(b)]


def work(case):
    kind = case["kind"]
    if kind == "attend":
        toks = sum(_lengths(case)) * case["heads"]
        rows = case["batch"] * case["heads"] * case["n_rep"]
        return {"bytes": toks * 160 + rows * D * 2 * 2, "flops": toks * case["n_rep"] * D * 4}
    if kind == "store":
        new = case["batch"] * case["tokens"] * case["heads"]
        back = case["batch"] * _window(case)[1] * case["heads"]
        rows = case["batch"] * case["back"] * case["heads"]
        return {"bytes": new * (2 * D * 2 + 160) + back * 160 + rows * 2 * D * 2,
                "flops": new * 2 * D * 5 + back * 2 * D * 2}
    if kind == "copy":
        pages = case["pages"] + (1 if case["branch"] else case["pages"])
        return {"bytes": pages * case["layers"] * 2 * PAGE * case["heads"] * D * 2,
                "flops": 0}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (2 if case["dtype"] == "float16" else 4) + case["rows"] * (12 + 12 * case["top"]),
            "flops": 5 * n}


def _window(case):
    """Of a store case: the first page read back, and the tokens read."""
    end = case["start"] + case["tokens"]
    first = (end - 1) // PAGE if case["back"] == PAGE else 0
    return first, end - first * PAGE


def _pools(nb, heads, gen):
    """Pools as some time of serving leaves them: codes of all values, steps
    and minima of keys and values around unit size."""
    def codes(*shape):
        return torch.randint(0, 256, shape, generator=gen, device=DEV, dtype=torch.uint8)

    def step(*shape):
        return 0.15 + 0.25 * torch.rand(*shape, generator=gen, device=DEV)

    ks, vs = step(nb, heads, PAGE, 4), step(nb, heads, 4, 4, 4)
    km = -7.5 * ks + 0.3 * torch.randn(ks.shape, generator=gen, device=DEV)
    vm = -7.5 * vs + 0.3 * torch.randn(vs.shape, generator=gen, device=DEV)
    return (codes(nb, heads, PAGE, 64), torch.stack((ks, km), -1).half().contiguous(),
            codes(nb, heads, 16, PAGE, 4), torch.stack((vs, vm), -2).half().contiguous())


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, st = case["kind"], {"case": case}
    if own:
        from latentserve_amd.kernels import logprobs
        from latentserve_amd.kernels.hip import int4_cache, page_copy
        st.update(cache4=int4_cache, pages=page_copy, scores=logprobs)
    if kind == "attend":
        b, h, lens = case["batch"], case["heads"], _lengths(case)
        width = -(-max(lens) // PAGE)
        nb = b * width + 7
        st["pools"] = _pools(nb, h, gen)
        st["tables"] = torch.randperm(nb, generator=gen, device=DEV)[:b * width] \
            .view(b, width).to(torch.int32)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["q"] = torch.randn(b, h, case["n_rep"], D, generator=gen, device=DEV).half()
        st["longest"] = max(lens)
    elif kind == "store":
        b, h, n, start = case["batch"], case["heads"], case["tokens"], case["start"]
        width = -(-(start + n) // PAGE)
        nb = b * width + 5
        st["pools"] = _pools(nb, h, gen)
        tables = torch.randperm(nb, generator=gen, device=DEV)[:b * width].view(b, width)
        pos = torch.arange(start, start + n, device=DEV)
        st["slots"] = (tables[:, pos // PAGE] * PAGE + pos % PAGE).reshape(-1)
        first, live = _window(case)
        st["tables"] = tables[:, first:].to(torch.int32).contiguous()
        st["lens"] = torch.full((b,), live, dtype=torch.int32, device=DEV)
        # k and v as views of one projection's output, a few channels larger than the rest
        x = torch.randn(b, n, 2 * h, D, generator=gen, device=DEV)
        x[..., ::37] *= 4
        x = x.half()
        st["k"], st["v"] = x[:, :, :h].transpose(1, 2), x[:, :, h:].transpose(1, 2)
    elif kind == "copy":
        nb, p = case["blocks"], case["pages"]
        st["all"] = torch.randn(case["layers"], 2, nb, PAGE, case["heads"], D, generator=gen,
                                device=DEV, dtype=torch.float16)
        st["tensors"] = [t for layer in st["all"] for t in layer]
        ids = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).tolist()
        st["src"], st["dst"] = ids[:1] * p if case["branch"] else ids[:p], ids[p:2 * p]
    else:
        r, v = case["rows"], case["vocab"]
        x = 2.5 * torch.randn(r, v, generator=gen, device=DEV)
        best = torch.randint(0, v, (r, 8), generator=gen, device=DEV)
        x.scatter_add_(1, best, 8 * torch.rand(r, 8, generator=gen, device=DEV))
        st["logits"] = x.to(getattr(torch, case["dtype"]))
        st["tokens"] = best[:, 0].contiguous()
    return st


def run(state):
    return _RUN[state["case"]["kind"]](state)


# ---- store ---------------------------------------------------------------------


def _words(codes):
    """Codes [..., 8 n] as bytes [..., 4 n]."""
    c = codes.to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _codes(words):
    """Bytes [..., n] as their codes [..., 2 n]."""
    return torch.stack((words & 15, words >> 4), -1).flatten(-2)


def _k_values(codes, affine):
    """[..., 16, 64] and [..., 16, 4, 2] -> [..., 16, 128] fp16."""
    c = _codes(codes).unflatten(-1, (4, 4, 8)).transpose(-3, -2).flatten(-3).unflatten(-1, (4, GROUP))
    a = affine.float()
    return (a[..., 1:] + a[..., :1] * c.float()).half().flatten(-2)


def _v_values(codes, affine):
    """[..., 16, 16, 4] and [..., 4, 4, 2, 4] -> [..., 16, 128] fp16."""
    c = _codes(codes).transpose(-3, -2).flatten(-2).unflatten(-1, (4, GROUP))
    a = affine.float().transpose(-2, -1).flatten(-3, -2).transpose(-3, -2)     # [..., 16, 4, 2]
    return (a[..., 1:] + a[..., :1] * c.float()).half().flatten(-2)


def _quantize(x):
    """[..., 128] fp16 -> codes [..., 128], (s, m) [..., 4, 2] fp16."""
    g = x.unflatten(-1, (4, GROUP)).float()
    lo = g.amin(-1, keepdim=True)
    s = ((g.amax(-1, keepdim=True) - lo) / 15).half()
    # (64 bits: values next to a border between two codes)
    c = torch.round((g.double() - lo.double()) / s.double()).clamp(0, 15)
    c = torch.where(s == 0, torch.zeros_like(c), c)
    return c.flatten(-2), torch.cat((s, lo.half()), -1)


def _store(st):
    case = st["case"]
    if own:
        st["cache4"].write(st["k"], st["v"], st["slots"], st["pools"])
        return st["cache4"].read(st["pools"], st["tables"], st["lens"], case["back"])
    k_codes, k_affine, v_codes, v_affine = st["pools"]
    blk, t = st["slots"] // PAGE, st["slots"] % PAGE
    kc, ka = _quantize(st["k"].transpose(1, 2).flatten(0, 1))              # [tokens, H, ...]
    vc, va = _quantize(st["v"].transpose(1, 2).flatten(0, 1))
    k_codes[blk, :, t] = _words(kc.unflatten(-1, (4, 4, 8)).transpose(-3, -2).flatten(-3))
    k_affine[blk, :, t] = ka
    v_codes[blk, :, :, t] = _words(vc.unflatten(-1, (16, 8)))
    v_affine[blk, :, :, t // 4, :, t % 4] = va
    tab = st["tables"].long()
    out = []
    for values, codes, affine in ((_k_values, k_codes, k_affine), (_v_values, v_codes, v_affine)):
        x = values(codes[tab], affine[tab])                                # [B, P, H, 16, D]
        x = x.transpose(1, 2).flatten(2, 3)[:, :, :case["back"]]
        live = torch.arange(x.shape[2], device=x.device) < st["lens"][:, None]
        out.append(torch.where(live[:, None, :, None], x, torch.zeros_like(x)))
    return tuple(out)


# ---- attend --------------------------------------------------------------------


def _attend(st):
    if own:
        return st["cache4"].paged_decode_int4(st["q"], st["pools"], st["tables"], st["lens"],
                                              st["longest"])
    tab = st["tables"].long()
    k_codes, k_affine, v_codes, v_affine = st["pools"]
    k = _k_values(k_codes[tab], k_affine[tab]).transpose(1, 2).flatten(2, 3).float()  # [B, H, T, D]
    x = torch.matmul(st["q"].float(), k.transpose(2, 3)) / math.sqrt(D)
    del k
    live = torch.arange(x.shape[-1], device=x.device) < st["lens"][:, None]
    live = live[:, None, None, :]
    x = torch.where(live, x, torch.full_like(x, -math.inf))
    p = torch.where(live, torch.exp(x - x.amax(-1, keepdim=True)), torch.zeros_like(x))
    v = _v_values(v_codes[tab], v_affine[tab]).transpose(1, 2).flatten(2, 3).float()
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-20)).half()


# ---- copy ----------------------------------------------------------------------


def _copy(st):
    if own:
        st["pages"].copy_pages(st["tensors"], st["src"], st["dst"])
        return st["all"]
    ids = torch.tensor([st["src"], st["dst"]], device=DEV)
    for t in st["tensors"]:
        t[ids[1]] = t[ids[0]]
    return st["all"]


# ---- score ---------------------------------------------------------------------


def _score(st):
    top = st["case"]["top"]
    if own:
        return tuple(x for x in st["scores"].token_logprobs(st["logits"], st["tokens"], top)
                     if x is not None)
    x = st["logits"].float()
    best = x.amax(-1, keepdim=True)
    e = torch.exp(x - best)
    z = e.sum(-1, keepdim=True)
    lse = best + torch.log(z)
    out = [(x.gather(1, st["tokens"][:, None]) - lse)[:, 0],
           (torch.log(z) - (e * (x - best)).sum(-1, keepdim=True) / z)[:, 0]]
    if top:
        # value first, then the lower index: one whole number a token
        bits = x.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        index = torch.arange(x.shape[1], device=x.device)
        key = torch.topk(order * (1 << 24) + (x.shape[1] - 1 - index), top, dim=-1).values
        ids = x.shape[1] - 1 - (key & ((1 << 24) - 1))
        out += [x.gather(1, ids) - lse, ids]
    return tuple(out)


_RUN = {"store": _store, "attend": _attend, "copy": _copy, "score": _score}


# ---- 64 bits, from the definitions ------------------------------------------------


def _entry64(codes, affine, value, blk, t):
    """Value of pool rows (page blk[i], token t[i]): [n, H, 128] in 64 bits."""
    c = torch.arange(D, device=blk.device)
    word = 4 * (c // 8 % 4) + c // 32 if not value else c // 8
    byte, shift = c % 8 // 2, c % 2 * 4
    rows = codes[blk].long()                                               # [n, H, ...]
    n, i = blk.shape[0], torch.arange(blk.shape[0], device=blk.device)[:, None]
    if value:
        raw = rows[i, :, word[None], t[:, None], byte[None]]               # [n, 128, H]
        s, m = (affine[blk].double()[i, :, c[None] // 32, t[:, None] // 4, z, t[:, None] % 4]
                for z in (0, 1))
    else:
        raw = rows[i, :, t[:, None], (4 * word + byte)[None]]
        s, m = (affine[blk].double()[i, :, t[:, None], c[None] // 32, z] for z in (0, 1))
    code = (raw >> shift[None, :, None]) & 15
    return (m + s * code).half().double().transpose(1, 2)


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "copy":
        y = st["all"]
        for a, b in zip(st["src"], st["dst"]):
            y[:, :, b] = y[:, :, a]
        return y
    if kind == "score":
        x = st["logits"].double()
        lse = torch.logsumexp(x, -1, keepdim=True)
        logp = x - lse
        out = [logp.gather(1, st["tokens"][:, None])[:, 0], -(logp.exp() * logp).sum(-1)]
        if case["top"]:
            val, ids = torch.sort(x, dim=-1, descending=True, stable=True)
            out += [val[:, :case["top"]] - lse, ids[:, :case["top"]].contiguous()]
        return tuple(out)
    k_codes, k_affine, v_codes, v_affine = st["pools"]
    if kind == "attend":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
        for b, length in enumerate(_lengths(case)):
            pos = torch.arange(length, device=DEV)
            blk, t = st["tables"][b].long()[pos // PAGE], pos % PAGE
            acc = []
            for lo in range(0, length, 8192):           # keys, in pieces
                acc.append(_entry64(k_codes, k_affine, False, blk[lo:lo + 8192], t[lo:lo + 8192]))
            k = torch.cat(acc).transpose(0, 1)                             # [H, T, D]
            x = st["q"][b].double() @ k.transpose(1, 2).contiguous() / math.sqrt(D)
            p = torch.softmax(x, -1)
            for lo in range(0, length, 8192):
                v = _entry64(v_codes, v_affine, True, blk[lo:lo + 8192], t[lo:lo + 8192])
                out[b] += p[:, :, lo:lo + 8192].contiguous() @ v.transpose(0, 1).contiguous()
        return out
    # store: what is read back is the new tokens' entries where they were written,
    # the pools' elsewhere
    first, live = _window(case)
    b, h, n = case["batch"], case["heads"], case["tokens"]
    out = []
    for z, (codes, affine, new) in enumerate(((k_codes, k_affine, st["k"]),
                                              (v_codes, v_affine, st["v"]))):
        y = torch.zeros(b, h, case["back"], D, dtype=torch.float64, device=DEV)
        pos = torch.arange(live, device=DEV)
        for i in range(b):
            y[i, :, :live] = _entry64(codes, affine, z == 1, st["tables"][i].long()[pos // PAGE],
                                      pos % PAGE).transpose(0, 1)
        g = new.double().reshape(b, h, n, 4, GROUP)
        lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        s = ((hi.float() - lo.float()) / 15).half().double()
        code = torch.where(s > 0, torch.round((g - lo) / torch.where(s > 0, s, 1.0)), 0.0)
        val = (lo + s * code.clamp(0, 15)).half().double().reshape(b, h, n, D)
        at = case["start"] - first * PAGE
        y[:, :, at:at + n] = val
        out.append(y)
    return tuple(out)
