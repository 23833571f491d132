"""Workloads of the operators for scores and masks of other models over a paged K/V cache, and for drafted tokens: flash_forward_paged with scores capped
by a tanh, with a bias by distance, with a prefix that all tokens see, or with a tree of drafted tokens; flash_tree_mask (masks and
positions from the parents of a tree's tokens) and flash_keep_paged (the accepted path of a tree moves to its places in the cache).

listed() names twelve of them, draw() gives more of the same ranges.  prepare() makes what a program has in hand before the
call, run() is one call.  With `own` set run() calls the package, otherwise it computes the same in elementary operations in 32 bits; exact() is
the definition in 64 bits.

Shapes: B sequences share one call.  Their new tokens lie one after the other, [T, H, d], sequence b in rows cu[b] ... cu[b + 1] - 1;
a cache is [pages, Hk, page, d] (of several layers: [layers, pages, Hk, page, d]); key j of sequence b lies in row j % page of page
table[b, j // page]; lens[b] counts the keys with the new ones, which are the last of their sequence.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# ---------------------------------------------------------------------------------------------------- cases
# forward: B, H, Hk, d, page, new (tokens of the longest chunk), old (keys in front of it in the longest cache), type,
#          cap (scores are cap * tanh(score / cap), 0: as they are), slopes (score -= slope of the head * distance), prefix (keys at the sequence's
#          begin that every token sees, 0: none), left (window, -1: none), tree (the new tokens are a tree's; otherwise causal)
# mask:    B, new: parents -> masks and positions
# keep:    B, Hk, d, page, new, old, layers, kept (tokens of the longest accepted path), type
# ragged:  sequences have lengths of their own, odd ones, up to new and old


def _forward(name, B, H, Hk, d, new, old, type, **more):
    c = {"op": "forward", "B": B, "H": H, "Hk": Hk, "d": d, "new": new, "old": old, "type": type, "page": 16, "ragged": False, "cap": 0.0, "slopes": False,
         "prefix": 0, "left": -1, "tree": False}
    return _named(name, c, more)


def _mask(name, B, new, old, **more):
    return _named(name, {"op": "mask", "B": B, "new": new, "old": old, "ragged": False}, more)


def _keep(name, B, Hk, d, new, old, layers, kept, type, **more):
    c = {"op": "keep", "B": B, "Hk": Hk, "d": d, "new": new, "old": old, "layers": layers, "kept": kept, "type": type, "page": 16, "ragged": False}
    return _named(name, c, more)


def _named(name, c, more):
    assert set(more) <= set(c)
    c.update(more)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # generation with capped scores, a full batch: the largest number of bytes read
        _forward("capped decode batch", 32, 16, 8, 128, 1, 8192, "bf16", page=64, ragged=True, cap=50.0),
        # prompts with capped scores: the largest number of operations
        _forward("capped prompts", 2, 16, 8, 128, 4096, 0, "bf16", page=32, cap=50.0),
        # a sliding-window layer with capped scores and narrow heads, chunks of prompts on what came before
        _forward("capped window d64", 3, 12, 4, 64, 1000, 2900, "fp16", ragged=True, cap=30.0, left=1023),
        # generation with a bias by distance, one K/V head per query head
        _forward("slopes decode", 8, 32, 32, 128, 1, 4001, "fp16", slopes=True),
        # prompts of several lengths with a bias by distance
        _forward("slopes prompts ragged", 6, 16, 16, 64, 2048, 0, "bf16", page=32, ragged=True, slopes=True),
        # prompts whose first part (an image, a question) all tokens see
        _forward("prefix prompts", 4, 32, 8, 128, 1531, 0, "bf16", page=128, ragged=True, prefix=1024),
        # one user's drafted tree over a cache of moderate length
        _forward("tree one", 1, 32, 8, 128, 25, 5002, "fp16", tree=True),
        # a batch of larger trees over caches of all lengths
        _forward("tree batch", 16, 32, 8, 128, 64, 4096, "bf16", page=64, ragged=True, tree=True),
        # masks of one small tree, and of a batch of the largest
        _mask("mask one", 1, 25, 5002),
        _mask("masks batch", 256, 256, 4096, ragged=True),
        # what one user's tree has left, in one layer's cache
        _keep("keep one", 1, 8, 128, 25, 5002, 1, 6, "fp16"),
        # what a batch has left, in the caches of all layers together
        _keep("keep batch", 32, 8, 128, 64, 200, 16, 12, "bf16", page=64, ragged=True),
    ]


def _size(rng, lo, hi):
    """An integer spread over the logarithm of the range, every other time a multiple of 64 where it is large enough."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if n >= 128 and rng.random() < 0.5:
        n = n // 64 * 64
    return max(lo, min(hi, n))


_DIMS = (64, 64, 128, 128, 128, 128, 32, 96, 80, 40, 72, 112)
_MOST_BYTES = {"forward": 1.0e9, "mask": 1.0e7, "keep": 2.0e8}
_MOST_FLOPS = 1.3e11
_MOST_SCORES = 1.5e9  # of the padded batch
_MOST_CACHE = 1.2e9   # elements of a cache


def draw(rng):
    while True:
        op = rng.choice(("decode", "decode", "chunk", "chunk", "prompt", "prompt", "tree", "tree", "tree", "mask", "keep", "keep"))
        d, kind = rng.choice(_DIMS), rng.choice(("fp16", "bf16"))
        hk, group = rng.choice((1, 2, 4, 8, 8, 12, 16)), rng.choice((1, 1, 2, 4, 4, 8, 5))
        pages = {"page": rng.choice((16, 16, 32, 48, 64, 128, 256)), "ragged": rng.random() < 0.7}
        if op == "mask":
            c = _mask(None, _size(rng, 1, 256), _size(rng, 1, 256), _size(rng, 1, 32768), ragged=pages["ragged"])
        elif op == "keep":
            new = _size(rng, 1, 256)
            c = _keep(None, _size(rng, 1, 64), hk, d, new, _size(rng, 1, 4096), rng.choice((1, 1, 2, 5, 16, 32)), _size(rng, 1, min(new, 32)), kind, **pages)
        else:
            scores = rng.choice(("cap", "cap", "slopes", "slopes", "both", "prefix")) if op != "tree" else rng.choice(("", "", "", "cap", "slopes", "both"))
            how = {"cap": rng.choice((20.0, 30.0, 50.0)) if scores in ("cap", "both") else 0.0, "slopes": scores in ("slopes", "both"), "tree": op == "tree"}
            if op == "decode":
                new, old = 1, _size(rng, 1, 32768)
            elif op == "chunk":
                new, old = _size(rng, 2, 2048), _size(rng, 16, 16384)
            elif op == "prompt":
                new, old = _size(rng, 16, 4096), 0
            else:
                new, old = _size(rng, 1, 256), _size(rng, 1, 32768)
            if scores == "prefix":
                how["prefix"] = _size(rng, 1, new + old)
            elif rng.random() < 0.3:
                how["left"] = _size(rng, 256, 4096)
            c = _forward(None, _size(rng, 1, 64 if op in ("decode", "tree") else 8), hk * group, hk, d, new, old, kind, **how, **pages)
        w = work(c)
        if w["bytes"] > _MOST_BYTES[c["op"]] or w["flops"] > _MOST_FLOPS:
            continue
        if c["op"] == "forward" and c["B"] * c["H"] * c["new"] * (c["new"] + c["old"] + c["page"]) > _MOST_SCORES:
            continue
        if c["op"] != "mask" and c.get("layers", 1) * c["B"] * hk * (c["new"] + c["old"] + c["page"]) * d > _MOST_CACHE / (4 if c["op"] == "keep" else 1):
            continue
        return c


# ---------------------------------------------------------------------------------------------------- inputs


def _lengths(case):
    """(new, old) tokens of each sequence: the longest first, the others, where ragged, a fixed odd mixture below."""
    B, new, old = case["B"], case["new"], case["old"]
    if not case["ragged"]:
        return [(new, old)] * B
    news = [new if b == 0 else 1 + (new - 1) * ((37 * b + 11) % 64) // 64 for b in range(B)]
    olds = [old if b == 0 else old * ((29 * b + 7) % 64) // 64 - (b % 3 if old > 64 else 0) for b in range(B)]
    return [(n, max(0, o)) for n, o in zip(news, olds)]


def _kept(case):
    """Tokens of each sequence's accepted path: from one up, at most all."""
    return [min(n, 1 + (case["kept"] - 1) * (64 - (23 * b) % 64) // 64) for b, (n, _) in enumerate(_lengths(case))]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lengths = _lengths(case)
    B, news, lens = case["B"], [n for n, _ in lengths], [n + o for n, o in lengths]
    T, most = sum(news), max(news)
    starts = [sum(news[:b]) for b in range(B + 1)]
    s = {"case": case, "most_new": most, "most_keys": max(lens), "tokens": T,
         "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "cu": torch.tensor(starts, dtype=torch.int32, device="cuda")}
    within = torch.cat([torch.arange(n) for n in news]).cuda()  # index of a token in its chunk
    if case["op"] == "mask" or case.get("tree"):
        # drafted tokens hang on one of the twelve in front of them or so, the first on the context
        back = 1 + (torch.rand(T, generator=g, device="cuda") ** 2 * 12).long()
        s["parents"] = torch.where(within == 0, -1, (within - back).clamp(min=0)).to(torch.int32)
        if case["op"] == "mask":
            return s
        s["mask"] = _plain_mask(s)[0]
    Hk, d, page, kind = case["Hk"], case["d"], case["page"], _TYPES[case["type"]]

    def normal(*shape, size=1.0):
        x = torch.randn(shape, generator=g, dtype=torch.float32, device="cuda")
        return (x * size).to(kind)

    need = [-(-n // page) for n in lens]
    width, total = max(need), sum(need) + 3
    # (pages are handed out in the order in which they came free; entries behind a sequence's last page are not set)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    table = table.cuda()
    s["table"] = torch.where(table < 0, table, order[table.long().clamp(min=0)])
    if case["op"] == "keep":
        shape = (case["layers"], total, Hk, page, d)
        s.update(k_cache=normal(*shape), v_cache=normal(*shape))
        # a path through a tree numbered level by level: its tokens' numbers grow, and lie behind those that end up in front
        counts = _kept(case)
        L = max(counts)
        path = torch.full((B, L), -1, dtype=torch.int32)
        pick = torch.rand((B, most), generator=g, device="cuda").cpu()
        for b, (n, k) in enumerate(zip(news, counts)):
            own_place = max(1, 2 * k - n)  # (of short trees the first ones stay where they are)
            rest = torch.argsort(pick[b, : n - k]) if n > k else torch.zeros(0, dtype=torch.int64)
            later = (k + rest[: k - own_place]).sort().values
            path[b, :k] = torch.cat((torch.arange(own_place), later))[:k].to(torch.int32)
        s.update(path=path.cuda(), accepted=torch.tensor(counts, dtype=torch.int32, device="cuda"))
        return s
    # (scores of models that cap them are large)
    s.update(q=normal(T, case["H"], d, size=6.0 if case["cap"] else 1.0), k_cache=normal(total, Hk, page, d), v_cache=normal(total, Hk, page, d))
    if case["slopes"]:
        H = case["H"]
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device="cuda")
    if case["prefix"]:
        s["prefix"] = torch.tensor([min(n, case["prefix"] - 5 * b % 64 if case["prefix"] > 64 else case["prefix"]) for b, n in enumerate(lens)], dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------- one pass


def run(s):
    op = s["case"]["op"]
    if own:
        return {"forward": _own_forward, "mask": _own_mask, "keep": _own_keep}[op](s)
    return {"forward": _plain_forward, "mask": _plain_mask, "keep": _plain_keep}[op](s)


def _own_forward(s):
    import flash_attn_amd as fa

    c = s["case"]
    return fa.flash_forward_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"], s["most_new"], s["most_keys"], causal=True,
                                  window=(c["left"], -1), softcap=c["cap"], alibi_slopes=s.get("slopes"), prefix_lens=s.get("prefix"),
                                  tree_mask=s.get("mask"))


def _own_mask(s):
    import flash_attn_amd as fa

    return fa.flash_tree_mask(s["parents"], s["cu"], s["lens"], s["most_new"])


def _own_keep(s):
    import flash_attn_amd as fa

    lens = fa.flash_keep_paged(s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"], s["path"], s["accepted"])
    return {"lens": lens, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _tokens(s):
    """Sequence of every new token, and its index in the chunk."""
    cu = s["cu"].long()
    t = torch.arange(s["tokens"], device=cu.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return b, t - cu[b]


def _plain_mask(s):
    """Word w of token t: which of the tokens 64 w ... 64 w + 63 of its chunk lie on its path from the root, itself among them."""
    cu, lens, most = s["cu"].long(), s["lens"].long(), s["most_new"]
    b, i = _tokens(s)
    words = (most + 63) // 64
    up = torch.where(s["parents"] >= 0, cu[b] + s["parents"].long(), -1)  # the parent's row
    on = torch.zeros((s["tokens"] + 1, words * 64), dtype=torch.bool, device=cu.device)  # (the last row: nobody's)
    on[torch.arange(s["tokens"], device=cu.device), i] = True
    up = torch.cat((up, up.new_tensor([-1])))
    for _ in range(max(1, (most - 1).bit_length())):  # paths double in length
        on = on | on[up]
        up = torch.where(up >= 0, up[up], -1)
    on = on[:-1]
    bits = torch.ones((), dtype=torch.int64, device=cu.device) << torch.arange(64, device=cu.device)
    mask = torch.where(on.view(-1, words, 64), bits, 0).sum(-1)
    depth = on.sum(-1) - 1
    return mask, (lens[b] - (cu[b + 1] - cu[b]) + depth).to(torch.int32)


def _plain_keep(s):
    page, path = s["case"]["page"], s["path"].long()
    count = (s["cu"][1:] - s["cu"][:-1]).long()
    base = s["lens"].long() - count
    i = torch.arange(path.shape[1], device=path.device)
    # a path ends where its numbers do not grow any more, or where there is no such token
    before = torch.cat((torch.full_like(path[:, :1], -1), path[:, :-1]), 1)
    good = (i < s["accepted"].long()[:, None]) & (path > before) & (path < count[:, None])
    good = good.long().cumprod(1).bool()
    b, k = good.nonzero(as_tuple=True)
    source, to = base[b] + path[b, k], base[b] + k
    table = s["table"].long()
    for c in (s["k_cache"], s["v_cache"]):
        rows = c.transpose(2, 3)  # [layers, pages, page, Hk, d]
        rows[:, table[b, to // page], to % page] = rows[:, table[b, source // page], source % page]
    return {"lens": (base + good.sum(1)).to(torch.int32), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_forward(s):
    c = s["case"]
    B, H, Hk, d, new = (c[x] for x in ("B", "H", "Hk", "d", "new"))
    G, q, table = H // Hk, s["q"], s["table"].long().clamp(min=0)
    K, V = (x[table].transpose(1, 2).reshape(B, Hk, -1, d).float() for x in (s["k_cache"], s["v_cache"]))
    cu, lens = s["cu"].long(), s["lens"].long()
    count = cu[1:] - cu[:-1]
    base = lens - count
    i, j = torch.arange(new, device=q.device), torch.arange(K.shape[2], device=q.device)
    rows = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)  # [B, new], those behind a chunk belong to others
    Q = q[rows].view(B, new, Hk, G, d).transpose(1, 2).reshape(B, Hk, new * G, d).float()
    at = base[:, None] + i  # [B, new] positions of the rows
    place = j.expand(B, -1)  # [B, keys] of the keys
    seen = (j < lens[:, None])[:, None, :].expand(B, new, -1)
    if c["tree"]:
        bit = (s["mask"][rows][..., None] >> torch.arange(64, device=q.device)) & 1
        on = bit.flatten(-2).bool()  # [B, new, 64 words]
        depth = on.sum(-1) - 1
        at = base[:, None] + depth
        drafted = (j - base[:, None]).clamp(min=0, max=new - 1)  # [B, keys]
        place = torch.where(j >= base[:, None], base[:, None] + torch.gather(depth, 1, drafted), place)
        old = (j < base[:, None])[:, None, :]
        seen = seen & (old | torch.gather(on, 2, drafted[:, None, :].expand(B, new, -1)))
    elif c["prefix"]:
        seen = seen & ((j <= at[..., None]) | (j < s["prefix"].long()[:, None])[:, None, :])
    else:
        seen = seen & (j <= at[..., None])
    distance = at[..., None] - place[:, None, :]
    if c["left"] >= 0:
        seen = seen & (distance <= c["left"])
    S = torch.matmul(Q, K.transpose(2, 3)) * d ** -0.5
    if c["cap"]:
        S = torch.tanh(S.div_(c["cap"])).mul_(c["cap"])
    S = S.view(B, Hk, new, G, -1)
    if c["slopes"]:
        S -= distance.abs().float()[:, None, :, None, :] * s["slopes"].view(Hk, 1, G, 1)
    S = S.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = S.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    S = S.sub_(m).exp_()
    total = S.sum(-1)
    O = torch.matmul(S.view(B, Hk, new * G, -1), V).view(B, Hk, new, G, d)
    O = O / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    L = m[..., 0] + total.log()
    b, i = _tokens(s)
    return O[b, :, i].reshape(-1, H, d).to(q.dtype), L[b, :, i].reshape(-1, H)


# ---------------------------------------------------------------------------------------------------- in 64 bits


def _ancestors(parents):
    """Of one chunk: the set of each token's path, as a whole number's bits."""
    paths = []
    for i, p in enumerate(parents):
        paths.append((paths[p] if p >= 0 else 0) | 1 << i)
    return paths


def exact(case, seed):
    s = prepare(case, seed)
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    B, top = case["B"], 1 << 64
    if case["op"] == "mask":
        words, parents = (case["new"] + 63) // 64, s["parents"].tolist()
        mask, positions = [], []
        for b in range(B):
            for x in _ancestors(parents[cu[b] : cu[b + 1]]):
                row = [(x >> 64 * w) % top for w in range(words)]
                mask.append([v - top if v >= top // 2 else v for v in row])
                positions.append(lens[b] - (cu[b + 1] - cu[b]) + bin(x).count("1") - 1)
        return torch.tensor(mask, dtype=torch.int64, device="cuda"), torch.tensor(positions, dtype=torch.int32, device="cuda")
    page, table = case["page"], s["table"].tolist()
    if case["op"] == "keep":
        path, accepted, after = s["path"].tolist(), s["accepted"].tolist(), []
        out = {"k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
        for b in range(B):
            base = lens[b] - (cu[b + 1] - cu[b])
            where = [(table[b][(base + x) // page], (base + x) % page) for x in range(cu[b + 1] - cu[b])]
            for to, x in enumerate(path[b][: accepted[b]]):
                for name in ("k_cache", "v_cache"):
                    out[name][:, where[to][0], :, where[to][1]] = s[name][:, where[x][0], :, where[x][1]].double()
            after.append(base + accepted[b])
        return {"lens": torch.tensor(after, dtype=torch.int32, device="cuda"), **out}
    H, Hk, d = (case[x] for x in ("H", "Hk", "d"))
    O = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    L = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        m = cu[b + 1] - cu[b]
        used = torch.tensor(table[b][: -(-n // page)], device="cuda")
        keys, rows = torch.arange(n, device="cuda"), torch.arange(n - m, n, device="cuda")
        hidden = keys[None, :] > rows[:, None]
        if case["prefix"]:
            hidden[:, : int(s["prefix"][b])] = False
        if case["tree"]:
            paths = _ancestors(s["parents"][cu[b] : cu[b + 1]].tolist())
            on = torch.tensor([[x >> y & 1 for y in range(m)] for x in paths], device="cuda").bool()
            hidden[:, n - m :] = ~on
            rows = n - m + on.sum(1) - 1
            keys = torch.cat((keys[: n - m], rows))
        apart = (rows[:, None] - keys[None, :]).double()
        if case["left"] >= 0:
            hidden |= apart > case["left"]
        for h in range(Hk):
            G = H // Hk
            heads = slice(h * G, (h + 1) * G)
            k, v = (x[used, h].reshape(-1, d)[:n].double() for x in (s["k_cache"], s["v_cache"]))
            q = s["q"][cu[b] : cu[b + 1], heads].double()
            score = torch.tensordot(q, k, dims=([2], [1])) / math.sqrt(d)
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            if case["slopes"]:
                score = score - apart.abs()[:, None, :] * s["slopes"][heads].double()[None, :, None]
            score.masked_fill_(hidden[:, None, :], -math.inf)
            L[cu[b] : cu[b + 1], heads] = torch.logsumexp(score, -1)
            O[cu[b] : cu[b + 1], heads] = torch.tensordot(torch.softmax(score, -1).nan_to_num_(0.0), v, dims=([2], [0]))
    return O, L


# ---------------------------------------------------------------------------------------------------- work


def work(case):
    B, lengths = case["B"], _lengths(case)
    T = sum(n for n, _ in lengths)
    if case["op"] == "mask":
        words = (case["new"] + 63) // 64
        return {"bytes": 4 * T + 4 * (2 * B + 1) + 8 * T * words + 4 * T, "flops": T * words}
    Hk, d, page = case["Hk"], case["d"], case["page"]
    if case["op"] == "keep":
        counts = _kept(case)
        moved = sum(k - max(1, 2 * k - n) for k, (n, _) in zip(counts, lengths))  # (the others stay where they are)
        return {"bytes": 2 * 2 * 2 * moved * Hk * d * case["layers"] + 4 * (B * max(counts) + 4 * B + 1), "flops": max(1, moved)}
    H, cap, left, prefix = case["H"], case["cap"], case["left"], case["prefix"]
    keys = pairs = 0
    for b, (n, o) in enumerate(lengths):
        back = left if left >= 0 else n + o
        ahead = min(n + o, prefix - 5 * b % 64 if prefix > 64 else prefix)
        keys += n + o - max(0, o - back)  # that some row sees
        if case["tree"]:
            pairs += n * min(o, back) + n * min(n, 8)  # (paths of some eight tokens)
        else:
            for i in range(o, o + n):
                pairs += max(i + 1, ahead) - max(0, i - back)
    table = sum(-(-(n + o) // page) for n, o in lengths)
    each = 4 * d + (4 if cap else 0) + (2 if case["slopes"] else 0)
    extra = (4 * H if case["slopes"] else 0) + (4 * B if prefix else 0) + (8 * T * ((case["new"] + 63) // 64) if case["tree"] else 0)
    return {"bytes": 2 * (2 * T * H * d + 2 * keys * Hk * d) + 4 * (T * H + table + 2 * B) + extra, "flops": each * H * pairs}
