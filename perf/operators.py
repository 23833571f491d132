"""Workloads of the operators around a paged K/V cache: flash_rotary (rotary positions and their gradient),
flash_append_paged (new tokens into the pages, rotated on the way) and flash_forward_paged (attention of a chunk of new
tokens, down to a single one per sequence, over the pages).

listed() names twelve of them, draw() gives more of the same ranges.  prepare() makes what a program has in hand before the
call, run() is one call.  With `own` set run() calls the package, otherwise it computes the same in elementary operations in
32 bits (angles in 64); exact() is the definition in 64 bits.

Shapes: B sequences share one call.  Their new tokens lie one after the other, [T, H, d], sequence b in rows cu[b] ... cu[b + 1] - 1;
a cache is [pages, Hk, page, d]; key j of sequence b lies in row j % page of page table[b, j // page]; lens[b] counts the keys
with the new ones, which are the last of their sequence.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}

# ---------------------------------------------------------------------------------------------------- cases
# rotary: B, H, N, d, order ("bhnd": heads first in memory, "bnhd": as a projection leaves them), rot (leading elements of a head that
#         turn), first (position of the first row), stretch (factor by which frequencies are lowered for long contexts), factor
#         (of the outputs), interleaved, inverse (the gradient), type
# append: B, H, Hk, d, page, new (tokens of the longest chunk), old (keys in the longest cache), rot (0: stored as they are), ...
# forward: B, H, Hk, d, page, new, old, causal, left (window, -1: none), type
# ragged: sequences have lengths of their own, odd ones, up to new and old


def _rotary(name, B, H, N, d, type, **more):
    c = {"op": "rotary", "B": B, "H": H, "N": N, "d": d, "type": type, "order": "bnhd", "rot": d, "first": 0, "stretch": 1.0, "factor": 1.0,
         "interleaved": False, "inverse": False}
    return _named(name, c, more)


def _append(name, B, H, Hk, d, new, old, type, **more):
    c = {"op": "append", "B": B, "H": H, "Hk": Hk, "d": d, "new": new, "old": old, "type": type, "page": 16, "ragged": False, "rot": d,
         "interleaved": False, "stretch": 1.0, "factor": 1.0}
    return _named(name, c, more)


def _forward(name, B, H, Hk, d, new, old, type, **more):
    c = {"op": "forward", "B": B, "H": H, "Hk": Hk, "d": d, "new": new, "old": old, "type": type, "page": 16, "ragged": False, "causal": True,
         "left": -1}
    return _named(name, c, more)


def _named(name, c, more):
    assert set(more) <= set(c)
    c.update(more)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # generation, one user: the queries of one token
        _rotary("rotate one token", 1, 32, 1, 128, "fp16", first=4095),
        # prompts of odd length, neighbours in pairs, the leading part of narrow heads
        _rotary("rotate part d80", 3, 12, 1777, 80, "bf16", rot=32, interleaved=True),
        # a training step's gradient with stretched positions, the largest of its kind
        _rotary("rotate gradient d128", 4, 32, 4096, 128, "bf16", first=1000003, stretch=8.0, factor=1.2, inverse=True),
        # generation, a full batch: one token per sequence into the pages
        _append("append decode", 64, 32, 8, 128, 1, 8000, "fp16", ragged=True),
        # prompts of several lengths arrive together, neighbours in pairs
        _append("append ragged d64", 5, 16, 4, 64, 1021, 900, "bf16", page=32, ragged=True, interleaved=True),
        # a long prompt in one piece, the largest number of bytes written
        _append("append prompt", 2, 32, 8, 128, 8192, 0, "bf16", page=64),
        # generation, one user, a cache of moderate length that ends in the middle of a page
        _forward("decode one", 1, 32, 8, 128, 1, 5002, "fp16"),
        # generation, a full batch with long caches of all lengths: the largest number of bytes read
        _forward("decode batch", 64, 32, 8, 128, 1, 16384, "bf16", page=64, ragged=True),
        # generation with one K/V head per query head and narrow heads
        _forward("decode heads d64", 16, 16, 16, 64, 1, 4096, "fp16", page=128),
        # a chunk of a prompt against the pages of what came before
        _forward("chunk on pages", 1, 32, 8, 128, 512, 16384, "bf16"),
        # prompts of several lengths in one call: the largest number of operations
        _forward("prompts ragged", 4, 32, 4, 128, 4096, 0, "fp16", page=32, ragged=True),
        # a sliding-window layer with a head dimension between the powers of two
        _forward("window chunk d80", 3, 12, 12, 80, 1777, 2048, "bf16", left=512),
    ]


def _size(rng, lo, hi):
    """An integer spread over the logarithm of the range, every other time a multiple of 64 where it is large enough."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if n >= 128 and rng.random() < 0.5:
        n = n // 64 * 64
    return max(lo, min(hi, n))


_DIMS = (64, 64, 128, 128, 128, 128, 32, 96, 80, 40, 72, 112)
_MOST_BYTES = {"rotary": 2.6e8, "append": 4.0e8, "forward": 2.0e9}
_MOST_FLOPS = 4.0e11
_MOST_SCORES = 2.1e9  # of the padded batch


def draw(rng):
    while True:
        op = rng.choice(("rotary", "append", "decode", "decode", "chunk", "chunk", "prompt"))
        d, kind = rng.choice(_DIMS), rng.choice(("fp16", "bf16"))
        hk, group = rng.choice((1, 2, 4, 8, 8, 12, 16)), rng.choice((1, 1, 2, 4, 4, 8, 5))
        H = hk * group
        turn = {"rot": rng.choice((d, d, d // 2 // 8 * 8 or 8)), "interleaved": rng.random() < 0.4, "stretch": rng.choice((1.0, 1.0, 4.0, 16.0)),
                "factor": rng.choice((1.0, 1.0, 1.1386))}
        pages = {"page": rng.choice((16, 16, 32, 48, 64, 128, 256)), "ragged": rng.random() < 0.7}
        if op == "rotary":
            c = _rotary(None, _size(rng, 1, 16), H, _size(rng, 1, 8192), d, rng.choice((kind, kind, "fp32")), order=rng.choice(("bnhd", "bhnd")),
                        first=rng.choice((0, 0, _size(rng, 1, 2000000))), inverse=rng.random() < 0.4, **turn)
        elif op == "append":
            if rng.random() < 0.2:
                turn["rot"] = 0
            c = _append(None, _size(rng, 1, 64), H, hk, d, rng.choice((1, _size(rng, 1, 8192))), rng.choice((0, _size(rng, 1, 16384))), kind, **turn, **pages)
        elif op == "decode":
            c = _forward(None, _size(rng, 1, 64), H, hk, d, 1, _size(rng, 1, 32768), kind, **pages)
        elif op == "chunk":
            c = _forward(None, _size(rng, 1, 8), H, hk, d, _size(rng, 2, 2048), _size(rng, 16, 32768), kind, left=rng.choice((-1, -1, _size(rng, 16, 4096))),
                         **pages)
        else:
            c = _forward(None, _size(rng, 1, 8), H, hk, d, _size(rng, 16, 4096), 0, kind, causal=rng.random() < 0.8, **pages)
        w = work(c)
        if w["bytes"] > _MOST_BYTES[c["op"]] or w["flops"] > _MOST_FLOPS:
            continue
        if c["op"] == "forward" and c["B"] * H * c["new"] * (c["new"] + c["old"] + c["page"]) > _MOST_SCORES:
            continue
        if c["op"] != "rotary" and c["B"] * hk * (c["new"] + c["old"] + c["page"]) * d > 1.2e9:  # elements of a cache
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


def _frequencies(rot, stretch, device):
    i = torch.arange(rot // 2, dtype=torch.float64)
    return (10000.0 ** (-2.0 * i / rot) / stretch).float().to(device)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, dtype=torch.float32, device="cuda").to(kind)

    s = {"case": case}
    if case["op"] == "rotary":
        B, H, N, d = (case[x] for x in ("B", "H", "N", "d"))
        s["x"] = normal(B, H, N, d) if case["order"] == "bhnd" else normal(B, N, H, d).transpose(1, 2)
        s["positions"] = case["first"] + torch.arange(N, device="cuda")
        s["inv_freq"] = _frequencies(case["rot"], case["stretch"], "cuda")
        return s
    B, H, Hk, d, page = (case[x] for x in ("B", "H", "Hk", "d", "page"))
    lengths = _lengths(case)
    T, lens = sum(n for n, _ in lengths), [n + o for n, o in lengths]
    need = [-(-n // page) for n in lens]
    width, total = max(need), sum(need) + 3
    # (pages are handed out in the order in which they came free; entries behind a sequence's last page are not set)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    where = torch.zeros((B, width), dtype=torch.int64)
    for b, n in enumerate(need):
        where[b, :n] = torch.arange(at, at + n)
        table[b, :n] = 0
        at += n
    table = torch.where(table.cuda() < 0, table.cuda(), order[where.cuda()])
    s.update(q=normal(T, H, d), k_cache=normal(total, Hk, page, d), v_cache=normal(total, Hk, page, d), table=table,
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             cu=torch.tensor([0] + [sum(n for n, _ in lengths[: b + 1]) for b in range(B)], dtype=torch.int32, device="cuda"),
             most_new=max(n for n, _ in lengths), most_keys=max(lens))
    if case["op"] == "append":
        s.update(k=normal(T, Hk, d), v=normal(T, Hk, d), inv_freq=_frequencies(case["rot"], case["stretch"], "cuda") if case["rot"] else None)
    return s


# ---------------------------------------------------------------------------------------------------- one pass


def run(s):
    op = s["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "append": _own_append, "forward": _own_forward}[op](s)
    return {"rotary": _plain_rotary, "append": _plain_append, "forward": _plain_forward}[op](s)


def _own_rotary(s):
    import flash_attn_amd as fa

    c = s["case"]
    return fa.flash_rotary(s["x"], s["positions"], s["inv_freq"], interleaved=c["interleaved"], factor=c["factor"], inverse=c["inverse"])


def _own_append(s):
    import flash_attn_amd as fa

    c = s["case"]
    if c["rot"] == 0:
        fa.flash_append_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    q = fa.flash_append_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"], q=s["q"], inv_freq=s["inv_freq"],
                              interleaved=c["interleaved"], factor=c["factor"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_forward(s):
    import flash_attn_amd as fa

    c = s["case"]
    return fa.flash_forward_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"], s["most_new"], s["most_keys"],
                                  causal=c["causal"], window=(c["left"], -1))


def _turn(x, positions, inv_freq, interleaved, factor, inverse=False):
    """x [..., d] turned by positions [...] (broadcast), in 32 bits, rounded once."""
    rot = 2 * inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq.double()
    cos, sin = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()
    if inverse:
        sin = -sin
    y = x.float()
    part, rest = y[..., :rot], y[..., rot:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = part[..., : rot // 2], part[..., rot // 2 :]
        part = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((part, rest), -1).to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    return _turn(s["x"], s["positions"], s["inv_freq"], c["interleaved"], c["factor"], c["inverse"])


def _tokens(s):
    """Sequence, row within the chunk and position of every new token."""
    cu, lens = s["cu"].long(), s["lens"].long()
    t = torch.arange(s["q"].shape[0], device=cu.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    i = t - cu[b]
    return b, i, lens[b] - (cu[b + 1] - cu[b]) + i


def _plain_append(s):
    c = s["case"]
    b, _, position = _tokens(s)
    page = c["page"]
    at, row = s["table"].long()[b, position // page], position % page
    k, q = s["k"], None
    if c["rot"]:
        k = _turn(k, position[:, None], s["inv_freq"], c["interleaved"], c["factor"])
        q = _turn(s["q"], position[:, None], s["inv_freq"], c["interleaved"], c["factor"])
    s["k_cache"][at, :, row] = k
    s["v_cache"][at, :, row] = s["v"]
    out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return out if q is None else {"q": q, **out}


def _plain_forward(s):
    c = s["case"]
    B, H, Hk, d, page, new = (c[x] for x in ("B", "H", "Hk", "d", "page", "new"))
    G, q, table = H // Hk, s["q"], s["table"].long().clamp(min=0)
    K, V = (x[table].transpose(1, 2).reshape(B, Hk, -1, d).float() for x in (s["k_cache"], s["v_cache"]))
    cu, lens = s["cu"].long(), s["lens"].long()
    count = cu[1:] - cu[:-1]
    i, j = torch.arange(new, device=q.device), torch.arange(K.shape[2], device=q.device)
    Q = q[(cu[:-1, None] + i).clamp(max=q.shape[0] - 1)]  # [B, new, H, d], rows behind a chunk belong to others
    Q = Q.view(B, new, Hk, G, d).transpose(1, 2).reshape(B, Hk, new * G, d).float()
    position = (lens - count)[:, None] + i
    seen = (j < lens[:, None])[:, None, :].expand(B, new, -1)
    if c["causal"]:
        seen = seen & (j <= position[..., None])
    if c["left"] >= 0:
        seen = seen & (j >= position[..., None] - c["left"])
    S = torch.matmul(Q, K.transpose(2, 3)) * d ** -0.5
    S = S.view(B, Hk, new, G, -1).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = S.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    S = S.sub_(m).exp_()
    total = S.sum(-1)
    O = torch.matmul(S.view(B, Hk, new * G, -1), V).view(B, Hk, new, G, d)
    O = O / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    L = m[..., 0] + total.log()
    b, i, _ = _tokens(s)
    return O[b, :, i].reshape(-1, H, d).to(q.dtype), L[b, :, i].reshape(-1, H)


# ---------------------------------------------------------------------------------------------------- in 64 bits


def _rotated64(x, angle, interleaved, factor):
    """The leading 2 * angle.shape[-1] elements of x as complex numbers, times factor * e^(i angle)."""
    n = angle.shape[-1]
    y = x.double().clone()
    turned = y[..., : 2 * n]
    re, im = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :n], turned[..., n:])
    z = torch.complex(re.contiguous(), im.contiguous()) * torch.polar(torch.full_like(angle, factor), angle)
    if interleaved:
        y[..., 0 : 2 * n : 2], y[..., 1 : 2 * n : 2] = z.real, z.imag
    else:
        y[..., :n], y[..., n : 2 * n] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        angle = s["positions"].double()[:, None] * s["inv_freq"].double()[None, :]
        return _rotated64(s["x"], -angle if case["inverse"] else angle, case["interleaved"], case["factor"])
    H, Hk, d, page = (case[x] for x in ("H", "Hk", "d", "page"))
    table, lens, cu = s["table"].tolist(), s["lens"].tolist(), s["cu"].tolist()
    if case["op"] == "append":
        out = {"k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
        if case["rot"]:
            out = {"q": torch.empty_like(s["q"], dtype=torch.float64), **out}
        for b, n in enumerate(lens):
            new = slice(cu[b], cu[b + 1])
            position = torch.arange(n - (cu[b + 1] - cu[b]), n, device="cuda")
            k = s["k"][new].double()
            if case["rot"]:
                angle = position.double()[:, None, None] * s["inv_freq"].double()
                k = _rotated64(k, angle, case["interleaved"], case["factor"])
                out["q"][new] = _rotated64(s["q"][new], angle, case["interleaved"], case["factor"])
            pages = s["table"][b].long()[position // page]
            out["k_cache"][pages, :, position % page] = k
            out["v_cache"][pages, :, position % page] = s["v"][new].double()
        return out
    O = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    L = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        m = cu[b + 1] - cu[b]
        used = torch.tensor(table[b][: -(-n // page)], device="cuda")
        keys = torch.arange(n, device="cuda")
        rows = torch.arange(n - m, n, device="cuda")
        hidden = torch.zeros((m, n), dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= keys[None, :] > rows[:, None]
        if case["left"] >= 0:
            hidden |= keys[None, :] < rows[:, None] - case["left"]
        for h in range(Hk):
            heads = slice(h * (H // Hk), (h + 1) * (H // Hk))
            k, v = (x[used, h].reshape(-1, d)[:n].double() for x in (s["k_cache"], s["v_cache"]))
            q = s["q"][cu[b] : cu[b + 1], heads].double()
            score = torch.tensordot(q, k, dims=([2], [1])) / math.sqrt(d)
            score.masked_fill_(hidden[:, None, :], -math.inf)
            L[cu[b] : cu[b + 1], heads] = torch.logsumexp(score, -1)
            O[cu[b] : cu[b + 1], heads] = torch.tensordot(torch.softmax(score, -1).nan_to_num_(0.0), v, dims=([2], [0]))
    return O, L


# ---------------------------------------------------------------------------------------------------- work


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "rotary":
        n = case["B"] * case["H"] * case["N"]
        return {"bytes": 2 * size * n * case["d"] + 8 * case["N"], "flops": 3 * n * case["rot"]}
    B, H, Hk, d, page = (case[x] for x in ("B", "H", "Hk", "d", "page"))
    lengths = _lengths(case)
    T = sum(n for n, _ in lengths)
    if case["op"] == "append":
        rows = 2 * Hk + (H if case["rot"] else 0)  # read once, written once
        return {"bytes": 2 * size * T * rows * d + 4 * (T + 2 * B), "flops": max(1, 3 * T * (H + Hk) * case["rot"])}
    keys = pairs = 0
    for n, o in lengths:
        left = case["left"] if case["left"] >= 0 else n + o
        keys += min(n + o, o + n - max(0, o - left))  # that some row sees
        if case["causal"]:
            for i in range(o, o + n):
                pairs += i + 1 - max(0, i - left)
        else:
            pairs += sum(n + o - max(0, i - left) for i in range(o, o + n))
    table = sum(-(-(n + o) // page) for n, o in lengths)
    return {"bytes": size * (2 * T * H * d + 2 * keys * Hk * d) + 4 * (T * H + table + 2 * B), "flops": 4 * d * H * pairs}
