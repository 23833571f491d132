"""Plain 64-bit forms of the paged attention's other scores and masks and of the operators for drafted tokens, on the CPU, and the bounds that the library
is held to."""
import math

import torch

from paged_reference import gather, half_step


def tree_paths(parents, n):
    """[n, n] of token i's path from the root, itself among them."""
    on = torch.eye(n, dtype=torch.bool)
    for i in range(n):
        p = int(parents[i])
        if 0 <= p < i:
            on[i] |= on[p]
    return on


def tree_mask(parents, cu, lens, words):
    """(mask, positions) of flash_tree_mask; rows of no sequence 0."""
    T = parents.shape[0]
    mask, positions = torch.zeros((T, words), dtype=torch.int64), torch.zeros(T, dtype=torch.int32)
    for b in range(len(cu) - 1):
        t0, t1 = int(cu[b]), int(cu[b + 1])
        n = t1 - t0
        base = int(lens[b]) - n if lens is not None else 0
        m = min(n, 64 * words)
        on = tree_paths(parents[t0:t1], m)
        for i in range(n):
            x = sum(1 << j for j in range(m) if on[i, j]) if i < m else 0
            for w in range(words):
                v = (x >> 64 * w) % 2 ** 64
                mask[t0 + i, w] = v - 2 ** 64 if v >= 2 ** 63 else v
            positions[t0 + i] = base + (bin(x).count("1") - 1 if i < m else 0)
    return mask, positions


def random_parents(news, seed, back=6):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in news:
        p = [max(-1, i - 1 - int(torch.randint(0, back, (1,), generator=g))) for i in range(n)]
        out += p
    return torch.tensor(out, dtype=torch.int32)


def seen_bits(mask_rows, n):
    """[m, n] from a mask's rows"""
    m, words = mask_rows.shape
    j = torch.arange(n)
    ok = torch.zeros((m, n), dtype=torch.bool)
    inside = j < 64 * words
    ok[:, inside] = (mask_rows[:, j[inside] // 64] >> (j[inside] % 64)) & 1 == 1
    return ok


def view(m, n, causal, window, prefix, mask_rows):
    """([m, n] what row i of m sees of the n keys, [m, n] distance row - key of positions)"""
    base = n - m
    rows, keys = torch.arange(base, n), torch.arange(n)
    ok = torch.ones((m, n), dtype=torch.bool)
    if mask_rows is not None:
        on = seen_bits(mask_rows, m)
        depth = (on.sum(1) - 1).clamp(min=0)
        rows = base + depth
        keys = torch.cat((keys[:max(base, 0)], rows))[-n:] if n else keys
        if n:
            ok[:, max(base, 0):] = on[:, max(-base, 0):]
    apart = rows[:, None] - keys[None, :]
    if mask_rows is None:
        if causal:
            ok &= apart >= 0
        if window[1] >= 0:
            ok &= -apart <= window[1]
        ok |= torch.arange(n)[None, :] < prefix
    if window[0] >= 0:
        ok &= apart <= window[0]
    return ok, apart


def attention(q, k_cache, v_cache, table, lens, cu, scale=None, causal=False, window=(-1, -1), softcap=0.0, slopes=None, prefix=None, mask=None):
    """(O, LSE, bound on O, bound on LSE, rows of a sequence).  CPU tensors, everything that a row sees finite.

    The bounds, with u half a step of the type, e = 2^-24, n keys, and for a key: S = sum |q k| scale, B = slope * distance, c the cap, w its weight:
      score  d products and sums in 32 bits, the scaling and the reference (d + 6) e (S + B), as the bias is what the sums begin with; the slope's unit, its
             product and the distance's place 5 e B; the reference's own rounding 2 e max |score|;
             capped: t = -1 / (1 + 2^x) has the roundings of x (2 of |x|, which 2^x / (1 + 2^x)^2 brings below 1 e), of v_exp_f32 (2 e, a quarter of it),
             of the sum (e) and of v_rcp_f32 (2 e): 4.5 e of 2 c; the factor, the fma and the reference 2 e of c each: 16 e c
      p      E = that + 4 e for 2^x, relative, which moves LSE by sum w E and O by sum w E |v| + (sum w E) sum w |v|
      LSE    sum w E, n sums, merges (40 e), the logarithm and the cap's sum (4 e (|LSE| + c))
      O      (u + (2 n + 40) e) sum w |v|: P rounded once; O rounded (u |O|); fp16 probabilities below 2^-14 are multiples of 2^-24, as are results"""
    T, H, d = q.shape
    Hk = k_cache.shape[1]
    G = H // Hk
    u, e = half_step(q.dtype), 2.0 ** -24
    half = q.dtype == torch.float16
    scale = d ** -0.5 if scale is None else scale
    O, L = torch.zeros((T, H, d), dtype=torch.float64), torch.full((T, H), -math.inf, dtype=torch.float64)
    bO, bL, mine = torch.zeros_like(O), torch.zeros_like(L), torch.zeros(T, dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        t0, t1 = int(cu[b]), int(cu[b + 1])
        m = t1 - t0
        mine[t0:t1] = True
        if m == 0 or n == 0:
            continue
        K, V = gather(k_cache, table[b], n), gather(v_cache, table[b], n)
        ok, apart = view(m, n, causal, window, int(prefix[b]) if prefix is not None else 0, mask[t0:t1] if mask is not None else None)
        for h in range(H):
            Q, k, v = q[t0:t1, h].double(), K[h // G], V[h // G]
            seen = ok.any(0)
            k, v = torch.where(seen[:, None], k, 0.0), torch.where(seen[:, None], v, 0.0)
            s, S = (Q @ k.T) * scale, (Q.abs() @ k.abs().T) * scale
            B = torch.zeros_like(S)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                B = float(slopes[h].double().abs()) * apart.abs().double()
                s = s - float(slopes[h].double()) * apart.abs().double()
            s = torch.where(ok, s, -math.inf)
            top = s.amax(1, keepdim=True)
            top0 = torch.where(top == -math.inf, 0.0, top)
            p = torch.where(ok, torch.exp(s - top0), 0.0)
            total = p.sum(1, keepdim=True)
            w = p / torch.where(total > 0, total, 1.0)
            E = (d + 6) * e * (S + B) + 5 * e * B + 16 * e * softcap + 2 * e * top0.abs() + 4 * e
            x = (w * E).sum(1, keepdim=True)
            size = w @ v.abs()
            O[t0:t1, h], L[t0:t1, h] = w @ v, (torch.log(total) + top)[:, 0]
            l = L[t0:t1, h].abs().nan_to_num(0, 0, 0)
            bL[t0:t1, h] = (x[:, 0] + (n + 40) * e + 4 * e * (l + softcap)) * 1.01
            bO[t0:t1, h] = ((u + (2 * n + 40) * e + x) * size + (w * E) @ v.abs()) * 1.01 + u * (w @ v).abs() + 1e-30
            if half:
                bO[t0:t1, h] += 2.0 ** -25 * (n * v.abs().max() + 1)
    return O, L, bO, bL, mine


def check(o, lse, want, what=""):
    O, L, bO, bL, mine = want
    o, lse = o.cpu().double()[mine], lse.cpu().double()[mine]
    O, L, bO, bL = O[mine], L[mine], bO[mine], bL[mine]
    empty = torch.isneginf(L)
    assert torch.equal(torch.isneginf(lse), empty), f"{what}: other rows see nothing"
    assert (o[empty] == 0).all(), f"{what}: rows that see nothing are not 0"
    assert torch.isfinite(o).all() and torch.isfinite(lse[~empty]).all(), f"{what}: not finite"
    off = (o - O).abs() - bO
    assert off.numel() == 0 or off.max() <= 0, f"{what}: O off by {(o - O).abs().max():.3e}, {off.max():.3e} more than it may be"
    off = ((lse - L).abs() - bL)[~empty]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: LSE {off.max():.3e} more off than it may be"


def keep(k_cache, v_cache, table, lens, cu, path, accepted):
    """New (k_cache, v_cache, lengths) of flash_keep_paged; caches with a dimension of layers in front, or none."""
    page = k_cache.shape[-2]
    K, V = k_cache.clone(), v_cache.clone()
    after = []
    for b, n in enumerate(lens.tolist()):
        count = int(cu[b + 1]) - int(cu[b])
        base, last, kept = n - count, -1, 0
        for i in range(min(max(int(accepted[b]), 0), path.shape[1])):
            p = int(path[b, i])
            if not last < p < count:
                break
            last, kept = p, i + 1
            s, t = base + p, base + i
            if t < 0 or s >= page * table.shape[1]:
                continue
            a, z = int(table[b, s // page]), int(table[b, t // page])
            if not (0 <= a < k_cache.shape[-4] and 0 <= z < k_cache.shape[-4]):
                continue
            for c, old in ((K, k_cache), (V, v_cache)):
                c[..., z, :, t % page, :] = old[..., a, :, s % page, :]
        after.append(max(base + kept, 0))
    return K, V, torch.tensor(after, dtype=torch.int32)
