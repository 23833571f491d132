"""Attention over a paged cache in 64 bits, with values that are not finite worked out by their class: what check() holds a result to, element by
element, is a bound that is finite wherever the value is, not a number where the definition has none, and the infinity of the right sign.

Written apart from paged_reference.py, whose bounds grow without limit beside a score of -inf and whose comparison takes any value that is not
finite for any other."""
import math

import torch


def _dense(cache, row, n, page):
    """[H_kv, n, d] of the first n keys"""
    j = torch.arange(n)
    return cache[row.long()[j // page], :, j % page].transpose(0, 1).double()


def attention(q, k_cache, v_cache, table, lens, cu, scale=None, causal=False, window=(-1, -1)):
    """(O, LSE, bound on O, bound on LSE, rows of a sequence) on the CPU.

    Bounds, with u half a step of the type, e = 2^-24, n keys and S the largest sum of scale |q k| among the row's keys that have a weight (a key whose
    score is -inf has the weight 0 on either side):
      p, relative   x = (d + 6) e S + 4 e: d products and sums in 32 bits, the scaling, the subtraction of the reference, the exponential
      LSE           x + (n + 40) e + 4 e |LSE|: n sums, the merge of waves and splits, the logarithm
      O             (u + 2 x + (2 n + 40) e) sum p |v| + u |O|: P and O rounded once each; in fp16 probabilities below 2^-14 are multiples of 2^-24
                    (n 2^-25 max |v|) and so are results (2^-25)"""
    T, H, d = q.shape
    Hk, page = k_cache.shape[1], k_cache.shape[2]
    G, u, e = H // Hk, torch.finfo(q.dtype).eps / 2, 2.0 ** -24
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
        at, j = torch.arange(n - m, n)[:, None], torch.arange(n)[None, :]
        sees = torch.ones((m, n), dtype=torch.bool)
        if causal:
            sees &= j <= at
        if window[0] >= 0:
            sees &= j >= at - window[0]
        if window[1] >= 0:
            sees &= j <= at + window[1]
        K, V = _dense(k_cache, table[b], n, page), _dense(v_cache, table[b], n, page)
        for h in range(H):
            Q, k, v = q[t0:t1, h].double(), K[h // G], V[h // G]
            # scores: of finite keys by the product, of others by element (their rows are few)
            odd = ~torch.isfinite(k).all(1)
            kf = torch.where(odd[:, None], 0.0, k)
            s, size = Q @ kf.T * scale, Q.abs() @ kf.abs().T * scale
            for i in odd.nonzero()[:, 0].tolist():
                s[:, i] = (Q * k[i]).sum(1) * scale
            weighs = sees & (s != -math.inf)
            s = torch.where(weighs, s, -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.where(weighs, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(1, keepdim=True)
            w = p / torch.where(total > 0, total, torch.where(torch.isnan(total), total, 1.0))
            fine = torch.where(torch.isfinite(v) & weighs.any(0)[:, None], v, 0.0)
            o = w @ fine
            big = torch.where(weighs, size, 0.0).amax(1)
            # what is not finite among the values that the row gives a weight
            there = weighs.double()
            nan, pos, neg = (there @ c.double() > 0 for c in (torch.isnan(v), v == math.inf, v == -math.inf))
            o = torch.where(pos, math.inf, torch.where(neg, -math.inf, o))
            o = torch.where(nan | (pos & neg) | torch.isnan(total), math.nan, o)
            x = (d + 6) * e * big + 4 * e
            O[t0:t1, h], L[t0:t1, h] = o, (torch.log(total) + top)[:, 0]
            bO[t0:t1, h] = ((u + 2 * x + (2 * n + 40) * e)[:, None] * (w.nan_to_num(0) @ fine.abs()) * 1.01 + u * o.nan_to_num(0, 0, 0).abs() + 1e-30
                            + (2.0 ** -25 * (n * fine.abs().max() + 1) if half else 0))
            bL[t0:t1, h] = x + (n + 40) * e + 4 * e * L[t0:t1, h].abs().nan_to_num(0, 0, 0)
    return O, L, bO, bL, mine


def check(o, lse, want, what=""):
    """Rows of no sequence are not looked at."""
    O, L, bO, bL, mine = want
    for name, got, ref, bound in (("O", o, O, bO), ("LSE", lse, L, bL)):
        got, ref, bound = got.cpu().double()[mine], ref[mine], bound[mine]
        fine = torch.isfinite(ref)
        assert torch.isfinite(bound[fine]).all()
        assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: {name} is not a number in other places"
        odd = ~fine & ~torch.isnan(ref)
        assert torch.equal(got[odd], ref[odd]), f"{what}: {name} has other infinities"
        assert torch.isfinite(got[fine]).all(), f"{what}: {name} is not finite where it should be"
        off = ((got - ref).abs() - bound)[fine]
        assert off.numel() == 0 or off.max() <= 0, f"{what}: {name} off by {off.max():.3e} more than it may be"
