"""Plain 64-bit forms of rotary positions, paged caches and the attention over them, on the CPU, and the bounds that the library is held to."""
import math
from decimal import Decimal, localcontext

import numpy as np
import torch


def half_step(dtype):
    """Largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


# ---- rotary


def angles(positions, inv_freq):
    """cos and sin [..., rot / 2] of position * inv_freq, the product and its remainder taken in 80 bits, from 2^33 on in 80 digits."""
    if np.abs(np.asarray(positions)).max(initial=0) >= 2 ** 33:
        with localcontext() as digits:
            digits.prec = 80
            two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")
            turns = [[Decimal(int(p)) * Decimal(float(w)) / two_pi for w in inv_freq] for p in np.asarray(positions).reshape(-1)]
            a = np.array([[float((t - t.to_integral_value()) * two_pi) for t in row] for row in turns]).reshape(*np.shape(positions), len(inv_freq))
        return torch.from_numpy(np.cos(a)), torch.from_numpy(np.sin(a))
    a = np.asarray(positions, dtype=np.longdouble)[..., None] * np.asarray(inv_freq, dtype=np.longdouble)
    two_pi = np.longdouble("6.283185307179586476925286766559005768394")
    a = a - np.rint(a / two_pi) * two_pi
    return torch.from_numpy(np.cos(a).astype(np.float64)), torch.from_numpy(np.sin(a).astype(np.float64))


def rotate(x, cos, sin, interleaved, factor):
    """x [..., d] in 64 bits, cos and sin broadcast against [..., rot / 2]"""
    n = cos.shape[-1]
    y = x.double().clone()
    a, b = (x[..., 0:2 * n:2].double(), x[..., 1:2 * n:2].double()) if interleaved else (x[..., :n].double(), x[..., n:2 * n].double())
    u, v = factor * (a * cos - b * sin), factor * (a * sin + b * cos)
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = u, v
    else:
        y[..., :n], y[..., n:2 * n] = u, v
    return y


def rotate_bound(x, cos, interleaved, factor, dtype, ref):
    """One rounding of the result to its type; in 32 bits: the fraction of a turn is rounded once (its angle is at most pi, so an error of
    pi 2^-24 in either of sine and cosine), sine and cosine are good to 4 half steps, their product with factor is rounded, and so are the two
    products and the sum.  Together below 12 half steps of |a| + |b| per element."""
    n = cos.shape[-1]
    size = x.double().abs()
    big = torch.zeros_like(size)
    if interleaved:
        big[..., :2 * n] = (size[..., 0:2 * n:2] + size[..., 1:2 * n:2]).repeat_interleave(2, -1)
    else:
        s = size[..., :n] + size[..., n:2 * n]
        big[..., :2 * n] = torch.cat((s, s), -1)
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}[dtype]
    return half_step(dtype) * ref.abs() * (0 if dtype == torch.float32 else 1) + 12 * 2.0 ** -24 * abs(factor) * big + tiny


# ---- paged attention


def gather(cache, table_row, n):
    """K or V of a sequence, [H_kv, n, d], from the pages."""
    page = cache.shape[2]
    if n == 0:
        return torch.zeros((cache.shape[1], 0, cache.shape[3]), dtype=torch.float64)
    pages = table_row[: -(-n // page)].long()
    return cache[pages].transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :n].double()


def visible(m, n, causal, window):
    """[m, n] of row i of m standing at n - m + i"""
    p = torch.arange(n - m, n)[:, None]
    j = torch.arange(n)[None, :]
    ok = torch.ones((m, n), dtype=torch.bool)
    if causal:
        ok &= j <= p
    if window[0] >= 0:
        ok &= j >= p - window[0]
    if window[1] >= 0:
        ok &= j <= p + window[1]
    return ok


def attention(q, k_cache, v_cache, table, lens, cu, scale, causal, window):
    """(O, LSE, bound on O, bound on LSE), LSE +inf in rows of no sequence.  CPU tensors.

    The bounds, with u = half a step of the type (P and O are rounded to it), e = 2^-24, n keys, and S the largest sum of |q k| scale of the row:
      score     products are exact in 32 bits, d sums, one multiplication by scale log2 e (itself rounded), one subtraction of the
                reference, whose size is that of a score: (d + 6) e S; 2^x is good to two half steps
      p         relative error x <= (d + 6) e S + 4 e
      LSE       x, n sums of the denominator, the merge of waves and splits (40 e), the logarithm (2 e relative)
      O         numerator and denominator x and n e each, P rounded (u), all of it relative to sum p |v|; fp16 probabilities below 2^-14 are rounded
                to multiples of 2^-24: n 2^-25 of the largest |v| (the row's largest probability is at least 1); O rounded (u |O|)"""
    T, H, d = q.shape
    Hk = k_cache.shape[1]
    G = H // Hk
    u, e = half_step(q.dtype), 2.0 ** -24
    O = torch.full((T, H, d), math.nan, dtype=torch.float64)
    L = torch.full((T, H), math.inf, dtype=torch.float64)
    bO, bL = torch.zeros_like(O), torch.zeros_like(L)
    for b, n in enumerate(lens.tolist()):
        t0, t1 = int(cu[b]), int(cu[b + 1])
        m = t1 - t0
        if m == 0:
            continue
        K, V = gather(k_cache, table[b], n), gather(v_cache, table[b], n)
        ok = visible(m, n, causal, window)
        for h in range(H):
            Q, k, v = q[t0:t1, h].double(), K[h // G], V[h // G]
            # what a row does not see does not count, whatever it holds
            seen = ok.any(0)
            k, v = torch.where(seen[:, None], k, 0.0), torch.where(seen[:, None], v, 0.0)
            s = torch.where(ok, (Q @ k.T) * scale, -math.inf)
            big = torch.where(ok, (Q.abs() @ k.abs().T) * scale, 0.0).amax(1) if n else torch.zeros(m, dtype=torch.float64)
            top = s.amax(1, keepdim=True) if n else torch.full((m, 1), -math.inf, dtype=torch.float64)
            p = torch.where(ok, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(1, keepdim=True)
            w = p / torch.where(total > 0, total, 1.0)
            # (0 times a value that is not finite: only visible ones count)
            if torch.isfinite(v).all():
                o, size = w @ v, w @ v.abs()
            else:
                o = torch.stack([(torch.where(ok[i][:, None], v, 0.0) * w[i][:, None]).sum(0) for i in range(m)])
                size = w @ v.abs().nan_to_num(0, 0, 0)
            O[t0:t1, h] = o
            L[t0:t1, h] = (torch.log(total) + top)[:, 0]
            x = (d + 6) * e * big + 4 * e
            fine = v.abs().nan_to_num(0, 0, 0).max() if n else 0.0
            bO[t0:t1, h] = (u + 2 * x + (2 * n + 40) * e)[:, None] * size * 1.01 + u * o.abs() + n * fine * (2.0 ** -25 if q.dtype == torch.float16 else 0) + 1e-30
            if q.dtype == torch.float16:
                bO[t0:t1, h] += 2.0 ** -25
            bL[t0:t1, h] = x + (n + 40) * e + 4 * e * L[t0:t1, h].abs().nan_to_num(0, 0, 0)
    return O, L, bO, bL


def check_attention(o, lse, ref, what=""):
    O, L, bO, bL = ref
    mine = ~torch.isposinf(L)  # rows of a sequence
    o, lse = o.cpu().double(), lse.cpu().double()
    empty = torch.isneginf(L)
    assert torch.equal(torch.isneginf(lse)[mine], empty[mine]), f"{what}: rows without a key differ"
    assert (o[empty] == 0).all(), f"{what}: rows without a key are not 0"
    assert torch.equal(torch.isnan(lse)[mine], torch.isnan(L)[mine]), f"{what}: other rows have a LSE that is not a number"
    ok = mine & ~empty
    fine = torch.isfinite(O)
    assert torch.equal(torch.isfinite(o)[ok], fine[ok]), f"{what}: other elements of O are finite"
    off = torch.where(fine & ok[..., None], (o - O).abs() - bO, -1.0)
    assert off.max() <= 0, f"{what}: O off by {(o - O).abs()[fine & ok[..., None]].max():.3e}, {off.max():.3e} more than it may be"
    off = torch.where(ok & ~torch.isnan(L), (lse - L).abs() - bL, -1.0)
    assert off.max() <= 0, f"{what}: LSE {off.max():.3e} more off than it may be"


class Batch:
    """Sequences with `news` new tokens and `lens` keys in shuffled pages, on the CPU; .cuda() has the tensors of a call."""

    def __init__(self, news, lens, H, Hk, d, page, dtype, seed=0, first=0, behind=0, spare=2, stale=None):
        g = torch.Generator().manual_seed(seed)
        self.news, self.page = news, page
        need = [-(-n // page) for n in lens]
        total = sum(need) + spare
        order = torch.randperm(total, generator=g, dtype=torch.int32)
        self.table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n

        def normal(*shape):
            return torch.randn(shape, generator=g).to(dtype)

        T = first + sum(news) + behind
        self.q = normal(T, H, d)
        self.k_cache, self.v_cache = normal(total, Hk, page, d), normal(total, Hk, page, d)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.cu = torch.tensor([first + sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32)
        if stale is not None:  # everything that no sequence has
            used = torch.zeros((total, page), dtype=torch.bool)
            for b, n in enumerate(lens):
                j = torch.arange(n)
                used[self.table[b].long()[j // page], j % page] = True
            for c in (self.k_cache, self.v_cache):
                c.transpose(1, 2)[~used] = stale

    def cuda(self):
        return tuple(t.cuda() for t in (self.q, self.k_cache, self.v_cache, self.table, self.lens, self.cu))

    def reference(self, causal=False, window=(-1, -1), scale=None):
        d = self.q.shape[2]
        return attention(self.q, self.k_cache, self.v_cache, self.table, self.lens, self.cu, d ** -0.5 if scale is None else scale, causal, window)
