"""Plain restatements in 64 bits, on the CPU, of the paged cache, the attention over it and the verification of drafted
tokens.  One loop per sequence; no cleverness (test infrastructure only)."""
import math

import torch

FP8 = torch.float8_e4m3fn


def quantise(x):
    """(codes, scale) of rows of bf16, in fp32 as the definition has it."""
    x = x.float()
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros(())).amax(-1).clamp(min=1e-30)
    y = x * (torch.full_like(a, 448.0) / a).unsqueeze(-1)        # number / tensor would be the number times a rounded reciprocal
    y = torch.where(torch.isfinite(x), y, torch.full((), math.nan))
    return y.to(FP8), a / 448.0


def place(table, b, j, block):
    return int(table[b, j // block]), j % block


def held(cache, scale):
    """A cache's values in 64 bits."""
    x = cache.float().double()
    return x if scale is None else x * scale.double().unsqueeze(-1)


def write(k_cache, k_scale, new, table, lens, cu):
    """new rows into one of the two caches, in place."""
    block = k_cache.shape[1]
    for b in range(len(lens)):
        n = int(cu[b + 1] - cu[b])
        for i in range(n):
            j = int(lens[b]) - n + i
            if j < 0:
                continue
            p, at = place(table, b, j, block)
            row = new[int(cu[b]) + i]
            if k_scale is None:
                k_cache[p, at] = row
            else:
                code, s = quantise(row)
                k_cache.view(torch.uint8)[p, at] = code.view(torch.uint8)
                k_scale[p, at] = s


def gather(values, table, b, n, block):
    return torch.stack([values[place(table, b, j, block)] for j in range(n)]) if n else values.new_zeros(0, *values.shape[2:])


def attention(q, k, v, table, lens, cu, block, scale=None, causal=True):
    """(out [T, Hq, D], lse [Hq, T], sum of p |v| [T, Hq, D]) in 64 bits; ``k`` / ``v`` from ``held``.  Rows of no sequence are NaN."""
    T, Hq, D = q.shape
    G = Hq // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    size = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((Hq, T), math.nan, dtype=torch.float64)
    for b in range(len(lens)):
        lo, hi, L = int(cu[b]), int(cu[b + 1]), int(lens[b])
        if hi <= lo:
            continue
        kb, vb = gather(k, table, b, L, block), gather(v, table, b, L, block)
        at = torch.arange(hi - lo) + L - (hi - lo)
        seen = (torch.arange(L)[None, :] <= at[:, None]) if causal else torch.ones(hi - lo, L, dtype=torch.bool)
        for h in range(Hq):
            s = (q[lo:hi, h].double() @ kb[:, h // G].T) * scale
            s = s.masked_fill(~seen, -math.inf)
            l = torch.logsumexp(s, 1) if L else torch.full((hi - lo,), -math.inf, dtype=torch.float64)
            p = torch.where(seen, torch.exp(s - torch.where(torch.isfinite(l), l, torch.zeros(()).double())[:, None]), torch.zeros(()).double())
            vh = vb[:, h // G]
            out[lo:hi, h] = p @ vh
            size[lo:hi, h] = p @ vh.abs()
            lse[h, lo:hi] = l
    return out, lse, size


def verify(target, draft, ids, u, cu):
    """(accepted, tokens) with -2 in rows of no sequence."""
    accepted, tokens = [], [-2] * target.shape[0]
    clean = lambda x: torch.where(torch.isfinite(x) & (x > 0), x, torch.zeros_like(x)).double()      # noqa: E731
    V, first = target.shape[1], 0                # first: the sequence's first row of draft
    for b in range(len(cu) - 1):
        lo, hi = int(cu[b]), int(cu[b + 1])
        if hi <= lo:
            accepted.append(0)
            continue
        K, n = hi - lo - 1, 0
        for n in range(K + 1):
            if n == K:
                break
            d = int(ids[lo + n + 1])
            if not 0 <= d < V:
                break
            qd = 1.0 if draft is None else float(clean(draft[first + n])[d])
            if not float(u[lo + n]) * qd < float(clean(target[lo + n])[d]):
                break
        p = clean(target[lo + n])
        rest = p
        if n < K:
            if draft is None:
                gone = torch.zeros_like(p)
                if 0 <= int(ids[lo + n + 1]) < V:
                    gone[int(ids[lo + n + 1])] = 1.0
            else:
                gone = clean(draft[first + n])
            rest = (p - gone).clamp(min=0)
            if float(rest.sum()) == 0:
                rest = p
        sums = rest.cumsum(0)
        over = (sums > float(u[lo + n]) * float(sums[-1])) & (rest > 0)
        some = rest > 0
        token = int(over.nonzero()[0]) if bool(over.any()) else int(some.nonzero()[-1]) if bool(some.any()) else -1
        accepted.append(n)
        first += K
        for i in range(K + 1):
            tokens[lo + i] = int(ids[lo + i + 1]) if i < n else token if i == n else -1
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int64)
