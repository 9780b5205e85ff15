"""Plain forms in 64 bits, on the CPU, of serving with trees of drafts and with caches of limited length, from their definitions in include/ftk.h."""
import math

import torch


def way(parents, t):
    """The nodes from t up to its root; a parent that does not come before its child is none."""
    out = [t]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(parents[out[-1]])
    return out


def tree_sees(parents, n, first, length, window=0):
    """[n, length]: which positions each of n new tokens sees, and how deep it lies."""
    seen = torch.zeros((n, length), dtype=torch.bool)
    for t in range(n):
        up = way(parents, t)
        depth = len(up) - 1
        lo = first + depth - window + 1 if window else 0
        seen[t, max(lo, 0):max(0, min(first, length))] = True
        for i, x in enumerate(up):
            if 0 <= first + x < length and (not window or i < window):
                seen[t, first + x] = True
    return seen


def causal_sees(n, first, length, causal=True, window=0):
    position, key = first + torch.arange(n)[:, None], torch.arange(length)
    seen = torch.ones((n, length), dtype=torch.bool)
    if causal:
        seen &= key <= position
    if window:
        seen &= key > position - window
    return seen


def sequences(batch):
    """(sequence, first packed row, new tokens, position of the first of them, length as far as the table has room)."""
    for b, length in enumerate(batch['lens']):
        s, e = batch['starts'][b], batch['starts'][b + 1]
        yield b, s, e - s, length - (e - s), min(length, len(batch['table'][b]) * batch['page'])


def rows_of(batch, x, b, h, length):
    """Rows of a head of x [pages, heads, page, ..] in the order of their positions."""
    ids = [min(max(t, 0), batch['pages'] - 1) for t in batch['table'][b]]
    return x[ids, h].reshape(-1, *x.shape[3:])[:length]


def attention(q, k, v, batch, heads, scale, sees):
    """As serving_reference.attention, for any masks: sees(b, n, first, length) -> [n, length]."""
    tokens, Hq, D = q.shape
    G, qd = Hq // heads, q.cpu().double()
    o, lse = torch.zeros((tokens, Hq, D), dtype=torch.float64), torch.full((tokens, Hq), -math.inf, dtype=torch.float64)
    mean, most, count, top = torch.zeros_like(o), torch.zeros_like(lse), torch.zeros_like(lse), torch.zeros_like(o)
    for b, s, n, first, length in sequences(batch):
        if n == 0 or length == 0:
            continue
        seen = sees(b, n, first, length)
        for h in range(heads):
            kk, vv = rows_of(batch, k, b, h, length), rows_of(batch, v, b, h, length)
            clean = torch.nan_to_num(kk, nan=0.0, posinf=0.0, neginf=0.0)
            bad = ~torch.isfinite(kk).all(1)
            value = torch.where(torch.isfinite(vv), vv, 0.0)
            for g in range(G):
                x = qd[s:s + n, h * G + g]
                scores = torch.where(bad[None, :], torch.nan, (x @ clean.T) * scale).masked_fill(~seen, -math.inf)
                at = (slice(s, s + n), h * G + g)
                lse[at] = torch.logsumexp(scores, 1)
                w = torch.where(seen, torch.exp(scores - lse[at][:, None]), 0.0)
                o[at] = w @ value
                o[at][(seen.double() @ (~torch.isfinite(vv)).double()) > 0] = math.nan
                none = ~seen.any(1)
                o[at][none] = 0.0
                lse[at][none] = -math.inf
                mean[at] = torch.nan_to_num(w @ value.abs())
                most[at] = ((x.abs() @ clean.abs().T) * scale).masked_fill(~seen, 0.0).amax(1)
                count[at] = seen.sum(1).double()
                top[at] = (seen.double() @ value.abs()) / seen.sum(1, keepdim=True).clamp(min=1)
    return dict(o=o, lse=lse, mean=mean, most=most, count=count, top=top)


def weigh(q, lse, k, weights, batch, heads, scale, sees, decay=1.0):
    """(weights, how far fp32 may be from them).  A score is a sum of D products, exact in fp32 each, off by at most D 2^-24 of the sum of magnitudes, then scaled and shifted by the lse with a
    rounding of each factor and of the result; the hardware's exponential adds 2^-22 of a weight; sums of n weights, of the four lanes and of what was there before
    n + 4 half steps of what they come to."""
    tokens, Hq, D = q.shape
    G, qd, ld = Hq // heads, q.cpu().double(), lse.cpu().double()
    out, off = weights.clone().double(), torch.zeros(weights.shape, dtype=torch.float64)
    for b, s, n, first, length in sequences(batch):
        if n == 0 or length == 0:
            continue
        seen = sees(b, n, first, length)
        pages = torch.tensor(batch['table'][b])[torch.arange(length) // batch['page']]
        rows = torch.arange(length) % batch['page']
        for h in range(heads):
            kk = rows_of(batch, k, b, h, length)
            total, error = torch.zeros(length, dtype=torch.float64), torch.zeros(length, dtype=torch.float64)
            for g in range(G):
                x, z = qd[s:s + n, h * G + g], ld[s:s + n, h * G + g]
                scores = torch.where(seen, (x @ kk.T) * scale, -math.inf)
                w = torch.where(seen & (z != -math.inf)[:, None], torch.exp(scores - z[:, None]), 0.0)
                size = (x.abs() @ kk.abs().T) * scale
                total += w.sum(0)
                error += (w * (((D + 4) * size + 3 * z.abs()[:, None]) * 2.0 ** -24 + 2.0 ** -22)).nan_to_num().sum(0)
            there = (pages >= 0) & (pages < batch['pages'])
            p, r = pages[there], rows[there]
            before = torch.where(torch.arange(length)[there] < first, weights[p, h, r].double() * decay if decay else 0.0, 0.0)
            out[p, h, r] = before + total[there]
            off[p, h, r] = error[there] + (before.abs() + total[there].abs()) * (n * G + 4) * 2.0 ** -24 + 2.0 ** -126
    return out, off


def select(weights, table, lens, page, budget, sinks, recent):
    pages, heads = weights.shape[:2]
    out = torch.full((len(lens), heads, budget), -1, dtype=torch.int32)
    for b, length in enumerate(lens):
        length = max(0, min(length, len(table[b]) * page))
        for h in range(heads):
            if length <= budget:
                out[b, h, :length] = torch.arange(length)
                continue
            def key(p):
                t = table[b][p // page]
                x = float(weights[t, h, p % page]) if 0 <= t < pages else math.nan
                return (x == x, x if x == x else 0.0)
            middle = sorted(range(sinks, length - recent), key=lambda p: (key(p), -p), reverse=True)[:budget - sinks - recent]
            stay = sorted(list(range(sinks)) + middle + list(range(length - recent, length)))
            out[b, h] = torch.tensor(stay)
    return out


def keep(arrays, table, lens, firsts, kept, page):
    """Arrays [pages, heads, page, ..] moved in place, and the new lengths."""
    pages, heads = arrays[0].shape[:2]
    out = []
    for b in range(len(lens)):
        count = 0
        for h in range(heads):
            row = (kept[b] if kept.dim() == 2 else kept[b, h]).tolist()
            row = row[:row.index(-1)] if -1 in row else row
            count = len(row) if h == 0 else count

            def place(p):
                if not 0 <= p < min(lens[b], len(table[b]) * page):
                    return None
                t = table[b][p // page]
                return (t, h, p % page) if 0 <= t < pages else None
            moves = [(place(firsts[b] + x), place(firsts[b] + j)) for j, x in enumerate(row) if x != j]
            moves = [(s, d) for s, d in moves if s is not None and d is not None]
            for a in arrays:
                got = [a[s].clone() for s, _ in moves]
                for x, (_, d) in zip(got, moves):
                    a[d] = x
        out.append(max(0, firsts[b] + count))
    return torch.tensor(out, dtype=torch.int32)


def verify(target, ids, parents, starts, uniforms):
    target, ids, parents, uniforms = (t.cpu() for t in (target, ids, parents, uniforms))
    B, M = uniforms.shape
    tokens, path, accepted = torch.full((B, M), -1, dtype=ids.dtype), torch.full((B, M), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        s, n = starts[b], starts[b + 1] - starts[b]
        node, steps = (0 if n > 0 else -1), 0
        while node >= 0 and steps < M:
            w = target[s + node].double()
            w = torch.where(w > 0, w, 0.0).tolist()
            aim, at, token, last = float(uniforms[b, steps]) * math.fsum(w), 0.0, -1, -1
            for t, x in enumerate(w):
                at += x
                if x > 0:
                    last = t
                    if at > aim:
                        token = t
                        break
            token = token if token >= 0 else last
            tokens[b, steps], path[b, steps] = token, node
            steps += 1
            node = next((i for i in range(node + 1, n) if int(parents[s + i]) == node and int(ids[s + i]) == token), -1) if token >= 0 else -1
        accepted[b] = max(0, steps - 1)
    return tokens, path, accepted
