"""Plain forms of the serving operators in 64 bits, on the CPU, from their definitions in include/ftk.h; and small caches and batches to try them on."""
import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
LEAST = {(torch.float16, torch.float8_e4m3fn): -15, (torch.float16, torch.int8): -24, (torch.bfloat16, torch.float8_e4m3fn): -100, (torch.bfloat16, torch.int8): -100}
REACH = {(torch.float16, torch.float8_e4m3fn): 61440.0, (torch.float16, torch.int8): 65024.0,
         (torch.bfloat16, torch.float8_e4m3fn): 1.875 * 2.0 ** 127, (torch.bfloat16, torch.int8): 127 * 2.0 ** 121}


def e4m3_values():
    """What each of the 256 codes stands for."""
    out = []
    for c in range(256):
        sign, e, f = -1.0 if c & 128 else 1.0, c >> 3 & 15, c & 7
        out.append(float('nan') if e == 15 and f == 7 else sign * (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)))
    return torch.tensor(out, dtype=torch.float64)


def quantise_row(row, dtype, cache):
    """(values of the codes, exponent) of one row."""
    x = [float(v) for v in row]
    x = [v if math.isnan(v) else max(-REACH[dtype, cache], min(REACH[dtype, cache], v)) for v in x]
    big = max([abs(v) for v in x if not math.isnan(v)], default=0.0)
    e = LEAST[dtype, cache]
    while big > LARGEST[cache] * 2.0 ** e:
        e += 1
    codes = []
    for v in x:
        if math.isnan(v):
            codes.append(float('nan') if cache == torch.float8_e4m3fn else 0.0)
            continue
        y = abs(v) * 2.0 ** -e
        step = 1.0 if cache == torch.int8 else 2.0 ** (max(math.frexp(y)[1] - 1, -6) - 3)
        codes.append(math.copysign(round(y / step) * step, v))       # round() takes the even one of two
    return codes, e


def code_values(pages):
    """Codes or 16-bit elements as float64 numbers, on the CPU."""
    if pages.dtype == torch.float8_e4m3fn:
        return e4m3_values()[pages.cpu().view(torch.uint8).long()]
    return pages.cpu().double()


def places(batch, b):
    """(packed row, page, row in the page) of the new tokens of sequence b that have a place in the cache."""
    starts, lens, table, page = batch['starts'], batch['lens'], batch['table'], batch['page']
    out = []
    for row in range(starts[b], starts[b + 1]):
        p = lens[b] - starts[b + 1] + row
        if 0 <= p < len(table[b]) * page and 0 <= table[b][p // page] < batch['pages']:
            out.append((row, table[b][p // page], p % page))
    return out


def make_batch(new, lens, page, seed, spare=2, tail=0):
    """A batch on pages in any order; `tail` rows behind the last sequence."""
    g = torch.Generator().manual_seed(seed)
    widths = [max(1, -(-n // page)) for n in lens]
    order = torch.randperm(sum(widths) + spare, generator=g).tolist()
    table, at = [], 0
    for w in widths:
        table.append(order[at:at + w] + [order[-1]] * (max(widths) - w))
        at += w
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(starts=starts, lens=list(lens), table=table, page=page, pages=sum(widths) + spare, tokens=starts[-1] + tail)


def on_device(batch):
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device='cuda')
    return ints(batch['table']), ints(batch['lens']), ints(batch['starts'])


def make_pages(batch, heads, D, cache, dtype, seed, scale=1.0):
    """k_pages, v_pages, k_exps, v_exps with anything in them that is finite; exponents None for pages of 16 bits."""
    g = torch.Generator().manual_seed(seed)
    shape = (batch['pages'], heads, batch['page'], D)
    if cache is None:
        return [(torch.randn(shape, generator=g) * scale).to(dtype) for _ in range(2)] + [None, None]
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=g)
        out.append((x * 120).clamp(-448, 448).to(torch.float8_e4m3fn) if cache == torch.float8_e4m3fn else (x * 40).round().clamp(-127, 127).to(torch.int8))
    unit = -7 if cache == torch.float8_e4m3fn else -6
    return out + [torch.randint(unit - 1, unit + 2, shape[:3], generator=g).to(torch.int8) for _ in range(2)]


def held(pages, exps):
    x = code_values(pages)
    return x if exps is None else x * torch.pow(2.0, exps.cpu().double()).unsqueeze(-1)


def attention(q, k, v, batch, heads, scale, causal=True, window=0):
    """o, lse, and what the bounds of rounding errors are made of: the weighted mean of |v|, the largest sum of |q k| scale, the number of keys, and the
    largest |v|; k, v: held()."""
    tokens, Hq, D = q.shape
    G, page = Hq // heads, batch['page']
    qd = q.cpu().double()
    o, lse = torch.zeros((tokens, Hq, D), dtype=torch.float64), torch.full((tokens, Hq), -math.inf, dtype=torch.float64)
    mean, most, count, top = torch.zeros_like(o), torch.zeros_like(lse), torch.zeros_like(lse), torch.zeros_like(o)
    for b in range(len(batch['lens'])):
        s, e = batch['starts'][b], batch['starts'][b + 1]
        length = min(batch['lens'][b], len(batch['table'][b]) * page)
        if e == s or length == 0:
            continue
        ids = [min(max(t, 0), batch['pages'] - 1) for t in batch['table'][b]]
        position = batch['lens'][b] - (e - s) + torch.arange(e - s)
        key = torch.arange(length)
        seen = torch.ones((e - s, length), dtype=torch.bool)
        if causal:
            seen &= key <= position[:, None]
        if window:
            seen &= key > position[:, None] - window
        for h in range(heads):
            kk, vv = (x[ids, h].reshape(-1, D)[:length] for x in (k, v))
            for g in range(G):
                x = qd[s:e, h * G + g]
                scores = (x @ torch.nan_to_num(kk, nan=0.0, posinf=0.0, neginf=0.0).T) * scale
                bad = ~torch.isfinite(kk).all(1)
                scores = torch.where(bad[None, :], torch.nan, scores).masked_fill(~seen, -math.inf)
                at = (slice(s, e), h * G + g)
                lse[at] = torch.logsumexp(scores, 1)
                w = torch.exp(scores - lse[at][:, None])
                w = torch.where(seen, w, 0.0)
                value = torch.where(torch.isfinite(vv), vv, 0.0)
                o[at] = w @ value
                hits = seen.double() @ (~torch.isfinite(vv)).double()
                o[at][hits > 0] = math.nan
                none = ~seen.any(1)
                o[at][none] = 0.0
                lse[at][none] = -math.inf
                mean[at] = torch.nan_to_num(w @ value.abs())
                most[at] = ((x.abs() @ torch.nan_to_num(kk, nan=0.0, posinf=0.0, neginf=0.0).abs().T) * scale).masked_fill(~seen, 0.0).amax(1)
                count[at] = seen.sum(1).double()
                top[at] = (seen.double() @ value.abs()) / seen.sum(1, keepdim=True).clamp(min=1)
    return dict(o=o, lse=lse, mean=mean, most=most, count=count, top=top)


def attention_bounds(ref, dtype, D):
    """How far o and lse may be from the reference.  Half a step for the weights (each relative to itself) and for the result; in
    fp16, whose steps end at 2^-24, 2^-25 for each weight of one sequence part whose largest is 1 or more.  fp32: products of 16-bit elements are exact, a sum of D
    of them is off by at most D 2^-24 of the sum of magnitudes, three more roundings scale and shift it; a score's error is the relative one of its weight, and of the
    sum; the hardware's exponential and the sums of n weights add (n + 16) 2^-24."""
    u = torch.finfo(dtype).eps / 2
    scores = ((D + 4) * ref['most'] + ref['lse'].abs().nan_to_num(posinf=0.0, neginf=0.0)) * 2.0 ** -24
    rest = 2 * scores + (ref['count'] + 16) * 2.0 ** -24
    o = 1.01 * u * (ref['o'].abs() + ref['mean']) + rest.unsqueeze(-1) * ref['mean'] + 2.0 ** -126
    if dtype == torch.float16:
        o = o + 2.0 ** -25 * (1 + ref['count'].unsqueeze(-1) * ref['top'])
    return o, rest + 2.0 ** -22 * (1 + ref['lse'].abs().nan_to_num(posinf=0.0, neginf=0.0))


def attention_bounds_by_largest(ref, dtype, D, split=False):
    """As attention_bounds, but for weights that are held as multiples of 2^9 of the row's largest or more: in fp16, whose steps end at 2^-24, what a
    weight loses besides its own half step is at most 2^-25 / 2^9 = 2^-34 of the largest weight, which is no more than the sum of all; and the result itself ends at steps of
    2^-24.  split: weights in two parts of 16 bits, the second of which is off by a half step of what the first leaves, so that the result's own half step is what counts."""
    u = torch.finfo(dtype).eps / 2
    scores = ((D + 4) * ref['most'] + ref['lse'].abs().nan_to_num(posinf=0.0, neginf=0.0)) * 2.0 ** -24
    rest = 2 * scores + (ref['count'] + 16) * 2.0 ** -24
    o = 1.01 * u * (ref['o'].abs() + (u if split else 1.0) * ref['mean']) + rest.unsqueeze(-1) * ref['mean'] + 2.0 ** -126
    if dtype == torch.float16:
        o = o + 2.0 ** -25 + 2.0 ** -34 * ref['count'].unsqueeze(-1) * ref['top']
    return o


def verify(target, draft, drafts, accept, sample, counts=None):
    target, drafts, accept, sample = (t.cpu() for t in (target, drafts, accept, sample))
    B, K = drafts.shape
    V = target.shape[2]
    tokens, accepted = torch.full((B, K + 1), -1, dtype=drafts.dtype), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        count = K if counts is None else min(max(int(counts[b]), 0), K)
        n = 0
        while n < count:
            d = int(drafts[b, n])
            if not 0 <= d < V:
                break
            q = 1.0 if draft is None else float(draft[b, n, d])
            if not float(accept[b, n]) * q < float(target[b, n, d]):
                break
            tokens[b, n] = d
            n += 1
        p = target[b, n].double()
        w = p
        if n < count:
            if draft is None:
                w = p.clone()
                if 0 <= int(drafts[b, n]) < V:
                    w[int(drafts[b, n])] = 0.0
            else:
                w = p - draft[b, n].cpu().double()
            w = torch.where(w > 0, w, 0.0)
            if float(w.sum()) == 0.0:
                w = p
        w = torch.where(w > 0, w, 0.0).tolist()
        aim, at, token, last = float(sample[b]) * math.fsum(w), 0.0, -1, -1
        for t, x in enumerate(w):
            at += x
            if x > 0:
                last = t
                if at > aim and token < 0:
                    token = t
        tokens[b, n] = token if token >= 0 else last
        accepted[b] = n
    return tokens, accepted
