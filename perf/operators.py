"""The operators of serving on a paged cache of keys and values, as workloads with a plain form beside each.

`listed()` gives fixed cases, `draw(rng)` further ones of the same ranges.  For a case, `prepare(case, seed)` makes what
a program holds before the call, `run(state)` makes one pass and returns its outputs: in plain torch operations where
`own` is false, through the package's entry points where it is true.  `work(case)` says what a pass cannot do without and
`exact(case, seed)` what it returns in 64 bits.

The operators:

  write    core.kv_cache_write: the keys and values of new tokens into the pages of a cache, in 8 bits or as they are
  read     core.kv_cache_read: what the cache holds for the last positions of every sequence, as dense rows again
  attend   core.paged_attention: attention of new tokens (one to a whole prompt for each sequence) over the cache
  verify   core.verify_drafts: which drafted tokens the target model accepts, and the token that follows them

A batch is three arrays: `starts` [B + 1] says which rows of the packed tokens are whose, `lens` [B] how long each sequence
is with its new tokens, `table` [B, W] which pages hold it.  Pages are [pages, kv heads, page size, head size]; a cache of 8 bits
has a power of two for each row, kept as its exponent.
"""
from __future__ import annotations

import torch

own = False

TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
CODES = {'e4m3': torch.float8_e4m3fn, 'int8': torch.int8}


def listed():
    return [
        # a decoding step's new keys and values, one row each for 32 sequences: latency
        dict(name='write_token', op='write', B=32, n=1, L=1500, mix='even', Hkv=8, D=128, page=16, type='fp16', cache='e4m3'),
        # a batch of prompts on its way into a cache of 8 bits
        dict(name='write_prompts', op='write', B=4, n=2048, L=6000, mix='ragged', Hkv=8, D=128, page=64, type='bf16', cache='int8'),
        # prefixes of a few sequences taken out of the cache again
        dict(name='read_prefixes', op='read', B=8, n=1000, L=1000, mix='ragged', Hkv=12, D=64, page=32, type='fp16', cache='e4m3'),
        # two long sequences as dense rows
        dict(name='read_long', op='read', B=2, n=30000, L=30000, mix='ragged', Hkv=8, D=128, page=128, type='bf16', cache='int8'),
        # one token each for a few short sequences: latency
        dict(name='attend_token_few', op='attend', B=3, n=1, L=777, mix='ragged', Hq=12, Hkv=12, D=64, page=16, type='fp16', cache='same', window=0, lse=False),
        # a full decoding batch with grouped heads on a cache of 8 bits: bandwidth
        dict(name='attend_token_batch', op='attend', B=64, n=1, L=8192, mix='lens', Hq=32, Hkv=8, D=128, page=64, type='bf16', cache='e4m3', window=0, lse=False),
        # one token of one very long sequence
        dict(name='attend_token_long', op='attend', B=1, n=1, L=131072, mix='even', Hq=16, Hkv=4, D=128, page=256, type='fp16', cache='int8', window=0, lse=True),
        # drafted tokens on their way to verification
        dict(name='attend_drafts', op='attend', B=16, n=5, L=4096, mix='lens', Hq=32, Hkv=8, D=96, page=32, type='fp16', cache='same', window=0, lse=False),
        # one prompt's chunk beside sequences that decode
        dict(name='attend_chunk', op='attend', B=6, n=512, L=16384, mix='mixed', Hq=16, Hkv=4, D=128, page=32, type='bf16', cache='int8', window=0, lse=True),
        # whole prompts
        dict(name='attend_prompts', op='attend', B=4, n=4096, L=4096, mix='ragged', Hq=16, Hkv=16, D=128, page=128, type='fp16', cache='same', window=0, lse=False),
        # drafts of a few sequences: latency
        dict(name='verify_few', op='verify', B=4, K=4, V=32000, type='fp32', short=False),
        # drafts of a full batch over a large vocabulary, some of them cut short
        dict(name='verify_batch', op='verify', B=64, K=7, V=131072, type='fp32', short=True),
    ]


def _log(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return max(low, min(high, round(low * (max(high, low) / low) ** rng.random())))


def draw(rng):
    op = rng.choice(['write', 'read', 'attend', 'attend', 'attend', 'attend', 'verify'])
    if op == 'verify':
        B, K = _log(rng, 1, 64), rng.randint(1, 7)
        return dict(op=op, B=B, K=K, V=_log(rng, 1000, 131072), type=rng.choice(['fp32', 'fp32', 'fp16', 'bf16']), short=rng.random() < 0.5)
    case = dict(op=op, B=_log(rng, 1, 64), n=1, L=1, mix='even', Hkv=rng.choice([1, 2, 4, 8, 12, 16]), D=rng.choice([32, 64, 64, 96, 128, 128]),
                page=rng.choice([16, 32, 64, 128, 256]), type=rng.choice(['fp16', 'bf16']), cache=rng.choice(['same', 'e4m3', 'int8']))
    row = case['B'] * case['Hkv'] * case['D']                     # elements of a position over the batch
    if op != 'attend':
        most = max(1, (1 << 25) // row)
        case['L'] = _log(rng, 1, min(30000, most))
        case['n'] = case['L'] if op == 'read' else _log(rng, 1, case['L'])
        case['mix'] = rng.choice(['even', 'ragged'])
        return case
    case['Hq'] = case['Hkv'] * rng.choice([1, 1, 2, 4, 4, 7, 8])
    case['L'] = _log(rng, 64, min(131072, max(64, (1 << 28) // row)))
    kind = rng.choice(['token', 'drafts', 'chunk'])
    if kind == 'token':
        case['mix'] = rng.choice(['even', 'lens'])
    elif kind == 'drafts':
        case.update(n=rng.randint(2, 8), mix='lens')
    else:
        case['n'] = min(case['L'], _log(rng, 16, 4096))
        case['mix'] = rng.choice(['ragged', 'mixed', 'mixed'])
    case['window'] = 0 if rng.random() < 0.75 else _log(rng, 16, 4096)
    case['lse'] = rng.random() < 0.3
    while work(case)['flops'] > 1.2e11:
        case['n'] = max(1, case['n'] // 2)
        case['L'] = max(case['n'], case['L'] // 2)
    return case


def _lengths(case):
    """How many new tokens each sequence has, and how long it is with them."""
    B, n, L, mix = case['B'], case['n'], case['L'], case['mix']
    share = [1.0 if b == 0 else 0.25 + 0.75 * ((b + 1) * 0.6180339887498949 % 1.0) for b in range(B)]
    if mix == 'even':                                              # all alike
        return [n] * B, [L] * B
    lens = [max(1, round(L * s)) for s in share]
    if mix == 'lens':                                              # lengths as they come, the same number of new tokens
        lens = [max(n, x) for x in lens]
        return [n] * B, lens
    if mix == 'mixed':                                             # one sequence brings a chunk, the others a token each
        return [min(n, lens[0])] + [1] * (B - 1), lens
    new = [max(1, round(n * s)) for s in share]                    # 'ragged': both as they come; every fourth sequence pauses
    new = [0 if b % 4 == 3 else min(x, y) for b, (x, y) in enumerate(zip(new, lens))]
    return new, lens


def _pairs(case):
    """How many (new token, visible position) pairs there are."""
    total = 0
    for n, length in zip(*_lengths(case)):
        for_all = n * (length - n) + n * (n + 1) // 2
        w = case['window']
        if w:
            first = length - n                                     # position of the first new token, which sees first + 1 positions
            whole = max(0, min(n, w - first))                      # new tokens that see fewer than w
            for_all = whole * first + whole * (whole + 1) // 2 + (n - whole) * w
        total += for_all
    return total


def _seen(case):
    """Positions of the cache that some new token sees."""
    w = case['window']
    return sum(0 if n == 0 else length if not w else length - max(0, length - n - w + 1) for n, length in zip(*_lengths(case)))


def work(case):
    if case['op'] == 'verify':
        size = 4 if case['type'] == 'fp32' else 2
        # the rows where a sequence ends: the target's, and the draft's where a token was rejected
        return dict(bytes=2 * case['B'] * case['V'] * size + case['B'] * case['K'] * (2 * size + 20), flops=4 * case['B'] * case['V'])
    wide = 2
    held = wide * case['D'] if case['cache'] == 'same' else case['D'] + 1
    rows = sum(_lengths(case)[0]) * case['Hkv']
    if case['op'] in ('write', 'read'):
        return dict(bytes=2 * rows * (case['D'] * wide + held), flops=2 * rows * case['D'])
    tokens = sum(_lengths(case)[0])
    return dict(bytes=2 * _seen(case) * case['Hkv'] * held + tokens * case['Hq'] * (2 * case['D'] * wide + (4 if case['lse'] else 0)),
                flops=4 * case['D'] * case['Hq'] * _pairs(case))


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device='cuda')


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    if case['op'] == 'verify':
        return _prepare_verify(case, gen)
    B, Hkv, D, page, dtype = case['B'], case['Hkv'], case['D'], case['page'], TYPES[case['type']]
    new, lens = _lengths(case)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    widths = [-(-x // page) for x in lens]
    used = sum(widths)
    order = torch.randperm(used + 3, generator=gen, device='cuda').to(torch.int32)      # three pages are nobody's
    table = torch.zeros((B, max(widths)), dtype=torch.int32, device='cuda')
    at = 0
    for b, w in enumerate(widths):
        table[b, :w] = order[at:at + w]
        at += w
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device='cuda')
    state = dict(case=case, new=new, lengths=lens, table=table, lens=ints(lens), starts=ints(starts), k_exps=None, v_exps=None)
    # keys have channels that differ in size and centre, values do not
    size, centre = torch.exp(0.4 * _normal(gen, 1, Hkv, 1, D)), 0.5 * _normal(gen, 1, Hkv, 1, D)
    pages = used + 3
    step = max(1, (1 << 26) // (Hkv * page * D))
    for name, of in (('k', lambda x: x * size + centre), ('v', lambda x: x)):
        parts, exps = [], []
        for i in range(0, pages, step):
            x = of(_normal(gen, min(step, pages - i), Hkv, page, D)).to(dtype)
            if case['cache'] != 'same':
                x, e = _quantise(x.float(), case['type'], case['cache'])
                exps.append(e)
            parts.append(x)
        state[name + '_pages'] = torch.cat([p.view(torch.uint8) for p in parts]).view(parts[0].dtype)
        if exps:
            state[name + '_exps'] = torch.cat(exps)
    total = starts[-1]
    if case['op'] == 'write':
        state['keys'] = (_normal(gen, total, Hkv, D) * size[:, :, 0] + centre[:, :, 0]).to(dtype)
        state['values'] = _normal(gen, total, Hkv, D).to(dtype)
    elif case['op'] == 'attend':
        state['q'] = _normal(gen, total, case['Hq'], D).to(dtype)
        if own:                                                    # the workspace that such a program keeps
            from fractaltensor_amd import _core as core
            need = core.paged_attention_workspace_bytes(state['q'], state['k_pages'], table, max(new), max(lens), case['window'])
            state['workspace'] = torch.empty(need, dtype=torch.uint8, device='cuda')
    return state


def _prepare_verify(case, gen):
    B, K, V, dtype = case['B'], case['K'], case['V'], TYPES[case['type']]
    logits = 2.5 * _normal(gen, B, K + 1, V)
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :K] + 0.5 * _normal(gen, B, K, V), -1).to(dtype)     # a smaller model's, near the target's
    drafts = torch.searchsorted(draft.double().cumsum(-1), torch.rand((B, K, 1), generator=gen, device='cuda', dtype=torch.float64) * 0.999)
    uniform = lambda *shape: torch.rand(shape, generator=gen, device='cuda')
    counts = None
    if case['short']:
        counts = torch.tensor([(3 * b) % (K + 1) for b in range(B)], dtype=torch.int32, device='cuda')
    return dict(case=case, target=target, draft=draft, drafts=drafts.squeeze(-1).clamp(max=V - 1), accept=uniform(B, K), sample=uniform(B), counts=counts)


def run(state):
    op = state['case']['op']
    if not own:
        return {'write': _plain_write, 'read': _plain_read, 'attend': _plain_attend, 'verify': _plain_verify}[op](state)
    from fractaltensor_amd import _core as core
    s, case = state, state['case']
    if op == 'verify':
        return core.verify_drafts(s['target'], s['draft'], s['drafts'], s['accept'], s['sample'], draft_lens=s['counts'])
    batch = (s['k_pages'], s['v_pages'], s['table'], s['lens'], s['starts'])
    exps = dict(k_exps=s['k_exps'], v_exps=s['v_exps'])
    if op == 'write':
        core.kv_cache_write(s['keys'], s['values'], *batch, **exps)
        return _held(s)
    if op == 'read':
        return core.kv_cache_read(*batch, tokens=sum(s['new']), dtype=TYPES[case['type']], **exps)
    return core.paged_attention(s['q'], *batch, window=case['window'], max_queries=max(s['new']), max_keys=max(s['lengths']), return_lse=case['lse'],
                                workspace=s['workspace'], **exps)


def _held(s):
    return [t for t in (s['k_pages'], s['v_pages'], s['k_exps'], s['v_exps']) if t is not None]


# ---- the plain forms -------------------------------------------------------------------

# the largest code, and how far a row may reach: the largest value of a code that the type it comes from can hold
LARGEST = {'int8': 127.0, 'e4m3': 448.0}
REACH = {('fp16', 'int8'): 127 * 2.0 ** 9, ('fp16', 'e4m3'): 1.875 * 2.0 ** 15, ('bf16', 'int8'): 127 * 2.0 ** 121, ('bf16', 'e4m3'): 1.875 * 2.0 ** 127}
# the least exponent: with fp16 the finest codes are then 2^-24 apart, as its own finest values are
LEAST = {('fp16', 'int8'): -24, ('fp16', 'e4m3'): -15, ('bf16', 'int8'): -100, ('bf16', 'e4m3'): -100}


def _power(e):
    """2^e of whole numbers from -126 to 127, by its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x, kind, cache):
    """Codes and exponents of the rows of x (fp32): the least power of two, from 2^LEAST up, under which a row's largest magnitude is no larger than
    the largest code."""
    x = x.clamp(-REACH[kind, cache], REACH[kind, cache])
    m, e = torch.frexp(x.abs().amax(-1))                           # m in [1/2, 1)
    m_top, e_top = (127 / 128, 7) if cache == 'int8' else (7 / 8, 9)
    least = LEAST[kind, cache]
    e = torch.where(m > 0, e - e_top + (m > m_top), least).clamp(min=least)
    scaled = x * _power(-e).unsqueeze(-1)
    return (scaled.round() if cache == 'int8' else scaled).to(CODES[cache]), e.to(torch.int8)


def _places(s):
    """Of every packed row: its page and its row there."""
    starts, lens = s['starts'].long(), s['lens'].long()
    row = torch.arange(sum(s['new']), device='cuda')
    b = torch.searchsorted(starts[1:], row, right=True)
    position = lens[b] - starts[b + 1] + row
    page = s['case']['page']
    return s['table'].long()[b, position // page], position % page


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _plain_write(s):
    pages, rows = _places(s)
    for name, x in (('k', s['keys']), ('v', s['values'])):
        if s['k_exps'] is not None:
            x, e = _quantise(x.float(), s['case']['type'], s['case']['cache'])
            s[name + '_exps'][pages, :, rows] = e
        _bytes(s[name + '_pages'])[pages, :, rows] = _bytes(x)
    return _held(s)


def _plain_read(s):
    pages, rows = _places(s)
    out = []
    for name in 'kv':
        held = s[name + '_pages']
        x = _bytes(held)[pages, :, rows].view(held.dtype).float()
        if s['k_exps'] is not None:
            x = x * _power(s[name + '_exps'][pages, :, rows]).unsqueeze(-1)
        out.append(x.to(TYPES[s['case']['type']]))
    return out


def _sequence(s, b, name):
    """The keys or values of sequence b, [kv heads, length, head size] in fp32."""
    ids = s['table'][b, :-(-s['lengths'][b] // s['case']['page'])].long()
    held = s[name + '_pages']
    x = _bytes(held)[ids].view(held.dtype).float()
    if s['k_exps'] is not None:
        x = x * _power(s[name + '_exps'][ids]).unsqueeze(-1)
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :s['lengths'][b]]


def _plain_attend(s):
    case = s['case']
    Hq, Hkv, D, dtype = case['Hq'], case['Hkv'], case['D'], TYPES[case['type']]
    out, lse, at = torch.empty_like(s['q']), torch.empty(s['q'].shape[:2], device='cuda'), 0
    for b, (n, length) in enumerate(zip(s['new'], s['lengths'])):
        if n == 0:
            continue
        k, v = _sequence(s, b, 'k'), _sequence(s, b, 'v')
        q = s['q'][at:at + n].float().view(n, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3)                     # [Hkv, G, n, D]
        scores = torch.matmul(q.reshape(Hkv, -1, D), k.transpose(1, 2)).view(Hkv, Hq // Hkv, n, length) * D ** -0.5
        position = torch.arange(length - n, length, device='cuda').unsqueeze(1)
        key = torch.arange(length, device='cuda')
        hidden = key > position
        if case['window']:
            hidden |= key <= position - case['window']
        scores.masked_fill_(hidden, float('-inf'))
        top = scores.amax(-1, keepdim=True)
        weights = torch.exp(scores - top)
        total = weights.sum(-1, keepdim=True)
        o = torch.matmul(weights.view(Hkv, -1, length), v).view(Hkv, Hq // Hkv, n, D) / total
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, Hq, D).to(dtype)
        lse[at:at + n] = (top + torch.log(total)).squeeze(-1).permute(2, 0, 1).reshape(n, Hq)
        at += n
    return (out, lse) if case['lse'] else out


def _plain_verify(s):
    target, draft, drafts = s['target'], s['draft'], s['drafts']
    B, K, V = draft.shape
    counts = s['counts'].long() if s['counts'] is not None else torch.full((B,), K, device='cuda')
    step = torch.arange(K, device='cuda')
    p = target[:, :K].gather(2, drafts.unsqueeze(-1)).squeeze(-1).double()
    q = draft.gather(2, drafts.unsqueeze(-1)).squeeze(-1).double()
    taken = (s['accept'].double() * q < p) & (step < counts.unsqueeze(1))
    accepted = taken.long().cumprod(1).sum(1)
    row = torch.arange(B, device='cuda')
    last = target[row, accepted].double()
    rest = (last - draft[row, accepted.clamp(max=K - 1)].double()).clamp(min=0)
    rejected = (accepted < counts) & (rest.sum(1) > 0)
    weights = torch.where(rejected.unsqueeze(1), rest, last)
    sums = weights.cumsum(1)
    token = (sums <= s['sample'].double().unsqueeze(1) * sums[:, -1:]).sum(1).clamp(max=V - 1)
    tokens = torch.full((B, K + 1), -1, dtype=drafts.dtype, device='cuda')
    tokens[:, :K] = torch.where(step < accepted.unsqueeze(1), drafts, -1)
    tokens[row, accepted] = token
    return tokens, accepted.to(torch.int32)


# ---- in 64 bits ------------------------------------------------------------------------

def _value(code, e, cache):
    """What codes stand for."""
    return code.double() if e is None else code.double() * torch.pow(2.0, e.double()).unsqueeze(-1)


def _rounded(x, kind, cache):
    """Codes (as float64) and exponents of the rows of x (float64), from the definition: the least 2^e that keeps a row within the codes, then the nearest code,
    the even one of two."""
    x = torch.clamp(x, -REACH[kind, cache], REACH[kind, cache])
    big = x.abs().amax(-1)
    e = torch.full_like(big, float(LEAST[kind, cache]))
    e = torch.maximum(e, torch.floor(torch.log2(torch.where(big > 0, big, 1e-300) / LARGEST[cache])))
    e = torch.where(big > LARGEST[cache] * torch.pow(2.0, e), e + 1, e)
    y = x / torch.pow(2.0, e).unsqueeze(-1)
    if cache == 'int8':
        return torch.round(y), e
    grid = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)     # spacing of the codes: 2^-9 from 0 to 2^-6
    return torch.round(y / grid) * grid, e


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'verify':
        return _exact_verify(s)
    new, lens, page = s['new'], s['lengths'], case['page']
    where = []                                                     # of every packed row: (page, row there)
    for b in range(case['B']):
        p = torch.arange(lens[b] - new[b], lens[b], device='cuda')
        where.append(torch.stack([s['table'][b].long()[torch.div(p, page, rounding_mode='floor')], p.remainder(page)]))
    where = torch.cat(where, 1)
    if case['op'] == 'write':
        held, exps = [], []
        for name, x in (('k', s['keys']), ('v', s['values'])):
            pages, e = s[name + '_pages'].double(), s[name + '_exps']
            codes = x.double()
            if e is not None:
                codes, power = _rounded(codes, case['type'], case['cache'])
                e = e.double()
                e[where[0], :, where[1]] = power
                exps.append(e)
            pages[where[0], :, where[1]] = codes
            held.append(pages)
        return held + exps
    if case['op'] == 'read':
        out = []
        for name in 'kv':
            e = s[name + '_exps']
            out.append(_value(_bytes(s[name + '_pages'])[where[0], :, where[1]].view(s[name + '_pages'].dtype), None if e is None else e[where[0], :, where[1]], case['cache']))
        return out
    Hq, Hkv, D = case['Hq'], case['Hkv'], case['D']
    out, lse = torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda'), torch.zeros(s['q'].shape[:2], dtype=torch.float64, device='cuda')
    at = 0
    for b in range(case['B']):
        n, length = new[b], lens[b]
        ids = s['table'][b, :-(-length // page)].long()
        position = torch.arange(length - n, length, device='cuda')
        key = torch.arange(length, device='cuda')
        seen = key[None] <= position[:, None]
        if case['window']:
            seen &= key[None] > position[:, None] - case['window']
        for h in range(Hkv if n else 0):
            k, v = (_value(_bytes(s[x + '_pages'])[ids, h].view(s[x + '_pages'].dtype), None if s[x + '_exps'] is None else s[x + '_exps'][ids, h],
                           case['cache']).reshape(-1, D)[:length] for x in 'kv')
            for head in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                scores = torch.where(seen, s['q'][at:at + n, head].double() @ k.t() / D ** 0.5, float('-inf'))
                lse[at:at + n, head] = torch.logsumexp(scores, 1)
                out[at:at + n, head] = torch.exp(scores - lse[at:at + n, head, None]) @ v
        at += n
    return (out, lse) if case['lse'] else out


def _exact_verify(s):
    K, V = s['draft'].shape[1:]
    tokens, accepted = [], []
    for b in range(s['draft'].shape[0]):
        count = K if s['counts'] is None else int(s['counts'][b])
        ids = s['drafts'][b].tolist()
        j = 0
        while j < count and float(s['accept'][b, j]) * float(s['draft'][b, j, ids[j]]) < float(s['target'][b, j, ids[j]]):
            j += 1
        weights = s['target'][b, j].double()
        if j < count:
            rest = torch.relu(weights - s['draft'][b, j].double())
            weights = rest if float(rest.sum()) > 0 else weights
        sums = weights.cumsum(0)
        token = int(torch.searchsorted(sums, sums[-1:] * s['sample'][b].double(), right=True))
        tokens.append(ids[:j] + [min(token, V - 1)] + [-1] * (K - j))
        accepted.append(j)
    return torch.tensor(tokens, device='cuda'), torch.tensor(accepted, dtype=torch.int32, device='cuda')
