"""Operators of serving with trees of drafted tokens and with caches of limited length, as workloads with a plain form beside each.

`listed()` gives fixed cases, `draw(rng)` further ones of the same ranges.  For a case, `prepare(case, seed)` makes what
a program holds before the call, `run(state)` makes one pass and returns its outputs: in plain torch operations where
`own` is false, through the package's entry points where it is true.  `work(case)` says what a pass cannot do without and
`exact(case, seed)` what it returns in 64 bits.

The operators, all on a paged cache of keys and values:

  tree     core.paged_tree_attention: attention of drafted tokens that form a tree: each sees the cache in front of the tree, its ancestors and itself
  verify   core.verify_tree: the path through such a tree that the target model's own draws follow, and the token behind it
  weigh    core.kv_cache_weigh: the attention weights that new tokens give to each position, added to what the position has gathered before
  select   core.kv_cache_select: which positions of each head stay when a sequence is cut to a budget: first and last ones, and those of most weight
  keep     core.kv_cache_keep: the rows that stay (a path of a tree, or what was selected), moved together in their order

A batch is three arrays: `starts` [B + 1] says which rows of the packed tokens are whose, `lens` [B] how long each sequence
is with its new tokens, `table` [B, W] which pages hold it.  Pages are [pages, kv heads, page size, head size]; a cache of 8 bits
has a power of two for each row, kept as its exponent.  Weights are fp32 [pages, kv heads, page size], one for each row of keys.
"""
from __future__ import annotations

import torch

own = False

TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
CODES = {'e4m3': torch.float8_e4m3fn, 'int8': torch.int8}


def listed():
    return [
        # small trees of a few short sequences: latency
        dict(name='tree_few', op='tree', B=3, n=16, L=777, mix='ragged', Hq=12, Hkv=12, D=64, page=16, type='fp16', cache='same', window=0, lse=False),
        # a full decoding batch with a tree each, grouped heads on a cache of 8 bits
        dict(name='tree_batch', op='tree', B=16, n=60, L=8192, mix='lens', Hq=32, Hkv=8, D=128, page=64, type='bf16', cache='e4m3', window=0, lse=False),
        # a tree at the end of one very long sequence
        dict(name='tree_long', op='tree', B=1, n=25, L=131072, mix='even', Hq=16, Hkv=4, D=128, page=256, type='fp16', cache='int8', window=0, lse=True),
        # which path of a small tree is taken, a few sequences: latency
        dict(name='verify_few', op='verify', B=4, n=25, M=6, V=32000, type='fp32', mix='even'),
        # the same for a full batch over a large vocabulary
        dict(name='verify_batch', op='verify', B=64, n=31, M=8, V=131072, type='bf16', mix='ragged'),
        # weights of one token each of a few short sequences: latency
        dict(name='weigh_few', op='weigh', B=3, n=1, L=777, mix='ragged', Hq=12, Hkv=12, D=64, page=16, type='fp16', cache='same', window=0, decay=1.0),
        # a decoding step of a full batch
        dict(name='weigh_batch', op='weigh', B=64, n=1, L=8192, mix='lens', Hq=32, Hkv=8, D=128, page=64, type='bf16', cache='e4m3', window=0, decay=0.99),
        # whole prompts, whose tokens' weights decide what stays of them
        dict(name='weigh_prompts', op='weigh', B=4, n=4096, L=4096, mix='ragged', Hq=16, Hkv=16, D=128, page=128, type='fp16', cache='same', window=0, decay=1.0),
        # a full batch that has grown past its budget while decoding
        dict(name='select_batch', op='select', B=64, L=1280, mix='lens', Hkv=8, page=64, budget=1024, sinks=4, recent=256),
        # two very long prompts cut down to their budget
        dict(name='select_long', op='select', B=2, L=131072, mix='ragged', Hkv=8, page=256, budget=4096, sinks=16, recent=512),
        # the accepted paths of trees: latency
        dict(name='keep_paths', op='keep', B=32, n=60, L=4096, M=8, mix='lens', of='tree', Hkv=8, D=128, page=32, type='bf16', cache='int8', weights=False),
        # what was selected of a full batch, moved together
        dict(name='keep_selected', op='keep', B=64, n=0, L=2560, M=2048, mix='lens', of='heads', Hkv=8, D=128, page=64, type='bf16', cache='e4m3', weights=True),
    ]


def _log(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return max(low, min(high, round(low * (max(high, low) / low) ** rng.random())))


def draw(rng):
    op = rng.choice(['tree', 'tree', 'tree', 'weigh', 'weigh', 'weigh', 'verify', 'select', 'keep', 'keep'])
    B, page = _log(rng, 1, 64), rng.choice([16, 32, 64, 128, 256])
    if op == 'verify':
        return dict(op=op, B=B, n=_log(rng, 1, 64), M=rng.randint(1, 10), V=_log(rng, 1000, 131072), type=rng.choice(['fp32', 'fp32', 'fp16', 'bf16']),
                    mix=rng.choice(['even', 'ragged']))
    Hkv, D = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([32, 64, 64, 96, 128, 128])
    if op == 'select':
        L = _log(rng, 64, min(131072, (1 << 21) // (B * Hkv)))
        budget = max(4, round(L * rng.uniform(0.03, 0.9)))
        return dict(op=op, B=B, L=L, mix=rng.choice(['even', 'lens', 'ragged']), Hkv=Hkv, page=page, budget=budget, sinks=min(budget // 4, rng.choice([0, 1, 4, 16])),
                    recent=rng.randint(0, budget // 2))
    case = dict(op=op, B=B, n=1, L=1, mix='lens', Hkv=Hkv, D=D, page=page, type=rng.choice(['fp16', 'bf16']), cache=rng.choice(['same', 'e4m3', 'int8']))
    row = B * Hkv * D                                             # elements of a position over the batch
    if op == 'keep':
        case['of'] = rng.choice(['tree', 'heads', 'all'])
        case['L'] = _log(rng, 16, min(30000, max(16, (1 << 27) // row)))
        if case['of'] == 'tree':
            case['n'] = min(case['L'], _log(rng, 1, 64))
            case['M'] = rng.randint(1, min(10, case['n']))
        else:
            case.update(n=0, M=max(1, round(case['L'] * rng.uniform(0.05, 1.0))))
        case['weights'] = rng.random() < 0.5
        return case
    case['Hq'] = Hkv * rng.choice([1, 1, 2, 4, 4, 7, 8])
    case['L'] = _log(rng, 64, min(131072, max(64, (1 << 28) // row)))
    if op == 'tree':
        case.update(n=min(case['L'], _log(rng, 1, 64)), mix=rng.choice(['even', 'lens', 'ragged']))
    elif rng.random() < 0.5:
        case['n'] = rng.choice([1, 1, rng.randint(2, 8)])
    else:
        case.update(n=min(case['L'], _log(rng, 16, 4096)), mix=rng.choice(['ragged', 'mixed']))
    case['window'] = 0 if rng.random() < 0.75 else _log(rng, 16, 4096)
    if op == 'tree':
        case['lse'] = rng.random() < 0.3
    else:
        case['decay'] = rng.choice([1.0, 0.9])
    # no more work, and no more scores at once in the plain form, than the largest listed cases have
    while work(case)['flops'] > 1.2e11 or B * case['Hq'] * case['n'] * case['L'] > 1 << 30:
        case['n'] = max(1, case['n'] // 2)
        case['L'] = max(case['n'], case['L'] // 2)
    return case


def _lengths(case):
    """How many new tokens each sequence has, and how long it is with them."""
    B, n, L, mix = case['B'], case.get('n', 0), case.get('L', 0), case['mix']
    share = [1.0 if b == 0 else 0.25 + 0.75 * ((b + 1) * 0.6180339887498949 % 1.0) for b in range(B)]
    if mix == 'even':                                              # all alike
        return [n] * B, [L] * B
    lens = [max(1, round(L * s)) for s in share]
    if mix == 'lens':                                              # lengths as they come, the same number of new tokens
        lens = [max(n, x) for x in lens]
        return [n] * B, lens
    if mix == 'mixed':                                             # one sequence brings a chunk, the others a token each
        return [min(n, lens[0])] + [1] * (B - 1), lens
    new = [max(1, round(n * s)) if n else 0 for s in share]        # 'ragged': both as they come; every fourth sequence pauses
    if case['op'] != 'verify':
        new = [min(x, y) for x, y in zip(new, lens)]
    return [0 if b % 4 == 3 else x for b, x in enumerate(new)], lens


def _pairs(case):
    """How many (new token, visible position) pairs there are at least."""
    total = 0
    for n, length in zip(*_lengths(case)):
        first, w = length - n, case['window']
        if case['op'] == 'tree':                                   # the prefix and itself
            total += n * (min(first, w - 1) if w else first) + n
            continue
        for_all = n * first + n * (n + 1) // 2
        if w:
            whole = max(0, min(n, w - first))                      # new tokens that see fewer than w
            for_all = whole * first + whole * (whole + 1) // 2 + (n - whole) * w
        total += for_all
    return total


def _seen(case):
    """Positions of the cache that some new token sees."""
    w = case['window']
    return sum(0 if n == 0 else length if not w else length - max(0, length - n - w + 1) for n, length in zip(*_lengths(case)))


def work(case):
    op = case['op']
    new, lens = _lengths(case)
    if op == 'verify':
        # a row where a draw is made: the root's, and one more for each accepted token; a sequence of more than one token accepts about one
        rows = sum(0 if n == 0 else min(2, n, case['M']) for n in new)
        return dict(bytes=rows * case['V'] * (4 if case['type'] == 'fp32' else 2) + sum(new) * 12 + case['B'] * case['M'] * 16, flops=2 * rows * case['V'])
    if op == 'select':
        return dict(bytes=case['Hkv'] * (4 * sum(lens) + 4 * case['B'] * case['budget']), flops=case['Hkv'] * sum(lens))
    held = 2 * case['D'] if case['cache'] == 'same' else case['D'] + 1
    if op == 'keep':
        lists = case['Hkv'] if case['of'] == 'heads' else 1
        moved = sum(min(case['M'], n) - 1 for n in new if n) if case['of'] == 'tree' else sum(min(case['M'], x) if case['M'] < x else 0 for x in lens)
        return dict(bytes=2 * moved * case['Hkv'] * (2 * held + (4 if case['weights'] else 0)) + 4 * case['B'] * case['M'] * lists, flops=0)
    tokens = sum(new)
    if op == 'weigh':
        every = sum(x for n, x in zip(new, lens) if n)
        return dict(bytes=_seen(case) * case['Hkv'] * held + 8 * every * case['Hkv'] + tokens * case['Hq'] * (2 * case['D'] + 4), flops=2 * case['D'] * case['Hq'] * _pairs(case))
    return dict(bytes=2 * _seen(case) * case['Hkv'] * held + tokens * (case['Hq'] * (4 * case['D'] + (4 if case['lse'] else 0)) + 4), flops=4 * case['D'] * case['Hq'] * _pairs(case))


# ---- what a program holds before the call -------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device='cuda')


def _uniform(gen, *shape):
    return torch.rand(shape, generator=gen, device='cuda')


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _starts(new):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return starts


def _parents(gen, new):
    """A tree for each sequence, the parent of each token by its number in the sequence: the first is the root, the others hang on any earlier one."""
    at = torch.cat([torch.arange(n, device='cuda') for n in new])
    return (torch.floor(_uniform(gen, sum(new)) * at).long().clamp(max=at - 1)).to(torch.int32)        # (-1 for the root)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    new, lens = _lengths(case)
    starts = _starts(new)
    s = dict(case=case, starts=_ints(starts), lens=_ints(lens), max_new=max(new), max_len=max(lens), tokens=starts[-1])
    if case['op'] == 'verify':
        return _prepare_verify(s, case, gen, new)
    page = case['page']
    widths = [-(-x // page) for x in lens]
    used = sum(widths)
    order = torch.randperm(used + 3, generator=gen, device='cuda').to(torch.int32)      # three pages are nobody's
    table = torch.zeros((case['B'], max(widths)), dtype=torch.int32, device='cuda')
    at = 0
    for b, w in enumerate(widths):
        table[b, :w] = order[at:at + w]
        at += w
    s['table'] = table
    Hkv, pages = case['Hkv'], used + 3
    if case['op'] == 'select':
        s['weights'] = torch.exp(2 * _normal(gen, pages, Hkv, page))                     # a few positions have most of the weight
        return s
    D, dtype = case['D'], TYPES[case['type']]
    # keys have channels that differ in size and centre, values do not
    size, centre = torch.exp(0.4 * _normal(gen, 1, Hkv, 1, D)), 0.5 * _normal(gen, 1, Hkv, 1, D)
    step = max(1, (1 << 26) // (Hkv * page * D))
    for name, of in (('k', lambda x: x * size + centre), ('v', lambda x: x)):
        parts, exps = [], []
        for i in range(0, pages if name == 'k' or case['op'] != 'weigh' else 0, step):
            x = of(_normal(gen, min(step, pages - i), Hkv, page, D)).to(dtype)
            if case['cache'] != 'same':
                x, e = _codes(x.float(), case['cache'])
                exps.append(e)
            parts.append(x)
        s[name + '_pages'] = torch.cat([p.view(torch.uint8) for p in parts]).view(parts[0].dtype) if parts else None
        s[name + '_exps'] = torch.cat(exps) if exps else None
    if case['op'] == 'keep':
        s['weights'] = torch.exp(2 * _normal(gen, pages, Hkv, page)) if case['weights'] else None
        s['kept'] = _prepare_kept(s, case, gen, new, lens)
        return s
    s['q'] = _normal(gen, starts[-1], case['Hq'], D).to(dtype)
    if case['op'] == 'tree':
        s['parents'] = _parents(gen, new)
    else:
        # what some passes before this one have left
        s['weights'] = torch.exp(_normal(gen, pages, Hkv, page)) * (4 * case['n'] * case['Hq'] / Hkv / case['L'])
        scores = _scores(s)                                        # as the attention in front of the call leaves it
        s['lse'] = _packed(s, torch.logsumexp(scores, -1).unsqueeze(-1)).squeeze(-1).contiguous()
    return s


def _codes(x, cache):
    """Codes and exponents of rows (fp32): the least power of two under which the row's largest is no larger than the largest code."""
    m, e = torch.frexp(x.abs().amax(-1))
    top, bits = (127 / 128, 7) if cache == 'int8' else (7 / 8, 9)
    e = (e - bits + (m > top)).to(torch.int32)
    x = torch.ldexp(x, -e.unsqueeze(-1))
    return (x.round() if cache == 'int8' else x).to(CODES[cache]), e.to(torch.int8)


def _prepare_kept(s, case, gen, new, lens):
    """Which rows stay, in their order, -1 behind them: a root-to-leaf path's numbers, or positions, for each head or for all alike."""
    B, M = case['B'], case['M']
    many = _ints(new if case['of'] == 'tree' else lens).view(B, 1, 1)
    stay = torch.clamp(many, max=M)                                # how many
    lists = case['Hkv'] if case['of'] == 'heads' else 1
    order = _uniform(gen, B, lists, max(new) if case['of'] == 'tree' else max(lens))
    at = torch.arange(order.shape[2], device='cuda')
    order = torch.where(at < many, order, 2.0)
    if case['of'] == 'tree':
        order[:, :, 0] = -1.0                                      # the root stays
    rank = order.argsort(-1).argsort(-1)
    kept = torch.where(rank < stay, at, order.shape[2]).sort(-1).values[:, :, :M]
    kept = torch.cat([kept, torch.full((B, lists, M - kept.shape[2]), order.shape[2], device='cuda')], 2)
    kept = torch.where(kept < order.shape[2], kept, -1).to(torch.int32)
    return kept if case['of'] == 'heads' else kept.squeeze(1)


def _prepare_verify(s, case, gen, new):
    V, T = case['V'], sum(new)
    logits = 2.5 * _normal(gen, T, V)
    s['parents'] = _parents(gen, new)
    s['ids'] = torch.randint(0, V, (T,), generator=gen, device='cuda')
    # a drafted token is about as likely as all that were not drafted together
    begin = torch.repeat_interleave(s['starts'][:-1].long(), torch.tensor(new, device='cuda'))
    child = s['parents'] >= 0
    row = (begin + s['parents'].long())[child]
    logits[row, s['ids'][child]] = torch.logsumexp(logits, -1)[row] + 0.3 * _normal(gen, T)[child]
    s['target'] = torch.softmax(logits, -1).to(TYPES[case['type']])
    s['uniforms'] = _uniform(gen, case['B'], case['M'])
    return s


def run(state):
    op = state['case']['op']
    if not own:
        return {'tree': _plain_tree, 'verify': _plain_verify, 'weigh': _plain_weigh, 'select': _plain_select, 'keep': _plain_keep}[op](state)
    from fractaltensor_amd import _core as core
    s, case = state, state['case']
    if op == 'verify':
        return core.verify_tree(s['target'], s['ids'], s['parents'], s['starts'], s['uniforms'])
    if op == 'select':
        return core.kv_cache_select(s['weights'], s['table'], s['lens'], case['budget'], sinks=case['sinks'], recent=case['recent'], max_keys=s['max_len'])
    if op == 'keep':
        lens = core.kv_cache_keep(s['k_pages'], s['v_pages'], s['table'], s['lens'], s['kept'], starts=s['starts'] if case['of'] == 'tree' else None,
                                  k_exps=s['k_exps'], v_exps=s['v_exps'], weights=s['weights'])
        return _held(s, lens)
    limits = dict(window=case['window'], max_queries=s['max_new'], max_keys=s['max_len'])
    if op == 'weigh':
        core.kv_cache_weigh(s['q'], s['lse'], s['k_pages'], s['weights'], s['table'], s['lens'], s['starts'], k_exps=s['k_exps'], decay=case['decay'], **limits)
        return s['weights']
    return core.paged_tree_attention(s['q'], s['k_pages'], s['v_pages'], s['table'], s['lens'], s['starts'], s['parents'], k_exps=s['k_exps'], v_exps=s['v_exps'],
                                     return_lse=case['lse'], **limits)


def _held(s, lens):
    return [lens] + [t for t in (s['k_pages'], s['v_pages'], s['k_exps'], s['v_exps'], s['weights']) if t is not None]


# ---- the plain forms: all sequences at once, as long as the longest ----------------------

def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _of_positions(s, position):
    """Of positions [B, ..]: their pages and rows there."""
    page, b = s['case']['page'], torch.arange(s['case']['B'], device='cuda').view(-1, *[1] * (position.dim() - 1))
    return s['table'].long()[b, position // page], position % page


def _rows(s, name):
    """Keys or values of all sequences, [B, kv heads, positions, D] in fp32."""
    ids = s['table'].long()
    held = s[name + '_pages']
    x = _bytes(held)[ids].view(held.dtype).float()                 # [B, W, kv heads, page, D]
    if s[name + '_exps'] is not None:
        x = torch.ldexp(x, s[name + '_exps'][ids].to(torch.int32).unsqueeze(-1))
    return x.transpose(1, 2).flatten(2, 3)[:, :, :s['max_len']]


def _packed_rows(s):
    """Of every packed row: its sequence and its number there."""
    row = torch.arange(s['tokens'], device='cuda')
    b = torch.searchsorted(s['starts'][1:].long(), row, right=True)
    return b, row - s['starts'].long()[b]


def _padded(s, x):
    """Packed rows [tokens, ..] -> [B, most new tokens, ..], zeros behind."""
    out = x.new_zeros((s['case']['B'], s['max_new'], *x.shape[1:]))
    out[_packed_rows(s)] = x
    return out


def _packed(s, x):
    """[B, kv heads, group, most new tokens, ..] -> packed rows [tokens, heads, ..]."""
    return x.permute(0, 3, 1, 2, *range(4, x.dim())).flatten(2, 3)[_packed_rows(s)]


def _visible(s):
    """[B, new tokens, positions]: who sees what; for a tree also what lies on the way to its root."""
    case = s['case']
    new = (s['starts'][1:] - s['starts'][:-1]).long().view(-1, 1, 1)
    lens = s['lens'].long().view(-1, 1, 1)
    t, key = torch.arange(s['max_new'], device='cuda').view(1, -1, 1), torch.arange(s['max_len'], device='cuda').view(1, 1, -1)
    first = lens - new
    position = first + t
    if case['op'] != 'tree':
        seen = key <= position
    else:
        parents = _padded(s, s['parents'].long() + 1)              # 0: none
        n = s['max_new'] + 1
        up = torch.nn.functional.one_hot(torch.cat([torch.zeros_like(parents[:, :1]), parents], 1), n).float()
        up[:, 0] = 0                                               # [B, token + 1, its parent + 1]
        reach = torch.eye(n, device='cuda').expand_as(up)
        for _ in range(max(1, (n - 1).bit_length())):              # ways of up to 1, 3, 7, .. steps
            reach = ((reach + torch.matmul(up, reach)) > 0).float()
            up = torch.matmul(up, up)
        reach = reach[:, 1:, 1:]                                   # [B, token, what lies on its way]
        depth = reach.sum(-1).long().unsqueeze(-1) - 1
        position = first + depth
        at = torch.clamp(key - first, 0, s['max_new'] - 1).expand(-1, s['max_new'], -1)
        seen = torch.where(key < first, True, (reach.gather(2, at) > 0) & (key < lens))
        if case['window']:
            place = torch.where(key < first, key, first + depth.transpose(1, 2).gather(2, at[:, :1]))
            seen &= place > position - case['window']
        return seen & (t < new)
    if case['window']:
        seen &= key > position - case['window']
    return seen & (t < new) & (key < lens)


def _scores(s):
    """[B, kv heads, group, new tokens, positions], -inf where a token does not see a position."""
    case = s['case']
    G, Hkv = case['Hq'] // case['Hkv'], case['Hkv']
    q = _padded(s, s['q'].float()).unflatten(2, (Hkv, G)).permute(0, 2, 3, 1, 4)          # [B, kv heads, G, n, D]
    scores = torch.matmul(q.flatten(2, 3), _rows(s, 'k').transpose(2, 3)).unflatten(2, (G, -1)) * case['D'] ** -0.5
    return scores.masked_fill_(~_visible(s)[:, None, None], float('-inf'))


def _plain_tree(s):
    scores = _scores(s)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)           # (rows that are nobody's see nothing)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    o = torch.matmul(weights.flatten(2, 3), _rows(s, 'v')).unflatten(2, weights.shape[2:4]) / total
    o = _packed(s, o).to(s['q'].dtype)
    return (o, _packed(s, top + torch.log(total)).squeeze(-1)) if s['case']['lse'] else o


def _plain_weigh(s):
    scores = _scores(s)
    lse = _padded(s, s['lse']).unflatten(2, (s['case']['Hkv'], -1)).permute(0, 2, 3, 1).unsqueeze(-1)
    added = torch.exp(scores - lse).sum((2, 3))                    # [B, kv heads, positions]
    new, lens = s['starts'][1:] - s['starts'][:-1], s['lens']
    key = torch.arange(s['max_len'], device='cuda')
    pages, rows = _of_positions(s, key.expand(s['case']['B'], -1))
    before = s['weights'][pages, :, rows].transpose(1, 2)          # [B, kv heads, positions]
    total = added + torch.where(key < (lens - new).view(-1, 1, 1), before * s['case']['decay'], 0.0)
    b, at = torch.nonzero((key < lens.unsqueeze(1)) & (new > 0).unsqueeze(1), as_tuple=True)
    s['weights'][pages[b, at], :, rows[b, at]] = total[b, :, at]
    return s['weights']


def _plain_select(s):
    case = s['case']
    key = torch.arange(s['max_len'], device='cuda')
    pages, rows = _of_positions(s, key.expand(case['B'], -1))
    lens = s['lens'].long().view(-1, 1, 1)
    x = s['weights'][pages, :, rows].transpose(1, 2)               # [B, kv heads, positions]
    x = torch.where((key < case['sinks']) | (key >= lens - case['recent']), float('inf'), x)
    x = torch.where(key < lens, x, float('-inf'))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :case['budget']]
    stay = torch.arange(order.shape[-1], device='cuda') < lens
    kept = torch.where(stay, order, s['max_len']).sort(-1).values
    kept = torch.where(kept < s['max_len'], kept, -1).to(torch.int32)
    return torch.nn.functional.pad(kept, (0, case['budget'] - kept.shape[-1]), value=-1)


def _plain_keep(s):
    case = s['case']
    B, Hkv, M = case['B'], case['Hkv'], case['M']
    first = (s['lens'] - (s['starts'][1:] - s['starts'][:-1])).long() if case['of'] == 'tree' else torch.zeros(B, dtype=torch.int64, device='cuda')
    kept = s['kept'].long() if case['of'] == 'heads' else s['kept'].long().unsqueeze(1).expand(-1, Hkv, -1)
    b, h, j = torch.nonzero(kept >= 0, as_tuple=True)
    table, page = s['table'].long(), case['page']
    source, target = first[b] + kept[b, h, j], first[b] + j
    source, target = (table[b, source // page], h, source % page), (table[b, target // page], h, target % page)
    for t in _held(s, None)[1:]:
        _bytes(t)[target] = _bytes(t)[source]
    return _held(s, (first + (kept[:, 0] >= 0).sum(1)).to(torch.int32))


def _plain_verify(s):
    case = s['case']
    B, M = case['B'], case['M']
    starts, parents, ids = s['starts'].long(), s['parents'].long(), s['ids']
    owner, number = _packed_rows(s)
    n = starts[1:] - starts[:-1]
    node = torch.where(n > 0, 0, -1)                               # -1: the way has ended
    tokens, path = torch.full((B, M), -1, dtype=ids.dtype, device='cuda'), torch.full((B, M), -1, dtype=torch.int32, device='cuda')
    for i in range(M):
        at = (starts[:-1] + node).clamp(0, s['tokens'] - 1)
        sums = s['target'][at].double().cumsum(-1)
        token = (sums <= s['uniforms'][:, i:i + 1].double() * sums[:, -1:]).sum(1).clamp(max=case['V'] - 1)
        tokens[:, i] = torch.where(node >= 0, token, -1)
        path[:, i] = node.to(torch.int32)
        follows = (parents == node[owner]) & (node[owner] >= 0) & (ids == token[owner])
        child = torch.full((B,), s['tokens'], device='cuda').scatter_reduce(0, owner, torch.where(follows, number, s['tokens']), 'amin')
        node = torch.where(child < s['tokens'], child, -1)
    return tokens, path, ((path >= 0).sum(1) - 1).clamp(min=0).to(torch.int32)


# ---- in 64 bits ------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {'tree': _exact_attention, 'weigh': _exact_attention, 'verify': _exact_verify, 'select': _exact_select, 'keep': _exact_keep}[case['op']](s)


def _value(s, name, ids, h):
    """What the rows of a head stand for, of the pages `ids` one behind the other."""
    held = s[name + '_pages']
    x = _bytes(held)[ids, h].view(held.dtype).double()
    if s[name + '_exps'] is not None:
        x = x * torch.pow(2.0, s[name + '_exps'][ids, h].double()).unsqueeze(-1)
    return x.reshape(-1, x.shape[-1])


def _exact_attention(s):
    """Attention over trees, or the weights that new tokens give."""
    case = s['case']
    tree, Hkv, D, page, w = case['op'] == 'tree', case['Hkv'], case['D'], case['page'], case['window']
    G = case['Hq'] // Hkv
    starts, lens = s['starts'].tolist(), s['lens'].tolist()
    out, lse = torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda'), torch.zeros(s['q'].shape[:2], dtype=torch.float64, device='cuda')
    weights = None if tree else s['weights'].double()
    up = s['parents'].tolist() if tree else None
    for b in range(case['B']):
        at, n, length = starts[b], starts[b + 1] - starts[b], lens[b]
        if n == 0:
            continue
        first = length - n
        seen = torch.ones((n, length), dtype=torch.bool)
        place, where = torch.arange(n), torch.arange(length)       # of tokens, and of what lies in the cache: how many steps from the first
        if tree:
            seen[:, first:] = False
            for t in range(n):
                way = [t]
                while up[at + way[-1]] >= 0:
                    way.append(up[at + way[-1]])
                seen[t, [first + x for x in way]] = True
                place[t] = len(way) - 1
            where[first:] = first + place
        else:
            seen = where[None] <= first + place[:, None]
        if w:
            seen &= where[None] > first + place[:, None] - w
        seen = seen.cuda()
        ids = s['table'][b, :-(-length // page)].long()
        for h in range(Hkv):
            k = _value(s, 'k', ids, h)[:length]
            v = _value(s, 'v', ids, h)[:length] if tree else None
            given = torch.zeros(length, dtype=torch.float64, device='cuda')
            for head in range(h * G, (h + 1) * G):
                scores = torch.where(seen, s['q'][at:at + n, head].double() @ k.t() / D ** 0.5, float('-inf'))
                if tree:
                    lse[at:at + n, head] = torch.logsumexp(scores, 1)
                    out[at:at + n, head] = torch.exp(scores - lse[at:at + n, head, None]) @ v
                else:
                    given += torch.exp(scores - s['lse'][at:at + n, head, None].double()).sum(0)
            if not tree:
                flat = weights[ids, h].reshape(-1)
                flat[:first] *= case['decay']
                flat[first:length] = 0.0
                flat[:length] += given
                weights[ids, h] = flat.view(-1, page)
    return weights if not tree else (out, lse) if case['lse'] else out


def _exact_verify(s):
    case = s['case']
    starts, up, ids = s['starts'].tolist(), s['parents'].tolist(), s['ids'].tolist()
    tokens, paths, accepted = [], [], []
    for b in range(case['B']):
        got, path = [], []
        node = 0 if starts[b + 1] > starts[b] else -1
        while node >= 0 and len(path) < case['M']:
            path.append(node)
            sums = s['target'][starts[b] + node].double().cumsum(0)
            token = min(int(torch.searchsorted(sums, sums[-1:] * s['uniforms'][b, len(got)].double(), right=True)), case['V'] - 1)
            got.append(token)
            node = next((i for i in range(starts[b + 1] - starts[b]) if up[starts[b] + i] == node and ids[starts[b] + i] == token), -1)
        tokens.append(got + [-1] * (case['M'] - len(got)))
        paths.append(path + [-1] * (case['M'] - len(path)))
        accepted.append(max(0, len(path) - 1))
    return torch.tensor(tokens, device='cuda'), torch.tensor(paths, dtype=torch.int32, device='cuda'), torch.tensor(accepted, dtype=torch.int32, device='cuda')


def _exact_select(s):
    case = s['case']
    out = torch.full((case['B'], case['Hkv'], case['budget']), -1, dtype=torch.int32)
    for b, length in enumerate(s['lens'].tolist()):
        ids = s['table'][b, :-(-length // case['page'])].long()
        for h in range(case['Hkv']):
            x = s['weights'][ids, h].reshape(-1)[:length].cpu()
            low, high = min(case['sinks'], length), max(length - case['recent'], min(case['sinks'], length))
            stay = torch.zeros(length, dtype=torch.bool)
            stay[:low] = True
            stay[high:] = True
            rest = min(case['budget'], length) - int(stay.sum())
            order = torch.argsort(-x[low:high].double(), stable=True)[:rest]
            stay[low + order] = True
            at = torch.nonzero(stay).squeeze(1)
            out[b, h, :len(at)] = at.to(torch.int32)
    return out.cuda()


def _exact_keep(s):
    case = s['case']
    page, starts, lens = case['page'], s['starts'].tolist(), s['lens'].tolist()
    before = _held(s, None)[1:]
    whole = [not t.is_floating_point() for t in before]
    before = [_bytes(t) for t in before]
    after, left = [t.clone() for t in before], []
    for b in range(case['B']):
        first = lens[b] - (starts[b + 1] - starts[b]) if case['of'] == 'tree' else 0
        for h in range(case['Hkv']):
            kept = s['kept'][b, h] if case['of'] == 'heads' else s['kept'][b]
            kept = kept[kept >= 0].long()
            to, source = first + torch.arange(len(kept), device='cuda'), first + kept
            row = lambda p: (s['table'][b].long()[torch.div(p, page, rounding_mode='floor')], p.remainder(page))
            (p, r), (x, y) = row(to), row(source)
            for t, u in zip(after, before):
                t[p, h, r] = u[x, h, y]
        left.append(first + len(kept))
    named = [t.view(u.dtype) for t, u in zip(after, _held(s, None)[1:])]
    return [torch.tensor(left, dtype=torch.int32, device='cuda')] + [t if w else t.double() for t, w in zip(named, whole)]
