"""Serving with trees of drafts and with caches of limited length against the definitions in 64 bits: attention over a tree, its verification, the weights that positions
gather, selection by them, moving what stays, and runs of them together."""
import math

import pytest
import torch

import serving_reference as base
import tree_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32, E4M3, I8 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8


@pytest.fixture(scope='module')
def core():
    import fractaltensor_amd._core as c
    return c


def _cuda(tensors):
    return [None if t is None else t.cuda() for t in tensors]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device='cuda')


def _bits(t):
    return t.cpu().contiguous().view(torch.uint8)


def _trees(new, seed, kind='any'):
    """Parents of the packed rows of trees of those sizes."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in new:
        for i in range(n):
            if i == 0:
                out.append(-1)
            elif kind == 'chain':
                out.append(i - 1)
            elif kind == 'star':
                out.append(0)
            elif kind == 'forest':
                out.append(-3 if i % 3 == 0 else int(torch.randint(0, i, (1,), generator=g)))
            elif kind == 'wild':                                   # numbers that point nowhere, forward, or at the token itself, too
                out.append(int(torch.randint(-2, 2 * n, (1,), generator=g)))
            else:
                out.append(int(torch.randint(0, i, (1,), generator=g)))
    return out


def _junk_unseen(batch, pages, heads):
    """NaN wherever no position of a sequence lies."""
    used = torch.zeros((batch['pages'], batch['page']), dtype=torch.bool)
    for b, length in enumerate(batch['lens']):
        for p in range(min(length, len(batch['table'][b]) * batch['page'])):
            used[batch['table'][b][p // batch['page']], p % batch['page']] = True
    for t in pages:
        if t is not None:
            raw = t.view(torch.uint8).view(*t.shape[:3], -1) if t.dim() == 4 else t.view(torch.uint8).view(*t.shape, 1)
            raw[~used[:, None, :].expand(-1, heads, -1)] = 0x7f
    return pages


def _tree_case(core, dtype, cache, D, page, heads, G, new, lens, seed, kind='any', window=0, scale=None, tail=0, pages=None, hints=True, workspace=None, parents=None, narrow=None):
    batch = base.make_batch(new, lens, page, seed, tail=tail)
    pages = base.make_pages(batch, heads, D, cache, dtype, seed + 1) if pages is None else pages(batch)
    pages = _junk_unseen(batch, pages, heads)
    parents = _trees(new, seed + 2, kind) if parents is None else parents
    g = torch.Generator().manual_seed(seed + 3)
    q = torch.randn((batch['tokens'], heads * G, D), generator=g).to(dtype)
    if tail:
        q[batch['starts'][-1]:] = math.nan
    scale = D ** -0.5 if scale is None else scale
    dev = _cuda(pages)
    out = torch.full(q.shape, 7.0, dtype=dtype, device='cuda')
    lse = torch.full(q.shape[:2], 7.0, device='cuda')
    most = max(new) if hints else 0
    o, got_lse = core.paged_tree_attention(q.cuda(), *dev[:2], *base.on_device(batch), _ints(parents + [5] * tail), *dev[2:], scale, window, most, max(lens) if hints else 0,
                                           out=out, return_lse=lse, workspace=workspace)
    assert o.data_ptr() == out.data_ptr() and got_lse.data_ptr() == lse.data_ptr()
    k, v = base.held(pages[0], pages[2]), base.held(pages[1], pages[3])
    if dtype == F16:                                               # codes of 8 bits count as what fp16 rounds them to, infinite beyond its largest
        k, v = k.half().double(), v.half().double()
    at = batch['starts']
    want = ref.attention(q[:at[-1]], k, v, batch | dict(tokens=at[-1]), heads, scale, lambda b, n, first, length: ref.tree_sees(parents[at[b]:at[b + 1]], n, first, length, window))
    narrow = (most or batch['tokens']) * G <= 16 if narrow is None else narrow
    bound = base.attention_bounds_by_largest(want, dtype, D, split=narrow)
    lse_bound = base.attention_bounds(want, dtype, D)[1]
    o, got_lse = o.cpu().double(), got_lse.cpu().double()
    assert bool((o[at[-1]:] == 7).all()) and bool((got_lse[at[-1]:] == 7).all())
    o, got_lse = o[:at[-1]], got_lse[:at[-1]]
    assert torch.equal(torch.isnan(o), torch.isnan(want['o']))
    fine = torch.isfinite(want['o'])
    assert bool(((o - want['o']).abs() <= bound)[fine].all()), float(((o - want['o']).abs() / bound)[fine].max())
    none = want['lse'] == -math.inf
    assert torch.equal(got_lse == -math.inf, none)
    fine = torch.isfinite(want['lse'])
    assert bool(((got_lse - want['lse']).abs() <= lse_bound)[fine].all())
    return o


# ---- attention over trees ------------------------------------------------------------------

@pytest.mark.parametrize('kind', ['any', 'chain', 'star', 'forest', 'wild'])
@pytest.mark.parametrize('dtype,cache,D,page,heads,G,new,lens', [
    (F16, None, 64, 16, 3, 1, [1, 7, 0, 16, 3], [1, 300, 40, 16, 50]),
    (BF16, E4M3, 128, 32, 2, 4, [4, 1, 8, 0], [90, 33, 8, 5]),
    (F16, I8, 96, 16, 1, 7, [9, 2, 5], [200, 2, 64]),
    (BF16, None, 32, 64, 2, 2, [32, 31, 1, 17], [32, 95, 1, 400]),
    (F16, E4M3, 128, 16, 1, 1, [64, 63, 5], [64, 190, 150]),
    (BF16, I8, 64, 128, 2, 8, [33, 7, 60, 1], [700, 7, 61, 300]),
    (F16, None, 128, 16, 1, 4, [100, 64, 3, 129], [100, 300, 3, 513]),
    (BF16, None, 96, 32, 2, 1, [256, 1, 65], [256, 400, 90]),
    (F16, I8, 32, 16, 1, 3, [255, 2, 200], [1000, 2, 263]),
])
def test_attention_over_trees(core, kind, dtype, cache, D, page, heads, G, new, lens):
    _tree_case(core, dtype, cache, D, page, heads, G, new, lens, 300, kind, tail=2)


@pytest.mark.parametrize('window', [1, 2, 3, 5, 40, 1000])
@pytest.mark.parametrize('kind', ['any', 'chain', 'forest'])
@pytest.mark.parametrize('dtype,cache,D,page,heads,G,new,lens', [(F16, I8, 64, 16, 2, 2, [16, 1, 9, 0], [60, 30, 9, 4]), (BF16, None, 128, 32, 1, 4, [70, 12, 1], [75, 400, 33])])
def test_windows_over_trees(core, window, kind, dtype, cache, D, page, heads, G, new, lens):
    _tree_case(core, dtype, cache, D, page, heads, G, new, lens, 310, kind, window=window)


@pytest.mark.parametrize('dtype,cache,D,page,heads,G,new,lens,window', [
    (F16, I8, 128, 64, 2, 4, [12], [9000], 0), (BF16, E4M3, 64, 256, 1, 8, [25], [20000], 0), (F16, None, 128, 32, 1, 1, [60, 3], [5000, 7000], 0),
    (BF16, I8, 96, 128, 2, 4, [60], [12000], 5000), (F16, None, 32, 16, 1, 2, [20, 200, 5, 1], [6000, 9000, 4000, 3000], 0)])
def test_trees_behind_long_sequences_in_parts(core, dtype, cache, D, page, heads, G, new, lens, window):
    _tree_case(core, dtype, cache, D, page, heads, G, new, lens, 320, window=window)
    _tree_case(core, dtype, cache, D, page, heads, G, new, lens, 320, window=window, hints=False, workspace=torch.empty(0, dtype=torch.uint8, device='cuda'),
               narrow=sum(new) * G <= 16)


@pytest.mark.parametrize('dtype,cache,D,page,heads,G,new,lens,window', [
    (BF16, E4M3, 64, 64, 3, 8, [(7 * i) % 6 + 1 for i in range(70)], [40 + (1237 * i) % 2600 for i in range(69)] + [3000], 0),
    (F16, None, 32, 32, 2, 8, [60, 0, 33, 5, 1, 40], [5000, 10, 3000, 700, 2500, 64], 0),
    (F16, I8, 128, 16, 1, 4, [30, 32, 9, 1, 0, 17], [4000, 1000, 2500, 30, 7, 3333], 700),
    (BF16, None, 96, 128, 5, 2, [17, 64, 3], [2100, 6000, 129], 0),
    (BF16, I8, 64, 32, 1, 16, [100, 3, 50], [3000, 3500, 2900], 0)])
def test_trees_of_sequences_of_different_lengths_shared_out(core, dtype, cache, D, page, heads, G, new, lens, window):
    """Blocks of rows and sequences that workgroups share, begin and end in: more than 64 of them, several blocks of rows in some and none in others."""
    _tree_case(core, dtype, cache, D, page, heads, G, new, lens, 325, window=window, tail=1)
    _tree_case(core, dtype, cache, D, page, heads, G, new, lens, 325, window=window, workspace=torch.empty(0, dtype=torch.uint8, device='cuda'))


def test_one_graph_for_lengths_that_change(core):
    """The arrays on the device alone say how the work is shared out: each replay against the eager result, with other lengths and numbers of new tokens."""
    heads, G, D, page, most = 2, 4, 64, 32, 40
    g = torch.Generator().manual_seed(340)
    batch = base.make_batch([most] * 4, [6000] * 4, page, 341)
    pages = _cuda(base.make_pages(batch, heads, D, E4M3, BF16, 342))
    table = _ints(batch['table'])
    lens, starts, parents = _ints([6000] * 4), _ints([0, most, 2 * most, 3 * most, 4 * most]), _ints(_trees([most] * 4, 343))
    q = torch.randn((4 * most, heads * G, D), generator=g).to(BF16).cuda()
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device='cuda')
    size = core.paged_tree_attention_workspace_bytes(q, pages[0], table, most, 6000)
    assert size > 0
    space = torch.empty(size, dtype=torch.uint8, device='cuda')
    call = lambda o, z, w: core.paged_tree_attention(q, *pages[:2], table, lens, starts, parents, *pages[2:], max_queries=most, max_keys=6000, out=o, return_lse=z, workspace=w)
    call(out, lse, space)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, lse, space)
    for new, length in (([40, 40, 40, 40], [6000, 6000, 6000, 6000]), ([1, 40, 0, 7], [50, 6000, 3, 4000]), ([40, 5, 5, 5], [40, 5, 5, 5]), ([30, 30, 30, 30], [777, 6000, 5999, 31])):
        at = [0]
        for n in new:
            at.append(at[-1] + n)
        lens.copy_(_ints(length))
        starts.copy_(_ints(at))
        parents[:at[-1]] = _ints(_trees(new, 344))
        out.fill_(7.0)
        lse.fill_(7.0)
        graph.replay()
        o, z = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device='cuda')
        call(o, z, None)
        torch.cuda.synchronize()
        assert torch.equal(_bits(out), _bits(o)) and torch.equal(lse, z) and bool((out[at[-1]:] == 7).all())


@pytest.mark.parametrize('dtype,cache', [(F16, None), (BF16, E4M3)])
def test_a_chain_is_what_a_tree_without_branches_is(core, dtype, cache):
    """What attention of new tokens one behind the other gives.  Trees have their keys summed in another order, and where many rows share a head's keys each weight is
    rounded to 16 bits, at most half a step, eps / 2 of it, in both: the sums differ by at most eps of the same sum over |values|, and their own rounding by eps of
    them, which is less.  (1 % is for sums in fp32.)"""
    for new, lens, G in (([5, 1, 16, 0], [900, 40, 16, 9], 4), ([200, 3, 256], [1500, 60, 300], 2)):
        batch = base.make_batch(new, lens, 32, 330)
        pages = _cuda(base.make_pages(batch, 2, 128, cache, dtype, 331))
        q = torch.randn((batch['tokens'], 2 * G, 128), generator=torch.Generator().manual_seed(332)).to(dtype).cuda()
        sizes = (pages[0], pages[1].float().abs().to(pages[1].dtype))
        for window in (0, 3, 50):
            args = dict(window=window, max_queries=max(new), max_keys=max(lens))
            a = core.paged_attention(q, *pages[:2], *base.on_device(batch), *pages[2:], **args)
            b = core.paged_tree_attention(q, *pages[:2], *base.on_device(batch), _ints(_trees(new, 0, 'chain')), *pages[2:], **args)
            most = core.paged_attention(q, *sizes, *base.on_device(batch), *pages[2:], **args).float()
            assert ((a.float() - b.float()).abs() <= 2.02 * torch.finfo(dtype).eps * most).all()


@pytest.mark.parametrize('dtype,cache,G,new,lens', [(F16, None, 2, [20, 6], [70, 6]), (BF16, E4M3, 4, [60, 2], [200, 31]), (F16, I8, 1, [256], [290])])
def test_what_a_token_does_not_see_of_a_tree_never_matters(core, dtype, cache, G, new, lens):
    """NaN in the values of some tokens, and in the keys of others, reaches their descendants and nobody else."""
    D, page, heads = 64, 16, 1
    chosen = {1: 3, 0: 5}                                          # new token 3's value, new token 5's key

    def pages(batch):
        p = base.make_pages(batch, heads, D, cache, dtype, 341)
        for which, t in chosen.items():
            position = lens[0] - new[0] + t
            at, r = batch['table'][0][position // page], position % page
            if cache == I8:
                p[3 if which else 2][at, 0, r] = 127               # an infinite element in fp16
                p[which][at, 0, r] = 0
                p[which][at, 0, r, 7] = 100
            else:
                p[which][at, 0, r, 7] = math.nan
        return p
    if cache == I8:
        chosen = {1: 3}                                            # (codes of 8 bits have no NaN, and a score of either infinity depends on a sign)
    _tree_case(core, dtype, cache, D, page, heads, G, new, lens, 340, pages=pages)


@pytest.mark.parametrize('dtype,cache,G,new,lens', [(BF16, E4M3, 4, [20, 2], [200, 31]), (F16, I8, 2, [50], [90]), (BF16, None, 1, [200], [300])])
def test_what_a_token_does_not_see_of_other_trees_never_matters(core, dtype, cache, G, new, lens):
    test_what_a_token_does_not_see_of_a_tree_never_matters(core, dtype, cache, G, new, lens)


def test_sequences_that_make_no_sense_beside_one_that_does(core):
    """Lengths past the table's room and below zero, pages that are not there: the work is shared out all the same, and the first sequence has its own results (to the sums'
    order and the weights' rounding, as above)."""
    heads, G, D, page, new = 2, 2, 64, 32, [40, 30, 50]
    batch = base.make_batch(new, [3000] * 3, page, 350)
    pages = _cuda(base.make_pages(batch, heads, D, E4M3, BF16, 351))
    table, lens, starts = base.on_device(batch)
    parents = _ints(_trees(new, 352))
    q = torch.randn((120, heads * G, D), generator=torch.Generator().manual_seed(353)).to(BF16).cuda()
    call = lambda v, t, n, s: core.paged_tree_attention(q, pages[0], v, t, n, s, parents, *pages[2:], max_queries=50, max_keys=3000)
    want, most = call(pages[1], table, lens, starts), call(pages[1].float().abs().to(E4M3), table, lens, starts).float()
    table[1:] = _ints([[(7919 * i) % 2 ** 31 - 2 ** 30 for i in range(table.shape[1])]] * 2)
    for bad_lens, bad_starts in (([3000, 2 ** 31 - 1, -7], [0, 40, 70, 120]), ([3000, 10, 0], [0, 40, 70, 2 ** 31 - 1]), ([3000, -2 ** 31, 5], [0, 40, -3, 1000]), ([3000, 9, 9], [0, 40, 40, 40])):
        got = call(pages[1], table, _ints(bad_lens), _ints(bad_starts))
        assert ((got[:40].float() - want[:40].float()).abs() <= 2.02 * torch.finfo(BF16).eps * most[:40]).all()


def test_trees_on_batches_that_make_no_sense(core):
    """More new tokens than positions, lengths past the table, pages that do not exist: nothing outside is touched, and who is right is served."""
    dtype, D, page, heads, G = F16, 64, 16, 2, 2
    new, lens = [6, 8, 5, 9], [3, 200, 40, 33]
    for most in (9, 100):                                          # both kernels
        batch = base.make_batch(new, [16, 40, 40, 33], page, 350)
        pages = base.make_pages(batch, heads, D, None, dtype, 351)
        parents = _trees(new, 352)
        q = torch.randn((batch['tokens'], heads * G, D), generator=torch.Generator().manual_seed(353)).to(dtype)
        table = [list(r) for r in batch['table']]
        table[2] = [10 ** 9] * len(table[2])
        dev = _cuda(pages)
        guard = torch.full((batch['tokens'] + 8, heads * G, D), 7.0, dtype=dtype, device='cuda')
        out = guard[4:-4]
        o = core.paged_tree_attention(q.cuda(), *dev[:2], _ints(table), _ints(lens), _ints(batch['starts']), _ints(parents), max_queries=most, out=out)
        torch.cuda.synchronize()
        assert bool((guard[:4] == 7).all()) and bool((guard[-4:] == 7).all())
        held = [base.held(p, None) for p in pages[:2]]
        at = batch['starts']
        want = ref.attention(q, *held, batch | dict(lens=lens), heads, D ** -0.5, lambda b, n, first, length: ref.tree_sees(parents[at[b]:at[b + 1]], n, first, length))
        bound = base.attention_bounds_by_largest(want, dtype, D)
        for b in (0, 1, 3):
            rows = slice(at[b], at[b + 1])
            assert bool(((o[rows].cpu().double() - want['o'][rows]).abs() <= bound[rows]).all()), (most, b)
        assert all(torch.equal(x.cpu(), y) for x, y in zip(dev[:2], pages[:2]))


def test_more_new_tokens_than_promised_write_nothing_outside(core):
    dtype, D, page, heads, G = BF16, 64, 16, 1, 4
    batch = base.make_batch([300, 20], [300, 60], page, 360)
    pages = _cuda(base.make_pages(batch, heads, D, None, dtype, 361))
    q = torch.randn((320, G, D), generator=torch.Generator().manual_seed(362)).to(dtype).cuda()
    parents = _ints(_trees([300, 20], 363))
    small = core.paged_tree_attention(q[300:].contiguous(), *pages[:2], _ints(batch['table'][1:]), _ints([60]), _ints([0, 20]), parents[300:].contiguous(), max_queries=20)
    for most in (10, 20, 256):
        guard = torch.full((328, G, D), 7.0, dtype=dtype, device='cuda')
        o = core.paged_tree_attention(q, *pages[:2], *base.on_device(batch), parents, max_queries=most, out=guard[4:-4])
        torch.cuda.synchronize()
        assert bool((guard[:4] == 7).all()) and bool((guard[-4:] == 7).all())
        if most >= 20:
            assert bool(((o[300:] - small).abs().float() <= 2 ** -6 * (1 + small.abs().float())).all())


def test_trees_with_queries_as_views(core):
    joint = torch.randn((21, 10, 64), generator=torch.Generator().manual_seed(370)).to(F16).cuda()
    batch = base.make_batch([5, 16], [40, 33], 16, 371)
    pages = _cuda(base.make_pages(batch, 2, 64, I8, F16, 372))
    parents = _ints(_trees([5, 16], 373))
    for q in (joint[:, 2:8], joint.permute(1, 0, 2).contiguous().permute(1, 0, 2)[:, 4:10]):
        a = core.paged_tree_attention(q, *pages[:2], *base.on_device(batch), parents, *pages[2:], max_queries=16)
        b = core.paged_tree_attention(q.contiguous(), *pages[:2], *base.on_device(batch), parents, *pages[2:], max_queries=16)
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype,cache,D,page,heads,G,new,lens,window', [
    (BF16, E4M3, 128, 64, 2, 4, [16, 9, 3, 0, 5], [900, 2500, 40, 9, 17], 0), (F16, I8, 128, 32, 1, 4, [16], [9000], 0), (BF16, None, 128, 16, 2, 4, [10, 5], [300, 900], 0),
    (F16, None, 64, 32, 1, 2, [32, 1, 20], [400, 50, 33], 7), (BF16, I8, 96, 16, 1, 7, [9, 3], [333, 5000], 0), (F16, E4M3, 32, 128, 2, 1, [64, 40, 17], [64, 3000, 18], 0)])
def test_trees_of_up_to_64_rows_are_off_by_their_own_rounding(core, dtype, cache, D, page, heads, G, new, lens, window):
    """Their weights enter the second product as the rounded one and what that leaves, on either kernel: the bounds are those of few rows."""
    for kind in ('any', 'chain', 'wild'):
        _tree_case(core, dtype, cache, D, page, heads, G, new, lens, 380, kind, window=window, narrow=True)


@pytest.mark.parametrize('dtype,cache,tree', [(BF16, None, 3), (F16, E4M3, 3), (BF16, I8, 3), (BF16, E4M3, 16), (F16, I8, 16), (F16, None, 7)])
def test_a_small_tree_does_not_depend_on_the_trees_beside_it(core, dtype, cache, tree):
    """Trees of 12 to 64 rows alone, and beside one of 40 rows, of 128 and of 256: each is off from the definition by its own rounding alone."""
    heads, G, D, page, length = 2, 4, 64, 32, 700
    for other in (0, 10, 32, 64):
        new, lens = ([tree, other], [length, 1500]) if other else ([tree], [length])
        batch = base.make_batch([tree, 64], [length, 1500], page, 390)
        pages = base.make_pages(batch, heads, D, cache, dtype, 392)
        q = torch.randn((tree + 64, heads * G, D), generator=torch.Generator().manual_seed(391)).to(dtype)
        batch.update(table=batch['table'][:len(new)], lens=lens, starts=[0, tree, tree + other][:len(new) + 1], tokens=sum(new))
        q, parents, dev = q[:sum(new)], _trees(new, 393), _cuda(pages)
        o = core.paged_tree_attention(q.cuda(), *dev[:2], *base.on_device(batch), _ints(parents), *dev[2:], max_queries=max(new), max_keys=max(lens)).cpu().double()
        k, v = base.held(pages[0], pages[2]), base.held(pages[1], pages[3])
        if dtype == F16:
            k, v = k.half().double(), v.half().double()
        at = batch['starts']
        want = ref.attention(q, k, v, batch, heads, D ** -0.5, lambda b, n, first, length: ref.tree_sees(parents[at[b]:at[b + 1]], n, first, length))
        off = (o - want['o']).abs() / base.attention_bounds_by_largest(want, dtype, D, split=True)
        assert bool((off[:tree] <= 1).all()), (other, float(off[:tree].max()))


def test_more_tokens_than_trees_have_are_refused_at_once(core):
    """A large batch whose program does not say how many tokens a sequence has at most: nothing to allocate, and an error."""
    q, pages = torch.zeros((1 << 16, 64, 32), dtype=F16, device='cuda'), torch.zeros((4, 1, 16, 32), dtype=F16, device='cuda')
    table, lens, starts, parents = (torch.zeros(s, dtype=torch.int32, device='cuda') for s in ((4096, 1024), 4096, 4097, 1 << 16))
    assert core.paged_tree_attention_workspace_bytes(q, pages, table) == 0 and core.paged_tree_attention_workspace_bytes(q, pages, table, 257) == 0
    with pytest.raises(core.FtkError, match='256'):
        core.paged_tree_attention(q, pages, pages, table, lens, starts, parents)
    # none of the sequences has any: nothing is written
    out = torch.full_like(q, 7.0)
    core.paged_tree_attention(q, pages, pages, table, lens, starts, parents, max_queries=256, out=out)
    assert bool((out == 7).all())


def test_grids_that_are_too_large_are_refused_by_name(core):
    B, heads = 1 << 20, 4096
    q, pages = torch.zeros((1, heads, 32), dtype=F16, device='cuda'), torch.zeros((1, heads, 16, 32), dtype=F16, device='cuda')
    table, lens, starts, parents = (torch.zeros(s, dtype=torch.int32, device='cuda') for s in ((B, 1), B, B + 1, 1))
    with pytest.raises(core.FtkError, match='ftk_paged_tree_attn: grid too large'):
        core.paged_tree_attention(q, pages, pages, table, lens, starts, parents, max_queries=1)
    with pytest.raises(core.FtkError, match='ftk_paged_attn: grid too large'):
        core.paged_attention(q, pages, pages, table, lens, starts, max_queries=1)


# ---- verification ------------------------------------------------------------------------------

def _verify_case(core, dtype, new, V, M, seed, ids_type=torch.int64, kind='any', shift=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(new)
    parents = _trees(new, seed + 1, kind)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    logits = 2.0 * torch.randn((T, V), generator=g)
    ids = torch.randint(0, V, (T,), generator=g)
    for b, n in enumerate(new):
        for i in range(n):
            p = parents[starts[b] + i]
            if 0 <= p < i:
                logits[starts[b] + p, ids[starts[b] + i]] = math.log(V) + 2.0
    target = torch.softmax(logits, -1).to(dtype)
    uniforms = torch.rand((len(new), M), generator=g)
    buffer = torch.empty(T * V + shift, dtype=dtype, device='cuda')
    t = buffer[shift:].view(T, V)
    t.copy_(target)
    ids = ids.to(ids_type)
    want = ref.verify(target, ids, torch.tensor(parents), starts, uniforms)
    for workspace in (None, torch.empty(0, dtype=torch.uint8, device='cuda')):       # drawn all at once where that is less, and one behind the other
        got = core.verify_tree(t, ids.cuda(), _ints(parents), _ints(starts), uniforms.cuda(), workspace)
        for x, y, name in zip(got, want, ('next', 'path', 'accepted')):
            assert x.dtype == y.dtype and torch.equal(x.cpu(), y), (name, x.cpu(), y)
    return want


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('new,V,M,kind', [([1], 17, 1, 'any'), ([5, 0, 26, 1, 60], 1000, 7, 'any'), ([12, 30], 32000, 5, 'star'), ([9, 8, 7], 4099, 12, 'chain'), ([40, 3], 50257, 6, 'wild'),
                                          ([20] * 5, 1, 4, 'any'), ([64], 131072, 3, 'any'),
                                          ([600, 300], 500, 10, 'any'), ([700], 300, 20, 'star'), ([3, 2], 200003, 4, 'any')])
def test_verified_trees(core, dtype, new, V, M, kind):
    want = _verify_case(core, dtype, new, V, M, 400 + V, kind=kind)
    if V > 1 and M > 2 and max(new) > 8:
        assert int(want[2].max()) > 0                              # (some draft is accepted)


def test_verified_trees_of_narrow_ids_and_at_odd_addresses(core):
    for dtype in (F32, F16, BF16):
        for shift in (1, 2, 3):
            _verify_case(core, dtype, [7, 20], 1001, 6, 410 + shift, ids_type=torch.int32, shift=shift)
            _verify_case(core, dtype, [7, 20], 1000, 6, 420 + shift, ids_type=torch.int32, shift=shift)


def test_verification_at_the_ends_of_its_ranges(core):
    """Rows without a positive weight, with NaN, infinities of the other sign and negative weights; uniforms of zero and next to one; ids outside; two children alike."""
    nan = math.nan
    target = torch.tensor([[0, 0, 0, 0], [nan, -1, 0, 0], [nan, 0.25, -3, 0.75], [0.5, 0.5, 0, 0], [0, 1, 0, 0], [0, 0, 0, 1.0], [1, 0, 0, 0]])
    ids = torch.tensor([-1, 0, 0, 1, 1, 1, 10 ** 12])
    below = 1 - 2.0 ** -24
    for starts, parents, u in (([0, 1, 2, 3], [-1] * 7, [[0.5], [0.5], [0.0]]), ([2, 3, 4, 5], [-1] * 7, [[below], [below], [0.0]]), ([3, 7, 7], [0, 0, 0, -1, 0, 0, 0], [[below, 0.3, 0.1]] * 2)):
        got = core.verify_tree(target.cuda(), ids.cuda(), _ints(parents), _ints(starts), torch.tensor(u).cuda())
        want = ref.verify(target, ids, torch.tensor(parents), starts, torch.tensor(u))
        assert all(torch.equal(x.cpu(), y) for x, y in zip(got, want)), (starts, got, want)
    # starts that point past the rows
    got = core.verify_tree(target.cuda(), ids.cuda(), _ints([-1] * 7), _ints([-5, 3, 100, 90]), torch.rand(3, 2).cuda())
    torch.cuda.synchronize()
    assert got[1][2].tolist() == [-1, -1]
    empty = core.verify_tree(target[:0].cuda(), ids[:0].cuda(), _ints([]), _ints([0, 0]), torch.rand(1, 2).cuda())
    assert [t.tolist() for t in empty] == [[[-1, -1]], [[-1, -1]], [0]]
    none = core.verify_tree(target.cuda(), ids.cuda(), _ints([-1] * 7), _ints([0]), torch.rand(0, 2).cuda())
    assert [tuple(t.shape) for t in none] == [(0, 2), (0, 2), (0,)]


# ---- weighing --------------------------------------------------------------------------------

def _weigh_case(core, dtype, cache, D, page, heads, G, new, lens, seed, causal=True, window=0, decay=1.0, scale=None, tail=0, hints=True, lens_given=None, table_given=None):
    batch = base.make_batch(new, lens, page, seed, tail=tail)
    pages = _junk_unseen(batch, base.make_pages(batch, heads, D, cache, dtype, seed + 1), heads)
    if lens_given:
        batch = batch | dict(lens=lens_given)
    if table_given:
        batch = batch | dict(table=table_given(batch['table']))
    g = torch.Generator().manual_seed(seed + 2)
    q = torch.randn((batch['tokens'], heads * G, D), generator=g).to(dtype)
    weights = torch.rand((batch['pages'], heads, page), generator=g)
    k = base.held(pages[0], pages[2])
    scale = D ** -0.5 if scale is None else scale
    sees = lambda b, n, first, length: ref.causal_sees(n, first, length, causal, window)
    at = batch['starts'][-1]
    lse = torch.full((batch['tokens'], heads * G), math.nan)
    lse[:at] = ref.attention(q[:at], k, k, batch | dict(tokens=at), heads, scale, sees)['lse'].float()
    if tail:
        q[at:] = math.nan
    for b, s, n, first, length in ref.sequences(batch):            # what new positions held does not matter
        for p in range(max(first, 0), length if n else 0):
            t = batch['table'][b][p // page]
            if 0 <= t < batch['pages']:
                weights[t, :, p % page] = math.nan
    dev = _cuda(pages)
    w = weights.cuda()
    core.kv_cache_weigh(q.cuda(), lse.cuda(), dev[0], w, *base.on_device(batch), dev[2], scale, decay, causal, window, max(new) if hints else 0, max(batch['lens']) if hints else 0)
    clean = torch.nan_to_num(weights)
    want, off = ref.weigh(q[:at], lse[:at], k, clean, batch | dict(tokens=at), heads, scale, sees, decay)
    w = w.cpu().double()
    touched = off != 0
    assert torch.equal(_bits(w[~touched].float()), _bits(weights[~touched]))           # all else is as it was
    assert torch.equal(torch.isnan(w[touched]), torch.isnan(want[touched]))              # (keys that are NaN)
    fine = touched & ~torch.isnan(want)
    assert bool(((w - want).abs() <= off)[fine].all()), float(((w - want).abs() / off)[fine].max())
    return w


@pytest.mark.parametrize('decay', [1.0, 0.9, 0.0])
@pytest.mark.parametrize('dtype,cache,D,page,heads,G,new,lens', [
    (F16, None, 64, 16, 3, 1, [1, 1, 0, 1, 2], [1, 300, 40, 16, 50]),
    (BF16, E4M3, 128, 32, 2, 4, [1, 1, 8, 0], [90, 33, 8, 5]),
    (F16, I8, 96, 16, 1, 7, [9, 2, 5], [200, 2, 64]),
    (BF16, None, 32, 64, 2, 2, [32, 31, 1, 70], [32, 95, 1, 400]),
    (F16, E4M3, 32, 16, 1, 3, [64, 63, 5], [64, 190, 150]),
    (BF16, I8, 64, 128, 2, 8, [300, 7, 60, 1], [700, 7, 61, 300]),
    (F16, None, 128, 16, 2, 5, [100, 1, 0, 129], [100, 300, 3, 513]),
    (BF16, None, 96, 1024, 1, 1, [257, 1, 65], [257, 400, 90]),
    (F16, I8, 128, 256, 1, 16, [1, 17], [1500, 600]),
])
def test_weights_that_positions_gather(core, decay, dtype, cache, D, page, heads, G, new, lens):
    _weigh_case(core, dtype, cache, D, page, heads, G, new, lens, 500, decay=decay, tail=2)


@pytest.mark.parametrize('causal,window', [(True, 1), (True, 7), (True, 100), (False, 0), (False, 9)])
@pytest.mark.parametrize('dtype,cache,D,page,G,new,lens', [(F16, I8, 64, 16, 2, [16, 1, 90, 0], [60, 300, 90, 4]), (BF16, None, 128, 32, 4, [70, 12, 1], [75, 400, 33])])
def test_weights_under_windows_and_without_a_causal_mask(core, causal, window, dtype, cache, D, page, G, new, lens):
    _weigh_case(core, dtype, cache, D, page, 2, G, new, lens, 510, causal, window, 0.5)
    _weigh_case(core, dtype, cache, D, page, 2, G, new, lens, 510, causal, window, 1.0, hints=False)


@pytest.mark.parametrize('heads,G,new,lens', [(16, 2, [1] * 20, [700 + 37 * i for i in range(20)]), (32, 1, [200, 1, 1, 150] * 3, [800, 900, 1, 600] * 3)])
def test_weights_of_many_sequences(core, heads, G, new, lens):
    """Where a workgroup has 256 keys."""
    _weigh_case(core, BF16, E4M3, 64, 32, heads, G, new, lens, 520)
    _weigh_case(core, F16, None, 32, 16, heads, G, new, lens, 521, window=300)


def test_weights_where_batches_make_no_sense(core):
    """More new tokens than positions, lengths past the table, pages that do not exist."""
    broken = lambda table: [row if b != 2 else [10 ** 9] + row[1:] for b, row in enumerate(table)]
    _weigh_case(core, F16, None, 64, 16, 2, 2, [6, 3, 1, 9], [16, 40, 40, 33], 530, lens_given=[4, 200, 40, 33], table_given=None)
    w = None
    batch = base.make_batch([1, 1], [40, 40], 16, 531)
    pages = _cuda(base.make_pages(batch, 1, 64, I8, BF16, 532))
    table = broken([batch['table'][0], batch['table'][0], batch['table'][1]])
    weights = torch.full((batch['pages'] + 2, 1, 16), 7.0, device='cuda')
    w = weights[1:-1].contiguous()
    core.kv_cache_weigh(torch.ones((3, 1, 64), dtype=BF16, device='cuda'), torch.zeros((3, 1), device='cuda'), pages[0], w, _ints(table), _ints([0, 0, 40]), _ints([0, 1, 2, 3]), pages[2])
    torch.cuda.synchronize()
    touched = {int(p) for p in torch.nonzero((w != 7).any(2).any(1))}
    assert touched == set(batch['table'][1][1:3])


def test_rows_that_see_nothing_give_nothing(core):
    batch = base.make_batch([2, 1], [40, 20], 16, 540)
    pages = _cuda(base.make_pages(batch, 1, 64, None, F16, 541))
    q = torch.randn((3, 2, 64), generator=torch.Generator().manual_seed(542)).half().cuda()
    _, lse = core.paged_attention(q, *pages[:2], *base.on_device(batch), return_lse=True)
    lse[1] = -math.inf
    w = torch.zeros((batch['pages'], 1, 16), device='cuda')
    core.kv_cache_weigh(q, lse, pages[0], w, *base.on_device(batch))
    one = torch.zeros_like(w)
    core.kv_cache_weigh(q, lse.index_fill(0, _ints([0, 2]).long(), -math.inf), pages[0], one, *base.on_device(batch))
    assert float(one.sum()) == 0.0 and abs(float(w.sum()) - 4.0) < 1e-4          # two rows of two heads, each of which gives one


@pytest.mark.parametrize('dtype', [F16, BF16])
def test_keys_that_are_not_finite_reach_their_own_weight_alone(core, dtype):
    new, lens, page = [20, 1], [70, 33], 16
    batch = base.make_batch(new, lens, page, 550)
    pages = base.make_pages(batch, 1, 64, None, dtype, 551)
    q = torch.randn((21, 2, 64), generator=torch.Generator().manual_seed(552)).to(dtype)
    lse = torch.full((21, 2), 3.0)
    sees = lambda b, n, first, length: ref.causal_sees(n, first, length)
    want, off = ref.weigh(q, lse, base.held(pages[0], None), torch.zeros((batch['pages'], 1, page)), batch, 1, 0.125, sees)
    odd = [(0, 3, math.nan), (0, 69, math.nan), (0, 60, math.inf), (1, 32, math.inf)]
    for b, p, x in odd:
        pages[0][batch['table'][b][p // page], 0, p % page, 5] = x
    w = torch.zeros((batch['pages'], 1, page), device='cuda')
    core.kv_cache_weigh(q.cuda(), lse.cuda(), pages[0].cuda(), w, *base.on_device(batch), scale=0.125)
    w, near = w.cpu().double(), torch.ones(w.shape, dtype=torch.bool)
    for b, p, x in odd:
        at = (batch['table'][b][p // page], 0, p % page)
        near[at] = False
        if x != x:
            assert math.isnan(float(w[at]))
    assert bool(((w - want).abs() <= off + (off == 0) * 0.0)[near].all())


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('new,lens', [([1, 1], [70, 33]), ([20, 1], [70, 33]), ([150, 1], [300, 33]), ([3000, 1], [3000, 33])])
def test_an_infinite_key_makes_nan_or_zero_of_its_weight(core, dtype, new, lens):
    """A score of +inf gives NaN, which selection ranks below everything, and one of -inf nothing: few rows, many, and many in parts."""
    page, D, G, scale = 16, 64, 2, 0.125
    batch = base.make_batch(new, lens, page, 556)
    pages = base.make_pages(batch, 1, D, None, dtype, 557)
    q = torch.randn((sum(new), G, D), generator=torch.Generator().manual_seed(558)).to(dtype)
    q[:, :, 5], q[:, 0, 6], q[:, 1, 6] = 0.75, 0.5, -0.5
    lse = torch.full((sum(new), G), 3.0)
    before = torch.rand((batch['pages'], 1, page), generator=torch.Generator().manual_seed(559))
    sees = lambda b, n, first, length: ref.causal_sees(n, first, length)
    want, off = ref.weigh(q, lse, base.held(pages[0], None), before, batch, 1, scale, sees, 0.5)
    # element 5: all rows score +inf; element 5 negative: all -inf; element 6: of the two heads one each
    odd = [(0, 3, 5, math.inf), (0, lens[0] - 1, 5, math.inf), (1, 32, 5, -math.inf), (0, 17, 5, -math.inf), (0, 40, 6, math.inf), (1, 9, 6, -math.inf)]
    for b, p, e, x in odd:
        at = (batch['table'][b][p // page], 0, p % page)
        pages[0][(*at, e)] = x
        old = p < lens[b] - new[b]
        want[at] = math.nan if x > 0 or e == 6 else 0.5 * float(before[at]) if old else 0.0
    w = before.cuda()
    core.kv_cache_weigh(q.cuda(), lse.cuda(), pages[0].cuda(), w, *base.on_device(batch), scale=scale, decay=0.5, max_queries=max(new), max_keys=max(lens))
    kept = core.kv_cache_select(w, _ints(batch['table']), _ints(lens), 30).cpu()
    w = w.cpu().double()
    assert torch.equal(torch.isnan(w), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert bool(((w - want).abs() <= off)[fine].all())
    for b in (0, 1):
        finite = [p for p in range(lens[b]) if (b, p) not in [o[:2] for o in odd if o[3] > 0 or o[2] == 6]]
        if len(finite) >= 30:
            assert set(kept[b, 0].tolist()) <= set(finite)


# ---- selecting ---------------------------------------------------------------------------------

def _select_case(core, lens, page, heads, budget, sinks, recent, weights, seed, hints=True, table=None):
    batch = base.make_batch([0] * len(lens), lens, page, seed)
    g = torch.Generator().manual_seed(seed + 1)
    w = weights((batch['pages'], heads, page), g)
    table = batch['table'] if table is None else table(batch['table'])
    got = core.kv_cache_select(w.cuda(), _ints(table), _ints(lens), budget, sinks, recent, max(lens) if hints else 0)
    want = ref.select(w, table, lens, page, budget, sinks, recent)
    assert torch.equal(got.cpu(), want), torch.nonzero(got.cpu() != want)[:5]


KINDS = {
    'normal': lambda s, g: torch.exp(2 * torch.randn(s, generator=g)),
    'few values': lambda s, g: torch.randint(0, 4, s, generator=g).float() / 3,
    'all alike': lambda s, g: torch.full(s, 0.25),
    'odd': lambda s, g: torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38, 1.0, -2.5])[torch.randint(0, 10, s, generator=g)],
    'next to each other': lambda s, g: (torch.randint(0, 3000, s, generator=g).to(torch.int32) + 0x3f7ff000).view(torch.float32),
    'all bits': lambda s, g: torch.randint(-2 ** 31, 2 ** 31, s, generator=g).to(torch.int32).view(torch.float32),
}


@pytest.mark.parametrize('kind', sorted(KINDS))
@pytest.mark.parametrize('lens,page,heads,budget,sinks,recent', [
    ([40, 1, 0, 17, 16], 16, 2, 16, 0, 0), ([300, 255, 257, 700], 32, 3, 100, 4, 20), ([1000, 1500, 64], 64, 1, 64, 64, 0), ([1000, 1500, 64], 128, 1, 64, 0, 64),
    ([4096, 4095], 256, 1, 1, 0, 0), ([900], 1024, 1, 899, 3, 5), ([5000, 4097, 3000], 16, 1, 1000, 1, 1), ([1300, 1301], 16, 2, 50, 20, 30)])
def test_selected_positions(core, kind, lens, page, heads, budget, sinks, recent):
    _select_case(core, lens, page, heads, budget, sinks, recent, KINDS[kind], 600)
    _select_case(core, lens, page, heads, budget, sinks, recent, KINDS[kind], 600, hints=False)


@pytest.mark.parametrize('kind', ['normal', 'few values', 'next to each other', 'all bits'])
@pytest.mark.parametrize('lens,budget', [([20000, 16385], 3000), ([70000], 60000), ([131072, 100], 512)])
def test_selected_positions_of_long_sequences(core, kind, lens, budget):
    _select_case(core, lens, 256, 1, budget, 4, 100, KINDS[kind], 610)


@pytest.mark.parametrize('kind', ['normal', 'few values', 'all bits'])
def test_selected_positions_of_the_longest_sequences(core, kind):
    _select_case(core, [524288 + 77, 131073], 1024, 1, 20000, 4, 100, KINDS[kind], 615)


def test_selection_on_tables_that_point_nowhere(core):
    _select_case(core, [300, 100], 16, 2, 90, 2, 3, KINDS['normal'], 620, table=lambda t: [[10 ** 9 if i % 3 == 1 else -5 if i % 3 == 2 else x for i, x in enumerate(row)] for row in t])
    got = core.kv_cache_select(torch.rand((2, 1, 16), device='cuda'), _ints([[0, 1]]), _ints([10 ** 9]), 20)     # a length past the table
    assert got.tolist()[0][0] == sorted(got.tolist()[0][0]) and 0 <= got.min() and got.max() < 32
    assert core.kv_cache_select(torch.rand((2, 1, 16), device='cuda'), _ints([[0, 1]]), _ints([-3]), 4).tolist() == [[[-1] * 4]]
    assert tuple(core.kv_cache_select(torch.rand((2, 3, 16), device='cuda'), torch.empty((0, 2), dtype=torch.int32, device='cuda'), _ints([]), 4).shape) == (0, 3, 4)


# ---- keeping -------------------------------------------------------------------------------------

def _lists(lens, heads, M, seed, share=0.5):
    """Ascending lists of M entries at most, [B, heads, M], those of a sequence of one length."""
    g = torch.Generator().manual_seed(seed)
    kept = torch.full((len(lens), heads, M), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        count = min(M, max(0, round(n * share)))
        for h in range(heads):
            kept[b, h, :count] = torch.randperm(n, generator=g)[:count].sort().values.to(torch.int32)
    return kept


def _keep_case(core, dtype, cache, D, page, heads, lens, kept, seed, starts=None, weights=True):
    batch = base.make_batch([0] * len(lens), lens, page, seed)
    arrays = base.make_pages(batch, heads, D, cache, dtype, seed + 1)
    w = torch.rand((batch['pages'], heads, page), generator=torch.Generator().manual_seed(seed + 2)) if weights else None
    dev = _cuda(arrays + [w])
    firsts = [0] * len(lens) if starts is None else [n - (starts[b + 1] - starts[b]) for b, n in enumerate(lens)]
    got = core.kv_cache_keep(*dev[:2], _ints(batch['table']), _ints(lens), kept.cuda(), None if starts is None else _ints(starts), *dev[2:])
    there = [t for t in arrays + [w] if t is not None]
    want = ref.keep(there, batch['table'], lens, firsts, kept, page)
    assert got.cpu().tolist() == want.tolist()
    for x, y in zip([t for t in dev if t is not None], there):
        assert torch.equal(_bits(x), _bits(y))


@pytest.mark.parametrize('per_head', [True, False])
@pytest.mark.parametrize('dtype,cache,D,page,heads,lens,M,share', [
    (F16, None, 64, 16, 3, [40, 1, 0, 17, 16], 20, 0.5), (BF16, E4M3, 128, 32, 2, [300, 33, 500], 400, 0.7), (F16, I8, 96, 16, 1, [200, 700], 150, 0.9), (BF16, None, 32, 64, 2, [1000, 3], 1000, 1.0),
    (F16, None, 96, 128, 1, [2000, 1500, 1], 1300, 0.6), (BF16, I8, 32, 16, 5, [100, 90], 1, 0.1), (F16, E4M3, 64, 256, 2, [900, 901], 512, 0.3), (BF16, None, 128, 1024, 1, [3000], 2048, 0.95)])
def test_rows_that_stay_move_together(core, per_head, dtype, cache, D, page, heads, lens, M, share):
    kept = _lists(lens, heads, M, 700, share)
    _keep_case(core, dtype, cache, D, page, heads, lens, kept if per_head else kept[:, 0].contiguous(), 701, weights=per_head)


def test_many_sequences_and_heads_move_at_once(core):
    lens = [200 + 11 * i for i in range(24)]
    _keep_case(core, BF16, E4M3, 128, 32, 16, lens, _lists(lens, 16, 256, 710, 0.6), 711)
    _keep_case(core, F16, None, 32, 16, 16, lens, _lists(lens, 16, 500, 712, 0.9), 713, weights=False)


def test_lists_of_thousands_of_rows(core):
    lens = [9000, 2049, 7001]
    _keep_case(core, F16, I8, 64, 64, 2, lens, _lists(lens, 2, 6500, 714, 0.8), 715)


def test_paths_of_trees_move_behind_the_cache(core):
    new, lens = [8, 0, 60, 1, 5], [50, 20, 60, 300, 33]
    starts = [0, 8, 8, 68, 69, 74]
    kept = torch.tensor([[0, 2, 7, -1], [-1] * 4, [0, 1, 2, 3], [0, -1, -1, -1], [0, 3, 4, -1]], dtype=torch.int32)
    for dtype, cache, D, page in ((F16, None, 128, 16), (BF16, I8, 64, 32), (F16, E4M3, 96, 16)):
        _keep_case(core, dtype, cache, D, page, 4, lens, kept, 720, starts)
        _keep_case(core, dtype, cache, D, page, 4, lens, kept[:, None].expand(-1, 4, -1).contiguous(), 721, starts)


def test_keeping_where_lists_make_no_sense(core):
    """Entries past the sequence and pages that do not exist move nothing; lists that do not ascend stay inside; lists of nothing."""
    _keep_case(core, F16, None, 64, 16, 2, [40, 30], torch.tensor([[0, 5, 39, 40, 1000], [1, 29, 30, 10 ** 9, -1]], dtype=torch.int32), 730)
    batch = base.make_batch([0], [40], 16, 731)
    arrays = base.make_pages(batch, 2, 64, None, F16, 732)
    dev = _cuda(arrays)
    core.kv_cache_keep(*dev[:2], _ints([[10 ** 9, -7, batch['table'][0][2]]]), _ints([40]), _ints([[1, 20, 33, 35]]))
    core.kv_cache_keep(*dev[:2], _ints(batch['table']), _ints([-4]), _ints([[0, 1, 2]]))
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(dev[:2], arrays[:2]))
    core.kv_cache_keep(*dev[:2], _ints(batch['table']), _ints([40]), _ints([[39, 3, 3, 0, 17]]))
    spare = [p for p in range(batch['pages']) if p not in batch['table'][0]]
    assert all(torch.equal(_bits(x[spare]), _bits(y[spare])) for x, y in zip(dev[:2], arrays[:2]))
    assert core.kv_cache_keep(*dev[:2], _ints(batch['table']), _ints([40]), torch.empty((1, 0), dtype=torch.int32, device='cuda')).tolist() == [0]
    assert core.kv_cache_keep(*dev[:2], _ints(batch['table']), _ints([40]), torch.empty((1, 0), dtype=torch.int32, device='cuda'), _ints([0, 3])).tolist() == [37]
    assert core.kv_cache_keep(*dev[:2], torch.empty((0, 1), dtype=torch.int32, device='cuda'), _ints([]), torch.empty((0, 3), dtype=torch.int32, device='cuda')).tolist() == []


def test_a_large_cache_past_32_bits(core):
    """Pages of 5 GB: the last ones."""
    heads, D, page = 4, 128, 64
    n = 5 * (1 << 30) // (heads * D * page) + 3
    pages = [torch.empty((n, heads, page, D), dtype=I8, device='cuda') for _ in range(2)]
    exps = [torch.empty((n, heads, page), dtype=I8, device='cuda') for _ in range(2)]
    ids = torch.tensor([n - 1, 0, n - 2], device='cuda')
    g = torch.Generator(device='cuda').manual_seed(740)
    small = [torch.randint(-100, 100, (3, heads, page, D), generator=g, device='cuda').to(I8) for _ in range(2)] + [torch.randint(-8, -4, (3, heads, page), generator=g, device='cuda').to(I8) for _ in range(2)]
    for t, s in zip((*pages, *exps), small):
        t[ids] = s
    weights = torch.zeros((n, heads, page), device='cuda')
    w = torch.zeros((3, heads, page), device='cuda')
    table, near = _ints([[n - 1, 0, n - 2]]), _ints([[0, 1, 2]])
    lens, starts = _ints([150]), _ints([0, 20])
    q = torch.randn((20, 8, D), generator=g, device='cuda').to(BF16)
    parents = _ints(_trees([20], 741))
    a, lse = core.paged_tree_attention(q, *pages, table, lens, starts, parents, *exps, return_lse=True)
    b = core.paged_tree_attention(q, *small[:2], near, lens, starts, parents, *small[2:])
    assert torch.equal(a, b)
    _, lse = core.paged_attention(q, *small[:2], near, lens, starts, *small[2:], return_lse=True)
    core.kv_cache_weigh(q, lse, pages[0], weights, table, lens, starts, exps[0])
    core.kv_cache_weigh(q, lse, small[0], w, near, lens, starts, small[2])
    assert torch.equal(weights[ids], w) and float(w.sum()) > 100
    kept = core.kv_cache_select(weights, table, lens, 70, 2, 8)
    assert torch.equal(kept, core.kv_cache_select(w, near, lens, 70, 2, 8))
    assert core.kv_cache_keep(*pages, table, lens, kept, None, *exps, weights).tolist() == [70]
    core.kv_cache_keep(*small[:2], near, lens, kept, None, *small[2:], w)
    assert all(torch.equal(_bits(t[ids]), _bits(s)) for t, s in zip((*pages, *exps, weights), (*small, w)))


# ---- together ------------------------------------------------------------------------------------

@pytest.mark.parametrize('dtype,cache', [(F16, None), (BF16, E4M3), (F16, I8)])
def test_a_step_with_a_tree(core, dtype, cache):
    """Write a tree's keys and values, attend, verify, keep the path: then a next token sees what a cache of the accepted tokens alone would show it."""
    heads, G, D, page, V = 2, 4, 64, 16, 500
    first, new = [37, 0, 80], [12, 7, 20]
    g = torch.Generator().manual_seed(800)
    batch = base.make_batch(new, [f + n for f, n in zip(first, new)], page, 801, spare=3)
    table, lens, starts = base.on_device(batch)
    pages = _cuda(base.make_pages(batch, heads, D, cache, dtype, 802))
    parents = _trees(new, 803)
    T = sum(new)
    keys, values, q = (torch.randn((T, h, D), generator=g).to(dtype).cuda() for h in (heads, heads, heads * G))
    core.kv_cache_write(keys, values, *pages[:2], table, lens, starts, *pages[2:])
    o = core.paged_tree_attention(q, *pages[:2], table, lens, starts, _ints(parents), *pages[2:], max_queries=20, max_keys=100)
    assert bool(torch.isfinite(o).all())
    logits = torch.randn((T, V), generator=g)
    ids = torch.randint(0, V, (T,), generator=g)
    for b, n in enumerate(new):
        for i in range(1, n):
            logits[batch['starts'][b] + parents[batch['starts'][b] + i], ids[batch['starts'][b] + i]] = 8.0
    target, uniforms = torch.softmax(logits, -1), torch.rand((3, 6), generator=g)
    tokens, path, accepted = core.verify_tree(target.cuda(), ids.cuda(), _ints(parents), starts, uniforms.cuda())
    assert int(accepted.sum()) > 0
    before = [None if t is None else t.clone() for t in pages]
    left = core.kv_cache_keep(*pages[:2], table, lens, path, starts, *pages[2:])
    assert left.tolist() == [f + a + 1 for f, a in zip(first, accepted.tolist())]
    # the same rows written one behind the other into the cache as it was in front of the tree
    rows = torch.cat([batch['starts'][b] + path[b][path[b] >= 0].cpu().long() for b in range(3)])
    counts = [a + 1 for a in accepted.tolist()]
    at = _ints([0, counts[0], counts[0] + counts[1], sum(counts)])
    core.kv_cache_write(keys[rows].contiguous(), values[rows].contiguous(), *before[:2], table, left, at, *before[2:])
    q2, one = torch.randn((3, heads * G, D), generator=g).to(dtype).cuda(), _ints([0, 1, 2, 3])
    a, b = (core.paged_attention(q2, *p[:2], table, left, one, *p[2:], max_queries=1) for p in (pages, before))
    assert torch.equal(a, b)
    # the last accepted token saw what it now sees as the last of its sequence
    for s in range(3):
        last = batch['starts'][s] + int(path[s][counts[s] - 1])
        again = core.paged_attention(q[last:last + 1].contiguous(), *pages[:2], table[s:s + 1].contiguous(), left[s:s + 1].contiguous(), _ints([0, 1]), *pages[2:], max_queries=1)
        assert bool(((again - o[last]).abs().float() <= 4 * torch.finfo(dtype).eps * (1 + o[last].abs().float())).all())


@pytest.mark.parametrize('dtype,cache', [(F16, None), (BF16, I8)])
def test_a_cache_of_limited_length(core, dtype, cache):
    """Tokens one by one, each attended, weighed and, when the budget is passed, what has least weight evicted; against the same in 64 bits with the same choices."""
    heads, G, D, page, budget, sinks, recent = 2, 2, 64, 16, 40, 2, 8
    B, g = 2, torch.Generator().manual_seed(810)
    batch = base.make_batch([0] * B, [64] * B, page, 811)
    table = _ints(batch['table'])
    pages = _cuda(base.make_pages(batch, heads, D, cache, dtype, 812))
    weights = torch.full((batch['pages'], heads, page), math.nan, device='cuda')
    lens, starts = _ints([0] * B), _ints([0, 1, 2])
    held = [[[] for _ in range(heads)] for _ in range(B)]           # (key, value, weight) in 64 bits
    gathered = 0.0
    for step in range(90):
        keys, values, q = (torch.randn((B, h, D), generator=g).to(dtype) for h in (heads, heads, heads * G))
        lens = lens + 1
        core.kv_cache_write(keys.cuda(), values.cuda(), *pages[:2], table, lens, starts, *pages[2:])
        at = core.kv_cache_read(*pages[:2], table, lens, starts, B, F32, *pages[2:])
        o, lse = core.paged_attention(q.cuda(), *pages[:2], table, lens, starts, *pages[2:], max_queries=1, return_lse=True)
        core.kv_cache_weigh(q.cuda(), lse, pages[0], weights, table, lens, starts, pages[2], max_queries=1)
        for b in range(B):
            for h in range(heads):
                held[b][h].append([at[0][b, h].cpu().double(), at[1][b, h].cpu().double(), 0.0])
                k, v = (torch.stack([x[i] for x in held[b][h]]) for i in (0, 1))
                for i in range(G):
                    w = torch.softmax(k @ q[b, h * G + i].double() * D ** -0.5, 0)
                    assert float((o[b, h * G + i].cpu().double() - w @ v).abs().max()) <= 1.1 * torch.finfo(dtype).eps * float((w @ v.abs()).max()) + 1e-5
                    for x, y in zip(held[b][h], w.tolist()):
                        x[2] += y
                got = weights[table[b].long(), h].reshape(-1)[:len(held[b][h])].cpu().double()
                gathered = max(gathered, float((got - torch.tensor([x[2] for x in held[b][h]], dtype=torch.float64)).abs().max()))
        if int(lens.max()) > budget + 12:
            kept = core.kv_cache_select(weights, table, lens, budget, sinks, recent)
            lens = core.kv_cache_keep(*pages[:2], table, lens, kept, None, *pages[2:], weights)
            assert lens.tolist() == [budget] * B
            for b in range(B):
                for h in range(heads):
                    rows = kept[b, h].tolist()
                    assert rows[:sinks] == list(range(sinks)) and rows[-recent:] == list(range(budget + 13 - recent, budget + 13))
                    out = [x[2] for i, x in enumerate(held[b][h]) if i not in rows]
                    inside = [held[b][h][i][2] for i in rows[sinks:-recent]]
                    assert max(out) <= min(inside) + 1e-4          # what goes has least weight
                    held[b][h] = [held[b][h][i] for i in rows]
    # 90 sums of weights that are off by 2^-22 and their scores' error, of a few units each
    assert gathered <= 90 * G * 1e-5


def test_other_streams_and_replays(core):
    """All five on a stream of their own, and captured: each replay against the eager result on new data, with eager work between the replays."""
    dtype, cache, heads, G, D, page, V = F16, I8, 2, 4, 64, 16, 700
    new, lens = [9, 16, 3], [200, 90, 40]
    batch = base.make_batch(new, lens, page, 820)
    table, dlens, starts = base.on_device(batch)
    parents = _ints(_trees(new, 821))
    T = sum(new)
    g = torch.Generator(device='cuda').manual_seed(822)

    def inputs():
        pages = _cuda(base.make_pages(batch, heads, D, cache, dtype, int(torch.randint(0, 10 ** 6, (1,), generator=g, device='cuda'))))
        return dict(q=torch.randn((T, heads * G, D), generator=g, device='cuda').to(dtype), k=pages[0], v=pages[1], ke=pages[2], ve=pages[3],
                    w=torch.rand((batch['pages'], heads, page), generator=g, device='cuda'), p=torch.softmax(torch.randn((T, V), generator=g, device='cuda'), -1),
                    u=torch.rand((3, 5), generator=g, device='cuda'), ids=torch.randint(0, V, (T,), generator=g, device='cuda'))

    def step(x, workspace):
        o, _ = core.paged_tree_attention(x['q'], x['k'], x['v'], table, dlens, starts, parents, x['ke'], x['ve'], max_queries=16, max_keys=200, return_lse=True, workspace=workspace)
        _, lse = core.paged_attention(x['q'], x['k'], x['v'], table, dlens, starts, x['ke'], x['ve'], max_queries=16, max_keys=200, return_lse=True, workspace=workspace)
        core.kv_cache_weigh(x['q'], lse, x['k'], x['w'], table, dlens, starts, x['ke'], max_keys=200)
        tokens, path, accepted = core.verify_tree(x['p'], x['ids'], parents, starts, x['u'])
        left = core.kv_cache_keep(x['k'], x['v'], table, dlens, path, starts, x['ke'], x['ve'], x['w'])
        kept = core.kv_cache_select(x['w'], table, left, 30, 2, 5, max_keys=200)
        last = core.kv_cache_keep(x['k'], x['v'], table, left, kept, None, x['ke'], x['ve'], x['w'])
        return [o, tokens, path, accepted, left, kept, last, x['k'], x['v'], x['ke'], x['ve'], x['w']]

    x = inputs()
    size = core.paged_tree_attention_workspace_bytes(x['q'], x['k'], table, 16, 200)
    workspaces = [torch.empty(max(size, 16) * 4, dtype=torch.uint8, device='cuda') for _ in range(2)]
    copy = lambda d: {n: t.clone() for n, t in d.items()}
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    want = step(copy(x), workspaces[0])
    torch.cuda.synchronize()
    mine = copy(x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(mine, workspaces[1])
    side.synchronize()
    assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(got, want))
    graphs = []
    for i in range(2):
        s = copy(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(s, workspaces[i])
        graphs.append((graph, s, out))
    for r in range(4):
        for graph, s, out in graphs:
            fresh = inputs()
            for n, t in fresh.items():
                s[n].copy_(t)
            graph.replay()
            want = step(copy(fresh), None)
            torch.cuda.synchronize()
            assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(out, want)), r


def test_the_same_call_gives_the_same_bits(core):
    new, lens = [60, 1, 200], [4000, 3000, 900]
    batch = base.make_batch(new, lens, 32, 830)
    at = base.on_device(batch)
    pages = _cuda(base.make_pages(batch, 4, 64, E4M3, BF16, 831))
    q = torch.randn((261, 16, 64), generator=torch.Generator().manual_seed(832)).to(BF16).cuda()
    _, lse = core.paged_attention(q, *pages[:2], *at, *pages[2:], return_lse=True)
    runs = []
    for _ in range(3):
        w = torch.zeros((batch['pages'], 4, 32), device='cuda')
        core.kv_cache_weigh(q, lse, pages[0], w, *at, pages[2], max_keys=4000)
        runs.append((w, core.kv_cache_select(w, at[0], at[1], 500), core.paged_tree_attention(q, *pages[:2], *at, _ints(_trees(new, 833)), *pages[2:], max_queries=200)))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_refusals_on_the_device(core):
    batch = base.make_batch([5, 3], [40, 30], 16, 840)
    table, lens, starts = base.on_device(batch)
    k, v, ke, ve = _cuda(base.make_pages(batch, 2, 64, I8, F16, 841))
    q, parents = torch.zeros((8, 4, 64), dtype=F16, device='cuda'), _ints([-1, 0, 0, 0, 0, -1, 0, 0])
    lse, w = torch.zeros((8, 4), device='cuda'), torch.zeros((batch['pages'], 2, 16), device='cuda')
    tree = lambda **o: core.paged_tree_attention(*[o.get(n, d) for n, d in (('q', q), ('k', k), ('v', v), ('table', table), ('lens', lens), ('starts', starts), ('parents', parents), ('ke', ke), ('ve', ve))],
                                                 **{n: x for n, x in o.items() if n in ('scale', 'window', 'max_queries', 'out', 'return_lse')})
    for error, over in ((ValueError, dict(parents=parents[:7])), (TypeError, dict(parents=parents.long())), (TypeError, dict(parents=None)), (RuntimeError, dict(parents=parents.cpu())),
                        (ValueError, dict(ke=None)), (TypeError, dict(q=q.float())), (ValueError, dict(q=q[:, :, :32])), (ValueError, dict(window=-1)), (core.FtkError, dict(scale=0.0)),
                        (ValueError, dict(max_queries=-1)), (ValueError, dict(starts=starts[:2])), (ValueError, dict(out=q[:7])), (core.FtkError, dict(q=q[:, :3]))):
        with pytest.raises(error):
            tree(**over)
    weigh = lambda **o: core.kv_cache_weigh(*[o.get(n, d) for n, d in (('q', q), ('lse', lse), ('k', k), ('w', w), ('table', table), ('lens', lens), ('starts', starts), ('ke', ke))],
                                            **{n: x for n, x in o.items() if n in ('decay', 'scale', 'window', 'max_keys')})
    for error, over in ((ValueError, dict(lse=lse[:7])), (TypeError, dict(lse=lse.half())), (TypeError, dict(lse=None)), (ValueError, dict(w=w[:1])), (TypeError, dict(w=w.double())), (core.FtkError, dict(decay=1.5)),
                        (core.FtkError, dict(decay=math.nan)), (ValueError, dict(window=-2)), (ValueError, dict(max_keys=1.5)), (ValueError, dict(ke=None)), (RuntimeError, dict(w=w.cpu())),
                        (TypeError, dict(q=q.double())), (ValueError, dict(lse=lse.t().contiguous().t()))):
        with pytest.raises(error):
            weigh(**over)
    select = lambda *a, **o: core.kv_cache_select(o.pop('w', w), o.pop('table', table), o.pop('lens', lens), *a, **o)
    for error, args, over in ((core.FtkError, (0,), {}), (core.FtkError, (4, 3, 2), {}), (ValueError, (-1,), {}), (ValueError, (4, -1), {}), (ValueError, (2.5,), {}), (TypeError, (4,), dict(w=w.double())),
                              (ValueError, (4,), dict(w=w[0])), (ValueError, (4,), dict(lens=lens[:1])), (TypeError, (4,), dict(table=table.long())), (ValueError, (4,), dict(max_keys=-1))):
        with pytest.raises(error):
            select(*args, **over)
    kept = _ints([[0, 2], [0, 1]])
    keep = lambda **o: core.kv_cache_keep(*[o.get(n, d) for n, d in (('k', k), ('v', v), ('table', table), ('lens', lens), ('kept', kept), ('starts', None), ('ke', ke), ('ve', ve), ('w', None))])
    for error, over in ((TypeError, dict(kept=kept.long())), (ValueError, dict(kept=kept[:1])), (ValueError, dict(kept=kept[0])), (ValueError, dict(kept=kept[:, None].expand(2, 3, 2).contiguous())), (ValueError, dict(w=w[:1])),
                        (ValueError, dict(starts=starts[:2])), (ValueError, dict(ke=None)), (TypeError, dict(v=v.short())), (RuntimeError, dict(kept=kept.cpu()))):
        with pytest.raises(error):
            keep(**over)
    p, ids, u = torch.rand((8, 50), device='cuda'), torch.zeros(8, dtype=torch.int64, device='cuda'), torch.rand((2, 3), device='cuda')
    for error, args in ((ValueError, (p, ids[:7], parents, starts, u)), (TypeError, (p.double(), ids, parents, starts, u)), (TypeError, (p, ids.float(), parents, starts, u)),
                        (TypeError, (p, ids, parents.long(), starts, u)), (ValueError, (p, ids, parents, starts, u[:1])), (ValueError, (p.t(), ids, parents, starts, u)),
                        (core.FtkError, (p, ids, parents, starts, torch.rand((2, 65), device='cuda'))), (core.FtkError, (p, ids, parents, starts, u[:, :0])), (RuntimeError, (p, ids, parents, starts, u.cpu()))):
        with pytest.raises(error):
            core.verify_tree(*args)


# ---- FractalTensors --------------------------------------------------------------------------------

@pytest.mark.parametrize('dtype,cache,window', [(F16, I8, 0), (BF16, None, 0), (BF16, E4M3, 20)])
def test_weights_of_an_accepted_path(core, dtype, cache, window):
    """Behind kv_cache_keep a path is a chain: its queries, with what attention over the tree left for them, give the weights of their positions and of all in front."""
    heads, G, D, page, V = 2, 4, 64, 16, 50
    new, lens = [12, 0, 40, 1], [60, 20, 300, 9]
    g = torch.Generator().manual_seed(930)
    batch = base.make_batch(new, lens, page, 931)
    table, dlens, starts = base.on_device(batch)
    pages = _cuda(base.make_pages(batch, heads, D, cache, dtype, 932))
    parents = _ints(_trees(new, 933))
    q = torch.randn((53, heads * G, D), generator=g).to(dtype).cuda()
    _, lse = core.paged_tree_attention(q, *pages[:2], table, dlens, starts, parents, *pages[2:], window=window, max_queries=40, max_keys=300, return_lse=True)
    p, ids = torch.zeros((53, V)), torch.arange(53) % V
    for b, n in enumerate(new):                                    # the way goes on at a node's last child
        for i in range(n):
            children = [c for c in range(n) if int(parents[batch['starts'][b] + c]) == i]
            p[batch['starts'][b] + i, int(ids[batch['starts'][b] + children[-1]]) if children else V - 1] = 1.0
    _, path, accepted = core.verify_tree(p.cuda(), ids.cuda(), parents, starts, torch.rand((4, 8), generator=g).cuda())
    assert int(accepted[0]) > 0 and int(accepted[2]) > 1
    weights = torch.rand((batch['pages'], heads, page), generator=g).cuda()
    left = core.kv_cache_keep(*pages[:2], table, dlens, path, starts, *pages[2:], weights)
    rows = (path + starts[:-1, None])[path >= 0].long()
    count = (path >= 0).sum(1).tolist()
    at = [sum(count[:b]) for b in range(5)]
    before = weights.cpu()
    qp, lp = q[rows].contiguous(), lse[rows].contiguous()
    core.kv_cache_weigh(qp, lp, pages[0], weights, table, left, _ints(at), pages[2], decay=0.5, window=window, max_queries=max(count), max_keys=300)
    k = base.held(pages[0].cpu(), None if pages[2] is None else pages[2].cpu())
    kept = batch | dict(starts=at, lens=left.tolist(), tokens=at[-1])
    sees = lambda b, n, first, length: ref.causal_sees(n, first, length, True, window)
    want, off = ref.weigh(qp, lp, k, before, kept, heads, D ** -0.5, sees, 0.5)
    assert bool(((weights.cpu().double() - want).abs() <= off).all())
    given = ref.weigh(qp, lp, k, torch.zeros_like(before), kept, heads, D ** -0.5, sees)[0].sum()
    exact = ref.attention(qp.cpu(), k.half().double() if dtype == F16 else k, k, kept, heads, D ** -0.5, sees)
    assert bool(((lp.cpu().double() - exact['lse']).abs() <= base.attention_bounds(exact, dtype, D)[1]).all())
    assert abs(float(given) - at[-1] * heads * G) < 1e-3 * at[-1] * heads * G      # each row gives one in all


def test_a_step_with_a_tree_on_fractal_tensors(core):
    from fractaltensor_amd.kaleido import FractalTensor, operations as ops
    heads, G, D, page, V = 2, 2, 64, 16, 300
    new, lens = [9, 0, 4], [50, 20, 4]
    g = torch.Generator().manual_seed(900)
    batch = base.make_batch(new, lens, page, 901)
    table, dlens, starts = base.on_device(batch)
    pages = _cuda(base.make_pages(batch, heads, D, E4M3, F16, 902))
    other = [t.clone() for t in pages]
    parents = _ints(_trees(new, 903))
    ft = lambda t: ops.fused._by_sequence(t, new)
    q = torch.randn((13, heads * G, D), generator=g).half().cuda()
    o = ops.fused.paged_tree_attention(ft(q), ft(parents.reshape(-1, 1)), *pages[:2], table, dlens, *pages[2:], scale=0.2, window=30, max_keys=50)
    assert o.width_by_depth(1) == new
    assert torch.equal(o.data.reshape(13, heads * G, D), core.paged_tree_attention(q, *pages[:2], table, dlens, starts, parents, *pages[2:], 0.2, 30, 9, 50))
    p = torch.softmax(torch.randn((13, V), generator=g), -1).cuda()
    ids, u = torch.randint(0, 4, (13,), generator=g).cuda(), torch.rand((3, 4), generator=g).cuda()
    p[:, 4:] = 0
    drawn, path = ops.fused.verify_tree(ft(p.reshape(13, 1, V)), ft(ids.reshape(-1, 1)), ft(parents.reshape(-1, 1)), u)
    want, where, accepted = core.verify_tree(p, ids, parents, starts, u)
    assert torch.equal(path, where) and drawn.width_by_depth(1) == [int((r >= 0).sum()) for r in want]
    assert torch.equal(drawn.data.reshape(-1), want[want >= 0])
    left = ops.fused.kv_cache_keep(*pages[:2], table, dlens, path, new, *pages[2:])
    assert torch.equal(left, core.kv_cache_keep(*other[:2], table, dlens, where, starts, *other[2:]))
    assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(pages, other))
    with pytest.raises(ValueError, match='tokens a sequence'):
        ops.fused.paged_tree_attention(ft(q), ops.fused._by_sequence(parents.reshape(-1, 1), [13]), *pages[:2], table, dlens, *pages[2:])
    with pytest.raises(TypeError, match='int32 or int64'):
        ops.fused.verify_tree(ft(p.reshape(13, 1, V)), ft(ids.float().reshape(-1, 1)), ft(parents.reshape(-1, 1)), u)
    with pytest.raises(ValueError, match='single integers'):
        ops.fused.verify_tree(ft(p.reshape(13, 1, V)), FractalTensor.from_dense(ids, 1), ft(parents.reshape(-1, 1)), u)
    with pytest.raises(ValueError, match=r'\[1, V\]'):
        ops.fused.verify_tree(ft(p), ft(ids.reshape(-1, 1)), ft(parents.reshape(-1, 1)), u)


def test_parents_past_32_bits_on_fractal_tensors(core):
    """Numbers that wrap to those of earlier tokens point nowhere all the same: their tokens follow the cache itself."""
    from fractaltensor_amd.kaleido import operations as ops
    heads, G, D, page, V, new, lens = 1, 2, 32, 16, 6, [6, 5], [30, 9]
    g = torch.Generator().manual_seed(905)
    batch = base.make_batch(new, lens, page, 906)
    table, dlens, starts = base.on_device(batch)
    pages = _cuda(base.make_pages(batch, heads, D, None, F16, 907))[:2]
    ft = lambda t: ops.fused._by_sequence(t, new)
    q = torch.randn((11, heads * G, D), generator=g).half().cuda()
    wide = torch.tensor([-1, 0, 2 ** 32, 2 ** 32 + 1, 1, 2 ** 33 + 4, -1, 2 ** 32, -2 ** 32, -2 ** 32 + 1, 0])
    none = _ints([-1, 0, -1, -1, 1, -1, -1, -1, -1, -1, 0])
    o = ops.fused.paged_tree_attention(ft(q), ft(wide.reshape(-1, 1).cuda()), *pages, table, dlens, max_keys=30)
    assert torch.equal(o.data.reshape(11, heads * G, D), core.paged_tree_attention(q, *pages, table, dlens, starts, none, scale=1.0, max_queries=6, max_keys=30))
    p, ids, u = torch.full((11, V), 1 / V).cuda(), torch.arange(11).cuda() % V, torch.rand((2, 4), generator=g).cuda()
    _, path = ops.fused.verify_tree(ft(p.reshape(11, 1, V)), ft(ids.reshape(-1, 1)), ft(wide.reshape(-1, 1).cuda()), u)
    assert torch.equal(path, core.verify_tree(p, ids, none, starts, u)[1])


def test_a_cache_of_limited_length_on_fractal_tensors(core):
    from fractaltensor_amd.kaleido import operations as ops
    heads, G, D, page, new, lens = 2, 2, 64, 16, [3, 30], [60, 30]
    batch = base.make_batch(new, lens, page, 910)
    table, dlens, starts = base.on_device(batch)
    pages = _cuda(base.make_pages(batch, heads, D, None, F16, 911))[:2]
    q = torch.randn((33, heads * G, D), generator=torch.Generator().manual_seed(912)).half().cuda()
    weights = torch.rand((batch['pages'], heads, page), generator=torch.Generator().manual_seed(913)).cuda()
    mine = weights.clone()
    o = ops.fused.paged_attention(ops.fused._by_sequence(q, new), *pages, table, dlens, scale=0.2, max_keys=60, weights=weights, decay=0.5)
    want, lse = core.paged_attention(q, *pages, table, dlens, starts, scale=0.2, max_queries=30, max_keys=60, return_lse=True)
    core.kv_cache_weigh(q, lse, pages[0], mine, table, dlens, starts, None, 0.2, 0.5, max_queries=30, max_keys=60)
    assert torch.equal(o.data.reshape(33, heads * G, D), want) and torch.equal(weights, mine)
    kept = ops.fused.kv_cache_select(weights, table, dlens, 25, 2, 5, 60)
    assert torch.equal(kept, core.kv_cache_select(weights, table, dlens, 25, 2, 5))
    assert ops.fused.kv_cache_keep(*pages, table, dlens, kept, weights=weights).tolist() == [25, 25]
