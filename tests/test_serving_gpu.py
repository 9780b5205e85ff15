"""The serving kernels against their definitions in 64 bits: writing to and reading from a paged cache, attention over it, verification of drafts,
and a run of them together."""
import math

import pytest
import torch

import serving_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32, E4M3, I8 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8


@pytest.fixture(scope='module')
def core():
    import fractaltensor_amd._core as c
    return c


def _cuda(tensors):
    return [None if t is None else t.cuda() for t in tensors]


def _junk(pages):
    """Fills pages and exponents with what must never matter."""
    for t in pages:
        if t is not None:
            t.view(torch.uint8).fill_(0x7f)                      # NaN in e4m3 and fp16; 2^127 as an exponent
    return pages


def _same(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


# ---- writing and reading -----------------------------------------------------------------

def _rows(kind, n, heads, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, heads, D), generator=g)
    if kind == 'edges':                                          # rows whose largest is at, just above and just below a change of the exponent; ties; ends of the range
        tops = [127.0, 127.25, 126.75, 448.0, 450.0, 446.0, 1.0, 0.0, 2.0 ** -24, 2.0 ** -16, 1e-5, 65504.0, 61440.0, 65024.0, 30000.0, 3e38, 1e-38, 1e-41]
        x = torch.round(x * 8) / 2
        for i in range(n):
            for h in range(heads):
                top = tops[(i * heads + h) % len(tops)]
                if dtype == F16:
                    top = min(top, 65504.0)
                x[i, h] = x[i, h] / 32 * top
                x[i, h, (i + h) % D] = top
    elif kind == 'odd':                                          # infinities and NaN among others
        x[0, 0, 0] = math.inf
        x[n // 2, heads - 1, D - 1] = -math.inf
        x[n - 1, 0, D // 2] = math.nan
        x[n // 3, 0] = math.nan
        x[n // 4, heads - 1] = math.inf
    return x.to(dtype)


@pytest.mark.parametrize('kind', ['normal', 'edges', 'odd'])
@pytest.mark.parametrize('dtype,cache,D,page,heads', [
    (F16, E4M3, 128, 16, 2), (F16, I8, 64, 32, 3), (BF16, E4M3, 32, 64, 1), (BF16, I8, 96, 16, 2), (F16, I8, 128, 256, 1), (BF16, E4M3, 96, 1024, 5),
    (F16, None, 96, 16, 3), (BF16, None, 32, 128, 2),
])
def test_written_rows_are_the_nearest_codes(core, kind, dtype, cache, D, page, heads):
    new, lens = [3, 0, 17, 1, 5], [3, 40, 50, 300, 2]            # the last has three new tokens without a position
    batch = ref.make_batch(new, lens, page, 1, tail=2)
    keys, values = _rows(kind, batch['tokens'], heads, D, dtype, 2), _rows(kind, batch['tokens'], heads, D, dtype, 3)
    pages = ref.make_pages(batch, heads, D, cache, dtype, 4)
    want = [None if t is None else t.clone() for t in pages]
    for x, p, e in ((keys, want[0], want[2]), (values, want[1], want[3])):
        for b in range(len(lens)):
            for row, at, r in ref.places(batch, b):
                for h in range(heads):
                    if cache is None:
                        p[at, h, r] = x[row, h]
                    else:
                        codes, exponent = ref.quantise_row(x[row, h].double(), dtype, cache)
                        p[at, h, r] = torch.tensor(codes, dtype=torch.float64).to(cache)
                        e[at, h, r] = exponent
    pages = _cuda(pages)
    core.kv_cache_write(keys.cuda(), values.cuda(), *pages[:2], *ref.on_device(batch), *pages[2:])
    for got, expected in zip(pages, want):
        if got is None:
            continue
        if cache == E4M3 and got.dtype == E4M3 and kind == 'odd':   # a NaN has two codes
            assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=-1e9), torch.nan_to_num(expected.float(), nan=-1e9))
        else:
            assert _same(got, expected)


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('cache,D,page,heads,came_from', [(E4M3, 128, 16, 2, F16), (I8, 64, 32, 3, F16), (E4M3, 32, 64, 1, F16), (I8, 96, 256, 2, F16), (None, 128, 32, 2, F16),
                                                        (None, 96, 16, 3, BF16)])
def test_read_rows_are_what_the_codes_stand_for(core, dtype, cache, D, page, heads, came_from):
    if cache is None and dtype not in (came_from, F32):
        pytest.skip('pages of 16 bits are read in their type or in fp32')
    new, lens = [7, 0, 64, 1, 5], [7, 40, 64, 300, 2]
    batch = ref.make_batch(new, lens, page, 5, tail=3)
    pages = ref.make_pages(batch, heads, D, cache, came_from, 6)
    want = [ref.held(pages[0], pages[2]).to(dtype), ref.held(pages[1], pages[3]).to(dtype)]
    pages = _cuda(pages)
    out = [torch.full((batch['tokens'], heads, D), 7.0, dtype=dtype, device='cuda') for _ in range(2)]
    got = core.kv_cache_read(*pages[:2], *ref.on_device(batch), batch['tokens'], dtype, *pages[2:], out=tuple(out))
    assert got[0].data_ptr() == out[0].data_ptr()
    for x, w in zip(got, want):
        expected = torch.full((batch['tokens'], heads, D), 7.0, dtype=dtype)
        expected[:batch['starts'][-1]] = 0.0                      # positions below zero are read as zeros
        for b in range(len(lens)):
            for row, at, r in ref.places(batch, b):
                expected[row] = w[at, :, r]
        assert torch.equal(x.cpu(), expected)


@pytest.mark.parametrize('cache', [E4M3, I8])
@pytest.mark.parametrize('dtype', [F16, BF16, F32])
def test_read_rows_under_any_exponent(core, cache, dtype):
    """Every signed byte for an exponent, once with each code: the product, rounded once, infinite beyond the type's largest."""
    batch = ref.make_batch([256], [256], 256, 171, spare=0)
    codes = torch.arange(256, dtype=torch.uint8)
    if cache == E4M3:
        codes[0x7f], codes[0xff] = 0, 0                            # NaN
    pages = [codes.view(cache).view(2, 1, 128).expand(2, 256, 128).contiguous().view(1, 2, 256, 128) for _ in range(2)]
    exps = [torch.arange(-128, 128).to(torch.int8).view(1, 1, 256).expand(1, 2, 256).contiguous() for _ in range(2)]
    got = core.kv_cache_read(*_cuda(pages), *ref.on_device(batch), 256, dtype, *_cuda(exps))
    want = ref.held(pages[0], exps[0])[0].transpose(0, 1).float().to(dtype)      # exact in fp32 where it is not beyond it
    assert torch.equal(got[0].cpu(), want) and torch.equal(got[1].cpu(), want)


def test_rows_of_a_joint_projection_are_written_in_place(core):
    """Views of one [tokens, query + key + value heads, D] product, and of one with the heads outermost."""
    heads, D, page = 2, 64, 16
    batch = ref.make_batch([5, 9], [20, 9], page, 7)
    joint = torch.randn((batch['tokens'], 4 + 2 * heads, D), generator=torch.Generator().manual_seed(8)).to(BF16).cuda()
    for k, v in ((joint[:, 4:6], joint[:, 6:8]), (joint.permute(1, 0, 2).contiguous().permute(1, 0, 2)[:, 4:6], joint[:, 6:8])):
        first, second = (_cuda(ref.make_pages(batch, heads, D, I8, BF16, 9)) for _ in range(2))
        core.kv_cache_write(k, v, *first[:2], *ref.on_device(batch), *first[2:])
        core.kv_cache_write(k.contiguous(), v.contiguous(), *second[:2], *ref.on_device(batch), *second[2:])
        assert all(_same(a, b) for a, b in zip(first, second))


def test_a_large_cache_is_written_and_read_past_32_bits(core):
    """Pages of 5 GB: the last ones."""
    heads, D, page = 4, 128, 64
    n = 5 * (1 << 30) // (heads * D * page) + 3
    pages = [torch.empty((n, heads, page, D), dtype=I8, device='cuda') for _ in range(2)]
    exps = [torch.empty((n, heads, page), dtype=I8, device='cuda') for _ in range(2)]
    table = torch.tensor([[n - 1, 0, n - 2]], dtype=torch.int32, device='cuda')
    lens, starts = torch.tensor([150], dtype=torch.int32, device='cuda'), torch.tensor([0, 150], dtype=torch.int32, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(10)
    keys, values, q = (torch.randn((150, h, D), generator=g, device='cuda').to(BF16) for h in (heads, heads, 8))
    core.kv_cache_write(keys, values, *pages, table, lens, starts, *exps)
    k, v = core.kv_cache_read(*pages, table, lens, starts, 150, F32, *exps)
    for got, x in ((k, keys.float()), (v, values.float())):
        step = 2.0 ** torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 127))
        assert bool(((got - x).abs() <= step / 2).all())
    small_table = torch.arange(3, dtype=torch.int32, device='cuda')[None]
    small = [t[torch.tensor([n - 1, 0, n - 2], device='cuda')].contiguous() for t in (*pages, *exps)]
    for hint in (0, 150):                                          # and both kernels of attention
        got = core.paged_attention(q, *pages, table, lens, starts, *exps, max_queries=hint)
        assert torch.equal(got, core.paged_attention(q, *small[:2], small_table, lens, starts, *small[2:], max_queries=hint))
    one = torch.tensor([0, 1], dtype=torch.int32, device='cuda')
    assert torch.equal(core.paged_attention(q[:1].contiguous(), *pages, table, lens, one, *exps, max_queries=1),
                       core.paged_attention(q[:1].contiguous(), *small[:2], small_table, lens, one, *small[2:], max_queries=1))


@pytest.mark.parametrize('dtype,cache,D,page,heads', [(F16, None, 128, 32, 12), (BF16, I8, 128, 16, 3), (F16, E4M3, 96, 64, 40), (BF16, E4M3, 64, 128, 7), (F16, I8, 32, 16, 5), (BF16, None, 64, 16, 1)])
def test_many_rows_at_once_are_those_of_few(core, dtype, cache, D, page, heads):
    """Long prompts among short ones, pauses and sequences of no length, in one call: the bytes that a call for each piece of ten tokens leaves and reads."""
    new = [700, 0, 1, 3000, 0, 0, 17, 1, 1, 1, 900, 0] * (6 if heads < 6 else 2) + [2000] * (12 if heads == 1 else 0)
    batch = ref.make_batch(new, [n + (5 * b) % 40 for b, n in enumerate(new)], page, 181, tail=3)
    table, lens, starts = ref.on_device(batch)
    a, b = (_junk(_cuda(ref.make_pages(batch, heads, D, cache, dtype, 182))) for _ in range(2))
    g = torch.Generator(device='cuda').manual_seed(183)
    keys, values = ((torch.randn((batch['tokens'], heads, D), generator=g, device='cuda') * torch.rand((batch['tokens'], heads, 1), generator=g, device='cuda') * 8).to(dtype) for _ in range(2))
    core.kv_cache_write(keys, values, *a[:2], table, lens, starts, *a[2:])
    k, v = (torch.full((batch['tokens'], heads, D), 7.0, device='cuda') for _ in range(2))
    core.kv_cache_read(*a[:2], table, lens, starts, batch['tokens'], F32, *a[2:], out=(k, v))
    ends = batch['starts'][-1]
    assert bool((k[ends:] == 7).all()) and bool((v[ends:] == 7).all())
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device='cuda')
    for s, n in enumerate(new):
        for t in range(0, n, max(10, n // 20)):
            m, at = min(max(10, n // 20), n - t), batch['starts'][s] + t
            one = (table[s:s + 1], ints([batch['lens'][s] - n + t + m]), ints([0, m]))
            core.kv_cache_write(keys[at:at + m].contiguous(), values[at:at + m].contiguous(), *b[:2], *one, *b[2:])
            few = core.kv_cache_read(*a[:2], *one, m, F32, *a[2:])
            assert torch.equal(few[0], k[at:at + m]) and torch.equal(few[1], v[at:at + m]), (s, t)
    assert all(x is None or _same(x, y) for x, y in zip(a, b))


# ---- attention --------------------------------------------------------------------------

def _attention_case(core, dtype, cache, D, page, heads, G, new, lens, seed, causal=True, window=0, hints=True, scale=None, tail=0, junk=True, workspace=None, pages=None):
    batch = ref.make_batch(new, lens, page, seed, tail=tail)
    if pages is None:
        pages = ref.make_pages(batch, heads, D, cache, dtype, seed + 1)
    if junk:                                                       # what no position of a sequence holds must not matter
        used = torch.zeros(pages[0].shape[:3], dtype=torch.bool)
        for b, n in enumerate(lens):
            for p in range(min(n, len(batch['table'][b]) * page)):
                used[batch['table'][b][p // page], :, p % page] = True
        for t in pages[:2]:
            t.view(torch.uint8).view(*used.shape, -1)[~used] = 0x7f
        for t in pages[2:]:
            if t is not None:
                t[~used] = 127
    q = torch.randn((batch['tokens'], heads * G, D), generator=torch.Generator().manual_seed(seed + 2)).to(dtype)
    scale = D ** -0.5 if scale is None else scale
    want = ref.attention(q, ref.held(pages[0], pages[2]), ref.held(pages[1], pages[3]), batch, heads, scale, causal, window)
    dev = _cuda(pages)
    out = torch.full(q.shape, 7.0, dtype=dtype, device='cuda')
    lse = torch.full(q.shape[:2], 7.0, device='cuda')
    core.paged_attention(q.cuda(), *dev[:2], *ref.on_device(batch), *dev[2:], scale=scale, causal=causal, window=window, max_queries=max(new) if hints else 0,
                         max_keys=max(lens) if hints else 0, out=out, return_lse=lse, workspace=workspace)
    bo, bl = ref.attention_bounds(want, dtype, D)
    got, got_lse = out.cpu().double(), lse.cpu().double()
    n = batch['starts'][-1]
    assert bool((got[n:] == 7).all()) and bool((got_lse[n:] == 7).all()), 'rows behind the last sequence were written'
    nans = torch.isnan(want['o'][:n])
    assert torch.equal(torch.isnan(got[:n]), nans)
    worst = ((got[:n] - want['o'][:n]).abs() / bo[:n])[~nans]
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, f'o is {float(worst.max()):.3g} times its bound off'
    ends = torch.isneginf(want['lse'][:n])
    assert torch.equal(torch.isneginf(got_lse[:n]), ends)
    fine = ~ends & ~torch.isnan(want['lse'][:n])
    off = ((got_lse[:n] - want['lse'][:n]).abs() / bl[:n])[fine]
    assert off.numel() == 0 or float(off.max()) <= 1.0, f'lse is {float(off.max()):.3g} times its bound off'
    return batch, q, dev, out


SHAPES = [
    # new tokens and lengths: decoding, drafts, chunks, whole prompts, sequences that pause, no length, fewer positions than tokens
    ([1, 1, 1], [1, 37, 200]),
    ([1, 0, 1, 1, 0], [64, 10, 129, 33, 0]),
    ([5, 3, 4], [5, 100, 333]),
    ([17, 1, 0, 40], [17, 300, 5, 250]),
    ([130, 1, 65], [130, 70, 400]),
    ([3, 9, 2], [1, 4, 0]),
]


@pytest.mark.parametrize('new,lens', SHAPES)
@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('cache', [None, E4M3, I8])
@pytest.mark.parametrize('D,page,heads,G', [(128, 16, 2, 4), (64, 32, 1, 1), (96, 64, 3, 2), (32, 16, 2, 7)])
def test_attention_over_a_paged_cache(core, dtype, cache, D, page, heads, G, new, lens):
    _attention_case(core, dtype, cache, D, page, heads, G, new, lens, 11, tail=2)


def _slots_are_packed(new, G, most):
    """Whether the wide kernel numbers its row blocks over the packed rows: with as many for each sequence as `most` tokens have, most would be empty."""
    B, tokens = len(new), sum(new)
    return most * G > 64 and B * -(-most * G // 256) > 2 * (tokens * G // 256 + B)


@pytest.mark.parametrize('dtype,cache,D,page,heads,G', [(F16, None, 128, 16, 1, 4), (BF16, I8, 64, 32, 2, 4), (F16, E4M3, 96, 64, 1, 5)])
@pytest.mark.parametrize('hints', [True, False])
@pytest.mark.parametrize('new,lens', [
    ([600, 1, 1, 0, 1, 1, 1], [650, 300, 40, 20, 1, 128, 77]),
    ([1, 0, 1, 600, 1, 20, 0], [1, 0, 90, 600, 333, 64, 5]),
    ([1, 0, 1] * 11 + [550] + [1, 1, 0] * 12, [(37 * b) % 90 + 1 for b in range(33)] + [700] + [(53 * b) % 90 + 1 for b in range(36)]),
])
def test_a_chunk_beside_sequences_that_decode_or_pause(core, dtype, cache, D, page, heads, G, hints, new, lens):
    """Row blocks numbered over the packed rows, of up to 70 sequences."""
    assert _slots_are_packed(new, G, max(new) if hints else sum(new))
    _attention_case(core, dtype, cache, D, page, heads, G, new, lens, 271, hints=hints, tail=1)


@pytest.mark.parametrize('dtype,cache,D', [(F16, None, 128), (BF16, E4M3, 128), (BF16, None, 64)])
def test_small_sequences_alone_are_cut(core, dtype, cache, D):
    """Room for the parts of sequences of up to 16 rows and for no others': sixteen rows to a wave that joins, most of which have nothing to join."""
    heads, G, page = 2, 2, 16
    long = 4000 * (1 if cache is None else 2) * (128 // D)
    new, lens = [200, 1, 0, 300, 1, 8, 2], [210, long, 50, 300, long - 100, long - 700, 9]
    keys, held = max(lens), 4 * D if cache is None else 2 * D + 2  # bytes of a position and head
    n = min(keys * held // (20 * 17000), keys // 256 + 1)
    part = -(-(-(-keys // n)) // 128) * 128
    parts = -(-keys // part)
    assert 1 < parts < 16                                          # (16 and few rows: a block to a row)
    room = len(new) * heads * 16 * parts * (D + 2) * 4
    _attention_case(core, dtype, cache, D, page, heads, G, new, lens, 281, tail=3, workspace=torch.empty(room, dtype=torch.uint8, device='cuda'))


@pytest.mark.parametrize('causal,window', [(False, 0), (True, 1), (True, 16), (True, 50), (False, 33)])
@pytest.mark.parametrize('cache,D,page,G', [(None, 64, 16, 3), (E4M3, 128, 64, 1), (I8, 96, 32, 8)])
@pytest.mark.parametrize('new,lens', [([1, 1], [200, 31]), ([6, 2], [150, 40]), ([100, 3], [150, 90])])
def test_attention_windows_and_without_a_causal_mask(core, causal, window, cache, D, page, G, new, lens):
    _attention_case(core, BF16 if D == 96 else F16, cache, D, page, 2, G, new, lens, 21, causal=causal, window=window, hints=window != 16)


@pytest.mark.parametrize('dtype,cache,D,page,heads,G,new,lens', [
    (F16, None, 128, 16, 1, 4, [1, 1], [3000, 700]),
    (BF16, E4M3, 128, 128, 2, 8, [1, 2], [2500, 100]),
    (F16, I8, 64, 32, 1, 1, [1], [5000]),
    (F16, E4M3, 32, 16, 1, 2, [3], [4000]),
    (BF16, None, 96, 64, 1, 5, [8, 1], [2600, 2000]),
    (BF16, I8, 128, 256, 1, 4, [40, 1], [3100, 2600]),       # the wide kernel, in parts
    (F16, None, 64, 16, 1, 2, [150], [2777]),
    (F16, I8, 96, 16, 1, 2, [70], [2100]),
    (F16, E4M3, 32, 32, 1, 2, [70], [9000]),
])
@pytest.mark.parametrize('window', [0, 1111])
def test_long_sequences_in_parts(core, dtype, cache, D, page, heads, G, new, lens, window):
    batch = ref.make_batch(new, lens, page, 31)
    q = torch.empty((batch['tokens'], heads * G, D), dtype=dtype, device='cuda')
    like = torch.empty((batch['pages'], heads, page, D), dtype=cache or dtype, device='cuda')
    need = core.paged_attention_workspace_bytes(q, like, ref.on_device(batch)[0], max(new), max(lens), window)
    assert need > 0 or window                                    # more than one part
    for space in (None, torch.empty(max(need // 2, 16), dtype=torch.uint8, device='cuda'), torch.empty(0, dtype=torch.uint8, device='cuda')):
        _attention_case(core, dtype, cache, D, page, heads, G, new, lens, 31, window=window, workspace=space)


@pytest.mark.parametrize('dtype,cache,D,page,heads,G,n,B,L', [
    (F16, None, 128, 16, 4, 8, 3, 16, 1100),                     # 24 rows: one block of 32
    (BF16, I8, 128, 64, 4, 8, 6, 16, 1100),                      # 48 rows: two, the second of which is not full
    (F16, E4M3, 96, 32, 5, 7, 9, 12, 1100),                      # 63
    (BF16, E4M3, 64, 16, 9, 2, 32, 10, 700),                     # 64
    (F16, I8, 32, 128, 12, 5, 8, 12, 600),                       # 40
    (BF16, None, 128, 16, 3, 4, 11, 11, 300),                    # 44 rows of few keys: blocks of 16
    (F16, None, 64, 16, 8, 1, 9, 40, 200),                       # 9 rows: many results
    (F16, I8, 128, 16, 8, 4, 4, 9, 300),                         # 16 rows
])
def test_drafts_of_many_sequences(core, dtype, cache, D, page, heads, G, n, B, L):
    new = [max(0, n - (b % 5 if b % 3 == 1 else 0)) for b in range(B)]
    lens = [max(1, L - 41 * b) if b % 4 else L for b in range(B)]
    _attention_case(core, dtype, cache, D, page, heads, G, new, lens, 191, tail=1)


@pytest.mark.parametrize('new,lens', [([6], [70]), ([5, 100], [33, 130]), ([2], [64])])
@pytest.mark.parametrize('dtype,cache', [(F16, None), (BF16, None), (F16, E4M3), (BF16, E4M3)])
def test_keys_and_values_that_are_not_finite_reach_only_who_sees_them(core, dtype, cache, new, lens):
    """The last new key of every sequence and one in the middle of its chunk: earlier tokens do not see them."""
    D, page, heads, G = 64, 16, 2, 2
    batch = ref.make_batch(new, lens, page, 41)
    pages = ref.make_pages(batch, heads, D, cache, dtype, 42)
    nan = math.nan if cache == E4M3 else math.inf
    for b, n in enumerate(lens):
        last, middle = n - 1, n - 1 - new[b] // 2
        at = lambda p: (batch['table'][b][p // page], p % page)
        pages[1][at(last)[0], 0, at(last)[1], 5] = math.nan
        pages[1][at(last)[0], 1, at(last)[1], D - 1] = nan
        pages[1][at(middle)[0], 1, at(middle)[1], 3] = nan
        pages[0][at(last)[0], 1, at(last)[1], 0] = math.nan
    _attention_case(core, dtype, cache, D, page, heads, G, new, lens, 41, junk=True, pages=pages)


@pytest.mark.parametrize('D,cache', [(64, None), (128, I8)])
@pytest.mark.parametrize('new', [1, 40])
def test_scores_of_any_size(core, D, cache, new):
    """Scores far from zero on both sides, and keys whose scores are all alike."""
    for scale in (1e-6, 3.0):
        _attention_case(core, F16, cache, D, 16, 1, 2, [new], [200], 51, scale=scale)


def test_small_and_large_rows_of_codes(core):
    """Exponents at both ends of what fp16 rows get: values of 2^-24, and of tens of thousands, in one cache."""
    for cache, least, most in ((I8, -24, 9), (E4M3, -15, 7)):
        batch = ref.make_batch([1, 30], [100, 90], 16, 61)
        pages = ref.make_pages(batch, 1, 64, cache, F16, 62)
        g = torch.Generator().manual_seed(63)
        pages[3] = torch.where(torch.rand(pages[3].shape, generator=g) < 0.5, least, most).to(torch.int8)
        for new, lens in (([1, 2], [100, 90]), ([1, 130], [100, 140])):
            batch = ref.make_batch(new, lens, 16, 61)
            big = ref.make_pages(batch, 1, 64, cache, F16, 62)
            big[3] = torch.where(torch.rand(big[3].shape, generator=g) < 0.5, least, most).to(torch.int8)
            _attention_case(core, F16, cache, 64, 16, 1, 4, new, lens, 61, pages=big)


def test_pages_that_point_nowhere_hurt_nobody_else(core):
    """Table entries outside the pages: the sequence beside them is as without, nothing else is written, and reads give zeros."""
    D, page, heads = 64, 16, 2
    batch = ref.make_batch([20, 3], [50, 40], page, 71)
    good = ref.on_device(batch)
    bad = good[0].clone()
    bad[0, 1], bad[0, 2], bad[0, 3] = -7, batch['pages'], 2 ** 31 - 1
    g = torch.Generator().manual_seed(72)
    keys, values, q = (torch.randn((23, h, D), generator=g).to(F16).cuda() for h in (heads, heads, 4))
    a, b = (_cuda(ref.make_pages(batch, heads, D, I8, F16, 73)) for _ in range(2))
    core.kv_cache_write(keys, values, *a[:2], *good, *a[2:])
    core.kv_cache_write(keys, values, *b[:2], bad, *good[1:], *b[2:])
    own = [p for p in batch['table'][1][:3]]
    assert all(_same(x[own], y[own]) for x, y in zip(a, b))
    others = [p for p in range(batch['pages']) if p not in batch['table'][0][:4] and p not in own]
    fresh = _cuda(ref.make_pages(batch, heads, D, I8, F16, 73))
    assert all(_same(x[others], y[others]) for x, y in zip(b, fresh))
    k, _ = core.kv_cache_read(*a[:2], bad, *good[1:], 23, F32, *a[2:])
    assert bool((k[:18] == 0).all())                             # positions 30 to 47 lie in pages 1 and 2 of the table
    for hint in (20, 0):
        x, y = (core.paged_attention(q, *a[:2], t, *good[1:], *a[2:], max_queries=hint) for t in (good[0], bad))
        assert torch.equal(x[20:], y[20:])


def test_batches_that_make_no_sense_write_nothing_outside(core):
    """starts that decrease or point past the rows, lengths past the table: in bounds (a launch that was not would fault), and what lies
    around the outputs is left alone."""
    D, page, heads = 64, 16, 2
    batch = ref.make_batch([4, 4, 4], [30, 40, 50], page, 75)
    table, lens, starts = ref.on_device(batch)
    g = torch.Generator().manual_seed(76)
    keys, values, q = (torch.randn((12, h, D), generator=g).to(F16).cuda() for h in (heads, heads, 4))
    for s, n in (([0, 8, 4, 12], [30, 40, 50]), ([0, 4, 8, 2 ** 31 - 1], [30, 40, 50]), ([-5, 4, 8, 12], [30, -40, 50]), ([0, 4, 8, 12], [30, 4000, 2 ** 31 - 1]), ([12, 0, 0, 0], [0, 0, 0])):
        ints = [torch.tensor(v, dtype=torch.int32, device='cuda') for v in (n, s)]
        pages = _cuda(ref.make_pages(batch, heads, D, E4M3, F16, 77))
        core.kv_cache_write(keys, values, *pages[:2], table, *ints, *pages[2:])
        core.kv_cache_read(*pages[:2], table, *ints, 12, F16, *pages[2:])
        for hint in (0, 4, 1):
            whole = torch.full((14, 4, D), 7.0, dtype=F16, device='cuda')
            core.paged_attention(q, *pages[:2], table, *ints, *pages[2:], max_queries=hint, out=whole[1:13])
            assert bool((whole[0] == 7).all()) and bool((whole[13] == 7).all())
    torch.cuda.synchronize()


def test_batches_that_make_no_sense_leave_what_lies_around_alone(core):
    """Pages, exponents, dense rows, results and log-sum-exps lie inside larger buffers of a pattern: what is written lies in them, and in pages that the table names."""
    D, page, heads = 64, 16, 2
    batch = ref.make_batch([4, 4, 4], [30, 40, 50], page, 75)
    table = ref.on_device(batch)[0]
    named = set(sum(batch['table'], []))
    g = torch.Generator().manual_seed(76)
    keys, values, q = (torch.randn((12, h, D), generator=g).to(F16).cuda() for h in (heads, heads, 4))
    inside = lambda shape, dtype: torch.full((shape[0] + 2 * 8, *shape[1:]), 0x55, dtype=torch.uint8, device='cuda').view(dtype)
    P = batch['pages']
    for s, n in (([0, 8, 4, 12], [30, 40, 50]), ([0, 4, 8, 2 ** 31 - 1], [30, 40, 50]), ([-5, 4, 8, 12], [30, -40, 50]), ([0, 4, 8, 12], [30, 4000, 2 ** 31 - 1]), ([12, 0, 0, 0], [0, 0, 0]),
                 ([3, 4, 9, 11], [-2 ** 31, 2 ** 31 - 1, 1])):
        ints = [torch.tensor(v, dtype=torch.int32, device='cuda') for v in (n, s)]
        whole = [inside((P, heads, page, D), E4M3) for _ in range(2)] + [inside((P, heads, page), I8) for _ in range(2)]
        pages = [t[8:-8] for t in whole]
        core.kv_cache_write(keys, values, *pages[:2], table, *ints, *pages[2:])
        for t in whole:
            raw = t.view(torch.uint8)
            for i in range(len(raw)):
                assert i - 8 in named or bool((raw[i] == 0x55).all()), (s, n, i)
        before = [t.view(torch.uint8).clone() for t in whole]
        rows = [inside((12, heads, D * 2), F16) for _ in range(2)]
        core.kv_cache_read(*pages[:2], table, *ints, 12, F16, *pages[2:], out=tuple(t[8:-8] for t in rows))
        for hint in (0, 4, 1):
            o, lse = inside((12, 4, D * 2), F16), inside((12, 4 * 4), F32)
            core.paged_attention(q, *pages[:2], table, *ints, *pages[2:], max_queries=hint, out=o[8:-8], return_lse=lse[8:-8])
            for t in (*rows, o, lse):
                raw = t.view(torch.uint8)
                assert bool((raw[:8] == 0x55).all()) and bool((raw[-8:] == 0x55).all()), (s, n, hint)
        assert all(torch.equal(a.view(torch.uint8), b) for a, b in zip(whole, before))


@pytest.mark.parametrize('new,lens,rows', [([1, 6], [40, 90], 4), ([5, 100], [30, 300], 60), ([3], [2900], 2), ([90], [3000], 70)])
def test_packed_rows_that_end_inside_a_sequence(core, new, lens, rows):
    """Fewer packed rows than `starts` speaks of: those that are there are at their positions, as for writing and reading."""
    D, page, heads, G = 64, 16, 2, 4
    batch = ref.make_batch(new, lens, page, 87)
    pages = ref.make_pages(batch, heads, D, None, F16, 88)
    q = torch.randn((batch['tokens'], heads * G, D), generator=torch.Generator().manual_seed(89)).to(F16)
    want = ref.attention(q, ref.held(pages[0], None), ref.held(pages[1], None), batch, heads, D ** -0.5)
    bound, _ = ref.attention_bounds(want, F16, D)
    dev = _cuda(pages)
    got = core.paged_attention(q[:rows].cuda(), *dev[:2], *ref.on_device(batch), max_queries=max(new), max_keys=max(lens)).cpu().double()
    assert bool(((got - want['o'][:rows]).abs() <= bound[:rows]).all())
    k, _ = core.kv_cache_read(*dev[:2], *ref.on_device(batch), rows)
    for b in range(len(new)):
        for row, at, r in ref.places(batch, b):
            assert row >= rows or torch.equal(k[row].cpu(), pages[0][at, :, r])


@pytest.mark.parametrize('new,lens', [([1, 1], [100, 40]), ([100, 1], [130, 40])])
def test_queries_as_views_and_results_in_their_place(core, new, lens):
    D, page, heads, G = 128, 32, 2, 4
    batch = ref.make_batch(new, lens, page, 81)
    pages = _cuda(ref.make_pages(batch, heads, D, None, BF16, 82))
    joint = torch.randn((batch['tokens'], heads * G + 2 * heads, D), generator=torch.Generator().manual_seed(83)).to(BF16).cuda()
    q = joint[:, :heads * G]
    args = (*pages[:2], *ref.on_device(batch))
    want = core.paged_attention(q.contiguous(), *args)
    assert torch.equal(core.paged_attention(q, *args), want)
    turned = q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert torch.equal(core.paged_attention(turned, *args), want)
    own = q.contiguous()
    core.paged_attention(own, *args, out=own)
    assert torch.equal(own, want)


def test_empty_calls(core):
    pages = _cuda(ref.make_pages(dict(pages=2, page=16), 2, 64, None, F16, 1))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device='cuda')
    table = torch.zeros((1, 1), dtype=torch.int32, device='cuda')
    none = torch.empty((0, 2, 64), dtype=F16, device='cuda')
    core.kv_cache_write(none, none, *pages[:2], table, ints(0), ints(0, 0))
    assert core.kv_cache_read(*pages[:2], table, ints(0), ints(0, 0), 0)[0].shape == (0, 2, 64)
    assert core.paged_attention(none, *pages[:2], table, ints(0), ints(0, 0)).shape == (0, 2, 64)
    some = torch.ones((3, 2, 64), dtype=F16, device='cuda')
    out = torch.full_like(some, 7.0)
    core.paged_attention(some, *pages[:2], table[:0], ints(), ints(0), out=out)
    assert bool((out == 7).all())
    tokens, accepted = core.verify_drafts(torch.ones((0, 3, 8), device='cuda'), None, torch.zeros((0, 2), dtype=torch.int64, device='cuda'), torch.zeros((0, 2), device='cuda'),
                                          torch.zeros(0, device='cuda'))
    assert tokens.shape == (0, 3) and accepted.shape == (0,)


def test_refusals_on_the_device(core):
    pages = _cuda(ref.make_pages(dict(pages=2, page=16), 2, 64, None, F16, 1))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device='cuda')
    batch = (torch.zeros((1, 1), dtype=torch.int32, device='cuda'), ints(1), ints(0, 1))
    q = torch.ones((1, 4, 64), dtype=F16, device='cuda')
    call = lambda q=q, p=pages, b=batch, **kw: core.paged_attention(q, *p[:2], *b, **kw)
    with pytest.raises(TypeError, match='type of the pages'):
        call(q.to(BF16))
    with pytest.raises(TypeError, match='float16 or bfloat16'):
        call(q.float())
    with pytest.raises(ValueError, match=r'\[tokens, heads, 64\]'):
        call(q[:, :, :32])
    with pytest.raises(core.FtkError) as info:
        call(q[:, :3].contiguous())
    assert info.value.code == -1
    with pytest.raises(ValueError, match='strides'):
        call(torch.ones((2, 4, 68), dtype=F16, device='cuda')[:, :, 2:66])
    with pytest.raises(ValueError, match='out must be'):
        call(out=torch.empty((2, 4, 64), dtype=F16, device='cuda'))
    with pytest.raises(ValueError, match='window'):
        call(window=-1)
    with pytest.raises(core.FtkError):
        call(scale=0.0)
    with pytest.raises(ValueError, match='CUDA tensor'):
        call(workspace=torch.empty(1 << 20, dtype=torch.uint8))
    with pytest.raises(TypeError, match='table must be'):
        call(b=(batch[0].long(), *batch[1:]))
    with pytest.raises(ValueError, match='starts must be'):
        call(b=(*batch[:2], ints(0)))
    with pytest.raises(ValueError, match='have no k_exps'):
        call(k_exps=torch.zeros((2, 2, 16), dtype=torch.int8, device='cuda'))
    with pytest.raises(ValueError, match='need k_exps'):
        call(p=[t.to(torch.int8) for t in pages[:2]])
    k = torch.ones((1, 2, 64), dtype=F16, device='cuda')
    with pytest.raises(ValueError, match='as many tokens'):
        core.kv_cache_write(k, torch.ones((2, 2, 64), dtype=F16, device='cuda'), *pages[:2], *batch)
    with pytest.raises(TypeError, match='read in that type'):
        core.kv_cache_read(*pages[:2], *batch, 1, BF16)
    with pytest.raises(ValueError, match='tokens must be'):
        core.kv_cache_read(*pages[:2], *batch, -1)
    with pytest.raises(core.FtkError) as info:                   # page sizes that the kernels do not have
        core.kv_cache_write(k, k, *[t[:, :, :8].contiguous() for t in pages[:2]], *batch)
    assert info.value.code == -2


@pytest.mark.parametrize('above', [12.0, 16.0, 20.0])
@pytest.mark.parametrize('at', [0, 1500])
@pytest.mark.parametrize('dtype,cache,D,page,G,new', [(F16, None, 64, 16, 4, 1), (F16, I8, 128, 64, 4, 5), (F16, E4M3, 96, 32, 2, 9), (F16, None, 128, 16, 2, 70), (F16, I8, 64, 16, 2, 90),
                                                      (F16, E4M3, 32, 128, 1, 150), (BF16, None, 64, 16, 4, 1), (BF16, I8, 64, 16, 2, 90)])
def test_keys_beside_one_that_outweighs_them(core, dtype, cache, D, page, G, new, at, above):
    """A key whose score is far above the others' and whose value is zero, at the first position or later: the result is what the others leave, by weights
    of e^-12 to e^-20 of the largest."""
    length, heads = 4096, 2
    batch = ref.make_batch([new], [length], page, 201)
    pages = ref.make_pages(batch, heads, D, None, dtype, 202)
    pages[1] = pages[1].abs()
    keys, row = batch['table'][0][at // page], at % page
    pages[0][..., 0] = 0.0
    pages[0][keys, :, row] = 0.0
    pages[0][keys, :, row, 0] = above * 2                          # q 4, scale 1 / 8; a value of both codes
    pages[1][keys, :, row] = 0.0
    exps = [None, None]
    if cache is not None:
        for i in range(2):
            x = pages[i].float()
            e = torch.ceil(torch.log2(x.abs().amax(-1).clamp(min=0.1) / ref.LARGEST[cache])).to(torch.int8)
            scaled = x / torch.pow(2.0, e.float()).unsqueeze(-1)
            pages[i], exps[i] = (scaled.round() if cache == I8 else scaled).to(cache), e
    q = torch.randn((new, heads * G, D), generator=torch.Generator().manual_seed(203)).to(dtype)
    q[..., 0] = 4.0
    held = [ref.held(pages[i], exps[i]) for i in range(2)]
    want = ref.attention(q, *held, batch, heads, 0.125)
    bound = ref.attention_bounds_by_largest(want, dtype, D)
    dev = _cuda([*pages[:2], *exps])
    got = core.paged_attention(q.cuda(), *dev[:2], *ref.on_device(batch), *dev[2:], scale=0.125, max_queries=new, max_keys=length).cpu().double()
    worst = float(((got - want['o']).abs() / bound).max())
    assert worst <= 1.0, f'o is {worst:.3g} times its bound off'


@pytest.mark.parametrize('dtype,cache,D,G', [(F16, None, 128, 4), (BF16, E4M3, 128, 4), (BF16, None, 64, 1), (F16, I8, 96, 8), (F16, E4M3, 32, 16)])
def test_a_result_does_not_depend_on_what_else_the_call_holds(core, dtype, cache, D, G):
    """One token of a sequence alone, among sixty-four that decode, and beside a prompt: the same bits where the keys are not cut, and the error of the result's own rounding
    alone each time."""
    heads, page, length = 2, 16, 333
    lens = [length] + [17 * b % 500 + 1 for b in range(1, 64)]
    batch = ref.make_batch([1] * 64, lens, page, 211)
    pages = ref.make_pages(batch, heads, D, cache, dtype, 212)
    q = 3 * torch.randn((64, heads * G, D), generator=torch.Generator().manual_seed(213))      # a few keys have most of a row's weight
    q = q.to(dtype)
    want = ref.attention(q, ref.held(pages[0], pages[2]), ref.held(pages[1], pages[3]), batch, heads, D ** -0.5)
    bound = ref.attention_bounds_by_largest(want, dtype, D, split=True)
    dev, (table, at, starts) = _cuda(pages), ref.on_device(batch)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device='cuda')
    uncut = torch.empty(0, dtype=torch.uint8, device='cuda')
    call = lambda rows, t, n, s, most: core.paged_attention(rows, *dev[:2], t, n, s, *dev[2:], max_queries=most, max_keys=500, workspace=uncut, return_lse=True)
    many = call(q.cuda(), table, at, starts, 1)
    alone = call(q[:1].cuda(), table[:1], at[:1], ints([0, 1]), 1)
    prompt = torch.cat([q[:1], q[:1].expand(100, -1, -1)]).cuda()
    beside = call(prompt, table[:1].expand(2, -1).contiguous(), ints([length, 100]), ints([0, 1, 101]), 100)
    for x in (alone, beside):
        assert torch.equal(x[0][:1], many[0][:1]) and torch.equal(x[1][:1], many[1][:1])
    worst = ((many[0].cpu().double() - want['o']).abs() / bound).max()
    assert float(worst) <= 1.0, f'o is {float(worst):.3g} times its bound off'


@pytest.mark.parametrize('dtype,cache,D,G,n', [(F16, None, 128, 4, 5), (BF16, E4M3, 64, 8, 8), (BF16, I8, 128, 8, 6), (F16, I8, 96, 4, 16), (BF16, None, 96, 2, 9)])
def test_drafts_are_off_by_the_rounding_of_results_alone(core, dtype, cache, D, G, n):
    """Sequences of 17 to 64 rows, in blocks of 16 and of 32."""
    for B, L in ((2, 100), (24, 300)):
        batch = ref.make_batch([n] * B, [L - 3 * b for b in range(B)], 16, 221)
        pages = ref.make_pages(batch, 6, D, cache, dtype, 222)
        q = (3 * torch.randn((batch['tokens'], 6 * G, D), generator=torch.Generator().manual_seed(223))).to(dtype)
        want = ref.attention(q, ref.held(pages[0], pages[2]), ref.held(pages[1], pages[3]), batch, 6, D ** -0.5)
        bound = ref.attention_bounds_by_largest(want, dtype, D, split=True)
        dev = _cuda(pages)
        got = core.paged_attention(q.cuda(), *dev[:2], *ref.on_device(batch), *dev[2:], max_queries=n, max_keys=L).cpu().double()
        worst = ((got - want['o']).abs() / bound).max()
        assert float(worst) <= 1.0, f'o is {float(worst):.3g} times its bound off'


@pytest.mark.parametrize('dtype,cache,new,lens', [(F16, None, [1, 3], [400, 200]), (BF16, None, [1], [3000]), (F16, None, [100, 1], [400, 300]), (BF16, None, [90], [3000])])
def test_infinite_values_make_nan_wherever_they_lie(core, dtype, cache, new, lens):
    """In tiles that all rows see, in those that a mask cuts, and beside one another: the same component is NaN, all others are what they were."""
    D, page, heads, G = 64, 16, 2, 2
    batch = ref.make_batch(new, lens, page, 231)
    pages = ref.make_pages(batch, heads, D, cache, dtype, 232)
    for b, n in enumerate(lens):
        for i, p in enumerate([0, 5, 70, 71, 100, n - new[b] - 1, n - 1]):
            at, row = batch['table'][b][p // page], p % page
            pages[1][at, i % heads, row, 7 * i + 1] = (math.inf, -math.inf)[i % 3 == 1]
            pages[1][at, 1 - i % heads, row, 60] = (math.inf, -math.inf)[i % 2]
    _attention_case(core, dtype, cache, D, page, heads, G, new, lens, 231, pages=pages)


@pytest.mark.parametrize('dtype,new,length', [(F16, 2, 300), (BF16, 1, 3000), (F16, 80, 300), (BF16, 90, 3000)])
def test_infinite_keys_give_the_scores_that_they_give(core, dtype, new, length):
    """-inf: a weight of zero, as that of a score far below all others; inf: NaN."""
    D, page, G = 64, 16, 2
    batch = ref.make_batch([new], [length], page, 241)
    pages = ref.make_pages(batch, 1, D, None, dtype, 242)
    q = torch.randn((new, G, D), generator=torch.Generator().manual_seed(243)).to(dtype)
    q[:, 0, 0], q[:, 1, 0] = -1.0, 1.0                              # the first head's scores are -inf, the second's inf

    def with_keys(x):
        for p in (0, 77, length - new):
            pages[0][batch['table'][0][p // page], 0, p % page, 0] = x
        return ref.attention(q, ref.held(pages[0], None), ref.held(pages[1], None), batch, 1, 0.125)

    # the weight of a score of -7500 is zero as well; what the other keys' scores are off by is what the bound is made of (rows of a wave move their reference
    # together, so that one head's scores can change another's last bits)
    most, want = with_keys(0.0)['most'], with_keys(60000.0)
    want['most'] = most
    bound, exact = ref.attention_bounds_by_largest(want, dtype, D), want['o']
    with_keys(math.inf)
    dev = _cuda(pages)
    o, lse = core.paged_attention(q.cuda(), *dev[:2], *ref.on_device(batch), scale=0.125, max_queries=new, max_keys=length, return_lse=True)
    assert bool(((o[:, 0].cpu().double() - exact[:, 0]).abs() <= bound[:, 0]).all())
    assert bool(((lse[:, 0].cpu().double() - want['lse'][:, 0]).abs() <= ref.attention_bounds(want, dtype, D)[1][:, 0]).all())
    assert bool(torch.isnan(o[:, 1]).all()) and bool(torch.isnan(lse[:, 1]).all())


@pytest.mark.parametrize('cache', [I8, E4M3])
@pytest.mark.parametrize('D,page,G,new,lens', [(64, 16, 4, [1, 3], [300, 90]), (96, 32, 4, [9, 4], [200, 150]), (128, 16, 8, [6] * 3, [900, 70, 6]), (64, 32, 2, [100, 1], [300, 200]),
                                               (128, 16, 1, [80], [2500]), (32, 16, 1, [70, 2], [100, 300])])
def test_queries_of_fp16_on_codes_of_bf16_rows(core, cache, D, page, G, new, lens):
    """Rows of zeros, of values below and at the end of fp16's range and beyond it: elements count as fp16 numbers, on all kernels."""
    heads, g = 2, torch.Generator().manual_seed(251)
    batch = ref.make_batch(new, lens, page, 252)
    factors = torch.tensor([1.0, 1.0, 0.0, 1e-5, 1e-6, 1e-7, 1e-8, 1e-12])
    k, v = (torch.randn((sum(lens), heads, D), generator=g).clamp(-4, 4) * factors[torch.randint(0, 8, (sum(lens), heads, 1), generator=g)] for _ in range(2))
    v[::7] = (v[::7] * 14000).clamp(-60000, 60000)
    k[11:13], v[13], v[14] = 0.0, 0.0, 0.0
    k[11, :, 0], k[12, :, 0] = 1e7, 3e30                            # q is -1 there: a score of -inf
    v[13, :, 3], v[14, 1, 5] = 1e5, -1e20
    pages = _cuda(ref.make_pages(batch, heads, D, cache, BF16, 253))
    table, at, _ = ref.on_device(batch)
    whole = torch.tensor([sum(lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device='cuda')
    core.kv_cache_write(k.to(BF16).cuda(), v.to(BF16).cuda(), *pages[:2], table, at, whole, *pages[2:])
    q = torch.randn((batch['tokens'], heads * G, D), generator=g).to(F16)
    q[..., 0] = -1.0
    as_half = lambda x: x.float().to(F16).double()                  # exact in fp32
    keys, values = as_half(ref.held(pages[0], pages[2])), as_half(ref.held(pages[1], pages[3]))
    assert int(torch.isinf(keys).sum()) == 2 * heads and int(torch.isinf(values).sum()) == heads + 1
    most = ref.attention(q, torch.where(torch.isinf(keys), 0.0, keys), values, batch, heads, 0.125)['most']
    want = ref.attention(q, torch.where(torch.isinf(keys), 60000.0, keys), values, batch, heads, 0.125)
    want['most'] = most
    # keys below 2^-14 may be as they are, less than 2^-25 off their fp16 number
    bound = ref.attention_bounds_by_largest(want, F16, D) + (2 * 0.125 * 2.0 ** -25) * q.double().abs().sum(-1, keepdim=True) * want['mean']
    got = core.paged_attention(q.cuda(), *pages[:2], *ref.on_device(batch), *pages[2:], scale=0.125, max_queries=max(new), max_keys=max(lens)).cpu().double()
    nans = torch.isnan(want['o'])
    assert bool(nans.any()) and not bool(nans.all()) and torch.equal(torch.isnan(got), nans)
    worst = float(((got - want['o']).abs() / bound)[~nans].max())
    assert worst <= 1.0, f'o is {worst:.3g} times its bound off'


# ---- verification -----------------------------------------------------------------------

def _drafts(B, K, V, dtype, wide, seed):
    g = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn((B, K + 1, V), generator=g)
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :K] + 0.7 * torch.randn((B, K, V), generator=g), -1).to(dtype)
    drafts = torch.multinomial(draft.float().view(-1, V), 1, generator=g).view(B, K) if B * K else torch.zeros((B, K), dtype=torch.int64)
    return target, draft, drafts.to(torch.int64 if wide else torch.int32), torch.rand((B, K), generator=g), torch.rand(B, generator=g)


def _verified(core, target, draft, drafts, accept, sample, counts=None):
    want = ref.verify(target, draft, drafts, accept, sample, None if counts is None else counts.tolist())
    got = core.verify_drafts(target.cuda(), None if draft is None else draft.cuda(), drafts.cuda(), accept.cuda(), sample.cuda(), None if counts is None else counts.cuda())
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0])
    return want


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('B,K,V', [(1, 1, 1), (3, 2, 7), (5, 4, 1000), (2, 5, 2048), (4, 3, 2049), (3, 0, 4096), (2, 63, 301), (2, 2, 65536), (2, 2, 70001), (3, 1, 131072), (2, 1, 150003), (2, 1, 262145)])
def test_verified_drafts(core, dtype, B, K, V):
    t = _drafts(B, K, V, dtype, K % 2, 91)
    _verified(core, *t)
    _verified(core, t[0], None, *t[2:])
    _verified(core, *t, counts=torch.tensor([(2 * b) % (K + 2) - (b == 2) for b in range(B)], dtype=torch.int32))


def test_verified_drafts_at_the_ends_of_their_ranges(core):
    B, K, V = 8, 3, 5000
    target, draft, drafts, accept, sample = _drafts(B, K, V, F32, True, 92)
    target[0] = draft[0, :1]                                      # nothing left of the target's row
    accept[0] = 1.0                                               # (a uniform of 1: rejected even so)
    drafts[1, 1], drafts[2, 0] = V, -1                            # no such tokens
    target[3, 0, drafts[3, 0]] = 0.0                              # impossible
    accept[4], sample[4] = 0.0, 0.0                               # every draft with a chance is accepted; the first token with one
    target[4, K, :17] = 0.0
    sample[5] = 1.0 - 2.0 ** -24
    target[6, 0] = 0.0                                            # no token has a chance
    accept[6] = 0.5
    target[7, 0, 5], draft[7, 0, 6] = math.nan, math.nan
    accept[7] = 1.0
    want = _verified(core, target, draft, drafts, accept, sample)
    assert want[1].tolist()[0] == 0 and int(want[1][1]) <= 1 and int(want[1][2]) == 0 and int(want[1][3]) == 0 and int(want[0][6][0]) == -1


@pytest.mark.parametrize('V', [(1 << 21) + 8, (1 << 21) + 1001])
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_verification_of_vocabularies_whose_segments_take_two_passes(core, V, dtype):
    """Beyond 2^21 a segment has 4096 tokens, read 2048 at a time: drawn tokens in both halves of a segment, in the first, a late and the last one, from the target's row
    and from what is left of it."""
    g = torch.Generator().manual_seed(94)
    weights = torch.rand((1, 2, V), generator=g)
    wanted = [5, 2048 + 77, 300 * 4096 + 4000, (V // 4096 - 1) * 4096 + 1000, V - 1]
    weights[0, :, wanted] = 500.0
    target = (weights / weights.sum(-1, keepdim=True, dtype=torch.float64)).to(dtype)
    draft = (target[:, :1].double() * 0.5).to(dtype)
    for token in wanted:
        for drafts, accept in (([[7]], 0.0), ([[7]], 1.0)):
            n = 0 if accept else 1
            draft[0, 0, 7] = 1.0 if accept else draft[0, 0, 8]      # rejected: 1 * 1 < target does not hold
            w = target[0, n].double() - (draft[0, 0].double() if accept else 0.0)
            ends = torch.where(w > 0, w, 0.0).cumsum(0)
            u = float((ends[token] - w[token] / 2) / ends[-1])     # the middle of its weight, some 2^-13 of all
            want = _verified(core, target, draft, torch.tensor(drafts), torch.tensor([[accept]]), torch.tensor([u]))
            assert int(want[1][0]) == n and int(want[0][0, n]) == token


def test_verified_drafts_at_odd_addresses(core):
    """Rows that do not begin at 16-byte boundaries, by the size of the vocabulary and by the place of the tensors."""
    for V in (999, 4096):
        target, draft, drafts, accept, sample = _drafts(3, 2, V, F16, False, 93)
        space = [torch.empty(t.numel() + 1, dtype=F16, device='cuda')[1:] for t in (target, draft)]
        views = [s.copy_(t.flatten()).view(t.shape) for s, t in zip(space, (target, draft))]
        want = ref.verify(target, draft, drafts, accept, sample)
        got = core.verify_drafts(*views, drafts.cuda(), accept.cuda(), sample.cuda())
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


# ---- together -----------------------------------------------------------------------------

def _step_inputs(seed, new, heads, G, D, V, dtype):
    g = torch.Generator(device='cuda').manual_seed(seed)
    n = sum(new)
    rows = [torch.randn((n, h, D), generator=g, device='cuda').to(dtype) for h in (heads, heads, heads * G)]
    return rows, torch.randn((heads * G * D, V), generator=g, device='cuda') * 0.3, [torch.rand(s, generator=g, device='cuda') for s in ((len(new), new[0] - 1), (len(new),))]


@pytest.mark.parametrize('dtype,cache', [(F16, E4M3), (BF16, I8), (BF16, None)])
def test_a_served_step(core, dtype, cache):
    """Prompts into the cache, then drafts: written, attended to, turned into probabilities, verified; the rejected ones are overwritten by the next step.
    Attention of a chunk equals attention of its tokens one by one to rounding, and what it reads is what was written."""
    heads, G, D, V, page, K = 2, 4, 64, 500, 16, 3
    prompts = [40, 7, 90]
    batch = ref.make_batch(prompts, [n + 20 for n in prompts], page, 101)
    table = ref.on_device(batch)[0]
    pages = _junk(_cuda(ref.make_pages(batch, heads, D, cache, dtype, 102)))
    kv, exps = pages[:2], pages[2:]
    lens = list(prompts)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device='cuda')
    starts = lambda new: ints([sum(new[:i]) for i in range(len(new) + 1)])
    (k, v, q), _, _ = _step_inputs(103, prompts, heads, G, D, V, dtype)
    at = (table, ints(lens), starts(prompts))
    core.kv_cache_write(k, v, *kv, *at, *exps)
    whole = core.paged_attention(q, *kv, *at, *exps, max_queries=max(prompts), max_keys=max(lens))
    last = torch.tensor([sum(prompts[:i + 1]) - 1 for i in range(3)], device='cuda')
    single = core.paged_attention(q[last].contiguous(), *kv, table, ints(lens), starts([1] * 3), *exps, max_queries=1, max_keys=max(lens))
    u = torch.finfo(dtype).eps
    assert bool(((whole[last].float() - single.float()).abs() <= 4 * u * (1 + single.float().abs())).all())
    generated = [[] for _ in prompts]
    for step in range(4):
        new = [K + 1] * 3
        lens = [n + K + 1 for n in lens]
        (k, v, q), head, (accept, sample) = _step_inputs(200 + step, new, heads, G, D, V, dtype)
        at = (table, ints(lens), starts(new))
        core.kv_cache_write(k, v, *kv, *at, *exps)
        o = core.paged_attention(q, *kv, *at, *exps, max_queries=K + 1, max_keys=max(lens))
        target = core.online_softmax((o.float().view(sum(new), -1) @ head).contiguous()).view(3, K + 1, V)
        draft = core.online_softmax((target[:, :K] + 1e-3).log().mul(0.8).reshape(-1, V)).view(3, K, V)
        drafts = torch.multinomial(draft.view(-1, V), 1, generator=torch.Generator(device='cuda').manual_seed(step)).view(3, K)
        tokens, accepted = core.verify_drafts(target, draft, drafts, accept, sample)
        want = ref.verify(target.cpu(), draft.cpu(), drafts.cpu(), accept.cpu(), sample.cpu())
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(accepted.cpu(), want[1])
        read_k, _ = core.kv_cache_read(*kv, *at, sum(new), F32, *exps)
        if cache is None:
            assert torch.equal(read_k, k.float())
        else:
            # int8: top > 127 2^(e - 1), so half a step, 2^(e - 1), is less than top / 127 (and may be more than top / 128); e4m3: half a step of three bits
            top = k.float().abs().amax(-1, keepdim=True)
            assert bool(((read_k - k.float()).abs() <= top * (2.0 ** -4 if cache == E4M3 else 1 / 127)).all())
        for b, n in enumerate(accepted.tolist()):
            generated[b] += tokens[b, :n + 1].tolist()
            lens[b] -= K - n                                     # the rejected positions are free again
    assert all(0 <= t < V for s in generated for t in s)


def test_other_streams_and_replays(core):
    """The calls on a stream of their own, recorded and replayed with other contents of the same buffers (lengths, pages, tokens among them), with eager work between the
    replays; two graphs on workspaces of their own."""
    heads, G, D, V, page, K = 2, 4, 128, 3000, 16, 3
    batch = ref.make_batch([4, 4], [2600, 2200], page, 111)
    need = None
    variants = []
    for i, (lens, seed) in enumerate([([2600, 2200], 1), ([100, 2000], 2), ([4, 37], 3)]):
        g = torch.Generator(device='cuda').manual_seed(seed)
        rows = [torch.randn((8, h, D), generator=g, device='cuda').to(F16) for h in (heads, heads, heads * G)]
        probs = [torch.softmax(torch.randn((2, n, V), generator=g, device='cuda') * 2, -1) for n in (K + 1, K)]
        ids = torch.randint(0, V, (2, K), generator=g, device='cuda')
        uniforms = [torch.rand(s, generator=g, device='cuda') * 0.2 for s in ((2, K), (2,))]
        table = torch.tensor(batch['table'], dtype=torch.int32, device='cuda').roll(i, 1)
        variants.append([*rows, table, torch.tensor(lens, dtype=torch.int32, device='cuda'), *probs, ids, *uniforms])
    starts = torch.tensor([0, 4, 8], dtype=torch.int32, device='cuda')
    fresh = lambda: _cuda(ref.make_pages(batch, heads, D, I8, F16, 112))

    def step(x, pages, space, spare):
        k, v, q, table, lens, target, draft, ids, accept, sample = x
        core.kv_cache_write(k, v, *pages[:2], table, lens, starts, *pages[2:])
        read = core.kv_cache_read(*pages[:2], table, lens, starts, 8, F16, *pages[2:])
        o, lse = core.paged_attention(q, *pages[:2], table, lens, starts, *pages[2:], max_queries=4, max_keys=2600, return_lse=True, workspace=space)
        return [*read, o, lse, *core.verify_drafts(target, draft, ids, accept, sample, workspace=spare)]

    need = core.paged_attention_workspace_bytes(variants[0][2], fresh()[0], variants[0][3], 4, 2600)
    assert need > 0
    spaces = lambda: (torch.empty(need, dtype=torch.uint8, device='cuda'), torch.empty(1 << 16, dtype=torch.uint8, device='cuda'))
    want = [[t.clone() for t in step(x, fresh(), *spaces())] for x in variants]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = step(variants[1], fresh(), *spaces())
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    graphs = []
    for _ in range(2):
        x, pages, space = [t.clone() for t in variants[0]], fresh(), spaces()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(x, pages, *space)
        graphs.append((graph, x, pages, space, out))
    clean = fresh()
    for turn in range(6):
        for i, (graph, x, pages, space, out) in enumerate(graphs):
            for a, b in zip(pages, clean):
                a.copy_(b)
            for a, b in zip(x, variants[(turn + i) % 3]):
                a.copy_(b)
        torch.cuda.synchronize()
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i, (_, _, _, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(turn + i) % 3])), (turn, i)
        eager = step(variants[turn % 3], fresh(), *spaces())
        assert all(torch.equal(a, b) for a, b in zip(eager, want[turn % 3]))


# ---- on FractalTensors --------------------------------------------------------------------

@pytest.mark.parametrize('new,dtype,cache', [([3, 1, 17], F16, E4M3), ([2, 2], F32, I8), ([4, 0, 1], F32, 'bf16')])
def test_serving_on_fractal_tensors(core, new, dtype, cache):
    """Sequences of any number of tokens as FractalTensors: the same as the packed rows, to the bit."""
    from fractaltensor_amd.kaleido import FractalTensor, operations as ops
    heads, G, D, page = 2, 3, 64, 16
    held = BF16 if cache == 'bf16' else F16                      # what the tokens are rounded to
    batch = ref.make_batch(new, [n + 21 for n in new], page, 121)
    table, lens, starts = ref.on_device(batch)
    pages = _cuda(ref.make_pages(batch, heads, D, None if cache == 'bf16' else cache, held, 122))
    other = [None if t is None else t.clone() for t in pages]
    g = torch.Generator(device='cuda').manual_seed(123)
    k, v, q = [torch.randn((sum(new), h, D), generator=g, device='cuda').to(dtype) for h in (heads, heads, heads * G)]
    as_ft = lambda t: ops.fused._by_sequence(t, new)
    assert as_ft(q).width_by_depth(1) == new and isinstance(as_ft(q), FractalTensor)
    core.kv_cache_write(k.to(held), v.to(held), *pages[:2], table, lens, starts, *pages[2:])
    want = core.paged_attention(q.to(held), *pages[:2], table, lens, starts, *pages[2:], scale=0.2, window=30, max_queries=max(new), max_keys=40).to(dtype)
    ops.fused.kv_cache_write(as_ft(k), as_ft(v), *other[:2], table, lens, *other[2:])
    assert all(a is None or _same(a, b) for a, b in zip(pages, other))
    got = ops.fused.paged_attention(as_ft(q), *other[:2], table, lens, *other[2:], scale=0.2, window=30, max_keys=40)
    assert got.depth == 2 and got.width_by_depth(1) == new and got.element_shape == (heads * G, D) and got.data.dtype == dtype
    assert torch.equal(got.data.view_as(want), want)
    back = ops.fused.kv_cache_read(*other[:2], table, lens, new, F32, *other[2:])
    for a, b in zip(back, core.kv_cache_read(*pages[:2], table, lens, starts, sum(new), F32, *pages[2:])):
        assert a.width_by_depth(1) == new and torch.equal(a.data.view_as(b), b)
    one = got[0][0].data                                         # the first token alone, through an ordinary index
    assert torch.equal(one, want[0])
    with pytest.raises(ValueError, match='one structure'):
        ops.fused.kv_cache_write(as_ft(k), ops.fused._by_sequence(v, [sum(new)]), *other[:2], table, lens, *other[2:])
    with pytest.raises(ValueError, match='depth 2'):
        ops.fused.paged_attention(FractalTensor.from_dense(q, 1), *other[:2], table, lens, *other[2:])


@pytest.mark.parametrize('cache', [E4M3, I8])
def test_bf16_rows_in_codes_on_fractal_tensors(core, cache):
    """Values beyond fp16's range: written and attended to in bf16, as the packed rows are, to the bit."""
    from fractaltensor_amd.kaleido import operations as ops
    heads, G, D, page, new = 2, 3, 64, 16, [3, 1, 17]
    batch = ref.make_batch(new, new, page, 261)
    table, lens, starts = ref.on_device(batch)
    pages, other = ([t.cuda() for t in ref.make_pages(batch, heads, D, cache, BF16, 262)] for _ in range(2))
    g = torch.Generator(device='cuda').manual_seed(263)
    k, v, q = (torch.randn((sum(new), h, D), generator=g, device='cuda') for h in (heads, heads, heads * G))
    v *= 1e6
    core.kv_cache_write(k.to(BF16), v.to(BF16), *pages[:2], table, lens, starts, *pages[2:])
    want = core.paged_attention(q.to(BF16), *pages[:2], table, lens, starts, *pages[2:], scale=0.2, max_queries=max(new)).float()
    as_ft = lambda t: ops.fused._by_sequence(t, new)
    ops.fused.kv_cache_write(as_ft(k), as_ft(v), *other[:2], table, lens, *other[2:], dtype=BF16)
    assert all(_same(a, b) for a, b in zip(pages, other))
    got = ops.fused.paged_attention(as_ft(q), *other[:2], table, lens, *other[2:], scale=0.2, dtype=BF16)
    assert bool(torch.isfinite(want).all()) and float(want.abs().max()) > 1e5 and torch.equal(got.data.view_as(want), want)
    with pytest.raises(TypeError, match='float16 or bfloat16'):
        ops.fused.paged_attention(as_ft(q), *other[:2], table, lens, *other[2:], dtype=F32)
    with pytest.raises(TypeError, match='that of the pages'):
        ops.fused.paged_attention(as_ft(q), *[t.half() for t in pages[:2]], table, lens, dtype=BF16)


def test_verification_on_fractal_tensors(core):
    from fractaltensor_amd.kaleido import FractalTensor, operations as ops
    B, K, V = 5, 4, 300
    target, draft, drafts, accept, sample = _drafts(B, K, V, F32, True, 131)
    want = ref.verify(target, draft, drafts, accept, sample)
    target, draft, drafts, accept, sample = (t.cuda() for t in (target, draft, drafts, accept, sample))
    ft = lambda t: FractalTensor.from_dense(t.reshape(*t.shape[:2], 1, V), 2)
    got = ops.fused.verify_drafts(ft(target), FractalTensor.from_dense(drafts.reshape(B, K, 1), 2), accept, sample, ft(draft))
    counts = [n + 1 for n in want[1].tolist()]
    assert got.depth == 2 and got.width_by_depth(1) == counts and got.data.dtype == torch.int64
    assert got.data.tolist() == [t for b, n in enumerate(counts) for t in want[0][b, :n].tolist()]
    with pytest.raises(ValueError, match=r'\[1, V\] items'):
        ops.fused.verify_drafts(FractalTensor.from_dense(target, 2), FractalTensor.from_dense(drafts.reshape(B, K, 1), 2), accept, sample)


@pytest.mark.parametrize('counts', [[3, 0, 5, 1], [0, 0, 0], [2, 2, 0]])
@pytest.mark.parametrize('drawn', [True, False])
def test_ragged_drafts_on_fractal_tensors(core, counts, drawn):
    """Sequences with different numbers of drafts, none among them."""
    from fractaltensor_amd.kaleido import operations as ops
    B, K, V = len(counts), max(counts), 300
    target, draft, drafts, accept, sample = _drafts(B, K, V, F32, True, 141)
    want = ref.verify(target, draft if drawn else None, drafts, accept, sample, counts)
    rows = lambda t, more: torch.cat([t[b, :n + more] for b, n in enumerate(counts)]).cuda()
    as_ft = lambda t, more: ops.fused._by_sequence(t, [n + more for n in counts])
    p, q, d = as_ft(rows(target, 1).view(-1, 1, V), 1), as_ft(rows(draft, 0).view(-1, 1, V), 0), as_ft(rows(drafts, 0).view(-1, 1), 0)
    got = ops.fused.verify_drafts(p, d, accept.cuda(), sample.cuda(), q if drawn else None)
    left = [n + 1 for n in want[1].tolist()]
    assert got.width_by_depth(1) == left and got.data.tolist() == [t for b, n in enumerate(left) for t in want[0][b, :n].tolist()]
    if counts[0]:
        with pytest.raises(ValueError, match='tokens a sequence'):
            ops.fused.verify_drafts(q, d, accept.cuda(), sample.cuda())
