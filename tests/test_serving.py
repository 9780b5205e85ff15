"""The serving entry points: what they refuse, before anything touches a device, and their plain forms against hand-made values."""
import ctypes
import math

import pytest
import torch

import serving_reference as ref


@pytest.fixture(scope='module')
def core():
    import fractaltensor_amd._core as c
    return c


ONE = 16            # never dereferenced: validation fails first


def _pages(core, **over):
    d = dict(k=ONE, v=ONE, k_exps=None, v_exps=None, type=0, pages=4, heads=2, page_size=16, head_size=64)
    d.update(over)
    return core.KvPages(*[d[n] for n, _ in core.KvPages._fields_])


def _batch(core, **over):
    d = dict(table=ONE, lens=ONE, starts=ONE, sequences=1, table_width=1, tokens=1)
    d.update(over)
    return core.KvBatch(*[d[n] for n, _ in core.KvBatch._fields_])


BAD_CACHES = [
    (dict(k=None), {}, -1, b'non-NULL'),
    (dict(type=4), {}, -1, b'type of pages'),
    (dict(pages=0), {}, -1, b'positive'),
    (dict(heads=-1), {}, -1, b'positive'),
    (dict(page_size=24), {}, -2, b'page size'),
    (dict(page_size=8), {}, -2, b'page size'),
    (dict(page_size=2048), {}, -2, b'page size'),
    (dict(head_size=80), {}, -2, b'head size'),
    (dict(type=2), {}, -1, b'exponents'),
    (dict(k_exps=ONE, v_exps=ONE), {}, -1, b'exponents'),
    (dict(type=3, k_exps=ONE), {}, -1, b'exponents'),
    (dict(k=24), {}, -1, b'aligned'),
    ({}, dict(table=None), -1, b'non-NULL'),
    ({}, dict(sequences=-1), -1, b'negative'),
    ({}, dict(tokens=-1), -1, b'negative'),
    ({}, dict(table_width=0), -1, b'columns'),
    ({}, dict(lens=18), -1, b'aligned'),
    ({}, dict(tokens=(1 << 28) + 1), -2, b'2^28'),
]


@pytest.mark.parametrize('pages,batch,code,text', BAD_CACHES)
def test_bad_caches_and_batches_are_refused(core, pages, batch, code, text):
    lib, ci, cl, one, nul = core.lib, ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p(ONE), ctypes.c_void_p(0)
    p, b = ctypes.byref(_pages(core, **pages)), ctypes.byref(_batch(core, **batch))
    calls = [lambda: lib.ftk_kv_cache_write(one, one, ci(0), cl(128), cl(64), cl(128), cl(64), p, b, nul),
             lambda: lib.ftk_kv_cache_read(p, b, ci(0), one, one, nul),
             lambda: lib.ftk_paged_attn(one, ci(0), cl(128), cl(64), p, b, one, nul, ci(4), ctypes.c_float(1), ci(1), ci(0), ci(0), ci(0), nul, ctypes.c_size_t(0), nul)]
    for call in calls:
        assert call() == code
        assert text in lib.ftk_last_error()


def test_bad_operands_of_the_cache_calls_are_refused(core):
    lib, ci, cl, nul = core.lib, ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p(0)
    vp = ctypes.c_void_p
    p, b = ctypes.byref(_pages(core)), ctypes.byref(_batch(core))
    write = lambda k=ONE, v=ONE, type=0, kt=128, vh=64: lib.ftk_kv_cache_write(vp(k), vp(v), ci(type), cl(kt), cl(64), cl(128), cl(vh), p, b, nul)
    assert write(k=None) == -1
    assert write(type=1) == -1 and b'type' in lib.ftk_last_error()          # bf16 into fp16 pages
    assert write(type=4) == -1
    assert write(kt=100) == -1 and b'strides' in lib.ftk_last_error()
    assert write(vh=-64) == -1
    assert write(v=24) == -1 and b'aligned' in lib.ftk_last_error()
    read = lambda type=0, k=ONE: lib.ftk_kv_cache_read(p, b, ci(type), vp(k), vp(ONE), nul)
    assert read(type=1) == -1
    assert read(type=2) == -1
    assert read(k=8) == -1
    assert read(k=None) == -1
    f = lambda q=ONE, type=0, qt=256, heads=4, scale=1.0, window=0, mq=0, ws=None, n=0, lse=None, o=ONE: lib.ftk_paged_attn(
        vp(q), ci(type), cl(qt), cl(64), p, b, vp(o), vp(lse), ci(heads), ctypes.c_float(scale), ci(1), ci(window), ci(mq), ci(0), vp(ws), ctypes.c_size_t(n), nul)
    assert f(heads=3) == -1 and b'multiple' in lib.ftk_last_error()
    assert f(heads=0) == -1
    assert f(type=1) == -1
    assert f(type=3) == -1
    assert f(scale=0.0) == -1 and f(scale=-1.0) == -1 and f(scale=math.inf) == -1 and f(scale=math.nan) == -1
    assert f(window=-1) == -1
    assert f(mq=-1) == -1
    assert f(q=None) == -1 and f(o=24) == -1
    assert f(qt=100) == -1
    assert f(lse=18) == -1
    # nothing to do: no rows, no sequences
    for empty in (dict(tokens=0), dict(sequences=0, table=None, lens=None, starts=None)):
        e = ctypes.byref(_batch(core, **empty))
        assert lib.ftk_kv_cache_write(vp(None), vp(None), ci(0), cl(0), cl(0), cl(0), cl(0), p, e, nul) == 0
        assert lib.ftk_kv_cache_read(p, e, ci(0), vp(None), vp(None), nul) == 0
        assert lib.ftk_paged_attn(vp(None), ci(0), cl(0), cl(0), p, e, vp(None), nul, ci(4), ctypes.c_float(1), ci(1), ci(0), ci(0), ci(0), nul, ctypes.c_size_t(0), nul) == 0
    assert lib.ftk_paged_attn_workspace_bytes(None, None, 1, 0, 0, 0) == 0


def test_bad_operands_of_the_verification_are_refused(core):
    lib, ci, vp, nul = core.lib, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p(0)
    need = lib.ftk_verify_drafts_workspace_bytes(2, 5000)
    assert need == 2 * 3 * 16                                               # three segments of 2048, two sums of 64 bits each
    f = lambda target=ONE, draft=ONE, type=4, drafts=ONE, wide=0, acc=ONE, smp=ONE, lens=None, out=ONE, B=2, K=3, V=5000, ws=ONE, n=1 << 20: lib.ftk_verify_drafts(
        vp(target), vp(draft), ci(type), vp(drafts), ci(wide), vp(acc), vp(smp), vp(lens), vp(out), vp(ONE), ci(B), ci(K), ci(V), vp(ws), ctypes.c_size_t(n), nul)
    assert f(B=-1) == -1 and f(V=0) == -1 and f(K=-1) == -1
    assert f(K=64) == -2 and f(V=(1 << 30) + 1) == -2
    assert f(type=2) == -1 and f(type=3) == -1
    assert f(target=None) == -1 and f(drafts=None) == -1 and f(acc=None) == -1 and f(smp=None) == -1 and f(out=None) == -1
    assert f(target=18) == -1 and f(drafts=20, wide=1) == -1 and f(lens=18) == -1
    assert f(ws=None) == -3 and f(n=need - 1) == -3 and f(ws=20) == -3
    assert f(B=0) == 0


def test_wrappers_say_what_is_wrong(core):
    """Host tensors are refused by name; types and shapes before devices."""
    h = torch.float16
    pages = torch.zeros((2, 2, 16, 64), dtype=h)
    table, lens, starts = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    rows = torch.zeros((1, 2, 64), dtype=h)
    with pytest.raises(RuntimeError, match='no CPU path'):
        core.kv_cache_write(rows, rows, pages, pages, table, lens, starts)
    with pytest.raises(RuntimeError, match='no CPU path'):
        core.kv_cache_read(pages, pages, table, lens, starts, tokens=1)
    with pytest.raises(RuntimeError, match='no CPU path'):
        core.paged_attention(rows, pages, pages, table, lens, starts)
    with pytest.raises(TypeError, match='k_pages must be float16'):
        core.paged_attention(rows, pages.double(), pages, table, lens, starts)
    with pytest.raises(ValueError, match='kv heads'):
        core.paged_attention(rows, pages[0], pages, table, lens, starts)
    with pytest.raises(RuntimeError, match='no CPU path'):
        core.verify_drafts(torch.zeros(1, 2, 8), None, torch.zeros((1, 1), dtype=torch.int64), torch.zeros(1, 1), torch.zeros(1))
    with pytest.raises(TypeError, match='drafts must be int32'):
        core.verify_drafts(torch.zeros(1, 2, 8), None, torch.zeros((1, 1)), torch.zeros(1, 1), torch.zeros(1))
    with pytest.raises(TypeError, match='target must be'):
        core.verify_drafts(torch.zeros(1, 2, 8).double(), None, torch.zeros((1, 1), dtype=torch.int64), torch.zeros(1, 1), torch.zeros(1))


def test_what_is_not_a_tensor_is_refused_by_name(core):
    pages = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    table, lens, starts = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    rows = torch.zeros((1, 2, 64), dtype=torch.float16)
    for dtype in (None, torch.float32):
        with pytest.raises(TypeError, match='k_pages must be a torch.Tensor'):
            core.kv_cache_read([pages], pages, table, lens, starts, 1, dtype)
    with pytest.raises(TypeError, match='v_pages must be a torch.Tensor'):
        core.kv_cache_read(pages, None, table, lens, starts, 1)
    with pytest.raises(TypeError, match='k_pages must be a torch.Tensor'):
        core.kv_cache_write(rows, rows, None, pages, table, lens, starts)
    with pytest.raises(TypeError, match='k_pages must be a torch.Tensor'):
        core.paged_attention(rows, pages.numpy(), pages, table, lens, starts)
    with pytest.raises(TypeError, match='must be torch.Tensors'):
        core.verify_drafts([0.5], None, [1], [0.5], [0.5])


def test_scales_whose_product_with_log2_e_is_not_finite_are_refused(core):
    lib, ci, cl, vp = core.lib, ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p
    p, b = ctypes.byref(_pages(core)), ctypes.byref(_batch(core))
    f = lambda scale, o: lib.ftk_paged_attn(vp(ONE), ci(0), cl(256), cl(64), p, b, vp(o), vp(None), ci(4), ctypes.c_float(scale), ci(1), ci(0), ci(0), ci(0), vp(None), ctypes.c_size_t(0),
                                            vp(None))
    for scale in (2.4e38, 2.9e38, 3.4e38):
        assert f(scale, 24) == -1 and b'scale' in lib.ftk_last_error()
    assert f(2.3e38, 24) == -1 and b'aligned' in lib.ftk_last_error()          # (refused for the address of o)


# ---- the reference itself ------------------------------------------------------------

def test_reference_codes():
    h, b, e4, i8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn, torch.int8
    assert ref.quantise_row([127.0, 0.5, 1.5, -2.5], h, i8) == ([127.0, 0.0, 2.0, -2.0], 0)
    assert ref.quantise_row([127.5, 1.0], h, i8) == ([64.0, 0.0], 1)                # half a code: to the even one
    assert ref.quantise_row([448.0, 17.0, 19.0], b, e4) == ([448.0, 16.0, 20.0], 0)
    assert ref.quantise_row([0.0, 0.0], b, e4) == ([0.0, 0.0], -100)
    assert ref.quantise_row([2.0 ** -24], h, i8) == ([1.0], -24)
    assert ref.quantise_row([2.0 ** -24], h, e4) == ([2.0 ** -9], -15)
    assert ref.quantise_row([65504.0], h, i8) == ([127.0], 9)
    assert ref.quantise_row([math.inf], h, e4) == ([240.0], 8)
    values = ref.e4m3_values()
    codes = torch.arange(256, dtype=torch.uint8).view(e4).double()
    assert torch.equal(torch.nan_to_num(values, nan=-1.0), torch.nan_to_num(codes, nan=-1.0))


@pytest.mark.parametrize('dtype,cache', [(d, c) for d in (torch.float16, torch.bfloat16) for c in (torch.float8_e4m3fn, torch.int8)])
def test_reference_codes_stand_for_values_of_their_type(dtype, cache):
    """code * 2^e is a number of the 16-bit type a row came from, at both ends of its range too."""
    g = torch.Generator().manual_seed(1)
    info = torch.finfo(dtype)
    for scale in (1.0, info.max / 4, info.tiny, 2.0 ** -24, 1e-3):
        x = (torch.randn(64, generator=g) * scale).clamp(-info.max, info.max).to(dtype)
        codes, e = ref.quantise_row(x, dtype, cache)
        for c in codes:
            v = torch.tensor(c * 2.0 ** e, dtype=torch.float64)
            assert float(v.to(dtype)) == float(v)
        if scale == info.max / 4:
            codes, e = ref.quantise_row(torch.tensor([info.max]), dtype, cache)
            assert math.isfinite(float(torch.tensor(codes[0] * 2.0 ** e, dtype=torch.float64).to(dtype)))


def test_fractal_tensors_on_the_cpu_are_refused():
    from fractaltensor_amd.kaleido import FractalTensor, operations as ops
    x = FractalTensor.from_dense(torch.zeros(2, 3, 2, 64), 2)
    pages = [torch.zeros(4, 2, 16, 64, dtype=torch.float16) for _ in range(2)]
    table, lens = torch.zeros((2, 2), dtype=torch.int32), torch.full((2,), 3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match='GPU only'):
        ops.fused.kv_cache_write(x, x, *pages, table, lens)
    with pytest.raises(RuntimeError, match='GPU only'):
        ops.fused.paged_attention(x, *pages, table, lens)
    with pytest.raises(ValueError, match='not be negative'):
        ops.fused.kv_cache_read(*pages, table, lens, [1, -1])
    with pytest.raises(TypeError, match='should be a FractalTensor'):
        ops.fused.paged_attention(x.data, *pages, table, lens)
    probs, ids = FractalTensor.from_dense(torch.zeros(2, 3, 1, 8), 2), FractalTensor.from_dense(torch.zeros(2, 2, 1, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match='GPU only'):
        ops.fused.verify_drafts(probs, ids, torch.zeros(2, 2), torch.zeros(2))
