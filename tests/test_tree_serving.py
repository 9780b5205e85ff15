"""Trees of drafts and caches of limited length: what the calls refuse, before anything touches a device, and their plain forms against hand-made values."""
import ctypes
import math

import pytest
import torch

import tree_reference as ref


@pytest.fixture(scope='module')
def core():
    import fractaltensor_amd._core as c
    return c


ONE = 16            # never dereferenced: validation fails first
ci, cl, cf, vp, NUL = ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_void_p, ctypes.c_void_p(0)


def _pages(core, **over):
    d = dict(k=ONE, v=ONE, k_exps=None, v_exps=None, type=0, pages=4, heads=2, page_size=16, head_size=64)
    d.update(over)
    return core.KvPages(*[d[n] for n, _ in core.KvPages._fields_])


def _batch(core, **over):
    d = dict(table=ONE, lens=ONE, starts=ONE, sequences=1, table_width=1, tokens=1)
    d.update(over)
    return core.KvBatch(*[d[n] for n, _ in core.KvBatch._fields_])


def _tree(core, q=ONE, type=0, qt=256, heads=4, scale=1.0, window=0, mq=0, mk=0, ws=None, n=0, lse=None, o=ONE, parents=ONE, pages={}, batch={}):
    return core.lib.ftk_paged_tree_attn(vp(q), ci(type), cl(qt), cl(64), ctypes.byref(_pages(core, **pages)), ctypes.byref(_batch(core, **batch)), vp(parents), vp(o), vp(lse),
                                        ci(heads), cf(scale), ci(window), ci(mq), ci(mk), vp(ws), ctypes.c_size_t(n), NUL)


def _weigh(core, q=ONE, type=0, qt=256, lse=ONE, weights=ONE, heads=4, scale=1.0, decay=1.0, window=0, mq=0, mk=0, ws=None, n=0, pages={}, batch={}):
    return core.lib.ftk_kv_cache_weigh(vp(q), ci(type), cl(qt), cl(64), vp(lse), ctypes.byref(_pages(core, **pages)), vp(weights), ctypes.byref(_batch(core, **batch)), ci(heads),
                                       cf(scale), cf(decay), ci(1), ci(window), ci(mq), ci(mk), vp(ws), ctypes.c_size_t(n), NUL)


def _keep(core, table=ONE, lens=ONE, starts=None, B=1, W=1, kept=ONE, most=4, per_head=0, weights=None, out=32, pages={}):
    return core.lib.ftk_kv_cache_keep(ctypes.byref(_pages(core, **pages)), vp(table), vp(lens), vp(starts), ci(B), ci(W), vp(kept), ci(most), ci(per_head), vp(weights), vp(out), NUL)


BAD_PAGES = [(dict(k=None), -1, b'non-NULL'), (dict(type=4), -1, b'type of pages'), (dict(pages=0), -1, b'positive'), (dict(page_size=24), -2, b'page size'),
             (dict(head_size=80), -2, b'head size'), (dict(type=2), -1, b'exponents'), (dict(k_exps=ONE, v_exps=ONE), -1, b'exponents'), (dict(k=24), -1, b'aligned')]
BAD_BATCHES = [(dict(table=None), -1, b'non-NULL'), (dict(sequences=-1), -1, b'negative'), (dict(tokens=-1), -1, b'negative'), (dict(table_width=0), -1, b'columns'),
               (dict(lens=18), -1, b'aligned'), (dict(tokens=(1 << 28) + 1), -2, b'2^28')]


@pytest.mark.parametrize('pages,code,text', BAD_PAGES)
def test_bad_caches_are_refused(core, pages, code, text):
    for call in (_tree, _weigh, _keep):
        assert call(core, pages=pages) == code and text in core.lib.ftk_last_error()


@pytest.mark.parametrize('batch,code,text', BAD_BATCHES)
def test_bad_batches_are_refused(core, batch, code, text):
    for call in (_tree, _weigh):
        assert call(core, batch=batch) == code and text in core.lib.ftk_last_error()


def test_bad_operands_of_attention_over_a_tree_are_refused(core):
    f = lambda **over: _tree(core, **over)
    assert f(heads=3) == -1 and b'multiple' in core.lib.ftk_last_error()
    assert f(type=1) == -1 and f(type=3) == -1 and f(window=-1) == -1 and f(mq=-1) == -1 and f(mk=-1) == -1
    assert f(scale=0.0) == -1 and f(scale=math.nan) == -1 and f(scale=2.9e38) == -1
    assert f(parents=None) == -1 and b'parents' in core.lib.ftk_last_error()
    assert f(parents=18) == -1
    assert f(q=None) == -1 and f(o=24) == -1 and f(qt=100) == -1 and f(lse=18) == -1
    # 257 new tokens are too many for a tree, whether promised or possible
    assert f(batch=dict(tokens=300), o=24) == -2 and b'256' in core.lib.ftk_last_error()
    assert f(batch=dict(tokens=300), mq=257, o=24) == -2
    assert f(batch=dict(tokens=300), mq=256, o=24) == -1 and b'aligned' in core.lib.ftk_last_error()
    assert f(batch=dict(tokens=256), o=24) == -1
    assert f(batch=dict(tokens=0), q=None, o=None, parents=None) == 0
    assert core.lib.ftk_paged_tree_attn_workspace_bytes(None, None, 1, 0, 0, 0) == 0


def test_bad_operands_of_weighing_are_refused(core):
    f = lambda **over: _weigh(core, **over)
    assert f(heads=3) == -1 and f(heads=0) == -1 and f(type=1) == -1 and f(type=4) == -1 and f(window=-1) == -1 and f(mq=-1) == -1 and f(mk=-1) == -1
    assert f(scale=-1.0) == -1 and f(scale=math.inf) == -1 and f(scale=2.9e38) == -1
    assert f(decay=-0.1) == -1 and f(decay=1.1) == -1 and f(decay=math.nan) == -1 and b'decay' in core.lib.ftk_last_error()
    assert f(q=None) == -1 and f(lse=None) == -1 and f(weights=None) == -1 and f(q=24) == -1 and f(lse=18) == -1 and f(weights=18) == -1 and f(qt=100) == -1 and f(ws=24, n=100) == -1
    assert core.lib.ftk_kv_cache_weigh_workspace_bytes(None, None, 1, 0, 0) == 0
    assert f(batch=dict(tokens=0), q=None, lse=None, weights=None) == 0
    assert f(pages=dict(v=None), batch=dict(tokens=0)) == 0                    # values are not looked at


def test_bad_operands_of_selecting_are_refused(core):
    f = lambda weights=ONE, pages=4, heads=2, page=16, table=ONE, lens=ONE, B=1, W=1, budget=8, sinks=0, recent=0, mk=0, kept=ONE: core.lib.ftk_kv_cache_select(
        vp(weights), ci(pages), ci(heads), ci(page), vp(table), vp(lens), ci(B), ci(W), ci(budget), ci(sinks), ci(recent), ci(mk), vp(kept), NUL)
    assert f(weights=None) == -1 and f(weights=20) == -1 and f(pages=0) == -1 and f(heads=0) == -1 and f(page=24) == -2 and f(page=2048) == -2
    assert f(B=-1) == -1 and f(W=-1) == -1 and f(mk=-1) == -1 and f(W=0) == -1
    assert f(budget=0) == -1 and f(sinks=-1) == -1 and f(recent=-1) == -1 and f(sinks=5, recent=4) == -1 and b'budget' in core.lib.ftk_last_error()
    assert f(budget=2 ** 31 - 1, sinks=2 ** 31 - 1, recent=2 ** 31 - 1) == -1
    assert f(table=None) == -1 and f(lens=None) == -1 and f(kept=None) == -1 and f(kept=18) == -1
    assert f(B=1 << 20, heads=1 << 12) == -2
    assert f(B=0, table=None, lens=None, kept=None) == 0


def test_bad_operands_of_keeping_are_refused(core):
    f = lambda **over: _keep(core, **over)
    assert f(B=-1) == -1 and f(W=-1) == -1 and f(most=-1) == -1 and f(W=0) == -1
    assert f(table=None) == -1 and f(lens=None) == -1 and f(kept=None) == -1 and f(out=None) == -1
    assert f(kept=18) == -1 and f(starts=18) == -1 and f(weights=18) == -1
    assert f(out=ONE) == -1 and b'old ones' in core.lib.ftk_last_error()
    assert f(B=0, table=None, lens=None, kept=None) == 0


def test_bad_operands_of_the_verification_are_refused(core):
    f = lambda target=ONE, type=4, ids=ONE, wide=0, parents=ONE, starts=ONE, u=ONE, out=ONE, path=ONE, acc=ONE, B=2, T=5, M=4, V=100, ws=None: core.lib.ftk_verify_tree(
        vp(target), ci(type), vp(ids), ci(wide), vp(parents), vp(starts), vp(u), vp(out), vp(path), vp(acc), ci(B), ci(T), ci(M), ci(V), vp(ws), ctypes.c_size_t(1 << 20), NUL)
    assert f(B=-1) == -1 and f(T=-1) == -1 and f(V=0) == -1 and f(M=0) == -1
    assert f(M=65) == -2 and f(V=(1 << 30) + 1) == -2
    assert f(type=2) == -1 and f(type=3) == -1
    for name in ('target', 'ids', 'parents', 'starts', 'u', 'out', 'path', 'acc'):
        assert f(**{name: None}) == -1 and f(**{name: 18 if name != 'target' else 17}) == -1
    assert f(ids=20, wide=1) == -1 and f(ws=24) == -1
    assert core.lib.ftk_verify_tree_workspace_bytes(5) == 20 and core.lib.ftk_verify_tree_workspace_bytes(-1) == 0
    assert f(B=0) == 0


def test_wrappers_say_what_is_wrong(core):
    """Host tensors are refused by name; types and shapes before devices."""
    h, i32 = torch.float16, torch.int32
    pages = torch.zeros((2, 2, 16, 64), dtype=h)
    table, lens, starts, parents = torch.zeros((1, 1), dtype=i32), torch.ones(1, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32)
    rows, lse, weights = torch.zeros((1, 2, 64), dtype=h), torch.zeros((1, 2)), torch.zeros((2, 2, 16))
    for call in (lambda: core.paged_tree_attention(rows, pages, pages, table, lens, starts, parents), lambda: core.kv_cache_weigh(rows, lse, pages, weights, table, lens, starts),
                 lambda: core.kv_cache_select(weights, table, lens, 4), lambda: core.kv_cache_keep(pages, pages, table, lens, torch.zeros((1, 2), dtype=i32)),
                 lambda: core.verify_tree(torch.zeros(1, 8), parents, parents, starts, torch.zeros(1, 2))):
        with pytest.raises(RuntimeError, match='no CPU path'):
            call()
    with pytest.raises(TypeError, match='k_pages must be float16'):
        core.paged_tree_attention(rows, pages.double(), pages, table, lens, starts, parents)
    with pytest.raises(TypeError, match='k_pages must be a torch.Tensor'):
        core.kv_cache_weigh(rows, lse, None, weights, table, lens, starts)
    with pytest.raises(TypeError, match='k_pages must be a torch.Tensor'):
        core.kv_cache_keep([pages], pages, table, lens, parents)
    with pytest.raises(TypeError, match='weights must be a torch.Tensor'):
        core.kv_cache_select([1.0], table, lens, 4)
    with pytest.raises(TypeError, match='must be torch.Tensors'):
        core.verify_tree([0.5], None, None, None, None)
    with pytest.raises(TypeError, match='ids must be int32'):
        core.verify_tree(torch.zeros(1, 8), torch.zeros(1), parents, starts, torch.zeros(1, 2))
    with pytest.raises(ValueError, match=r'target must be \[tokens, V\]'):
        core.verify_tree(torch.zeros(1, 1, 8), parents, parents, starts, torch.zeros(1, 2))


# ---- the reference itself ------------------------------------------------------------

def test_reference_trees():
    #      0
    #    1   2
    #   3   4 5
    parents = [-1, 0, 0, 1, 2, 2]
    assert ref.way(parents, 5) == [5, 2, 0] and ref.way(parents, 3) == [3, 1, 0]
    assert ref.way([-1, 1, 7], 1) == [1] and ref.way([-1, 1, 7], 2) == [2]
    seen = ref.tree_sees(parents, 6, 2, 8)
    assert seen[5].tolist() == [True, True, True, False, True, False, False, True]
    seen = ref.tree_sees(parents, 6, 2, 8, window=2)
    assert seen[5].tolist() == [False, False, False, False, True, False, False, True]
    assert seen[0].tolist() == [False, True, True, False, False, False, False, False]
    chain = list(range(-1, 4))
    for window in (0, 1, 3, 6, 50):
        assert torch.equal(ref.tree_sees(chain, 5, 7, 12, window), ref.causal_sees(5, 7, 12, True, window))


def test_reference_selection_and_moves():
    w = torch.tensor([3.0, 1.0, 4.0, 1.0, 5.0, 9.0, 2.0, 6.0] + [0.0] * 8).view(1, 1, 16)
    assert ref.select(w, [[0]], [8], 16, 4, 0, 0).tolist() == [[[2, 4, 5, 7]]]
    assert ref.select(w, [[0]], [8], 16, 5, 2, 1).tolist() == [[[0, 1, 4, 5, 7]]]
    assert ref.select(w, [[0]], [8], 16, 6, 0, 0).tolist() == [[[0, 2, 4, 5, 6, 7]]]
    assert ref.select(w, [[0]], [8], 16, 7, 0, 0).tolist() == [[[0, 1, 2, 4, 5, 6, 7]]]       # of two ones the earlier
    assert ref.select(w, [[0]], [3], 16, 4, 0, 0).tolist() == [[[0, 1, 2, -1]]]
    a = torch.arange(16.0).view(1, 1, 16)
    assert ref.keep([a], [[0]], [10], [4], torch.tensor([[0, 2, 5, -1]]), 16).tolist() == [7]
    assert a.view(-1).tolist() == [0, 1, 2, 3, 4, 6, 9, 7, 8, 9, 10, 11, 12, 13, 14, 15]


def test_reference_verification():
    p = torch.tensor([[0.0, 0.5, 0.5], [1.0, 0.0, 0.0], [0.25, 0.25, 0.5]])
    ids, parents = torch.tensor([9, 1, 2]), torch.tensor([-1, 0, 0])
    got = ref.verify(p, ids, parents, [0, 3], torch.tensor([[0.6, 0.3, 0.0]]))
    assert [t.tolist() for t in got] == [[[2, 1, -1]], [[0, 2, -1]], [1]]
    got = ref.verify(p, ids, parents, [0, 3], torch.tensor([[0.0]]))
    assert [t.tolist() for t in got] == [[[1]], [[0]], [0]]


def test_fractal_tensors_are_refused_by_name():
    from fractaltensor_amd.kaleido import FractalTensor, operations as ops
    pages, table, lens = torch.zeros((2, 2, 16, 32), dtype=torch.float16), torch.zeros((2, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = FractalTensor.from_dense(torch.zeros((2, 3, 4, 32), dtype=torch.float16), 2)
    ids = FractalTensor.from_dense(torch.zeros((2, 3, 1), dtype=torch.int64), 2)
    for call, error, text in (
            (lambda: ops.fused.paged_tree_attention(q, ids, pages, pages, table, lens), RuntimeError, 'qss lives on cpu'),
            (lambda: ops.fused.paged_tree_attention(table, ids, pages, pages, table, lens), TypeError, 'qss should be a FractalTensor'),
            (lambda: ops.fused.verify_tree(q, ids, ids, torch.zeros(2, 2)), RuntimeError, 'tokens lives on cpu'),
            (lambda: ops.fused.verify_tree(q, table, ids, torch.zeros(2, 2)), TypeError, 'tokens should be a FractalTensor'),
            (lambda: ops.fused.verify_tree(q, q, ids, torch.zeros(2, 2)), ValueError, 'single integers'),
            (lambda: ops.fused.kv_cache_select(table, table, lens, 3), (TypeError, RuntimeError, ValueError), 'weights'),
            (lambda: ops.fused.kv_cache_keep(pages, pages, table, lens, table), (TypeError, RuntimeError, ValueError), 'k_pages')):
        with pytest.raises(error, match=text):
            call()


def test_parents_outside_of_int32_stay_none():
    from fractaltensor_amd.kaleido.operations import fused
    wide = torch.tensor([2 ** 32, 2 ** 32 + 3, -2 ** 32, -2 ** 63, 2 ** 63 - 1, 2 ** 31, -1, 0, 5, 255])
    assert fused._narrowed(wide).tolist() == [2 ** 31 - 1, 2 ** 31 - 1, -1, -1, 2 ** 31 - 1, 2 ** 31 - 1, -1, 0, 5, 255]
    narrow = torch.tensor([-7, 3], dtype=torch.int32)
    assert fused._narrowed(narrow) is narrow
