"""GPU fast paths: the three hot-path programs of the reference as single
kernel calls on FractalTensors that live on the GPU.

  stacked_lstm   the fold-over-layers / scan-over-time / map-over-batch program of
                 examples/stacked_rnn/stacked_rnn.py:23-79
  dilated_lstm   the dilated_map program of examples/dilated_rnn/dilated_rnn.py:16-41
  flash_attention  the map / reduce program of examples/flash_attention/flash_attention.py:14-91
  b2b_gemm       (a @ b) @ c, the computation of benchmarks/fused_two_hgemms
  grid_rnn       the nested-scan program of examples/grid_rnn/grid_rnn.py:40-137 over a batch of samples
  windowed_attention  shifted_slide + the map of sparse_attn of examples/sparse_attention/sparse_attention.py:25-71
  kv_cache_write, kv_cache_read, paged_attention, verify_drafts   serving: the new tokens of a batch of sequences and a paged cache
                 of keys and values; one sequence is one item of a FractalTensor, of any length
  paged_tree_attention, verify_tree, kv_cache_keep   the same with trees of drafts: what a target model makes of one in a step, and the cache behind it
  kv_cache_select, kv_cache_keep   caches of limited length: which positions stay, by the weights that paged_attention gathers, and moving those

A regular (non-ragged) FractalTensor already is a dense row-major tensor in
its flat buffer, so inputs are handed to the kernels as views and outputs are
wrapped back without copies.  Everything here runs through the C ABI in
fractaltensor_amd._core; there is no CPU or PyTorch fallback: CPU inputs are
rejected, and a missing library is an ImportError.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from ..fractal_tensor import FractalTensor
from ..tensor import Tensor
from ..types import FractalTensorStorage, TensorStorage, torch_type_to_internal_type

__all__ = ['pack_lstm_weights', 'pad_time_major', 'unpad_time_major', 'stacked_lstm', 'dilated_lstm', 'lstm_cell', 'flash_attention', 'b2b_gemm', 'mm',
           'online_softmax', 'embedding_lookup', 'grid_rnn', 'windowed_attention', 'kv_cache_write', 'kv_cache_read', 'paged_attention',
           'verify_drafts', 'paged_tree_attention', 'verify_tree', 'kv_cache_select', 'kv_cache_keep']


def _core():
    from ... import _core
    return _core


def _dense_gpu(ft: FractalTensor, name: str, depth: int) -> torch.Tensor:
    if not isinstance(ft, FractalTensor):
        raise TypeError(f'{name} should be a FractalTensor.')
    if ft.depth != depth:
        raise ValueError(f'{name} should have depth {depth}, got {ft.depth}.')
    if not ft.is_regular():
        raise ValueError(f'{name} is ragged; the fused kernels take regular batches.')
    t = ft.as_dense()
    if not t.is_cuda:
        raise RuntimeError(f'{name} lives on {t.device}; the fused kernels run on the GPU only.')
    return t


def pack_lstm_weights(Wss: FractalTensor, Uss: FractalTensor, bss: Optional[FractalTensor] = None):
    """Per-gate parameters -> the fused layout of the kernels.

    Wss, Uss: depth-2 [L][4] of [H, H] (gate order i, f, o, candidate, as in
    examples/stacked_rnn/rnn_utils.py:28-36); bss: depth-2 [L][4] of [1, H].
    Returns WU [L, 2H, 4H] with column blocks i|f|o|c~ (x rows, then h rows)
    and bias [L, 4H] or None."""
    W = _dense_gpu(Wss, 'Wss', 2)   # [L, 4, H, H]
    U = _dense_gpu(Uss, 'Uss', 2)
    L, G, H, H2 = W.shape
    if G != 4 or H != H2 or U.shape != W.shape:
        raise ValueError('Wss and Uss should be [L][4] of [H, H].')
    WU = torch.cat([W.permute(0, 2, 1, 3).reshape(L, H, 4 * H), U.permute(0, 2, 1, 3).reshape(L, H, 4 * H)], dim=1)
    bias = None
    if bss is not None:
        b = _dense_gpu(bss, 'bss', 2)   # [L, 4, 1, H]
        bias = b.reshape(L, 4 * H).contiguous()
    return WU.contiguous(), bias


def pad_time_major(xss: FractalTensor):
    """Time-major batch [T][B_t] of [1, H] -> (dense [T, B_0, H], batch sizes or None).

    A regular batch is returned as a view.  A ragged one must be what
    examples/utils/data_utils.py:42-66 builds for sequences sorted by length:
    step t holds the first B_t sequences, B_t non-increasing.  It is padded with
    zero rows; rows of a batch are independent in every LSTM layer, so the
    padding rows compute values nobody reads and the rows that matter are exact."""
    if not isinstance(xss, FractalTensor):
        raise TypeError('xss should be a FractalTensor.')
    if xss.depth != 2:
        raise ValueError(f'xss should have depth 2, got {xss.depth}.')
    if xss.is_regular():
        xs = _dense_gpu(xss, 'xss', 2)
        return xs.reshape(xs.shape[0], xs.shape[1], xs.shape[-1]), None
    sizes = [len(step) for step in xss.indices]
    if any(b <= 0 for b in sizes) or any(a < b for a, b in zip(sizes, sizes[1:])):
        raise ValueError('a ragged batch must be time-major with non-increasing, positive batch sizes per step.')
    H = xss.element_shape[-1]
    flat = xss.data.view(-1, H)
    if not flat.is_cuda:
        raise RuntimeError(f'xss lives on {flat.device}; the fused kernels run on the GPU only.')
    xs = torch.zeros((len(sizes), sizes[0], H), dtype=flat.dtype, device=flat.device)
    off = 0
    for t, b in enumerate(sizes):
        xs[t, :b] = flat[off:off + b]
        off += b
    return xs, sizes


def unpad_time_major(dense: torch.Tensor, sizes) -> FractalTensor:
    """dense [T, B_0, H] -> depth-2 [T][B_t] of [1, H] keeping the first B_t rows of step t."""
    T, B0, H = dense.shape
    if sizes is None:
        return FractalTensor.from_dense(dense.reshape(T, B0, 1, H), 2)
    return FractalTensor.from_fractaltensors(
        *[FractalTensor.from_dense(dense[t, :b].reshape(b, 1, H), 1) for t, b in enumerate(sizes)])


def _run_stack(xss, Wss, Uss, bss, dilations, return_all_layers):
    core = _core()
    xs, sizes = pad_time_major(xss)
    WU, bias = pack_lstm_weights(Wss, Uss, bss)
    # a ragged batch goes down with its per-step row counts: 32-row blocks that have ended are skipped
    T_, B_, H_ = xs.shape
    if xs.dtype == torch.float16 and WU.dtype == torch.float16 and H_ % 32 == 0:
        # fp16 program, fp16 kernel: h and c are kept in fp16 like every other tensor of the program
        hsss, csss = core.stacked_lstm_f16(xs, WU, None if bias is None else bias.float(), dilations=dilations,
                                           active_rows=sizes)
    else:
        hsss, csss = core.stacked_lstm(xs.float(), WU.float(), None if bias is None else bias.float(), dilations=dilations,
                                       active_rows=sizes, exact_small_states=True)
    L = WU.shape[0]
    if return_all_layers:
        if sizes is None:
            T, B, H = xs.shape
            return (FractalTensor.from_dense(hsss.view(L, T, B, 1, H), 3),
                    FractalTensor.from_dense(csss.view(L, T, B, 1, H), 3))
        return (FractalTensor.from_fractaltensors(*[unpad_time_major(hsss[l], sizes) for l in range(L)]),
                FractalTensor.from_fractaltensors(*[unpad_time_major(csss[l], sizes) for l in range(L)]))
    return unpad_time_major(hsss[L - 1], sizes)


def stacked_lstm(xss: FractalTensor, Wss: FractalTensor, Uss: FractalTensor, bss: Optional[FractalTensor] = None,
                 return_all_layers: bool = False):
    """Stacked LSTM over a time-major batch.

    xss: depth-2 [T][B_t] of [1, H]: what stacked_rnn.py's `embs` is, either for
    equal-length sequences or the ragged time-major batch of length-sorted
    sequences (shrinking batch per step, stacked_rnn.py:49).  Returns the last layer's hidden sequence as depth-2 [T][B] of
    [1, H], which is what the reference's stacked_lstm returns; with
    return_all_layers the (h, c) of every layer as depth-3 [L][T][B]."""
    return _run_stack(xss, Wss, Uss, bss, None, return_all_layers)


def dilated_lstm(xss: FractalTensor, Wss: FractalTensor, Uss: FractalTensor, bss: Optional[FractalTensor] = None,
                 dilations: Optional[Sequence[int]] = None, return_all_layers: bool = False):
    """Dilated stack: layer k takes its state from step t - dilations[k]
    (default 2**k, the reference's choice, dilated_rnn.py:26).  xss as in stacked_lstm."""
    L = len(Wss)
    if dilations is None:
        dilations = [2 ** k for k in range(L)]
    return _run_stack(xss, Wss, Uss, bss, list(dilations), return_all_layers)


def lstm_cell(hs_prev: FractalTensor, cs_prev: FractalTensor, xs: FractalTensor, ws: FractalTensor,
              us: FractalTensor, bs: Optional[FractalTensor] = None):
    """One batched cell: the `batched_cell` of stacked_rnn.py:40-50 as one launch.
    hs_prev, cs_prev, xs: depth-1 [B] of [1, H]; ws, us: depth-1 [4] of [H, H]; bs: [4] of [1, H]."""
    core = _core()
    x = _dense_gpu(xs, 'xs', 1)
    B, H = x.shape[0], x.shape[-1]
    hp = _dense_gpu(hs_prev, 'hs_prev', 1).reshape(-1, H)[:B].contiguous()
    cp = _dense_gpu(cs_prev, 'cs_prev', 1).reshape(-1, H)[:B].contiguous()
    W = _dense_gpu(ws, 'ws', 1)
    U = _dense_gpu(us, 'us', 1)
    WU = torch.cat([W.permute(1, 0, 2).reshape(W.shape[1], 4 * H), U.permute(1, 0, 2).reshape(H, 4 * H)], dim=0).contiguous()
    bias = None if bs is None else _dense_gpu(bs, 'bs', 1).reshape(4 * H).contiguous()
    h, c = core.lstm_cell(x.reshape(B, -1).contiguous(), hp, cp, WU, bias)
    return FractalTensor.from_dense(h.view(B, 1, H), 1), FractalTensor.from_dense(c.view(B, 1, H), 1)


def flash_attention(qsss: FractalTensor, ksss: FractalTensor, vsss: FractalTensor, scale: Optional[float] = None):
    """Blockwise attention.  qsss, ksss, vsss: depth-3 [batch][head][block] of
    [block_rows, head_dim], the layout flash_attention_utils.create_input builds.
    The result has the structure of qsss.  fp32 inputs are converted to fp16 for
    the kernel (which accumulates in fp32) and the result converted back; `scale`
    multiplies the scores and defaults to 1.0, the reference program's maths
    (attn_func forms query @ key.T unscaled); pass head_dim ** -0.5 for the usual one."""
    core = _core()
    q = _dense_gpu(qsss, 'qsss', 3)   # [B, Hd, nb, rows, D]
    k = _dense_gpu(ksss, 'ksss', 3)
    v = _dense_gpu(vsss, 'vsss', 3)
    B, Hd, nbq, rq, D = q.shape
    to4 = lambda t: t.reshape(t.shape[0], t.shape[1], t.shape[2] * t.shape[3], t.shape[4])
    in_dtype = q.dtype
    O = core.flash_attention(to4(q).half().contiguous(), to4(k).half().contiguous(), to4(v).half().contiguous(),
                             1.0 if scale is None else float(scale))
    return FractalTensor.from_dense(O.to(in_dtype).view(B, Hd, nbq, rq, D), 3)


def b2b_gemm(a, b, c):
    """(a @ b) @ c in one kernel.  a [M,K], b [K,N], c [N,P] Tensors, or
    depth-1 FractalTensors of them (independent problems).  fp16 on the GPU."""
    core = _core()

    def dense(x, name):
        if isinstance(x, FractalTensor):
            return _dense_gpu(x, name, 1)
        if isinstance(x, Tensor):
            if not x.data.is_cuda:
                raise RuntimeError(f'{name} lives on {x.data.device}; the fused kernels run on the GPU only.')
            return x.data.unsqueeze(0)
        raise TypeError(f'{name} should be a Tensor or a FractalTensor.')

    A, Bm, Cm = dense(a, 'a'), dense(b, 'b'), dense(c, 'c')
    in_dtype = A.dtype
    K_, N_, P_ = A.shape[2], Bm.shape[2], Cm.shape[2]
    if core.b2b_gemm_rowmajor_supported(N_, K_, P_):
        # b and c as they are: the kernel transposes them between LDS and the matrix unit
        D = core.b2b_gemm_rowmajor(A.half().contiguous(), Bm.half().contiguous(), Cm.half().contiguous()).to(in_dtype)
    else:
        # the general kernel takes B and C with the contraction index contiguous
        D = core.b2b_gemm(A.half().contiguous(), Bm.half().transpose(1, 2).contiguous(),
                          Cm.half().transpose(1, 2).contiguous()).to(in_dtype)
    if isinstance(a, Tensor):
        return Tensor.from_tensor(D[0])
    return FractalTensor.from_dense(D, 1)


def mm(a: Tensor, b: Tensor) -> Tensor:
    """a @ b for fp16 Tensors on the GPU through the library's own MFMA product (ftk_gemm_f16): a [M,K], b [K,N],
    N a multiple of 128, K of 32, whatever the size.  `ops.mm` routes a product here by itself when it is large enough
    for this kernel to be the faster one (N a multiple of 256 and a 256 x 256 tile per compute unit) and leaves the
    rest with torch; this calls it on any shape the kernel takes."""
    for x, name in ((a, 'a'), (b, 'b')):
        if not isinstance(x, Tensor):
            raise TypeError(f'{name} should be a Tensor.')
        if not x.data.is_cuda:
            raise RuntimeError(f'{name} lives on {x.data.device}; the fused kernels run on the GPU only.')
    in_dtype = a.data.dtype
    return Tensor.from_tensor(_core().gemm(a.data.half().contiguous(), b.data.half().contiguous()).to(in_dtype))


def online_softmax(x: Tensor) -> Tensor:
    """Row softmax of a [rows, cols] fp32 Tensor through the online (max, sum) kernel."""
    return Tensor.from_tensor(_core().online_softmax(x.data.contiguous()))


def embedding_lookup(embedding: Tensor, words: FractalTensor) -> FractalTensor:
    """Rows of `embedding` [V, E] for every word id of `words`: what
    ops.map(lambda ws: ops.map(lambda word: ops.index(ops.slices(embedding, dim=0), word), ws), words)
    builds (examples/stacked_rnn/rnn_utils.py:81-90), as one gather.  `words` is a FractalTensor of any depth
    (regular or ragged) of single integers; the result has its structure with [1, E] elements.  An id outside
    [0, V) raises IndexError, as indexing the sliced matrix does."""
    if not isinstance(words, FractalTensor):
        raise TypeError('words should be a FractalTensor.')
    if not isinstance(embedding, Tensor):
        raise TypeError('embedding should be a Tensor.')
    table = embedding.data
    if table.dim() != 2:
        raise ValueError('embedding should be a [V, E] matrix.')
    if words.element_size != 1:
        raise ValueError('words should hold single integers.')
    ids = words._T
    if ids is None or words.indices is None:
        raise RuntimeError('FractalTensor is not initialized.')
    if not table.is_cuda or not ids.is_cuda:
        raise RuntimeError('embedding_lookup runs on the GPU only; move the embedding and the words there.')
    V, E = table.shape
    out = _core().embedding_gather(table.contiguous().float(), ids.reshape(-1).contiguous())
    typ = TensorStorage((1, E), torch_type_to_internal_type(out.dtype), device=out.device.type)
    for _ in range(words.depth - 1):
        typ = FractalTensorStorage(typ)
    ft = FractalTensor(typ)
    ft.indices = words.indices
    ft._T = out.reshape(-1)
    return ft


def grid_rnn(srcs: FractalTensor, trgs: FractalTensor, params):
    """The stacked grid RNN of examples/grid_rnn/grid_rnn.py:40-137 for a batch of samples in one call per plane
    of the (block, target, source) grid.

    srcs: depth-2 [N][S] of [1, H], trgs: depth-2 [N][Tg] of [1, H] (the two sides of the reference's outer map
    over samples, :127-137; equal lengths within the batch); params: per block ((i2h [2H, H], h2h [H, H],
    bias [1, H]) for the x direction, the same for y), Tensors on the GPU.  Returns (h_x, h_y), each depth-3
    [N][Tg][S] of [1, H]: the last block's outputs at every grid position, as the eager program returns them."""
    core = _core()
    xs = _dense_gpu(srcs, 'srcs', 2)   # [N, S, 1, H]
    ys = _dense_gpu(trgs, 'trgs', 2)   # [N, Tg, 1, H]
    N, S, one, H = xs.shape
    if one != 1 or ys.shape[0] != N or tuple(ys.shape[2:]) != (1, H):
        raise ValueError('srcs and trgs should be [N][S] and [N][Tg] of [1, H].')
    Tg = ys.shape[1]

    def stack(direction: int, which: int, shape):
        ts = []
        for block in params:
            t = block[direction][which]
            t = t.data if isinstance(t, Tensor) else t
            if tuple(t.shape) != shape:
                raise ValueError(f'grid parameter of shape {tuple(t.shape)}, expected {shape}.')
            if not t.is_cuda:
                raise RuntimeError('grid_rnn runs on the GPU only; move the parameters there.')
            ts.append(t.float())
        return torch.stack(ts).contiguous()

    Ux, Wx, bx = stack(0, 0, (2 * H, H)), stack(0, 1, (H, H)), stack(0, 2, (1, H))
    Uy, Wy, by = stack(1, 0, (2 * H, H)), stack(1, 1, (H, H)), stack(1, 2, (1, H))
    xs_t = xs.reshape(N, S, H).transpose(0, 1).contiguous().float()    # [S, N, H]: the source runs along the inner axis
    ys_t = ys.reshape(N, Tg, H).transpose(0, 1).contiguous().float()   # [Tg, N, H]
    hsss = core.grid_rnn(xs_t, ys_t, Wx, Ux, bx, Wy, Uy, by, crossed=True)   # [D, Tg, S, 2, N, H]
    last = hsss[-1].permute(2, 3, 0, 1, 4).contiguous()                      # [2, N, Tg, S, H]
    return (FractalTensor.from_dense(last[0].reshape(N, Tg, S, 1, H), 3),
            FractalTensor.from_dense(last[1].reshape(N, Tg, S, 1, H), 3))


def windowed_attention(query: FractalTensor, key: FractalTensor, value: FractalTensor, window_size: int,
                       dilation: int = 1, random_attn_pos: Optional[FractalTensor] = None) -> FractalTensor:
    """ops.shifted_slide(ops.zip(key, value), window_size, dilation) followed by the map of sparse_attn over the
    tokens (examples/sparse_attention/sparse_attention.py:25-38, 51-53, 69-71), as one kernel.

    query, key, value: regular FractalTensors of one structure, depth >= 1, of [1, D] tokens; the innermost level is
    the sequence, the outer ones (heads, batch) are independent.  random_attn_pos: the same structure of [1, R]
    integer tokens, or None.  The result has the structure of `query`."""
    if not all(isinstance(t, FractalTensor) for t in (query, key, value)):
        raise TypeError('query, key and value should be FractalTensors.')
    depth = query.depth
    q = _dense_gpu(query, 'query', depth)
    k = _dense_gpu(key, 'key', depth)
    v = _dense_gpu(value, 'value', depth)
    if q.shape != k.shape or q.shape != v.shape or q.shape[-2] != 1:
        raise ValueError('query, key and value should have one structure of [1, D] tokens.')
    S, D = q.shape[-3], q.shape[-1]
    extra = None
    if random_attn_pos is not None:
        r = _dense_gpu(random_attn_pos, 'random_attn_pos', depth)
        if r.shape[:-1] != q.shape[:-1] or r.is_floating_point():
            raise ValueError('random_attn_pos should have the structure of query and hold [1, R] integers.')
        extra = r.reshape(-1, S, r.shape[-1]).to(torch.int32).contiguous()
    out = _core().windowed_attention(q.reshape(-1, S, D).float().contiguous(), k.reshape(-1, S, D).float().contiguous(),
                                     v.reshape(-1, S, D).float().contiguous(), window_size, dilation, extra, 1.0)
    return FractalTensor.from_dense(out.reshape(q.shape), depth)


def _new_tokens(tss: FractalTensor, name: str, pages: torch.Tensor, dtype: Optional[torch.dtype]):
    """[sequence][token] of [heads, D], ragged or not -> (the packed rows [tokens, heads, D] in the type that goes with the pages (for codes of 8 bits: dtype, or
    fp16), tokens of each sequence)."""
    if not isinstance(tss, FractalTensor):
        raise TypeError(f'{name} should be a FractalTensor.')
    if tss.depth != 2 or len(tss.element_shape) != 2:
        raise ValueError(f'{name} should have depth 2 and [heads, D] items, got depth {tss.depth} of {list(tss.element_shape)}.')
    if tss._T is None or not tss.has_indices:
        raise RuntimeError('FractalTensor is not initialized.')
    rows = tss.data.reshape(-1, *tss.element_shape)
    if not rows.is_cuda:
        raise RuntimeError(f'{name} lives on {rows.device}; the fused kernels run on the GPU only.')
    own = pages.dtype if pages.dtype in (torch.float16, torch.bfloat16) else None
    if dtype not in ((None, own) if own else (None, torch.float16, torch.bfloat16)):
        raise TypeError(f'dtype should be {"that of the pages" if own else "float16 or bfloat16"}, got {dtype}.')
    return rows.to(own or dtype or torch.float16), tss.width_by_depth(1)


def _starts(counts, device) -> torch.Tensor:
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return torch.tensor(starts, dtype=torch.int32, device=device)


def _by_sequence(rows: torch.Tensor, counts) -> FractalTensor:
    """Packed rows -> [sequence][token] of what a row is."""
    if counts and counts[0] > 0 and all(n == counts[0] for n in counts):
        return FractalTensor.from_dense(rows.reshape(len(counts), counts[0], *rows.shape[1:]), 2)
    ft = FractalTensor(FractalTensorStorage(TensorStorage(tuple(rows.shape[1:]), torch_type_to_internal_type(rows.dtype), device=rows.device.type)))
    indices, at = [], 0
    for n in counts:
        indices.append(list(range(at, at + n)))
        at += n
    ft.indices = indices
    ft._T = rows.reshape(-1)
    return ft


def kv_cache_write(keyss: FractalTensor, valuess: FractalTensor, k_pages, v_pages, table, lens, k_exps=None, v_exps=None,
                   dtype: Optional[torch.dtype] = None) -> None:
    """Writes the keys and values of new tokens, [sequence][token] of [kv heads, D] (any number of tokens in each sequence, none too), into their
    pages: the last positions of the lens[b] that sequence b has with them.  Pages [pages, kv heads, page size, D] are fp16, bf16, or 8-bit codes
    (float8_e4m3fn or int8) with an exponent for each row in k_exps, v_exps [pages, kv heads, page size] int8; table [B, columns] and lens [B] are int32.
    Tokens are rounded first: to the type of 16-bit pages, and for codes to `dtype`, fp16 (the default) or bf16, which keeps fewer bits and values beyond
    65504."""
    keys, counts = _new_tokens(keyss, 'keyss', k_pages, dtype)
    values, same = _new_tokens(valuess, 'valuess', k_pages, dtype)
    if counts != same:
        raise ValueError('keyss and valuess should have one structure.')
    _core().kv_cache_write(keys, values, k_pages, v_pages, table, lens, _starts(counts, keys.device), k_exps, v_exps)


def kv_cache_read(k_pages, v_pages, table, lens, counts: Sequence[int], dtype=torch.float32, k_exps=None, v_exps=None):
    """The last counts[b] positions of every sequence, as kv_cache_write would have been given them: (keyss, valuess), [sequence][token] of [kv
    heads, D] of fp32 (fp16 if asked for and the pages are not bf16)."""
    counts = [int(n) for n in counts]
    if any(n < 0 for n in counts):
        raise ValueError('counts should not be negative.')
    keys, values = _core().kv_cache_read(k_pages, v_pages, table, lens, _starts(counts, k_pages.device), sum(counts), dtype, k_exps, v_exps)
    return _by_sequence(keys, counts), _by_sequence(values, counts)


def paged_attention(qss: FractalTensor, k_pages, v_pages, table, lens, k_exps=None, v_exps=None, scale: Optional[float] = None, causal: bool = True,
                    window: int = 0, max_keys: int = 0, dtype: Optional[torch.dtype] = None, weights: Optional[torch.Tensor] = None,
                    decay: float = 1.0) -> FractalTensor:
    """Attention of new tokens, [sequence][token] of [heads, D], over a paged cache that holds their keys and values already (kv_cache_write): one
    token a sequence, drafted ones, chunks of prompts and whole prompts, in any mixture.  heads is a multiple of the cache's.  `scale` multiplies the
    scores and defaults to 1.0, as in flash_attention.  causal: a token sees the positions up to its own; window > 0: no more than that many of them.
    max_keys: the greatest of lens where the program knows it.  The result has the structure and the type of qss; a token that sees nothing gets zeros.
    dtype: what the computation runs in on codes of 8 bits, that which they were written in: fp16 (the default) or bf16.
    weights [pages, kv heads, page size] fp32: what each position gets of the new tokens' attention is added there, behind a product of what older ones had with decay
    (for kv_cache_select); new positions begin at zero."""
    q, counts = _new_tokens(qss, 'qss', k_pages, dtype)
    core, starts, scale, most = _core(), _starts(counts, q.device), 1.0 if scale is None else float(scale), max(counts, default=0)
    o = core.paged_attention(q, k_pages, v_pages, table, lens, starts, k_exps, v_exps, scale, causal, window, most, max_keys, return_lse=weights is not None)
    if weights is not None:
        o, lse = o
        core.kv_cache_weigh(q, lse, k_pages, weights, table, lens, starts, k_exps, scale, decay, causal, window, most, max_keys)
    return _by_sequence(o.to(qss.data.dtype), counts)


def _integers(ft: FractalTensor, name: str, counts, dtypes=(torch.int32, torch.int64)) -> torch.Tensor:
    """[sequence][token] of [1] integers, counts[b] tokens in sequence b -> packed [tokens]."""
    if not isinstance(ft, FractalTensor):
        raise TypeError(f'{name} should be a FractalTensor.')
    if ft.depth != 2 or ft.element_size != 1:
        raise ValueError(f'{name} should have depth 2 and hold single integers, got depth {ft.depth} of {list(ft.element_shape)}.')
    if ft._T is None or not ft.has_indices:
        raise RuntimeError('FractalTensor is not initialized.')
    if not ft.data.is_cuda:
        raise RuntimeError(f'{name} lives on {ft.data.device}; the fused kernels run on the GPU only.')
    if ft.data.dtype not in dtypes:
        raise TypeError(f'{name} should be int32 or int64, got {ft.data.dtype}.')
    if counts is not None and ft.width_by_depth(1) != counts:
        raise ValueError(f'{name} should have {counts} tokens a sequence, got {ft.width_by_depth(1)}.')
    return ft.data.reshape(-1)


def _parents(ft: FractalTensor, counts) -> torch.Tensor:
    """Parents of the packed tokens in int32.  A number that has no place there stays one that comes before no token: it counts as none, as in int64."""
    return _narrowed(_integers(ft, 'parentss', counts))


def _narrowed(x: torch.Tensor) -> torch.Tensor:
    return x if x.dtype == torch.int32 else x.clamp(-1, 2 ** 31 - 1).to(torch.int32)


def paged_tree_attention(qss: FractalTensor, parentss: FractalTensor, k_pages, v_pages, table, lens, k_exps=None, v_exps=None, scale: Optional[float] = None,
                         window: int = 0, max_keys: int = 0, dtype: Optional[torch.dtype] = None) -> FractalTensor:
    """paged_attention of new tokens that form a tree in each sequence, at most 256 of them: each sees what is in front of its sequence's new tokens, its ancestors and
    itself.  parentss: [sequence][token] of [1] int32 or int64, the number of a token's parent among its sequence's new tokens, one in front of it; negative: none.
    window > 0: the last that many on the way that ends with the token.  All else as in paged_attention."""
    q, counts = _new_tokens(qss, 'qss', k_pages, dtype)
    parents = _parents(parentss, counts)
    o = _core().paged_tree_attention(q, k_pages, v_pages, table, lens, _starts(counts, q.device), parents, k_exps, v_exps, 1.0 if scale is None else float(scale), window,
                                     max(counts, default=0), max_keys)
    return _by_sequence(o.to(qss.data.dtype), counts)


def verify_tree(targets: FractalTensor, tokens: FractalTensor, parentss: FractalTensor, uniforms: torch.Tensor):
    """The path through each sequence's tree of drafts that the target model's own draws follow: (nextss, path).

    tokens: [B][n] of [1] int32 or int64, in each sequence the last token that is known, which is the root, and behind it the drafts; parentss: as in
    paged_tree_attention; targets: [B][n] of [1, V], the target's probabilities of what follows each token.  uniforms [B, M]: uniform numbers of [0, 1), fp32, one
    for each draw.  nextss, [B][token] of [1]: what was drawn, the accepted drafts and one token more (nothing for a sequence without tokens).  path [B, M] int32: the
    places of the tokens that stay in the cache, behind them -1, for kv_cache_keep."""
    ids = _integers(tokens, 'tokens', None)
    counts = tokens.width_by_depth(1)
    parents = _parents(parentss, counts)
    if not isinstance(targets, FractalTensor):
        raise TypeError('targets should be a FractalTensor.')
    if targets.depth != 2 or len(targets.element_shape) != 2 or targets.element_shape[0] != 1:
        raise ValueError(f'targets should have depth 2 and [1, V] items, got depth {targets.depth} of {list(targets.element_shape)}.')
    if targets.width_by_depth(1) != counts:
        raise ValueError(f'targets should have {counts} tokens a sequence, got {targets.width_by_depth(1)}.')
    drawn, path, _ = _core().verify_tree(targets.data.reshape(-1, targets.element_shape[1]), ids, parents, _starts(counts, ids.device), uniforms)
    there = drawn >= 0
    return _by_sequence(drawn[there].reshape(-1, 1), there.sum(1).tolist()), path


def kv_cache_select(weights: torch.Tensor, table, lens, budget: int, sinks: int = 0, recent: int = 0, max_keys: int = 0) -> torch.Tensor:
    """The positions of every sequence and head that a cache of `budget` positions keeps, [B, kv heads, budget] int32, ascending, then -1 (for kv_cache_keep): the first
    `sinks`, the last `recent`, and of the others those of the largest weights (paged_attention), of equal ones the earlier.  max_keys: the greatest of lens where the
    program knows it."""
    return _core().kv_cache_select(weights, table, lens, budget, sinks, recent, max_keys)


def kv_cache_keep(k_pages, v_pages, table, lens, kept: torch.Tensor, counts: Optional[Sequence[int]] = None, k_exps=None, v_exps=None,
                  weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Moves the positions that stay together, in place, and returns the new lens [B] int32: kept [B, M], or [B, kv heads, M] with as many in each head of a sequence, int32,
    ascends and has -1 behind its end.  It counts from a sequence's begin (kv_cache_select), or with counts, the number of new tokens of each sequence, from the first of
    these (verify_tree).  weights: theirs move with them."""
    starts = None if counts is None else _starts([int(n) for n in counts], k_pages.device)
    return _core().kv_cache_keep(k_pages, v_pages, table, lens, kept, starts, k_exps, v_exps, weights)


def _padded(ft: FractalTensor, name: str, counts) -> torch.Tensor:
    """[sequence][token], counts[b] tokens in sequence b -> dense [B, max(counts), *item]; what lies behind a sequence's tokens is not defined."""
    if not isinstance(ft, FractalTensor):
        raise TypeError(f'{name} should be a FractalTensor.')
    if ft.depth != 2:
        raise ValueError(f'{name} should have depth 2, got {ft.depth}.')
    if ft._T is None or not ft.has_indices:
        raise RuntimeError('FractalTensor is not initialized.')
    if not ft.data.is_cuda:
        raise RuntimeError(f'{name} lives on {ft.data.device}; the fused kernels run on the GPU only.')
    if ft.width_by_depth(1) != counts:
        raise ValueError(f'{name} should have {counts} tokens a sequence, got {ft.width_by_depth(1)}.')
    rows, most = ft.data.reshape(-1, *ft.element_shape), max(counts, default=0)
    if all(n == most for n in counts):
        return rows.view(len(counts), most, *ft.element_shape)
    out = rows.new_empty((len(counts), most, *ft.element_shape))
    out[torch.tensor([[i < n for i in range(most)] for n in counts], device=rows.device)] = rows
    return out


def verify_drafts(targets: FractalTensor, drafts: FractalTensor, accept_uniforms: torch.Tensor, sample_uniforms: torch.Tensor,
                  draft_probabilities: Optional[FractalTensor] = None) -> FractalTensor:
    """Which drafted tokens a target model accepts, and the token that follows them: [sequence][token] of [1] integers, from one to K + 1 tokens a sequence.

    targets: [B][K + 1] of [1, V], the target's probabilities before each draft and behind the last; drafts: [B][K] of [1] int32 or int64; draft_probabilities:
    [B][K] of [1, V] that the drafts were drawn from, or None for drafts that were not drawn at random.  Sequences may have different numbers of drafts, K at
    most, or none (dense arrays of all are made then, a copy).  accept_uniforms [B, K] and sample_uniforms [B]: uniform numbers of [0, 1), fp32.
    The tokens left are distributed as the target's own."""
    if not isinstance(drafts, FractalTensor):
        raise TypeError('drafts should be a FractalTensor.')
    if drafts.depth != 2 or drafts.element_size != 1:
        raise ValueError(f'drafts should have depth 2 and hold single integers, got depth {drafts.depth} of {list(drafts.element_shape)}.')
    counts = drafts.width_by_depth(1)
    d = _padded(drafts, 'drafts', counts)
    p = _padded(targets, 'targets', [n + 1 for n in counts])
    q = None if draft_probabilities is None else _padded(draft_probabilities, 'draft_probabilities', counts)
    if p.dim() != 4 or p.shape[2] != 1 or (q is not None and (q.dim() != 4 or q.shape[2] != 1)):
        raise ValueError('targets and draft_probabilities should have [1, V] items.')
    lens = None if all(n == d.shape[1] for n in counts) else torch.tensor(counts, dtype=torch.int32, device=d.device)
    tokens, accepted = _core().verify_drafts(p.squeeze(2), None if q is None else q.squeeze(2), d.reshape(d.shape[0], d.shape[1]), accept_uniforms, sample_uniforms, lens)
    kept = torch.arange(tokens.shape[1], device=tokens.device) <= accepted[:, None]
    return _by_sequence(tokens[kept].reshape(-1, 1), [n + 1 for n in accepted.tolist()])
