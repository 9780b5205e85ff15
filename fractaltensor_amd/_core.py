"""ctypes binding of libftkernels.so, the C ABI declared in include/ftk.h.

This is the only place the package touches native code.  The library is
required: importing this module without a built libftkernels.so (and the
module beside it, _fast) raises, and no function here has a CPU or PyTorch
fallback.

The fused entry points first hand their arguments to _fast, which checks,
allocates and launches in one native call and returns None, with nothing done,
for whatever is not plainly right; the code below it then says what is wrong
(or handles the rarer options).
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional, Sequence, Tuple

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, 'libftkernels.so')

# every symbol include/ftk.h declares; checked at load time
EXPORTS = (
    'ftk_version', 'ftk_last_error', 'ftk_device_info_query',
    'ftk_lstm_cell_f32', 'ftk_lstm_cell_f16', 'ftk_lstm_layer_f32', 'ftk_lstm_layer_f16', 'ftk_lstm_elementwise_f32',
    'ftk_stacked_lstm_workspace_bytes', 'ftk_stacked_lstm_f32', 'ftk_dilated_lstm_f32',
    'ftk_stacked_lstm_wavefront_f32', 'ftk_stacked_lstm_ragged_f32', 'ftk_lstm_set_products', 'ftk_lstm_get_products',
    'ftk_stacked_lstm_opts_f32', 'ftk_stacked_lstm_status', 'ftk_stacked_lstm_small_states', 'ftk_stacked_lstm_result', 'ftk_stacked_lstm_noalloc_f32',
    'ftk_stacked_lstm_f16_workspace_bytes', 'ftk_stacked_lstm_f16',
    'ftk_b2b_gemm_f16', 'ftk_b2b_gemm_f16_supported', 'ftk_b2b_gemm_rowmajor_f16', 'ftk_gemm_f16', 'ftk_batched_gemm_f16', 'ftk_flash_attn_f16', 'ftk_flash_attn_f16_workspace_bytes', 'ftk_flash_attn_ws_f16', 'ftk_flash_attn_f32_workspace_bytes', 'ftk_flash_attn_f32', 'ftk_online_softmax_f32', 'ftk_embedding_gather_f32',
    'ftk_grid_rnn_workspace_bytes', 'ftk_grid_rnn_f32', 'ftk_windowed_attn_f32',
    'ftk_kv_cache_write', 'ftk_kv_cache_read', 'ftk_paged_attn_workspace_bytes', 'ftk_paged_attn', 'ftk_verify_drafts_workspace_bytes', 'ftk_verify_drafts',
    'ftk_paged_tree_attn_workspace_bytes', 'ftk_paged_tree_attn', 'ftk_verify_tree_workspace_bytes', 'ftk_verify_tree', 'ftk_kv_cache_weigh_workspace_bytes', 'ftk_kv_cache_weigh', 'ftk_kv_cache_select', 'ftk_kv_cache_keep',
)


class FtkError(RuntimeError):
    """A non-zero return from the C ABI; carries the code and ftk_last_error()."""

    def __init__(self, code: int, message: str):
        super().__init__(f'libftkernels error {code}: {message}')
        self.code = code


class LstmOptions(ctypes.Structure):
    """ftk_lstm_options of include/ftk.h."""
    _fields_ = [('products', ctypes.c_int), ('spin_limit', ctypes.c_int)]


class KvPages(ctypes.Structure):
    """ftk_kv_pages of include/ftk.h."""
    _fields_ = [('k', ctypes.c_void_p), ('v', ctypes.c_void_p), ('k_exps', ctypes.c_void_p), ('v_exps', ctypes.c_void_p), ('type', ctypes.c_int),
                ('pages', ctypes.c_int), ('heads', ctypes.c_int), ('page_size', ctypes.c_int), ('head_size', ctypes.c_int)]


class KvBatch(ctypes.Structure):
    """ftk_kv_batch of include/ftk.h."""
    _fields_ = [('table', ctypes.c_void_p), ('lens', ctypes.c_void_p), ('starts', ctypes.c_void_p), ('sequences', ctypes.c_int),
                ('table_width', ctypes.c_int), ('tokens', ctypes.c_int)]


class DeviceInfo(ctypes.Structure):
    _fields_ = [('compute_units', ctypes.c_int), ('lds_bytes_per_block', ctypes.c_int),
                ('clock_khz', ctypes.c_int), ('wavefront_size', ctypes.c_int),
                ('persistent_slots', ctypes.c_int), ('arch', ctypes.c_char * 32)]


def _load() -> ctypes.CDLL:
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f'{LIB_PATH} is missing: build it with `make -C fractaltensor_amd/csrc` '
            '(or __graft_entry__.build()); there is no fallback path')
    lib = ctypes.CDLL(LIB_PATH)
    for name in EXPORTS:
        if not hasattr(lib, name):
            raise ImportError(f'{LIB_PATH} does not export {name}')
    lib.ftk_version.restype = ctypes.c_int
    lib.ftk_last_error.restype = ctypes.c_char_p
    lib.ftk_stacked_lstm_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_stacked_lstm_workspace_bytes.argtypes = [ctypes.c_int] * 4
    lib.ftk_stacked_lstm_f16_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_stacked_lstm_f16_workspace_bytes.argtypes = [ctypes.c_int] * 4
    lib.ftk_grid_rnn_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_grid_rnn_workspace_bytes.argtypes = [ctypes.c_int] * 2
    lib.ftk_flash_attn_f32_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_flash_attn_f32_workspace_bytes.argtypes = [ctypes.c_int] * 5
    lib.ftk_flash_attn_f16_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_flash_attn_f16_workspace_bytes.argtypes = [ctypes.c_int] * 5
    lib.ftk_paged_attn_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_paged_attn_workspace_bytes.argtypes = [ctypes.POINTER(KvPages), ctypes.POINTER(KvBatch)] + [ctypes.c_int] * 4
    lib.ftk_paged_tree_attn_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_paged_tree_attn_workspace_bytes.argtypes = lib.ftk_paged_attn_workspace_bytes.argtypes
    lib.ftk_verify_tree_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_verify_tree_workspace_bytes.argtypes = [ctypes.c_int]
    lib.ftk_kv_cache_weigh_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_kv_cache_weigh_workspace_bytes.argtypes = [ctypes.POINTER(KvPages), ctypes.POINTER(KvBatch)] + [ctypes.c_int] * 3
    lib.ftk_verify_drafts_workspace_bytes.restype = ctypes.c_size_t
    lib.ftk_verify_drafts_workspace_bytes.argtypes = [ctypes.c_int] * 2
    for name in EXPORTS:
        if name not in ('ftk_last_error', 'ftk_stacked_lstm_workspace_bytes', 'ftk_stacked_lstm_f16_workspace_bytes', 'ftk_grid_rnn_workspace_bytes',
                        'ftk_flash_attn_f32_workspace_bytes', 'ftk_flash_attn_f16_workspace_bytes', 'ftk_paged_attn_workspace_bytes',
                        'ftk_verify_drafts_workspace_bytes', 'ftk_paged_tree_attn_workspace_bytes',
                        'ftk_kv_cache_weigh_workspace_bytes', 'ftk_verify_tree_workspace_bytes'):
            getattr(lib, name).restype = ctypes.c_int
    return lib


lib = _load()


def _check(rc: int) -> None:
    if rc != 0:
        raise FtkError(rc, lib.ftk_last_error().decode('utf-8', 'replace'))


def _ptr(t: Optional[torch.Tensor]):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _req(t: torch.Tensor, dtype, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{name} must be a torch.Tensor')
    if not t.is_cuda:
        raise RuntimeError(f'{name} must live on the GPU (got {t.device}); there is no CPU path')
    if t.dtype != dtype:
        raise TypeError(f'{name} must be {dtype}, got {t.dtype}')
    if not t.is_contiguous():
        raise ValueError(f'{name} must be contiguous')
    return t


def _req_out(t: torch.Tensor, dtype, shape, name: str) -> torch.Tensor:
    """A caller-supplied output: the kernels write the full shape, so anything smaller would be overrun."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{name} must be a torch.Tensor')
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name} must be {tuple(shape)}, got {tuple(t.shape)}')
    return _req(t, dtype, name)


def _req_workspace(t: torch.Tensor) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or not t.is_contiguous():
        raise ValueError('workspace must be a contiguous CUDA tensor')
    return t


# calls of the fused entry points made through this binding, by name (what routed an operator program here)
launch_counts: dict = {}


def _count(name: str) -> None:
    launch_counts[name] = launch_counts.get(name, 0) + 1


try:
    from . import _fast, _serving
except ImportError as e:
    raise ImportError(f'{_HERE}/_fast.so or _serving.so cannot be loaded ({e}): build them with `make -C fractaltensor_amd/csrc` '
                      '(or __graft_entry__.build()); there is no fallback path') from e
_fast.init(launch_counts, _check)
_serving.init(launch_counts, _check)


def version() -> int:
    return lib.ftk_version()


def device_info() -> DeviceInfo:
    info = DeviceInfo()
    _check(lib.ftk_device_info_query(ctypes.byref(info)))
    return info


def lstm_cell(x, h_prev, c_prev, WU, bias=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Fused cell: x [B,I], h_prev/c_prev [B,H] or None, WU [(I+H),4H], bias [4H] or None."""
    f32 = torch.float32
    _req(x, f32, 'x'); _req(WU, f32, 'WU')
    B, I = x.shape
    H = WU.shape[1] // 4
    if WU.shape != (I + H, 4 * H):
        raise ValueError(f'WU must be [(I+H), 4H] = [{I + H}, {4 * H}], got {tuple(WU.shape)}')
    for t, n in ((h_prev, 'h_prev'), (c_prev, 'c_prev')):
        if t is not None and _req(t, f32, n).shape != (B, H):
            raise ValueError(f'{n} must be [{B}, {H}]')
    if bias is not None and _req(bias, f32, 'bias').numel() != 4 * H:
        raise ValueError('bias must have 4H elements')
    h = torch.empty((B, H), dtype=f32, device=x.device)
    c = torch.empty((B, H), dtype=f32, device=x.device)
    _check(lib.ftk_lstm_cell_f32(_ptr(x), _ptr(h_prev), _ptr(c_prev), _ptr(WU), _ptr(bias), _ptr(h), _ptr(c),
                                 ctypes.c_int(B), ctypes.c_int(I), ctypes.c_int(H), _stream()))
    return h, c


def lstm_layer(xs, WU, bias=None, h0=None, c0=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One layer over T steps from an initial state: xs [T,B,I], WU [(I+H),4H], bias [4H] or None, h0/c0 [B,H] or
    None (zero state) -> hs, cs [T,B,H].  fp32 throughout, or fp16 storage (bias fp32) when xs is fp16."""
    dt = xs.dtype
    if dt not in (torch.float32, torch.float16):
        raise TypeError('xs must be float32 or float16')
    _req(xs, dt, 'xs'); _req(WU, dt, 'WU')
    T, B, I = xs.shape
    H = WU.shape[1] // 4
    if WU.shape != (I + H, 4 * H):
        raise ValueError(f'WU must be [(I+H), 4H] = [{I + H}, {4 * H}], got {tuple(WU.shape)}')
    for t, n in ((h0, 'h0'), (c0, 'c0')):
        if t is not None and _req(t, dt, n).shape != (B, H):
            raise ValueError(f'{n} must be [{B}, {H}]')
    if bias is not None and _req(bias, torch.float32, 'bias').numel() != 4 * H:
        raise ValueError('bias must have 4H elements')
    hs = torch.empty((T, B, H), dtype=dt, device=xs.device)
    cs = torch.empty((T, B, H), dtype=dt, device=xs.device)
    fn = lib.ftk_lstm_layer_f32 if dt == torch.float32 else lib.ftk_lstm_layer_f16
    ci = ctypes.c_int
    _check(fn(_ptr(xs), _ptr(WU), _ptr(bias), _ptr(h0), _ptr(c0), _ptr(hs), _ptr(cs), ci(T), ci(B), ci(I), ci(H), _stream()))
    return hs, cs


def lstm_cell_f16(x, h_prev, c_prev, WU, bias=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The fused cell with fp16 storage: x [B,I], h_prev/c_prev [B,H] or None, WU [(I+H),4H] fp16, bias [4H]
    fp32 or None; I and H multiples of 32.  Gate sums in fp32, h and c rounded to fp16 when written."""
    f16 = torch.float16
    _req(x, f16, 'x'); _req(WU, f16, 'WU')
    B, I = x.shape
    H = WU.shape[1] // 4
    if WU.shape != (I + H, 4 * H):
        raise ValueError(f'WU must be [(I+H), 4H] = [{I + H}, {4 * H}], got {tuple(WU.shape)}')
    for t, n in ((h_prev, 'h_prev'), (c_prev, 'c_prev')):
        if t is not None and _req(t, f16, n).shape != (B, H):
            raise ValueError(f'{n} must be [{B}, {H}]')
    if bias is not None and _req(bias, torch.float32, 'bias').numel() != 4 * H:
        raise ValueError('bias must have 4H elements')
    h = torch.empty((B, H), dtype=f16, device=x.device)
    c = torch.empty((B, H), dtype=f16, device=x.device)
    _check(lib.ftk_lstm_cell_f16(_ptr(x), _ptr(h_prev), _ptr(c_prev), _ptr(WU), _ptr(bias), _ptr(h), _ptr(c),
                                 ctypes.c_int(B), ctypes.c_int(I), ctypes.c_int(H), _stream()))
    return h, c


def lstm_elementwise(gates, bias, c_prev, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """State update on pre-activation gates [B,4H] (the unfused baseline's second kernel)."""
    f32 = torch.float32
    _req(gates, f32, 'gates')
    B, H4 = gates.shape
    H = H4 // 4
    if gates.dim() != 2 or H4 % 4:
        raise ValueError(f'gates must be [B, 4H], got {tuple(gates.shape)}')
    if bias is not None and _req(bias, f32, 'bias').numel() != 4 * H:
        raise ValueError('bias must have 4H elements')
    if c_prev is not None and tuple(_req(c_prev, f32, 'c_prev').shape) != (B, H):
        raise ValueError(f'c_prev must be [{B}, {H}], got {tuple(c_prev.shape)}')
    if out is None:
        h = torch.empty((B, H), dtype=f32, device=gates.device)
        c = torch.empty((B, H), dtype=f32, device=gates.device)
    else:
        h, c = out
        _req_out(h, f32, (B, H), 'h'); _req_out(c, f32, (B, H), 'c')
    _check(lib.ftk_lstm_elementwise_f32(_ptr(gates), _ptr(bias), _ptr(c_prev), _ptr(h), _ptr(c),
                                        ctypes.c_int(B), ctypes.c_int(H), _stream()))
    return h, c


def stacked_lstm_workspace_bytes(L: int, T: int, B: int, H: int) -> int:
    return int(lib.ftk_stacked_lstm_workspace_bytes(L, T, B, H))


def stacked_lstm(xs, WU, bias=None, dilations: Optional[Sequence[int]] = None, schedule: str = 'auto',
                 out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                 workspace: Optional[torch.Tensor] = None,
                 active_rows: Optional[Sequence[int]] = None, products: Optional[str] = None,
                 spin_limit: int = 0, check: Optional[bool] = None, exact_small_states: bool = False
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """xs [T,B,H], WU [L,2H,4H], bias [L,4H] or None -> hsss, csss [L,T,B,H].

    schedule: 'auto' (persistent kernel when the shape allows, else per-stage
    launches) or 'wavefront' (always per-stage launches).
    active_rows: for a ragged time-major batch (rows sorted by decreasing length), the number of rows still
    running at each step; only the live (t, row) places of the outputs are defined then.
    products: 'f32' / 'f16x3' for this call, None for the process-wide mode (set_lstm_products).
    spin_limit: polls a bounded wait of the persistent kernel makes before giving up (0 = the default).
    check: wait for the stream and raise FtkError (code -6) if the persistent launch gave up a wait and left
    the outputs incomplete.  Default: True when the workspace is allocated here (nobody else could look at its
    status word afterwards), False when the caller passes one (check it with stacked_lstm_check(workspace)).
    exact_small_states: after a call on split products, wait for the stream and, if hidden states too small for
    the fixed scale of their fp16 planes were written (stacked_lstm_small_states), compute the stack again on fp32
    products, so that layers that fade towards zero are accurate relative to their own size as well.
    """
    if schedule == 'auto' and active_rows is None and not spin_limit and (products is None or products in LSTM_PRODUCTS):
        small = exact_small_states and products != 'f32'
        done = _fast.stacked_lstm(False, xs, WU, bias, dilations, out, workspace, -1 if products is None else LSTM_PRODUCTS[products],
                                  check, small)
        if done is not None:
            if not (small and done[2]):
                return done[0], done[1]
            _count('stacked_lstm_repeated_on_f32_products')
            return stacked_lstm(xs, WU, bias, dilations=dilations, out=(done[0], done[1]), workspace=workspace, products='f32',
                                check=workspace is None if check is None else check)
    f32 = torch.float32
    _req(xs, f32, 'xs'); _req(WU, f32, 'WU')
    T, B, H = xs.shape
    L = WU.shape[0]
    if WU.shape != (L, 2 * H, 4 * H):
        raise ValueError(f'WU must be [L, 2H, 4H] = [{L}, {2 * H}, {4 * H}], got {tuple(WU.shape)}')
    if bias is not None and _req(bias, f32, 'bias').shape != (L, 4 * H):
        raise ValueError('bias must be [L, 4H]')
    if out is None:
        hsss = torch.empty((L, T, B, H), dtype=f32, device=xs.device)
        csss = torch.empty((L, T, B, H), dtype=f32, device=xs.device)
    else:
        hsss, csss = out
        _req_out(hsss, f32, (L, T, B, H), 'hsss'); _req_out(csss, f32, (L, T, B, H), 'csss')
    if products is not None and products not in LSTM_PRODUCTS:
        raise ValueError(f"products must be one of {sorted(LSTM_PRODUCTS)} or None, got {products!r}")
    _count('stacked_lstm')
    dil = None
    if dilations is not None:
        if len(dilations) != L:
            raise ValueError('dilations must have one entry per layer')
        dil = (ctypes.c_int * L)(*[int(d) for d in dilations])
    ci = ctypes.c_int
    if schedule == 'wavefront':
        _check(lib.ftk_stacked_lstm_wavefront_f32(_ptr(xs), _ptr(WU), _ptr(bias), dil, _ptr(hsss), _ptr(csss),
                                                  ci(L), ci(T), ci(B), ci(H), _stream()))
        return hsss, csss
    if schedule != 'auto':
        raise ValueError("schedule must be 'auto' or 'wavefront'")
    need = stacked_lstm_workspace_bytes(L, T, B, H)
    if check is None:
        check = workspace is None
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=xs.device)
    _req_workspace(workspace)
    ws_bytes = ctypes.c_size_t(workspace.numel() * workspace.element_size())
    act = None
    if active_rows is not None:
        if len(active_rows) != T:
            raise ValueError('active_rows must have one entry per step')
        act = (ctypes.c_int * T)(*[int(v) for v in active_rows])
    if products is not None or spin_limit:
        opts = LstmOptions(LSTM_PRODUCTS[products] if products is not None else -1, int(spin_limit))
        _check(lib.ftk_stacked_lstm_opts_f32(_ptr(xs), _ptr(WU), _ptr(bias), dil, act, _ptr(hsss), _ptr(csss), ci(L), ci(T),
                                             ci(B), ci(H), ctypes.byref(opts), _ptr(workspace), ws_bytes, _stream()))
    elif act is not None:
        _check(lib.ftk_stacked_lstm_ragged_f32(_ptr(xs), _ptr(WU), _ptr(bias), dil, act, _ptr(hsss), _ptr(csss),
                                               ci(L), ci(T), ci(B), ci(H), _ptr(workspace), ws_bytes, _stream()))
    elif dil is None:
        _check(lib.ftk_stacked_lstm_f32(_ptr(xs), _ptr(WU), _ptr(bias), _ptr(hsss), _ptr(csss),
                                        ci(L), ci(T), ci(B), ci(H), _ptr(workspace), ws_bytes, _stream()))
    else:
        _check(lib.ftk_dilated_lstm_f32(_ptr(xs), _ptr(WU), _ptr(bias), dil, _ptr(hsss), _ptr(csss),
                                        ci(L), ci(T), ci(B), ci(H), _ptr(workspace), ws_bytes, _stream()))
    if check:
        stacked_lstm_check(workspace)
    if exact_small_states and products != 'f32' and stacked_lstm_small_states(workspace):
        _count('stacked_lstm_repeated_on_f32_products')
        return stacked_lstm(xs, WU, bias, dilations=dilations, out=(hsss, csss), workspace=workspace, active_rows=active_rows,
                            products='f32', spin_limit=spin_limit, check=check)
    return hsss, csss


def stacked_lstm_launch(xs, WU, bias, dilations: Optional[Sequence[int]] = None, products: Optional[str] = None):
    """The launch of stacked_lstm(..., exact_small_states=True) without its wait, so that a caller can do something meanwhile:
    (hsss, csss, what stacked_lstm_finish takes), or None for operands that stacked_lstm has to look at more closely."""
    if products is not None and products not in LSTM_PRODUCTS or xs.dim() != 3 or WU.dim() != 3 or not xs.is_cuda:
        return None
    workspace = _fast.stacked_lstm_workspace(False, xs, WU)
    done = _fast.stacked_lstm(False, xs, WU, bias, dilations, None, workspace, -1 if products is None else LSTM_PRODUCTS[products],
                              False, False)
    return None if done is None else (done[0], done[1], (xs, WU, bias, dilations, products, workspace))


def stacked_lstm_finish(launched) -> bool:
    """Waits for a stacked_lstm_launch, raises FtkError if it gave up a wait, and repeats it on fp32 products, into the same
    outputs, if it met states too small for split ones; says whether it did."""
    hsss, csss, (xs, WU, bias, dilations, products, workspace) = launched
    small = _fast.stacked_lstm_result(workspace)
    if not small or products == 'f32':
        return False
    _count('stacked_lstm_repeated_on_f32_products')
    stacked_lstm(xs, WU, bias, dilations=dilations, out=(hsss, csss), workspace=workspace, products='f32', check=True)
    return True


def stacked_lstm_noalloc(xs, WU, bias, out: Tuple[torch.Tensor, torch.Tensor], dilations: Optional[Sequence[int]] = None) -> None:
    """ftk_stacked_lstm_noalloc_f32: the fp32-product persistent stack (H = 256) into caller-supplied hsss, csss
    [L,T,B,H], with the launch's flags in the library's built-in per-device scratch.  Nothing is allocated, here or in
    the library; the status word is read with stacked_lstm_check(None)."""
    f32 = torch.float32
    _req(xs, f32, 'xs'); _req(WU, f32, 'WU')
    T, B, H = xs.shape
    L = WU.shape[0]
    if WU.shape != (L, 2 * H, 4 * H):
        raise ValueError(f'WU must be [L, 2H, 4H] with H={H}, got {tuple(WU.shape)}')
    if bias is not None and _req(bias, f32, 'bias').numel() != L * 4 * H:
        raise ValueError('bias must be [L, 4H]')
    hsss, csss = out
    _req_out(hsss, f32, (L, T, B, H), 'hsss'); _req_out(csss, f32, (L, T, B, H), 'csss')
    dil = None
    if dilations is not None:
        if len(dilations) != L:
            raise ValueError('one dilation per layer')
        dil = (ctypes.c_int * L)(*[int(d) for d in dilations])
    ci = ctypes.c_int
    _check(lib.ftk_stacked_lstm_noalloc_f32(_ptr(xs), _ptr(WU), _ptr(bias), dil, _ptr(hsss), _ptr(csss), ci(L), ci(T), ci(B),
                                            ci(H), _stream()))


def stacked_lstm_check(workspace: Optional[torch.Tensor]) -> None:
    """Waits for the current stream and raises FtkError (code -6) if the last stacked-LSTM call given this
    workspace drained early because a bounded wait of the persistent kernel ran out.  None: the built-in scratch
    that stacked_lstm_noalloc uses on the current device."""
    if workspace is not None:
        _req_workspace(workspace)
    _check(lib.ftk_stacked_lstm_status(_ptr(workspace), _stream()))


def stacked_lstm_small_states(workspace: torch.Tensor) -> bool:
    """Waits for the current stream; True if the last fp32 stacked-LSTM call given this workspace ran on split
    products and wrote hidden states too small for the fixed scale of their fp16 planes (four neighbouring units of a
    row all below 2^-26 and not all zero): such values reach the cells that read them with fewer than 13 bits.
    The whole output is still accurate relative to its largest value; layers that faded that far are not accurate
    relative to themselves.  stacked_lstm(..., exact_small_states=True) repeats such a call on fp32 products."""
    _req_workspace(workspace)
    rc = lib.ftk_stacked_lstm_small_states(_ptr(workspace), _stream())
    if rc < 0:
        _check(rc)
    return rc == 1


def stacked_lstm_f16(xs, WU, bias=None, dilations: Optional[Sequence[int]] = None,
                     out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, workspace: Optional[torch.Tensor] = None,
                     active_rows: Optional[Sequence[int]] = None, check: Optional[bool] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp16 storage: xs [T,B,H], WU [L,2H,4H] fp16, bias [L,4H] fp32 or None -> hsss, csss [L,T,B,H] fp16.
    H a multiple of 32.  H = 256, 512 and 1024 run in one launch per group of layers whose weights the chip holds,
    where that is faster; every other shape streams its weights through the cell kernels, in one launch or one per stage
    of independent cells."""
    if active_rows is None:
        done = _fast.stacked_lstm(True, xs, WU, bias, dilations, out, workspace, -1, check, False)
        if done is not None:
            return done[0], done[1]
    f16 = torch.float16
    _req(xs, f16, 'xs'); _req(WU, f16, 'WU')
    T, B, H = xs.shape
    L = WU.shape[0]
    if WU.shape != (L, 2 * H, 4 * H):
        raise ValueError(f'WU must be [L, 2H, 4H] = [{L}, {2 * H}, {4 * H}], got {tuple(WU.shape)}')
    if bias is not None and _req(bias, torch.float32, 'bias').shape != (L, 4 * H):
        raise ValueError('bias must be [L, 4H]')
    if out is None:
        hsss = torch.empty((L, T, B, H), dtype=f16, device=xs.device)
        csss = torch.empty((L, T, B, H), dtype=f16, device=xs.device)
    else:
        hsss, csss = out
        _req_out(hsss, f16, (L, T, B, H), 'hsss'); _req_out(csss, f16, (L, T, B, H), 'csss')
    _count('stacked_lstm_f16')
    dil = None
    if dilations is not None:
        if len(dilations) != L:
            raise ValueError('dilations must have one entry per layer')
        dil = (ctypes.c_int * L)(*[int(d) for d in dilations])
    act = None
    if active_rows is not None:
        if len(active_rows) != T:
            raise ValueError('active_rows must have one entry per step')
        act = (ctypes.c_int * T)(*[int(v) for v in active_rows])
    if check is None:
        check = workspace is None
    if workspace is None:
        workspace = torch.empty(int(lib.ftk_stacked_lstm_f16_workspace_bytes(L, T, B, H)), dtype=torch.uint8, device=xs.device)
    _req_workspace(workspace)
    ci = ctypes.c_int
    _check(lib.ftk_stacked_lstm_f16(_ptr(xs), _ptr(WU), _ptr(bias), dil, act, _ptr(hsss), _ptr(csss), ci(L), ci(T), ci(B),
                                    ci(H), _ptr(workspace), ctypes.c_size_t(workspace.numel() * workspace.element_size()),
                                    _stream()))
    if check:
        stacked_lstm_check(workspace)
    return hsss, csss


LSTM_PRODUCTS = {'f32': 0, 'f16x3': 1}


def set_lstm_products(mode: str) -> None:
    """How the persistent stacked-LSTM kernel forms the gate GEMM's products.

    'f32': one fp32 MFMA per product.  'f16x3' (default): each fp32 operand as an fp16 value plus an fp16
    remainder under a shared power-of-two scale, three fp16 MFMAs per fp32 one, fp32 accumulation; only the
    remainder-times-remainder term (2^-22 of a product) is dropped.
    """
    if mode not in LSTM_PRODUCTS:
        raise ValueError(f"mode must be one of {sorted(LSTM_PRODUCTS)}, got {mode!r}")
    _check(lib.ftk_lstm_set_products(ctypes.c_int(LSTM_PRODUCTS[mode])))


def get_lstm_products() -> str:
    code = int(lib.ftk_lstm_get_products())
    return next(k for k, v in LSTM_PRODUCTS.items() if v == code)


def persistent_status(workspace: torch.Tensor) -> int:
    """Error word a persistent stacked-LSTM launch left in its workspace (synchronises).

    0 = every bounded wait completed; 1 = a wait ran out of polls and the launch drained early.
    """
    torch.cuda.synchronize()
    return int(workspace[:4].view(torch.int32).item())


def b2b_gemm(A, B_nk, C_pn, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """D = (A @ B) @ C.  A [G,M,K]; B_nk [G,N,K] (B stored column-major); C_pn [G,P,N]; D [G,M,P]; fp16."""
    D = _fast.b2b_gemm(A, B_nk, C_pn, out)
    if D is not None:
        return D
    f16 = torch.float16
    _req(A, f16, 'A'); _req(B_nk, f16, 'B_nk'); _req(C_pn, f16, 'C_pn')
    squeeze = A.dim() == 2
    if squeeze:
        A, B_nk, C_pn = A[None], B_nk[None], C_pn[None]
    G, M, K = A.shape
    N = B_nk.shape[1]
    P = C_pn.shape[1]
    if B_nk.shape != (G, N, K) or C_pn.shape != (G, P, N):
        raise ValueError(f'shape mismatch: A {tuple(A.shape)}, B_nk {tuple(B_nk.shape)}, C_pn {tuple(C_pn.shape)}')
    D = out if out is not None else torch.empty((G, M, P), dtype=f16, device=A.device)
    _req_out(D, f16, (G, M, P), 'D')
    _count('b2b_gemm')
    ci = ctypes.c_int
    _check(lib.ftk_b2b_gemm_f16(_ptr(A), _ptr(B_nk), _ptr(C_pn), _ptr(D), ci(G), ci(M), ci(N), ci(K), ci(P), _stream()))
    return D[0] if squeeze and out is None else D


def b2b_gemm_supported(N: int, K: int, P: int) -> bool:
    """Shapes ftk_b2b_gemm_f16 takes on the current device (the fused kernels' LDS fit, or N <= 2048 for the general one)."""
    return bool(lib.ftk_b2b_gemm_f16_supported(ctypes.c_int(N), ctypes.c_int(K), ctypes.c_int(P)))


def b2b_gemm_rowmajor_supported(N: int, K: int, P: int) -> bool:
    """Shapes ftk_b2b_gemm_rowmajor_f16 is built for."""
    return K in (64, 128) and N in (64, 128) and P % 128 == 0


def b2b_gemm_rowmajor(A, B, C, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """D = (A @ B) @ C with every operand row-major: A [G,M,K], B [G,K,N], C [G,N,P], D [G,M,P]; fp16.
    K and N in {64, 128}, P a multiple of 128."""
    f16 = torch.float16
    _req(A, f16, 'A'); _req(B, f16, 'B'); _req(C, f16, 'C')
    squeeze = A.dim() == 2
    if squeeze:
        A, B, C = A[None], B[None], C[None]
    G, M, K = A.shape
    N = B.shape[2]
    P = C.shape[2]
    if B.shape != (G, K, N) or C.shape != (G, N, P):
        raise ValueError(f'shape mismatch: A {tuple(A.shape)}, B {tuple(B.shape)}, C {tuple(C.shape)}')
    D = out if out is not None else torch.empty((G, M, P), dtype=f16, device=A.device)
    _req_out(D, f16, (G, M, P), 'D')
    _count('b2b_gemm_rowmajor')
    ci = ctypes.c_int
    _check(lib.ftk_b2b_gemm_rowmajor_f16(_ptr(A), _ptr(B), _ptr(C), _ptr(D), ci(G), ci(M), ci(N), ci(K), ci(P), _stream()))
    return D[0] if squeeze and out is None else D


def gemm(A, B, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """C = A @ B, fp16 storage, fp32 accumulation, row-major: A [M,K] or [G,M,K], B [K,N] or [G,K,N].
    N a multiple of 128, K of 32."""
    f16 = torch.float16
    _req(A, f16, 'A'); _req(B, f16, 'B')
    if A.dim() != B.dim() or A.dim() not in (2, 3):
        raise ValueError('A and B must both be matrices or both be batches of matrices')
    batched = A.dim() == 3
    G = A.shape[0] if batched else 1
    M, K = A.shape[-2:]
    N = B.shape[-1]
    if B.shape[-2] != K or (batched and B.shape[0] != G):
        raise ValueError(f'shape mismatch: A {tuple(A.shape)}, B {tuple(B.shape)}')
    C = out if out is not None else torch.empty((*A.shape[:-1], N), dtype=f16, device=A.device)
    _req_out(C, f16, (*A.shape[:-1], N), 'C')
    ci = ctypes.c_int
    _count('gemm')
    if batched:
        _check(lib.ftk_batched_gemm_f16(_ptr(A), _ptr(B), _ptr(C), ci(G), ci(M), ci(N), ci(K), _stream()))
    else:
        _check(lib.ftk_gemm_f16(_ptr(A), _ptr(B), _ptr(C), ci(M), ci(N), ci(K), _stream()))
    return C


def flash_attention(Q, K, V, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None, split_keys: bool = True) -> torch.Tensor:
    """O = softmax(Q K^T scale) V.  Q [B,Hd,Sq,D], K/V [B,Hd,Skv,D], fp16, non-causal.
    A grid that does not fill the chip (few queries, heads and samples) with many keys is split over the keys and
    merged (ftk_flash_attn_ws_f16); the workspace for that is allocated here unless one is given, split_keys=False
    keeps the single launch."""
    O = _fast.flash_attention(True, Q, K, V, scale, out, workspace, split_keys)
    if O is not None:
        return O
    f16 = torch.float16
    _req(Q, f16, 'Q'); _req(K, f16, 'K'); _req(V, f16, 'V')
    B, Hd, Sq, D = Q.shape
    Skv = K.shape[2]
    if K.shape != (B, Hd, Skv, D) or V.shape != (B, Hd, Skv, D):
        raise ValueError(f'shape mismatch: Q {tuple(Q.shape)}, K {tuple(K.shape)}, V {tuple(V.shape)}')
    if scale is None:
        scale = D ** -0.5
    O = out if out is not None else torch.empty_like(Q)
    _req_out(O, f16, Q.shape, 'O')
    _count('flash_attention')
    ci = ctypes.c_int
    need = int(lib.ftk_flash_attn_f16_workspace_bytes(B, Hd, Sq, Skv, D)) if split_keys else 0
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=Q.device)
        _req_workspace(workspace)
        _count('flash_attention_split_keys')
        _check(lib.ftk_flash_attn_ws_f16(_ptr(Q), _ptr(K), _ptr(V), _ptr(O), ci(B), ci(Hd), ci(Sq), ci(Skv), ci(D), ctypes.c_float(scale),
                                         _ptr(workspace), ctypes.c_size_t(workspace.numel() * workspace.element_size()), _stream()))
        return O
    _check(lib.ftk_flash_attn_f16(_ptr(Q), _ptr(K), _ptr(V), _ptr(O), ci(B), ci(Hd), ci(Sq), ci(Skv), ci(D),
                                  ctypes.c_float(scale), _stream()))
    return O


def flash_attention_f32_flat(q, k, v, B: int, Hd: int, Sq: int, Skv: int, D: int, scale: float) -> torch.Tensor:
    """flash_attention_f32 on the flat buffers of Q [B,Hd,Sq,D] and K, V [B,Hd,Skv,D]: the flat buffer of O."""
    O = _fast.flash_attention_f32_flat(q, k, v, B, Hd, Sq, Skv, D, scale)
    if O is not None:
        return O
    q, k, v = q.view(B, Hd, Sq, D), k.view(B, Hd, Skv, D), v.view(B, Hd, Skv, D)
    return flash_attention_f32(q.contiguous(), k.contiguous(), v.contiguous(), scale).view(-1)


def flash_attention_f32(Q, K, V, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                        workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Non-causal attention with fp32 Q [B,Hd,Sq,D], K, V [B,Hd,Skv,D] -> O [B,Hd,Sq,D] fp32; D of 32, 64, 96 or 128.
    Every product as three fp16 MFMAs of split operands, fp32 accumulation and softmax state."""
    O = _fast.flash_attention(False, Q, K, V, scale, out, workspace, False)
    if O is not None:
        return O
    f32 = torch.float32
    _req(Q, f32, 'Q'); _req(K, f32, 'K'); _req(V, f32, 'V')
    if Q.dim() != 4 or K.dim() != 4 or K.shape != V.shape or Q.shape[:2] != K.shape[:2] or Q.shape[3] != K.shape[3]:
        raise ValueError(f'Q [B,Hd,Sq,D] and K, V [B,Hd,Skv,D] expected, got {tuple(Q.shape)}, {tuple(K.shape)}, {tuple(V.shape)}')
    B, Hd, Sq, D = Q.shape
    Skv = K.shape[2]
    if scale is None:
        scale = D ** -0.5
    O = out if out is not None else torch.empty_like(Q)
    _req_out(O, f32, (B, Hd, Sq, D), 'O')
    need = int(lib.ftk_flash_attn_f32_workspace_bytes(B, Hd, Sq, Skv, D))
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=Q.device)
    _req_workspace(workspace)
    _count('flash_attention_f32')
    ci = ctypes.c_int
    _check(lib.ftk_flash_attn_f32(_ptr(Q), _ptr(K), _ptr(V), _ptr(O), ci(B), ci(Hd), ci(Sq), ci(Skv), ci(D), ctypes.c_float(scale),
                                  _ptr(workspace), ctypes.c_size_t(workspace.numel() * workspace.element_size()), _stream()))
    return O


def read_fa_trace(tiles: int):
    """Timeline of one wave of workgroup 0 of the last flash-attention launch: [tiles, 6] in us.  Only a tuning
    build of the library (make TRACE=1, run with FTK_FA_TRACE=1+wave) records it."""
    import numpy as np
    fn = getattr(lib, 'ftk_debug_read_fa_trace', None)
    if fn is None:
        raise RuntimeError('this build of libftkernels.so has no attention timeline: build it with make TRACE=1')
    fn.restype = ctypes.c_int
    buf = (ctypes.c_longlong * (tiles * 6))()
    _check(fn(buf, ctypes.c_int(tiles * 6)))
    return np.frombuffer(buf, dtype=np.int64).reshape(tiles, 6).astype(np.float64) / 100.0


def embedding_gather(table: torch.Tensor, ids: torch.Tensor, out: Optional[torch.Tensor] = None,
                     check: bool = True) -> torch.Tensor:
    """table [V,E] fp32, ids int32/int64 of any shape -> [*ids.shape, E]: rows of the table.

    check=True reads back the count of ids outside [0,V) (one synchronising copy of 4 bytes) and raises
    IndexError like indexing a FractalTensor does; check=False leaves such rows zero-filled."""
    _req(table, torch.float32, 'table')
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f'ids must be int32 or int64, got {ids.dtype}')
    if not ids.is_cuda or not ids.is_contiguous():
        raise RuntimeError('ids must be a contiguous CUDA tensor')
    if table.dim() != 2:
        raise ValueError('table must be [V, E]')
    V, E = table.shape
    n = ids.numel()
    if out is None:
        out = torch.empty((*ids.shape, E), dtype=torch.float32, device=table.device)
    else:
        _req(out, torch.float32, 'out')
        if out.numel() != n * E:
            raise ValueError('out must hold ids.numel() * E elements')
    if n == 0:
        return out
    bad = torch.zeros(1, dtype=torch.int32, device=table.device) if check else None
    _check(lib.ftk_embedding_gather_f32(_ptr(table), _ptr(ids), ctypes.c_int(1 if ids.dtype == torch.int64 else 0),
                                        _ptr(out), ctypes.c_longlong(n), ctypes.c_int(V), ctypes.c_int(E),
                                        _ptr(bad), _stream()))
    if check and int(bad.item()) != 0:
        raise IndexError(f'{int(bad.item())} ids are outside [0, {V})')
    return out


def online_softmax(x) -> torch.Tensor:
    """Row softmax of x [rows, cols], fp32."""
    _req(x, torch.float32, 'x')
    rows, cols = x.shape
    y = torch.empty_like(x)
    _check(lib.ftk_online_softmax_f32(_ptr(x), _ptr(y), ctypes.c_int(rows), ctypes.c_int(cols), _stream()))
    return y


def grid_rnn(xs, ys, Wx, Ux, bx, Wy, Uy, by, crossed: bool = False, out: Optional[torch.Tensor] = None,
             workspace: Optional[torch.Tensor] = None, relay_weights: bool = True) -> torch.Tensor:
    """Stacked grid RNN, fp32.  W* [D, H, H], U* [D, 2H, H], biases [D, 1 or B, H] or both None.
    crossed=False: xs [L1, B, H] feeds the first grid axis, ys [L2, B, H] the second (the layout of the
    reference's grid benchmark); crossed=True: xs [L2, B, H] is indexed by the second axis and ys [L1, B, H] by the
    first (the layout of its frontend program).  Returns hsss [D, L1, L2, 2, B, H]: h_x at index 0, h_y at 1.
    workspace: uint8 device tensor for the re-laid parameters (allocated here if None); relay_weights=False runs
    the kernel that reads the parameters where they lie."""
    for name, t in (('xs', xs), ('ys', ys), ('Wx', Wx), ('Ux', Ux), ('Wy', Wy), ('Uy', Uy)):
        _req(t, torch.float32, name)
    if xs.dim() != 3 or ys.dim() != 3 or xs.shape[1:] != ys.shape[1:]:
        raise ValueError(f'xs and ys must be [L, B, H] with equal B and H, got {tuple(xs.shape)} and {tuple(ys.shape)}')
    _, B, H = xs.shape
    L1, L2 = (ys.shape[0], xs.shape[0]) if crossed else (xs.shape[0], ys.shape[0])
    D = Wx.shape[0]
    for name, t, shape in (('Wx', Wx, (D, H, H)), ('Wy', Wy, (D, H, H)), ('Ux', Ux, (D, 2 * H, H)), ('Uy', Uy, (D, 2 * H, H))):
        if tuple(t.shape) != shape:
            raise ValueError(f'{name} must be {shape}, got {tuple(t.shape)}')
    if (bx is None) != (by is None):
        raise ValueError('give both biases or neither')
    bias_rows = 1
    if bx is not None:
        _req(bx, torch.float32, 'bx')
        _req(by, torch.float32, 'by')
        bias_rows = bx.shape[1]
        if tuple(bx.shape) != (D, bias_rows, H) or bx.shape != by.shape or bias_rows not in (1, B):
            raise ValueError(f'biases must both be [D, 1 or B, H], got {tuple(bx.shape)} and {tuple(by.shape)}')
    if out is None:
        out = torch.empty((D, L1, L2, 2, B, H), dtype=torch.float32, device=xs.device)
    else:
        _req(out, torch.float32, 'out')
        if tuple(out.shape) != (D, L1, L2, 2, B, H):
            raise ValueError(f'out must be {(D, L1, L2, 2, B, H)}, got {tuple(out.shape)}')
    if relay_weights and workspace is None:
        shared = Wx.data_ptr() == Wy.data_ptr() and Ux.data_ptr() == Uy.data_ptr()
        workspace = torch.empty(lib.ftk_grid_rnn_workspace_bytes(D, H) // (2 if shared else 1), dtype=torch.uint8, device=xs.device)
    ws_ptr, ws_bytes = (_ptr(workspace), workspace.numel()) if relay_weights else (None, 0)
    _check(lib.ftk_grid_rnn_f32(_ptr(xs), _ptr(ys), _ptr(Wx), _ptr(Ux), _ptr(bx), _ptr(Wy), _ptr(Uy), _ptr(by), _ptr(out),
                                ctypes.c_int(D), ctypes.c_int(L1), ctypes.c_int(L2), ctypes.c_int(B), ctypes.c_int(H),
                                ctypes.c_int(bias_rows), ctypes.c_int(1 if crossed else 0), ws_ptr, ctypes.c_size_t(ws_bytes), _stream()))
    return out


def windowed_attention(Q, K, V, window: int, dilation: int = 1, extra_idx: Optional[torch.Tensor] = None,
                       scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Q, K, V [G, S, D] fp32: every token attends to the `window` positions centred on it (`dilation` apart,
    wrapped at the ends as shifted_slide wraps them) and to extra_idx[g, t, :] (int32 [G, S, R]) if given."""
    for name, t in (('Q', Q), ('K', K), ('V', V)):
        _req(t, torch.float32, name)
    if Q.dim() != 3 or K.shape != Q.shape or V.shape != Q.shape:
        raise ValueError(f'Q, K and V must be [G, S, D] of one shape, got {tuple(Q.shape)}, {tuple(K.shape)}, {tuple(V.shape)}')
    G, S, D = Q.shape
    R = 0
    if extra_idx is not None:
        _req(extra_idx, torch.int32, 'extra_idx')
        if extra_idx.dim() != 3 or tuple(extra_idx.shape[:2]) != (G, S):
            raise ValueError(f'extra_idx must be [G, S, R], got {tuple(extra_idx.shape)}')
        R = extra_idx.shape[2]
        if R == 0:
            extra_idx = None
        elif int(extra_idx.min()) < 0 or int(extra_idx.max()) >= S:
            raise IndexError(f'extra_idx holds a position outside [0, {S})')
    if out is None:
        out = torch.empty_like(Q)
    else:
        _req(out, torch.float32, 'out')
        if out.shape != Q.shape:
            raise ValueError(f'out must be {tuple(Q.shape)}, got {tuple(out.shape)}')
    _check(lib.ftk_windowed_attn_f32(_ptr(Q), _ptr(K), _ptr(V), _ptr(extra_idx), _ptr(out), ctypes.c_int(G), ctypes.c_int(S),
                                     ctypes.c_int(D), ctypes.c_int(window), ctypes.c_int(dilation), ctypes.c_int(R),
                                     ctypes.c_float(scale), _stream()))
    return out


# ---- serving on a paged cache of keys and values ------------------------------------------
#
# The cache: k_pages, v_pages [pages, kv heads, page size, D], fp16, bf16, float8_e4m3fn or int8; the last two with
# k_exps, v_exps [pages, kv heads, page size] int8, an exponent for each row (element = code * 2^exponent).
# The batch, int32: starts [B + 1], the packed rows starts[b] .. starts[b + 1] - 1 are the new tokens of sequence b; lens [B], its length
# with them, so that they are its last positions; table [B, W], position p lies in row p % page size of page table[b, p // page size].
# What these arrays hold is looked at on the device only (include/ftk.h says what becomes of entries that point nowhere).

KV_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float8_e4m3fn: 2, torch.int8: 3}


def _req_on(t, dtype, shape, device, name: str) -> None:
    _req(t, dtype, name)
    if t.device != device:
        raise RuntimeError(f'{name} lives on {t.device}, the others on {device}')
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name} must be {tuple(shape)}, got {tuple(t.shape)}')


def _req_rows(t, dtype, heads, D: int, device, name: str) -> None:
    """[tokens, heads, D] with the elements of a head next to each other and strides of 8 elements otherwise."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{name} must be a torch.Tensor')
    if not t.is_cuda:
        raise RuntimeError(f'{name} must live on the GPU (got {t.device}); there is no CPU path')
    if t.device != device:
        raise RuntimeError(f'{name} lives on {t.device}, the others on {device}')
    if t.dtype != dtype:
        raise TypeError(f'{name} must be {dtype}, got {t.dtype}')
    if t.dim() != 3 or (heads is not None and t.shape[1] != heads) or t.shape[2] != D:
        raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {D}], got {tuple(t.shape)}")
    if t.stride(2) != 1 or any(t.shape[i] > 1 and t.stride(i) % 8 for i in (0, 1)):
        raise ValueError(f'{name}: the elements of a head must be contiguous and the other strides multiples of 8, got strides {t.stride()}')


def _req_cache(k_pages, v_pages, table, lens, starts, k_exps, v_exps) -> None:
    """Says what is wrong with a cache and a batch, if something is."""
    for t, name in ((k_pages, 'k_pages'), (v_pages, 'v_pages')):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f'{name} must be a torch.Tensor')
        if t.dtype not in KV_TYPES:
            raise TypeError(f'{name} must be float16, bfloat16, float8_e4m3fn or int8, got {t.dtype}')
        if t.dim() != 4:
            raise ValueError(f'{name} must be [pages, kv heads, page size, D], got {tuple(t.shape)}')
    device = k_pages.device
    _req(k_pages, k_pages.dtype, 'k_pages')
    _req_on(v_pages, k_pages.dtype, k_pages.shape, device, 'v_pages')
    codes = k_pages.dtype in (torch.float8_e4m3fn, torch.int8)
    for t, name in ((k_exps, 'k_exps'), (v_exps, 'v_exps')):
        if codes:
            if t is None:
                raise ValueError(f'pages of {k_pages.dtype} need {name}')
            _req_on(t, torch.int8, k_pages.shape[:3], device, name)
        elif t is not None:
            raise ValueError(f'pages of {k_pages.dtype} have no {name}')
    _req_on(lens, torch.int32, None, device, 'lens')
    if lens.dim() != 1:
        raise ValueError(f'lens must be [B], got {tuple(lens.shape)}')
    _req_on(starts, torch.int32, (lens.shape[0] + 1,), device, 'starts')
    _req_on(table, torch.int32, None, device, 'table')
    if table.dim() != 2 or table.shape[0] != lens.shape[0]:
        raise ValueError(f'table must be [B, W] with B = {lens.shape[0]}, got {tuple(table.shape)}')


def _req_pages_of(dtype, k_pages, name: str) -> None:
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f'{name} must be float16 or bfloat16, got {dtype}')
    if k_pages.dtype in (torch.float16, torch.bfloat16) and k_pages.dtype != dtype:
        raise TypeError(f'{name} must have the type of the pages, {k_pages.dtype}, got {dtype}')


def _not_negative(**values) -> None:
    for name, v in values.items():
        if isinstance(v, bool) or not isinstance(v, int) or not 0 <= v < 2 ** 31:
            raise ValueError(f'{name} must be a whole number from 0 up, got {v!r}')


def kv_cache_write(keys, values, k_pages, v_pages, table, lens, starts, k_exps=None, v_exps=None) -> None:
    """Writes the keys and values of new tokens, [tokens, kv heads, D] fp16 or bf16 (views with strides that are multiples of 8 are fine), into
    their pages: as they are into pages of their type, else as codes of 8 bits under the least power of two of each row and head that keeps it
    within the codes, rounded to nearest."""
    if _serving.kv_cache_write(keys, values, k_pages, v_pages, table, lens, starts, k_exps, v_exps):
        return
    _req_cache(k_pages, v_pages, table, lens, starts, k_exps, v_exps)
    for t, name in ((keys, 'keys'), (values, 'values')):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f'{name} must be a torch.Tensor')
        _req_pages_of(t.dtype, k_pages, name)
        _req_rows(t, keys.dtype, k_pages.shape[1], k_pages.shape[3], k_pages.device, name)
    raise ValueError(f'keys and values must have as many tokens, got {keys.shape[0]} and {values.shape[0]}')


def kv_cache_read(k_pages, v_pages, table, lens, starts, tokens: int, dtype=None, k_exps=None, v_exps=None,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The last starts[b + 1] - starts[b] positions of every sequence as dense keys and values [tokens, kv heads, D]; tokens is what the
    arrays hold rows of (rows that are no sequence's are left as they were).  dtype: fp16, bf16 or fp32, for pages of 16 bits their own type (the
    default) or fp32; for codes of 8 bits there is no default."""
    own = getattr(k_pages, 'dtype', None)
    if dtype is None:
        dtype = own
    ok, ov = (None, None) if out is None else out
    if dtype in (torch.float16, torch.bfloat16, torch.float32) and (own not in (torch.float16, torch.bfloat16) or dtype in (own, torch.float32)):
        done = _serving.kv_cache_read(_LIKE[dtype], k_pages, v_pages, table, lens, starts, k_exps, v_exps, tokens, ok, ov)
        if done is not None:
            return done
    _req_cache(k_pages, v_pages, table, lens, starts, k_exps, v_exps)
    _not_negative(tokens=tokens)
    if dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError(f'dtype must be float16, bfloat16 or float32, got {dtype}')
    if k_pages.dtype in (torch.float16, torch.bfloat16) and dtype not in (k_pages.dtype, torch.float32):
        raise TypeError(f'pages of {k_pages.dtype} are read in that type or in float32, not {dtype}')
    shape = (tokens, k_pages.shape[1], k_pages.shape[3])
    for t, name in ((ok, 'out[0]'), (ov, 'out[1]')):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f'{name} must be a torch.Tensor')
        _req_out(t, dtype, shape, name)
        _req_on(t, dtype, shape, k_pages.device, name)
    raise ValueError('kv_cache_read: these arguments are not taken')


_LIKE = {t: torch.empty(0, dtype=t) for t in (torch.float16, torch.bfloat16, torch.float32)}


def paged_attention_workspace_bytes(q, k_pages, table, max_queries: int = 0, max_keys: int = 0, window: int = 0) -> int:
    """Bytes that paged_attention wants for a batch of this shape on the device of q; 0 where the keys are not cut into parts."""
    pages = KvPages(None, None, None, None, KV_TYPES[k_pages.dtype], *k_pages.shape)
    batch = KvBatch(None, None, None, table.shape[0], table.shape[1], q.shape[0])
    with torch.cuda.device(q.device):
        return int(lib.ftk_paged_attn_workspace_bytes(ctypes.byref(pages), ctypes.byref(batch), q.shape[1], window, max_queries, max_keys))


def _req_attention(q, args, out, lse, workspace, **numbers) -> None:
    """Says what is wrong with queries, a cache and a batch, and where the results go, if something is."""
    _req_cache(*args)
    k_pages = args[0]
    if not isinstance(q, torch.Tensor):
        raise TypeError('q must be a torch.Tensor')
    _req_pages_of(q.dtype, k_pages, 'q')
    _req_rows(q, q.dtype, None, k_pages.shape[3], k_pages.device, 'q')
    _not_negative(**numbers)
    if out is not None:
        _req_out(out, q.dtype, q.shape, 'out')
        _req_on(out, q.dtype, q.shape, q.device, 'out')
    if isinstance(lse, torch.Tensor):
        _req_out(lse, torch.float32, q.shape[:2], 'return_lse')
        _req_on(lse, torch.float32, q.shape[:2], q.device, 'return_lse')
    if workspace is not None:
        _req_on(_req_workspace(workspace), workspace.dtype, None, q.device, 'workspace')


def paged_attention(q, k_pages, v_pages, table, lens, starts, k_exps=None, v_exps=None, scale: Optional[float] = None, causal: bool = True,
                    window: int = 0, max_queries: int = 0, max_keys: int = 0, out: Optional[torch.Tensor] = None, return_lse=False,
                    workspace: Optional[torch.Tensor] = None):
    """Attention of new tokens q [tokens, heads, D] (fp16 or bf16; views with strides that are multiples of 8 are fine) over the cache, which holds
    their own keys and values already: one token a sequence, drafts, chunks of prompts or whole ones, in any mixture.  heads is a multiple
    of the kv heads; each of these serves heads / kv heads neighbours.  causal: the token at position p sees positions up to p; window > 0: from
    p - window + 1 on.  scale defaults to D ** -0.5.  A token that sees nothing gets zeros (and -inf).
    max_queries, max_keys: the most new tokens and the greatest length of a sequence, where the program knows them (0: not known); they decide which
    kernel runs and how it cuts the keys, and no sequence may have more new tokens than max_queries.
    Returns o [tokens, heads, D], or (o, lse [tokens, heads] fp32) with return_lse (True, or the tensor to write to): the logs of the sums of
    exponentials.  The workspace (paged_attention_workspace_bytes) is allocated here unless one is given."""
    args = (k_pages, v_pages, table, lens, starts, k_exps, v_exps)
    done = _serving.paged_attention(q, *args, scale, causal, window, max_queries, max_keys, out, return_lse, workspace)
    if done is None:
        _req_attention(q, args, out, return_lse, workspace, window=window, max_queries=max_queries, max_keys=max_keys)
        done = _serving.paged_attention(q, *args, None if scale is None else float(scale), bool(causal), window, max_queries, max_keys, out,
                                        return_lse if isinstance(return_lse, torch.Tensor) else bool(return_lse), workspace)
        if done is None:
            raise ValueError('paged_attention: these arguments are not taken')
    return done[0] if done[1] is None else done


def verify_drafts(target, draft, drafts, accept_uniforms, sample_uniforms, draft_lens=None,
                  workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which drafted tokens a target model accepts, and the token that follows them.

    target [B, K + 1, V]: the target's probabilities before each draft and behind the last; draft [B, K, V]: those the drafts were drawn from
    (the same type: fp32, fp16 or bf16), or None for drafts that were not drawn at random; drafts [B, K] int32 or int64; uniform numbers of
    [0, 1) accept_uniforms [B, K] and sample_uniforms [B] fp32; draft_lens [B] int32: how many drafts a sequence has (None: K).
    A draft is accepted, if all before it are, where uniform * draft < target; the next token is drawn from max(target - draft, 0) of the
    first that is not, or from the target behind the last.  Returns tokens [B, K + 1] of drafts' type (the accepted ones, the next, then -1) and
    accepted [B] int32.  The numbers decide everything: the same ones give the same tokens."""
    args = (target, draft, drafts, accept_uniforms, sample_uniforms, draft_lens, workspace)
    done = _serving.verify_drafts(*args)
    if done is not None:
        return done
    if not isinstance(target, torch.Tensor) or not isinstance(drafts, torch.Tensor):
        raise TypeError('target and drafts must be torch.Tensors')
    if target.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f'target must be float32, float16 or bfloat16, got {target.dtype}')
    if drafts.dtype not in (torch.int32, torch.int64):
        raise TypeError(f'drafts must be int32 or int64, got {drafts.dtype}')
    if target.dim() != 3 or drafts.dim() != 2:
        raise ValueError(f'target must be [B, K + 1, V] and drafts [B, K], got {tuple(target.shape)} and {tuple(drafts.shape)}')
    (B, K), V, device = drafts.shape, target.shape[2], target.device
    _req_on(target, target.dtype, (B, K + 1, V), device, 'target')
    _req_on(drafts, drafts.dtype, None, device, 'drafts')
    if draft is not None:
        _req_on(draft, target.dtype, (B, K, V), device, 'draft')
    _req_on(accept_uniforms, torch.float32, (B, K), device, 'accept_uniforms')
    _req_on(sample_uniforms, torch.float32, (B,), device, 'sample_uniforms')
    if draft_lens is not None:
        _req_on(draft_lens, torch.int32, (B,), device, 'draft_lens')
    if workspace is not None:
        _req_on(_req_workspace(workspace), workspace.dtype, None, device, 'workspace')
    raise ValueError('verify_drafts: these arguments are not taken')


# ---- trees of drafted tokens, and caches of limited length ----------------------------------
#
# A tree of drafts: the new tokens of a sequence, and for each of them parents [tokens] int32, the number of the token that it follows among those of
# its sequence (counted from 0; a parent comes before its children), or a negative one for what follows the cache itself.
# Weights [pages, kv heads, page size] fp32: what each position of the cache has been given, beside its keys.

TREE_TOKENS = 256


def paged_tree_attention_workspace_bytes(q, k_pages, table, max_queries: int = 0, max_keys: int = 0, window: int = 0) -> int:
    """Bytes that paged_tree_attention wants for a batch of this shape on the device of q; 0 where the keys are not cut into parts."""
    pages = KvPages(None, None, None, None, KV_TYPES[k_pages.dtype], *k_pages.shape)
    batch = KvBatch(None, None, None, table.shape[0], table.shape[1], q.shape[0])
    with torch.cuda.device(q.device):
        return int(lib.ftk_paged_tree_attn_workspace_bytes(ctypes.byref(pages), ctypes.byref(batch), q.shape[1], window, max_queries, max_keys))


def paged_tree_attention(q, k_pages, v_pages, table, lens, starts, parents, k_exps=None, v_exps=None, scale: Optional[float] = None, window: int = 0,
                         max_queries: int = 0, max_keys: int = 0, out: Optional[torch.Tensor] = None, return_lse=False, workspace: Optional[torch.Tensor] = None):
    """paged_attention for new tokens that form a tree: each sees the cache in front of its sequence's new tokens, its ancestors and itself, whose keys and
    values the cache holds already, at the sequence's last positions in the order of their rows.  window > 0: of these the last `window` on the way that
    ends with it.  At most 256 new tokens a sequence, which max_queries has to say where the call has more of all sequences together.  All else is as
    in paged_attention, what it returns too."""
    args = (k_pages, v_pages, table, lens, starts, k_exps, v_exps)
    done = _serving.paged_tree_attention(q, *args, scale, parents, window, max_queries, max_keys, out, return_lse, workspace)
    if done is None:
        _req_attention(q, args, out, return_lse, workspace, window=window, max_queries=max_queries, max_keys=max_keys)
        _req_on(parents, torch.int32, q.shape[:1], q.device, 'parents')
        done = _serving.paged_tree_attention(q, *args, None if scale is None else float(scale), parents, window, max_queries, max_keys, out,
                                             return_lse if isinstance(return_lse, torch.Tensor) else bool(return_lse), workspace)
        if done is None:
            raise ValueError('paged_tree_attention: these arguments are not taken')
    return done[0] if done[1] is None else done


def verify_tree(target, ids, parents, starts, uniforms, workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The path through a tree of drafts that the target model's own draws follow, and the token behind it.

    The packed rows starts[b] .. starts[b + 1] - 1 are the tokens of sequence b: first the root, the last token that is known already, then the drafts.
    target [tokens, V] (fp32, fp16 or bf16): the target's probabilities of what follows each; ids [tokens] int32 or int64; parents [tokens] int32; uniforms
    [B, M] fp32 of [0, 1), one for each step.  From the root on a token is drawn at each node; where the node has a child with it, the way goes on
    there.  Returns next [B, M] of ids' type (the tokens that were drawn: the accepted drafts and one more, then -1), path [B, M] int32 (the nodes that
    stay in the cache, by their number in the sequence, then -1: a list for kv_cache_keep) and accepted [B] int32.  The tokens are distributed as
    the target's own, however the drafts were chosen.  The workspace (4 bytes a token) is allocated here unless one is given."""
    done = _serving.verify_tree(target, ids, parents, starts, uniforms, workspace)
    if done is not None:
        return done
    if not isinstance(target, torch.Tensor) or not isinstance(ids, torch.Tensor):
        raise TypeError('target and ids must be torch.Tensors')
    if target.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f'target must be float32, float16 or bfloat16, got {target.dtype}')
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f'ids must be int32 or int64, got {ids.dtype}')
    if target.dim() != 2:
        raise ValueError(f'target must be [tokens, V], got {tuple(target.shape)}')
    _req_on(target, target.dtype, None, target.device, 'target')
    _req_on(ids, ids.dtype, target.shape[:1], target.device, 'ids')
    _req_on(parents, torch.int32, target.shape[:1], target.device, 'parents')
    _req_on(starts, torch.int32, None, target.device, 'starts')
    if starts.dim() != 1 or starts.shape[0] < 1:
        raise ValueError(f'starts must be [B + 1], got {tuple(starts.shape)}')
    _req_on(uniforms, torch.float32, None, target.device, 'uniforms')
    if uniforms.dim() != 2 or uniforms.shape[0] != starts.shape[0] - 1:
        raise ValueError(f'uniforms must be [B, M] with B = {starts.shape[0] - 1}, got {tuple(uniforms.shape)}')
    if workspace is not None:
        _req_on(_req_workspace(workspace), workspace.dtype, None, target.device, 'workspace')
    raise ValueError('verify_tree: these arguments are not taken')


def _req_weights(weights, pages, device) -> None:
    _req_on(weights, torch.float32, pages, device, 'weights')
    if weights.dim() != 3:
        raise ValueError(f'weights must be [pages, kv heads, page size], got {tuple(weights.shape)}')


def kv_cache_weigh_workspace_bytes(q, k_pages, table, max_queries: int = 0, max_keys: int = 0) -> int:
    """Bytes that kv_cache_weigh wants for a batch of this shape on the device of q; 0 where the rows are not cut into parts."""
    pages = KvPages(None, None, None, None, KV_TYPES[k_pages.dtype], *k_pages.shape)
    batch = KvBatch(None, None, None, table.shape[0], table.shape[1], q.shape[0])
    with torch.cuda.device(q.device):
        return int(lib.ftk_kv_cache_weigh_workspace_bytes(ctypes.byref(pages), ctypes.byref(batch), q.shape[1], max_queries, max_keys))


def kv_cache_weigh(q, lse, k_pages, weights, table, lens, starts, k_exps=None, scale: Optional[float] = None, decay: float = 1.0, causal: bool = True,
                   window: int = 0, max_queries: int = 0, max_keys: int = 0, workspace: Optional[torch.Tensor] = None) -> None:
    """Adds to weights, of every position of the sequences that have new tokens, the attention weights that these give it: the sum of exp(scale q . k - lse) over
    the new tokens that see it and the query heads that read its head.  q [tokens, heads, D] and lse [tokens, heads] as in, and out of, paged_attention
    with the same scale, causal and window.  What older positions had is multiplied by decay (0 to 1) first, new ones begin at zero.  max_queries, max_keys: as in
    paged_attention.  The workspace (kv_cache_weigh_workspace_bytes) is allocated here unless one is given."""
    decay = decay if isinstance(decay, float) else float(decay)
    if _serving.kv_cache_weigh(q, lse, k_pages, weights, table, lens, starts, k_exps, scale, decay, causal, window, max_queries, max_keys, workspace):
        return
    _req_attention(q, (k_pages, k_pages, table, lens, starts, k_exps, k_exps), None, None, workspace, window=window, max_queries=max_queries, max_keys=max_keys)
    _req_on(lse, torch.float32, q.shape[:2], q.device, 'lse')
    _req_weights(weights, k_pages.shape[:3], q.device)
    if not _serving.kv_cache_weigh(q, lse, k_pages, weights, table, lens, starts, k_exps, None if scale is None else float(scale), decay, bool(causal), window, max_queries, max_keys,
                                   workspace):
        raise ValueError('kv_cache_weigh: these arguments are not taken')


def kv_cache_select(weights, table, lens, budget: int, sinks: int = 0, recent: int = 0, max_keys: int = 0) -> torch.Tensor:
    """Which positions of every sequence and head stay in a cache of `budget` positions: the first `sinks`, the last `recent` and of the others those of the largest
    weights, of equal ones the earlier.  Returns kept [B, kv heads, budget] int32, ascending, then -1: lists for kv_cache_keep.  A sequence of at most
    `budget` positions keeps them all.  max_keys: the greatest length where the program knows it."""
    done = _serving.kv_cache_select(weights, table, lens, budget, sinks, recent, max_keys)
    if done is not None:
        return done
    _req(weights, torch.float32, 'weights')
    _req_weights(weights, None, weights.device)
    _req_on(lens, torch.int32, None, weights.device, 'lens')
    if lens.dim() != 1:
        raise ValueError(f'lens must be [B], got {tuple(lens.shape)}')
    _req_on(table, torch.int32, None, weights.device, 'table')
    if table.dim() != 2 or table.shape[0] != lens.shape[0]:
        raise ValueError(f'table must be [B, W] with B = {lens.shape[0]}, got {tuple(table.shape)}')
    _not_negative(budget=budget, sinks=sinks, recent=recent, max_keys=max_keys)
    raise ValueError('kv_cache_select: these arguments are not taken')


def kv_cache_keep(k_pages, v_pages, table, lens, kept, starts=None, k_exps=None, v_exps=None, weights=None) -> torch.Tensor:
    """Moves the rows that stay together, in place: row kept[b, j] (or kept[b, head, j]) of sequence b goes to place j, for keys, values, exponents and, where they are
    given, weights.  Rows are counted from the sequence's begin, or with starts from its first new token.  kept [B, M] or [B, kv heads, M] int32
    ascends and has -1 behind its end; the lists of a sequence's heads are of one length.  Returns the new lengths [B] int32."""
    done = _serving.kv_cache_keep(k_pages, v_pages, table, lens, kept, starts, k_exps, v_exps, weights)
    if done is not None:
        return done
    if starts is None and isinstance(lens, torch.Tensor) and lens.dim() == 1:
        _req_cache(k_pages, v_pages, table, lens, lens.new_zeros(lens.shape[0] + 1, dtype=torch.int32), k_exps, v_exps)
    else:
        _req_cache(k_pages, v_pages, table, lens, starts, k_exps, v_exps)
    _req_on(kept, torch.int32, None, k_pages.device, 'kept')
    if kept.dim() not in (2, 3) or kept.shape[0] != lens.shape[0] or (kept.dim() == 3 and kept.shape[1] != k_pages.shape[1]):
        raise ValueError(f'kept must be [B, M] or [B, kv heads, M] with B = {lens.shape[0]}, got {tuple(kept.shape)}')
    if weights is not None:
        _req_weights(weights, k_pages.shape[:3], k_pages.device)
    raise ValueError('kv_cache_keep: these arguments are not taken')
