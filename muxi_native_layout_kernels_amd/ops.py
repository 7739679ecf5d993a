"""Host-side mirror of the reference's operator interface for the hot path.

Same names, positional order, keyword names and defaults as the pybind module
of the reference (csrc/ffi.cu:32-143); each function checks its arguments the way
the reference's host launcher does, looks up launch parameters in the csv
tables, allocates the output and calls the C-ABI library on torch's current HIP
stream.  PyTorch is used for device memory and streams only.

Reference naming: `m` = weight rows (output features), `k` = reduction,
`n` = activation rows (tokens).
"""
import ctypes
import threading

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib, arg_selector

_KIND = {torch.float16: 0, torch.bfloat16: 1}
_FP8_KIND = 2


def _stream():
    return torch.cuda.current_stream().cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_of(t):
    """Raw handle of torch's current stream on the tensor's device (the short way when torch offers it)."""
    if _raw_stream is not None:
        return _raw_stream(t.get_device())
    return torch.cuda.current_stream(t.device).cuda_stream


# Launch plans of the eager entry points.  The first call with a given combination of shapes, dtypes and device
# runs every argument check and the table lookup, and leaves the launch arguments here; later calls with the same
# combination only check what a shape does not tell (contiguity, alpha / beta), allocate the output and call the
# library.  A plan is a few integers: the cache is never cleared.
_plans = {}


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _check(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _is_fp8(t):
    return t.element_size() == 1


def _kind(t):
    if _is_fp8(t):
        return _FP8_KIND
    _check(t.dtype in _KIND, "Unsupported data type")
    return _KIND[t.dtype]


# --------------------------------------------------------------- workspaces
class WorkspacePool:
    """Device scratch handed to the kernels as raw pointers (cross-workgroup K-split partials and their
    arrival counters, the MoE alignment tables and intermediate).

    * One buffer per (device, stream): two calls that run side by side on different streams never share
      counters or partials.  Calls on one stream are ordered, so they can share.
    * A buffer that has been handed out stays allocated for the life of the process.  A HIP graph captured
      earlier replays with the pointer it was captured with; when a later call needs more room, a new, larger
      buffer takes over for new calls and the old one is retired, not freed.
    * `zero_prefix` bytes at the front are cleared when a buffer is created (the K-split kernels count
      arrivals there and leave the counters at zero).
    """

    def __init__(self, min_bytes, zero_prefix=False):
        self.min_bytes = int(min_bytes)
        self.zero_prefix = zero_prefix
        self._lock = threading.Lock()
        self._live = {}
        self._retired = []

    def get(self, device, stream, nbytes, prefix_bytes=0):
        key = (device.type, device.index, int(stream))
        with self._lock:
            buf = self._live.get(key)
            if buf is None or buf.numel() < nbytes:
                old = buf
                grown = 0 if old is None else old.numel() + old.numel() // 2      # few retirements on a growing series
                size = max(int(nbytes), self.min_bytes, grown)
                buf = torch.empty(size, dtype=torch.uint8, device=device)
                if self.zero_prefix and prefix_bytes:
                    buf[:prefix_bytes].zero_()
                if old is not None:                    # only now: where there is no room for more, it stays in use
                    self._retired.append(old)
                self._live[key] = buf
            return buf

    def owned(self):
        """Every buffer ever handed out (live and retired)."""
        with self._lock:
            return list(self._live.values()) + list(self._retired)

    def held_bytes(self):
        with self._lock:
            return sum(b.numel() for b in self._live.values()) + sum(b.numel() for b in self._retired)

    def release(self, retired_only=False):
        """Drop the retired buffers and, unless `retired_only`, the live ones too (they are re-created on the next
        call).  Only for callers that hold no captured graph which replays one of these pointers, and with no call
        of this library in flight on the device."""
        with self._lock:
            freed = sum(b.numel() for b in self._retired)
            self._retired = []
            if not retired_only:
                freed += sum(b.numel() for b in self._live.values())
                self._live = {}
        return freed


_gemm_pool = WorkspacePool(1 << 22, zero_prefix=True)
_moe_pool = WorkspacePool(1 << 20)
_balance_pool = WorkspacePool(1 << 16, zero_prefix=True)


def workspace_bytes_held():
    """Device bytes the library's scratch pools hold right now (K-split partials, MoE tables and intermediates, sums of the balance loss)."""
    return _gemm_pool.held_bytes() + _moe_pool.held_bytes() + _balance_pool.held_bytes()


def release_workspaces(retired_only=False):
    """Give the scratch memory of the K-split GeMMs, of the fused MoE and of the balance loss back to torch's allocator and
    return the number of bytes released.  The pools keep one buffer per (device, stream) and never free by themselves, so that
    a HIP graph captured around a call replays with valid pointers; a caller that holds no such graph (or has
    dropped it) calls this after a burst of large batches, or when streams it used are gone.  `retired_only`
    releases just the buffers that a larger one has replaced.  Synchronize the device first."""
    return _gemm_pool.release(retired_only) + _moe_pool.release(retired_only) + _balance_pool.release(retired_only)


def _workspace(device, nbytes, counter_bytes, stream=None):
    """Scratch for cross-workgroup K splits on `stream` (default: torch's current stream)."""
    return _gemm_pool.get(device, _stream() if stream is None else stream, nbytes, counter_bytes)


def _split_scratch(device, stream, nbytes, counter_bytes):
    """The same, or None where the card has no room: every kernel also runs in one slice, which needs none."""
    try:
        return _gemm_pool.get(device, stream, nbytes, counter_bytes)
    except torch.OutOfMemoryError:
        return None


# ------------------------------------------------------------------ relayout
def pack_layout_a(weight):
    """[N, K] or [E, N, K] (16-bit or 1-byte elements) -> layout-A [.., N/16, K/8, 16, 8].

    Device counterpart of the offline `A.view(m//16,16,k//8,8).permute(0,2,1,3)`
    (benchmark_and_test/gemv_benchmark.py:47-48, test_muxi_moe.py:74-81)."""
    _check(weight.is_cuda, "weight must be a CUDA tensor")
    _check(weight.is_contiguous(), "weight must be contiguous")
    _check(weight.dim() in (2, 3), "weight must be 2D or 3D")
    n, k = weight.shape[-2], weight.shape[-1]
    _check(n % 16 == 0 and k % 8 == 0, "N % 16 and K % 8 must be 0")
    batch = weight.shape[0] if weight.dim() == 3 else 1
    out = torch.empty(tuple(weight.shape[:-2]) + (n // 16, k // 8, 16, 8), dtype=weight.dtype, device=weight.device)
    lib = _lib.load()
    _lib.check(lib.mlk_pack_layout_a(_ptr(weight), _ptr(out), batch, n, k, weight.element_size(), _stream()),
               "pack_layout_a")
    return out


def unpack_layout_a(a_nat):
    """layout-A [.., N/16, K/8, 16, 8] -> [.., N, K]."""
    _check(a_nat.is_cuda and a_nat.is_contiguous(), "A must be a contiguous CUDA tensor")
    _check(a_nat.dim() in (4, 5) and a_nat.shape[-2] == 16 and a_nat.shape[-1] == 8, "A must be in layout-A")
    n, k = a_nat.shape[-4] * 16, a_nat.shape[-3] * 8
    batch = a_nat.shape[0] if a_nat.dim() == 5 else 1
    out = torch.empty(tuple(a_nat.shape[:-4]) + (n, k), dtype=a_nat.dtype, device=a_nat.device)
    lib = _lib.load()
    _lib.check(lib.mlk_unpack_layout_a(_ptr(a_nat), _ptr(out), batch, n, k, a_nat.element_size(), _stream()),
               "unpack_layout_a")
    return out


def layoutB(B):
    """Row-major activations [n, k] -> layout-B [k/32, n/16, 4, 16, 8] (csrc/layout_b.cu:65-99)."""
    _check(B.is_cuda, "B must be a CUDA tensor")
    _check(B.is_contiguous(), "B must be contiguous")
    _check(B.dim() == 2, "B must be a 2D tensor")
    n, k = B.shape
    _check(n % 16 == 0, "n must be a multiple of 16")
    _check(k % 32 == 0, "k must be a multiple of 32")
    _check(B.dtype in _KIND, "Unsupported data type")
    out = torch.empty((k // 32, n // 16, 4, 16, 8), dtype=B.dtype, device=B.device)
    _lib.check(_lib.load().mlk_layout_b(_ptr(B), _ptr(out), n, k, _stream()), "layoutB")
    return out


def reLayoutC(C):
    """layout-C [m/32, n/16, 4, 16, 8] -> row-major [n, m] (csrc/re_layout_c.cu:63-95)."""
    _check(C.is_cuda, "C must be a CUDA tensor")
    _check(C.is_contiguous(), "C must be contiguous")
    _check(C.dim() == 5, "C must be a 5D tensor")
    _check(C.shape[2] == 4 and C.shape[3] == 16 and C.shape[4] == 8, "C must be in layout-C [m/32, n/16, 4, 16, 8]")
    _check(C.dtype in _KIND, "Unsupported data type")
    m, n = C.shape[0] * 32, C.shape[1] * 16
    out = torch.empty((n, m), dtype=C.dtype, device=C.device)
    _lib.check(_lib.load().mlk_re_layout_c(_ptr(C), _ptr(out), n, m, _stream()), "reLayoutC")
    return out


def fp8_weight_repack(weight):
    """Swap bytes 1 and 2 of every 4-byte group (csrc/fp8_weight_repack.cu:44-67)."""
    _check(weight.is_cuda, "weight must be a CUDA tensor")
    _check(weight.is_contiguous(), "weight must be contiguous")
    _check(weight.element_size() == 1, "weight must hold one byte per element")
    _check(weight.numel() % 4 == 0, "weight size must be a multiple of 4 bytes")
    out = torch.empty_like(weight)
    _lib.check(_lib.load().mlk_fp8_weight_repack(_ptr(weight), _ptr(out), weight.numel(), _stream()),
               "fp8_weight_repack")
    return out


# ---------------------------------------------------------------------- GeMV
def _check_beta(beta):
    # The reference accepts beta everywhere and no kernel of it ever reads it
    # (csrc/layout_gemv_kernel.cuh:377 only derives an unused flag); C is never an input.
    _check(float(beta) == 0.0, "beta != 0 is not supported: the output is never read (the reference ignores beta)")


def _layout_a_dims(A):
    _check(A.dim() == 4, "A must be a 4D tensor")
    _check(A.size(2) == 16, "A.shape[2] must be 16")
    _check(A.size(3) == 8, "A.shape[3] must be 8")
    return A.size(0) * 16, A.size(1) * 8


def gemv_layoutA_wapper(A, B, m, k, alpha=1, beta=0, blockDimX=256, kernelId=1, kernelParam1=1, kernelParam2=1,
                        scale_matrix=None, bias=None):
    """Run the GeMV with explicit launch parameters (csrc/gemv_layout_a.cu:17-71)."""
    _check_beta(beta)
    _check(A.is_cuda and B.is_cuda, "A and B must be CUDA tensors")
    _check(B.dtype in _KIND, "Unsupported data type")
    a_kind = _kind(A)
    if a_kind == _FP8_KIND:
        _check(B.dtype == torch.bfloat16, "Unsupported data type")
        if scale_matrix is not None:
            _check(scale_matrix.dtype == torch.float32 and scale_matrix.is_contiguous(),
                   "scale_matrix must be contiguous fp32")
            _check(tuple(scale_matrix.shape) == ((m + 127) // 128, (k + 127) // 128),
                   "scale_matrix must be [ceil(m/128), ceil(k/128)]")
    else:
        _check(A.dtype == B.dtype, "Unsupported data type")
        scale_matrix = None
    if bias is not None:
        _check(bias.dtype == B.dtype and bias.numel() == m, "bias must be [1, m] of the activation dtype")
    rows = B.size(0)
    C = torch.empty((rows, m), dtype=B.dtype, device=B.device)
    _lib.check(_lib.load().mlk_gemv_layout_a(_ptr(A), _ptr(B), _ptr(C), rows, m, k, a_kind, _KIND[B.dtype],
                                             float(alpha), _ptr(bias), _ptr(scale_matrix), int(blockDimX),
                                             int(kernelId), int(kernelParam1), int(kernelParam2), _stream()),
               "gemv_layoutA")
    return C


def gemv_layoutA(A, B, alpha=1, beta=0, scale_matrix=None, bias=None):
    """y[1, m] = alpha * B[1, k] . A^T (+ bias), A in layout-A (csrc/gemv_layout_a.cu:73-150)."""
    key = ("gemv", A.shape, B.shape, A.dtype, B.dtype, A.device, B.device,
           None if scale_matrix is None else (scale_matrix.shape, scale_matrix.dtype, scale_matrix.device),
           None if bias is None else (bias.shape, bias.dtype, bias.device))
    plan = _plans.get(key)
    if plan is not None and beta == 0 and A.is_contiguous() and B.is_contiguous() and \
            (scale_matrix is None or scale_matrix.is_contiguous()) and (bias is None or bias.is_contiguous()):
        m, k, a_kind, x_kind, block, kid, p1, p2, use_scale, fn = plan
        C = torch.empty((1, m), dtype=B.dtype, device=B.device)
        rc = fn(A.data_ptr(), B.data_ptr(), C.data_ptr(), 1, m, k, a_kind, x_kind, float(alpha),
                0 if bias is None else bias.data_ptr(), scale_matrix.data_ptr() if use_scale else 0,
                block, kid, p1, p2, _stream_of(B))
        if rc != 0:
            _lib.check(rc, "gemv_layoutA")
        return C
    C = _gemv_layoutA_checked(A, B, alpha, beta, scale_matrix, bias)
    m, k = A.size(0) * 16, A.size(1) * 8
    if _is_fp8(A) and B.dtype == torch.bfloat16:
        table = "gemv_soft_fp8"
    else:
        table = "gemv_fp16" if B.dtype == torch.float16 else "gemv_bf16"
    block, kid, p1, p2 = arg_selector.gemv_guard(arg_selector.selector(table).get_args((m, k)), m, k)
    _plans[key] = (m, k, _kind(A), _KIND[B.dtype], block, kid, p1, p2, _is_fp8(A) and scale_matrix is not None,
                   _lib.load().mlk_gemv_layout_a)
    return C


def _gemv_layoutA_checked(A, B, alpha=1, beta=0, scale_matrix=None, bias=None):
    """Every argument check of the reference's host launcher, the table lookup, the launch."""
    _check(A.is_cuda, "A must be a CUDA tensor")
    _check(B.is_cuda, "B must be a CUDA tensor")
    _check(A.is_contiguous(), "A must be contiguous")
    _check(B.is_contiguous(), "B must be contiguous")
    m, a_k = _layout_a_dims(A)
    _check(B.dim() == 2 and B.size(0) == 1, "B must be a vector")
    _check(a_k == B.size(1), "A and B must have the same k")
    k = a_k
    _check(m % 16 == 0, "GEMV m % 16(at least) must be 0")
    _check(k % 32 == 0, "GEMV k % 32(at least) must be 0")
    if _is_fp8(A) and B.dtype == torch.bfloat16:
        sel = arg_selector.selector("gemv_soft_fp8")
    elif B.dtype == torch.float16:
        sel = arg_selector.selector("gemv_fp16")
    elif B.dtype == torch.bfloat16:
        sel = arg_selector.selector("gemv_bf16")
    else:
        raise RuntimeError("Unsupported data type")
    block, kid, p1, p2 = arg_selector.gemv_guard(sel.get_args((m, k)), m, k)
    return gemv_layoutA_wapper(A, B, m, k, alpha, beta, block, kid, p1, p2, scale_matrix, bias)


# ---------------------------------------------------------------------- GEMM
_B_ROWMAJOR, _B_NATIVE = 0, 1
_C_ROWMAJOR, _C_NATIVE = 0, 1


def _gemm_call(A, A_Scale, B, m, n, k, alpha, beta, bias, b_mode, c_mode, kernel_id, p1, p2, p3, what):
    _check_beta(beta)
    _check(B.dtype in _KIND, "Unsupported data type")
    a_kind = _kind(A)
    if a_kind == _FP8_KIND:
        _check(B.dtype == torch.bfloat16, "soft-FP8 weights need bf16 activations")
        if A_Scale is not None:
            _check(A_Scale.dtype == torch.float32 and A_Scale.is_contiguous(), "A_Scale must be contiguous fp32")
            _check(tuple(A_Scale.shape) == ((m + 127) // 128, (k + 127) // 128),
                   "A_Scale must be [ceil(m/128), ceil(k/128)]")
    else:
        _check(A.dtype == B.dtype, "Unsupported data type")
        A_Scale = None
    if bias is not None:
        _check(bias.dtype == B.dtype and bias.numel() == m, "bias must be [1, m] of the activation dtype")
    if c_mode == _C_NATIVE:
        C = torch.empty((m // 32, n // 16, 4, 16, 8), dtype=B.dtype, device=B.device)
    else:
        C = torch.empty((n, m), dtype=B.dtype, device=B.device)
    lib = _lib.load()
    ws = None
    ws_bytes = 0
    if _off_panels(kernel_id, _ptr(A) | _ptr(B)) and p1 in (2, 4) and 1 <= p2 <= 4 and 1 <= p3 <= 64 and k % 128 == 0:
        copy = _on16(A, B, n)
        if copy is not None:
            B = copy
        else:
            kernel_id, p1, p2, p3, _ = _off16_plan(m, n, k, a_kind, b_mode, c_mode)
    if p3 > 1:
        ws = _split_scratch(B.device, _stream(), _gemm_workspace_bytes(lib, m, n, k, int(kernel_id), int(p1), int(p2), int(p3)),
                            lib.mlk_gemm_counter_bytes())
        if ws is None:
            p3 = 1
        else:
            ws_bytes = ws.numel()
    _lib.check(lib.mlk_gemm_layout_a(_ptr(A), _ptr(B), _ptr(C), n, m, k, a_kind, _KIND[B.dtype], b_mode, c_mode,
                                     float(alpha), _ptr(bias), _ptr(A_Scale), int(kernel_id), int(p1), int(p2),
                                     int(p3), _ptr(ws), ws_bytes, _stream()), what)
    return C


def _off_panels(kid, addresses):
    """Whether operands that do not lie on 16 bytes keep a launch off the eight-wave panels it names."""
    return kid == 8 and addresses & 15 != 0


def _on16(A, B, n):
    """A copy of activations off 16 bytes, where the panels are worth it: above 64 tokens (copy and panels against the kernels that take any
    address: bf16 4096 x 4096 at 100 tokens 19 against 24.5 us, soft-FP8 13824 x 5120 at 1000 tokens 146 against 215 us).  None for fewer
    tokens, for weights off 16 bytes, and where there is no room."""
    if n <= 64 or A.data_ptr() & 15:
        return None
    try:
        return B.clone()
    except torch.OutOfMemoryError:
        return None


def _off16_plan(m, n, k, a_kind, b_mode, c_mode):
    """Launch parameters and workspace bytes for such operands."""
    key = ("off 16 bytes", m, n, k, a_kind, b_mode, c_mode)
    plan = _plans.get(key)
    if plan is None:
        lib, out = _lib.load(), (ctypes.c_int32 * 4)()
        _lib.check(lib.mlk_gemm_plan_off16(n, m, k, a_kind, b_mode, c_mode, out), "gemm")
        plan = _plans[key] = (*out, lib.mlk_gemm_workspace_bytes(n, m, out[1], out[3]))
    return plan


def _gemm_workspace_bytes(lib, m, n, k, kid, p1, p2, p3):
    if kid == 8:
        return lib.mlk_gemm_panel_workspace_bytes(n, m, k, p1, p2, p3)
    return lib.mlk_gemm_workspace_bytes(n, m, p1, p3)


def _gemm_guard(args, m):
    kid, p1, p2, p3 = args
    if kid == 8:
        return args if p1 in (2, 4) and p2 in (1, 2, 3, 4) and 1 <= p3 <= 64 else (1, 1, 4, 1)
    if kid not in (1, 2, 3, 4, 5, 12, 14, 16, 18) or p1 not in (1, 2, 4, 8) or \
            (kid not in (3, 5) and (m // 16) % p1 != 0) or \
            p2 not in (1, 2, 4, 8, 16) or p3 < 1:
        return (1, 1, 4, 1)
    return args


def _gemm_args(table, m, n, k, a_kind, b_mode=_B_ROWMAJOR):
    """Launch parameters of a table-driven GeMM call: the table's row of this very shape; else the row of a nearby token count (up to
    64 tokens, or above); else what the library expects to be fastest (`mlk_gemm_plan_placed`: a fitted cost of every launch it considers),
    else what the selector makes of it.  The packaged tables hold no rows above 64 tokens: on 24 weight shapes at 14 token counts from 65 to
    3000 the eight-wave panels were 1.29 (bf16) to 1.40 (soft-FP8) times as fast as the rows that had been scanned for the older panel
    kernels (geometric mean), and in native layouts, where those do not run, up to fifteen times.  Weight shapes outside the tables
    at up to 64 tokens: 1.37 times the fixed launch parameters they had."""
    def plan():
        out = (ctypes.c_int32 * 4)()
        if k % 128 or n * k >= 1 << 31 or _lib.load().mlk_gemm_plan_placed(n, m, k, a_kind, b_mode, out) != 0:
            return None
        return tuple(out)
    return _gemm_guard(arg_selector.selector(table).get_args((m, n, k), plan), m)


def _gemm_eager(tag, table, checked, A, A_Scale, B, alpha, beta, bias, b_mode, c_mode):
    """The table-driven GeMM entry points behind their launch plans (see `_plans`): `checked` is the function that
    runs every argument check, the table lookup and the launch for a combination not seen before."""
    key = (tag, A.shape, B.shape, A.dtype, B.dtype, A.device, B.device,
           None if A_Scale is None else (A_Scale.shape, A_Scale.dtype, A_Scale.device),
           None if bias is None else (bias.shape, bias.dtype, bias.device))
    plan = _plans.get(key)
    if plan is not None and beta == 0 and A.is_contiguous() and B.is_contiguous() and \
            (A_Scale is None or A_Scale.is_contiguous()) and (bias is None or bias.is_contiguous()):
        m, n, k, a_kind, x_kind, kid, p1, p2, p3, ws_need, counter_bytes, use_scale, c_shape, fn = plan
        C = torch.empty(c_shape, dtype=B.dtype, device=B.device)
        stream = _stream_of(B)
        a_ptr, b_ptr = A.data_ptr(), B.data_ptr()
        if _off_panels(kid, a_ptr | b_ptr):
            copy = _on16(A, B, n)
            if copy is not None:
                b_ptr = copy.data_ptr()
            else:
                kid, p1, p2, p3, ws_need = _off16_plan(m, n, k, a_kind, b_mode, c_mode)
        ws_ptr = ws_len = 0
        if p3 > 1:
            ws = _split_scratch(B.device, stream, ws_need, counter_bytes)
            if ws is None:
                p3 = 1
            else:
                ws_ptr, ws_len = ws.data_ptr(), ws.numel()
        rc = fn(a_ptr, b_ptr, C.data_ptr(), n, m, k, a_kind, x_kind, b_mode, c_mode, float(alpha),
                0 if bias is None else bias.data_ptr(), A_Scale.data_ptr() if use_scale else 0, kid, p1, p2, p3,
                ws_ptr, ws_len, stream)
        if rc != 0:
            _lib.check(rc, tag)
        return C
    C = checked()
    lib = _lib.load()
    m, k = A.size(0) * 16, A.size(1) * 8
    n = B.size(0) if b_mode == _B_ROWMAJOR else B.size(1) * 16
    kid, p1, p2, p3 = _gemm_args(table, m, n, k, _kind(A), b_mode)
    _plans[key] = (m, n, k, _kind(A), _KIND[B.dtype], kid, p1, p2, p3,
                   _gemm_workspace_bytes(lib, m, n, k, kid, p1, p2, p3) if p3 > 1 else 0, lib.mlk_gemm_counter_bytes(),
                   _is_fp8(A) and A_Scale is not None, tuple(C.shape), lib.mlk_gemm_layout_a)
    return C


def gemm_layoutA_wapper(A, B, m, n, k, alpha=1, beta=0, kernelParam1=1, kernelParam2=1, kernelParam3=1, kernelId=1,
                        bias=None):
    """csrc/gemm_layout_A.cu:684-750 with explicit launch parameters."""
    return _gemm_call(A, None, B, m, n, k, alpha, beta, bias, _B_ROWMAJOR, _C_ROWMAJOR, kernelId, kernelParam1,
                      kernelParam2, kernelParam3, "gemm_layoutA")


def _check_gemm_common(A, B):
    _check(A.is_cuda, "A must be a CUDA tensor")
    _check(B.is_cuda, "B must be a CUDA tensor")
    _check(A.is_contiguous(), "A must be contiguous")
    _check(B.is_contiguous(), "B must be contiguous")


def gemm_layoutA(A, B, alpha=1, beta=0, bias=None):
    """C[n, m] = alpha * B[n, k] . A^T (+ bias); A layout-A, B and C row-major
    (csrc/gemm_layout_A.cu:752-787)."""
    return _gemm_eager("gemm_layoutA", "layoutA_gemm", lambda: _gemm_layoutA_checked(A, B, alpha, beta, bias), A, None, B, alpha, beta, bias,
                       _B_ROWMAJOR, _C_ROWMAJOR)


def _gemm_layoutA_checked(A, B, alpha=1, beta=0, bias=None):
    """Every argument check of the reference's host launcher, the table lookup, the launch."""
    _check_gemm_common(A, B)
    m, a_k = _layout_a_dims(A)
    _check(B.dim() == 2, "B must be a 2D tensor")
    n, b_k = B.size(0), B.size(1)
    _check(a_k == b_k, "A and B must have the same k")
    k = a_k
    _check(m % 128 == 0, "GEMM m % 128 == 0, currently, will be revised soon")
    _check(k % 128 == 0, "GEMM k % 128 must be 0")
    kid, p1, p2, p3 = _gemm_args("layoutA_gemm", m, n, k, _kind(A), _B_ROWMAJOR)
    return gemm_layoutA_wapper(A, B, m, n, k, alpha, beta, p1, p2, p3, kid, bias)


def gemm_layoutA_soft_fp8_wapper(A, A_Scale, B, m, n, k, alpha=1, beta=0, kernelParam1=1, kernelParam2=1,
                                 kernelParam3=1, kernelId=1, bias=None):
    """csrc/gemm_layout_A_soft_fp8.cu:749-823 with explicit launch parameters."""
    _check(_is_fp8(A), "A must hold one e4m3 byte per element")
    return _gemm_call(A, A_Scale, B, m, n, k, alpha, beta, bias, _B_ROWMAJOR, _C_ROWMAJOR, kernelId, kernelParam1,
                      kernelParam2, kernelParam3, "gemm_layoutA_soft_fp8")


def gemm_layoutA_soft_fp8(A, A_Scale, B, alpha=1, beta=0, bias=None):
    """Soft-FP8 weights (e4m3 bytes in layout-A + fp32 scale per 128x128 block), bf16
    activations (csrc/gemm_layout_A_soft_fp8.cu:825-862)."""
    return _gemm_eager("gemm_layoutA_soft_fp8", "layoutA_soft_fp8_gemm", lambda: _gemm_layoutA_soft_fp8_checked(A, A_Scale, B, alpha, beta, bias), A, A_Scale, B, alpha,
                       beta, bias, _B_ROWMAJOR, _C_ROWMAJOR)


def _gemm_layoutA_soft_fp8_checked(A, A_Scale, B, alpha=1, beta=0, bias=None):
    """Every argument check of the reference's host launcher, the table lookup, the launch."""
    _check_gemm_common(A, B)
    m, a_k = _layout_a_dims(A)
    _check(B.dim() == 2, "B must be a 2D tensor")
    n, b_k = B.size(0), B.size(1)
    _check(a_k == b_k, "A and B must have the same k")
    k = a_k
    _check(m % 128 == 0, "GEMM m % 128 == 0, currently, will be revised soon")
    _check(k % 128 == 0, "GEMM k % 128 must be 0")
    _check(B.dtype == torch.bfloat16, "soft-FP8 weights need bf16 activations")
    kid, p1, p2, p3 = _gemm_args("layoutA_soft_fp8_gemm", m, n, k, _kind(A), _B_ROWMAJOR)
    return gemm_layoutA_soft_fp8_wapper(A, A_Scale, B, m, n, k, alpha, beta, p1, p2, p3, kid, bias)


def gemm_layoutA_linear(A, B, alpha=1, beta=0, scale_matrix=None, bias=None):
    """Route on the presence of a scale matrix (csrc/gemm_layoutA_linear.cu:9-18)."""
    if scale_matrix is not None:
        return gemm_layoutA_soft_fp8(A, scale_matrix, B, alpha, beta, bias)
    return gemm_layoutA(A, B, alpha, beta, bias)


def _native_b_dims(B):
    _check(B.dim() == 5, "B must be a 5D tensor")
    _check(B.size(2) == 4, "B.shape[2] must be 4")
    _check(B.size(3) == 16, "B.shape[3] must be 16")
    _check(B.size(4) == 8, "B.shape[4] must be 8")
    return B.size(1) * 16, B.size(0) * 32


def gemm_layoutAB_ContinuousC_wapper(A, B, m, n, k, alpha=1, beta=0, kernelParam1=1, kernelParam2=1, kernelParam3=1,
                                     kernelId=1, bias=None):
    """csrc/gemm_layout_ab_continuous_c.cu with explicit launch parameters."""
    return _gemm_call(A, None, B, m, n, k, alpha, beta, bias, _B_NATIVE, _C_ROWMAJOR, kernelId, kernelParam1,
                      kernelParam2, kernelParam3, "gemm_layoutAB_ContinuousC")


def gemm_layoutAB_ContinuousC(A, B, alpha=1, beta=0, bias=None):
    """A layout-A, B layout-B, C row-major [n, m] (csrc/gemm_layout_ab_continuous_c.cu:1051-1093)."""
    return _gemm_eager("gemm_layoutAB_ContinuousC", "continuous_gemm", lambda: _gemm_layoutAB_ContinuousC_checked(A, B, alpha, beta, bias), A, None, B, alpha, beta, bias,
                       _B_NATIVE, _C_ROWMAJOR)


def _gemm_layoutAB_ContinuousC_checked(A, B, alpha=1, beta=0, bias=None):
    """Every argument check of the reference's host launcher, the table lookup, the launch."""
    _check_gemm_common(A, B)
    m, a_k = _layout_a_dims(A)
    n, b_k = _native_b_dims(B)
    _check(a_k == b_k, "A and B must have the same k")
    k = a_k
    _check(m % 128 == 0, "GEMM m % 128 == 0, currently, will be revised soon")
    _check(k % 128 == 0, "GEMM k % 128 must be 0")
    kid, p1, p2, p3 = _gemm_args("continuous_gemm", m, n, k, _kind(A), _B_NATIVE)
    return gemm_layoutAB_ContinuousC_wapper(A, B, m, n, k, alpha, beta, p1, p2, p3, kid, bias)


def gemm_layoutABC_wapper(A, B, m, n, k, alpha=1, beta=0, kernelParam1=1, kernelParam2=1, kernelParam3=1,
                          kernelId=1, bias=None):
    """csrc/gemm_layout_abc.cu with explicit launch parameters."""
    return _gemm_call(A, None, B, m, n, k, alpha, beta, bias, _B_NATIVE, _C_NATIVE, kernelId, kernelParam1,
                      kernelParam2, kernelParam3, "gemm_layoutABC")


def gemm_layoutABC(A, B, alpha=1, beta=0, bias=None):
    """A layout-A, B layout-B, C layout-C [m/32, n/16, 4, 16, 8], ready to be the B of the
    next product (csrc/gemm_layout_abc.cu:754-791)."""
    return _gemm_eager("gemm_layoutABC", "layout_gemm", lambda: _gemm_layoutABC_checked(A, B, alpha, beta, bias), A, None, B, alpha, beta, bias,
                       _B_NATIVE, _C_NATIVE)


def _gemm_layoutABC_checked(A, B, alpha=1, beta=0, bias=None):
    """Every argument check of the reference's host launcher, the table lookup, the launch."""
    _check_gemm_common(A, B)
    m, a_k = _layout_a_dims(A)
    n, b_k = _native_b_dims(B)
    _check(a_k == b_k, "A and B must have the same k")
    k = a_k
    _check(m % 128 == 0, "GEMM m % 128 == 0, currently, will be revised soon")
    _check(k % 128 == 0, "GEMM k % 128 must be 0")
    kid, p1, p2, p3 = _gemm_args("layout_gemm", m, n, k, _kind(A), _B_NATIVE)
    return gemm_layoutABC_wapper(A, B, m, n, k, alpha, beta, p1, p2, p3, kid, bias)


# ------------------------------------------------------------- 4-bit weights
class _OnDevice:
    """The library launches on the current device: makes the tensor's device current for the call where it is another one."""

    def __init__(self, t):
        self.guard = torch.cuda.device(t.device) if t.device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _check_tensors(named, device):
    for t, name in named:
        if t is not None:
            _check(t.is_cuda, "%s must be a CUDA tensor" % name)
            _check(t.device == device, "%s must be on the same device as the others" % name)
            _check(t.is_contiguous(), "%s must be contiguous" % name)


def pack_layout_a_w4(codes, scales, zeros=None):
    """4-bit weights W = s (q - z), row-major, to the layout of `gemm_layoutA_w4` and `fused_experts_w4`.

    codes  uint8 [N, K/2] or [E, N, K/2], two codes 0..15 in a byte, element 2 i in the low half of byte i
    scales fp16 / bf16 [.., N, K/G], one for G consecutive weights of a row; G = 32, 64 or a multiple of 128
    zeros  uint8 [.., N, K/G], 0..15, or None: 8 everywhere.  Larger ones, which the kernels would not take alike, are refused: the call waits for the device
           to look at them, so with zeros it cannot be recorded into a graph
    Returns (A [.., N/16, K/128, 64, 16] uint8, scale and zero [.., N/16, K/max(G,128), 16, max(1,128/G)])."""
    _check(codes.dtype == torch.uint8 and codes.dim() in (2, 3), "codes must be uint8 [N, K/2] or [E, N, K/2]")
    _check(scales.dtype in _KIND, "scales must be fp16 or bf16")
    _check(zeros is None or zeros.dtype == torch.uint8, "zeros must be uint8")
    n, k = codes.shape[-2], codes.shape[-1] * 2
    lead = tuple(codes.shape[:-2])
    _check(n % 16 == 0 and k % 128 == 0 and n > 0 and k > 0, "N % 16 and K % 128 must be 0")
    _check(scales.dim() == codes.dim() and tuple(scales.shape[:-1]) == lead + (n,), "scales must be [.., N, K/G]")
    groups = scales.shape[-1]
    _check(groups > 0 and k % groups == 0, "scales must be [.., N, K/G]")
    group = k // groups
    _check(group in (32, 64) or group % 128 == 0, "the group must be 32, 64 or a multiple of 128")
    _check(zeros is None or zeros.shape == scales.shape, "zeros must have the shape of scales")
    _check(zeros is None or zeros.numel() == 0 or int(zeros.max()) <= 15, "zeros must be 0..15")
    _check_tensors(((codes, "codes"), (scales, "scales"), (zeros, "zeros")), codes.device)
    batch = codes.shape[0] if codes.dim() == 3 else 1
    per = max(1, 128 // group)
    lib, shape = _lib.load(), lead + (n // 16, groups // per, 16, per)
    with _OnDevice(codes):
        stream = _stream_of(codes)
        A = torch.empty(lead + (n // 16, k // 128, 64, 16), dtype=torch.uint8, device=codes.device)
        _lib.check(lib.mlk_pack_layout_a_w4(_ptr(codes), _ptr(A), batch, n, k, stream), "pack_layout_a_w4")
        out = []
        for t in (scales, zeros):
            p = None
            if t is not None:
                p = torch.empty(shape, dtype=t.dtype, device=t.device)
                _lib.check(lib.mlk_pack_scales_w4(_ptr(t), _ptr(p), batch, n, k, group, t.element_size(), stream), "pack_layout_a_w4")
            out.append(p)
    return A, out[0], out[1]


def unpack_layout_a_w4(A, A_Scale, A_Zero=None):
    """Inverse of `pack_layout_a_w4`: (codes [.., N, K/2], scales [.., N, K/G], zeros or None)."""
    n, k, group = _w4_dims(A, A_Scale, A_Zero, A.dim() - 4)
    _check_tensors(((A, "A"), (A_Scale, "A_Scale"), (A_Zero, "A_Zero")), A.device)
    lead = tuple(A.shape[:-4])
    batch = A.shape[0] if lead else 1
    lib = _lib.load()
    with _OnDevice(A):
        stream = _stream_of(A)
        codes = torch.empty(lead + (n, k // 2), dtype=torch.uint8, device=A.device)
        _lib.check(lib.mlk_unpack_layout_a_w4(_ptr(A), _ptr(codes), batch, n, k, stream), "unpack_layout_a_w4")
        out = []
        for t in (A_Scale, A_Zero):
            p = None
            if t is not None:
                p = torch.empty(lead + (n, k // group), dtype=t.dtype, device=t.device)
                _lib.check(lib.mlk_unpack_scales_w4(_ptr(t), _ptr(p), batch, n, k, group, t.element_size(), stream), "unpack_layout_a_w4")
            out.append(p)
    return codes, out[0], out[1]


def _w4_dims(A, scale, zero, lead, what="A"):
    """(N, K, group) of packed 4-bit weights with `lead` leading dimensions (0 or 1)."""
    _check(lead in (0, 1) and A.dim() == 4 + lead and A.dtype == torch.uint8 and tuple(A.shape[-2:]) == (64, 16),
           "%s must be uint8 [N/16, K/128, 64, 16] (pack_layout_a_w4)" % what)
    n, k = A.size(-4) * 16, A.size(-3) * 128
    _check(scale.dim() == A.dim() and scale.size(-2) == 16 and tuple(scale.shape[:-3]) == tuple(A.shape[:-3]) and scale.size(-3) > 0,
           "the scales of %s must be [N/16, K/max(G,128), 16, max(1,128/G)]" % what)
    blocks, per = scale.size(-3), scale.size(-1)
    _check((per in (2, 4) and blocks * 128 == k) or (per == 1 and k % (blocks * 128) == 0 and k > 0),
           "the scales of %s must be [N/16, K/max(G,128), 16, max(1,128/G)]" % what)
    _check(scale.dtype in _KIND, "the scales of %s must be fp16 or bf16" % what)
    _check(zero is None or (zero.dtype == torch.uint8 and zero.shape == scale.shape), "the zero points of %s must be uint8 of the scales' shape" % what)
    return n, k, 128 // per if per > 1 else k // blocks


def _w4_call(A, A_Scale, B, A_Zero, alpha, beta, bias, what):
    device = B.get_device()
    key = ("w4", A.shape, A_Scale.shape, B.shape, A.dtype, A_Scale.dtype, B.dtype, A.get_device(), A_Scale.get_device(), device,
           None if A_Zero is None else (A_Zero.shape, A_Zero.dtype, A_Zero.get_device()), None if bias is None else (bias.shape, bias.dtype, bias.get_device()))
    plan = _plans.get(key)
    if plan is None or beta != 0 or not (A.is_contiguous() and A_Scale.is_contiguous() and B.is_contiguous() and
                                         (A_Zero is None or A_Zero.is_contiguous()) and (bias is None or bias.is_contiguous())):
        _check_beta(beta)
        m, k, group = _w4_dims(A, A_Scale, A_Zero, 0)
        _check(B.dim() == 2, "B must be a 2D tensor")
        _check(B.size(1) == k, "A and B must have the same k")
        _check(B.dtype in _KIND, "Unsupported data type")
        _check(A_Scale.dtype == B.dtype, "A_Scale must have the activation dtype")
        _check(bias is None or (bias.dtype == B.dtype and bias.numel() == m), "bias must be [1, m] of the activation dtype")
        _check_tensors(((A, "A"), (A_Scale, "A_Scale"), (B, "B"), (A_Zero, "A_Zero"), (bias, "bias")), B.device)
        lib = _lib.load()
        plan = _plans[key] = (B.size(0), m, k, group, _KIND[B.dtype], lib.mlk_gemm_w4_workspace_bytes(B.size(0), m, k, group),
                              lib.mlk_gemm_counter_bytes(), lib.mlk_gemm_layout_a_w4)
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _w4_launch(plan, A, A_Scale, B, A_Zero, alpha, bias, what)
    return _w4_launch(plan, A, A_Scale, B, A_Zero, alpha, bias, what)


def _w4_launch(plan, A, A_Scale, B, A_Zero, alpha, bias, what):
    n, m, k, group, kind, ws_need, counter_bytes, fn = plan
    b_ptr = B.data_ptr()
    if b_ptr & 15:
        B = B.clone()
        b_ptr = B.data_ptr()
    C = B.new_empty((n, m))
    stream = _stream_of(B)
    ws_ptr = ws_len = 0
    if ws_need:
        ws = _gemm_pool.get(B.device, stream, ws_need, counter_bytes)
        ws_ptr, ws_len = ws.data_ptr(), ws.numel()
    rc = fn(A.data_ptr(), A_Scale.data_ptr(), _ptr(A_Zero), b_ptr, C.data_ptr(), n, m, k, group, kind, float(alpha), _ptr(bias), ws_ptr, ws_len, stream)
    if rc != 0:
        _lib.check(rc, what)
    return C


def gemm_layoutA_w4(A, A_Scale, B, A_Zero=None, alpha=1, beta=0, bias=None):
    """C[n, m] = alpha * B[n, k] . W^T (+ bias) with 4-bit weights W = s (q - z) from `pack_layout_a_w4`; any n >= 0, m % 16 == 0,
    k % 128 == 0.  fp32 sums, one rounding at the end, no weight rounded.  A row of B that holds an infinity, or bf16 numbers so large that 64
    times the sum of their magnitudes passes the fp32 range, gives NaN.  No gradient: the result is detached."""
    return _w4_call(A, A_Scale, B, A_Zero, alpha, beta, bias, "gemm_layoutA_w4")


def gemv_layoutA_w4(A, A_Scale, B, A_Zero=None, alpha=1, beta=0, bias=None):
    """The same for one token: B [1, k]."""
    _check(B.dim() == 2 and B.size(0) == 1, "B must be a vector")
    return _w4_call(A, A_Scale, B, A_Zero, alpha, beta, bias, "gemv_layoutA_w4")


# ----------------------------------------------------------------------- MoE
def _check_gating_bias(bias, gating_output):
    """The router reads one element for every expert."""
    if bias is not None:
        _check(bias.dtype == gating_output.dtype, "Mismatched dtypes: load_balance_bias and gating_output.")
        _check(bias.numel() >= gating_output.size(-1), "load_balance_bias must have an element for every expert")
        _check(bias.device == gating_output.device and bias.is_contiguous(), "load_balance_bias must be contiguous and on gating_output's device")


def fused_routing_gate(gating_output, score_fun, batch_size, hidden_size, n_groups, topK_groups, experts_ids,
                       selected_experts_weights, topK, load_balance_bias=None, renormalize=False):
    """Router: writes `experts_ids` (int32 [T, K]) and `selected_experts_weights` ([T, K]) in place and
    returns None (csrc/moe_kernels/fused_gating.cu:5-67).  `renormalize` is an extension: the reference
    leaves the division to its Python caller (muxi_moe_planC.py:69-70)."""
    _check(gating_output.dtype == selected_experts_weights.dtype,
           "Mismatched dtypes: gating_output and selected_experts_weights.")
    _check_gating_bias(load_balance_bias, gating_output)
    _check(gating_output.dtype in _KIND, "Invalid dtype for gating_output: must be kFloat16 or kBFloat16.")
    _check(experts_ids.dtype == torch.int32, "Invalid dtype for experts_ids: must be kInt32.")
    _check(experts_ids.device == selected_experts_weights.device,
           "Device mismatch: experts_ids and selected_experts_weights.")
    _check(gating_output.is_cuda and gating_output.is_contiguous(), "gating_output must be a contiguous CUDA tensor")
    n_experts = gating_output.size(-1)
    _check(int(batch_size) * n_experts == gating_output.numel(), "batch_size does not match gating_output")
    _check(1 <= n_experts <= 256, "the router supports at most 256 experts")
    _check(n_groups >= 1 and n_experts % n_groups == 0, "n_groups must divide the number of experts")
    _check(1 <= topK_groups <= n_groups, "topK_groups must be in 1..n_groups")
    _check(1 <= topK <= min(32, n_experts), "topK must be in 1..min(32, experts)")
    _check(experts_ids.numel() >= batch_size * topK and selected_experts_weights.numel() >= batch_size * topK,
           "output tensors are too small")
    _lib.check(_lib.load().mlk_fused_routing_gate(_ptr(gating_output), _KIND[gating_output.dtype], int(score_fun),
                                                  int(batch_size), n_experts, int(n_groups), int(topK_groups),
                                                  int(topK), _ptr(load_balance_bias), int(bool(renormalize)),
                                                  _ptr(experts_ids), _ptr(selected_experts_weights), _stream()),
               "fused_routing_gate")
    return None


def batched_routed_activation_indexed_to_expert_block_indexed(batchSize, expertCount, topK, microBatchSize,
                                                              expertsIds, dev_sorted_token_ids, dev_cumsum_buffer,
                                                              dev_padded_num_experts, dev_experts_ids,
                                                              experts_map=None):
    """Token -> expert-block permutation (csrc/moe_kernels/fused_experts_compute.cu:6-48)."""
    _check(expertsIds.dtype == torch.int32, "expertsIds must be of type torch::kInt32.")
    for t, name in ((dev_sorted_token_ids, "dev_sorted_token_ids"), (dev_cumsum_buffer, "dev_cumsum_buffer"),
                    (dev_padded_num_experts, "dev_padded_num_experts"), (dev_experts_ids, "dev_experts_ids")):
        _check(expertsIds.device == t.device, "expertsIds must be on the same device as %s." % name)
        _check(t.dtype == torch.int32, "%s must be int32" % name)
    _check(microBatchSize == 16, "microBatchSize must be 16")
    _check(1 <= expertCount <= 1024, "expertCount must be in 1..1024")
    n_pairs = int(batchSize) * int(topK)
    _check(expertsIds.numel() >= n_pairs, "expertsIds is too small")
    padded = n_pairs + expertCount * (microBatchSize - 1)
    _check(dev_sorted_token_ids.numel() >= padded, "dev_sorted_token_ids is too small")
    _check(dev_cumsum_buffer.numel() >= expertCount + 1, "dev_cumsum_buffer is too small")
    _check(dev_experts_ids.numel() >= (padded + microBatchSize - 1) // microBatchSize, "dev_experts_ids is too small")
    if experts_map is not None:
        _check(experts_map.dtype == torch.int32, "experts_map must be int32")
    _lib.check(_lib.load().mlk_moe_align_tokens(_ptr(expertsIds), n_pairs, int(expertCount), int(microBatchSize),
                                                _ptr(experts_map), _ptr(dev_sorted_token_ids),
                                                _ptr(dev_cumsum_buffer), _ptr(dev_padded_num_experts),
                                                _ptr(dev_experts_ids), _stream()), "moe_align_tokens")
    return None


def _moe_workspace(device, nbytes, stream=None):
    return _moe_pool.get(device, _stream() if stream is None else stream, nbytes)


def _moe_scratch(device, T, E, K, hidden, inter):
    """Scratch for T tokens: that of the wide kernels, or, where the card has no room for it, that of passes of 256 tokens
    (8 experts, H 4096, I 14336 at 4096 tokens: 487 and 63 MiB), in which the call then runs."""
    lib = _lib.load()
    try:
        return _moe_workspace(device, lib.mlk_moe_wide_workspace_bytes(T, E, K, hidden, inter))
    except torch.OutOfMemoryError:
        if T <= 256:
            raise
        return _moe_workspace(device, lib.mlk_moe_workspace_bytes(T, E, K, hidden, inter))


def fused_experts_compute(experts_weights_matrix1, experts_weights_matrix2, activations, batch_size, expert_count,
                          dynamic_experts_per_act, topk_ids, actived_experts_weights, sorted_token_ids, cumsum_buffer,
                          padded_num_experts, experts_ids, C, y, *args, **kwargs):
    """Both overloads of the reference's `fused_experts_compute` (ffi.cu:112-143):

    16-bit weights: (..., APerWarp=2, splitK=3, tile_m_2=128, tile_n_2=16, tile_k_2=128, block_dim_x_gemm=256,
                     microBatchSize=16, experts_map=None)
    soft-FP8:       (..., w1_scale, w2_scale, block_shape, soft_fp8=False, microBatchSize=16, experts_map=None)

    The overload is chosen as pybind does, from the type of the first extra argument.  Runs the alignment,
    the grouped gate/up GeMM with SiLU*up, the grouped down GeMM and the weighted sum into `y`.  `C` (the
    reference's intermediate buffer) is accepted and left untouched: the intermediate lives in a cached
    workspace in a layout the second GeMM can stream.  The MetaX tile parameters are accepted and ignored."""
    w1, w2, x = experts_weights_matrix1, experts_weights_matrix2, activations
    fp8 = (len(args) > 0 and isinstance(args[0], torch.Tensor)) or "w1_scale" in kwargs
    if fp8:
        names = ["w1_scale", "w2_scale", "block_shape", "soft_fp8", "microBatchSize", "experts_map"]
        defaults = {"soft_fp8": False, "microBatchSize": 16, "experts_map": None}
    else:
        names = ["APerWarp", "splitK", "tile_m_2", "tile_n_2", "tile_k_2", "block_dim_x_gemm", "microBatchSize",
                 "experts_map"]
        defaults = {"APerWarp": 2, "splitK": 3, "tile_m_2": 128, "tile_n_2": 16, "tile_k_2": 128,
                    "block_dim_x_gemm": 256, "microBatchSize": 16, "experts_map": None}
    _check(len(args) <= len(names), "fused_experts_compute: too many positional arguments")
    opts = dict(defaults)
    for name, val in zip(names, args):
        opts[name] = val
    for name, val in kwargs.items():
        _check(name in names and name not in names[:len(args)], "fused_experts_compute: unexpected argument %s" % name)
        opts[name] = val
    for name in names:
        _check(name in opts, "fused_experts_compute: missing argument %s" % name)

    _check(w1.dtype == w2.dtype, "experts_weights_matrix1 and experts_weights_matrix2 must have the same dtype.")
    _check(topk_ids.dtype == torch.int32, "expertsIds must be of type torch::kInt32.")
    _check(x.dtype == actived_experts_weights.dtype, "activations and activedExpertsWeights must have the same dtype.")
    _check(x.dtype == y.dtype, "activations and y must have the same dtype.")
    _check(x.dtype in _KIND, "activations must be fp16 or bf16")
    for t in (w1, w2, x, topk_ids, actived_experts_weights, sorted_token_ids, cumsum_buffer, padded_num_experts,
              experts_ids, y):
        _check(t.is_cuda and t.is_contiguous(), "all tensors must be contiguous CUDA tensors")
    w1_scale = w2_scale = None
    if fp8:
        _check(w1.element_size() == 1, "experts weights must be float8_e4m3fn bytes for the soft-FP8 overload.")
        w1_scale, w2_scale = opts["w1_scale"], opts["w2_scale"]
        _check(w1_scale.dtype == torch.float32 and w2_scale.dtype == torch.float32, "scales must be float32.")
        _check(w1_scale.device == w2_scale.device, "w1_scale and w2_scale must be on the same device.")
        block_shape = list(opts["block_shape"])
        _check(len(block_shape) == 2, "block_shape must have size 2.")
        _check(block_shape[0] == 128 and block_shape[1] == 128, "block_shape must be (128, 128) for float8_e4m3fn.")
        _check(bool(opts["soft_fp8"]), "soft_fp8 must be true for float8_e4m3fn.")
        _check(x.dtype == torch.bfloat16, "Weight date type and activation date type mismatch")
        w_kind = _FP8_KIND
    else:
        _check(w1.dtype == x.dtype, "Weight date type and activation date type mismatch")
        w_kind = _KIND[w1.dtype]
    _check(opts["microBatchSize"] == 16, "microBatchSize must be 16")
    # per-expert slabs: either the flattened [E, 2I, H] view the reference's tests pass or [E, 2I/16, H/8, 16, 8]
    if w1.dim() == 5:
        e1, m1, k1 = w1.shape[0], w1.shape[1] * 16, w1.shape[2] * 8
        e2, m2, k2 = w2.shape[0], w2.shape[1] * 16, w2.shape[2] * 8
    else:
        _check(w1.dim() == 3 and w2.dim() == 3, "expert weights must be [E, rows, cols]")
        e1, m1, k1 = w1.shape
        e2, m2, k2 = w2.shape
    _check(e1 == e2 == expert_count, "expert count mismatch")
    _check(k1 == m2 and m1 == 2 * k2, "w1 must be [E, 2I, H] and w2 [E, H, I]")
    hidden, inter = k1, k2
    _check(hidden % 128 == 0 and inter % 128 == 0, "hidden and intermediate sizes must be multiples of 128")
    T, K = int(batch_size), int(dynamic_experts_per_act)
    _check(x.numel() == T * hidden and y.numel() == T * hidden, "activations / y must be [batch, hidden]")
    if fp8:
        _check(tuple(w1_scale.shape) == (e1, m1 // 128, k1 // 128) and w1_scale.is_contiguous(),
               "w1_scale must be [E, 2I/128, H/128]")
        _check(tuple(w2_scale.shape) == (e2, m2 // 128, k2 // 128) and w2_scale.is_contiguous(),
               "w2_scale must be [E, H/128, I/128]")
    experts_map = opts["experts_map"]
    if experts_map is not None:
        _check(experts_map.dtype == torch.int32 and experts_map.is_cuda, "experts_map must be an int32 CUDA tensor")
    # the reference fills the caller's alignment buffers as a side effect of this call
    batched_routed_activation_indexed_to_expert_block_indexed(T, e1, K, 16, topk_ids, sorted_token_ids, cumsum_buffer,
                                                              padded_num_experts, experts_ids, experts_map)
    experts_compute_raw(w1, w2, x, T, e1, K, hidden, inter, w_kind, topk_ids, actived_experts_weights, experts_map,
                        w1_scale, w2_scale, y)
    return None


def experts_compute_raw(w1, w2, x, T, E, K, hidden, inter, w_kind, topk_ids, topk_weights, experts_map, w1_scale,
                        w2_scale, y):
    """Thin call of the C entry point (alignment + both grouped GeMMs + weighted sum); no checks."""
    lib = _lib.load()
    ws = _moe_scratch(x.device, T, E, K, hidden, inter)
    _lib.check(lib.mlk_fused_experts_compute(_ptr(w1), _ptr(w2), _ptr(x), T, E, K, hidden, inter, w_kind,
                                             _KIND[x.dtype], _ptr(topk_ids), _ptr(topk_weights), _ptr(experts_map),
                                             _ptr(w1_scale), _ptr(w2_scale), _ptr(y), _ptr(ws), ws.numel(),
                                             _stream()), "fused_experts_compute")


def fused_moe_raw(w1, w2, x, logits, T, E, K, hidden, inter, w_kind, score_fun, n_groups, topk_groups, bias,
                  renormalize, experts_map, w1_scale, w2_scale, topk_ids, topk_weights, y):
    """Thin call of the whole-layer entry point (router + alignment + both grouped GeMMs + weighted sum); no
    checks.  `topk_ids` / `topk_weights` receive the routing."""
    lib = _lib.load()
    ws = _moe_scratch(x.device, T, E, K, hidden, inter)
    _lib.check(lib.mlk_fused_moe(_ptr(w1), _ptr(w2), _ptr(x), _ptr(logits), T, logits.size(-1), E, K, hidden, inter,
                                 w_kind, _KIND[x.dtype], score_fun, n_groups, topk_groups, _ptr(bias),
                                 int(bool(renormalize)), _ptr(experts_map), _ptr(w1_scale), _ptr(w2_scale),
                                 _ptr(topk_ids), _ptr(topk_weights), _ptr(y), _ptr(ws), ws.numel(), _stream()),
               "fused_moe")


def fused_experts_w4(hidden_states, w1, w2, topk_ids, topk_weights, w1_scale, w2_scale, w1_zero=None, w2_zero=None, experts_map=None):
    """The two products of an expert layer over 4-bit weights, from a routing decision (`fused_routing_gate`, or a caller's own).

    hidden_states [T, H] fp16 / bf16; w1 [E, 2I/16, H/128, 64, 16] (gate rows, then up rows), w2 [E, H/16, I/128, 64, 16], their scales and zero
    points from `pack_layout_a_w4`; topk_ids int32 [T, K], topk_weights [T, K] of the activation dtype; experts_map int32 [experts of
    the router]: the expert's place in w1 / w2, -1 = on another card.  Ids outside the router's experts are dropped too; a token without an expert here
    gets zeros.  Returns y [T, H].  fp32 sums; the SiLU intermediate is rounded to the activation dtype, which the second product's matrix
    instructions take, as in `fused_moe`.  A token with an infinity, or whose intermediate passes the range of that type (fp16: 65504), gives a row of NaN; other rows keep theirs.
    No gradient: the result is detached."""
    plan = _experts_w4_plan(hidden_states, w1, w2, topk_ids, topk_weights, w1_scale, w2_scale, w1_zero, w2_zero, experts_map)
    return _experts_w4_launch(plan, hidden_states, w1, w2, topk_ids, topk_weights, w1_scale, w2_scale, w1_zero, w2_zero, experts_map)


def _check_experts_w4_aligned(w1, w2, w1_scale, w2_scale, w1_zero, w2_zero):
    """What the library would say of them, for a caller that launches something ahead of it."""
    _check(((w1.data_ptr() | w2.data_ptr()) & 15) == 0, "w1 and w2 must lie on 16 bytes")
    _check(((w1_scale.data_ptr() | w2_scale.data_ptr()) & 7) == 0, "scales must lie on 8 bytes")
    _check(((_ptr(w1_zero) | _ptr(w2_zero)) & 3) == 0, "zero points must lie on 4 bytes")


def _experts_w4_plan(x, w1, w2, topk_ids, topk_weights, w1_scale, w2_scale, w1_zero, w2_zero, experts_map):
    key = ("experts_w4", x.shape, w1.shape, w2.shape, topk_ids.shape, topk_weights.shape, w1_scale.shape, w2_scale.shape, x.dtype, w1.dtype, w2.dtype,
           topk_ids.dtype, topk_weights.dtype, w1_scale.dtype, w2_scale.dtype, x.device, w1.device, w2.device, topk_ids.device, topk_weights.device,
           w1_scale.device, w2_scale.device,
           None if w1_zero is None else (w1_zero.shape, w1_zero.dtype, w1_zero.device),
           None if w2_zero is None else (w2_zero.shape, w2_zero.dtype, w2_zero.device),
           None if experts_map is None else (experts_map.shape, experts_map.dtype, experts_map.device))
    plan = _plans.get(key)
    if plan is None or not (x.is_contiguous() and w1.is_contiguous() and w2.is_contiguous() and topk_ids.is_contiguous() and topk_weights.is_contiguous() and
                            w1_scale.is_contiguous() and w2_scale.is_contiguous() and (w1_zero is None or w1_zero.is_contiguous()) and
                            (w2_zero is None or w2_zero.is_contiguous()) and (experts_map is None or experts_map.is_contiguous())):
        m1, hidden, group = _w4_dims(w1, w1_scale, w1_zero, 1, "w1")
        m2, inter, group2 = _w4_dims(w2, w2_scale, w2_zero, 1, "w2")
        E = w1.size(0)
        _check(w2.size(0) == E and m1 == 2 * inter and m2 == hidden, "w1 must be [E, 2I, H] and w2 [E, H, I]")
        _check(group == group2, "w1 and w2 must have the same group size")
        _check((w1_zero is None) == (w2_zero is None), "zero points for both w1 and w2 or for none")
        _check(inter % 128 == 0 and hidden % 128 == 0, "hidden and intermediate sizes must be multiples of 128")
        _check(max(hidden, inter) < 1 << 23, "hidden and intermediate sizes must be below 2^23")
        _check(1 <= E <= 256, "at most 256 experts")
        _check(x.dim() == 2 and x.size(1) == hidden, "hidden_states must be [T, H]")
        _check(x.dtype in _KIND, "hidden_states must be fp16 or bf16")
        _check(w1_scale.dtype == x.dtype and w2_scale.dtype == x.dtype, "scales must have the activation dtype")
        _check(topk_ids.dim() == 2 and topk_ids.size(0) == x.size(0) and topk_ids.dtype == torch.int32, "topk_ids must be int32 [T, K]")
        _check(topk_weights.shape == topk_ids.shape and topk_weights.dtype == x.dtype, "topk_weights must be [T, K] of the activation dtype")
        K = topk_ids.size(1)
        _check(1 <= K <= 32, "topK must be in 1..32")
        _check(experts_map is None or (experts_map.dtype == torch.int32 and experts_map.dim() == 1 and experts_map.numel() > 0),
               "experts_map must be int32 [experts of the router]")
        _check_tensors(((x, "hidden_states"), (w1, "w1"), (w2, "w2"), (topk_ids, "topk_ids"), (topk_weights, "topk_weights"), (w1_scale, "w1_scale"),
                     (w2_scale, "w2_scale"), (w1_zero, "w1_zero"), (w2_zero, "w2_zero"), (experts_map, "experts_map")), x.device)
        lib = _lib.load()
        E_router = E if experts_map is None else experts_map.numel()
        plan = _plans[key] = (x.size(0), E, E_router, K, hidden, inter, group, _KIND[x.dtype],
                              lib.mlk_experts_w4_workspace_bytes(x.size(0), E, E_router, K, hidden, inter, group), lib.mlk_fused_experts_w4)
    return plan


def _experts_w4_launch(plan, x, w1, w2, topk_ids, topk_weights, w1_scale, w2_scale, w1_zero, w2_zero, experts_map):
    T, E, E_router, K, hidden, inter, group, kind, ws_need, fn = plan
    with _OnDevice(x):
        if x.data_ptr() & 15:
            x = x.clone()
        y = torch.empty((T, hidden), dtype=x.dtype, device=x.device)
        if T == 0:
            return y
        stream = _stream_of(x)
        ws = _moe_pool.get(x.device, stream, ws_need)
        rc = fn(w1.data_ptr(), w1_scale.data_ptr(), _ptr(w1_zero), w2.data_ptr(), w2_scale.data_ptr(), _ptr(w2_zero), x.data_ptr(), T, E, E_router, K,
                hidden, inter, group, kind, topk_ids.data_ptr(), topk_weights.data_ptr(), _ptr(experts_map), y.data_ptr(), ws.data_ptr(), ws.numel(),
                stream)
        if rc != 0:
            _lib.check(rc, "fused_experts_w4")
    return y


# ------------------------------------------------------------- router balance
def _check_routing(experts_ids, token_mask, device):
    _check(experts_ids.dtype == torch.int32 and experts_ids.dim() == 2 and experts_ids.size(1) >= 1, "experts_ids must be int32 [T, K]")
    _check(token_mask is None or (token_mask.dtype in (torch.bool, torch.uint8) and token_mask.dim() == 1 and
                                  token_mask.size(0) == experts_ids.size(0)), "token_mask must be bool [T]")
    _check_tensors(((experts_ids, "experts_ids"), (token_mask, "token_mask")), device)


def expert_counts(experts_ids, n_experts, token_mask=None, out=None):
    """How many routed pairs each expert got: int32 [n_experts].  experts_ids int32 [T, K] (`fused_routing_gate`), ids outside 0..n_experts-1
    count nowhere; token_mask bool [T]: False for padded rows.  With `out` the counts are added to it, for a load that builds up over
    the steps of a server."""
    device = experts_ids.get_device()
    key = ("counts", n_experts, experts_ids.shape, experts_ids.dtype, device,
           None if token_mask is None else (token_mask.shape, token_mask.dtype, token_mask.get_device()),
           None if out is None else (out.shape, out.dtype, out.get_device()))
    plan = _plans.get(key)
    if plan is None or not (experts_ids.is_contiguous() and (token_mask is None or token_mask.is_contiguous()) and (out is None or out.is_contiguous())):
        _check_routing(experts_ids, token_mask, experts_ids.device)
        _check(1 <= n_experts <= 256, "1..256 experts")
        if out is not None:
            _check(out.dtype == torch.int32 and tuple(out.shape) == (n_experts,), "out must be int32 [n_experts]")
            _check_tensors(((out, "out"),), experts_ids.device)
        lib = _lib.load()
        ws_need = lib.mlk_balance_counter_bytes() if out is None and experts_ids.numel() > 4096 else 0
        plan = _plans[key] = (experts_ids.size(0), experts_ids.size(1), ws_need, lib.mlk_expert_counts)
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _counts_launch(plan, experts_ids, n_experts, token_mask, out)
    return _counts_launch(plan, experts_ids, n_experts, token_mask, out)


def _counts_launch(plan, experts_ids, n_experts, token_mask, out):
    n_tokens, topk, ws_need, fn = plan
    add, stream = out is not None, _stream_of(experts_ids)
    if not add:
        out = experts_ids.new_empty(n_experts)
    ws = _balance_pool.get(experts_ids.device, stream, ws_need, ws_need).data_ptr() if ws_need else 0
    rc = fn(experts_ids.data_ptr(), _ptr(token_mask), n_tokens, topk, n_experts, add, out.data_ptr(), ws, stream)
    if rc != 0:
        _lib.check(rc, "expert_counts")
    return out


_LOGIT_KIND = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 3}


def _balance_forward(logits, ids, mask, cu, score_fun, coef, plan):
    if logits.get_device() != torch.cuda.current_device():
        with torch.cuda.device(logits.device):
            return _balance_launch(logits, ids, mask, cu, score_fun, coef, plan)
    return _balance_launch(logits, ids, mask, cu, score_fun, coef, plan)


def _balance_launch(logits, ids, mask, cu, score_fun, coef, plan):
    T, E, K, kind, n_seq, ws_need, counter_bytes, fn, _ = plan
    stream = _stream_of(logits)
    loss = logits.new_empty((), dtype=torch.float32)
    counts = ids.new_empty(E)
    share = logits.new_empty(n_seq * E, dtype=torch.float32)
    ws = _balance_pool.get(logits.device, stream, ws_need, counter_bytes)
    rc = fn(logits.data_ptr(), kind, score_fun, T, E, K, ids.data_ptr(), _ptr(mask), _ptr(cu), n_seq, coef, loss.data_ptr(), counts.data_ptr(),
            share.data_ptr(), ws.data_ptr(), ws.numel(), stream)
    if rc != 0:
        _lib.check(rc, "moe_balance_loss")
    return loss, counts, share


def _check_no_tangent(t):
    _check(unpack_dual(t).tangent is None, "moe_balance_loss: there is no forward-mode derivative")


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask, cu, score_fun, coef, plan):
        loss, counts, share = _balance_forward(logits, ids, mask, cu, score_fun, coef, plan)
        ctx.save_for_backward(logits, mask, cu, share)
        ctx.score_fun, ctx.plan = score_fun, plan
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    def backward(ctx, dloss, _):
        if torch.is_grad_enabled() and dloss is not None:                       # create_graph
            with torch.no_grad():
                grad = _balance_backward(ctx, dloss)[0]
            return _FirstDerivative.apply(grad.requires_grad_(True)), None, None, None, None, None, None
        return _balance_backward(ctx, dloss)


class _FirstDerivative(torch.autograd.Function):
    """The gradient as it is; its own derivative is refused, not taken for zero."""

    @staticmethod
    def forward(ctx, grad):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("moe_balance_loss: the gradient cannot be differentiated again")


def _balance_backward(ctx, dloss):
    if dloss is None:
        return None, None, None, None, None, None, None
    _check_no_tangent(dloss)
    logits, mask, cu, share = ctx.saved_tensors
    if logits.get_device() != torch.cuda.current_device():
        with torch.cuda.device(logits.device):
            grad = _balance_grad_launch(ctx, dloss, logits, mask, cu, share)
    else:
        grad = _balance_grad_launch(ctx, dloss, logits, mask, cu, share)
    return grad, None, None, None, None, None, None


def _balance_grad_launch(ctx, dloss, logits, mask, cu, share):
    T, E, _, kind, n_seq, _, _, _, fn = ctx.plan
    grad = torch.empty_like(logits)
    rc = fn(logits.data_ptr(), kind, ctx.score_fun, T, E, _ptr(mask), _ptr(cu), n_seq, share.data_ptr(), dloss.data_ptr(), grad.data_ptr(),
            _stream_of(logits))
    if rc != 0:
        _lib.check(rc, "moe_balance_loss")
    return grad


def moe_balance_loss(gating_output, experts_ids, score_func="softmax", coef=1.0, token_mask=None, cu_seqlens=None):
    """Balance loss of a router and its per-expert counts: (loss fp32 [], counts int32 [E]); differentiable in gating_output.

    loss = coef * mean over the sequences that have a valid token of E * sum_e f_e P_e, f_e = share of their valid tokens' routed pairs that went to e
    (a constant of the differentiation), P_e = mean over them of the router's probabilities: softmax of the logits, or with "sigmoid" the
    sigmoids over their sum.  counts: routed pairs of all valid tokens.

    gating_output [T, E] fp16 / bf16 / fp32, E <= 256; experts_ids int32 [T, K] (`fused_routing_gate`); token_mask bool [T], False for padded
    tokens; cu_seqlens int32 [sequences + 1] on the device, non-decreasing, where each sequence begins and the last one ends (None: all tokens are
    one).  Masked rows and rows outside the sequences may hold anything; their gradient is 0.  A second derivative
    and a derivative in forward mode are refused.
    Both passes may be recorded into a HIP graph, once run on its stream; as with any torch function no earlier loss of the same leaf may then be alive."""
    logits = gating_output
    _check_no_tangent(logits)
    key = ("balance", logits.shape, logits.dtype, logits.get_device(), experts_ids.shape, experts_ids.dtype, experts_ids.get_device(),
           None if token_mask is None else (token_mask.shape, token_mask.dtype, token_mask.get_device()),
           None if cu_seqlens is None else (cu_seqlens.shape, cu_seqlens.dtype, cu_seqlens.get_device()))
    plan = _plans.get(key)
    if plan is None or not (logits.is_contiguous() and experts_ids.is_contiguous() and (token_mask is None or token_mask.is_contiguous()) and
                            (cu_seqlens is None or cu_seqlens.is_contiguous())):
        _check(logits.dim() == 2 and 1 <= logits.size(1) <= 256, "gating_output must be [T, E], at most 256 experts")
        _check(logits.dtype in _LOGIT_KIND, "gating_output must be fp16, bf16 or fp32")
        _check(logits.is_cuda and logits.is_contiguous(), "gating_output must be a contiguous CUDA tensor")
        _check_routing(experts_ids, token_mask, logits.device)
        _check(experts_ids.size(0) == logits.size(0), "experts_ids must be int32 [T, K]")
        _check(cu_seqlens is None or (cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and 1 <= cu_seqlens.numel() <= 65536),
               "cu_seqlens must be int32 [sequences + 1], at most 65535 sequences")
        _check_tensors(((cu_seqlens, "cu_seqlens"),), logits.device)
        lib, (T, E), n_seq = _lib.load(), logits.shape, 1 if cu_seqlens is None else cu_seqlens.numel() - 1
        plan = _plans[key] = (T, E, experts_ids.size(1), _LOGIT_KIND[logits.dtype], n_seq, lib.mlk_balance_workspace_bytes(T, E, n_seq),
                              lib.mlk_balance_counter_bytes(), lib.mlk_balance_loss, lib.mlk_balance_loss_grad)
    if score_func not in ("softmax", "sigmoid"):
        raise ValueError("Unsupported scoring function")
    score_fun = 0 if score_func == "softmax" else 1
    if logits.requires_grad and torch.is_grad_enabled():
        return _BalanceLoss.apply(logits, experts_ids, token_mask, cu_seqlens, score_fun, float(coef), plan)
    return _balance_forward(logits, experts_ids, token_mask, cu_seqlens, score_fun, float(coef), plan)[:2]


# ------------------------------------------------- names outside the hot path
def _out_of_scope(name, why):
    def fn(*args, **kwargs):
        raise NotImplementedError("%s is outside the weight-stationary hot path: %s" % (name, why))
    fn.__name__ = name
    return fn


gemmEx = _out_of_scope("gemmEx", "it wraps the vendor BLAS of the reference (csrc/gemm_ex.cu); use torch.matmul")
muxi_hgemm = _out_of_scope("muxi_hgemm", "large-tile prefill GEMM (csrc/muxi_hgemm.cu); use torch.matmul / hipBLASLt")
muxi_hgemm_layout = _out_of_scope("muxi_hgemm_layout", "large-tile prefill GEMM (csrc/muxi_hgemm_layout.cu)")
muxi_hgemm_layoutA = _out_of_scope("muxi_hgemm_layoutA", "large-tile prefill GEMM (csrc/muxi_hgemm_layoutA.cu)")
muxi_hgemm_layoutC = _out_of_scope("muxi_hgemm_layoutC", "large-tile prefill GEMM (csrc/muxi_hgemm_layoutC.cu)")
routing_gate = _out_of_scope("routing_gate", "legacy split MoE (csrc/moe_kernels/routing_gate.cu); use fused_routing_gate")
experts_compute = _out_of_scope("experts_compute",
                                "legacy split MoE (csrc/moe_kernels/experts_compute.cu); use fused_experts_compute")

__all__ = [
    "layoutB", "reLayoutC", "gemm_layoutABC", "gemm_layoutA_linear", "gemm_layoutA", "gemm_layoutA_soft_fp8",
    "gemm_layoutAB_ContinuousC", "gemmEx", "muxi_hgemm", "muxi_hgemm_layout", "muxi_hgemm_layoutA",
    "muxi_hgemm_layoutC", "gemv_layoutA", "gemm_layoutABC_wapper", "gemm_layoutA_wapper",
    "gemm_layoutA_soft_fp8_wapper", "gemm_layoutAB_ContinuousC_wapper", "gemv_layoutA_wapper", "fp8_weight_repack",
    "routing_gate", "experts_compute", "fused_routing_gate",
    "batched_routed_activation_indexed_to_expert_block_indexed", "fused_experts_compute",
    "pack_layout_a", "unpack_layout_a", "experts_compute_raw", "release_workspaces", "workspace_bytes_held",
    "fused_moe_raw", "pack_layout_a_w4", "unpack_layout_a_w4", "gemm_layoutA_w4", "gemv_layoutA_w4",
    "fused_experts_w4", "expert_counts", "moe_balance_loss",
]
