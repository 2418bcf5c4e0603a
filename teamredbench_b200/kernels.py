"""torch-tensor front end of the native kernels.

Thin: it checks shapes / dtypes / devices, takes raw device pointers and the
current CUDA stream, and calls libtrb_b200 through ``_native``.  torch provides
device memory and streams only; all arithmetic happens in the CUDA kernels.
"""
from __future__ import annotations

from typing import Any

from teamredbench_b200 import _native

_TORCH_TO_TRB = {
    "torch.float32": "float32",
    "torch.bfloat16": "bfloat16",
    "torch.float16": "float16",
    "torch.float64": "float64",
    "torch.int8": "int8",
    "torch.uint8": "int8",
    "torch.float8_e4m3fn": "float8_e4m3fn",
}


_DTYPE_CACHE: dict[Any, str] = {}  # torch.dtype object -> library dtype name, filled on first use


def trb_dtype(tensor: Any) -> str:
    name = _DTYPE_CACHE.get(tensor.dtype)
    if name is None:
        name = _TORCH_TO_TRB.get(str(tensor.dtype))
        if name is None:
            raise _native.NativeSkipped(1, f"unsupported tensor dtype {tensor.dtype}")
        _DTYPE_CACHE[tensor.dtype] = name
    return name


_RAW_STREAM: Any = None  # device index -> raw handle of its current stream, found on first use


def _stream_handle(tensor: Any, stream: Any | None) -> int:
    """Raw cudaStream_t of ``stream``, or of the device's current stream.

    The current stream is read through torch's raw-handle query (one C call,
    no Stream object built), which keeps the per-call host cost of a small
    GEMM close to the bare ctypes call; torch builds without it take the
    public ``torch.cuda.current_stream``."""
    global _RAW_STREAM
    if stream is not None:
        device = tensor.get_device()
        if getattr(stream, "device_index", device) != device:
            raise ValueError(f"stream is on cuda:{stream.device_index}, the tensors on cuda:{device}")
        return int(stream.cuda_stream)
    if _RAW_STREAM is None:
        import torch

        _RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda device: torch.cuda.current_stream(device).cuda_stream)
    return int(_RAW_STREAM(tensor.get_device()))


_CURRENT_DEVICE: Any = None  # () -> index of the calling thread's current device, found on first use


def _launch_on(device: int, launch: Any, *args: Any) -> None:
    """launch(*args) with `device`, the operands' own, as the current one.  The
    library launches on the current device, and the default streams of all
    devices have the same raw handle, so a stream alone does not name it."""
    global _CURRENT_DEVICE
    if _CURRENT_DEVICE is None:
        import torch

        _CURRENT_DEVICE = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    if _CURRENT_DEVICE() == device:
        launch(*args)
        return
    import torch

    with torch.cuda.device(device):
        launch(*args)


def _require_cuda_contiguous(*tensors: Any) -> None:
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("tensor must live on a CUDA device")
        if not t.is_contiguous():
            raise ValueError("tensor must be contiguous")


def stream_op(mode: str, dst: Any, src: Any, aux: Any | None = None, scale: float = 1.0, variant: str = "auto",
              blocks_per_sm: int = 0, stream: Any | None = None) -> Any:
    """dst = copy / scale / triad of src (and aux) -- the hbm benchmark's op
    (reference src/teamredbench/benchmarks/hbm.py:29-39), on the GPU."""
    _require_cuda_contiguous(dst, src, aux)
    if src.dtype != dst.dtype or (aux is not None and aux.dtype != src.dtype):
        raise ValueError("dst, src and aux must share one dtype")
    if src.numel() != dst.numel() or (aux is not None and aux.numel() != src.numel()):
        raise ValueError("dst, src and aux must have the same number of elements")
    if mode == "triad" and aux is None:
        raise ValueError("triad needs aux")
    _launch_on(src.get_device(), _native.hbm_launch, trb_dtype(src), mode, dst.data_ptr(), src.data_ptr(),
               aux.data_ptr() if aux is not None else None, src.numel(), float(scale), variant, blocks_per_sm,
               _stream_handle(src, stream))
    return dst


def gemm(a: Any, b: Any, out: Any, *, dtype: str | None = None, scale_a: float = 1.0, scale_b: float = 1.0,
         splits: int = 0, cta_pair: int = -1, b_transposed: bool = False, stream: Any | None = None,
         tile_n: int = 0) -> Any:
    """out = a @ b on the tcgen05 kernel; a (m x k) and b (k x n) row-major.
    With b_transposed=True, `b` holds B^T as a row-major (n x k) tensor.

    dtype defaults to the tensors' dtype; pass ``dtype="tfloat32"`` to run
    float32 tensors on the tf32 tensor-core path (float32 itself runs as three
    tf32 products, float64 on the DMMA tensor path).  Output dtypes: bf16 for bf16 /
    e4m3 inputs, f16 for f16, f32 for tf32 and float32, f64 for float64, int32
    for int8.
    splits: 0 = automatic split-K, >= 1 forces that many K splits reduced
    through a global workspace, -2 / -4 / -8 that many splits reduced inside a
    thread-block cluster (distributed shared memory).
    cta_pair: -1 automatic, 0 single-CTA 128x256 kernel, 1 CTA-pair 256x256 kernel,
    2 CTA pair with 256x512 tiles (bf16 / f16 / e4m3 inputs, no split-K; bit-identical
    to cta_pair=1).
    tile_n: 0 automatic, 64/128/256 single-CTA tile width, -1 the
    swapped-operand skinny kernel (C^T = B^T A^T, m <= 64; automatic for
    m <= 64)."""
    _require_cuda_contiguous(a, b, out)
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError(f"gemm operands must be 2-D, got {tuple(a.shape)} x {tuple(b.shape)}")
    m, k = a.shape
    n, bk = b.shape if b_transposed else reversed(b.shape)
    if bk != k:
        raise ValueError(f"incompatible shapes {tuple(a.shape)} x {tuple(b.shape)} (b_transposed={b_transposed})")
    if out.shape != (m, n):
        raise ValueError(f"out must be {(m, n)}, got {tuple(out.shape)}")
    name = dtype or trb_dtype(a)
    _launch_on(a.get_device(), _native.gemm_launch_ex, name, m, n, k, a.data_ptr(), b.data_ptr(), out.data_ptr(),
               float(scale_a), float(scale_b), int(splits), int(cta_pair), "k_major" if b_transposed else "row_major",
               _stream_handle(a, stream), int(tile_n))
    return out


_INT32: Any = None  # torch.int32 and torch.uint8, looked up on first use
_UINT8: Any = None


def _check_operands(*tensors: Any) -> int:
    """The one CUDA device (its index) that all tensors are on, contiguous.  A
    call of a few microseconds is made of such checks: two queries a tensor,
    and the wording of an error only once there is one."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is None:
            continue
        if t.get_device() != device or device < 0 or not t.is_contiguous():
            _require_cuda_contiguous(*tensors)
            raise ValueError(f"tensors must share one device, got {t.device} beside {tensors[0].device}")
    return device


def _check_offsets(offsets: Any, groups: int) -> None:
    global _INT32
    if _INT32 is None:
        import torch

        _INT32 = torch.int32
    if offsets.dtype is not _INT32 or offsets.dim() != 1 or offsets.numel() != groups + 1:
        raise ValueError(f"offsets must be {groups + 1} int32 values, got {tuple(offsets.shape)} {offsets.dtype}")


def grouped_gemm(a: Any, b: Any, offsets: Any, out: Any, *, b_transposed: bool = False, stream: Any | None = None) -> Any:
    """out[r] = a[r] @ b[e] for the rows r of group (expert) e, bf16 or f16.

    a (rows x k) and out (rows x n) are sorted by group; offsets (groups + 1
    int32 on the device) gives group e the rows [offsets[e], offsets[e + 1]).
    b is (groups x k x n), or (groups x n x k) with b_transposed=True; the
    gradient of a is the same call on the gradient of out with the other value
    of b_transposed.  Groups may be empty; rows outside every group are left as
    they are.  n and k must be multiples of 8.  Offsets that decrease or leave
    [0, rows] compute nothing and set the device error word to 7
    (``_native.device_error``), which the host does not wait for here."""
    device = _check_operands(a, b, offsets, out)
    if a.dim() != 2 or b.dim() != 3:
        raise ValueError(f"grouped_gemm takes a 2-D a and a 3-D b, got {tuple(a.shape)} and {tuple(b.shape)}")
    rows, k = a.shape
    groups, bk, n = b.shape
    if b_transposed:
        bk, n = n, bk
    if bk != k:
        raise ValueError(f"incompatible shapes {tuple(a.shape)} x {tuple(b.shape)} (b_transposed={b_transposed})")
    if out.shape != (rows, n):
        raise ValueError(f"out must be {(rows, n)}, got {tuple(out.shape)}")
    dtype = a.dtype
    if b.dtype is not dtype or out.dtype is not dtype:
        raise ValueError("a, b and out must share one dtype")
    _check_offsets(offsets, groups)
    _launch_on(device, _native.grouped_gemm_launch, trb_dtype(a), groups, rows, n, k, a.data_ptr(), b.data_ptr(),
               "k_major" if b_transposed else "row_major", offsets.data_ptr(), out.data_ptr(),
               _stream_handle(a, stream))
    return out


def grouped_gemm_wgrad(a: Any, grad: Any, offsets: Any, out: Any, *, stream: Any | None = None) -> Any:
    """out[e] = a[rows of e].T @ grad[rows of e]: the gradient of grouped_gemm's
    (groups x k x n) weights from a (rows x k) and the gradient of its output
    (rows x n); zeros for a group without rows.  For weights kept
    (groups x n x k) pass grad first and a second.  offsets, types, sizes and
    errors as in grouped_gemm."""
    device = _check_operands(a, grad, offsets, out)
    if a.dim() != 2 or grad.dim() != 2 or out.dim() != 3:
        raise ValueError(f"grouped_gemm_wgrad takes 2-D a and grad and a 3-D out, got {tuple(a.shape)}, "
                         f"{tuple(grad.shape)} and {tuple(out.shape)}")
    rows, k = a.shape
    grad_rows, n = grad.shape
    groups, out_k, out_n = out.shape
    if grad_rows != rows:
        raise ValueError(f"a and grad must have the same number of rows, got {rows} and {grad_rows}")
    if out_k != k or out_n != n:
        raise ValueError(f"out must be {(groups, k, n)}, got {tuple(out.shape)}")
    dtype = a.dtype
    if grad.dtype is not dtype or out.dtype is not dtype:
        raise ValueError("a, grad and out must share one dtype")
    _check_offsets(offsets, groups)
    _launch_on(device, _native.grouped_wgrad_launch, trb_dtype(a), groups, rows, n, k, a.data_ptr(), grad.data_ptr(),
               offsets.data_ptr(), out.data_ptr(), _stream_handle(a, stream))
    return out


def gemv_w4(x: Any, q: Any, scales: Any, out: Any, *, zeros: Any | None = None, offsets: Any | None = None,
            stream: Any | None = None) -> Any:
    """out[r] = W[e] @ x[r] for the rows r of group (expert) e, with 4-bit weights
    W[e, n, k] = (q[e, n, k] - zeros[e, n, k // g]) * scales[e, n, k // g].

    x is (rows x k) and out (rows x n), bf16 or f16; q is uint8 (groups x n x k/2),
    two weights a byte, the even k in the low four bits; scales (groups x n x k/g),
    of x's dtype, sets the group size g (a power of two of at least 32); zeros is
    uint8 of the same shape (values 0 to 15), or None for 8.  A single matrix may
    be given without the leading dimension, and needs no offsets; otherwise
    offsets are those of grouped_gemm.  Meant for few rows a group: their weights
    are read once for the rows taken at once, 8 or 16 of them and no more than
    65536 / k.  k is at most 65536; n is free."""
    global _UINT8
    device = _check_operands(x, q, scales, out, zeros, offsets)
    if x.dim() != 2 or q.dim() not in (2, 3):
        raise ValueError(f"gemv_w4 takes a 2-D x and a 2-D or 3-D q, got {tuple(x.shape)} and {tuple(q.shape)}")
    rows, k = x.shape
    outputs, scale_shape = q.shape, scales.shape
    groups = 1 if len(outputs) == 2 else outputs[0]
    n, k_bytes = outputs[-2:]
    if 2 * k_bytes != k:
        raise ValueError(f"q holds {2 * k_bytes} weights a row for k = {k}")
    k_groups = scale_shape[-1] if len(scale_shape) else 0
    if scale_shape[:-1] != outputs[:-1] or k_groups == 0 or k % k_groups:
        raise ValueError(f"scales must be {tuple(outputs[:-1])} x a divisor of {k}, got {tuple(scale_shape)}")
    if zeros is not None and zeros.shape != scale_shape:
        raise ValueError(f"zeros must be {tuple(scales.shape)}, got {tuple(zeros.shape)}")
    if out.shape != (rows, n):
        raise ValueError(f"out must be {(rows, n)}, got {tuple(out.shape)}")
    dtype = x.dtype
    if scales.dtype is not dtype or out.dtype is not dtype:
        raise ValueError("x, scales and out must share one dtype")
    if _UINT8 is None:
        import torch

        _UINT8 = torch.uint8
    if q.dtype is not _UINT8 or (zeros is not None and zeros.dtype is not _UINT8):
        raise ValueError("q and zeros must be uint8")
    if offsets is not None:
        _check_offsets(offsets, groups)
    elif groups != 1:
        raise ValueError(f"{groups} groups need offsets")
    _launch_on(device, _native.gemv_w4_launch, trb_dtype(x), groups, rows, n, k, k // k_groups, x.data_ptr(),
               q.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(),
               None if offsets is None else offsets.data_ptr(), out.data_ptr(), _stream_handle(x, stream))
    return out
