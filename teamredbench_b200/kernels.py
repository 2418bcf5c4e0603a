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


_SHORT: Any = None  # the compiled way from tensors to the library (csrc/trb_torch.cpp), False without it; found on first use


def _find_short() -> Any:
    """The functions of lib/trb_torch.*.so, each for the front end of its name: it
    makes the call and returns True where all arguments are as they have to be
    and the tensors' device is the current one, and does nothing and returns
    False otherwise.  The checks below are the same ones, with the words."""
    global _SHORT
    _SHORT = _native.load_torch_binding() or False
    return _SHORT


_ID_BYTES: Any = None  # {torch.int32: 4, torch.int64: 8}, found on first use


def expert_sort(experts: Any, offsets: Any, slots: Any, *, stream: Any | None = None) -> tuple[Any, Any]:
    """Sorts a router's choices by expert; returns (offsets, slots).

    experts (tokens x choices, int32 or int64, as topk's indices) holds the
    expert of each choice.  offsets (int32, one more than there are experts)
    gets what the grouped products take, slots (tokens x choices, int32) the row
    of each choice among the rows sorted by expert, in the order of the tokens
    inside an expert.  A choice outside [0, experts) -- another rank's expert,
    or -1 for a token left out -- gets the slot -1 and no row.  One launch,
    nothing allocated, the same result at every call.  As for the functions
    below, results must not share memory with operands or each other."""
    short = _SHORT if _SHORT is not None else _find_short()
    if stream is None and short and short.expert_sort(experts, offsets, slots):
        return offsets, slots
    global _ID_BYTES
    device = _check_operands(experts, offsets, slots)
    if _ID_BYTES is None:
        import torch

        _ID_BYTES = {torch.int32: 4, torch.int64: 8}
    id_bytes = _ID_BYTES.get(experts.dtype)
    if experts.dim() != 2 or id_bytes is None:
        raise ValueError(f"experts must be tokens x choices in int32 or int64, got {tuple(experts.shape)} {experts.dtype}")
    tokens, choices = experts.shape
    _check_slots(slots, tokens, choices)
    groups = offsets.numel() - 1
    if groups < 1:
        raise ValueError("offsets must hold one more value than there are experts")
    _check_offsets(offsets, groups)
    _launch_on(device, _native.expert_sort_launch, id_bytes, tokens, choices, groups, experts.data_ptr(),
               offsets.data_ptr(), slots.data_ptr(), _stream_handle(slots, stream))
    return offsets, slots


def _check_slots(slots: Any, tokens: int, choices: int | None = None) -> int:
    """The number of choices of (tokens x choices) int32 slots."""
    global _INT32
    if _INT32 is None:
        import torch

        _INT32 = torch.int32
    if slots.dtype is not _INT32 or slots.dim() != 2:
        raise ValueError(f"slots must be tokens x choices in int32, got {tuple(slots.shape)} {slots.dtype}")
    if slots.shape[0] != tokens or (choices is not None and slots.shape[1] != choices):
        want = f"{tokens} x {'choices' if choices is None else choices}"
        raise ValueError(f"slots must be {want}, got {tuple(slots.shape)}")
    return slots.shape[1]


def _check_rows(tokens_side: Any, rows_side: Any, slots: Any, weights: Any, name: str) -> tuple[int, int, int, int]:
    """(tokens, choices, rows, width) of the rows of tokens and of their experts."""
    if tokens_side.dim() != 2 or rows_side.dim() != 2 or tokens_side.shape[1] != rows_side.shape[1]:
        raise ValueError(f"{name} must be 2-D and equally wide, got {tuple(tokens_side.shape)} and "
                         f"{tuple(rows_side.shape)}")
    if tokens_side.dtype is not rows_side.dtype:
        raise ValueError(f"{name} must share one dtype")
    tokens, width = tokens_side.shape
    choices = _check_slots(slots, tokens)
    if weights is not None and weights.shape != slots.shape:
        raise ValueError(f"weights must be {tuple(slots.shape)}, got {tuple(weights.shape)}")
    return tokens, choices, rows_side.shape[0], width


def expert_dispatch(x: Any, slots: Any, out: Any, *, weights: Any | None = None, stream: Any | None = None) -> Any:
    """out[slots[t, j]] = x[t], times weights[t, j] if they are given: the rows of
    tokens to the rows of their experts.

    x is (tokens x width) and out (rows x width), bf16, f16 or float32; slots are
    expert_sort's, which differ (a row that two slots name gets values of both);
    weights (tokens x choices) are float32 or of x's dtype.  Rows
    of out that no slot names stay as they are, a negative slot is skipped, and
    one behind the last row is skipped and sets the device error word to 8
    (``_native.device_error``), which the host does not wait for here.  The
    gradient of x is expert_combine on the gradient of out, with the same
    weights.  That of the weights is grad_weights of expert_combine_grad(x,
    grad_out, slots, weights, grad_y, grad_weights), where grad_y, which gets
    dispatch's own result again, may be grad_out itself once x's gradient is
    made."""
    short = _SHORT if _SHORT is not None else _find_short()
    if stream is None and short and short.expert_dispatch(x, slots, out, weights):
        return out
    device = _check_operands(x, slots, out, weights)
    tokens, choices, rows, width = _check_rows(x, out, slots, weights, "x and out")
    dtype = trb_dtype(x)
    _launch_on(device, _native.expert_dispatch_launch, dtype, dtype if weights is None else trb_dtype(weights), tokens,
               choices, rows, width, x.data_ptr(), slots.data_ptr(), None if weights is None else weights.data_ptr(),
               out.data_ptr(), _stream_handle(x, stream))
    return out


def expert_combine(y: Any, slots: Any, out: Any, *, weights: Any | None = None, stream: Any | None = None) -> Any:
    """out[t] = the sum over j of weights[t, j] * y[slots[t, j]] (of the rows
    themselves without weights): the rows of experts back to their tokens.

    y is (rows x width) and out (tokens x width); a token without a row gets
    zeros.  fp32 sums in the order of the choices, rounded once.  Types, slots and
    errors as in expert_dispatch, whose gradient for x this is; its own
    gradient is expert_combine_grad."""
    short = _SHORT if _SHORT is not None else _find_short()
    if stream is None and short and short.expert_combine(y, slots, out, weights):
        return out
    device = _check_operands(y, slots, out, weights)
    tokens, choices, rows, width = _check_rows(out, y, slots, weights, "out and y")
    dtype = trb_dtype(y)
    _launch_on(device, _native.expert_combine_launch, dtype, dtype if weights is None else trb_dtype(weights), tokens,
               choices, rows, width, y.data_ptr(), slots.data_ptr(), None if weights is None else weights.data_ptr(),
               out.data_ptr(), _stream_handle(y, stream))
    return out


def expert_combine_grad(grad: Any, y: Any, slots: Any, weights: Any, grad_y: Any, grad_weights: Any, *,
                        stream: Any | None = None) -> tuple[Any, Any]:
    """The gradients of expert_combine's y and weights from grad, that of its
    result, in one pass; returns (grad_y, grad_weights).

    grad_y[slots[t, j]] = weights[t, j] * grad[t] (rows x width; rows that no
    slot names stay as they are), grad_weights[t, j] = the sum of grad[t] *
    y[slots[t, j]] over the width (tokens x choices, 0 for a negative slot), of
    the weights' dtype, summed in fp32.  grad_y may be y itself, which saves a
    matrix where y is not needed any more.  Types, slots and errors as in
    expert_dispatch."""
    short = _SHORT if _SHORT is not None else _find_short()
    if stream is None and short and short.expert_combine_grad(grad, y, slots, weights, grad_y, grad_weights):
        return grad_y, grad_weights
    device = _check_operands(grad, y, slots, weights, grad_y, grad_weights)
    tokens, choices, rows, width = _check_rows(grad, y, slots, weights, "grad and y")
    if grad_y.shape != y.shape or grad_y.dtype is not y.dtype:
        raise ValueError(f"grad_y must be {tuple(y.shape)} {y.dtype}, got {tuple(grad_y.shape)} {grad_y.dtype}")
    if grad_weights.shape != weights.shape or grad_weights.dtype is not weights.dtype:
        raise ValueError(f"grad_weights must be {tuple(weights.shape)} {weights.dtype}, got "
                         f"{tuple(grad_weights.shape)} {grad_weights.dtype}")
    _launch_on(device, _native.expert_combine_grad_launch, trb_dtype(grad), trb_dtype(weights), tokens, choices, rows,
               width, grad.data_ptr(), y.data_ptr(), slots.data_ptr(), weights.data_ptr(), grad_y.data_ptr(),
               grad_weights.data_ptr(), _stream_handle(grad, stream))
    return grad_y, grad_weights


def fp4_scale_pitch(k: int) -> int:
    """Bytes of scales a row of k values of 4-bit floating point has: one for 32
    values, up to a multiple of 16."""
    return (k // 32 + 15) // 16 * 16


def _check_fp4(q: Any, scales: Any, name: str) -> None:
    """q (... x k/2) and scales (... x pitch) belong together."""
    global _UINT8
    if _UINT8 is None:
        import torch

        _UINT8 = torch.uint8
    if q.dtype is not _UINT8 or scales.dtype is not _UINT8:
        raise ValueError(f"{name} and its scales must be uint8")
    shape = q.shape
    if shape[-1] % 16:
        raise ValueError(f"k must be a multiple of 32, got {2 * shape[-1]}")
    if scales.shape[:-1] != shape[:-1] or scales.shape[-1] != (shape[-1] // 16 + 15) // 16 * 16:
        raise ValueError(f"the scales of {name} must be {(*shape[:-1], fp4_scale_pitch(2 * shape[-1]))}, got "
                         f"{tuple(scales.shape)}")


def quantize_fp4(x: Any, q: Any, scales: Any, *, slots: Any | None = None, stream: Any | None = None) -> tuple[Any, Any]:
    """Rows of x (rows x k, bf16, f16 or float32) to microscaled 4-bit floating
    point; returns (q, scales).

    q (rows x k/2, uint8) holds two e2m1 values a byte, the even k in the low
    four bits; scales (rows x fp4_scale_pitch(k), uint8) one power of two (e8m0)
    for 32 values, 2^(floor(log2 max|x|) - 2), and zeros behind the last block.
    Values are rounded to the nearest code, ties to the even one, and stop at 6
    times the scale; a block with a NaN or an infinity becomes NaN.  k is a
    multiple of 32.  With slots (expert_sort's) row t of x goes to the rows
    slots[t, j] of q and scales, quantised once: expert_dispatch in 4 bits, with
    its rules for slots and other rows.  A matrix of weights (n x k) is
    quantised the same way, and a stack of them as its rows."""
    short = _SHORT if _SHORT is not None else _find_short()
    if stream is None and short and short.quantize_fp4(x, q, scales, slots):
        return q, scales
    device = _check_operands(x, q, scales, slots)
    if x.dim() != 2 or q.dim() != 2 or scales.dim() != 2:
        raise ValueError(f"quantize_fp4 takes a 2-D x, q and scales, got {tuple(x.shape)}, {tuple(q.shape)} and "
                         f"{tuple(scales.shape)}")
    rows, k = x.shape
    _check_fp4(q, scales, "q")
    if 2 * q.shape[1] != k or (slots is None and q.shape[0] != rows):
        raise ValueError(f"q must be {(rows if slots is None else 'rows', k // 2)} for k = {k}, got {tuple(q.shape)}")
    choices = 1 if slots is None else _check_slots(slots, rows)
    _launch_on(device, _native.quantize_fp4_launch, trb_dtype(x), rows, k, x.data_ptr(), choices,
               None if slots is None else slots.data_ptr(), q.shape[0], q.data_ptr(), scales.data_ptr(),
               _stream_handle(x, stream))
    return q, scales


def dequantize_fp4(q: Any, scales: Any, out: Any, *, stream: Any | None = None) -> Any:
    """out (rows x k, bf16, f16 or float32) = the values of quantize_fp4's q and
    scales: exact in bf16 and float32, except that values of 2^128 or more, which
    the scale bytes 253 and 254 can give and quantize_fp4 never writes, are
    infinite there.  f16 rounds what is too small for it, and what is too large
    is infinite."""
    short = _SHORT if _SHORT is not None else _find_short()
    if stream is None and short and short.dequantize_fp4(q, scales, out):
        return out
    device = _check_operands(q, scales, out)
    if q.dim() != 2 or scales.dim() != 2 or out.dim() != 2:
        raise ValueError(f"dequantize_fp4 takes a 2-D q, scales and out, got {tuple(q.shape)}, {tuple(scales.shape)} and "
                         f"{tuple(out.shape)}")
    _check_fp4(q, scales, "q")
    rows, k = out.shape
    if q.shape[0] != rows or 2 * q.shape[1] != k:
        raise ValueError(f"out must be {(q.shape[0], 2 * q.shape[1])}, got {tuple(out.shape)}")
    _launch_on(device, _native.dequantize_fp4_launch, trb_dtype(out), rows, k, q.data_ptr(), scales.data_ptr(),
               out.data_ptr(), _stream_handle(out, stream))
    return out


def gemm_fp4(a: Any, a_scales: Any, b: Any, b_scales: Any, out: Any, *, offsets: Any | None = None,
             stream: Any | None = None) -> Any:
    """out[r] = b[e] @ a[r] for the rows r of group (expert) e, both operands in
    microscaled 4-bit floating point as quantize_fp4 makes it.

    a and a_scales hold (rows x k), b and b_scales (groups x n x k); a single
    matrix may be given without the leading dimension, and needs no offsets;
    otherwise offsets are those of grouped_gemm.  out is (rows x n), bf16 or f16:
    fp32 sums, rounded once.  k is a multiple of 32, n is free.  What stands
    behind the last scale of a row does not matter.  Rows outside every group
    and wrong offsets as in grouped_gemm."""
    short = _SHORT if _SHORT is not None else _find_short()
    if stream is None and short and short.gemm_fp4(a, a_scales, b, b_scales, out, offsets):
        return out
    device = _check_operands(a, a_scales, b, b_scales, out, offsets)
    if a.dim() != 2 or b.dim() not in (2, 3) or out.dim() != 2:
        raise ValueError(f"gemm_fp4 takes a 2-D a, a 2-D or 3-D b and a 2-D out, got {tuple(a.shape)}, {tuple(b.shape)} "
                         f"and {tuple(out.shape)}")
    _check_fp4(a, a_scales, "a")
    _check_fp4(b, b_scales, "b")
    rows, k_bytes = a.shape
    outputs = b.shape
    groups = 1 if len(outputs) == 2 else outputs[0]
    n = outputs[-2]
    if outputs[-1] != k_bytes:
        raise ValueError(f"incompatible shapes {tuple(a.shape)} and {tuple(b.shape)}")
    if out.shape != (rows, n):
        raise ValueError(f"out must be {(rows, n)}, got {tuple(out.shape)}")
    if offsets is not None:
        _check_offsets(offsets, groups)
    elif groups != 1:
        raise ValueError(f"{groups} groups need offsets")
    _launch_on(device, _native.gemm_fp4_launch, trb_dtype(out), groups, rows, n, 2 * k_bytes, a.data_ptr(),
               a_scales.data_ptr(), b.data_ptr(), b_scales.data_ptr(), None if offsets is None else offsets.data_ptr(),
               out.data_ptr(), _stream_handle(a, stream))
    return out
