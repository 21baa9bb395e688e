"""int8 products next to the emulated FP8 GEMM: quantize_int8, int8_scaled_mm, int8_grouped_scaled_mm.

    xq, sx = quantize_int8(x)                        # codes [.., K] int8, one fp32 scale per row [.., 1]
    wq, sw = quantize_int8(w)                        # w: [N, K], one scale per output channel
    y = int8_scaled_mm(xq, wq.t(), sx, sw.t(), bias, torch.bfloat16)

Integer tensor-core sums are exact on every GPU, so no profile takes part: the result is

    y = out_dtype(RN32(RN32(sum_k a[m, k] b[k, n]) * RN32(scale_a[m] * scale_b[n]) + bias[n]))

with one rounding for the product and the bias together (+0 without one, so a zero result is +0): the epilogue of
`scaled_mm` with a scale for each row and column.
The reference has no int8 path. Errors are TypeError for argument types, ValueError for shapes, layouts and devices,
UnsupportedFeatureError for inputs that require grad, BackendUnavailableError without an sm_100 device. Calls run on the
current stream of the operands' device, do not synchronise and can be captured into CUDA graphs. With
$MMAEMU_B200_CHECK_STATUS=1 a product waits for its own kernels and raises when one of their bounded waits has run out.
"""
from __future__ import annotations

import torch

from . import _lib
from .api import _SUPPORTED, _require_device
from .errors import UnsupportedFeatureError

__all__ = ["quantize_int8", "int8_scaled_mm", "int8_grouped_scaled_mm"]

_Tensor, _INT8, _F32 = torch.Tensor, torch.int8, torch.float32
MAX_K = 131071                     # 2^14 * K < 2^31: the int32 sums cannot overflow
MAX_ROWS = 1 << 23
MAX_N = 1 << 30                    # also of the values in a row of quantize_int8
MAX_GROUPS = 4096
_REAL_CODES = {torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}           # MMB200_HP_*
_OUT_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}            # MMB200_OUT_*


def _not_a_tensor(who: str, name: str, t) -> TypeError:
    return TypeError(f"{who}(): argument '{name}' must be Tensor, not {type(t).__name__}")


def _no_grad(who: str) -> UnsupportedFeatureError:
    return UnsupportedFeatureError(f"{who}(): inference only: an input requires grad while grad mode is enabled")


def _quantise(rows, ld, code, codes, scale, n, K, index) -> None:
    rc = _lib.load().mmb200_quantize_int8(rows.data_ptr(), ld, code, codes.data_ptr(), K, scale.data_ptr(), n, K,
                                          torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check("mmb200_quantize_int8", rc)


def quantize_int8(x):
    """Symmetric int8 quantisation of every row (last dimension) of x, fp32, bf16 or fp16: (codes, scale).

    scale = amax / 127 (fp32, shape [..., 1]) and codes = the integer nearest to x * 127 / amax, ties to even, decided
    exactly (int8, the shape of x, contiguous; between -127 and 127). A row of zeros has scale 0; a row with a NaN or an
    infinity has scale NaN and codes 0, which makes every product with it NaN. Rows quantised this way are the operands of
    int8_scaled_mm: activations [M, K] give scale_a [M, 1], weights [N, K] give scale_b.t() [1, N]."""
    if not isinstance(x, torch.Tensor):
        raise _not_a_tensor("quantize_int8", "x", x)
    code = _REAL_CODES.get(x.dtype)
    if code is None:
        raise TypeError(f"quantize_int8(): x must be float32, bfloat16 or float16, got {x.dtype}")
    if x.is_neg():                       # the imaginary part of a conjugate: its sign is a bit of the tensor, not of the memory
        x = x.resolve_neg()
    shape = x.shape
    if not shape:
        raise ValueError("quantize_int8(): x must have at least one dimension")
    if x.requires_grad and torch.is_grad_enabled():
        raise _no_grad("quantize_int8")
    K = shape[-1]
    if K > MAX_N:
        raise ValueError(f"quantize_int8(): a row has at most {MAX_N} values, got {K}")
    index = x.get_device()
    if index not in _SUPPORTED:
        _require_device(x.device)
    rows, n = x, shape[0]
    if len(shape) != 2:
        n = shape[:-1].numel()
        rows = x.detach().reshape(n, K)
    ld = rows.stride(0) if n > 1 else K
    if ld < K or (rows.stride(1) != 1 and K > 1):
        rows = rows.detach().contiguous()
        ld = K
    # (the cheapest ways to allocate: 1.4 and 1.9 us of a call, torch.empty takes 3.1 and 2.3)
    codes = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    scale = x.new_empty((n, 1) if len(shape) == 2 else (*shape[:-1], 1), dtype=torch.float32)
    if n == 0:
        return codes, scale
    if index == torch._C._cuda_getDevice():
        _quantise(rows, ld, code, codes, scale, n, K, index)
    else:
        with torch.cuda.device(index):
            _quantise(rows, ld, code, codes, scale, n, K, index)
    return codes, scale


def _check_operands(who, input, mat2, scale_a, scale_b, bias, out) -> int:
    """Types, one device (its index; -1: no GPU), no gradients."""
    if not (isinstance(input, _Tensor) and isinstance(mat2, _Tensor) and isinstance(scale_a, _Tensor) and isinstance(scale_b, _Tensor)
            and (bias is None or isinstance(bias, _Tensor)) and (out is None or isinstance(out, _Tensor))):
        for name, t in (("input", input), ("mat2", mat2), ("scale_a", scale_a), ("scale_b", scale_b), ("bias", bias), ("out", out)):
            if not isinstance(t, _Tensor) and (t is not None or name not in ("bias", "out")):
                raise _not_a_tensor(who, name, t)
    if input.dtype is not _INT8 or mat2.dtype is not _INT8:
        raise TypeError(f"{who}(): input and mat2 must be int8, got {input.dtype} and {mat2.dtype}")
    index = input.get_device()
    if not (index == mat2.get_device() == scale_a.get_device() == scale_b.get_device() and (bias is None or bias.get_device() == index)
            and (out is None or out.get_device() == index)):
        raise ValueError(f"{who}(): expected all tensors on one device, found "
                         f"{sorted({str(t.device) for t in (input, mat2, scale_a, scale_b, bias, out) if t is not None})}")
    if (scale_a.requires_grad or scale_b.requires_grad or (bias is not None and bias.requires_grad)
            or (out is not None and out.requires_grad)) and torch.is_grad_enabled():
        raise _no_grad(who)
    if scale_a.dtype is not _F32 or scale_b.dtype is not _F32:
        raise ValueError(f"{who}(): scale_a and scale_b must be float32, got {scale_a.dtype} and {scale_b.dtype}")
    return index


def _rows_of(t: torch.Tensor, rows: int, K: int):
    """(tensor, row stride) of a [rows, K] int8 operand whose rows the kernels can read: unit stride along K, no overlap."""
    ld, unit = t.stride()
    if (unit != 1 and K > 1) or (rows > 1 and ld < K):
        return t.contiguous(), K
    return t, (ld if rows > 1 else K)


def _scale_a(who, scale_a, rows):
    """Stride of scale_a over the rows; 0: one element."""
    if scale_a.numel() == 1:
        return 0
    if scale_a.dim() != 2 or scale_a.shape[0] != rows or scale_a.shape[1] != 1:
        raise ValueError(f"{who}(): scale_a must have one element or shape {(rows, 1)}, got {tuple(scale_a.shape)}")
    return scale_a.stride(0)


def _output(who, input, out, out_dtype, rows, N):
    """(tensor, row stride, code of the dtype) of the output."""
    if out_dtype is not None and not isinstance(out_dtype, torch.dtype):
        raise TypeError(f"{who}(): argument 'out_dtype' must be torch.dtype, not {type(out_dtype).__name__}")
    if out is not None and out_dtype is not None and out_dtype != out.dtype:
        raise ValueError(f"{who}(): out_dtype must match the dtype of out ({out_dtype}, {out.dtype})")
    dtype = out.dtype if out is not None else torch.bfloat16 if out_dtype is None else out_dtype
    code = _OUT_CODES.get(dtype)
    if code is None:
        raise ValueError(f"{who}(): the output is float32, bfloat16 or float16, got {dtype}")
    if out is None:
        return (input.new_empty((rows, N), dtype=dtype) if input.is_cuda else None), N, code
    if tuple(out.shape) != (rows, N) or (N > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < N) or out.is_neg():
        raise ValueError(f"{who}(): out must be a row-major tensor of shape {(rows, N)}, got shape {tuple(out.shape)} with strides "
                         f"{tuple(out.stride())}")
    return out, (out.stride(0) if rows > 1 else N), code


def _bias(who, bias, shape):
    """(tensor, code of the dtype)"""
    code = _REAL_CODES.get(bias.dtype)
    if code is None:
        raise ValueError(f"{who}(): bias must be float32, bfloat16 or float16, got {bias.dtype}")
    if tuple(bias.shape) != shape:
        raise ValueError(f"{who}(): bias must have shape {shape}, got {tuple(bias.shape)}")
    return bias.detach().contiguous(), code


def _run(index, ap, lda, wp, ldw, gsw, y, *rest) -> None:
    """The call into the library. rest: what follows D_dev in mmb200_int8_args, up to zero_rest."""
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _run(index, ap, lda, wp, ldw, gsw, y, *rest)
    L = _lib.load()
    ws, ws_ptr, n = None, 0, 0
    if (ap | wp | lda | ldw | gsw) & 15 or (rest[5] > 1 and not gsw):   # rows that TMA cannot read in place: room for copies
        n = L.mmb200_int8_workspace_bytes(ap, lda, wp, ldw, gsw, *rest[2:6])
        if n:
            ws = y.new_empty(n, dtype=torch.uint8)
            ws_ptr = ws.data_ptr()
    rc = L.mmb200_int8_scaled_mm(_lib.int8_args(ap, lda, wp, ldw, gsw, y.data_ptr(), *rest, ws_ptr, n,
                                                torch._C._cuda_getCurrentRawStream(index)))
    if rc:
        _lib.check("mmb200_int8_scaled_mm", rc)


def int8_scaled_mm(input, mat2, scale_a, scale_b, bias=None, out_dtype=None, *, out=None):
    """input [M, K] int8 times mat2 [K, N] int8 (column-major: w.t() of a row-major [N, K] weight) with exact int32 sums,
    scaled: out_dtype(sum * (scale_a * scale_b) + bias), the arithmetic of the module docstring.

    scale_a: one element or [M, 1], scale_b: one element or [1, N], fp32. bias: [N] fp32, bf16 or fp16. out_dtype: bfloat16
    (default), float16 or float32. out: a row-major [M, N] tensor of the output dtype (any row stride) to write into.
    K <= 131071, M <= 2^23, N <= 2^30. Rows of any alignment and stride are served; those that do not start on 16 bytes are copied
    first."""
    who = "int8_scaled_mm"
    index = _check_operands(who, input, mat2, scale_a, scale_b, bias, out)
    if scale_a.is_neg() or scale_b.is_neg() or (bias is not None and bias.is_neg()):
        scale_a, scale_b, bias = scale_a.resolve_neg(), scale_b.resolve_neg(), None if bias is None else bias.resolve_neg()
    sizes, sizes2 = input.shape, mat2.shape
    if len(sizes) != 2 or len(sizes2) != 2 or sizes[1] != sizes2[0]:
        raise ValueError(f"{who}(): expected input [M, K] and mat2 [K, N], got {tuple(sizes)} and {tuple(sizes2)}")
    (M, K), N = sizes, sizes2[1]
    if K > MAX_K or M > MAX_ROWS or N > MAX_N:
        raise ValueError(f"{who}(): K is at most {MAX_K} (int32 sums), M at most {MAX_ROWS} and N at most {MAX_N}, got K = {K}, "
                         f"M = {M}, N = {N}")
    unit, ldw = mat2.stride()
    if K > 1 and N > 0 and unit != 1:
        raise ValueError(f"{who}(): mat2 must be column-major (the transpose of a row-major [N, K] weight), got strides "
                         f"{(unit, ldw)}")
    sa = _scale_a(who, scale_a, M)
    if scale_b.numel() == 1:
        sb = 0
    elif scale_b.dim() == 2 and scale_b.shape[0] == 1 and scale_b.shape[1] == N:
        sb = scale_b.stride(1)
    else:
        raise ValueError(f"{who}(): scale_b must have one element or shape {(1, N)}, got {tuple(scale_b.shape)}")
    bias_code = 0
    if bias is not None:
        bias, bias_code = _bias(who, bias, (N,))
    y, ldd, code = _output(who, input, out, out_dtype, M, N)
    if index not in _SUPPORTED:
        _require_device(input.device)
    if M == 0 or N == 0:
        return y
    a, lda = _rows_of(input, M, K)
    if N == 1:
        ldw = K
    elif ldw < K:                                        # overlapping rows
        mat2, ldw = mat2.t().contiguous(), K
    _run(index, a.data_ptr(), lda, mat2.data_ptr(), ldw, 0, y, ldd, code, M, N, K, 1, 0, scale_a.data_ptr(), sa, scale_b.data_ptr(), 0,
         sb, 0 if bias is None else bias.data_ptr(), bias_code, 0, 0)
    return y


def int8_grouped_scaled_mm(input, mat2, offs, scale_a, scale_b, bias=None, out_dtype=None, *, out=None):
    """int8_scaled_mm for ragged groups of rows with weights of their own (rows sorted by expert): the rows
    offs[e - 1] .. offs[e] - 1 of input [T, K] are multiplied with mat2[e].

    mat2: [E, K, N] int8, every matrix column-major (w.transpose(1, 2) of [E, N, K] weights). offs: int32 [E] on the device,
    the end of every group's rows; it is read by the kernels, never by the host, so routing decided on the GPU needs no
    synchronisation. Groups may be empty. Ends are taken as a running maximum and clamped to [0, T]. scale_a: one element or
    [T, 1]; scale_b: one element or [E, 1, N]; bias: [E, N]. Rows behind the last group (a padded batch) are zero in a new
    output and keep their contents in `out`. Everything else as int8_scaled_mm; E <= 4096."""
    who = "int8_grouped_scaled_mm"
    if not isinstance(offs, torch.Tensor):
        raise _not_a_tensor(who, "offs", offs)
    index = _check_operands(who, input, mat2, scale_a, scale_b, bias, out)
    if scale_a.is_neg() or scale_b.is_neg() or (bias is not None and bias.is_neg()):
        scale_a, scale_b, bias = scale_a.resolve_neg(), scale_b.resolve_neg(), None if bias is None else bias.resolve_neg()
    if offs.get_device() != index:
        raise ValueError(f"{who}(): expected all tensors on one device, found {input.device} and {offs.device}")
    sizes, sizes2 = input.shape, mat2.shape
    if len(sizes) != 2 or len(sizes2) != 3 or sizes[1] != sizes2[1]:
        raise ValueError(f"{who}(): expected input [T, K] and mat2 [E, K, N], got {tuple(sizes)} and {tuple(sizes2)}")
    (T, K), (E, _, N) = sizes, sizes2
    if K > MAX_K or T > MAX_ROWS or E > MAX_GROUPS or N > MAX_N:
        raise ValueError(f"{who}(): K is at most {MAX_K} (int32 sums), T at most {MAX_ROWS}, E at most {MAX_GROUPS} and N at most "
                         f"{MAX_N}, got K = {K}, T = {T}, E = {E}, N = {N}")
    if offs.dtype != torch.int32 or offs.dim() != 1 or offs.shape[0] != E:
        raise ValueError(f"{who}(): offs must be int32 of shape {(E,)}, got {offs.dtype} of shape {tuple(offs.shape)}")
    gsw, unit, ldw = mat2.stride()
    if K > 1 and N > 0 and E > 0 and unit != 1:
        raise ValueError(f"{who}(): every matrix of mat2 must be column-major (the transpose of row-major [E, N, K] weights), got "
                         f"strides {(gsw, unit, ldw)}")
    sa = _scale_a(who, scale_a, T)
    if scale_b.numel() == 1:
        sb_group = sb = 0
    elif tuple(scale_b.shape) == (E, 1, N):
        sb_group, _, sb = scale_b.stride()
    else:
        raise ValueError(f"{who}(): scale_b must have one element or shape {(E, 1, N)}, got {tuple(scale_b.shape)}")
    bias_code = 0
    if bias is not None:
        bias, bias_code = _bias(who, bias, (E, N))
    y, ldd, code = _output(who, input, out, out_dtype, T, N)
    if index not in _SUPPORTED:
        _require_device(input.device)
    if T == 0 or N == 0:
        return y
    if E == 0:
        return y.zero_() if out is None else y
    a, lda = _rows_of(input, T, K)
    if N > 1 and ldw < K:                                # overlapping rows
        mat2 = mat2.transpose(1, 2).contiguous()
        gsw, ldw = N * K, K
    offs = offs.contiguous()
    _run(index, a.data_ptr(), lda, mat2.data_ptr(), ldw if N > 1 else K, gsw if E > 1 else 0, y, ldd, code, T, N, K, E, offs.data_ptr(),
         scale_a.data_ptr(), sa, scale_b.data_ptr(), sb_group, sb, 0 if bias is None else bias.data_ptr(), bias_code, N,
         int(out is None))
    return y


# torch.compile must not trace into these entry points (they call a foreign library through ctypes)
quantize_int8 = torch.compiler.disable(quantize_int8)
int8_scaled_mm = torch.compiler.disable(int8_scaled_mm)
int8_grouped_scaled_mm = torch.compiler.disable(int8_grouped_scaled_mm)
