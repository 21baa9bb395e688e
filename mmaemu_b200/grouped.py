"""grouped_scaled_mm: the emulated FP8 GEMM for ragged groups of rows with weights of their own, in one call.

A mixture-of-experts layer sorts its rows by expert and multiplies every expert's rows with that expert's weights; on the
emulated platform that is one torch._scaled_mm (Transformer Engine: one cuBLASLt GEMM) per expert. The result here has the
bits of that loop over `scaled_mm`. The split-K decision of the emulated cuBLASLt depends on a group's number of rows, so
the group sizes are host integers, as Transformer Engine's grouped linear layers take them (m_splits). The reference has no
grouped call; its checks and raises (astding/mmaemu, mmaemu/api.py:280-326) apply to every group.
"""
from __future__ import annotations

import ctypes
import os

import torch

from . import _lib
from .api import (_check_argument_types, _check_like_cublas, _check_like_torch, _check_scope, _emit_maturity, _kernel_choice,
                  _kernel_code, _on_device, _require_device, _scalar_ptr, _stream_ptr)
from .errors import ReferenceRejectsError
from .formats import E5M2, NAME_OF, OUT_DTYPE_NAMES, fmt_of
from .numerics import check_plan, get_preset
from .platforms import get_profile
from .splitk import resolve_splitk

__all__ = ["grouped_scaled_mm"]

MAX_GROUPS = 4096
_PLAIN_OUT = (torch.bfloat16, torch.float16, torch.float32)


def _sizes(m_splits, E: int, T: int) -> list:
    if isinstance(m_splits, torch.Tensor):
        if m_splits.device.type != "cpu":
            raise TypeError("grouped_scaled_mm(): m_splits is read on the host (the split-K decision depends on it); got a tensor "
                            f"on {m_splits.device}")
        if m_splits.is_floating_point() or m_splits.is_complex() or m_splits.dtype == torch.bool:
            raise TypeError(f"grouped_scaled_mm(): m_splits must hold integers, got {m_splits.dtype}")
        m_splits = m_splits.tolist()
    if not isinstance(m_splits, (list, tuple)) or not all(type(m) is int for m in m_splits):
        raise TypeError("grouped_scaled_mm(): m_splits must be a list of ints (or a CPU tensor of integers)")
    if len(m_splits) != E:
        raise ValueError(f"grouped_scaled_mm(): mat2 has {E} matrices, m_splits {len(m_splits)} entries")
    if min(m_splits) < 0 or sum(m_splits) != T:
        raise ValueError(f"grouped_scaled_mm(): m_splits must be non-negative and add up to the {T} rows of input, got a sum of "
                         f"{sum(m_splits)}")
    return list(m_splits)


def _group_scale(name: str, t: torch.Tensor, E: int) -> int:
    """Stride of a scale over the groups: 0 for one element, else of an [E] tensor."""
    if t.numel() == 1:
        return 0
    if tuple(t.shape) != (E,):
        raise ValueError(f"grouped_scaled_mm(): {name} must have one element or shape {(E,)}, got {tuple(t.shape)}")
    return t.stride(0)


def _plainly_valid(input, mat2, scale_a, scale_b, scale_result, out_dtype, out) -> bool:
    """Whether the checks of a scaled_mm call would let every group pass as it is, seen from the whole call: the usual layouts
    and dtypes. False says nothing; the checks themselves decide then (15 us more)."""
    if input.dim() != 2 or scale_result is not None or out is not None or out_dtype not in _PLAIN_OUT or input.dtype not in NAME_OF or \
            mat2.dtype not in NAME_OF or (input.dtype == E5M2 and mat2.dtype == E5M2):
        return False
    (T, K), (E, K2, N) = input.shape, mat2.shape
    (lda, unit), (gsb, unit2, ldb) = input.stride(), mat2.stride()
    index = input.get_device()
    return (K == K2 and K % 16 == 0 and N % 16 == 0 and T > 1 and N > 1 and K > 1 and unit == 1 and unit2 == 1 and lda >= K and ldb >= K
            and not (lda | ldb | gsb | input.data_ptr() | mat2.data_ptr()) & 15 and index >= 0 and index == mat2.get_device()
            and index == scale_a.get_device() and index == scale_b.get_device() and scale_a.dtype == scale_b.dtype == torch.float32)


def _scratch(L, input, kernel, sizes, plan):
    """(tensor or None, pointer or None, bytes) of the scratch memory: for all groups at once (about four times the operands), where
    the device has too little left for that for one group after the other, as a loop of scaled_mm calls would have it, else none."""
    n = L.mmb200_grouped_workspace_bytes(*sizes, *plan)
    while n:
        try:
            ws = input.new_empty(n, dtype=torch.uint8)
            return ws, ws.data_ptr(), n
        except torch.OutOfMemoryError:
            one_by_one = L.mmb200_grouped_workspace_bytes_one_by_one(*sizes)
            if one_by_one >= n and kernel != "auto":
                raise                                    # a request for the fast kernels by name
            n = one_by_one if one_by_one < n else 0
    return None, None, 0


def grouped_scaled_mm(input, mat2, m_splits, scale_a, scale_b, scale_result=None, out_dtype=None, use_fast_accum=False, *,
                      out=None, profile=None, splitk="auto", backend="auto"):
    """scaled_mm of every group of rows, bit for bit: the first m_splits[0] rows of input [T, K] with mat2[0], the next
    m_splits[1] rows with mat2[1], and so on.

    mat2: [E, K, N] FP8, every matrix column-major (w.transpose(1, 2) of [E, N, K] weights). m_splits: E host integers that
    add up to T; groups may be empty. scale_a, scale_b: fp32, one element or one per group ([E]). out: a row-major [T, N]
    tensor of the output dtype to write into. profile, splitk, use_fast_accum, scale_result, out_dtype, backend and every
    raise: scaled_mm's; splitk="auto" decides for every group by its own number of rows. E <= 4096. Returns [T, N]."""
    fast = use_fast_accum
    _check_argument_types(input, mat2, scale_a, scale_b, None, scale_result, out_dtype, fast, out)
    if mat2.dim() != 3:
        raise ValueError(f"grouped_scaled_mm(): mat2 must be [E, K, N], got {tuple(mat2.shape)}")
    if input.dim() != 2:
        raise ReferenceRejectsError("mat1 must be a matrix")
    E, N, (T, K) = mat2.shape[0], mat2.shape[2], input.shape
    if E < 1 or E > MAX_GROUPS:
        raise ValueError(f"grouped_scaled_mm(): between 1 and {MAX_GROUPS} groups, got {E}")
    if max(T, N, K) >= 1 << 31:
        raise ValueError(f"grouped_scaled_mm(): sizes are below 2^31, got {T} rows, N = {N}, K = {K}")
    sizes = _sizes(m_splits, E, T)
    if scale_a.is_neg() or scale_b.is_neg():
        scale_a, scale_b = scale_a.resolve_neg(), scale_b.resolve_neg()
    sa, sb = _group_scale("scale_a", scale_a, E), _group_scale("scale_b", scale_b, E)
    plain = _plainly_valid(input, mat2, scale_a, scale_b, scale_result, out_dtype, out)
    if plain:
        scaling, od = "tensorwise", out_dtype
    else:
        w0 = mat2[0]
        scaling, od = _check_like_torch(input, w0, scale_a if scale_a.numel() == 1 else scale_a[:1],
                                        scale_b if scale_b.numel() == 1 else scale_b[:1], None, scale_result, out_dtype, out)
    prof = get_profile(profile)
    preset = get_preset(prof.preset)
    if out is not None and (tuple(out.shape) != (T, N) or (N > 1 and out.stride(1) != 1) or (T > 1 and out.stride(0) < N)):
        raise ValueError(f"grouped_scaled_mm(): out must be a row-major tensor of shape {(T, N)}, got shape {tuple(out.shape)} with "
                         f"strides {tuple(out.stride())}")
    if T == 0 or N == 0 or K == 0:
        return torch.zeros((T, N), dtype=od, device=input.device) if out is None else out.zero_()
    mat1 = input if plain else _check_like_cublas(input, w0, scaling, od)
    if E > 1 and mat2.stride(0) % 16:
        raise ReferenceRejectsError("CUBLAS_STATUS_NOT_SUPPORTED when calling cublasLtMatmul (operand pointer not 16-byte aligned)")
    fa, fb = fmt_of(mat1.dtype), fmt_of(mat2.dtype)
    rule = prof.rejection(fa, fb, od)
    if rule is not None:
        raise ReferenceRejectsError(f"{rule.message} [profile {prof.name}]")
    _check_scope(scaling, None, (mat1, mat2, scale_a, scale_b, scale_result))
    _emit_maturity(prof, preset)
    rows_std, weights_std = mat1.is_contiguous(), mat2.stride(1) == 1 and (mat2.stride(2) == K or N == 1)

    def plan_of(m):
        layout_std = weights_std and (rows_std or m == 1)      # one row is contiguous whatever the input's row stride
        d = resolve_splitk(m, N, K, a_dtype=mat1.dtype, b_dtype=mat2.dtype, out_dtype=od, use_fast_accum=fast, profile=prof, splitk=splitk,
                           layout_std=layout_std, dry=False)
        return d.S, check_plan(preset, K, d.S, d.scheme, fast)

    # (splits, scheme) of the groups by their rows; a split given by the caller holds for all of them
    split, plans = False, None
    if type(splitk) is int and splitk == 1:
        check_plan(preset, K, 1, "none", fast)
    elif isinstance(splitk, str) and splitk == "auto":
        plans = {m: plan_of(m) for m in set(sizes) if m}
        split = any(S > 1 for S, _ in plans.values())
    else:
        plan = plan_of(T)
        split = plan[0] > 1
        plans = dict.fromkeys(sizes, plan) if split else None
    kernel = _kernel_choice(backend)
    dev = mat1.device
    _require_device(dev)
    lda = mat1.stride(0) if T > 1 else K
    ldb = mat2.stride(2) if N > 1 else K
    y = input.new_empty((T, N), dtype=od) if out is None else out
    ints = ctypes.c_int * E
    rows, splits, schemes = ints(*sizes), None, None
    if split:
        splits = ints(*[plans[m][0] if m else 1 for m in sizes])
        schemes = ints(*[_lib.SCHEME_CODES[plans[m][1]] if m else 0 for m in sizes])
    keep_r, pr = (None, None) if scale_result is None else _scalar_ptr(scale_result, dev)
    L = _lib.load()
    with _on_device(dev):
        ws, ws_ptr, n = None, None, 0
        if kernel not in ("integer", "direct") and not preset.late_c and os.environ.get("MMAEMU_B200_WORKSPACE", "1") != "0":
            ws, ws_ptr, n = _scratch(L, input, kernel, (rows, splits, E, N, K), (_lib.FMT_CODES[fa], _lib.FMT_CODES[fb], preset.code,
                                                                                int(fast)))
        rc = L.mmb200_grouped_scaled_mm(mat1.data_ptr(), lda, _lib.FMT_CODES[fa], mat2.data_ptr(), ldb, mat2.stride(0) if E > 1 else 0,
                                        _lib.FMT_CODES[fb], y.data_ptr(), y.stride(0) if T > 1 else N,
                                        _lib.OUT_CODES[OUT_DTYPE_NAMES[od]], rows, splits, schemes, E, N, K, preset.code, int(fast),
                                        scale_a.data_ptr(), sa, scale_b.data_ptr(), sb, pr, _kernel_code(kernel), ws_ptr, n,
                                        _stream_ptr(dev))
        _lib.check("mmb200_grouped_scaled_mm", rc)
        if ws is not None and os.environ.get("MMAEMU_B200_CHECK_STATUS", "0") == "1":
            _lib.check("mmb200_grouped_status", L.mmb200_grouped_status(ws_ptr, _stream_ptr(dev)))
    del keep_r, ws
    return y


grouped_scaled_mm = torch.compiler.disable(grouped_scaled_mm)
