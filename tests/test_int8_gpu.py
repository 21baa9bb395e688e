"""int8 operators on a B200 (-m gpu): quantize_int8, int8_scaled_mm, int8_grouped_scaled_mm against plain computations in
64 bits.

Sums of int8 products are exact in fp64 (2^14 K < 2^53), so without a bias the result is known bit for bit: two fp32
roundings and the conversion. With a bias the 64-bit value is compared: the kernel rounds the sum to fp32 (2^-24 relative),
the product of the scales (2^-24), the fused multiply-add (2^-24) and the output (half a step), so
    |y - y64| <= eps_out / 2 |y64| + 3 * 2^-24 (|acc sa sb| + |y64|), and a little for the products of these errors."""
import ctypes
import math
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import mmaemu_b200 as mm
from mmaemu_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
VIEW = {4: torch.int32, 2: torch.int16}


def same(x, y):
    assert x.dtype == y.dtype and x.shape == y.shape
    v = VIEW[x.element_size()]
    bad = (x.contiguous().view(v) != y.contiguous().view(v))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outputs differ, first at {bad.nonzero()[0].tolist()}"


def codes(*shape, seed=0, lo=-128):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(lo, 128, shape, generator=g, device=DEV).to(torch.int8)


def scales(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(1000 + seed)
    return torch.rand(shape, generator=g, device=DEV) * 0.05 + 0.001


def want_bits(a, w, sa, sb, out):
    """a [M, K], w [N, K]; no bias: sum rounded to fp32, times the fp32 product of the scales, plus +0 (so a zero is +0, as
    scaled_mm has it), converted."""
    acc = a.double() @ w.double().t()
    y = acc.float() * (sa * sb) + 0.0
    y = torch.where(torch.isnan(y), torch.full_like(y, math.nan), y).to(out)
    return y


def check_close(y, a, w, sa, sb, bias):
    prod = (a.double() @ w.double().t()) * sa.double() * sb.double()
    ref = prod + bias.double()
    step = torch.finfo(y.dtype).eps / 2
    tol = step * ref.abs() + 3.1 * 2.0 ** -24 * (prod.abs() + ref.abs()) + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    assert ((y.double() - ref).abs() <= tol).all()


SHAPES = [(1, 1, 1), (1, 16, 16), (2, 8, 15), (3, 100, 31), (16, 128, 128), (16, 4096, 512), (17, 129, 127), (32, 256, 4096), (33, 64, 129),
          (64, 300, 1000), (65, 127, 2048), (100, 1003, 333), (128, 128, 16384), (129, 384, 640), (200, 2064, 1936), (256, 128, 128),
          (257, 640, 256), (300, 129, 65), (517, 1003, 2001), (1024, 1024, 1024), (5, 24576, 96), (2000, 16, 272)]


@pytest.mark.parametrize("out", DT)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_bits(M, N, K, out):
    a, w = codes(M, K, seed=M), codes(N, K, seed=N + 1)
    sa, sb = scales(M, 1, seed=K), scales(1, N, seed=K + 1)
    same(mm.int8_scaled_mm(a, w.t(), sa, sb, out_dtype=DT[out]), want_bits(a, w, sa, sb, DT[out]))


# every kernel, by the rule's choice: (kind, rows of a tile, parts of K) -> rows, channels, K; a worker's second and third tile,
# ragged rows, channels and K among them
KERNELS = [((0, 16, 1), 40, 300, 100), ((0, 16, 2), 1, 5622, 2083), ((0, 16, 4), 1, 5000, 2000), ((0, 16, 4), 300, 16, 2000), ((0, 16, 8), 7, 130, 2001),
           ((0, 16, 1), 3000, 16, 48), ((0, 16, 1), 17, 5000, 2000), ((0, 16, 1), 1500, 16, 2000), ((0, 32, 1), 5000, 16, 40),
           ((0, 32, 2), 17, 5676, 2475), ((0, 32, 4), 700, 16, 2000), ((0, 32, 8), 300, 17, 5000), ((0, 32, 8), 700, 16, 5000),
           ((0, 64, 1), 33, 20000, 17), ((0, 64, 2), 4631, 16, 3445), ((0, 64, 4), 3000, 16, 5000), ((0, 64, 8), 1500, 16, 5000),
           ((1, 64, 1), 65, 20000, 130), ((1, 128, 1), 1000, 2064, 1936), ((1, 128, 1), 1030, 5000, 300), ((1, 256, 1), 5000, 500, 1000),
           ((2, 256, 1), 2050, 5000, 300), ((2, 256, 1), 2000, 8200, 528)]
RAGGED = [((0, 16, 8), [0, 33, 0, 1], 16, 5000), ((0, 32, 8), [100, 0, 200], 16, 5000), ((0, 64, 1), [60, 0, 40], 9000, 16), ((1, 64, 1), [25, 0, 70, 3] * 10, 2000, 500),
          ((1, 128, 1), [300, 0, 1, 128, 129, 900, 42, 600], 4100, 300), ((1, 256, 1), [3, 257, 256, 0, 484, 0, 0, 0], 2000, 1000),
          ((2, 256, 1), [1, 800, 256, 0, 1300, 33, 1610], 2050, 1040)]


def kind_of(T, N, K, E=1, ragged=0):
    c = _lib.load().mmb200_int8_kernel_for(T, N, K, E, ragged)
    return c >> 16, (c >> 4) & 0xFFF, c & 15


@pytest.mark.parametrize("out", DT)
@pytest.mark.parametrize("kind,M,N,K", KERNELS, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_every_kernel(kind, M, N, K, out):
    assert kind_of(M, N, K) == kind
    a, w = codes(M, K, seed=M), codes(N, K, seed=N + 1)
    sa, sb = scales(M, 1, seed=K), scales(1, N, seed=K + 1)
    for _ in range(2):
        same(mm.int8_scaled_mm(a, w.t(), sa, sb, out_dtype=DT[out]), want_bits(a, w, sa, sb, DT[out]))


@pytest.mark.parametrize("kind,sizes,N,K", RAGGED, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else None)
@pytest.mark.parametrize("spare", [0, 37])
def test_every_kernel_with_ragged_groups(kind, sizes, N, K, spare):
    E, T = len(sizes), sum(sizes) + spare
    if not spare:
        assert kind_of(T, N, K, E, 1) == kind
    a, w = codes(T, K, seed=T), codes(E, N, K, seed=N)
    sa, sb = scales(T, 1, seed=1), scales(E, 1, N, seed=2)
    ends = torch.tensor(sizes, device=DEV).cumsum(0).to(torch.int32)
    same(mm.int8_grouped_scaled_mm(a, w.transpose(1, 2), ends, sa, sb), grouped_want(a, w, ends.tolist(), sa, sb, torch.bfloat16))


@pytest.mark.parametrize("M", [1, 16, 130, 300])
@pytest.mark.parametrize("K", [131071, 131056])
def test_largest_sums(M, K):
    """-128 times -128 over the largest K: 2^14 K, just below 2^31; and its negative."""
    a = torch.full((M, K), -128, dtype=torch.int8, device=DEV)
    w = torch.full((40, K), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    one = torch.ones(1, device=DEV)
    y = mm.int8_scaled_mm(a, w.t(), one, one, out_dtype=torch.float32)
    same(y, want_bits(a, w, one, one, torch.float32))
    assert y[0, 0] == float(16384 * K)


@pytest.mark.parametrize("M,N,K", [(7, 100, 300), (130, 260, 500), (300, 128, 1024)])
@pytest.mark.parametrize("bias", DT)
@pytest.mark.parametrize("out", DT)
def test_bias(M, N, K, bias, out):
    a, w = codes(M, K, seed=1), codes(N, K, seed=2)
    sa, sb = scales(M, 1, seed=3) * 0.01, scales(1, N, seed=4)
    b = (torch.randn(N, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)) * 3).to(DT[bias])
    check_close(mm.int8_scaled_mm(a, w.t(), sa, sb, b, DT[out]), a, w, sa, sb, b)
    big = torch.randn(2 * N, device=DEV).to(DT[bias])[::2]           # a strided bias
    check_close(mm.int8_scaled_mm(a, w.t(), sa, sb, big, DT[out]), a, w, sa, sb, big)


@pytest.mark.parametrize("M", [4, 200])
def test_scales_of_every_form(M):
    N, K = 144, 256
    a, w = codes(M, K, seed=1), codes(N, K, seed=2)
    row, col = scales(M, 1, seed=3), scales(1, N, seed=4)
    strided_row, strided_col = scales(M, 5, seed=6)[:, 2:3], scales(3, N * 2, seed=7)[1:2, ::2]
    for sa in (row, strided_row, row[:1, 0], row[0, 0], row[:1]):
        for sb in (col, strided_col, col[0, :1], col[0, 0], col[:, :1]):
            same(mm.int8_scaled_mm(a, w.t(), sa, sb), want_bits(a, w, sa, sb, torch.bfloat16))


def test_scales_that_are_not_finite():
    M, N, K = 20, 40, 64
    a, w = codes(M, K, seed=1), codes(N, K, seed=2)
    a[3] = 0
    sa, sb = scales(M, 1, seed=3), scales(1, N, seed=4)
    sa[3], sa[5], sb[0, 7], sa[9] = math.inf, math.nan, math.inf, 0.0
    for out in DT.values():
        y, want = mm.int8_scaled_mm(a, w.t(), sa, sb, out_dtype=out), want_bits(a, w, sa, sb, out)
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        same(torch.nan_to_num(y), torch.nan_to_num(want))
        v = y[5, 0].view(VIEW[y.element_size()]).item() & (0xFFFFFFFF if out == torch.float32 else 0xFFFF)
        assert v == (0x7FFFFFFF if out == torch.float32 else 0x7FFF)          # the framework's NaN


@pytest.mark.parametrize("M,N,K", [(5, 48, 100), (70, 130, 256), (260, 200, 97)])
@pytest.mark.parametrize("off_a,off_w,pad_a,pad_w", [(0, 0, 0, 0), (16, 32, 16, 48), (1, 0, 0, 0), (0, 3, 0, 0), (0, 0, 7, 0), (0, 0, 0, 1), (5, 9, 11, 13)])
def test_any_alignment_and_stride(M, N, K, off_a, off_w, pad_a, pad_w):
    ha, hw = codes(M * (K + pad_a) + off_a + 64, seed=1), codes(N * (K + pad_w) + off_w + 64, seed=2)
    a = ha.as_strided((M, K), (K + pad_a, 1), off_a)
    w = hw.as_strided((N, K), (K + pad_w, 1), off_w)
    sa, sb = scales(M, 1, seed=3), scales(1, N, seed=4)
    same(mm.int8_scaled_mm(a, w.t(), sa, sb, out_dtype=torch.float32), want_bits(a, w, sa, sb, torch.float32))


def test_operands_without_unit_stride_and_overlapping_rows():
    a, w = codes(96, 40, seed=1), codes(64, 96, seed=2)
    sa, sb = scales(40, 1, seed=3), scales(1, 64, seed=4)
    same(mm.int8_scaled_mm(a.t(), w.t(), sa, sb), want_bits(a.t(), w, sa, sb, torch.bfloat16))     # column-major input
    row = codes(1, 96, seed=5).expand(40, 96)                                                        # one row, repeated
    same(mm.int8_scaled_mm(row, w.t(), sa, sb), want_bits(row, w, sa, sb, torch.bfloat16))
    col = codes(1, 96, seed=6).expand(64, 96)
    same(mm.int8_scaled_mm(row, col.t(), sa, sb), want_bits(row, col, sa, sb, torch.bfloat16))


@pytest.mark.parametrize("out", DT)
@pytest.mark.parametrize("M,N", [(9, 33), (140, 130), (300, 257)])
def test_out_argument(M, N, out):
    """out= with any row stride and offset: written in place, nothing around it touched."""
    K = 192
    a, w = codes(M, K, seed=1), codes(N, K, seed=2)
    sa, sb = scales(M, 1, seed=3), scales(1, N, seed=4)
    home = torch.full((M + 2, N + 5), 7.0, dtype=DT[out], device=DEV)
    y = home[1:M + 1, 3:N + 3]
    assert mm.int8_scaled_mm(a, w.t(), sa, sb, out=y) is y
    want = torch.full_like(home, 7.0)
    want[1:M + 1, 3:N + 3] = want_bits(a, w, sa, sb, DT[out])
    same(home, want)


def test_empty_sizes():
    one = torch.ones(1, device=DEV)
    for M, N, K in ((0, 16, 16), (16, 0, 16), (0, 0, 0)):
        assert mm.int8_scaled_mm(codes(M, K), codes(N, K).t(), one, one).shape == (M, N)
    bias = torch.arange(24, device=DEV, dtype=torch.float32)
    y = mm.int8_scaled_mm(codes(20, 0), codes(24, 0).t(), one, one, bias, torch.float32)
    assert torch.equal(y, bias.expand(20, 24))                       # an empty sum is zero
    for M, N in ((300, 24), (1000, 2064), (2050, 5000)):
        assert not mm.int8_scaled_mm(codes(M, 0), codes(N, 0).t(), one, one).any()
    ends = torch.tensor([3, 900], dtype=torch.int32, device=DEV)
    assert not mm.int8_grouped_scaled_mm(codes(1000, 0), codes(2, 2000, 0).transpose(1, 2), ends, one, one).any()


# ---------------------------------------------------------------------------------------------------------------
def grouped_want(a, w, ends, sa, sb, out):
    T, N = a.shape[0], w.shape[1]
    y = torch.zeros((T, N), dtype=out, device=DEV)
    start = 0
    for e, end in enumerate(ends):
        if end > start:
            rs = sa if sa.numel() == 1 else sa[start:end]
            y[start:end] = want_bits(a[start:end], w[e], rs, sb if sb.numel() == 1 else sb[e], out)
        start = max(start, end)
    return y


GROUPS = [[1], [0, 0, 5], [16, 16, 16], [17, 0, 1, 31, 0], [128, 129, 127], [256, 1, 255, 300], [600, 3], [2] * 70, [0] * 40 + [9] + [0] * 30,
          [33, 64, 65, 100, 0, 1], list(range(40)), [3, 0, 1] * 100]


@pytest.mark.parametrize("sizes", GROUPS, ids=lambda s: f"{len(s)}groups{sum(s)}rows")
@pytest.mark.parametrize("N,K,spare", [(128, 128, 0), (130, 272, 3), (1000, 100, 300)])
def test_grouped_bits(sizes, N, K, spare):
    E, T = len(sizes), sum(sizes) + spare
    a, w = codes(T, K, seed=T), codes(E, N, K, seed=N)
    sa, sb = scales(T, 1, seed=1), scales(E, 1, N, seed=2)
    ends = torch.tensor(sizes, device=DEV).cumsum(0).to(torch.int32)
    want = grouped_want(a, w, ends.tolist(), sa, sb, torch.bfloat16)
    same(mm.int8_grouped_scaled_mm(a, w.transpose(1, 2), ends, sa, sb), want)
    # rows behind the last group keep what out= holds
    out = torch.full((T, N), 5.0, dtype=torch.bfloat16, device=DEV)
    assert mm.int8_grouped_scaled_mm(a, w.transpose(1, 2), ends, sa, sb, out=out) is out
    want[sum(sizes):] = 5.0
    same(out, want)


@pytest.mark.parametrize("ends", [[-5, 10, 4, 40], [50, 20, 30, 45], [1000, 3, 2000, 1], [0, 0, 0, 0], [-1, -2, -3, -4], [2 ** 31 - 1] * 4,
                                  [-2 ** 31, 45, -2 ** 31, 45]])
def test_grouped_ends_of_any_value(ends):
    """Ends that decrease, are negative or pass the rows: a running maximum inside [0, T]."""
    T, N, K = 45, 48, 64
    a, w = codes(T, K, seed=1), codes(4, N, K, seed=2)
    sa, sb = scales(T, 1, seed=3), scales(4, 1, N, seed=4)
    meant, top = [], 0
    for e in ends:
        top = max(top, min(max(e, 0), T))
        meant.append(top)
    offs = torch.tensor(ends, dtype=torch.int32, device=DEV)
    same(mm.int8_grouped_scaled_mm(a, w.transpose(1, 2), offs, sa, sb), grouped_want(a, w, meant, sa, sb, torch.bfloat16))


@pytest.mark.parametrize("out", DT)
@pytest.mark.parametrize("sizes", [[3, 0, 20], [200, 90, 0, 60]])
def test_grouped_bias_scales_and_types(sizes, out):
    E, T, N, K = len(sizes), sum(sizes), 200, 144
    a, w = codes(T, K, seed=1), codes(E, N, K, seed=2)
    one = torch.full((1,), 0.0007, device=DEV)
    ends = torch.tensor(sizes, device=DEV).cumsum(0).to(torch.int32)
    wt = w.transpose(1, 2)
    same(mm.int8_grouped_scaled_mm(a, wt, ends, one, one * 3, out_dtype=DT[out]), grouped_want(a, w, ends.tolist(), one, one * 3, DT[out]))
    sb = scales(E, 1, 2 * N, seed=5)[:, :, ::2]
    same(mm.int8_grouped_scaled_mm(a, wt, ends, one, sb, out_dtype=DT[out]), grouped_want(a, w, ends.tolist(), one, sb, DT[out]))
    bias = torch.randn(E, N, device=DEV).to(DT[out])
    y = mm.int8_grouped_scaled_mm(a, wt, ends, one, sb, bias, DT[out])
    start = 0
    for e, end in enumerate(ends.tolist()):
        if end > start:
            check_close(y[start:end], a[start:end], w[e], one, sb[e], bias[e])
        start = end


@pytest.mark.parametrize("make", ["offset", "row stride", "group stride", "shared weights", "odd K"])
def test_grouped_operands_of_any_layout(make):
    sizes = [5, 0, 40, 3]
    E, T, N, K = 4, 48, 72, 33 if make == "odd K" else 96
    a = codes(T, K, seed=1)
    home = codes(E * (N + 4) * (K + 16) + 64, seed=2)
    strides = {"offset": (N * K, K, 3), "row stride": (N * (K + 5), K + 5, 0), "group stride": (N * K + 7, K, 0),
               "shared weights": (0, K, 0), "odd K": (N * K, K, 0)}[make]
    w = home.as_strided((E, N, K), (strides[0], strides[1], 1), strides[2])
    sa, sb = scales(T, 1, seed=3), scales(E, 1, N, seed=4)
    ends = torch.tensor(sizes, device=DEV).cumsum(0).to(torch.int32)
    same(mm.int8_grouped_scaled_mm(a, w.transpose(1, 2), ends, sa, sb), grouped_want(a, w, ends.tolist(), sa, sb, torch.bfloat16))


@pytest.mark.parametrize("T,N", [(5000, 16), (5000, 2000), (300000, 16)])
def test_as_many_groups_as_there_may_be(T, N):
    """4096 groups, most of them empty or of a row; tiles per CTA and persistent CTAs."""
    E, K = 4096, 48
    g = torch.Generator().manual_seed(T)
    at = torch.sort(torch.randint(0, T + 1, (E,), generator=g))[0]
    at[-1] = T - 3
    at = at.clamp(max=T - 3)
    a, w = codes(T, K, seed=1), codes(E, N, K, seed=2)
    sa, sb = scales(T, 1, seed=3), scales(E, 1, N, seed=4)
    y = mm.int8_grouped_scaled_mm(a, w.transpose(1, 2), at.to(torch.int32).to(DEV), sa, sb, out_dtype=torch.float32)
    e = torch.searchsorted(at, torch.arange(T), right=True).to(DEV)
    real = e < E
    e = e.clamp(max=E - 1)
    for lo in range(0, T, 4096):                                     # row by row in pieces: one weight matrix per row
        rows = slice(lo, min(T, lo + 4096))
        for c in range(0, N, 500):
            cols = slice(c, min(N, c + 500))
            acc = torch.einsum("tk,tnk->tn", a[rows].float(), w[:, cols][e[rows]].float())        # exact: at most 48 * 2^14
            want = acc * (sa[rows] * sb[e[rows], 0, cols]) + 0.0
            same(y[rows, cols], torch.where(real[rows, None], want, 0.0))


def test_grouped_without_groups_or_rows():
    one = torch.ones(1, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert not mm.int8_grouped_scaled_mm(codes(5, 32), codes(0, 16, 32).transpose(1, 2), none, one, one).any()
    ends = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert mm.int8_grouped_scaled_mm(codes(0, 32), codes(3, 16, 32).transpose(1, 2), ends, one, one).shape == (0, 16)
    assert not mm.int8_grouped_scaled_mm(codes(9, 32), codes(3, 16, 32).transpose(1, 2), ends, one, one).any()


# ---------------------------------------------------------------------------------------------------------------
def quantise_want(x):
    """Integer arithmetic on fp64 values: floor((254 |x| + amax) / (2 amax)), ties to even."""
    d = x.double()
    top = d.abs().amax(-1, keepdim=True)
    good = torch.isfinite(top)
    whole = torch.where(good & (top > 0), top, 1.0)
    twice = 254.0 * torch.where(good, d, 0.0).abs() + whole
    q = torch.floor(twice / (2 * whole))
    q = q - ((q * 2 * whole == twice) & (q % 2 == 1)).double()
    return (q * torch.sign(torch.where(good, d, 0.0))).to(torch.int8), torch.where(good, top / 127.0, math.nan)


def check_quantised(x):
    c, s = mm.quantize_int8(x)
    want_c, want_s = quantise_want(x)
    assert c.dtype == torch.int8 and c.shape == x.shape and c.is_contiguous()
    assert s.dtype == torch.float32 and s.shape == x.shape[:-1] + (1,)
    assert torch.equal(c, want_c), f"{int((c != want_c).sum())} codes differ"
    assert torch.equal(torch.isnan(s), torch.isnan(want_s))
    ok = ~torch.isnan(want_s)
    # one rounding to fp32: half a step, or half the smallest subnormal
    assert ((s[ok].double() - want_s[ok]).abs() <= 2.0 ** -24 * want_s[ok] + 2.0 ** -150).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 4096), (3, 7), (5, 64), (9, 129), (4, 511), (7, 512), (16, 513), (3, 2048), (2, 2049), (2, 4100), (3, 8192),
                                    (2, 8200), (1, 16384), (2, 16400), (2, 40000), (1000, 96), (517, 2001)])
def test_quantise(rows, K, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows * K)
    check_quantised((torch.randn(rows, K, generator=g, device=DEV) * torch.exp(torch.randn(rows, 1, generator=g, device=DEV))).to(DT[dtype]))


@pytest.mark.parametrize("dtype", DT)
def test_quantise_ties_and_borders(dtype):
    """Rows whose values lie on or next to the borders between codes."""
    half = torch.arange(-127, 127, device=DEV) + 0.5
    rows = []
    for top in (127.0, 63.5, 1.0, 448.0, 0.371, 3.0):
        x = (half * top / 127.0).to(DT[dtype])
        x[0] = top
        bits = x.view(VIEW[x.element_size()])
        rows += [x, (bits + 1).view(DT[dtype]).clone(), (bits - 1).view(DT[dtype]).clone()]
        for r in rows[-2:]:
            r[0] = top
    check_quantised(torch.stack(rows))


@pytest.mark.parametrize("dtype", DT)
def test_quantise_extreme_rows(dtype):
    t = DT[dtype]
    fi = torch.finfo(t)
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(12, 300, generator=g, device=DEV).clamp(-1, 1).to(t)
    x[0] = 0
    x[1] = -0.0
    x[2] = (x[2].double() * fi.max).to(t)
    x[3] = (x[3].double() * fi.tiny).to(t)                            # subnormal values
    x[4] = 0
    x[4, 7] = fi.smallest_normal
    x[5] = 0
    x[5, 8] = -fi.tiny * fi.eps                                       # the smallest number
    x[6, 3] = math.inf
    x[7, 299] = -math.inf
    x[8, 0] = math.nan
    x[9, :] = math.nan
    x[10] = fi.max
    check_quantised(x)
    c, s = mm.quantize_int8(x)
    assert not c[6:10].any() and torch.isnan(s[6:10]).all() and s[0] == 0 and s[1] == 0
    assert (s[8].view(torch.int32) == 0x7FFFFFFF).all()


@pytest.mark.parametrize("dtype", DT)
def test_quantise_layouts(dtype):
    t = DT[dtype]
    g = torch.Generator(device=DEV).manual_seed(4)
    home = torch.randn(40, 330, generator=g, device=DEV).to(t)
    check_quantised(home[:, 1:301])                                   # rows that are not 16-byte aligned
    check_quantised(home[::3, :256])
    check_quantised(home.t())                                         # no unit stride
    check_quantised(home.view(2, 20, 330)[:, 3:9])
    check_quantised(home[0].expand(5, 330))
    check_quantised(home[0])
    check_quantised(home.view(4, 10, 330).transpose(0, 1))
    assert mm.quantize_int8(home[:0])[0].shape == (0, 330)
    c, s = mm.quantize_int8(home[:, :0])
    assert c.shape == (40, 0) and s.shape == (40, 1) and not s.any()


# ---------------------------------------------------------------------------------------------------------------
def test_quantised_layer_and_experts_together():
    """quantise -> product -> quantise -> grouped product, as a quantised model runs them. Each code is off by at most half a
    step, amax / 254, so an output of K terms is off by at most sum |x| sw / 2 + |w| sx / 2 + K sx sw / 4."""
    g = torch.Generator(device=DEV).manual_seed(6)
    T, K, N, E, F = 70, 320, 264, 4, 136
    x, w = torch.randn(T, K, generator=g, device=DEV), torch.randn(N, K, generator=g, device=DEV)
    v = torch.randn(E, F, N, generator=g, device=DEV)
    xq, sx = mm.quantize_int8(x)
    wq, sw = mm.quantize_int8(w)
    h = mm.int8_scaled_mm(xq, wq.t(), sx, sw.t(), out_dtype=torch.float32)
    err = x.abs().double().sum(1, keepdim=True) * sw.double().t() / 2 + sx.double() * w.abs().double().sum(1)[None] / 2 + K * sx.double() * sw.double().t() / 4
    ref = x.double() @ w.double().t()
    assert ((h.double() - ref).abs() <= err * 1.001 + 1e-6 * ref.abs()).all()
    hq, sh = mm.quantize_int8(h)
    vq, sv = mm.quantize_int8(v)
    ends = torch.tensor([10, 10, 50, 70], dtype=torch.int32, device=DEV)
    y = mm.int8_grouped_scaled_mm(hq, vq.transpose(1, 2), ends, sh, sv.transpose(1, 2), out_dtype=torch.float32)
    same(y, grouped_want(hq, vq, ends.tolist(), sh, sv.transpose(1, 2), torch.float32))


def test_streams_and_graphs():
    """Calls run on the current stream; a captured run of all of them replays on new contents, new group ends among them."""
    T, K, N, E = 60, 256, 192, 3
    x = torch.randn(T, K, device=DEV)
    wq, w3 = codes(N, K, seed=1), codes(E, 40, N, seed=2)
    sw, s3 = scales(1, N, seed=3), scales(E, 1, 40, seed=4)
    ends = torch.tensor([20, 20, 60], dtype=torch.int32, device=DEV)

    def step():
        xq, sx = mm.quantize_int8(x)
        h = mm.int8_scaled_mm(xq, wq.t(), sx, sw)
        hq, sh = mm.quantize_int8(h)
        return mm.int8_grouped_scaled_mm(hq, w3.transpose(1, 2), ends, sh, s3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y_side = step()
    torch.cuda.current_stream().wait_stream(side)
    same(y_side, step())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for seed in (1, 2):
        x.copy_(torch.randn(T, K, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)))
        ends.copy_(torch.tensor([[7, 40, 41], [0, 60, 60]][seed - 1], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        same(got, step())


FRESH = """
import torch, mmaemu_b200 as mm
dev = torch.device("cuda:0")
x = torch.randn(70, 256, device=dev, dtype=torch.bfloat16)
w = torch.randint(-127, 128, (3, 192, 256), device=dev).to(torch.int8)
big = torch.randint(-127, 128, (2064, 256), device=dev).to(torch.int8)
ends = torch.tensor([20, 20, 70], dtype=torch.int32, device=dev)
one = torch.full((1,), 0.01, device=dev)
f8 = torch.float8_e4m3fn
xa, wa = x.to(f8), w.to(torch.bfloat16).to(f8)
xb = torch.randint(-127, 128, (1000, 256), device=dev).to(torch.int8)
def step():
    xq, sx = mm.quantize_int8(x)
    return (mm.int8_grouped_scaled_mm(xq, w.transpose(1, 2), ends, sx, one), mm.int8_scaled_mm(xq, w[0].t(), sx, one),
            mm.int8_scaled_mm(xb, big.t(), one, one),
            mm.grouped_scaled_mm(xa, wa.transpose(1, 2), [20, 0, 50], one, one, None, torch.bfloat16, profile="hopper", splitk=1))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("same")
"""


def test_the_first_calls_of_a_process_can_be_captured():
    """Nothing that a first call looks up or sets breaks a capture."""
    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, "-c", FRESH], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stderr[-2000:]


def test_calls_on_two_streams_at_once():
    """Two threads on streams of their own, every kind of kernel: no call sees the other's scratch memory or barriers."""
    shapes = [(7, 130, 2001), (65, 2000, 130), (300, 1000, 333), (1000, 2064, 520)]
    work = [(codes(M, K, seed=i), codes(N, K, seed=i + 9), scales(M, 1, seed=i), scales(1, N, seed=i + 1)) for i, (M, N, K) in enumerate(shapes)]
    want = [want_bits(*w, torch.bfloat16) for w in work]
    torch.cuda.synchronize()
    got = [None, None]

    def run(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[k] = [[mm.int8_scaled_mm(a, w.t(), sa, sb) for a, w, sa, sb in work] for _ in range(20)]
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        for round_ in got[k]:
            for y, w in zip(round_, want):
                same(y, w)


@pytest.mark.parametrize("M,N,K", [(4, 512, 2048)])
def test_status_check_after_every_call(M, N, K, monkeypatch):
    """$MMAEMU_B200_CHECK_STATUS=1: the call itself raises."""
    monkeypatch.setenv("MMAEMU_B200_CHECK_STATUS", "1")
    a, w, one = codes(M, K, seed=1), codes(N, K, seed=2), torch.ones(1, device=DEV)
    want = mm.int8_scaled_mm(a, w.t(), one, one)
    L = _lib.load()
    L.mmb200_test_hooks(200, 16)
    try:
        with pytest.raises(_lib.NativeError) as e:
            mm.int8_scaled_mm(a, w.t(), one, one)
        assert e.value.status == _lib.ERR_TIMEOUT
    finally:
        L.mmb200_test_hooks(0, 0)
    same(mm.int8_scaled_mm(a, w.t(), one, one), want)


@pytest.mark.parametrize("M,N,K", [(4, 512, 2048), (100, 512, 2048), (400, 512, 2048), (65, 20000, 1300), (1000, 2064, 1936), (5000, 500, 1000),
                                   (2000, 8200, 1280)])
def test_a_wait_that_runs_out_is_reported(M, N, K):
    """The test hook announces more bytes than arrive: the bounded waits run out, the call reports it, the next call works."""
    a, w = codes(M, K, seed=1), codes(N, K, seed=2)
    one = torch.ones(1, device=DEV)
    want = mm.int8_scaled_mm(a, w.t(), one, one)
    L = _lib.load()
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert L.mmb200_int8_status(st) == _lib.OK
    L.mmb200_test_hooks(200, 16)
    try:
        mm.int8_scaled_mm(a, w.t(), one, one)
        torch.cuda.synchronize()
    finally:
        L.mmb200_test_hooks(0, 0)
    assert L.mmb200_int8_status(st) == _lib.ERR_TIMEOUT
    assert L.mmb200_int8_status(st) == _lib.OK                       # read once
    same(mm.int8_scaled_mm(a, w.t(), one, one), want)


def test_a_checked_call_reports_its_own_waits_only(monkeypatch):
    """A wait that has run out in another call is neither raised by a checked call nor taken from the device's word by it, and
    the other way round."""
    M, N, K = 4, 512, 2048
    a, w, one = codes(M, K, seed=1), codes(N, K, seed=2), torch.ones(1, device=DEV)
    want = mm.int8_scaled_mm(a, w.t(), one, one)
    L = _lib.load()
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert L.mmb200_int8_status(st) == _lib.OK
    L.mmb200_test_hooks(200, 16)
    try:
        mm.int8_scaled_mm(a, w.t(), one, one)
        torch.cuda.synchronize()
    finally:
        L.mmb200_test_hooks(0, 0)
    monkeypatch.setenv("MMAEMU_B200_CHECK_STATUS", "1")
    got = []

    def run():
        with torch.cuda.stream(torch.cuda.Stream()):
            got.extend(mm.int8_scaled_mm(a, w.t(), one, one) for _ in range(10))

    threads = [threading.Thread(target=run) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 40
    for y in got:
        same(y, want)
    assert L.mmb200_int8_status(st) == _lib.ERR_TIMEOUT              # the unchecked call's
    L.mmb200_test_hooks(200, 16)
    try:
        for _ in range(70):                                          # more calls than there are words
            with pytest.raises(_lib.NativeError):
                mm.int8_scaled_mm(a, w.t(), one, one)
    finally:
        L.mmb200_test_hooks(0, 0)
    assert L.mmb200_int8_status(st) == _lib.OK
    same(mm.int8_scaled_mm(a, w.t(), one, one), want)


def negated(*shape, seed=0):
    """The imaginary part of a conjugate: a view whose sign is a bit of the tensor, and the same values in memory."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    v = torch.randn(*shape, dtype=torch.complex64, generator=g, device=DEV).conj().imag
    assert v.is_neg()
    return v, v.resolve_neg().contiguous()


def test_views_whose_sign_is_a_bit():
    for shape in ((6, 1), (6, 40)):
        x, plain = negated(*shape, seed=1)
        for got, want in zip(mm.quantize_int8(x), mm.quantize_int8(plain)):
            assert torch.equal(got, want)
        check_quantised(plain)
    M, N, K, E = 7, 33, 64, 2
    a, w, w3 = codes(M, K, seed=1), codes(N, K, seed=2), codes(E, N, K, seed=3)
    (va, sa), (vb, sb), (vc, sc), (v3, s3) = negated(M, 1, seed=2), negated(1, N, seed=3), negated(1, seed=4), negated(E, 1, N, seed=5)
    same(mm.int8_scaled_mm(a, w.t(), va, vb), want_bits(a, w, sa, sb, torch.bfloat16))
    same(mm.int8_scaled_mm(a, w.t(), vc, sb), want_bits(a, w, sc, sb, torch.bfloat16))
    same(mm.int8_scaled_mm(a, w[:1].t(), sa, sb[:, :1], vc), mm.int8_scaled_mm(a, w[:1].t(), sa, sb[:, :1], sc))
    ends = torch.tensor([3, 7], dtype=torch.int32, device=DEV)
    same(mm.int8_grouped_scaled_mm(a, w3.transpose(1, 2), ends, va, v3), grouped_want(a, w3, [3, 7], sa, s3, torch.bfloat16))
    with pytest.raises(ValueError):
        mm.int8_scaled_mm(a, w[:1].t(), sa, sb[:, :1], out=negated(M, 1)[0])


@pytest.mark.parametrize("layout", ["groups inside rows", "gap between groups", "overlapping groups", "one channel, strided groups"])
@pytest.mark.parametrize("sizes", [[5, 0, 40, 3], [300, 0, 129, 600]])
def test_grouped_weights_in_place_with_any_group_stride(layout, sizes):
    """Group strides that are below the row stride, no multiple of it, or below a matrix: read in place all the same."""
    E, T, N, K = 4, sum(sizes), 1 if "one channel" in layout else 272, 320
    strides = {"groups inside rows": (K, E * K), "gap between groups": (N * K + 48, K), "overlapping groups": (16, K),
               "one channel, strided groups": (48 + K, K)}[layout]
    a, home = codes(T, K, seed=1), codes(E * (N * K + 400), seed=2)
    w = home.as_strided((E, N, K), (*strides, 1))
    sa, sb = scales(T, 1, seed=3), scales(E, 1, N, seed=4)
    ends = torch.tensor(sizes, device=DEV).cumsum(0).to(torch.int32)
    assert _lib.load().mmb200_int8_workspace_bytes(a.data_ptr(), K, w.data_ptr(), strides[1], strides[0], T, N, K, E) == 0
    same(mm.int8_grouped_scaled_mm(a, w.transpose(1, 2), ends, sa, sb), grouped_want(a, w, ends.tolist(), sa, sb, torch.bfloat16))


def test_offsets_beyond_32_bits():
    """More than 2^31 outputs, input codes and quantised values; the first, middle and last rows are compared."""
    T, N, K = 131079, 20000, 48
    a, w = codes(T, K, seed=1), codes(N, K, seed=2)
    sa, sb = scales(T, 1, seed=3), scales(1, N, seed=4)
    ends = torch.tensor([70001, T - 5], dtype=torch.int32, device=DEV)
    y, z = mm.int8_scaled_mm(a, w.t(), sa, sb), mm.int8_grouped_scaled_mm(a, torch.stack([w, w.flip(0)]).transpose(1, 2), ends, sa, sb[0, 0])
    assert y.numel() > 2 ** 31
    for lo in (0, 69990, T - 40):
        rows = slice(lo, min(lo + 40, T))
        same(y[rows], want_bits(a[rows], w, sa[rows], sb, torch.bfloat16))
        first, second = (want_bits(a[rows], v, sa[rows], sb[0, 0], torch.bfloat16) for v in (w, w.flip(0)))
        row = torch.arange(T, device=DEV)[rows, None]
        same(z[rows], torch.where(row < 70001, first, torch.where(row < T - 5, second, 0.0)))
    del y, z
    T, K = 70001, 32768
    x = torch.empty(T, K, dtype=torch.float16, device=DEV)
    for lo in range(0, T, 10000):
        x[lo:lo + 10000].normal_(generator=torch.Generator(device=DEV).manual_seed(lo))
    xq, sx = mm.quantize_int8(x)
    assert xq.numel() > 2 ** 31
    for lo in (0, 65530, T - 20):
        rows = slice(lo, min(lo + 20, T))
        assert torch.equal(xq[rows], quantise_want(x[rows])[0]) and torch.equal(sx[rows], mm.quantize_int8(x[rows].clone())[1])
    w, sb = codes(40, K, seed=5), scales(1, 40, seed=6)
    y = mm.int8_scaled_mm(xq, w.t(), sx, sb)
    for lo in (0, 65530, T - 20):
        rows = slice(lo, min(lo + 20, T))
        same(y[rows], want_bits(xq[rows], w, sx[rows], sb, torch.bfloat16))


@pytest.mark.parametrize("dtype", DT)
def test_quantise_rows_of_one_repeated_value(dtype):
    """Rows of one value without a stride between them."""
    one = torch.tensor([[-0.75]], dtype=DT[dtype], device=DEV)
    check_quantised(one.expand(5, 1))
    check_quantised(one.expand(2, 300, 1))
    check_quantised(one.expand(5, 40))
    check_quantised(one[0].expand(7))
