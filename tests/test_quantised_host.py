"""Refusals and host logic of quantize_int8, int8_scaled_mm, int8_grouped_scaled_mm and grouped_scaled_mm; no GPU."""
import ctypes

import pytest
import torch

import mmaemu_b200 as mm
from mmaemu_b200 import _lib

I8, F32 = torch.int8, torch.float32


def z(*shape, dtype=I8):
    return torch.zeros(shape, dtype=dtype)


def s(*shape):
    return torch.ones(shape, dtype=F32)


ONE = s(1)


def dense(**kw):
    args = dict(input=z(4, 32), mat2=z(16, 32).t(), scale_a=ONE, scale_b=ONE)
    args.update(kw)
    return mm.int8_scaled_mm(**args)


def grouped(**kw):
    args = dict(input=z(4, 32), mat2=z(3, 16, 32).transpose(1, 2), offs=z(3, dtype=torch.int32), scale_a=ONE, scale_b=ONE)
    args.update(kw)
    return mm.int8_grouped_scaled_mm(**args)


def fp8(**kw):
    f = torch.float8_e4m3fn
    args = dict(input=z(4, 32, dtype=f), mat2=z(3, 16, 32, dtype=f).transpose(1, 2), m_splits=[1, 0, 3], scale_a=ONE, scale_b=ONE,
                out_dtype=torch.bfloat16, splitk=1)
    args.update(kw)
    return mm.grouped_scaled_mm(**args)


def test_valid_calls_on_cpu_tensors_ask_for_a_device():
    for call in (dense, grouped, fp8, lambda: mm.quantize_int8(s(3, 4))):
        with pytest.raises(mm.BackendUnavailableError):
            call()


@pytest.mark.parametrize("kw,exc", [
    (dict(input=[1]), TypeError), (dict(mat2=None), TypeError), (dict(scale_a=1.0), TypeError), (dict(scale_b=1.0), TypeError),
    (dict(bias=3), TypeError), (dict(out=3), TypeError), (dict(out_dtype="bf16"), TypeError),
    (dict(input=z(4, 32, dtype=torch.uint8)), TypeError), (dict(mat2=z(16, 32, dtype=torch.float8_e4m3fn).t()), TypeError),
    (dict(input=z(32)), ValueError), (dict(input=z(4, 31)), ValueError),
    (dict(scale_a=s(3, 1)), ValueError), (dict(scale_a=s(4)), ValueError), (dict(scale_a=ONE.double()), ValueError),
    (dict(scale_b=ONE.half()), ValueError), (dict(bias=s(15)), ValueError), (dict(bias=z(16)), ValueError),
    (dict(out_dtype=torch.float8_e4m3fn), ValueError), (dict(out_dtype=torch.int32), ValueError),
    (dict(out=z(4, 15, dtype=F32)), ValueError), (dict(out=z(16, 4, dtype=F32).t()), ValueError),
    (dict(out=z(4, 16, dtype=F32), out_dtype=torch.bfloat16), ValueError),
])
@pytest.mark.parametrize("call", [dense, grouped])
def test_refusals(call, kw, exc):
    if call is grouped and isinstance(kw.get("bias"), torch.Tensor):
        kw = dict(bias=z(3, 16) if kw["bias"].dtype == I8 else s(3, 15))
    with pytest.raises(exc):
        call(**kw)


@pytest.mark.parametrize("kw", [
    dict(mat2=z(32, 16)), dict(scale_b=s(16, 1)), dict(scale_b=s(1, 15)), dict(mat2=z(16, 32)), dict(mat2=z(2, 16, 32).transpose(1, 2)),
    dict(input=z(1, 131072), mat2=z(1, 131072).t()), dict(input=torch.zeros(1, dtype=I8).expand((1 << 23) + 1, 1), mat2=z(1, 1)),
    dict(input=z(1, 1), mat2=z(1, 1).expand(1, (1 << 30) + 1)),
])
def test_refusals_of_the_dense_product(kw):
    with pytest.raises(ValueError):
        dense(**kw)


@pytest.mark.parametrize("kw,exc", [
    (dict(offs=[1, 2, 3]), TypeError), (dict(offs=z(3, dtype=torch.int64)), ValueError), (dict(offs=z(2, dtype=torch.int32)), ValueError),
    (dict(offs=z(3, 1, dtype=torch.int32)), ValueError), (dict(mat2=z(3, 32, 16)), ValueError), (dict(mat2=z(16, 32).t()), ValueError),
    (dict(scale_b=s(3, 16)), ValueError), (dict(scale_b=s(3, 1, 15)), ValueError), (dict(scale_b=s(3)), ValueError),
    (dict(bias=s(16)), ValueError),
    (dict(mat2=z(1, 16, 32).expand(4097, 16, 32).transpose(1, 2), offs=z(4097, dtype=torch.int32)), ValueError),
])
def test_refusals_of_the_grouped_product(kw, exc):
    with pytest.raises(exc):
        grouped(**kw)


def test_gradients_are_refused():
    w = ONE.clone().requires_grad_()
    for call in (dense, grouped, fp8):
        with pytest.raises(mm.UnsupportedFeatureError):
            call(scale_a=w)
    with pytest.raises(mm.UnsupportedFeatureError):
        mm.quantize_int8(torch.ones(2, 4, requires_grad=True))
    with torch.no_grad(), pytest.raises(mm.BackendUnavailableError):
        dense(scale_a=w)


@pytest.mark.parametrize("x,exc", [([1.0], TypeError), (z(3, 4), TypeError), (s(3, 4).double(), TypeError), (torch.tensor(1.0), ValueError),
                                   (s(1, 1).expand(1, (1 << 30) + 1), ValueError)])
def test_refusals_of_the_quantiser(x, exc):
    with pytest.raises(exc):
        mm.quantize_int8(x)


@pytest.mark.parametrize("kw,exc", [
    (dict(m_splits=[1, 3]), ValueError), (dict(m_splits=[1, 0, 2]), ValueError), (dict(m_splits=[5, -1, 0]), ValueError),
    (dict(m_splits=[1.0, 0, 3]), TypeError), (dict(m_splits=[True, 0, 3]), TypeError), (dict(m_splits=torch.tensor([1.0, 0, 3])), TypeError),
    (dict(m_splits="103"), TypeError), (dict(m_splits=None), TypeError),
    (dict(scale_a=s(2)), ValueError), (dict(scale_b=s(3, 1)), ValueError),
    (dict(mat2=z(16, 32, dtype=torch.float8_e4m3fn).t()), ValueError),
    (dict(mat2=z(0, 16, 32, dtype=torch.float8_e4m3fn).transpose(1, 2), m_splits=[]), ValueError),
    (dict(input=z(4, 24, dtype=torch.float8_e4m3fn)), mm.ReferenceRejectsError),
    (dict(input=z(4, 32, dtype=torch.float8_e5m2), mat2=z(3, 16, 32, dtype=torch.float8_e5m2).transpose(1, 2)), mm.ReferenceRejectsError),
    (dict(mat2=z(3, 32, 16, dtype=torch.float8_e4m3fn)), mm.ReferenceRejectsError),
    (dict(out=z(4, 15, dtype=torch.bfloat16)), ValueError), (dict(out=z(16, 4, dtype=torch.bfloat16).t()), ValueError),
    (dict(out=z(4, 16, dtype=torch.float16)), mm.ReferenceRejectsError), (dict(use_fast_accum=1), TypeError),
    (dict(input=z(1, 32, dtype=torch.float8_e4m3fn).expand(1 << 31, 32), m_splits=[1 << 31, 0, 0]), ValueError),
    (dict(profile="nothing"), Exception), (dict(splitk=(2, "serial")), ValueError), (dict(backend="cuda:h4"), mm.BackendUnavailableError),
    (dict(mat2=torch.zeros(3 * 520, dtype=torch.float8_e4m3fn).as_strided((3, 32, 16), (520, 1, 32))), mm.ReferenceRejectsError),
])
def test_refusals_of_the_emulated_grouped_product(kw, exc):
    with pytest.raises(exc):
        fp8(**kw)


def test_a_cpu_tensor_of_sizes_is_taken():
    with pytest.raises(mm.BackendUnavailableError):
        fp8(m_splits=torch.tensor([1, 0, 3]))
    with pytest.raises(mm.BackendUnavailableError):
        fp8(m_splits=(1, 0, 3), scale_a=s(3), scale_b=s(3))


# ---- the C ABI, without a device
@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as entry
    entry.build()
    return _lib.load()


def test_argument_checks_of_the_entry_points(lib):
    buf = ctypes.create_string_buffer(1024)
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def i8(a=p, lda=16, w=p, ldw=16, gsw=0, d=p, ldd=16, out=1, T=2, N=16, K=16, E=1, offs=0, sa=p, sas=0, sb=p, sbg=0, sbs=0, bias=0,
           bt=0, bg=0):
        return lib.mmb200_int8_scaled_mm(_lib.int8_args(a, lda, w, ldw, gsw, d, ldd, out, T, N, K, E, offs, sa, sas, sb, sbg, sbs, bias, bt, bg, 0,
                                                        0, 0, 0))

    assert lib.mmb200_int8_scaled_mm(None) == _lib.ERR_BAD_ARG
    for kw in (dict(T=-1), dict(N=-1), dict(K=-1), dict(E=-1), dict(E=2), dict(out=3), dict(out=-1), dict(bias=p, bt=0), dict(sa=0),
               dict(sb=0), dict(sas=-1), dict(sbs=-1), dict(sbg=-1), dict(gsw=-1), dict(bg=-1), dict(d=0), dict(a=0), dict(w=0),
               dict(lda=15), dict(ldw=15), dict(ldd=15), dict(d=p + 1)):
        assert i8(**kw) == _lib.ERR_BAD_ARG, kw
    for kw in (dict(K=131072, lda=131072, ldw=131072), dict(T=(1 << 23) + 1), dict(E=4097, offs=p), dict(N=(1 << 30) + 1, ldd=1 << 31),
               dict(N=(1 << 32) + 16), dict(T=1 << 40)):
        assert i8(**kw) == _lib.ERR_TOO_LARGE, kw
    assert i8(T=0) == _lib.OK and i8(N=0) == _lib.OK
    q = lib.mmb200_quantize_int8
    assert q(p, 16, 0, p, 16, p, 2, 16, None) == _lib.ERR_BAD_ARG and q(p, 16, 4, p, 16, p, 2, 16, None) == _lib.ERR_BAD_ARG
    assert q(p, 15, 1, p, 16, p, 2, 16, None) == _lib.ERR_BAD_ARG and q(p, 16, 1, p, 15, p, 2, 16, None) == _lib.ERR_BAD_ARG
    assert q(None, 16, 1, p, 16, p, 2, 16, None) == _lib.ERR_BAD_ARG and q(p, 16, 1, p, 16, None, 2, 16, None) == _lib.ERR_BAD_ARG
    assert q(p + 2, 16, 1, p, 16, p, 2, 16, None) == _lib.ERR_BAD_ARG and q(p, 16, 1, p, 16, p, -1, 16, None) == _lib.ERR_BAD_ARG
    assert q(p, 1 << 31, 1, p, 1 << 31, p, 2, (1 << 30) + 1, None) == _lib.ERR_TOO_LARGE
    assert q(p, 16, 1, p, 16, p, 0, 16, None) == _lib.OK


def test_scratch_memory_of_the_int8_products(lib):
    """Operands whose rows start on 16 bytes are read in place; others get rows of a multiple of 128 bytes."""
    need = lib.mmb200_int8_workspace_bytes
    assert need(1 << 12, 64, 1 << 13, 64, 640, 5, 10, 50, 3) == 0
    assert need((1 << 12) + 8, 64, 1 << 13, 64, 640, 5, 10, 50, 3) == 5 * 128
    assert need(1 << 12, 50, 1 << 13, 64, 640, 5, 10, 50, 3) == 5 * 128
    assert need(1 << 12, 50, 1 << 13, 64, 640, 1, 10, 50, 3) == 0               # one row: its stride is not used
    assert need(1 << 12, 64, 1 << 13, 50, 640, 5, 10, 50, 3) == 3 * 10 * 128
    assert need(1 << 12, 64, 1 << 13, 64, 648, 5, 10, 50, 3) == 3 * 10 * 128
    assert need(1 << 12, 64, 1 << 13, 64, 0, 5, 10, 130, 3) == 3 * 10 * 256     # weights shared by a stride of zero
    assert need(1 << 12, 64, 1 << 13, 64, 0, 5, 10, 50, 1) == 0
    assert need(1, 1, 1, 1, 1, 0, 10, 50, 3) == 0 and need(1, 1, 1, 1, 1, 5, 10, 0, 3) == 0


def test_argument_checks_of_the_emulated_grouped_entry_point(lib):
    buf = ctypes.create_string_buffer(1024)
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def call(m=(1, 0, 2), S=None, scheme=None, E=None, fmt=0, out=1, sa=p, K=16, sas=0, gs=16):
        ints = lambda v: None if v is None else (ctypes.c_int * len(v))(*v)  # noqa: E731
        return lib.mmb200_grouped_scaled_mm(p, 16, fmt, p, 16, gs, 0, p, 16, out, ints(m), ints(S), ints(scheme), len(m) if E is None else E, 16,
                                            K, 32, 1, sa, sas, p, 0, None, 0, None, 0, None)

    for kw in (dict(E=-1), dict(m=(1, -1)), dict(S=(1, 1, 1)), dict(fmt=7), dict(out=5), dict(sa=None), dict(sas=-1), dict(gs=-1), dict(K=-1),
               dict(S=(0, 1, 1), scheme=(0, 0, 0)), dict(S=(2, 1, 1), scheme=(0, 0, 0))):
        assert call(**kw) == _lib.ERR_BAD_ARG, kw
    assert call(m=(2 ** 31 - 1, 1)) == _lib.ERR_TOO_LARGE and call(m=(1,), E=4097) == _lib.ERR_TOO_LARGE
    assert call(m=(0, 0)) == _lib.OK
    m = (ctypes.c_int * 2)(100, 300)
    need = lib.mmb200_grouped_workspace_bytes
    assert need((ctypes.c_int * 2)(0, 300), None, 2, 64, 64, 0, 0, 32, 0) >= lib.mmb200_workspace_bytes(300, 64, 64)
    assert need(m, None, 2, 64, 64, 0, 0, 32, 0) > 0
    assert need((ctypes.c_int * 2)(0, 0), None, 2, 64, 64, 0, 0, 32, 0) == 0
    # the decoded operands of all groups would take 16 GB: group by group
    most = (ctypes.c_int * 64)(*[100] * 64)
    assert need(most, None, 64, 8192, 8192, 0, 0, 32, 1) < 1 << 30


@pytest.mark.parametrize("profile", ["hopper", "hopper-te", "ada"])
@pytest.mark.parametrize("pad", [0, 16])
@pytest.mark.parametrize("sizes", [[1, 1], [1, 128], [128, 0, 1], [16, 64, 1, 1], [1]])
def test_split_decisions_are_those_of_the_loop(sizes, pad, profile, monkeypatch):
    """splitk="auto": the layout that the decision goes by is each group's own (one row of a padded input is contiguous). What every
    group resolves to, or the error that the first undecided one raises, is what scaled_mm of the group has."""
    from mmaemu_b200 import api
    from mmaemu_b200 import grouped as grouped_module
    f, N, K = torch.float8_e4m3fn, 2048, 2048
    a, w = z(sum(sizes), K + pad, dtype=f)[:, :K], z(len(sizes), N, K, dtype=f)
    kw = dict(out_dtype=torch.bfloat16, profile=profile)
    seen = {}

    def record(M, *args, **kwargs):
        seen[M] = None
        d = mm.resolve_splitk(M, *args, **kwargs)
        seen[M] = (d.S, d.scheme, d.source)
        return d

    monkeypatch.setattr(api, "resolve_splitk", record)
    monkeypatch.setattr(grouped_module, "resolve_splitk", record)
    loop, start = {}, 0
    for e, m in enumerate(sizes):
        if m:
            with pytest.raises((mm.BackendUnavailableError, mm.SplitKUnknownError)):
                mm.scaled_mm(a[start:start + m], w[e].t(), ONE, ONE, **kw)
        start += m
    loop, seen = seen, {}
    undecided = any(d is None for d in loop.values())
    with pytest.raises(mm.SplitKUnknownError if undecided else mm.BackendUnavailableError):
        mm.grouped_scaled_mm(a, w.transpose(1, 2), sizes, ONE, ONE, **kw)
    assert undecided or seen == loop


def test_scratch_memory_of_groups_one_after_the_other(lib):
    """What a call asks for where there is no room for the decoded operands of all groups: the largest group's, by itself."""
    ints = lambda *v: (ctypes.c_int * len(v))(*v)  # noqa: E731
    one = lib.mmb200_grouped_workspace_bytes_one_by_one
    alone = [lib.mmb200_workspace_bytes_split(m, 4096, 4096, 1) for m in (128, 300)]
    assert one(ints(128, 0, 300, 128), None, 4, 4096, 4096) == 256 + max(alone)
    many = ints(*[128] * 32)
    assert one(many, None, 32, 4096, 4096) == 256 + alone[0] < lib.mmb200_grouped_workspace_bytes(many, None, 32, 4096, 4096, 0, 0, 32, 0) / 8
    split = lib.mmb200_workspace_bytes_split(128, 4096, 4096, 4)
    assert one(ints(128, 300), ints(4, 1), 2, 4096, 4096) == 256 + max(split, alone[1])
    assert one(ints(0, 0), None, 2, 64, 64) == 0 and one(None, None, 2, 64, 64) == 0 and one(ints(5), None, 0, 64, 64) == 0
