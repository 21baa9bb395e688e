"""grouped_scaled_mm on a B200 (-m gpu): the bits of the CPU oracle for every group, and of a loop of scaled_mm calls."""
import ctypes
import warnings

import numpy as np
import pytest
import torch

import datagen
import mmaemu_b200 as mm
from mmaemu_b200 import _lib
from oracle import oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
NPV = {4: (torch.int32, np.uint32), 2: (torch.int16, np.uint16), 1: (torch.uint8, np.uint8)}


def bits(t):
    tv, nv = NPV[t.element_size()]
    return t.detach().cpu().contiguous().view(tv).numpy().view(nv)


def operands(sizes, N, K, fa="e4m3", fb="e4m3", cls="gauss40", seed=0):
    rng = np.random.default_rng(seed)
    T, E = sum(sizes), len(sizes)
    a, w = datagen.codes(rng, max(T, 1), K, fa, cls)[:T], datagen.codes(rng, E * N, K, fb, cls, 1).reshape(E, N, K)
    return a, w, torch.from_numpy(a.copy()).to(DEV).view(F8[fa]), torch.from_numpy(w).to(DEV).view(F8[fb])


def loop(ta, tw, sizes, sa, sb, **kw):
    """scaled_mm, group by group."""
    got, start = [], 0
    for e, m in enumerate(sizes):
        one = lambda s: s if s.numel() == 1 else s[e]  # noqa: E731, B023
        got.append(mm.scaled_mm(ta[start:start + m], tw[e].t(), one(sa), one(sb), **kw))
        start += m
    return torch.cat(got)


def check(ta, tw, sizes, sa, sb, **kw):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        y = mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, **kw)
        want = loop(ta, tw, sizes, sa, sb, **kw)
    assert y.dtype == want.dtype and y.shape == want.shape
    bad = bits(y) != bits(want)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} outputs differ, first at {np.argwhere(bad)[0].tolist()}"
    return y


SCALES = (torch.tensor([0.5, 0.25, 3.0, 0.011, 1.0, 0.7]), torch.tensor([1.25, 0.5, 0.1, 2.0, 1.0, 0.3]))


def group_scales(E):
    return SCALES[0].repeat(E)[:E].to(DEV), SCALES[1].repeat(E)[:E].to(DEV)


SIZES = [[1], [5, 0, 11], [16, 16, 1, 0, 7], [0, 17, 128, 33], [129, 3, 200, 0, 64], [300, 260], [1] * 40, [0, 0, 90, 0]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}groups{sum(s)}rows")
@pytest.mark.parametrize("fa,fb", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2")])
@pytest.mark.parametrize("profile", ["hopper", "ada"])
@pytest.mark.parametrize("fast", [True, False])
def test_groups_against_the_oracle(sizes, fa, fb, profile, fast):
    N, K = 144, 400
    a, w, ta, tw = operands(sizes, N, K, fa, fb, seed=sum(sizes))
    sa, sb = group_scales(len(sizes))
    y = mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, out_dtype=torch.bfloat16, use_fast_accum=fast, profile=profile, splitk=1)
    start = 0
    for e, m in enumerate(sizes):
        if m:
            want = oracle.scaled_mm(a[start:start + m], w[e], float(sa[e]), float(sb[e]), out="bfloat16", fmt_a=fa, fmt_b=fb, preset=profile, fast=fast)
            bad = bits(y[start:start + m]) != want
            assert not bad.any(), f"group {e}: {int(bad.sum())} of {bad.size} outputs differ, first at {np.argwhere(bad)[0].tolist()}"
        start += m


@pytest.mark.parametrize("cls", datagen.CLASSES)
@pytest.mark.parametrize("fast", [True, False])
def test_groups_of_every_class_of_data(cls, fast):
    sizes = [20, 0, 140, 7]
    _, _, ta, tw = operands(sizes, 272, 512, cls=cls, seed=3)
    check(ta, tw, sizes, *group_scales(4), out_dtype=torch.float32, use_fast_accum=fast, profile="hopper", splitk=1)


@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16", "float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("sizes", [[9, 0, 3], [150, 20, 0, 33]])
def test_output_types_and_scale_result(out, sizes):
    _, _, ta, tw = operands(sizes, 160, 256, "e5m2", "e4m3", seed=5)
    sr = torch.tensor(0.37, device=DEV) if out.startswith("float8") else None
    check(ta, tw, sizes, *group_scales(len(sizes)), scale_result=sr, out_dtype=getattr(torch, out), profile="hopper", splitk=1)
    one = torch.tensor([0.01], device=DEV)
    check(ta, tw, sizes, one, one, scale_result=sr, out_dtype=getattr(torch, out), profile="ada", splitk=1, use_fast_accum=True)


@pytest.mark.parametrize("sizes", [[4, 12, 0, 1], [130, 0, 40]])
def test_special_codes_stay_in_their_rows_columns_and_groups(sizes):
    _, _, ta, tw = operands(sizes, 144, 272, "e5m2", "e4m3", seed=6)
    au, wu = ta.view(torch.uint8), tw.view(torch.uint8)
    au[1, 7], au[3, 0], au[sizes[0] + 1, 5] = 0x7C, 0x7F, 0xFC      # +Inf, NaN, -Inf
    second = next(e for e in range(1, len(sizes)) if sizes[e])       # the group of row sizes[0] + 1
    wu[0, 9, 3], wu[second, 20, 5], wu[second, 21, 5] = 0x7F, 0x00, 0x80
    y = check(ta, tw, sizes, *group_scales(len(sizes)), out_dtype=torch.float32, profile="hopper", splitk=1)
    assert torch.isnan(y[3]).all() and torch.isnan(y[0, 9]) and not torch.isnan(y[sizes[0], 9])
    assert torch.isnan(y[sizes[0] + 1, 20]) and torch.isnan(y[sizes[0] + 1, 21])    # Inf times zero


@pytest.mark.parametrize("profile", ["hopper", "hopper-te", "ada", "hopper-ws0"])
def test_split_decision_of_every_group(profile):
    """The automatic decision goes by each group's rows: some groups are split, in other ways, and some are not."""
    sizes, N, K = [16, 0, 128, 256, 64, 128], 512, 8192
    _, _, ta, tw = operands(sizes, N, K, cls="gauss1", seed=7)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        S = {m: mm.resolve_splitk(m, N, K, a_dtype=ta.dtype, b_dtype=tw.dtype, out_dtype=torch.bfloat16, use_fast_accum=False, profile=profile,
                                  dry=True).S for m in sizes if m}
    assert len(set(S.values())) > 1 or profile == "hopper-ws0"       # the case reaches both
    check(ta, tw, sizes, *group_scales(6), out_dtype=torch.bfloat16, profile=profile)


@pytest.mark.parametrize("fast", [True, False])
@pytest.mark.parametrize("profile,scheme", [("hopper", "contiguous"), ("ada", "serial"), ("ada", "pairwise")])
def test_explicit_splits(profile, scheme, fast):
    sizes = [3, 0, 140]
    _, _, ta, tw = operands(sizes, 128, 1040, seed=8)
    check(ta, tw, sizes, *group_scales(3), out_dtype=torch.float32, profile=profile, splitk=(3, scheme), use_fast_accum=fast)


@pytest.mark.parametrize("backend", ["cuda", "cuda:b200-integer", "cuda:b200-fast", "cuda:b200-direct"])
def test_kernel_families(backend):
    sizes = [5, 0, 140, 30]
    _, _, ta, tw = operands(sizes, 144, 272, seed=9)
    check(ta, tw, sizes, *group_scales(4), out_dtype=torch.bfloat16, profile="hopper", splitk=1, backend=backend)


@pytest.mark.parametrize("env", [{"MMAEMU_B200_TC_EPASS": "0"}, {"MMAEMU_B200_WORKSPACE": "0"}, {"MMAEMU_B200_ROW_GROUPS": "0"}, {"MMAEMU_B200_SLICES": "0"},
                                 {"MMAEMU_B200_CHECK_STATUS": "1"}])
@pytest.mark.parametrize("sizes", [[5, 0, 140, 30], [2, 9, 1]])
def test_environment_switches(env, sizes, monkeypatch):
    for k, v in env.items():
        monkeypatch.setenv(k, v)
    _, _, ta, tw = operands(sizes, 144, 272, seed=10)
    for fast in (True, False):
        check(ta, tw, sizes, *group_scales(len(sizes)), out_dtype=torch.bfloat16, profile="hopper", splitk=1, use_fast_accum=fast)


def test_late_accumulator_profile():
    """The experimental preset runs group by group on the integer kernel; slow accumulation is refused as in scaled_mm."""
    sizes = [5, 0, 30]
    _, _, ta, tw = operands(sizes, 48, 256, seed=15)
    kw = dict(out_dtype=torch.bfloat16, profile="b200-mma-sync-experimental", splitk=1)
    check(ta, tw, sizes, *group_scales(3), use_fast_accum=True, **kw)
    with pytest.raises(mm.UnsupportedFeatureError), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, *group_scales(3), **kw)


def test_many_groups():
    """More groups than one launch of the list kernel takes (512)."""
    rng = np.random.default_rng(16)
    sizes = [int(m) for m in rng.integers(0, 4, 1100)]
    sizes[700] = 40
    _, _, ta, tw = operands(sizes, 16, 64, seed=17)
    sa, sb = group_scales(len(sizes))
    y = mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, out_dtype=torch.bfloat16, profile="hopper", splitk=1)
    z = mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, out_dtype=torch.bfloat16, profile="hopper", splitk=1,
                             backend="cuda:b200-integer")
    assert np.array_equal(bits(y), bits(z))


@pytest.mark.parametrize("fast", [True, False])
@pytest.mark.parametrize("profile,fa", [("hopper", "e4m3"), ("hopper", "e5m2"), ("ada", "e4m3"), ("ada", "e5m2")])
def test_wide_outputs_and_mixed_sizes(profile, fa, fast):
    """Enough tiles for 256 columns per CTA, groups of few rows beside long ones."""
    sizes = [700, 3, 0, 128, 16, 300, 33, 900]
    _, _, ta, tw = operands(sizes, 2064, 144, fa=fa, seed=18)
    sa, sb = group_scales(8)
    y = mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, out_dtype=torch.float32, profile=profile, splitk=1, use_fast_accum=fast)
    z = mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, out_dtype=torch.float32, profile=profile, splitk=1, use_fast_accum=fast,
                             backend="cuda:b200-integer")
    assert np.array_equal(bits(y), bits(z))


def test_layouts():
    """Row strides of both operands, a group stride that leaves gaps, an input that is a view; out= with a row stride."""
    sizes, N, K = [5, 0, 140, 30], 144, 272
    _, _, ta, tw = operands(sizes, N, K, seed=11)
    T, E = sum(sizes), len(sizes)
    home = torch.zeros(T, K + 48, dtype=torch.uint8, device=DEV)
    home[:, 16:16 + K] = ta.view(torch.uint8)
    wide = torch.zeros(E, N + 3, K + 16, dtype=torch.uint8, device=DEV)
    wide[:, 1:N + 1, :K] = tw.view(torch.uint8)
    sa, sb = group_scales(E)
    kw = dict(out_dtype=torch.bfloat16, profile="hopper", splitk=1)
    want = loop(ta, tw, sizes, sa, sb, **kw)
    a2, w2 = home[:, 16:16 + K].view(ta.dtype), wide[:, 1:N + 1, :K].view(tw.dtype)
    y = mm.grouped_scaled_mm(a2, w2.transpose(1, 2), sizes, sa, sb, **kw)
    assert np.array_equal(bits(y), bits(want))
    strided = torch.stack([sa, sb], 1)
    y = mm.grouped_scaled_mm(a2, w2.transpose(1, 2), torch.tensor(sizes), strided[:, 0], strided[:, 1], **kw)
    assert np.array_equal(bits(y), bits(want))
    same = sa[:1].expand(E)                                          # one scale, expanded
    y = mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, same, same, **kw)
    assert np.array_equal(bits(y), bits(loop(ta, tw, sizes, same, same, **kw)))
    big = torch.full((T + 2, N + 7), 3.0, dtype=torch.bfloat16, device=DEV)
    out = big[1:T + 1, 4:N + 4]
    assert mm.grouped_scaled_mm(a2, w2.transpose(1, 2), sizes, sa, sb, out=out, profile="hopper", splitk=1) is out
    ref = torch.full_like(big, 3.0)
    ref[1:T + 1, 4:N + 4] = want
    assert np.array_equal(bits(big), bits(ref))
    shared = tw[:1].expand(E, N, K)                                  # one matrix for all groups
    y = mm.grouped_scaled_mm(ta, shared.transpose(1, 2), sizes, sa, sb, **kw)
    assert np.array_equal(bits(y), bits(loop(ta, shared, sizes, sa, sb, **kw)))


@pytest.mark.parametrize("K,lda,ldb,shift", [(67, 70, 69, 1), (400, 400, 401, 0), (128, 144, 128, 3), (1, 1, 1, 0)])
@pytest.mark.parametrize("sizes", [[5, 0, 140, 30], [3, 1, 2]])
def test_c_entry_point_takes_operands_of_any_alignment(K, lda, ldb, shift, sizes):
    """K, leading dimensions, group stride and base addresses that no 16-byte load fits (the Python entry point refuses them, as
    the emulated platform does)."""
    N, E, T = 50, len(sizes), sum(sizes)
    rng = np.random.default_rng(K)
    a, w = datagen.codes(rng, T, K, "e4m3", "gauss40"), datagen.codes(rng, E * N, K, "e4m3", "gauss40", 1)
    ha = torch.zeros(T * lda + 8, dtype=torch.uint8, device=DEV)
    hw = torch.zeros(E * (N * ldb + 5) + 8, dtype=torch.uint8, device=DEV)
    ha.as_strided((T, K), (lda, 1), shift).copy_(torch.from_numpy(a))
    hw.as_strided((E, N, K), (N * ldb + 5, ldb, 1), shift).copy_(torch.from_numpy(w).view(E, N, K))
    sa, sb = group_scales(E)
    L = _lib.load()
    ints = (ctypes.c_int * E)(*sizes)
    for fast in (0, 1):
        n = L.mmb200_grouped_workspace_bytes(ints, None, E, N, K, 0, 0, 32, fast)
        ws = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
        y = torch.zeros(T, N, dtype=torch.float32, device=DEV)
        rc = L.mmb200_grouped_scaled_mm(ha.data_ptr() + shift, lda, 0, hw.data_ptr() + shift, ldb, N * ldb + 5, 0, y.data_ptr(), N, 0, ints, None,
                                        None, E, N, K, 32, fast, sa.data_ptr(), 1, sb.data_ptr(), 1, None, 0, ws.data_ptr(), n,
                                        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        _lib.check("mmb200_grouped_scaled_mm", rc)
        start = 0
        for e, m in enumerate(sizes):
            if m:
                want = oracle.scaled_mm(a[start:start + m], w.reshape(E, N, K)[e], float(sa[e]), float(sb[e]), out="float32", preset="hopper", fast=bool(fast))
                assert np.array_equal(bits(y[start:start + m]), want), (fast, e)
            start += m


def test_empty_results():
    one = torch.ones(1, device=DEV)
    f = torch.float8_e4m3fn

    def z(*shape):
        return torch.zeros(shape, dtype=torch.uint8, device=DEV).view(f)
    kw = dict(out_dtype=torch.bfloat16, profile="hopper", splitk=1)
    assert mm.grouped_scaled_mm(z(0, 32), z(3, 16, 32).transpose(1, 2), [0, 0, 0], one, one, **kw).shape == (0, 16)
    assert mm.grouped_scaled_mm(z(4, 32), z(2, 0, 32).transpose(1, 2), [1, 3], one, one, **kw).shape == (4, 0)
    assert not mm.grouped_scaled_mm(z(4, 0), z(2, 16, 0).transpose(1, 2), [1, 3], one, one, **kw).any()


def test_streams_and_graphs():
    sizes = [5, 0, 140, 30]
    _, _, ta, tw = operands(sizes, 144, 272, seed=12)
    sa, sb = group_scales(4)
    kw = dict(out_dtype=torch.bfloat16, profile="hopper", splitk=1)

    def call():
        return mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, **kw)

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = call()
    torch.cuda.current_stream().wait_stream(side)
    assert np.array_equal(bits(y), bits(want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    _, _, tb, _ = operands(sizes, 144, 272, seed=13)
    ta.copy_(tb)
    graph.replay()
    torch.cuda.synchronize()
    got = y.clone()
    assert np.array_equal(bits(got), bits(call()))


@pytest.mark.parametrize("sizes", [[140, 0, 300], [1, 2, 3]])
def test_a_wait_that_runs_out_is_reported(sizes, monkeypatch):
    """$MMAEMU_B200_CHECK_STATUS=1 with the test hook of the bounded waits: an error, and the next call works. Groups of few
    rows run on kernels without waits."""
    monkeypatch.setenv("MMAEMU_B200_CHECK_STATUS", "1")
    monkeypatch.setenv("MMAEMU_B200_ROW_GROUPS", "0")                # 128-row tiles, whose copies are waited for
    _, _, ta, tw = operands(sizes, 256, 1024, seed=14)
    sa, sb = group_scales(3)
    kw = dict(out_dtype=torch.bfloat16, profile="hopper", splitk=1)
    L = _lib.load()
    L.mmb200_test_hooks(200, 16)
    try:
        if max(sizes) > 16:
            with pytest.raises(_lib.NativeError) as e:
                mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, **kw)
            assert e.value.status == _lib.ERR_TIMEOUT
        else:
            mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, **kw)
    finally:
        L.mmb200_test_hooks(0, 0)
    check(ta, tw, sizes, sa, sb, **kw)


@pytest.mark.parametrize("profile,fast,N,K,sizes", [("hopper", False, 2048, 8192, [1, 300, 0, 1]), ("hopper-te", True, 2048, 8192, [300, 1]),
                                                    ("ada", True, 512, 8192, [1, 600, 1]), ("ada", False, 128, 8192, [1, 0, 1, 1])])
def test_split_decisions_with_a_padded_input(profile, fast, N, K, sizes):
    """Rows of a wider buffer: a group of one row is contiguous for scaled_mm and split by the table, a longer one is not."""
    T = sum(sizes)
    _, _, ta, tw = operands(sizes, N, K, cls="gauss1", seed=19)
    home = torch.zeros(T, K + 32, dtype=torch.uint8, device=DEV)
    home[:, :K] = ta.view(torch.uint8)
    a2 = home[:, :K].view(ta.dtype)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        assert mm.resolve_splitk(1, N, K, a_dtype=ta.dtype, b_dtype=tw.dtype, out_dtype=torch.bfloat16, use_fast_accum=fast, profile=profile,
                                 dry=True).S > 1
    check(a2, tw, sizes, *group_scales(len(sizes)), out_dtype=torch.bfloat16, profile=profile, use_fast_accum=fast)


@pytest.mark.parametrize("splitk", [1, (2, "contiguous")])
@pytest.mark.parametrize("fast", [True, False])
def test_without_memory_for_the_scratch_of_all_groups(fast, splitk, monkeypatch):
    """Where the decoded operands of all groups do not fit, every group runs on the scratch-memory kernels by itself; without memory
    for that either, on the kernels that need none. The allocations fail because the test makes them fail."""
    monkeypatch.setenv("MMAEMU_B200_ROW_GROUPS", "0")                # 128-row tiles, whose operands are decoded into scratch memory
    sizes = [130, 0, 200, 40] * 6
    E = len(sizes)
    _, _, ta, tw = operands(sizes, 400, 272, seed=20)
    sa, sb = group_scales(E)
    kw = dict(out_dtype=torch.bfloat16, profile="hopper", splitk=splitk, use_fast_accum=fast)
    L = _lib.load()
    want = loop(ta, tw, sizes, sa, sb, **kw)
    before = L.mmb200_launch_count()
    loop(ta, tw, sizes, sa, sb, **kw)
    launches_of_loop = L.mmb200_launch_count() - before
    new_empty, asked, most = torch.Tensor.new_empty, [], [0]

    def limited(self, size, *args, dtype=None, **kwargs):
        if dtype is torch.uint8:
            asked.append(size)
            if size > most[0]:
                raise torch.OutOfMemoryError("no memory left")
        return new_empty(self, size, *args, dtype=dtype, **kwargs)

    monkeypatch.setattr(torch.Tensor, "new_empty", limited)
    one_by_one = L.mmb200_grouped_workspace_bytes_one_by_one((ctypes.c_int * E)(*sizes), None if splitk == 1 else (ctypes.c_int * E)(*[2, 1, 2, 2] * 6),
                                                             E, 400, 272)
    for backend in ("auto", "cuda:b200-fast"):
        most[0] = one_by_one
        asked.clear()
        before = L.mmb200_launch_count()
        y = mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, backend=backend, **kw)
        assert asked[-1] == one_by_one and (len(asked) == 2 or splitk != 1)
        assert L.mmb200_launch_count() - before == launches_of_loop
        assert np.array_equal(bits(y), bits(want))
    most[0] = 0
    assert np.array_equal(bits(mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, **kw)), bits(want))
    with pytest.raises(torch.OutOfMemoryError):
        mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, backend="cuda:b200-fast", **kw)


@pytest.mark.parametrize("one_by_one", [False, True])
@pytest.mark.parametrize("sizes", [[300, 5, 0, 3], [2, 130, 16]])
def test_a_wait_that_runs_out_in_one_group_leaves_the_others_written(sizes, one_by_one, monkeypatch):
    """The test hook makes the waits of the 128-row tiles run out; groups of few rows (K slices and their combination) do not wait
    and are written, in the fused launches and one after the other. The call's status word tells."""
    from mmaemu_b200 import grouped as grouped_module
    monkeypatch.setenv("MMAEMU_B200_ROW_GROUPS", "0")                # more than 16 rows: 128-row tiles, whose copies are waited for
    E, N, K = len(sizes), 256, 1024
    _, _, ta, tw = operands(sizes, N, K, seed=21)
    sa, sb = group_scales(E)
    kw = dict(profile="hopper", splitk=1)
    want = loop(ta, tw, sizes, sa, sb, out_dtype=torch.float32, **kw)
    out = torch.full((sum(sizes), N), 7.0, device=DEV)
    L = _lib.load()
    kept = []

    def scratch(L, input, kernel, shape, plan):
        n = L.mmb200_grouped_workspace_bytes_one_by_one(*shape) if one_by_one else L.mmb200_grouped_workspace_bytes(*shape, *plan)
        kept.append(torch.empty(n, dtype=torch.uint8, device=DEV))
        return kept[-1], kept[-1].data_ptr(), n

    monkeypatch.setattr(grouped_module, "_scratch", scratch)
    L.mmb200_test_hooks(200, 16)
    try:
        mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, out=out, **kw)
        torch.cuda.synchronize()
    finally:
        L.mmb200_test_hooks(0, 0)
    start = 0
    for m in sizes:
        rows = slice(start, start + m)
        assert np.array_equal(bits(out[rows]), bits(want[rows])) if m <= 16 else (out[rows] == 7.0).all(), m
        start += m
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert L.mmb200_grouped_status(kept[0].data_ptr(), st) == _lib.ERR_TIMEOUT
    mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, out=out, **kw)
    assert np.array_equal(bits(out), bits(want))
    assert L.mmb200_grouped_status(kept[1].data_ptr(), st) == _lib.OK


def test_scales_whose_sign_is_a_bit():
    """Scales that are the imaginary part of a conjugate: the sign is a bit of the tensor, not of the memory."""
    sizes, N, K = [5, 0, 140], 144, 272
    a, w, ta, tw = operands(sizes, N, K, seed=22)
    z = torch.complex(torch.zeros(3, device=DEV), torch.tensor([0.5, -2.0, 0.25], device=DEV)).conj().imag
    assert z.is_neg()
    plain = torch.tensor([-0.5, 2.0, -0.25], device=DEV)
    kw = dict(out_dtype=torch.float32, profile="hopper", splitk=1)
    want = loop(ta, tw, sizes, plain, plain[1:2], **kw)
    assert np.array_equal(bits(want[:5]), oracle.scaled_mm(a[:5], w[0], -0.5, 2.0, out="float32", preset="hopper", fast=False))
    assert np.array_equal(bits(mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, z, z[1:2], **kw)), bits(want))
    assert np.array_equal(bits(loop(ta, tw, sizes, z, z[1:2], **kw)), bits(want))


def test_offsets_beyond_32_bits():
    """More than 2^32 bytes of weights and more than 2^31 outputs."""
    E, N, K = 5, 16384, 65536
    base = operands([1], 256, K, seed=23)
    tw = base[3].view(torch.uint8).repeat(E, N // 256, 1)
    tw[-1] = 0x3C                                                    # the last group's weights: 1.5
    tw = tw.view(F8["e4m3"])
    assert tw.numel() > 2 ** 32
    sizes = [1, 0, 2, 0, 2]
    _, _, ta, _ = operands(sizes, 16, K, seed=24)
    check(ta, tw, sizes, *group_scales(E), out_dtype=torch.float32, profile="hopper", splitk=1)
    del tw, base
    sizes, N, K = [130000, 3, 1100], 16512, 32
    _, _, ta, tw = operands(sizes, N, K, seed=25)
    sa, sb = group_scales(3)
    kw = dict(out_dtype=torch.bfloat16, profile="hopper", splitk=1, use_fast_accum=True)
    y = mm.grouped_scaled_mm(ta, tw.transpose(1, 2), sizes, sa, sb, **kw)
    assert y.numel() > 2 ** 31
    for e, lo, hi in ((0, 0, 100), (0, 129900, 130000), (1, 130000, 130003), (2, 130003, 131103)):
        assert np.array_equal(bits(y[lo:hi]), bits(mm.scaled_mm(ta[lo:hi], tw[e].t(), sa[e], sb[e], **kw)))
