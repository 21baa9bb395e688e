"""The quantised operators next to the emulated FP8 GEMM, as a program calls them, and their plain forms.

quantise   int8 codes and one scale per row (token or output channel) of fp32 / bf16 / fp16 data
int8       product of two int8 matrices with a scale for each row and each column, optional bias
int8 moe   the same for rows sorted by expert: ragged groups, one weight matrix per group, group ends on the device
fp8 moe    the emulated FP8 GEMM of an H100 or an RTX 4060, ragged groups with one weight matrix each, group sizes on the host

`run` computes the plain forms with elementary torch operations, or, where `own` is true, calls the package.
"""
import math
import random

import torch

own = False

_DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16,
       "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


# ---------------------------------------------------------------------------------------------------------------
# cases
def _quantise(rows, K, dtype="bfloat16", name=None):
    return _named({"op": "quantise", "rows": rows, "K": K, "dtype": dtype}, name)


def _int8(M, N, K, out="bfloat16", bias=False, per_row=True, name=None):
    """per_row: a scale for each row and column; else one for each matrix."""
    return _named({"op": "int8", "M": M, "N": N, "K": K, "out": out, "bias": bias, "per_row": per_row}, name)


def _int8_moe(T, E, N, K, out="bfloat16", bias=False, skew=1.0, spare=0, name=None):
    """T rows in E groups, `spare` more rows behind the last group (a padded batch)."""
    return _named({"op": "int8 moe", "T": T, "E": E, "N": N, "K": K, "out": out, "bias": bias, "skew": skew, "spare": spare}, name)


def _fp8_moe(T, E, N, K, fa="e4m3", fb="e4m3", out="bfloat16", fast=False, profile="hopper", skew=1.0, name=None):
    return _named({"op": "fp8 moe", "T": T, "E": E, "N": N, "K": K, "fa": fa, "fb": fb, "out": out, "fast": fast,
                   "profile": profile, "skew": skew}, name)


def _named(case, name):
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # the activations of one decode step of 16 sequences: launch latency
        _quantise(16, 4096, name="quantise_16x4096"),
        # the activations of a prefill of 8192 tokens
        _quantise(8192, 8192, name="quantise_8192x8192"),
        # one decode step: 16 sequences through a projection, bound by the weights
        _int8(16, 4096, 8192, name="int8_16x4096x8192"),
        # sizes that fill no tile, fp16 with a bias (a QKV projection)
        _int8(1000, 2064, 1936, "float16", bias=True, name="int8_1000x2064x1936_bias"),
        # operands whose rows are not 16-byte aligned, fp32 out, one scale per matrix
        _int8(517, 1003, 2001, "float32", per_row=False, name="int8_517x1003x2001_f32"),
        # the projection stack at its largest width
        _int8(8192, 24576, 8192, name="int8_8192x24576x8192"),
        # one decode step of 16 sequences routed to 8 experts, two experts per sequence
        _int8_moe(32, 8, 4096, 4096, name="int8_moe_decode_32x8"),
        # a prefill of 4096 rows over 64 small experts, padded batch
        _int8_moe(4096, 64, 1536, 2048, skew=0.7, spare=100, name="int8_moe_4096x64"),
        # a large prefill over 8 large experts
        _int8_moe(16384, 8, 8192, 4096, name="int8_moe_16384x8"),
        # decode: 16 rows over 8 experts with the numbers of an H100
        _fp8_moe(16, 8, 1024, 2048, skew=0.5, name="fp8_moe_decode_16x8"),
        # a short prefill, activations in E5M2, fast accumulation, ragged sizes
        _fp8_moe(1000, 8, 1040, 2064, fa="e5m2", fast=True, name="fp8_moe_1000x8_fast"),
        # a prefill, slow accumulation
        _fp8_moe(4096, 8, 2048, 2048, skew=0.5, name="fp8_moe_4096x8"),
    ]


_MOST = {"quantise": 8192 * 8192, "int8": 8192 * 24576 * 8192, "int8 moe": 16384 * 8192 * 4096, "fp8 moe": 4096 * 2048 * 2048}
_MOST_ELEMENTS = 8192 * 24576          # of all weight matrices of a drawn case; of its groups padded to the longest one


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choices(("quantise", "int8", "int8 moe", "fp8 moe"), (2, 4, 4, 3))[0]
    while True:
        if op == "quantise":
            c = _quantise(_log(rng, 1, 16384), _log(rng, 16, 24576), rng.choice(("bfloat16", "bfloat16", "float16", "float32")))
            cost, elements = c["rows"] * c["K"], 0
        elif op == "int8":
            step = rng.choice((1, 16, 16, 64))
            c = _int8(_log(rng, 1, 8192), _log(rng, 16, 24576, step), _log(rng, 32, 16384, step),
                      rng.choice(("bfloat16", "bfloat16", "float16", "float32")), rng.random() < 0.3, rng.random() < 0.8)
            cost, elements = c["M"] * c["N"] * c["K"], c["N"] * c["K"]
        elif op == "int8 moe":
            step = rng.choice((1, 16, 16, 64))
            c = _int8_moe(_log(rng, 1, 16384), _log(rng, 1, 128), _log(rng, 64, 8192, step), _log(rng, 64, 8192, step),
                          rng.choice(("bfloat16", "bfloat16", "float16", "float32")), rng.random() < 0.3,
                          rng.choice((0.0, 0.5, 1.0, 2.0)), rng.choice((0, 0, 0, 1, 77)))
        else:
            fa, fb = rng.choice((("e4m3", "e4m3"), ("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2")))
            c = _fp8_moe(_log(rng, 1, 2048), _log(rng, 1, 32), _log(rng, 32, 4096, 16), _log(rng, 64, 4096, 16), fa, fb,
                         rng.choice(("bfloat16", "bfloat16", "float16", "float32")), rng.random() < 0.5,
                         rng.choice(("hopper", "hopper", "ada")), rng.choice((0.0, 0.5, 1.0)))
        if "moe" in op:
            padded = c["E"] * max(_counts(c))               # rows of the plain forms, which pad every group to the longest one
            cost, elements = padded * c["N"] * c["K"], max(c["E"] * c["N"] * c["K"], padded * c["N"], padded * c["K"])
        if cost <= _MOST[op] and elements <= _MOST_ELEMENTS:
            return c


def _counts(case):
    """Rows of each group: a routing whose popularity has a spread of `skew` (0: even); a function of the case alone."""
    T, E = case["T"], case["E"]
    r = random.Random(T * 1009 + E)
    w = [math.exp(case["skew"] * r.gauss(0.0, 1.0)) for _ in range(E)]
    got = [0] * E
    for e in r.choices(range(E), w, k=T):
        got[e] += 1
    return got


def work(case):
    if case["op"] == "quantise":
        n = case["rows"] * case["K"]
        return {"bytes": n * (_BYTES[case["dtype"]] + 1) + 4 * case["rows"], "flops": 3 * n}
    if case["op"] == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        scales = 4 * (M + N) if case["per_row"] else 8
        return {"bytes": (M + N) * K + M * N * _BYTES[case["out"]] + scales + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    T, N, K = case["T"], case["N"], case["K"]
    used = sum(1 for c in _counts(case) if c)              # the weights of groups without rows are not needed
    rows = T + case.get("spare", 0)
    by = T * K + used * N * K + rows * N * _BYTES[case["out"]]
    by += 4 * (T + used * N + case["E"]) + (4 * used * N if case["bias"] else 0) if case["op"] == "int8 moe" else 8 * case["E"]
    return {"bytes": by, "flops": 2 * T * N * K}


# ---------------------------------------------------------------------------------------------------------------
# inputs
def _activations(shape, g, dtype=torch.float32):
    """Rows as a model has them: a spread of magnitudes between rows, a few large channels."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device="cuda"))
    x *= torch.exp(0.7 * torch.randn(shape[-1:], generator=g, device="cuda"))
    return x.to(dtype)


def _codes(shape, g):
    """int8 codes of symmetric quantisation, as a quantiser with one scale per row leaves them."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= 127.0 / x.abs().amax(-1, keepdim=True)
    return x.round_().clamp_(-127, 127).to(torch.int8)


def _scales(shape, g, size):
    return torch.rand(shape, generator=g, device="cuda").add_(0.5).mul_(size)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    if op == "quantise":
        return dict(case, x=_activations((case["rows"], case["K"]), g, _DT[case["dtype"]]))
    if op == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        many = case["per_row"]
        return dict(case, a=_codes((M, K), g), w=_codes((N, K), g), sa=_scales((M, 1) if many else (1,), g, 0.02),
                    sb=_scales((1, N) if many else (1,), g, 0.002),
                    b=torch.randn(N, generator=g, device="cuda") if case["bias"] else None)
    E, N, K = case["E"], case["N"], case["K"]
    counts = _counts(case)
    random.Random(int(seed)).shuffle(counts)               # other inputs route to other experts
    longest = max(counts)
    if op == "int8 moe":
        rows = case["T"] + case["spare"]
        offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
        return dict(case, a=_codes((rows, K), g), w=_codes((E, N, K), g), offs=offs, longest=longest,
                    sa=_scales((rows, 1), g, 0.02), sb=_scales((E, 1, N), g, 0.002),
                    b=torch.randn((E, N), generator=g, device="cuda") if case["bias"] else None)
    a = (torch.randn((case["T"], K), generator=g, device="cuda") * 4.0).to(_DT[case["fa"]])
    w = (torch.randn((E, N, K), generator=g, device="cuda") * 4.0).to(_DT[case["fb"]])
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    return dict(case, a=a, w=w, counts=counts, offs=offs, longest=longest, sa=_scales((E,), g, 0.02), sb=_scales((E,), g, 0.002))


# ---------------------------------------------------------------------------------------------------------------
# one pass
def run(s):
    if own:
        return _own(s)
    if s["op"] == "quantise":
        return _plain_quantise(s["x"])
    if s["op"] == "int8":
        acc = (s["a"].double() @ s["w"].double().t()).float()
        y = acc * (s["sa"] * s["sb"])
        return (y if s["b"] is None else y + s["b"]).to(_DT[s["out"]])
    # groups padded to the longest one: row t of group e goes to place e * longest + t - start(e)
    rows, longest, offs = s["a"].shape[0], s["longest"], s["offs"].long()
    t = torch.arange(rows, device="cuda")
    e = torch.searchsorted(offs, t, right=True)
    real = e < s["E"]
    e = e.clamp(max=s["E"] - 1)
    starts = torch.cat([offs.new_zeros(1), offs[:-1]])
    place = torch.where(real, e * longest + t - starts[e], s["E"] * longest)     # rows behind the last group: one spare place
    if s["op"] == "int8 moe":
        pad = torch.zeros((s["E"] * longest + 1, s["K"]), dtype=torch.float64, device="cuda")
        pad[place] = s["a"].double()
        acc = torch.bmm(pad[:-1].view(s["E"], longest, s["K"]), s["w"].double().transpose(1, 2)).float()
        y = torch.cat([acc.view(-1, s["N"]), acc.new_zeros((1, s["N"]))])[place]
        y = y * (s["sa"] * s["sb"][e, 0])
        y = y if s["b"] is None else y + s["b"][e]
        return torch.where(real[:, None], y, 0.0).to(_DT[s["out"]])
    pad = torch.zeros((s["E"] * longest + 1, s["K"]), device="cuda")
    pad[place] = s["a"].float()
    acc = _plain_emulated(pad[:-1].view(s["E"], longest, s["K"]), s["w"].float(), s["fa"], s["fb"], s["profile"], s["fast"])
    y = acc.view(-1, s["N"])[place] * (s["sa"] * s["sb"])[e][:, None]
    return y.to(_DT[s["out"]])


def _own(s):
    import mmaemu_b200 as mm
    if s["op"] == "quantise":
        return mm.quantize_int8(s["x"])
    if s["op"] == "int8":
        return mm.int8_scaled_mm(s["a"], s["w"].t(), s["sa"], s["sb"], s["b"], _DT[s["out"]])
    if s["op"] == "int8 moe":
        return mm.int8_grouped_scaled_mm(s["a"], s["w"].transpose(1, 2), s["offs"], s["sa"], s["sb"], s["b"], _DT[s["out"]])
    return mm.grouped_scaled_mm(s["a"], s["w"].transpose(1, 2), s["counts"], s["sa"], s["sb"], None, _DT[s["out"]], s["fast"],
                                profile=s["profile"], splitk=1)


def _plain_quantise(x):
    """codes = x * 127 / amax to the nearest integer, ties to even, decided in 64 bits; scale = amax / 127."""
    amax = x.abs().amax(-1, keepdim=True).float()
    good = torch.isfinite(amax)
    top = torch.where(good & (amax > 0), amax, 1.0).double()
    codes = torch.where(good, (x.double() * 127.0 / top).round(), 0.0).to(torch.int8)
    scale = torch.where(good, amax / torch.full_like(amax, 127.0), math.nan)
    return codes, scale


def _power(e):
    return (e + 127).to(torch.int32).bitwise_left_shift(23).view(torch.float32)


def _exponent(x, smallest):
    """floor(log2 |x|), at least `smallest`; far below everything for zero."""
    return torch.where(x == 0, -1000, (torch.frexp(x)[1] - 1).clamp(min=smallest))


def _plain_emulated(a, b, fa, fb, profile, fast):
    """The emulated chains of a [E, M, K] x b [E, N, K]: per block of products, align to the largest exponent, truncate below
    13 fraction bits, add, cut to 14 significant bits. Every step is exact in fp32 (at most 2^20 units per block)."""
    n = {"hopper": 32, "ada": 16}[profile]
    least = {"e4m3": -6, "e5m2": -14}
    ea, eb = _exponent(a, least[fa]), _exponent(b, least[fb])
    acc = torch.zeros((a.shape[0], a.shape[1], b.shape[1]), device=a.device)
    total = torch.zeros_like(acc)
    for k in range(0, a.shape[2], n):
        if not fast and k and k % 128 == 0:
            total, acc = total + acc, torch.zeros_like(acc)
        top = (ea[:, :, None, k:k + n] + eb[:, None, :, k:k + n]).amax(-1)
        top = torch.maximum(top, _exponent(acc, -126)).clamp(min=-60)
        scale = _power(13 - top)
        units = (a[:, :, None, k:k + n] * b[:, None, :, k:k + n] * scale[..., None]).trunc().sum(-1) + (acc * scale).trunc()
        drop = (torch.frexp(units)[1] - 14).clamp(min=0)
        acc = (units * _power(-drop)).trunc() * _power(drop) * _power(top - 13) + 0.0
    return total + acc


# ---------------------------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantise":
        x = s["x"].double()
        top = x.abs().max(dim=-1, keepdim=True)[0]
        whole = torch.where(top > 0, top, 1.0)
        twice = 254.0 * x.abs() + whole                    # nearest integer of 127 |x| / top: floor of twice / (2 top)
        q = torch.floor(twice / (2.0 * whole))
        q -= ((q * 2.0 * whole == twice) & (q % 2 == 1)).double()      # halfway: to even
        return (q * torch.sign(x)).to(torch.int8), top / 127.0
    if case["op"] == "int8":
        acc = torch.mm(s["a"].double(), s["w"].double().t())
        y = acc * s["sa"].double() * s["sb"].double()
        return y if s["b"] is None else y + s["b"].double()
    y = torch.zeros((s["a"].shape[0], case["N"]), dtype=torch.float64, device="cuda")
    start = 0
    for g, end in enumerate(s["offs"].tolist()):
        rows = slice(start, end)
        start = end
        if rows.start == end:
            continue
        if case["op"] == "int8 moe":
            y[rows] = torch.mm(s["a"][rows].double(), s["w"][g].double().t()) * s["sa"][rows].double() * s["sb"][g].double()
            if s["b"] is not None:
                y[rows] += s["b"][g].double()
        else:
            acc = _exact_chains(s["a"][rows], s["w"][g], case["fa"], case["fb"], case["profile"], case["fast"])
            y[rows] = acc * s["sa"][g].double() * s["sb"][g].double()
    return y


def _significands(codes, fmt):
    """Signed integer significand and exponent of FP8 codes (value = significand * 2^(exponent - fraction bits))."""
    bits, low, bias = (3, -6, 7) if fmt == "e4m3" else (2, -14, 15)
    u = codes.view(torch.uint8).long()
    field, frac = (u & 127) >> bits, u & ((1 << bits) - 1)
    m = torch.where(field > 0, frac + (1 << bits), frac)
    return torch.where(u >= 128, -m, m), torch.where(field > 0, field - bias, low), bits


def _exact_chains(a, b, fa, fb, profile, fast):
    """The emulated accumulator in integers: mantissa and exponent of the chain kept apart, chains added as fp32 numbers."""
    n = 32 if profile == "hopper" else 16
    ma, xa, la = _significands(a, fa)
    mb, xb, lb = _significands(b, fb)
    K = a.shape[1]
    total = torch.zeros((a.shape[0], b.shape[0]), device=a.device)
    for first in range(0, K, K if fast else 128):
        last = K if fast else min(K, first + 128)
        mant = torch.zeros(total.shape, dtype=torch.int64, device=a.device)    # value: mant * 2^(grid - 13)
        grid = torch.full_like(mant, -500)
        for k in range(first, last, n):
            j = slice(k, min(k + n, last))
            product = ma[:, None, j] * mb[None, :, j]
            level = xa[:, None, j] + xb[None, :, j]
            length = torch.frexp(mant.double())[1].long()                       # bits of |mant|
            own_level = torch.where(mant == 0, -500, grid - 13 + length - 1)
            top = torch.maximum(torch.where(product == 0, -500, level).amax(-1), own_level)
            shift = level - top[..., None] + 13 - la - lb
            size = torch.where(shift >= 0, product.abs() << shift.clamp(0, 40), product.abs() >> (-shift).clamp(0, 40))
            kept = (mant.abs() << 20) >> (top - grid + 20).clamp(0, 60)
            add = (torch.sign(product) * size).sum(-1) + torch.sign(mant) * kept
            cut = (torch.frexp(add.double())[1].long() - 14).clamp(min=0)
            mant = torch.sign(add) * ((add.abs() >> cut) << cut)
            grid = top
        total = total + torch.ldexp(mant.double(), (grid - 13).double()).float()
    return total.double()
