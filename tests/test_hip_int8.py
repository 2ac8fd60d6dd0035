"""The 8-bit path of a step's projections (``hip_int8``) against its definitions in 64 bits.

Codes: ``t = v * 127 / a`` in float64, ``a = max|v|``; the kernel's code is an integer within half
a step of its own float32 ``t``, so ``|code - t| <= 1/2 + d`` with d = 127 x the relative error
of the float32 chain (each operation rounds by at most 2^-24):

- plain rows: v and a are exact; 127 / a and the product round: d = 127 * 2^-23;
- norms: v = x * w and so a round once more each: d = 127 * 2^-22;
- SiLU: expf within 2^-22, then a sum, a quotient and a product: v and a are within 2^-21,
  d = 127 * (2^-20 + 2^-23).

Scales: a / 127 rounds once (2^-24) besides a's own error; under a norm the sum of squares of up
to 32 terms a lane, 6 lane steps and 16 waves is within 54 * 2^-24, its square root within half
of that, and the mean, eps, root, quotient and products round five times more: 2^-19.

The product's integer sums are exact, so its outputs equal the same three float32 roundings bit
for bit; so do the lookup's.
"""

from __future__ import annotations

import pytest
import torch

from tinyserve_amd import _lib, hip_int8
from tinyserve_amd.hip_int8 import (Int8Rows, add_rms_norm_rows_int8, dequantize_rows, int8_embedding, int8_linear,
                                    quantize_rows, rms_norm_rows_int8, silu_mul_int8)  # fmt: skip

DEVICE = "cuda"
EPS = 1e-6
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
FORMS = ["plain", "norm", "add", "silu"]
TINY = 2.0**-100
CODE_SLACK = {"plain": 127 * 2.0**-23, "norm": 127 * 2.0**-22, "add": 127 * 2.0**-22,
              "silu": 127 * (2.0**-20 + 2.0**-23)}  # fmt: skip
SCALE_ERR = {"plain": 2.0**-24, "norm": 2.0**-19, "add": 2.0**-19, "silu": 2.0**-21 + 2.0**-24}


def rows_of(t: int, n: int, dtype: torch.dtype, seed: int, form: str = "plain") -> dict[str, torch.Tensor]:
    g = torch.Generator().manual_seed(seed)
    wide = 2 * n if form == "silu" else n
    size = 0.25 + torch.rand(t, 1, generator=g)
    return {"x": (torch.randn(t, wide, generator=g) * size).to(dtype),
            "y": (torch.randn(t, n, generator=g) * 0.5).to(dtype),
            "w": (1 + 0.1 * torch.randn(n, generator=g)).to(dtype)}  # fmt: skip


def call(form: str, c: dict[str, torch.Tensor]) -> Int8Rows:
    if form == "plain":
        return quantize_rows(c["x"])
    if form == "silu":
        return silu_mul_int8(c["x"])
    if form == "norm":
        return rms_norm_rows_int8(c["x"], c["w"], EPS)
    return add_rms_norm_rows_int8(c["x"], c["y"], c["w"], EPS)


def definition(form: str, c: dict[str, torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(v, r, x)`` in float64: what is quantised, the row factor of its scale, and the residual."""
    x = c["x"].double()
    one = torch.ones(x.shape[0], 1, dtype=torch.float64)
    if form == "plain":
        return x, one, x
    if form == "silu":
        gate, up = x.chunk(2, dim=1)
        return gate / (1 + torch.exp(-gate)) * up, one, x
    if form == "add":
        x = (c["x"].float() + c["y"].float()).to(c["x"].dtype).double()
    return x * c["w"].double(), (x.square().mean(1, keepdim=True) + EPS).rsqrt(), x


def check_rows(form: str, got: Int8Rows, c: dict[str, torch.Tensor]) -> None:
    v, r, _ = definition(form, c)
    t, n = v.shape
    assert got.q.shape == (t, n) and got.q.dtype == torch.int8
    assert got.scale.shape == (t,) and got.scale.dtype == torch.float32
    q, scale = got.q.cpu().double(), got.scale.cpu().double()
    a = v.abs().amax(1, keepdim=True)
    code = torch.where(a < TINY, 0.0, v * 127 / a.clamp_min(TINY))
    assert float((q - code).abs().max()) <= 0.5 + CODE_SLACK[form]
    want = torch.where(a < TINY, 0.0, a / 127 * r)[:, 0]
    err = (scale - want).abs()
    assert bool((err <= SCALE_ERR[form] * want).all()), float((err / want.clamp_min(1e-300)).max())


def device(c: dict[str, torch.Tensor]) -> dict[str, torch.Tensor]:
    return {k: z.to(DEVICE) for k, z in c.items()}


def codes(m: int, k: int, seed: int, full: bool = False) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    if full:  # the whole range of the type, its lowest value too
        return torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    return (torch.randn(m, k, generator=g) * 31).round().clamp(-127, 127).to(torch.int8)


def scales(m: int, seed: int) -> torch.Tensor:
    return torch.rand(m, generator=torch.Generator().manual_seed(seed)) * 0.01 + 1e-4


def linear_want(x: Int8Rows, w: Int8Rows, dtype: torch.dtype) -> torch.Tensor:
    acc = x.q.cpu().double() @ w.q.cpu().double().t()  # integers below 2^53
    return (acc.float() * x.scale.cpu()[:, None] * w.scale.cpu()).to(dtype)


def same(got: torch.Tensor, want: torch.Tensor) -> bool:
    """Equal, NaN for NaN."""
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


@pytest.fixture(params=["compiled", "python"])
def host_path(request: pytest.FixtureRequest, monkeypatch: pytest.MonkeyPatch) -> str:
    """Both host paths of the calls: the compiled one (bound by a first call) and Python's."""
    quantize_rows(torch.ones(1, 16, device=DEVICE))
    if request.param == "python":
        monkeypatch.setattr(hip_int8, "_fast", None)
    else:
        assert hip_int8._fast is not None
    return request.param


# ---- refusals (CPU) ------------------------------------------------------------------------------
def test_refusals_come_before_the_device() -> None:
    x = torch.zeros(2, 8, dtype=torch.float16)
    w = torch.ones(8, dtype=torch.float16)
    r = Int8Rows(torch.zeros(2, 8, dtype=torch.int8), torch.ones(2))
    for bad in (x[0], x.t(), x.double(), x.to(torch.int32)):
        with pytest.raises(ValueError):
            quantize_rows(bad)
    for bad in (w[:7], w.float(), torch.ones(16, dtype=torch.float16)[::2], torch.ones(1, 8, dtype=torch.float16)):
        with pytest.raises(ValueError, match="weight"):
            rms_norm_rows_int8(x, bad, EPS)
        with pytest.raises(ValueError, match="weight"):
            add_rms_norm_rows_int8(x, x.clone(), bad, EPS)
    for eps in (0.0, -1e-6, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            rms_norm_rows_int8(x, w, eps)
        with pytest.raises(ValueError, match="eps"):
            add_rms_norm_rows_int8(x, x.clone(), w, eps)
    for bad in (x[:1], x.float(), torch.zeros(8, 2, dtype=torch.float16).t()):
        with pytest.raises(ValueError, match="y must be"):
            add_rms_norm_rows_int8(x, bad, w, EPS)
    with pytest.raises(ValueError, match="even width"):
        silu_mul_int8(x[:, :7])
    for bad in (Int8Rows(r.q.to(torch.int16), r.scale), Int8Rows(r.q.t(), r.scale), Int8Rows(r.q[0], r.scale),
                Int8Rows(r.q, r.scale[:1]), Int8Rows(r.q, r.scale.double()), Int8Rows(r.q, torch.ones(4)[::2])):  # fmt: skip
        for op in (lambda z: int8_linear(z, r, torch.float16), lambda z: int8_linear(r, z, torch.float16),
                   lambda z: dequantize_rows(z, torch.float16)):  # fmt: skip
            with pytest.raises(ValueError):
                op(bad)
    with pytest.raises(ValueError, match="columns"):
        int8_linear(r, Int8Rows(r.q[:, :7], r.scale), torch.float16)
    with pytest.raises(ValueError, match="dtype"):
        int8_linear(r, r, torch.float64)
    with pytest.raises(ValueError, match="dtype"):
        dequantize_rows(r, torch.int8)
    long = torch.zeros(1, hip_int8.MAX_K + 1, dtype=torch.int8)
    with pytest.raises(ValueError, match="at most 131071"):
        int8_linear(Int8Rows(long, torch.ones(1)), Int8Rows(long, torch.ones(1)), torch.float16)
    for bad in (torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, dtype=torch.int16), torch.zeros(2)):
        with pytest.raises(ValueError, match="ids"):
            int8_embedding(r, bad, torch.float16)
    with pytest.raises(ValueError, match="no rows"):
        int8_embedding(Int8Rows(r.q[:0], r.scale[:0]), torch.zeros(1, dtype=torch.int64), torch.float16)


def test_cpu_tensors_are_refused() -> None:
    x = torch.zeros(2, 8, dtype=torch.float16)
    w = torch.ones(8, dtype=torch.float16)
    r = Int8Rows(torch.zeros(2, 8, dtype=torch.int8), torch.ones(2))
    for op in (lambda: quantize_rows(x), lambda: rms_norm_rows_int8(x, w, EPS),
               lambda: add_rms_norm_rows_int8(x, x.clone(), w, EPS), lambda: silu_mul_int8(x),
               lambda: int8_linear(r, r, torch.float16), lambda: dequantize_rows(r, torch.float16),
               lambda: int8_embedding(r, torch.zeros(1, dtype=torch.int64), torch.float16)):  # fmt: skip
        with pytest.raises(RuntimeError, match="HIP device only"):
            op()


def test_c_abi_refuses_before_any_launch() -> None:
    lib = _lib.load()
    big = (1 << 30) + 1

    def quant(t=2, n=8, xs=8, ys=8, qs=16, form=0, dtype=1, x=0x1000, y=0x9000, w=0x2000, q=0x4000, scale=0x3000):  # noqa: ANN001, ANN202
        return lib.ts_int8_quantize_rows(x, y, w, q, scale, t, n, xs, ys, qs, 1e-6, form, dtype, None)

    assert quant(t=0) == 0  # nothing to launch
    for bad in ({"t": -1}, {"t": big}, {"n": 0}, {"n": big}, {"form": 4}, {"form": -1}, {"qs": 8}, {"qs": 24}, {"q": 0x4008},
                {"x": None}, {"q": None, "t": 1}, {"scale": None}, {"xs": -1}, {"form": 1, "w": None},
                {"form": 2, "y": None}, {"form": 2, "w": None}, {"form": 2, "ys": -1}):  # fmt: skip
        assert quant(**bad) == -1, bad
    assert quant(dtype=3) == -2
    # The residual is written: rows over each other, or over another tensor's.
    for bad in ({"xs": 4}, {"xs": 0}, {"y": 0x1000, "ys": 16, "xs": 8}, {"y": 0x1002}, {"y": 0x1008, "xs": 12, "ys": 12},
                {"y": 0x1000 - 14, "t": 1}, {"xs": 16, "ys": 16, "y": 0x1000 + 2 * 16 + 14}):  # fmt: skip
        assert quant(form=2, **bad) == -1, bad

    def linear(m=2, n=3, k=4, xs=4, ws=4, os=3, padded=0, dtype=1, x=0x1000, w=0x2000, out=0x3000, a=0x4000, b=0x5000, s=None, sb=0):  # noqa: ANN001, ANN202
        return lib.ts_int8_linear(x, xs, a, w, ws, b, out, os, m, n, k, padded, dtype, s, sb, None)

    assert linear(m=0) == 0 and linear(n=0) == 0
    for bad in ({"m": -1}, {"m": big}, {"n": -1}, {"n": big}, {"k": -1}, {"k": 131072}, {"xs": -1}, {"ws": -1}, {"os": 2},
                {"x": None}, {"w": None}, {"out": None}, {"a": None}, {"b": None}, {"s": 0x6008, "sb": 64}, {"sb": -1}):  # fmt: skip
        assert linear(**bad) == -1, bad
    assert linear(dtype=7) == -2
    tiled = {"m": 4000, "n": 4000, "os": 4000, "k": 20, "xs": 32, "ws": 32}  # many rows: aligned and readable to 32 columns, or not taken
    for bad in ({"padded": 0}, {"padded": 1, "xs": 20}, {"padded": 1, "ws": 24}, {"padded": 1, "x": 0x1008},
                {"padded": 1, "w": 0x2001}, {"padded": 1, "xs": (1 << 23) + 16}):  # fmt: skip
        assert linear(**{**tiled, **bad}) == -2, bad

    def pad(m=2, m2=2, n=20, qs=20, qs2=20, os=32, q=0x1000, q2=0x3000, out=0x2000, out2=0x4000):  # noqa: ANN001, ANN202
        return lib.ts_int8_pad_rows(q, qs, out, m, q2, qs2, out2, m2, os, n, None)

    assert pad(m=0, m2=0) == 0 and pad(n=0) == 0
    for bad in ({"m": -1}, {"m2": -1}, {"m": big}, {"m2": big}, {"n": big}, {"qs": -1}, {"qs2": -1}, {"os": 16}, {"os": 40},
                {"out": 0x2008}, {"out2": 0x4004}, {"q": None}, {"q2": None}, {"out": None}, {"out2": None}):  # fmt: skip
        assert pad(**bad) == -1, bad

    def embed(t=2, n=4, rows=5, ts=4, os=4, dtype=1, table=0x1000, scale=0x2000, ids=0x3000, out=0x4000):  # noqa: ANN001, ANN202
        return lib.ts_int8_embedding(table, ts, scale, rows, ids, out, os, t, n, dtype, None)

    assert embed(t=0) == 0 and embed(n=0) == 0
    for bad in ({"t": -1}, {"t": big}, {"n": big}, {"rows": 0}, {"rows": -1}, {"ts": -1}, {"os": 3}, {"table": None},
                {"scale": None}, {"out": None}, {"ids": None, "t": 6}):  # fmt: skip
        assert embed(**bad) == -1, bad
    assert embed(dtype=-1) == -2


# ---- quantised rows --------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 9, 15, 64, 509, 512, 1000, 1024, 1029, 2048, 2051, 4096, 4097, 8192, 8200])
def test_rows_equal_the_definition(form: str, n: int, dtype: torch.dtype) -> None:
    for t in (1, 5, 700):
        if t * n > 3_000_000:
            continue
        c = rows_of(t, n, dtype, seed=t * 31 + n, form=form)
        d = device(c)
        got = call(form, d)
        check_rows(form, got, c)
        if form == "add":
            assert torch.equal(d["x"].cpu().double(), definition(form, c)[2])
            assert torch.equal(d["y"].cpu(), c["y"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("n", [16384, 16411, 32768, 32775, 70001])
def test_long_rows_equal_the_definition(form: str, n: int, dtype: torch.dtype) -> None:
    c = rows_of(3, n, dtype, seed=n, form=form)
    d = device(c)
    check_rows(form, call(form, d), c)
    if form == "add":
        assert torch.equal(d["x"].cpu().double(), definition(form, c)[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5, 520, 1032, 9000, 40000])
@pytest.mark.parametrize("form", FORMS)
def test_rows_that_have_no_scale(form: str, n: int, dtype: torch.dtype) -> None:
    """Zeros, values below 2^-100, an infinity, a NaN: their rows alone, and no others."""
    c = rows_of(7, n, dtype, seed=n, form=form)
    wide = c["x"].shape[1]
    c["y"].zero_()
    c["x"][0] = 0
    c["x"][1] = 1e-38 if dtype != torch.float16 else 0  # with SiLU the product underflows too
    c["x"][2, wide - 1] = float("nan")
    c["x"][3, wide // 2] = float("inf")
    c["x"][4, 0] = -float("inf")
    if form == "silu":
        c["x"][4, n:] = 1.0  # silu(-inf) is -0 * inf in the formula: NaN
    d = device(c)
    got = call(form, d)
    scale = got.scale.cpu()
    assert float(scale[0]) == 0 and float(scale[1]) == 0
    assert bool(scale[2:5].isnan().all())
    assert not bool(got.q[:5].cpu().any())
    rest = Int8Rows(got.q[5:], got.scale[5:])
    check_rows(form, rest, {"x": c["x"][5:], "y": c["y"][5:], "w": c["w"]})
    out = int8_linear(got, Int8Rows(codes(3, n, 1).to(DEVICE), scales(3, 2).to(DEVICE)), torch.float32).cpu()
    assert bool(out[2:5].isnan().all()) and not bool(out[:2].any()) and bool(out[5:].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5, 40, 700, 40000])
def test_gates_of_every_size(n: int, dtype: torch.dtype) -> None:
    """SiLU where its exponential overflows, underflows or does neither, one size a row."""
    gates = [0.0, 1e-6, -1e-6, 1.0, -1.0, 10.0, -10.0, 50.0, -50.0, 80.0, -80.0, 88.0, 89.0, 130.0, 1e4, 6e4]
    x = torch.randn(len(gates), 2 * n, generator=torch.Generator().manual_seed(n)).to(dtype)
    x[:, :n] = torch.tensor(gates)[:, None].to(dtype)
    check_rows("silu", silu_mul_int8(x.to(DEVICE)), {"x": x})
    # Where exp(-g) passes float32 the value is 0 to within 1e-36: the rest of the row decides.
    x[:, 0] = torch.tensor([-88.5, -89.0, -95.0, -130.0, -1e3, -6e4] * 3)[: len(gates)].to(dtype)
    check_rows("silu", silu_mul_int8(x[3:].to(DEVICE)), {"x": x[3:]})
    if dtype == torch.float32:
        x[:, :n], x[:, n:] = torch.tensor([3e38, -3e38] * 8)[:, None], 0.1
        got = silu_mul_int8(x.to(DEVICE))
        assert bool((got.q[::2] == 127).all()) and bool((got.scale[1::2] < 1e-36).all())


@pytest.mark.gpu
def test_sums_of_squares_past_float32_are_nan_rows() -> None:
    x = torch.full((2, 64), 2.0**64)
    x[1] = 2.0**50
    got = rms_norm_rows_int8(x.to(DEVICE), torch.ones(64, device=DEVICE), EPS)
    assert bool(got.scale[0].isnan()) and not bool(got.q[0].any())
    assert bool((got.q[1] == 127).all()) and abs(float(got.scale[1]) * 127 - 1) < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("n", [24, 1025, 3000])
def test_strided_and_unaligned_rows(form: str, n: int, dtype: torch.dtype) -> None:
    """Rows cut out of wider ones, from an odd element on; nothing outside them is touched."""
    c = rows_of(6, n, dtype, seed=n + 1, form=form)
    wide = c["x"].shape[1]
    buf = torch.full((6, wide + 7), 3.0, dtype=dtype, device=DEVICE)
    ybuf = torch.full((6, n + 2), 5.0, dtype=dtype, device=DEVICE)
    wbuf = torch.full((n + 1,), 9.0, dtype=dtype, device=DEVICE)
    d = {"x": buf[:, 3 : 3 + wide], "y": ybuf[:, 1 : 1 + n], "w": wbuf[1:]}
    for k in d:
        d[k].copy_(c[k])
    check_rows(form, call(form, d), c)
    assert bool((buf[:, :3] == 3).all()) and bool((buf[:, 3 + wide :] == 3).all())
    if form == "add":
        assert torch.equal(d["x"].cpu().double(), definition(form, c)[2])
    else:
        assert torch.equal(d["x"].cpu(), c["x"])


@pytest.mark.gpu
def test_residual_and_addend_in_the_same_memory() -> None:
    """y may be x, or lie beside x in the same rows; rows over each other are refused."""
    g = torch.Generator().manual_seed(3)
    buf = torch.randn(4, 64, generator=g).half()
    w = torch.ones(32, dtype=torch.float16)
    d = buf.to(DEVICE)
    got = add_rms_norm_rows_int8(d[:, :32], d[:, 32:], w.to(DEVICE), EPS)
    check_rows("add", got, {"x": buf[:, :32], "y": buf[:, 32:], "w": w})
    assert torch.equal(d[:, 32:].cpu(), buf[:, 32:])
    d = buf.to(DEVICE)
    got = add_rms_norm_rows_int8(d[:, :32], d[:, :32], w.to(DEVICE), EPS)
    check_rows("add", got, {"x": buf[:, :32], "y": buf[:, :32], "w": w})
    assert torch.equal(d[:, :32].cpu(), (buf[:, :32] * 2))
    for x, y in ((d[:, :32], d[:, 16:48]), (d[:3, :32], d[1:, :32]), (d[:1].expand(4, 64)[:, :32], d[:, 32:])):
        with pytest.raises(ValueError, match="invalid"):
            add_rms_norm_rows_int8(x, y, w.to(DEVICE), EPS)


@pytest.mark.gpu
def test_rows_and_columns_of_length_zero() -> None:
    w = torch.ones(16, dtype=torch.float16, device=DEVICE)
    empty = torch.empty(0, 16, dtype=torch.float16, device=DEVICE)
    for got in (quantize_rows(empty), rms_norm_rows_int8(empty, w, EPS), add_rms_norm_rows_int8(empty, empty, w, EPS)):
        assert got.q.shape == (0, 16) and got.scale.shape == (0,)
    assert silu_mul_int8(empty).q.shape == (0, 8)
    thin = quantize_rows(torch.empty(3, 0, dtype=torch.float16, device=DEVICE))
    assert thin.q.shape == (3, 0) and not bool(thin.scale.any())
    rows = Int8Rows(codes(3, 16, 0).to(DEVICE), scales(3, 1).to(DEVICE))
    none = Int8Rows(rows.q[:0], rows.scale[:0])
    assert int8_linear(none, rows, torch.float16).shape == (0, 3)
    assert int8_linear(rows, none, torch.float16).shape == (3, 0)
    zero = int8_linear(Int8Rows(rows.q[:, :0], rows.scale), Int8Rows(rows.q[:, :0], rows.scale), torch.float32)
    assert torch.equal(zero.cpu(), torch.zeros(3, 3))
    assert dequantize_rows(none, torch.float16).shape == (0, 16)
    assert int8_embedding(rows, torch.empty(0, dtype=torch.int64, device=DEVICE), torch.float16).shape == (0, 16)
    assert int8_embedding(none, torch.empty(0, dtype=torch.int64, device=DEVICE), torch.float16).shape == (0, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_more_rows_than_one_launch_takes(form: str) -> None:
    """Over 2^21 rows go in several launches: the rows around the seam, as they are alone."""
    t, n = (1 << 21) + 5, 8
    x = torch.randn(t, 2 * n if form == "silu" else n, device=DEVICE, generator=torch.Generator(DEVICE).manual_seed(1)).half()
    c = {"x": x, "y": torch.randn(t, n, device=DEVICE).half(), "w": torch.ones(n, dtype=torch.float16, device=DEVICE)}
    seam = slice((1 << 21) - 4, t)
    part = {k: (v if k == "w" else v[seam].clone()) for k, v in c.items()}
    before = {k: v.cpu() for k, v in part.items()}
    got, alone = call(form, c), call(form, part)
    assert torch.equal(got.q[seam], alone.q) and torch.equal(got.scale[seam], alone.scale)
    assert torch.equal(c["x"][seam], part["x"])
    check_rows(form, alone, before)
    assert bool((got.q.abs().amax(1) == 127).all())


# ---- the product -----------------------------------------------------------------------------------
ODD = [(1, 1, 1), (2, 3, 5), (1, 17, 16), (16, 16, 64), (17, 33, 65), (5, 100, 127), (31, 64, 128), (33, 130, 129),
       (64, 48, 200), (65, 1003, 531), (100, 36, 1531), (128, 128, 256), (129, 257, 255), (255, 70, 1024),
       (300, 513, 640), (513, 300, 77), (1, 5000, 40), (3, 20, 9000), (200, 400, 4112)]  # fmt: skip


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("m", "n", "k"), ODD)
def test_linear_equals_the_definition(m: int, n: int, k: int, dtype: torch.dtype) -> None:
    x = Int8Rows(codes(m, k, m + k, full=k <= 64).to(DEVICE), scales(m, m).to(DEVICE))
    w = Int8Rows(codes(n, k, n - k, full=k <= 64).to(DEVICE), scales(n, n).to(DEVICE))
    got = int8_linear(x, w, dtype)
    assert got.dtype == dtype and got.shape == (m, n)
    assert same(got.cpu(), linear_want(x, w, dtype))
    # The same rows at 16-byte aligned strides, as the quantising functions lay them out.
    pad = torch.full((max(m, n), (k + 15) // 16 * 16), 77, dtype=torch.int8, device=DEVICE)
    xa, wa = pad.clone()[:m, :k], pad.clone()[:n, :k]
    xa.copy_(x.q)
    wa.copy_(w.q)
    assert same(int8_linear(Int8Rows(xa, x.scale), Int8Rows(wa, w.scale), dtype).cpu(), got.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize(("m", "n"), [(4100, 4100), (2751, 6144), (1030, 4090), (520, 4100), (260, 1030), (129, 70)])
def test_every_tile_shape_and_last_columns(m: int, n: int) -> None:
    """Sizes that take each of the tile shapes, at column counts around their tiles of 128."""
    for k in (1, 15, 16, 17, 112, 113, 127, 128, 129, 136, 144, 255, 256, 400, 515):
        x = Int8Rows(codes(m, k, m + k, full=True).to(DEVICE), scales(m, m).to(DEVICE))
        w = Int8Rows(codes(n, k, n - k, full=True).to(DEVICE), scales(n, n).to(DEVICE))
        got = int8_linear(x, w, torch.float32)
        acc = (x.q.float() @ w.q.float().t()) if k <= 1024 else None  # integers below 2^24: exact
        assert same(got, acc * x.scale[:, None] * w.scale), k
        half = int8_linear(x, w, torch.bfloat16)
        assert same(half, (acc * x.scale[:, None] * w.scale).bfloat16()), k


@pytest.mark.gpu
@pytest.mark.parametrize(("m", "n"), [(1_100_003, 3), (3, 1_100_003), (70_001, 40)])
def test_many_rows_of_one_side(m: int, n: int) -> None:
    """Grids past 65535 workgroups along either side."""
    k = 48
    g = torch.Generator(DEVICE).manual_seed(m)
    x = Int8Rows(torch.randint(-128, 128, (m, k), dtype=torch.int8, device=DEVICE, generator=g), torch.rand(m, device=DEVICE))
    w = Int8Rows(torch.randint(-128, 128, (n, k), dtype=torch.int8, device=DEVICE, generator=g), torch.rand(n, device=DEVICE))
    acc = x.q.float() @ w.q.float().t()  # integers below 2^24: exact
    assert same(int8_linear(x, w, torch.float32), acc * x.scale[:, None] * w.scale)
    odd = Int8Rows(x.q[:, :47], x.scale)  # rows that are not 16-byte aligned from 47 columns on
    acc = odd.q.float() @ w.q[:, :47].float().t()
    assert same(int8_linear(odd, Int8Rows(w.q[:, :47].contiguous(), w.scale), torch.float32), acc * x.scale[:, None] * w.scale)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [(127, 127), (-128, -128), (127, -128)])
def test_largest_sums_are_exact(value: tuple[int, int]) -> None:
    k = hip_int8.MAX_K
    x = Int8Rows(torch.full((3, k), value[0], dtype=torch.int8, device=DEVICE), torch.ones(3, device=DEVICE))
    w = Int8Rows(torch.full((20, k), value[1], dtype=torch.int8, device=DEVICE), torch.ones(20, device=DEVICE))
    want = torch.tensor(float(value[0] * value[1] * k))  # the int32, rounded to float32
    assert bool((int8_linear(x, w, torch.float32).cpu() == want).all())


# Products that run in parts of K: 2, 3, 4, 6 and 8 of them, in 128 x 128 tiles but for the last one
# (256 x 256), with odd outputs and columns.
PARTS = [(146, 6602, 5805), (3270, 263, 5441), (40, 5460, 13418), (2, 4132, 40592), (2, 911, 104701), (2700, 47, 20001), (136, 5787, 15353)]


def test_workspace_of_products() -> None:
    need = _lib.load().ts_int8_linear_workspace
    for m, n, k in PARTS:
        parts, rest = divmod(need(m, n, k), m * ((n + 3) // 4) * 16)
        assert parts in (2, 3, 4, 6, 8) and rest == 0, (m, n, k)
    for m, n, k in [(0, 4, 9000), (4, 0, 9000), (-1, 4, 9000), (4, 4, -1), (4, 4, 131072), (4, 4, 0), (16, 16, 4096),
                    (16, 16, 131071), (8192, 8192, 8192), (1 << 30, 1, 131071), (1, 1 << 30, 131071), (1 << 30, 1 << 30, 131071)]:  # fmt: skip
        assert need(m, n, k) == 0, (m, n, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("m", "n", "k"), PARTS)
def test_parts_of_the_columns(m: int, n: int, k: int, dtype: torch.dtype, host_path: str) -> None:
    x = Int8Rows(codes(m, k, 1, full=True).to(DEVICE), scales(m, 2).to(DEVICE))
    w = Int8Rows(codes(n, k, 3, full=True).to(DEVICE), scales(n, 4).to(DEVICE))
    want = linear_want(x, w, dtype)
    wide = torch.full((m, n + 5), 5.0, dtype=dtype, device=DEVICE)
    assert torch.equal(int8_linear(x, w, dtype).cpu(), want)
    int8_linear(x, w, dtype, wide[:, 3 : n + 3])
    assert torch.equal(wide[:, 3 : n + 3].cpu(), want)
    assert bool((wide[:, :3] == 5).all()) and bool((wide[:, n + 3 :] == 5).all())


@pytest.mark.gpu
@pytest.mark.parametrize(("m", "n", "k"), [(2, 4132, 40592), (40, 5460, 13424)])
def test_workspace_given_short_and_none(m: int, n: int, k: int) -> None:
    """The same bits with the workspace, with a byte less and without; nothing past it is written."""
    lib = _lib.load()
    x, w, xs, ws = codes(m, k, 1).to(DEVICE), codes(n, k, 2).to(DEVICE), scales(m, 3).to(DEVICE), scales(n, 4).to(DEVICE)
    want = linear_want(Int8Rows(x, xs), Int8Rows(w, ws), torch.float32)
    need = lib.ts_int8_linear_workspace(m, n, k)
    assert need > 0
    work = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device=DEVICE)
    for given in (need, need - 1, 0):
        out = torch.zeros(m, n, device=DEVICE)
        work.fill_(0x5A)
        rc = lib.ts_int8_linear(x.data_ptr(), k, xs.data_ptr(), w.data_ptr(), k, ws.data_ptr(), out.data_ptr(), n, m, n, k, 1, _lib.DTYPES[torch.float32],
                                work.data_ptr() if given else None, given, torch.cuda.current_stream().cuda_stream)  # fmt: skip
        torch.cuda.synchronize()
        assert rc == 0
        assert torch.equal(out.cpu(), want), given
        assert bool((work[need if given == need else 0 :] == 0x5A).all()), given


@pytest.mark.gpu
def test_parts_captured_and_replayed_between_eager_calls(host_path: str) -> None:
    """Two captured products in parts and eager ones in turn: each has its own sums."""
    sets = []
    for m, n, k in ((2, 911, 104701), (40, 5460, 13418)):
        x = Int8Rows(codes(m, k, 1).to(DEVICE), scales(m, 2).to(DEVICE))
        w = Int8Rows(codes(n, k, 3).to(DEVICE), scales(n, 4).to(DEVICE))
        sets.append((x, w, torch.empty(m, n, device=DEVICE)))
    for x, w, out in sets:
        int8_linear(x, w, torch.float32, out)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in sets]
    for g, (x, w, out) in zip(graphs, sets, strict=True):
        with torch.cuda.graph(g):
            int8_linear(x, w, torch.float32, out)
    for round_ in range(3):
        for i, (x, w, out) in enumerate(sets):
            x.q.copy_(codes(*x.q.shape, 10 * round_ + i))
            out.zero_()
        for g in graphs:
            g.replay()
        eager = [int8_linear(x, w, torch.float32) for x, w, _ in sets]
        torch.cuda.synchronize()
        for (x, w, out), e in zip(sets, eager, strict=True):
            want = linear_want(x, w, torch.float32)
            assert torch.equal(out.cpu(), want) and torch.equal(e.cpu(), want)


@pytest.mark.gpu
def test_parts_on_two_streams_at_once(host_path: str) -> None:
    m, n, k = 2, 911, 104701
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [(Int8Rows(codes(m, k, i).to(DEVICE), scales(m, i).to(DEVICE)), Int8Rows(codes(n, k, 9 + i).to(DEVICE), scales(n, 9 + i).to(DEVICE))) for i in range(2)]  # fmt: skip
    torch.cuda.synchronize()
    outs: list[list[torch.Tensor]] = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(int8_linear(*sets[i], torch.bfloat16))
    torch.cuda.synchronize()
    for (x, w), got in zip(sets, outs, strict=True):
        want = linear_want(x, w, torch.bfloat16)
        assert all(torch.equal(o.cpu(), want) for o in got)


@pytest.mark.gpu
@pytest.mark.parametrize(("m", "n", "k"), [(7, 50, 96), (70, 260, 512), (300, 300, 300)])
def test_linear_of_strided_rows_into_strided_rows(m: int, n: int, k: int) -> None:
    xb, wb = codes(m, k + 9, 1).to(DEVICE), codes(n, k + 5, 2).to(DEVICE)
    x = Int8Rows(xb[:, 3 : 3 + k], scales(m + 1, 3).to(DEVICE)[1:])
    w = Int8Rows(wb[:, 5:], scales(n + 3, 4).to(DEVICE)[3:])
    out = torch.full((m, n + 3), 5.0, dtype=torch.float16, device=DEVICE)
    got = int8_linear(x, w, torch.float16, out=out[:, 1 : 1 + n])
    assert got.data_ptr() == out[:, 1:].data_ptr()
    assert torch.equal(out[:, 1 : 1 + n].cpu(), linear_want(x, w, torch.float16))
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 1 + n :] == 5).all())
    # One row of x for every token (stride 0).
    one = Int8Rows(x.q[:1].expand(m, k), x.scale)
    assert torch.equal(int8_linear(one, w, torch.float32).cpu(), linear_want(one, w, torch.float32))
    for bad in (out, out[:, 1 : 1 + n].float(), out[:1].expand(m, n + 3)[:, :n] if m > 1 else out,
                torch.empty(n, m, dtype=torch.float16, device=DEVICE).t()):  # fmt: skip
        with pytest.raises(ValueError, match="out must be"):
            int8_linear(x, w, torch.float16, out=bad)


@pytest.mark.gpu
def test_rows_of_the_product_do_not_depend_on_their_batch() -> None:
    """A token alone, in a batch of 40 and in one of 600 gives the same bits: the sums are exact."""
    x = Int8Rows(codes(600, 1024, 1).to(DEVICE), scales(600, 2).to(DEVICE))
    w = Int8Rows(codes(520, 1024, 3).to(DEVICE), scales(520, 4).to(DEVICE))
    full = int8_linear(x, w, torch.bfloat16)
    for lo, hi in ((0, 1), (599, 600), (10, 50), (100, 300)):
        part = int8_linear(Int8Rows(x.q[lo:hi], x.scale[lo:hi]), w, torch.bfloat16)
        assert torch.equal(part, full[lo:hi])


@pytest.mark.gpu
def test_scales_of_zero_infinity_and_nan() -> None:
    x = Int8Rows(codes(4, 64, 1).to(DEVICE), torch.tensor([1.0, 0.0, float("inf"), float("nan")], device=DEVICE))
    w = Int8Rows(codes(5, 64, 2).to(DEVICE), torch.tensor([1.0, 0.0, 2.0, float("nan"), 1e38], device=DEVICE))
    for dtype in DTYPES:
        assert same(int8_linear(x, w, dtype).cpu(), linear_want(x, w, dtype))


# ---- rows of a table -------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 15, 16, 17, 100, 1024, 1031])
def test_embedding_equals_the_definition(n: int, dtype: torch.dtype) -> None:
    table = Int8Rows(codes(300, n, n, full=True).to(DEVICE), scales(300, 1).to(DEVICE))
    want = (table.q.cpu().float() * table.scale.cpu()[:, None]).to(dtype)
    assert torch.equal(dequantize_rows(table, dtype).cpu(), want)
    ids = torch.randint(0, 300, (517,), generator=torch.Generator().manual_seed(n))
    ids[:4] = torch.tensor([0, 299, 7, 7])
    for kind in (torch.int64, torch.int32):
        at = ids.to(kind)
        assert torch.equal(int8_embedding(table, at.to(DEVICE), dtype).cpu(), want[ids])
    wide = torch.stack([ids, ids.flip(0)], 1).to(DEVICE)
    assert torch.equal(int8_embedding(table, wide[:, 1], dtype).cpu(), want[ids.flip(0)])


@pytest.mark.gpu
def test_ids_outside_the_table_give_nan_rows() -> None:
    table = Int8Rows(codes(10, 40, 0).to(DEVICE), scales(10, 1).to(DEVICE))
    ids = torch.tensor([3, -1, 10, 2**40, -(2**62), 9], device=DEVICE)
    got = int8_embedding(table, ids, torch.float16).cpu()
    assert bool(got[1:5].isnan().all())
    assert torch.equal(got[[0, 5]], dequantize_rows(table, torch.float16).cpu()[[3, 9]])


# ---- together --------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t", [1, 33, 300])
def test_mlp_of_a_layer_stage_by_stage(t: int, dtype: torch.dtype) -> None:
    """The MLP half of a decoder layer: every stage against its definition on what the stage
    before it gave, the way the functions are used together."""
    hidden, inter = 256, 704
    g = torch.Generator().manual_seed(t)
    x, y = torch.randn(t, hidden, generator=g).to(dtype), torch.randn(t, hidden, generator=g).to(dtype)
    w = (1 + 0.1 * torch.randn(hidden, generator=g)).to(dtype)
    gate_up = quantize_rows((torch.randn(2 * inter, hidden, generator=g) * 0.05).to(dtype).to(DEVICE))
    down = quantize_rows((torch.randn(hidden, inter, generator=g) * 0.05).to(dtype).to(DEVICE))
    dx = x.to(DEVICE)
    h = add_rms_norm_rows_int8(dx, y.to(DEVICE), w.to(DEVICE), EPS)
    check_rows("add", h, {"x": x, "y": y, "w": w})
    gu = int8_linear(h, gate_up, dtype)
    assert torch.equal(gu.cpu(), linear_want(h, gate_up, dtype))
    act = silu_mul_int8(gu)
    check_rows("silu", act, {"x": gu.cpu()})
    out = int8_linear(act, down, dtype)
    assert torch.equal(out.cpu(), linear_want(act, down, dtype))


@pytest.mark.gpu
def test_captured_and_replayed() -> None:
    """One graph of the chain, replayed on new inputs with eager work between the replays."""
    t, hidden, inter = 24, 512, 640
    g = torch.Generator().manual_seed(5)
    w = (1 + 0.1 * torch.randn(hidden, generator=g)).half().to(DEVICE)
    up = quantize_rows((torch.randn(2 * inter, hidden, generator=g) * 0.05).half().to(DEVICE))
    down = quantize_rows((torch.randn(hidden, inter, generator=g) * 0.05).half().to(DEVICE))
    ids = torch.zeros(t, dtype=torch.int64, device=DEVICE)
    table = quantize_rows(torch.randn(100, hidden, generator=g).half().to(DEVICE))

    def chain() -> torch.Tensor:
        x = int8_embedding(table, ids, torch.float16)
        act = silu_mul_int8(int8_linear(rms_norm_rows_int8(x, w, EPS), up, torch.float16))
        y = int8_linear(act, down, torch.float16)
        h = add_rms_norm_rows_int8(x, y, w, EPS)
        return int8_linear(h, table, torch.float32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    for seed in range(4):
        ids.copy_(torch.randint(0, 100, (t,), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, chain()), seed
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("t", "n"), [(1, 16), (3, 40), (300, 257), (700, 1024)])
def test_both_host_paths(t: int, n: int, dtype: torch.dtype, host_path: str) -> None:
    for form in FORMS:
        c = rows_of(t, n, dtype, seed=t, form=form)
        d = device(c)
        got = call(form, d)
        assert type(got) is Int8Rows and got.q.stride(0) % 16 == 0
        check_rows(form, got, c)
        if form == "add":
            assert torch.equal(d["x"].cpu().double(), definition(form, c)[2])
    w = Int8Rows(codes(n, n, 1).to(DEVICE), scales(n, 2).to(DEVICE))
    assert torch.equal(int8_linear(got, w, dtype).cpu(), linear_want(got, w, dtype))
    out = torch.full((t, n + 5), 2.0, dtype=dtype, device=DEVICE)
    view = out[:, 2 : n + 2]
    assert int8_linear(got, w, dtype, view) is view
    assert torch.equal(view.cpu(), linear_want(got, w, dtype)) and bool((out[:, :2] == 2).all()) and bool((out[:, n + 2 :] == 2).all())
    want = (got.q.cpu().float() * got.scale.cpu()[:, None]).to(dtype)
    assert torch.equal(dequantize_rows(got, dtype).cpu(), want)
    ids = torch.arange(t - 1, -1, -1)
    for kind in (torch.int64, torch.int32):
        assert torch.equal(int8_embedding(got, ids.to(kind).to(DEVICE), dtype).cpu(), want.flip(0))


@pytest.mark.gpu
@pytest.mark.parametrize(("xk", "wk"), [(1003, 1003), (1003, 1008), (1008, 1003), (1008, 1008), (1024, 1003)])
def test_both_host_paths_copy_what_tiles_cannot_read(xk: int, wk: int, host_path: str) -> None:
    """1003 columns of rows of xk and wk bytes: neither, one or both are copied first."""
    m, n, k = 700, 900, 1003
    xb, wb = codes(m, xk, 1).to(DEVICE), codes(n, wk, 2).to(DEVICE)
    x = Int8Rows(xb[:, :k], scales(m, 3).to(DEVICE))
    w = Int8Rows(wb[:, :k], scales(n, 4).to(DEVICE))
    out = torch.full((m, n + 2), 5.0, dtype=torch.bfloat16, device=DEVICE)
    assert torch.equal(int8_linear(x, w, torch.bfloat16).cpu(), linear_want(x, w, torch.bfloat16))
    assert torch.equal(int8_linear(x, w, torch.bfloat16, out[:, :n]).cpu(), linear_want(x, w, torch.bfloat16))
    assert bool((out[:, n:] == 5).all())


@pytest.mark.gpu
def test_both_host_paths_refuse(host_path: str) -> None:
    x = torch.randn(4, 32, device=DEVICE).half()
    w = torch.ones(32, dtype=torch.float16, device=DEVICE)
    r = quantize_rows(x)
    for op in (lambda: quantize_rows(x.t()), lambda: quantize_rows(x.double()), lambda: quantize_rows(x[0]),
               lambda: rms_norm_rows_int8(x, w[:31], EPS), lambda: rms_norm_rows_int8(x, w.float(), EPS),
               lambda: rms_norm_rows_int8(x, w, 0.0), lambda: add_rms_norm_rows_int8(x, x[:2], w, EPS),
               lambda: add_rms_norm_rows_int8(x[:, :16], x[:, 8:24], w[:16], EPS),
               lambda: add_rms_norm_rows_int8(x[:1].expand(4, 32), x, w, EPS), lambda: silu_mul_int8(x[:, :31]),
               lambda: int8_linear(r, quantize_rows(x[:, :16].contiguous()), torch.float16),
               lambda: int8_linear(r, r, torch.int8), lambda: int8_linear(Int8Rows(r.q, r.scale[:3]), r, torch.float16),
               lambda: int8_linear(r, r, torch.float16, torch.empty(4, 5, dtype=torch.float16, device=DEVICE)),
               lambda: dequantize_rows(r, torch.float64), lambda: int8_embedding(r, torch.zeros(2, device=DEVICE), torch.float16)):  # fmt: skip
        with pytest.raises(ValueError):
            op()
    for op in (lambda: rms_norm_rows_int8(x, w.cpu(), EPS), lambda: add_rms_norm_rows_int8(x, x.cpu(), w, EPS),
               lambda: int8_linear(r, Int8Rows(r.q.cpu(), r.scale.cpu()), torch.float16),
               lambda: int8_embedding(r, torch.zeros(2, dtype=torch.int64), torch.float16)):  # fmt: skip
        with pytest.raises(RuntimeError, match="HIP device only"):
            op()
    assert torch.equal(quantize_rows(x).q, r.q)  # x as it was: nothing was launched


@pytest.mark.gpu
def test_two_streams_at_once() -> None:
    cases = []
    for s in range(2):
        x = quantize_rows(torch.randn(200, 2048, generator=torch.Generator().manual_seed(s)).half().to(DEVICE))
        w = quantize_rows(torch.randn(1000, 2048, generator=torch.Generator().manual_seed(s + 9)).half().to(DEVICE))
        cases.append((x, w, int8_linear(x, w, torch.float16)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got: list[list[torch.Tensor]] = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(int8_linear(cases[i][0], cases[i][1], torch.float16))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert all(torch.equal(o, cases[i][2]) for o in outs)
