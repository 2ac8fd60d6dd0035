"""The 8-bit integer path of a step's projections, as cases that can be timed and compared.

Rows quantised to 8 bits with a scale each (as they stand, after the residual add and RMSNorm, after
SiLU x up), the product of two such matrices with a scale for each token and channel, and the lookup
of rows of an 8-bit table. What is held in 8 bits is returned as the values it stands for, in 16 bits,
beside its scales. ``run`` computes a case in elementary operations of torch, or, where ``own`` is
true, through the package's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-6
HIDDEN, QKV, GATE_UP, VOCAB = 1024, 4096, 6144, 151936
TINY = 2.0**-100  # a row whose largest magnitude is below this is a row of zeros
MOST = 8192**3  # products of the largest case


def listed() -> list[dict]:
    return [
        # A lone sequence's decode step: the qkv projection of one row, all latency.
        linear("linear_1x4096x1024_fp16", 1, QKV, HIDDEN, "fp16"),
        # A small ragged batch against a layer of odd sizes, whose rows are not 16-byte aligned.
        linear("linear_37x1003x1531_bf16", 37, 1003, 1531, "bf16"),
        # The output head on a decode batch of 64: a stream of 156 MB of weights, float32 logits.
        linear("linear_64x151936x1024_fp32", 64, VOCAB, HIDDEN, "fp32"),
        # The gate / up projection of a mixed step of 2751 rows.
        linear("linear_2751x6144x1024_fp16", 2751, GATE_UP, HIDDEN, "fp16"),
        # The largest: a long prompt batch through a wide layer, bound by the matrix cores.
        linear("linear_8192x8192x8192_bf16", 8192, 8192, 8192, "bf16"),
        # The residual add and norm before a projection: a decode batch, and a long prefill of a wide model.
        norm("add_norm_32x1024_fp16", 32, HIDDEN, "fp16", "add"),
        norm("add_norm_8192x8192_bf16", 8192, 8192, "bf16", "add"),
        # Attention outputs before their projection, float32 rows of an odd width.
        norm("quantize_513x2049_fp32", 513, 2049, "fp32", "plain"),
        # SiLU x up before the down projection: a decode batch, and a prefill step's rows.
        {"name": "silu_48x2560_fp16", "kind": "silu", "rows": 48, "cols": 2560, "dtype": "fp16"},
        {"name": "silu_4096x11008_bf16", "kind": "silu", "rows": 4096, "cols": 11008, "dtype": "bf16"},
        # Token embeddings out of the 8-bit table: a decode batch, and a prefill step's tokens.
        {"name": "embed_64x1024_fp16", "kind": "embed", "rows": 64, "cols": HIDDEN, "vocab": VOCAB, "dtype": "fp16"},
        {"name": "embed_16384x4096_bf16", "kind": "embed", "rows": 16384, "cols": 4096, "vocab": 32000,
         "dtype": "bf16"},
    ]  # fmt: skip


def linear(name: str | None, rows: int, out: int, cols: int, dtype: str) -> dict:
    c = {"kind": "linear", "rows": rows, "out": out, "cols": cols, "dtype": dtype}
    return {"name": name, **c} if name else c


def norm(name: str | None, rows: int, cols: int, dtype: str, form: str) -> dict:
    c = {"kind": "norm", "rows": rows, "cols": cols, "dtype": dtype, "form": form}
    return {"name": name, **c} if name else c


def draw(rng) -> dict:  # noqa: ANN001
    def log(lo: int, hi: int) -> int:
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))

    def width(lo: int, hi: int) -> int:
        """Columns: half of them multiples of 64, as a model has them, half any number."""
        n = log(lo, hi)
        return max(64, n // 64 * 64) if rng.random() < 0.5 else n

    kind = rng.choice(["linear", "linear", "linear", "norm", "norm", "silu", "embed"])
    dtype = rng.choice(["fp16", "bf16", "fp16", "bf16", "fp32"])
    if kind == "linear":
        rows = log(1, 16384)
        if rows <= 256 and rng.random() < 0.2:
            return linear(None, rows, log(16384, VOCAB), width(64, 1024), dtype)
        cols = width(16, 16384)
        out = width(16, 16384)
        return linear(None, max(1, min(rows, MOST // (out * cols))), out, cols, dtype)
    cols = width(16, 16384)
    rows = log(1, max(1, min(32768, 8192 * 8192 // cols)))
    if kind == "norm":
        if dtype == "fp32":
            rows = max(1, rows // 2)
        return norm(None, rows, cols, dtype, rng.choice(["plain", "norm", "add", "add"]))
    if kind == "silu":
        return {"kind": "silu", "rows": max(1, rows // 2), "cols": cols, "dtype": dtype}
    vocab = log(1000, min(VOCAB, 200_000_000 // cols))
    return {"kind": "embed", "rows": rows, "cols": cols, "vocab": vocab, "dtype": rng.choice(["fp16", "bf16"])}


def _values(dtype: str) -> torch.dtype:
    """The 16-bit type in which a case's 8-bit rows are returned."""
    return DTYPES["bf16" if dtype == "bf16" else "fp16"]


# ---- inputs ------------------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    rows, cols = case["rows"], case["cols"]

    def normal(*size: int, dtype: torch.dtype = dt, by: float = 1.0, at: float = 0.0) -> torch.Tensor:
        return torch.empty(*size, dtype=dtype, device=DEVICE).normal_(at, by, generator=g)

    def codes(*size: int) -> torch.Tensor:
        """Codes of normally distributed rows whose largest magnitudes are near four deviations."""
        return normal(*size, dtype=torch.float16, by=31.0).round_().clamp_(-127, 127).to(torch.int8)

    def scales(n: int, by: float) -> torch.Tensor:
        return torch.empty(n, device=DEVICE).uniform_(0.5 * by, 1.5 * by, generator=g)

    s = {"case": case, "dtype": dt, "values": _values(case["dtype"])}
    if case["kind"] == "linear":
        s |= {"xq": codes(rows, cols), "xs": scales(rows, 0.03), "wq": codes(case["out"], cols),
              "ws": scales(case["out"], 0.0006)}  # fmt: skip
    elif case["kind"] == "embed":
        s |= {"q": codes(case["vocab"], cols), "scale": scales(case["vocab"], 0.0006),
              "ids": torch.randint(0, case["vocab"], (rows,), generator=g, device=DEVICE)}  # fmt: skip
    elif case["kind"] == "silu":
        s["x"] = normal(rows, 2 * cols)
    else:
        # Every row with a size of its own; in a batch the padding row holds zeros.
        s["x"] = normal(rows, cols).mul_(scales(rows, 1.0)[:, None])
        if rows > 2:
            s["x"][rows // 2] = 0
        if case["form"] != "plain":
            s["weight"] = normal(cols, by=0.1, at=1.0)
        if case["form"] == "add":
            s["y"] = normal(rows, cols, by=0.5)
            if rows > 2:
                s["y"][rows // 2] = 0
    return s


# ---- one pass ----------------------------------------------------------------------------
def run(s: dict) -> dict:
    kind = s["case"]["kind"]
    if own:
        return _own(s, kind)
    if kind == "linear":
        acc = s["xq"].float() @ s["wq"].float().t()
        return {"out": (acc * s["xs"][:, None] * s["ws"]).to(s["dtype"])}
    if kind == "embed":
        return {"out": (s["q"][s["ids"]].float() * s["scale"][s["ids"]][:, None]).to(s["dtype"])}
    if kind == "silu":
        gate, up = s["x"].float().chunk(2, dim=1)
        return _quantized(gate / (1 + torch.exp(-gate)) * up, None, s["values"])
    if s["case"]["form"] == "plain":
        return _quantized(s["x"].float(), None, s["values"])
    if s["case"]["form"] == "add":
        s["x"].copy_(s["x"].float() + s["y"].float())
    x = s["x"].float()
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    got = _quantized(x * s["weight"].float(), r, s["values"])
    return {**got, "x": s["x"]} if s["case"]["form"] == "add" else got


def _quantized(v: torch.Tensor, r: torch.Tensor | None, dtype: torch.dtype) -> dict:
    """Rows of ``v`` (times ``r``) as 8-bit codes with a scale each, and the values they stand for."""
    top = v.abs().amax(1, keepdim=True)
    top = torch.where(top < TINY, 0.0, top)
    q = torch.where(top > 0, torch.round(v * (127 / top)), 0.0)
    scale = top / 127 if r is None else top / 127 * r
    return {"values": (q * scale).to(dtype), "scale": scale[:, 0]}


def _own(s: dict, kind: str) -> dict:
    from tinyserve_amd import hip_int8

    if kind == "linear":
        x, w = hip_int8.Int8Rows(s["xq"], s["xs"]), hip_int8.Int8Rows(s["wq"], s["ws"])
        return {"out": hip_int8.int8_linear(x, w, s["dtype"])}
    if kind == "embed":
        return {"out": hip_int8.int8_embedding(hip_int8.Int8Rows(s["q"], s["scale"]), s["ids"], s["dtype"])}
    if kind == "silu":
        rows = hip_int8.silu_mul_int8(s["x"])
    elif s["case"]["form"] == "plain":
        rows = hip_int8.quantize_rows(s["x"])
    elif s["case"]["form"] == "norm":
        rows = hip_int8.rms_norm_rows_int8(s["x"], s["weight"], EPS)
    else:
        rows = hip_int8.add_rms_norm_rows_int8(s["x"], s["y"], s["weight"], EPS)
    got = {"values": hip_int8.dequantize_rows(rows, s["values"]), "scale": rows.scale}
    return {**got, "x": s["x"]} if kind == "norm" and s["case"]["form"] == "add" else got


# ---- what a pass cannot do without -------------------------------------------------------
def work(case: dict) -> dict:
    rows, cols, e = case["rows"], case["cols"], BYTES[case["dtype"]]
    if case["kind"] == "linear":
        out = case["out"]
        return {"bytes": rows * cols + out * cols + rows * out * e + 4 * (rows + out), "flops": 2 * rows * out * cols}
    if case["kind"] == "embed":
        seen = min(rows, case["vocab"])  # rows of the table, at most
        return {"bytes": seen * (cols + 4) + rows * (8 + cols * e), "flops": rows * cols}
    n = rows * cols
    if case["kind"] == "silu":
        return {"bytes": n * (2 * e + 2) + 4 * rows, "flops": 8 * n}
    moved = {"plain": e, "norm": e, "add": 3 * e}[case["form"]]
    return {"bytes": n * (moved + 2) + 4 * rows + (cols * e if case["form"] != "plain" else 0), "flops": 6 * n}


# ---- the definitions in 64 bits ----------------------------------------------------------
def exact(case: dict, seed: int) -> dict | None:
    s = prepare(case, seed)
    if case["kind"] == "linear":
        return {"out": torch.mm(s["xq"].double() * s["xs"].double().unsqueeze(1),
                                (s["wq"].double() * s["ws"].double().unsqueeze(1)).T.contiguous())}  # fmt: skip
    if case["kind"] == "embed":
        return {"out": s["q"].index_select(0, s["ids"]).double()
                * s["scale"].double().index_select(0, s["ids"]).unsqueeze(1)}  # fmt: skip
    x = s["x"].double()
    if case["kind"] == "silu":
        n = case["cols"]
        y = x[:, :n] * torch.sigmoid(x[:, :n]) * x[:, n:]
    elif case["form"] == "plain":
        y = x
    else:
        if case["form"] == "add":
            x = (x + s["y"].double()).to(s["dtype"]).double()
        y = x * s["weight"].double() * (x.pow(2).sum(1, keepdim=True) / case["cols"] + EPS).rsqrt()
    step = y.abs().max(1, keepdim=True).values / 127
    got = {"values": torch.round(y / step.clamp_min(TINY)) * step, "scale": step.squeeze(1)}
    return {**got, "x": x} if case["kind"] == "norm" and case["form"] == "add" else got
