"""The decode step with 8-bit weights (``decode_step.int8_weights``) on the GPU.

Each call that the step makes of ``hip_int8`` is checked against its definition on the inputs
that it got (the products bit for bit), so nothing adds up over the layers. The step as a whole
is held to the float32 step with the same (dequantised) weights, whose only difference is the
rounding of activations: codes are off by at most half of a / 127, so by a / 440 in the root
mean square, and rows whose largest magnitude a is 3 to 6 deviations are off by 1.4% at most
where they enter a product. The products of a row's path, at most five a layer (one of them
twice, through k and v) and the head, add at most in quadrature: sqrt(6 * 2 + 1) * 1.4% = 5% of
the logits at two layers; the bound is 10%, where a part taken from the wrong place gives
about 100%.
"""

from __future__ import annotations

import pytest
import torch

from tests.test_decode_step import DEVICE, TINY, reference_step, setup
from tests.test_hip_int8 import EPS, check_rows, linear_want, same
from tinyserve_amd import decode_step, hip_int8
from tinyserve_amd.decode_step import DecodeGraph, DecodeStep, int8_weights, rope_tables
from tinyserve_amd.hip_int8 import Int8Rows, dequantize_rows
from tinyserve_amd.step_inputs import DecodeInputs, build_batch, fill_decode_inputs

pytestmark = pytest.mark.gpu
LENS = [9, 30, 2, 17, 5]


def dequantized(w: dict) -> dict[str, torch.Tensor]:
    return {k: dequantize_rows(v, torch.float32) if isinstance(v, Int8Rows) else v.float() for k, v in w.items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [5, 8])
def test_step_with_8_bit_weights(dtype: torch.dtype, rows: int, monkeypatch: pytest.MonkeyPatch) -> None:
    w, pool, _, inp = setup(LENS, rows, dtype, seed=13)
    w8 = int8_weights(w)
    assert all(isinstance(v, Int8Rows) == (w[k].dim() == 2) for k, v in w8.items())
    calls: list[str] = []

    def watched(name: str, form: str):  # noqa: ANN202
        kernel = getattr(hip_int8, name)

        def call(x: torch.Tensor, *rest):  # noqa: ANN002, ANN202
            c = {"x": x.cpu().clone()}
            if form == "add":
                c["y"] = rest[0].cpu()
            if form in ("norm", "add"):
                c["w"] = rest[-2].cpu()
                assert rest[-1] == EPS
            got = kernel(x, *rest)
            check_rows(form, got, c)
            calls.append(form)
            return got

        monkeypatch.setattr(hip_int8, name, call)

    for name, form in (("quantize_rows", "plain"), ("rms_norm_rows_int8", "norm"), ("add_rms_norm_rows_int8", "add"),
                       ("silu_mul_int8", "silu")):  # fmt: skip
        watched(name, form)
    linear = hip_int8.int8_linear

    def watched_linear(x: Int8Rows, wt: Int8Rows, dt: torch.dtype) -> torch.Tensor:
        got = linear(x, wt, dt)
        assert same(got.cpu(), linear_want(x, wt, dt))
        calls.append("linear")
        return got

    monkeypatch.setattr(hip_int8, "int8_linear", watched_linear)
    kr, vr = pool.k.float().cpu(), pool.v.float().cpu()
    want = reference_step(TINY, dequantized(w8), kr, vr, inp, pool.block_size)[: len(LENS)]
    step = DecodeStep(TINY, w8, pool)
    assert step.projections == "int8"
    got = step.forward(inp)
    assert got.shape == (rows, TINY.vocab) and got.dtype == torch.float32
    layer = ["linear", "plain", "linear", "add", "linear", "silu", "linear"]
    assert calls == ["norm", *layer, *(["add", *layer] * (TINY.num_layers - 1)), "add", "linear"]
    off = float((got[: len(LENS)].cpu() - want).norm() / want.norm())
    print(f"[int8 step {dtype}] logits off by {off:.3g} of their norm")
    assert off <= 0.1


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_graph_replays_equal_the_eager_step(dtype: torch.dtype) -> None:
    w, pool, tabs, inp = setup(LENS, 8, dtype, seed=7)
    step = DecodeStep(TINY, int8_weights(w), pool)
    graph = DecodeGraph(step.forward, inp)
    spare = iter(range(pool.pad_block - 3, pool.pad_block))
    for it in range(3):
        for t in tabs:
            t.num_tokens += 1
            if len(t.blocks) * t.block_size < t.num_tokens:
                t.blocks.append(next(spare))
        fill_decode_inputs(inp, [((it * 5 + j) % TINY.vocab, t) for j, t in enumerate(tabs)], pool.pad_block)
        k0, v0 = pool.k.clone(), pool.v.clone()
        got = graph.replay().clone()
        k1, v1 = pool.k.clone(), pool.v.clone()
        pool.k.copy_(k0)
        pool.v.copy_(v0)
        assert torch.equal(got, step.forward(inp))
        assert torch.equal(pool.k, k1) and torch.equal(pool.v, v1)
        torch.randn(1 << 20, device=DEVICE).sum().item()


def test_decode_only_batch_equals_the_decode_step() -> None:
    w, pool, tabs, _ = setup(LENS, len(LENS), torch.float16, seed=5)
    items = [((7 * i + 3) % TINY.vocab, t) for i, t in enumerate(tabs)]
    batch = build_batch([([tok], tab) for tok, tab in items], DEVICE)
    inp = DecodeInputs.empty(len(LENS), batch.block_tables.shape[1], DEVICE)
    fill_decode_inputs(inp, items, pool.pad_block)
    k0, v0 = pool.k.clone(), pool.v.clone()
    step = DecodeStep(TINY, int8_weights(w), pool)
    want = step.forward(inp)
    pool.k.copy_(k0)
    pool.v.copy_(v0)
    assert torch.equal(step.forward_batch(batch), want)


def test_mixed_step_matches_the_reference_step() -> None:
    """Prompts of one and many tokens beside decodes: 300 rows, so that products run in tiles."""
    cached, new = [5, 0, 9, 2, 0], [3, 255, 1, 1, 40]
    w, pool, tabs, _ = setup([c + n for c, n in zip(cached, new)], len(cached), torch.float16, seed=17)
    g = torch.Generator(device="cpu").manual_seed(19)
    batch = build_batch([(torch.randint(0, TINY.vocab, (n,), generator=g).tolist(), t) for n, t in zip(new, tabs)], DEVICE)
    w8 = int8_weights(w)
    kr, vr = pool.k.float().cpu(), pool.v.float().cpu()
    want = reference_step(TINY, dequantized(w8), kr, vr, batch, pool.block_size)[batch.last_rows.cpu()]
    got = DecodeStep(TINY, w8, pool).forward_batch(batch).cpu()
    assert got.shape == (len(new), TINY.vocab)
    assert float((got - want).norm() / want.norm()) <= 0.1


def test_layers_one_by_one_give_the_step() -> None:
    w, pool, _, inp = setup([3, 17, 40, 9, 1, 22, 5, 13], 8, torch.float16)
    w8 = int8_weights(w)
    step = DecodeStep(TINY, w8, pool)
    want = step.forward(inp)
    cos, sin = rope_tables(TINY.head_dim, TINY.rope_theta, inp.positions)
    table = w8["model.embed_tokens.weight"]
    x = hip_int8.int8_embedding(table, inp.token_ids, torch.float16)
    for i in range(TINY.num_layers):
        x = step.layer(i, x, cos, sin, inp.slots, lambda i, q: step._attention(i, q, inp))
    h = hip_int8.rms_norm_rows_int8(x, w8["model.norm.weight"], TINY.rms_norm_eps)
    assert torch.equal(hip_int8.int8_linear(h, table, torch.float32), want)


def test_projection_choice() -> None:
    w, pool, _, _ = setup([3], 1, torch.float16)
    w8 = int8_weights(w)
    assert DecodeStep(TINY, w8, pool, projections="int8").projections == "int8"
    for weights, projections in ((w, "int8"), (w8, "rows"), (w8, "library")):
        with pytest.raises(ValueError, match="projections"):
            DecodeStep(TINY, weights, pool, projections=projections)
    assert decode_step.DecodeStep(TINY, w, pool).projections == "rows"
