"""A model whose projections are held in 8 bits: loading, its layers, and generation through the engine."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import device_model, random_tokens
from plain import qwen2_plain as plain
from test_config_weights import TINY_B, make_model_folder
from test_kernels import make_ctx
from llm_inference_b200 import models  # noqa: F401
from llm_inference_b200.config import parse_config
from llm_inference_b200.cli.presets import PRESETS
from llm_inference_b200.engine.loading import load_model
from llm_inference_b200.parts import float8
from llm_inference_b200.parts.model import Model

gpu = pytest.mark.gpu

SHAPE = dict(PRESETS["tiny-a"], hidden_size=256, num_attention_heads=4, num_key_value_heads=2, intermediate_size=704, vocab_size=500, num_hidden_layers=3,
             max_position_embeddings=512)


def test_loading(tmp_path):
    folder = make_model_folder(tmp_path / "m", TINY_B, seed=3)
    wide = load_model(folder, "bfloat16", "cpu")
    model = load_model(folder, "bfloat16", "cpu", weights="float8")
    assert model.weights == "float8" and wide.weights is None
    for block, other in zip(model.blocks, wide.blocks):
        for part, beside, names in ((block.mixer, other.mixer, ("w_qkv", "w_o")), (block.feed_forward, other.feed_forward, ("w_gate_up", "w_down"))):
            assert part.float8 and not beside.float8
            for name in names:
                rows, whole = getattr(part, name), getattr(beside, name)
                assert rows.constant and rows.shape == tuple(whole.shape)
                again = float8.from_tensor(whole)
                assert torch.equal(rows.values.view(torch.uint8), again.values.view(torch.uint8)) and torch.equal(rows.scales, again.scales)
            assert part.weight_bytes() < 0.6 * beside.weight_bytes()
    assert model.weight_bytes() < wide.weight_bytes()
    before = model.blocks[0].mixer.w_qkv
    model.to_float8()  # once is enough
    assert model.blocks[0].mixer.w_qkv is before


def test_refusals(tmp_path):
    folder = make_model_folder(tmp_path / "m", TINY_B, seed=3)
    with pytest.raises(ValueError, match="bfloat16"):
        load_model(folder, "float32", "cpu", weights="float8")
    with pytest.raises(ValueError, match="unknown weights"):
        load_model(folder, "bfloat16", "cpu", weights="int4")
    for name in ("tunadra-small", "tosipel-small", "lerorax-small"):
        entry, config = parse_config(PRESETS[name])
        model = Model(entry.recipe(config))
        model.dtype = torch.bfloat16
        with pytest.raises(ValueError, match="layer 0 cannot"):
            model.to_float8()


def rows8(v: np.ndarray) -> np.ndarray:
    """Rows as they are after a trip through e4m3 with a scale each."""
    scale = np.maximum(np.abs(v).max(axis=-1, keepdims=True) / 448.0, 2.0**-126)
    u = v / scale
    step = np.exp2(np.maximum(np.frexp(u)[1] - 1, -6) - 3.0)
    return np.round(u / step) * step * scale


def plain_float8(config: dict, weights, tokens) -> np.ndarray:
    """The plain model with every product's operands taken through 8 bits."""

    def linear(h, name, bias=None):
        return plain.linear(rows8(h), rows8(weights[name]), None if bias is None else weights[bias])

    x = plain.embed(weights["model.embed_tokens.weight"], tokens)
    heads, kv_heads, eps = config["num_attention_heads"], config["num_key_value_heads"], config["rms_norm_eps"]
    dim = config["hidden_size"] // heads
    for layer in range(config["num_hidden_layers"]):
        p = f"model.layers.{layer}."
        h = plain.rms_norm(x, weights[p + "input_layernorm.weight"], eps)
        q, k, v = (linear(h, f"{p}self_attn.{n}_proj.weight", f"{p}self_attn.{n}_proj.bias") for n in "qkv")
        positions = np.arange(len(tokens))
        q = plain.rope(q.reshape(-1, heads, dim), positions, config["rope_theta"])
        k = plain.rope(k.reshape(-1, kv_heads, dim), positions, config["rope_theta"])
        x = x + linear(plain.attention(q, k, v.reshape(-1, kv_heads, dim), dim**-0.5), p + "self_attn.o_proj.weight")
        h = plain.rms_norm(x, weights[p + "post_attention_layernorm.weight"], eps)
        gate, up = linear(h, p + "mlp.gate_proj.weight"), linear(h, p + "mlp.up_proj.weight")
        x = x + linear(gate / (1 + np.exp(-gate)) * up, p + "mlp.down_proj.weight")
    return plain.output_logits(config, weights, x)


@pytest.fixture(scope="module")
def built():
    model, config, weights = device_model(SHAPE, 7, "bfloat16", 0.05)
    model.to_float8()
    return model, config, weights


def make_engine(model, **options):
    from llm_inference_b200 import create_engine

    return create_engine(model=model, max_num_sequences=8, max_model_length=512, kv_cache_bytes=64 << 20, **options)


@gpu
def test_logits_of_prompts_and_decoded_tokens(built):
    """Against the plain model with the same operands in 8 bits. What a bfloat16 rounding moves across an e4m3 border comes out a whole step away, and a stream
    that differs by that moves more across the next layers' borders, up to where the two sides' roundings have nothing to do with each other. Both carry
    rounding noise of the same size n (the plain 8-bit model's distance from the one without), so they are then sqrt(2) n = 1.41 n apart,
    before that less, and the engine is n (1 +- its spread) from the model without 8 bits: 1.5 n bounds both. (A fixed bound of 7 % for the first, from one
    product's roundings alone, left the later layers' out: with these weights n is 10 to 20 %.) Wrong weights, scales or rows are off by 100 %."""
    from llm_inference_b200.cache.paged_cache import PagedCache
    from llm_inference_b200.engine.runner import ModelRunner, StepEntry

    model, config, weights = built
    cache = PagedCache(model.cache_specs(), dtype=torch.bfloat16, device=model.device, page_size=64, max_num_sequences=4, max_model_length=512, step_tokens=512,
                       num_pages=64)
    runner = ModelRunner(model, cache, max_batch_tokens=512)
    rng = np.random.default_rng(3)
    prompts = [random_tokens(rng, 500, n) for n in (37, 130, 1)]
    for rid, prompt in enumerate(prompts, 1):
        cache.open(rid)
    logits = runner.step([StepEntry(rid, p, (len(p) - 1,)) for rid, p in enumerate(prompts, 1)], check=True).double().cpu().numpy()
    for turn in range(3):  # the third is replayed from a graph
        for row, prompt in zip(logits, prompts):
            want = plain_float8(config, weights, prompt)[-1]
            whole = plain.output_logits(config, weights, plain.hidden_states(config, weights, prompt))[-1]
            noise = np.linalg.norm(want - whole)
            assert np.linalg.norm(row - want) < 1.5 * noise and np.linalg.norm(row - whole) < 1.5 * noise
        new = [int(t) for t in rng.integers(0, 500, 3)]
        for prompt, token in zip(prompts, new):
            prompt.append(token)
        logits = runner.step([StepEntry(rid, (t,), (0,)) for rid, t in enumerate(new, 1)], check=True).double().cpu().numpy()


@gpu
def test_generation(built):
    """The same greedy tokens with and without graphs and steps launched ahead, alone and beside others of another length."""
    model, _, _ = built
    rng = np.random.default_rng(4)
    prompts = [random_tokens(rng, 500, n) for n in (5, 70, 200)]
    with make_engine(model, weights="float8") as engine:
        alone = [engine.generate(p, max_new_tokens=24) for p in prompts]
        assert engine.generate(prompts[0], max_new_tokens=24) == alone[0]
    with make_engine(model, cuda_graphs=False, run_ahead=False) as engine:
        assert [engine.generate(p, max_new_tokens=24) for p in prompts] == alone
    with make_engine(model, decode_kernel="resident", fold_norms=True) as engine:  # neither has a form for 8 bits: the chain of kernels
        assert engine.generate(prompts[1], max_new_tokens=24) == alone[1]


@gpu
def test_engine_refusals(built):
    from llm_inference_b200.engine.loading import random_model

    model, _, _ = built
    with pytest.raises(ValueError, match="plain kernels"):
        make_engine(model, kernels="plain")
    wide = random_model(parse_config(SHAPE)[1], 1)
    with pytest.raises(ValueError, match="compute dtype"):
        make_engine(wide, weights="float8")


@gpu
@pytest.mark.parametrize("tokens", [1, 9, 40, 300])
def test_a_layers_operators_as_they_are_used(built, tokens):
    """Norm with the residual's add, gated product, its rows to 8 bits and the down product with the residual in its epilogue: against 64 bits, each
    stage from what the stage before left, and the part's own forward bit by bit."""
    from llm_inference_b200.csrc.library import kernels
    from test_float8 import check_rows, half_step, slope, sum_off, wide_activation, wide_product

    model, _, _ = built
    ff, norm = model.blocks[1].feed_forward, model.blocks[1].feed_forward_norm
    ctx = make_ctx(kernels(), positions=[0] * tokens)
    ctx.buffer = lambda name, shape, dtype=None, per_token=True: ctx.workspace.get(name, shape, dtype or torch.bfloat16, per_token=per_token)  # as a step's
    torch.manual_seed(tokens)
    x, delta = torch.randn(tokens, 256, device="cuda") * 2, torch.randn(tokens, 256, device="cuda").bfloat16()
    s = x + delta.float()
    rows = norm.forward_float8(ctx, x, delta)
    assert torch.equal(x, s)
    v = s.double()
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + norm.eps) * norm.weight.double()
    check_rows(rows, v, 2.0**-18, 2.0**-21)
    act = float8.linear_gated(ctx, rows, ff.w_gate_up, torch.empty(tokens, 704, device="cuda", dtype=torch.bfloat16))
    y, magnitudes = wide_product(rows, ff.w_gate_up)
    off = sum_off(256, magnitudes, torch.bfloat16)
    g, u, og, ou = y[:, 0::2], y[:, 1::2], off[:, 0::2], off[:, 1::2]
    a = wide_activation(g, "silu")
    want = a * u
    assert torch.all((act.double() - want).abs() <= slope(g, og, "silu") * (u.abs() + ou) + a.abs() * ou + (half_step(torch.bfloat16) * 1.01 + 2.0**-22) * want.abs())
    rows8_ = float8.quantize(ctx, act, float8.empty_rows(tokens, 704, "cuda:0"))
    check_rows(rows8_, act.double(), 2.0**-23, 2.0**-22)
    into = float8.linear(ctx, rows8_, ff.w_down, s.clone(), residual=s)
    y, magnitudes = wide_product(rows8_, ff.w_down)
    want = s.double() + y
    assert torch.all((into.double() - want).abs() <= sum_off(704, magnitudes, torch.float32) + s.double().abs() * 2.0**-23 + half_step(torch.float32) * 1.01 * want.abs())
    branch = float8.linear(ctx, rows8_, ff.w_down, torch.empty(tokens, 256, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(ff.forward(ctx, norm.forward_float8(ctx, s.clone(), None)), branch)
    assert int(ctx.err.item()) == 0
