"""The 8-bit attention sublayer stage by stage, and batches of several requests."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import device_model, random_tokens
from plain import qwen2_plain as plain
from test_float8 import check_rows, half_step, sum_off, wide_product
from test_float8_engine import SHAPE, plain_float8
from test_kernels import make_ctx

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("starts,runs", [([11], [1]), ([70, 5, 0], [1, 1, 1]), ([9, 0, 3], [1, 40, 21]), ([0], [300])])
def test_attention_stage_by_stage(starts, runs):
    """Each stage in 64 bits from what the stage before left. Biases are of the products' own size, so that a lost or swapped one shows."""
    from llm_inference_b200.csrc.library import kernels
    from llm_inference_b200.parts.context import CacheView

    model, config, _ = device_model(SHAPE, 7, "bfloat16", 0.05)
    mixer, norm = model.blocks[1].mixer, model.blocks[1].mixer_norm
    heads, kv_heads, dim, hidden = 4, 2, 64, 256
    torch.manual_seed(70)
    mixer.b_qkv = torch.randn((heads + 2 * kv_heads) * dim, device="cuda")
    model.to_float8()
    page, per_request = 16, 24
    tables = np.random.default_rng(5).permutation(len(runs) * per_request).astype(np.int32).reshape(len(runs), per_request)
    keys = torch.randn(tables.size, kv_heads, page, dim, device="cuda").bfloat16()
    values = torch.randn_like(keys)
    view = CacheView(0, True, keys, values, torch.from_numpy(tables).cuda(), tables.size, per_request, page)
    positions = [s + i for s, r in zip(starts, runs) for i in range(r)]
    requests = [i for i, r in enumerate(runs) for _ in range(r)]
    t = len(positions)
    ctx = make_ctx(kernels(), positions=positions, token_seq=requests, starts=starts, runs=runs)
    ctx.buffer = lambda name, shape, dtype=None, per_token=True: ctx.workspace.get(name, shape, dtype or torch.bfloat16, per_token=per_token)  # as a step's
    x = torch.randn(t, hidden, device="cuda") * 2
    h = norm.forward_float8(ctx, x, None)
    branch = mixer.forward(ctx, view, h)
    assert int(ctx.err.item()) == 0

    qkv = ctx.buffer("qkv", (t, (heads + 2 * kv_heads) * dim))
    y, magnitudes = wide_product(h, mixer.w_qkv)
    want = y + mixer.b_qkv.double()
    off = sum_off(hidden, magnitudes + mixer.b_qkv.double().abs(), torch.bfloat16)
    assert torch.all((qkv.double() - want).abs() <= off + half_step(torch.bfloat16) * 1.01 * want.abs())

    # Rotation: two products of 32 bits with sines and cosines good to 2^-18 (positions below 2^9, angles rounded to 2^-24 of themselves: 2^-15), one rounding.
    parts = qkv.double().cpu().numpy()
    q = parts[:, : heads * dim].reshape(t, heads, dim)
    k = parts[:, heads * dim : (heads + kv_heads) * dim].reshape(t, kv_heads, dim)
    v = parts[:, (heads + kv_heads) * dim :].reshape(t, kv_heads, dim)

    def rotated(got, before):
        want = plain.rope(before, positions, config["rope_theta"])
        half = np.abs(before[..., : dim // 2]) + np.abs(before[..., dim // 2 :])
        size = np.concatenate([half, half], axis=-1)
        assert np.all(np.abs(got - want) <= 2.0**-14 * size + half_step(torch.bfloat16) * 1.01 * np.abs(want))

    turned = ctx.buffer("q", (t, heads * dim)).double().cpu().numpy().reshape(t, heads, dim)
    rotated(turned, q)
    held_k, held_v = keys.double().cpu().numpy(), values.double().cpu().numpy()
    at = [(tables[r, p // page], p % page) for r, p in zip(requests, positions)]
    rotated(np.stack([held_k[a, :, o] for a, o in at]), k)
    assert np.array_equal(np.stack([held_v[a, :, o] for a, o in at]), v)

    # Attention over the cache as it now is: weights are rounded to bfloat16 (2^-8 of each), and their sum's counterpart, and the output once more.
    attn = ctx.buffer("attn", (t, heads * dim))
    got = attn.double().cpu().numpy().reshape(t, heads, dim)
    for i, (r, p) in enumerate(zip(requests, positions)):
        seen_k = np.stack([held_k[tables[r, j // page], :, j % page] for j in range(p + 1)])
        seen_v = np.stack([held_v[tables[r, j // page], :, j % page] for j in range(p + 1)])
        for head in range(heads):
            weights = plain.softmax(seen_k[:, head // 2] @ turned[i, head] * dim**-0.5)
            want, size = weights @ seen_v[:, head // 2], weights @ np.abs(seen_v[:, head // 2])
            assert np.all(np.abs(got[i, head] - want) <= 3.1 * 2.0**-8 * size), (i, head)

    rows = mixer_rows(ctx, t, heads * dim)
    check_rows(rows, attn.double(), 2.0**-23, 2.0**-22)
    want, magnitudes = wide_product(rows, mixer.w_o)
    assert torch.all((branch.double() - want).abs() <= sum_off(heads * dim, magnitudes, torch.bfloat16) + half_step(torch.bfloat16) * 1.01 * want.abs())


def mixer_rows(ctx, rows: int, columns: int):
    from llm_inference_b200.parts import float8

    return float8.buffer_rows(ctx, "attn8", rows, columns)


@gpu
def test_requests_that_share_batches():
    """Decoded tokens beside prompt portions, and three decoded requests in a step of four: against the plain model with its operands in 8 bits, request by
    request. The bound is that of the logits of single requests: both sides' rounding noise is as large as the distance n between the plain
    models with and without 8 bits, and 1.5 n bounds their distance. Another request's rows would be off by all of a logit row, seven times that or more."""
    from llm_inference_b200.cache.paged_cache import PagedCache
    from llm_inference_b200.engine.runner import ModelRunner, StepEntry

    model, config, weights = device_model(SHAPE, 7, "bfloat16", 0.05)
    model.to_float8()
    cache = PagedCache(model.cache_specs(), dtype=torch.bfloat16, device=model.device, page_size=64, max_num_sequences=4, max_model_length=512, step_tokens=512,
                       num_pages=64)
    runner = ModelRunner(model, cache, max_batch_tokens=512)
    rng = np.random.default_rng(9)
    for rid in (1, 2, 3):
        cache.open(rid)
    fed: dict[int, list[int]] = {1: [], 2: [], 3: []}
    # Tokens of requests 1, 2, 3 in each step; the last four steps are decoded tokens only (the later ones replayed from a graph).
    for counts in ((37, 1, 0), (1, 1, 70), (1, 1, 60), (1, 12, 1), (1, 1, 1), (1, 1, 1), (1, 1, 1), (1, 1, 1)):
        entries = []
        for rid, count in enumerate(counts, 1):
            if count:
                tokens = random_tokens(rng, 500, count)
                fed[rid] += tokens
                entries.append(StepEntry(rid, tokens, (count - 1,)))
        logits = runner.step(entries, check=True).double().cpu().numpy()
        for row, entry in zip(logits, entries):
            sequence = fed[entry.request_id]
            want = plain_float8(config, weights, sequence)[-1]
            whole = plain.output_logits(config, weights, plain.hidden_states(config, weights, sequence))[-1]
            noise = np.linalg.norm(want - whole)
            assert np.linalg.norm(row - want) < 1.5 * noise and np.linalg.norm(row - whole) < 1.5 * noise
    assert runner.graph_replays >= 1
