"""The decode loops over 4-bit weights and with sampled tokens: a step's logits against the same step over
the dequantized weights, sampled tokens against the definition applied to the loop's own logits, eager runs
against replayed graphs, and what the loop refuses."""
import dataclasses

import pytest
import torch

from rdkv_amd import blockwise_decode as bw
from rdkv_amd import fast_decode, knapsack_solver as ks, sampling, weight_quant as wq
from tests.gpu_util import DEV, require_gpu
from tests.test_gpu_decode_loop import T_PROMPT, VOCAB, _build_setup, _mixed_bits, _pack
from tests.test_gpu_sampling import oracle


@pytest.fixture(scope="module")
def setup():
    require_gpu()
    model, prompt, pre, kv = _build_setup()
    return model, pre.logits[0, -1], kv


def _decode(model, kv, first, n, **kw):
    return fast_decode.greedy_decode_fast(model, _pack(kv, *_mixed_bits(11)), first, n, [], torch.device(DEV), T_PROMPT, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("group,lm_head", [(32, True), (128, True), (64, False)])
def test_loop_over_4_bit_weights(setup, group, lm_head):
    model, first, kv = setup
    W = fast_decode.quantize_weights(model, group, lm_head)
    assert isinstance(W.lm_head_weight, wq.QuantizedWeight) == lm_head
    assert not isinstance(fast_decode.pre_extract_weights(model).lm_head_weight, wq.QuantizedWeight)
    ids, logits = _decode(model, kv, first, 5, weights=W, return_logits=True)
    # the same loop over the dequantized values (rounded to fp16: 2^-11 of each weight more)
    names = ("qkv_weight", "o_proj_weight", "gate_up_weight", "down_proj_weight")
    V = dataclasses.replace(W, layers=[dataclasses.replace(lq, **{n: wq.dequantize_weight(getattr(lq, n)) for n in names})
                                       for lq in W.layers])
    if lm_head:
        V = dataclasses.replace(V, lm_head_weight=wq.dequantize_weight(W.lm_head_weight))
    exp_ids, exp = _decode(model, kv, first, 5, weights=V, return_logits=True)
    # the fp16 model's own bar for logits whose intermediate roundings differ (5e-2 of the largest)
    assert float((logits[0] - exp[0]).abs().max()) <= 5e-2 * float(exp[0].abs().max())
    assert float((logits[0] - exp[0]).norm()) <= 1e-2 * float(exp[0].norm())
    assert ids[0] == exp_ids[0] == int(first.argmax()) and all(t == int(l.argmax()) for t, l in zip(ids[1:], logits))
    assert _decode(model, kv, first, 5, weights=W) == ids
    assert _decode(model, kv, first, 5, weights=W, use_cuda_graph=True) == ids


@pytest.mark.gpu
@pytest.mark.parametrize("settings", [dict(temperature=0.9, top_p=0.95), dict(temperature=1.5, top_k=20, min_p=0.01), dict()])
@pytest.mark.parametrize("quantized", [False, True])
def test_sampled_loop(setup, settings, quantized):
    model, first, kv = setup
    weights = fast_decode.quantize_weights(model) if quantized else None
    u = torch.rand(9, generator=torch.Generator().manual_seed(17)).to(DEV)
    s = sampling.Sampling(**settings)
    ids, logits = _decode(model, kv, first, 8, weights=weights, sampling=s, uniforms=u, return_logits=True)
    seen = [first.float().cpu().view(1, -1)] + logits
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    for i, token in enumerate(ids):
        assert token == oracle(seen[i][0].double().numpy(), float(u[i]), f32(s.temperature), s.top_k, f32(s.top_p), f32(s.min_p))[0]
    for graph in (False, True):
        assert _decode(model, kv, first, 8, weights=weights, sampling=s, uniforms=u, use_cuda_graph=graph) == ids
    assert _decode(model, kv, first, 1, weights=weights, sampling=s, uniforms=u) == ids[:1]
    assert _decode(model, kv, first, 0, sampling=s, uniforms=u[:0]) == []


@pytest.mark.gpu
def test_temperature_zero_is_the_greedy_loop(setup):
    model, first, kv = setup
    u = torch.rand(6, device=DEV)
    greedy = _decode(model, kv, first, 6)
    assert _decode(model, kv, first, 6, sampling=sampling.Sampling(temperature=0.0), uniforms=u) == greedy
    assert _decode(model, kv, first, 6, sampling=sampling.Sampling(top_k=1), uniforms=u, use_cuda_graph=True) == greedy


@pytest.mark.gpu
def test_loop_refusals(setup):
    model, first, kv = setup
    s, u = sampling.Sampling(), torch.rand(4, device=DEV)
    with pytest.raises(ValueError):
        _decode(model, kv, first, 2, sampling=s)
    with pytest.raises(ValueError):
        _decode(model, kv, first, 2, uniforms=u)
    for bad in (u[:1], u.double(), u.view(2, 2), u.cpu()):
        with pytest.raises(AssertionError):
            _decode(model, kv, first, 2, sampling=s, uniforms=bad)
    with pytest.raises(RuntimeError, match="no token to draw"):
        _decode(model, kv, torch.full_like(first, float("-inf")), 2, sampling=s, uniforms=u)


@pytest.mark.gpu
def test_blockwise_loop_over_4_bit_weights(setup):
    model, first, kv = setup
    W = fast_decode.quantize_weights(model)
    config = bw.BlockwiseRDKVConfig(block_size=8, block_budget_tokens=4, k_budget_ratio=0.5, obs_window=4, pool_kernel_size=3,
                                    pool_padding="reflect", v_bit_options=torch.tensor([0., 2, 4, 8, 16]),
                                    k_bit_options=torch.tensor([0., 2, 4, 8]), epsilon_v=ks.DEFAULT_EPSILON_V,
                                    epsilon_k=ks.DEFAULT_EPSILON_K, correctness_check=True)
    runs = []
    for graph in (False, True):
        ids, report = bw.greedy_decode_blockwise(
            model=model, dual_cache=_pack(kv, *_mixed_bits(11)), next_token_logits=first, max_new_tokens=20, eos_token_ids=[],
            primary_device=torch.device(DEV), decode_position_start=T_PROMPT, config=config, use_cuda_graph=graph, weights=W)
        assert report["num_compressed_decode_blocks"] > 0 and all(0 <= t < VOCAB for t in ids)
        runs.append(ids)
    assert runs[0] == runs[1] and runs[0][:8] == _decode(model, kv, first, 8, weights=W)


def test_quantize_weights_has_no_cpu_path():
    from transformers import LlamaConfig, LlamaForCausalLM
    cfg = LlamaConfig(hidden_size=128, intermediate_size=128, num_hidden_layers=1, num_attention_heads=1, num_key_value_heads=1,
                      head_dim=128, vocab_size=64)
    with pytest.raises(RuntimeError):
        fast_decode.quantize_weights(LlamaForCausalLM(cfg).half())
