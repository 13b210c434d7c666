"""NativeDecodeSession on a 4-bit cache and with a sliding window: the session's own chain
against the same chain with its attention formed from the definition in 64 bits.

Two chains that differ in the rounding of the attention's output alone: the bars are those
of the session against the HF modules, which differ in every module's (log-probs within 0.05,
logits NRMSE within 0.02, test_native_decode_gpu.py).
"""
import pytest
import torch

from marlin_style_fluxbin_amd import native_decode
from marlin_style_fluxbin_amd.full_model_trial import compare_trace
from marlin_style_fluxbin_amd.native_decode import NativeDecodeSession
from marlin_style_fluxbin_amd.qwen3 import qwen3_config, random_qwen3_model, w3_quantize_qwen3_model
from tests.attention_reference import reference

pytestmark = pytest.mark.gpu


def setup(gpu, quantize, **kw):
    config = qwen3_config(hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4,
                          num_key_value_heads=2, head_dim=64, vocab_size=512, max_position_embeddings=512)
    model = random_qwen3_model(config, device=gpu, dtype=torch.bfloat16, seed=2)
    if quantize:
        w3_quantize_qwen3_model(model, **kw)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 512, (1, 90), generator=g).to(gpu)
    forced = torch.randint(0, 512, (1, 12), generator=g).to(gpu)
    return model, ids, forced


def exact_window(q, k, v, *, lengths, window, sinks, scale, out):
    n = int(lengths[0])
    out.copy_(reference(q, k, v, [(n, 1)], window, sinks, scale)[0])
    return out


def exact_kv4(q, cache, **kw):
    def widen(codes, pairs):
        word = codes.view(torch.int16).to(torch.int32).view(*codes.shape[:3], 16, -1)  # [.., c, g]
        code = torch.stack([(word >> (4 * i)) & 15 for i in range(4)], -1).transpose(-2, -3).flatten(-2)
        pairs = pairs.double()
        return (code.double() * pairs[..., :1] + pairs[..., 1:]).flatten(-2)

    return exact_window(q, widen(cache.k_codes, cache.k_scales), widen(cache.v_codes, cache.v_scales), **kw)


@pytest.mark.parametrize("quantize,order", [(False, None), (True, None), (True, 7)])
@pytest.mark.parametrize("kw", [dict(kv_cache="int4"), dict(kv_cache="int4", window=40, sinks=3),
                                dict(window=40, sinks=3), dict(window=1)])
def test_session_attention(gpu, monkeypatch, quantize, order, kw):
    model, ids, forced = setup(gpu, quantize, **({} if order is None else {"desc_act_seed": order}))
    session = NativeDecodeSession(model, ids, forced, **kw)
    eager = session.audit()
    graph = session.capture()
    assert torch.equal(graph["logits"], eager["logits"])
    for _ in range(2):
        session.audit()  # the program's own work between the replays
        _, again = session.measure("sequence_graph")
        assert torch.equal(again["logits"], eager["logits"])
    other = NativeDecodeSession(model, ids, forced, **kw)
    other.prefix_k, other.prefix_v, other.prefill_logits = session.prefix_k, session.prefix_v, session.prefill_logits
    monkeypatch.setattr(native_decode, "kv4_attention", exact_kv4)
    monkeypatch.setattr(native_decode, "window_attention", exact_window)
    report = compare_trace(graph, other.audit(), logprob_tolerance=0.05)
    assert report["max_abs_logprob_error"] <= 0.05, report
    assert report["logits"]["normalized_rmse"] <= 0.02, report


def test_a_window_over_everything_is_the_session_without_one(gpu):
    model, ids, forced = setup(gpu, True)
    plain = NativeDecodeSession(model, ids, forced)
    wide = NativeDecodeSession(model, ids, forced, window=1000)
    wide.prefix_k, wide.prefix_v, wide.prefill_logits = plain.prefix_k, plain.prefix_v, plain.prefill_logits
    report = compare_trace(wide.audit(), plain.audit(), logprob_tolerance=0.05)
    assert report["max_abs_logprob_error"] <= 0.05 and report["logits"]["normalized_rmse"] <= 0.02, report


def test_session_refusals(gpu):
    model, ids, forced = setup(gpu, False)
    for kw, message in ((dict(kv_cache="fp8"), "kv_cache"), (dict(window=0), "window"), (dict(window=1.5), "window"),
                        (dict(sinks=-1), "sinks")):
        with pytest.raises(ValueError, match=message):
            NativeDecodeSession(model, ids, forced, **kw)


@pytest.mark.parametrize("kw", [dict(kv_cache="int4"), dict(window=40)])
def test_session_refuses_other_head_dims(gpu, kw):
    config = qwen3_config(hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4,
                          num_key_value_heads=2, head_dim=32, vocab_size=512, max_position_embeddings=512)
    model = random_qwen3_model(config, device=gpu, dtype=torch.bfloat16, seed=2)
    ids = torch.zeros(1, 9, dtype=torch.long, device=gpu)
    with pytest.raises(ValueError, match="head_dim"):
        NativeDecodeSession(model, ids, ids[:, :3], **kw)
