"""NativeDecodeSession on 8-bit Linears: the session's own chain against the same chain with the
8-bit operators formed from their definitions in 64 bits.

Two chains whose stored tensors round alike and that differ in fp32 against 64-bit arithmetic
between them (a code or a 16-bit value that flips now and then): the bars are those of the session
against the HF modules, which differ in every module's (log-probs within 0.05, logits NRMSE
within 0.02, test_native_decode_gpu.py).
"""
import pytest
import torch

from marlin_style_fluxbin_amd import PackedInt8Linear, native_decode
from marlin_style_fluxbin_amd.full_model_trial import compare_trace
from marlin_style_fluxbin_amd.native_decode import NativeDecodeSession
from marlin_style_fluxbin_amd.qwen3 import int8_quantize_qwen3_model, qwen3_config, random_qwen3_model
from marlin_style_fluxbin_amd.static_decode import StaticDecodeSession, prepared_linears
from tests.int8_reference import held, norm_rows, product, swiglu_rows

pytestmark = pytest.mark.gpu


def setup(gpu, dtype=torch.bfloat16, **config):
    sizes = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4,
                 num_key_value_heads=2, head_dim=64, vocab_size=512, max_position_embeddings=512) | config
    model = random_qwen3_model(qwen3_config(**sizes), device=gpu, dtype=dtype, seed=2)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 512, (1, 90), generator=g).to(gpu)
    forced = torch.randint(0, 512, (1, 12), generator=g).to(gpu)
    return model, ids, forced


def write(out, codes, scales):
    out[0].copy_(codes)
    out[1].copy_(scales)


def exact_norm(x, weight, eps, *, out):
    p, inverse, _ = norm_rows(x, weight, eps)
    write(out, held(p)[0], held(p * inverse)[1])


def exact_add_norm(x, residual, weight, eps, *, residual_out, out):
    p, inverse, s = norm_rows(x, weight, eps, residual)
    write(out, held(p)[0], held(p * inverse)[1])
    residual_out.copy_(s)


def exact_silu(gate, up, *, out):
    write(out, *held(swiglu_rows(gate, up)))


def exact_matmul(a, a_scales, w, w_scales, *, bias, dtype, out):
    out.copy_(product(a, a_scales, w, w_scales, bias)[0])


def exact_kernel(module, rows, device):
    def run(x, out):
        a, sa = held(x)
        out.copy_(product(a, sa, module.codes[:, :module.in_features], module.scales, module.bias)[0])
    return run


def patch(monkeypatch):
    for name, exact in (("rms_norm_int8", exact_norm), ("add_rms_norm_int8", exact_add_norm),
                        ("silu_mul_int8", exact_silu), ("int8_matmul", exact_matmul)):
        monkeypatch.setattr(native_decode, name, exact)
    monkeypatch.setattr(PackedInt8Linear, "_packed_kernel", exact_kernel)


def compare(monkeypatch, model, ids, forced, chain, **kw):
    session = NativeDecodeSession(model, ids, forced, **kw)
    assert (session.int8 is not None) is chain
    eager = session.audit()
    graph = session.capture()
    assert torch.equal(graph["logits"], eager["logits"])
    for _ in range(2):
        session.audit()  # the program's own work between the replays
        _, again = session.measure("sequence_graph")
        assert torch.equal(again["logits"], eager["logits"])
    with monkeypatch.context() as m:
        patch(m)
        other = NativeDecodeSession(model, ids, forced, **kw)
        # (its own prefill ran on the exact Linears; the decode steps are compared on one prefix)
        if session.int4_cache is None:
            other.prefix_k, other.prefix_v = session.prefix_k, session.prefix_v
        else:
            other.int4_cache = session.int4_cache
        other.prefill_logits = session.prefill_logits
        want = other.audit()
    report = compare_trace(graph, want, logprob_tolerance=0.05)
    assert report["max_abs_logprob_error"] <= 0.05, report
    assert report["logits"]["normalized_rmse"] <= 0.02, report


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [{}, dict(window=40, sinks=3), dict(kv_cache="int4")])
def test_session_of_int8_linears(gpu, monkeypatch, dtype, kw):
    model, ids, forced = setup(gpu, dtype)
    assert int8_quantize_qwen3_model(model) == 21
    compare(monkeypatch, model, ids, forced, True, **kw)


def test_session_with_biases(gpu, monkeypatch):
    model, ids, forced = setup(gpu)
    for block in model.model.layers:
        for name in ("self_attn.q_proj", "self_attn.v_proj", "mlp.down_proj"):
            linear = block.get_submodule(name)
            linear.bias = torch.nn.Parameter(0.1 * torch.randn(linear.out_features, device=gpu).bfloat16())
    int8_quantize_qwen3_model(model)
    compare(monkeypatch, model, ids, forced, True)


@pytest.mark.parametrize("which", ["odd width", "some Linears"])
def test_session_of_other_int8_linears(gpu, monkeypatch, which):
    """Widths that are no whole 16, and models of which some Linears are 8-bit: each quantizes its input."""
    model, ids, forced = setup(gpu, intermediate_size=520 if which == "odd width" else 512)
    if which == "odd width":
        int8_quantize_qwen3_model(model)
    else:
        for block in model.model.layers:
            for name in ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "mlp.down_proj"):
                parent, attribute = name.rsplit(".", 1)
                setattr(block.get_submodule(parent), attribute, PackedInt8Linear.from_linear(block.get_submodule(name)))
    compare(monkeypatch, model, ids, forced, False)


def test_prefill_is_the_quantized_models(gpu):
    """The model's own forward on 8-bit Linears, against one whose Linears hold the values that the
    codes stand for: they differ by the rows' quantization."""
    model, ids, _ = setup(gpu)
    other, _, _ = setup(gpu)
    int8_quantize_qwen3_model(model)
    with torch.no_grad():
        for block, plain in zip(model.model.layers, other.model.layers):
            for name in native_decode._ATTN + native_decode._MLP:
                plain.get_submodule(name).weight.copy_(block.get_submodule(name)._dense_weight(torch.bfloat16))
        got, want = model(ids).logits.float(), other(ids).logits.float()
    assert all(m.route_counts["packed_small_m"] == 1 for m in model.modules() if isinstance(m, PackedInt8Linear))
    # a row of normal values has its largest near 3 to 4 and a step of 1/36 and less: 0.8% of the
    # row's norm (step / sqrt(12)) for each of the 12 inputs in turn, 5% with all against each other
    assert float((got - want).norm() / want.norm()) <= 0.05


def test_module_tree_session_with_bound_linears(gpu):
    """The HF module tree's own session, its Linears bound: the same as unbound, and in a graph."""
    model, ids, forced = setup(gpu)
    int8_quantize_qwen3_model(model)
    session = StaticDecodeSession(model, ids, forced)
    want = session.audit()
    with prepared_linears(model, torch.bfloat16) as modules:
        assert len(modules) == 21
        got = session.audit()
        assert torch.equal(got["logits"], want["logits"])
        assert torch.equal(session.capture()["logits"], want["logits"])
    assert all(m._decode_binding is None for m in modules.values())
