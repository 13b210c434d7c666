"""What the 8-bit operators write into a caller's memory counts as a change of it, as torch's own
``out=`` does: a graph that saved the memory before does not use it with other values."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from marlin_style_fluxbin_amd import add_rms_norm_int8, int8_linear, int8_matmul, quantize_int8, rms_norm_int8, silu_mul_int8

BF, I8, F32 = torch.bfloat16, torch.int8, torch.float32


def calls(make):
    """(the call, the tensors that it writes, those that it must leave)"""
    x, r, w = make(4, 64, BF), make(4, 64, BF), make(64, BF)
    codes, scales, total, y = make(4, 64, I8), make(4, F32), make(4, 64, BF), make(4, 32, BF)
    b, sb = make(32, 64, I8), make(32, F32)
    out = dict(out=(codes, scales))
    return [(lambda: quantize_int8(x, **out), (codes, scales), (x,)),
            (lambda: rms_norm_int8(x, w, 1e-6, **out), (codes, scales), (x, w)),
            (lambda: add_rms_norm_int8(x, r, w, 1e-6, **out), (codes, scales), (x, r, w)),
            (lambda: add_rms_norm_int8(x, r, w, 1e-6, residual_out=total), (total,), (x, r, w)),
            (lambda: add_rms_norm_int8(x, r, w, 1e-6, residual_out=r, **out), (r, codes, scales), (x, w)),
            (lambda: silu_mul_int8(x, r, **out), (codes, scales), (x, r)),
            (lambda: int8_matmul(codes, scales, b, sb, out=y), (y,), (codes, scales, b, sb))]


@pytest.mark.parametrize("which", range(7))
def test_outputs_given_count_a_change(monkeypatch, which):
    """On the host: fake tensors of a GPU device, no launch."""
    monkeypatch.setattr(int8_linear, "_launch", lambda *args: None)
    with FakeTensorMode(), torch.no_grad():
        call, written, left = calls(lambda *a: torch.empty(*a[:-1], dtype=a[-1], device="cuda:0"))[which]
        before = [t._version for t in written + left]
        call()
        change = [t._version - v for t, v in zip(written + left, before)]
    assert all(n >= 1 for n in change[:len(written)]) and not any(change[len(written):]), change


@pytest.mark.parametrize("kind", [tuple, list, iter])
def test_outputs_given_by_any_pair_count_a_change(monkeypatch, kind):
    monkeypatch.setattr(int8_linear, "_launch", lambda *args: None)
    with FakeTensorMode(), torch.no_grad():
        make = lambda *a: torch.empty(*a[:-1], dtype=a[-1], device="cuda:0")
        x, w, pair = make(4, 64, BF), make(64, BF), (make(4, 64, I8), make(4, F32))
        for call in (lambda: quantize_int8(x, out=kind(pair)), lambda: rms_norm_int8(x, w, 1e-6, out=kind(pair)),
                     lambda: silu_mul_int8(x, x, out=kind(pair))):
            before = [t._version for t in pair]
            call()
            assert all(t._version > v for t, v in zip(pair, before))


@pytest.mark.gpu
def test_a_graph_does_not_read_what_a_call_overwrote(gpu):
    x, w = torch.randn(4, 64, device=gpu).to(BF), torch.ones(64, dtype=BF, device=gpu)
    b, sb = torch.randint(-127, 128, (32, 64), device=gpu, dtype=I8), torch.rand(32, device=gpu)
    a, sa = quantize_int8(x)
    leaf = torch.ones((), device=gpu, requires_grad=True)
    y, total, scales = int8_matmul(a, sa, b, sb), x.clone(), sa.clone()
    for memory, write in ((y, lambda: int8_matmul(a, sa, b, sb, out=y)),
                          (total, lambda: add_rms_norm_int8(x, x, w, 1e-6, residual_out=total)),
                          (scales, lambda: quantize_int8(x * 2, out=(torch.empty_like(a), scales)))):
        loss = (memory * leaf).sum()  # saves `memory` for the gradient of `leaf`
        with torch.no_grad():
            write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():  # inference tensors have no counter, and need none
        held = torch.empty_like(a), torch.empty_like(sa)
        quantize_int8(x, out=held)
    assert torch.equal(held[0], a) and torch.equal(held[1], sa)
    with torch.no_grad():
        quantize_int8(x * 3, out=held)
    assert torch.equal(held[0], quantize_int8(x * 3)[0])


@pytest.mark.gpu
def test_a_compiled_caller_writes_into_given_memory(gpu):
    x, w = torch.randn(4, 64, device=gpu).to(BF), torch.ones(64, dtype=BF, device=gpu)
    b, sb = torch.randint(-127, 128, (32, 64), device=gpu, dtype=I8), torch.rand(32, device=gpu)

    def step(x, total, y):
        a, sa, _ = add_rms_norm_int8(x * 1, x, w, 1e-6, residual_out=total)
        return int8_matmul(a, sa, b, sb, out=y) * 2

    with torch.no_grad():
        total, y = torch.zeros_like(x), torch.zeros(4, 32, device=gpu, dtype=BF)
        want = step(x, total, y)
        other, z = torch.zeros_like(x), torch.zeros_like(y)
        got = torch.compile(step, backend="eager")(x, other, z)
    assert torch.equal(got, want) and torch.equal(other, total) and torch.equal(z, y)


@pytest.mark.gpu
def test_captured_calls_write_into_given_memory(gpu):
    x, w = torch.randn(4, 64, device=gpu).to(BF), torch.ones(64, dtype=BF, device=gpu)
    total, held = torch.empty_like(x), (torch.empty(4, 64, dtype=I8, device=gpu), torch.empty(4, device=gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        add_rms_norm_int8(x, x, w, 1e-6, residual_out=total, out=held)
        with torch.cuda.graph(graph):
            add_rms_norm_int8(x, x, w, 1e-6, residual_out=total, out=held)
        for _ in range(3):
            x.copy_(torch.randn(4, 64, device=gpu))
            graph.replay()
            want = add_rms_norm_int8(x, x, w, 1e-6)
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip((*held, total), want))
