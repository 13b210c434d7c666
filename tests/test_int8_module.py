"""PackedInt8Linear's payload: memory of its own, laid out as the kernels read it whatever brings it.
CPU-only but for the last test."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from marlin_style_fluxbin_amd import PackedInt8Linear, int8_linear


def payload(columns, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (7, columns), generator=g, dtype=torch.int8), torch.rand(7, generator=g) + 0.5


@pytest.mark.parametrize("columns", [48, 40])
@torch.no_grad()
def test_a_module_shares_no_memory_with_what_it_was_made_of(columns):
    codes, scales = payload(columns)
    bias = torch.rand(7)
    before = codes.clone(), scales.clone(), bias.clone()
    one, two = (PackedInt8Linear(codes, scales, bias=bias, fallback="dense") for _ in range(2))
    x = torch.randn(3, columns, generator=torch.Generator().manual_seed(1))
    want = two(x)
    # another checkpoint into one of them
    one.load_state_dict(PackedInt8Linear(*payload(columns, 5), bias=torch.zeros(7)).state_dict())
    assert all(torch.equal(t, b) for t, b in zip((codes, scales, bias), before))
    assert torch.equal(two(x), want) and not torch.equal(one(x), want)
    # and the caller's memory used for something else
    for t in (codes, scales, bias):
        t.zero_()
    assert torch.equal(two(x), want)


@torch.no_grad()
def test_scales_with_a_lazy_negation_are_held_as_values():
    codes, scales = payload(48)
    module = PackedInt8Linear(codes, torch._neg_view(scales))
    assert not module.scales.is_neg() and torch.equal(module.scales, -scales)


@torch.no_grad()
def test_any_layout_becomes_whole_rows():
    codes, scales = payload(48)
    for given in (codes.t().contiguous().t(), torch.cat([codes, codes], 1)[:, :48], torch.cat([codes, codes], 1)[:, 3:51]):
        module = PackedInt8Linear(given, scales.repeat_interleave(2)[::2])
        assert module.codes.is_contiguous() and module.scales.is_contiguous() and module.codes.data_ptr() % 16 == 0
        assert torch.equal(module.codes, given) and torch.equal(module.scales, scales)
    one = PackedInt8Linear(codes[:1].expand(7, 48), scales[:1].expand(7))
    assert torch.equal(one.codes, codes[:1].repeat(7, 1)) and one.codes.is_contiguous() and one.scales.is_contiguous()


# ------------------------------------------------------------------ tensors that a state dict assigns
class Launched(Exception):
    pass


@pytest.fixture
def fake(monkeypatch):
    """Fake tensors of a GPU device; a call that would reach the library ends."""
    def launch(name, index, *args):
        raise Launched(name)

    monkeypatch.setattr(int8_linear, "_launch", launch)
    with FakeTensorMode(), torch.no_grad():
        yield lambda *shape, dtype=torch.bfloat16, device="cuda:0": torch.empty(*shape, dtype=dtype, device=device)


def fake_module(fake, bias=True):
    return PackedInt8Linear(fake(8, 32, dtype=torch.int8), fake(8, dtype=torch.float32), bias=fake(8) if bias else None)


@torch.no_grad()
def test_assigned_tensors_are_held_as_the_kernels_read_them():
    """Strided, lazily negated and unaligned ones as copies, others as they are."""
    codes, scales = payload(48)
    bias = torch.rand(7)
    module = PackedInt8Linear(codes, scales, bias=bias)
    odd = torch.empty(7 * 48 + 3, dtype=torch.int8)[3:].view(7, 48).copy_(codes)
    for given in (dict(codes=codes.t().contiguous().t(), scales=scales.repeat_interleave(2)[::2],
                       bias=bias.repeat_interleave(2)[::2]),
                  dict(codes=odd, scales=torch._neg_view(-scales), bias=torch._neg_view(-bias))):
        module.load_state_dict(given, assign=True)
        for name, want in (("codes", codes), ("scales", scales), ("bias", bias)):
            held = getattr(module, name)
            assert held.is_contiguous() and not held.is_neg() and held.data_ptr() % 16 == 0 and torch.equal(held, want)
    module.load_state_dict(dict(codes=codes, scales=scales, bias=bias), assign=True)
    assert module.codes.data_ptr() == codes.data_ptr()


@pytest.mark.parametrize("which", ["codes", "scales", "bias"])
def test_tensors_of_two_devices_are_refused(fake, which):
    module = fake_module(fake)
    with pytest.raises(Launched):
        module(fake(3, 32))
    shape, dtype = dict(codes=((8, 32), torch.int8), scales=((8,), torch.float32), bias=((8,), torch.bfloat16))[which]
    module.load_state_dict({which: fake(*shape, dtype=dtype, device="cpu")}, assign=True, strict=False)
    for x in (fake(3, 32), fake(1, 1, 32)):
        with pytest.raises(ValueError, match="device|fallback"):
            module(x)
    with pytest.raises(ValueError, match="device|CUDA"):
        module.bind_prepared_decode(torch.bfloat16)


def test_an_assigned_payload_ends_a_binding_of_the_old_one(fake):
    module = fake_module(fake)
    module.bind_prepared_decode(torch.bfloat16)
    module.load_state_dict(fake_module(fake).state_dict())  # written into the buffers that are bound
    assert module._decode_binding is not None
    module.load_state_dict(fake_module(fake).state_dict(), assign=True)
    assert module._decode_binding is None and module._decode_output is None
    for given in (dict(codes=fake(32, 8, dtype=torch.int8).t()), dict(scales=fake(16, dtype=torch.float32)[::2]),
                  dict(bias=fake(16)[::2])):  # each held as a copy
        module.bind_prepared_decode(torch.bfloat16)
        module.load_state_dict(given, assign=True, strict=False)
        assert module._decode_binding is None


# ------------------------------------------------------------------ bound calls
def test_a_bound_call_reads_values_and_refuses_records(fake, monkeypatch):
    from torch.autograd import forward_ad

    module = fake_module(fake)
    module.bind_prepared_decode(torch.bfloat16)
    x = fake(1, 1, 32)
    addresses = []
    monkeypatch.setattr(module, "_decode_binding", lambda t: addresses.append(t.is_neg()))
    module(x)
    module(torch._neg_view(x))
    assert addresses == [False, False]
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            module(forward_ad.make_dual(x, torch.ones_like(x)))
        module(x)
    assert len(addresses) == 3


@pytest.mark.gpu
def test_bound_calls_on_the_gpu(gpu):
    from torch.fx.experimental.proxy_tensor import make_fx

    codes, scales = payload(48)
    module = PackedInt8Linear(codes.to(gpu), scales.to(gpu))
    x = torch.randn(1, 1, 48, generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu)
    with torch.no_grad():
        want, minus = module(x), module(-x)
        module.bind_prepared_decode(torch.bfloat16)
        assert torch.equal(module(x), want) and torch.equal(module(torch._neg_view(x)), minus)
        for record in (lambda: torch.jit.trace(module, (x,), check_trace=False), lambda: make_fx(module)(x)):
            with pytest.raises(ValueError, match="traced"):
                record()
        module.load_state_dict({name: t.clone() for name, t in PackedInt8Linear(codes.to(gpu), 2 * scales.to(gpu))
                                .state_dict().items()}, assign=True)
        assert torch.equal(module(x), 2 * want)  # a power of two: exact
