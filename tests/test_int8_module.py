"""PackedInt8Linear's payload: memory of its own.  CPU-only."""
import pytest
import torch

from marlin_style_fluxbin_amd import PackedInt8Linear


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
