"""The oracle of the four-bit products of whole numbers, on the CPU: it holds the rows exactly, and what a wrong kernel would give
is not equal to it in any row."""
import pytest
import torch

import mxfp4_whole as whole

M, N, K = 6, 40, 2048


@pytest.fixture(scope="module")
def drawn():
    a, (codes, scales) = whole.rows(M, K, 1, device="cpu"), whole.weight_codes((N,), K, 2, device="cpu")
    return a, codes, scales, whole.product(a, whole.numbers(codes, scales))


def test_two_parts_hold_whole_numbers(drawn):
    a = drawn[0]
    first, second = whole.split(a)
    assert torch.equal(first + second, a.double()) and bool((second != 0).any(1).all())


def test_rows_lose_at_most_the_stated_part_of_their_blocks_largest():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(64, 256, generator=g) * torch.exp2(torch.linspace(-133, 120, 64)).unsqueeze(1)
    x[:, ::32] *= torch.exp2(torch.arange(8.0) * 3)                    # a number far above its block's others
    x = x.clamp(-3e38, 3e38).bfloat16()
    first, second = whole.split(x)
    top = x.double().abs().view(64, -1, 32).amax(-1).repeat_interleave(32, 1)
    assert bool(((first + second - x.double()).abs() <= 2.0 ** -22 * top.clamp(min=2.0 ** -115)).all())


def mistakes(a, codes, scales):
    w = whole.numbers(codes, scales)
    first, _ = whole.split(a)
    yield "no second parts", first @ w.T
    for tile in (0, 7, 15):
        at = slice(128 * tile, 128 * tile + 128)
        part = a[:, at].double() @ w[:, at].T
        yield f"tile {tile} lost", a.double() @ w.T - part
        yield f"tile {tile} twice", a.double() @ w.T + part
    yield "scales of the blocks before", a.double() @ whole.numbers(codes, scales.roll(1, 1)).T
    yield "scales of the features before", a.double() @ whole.numbers(codes, scales.roll(1, 0)).T
    shifted = a.clone().double()
    shifted[:, 64:96] *= 2
    yield "a block of rows under another scale", shifted @ w.T
    halves = (codes << 4) | (codes >> 4)
    halves[:, 16:] = codes[:, 16:]
    yield "the halves of a block's bytes", a.double() @ whole.numbers(halves, scales).T


def test_what_a_wrong_kernel_gives_is_not_equal(drawn):
    a, codes, scales, want = drawn
    for name, got in mistakes(a, codes, scales):
        assert bool((got != want).any(1).all()) and bool((got != want).any(0).all()), name
