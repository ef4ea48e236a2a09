"""What four-bit weights multiply: rows as two e4m3 numbers under their block's power of two.  Rows with numbers far above their
block's others, rows at both ends of bfloat16's range, and rows with an infinity or a NaN, in every form."""
import math

import pytest
import torch

import mxfp4_whole as whole
from mxfp4_whole import step

pytestmark = pytest.mark.gpu


# (rows, outputs, inputs): split by the product itself, ahead of a narrow one (few rows of a long stretch, and more), wide, in pairs
FORMS = [(5, 200, 1024), (8, 16384, 9216), (20, 200, 1024), (40, 200, 1024), (100, 28790, 512), (300, 200, 1024)]


def products(a, codes, scales, ctx):
    """a with the weight, by the dense form and by the grouped ones (every tile of group 1 of 2, of which group 0 is none of it)."""
    from flambeau_b200.kernels import ops
    M, K = a.shape
    N = codes.shape[0]
    out = torch.empty(M, N, device="cuda")
    ops.linear(a, ops.Mxfp4Weight(codes, scales, K), out, ctx)
    yield "dense", out
    if M > 100 or N > 1000:
        return
    stack = ops.Mxfp4Weight(torch.stack([codes.flip(0), codes]), torch.stack([scales.flip(0), scales]), K)
    for tile in (16, 64, 128):
        n = -(-M // tile)
        index = torch.full((n * tile,), -1, dtype=torch.int32, device="cuda")
        index[:M] = torch.arange(M, dtype=torch.int32, device="cuda")
        out = torch.empty(n * tile, N, device="cuda")
        ops.grouped_linear(a, index, stack, torch.ones(n, dtype=torch.int32, device="cuda"), tile, out, None, ctx)
        yield f"tiles of {tile}", out[:M]


@pytest.mark.parametrize("power", [8, 13, 16, 20])
@pytest.mark.parametrize("M,N,K", FORMS)
def test_a_number_far_above_its_blocks_others(M, N, K, power):
    """One number 2^power in every block, over weights of code 0: the others lose up to 2^-22 of it, no more, and the product is that
    of what is left."""
    a = whole.rows(M, K, 1) / 256                # multiples of 2^-8 below 1
    codes, scales = whole.weight_codes((N,), K, 2)
    codes.view(N, -1, 16)[:, :, 5] &= 0x0f       # column 11 of every block, of either sign
    codes.view(N, -1, 16)[:, ::2, 5] |= 0x80
    a[:, 11::32] = 2.0 ** power
    a[::2, 11::32] *= -1
    w = whole.numbers(codes, scales)
    held = sum(whole.split(a))
    lost = (held - a.double()).abs()
    assert bool((lost <= 2.0 ** (power - 22)).all()) and bool((lost > 0).any()) == (power > 13)
    want = whole.product(held * 256, w) / 256    # (whole numbers again: sums of them are exact)
    ctx = step()
    for name, out in products(a, codes, scales, ctx):
        assert torch.equal(out.double(), want), name
        assert bool(((out.double() - a.double() @ w.T).abs() <= 2.0 ** (power - 22) * w.abs().sum(1)).all()), name
    ctx.runtime.check_status()


@pytest.mark.parametrize("power", [-133, -126, -120, 118])
@pytest.mark.parametrize("M,N,K", FORMS)
def test_rows_at_the_ends_of_bfloat16s_range(M, N, K, power):
    """Multiples of 2^power (the lowest are subnormal): blocks below 2^-115 share one scale, under which 2^-136 is the last place."""
    a = (whole.rows(M, K, 3).float() * 2.0 ** max(power, -126) * 2.0 ** min(0, power + 126)).bfloat16()
    codes, scales = whole.weight_codes((N,), K, 4)
    scales = scales - 40 if power > 0 else scales + 60                   # (sums of ordinary size)
    w = whole.numbers(codes, scales)
    assert torch.equal(sum(whole.split(a)), a.double()) and int((a != 0).sum()) > a.numel() // 2
    want = a.double() @ w.T
    ctx = step()
    for name, out in products(a, codes, scales, ctx):
        assert torch.equal(out.double(), want), name
    ctx.runtime.check_status()


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("M,N,K", FORMS)
def test_a_row_with_an_infinity_or_a_nan(M, N, K, what):
    """Its sums are NaN, of weights of code 0 too; every other row is as if it were not there."""
    a = whole.rows(M, K, 5)
    codes, scales = whole.weight_codes((N,), K, 6)
    want = whole.product(a, whole.numbers(codes, scales))
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    for r, c in ((0, 0), (M // 2, K - 1), (M - 1, K // 2 + 37)):
        a[r, c] = what
        bad[r] = True
    ctx = step()
    for name, out in products(a, codes, scales, ctx):
        assert bool(out[bad].isnan().all()) and torch.equal(out[~bad].double(), want[~bad]), name
    ctx.runtime.check_status()


@pytest.mark.parametrize("tile", [16, 32, 64, 128])
def test_a_tile_whose_group_is_none_of_the_weights(tile):
    """Its rows of the output become NaN, and those of the other tiles are what they are without it."""
    from flambeau_b200.kernels import ops
    N, K = 130, 320
    codes, scales = whole.weight_codes((3, N), K, 7)
    w, dense = ops.Mxfp4Weight(codes, scales, K), whole.numbers(codes, scales)
    order = [0, 3, 1, 1, 2 ** 31 - 1, -1, 2, 2, 70]
    M = tile * len(order)
    a = whole.rows(M, K, 8)
    tiles = torch.tensor(order, dtype=torch.int32, device="cuda")
    of = tiles.repeat_interleave(tile)
    ctx = step()
    for index in (None, torch.arange(M, dtype=torch.int32, device="cuda")):
        for dtype in (torch.float32, torch.bfloat16):
            out, act = torch.full((M, N), 7.0, dtype=dtype, device="cuda"), torch.full((M, N // 2), 7.0, dtype=dtype, device="cuda")
            ops.grouped_linear(a, index, w, tiles, tile, out, None, ctx)
            ops.grouped_gated_linear(a, index, w, tiles, tile, act, "silu", ctx)
            for g in range(3):
                assert torch.equal(out[of == g], whole.product(a[of == g], dense[g]).to(dtype)) and bool(act[of == g].isfinite().all())
            assert bool(out[of > 2].isnan().all()) and bool(act[of > 2].isnan().all())
            assert bool((out[of < 0] == 7.0).all()) and bool((act[of < 0] == 7.0).all())
    ctx.runtime.check_status()
