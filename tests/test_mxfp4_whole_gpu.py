"""Products of whole numbers with four-bit weights are equal to the formula's, in every form: a tile along K, a share, a scale or a
second part that is lost, repeated or taken from elsewhere shows however long the sums are."""
import pytest
import torch

import mxfp4_whole as whole
from mxfp4_whole import step

pytestmark = pytest.mark.gpu


def weight(shape, K, seed):
    """(the weight for K inputs, its float64 numbers); columns behind K are codes that nobody may read."""
    from flambeau_b200.kernels import ops
    wide = -(-K // 32) * 32
    codes, scales = whole.weight_codes(shape, wide, seed)
    return ops.Mxfp4Weight(codes, scales, K), whole.numbers(codes, scales)[..., :K]


def finished(ctx):
    ctx.runtime.check_status()
    assert int(ctx.ws.counters.abs().sum()) == 0


def linear_is_equal(a, w, want, ctx):
    from flambeau_b200.kernels import ops
    M, N = want.shape
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((M, N + 3), 7.0, dtype=dtype, device="cuda")
        for view in (out[:, :N], torch.full((M, N), 7.0, dtype=dtype, device="cuda")):
            ops.linear(a, w, view, ctx)
            assert torch.equal(view, want.to(dtype))                     # (one rounding, of a float32 number)
        assert bool((out[:, N:] == 7.0).all())


def every_entry_is_equal(a, w, want, ctx):
    from flambeau_b200.kernels import ops
    M, N = want.shape
    linear_is_equal(a, w, want, ctx)
    act = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    ops.activated_linear(a, w, act, "relu_squared", ctx)
    assert torch.equal(act, want.float().clamp(min=0).square().bfloat16())
    for most in (1, 2, 3, 8):
        slabs = torch.full((most + 1, M, N), 7.0, device="cuda")
        k = ops.linear_slabs(a, w, slabs[:most], ctx)
        assert 1 <= k <= most and torch.equal(slabs[:k].sum(0).double(), want) and bool((slabs[k:] == 7.0).all())
    stream = torch.randint(-1000, 1000, (M, N), device="cuda").float()
    before = stream.double()
    if ops.linear_add(a, w, stream, ctx):
        assert M > 128 and torch.equal(stream.double(), before + want)
    if N % 2 == 0:
        for dtype, rounding in ((torch.float32, 2.0 ** -20), (torch.bfloat16, 2.0 ** -8 + 2.0 ** -20)):
            out = torch.empty(M, N // 2, dtype=dtype, device="cuda")
            ops.gated_linear(a, w, out, "silu", ctx)
            assert gated_is_near(out, want, rounding)


def gated_is_near(out, want, rounding):
    """silu(g) u of exact g and u: roundings where g > 0; below, the exponential of a large number, and nothing below -87."""
    g, u = want[:, 0::2], want[:, 1::2]
    ref = g * torch.sigmoid(g) * u
    low = 2.0 ** -21 * g.clamp(max=0).abs() * ref.abs() + 2.0 ** -126 * (g * u).abs()
    return bool(((out.double() - ref).abs() <= rounding * ref.abs() + low).all())


@pytest.mark.parametrize("M", [1, 3, 8, 9, 20, 32, 33, 48, 64, 65, 100, 128, 130, 301])
@pytest.mark.parametrize("N,K", [(2, 8), (130, 1000), (384, 14336), (1024, 4096), (4096, 2048)])
def test_product(M, N, K):
    w, dense = weight((N,), K, 1)
    a = whole.rows(M, K, 2 + M)
    ctx = step()
    every_entry_is_equal(a, w, whole.product(a, dense), ctx)
    finished(ctx)


@pytest.mark.parametrize("M,N,K", [(48, 384, 14336), (100, 256, 8192), (130, 200, 16384), (17, 128, 28672), (3, 64, 28672), (96, 130, 28672)])
def test_shares_meet(M, N, K):
    w, dense = weight((N,), K, 3)
    a = whole.rows(M, K, 4, top=31)
    ctx = step()
    every_entry_is_equal(a, w, whole.product(a, dense), ctx)
    finished(ctx)


@pytest.mark.parametrize("M,N,K", [(8, 16384, 9216), (1, 16384, 9216), (40, 28790, 4160), (64, 28790, 4096), (100, 28790, 4096), (128, 28790, 4096),
                                   (256, 28790, 4096), (301, 28672, 4096), (2048, 1543, 1001)])
def test_sizes_that_only_some_forms_see(M, N, K):
    """Long stretches of few rows, an odd number of feature tiles in pairs, many tiles of tokens."""
    w, dense = weight((N,), K, 5)
    a = whole.rows(M, K, 6)
    ctx = step()
    every_entry_is_equal(a, w, whole.product(a, dense), ctx)
    finished(ctx)


@pytest.mark.parametrize("M", [3, 30, 70])
def test_a_matrix_whose_offsets_pass_32_bits(M):
    N = K = 1 << 16
    from flambeau_b200.kernels import ops
    codes, scales = whole.weight_codes((N,), K, 7)
    w = ops.Mxfp4Weight(codes, scales, K)
    a = whole.rows(M, K, 8, top=31)
    ctx = step()
    out = torch.empty(M, N, device="cuda")
    ops.linear(a, w, out, ctx)
    for part in (slice(0, 300), slice(N // 2 - 150, N // 2 + 150), slice(N - 300, N)):
        assert torch.equal(out[:, part].double(), whole.product(a, whole.numbers(codes[part], scales[part])))
    finished(ctx)


TILES = {"runs": [0] * 6 + [1] * 8 + [2] * 9 + [3] + [4] * 17 + [-1] * 3, "mixed": [2, 2, -1, 0, 2, 1, 1, -1, -1, 4, 3, 3, 3],
         "many": [i % 5 for i in range(450)] + [3] * 12 + [-1, 0]}


@pytest.mark.parametrize("groups", [5, 300])                             # (of 300 groups most are empty: units of 64 rows)
@pytest.mark.parametrize("tile", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("pattern", list(TILES))
def test_groups(pattern, tile, groups):
    from flambeau_b200.kernels import ops
    N, K = 258, 1000
    order = [g * (groups // 5) for g in TILES[pattern]]                  # (-1 stays negative)
    M = tile * len(order)
    w, dense = weight((groups, N), K, 9)
    tiles = torch.tensor(order, dtype=torch.int32, device="cuda")
    of = tiles.repeat_interleave(tile)
    kept = of >= 0
    x = whole.rows(90, K, 10)
    index = torch.randint(-1, 90, (M,), generator=torch.Generator().manual_seed(11)).int().cuda()
    pair = torch.randperm(M, generator=torch.Generator().manual_seed(12)).int().cuda()
    share = 2.0 ** torch.randint(-1, 2, (M,), generator=torch.Generator().manual_seed(13)).float().cuda()
    ctx = step()
    for shares in (False, True):
        a = torch.where((index >= 0).unsqueeze(1), x[index.clamp(min=0).long()], 0)
        if shares:                               # (powers of two: the scaled rows are exact)
            a = a * share[pair.long()].unsqueeze(1).bfloat16()
        want = torch.zeros(M, N, dtype=torch.float64, device="cuda")
        for g in set(order):
            if g >= 0:
                want[of == g] = whole.product(a[of == g], dense[g])
        more = dict(row_share=share, row_pair=pair) if shares else {}
        for dtype in (torch.float32, torch.bfloat16):
            out = torch.full((M, N), 7.0, dtype=dtype, device="cuda")
            ops.grouped_linear(x, index, w, tiles, tile, out, None, ctx, **more)
            assert torch.equal(out[kept], want[kept].to(dtype)) and bool((out[~kept] == 7.0).all())
            if not shares:
                out.fill_(7.0)
                ops.grouped_linear(a, None, w, tiles, tile, out, None, ctx)
                assert torch.equal(out[kept], want[kept].to(dtype)) and bool((out[~kept] == 7.0).all())
            act = torch.full((M, N // 2), 7.0, dtype=dtype, device="cuda")
            ops.grouped_gated_linear(x, index, w, tiles, tile, act, "silu", ctx, **more)
            assert gated_is_near(act[kept], want[kept], 2.0 ** -20 + (0 if dtype == torch.float32 else 2.0 ** -8))
            assert bool((act[~kept] == 7.0).all())
        act = torch.full((M, N), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.grouped_linear(x, index, w, tiles, tile, act, "relu_squared", ctx, **more)
        assert torch.equal(act[kept], want[kept].float().clamp(min=0).square().bfloat16()) and bool((act[~kept] == 7.0).all())
    ctx.runtime.check_status()


@pytest.mark.parametrize("tile", [16, 32, 64, 128])
def test_more_units_than_are_listed(tile):
    """Thousands of runs of one to five tiles, skipped tiles among them: units behind the first 512 are counted on."""
    from flambeau_b200.kernels import ops
    N, K, groups = 200, 96, 7
    g = torch.Generator().manual_seed(tile)
    order = torch.repeat_interleave(torch.randint(-1, groups, (1500,), generator=g), torch.randint(1, 6, (1500,), generator=g))
    tiles = order.int().cuda()
    M = tile * len(order)
    w, dense = weight((groups, N), K, 14)
    x = whole.rows(M, K, 15)
    of = tiles.repeat_interleave(tile)
    want = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    for e in range(groups):
        want[of == e] = whole.product(x[of == e], dense[e])
    ctx = step()
    out = torch.full((M, N), 7.0, device="cuda")
    ops.grouped_linear(x, None, w, tiles, tile, out, None, ctx)
    assert torch.equal(out[of >= 0].double(), want[of >= 0]) and bool((out[of < 0] == 7.0).all())
    ctx.runtime.check_status()


@pytest.mark.parametrize("M,N,K", [(70001, 130, 96), (300000, 8, 32)])
def test_many_rows(M, N, K):
    from flambeau_b200.kernels import ops
    w, dense = weight((N,), K, 16)
    a = whole.rows(M, K, 17)
    ctx = step()
    linear_is_equal(a, w, whole.product(a, dense), ctx)
    finished(ctx)


def test_slabs_of_any_number_and_stride():
    """As many slabs as are given, apart by more than their rows, in rows apart; what lies between is not touched."""
    from flambeau_b200.kernels import ops
    N, K = 130, 14336
    w, dense = weight((N,), K, 18)
    ctx = step()
    for M in (1, 8, 20, 40, 130):
        a = whole.rows(M, K, 19)
        want = whole.product(a, dense)
        for most in (2, 5, 40):
            for pad in (2, 6):
                room = torch.full((most, M + 1, N + pad), 7.0, device="cuda")
                slabs = room[:, :M, :N]
                k = ops.linear_slabs(a, w, slabs, ctx)
                assert 1 <= k <= most and torch.equal(slabs[:k].sum(0).double(), want)
                assert bool((room[:, M:] == 7.0).all()) and bool((room[:, :, N:] == 7.0).all()) and bool((room[k:] == 7.0).all())
    finished(ctx)
