"""Four-bit weights: rows into blocks and back against the definition, the products against float64 with the same numbers, at the
sizes where tiles, blocks and copies end, and what is refused."""
import math
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def step(dtype="bfloat16"):
    from flambeau_b200.engine.runtime import Runtime
    rt = Runtime("cuda:0", dtype)
    return SimpleNamespace(runtime=rt, ws=rt.ws)


def values(codes, scales, columns):
    """float64 numbers of codes and scales, from the definition."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = torch.tensor(GRID + [-x for x in GRID], dtype=torch.float64, device=codes.device)[c]
    s = torch.exp2(scales.double() - 127.0)
    s[scales == 255] = math.nan
    return (v * s.repeat_interleave(32, -1))[..., :columns]


def nearest(x):
    """(numbers, scale exponents) of x [rows, 32 n] by trying every scale and every point of the grid, one block at a time."""
    x = x.double()
    blocks = x.view(-1, 32)
    exps = torch.arange(-127, 128, dtype=torch.float64, device=x.device)
    top = blocks.abs().amax(1, keepdim=True)
    fits = (top < 7.0 * torch.exp2(exps)) | (exps == 125.0)              # (scales end there)
    fits &= exps <= 125.0                                  # (a row a block, a column a scale)
    e = exps[fits.double().argmax(1)].unsqueeze(1)
    y = blocks.abs() / torch.exp2(e)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    d = (y.unsqueeze(-1) - grid).abs()
    tie = torch.arange(8, device=x.device) % 2                           # among equals the even code
    best = d.amin(-1, keepdim=True)
    code = torch.where(d == best, tie, 9).argmin(-1)
    out = grid[code] * torch.where(torch.signbit(blocks), -1.0, 1.0) * torch.exp2(e)
    none = ~blocks.isfinite().all(1, keepdim=True)                       # a block with an infinity or a NaN is no number
    return torch.where(none, math.nan, out).view(x.shape), torch.where(none, 128.0, e)


def same(a, b):
    return a.shape == b.shape and bool(((a.double() == b.double()) | (a.isnan() & b.isnan())).all())


def test_rows_into_blocks_and_back_over_the_range():
    from flambeau_b200.kernels import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(64, 256, generator=g, device="cuda")
    x *= torch.exp2(torch.linspace(-130, 110, 64, device="cuda")).unsqueeze(1)
    x[3] = 0.0
    x[5, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4, device="cuda")        # ties under scale 1
    x[6, :32] = 7.0
    x[6, 32:64] = torch.nextafter(torch.tensor(7.0), torch.tensor(0.0)).cuda()
    x[7, :32] = -x[5, :32]
    x[8, 0], x[8, 1:32] = 3.4028234e38, 1e-45
    x[9, :32], x[9, 32:64] = 1e-45, 2.0 ** -126
    for t in (x, x.bfloat16()):
        codes, scales = ops.quantize_mxfp4(t)
        want, e = nearest(t)
        got = values(codes, scales, 256)
        assert same(got, want)
        assert torch.equal(scales.view(-1).double() - 127.0, torch.where(t.reshape(-1, 32).abs().amax(1) > 0, e.view(-1), -127.0))
        assert same(ops.dequantize_mxfp4(codes, scales, 256), want)
        assert same(ops.dequantize_mxfp4(codes, scales, 256, torch.bfloat16), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 31), (3, 33), (7, 100), (129, 1000), (2, 4097)])
def test_rows_of_odd_sizes_and_strides(rows, columns, dtype):
    from flambeau_b200.kernels import ops
    g = torch.Generator(device="cuda").manual_seed(rows)
    wide = torch.randn(rows, columns + 5, generator=g, device="cuda").to(dtype)
    blocks = -(-columns // 32)
    for x in (wide[:, :columns], wide[:, 3:columns + 3], wide[:, :columns].contiguous()):
        codes, scales = ops.quantize_mxfp4(x)
        padded = torch.nn.functional.pad(x, (0, 32 * blocks - columns))
        assert codes.shape == (rows, 16 * blocks) and scales.shape == (rows, blocks)
        assert torch.equal(values(codes, scales, 32 * blocks), nearest(padded)[0])
        assert torch.equal(ops.dequantize_mxfp4(codes, scales, columns, dtype).double(), nearest(padded)[0][:, :columns])
    empty = ops.quantize_mxfp4(wide[:0])
    assert empty[0].shape == (0, 16 * -(-(columns + 5) // 32)) and ops.dequantize_mxfp4(*empty, columns + 5).shape == (0, columns + 5)


def test_blocks_that_are_no_numbers():
    from flambeau_b200.kernels import ops
    x = torch.ones(4, 128, device="cuda")
    x[0, 5], x[1, 40], x[2, 100] = math.inf, -math.inf, math.nan
    codes, scales = ops.quantize_mxfp4(x)
    bad = torch.zeros(4, 4, dtype=torch.bool, device="cuda")
    bad[0, 0] = bad[1, 1] = bad[2, 3] = True
    assert torch.equal(scales == 255, bad)
    y = ops.dequantize_mxfp4(codes, scales, 128)
    assert torch.equal(y.isnan(), bad.repeat_interleave(32, 1)) and bool((y[~y.isnan()] == 1.0).all())
    out = torch.empty(3, 4, device="cuda")
    ops.linear(torch.ones(3, 128, device="cuda").bfloat16(), ops.Mxfp4Weight(codes, scales, 128), out, step())
    assert torch.equal(out.isnan(), torch.tensor([[True, True, True, False]] * 3, device="cuda")) and bool((out[:, 3] == 128.0).all())


def operands(M, N, K, seed=0, groups=None):
    from flambeau_b200.kernels import ops
    g = torch.Generator(device="cuda").manual_seed(seed + M)
    a = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    codes, scales = ops.quantize_mxfp4(torch.randn(*([groups] if groups else []), N, K, generator=g, device="cuda") / K ** 0.5)
    return a, ops.Mxfp4Weight(codes, scales, K), values(codes, scales, K)


def bounds(a, w, out_dtype):
    """(product, how far a sum of K float32 terms that the tensor cores cut off may be from it, then the output's rounding)."""
    want = a.double() @ w.T
    sums = a.shape[1] * 2.0 ** -23 * (a.double().abs() @ w.abs().T)
    return want, sums, sums + (0 if out_dtype == torch.float32 else 2.0 ** -8 * (want.abs() + sums))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 2, 16, 17, 32, 33, 64, 100, 129, 192, 193, 385, 700])
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (130, 64), (257, 1000), (384, 2056), (1024, 4096)])
def test_product(M, N, K, dtype):
    from flambeau_b200.kernels import ops
    a, w, dense = operands(M, N, K)
    ctx = step()
    out = torch.full((M, N + 3), 7.0, dtype=dtype, device="cuda")
    want, _, bound = bounds(a, dense, dtype)
    for view in (out[:, :N], torch.full((M, N), 7.0, dtype=dtype, device="cuda")):
        ops.linear(a, w, view, ctx)
        assert bool(((view.double() - want).abs() <= bound).all())
    assert bool((out[:, N:] == 7.0).all())
    ctx.runtime.check_status()
    assert int(ctx.ws.counters.abs().sum()) == 0


def silu_bound(want, sums, rounding):
    """|act(g) u| of alternating columns: silu's slope is below 1.1."""
    g, u, eg, eu = want[:, 0::2], want[:, 1::2], sums[:, 0::2], sums[:, 1::2]
    ref = torch.nn.functional.silu(g) * u
    return ref, 1.1 * eg * (u.abs() + eu) + g.abs() * eu + rounding * ref.abs() + 1e-30


@pytest.mark.parametrize("M", [1, 8, 33, 130, 400])
@pytest.mark.parametrize("N,K", [(2, 8), (258, 520), (1792, 2048), (256, 4104)])
def test_epilogues_shares_and_sums(M, N, K):
    from flambeau_b200.kernels import ops
    a, w, dense = operands(M, N, K, seed=3)
    ctx = step()
    want, sums, bound = bounds(a, dense, torch.float32)
    # the activation of a gated feed-forward, whole or from shares that meet in scratch
    for dtype, rounding in ((torch.float32, 2.0 ** -20), (torch.bfloat16, 2.0 ** -8)):
        out = torch.empty(M, N // 2, dtype=dtype, device="cuda")
        ops.gated_linear(a, w, out, "silu", ctx)
        ref, allowed = silu_bound(want, sums, rounding)
        assert bool(((out.double() - ref).abs() <= allowed).all())
    act = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    ops.activated_linear(a, w, act, "relu_squared", ctx)
    ref = torch.relu(want).square()
    assert bool(((act.double() - ref).abs() <= 2 * sums * (want.abs() + sums) + 2.0 ** -8 * (want.abs() + sums) ** 2).all())
    # shares of K that the next kernel adds: their count comes back, slabs behind them are not touched
    slabs = torch.full((5, M, N), 7.0, device="cuda")
    k = ops.linear_slabs(a, w, slabs, ctx)
    assert 1 <= k <= 5 and bool(((slabs[:k].double().sum(0) - want).abs() <= bound).all()) and bool((slabs[k:] == 7.0).all())
    assert ops.linear_slabs(a, w, slabs[:1], ctx) == 1 and bool(((slabs[0].double() - want).abs() <= bound).all())
    # added to a stream: one float32 add an element
    stream = torch.randn(M, N, device="cuda")
    before = stream.clone()
    if ops.linear_add(a, w, stream, ctx):
        assert M > 128
        total = want + before.double()
        assert bool(((stream.double() - total).abs() <= bound + 2.0 ** -24 * (total.abs() + bound)).all())
    else:
        assert M <= 128 and torch.equal(stream, before)
    ctx.runtime.check_status()
    assert int(ctx.ws.counters.abs().sum()) == 0


def test_scales_at_both_ends():
    """Weights of 2^100 and of 2^-120, and both in one matrix: only what lies 2^127 below the largest scale may vanish."""
    from flambeau_b200.kernels import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    a = torch.randn(9, 256, generator=g, device="cuda").bfloat16()
    base = torch.randn(130, 256, generator=g, device="cuda")
    for size in (2.0 ** 100, 2.0 ** 20, 24.0, 2.0 ** -120, 2.0 ** -126):
        codes, scales = ops.quantize_mxfp4(base * size)
        dense = values(codes, scales, 256)
        out = torch.empty(9, 130, device="cuda")
        ops.linear(a, ops.Mxfp4Weight(codes, scales, 256), out, step())
        want, _, bound = bounds(a, dense, torch.float32)
        # (below 2^-126 sums are subnormal, 2^-149 apart, which the tensor cores need not keep)
        assert bool(((out.double() - want).abs() <= bound + 256 * 2.0 ** -126).all())
    mixed = base.clone()
    mixed[::2] *= 2.0 ** 60
    codes, scales = ops.quantize_mxfp4(mixed)
    out = torch.empty(9, 130, device="cuda")
    ops.linear(a, ops.Mxfp4Weight(codes, scales, 256), out, step())
    want, _, bound = bounds(a, values(codes, scales, 256), torch.float32)
    assert bool(((out.double() - want).abs() <= bound).all())


def test_rows_of_other_strides_and_no_rows():
    from flambeau_b200.kernels import ops
    g = torch.Generator(device="cuda").manual_seed(6)
    ctx = step()
    codes, scales = ops.quantize_mxfp4(torch.randn(200, 333, generator=g, device="cuda"))
    w, dense = ops.Mxfp4Weight(codes, scales, 333), values(codes, scales, 333)
    wide = torch.randn(140, 700, generator=g, device="cuda").bfloat16()
    wide[:, :5] = math.nan                       # beside the rows, nothing of it may be read
    wide[:, 338:] = math.nan
    for a in (wide[:, 5:338], wide[::2, 5:338], wide[:, 5:338].contiguous(), wide[3:4, 5:338]):
        out = torch.empty(a.shape[0], 200, device="cuda")
        ops.linear(a, w, out, ctx)
        want, _, bound = bounds(a, dense, torch.float32)
        assert bool(((out.double() - want).abs() <= bound).all())
    for a in (wide[:, 8:341], ):                 # aligned rows apart: what is behind a row's end stays out as well
        a = a.clone(memory_format=torch.preserve_format)
        padded = torch.full((140, 336), math.nan, dtype=torch.bfloat16, device="cuda")
        padded[:, :333] = wide[:, 5:338]
        out = torch.empty(140, 200, device="cuda")
        ops.linear(padded[:, :333], w, out, ctx)
        want, _, bound = bounds(padded[:, :333], dense, torch.float32)
        assert bool(((out.double() - want).abs() <= bound).all())
    ops.linear(wide[:0, 5:338], w, torch.empty(0, 200, device="cuda"), ctx)
    assert ops.linear_slabs(wide[:0, 5:338], w, torch.empty(3, 0, 200, device="cuda"), ctx) == 1


TILES = {"sorted": [0] * 6 + [1] * 8 + [2] * 9 + [3] + [4] * 17 + [-1] * 3, "mixed": [2, 2, -1, 0, 2, 1, 1, -1, -1, 4, 3, 3, 3],
         "one": [1], "none": [-1, -1], "many": [i % 5 for i in range(450)] + [3] * 12 + [-1, 0]}


@pytest.mark.parametrize("tile", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("pattern", list(TILES))
@pytest.mark.parametrize("N,K", [(64, 64), (258, 328), (512, 1032)])
def test_groups(pattern, tile, N, K):
    from flambeau_b200.kernels import ops
    group = TILES[pattern]
    ctx = step()
    M = tile * len(group)
    x, w, dense = operands(M, N, K, seed=7, groups=5)
    tiles = torch.tensor(group, dtype=torch.int32, device="cuda")
    of = tiles.repeat_interleave(tile)
    kept = of >= 0
    want, sums = (torch.zeros(M, N, dtype=torch.float64, device="cuda") for _ in range(2))
    for e in range(5):
        want[of == e], sums[of == e], _ = bounds(x[of == e], dense[e], torch.float32)
    for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        out = torch.full((M, N), 7.0, dtype=dtype, device="cuda")
        ops.grouped_linear(x, None, w, tiles, tile, out, None, ctx)
        assert bool(((out.double() - want).abs() <= sums + rounding * (want.abs() + sums))[kept].all()) and bool((out[~kept] == 7.0).all())
    gated = torch.full((M, N // 2), 7.0, dtype=torch.bfloat16, device="cuda")
    # rows fetched by index, some of them nobody's
    index = torch.randperm(M, generator=torch.Generator().manual_seed(1)).int().cuda()
    index[::5] = -1
    rows = torch.where((index >= 0).unsqueeze(1), x[index.clamp(min=0).long()], 0)
    ops.grouped_gated_linear(x, index, w, tiles, tile, gated, "silu", ctx)
    for e in range(5):
        want[of == e], sums[of == e], _ = bounds(rows[of == e], dense[e], torch.float32)
    ref, allowed = silu_bound(want, sums, 2.0 ** -8)
    assert bool(((gated.double() - ref).abs() <= allowed)[kept].all()) and bool((gated[~kept] == 7.0).all())
    act = torch.full((M, N), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.grouped_linear(rows, None, w, tiles, tile, act, "relu_squared", ctx)
    ref = torch.relu(want).square()
    allowed = 2 * sums * (want.abs() + sums) + 2.0 ** -8 * (want.abs() + sums) ** 2
    assert bool(((act.double() - ref).abs() <= allowed)[kept].all()) and bool((act[~kept] == 7.0).all())
    ctx.runtime.check_status()


def test_refusals():
    from flambeau_b200.kernels import ops
    from flambeau_b200.kernels.library import KernelError
    ctx = step()
    x = torch.randn(64, 96, device="cuda")
    codes, scales = ops.quantize_mxfp4(x)
    w = ops.Mxfp4Weight(codes, scales, 96)
    a, out = torch.randn(4, 96, device="cuda").bfloat16(), torch.empty(4, 64, device="cuda")
    stack = ops.Mxfp4Weight.from_dense(torch.randn(3, 64, 96, device="cuda"))
    group = torch.zeros(2, dtype=torch.int32, device="cuda")
    rows = torch.randn(32, 96, device="cuda").bfloat16()
    refused = [
        lambda: ops.quantize_mxfp4(x.half()), lambda: ops.quantize_mxfp4(x.cpu()), lambda: ops.quantize_mxfp4(x.t()),
        lambda: ops.quantize_mxfp4(x[0]), lambda: ops.quantize_mxfp4(x.view(2, 32, 96)[:, ::2]), lambda: ops.quantize_mxfp4(x[:, :0]),
        lambda: ops.dequantize_mxfp4(codes, scales, 97), lambda: ops.dequantize_mxfp4(codes, scales[:, :2], 96),
        lambda: ops.dequantize_mxfp4(codes.int(), scales, 96), lambda: ops.dequantize_mxfp4(codes, scales, 96, torch.float16),
        lambda: ops.dequantize_mxfp4(codes[:, 16:], scales[:, 1:], 64), lambda: ops.Mxfp4Weight(codes, scales, 160),
        lambda: ops.Mxfp4Weight(codes[:0], scales[:0], 96), lambda: ops.Mxfp4Weight(codes.cpu(), scales.cpu(), 96),
        lambda: ops.linear(a.float(), w, out, ctx), lambda: ops.linear(a[:, :90], w, out, ctx), lambda: ops.linear(a, w, out[:3], ctx),
        lambda: ops.linear(a, w, out.half(), ctx), lambda: ops.linear(a, stack, out, ctx), lambda: ops.linear(a, w, out.t(), ctx),
        lambda: ops.gated_linear(a, w, out, "silu", ctx), lambda: ops.gated_linear(a, w, out[:, :32], "tanh", ctx),
        lambda: ops.activated_linear(a, w, out, "tanh", ctx), lambda: ops.linear_slabs(a, w, out, ctx),
        lambda: ops.linear_slabs(a, w, torch.empty(2, 4, 64, device="cuda").bfloat16(), ctx),
        lambda: ops.linear_add(a, w, out.bfloat16(), ctx),
        lambda: ops.grouped_linear(rows, None, w, group, 16, torch.empty(32, 64, device="cuda"), None, ctx),
        lambda: ops.grouped_linear(rows, None, stack, group, 24, torch.empty(32, 64, device="cuda"), None, ctx),
        lambda: ops.grouped_linear(rows, None, stack, group.long(), 16, torch.empty(32, 64, device="cuda"), None, ctx),
        lambda: ops.grouped_linear(rows, None, stack, group[:1], 16, torch.empty(32, 64, device="cuda"), None, ctx),
        lambda: ops.grouped_linear(rows, None, stack, group, 16, torch.empty(32, 64, device="cuda"), None, None),
        lambda: ops.grouped_linear(rows[:16], None, stack, group, 16, torch.empty(32, 64, device="cuda"), None, ctx),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(KernelError):             # a gate over an odd number of rows
        odd = ops.Mxfp4Weight(codes[:63].contiguous(), scales[:63].contiguous(), 96)
        ops.gated_linear(a, odd, out[:, :31], "silu", ctx)
    ctx.runtime.check_status()
