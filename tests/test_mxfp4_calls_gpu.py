"""Four-bit weights as programs call them: captured and replayed, on other streams and two at a time, with rows fetched twice, in the
forms that only certain sizes reach, and where offsets pass 32 bits."""
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def step():
    from flambeau_b200.engine.runtime import Runtime
    rt = Runtime("cuda:0", "bfloat16")
    return SimpleNamespace(runtime=rt, ws=rt.ws)


def numbers(codes, scales):
    """float64 numbers of codes and scales, from the definition."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    grid = torch.tensor(GRID + [-x for x in GRID], dtype=torch.float64, device=codes.device)
    return grid[c.int()] * torch.exp2(scales.double() - 127.0).repeat_interleave(32, -1)


def drawn(shape, K, seed):
    """A weight of random codes under scales around 1 / 64, with its codes and scales."""
    from flambeau_b200.kernels import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = K // 32
    codes = torch.randint(0, 256, (*shape, 16 * blocks), generator=g, dtype=torch.uint8, device="cuda")
    scales = torch.randint(119, 123, (*shape, blocks), generator=g, dtype=torch.uint8, device="cuda")
    return ops.Mxfp4Weight(codes, scales, K), codes, scales


def rows(M, K, seed):
    return torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()


def product(a, w):
    """(a w^T, how far a sum of K float32 terms that the tensor cores cut off may be from it), in float64."""
    a = a.double()
    return a @ w.T, a.shape[1] * 2.0 ** -23 * (a.abs() @ w.abs().T)


def close(got, want, allowed, rounding=0.0):
    return bool(((got.double() - want).abs() <= allowed + rounding * (want.abs() + allowed)).all())


def gated(want, sums, rounding):
    """silu(g) u of alternating columns (silu's slope is below 1.1), how far it may be off."""
    g, u, eg, eu = want[:, 0::2], want[:, 1::2], sums[:, 0::2], sums[:, 1::2]
    ref = torch.nn.functional.silu(g) * u
    return ref, 1.1 * eg * (u.abs() + eu) + g.abs() * eu + rounding * ref.abs() + 1e-30


@pytest.mark.parametrize("M", [1, 8])
def test_few_rows_of_a_large_matrix(M):
    """Stretches of K so long that the rows are split ahead of the product, and ones so short that the product does it."""
    from flambeau_b200.kernels import ops
    ctx = step()
    for N, K in ((16384, 9216), (4096, 2048)):
        w, codes, scales = drawn((N,), K, 1)
        dense = numbers(codes, scales)
        a = rows(M, K, 2)
        want, sums = product(a, dense)
        out, act = torch.empty(M, N, device="cuda"), torch.empty(M, N // 2, dtype=torch.bfloat16, device="cuda")
        ops.linear(a, w, out, ctx)
        assert close(out, want, sums)
        ops.gated_linear(a, w, act, "silu", ctx)
        ref, allowed = gated(want, sums, 2.0 ** -8)
        assert close(act, ref, allowed)
        slabs = torch.full((8, M, N), 7.0, device="cuda")
        k = ops.linear_slabs(a, w, slabs, ctx)
        assert close(slabs[:k].double().sum(0), want, sums) and bool((slabs[k:] == 7.0).all())
    ctx.runtime.check_status()
    assert int(ctx.ws.counters.abs().sum()) == 0


def test_an_odd_number_of_feature_tiles_in_pairs():
    """225 tiles of 128 features, of which the last holds 118: 113 pairs, the last one of a single tile."""
    from flambeau_b200.kernels import ops
    ctx = step()
    N, K = 28790, 4096
    w, codes, scales = drawn((N,), K, 3)
    dense = numbers(codes, scales)
    for M in (100, 128, 256):
        a = rows(M, K, M)
        want, sums = product(a, dense)
        for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
            out = torch.full((M, N + 2), 7.0, dtype=dtype, device="cuda")
            for view, rest in ((out[:, :N], out[:, N:]), (out[:, 1:N + 1], out[:, N + 1:])):
                out.fill_(7.0)
                ops.linear(a, w, view, ctx)
                assert close(view, want, sums, rounding) and bool((rest == 7.0).all())
            act = torch.empty(M, N // 2, dtype=dtype, device="cuda")
            ops.gated_linear(a, w, act, "silu", ctx)
            ref, allowed = gated(want, sums, rounding + 2.0 ** -20)
            assert close(act, ref, allowed)
        slabs = torch.full((3, M, N), 7.0, device="cuda")
        k = ops.linear_slabs(a, w, slabs, ctx)
        assert close(slabs[:k].double().sum(0), want, sums) and bool((slabs[k:] == 7.0).all())
        stream = torch.randn(M, N, device="cuda")
        before = stream.double()
        if ops.linear_add(a, w, stream, ctx):
            assert close(stream, want + before, sums, 2.0 ** -24)
    ctx.runtime.check_status()
    assert int(ctx.ws.counters.abs().sum()) == 0


@pytest.mark.parametrize("M", [40, 64])
def test_pairs_of_feature_tiles_and_up_to_64_rows(M):
    """Both parts of the rows side by side, two feature tiles a unit, the last one alone."""
    from flambeau_b200.kernels import ops
    ctx = step()
    N, K = 28790, 4096 + 64
    w, codes, scales = drawn((N,), K, 31)
    a = rows(M, K, M)
    want, sums = product(a, numbers(codes, scales))
    for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        out = torch.full((M, N + 2), 7.0, dtype=dtype, device="cuda")
        ops.linear(a, w, out[:, :N], ctx)
        assert close(out[:, :N], want, sums, rounding) and bool((out[:, N:] == 7.0).all())
        act = torch.empty(M, N // 2, dtype=dtype, device="cuda")
        ops.gated_linear(a, w, act, "silu", ctx)
        ref, allowed = gated(want, sums, rounding + 2.0 ** -20)
        assert close(act, ref, allowed)
    slabs = torch.full((3, M, N), 7.0, device="cuda")
    k = ops.linear_slabs(a, w, slabs, ctx)
    assert close(slabs[:k].double().sum(0), want, sums) and bool((slabs[k:] == 7.0).all())
    ctx.runtime.check_status()
    assert int(ctx.ws.counters.abs().sum()) == 0


@pytest.mark.parametrize("M,N,K", [(48, 384, 14336), (100, 256, 8192), (130, 200, 16384)])
def test_shares_of_many_rows_meet(M, N, K):
    """So few tiles that K is split, by rows that leave the last tile of tokens open."""
    from flambeau_b200.kernels import ops
    ctx = step()
    w, codes, scales = drawn((N,), K, 4)
    dense = numbers(codes, scales)
    a = rows(M, K, 5)
    want, sums = product(a, dense)
    for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        out = torch.full((M, N + 1), 7.0, dtype=dtype, device="cuda")
        ops.linear(a, w, out[:, :N], ctx)
        assert close(out[:, :N], want, sums, rounding) and bool((out[:, N] == 7.0).all())
    for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        act = torch.empty(M, N // 2, dtype=dtype, device="cuda")
        ops.gated_linear(a, w, act, "silu", ctx)
        ref, allowed = gated(want, sums, rounding + 2.0 ** -20)
        assert close(act, ref, allowed)
    relu = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    ops.activated_linear(a, w, relu, "relu_squared", ctx)
    ref = torch.relu(want).square()
    assert bool(((relu.double() - ref).abs() <= 2 * sums * (want.abs() + sums) + 2.0 ** -8 * (want.abs() + sums) ** 2).all())
    stream = torch.randn(M, N, device="cuda")
    before = stream.double()
    if ops.linear_add(a, w, stream, ctx):
        # (the shares' sum is rounded once more when it is added)
        assert close(stream, want + before, sums, 2.0 ** -24)
    ctx.runtime.check_status()
    assert int(ctx.ws.counters.abs().sum()) == 0


RUNS = {32: [1, 2, 3, 4, 1, 2, 2, 1, 3, 1, 2, 2], 64: [1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1], 48: [1, 2, 1, 1, 2, 1, 1, 1, 1, 1, 1, 1]}


@pytest.mark.parametrize("tile", list(RUNS))
@pytest.mark.parametrize("N,K", [(64, 96), (386, 640)])
def test_groups_of_few_rows(tile, N, K):
    """Many groups with a tile or two each: rows by index, the same one several times, some of them nobody's, with shares."""
    from flambeau_b200.kernels import ops
    ctx = step()
    groups = 24
    w, codes, scales = drawn((groups, N), K, 6)
    dense = numbers(codes, scales)
    order = [g for g, n in zip((3, 5, 0, 7, 11, 2, 23, 9, 1, 22, 4, 6), RUNS[tile]) for _ in range(n)] + [-1, -1]
    M = tile * len(order)
    assert M <= 64 * groups
    tiles = torch.tensor(order, dtype=torch.int32, device="cuda")
    of = tiles.repeat_interleave(tile)
    kept = of >= 0
    x = rows(90, K, 7)
    index = torch.randint(-1, 90, (M,), generator=torch.Generator().manual_seed(2)).int().cuda()
    index[:3] = 5
    pair = torch.randperm(M, generator=torch.Generator().manual_seed(3)).int().cuda()
    share = torch.rand(M, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    for shares in (False, True):
        a = torch.where((index >= 0).unsqueeze(1), x[index.clamp(min=0).long()], 0)
        if shares:                               # (the scaled row is rounded to bfloat16 once)
            a = (a.float() * share[pair.long()].unsqueeze(1)).bfloat16()
        want, sums = (torch.zeros(M, N, dtype=torch.float64, device="cuda") for _ in range(2))
        for e in set(order) - {-1}:
            want[of == e], sums[of == e] = product(a[of == e], dense[e])
        more = dict(row_share=share, row_pair=pair) if shares else {}
        for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
            out = torch.full((M, N), 7.0, dtype=dtype, device="cuda")
            ops.grouped_linear(x, index, w, tiles, tile, out, None, ctx, **more)
            assert close(out[kept], want[kept], sums[kept], rounding) and bool((out[~kept] == 7.0).all())
            act = torch.full((M, N // 2), 7.0, dtype=dtype, device="cuda")
            ops.grouped_gated_linear(x, index, w, tiles, tile, act, "silu", ctx, **more)
            ref, allowed = gated(want, sums, rounding + 2.0 ** -20)
            assert close(act[kept], ref[kept], allowed[kept]) and bool((act[~kept] == 7.0).all())
    ctx.runtime.check_status()


@pytest.mark.parametrize("name", ["silu", "gelu_tanh", "limited"])
def test_every_gate(name):
    """The gates' own kernel on the product's float32 numbers is the reference: within its error, and the product's times the gates' slopes."""
    from flambeau_b200.kernels import ops
    gate = ops.GateActivation(name, limit=1.5, slope=1.702) if name == "limited" else name
    ctx = step()
    for M in (3, 20, 40, 128):
        w, codes, scales = drawn((260,), 512, 8)
        a = rows(M, 512, 9)
        plain, want, out = torch.empty(M, 260, device="cuda"), torch.empty(M, 130, device="cuda"), torch.empty(M, 130, device="cuda")
        ops.linear(a, w, plain, ctx)
        ops.gate_mul(plain, want, activation=gate)
        ops.gated_linear(a, w, out, gate, ctx)
        # both epilogues start from float32 sums of the same terms, cut off in another order at most; slopes of gates stay below 2
        sums = 512 * 2.0 ** -22 * (a.float().abs() @ numbers(codes, scales).float().abs().T)
        g, u = plain[:, 0::2].abs(), plain[:, 1::2].abs()
        allowed = 2 * sums[:, 0::2] * (u + 1) + (g + 1) * sums[:, 1::2] + 2.0 ** -18 * (g + 1) * (u + 1)
        assert bool(((out - want).abs() <= allowed).all())
    ctx.runtime.check_status()


def test_captured_and_replayed():
    """Two graphs over one workspace, replayed in turn with new rows in the same tensors, give what the eager calls give."""
    from flambeau_b200.kernels import ops
    ctx = step()
    calls = []
    for M, N, K in ((8, 4096, 2048), (8, 1024, 4096), (67, 640, 4096), (300, 1024, 512)):
        w, _, _ = drawn((N,), K, M)
        a, out = rows(M, K, 10), torch.empty(M, N // 2, dtype=torch.bfloat16, device="cuda")
        calls.append((a, out, lambda a=a, w=w, out=out: ops.gated_linear(a, w, out, "silu", ctx)))
    stack, _, _ = drawn((6, 256), 512, 11)
    tiles = torch.tensor([0, 0, 3, 5, -1, 1], dtype=torch.int32, device="cuda")
    for tile in (16, 64):
        a, out = rows(6 * tile, 512, 12), torch.zeros(6 * tile, 256, device="cuda")
        calls.append((a, out, lambda a=a, out=out, tile=tile: ops.grouped_linear(a, None, stack, tiles, tile, out, None, ctx)))
    for _, _, call in calls:
        call()                                   # (the workspace has its size, the kernels are loaded)
    torch.cuda.synchronize()
    graphs = []
    for part in (calls[::2], calls[1::2]):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _, _, call in part:
                call()
        graphs.append(graph)
    for turn in range(3):
        for i, (a, _, _) in enumerate(calls):
            a.copy_(rows(*a.shape, seed=100 * turn + i))
        want = []
        for _, out, call in calls:
            call()
            want.append(out.clone())
            out.fill_(-1.0)
        kept = want[-1] != 0
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (a, out, _), ref in zip(calls[:4], want):
            assert torch.equal(out, ref)
        for (a, out, _), ref in zip(calls[4:], want[4:]):
            tile = a.shape[0] // 6
            used = (tiles >= 0).repeat_interleave(tile)
            assert torch.equal(out[used], ref[used]) and bool((out[~used] == -1.0).all())
    ctx.runtime.check_status()


def test_on_two_streams_at_a_time():
    """Two contexts, each on a stream of its own, with products of the same weights in flight together."""
    from flambeau_b200.kernels import ops
    contexts, streams = [step(), step()], [torch.cuda.Stream(), torch.cuda.Stream()]
    shapes = ((8, 4096, 4096), (67, 1024, 4096), (300, 2048, 1024), (1, 1024, 8192))
    weights = [drawn((N,), K, i)[0] for i, (_, N, K) in enumerate(shapes)]
    inputs = [[rows(M, K, 20 + 10 * s + i) for i, (M, _, K) in enumerate(shapes)] for s in range(2)]
    want = [[torch.empty(M, N, device="cuda") for M, N, _ in shapes] for _ in range(2)]
    got = [[torch.empty(M, N, device="cuda") for M, N, _ in shapes] for _ in range(2)]
    for s in range(2):
        for a, w, out in zip(inputs[s], weights, want[s]):
            ops.linear(a, w, out, contexts[s])
    torch.cuda.synchronize()
    for _ in range(5):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                for a, w, out in zip(inputs[s], weights, got[s]):
                    ops.linear(a, w, out, contexts[s])
    torch.cuda.synchronize()
    for s in range(2):
        assert all(torch.equal(g, w) for g, w in zip(got[s], want[s]))
        contexts[s].runtime.check_status()


def test_offsets_past_32_bits():
    """2^32 weights of one matrix, more than 2^31 numbers of rows to quantise: the last ones are as right as the first."""
    from flambeau_b200.kernels import ops
    ctx = step()
    N = K = 1 << 16
    w, codes, scales = drawn((N,), K, 13)
    a = rows(3, K, 14)
    out = torch.empty(3, N, device="cuda")
    ops.linear(a, w, out, ctx)
    for part in (slice(0, 200), slice(N - 200, N)):
        want, sums = product(a, numbers(codes[part], scales[part]))
        assert close(out[:, part], want, sums)
    del w, codes, scales, out
    x = torch.empty((1 << 16) + 1, 1 << 15, dtype=torch.bfloat16, device="cuda")
    x.fill_(0.25)
    x[-2:] = rows(2, 1 << 15, 15)
    codes, scales = ops.quantize_mxfp4(x)
    ends = ops.quantize_mxfp4(x[-2:].clone())
    assert torch.equal(codes[-2:], ends[0]) and torch.equal(scales[-2:], ends[1]) and int(scales[:-2].max()) == int(scales[:-2].min())
    back = ops.dequantize_mxfp4(codes, scales, 1 << 15, torch.bfloat16)
    assert torch.equal(back[-2:].double(), numbers(*ends)) and bool((back[:-2] == 0.25).all())
    ctx.runtime.check_status()


def test_indexes_that_name_no_row_and_no_group():
    """A row that is none of the input's counts as zeros, as a negative one does; a group beyond the last one reads no weights of others."""
    from flambeau_b200.kernels import ops
    ctx = step()
    w, codes, scales = drawn((3, 96), 64, 18)
    dense = numbers(codes, scales)
    x = rows(10, 64, 19)
    for tile in (16, 32):
        M = 3 * tile
        tiles = torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda")
        index = (torch.arange(M, device="cuda") % 10).int()
        index[1], index[tile + 2], index[2 * tile + 3] = 10, 2 ** 31 - 1, -2 ** 31
        a = torch.where(((index >= 0) & (index < 10)).unsqueeze(1), x[index.clamp(0, 9).long()], 0)
        out = torch.empty(M, 96, device="cuda")
        ops.grouped_linear(x, index, w, tiles, tile, out, None, ctx)
        for i, g in enumerate((0, 2, 1)):
            part = slice(i * tile, (i + 1) * tile)
            want, sums = product(a[part], dense[g])
            assert close(out[part], want, sums)
        ops.grouped_linear(x, index, w, torch.tensor([0, 7, 1], dtype=torch.int32, device="cuda"), tile, out, None, ctx)
        want, sums = product(a[:tile], dense[0])
        assert close(out[:tile], want, sums)
    ctx.runtime.check_status()


def test_what_products_refuse():
    from flambeau_b200.kernels import ops
    from flambeau_b200.kernels.library import KernelError
    w, _, _ = drawn((64,), 96, 16)
    a, out = rows(4, 96, 17), torch.empty(4, 64, device="cuda")
    ctx = step()
    for call in (lambda: ops.linear(a, w, out), lambda: ops.linear(rows(4, 192, 1)[:, ::2], w, out, ctx),
                 lambda: ops.linear(a[:1].expand(4, 96), w, out, ctx), lambda: ops.linear(a.cpu(), w, out, ctx),
                 lambda: ops.linear(a, w, out.cpu(), ctx), lambda: ops.gated_linear(a, w, out[:, :32], "silu", None)):
        with pytest.raises(KernelError):
            call()
            pytest.fail("not refused")
    ctx.runtime.check_status()
