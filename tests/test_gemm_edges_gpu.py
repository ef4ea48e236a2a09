"""Stored-weight products on the two-SM kernel whose output rows end inside 16 bytes: nothing beyond a row's end is written."""
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu


def operands(M, N, K, seed):
    """Whole numbers up to 15: float32 holds every sum of their products, in any order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randint(-15, 16, (M, K), generator=g, device="cuda").bfloat16()
    w = torch.randint(-15, 16, (N, K), generator=g, device="cuda").bfloat16()
    return a, w, a.double() @ w.double().T


@pytest.mark.parametrize("columns", [10001, 10002, 10003, 10004, 10006])
@pytest.mark.parametrize("M", [300, 515])
def test_rows_that_end_inside_16_bytes(M, columns):
    from flambeau_b200.engine.runtime import Runtime
    from flambeau_b200.kernels import ops
    rt = Runtime("cuda:0", "bfloat16")
    ctx = SimpleNamespace(runtime=rt, ws=rt.ws)
    a, w, want = operands(M, columns, 200, M)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.full((M, 10016), 7.0, dtype=dtype, device="cuda")   # (rows on 16-byte borders)
        ops.linear(a, w, wide[:, :columns], ctx)
        assert torch.equal(wide[:, :columns], want.to(dtype)) and bool((wide[:, columns:] == 7.0).all())
        act = torch.full((M, 10016), 7.0, dtype=dtype, device="cuda")
        ops.activated_linear(a, w, act[:, :columns], "relu_squared", ctx)
        assert torch.equal(act[:, :columns], want.float().clamp(min=0).square().to(dtype)) and bool((act[:, columns:] == 7.0).all())
    wide = torch.full((M, 10016), 7.0, device="cuda")
    if ops.linear_add(a, w, wide[:, :columns], ctx):
        assert torch.equal(wide[:, :columns].double(), want + 7.0)
    assert bool((wide[:, columns:] == 7.0).all())
    rt.check_status()


@pytest.mark.parametrize("columns", [5001, 5002, 5004])
def test_gated_rows_that_end_inside_16_bytes(columns):
    from flambeau_b200.engine.runtime import Runtime
    from flambeau_b200.kernels import ops
    rt = Runtime("cuda:0", "bfloat16")
    ctx = SimpleNamespace(runtime=rt, ws=rt.ws)
    M = 515
    a, w, want = operands(M, 2 * columns, 200, 1)
    g, u = want[:, 0::2], want[:, 1::2]
    ref = g * torch.sigmoid(g) * u
    for dtype, rounding in ((torch.float32, 2.0 ** -20), (torch.bfloat16, 2.0 ** -8 + 2.0 ** -20)):
        wide = torch.full((M, 5008), 7.0, dtype=dtype, device="cuda")
        ops.gated_linear(a, w, wide[:, :columns], "silu", ctx)
        assert bool(((wide[:, :columns].double() - ref).abs() <= rounding * ref.abs() + 2.0 ** -126 * (g * u).abs()).all())
        assert bool((wide[:, columns:] == 7.0).all())
    rt.check_status()
