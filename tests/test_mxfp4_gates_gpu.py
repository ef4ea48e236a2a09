"""SiLU gates in the epilogue of products with four-bit weights, over the whole range of the gate."""
import pytest
import torch

from mxfp4_whole import step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [3, 20, 40, 130])
def test_silu_over_the_gates_range(M, dtype):
    """Every gate and every factor is one number of a row, so that both sides of the activation are exact.

    The bound, in 2^-24: an exponential of half the gate within 4 of itself and a rounding of its correction, twice for gates below
    zero (10), a reciprocal within 2, five roundings (the sum below the line, four products): 17, and 20 are allowed; what
    lies below float32's normal numbers may be zero."""
    from flambeau_b200.kernels import ops
    n = 65                                       # gates; each in a block of its own, its factor in another
    K = 64 * n
    weight = torch.zeros(2 * n, K, device="cuda")
    at = torch.arange(n, device="cuda")
    weight[2 * at, 64 * at] = 1.0
    weight[2 * at + 1, 64 * at + 32] = 1.0
    g = torch.linspace(-170, 100, M * n, dtype=torch.float64)[torch.randperm(M * n, generator=torch.Generator().manual_seed(1))]
    special = torch.tensor([0.0, -0.0, 1.0, -1.0, -87.0, -87.5, -88.0, -89.0, -100.0, -104.0, 88.0, 3e38, 1e-38, -1e-38, -300.0, -3e38])
    g[:16] = special.double()
    g = g.view(M, n).cuda().bfloat16()
    u = torch.exp2(torch.randint(-20, 100, (M, n), generator=torch.Generator().manual_seed(2)).double())
    u = (u * torch.where(torch.arange(M * n).view(M, n) % 3 == 0, -1.5, 1.0)).cuda()
    u[g > 1e30] = 0.5
    u = u.bfloat16()
    a = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    a[:, 0::64], a[:, 32::64] = g, u
    ref = g.double() * torch.sigmoid(g.double()) * u.double()
    ctx = step()
    w = ops.Mxfp4Weight.from_dense(weight)
    out = torch.empty(M, n, dtype=dtype, device="cuda")
    ops.gated_linear(a, w, out, "silu", ctx)
    rounding = 20 * 2.0 ** -24 + (0.0 if dtype == torch.float32 else 2.0 ** -8)
    assert bool(((out.double() - ref).abs() <= rounding * ref.abs() + 2.0 ** -126).all())
    ctx.runtime.check_status()


@pytest.mark.parametrize("M", [3, 40])
def test_silu_of_no_numbers(M):
    """Gates whose sums pass float32, and NaN, as the formula has them."""
    from flambeau_b200.kernels import ops
    weight = torch.zeros(4, 64, device="cuda")
    weight[0, 0] = weight[1, 32] = weight[2, 0] = weight[3, 32] = 2.0 ** 100
    ctx = step()
    a = torch.zeros(M, 64, dtype=torch.bfloat16, device="cuda")
    a[:, 0], a[:, 32] = 2.0 ** 60, 1.0           # the sum is infinite: so is the result
    out = torch.empty(M, 2, device="cuda")
    ops.gated_linear(a, ops.Mxfp4Weight.from_dense(weight), out, "silu", ctx)
    assert bool((out == float("inf")).all())
    a[:, 0] = float("nan")
    ops.gated_linear(a, ops.Mxfp4Weight.from_dense(weight), out, "silu", ctx)
    assert bool(out.isnan().all())
    ctx.runtime.check_status()
