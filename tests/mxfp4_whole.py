"""Rows and four-bit weights of whole numbers: every sum of a product with them is a float32 number whatever the order of its
terms, so that a product is right when it is equal.  Used by the tests of four-bit weights; runs on any device."""
from types import SimpleNamespace

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def step():
    """What a product wants of a step: the runtime and its arena."""
    from flambeau_b200.engine.runtime import Runtime
    rt = Runtime("cuda:0", "bfloat16")
    return SimpleNamespace(runtime=rt, ws=rt.ws)


def numbers(codes, scales):
    """float64 numbers of codes and scales, from the definition."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    grid = torch.tensor(GRID + tuple(-x for x in GRID), dtype=torch.float64, device=codes.device)
    return grid[c.int()] * torch.exp2(scales.double() - 127.0).repeat_interleave(32, -1)


def rows(M, K, seed, top=63, device="cuda"):
    """Whole numbers up to 4 `top` of more bits than an e4m3 number has: every block of 32 times 1, 2 or 4, so that no block's
    scale can stand for its neighbour's."""
    g = torch.Generator(device=device).manual_seed(seed)
    a = torch.randint(-top, top + 1, (M, K), generator=g, device=device)
    size = torch.randint(0, 3, (M, -(-K // 32)), generator=g, device=device).repeat_interleave(32, 1)[:, :K]
    return (a << size).bfloat16()


def weight_codes(shape, K, seed, device="cuda"):
    """Random codes under scales of 2 and 4 (whole numbers up to 24), for K a multiple of 32."""
    g = torch.Generator(device=device).manual_seed(seed)
    codes = torch.randint(0, 256, (*shape, K // 2), generator=g, dtype=torch.uint8, device=device)
    scales = torch.randint(128, 130, (*shape, K // 32), generator=g, dtype=torch.uint8, device=device)
    return codes, scales


def product(a, w):
    """a w^T in float64, for sums that float32 holds in any order: the positive terms of each, and the negative ones, add up to
    less than 2^24 (an eighth less, for rows whose first part is rounded up)."""
    a = a.double()
    want = a @ w.T
    assert float((a.abs() @ w.abs().T + want.abs()).max()) / 2 < 2.0 ** 24 * 8 / 9, "float32 does not hold every sum of these"
    return want


def split(x):
    """The numbers that the products take for rows x [M, K] (bfloat16; K a multiple of 32), in float64: a block's two e4m3 parts,
    the second a 32nd of the first's size, under the power of two that brings its largest magnitude to 2^7 .. 2^8 (blocks below
    2^-115 under that one's)."""
    b = x.double().view(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top)[1] - 1, -115).clamp(min=-115).double()
    y = b * torch.exp2(7 - e)
    first = y.float().to(torch.float8_e4m3fn).double()
    second = ((y - first) * 32).float().to(torch.float8_e4m3fn).double() / 32
    return (first * torch.exp2(e - 7)).view(x.shape), (second * torch.exp2(e - 7)).view(x.shape)
