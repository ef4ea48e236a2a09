"""What the C entries of four-bit weights refuse, and the sizes that they name, on the CPU: nothing is launched."""
import pytest

from flambeau_b200.kernels.library import lib

LARGEST = 2 ** 31 - 1
A = 1 << 20                                      # an address that is never followed


def refused(code, what):
    message = lib().fb_last_error().decode()
    assert code < 0 and what in message, (code, message)


@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (129, 257), (LARGEST, 1), (1, LARGEST), (LARGEST, LARGEST)])
def test_bytes_of_tiles(N, K):
    assert lib().fb_mxfp4_tile_bytes(N, K) == -(-N // 128) * -(-K // 128) * 8704


def test_sizes_of_weights():
    for groups, N, K in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (65536, 1, 1), (1, 65535 * 128 + 1, 1), (1, LARGEST, 1), (1, 1, LARGEST),
                         (1, 1, (1 << 30) + 1)):
        refused(lib().fb_mxfp4_tiles(A, A, groups, N, K, A, 0), "bad sizes")
    refused(lib().fb_mxfp4_tiles(A + 1, A, 1, 1, 1, A, 0), "aligned")
    refused(lib().fb_mxfp4_tiles(A, A, 1, 1, 1, A + 8, 0), "aligned")
    for K in (0, -1, (1 << 30) + 1, LARGEST):
        refused(lib().fb_quantize_mxfp4(A, 0, LARGEST, 1, K, A, A, 0), "bad sizes")
        refused(lib().fb_dequantize_mxfp4(A, A, 1, K, A, 0, LARGEST, 0), "bad sizes")
    refused(lib().fb_quantize_mxfp4(A, 0, 31, 2, 32, A, A, 0), "stride")
    refused(lib().fb_quantize_mxfp4(A, 0, 32, 2, 32, A + 4, A, 0), "aligned")


def product(M=4, N=64, K=96, **changed):
    a = dict(X=A, lda=K, W=A, out=A, dtype=0, ldo=N, slab_stride=0, slabs=0, used=None, act=0, limit=0.0, slope=0.0, plain=0, add=0,
             counters=A, n_counters=64, scratch=A, bytes=1 << 40, status=A)
    a.update(changed)
    return lib().fb_gemm_mxfp4(a["X"], a["lda"], a["W"], a["out"], a["dtype"], a["ldo"], a["slab_stride"], a["slabs"], a["used"], M, N, K,
                               a["act"], a["limit"], a["slope"], a["plain"], a["add"], a["counters"], a["n_counters"], a["scratch"],
                               a["bytes"], a["status"], 0)


def test_products():
    for sizes in (dict(M=-1), dict(N=0), dict(K=0)):
        refused(product(**sizes), "bad sizes")
    for sizes in (dict(N=LARGEST, K=LARGEST), dict(N=LARGEST, K=129), dict(N=1, K=LARGEST)):
        refused(product(**sizes), "too many weights")
    refused(product(lda=95), "stride")
    refused(product(ldo=63), "stride")
    refused(product(dtype=7), "dtype")
    refused(product(act=9), "gate")
    refused(product(act=1, plain=1), "gate")
    refused(product(N=63, act=1), "gate")
    refused(product(act=3, limit=0.0), "gate")
    refused(product(plain=9), "activation")
    for wrong in (dict(X=A + 1), dict(W=A + 8), dict(W=0), dict(status=0)):
        refused(product(**wrong), "unaligned rows or weights")
    refused(product(out=A + 2), "unaligned output")
    refused(product(slab_stride=4 * 64 - 1, slabs=2), "slabs")
    refused(product(slab_stride=4 * 64, slabs=2, dtype=1), "slabs")
    refused(product(add=1, dtype=1), "added")
    refused(product(counters=0), "counters")
    refused(product(n_counters=0), "counters")


def test_the_largest_product_is_looked_up_without_an_overflow():
    """Sizes up to what a weight may have: bytes of scratch are named, never less than the rows' two parts."""
    for M, N, K in ((1, 65535 * 128, 128), (8, 128, 1 << 30), (33, 65535 * 128, 128), (LARGEST // 2, 128, 128)):
        for slabs in (0, 1):
            got = lib().fb_gemm_mxfp4_scratch_bytes(M, N, K, 1 << 16, slabs, 0)
            assert got == 0 or got >= 2 * M * K


def test_grouped_products():
    def call(M=64, N=64, K=96, groups=2, tiles=A, tile=16, x_rows=64, index=0, share=0, pair=0, scratch=A, size=1 << 40):
        return lib().fb_gemm_mxfp4_grouped(A, K, x_rows, index, share, pair, A, groups, tiles, tile, A, 0, N, M, N, K, 0, 0.0, 0.0, 0,
                                           scratch, size, A, 0)
    for groups in (dict(groups=0), dict(tiles=0)):
        refused(call(**groups), "no groups")
    refused(call(x_rows=63), "fewer than")
    for tile in (8, 24, 144, 48):
        refused(call(tile=tile), "whole tiles")
    refused(call(share=A), "shares need")
    refused(call(index=A, share=A), "shares need")
    refused(call(scratch=0), "scratch missing")
    refused(call(scratch=A + 64), "scratch missing")
    refused(call(size=1000), "scratch missing")
