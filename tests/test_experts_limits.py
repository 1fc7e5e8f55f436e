"""Limits of sizes of the experts' operators and the 4-bit values, without a GPU:
refused by the check of the entry point (error 1), before any CUDA call."""
from test_experts_abi import A, _lib, _refused


def test_route_limits():
    lib = _lib()
    for tokens in (2 ** 31 - 1, 2 ** 31 - 128, 2 ** 31 - 1024):
        _refused(lib.tdb_moe_route(A, 0, 8, tokens, 8, 1, 1, A, A, A, A, A, A, None), b"tokens")
        _refused(lib.tdb_moe_route_bwd(A, 0, 8, tokens, 8, 1, 1, A, A, A, A, 0, 8, None), b"tokens")


def test_4_bit_limits():
    """A grid has at most 65535 blocks of 1024 values along K."""
    lib = _lib()
    for K in (2 ** 26 - 992, 2 ** 26 - 32, 2 ** 26):
        _refused(lib.tdb_mx4_quantize(A, K, 1, 8, K, None, 0, A, A, None), b"multiple of 32")
        _refused(lib.tdb_mx4_dequantize(A, A, 1, 8, K, None, 0, A, K, None), b"multiple of 32")
        _refused(lib.tdb_mx4_gemm(A, A, A, A, None, 1, A, 32, 8, 32, K, None, 0, None), b"K of 32")
