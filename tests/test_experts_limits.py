"""Limits of sizes of the experts' operators and the 4-bit values, without a GPU:
refused by the check of the entry point (error 1), before any CUDA call."""
from test_experts_abi import A, _lib, _refused


def test_route_limits():
    lib = _lib()
    for tokens in (2 ** 31 - 1, 2 ** 31 - 128, 2 ** 31 - 1024):
        _refused(lib.tdb_moe_route(A, 0, 8, tokens, 8, 1, 1, A, A, A, A, A, A, None), b"tokens")
        _refused(lib.tdb_moe_route_bwd(A, 0, 8, tokens, 8, 1, 1, A, A, A, A, 0, 8, None), b"tokens")
