"""Entry points of the experts' operators and the 4-bit products, without a GPU:
the ctypes signatures against csrc/tdb.h, and the refusals that come before any
CUDA call (with made-up addresses)."""
import ctypes

import pytest

A, ODD = 0x10000, 0x10008  # aligned and misaligned made-up device addresses


def _lib():
    import tempname_dcu_b200.ops.grouped  # noqa: F401
    import tempname_dcu_b200.ops.moe  # noqa: F401
    import tempname_dcu_b200.ops.mx4  # noqa: F401
    from tempname_dcu_b200.ops import native
    return native.lib()


def test_signatures_match_the_header():
    from test_abi_header import _ctypes_kind, _prototypes
    _lib()
    from tempname_dcu_b200.ops import native
    protos = _prototypes()
    names = [n for n in protos if n.startswith(("tdb_moe_", "tdb_grouped_", "tdb_mx4_"))]
    assert len(names) >= 14
    for name in names:
        if name in native.SIGNATURES:
            assert [_ctypes_kind(t) for t in native.SIGNATURES[name]] == protos[name], name
    assert sum(n in native.SIGNATURES for n in names) == len(names)


def _refused(rc, text):
    from tempname_dcu_b200.ops import native
    assert rc == 1 and text in native.lib().tdb_last_error(), native.lib().tdb_last_error()


def test_moe_refusals():
    lib = _lib()

    def route(ld=8, tokens=4, E=8, k=2, logits=A, scratch=None):
        return lib.tdb_moe_route(logits, 0, ld, tokens, E, k, 1, A, A, A, A, A, scratch, None)
    for bad in (dict(E=0), dict(E=513, ld=600), dict(k=0), dict(k=9), dict(k=17, E=20, ld=20), dict(ld=7),
                dict(tokens=-1), dict(tokens=2 ** 30, k=2)):
        _refused(route(**bad), b"experts")
    _refused(route(logits=None), b"null")
    _refused(route(tokens=1000), b"null")  # more than one block needs scratch
    assert lib.tdb_moe_route_scratch_ints(128, 8) == 0 and lib.tdb_moe_route_scratch_ints(129, 8) == 16
    _refused(lib.tdb_moe_route_bwd(A, 0, 8, 4, 8, 2, 1, A, A, A, A, 0, 7, None), b"experts")
    _refused(lib.tdb_moe_dispatch(A, 64, 4, 2, 60, A, A, 64, None), b"multiple of 8")
    _refused(lib.tdb_moe_dispatch(ODD, 64, 4, 2, 64, A, A, 64, None), b"aligned")
    _refused(lib.tdb_moe_dispatch(A, 68, 4, 2, 64, A, A, 64, None), b"aligned")
    _refused(lib.tdb_moe_dispatch(A, 64, 4, 17, 64, A, A, 64, None), b"choices")
    _refused(lib.tdb_moe_combine(A, 64, 4, 2, 64, A, A, ODD, 64, A, 64, None), b"aligned")
    _refused(lib.tdb_moe_combine_bwd(A, 64, A, 56, 4, 2, 64, A, A, A, 64, A, None), b"aligned")
    assert lib.tdb_moe_dispatch(None, 64, 0, 2, 64, None, None, 64, None) == 0  # no tokens


def test_grouped_refusals():
    lib = _lib()

    def gemm(lda=64, groups=2, ldc=32, rows=8, N=32, K=64, mode=0, bias=None, aux=None, ld_aux=0, aux_out=None, tile=0,
             a=A, dg=0):
        return lib.tdb_grouped_gemm(a, lda, A, dg, A, groups, A, ldc, rows, N, K, mode, bias, aux, ld_aux, aux_out, tile,
                                    None)
    for bad in (dict(groups=0), dict(groups=1025), dict(N=36, ldc=40), dict(K=60), dict(rows=-1), dict(N=0),
                dict(rows=2 ** 31 - 8), dict(N=2 ** 31 - 8, ldc=2 ** 31)):
        _refused(gemm(**bad), b"groups")
    for bad in (dict(lda=60), dict(lda=56), dict(ldc=28), dict(a=ODD), dict(mode=1, bias=ODD)):
        _refused(gemm(**bad), b"aligned")
    for bad in (dict(mode=1), dict(mode=3), dict(mode=4), dict(mode=2, dg=1), dict(mode=9)):
        _refused(gemm(**bad), b"mode")
    _refused(gemm(mode=2, aux_out=A, ld_aux=24), b"pre-activation")
    _refused(gemm(mode=3, dg=1), b"pre-activation")
    _refused(gemm(tile=64), b"tile")
    _refused(gemm(tile=16, dg=1), b"tile")
    _refused(gemm(tile=16, rows=17), b"tile")
    _refused(gemm(tile=16, N=2 ** 27, ldc=2 ** 27), b"tile")
    assert gemm(rows=0, a=None) == 0
    _refused(lib.tdb_grouped_weight_grad(A, 32, A, 64, A, 2, ODD, 8, 32, 64, 0, 0, None), b"aligned")
    _refused(lib.tdb_grouped_weight_grad(A, 28, A, 64, A, 2, A, 8, 32, 64, 0, 0, None), b"aligned")
    _refused(lib.tdb_grouped_weight_grad(A, 32, A, 64, A, 2, A, 8, 32, 64, 0, 32, None), b"tile")
    assert lib.tdb_grouped_weight_grad(None, 32, None, 64, None, 2, A, 0, 32, 64, 1, 0, None) == 0
    _refused(lib.tdb_grouped_bias_grad(A, 30, A, 2, A, 8, 32, 0, None), b"aligned")


def test_mx4_refusals():
    lib = _lib()
    _refused(lib.tdb_mx4_quantize(A, 64, 1, 8, 48, None, 0, A, A, None), b"multiple of 32")
    _refused(lib.tdb_mx4_quantize(A, 64, 2, 8, 64, A, 2, A, A, None), b"one matrix")
    _refused(lib.tdb_mx4_quantize(ODD, 64, 1, 8, 64, None, 0, A, A, None), b"aligned")
    _refused(lib.tdb_mx4_dequantize(A, A, 1, 8, 64, None, 0, A, 60, None), b"aligned")
    assert lib.tdb_mx4_quantize(None, 64, 1, 0, 64, None, 0, None, None, None) == 0

    def gemm(offsets=None, groups=1, ldc=32, rows=8, N=32, K=64, bias=None, tile=0, q=A):
        return lib.tdb_mx4_gemm(q, A, A, A, offsets, groups, A, ldc, rows, N, K, bias, tile, None)
    for bad in (dict(groups=2), dict(N=36), dict(K=48), dict(offsets=A, groups=1025), dict(rows=-1), dict(rows=2 ** 31 - 8)):
        _refused(gemm(**bad), b"groups")
    for bad in (dict(ldc=28), dict(q=ODD), dict(bias=ODD)):
        _refused(gemm(**bad), b"aligned")
    for bad in (dict(tile=64), dict(rows=64, tile=32), dict(offsets=A, groups=2, rows=8, tile=128),
                dict(offsets=A, groups=2, rows=100, tile=32)):
        _refused(gemm(**bad), b"tile")
    # 32-row scale blocks while the groups hold at most 32 rows on average
    assert lib.tdb_mx4_scale_bytes(1, 64, 256, 2) == (2 + 2) * 1024
    assert lib.tdb_mx4_scale_bytes(1, 65, 256, 2) == (0 + 2) * 1024
    assert lib.tdb_mx4_scale_bytes(3, 130, 300, 0) == 3 * 2 * 2 * 1024
    from tempname_dcu_b200.ops import mx4
    for rows in (0, 1, 31, 32, 33, 64, 65, 127, 128, 129, 5000):
        for k in (32, 256, 288):
            for groups, matrices in ((0, 1), (0, 3), (1, 1), (2, 1), (7, 1), (200, 1)):
                assert mx4.scale_bytes(rows, k, groups, matrices) == lib.tdb_mx4_scale_bytes(matrices, rows, k, groups)


def test_python_refusals_without_a_gpu():
    import torch
    from tempname_dcu_b200.ops import grouped, moe, mx4
    z, x = torch.zeros(4, 8), torch.zeros(4, 64, dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    w = torch.zeros(2, 32, 64, dtype=torch.bfloat16)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    flat = torch.zeros(8, dtype=torch.int32)
    r = moe.Routing(ids=ids, weights=torch.zeros(4, 2), offsets=torch.zeros(9, dtype=torch.int32), order=flat, slots=flat)
    assert (r.tokens, r.top_k, r.experts) == (4, 2, 8)
    for call in (lambda: moe.route(z, 2), lambda: moe.dispatch(x, r), lambda: moe.combine(x, r),
                 lambda: moe.route_bwd(z, r, torch.zeros(4, 2)), lambda: moe.combine_bwd(x, x, r),
                 lambda: grouped.linear(x, w, off), lambda: grouped.matmul_nt(x, w, off),
                 lambda: grouped.weight_grad(x, x, off), lambda: grouped.bias_grad(x, off), lambda: mx4.quantize(x),
                 lambda: mx4.dequantize(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            call()
    for bad in (dict(ids=ids.long()), dict(weights=torch.zeros(4, 3)), dict(slots=flat[:7]), dict(order=flat.float()),
                dict(offsets=torch.zeros(1, dtype=torch.int32)), dict(ids=ids.t())):
        with pytest.raises(ValueError):
            moe.Routing(**dict(dict(ids=ids, weights=torch.zeros(4, 2), offsets=off, order=flat, slots=flat), **bad))
    for call in (lambda: moe.route(logits=z, top_k=2), lambda: mx4.quantize(x=x)):  # by keyword: the same refusals
        with pytest.raises(ValueError):
            call()
    assert r == r and r != moe.Routing(ids=ids, weights=torch.zeros(4, 2), offsets=off, order=flat, slots=flat)
    with pytest.raises(Exception):
        r.ids = None  # frozen: the checks hold for its life
