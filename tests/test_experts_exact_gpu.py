"""Sums of the grouped and 4-bit products with nothing to round: operands of 1
and -1, whose sums are whole numbers that fp32 holds.  One row or value lost or
taken twice, at the border of a tile, of a chain or of a block's share, changes
a result by 1 or 2, and fp32 outputs have to be equal.  bf16 outputs have to be
the rounding of the whole number; below 256 they hold it.

Random operands measure the fp32 gradients' error by its relative 2-norm.  The
tensor cores truncate when they add to their accumulator, once for 16 rows.  In
a chain of 512 rows the j-th of 32 running sums is sqrt(j / 32) of the last; an
addition loses 0.36 x 2^-23 of it on average (half a unit in the last place,
which is between 2^-24 and 2^-23 of the value), together 21.7 x 0.36 x 2^-23 =
9.3e-7 if all have one sign.  Chains are joined rounding to nearest and their
errors are independent, so the bound 2^-20 holds for any number of rows.  One
chain of all 8192 rows would be 4.4e-6 off.
"""
import pytest

pytestmark = pytest.mark.gpu


def _signs(*shape):
    import torch
    return (torch.randint(0, 2, shape, device="cuda") * 2 - 1).to(torch.bfloat16)


def _offsets(counts, start=0):
    import torch
    bounds = [start]
    for n in counts:
        bounds.append(bounds[-1] + n)
    return torch.tensor(bounds, dtype=torch.int32, device="cuda"), list(zip(bounds, bounds[1:]))


GROUPS = [[1027], [5000, 3, 0, 1], [0, 0, 3500], [64, 8128], [1100] * 5, [513, 511, 1536, 16, 15, 17], [100000]]


@pytest.mark.parametrize("tile", [0, 128, 512])
@pytest.mark.parametrize("counts", GROUPS, ids=str)
@pytest.mark.parametrize("N,K", [(64, 64), (520, 136), (264, 512)])
def test_weight_and_bias_gradient(cuda, N, K, counts, tile):
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(N + len(counts))
    off, spans = _offsets(counts, start=3)
    rows = sum(counts) + 7
    dy, x = _signs(rows, N), _signs(rows, K)
    exact = torch.stack([dy[a:b].double().t() @ x[a:b].double() for a, b in spans])
    base = torch.randint(-50, 50, (len(counts), N, K), device=cuda).float()
    acc = base.clone()
    assert torch.equal(grouped.weight_grad(dy, x, off, tile=tile).double(), exact)
    grouped.weight_grad(dy, x, off, acc, accumulate=True, tile=tile)
    assert torch.equal(acc.double(), exact + base.double())
    if tile == 0:
        exact = torch.stack([dy[a:b].double().sum(0) for a, b in spans])
        assert torch.equal(grouped.bias_grad(dy, off).double(), exact)


@pytest.mark.parametrize("tile", [0, 128, 512])
@pytest.mark.parametrize("counts", [[512], [8192], [64, 8128], [1170] * 7, [16384, 1, 4000], [100000]], ids=str)
def test_error_of_the_weight_gradient(cuda, counts, tile):
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(len(counts))
    off, spans = _offsets(counts)
    dy, x = (torch.randn(sum(counts), n, device=cuda).to(torch.bfloat16) for n in (264, 136))
    got = grouped.weight_grad(dy, x, off, tile=tile)
    db = grouped.bias_grad(dy, off)
    for g, (a, b) in enumerate(spans):
        exact = dy[a:b].double().t() @ x[a:b].double()
        assert (got[g].double() - exact).norm() <= 2.0 ** -20 * exact.norm()
        # the bias: a thread adds at most b - a over 256 values in a row, rounding to nearest, then 40 joins:
        # independent errors of half a step, sqrt(n) 2^-24 in all
        exact = dy[a:b].double().sum(0)
        assert (db[g].double() - exact).norm() <= 2.0 ** -24 * ((b - a) / 32 + 40) ** 0.5 * exact.norm() + 1e-12


@pytest.mark.parametrize("tile", [0, 32, 128, 512])
@pytest.mark.parametrize("counts", [[17], [40, 0, 3, 129], [100, 260], [1] * 20, [300] * 3, [33, 255, 257]], ids=str)
@pytest.mark.parametrize("width,terms", [(72, 512), (264, 1032), (136, 4104), (72, 8192), (264, 16384)])
def test_products(cuda, width, terms, counts, tile):
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(terms + len(counts))
    off, spans = _offsets(counts, start=1)
    x, w = _signs(sum(counts) + 4, terms), _signs(len(counts), width, terms)
    rows = slice(1, 1 + sum(counts))
    exact = torch.cat([x[a:b].double() @ w[g].double().t() for g, (a, b) in enumerate(spans)]).to(torch.bfloat16)
    assert torch.equal(grouped.linear(x, w, off, tile=tile)[rows], exact)
    assert torch.equal(grouped.matmul_nt(x, w.transpose(1, 2).contiguous(), off, tile=tile)[rows], exact)


@pytest.mark.parametrize("counts", [[1], [9, 0, 7], [1] * 16, [3, 0, 0, 4, 5]], ids=str)
@pytest.mark.parametrize("N,K", [(24, 40), (264, 1032), (512, 4096), (40, 16384)])
def test_few_rows(cuda, N, K, counts):
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(N + K)
    off, spans = _offsets(counts)
    x, w = _signs(sum(counts), K), _signs(len(counts), N, K)
    exact = torch.cat([x[a:b].double() @ w[g].double().t() for g, (a, b) in enumerate(spans)]).to(torch.bfloat16)
    for tile in (0, 16, 32):
        assert torch.equal(grouped.linear(x, w, off, tile=tile), exact)


@pytest.mark.parametrize("counts", [[1], [0, 140, 0], [40, 0, 1, 70], [9] * 12, [600, 33]], ids=str)
@pytest.mark.parametrize("N,K", [(136, 2048), (64, 2592), (264, 8192), (520, 288)])
def test_4_bit_products(cuda, N, K, counts):
    """1 and -1 times a power of two that differs from row to row: 4 bits hold them."""
    import torch
    from tempname_dcu_b200.ops import mx4
    torch.manual_seed(N + K)
    off, spans = _offsets(counts)
    power = torch.exp2(torch.randint(-3, 4, (sum(counts), 1), device=cuda)).to(torch.bfloat16)
    x, w = _signs(sum(counts), K) * power, _signs(len(counts), N, K)
    exact = torch.cat([x[a:b].double() @ w[g].double().t() for g, (a, b) in enumerate(spans)]).to(torch.bfloat16)
    qw, sfw = mx4.quantize(w)
    q, sf = mx4.quantize(x, offsets=off)
    assert torch.equal(mx4.dequantize(q, sf, offsets=off), x) and torch.equal(mx4.dequantize(qw, sfw), w)
    assert torch.equal(mx4.grouped_linear(q, sf, qw, sfw, off), exact)
    dense = (x.double() @ w[0].double().t()).to(torch.bfloat16)
    assert torch.equal(mx4.linear(*mx4.quantize(x), *mx4.quantize(w[0])), dense)
