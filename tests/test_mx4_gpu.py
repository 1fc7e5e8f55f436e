"""Microscaled 4-bit values and products (csrc/mx4.cu) against their
definitions in 64 bits: the quantizer value for value, the products within the
fp32 accumulation (products of two such values are exact in fp32; the sum of n
of them is off by less than n 2^-22 of the sum of their magnitudes) and half a
bf16 step.
"""
import pytest

pytestmark = pytest.mark.gpu


def _values(x):
    """The 4-bit values of x (float64): nearest grid point, ties to the even code."""
    import torch
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -127.0)
    for _ in range(300):  # the smallest e >= -127 with top / 2^e <= 6
        e = torch.where(torch.isfinite(top) & (top * torch.exp2(-e) > 6), e + 1, e)
    scale = torch.exp2(e)
    size = b.abs() / scale
    code = torch.zeros_like(size, dtype=torch.int64)
    for c in range(1, 8):
        middle = 0.5 * (grid[c - 1] + grid[c])
        code += (size >= middle if c % 2 == 0 else size > middle).long()
    out = torch.copysign(grid[code.clamp(max=7)] * scale, b)
    out = torch.where(torch.isfinite(b).all(-1, keepdim=True), out, torch.full_like(out, float("nan")))
    return out.reshape(x.shape)


def _status_ok():
    from tempname_dcu_b200.ops import native
    assert native.read_status() == [0, 0, 0, 0]


def _same(a, b):
    import torch
    return torch.equal(torch.nan_to_num(a.double(), nan=1e30), torch.nan_to_num(b.double(), nan=1e30))


@pytest.mark.parametrize("rows,K", [(1, 32), (3, 64), (128, 256), (130, 288), (257, 1056), (31, 4096)])
def test_quantize_and_back(cuda, rows, K):
    import torch
    from tempname_dcu_b200.ops import mx4
    torch.manual_seed(rows + K)
    x = (torch.randn(rows, K, device=cuda) * torch.logspace(-20, 20, K, device=cuda)).to(torch.bfloat16)
    x[0, :32] = 0
    assert _same(mx4.dequantize(*mx4.quantize(x)), _values(x))
    wide = torch.full((rows, K + 24), 7.0, device=cuda, dtype=torch.bfloat16)
    wide[:, 8:8 + K] = x
    q, sf = mx4.quantize(wide[:, 8:8 + K])
    out = torch.full((rows, K + 8), 9.0, device=cuda, dtype=torch.bfloat16)
    mx4.dequantize(q, sf, out=out[:, :K])
    assert _same(out[:, :K], _values(x)) and (out[:, K:] == 9).all()
    _status_ok()


def test_every_tie_sign_and_extreme(cuda):
    """Blocks that hold every bf16 between 0 and 6 times a scale, at scales
    from the smallest to the largest; subnormals, infinities and NaN."""
    import torch
    from tempname_dcu_b200.ops import mx4
    bits = torch.arange(0, 0x40c1, dtype=torch.int32, device=cuda).to(torch.int16).view(torch.bfloat16)  # 0 .. 6.0
    pad = -(-bits.numel() // 31) * 31 - bits.numel()
    body = torch.cat([bits, bits[:pad]]).view(-1, 31)
    body = torch.cat([torch.full_like(body[:, :1], 6.0), body], 1)  # the block's maximum: scale 1
    body[:, 1::2] *= -1
    for e in (0, -124, 125, 7):
        x = (body.double() * 2.0 ** e).to(torch.bfloat16)
        assert _same(mx4.dequantize(*mx4.quantize(x)), _values(x)), e
    x = bits.view(-1)[: 0x40c0].view(-1, 32)  # every block has its own scale, subnormals among them
    assert _same(mx4.dequantize(*mx4.quantize(x)), _values(x))
    x = torch.randn(4, 96, device=cuda).to(torch.bfloat16)
    x[1, 40], x[2, 0], x[3, 95] = float("inf"), float("nan"), -float("inf")
    got = mx4.dequantize(*mx4.quantize(x))
    assert _same(got, _values(x)) and got.isnan().sum() == 96
    x = torch.full((2, 32), torch.finfo(torch.bfloat16).max, device=cuda, dtype=torch.bfloat16)
    # (2 - 2^-7) 2^127 / 2^126 = 3.984 rounds to 4: the format's value is 4 * 2^126 = 2^128, which lies above
    # the largest bf16 (and fp32); its bf16 rounding is the infinity
    assert (_values(x) == 2.0 ** 128).all()
    assert _same(mx4.dequantize(*mx4.quantize(x)), _values(x).to(torch.bfloat16))
    _status_ok()


def test_quantize_matrices_and_groups(cuda):
    import torch
    from tempname_dcu_b200.ops import mx4
    torch.manual_seed(1)
    w = torch.randn(3, 200, 96, device=cuda).to(torch.bfloat16)
    assert _same(mx4.dequantize(*mx4.quantize(w)), _values(w))
    off = torch.tensor([4, 4, 133, 134, 134, 300], dtype=torch.int32, device=cuda)
    x = torch.randn(310, 320, device=cuda).to(torch.bfloat16)
    q, sf = mx4.quantize(x, offsets=off, q=torch.full((310, 160), 0x77, device=cuda, dtype=torch.uint8))
    assert (q[:4] == 0x77).all() and (q[300:] == 0x77).all()
    out = torch.full((310, 320), 5.0, device=cuda, dtype=torch.bfloat16)
    mx4.dequantize(q, sf, offsets=off, out=out)
    assert _same(out[4:300], _values(x[4:300])) and (out[:4] == 5).all() and (out[300:] == 5).all()
    assert mx4.dequantize(*mx4.quantize(x[:0])).shape == (0, 320)
    _status_ok()


def _within(got, exact, size, terms):
    return ((got.double() - exact).abs() <= exact.abs() * 2.0 ** -8 + size * terms * 2.0 ** -22).all()


@pytest.mark.parametrize("tile", [0, 128, 512])
@pytest.mark.parametrize("M,N,K", [(1, 8, 32), (7, 64, 64), (128, 128, 256), (129, 264, 288), (300, 520, 1056),
                                   (512, 1024, 4096), (700, 72, 2080)])
def test_linear(cuda, M, N, K, tile):
    import torch
    from tempname_dcu_b200.ops import mx4
    torch.manual_seed(M + N + K)
    # scales that differ from block to block and row to row
    x = (torch.randn(M, K, device=cuda) * torch.exp2(torch.randint(-4, 5, (M, K // 32), device=cuda))
         .repeat_interleave(32, 1)).to(torch.bfloat16)
    w = (torch.randn(N, K, device=cuda) * torch.exp2(torch.randint(-4, 5, (N, K // 32), device=cuda))
         .repeat_interleave(32, 1)).to(torch.bfloat16)
    b = torch.randn(N, device=cuda).to(torch.bfloat16)
    xv, wv = _values(x), _values(w)
    exact, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    qx, sfx = mx4.quantize(x)
    qw, sfw = mx4.quantize(w)
    assert _within(mx4.linear(qx, sfx, qw, sfw, tile=tile), exact, size, K)
    out = torch.full((M, N + 8), 7.0, device=cuda, dtype=torch.bfloat16)
    mx4.linear(qx, sfx, qw, sfw, bias=b, out=out[:, :N], tile=tile)
    assert _within(out[:, :N], exact + b.double(), size + b.double().abs(), K) and (out[:, N:] == 7).all()
    _status_ok()


@pytest.mark.parametrize("tile", [0, 128, 512])
@pytest.mark.parametrize("counts", [[130], [0, 103, 0], [130, 0, 257, 64, 1, 0, 77], [256, 128, 384], [31, 33, 513, 127]])
@pytest.mark.parametrize("N,K", [(64, 64), (264, 320), (520, 1056)])
def test_grouped_linear(cuda, counts, N, K, tile):
    import torch
    from tempname_dcu_b200.ops import mx4
    torch.manual_seed(N + K)
    lead, R, G = 5, sum(counts) + 11, len(counts)
    bounds = [lead]
    for n in counts:
        bounds.append(bounds[-1] + n)
    off = torch.tensor(bounds, dtype=torch.int32, device=cuda)
    x = torch.randn(R, K, device=cuda).to(torch.bfloat16)
    x[:lead] = float("nan")
    x[bounds[-1]:] = float("inf")
    w = (torch.randn(G, N, K, device=cuda) * 0.02).to(torch.bfloat16)
    b = torch.randn(G, N, device=cuda).to(torch.bfloat16)
    xv, wv = _values(x), _values(w)
    qx, sfx = mx4.quantize(x, offsets=off)
    qw, sfw = mx4.quantize(w)
    out = torch.full((R, N), 7.0, device=cuda, dtype=torch.bfloat16)
    mx4.grouped_linear(qx, sfx, qw, sfw, off, bias=b, out=out, tile=tile)
    for g in range(G):
        lo, hi = bounds[g], bounds[g + 1]
        exact = xv[lo:hi] @ wv[g].t() + b[g].double()
        assert _within(out[lo:hi], exact, xv[lo:hi].abs() @ wv[g].abs().t() + b[g].double().abs(), K)
    assert (out[:lead] == 7).all() and (out[bounds[-1]:] == 7).all()
    _status_ok()


@pytest.mark.parametrize("counts", [[1], [0, 3, 0], [40, 0, 1, 70, 0, 9], [0] * 60 + [200] + [1] * 9, [32, 33, 31, 0]])
@pytest.mark.parametrize("N,K", [(8, 32), (264, 320), (520, 1056)])
def test_grouped_linear_with_small_groups(cuda, counts, N, K):
    """At most 32 rows per group on average: scale blocks and tiles of 32 rows."""
    import torch
    from tempname_dcu_b200.ops import mx4, native
    torch.manual_seed(N + K)
    lead, G = 2, len(counts)
    R = sum(counts) + lead
    bounds = [lead]
    for n in counts:
        bounds.append(bounds[-1] + n)
    assert native.lib().tdb_mx4_pick_tile(R, G, N) == (32 if R <= 32 * G else 128)
    off = torch.tensor(bounds, dtype=torch.int32, device=cuda)
    x = torch.randn(R, K, device=cuda).to(torch.bfloat16)
    x[:lead] = float("nan")
    w = (torch.randn(G, N, K, device=cuda) * 0.02).to(torch.bfloat16)
    xv, wv = _values(x), _values(w)
    qx, sfx = mx4.quantize(x, offsets=off)
    assert _same(mx4.dequantize(qx, sfx, offsets=off)[lead:], xv[lead:])
    qw, sfw = mx4.quantize(w)
    out = torch.full((R, N), 7.0, device=cuda, dtype=torch.bfloat16)
    mx4.grouped_linear(qx, sfx, qw, sfw, off, out=out)
    for g in range(G):
        lo, hi = bounds[g], bounds[g + 1]
        assert _within(out[lo:hi], xv[lo:hi] @ wv[g].t(), xv[lo:hi].abs() @ wv[g].abs().t(), K)
    assert (out[:lead] == 7).all()
    _status_ok()


@pytest.mark.parametrize("counts", [[1], [0, 140, 0], [40, 0, 1, 70], [9] * 12])
@pytest.mark.parametrize("K", [2048, 2592, 8192])
def test_long_sums_of_few_tiles(cuda, counts, K):
    """Tiles whose summed values several blocks share."""
    import torch
    from tempname_dcu_b200.ops import mx4
    torch.manual_seed(K)
    G, N, R = len(counts), 136, sum(counts)
    bounds = [sum(counts[:g]) for g in range(G + 1)]
    off = torch.tensor(bounds, dtype=torch.int32, device=cuda)
    x = torch.randn(R, K, device=cuda).to(torch.bfloat16)
    w = (torch.randn(G, N, K, device=cuda) * 0.02).to(torch.bfloat16)
    b = torch.randn(G, N, device=cuda).to(torch.bfloat16)
    xv, wv = _values(x), _values(w)
    qw, sfw = mx4.quantize(w)
    out = mx4.grouped_linear(*mx4.quantize(x, offsets=off), qw, sfw, off, bias=b)
    for g in range(G):
        lo, hi = bounds[g], bounds[g + 1]
        assert _within(out[lo:hi], xv[lo:hi] @ wv[g].t() + b[g].double(),
                       xv[lo:hi].abs() @ wv[g].abs().t() + b[g].double().abs(), K)
    y = mx4.linear(*mx4.quantize(x), *mx4.quantize(w[0]))
    assert _within(y, xv @ wv[0].t(), xv.abs() @ wv[0].abs().t(), K)
    assert torch.equal(y, mx4.linear(*mx4.quantize(x), *mx4.quantize(w[0])))
    _status_ok()


def test_nan_stays_in_its_row(cuda):
    import torch
    from tempname_dcu_b200.ops import mx4
    torch.manual_seed(4)
    x = torch.randn(200, 512, device=cuda).to(torch.bfloat16)
    x[17, 300] = float("nan")
    w = torch.randn(136, 512, device=cuda).to(torch.bfloat16)
    qw, sfw = mx4.quantize(w)
    y = mx4.linear(*mx4.quantize(x), qw, sfw)
    assert y[17].isnan().all()
    keep = torch.arange(200, device=cuda) != 17
    assert not y[keep].isnan().any()
    _status_ok()


def test_captured_and_replayed(cuda):
    import torch
    from tempname_dcu_b200.ops import mx4
    torch.manual_seed(6)
    off = torch.tensor([0, 40, 40, 100], dtype=torch.int32, device=cuda)
    x = torch.randn(100, 256, device=cuda).to(torch.bfloat16)
    qw, sfw = mx4.quantize(torch.randn(3, 136, 256, device=cuda).to(torch.bfloat16))

    def step():
        return mx4.grouped_linear(*mx4.quantize(x, offsets=off), qw, sfw, off)
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    x.copy_(torch.randn(100, 256, device=cuda))
    off.copy_(torch.tensor([0, 3, 90, 100], dtype=torch.int32, device=cuda))
    g.replay()
    assert torch.equal(captured, step())
    _status_ok()


def test_refusals(cuda):
    import torch
    from tempname_dcu_b200.ops import mx4, native
    x = torch.randn(8, 64, device=cuda).to(torch.bfloat16)
    w = torch.randn(2, 32, 64, device=cuda).to(torch.bfloat16)
    off = torch.tensor([0, 3, 8], dtype=torch.int32, device=cuda)
    q, sf = mx4.quantize(x)
    qw, sfw = mx4.quantize(w)
    for call in (lambda: mx4.quantize(x.float()), lambda: mx4.quantize(x[:, :48]), lambda: mx4.quantize(x.t()),
                 lambda: mx4.quantize(x.cpu()), lambda: mx4.quantize(w, offsets=off), lambda: mx4.quantize(w[:, :16]),
                 lambda: mx4.quantize(x, sf=sf[:512]), lambda: mx4.quantize(x, offsets=off.long()),
                 lambda: mx4.dequantize(q, sf[:512]), lambda: mx4.dequantize(q, sf, out=x[:, :32]),
                 lambda: mx4.linear(q, sf, qw, sfw), lambda: mx4.linear(q, sf, qw[0], sfw, bias=x[0]),
                 lambda: mx4.linear(q, sf, qw[0, :, :16].contiguous(), sfw),
                 lambda: mx4.linear(q, sf, qw[0, :20].contiguous(), sfw),
                 lambda: mx4.grouped_linear(q, sf, qw, sfw, off[:2]),
                 lambda: mx4.grouped_linear(q, sf, qw, sfw, None),
                 lambda: mx4.linear(q, sf, qw[0], sfw, out=x)):
        with pytest.raises((ValueError, TypeError)):
            call()
    with pytest.raises(native.NativeError):  # scale blocks of 32 rows go with tiles of 32 rows
        mx4.grouped_linear(*mx4.quantize(x, offsets=off), qw, sfw, off, tile=128)
    with pytest.raises(native.NativeError):
        mx4.linear(*mx4.quantize(torch.cat([x] * 5)), qw[0].contiguous(), sfw, tile=32)
    native.clear_status()
    mx4.quantize(x, offsets=torch.tensor([0, 9, 8], dtype=torch.int32, device=cuda))
    with pytest.raises(native.NativeError):
        native.raise_on_status()
    _status_ok()
