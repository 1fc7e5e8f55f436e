"""Products grouped by expert (csrc/grouped.cu) against plain products in 64
bits.

Tolerances: a bf16 product is exact in fp32 and the sum of n of them in fp32 is
off by less than n 2^-23 of the sum of their magnitudes, here taken as
n 2^-24 * 4 because the tensor cores may truncate; a bf16 output adds half a
step, 2^-8 relative.
"""
import pytest

pytestmark = pytest.mark.gpu

SIZES = {
    "one_row": [1], "single_empty": [0, 0, 5, 0], "few": [3, 0, 1, 2], "ragged": [130, 0, 257, 64, 1, 0, 77],
    "full_tiles": [256, 128, 384], "tail_rows": [31, 33, 65, 127, 129, 255, 1], "big": [700, 1, 0, 1300],
}
SHAPES = [(8, 8), (64, 64), (264, 200), (512, 264), (1032, 72)]


def _offsets(sizes, device, start=0):
    import torch
    return torch.tensor([start] + [start + sum(sizes[:i + 1]) for i in range(len(sizes))], dtype=torch.int32,
                        device=device)


def _bf(*shape, device, scale=1.0):
    import torch
    return (torch.randn(*shape, device=device) * scale).to(torch.bfloat16)


def _within(got, exact, size, terms, half_step=2.0 ** -8):
    err = (got.double() - exact).abs()
    return (err <= exact.abs() * half_step + size * terms * 2.0 ** -22).all()


def _status_ok():
    from tempname_dcu_b200.ops import native
    assert native.read_status() == [0, 0, 0, 0]


@pytest.mark.parametrize("tile", [0, 32, 128, 512])
@pytest.mark.parametrize("N,K", SHAPES)
@pytest.mark.parametrize("sizes", list(SIZES))
def test_linear(cuda, sizes, N, K, tile):
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(N + K)
    counts = SIZES[sizes]
    R, G = sum(counts), len(counts)
    off = _offsets(counts, cuda)
    x, w, b = _bf(R, K, device=cuda), _bf(G, N, K, device=cuda, scale=0.1), _bf(G, N, device=cuda)
    group = torch.repeat_interleave(torch.arange(G, device=cuda), torch.tensor(counts, device=cuda))
    exact = torch.einsum("rk,rnk->rn", x.double(), w.double()[group]) if R * N * K < 2e7 else \
        torch.cat([x[a:c].double() @ w[g].double().t() for g, (a, c) in enumerate(zip(off.tolist(), off.tolist()[1:]))])
    size = torch.cat([x[a:c].double().abs() @ w[g].double().abs().t()
                      for g, (a, c) in enumerate(zip(off.tolist(), off.tolist()[1:]))])
    assert _within(grouped.linear(x, w, off, tile=tile), exact, size, K)
    z = exact + b.double()[group]
    zs = size + b.double().abs()[group]
    assert _within(grouped.linear(x, w, off, b, tile=tile), z, zs, K)
    h, pre = grouped.linear_gelu(x, w, off, b, tile=tile)
    assert _within(pre, z, zs, K)
    gelu = 0.5 * z * torch.erfc(-z / 2 ** 0.5)
    # |gelu'| < 1.13; the distribution function is off by less than 1.5e-7 / 2 (its approximation) + 2^-22, times z
    assert ((h.double() - gelu).abs() <= gelu.abs() * 2.0 ** -8 + 1.2 * zs * K * 2.0 ** -22 + z.abs() * 4e-7).all()
    _status_ok()


@pytest.mark.parametrize("tile", [0, 32, 128, 512])
@pytest.mark.parametrize("N,K", SHAPES)
@pytest.mark.parametrize("sizes", list(SIZES))
def test_data_gradient(cuda, sizes, N, K, tile):
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(N * K)
    counts = SIZES[sizes]
    R, G = sum(counts), len(counts)
    off = _offsets(counts, cuda)
    spans = list(zip(off.tolist(), off.tolist()[1:]))
    dy, w, pre = _bf(R, N, device=cuda), _bf(G, N, K, device=cuda, scale=0.1), _bf(R, K, device=cuda)
    exact = torch.cat([dy[a:c].double() @ w[g].double() for g, (a, c) in enumerate(spans)])
    size = torch.cat([dy[a:c].double().abs() @ w[g].double().abs() for g, (a, c) in enumerate(spans)])
    assert _within(grouped.matmul_nt(dy, w, off, tile=tile), exact, size, N)
    z = pre.double()
    slope = 0.5 * torch.erfc(-z / 2 ** 0.5) + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    got = grouped.matmul_nt(dy, w, off, gelu_pre=pre, tile=tile)
    # the slope in fp32: its terms are below 1.2, each within 2^-20
    assert ((got.double() - exact * slope).abs() <=
            (exact * slope).abs() * 2.0 ** -8 + 1.2 * size * N * 2.0 ** -22 + exact.abs() * 2.0 ** -19).all()
    _status_ok()


@pytest.mark.parametrize("tile", [0, 128, 512])
@pytest.mark.parametrize("N,K", SHAPES)
@pytest.mark.parametrize("sizes", list(SIZES))
def test_weight_and_bias_gradient(cuda, sizes, N, K, tile):
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(N - K)
    counts = SIZES[sizes]
    R, G = sum(counts), len(counts)
    off = _offsets(counts, cuda)
    spans = list(zip(off.tolist(), off.tolist()[1:]))
    dy, x = _bf(R, N, device=cuda), _bf(R, K, device=cuda)
    exact = torch.stack([dy[a:c].double().t() @ x[a:c].double() for a, c in spans])
    size = torch.stack([dy[a:c].double().abs().t() @ x[a:c].double().abs() for a, c in spans])
    terms = max(max(counts), 1)
    base = torch.randn(G, N, K, device=cuda)
    acc = base.clone()
    grouped.weight_grad(dy, x, off, acc, accumulate=True, tile=tile)
    assert _within(acc, exact + base.double(), size + base.double().abs(), terms, 2.0 ** -24)
    fresh = torch.full((G, N, K), float("nan"), device=cuda)
    grouped.weight_grad(dy, x, off, fresh, accumulate=False, tile=tile)
    assert _within(fresh, exact, size, terms, 2.0 ** -24)
    assert torch.equal(fresh, grouped.weight_grad(dy, x, off, tile=tile))
    for g, n in enumerate(counts):
        if n == 0:
            assert torch.equal(acc[g], base[g]) and (fresh[g] == 0).all()
    db = grouped.bias_grad(dy, off)
    bias_exact = torch.stack([dy[a:c].double().sum(0) for a, c in spans])
    bias_size = torch.stack([dy[a:c].double().abs().sum(0) for a, c in spans])
    assert _within(db, bias_exact, bias_size, terms, 2.0 ** -24)
    again = db.clone()
    grouped.bias_grad(dy, off, again, accumulate=True)
    assert torch.equal(again, db + db)
    _status_ok()


@pytest.mark.parametrize("tile", [32, 128, 512])
def test_foreign_rows_hold_nan_and_stay_as_they_were(cuda, tile):
    """Rows before the first and behind the last group, and rows of other
    groups, are full of NaN and infinities; strided operands and outputs."""
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(11)
    counts, lead, trail = [5, 70, 0, 300], 3, 40
    R, G, N, K = lead + sum(counts) + trail, 4, 264, 136
    off = _offsets(counts, cuda, start=lead)
    wide_x, wide_dy = _bf(R, K + 24, device=cuda), _bf(R, N + 8, device=cuda)
    x, dy = wide_x[:, 16:16 + K], wide_dy[:, :N]
    w = _bf(G, N, K, device=cuda, scale=0.1)
    for t in (wide_x, wide_dy):
        t[:lead] = float("nan")
        t[R - trail:] = float("inf")
    for g in (1, 3):  # one group at a time is finite
        lo, hi = off[g].item(), off[g + 1].item()
        xs, dys = x.clone(), dy.clone()
        only = torch.zeros(R, dtype=torch.bool, device=cuda)
        only[lo:hi] = True
        xs[~only] = float("nan")
        dys[~only] = float("nan")
        out = torch.full((R, N + 8), 7.0, device=cuda, dtype=torch.bfloat16)
        grouped.linear(xs, w, off, out=out[:, :N], tile=tile)
        exact = xs[lo:hi].double() @ w[g].double().t()
        size = xs[lo:hi].double().abs() @ w[g].double().abs().t()
        assert _within(out[lo:hi, :N], exact, size, K)
        assert (out[:lead] == 7).all() and (out[R - trail:] == 7).all() and (out[:, N:] == 7).all()
        dx = torch.full((R, K), 7.0, device=cuda, dtype=torch.bfloat16)
        grouped.matmul_nt(dys, w, off, out=dx, tile=tile)
        assert _within(dx[lo:hi], dys[lo:hi].double() @ w[g].double(),
                       dys[lo:hi].double().abs() @ w[g].double().abs(), N)
        assert (dx[:lead] == 7).all() and (dx[R - trail:] == 7).all()
        dw = grouped.weight_grad(dys, xs, off, tile=max(tile, 128))
        assert _within(dw[g], dys[lo:hi].double().t() @ xs[lo:hi].double(),
                       dys[lo:hi].double().abs().t() @ xs[lo:hi].double().abs(), hi - lo, 2.0 ** -24)
        assert (dw[2] == 0).all()
    _status_ok()


@pytest.mark.parametrize("counts", [[1], [0, 2, 0], [1] * 16, [0, 16], [9, 0, 7], [3, 0, 0, 4, 5], [0] * 70 + [2, 0, 1]])
@pytest.mark.parametrize("N,K", [(8, 8), (24, 40), (264, 1032), (512, 4096)])
def test_few_rows(cuda, counts, N, K):
    """At most 16 rows: the streaming kernel, with rows outside the groups and strided operands."""
    import torch
    from tempname_dcu_b200.ops import grouped, native
    torch.manual_seed(len(counts) + N)
    used, G = sum(counts), len(counts)
    lead = min(1, 16 - used)
    R = 16
    off = _offsets(counts, cuda, start=lead)
    wide = _bf(R, K + 8, device=cuda)
    wide[:lead] = float("nan")
    wide[lead + used:] = float("inf")
    x = wide[:, :K]
    w, b = _bf(G, N, K, device=cuda, scale=0.1), _bf(G, N, device=cuda)
    assert native.lib().tdb_grouped_pick_tile(0, R, G, 0, N) == 16 or G * N > 8000
    out = torch.full((R, N + 16), 7.0, device=cuda, dtype=torch.bfloat16)
    grouped.linear(x, w, off, out=out[:, :N], tile=16)
    h, z = torch.full_like(out, 7.0)[:, :N], torch.full_like(out, 7.0)[:, :N]
    grouped.linear_gelu(x, w, off, b, pre_out=z, out=h, tile=16)
    group = torch.repeat_interleave(torch.arange(G, device=cuda), torch.tensor(counts, device=cuda))
    rows = slice(lead, lead + used)
    exact = torch.einsum("rk,rnk->rn", x[rows].double(), w.double()[group])
    size = torch.einsum("rk,rnk->rn", x[rows].double().abs(), w.double().abs()[group])
    assert _within(out[rows, :N], exact, size, K)
    ze, zs = exact + b.double()[group], size + b.double().abs()[group]
    assert _within(z[rows], ze, zs, K)
    gelu = 0.5 * ze * torch.erfc(-ze / 2 ** 0.5)
    # the approximation of the distribution function is off by less than 1.5e-7 / 2 + 2^-22 (times z)
    assert ((h[rows].double() - gelu).abs() <= gelu.abs() * 2.0 ** -8 + 1.2 * zs * K * 2.0 ** -22 + ze.abs() * 4e-7).all()
    for t in (out[:, :N], h, z):
        assert (t[:lead] == 7).all() and (t[lead + used:] == 7).all()
    assert (out[:, N:] == 7).all()
    assert torch.equal(grouped.linear(x, w, off, tile=16)[rows], out[rows, :N])
    _status_ok()


@pytest.mark.parametrize("tile", [0, 32, 128])
@pytest.mark.parametrize("counts", [[17], [40, 0, 3, 129], [100, 260], [1] * 20])
@pytest.mark.parametrize("terms", [512, 1000, 4104, 8192])
def test_long_sums_of_few_tiles(cuda, terms, counts, tile):
    """Tiles whose summed values several blocks share."""
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(terms)
    G, width = len(counts), 72
    off = _offsets(counts, cuda, start=2)
    R = sum(counts) + 5
    spans = list(zip(off.tolist(), off.tolist()[1:]))
    x = _bf(R, terms, device=cuda)
    x[:2] = float("nan")
    x[-3:] = float("inf")
    rows = slice(2, R - 3)
    w, b, pre = _bf(G, width, terms, device=cuda, scale=0.1), _bf(G, width, device=cuda), _bf(R, width, device=cuda)
    group = torch.repeat_interleave(torch.arange(G, device=cuda), torch.tensor(counts, device=cuda))
    exact = torch.cat([x[a:c].double() @ w[g].double().t() for g, (a, c) in enumerate(spans)])
    size = torch.cat([x[a:c].double().abs() @ w[g].double().abs().t() for g, (a, c) in enumerate(spans)])
    out = torch.full((R, width + 8), 7.0, device=cuda, dtype=torch.bfloat16)
    grouped.linear(x, w, off, out=out[:, :width], tile=tile)
    assert _within(out[rows, :width], exact, size, terms)
    assert (out[:2] == 7).all() and (out[-3:] == 7).all() and (out[:, width:] == 7).all()
    assert torch.equal(grouped.linear(x, w, off, tile=tile)[rows], out[rows, :width])
    z, zs = exact + b.double()[group], size + b.double().abs()[group]
    h, got = grouped.linear_gelu(x, w, off, b, tile=tile)
    assert _within(got[rows], z, zs, terms)
    gelu = 0.5 * z * torch.erfc(-z / 2 ** 0.5)
    # |gelu'| < 1.13; the distribution function is off by less than 1.5e-7 / 2 (its approximation) + 2^-22, times z
    assert ((h[rows].double() - gelu).abs() <= gelu.abs() * 2.0 ** -8 + 1.2 * zs * terms * 2.0 ** -22 + z.abs() * 4e-7).all()
    wt = w.transpose(1, 2).contiguous()  # [G, terms, width]: the gradient of x sums over its rows
    dx = torch.full((R, width), 7.0, device=cuda, dtype=torch.bfloat16)
    grouped.matmul_nt(x, wt, off, out=dx, tile=tile)
    assert _within(dx[rows], exact, size, terms)
    p = pre[rows].double()
    slope = 0.5 * torch.erfc(-p / 2 ** 0.5) + p * torch.exp(-p * p / 2) / (2 * torch.pi) ** 0.5
    grouped.matmul_nt(x, wt, off, gelu_pre=pre, out=dx, tile=tile)
    # the slope in fp32: its terms are below 1.2, each within 2^-20
    assert ((dx[rows].double() - exact * slope).abs() <=
            (exact * slope).abs() * 2.0 ** -8 + 1.2 * size * terms * 2.0 ** -22 + exact.abs() * 2.0 ** -19).all()
    assert (dx[:2] == 7).all() and (dx[-3:] == 7).all()
    _status_ok()


@pytest.mark.parametrize("tile", [0, 128])
@pytest.mark.parametrize("counts", [[1027], [5000, 3, 0, 1], [0, 0, 3500], [9, 4000], [1100] * 5, [64, 8128]])
@pytest.mark.parametrize("N,K", [(8, 8), (72, 264), (520, 136)])
def test_weight_gradient_of_few_tiles(cuda, N, K, counts, tile):
    """Tiles whose rows several blocks share, groups shorter than the shares too."""
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(N + len(counts))
    off = _offsets(counts, cuda, start=2)
    spans = list(zip(off.tolist(), off.tolist()[1:]))
    dy, x = _bf(sum(counts) + 5, N + 8, device=cuda)[:, :N], _bf(sum(counts) + 5, K + 8, device=cuda)[:, 8:]
    for t in (dy, x):
        t[:2] = float("nan")
        t[-3:] = float("inf")
    exact = torch.stack([dy[a:c].double().t() @ x[a:c].double() for a, c in spans])
    size = torch.stack([dy[a:c].double().abs().t() @ x[a:c].double().abs() for a, c in spans])
    base = torch.randn(len(counts), N, K, device=cuda)
    acc = base.clone()
    grouped.weight_grad(dy, x, off, acc, accumulate=True, tile=tile)
    assert _within(acc, exact + base.double(), size + base.double().abs(), max(counts), 2.0 ** -24)
    fresh = torch.full_like(base, float("nan"))
    grouped.weight_grad(dy, x, off, fresh, accumulate=False, tile=tile)
    assert _within(fresh, exact, size, max(counts), 2.0 ** -24)
    assert torch.equal(fresh, grouped.weight_grad(dy, x, off, tile=tile))
    for g, n in enumerate(counts):
        if n == 0:
            assert torch.equal(acc[g], base[g]) and (fresh[g] == 0).all()
    _status_ok()


def test_shared_sums_captured_on_two_streams(cuda):
    """Calls whose sums several blocks share, first made inside a capture; two graphs at once."""
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(8)
    off = _offsets([40, 0, 1500, 20], cuda)
    x, w = _bf(1560, 2056, device=cuda), _bf(4, 40, 2056, device=cuda, scale=0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for s in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = grouped.linear(x, w, off)
            outs.append((y, grouped.weight_grad(y, x, off), grouped.matmul_nt(y, w, off)))
        graphs.append(g)
    x.copy_(_bf(1560, 2056, device=cuda))
    off.copy_(_offsets([0, 1000, 60, 500], cuda))
    torch.cuda.synchronize()
    for s, g in zip(streams, graphs):
        with torch.cuda.stream(s):
            for _ in range(5):
                g.replay()
    torch.cuda.synchronize()
    y = grouped.linear(x, w, off)
    for got in outs:
        for have, want in zip(got, (y, grouped.weight_grad(y, x, off), grouped.matmul_nt(y, w, off))):
            assert torch.equal(have, want)
    spans = list(zip(off.tolist(), off.tolist()[1:]))
    exact = torch.cat([x[a:c].double() @ w[g].double().t() for g, (a, c) in enumerate(spans)])
    size = torch.cat([x[a:c].double().abs() @ w[g].double().abs().t() for g, (a, c) in enumerate(spans)])
    assert _within(y, exact, size, 2056)
    _status_ok()


@pytest.mark.parametrize("counts", [[5000, 3, 0, 1], [0, 0], [9, 4000], [130] * 40])
@pytest.mark.parametrize("N", [8, 72, 1000, 4096])
def test_bias_gradient_of_long_groups(cuda, counts, N):
    """Groups whose rows several blocks share, and outputs that need no sharing."""
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(N)
    off = _offsets(counts, cuda, start=2)
    dy = _bf(sum(counts) + 5, N + 8, device=cuda)[:, :N]
    dy[:2] = float("nan")
    dy[-3:] = float("inf")
    spans = list(zip(off.tolist(), off.tolist()[1:]))
    exact = torch.stack([dy[a:c].double().sum(0) for a, c in spans])
    size = torch.stack([dy[a:c].double().abs().sum(0) for a, c in spans])
    got = grouped.bias_grad(dy, off)
    assert _within(got, exact, size, max(max(counts), 1), 2.0 ** -24)
    again = got.clone()
    grouped.bias_grad(dy, off, again)
    assert torch.equal(again, got + got) and torch.equal(got, grouped.bias_grad(dy, off))
    _status_ok()


@pytest.mark.parametrize("tile", [16, 32, 128, 512])
def test_gelu_of_infinities_and_nan(cuda, tile):
    import torch
    from tempname_dcu_b200.ops import grouped
    off = _offsets([5, 7], cuda)
    x, w, b = _bf(12, 64, device=cuda), _bf(2, 32, 64, device=cuda), torch.zeros(2, 32, device=cuda, dtype=torch.bfloat16)
    b[1, 0], b[1, 1], b[1, 2], b[1, 3], b[1, 4] = float("inf"), -float("inf"), float("nan"), 1e20, -1e20
    h, z = grouped.linear_gelu(x, w, off, b, tile=tile)
    assert torch.isfinite(h[:5]).all() and torch.isfinite(h[5:, 3:]).all()
    assert (h[5:, 0] == float("inf")).all() and (h[5:, 1] == 0).all() and h[5:, 2].isnan().all()
    assert torch.equal(h[5:, 3], z[5:, 3]) and (h[5:, 4] == 0).all()


def test_many_groups_and_repeat_bitwise(cuda):
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(2)
    counts = [(i * 7) % 11 for i in range(1024)]
    R, G, N, K = sum(counts), 1024, 72, 40
    off = _offsets(counts, cuda)
    x, w = _bf(R, K, device=cuda), _bf(G, N, K, device=cuda)
    group = torch.repeat_interleave(torch.arange(G, device=cuda), torch.tensor(counts, device=cuda))
    exact = (w.double()[group] * x.double()[:, None]).sum(2)
    size = (w.double()[group] * x.double()[:, None]).abs().sum(2)
    y = grouped.linear(x, w, off)
    assert _within(y, exact, size, K)
    assert torch.equal(y, grouped.linear(x, w, off))
    _status_ok()


@pytest.mark.parametrize("call", ["linear", "data", "weight", "bias"])
def test_bad_offsets_are_reported(cuda, call):
    """Offsets are checked by the kernel before any row is addressed."""
    import torch
    from tempname_dcu_b200.ops import grouped, native
    x, w = _bf(64, 64, device=cuda), _bf(2, 64, 64, device=cuda)
    for values in ([0, 40, 65], [0, 50, 20], [-1, 10, 64]):
        native.clear_status()
        off = torch.tensor(values, dtype=torch.int32, device=cuda)
        if call == "linear":
            grouped.linear(x, w, off)
        elif call == "data":
            grouped.matmul_nt(x, w, off)
        elif call == "weight":
            grouped.weight_grad(x, x, off)
        else:
            grouped.bias_grad(x, off)
        with pytest.raises(native.NativeError):
            native.raise_on_status()
    _status_ok()


def test_no_rows(cuda):
    import torch
    from tempname_dcu_b200.ops import grouped
    off = torch.zeros(4, dtype=torch.int32, device=cuda)
    x, w = _bf(0, 64, device=cuda), _bf(3, 32, 64, device=cuda)
    assert grouped.linear(x, w, off).shape == (0, 32)
    assert (grouped.weight_grad(_bf(0, 32, device=cuda), x, off) == 0).all()
    assert (grouped.bias_grad(x, off) == 0).all()
    kept = torch.ones(3, 32, 64, device=cuda)
    grouped.weight_grad(_bf(0, 32, device=cuda), x, off, kept)
    assert (kept == 1).all()
    _status_ok()


def test_other_streams_and_graphs(cuda):
    import torch
    from tempname_dcu_b200.ops import grouped
    torch.manual_seed(9)
    counts = [40, 0, 200, 17]
    off = _offsets(counts, cuda)
    x, w, dy = _bf(257, 136, device=cuda), _bf(4, 264, 136, device=cuda), _bf(257, 264, device=cuda)

    def step():
        h, z = grouped.linear_gelu(x, w, off)
        return h, grouped.matmul_nt(dy, w, off), grouped.weight_grad(dy, x, off), grouped.bias_grad(dy, off)
    ref = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    # new sizes and rows on replay: the offsets are read on the device
    off.copy_(_offsets([0, 250, 3, 4], cuda))
    x.copy_(_bf(257, 136, device=cuda))
    g.replay()
    ref = step()
    assert all(torch.equal(a, b) for a, b in zip(ref, captured))
    _status_ok()


def test_refusals(cuda):
    import torch
    from tempname_dcu_b200.ops import grouped, native
    off = _offsets([3, 5], cuda)
    x, w = _bf(8, 64, device=cuda), _bf(2, 32, 64, device=cuda)
    grad = torch.zeros(2, 32, 64, device=cuda)
    dy = _bf(8, 32, device=cuda)
    for call in (lambda: grouped.linear(x.float(), w, off), lambda: grouped.linear(x, w.float(), off),
                 lambda: grouped.linear(x, w, off.long()), lambda: grouped.linear(x, w, off[:2]),
                 lambda: grouped.linear(x, w[:, :30], off), lambda: grouped.linear(x[:, :56], w, off),
                 lambda: grouped.linear(x, w[:, :, :60].contiguous(), off),
                 lambda: grouped.linear(x, w, off, _bf(32, device=cuda)),
                 lambda: grouped.linear(x, w, off, out=torch.empty(8, 32, device=cuda)),
                 lambda: grouped.linear(x.cpu(), w, off), lambda: grouped.linear(x, w, off.cpu()),
                 lambda: grouped.linear(x.t(), w, off), lambda: grouped.linear_gelu(x, w, off, pre_out=x),
                 lambda: grouped.matmul_nt(dy, w, off, gelu_pre=dy), lambda: grouped.weight_grad(dy, x[:7], off),
                 lambda: grouped.weight_grad(dy, x, off, grad.to(torch.bfloat16)),
                 lambda: grouped.weight_grad(dy, x, off, grad[:1]), lambda: grouped.bias_grad(dy[:, :30], off)):
        with pytest.raises((ValueError, TypeError)):
            call()
    with pytest.raises(native.NativeError):
        grouped.linear(x, w, off, tile=64)
    odd = torch.empty(8 * 64 + 4, device=cuda, dtype=torch.bfloat16)[4:].view(8, 64)
    with pytest.raises(native.NativeError):
        grouped.linear(odd, w, off)
