"""What the experts' entry points promise beside their results: outputs of a
refused call stay as they were, limits of GELU and its slope, cost of routing
in proportion to the tokens, results under a grid limit."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", ["linear", "few", "gelu", "data", "weight", "weight_acc", "bias", "bias_acc"])
@pytest.mark.parametrize("values", [[0, 40, 65], [0, 50, 20], [-1, 10, 64], [0, 64, 80], [70, 70, 70]])
def test_bad_offsets_leave_the_outputs(cuda, values, call):
    import torch
    from tempname_dcu_b200.ops import grouped, native
    rows = 16 if call == "few" else 64
    bf = lambda *s: torch.randn(*s, device=cuda).to(torch.bfloat16)
    x, w = bf(rows, 64), bf(2, 64, 64)
    off = torch.tensor(values, dtype=torch.int32, device=cuda)
    native.clear_status()
    if call in ("linear", "few", "gelu", "data"):
        outs = [torch.full((rows, 64), 7.0, device=cuda, dtype=torch.bfloat16) for _ in range(2)]
        if call == "data":
            grouped.matmul_nt(x, w, off, out=outs[0])
        elif call == "gelu":
            grouped.linear_gelu(x, w, off, out=outs[0], pre_out=outs[1])
        else:
            grouped.linear(x, w, off, out=outs[0], tile=16 if call == "few" else 0)
    else:
        shape = (2, 64, 64) if call.startswith("weight") else (2, 64)
        outs = [torch.full(shape, 7.0, device=cuda)]
        grad = grouped.weight_grad if call.startswith("weight") else grouped.bias_grad
        grad(x, *([x] if call.startswith("weight") else []), off, outs[0], accumulate=call.endswith("acc"))
    with pytest.raises(native.NativeError):
        native.raise_on_status()
    assert all((t == 7).all() for t in outs)


@pytest.mark.parametrize("groups,width", [(2, 4096), (700, 64), (1024, 8)])
def test_one_bad_offset_among_many_groups(cuda, groups, width):
    """Also where each group has its own blocks, and where the fault lies in the last of many entries."""
    import torch
    from tempname_dcu_b200.ops import grouped, native
    dy = torch.randn(2048, width, device=cuda).to(torch.bfloat16)
    good = torch.arange(groups + 1, dtype=torch.int32, device=cuda)
    for at, value in ((groups, 2049), (groups, 0), (0, -1), (groups // 2, 2048)):
        off = good.clone()
        off[at] = value
        for accumulate in (False, True):
            native.clear_status()
            out = torch.full((groups, width), 7.0, device=cuda)
            grouped.bias_grad(dy, off, out, accumulate=accumulate)
            with pytest.raises(native.NativeError):
                native.raise_on_status()
            assert (out == 7).all()
    native.clear_status()


def _route_time(tokens, experts, top_k):
    """Shortest of five calls, in milliseconds."""
    import torch
    from tempname_dcu_b200.ops import moe
    z = torch.randn(tokens, experts, device="cuda")
    moe.route(z, top_k)
    best = float("inf")
    for _ in range(5):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        moe.route(z, top_k)
        end.record()
        torch.cuda.synchronize()
        best = min(best, start.elapsed_time(end))
    return best


def test_routing_time_grows_with_the_tokens(cuda):
    """Eight times the tokens take eight times the time; 24 leaves room for a
    busy machine, and a cost of their square (64) fails."""
    assert _route_time(2 ** 20, 128, 2) < 24 * _route_time(2 ** 17, 128, 2)


@pytest.mark.parametrize("tokens,experts,top_k", [(16384, 128, 2), (16385, 7, 3), (20001, 512, 1), (65535, 60, 4),
                                                  (65536 * 3 + 1, 8, 2), (2 ** 20 + 77, 33, 1)])
def test_many_tokens_against_a_sort(cuda, tokens, experts, top_k):
    import torch
    from tempname_dcu_b200.ops import moe
    torch.manual_seed(tokens)
    z = torch.randn(tokens, experts, device=cuda)
    z[: tokens // 3, 0] += 8  # a long stretch of tokens that choose one expert
    for _ in range(2):
        r = moe.route(z, top_k)
        ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top_k]
        assert torch.equal(r.ids.long(), ids)
        order = torch.sort(ids.reshape(-1), stable=True).indices
        assert torch.equal(r.order.long(), order)
        assert torch.equal(r.slots.long()[order], torch.arange(order.numel(), device=cuda))
        counts = torch.bincount(ids.reshape(-1), minlength=experts)
        assert r.offsets[0] == 0 and torch.equal(r.offsets[1:].long(), counts.cumsum(0))


def test_choices_up_to_2_to_the_31(cuda):
    """The most tokens that the router takes, with the most choices: the last
    choice has the index 2^31 - 17.  Equal logits: every token chooses all
    experts in order, so the row of choice (t, j) is j * tokens + t."""
    import torch
    from tempname_dcu_b200.ops import moe, native
    T, k = 2 ** 27 - 1, 16
    r = moe.route(torch.zeros(T, k, device=cuda, dtype=torch.bfloat16), k)
    assert torch.equal(r.offsets.long(), torch.arange(k + 1, device=cuda) * T)
    expert = torch.arange(k, device=cuda)
    for t0 in (0, T // 2, T - 4000):
        rows = slice(t0, t0 + 4000)
        t = torch.arange(t0, min(t0 + 4000, T), device=cuda)
        assert torch.equal(r.ids[rows].long(), expert.expand(t.numel(), k))
        assert (r.weights[rows] == 1 / 16).all()
        slots = expert * T + t[:, None]
        assert torch.equal(r.slots.view(T, k)[rows].long(), slots)
        assert torch.equal(r.order[slots.reshape(-1)].long(), (t[:, None] * k + expert).reshape(-1))
    native.raise_on_status()


@pytest.mark.parametrize("tile", [32, 128, 512])
def test_gelu_slope_at_its_limits(cuda, tile):
    """The gradient is the slope itself where the product is 1.  Its formula is
    off by less than 7.5e-8, fp32 adds 2^-24 near 1; below -4 the error is relative:
    the tail's (3 % at -12) divided by x^2, far below 2^-10."""
    import torch
    from tempname_dcu_b200.ops import grouped
    inf, nan = float("inf"), float("nan")
    special = [inf, -inf, nan, 0.0, -0.0, 1e20, -1e20, 3e38, -3e38, 1e-30, -1e-30, 14.0, -14.0, 40.0, -40.0, 1.0]
    pre = torch.cat([torch.tensor(special), torch.linspace(-12, 12, 2048 - 16)]).to(cuda, torch.bfloat16).view(32, 64)
    dy, w = torch.zeros(32, 8, device=cuda, dtype=torch.bfloat16), torch.ones(1, 8, 64, device=cuda, dtype=torch.bfloat16)
    dy[:, 3] = 1
    off = torch.tensor([0, 32], dtype=torch.int32, device=cuda)
    got = grouped.matmul_nt(dy, w, off, gelu_pre=pre, tile=tile).double().view(-1)
    assert got[:2].tolist() == [1.0, 0.0] and got[2].isnan() and got[3:5].tolist() == [0.5, 0.5]
    assert got[5:9].tolist() == [1.0, 0.0, 1.0, 0.0] and got[9:12].tolist() == [0.5, 0.5, 1.0]
    x = pre.double().view(-1)[11:]
    exact = 0.5 * torch.erfc(-x / 2 ** 0.5) + x * torch.exp(-x * x / 2) / (2 * torch.pi) ** 0.5
    err = (got[11:] - exact).abs()
    assert (err <= exact.abs() * 2.0 ** -8 + 1.5e-7).all()
    low = (x <= -4) & (x >= -12)
    assert low.sum() > 600 and (err[low] <= exact[low].abs() * (2.0 ** -8 + 2.0 ** -10)).all()


def test_longest_4_bit_rows(cuda):
    """The largest K: one row as an operand of a product of two rows' worth of ones."""
    import torch
    from tempname_dcu_b200.ops import mx4, native
    K = mx4.MAX_K
    x = torch.zeros(1, K, device=cuda, dtype=torch.bfloat16)
    x[0, -1], x[0, 0], x[0, K // 2] = 3, 1, -0.5
    q, sf = mx4.quantize(x)
    assert torch.equal(mx4.dequantize(q, sf), x)
    w = torch.zeros(8, K, device=cuda, dtype=torch.bfloat16)
    w[:, -1] = torch.arange(8, device=cuda) % 4
    w[:, 0] = 2
    y = mx4.linear(q, sf, *mx4.quantize(w))
    assert y.tolist() == [[2.0 + 3 * (n % 4) for n in range(8)]]
    with pytest.raises(ValueError):
        mx4.quantize(torch.empty(1, K + 32, device=cuda, dtype=torch.bfloat16))
    native.raise_on_status()


def test_shared_sums_under_a_grid_limit(cuda):
    """A limited grid shares no sums: the order of the additions differs from the
    unlimited call's, so the results agree within their error and, among calls
    of either kind, bit for bit."""
    import torch
    from tempname_dcu_b200.ops import grouped, mx4, native
    torch.manual_seed(7)
    K, rows = 4104, 1500
    off = torch.tensor([0, 40, 40, 1480, rows], dtype=torch.int32, device=cuda)
    spans = [(0, 40), (40, 40), (40, 1480), (1480, rows)]
    x = torch.randn(rows, K, device=cuda).to(torch.bfloat16)
    w = (torch.randn(4, 40, K, device=cuda) * 0.1).to(torch.bfloat16)
    x4, w4 = torch.randn(40, 4096, device=cuda).to(torch.bfloat16), torch.randn(64, 4096, device=cuda).to(torch.bfloat16)
    q4 = (*mx4.quantize(x4), *mx4.quantize(w4))

    def calls():
        y = grouped.linear(x, w, off)
        return y, grouped.weight_grad(y, x, off), grouped.bias_grad(y, off), mx4.linear(*q4)
    free, again = calls(), calls()
    with native.grid_limit(20):
        limited, repeated = calls(), calls()
    assert all(torch.equal(a, b) for a, b in zip(free, again))
    assert all(torch.equal(a, b) for a, b in zip(limited, repeated))
    v4 = [mx4.dequantize(*q4[i:i + 2]).double() for i in (0, 2)]
    for y, dw, db, y4 in (free, limited):
        for g, (a, b) in enumerate(spans):
            exact, size = x[a:b].double() @ w[g].double().t(), x[a:b].double().abs() @ w[g].double().abs().t()
            assert ((y[a:b].double() - exact).abs() <= exact.abs() * 2.0 ** -8 + size * K * 2.0 ** -22).all()
            exact = y[a:b].double().t() @ x[a:b].double()
            assert (dw[g].double() - exact).norm() <= 2.0 ** -20 * exact.norm()  # see test_experts_exact_gpu.py
        exact, size = v4[0] @ v4[1].t(), v4[0].abs() @ v4[1].abs().t()
        assert ((y4.double() - exact).abs() <= exact.abs() * 2.0 ** -8 + size * 4096 * 2.0 ** -22).all()
    native.raise_on_status()
