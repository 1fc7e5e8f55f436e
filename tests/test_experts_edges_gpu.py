"""The experts' operators where calls leave the beaten path: first call inside a
capture, two streams at once, a limited grid, offsets beyond 32 bits, the whole
layer in one run."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]

FIRST_CALL = """
import torch
from tempname_dcu_b200.ops import grouped, moe, mx4, native
torch.cuda.set_device(0)
bf = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
z, x, w1, w2 = torch.randn(300, 8, device="cuda"), bf(300, 256), bf(8, 512, 256), bf(8, 256, 512)
q, sf = torch.empty(8, 512, 128, dtype=torch.uint8, device="cuda"), torch.empty(8 * 4 * 1024, dtype=torch.uint8, device="cuda")

def layer():
    r = moe.route(z, 2)
    xs = moe.dispatch(x, r)
    h, pre = grouped.linear_gelu(xs, w1, r.offsets)
    ys = grouped.linear(h, w2, r.offsets)
    out = moe.combine(ys, r, residual=x)
    dys, dw = moe.combine_bwd(x, ys, r)
    dz = grouped.matmul_nt(dys, w2, r.offsets, gelu_pre=pre)
    g1, b1 = grouped.weight_grad(dz, xs, r.offsets), grouped.bias_grad(dz, r.offsets)
    dx = moe.dispatch_bwd(grouped.matmul_nt(dz, w1, r.offsets), r)
    dl = moe.route_bwd(z, r, dw)
    mx4.quantize(w1, q=q, sf=sf)
    y4 = mx4.grouped_linear(*mx4.quantize(xs, offsets=r.offsets), q, sf, r.offsets)
    few = grouped.linear(x[:2], w1[:2], small)
    return [out, g1, b1, dx, dl, y4, few]

small = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):  # nothing has been launched before
    captured = layer()
graph.replay()
eager = layer()
assert all(torch.equal(a, b) for a, b in zip(captured, eager))
native.raise_on_status()
print("ok")
"""


def test_first_call_inside_a_capture(cuda):
    out = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip().endswith("ok"), out.stderr[-2000:]


def test_two_streams_at_once_and_a_limited_grid(cuda):
    import torch
    from tempname_dcu_b200.ops import grouped, moe, mx4, native
    torch.manual_seed(0)
    bf = lambda *s: torch.randn(*s, device=cuda).to(torch.bfloat16)
    data = []
    for seed in range(2):
        z, x, w = torch.randn(1500, 16, device=cuda), bf(1500, 512), bf(16, 520, 512)
        data.append((z, x, w, mx4.quantize(w)))

    def layer(z, x, w, w4):
        r = moe.route(z, 2)
        xs = moe.dispatch(x, r)
        y = grouped.linear(xs, w, r.offsets)
        g = grouped.weight_grad(y, xs, r.offsets)
        y4 = mx4.grouped_linear(*mx4.quantize(xs, offsets=r.offsets), *w4, r.offsets)
        return r.slots, y, g, grouped.matmul_nt(y, w, r.offsets), y4
    expected = [layer(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = layer(*data[i])
    torch.cuda.synchronize()
    for a, b in zip(expected, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    with native.grid_limit(7):
        limited = layer(*data[0])
    assert all(torch.equal(u, v) for u, v in zip(limited, expected[0]))
    native.raise_on_status()


def test_rows_beyond_32_bit_offsets(cuda):
    """Row operands of more than 2^31 elements; only the last rows are compared."""
    import torch
    from tempname_dcu_b200.ops import grouped, moe, mx4, native
    H, tokens = 8192, 2 ** 18 + 300
    assert tokens * H > 2 ** 31
    x = torch.zeros(tokens, H, device=cuda, dtype=torch.bfloat16)
    x[-300:] = torch.randn(300, H, device=cuda).to(torch.bfloat16)
    r = moe.route(torch.zeros(tokens, 8, device=cuda), 1)  # ties: every token to expert 0, in order
    xs = moe.dispatch(x, r)
    assert torch.equal(xs[-300:], x[-300:])
    assert torch.equal(moe.combine(xs, r)[-300:], x[-300:])
    dys, dw = moe.combine_bwd(x, xs, r)
    assert torch.equal(dys[-300:], x[-300:])
    ref = x[-300:].double().square().sum(1)
    assert ((dw[-300:, 0].double() - ref).abs() <= ref * H * 2.0 ** -24).all()
    del xs, dys
    off = torch.tensor([0, tokens - 299, tokens], dtype=torch.int32, device=cuda)
    w = torch.randn(2, 8, H, device=cuda).to(torch.bfloat16)
    y = grouped.linear(x, w, off)
    exact = x[-299:].double() @ w[1].double().t()
    size = x[-299:].double().abs() @ w[1].double().abs().t()
    assert ((y[-299:].double() - exact).abs() <= exact.abs() * 2.0 ** -8 + size * H * 2.0 ** -22).all()
    wide = grouped.matmul_nt(y, w, off)  # an output of more than 2^31 elements
    exact = y[-299:].double() @ w[1].double()
    size = y[-299:].double().abs() @ w[1].double().abs()
    assert ((wide[-299:].double() - exact).abs() <= exact.abs() * 2.0 ** -8 + size * 8 * 2.0 ** -22).all()
    del wide
    g = grouped.weight_grad(y, x, off)
    exact = y[-299:].double().t() @ x[-299:].double()
    size = y[-299:].double().abs().t() @ x[-299:].double().abs()
    assert ((g[1].double() - exact).abs() <= exact.abs() * 2.0 ** -24 + size * 299 * 2.0 ** -22).all()
    q, sf = mx4.quantize(x)
    tail = mx4.dequantize(*mx4.quantize(x[-300:].contiguous()))
    assert torch.equal(mx4.dequantize(q, sf)[-300:], tail)
    native.raise_on_status()


def test_tensors_by_keyword(cuda):
    import torch
    from tempname_dcu_b200.ops import grouped, moe
    z, x = torch.randn(9, 8, device=cuda), torch.randn(9, 64, device=cuda).to(torch.bfloat16)
    r = moe.route(logits=z, top_k=2)
    w = torch.randn(8, 32, 64, device=cuda).to(torch.bfloat16)
    y = grouped.linear(x=moe.dispatch(x=x, routing=r), w=w, offsets=r.offsets)
    assert torch.equal(y, grouped.linear(moe.dispatch(x, r), w, r.offsets))


def test_layer_against_64_bits(cuda):
    """Router, exchange and both products as a layer uses them, with the
    gradients, for a ragged batch with a closed expert."""
    import torch
    from tempname_dcu_b200.ops import grouped, moe, native
    torch.manual_seed(4)
    T, E, k, H, Fh = 333, 16, 3, 264, 520
    bf = lambda *s, scale=1.0: (torch.randn(*s, device=cuda) * scale).to(torch.bfloat16)
    x, z = bf(T, H), torch.randn(T, E, device=cuda)
    z[:, 5] = float("-inf")
    w1, b1, w2, b2 = bf(E, Fh, H, scale=0.06), bf(E, Fh, scale=0.1), bf(E, H, Fh, scale=0.04), bf(E, H, scale=0.1)
    dout = bf(T, H)
    r = moe.route(z, k)
    xs = moe.dispatch(x, r)
    h, pre = grouped.linear_gelu(xs, w1, r.offsets, b1)
    ys = grouped.linear(h, w2, r.offsets, b2)
    out = moe.combine(ys, r, residual=x)
    dys, dw = moe.combine_bwd(dout, ys, r)
    got = dict(w2=grouped.weight_grad(dys, h, r.offsets), b2=grouped.bias_grad(dys, r.offsets))
    dz = grouped.matmul_nt(dys, w2, r.offsets, gelu_pre=pre)
    got.update(w1=grouped.weight_grad(dz, xs, r.offsets), b1=grouped.bias_grad(dz, r.offsets),
               x=moe.dispatch_bwd(grouped.matmul_nt(dz, w1, r.offsets), r, residual=dout), z=moe.route_bwd(z, r, dw))
    leaf = {n: t.double().requires_grad_(True) for n, t in dict(x=x, z=z, w1=w1, b1=b1, w2=w2, b2=b2).items()}
    weights = leaf["z"].gather(1, r.ids.long()).softmax(1)
    ref = leaf["x"]
    y = torch.zeros_like(ref)
    for e in range(E):
        t, j = (r.ids == e).nonzero(as_tuple=True)
        u = torch.nn.functional.gelu(leaf["x"][t] @ leaf["w1"][e].t() + leaf["b1"][e])
        y = y.index_add(0, t, weights[t, j][:, None] * (u @ leaf["w2"][e].t() + leaf["b2"][e]))
    ref = ref + y
    ref.backward(dout.double())
    # each result passes at most five bf16 roundings of independent elements: sqrt(5) 2^-9 of its 2-norm, twice that
    assert (out.double() - ref).norm() / ref.norm() < 2 * 5 ** 0.5 * 2.0 ** -9
    for name, value in got.items():
        exact = torch.nan_to_num(leaf[name].grad)
        assert (value.double() - exact).norm() / exact.norm() < 2 * 5 ** 0.5 * 2.0 ** -9, name
    assert (got["w1"][5] == 0).all() and (got["z"][:, 5] == 0).all() and r.offsets[5] == r.offsets[6]
    native.raise_on_status()
