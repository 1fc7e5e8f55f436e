"""Routing and row exchange (csrc/moe.cu) against plain implementations in 64
bits.

Tolerances: fp32 softmax weights.  expf is off by at most 2 ulp (2^-22), the
subtraction z - m rounds by 2^-24 |z - m|, which exp turns into a relative
error of the same size (|z - m| < 32 here: 2^-19), the sums of at most 512
terms and the quotient add below 2^-20: 2^-18 in all, relative to the weight.
bf16 outputs: half a step, 2^-8 relative, plus the fp32 sum's error, which is
below 2^-20 of the sum of the terms' magnitudes.
"""
import pytest

pytestmark = pytest.mark.gpu


def _plain_route(z, k, normalize):
    """Definition in 64 bits: z [T, E] float64 -> ids, weights, offsets, order, slots."""
    import torch
    T, E = z.shape
    ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    top = z.amax(1, keepdim=True)
    p = torch.where(top == float("-inf"), torch.zeros_like(z), torch.exp(z - top))
    chosen = p.gather(1, ids)
    total = (chosen if normalize else p).sum(1, keepdim=True)
    weights = torch.where(total > 0, chosen / total, torch.zeros_like(chosen))
    flat = ids.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(T * k, device=z.device)
    offsets = torch.zeros(E + 1, dtype=torch.int64, device=z.device)
    offsets[1:] = torch.bincount(flat, minlength=E).cumsum(0)
    return ids, weights, offsets, order, slots


def _check_route(r, z, k, normalize):
    import torch
    ids, weights, offsets, order, slots = _plain_route(z.double(), k, normalize)
    assert torch.equal(r.ids.long(), ids)
    assert torch.equal(r.offsets.long(), offsets)
    assert torch.equal(r.order.long(), order)
    assert torch.equal(r.slots.long(), slots)
    assert ((r.weights.double() - weights).abs() <= 2.0 ** -18 * weights + 1e-40).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (2, 512, 16), (63, 5, 5), (64, 33, 3), (65, 33, 3), (129, 64, 8),
                                   (1000, 100, 4), (4099, 256, 7), (5000, 512, 2), (3000, 3, 1)])
@pytest.mark.parametrize("normalize", [True, False])
def test_route(cuda, T, E, k, normalize, dtype):
    import torch
    from tempname_dcu_b200.ops import moe
    torch.manual_seed(T + E + k)
    # bf16 logits and coarse fp32 ones hold many ties
    z = (torch.randn(T, E, device=cuda) * 2).to(getattr(torch, dtype))
    if dtype == "float32":
        z[: T // 2] = torch.round(z[: T // 2])
    _check_route(moe.route(z, k, normalize=normalize), z, k, normalize)


def test_route_closed_experts_strides_and_zeros(cuda):
    import torch
    from tempname_dcu_b200.ops import moe
    torch.manual_seed(1)
    wide = torch.randn(200, 96, device=cuda)
    z = wide[:, 7:47]  # a row stride of 96 and an odd start
    z[::3, :35] = float("-inf")   # five experts left, k of them
    z[5] = float("-inf")          # nothing left
    z[6] = torch.finfo(torch.float32).min
    z[7] = 0.0
    z[7, ::2] = -0.0              # equal to +0: the order stays by index
    for normalize in (True, False):
        r = moe.route(z, 6, normalize=normalize)
        _check_route(r, z, 6, normalize)
        assert (r.weights[5] == 0).all() and r.ids[5].tolist() == [0, 1, 2, 3, 4, 5]
        assert r.ids[7].tolist() == [0, 1, 2, 3, 4, 5]


def test_route_without_tokens_and_with_nan(cuda):
    import torch
    from tempname_dcu_b200.ops import moe
    r = moe.route(torch.empty(0, 8, device=cuda), 2)
    assert r.offsets.tolist() == [0] * 9 and r.ids.shape == (0, 2)
    assert moe.route_bwd(torch.empty(0, 8, device=cuda), r, torch.empty(0, 2, device=cuda)).shape == (0, 8)
    x = torch.empty(0, 64, device=cuda, dtype=torch.bfloat16)
    assert moe.dispatch(x, r).shape == (0, 64) and moe.combine(x, r).shape == (0, 64)
    z = torch.randn(70, 8, device=cuda)
    z[3, 5] = float("nan")
    r = moe.route(z, 2)
    assert r.ids[3, 0] == 5 and r.weights[3].isnan().all()  # NaN counts as the largest and shows
    clean = [t for t in range(70) if t != 3]
    ids, weights, *_ = _plain_route(z[clean].double(), 2, True)
    assert torch.equal(r.ids[clean].long(), ids)
    assert torch.equal(r.slots.sort().values.long(), torch.arange(140, device=cuda))


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (77, 33, 5), (300, 128, 8), (50, 512, 16), (9, 1, 1)])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_route_gradient(cuda, T, E, k, normalize, out):
    import torch
    from tempname_dcu_b200.ops import moe
    torch.manual_seed(T * E + k)
    z = torch.randn(T, E, device=cuda)
    if E > 8:
        z[0, 3:] = float("-inf")  # fewer open experts than choices for k > 3
    dw = torch.randn(T, k, device=cuda)
    r = moe.route(z, k, normalize=normalize)
    got = moe.route_bwd(z, r, dw, out=torch.full((T, E), 7.0, device=cuda, dtype=getattr(torch, out)))
    p = torch.softmax(z.double(), 1)
    w = p.gather(1, r.ids.long())
    if normalize:
        w = w / w.sum(1, keepdim=True)
        g = w * (dw.double() - (w * dw.double()).sum(1, keepdim=True))
        ref = torch.zeros_like(p).scatter(1, r.ids.long(), g)
    else:
        ref = p * (torch.zeros_like(p).scatter(1, r.ids.long(), dw.double()) - (w * dw.double()).sum(1, keepdim=True))
    # dz = w (dw - dot): the difference carries the weights' 2^-18 of |dw| + |dot|; bf16 adds half a step
    scale = dw.abs().amax().item() * 2
    tol = 2.0 ** -18 * scale + (ref.abs() * 2.0 ** -8 if out == "bfloat16" else 0)
    assert ((got.double() - ref).abs() <= tol).all()


def test_route_gradient_against_differences(cuda):
    import torch
    from tempname_dcu_b200.ops import moe
    torch.manual_seed(0)
    z = torch.randn(6, 12, device=cuda)
    z[2] = float("-inf")
    for normalize in (True, False):
        r = moe.route(z, 3, normalize=normalize)
        dw = torch.randn(6, 3, device=cuda)
        got = moe.route_bwd(z, r, dw)
        assert (got[2] == 0).all()  # a row without an open expert
        h = 1e-5
        for t in (0, 5):
            for e in range(12):
                up, dn = z.double().clone(), z.double().clone()
                up[t, e] += h
                dn[t, e] -= h

                def loss(v):
                    p = torch.softmax(v[t], 0)[r.ids[t].long()]
                    return ((p / p.sum() if normalize else p) * dw[t].double()).sum()
                # central differences: h^2 |f'''| + 2^-52 / h < 1e-9; the kernel: 2^-18 of the terms
                assert abs((loss(up) - loss(dn)) / (2 * h) - got[t, e]) < 2.0 ** -17 * dw.abs().max() + 1e-8


@pytest.mark.parametrize("T,k,H", [(1, 1, 8), (1, 2, 4096), (77, 3, 264), (130, 16, 72), (33, 5, 2056), (4, 4, 16384)])
def test_exchange(cuda, T, k, H):
    import torch
    from tempname_dcu_b200.ops import moe
    torch.manual_seed(T + k + H)
    E = max(k, 6)
    r = moe.route(torch.randn(T, E, device=cuda), k)
    bf = torch.bfloat16
    x = torch.randn(T, H + 16, device=cuda).to(bf)[:, 8:8 + H]  # strided rows
    slots = r.slots.long().view(T, k)
    ref = torch.empty(T * k, H, device=cuda, dtype=bf)
    ref[slots.reshape(-1)] = x.repeat_interleave(k, 0)
    assert torch.equal(moe.dispatch(x, r), ref)
    ys = torch.randn(T * k, H, device=cuda).to(bf)
    res = torch.randn(T, H, device=cuda).to(bf)
    w = r.weights.double()
    terms = w[:, :, None] * ys.double()[slots]
    for residual in (None, res):
        exact = terms.sum(1) + (0 if residual is None else residual.double())
        size = terms.abs().sum(1) + (0 if residual is None else residual.double().abs())
        got = moe.combine(ys, r, residual=residual).double()
        assert ((got - exact).abs() <= exact.abs() * 2.0 ** -8 + size * 2.0 ** -19).all()
    dout = torch.randn(T, H, device=cuda).to(bf)
    dys, dw = moe.combine_bwd(dout, ys, r)
    exact = torch.empty(T * k, H, device=cuda, dtype=torch.float64)
    exact[slots.reshape(-1)] = (w[:, :, None] * dout.double()[:, None]).reshape(T * k, H)
    assert ((dys.double() - exact).abs() <= exact.abs() * (2.0 ** -8 + 2.0 ** -23)).all()
    prod = dout.double()[:, None] * ys.double()[slots]
    # H fp32 additions in partial sums: below H 2^-24 of the magnitudes' sum
    assert ((dw.double() - prod.sum(2)).abs() <= prod.abs().sum(2) * H * 2.0 ** -24).all()
    dxs = torch.randn(T * k, H, device=cuda).to(bf)
    terms = dxs.double()[slots]
    got = moe.dispatch_bwd(dxs, r).double()
    assert ((got - terms.sum(1)).abs() <= terms.sum(1).abs() * 2.0 ** -8 + terms.abs().sum(1) * 2.0 ** -19).all()


def test_exchange_does_not_mix_nan_rows_and_repeats_bitwise(cuda):
    import torch
    from tempname_dcu_b200.ops import moe
    torch.manual_seed(3)
    r = moe.route(torch.randn(40, 8, device=cuda), 2)
    ys = torch.randn(80, 512, device=cuda).to(torch.bfloat16)
    ys[r.slots.long().view(40, 2)[7, 1]] = float("nan")
    a, b = moe.combine(ys, r), moe.combine(ys, r)
    bad = a.isnan().any(1).nonzero().flatten().tolist()
    assert bad == [7]
    keep = [t for t in range(40) if t != 7]
    assert torch.equal(a[keep], b[keep])


def test_slots_outside_the_rows_are_reported(cuda):
    """The kernel checks every slot before it uses it, so nothing is read or
    written out of range; the status word says so."""
    import torch
    from tempname_dcu_b200.ops import moe, native
    native.clear_status()
    r = moe.route(torch.randn(4, 8, device=cuda), 2)
    r.slots[3] = 99
    r.slots[4] = -1
    x = torch.randn(4, 64, device=cuda).to(torch.bfloat16)
    moe.dispatch(x, r, out=torch.zeros(8, 64, device=cuda, dtype=torch.bfloat16))
    with pytest.raises(native.NativeError):
        native.raise_on_status()
    assert native.read_status()[0] == 0


def test_captured_and_replayed(cuda):
    import torch
    from tempname_dcu_b200.ops import moe
    torch.manual_seed(5)
    z = torch.randn(700, 16, device=cuda)
    x = torch.randn(700, 128, device=cuda).to(torch.bfloat16)

    def layer():
        r = moe.route(z, 2)
        return r, moe.combine(moe.dispatch(x, r), r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs alive at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer()
        graphs.append((g, out))
    z.copy_(torch.randn(700, 16, device=cuda))
    x.copy_(torch.randn(700, 128, device=cuda))
    for g, _ in graphs:
        g.replay()
    r, y = layer()
    for _, (rg, yg) in graphs:
        assert torch.equal(rg.ids, r.ids) and torch.equal(rg.slots, r.slots) and torch.equal(yg, y)


def test_refusals(cuda):
    import torch
    from tempname_dcu_b200.ops import moe
    z = torch.randn(4, 8, device=cuda)
    x = torch.randn(4, 64, device=cuda).to(torch.bfloat16)
    r = moe.route(z, 2)
    for call in (lambda: moe.route(z, 0), lambda: moe.route(z, 9), lambda: moe.route(z.half(), 2),
                 lambda: moe.route(z.t(), 2), lambda: moe.route(torch.randn(2, 513, device=cuda), 2),
                 lambda: moe.route(z[0], 2), lambda: moe.route_bwd(z[:3], r, torch.zeros(3, 2, device=cuda)),
                 lambda: moe.route_bwd(z, r, torch.zeros(4, 3, device=cuda)),
                 lambda: moe.route_bwd(z, r, torch.zeros(4, 2, device=cuda, dtype=torch.float64)),
                 lambda: moe.dispatch(x[:, :60], r), lambda: moe.dispatch(x[:3], r), lambda: moe.dispatch(x.float(), r),
                 lambda: moe.dispatch(x, r, out=torch.empty(4, 64, device=cuda, dtype=torch.bfloat16)),
                 lambda: moe.combine(x, r), lambda: moe.combine_bwd(x, x, r),
                 lambda: moe.combine(torch.cat([x, x]), r, residual=x[:, :32])):
        with pytest.raises((ValueError, TypeError)):
            call()
    from tempname_dcu_b200.ops import native
    odd = torch.empty(4 * 64 + 4, device=cuda, dtype=torch.bfloat16)[4:].view(4, 64)  # 8-byte aligned rows
    with pytest.raises(native.NativeError):
        moe.dispatch(odd, r)
