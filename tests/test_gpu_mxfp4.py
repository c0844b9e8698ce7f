"""MXFP4 quantisation and the routed operators on 4-bit weights against the 64-bit oracle.

Quantisation is compared bit for bit.  Products are compared element by element with bounds that the oracle derives
from the roundings on the way (``oracle/mxfp4_ref.py``)."""
import copy
import io
import threading
import time

import pytest
import torch

from ffn_kernel_b200 import (GraphedMaskedFFN, MaskedFFN, MaskedFFNModule, MaskedLinearModule, MXFP4MaskedFFN, MXFP4MaskedFFNModule,
                             MXFP4MaskedLinear, MXFP4MaskedLinearModule, MXFP4Tensor, check_status, dequantize_mxfp4,
                             quantize_mxfp4)
from ffn_kernel_b200.synth import edge_mask
from oracle import mxfp4_ref as R

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def spread(rows, cols, seed, dtype=torch.bfloat16):
    """Magnitudes that differ by row and column."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randn(rows, 1, generator=g))
    return (x * torch.exp2(2 * torch.randn(1, cols, generator=g))).to(dtype)


def poison(dev):
    """Freed blocks full of NaN, for the allocator to hand out again as outputs and workspaces."""
    junk = [torch.full((n,), float("nan"), device=dev) for n in (1 << 10, 1 << 14, 1 << 18, 1 << 22)]
    del junk


def same_matrix(q: MXFP4Tensor, x: torch.Tensor):
    codes, scales = R.quantize(x.cpu().double())
    assert torch.equal(q.codes.cpu(), codes)
    assert torch.equal(q.scales.cpu(), scales)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 31), (37, 200), (64, 32), (130, 72), (129, 257), (5, 2049)])
def test_quantize_bit_for_bit(dev, name, rows, cols):
    x = spread(rows, cols, rows * 1000 + cols, DTYPES[name])
    poison(dev)
    same_matrix(quantize_mxfp4(x.to(dev)), x)
    poison(dev)
    same_matrix(quantize_mxfp4(x.T.contiguous().to(dev), dim=0), x)      # blocks along the strided dimension
    same_matrix(quantize_mxfp4(x.to(dev).T, dim=0), x)                   # the nn.Linear weight seen as [in, out]


def test_quantize_strided_and_offset_views(dev):
    base = spread(70, 300, 1).to(dev)
    for v in (base[:, 3:203], base[::2, :128], base[1:, 1:], base[:, ::3], base[5:6], base[:, 7:8]):
        same_matrix(quantize_mxfp4(v), v)
        same_matrix(quantize_mxfp4(v, dim=0), v.T)


@pytest.mark.parametrize("name", list(DTYPES))
def test_quantize_every_tie_and_special_value(dev, name):
    dt = DTYPES[name]
    ties = torch.tensor([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, 7.5, 7, -7.5, 0, -0.0])
    x = torch.zeros(12, 64)
    x[0, :20], x[1, 32:52], x[2, :20] = ties, ties * 2 ** -10, ties * 2 ** 8
    x[3, 5], x[4, 5], x[5, 5] = float("inf"), float("-inf"), float("nan")
    x[3, 6] = x[4, 40] = 3.0
    x[6, :4] = torch.tensor([torch.finfo(dt).max, -torch.finfo(dt).max, 1.0, torch.finfo(dt).tiny])
    x[7, :4] = torch.tensor([torch.finfo(dt).smallest_normal, -torch.finfo(dt).smallest_normal / 2, 0.0, 0.0])
    x = x.to(dt)
    x[8, 0] = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps      # the smallest subnormal alone
    x[9, 33] = -torch.finfo(dt).smallest_normal
    q = quantize_mxfp4(x.to(dev))
    same_matrix(q, x)
    back = dequantize_mxfp4(q, torch.float32).cpu().double()
    want = R.values(q.codes, q.scales, 12, 64)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(back), torch.nan_to_num(want))


@pytest.mark.parametrize("name", list(DTYPES))
def test_special_values_in_every_place(dev, name):
    dt = DTYPES[name]
    info = torch.finfo(dt)
    some = torch.tensor([float("inf"), float("-inf"), float("nan"), info.max, -info.max, info.smallest_normal, info.smallest_normal * info.eps,
                         -info.smallest_normal * info.eps, -0.0])
    x = spread(300, 520, 1, dt)
    g = torch.Generator().manual_seed(2)
    for i in range(400):
        r, c = (int(torch.randint(0, n, (), generator=g)) for n in x.shape)
        x[r, c] = some[i % len(some)].to(dt)
        if i % len(some) > 4:                       # small ones matter where nothing hides them
            b = c // 32 * 32
            x[r, b:b + 32] = 0
            x[r, c] = some[i % len(some)].to(dt)
    minus_nan = torch.tensor([-1], dtype=torch.int32 if dt is torch.float32 else torch.int16).view(dt)
    x[7, 9] = x[299, 519] = x[150, 260] = minus_nan[0]
    same_matrix(quantize_mxfp4(x.to(dev)), x)
    same_matrix(quantize_mxfp4(x.T.contiguous().to(dev), dim=0), x)
    wide = torch.empty(520, 333, dtype=dt, device=dev)[:, 1:301]             # columns that are not 4-byte aligned in 16 bits
    wide.copy_(x.T)
    same_matrix(quantize_mxfp4(wide, dim=0), x)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (130, 72), (257, 300), (9, 1031)])
def test_dequantize_any_codes_and_scales(dev, rows, cols):
    g = torch.Generator().manual_seed(rows)
    q = MXFP4Tensor(torch.randint(0, 256, (rows, -(-cols // 32) * 16), generator=g, dtype=torch.uint8).to(dev),
                    torch.randint(0, 256, (-(-rows // 128), -(-cols // 128), 32, 4, 4), generator=g, dtype=torch.uint8).to(dev),
                    rows, cols)
    want = R.values(q.codes, q.scales, rows, cols)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        got = dequantize_mxfp4(q, dt).cpu()
        # 6 * 2^127 is beyond bf16 and fp32: infinity, as the rounding of the value gives
        ref = want.to(torch.float32).to(dt)
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(ref.float()))


def test_empty_matrices(dev):
    for shape in ((0, 64), (5, 0)):
        q = quantize_mxfp4(torch.empty(shape, dtype=torch.bfloat16, device=dev))
        assert q.shape == shape and tuple(dequantize_mxfp4(q).shape) == shape


# ------------------------------------------------------------------------------------------------ products
def weights(shapes, seed, dev):
    qs = [quantize_mxfp4((spread(r, c, seed + i) * (0.5 * c ** -0.5)).to(dev)) for i, (r, c) in enumerate(shapes)]
    return qs, [R.values(q.codes, q.scales, q.rows, q.cols) for q in qs]


def inside(got, want_and_bound):
    want, bound = want_and_bound
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), f"worst: {(off / bound).max().item():.3f} of the bound"


MASKS = ["all_visual", "all_text", "alternating", "bernoulli", "span"]
LINEAR_SIZES = [(1, 64, 64), (3, 2056, 328), (1, 4096, 264), (2, 8, 8), (7, 40, 136), (33, 1000, 72), (127, 264, 520), (128, 256, 256),
                (129, 128, 1032), (300, 2056, 328), (515, 96, 2048), (1030, 520, 264), (8200, 72, 64), (33000, 40, 72)]


@pytest.mark.parametrize("M,K,N", LINEAR_SIZES)
@pytest.mark.parametrize("kind", MASKS)
def test_linear_forward_and_gradient(dev, M, K, N, kind):
    x, mask, g = spread(M, K, M + K), edge_mask(M, kind, seed=M), spread(M, N, M + N + 1)
    (b1, b2), (v1, v2) = weights([(N, K)] * 2, K, dev)
    poison(dev)
    with torch.no_grad():
        y0 = MXFP4MaskedLinear.apply(x.to(dev), b1, b2, mask.to(dev))
    xg = x.to(dev).requires_grad_(True)
    y = MXFP4MaskedLinear.apply(xg, b1, b2, mask.to(dev))
    poison(dev)
    y.backward(g.to(dev))
    check_status()
    assert torch.equal(y0, y.detach())
    inside(y.detach(), R.linear(x, v1, v2, mask))
    inside(xg.grad, R.linear_dx(g, v1, v2, mask))


@pytest.mark.parametrize("M,K,N", [(300, 4104, 264), (513, 4104, 136), (1000, 8200, 72), (200, 11008, 1032)])
@pytest.mark.parametrize("kind", MASKS)
def test_linear_of_several_row_tiles_and_a_long_contraction(dev, M, K, N, kind):
    x, mask = spread(M, K, M + K), edge_mask(M, kind, seed=M)
    (b1, b2), (v1, v2) = weights([(N, K)] * 2, K, dev)
    poison(dev)
    inside(MXFP4MaskedLinear.apply(x.to(dev), b1, b2, mask.to(dev)), R.linear(x, v1, v2, mask))
    check_status()


FFN_SIZES = [(1, 64, 64), (1, 1024, 1416), (2, 8, 8), (7, 40, 136), (33, 1000, 72), (127, 264, 520), (128, 256, 256),
             (130, 128, 1032), (300, 512, 328), (515, 96, 1000), (1030, 264, 136), (8200, 64, 72)]


def ffn_weights(d, h, seed, dev):
    return weights([(h, d), (d, h), (h, d)] * 2, seed, dev)


@pytest.mark.parametrize("M,d,h", FFN_SIZES)
@pytest.mark.parametrize("kind", MASKS)
def test_ffn_forward_and_gradient(dev, M, d, h, kind):
    x, mask, g = spread(M, d, M + d), edge_mask(M, kind, seed=M), spread(M, d, M + h)
    qs, vs = ffn_weights(d, h, d + h, dev)
    poison(dev)
    with torch.no_grad():
        y0 = MXFP4MaskedFFN.apply(x.to(dev), *qs, mask.to(dev))
    xg = x.to(dev).requires_grad_(True)
    y = MXFP4MaskedFFN.apply(xg, *qs, mask.to(dev))
    poison(dev)
    y.backward(g.to(dev))
    check_status()
    assert torch.equal(y0, y.detach())
    inside(y.detach(), R.ffn(x, vs, mask))
    inside(xg.grad, R.ffn_dx(g, x, vs, mask))


def test_linear_gradient_is_a_difference_of_outputs(dev):
    # activations that the format holds exactly, moved to others that it holds exactly: y moves by d @ W^T
    M, K, N = 40, 96, 128
    g = torch.Generator().manual_seed(5)
    grid = torch.tensor([1.0, 1.5, 2.0, 3.0, 4.0])
    x, x2 = (grid[torch.randint(0, 5, (M, K), generator=g)].to(torch.bfloat16) for _ in range(2))
    x[:, ::32] = x2[:, ::32] = 4.0                  # every block's largest value, so that its exponent is 0
    mask = edge_mask(M, "bernoulli", 3).to(dev)
    (b1, b2), _ = weights([(N, K)] * 2, 9, dev)
    up = spread(M, N, 2).to(dev)
    xg = x.to(dev).requires_grad_(True)
    y = MXFP4MaskedLinear.apply(xg, b1, b2, mask)
    y.backward(up)
    y2 = MXFP4MaskedLinear.apply(x2.to(dev), b1, b2, mask)
    moved = ((y2.double() - y.detach().double()) * up.double()).sum()
    told = (xg.grad.double() * (x2 - x).double().to(dev)).sum()
    # y, y2 and dx are each rounded to bf16 once (half a step, 2^-8 relative)
    bound = R.U16 * (((y.detach().abs() + y2.abs()).double() * up.abs().double()).sum()
                     + (xg.grad.abs().double() * (x2 - x).abs().double().to(dev)).sum()) * 1.01
    assert (moved - told).abs() <= bound


def test_ffn_gradient_is_a_difference_of_the_formula(dev):
    # the layer without its roundings to 4 bits, at the activations that the 4 bits hold
    M, d, h = 24, 64, 96
    x, mask, g = spread(M, d, 3), edge_mask(M, "bernoulli", 1), spread(M, d, 4)
    qs, vs = ffn_weights(d, h, 7, dev)
    xg = x.to(dev).requires_grad_(True)
    MXFP4MaskedFFN.apply(xg, *qs, mask.to(dev)).backward(g.to(dev))
    w1, w2, w3, u1, u2, u3 = vs

    def value(a):
        t1, t3 = R.by_rows(a, mask, w1.T, u1.T), R.by_rows(a, mask, w3.T, u3.T)
        return (R.by_rows(t1 * torch.sigmoid(t1) * t3, mask, w2.T, u2.T) * g.double()).sum()

    q, bound = R.rounded(x.double()), R.ffn_dx(g, x, vs, mask)[1]
    for i in range(6):
        way = torch.randn(M, d, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        eps = 1e-5
        diff = (value(q + eps * way) - value(q - eps * way)) / (2 * eps)
        told = (xg.grad.cpu().double() * way).sum()
        # central difference: its own error is of the order eps^2 times third derivatives, far below 1e-4 relative here
        assert (diff - told).abs() <= (bound * way.abs()).sum() + 1e-4 * diff.abs()


def test_rows_do_not_depend_on_one_another(dev):
    M, d, h = 700, 136, 264
    x, mask = spread(M, d, 1).to(dev), edge_mask(M, "span", 2).to(dev)
    qs, _ = ffn_weights(d, h, 3, dev)
    y = MXFP4MaskedFFN.apply(x, *qs, mask)
    for n in (1, 5, 130):
        assert torch.equal(MXFP4MaskedFFN.apply(x[:n], *qs, mask[:n]), y[:n])
    bad = x.clone()
    bad[::7] = float("nan")
    y2 = MXFP4MaskedFFN.apply(bad, *qs, mask)
    keep = torch.ones(M, dtype=torch.bool, device=dev)
    keep[::7] = False
    assert torch.equal(y2[keep], y[keep]) and torch.isnan(y2[::7]).all()


def test_infinite_activations_and_weights_give_nan_where_they_are_used(dev):
    M, K, N = 9, 96, 136
    x, mask = spread(M, K, 1), edge_mask(M, "alternating")
    x[4, 33] = float("inf")
    w = [spread(N, K, i) for i in (2, 3)]
    w[0][17, 5] = float("-inf")                # a visual weight row
    y = MXFP4MaskedLinear.apply(x.to(dev), *[quantize_mxfp4(t.to(dev)) for t in w], mask.to(dev)).cpu()
    want = torch.zeros(M, N, dtype=torch.bool)
    want[4] = True
    want[mask, 17] = True
    assert torch.equal(torch.isnan(y), want)


def test_strided_activations_gradients_and_uint8_mask(dev):
    M, K, N = 200, 72, 136
    wide = spread(M, K + 40, 1).to(dev)
    mask = edge_mask(M, "bernoulli", 1).to(dev)
    (b1, b2), _ = weights([(N, K)] * 2, 2, dev)
    want = MXFP4MaskedLinear.apply(wide[:, 8:8 + K].contiguous(), b1, b2, mask)
    for v in (wide[:, 8:8 + K], wide[:, 8:8 + K].T.contiguous().T):
        assert torch.equal(MXFP4MaskedLinear.apply(v, b1, b2, mask.to(torch.uint8) * 3), want)
    xg = wide[:, 8:8 + K].clone().requires_grad_(True)
    y = MXFP4MaskedLinear.apply(xg, b1, b2, mask)
    g = spread(M, N, 5).to(dev)
    a = torch.autograd.grad(y, xg, g, retain_graph=True)[0]
    b = torch.autograd.grad(y, xg, torch.cat([g, g], 1)[:, :N], retain_graph=True)[0]      # strided upstream gradient
    c = torch.autograd.grad(y.sum(), xg)[0]                                                # an expanded one
    assert torch.equal(a, b) and torch.isfinite(c).all()


@pytest.mark.parametrize("M", [1, 2, 5, 31, 32, 33, 64, 65, 127, 128, 129, 300, 8193, 32768, 32769])
@pytest.mark.parametrize("kind", MASKS)
def test_routing_lists_are_those_of_route(dev, M, kind):
    # few tokens are routed inside the product's kernel (K <= 512: up to 16 of them), more by a kernel before it
    from ffn_kernel_b200 import route
    from ffn_kernel_b200.mxfp4 import _mxfp4_linear_forward
    mask = edge_mask(M, kind, seed=M + 1).to(dev)
    want = route(mask)
    for K in (64, 2056):
        (b1, b2), _ = weights([(72, K)] * 2, 1, dev)
        lists = _mxfp4_linear_forward(spread(M, K, 1).to(dev), b1, b2, mask, keep=True)[1].view(torch.int32)
        perm, counts = lists[:-8], lists[-8:]
        assert torch.equal(counts[:5], want.counts[:5])
        mv = int(counts[0])
        assert torch.equal(perm[:mv], want.perm[:mv]) and torch.equal(perm[want.cap:want.cap + M - mv], want.perm[want.cap:want.cap + M - mv])


def test_a_few_strided_tokens(dev):
    K, N = 264, 136
    wide = spread(40, 3 * K + 8, 1).to(dev)
    (b1, b2), vs = weights([(N, K)] * 2, 2, dev)
    mask = edge_mask(20, "alternating").to(dev)
    for v in (wide[::2, 8:8 + K], wide[1::2, K + 8:2 * K + 8], wide[::2, 1:1 + K], wide[:20, :K].T.contiguous().T):
        for n in (1, 3, 20):
            inside(MXFP4MaskedLinear.apply(v[:n], b1, b2, mask[:n]), R.linear(v[:n].cpu(), *vs, mask[:n].cpu()))


def test_a_second_backward_needs_retain_graph(dev):
    M, d, h = 6, 64, 96
    qs, _ = ffn_weights(d, h, 1, dev)
    x = spread(M, d, 1).to(dev).requires_grad_(True)
    y = MXFP4MaskedFFN.apply(x, *qs, edge_mask(M, "alternating").to(dev))
    first = torch.autograd.grad(y.sum(), x, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], first)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), x)


def test_no_tokens(dev):
    mask = torch.zeros(0, dtype=torch.bool, device=dev)
    (b1, b2), _ = weights([(64, 32)] * 2, 1, dev)
    qs, _ = ffn_weights(32, 64, 1, dev)
    x = torch.empty(0, 32, dtype=torch.bfloat16, device=dev, requires_grad=True)
    y, z = MXFP4MaskedLinear.apply(x, b1, b2, mask), MXFP4MaskedFFN.apply(x, *qs, mask)
    assert tuple(y.shape) == (0, 64) and tuple(z.shape) == (0, 32)
    (y.sum() + z.sum()).backward()
    assert tuple(x.grad.shape) == (0, 32)


def test_refusals(dev):
    M, K, N = 16, 64, 96
    x, mask = spread(M, K, 1).to(dev), edge_mask(M, "alternating").to(dev)
    (b1, b2), _ = weights([(N, K)] * 2, 1, dev)
    qs, _ = ffn_weights(K, N, 1, dev)
    lin, ffn = MXFP4MaskedLinear.apply, MXFP4MaskedFFN.apply
    refused = [
        lambda: lin(x.float(), b1, b2, mask), lambda: lin(x[0], b1, b2, mask), lambda: lin(x, b1, b2, mask[1:]),
        lambda: lin(x, b1, b2, mask.float()), lambda: lin(x, b1, b2, mask.cpu()), lambda: lin(x, b1, b1.codes, mask),
        lambda: lin(x[:, :56], b1, b2, mask), lambda: lin(x, b1, qs[1], mask), lambda: ffn(x, *qs[:5], b1, mask[:4]),
        lambda: ffn(x, qs[1], *qs[1:], mask), lambda: ffn(x, *qs[:5], x, mask),
        lambda: quantize_mxfp4(x.double()), lambda: quantize_mxfp4(x[0]), lambda: quantize_mxfp4(x, dim=2),
        lambda: dequantize_mxfp4(b1, torch.float64), lambda: dequantize_mxfp4(b1.codes),
        lambda: MXFP4Tensor(b1.codes, b1.scales, N, K + 64), lambda: MXFP4Tensor(b1.codes.int(), b1.scales, N, K),
        lambda: MXFP4Tensor(b1.codes, b1.scales.permute(0, 1, 3, 2, 4).permute(0, 1, 3, 2, 4)[:, :, :, :, :2], N, K),
        lambda: MXFP4Tensor(b1.codes.cpu(), b1.scales, N, K),
        lambda: MXFP4Tensor(torch.cat([b1.codes] * 2, 1)[:, :32], b1.scales, N, K),
    ]
    for call in refused:
        with pytest.raises((RuntimeError, TypeError)):
            call()
    q36 = quantize_mxfp4(spread(96, 36, 1).to(dev))           # the format holds 36 columns, the product does not
    with pytest.raises(RuntimeError):
        lin(spread(M, 36, 1).to(dev), q36, q36, mask)
    check_status()


# ------------------------------------------------------------------------------------------------ as they are used together
def test_modules_and_graph_replay(dev):
    torch.manual_seed(3)
    d, h, T = 136, 264, 50
    ffn, lin = MaskedFFNModule(d, h, device=dev), MaskedLinearModule(d, d, device=dev)
    f4, l4 = MXFP4MaskedFFNModule.from_module(ffn), MXFP4MaskedLinearModule.from_module(lin)
    x = torch.randn(2, T // 2, d, device=dev, dtype=torch.bfloat16)
    mask = torch.rand(2, T // 2, device=dev) < 0.5
    xg = x.clone().requires_grad_(True)
    y = f4(l4(xg, mask), mask)                                # the two layers one after the other, trained through
    y.sum().backward()
    assert y.shape == x.shape and xg.grad.shape == x.shape and torch.isfinite(xg.grad).all()
    # what the layers hold is what the operators compute on
    mid = MXFP4MaskedLinear.apply(x.view(-1, d), quantize_mxfp4(lin.linear_v.weight), quantize_mxfp4(lin.linear_t.weight.T, dim=0),
                                  mask.view(-1))
    want = MXFP4MaskedFFN.apply(mid, *[quantize_mxfp4(getattr(ffn, n).weight) for n in f4.NAMES], mask.view(-1))
    assert torch.equal(want.view_as(x), y.detach())
    again = MXFP4MaskedFFNModule(d, h, device=dev)
    again.load_state_dict(f4.state_dict())
    graphed = GraphedMaskedFFN(again, T)
    for seed in range(3):
        xi = spread(T, d, seed).to(dev)
        mi = edge_mask(T, MASKS[seed], seed).to(dev)
        assert torch.equal(graphed(xi, mi), f4(xi, mi))
    check_status()


def test_two_streams_at_once_and_captured_training(dev):
    M, d, h = 600, 128, 264
    qs, _ = ffn_weights(d, h, 1, dev)
    (b1, b2), _ = weights([(d, d)] * 2, 2, dev)
    xs = [spread(M, d, s).to(dev) for s in range(4)]
    mask = edge_mask(M, "span", 1).to(dev)

    def step(x):
        x = x.detach().requires_grad_(True)
        y = MXFP4MaskedFFN.apply(MXFP4MaskedLinear.apply(x, b1, b2, mask), *qs, mask)
        return y.detach(), torch.autograd.grad(y, x, x.detach())[0]

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    got = [None] * 4
    for rep in range(3):
        for i, x in enumerate(xs):
            with torch.cuda.stream(streams[i % 2]):
                got[i] = step(x)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    static = xs[0].clone()
    streams[0].wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(streams[0]):
        step(static)
    torch.cuda.current_stream(dev).wait_stream(streams[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in (2, 1):
        static.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])
    check_status()


def test_repeated_calls_give_the_same_bits(dev):
    M, d, h = 3000, 264, 520
    x, mask = spread(M, d, 1).to(dev), edge_mask(M, "span", 1).to(dev)
    qs, _ = ffn_weights(d, h, 2, dev)
    y = MXFP4MaskedFFN.apply(x, *qs, mask)
    for _ in range(5):
        assert torch.equal(MXFP4MaskedFFN.apply(x, *qs, mask), y)


def test_a_single_row_of_any_stride(dev):
    # PyTorch calls a one-row view contiguous whatever its stride
    K, N = 72, 136
    wide = spread(4, 77, 1).to(dev)
    (b1, b2), _ = weights([(N, K)] * 2, 2, dev)
    qs, _ = ffn_weights(K, N, 3, dev)
    mask = torch.ones(1, dtype=torch.bool, device=dev)
    for v in (wide[0:1, :K], wide[1:2, :K], wide[:, 1:].as_strided((1, K), (1, 1)), wide[2:3, 5:]):
        plain = v.reshape(-1).clone().view(1, K)
        assert torch.equal(MXFP4MaskedLinear.apply(v, b1, b2, mask), MXFP4MaskedLinear.apply(plain, b1, b2, mask))
        a, b = v.detach().requires_grad_(True), plain.requires_grad_(True)
        ya, yb = MXFP4MaskedFFN.apply(a, *qs, mask), MXFP4MaskedFFN.apply(b, *qs, mask)
        assert torch.equal(ya, yb)
        assert torch.equal(torch.autograd.grad(ya, a, v)[0], torch.autograd.grad(yb, b, plain)[0])
    for v in (wide[0:1, ::3], wide[1:2, 1::2], wide[:, 3:4]):
        same_matrix(quantize_mxfp4(v), v)
        same_matrix(quantize_mxfp4(v, dim=0), v.T)


def test_a_copied_or_loaded_matrix_has_its_own_memory(dev):
    q = quantize_mxfp4(spread(70, 200, 1).to(dev))
    want = dequantize_mxfp4(q)
    stored = io.BytesIO()
    torch.save(q, stored)
    stored.seek(0)
    twins = [copy.deepcopy(q), torch.load(stored, weights_only=False), copy.copy(q)]
    assert twins[0].codes.data_ptr() != q.codes.data_ptr() != twins[1].codes.data_ptr()
    del q
    poison(dev)
    for t in twins:
        assert torch.equal(dequantize_mxfp4(t), want) and t.shape == (70, 200)
        for name in ("codes", "scales", "rows", "cols", "shape", "device"):
            with pytest.raises(AttributeError):
                setattr(t, name, getattr(t, name))


def test_weights_changed_before_the_backward_pass_are_noticed(dev):
    K, N = 64, 96
    mask = edge_mask(6, "alternating").to(dev)
    x = spread(6, K, 1).to(dev).requires_grad_(True)
    for run, ws in ((MXFP4MaskedLinear, [(N, K)] * 2), (MXFP4MaskedFFN, [(N, K), (K, N), (N, K)] * 2)):
        qs, _ = weights(ws, 1, dev)
        y = run.apply(x, *qs, mask)
        qs[-1].scales.add_(1)
        with pytest.raises(RuntimeError):
            y.sum().backward()
        with torch.inference_mode():
            frozen = [quantize_mxfp4(spread(r, c, 1).to(dev)) for r, c in ws]
        assert torch.isfinite(torch.autograd.grad(run.apply(x, *frozen, mask).sum(), x)[0]).all()
        with torch.autograd.forward_ad.dual_level():              # no forward-mode derivative: refused, not dropped
            with pytest.raises((RuntimeError, NotImplementedError)):
                run.apply(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()), *qs, mask)


def test_a_graph_outlives_the_module_it_was_captured_from(dev):
    d, h, T = 136, 264, 9
    torch.manual_seed(1)
    ffn = MaskedFFNModule(d, h, device=dev)
    x, mask = spread(T, d, 1).to(dev), edge_mask(T, "span").to(dev)
    with torch.no_grad():                     # a graph holds the inference forward
        want4, want = MXFP4MaskedFFNModule.from_module(ffn)(x, mask), ffn(x, mask)
    g4, g = GraphedMaskedFFN(MXFP4MaskedFFNModule.from_module(ffn), T), GraphedMaskedFFN(ffn, T)
    del ffn
    poison(dev)
    assert torch.equal(g4(x, mask), want4) and torch.equal(g(x, mask), want)


def test_nothing_of_the_workspace_reaches_the_results(dev):
    # every byte 255: scales that stand for NaN, in rows and blocks that exist only as padding
    def stain():
        junk = [torch.full((n,), 255, dtype=torch.uint8, device=dev) for n in (1 << 12, 1 << 16, 1 << 20, 1 << 24, 1 << 26)]
        del junk

    for M, d, h in ((1, 40, 72), (5, 200, 136), (130, 328, 1000), (700, 136, 264), (8200, 72, 136), (33000, 40, 72)):
        x, mask, g = spread(M, d, 1).to(dev), edge_mask(M, "span", 2).to(dev), spread(M, d, 3).to(dev)
        qs, _ = ffn_weights(d, h, 4, dev)
        x.requires_grad_(True)
        runs = []
        for _ in range(2):
            stain()
            z = MXFP4MaskedLinear.apply(x, qs[0], qs[3], mask)
            stain()
            y = MXFP4MaskedFFN.apply(x, *qs, mask)
            stain()
            dz = torch.autograd.grad(z, x, z.detach())[0]
            stain()
            runs.append((z.detach(), y.detach(), dz, torch.autograd.grad(y, x, g)[0]))
        for a, b in zip(*runs):
            assert torch.isfinite(a).all() and torch.equal(a, b)


def test_offsets_beyond_32_bits(dev):
    K = 32768
    x = torch.randn(140000, K, device=dev, dtype=torch.bfloat16)          # 4.6e9 values, 2.3e9 bytes of codes
    q = quantize_mxfp4(x)
    back = dequantize_mxfp4(q)
    for s in (slice(65500, 65700), slice(131000, 131200), slice(139900, 140000)):
        part = quantize_mxfp4(x[s].clone())
        assert torch.equal(q.codes[s], part.codes) and torch.equal(back[s], dequantize_mxfp4(part))
    del back
    q = quantize_mxfp4(x, dim=0)
    part = quantize_mxfp4(x[:, -128:].contiguous(), dim=0)
    assert torch.equal(q.codes[-128:], part.codes) and torch.equal(q.scales[-1], part.scales[0])
    del x, q, part
    torch.cuda.empty_cache()

    def tail(M, d, ws, run, forward, backward):
        qs, vs = weights(ws, 1, dev)
        x = torch.randn(M, d, device=dev, dtype=torch.bfloat16, requires_grad=True)
        mask = edge_mask(M, "bernoulli", 1)
        y = run.apply(x, *qs, mask.to(dev))
        g = torch.randn_like(y)
        dx = torch.autograd.grad(y, x, g)[0]
        check_status()
        for s in (slice(0, 40), slice(M // 2, M // 2 + 40), slice(M - 60, M)):
            xs, gs, ms = x[s].detach().cpu(), g[s].cpu(), mask[s]
            inside(y[s].detach(), forward(xs, vs, ms))
            inside(dx[s], backward(gs, xs, vs, ms))

    tail(1_100_000, 4096, [(4104, 4096)] * 2, MXFP4MaskedLinear, lambda x, vs, m: R.linear(x, *vs, m),
         lambda g, x, vs, m: R.linear_dx(g, *vs, m))
    torch.cuda.empty_cache()
    tail(540_000, 64, [(8200, 64), (64, 8200), (8200, 64)] * 2, MXFP4MaskedFFN, R.ffn, R.ffn_dx)
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------ hidden values below 2^-126
def tiny_hidden(M, d, h, dev):
    """FFN weights and activations whose hidden values are all 2^-127: the smallest block exponent, code 1.0."""
    w1, w3, w2 = torch.zeros(h, d), torch.zeros(h, d), torch.zeros(d, h)
    x = torch.zeros(M, d)
    x[:, 0], w1[:, 0], w3[:, 0], w2[:, 0] = 2.0 ** -30, 2.0 ** -40, 2.0 ** -26, 2.0 ** 100    # t1 2^-70 (silu: half of it), t3 2^-56
    qs = [quantize_mxfp4(w.to(torch.bfloat16).to(dev)) for w in (w1, w2, w3)] * 2
    return x.to(torch.bfloat16).to(dev), qs, torch.full((M, d), 2.0 ** -27, dtype=torch.bfloat16, device=dev)


# a few tokens (split kernel), single CTAs, CTA pairs
@pytest.mark.parametrize("M,d,h", [(1, 64, 96), (40, 64, 96), (200, 64, 96), (2305, 2048, 96)])
@pytest.mark.parametrize("train", [False, True])
def test_hidden_values_keep_subnormals(dev, M, d, h, train):
    # every step is a power of two: silu(2^-70) = 2^-71 to fp32, so the result is exact
    x, qs, want = tiny_hidden(M, d, h, dev)
    y = MXFP4MaskedFFN.apply(x.requires_grad_(train), *qs, edge_mask(M, "alternating").to(dev))
    assert torch.equal(y.detach(), want)


# ------------------------------------------------------------------------------------------------ CTA pairs
def test_repeated_calls_on_cta_pairs_give_the_same_bits(dev):
    # enough tiles that every pair hands its accumulators over several times, 4-bit and bf16 products alike
    M, d, h = 9001, 2056, 2824
    x, g, mask = spread(M, d, 1).to(dev), spread(M, d, 2).to(dev), edge_mask(M, "span", 1).to(dev)
    qs, _ = ffn_weights(d, h, 2, dev)
    ws = [dequantize_mxfp4(q).T.contiguous() for q in qs]
    x.requires_grad_(True)

    def once():
        y, z = MXFP4MaskedFFN.apply(x, *qs, mask), MaskedFFN.apply(x, *ws, mask)
        return [y.detach(), z.detach(), *torch.autograd.grad((y, z), (x,), (g, g))]

    first = once()
    for _ in range(10):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)
    check_status()


@pytest.fixture
def forced(libffnk):
    """forced(pair=1, narrow=0): kernel choices set for one test (the tables decide again afterwards)."""
    names = []

    def choose(**choices):
        for name, value in choices.items():
            names.append(name)
            assert libffnk.ffnk_tune_override(name.encode(), value) == 0
    yield choose
    for name in names:
        libffnk.ffnk_tune_override(name.encode(), -1)


# CTA pairs by the rule of the library, at its small end and started early beside the routing kernel; a last pair with rows
# in its first CTA only, a contraction that ends inside a k-step, an odd number of scale atoms, output columns that end in a tile
PAIR_LINEAR = [(1030, 1544, 264), (1153, 2056, 136), (8200, 1032, 72)]
PAIR_FFN = [(2050, 2056, 136), (2305, 2056, 328), (4100, 2048, 72)]


@pytest.mark.parametrize("M,K,N", PAIR_LINEAR)
@pytest.mark.parametrize("kind", MASKS)
def test_linear_on_cta_pairs(dev, M, K, N, kind):
    test_linear_forward_and_gradient(dev, M, K, N, kind)


@pytest.mark.parametrize("M,d,h", PAIR_FFN)
@pytest.mark.parametrize("kind", MASKS)
def test_ffn_on_cta_pairs(dev, M, d, h, kind):
    test_ffn_forward_and_gradient(dev, M, d, h, kind)


# one choice or the other whatever the rule: tile kernels with and without pairs down to one token, and the split kernel
@pytest.mark.parametrize("choices", [dict(pair=1, narrow=0), dict(pair=0, narrow=0), dict(narrow=1, permute=0)], ids=["pairs", "single", "split"])
@pytest.mark.parametrize("M,d,h", [(1, 64, 136), (130, 1000, 328), (515, 96, 1000)])
@pytest.mark.parametrize("kind", ["all_text", "alternating", "span"])
def test_every_kernel_at_every_size(dev, forced, choices, M, d, h, kind):
    forced(**choices)
    test_linear_forward_and_gradient(dev, M, d, h, kind)
    test_ffn_forward_and_gradient(dev, M, d, h, kind)


def test_cta_pairs_with_dirty_workspaces_and_two_streams(dev):
    M, d, h = 2305, 2056, 1544
    x, mask, g = spread(M, d, 1).to(dev), edge_mask(M, "span", 2).to(dev), spread(M, d, 3).to(dev)
    qs, _ = ffn_weights(d, h, 4, dev)

    def step(fill):
        junk = [torch.full((n,), fill, dtype=torch.uint8, device=dev) for n in (1 << 12, 1 << 16, 1 << 20, 1 << 24, 1 << 26)]
        del junk
        a = x.detach().requires_grad_(True)
        z, y = MXFP4MaskedLinear.apply(a, qs[0], qs[3], mask), MXFP4MaskedFFN.apply(a, *qs, mask)
        return z.detach(), y.detach(), *torch.autograd.grad((z, y), a, (z.detach(), g))

    want = step(0)
    assert all(torch.isfinite(t).all() for t in want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    got = []
    for rep in range(4):
        with torch.cuda.stream(streams[rep % 2]):
            got.append(step(255))
    torch.cuda.synchronize()
    for other in got:
        assert all(torch.equal(a, b) for a, b in zip(want, other))
    check_status()


# ------------------------------------------------------------------------------------------------ kernels by the number of tokens
def test_a_token_among_few_and_among_many(dev):
    # rows do not mix; the order of a row's fp32 sums goes by the number of tokens, so that here every batch is held to the
    # oracle's bound, and to the same bits only against batches of the same size
    K, N, d, h = 8200, 264, 4104, 328
    M = 1300
    mask = edge_mask(M, "span", 3)
    (b1, b2), vs = weights([(N, K)] * 2, 5, dev)
    qs, ws = ffn_weights(d, h, 6, dev)
    x, z, m = spread(M, K, 1), spread(M, d, 2), mask.to(dev)
    want, bound = R.linear(x[:130], *vs, mask[:130])
    fwant, fbound = R.ffn(z[:130], ws, mask[:130])
    for n in (1, 2, 16, 17, 64, 65, 129, 300, 520, M):
        y, f = MXFP4MaskedLinear.apply(x[:n].to(dev), b1, b2, m[:n]), MXFP4MaskedFFN.apply(z[:n].to(dev), *qs, m[:n])
        inside(y[:130], (want[:n], bound[:n]))
        inside(f[:130], (fwant[:n], fbound[:n]))
        # the same size with other neighbours
        xo, zo = spread(n, K, 8).to(dev), spread(n, d, 9).to(dev)
        keep = n // 2
        xo[keep], zo[keep] = x[keep].to(dev), z[keep].to(dev)
        assert torch.equal(MXFP4MaskedLinear.apply(xo, b1, b2, m[:n])[keep], y[keep])
        assert torch.equal(MXFP4MaskedFFN.apply(zo, *qs, m[:n])[keep], f[keep])
    check_status()


def test_split_kernel_of_more_tokens_than_a_cta_counts(dev):
    # few output columns, a contraction so long that 4200 tokens still take the split kernel, whose CTAs then read the
    # counts of the routing kernel instead of counting the mask
    M, K, N = 4200, 33800, 72
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(M, K, device=dev, generator=g).to(torch.bfloat16)
    (b1, b2), vs = weights([(N, K)] * 2, 5, dev)
    for kind in ("span", "all_text", "all_visual"):
        mask = edge_mask(M, kind, 2)
        poison(dev)
        y = MXFP4MaskedLinear.apply(x, b1, b2, mask.to(dev))
        for s in (slice(0, 40), slice(2030, 2070), slice(M - 60, M)):
            inside(y[s], R.linear(x[s].cpu(), *vs, mask[s]))
        check_status()


# 72 and 200 columns: three and seven blocks, the contraction ends inside a pair of blocks; 136 and 264 rows fill no atom
@pytest.mark.parametrize("M", [1, 40, 300, 1100])
@pytest.mark.parametrize("rows,cols", [(136, 72), (264, 200)])
def test_matrices_made_elsewhere(dev, M, rows, cols):
    # packed by the oracle; scales of rows and blocks that do not exist are 0, or any byte but the 255 that stands for NaN
    shapes = [(rows, cols), (cols, rows), (rows, cols)] * 2
    plain = [spread(r, c, 10 + i) * 0.25 for i, (r, c) in enumerate(shapes)]
    packed = [R.quantize(w.double()) for w in plain]
    zero = [MXFP4Tensor(c.to(dev), s.to(dev), r, k) for (c, s), (r, k) in zip(packed, shapes)]
    other = []
    for (c, s), (r, k) in zip(packed, shapes):
        row = torch.arange(s.shape[0] * 128).view(-1, 1, 4, 32, 1).transpose(2, 3).expand(s.shape)
        block = torch.arange(s.shape[1] * 4).view(1, -1, 1, 1, 4).expand(s.shape)
        junk = torch.randint(0, 255, s.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(r))
        other.append(MXFP4Tensor(c.to(dev), torch.where((row < r) & (block < -(-k // 32)), s, junk).contiguous().to(dev), r, k))
    for q, w in zip(zero, plain):
        same_matrix(quantize_mxfp4(w.to(dev)), w)
        assert torch.equal(quantize_mxfp4(w.to(dev)).scales, q.scales) and torch.equal(quantize_mxfp4(w.to(dev)).codes, q.codes)
    mask, x = edge_mask(M, "alternating"), spread(M, cols, 3)
    values = [R.values(q.codes, q.scales, q.rows, q.cols) for q in zero]
    for qs in (zero, other):
        inside(MXFP4MaskedLinear.apply(x.to(dev), qs[0], qs[3], mask.to(dev)), R.linear(x, values[0], values[3], mask))
        inside(MXFP4MaskedFFN.apply(x.to(dev), *qs, mask.to(dev)), R.ffn(x, values, mask))
        assert all(torch.equal(dequantize_mxfp4(q), dequantize_mxfp4(z)) for q, z in zip(qs, zero))
    check_status()


def test_kernel_choices_may_change_between_calls_of_another_thread(dev, libffnk):
    # the overrides and the SM margin are process-wide: a call looks each up once and goes by what it saw
    K, N = 520, 1032
    (b1, b2), vs = weights([(N, K)] * 2, 5, dev)
    qs, ws = ffn_weights(K, 264, 6, dev)
    cases = []
    for M in (1, 3, 8, 130):
        x, mask = spread(M, K, M), edge_mask(M, "alternating")
        cases.append((x.to(dev), mask.to(dev), R.linear(x, *vs, mask), R.ffn(x, ws, mask)))
    stop = threading.Event()

    def change():
        i = 0
        while not stop.is_set():
            i += 1
            libffnk.ffnk_set_sm_margin(i * 37 % 140)
            libffnk.ffnk_tune_override(b"narrow", (-1, 0, -1, 1)[i % 4])
            time.sleep(1e-5)

    other = threading.Thread(target=change)
    other.start()
    try:
        got = [(MXFP4MaskedLinear.apply(x, b1, b2, m), MXFP4MaskedFFN.apply(x, *qs, m)) for _ in range(200) for x, m, *_ in cases]
    finally:
        stop.set()
        other.join()
        libffnk.ffnk_set_sm_margin(0)
        libffnk.ffnk_tune_override(b"narrow", -1)
    check_status()
    for i, (y, f) in enumerate(got):
        inside(y, cases[i % 4][2])
        inside(f, cases[i % 4][3])


def test_a_replayed_graph_is_no_part_of_a_backward_pass(dev):
    d, h, T = 136, 264, 9
    for module in (MaskedFFNModule(d, h, device=dev), MXFP4MaskedFFNModule.from_module(MaskedFFNModule(d, h, device=dev))):
        graphed = GraphedMaskedFFN(module, T)
        x, mask = spread(T, d, 1).to(dev), edge_mask(T, "span").to(dev)
        want = graphed(x, mask).clone()
        for _ in range(2):                        # an input that wants a gradient: inference all the same
            y = graphed(x.clone().requires_grad_(True), mask)
            assert torch.equal(y, want) and not y.requires_grad and not graphed.x.requires_grad
