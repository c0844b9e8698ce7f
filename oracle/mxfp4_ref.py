"""64-bit CPU restatement of the MXFP4 format and of the routed operators on it.

Written from the definition of the format (blocks of 32 along the contraction, E = floor(log2 max|x|) - 2, values
0, 0.5, 1, 1.5, 2, 3, 4, 6 rounded to nearest even) and from the operators' formulas; no code of the package.
"""
from __future__ import annotations

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def two(e: torch.Tensor) -> torch.Tensor:
    """2^e in float64, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _blocks(x):
    rows, cols = x.shape
    nb = -(-cols // 32)
    p = torch.zeros(rows, nb * 32, dtype=torch.float64)
    p[:, :cols] = x.double()
    return p.view(rows, nb, 32)


def exponent(x: torch.Tensor) -> torch.Tensor:
    """E of every block of x [rows, cols] -> [rows, blocks]; 128 marks a block that is not finite."""
    top = _blocks(x).abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, torch.tensor(-127)).clamp(-127, 127)
    return torch.where(torch.isfinite(top), e, torch.tensor(128))


def to_grid(x: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """x rounded to the grid of the block exponents e [rows, blocks], as code 0..15 [rows, 32 * blocks]."""
    b = _blocks(x)
    finite = (e < 128)[..., None]
    r = torch.where(finite, b, torch.zeros(())) * two(-e.clamp(max=127))[..., None]
    d = (r.abs()[..., None] - GRID).abs()
    near = d.amin(-1, keepdim=True)
    # ties to even: of two magnitudes at the same distance the one with an even code
    cand = d == near
    even = cand & (torch.arange(8) % 2 == 0)
    pick = torch.where(even.any(-1, keepdim=True), even, cand)
    code = pick.double().argmax(-1)
    code = code + 8 * torch.signbit(b).long()
    return torch.where(finite, code, torch.zeros((), dtype=torch.long)).flatten(1)


def pack(code: torch.Tensor, e: torch.Tensor):
    """codes and scales in the layout of storage."""
    rows, nb = e.shape
    c = code.to(torch.uint8)
    codes = c[:, 0::2] | (c[:, 1::2] << 4)
    scales = torch.zeros(-(-rows // 128), -(-nb // 4), 32, 4, 4, dtype=torch.uint8)
    r, b = torch.arange(rows)[:, None], torch.arange(nb)[None, :]
    scales[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = (e + 127).to(torch.uint8)
    return codes, scales


def quantize(x: torch.Tensor):
    e = exponent(x)
    return pack(to_grid(x, e), e)


def values(codes, scales, rows, cols) -> torch.Tensor:
    """float64 values of a matrix in storage."""
    codes, scales = codes.cpu(), scales.cpu()
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(rows, -1)[:, :cols].long()
    v = GRID[c & 7] * torch.where(c >= 8, -1.0, 1.0)
    r, b = torch.arange(rows)[:, None], (torch.arange(cols) // 32)[None, :]
    s = scales[r // 128, b // 4, r % 32, r % 128 // 32, b % 4].long()
    return torch.where(s == 255, torch.tensor(float("nan"), dtype=torch.float64), v * two(s - 127))


def rounded(x: torch.Tensor, e: torch.Tensor | None = None) -> torch.Tensor:
    """x through the format and back, float64; NaN where the block is not finite."""
    e = exponent(x) if e is None else e
    code = to_grid(x, e)
    v = GRID[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    s = e.repeat_interleave(32, 1)
    v = torch.where(s == 128, torch.tensor(float("nan"), dtype=torch.float64), v * two(s.clamp(max=127)))
    return v[:, : x.shape[1]]


def by_rows(x, mask, wv, wt):
    """x[m] @ (wv if mask[m] else wt), float64."""
    m = mask.bool()
    y = torch.zeros(x.shape[0], wv.shape[1], dtype=torch.float64)
    y[m] = x[m].double() @ wv
    y[~m] = x[~m].double() @ wt
    return y


U16, U32 = 2.0 ** -8, 2.0 ** -24      # half a step of bf16 and of fp32


def linear(x, wv, wt, mask):
    """Forward on float64 weights [N, K] -> (y, bound on |computed - y|).

    The products are exact; K of them are added in fp32 in some order, each addition off by at most a whole step
    2 * U32 of the sum of magnitudes (tensor cores may cut instead of round); the result is rounded to bf16."""
    q = rounded(x.cpu().double())
    y = by_rows(q, mask, wv.T, wt.T)
    s = by_rows(q.abs(), mask, wv.T.abs(), wt.T.abs())
    acc = 2 * U32 * x.shape[1] * s
    return y, U16 * (y.abs() + acc) + acc + 2.0 ** -133


def linear_dx(g, wv, wt, mask):
    y = by_rows(g.cpu().double(), mask, wv, wt)
    acc = 2 * U32 * g.shape[1] * by_rows(g.cpu().double().abs(), mask, wv.abs(), wt.abs())
    return y, U16 * (y.abs() + acc) + acc + 2.0 ** -133


def ffn(x, w, mask):
    """Forward on float64 weights (w1, w2, w3, u1, u2, u3) in nn.Linear order -> (y, bound).

    The hidden value is known to within `dh` (fp32 sums of t1 and t3, the exponential and the reciprocal: 16 * U32
    relative is ample for both), so it may round to a neighbour on the 4-bit grid, or its block may take the
    neighbouring exponent, exactly where that interval crosses a tie or a power of two."""
    w1, w2, w3, u1, u2, u3 = w
    q = rounded(x.cpu().double())
    t1, t3 = by_rows(q, mask, w1.T, u1.T), by_rows(q, mask, w3.T, u3.T)
    e1 = 2 * U32 * q.shape[1] * by_rows(q.abs(), mask, w1.T.abs(), u1.T.abs())
    e3 = 2 * U32 * q.shape[1] * by_rows(q.abs(), mask, w3.T.abs(), u3.T.abs())
    s = torch.sigmoid(t1)
    silu, dsilu = t1 * s, s * (1 + t1 * (1 - s))
    hid = silu * t3
    dh = (dsilu * t3).abs() * e1 + silu.abs() * e3 + 1.1 * e1 * e3 + 16 * U32 * hid.abs() * (1 + t1.abs() / 8) + 2.0 ** -126
    hq = rounded(hid)
    far = torch.zeros_like(hid)
    lo, hi = (hid.abs() - dh).clamp(min=0), hid.abs() + dh
    for e in (exponent(lo), exponent(hi)):
        for v in (hid - dh, hid + dh):
            far = torch.maximum(far, (rounded(v, e) - hq).abs())
    y = by_rows(hq, mask, w2.T, u2.T)
    off = by_rows(far, mask, w2.T.abs(), u2.T.abs())
    off = off + 2 * U32 * hid.shape[1] * by_rows(hq.abs() + far, mask, w2.T.abs(), u2.T.abs())
    return y, off + U16 * (y.abs() + off) + 2.0 ** -133


def ffn_dx(g, x, w, mask):
    """Gradient of the activations, the roundings to 4 bits counting as the identity -> (dx, bound).

    On the way: the factors f1 = dh/dt1 and f3 = dh/dt3 from fp32 t1, t3 and the exponential (as in `ffn`), kept in
    fp16 with a shared power of two per 32 (half a step 2^-11 relative, and 2^-39 of the block's largest below its
    normal range); dH in fp32; dT1, dT3 rounded to bf16; fp32 sums; dx rounded to bf16."""
    w1, w2, w3, u1, u2, u3 = w
    q = rounded(x.cpu().double())
    g = g.cpu().double()
    t1, t3 = by_rows(q, mask, w1.T, u1.T), by_rows(q, mask, w3.T, u3.T)
    s = torch.sigmoid(t1)
    dh = by_rows(g, mask, w2, u2)
    edh = 2 * U32 * g.shape[1] * by_rows(g.abs(), mask, w2.abs(), u2.abs())
    f1, f3 = t3 * s * (1 + t1 * (1 - s)), t1 * s
    d1, d3 = dh * f1, dh * f3
    et = 2 * U32 * q.shape[1]
    et1 = et * by_rows(q.abs(), mask, w1.T.abs(), u1.T.abs())
    et3 = et * by_rows(q.abs(), mask, w3.T.abs(), u3.T.abs())
    # silu'(t1) is below 1.1, its slope below 0.5; 16 * U32 relative (and 2 * U32 |t1| from the exponential) of the terms
    fine = 16 * U32 * (1 + t1.abs() / 8)
    ef1 = 1.1 * et3 + 0.5 * (t3.abs() + et3) * et1 + fine * t3.abs() * (s + t1.abs() * s * (1 - s))
    ef3 = 1.1 * et1 + fine * f3.abs()
    top1, top3 = (_blocks(f).abs().amax(-1).repeat_interleave(32, 1)[:, : f.shape[1]] for f in (f1, f3))
    ef1 = ef1 + 2.0 ** -11 * (f1.abs() + ef1) + 2.0 ** -38 * top1 + 2.0 ** -126
    ef3 = ef3 + 2.0 ** -11 * (f3.abs() + ef3) + 2.0 ** -38 * top3 + 2.0 ** -126
    off1 = dh.abs() * ef1 + edh * (f1.abs() + ef1)
    off3 = dh.abs() * ef3 + edh * (f3.abs() + ef3)
    off1 = off1 + U16 * (d1.abs() + off1) + 8 * U32 * d1.abs() + 2.0 ** -126
    off3 = off3 + U16 * (d3.abs() + off3) + 8 * U32 * d3.abs() + 2.0 ** -126
    dx = by_rows(d1, mask, w1, u1) + by_rows(d3, mask, w3, u3)
    off = by_rows(off1, mask, w1.abs(), u1.abs()) + by_rows(off3, mask, w3.abs(), u3.abs())
    mag = by_rows(d1.abs() + off1, mask, w1.abs(), u1.abs()) + by_rows(d3.abs() + off3, mask, w3.abs(), u3.abs())
    off = off + 4 * U32 * d1.shape[1] * mag
    return dx, off + U16 * (dx.abs() + off) + 2.0 ** -133
