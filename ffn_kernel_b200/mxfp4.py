"""MXFP4: 4-bit floating point with one power-of-two scale per 32 values, and the routed operators on it.

The reference computes in bf16 only; this module adds the same two layers with weights held in 4 bits (4.25
bits a value with its share of the scales) and multiplied on the 4-bit tensor-core path:

``quantize_mxfp4(x, dim)`` / ``dequantize_mxfp4(q, dtype)``  a matrix into the format and back,
``MXFP4MaskedLinear.apply(a, q1, q2, mask)``                 ``MaskedLinear`` on 4-bit weights,
``MXFP4MaskedFFN.apply(a, q_w1, ..., q_u3, mask)``           ``MaskedFFN`` on 4-bit weights.

Activations come and go in bf16 and are quantised inside the call, row by row in blocks of 32 along the contraction: no
token's values reach another's result.  The number of tokens chooses the kernel, and with it the order of the fp32 sums, so
between batches of different sizes the last bits may differ (in the FFN a hidden value next to a tie by its 4-bit step).
Gradients reach the activations (the rounding to 4 bits counts as the identity); the weights are frozen.  A block that
holds an infinity or a NaN reads back as NaN.
"""
from __future__ import annotations

import struct
from functools import lru_cache

import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from ._lib import check, lib
from .linear import _activation, _check_dims
from .route import _require_cuda, maybe_check, status_word, stream_ptr

__all__ = ["MXFP4Tensor", "quantize_mxfp4", "dequantize_mxfp4", "MXFP4MaskedLinear", "MXFP4MaskedFFN"]

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_six = struct.Struct("6P").pack        # a host array of six pointers


@lru_cache(maxsize=1024)
def _workspace_bytes(M: int, K: int, h: int) -> int:
    return lib().ffnk_mxfp4_workspace_bytes(M, K, h)


@lru_cache(maxsize=1024)
def _backward_bytes(M: int, K: int, N: int, h: int) -> int:
    return lib().ffnk_mxfp4_backward_workspace_bytes(M, K, N, h)


def _elsewhere(dev) -> bool:
    """Is ``dev`` another device than the current one?  (Then the call is made again with it current.)"""
    return torch.cuda.current_device() != dev.index


def _rows(t, name):
    """``_activation`` with the common case, a contiguous matrix with 16-byte rows, decided at once."""
    if (isinstance(t, torch.Tensor) and t.dtype is torch.bfloat16 and t.is_cuda and t.dim() == 2 and t.is_contiguous()
            and not t.shape[1] & 7 and not t.data_ptr() & 15):
        return t
    t = _activation(t, name)
    # a single row at an odd address counts as contiguous and comes back as it was
    return t.clone() if t.data_ptr() & 15 else t


def _ld(t) -> int:
    """Elements from one row to the next; the stride of a single row may be anything."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class MXFP4Tensor:
    """A matrix [rows, cols] in MXFP4, blocks of 32 along the columns (the contraction: a weight is [out, in]).

    codes   uint8 [rows, 16 * ceil(cols / 32)], two values a byte, the lower column in the low half
    scales  uint8 [ceil(rows / 128), ceil(cols / 128), 32, 4, 4]; 2^(byte - 127) of (row r, block b) sits at
            [r // 128, b // 4, r % 32, r % 128 // 32, b % 4]; entries without a row or block are 0 (they are not looked
            at but for one: with an odd number of blocks a 255 in the block after the last makes products NaN)
    """
    __slots__ = ("_codes", "_scales", "_rows", "_cols", "_device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int):
        try:
            device = codes.device
            ok = (codes.dtype is torch.uint8 and scales.dtype is torch.uint8 and codes.is_cuda and scales.device == device
                  and codes.shape == (rows, (cols + 31) // 32 * 16)
                  and scales.shape == ((rows + 127) // 128, (cols + 127) // 128, 32, 4, 4)
                  and codes.is_contiguous() and scales.is_contiguous() and not (codes.data_ptr() | scales.data_ptr()) & 15)
        except AttributeError:
            ok = False
        if not ok:
            raise RuntimeError(
                f"an MXFP4 matrix [{rows}, {cols}] takes codes torch.uint8 [{rows}, {-(-cols // 32) * 16}] and scales torch.uint8 "
                f"[{-(-rows // 128)}, {-(-cols // 128)}, 32, 4, 4], both contiguous, 16-byte aligned and on one CUDA device; got "
                + " and ".join(f"{t.dtype} {list(t.shape)} strides {list(t.stride())} on {t.device}" if isinstance(t, torch.Tensor)
                               else type(t).__name__ for t in (codes, scales)))
        self._codes, self._scales, self._rows, self._cols, self._device = codes, scales, rows, cols, device

    # the fields have been checked against one another: they can be read, not replaced
    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    rows = property(lambda self: self._rows)
    cols = property(lambda self: self._cols)
    device = property(lambda self: self._device)
    shape = property(lambda self: (self._rows, self._cols))

    def _ptrs(self):
        return self._codes.data_ptr(), self._scales.data_ptr()

    def __reduce__(self):
        return MXFP4Tensor, (self._codes, self._scales, self._rows, self._cols)

    def __repr__(self):
        return f"MXFP4Tensor([{self.rows}, {self.cols}], device={self.codes.device})"


def quantize_mxfp4(x: torch.Tensor, dim: int = 1) -> MXFP4Tensor:
    """``x`` (2-D; bf16, fp16 or fp32) with blocks along ``dim``.  The result's columns are ``x``'s dimension
    ``dim`` and it carries no gradient: an ``nn.Linear`` weight [out, in] is quantised along 1, its ``.T`` view or an [in, out] weight along 0."""
    _require_cuda(x, "x")
    if x.dim() != 2:
        raise RuntimeError(f"x must be 2-D, got shape {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"x must be torch.bfloat16, torch.float16 or torch.float32, got {x.dtype}")
    if dim not in (0, 1, -1, -2):
        raise RuntimeError(f"dim must be 0 or 1, got {dim}")
    rows, cols = x.shape
    rs, cs = x.stride()
    if not (cs == 1 or cols == 1 or rs == 1 or rows == 1):
        x = x.contiguous()
        rs, cs = cols, 1
    if dim in (0, -2):
        rows, cols, rs, cs = cols, rows, cs, rs
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return quantize_mxfp4(x, 1 if dim in (1, -1) else 0)
    codes = torch.empty(rows, -(-cols // 32) * 16, dtype=torch.uint8, device=dev)
    scales = torch.empty(-(-rows // 128), -(-cols // 128), 32, 4, 4, dtype=torch.uint8, device=dev)
    q = MXFP4Tensor.__new__(MXFP4Tensor)
    q._codes, q._scales, q._rows, q._cols, q._device = codes, scales, rows, cols, dev
    check("ffnk_mxfp4_quantize", lib().ffnk_mxfp4_quantize(
        x.data_ptr(), _DTYPES[x.dtype], rs, cs, rows, cols, *q._ptrs(), stream_ptr(dev)))
    return q


def dequantize_mxfp4(q: MXFP4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The matrix [rows, cols] that ``q`` stands for: exact in bf16 and fp32, rounded to nearest in fp16."""
    if not isinstance(q, MXFP4Tensor):
        raise RuntimeError(f"q must be an MXFP4Tensor, got {type(q).__name__}")
    if dtype not in _DTYPES:
        raise RuntimeError(f"dtype must be torch.bfloat16, torch.float16 or torch.float32, got {dtype}")
    dev = q.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return dequantize_mxfp4(q, dtype)
    out = torch.empty(q.rows, q.cols, dtype=dtype, device=dev)
    check("ffnk_mxfp4_dequantize", lib().ffnk_mxfp4_dequantize(
        *q._ptrs(), q.rows, q.cols, out.data_ptr(), _DTYPES[dtype], q.cols, stream_ptr(dev)))
    return out


def _check_weights(ws, names, shapes, dev):
    for w, n, s in zip(ws, names, shapes):
        if not isinstance(w, MXFP4Tensor):
            raise RuntimeError(f"{n} must be an MXFP4Tensor, got {type(w).__name__}")
        if w._rows != s[0] or w._cols != s[1]:
            raise RuntimeError(f"{n} must have shape {list(s)} ([out, in]), got [{w.rows}, {w.cols}]")
        if w._device != dev:
            raise RuntimeError(f"{n} must be on the same device as the activations")


def _check_mask(mask, M, dev):
    if not isinstance(mask, torch.Tensor) or mask.dim() != 1 or mask.shape[0] != M or mask.device != dev:
        raise RuntimeError(f"mask must have shape [{M}] on {dev}")
    if mask.dtype is not torch.bool and mask.dtype is not torch.uint8:
        raise RuntimeError(f"mask must be torch.bool (or uint8), got {mask.dtype}")
    return mask if mask.is_contiguous() else mask.contiguous()


@lru_cache(maxsize=1024)
def _kept_bytes(M: int, h: int) -> int:
    return lib().ffnk_mxfp4_kept_bytes(M, h)


def _scratch(nbytes, M, dev, keep: bool, factors: int = 0):
    """Workspace, and the routing lists (perm int32 [2 * cap], counts int32 [8]) of one call -> (tensors to hold, workspace,
    perm, counts).  Inference takes one allocation for both; what a backward pass wants, the lists behind ``factors``
    bytes, gets one of its own."""
    cap = (M + 127) // 128 * 128
    if keep:
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        kept = torch.empty(factors + 8 * cap + 32, device=dev, dtype=torch.uint8)
        p = kept.data_ptr() + factors
        return ws, kept, ws.data_ptr(), p, p + 8 * cap
    ws = torch.empty(nbytes + 8 * cap + 32, device=dev, dtype=torch.uint8)
    p = ws.data_ptr()
    return ws, None, p, p + nbytes, p + nbytes + 8 * cap


def _lists(kept, M):
    """(perm, counts) at the end of what ``_scratch`` keeps."""
    p = kept.data_ptr() + kept.numel() - 32
    return p - 8 * ((M + 127) // 128 * 128), p


def _mxfp4_linear_forward(a, b1, b2, mask, keep: bool = False):
    """y[m] = Q(a[m]) @ (b1 if mask[m] else b2).T -> (y [M, N] bf16, with ``keep`` what the backward pass needs)."""
    a = _rows(a, "a")
    M, K = a.shape
    dev = a.device
    N = b1.rows if isinstance(b1, MXFP4Tensor) else -1
    _check_weights((b1, b2), ("b1", "b2"), ((N, K), (N, K)), dev)
    if K & 7 or N & 7 or not K or not N:
        _check_dims(K=K, N=N)
    mask = _check_mask(mask, M, dev)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _mxfp4_linear_forward(a, b1, b2, mask, keep)
    y = a.new_empty(M, N)
    if M == 0:
        return y, None
    nbytes = _workspace_bytes(M, K, 0)
    ws, kept, wp, perm, counts = _scratch(nbytes, M, dev, keep)
    check("ffnk_mxfp4_linear_forward", lib().ffnk_mxfp4_linear_forward(
        a.data_ptr(), _ld(a), *b1._ptrs(), *b2._ptrs(), mask.data_ptr(), perm, counts, wp, nbytes, y.data_ptr(), N, M, N, K,
        status_word(dev).data_ptr(), stream_ptr(dev)))
    maybe_check(dev)
    return y, kept


def _mxfp4_linear_backward(g, b1, b2, kept):
    """dx[m] = g[m] @ (b1 if mask[m] else b2)."""
    g = _rows(g, "grad")
    M, (N, K) = g.shape[0], b1.shape
    dev = g.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _mxfp4_linear_backward(g, b1, b2, kept)
    dx = g.new_empty(M, K)
    if M == 0:
        return dx
    nbytes = _backward_bytes(M, K, N, 0)
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    check("ffnk_mxfp4_linear_backward", lib().ffnk_mxfp4_linear_backward(
        g.data_ptr(), _ld(g), *b1._ptrs(), *b2._ptrs(), *_lists(kept, M), ws.data_ptr(), nbytes, dx.data_ptr(), K, M, N, K,
        status_word(dev).data_ptr(), stream_ptr(dev)))
    maybe_check(dev)
    return dx


_FFN_NAMES = ("w1", "w2", "w3", "u1", "u2", "u3")


def _mxfp4_ffn_forward(x, ws6, mask, keep: bool):
    """The whole FFN forward -> (y [M, d] bf16, with ``keep`` what the backward pass needs)."""
    x = _rows(x, "x")
    M, d = x.shape
    dev = x.device
    h = ws6[0].rows if isinstance(ws6[0], MXFP4Tensor) else -1
    _check_weights(ws6, _FFN_NAMES, ((h, d), (d, h), (h, d), (h, d), (d, h), (h, d)), dev)
    if d & 7 or h & 7 or not d or not h:
        _check_dims(d=d, h=h)
    mask = _check_mask(mask, M, dev)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _mxfp4_ffn_forward(x, ws6, mask, keep)
    L = lib()
    y = x.new_empty(M, d)
    if M == 0:
        return y, None
    nbytes = _workspace_bytes(M, d, h)
    n = _kept_bytes(M, h) if keep else 0
    ws, kept, wp, perm, counts = _scratch(nbytes, M, dev, keep, 2 * n)
    f1 = f3 = None
    if keep:
        f1 = kept.data_ptr()
        f3 = f1 + n
    check("ffnk_mxfp4_ffn_forward", L.ffnk_mxfp4_ffn_forward(
        x.data_ptr(), _ld(x), _six(*[w._codes.data_ptr() for w in ws6]), _six(*[w._scales.data_ptr() for w in ws6]), mask.data_ptr(), perm,
        counts, wp, nbytes, f1, f3, y.data_ptr(), d, M, d, h, status_word(dev).data_ptr(), stream_ptr(dev)))
    maybe_check(dev)
    return y, kept


def _mxfp4_ffn_backward(gy, ws6, kept):
    """Gradient of the activations."""
    gy = _rows(gy, "grad")
    M, (h, d) = gy.shape[0], ws6[0].shape
    dev = gy.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _mxfp4_ffn_backward(gy, ws6, kept)
    dx = gy.new_empty(M, d)
    if M == 0:
        return dx
    nbytes = _backward_bytes(M, d, d, h)
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    f1 = kept.data_ptr()
    check("ffnk_mxfp4_ffn_backward", lib().ffnk_mxfp4_ffn_backward(
        gy.data_ptr(), _ld(gy), _six(*[w._codes.data_ptr() for w in ws6]), _six(*[w._scales.data_ptr() for w in ws6]), f1,
        f1 + _kept_bytes(M, h), *_lists(kept, M), ws.data_ptr(), nbytes, dx.data_ptr(), d, M, d, h,
        status_word(dev).data_ptr(), stream_ptr(dev)))
    maybe_check(dev)
    return dx


def _wants_grad(a) -> bool:
    """Does this call go through autograd?  (Under forward-mode differentiation too, for its refusal; where torch no longer
    tells the level, always: right as well, but slower.)"""
    return isinstance(a, torch.Tensor) and (a.requires_grad and torch.is_grad_enabled()
                                            or getattr(forward_ad, "_current_level", 0) >= 0)


def _storage(ws):
    """The weights' tensors, saved so that a change between the forward and the backward pass is noticed (one made in
    inference mode has no version to compare and cannot be saved)."""
    return [t for w in ws for t in (w._codes, w._scales) if not t.is_inference()]


class MXFP4MaskedLinear(Function):
    """``MXFP4MaskedLinear.apply(a, b1, b2, mask)``: ``Q(a[m]) @ b1.T`` where ``mask[m]`` else ``Q(a[m]) @ b2.T``.

    a [M, K] bf16; b1 (visual), b2 (text): ``MXFP4Tensor`` [N, K], the ``nn.Linear`` weights quantised.  Gradient
    of ``a`` only."""

    @classmethod
    def apply(cls, a, b1, b2, mask):
        return super().apply(a, b1, b2, mask) if _wants_grad(a) else _mxfp4_linear_forward(a, b1, b2, mask)[0]

    @staticmethod
    def forward(ctx, a, b1, b2, mask):
        y, kept = _mxfp4_linear_forward(a, b1, b2, mask, keep=True)
        ctx.save_for_backward(kept, *_storage((b1, b2)))
        ctx.weights = (b1, b2)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _mxfp4_linear_backward(grad, *ctx.weights, ctx.saved_tensors[0]), None, None, None


class MXFP4MaskedFFN(Function):
    """``MXFP4MaskedFFN.apply(a, w1, w2, w3, u1, u2, u3, mask)``: the routed SwiGLU FFN on 4-bit weights.

    y = Q(silu(Q(a) w1.T) * (Q(a) w3.T)) w2.T for visual tokens, u* for text tokens; the weights are ``MXFP4Tensor``
    in ``nn.Linear`` order (w1, w3, u1, u3 [h, d]; w2, u2 [d, h]).  Gradient of ``a`` only."""

    @classmethod
    def apply(cls, a, w1, w2, w3, u1, u2, u3, mask):
        if _wants_grad(a):
            return super().apply(a, w1, w2, w3, u1, u2, u3, mask)
        return _mxfp4_ffn_forward(a, (w1, w2, w3, u1, u2, u3), mask, keep=False)[0]

    @staticmethod
    def forward(ctx, a, w1, w2, w3, u1, u2, u3, mask):
        ctx.weights = (w1, w2, w3, u1, u2, u3)
        y, kept = _mxfp4_ffn_forward(a, ctx.weights, mask, keep=True)
        ctx.save_for_backward(kept, *_storage(ctx.weights))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return (_mxfp4_ffn_backward(grad, ctx.weights, ctx.saved_tensors[0]), *([None] * 7))
