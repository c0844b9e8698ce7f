"""The MXFP4 operators of this package as measured cases: quantisation, its inverse, and the routed
MaskedLinear / MaskedFFN whose weights (and, inside the call, activations) are held in 4 bits.

MXFP4 (the OCP microscaling format): 32 consecutive values along the contraction share one power of two,
2^E with E = floor(log2(max |x|)) - 2 held in eight bits (E + 127; 255 = the block holds an infinity or a
NaN); each value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, rounded to nearest even.

In storage a [rows, cols] matrix is ``codes`` uint8 [rows, 16 * ceil(cols / 32)] (two values a byte, the
lower index in the low half) and ``scales`` uint8 [ceil(rows / 128), ceil(cols / 128), 32, 4, 4]: the scale of
row r and block b sits at [r // 128, b // 4, r % 32, r % 128 // 32, b % 4].

Where ``own`` is false, ``run`` computes the operators in elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a handful of calibration rows through the format and back: a call of the smallest kind
        {"name": "quantize_small", "op": "quantize", "rows": 37, "cols": 200, "dim": 1, "dtype": "fp16"},
        # one [in, out] fp32 master weight of the 4096/11008 FFN, quantised along its strided dimension and read back
        {"name": "quantize_weight", "op": "quantize", "rows": 11008, "cols": 4096, "dim": 0, "dtype": "fp32"},
        # a small adapter-sized weight back to fp32, columns that end inside a block
        {"name": "dequantize_small", "op": "dequantize", "rows": 130, "cols": 72, "dtype": "fp32"},
        # one weight of the 4096/11008 FFN back to bf16, as the backward pass reads it
        {"name": "dequantize_weight", "op": "dequantize", "rows": 11008, "cols": 4096, "dtype": "bf16"},
        # serving, one token through a square projection
        {"name": "linear_1_token", "op": "linear", "M": 1, "K": 4096, "N": 4096, "mask": "visual", "train": False},
        # a short ragged prompt, a contraction that ends inside a block
        {"name": "linear_odd", "op": "linear", "M": 1000, "K": 1000, "N": 1416, "mask": "span", "train": False},
        # the framework's linear workload: 32768 tokens, 4096 x 4096
        {"name": "linear_large", "op": "linear", "M": 32768, "K": 4096, "N": 4096, "mask": "span", "train": False},
        # fine-tuning through frozen 4-bit weights: forward and the gradient of the activations
        {"name": "linear_train", "op": "linear", "M": 8192, "K": 4096, "N": 4096, "mask": "span", "train": True},
        # serving, one token through the 4096/11008 FFN
        {"name": "ffn_1_token", "op": "ffn", "M": 1, "d": 4096, "h": 11008, "mask": "text", "train": False},
        # a decoding batch of both modalities through the 1024/2816 FFN
        {"name": "ffn_127_tokens", "op": "ffn", "M": 127, "d": 1024, "h": 2816, "mask": "random", "train": False},
        # the framework's headline workload: 16384 tokens through the 4096/11008 FFN
        {"name": "ffn_large", "op": "ffn", "M": 16384, "d": 4096, "h": 11008, "mask": "span", "train": False},
        # fine-tuning through the 1024/2816 FFN with frozen 4-bit weights, an odd number of tokens
        {"name": "ffn_train", "op": "ffn", "M": 4099, "d": 1024, "h": 2816, "mask": "span", "train": True},
    ]


def _log(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v // step * step))


def draw(rng):
    op = rng.choice(["quantize", "dequantize", "linear", "linear", "ffn", "ffn"])
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 11008), "cols": _log(rng, 8, 4096), "dim": rng.choice([0, 1]),
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "dequantize":
        return {"op": op, "rows": _log(rng, 1, 11008), "cols": _log(rng, 8, 4096), "dtype": rng.choice(["bf16", "fp32"])}
    c = {"op": op, "M": _log(rng, 1, 16384), "mask": rng.choice(["span", "random", "visual", "text"]), "train": rng.random() < 0.35}
    if op == "linear":
        return {**c, "K": _log(rng, 64, 4096, 8), "N": _log(rng, 64, 4096, 8)}
    return {**c, "d": _log(rng, 64, 2048, 8), "h": _log(rng, 128, 5504, 8)}


# ------------------------------------------------------------------------------------------------ inputs
def _mask(M, kind, gen):
    if kind == "visual":
        return torch.ones(M, dtype=torch.bool, device="cuda")
    if kind == "text":
        return torch.zeros(M, dtype=torch.bool, device="cuda")
    if kind == "random":
        return torch.rand(M, device="cuda", generator=gen) < 0.5
    rng = np.random.RandomState(int(torch.randint(1 << 30, (1,), device="cuda", generator=gen).item()))
    m, at = np.zeros(M, dtype=bool), 0       # images of 576 tokens between texts of random length
    while at < M:
        at += int(rng.randint(64, 1200))
        m[at:at + 576] = True
        at += 576
    return torch.from_numpy(m).cuda()


def _stored(values):
    """Codes and scales, in storage, of a weight [rows, cols] that a program quantised when it loaded its model."""
    rows, cols = values.shape
    blocks = -(-cols // 32)
    v = torch.nn.functional.pad(values.float(), (0, blocks * 32 - cols)).view(rows, blocks, 32)
    e = torch.frexp(v.abs().amax(-1))[1].clamp(min=-124, max=130) - 3
    a = torch.ldexp(v, -e[..., None])
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=v.device)
    code = (torch.bucketize(a.abs(), grid) + (a < 0) * 8).to(torch.uint8).view(rows, -1)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    ra, ka = -(-rows // 128), -(-blocks // 4)
    s = torch.zeros(ra * 128, ka * 4, dtype=torch.uint8, device=v.device)
    s[:rows, :blocks] = (e + 127).to(torch.uint8)
    return codes, s.view(ra, 4, 32, ka, 4).permute(0, 3, 2, 1, 4).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    bf = torch.bfloat16

    def randn(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    def weight(rows, cols):
        return _stored(randn(rows, cols, std=cols ** -0.5))

    op = case["op"]
    s = {"case": dict(case)}
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        shape = (rows, cols) if case["dim"] == 1 else (cols, rows)
        # magnitudes that spread over rows and columns, as activations and weights do
        x = randn(*shape) * torch.exp2(randn(shape[0], 1)) * torch.exp2(2 * randn(1, shape[1]))
        s["x"] = x.to(DTYPES[case["dtype"]])
    elif op == "dequantize":
        s["w"] = weight(case["rows"], case["cols"])
    elif op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = (randn(M, K) * torch.exp2(randn(1, K))).to(bf)
        s["mask"] = _mask(M, case["mask"], gen)
        s["w"] = [weight(N, K) for _ in range(2)]
        s["g"] = randn(M, N).to(bf) if case["train"] else None
    else:
        M, d, h = case["M"], case["d"], case["h"]
        s["x"] = (randn(M, d) * torch.exp2(randn(1, d))).to(bf)
        s["mask"] = _mask(M, case["mask"], gen)
        s["w"] = [weight(*((d, h) if i in (1, 4) else (h, d))) for i in range(6)]     # w1 w2 w3 u1 u2 u3
        s["g"] = randn(M, d).to(bf) if case["train"] else None
    return s


# ------------------------------------------------------------------------------------------------ plain form, 32 bits
def _round4(x):
    """[rows, cols] fp32 -> (values that 4 bits hold, scale bytes [rows, blocks])."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.nn.functional.pad(x, (0, blocks * 32 - cols)).view(rows, blocks, 32)
    top = v.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(-127, 127)
    a = torch.ldexp(v.abs(), -e[..., None])
    q = 0.5 * ((a > 0.25).float() + (a >= 0.75).float() + (a > 1.25).float() + (a >= 1.75).float())
    q = q + (a > 2.5).float() + (a >= 3.5).float() + 2.0 * (a > 5.0).float()
    q = torch.ldexp(torch.where(v < 0, -q, q), e[..., None])
    return q.view(rows, -1)[:, :cols], (e + 127).to(torch.uint8)


def _block_scales(s, rows, blocks):
    """Scale bytes [rows, blocks] in the order of storage."""
    ra, ka = -(-rows // 128), -(-blocks // 4)
    t = torch.zeros(ra * 128, ka * 4, dtype=torch.uint8, device=s.device)
    t[:rows, :blocks] = s
    return t.view(ra, 4, 32, ka, 4).permute(0, 3, 2, 1, 4).contiguous()


def _values(w, rows, cols):
    """The fp32 values of a matrix in storage."""
    codes, scales = w
    ra, ka = scales.shape[:2]
    sc = scales.permute(0, 3, 2, 1, 4).reshape(ra * 128, ka * 4)[:rows, : -(-cols // 32)]
    c = torch.stack((codes & 15, codes >> 4), -1).view(rows, -1, 32)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    v = grid[(c & 7).int()] * (1.0 - 2.0 * (c >> 3).float())
    return torch.ldexp(v, sc[..., None].int() - 127).view(rows, -1)[:, :cols]


def _by_rows(x, mask, wv, wt):
    """x[m] @ (wv if mask[m] else wt).T, each token by its own modality's weight."""
    y = torch.empty(x.shape[0], wv.shape[0], device=x.device)
    iv, it = mask.nonzero()[:, 0], (~mask).nonzero()[:, 0]
    y[iv] = x[iv] @ wv.T
    y[it] = x[it] @ wt.T
    return y


def _run_plain(s):
    c = s["case"]
    op, bf = c["op"], torch.bfloat16
    if op == "quantize":
        x = s["x"].float() if c["dim"] == 1 else s["x"].float().T
        v, e = _round4(x)
        return {"values": v.to(s["x"].dtype), "scales": _block_scales(e, *e.shape)}
    if op == "dequantize":
        return {"values": _values(s["w"], c["rows"], c["cols"]).to(DTYPES[c["dtype"]])}
    mask = s["mask"]
    x = _round4(s["x"].float())[0]
    if op == "linear":
        wv, wt = (_values(w, c["N"], c["K"]) for w in s["w"])
        out = {"y": _by_rows(x, mask, wv, wt).to(bf)}
        if c["train"]:
            out["dx"] = _by_rows(s["g"].float(), mask, wv.T, wt.T).to(bf)
        return out
    d, h = c["d"], c["h"]
    w1, w2, w3, u1, u2, u3 = (_values(w, *((d, h) if i in (1, 4) else (h, d))) for i, w in enumerate(s["w"]))
    t1, t3 = _by_rows(x, mask, w1, u1), _by_rows(x, mask, w3, u3)
    sg = 1.0 / (1.0 + torch.exp(-t1))
    out = {"y": _by_rows(_round4(t1 * sg * t3)[0], mask, w2, u2).to(bf)}
    if c["train"]:
        dh = _by_rows(s["g"].float(), mask, w2.T, u2.T)      # the rounding to 4 bits counts as the identity
        d1, d3 = dh * t3 * sg * (1.0 + t1 * (1.0 - sg)), dh * t1 * sg
        out["dx"] = (_by_rows(d1, mask, w1.T, u1.T) + _by_rows(d3, mask, w3.T, u3.T)).to(bf)
    return out


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    import ffn_kernel_b200 as F
    c = s["case"]
    op = c["op"]
    if op == "quantize":
        q = F.quantize_mxfp4(s["x"], dim=c["dim"])
        return {"values": F.dequantize_mxfp4(q, dtype=s["x"].dtype), "scales": q.scales}
    if op == "dequantize":
        q = F.MXFP4Tensor(*s["w"], c["rows"], c["cols"])
        return {"values": F.dequantize_mxfp4(q, dtype=DTYPES[c["dtype"]])}
    if op == "linear":
        fn, ws = F.MXFP4MaskedLinear, [F.MXFP4Tensor(*w, c["N"], c["K"]) for w in s["w"]]
    else:
        d, h = c["d"], c["h"]
        fn = F.MXFP4MaskedFFN
        ws = [F.MXFP4Tensor(*w, *((d, h) if i in (1, 4) else (h, d))) for i, w in enumerate(s["w"])]
    if not c["train"]:
        return {"y": fn.apply(s["x"], *ws, s["mask"])}
    x = s["x"].detach().requires_grad_(True)
    y = fn.apply(x, *ws, s["mask"])
    return {"y": y.detach(), "dx": torch.autograd.grad(y, x, s["g"])[0]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ what it costs
def work(case):
    op = case["op"]

    def held(rows, cols):          # bytes of a matrix in 4 bits with its scales
        return rows * (-(-cols // 32)) * 17

    if op == "quantize":           # read the values, write codes and scales; read those, write the values back
        n = case["rows"] * case["cols"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * n * size + 2 * held(case["rows"], case["cols"]), "flops": 0}
    if op == "dequantize":
        n = case["rows"] * case["cols"]
        return {"bytes": held(case["rows"], case["cols"]) + n * (4 if case["dtype"] == "fp32" else 2), "flops": 0}
    M, present = case["M"], 1 if case["mask"] in ("visual", "text") or case["M"] == 1 else 2
    if op == "linear":
        K, N = case["K"], case["N"]
        b, f = M * K * 2 + M * N * 2 + M + present * held(N, K), 2.0 * M * K * N
        if case["train"]:
            b, f = b + M * N * 2 + M * K * 2 + present * held(N, K), 2 * f
        return {"bytes": b, "flops": f}
    d, h = case["d"], case["h"]
    weights = present * (2 * held(h, d) + held(d, h))
    b, f = M * d * 4 + M + weights, 6.0 * M * d * h
    if case["train"]:
        b, f = b + M * d * 4 + weights, 2 * f
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------------------ 64 bits, from the definition
def _two64(e):
    """2^e as float64, exact (its bits): a power function may be a unit in the last place off."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest4(x):
    """The value of the format nearest to each x (float64), ties to even, and the block exponents."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    out = torch.zeros(rows, blocks * 32, dtype=torch.float64, device=x.device)
    out[:, :cols] = x
    out = out.reshape(rows * blocks, 32)
    top = out.abs().max(dim=1).values
    m, ex = torch.frexp(top)
    E = torch.where(top == 0, torch.full_like(ex, -127), ex - 1 - 2).clamp(-127, 127)
    r = out * _two64(-E)[:, None]
    # spacing of the grid around r: 0.5 below 2, 1 below 4, 2 from there
    step = torch.where(r.abs() < 2, 0.5, torch.where(r.abs() < 4, 1.0, 2.0)).double()
    q = (torch.round(r / step) * step).clamp(-6, 6)
    q = q * _two64(E)[:, None]
    return q.reshape(rows, -1)[:, :cols], (E + 127).reshape(rows, blocks)


def _read64(w, rows, cols):
    codes, scales = w
    i = torch.arange(cols, device=codes.device)
    nib = (codes[:, i // 2].int() >> (4 * (i % 2)).int()) & 15
    mag, ex = (nib & 1).double(), ((nib >> 1) & 3).double()
    v = torch.where(ex == 0, mag / 2, (1 + mag / 2) * _two64(ex - 1))
    v = torch.where(nib >= 8, -v, v)
    r = torch.arange(rows, device=codes.device)[:, None]
    b = (i // 32)[None, :]
    sc = scales[r // 128, b // 4, r % 32, r % 128 // 32, b % 4].long()
    return v * _two64(sc - 127)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = s["x"].double() if case["dim"] == 1 else s["x"].double().t()
        v, e = _nearest4(x)
        rows, blocks = e.shape
        sc = torch.zeros(-(-rows // 128), -(-blocks // 4), 32, 4, 4, dtype=torch.uint8, device=x.device)
        r, b = torch.arange(rows, device=x.device)[:, None], torch.arange(blocks, device=x.device)[None, :]
        sc[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = e.to(torch.uint8)
        return {"values": v, "scales": sc}
    if op == "dequantize":
        return {"values": _read64(s["w"], case["rows"], case["cols"])}
    x, m = _nearest4(s["x"].double())[0], s["mask"]

    def times(a, wv, wt):
        y = torch.zeros(a.shape[0], wv.shape[1], dtype=torch.float64, device=a.device)
        y[m] = a[m] @ wv
        y[~m] = a[~m] @ wt
        return y

    if op == "linear":
        wv, wt = (_read64(w, case["N"], case["K"]) for w in s["w"])
        out = {"y": times(x, wv.t(), wt.t())}
        if case["train"]:
            out["dx"] = times(s["g"].double(), wv, wt)
        return out
    d, h = case["d"], case["h"]
    w1, w2, w3, u1, u2, u3 = (_read64(w, *((d, h) if i in (1, 4) else (h, d))) for i, w in enumerate(s["w"]))
    a, b = times(x, w1.t(), u1.t()), times(x, w3.t(), u3.t())
    sig = torch.sigmoid(a)
    out = {"y": times(_nearest4(a * sig * b)[0], w2.t(), u2.t())}
    if case["train"]:
        gh = times(s["g"].double(), w2, u2)
        da, db = gh * b * (sig + a * sig * (1 - sig)), gh * a * sig
        out["dx"] = times(da, w1, u1) + times(db, w3, u3)
    return out
