"""The MXFP4 operators without a GPU: the oracle against the format's definition, and every refusal."""
import ctypes

import pytest
import torch

from ffn_kernel_b200 import (MXFP4MaskedFFN, MXFP4MaskedFFNModule, MXFP4MaskedLinear, MXFP4MaskedLinearModule, MXFP4Tensor,
                             dequantize_mxfp4, quantize_mxfp4)
from oracle import mxfp4_ref as R


def test_oracle_rounds_ties_to_even_and_saturates():
    x = torch.tensor([[6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, -0.25, 0.26, 7.9]], dtype=torch.float64)
    want = [[6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -4.0, -0.0, 0.5, 6.0]]
    assert R.rounded(x).tolist() == want
    assert R.exponent(x).tolist() == [[0]]


def test_oracle_special_blocks():
    x = torch.zeros(1, 160, dtype=torch.float64)
    x[0, 32] = 2.0 ** -130            # smaller than any block exponent reaches
    x[0, 64] = float("inf")
    x[0, 96] = float("nan")
    x[0, 128] = 3.0e38
    e = R.exponent(x)
    assert e.tolist() == [[-127, -127, 128, 128, 125]]
    v = R.rounded(x)
    assert torch.isnan(v[0, 64:128]).all() and torch.isfinite(v[0, :64]).all() and torch.isfinite(v[0, 128:]).all()
    codes, scales = R.quantize(x)
    back = R.values(codes, scales, 1, 160)
    assert torch.equal(torch.nan_to_num(back, nan=-1.0), torch.nan_to_num(v, nan=-1.0))


def test_sizes_of_storage(libffnk):
    L = libffnk
    assert L.ffnk_mxfp4_code_bytes(130, 72) == 130 * 48
    assert L.ffnk_mxfp4_scale_bytes(130, 72) == 2 * 512
    assert L.ffnk_mxfp4_scale_bytes(128, 129) == 2 * 512
    assert L.ffnk_mxfp4_code_bytes(-1, 8) < 0 and L.ffnk_mxfp4_scale_bytes(8, 1 << 30) < 0
    assert L.ffnk_mxfp4_workspace_bytes(0, 64, 0) > 0
    assert L.ffnk_mxfp4_workspace_bytes(1, 64, 64) > L.ffnk_mxfp4_workspace_bytes(1, 64, 0)


def test_argument_errors_are_reported_before_any_launch(libffnk):
    L, p, odd = libffnk, ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1008)
    six, six_odd, holes = (ctypes.c_void_p * 6)(*[0x1000] * 6), (ctypes.c_void_p * 6)(*[0x1008] * 6), (ctypes.c_void_p * 6)()
    q = L.ffnk_mxfp4_quantize
    assert q(None, 0, 8, 1, 4, 8, p, p, None) == -1
    assert q(p, 3, 8, 1, 4, 8, p, p, None) == -2
    assert q(p, 0, 8, 1, -4, 8, p, p, None) == -2
    assert q(p, 0, 16, 2, 4, 8, p, p, None) == -4
    assert q(p, 0, -8, 1, 4, 8, p, p, None) == -4
    assert q(p, 0, 8, 1, 4, 8, odd, p, None) == -3
    assert q(None, 0, 8, 1, 0, 8, None, None, None) == 0
    d = L.ffnk_mxfp4_dequantize
    assert d(p, p, 4, 8, None, 0, 8, None) == -1
    assert d(p, p, 4, 8, p, 0, 7, None) == -3
    assert d(p, p, 4, 8, p, 9, 8, None) == -2
    assert d(None, None, 4, 0, None, 0, 8, None) == 0
    f = L.ffnk_mxfp4_linear_forward
    big = 1 << 30
    assert f(p, 64, p, p, p, p, p, p, p, None, big, p, 64, 4, 64, 64, p, None) == -1
    assert f(p, 64, p, p, p, p, p, p, p, p, big, p, 64, 4, 60, 64, p, None) == -2
    assert f(p, 64, p, p, p, p, p, p, p, p, big, p, 64, 4, 64, 0, p, None) == -2
    assert f(p, 60, p, p, p, p, p, p, p, p, big, p, 64, 4, 64, 64, p, None) == -3
    assert f(p, 64, odd, p, p, p, p, p, p, p, big, p, 64, 4, 64, 64, p, None) == -3
    assert f(p, 64, p, p, p, p, p, p, p, p, 16, p, 64, 4, 64, 64, p, None) == -8
    assert f(None, 64, None, None, None, None, None, None, None, None, 0, None, 64, 0, 64, 64, None, None) == 0
    b = L.ffnk_mxfp4_linear_backward
    assert b(p, 64, p, p, p, p, p, None, p, big, p, 64, 4, 64, 64, p, None) == -1
    assert b(p, 64, p, p, p, p, p, p, p, big, p, 64, 4, 64, 60, p, None) == -2
    assert b(p, 64, p, p, p, p, p, p, p, 16, p, 64, 4, 64, 64, p, None) == -8
    g = L.ffnk_mxfp4_ffn_forward
    assert g(p, 64, six, holes, p, p, p, p, big, None, None, p, 64, 4, 64, 64, p, None) == -1
    assert g(p, 64, six, six, p, p, p, p, big, p, None, p, 64, 4, 64, 64, p, None) == -1       # f1 without f3
    assert g(p, 64, six, six_odd, p, p, p, p, big, None, None, p, 64, 4, 64, 64, p, None) == -3
    assert g(p, 64, six, six, p, p, p, p, big, None, None, p, 64, 4, 64, 68, p, None) == -2
    assert g(p, 64, six, six, p, p, p, p, 16, None, None, p, 64, 4, 64, 64, p, None) == -8
    w = L.ffnk_mxfp4_ffn_backward
    assert w(p, 64, six, six, None, p, p, p, p, big, p, 64, 4, 64, 64, p, None) == -1
    assert w(p, 64, six, six, p, p, p, p, p, 16, p, 64, 4, 64, 64, p, None) == -8


def test_python_refuses_cpu_tensors_and_wrong_arguments():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: quantize_mxfp4(x), lambda: dequantize_mxfp4(x),
                 lambda: MXFP4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), 4, 64),
                 lambda: MXFP4MaskedLinear.apply(x, x, x, torch.zeros(4, dtype=torch.bool)),
                 lambda: MXFP4MaskedFFN.apply(x, x, x, x, x, x, x, torch.zeros(4, dtype=torch.bool))):
        with pytest.raises(RuntimeError):
            call()


def test_modules_hold_their_weights_as_buffers():
    m = MXFP4MaskedFFNModule(64, 160)
    assert not list(m.parameters())
    sd = m.state_dict()
    assert sorted(sd) == sorted(f"{n}_{k}" for n in MXFP4MaskedFFNModule.NAMES for k in ("codes", "scales"))
    assert tuple(sd["w1_codes"].shape) == (160, 32) and tuple(sd["w2_codes"].shape) == (64, 80)
    assert tuple(sd["w1_scales"].shape) == (2, 1, 32, 4, 4) and tuple(sd["w2_scales"].shape) == (1, 2, 32, 4, 4)
    m.to(torch.bfloat16)                                   # a cast of the model leaves codes alone
    assert all(v.dtype == torch.uint8 for v in m.state_dict().values())
    with pytest.raises(RuntimeError):
        m.load_weight("w1", torch.zeros(64, 160))
    assert sorted(MXFP4MaskedLinearModule(64, 96).state_dict()) == ["linear_t_codes", "linear_t_scales", "linear_v_codes",
                                                                    "linear_v_scales"]


def test_calls_do_not_need_private_names_of_torch(monkeypatch):
    from ffn_kernel_b200 import mxfp4
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    assert not mxfp4._wants_grad(x) and mxfp4._wants_grad(x.requires_grad_(True)) and not mxfp4._wants_grad(None)
    monkeypatch.delattr(torch.autograd.forward_ad, "_current_level")
    assert mxfp4._wants_grad(x.detach()) and not mxfp4._wants_grad(None)
