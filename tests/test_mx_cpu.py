"""Microscaled formats without a GPU: the oracle against the element types' known values, and every refusal."""
import ctypes

import numpy as np
import pytest
import torch

import mx_oracle as mxo


@pytest.fixture(scope="module")
def s24():
    import build as s24_build
    s24_build.build()
    import s24
    return s24


def test_oracle_rounds_like_the_element_types():
    assert list(mxo.element_values(4)) == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(mxo.element_values(8), every)
    # ties to even, saturation and signs of e2m1 under a scale of one (the block's largest value is 4..8)
    v = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25, -5.1] + [0.0] * 22])
    code, scale = mxo.quantize(v, 4)
    assert scale.tolist() == [[127]]
    assert mxo.dequantize(code, scale, 4)[0, :10].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 0, -6]
    # e4m3 against torch's own conversion, on values whose block scale is one (amax in 256..511)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(64, 32, generator=g, dtype=torch.float64) * torch.exp(3 * torch.randn(64, 32, generator=g, dtype=torch.float64))
    x[:, 0] = 300.0
    x = x.clamp(-448, 448).float()
    code, scale = mxo.quantize(x.double().numpy(), 8)
    assert (scale == 127).all()
    assert np.array_equal(code, x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_oracle_special_blocks():
    x = np.zeros((5, 32))
    x[1, 3] = np.nan
    x[2, 4] = -np.inf
    x[3, 5] = 2.0 ** -140
    x[4, 6] = 2.0 ** 127
    for bits, emax in ((4, 2), (8, 8)):
        code, scale = mxo.quantize(x, bits)
        assert scale[:, 0].tolist() == [0, 255, 255, 0, 254 - emax]
        back = mxo.dequantize(code, scale, bits)
        assert (back[0] == 0).all() and np.isnan(back[1]).all() and np.isnan(back[2]).all() and back[4, 6] == 2.0 ** 127


def test_scale_buffer_sizes(s24):
    assert s24.mx_scales_numel(1, 32) == 512
    assert s24.mx_scales_numel(128, 128) == 512
    assert s24.mx_scales_numel(129, 160) == 4 * 512
    assert s24.mx_scales_numel(0, 128) == 0


def test_front_end_refusals_need_no_gpu(s24):
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        s24.mx_quantize(x)
    with pytest.raises(RuntimeError, match="divisible by 32"):
        s24.mx_quantize(x[:, :48])
    with pytest.raises(RuntimeError, match="Invalid datatype"):
        s24.mx_quantize(x.double())
    with pytest.raises(ValueError, match="unknown format"):
        s24.mx_quantize(x, "mxfp6")
    with pytest.raises(RuntimeError, match="at least one dimension"):
        s24.mx_quantize(torch.tensor(1.0))
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        s24.mx_dequantize(codes, scales)
    with pytest.raises(RuntimeError, match="contiguous bytes"):
        s24.mx_dequantize(codes, scales[:3])
    with pytest.raises(RuntimeError, match="contiguous bytes"):
        s24.mx_dequantize(codes, scales, layout="tc")
    with pytest.raises(ValueError, match="unknown scale layout"):
        s24.mx_dequantize(codes, scales, layout="columns")
    with pytest.raises(RuntimeError, match="Invalid datatype"):
        s24.mx_dequantize(codes, scales, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="Invalid datatype"):
        s24.mx_dequantize(codes.to(torch.int32), scales)
    with pytest.raises(ValueError, match="cannot convert"):
        s24.mx_scales_convert(scales, "rows", "rows", 4, 64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        s24.mx_scales_convert(scales, "rows", "tc", 4, 64)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        s24.mx_rms_norm(x, w)
    with pytest.raises(RuntimeError, match="`weight` must be"):
        s24.mx_rms_norm(x, w[:32])
    with pytest.raises(RuntimeError, match="`weight` must be"):
        s24.mx_rms_norm(x, w.half())
    with pytest.raises(RuntimeError, match="`residual` must be"):
        s24.mx_rms_norm(x, w, residual=x[:2])
    with pytest.raises(RuntimeError, match="Invalid datatype"):
        s24.mx_rms_norm(x.float(), w.float())
    with pytest.raises(RuntimeError, match="at most 65536"):
        s24.mx_rms_norm(torch.zeros(1, 65568, dtype=torch.bfloat16), torch.zeros(65568, dtype=torch.bfloat16))
    tc = torch.zeros(s24.mx_scales_numel(4, 64), dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        s24.mx_matmul(codes, tc, codes, tc)
    with pytest.raises(RuntimeError, match="must be equal"):
        s24.mx_matmul(codes, tc, codes[:, :16], tc)
    with pytest.raises(RuntimeError, match="K % 128"):
        s24.mx_matmul(torch.zeros(4, 64, dtype=torch.float8_e4m3fn), tc, codes, tc)
    with pytest.raises(RuntimeError, match="contiguous bytes"):
        s24.mx_matmul(codes, scales, codes, tc)
    with pytest.raises(RuntimeError, match="Invalid datatype"):
        s24.mx_matmul(codes, tc, codes, tc, out_dtype=torch.int8)
    with pytest.raises(RuntimeError, match="2-dimensional"):
        s24.mx_matmul(codes, tc, codes.view(1, 4, 32), tc)


def test_c_entry_refusals_need_no_gpu(s24):
    """every argument rule is checked before the first CUDA call"""
    from s24 import _lib
    L = _lib.lib()
    p = ctypes.cast(ctypes.create_string_buffer(4096 + 64), ctypes.c_void_p)
    p = ctypes.c_void_p((p.value + 63) & ~63)
    odd = ctypes.c_void_p(p.value + 2)
    I, S, U = _lib.ERR_INVALID_ARG, _lib.ERR_SHAPE, _lib.ERR_UNSUPPORTED
    q = L.s24_mx_quantize
    assert q(None, 4, 64, 64, 1, 0, p, p, None, None) == I
    assert q(p, 4, 64, 64, 1, 0, p, None, None, None) == I                 # no layout of the scales
    assert q(p, 4, 48, 64, 1, 0, p, p, None, None) == S
    assert q(p, -1, 64, 64, 1, 0, p, p, None, None) == S
    assert q(p, 4, 64, 32, 1, 0, p, p, None, None) == S                    # rows overlap
    assert q(p, 4, 64, 68, 1, 0, p, p, None, None) == S                    # stride not a multiple of 16 bytes
    assert q(p, 4, 64, 64, 2, 0, p, p, None, None) == I and q(p, 4, 64, 64, 1, 2, p, p, None, None) == I
    assert q(odd, 4, 64, 64, 1, 0, p, p, None, None) == I and q(p, 4, 64, 64, 1, 0, p, None, odd, None) == I
    assert q(p, 1 << 30, 1 << 20, 1 << 20, 1, 0, p, p, None, None) == S    # too many blocks
    assert q(None, 0, 64, 64, 1, 0, None, None, None, None) == _lib.OK     # nothing to do
    d = L.s24_mx_dequantize
    assert d(None, p, 0, p, 4, 64, 0, 1, None) == I and d(p, p, 2, p, 4, 64, 0, 1, None) == I
    assert d(p, p, 0, p, 4, 40, 0, 1, None) == S and d(p, p, 0, odd, 4, 64, 0, 1, None) == I
    assert d(p, p, 0, p, 4, 64, 3, 1, None) == I and d(p, p, 0, p, 4, 64, 0, 3, None) == I
    c = L.s24_mx_scales_convert
    assert c(p, 0, p, 0, 4, 64, None) == U and c(p, 0, p, 2, 4, 64, None) == I and c(None, 0, p, 1, 4, 64, None) == I
    assert c(p, 0, p, 1, 4, 65, None) == S
    n = L.s24_mx_rms_norm
    assert n(p, None, None, None, 4, 64, 64, 0, 1e-6, 1, 1, p, p, None, None) == I
    assert n(p, p, p, None, 4, 64, 64, 64, 1e-6, 1, 1, p, p, None, None) == I       # a residual needs h
    assert n(p, None, p, None, 4, 64, 64, 0, 0.0, 1, 1, p, p, None, None) == I      # eps
    assert n(p, None, p, None, 4, 64, 64, 0, float("nan"), 1, 1, p, p, None, None) == I
    assert n(p, None, p, None, 4, 64, 64, 0, 1e-6, 4, 1, p, p, None, None) == I     # fp32 rows
    assert n(p, None, p, None, 4, 72, 72, 0, 1e-6, 1, 1, p, p, None, None) == S
    assert n(p, None, p, None, 4, 65568, 65568, 0, 1e-6, 1, 1, p, p, None, None) == U
    assert n(p, p, p, p, 4, 64, 64, 60, 1e-6, 1, 1, p, p, None, None) == S
    assert n(odd, None, p, None, 4, 64, 64, 0, 1e-6, 1, 1, p, p, None, None) == I
    m = L.s24_mx_matmul
    assert m(None, p, p, p, p, 4, 4, 64, 32, 32, 4, 0, 0, 1, None, None) == I
    assert m(p, p, p, p, p, 4, 4, 48, 32, 32, 4, 0, 0, 1, None, None) == S
    assert m(p, p, p, p, p, 4, 4, 0, 32, 32, 4, 0, 0, 1, None, None) == S
    assert m(p, p, p, p, p, 4, 4, 64, 64, 32, 4, 1, 0, 1, None, None) == S          # formats differ: K % 128
    assert m(p, p, p, p, p, 4, 4, 64, 24, 32, 4, 0, 0, 1, None, None) == S
    assert m(p, p, p, p, p, 4, 4, 64, 32, 32, 3, 0, 0, 1, None, None) == S
    assert m(p, p, p, p, odd, 4, 4, 64, 32, 32, 4, 0, 0, 4, None, None) == I        # fp32 C on 4 bytes
    assert m(p, p, p, p, p, 4, 4, 64, 32, 32, 4, 2, 0, 1, None, None) == I
    assert m(p, p, p, p, p, 4, 4, 64, 32, 32, 4, 0, 0, 2, None, None) == I
    assert m(p, p, p, p, p, 1 << 40, 4, 64, 32, 32, 4, 0, 0, 1, None, None) == S
    assert m(None, None, None, None, None, 0, 4, 64, 32, 32, 4, 0, 0, 1, None, None) == _lib.OK


def test_split_refusals_need_no_gpu(s24):
    """a split that is not a power of two up to 8, that a side has too many rows for, or that comes with a tile"""
    from s24 import _lib
    p = ctypes.cast(ctypes.create_string_buffer(4096 + 64), ctypes.c_void_p)
    p = ctypes.c_void_p((p.value + 63) & ~63)

    def product(m, n, *cfg):
        return _lib.lib().s24_mx_matmul(p, p, p, p, p, m, n, 1024, 512, 512, n, 0, 0, 1, ctypes.byref(_lib.TileCfg(*cfg)), None)

    for split in (3, 16, -1):
        assert product(4, 4, 0, 0, 0, split) == _lib.ERR_UNSUPPORTED
    assert product(8193, 8193, 0, 0, 0, 2) == _lib.ERR_UNSUPPORTED
    assert product(4, 65535 * 128 + 1, 0, 0, 0, 2) == _lib.ERR_UNSUPPORTED
    for bm, bn in ((256, 256), (256, 0), (0, 128), (128, 128)):
        assert product(4, 4, bm, bn, 0, 2) == _lib.ERR_UNSUPPORTED and "tiles of its own" in _lib.last_error()
