"""Microscaled formats on the GPU against the 64-bit oracle.

Codes and scales are compared bit for bit (the only rounding is the one to the element type), read-back values
exactly.  Products are compared exactly where every partial sum is a whole multiple of a small power of two
below 2^24 of it, and otherwise within K * 2^-24 * sum |a b| (K additions, each off by at most half a step of a
partial sum, which sum |a b| bounds) plus half a step of the output type.
"""
import numpy as np
import pytest
import torch

import mx_oracle as mxo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BITS = {"mxfp4": 4, "mxfp8": 8}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def s24():
    import s24
    return s24


def _codes(t):
    """codes of a tensor as one uint8 per element"""
    t = t.cpu()
    return mxo.unpack(t.numpy(), 4) if t.dtype == torch.uint8 else t.view(torch.uint8).numpy()


def _activations(r, k, dtype, seed):
    """values over many scales, with zero blocks, ties, both ends of the type and non-finite blocks among them"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(r, k, generator=g) * torch.exp2(torch.randint(-12, 8, (r, k // 32), generator=g).float()).repeat_interleave(32, 1)
    x = x.to(dtype)
    flat = x.view(-1, 32)
    n = flat.shape[0]
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, 6.0, 7.0, -0.25, -0.75, -5.0, -0.0, 0.0, 7.96875]).repeat(2).to(dtype)
    for i, block in enumerate((torch.zeros(32), ties, torch.full((32,), torch.finfo(dtype).max), torch.full((32,), torch.finfo(dtype).smallest_normal / 8),
                               torch.tensor([float("nan")] + [1.0] * 31), torch.tensor([1.0] * 31 + [float("-inf")]),
                               torch.tensor([448.0, 464.0, 480.0, 0.01] * 8), torch.full((32,), -0.0))):
        if n > 8:
            flat[(i * 37 + 5) % n] = block.to(dtype)
    return x


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r,k", [(1, 32), (1, 4096), (3, 96), (33, 160), (127, 128), (128, 256), (129, 288), (300, 1056), (1000, 8192)])
def test_quantize_is_bit_exact_and_reads_back(s24, r, k, dtype, fmt):
    x = _activations(r, k, dtype, r + k)
    want_c, want_s = mxo.quantize(x.double().numpy(), BITS[fmt])
    codes, scales, tc = s24.mx_quantize(x.to(DEV), fmt, want_rows=True, want_tc=True)
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(_codes(codes), want_c)
    assert np.array_equal(tc.cpu().numpy(), mxo.tc_order(want_s))
    # one layout at a time, and from one to the other
    only = s24.mx_quantize(x.to(DEV), fmt, want_rows=False, want_tc=True)
    assert only[1] is None and torch.equal(only[2], tc) and torch.equal(only[0].view(torch.uint8), codes.view(torch.uint8))
    assert torch.equal(s24.mx_scales_convert(scales, "rows", "tc", r, k), tc)
    assert torch.equal(s24.mx_scales_convert(tc, "tc", "rows", r, k), scales)
    # back, rounded once to each type
    want = torch.from_numpy(mxo.dequantize(want_c, want_s, BITS[fmt]))
    for out in DTYPES:
        for layout, s in (("rows", scales), ("tc", tc)):
            got = s24.mx_dequantize(codes, s, layout=layout, dtype=out).cpu()
            torch.testing.assert_close(got, want.to(out), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_every_code_and_scale_reads_back(s24, fmt):
    """all element codes under all 256 scales: NaN codes of e4m3, the subnormal scale 0 and NaN scales among them"""
    bits = BITS[fmt]
    n = 16 if bits == 4 else 256
    code = np.tile(np.arange(n, dtype=np.uint8), max(1, 32 // n))
    code = np.broadcast_to(code, (256, len(code))).copy()
    scale = np.broadcast_to(np.arange(256, dtype=np.uint8)[:, None], (256, code.shape[1] // 32)).copy()
    packed = torch.from_numpy(mxo.pack(code, bits)).to(DEV)
    packed = packed if bits == 4 else packed.view(torch.float8_e4m3fn)
    want = torch.from_numpy(mxo.dequantize(code, scale, bits))
    for out in DTYPES:
        got = s24.mx_dequantize(packed, torch.from_numpy(scale).to(DEV), dtype=out).cpu()
        torch.testing.assert_close(got, want.to(out), rtol=0, atol=0, equal_nan=True)


def test_quantize_takes_strided_unaligned_and_higher_dimensional_inputs(s24):
    base = _activations(40, 1024, torch.bfloat16, 7).to(DEV)
    for x in (base[:, 256:768], base[::2], base[:, 4:4 + 512], base.view(-1)[2:2 + 64 * 96].view(64, 96), base.t()[:, :32], base[:1].expand(5, 1024),
              base.view(5, 8, 1024), base.view(2, 4, 5, 1024)[:, 1:3], base[3]):
        codes, scales, tc = s24.mx_quantize(x, "mxfp8", want_tc=True)
        flat = x.reshape(-1, x.shape[-1])
        want_c, want_s = mxo.quantize(flat.double().cpu().numpy(), 8)
        assert codes.shape == x.shape and scales.shape == (*x.shape[:-1], x.shape[-1] // 32)
        assert np.array_equal(codes.view(torch.uint8).cpu().numpy().reshape(want_c.shape), want_c)
        assert np.array_equal(scales.cpu().numpy().reshape(want_s.shape), want_s)
        assert np.array_equal(tc.cpu().numpy(), mxo.tc_order(want_s))


def test_refusals_on_the_gpu(s24):
    x = torch.zeros(8, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="at least one layout"):
        s24.mx_quantize(x, want_rows=False)
    with pytest.raises(RuntimeError, match="at least one layout"):
        s24.mx_rms_norm(x, w, want_rows=False)
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(s24.S24Error, match="eps must be"):
            s24.mx_rms_norm(x, w, eps=eps)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        s24.mx_rms_norm(x, w.cpu())
    codes, scales, tc = s24.mx_quantize(x, want_tc=True)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        s24.mx_dequantize(codes, scales.cpu())
    with pytest.raises(RuntimeError, match="contiguous bytes"):
        s24.mx_matmul(codes, tc[:256], codes, tc)
    for config in ({"BM": 64, "BN": 64}, {"BM": 128, "BN": 256}, {"SPLIT": 3}):
        with pytest.raises(s24.S24Error):
            s24.mx_matmul(codes, tc, codes, tc, manual_config=config)
    torch.cuda.synchronize()


def test_empty_inputs(s24):
    x = torch.empty(0, 64, dtype=torch.float16, device=DEV)
    codes, scales, tc = s24.mx_quantize(x, want_tc=True)
    assert codes.shape == (0, 32) and scales.shape == (0, 2) and tc.numel() == 0
    assert s24.mx_dequantize(codes, scales).shape == (0, 64)
    b, _, bt = s24.mx_quantize(torch.ones(8, 64, dtype=torch.float16, device=DEV), want_tc=True)
    assert s24.mx_matmul(codes, tc, b, bt).shape == (0, 8)
    assert s24.mx_matmul(b, bt, codes, tc).shape == (8, 0)
    assert s24.mx_quantize(torch.empty(4, 0, dtype=torch.float16, device=DEV), "mxfp8")[0].shape == (4, 0)
    out = s24.mx_rms_norm(x, torch.ones(64, dtype=torch.float16, device=DEV), residual=x)
    assert out[0].shape == (0, 64) and out[3].shape == (0, 64)


# ------------------------------------------------------------------ norm

@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("r,k", [(1, 32), (5, 96), (9, 128), (7, 224), (130, 512), (33, 1056), (3, 2080), (20, 4128), (16, 8192), (129, 8192),
                                 (2, 16384), (3, 20000), (2, 32768), (1, 65536)])
def test_norm_is_the_formula_in_64_bits(s24, r, k, residual, dtype, fmt):
    g = torch.Generator().manual_seed(r * 7 + k)
    x = (torch.randn(r, k, generator=g) * torch.exp(torch.randn(k, generator=g))).to(dtype)
    res = (3 * torch.randn(r, k, generator=g)).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(k, generator=g)).to(dtype)
    if r > 8:
        x[r // 2] = 0
        if residual:
            res[r // 2] = 0
    h, y = mxo.rms_norm(x.double().numpy(), None if res is None else res.double().numpy(), w.double().numpy(), 1e-6,
                        lambda v: torch.from_numpy(v).to(dtype).double().numpy())
    want_c, want_s = mxo.quantize(y, BITS[fmt])
    codes, scales, tc, got_h = s24.mx_rms_norm(x.to(DEV), w.to(DEV), eps=1e-6, residual=None if res is None else res.to(DEV), fmt=fmt, want_tc=True)
    assert np.array_equal(got_h.double().cpu().numpy(), h)
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(_codes(codes), want_c)
    assert np.array_equal(tc.cpu().numpy(), mxo.tc_order(want_s))


def test_norm_special_rows(s24):
    """a row of zeros, an infinity, a NaN, very large and very small rows; strided inputs; only one layout"""
    x = torch.randn(6, 256, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    x[0] = 0
    x[1, 40] = float("inf")
    x[2, 70] = float("nan")
    x[3] *= 1e30
    x[4] *= 1e-30
    wide = torch.zeros(6, 512, dtype=torch.bfloat16)
    wide[:, 64:320] = x
    xd = wide.to(DEV)[:, 64:320]
    w = torch.linspace(-2, 2, 256).to(torch.bfloat16)
    _, y = mxo.rms_norm(x.double().numpy(), None, w.double().numpy(), 1e-6, None)
    for bits, fmt in ((8, "mxfp8"), (4, "mxfp4")):
        want_c, want_s = mxo.quantize(y, bits)
        codes, scales, tc, h = s24.mx_rms_norm(xd, w.to(DEV), fmt=fmt, want_rows=False, want_tc=True)
        assert scales is None and h is xd
        assert np.array_equal(tc.cpu().numpy(), mxo.tc_order(want_s)) and np.array_equal(_codes(codes), want_c)
        # the infinity's block is not a number, the row's other blocks are zeros; a NaN takes its whole row
        assert (want_s[1] == 255).sum() == 1 and (want_s[2] == 255).all()


def test_norm_writes_the_new_residual_in_place_through_the_c_entry(s24):
    import ctypes
    from s24 import _lib
    g = torch.Generator(device=DEV).manual_seed(5)
    x, res = (torch.randn(64, 1024, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(1024, dtype=torch.bfloat16, device=DEV)
    codes, scales, _, h = s24.mx_rms_norm(x, w, residual=res)
    c2, s2 = torch.empty_like(codes), torch.empty_like(scales)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(_lib.lib().s24_mx_rms_norm(p(x), p(res), p(w), p(res), 64, 1024, 1024, 1024, 1e-6, _lib.BF16, _lib.MXFP8, p(c2), p(s2), None, stream))
    torch.cuda.synchronize()
    assert torch.equal(res, h) and torch.equal(c2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s2, scales)


# ------------------------------------------------------------------ product

def _operand(s24, r, k, fmt, seed, exact):
    """codes and scales of an operand, on the GPU, and its values in float64"""
    rng = np.random.default_rng(seed)
    bits = BITS[fmt]
    if exact:   # elements of at most 2 in steps of a half under scales of 1/4..4: products are multiples of 2^-6, at most 2^6
        code = rng.integers(0, 5, (r, k)).astype(np.uint8)
        code = np.array([0, 1, 2, 3, 4], np.uint8)[code] if bits == 4 else np.array([0, 0x30, 0x38, 0x3C, 0x40], np.uint8)[code]
        code |= (rng.integers(0, 2, (r, k)) * (8 if bits == 4 else 128)).astype(np.uint8)
        scale = rng.integers(125, 130, (r, k // 32)).astype(np.uint8)
    else:
        x = rng.standard_normal((r, k)) * np.exp(rng.standard_normal((r, k // 32))).repeat(32, 1)
        code, scale = mxo.quantize(x, bits)
    t = torch.from_numpy(mxo.pack(code, bits)).to(DEV)
    return (t if bits == 4 else t.view(torch.float8_e4m3fn)), torch.from_numpy(mxo.tc_order(scale)).to(DEV), mxo.dequantize(code, scale, bits)


PAIRS = [("mxfp4", "mxfp4"), ("mxfp8", "mxfp8"), ("mxfp8", "mxfp4"), ("mxfp4", "mxfp8")]
SPLITS = [{"SPLIT": 1}, {"SPLIT": 2}, {"SPLIT": 4}, {"SPLIT": 8}]    # K split over that many CTAs
TILES = [None, {"BM": 128, "BN": 128}, {"BM": 256, "BN": 128}, {"BM": 256, "BN": 256}]


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 8, 128), (3, 5, 96), (1, 257, 256), (2, 1000, 1024), (17, 130, 384), (40, 520, 2048), (64, 64, 160),
                                   (100, 4099, 512), (128, 128, 128), (129, 127, 256), (200, 333, 640), (256, 256, 512), (257, 515, 416), (1000, 300, 1024),
                                   (2048, 1544, 512), (513, 2049, 128),
                                   (1537, 6150, 1024), (1540, 6144, 512), (6200, 1536, 512)])
def test_product_is_exact_where_sums_are(s24, m, n, k, fa, fb):
    if fa != fb:
        k = -(-k // 128) * 128
    a, sa, va = _operand(s24, m, k, fa, 1000 * m + k, True)
    b, sb, vb = _operand(s24, n, k, fb, 1000 * n + k + 1, True)
    want = torch.from_numpy(va) @ torch.from_numpy(vb).t()      # below 2^6 * 2048 * ..., whole multiples of 2^-6: exact in fp32
    for tile in TILES + SPLITS:
        got = s24.mx_matmul(a, sa, b, sb, out_dtype=torch.float32, manual_config=tile)
        assert torch.equal(got.cpu().double(), want), f"tile {tile}: {(got.cpu().double() != want).sum()} of {want.numel()} differ"
    for out in (torch.bfloat16, torch.float16):
        got = s24.mx_matmul(a, sa, b, sb, out_dtype=out)
        assert torch.equal(got.cpu(), want.to(out))
    assert s24.lib().s24_device_status(None) == 0


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("m,n,k", [(2560, 2050, 256), (2560, 2178, 384), (5000, 1040, 512), (4100, 1281, 256), (300, 11000, 512), (2500, 2700, 128)])
def test_product_whose_last_pass_is_shared(s24, m, n, k, fa, fb):
    """some more tiles than the device has SM pairs, in a window of a wider result that keeps what surrounds it"""
    a, sa, va = _operand(s24, m, k, fa, 1000 * m + k, True)
    b, sb, vb = _operand(s24, n, k, fb, 1000 * n + k + 1, True)
    want = (torch.from_numpy(va).to(DEV) @ torch.from_numpy(vb).to(DEV).t()).float()
    for left, width in ((0, n), (32, -(-n // 32) * 32 + 96), (3, n + 8)):
        for tile in (None, {"BM": 256, "BN": 256}, {"BM": 256, "BN": 128}):
            full = torch.full((m + 2, width), 7.0, dtype=torch.float32, device=DEV)
            s24.mx_matmul(a, sa, b, sb, out_dtype=torch.float32, out=full[1:m + 1, left:left + n], manual_config=tile)
            assert torch.equal(full[1:m + 1, left:left + n], want), f"tile {tile}"
            full[1:m + 1, left:left + n] = 7.0
            assert bool((full == 7.0).all()), f"tile {tile}: written outside"


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("m,n,k", [(5, 300, 4096), (300, 700, 2048), (64, 256, 16384), (1030, 520, 8192)])
def test_product_of_quantized_data(s24, m, n, k, fa, fb):
    a, sa, va = _operand(s24, m, k, fa, m + k, False)
    b, sb, vb = _operand(s24, n, k, fb, n + k + 1, False)
    ta, tb = torch.from_numpy(va).to(DEV), torch.from_numpy(vb).to(DEV)
    want, most = ta @ tb.t(), ta.abs() @ tb.abs().t()
    for out in (torch.float32, torch.bfloat16, torch.float16):
        got = s24.mx_matmul(a, sa, b, sb, out_dtype=out).double()
        bound = k * 2.0 ** -24 * most + torch.finfo(out).eps / 2 * want.abs() * (1 + k * 2.0 ** -24)
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


def test_product_takes_strided_codes_leading_dimensions_and_out(s24):
    a, sa, va = _operand(s24, 24, 256, "mxfp8", 1, True)
    b, sb, vb = _operand(s24, 200, 256, "mxfp4", 2, True)
    want = torch.from_numpy(va @ vb.T)
    wide = torch.zeros(24, 512, dtype=torch.uint8, device=DEV)
    wide[:, 64:320] = a.view(torch.uint8)
    got = s24.mx_matmul(wide[:, 64:320].view(torch.float8_e4m3fn), sa, b, sb, out_dtype=torch.float32)
    assert torch.equal(got.cpu().double(), want)
    shifted = torch.zeros(24 * 256 + 8, dtype=torch.uint8, device=DEV)
    shifted[8:] = a.view(torch.uint8).reshape(-1)
    got = s24.mx_matmul(shifted[8:].view(24, 256).view(torch.float8_e4m3fn), sa, b, sb, out_dtype=torch.float32)
    assert torch.equal(got.cpu().double(), want)
    got = s24.mx_matmul(a.view(2, 3, 4, 256), sa, b, sb)
    assert got.shape == (2, 3, 4, 200) and torch.equal(got.cpu().view(24, 200), want.to(torch.bfloat16))
    # into a window of a larger tensor whose rows are not 16-byte aligned: nothing outside it changes
    big = torch.full((30, 333), -77.0, device=DEV)
    s24.mx_matmul(a, sa, b, sb, out_dtype=torch.float32, out=big[3:27, 5:205])
    full = torch.full((30, 333), -77.0, dtype=torch.float64)
    full[3:27, 5:205] = want
    assert torch.equal(big.cpu().double(), full)
    for bad in (torch.empty(24, 200, device=DEV, dtype=torch.float16), torch.empty(24, 199, device=DEV), torch.empty(200, 24, device=DEV).t(),
                torch.empty(1, 200, device=DEV).expand(24, 200)):
        with pytest.raises(RuntimeError, match="`out` must be"):
            s24.mx_matmul(a, sa, b, sb, out_dtype=torch.float32, out=bad)


def test_product_keeps_nan_blocks_to_their_rows_and_columns(s24):
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(70, 512, generator=g).to(torch.bfloat16), torch.randn(150, 512, generator=g).to(torch.bfloat16)
    x[11, 100] = float("nan")
    w[140, 7] = float("inf")
    for fa, fb in PAIRS:
        a, _, sa = s24.mx_quantize(x.to(DEV), fa, want_tc=True)
        b, _, sb = s24.mx_quantize(w.to(DEV), fb, want_tc=True)
        c = s24.mx_matmul(a, sa, b, sb).isnan().cpu()
        want = torch.zeros(70, 150, dtype=torch.bool)
        want[11] = True
        want[:, 140] = True
        assert torch.equal(c, want)


def test_a_chain_of_them_on_another_stream_and_in_a_graph(s24):
    """norm -> product -> quantise -> product, as an MLP uses them: eager, on a side stream, captured and replayed with new
    inputs, two graphs of the same operands in turn"""
    g = torch.Generator(device=DEV).manual_seed(11)
    x, res = (torch.randn(48, 1024, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(1024, dtype=torch.bfloat16, device=DEV)
    up = s24.mx_quantize((0.02 * torch.randn(2048, 1024, generator=g, device=DEV)).to(torch.bfloat16), "mxfp4", False, True)
    down = s24.mx_quantize((0.02 * torch.randn(1024, 2048, generator=g, device=DEV)).to(torch.bfloat16), "mxfp4", False, True)

    def block(x, res):
        q, _, s, h = s24.mx_rms_norm(x, w, residual=res, fmt="mxfp8", want_rows=False, want_tc=True)
        mid = s24.mx_matmul(q, s, up[0], up[2])
        q, _, s = s24.mx_quantize(torch.relu(mid), "mxfp8", False, True)
        return s24.mx_matmul(q, s, down[0], down[2]), h

    def plain(x, res):
        deq = lambda q, s, k: s24.mx_dequantize(q, s, layout="tc", dtype=torch.float32).double()  # noqa: E731
        q, _, s, h = s24.mx_rms_norm(x, w, residual=res, want_rows=False, want_tc=True)
        mid = (deq(q, s, 1024) @ deq(up[0], up[2], 1024).t()).to(torch.bfloat16)
        q, _, s = s24.mx_quantize(torch.relu(mid), "mxfp8", False, True)
        return deq(q, s, 2048) @ deq(down[0], down[2], 2048).t(), h

    y, h = block(x, res)
    want, _ = plain(x, res)
    # a bf16 intermediate that rounds the other way moves by 2^-8, and so may its e4m3 code by 2^-3: a few of 2048 terms
    assert float((y.double() - want).norm() / want.norm()) < 2.0 ** -6
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, _ = block(x, res)
    side.synchronize()
    assert torch.equal(y2, y)
    sx, sr = x.clone(), res.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = block(sx, sr)
        graphs.append((graph, out))
    for seed in (1, 2, 3):
        sx.copy_(torch.randn(48, 1024, generator=g, device=DEV).to(torch.bfloat16))
        eager, _ = block(sx, sr)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, eager) for _, out in graphs)
    assert s24.lib().s24_device_status(None) == 0


def test_offsets_beyond_32_bits(s24):
    """operands, scales and results whose last rows lie past 4 GB: the same bits as for those rows by themselves"""
    r, k = 140032, 16384                                   # 4.6 GB in 16 bits
    x = torch.empty(r, k, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(128, k, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(torch.bfloat16)
    x.zero_()
    x[-128:] = tail
    codes, scales, tc = s24.mx_quantize(x, "mxfp8", want_tc=True)
    c2, s2, t2 = s24.mx_quantize(tail, "mxfp8", want_tc=True)
    assert torch.equal(codes[-128:].view(torch.uint8), c2.view(torch.uint8)) and torch.equal(scales[-128:], s2) and torch.equal(tc[-t2.numel():], t2)
    w = torch.ones(k, dtype=torch.bfloat16, device=DEV)
    n1, n2 = s24.mx_rms_norm(x, w, residual=x), s24.mx_rms_norm(tail, w, residual=tail)
    for a, b in zip(n1, n2):
        assert (a is None) == (b is None) and (a is None or torch.equal(a[-128:].view(torch.uint8), b.view(torch.uint8)))
    del n1, x
    back = s24.mx_dequantize(codes, scales, dtype=torch.bfloat16)
    assert torch.equal(back[-128:], s24.mx_dequantize(c2, s2, dtype=torch.bfloat16))
    del back
    b, _, bt = s24.mx_quantize(tail[:, :].contiguous(), "mxfp8", False, True)
    few = s24.mx_matmul(b[:3], s24.mx_quantize(tail[:3], "mxfp8", False, True)[2], codes, tc)        # (3, r): rows of the long side past 2 GB
    assert torch.equal(few[:, -128:], s24.mx_matmul(b[:3], s24.mx_quantize(tail[:3], "mxfp8", False, True)[2], c2, t2))
    del codes, scales, tc
    # a result past 4 GB, through the tiles: its last block against the product of those rows
    a8, _, a8t = s24.mx_quantize(torch.randn(70016, 128, device=DEV).to(torch.bfloat16), "mxfp4", False, True)
    b8, _, b8t = s24.mx_quantize(torch.randn(32896, 128, device=DEV).to(torch.bfloat16), "mxfp4", False, True)
    c = s24.mx_matmul(a8, a8t, b8, b8t)
    one = s24.mx_matmul(a8[-128:], a8t[-512:], b8[-128:], b8t[-512:])
    assert torch.equal(c[-128:, -128:], one)
    assert s24.lib().s24_device_status(None) == 0


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("seed", [1, 2])
def test_norm_of_many_elements_is_the_formula_in_64_bits(s24, seed, fmt):
    """134 million elements, of which several lie within a unit in the last place of a border: every code and scale"""
    r, k = 16384, 8192
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(r, k, generator=g, device=DEV).mul_(torch.exp(0.5 * torch.randn(k, generator=g, device=DEV))).to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(k, generator=g, device=DEV)).to(torch.bfloat16)
    codes, scales, _, _ = s24.mx_rms_norm(x, w, eps=1e-6, residual=x, fmt=fmt)
    emax, top = (2, 6.0) if fmt == "mxfp4" else (8, 448.0)
    low, fraction = (0, 1) if fmt == "mxfp4" else (-6, 3)
    for i in range(0, r, 2048):
        h = (2 * x[i:i + 2048].float()).to(torch.bfloat16).double()
        y = (h / torch.sqrt((h * h).sum(-1, keepdim=True) / k + 1e-6) * w.double()).view(2048, k // 32, 32)
        s = torch.frexp(y.abs().amax(-1))[1] - 1 - emax
        assert torch.equal(scales[i:i + 2048].int() - 127, s.int())
        u = torch.ldexp(y, -s.unsqueeze(-1))
        step = torch.ldexp(torch.ones_like(u), (torch.frexp(u.abs())[1] - 1).clamp(min=low) - fraction)
        q = (torch.round(u / step) * step).clamp(-top, top)
        got = s24.mx_dequantize(codes[i:i + 2048], torch.full_like(scales[i:i + 2048], 127), dtype=torch.float32).view_as(q)
        assert int((got.double() != q).sum()) == 0


def test_products_of_random_shapes(s24):
    """shapes drawn over the whole range of tiles, splits and unaligned rows, windows of larger results among them"""
    rng = np.random.default_rng(42)
    for i in range(60):
        fa, fb = PAIRS[int(rng.integers(4))]
        m, n = (int(np.exp(rng.uniform(0, np.log(1500)))) for _ in range(2))
        k = 128 * int(rng.integers(1, 13)) if fa != fb else 32 * int(rng.integers(1, 49))
        out = DTYPES[int(rng.integers(3))]
        a, sa, va = _operand(s24, m, k, fa, 10 * i, True)
        b, sb, vb = _operand(s24, n, k, fb, 10 * i + 1, True)
        want = (torch.from_numpy(va) @ torch.from_numpy(vb).t()).to(out)
        pad, first = int(rng.integers(0, 40)), int(rng.integers(0, 8))
        big = torch.full((m + 2, first + n + pad), 5.0, dtype=out, device=DEV)
        s24.mx_matmul(a, sa, b, sb, out_dtype=out, out=big[1:m + 1, first:first + n])
        full = torch.full((m + 2, first + n + pad), 5.0, dtype=out)
        full[1:m + 1, first:first + n] = want
        assert torch.equal(big.cpu(), full), (i, fa, fb, m, n, k, out, pad, first)
        assert torch.equal(s24.mx_matmul(a, sa, b, sb, out_dtype=out).cpu(), want), (i, fa, fb, m, n, k, out)


def test_two_streams_at_once(s24):
    """products of every kind, norms and quantisations on two streams that run together: the bits of one stream alone"""
    def work(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        x = torch.randn(300, 2048, generator=g, device=DEV).to(torch.bfloat16)
        w = torch.randn(1500, 2048, generator=g, device=DEV).to(torch.bfloat16)
        gamma = torch.ones(2048, dtype=torch.bfloat16, device=DEV)
        return x, w, gamma

    def steps(x, w, gamma):
        out = []
        for fmt in ("mxfp4", "mxfp8"):
            wq, _, ws = s24.mx_quantize(w, "mxfp4", False, True)
            for rows in (1, 40, 300):
                q, _, s, _ = s24.mx_rms_norm(x[:rows], gamma, residual=x[:rows], fmt=fmt, want_rows=False, want_tc=True)
                out.append(s24.mx_matmul(q, s, wq, ws))
                out.append(s24.mx_dequantize(q, s, layout="tc"))
        return out

    inputs = [work(1), work(2)]
    alone = [steps(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        together = []
        for stream, i in zip(streams, inputs):
            with torch.cuda.stream(stream):
                together.append(steps(*i))
        torch.cuda.synchronize()
        for a, b in zip(alone, together):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert s24.lib().s24_device_status(None) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_norm_on_exact_borders(s24, fmt, dtype):
    """rows of +-1 (and +-2): 1 / sqrt(mean + 1e-30) is exactly 1 (a half), so y is the weight itself, which runs through
    values exactly between two elements and blocks whose largest value is a power of two or one step to its side; zero
    rows and rows with a single non-zero among them"""
    k = 4096
    g = torch.Generator().manual_seed(4)
    x = torch.where(torch.rand(12, k, generator=g) < 0.5, -1.0, 1.0)
    x[3] *= 2
    x[5] = 0
    x[7] = 0
    x[7, 100] = 8.0
    w = torch.ldexp((torch.randint(16, 33, (k,), generator=g) / 16.0 + torch.randint(0, 2, (k,), generator=g) / 32.0),
                    torch.randint(-9, 1, (k,), generator=g).int())
    blocks = w.view(-1, 32)
    blocks[::3, 7] = 2.0
    blocks[1::3, 7] = 2.0 + torch.finfo(dtype).eps * 2
    blocks[2::3, 7] = 2.0 - torch.finfo(dtype).eps
    x, w = x.to(dtype), w.to(dtype)
    h, y = mxo.rms_norm(x.double().numpy(), None, w.double().numpy(), 1e-30, None)
    want_c, want_s = mxo.quantize(y, BITS[fmt])
    codes, scales, _, _ = s24.mx_rms_norm(x.to(DEV), w.to(DEV), eps=1e-30, fmt=fmt)
    assert np.array_equal(scales.cpu().numpy(), want_s) and np.array_equal(_codes(codes), want_c)


def _check_norm(s24, x, w, eps, fmt):
    """codes and scales against the formula in 64 bits, where values from 2^128 on count as infinite"""
    _, y = mxo.rms_norm(x.double().numpy(), None, w.double().numpy(), eps, None)
    want_c, want_s = mxo.quantize(np.where(np.abs(y) < 2.0 ** 128, y, np.inf), BITS[fmt])
    codes, scales, tc, _ = s24.mx_rms_norm(x.to(DEV), w.to(DEV), eps=eps, fmt=fmt, want_tc=True)
    assert np.array_equal(scales.cpu().numpy(), want_s), f"{(scales.cpu().numpy() != want_s).sum()} scales differ"
    assert np.array_equal(_codes(codes), want_c), f"{(_codes(codes) != want_c).sum()} codes differ"
    assert np.array_equal(tc.cpu().numpy(), mxo.tc_order(want_s))


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [96, 1568, 4096, 4128, 40000])
def test_norm_keeps_ties_of_the_formula(s24, k, dtype, fmt):
    """rows of one magnitude c: h / sqrt(mean) is exactly +-1 in 64 bits though 1 / c has no end, so y is +-w, which runs
    through values exactly between two elements; a row with a single non-zero, and magnitudes near the end of the type"""
    g = torch.Generator().manual_seed(k)
    magnitudes = [3.0, 5.0, 7.0, 11.0, 100.0, 1.5 * 2.0 ** 13]
    if dtype == torch.bfloat16:
        magnitudes += [196608.0, 2.0 ** 100 * 1.75, 1.5 * 2.0 ** 126, 1.25 * 2.0 ** 127, 3.0 * 2.0 ** -20]
    x = torch.where(torch.rand(len(magnitudes) + 1, k, generator=g) < 0.5, -1.0, 1.0) * torch.tensor([*magnitudes, 0.0]).unsqueeze(1)
    x[-1, 41] = 7.0
    w = torch.ldexp((torch.randint(16, 33, (k,), generator=g) / 16.0 + torch.randint(0, 2, (k,), generator=g) / 32.0),
                    torch.randint(-9, 1, (k,), generator=g).int())
    w.view(-1, 32)[::2, 7] = 2.0
    for eps in (1e-30, 1e-12, 1e-6):
        _check_norm(s24, x.to(dtype), w.to(dtype), eps, fmt)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("scale", [1e31, 1e38])
def test_norm_of_very_large_rows(s24, scale, fmt):
    """1 / sqrt(mean) is below what fp32 holds with all its bits"""
    g = torch.Generator().manual_seed(6)
    x = (torch.randn(1024, 4096, generator=g, dtype=torch.float64) * scale).clamp(-3.3e38, 3.3e38).to(torch.bfloat16)
    _check_norm(s24, x, (1 + 0.3 * torch.randn(4096, generator=g)).to(torch.bfloat16), 1e-6, fmt)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_rounds_like_the_formula_next_to_ties(s24, dtype, fmt):
    """rows whose mean of squares is c^2 and whose elements are c / 3 and 5 c / 3: h / sqrt(mean) is a rounded third, and times
    three times a value between two elements it is again such a value, or the double next to it"""
    k = 1536
    c = torch.tensor([3.0, 6.0, 12.0, 1.5, 0.75])
    g = torch.Generator().manual_seed(8)
    pattern = torch.tensor([1.0, 1.0, 5.0]).repeat(k // 3) / 3.0
    x = torch.stack([pattern[torch.randperm(k, generator=g)] for _ in c]) * c.unsqueeze(1)
    w = 3.0 * torch.ldexp((torch.randint(16, 33, (k,), generator=g) / 16.0 + torch.randint(0, 2, (k,), generator=g) / 32.0),
                          torch.randint(-6, 1, (k,), generator=g).int())
    _check_norm(s24, x.to(dtype), w.to(dtype), 1e-30, fmt)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("eps", [1e-30, 1e-6, 1e30])
def test_norm_over_the_whole_range_of_bf16(s24, eps, fmt):
    """rows and weights of every exponent that bf16 has: h / sqrt(mean) or y below and beyond what fp32 holds in between"""
    def numbers(g, shape, low, high):
        e = torch.rand(shape, generator=g, dtype=torch.float64) * (high - low) + low
        return (torch.exp2(e) * torch.where(torch.rand(shape, generator=g) < 0.5, -1.0, 1.0)).to(torch.bfloat16)

    g = torch.Generator().manual_seed(10)
    k = 2048
    for low, high in ((-133, 127), (-40, 127), (-133, -100), (-133, 0), (-70, -40), (60, 127)):
        x = numbers(g, (32, k), low, high)
        x[::3, ::2] = 0
        for wlow, whigh in ((-133, 127), (100, 127), (-5, 5), (-133, -60)):
            w = numbers(g, (k,), wlow, whigh)
            w.view(-1, 32)[::5] = 0
            _check_norm(s24, x, w, eps, fmt)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_norm_of_small_elements_beside_large_ones(s24, fmt):
    """elements whose h / sqrt(mean) fp32 has only few bits for, or none, under weights that bring y back into its range"""
    rows = [(2.0 ** 127, 1.0703125 * 2.0 ** -20, 2.0 ** 120), (2.0 ** 127, 1.0703125 * 2.0 ** -20, 2.0 ** 127), (2.0 ** 127, 2.0 ** -133, 1.5 * 2.0 ** 127),
            (2.0 ** 100, 1.4375 * 2.0 ** -126, 1.75 * 2.0 ** 127), (2.0 ** 90, -2.0 ** -132, 2.0 ** 127), (1.0, 1.0703125 * 2.0 ** -126, 2.0 ** 127)]
    for big, small, weight in rows:
        x, w = torch.zeros(3, 64), torch.ones(64)
        x[:2, 0], x[:, 32], x[1, 33], w[32:] = big, small, 3 * small, weight
        _check_norm(s24, x.to(torch.bfloat16), w.to(torch.bfloat16), 1e-6, fmt)
        _check_norm(s24, x.to(torch.bfloat16), w.to(torch.bfloat16), 1e-30, fmt)


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("m,n", [(1, 130), (7, 1000), (33, 257), (130, 70), (300, 200)])
def test_product_with_k_really_split(s24, m, n, fa, fb):
    """as many k-tiles as CTAs that share them, and a few more; a tile with it is refused"""
    for k in (2048, 2560):
        a, sa, va = _operand(s24, m, k, fa, m + k, True)
        b, sb, vb = _operand(s24, n, k, fb, n + k + 1, True)
        want = torch.from_numpy(va) @ torch.from_numpy(vb).t()
        for split in SPLITS:
            got = s24.mx_matmul(a, sa, b, sb, out_dtype=torch.float32, manual_config=split)
            assert torch.equal(got.cpu().double(), want), (k, split)
    with pytest.raises(s24.S24Error, match="tiles of its own"):
        s24.mx_matmul(a, sa, b, sb, manual_config={"BM": 256, "BN": 128, "SPLIT": 2})
    assert s24.lib().s24_device_status(None) == 0


def test_mlp_bench_in_microscaled_formats_makes_no_sparse_operand(s24, monkeypatch, capsys):
    """a small case of the benchmark's --mx form, with the sparse path out of reach"""
    import json
    import sys

    import mlp_bench

    def out_of_reach(*args, **kwargs):
        raise AssertionError("called for a run without a sparse operand")

    for name, value in (("M", 512), ("K", 256), ("N", 384)):
        monkeypatch.setattr(mlp_bench, name, value)
    monkeypatch.setattr(s24, "prune_compress", out_of_reach)
    monkeypatch.setattr(mlp_bench, "NShardedSpmm", out_of_reach)
    for name in ("RANK", "WORLD_SIZE", "LOCAL_RANK"):
        monkeypatch.delenv(name, raising=False)
    monkeypatch.setattr(sys, "argv", ["mlp_bench.py", "--mx", "--steps", "2"])
    mlp_bench.main()
    line = json.loads(capsys.readouterr().out.splitlines()[-1])
    assert line["n_gpus"] == 1 and line["mx"]["ms"] > 0
