"""The microscaled formats in 64-bit numpy, from their definition: element values are looked up in the list of
numbers that the element type has, scales by comparison with the powers of two."""
import numpy as np

BLOCK = 32


def element_values(bits):
    """the element type's non-negative finite values, in code order"""
    fraction, low, top, largest = (1, 0, 2, 6.0) if bits == 4 else (3, -6, 8, 448.0)
    n = 1 << fraction
    v = [2.0 ** low * i / n for i in range(n)] + [2.0 ** e * (1 + i / n) for e in range(low, top + 1) for i in range(n)]
    return np.array([x for x in v if x <= largest])


def quantize(x, bits):
    """codes (R, K) uint8, one element each, and scales (R, K / 32) uint8 of a float64 matrix"""
    r, k = x.shape
    emax = 2 if bits == 4 else 8
    blocks = x.astype(np.float64).reshape(r, k // BLOCK, BLOCK)
    finite = np.isfinite(blocks).all(-1)
    blocks = np.where(finite[..., None], blocks, 0.0)
    amax = np.abs(blocks).max(-1)
    # floor(log2 amax) as the number of powers of two not above it
    powers = np.ldexp(1.0, np.arange(-400, 200))
    exponent = np.searchsorted(powers, amax, side="right") - 1 - 400
    scale = np.where(amax > 0, np.clip(exponent - emax + 127, 0, 254), 0)
    mag = np.abs(blocks) / np.ldexp(1.0, scale - 127)[..., None]
    table = element_values(bits)
    middle = (table[1:] + table[:-1]) / 2
    below, through = np.searchsorted(middle, mag, side="left"), np.searchsorted(middle, mag, side="right")
    code = np.where((below != through) & (below % 2 == 1), through, below)     # a tie goes to the even code
    code = code | np.where(np.signbit(blocks), 8 if bits == 4 else 128, 0)
    code = np.where(finite[..., None], code, 0)
    return code.reshape(r, k).astype(np.uint8), np.where(finite, scale, 255).astype(np.uint8)


def pack(code, bits):
    return code if bits == 8 else (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed, bits):
    if bits == 8:
        return packed
    out = np.empty((*packed.shape[:-1], 2 * packed.shape[-1]), np.uint8)
    out[..., 0::2], out[..., 1::2] = packed & 15, packed >> 4
    return out


def dequantize(code, scale, bits):
    """float64 values of one-element-each codes"""
    sign = 8 if bits == 4 else 128
    table = element_values(bits)
    table = np.concatenate([table, np.full(sign - len(table), np.nan)])
    v = np.where(code >= sign, -1.0, 1.0) * table[code % sign]
    s = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(np.int64) - 127))
    return (v.reshape(*scale.shape, BLOCK) * s[..., None]).reshape(code.shape)


def tc_order(scale):
    """(R, K / 32) scales in tensor-core order, byte by byte"""
    r, kb = scale.shape
    chunks = -(-kb // 4)
    out = np.zeros(-(-r // 128) * chunks * 512, np.uint8)
    i, j = np.meshgrid(np.arange(r), np.arange(kb), indexing="ij")
    out[((i // 128) * chunks + j // 4) * 512 + (i % 32) * 16 + (i % 128) // 32 * 4 + j % 4] = scale
    return out


def rms_norm(x, residual, weight, eps, round_h):
    """(h, y) in float64; round_h rounds to the activations' type"""
    h = x if residual is None else round_h(x + residual)
    with np.errstate(invalid="ignore"):
        y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * weight
    return h, y
