// mx_norm.cu -- root-mean-square norm with the residual's addition, quantised as it is computed.
//
//   h = round(x + residual)   (or x),   y = h * w / sqrt(mean(h^2) + eps),   (codes, scales) = quantise(y)
//
// y is never rounded to 16 bits in between, and codes and scales are those of the formula in 64 bits: a
// rounding to 8 or 4 bits turns the last bit of y into a whole step of the format wherever y lies at a
// border, so near one y is carried further than fp32.
//   * the sum of squares is held in fp64 (squares of 16-bit values are exact there), in a fixed order;
//   * 1 / sqrt(.) is computed once per row in fp64 and used as a sum of two fp32 numbers;
//   * y is first computed in fp32 (off by at most 2.5 * 2^-24 of itself) and rounded to the element type
//     from both ends of y * (1 +- 2^-21): where the two agree, the code is certain.  About one element in
//     10^5 lies nearer to a border; its thread computes y again with the rounding error of each product
//     kept (one fused multiply-add) and rounds it to odd: an inexact y gets its last bit set, so the one
//     rounding to the element type sees on which side of the border y lies (rounding to odd, then to
//     nearest with at least two bits fewer, is a single rounding).
// Values of y beyond the fp32 range count as infinite.
#include "mx_common.cuh"

namespace s24 {

using namespace mx;

// value + error, where value is the nearest fp32 number to the sum, rounded to odd
__device__ __forceinline__ float round_to_odd(float value, float error)
{
    const uint32_t b = __float_as_uint(value), e = __float_as_uint(error);
    const uint32_t exponent = b & 0x7F800000u;
    // even and inexact: the odd neighbour towards the exact value
    if (error != 0.0f && !(b & 1u) && exponent != 0x7F800000u && (b & 0x7FFFFFFFu) != 0u)
        return __uint_as_float(((b ^ e) >> 31) ? b - 1u : b + 1u);
    return value;
}

// 1 / sqrt(m) in fp64: an fp32 start (22 bits) and two Newton steps, a tenth of the instructions of a division of a
// square root, which cost a fifth of the kernel's time
__device__ __forceinline__ double inverse_sqrt(double m)
{
    if (!(m < 1e38)) return 1.0 / sqrt(m);   // beyond fp32, or not a number
    double r = (double)rsqrtf((float)m);
#pragma unroll
    for (int i = 0; i < 2; ++i) r = fma(r * 0.5, fma(-m * r, r, 1.0), r);
    return r;
}

struct NormParams {
    const uint8_t* x;
    const uint8_t* residual;   // null: h = x and is not written
    const uint8_t* weight;
    uint8_t* h;
    uint8_t* codes;
    uint8_t* scales;
    uint8_t* scales_tc;
    int64_t x_row_bytes, r_row_bytes;
    uint32_t R, R_pad, KB, KB_pad;   // rows, rows to visit (whole records with scales_tc), blocks a row, blocks of whole chunks
    double eps, inv_k;
};


// The exact form of one value of y = h * rinv * w with rinv = rhi + rlo, rounded to odd.  h and w are read again: this runs
// for one element in 10^5, and registers that it kept would be the common path's.
template <int DT>
__device__ __forceinline__ float norm_exact(const uint8_t* h, const uint8_t* w, float rhi, float rlo)
{
    const float hv = unpack2<DT>(*reinterpret_cast<const uint16_t*>(h)).x, wv = unpack2<DT>(*reinterpret_cast<const uint16_t*>(w)).x;
    const float t = hv * rhi;
    const float t_err = fmaf(hv, rlo, fmaf(hv, rhi, -t));
    const float v = t * wv;
    const float v_err = fmaf(t_err, wv, fmaf(t, wv, -v));   // as much as two units in the last place of v,
    const float y = v + v_err;                              // so the pair is brought to a nearest value and its rest
    return round_to_odd(y, v_err - (y - v));
}

// codes of a piece times up
template <int FMT>
__device__ __forceinline__ void encode_piece(const Pair (&y)[8], float up, uint32_t (&c)[FMT == S24_MXFP4 ? 2 : 4])
{
    float u[16];
    const Pair up2 = make_pair(up, up);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = split(y[i] * up2);
        u[2 * i] = f.x;
        u[2 * i + 1] = f.y;
    }
#pragma unroll
    for (int i = 0; i < (FMT == S24_MXFP4 ? 2 : 4); ++i) c[i] = FMT == S24_MXFP4 ? to_e2m1x8(u + 8 * i) : to_e4m3x4(u + 4 * i);
}

// A row belongs to TPR threads (4 to 32) of a CTA of 128, or, with TPR = 0, to a whole CTA of as many warps as it takes.
// Two threads hold a block of 32 elements: thread t takes elements 16 t .. 16 t + 15 and every 16 TPR further, NC pieces in
// all, 32 bytes each, so that a warp's accesses are whole lines.  The row stays in registers between the sum and the
// quantisation: x and the residual are read once.
//
// What bounds it: with a residual the 7.03 bytes an element (8 bits out), without one the instructions, about 14 an
// element.  Measured, 8192 x 8192 bf16 with a residual: a block per thread 117 us, an eighth of a block (8 elements) per
// thread 74 to 80 us with 22 to 28 instructions an element; 4099 x 6144 fp16 to 4 bits 34, 25 to 27 us.
template <int DT, int FMT, int TPR, int NC>
__global__ void __launch_bounds__(TPR == 0 ? 1024 : 128, TPR == 0 ? 1 : 8)
mx_rms_norm_kernel(const NormParams p)
{
    const uint32_t tpr = TPR == 0 ? blockDim.x : TPR;
    const uint32_t sub = TPR == 0 ? threadIdx.x : threadIdx.x % (TPR == 0 ? 1 : TPR);
    const uint32_t r = TPR == 0 ? blockIdx.x : blockIdx.x * (128 / (TPR == 0 ? 1 : TPR)) + threadIdx.x / (TPR == 0 ? 1 : TPR);
    const uint32_t pieces = r < p.R ? p.KB * 2 : 0;

    wait_for_predecessors();   // and no early start of the next kernel: its CTAs would share the issue slots that this one lives on
    uint32_t h[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const uint32_t at = sub + c * tpr;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[c][i] = 0u;
        if (at < pieces) load32(p.x + (int64_t)r * p.x_row_bytes + at * 32, h[c]);
    }
    if (p.residual != nullptr) {
        uint32_t v[NC][8];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const uint32_t at = sub + c * tpr;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = 0u;
            if (at < pieces) load32(p.residual + (int64_t)r * p.r_row_bytes + at * 32, v[c]);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const uint32_t at = sub + c * tpr;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // the fp32 sum of two 16-bit values rounds to 16 bits as the exact sum does
                // (24 bits are at least twice the type's plus two)
                const float2 a = unpack2<DT>(h[c][i]), b = unpack2<DT>(v[c][i]);
                const float2 f = split(make_pair(a.x, a.y) + make_pair(b.x, b.y));
                h[c][i] = mx::pack2<DT>(f.x, f.y);
            }
            if (at < pieces) store32(p.h + (int64_t)r * (p.KB * 64) + at * 32, h[c]);
        }
    }
    double s0 = 0.0, s1 = 0.0;   // two chains: one alone waits for itself
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 a = unpack2<DT>(h[c][i]);
            s0 = fma((double)a.x, (double)a.x, s0);
            s1 = fma((double)a.y, (double)a.y, s1);
        }
    }
    double sum = s0 + s1;
#pragma unroll
    for (int o = (TPR == 0 ? 32 : TPR) / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if constexpr (TPR == 0) {
        __shared__ double part[32];
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = part[0];
        for (uint32_t i = 1; i < blockDim.x >> 5; ++i) sum += part[i];
    }
    const double rinv = inverse_sqrt(sum * p.inv_k + p.eps);
    const float rhi = (float)rinv;
    const float rlo = (float)(rinv - (double)rhi);

    uint8_t* codes = p.codes + (int64_t)r * (p.KB * Format<FMT>::kBytes);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const uint32_t at = sub + c * tpr, kb = at >> 1;
        const bool ok = at < pieces;   // the same for the two threads of a block
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0u;
        if (ok) load32(p.weight + at * 32, w);
        Pair y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 a = unpack2<DT>(h[c][i]), b = unpack2<DT>(w[i]);
            y[i] = make_pair(a.x, a.y) * make_pair(rhi, rhi) * make_pair(b.x, b.y);
        }
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = split(y[i]);
            m = max_magnitude(m, f.x, f.y);
        }
        uint32_t amax = __float_as_uint(m);   // a NaN among them gives a NaN's bits, the largest
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        const uint8_t* h_at = (p.residual != nullptr ? p.h + (int64_t)r * (p.KB * 64) : p.x + (int64_t)r * p.x_row_bytes) + at * 32;
        const uint8_t* w_at = p.weight + at * 32;
        // a power of two too near to tell the scale, or numbers too small for fp32's own rounding; not a block of zeros
        const bool unsure = amax != 0u && (((amax + 8u) & 0x7FFFFFu) < 16u || amax <= 0x0E800000u);
        if (__any_sync(0xFFFFFFFFu, unsure)) {
            uint32_t exact = 0;
            if (ok && unsure) {
#pragma unroll 1
                for (int e = 0; e < 16; ++e) exact = max(exact, magnitude_bits(norm_exact<DT>(h_at + 2 * e, w_at + 2 * e, rhi, rlo)));
            }
            exact = max(exact, __shfl_xor_sync(0xFFFFFFFFu, exact, 1));
            if (unsure) amax = exact;
        }
        const uint32_t s = scale_code<FMT>(amax);
        const float up = scale_up(s);
        constexpr int kWords = FMT == S24_MXFP4 ? 2 : 4, kBits = FMT == S24_MXFP4 ? 4 : 8;
        uint32_t code[kWords], other[kWords];
        encode_piece<FMT>(y, up * (1.0f - 0x1p-21f), code);
        encode_piece<FMT>(y, up * (1.0f + 0x1p-21f), other);
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            uint32_t d = ok ? (unsure ? 0xFFFFFFFFu : code[i] ^ other[i]) : 0u;
#pragma unroll 1
            while (d != 0u) {   // an element that the two do not agree on
                const int e = (__ffs((int)d) - 1) / kBits;
                const uint32_t mask = ((1u << kBits) - 1u) << (e * kBits);
                const int at_e = 2 * (i * (32 / kBits) + e);
                float one[8] = {norm_exact<DT>(h_at + at_e, w_at + at_e, rhi, rlo) * up, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                const uint32_t q = FMT == S24_MXFP4 ? to_e2m1x8(one) : to_e4m3x4(one);
                code[i] = (code[i] & ~mask) | ((q << (e * kBits)) & mask);
                d &= ~mask;
            }
        }
        if (s == 255u) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) code[i] = 0u;
        }
        if (ok) {
            if constexpr (FMT == S24_MXFP4) *reinterpret_cast<uint2*>(codes + at * 8) = make_uint2(code[0], code[1]);
            else *reinterpret_cast<uint4*>(codes + at * 16) = make_uint4(code[0], code[1], code[2], code[3]);
            if (p.scales != nullptr && (threadIdx.x & 1) == 0) p.scales[(int64_t)r * p.KB + kb] = (uint8_t)s;
        }
        if (p.scales_tc != nullptr && (threadIdx.x & 1) == 0 && r < p.R_pad && kb < p.KB_pad)
            p.scales_tc[tc_offset(r, kb, p.KB_pad >> 2)] = ok ? (uint8_t)s : (uint8_t)0;
    }
}

template <int DT, int FMT, int TPR, int NC>
static int launch_norm(const NormParams& p, int threads, cudaStream_t st)
{
    const uint32_t rows = TPR == 0 ? 1 : 128 / (TPR == 0 ? 1 : TPR);
    return check_cuda(launch_overlapped(mx_rms_norm_kernel<DT, FMT, TPR, NC>, dim3((p.R_pad + rows - 1) / rows), (unsigned)threads, 0, 1, st, p), "mx_rms_norm launch");
}

// Two pieces of 16 elements per thread: rows of at most 1024 share a CTA, longer ones have as many warps as it takes, and
// beyond 32768 elements the 1024 threads take four pieces each.  Few rows take one piece per thread: nothing but a row's
// latency counts then (16 x 8192 3.4 -> 3.0 us; 8192 x 8192 would take 90 instead of 72).
template <int DT, int FMT>
static int pick_norm(const NormParams& p, cudaStream_t st)
{
    const int threads = (int)((p.KB_pad + 31) / 32 * 32);   // KB_pad blocks are 2 KB_pad pieces
    const int single = (int)((p.KB_pad * 2 + 31) / 32 * 32);
    if (p.R <= (uint32_t)sm_count() && single > 64 && single <= 1024) return launch_norm<DT, FMT, 0, 1>(p, single, st);
    if (threads > 1024) return launch_norm<DT, FMT, 0, 4>(p, 1024, st);
    if (threads > 32) return launch_norm<DT, FMT, 0, 2>(p, threads, st);
    if (p.KB_pad > 16) return launch_norm<DT, FMT, 32, 2>(p, 128, st);
    if (p.KB_pad > 8) return launch_norm<DT, FMT, 16, 2>(p, 128, st);
    if (p.KB_pad > 4) return launch_norm<DT, FMT, 8, 2>(p, 128, st);
    return launch_norm<DT, FMT, 4, 2>(p, 128, st);
}

}  // namespace s24

using namespace s24;

extern "C" int s24_mx_rms_norm(const void* x, const void* residual, const void* weight, void* h, int64_t R, int64_t K, int64_t ldx,
                               int64_t ldr, double eps, int dtype, int fmt, void* codes, void* scales, void* scales_tc, void* stream)
{
    if (dtype != S24_FP16 && dtype != S24_BF16) return fail(S24_ERR_INVALID_ARG, "mx_rms_norm: bad dtype %d", dtype);
    if (fmt != S24_MXFP4 && fmt != S24_MXFP8) return fail(S24_ERR_INVALID_ARG, "mx_rms_norm: bad format %d", fmt);
    if (!(eps >= 1e-30 && eps <= 1e30)) return fail(S24_ERR_INVALID_ARG, "mx_rms_norm: eps must be between 1e-30 and 1e30 (got %g)", eps);
    if (R < 0 || K < 0 || K % kBlock != 0)
        return fail(S24_ERR_SHAPE, "mx_rms_norm: needs R >= 0 and K a multiple of 32 (got R=%lld K=%lld)", (long long)R, (long long)K);
    if (K > S24_MX_NORM_MAX_K) return fail(S24_ERR_UNSUPPORTED, "mx_rms_norm: rows of at most %d elements (got %lld)", S24_MX_NORM_MAX_K, (long long)K);
    if (R > 0x7FFFFF00ll) return fail(S24_ERR_SHAPE, "mx_rms_norm: dimension too large");
    if (R == 0 || K == 0) return S24_OK;
    if (x == nullptr || weight == nullptr || codes == nullptr || (scales == nullptr && scales_tc == nullptr) || (residual != nullptr && h == nullptr))
        return fail(S24_ERR_INVALID_ARG, "mx_rms_norm: null pointer");
    if (ldx < K || ldx > (INT64_MAX >> 2) / R || ldx % 16 != 0 || (residual != nullptr && (ldr < K || ldr > (INT64_MAX >> 2) / R || ldr % 16 != 0)))
        return fail(S24_ERR_SHAPE, "mx_rms_norm: row strides must be >= K and multiples of 16 (got %lld, %lld)", (long long)ldx, (long long)ldr);
    if (!aligned(x, 32) || !aligned(residual, 32) || !aligned(weight, 32) || (residual != nullptr && !aligned(h, 32)) || !aligned(codes, 16) ||
        !aligned(scales_tc, 16))
        return fail(S24_ERR_INVALID_ARG, "mx_rms_norm: x, residual, weight and h must be 32-byte aligned, codes and scales_tc 16");
    NormParams p;
    p.x = static_cast<const uint8_t*>(x);
    p.residual = static_cast<const uint8_t*>(residual);
    p.weight = static_cast<const uint8_t*>(weight);
    p.h = static_cast<uint8_t*>(h);
    p.codes = static_cast<uint8_t*>(codes);
    p.scales = static_cast<uint8_t*>(scales);
    p.scales_tc = static_cast<uint8_t*>(scales_tc);
    p.x_row_bytes = ldx * 2;
    p.r_row_bytes = ldr * 2;
    p.R = (uint32_t)R;
    p.R_pad = scales_tc ? (uint32_t)(row_tiles(R) * 128) : (uint32_t)R;
    p.KB = (uint32_t)(K / kBlock);
    p.KB_pad = (uint32_t)(k_chunks(K) * 4);
    p.eps = eps;
    p.inv_k = 1.0 / (double)K;
    auto st = static_cast<cudaStream_t>(stream);
    if (dtype == S24_BF16) return fmt == S24_MXFP4 ? pick_norm<S24_BF16, S24_MXFP4>(p, st) : pick_norm<S24_BF16, S24_MXFP8>(p, st);
    return fmt == S24_MXFP4 ? pick_norm<S24_FP16, S24_MXFP4>(p, st) : pick_norm<S24_FP16, S24_MXFP8>(p, st);
}
