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

// value + error, |error| below one unit in the last place of value, rounded to odd
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

// eight values of y, rounded to odd
template <int DT>
__device__ __forceinline__ void norm_exact(const uint32_t (&h)[4], const uint32_t (&w)[4], float rhi, float rlo, Pair (&y)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = unpack2<DT>(h[i]), c = unpack2<DT>(w[i]);
        float o[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float hv = j ? a.y : a.x, wv = j ? c.y : c.x;
            const float t = hv * rhi;
            const float t_err = fmaf(hv, rlo, fmaf(hv, rhi, -t));
            const float v = t * wv;
            o[j] = round_to_odd(v, fmaf(t_err, wv, fmaf(t, wv, -v)));
        }
        y[i] = make_pair(o[0], o[1]);
    }
}

// codes of eight values (four pairs) times up
template <int FMT>
__device__ __forceinline__ void encode8(const Pair (&y)[4], float up, uint32_t (&c)[FMT == S24_MXFP4 ? 1 : 2])
{
    float u[8];
    const Pair up2 = make_pair(up, up);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = split(y[i] * up2);
        u[2 * i] = f.x;
        u[2 * i + 1] = f.y;
    }
    if constexpr (FMT == S24_MXFP4) {
        c[0] = to_e2m1x8(u);
    } else {
        c[0] = to_e4m3x4(u);
        c[1] = to_e4m3x4(u + 4);
    }
}

// bits of the largest magnitude of eight values; a NaN among them gives the bits of a NaN
__device__ __forceinline__ uint32_t max8(const Pair (&y)[4])
{
    const float2 a = split(y[0]), b = split(y[1]), c = split(y[2]), d = split(y[3]);
    return __float_as_uint(max_magnitude(max_magnitude(a.x, a.y, b.x), max_magnitude(b.y, c.x, c.y), max_magnitude(d.x, d.y, 0.0f)));
}

// over the four threads that hold a block
__device__ __forceinline__ uint32_t max_of_block(uint32_t m)
{
    const uint32_t mask = 0xFu << (threadIdx.x & 28);
    m = max(m, __shfl_xor_sync(mask, m, 1));
    return max(m, __shfl_xor_sync(mask, m, 2));
}

// TPR threads per row, four to a block of 32 elements: thread t takes elements 8 t .. 8 t + 7 and every 8 TPR further, NC
// pieces in all, so that a warp's loads and stores are whole lines (with a block per thread the same kernel took 117 us
// instead of 78 at 8192 x 8192 with a residual: 18 accesses of 16 lines each per warp).  A row stays in registers between
// the sum and the quantisation: x and the residual are read once.
template <int DT, int FMT, int TPR, int NC>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR)
mx_rms_norm_kernel(const NormParams p)
{
    constexpr int kThreads = TPR < 128 ? 128 : TPR;
    constexpr int kRows = kThreads / TPR;
    constexpr int kWarps = TPR / 32;
    const uint32_t sub = threadIdx.x % TPR;
    const uint32_t r = blockIdx.x * kRows + threadIdx.x / TPR;
    const uint32_t pieces = r < p.R ? p.KB * 4 : 0;   // of eight elements

    uint32_t h[NC][4];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const uint32_t at = sub + c * TPR;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (at < pieces) v = reinterpret_cast<const uint4*>(p.x + (int64_t)r * p.x_row_bytes)[at];
        h[c][0] = v.x; h[c][1] = v.y; h[c][2] = v.z; h[c][3] = v.w;
    }
    if (p.residual != nullptr) {
        uint4 v[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const uint32_t at = sub + c * TPR;
            v[c] = make_uint4(0u, 0u, 0u, 0u);
            if (at < pieces) v[c] = reinterpret_cast<const uint4*>(p.residual + (int64_t)r * p.r_row_bytes)[at];
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const uint32_t at = sub + c * TPR;
            const uint32_t u[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // the fp32 sum of two 16-bit values rounds to 16 bits as the exact sum does
                // (24 bits are at least twice the type's plus two)
                const float2 a = unpack2<DT>(h[c][i]), b = unpack2<DT>(u[i]);
                const float2 f = split(make_pair(a.x, a.y) + make_pair(b.x, b.y));
                h[c][i] = mx::pack2<DT>(f.x, f.y);
            }
            if (at < pieces) reinterpret_cast<uint4*>(p.h + (int64_t)r * p.KB * 64)[at] = make_uint4(h[c][0], h[c][1], h[c][2], h[c][3]);
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpack2<DT>(h[c][i]);
            sum = fma((double)a.x, (double)a.x, sum);
            sum = fma((double)a.y, (double)a.y, sum);
        }
    }
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if constexpr (kWarps > 1) {
        __shared__ double part[kRows][kWarps];
        const uint32_t own = threadIdx.x / TPR;
        if ((threadIdx.x & 31) == 0) part[own][sub >> 5] = sum;
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) sum += part[own][i];
    }
    const double rinv = inverse_sqrt(sum * p.inv_k + p.eps);
    const float rhi = (float)rinv;
    const float rlo = (float)(rinv - (double)rhi);

#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const uint32_t at = sub + c * TPR, kb = at >> 2;
        uint32_t s = 0;
        if (at < pieces) {   // the same for the four threads of a block
            const uint4 q = reinterpret_cast<const uint4*>(p.weight)[at];
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
            Pair y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = unpack2<DT>(h[c][i]), b = unpack2<DT>(w[i]);
                y[i] = make_pair(a.x, a.y) * make_pair(rhi, rhi) * make_pair(b.x, b.y);
            }
            uint32_t amax = max_of_block(max8(y));
            // a power of two too near to tell the scale, or numbers too small for fp32's own rounding
            bool exact = ((amax + 8u) & 0x7FFFFFu) < 16u || amax - 1u < 0x0E800000u;
            if (exact) {
                norm_exact<DT>(h[c], w, rhi, rlo, y);
                amax = max_of_block(max8(y));
            }
            s = scale_code<FMT>(amax);
            const float up = scale_up(s);
            constexpr int kWords = FMT == S24_MXFP4 ? 1 : 2;
            uint32_t code[kWords], other[kWords];
            encode8<FMT>(y, exact ? up : up * (1.0f - 0x1p-21f), code);
            encode8<FMT>(y, exact ? up : up * (1.0f + 0x1p-21f), other);
            bool differ = code[0] != other[0];
            if (kWords == 2) differ = differ || code[kWords - 1] != other[kWords - 1];
            if (differ && s != 255u) {
                norm_exact<DT>(h[c], w, rhi, rlo, y);
                encode8<FMT>(y, up, code);
            }
            if (s == 255u) {
#pragma unroll
                for (int i = 0; i < kWords; ++i) code[i] = 0u;
            }
            uint8_t* dst = p.codes + (int64_t)r * p.KB * Format<FMT>::kBytes;
            if constexpr (FMT == S24_MXFP4) reinterpret_cast<uint32_t*>(dst)[at] = code[0];
            else reinterpret_cast<uint2*>(dst)[at] = make_uint2(code[0], code[1]);
            if (p.scales != nullptr && (threadIdx.x & 3) == 0) p.scales[(int64_t)r * p.KB + kb] = (uint8_t)s;
        }
        if (p.scales_tc != nullptr && (threadIdx.x & 3) == 0 && r < p.R_pad && kb < p.KB_pad)
            p.scales_tc[tc_offset(r, kb, p.KB_pad >> 2)] = (uint8_t)s;
    }
}

template <int DT, int FMT, int TPR, int NC>
static int launch_norm(const NormParams& p, cudaStream_t st)
{
    constexpr int kThreads = TPR < 128 ? 128 : TPR;
    constexpr uint32_t kRows = kThreads / TPR;
    mx_rms_norm_kernel<DT, FMT, TPR, NC><<<(p.R_pad + kRows - 1) / kRows, kThreads, 0, st>>>(p);
    return check_cuda(cudaGetLastError(), "mx_rms_norm launch");
}

// Four pieces of eight elements per thread, a block's worth, wherever the row allows it: the smallest power of two of
// threads that covers the row; beyond 512 threads, 8 or 16 pieces per thread.
template <int DT, int FMT>
static int pick_norm(const NormParams& p, cudaStream_t st)
{
    const uint32_t kb = p.KB_pad;
    if (kb <= 4) return launch_norm<DT, FMT, 4, 4>(p, st);
    if (kb <= 8) return launch_norm<DT, FMT, 8, 4>(p, st);
    if (kb <= 16) return launch_norm<DT, FMT, 16, 4>(p, st);
    if (kb <= 32) return launch_norm<DT, FMT, 32, 4>(p, st);
    if (kb <= 64) return launch_norm<DT, FMT, 64, 4>(p, st);
    if (kb <= 128) return launch_norm<DT, FMT, 128, 4>(p, st);
    if (kb <= 256) return launch_norm<DT, FMT, 256, 4>(p, st);
    if (kb <= 512) return launch_norm<DT, FMT, 512, 4>(p, st);
    if (kb <= 1024) return launch_norm<DT, FMT, 512, 8>(p, st);
    return launch_norm<DT, FMT, 512, 16>(p, st);
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
    if (ldx < K || ldx > (INT64_MAX >> 2) / R || ldx % 8 != 0 || (residual != nullptr && (ldr < K || ldr > (INT64_MAX >> 2) / R || ldr % 8 != 0)))
        return fail(S24_ERR_SHAPE, "mx_rms_norm: row strides must be >= K and multiples of 8 (got %lld, %lld)", (long long)ldx, (long long)ldr);
    if (!aligned(x, 16) || !aligned(residual, 16) || !aligned(weight, 16) || !aligned(h, 16) || !aligned(codes, 16) || !aligned(scales_tc, 16))
        return fail(S24_ERR_INVALID_ARG, "mx_rms_norm: pointers must be 16-byte aligned");
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
