// mx_norm.cu -- root-mean-square norm with the residual's addition, quantised as it is computed.
//
//   h = round(x + residual)   (or x),   y = h * w / sqrt(mean(h^2) + eps),   (codes, scales) = quantise(y)
//
// y is never rounded to 16 bits in between, and the result is that of the formula in 64 bits: a
// rounding to 8 or 4 bits turns the last bit of y into a whole step of the format wherever y lies at
// a border, so y is carried further than fp32 at the places where it costs little.
//   * the sum of squares is held in fp64 (squares of 16-bit values are exact there), in a fixed order;
//   * 1 / sqrt(.) is computed once per row in fp64 and used as a sum of two fp32 numbers;
//   * each product of the two-step h * rinv * w keeps its rounding error (one fused multiply-add),
//     and the final fp32 y is rounded to odd: an inexact y gets its last bit set, so the one
//     rounding to the element type that follows sees on which side of a border the exact y lies
//     (rounding to odd, then to nearest with at least two bits fewer, is a single rounding).
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
    double eps;
};

// TPR threads per row, NB blocks of 32 elements per thread (block i of a thread: its place in the row + i * TPR);
// a row stays in registers between the sum and the quantisation, so x and the residual are read once.
template <int DT, int FMT, int TPR, int NB>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR)
mx_rms_norm_kernel(const NormParams p)
{
    constexpr int kThreads = TPR < 128 ? 128 : TPR;
    constexpr int kRows = kThreads / TPR;
    constexpr int kWarps = TPR / 32;
    const uint32_t sub = threadIdx.x % TPR;
    const uint32_t r = blockIdx.x * kRows + threadIdx.x / TPR;
    const bool row_ok = r < p.R;

    uint32_t h[NB][16];
    double sum = 0.0;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const uint32_t kb = sub + b * TPR;
        if (!row_ok || kb >= p.KB) {
#pragma unroll
            for (int i = 0; i < 16; ++i) h[b][i] = 0u;
            continue;
        }
        const uint4* x = reinterpret_cast<const uint4*>(p.x + (int64_t)r * p.x_row_bytes + (int64_t)kb * 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 w = x[i];
            h[b][4 * i] = w.x; h[b][4 * i + 1] = w.y; h[b][4 * i + 2] = w.z; h[b][4 * i + 3] = w.w;
        }
        if (p.residual != nullptr) {
            const uint4* res = reinterpret_cast<const uint4*>(p.residual + (int64_t)r * p.r_row_bytes + (int64_t)kb * 64);
            uint4* out = reinterpret_cast<uint4*>(p.h + ((int64_t)r * p.KB + kb) * 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 w = res[i];
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // the fp32 sum of two 16-bit values rounds to 16 bits as the exact sum does
                    // (24 bits are at least twice the type's plus two)
                    const float2 a = unpack2<DT>(h[b][4 * i + j]), c = unpack2<DT>(u[j]);
                    h[b][4 * i + j] = mx::pack2<DT>(a.x + c.x, a.y + c.y);
                }
                out[i] = make_uint4(h[b][4 * i], h[b][4 * i + 1], h[b][4 * i + 2], h[b][4 * i + 3]);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 a = unpack2<DT>(h[b][i]);
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
    const double rinv = 1.0 / sqrt(sum / (double)(p.KB * kBlock) + p.eps);
    const float rhi = (float)rinv;
    const float rlo = (float)(rinv - (double)rhi);

#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const uint32_t kb = sub + b * TPR;
        uint32_t s = 0;
        if (row_ok && kb < p.KB) {
            const uint4* w = reinterpret_cast<const uint4*>(p.weight + (int64_t)kb * 64);
            float y[kBlock];
            uint32_t amax = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 q = w[i];
                const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 a = unpack2<DT>(h[b][4 * i + j]), c = unpack2<DT>(u[j]);
#pragma unroll
                    for (int l = 0; l < 2; ++l) {
                        const float hv = l ? a.y : a.x, wv = l ? c.y : c.x;
                        const float t = hv * rhi;
                        const float t_err = fmaf(hv, rlo, fmaf(hv, rhi, -t));
                        const float v = t * wv;
                        const float v_err = fmaf(t_err, wv, fmaf(t, wv, -v));
                        const float o = round_to_odd(v, v_err);
                        y[8 * i + 2 * j + l] = o;
                        amax = max(amax, magnitude_bits(o));
                    }
                }
            }
            s = scale_code<FMT>(amax);
            const float up = scale_up(s);
#pragma unroll
            for (int i = 0; i < kBlock; ++i) y[i] *= up;
            uint32_t c[Format<FMT>::kBytes / 4];
            encode_block<FMT>(y, s != 255u, c);
            const int64_t at = (int64_t)r * p.KB + kb;
            uint4* dst = reinterpret_cast<uint4*>(p.codes + at * Format<FMT>::kBytes);
#pragma unroll
            for (int i = 0; i < Format<FMT>::kBytes / 16; ++i) dst[i] = make_uint4(c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]);
            if (p.scales != nullptr) p.scales[at] = (uint8_t)s;
        }
        if (p.scales_tc != nullptr) {   // four neighbouring threads hold one word of tensor-core order
            uint32_t word = s << (8 * (threadIdx.x & 3));
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 1);
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2);
            if ((threadIdx.x & 3) == 0 && r < p.R_pad && kb < p.KB_pad)
                *reinterpret_cast<uint32_t*>(p.scales_tc + tc_offset(r, kb, p.KB_pad >> 2)) = word;
        }
    }
}

template <int DT, int FMT, int TPR, int NB>
static int launch_norm(const NormParams& p, cudaStream_t st)
{
    constexpr int kThreads = TPR < 128 ? 128 : TPR;
    constexpr uint32_t kRows = kThreads / TPR;
    mx_rms_norm_kernel<DT, FMT, TPR, NB><<<(p.R_pad + kRows - 1) / kRows, kThreads, 0, st>>>(p);
    return check_cuda(cudaGetLastError(), "mx_rms_norm launch");
}

// One block of 32 elements per thread wherever the row allows it: the smallest power of two of threads that
// covers the row; beyond 1024 threads, 2 or 4 blocks per thread.
template <int DT, int FMT>
static int pick_norm(const NormParams& p, cudaStream_t st)
{
    const uint32_t kb = p.KB_pad;
    if (kb <= 4) return launch_norm<DT, FMT, 4, 1>(p, st);
    if (kb <= 8) return launch_norm<DT, FMT, 8, 1>(p, st);
    if (kb <= 16) return launch_norm<DT, FMT, 16, 1>(p, st);
    if (kb <= 32) return launch_norm<DT, FMT, 32, 1>(p, st);
    if (kb <= 64) return launch_norm<DT, FMT, 64, 1>(p, st);
    if (kb <= 128) return launch_norm<DT, FMT, 128, 1>(p, st);
    if (kb <= 256) return launch_norm<DT, FMT, 256, 1>(p, st);
    if (kb <= 512) return launch_norm<DT, FMT, 512, 1>(p, st);
    if (kb <= 1024) return launch_norm<DT, FMT, 512, 2>(p, st);
    return launch_norm<DT, FMT, 512, 4>(p, st);
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
    auto st = static_cast<cudaStream_t>(stream);
    if (dtype == S24_BF16) return fmt == S24_MXFP4 ? pick_norm<S24_BF16, S24_MXFP4>(p, st) : pick_norm<S24_BF16, S24_MXFP8>(p, st);
    return fmt == S24_MXFP4 ? pick_norm<S24_FP16, S24_MXFP4>(p, st) : pick_norm<S24_FP16, S24_MXFP8>(p, st);
}
