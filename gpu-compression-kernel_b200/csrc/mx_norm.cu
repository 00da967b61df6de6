// mx_norm.cu -- root-mean-square norm with the residual's addition, quantised as it is computed.
//
//   h = round(x + residual)   (or x),   y = h * w / sqrt(mean(h^2) + eps),   (codes, scales) = quantise(y)
//
// y is never rounded to 16 bits in between, and codes and scales are those of the formula in 64 bits,
// h / sqrt(sum(h^2) / K + eps) * w with each operation rounded to fp64: a rounding to 8 or 4 bits turns the
// last bit of y into a whole step of the format wherever y lies at a border, so near one y is computed in
// fp64.
//   * the sum of squares is held in fp64 (squares of 16-bit values are exact there), in a fixed order;
//   * 1 / sqrt(.) is computed once per row in fp64, times 2^64, and rounded to fp32;
//   * 2^64 y is first computed in fp32 (off by at most 2.5 * 2^-24 of itself) and rounded to the element type
//     from both ends of y * (1 +- 2^-21): where the two agree, the code is certain.  The 2^64 stands in for
//     fp32's range, so that h / sqrt(.) may be small beside a large weight: where 2^64 h / sqrt(.) is subnormal,
//     2^64 y is off by at most 2^-150 times the weight, 2^-22, which is nothing in a block whose largest
//     2^64 y is above 2^20; with a row's root below 2^57 none is subnormal, and 2^-100 does.  Other blocks
//     (y below that or from 2^64 on, zeros in a row beyond 2^80) count as not certain.  About one element in
//     10^5 lies nearer to a border; its thread computes y again, in fp64 as the formula reads (a root and a
//     division: a value that the formula puts exactly on a border stays there), and rounds it to fp32 to
//     odd: an inexact y gets its last bit set, so the one rounding to the element type sees on which side
//     of the border y lies (rounding to odd, then to nearest with at least two bits fewer, is a single
//     rounding).
// Values of y from 2^128 on count as infinite.
#include "mx_common.cuh"

namespace s24 {

using namespace mx;

// y in fp32, rounded to odd: towards zero, and the last bit set if that dropped anything
__device__ __forceinline__ float round_to_odd(double y)
{
    if (fabs(y) >= 0x1p128) return y < 0.0 ? -INFINITY : INFINITY;
    const float f = __double2float_rz(y);
    return (double)f == y ? f : __uint_as_float(__float_as_uint(f) | 1u);   // a NaN stays one
}

// 1 / sqrt(m) in fp64 for m >= 1e-30: an fp32 start (22 bits) and two Newton steps, a tenth of the instructions of a
// division of a square root, which cost a fifth of the kernel's time.  m is brought into the fp32 range first.
__device__ __forceinline__ double inverse_sqrt(double m)
{
    const bool big = m >= 0x1p100;
    if (big) m *= 0x1p-160;
    double r = (double)rsqrtf((float)m);
#pragma unroll
    for (int i = 0; i < 2; ++i) r = fma(r * 0.5, fma(-m * r, r, 1.0), r);
    return m == INFINITY ? 0.0 : big ? r * 0x1p-80 : r;
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
    double eps, k, inv_k;
};

// a / b, rounded once, from inv = 1 / b to about its last bit: the remainder of the rounded product is exact in a fused
// multiply-add and corrects it (Markstein, IBM J. Res. Dev. 34, 1990); likewise the root of m from 1 / sqrt(m).  Exact
// quotients and roots come out exactly.  b >= 0 and finite; a zero keeps its sign.  A few instructions each instead of the
// operators' some dozens, which the one thread that needs them would wait for (300 x 4096 5.0 us, so 4.4).
__device__ __forceinline__ double quotient(double a, double b, double inv)
{
    const double q = a * inv;
    return copysign(fma(fma(-q, b, a), inv, q), a);
}

// sqrt(sum / K + eps) of a row and its inverse; both 0 where it is infinite, which makes the quotients 0 or, of infinities, NaN
struct NormRoot {
    double root, inv;
    __device__ __forceinline__ NormRoot(double sum, const NormParams& p)
    {
        const double m = sum == INFINITY ? sum : quotient(sum, p.k, p.inv_k) + p.eps;
        inv = inverse_sqrt(m);
        const double g = m * inv;
        root = m == INFINITY ? 0.0 : fma(fma(-g, g, m), 0.5 * inv, g);
    }
};

// y of one element in fp64, rounded to odd
template <int DT>
__device__ __forceinline__ float norm_exact(const uint8_t* h, const uint8_t* w, const NormRoot& row)
{
    const float hv = unpack2<DT>(*reinterpret_cast<const uint16_t*>(h)).x, wv = unpack2<DT>(*reinterpret_cast<const uint16_t*>(w)).x;
    return round_to_odd(quotient((double)hv, row.root, row.inv) * (double)wv);
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
// What bounds it: with a residual the 7.03 bytes an element (8 bits out): 8192 x 8192 bf16 71.5 us, the measured
// copy rate.  Without one neither bytes nor a pipe: 4099 x 6144 fp16 to 4 bits is 18.8 us for 9.9 us of bytes, at 16
// instructions an element, 52 % of the issue slots (63 % while an SM is active) and no pipe above 35 %.  A CTA's loads, its
// sum and its encoding follow one another, and what warps wait for most is the loads.  The second rounding and what
// follows from it are 11 %.  Steps, 8192 x 8192 with a residual: a block per thread 117 us, an eighth of a block (8 elements)
// per thread 74 to 80, half a block 72.
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
    const float rinv = (float)(inverse_sqrt(sum * p.inv_k + p.eps) * 0x1p64);

    // the largest 2^64 y of a block has to be above 2^20, or above 2^-100 where h of 2^-133 still makes a normal number
    const uint32_t low = rinv < 128.0f ? 0x49800000u : 0x0D800000u;

    uint8_t* codes = p.codes + (int64_t)r * (p.KB * Format<FMT>::kBytes);
    const auto store_scale = [&](uint32_t at, uint32_t s, bool ok) {
        const uint32_t kb = at >> 1;
        if ((threadIdx.x & 1) != 0) return;
        if (p.scales != nullptr && ok) p.scales[(int64_t)r * p.KB + kb] = (uint8_t)s;
        if (p.scales_tc != nullptr && r < p.R_pad && kb < p.KB_pad) p.scales_tc[tc_offset(r, kb, p.KB_pad >> 2)] = ok ? (uint8_t)s : (uint8_t)0;
    };
    constexpr int kBytes = FMT == S24_MXFP4 ? 8 : 16, kWords = kBytes / 4;   // of a piece's codes
    uint32_t todo[NC];   // of a piece: a bit per byte of codes that is not certain, the scale from bit 16, bit 24 where that is not either
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const uint32_t at = sub + c * tpr;
        const bool ok = at < pieces;   // the same for the two threads of a block
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0u;
        if (ok) load32(p.weight + at * 32, w);
        Pair y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 a = unpack2<DT>(h[c][i]), b = unpack2<DT>(w[i]);
            y[i] = make_pair(a.x, a.y) * make_pair(rinv, rinv) * make_pair(b.x, b.y);
        }
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = split(y[i]);
            m = max_magnitude(m, f.x, f.y);
        }
        uint32_t amax = __float_as_uint(m);   // a NaN among them gives a NaN's bits, the largest
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        // a power of two too near to tell the scale, numbers outside low .. 2^128; not a block of zeros that are zeros
        const bool unsure = amax != 0u ? amax - low >= 0x7F800000u - low || ((amax + 8u) & 0x7FFFFFu) < 16u : rinv < 0x1p-16f;
        const uint32_t s = (uint32_t)max((int)(amax >> 23) - 64 - Format<FMT>::kEmax, 0);   // of no use where unsure
        const float up = __uint_as_float((254u - 64u - s) << 23);                       // 2^(127 - s) of y is this of 2^64 y
        uint32_t code[kWords], other[kWords];
        encode_piece<FMT>(y, up * (1.0f - 0x1p-21f), code);
        encode_piece<FMT>(y, up * (1.0f + 0x1p-21f), other);
        if (ok) {
            if constexpr (FMT == S24_MXFP4) *reinterpret_cast<uint2*>(codes + at * 8) = make_uint2(code[0], code[1]);
            else *reinterpret_cast<uint4*>(codes + at * 16) = make_uint4(code[0], code[1], code[2], code[3]);
        }
        store_scale(at, s, ok);
        uint32_t differ = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i) differ |= code[i] ^ other[i];
        todo[c] = ok && unsure ? 1u << 24 : 0u;
        if (ok && !unsure && differ != 0u) {
            todo[c] = s << 16;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {   // which bytes are not zero: the last bit of each, brought together
                uint32_t d = code[i] ^ other[i];
                d |= d >> 4;
                d |= d >> 2;
                d |= d >> 1;
                todo[c] |= ((d & 0x01010101u) * 0x01020408u >> 24) << (4 * i);
            }
        }
    }

    // What was not certain, again in fp64; h and w are read once more.  Here and not in the loop above, whose registers it
    // would take (44 bytes of spills there).
    uint32_t any = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) any |= todo[c];
    if (!__any_sync(0xFFFFFFFFu, any != 0u)) return;
    const NormRoot row(sum, p);
    const uint8_t* h_row = p.residual != nullptr ? p.h + (int64_t)r * (p.KB * 64) : p.x + (int64_t)r * p.x_row_bytes;
#pragma unroll 1
    for (int c = 0; c < NC; ++c) {
        uint32_t t = todo[0];
#pragma unroll
        for (int i = 1; i < NC; ++i) t = c == i ? todo[i] : t;
        const uint32_t at = sub + c * tpr;
        const uint8_t *h_at = h_row + at * 32, *w_at = p.weight + at * 32;
        uint32_t s = (t >> 16) & 0xFFu;
        const bool unsure = (t >> 24) != 0u;   // the same for the two threads of a block
        if (__any_sync(0xFFFFFFFFu, unsure)) {
            uint32_t amax = 0;
            if (unsure) {
#pragma unroll 1
                for (int e = 0; e < 16; ++e) amax = max(amax, magnitude_bits(norm_exact<DT>(h_at + 2 * e, w_at + 2 * e, row)));
            }
            amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
            if (unsure) {
                s = scale_code<FMT>(amax);
                store_scale(at, s, true);
                t = kBytes == 16 ? 0xFFFFu : 0xFFu;
            }
        }
        const float up = scale_up(s);
        t &= 0xFFFFu;
#pragma unroll 1
        while (t != 0u) {
            const int byte = __ffs((int)t) - 1, e = byte * (16 / kBytes);
            float v[8] = {};
            v[0] = norm_exact<DT>(h_at + 2 * e, w_at + 2 * e, row) * up;
            if (FMT == S24_MXFP4) v[1] = norm_exact<DT>(h_at + 2 * e + 2, w_at + 2 * e + 2, row) * up;
            const uint32_t q = s == 255u ? 0u : FMT == S24_MXFP4 ? to_e2m1x8(v) : to_e4m3x4(v);
            codes[at * kBytes + byte] = (uint8_t)q;
            t &= t - 1u;
        }
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
    p.k = (double)K;
    p.inv_k = 1.0 / (double)K;
    auto st = static_cast<cudaStream_t>(stream);
    if (dtype == S24_BF16) return fmt == S24_MXFP4 ? pick_norm<S24_BF16, S24_MXFP4>(p, st) : pick_norm<S24_BF16, S24_MXFP8>(p, st);
    return fmt == S24_MXFP4 ? pick_norm<S24_FP16, S24_MXFP4>(p, st) : pick_norm<S24_FP16, S24_MXFP8>(p, st);
}
