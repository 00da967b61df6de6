// mx_quantize.cu -- block quantisation to the microscaled formats, reading back, and the re-layout
// of scales.
#include "mx_common.cuh"

namespace s24 {

using namespace mx;

constexpr int kQuantThreads = 256;

// scale code and codes of a block
template <int FMT>
__device__ __forceinline__ uint32_t quantize_block(const Pair (&v)[kBlock / 2], uint32_t (&c)[Format<FMT>::kBytes / 4])
{
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < kBlock / 2; ++i) {
        const float2 f = split(v[i]);
        m = max_magnitude(m, f.x, f.y);
    }
    const uint32_t s = scale_code<FMT>(__float_as_uint(m));   // a NaN among them gives a NaN's bits
    const float up = scale_up(s);
    float u[kBlock];
#pragma unroll
    for (int i = 0; i < kBlock / 2; ++i) {
        const float2 f = split(v[i] * make_pair(up, up));
        u[2 * i] = f.x;
        u[2 * i + 1] = f.y;
    }
    encode_block<FMT>(u, s != 255u, c);
    return s;
}

// One thread per block of 32 elements; four neighbouring threads share a 128-column chunk and put its
// scales together into the one word that tensor-core order keeps together.  With TC the index space
// covers whole 128 x 128 records, and threads outside the matrix only write the filler scale 0.
template <int DT, int FMT, bool TC>
__global__ void __launch_bounds__(kQuantThreads)
mx_quantize_kernel(const uint8_t* __restrict__ x, uint32_t R, uint32_t KB, uint32_t KB_pad, uint32_t total, int64_t row_bytes,
                   uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, uint8_t* __restrict__ scales_tc)
{
    constexpr int kElem = DT == S24_FP32 ? 4 : 2;
    const uint32_t t = blockIdx.x * kQuantThreads + threadIdx.x;
    const uint32_t r = t / KB_pad, kb = t - r * KB_pad;
    uint32_t s = 0;
    start_dependents();
    wait_for_predecessors();
    if (t < total && r < R && kb < KB) {
        const uint8_t* src = x + (int64_t)r * row_bytes + (int64_t)kb * (kBlock * kElem);
        Pair v[kBlock / 2];
#pragma unroll
        for (int i = 0; i < kElem; ++i) {
            uint32_t u[8];
            load32(src + 32 * i, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (DT == S24_FP32) {
                    if (j & 1) v[4 * i + j / 2] = make_pair(__uint_as_float(u[j - 1]), __uint_as_float(u[j]));
                } else {
                    const float2 f = unpack2<DT>(u[j]);
                    v[8 * i + j] = make_pair(f.x, f.y);
                }
            }
        }
        uint32_t c[Format<FMT>::kBytes / 4];
        s = quantize_block<FMT>(v, c);
        const int64_t at = (int64_t)r * KB + kb;
        if constexpr (FMT == S24_MXFP4) *reinterpret_cast<uint4*>(codes + at * 16) = make_uint4(c[0], c[1], c[2], c[3]);
        else store32(codes + at * 32, c);
        if (scales != nullptr) scales[at] = (uint8_t)s;
    }
    if constexpr (TC) {
        uint32_t word = s << (8 * (threadIdx.x & 3));
        word |= __shfl_xor_sync(0xFFFFFFFFu, word, 1);
        word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2);
        if (t < total && (threadIdx.x & 3) == 0) *reinterpret_cast<uint32_t*>(scales_tc + tc_offset(r, kb, KB_pad >> 2)) = word;
    }
}

// One thread per block.
template <int DT, int FMT>
__global__ void __launch_bounds__(kQuantThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int tc, uint32_t KB, uint32_t total,
                     uint8_t* __restrict__ out)
{
    constexpr int kElem = DT == S24_FP32 ? 4 : 2;
    const uint32_t t = blockIdx.x * kQuantThreads + threadIdx.x;
    start_dependents();
    wait_for_predecessors();
    if (t >= total) return;
    const uint32_t r = t / KB, kb = t - r * KB;
    const float s = scale_value(scales[tc ? tc_offset(r, kb, (KB + 3) / 4) : (int64_t)t]);
    const uint8_t* src = codes + (int64_t)t * Format<FMT>::kBytes;
    uint32_t u[Format<FMT>::kBytes / 4];
    if constexpr (FMT == S24_MXFP4) {
        const uint4 w = *reinterpret_cast<const uint4*>(src);
        u[0] = w.x; u[1] = w.y; u[2] = w.z; u[3] = w.w;
    } else {
        load32(src, u);
    }
    uint8_t* dst = out + (int64_t)t * (kBlock * kElem);
    constexpr int kPer = 32 / kElem;   // elements of a 32-byte store
#pragma unroll
    for (int i = 0; i < kElem; ++i) {
        float v[kPer];
#pragma unroll
        for (int j = 0; j < kPer; j += 4) {
            const int e = kPer * i + j;
            if constexpr (FMT == S24_MXFP4) {
                from_e2m1x4((u[e / 8] >> (4 * (e & 7))) & 0xFFFFu, &v[j]);
            } else {
                from_e4m3x2(u[e / 4] & 0xFFFFu, &v[j]);
                from_e4m3x2(u[e / 4] >> 16, &v[j + 2]);
            }
        }
        uint32_t q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (DT == S24_FP32) q[j] = __float_as_uint(v[j] * s);
            else q[j] = mx::pack2<DT>(v[2 * j] * s, v[2 * j + 1] * s);
        }
        store32(dst + 32 * i, q);
    }
}

// One thread per scale of the destination; positions of tensor-core order outside the matrix get 0.  Bound by its byte
// accesses: 28672 x 8192 31 us either way for 2.3 us of bytes.  It runs once per weight, when a checkpoint is loaded; what
// runs in a step writes the order that it needs itself.
template <bool TO_TC>
__global__ void __launch_bounds__(kQuantThreads)
mx_scales_convert_kernel(const uint8_t* __restrict__ src, uint8_t* __restrict__ dst, uint32_t R, uint32_t KB, uint32_t total)
{
    const uint32_t t = blockIdx.x * kQuantThreads + threadIdx.x;
    start_dependents();
    wait_for_predecessors();
    if (t >= total) return;
    const uint32_t chunks = (KB + 3) / 4;
    if constexpr (TO_TC) {
        const uint32_t rec = t >> 9, in = t & 511;
        const uint32_t tile = rec / chunks, chunk = rec - tile * chunks;
        const uint32_t r = tile * 128 + ((in >> 2) & 3) * 32 + (in >> 4), kb = chunk * 4 + (in & 3);
        dst[t] = (r < R && kb < KB) ? src[(int64_t)r * KB + kb] : (uint8_t)0;
    } else {
        const uint32_t r = t / KB;
        dst[t] = src[tc_offset(r, t - r * KB, chunks)];
    }
}

// shape rules shared by the entry points; the index space of blocks has to fit 31 bits
static int check_mx_shape(const char* who, int64_t R, int64_t K)
{
    if (R < 0 || K < 0 || K % kBlock != 0)
        return fail(S24_ERR_SHAPE, "%s: needs R >= 0 and K a multiple of 32 (got R=%lld K=%lld)", who, (long long)R, (long long)K);
    if (R > 0x7FFFFF00ll || K > 0x7FFFFF00ll || (K > 0 && row_tiles(R) * 128 > 0x7FFFFF00ll / (k_chunks(K) * 4)))
        return fail(S24_ERR_SHAPE, "%s: %lld x %lld has too many blocks of 32", who, (long long)R, (long long)K);
    return S24_OK;
}

template <int DT, int FMT>
static int launch_quantize(const void* x, int64_t R, int64_t K, int64_t row_bytes, void* codes, void* scales, void* tc, cudaStream_t st)
{
    const uint32_t KB = (uint32_t)(K / kBlock);
    const uint32_t KB_pad = tc ? (uint32_t)(k_chunks(K) * 4) : KB;
    const uint32_t total = (uint32_t)(tc ? row_tiles(R) * 128 : R) * KB_pad;
    const unsigned grid = (total + kQuantThreads - 1) / kQuantThreads;
    auto* xs = static_cast<const uint8_t*>(x);
    auto* c = static_cast<uint8_t*>(codes);
    auto* s = static_cast<uint8_t*>(scales);
    auto* t = static_cast<uint8_t*>(tc);
    return check_cuda(launch_overlapped(tc ? mx_quantize_kernel<DT, FMT, true> : mx_quantize_kernel<DT, FMT, false>, dim3(grid), kQuantThreads, 0, 1, st,
                                        xs, (uint32_t)R, KB, KB_pad, total, row_bytes, c, s, t),
                      "mx_quantize launch");
}

template <int DT, int FMT>
static int launch_dequantize(const void* codes, const void* scales, int layout, void* out, int64_t R, int64_t K, cudaStream_t st)
{
    const uint32_t KB = (uint32_t)(K / kBlock), total = (uint32_t)R * KB;
    return check_cuda(launch_overlapped(mx_dequantize_kernel<DT, FMT>, dim3((total + kQuantThreads - 1) / kQuantThreads), kQuantThreads, 0, 1, st,
                                        static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), (int)(layout == S24_SCALES_TC), KB, total,
                                        static_cast<uint8_t*>(out)),
                      "mx_dequantize launch");
}

}  // namespace s24

using namespace s24;

extern "C" size_t s24_mx_scales_tc_bytes(int64_t R, int64_t K)
{
    if (R <= 0 || K <= 0) return 0;
    return (size_t)row_tiles(R) * (size_t)k_chunks(K) * kRecordBytes;
}

extern "C" int s24_mx_quantize(const void* x, int64_t R, int64_t K, int64_t ld, int dtype, int fmt, void* codes, void* scales,
                               void* scales_tc, void* stream)
{
    if (dtype != S24_FP16 && dtype != S24_BF16 && dtype != S24_FP32) return fail(S24_ERR_INVALID_ARG, "mx_quantize: bad dtype %d", dtype);
    if (fmt != S24_MXFP4 && fmt != S24_MXFP8) return fail(S24_ERR_INVALID_ARG, "mx_quantize: bad format %d", fmt);
    int rc = check_mx_shape("mx_quantize", R, K);
    if (rc) return rc;
    if (R == 0 || K == 0) return S24_OK;
    if (x == nullptr || codes == nullptr || (scales == nullptr && scales_tc == nullptr))
        return fail(S24_ERR_INVALID_ARG, "mx_quantize: null pointer");
    const int64_t elem = dtype == S24_FP32 ? 4 : 2;
    if (ld < K || ld > (INT64_MAX >> 2) / R || (ld * elem) % 32 != 0)
        return fail(S24_ERR_SHAPE, "mx_quantize: the row stride must be >= K and a multiple of 32 bytes (got %lld elements)", (long long)ld);
    if (!aligned(x, 32) || !aligned(codes, 32) || !aligned(scales_tc, 16))
        return fail(S24_ERR_INVALID_ARG, "mx_quantize: x and codes must be 32-byte aligned, scales_tc 16");
    auto st = static_cast<cudaStream_t>(stream);
    if (fmt == S24_MXFP4) {
        if (dtype == S24_FP16) return launch_quantize<S24_FP16, S24_MXFP4>(x, R, K, ld * elem, codes, scales, scales_tc, st);
        if (dtype == S24_BF16) return launch_quantize<S24_BF16, S24_MXFP4>(x, R, K, ld * elem, codes, scales, scales_tc, st);
        return launch_quantize<S24_FP32, S24_MXFP4>(x, R, K, ld * elem, codes, scales, scales_tc, st);
    }
    if (dtype == S24_FP16) return launch_quantize<S24_FP16, S24_MXFP8>(x, R, K, ld * elem, codes, scales, scales_tc, st);
    if (dtype == S24_BF16) return launch_quantize<S24_BF16, S24_MXFP8>(x, R, K, ld * elem, codes, scales, scales_tc, st);
    return launch_quantize<S24_FP32, S24_MXFP8>(x, R, K, ld * elem, codes, scales, scales_tc, st);
}

extern "C" int s24_mx_dequantize(const void* codes, const void* scales, int layout, void* out, int64_t R, int64_t K, int fmt, int dtype,
                                 void* stream)
{
    if (dtype != S24_FP16 && dtype != S24_BF16 && dtype != S24_FP32) return fail(S24_ERR_INVALID_ARG, "mx_dequantize: bad dtype %d", dtype);
    if (fmt != S24_MXFP4 && fmt != S24_MXFP8) return fail(S24_ERR_INVALID_ARG, "mx_dequantize: bad format %d", fmt);
    if (layout != S24_SCALES_ROWS && layout != S24_SCALES_TC) return fail(S24_ERR_INVALID_ARG, "mx_dequantize: bad layout %d", layout);
    int rc = check_mx_shape("mx_dequantize", R, K);
    if (rc) return rc;
    if (R == 0 || K == 0) return S24_OK;
    if (codes == nullptr || scales == nullptr || out == nullptr) return fail(S24_ERR_INVALID_ARG, "mx_dequantize: null pointer");
    if (!aligned(codes, 32) || !aligned(out, 32)) return fail(S24_ERR_INVALID_ARG, "mx_dequantize: codes and out must be 32-byte aligned");
    auto st = static_cast<cudaStream_t>(stream);
    if (fmt == S24_MXFP4) {
        if (dtype == S24_FP16) return launch_dequantize<S24_FP16, S24_MXFP4>(codes, scales, layout, out, R, K, st);
        if (dtype == S24_BF16) return launch_dequantize<S24_BF16, S24_MXFP4>(codes, scales, layout, out, R, K, st);
        return launch_dequantize<S24_FP32, S24_MXFP4>(codes, scales, layout, out, R, K, st);
    }
    if (dtype == S24_FP16) return launch_dequantize<S24_FP16, S24_MXFP8>(codes, scales, layout, out, R, K, st);
    if (dtype == S24_BF16) return launch_dequantize<S24_BF16, S24_MXFP8>(codes, scales, layout, out, R, K, st);
    return launch_dequantize<S24_FP32, S24_MXFP8>(codes, scales, layout, out, R, K, st);
}

extern "C" int s24_mx_scales_convert(const void* src, int from_layout, void* dst, int to_layout, int64_t R, int64_t K, void* stream)
{
    if ((from_layout != S24_SCALES_ROWS && from_layout != S24_SCALES_TC) || (to_layout != S24_SCALES_ROWS && to_layout != S24_SCALES_TC))
        return fail(S24_ERR_INVALID_ARG, "mx_scales_convert: bad layout %d -> %d", from_layout, to_layout);
    if (from_layout == to_layout) return fail(S24_ERR_UNSUPPORTED, "mx_scales_convert: source and destination layouts are the same");
    int rc = check_mx_shape("mx_scales_convert", R, K);
    if (rc) return rc;
    if (R == 0 || K == 0) return S24_OK;
    if (src == nullptr || dst == nullptr) return fail(S24_ERR_INVALID_ARG, "mx_scales_convert: null pointer");
    auto st = static_cast<cudaStream_t>(stream);
    auto* s = static_cast<const uint8_t*>(src);
    auto* d = static_cast<uint8_t*>(dst);
    const uint32_t KB = (uint32_t)(K / kBlock);
    if (to_layout == S24_SCALES_TC) {
        const uint32_t total = (uint32_t)s24_mx_scales_tc_bytes(R, K);
        return check_cuda(launch_overlapped(mx_scales_convert_kernel<true>, dim3((total + kQuantThreads - 1) / kQuantThreads), kQuantThreads, 0, 1, st, s, d,
                                            (uint32_t)R, KB, total),
                          "mx_scales_convert launch");
    }
    const uint32_t total = (uint32_t)R * KB;
    return check_cuda(launch_overlapped(mx_scales_convert_kernel<false>, dim3((total + kQuantThreads - 1) / kQuantThreads), kQuantThreads, 0, 1, st, s, d,
                                        (uint32_t)R, KB, total),
                      "mx_scales_convert launch");
}
