// mx_common.cuh -- the microscaled number formats: what a block of 32 elements and its scale are,
// and the conversions every kernel of them uses.
//
// A block is 32 consecutive elements of a row.  With a = max |v_i| and emax the exponent of the
// element type's largest power of two (e2m1: 2, e4m3: 8),
//   scale code s = clamp(floor(log2 a) - emax + 127, 0, 254)   (s = 0 for a = 0),
//   element    q = round(v * 2^(127 - s)) to the element type, half to even, saturating,
// and the block reads back as q * 2^(s - 127).  A block that holds a NaN or an infinity has s = 255
// and codes 0 and reads back as NaN throughout.  v * 2^(127 - s) is exact in fp32, so the only
// rounding is the one to the element type.
#pragma once

#include "s24_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace s24 {
namespace mx {

constexpr int kBlock = 32;          // elements that share a scale
constexpr int kRecordBytes = 512;   // scales of 128 rows x 128 columns in tensor-core order

template <int FMT>
struct Format {
    static constexpr int kEmax = (FMT == S24_MXFP4) ? 2 : 8;
    static constexpr int kBytes = (FMT == S24_MXFP4) ? 16 : 32;   // codes of one block
};

__host__ __device__ inline int64_t row_tiles(int64_t R) { return (R + 127) / 128; }
__host__ __device__ inline int64_t k_chunks(int64_t K) { return (K + 127) / 128; }

// byte offset in tensor-core order of the scale of row r, block kb
__host__ __device__ inline int64_t tc_offset(int64_t r, int64_t kb, int64_t chunks)
{
    return ((r >> 7) * chunks + (kb >> 2)) * kRecordBytes + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (kb & 3);
}

// the scale code of a block from the largest magnitude's fp32 bits
template <int FMT>
__device__ __forceinline__ uint32_t scale_code(uint32_t amax_bits)
{
    const int e = (int)(amax_bits >> 23);   // floor(log2 a) + 127 for normal numbers; smaller ones give s = 0 anyway
    return e == 255 ? 255u : (uint32_t)max(e - Format<FMT>::kEmax, 0);
}

// 2^(127 - s); s is at most 252, so this is a normal number
__device__ __forceinline__ float scale_up(uint32_t code) { return __uint_as_float((254u - code) << 23); }

// 2^(s - 127), NaN for 255
__device__ __forceinline__ float scale_value(uint32_t code)
{
    return __uint_as_float(code == 255u ? 0x7FFFFFFFu : code == 0u ? 0x00400000u : code << 23);
}

// eight fp32 values to e2m1, element 0 in the lowest four bits
__device__ __forceinline__ uint32_t to_e2m1x8(const float* v)
{
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// four fp32 values to e4m3, element 0 in the lowest byte
__device__ __forceinline__ uint32_t to_e4m3x4(const float* v)
{
    uint32_t r;
    asm("{\n\t.reg .b16 h0, h1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h0, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h1, %4, %3;\n\t"
        "mov.b32 %0, {h0, h1};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
    return r;
}

// the codes of a block whose elements are already multiplied by 2^(127 - s); zeros if !finite
template <int FMT>
__device__ __forceinline__ void encode_block(const float (&v)[kBlock], bool finite, uint32_t (&codes)[Format<FMT>::kBytes / 4])
{
    if constexpr (FMT == S24_MXFP4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) codes[i] = finite ? to_e2m1x8(&v[8 * i]) : 0u;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) codes[i] = finite ? to_e4m3x4(&v[4 * i]) : 0u;
    }
}

// four e2m1 codes (16 bits) or two e4m3 codes (16 bits) to fp32, exact
__device__ __forceinline__ void from_e2m1x4(uint32_t bits16, float* v)
{
    uint32_t lo, hi;
    asm("{\n\t.reg .b8 b0, b1;\n\t.reg .b16 h;\n\t"
        "cvt.u16.u32 h, %2;\n\t"
        "mov.b16 {b0, b1}, h;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(bits16));
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}

__device__ __forceinline__ void from_e4m3x2(uint32_t bits16, float* v)
{
    uint32_t h;
    asm("{\n\t.reg .b16 t;\n\t"
        "cvt.u16.u32 t, %1;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, t;\n\t}"
        : "=r"(h)
        : "r"(bits16));
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&h));
    v[0] = a.x; v[1] = a.y;
}

// two 16-bit values of a register to fp32
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t w)
{
    if constexpr (DT == S24_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    if constexpr (DT == S24_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Launches that follow one another overlap: a kernel lets the next one of its stream start as soon as all its own CTAs have
// (start_dependents), and touches global memory only when the kernels before it have completed and their writes are visible
// (wait_for_predecessors).  What it does before that, setting up barriers, tensor memory and descriptors, costs nothing then.
// A kernel of another library neither starts early nor is overtaken.
__device__ __forceinline__ void start_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_predecessors() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... Params, class... Args>
inline cudaError_t launch_overlapped(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t stream, Args... args)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim = grid;
    lc.blockDim = dim3(threads);
    lc.dynamicSmemBytes = smem;
    lc.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&lc, kernel, args...);
}

// two fp32 numbers in one 64-bit register pair, and operations on both at once
struct Pair {
    uint64_t v;
};
__device__ __forceinline__ Pair make_pair(float a, float b)
{
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ float2 split(Pair p)
{
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
    return f;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b)
{
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b)
{
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

// largest magnitude of three, NaN if one is
__device__ __forceinline__ float max_magnitude(float a, float b, float c)
{
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 32-byte accesses
__device__ __forceinline__ void load32(const void* p, uint32_t (&r)[8])
{
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void store32(void* p, const uint32_t* r)
{
    asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

}  // namespace mx
}  // namespace s24
