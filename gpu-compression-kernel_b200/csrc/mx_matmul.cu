// mx_matmul.cu -- product of two matrices in microscaled formats on the block-scaled tcgen05.mma.
//
//   C (M, N) = deq(A) (M, K) . deq(B) (N, K)^T,  both operands K-major, fp32 accumulation in tensor memory.
//
// Both 4-bit: kind::mxf4, 64 elements of K per instruction.  Otherwise kind::mxf8f6f4, 32 per instruction, where a
// 4-bit operand lies in shared memory with every 16 elements in 8 of 16 bytes; the tensor map's 16U4 type spreads
// them that way while they are copied, so memory is read at 4 bits an element.  Either way one k-tile is 128
// bytes of shared memory per row and four instructions.
//
// One CTA, or a CTA pair working as one tile engine, walks the output tiles (persistent grid):
//   * warp 0: TMA producer, one ring of k-tiles (A rows, B rows, and the scale records of both);
//   * warp 1: MMA issuer.  Per k-tile tcgen05.cp brings the scale records into tensor memory (each 512-byte
//     record is 32 lanes x 4 columns, copied to all four lane quadrants), then four MMAs;
//   * warps 2-9: epilogue, two per 32-lane quadrant, each half of the tile's columns.
// In a pair each CTA holds its own 128 rows of A and half of the rows of B, but the scales of all rows of B.
// Every wait is bounded as in the sparse GEMM (s24_device_status).
#include "mx_common.cuh"
#include "sm100_ptx.cuh"
#include "spmm_shared.cuh"

namespace s24 {

using namespace ptx;

constexpr int kMxThreads = 320;

// ---------------------------------------------------------------- the instructions only this file uses

template <int G>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar)
{
    if (G == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                     : "memory");
}

template <int G>
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    if (G == 1) tma_load_2d(dst, map, x, y, bar);
    else tma_load_2d_pair(dst, map, x, y, bar);
}

// one scale record: 32 rows x 16 bytes of shared memory -> 32 lanes x 4 columns, in all four lane quadrants
template <int G>
__device__ __forceinline__ void tc_cp_scales(uint32_t taddr, uint64_t sdesc)
{
    if (G == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

template <int G, bool F4>
__device__ __forceinline__ void tc_mma_scaled(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                              uint32_t accumulate)
{
#define S24_MX_MMA(GROUP, KIND)                                                                                                       \
    asm volatile("{\n\t.reg .pred p;\n\t"                                                                                             \
                 "setp.ne.b32 p, %6, 0;\n\t"                                                                                          \
                 "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d), "l"(adesc), \
                 "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                                                          \
                 : "memory")
    if constexpr (G == 1) {
        if constexpr (F4) S24_MX_MMA("1", "mxf4.block_scale.scale_vec::2X");
        else S24_MX_MMA("1", "mxf8f6f4.block_scale.scale_vec::1X");
    } else {
        if constexpr (F4) S24_MX_MMA("2", "mxf4.block_scale.scale_vec::2X");
        else S24_MX_MMA("2", "mxf8f6f4.block_scale.scale_vec::1X");
    }
#undef S24_MX_MMA
}

// Instruction descriptor of the block-scaled kinds: bits 4-5 / 29-30 which byte of a scale column the B / A scales
// start at (set per instruction), 7-9 A format, 10-12 B format (kind::mxf4: 1 = e2m1; kind::mxf8f6f4: 0 = e4m3,
// 5 = e2m1), 15 / 16 majors (0 = K), 17-22 N >> 3, 23 scale type (1 = power of two), 24-28 M >> 4
__host__ __device__ constexpr uint32_t make_idesc_scaled(uint32_t a_format, uint32_t b_format, int m, int n)
{
    return (a_format << 7) | (b_format << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}

// after a wait that gave up: copies and MMAs still in flight end within this millisecond, before the block's
// shared and tensor memory go to another
__device__ __forceinline__ void settle_after_abort(volatile int* abort_flag)
{
    if (!*abort_flag) return;
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 1000000ull) {}
}

struct MxParams {
    void* C;
    int64_t ldc;
    int M, N, K;
    int out;                 // S24_FP16 / S24_BF16 / S24_FP32
    uint32_t a_format, b_format;
    uint32_t tx_bytes;       // bytes a CTA's copies of one k-tile deliver
    int wide;                // rows of C allow 16-byte stores
    int* status;
    unsigned long long wait_limit_ns;
};

template <int G, int BN, bool F4, int ST>
struct MxCfg {
    static constexpr int kG = G;
    static constexpr int kBN = BN;
    static constexpr bool kF4 = F4;
    static constexpr int kStages = ST;
    static constexpr int kKTile = F4 ? 256 : 128;               // elements of K: 128 bytes of a row
    static constexpr int kChunks = kKTile / 128;                // scale records per 128 rows
    static constexpr int kBNCta = BN / G;
    static constexpr int kTilesB = (BN + 127) / 128;            // record rows of B's scales
    static constexpr int kABytes = 128 * 128;
    static constexpr int kBBytes = kBNCta * 128;
    static constexpr int kSABytes = kChunks * mx::kRecordBytes;
    static constexpr int kSBBytes = kTilesB * kChunks * mx::kRecordBytes;
    static constexpr int kStageBytes = kABytes + kBBytes + kSABytes + kSBBytes;
    static constexpr int kAcc = BN >= 256 ? 1 : 2;
    static constexpr int kScaleCol0 = kAcc * BN;
    static constexpr int kScaleCols = 4 * kChunks * (1 + kTilesB);
    static constexpr int kSmemBytes = ST * kStageBytes + 1024 + 256;
    static_assert(kScaleCol0 + ST * kScaleCols <= (int)kTmemCols, "tensor memory budget");
    static_assert(kSmemBytes <= 232448, "shared memory budget");
    static_assert(8 * (2 * ST + 2 * kAcc) + 16 <= 256, "barrier block");
};

// one row's 32 accumulator columns to memory
__device__ __forceinline__ void mx_store32(const MxParams& p, int row, int col, const uint32_t* r)
{
    if (row >= p.M || col >= p.N) return;
    const int64_t at = (int64_t)row * p.ldc + col;
    const bool whole = p.wide && col + 32 <= p.N;
    if (p.out == S24_FP32) {
        float* c = static_cast<float*>(p.C) + at;
        if (whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<uint4*>(c)[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (col + i < p.N) c[i] = __uint_as_float(r[i]);
        }
        return;
    }
    uint16_t* c = static_cast<uint16_t*>(p.C) + at;
    uint32_t q[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), p.out == S24_BF16);
    if (whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(c)[i] = make_uint4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (col + i < p.N) c[i] = (uint16_t)(q[i >> 1] >> (16 * (i & 1)));
    }
}

template <class Cfg>
__global__ void __launch_bounds__(kMxThreads, 1)
mx_matmul_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                 const __grid_constant__ CUtensorMap tm_sa, const __grid_constant__ CUtensorMap tm_sb, const MxParams p)
{
    constexpr int G = Cfg::kG, BN = Cfg::kBN, ST = Cfg::kStages, ACC = Cfg::kAcc;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t smem_a = smem_base;
    const uint32_t smem_b = smem_a + ST * Cfg::kABytes;
    const uint32_t smem_sa = smem_b + ST * Cfg::kBBytes;
    const uint32_t smem_sb = smem_sa + ST * Cfg::kSABytes;
    const uint32_t bars = smem_sb + ST * Cfg::kSBBytes;
    const uint32_t bar_full = bars;
    const uint32_t bar_empty = bar_full + 8 * ST;
    const uint32_t bar_acc_full = bar_empty + 8 * ST;
    const uint32_t bar_acc_empty = bar_acc_full + 8 * ACC;
    const uint32_t tmem_slot = bar_acc_empty + 8 * ACC;
    const uint32_t abort_addr = tmem_slot + 8;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_gen + (tmem_slot - smem_base));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + (abort_addr - smem_base));

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t cta_rank = (G == 2) ? cluster_ctarank() : 0u;
    const bool leader = cta_rank == 0;

    const int num_m = (p.M + 128 * G - 1) / (128 * G);
    const int num_n = (p.N + BN - 1) / BN;
    const int num_tiles = num_m * num_n;
    const int num_units = (int)gridDim.x / G;
    const int unit = (int)blockIdx.x / G;
    const int ktiles = (p.K + Cfg::kKTile - 1) / Cfg::kKTile;   // elements and scales beyond K read as zeros

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(bar_full + 8 * s, 1);   // one arrive (the leader's producer) + both CTAs' bytes
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < ACC; ++a) {
            mbar_init(bar_acc_full + 8 * a, 1);
            mbar_init(bar_acc_empty + 8 * a, 8 * G);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tensormap(&tm_a);
        prefetch_tensormap(&tm_b);
        prefetch_tensormap(&tm_sa);
        prefetch_tensormap(&tm_sb);
    }
    if (warp == 1) {
        tmem_alloc<G>(tmem_slot, kTmemCols);
        tmem_relinquish<G>();
    }
    tc_fence_before();
    __syncthreads();
    if (G == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot_ptr;

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (elect_one()) {
            int s = 0;
            uint32_t ph = 0;
            bool stopped = false;
            // 4-bit operands of kind::mxf4 are copied as bytes, two elements each; the others by element
            constexpr int kStep = 128;
            for (int t = unit; t < num_tiles && !stopped && !*abort_flag; t += num_units) {
                int tm, tn;
                tile_coords(t, num_m, num_n, tm, tn);
                const int row0 = (tm * G + (int)cta_rank) * 128;
                const int col0 = tn * BN + (int)cta_rank * Cfg::kBNCta;
                for (int kt = 0; kt < ktiles; ++kt) {
                    if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, p.wait_limit_ns)) {
                        report_timeout(p.status, abort_flag, 1);
                        stopped = true;
                        break;
                    }
                    const uint32_t full = (G == 2) ? mapa(bar_full + 8 * s, 0) : (bar_full + 8 * s);
                    if (leader) mbar_arrive_expect_tx(bar_full + 8 * s, G * p.tx_bytes);
                    tma_load_rows<G>(smem_a + s * Cfg::kABytes, &tm_a, kt * kStep, row0, full);
                    tma_load_rows<G>(smem_b + s * Cfg::kBBytes, &tm_b, kt * kStep, col0, full);
                    tma_load_3d<G>(smem_sa + s * Cfg::kSABytes, &tm_sa, 0, kt * Cfg::kChunks, row0 / 128, full);
                    tma_load_3d<G>(smem_sb + s * Cfg::kSBBytes, &tm_sb, 0, kt * Cfg::kChunks, tn * BN / 128, full);
                    if (++s == ST) { s = 0; ph ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (leader CTA only)
        if (leader && elect_one()) {
            const uint32_t idesc = make_idesc_scaled(p.a_format, p.b_format, 128 * G, BN);
            int s = 0, a = 0;
            uint32_t ph = 0, acc_phase = 0;
            bool ok = true;
            for (int t = unit; t < num_tiles && ok && !*abort_flag; t += num_units) {
                if (!mbar_wait(bar_acc_empty + 8 * a, acc_phase ^ 1u, p.wait_limit_ns)) {
                    report_timeout(p.status, abort_flag, 3);
                    break;
                }
                tc_fence_after();
                const uint32_t tmem_d = tmem_base + (uint32_t)(a * BN);
                for (int kt = 0; kt < ktiles; ++kt) {
                    if (!mbar_wait(bar_full + 8 * s, ph, p.wait_limit_ns)) {
                        report_timeout(p.status, abort_flag, 2);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sfa = tmem_base + (uint32_t)(Cfg::kScaleCol0 + s * Cfg::kScaleCols);
                    const uint32_t sfb = sfa + 4 * Cfg::kChunks;
#pragma unroll
                    for (int c = 0; c < Cfg::kChunks; ++c) {
                        tc_cp_scales<G>(sfa + 4 * c, make_smem_desc(smem_sa + s * Cfg::kSABytes + c * mx::kRecordBytes, 128, 128, kSwizzleNone));
#pragma unroll
                        for (int b = 0; b < Cfg::kTilesB; ++b)
                            tc_cp_scales<G>(sfb + 4 * (c * Cfg::kTilesB + b),
                                            make_smem_desc(smem_sb + s * Cfg::kSBBytes + (b * Cfg::kChunks + c) * mx::kRecordBytes, 128, 128, kSwizzleNone));
                    }
                    const uint64_t adesc = make_smem_desc(smem_a + s * Cfg::kABytes, 16, 1024, kSwizzle128B);
                    const uint64_t bdesc = make_smem_desc(smem_b + s * Cfg::kBBytes, 16, 1024, kSwizzle128B);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        // 32 bytes of a row per instruction; its scales: two bytes of a record's word, or one
                        const uint32_t c = Cfg::kF4 ? j >> 1 : 0, id = Cfg::kF4 ? (j & 1) * 2 : j;
                        tc_mma_scaled<G, Cfg::kF4>(tmem_d, adesc + (uint64_t)(j * 2), bdesc + (uint64_t)(j * 2), idesc | (id << 4) | (id << 29),
                                                   sfa + 4 * c, sfb + 4 * Cfg::kTilesB * c, (kt | j) != 0 ? 1u : 0u);
                    }
                    if (G == 2) tc_commit_pair(bar_empty + 8 * s, 3);
                    else tc_commit<1>(bar_empty + 8 * s);
                    if (++s == ST) { s = 0; ph ^= 1u; }
                }
                if (!ok) break;
                if (G == 2) tc_commit_pair(bar_acc_full + 8 * a, 3);
                else tc_commit<1>(bar_acc_full + 8 * a);
                if (++a == ACC) { a = 0; acc_phase ^= 1u; }
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue warps
        const int quad = warp & 3;
        const int half = (warp - 2) >> 2;
        constexpr int CW = BN / 2;
        int a = 0;
        uint32_t acc_phase = 0;
        const uint32_t acc_empty = (G == 2) ? mapa(bar_acc_empty, 0) : bar_acc_empty;
        for (int t = unit; t < num_tiles && !*abort_flag; t += num_units) {
            int tm, tn;
            tile_coords(t, num_m, num_n, tm, tn);
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(bar_acc_full + 8 * a, acc_phase, p.wait_limit_ns))) {
                if (lane == 0) report_timeout(p.status, abort_flag, 4);
                break;
            }
            tc_fence_after();
            const uint32_t tacc = tmem_base + (uint32_t)(a * BN + half * CW) + ((uint32_t)(32 * quad) << 16);
            const int row = (tm * G + (int)cta_rank) * 128 + 32 * quad + lane;
            const int col = tn * BN + half * CW;
#pragma unroll 1
            for (int c = 0; c < CW; c += 32) {
                uint32_t r[32];
                tc_ld_32x32b_x32(tacc + (uint32_t)c, r);
                tc_wait_ld();
                if (c + 32 == CW) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(acc_empty + 8 * a);
                }
                mx_store32(p, row, col + c, r);
                __syncwarp();
            }
            if (++a == ACC) { a = 0; acc_phase ^= 1u; }
        }
    }

    // ------------------------------------------------------------ teardown
    settle_after_abort(abort_flag);
    tc_fence_before();
    __syncthreads();
    if (G == 2) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<G>(tmem_base, kTmemCols);
    }
}

// ---------------------------------------------------------------- host side

struct MxOperand {
    const void* codes;
    const void* scales;   // tensor-core order
    int64_t rows, ld;     // row stride in bytes
    int fmt;
};

// codes of an operand: boxes of 128 bytes of shared memory per row
static int make_code_map(CUtensorMap* map, const MxOperand& o, int64_t K, bool both4, int box_rows, const char* what)
{
    if (both4 || o.fmt == S24_MXFP8)
        return make_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, o.codes, (uint64_t)(both4 ? K / 2 : K), (uint64_t)o.rows, (uint64_t)o.ld, 128,
                           (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B, what);
    return make_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 1, o.codes, (uint64_t)K, (uint64_t)o.rows, (uint64_t)o.ld, 128,
                       (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B, what);
}

static int make_scale_map(CUtensorMap* map, const MxOperand& o, int64_t K, int chunks, int tiles, const char* what)
{
    const uint64_t nk = (uint64_t)mx::k_chunks(K);
    const uint64_t dims[3] = {mx::kRecordBytes / 4, nk, (uint64_t)mx::row_tiles(o.rows)};
    const uint64_t strides[2] = {mx::kRecordBytes, nk * mx::kRecordBytes};
    const uint32_t box[3] = {mx::kRecordBytes / 4, (uint32_t)chunks, (uint32_t)tiles};
    return make_map_3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, o.scales, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE, what);
}

// bytes a copy of `rows` rows of one k-tile signals on its barrier: what was read, so a spread 4-bit row counts
// 64 of the 128 bytes it covers (measured; the padding is not written either)
static uint32_t code_tx(const MxOperand& o, bool both4, int rows) { return (uint32_t)rows * ((both4 || o.fmt == S24_MXFP8) ? 128u : 64u); }

template <class Cfg>
static int launch_mx(const MxOperand& a, const MxOperand& b, MxParams p, cudaStream_t stream)
{
    CUtensorMap tm_a, tm_b, tm_sa, tm_sb;
    int rc = make_code_map(&tm_a, a, p.K, Cfg::kF4, 128, "A codes");
    if (!rc) rc = make_code_map(&tm_b, b, p.K, Cfg::kF4, Cfg::kBNCta, "B codes");
    if (!rc) rc = make_scale_map(&tm_sa, a, p.K, Cfg::kChunks, 1, "A scales");
    if (!rc) rc = make_scale_map(&tm_sb, b, p.K, Cfg::kChunks, Cfg::kTilesB, "B scales");
    if (rc) return rc;
    p.tx_bytes = code_tx(a, Cfg::kF4, 128) + code_tx(b, Cfg::kF4, Cfg::kBNCta) + Cfg::kSABytes + Cfg::kSBBytes;
    {
        static bool opted_in[64] = {false};
        int dev = 0;
        rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
        if (rc) return rc;
        if (dev < 0 || dev >= 64 || !opted_in[dev]) {
            rc = check_cuda(cudaFuncSetAttribute(mx_matmul_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes),
                            "cudaFuncSetAttribute(max dynamic shared memory)");
            if (rc) return rc;
            if (dev >= 0 && dev < 64) opted_in[dev] = true;
        }
    }
    const int64_t tiles = (int64_t)((p.M + 128 * Cfg::kG - 1) / (128 * Cfg::kG)) * ((p.N + Cfg::kBN - 1) / Cfg::kBN);
    if (tiles > 0x7FFFFFFFll / kGroupM) return fail(S24_ERR_SHAPE, "mx_matmul: too many output tiles");
    int units = sm_count() / Cfg::kG;
    if (units > tiles) units = (int)tiles;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(units * Cfg::kG));
    lc.blockDim = dim3(kMxThreads);
    lc.dynamicSmemBytes = Cfg::kSmemBytes;
    lc.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = Cfg::kG;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&lc, mx_matmul_kernel<Cfg>, tm_a, tm_b, tm_sa, tm_sb, p), "mx_matmul launch");
}

template <bool F4>
static int pick_mx(const MxOperand& a, const MxOperand& b, const MxParams& p, const s24_tile_cfg* cfg, cudaStream_t stream)
{
    int bm = cfg ? cfg->bm : 0, bn = cfg ? cfg->bn : 0;
    if (bm == 0) bm = p.M > 128 ? 256 : 128;
    if (bn == 0) bn = bm == 256 && p.N > 128 ? 256 : 128;
    if (bm == 256 && bn == 256) return launch_mx<MxCfg<2, 256, F4, 6>>(a, b, p, stream);
    if (bm == 256 && bn == 128) return launch_mx<MxCfg<2, 128, F4, 8>>(a, b, p, stream);
    if (bm == 128 && bn == 128) return launch_mx<MxCfg<1, 128, F4, 6>>(a, b, p, stream);
    return fail(S24_ERR_UNSUPPORTED, "mx_matmul: no kernel for tile %d x %d (have 256x256, 256x128, 128x128)", bm, bn);
}

}  // namespace s24

using namespace s24;

extern "C" int s24_mx_matmul(const void* a, const void* a_scales, const void* b, const void* b_scales, void* C, int64_t M, int64_t N, int64_t K,
                             int64_t lda, int64_t ldb, int64_t ldc, int fmt_a, int fmt_b, int out_dtype, const s24_tile_cfg* cfg, void* stream)
{
    if ((fmt_a != S24_MXFP4 && fmt_a != S24_MXFP8) || (fmt_b != S24_MXFP4 && fmt_b != S24_MXFP8))
        return fail(S24_ERR_INVALID_ARG, "mx_matmul: bad format %d, %d", fmt_a, fmt_b);
    if (out_dtype != S24_FP16 && out_dtype != S24_BF16 && out_dtype != S24_FP32) return fail(S24_ERR_INVALID_ARG, "mx_matmul: bad dtype %d", out_dtype);
    if (M < 0 || N < 0 || K <= 0 || K % 32 != 0)
        return fail(S24_ERR_SHAPE, "mx_matmul: needs M, N >= 0 and K a positive multiple of 32 (got M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
    if (fmt_a != fmt_b && K % 128 != 0)
        return fail(S24_ERR_SHAPE, "mx_matmul: operands of different formats need K %% 128 == 0 (got %lld)", (long long)K);
    if (M > 0x7FFFFF00ll || N > 0x7FFFFF00ll || K > 0x7FFFFF00ll) return fail(S24_ERR_SHAPE, "mx_matmul: dimension too large");
    if (M == 0 || N == 0) return S24_OK;
    if (a == nullptr || a_scales == nullptr || b == nullptr || b_scales == nullptr || C == nullptr) return fail(S24_ERR_INVALID_ARG, "mx_matmul: null pointer");
    // bytes of a row; the copies want strides of 16 bytes, of 32 where 4-bit codes are spread on the way
    const int64_t wa = fmt_a == S24_MXFP4 ? K / 2 : K, wb = fmt_b == S24_MXFP4 ? K / 2 : K;
    const int64_t step_a = (fmt_a == S24_MXFP4 && fmt_b == S24_MXFP8) ? 32 : 16, step_b = (fmt_b == S24_MXFP4 && fmt_a == S24_MXFP8) ? 32 : 16;
    if (lda < wa || lda % step_a != 0 || ldb < wb || ldb % step_b != 0 || lda >= (1ll << 40) || ldb >= (1ll << 40))
        return fail(S24_ERR_SHAPE, "mx_matmul: row strides of the codes must cover K and be multiples of %lld / %lld bytes (got %lld, %lld)",
                    (long long)step_a, (long long)step_b, (long long)lda, (long long)ldb);
    if (ldc < N || ldc >= (1ll << 40)) return fail(S24_ERR_SHAPE, "mx_matmul: ldc must be >= N (got %lld)", (long long)ldc);
    const int64_t esz = out_dtype == S24_FP32 ? 4 : 2;
    if (!aligned(a, step_a) || !aligned(b, step_b) || !aligned(a_scales, 16) || !aligned(b_scales, 16) || !aligned(C, esz))
        return fail(S24_ERR_INVALID_ARG, "mx_matmul: codes must be %lld / %lld-byte aligned, scales 16-byte and C by its element", (long long)step_a,
                    (long long)step_b);
    int* status = status_word_address();
    if (status == nullptr) return fail(S24_ERR_CUDA, "mx_matmul: cannot resolve the device status word");

    const bool both4 = fmt_a == S24_MXFP4 && fmt_b == S24_MXFP4;
    MxParams p;
    p.C = C;
    p.ldc = ldc;
    p.M = (int)M;
    p.N = (int)N;
    p.K = (int)K;
    p.out = out_dtype;
    p.a_format = both4 ? 1u : fmt_a == S24_MXFP4 ? 5u : 0u;
    p.b_format = both4 ? 1u : fmt_b == S24_MXFP4 ? 5u : 0u;
    p.tx_bytes = 0;
    p.wide = aligned(C, 16) && (ldc * esz) % 16 == 0;
    p.status = status;
    p.wait_limit_ns = kWaitTimeoutNs;
    const MxOperand oa = {a, a_scales, M, lda, fmt_a}, ob = {b, b_scales, N, ldb, fmt_b};
    auto st = static_cast<cudaStream_t>(stream);
    return both4 ? pick_mx<true>(oa, ob, p, cfg, st) : pick_mx<false>(oa, ob, p, cfg, st);
}
