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
//   * warps 2-9: epilogue, two per 32-lane quadrant, 64 of the tile's columns each in turn (with a half of the tile for
//     each the sectors that unaligned rows share were written further apart: 4078 x 13733 x 384 55 us, so 50).
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
    uint32_t tx_bytes;       // bytes a CTA's copies of one k-tile deliver, B's codes aside
    uint32_t tx_box;         // and each box of B's codes
    int wide;                // rows of C allow 32-byte stores
    int whole, steps;        // mx_tile
    int* status;
    unsigned long long wait_limit_ns;
};

constexpr int kStorePitch = 33;                              // words: 32 of a row and one against bank conflicts
constexpr int kStoreWarpBytes = 32 * kStorePitch * 4;

// Output tiles in groups of 16 row tiles swept along N.  Of groups of 4 / 8 / 16 / 32, seconds under load:
// 8192^3 4-bit 210 / 210 / 208 / 207 us, 8-bit 438 / 428 / 421 / 468, 4001 x 28672 x 8192 700 / 689 / 682 / 682,
// 16384^3 4-bit 1639 / 1577 / 1550 / 1746 (with 16 now 200, 409, 674 and 1518).
constexpr int kMxGroupM = 16;
// Parts of a tile start on whole records of B's scales; from a record's middle they would be read two tensor-memory columns
// further on, which is not built.
constexpr int kMxPart = 128;

struct MxTile {
    int m, col, width;   // row tile, first column, columns the MMA makes: a multiple of 64; none: nothing left to do
};

// Step t of the persistent walk.  The tiles of a last pass that leaves half of the units idle, those from p.whole on, are
// two steps of 128 columns each, and a tile that N ends in is as narrow as it can be (1537 x 6150 x 4128 8-bit 41.2 -> 38.4
// us, 2000 x 10000 x 4096 8-by-4-bit 60.1 -> 57.6, 2560 x 2048 x 4096 4-bit 15.1 -> 13.2).
template <int BN>
__device__ __forceinline__ MxTile mx_tile(const MxParams& p, int t, int num_m, int num_n)
{
    int part = 0, columns = BN;
    if (BN > kMxPart && t >= p.whole) {
        part = (t - p.whole) & 1;
        t = p.whole + ((t - p.whole) >> 1);
        columns = kMxPart;
    }
    const int group_size = kMxGroupM * num_n;
    const int group = t / group_size;
    const int first_m = group * kMxGroupM;
    const int gm = min(num_m - first_m, kMxGroupM);
    const int in_group = t - group * group_size;
    MxTile tile;
    tile.m = first_m + in_group % gm;
    tile.col = in_group / gm * BN + part * kMxPart;
    tile.width = min(columns, (p.N - tile.col + 63) / 64 * 64);
    return tile;
}

// ALIGNED: rows of C start on 32 bytes; otherwise a stage of the ring makes room for the stores' staging
template <int G, int BN, bool F4, int ST, bool ALIGNED>
struct MxCfg {
    static constexpr bool kAligned = ALIGNED;
    static constexpr int kG = G;
    static constexpr int kBN = BN;
    static constexpr bool kF4 = F4;
    static constexpr int kStages = ST;
    static constexpr int kKTile = F4 ? 256 : 128;               // elements of K: 128 bytes of a row
    static constexpr int kChunks = kKTile / 128;                // scale records per 128 rows
    static constexpr int kBNCta = BN / G;
    // rows of B in one copy: a tile's half is copied alone (an SM takes in 64 bytes a cycle, so an MMA half as wide is no
    // faster where the rows of a whole one come with it), and whole tiles run 2 to 3 % faster with two copies as well
    static constexpr int kBox = kBNCta < kMxPart / G ? kBNCta : kMxPart / G;
    static constexpr int kTilesB = (BN + 127) / 128;            // record rows of B's scales
    static constexpr int kABytes = 128 * 128;
    static constexpr int kBBytes = kBNCta * 128;
    static constexpr int kSABytes = kChunks * mx::kRecordBytes;
    static constexpr int kSBBytes = kTilesB * kChunks * mx::kRecordBytes;
    static constexpr int kStageBytes = kABytes + kBBytes + kSABytes + kSBBytes;
    static constexpr int kAccStep = BN >= 256 ? 224 : BN;       // first column of the second accumulator
    static constexpr int kScaleCol0 = kAccStep + BN;
    static constexpr int kScaleCols = 4 * kChunks * (1 + kTilesB);
    static constexpr int kStoreBytes = ALIGNED ? 0 : 8 * kStoreWarpBytes;
    static constexpr int kSmemBytes = ST * kStageBytes + kStoreBytes + 1024 + 256;
    static_assert(kScaleCol0 + kScaleCols <= (int)kTmemCols, "tensor memory budget");
    static_assert(kSmemBytes <= 232448, "shared memory budget");
    static_assert(8 * (2 * ST + 2) + 16 <= 256, "barrier block");
};

__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr)
{
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// 32 rows (one per lane) x 64 accumulator columns to C, whose rows start on 32 bytes: whole sectors straight from the
// registers, and single elements where N ends inside one.
__device__ __forceinline__ void mx_store_aligned(const MxParams& p, int row0, int col, const uint32_t (&r)[64], int lane)
{
    const int row = row0 + lane;
    if (row >= p.M) return;
    if (p.out == S24_FP32) {
        float* c = static_cast<float*>(p.C) + (int64_t)row * p.ldc + col;
#pragma unroll
        for (int i = 0; i < 64; i += 8) {
            if (col + i + 8 <= p.N) {
                mx::store32(c + i, &r[i]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (col + i + k < p.N) c[i + k] = __uint_as_float(r[i + k]);
            }
        }
        return;
    }
    uint16_t* c = static_cast<uint16_t*>(p.C) + (int64_t)row * p.ldc + col;
#pragma unroll
    for (int i = 0; i < 64; i += 16) {
        uint32_t q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = pack2(__uint_as_float(r[i + 2 * k]), __uint_as_float(r[i + 2 * k + 1]), p.out == S24_BF16);
        if (col + i + 16 <= p.N) {
            mx::store32(c + i, q);
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (col + i + k < p.N) c[i + k] = (uint16_t)(q[k >> 1] >> (16 * (k & 1)));
        }
    }
}

// The same for rows that start anywhere: through shared memory, so that 32 lanes write 128 bytes of one row.  Of 16-bit
// rows every second starts on the same half of a word: rows that start on a whole word are written as words, the others
// as words from their second element on, with their first and last elements by themselves.
__device__ __forceinline__ void mx_store_any(const MxParams& p, int row0, int col, const uint32_t (&r)[64], uint32_t staging, int lane)
{
    const bool f32 = p.out == S24_FP32;
    const int rows = min(32, p.M - row0);   // the same for the whole warp
    const uint32_t own = staging + (uint32_t)lane * 4;
    constexpr uint32_t kRow = kStorePitch * 4;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        if (part == 1 && !f32) break;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint32_t w = f32 ? r[32 * part + i] : pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), p.out == S24_BF16);
            st_shared_u32(staging + (uint32_t)lane * kRow + 4 * i, w);
        }
        __syncwarp();
        if (f32) {
            const int c = col + 32 * part + lane;
            float* dst = static_cast<float*>(p.C) + (int64_t)row0 * p.ldc + c;
            if (rows == 32 && col + 32 * part + 32 <= p.N) {
#pragma unroll
                for (int rr = 0; rr < 32; ++rr) dst[rr * p.ldc] = __uint_as_float(ld_shared_u32(own + rr * kRow));
            } else if (c < p.N) {
                for (int rr = 0; rr < rows; ++rr) dst[rr * p.ldc] = __uint_as_float(ld_shared_u32(own + rr * kRow));
            }
        } else if (rows == 32 && col + 64 <= p.N) {
            uint16_t* first = static_cast<uint16_t*>(p.C) + (int64_t)row0 * p.ldc + col;
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                uint16_t* start = first + odd * p.ldc;
                const uint32_t from = own + odd * kRow;
                if ((reinterpret_cast<uintptr_t>(start) & 3u) == 0) {   // the same for the whole warp
                    uint32_t* dst = reinterpret_cast<uint32_t*>(start) + lane;
#pragma unroll
                    for (int i = 0; i < 16; ++i) dst[i * p.ldc] = ld_shared_u32(from + 2 * i * kRow);
                } else {
                    uint32_t* dst = reinterpret_cast<uint32_t*>(start + 1) + lane;
                    if (lane < 31) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            dst[i * p.ldc] = __byte_perm(ld_shared_u32(from + 2 * i * kRow), ld_shared_u32(from + 2 * i * kRow + 4), 0x5432);
                    }
                    // lanes 0-15: the first elements of the 16 rows, 16-31: their last
                    const int i = lane & 15, last = lane >> 4;
                    const uint32_t w = ld_shared_u32(staging + (uint32_t)(odd + 2 * i) * kRow + (last ? 124u : 0u));
                    start[(int64_t)(2 * i) * p.ldc + (last ? 63 : 0)] = (uint16_t)(last ? w >> 16 : w);
                }
            }
        } else {
            const int c = col + 2 * lane;
            uint16_t* dst = static_cast<uint16_t*>(p.C) + (int64_t)row0 * p.ldc + c;
            for (int rr = 0; rr < rows; ++rr, dst += p.ldc) {
                const uint32_t v = ld_shared_u32(own + rr * kRow);
                if (c < p.N) dst[0] = (uint16_t)v;
                if (c + 1 < p.N) dst[1] = (uint16_t)(v >> 16);
            }
        }
    }
}

template <class Cfg>
__global__ void __launch_bounds__(kMxThreads, 1)
mx_matmul_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                 const __grid_constant__ CUtensorMap tm_sa, const __grid_constant__ CUtensorMap tm_sb, const MxParams p)
{
    constexpr int G = Cfg::kG, BN = Cfg::kBN, ST = Cfg::kStages;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t smem_a = smem_base;
    const uint32_t smem_b = smem_a + ST * Cfg::kABytes;
    const uint32_t smem_sa = smem_b + ST * Cfg::kBBytes;
    const uint32_t smem_sb = smem_sa + ST * Cfg::kSABytes;
    const uint32_t smem_store = smem_sb + ST * Cfg::kSBBytes;
    const uint32_t bar_full = smem_store + Cfg::kStoreBytes;
    const uint32_t bar_empty = bar_full + 8 * ST;
    const uint32_t bar_acc_full = bar_empty + 8 * ST;
    const uint32_t bar_acc_empty = bar_acc_full + 8;
    const uint32_t tmem_slot = bar_acc_empty + 8;
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
    const int num_units = (int)gridDim.x / G;
    const int unit = (int)blockIdx.x / G;
    const int ktiles = (p.K + Cfg::kKTile - 1) / Cfg::kKTile;   // elements and scales beyond K read as zeros

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(bar_full + 8 * s, 1);   // one arrive (the leader's producer) + both CTAs' bytes
            mbar_init(bar_empty + 8 * s, 1);
        }
        mbar_init(bar_acc_full, 1);
        mbar_init(bar_acc_empty, 8 * G);   // the epilogue warps of every CTA
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
    mx::start_dependents();
    mx::wait_for_predecessors();

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (elect_one()) {
            int s = 0;
            uint32_t ph = 0;
            bool stopped = false;
            // 4-bit operands of kind::mxf4 are copied as bytes, two elements each; the others by element
            constexpr int kStep = 128;
            for (int t = unit; t < p.steps && !stopped && !*abort_flag; t += num_units) {
                const MxTile tile = mx_tile<BN>(p, t, num_m, num_n);
                if (tile.width <= 0) break;   // the second half of a narrow tile: a unit's last step
                const int row0 = (tile.m * G + (int)cta_rank) * 128;
                const int col0 = tile.col + (int)cta_rank * (tile.width / G);
                const int boxes = Cfg::kBNCta > Cfg::kBox && tile.width > kMxPart ? 2 : 1;
                const uint32_t tx_bytes = G * (p.tx_bytes + (uint32_t)boxes * p.tx_box);
                for (int kt = 0; kt < ktiles; ++kt) {
                    if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, p.wait_limit_ns)) {
                        report_timeout(p.status, abort_flag, 1);
                        stopped = true;
                        break;
                    }
                    const uint32_t full = (G == 2) ? mapa(bar_full + 8 * s, 0) : (bar_full + 8 * s);
                    if (leader) mbar_arrive_expect_tx(bar_full + 8 * s, tx_bytes);
                    tma_load_rows<G>(smem_a + s * Cfg::kABytes, &tm_a, kt * kStep, row0, full);
                    tma_load_rows<G>(smem_b + s * Cfg::kBBytes, &tm_b, kt * kStep, col0, full);
                    if (boxes > 1) tma_load_rows<G>(smem_b + s * Cfg::kBBytes + Cfg::kBox * 128, &tm_b, kt * kStep, col0 + Cfg::kBox, full);
                    tma_load_3d<G>(smem_sa + s * Cfg::kSABytes, &tm_sa, 0, kt * Cfg::kChunks, row0 / 128, full);
                    tma_load_3d<G>(smem_sb + s * Cfg::kSBBytes, &tm_sb, 0, kt * Cfg::kChunks, tile.col / 128, full);
                    if (++s == ST) { s = 0; ph ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (leader CTA only)
        if (leader && elect_one()) {
            const uint32_t sfa = tmem_base + (uint32_t)Cfg::kScaleCol0;
            const uint32_t sfb = sfa + 4 * Cfg::kChunks;
            int s = 0, n = 0;   // n: tiles done
            uint32_t ph = 0;
            bool ok = true;
            for (int t = unit; t < p.steps && ok && !*abort_flag; t += num_units, ++n) {
                const int width = mx_tile<BN>(p, t, num_m, num_n).width;
                if (width <= 0) break;
                const uint32_t idesc = make_idesc_scaled(p.a_format, p.b_format, 128 * G, width);
                const uint32_t tmem_d = tmem_base + (uint32_t)((n & 1) * Cfg::kAccStep);
                for (int kt = 0; kt < ktiles; ++kt) {
                    if (!mbar_wait(bar_full + 8 * s, ph, p.wait_limit_ns)) {
                        report_timeout(p.status, abort_flag, 2);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    // tcgen05.cp and tcgen05.mma run in the order of issue, so one set of scale columns does
#pragma unroll
                    for (int c = 0; c < Cfg::kChunks; ++c) {
                        tc_cp_scales<G>(sfa + 4 * c, make_smem_desc(smem_sa + s * Cfg::kSABytes + c * mx::kRecordBytes, 128, 128, kSwizzleNone));
#pragma unroll
                        for (int b = 0; b < Cfg::kTilesB; ++b)
                            tc_cp_scales<G>(sfb + 4 * (c * Cfg::kTilesB + b),
                                            make_smem_desc(smem_sb + s * Cfg::kSBBytes + (b * Cfg::kChunks + c) * mx::kRecordBytes, 128, 128, kSwizzleNone));
                    }
                    // the epilogue has read what the previous tile's accumulator shares with this one's (and, before it, all
                    // of the tile before that, which had this accumulator)
                    if (kt == 0 && n > 0) {
                        if (!mbar_wait(bar_acc_empty, (uint32_t)(n - 1) & 1u, p.wait_limit_ns)) {
                            report_timeout(p.status, abort_flag, 3);
                            ok = false;
                            break;
                        }
                        tc_fence_after();
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
                if (G == 2) tc_commit_pair(bar_acc_full, 3);
                else tc_commit<1>(bar_acc_full);
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue warps
        const int quad = warp & 3;
        const int half = (warp - 2) >> 2;
        const uint32_t staging = Cfg::kAligned ? 0u : smem_store + (uint32_t)(warp - 2) * kStoreWarpBytes;
        const uint32_t acc_empty = (G == 2) ? mapa(bar_acc_empty, 0) : bar_acc_empty;
        int n = 0;
        for (int t = unit; t < p.steps && !*abort_flag; t += num_units, ++n) {
            const MxTile tile = mx_tile<BN>(p, t, num_m, num_n);
            if (tile.width <= 0) break;
            const int turns = BN > 128 && tile.width > 128 ? 2 : 1;
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(bar_acc_full, (uint32_t)n & 1u, p.wait_limit_ns))) {
                if (lane == 0) report_timeout(p.status, abort_flag, 4);
                break;
            }
            tc_fence_after();
            const uint32_t tacc = tmem_base + (uint32_t)((n & 1) * Cfg::kAccStep) + ((uint32_t)(32 * quad) << 16);
            const int row0 = (tile.m * G + (int)cta_rank) * 128 + 32 * quad;
            // The 32 columns that both accumulators cover are the first's last ones and the second's first ones: the warp
            // that owns them reads its 64 columns with them first and hands them back; every warp arrives, whether it has a
            // share or not.
            const bool shares = half == ((n & 1) ? 0 : 1);
            if (!shares) {
                tc_fence_before();   // its reads of the tile before
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(acc_empty);
            }
#pragma unroll 1
            for (int i = 0; i < turns; ++i) {
                const int c = 128 * ((n & 1) ? i : turns - 1 - i) + 64 * half;
                uint32_t r[64];
                tc_ld_32x32b_x64(tacc + (uint32_t)c, r);
                tc_wait_ld();
                if (shares && i == 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_remote(acc_empty);
                }
                if (row0 < p.M && c < tile.width) {   // the same for the whole warp
                    if constexpr (Cfg::kAligned) mx_store_aligned(p, row0, tile.col + c, r, lane);
                    else mx_store_any(p, row0, tile.col + c, r, staging, lane);
                }
                __syncwarp();
            }
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

// ---------------------------------------------------------------- few rows
//
// With few rows on one side (a decoding step) the product is the reading of the other side's codes.  That side
// ("long") takes the 128 rows of the MMA, the few rows its NT columns, and K is split over the S CTAs of a cluster so
// that all SMs read; a product of any size that has too few 128 x 128 tiles for the SMs is split the same way.  Each
// CTA multiplies its share of the k-tiles, leaves its partial sums (fp32) in its shared memory, and each then adds 1 / S
// of the columns over the S CTAs, in the order of their ranks, and stores them.  No workspace, no atomics, one launch,
// the same sums whatever order the CTAs run in.

struct FewParams {
    void* C;
    int64_t stride_long, stride_few;   // elements of C between rows of the long side, and of the few
    int n_long, n_few, ktiles;
    int out;
    uint32_t a_format, b_format;       // of the long side, and of the few
    uint32_t tx_bytes;
    int* status;
    unsigned long long wait_limit_ns;
};

constexpr int kFewThreads = 192;   // producer, MMA issuer, four epilogue warps

// DEEP: as many stages as one CTA's shared memory holds, where no SM gets a second CTA (128 x 8192 x 28672 57 -> 40 us, one
// CTA per tile 64 x 8192 x 8192 24 -> 14); otherwise as many as two have room for
template <bool F4, int NT, bool DEEP>
struct FewCfg {
    static constexpr bool kF4 = F4;
    static constexpr int kNT = NT;
    static constexpr int kChunks = F4 ? 2 : 1;
    static constexpr int kABytes = 128 * 128;
    static constexpr int kBBytes = NT * 128;
    static constexpr int kSBytes = kChunks * mx::kRecordBytes;
    static constexpr int kStageBytes = kABytes + kBBytes + 2 * kSBytes;
    static constexpr int kOtherBytes = 1024 + 256;   // alignment and barriers
    static constexpr int kFit = ((DEEP ? 232448 : 233472 / 2 - 1024) - kOtherBytes) / kStageBytes;
    static constexpr int ST = kFit < 12 ? kFit : 12;
    static constexpr int kStages = ST;
    static constexpr int kScaleCols = 8 * kChunks;
    static constexpr int kScaleCol0 = NT;
    static constexpr int kTmem = NT + kScaleCols <= 32 ? 32 : NT + kScaleCols <= 64 ? 64 : NT + kScaleCols <= 128 ? 128 : 256;
    static constexpr int kSmemBytes = ST * kStageBytes + kOtherBytes;
    static_assert(ST * kStageBytes >= NT * 128 * 4, "the partial sums take the place of the stages");
    static_assert(8 * (2 * ST + 1) + 16 <= 256, "barrier block");
};

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t cluster_addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
    return v;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}

__device__ __forceinline__ void few_store(const FewParams& p, int i, int j, float v)
{
    if (i >= p.n_long || j >= p.n_few) return;
    const int64_t at = (int64_t)i * p.stride_long + (int64_t)j * p.stride_few;
    if (p.out == S24_FP32) static_cast<float*>(p.C)[at] = v;
    else if (p.out == S24_BF16) static_cast<__nv_bfloat16*>(p.C)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p.C)[at] = __float2half_rn(v);
}

// columns j .. j + 7 of row i of the long side, where they are neighbours in C: 16 bytes at once where they are all there
// and aligned (3913 x 64 x 256: element by element 11 us, so 3.5)
__device__ __forceinline__ void few_store_row8(const FewParams& p, int i, int j, const float* v)
{
    if (i >= p.n_long || j >= p.n_few) return;
    const int64_t at = (int64_t)i * p.stride_long + j;
    if (p.out != S24_FP32 && j + 8 <= p.n_few) {
        uint16_t* c = static_cast<uint16_t*>(p.C) + at;
        if ((reinterpret_cast<uintptr_t>(c) & 15u) == 0) {
            const int bf16 = p.out == S24_BF16;
            *reinterpret_cast<uint4*>(c) = make_uint4(pack2(v[0], v[1], bf16), pack2(v[2], v[3], bf16), pack2(v[4], v[5], bf16), pack2(v[6], v[7], bf16));
            return;
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) few_store(p, i, j + k, v[k]);
}

// This CTA's share of the columns, summed over the S partial sums in the order of the ranks; the S loads of a step do not
// wait for one another (one at a time cost 35 us of 75 with 128 rows and S = 2).  Where rows of the long side are
// neighbours in C: every S-th column, four rows per thread and step.
template <int S>
__device__ __forceinline__ void few_reduce(const FewParams& p, uint32_t sums, int rank, int row0, int j0, int columns, int thread)
{
    for (int it = thread; it < 32 * ((columns - rank + S - 1) / S); it += 128) {
        const int j = rank + S * (it >> 5), row = (it & 31) * 4;
        float4 v[S];
#pragma unroll
        for (int r = 0; r < S; ++r) v[r] = ld_cluster_f32x4(mapa(sums + (uint32_t)(j * 128 + row) * 4, (uint32_t)r));
#pragma unroll
        for (int r = 1; r < S; ++r) {
            v[0].x += v[r].x;
            v[0].y += v[r].y;
            v[0].z += v[r].z;
            v[0].w += v[r].w;
        }
        few_store(p, row0 + row, j0 + j, v[0].x);
        few_store(p, row0 + row + 1, j0 + j, v[0].y);
        few_store(p, row0 + row + 2, j0 + j, v[0].z);
        few_store(p, row0 + row + 3, j0 + j, v[0].w);
    }
}

// Where the columns are neighbours in C: a row per thread, every S-th eight columns.
template <int S>
__device__ __forceinline__ void few_reduce_rows(const FewParams& p, uint32_t sums, int rank, int row0, int j0, int columns, int row)
{
    for (int j = 8 * rank; j < columns; j += 8 * S) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float w[S];
#pragma unroll
            for (int r = 0; r < S; ++r) w[r] = ld_cluster_f32(mapa(sums + (uint32_t)((j + k) * 128 + row) * 4, (uint32_t)r));
            v[k] = w[0];
#pragma unroll
            for (int r = 1; r < S; ++r) v[k] += w[r];
        }
        few_store_row8(p, row0 + row, j0 + j, v);
    }
}

template <int S>
__device__ __forceinline__ void few_reduce_any(const FewParams& p, uint32_t sums, int rank, int row0, int j0, int columns, int thread)
{
    if (p.stride_few == 1) few_reduce_rows<S>(p, sums, rank, row0, j0, columns, thread);
    else few_reduce<S>(p, sums, rank, row0, j0, columns, thread);
}

template <class Cfg>
__global__ void __launch_bounds__(kFewThreads)
mx_matmul_few_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                     const __grid_constant__ CUtensorMap tm_sa, const __grid_constant__ CUtensorMap tm_sb, const FewParams p)
{
    constexpr int ST = Cfg::kStages, NT = Cfg::kNT;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t smem_a = smem_base;
    const uint32_t smem_b = smem_a + ST * Cfg::kABytes;
    const uint32_t smem_sa = smem_b + ST * Cfg::kBBytes;
    const uint32_t smem_sb = smem_sa + ST * Cfg::kSBytes;
    const uint32_t bar_full = smem_sb + ST * Cfg::kSBytes;
    const uint32_t bar_empty = bar_full + 8 * ST;
    const uint32_t bar_acc = bar_empty + 8 * ST;
    const uint32_t tmem_slot = bar_acc + 8;
    const uint32_t abort_addr = tmem_slot + 8;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_gen + (tmem_slot - smem_base));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + (abort_addr - smem_base));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = (int)gridDim.x;                 // the cluster spans the grid's x
    const int rank = (int)blockIdx.x;
    const int row0 = (int)blockIdx.y * 128;
    const int j0 = (int)blockIdx.z * NT, columns = min(NT, p.n_few - j0);   // more than one z: NT = 128
    const int kt0 = (int)((int64_t)p.ktiles * rank / split), kt1 = (int)((int64_t)p.ktiles * (rank + 1) / split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        mbar_init(bar_acc, 1);
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
        tmem_alloc<1>(tmem_slot, Cfg::kTmem);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot_ptr;
    mx::start_dependents();
    mx::wait_for_predecessors();

    if (warp == 0) {
        if (elect_one()) {
            int s = 0;
            uint32_t ph = 0;
            for (int kt = kt0; kt < kt1; ++kt) {
                if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, p.wait_limit_ns)) {
                    report_timeout(p.status, abort_flag, 1);
                    break;
                }
                const uint32_t full = bar_full + 8 * s;
                mbar_arrive_expect_tx(full, p.tx_bytes);
                tma_load_2d(smem_a + s * Cfg::kABytes, &tm_a, kt * 128, row0, full);
                tma_load_3d<1>(smem_sa + s * Cfg::kSBytes, &tm_sa, 0, kt * Cfg::kChunks, row0 / 128, full);
                tma_load_2d(smem_b + s * Cfg::kBBytes, &tm_b, kt * 128, j0, full);
                tma_load_3d<1>(smem_sb + s * Cfg::kSBytes, &tm_sb, 0, kt * Cfg::kChunks, j0 / 128, full);
                if (++s == ST) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = make_idesc_scaled(p.a_format, p.b_format, 128, NT);
            const uint32_t sfa = tmem_base + (uint32_t)Cfg::kScaleCol0, sfb = sfa + 4 * Cfg::kChunks;
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int kt = kt0; kt < kt1; ++kt) {
                if (!mbar_wait(bar_full + 8 * s, ph, p.wait_limit_ns)) {
                    report_timeout(p.status, abort_flag, 2);
                    ok = false;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < Cfg::kChunks; ++c) {
                    tc_cp_scales<1>(sfa + 4 * c, make_smem_desc(smem_sa + s * Cfg::kSBytes + c * mx::kRecordBytes, 128, 128, kSwizzleNone));
                    tc_cp_scales<1>(sfb + 4 * c, make_smem_desc(smem_sb + s * Cfg::kSBytes + c * mx::kRecordBytes, 128, 128, kSwizzleNone));
                }
                const uint64_t adesc = make_smem_desc(smem_a + s * Cfg::kABytes, 16, 1024, kSwizzle128B);
                const uint64_t bdesc = make_smem_desc(smem_b + s * Cfg::kBBytes, 16, 1024, kSwizzle128B);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t c = Cfg::kF4 ? j >> 1 : 0, id = Cfg::kF4 ? (j & 1) * 2 : j;
                    tc_mma_scaled<1, Cfg::kF4>(tmem_base, adesc + (uint64_t)(j * 2), bdesc + (uint64_t)(j * 2), idesc | (id << 4) | (id << 29), sfa + 4 * c,
                                               sfb + 4 * c, (kt != kt0 || j != 0) ? 1u : 0u);
                }
                tc_commit<1>(bar_empty + 8 * s);
                if (++s == ST) { s = 0; ph ^= 1u; }
            }
            if (ok) tc_commit<1>(bar_acc);
        }
    } else {
        const int quad = warp & 3;
        const int row = 32 * quad + lane;
        if (__all_sync(0xFFFFFFFFu, mbar_wait(bar_acc, 0, p.wait_limit_ns))) {
            tc_fence_after();
            const uint32_t tacc = tmem_base + ((uint32_t)(32 * quad) << 16);
#pragma unroll
            for (int c = 0; c < NT; c += 16) {
                if (c >= columns) break;
                uint32_t r[16];
                tc_ld_32x32b_x16(tacc + (uint32_t)c, r);
                tc_wait_ld();
                if (split == 1 && p.stride_few == 1) {
                    few_store_row8(p, row0 + row, j0 + c, reinterpret_cast<const float*>(r));
                    few_store_row8(p, row0 + row, j0 + c + 8, reinterpret_cast<const float*>(r + 8));
                } else if (split == 1) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) few_store(p, row0 + row, j0 + c + j, __uint_as_float(r[j]));
                } else {   // every copy into the stages and every MMA that reads them is done
#pragma unroll
                    for (int j = 0; j < 16; ++j) st_shared_u32(smem_base + (uint32_t)((c + j) * 128 + row) * 4, r[j]);
                }
            }
        } else if (lane == 0) {
            report_timeout(p.status, abort_flag, 4);
        }
    }

    settle_after_abort(abort_flag);
    __syncwarp();
    if (split > 1) {
        cluster_sync();
        if (warp >= 2) {
            const int thread = (int)threadIdx.x - 64;
            if (split == 2) few_reduce_any<2>(p, smem_base, rank, row0, j0, columns, thread);
            else if (split == 4) few_reduce_any<4>(p, smem_base, rank, row0, j0, columns, thread);
            else few_reduce_any<8>(p, smem_base, rank, row0, j0, columns, thread);
        }
        __syncwarp();
        cluster_sync();   // nobody leaves while another reads its sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, Cfg::kTmem);
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

// the opt-in to more than 48 KB of shared memory, once per kernel and device
template <auto* Kernel>
static int allow_smem(int bytes)
{
    static bool opted_in[64] = {false};
    int dev = 0;
    int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (rc) return rc;
    if (dev >= 0 && dev < 64 && opted_in[dev]) return S24_OK;
    rc = check_cuda(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "cudaFuncSetAttribute(max dynamic shared memory)");
    if (rc == S24_OK && dev >= 0 && dev < 64) opted_in[dev] = true;
    return rc;
}

template <class Cfg>
static int launch_mx(const MxOperand& a, const MxOperand& b, MxParams p, cudaStream_t stream)
{
    CUtensorMap tm_a, tm_b, tm_sa, tm_sb;
    int rc = make_code_map(&tm_a, a, p.K, Cfg::kF4, 128, "A codes");
    if (!rc) rc = make_code_map(&tm_b, b, p.K, Cfg::kF4, Cfg::kBox, "B codes");
    if (!rc) rc = make_scale_map(&tm_sa, a, p.K, Cfg::kChunks, 1, "A scales");
    if (!rc) rc = make_scale_map(&tm_sb, b, p.K, Cfg::kChunks, Cfg::kTilesB, "B scales");
    if (rc) return rc;
    p.tx_bytes = code_tx(a, Cfg::kF4, 128) + Cfg::kSABytes + Cfg::kSBBytes;
    p.tx_box = code_tx(b, Cfg::kF4, Cfg::kBox);
    rc = allow_smem<mx_matmul_kernel<Cfg>>(Cfg::kSmemBytes);
    if (rc) return rc;
    const int64_t tiles = (int64_t)((p.M + 128 * Cfg::kG - 1) / (128 * Cfg::kG)) * ((p.N + Cfg::kBN - 1) / Cfg::kBN);
    if (tiles > 0x7FFFFFFFll / kMxGroupM) return fail(S24_ERR_SHAPE, "mx_matmul: too many output tiles");
    int units = sm_count() / Cfg::kG;
    if (units > tiles) units = (int)tiles;
    // a last pass for at most half of the units: each tile's halves to two of them
    const int last = (int)(tiles % units);
    p.whole = (int)(Cfg::kBN > kMxPart && tiles > units && 2 * last <= units ? tiles - last : tiles);
    p.steps = p.whole + 2 * (int)(tiles - p.whole);
    return check_cuda(mx::launch_overlapped(mx_matmul_kernel<Cfg>, dim3((unsigned)(units * Cfg::kG)), kMxThreads, Cfg::kSmemBytes, Cfg::kG, stream, tm_a, tm_b,
                                            tm_sa, tm_sb, p),
                      "mx_matmul launch");
}

// CTAs of the kernel for few rows that the device holds at once with one per SM, in clusters of `split`: fewer than SMs
// where clusters do not divide the SMs of a GPC (148, 148, 132 and 120 on the device of these measurements)
static int few_slots(int split)
{
    static int cached[64][4] = {};   // each written with the same value, whichever thread gets there first
    const int log = split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sm_count();
    int& slots = cached[dev][log];
    if (slots == 0) {
        using Cfg = FewCfg<false, 16, true>;
        cudaLaunchConfig_t lc = {};
        lc.gridDim = dim3((unsigned)split, 1024);
        lc.blockDim = dim3(kFewThreads);
        lc.dynamicSmemBytes = Cfg::kSmemBytes;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)split;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        lc.attrs = attr;
        lc.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(mx_matmul_few_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, mx_matmul_few_kernel<Cfg>, &lc) != cudaSuccess)
            cudaGetLastError();
        slots = n > 0 ? n * split : sm_count();
    }
    return slots;
}

template <class Cfg>
static int launch_few_cfg(const MxOperand& a, const MxOperand& b, FewParams p, int64_t K, int split, cudaStream_t stream)
{
    CUtensorMap tm_a, tm_b, tm_sa, tm_sb;
    int rc = make_code_map(&tm_a, a, K, Cfg::kF4, 128, "codes of the long side");
    if (!rc) rc = make_code_map(&tm_b, b, K, Cfg::kF4, Cfg::kNT, "codes of the few rows");
    if (!rc) rc = make_scale_map(&tm_sa, a, K, Cfg::kChunks, 1, "scales of the long side");
    if (!rc) rc = make_scale_map(&tm_sb, b, K, Cfg::kChunks, 1, "scales of the few rows");
    if (rc) return rc;
    p.tx_bytes = code_tx(a, Cfg::kF4, 128) + code_tx(b, Cfg::kF4, Cfg::kNT) + 2 * Cfg::kSBytes;
    rc = allow_smem<mx_matmul_few_kernel<Cfg>>(Cfg::kSmemBytes);
    if (rc) return rc;
    const int tiles = (p.n_long + 127) / 128, across = (p.n_few + Cfg::kNT - 1) / Cfg::kNT;
    return check_cuda(mx::launch_overlapped(mx_matmul_few_kernel<Cfg>, dim3((unsigned)split, (unsigned)tiles, (unsigned)across), kFewThreads, Cfg::kSmemBytes, (unsigned)split, stream,
                                            tm_a, tm_b, tm_sa, tm_sb, p),
                      "mx_matmul launch");
}

template <bool F4, int NT>
static int launch_few(const MxOperand& a, const MxOperand& b, FewParams p, int64_t K, int split, cudaStream_t stream)
{
    p.ktiles = (int)((K + (F4 ? 255 : 127)) / (F4 ? 256 : 128));
    if (split > p.ktiles) split = 1;
    const int64_t ctas = (int64_t)((p.n_long + 127) / 128) * ((p.n_few + NT - 1) / NT) * split;
    if (ctas <= few_slots(split)) return launch_few_cfg<FewCfg<F4, NT, true>>(a, b, p, K, split, stream);
    return launch_few_cfg<FewCfg<F4, NT, false>>(a, b, p, K, split, stream);
}

template <bool F4>
static int run_few(const MxOperand& a, const MxOperand& b, const MxParams& p, int split, cudaStream_t stream)
{
    // the few rows are A's, and A's too where neither side's are few: then a warp's 32 rows of B are neighbours in C
    const bool swap = p.M <= p.N || p.N > 128;
    const MxOperand& lng = swap ? b : a;
    const MxOperand& few = swap ? a : b;
    FewParams f;
    f.C = p.C;
    f.stride_long = swap ? 1 : p.ldc;
    f.stride_few = swap ? p.ldc : 1;
    f.n_long = (int)lng.rows;
    f.n_few = (int)few.rows;
    f.ktiles = 0;
    f.out = p.out;
    f.a_format = swap ? p.b_format : p.a_format;
    f.b_format = swap ? p.a_format : p.b_format;
    f.tx_bytes = 0;
    f.status = p.status;
    f.wait_limit_ns = p.wait_limit_ns;
    // eight columns leave room for a sixth stage beside 8-bit rows: 4 x 28672 x 8192 with a 4-bit weight 23.0 -> 22.3 us
    if (f.n_few <= 8) return launch_few<F4, 8>(lng, few, f, p.K, split, stream);
    if (f.n_few <= 16) return launch_few<F4, 16>(lng, few, f, p.K, split, stream);
    if (f.n_few <= 32) return launch_few<F4, 32>(lng, few, f, p.K, split, stream);
    if (f.n_few <= 64) return launch_few<F4, 64>(lng, few, f, p.K, split, stream);
    return launch_few<F4, 128>(lng, few, f, p.K, split, stream);
}

// Which kernel and tile: the least of a time model, in microseconds.  A tile costs a fixed part (launch, first copies,
// last epilogue), one per k-tile and pass over the SMs, and one per further pass; a split of K a fixed part, one per
// k-tile of a CTA, more where SMs have two, and the sum over the cluster.  The constants are fitted to 220 shapes drawn
// over 1 to 4096 rows, 64 to 16384 columns and K of 256 to 16384 in three pairs of formats, each timed with every tile and
// split; on 216 others (profiles/mx_tile_choice.csv) what the model picks takes 1.02 times the best of them on average, 1.31
// at worst.  Examples (tiles 256 x 256, 256 x 128, 128 x 128, then 1, 2, 4, 8 CTAs sharing K): 8192^3 4-bit 183 / 235 / 287 and 341 to 1160 us;
// 543 x 1792 x 1792 8-by-4-bit 9.6 / 6.6 / 6.2, 12.1 / 12.1 / 10.0 / 20.5; 65 x 561 x 12032 41.8 / 25.0 / 24.4, 36.7 / 22.7 /
// 13.1 / 8.6; 1 x 4096 x 4096 15 / 16 / 10, 7.0 / 5.2 / 4.6 / 5.2; 4 x 28672 x 8192 54 / 74 / 59, 22.2 / 27.4 / 32.9 / 45.
struct MxPlan {
    double time;
    int bm, bn, split;   // split > 0: K split over that many CTAs on tiles of at most 128 x 128
};

static MxPlan plan_mx(int64_t M, int64_t N, int ktiles)
{
    struct Tile { int bm, bn, units; double fixed, per_ktile, per_pass; };
    const int sms = sm_count();
    const Tile tiles[3] = {{256, 256, sms / 2, 4.3, 0.31, 2.0}, {256, 128, sms / 2, 3.7, 0.19, 1.2}, {128, 128, sms, 3.2, 0.21, 1.1}};
    MxPlan best = {1e30, 0, 0, 0};
    for (const Tile& t : tiles) {
        const int64_t n = ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
        // a last pass in halves costs two thirds of one
        const int64_t last = n % t.units;
        const double passes = (double)(n / t.units) + (last == 0 ? 0.0 : t.bn > kMxPart && n > t.units && 2 * last <= t.units ? 0.67 : 1.0);
        const double time = t.fixed + passes * ktiles * t.per_ktile + (passes - 1) * t.per_pass;
        if (time < best.time) best = {time, t.bm, t.bn, 0};
    }
    const int64_t few = M < N ? M : N, lng = M < N ? N : M;
    if (few <= 8192 && lng <= 65535 * 128) {   // the grid's y and z
        const double fixed = few <= 16 ? 2.4 : few <= 32 ? 2.7 : few <= 64 ? 3.0 : 4.9;
        const double per_ktile = few <= 64 ? 0.15 : 0.20;
        const double sum = few <= 16 ? 1.1 : few <= 32 ? 1.7 : few <= 64 ? 2.2 : 3.0;
        const double second = few <= 64 ? 2.6 : 3.2;   // with a second CTA on an SM and half the stages for each
        const int64_t n = ((lng + 127) / 128) * ((few + 127) / 128);
        for (int s = 1; s <= 8 && s <= ktiles; s *= 2) {
            const double passes = (double)((n * s + 2 * few_slots(s) - 1) / (2 * few_slots(s)));
            const double time = fixed + passes * ktiles / s * per_ktile * (n * s > few_slots(s) ? second : 1.0) + (s > 1 ? sum : 0.0) + (passes - 1) * 4.0;
            if (time < best.time) best = {time, 0, 0, s};
        }
    }
    return best;
}

template <bool F4>
static int launch_plan(const MxOperand& a, const MxOperand& b, const MxParams& p, const MxPlan& plan, cudaStream_t stream)
{
    if (plan.split > 0) return run_few<F4>(a, b, p, plan.split, stream);
    if (p.wide) {
        if (plan.bm == 256 && plan.bn == 256) return launch_mx<MxCfg<2, 256, F4, 6, true>>(a, b, p, stream);
        if (plan.bm == 256 && plan.bn == 128) return launch_mx<MxCfg<2, 128, F4, 8, true>>(a, b, p, stream);
        if (plan.bm == 128 && plan.bn == 128) return launch_mx<MxCfg<1, 128, F4, 6, true>>(a, b, p, stream);
    } else {
        if (plan.bm == 256 && plan.bn == 256) return launch_mx<MxCfg<2, 256, F4, 5, false>>(a, b, p, stream);
        if (plan.bm == 256 && plan.bn == 128) return launch_mx<MxCfg<2, 128, F4, 7, false>>(a, b, p, stream);
        if (plan.bm == 128 && plan.bn == 128) return launch_mx<MxCfg<1, 128, F4, 5, false>>(a, b, p, stream);
    }
    return fail(S24_ERR_UNSUPPORTED, "mx_matmul: no kernel for tile %d x %d (have 256x256, 256x128, 128x128)", plan.bm, plan.bn);
}

template <bool F4>
static int pick_mx(const MxOperand& a, const MxOperand& b, const MxParams& p, const s24_tile_cfg* cfg, cudaStream_t stream)
{
    const int ktiles = (p.K + (F4 ? 255 : 127)) / (F4 ? 256 : 128);
    if (cfg != nullptr && (cfg->bm != 0 || cfg->bn != 0 || cfg->split != 0)) {
        MxPlan plan = {0.0, cfg->bm, cfg->bn, cfg->split};
        if (plan.bm == 0) plan.bm = plan.bn == 256 || p.M > 128 ? 256 : 128;
        if (plan.bn == 0) plan.bn = 128;
        return launch_plan<F4>(a, b, p, plan, stream);
    }
    return launch_plan<F4>(a, b, p, plan_mx(p.M, p.N, ktiles), stream);
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
    if (cfg != nullptr && cfg->split != 0) {
        const int64_t few = M < N ? M : N, lng = M < N ? N : M;
        const int split = cfg->split;
        if (cfg->bm != 0 || cfg->bn != 0) return fail(S24_ERR_UNSUPPORTED, "mx_matmul: a split of K has tiles of its own (got %d x %d with it)", cfg->bm, cfg->bn);
        if (few > 8192 || lng > 65535 * 128 || (split != 1 && split != 2 && split != 4 && split != 8))
            return fail(S24_ERR_UNSUPPORTED, "mx_matmul: K can be split 1, 2, 4 or 8 ways, with at most 8192 rows on one side (got %d)", split);
    }
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
    p.tx_bytes = p.tx_box = 0;
    p.wide = aligned(C, 32) && (ldc * esz) % 32 == 0;
    p.whole = p.steps = 0;
    p.status = status;
    p.wait_limit_ns = kWaitTimeoutNs;
    const MxOperand oa = {a, a_scales, M, lda, fmt_a}, ob = {b, b_scales, N, ldb, fmt_b};
    auto st = static_cast<cudaStream_t>(stream);
    return both4 ? pick_mx<true>(oa, ob, p, cfg, st) : pick_mx<false>(oa, ob, p, cfg, st);
}
