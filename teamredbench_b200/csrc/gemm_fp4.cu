// gemm_fp4.cu -- products of microscaled 4-bit floating point, dense or grouped by expert.
//
//   out[r, n] = sum over k of a[r, k] * b[e, n, k]   for the rows r of group e (one group of all rows without offsets)
//
// a and b are stored as trb_fp4.cuh says.  The tensor cores multiply them as they are
// (tcgen05.mma.kind::mxf4.block_scale, 64 k an instruction, a scale every 32), accumulate in fp32 in TMEM, and the
// result is rounded once to bf16 or f16.
//
// Measured in CUDA graphs of calls on several sets of inputs: 8192^3 200 us in a burst of 50 ms and 232 sustained, 5.5 and
// 4.7 PFLOP/s, both under the power cap, whose clock is 1.3 to 1.4 GHz from the first launch on (four times the measured
// 16-bit rates would be 164 and 195 us); the tensor pipe is busy in 83% of the cycles, 6% go to the change from tile to
// tile, the rest to instructions of 140 cycles instead of 128.  16436 rows of 16 experts, 4096 x 2048: 76 us (89
// sustained), a sixth of it the change of tiles of only four stages.  16 rows, 4096 x 4096: 5.5 us, launch and one round
// of loads; 256 rows of 32 experts, 2047 x 4096: 31.5 us, 4.6 TB/s, 30.3 with the products left out: the order and depth of
// the loads.  Where n is no multiple of 8 the pair kernel's results leave two bytes at a time: the case of 16 experts above
// with n = 4095 takes 329 us.
//
// No counterpart in the reference.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "trb_common.cuh"
#include "trb_fp4.cuh"
#include "trb_groups.cuh"
#include "trb_launch.cuh"

namespace trb {
namespace fp4 {

__device__ int g_fp4_gemm_error;

// ------------------------------------------------------------------ instructions
// Instruction descriptor of kind::mxf4: e2m1 x e2m1 (types 1), both K-major, e8m0 scales (bit 23), M / 128 at bit 27,
// N / 8 at bit 17; the byte of a scale word that the instruction starts at goes to bits 4 (B) and 29 (A).
__host__ __device__ constexpr uint32_t make_idesc(int m) {
    return (1u << 7) | (1u << 10) | (1u << 23) | ((uint32_t)(m >> 7) << 27);
}
__device__ __forceinline__ uint32_t idesc_n(uint32_t idesc, int n) { return idesc | ((uint32_t)(n >> 3) << 17); }
constexpr uint32_t kSecondHalf = (2u << 4) | (2u << 29);  // scale bytes 2 and 3

__device__ __forceinline__ void mma_pair_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                              uint32_t a_scales, uint32_t b_scales, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(a_scales), "r"(b_scales)
        : "memory");
}
// Arrival on a barrier of either CTA after reads or writes of TMEM, which tcgen05.wait and the fence before it have
// ordered: nothing in memory is handed over, and a release at cluster scope would take a thousand cycles.
__device__ __forceinline__ void mbar_arrive_tmem(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ void mma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t a_scales, uint32_t b_scales, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(a_scales), "r"(b_scales)
        : "memory");
}

// One lane of a warp that runs together.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(uint32_t lo, uint32_t hi) {
    if constexpr (DT == TRB_FLOAT16) {
        __half2 h = __floats2half2_rn(__uint_as_float(lo), __uint_as_float(hi));
        return *reinterpret_cast<uint32_t*>(&h);
    } else {
        __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
        return *reinterpret_cast<uint32_t*>(&h);
    }
}
// Four 8 x 8 blocks of 16-bit values from registers to shared memory, each transposed; thread 8i + j gives the 16-byte
// row that takes column j of block i.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r0),
                 "r"(r1), "r"(r2), "r"(r3)
                 : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr)
                 : "memory");
    return v;
}

// ------------------------------------------------------------------ the product
// A CTA pair computes the transposed tile out^T[256 columns n, R rows r] = b[n, k] * a[r, k]^T, as the 16-bit product
// grouped by expert does: the pair's 256 TMEM lanes run along n, the instruction's N side along up to 256 rows of one
// group in steps of 32, so that few rows cost few.
//
// A stage holds 512 k, two k-blocks of 128 bytes of each operand, by TMA; the MMA thread waits once a stage (a wait costs
// it as much as four products of few rows) and gives its k-blocks back one by one.
//
// The scales are in memory as rows and belong into TMEM as columns: lane l of columns 4i .. 4i + 3 holds the four bytes,
// 128 k, of rows l, 32 + l, 64 + l and 96 + l, and every quarter of the lanes holds a copy.  TMA brings 16 bytes a row
// (512 k) to shared memory, and four scale warps, one for each quarter, store them to TMEM (tcgen05.st), where four
// k-blocks have columns.  The tensor cores' own copy (tcgen05.cp) takes 33 ns of their time for every 128 rows x 128 k:
// with 12 a stage 8192^3 took 399 us where the products alone take 183.  Loads of the scale warps' own held up their
// signal to the MMA thread, which waits for them: 403 us.
//
// What is left of TMEM holds two accumulators of 256 columns that share 96: the epilogue takes the shared columns into
// registers first, and then the next tile's products may start.
constexpr int kEpiWarps = 8;                    // two for each quarter of the TMEM lanes
constexpr int kScaleWarps = 4;
constexpr int kProductThreads = 96 + 32 * (kEpiWarps + kScaleWarps);
constexpr int kTileN = 256;                     // columns of a tile (pair)
constexpr int kTileRows = 256;                  // most rows of a tile
constexpr int kBK = 256;                        // k of a k-block: 128 bytes
constexpr int kStageK = 2 * kBK;
constexpr int kStages = 3;
constexpr int kSlots = 2 * kStages;             // k-blocks
constexpr int kWBlock = 128 * 128;              // bytes of one CTA's share of a k-block
constexpr int kXBlock = kTileRows / 2 * 128;
constexpr int kScaleRows = 128 + kTileRows;     // of b and of a that a CTA's products need
constexpr int kScaleStage = kScaleRows * 16;    // a stage's scales as rows
constexpr int kScaleCols = kScaleRows / 32 * 2; // of a k-block in TMEM
constexpr int kScaleSlots = 4;                  // k-blocks whose scales TMEM holds
constexpr int kEpiBytes = 16 * 64;              // 16 rows x 32 columns of 16-bit results
constexpr int kMaxK = 1 << 26;                  // a tile takes less than the limit of a wait
constexpr int kTmemCols = 512;
constexpr int kTmemScales = kTmemCols - kScaleSlots * kScaleCols;
constexpr int kSecondAcc = kTmemScales - kTileRows;    // columns kSecondAcc .. kTileRows - 1 are both accumulators'
constexpr int kSharedBlocks = (kTileRows - kSecondAcc) / 32;
static_assert(kSecondAcc % 32 == 0 && kSecondAcc >= kTileRows - kSecondAcc, "whole blocks of 32 columns are shared");
constexpr size_t kProductSmem =
    (size_t)kSlots * (kWBlock + kXBlock) + 2 * kScaleStage + kEpiWarps * kEpiBytes + 1024;

struct ProductTile {
    int e, row0, rows, n0;
};

// Tile t: groups in order; inside a group, runs of 8 chunks walk the columns together (a panel of b is read by the
// chunks next to each other in time).  Without groups (0) there is one of all rows.
__device__ __forceinline__ ProductTile product_tile(int t, int groups, int total_rows, int num_n, const GroupTable& g) {
    const int e = groups > 0 ? group_of_chunk(t / num_n, groups, g) : 0;
    const int local = groups > 0 ? t - g.chunk0[e] * num_n : t;
    const int rows = groups > 0 ? g.rows[e] : total_rows;
    const int chunks = (rows + kTileRows - 1) / kTileRows;
    const int run = 8 * num_n;
    const int first = local / run * 8;
    const int width = min(8, chunks - first);
    const int in_run = local - first * num_n;
    const int chunk = first + in_run % width;
    const int per = ((rows + chunks - 1) / chunks + 31) & ~31;
    ProductTile p;
    p.e = e;
    p.row0 = (groups > 0 ? g.start[e] : 0) + chunk * per;
    p.rows = min(per, rows - chunk * per);
    p.n0 = in_run / width * kTileN;
    return p;
}

// Scale bytes from the first `valid` on are taken as 0 (2^-127): what stands behind a row's last block is anyone's, and
// meets only the zeros that TMA fills in there.
__device__ __forceinline__ uint4 first_bytes(uint4 v, int valid) {
    uint32_t* const w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = valid - 4 * i;
        if (n < 4) w[i] = n <= 0 ? 0 : w[i] & ((1u << (8 * n)) - 1u);
    }
    return v;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kProductThreads, 1)
    gemm_fp4_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX128,
                    const __grid_constant__ CUtensorMap tmX64, const __grid_constant__ CUtensorMap tmX32,
                    const __grid_constant__ CUtensorMap tmWS, const __grid_constant__ CUtensorMap tmXS, const int* offsets, uint16_t* out, int groups,
                    int total_rows, int N, int K) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ int group_words[3 * kMaxGroups + 1];
    __shared__ __align__(8) uint64_t full_bar[kStages];   // leader: both CTAs' TMA bytes land here, and their scale warps
    __shared__ __align__(8) uint64_t empty_bar[kSlots];   // both: the products that read the k-block are done
    __shared__ __align__(8) uint64_t scalef_bar[2];       // each CTA: a stage's scales have landed as rows
    __shared__ __align__(8) uint64_t scalee_bar[2];       // each CTA: its scale warps have read them
    __shared__ __align__(8) uint64_t accf_bar;            // both: accumulator ready for the epilogue
    __shared__ __align__(8) uint64_t acce_bar;            // leader: both CTAs' epilogues have taken the shared columns
    __shared__ __align__(8) uint64_t drain_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;

    const uint32_t sW = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sX = sW + kSlots * kWBlock;
    const uint32_t sScale = sX + kSlots * kXBlock;
    const uint32_t sEpi = sScale + 2 * kScaleStage;

    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int pair = blockIdx.x >> 1;
    const int num_pairs = gridDim.x >> 1;
    const int num_n = (N + kTileN - 1) / kTileN;
    const int num_stages = (K + kStageK - 1) / kStageK;
    const GroupTable table = {group_words, group_words + kMaxGroups, group_words + 2 * kMaxGroups};

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&full_bar[s]), 1 + 2 * kScaleWarps);
        for (int s = 0; s < kSlots; ++s) mbar_init(smem_u32(&empty_bar[s]), 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&scalef_bar[s]), 1);
            mbar_init(smem_u32(&scalee_bar[s]), kScaleWarps);
        }
        mbar_init(smem_u32(&accf_bar), 1);
        mbar_init(smem_u32(&acce_bar), 2 * kEpiWarps);  // of both CTAs
        mbar_init(smem_u32(&drain_bar), 1);
        abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX128);
        tma_prefetch_desc(&tmX64);
        tma_prefetch_desc(&tmX32);
        tma_prefetch_desc(&tmWS);
        tma_prefetch_desc(&tmXS);
    }
    if (warp == 0) {
        tmem_alloc_pair(smem_u32(&tmem_slot), kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // barrier inits of both CTAs visible before any cross-CTA signal
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;
    // Only now that this block has its TMEM: the next grid's blocks take theirs before they wait for this grid.
    grid_launch_dependents();
    grid_dependency_wait();  // offsets, operands and out may belong to the previous grid until here
    int num_tiles = (total_rows + kTileRows - 1) / kTileRows * num_n;
    if (offsets != nullptr) {
        groups = load_groups(offsets, groups, total_rows, table, &g_fp4_gemm_error);
        if (warp == 0) scan_chunks(groups, kTileRows, table, lane);
        __syncthreads();
        num_tiles = table.chunk0[groups] * num_n;
    } else {
        groups = 0;
    }

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer (both CTAs; completion on the leader's full barriers)
            uint32_t stage = 0, phase = 0;
            uint32_t issued_mask = 0, issued_phase = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
                const ProductTile p = product_tile(tile, groups, total_rows, num_n, table);
                const int half = ((p.rows + 31) & ~31) >> 1;  // rows this CTA loads
                const int x_row = p.row0 + (int)rank * half;
                // One box a k-block, of 128, 64 or 32 rows: a request costs more than the rows nobody uses.
                const CUtensorMap* tmX = half > 64 ? &tmX128 : half > 32 ? &tmX64 : &tmX32;
                const uint32_t x_bytes = (half > 64 ? 128 : half > 32 ? 64 : 32) * 128;
                const int w_col = p.n0 + (int)rank * 128;
                for (int s = 0; ok && s < num_stages; ++s) {
                    const int blocks = s * kStageK + kBK < K ? 2 : 1;
                    const uint32_t fb_local = smem_u32(&full_bar[stage]);
                    const uint32_t fb = fb_local & kPeerBitMask;
                    for (int i = 0; i < 2; ++i) {  // a k-block past K is not loaded, but its turn is taken
                        const uint32_t slot = 2 * stage + i;
                        if (!mbar_wait(smem_u32(&empty_bar[slot]), phase ^ 1u, &abort_flag)) {
                            atomicCAS(&g_fp4_gemm_error, 0, kErrProducerWait);
                            abort_flag = 1;
                            ok = false;
                            break;
                        }
                        if (i == 0) {
                            if (leader) mbar_arrive_expect_tx(fb_local, 2 * blocks * (kWBlock + x_bytes));
                            issued_mask |= 1u << stage;
                            issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                        }
                        if (i < blocks) {
                            const int byte = (s * 2 + i) * 128;
                            tma_load_3d_pair(sW + slot * kWBlock, &tmW, fb, byte, w_col, p.e);
                            tma_load_2d_pair(sX + slot * kXBlock, tmX, fb, byte, x_row);
                        }
                    }
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (leader)  // every armed phase completes only once both CTAs' bytes have landed
                for (int s = 0; s < kStages; ++s)
                    if (issued_mask & (1u << s))
                        if (!mbar_wait(smem_u32(&full_bar[s]), (issued_phase >> s) & 1u, nullptr))
                            atomicCAS(&g_fp4_gemm_error, 0, kErrDrainWait);
        }
    } else if (warp == 1) {
        if (leader) {
            // ---------------- MMA issuer: the leader CTA only; the whole warp goes along, so that what the instructions
            // take is in uniform registers
            const bool elected = elect_one();
            const uint64_t w_desc0 = make_sdesc(sW, 16, 1024), x_desc0 = make_sdesc(sX, 16, 1024);
            uint32_t stage = 0, phase = 0, scale_slot = 0;
            bool ok = true;
            int t_local = 0;
            for (int tile = pair; ok && tile < num_tiles; tile += num_pairs, ++t_local) {
                const ProductTile p = product_tile(tile, groups, total_rows, num_n, table);
                const uint32_t idesc = idesc_n(make_idesc(256), (p.rows + 31) & ~31);
                // The epilogue takes the tiles in order: with the last tile's shared columns, all of the one before.
                if (t_local > 0 && !mbar_wait(smem_u32(&acce_bar), (uint32_t)(t_local - 1) & 1u, &abort_flag)) {
                    if (elected) atomicCAS(&g_fp4_gemm_error, 0, kErrMmaWait);
                    abort_flag = 1;
                    break;
                }
                const uint32_t d_tmem = tmem_base + (t_local & 1 ? kSecondAcc : 0);
                for (int s = 0; s < num_stages; ++s) {
                    if (!mbar_wait(smem_u32(&full_bar[stage]), phase, &abort_flag)) {
                        if (elected) atomicCAS(&g_fp4_gemm_error, 0, kErrMmaWait);
                        abort_flag = 1;
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const int left = K - s * kStageK;
                    if (elected) {
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const uint32_t slot = 2 * stage + b;
                            const uint64_t w = w_desc0 + (uint64_t)((slot * kWBlock) >> 4);
                            const uint64_t x = x_desc0 + (uint64_t)((slot * kXBlock) >> 4);
                            const uint32_t scales = tmem_base + (uint32_t)(kTmemScales + (scale_slot + b) * kScaleCols);
#pragma unroll
                            for (int i = 0; i < kBK / 64; ++i) {  // 64 k: 32 bytes of a k-block's 128, half of a scale word
                                const uint32_t t = scales + (uint32_t)((i >> 1) * (kScaleCols / 2));
                                if (b * kBK + i * 64 < left)
                                    mma_pair_mxf4(d_tmem, w + (uint64_t)((i * 32) >> 4), x + (uint64_t)((i * 32) >> 4),
                                                  (i & 1) ? idesc | kSecondHalf : idesc, t, t + 4,
                                                  (s != 0 || b != 0 || i != 0) ? 1u : 0u);
                            }
                            tc_commit_pair_multicast(smem_u32(&empty_bar[slot]), 0x3);
                        }
                    }
                    __syncwarp();
                    scale_slot ^= 2;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (ok && elected) tc_commit_pair_multicast(smem_u32(&accf_bar), 0x3);
            }
            if (elected) tc_commit_pair_multicast(smem_u32(&drain_bar), 0x1);
            if (!mbar_wait(smem_u32(&drain_bar), 0, nullptr)) atomicCAS(&g_fp4_gemm_error, 0, kErrDrainWait);
        }
    } else if (warp < 2 + kEpiWarps) {
        // ---------------- epilogue (both CTAs): a TMEM lane quarter (32 columns of out) and every other block of 32 rows
        // each.  TMEM holds out^T, so the blocks go through shared memory transposed (stmatrix.trans), 16 rows at a time,
        // and leave as 64-byte runs of a row, 16 bytes a lane.
        const int q = warp & 3, own = (warp - 2) >> 2;
        const uint32_t acce_leader = mapa_shared(smem_u32(&acce_bar), 0);
        const uint32_t buf = sEpi + (uint32_t)((warp - 2) * kEpiBytes);
        // block row j is 64 bytes; its 16-byte piece i stands at i ^ ((j >> 1) & 3), free of bank conflicts both ways
        const uint32_t st_row = buf + (uint32_t)((lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) * 16));
        const uint32_t ld_row = buf + (uint32_t)((lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) * 16));
        const bool whole = N % 8 == 0;  // rows of out begin at 16 bytes
        int t_local = 0;
        for (int tile = pair; tile < num_tiles; tile += num_pairs, ++t_local) {
            const ProductTile p = product_tile(tile, groups, total_rows, num_n, table);
            const bool odd = t_local & 1;
            bool ok = mbar_wait(smem_u32(&accf_bar), (uint32_t)t_local & 1u, &abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                if (lane == 0) {
                    atomicCAS(&g_fp4_gemm_error, 0, kErrEpilogueWait);
                    abort_flag = 1;
                }
                break;
            }
            tc_fence_after();
            const uint32_t t_tile = tmem_base + ((uint32_t)(q * 32) << 16) + (odd ? kSecondAcc : 0);
            const int col = p.n0 + (int)rank * 128 + q * 32 + (lane & 3) * 8;
            uint16_t* const out_lane = out + (size_t)(p.row0 + (lane >> 2)) * N + col;
            const auto take = [&](int c, uint32_t (&r)[16]) {  // 32 rows, rounded
                uint32_t lo[16], hi[16];  // TMEM lanes 0..15 and 16..31 of the quarter
                tmem_ld_16x256b_x4(t_tile + (uint32_t)(c * 32), lo);
                tmem_ld_16x256b_x4(t_tile + (16u << 16) + (uint32_t)(c * 32), hi);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    r[4 * j] = pack2<DT>(lo[4 * j], lo[4 * j + 1]);
                    r[4 * j + 1] = pack2<DT>(lo[4 * j + 2], lo[4 * j + 3]);
                    r[4 * j + 2] = pack2<DT>(hi[4 * j], hi[4 * j + 1]);
                    r[4 * j + 3] = pack2<DT>(hi[4 * j + 2], hi[4 * j + 3]);
                }
            };
            const auto put = [&](int c, const uint32_t (&r)[16]) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    __syncwarp();  // what was in buf has been read
#pragma unroll
                    for (int j = 0; j < 2; ++j) {  // rows 8j .. 8j + 7; columns in octets 0..3
                        const uint32_t* const v = r + 8 * half + 4 * j;
                        stmatrix_x4_trans(st_row + (uint32_t)(j * 8 * 64), v[0], v[1], v[2], v[3]);
                    }
                    __syncwarp();
                    if (col >= N) continue;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = c * 32 + half * 16 + i * 8;
                        if (row + (lane >> 2) >= p.rows) continue;
                        const uint4 v = ld_shared_v4(ld_row + (uint32_t)(i * 8 * 64));
                        uint16_t* const to = out_lane + (size_t)row * N;
                        if (whole) {
                            *reinterpret_cast<uint4*>(to) = v;
                        } else {
#pragma unroll
                            for (int h = 0; h < 8; ++h)
                                if (col + h < N) to[h] = (uint16_t)(word(v, h >> 1) >> (16 * (h & 1)));
                        }
                    }
                }
            };
            // The shared columns: the last ones of the first accumulator, the first ones of the second.
            const int shared0 = odd ? 0 : kSecondAcc / 32;
            uint32_t r[(kSharedBlocks + 1) / 2][16];
#pragma unroll
            for (int c = 0; c < kSharedBlocks; c += 2)
                if (c + own < kSharedBlocks && (shared0 + c + own) * 32 < p.rows) take(shared0 + c + own, r[c / 2]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_tmem(acce_leader);
#pragma unroll
            for (int c = 0; c < kSharedBlocks; c += 2)
                if (c + own < kSharedBlocks && (shared0 + c + own) * 32 < p.rows) put(shared0 + c + own, r[c / 2]);
            // The others; the warp that had one block less above begins.
            const int first = odd ? kSharedBlocks : 0, last = odd ? kTileRows / 32 : kSecondAcc / 32;
#pragma unroll 1
            for (int c = first + (own ^ 1); c < last && c * 32 < p.rows; c += 2) {
                take(c, r[0]);
                put(c, r[0]);
            }
        }
    } else if (warp < 2 + kEpiWarps + kScaleWarps) {
        // ---------------- scales (both CTAs, each for its 128 columns n and all rows of the tile), to this warp's quarter
        // of the TMEM lanes
        const int q = warp & 3;
        const uint32_t full_leader = mapa_shared(smem_u32(&full_bar[0]), 0);
        const uint32_t t_quarter = tmem_base + ((uint32_t)(q * 32) << 16) + kTmemScales;
        uint32_t stage = 0, scale_slot = 0, buffer = 0, phase = 0;
        int before = -kScaleSlots;  // the k-block whose columns are next
        uint32_t parity = 0;        // of the empty barrier's phase that ends with that k-block
        bool ok = true;
        for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
            const bool second = product_tile(tile, groups, total_rows, num_n, table).rows > 128;
            for (int s = 0; s < num_stages; ++s) {
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&scalef_bar[buffer]), phase, &abort_flag));
                const uint32_t rows = sScale + buffer * kScaleStage + lane * 16;
                uint4 v[3][4];  // of b, of the tile's first 128 rows of a, of the others
#pragma unroll
                for (int part = 0; part < 3; ++part)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (part < 2 || second) v[part][j] = ld_shared_v4(rows + (uint32_t)((part * 128 + 32 * j) * 16));
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&scalee_bar[buffer]));
                if (++buffer == 2) {
                    buffer = 0;
                    phase ^= 1u;
                }
                if ((s + 1) * kStageK > K)  // the last stage
#pragma unroll
                    for (int part = 0; part < 3; ++part)
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[part][j] = first_bytes(v[part][j], K / kBlock - s * (kStageK / kBlock));
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    if (before >= 0) {
                        const bool free = mbar_wait(smem_u32(&empty_bar[before]), parity, &abort_flag);
                        ok = __all_sync(0xffffffffu, free) && ok;
                    }
                    if (++before == kSlots) {
                        before = 0;
                        parity ^= 1u;
                    }
                    tc_fence_after();
                    // 128 k: 4 columns of b, 8 of a; then the other 128 k
                    const auto column = [&](int c) { return word(v[c % 12 / 4][c % 4], 2 * b + c / 12); };
                    uint32_t cols0[16], cols1[8];
#pragma unroll
                    for (int c = 0; c < 16; ++c) cols0[c] = column(c);
#pragma unroll
                    for (int c = 0; c < 8; ++c) cols1[c] = column(16 + c);
                    if (ok) {
                        tmem_st_32x32b_x16(t_quarter + (scale_slot + b) * kScaleCols, cols0);
                        tmem_st_32x32b_x8(t_quarter + (scale_slot + b) * kScaleCols + 16, cols1);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (!ok) {
                    if (lane == 0) {
                        atomicCAS(&g_fp4_gemm_error, 0, kErrProducerWait);
                        abort_flag = 1;
                    }
                    break;
                }
                if (lane == 0) mbar_arrive_tmem(full_leader + (uint32_t)(stage * sizeof(uint64_t)));
                scale_slot ^= 2;
                if (++stage == kStages) stage = 0;
            }
        }
    } else if (lane == 0) {
        // ---------------- TMA producer of the scales (both CTAs, each for itself)
        uint32_t buffer = 0, phase = 0;
        int issued = 0;
        bool ok = true;
        for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
            const ProductTile p = product_tile(tile, groups, total_rows, num_n, table);
            const uint32_t bytes = (p.rows > 128 ? 3 : 2) * 128 * 16;
            for (int s = 0; s < num_stages; ++s) {
                if (!mbar_wait(smem_u32(&scalee_bar[buffer]), phase ^ 1u, &abort_flag)) {
                    atomicCAS(&g_fp4_gemm_error, 0, kErrProducerWait);
                    abort_flag = 1;
                    ok = false;
                    break;
                }
                const uint32_t bar = smem_u32(&scalef_bar[buffer]), to = sScale + buffer * kScaleStage;
                mbar_arrive_expect_tx(bar, bytes);
                tma_load_3d(to, &tmWS, bar, s * 16, p.n0 + (int)rank * 128, p.e);
                tma_load_2d(to + 128 * 16, &tmXS, bar, s * 16, p.row0);
                if (p.rows > 128) tma_load_2d(to + 256 * 16, &tmXS, bar, s * 16, p.row0 + 128);
                ++issued;
                if (++buffer == 2) {
                    buffer = 0;
                    phase ^= 1u;
                }
            }
        }
        for (int i = min(issued, 2); i > 0; --i) {  // no copy in flight when this CTA ends
            if (buffer == 0) {
                buffer = 2;
                phase ^= 1u;
            }
            --buffer;
            if (!mbar_wait(smem_u32(&scalef_bar[buffer]), phase, nullptr))
                atomicCAS(&g_fp4_gemm_error, 0, kErrDrainWait);
        }
    }

    // Teardown: the leader's MMAs read the peer's shared memory and write its
    // TMEM, so neither CTA releases TMEM or exits before both are done.
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// ------------------------------------------------------------------ few tiles: K split over a cluster
// The same transposed product with single CTAs, 128 columns of out x up to R rows, when the tiles of pairs are too few to
// occupy the GPU: the CL CTAs of a cluster take a tile's K in CL parts, each streaming its own share of the weights.  CTA
// r owns columns [128 r / CL, ...) of the tile: the others send it their fp32 parts through distributed shared memory,
// and it adds them in the order of K, so the result does not depend on timing.  One tile a cluster.  Four warps bring the
// scales to TMEM, a stage ahead of the products, and read the results afterwards.
constexpr int kSplitThreads = 224;  // producer warp, MMA warp, 4 warps for scales and results, producer of the scales
constexpr int kSplitN = 128;
constexpr int kWStage = 2 * kWBlock;
template <int R>
struct SplitCfg {
    static constexpr int kStages = R == 64 ? 3 : 2;
    static constexpr int kX = 2 * R * 128;                 // a stage's rows of a
    static constexpr int kScales = (128 + R) * 16;
    static constexpr int kScaleCols = 16;                  // of a k-block in TMEM: 128 k of b and of a take 4 each
    static constexpr int kAcc = R < 32 ? 32 : R;
    static constexpr int kTmem = kAcc + kStages * 2 * kScaleCols <= 128 ? 128 : 256;
    static constexpr int kReceive = R * kSplitN * 4;
    static constexpr size_t kSmem = (size_t)kStages * (kWStage + kX + kScales) + kReceive + 1024;
    static constexpr int kPerSm = R == 64 ? 1 : 2;
};

__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

template <int DT>
__device__ __forceinline__ uint16_t round16(float v) {
    if constexpr (DT == TRB_FLOAT16) return __half_as_ushort(__float2half_rn(v));
    else return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

template <int DT, int R>
__global__ void __launch_bounds__(kSplitThreads, SplitCfg<R>::kPerSm)
    gemm_fp4_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                          const __grid_constant__ CUtensorMap tmWS, const __grid_constant__ CUtensorMap tmXS,
                          const int* offsets, uint16_t* out, int groups, int total_rows, int N, int K, int log2_cl) {
    using Cfg = SplitCfg<R>;
    constexpr int kRing = Cfg::kStages;

    extern __shared__ uint8_t smem_raw[];
    __shared__ int group_words[3 * kMaxGroups + 1];
    __shared__ __align__(8) uint64_t full_bar[kRing];    // operands have landed, and the four warps stored their scales
    __shared__ __align__(8) uint64_t scalef_bar[kRing];  // scales have landed as rows
    __shared__ __align__(8) uint64_t empty_bar[kRing];   // the products that read the stage are done
    __shared__ __align__(8) uint64_t done_bar;           // all products of the tile
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;

    const uint32_t sW = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sX = sW + kRing * kWStage;
    const uint32_t sScale = sX + kRing * Cfg::kX;
    const uint32_t receive = sScale + kRing * Cfg::kScales;

    const uint32_t rank = cluster_ctarank();
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int num_n = (N + kSplitN - 1) / kSplitN;
    const int num_stages = (K + kStageK - 1) / kStageK;
    const GroupTable table = {group_words, group_words + kMaxGroups, group_words + 2 * kMaxGroups};

    if (threadIdx.x == 0) {
        for (int s = 0; s < kRing; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1 + 4);
            mbar_init(smem_u32(&scalef_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        mbar_init(smem_u32(&done_bar), 1);
        abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmWS);
        tma_prefetch_desc(&tmXS);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_slot), Cfg::kTmem);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;
    grid_launch_dependents();  // after the allocation, as above
    grid_dependency_wait();
    const int tile = blockIdx.x >> log2_cl, chunk = tile / num_n;
    int e = 0, row0 = chunk * R, rows = min(R, total_rows - row0);
    bool some = rows > 0;
    if (offsets != nullptr) {
        groups = load_groups(offsets, groups, total_rows, table, &g_fp4_gemm_error);
        if (warp == 0) scan_chunks(groups, R, table, lane);
        __syncthreads();
        some = chunk < table.chunk0[groups];
        if (some) {
            e = group_of_chunk(chunk, groups, table);
            const int first = (chunk - table.chunk0[e]) * R;
            row0 = table.start[e] + first;
            rows = min(R, table.rows[e] - first);
        }
    }
    if (!some) {  // the whole cluster: the grid covers the most tiles there can be
        __syncthreads();
        if (warp == 1) tmem_dealloc(tmem_base, Cfg::kTmem);
        return;
    }

    const int cl = 1 << log2_cl;
    const int padded = (rows + 15) & ~15;
    const int n0 = (tile - chunk * num_n) * kSplitN;
    const int s0 = (num_stages * (int)rank) >> log2_cl, s1 = (num_stages * ((int)rank + 1)) >> log2_cl;

    cluster_arrive();  // peers may not write here before this CTA runs; the wait is before the first such write

    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer
            uint32_t stage = 0, phase = 0;
            int issued = 0;
            for (int s = s0; s < s1; ++s) {
                if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, &abort_flag)) {
                    atomicCAS(&g_fp4_gemm_error, 0, kErrProducerWait);
                    abort_flag = 1;
                    break;
                }
                const int blocks = s * kStageK + kBK < K ? 2 : 1;
                const uint32_t bar = smem_u32(&full_bar[stage]);
                const uint32_t w = sW + stage * kWStage, x = sX + stage * Cfg::kX;
                mbar_arrive_expect_tx(bar, blocks * (kWBlock + Cfg::kX / 2));
                for (int i = 0; i < blocks; ++i) {
                    tma_load_3d(w + i * kWBlock, &tmW, bar, (2 * s + i) * 128, n0, e);
                    tma_load_2d(x + i * (Cfg::kX / 2), &tmX, bar, (2 * s + i) * 128, row0);
                }
                ++issued;
                if (++stage == kRing) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            for (int i = min(issued, kRing); i > 0; --i) {  // no copy in flight when this CTA ends
                if (stage == 0) {
                    stage = kRing;
                    phase ^= 1u;
                }
                --stage;
                if (!mbar_wait(smem_u32(&full_bar[stage]), phase, nullptr))
                    atomicCAS(&g_fp4_gemm_error, 0, kErrDrainWait);
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer
        const bool elected = elect_one();
        const uint64_t w_desc0 = make_sdesc(sW, 16, 1024), x_desc0 = make_sdesc(sX, 16, 1024);
        const uint32_t idesc = idesc_n(make_idesc(128), padded);
        uint32_t stage = 0, phase = 0;
        for (int s = s0; s < s1; ++s) {
            if (!mbar_wait(smem_u32(&full_bar[stage]), phase, &abort_flag)) {
                if (elected) atomicCAS(&g_fp4_gemm_error, 0, kErrMmaWait);
                abort_flag = 1;
                break;
            }
            tc_fence_after();
            const uint32_t scales = tmem_base + Cfg::kAcc + stage * 2 * Cfg::kScaleCols;
            const int left = K - s * kStageK;
            if (elected) {
#pragma unroll
                for (int i = 0; i < kStageK / 64; ++i) {  // 64 k: 32 bytes of a k-block's 128, half of a scale word
                    const uint32_t t = scales + (uint32_t)((i >> 1) * (Cfg::kScaleCols / 2));
                    if (i * 64 < left)
                        mma_mxf4(tmem_base,
                                 w_desc0 + (uint64_t)((stage * kWStage + (i >> 2) * kWBlock + (i & 3) * 32) >> 4),
                                 x_desc0 + (uint64_t)((stage * Cfg::kX + (i >> 2) * (Cfg::kX / 2) + (i & 3) * 32) >> 4),
                                 (i & 1) ? idesc | kSecondHalf : idesc, t, t + 4, (s != s0 || i != 0) ? 1u : 0u);
                }
                tc_commit(smem_u32(&empty_bar[stage]));
            }
            __syncwarp();
            if (++stage == kRing) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (elected) tc_commit(smem_u32(&done_bar));
        if (!mbar_wait(smem_u32(&done_bar), 0, nullptr) && elected) atomicCAS(&g_fp4_gemm_error, 0, kErrDrainWait);
    } else if (warp == 6) {
        if (lane == 0) {
            // ---------------- TMA producer of the scales
            uint32_t stage = 0, phase = 0;
            int issued = 0;
            for (int s = s0; s < s1; ++s) {
                if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, &abort_flag)) {
                    atomicCAS(&g_fp4_gemm_error, 0, kErrProducerWait);
                    abort_flag = 1;
                    break;
                }
                const uint32_t bar = smem_u32(&scalef_bar[stage]), scale = sScale + stage * Cfg::kScales;
                mbar_arrive_expect_tx(bar, Cfg::kScales);
                tma_load_3d(scale, &tmWS, bar, s * 16, n0, e);
                tma_load_2d(scale + 128 * 16, &tmXS, bar, s * 16, row0);
                ++issued;
                if (++stage == kRing) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            for (int i = min(issued, kRing); i > 0; --i) {
                if (stage == 0) {
                    stage = kRing;
                    phase ^= 1u;
                }
                --stage;
                if (!mbar_wait(smem_u32(&scalef_bar[stage]), phase, nullptr))
                    atomicCAS(&g_fp4_gemm_error, 0, kErrDrainWait);
            }
        }
    } else {
        // ---------------- scales, to this warp's quarter of the TMEM lanes.  Rows that have landed mean that the stage's
        // last products are done: the producer waited for them.
        const uint32_t t_quarter = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + Cfg::kAcc;
        uint32_t stage = 0, phase = 0;
        for (int s = s0; s < s1; ++s) {
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&scalef_bar[stage]), phase, &abort_flag))) {
                if (lane == 0) {
                    atomicCAS(&g_fp4_gemm_error, 0, kErrProducerWait);
                    abort_flag = 1;
                }
                break;
            }
            tc_fence_after();
            const uint32_t scale = sScale + stage * Cfg::kScales + lane * 16;
            const int valid = K / kBlock - s * (kStageK / kBlock);
            uint4 v[2][4];  // of b, of a
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[0][j] = first_bytes(ld_shared_v4(scale + (uint32_t)(32 * j * 16)), valid);
                v[1][j] = make_uint4(0, 0, 0, 0);
                // Past the tile's rows: what meets the products nobody takes.
                if (32 * j + lane < R) v[1][j] = first_bytes(ld_shared_v4(scale + (uint32_t)((128 + 32 * j) * 16)), valid);
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t cols[16];  // 128 k: 4 columns of b, 4 of a; then the other 128 k
#pragma unroll
                for (int c = 0; c < 16; ++c) cols[c] = word(v[c % 8 / 4][c % 4], 2 * b + c / 8);
                tmem_st_32x32b_x16(t_quarter + (uint32_t)((stage * 2 + b) * Cfg::kScaleCols), cols);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&full_bar[stage]));
            if (++stage == kRing) {
                stage = 0;
                phase ^= 1u;
            }
        }
    }
    __syncwarp();
    cluster_wait();  // every CTA of the cluster runs
    const int log2_own = 7 - log2_cl, own = 1 << log2_own;  // columns this CTA owns
    const bool results = warp >= 2 && warp < 6;
    if (results) {
        // ---------------- lane = column of out, TMEM column = row
        const int n = (warp & 3) * 32 + lane;
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&done_bar), 0, &abort_flag));
        if (!ok && lane == 0) {
            atomicCAS(&g_fp4_gemm_error, 0, kErrEpilogueWait);
            abort_flag = 1;
        }
        if (ok) {
            tc_fence_after();
            const uint32_t owner = mapa_shared(receive, (uint32_t)(n >> log2_own)) +
                                   (uint32_t)((((int)rank * R << log2_own) + (n & (own - 1))) * 4);
            for (int c = 0; c < padded; c += 16) {
                uint32_t v[16];
                tmem_ld_32x32b_x16(tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (c + i < rows) st_cluster_f32(owner + (uint32_t)(((c + i) << log2_own) * 4), __uint_as_float(v[i]));
            }
            tc_fence_before();
        }
    }
    // The parts have arrived, and no CTA leaves while a peer may still write into it.
    __syncwarp();
    cluster_sync_all();
    if (results && ok) {  // four columns of a row a thread
        const int log2_quads = log2_own - 2;
        for (int i = threadIdx.x - 64; i < rows << log2_quads; i += 128) {
            const int r = i >> log2_quads, c = (i & ((1 << log2_quads) - 1)) * 4;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int src = 0; src < 8; ++src) {
                if (src >= cl) break;
                const uint4 p = ld_shared_v4(receive + (uint32_t)((((src * R + r) << log2_own) + c) * 4));
                v[0] += __uint_as_float(p.x);
                v[1] += __uint_as_float(p.y);
                v[2] += __uint_as_float(p.z);
                v[3] += __uint_as_float(p.w);
            }
            const int n = n0 + ((int)rank << log2_own) + c;
            uint16_t* const to = out + (size_t)(row0 + r) * N + n;
            if (N % 4 == 0) {
                const uint2 w = {pack2<DT>(__float_as_uint(v[0]), __float_as_uint(v[1])),
                                 pack2<DT>(__float_as_uint(v[2]), __float_as_uint(v[3]))};
                if (n < N) *reinterpret_cast<uint2*>(to) = w;
            } else {
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (n + x < N) to[x] = round16<DT>(v[x]);
            }
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, Cfg::kTmem);
    }
}

// ------------------------------------------------------------------ host side
static int pairs_for(int64_t tiles, int dev) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(tiles, device_sm_count(dev) / 2));
}

// The tensor maps of one call: b's rows and scales by group, a's scales; those of a's rows are the kernels'.
struct Operands {
    const void *a, *a_scales, *b, *b_scales;
    int groups, rows, n, k;
    int map_w(CUtensorMap* m) const {
        const uint64_t extent[3] = {(uint64_t)k / 2, (uint64_t)n, (uint64_t)groups};
        const uint32_t box[3] = {128, 128, 1};
        return gemm::encode_tiled(m, b, 1, 3, extent, box, CU_TENSOR_MAP_SWIZZLE_128B);
    }
    int map_w_scales(CUtensorMap* m) const {
        const uint64_t extent[3] = {(uint64_t)scale_pitch(k), (uint64_t)n, (uint64_t)groups};
        const uint32_t box[3] = {16, 128, 1};
        return gemm::encode_tiled(m, b_scales, 1, 3, extent, box, CU_TENSOR_MAP_SWIZZLE_NONE);
    }
    int map_x(CUtensorMap* m, uint32_t box_rows) const {
        const uint64_t extent[2] = {(uint64_t)k / 2, (uint64_t)rows};
        const uint32_t box[2] = {128, box_rows};
        return gemm::encode_tiled(m, a, 1, 2, extent, box, CU_TENSOR_MAP_SWIZZLE_128B);
    }
    int map_x_scales(CUtensorMap* m, uint32_t box_rows) const {
        const uint64_t extent[2] = {(uint64_t)scale_pitch(k), (uint64_t)rows};
        const uint32_t box[2] = {16, box_rows};
        return gemm::encode_tiled(m, a_scales, 1, 2, extent, box, CU_TENSOR_MAP_SWIZZLE_NONE);
    }
    // The most tiles of `tile_rows` rows and `tile_n` columns that there can be.
    int64_t tiles(int tile_rows, int tile_n, bool grouped) const {
        const int64_t chunks = grouped ? (int64_t)rows / tile_rows + std::min(groups, rows)
                                       : ((int64_t)rows + tile_rows - 1) / tile_rows;
        return chunks * ((n + tile_n - 1) / tile_n);
    }
};

template <int DT, int R>
static int launch_split(const Operands& op, const int* offsets, void* out, int log2_cl, int dev, cudaStream_t stream) {
    static bool attr_set[64] = {};
    CUtensorMap tmW, tmX, tmWS, tmXS;
    int rc = op.map_w(&tmW);
    if (rc == TRB_OK) rc = op.map_x(&tmX, R);
    if (rc == TRB_OK) rc = op.map_w_scales(&tmWS);
    if (rc == TRB_OK) rc = op.map_x_scales(&tmXS, R);
    if (rc != TRB_OK) return rc;
    return launch_kernel(gemm_fp4_split_kernel<DT, R>, (int)op.tiles(R, kSplitN, offsets != nullptr) << log2_cl, kSplitThreads,
                         1 << log2_cl, SplitCfg<R>::kSmem, dev, attr_set, stream, tmW, tmX, tmWS, tmXS, offsets,
                         static_cast<uint16_t*>(out), op.groups, op.rows, op.n, op.k, log2_cl);
}

template <int DT>
static int launch_product(const Operands& op, const int* offsets, void* out, int dev, cudaStream_t stream) {
    const bool grouped = offsets != nullptr;
    const int num_stages = (op.k + kStageK - 1) / kStageK;
    const int64_t num_n = (op.n + kSplitN - 1) / kSplitN, active = std::min(op.groups, op.rows);
    // Single CTAs with K split over clusters as far as every cluster has a place at once (16 rows, 4096 x 4096: 5.5 us
    // in clusters of 4, 6.1 of 8, of which 30 have places, and the pairs' 9.0).  Few rows take tiles of 16 of them, two CTAs
    // an SM, more take tiles of 64 (17 rows as above: 5.9 us, with tiles of 16 6.1; 128 rows: 7.2, the pairs 9.7).  How the
    // rows are dealt out to the groups is not known here: up to 8 a group on average count as one tile of 16 each, and are
    // worth it even without places for all (16 groups of 8 rows, 4096 x 2048: 19.6 us, the pairs 22.3; of 16 rows 24.8 and
    // 20.6); up to 32 count as one tile of 64 (8 groups of 24 rows, 2048 x 2048: 8.6 us, the pairs 9.6; of 48 11.9 and 9.5).
    const bool few = grouped ? op.rows <= 8 * active : op.rows <= 16;
    if (few || !grouped || op.rows <= 32 * active) {
        const int64_t tiles = num_n * (grouped ? active : ((int64_t)op.rows + 63) / 64);
        const auto fits = [&](int log2_cl) {
            static int places[4][64] = {};
            const int at_once = clusters_at_once(gemm_fp4_split_kernel<DT, 64>, kSplitThreads, SplitCfg<64>::kSmem,
                                                 1 << log2_cl, dev, places[log2_cl]);
            return tiles <= (few ? SplitCfg<16>::kPerSm : SplitCfg<64>::kPerSm) * at_once;
        };
        int log2_cl = -1;
        while (log2_cl < 3 && 1 << (log2_cl + 1) <= num_stages && fits(log2_cl + 1)) ++log2_cl;
        if (few && grouped && log2_cl < 0) log2_cl = 0;
        if (log2_cl >= 0 && op.tiles(few ? 16 : 64, kSplitN, grouped) << log2_cl <= INT32_MAX)
            return few ? launch_split<DT, 16>(op, offsets, out, log2_cl, dev, stream)
                       : launch_split<DT, 64>(op, offsets, out, log2_cl, dev, stream);
    }
    static bool attr_set[64] = {};
    CUtensorMap tmW, tmX128, tmX64, tmX32, tmWS, tmXS;
    int rc = op.map_w(&tmW);
    if (rc == TRB_OK) rc = op.map_x(&tmX128, 128);
    if (rc == TRB_OK) rc = op.map_x(&tmX64, 64);
    if (rc == TRB_OK) rc = op.map_x(&tmX32, 32);
    if (rc == TRB_OK) rc = op.map_w_scales(&tmWS);
    if (rc == TRB_OK) rc = op.map_x_scales(&tmXS, 128);
    if (rc != TRB_OK) return rc;
    const int64_t tiles = op.tiles(kTileRows, kTileN, grouped);
    if (tiles > INT32_MAX - 1024) {  // a pair steps past the last tile
        set_error("trb_gemm_fp4_launch: too many tiles (rows=%d n=%d groups=%d)", op.rows, op.n, op.groups);
        return TRB_SKIPPED;
    }
    return launch_kernel(gemm_fp4_kernel<DT>, 2 * pairs_for(tiles, dev), kProductThreads, 0, kProductSmem, dev, attr_set,
                         stream, tmW, tmX128, tmX64, tmX32, tmWS, tmXS, offsets, static_cast<uint16_t*>(out), op.groups,
                         op.rows, op.n, op.k);
}

int read_product_error(bool clear) {
    int v = 0;
    TRB_CUDA(cudaMemcpyFromSymbol(&v, g_fp4_gemm_error, sizeof(int)));
    if (clear) {
        const int zero = 0;
        TRB_CUDA(cudaMemcpyToSymbol(g_fp4_gemm_error, &zero, sizeof(int)));
    }
    return v;
}

}  // namespace fp4
}  // namespace trb

extern "C" int trb_gemm_fp4_launch(int dtype, int groups, int rows, int n, int k, const void* a, const void* a_scales,
                                   const void* b, const void* b_scales, const int32_t* offsets, void* out, void* stream) {
    using namespace trb;
    const char* const what = "trb_gemm_fp4_launch";
    clear_error();
    if (groups <= 0 || rows < 0 || n <= 0 || k <= 0) {
        set_error("%s: sizes must be positive (rows may be 0)", what);
        return TRB_ERR_ARGS;
    }
    if (groups > 1 && offsets == nullptr) {
        set_error("%s: several groups need offsets", what);
        return TRB_ERR_ARGS;
    }
    if (dtype != TRB_BFLOAT16 && dtype != TRB_FLOAT16) {
        set_error("%s: unsupported dtype %s (bfloat16 and float16)", what, dtype_name(dtype));
        return TRB_SKIPPED;
    }
    if (groups > kMaxGroups) {
        set_error("%s: at most %d groups (got %d)", what, kMaxGroups, groups);
        return TRB_SKIPPED;
    }
    if (std::max(rows, n) > kMaxExtent || k > fp4::kMaxK) {
        set_error("%s: rows and n at most %d, k at most %d (rows=%d n=%d k=%d)", what, kMaxExtent, fp4::kMaxK, rows, n, k);
        return TRB_SKIPPED;
    }
    if (k % fp4::kBlock != 0) {
        set_error("%s: k must be a multiple of %d (k=%d)", what, fp4::kBlock, k);
        return TRB_ERR_ALIGN;
    }
    if (rows == 0) return TRB_OK;
    if (a == nullptr || a_scales == nullptr || b == nullptr || b_scales == nullptr || out == nullptr) {
        set_error("%s: pointers must be non-null", what);
        return TRB_ERR_ARGS;
    }
    const auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    if ((bits(a) | bits(a_scales) | bits(b) | bits(b_scales) | bits(out)) % 16 != 0 || bits(offsets) % 4 != 0) {
        set_error("%s: matrices must be 16-byte aligned and offsets 4-byte aligned", what);
        return TRB_ERR_ALIGN;
    }
    const uint64_t codes = (uint64_t)k / 2, pitch = (uint64_t)fp4::scale_pitch(k);
    const int rc = check_apart(what, {{out, 2, (uint64_t)rows, (uint64_t)n}},
                               {{a, 1, (uint64_t)rows, codes},
                                {a_scales, 1, (uint64_t)rows, pitch},
                                {b, 1, (uint64_t)n, codes, (uint64_t)groups},
                                {b_scales, 1, (uint64_t)n, pitch, (uint64_t)groups},
                                {offsets, 4, (uint64_t)groups + 1}});
    if (rc != TRB_OK) return rc;
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const fp4::Operands op = {a, a_scales, b, b_scales, groups, rows, n, k};
    return dtype == TRB_BFLOAT16 ? fp4::launch_product<TRB_BFLOAT16>(op, offsets, out, dev, s)
                                 : fp4::launch_product<TRB_FLOAT16>(op, offsets, out, dev, s);
}
