// gemm_fp4.cu -- products of microscaled 4-bit floating point, dense or grouped by expert.
//
//   out[r, n] = sum over k of a[r, k] * b[e, n, k]   for the rows r of group e (one group of all rows without offsets)
//
// a and b are stored as trb_fp4.cuh says.  The tensor cores multiply them as they are
// (tcgen05.mma.kind::mxf4.block_scale, 64 k an instruction, a scale every 32), accumulate in fp32 in TMEM, and the
// result is rounded once to bf16 or f16.
//
// No counterpart in the reference.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "trb_common.cuh"
#include "trb_fp4.cuh"
#include "trb_groups.cuh"

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
// chunks next to each other in time).
__device__ __forceinline__ ProductTile product_tile(int t, int groups, int num_n, const GroupTable& g) {
    const int e = group_of_chunk(t / num_n, groups, g);
    const int local = t - g.chunk0[e] * num_n;
    const int rows = g.rows[e];
    const int chunks = (rows + kTileRows - 1) / kTileRows;
    const int run = 8 * num_n;
    const int first = local / run * 8;
    const int width = min(8, chunks - first);
    const int in_run = local - first * num_n;
    const int chunk = first + in_run % width;
    const int per = ((rows + chunks - 1) / chunks + 31) & ~31;
    ProductTile p;
    p.e = e;
    p.row0 = g.start[e] + chunk * per;
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
    groups = load_groups_or_all(offsets, groups, total_rows, table, &g_fp4_gemm_error);
    if (warp == 0) scan_chunks(groups, kTileRows, table, lane);
    __syncthreads();
    const int num_tiles = table.chunk0[groups] * num_n;

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer (both CTAs; completion on the leader's full barriers)
            uint32_t stage = 0, phase = 0;
            uint32_t issued_mask = 0, issued_phase = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
                const ProductTile p = product_tile(tile, groups, num_n, table);
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
                const ProductTile p = product_tile(tile, groups, num_n, table);
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
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint32_t slot = 2 * stage + b;
                        const uint64_t w = w_desc0 + (uint64_t)((slot * kWBlock) >> 4);
                        const uint64_t x = x_desc0 + (uint64_t)((slot * kXBlock) >> 4);
                        const uint32_t scales = tmem_base + (uint32_t)(kTmemScales + (scale_slot + b) * kScaleCols);
#pragma unroll
                        for (int i = 0; i < kBK / 64; ++i) {  // 64 k: 32 bytes of a k-block's 128, half of a scale word
                            if (s * kStageK + b * kBK + i * 64 >= K) break;
                            const uint32_t t = scales + (uint32_t)((i >> 1) * (kScaleCols / 2));
                            if (elected) mma_pair_mxf4(d_tmem, w + (uint64_t)((i * 32) >> 4), x + (uint64_t)((i * 32) >> 4),
                                          (i & 1) ? idesc | kSecondHalf : idesc, t, t + 4,
                                          (s != 0 || b != 0 || i != 0) ? 1u : 0u);
                        }
                        if (elected) tc_commit_pair_multicast(smem_u32(&empty_bar[slot]), 0x3);
                    }
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
            const ProductTile p = product_tile(tile, groups, num_n, table);
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
            const bool second = product_tile(tile, groups, num_n, table).rows > 128;
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
            const ProductTile p = product_tile(tile, groups, num_n, table);
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

// ------------------------------------------------------------------ host side
static int pairs_for(int64_t tiles, int dev) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(tiles, device_sm_count(dev) / 2));
}

template <int DT>
static int launch_product(int groups, int rows, int n, int k, const void* a, const void* a_scales, const void* b,
                          const void* b_scales, const int* offsets, void* out, int dev, cudaStream_t stream) {
    static bool attr_set[64] = {};
    CUtensorMap tmW, tmX128, tmX64, tmX32, tmWS, tmXS;
    const uint64_t we[3] = {(uint64_t)k / 2, (uint64_t)n, (uint64_t)groups}, xe[2] = {(uint64_t)k / 2, (uint64_t)rows};
    const uint32_t wb[3] = {128, 128, 1}, xb128[2] = {128, 128}, xb64[2] = {128, 64}, xb32[2] = {128, 32};
    int rc = gemm::encode_tiled(&tmW, b, 1, 3, we, wb, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmX128, a, 1, 2, xe, xb128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmX64, a, 1, 2, xe, xb64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmX32, a, 1, 2, xe, xb32, CU_TENSOR_MAP_SWIZZLE_128B);
    const uint64_t wse[3] = {(uint64_t)scale_pitch(k), (uint64_t)n, (uint64_t)groups};
    const uint64_t xse[2] = {(uint64_t)scale_pitch(k), (uint64_t)rows};
    const uint32_t scale_box[3] = {16, 128, 1};
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmWS, b_scales, 1, 3, wse, scale_box, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmXS, a_scales, 1, 2, xse, scale_box, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc != TRB_OK) return rc;
    const int64_t num_n = (n + kTileN - 1) / kTileN;
    const int64_t tiles = num_n * ((int64_t)rows / kTileRows + std::min(groups, rows));
    if (tiles > INT32_MAX) {
        set_error("trb_gemm_fp4_launch: too many tiles (rows=%d n=%d groups=%d)", rows, n, groups);
        return TRB_SKIPPED;
    }
    if (dev >= 64 || !attr_set[dev]) {
        TRB_CUDA(cudaFuncSetAttribute(gemm_fp4_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kProductSmem));
        if (dev < 64) attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)(2 * pairs_for(tiles, dev)));
    cfg.blockDim = dim3(kProductThreads);
    cfg.dynamicSmemBytes = kProductSmem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    TRB_CUDA(cudaLaunchKernelEx(&cfg, gemm_fp4_kernel<DT>, tmW, tmX128, tmX64, tmX32, tmWS, tmXS, offsets,
                                static_cast<uint16_t*>(out), groups, rows, n, k));
    return TRB_OK;
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
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == TRB_BFLOAT16
               ? fp4::launch_product<TRB_BFLOAT16>(groups, rows, n, k, a, a_scales, b, b_scales, offsets, out, dev, s)
               : fp4::launch_product<TRB_FLOAT16>(groups, rows, n, k, a, a_scales, b, b_scales, offsets, out, dev, s);
}
