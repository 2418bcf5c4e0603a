// gemv_w4.cu -- few rows times matrices of 4-bit weights with a scale per group of k.
//
//   out[r, n] = sum over groups g of k:  s[e, n, g] * sum over k in g of x[r, k] * (q[e, n, k] - z[e, n, g])
//
// for the rows r of expert e (one expert: a plain matrix).  q is stored two to
// a byte along k, the low four bits first.
//
// The bytes of q are its floor: 1/2 byte per weight, read once for the rows of
// x taken at once (up to 8 or 16, as far as they fit).  The products run on
// mma.sync m16n8k16, 16 outputs x 8 rows of x per instruction -- at one row
// the tensor pipe still does with one instruction per 256 weights what would
// take 256 FMA lanes, and the exact products of small whole numbers with
// 16-bit x accumulate in fp32.  Weights become 16-bit floats by bit
// operations: a 4-bit q ORed into the mantissa of 128 is 128 + q exactly, and
// subtracting 128 + z is exact too, so nothing is rounded before the product,
// and the scale is applied in fp32 to each group's sum.
//
// The order of k inside a product is free as long as q and x agree on it, so
// each of the four threads that share an output takes W consecutive words (8
// q each) straight from global memory into registers: no shared memory, no
// barrier between the loads and the products.  One step is 4 W words of an
// output, 32 W k, with W = 1, 2 or 4 so that a group of 32, 64 or 128 (or
// more) k covers whole steps; a pack of 512 k is 16 / W steps and 32 registers,
// and each step's registers take the same step of the next pack as soon as
// they are used, 64 KiB in flight on an SM.
//
// A CTA takes rows of 16 outputs of one group in jobs.  The packs of a job are
// one sequence, cut evenly among the 16 warps, so a warp works through
// neighbouring packs of one or two rows whatever k is, with nothing to wait for
// but its own loads.  What a warp has summed of a row goes to shared memory
// when it leaves the row, and at the job's end the parts of each row are added
// in the order of k.
//
// Measured (CUDA graph of calls on three sets of inputs): one row, 4096 x 4096,
// 4.9 us, launch and latency; one row, 16384 x 8192, zero points, groups of 64,
// 22.3 us, 3.3 TB/s; 40 rows of 22 experts, 2048 x 4096, 27.4 us, 3.6 TB/s; 15
// rows, 11009 x 4096, groups of 32, 17.9 us.  A copy that moves as many bytes
// takes 3.2, 13.3, 16.6 and 6.0 us.  What bounds the middle two is not known:
// they issue in 50% of the cycles, 42 instructions per 512 weights, half of
// them the conversion; with the conversion and the products taken out they ran
// 20 and 26 us; 12, 16 and 20 warps take the same; and it matters little
// whether the words come from L2 or from memory (8 rows of 5 experts, 4096 x
// 4096: 16.2 and 17.4 us).  Tried and slower: the words through TMA rings (a
// warp's own, 22 and 33 us, or a producer warp's, 26 and 35), through cp.async
// (26 and 32), asked into L2 packs ahead (25 and 35), 24 warps a CTA (29 and
// 31), k shared by clusters of 4 CTAs (45 us for the 15 rows), packs dealt to
// the warps in turn, so that an SM reads runs of whole rows.  14 of the 40
// variants spill 4 to 20 bytes at 128 registers.
//
// No counterpart in the reference.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "trb_common.cuh"
#include "trb_groups.cuh"

namespace trb {
namespace w4 {

__device__ int g_w4_error;

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;      // outputs of a row of a job
constexpr int kPackK = 512;    // k of a pack
constexpr int kJobRows = 32;   // rows of 16 outputs in a job, at most

struct Shape {
    int groups, rows, n, k;
    int k_groups;    // scales per output
    int group_log2;
    int tokens;      // rows of x taken at once
};

// d (+)= a * b on the tensor cores, 16 outputs x 8 rows of x x 16 k; `first` starts from zero.
#define TRB_MMA_16816(TYPE, C0, C1, C2, C3)                                                                 \
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, " \
                 "{%8, %9}, {%10, %11, %12, %13};"                                                          \
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                           \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(C0), "f"(C1), "f"(C2), "f"(C3))
template <int DT>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
    if constexpr (DT == TRB_BFLOAT16) {
        if (first) TRB_MMA_16816("bf16", 0.f, 0.f, 0.f, 0.f);
        else TRB_MMA_16816("bf16", d[0], d[1], d[2], d[3]);
    } else {
        if (first) TRB_MMA_16816("f16", 0.f, 0.f, 0.f, 0.f);
        else TRB_MMA_16816("f16", d[0], d[1], d[2], d[3]);
    }
}
#undef TRB_MMA_16816

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
// W words of q.  A step of W = 1 takes half a 32-byte sector of each output, the next step the other half, which
// stays in L1 for it; wider steps use whole sectors once.
// Predicated in place: as a branch around the load, every word was copied once more.
template <int W>
__device__ __forceinline__ void load_words(const uint8_t* p, int in, uint32_t (&v)[W]) {
    if constexpr (W == 4)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %5, 0;\n\t"
            "@p ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
            : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3])
            : "l"(p), "r"(in));
    else if constexpr (W == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %3, 0;\n\t"
            "@p ld.global.nc.L1::no_allocate.L2::256B.v2.u32 {%0, %1}, [%2];\n\t}"
            : "+r"(v[0]), "+r"(v[1])
            : "l"(p), "r"(in));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\t"
            "@p ld.global.nc.L2::256B.u32 %0, [%1];\n\t}"
            : "+r"(v[0])
            : "l"(p), "r"(in));
}

// Pair p of a word of eight q: (q[p], q[p + 4]) as two 16-bit floats.  bf16: 128 + q each.  f16 has mantissa bits
// enough to take q where it stands in the word or its upper half: 1024 + q for even p, 64 + q for odd p.
// One lop3 for the mask and the exponent together (written as & and |, it became two).
__device__ __forceinline__ uint32_t mask_or(uint32_t v, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));
    return r;
}
template <int DT>
__device__ __forceinline__ void biased_pairs(uint32_t w, uint32_t (&pair)[4]) {
    if constexpr (DT == TRB_BFLOAT16) {
#pragma unroll
        for (int p = 0; p < 4; ++p) pair[p] = mask_or(w >> (4 * p), 0x000F000Fu, 0x43004300u);
    } else {
        pair[0] = mask_or(w, 0x000F000Fu, 0x64006400u);
        pair[1] = mask_or(w, 0x00F000F0u, 0x54005400u);
        pair[2] = mask_or(w >> 8, 0x000F000Fu, 0x64006400u);
        pair[3] = mask_or(w >> 8, 0x00F000F0u, 0x54005400u);
    }
}
// Byte i of four zero points as two equal 16-bit floats with the same bias, for even and odd pairs.
template <int DT>
__device__ __forceinline__ void biased_zeros(uint32_t bytes, int i, uint32_t& even, uint32_t& odd) {
    const uint32_t twice = 0x4040u + 0x0101u * (uint32_t)i;
    if constexpr (DT == TRB_BFLOAT16) {
        even = odd = __byte_perm(bytes, 0x43u, twice);
    } else {
        even = __byte_perm(bytes, 0x64u, twice);
        odd = __byte_perm(bytes << 4, 0x54u, twice);
    }
}
template <int DT>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    if constexpr (DT == TRB_BFLOAT16) {
        __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    } else {
        __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    }
}
template <int DT>
__device__ __forceinline__ float scale_of(uint32_t pair, int i) {  // the lower or upper 16 bits
    if constexpr (DT == TRB_BFLOAT16) return __uint_as_float(i ? pair & 0xFFFF0000u : pair << 16);
    else return __half2float(__ushort_as_half((unsigned short)(i ? pair >> 16 : pair & 0xFFFFu)));
}
template <int DT>
__device__ __forceinline__ uint16_t round16(float v) {
    if constexpr (DT == TRB_BFLOAT16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
    else return __half_as_ushort(__float2half_rn(v));
}

// Rows of 16 outputs [row, row + rows) of group e for the rows of x in chunk q, and a warp's share of their packs:
// `left` packs from pack `pack` of row `p_row` on.
struct Job {
    int first;  // in the count of all rows of outputs of all chunks
    int rows, row, q, e;
    int p_row, pack, left;
};

// NT * 8 rows of x at once; W: words of a step; Z: zero points given; V: a thread's scales of a pack are one aligned
// read.
template <int DT, int NT, int W, bool Z, bool V>
__global__ void __launch_bounds__(kThreads, 1)
    gemv_w4_kernel(const uint8_t* weights, const uint16_t* x, const uint16_t* scales, const uint8_t* zeros,
                   const int* offsets, uint16_t* out, const Shape sh) {
    constexpr int kSteps = 16 / W;      // of a pack
    constexpr int kStepK = 32 * W;
    constexpr int kHeld = kSteps / 4;   // steps of a pack whose scale a thread holds for the four of an output
    constexpr int kScaleWords = (kHeld + 1) / 2;

    extern __shared__ __align__(16) uint8_t smem[];

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int num_pack = (sh.k + kPackK - 1) / kPackK;
    const int rows_n = (sh.n + kRows - 1) / kRows;

    // x, the parts of the sums, the groups
    float* red = reinterpret_cast<float*>(smem + (size_t)num_pack * (kPackK * 2) * sh.tokens);
    const int part = sh.tokens * kRows;  // one warp's sums of a row
    int* words = reinterpret_cast<int*>(red + (kWarps + kJobRows) * part);
    const GroupTable table = {words, words + sh.groups, words + 2 * sh.groups};

    // No operand is read before the wait: the plain pointers (no __restrict__, no read-only loads but the volatile
    // ones) keep the compiler from moving a load up over it.
    grid_launch_dependents();
    grid_dependency_wait();
    int groups = sh.groups;
    if (offsets != nullptr) {
        groups = load_groups(offsets, sh.groups, sh.rows, table, &g_w4_error);
        if (warp == 0) scan_chunks(groups, sh.tokens, table, lane);
    } else if (threadIdx.x == 0) {
        table.start[0] = 0;
        table.rows[0] = sh.rows;
        table.chunk0[0] = 0;
        table.chunk0[1] = (sh.rows + sh.tokens - 1) / sh.tokens;
    }
    __syncthreads();

    // This CTA's share of the rows of outputs, contiguous so that x stays in shared memory.
    const int64_t total = (int64_t)table.chunk0[groups] * rows_n;
    const int end = (int)(total * (blockIdx.x + 1) / gridDim.x);
    auto first_pack = [&](int rows, int w) { return rows * num_pack * w / kWarps; };
    auto job_at = [&](int first) {
        Job j = {};
        j.first = first;
        if (first >= end) return j;
        j.q = first / rows_n;
        j.row = first - j.q * rows_n;
        j.rows = min(min(end - first, rows_n - j.row), kJobRows);
        j.e = group_of_chunk(j.q, groups, table);
        const int p = first_pack(j.rows, warp);
        j.left = first_pack(j.rows, warp + 1) - p;
        j.p_row = p / num_pack;
        j.pack = p - j.p_row * num_pack;
        return j;
    };

    uint32_t lo[kSteps][W], hi[kSteps][W];  // q of outputs g and g + 8
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int w = 0; w < W; ++w) lo[i][w] = hi[i][w] = 0;
    uint32_t sc_next[2][kScaleWords], zr_next[2];
    // The pack to load next: this thread's first word for outputs g and g + 8, and its steps.  Outputs past n are
    // computed from the last one and not stored; steps past k keep old words and meet zeros in x.
    const uint8_t *q_lo = weights, *q_hi = weights;
    int steps = 0;
    auto at_pack = [&](int e, int row, int pack) {
        const size_t first = (size_t)e * sh.n;
        const int r_lo = min(row * kRows + g, sh.n - 1), r_hi = min(row * kRows + 8 + g, sh.n - 1);
        const int byte = pack * (kPackK / 2) + t * 4 * W;
        q_lo = weights + (first + r_lo) * (size_t)(sh.k / 2) + byte;
        q_hi = weights + (first + r_hi) * (size_t)(sh.k / 2) + byte;
        steps = min(kSteps, (sh.k - pack * kPackK) / kStepK);
        const int step = pack * kSteps + t * kHeld;
        const int kg = W == 4 ? (step * kStepK) >> sh.group_log2 : step;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const size_t at = (first + (i ? r_hi : r_lo)) * sh.k_groups + kg;
            const bool in = kg < sh.k_groups;
            if constexpr (kHeld == 1) {
                sc_next[i][0] = in ? scales[at] : 0;
                if constexpr (Z) zr_next[i] = in ? zeros[at] : 0;
            } else if constexpr (V && kHeld == 4) {  // k_groups is a multiple of kHeld
                const uint2 v = in ? *reinterpret_cast<const uint2*>(scales + at) : make_uint2(0, 0);
                sc_next[i][0] = v.x;
                sc_next[i][1] = v.y;
                if constexpr (Z) zr_next[i] = in ? *reinterpret_cast<const uint32_t*>(zeros + at) : 0;
            } else if constexpr (V) {
                sc_next[i][0] = in ? *reinterpret_cast<const uint32_t*>(scales + at) : 0;
                if constexpr (Z) zr_next[i] = in ? *reinterpret_cast<const uint16_t*>(zeros + at) : 0;
            } else {
                if constexpr (Z) zr_next[i] = 0;
#pragma unroll
                for (int j = 0; j < kHeld; ++j) {
                    const bool in_j = kg + j < sh.k_groups;
                    const uint32_t v = (uint32_t)(in_j ? scales[at + j] : 0) << (16 * (j & 1));
                    sc_next[i][j >> 1] = j & 1 ? sc_next[i][j >> 1] | v : v;
                    if constexpr (Z) zr_next[i] |= (uint32_t)(in_j ? zeros[at + j] : 0) << (8 * j);
                }
            }
        }
    };
    auto load_step = [&](int i) {
        load_words<W>(q_lo + i * 16 * W, i < steps, lo[i]);
        load_words<W>(q_hi + i * 16 * W, i < steps, hi[i]);
    };
    auto begin = [&](const Job& j) {  // a job's first pack
        if (j.left == 0) return;
        at_pack(j.e, j.row + j.p_row, j.pack);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) load_step(i);
    };

    Job job = job_at((int)(total * blockIdx.x / gridDim.x));
    begin(job);
    int chunk = -1, tokens = 0, row0 = 0;
    while (job.first < end) {
        if (job.q != chunk) {  // other rows of x: in shared memory, [step][word of a thread][row][t]: 8 values in the
            chunk = job.q;     // order the pairs of a word of q come in, zeros past k
            const int first = (chunk - table.chunk0[job.e]) * sh.tokens;
            row0 = table.start[job.e] + first;
            tokens = min(sh.tokens, table.rows[job.e] - first);
            uint4* x_out = reinterpret_cast<uint4*>(smem);
            for (int j = threadIdx.x; j < num_pack * (kPackK / 8); j += kThreads) {
                const bool in = j * 8 < sh.k;
                const uint4* src = reinterpret_cast<const uint4*>(x + (size_t)row0 * sh.k) + j;
                const int step = j / (4 * W), of = j / W % 4, w = j % W;
                uint4* dst = x_out + (step * W + w) * tokens * 4 + of;
#pragma unroll 8
                for (int c = 0; c < tokens; ++c) {
                    const uint4 v = in ? src[(size_t)c * (sh.k / 8)] : make_uint4(0, 0, 0, 0);
                    dst[c * 4] = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                                            __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
                }
            }
            __syncthreads();
        }
        // Columns of the products past the last row of x are computed from that row and not used.
        const uint32_t x_block = (uint32_t)tokens * 64;
        uint32_t x_lane[NT];
#pragma unroll
        for (int c = 0; c < NT; ++c) x_lane[c] = smem_u32(smem) + (uint32_t)(min(c * 8 + g, tokens - 1) * 64 + t * 16);

        float sum[NT][4];
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[c][i] = 0.0f;
        int row = job.p_row, pack = job.pack;
        for (int left = job.left; left > 0;) {
            uint32_t sc[2][kScaleWords], zr[2] = {};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int j = 0; j < kScaleWords; ++j) sc[i][j] = sc_next[i][j];
                if constexpr (Z) zr[i] = zr_next[i] & 0x0F0F0F0Fu;
            }
            uint32_t x_at[NT];
#pragma unroll
            for (int c = 0; c < NT; ++c) x_at[c] = x_lane[c] + (uint32_t)(pack * 16) * x_block;
            --left;
            const bool row_done = ++pack == num_pack;
            if (row_done) pack = 0;
            steps = 0;
            if (left > 0) at_pack(job.e, job.row + row + row_done, pack);

            uint32_t pair[2], zw[2];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int held = i % kHeld;
                uint32_t even[2], odd[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (held % 2 == 0) pair[h] = __shfl_sync(0xffffffffu, sc[h][held >> 1], i / kHeld, 4);
                    if constexpr (Z) {
                        if (held == 0) zw[h] = __shfl_sync(0xffffffffu, zr[h], i / kHeld, 4);
                        biased_zeros<DT>(zw[h], held, even[h], odd[h]);
                    } else {
                        biased_zeros<DT>(8u, 0, even[h], odd[h]);
                    }
                }
                float acc[NT][4];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    uint4 xv[NT];
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        xv[c] = lds128(x_at[c]);
                        x_at[c] += x_block;
                    }
                    uint32_t lo_pairs[4], hi_pairs[4];
                    biased_pairs<DT>(lo[i][w], lo_pairs);
                    biased_pairs<DT>(hi[i][w], hi_pairs);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t a[4] = {sub2<DT>(lo_pairs[2 * h], even[0]), sub2<DT>(hi_pairs[2 * h], even[1]),
                                               sub2<DT>(lo_pairs[2 * h + 1], odd[0]),
                                               sub2<DT>(hi_pairs[2 * h + 1], odd[1])};
#pragma unroll
                        for (int c = 0; c < NT; ++c)
                            mma_16816<DT>(acc[c], a, h ? xv[c].z : xv[c].x, h ? xv[c].w : xv[c].y, w == 0 && h == 0);
                    }
                }
                load_step(i);
                const float s_lo = scale_of<DT>(pair[0], held & 1), s_hi = scale_of<DT>(pair[1], held & 1);
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[c][j] = fmaf(j < 2 ? s_lo : s_hi, acc[c][j], sum[c][j]);
            }
            if (row_done || left == 0) {  // this warp is done with the row
                // (warp, row) pairs of a job go up one at a time, so their sums are places of their own
                float* mine = red + (warp + row) * part;
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int token = c * 8 + 2 * t + (i & 1);
                        if (token < tokens) mine[token * kRows + (i >> 1) * 8 + g] = sum[c][i];
                        sum[c][i] = 0.0f;
                    }
                ++row;
            }
        }

        const Job next = job_at(job.first + job.rows);
        begin(next);
        __syncthreads();
        const int packs = job.rows * num_pack;
        for (int i = threadIdx.x; i < job.rows * tokens * kRows; i += kThreads) {
            const int in_row = i % (tokens * kRows), r = i / (tokens * kRows);
            const int token = in_row / kRows, n = (job.row + r) * kRows + in_row % kRows;
            // warp w has pack p when packs * w / 16 <= p < packs * (w + 1) / 16 (whole quotients)
            const int w0 = (kWarps * (r * num_pack + 1) - 1) / packs, w1 = (kWarps * (r + 1) * num_pack - 1) / packs;
            float v = 0.0f;
            for (int w = w0; w <= w1; ++w)
                if (first_pack(job.rows, w) < first_pack(job.rows, w + 1)) v += red[(w + r) * part + in_row];
            if (n < sh.n) out[(size_t)(row0 + token) * sh.n + n] = round16<DT>(v);
        }
        __syncthreads();
        job = next;
    }
}

// ------------------------------------------------------------------ host side
constexpr size_t kMaxX = 128 * 1024;  // of x in shared memory
static size_t x_row_bytes(int k) { return (size_t)(k + kPackK - 1) / kPackK * kPackK * 2; }

struct Operands {
    const void *x, *q, *scales, *zeros;
    const int* offsets;
    void* out;
};

template <int DT, int NT, int W, bool Z, bool V>
static int launch_kernel(const Operands& op, Shape sh, int dev, cudaStream_t stream) {
    static bool attr_set[64] = {};
    constexpr size_t kMaxSmem = 226 * 1024;
    if (dev >= 64 || !attr_set[dev]) {
        TRB_CUDA(cudaFuncSetAttribute(gemv_w4_kernel<DT, NT, W, Z, V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)kMaxSmem));
        if (dev < 64) attr_set[dev] = true;
    }
    const size_t row_bytes = x_row_bytes(sh.k);
    sh.tokens = std::min({sh.rows, NT * 8, (int)(kMaxX / row_bytes)});
    const size_t smem = row_bytes * sh.tokens + (size_t)(kWarps + kJobRows) * sh.tokens * kRows * 4 +
                        (size_t)(3 * sh.groups + 1) * 4;
    const int64_t rows_n = (sh.n + kRows - 1) / kRows;
    const int64_t tiles = rows_n * ((int64_t)sh.rows / sh.tokens + std::min(sh.groups, sh.rows));
    if (tiles > INT32_MAX) {
        set_error("trb_gemv_w4_launch: too many outputs (rows=%d n=%d groups=%d)", sh.rows, sh.n, sh.groups);
        return TRB_SKIPPED;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(tiles, device_sm_count(dev)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    TRB_CUDA(cudaLaunchKernelEx(&cfg, gemv_w4_kernel<DT, NT, W, Z, V>, static_cast<const uint8_t*>(op.q),
                                static_cast<const uint16_t*>(op.x), static_cast<const uint16_t*>(op.scales),
                                static_cast<const uint8_t*>(op.zeros), op.offsets, static_cast<uint16_t*>(op.out), sh));
    return TRB_OK;
}

template <int DT, int NT, bool Z>
static int launch_group(const Operands& op, const Shape& sh, int dev, cudaStream_t stream) {
    auto vector = [&](int held) {
        return sh.k_groups % held == 0 && reinterpret_cast<uintptr_t>(op.scales) % (2 * held) == 0 &&
               reinterpret_cast<uintptr_t>(op.zeros) % held == 0;
    };
    switch (sh.group_log2) {
        case 5:
            return vector(4) ? launch_kernel<DT, NT, 1, Z, true>(op, sh, dev, stream)
                             : launch_kernel<DT, NT, 1, Z, false>(op, sh, dev, stream);
        case 6:
            return vector(2) ? launch_kernel<DT, NT, 2, Z, true>(op, sh, dev, stream)
                             : launch_kernel<DT, NT, 2, Z, false>(op, sh, dev, stream);
        default: return launch_kernel<DT, NT, 4, Z, false>(op, sh, dev, stream);
    }
}

template <int DT>
static int launch(const Operands& op, const Shape& sh, int dev, cudaStream_t stream) {
    // 16 rows at once where that takes fewer passes over the weights than 8, on average rows a group: 15 rows of one
    // 11009 x 4096 matrix in groups of 32, 18.5 against 22.5 us.  Less than 16 rows of a long k fit: 16 rows of 16384 x
    // 6144 in groups of 128 take two passes either way, 33.6 us as 10 and 6 rows and 26.7 as 8 and 8, 9 rows 21.4 as one
    // pass and 26.5 as two.
    const int64_t rows = (sh.rows + (int64_t)sh.groups - 1) / sh.groups;
    const auto passes = [&](int64_t at_once) {
        const int64_t taken = std::min<int64_t>(at_once, kMaxX / x_row_bytes(sh.k));
        return (rows + taken - 1) / taken;
    };
    if (passes(16) < passes(8))
        return op.zeros ? launch_group<DT, 2, true>(op, sh, dev, stream) : launch_group<DT, 2, false>(op, sh, dev, stream);
    return op.zeros ? launch_group<DT, 1, true>(op, sh, dev, stream) : launch_group<DT, 1, false>(op, sh, dev, stream);
}

int read_error(bool clear) {
    int v = 0;
    TRB_CUDA(cudaMemcpyFromSymbol(&v, g_w4_error, sizeof(int)));
    if (clear) {
        const int zero = 0;
        TRB_CUDA(cudaMemcpyToSymbol(g_w4_error, &zero, sizeof(int)));
    }
    return v;
}

}  // namespace w4
}  // namespace trb

extern "C" int trb_gemv_w4_launch(int dtype, int groups, int rows, int n, int k, int group_size, const void* x,
                                  const void* q, const void* scales, const void* zeros, const int32_t* offsets,
                                  void* out, void* stream) {
    using namespace trb;
    clear_error();
    if (groups <= 0 || rows < 0 || n <= 0 || k <= 0 || q == nullptr || scales == nullptr ||
        (rows > 0 && (x == nullptr || out == nullptr)) || (offsets == nullptr && groups != 1)) {
        set_error("trb_gemv_w4_launch: sizes must be positive (rows may be 0), pointers non-null, and several groups "
                  "need offsets");
        return TRB_ERR_ARGS;
    }
    if (dtype != TRB_BFLOAT16 && dtype != TRB_FLOAT16) {
        set_error("trb_gemv_w4_launch: unsupported dtype %s (bfloat16 and float16)", dtype_name(dtype));
        return TRB_SKIPPED;
    }
    if (group_size < 32 || (group_size & (group_size - 1)) != 0 || k % group_size != 0) {
        set_error("trb_gemv_w4_launch: the group size must be a power of two of at least 32 that divides k (group size "
                  "%d, k %d)", group_size, k);
        return TRB_SKIPPED;
    }
    if (k > 65536 || groups > kMaxGroups) {
        set_error("trb_gemv_w4_launch: k at most 65536 and at most %d groups (k=%d groups=%d)", kMaxGroups, k, groups);
        return TRB_SKIPPED;
    }
    if (std::max(rows, n) > kMaxExtent) {
        set_error("trb_gemv_w4_launch: rows and n at most %d (rows=%d n=%d)", kMaxExtent, rows, n);
        return TRB_SKIPPED;
    }
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(q)) & 15u) != 0 ||
        ((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(out)) & 1u) != 0 ||
        (reinterpret_cast<uintptr_t>(offsets) & 3u) != 0) {
        set_error("trb_gemv_w4_launch: x and q must be 16-byte aligned, the others as their elements");
        return TRB_ERR_ALIGN;
    }
    if (rows == 0) return TRB_OK;
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    w4::Shape sh = {};
    sh.groups = groups;
    sh.rows = rows;
    sh.n = n;
    sh.k = k;
    sh.k_groups = k / group_size;
    while ((1 << sh.group_log2) < group_size) ++sh.group_log2;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const w4::Operands op = {x, q, scales, zeros, offsets, out};
    return dtype == TRB_BFLOAT16 ? w4::launch<TRB_BFLOAT16>(op, sh, dev, s) : w4::launch<TRB_FLOAT16>(op, sh, dev, s);
}
