// expert_rows.cu -- rows of tokens to their experts and back, with weights, and the gradients.
//
// A router gives each token J choices of experts.  For the choice j of token t
//   sort      slots[t, j] = the place of (t, j) among all choices sorted by expert, in the order of (t, j) inside an
//             expert; -1 where the choice is no expert of this layer.  offsets[e] = where expert e's places begin
//   dispatch  out[slots[t, j]] = x[t], or w[t, j] * x[t]
//   combine   out[t] = sum over j of w[t, j] * y[slots[t, j]]
//   gradient  of combine: gy[slots[t, j]] = w[t, j] * g[t],  gw[t, j] = <g[t], y[slots[t, j]]>
// and the gradient of dispatch is combine.  offsets and the sorted rows are what the products of trb_groups.cuh take.
//
// What bounds all of it is the rows' bytes (the sort: launch and latency).  Measured in CUDA graphs of calls on several
// sets of inputs, floors at 6551 GB/s, a measured copy: dispatch of 4109 tokens to 8 rows of 2048 bf16 25.2 us (floor
// 23.1), of 16384 to 2 of 4096 62 to 65 (61.5); combine of the same 25.2 (23.2) and 60.7 (61.5); gradient of the same 48
// (43.7) and 116 (102); the sort of 2, 32872 and 131072 choices 2.4, 6.8 and 14.2 us.
//
// No counterpart in the reference.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "trb_common.cuh"
#include "trb_groups.cuh"
#include "trb_launch.cuh"

namespace trb {
namespace rows {

__device__ int g_rows_error;

// ------------------------------------------------------------------ sort
// Counting sort in one launch, by one cluster: no workspace, no atomics, and the order inside an expert is that of the
// choices.  A CTA takes a contiguous part of the choices, a warp a contiguous part of the CTA's, 32 at a time:
// match.any tells each lane which others chose its expert, so each choice's place inside the warp's part is the warp's
// count of its expert so far and the lanes before, and the first of them adds their number to the count.  The counts are
// then summed over the warps before, the CTAs before (distributed shared memory) and the experts before, and added.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortCtas = 16;  // the largest cluster
constexpr int kBatch = 8;  // groups of 32 choices that a warp loads at once

template <typename Id>
__device__ __forceinline__ int expert_of(const Id* ids, int i, int end, int experts) {
    if (i >= end) return -1;
    const Id id = ids[i];
    return id >= 0 && id < (Id)experts ? (int)id : -1;
}

template <typename Id>
__global__ void __launch_bounds__(kSortThreads)
    expert_sort_kernel(const Id* ids, int entries, int experts, int* offsets, int* slots) {
    extern __shared__ int counts[];  // [warps][experts], then the CTA's totals, where its places begin, where the expert's do
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int* const totals = counts + warps * experts;
    int* const begin = totals + experts;
    int* const offset = begin + experts;
    __shared__ int group_total[32];  // at most kMaxGroups experts
    const int ctas = gridDim.x, rank = blockIdx.x;  // the grid is one cluster
    int* const mine = counts + warp * experts;

    for (int i = threadIdx.x; i < warps * experts; i += blockDim.x) counts[i] = 0;
    grid_launch_dependents();
    grid_dependency_wait();
    __syncthreads();

    // Whole groups of 32 to every warp of the cluster, as evenly as they go.
    const int64_t groups = ((int64_t)entries + 31) / 32;
    const int64_t part = (int64_t)rank * warps + warp, parts = (int64_t)ctas * warps;
    const int first = (int)(groups * part / parts * 32);
    const int end = (int)min((int64_t)entries, groups * (part + 1) / parts * 32);
    const bool once = end - first <= 32 * kBatch;  // all of them stay in registers

    int e[kBatch], place[kBatch];
    for (int i = first; i < end; i += 32 * kBatch) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) e[b] = expert_of(ids, i + 32 * b + lane, end, experts);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (i + 32 * b >= end) break;
            const uint32_t same = __match_any_sync(0xffffffffu, e[b]);
            const int before = __popc(same & ((1u << lane) - 1u));
            place[b] = e[b] >= 0 ? mine[e[b]] + before : -1;
            __syncwarp();
            if (e[b] >= 0 && before == 0) mine[e[b]] = place[b] + __popc(same);
            __syncwarp();
        }
        if (!once)
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (i + 32 * b + lane < end) slots[i + 32 * b + lane] = place[b];
    }
    __syncthreads();
    for (int x = threadIdx.x; x < experts; x += blockDim.x) {
        int sum = 0;
#pragma unroll 8
        for (int w = 0; w < warps; ++w) {
            const int c = counts[w * experts + x];
            counts[w * experts + x] = sum;
            sum += c;
        }
        totals[x] = sum;
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
    // begin[x] = what the CTAs before have of expert x, and the experts of its group of 32 before it have in all.
    for (int x0 = warp * 32; x0 < experts; x0 += warps * 32) {
        const int x = x0 + lane;
        int before = 0, all = 0;
        if (x < experts) {
            if (ctas == 1) {
                all = totals[x];
            } else {
                const uint32_t at = smem_u32(totals + x);
                int c[kSortCtas];
#pragma unroll
                for (int r = 0; r < kSortCtas; ++r) {
                    c[r] = 0;
                    if (r < ctas) asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c[r]) : "r"(mapa_shared(at, r)));
                }
#pragma unroll
                for (int r = 0; r < kSortCtas; ++r) {
                    before += r < rank ? c[r] : 0;
                    all += c[r];
                }
            }
        }
        int sum = all;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        if (x < experts) {
            begin[x] = before;
            offset[x] = sum - all;
        }
        if (lane == 31) group_total[x0 >> 5] = sum;
    }
    __syncthreads();
    if (ctas > 1) cluster_arrive();  // the other CTAs' totals have been read
    if (warp == 0) {
        const int groups_of_32 = (experts + 31) >> 5;
        int sum = lane < groups_of_32 ? group_total[lane] : 0;
        const int own = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        group_total[lane] = sum - own;
        if (lane == 31 && rank == 0) offsets[experts] = sum;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < experts; x += blockDim.x) {
        const int at = offset[x] + group_total[x >> 5];
        if (rank == 0) offsets[x] = at;
        begin[x] += at;
    }
    __syncthreads();
    for (int i = first; i < end; i += 32 * kBatch) {
        if (!once) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int at = i + 32 * b + lane;
                e[b] = expert_of(ids, at, end, experts);
                place[b] = at < end ? slots[at] : -1;
            }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int at = i + 32 * b + lane;
            if (at < end) slots[at] = e[b] >= 0 ? begin[e[b]] + mine[e[b]] + place[b] : -1;
        }
    }
    if (ctas > 1) cluster_wait();
}

// ------------------------------------------------------------------ rows there and back
// V values of a row that move together, in one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T round_to(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load(const T* p) {
    return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const Pack<T, V>& v) {
    *reinterpret_cast<Pack<T, V>*>(p) = v;
}

// The row of a slot, or -1 where there is none.  A slot behind the last row is an error of the caller's.  This waits for
// the slot, so slots are read well before they are looked at.
__device__ __forceinline__ int row_of(int s, int rows) {
    if (s >= rows) {
        atomicCAS(&g_rows_error, 0, kErrSlots);
        return -1;
    }
    return s;
}

constexpr int kRowThreads = 256;

// Threads of a CTA: 1 << log2_lanes of them for one token's row, several tokens side by side; blockIdx.y shares a row
// among CTAs where there are few tokens.
struct RowWalk {
    int64_t token, token_step;
    int pack, pack_step;
};
__device__ __forceinline__ RowWalk row_walk(int log2_lanes) {
    RowWalk w;
    const int side = kRowThreads >> log2_lanes;
    w.token = (int64_t)blockIdx.x * side + (threadIdx.x >> log2_lanes);
    w.token_step = (int64_t)gridDim.x * side;
    w.pack = (int)(blockIdx.y << log2_lanes) + (threadIdx.x & ((1 << log2_lanes) - 1));
    w.pack_step = (int)(gridDim.y << log2_lanes);
    return w;
}

// Each row of x is read once, whatever the number of its choices.
template <typename T, typename W, int V, int U>
__global__ void __launch_bounds__(kRowThreads)
    expert_dispatch_kernel(const T* x, const int* slots, const W* weights, T* out, int64_t tokens, int choices, int rows,
                           int width, int log2_lanes) {
    // A slot is looked at as it is read, and then its weight is read.  Rows that begin anywhere lost by reading them ahead: with
    // four slots of single 16-bit values at once one row of 4095 for each of 16384 tokens took 108 us, two of them 126 (here
    // 75 and 103), 8 rows of 2047 for 4109 tokens 40 (42.5); with the weight ahead of the look 8 rows of 2046 36 (31), but 30
    // where weights are given (33).  Aligned rows do not mind.
    grid_launch_dependents();
    grid_dependency_wait();
    const RowWalk w = row_walk(log2_lanes);
    const int packs = width / V;
    for (int64_t t = w.token; t < tokens; t += w.token_step) {
        for (int p = w.pack; p < packs; p += U * w.pack_step) {
            Pack<T, V> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (p + u * w.pack_step < packs) v[u] = load<T, V>(x + t * width + (int64_t)(p + u * w.pack_step) * V);
            for (int j = 0; j < choices; ++j) {
                const int row = row_of(slots[t * choices + j], rows);
                if (row < 0) continue;
                const float f = weights != nullptr ? to_f32(weights[t * choices + j]) : 1.0f;
                T* const to = out + (int64_t)row * width + (int64_t)p * V;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (p + u * w.pack_step >= packs) break;
                    Pack<T, V> o = v[u];
                    if (weights != nullptr)
#pragma unroll
                        for (int i = 0; i < V; ++i) o.v[i] = round_to<T>(f * to_f32(v[u].v[i]));
                    store<T, V>(to + (int64_t)u * w.pack_step * V, o);
                }
            }
        }
    }
}

// Choices whose rows are on their way at the same time, in the gradient.
constexpr int kAtOnce = 4;

// Combine: sums in fp32, in the order of the choices, rounded once.  Loads into registers keep too few bytes in flight, for
// a slot has to be read before its row can be (16384 tokens of 2 rows of 4096 bf16: 119 us).  Here a thread copies its 16
// bytes of J rows to shared memory (cp.async) kDeep - 1 steps before it adds them up; nobody else reads them, so there is no
// barrier.  A lane reads the slot and weight of one of a step's choices a step before the rows are asked for and looks at
// them then, for a check behind the load would wait for it, and shuffles pass them round.  J = 2: 60.7 us three steps deep
// with four CTAs an SM; two, four and six steps 74, 60.7 and 65.8, three CTAs 71, five 67 (four steps), six 78; 64 tokens
// 1.9 us, with six steps 2.6.  J = 4: four steps and three CTAs are 3 to 4% faster where every choice has a row (16384
// tokens of 4 rows of 4096 99 us) and 6% slower where half have none.  Rows through a ring of bulk copies of 4 KB with a
// producer warp took two waits a row and, when slots were still checked at once, 73 us to this ring's 70.
//
// Rows that begin anywhere (kAny) go the same way in the aligned pieces around them: 4109 tokens of 8 rows of 2047 and 2046
// bf16 31 and 30 us, where accesses of 2 and 4 bytes straight to registers took 55 and 82, and of 2046 float32, 4 rows, 32.
template <int J>
struct Ring {
    static constexpr int kDeep = J == 8 ? 2 : 3;
    static constexpr int kCtas = J == 8 ? 3 : 4;  // of an SM
    static constexpr size_t smem(int pieces) { return (size_t)kDeep * J * (kRowThreads / 32) * pieces * 16; }
};

__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// The first `bytes` of the 16, zeros behind them; no more than these are read.
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// A row that begins at any value's place, in the 16-byte pieces that memory has: its values from e0 on stand `shift`
// bytes behind the beginning of the first piece.
template <typename T>
__device__ __forceinline__ int row_shift(const T* rows, int row, int width, int e0) {
    constexpr uint32_t S = sizeof(T);
    return (int)(((uint32_t)reinterpret_cast<uintptr_t>(rows) + S * ((uint32_t)row * (uint32_t)width + (uint32_t)e0)) & 15u);
}
// Copies a piece, which begins with value `first` of its row, as far as it is the row's.  The one that begins before the
// matrix goes value by value.
template <typename T>
__device__ __forceinline__ void copy_piece(uint32_t to, const T* from, int first, int width, const T* rows) {
    constexpr int S = sizeof(T), V = 16 / S;
    if (first + V <= 0 || first >= width) return;
    if (first >= 0 || from >= rows) {
        copy_async(to, from, min(V, width - first) * S);
    } else {
        for (int x = -first; x < V && first + x < width; ++x) {
            if constexpr (S == 2)
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + x * S),
                             "h"(reinterpret_cast<const unsigned short*>(from)[x]) : "memory");
            else
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + x * S),
                             "r"(reinterpret_cast<const uint32_t*>(from)[x]) : "memory");
        }
    }
}
// Four words of shared memory, 128 bytes apart, from any value's place on.
template <int S>
__device__ __forceinline__ void load_words(uint32_t (&words)[4], uint32_t at) {
    const uint32_t even = at & ~3u;
#pragma unroll
    for (int u = 0; u < 4; ++u) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(words[u]) : "r"(even + 128 * u) : "memory");
    if (S == 2 && (at & 2u)) {  // all of the warp or none
        uint32_t high[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(high[u]) : "r"(even + 128 * u + 4) : "memory");
#pragma unroll
        for (int u = 0; u < 4; ++u) words[u] = __byte_perm(words[u], high[u], 0x5432);
    }
}
// The values of a word.
template <typename T>
struct alignas(4) Word {
    static constexpr int kValues = 4 / sizeof(T);
    T v[kValues];
};
template <typename T>
__device__ __forceinline__ Word<T> as_word(uint32_t bits) {
    Word<T> w;
    memcpy(&w, &bits, 4);
    return w;
}
// Values e, e + 1 of a row (or e alone), which stand in one word there, as far as they are the row's.
template <typename T>
__device__ __forceinline__ void store_word(T* row, int e, int width, const Word<T>& w) {
    constexpr int N = Word<T>::kValues;
    if (e >= 0 && e + N <= width) {
        *reinterpret_cast<Word<T>*>(row + e) = w;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (e + i >= 0 && e + i < width) row[e + i] = w.v[i];
    }
}

// A warp's way through its tokens, 32 packs of their rows and J choices at a time.
struct Step {
    int64_t token;
    int pack0, chunk;
};
// What a warp has of a row in a step: 32 packs of 16 bytes, and one more piece where they stand anywhere.
constexpr int kPieces = 33;

// kAny: the rows and the tokens' rows begin at any value's place.  The warp's 512 bytes of a row are then copied as the 33
// pieces around them, and its lanes read words out of them, as the words of the token's row want them.
template <typename T, typename W, int J, bool kAny>
__global__ void __launch_bounds__(kRowThreads, Ring<J>::kCtas)
    expert_combine_ring_kernel(const T* y, const int* slots, const W* weights, T* out, int64_t tokens, int choices,
                               int rows, int width, int log2_lanes) {
    constexpr int S = sizeof(T), V = 16 / S, kDeep = Ring<J>::kDeep, N = Word<T>::kValues;
    // Shared memory for a warp's part of a row, and from one row of a step to the next.
    constexpr int kRow = kAny ? kPieces * 16 : 32 * 16, kNext = kAny ? kRow : kRow * (kRowThreads / 32);
    extern __shared__ __align__(16) uint8_t ring[];
    grid_launch_dependents();
    grid_dependency_wait();
    const RowWalk w = row_walk(log2_lanes);
    const int packs = kAny ? (width + N - 1 + V - 1) / V : width / V;
    const int lane = threadIdx.x & 31, chunks = (choices + J - 1) / J;
    const T* const y_end = y + (int64_t)rows * width;
    const uint32_t own = smem_u32(ring) + (threadIdx.x >> 5) * (kAny ? kDeep * J * kRow : kRow);
    const auto at = [&](int deep, int j) { return own + (uint32_t)((deep * J + j) * kNext); };
    const auto next = [&](Step& s) {
        if (++s.chunk < chunks) return;
        s.chunk = 0;
        s.pack0 += w.pack_step;
        if (s.pack0 < packs) return;
        s.pack0 = w.pack - lane;
        s.token += w.token_step;
    };
    // The value that a step's packs begin with: one before the row's pack where its words begin there.
    const auto first_value = [&](const Step& s) {
        const int e0 = s.pack0 * V;
        if constexpr (S == 4 || !kAny) return e0;
        else return e0 - (int)(((uint32_t)(reinterpret_cast<uintptr_t>(out) >> 1) + (uint32_t)s.token * (uint32_t)width) & 1u);
    };
    // Lane j has choice j of a step, as it was read.
    struct Choice {
        int slot;
        W weight;
    };
    const auto choice = [&](Step& s) {
        Choice c;
        c.slot = -1;
        const int j = s.chunk * J + lane;
        if (lane < J && j < choices && s.token < tokens) {
            c.slot = slots[s.token * choices + j];
            if (weights != nullptr) c.weight = weights[s.token * choices + j];
        }
        next(s);
        return c;
    };
    uint32_t present[kDeep];  // which of a step's choices have a row
    float weight[kDeep];      // (lane j) the weight of choice j
    int shift[kDeep];         // kAny, in place of present: (lane j) that of choice j, negative without a row
    const auto ask = [&](int deep, Step& s, const Choice& c) {
        const int own_row = row_of(c.slot, rows);
        if constexpr (!kAny) present[deep] = __ballot_sync(0xffffffffu, own_row >= 0);
        weight[deep] = weights != nullptr && c.slot >= 0 ? to_f32(c.weight) : 1.0f;
        if constexpr (kAny) {
            // Where the row's part stands in its pieces, the first of them, and whether all are the matrix's.
            const int e0 = first_value(s);
            const int own_shift = own_row < 0 ? -1 : row_shift(y, own_row, width, e0);
            const T* const own_from = own_row < 0 ? nullptr : y + (int64_t)own_row * width + (e0 - own_shift / S);
            shift[deep] = own_shift;
            if (__all_sync(0xffffffffu, own_row < 0 || (own_from >= y && own_from + kPieces * V <= y_end))) {
                // What stands before and behind the row in the pieces is read along and left out of the results.
                const bool needed = e0 + V * (lane - 1) < width;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const uint64_t from = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(own_from), j);
                    if (from != 0 && needed) copy_async(at(deep, j) + lane * 16, reinterpret_cast<const T*>(from) + lane * V);
                }
                if (own_shift >= 0 && e0 + V * 31 < width) copy_async(at(deep, lane) + 32 * 16, own_from + 32 * V);  // the last
            } else {
#pragma unroll 1
                for (int j = 0; j < J; ++j) {
                    const uint64_t from = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(own_from), j);
                    const int first = e0 - __shfl_sync(0xffffffffu, own_shift, j) / S + V * lane;
                    if (from != 0)
                        copy_piece(at(deep, j) + lane * 16, reinterpret_cast<const T*>(from) + lane * V, first, width, y);
                }
                if (own_shift >= 0) copy_piece(at(deep, lane) + 32 * 16, own_from + 32 * V, e0 - own_shift / S + 32 * V, width, y);
            }
        } else {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int row = __shfl_sync(0xffffffffu, own_row, j);
                if (row >= 0 && s.pack0 + lane < packs)
                    copy_async(at(deep, j) + lane * 16, y + (int64_t)row * width + (int64_t)(s.pack0 + lane) * V);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        next(s);
    };
    Step now = {w.token, w.pack - lane, 0};
    if (now.pack0 >= packs) return;  // more lanes than packs
    Step asked = now, read = now;
    Choice known = choice(read);
#pragma unroll
    for (int i = 0; i < kDeep - 1; ++i) {
        ask(i, asked, known);
        known = choice(read);
    }
    float sum[V];
    while (now.token < tokens) {
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
            if (now.token >= tokens) break;
            asm volatile("cp.async.wait_group %0;" ::"n"(kDeep - 2) : "memory");
            if constexpr (kAny) __syncwarp();  // the other lanes' pieces; and all have read what the next request overwrites
            if (now.chunk == 0)
#pragma unroll
                for (int x = 0; x < V; ++x) sum[x] = 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float f = __shfl_sync(0xffffffffu, weight[i], j);
                const int sh = kAny ? __shfl_sync(0xffffffffu, shift[i], j) : 0;
                if (kAny ? sh < 0 : !(present[i] >> j & 1)) continue;
                if constexpr (kAny) {
                    const uint32_t from = at(i, j) + sh + 4 * lane;
                    uint32_t words[4];
                    load_words<S>(words, from);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const Word<T> v = as_word<T>(words[u]);
#pragma unroll
                        for (int x = 0; x < N; ++x) sum[u * N + x] = fmaf(f, to_f32(v.v[x]), sum[u * N + x]);
                    }
                } else {
                    const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(ring + (i * J + j) * kNext + threadIdx.x * 16);
#pragma unroll
                    for (int x = 0; x < V; ++x) sum[x] = fmaf(f, to_f32(v.v[x]), sum[x]);
                }
            }
            if (now.chunk == chunks - 1) {
                if constexpr (kAny) {
                    const int e0 = first_value(now);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        Word<T> o;
#pragma unroll
                        for (int x = 0; x < N; ++x) o.v[x] = round_to<T>(sum[u * N + x]);
                        store_word(out + now.token * width, e0 + N * (lane + 32 * u), width, o);
                    }
                } else if (now.pack0 + lane < packs) {
                    Pack<T, V> o;
#pragma unroll
                    for (int x = 0; x < V; ++x) o.v[x] = round_to<T>(sum[x]);
                    store<T, V>(out + now.token * width + (int64_t)(now.pack0 + lane) * V, o);
                }
            }
            next(now);
            ask((i + kDeep - 1) % kDeep, asked, known);
            known = choice(read);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The sums of the weights' gradients over a row's lanes: in a thread, in its warp, then over the row's warps, always in
// the same order.  All threads of the CTA.
template <typename W>
__device__ __forceinline__ void store_dots(float (&dot)[kAtOnce], float (&part)[kRowThreads / 32][kAtOnce], W* grad_weights,
                                           int64_t t, int64_t tokens, int j0, int choices, int log2_lanes) {
    const int warps = (1 << log2_lanes) / 32, own = threadIdx.x >> log2_lanes, l = threadIdx.x & ((1 << log2_lanes) - 1);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], d);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][j] = dot[j];
    }
    __syncthreads();
    if (l < kAtOnce && j0 + l < choices && t < tokens) {
        float sum = 0.0f;
        for (int w = 0; w < warps; ++w) sum += part[own * warps + w][l];
        grad_weights[t * choices + j0 + l] = round_to<W>(sum);
    }
    __syncthreads();
}

// One pass over a token's rows for both gradients.
template <typename T, typename W, int V, int U>
__global__ void __launch_bounds__(kRowThreads)
    expert_combine_grad_kernel(const T* grad, const T* y, const int* slots, const W* weights, T* grad_y, W* grad_weights,
                               int64_t tokens, int choices, int rows, int width, int log2_lanes) {
    __shared__ float part[kRowThreads / 32][kAtOnce];
    // The next kernel does not start before the end: a combine, which divides the SM's memory otherwise, gained nothing from
    // an early start (both, 64 tokens of 4 rows of 4096 and 500 of 512 bf16: 7.4 and 6.9 us with it, 7.1 and 6.4 without).
    grid_dependency_wait();
    const int lanes = 1 << log2_lanes;  // 32 or more
    const int side = kRowThreads >> log2_lanes, own = threadIdx.x >> log2_lanes, l = threadIdx.x & (lanes - 1);
    const int packs = width / V;
    for (int64_t t0 = (int64_t)blockIdx.x * side; t0 < tokens; t0 += (int64_t)gridDim.x * side) {
        const int64_t t = t0 + own;
        for (int j0 = 0; j0 < choices; j0 += kAtOnce) {
            int row[kAtOnce];
            W weight[kAtOnce];
            float f[kAtOnce], dot[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                row[j] = -1;
                if (t >= tokens || j0 + j >= choices) continue;
                row[j] = slots[t * choices + j0 + j];
                weight[j] = weights[t * choices + j0 + j];
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                dot[j] = 0.0f;
                row[j] = row_of(row[j], rows);
                f[j] = row[j] >= 0 ? to_f32(weight[j]) : 0.0f;
            }
            if (t < tokens) {
                for (int p = l; p < packs; p += U * lanes) {
                    Pack<T, V> g[U], v[kAtOnce][U];
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (p + u * lanes < packs) g[u] = load<T, V>(grad + t * width + (int64_t)(p + u * lanes) * V);
#pragma unroll
                    for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (row[j] >= 0 && p + u * lanes < packs)
                                v[j][u] = load<T, V>(y + (int64_t)row[j] * width + (int64_t)(p + u * lanes) * V);
#pragma unroll
                    for (int j = 0; j < kAtOnce; ++j) {
                        if (row[j] < 0) continue;
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            if (p + u * lanes >= packs) continue;
                            Pack<T, V> o;
#pragma unroll
                            for (int i = 0; i < V; ++i) {
                                const float gi = to_f32(g[u].v[i]);
                                dot[j] = fmaf(gi, to_f32(v[j][u].v[i]), dot[j]);
                                o.v[i] = round_to<T>(f[j] * gi);
                            }
                            store<T, V>(grad_y + (int64_t)row[j] * width + (int64_t)(p + u * lanes) * V, o);
                        }
                    }
                }
            }
            store_dots<W>(dot, part, grad_weights, t, tokens, j0, choices, log2_lanes);
        }
    }
}

// The same for many tokens and rows that are 16-byte aligned: the parts of up to four rows and of the token's own come
// through a ring as in combine, a thread's 16 bytes of each, a step ahead.  A token is a CTA's (kWhole), whose warps add up
// the sums of the weights' gradients in order, or a warp's.  4109 tokens of 8 rows of 2048 bf16 47.7 us (the kernel above
// 57), 16384 of 2 rows of 4096 116 (146); two steps ahead with three CTAs an SM 50.4 and 115.6, and 77 where this takes 67.
constexpr int kGradRows = 4, kGradDeep = 2;
constexpr int kGradCtas = 4;  // of an SM
constexpr size_t kGradSmem = (size_t)kGradDeep * (kGradRows + 1) * kRowThreads * 16;

template <typename T, typename W, bool kWhole>
__global__ void __launch_bounds__(kRowThreads, kGradCtas)
    expert_combine_grad_ring_kernel(const T* grad, const T* y, const int* slots, const W* weights, T* grad_y,
                                    W* grad_weights, int64_t tokens, int choices, int rows, int width) {
    constexpr int V = 16 / sizeof(T), J = kGradRows, D = kGradDeep, kWarps = kRowThreads / 32;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float part[2][kWarps][J];
    // The next kernel does not start before the end.  Started early into this one's division of the SM's memory, a combine
    // found room for three CTAs an SM instead of four, and its fourth part came after the others (a training step's two
    // calls: 354 us instead of 303; the largest division for both kernels took 331 and slowed combine down).
    grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int packs = width / V, chunks = (choices + J - 1) / J;
    const int pack_first = kWhole ? warp * 32 : 0, pack_step = kWhole ? kRowThreads : 32;
    const int64_t token_first = kWhole ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kWarps + warp;
    const int64_t token_step = kWhole ? (int64_t)gridDim.x : (int64_t)gridDim.x * kWarps;
    uint8_t* const own = ring + threadIdx.x * 16;
    const auto at = [&](int deep, int j) { return own + (deep * (J + 1) + j) * (kRowThreads * 16); };
    const auto next_row = [&](Step& s) {
        s.pack0 = pack_first;
        if (++s.chunk < chunks) return;
        s.chunk = 0;
        s.token += token_step;
    };
    // True at the end of a row's packs.  A warp behind them goes through every row once, too, with nothing to do.
    const auto next = [&](Step& s) {
        s.pack0 += pack_step;
        if (s.pack0 < packs) return false;
        next_row(s);
        return true;
    };
    // Lane j has choice j of a token's row, as it was read; lane J has the token's own row.
    struct Choice {
        int slot;
        W weight;
        int64_t token;
    };
    const auto choice = [&](const Step& s) {
        Choice c;
        c.slot = -1;
        c.token = s.token;
        const int j = s.chunk * J + lane;
        if (lane < J && j < choices && s.token < tokens) {
            c.slot = slots[s.token * choices + j];
            c.weight = weights[s.token * choices + j];
        }
        return c;
    };
    // Where the warp's next packs of them are, if there are any.
    struct Part {
        int row;
        float weight;
        const T* from;
    };
    const auto part_of = [&](const Choice& choice) {
        Part c;
        c.row = row_of(choice.slot, rows);
        c.weight = c.row >= 0 ? to_f32(choice.weight) : 0.0f;
        c.from = c.row >= 0 ? y + (int64_t)c.row * width + pack_first * V : nullptr;
        if (lane == J && choice.token < tokens) c.from = grad + choice.token * width + pack_first * V;
        return c;
    };
    Step now = {token_first, pack_first, 0};
    Step asked = now, read = now;
    // The rows that are asked for, and the choices after them: a warp's tokens change often, and it looks at their slots when
    // it comes to them (16384 tokens of 4 rows of 256 and 1024 bf16 15.0 and 55.3 us, at once 15.7 and 56.2); a CTA's change
    // seldom, and it looks at them at once (of 2048 and 4096 95 and 201 us, later 100 and 204).
    Part known = part_of(choice(read)), then;
    next_row(read);
    Choice after = choice(read);
    if constexpr (kWhole) then = part_of(after);
    int row[D];  // (lane j) of a step's choice j
    float weight[D];
    const auto ask = [&](int deep) {
        row[deep] = known.row;
        weight[deep] = known.weight;
#pragma unroll
        for (int j = 0; j <= J; ++j) {
            const uint64_t from = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(known.from), j);
            if (from != 0 && asked.pack0 + lane < packs)
                copy_async(smem_u32(at(deep, j)), reinterpret_cast<const T*>(from) + lane * V);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (known.from != nullptr) known.from += pack_step * V;
        if (next(asked)) {
            known = kWhole ? then : part_of(after);
            next_row(read);
            after = choice(read);
            if constexpr (kWhole) then = part_of(after);
        }
    };
#pragma unroll
    for (int i = 0; i < D - 1; ++i) ask(i);
    float dot[J] = {};
    int turn = 0;
    while (now.token < tokens) {
#pragma unroll
        for (int i = 0; i < D; ++i) {
            if (now.token >= tokens) break;
            asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
            const int pack = now.pack0 + lane;
            const bool inside = pack < packs;
            Pack<T, V> g;
            if (inside) g = *reinterpret_cast<const Pack<T, V>*>(at(i, J));
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int r = __shfl_sync(0xffffffffu, row[i], j);
                const float f = __shfl_sync(0xffffffffu, weight[i], j);
                if (r < 0 || !inside) continue;
                const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(at(i, j));
                Pack<T, V> o;
#pragma unroll
                for (int x = 0; x < V; ++x) {
                    const float gx = to_f32(g.v[x]);
                    dot[j] = fmaf(gx, to_f32(v.v[x]), dot[j]);
                    o.v[x] = round_to<T>(f * gx);
                }
                store<T, V>(grad_y + (int64_t)r * width + (int64_t)pack * V, o);
            }
            const int64_t entry = now.token * choices + now.chunk * J;
            const int left = choices - now.chunk * J;
            if (next(now)) {
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < J; ++j) {
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], d);
                    if (kWhole && lane == 0) part[turn][warp][j] = dot[j];
                    if (!kWhole && lane == j) sum = dot[j];
                    dot[j] = 0.0f;
                }
                if constexpr (kWhole) {
                    // The warps come here after different numbers of steps.  The first one has read the turn before last
                    // before it came here the last time.
                    asm volatile("bar.sync 1, %0;" ::"n"(kRowThreads) : "memory");
                    if (warp == 0 && lane < J)
#pragma unroll
                        for (int x = 0; x < kWarps; ++x) sum += part[turn][x][lane];
                    turn ^= 1;
                }
                if ((!kWhole || warp == 0) && lane < J && lane < left) grad_weights[entry + lane] = round_to<W>(sum);
            }
            ask((i + D - 1) % D);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ------------------------------------------------------------------ host side
template <typename Kernel, typename... Args>
static int launch(Kernel kernel, dim3 grid, int threads, int cluster, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    TRB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return TRB_OK;
}

template <typename Id>
static int launch_sort(const void* ids, int entries, int experts, int* offsets, int* slots, int dev,
                       cudaStream_t stream) {
    constexpr size_t kMost = sizeof(int) * (kSortWarps + 3) * kMaxGroups;
    static bool attr_set[64] = {};
    if (dev >= 64 || !attr_set[dev]) {
        TRB_CUDA(cudaFuncSetAttribute(expert_sort_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost));
        TRB_CUDA(cudaFuncSetAttribute(expert_sort_kernel<Id>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (dev < 64) attr_set[dev] = true;
    }
    // 32872 choices of 128 experts in clusters of 8 and 16 CTAs 8.8 and 6.8 us, 131072 of 256 25.9 and 14.2; one CTA is
    // enough, and fastest, up to two groups of 32 choices a warp.  Clusters of 16 are more than every device has to offer.
    const int64_t groups = ((int64_t)entries + 31) / 32;
    int ctas = groups <= 2 * kSortWarps ? 1 : groups <= 8 * kSortWarps ? 4 : 8;
    if (groups > 16 * kSortWarps) {
        static int places[64] = {};
        if (clusters_at_once(expert_sort_kernel<Id>, kSortThreads, kMost, kSortCtas, dev, places) > 0) ctas = kSortCtas;
    }
    const int warps = (int)std::min<int64_t>(kSortWarps, std::max<int64_t>(groups, 8));
    const size_t smem = sizeof(int) * (size_t)(warps + 3) * experts;
    return launch(expert_sort_kernel<Id>, dim3((unsigned)ctas), 32 * warps, ctas, smem, stream,
                  static_cast<const Id*>(ids), entries, experts, offsets, slots);
}

struct RowShape {
    dim3 grid;
    int log2_lanes;
};
// As many lanes a token as its row has packs, at_once each, between a warp and a CTA; a row is shared among CTAs while the GPU is not full.
static RowShape row_shape(int64_t tokens, int packs, int at_once, bool whole_rows, int dev) {
    RowShape s;
    s.log2_lanes = 5;
    while (s.log2_lanes < 8 && at_once << s.log2_lanes < packs) ++s.log2_lanes;
    const int64_t side = kRowThreads >> s.log2_lanes, blocks = (tokens + side - 1) / side;
    const int64_t full = 8 * (int64_t)device_sm_count(dev);  // CTAs of 256 threads that the GPU holds
    const int64_t share = whole_rows ? 1 : std::max<int64_t>(1, std::min<int64_t>((packs + kRowThreads - 1) / kRowThreads,
                                                                                  full / std::max<int64_t>(blocks, 1)));
    s.grid = dim3((unsigned)std::min<int64_t>(blocks, 1 << 30), (unsigned)std::min<int64_t>(share, 1024));
    return s;
}

static int check(const char* what, int dtype, int weight_dtype, int tokens, int choices, int rows, int width,
                 const void* slots, const void* weights) {
    if (tokens < 0 || choices <= 0 || rows < 0 || width <= 0 || (tokens > 0 && slots == nullptr)) {
        set_error("%s: sizes must be positive (tokens and rows may be 0) and pointers non-null", what);
        return TRB_ERR_ARGS;
    }
    if (dtype != TRB_BFLOAT16 && dtype != TRB_FLOAT16 && dtype != TRB_FLOAT32) {
        set_error("%s: unsupported dtype %s (bfloat16, float16 and float32)", what, dtype_name(dtype));
        return TRB_SKIPPED;
    }
    if (weights != nullptr && weight_dtype != TRB_FLOAT32 && weight_dtype != dtype) {
        set_error("%s: weights must be float32 or %s, not %s", what, dtype_name(dtype), dtype_name(weight_dtype));
        return TRB_SKIPPED;
    }
    if (std::max({rows, width}) > kMaxExtent || (int64_t)tokens * choices > kMaxExtent) {
        set_error("%s: rows, width and tokens * choices at most %d (rows=%d width=%d tokens=%d choices=%d)", what,
                  kMaxExtent, rows, width, tokens, choices);
        return TRB_SKIPPED;
    }
    return TRB_OK;
}

static uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Pointers are aligned to their elements.  Wider accesses are chosen where they are aligned to more (access_bytes).
static int check_align(const char* what, int dtype, int weight_dtype, uintptr_t values, const void* weights,
                       const void* grad_weights, const void* slots) {
    const size_t size = dtype_size(dtype), weight_size = dtype_size(weight_dtype);
    if (values % size != 0 || bits(slots) % 4 != 0 ||
        (weights != nullptr && (bits(weights) | bits(grad_weights)) % weight_size != 0)) {
        set_error("%s: pointers must be aligned to their elements", what);
        return TRB_ERR_ALIGN;
    }
    return TRB_OK;
}

// The widest access, 16, 8, 4 or 2 bytes, that all rows are made of, aligned.
static int access_bytes(size_t size, int width, uintptr_t pointers) {
    const uint64_t all = (uint64_t)width * size | pointers | 16;
    return (int)std::min<uint64_t>(all & (~all + 1), 16);
}

template <typename T, typename W, int J, bool kAny>
static int launch_ring(const void* y, const int* slots, const void* weights, void* out, int tokens, int choices, int rows,
                       int width, int dev, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    constexpr size_t smem = Ring<J>::smem(kAny ? kPieces : 32);
    static bool attr_set[64] = {};
    if (dev >= 64 || !attr_set[dev]) {
        TRB_CUDA(cudaFuncSetAttribute(expert_combine_ring_kernel<T, W, J, kAny>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)smem));
        if (dev < 64) attr_set[dev] = true;
    }
    RowShape s = row_shape(tokens, kAny ? (width + Word<T>::kValues + V - 2) / V : width / V, 1, false, dev);
    // No more CTAs than the GPU holds, each for several tokens.
    const unsigned places = (unsigned)(device_sm_count(dev) * Ring<J>::kCtas);
    s.grid.x = std::max(1u, std::min(s.grid.x, places / s.grid.y));
    return launch(expert_combine_ring_kernel<T, W, J, kAny>, s.grid, kRowThreads, 0, smem, stream, static_cast<const T*>(y),
                  slots, static_cast<const W*>(weights), static_cast<T*>(out), (int64_t)tokens, choices, rows, width,
                  s.log2_lanes);
}

// One of the two moves with V values an access.
template <typename T, typename W, int V>
static int launch_move(bool back, const void* src, const int* slots, const void* weights, void* dst, int tokens,
                       int choices, int rows, int width, int dev, cudaStream_t stream) {
    constexpr int B = V * sizeof(T);
    if (back) {
        // Eight rows a step where each has shifting to do and there are as many: 4109 tokens of 8 rows of 2047 and 2048 bf16
        // 30.6 and 26.1 us, four rows 34.2 and 25.2.
        constexpr bool kAny = B != 16;
        if constexpr (kAny)
            if (choices > 4)
                return launch_ring<T, W, 8, kAny>(src, slots, weights, dst, tokens, choices, rows, width, dev, stream);
        return choices <= 2
                   ? launch_ring<T, W, 2, kAny>(src, slots, weights, dst, tokens, choices, rows, width, dev, stream)
                   : launch_ring<T, W, 4, kAny>(src, slots, weights, dst, tokens, choices, rows, width, dev, stream);
    }
    const auto run = [&](auto kernel, int at_once) {
        const RowShape s = row_shape(tokens, width / V, at_once, false, dev);
        return launch(kernel, s.grid, kRowThreads, 0, 0, stream, static_cast<const T*>(src), slots,
                      static_cast<const W*>(weights), static_cast<T*>(dst), (int64_t)tokens, choices, rows, width,
                      s.log2_lanes);
    };
    // Accesses of a lane on their way: 4109 tokens of 8 rows of 2047 bf16 with 2, 4 and 8 of them 49, 43 and 43 us.
    constexpr int U = B == 16 ? 1 : B == 8 ? 2 : 4;
    return run(expert_dispatch_kernel<T, W, V, U>, U);
}

template <typename T, typename W>
static int move_rows(bool back, const void* src, const int* slots, const void* weights, void* dst, int tokens, int choices,
                     int rows, int width, int dev, cudaStream_t stream) {
    constexpr int S = sizeof(T);
    switch (access_bytes(S, width, bits(src) | bits(dst))) {
        case 16: return launch_move<T, W, 16 / S>(back, src, slots, weights, dst, tokens, choices, rows, width, dev, stream);
        case 8: return launch_move<T, W, 8 / S>(back, src, slots, weights, dst, tokens, choices, rows, width, dev, stream);
        case 4: return launch_move<T, W, 4 / S>(back, src, slots, weights, dst, tokens, choices, rows, width, dev, stream);
        default: return launch_move<T, W, 1>(back, src, slots, weights, dst, tokens, choices, rows, width, dev, stream);
    }
}

static int move(const char* what, bool back, int dtype, int weight_dtype, int tokens, int choices, int rows, int width,
                const void* src, const int32_t* slots, const void* weights, void* dst, void* stream) {
    clear_error();
    int rc = check(what, dtype, weight_dtype, tokens, choices, rows, width, slots, weights);
    if (rc != TRB_OK) return rc;
    if (tokens == 0) return TRB_OK;
    const void* const tokens_side = back ? dst : src;
    const void* const rows_side = back ? src : dst;
    if (tokens_side == nullptr || (rows > 0 && rows_side == nullptr)) {
        set_error("%s: rows must be non-null", what);
        return TRB_ERR_ARGS;
    }
    rc = check_align(what, dtype, weight_dtype, bits(src) | bits(dst), weights, nullptr, slots);
    if (rc != TRB_OK) return rc;
    const uint64_t size = dtype_size(dtype), entries = (uint64_t)tokens * choices;
    rc = check_apart(what, {{dst, size, (uint64_t)(back ? tokens : rows), (uint64_t)width}},
                     {{src, size, (uint64_t)(back ? rows : tokens), (uint64_t)width},
                      {slots, 4, entries},
                      {weights, dtype_size(weight_dtype), entries}});
    if (rc != TRB_OK) return rc;
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f32 = weight_dtype == TRB_FLOAT32;
    const auto call = [&](auto f) { return f(back, src, slots, weights, dst, tokens, choices, rows, width, dev, s); };
    if (dtype == TRB_BFLOAT16)
        return f32 ? call(move_rows<__nv_bfloat16, float>) : call(move_rows<__nv_bfloat16, __nv_bfloat16>);
    if (dtype == TRB_FLOAT16) return f32 ? call(move_rows<__half, float>) : call(move_rows<__half, __half>);
    return call(move_rows<float, float>);
}

template <typename T, typename W, bool kWhole>
static int launch_grad_ring(const void* grad, const void* y, const int* slots, const void* weights, void* grad_y,
                            void* grad_weights, int tokens, int choices, int rows, int width, int dev,
                            cudaStream_t stream) {
    static bool attr_set[64] = {};
    if (dev >= 64 || !attr_set[dev]) {
        TRB_CUDA(cudaFuncSetAttribute(expert_combine_grad_ring_kernel<T, W, kWhole>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kGradSmem));
        if (dev < 64) attr_set[dev] = true;
    }
    const int64_t side = kWhole ? 1 : kRowThreads / 32, blocks = (tokens + side - 1) / side;
    const int64_t places = (int64_t)device_sm_count(dev) * kGradCtas;
    return launch(expert_combine_grad_ring_kernel<T, W, kWhole>, dim3((unsigned)std::min(blocks, places)), kRowThreads, 0,
                  kGradSmem, stream, static_cast<const T*>(grad), static_cast<const T*>(y), slots,
                  static_cast<const W*>(weights), static_cast<T*>(grad_y), static_cast<W*>(grad_weights), (int64_t)tokens,
                  choices, rows, width);
}

template <typename T, typename W>
static int launch_grad(const void* grad, const void* y, const int* slots, const void* weights, void* grad_y,
                       void* grad_weights, int tokens, int choices, int rows, int width, int dev, cudaStream_t stream) {
    constexpr int S = sizeof(T);
    const auto run = [&](auto kernel, int values, int at_once) {
        const RowShape s = row_shape(tokens, width / values, at_once, true, dev);
        return launch(kernel, s.grid, kRowThreads, 0, 0, stream, static_cast<const T*>(grad), static_cast<const T*>(y),
                      slots, static_cast<const W*>(weights), static_cast<T*>(grad_y), static_cast<W*>(grad_weights),
                      (int64_t)tokens, choices, rows, width, s.log2_lanes);
    };
    const int access = access_bytes(S, width, bits(grad) | bits(y) | bits(grad_y)), packs = width / (16 / S);
    // The ring has a CTA a token where its row keeps all threads busy (16384 tokens of 4 rows of 1024 and 2048 bf16: a CTA 67
    // and 95 us, a warp 57 and 110, without the ring 64 and 124), and is for tokens enough for all CTAs, or warps, of it to
    // be worth their start (a CTA: 64 and 500 tokens of 4 rows of 4096 bf16 4.0 and 8.6 us, without the ring 3.6 and 10.2;
    // a warp: 500 and 16384 of 4 rows of 512 4.0 and 28.7, without 3.2 and 34.4).  Rows a little wider than a CTA were
    // not measured with a warp a token; with a CTA 16384 tokens of 4 rows of 2056 and 2400 bf16 take 113 and 128 us (floors
    // 93 and 108).
    if (access == 16) {
        const int64_t sms = device_sm_count(dev);
        if (packs >= kRowThreads && tokens >= sms)
            return launch_grad_ring<T, W, true>(grad, y, slots, weights, grad_y, grad_weights, tokens, choices, rows, width,
                                                dev, stream);
        if (packs < kRowThreads && tokens >= sms * kGradCtas * (kRowThreads / 32))
            return launch_grad_ring<T, W, false>(grad, y, slots, weights, grad_y, grad_weights, tokens, choices, rows, width,
                                                 dev, stream);
    }
    switch (access) {
        case 16: return run(expert_combine_grad_kernel<T, W, 16 / S, 1>, 16 / S, 1);
        // Accesses of each row on their way: two of single values, one of more.  4109 tokens of 8 rows of 2047, 2046 and 2044
        // bf16 with one, two and four: 104, 91 and 87 us; 79, 97 and 255; 72, 75 and 146.  509 of 8 of 1001 float32: 11.6,
        // 10.1 and 11.9.
        case 8: return run(expert_combine_grad_kernel<T, W, 8 / S, 1>, 8 / S, 1);
        case 4: return run(expert_combine_grad_kernel<T, W, 4 / S, S == 4 ? 2 : 1>, 4 / S, S == 4 ? 2 : 1);
        default: return run(expert_combine_grad_kernel<T, W, 1, 2>, 1, 2);
    }
}

int read_error(bool clear) {
    int v = 0;
    TRB_CUDA(cudaMemcpyFromSymbol(&v, g_rows_error, sizeof(int)));
    if (clear) {
        const int zero = 0;
        TRB_CUDA(cudaMemcpyToSymbol(g_rows_error, &zero, sizeof(int)));
    }
    return v;
}

}  // namespace rows
}  // namespace trb

extern "C" int trb_expert_sort_launch(int id_bytes, int tokens, int choices, int experts, const void* ids,
                                      int32_t* offsets, int32_t* slots, void* stream) {
    using namespace trb;
    clear_error();
    if (tokens < 0 || choices <= 0 || experts <= 0 || offsets == nullptr ||
        (tokens > 0 && (ids == nullptr || slots == nullptr))) {
        set_error("trb_expert_sort_launch: sizes must be positive (tokens may be 0) and pointers non-null");
        return TRB_ERR_ARGS;
    }
    if (id_bytes != 4 && id_bytes != 8) {
        set_error("trb_expert_sort_launch: choices must be int32 or int64 (got %d bytes)", id_bytes);
        return TRB_SKIPPED;
    }
    if (experts > kMaxGroups) {
        set_error("trb_expert_sort_launch: at most %d experts (got %d)", kMaxGroups, experts);
        return TRB_SKIPPED;
    }
    if ((int64_t)tokens * choices > kMaxExtent) {
        set_error("trb_expert_sort_launch: tokens * choices at most %d (tokens=%d choices=%d)", kMaxExtent, tokens,
                  choices);
        return TRB_SKIPPED;
    }
    if (rows::bits(ids) % id_bytes != 0 || (rows::bits(offsets) | rows::bits(slots)) % 4 != 0) {
        set_error("trb_expert_sort_launch: pointers must be aligned to their elements");
        return TRB_ERR_ALIGN;
    }
    const uint64_t entries = (uint64_t)tokens * choices;
    const int rc = check_apart("trb_expert_sort_launch", {{offsets, 4, (uint64_t)experts + 1}, {slots, 4, entries}},
                               {{ids, (uint64_t)id_bytes, entries}});
    if (rc != TRB_OK) return rc;
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return id_bytes == 4 ? rows::launch_sort<int>(ids, tokens * choices, experts, offsets, slots, dev, s)
                         : rows::launch_sort<long long>(ids, tokens * choices, experts, offsets, slots, dev, s);
}

extern "C" int trb_expert_dispatch_launch(int dtype, int weight_dtype, int tokens, int choices, int rows, int width,
                                          const void* x, const int32_t* slots, const void* weights, void* out,
                                          void* stream) {
    return trb::rows::move("trb_expert_dispatch_launch", false, dtype, weight_dtype, tokens, choices, rows, width, x, slots,
                           weights, out, stream);
}

extern "C" int trb_expert_combine_launch(int dtype, int weight_dtype, int tokens, int choices, int rows, int width,
                                         const void* y, const int32_t* slots, const void* weights, void* out,
                                         void* stream) {
    return trb::rows::move("trb_expert_combine_launch", true, dtype, weight_dtype, tokens, choices, rows, width, y, slots,
                           weights, out, stream);
}

extern "C" int trb_expert_combine_grad_launch(int dtype, int weight_dtype, int tokens, int choices, int rows, int width,
                                              const void* grad, const void* y, const int32_t* slots, const void* weights,
                                              void* grad_y, void* grad_weights, void* stream) {
    using namespace trb;
    const char* const what = "trb_expert_combine_grad_launch";
    clear_error();
    int rc = rows::check(what, dtype, weight_dtype, tokens, choices, rows, width, slots, weights);
    if (rc != TRB_OK) return rc;
    if (tokens == 0) return TRB_OK;
    if (grad == nullptr || weights == nullptr || grad_weights == nullptr ||
        (rows > 0 && (y == nullptr || grad_y == nullptr))) {
        set_error("%s: pointers must be non-null", what);
        return TRB_ERR_ARGS;
    }
    rc = rows::check_align(what, dtype, weight_dtype, rows::bits(grad) | rows::bits(y) | rows::bits(grad_y), weights,
                           grad_weights, slots);
    if (rc != TRB_OK) return rc;
    const uint64_t size = dtype_size(dtype), weight_size = dtype_size(weight_dtype), entries = (uint64_t)tokens * choices;
    rc = check_apart(what, {{grad_y, size, (uint64_t)rows, (uint64_t)width}, {grad_weights, weight_size, entries}},
                     {{grad, size, (uint64_t)tokens, (uint64_t)width},
                      // The thread that writes a value of grad_y has read the one of y in its place, and nobody else does.
                      {y == grad_y ? nullptr : y, size, (uint64_t)rows, (uint64_t)width},
                      {slots, 4, entries},
                      {weights, weight_size, entries}});
    if (rc != TRB_OK) return rc;
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f32 = weight_dtype == TRB_FLOAT32;
    const auto call = [&](auto f) {
        return f(grad, y, slots, weights, grad_y, grad_weights, tokens, choices, rows, width, dev, s);
    };
    if (dtype == TRB_BFLOAT16)
        return f32 ? call(rows::launch_grad<__nv_bfloat16, float>) : call(rows::launch_grad<__nv_bfloat16, __nv_bfloat16>);
    if (dtype == TRB_FLOAT16) return f32 ? call(rows::launch_grad<__half, float>) : call(rows::launch_grad<__half, __half>);
    return call(rows::launch_grad<float, float>);
}
