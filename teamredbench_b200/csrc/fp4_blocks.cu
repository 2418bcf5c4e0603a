// fp4_blocks.cu -- rows to microscaled 4-bit floating point and back.
//
// For every block of 32 values of a row
//   e = floor(log2(max |x|)) - 2, at least -127,    q = x / 2^e on the grid of e2m1, ties to the even code, at most 6
// (the conversion of the OCP Microscaling Formats specification, version 1.0, section 6.3, with rounding to nearest
// even).  Dividing by a power of two is exact, so nothing is rounded but q itself.  A block that holds a NaN or an
// infinity gets the scale NaN and codes of 0: it is NaN as a whole.  A block of zeros gets the smallest scale.
//
// With slots, row t of x goes to the rows slots[t, j] of the result: tokens on their way to their experts are quantised
// once and written in 4 bits, instead of moved in 16 and quantised after.
//
// The bytes of the rows bound both ways: 16384 x 8192 bf16 to 4 bits in 49.6 us, 6.85 TB/s (two bytes read for 0.53
// written, a copy of as many bytes measures 6.55), and back in 52.6 us; 8192 x 8192 float32 in 46 us.
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

__device__ int g_fp4_error;

constexpr int kThreads = 256;
constexpr int kValues = 8;  // a thread's; four threads share a block

template <typename T>
struct alignas(16) Octet {
    T v[kValues];
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

// A word's two 16-bit values.
template <typename T>
__device__ __forceinline__ float2 pair_f32(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Eight values to eight codes, v[0] in the lowest four bits.
__device__ __forceinline__ uint32_t codes_of(const float (&v)[kValues]) {
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

// The four e2m1 pairs of a word as f16 pairs (exact).
__device__ __forceinline__ void halves_of(uint32_t codes, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
}

// Threads of a CTA: 1 << log2_lanes of them, 32 or more, for one row, several rows side by side; blockIdx.y shares a row
// among CTAs where there are few.
struct Walk {
    int first, step;  // octets
    int64_t row, row_step;
};
__device__ __forceinline__ Walk walk(int log2_lanes) {
    const int side = kThreads >> log2_lanes;
    return {(int)(blockIdx.y << log2_lanes) + (int)(threadIdx.x & ((1u << log2_lanes) - 1)), (int)(gridDim.y << log2_lanes),
            (int64_t)blockIdx.x * side + (threadIdx.x >> log2_lanes), (int64_t)gridDim.x * side};
}
constexpr int kAtOnce = 4;  // octets of a thread on their way, in dequantisation

// The exponent code of a block whose largest magnitude has the fp32 bits `largest`, and whether the block is all NaN.
__device__ __forceinline__ uint32_t scale_code(uint32_t largest, bool& nan) {
    const uint32_t exponent = largest >> 23;  // 127 + floor(log2), 0 below 2^-126, 255 for NaN and infinity
    nan = exponent == 255;
    return nan ? 255 : exponent > 2 ? exponent - 2 : 0;
}
__device__ __forceinline__ float inverse_of(uint32_t code) { return __uint_as_float((254 - code) << 23); }

// Calls put(row) for the row of x itself, or for every row that its slots name.
template <typename Put>
__device__ __forceinline__ void for_rows(const int* slots, int64_t t, int choices, int out_rows, const Put& put) {
    if (slots == nullptr) {
        put(t);
        return;
    }
    for (int j = 0; j < choices; ++j) {
        const int row = slots[t * choices + j];
        if (row >= out_rows) atomicCAS(&g_fp4_error, 0, kErrSlots);
        else if (row >= 0) put((int64_t)row);
    }
}

// 16-bit values: a thread takes a whole block, 64 bytes, so that there is one scale to work out for 32 values and
// nothing to exchange: 3.4 instructions a value, where eight values a thread took 13 and the issue slots bound it.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    quantize_fp4_kernel(const T* x, const int* slots, uint8_t* q, uint8_t* scales, int64_t rows, int choices, int out_rows,
                        int k) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int blocks = k / kBlock, pitch = scale_pitch(k);
    const int64_t total = rows * blocks;
    for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < total; g += (int64_t)gridDim.x * kThreads) {
        uint4 raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = reinterpret_cast<const uint4*>(x + g * kBlock)[i];
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[4 * i] = raw[i].x;
            w[4 * i + 1] = raw[i].y;
            w[4 * i + 2] = raw[i].z;
            w[4 * i + 3] = raw[i].w;
        }
        uint32_t most = 0;  // two magnitudes, whose bits are ordered as they are, NaN above all
#pragma unroll
        for (int i = 0; i < 16; ++i) most = __vmaxu2(most, w[i] & 0x7fff7fffu);
        most = max(most & 0xffffu, most >> 16);
        T largest;
        *reinterpret_cast<uint16_t*>(&largest) = (uint16_t)most;
        bool nan;
        const uint32_t code = scale_code(__float_as_uint(to_f32(largest)), nan);
        const float inverse = inverse_of(code);
        uint4 packed;
        uint32_t* const p = &packed.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[kValues];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 pair = pair_f32<T>(w[4 * i + j]);
                v[2 * j] = pair.x * inverse;
                v[2 * j + 1] = pair.y * inverse;
            }
            p[i] = nan ? 0 : codes_of(v);
        }
        int64_t t;
        int block;
        if (total <= UINT32_MAX) {
            t = (uint32_t)g / (uint32_t)blocks;
            block = (int)((uint32_t)g - (uint32_t)t * (uint32_t)blocks);
        } else {
            t = g / blocks;
            block = (int)(g - t * blocks);
        }
        for_rows(slots, t, choices, out_rows, [&](int64_t row) {
            *reinterpret_cast<uint4*>(q + (row * blocks + block) * (kBlock / 2)) = packed;
            scales[row * pitch + block] = (uint8_t)code;
            if (block == blocks - 1)
                for (int i = blocks; i < pitch; ++i) scales[row * pitch + i] = 0;
        });
    }
}

// 32-bit values: eight a thread, four threads a block.
__global__ void __launch_bounds__(kThreads)
    quantize_fp4_f32_kernel(const float* x, const int* slots, uint8_t* q, uint8_t* scales, int64_t rows, int choices,
                            int out_rows, int k, int log2_lanes) {
    grid_launch_dependents();
    grid_dependency_wait();
    const Walk w = walk(log2_lanes);
    const int octets = k / kValues, blocks = k / kBlock, pitch = scale_pitch(k);
    const uint32_t quad = 0xfu << (threadIdx.x & 28);
    for (int64_t t = w.row; t < rows; t += w.row_step) {
        for (int o = w.first; o < octets; o += w.step) {  // octets of a block: one quad of lanes
            Octet<float> in = *reinterpret_cast<const Octet<float>*>(x + t * k + (int64_t)o * kValues);
            uint32_t largest = 0;  // bits of a magnitude: ordered as the magnitudes are, NaN above all
#pragma unroll
            for (int i = 0; i < kValues; ++i) largest = max(largest, __float_as_uint(in.v[i]) & 0x7fffffffu);
            largest = max(largest, __shfl_xor_sync(quad, largest, 1));
            largest = max(largest, __shfl_xor_sync(quad, largest, 2));
            bool nan;
            const uint32_t code = scale_code(largest, nan);
            const float inverse = inverse_of(code);
#pragma unroll
            for (int i = 0; i < kValues; ++i) in.v[i] *= inverse;
            const uint32_t packed = nan ? 0 : codes_of(in.v);
            for_rows(slots, t, choices, out_rows, [&](int64_t row) {
                *reinterpret_cast<uint32_t*>(q + row * (k / 2) + (int64_t)o * (kValues / 2)) = packed;
                if (o % 4 == 0) scales[row * pitch + o / 4] = (uint8_t)code;
            });
        }
        if (w.first < pitch - blocks)  // behind the last block: zeros
            for_rows(slots, t, choices, out_rows, [&](int64_t row) { scales[row * pitch + blocks + w.first] = 0; });
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    dequantize_fp4_kernel(const uint8_t* q, const uint8_t* scales, T* out, int64_t rows, int k, int log2_lanes) {
    grid_launch_dependents();
    grid_dependency_wait();
    const Walk w = walk(log2_lanes);
    const int octets = k / kValues, pitch = scale_pitch(k);
    for (int64_t t = w.row; t < rows; t += w.row_step) {
        for (int o0 = w.first; o0 < octets; o0 += kAtOnce * w.step) {
            uint32_t packed[kAtOnce], code[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int o = o0 + u * w.step;
                if (o >= octets) break;
                packed[u] = *reinterpret_cast<const uint32_t*>(q + t * (k / 2) + (int64_t)o * (kValues / 2));
                code[u] = scales[t * pitch + o / (kBlock / kValues)];
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int o = o0 + u * w.step;
                if (o >= octets) break;
                const float scale = __uint_as_float(code[u] == 255 ? 0x7fffffffu : code[u] == 0 ? 0x00400000u : code[u] << 23);
                uint32_t h[4];
                halves_of(packed[u], h);
                Octet<T> v;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 pair = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
                    v.v[2 * i] = round_to<T>(pair.x * scale);
                    v.v[2 * i + 1] = round_to<T>(pair.y * scale);
                }
                *reinterpret_cast<Octet<T>*>(out + t * k + (int64_t)o * kValues) = v;
            }
        }
    }
}

// ------------------------------------------------------------------ host side
template <typename Kernel, typename... Args>
static int launch(Kernel kernel, dim3 grid, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    TRB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return TRB_OK;
}

// Rows of `octets`, at_once of them a thread.
template <typename Kernel, typename... Args>
static int launch_rows(Kernel kernel, int64_t rows, int octets, int at_once, int dev, cudaStream_t stream, Args... args) {
    int log2_lanes = 5;
    while (log2_lanes < 8 && (at_once << log2_lanes) < octets) ++log2_lanes;
    const int64_t blocks = (rows + (kThreads >> log2_lanes) - 1) / (kThreads >> log2_lanes);
    const int64_t full = 8 * (int64_t)device_sm_count(dev);  // CTAs that the GPU holds
    const int64_t share = std::max<int64_t>(1, std::min<int64_t>((octets + kThreads - 1) / kThreads, full / blocks));
    const dim3 grid((unsigned)std::min<int64_t>(blocks, 1 << 30), (unsigned)std::min<int64_t>(share, 1024));
    return launch(kernel, grid, stream, args..., log2_lanes);
}

static uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

static int check(const char* what, int dtype, int rows, int k, const void* values, const void* q, const void* scales) {
    if (rows < 0 || k <= 0) {
        set_error("%s: sizes must be positive (rows may be 0)", what);
        return TRB_ERR_ARGS;
    }
    if (dtype != TRB_BFLOAT16 && dtype != TRB_FLOAT16 && dtype != TRB_FLOAT32) {
        set_error("%s: unsupported dtype %s (bfloat16, float16 and float32)", what, dtype_name(dtype));
        return TRB_SKIPPED;
    }
    if (std::max(rows, k) > kMaxExtent) {
        set_error("%s: rows and k at most %d (rows=%d k=%d)", what, kMaxExtent, rows, k);
        return TRB_SKIPPED;
    }
    if (k % kBlock != 0) {
        set_error("%s: k must be a multiple of %d (k=%d)", what, kBlock, k);
        return TRB_ERR_ALIGN;
    }
    if (rows > 0 && (values == nullptr || q == nullptr || scales == nullptr)) {
        set_error("%s: pointers must be non-null", what);
        return TRB_ERR_ARGS;
    }
    if ((bits(values) | bits(q) | bits(scales)) % 16 != 0) {
        set_error("%s: pointers must be 16-byte aligned", what);
        return TRB_ERR_ALIGN;
    }
    return TRB_OK;
}

template <typename T>
static int launch_quantize(const void* x, const int* slots, void* q, void* scales, int rows, int choices, int out_rows,
                           int k, int dev, cudaStream_t stream) {
    if constexpr (sizeof(T) == 4) {
        return launch_rows(quantize_fp4_f32_kernel, rows, k / kValues, 1, dev, stream, static_cast<const float*>(x), slots,
                           static_cast<uint8_t*>(q), static_cast<uint8_t*>(scales), (int64_t)rows, choices, out_rows, k);
    } else {
        const int64_t ctas = ((int64_t)rows * (k / kBlock) + kThreads - 1) / kThreads;
        return launch(quantize_fp4_kernel<T>, dim3((unsigned)std::min<int64_t>(ctas, 1 << 30)), stream,
                      static_cast<const T*>(x), slots, static_cast<uint8_t*>(q), static_cast<uint8_t*>(scales),
                      (int64_t)rows, choices, out_rows, k);
    }
}

template <typename T>
static int launch_dequantize(const void* q, const void* scales, void* out, int rows, int k, int dev, cudaStream_t stream) {
    return launch_rows(dequantize_fp4_kernel<T>, rows, k / kValues, kAtOnce, dev, stream, static_cast<const uint8_t*>(q),
                       static_cast<const uint8_t*>(scales), static_cast<T*>(out), (int64_t)rows, k);
}

int read_error(bool clear) {
    int v = 0;
    TRB_CUDA(cudaMemcpyFromSymbol(&v, g_fp4_error, sizeof(int)));
    if (clear) {
        const int zero = 0;
        TRB_CUDA(cudaMemcpyToSymbol(g_fp4_error, &zero, sizeof(int)));
    }
    return v;
}

}  // namespace fp4
}  // namespace trb

extern "C" int trb_quantize_fp4_launch(int dtype, int rows, int k, const void* x, int choices, const int32_t* slots,
                                       int out_rows, void* q, void* scales, void* stream) {
    using namespace trb;
    const char* const what = "trb_quantize_fp4_launch";
    clear_error();
    // With slots and no row to write to, q and scales need not be there.
    const bool nothing = slots != nullptr && out_rows == 0;
    int rc = fp4::check(what, dtype, rows, k, x, nothing ? x : q, nothing ? x : scales);
    if (rc != TRB_OK) return rc;
    if (slots != nullptr && (choices <= 0 || out_rows < 0 || (fp4::bits(slots) & 3u) != 0)) {
        set_error("%s: slots need choices > 0, out_rows >= 0 and 4-byte alignment", what);
        return TRB_ERR_ARGS;
    }
    if (slots != nullptr && ((int64_t)rows * choices > kMaxExtent || out_rows > kMaxExtent)) {
        set_error("%s: out_rows and rows * choices at most %d (rows=%d choices=%d out_rows=%d)", what, kMaxExtent, rows,
                  choices, out_rows);
        return TRB_SKIPPED;
    }
    if (rows == 0) return TRB_OK;
    const uint64_t to = (uint64_t)(slots != nullptr ? out_rows : rows);
    rc = check_apart(what, {{q, 1, to, (uint64_t)k / 2}, {scales, 1, to, (uint64_t)fp4::scale_pitch(k)}},
                     {{x, dtype_size(dtype), (uint64_t)rows, (uint64_t)k},
                      {slots, 4, (uint64_t)rows, (uint64_t)(slots != nullptr ? choices : 0)}});
    if (rc != TRB_OK) return rc;
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == TRB_BFLOAT16)
        return fp4::launch_quantize<__nv_bfloat16>(x, slots, q, scales, rows, choices, out_rows, k, dev, s);
    if (dtype == TRB_FLOAT16) return fp4::launch_quantize<__half>(x, slots, q, scales, rows, choices, out_rows, k, dev, s);
    return fp4::launch_quantize<float>(x, slots, q, scales, rows, choices, out_rows, k, dev, s);
}

extern "C" int trb_dequantize_fp4_launch(int dtype, int rows, int k, const void* q, const void* scales, void* out,
                                         void* stream) {
    using namespace trb;
    clear_error();
    const char* const what = "trb_dequantize_fp4_launch";
    int rc = fp4::check(what, dtype, rows, k, out, q, scales);
    if (rc != TRB_OK || rows == 0) return rc;
    rc = check_apart(what, {{out, dtype_size(dtype), (uint64_t)rows, (uint64_t)k}},
                     {{q, 1, (uint64_t)rows, (uint64_t)k / 2}, {scales, 1, (uint64_t)rows, (uint64_t)fp4::scale_pitch(k)}});
    if (rc != TRB_OK) return rc;
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == TRB_BFLOAT16) return fp4::launch_dequantize<__nv_bfloat16>(q, scales, out, rows, k, dev, s);
    if (dtype == TRB_FLOAT16) return fp4::launch_dequantize<__half>(q, scales, out, rows, k, dev, s);
    return fp4::launch_dequantize<float>(q, scales, out, rows, k, dev, s);
}
