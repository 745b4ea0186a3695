// int8_rows.cu -- activation rows in 8 bits with one scale each, the left operand of the
// integer product (int8_gemm.cu):
//   a = max |x|, scale = a / 127, code = rint(x * (1 / scale)).
// The row is read once into registers, its largest magnitude found as an integer maximum of
// the absolute bits (which also finds an infinity or a NaN), and the codes written: input
// bytes + one byte per value is all the traffic, so the kernel is bound by HBM. f32 throughout;
// the products and the reciprocal are each rounded once, so the codes do not depend on the
// launch shape. Measured: 8192 rows of 12288 bf16 values 47 us = 6.4 TB/s, 97 % of a copy's rate; one row
// of 4096 in 1.3 us, a launch; 8192 x 12287 (rows at odd offsets, staged) 81 us.
#include <atomic>

#include "int8.cuh"

namespace evl {
namespace {

constexpr uint32_t kChunk = 8;  // values a thread loads together: one or two 16-byte loads, one 8-byte store

__device__ __forceinline__ uint32_t block_umax(uint32_t v, uint32_t* red) {
    v = __reduce_max_sync(0xffffffffu, v);
    const uint32_t warps = blockDim.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const uint32_t lane = threadIdx.x & 31;
    return __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
}

// One CTA per row, C chunks per thread, kept as they were loaded: no load waits for a conversion or
// stands behind a condition, so all are on their way together. The values after the last whole chunk
// are one more per thread.
template <class T> struct Chunk {
    uint4 w[sizeof(T) / 2];  // kChunk values
};
template <class T> __device__ __forceinline__ void widen(const Chunk<T>& c, float (&v)[kChunk]) {
    if constexpr (sizeof(T) == 4) {
        const uint4 a = c.w[0], b = c.w[1];
        v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y), v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
        v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y), v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
    } else {
        unpack2(c.w[0].x, T{}, v[0], v[1]);
        unpack2(c.w[0].y, T{}, v[2], v[3]);
        unpack2(c.w[0].z, T{}, v[4], v[5]);
        unpack2(c.w[0].w, T{}, v[6], v[7]);
    }
}
template <class T, int C> __global__ void __launch_bounds__(1024) quantize_rows_kernel(const QuantRowsArgs a) {
    __shared__ uint32_t red[32];
    pdl_wait();
    pdl_launch_dependents();
    const uint64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    int8_t* codes = a.codes + row * a.code_stride;
    const uint32_t chunks = a.cols / kChunk, tail = a.cols % kChunk, nt = blockDim.x;
    Chunk<T> raw[C];
    T last{};
    if (chunks) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const uint4* p = reinterpret_cast<const uint4*>(x + (uint64_t)min(threadIdx.x + i * nt, chunks - 1) * kChunk);
#pragma unroll
            for (uint32_t j = 0; j < sizeof(T) / 2; ++j) raw[i].w[j] = ldg_nc(p + j);
        }
    } else {
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (uint32_t j = 0; j < sizeof(T) / 2; ++j) raw[i].w[j] = make_uint4(0, 0, 0, 0);
    }
    if (threadIdx.x < tail) last = x[(uint64_t)chunks * kChunk + threadIdx.x];
    // (a thread past the end holds the last chunk again: the maximum is the same)
    uint32_t m = threadIdx.x < tail ? abs_bits(to_f32(last)) : 0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        float v[kChunk];
        widen(raw[i], v);
#pragma unroll
        for (uint32_t j = 0; j < kChunk; ++j) m = max(m, abs_bits(v[j]));
    }
    m = block_umax(m, red);
    const float scale = scale_of(m), inv = inverse_of(scale);
    if (threadIdx.x == 0) a.scales[row] = scale;
    const bool live = scale > 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const uint32_t c = threadIdx.x + i * nt;
        if (c >= chunks) break;
        float v[kChunk];
        uint32_t q[kChunk];
        widen(raw[i], v);
#pragma unroll
        for (uint32_t j = 0; j < kChunk; ++j) q[j] = live ? code_bits(v[j], inv) : 0u;
        *reinterpret_cast<uint2*>(codes + (uint64_t)c * kChunk) =
            make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
    }
    if (threadIdx.x < tail) codes[(uint64_t)chunks * kChunk + threadIdx.x] = live ? (int8_t)code_bits(to_f32(last), inv) : (int8_t)0;
}

// Rows that do not start on the boundaries of wide loads (an odd row length, a view), and rows too long
// for registers: the row is staged in shared memory in the 16-byte granules of its global addresses
// (asynchronous copies; the values before the first and after the last whole granule one by one, the
// rest of those granules zero). The maximum is taken granule by granule; eight values of a chunk come
// from the two (f32: three) granules that hold them, moved by the row's offset.
template <class T> __global__ void __launch_bounds__(512) quantize_rows_staged_kernel(const QuantRowsArgs a) {
    extern __shared__ __align__(16) uint8_t row_smem[];
    __shared__ uint32_t red[32];
    pdl_wait();
    pdl_launch_dependents();
    constexpr uint32_t ES = sizeof(T), NW = kChunk * ES / 4;  // words of a chunk
    const uint64_t row = blockIdx.x;
    const uint8_t* x = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.x) + row * a.x_stride);
    int8_t* codes = a.codes + row * a.code_stride;
    const uint32_t sh = (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15), bytes = a.cols * ES;
    const uint32_t g0 = sh ? 1 : 0, g1 = (sh + bytes) / 16;       // whole granules [g0, g1)
    const uint32_t granules = (sh + bytes + 15) / 16 + 2;         // with two of zeros, which a last chunk may reach into
    const uint32_t tid = threadIdx.x, nt = blockDim.x;
    for (uint32_t g = tid; g < granules; g += nt) {
        if (g >= g0 && g < g1)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(row_smem + 16 * g)), "l"(x + 16 * g - sh) : "memory");
        else
            *reinterpret_cast<uint4*>(row_smem + 16 * g) = make_uint4(0, 0, 0, 0);
    }
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    // the values of a first and a last granule that are not whole
    const uint32_t head = g0 ? min(16 - sh, bytes) / ES : 0;               // elements before the first whole granule
    const uint32_t from = max(head, g1 > g0 ? (16 * g1 - sh) / ES : head);  // and from here on
    if (tid < head) reinterpret_cast<T*>(row_smem + sh)[tid] = reinterpret_cast<const T*>(x)[tid];
    if (from + tid < a.cols) reinterpret_cast<T*>(row_smem + sh)[from + tid] = reinterpret_cast<const T*>(x)[from + tid];
    __syncthreads();
    uint32_t m = 0;
    for (uint32_t g = tid; g < granules; g += nt) {
        const uint4 w = *reinterpret_cast<const uint4*>(row_smem + 16 * g);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (ES == 4) {
                m = max(m, v[j] & 0x7fffffffu);
            } else {
                float p, q;
                unpack2(v[j], T{}, p, q);
                m = max(m, max(abs_bits(p), abs_bits(q)));
            }
        }
    }
    m = block_umax(m, red);
    const float scale = scale_of(m), inv = inverse_of(scale);
    if (tid == 0) a.scales[row] = scale;
    const bool live = scale > 0.f;
    const bool wide = (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    const uint32_t chunks = (a.cols + kChunk - 1) / kChunk, bits = 8 * (sh & 3);
    for (uint32_t c = tid; c < chunks; c += nt) {
        uint32_t w[NW + 4], v[NW];
#pragma unroll
        for (uint32_t j = 0; j < NW + 4; j += 4) {
            const uint4 g = *reinterpret_cast<const uint4*>(row_smem + c * (kChunk * ES) + 4 * j);
            w[j] = g.x, w[j + 1] = g.y, w[j + 2] = g.z, w[j + 3] = g.w;
        }
        auto move = [&](auto at) {
#pragma unroll
            for (uint32_t j = 0; j < NW; ++j) v[j] = __funnelshift_r(w[at + j], j + at + 1 < NW + 4 ? w[at + j + 1] : 0u, bits);
        };
        switch (sh >> 2) {  // (the same for the whole row)
            case 0: move(std::integral_constant<uint32_t, 0>{}); break;
            case 1: move(std::integral_constant<uint32_t, 1>{}); break;
            case 2: move(std::integral_constant<uint32_t, 2>{}); break;
            default: move(std::integral_constant<uint32_t, 3>{}); break;
        }
        float f[kChunk];
        uint32_t q[kChunk];
#pragma unroll
        for (uint32_t j = 0; j < kChunk; j += 4 / ES) {
            if constexpr (ES == 4) f[j] = __uint_as_float(v[j]);
            else unpack2(v[j / 2], T{}, f[j], f[j + 1]);
        }
#pragma unroll
        for (uint32_t j = 0; j < kChunk; ++j) q[j] = live ? code_bits(f[j], inv) : 0u;
        const uint32_t left = a.cols - c * kChunk;
        if (wide && left >= kChunk) {
            *reinterpret_cast<uint2*>(codes + (uint64_t)c * kChunk) =
                make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
        } else {
#pragma unroll
            for (uint32_t j = 0; j < kChunk; ++j)
                if (j < left) codes[(uint64_t)c * kChunk + j] = (int8_t)q[j];
        }
    }
}

// Rows that do not fit into shared memory: values one by one, neighbouring threads on neighbouring values,
// the row read a second time from L2.
template <class T> __global__ void __launch_bounds__(512) quantize_rows_long_kernel(const QuantRowsArgs a) {
    __shared__ uint32_t red[32];
    pdl_wait();
    pdl_launch_dependents();
    const uint64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    int8_t* codes = a.codes + row * a.code_stride;
    uint32_t m = 0;
#pragma unroll 8
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) m = max(m, abs_bits(to_f32(x[c])));
    m = block_umax(m, red);
    const float scale = scale_of(m), inv = inverse_of(scale);
    if (threadIdx.x == 0) a.scales[row] = scale;
    const bool live = scale > 0.f;
#pragma unroll 8
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x)
        codes[c] = live ? (int8_t)code_bits(to_f32(x[c]), inv) : (int8_t)0;
}

// shared memory of a staged row, and the most that a CTA may have
inline uint64_t staged_bytes(uint64_t row_bytes) { return row_bytes + 16 + 48; }
constexpr uint32_t kStagedCap = 200 * 1024;
template <auto kernel> cudaError_t opt_in(uint32_t smem) {
    static std::atomic<bool> done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (done[dev].load()) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) done[dev] = true;
    return e;
}

template <class T> cudaError_t launch(const QuantRowsArgs& a, int sms, cudaStream_t s) {
    const bool aligned = (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && (a.x_stride * sizeof(T)) % 16 == 0 &&
                         (reinterpret_cast<uintptr_t>(a.codes) & 7) == 0 && a.code_stride % 8 == 0;
    const uint32_t chunks = (a.cols + kChunk - 1) / kChunk;
    if (!aligned || chunks > 4 * 1024) {
        const uint64_t smem = staged_bytes((uint64_t)a.cols * sizeof(T));
        const uint32_t nt = a.cols >= 8192 ? 512 : a.cols >= 1024 ? 256 : 64;
        if (smem > kStagedCap) {
            return launch_chained(quantize_rows_long_kernel<T>, a.rows, 512, 0, s, a);
        }
        if (const cudaError_t e = opt_in<quantize_rows_staged_kernel<T>>(kStagedCap)) return e;
        return launch_chained(quantize_rows_staged_kernel<T>, a.rows, nt, (uint32_t)smem, s, a);
    }
    // few rows: as many threads as chunks, so that a row is one load deep; many rows: four
    // chunks per thread, all in flight, and more rows on each SM
    const int C = (a.rows <= (uint32_t)(2 * sms) && chunks <= 1024) ? 1 : chunks > 2048 || a.rows > (uint32_t)(2 * sms) ? 4 : 2;
    const uint32_t nt = ((chunks + C - 1) / C + 31) / 32 * 32;
    return launch_chained(C == 1 ? quantize_rows_kernel<T, 1> : C == 2 ? quantize_rows_kernel<T, 2> : quantize_rows_kernel<T, 4>,
                          a.rows, nt, 0, s, a);
}

}  // namespace

cudaError_t launch_quantize_rows(const QuantRowsArgs& a, int sms, cudaStream_t s) {
    switch (a.type) {
        case GGML_F32: return launch<float>(a, sms, s);
        case GGML_F16: return launch<__half>(a, sms, s);
        case GGML_BF16: return launch<__nv_bfloat16>(a, sms, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace evl
