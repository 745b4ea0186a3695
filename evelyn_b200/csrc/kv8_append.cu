// kv8_append.cu -- new keys and values into the 8-bit paged cache, and the queries made ready
// for it: per-head RMS norm (optional), rotation by the position's row of a table (optional),
// quantisation with one scale per block of 16 positions and kv head.
//
// A block's scale is the largest |value| / 127 that the block has held since its first position
// was written. A call that brings a larger value raises the scale, and the codes of the block's
// earlier positions are moved to it: code' = rint(code * (old / new)). So a block written by one
// call holds rint(x / scale), and one filled a token at a time is off by at most one more
// rounding for each time that its scale rose.
//
// Layout: a CTA of four warps owns one (block, kv head) of K or of V, so nothing else touches the
// block's scale or codes and no atomics are needed; its rows are dealt to the warps and stay in
// registers, the maximum meets in shared memory. A lane holds four values of a row, as two pairs
// (NeoX rotation: dims 2u, 2u+1 and the same + rope_dim / 2; else four neighbours), so both
// halves of a rotated pair sit in one lane. Query rows: a warp takes four heads of a token at a
// time. Bound: HBM (each new value read once, one byte written).
//
// Norm: the sum of squares and its root are computed in 64 bits and rounded once, then x * r * w
// in f32; rotation in f32, each product and sum rounded once. So codes and scales are the same
// for every launch shape and order of summation.
#include "int8.cuh"

namespace evl {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kQHeads = 4;  // q heads a warp takes together

struct Plan {
    Kv8AppendArgs a;
    uint32_t tile;        // tokens whose blocks one CTA looks for: 1 or 16
    uint32_t kv_ctas;     // (tile, K or V, kv head)
    uint32_t q_tokens;    // consecutive tokens of a warp
    uint32_t q_items;     // (q_tokens tokens, group of q heads), a warp each, in the CTAs after those
    uint32_t q_groups, q_per;
};

// the two pairs of unit u of a row: dims lo, lo+1 and hi, hi+1
struct Unit {
    uint32_t lo, hi;
    bool turns;
};
__device__ __forceinline__ Unit unit_of(uint32_t u, uint32_t rope_dim, bool interleaved) {
    if (interleaved) return {4 * u, 4 * u + 2, 4 * u < rope_dim};
    if (4 * u < rope_dim) return {2 * u, 2 * u + rope_dim / 2, true};
    return {4 * u, 4 * u + 2, false};
}

// x * 1/rms * w of one row held by the `width` lanes of a group (N units each)
template <int N>
__device__ __forceinline__ void norm_row(float (&x)[N][4], const float (&w)[N][4], uint32_t dim, float eps,
                                         uint32_t width) {
    double ss = 0.0;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fma((double)x[n][j], (double)x[n][j], ss);
    for (uint32_t o = width / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = (float)(1.0 / sqrt(ss / (double)dim + (double)eps));
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[n][j] = __fmul_rn(__fmul_rn(x[n][j], r), w[n][j]);
}
// rotation of a unit by the table row t = (cos, sin) of its two slots
__device__ __forceinline__ void turn(float (&x)[4], const float4 t, bool interleaved) {
    auto pair = [](float& a, float& b, float c, float s) {
        const float y = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
        b = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
        a = y;
    };
    if (interleaved) {
        pair(x[0], x[1], t.x, t.y);
        pair(x[2], x[3], t.z, t.w);
    } else {
        pair(x[0], x[2], t.x, t.y);
        pair(x[1], x[3], t.z, t.w);
    }
}

// The token's sequence, checked: new tokens [q0, q1), positions base + (t - q0).
struct Seq {
    int s;
    int32_t q0, q1, base;
    bool ok;
};
__device__ __forceinline__ Seq seq_of(const Kv8AppendArgs& a, int32_t t, uint32_t lane) {
    Seq r;
    r.ok = false;
    r.s = find_seq(a.b.cu, a.b.n_seqs, t, lane);
    if (r.s < 0) return r;
    r.q0 = a.b.cu[r.s];
    r.q1 = a.b.cu[r.s + 1];
    if (t < r.q0 || t >= r.q1) return r;  // a token of no sequence: behind the last one
    const int32_t len = a.b.len[r.s];
    r.base = len - (r.q1 - r.q0);
    r.ok = r.q0 >= 0 && r.q1 <= (int32_t)a.b.total && r.q1 - r.q0 <= (int32_t)a.b.max_new && r.base >= 0 &&
           len <= (int32_t)a.b.max_len && (uint64_t)len <= (uint64_t)a.b.table_stride * a.c.page_size && (!a.rope || len <= (int32_t)a.rope_len);
    if (!r.ok && lane == 0) flag_error(a.err, DEV_ERR_POSITION);
    return r;
}

// New rows of one block: positions base + (t - q0), tokens [t, t + rows), of head h of K or V.
// Called by the whole CTA.
template <class T, int HD, bool KEY>
__device__ __forceinline__ void write_block(const Kv8AppendArgs& a, const Seq& sq, int32_t t, uint32_t rows, uint32_t h,
                                            uint32_t warp, uint32_t lane, uint32_t* red) {
    constexpr uint32_t W = HD == 64 ? 16 : 32;       // lanes per row
    constexpr uint32_t P = 32 / W;                   // rows of a warp side by side
    constexpr int N = HD / (4 * W);                  // units per lane
    constexpr uint32_t S = P * kWarps, R = 16 / S;   // rows of the CTA side by side, passes
    const uint32_t pos = (uint32_t)(sq.base + (t - sq.q0)), row0 = pos % 16;
    const uint32_t pg = pos / a.c.page_size, blk = pos % a.c.page_size / 16;
    const uint32_t sub = lane / W, u0 = lane % W, first = warp * P + sub;  // this lane's rows: first, first + S, ...
    const T* src = static_cast<const T*>(KEY ? a.k : a.v) + h * HD;
    const uint64_t stride = KEY ? a.k_stride : a.v_stride;
    Unit un[N];
#pragma unroll
    for (int n = 0; n < N; ++n) un[n] = unit_of(u0 + n * W, KEY ? a.rope_dim : 0u, KEY && a.interleaved);
    float x[R][N][4];
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
        const uint32_t i = first + r * S;
        const T* p = src + (uint64_t)(t + (int32_t)min(i, rows - 1)) * stride;
        if (r == 0 || r * S < rows)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (!KEY) {
                    load4(p + un[n].lo, x[r][n]);
                } else {
                    load2(p + un[n].lo, x[r][n][0], x[r][n][1]);
                    load2(p + un[n].hi, x[r][n][2], x[r][n][3]);
                }
            }
    }
    const int32_t page = a.b.table[(uint64_t)sq.s * a.b.table_stride + pg];
    const bool fine = (uint32_t)page < a.c.n_pages;
    if (!fine) {
        if (threadIdx.x == 0) flag_error(a.err, DEV_ERR_POSITION);
        return;  // the whole CTA
    }
    float* scale_at = (KEY ? a.c.ks : a.c.vs) + (uint64_t)page * a.c.scale_stride + h * (a.c.page_size / 16) + blk;
    int8_t* codes = (KEY ? a.c.k : a.c.v) + (uint64_t)page * a.c.page_stride +
                    ((uint64_t)h * a.c.page_size + blk * 16) * HD;
    const float old = row0 ? *scale_at : 0.f;
    float w[N][4];
    if (KEY && a.k_norm) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            w[n][0] = a.k_norm[un[n].lo], w[n][1] = a.k_norm[un[n].lo + 1];
            w[n][2] = a.k_norm[un[n].hi], w[n][3] = a.k_norm[un[n].hi + 1];
        }
    }
    uint32_t m = 0;
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
        if (r * S < rows) {
            if (KEY) {
                if (a.k_norm) norm_row<N>(x[r], w, HD, a.eps, W);
                if (a.rope) {
                    const float* tr = a.rope + (uint64_t)(pos + min(first + r * S, rows - 1)) * a.rope_dim;
#pragma unroll
                    for (int n = 0; n < N; ++n)
                        if (un[n].turns)
                            turn(x[r][n], *reinterpret_cast<const float4*>(tr + 4 * (u0 + n * W)), a.interleaved);
                }
            }
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) m = max(m, abs_bits(x[r][n][j]));
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kWarps; ++k) m = max(m, red[k]);
    const float fresh = scale_of(m);
    // a NaN on either side (a value that is not finite, now or earlier in this block) stays
    const float now = (fresh != fresh || old != old) ? __uint_as_float(0x7fc00000u) : fmaxf(old, fresh);
    const float inv = inverse_of(now);
    const bool live = now > 0.f;
    if (row0 && __float_as_uint(now) != __float_as_uint(old)) {  // the earlier rows follow the scale
        const float ratio = live ? __fdiv_rn(old, now) : 0.f;
        for (uint32_t i = first; i < row0; i += S)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                uint32_t* at = reinterpret_cast<uint32_t*>(codes + i * HD + 4 * (u0 + n * W));
                const uint32_t c = *at;
                uint32_t q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = code_bits((float)(int8_t)(c >> (8 * j)), ratio);
                *at = pack4(q[0], q[1], q[2], q[3]);
            }
    }
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
        const uint32_t i = first + r * S;
        if (i < rows) {
            int8_t* at = codes + (row0 + i) * HD;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                uint32_t q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = live ? code_bits(x[r][n][j], inv) : 0u;
                const uint32_t c = pack4(q[0], q[1], q[2], q[3]);
                if (!KEY || un[n].hi == un[n].lo + 2) {
                    *reinterpret_cast<uint32_t*>(at + un[n].lo) = c;
                } else {
                    *reinterpret_cast<uint16_t*>(at + un[n].lo) = (uint16_t)c;
                    *reinterpret_cast<uint16_t*>(at + un[n].hi) = (uint16_t)(c >> 16);
                }
            }
        }
    }
    __syncthreads();  // every warp has read the old scale (and red) by now
    if (threadIdx.x == 0) *scale_at = now;
}

// q heads [h0, h0 + n) of token t: norm, rotation, one rounding to the output type.
template <class T, int HD>
__device__ __forceinline__ void write_q(const Kv8AppendArgs& a, uint32_t pos, int32_t t, uint32_t h0, uint32_t heads,
                                        uint32_t lane) {
    constexpr uint32_t W = HD == 64 ? 16 : 32;
    constexpr int P = 32 / W, N = HD / (4 * W), R = kQHeads / P;
    const uint32_t sub = lane / W, u0 = lane % W;
    const T* src = static_cast<const T*>(a.q) + (uint64_t)t * a.q_stride;
    T* dst = static_cast<T*>(a.q_out) + (uint64_t)t * a.q_out_stride;
    Unit un[N];
#pragma unroll
    for (int n = 0; n < N; ++n) un[n] = unit_of(u0 + n * W, a.rope_dim, a.interleaved);
    float x[R][N][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T* p = src + (uint64_t)min(h0 + r * P + sub, h0 + heads - 1) * HD;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            load2(p + un[n].lo, x[r][n][0], x[r][n][1]);
            load2(p + un[n].hi, x[r][n][2], x[r][n][3]);
        }
    }
    float4 tr[N];
    float w[N][4];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (a.rope && un[n].turns)
            tr[n] = *reinterpret_cast<const float4*>(a.rope + (uint64_t)pos * a.rope_dim + 4 * (u0 + n * W));
        if (a.q_norm) {
            w[n][0] = a.q_norm[un[n].lo], w[n][1] = a.q_norm[un[n].lo + 1];
            w[n][2] = a.q_norm[un[n].hi], w[n][3] = a.q_norm[un[n].hi + 1];
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t i = r * P + sub;
        if ((uint32_t)r * P >= heads) break;
        if (a.q_norm) norm_row<N>(x[r], w, HD, a.eps, W);
        if (a.rope) {
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (un[n].turns) turn(x[r][n], tr[n], a.interleaved);
        }
        if (i < heads) {
            T* p = dst + (uint64_t)(h0 + i) * HD;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                store2(p + un[n].lo, x[r][n][0], x[r][n][1]);
                store2(p + un[n].hi, x[r][n][2], x[r][n][3]);
            }
        }
    }
}

template <class T, int HD> __global__ void __launch_bounds__(32 * kWarps, 5) kv8_append_kernel(const __grid_constant__ Plan p) {
    __shared__ uint32_t red[kWarps];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Kv8AppendArgs& a = p.a;
    if (blockIdx.x >= p.kv_ctas) {
        const uint32_t item = (blockIdx.x - p.kv_ctas) * kWarps + warp;
        if (item >= p.q_items) return;
        const uint32_t h0 = item % p.q_groups * p.q_per;
        const int32_t t0 = (int32_t)(item / p.q_groups * p.q_tokens), t1 = min(t0 + (int32_t)p.q_tokens, (int32_t)a.b.total);
        Seq sq;
        sq.q1 = t0;
        for (int32_t t = t0; t < t1; ++t) {
            if (t >= sq.q1 || t == t0) sq = seq_of(a, t, lane);
            if (sq.ok) write_q<T, HD>(a, (uint32_t)(sq.base + (t - sq.q0)), t, h0, min(p.q_per, a.heads - h0), lane);
            else sq.q1 = t;  // (look again at the next one)
        }
        return;
    }
    const uint32_t per = 2 * a.c.kv_heads, hk = blockIdx.x % per, h = hk >> 1;
    const int32_t t0 = (int32_t)(blockIdx.x / per * p.tile), t1 = min(t0 + (int32_t)p.tile, (int32_t)a.b.total);
    // the blocks whose first new token is in [t0, t1); every warp looks for itself and finds the same
    for (int32_t t = t0; t < t1;) {
        const Seq sq = seq_of(a, t, lane);
        if (!sq.ok) {
            ++t;
            continue;
        }
        const uint32_t pos = (uint32_t)(sq.base + (t - sq.q0)), row = pos % 16;
        const int32_t end = min(sq.q1, t + 16 - (int32_t)row);  // the block's new tokens end here
        if (row == 0 || t == sq.q0) {
            if (hk & 1) write_block<T, HD, false>(a, sq, t, (uint32_t)(end - t), h, warp, lane, red);
            else write_block<T, HD, true>(a, sq, t, (uint32_t)(end - t), h, warp, lane, red);
        }
        t = end;
    }
}

template <class T> cudaError_t launch(const Plan& p, cudaStream_t s) {
    const uint32_t grid = p.kv_ctas + (p.q_items + kWarps - 1) / kWarps;
    if (p.a.c.head_dim == 64) kv8_append_kernel<T, 64><<<grid, 32 * kWarps, 0, s>>>(p);
    else if (p.a.c.head_dim == 128) kv8_append_kernel<T, 128><<<grid, 32 * kWarps, 0, s>>>(p);
    else kv8_append_kernel<T, 256><<<grid, 32 * kWarps, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t s) {
    Plan p;
    p.a = a;
    // prompts: a CTA covers 16 tokens, so nearly every CTA finds one block; decoding: every
    // token starts or continues a block of its own and gets its own CTAs
    p.tile = (uint64_t)a.b.total >= 8ull * a.b.n_seqs ? 16 : 1;
    const uint64_t tiles = (a.b.total + p.tile - 1) / p.tile;
    // few tokens: one q head per warp, for the shortest chain; many: four in flight, four tokens
    // one after the other under one look at the sequence
    p.q_per = p.tile == 1 ? 1 : kQHeads;
    p.q_tokens = p.tile == 1 ? 1 : 4;
    p.q_groups = a.q ? (a.heads + p.q_per - 1) / p.q_per : 0;
    const uint64_t kv = tiles * 2 * a.c.kv_heads, q = (uint64_t)((a.b.total + p.q_tokens - 1) / p.q_tokens) * p.q_groups;
    if (kv + q > 0x7fffffffull) return cudaErrorInvalidValue;
    p.kv_ctas = (uint32_t)kv;
    p.q_items = (uint32_t)q;
    switch (a.type) {
        case GGML_F32: return launch<float>(p, s);
        case GGML_F16: return launch<__half>(p, s);
        case GGML_BF16: return launch<__nv_bfloat16>(p, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace evl
