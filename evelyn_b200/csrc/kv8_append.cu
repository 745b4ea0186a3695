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
// Layout: a CTA of eight warps owns one (block, kv head), K and V, so nothing else touches the
// block's scales or codes and no atomics are needed; its rows are dealt to the warps and stay in
// registers, the maxima meet in shared memory behind one barrier. A lane holds four values of a row, as two
// pairs (NeoX rotation: dims 2u, 2u+1 and the same + rope_dim / 2; else four neighbours), so both
// halves of a rotated pair sit in one lane. Query rows: a warp takes up to 512 / head_dim heads of up to eight
// tokens in turn. Bound: HBM (each new value read once, one byte written). Measured: four
// prompts of 5003 tokens, 16 heads and 4 kv heads of 256 dims, 94 us = 3.6 TB/s, 55 % of a copy's rate (no norm there; issue
// 60 % busy at 24 warps an SM, and the 80 registers of three CTAs make the 256-dim kernels spill, 96 bytes stored and 272
// loaded in this one; 296 us with a warp per row of the cache, 127 before the next head's rows were loaded ahead). The
// same tokens with 32 and 8 heads of 128 dims, bf16, q and k normed, NeoX pairs: 165 us for 346 MB, 103 without
// the norm: its sums in 64 bits. 32 tokens of a decode step 3.9 us, a launch and one chain of dependent loads.
//
// Norm: the sum of squares and its root are computed in 64 bits and rounded once, then x * r * w
// in f32; rotation in f32, each product and sum rounded once. So codes and scales are the same
// for every launch shape and order of summation.
#include "int8.cuh"

namespace evl {
namespace {

constexpr uint32_t kWarps = 8;
// q heads that a warp takes together: 16 values per lane
__host__ __device__ constexpr int q_heads(int head_dim) { return 512 / head_dim; }

struct Plan {
    Kv8AppendArgs a;
    uint32_t tile;        // tokens whose blocks one CTA looks for: 1 or 16
    uint32_t kv_per;      // kv heads of a CTA
    uint32_t kv_ctas;     // (tile, group of kv heads)
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

// FOUR: every unit is four neighbours (no rotation, or interleaved pairs) and moves in one piece. Units are
// kept as they were loaded and widened where they are used: a conversion beside the load would wait
// for it before the next load is issued.
template <class T> struct Raw {
    uint32_t w[sizeof(T)];  // four values
};
template <bool FOUR, class T> __device__ __forceinline__ void load_unit(const T* p, const Unit& u, Raw<T>& x) {
    if constexpr (FOUR && sizeof(T) == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p + u.lo);
        x.w[0] = v.x, x.w[1] = v.y, x.w[2] = v.z, x.w[3] = v.w;
    } else if constexpr (FOUR) {
        const uint2 v = *reinterpret_cast<const uint2*>(p + u.lo);
        x.w[0] = v.x, x.w[1] = v.y;
    } else if constexpr (sizeof(T) == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p + u.lo), z = *reinterpret_cast<const uint2*>(p + u.hi);
        x.w[0] = v.x, x.w[1] = v.y, x.w[2] = z.x, x.w[3] = z.y;
    } else {
        x.w[0] = *reinterpret_cast<const uint32_t*>(p + u.lo);
        x.w[1] = *reinterpret_cast<const uint32_t*>(p + u.hi);
    }
}
template <class T> __device__ __forceinline__ void widen(const Raw<T>& r, float (&x)[4]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(r.w[j]);
    } else {
        unpack2(r.w[0], T{}, x[0], x[1]);
        unpack2(r.w[1], T{}, x[2], x[3]);
    }
}
template <bool FOUR, class T> __device__ __forceinline__ void store_unit(T* p, const Unit& u, const float (&x)[4]) {
    if constexpr (FOUR) {
        store4(p + u.lo, x);
    } else {
        store2(p + u.lo, x[0], x[1]);
        store2(p + u.hi, x[2], x[3]);
    }
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

// New rows of a block: tokens [t, t + rows) at positions from pos, in a page that is there.
struct Job {
    int32_t t;
    uint32_t rows, pos;
    uint64_t codes, scale;  // of kv head 0 of the block
};

// The rows of one (block, kv head) of K or of V that a thread of the CTA holds.
template <class T, int HD, bool FOUR, bool KEY> struct Rows {
    static constexpr uint32_t W = HD == 64 ? 16 : 32;     // lanes per row
    static constexpr uint32_t P = 32 / W;                 // rows of a warp side by side
    static constexpr int N = HD / (4 * W);                // units per lane
    static constexpr uint32_t S = P * kWarps, R = 16 / S;  // rows of the CTA side by side, passes
    Raw<T> raw[R][N];  // on their way, of the head that comes next
    float coming;      // and its block's scale
    float x[R][N][4];
    float4 tr[R][N];
    float old;

    __device__ __forceinline__ static Unit unit(const Kv8AppendArgs& a, uint32_t u) {
        return unit_of(u, KEY ? a.rope_dim : 0u, KEY && a.interleaved);
    }
    // whether pass r has a row for this warp
    __device__ __forceinline__ static bool some(uint32_t r, uint32_t rows) { return (threadIdx.x >> 5) * P + r * S < rows; }
    __device__ __forceinline__ void load(const Kv8AppendArgs& a, const Job& b, uint32_t h, uint32_t first, uint32_t u0) {
        const T* src = static_cast<const T*>(KEY ? a.k : a.v) + h * HD;
        const uint64_t stride = KEY ? a.k_stride : a.v_stride;
#pragma unroll
        for (uint32_t r = 0; r < R; ++r) {
            const uint32_t i = min(first + r * S, b.rows - 1);
            const T* p = src + (uint64_t)(b.t + (int32_t)i) * stride;
#pragma unroll
            for (int n = 0; n < N; ++n) load_unit<FOUR || !KEY>(p, unit(a, u0 + n * W), raw[r][n]);
        }
        coming = b.pos % 16 ? (KEY ? a.c.ks : a.c.vs)[b.scale + h * (a.c.page_size / 16)] : 0.f;
    }
    // the table rows of the block's positions, for all heads
    __device__ __forceinline__ void load_turns(const Kv8AppendArgs& a, const Job& b, uint32_t first, uint32_t u0) {
        if (!KEY || !a.rope) return;
#pragma unroll
        for (uint32_t r = 0; r < R; ++r)
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (unit(a, u0 + n * W).turns)
                    tr[r][n] = *reinterpret_cast<const float4*>(
                        a.rope + (uint64_t)(b.pos + min(first + r * S, b.rows - 1)) * a.rope_dim + 4 * (u0 + n * W));
    }
    // what load() brought becomes the current head
    __device__ __forceinline__ void take() {
        old = coming;
#pragma unroll
        for (uint32_t r = 0; r < R; ++r)
#pragma unroll
            for (int n = 0; n < N; ++n) widen(raw[r][n], x[r][n]);
    }
    // norm, rotation; the largest magnitude of the warp's rows
    __device__ __forceinline__ uint32_t ready(const Kv8AppendArgs& a, uint32_t rows, uint32_t u0) {
        if (KEY && a.k_norm) {
            float w[N][4];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const Unit u = unit(a, u0 + n * W);
                w[n][0] = a.k_norm[u.lo], w[n][1] = a.k_norm[u.lo + 1];
                w[n][2] = a.k_norm[u.hi], w[n][3] = a.k_norm[u.hi + 1];
            }
#pragma unroll
            for (uint32_t r = 0; r < R; ++r)
                if (some(r, rows)) norm_row<N>(x[r], w, HD, a.eps, W);
        }
        uint32_t m = 0;
#pragma unroll
        for (uint32_t r = 0; r < R; ++r)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (!some(r, rows)) continue;
                if (KEY && a.rope && unit(a, u0 + n * W).turns) turn(x[r][n], tr[r][n], a.interleaved);
#pragma unroll
                for (int j = 0; j < 4; ++j) m = max(m, abs_bits(x[r][n][j]));
            }
        return __reduce_max_sync(0xffffffffu, m);
    }
    // codes and scale, m the largest magnitude of all rows
    __device__ __forceinline__ void write(const Kv8AppendArgs& a, const Job& b, uint32_t h, uint32_t first, uint32_t u0,
                                          uint32_t m) {
        const uint32_t row0 = b.pos % 16;
        const float fresh = scale_of(m);
        // a NaN on either side (a value that is not finite, now or earlier in this block) stays
        const float now = (fresh != fresh || old != old) ? __uint_as_float(0x7fc00000u) : fmaxf(old, fresh);
        const float inv = inverse_of(now);
        const bool live = now > 0.f;
        int8_t* codes = (KEY ? a.c.k : a.c.v) + b.codes + (uint64_t)h * a.c.page_size * HD;
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
        // (every thread read the old scale before the barrier)
        if (threadIdx.x == 0) (KEY ? a.c.ks : a.c.vs)[b.scale + h * (a.c.page_size / 16)] = now;
#pragma unroll
        for (uint32_t r = 0; r < R; ++r) {
            const uint32_t i = first + r * S;
            if (i < b.rows) {
                int8_t* at = codes + (row0 + i) * HD;
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const Unit u = unit(a, u0 + n * W);
                    uint32_t q[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) q[j] = live ? code_bits(x[r][n][j], inv) : 0u;
                    const uint32_t c = pack4(q[0], q[1], q[2], q[3]);
                    if constexpr (FOUR || !KEY) {
                        *reinterpret_cast<uint32_t*>(at + u.lo) = c;
                    } else {
                        *reinterpret_cast<uint16_t*>(at + u.lo) = (uint16_t)c;
                        *reinterpret_cast<uint16_t*>(at + u.hi) = (uint16_t)(c >> 16);
                    }
                }
            }
        }
    }
};

// q heads [h0, h0 + heads) of tokens [t0, t1): norm, rotation, one rounding to the output type. A
// token's rows are on their way while the one before is written, and the sequence is looked up only
// where one ends.
template <class T, int HD, bool FOUR>
__device__ __forceinline__ void write_q(const Kv8AppendArgs& a, int32_t t0, int32_t t1, uint32_t h0, uint32_t heads,
                                        uint32_t lane) {
    constexpr uint32_t W = HD == 64 ? 16 : 32;
    constexpr int P = 32 / W, N = HD / (4 * W), R = q_heads(HD) / P;
    const uint32_t sub = lane / W, u0 = lane % W;
    Unit un[N];
#pragma unroll
    for (int n = 0; n < N; ++n) un[n] = unit_of(u0 + n * W, a.rope_dim, a.interleaved);
    auto load = [&](Raw<T>(&x)[R][N], int32_t t) {
        const T* src = static_cast<const T*>(a.q) + (uint64_t)t * a.q_stride;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const T* p = src + (uint64_t)min(h0 + r * P + sub, h0 + heads - 1) * HD;
#pragma unroll
            for (int n = 0; n < N; ++n) load_unit<FOUR>(p, un[n], x[r][n]);
        }
    };
    Raw<T> next[R][N];
    load(next, t0);
    float w[N][4];
    if (a.q_norm) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            w[n][0] = a.q_norm[un[n].lo], w[n][1] = a.q_norm[un[n].lo + 1];
            w[n][2] = a.q_norm[un[n].hi], w[n][3] = a.q_norm[un[n].hi + 1];
        }
    }
    Seq sq = seq_of(a, t0, lane);
    float4 tr[N], tr_next[N];
    auto load_turns = [&](float4(&r)[N], const Seq& q, int32_t t) {
        if (!q.ok || !a.rope) return;
        const float* row = a.rope + (uint64_t)(q.base + (t - q.q0)) * a.rope_dim;
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (un[n].turns) r[n] = *reinterpret_cast<const float4*>(row + 4 * (u0 + n * W));
    };
    load_turns(tr, sq, t0);
    for (int32_t t = t0;; ++t) {
        float x[R][N][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int n = 0; n < N; ++n) widen(next[r][n], x[r][n]);
        const bool same = sq.ok && t + 1 < min(sq.q1, t1);  // the next token is this sequence's too
        if (t + 1 < t1) load(next, t + 1);
        if (same) load_turns(tr_next, sq, t + 1);
        if (sq.ok) {
            T* dst = static_cast<T*>(a.q_out) + (uint64_t)t * a.q_out_stride;
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
#pragma unroll
                    for (int n = 0; n < N; ++n) store_unit<FOUR>(dst + (uint64_t)(h0 + i) * HD, un[n], x[r][n]);
                }
            }
        }
        if (t + 1 >= t1) break;
        if (same) {
#pragma unroll
            for (int n = 0; n < N; ++n) tr[n] = tr_next[n];
        } else {
            sq = seq_of(a, t + 1, lane);
            load_turns(tr, sq, t + 1);
        }
    }
}

template <class T, int HD, bool FOUR>
__global__ void __launch_bounds__(32 * kWarps, 3) kv8_append_kernel(const __grid_constant__ Plan p) {
    __shared__ uint2 red[2][kWarps];
    uint32_t turn_no = 0;  // (two sets of maxima, so that one barrier per block is enough)
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Kv8AppendArgs& a = p.a;
    pdl_wait();
    // (no pdl_launch_dependents: the attention's CTAs would take their places while these run, three beside one
    // another where there is room first -- a layer's step of 32 sequences 76 us against 64)
    if (blockIdx.x >= p.kv_ctas) {
        const uint32_t item = (blockIdx.x - p.kv_ctas) * kWarps + warp;
        if (item >= p.q_items) return;
        const uint32_t h0 = item % p.q_groups * p.q_per;
        const int32_t t0 = (int32_t)(item / p.q_groups * p.q_tokens);
        write_q<T, HD, FOUR>(a, t0, min(t0 + (int32_t)p.q_tokens, (int32_t)a.b.total), h0, min(p.q_per, a.heads - h0), lane);
        return;
    }
    using Keys = Rows<T, HD, FOUR, true>;
    using Values = Rows<T, HD, FOUR, false>;
    const uint32_t groups = (a.c.kv_heads + p.kv_per - 1) / p.kv_per, h0 = blockIdx.x % groups * p.kv_per;
    const uint32_t h1 = min(h0 + p.kv_per, a.c.kv_heads), tile = blockIdx.x / groups;
    const int32_t t0 = (int32_t)(tile * p.tile), t1 = min(t0 + (int32_t)p.tile, (int32_t)a.b.total);
    const uint32_t u0 = lane % Keys::W, first = warp * Keys::P + lane / Keys::W;
    // the blocks whose first new token is in [t0, t1); every warp looks for itself and finds the same
    for (int32_t t = t0; t < t1;) {
        const Seq sq = seq_of(a, t, lane);
        if (!sq.ok) {
            ++t;
            continue;
        }
        Job b;
        b.t = t;
        b.pos = (uint32_t)(sq.base + (t - sq.q0));
        const int32_t end = min(sq.q1, t + 16 - (int32_t)(b.pos % 16));  // the block's new tokens end here
        b.rows = (uint32_t)(end - t);
        t = end;
        if (b.pos % 16 && b.t != sq.q0) continue;  // (an earlier CTA's)
        const int32_t page = a.b.table[(uint64_t)sq.s * a.b.table_stride + b.pos / a.c.page_size];
        if ((uint32_t)page >= a.c.n_pages) {
            if (threadIdx.x == 0) flag_error(a.err, DEV_ERR_POSITION);
            continue;
        }
        const uint32_t blk = b.pos % a.c.page_size / 16;
        b.codes = (uint64_t)page * a.c.page_stride + (uint64_t)blk * 16 * HD;
        b.scale = (uint64_t)page * a.c.scale_stride + blk;
        Keys k;
        Values v;
        k.load(a, b, h0, first, u0);
        v.load(a, b, h0, first, u0);
        k.load_turns(a, b, first, u0);
        for (uint32_t h = h0; h < h1; ++h) {
            k.take();
            v.take();
            if (h + 1 < h1) {  // the next head's rows on their way meanwhile
                k.load(a, b, h + 1, first, u0);
                v.load(a, b, h + 1, first, u0);
            }
            uint2 m = make_uint2(k.ready(a, b.rows, u0), v.ready(a, b.rows, u0));
            if (lane == 0) red[turn_no & 1][warp] = m;
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < kWarps; ++i) {
                const uint2 o = red[turn_no & 1][i];
                m.x = max(m.x, o.x), m.y = max(m.y, o.y);
            }
            ++turn_no;
            k.write(a, b, h, first, u0, m.x);
            v.write(a, b, h, first, u0, m.y);
        }
    }
}

template <class T, int HD, bool FOUR> cudaError_t launch(const Plan& p, cudaStream_t s) {
    return launch_chained(kv8_append_kernel<T, HD, FOUR>, p.kv_ctas + (p.q_items + kWarps - 1) / kWarps, 32 * kWarps, 0, s, p);
}
template <class T, bool FOUR> cudaError_t by_dim(const Plan& p, cudaStream_t s) {
    return p.a.c.head_dim == 64    ? launch<T, 64, FOUR>(p, s)
           : p.a.c.head_dim == 128 ? launch<T, 128, FOUR>(p, s)
                                   : launch<T, 256, FOUR>(p, s);
}
template <class T> cudaError_t by_layout(const Plan& p, cudaStream_t s) {
    return p.a.interleaved || !p.a.rope ? by_dim<T, true>(p, s) : by_dim<T, false>(p, s);
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, int sms, cudaStream_t s) {
    Plan p;
    p.a = a;
    // prompts: a CTA covers 16 tokens, so nearly every CTA finds one block; decoding: every
    // token starts or continues a block of its own and gets its own CTAs
    p.tile = (uint64_t)a.b.total >= 8ull * a.b.n_seqs ? 16 : 1;
    const uint64_t tiles = (a.b.total + p.tile - 1) / p.tile;
    // queries: several heads and then several tokens per warp (one look at the sequence, the next rows
    // on their way), as long as the warps still fill the SMs twice (24 at a time on each)
    const uint64_t fill = 48ull * sms, rows = (uint64_t)a.b.total * a.heads;
    p.q_per = p.q_tokens = 1;
    while ((int)p.q_per < q_heads((int)a.c.head_dim) && rows / (2 * p.q_per) >= fill) p.q_per *= 2;
    while (p.q_tokens < 8 && rows / p.q_per / (2 * p.q_tokens) >= fill) p.q_tokens *= 2;
    p.q_groups = a.q ? (a.heads + p.q_per - 1) / p.q_per : 0;
    // kv heads one after the other in a CTA while the grid still covers the SMs four times
    p.kv_per = 1;
    while (p.kv_per < a.c.kv_heads && tiles * ((a.c.kv_heads + 2 * p.kv_per - 1) / (2 * p.kv_per)) >= 4ull * sms) p.kv_per *= 2;
    const uint64_t kv = tiles * ((a.c.kv_heads + p.kv_per - 1) / p.kv_per), q = (uint64_t)((a.b.total + p.q_tokens - 1) / p.q_tokens) * p.q_groups;
    if (kv + q > 0x7fffffffull) return cudaErrorInvalidValue;
    p.kv_ctas = (uint32_t)kv;
    p.q_items = (uint32_t)q;
    switch (a.type) {
        case GGML_F32: return by_layout<float>(p, s);
        case GGML_F16: return by_layout<__half>(p, s);
        case GGML_BF16: return by_layout<__nv_bfloat16>(p, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace evl
