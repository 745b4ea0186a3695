// kv8_attention.cu -- attention of new tokens over the 8-bit paged cache.
//
// o = sum_j softmax_j(scale * q . (sk_j ck_j)) sv_j cv_j over the positions j that the token
// sees, with 8-bit codes c and one scale s per block of 16 positions and kv head. The scales are
// constant over a block, so they leave the products: scores are integer products times one
// factor per block, and the value scale joins the softmax weight. One pass over the cache with
// a running maximum M and sum, all in the exponent's base 2:
//   x = q . ck (an integer) * (sk * scale * log2 e * step of q) + e,  e = exponent of sv
//   w = 2^(x - M),  l += w * 2^-e,  O += (w * sv 2^-e) * cv,  o = O / l
// so w times a mantissa in [1, 2) meets the codes, whatever the size of the value scale, and
// the power of two leaves the sum exactly.
//
// Small-batch kernel (kv8_split_kernel): up to 8 rows (token, head) per CTA that share a kv head;
// positions are the M dimension of the warp's products.
//   K: mma.sync m16n8k32 on the codes as they are. q is fixed point in three signed 8-bit limbs
//      (22 bits below the row's largest magnitude), the integer products are exact, so a score
//      is as good as an f32 dot product. The K order inside the product is permuted so that a
//      lane's fragment is 16 neighbouring bytes of a row: codes go from HBM to registers to the
//      tensor cores, with no shared memory and no conversion.
//   V: mma.sync m16n8k16 in f16: codes are exact in f16, the weights two f16 parts (22 bits).
//      A lane loads 16 neighbouring dims of four positions and pairs positions with byte
//      permutes; the weights move to the other operand's layout by two 8x8 transposes.
//   The maximum is raised only when a score passes it by 2^8, so most blocks cost one vote.
// A warp takes every 4th block of the CTA's chunk of positions, the next block's codes already
// in flight in registers. The warps' partials meet in shared memory; a sequence of more than one
// chunk leaves (O, M, l) in the workspace for kv8_join_kernel.
// Bound: HBM, (2 head_dim + 1/2) bytes per position and kv head.
#include <algorithm>

#include "int8.cuh"

namespace evl {
namespace {

constexpr uint32_t kRows = 8;     // rows of a tile (the product's N)
constexpr uint32_t kWarps = 4;
constexpr float kNegBig = -1e38f;  // a maximum that no score has reached
constexpr float kSlack = 8.f;      // weights stay below 2^8 (times a mantissa below 2: far inside f16)

struct Plan {
    Kv8AttnArgs a;
    uint32_t group;      // q heads per kv head
    uint32_t row_tiles;  // per (sequence, kv head)
    uint32_t chunk;      // blocks of 16 positions per split
    uint32_t splits;
    float* part_o;       // [sequence][kv head][row tile][split][kRows][head_dim]
    float2* part_ml;     // same without head_dim: (M, l)
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// bytes 0, 1 (or 2, 3) of w, biased codes c + 128, as an exact f16 pair: 0x6400 | b is 1024 + b
__device__ __forceinline__ uint32_t codes_h2(uint32_t w, uint32_t sel) {
    const uint32_t h = __byte_perm(w, 0x64646464u, sel), bias = 0x64806480u;  // 1024 + 128
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}

// What a tile attends: its sequence's length and the last position of each of its rows.
struct Span {
    int32_t q0, n_new, base;  // first token, tokens, position of the first one
    bool ok;
};
__device__ __forceinline__ Span span_of(const Kv8AttnArgs& a, uint32_t s) {
    Span r;
    r.q0 = a.b.cu[s];
    const int32_t q1 = a.b.cu[s + 1], len = a.b.len[s];
    r.n_new = q1 - r.q0;
    r.base = len - r.n_new;
    r.ok = r.q0 >= 0 && q1 >= r.q0 && q1 <= (int32_t)a.b.total && r.n_new <= (int32_t)a.b.max_new && len >= 0 &&
           len <= (int32_t)a.b.max_len && (uint64_t)len <= (uint64_t)a.b.table_stride * a.c.page_size;
    return r;
}

// The codes and scales of one block of 16 positions for one lane.
template <int HD> struct Block {
    uint32_t k[HD / 64][2][4];                       // rows g, g + 8: 16 bytes at 64 c + 16 t
    uint32_t v[HD <= 128 ? 1 : 2][4][HD < 128 ? 2 : 4];  // positions 2t, 2t+1, 2t+8, 2t+9: 16 (8) bytes of dims
    float sk, sv;
};
template <int HD>
__device__ __forceinline__ void load_block(Block<HD>& b, const Kv8Cache& c, int32_t page, uint32_t sub, uint32_t h,
                                           uint32_t g, uint32_t t) {
    const uint64_t row = (uint64_t)page * c.page_stride + ((uint64_t)h * c.page_size + sub * 16) * HD;
    const int8_t *k = c.k + row, *v = c.v + row;
    const uint64_t sc = (uint64_t)page * c.scale_stride + h * (c.page_size / 16) + sub;
    b.sk = __ldg(c.ks + sc);
    b.sv = __ldg(c.vs + sc);
#pragma unroll
    for (int i = 0; i < HD / 64; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint4 w = ldg_nc(k + (g + 8 * r) * HD + 64 * i + 16 * t);
            b.k[i][r][0] = w.x, b.k[i][r][1] = w.y, b.k[i][r][2] = w.z, b.k[i][r][3] = w.w;
        }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int8_t* at = v + (2 * t + (p & 1) + (p >> 1) * 8) * HD;
        if constexpr (HD == 64) {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(at + 8 * g));
            b.v[0][p][0] = w.x, b.v[0][p][1] = w.y;
        } else {
#pragma unroll
            for (int i = 0; i < HD / 128; ++i) {
                const uint4 w = ldg_nc(at + 128 * i + 16 * g);
                b.v[i][p][0] = w.x, b.v[i][p][1] = w.y, b.v[i][p][2] = w.z, b.v[i][p][3] = w.w;
            }
        }
    }
}

template <class T, int HD>
__global__ void __launch_bounds__(32 * kWarps) kv8_split_kernel(const __grid_constant__ Plan P) {
    constexpr int KC = HD / 64;                  // 64-dim chunks of the score product
    constexpr int VW = HD < 128 ? 2 : 4;         // words of a V load
    constexpr int VC = HD <= 128 ? 1 : 2;        // V loads per position
    constexpr int MT = HD / 16;                  // 16-dim tiles of the output
    constexpr int LD = HD / 8 < 16 ? HD / 8 : 16;  // neighbouring dims of a lane's load
    __shared__ float so[kWarps][kRows][HD];
    __shared__ float2 sml[kWarps][kRows];
    const Kv8AttnArgs& a = P.a;
    const uint32_t split = blockIdx.x, h = blockIdx.y % a.c.kv_heads, tile = blockIdx.y / a.c.kv_heads, s = blockIdx.z;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const Span sp = span_of(a, s);
    if (!sp.ok) {
        if (tid == 0) flag_error(a.err, DEV_ERR_POSITION);
        return;
    }
    const int32_t rows = sp.n_new * (int32_t)P.group, r0 = (int32_t)(tile * kRows);
    if (r0 >= rows) return;
    const int32_t nrow = min((int32_t)kRows, rows - r0);
    // positions [0, seen) are seen by the tile's last row
    const int32_t seen = sp.base + (r0 + nrow - 1) / (int32_t)P.group + 1;
    const int32_t nblk = seen > 0 ? (seen + 15) / 16 : 0;
    const int32_t b0 = (int32_t)(split * P.chunk), b1 = min(nblk, b0 + (int32_t)P.chunk);
    if (b0 >= nblk && split > 0) return;  // (split 0 of an empty tile writes its zeros)

    // ---- q of row g: fixed point, m = q 2^sh, |m| <= 2^22, in three signed limbs
    uint32_t qb[3][KC][4];
    float qstep;
    {
        const int32_t r = min(r0 + (int32_t)g, rows - 1), tok = sp.q0 + r / (int32_t)P.group;
        const T* q = static_cast<const T*>(a.q) + (uint64_t)tok * a.q_stride +
                     (uint64_t)(h * P.group + r % (int32_t)P.group) * HD;
        float x[KC][16];
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int j = 0; j < 16; j += 8) {
                float v[8];
                load8(q + 64 * c + 16 * t + j, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[c][j + i] = v[i];
                    m = max(m, abs_bits(v[i]));
                }
            }
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const bool bad = m >= 0x7f800000u;  // a query that is not finite: the row is NaN
        // 2^sh with amax 2^sh < 2^22; amax in [2^(e-127), 2^(e-126))
        const int sh = min(100, 22 - ((int)(m >> 23) - 126));
        const float up = bad ? 0.f : exp2f((float)sh);
        qstep = bad ? __uint_as_float(0x7fc00000u) : exp2f((float)-sh) * a.scale * 1.4426950408889634f;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t lb[3][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int v = bad ? 0 : __float2int_rn(x[c][4 * w + j] * up);
                    const int l0 = (int)(int8_t)v, v1 = (v - l0) >> 8, l1 = (int)(int8_t)v1, l2 = (v1 - l1) >> 8;
                    lb[0][j] = (uint32_t)l0, lb[1][j] = (uint32_t)l1, lb[2][j] = (uint32_t)l2;
                }
#pragma unroll
                for (int l = 0; l < 3; ++l) qb[l][c][w] = pack4(lb[l][0], lb[l][1], lb[l][2], lb[l][3]);
            }
    }
    // the lane's columns of the scores are rows 2t and 2t + 1
    float step[2];
    int32_t last[2];  // last position each row sees
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        step[j] = __shfl_sync(0xffffffffu, qstep, (2 * t + j) * 4);
        last[j] = 2 * (int32_t)t + j < nrow ? sp.base + (r0 + 2 * (int32_t)t + j) / (int32_t)P.group : -1;
    }
    const int32_t first_last = sp.base + r0 / (int32_t)P.group;  // the smallest of the tile's

    float o[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float M[2] = {kNegBig, kNegBig}, l[2] = {0.f, 0.f};

    const int32_t* table = a.b.table + (uint64_t)s * a.b.table_stride;
    const uint32_t bpp = a.c.page_size / 16;
    auto page_of = [&](int32_t blk) { return blk < b1 ? __ldg(table + (uint32_t)blk / bpp) : -1; };
    auto fine = [&](int32_t page) { return page >= 0 && (uint32_t)page < a.c.n_pages; };
    bool bad_page = false;
    Block<HD> cur, nxt;
    int32_t blk = b0 + (int32_t)warp;
    int32_t page = page_of(blk), page1 = page_of(blk + kWarps);
    if (fine(page)) load_block<HD>(cur, a.c, page, (uint32_t)blk % bpp, h, g, t);
    for (; blk < b1; blk += kWarps) {
        const bool have = fine(page);
        page = page1;
        page1 = page_of(blk + 2 * (int32_t)kWarps);
        if (fine(page)) load_block<HD>(nxt, a.c, page, (uint32_t)(blk + kWarps) % bpp, h, g, t);
        if (have) {
            // ---- scores
            int acc[3][4];
#pragma unroll
            for (int i = 0; i < 3; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = 0;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        mma_s8(acc[i], cur.k[c][0][2 * j], cur.k[c][1][2 * j], cur.k[c][0][2 * j + 1],
                               cur.k[c][1][2 * j + 1], qb[i][c][2 * j], qb[i][c][2 * j + 1]);
            // value scale = mant * 2^e; 0 (a block of zeros) and non-finite ones keep e = 0
            const uint32_t sb = __float_as_uint(cur.sv);
            const int eb = (int)((sb >> 23) & 0xffu);
            const bool plain = eb > 0 && eb < 255;
            const float e = plain ? (float)(eb - 127) : 0.f;
            const float mant = plain ? __uint_as_float((sb & 0x807fffffu) | 0x3f800000u) : cur.sv;
            const float down = plain ? __uint_as_float((uint32_t)(254 - eb) << 23) : 1.f;  // 2^-e
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float d = fmaf((float)acc[2][j], 65536.f, fmaf((float)acc[1][j], 256.f, (float)acc[0][j]));
                x[j] = fmaf(d, step[j & 1] * cur.sk, e);
            }
            if (blk * 16 + 15 > first_last) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (blk * 16 + (int32_t)g + (j >> 1) * 8 > last[j & 1]) x[j] = -INFINITY;
            }
            // ---- the running maximum
            const bool up = fmaxf(x[0], x[2]) > M[0] + kSlack || fmaxf(x[1], x[3]) > M[1] + kSlack;
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float m = fmaxf(x[j], x[j + 2]);
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(M[j], m);
                    const float f = exp2_fast(M[j] - m);
                    M[j] = m;
                    l[j] *= f;
#pragma unroll
                    for (int i = 0; i < MT; ++i) o[i][j] *= f, o[i][j + 2] *= f;
                }
            }
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = exp2_fast(x[j] - M[j & 1]);
            l[0] = fmaf(w[0] + w[2], down, l[0]);
            l[1] = fmaf(w[1] + w[3], down, l[1]);
            uint32_t ph[2], pl[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // (a hidden position has weight 0 even where the block's scale is not finite)
                const float p0 = w[2 * i] > 0.f ? w[2 * i] * mant : 0.f;
                const float p1 = w[2 * i + 1] > 0.f ? w[2 * i + 1] * mant : 0.f;
                const uint32_t hi = pack_h2(p0, p1);
                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                ph[i] = transpose8(hi);
                pl[i] = transpose8(pack_h2(p0 - back.x, p1 - back.y));
            }
            // ---- O^T += V^T w^T: lane dims (128 i + 16 g) + 2 j, + 1 are rows g, g + 8 of tile j
#pragma unroll
            for (int i = 0; i < VC; ++i)
#pragma unroll
                for (int q = 0; q < VW; ++q) {
                    const uint32_t w0 = cur.v[i][0][q] ^ 0x80808080u, w1 = cur.v[i][1][q] ^ 0x80808080u;
                    const uint32_t w2 = cur.v[i][2][q] ^ 0x80808080u, w3 = cur.v[i][3][q] ^ 0x80808080u;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t lo = __byte_perm(w0, w1, j ? 0x7362 : 0x5140);
                        const uint32_t hi = __byte_perm(w2, w3, j ? 0x7362 : 0x5140);
                        const uint32_t a0 = codes_h2(lo, 0x4140), a1 = codes_h2(lo, 0x4342);
                        const uint32_t a2 = codes_h2(hi, 0x4140), a3 = codes_h2(hi, 0x4342);
                        float(&d)[4] = o[(i * VW + q) * 2 + j];
                        mma_f16(d, a0, a1, a2, a3, ph[0], ph[1]);
                        mma_f16(d, a0, a1, a2, a3, pl[0], pl[1]);
                    }
                }
        } else {
            bad_page = true;
        }
        cur = nxt;
    }
    if (bad_page && lane == 0) flag_error(a.err, DEV_ERR_POSITION);

    // ---- the warps' partials
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 4);
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 8);
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 16);
        if (g == 0) sml[warp][2 * t + j] = make_float2(M[j], l[j]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int d = (i / (LD / 2)) * 128 + (int)g * LD + 2 * (i % (LD / 2));
#pragma unroll
        for (int j = 0; j < 2; ++j)
            *reinterpret_cast<float2*>(&so[warp][2 * t + j][d]) = make_float2(o[i][j], o[i][j + 2]);
    }
    __syncthreads();
    const uint64_t at = (((uint64_t)s * a.c.kv_heads + h) * P.row_tiles + tile) * P.splits + split;
    for (uint32_t i = tid * 4; i < (uint32_t)nrow * HD; i += 32 * kWarps * 4) {
        const uint32_t r = i / HD, d = i % HD;
        float m = kNegBig, sum = 0.f;
#pragma unroll
        for (uint32_t k = 0; k < kWarps; ++k) m = fmaxf(m, sml[k][r].x);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t k = 0; k < kWarps; ++k) {
            const float2 ml = sml[k][r];
            const float f = exp2_fast(ml.x - m);
            const float4 p = *reinterpret_cast<const float4*>(&so[k][r][d]);
            sum = fmaf(ml.y, f, sum);
            v[0] = fmaf(p.x, f, v[0]), v[1] = fmaf(p.y, f, v[1]), v[2] = fmaf(p.z, f, v[2]), v[3] = fmaf(p.w, f, v[3]);
        }
        if (P.splits == 1) {
            const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);  // a row that sees nothing: zeros
            const uint32_t row = (uint32_t)r0 + r;
            T* out = static_cast<T*>(a.out) + (uint64_t)(sp.q0 + row / P.group) * a.out_stride +
                     (uint64_t)(h * P.group + row % P.group) * HD + d;
            store2(out, v[0] * inv, v[1] * inv);
            store2(out + 2, v[2] * inv, v[3] * inv);
        } else {
            *reinterpret_cast<float4*>(P.part_o + (at * kRows + r) * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
            if (d == 0) P.part_ml[at * kRows + r] = make_float2(m, sum);
        }
    }
}

// One warp per (token, head): the chunks' partials under their common maximum, in chunk order.
template <class T, int HD> __global__ void __launch_bounds__(128) kv8_join_kernel(const __grid_constant__ Plan P) {
    const Kv8AttnArgs& a = P.a;
    const uint32_t lane = threadIdx.x & 31, head = blockIdx.y, s = blockIdx.z;
    const int32_t i = (int32_t)(blockIdx.x * 4 + (threadIdx.x >> 5));
    const Span sp = span_of(a, s);
    if (!sp.ok || i >= sp.n_new) return;
    const uint32_t h = head / P.group, row = (uint32_t)i * P.group + head % P.group, tile = row / kRows;
    const int32_t rows = sp.n_new * (int32_t)P.group;
    const int32_t seen = sp.base + (min((int32_t)((tile + 1) * kRows), rows) - 1) / (int32_t)P.group + 1;
    const uint32_t n = seen > 0 ? ((uint32_t)(seen + 15) / 16 + P.chunk - 1) / P.chunk : 1;
    const uint64_t at = (((uint64_t)s * a.c.kv_heads + h) * P.row_tiles + tile) * P.splits;
    float m = kNegBig;
    for (uint32_t k = lane; k < n; k += 32) m = fmaxf(m, P.part_ml[(at + k) * kRows + row % kRows].x);
    m = warp_max(m);
    constexpr int N = HD / 64;
    float v[N][2], sum = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) v[c][0] = v[c][1] = 0.f;
#pragma unroll 4
    for (uint32_t k = 0; k < n; ++k) {
        const uint64_t p = (at + k) * kRows + row % kRows;
        const float2 ml = P.part_ml[p];
        const float f = exp2_fast(ml.x - m);
        sum = fmaf(ml.y, f, sum);
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const float2 w = *reinterpret_cast<const float2*>(P.part_o + p * HD + 64 * c + 2 * lane);
            v[c][0] = fmaf(w.x, f, v[c][0]);
            v[c][1] = fmaf(w.y, f, v[c][1]);
        }
    }
    const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
    T* out = static_cast<T*>(a.out) + (uint64_t)(sp.q0 + i) * a.out_stride + (uint64_t)head * HD;
#pragma unroll
    for (int c = 0; c < N; ++c) store2(out + 64 * c + 2 * lane, v[c][0] * inv, v[c][1] * inv);
}

struct Shape {
    uint32_t group, row_tiles, chunk, splits;
    uint64_t slots;  // partials
};
Shape shape_of(const Kv8Cache& c, const Kv8Batch& b, uint32_t heads, int sms) {
    Shape r;
    r.group = heads / c.kv_heads;
    r.row_tiles = (uint32_t)(((uint64_t)std::max(1u, b.max_new) * r.group + kRows - 1) / kRows);
    const uint32_t blocks = std::max(1u, (b.max_len + 15) / 16);
    // chunks of positions: enough CTAs for three on every SM, at least 8 blocks (two per warp) each
    const uint64_t tiles = (uint64_t)b.n_seqs * c.kv_heads * r.row_tiles;
    const uint64_t want = std::max<uint64_t>(1, (3ull * sms) / std::max<uint64_t>(1, tiles));
    r.chunk = std::max(8u, (uint32_t)((blocks + want - 1) / want));
    r.splits = (blocks + r.chunk - 1) / r.chunk;
    r.slots = tiles * r.splits;
    return r;
}

template <class T, int HD> cudaError_t launch(const Plan& p, cudaStream_t s) {
    kv8_split_kernel<T, HD>
        <<<dim3(p.splits, p.row_tiles * p.a.c.kv_heads, p.a.b.n_seqs), 32 * kWarps, 0, s>>>(p);
    if (p.splits > 1)
        kv8_join_kernel<T, HD><<<dim3((p.a.b.max_new + 3) / 4, p.a.heads, p.a.b.n_seqs), 128, 0, s>>>(p);
    return cudaGetLastError();
}
template <class T> cudaError_t by_dim(const Plan& p, cudaStream_t s) {
    return p.a.c.head_dim == 64 ? launch<T, 64>(p, s) : p.a.c.head_dim == 128 ? launch<T, 128>(p, s) : launch<T, 256>(p, s);
}

}  // namespace

uint64_t kv8_attention_ws_bytes(const Kv8Cache& c, const Kv8Batch& b, uint32_t heads, int sms) {
    const Shape sh = shape_of(c, b, heads, sms);
    return sh.splits == 1 ? 0 : sh.slots * kRows * (c.head_dim + 2) * 4;
}

cudaError_t launch_kv8_attention(const Kv8AttnArgs& a, int sms, cudaStream_t s) {
    const Shape sh = shape_of(a.c, a.b, a.heads, sms);
    if ((uint64_t)sh.row_tiles * a.c.kv_heads > 65535 || a.heads > 65535) return cudaErrorInvalidValue;
    Plan p;
    p.a = a;
    p.group = sh.group;
    p.row_tiles = sh.row_tiles;
    p.chunk = sh.chunk;
    p.splits = sh.splits;
    p.part_o = reinterpret_cast<float*>(a.ws);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + sh.slots * kRows * a.c.head_dim);
    switch (a.type) {
        case GGML_F32: return by_dim<float>(p, s);
        case GGML_F16: return by_dim<__half>(p, s);
        case GGML_BF16: return by_dim<__nv_bfloat16>(p, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace evl
