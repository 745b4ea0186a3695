// kv8_attention.cu -- attention of new tokens over the 8-bit paged cache.
//
// o = sum_j softmax_j(scale * q . (sk_j ck_j)) sv_j cv_j over the positions j that the token
// sees, with 8-bit codes c and one scale s per block of 16 positions and kv head. The scales are
// constant over a block, so they leave the products: scores are integer products times one
// factor per block, and the value scale joins the softmax weight. One pass over the cache with
// a running maximum M of the scores and their sum, in the exponent's base 2:
//   x = q . ck (an integer) * (sk * scale * log2 e * step of q),
//   w = 2^(x - M),  l += w,  O += (w * sv) * cv,  o = O / l
// The codes meet w * sv in bf16 parts: codes of 8 bits are exact in bf16, and its exponents are f32's, so
// a weight keeps its bits however far below the maximum it lies (a head that puts nearly all weight on
// one position of value 0 is made of such weights; in f16 parts they were gone from 16 nats on). Three parts
// hold an f32 product exactly (f32 outputs), two are off by at most 2^-16 of it (16-bit outputs). Value
// scales near the ends of f32's range (below 2^-60, above 2^80) move the maximum that their positions
// ask for, so that their products stay inside (lift_of()).
//
// Small-batch kernel (kv8_split_kernel): up to 8 rows (token, head) per CTA that share a kv head;
// positions are the M dimension of the warp's products.
//   K: mma.sync m16n8k32 on the codes as they are. q is fixed point in three signed 8-bit limbs
//      (22 bits below the row's largest magnitude, so beside a loud channel the small values of q
//      keep fewer), the integer products are exact. The K order inside the product is permuted so that a
//      lane's fragment is 16 neighbouring bytes of a row: the codes reach the tensor cores as they
//      were copied, with no conversion.
//   V: mma.sync m16n8k16 in bf16. A lane loads 16 neighbouring dims of four positions and pairs positions
//      with byte permutes; the weights move to the other operand's layout by 8x8 transposes. For f32 a
//      block's products are summed there and the blocks in registers, since the tensor cores' own sums
//      are cut off (with the third part 64.7 -> 67.6 us at 131071 positions).
//   The maximum is raised only when a score passes it by 2^8, so most blocks cost one vote.
// A warp takes every 4th block of the CTA's chunk of positions, the next blocks already on their way
// into a ring of its own (asynchronous copies, each lane its own pieces: no barrier, no registers). The
// warps' partials meet in shared memory; a sequence of more than one chunk leaves (O, M, l) in the workspace for
// kv8_join_kernel.
// Bound: HBM, (2 head_dim + 1/2) bytes per position and kv head. Measured (32 heads, 8 kv heads of 128 dims):
// 131071 positions of one sequence, f32, 68 us = 4.0 TB/s, 61 % of a copy's rate; 32 sequences of up to
// 2100, bf16, 34 us = 3.0 TB/s; 517 positions 7.9 us. What holds the long one: its instructions, a third of them
// V's widening, issued by three warps a scheduler (issue 53 % busy, all waiting in turn on the ring, the
// products and the exponentials); the 32 sequences: 256 CTAs of four warps, seven warps an SM, of which the longest
// sequence's decide; all: about 4 us from a CTA's start to its first product and from its last one to the join.
#include <algorithm>
#include <atomic>

#include "int8.cuh"

namespace evl {
namespace {

constexpr uint32_t kRows = 8;     // rows of a tile (the product's N)
constexpr uint32_t kWarps = 4;
constexpr uint32_t kSumBlocks = 512;  // blocks that a warp sums on the tensor cores (16-bit types; see sum_steps)
constexpr float kNegBig = -1e38f;  // a maximum that no score has reached
constexpr float kSlack = 8.f;      // the maximum is raised when a score passes it by this: weights stay below 2^8

struct Plan {
    Kv8AttnArgs a;
    uint32_t group;      // q heads per kv head
    uint32_t row_tiles;  // per (sequence, kv head)
    uint32_t chunk;      // blocks of 16 positions per split
    uint32_t splits;
    uint32_t tile_rows;  // rows of a tile: kRows, or those of the prompt kernel
    float* part_o;       // [sequence][kv head][row tile][split][tile_rows][head_dim]
    float2* part_ml;     // same without head_dim: (M, l)
    float4* sums;        // of long chunks: [sequence][kv head][row tile][split][128 rows at a time][head_dim / 4][128]
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
// What the scores of a block are raised by where they ask for a new maximum: 0 for value scales from 2^-60 to 2^80 and
// for scales that are 0 (or subnormal, which count as 0) or not finite.
__device__ __forceinline__ float lift_of(float sv) {
    const int e = (int)(__float_as_uint(sv) >> 23 & 0xffu) - 127;
    return e == -127 || e == 128 ? 0.f : (float)(max(e - 80, 0) + min(e + 60, 0));
}
__device__ __forceinline__ float zero_if_subnormal(float sv) { return abs_bits(sv) < 0x00800000u ? 0.f : sv; }
// bytes 0, 1 (or 2, 3) of w, biased codes c + 128, as an exact f16 pair: 0x6400 | b is 1024 + b
__device__ __forceinline__ uint32_t codes_h2(uint32_t w, uint32_t sel) {
    const uint32_t h = __byte_perm(w, 0x64646464u, sel), bias = 0x64806480u;  // 1024 + 128
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// The same bytes of plain codes as an exact bf16 pair: 128 + the lower seven bits, less 128 or, for negative ones, 256.
__device__ __forceinline__ uint32_t codes_b2(uint32_t w, uint32_t sel) {
    const uint32_t t = __byte_perm(w, 0x43434343u, sel), a = t & 0xff7fff7fu, b = t & 0xff80ff80u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// A pair of products as PARTS bf16 pairs. Two: each rounded to nearest. Three: the upper half of each f32's bits, of what
// remains, and the rest (differences and the last part are exact).
template <int PARTS> __device__ __forceinline__ void split_b2(float a, float b, uint32_t (&part)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        if constexpr (PARTS == 2) {
            const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
            part[i] = *reinterpret_cast<const uint32_t*>(&r);
        } else {
            part[i] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
        }
        if (i + 1 < PARTS) a -= __uint_as_float(part[i] << 16), b -= __uint_as_float(part[i] & 0xffff0000u);
    }
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

// One block of 16 positions for one warp in shared memory: 16 (8) byte pieces, each in the place of the
// lane that will use it, so a lane reads what it copied itself and the warp needs no barrier:
// K rows g, g + 8 at 64 c + 16 t; V positions 2t, 2t+1, 2t+8, 2t+9 at 16 g (8 g); the two scales.
constexpr uint32_t ring_bytes(int hd) { return 32u * hd + 256; }
// blocks on their way per warp (a block in use besides): as many as leave room for three CTAs on an SM
constexpr int ring_depth(int hd) { return hd == 64 ? 6 : hd == 128 ? 4 : 3; }
constexpr uint32_t split_smem(int hd) { return kWarps * ring_depth(hd) * ring_bytes(hd); }

template <int N> __device__ __forceinline__ void cp_async(void* dst, const void* src) {
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr(dst)), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int HD>
__device__ __forceinline__ void fetch_block(uint8_t* slot, const Kv8Cache& c, int32_t page, uint32_t sub, uint32_t h,
                                            uint32_t lane) {
    const uint32_t g = lane >> 2, t = lane & 3;
    const uint64_t row = (uint64_t)page * c.page_stride + ((uint64_t)h * c.page_size + sub * 16) * HD;
    const int8_t *k = c.k + row, *v = c.v + row;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) cp_async<16>(slot + (i * 2 + r) * 512 + lane * 16, k + (g + 8 * r) * HD + 64 * i + 16 * t);
    slot += HD / 32 * 512;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int8_t* at = v + (2 * t + (p & 1) + (p >> 1) * 8) * HD;
        if constexpr (HD == 64) {
            cp_async<8>(slot + p * 256 + lane * 8, at + 8 * g);
        } else {
#pragma unroll
            for (int i = 0; i < HD / 128; ++i) cp_async<16>(slot + (p * (HD / 128) + i) * 512 + lane * 16, at + 128 * i + 16 * g);
        }
    }
    slot += HD * 16;
    const uint64_t sc = (uint64_t)page * c.scale_stride + h * (c.page_size / 16) + sub;
    cp_async<4>(slot + lane * 8, c.ks + sc);
    cp_async<4>(slot + lane * 8 + 4, c.vs + sc);
}
// The codes and scales of one block for one lane.
template <int HD> struct Block {
    uint32_t k[HD / 64][2][4];
    uint32_t v[HD <= 128 ? 1 : 2][4][HD < 128 ? 2 : 4];
    float sk, sv;
};
template <int HD> __device__ __forceinline__ void read_block(Block<HD>& b, const uint8_t* slot, uint32_t lane) {
#pragma unroll
    for (int i = 0; i < HD / 64; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint4 w = *reinterpret_cast<const uint4*>(slot + (i * 2 + r) * 512 + lane * 16);
            b.k[i][r][0] = w.x, b.k[i][r][1] = w.y, b.k[i][r][2] = w.z, b.k[i][r][3] = w.w;
        }
    slot += HD / 32 * 512;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        if constexpr (HD == 64) {
            const uint2 w = *reinterpret_cast<const uint2*>(slot + p * 256 + lane * 8);
            b.v[0][p][0] = w.x, b.v[0][p][1] = w.y;
        } else {
#pragma unroll
            for (int i = 0; i < HD / 128; ++i) {
                const uint4 w = *reinterpret_cast<const uint4*>(slot + (p * (HD / 128) + i) * 512 + lane * 16);
                b.v[i][p][0] = w.x, b.v[i][p][1] = w.y, b.v[i][p][2] = w.z, b.v[i][p][3] = w.w;
            }
        }
    }
    slot += HD * 16;
    const float2 s = *reinterpret_cast<const float2*>(slot + lane * 8);
    b.sk = s.x, b.sv = s.y;
}

template <class T, int HD>
__global__ void __launch_bounds__(32 * kWarps) kv8_split_kernel(const __grid_constant__ Plan P) {
    constexpr int KC = HD / 64;                  // 64-dim chunks of the score product
    constexpr int VW = HD < 128 ? 2 : 4;         // words of a V load
    constexpr int VC = HD <= 128 ? 1 : 2;        // V loads per position
    constexpr int MT = HD / 16;                  // 16-dim tiles of the output
    constexpr int LD = HD / 8 < 16 ? HD / 8 : 16;  // neighbouring dims of a lane's load
    constexpr int PARTS = sizeof(T) == 4 ? 3 : 2;  // bf16 parts of a weight
    constexpr int D = ring_depth(HD);
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ float2 sml[kWarps][kRows];
    static_assert(split_smem(HD) >= kWarps * kRows * HD * 4, "the warps' partials lie over the rings");
    const Kv8AttnArgs& a = P.a;
    const uint32_t split = blockIdx.x, h = blockIdx.y % a.c.kv_heads, tile = blockIdx.y / a.c.kv_heads, s = blockIdx.z;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
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

    // ---- the warp's blocks b0 + warp, + kWarps, ...: D - 1 of them on their way, the pages of one more
    // looked up
    const int32_t* table = a.b.table + (uint64_t)s * a.b.table_stride;
    const uint32_t lb = 31 - __clz(a.c.page_size / 16);  // log2 of the blocks of a page: 0, 1 or 2
    uint8_t* ring = ring_smem + warp * (D * ring_bytes(HD));
    auto page_of = [&](int32_t blk) { return blk < b1 ? __ldg(table + ((uint32_t)blk >> lb)) : -1; };
    uint32_t bad = 0;  // bits: slots whose block has no valid page
    bool bad_page = false;
    int32_t ahead = b0 + (int32_t)warp, page = page_of(ahead);
    auto fetch = [&](uint32_t slot) {
        const bool fine = page >= 0 && (uint32_t)page < a.c.n_pages;
        bad = fine ? bad & ~(1u << slot) : bad | 1u << slot;
        if (fine) fetch_block<HD>(ring + slot * ring_bytes(HD), a.c, page, (uint32_t)ahead & ((1u << lb) - 1), h, lane);
        cp_async_commit();
        ahead += kWarps;
        page = page_of(ahead);
    };
#pragma unroll
    for (int i = 0; i < D - 1; ++i) fetch((uint32_t)i);

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

    uint32_t slot = 0;
    for (int32_t blk = b0 + (int32_t)warp; blk < b1; blk += kWarps) {
        cp_async_wait<D - 2>();
        const bool have = !(bad >> slot & 1);
        Block<HD> cur;
        if (have) read_block<HD>(cur, ring + slot * ring_bytes(HD), lane);
        {
            const uint32_t next = slot == 0 ? D - 1 : slot - 1;  // the slot that the block before left
            fetch(next);
        }
        slot = slot + 1 == D ? 0 : slot + 1;
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
            const float sv = zero_if_subnormal(cur.sv), lift = lift_of(sv);
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // (the two lower limbs together stay below 2^30)
                const float d = fmaf((float)acc[2][j], 65536.f, (float)(acc[1][j] * 256 + acc[0][j]));
                x[j] = d * (step[j & 1] * cur.sk);
            }
            const bool edge = blk * 16 + 15 > first_last;
            if (edge) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (blk * 16 + (int32_t)g + (j >> 1) * 8 > last[j & 1]) x[j] = -INFINITY;
            }
            // ---- the running maximum
            const bool up = fmaxf(x[0], x[2]) + lift > M[0] + kSlack || fmaxf(x[1], x[3]) + lift > M[1] + kSlack;
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float m = fmaxf(x[j], x[j + 2]);
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(M[j], m + lift);
                    const float f = exp2_fast(M[j] - m);
                    l[j] *= f;
                    M[j] = m;
#pragma unroll
                    for (int i = 0; i < MT; ++i) o[i][j] *= f, o[i][j + 2] *= f;
                }
            }
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = exp2_fast(x[j] - M[j & 1]);
            l[0] += w[0] + w[2];
            l[1] += w[1] + w[3];
            uint32_t pw[PARTS][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float p[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    p[j] = w[2 * i + j] * sv;
                    // (a hidden position has weight 0 even where the block's scale is not finite)
                    if (edge && x[2 * i + j] == -INFINITY) p[j] = 0.f;
                }
                uint32_t part[PARTS];
                split_b2<PARTS>(p[0], p[1], part);
#pragma unroll
                for (int k = 0; k < PARTS; ++k) pw[k][i] = transpose8(part[k]);
            }
            // ---- O^T += V^T w^T: lane dims (128 i + 16 g) + 2 j, + 1 are rows g, g + 8 of tile j
#pragma unroll
            for (int i = 0; i < VC; ++i)
#pragma unroll
                for (int q = 0; q < VW; ++q) {
                    const uint32_t w0 = cur.v[i][0][q], w1 = cur.v[i][1][q], w2 = cur.v[i][2][q], w3 = cur.v[i][3][q];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t lo = __byte_perm(w0, w1, j ? 0x7362 : 0x5140);
                        const uint32_t hi = __byte_perm(w2, w3, j ? 0x7362 : 0x5140);
                        const uint32_t a0 = codes_b2(lo, 0x4140), a1 = codes_b2(lo, 0x4342);
                        const uint32_t a2 = codes_b2(hi, 0x4140), a3 = codes_b2(hi, 0x4342);
                        float(&sum)[4] = o[(i * VW + q) * 2 + j];
                        if constexpr (PARTS == 3) {
                            // (smallest parts first, into zeros: the tensor cores cut their sums off, O is added rounded)
                            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int k = PARTS - 1; k >= 0; --k) mma_bf16(d, a0, a1, a2, a3, pw[k][0], pw[k][1]);
#pragma unroll
                            for (int k = 0; k < 4; ++k) sum[k] += d[k];
                        } else {  // (at most kSumBlocks of them in a row)
#pragma unroll
                            for (int k = 0; k < PARTS; ++k) mma_bf16(sum, a0, a1, a2, a3, pw[k][0], pw[k][1]);
                        }
                    }
                }
        } else {
            bad_page = true;
        }
    }
    cp_async_wait<0>();
    // (not at the start: 32 sequences of 2100 positions 42 us against 32, with the next kernel's CTAs waiting
    // among this one's)
    pdl_launch_dependents();
    if (bad_page && lane == 0) flag_error(a.err, DEV_ERR_POSITION);

    // ---- the warps' partials, over the rings
    float(*so)[kRows][HD] = reinterpret_cast<float(*)[kRows][HD]>(ring_smem);
    __syncthreads();
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

// One CTA per (token, head): the chunks' partials under their common maximum. The warps deal the chunks
// among themselves, each keeps the order of its own, and their sums are added in warp order.
constexpr uint32_t kJoinWarps = 8;
template <class T, int HD> __global__ void __launch_bounds__(32 * kJoinWarps) kv8_join_kernel(const __grid_constant__ Plan P) {
    __shared__ float so[kJoinWarps][HD], sl[kJoinWarps];
    const Kv8AttnArgs& a = P.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = blockIdx.y, s = blockIdx.z;
    const int32_t i = (int32_t)blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    const Span sp = span_of(a, s);
    if (!sp.ok || i >= sp.n_new) return;
    const uint32_t h = head / P.group, row = (uint32_t)i * P.group + head % P.group, tile = row / P.tile_rows;
    const int32_t rows = sp.n_new * (int32_t)P.group;
    const int32_t seen = sp.base + (min((int32_t)((tile + 1) * P.tile_rows), rows) - 1) / (int32_t)P.group + 1;
    const uint32_t n = seen > 0 ? ((uint32_t)(seen + 15) / 16 + P.chunk - 1) / P.chunk : 1;
    const uint64_t at = ((((uint64_t)s * a.c.kv_heads + h) * P.row_tiles + tile) * P.splits) * P.tile_rows + row % P.tile_rows;
    float m = kNegBig;
    for (uint32_t k = lane; k < n; k += 32) m = fmaxf(m, P.part_ml[at + (uint64_t)k * P.tile_rows].x);
    m = warp_max(m);
    constexpr int N = HD / 64;
    float v[N][2], sum = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) v[c][0] = v[c][1] = 0.f;
#pragma unroll 4
    for (uint32_t k = warp; k < n; k += kJoinWarps) {
        const uint64_t p = at + (uint64_t)k * P.tile_rows;
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
#pragma unroll
    for (int c = 0; c < N; ++c) *reinterpret_cast<float2*>(&so[warp][64 * c + 2 * lane]) = make_float2(v[c][0], v[c][1]);
    if (lane == 0) sl[warp] = sum;
    __syncthreads();
    const uint32_t d = 2 * threadIdx.x;
    if (d >= HD) return;
    float2 o = make_float2(0.f, 0.f);
    sum = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < kJoinWarps; ++w) {
        const float2 x = *reinterpret_cast<const float2*>(&so[w][d]);
        o.x += x.x, o.y += x.y, sum += sl[w];
    }
    const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
    store2(static_cast<T*>(a.out) + (uint64_t)(sp.q0 + i) * a.out_stride + (uint64_t)head * HD + d, o.x * inv, o.y * inv);
}

// ------------------------------------------------------------------ prompts
// kv8_tile_kernel: many rows per kv head, on the 5th-generation tensor cores. A CTA takes RT row
// tiles of 128 rows (token, head) of one (sequence, kv head) and walks the positions NP at a time:
//   1 block warp      a lane per block looks its page up, copies its codes into a ring (one run of memory for
//                     K and one for V: two bulk copies) and makes the factors of its scales;
//   4 producer warps  codes to f16 (K; f32: as they are) and bf16 (V), exactly, into a ring of shared-memory
//                     stages: 64 dims x NP positions per 128-byte-swizzled panel. The score product reads
//                     them K-major, the value product MN-major, so no transpose is made;
//   RT MMA threads    one per row tile: S = q K^T into tensor memory (two to four buffers per row
//                     tile, so the next scores are multiplied while this step's softmax runs),
//                     O += P V with P read from tensor memory;
//   4 softmax warps   per row tile, one row per thread: scores to registers, running maximum,
//                     weights to bf16 parts over the scores' own columns. O is rescaled (read, multiplied,
//                     written back) only when a score passes the row's maximum by 2^8.
// 16-bit inputs: q is scaled by a power of two per row and held in f16, exactly down to 2^-24 (its largest just under
// 2^10); the weights are two bf16 parts, with the value scale as an added log2 in their exponent. f32 inputs: q is fixed
// point in three 8-bit limbs and the scores are integer products (kind::i8) of the codes as they are, summed exactly
// -- the f32 sums of kind::f16 are cut off, not rounded, and over long sums that shows; the weights are three bf16 parts.
// Bound: the tensor pipe and, close behind, shared memory: a step of 64 positions with two row tiles of 128 dims
// is 1536 clocks of products (512 of them the weights' second part), 1800 of shared-memory traffic (q is read again
// for every K panel, the codes pass it three times, V once for each part) and 1024 of exponentials on each scheduler.
// Measured (2048 tokens behind 6144 positions, 32 heads, 8 kv heads of 128 dims, bf16): 364 us = 660 TFLOP/s; the tensor
// pipe of the busiest SM is active 69 % of the time, and 256 CTAs on 148 SMs take two turns where 1.73 would do. 64 rows
// over 4099 positions of 8 sequences, 8 kv heads: 55 us; 512 f32 tokens over 4096 positions, 8 kv heads of 128: 182.
// (One f16 part took 297, 48 and 120 us, without the range.) Parts left out to time the rest: without the second
// product 3 us less, without its conversions 44, without both 79: softmax warps and products hold one another up.
// Tried and slower: parts cut instead of rounded (380 us against 375), scalar operations instead of pairs (380), the
// largest score looked for first so that parts can be stored at once (380); with one f16 part 128 positions a step with
// one score buffer (432 against 316), codes kept in registers instead of a ring (354 against 331), the store's end
// waited for one step late (293 against 297, but 54 against 48 with one row tile), polynomials for some exponentials.
constexpr uint32_t kTileRows = 128;
// Rows per (sequence, kv head) from which it may be used, and the blocks of 16 positions times tiles of eight rows
// that each warp of the other kernel would then have to take. Measured over 64 to 256 dims, bf16 and f32, 16 to 96
// rows, 600 to 16000 positions of 1 to 32 sequences: 1.4 % over the better kernel's time on average, 34 % at
// most; on either side of the rule, 32 rows over 4099 positions of 9 sequences with 8 kv heads of 128 dims,
// bf16: 50 us against 60; 16 rows: 47 against 40; 32 rows over 600 positions of 2 sequences: 14.0 against 11.9.
// (f32 has one row tile and more products, and its rows pay later: 48 rows over the 4099 positions 110 against 84,
// 64 rows 112 against 105.)
__host__ __device__ constexpr uint32_t tile_min(bool f32) { return f32 ? 64 : 24; }
constexpr uint64_t kTileWork = 3;

// Steps whose products are added up in tensor memory. Its sums are cut off, not rounded, by up to 2^-23 at
// each product of 16 positions and one part (values of one sign lose 4.4e-8 each on average); after 96 of them (f32;
// 1024: 16-bit types) O joins a sum in the workspace, rounded to nearest, and starts again from zero.
__host__ __device__ constexpr uint32_t sum_steps(uint32_t np, bool f32) { return (f32 ? 96u / 3 : 1024u / 2) / (np / 16); }

struct Role {  // per (HD, f32 or not): row tiles, positions per step, stages of f16 panels, of codes
    uint32_t rt, np, stages, raw;
};
__host__ __device__ constexpr Role role_of(int hd, bool f32) {
    return hd == 256 ? (f32 ? Role{1, 32, 2, 2} : Role{1, 32, 3, 3}) : f32 ? Role{1, 64, 2, 4} : Role{2, 64, 2, 4};
}
// bytes of one part of a row tile's q (f16; or an 8-bit limb), of a stage's K
__host__ __device__ constexpr uint32_t q_part(int hd, bool f32) { return kTileRows * hd * (f32 ? 1 : 2); }
__host__ __device__ constexpr uint32_t q_parts(bool f32) { return f32 ? 3 : 1; }
__host__ __device__ constexpr uint32_t k_stage(int hd, bool f32) { return role_of(hd, f32).np * hd * (f32 ? 1 : 2); }
__host__ __device__ constexpr uint32_t tile_smem(int hd, bool f32) {
    return role_of(hd, f32).rt * q_parts(f32) * q_part(hd, f32) +
           role_of(hd, f32).stages * (k_stage(hd, f32) + role_of(hd, f32).np * hd * 2) +
           role_of(hd, f32).raw * role_of(hd, f32).np * hd * 2 + 1024;
}
static_assert(tile_smem(256, true) <= 232448 && tile_smem(256, false) <= 232448 && tile_smem(128, false) <= 232448, "shared memory");

__device__ __forceinline__ bool bwait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*abort_flag) return false;
        if (global_ns() - t0 > kWaitNs) {
            *abort_flag = 1;
            return false;
        }
    }
    return true;
}
// the same for a whole warp, which stays together
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const uint64_t t0 = global_ns();
    while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
        if (__any_sync(0xffffffffu, *abort_flag || global_ns() - t0 > kWaitNs)) {
            *abort_flag = 1;
            return false;
        }
    return true;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
// one lane of a converged warp, in the form that tells the compiler so
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
// shared-memory operand, 128-byte swizzle. lbo: bytes between 64-element panels (MN-major), sbo: between 8-row groups
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// K-major 8-bit operand: rows of 128 bytes as above, or (64 dims) of 64 bytes with the 64-byte swizzle
template <int HD> __device__ __forceinline__ uint64_t bytes_desc(uint32_t addr) {
    constexpr uint64_t group = HD == 64 ? 512 : 1024, mode = HD == 64 ? 4 : 2;
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((group >> 4) << 32) | (1ull << 46) | (mode << 61);
}
// byte offset of 16-byte piece `p` of row r in such panels of `rows` rows
template <int HD> __device__ __forceinline__ uint32_t bytes_at(uint32_t rows, uint32_t r, uint32_t p) {
    if constexpr (HD == 64) return r * 64u + ((p ^ ((r >> 1) & 3u)) << 4);
    else return (p >> 3) * (rows * 128u) + r * 128u + (((p & 7u) ^ (r & 7u)) << 4);
}
__host__ __device__ constexpr uint32_t i8_idesc(uint32_t n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((kTileRows >> 4) << 24);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__host__ __device__ constexpr uint32_t f16_idesc(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((kTileRows >> 4) << 24); }
// bf16, B as [K][N]
__host__ __device__ constexpr uint32_t bf16_idesc(uint32_t n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((n >> 3) << 17) | ((kTileRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t t, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t t, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(t)
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t t, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two f32 operations in one instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    return (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
}
__device__ __forceinline__ uint64_t pack2(uint32_t a, uint32_t b) { return (uint64_t)a | (uint64_t)b << 32; }
__device__ __forceinline__ float lo2(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi2(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// byte offset of 16-byte piece `p` (8 f16 values) of row r in panels of `rows` rows
__device__ __forceinline__ uint32_t panel_at(uint32_t rows, uint32_t r, uint32_t p) {
    return (p >> 3) * (rows * 128u) + r * 128u + (((p & 7u) ^ (r & 7u)) << 4);
}
// 16 codes to f16 (keys) or bf16 (values), two 16-byte pieces
template <bool BF16> __device__ __forceinline__ void codes_to_panel(uint8_t* panel, uint32_t rows, uint32_t r, uint32_t c, uint4 w) {
    uint32_t h[8];
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF16) {
            h[2 * i] = codes_b2(in[i], 0x4140);
            h[2 * i + 1] = codes_b2(in[i], 0x4342);
        } else {
            const uint32_t b = in[i] ^ 0x80808080u;
            h[2 * i] = codes_h2(b, 0x4140);
            h[2 * i + 1] = codes_h2(b, 0x4342);
        }
    }
    *reinterpret_cast<uint4*>(panel + panel_at(rows, r, 2 * c)) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(panel + panel_at(rows, r, 2 * c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
}

template <class T, int HD>
__global__ void __launch_bounds__(32 * (5 * role_of(HD, sizeof(T) == 4).rt + 5), 1)
    kv8_tile_kernel(const __grid_constant__ Plan P) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int PARTS = F32 ? 3 : 2;  // bf16 parts of a weight
    constexpr Role R = role_of(HD, F32);
    constexpr uint32_t RT = R.rt, NP = R.np, ST = R.stages, RAW = R.raw, NB = NP / 16;
    constexpr uint32_t kQPart = q_part(HD, F32), kQParts = q_parts(F32);
    constexpr uint32_t kK = k_stage(HD, F32), kV = NP * HD * 2, kStage = kK + kV;  // K and V of a stage
    constexpr uint32_t kSCols = F32 ? 3 * NP : NP;  // tensor memory columns of a score buffer, then of its weights
    static_assert(PARTS * NP / 2 <= kSCols, "tensor memory");
    constexpr uint32_t G = sum_steps(NP, F32);
    // log2 of a row tile's score buffers: as many as its share of the tensor memory holds beside O, up to four
    constexpr uint32_t kMostBuffers = HD + 4 * kSCols <= 512 ? 2 : 1, kShared = RT == 1 ? kMostBuffers : 1;
    static_assert(RT * (HD + (kSCols << kShared)) <= 512 && (RT == 1 || HD + 2 * kSCols <= 256), "tensor memory");
    constexpr uint32_t kSoftWarps = 4 * RT, kTileCols = RT == 2 ? 256 : 512;  // tensor memory columns per row tile
    extern __shared__ uint8_t raw_smem[];
    constexpr uint32_t FG = 8, FS = 2 * FG;  // steps of block factors handed over together, and kept
    __shared__ __align__(8) uint64_t k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], f_full[2], f_empty[2], c_full[RAW], c_empty[RAW];
    __shared__ __align__(8) uint64_t s_full[RT][4], p_full[RT][4], o_done[RT][4], q_full, fin[RT];
    // key scale, log2 of the value scale (f32: 0; -infinity: no such page, infinity: a rare one), its inverse, itself
    __shared__ float4 f_blk[FS][NB];
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    const Kv8AttnArgs& a = P.a;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // the last row tiles see the most positions: they go first
    const uint32_t tile = P.row_tiles - 1 - blockIdx.x / P.splits, split = blockIdx.x % P.splits, h = blockIdx.y, s = blockIdx.z;
    pdl_wait();
    const Span sp = span_of(a, s);
    if (!sp.ok) {
        if (tid == 0) flag_error(a.err, DEV_ERR_POSITION);
        return;
    }
    const int32_t rows = sp.n_new * (int32_t)P.group, r0 = (int32_t)(tile * (RT * kTileRows));
    if (r0 >= rows) return;
    const int32_t nrow = min((int32_t)(RT * kTileRows), rows - r0);
    const int32_t seen = sp.base + (r0 + nrow - 1) / (int32_t)P.group + 1;
    const int32_t nblk = seen > 0 ? (seen + 15) / 16 : 0;
    const int32_t b0 = (int32_t)(split * P.chunk), b1 = min(nblk, b0 + (int32_t)P.chunk);
    if (b0 >= nblk && split > 0) return;
    const uint32_t steps = b1 > b0 ? (uint32_t)(b1 - b0 + (int32_t)NB - 1) / NB : 0;
    const uint32_t used = ((uint32_t)nrow + kTileRows - 1) / kTileRows;  // row tiles that hold rows; the others' warps rest
    const uint32_t lsb = RT == 2 && used == 1 ? kMostBuffers : kShared, nsb = 1u << lsb;  // score buffers of a row tile

    uint8_t* smem = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);
    uint8_t* sq = smem;                                  // [RT] q panels
    uint8_t* skv = smem + RT * kQParts * kQPart;         // [ST][K | V] panels
    uint8_t* sraw = skv + ST * kStage;                  // [RAW][K | V] codes, block after block
    if (tid == 0) {
        abort_flag = 0;
        for (uint32_t i = 0; i < ST; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&k_empty[i], used);
            mbar_init(&v_full[i], 4);
            mbar_init(&v_empty[i], used);
        }
        for (uint32_t i = 0; i < RAW; ++i) {
            mbar_init(&c_full[i], 1);
            mbar_init(&c_empty[i], 4);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&f_full[i], 1);
            mbar_init(&f_empty[i], 4 * used);
        }
        for (uint32_t i = 0; i < RT; ++i) {
            // (one of each per score buffer: a warp may finish the next step's weights before another has this
            // one's, and a parity tells only neighbouring phases apart)
            for (uint32_t k = 0; k < 4; ++k) {
                mbar_init(&s_full[i][k], 1);
                mbar_init(&p_full[i][k], 4);
                mbar_init(&o_done[i][k], 1);
            }
            mbar_init(&fin[i], 1);
        }
        mbar_init(&q_full, 4 * used);
        fence_barrier_init();
    }
    if (warp == kSoftWarps + 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = tmem_base;
    pdl_launch_dependents();  // (not before: a kernel that began meanwhile could hold the tensor memory)

    if (warp < 4 * used) {
        // ---------------------------------------------------------------- softmax: one row per thread
        const uint32_t rt = warp >> 2, quad = warp & 3, lr = quad * 32 + lane;
        const int32_t row = r0 + (int32_t)(rt * kTileRows + lr);
        const bool live = row < rows;
        const int32_t row_c = min(row, rows - 1), tok = row_c / (int32_t)P.group;
        const uint32_t head = h * P.group + (uint32_t)(row_c % (int32_t)P.group);
        float step;
        {
            const T* q = static_cast<const T*>(a.q) + (uint64_t)(sp.q0 + tok) * a.q_stride + (uint64_t)head * HD;
            uint32_t m = 0;
#pragma unroll 4
            for (int d = 0; d < HD; d += 8) {
                float v[8];
                load8(q + d, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
            }
            const bool bad = m >= 0x7f800000u;
            // largest magnitude just under 2^10 (f16) or 2^22 (limbs)
            const int sh = min(100, (F32 ? 22 : 10) - ((int)(m >> 23) - 126));
            const float up = copysignf(exp2f((float)sh), a.scale);  // (so that the factor is not negative)
            step = bad ? __uint_as_float(0x7fc00000u) : exp2f((float)-sh) * fabsf(a.scale) * 1.4426950408889634f;
            uint8_t* panel = sq + rt * kQParts * kQPart;
            if constexpr (!F32) {
#pragma unroll 4
                for (int d = 0; d < HD; d += 8) {
                    float v[8];
                    load8(q + d, v);
                    uint32_t hi[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) hi[i] = pack_h2(bad ? 0.f : v[2 * i] * up, bad ? 0.f : v[2 * i + 1] * up);
                    *reinterpret_cast<uint4*>(panel + panel_at(kTileRows, lr, d / 8)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                }
            } else {
#pragma unroll 1
                for (int d = 0; d < HD; d += 16) {
                    uint32_t w[3][4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float v[4];
                        uint32_t lb[3][4];
                        load4(q + d + 4 * k, v);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int x = bad ? 0 : __float2int_rn(v[i] * up);
                            const int l0 = (int)(int8_t)x, x1 = (x - l0) >> 8, l1 = (int)(int8_t)x1, l2 = (x1 - l1) >> 8;
                            lb[0][i] = (uint32_t)l0, lb[1][i] = (uint32_t)l1, lb[2][i] = (uint32_t)l2;
                        }
#pragma unroll
                        for (int i = 0; i < 3; ++i) w[i][k] = pack4(lb[i][0], lb[i][1], lb[i][2], lb[i][3]);
                    }
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        *reinterpret_cast<uint4*>(panel + i * kQPart + bytes_at<HD>(kTileRows, lr, d / 16)) =
                            make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
        }
        const int32_t last = sp.base + tok;  // (lanes past the last row do its work again and write nothing)
        const bool idle = r0 + (int32_t)(rt * kTileRows + quad * 32) >= rows;  // the whole warp
        // no row of this warp hides a position before this one
        const int32_t open = sp.base + min(r0 + (int32_t)(rt * kTileRows + quad * 32), rows - 1) / (int32_t)P.group;
        const uint32_t to = tm + rt * kTileCols + ((quad * 32) << 16);  // O, then the score buffers
        const uint64_t place = ((((uint64_t)s * a.c.kv_heads + h) * P.row_tiles + tile) * P.splits + split) * RT + rt;
        // (a warp's rows side by side: with a row's values side by side each access touched 32 lines, 283 us against 231
        // for 300 tokens over 4000 positions of 2 sequences, 256 dims)
        float4* sums = P.sums + place * (HD / 4 * kTileRows) + lr;
        float M = kNegBig, l = 0.f, Msum = 0.f;  // Msum: the maximum under which the sum in the workspace stands
        bool ok = true;
        for (uint32_t j = 0; j < steps && ok; ++j) {
            const uint32_t st = j % FS, fg = j / FG % 2;
            if (j % FG == 0) ok = warp_wait(&f_full[fg], (j / FG / 2) & 1, &abort_flag);
            ok = ok && warp_wait(&s_full[rt][j % nsb], (j >> lsb) & 1, &abort_flag);
            if (!ok) break;
            tc_after();
            auto done = [&] {
                tmem_st_wait();
                tc_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&p_full[rt][j % nsb]);
                    if (j % FG == FG - 1) mbar_arrive(&f_empty[fg]);
                }
            };
            if (idle) {  // (what these rows add up goes nowhere)
                done();
                continue;
            }
            if (j && j % G == 0) {  // (rows past the last one have their places in the workspace too)
                float4 x[2][8];
                auto fetch = [&](uint32_t c) {
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) x[c & 1][i] = sums[(8 * c + i) * kTileRows];
                };
                fetch(0);
                ok = warp_wait(&o_done[rt][(j - 1) % nsb], ((j - 1) >> lsb) & 1, &abort_flag);
                if (!ok) break;
                tc_after();
                const bool first = j == G;
                const float f = exp2_fast(Msum - M);
#pragma unroll
                for (uint32_t c = 0; c < HD / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(to + 32 * c, o);
                    if (c + 1 < HD / 32) fetch(c + 1);  // on their way meanwhile
                    tmem_ld_wait();
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        const float4 y = x[c & 1][i];
                        float4 z = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                        if (!first) z = make_float4(fmaf(y.x, f, z.x), fmaf(y.y, f, z.y), fmaf(y.z, f, z.z), fmaf(y.w, f, z.w));
                        sums[(8 * c + i) * kTileRows] = z;
                    }
                }
                Msum = M;
            }
            const uint32_t ts = to + HD + j % nsb * kSCols;
            const int32_t p0 = (b0 + (int32_t)(j * NB)) * 16;
            const bool masked = p0 + (int32_t)NP - 1 > open;
            float f[NB], e[NB], down[NB], sv[NB];
            bool rare = false;  // a block of zeros, of a scale near the ends of f32's range or not finite, or without a page
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const float4 w = f_blk[st][b];
                f[b] = step * w.x;
                e[b] = w.y, down[b] = w.z, sv[b] = w.w;
                rare |= fabsf(e[b]) == INFINITY;
            }
            // ---- the usual step: nothing hidden, and the maximum still holds. The weights are made
            // without looking for the maximum: their sum tells whether one passes it by far (or is
            // not a number), and then the scores are read again below.
            if (!F32 && j > 0 && !masked && !__any_sync(0xffffffffu, rare)) {
                uint32_t hi[NP / 2], lo[NP / 2], v[2][16];
                float add = 0.f;
                tmem_ld16(ts, v[0]);
                tmem_ld_wait();
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) {  // the next block's scores on their way meanwhile
                    if (b + 1 < NB) tmem_ld16(ts + 16 * (b + 1), v[(b + 1) & 1]);
                    const uint32_t(&x)[16] = v[b & 1];
                    const uint64_t ff = pack2(f[b], f[b]), off = pack2(e[b] - M, e[b] - M);
                    uint64_t sum = 0;
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        const uint64_t y = fma2(pack2(x[2 * i], x[2 * i + 1]), ff, off);
                        const float w0 = exp2_fast(lo2(y)), w1 = exp2_fast(hi2(y));
                        sum = add2(sum, pack2(w0, w1));
                        // (split_b2, the differences of a pair in one operation)
                        const __nv_bfloat162 h = __floats2bfloat162_rn(w0, w1);
                        const uint32_t hb = *reinterpret_cast<const uint32_t*>(&h);
                        const uint64_t left = fma2(pack2(hb << 16, hb & 0xffff0000u), pack2(-1.f, -1.f), pack2(w0, w1));
                        const __nv_bfloat162 r = __floats2bfloat162_rn(lo2(left), hi2(left));
                        hi[8 * b + i] = hb;
                        lo[8 * b + i] = *reinterpret_cast<const uint32_t*>(&r);
                    }
                    add = fmaf(lo2(sum) + hi2(sum), down[b], add);
                    if (b + 1 < NB) tmem_ld_wait();
                }
                if (__all_sync(0xffffffffu, add < 16384.f)) {
                    l += add;
#pragma unroll
                    for (uint32_t b = 0; b < NB; ++b) {
                        tmem_st8(ts + 8 * b, hi + 8 * b);
                        tmem_st8(ts + NP / 2 + 8 * b, lo + 8 * b);
                    }
                    done();
                    continue;
                }
            }
            uint32_t v[NP];
            if constexpr (!F32) {
#pragma unroll
                for (uint32_t c = 0; c < NP; c += 32) tmem_ld32(ts + c, *reinterpret_cast<uint32_t(*)[32]>(v + c));
                tmem_ld_wait();
            } else {
#pragma unroll
                for (uint32_t c = 0; c < NP; c += 16) {
                    uint32_t l0[16], l1[16], l2[16];
                    tmem_ld16(ts + c, l0);
                    tmem_ld16(ts + NP + c, l1);
                    tmem_ld16(ts + 2 * NP + c, l2);
                    tmem_ld_wait();
#pragma unroll
                    for (uint32_t i = 0; i < 16; ++i)  // (the two lower limbs together stay below 2^30)
                        v[c + i] = __float_as_uint(fmaf((float)(int)l2[i], 65536.f, (float)((int)l1[i] * 256 + (int)l0[i])));
                }
            }
            if (masked) {
#pragma unroll
                for (uint32_t i = 0; i < NP; ++i)
                    if (p0 + (int32_t)i > last) v[i] = 0xff800000u;  // -infinity
            }
            // the largest score: of each block's products, then by the block's factor (not negative)
            float mx = -INFINITY;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                float m = __uint_as_float(v[16 * b]);
#pragma unroll
                for (uint32_t i = 1; i < 16; ++i) m = fmaxf(m, __uint_as_float(v[16 * b + i]));
                // (a hidden block and a factor of 0: 0 * -infinity is not a number)
                mx = fmaxf(mx, m == -INFINITY || e[b] == -INFINITY ? -INFINITY : fmaf(m, f[b], lift_of(sv[b])));
            }
            if (__any_sync(0xffffffffu, mx > M + kSlack)) {
                const float m = fmaxf(M, mx), f8 = exp2_fast(M - m);
                l *= f8;
                M = m;
                if (j % G) {  // (a step that starts O again finds nothing to move)
                    ok = warp_wait(&o_done[rt][(j - 1) % nsb], ((j - 1) >> lsb) & 1, &abort_flag);
                    if (!ok) break;
                    tc_after();
#pragma unroll 1
                    for (uint32_t c = 0; c < HD; c += 8) {  // (rare: in few registers)
                        uint32_t o[8];
                        tmem_ld8(to + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f8);
                        tmem_st8(to + c, o);
                    }
                }
            }
            auto weights = [&](auto some) {  // some: hidden positions, or a block that is rare
                constexpr bool SOME = decltype(some)::value;
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) {
                    float sum = 0.f;
                    uint32_t part[PARTS][8];
                    const float off = SOME && e[b] == -INFINITY ? -INFINITY : -M;
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        float p[2];
#pragma unroll
                        for (uint32_t k = 0; k < 2; ++k) {
                            const float x = __uint_as_float(v[16 * b + 2 * i + k]);
                            const bool hidden = SOME && x == -INFINITY;  // (a product itself is never infinite)
                            const float w = hidden ? 0.f : exp2_fast(fmaf(x, f[b], off));
                            sum += w;
                            p[k] = hidden ? 0.f : w * sv[b];
                        }
                        uint32_t pp[PARTS];
                        split_b2<PARTS>(p[0], p[1], pp);
#pragma unroll
                        for (int k = 0; k < PARTS; ++k) part[k][i] = pp[k];
                    }
                    l += sum;
#pragma unroll
                    for (int k = 0; k < PARTS; ++k) tmem_st8(ts + k * (NP / 2) + 8 * b, part[k]);
                }
            };
            if (masked || __any_sync(0xffffffffu, rare)) weights(std::true_type{});
            else weights(std::false_type{});
            done();
        }
        if (steps && ok) ok = warp_wait(&o_done[rt][(steps - 1) % nsb], ((steps - 1) >> lsb) & 1, &abort_flag);
        tc_after();
        if (ok) {
            const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);  // a row that sees nothing: zeros
            T* out = static_cast<T*>(a.out) + (uint64_t)(sp.q0 + tok) * a.out_stride + (uint64_t)head * HD;
            const uint64_t slot = place * kTileRows + lr;
            if (live && P.splits > 1) P.part_ml[slot] = make_float2(M, l);
            for (uint32_t c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (steps) {
                    tmem_ld32(to + c, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                if (steps > G) {
                    const float f = exp2_fast(Msum - M);
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 4) {
                        const float4 x = sums[(c + i) / 4 * kTileRows];
                        o[i] = __float_as_uint(fmaf(x.x, f, __uint_as_float(o[i])));
                        o[i + 1] = __float_as_uint(fmaf(x.y, f, __uint_as_float(o[i + 1])));
                        o[i + 2] = __float_as_uint(fmaf(x.z, f, __uint_as_float(o[i + 2])));
                        o[i + 3] = __float_as_uint(fmaf(x.w, f, __uint_as_float(o[i + 3])));
                    }
                }
                __syncwarp();
                if (!live) {
                } else if (P.splits > 1) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4*>(P.part_o + slot * HD + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                } else if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(out + c + i) =
                            make_float4(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv,
                                        __uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        T y[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) y[k] = from_f32<T>(__uint_as_float(o[i + k]) * inv);
                        *reinterpret_cast<uint4*>(out + c + i) = *reinterpret_cast<uint4*>(y);
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp < kSoftWarps) {
    } else if (warp < kSoftWarps + 4) {
        // ---------------------------------------------------------------- producers
        const uint32_t pt = tid - 32 * kSoftWarps;  // 0..127
        constexpr uint32_t CPR = HD / 16, N = NP * CPR / 128;  // 16-code pieces per row, per thread and operand
        // Piece of a thread: row and 16-code column. Eight neighbouring lanes take two rows of four columns, so
        // that the f16 pieces that they write lie in eight different 16-byte columns of the banks.
        auto row_of = [](uint32_t p) { return CPR == 4 ? p / 4 : p / (2 * CPR) * 2 + (p >> 2 & 1); };
        auto col_of = [](uint32_t p) { return CPR == 4 ? p % 4 : (p & 3) | (p % (2 * CPR) >> 3) << 2; };
        auto piece = [&](uint32_t i) { return pt + 128 * i; };
        auto code_at = [&](uint32_t i) { return row_of(piece(i)) * HD + 16 * col_of(piece(i)); };
        // (blocks without a valid page were not copied: whatever codes lie there have weight 0)
        auto widen = [&](auto bf16, uint8_t* panel, const uint8_t* raw) {
            uint4 w[N];
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint4*>(raw + code_at(i));
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) codes_to_panel<decltype(bf16)::value>(panel, NP, row_of(piece(i)), col_of(piece(i)), w[i]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        auto copy = [&](uint8_t* panel, const uint8_t* raw) {  // the codes as they are
#pragma unroll
            for (uint32_t i = 0; i < N; ++i)
                *reinterpret_cast<uint4*>(panel + bytes_at<HD>(NP, row_of(piece(i)), col_of(piece(i)))) =
                    *reinterpret_cast<const uint4*>(raw + code_at(i));
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        for (uint32_t j = 0; j < steps; ++j) {  // (after an abort the loop runs out quickly: every wait gives up at once)
            const uint32_t st = j % ST, rs = j % RAW;
            const uint8_t* raw = sraw + rs * (2 * NP * HD);
            uint8_t* dst = skv + st * kStage;
            warp_wait(&c_full[rs], (j / RAW) & 1, &abort_flag);
            if (j >= ST) warp_wait(&k_empty[st], (j / ST - 1) & 1, &abort_flag);
            if (F32) copy(dst, raw);
            else widen(std::false_type{}, dst, raw);
            if (lane == 0) mbar_arrive(&k_full[st]);
            if (j >= ST) warp_wait(&v_empty[st], (j / ST - 1) & 1, &abort_flag);
            widen(std::true_type{}, dst + kK, raw + NP * HD);
            if (lane == 0) {
                mbar_arrive(&v_full[st]);
                mbar_arrive(&c_empty[rs]);
            }
        }
    } else if (warp == kSoftWarps + 4 + RT) {
        // ---------------------------------------------------------------- the blocks: their factors and codes
        // one lane per block, 32 / NB steps looked up together; a block's codes are one run of memory for
        // K and one for V, each copied by its lane
        constexpr uint32_t LS = 32 / NB;
        static_assert(LS % FG == 0, "whole groups of factors");
        const int32_t* table = a.b.table + (uint64_t)s * a.b.table_stride;
        const uint32_t lb = 31 - __clz(a.c.page_size / 16);  // log2 of the blocks of a page: 0, 1 or 2
        uint32_t n = 0;  // steps whose copies were issued
        bool ok = true;
        for (uint32_t j0 = 0; j0 < steps && ok; j0 += LS) {
            const int32_t blk = b0 + (int32_t)(j0 * NB + lane);
            const int32_t page = blk < b1 ? __ldg(table + ((uint32_t)blk >> lb)) : -1;
            const uint32_t sub = (uint32_t)blk & ((1u << lb) - 1);
            const bool hidden = (uint32_t)page >= a.c.n_pages;
            if (hidden && blk < b1) flag_error(a.err, DEV_ERR_POSITION);
            float sk = 0.f, sv = 0.f;
            if (!hidden) {
                const uint64_t at = (uint32_t)page * a.c.scale_stride + (h << lb) + sub;
                sk = __ldg(a.c.ks + at);
                sv = __ldg(a.c.vs + at);
            }
            const uint64_t code = hidden ? 0 : (uint32_t)page * a.c.page_stride + (uint64_t)(h * a.c.page_size + 16 * sub) * HD;
            auto copies = [&](uint32_t j) {
                const uint32_t rs = j % RAW, i = j - j0;
                if (j >= RAW) ok = warp_wait(&c_empty[rs], (j / RAW - 1) & 1, &abort_flag);
                if (!ok) return;
                const bool mine = lane / NB == i && !hidden;
                const uint32_t count = __popc(__ballot_sync(0xffffffffu, mine));
                if (lane == 0) mbar_arrive_expect_tx(&c_full[rs], count * (2 * 16 * HD));
                __syncwarp();
                if (mine) {
                    uint8_t* dst = sraw + rs * (2 * NP * HD) + lane % NB * (16 * HD);
                    tma_load_1d(dst, a.c.k + code, 16 * HD, &c_full[rs]);
                    tma_load_1d(dst + NP * HD, a.c.v + code, 16 * HD, &c_full[rs]);
                }
                ++n;
            };
            // (a page that is not there: weights of 0 that are not counted; a scale of 0: weights that are)
            sv = zero_if_subnormal(sv);
            const bool plain = sv > 0.f && sv < INFINITY && lift_of(sv) == 0.f;
            const float e = hidden ? -INFINITY : !plain ? INFINITY : F32 ? 0.f : log2f(sv), down = !F32 && plain ? __fdiv_rn(1.f, sv) : 0.f;
            for (uint32_t g = 0; g < LS / FG && j0 + g * FG < steps && ok; ++g) {
                const uint32_t grp = j0 / FG + g;
                if (grp >= 2) ok = warp_wait(&f_empty[grp % 2], (grp / 2 - 1) & 1, &abort_flag);
                __syncwarp();
                if (lane / NB / FG == g) f_blk[(j0 + lane / NB) % FS][lane % NB] = make_float4(sk, e, down, sv);
                __syncwarp();
                if (lane == 0) mbar_arrive(&f_full[grp % 2]);
                for (uint32_t i = 0; i < FG && j0 + g * FG + i < steps && ok; ++i) copies(j0 + g * FG + i);
            }
        }
        if (!ok)  // copies in flight land before the CTA leaves
            for (uint32_t i = 0; i < RAW && i < n; ++i) mbar_wait(&c_full[i], ((n - 1 - i) / RAW) & 1);
    } else if (warp < kSoftWarps + 4 + used && steps && elect_one()) {
        // ---------------------------------------------------------------- MMA: one thread per row tile, so that
        // one tile's products run while the other waits for its weights
        const uint32_t rt = warp - kSoftWarps - 4;
        const uint32_t d = tm + rt * kTileCols, qb = smem_addr(sq + rt * kQParts * kQPart);
        bool ok = bwait(&q_full, 0, &abort_flag);
        auto scores = [&](uint32_t j) {
            const uint32_t st = j % ST;
            // the buffer holds the weights of step j - nsb until their product has ended (products of
            // different shapes are not ordered by their issue)
            ok = ok && (j < nsb || bwait(&o_done[rt][j % nsb], ((j >> lsb) - 1) & 1, &abort_flag)) &&
                 bwait(&k_full[st], (j / ST) & 1, &abort_flag);
            if (!ok) return;
            tc_after();
            const uint32_t kb = smem_addr(skv + st * kStage), ds = d + HD + j % nsb * kSCols;
            if constexpr (!F32) {
#pragma unroll
                for (uint32_t k = 0; k < HD / 16; ++k)
                    mma_ss(ds, swizzled_desc(qb + (k / 4) * (kTileRows * 128) + (k % 4) * 32, 16),
                           swizzled_desc(kb + (k / 4) * (NP * 128) + (k % 4) * 32, 16), f16_idesc(NP), k > 0);
            } else {
#pragma unroll
                for (uint32_t x = 0; x < 3; ++x)
#pragma unroll
                    for (uint32_t k = 0; k < HD / 32; ++k)
                        mma_i8(ds + x * NP, bytes_desc<HD>(qb + x * kQPart + (k / 4) * (kTileRows * 128) + (k % 4) * 32),
                               bytes_desc<HD>(kb + (k / 4) * (NP * 128) + (k % 4) * 32), i8_idesc(NP), k > 0);
            }
            mma_commit(&s_full[rt][j % nsb]);
            mma_commit(&k_empty[st]);
        };
        scores(0);
        for (uint32_t j = 0; j < steps && ok; ++j) {
            if (j + 1 < steps) scores(j + 1);
            const uint32_t st = j % ST, vb = smem_addr(skv + st * kStage + kK);
            ok = ok && bwait(&v_full[st], (j / ST) & 1, &abort_flag) &&
                 bwait(&p_full[rt][j % nsb], (j >> lsb) & 1, &abort_flag);
            if (!ok) break;
            tc_after();
            const uint32_t pw = d + HD + j % nsb * kSCols;
#pragma unroll
            for (uint32_t x = 0; x < (uint32_t)PARTS; ++x)
#pragma unroll
                for (uint32_t k = 0; k < NP / 16; ++k)
                    mma_ts(d, pw + x * (NP / 2) + 8 * k, swizzled_desc(vb + k * 2048, NP * 128), bf16_idesc(HD),
                           j % G || x > 0 || k > 0);
            mma_commit(&o_done[rt][j % nsb]);
            mma_commit(&v_empty[st]);
        }
        if (!ok) {  // the MMAs in flight end before the tensor memory is freed
            mma_commit(&fin[rt]);
            mbar_wait(&fin[rt], 0);
        }
    }
    __syncwarp();
    tc_before();
    __syncthreads();
    if (tid == 0 && abort_flag) flag_error(a.err, DEV_ERR_WAIT_TIMEOUT);
    if (warp == kSoftWarps + 4)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512) : "memory");
}

struct Shape {
    uint32_t group, row_tiles, tile_rows, chunk, splits;
    bool tiles;      // the prompt kernel
    uint64_t slots, sums;  // tiles with partials in the workspace (0: one chunk), with sums there (0: they stay in tensor memory)
};
Shape shape_of(const Kv8Cache& c, const Kv8Batch& b, uint32_t heads, uint32_t type, int sms) {
    Shape r;
    r.group = heads / c.kv_heads;
    const bool f32 = type == GGML_F32;
    const uint64_t rows = (uint64_t)std::max(1u, b.max_new) * r.group;
    const uint32_t blocks = std::max(1u, (b.max_len + 15) / 16);
    r.tiles = rows >= tile_min(f32) &&
              (double)b.n_seqs * c.kv_heads * blocks * ((rows + kRows - 1) / kRows) >= (double)kTileWork * 3 * kWarps * sms;
    const Role role = role_of((int)c.head_dim, f32);
    r.tile_rows = r.tiles ? role.rt * kTileRows : kRows;
    r.row_tiles = (uint32_t)((rows + r.tile_rows - 1) / r.tile_rows);
    // chunks of positions: enough CTAs for three on every SM (the prompt kernel: one; one row tile of 256
    // dims: two, as many as run at once -- 32768 positions over 4 kv heads 27 us against 37 with three;
    // several row tiles read the same pages, and three measured better: 2 tokens over 4099 positions of 9 sequences 21
    // against 26, though 4 over 32768 of one 49 against 37), each with at
    // least 8 blocks (two per warp, two steps of the prompt kernel). More chunks measured slower: a
    // CTA's fixed cost is about 4 us.
    const uint64_t tiles = (uint64_t)b.n_seqs * c.kv_heads * r.row_tiles;
    const uint64_t want = std::max<uint64_t>(1, (r.tiles ? 1ull : c.head_dim == 256 && r.row_tiles == 1 ? 2ull : 3ull) * sms / std::max<uint64_t>(1, tiles));
    r.chunk = std::max(8u, (uint32_t)((blocks + want - 1) / want));
    r.chunk = (r.chunk + 3) / 4 * 4;
    if (!r.tiles && !f32) r.chunk = std::min(r.chunk, kSumBlocks * kWarps);
    r.splits = (blocks + r.chunk - 1) / r.chunk;
    r.slots = r.splits > 1 ? tiles * r.splits : 0;
    r.sums = r.tiles && std::min(r.chunk, blocks) * 16 > sum_steps(role.np, f32) * role.np ? tiles * r.splits : 0;
    return r;
}

// the kernel's shared memory beyond the default, once per device (the attribute is the same for every call)
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

template <class T, int HD> cudaError_t launch(const Plan& p, bool tiles, cudaStream_t s) {
    if (tiles) {
        constexpr bool f32 = sizeof(T) == 4;
        constexpr uint32_t smem = tile_smem(HD, f32), threads = 32 * (5 * role_of(HD, f32).rt + 5);
        cudaError_t e = opt_in<kv8_tile_kernel<T, HD>>(smem);
        if (e != cudaSuccess) return e;
        e = launch_chained(kv8_tile_kernel<T, HD>, dim3(p.row_tiles * p.splits, p.a.c.kv_heads, p.a.b.n_seqs), threads, smem, s, p);
        if (e != cudaSuccess) return e;
    } else {
        cudaError_t e = opt_in<kv8_split_kernel<T, HD>>(split_smem(HD));
        if (e != cudaSuccess) return e;
        e = launch_chained(kv8_split_kernel<T, HD>, dim3(p.splits, p.row_tiles * p.a.c.kv_heads, p.a.b.n_seqs), 32 * kWarps,
                           split_smem(HD), s, p);
        if (e != cudaSuccess) return e;
    }
    if (p.splits == 1) return cudaSuccess;
    return launch_chained(kv8_join_kernel<T, HD>, dim3(p.a.b.max_new, p.a.heads, p.a.b.n_seqs), 32 * kJoinWarps, 0, s, p);
}
template <class T> cudaError_t by_dim(const Plan& p, bool tiles, cudaStream_t s) {
    return p.a.c.head_dim == 64    ? launch<T, 64>(p, tiles, s)
           : p.a.c.head_dim == 128 ? launch<T, 128>(p, tiles, s)
                                   : launch<T, 256>(p, tiles, s);
}

}  // namespace

uint64_t kv8_attention_ws_bytes(const Kv8Cache& c, const Kv8Batch& b, uint32_t heads, uint32_t type, int sms) {
    const Shape sh = shape_of(c, b, heads, type, sms);
    return sh.slots * sh.tile_rows * (c.head_dim + 2) * 4 + sh.sums * sh.tile_rows * c.head_dim * 4;
}

cudaError_t launch_kv8_attention(const Kv8AttnArgs& a, int sms, cudaStream_t s) {
    const Shape sh = shape_of(a.c, a.b, a.heads, a.type, sms);
    if ((!sh.tiles && (uint64_t)sh.row_tiles * a.c.kv_heads > 65535) || (uint64_t)sh.row_tiles * sh.splits > 0x7fffffffull)
        return cudaErrorInvalidValue;
    Plan p;
    p.a = a;
    p.group = sh.group;
    p.row_tiles = sh.row_tiles;
    p.tile_rows = sh.tile_rows;
    p.chunk = sh.chunk;
    p.splits = sh.splits;
    p.part_o = reinterpret_cast<float*>(a.ws);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + sh.slots * sh.tile_rows * a.c.head_dim);
    p.sums = reinterpret_cast<float4*>(p.part_ml + sh.slots * sh.tile_rows);  // (tiles have 128 rows or 256: 16-byte aligned)
    switch (a.type) {
        case GGML_F32: return by_dim<float>(p, sh.tiles, s);
        case GGML_F16: return by_dim<__half>(p, sh.tiles, s);
        case GGML_BF16: return by_dim<__nv_bfloat16>(p, sh.tiles, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace evl
