// int8_gemm.cu -- y[m][n] = (sum_k x[m][k] w[n][k]) * xs[m] * ws[n] (+ add[m][n]) over 8-bit
// integers, on the 5th-generation tensor cores (tcgen05 kind::i8, exact int32 sums).
//
// The weight rows are the MMA's M dimension (128 TMEM lanes) and the tokens its N: a warp
// reading one accumulator column back then holds 32 neighbouring outputs of one token, so the
// row-major output is written in whole sectors without a transpose, and a product of few tokens
// costs N = 16, not 128.
//
// i8_gemm_kernel: one CTA works on tiles of 128 weight rows x NT tokens:
//   warp 0     TMA producer: 128-byte K slices (128-byte swizzle) of both operands into a ring
//              completing on mbarriers; ragged rows and a ragged K are zero-filled by TMA;
//   warp 1     owns the tensor memory; one thread issues 4 MMAs (K = 32 each) per slice;
//   the others epilogue, one TMEM lane quadrant each (eight warps: two share a quadrant's columns);
//              two accumulators, so a tile is written while the next one is multiplied.
// With few tiles the K range is split over the CTAs of a cluster: the int32 partial tiles meet
// through distributed shared memory, each CTA adding and writing its share of the columns, in
// one launch, without a workspace, and exactly (integer sums).
//
// i8_gemm_pair_kernel: many tokens, 256 weight rows x 256 tokens on two CTAs that share their MMAs
// (cta_group::2): each brings its own 128 weight rows and half of the tokens, so a slice costs each SM
// 32 KB from L2 for 512 cycles of the tensor pipe where a CTA alone (128 x 256) needs 48 KB.
//
// Clusters of different launches share no SM's tensor memory beyond its 512 columns (a ring of half an
// SM's shared memory goes with 64 columns at most, larger rings leave no room for a second CTA), so none
// waits for a cluster that waits for it.
//
// Bound: few tokens -- HBM, every weight byte once; many tokens -- the tensor pipe. Measured:
//   1 token, 6144 x 4096, f32 out           7.6 us   3.3 TB/s (a launch, one ring's fill and a cluster's exchange)
//   33 tokens, 5120 x 25600, bf16, added     28 us   4.7 TB/s (71 % of a copy's rate)
//   4096 tokens, 24576 x 4096, bf16         282 us   2920 TOP/s (tensor pipe busy 78 % of the cycles; 535 us with
//                                                    128 x 256 tiles on single CTAs)
// Every wait on an mbarrier is bounded; on a timeout the CTA records DEV_ERR_WAIT_TIMEOUT, lets its copies and
// MMAs land, frees its tensor memory and leaves. The allocation of tensor memory and the cluster's barriers have no
// limit of their own: a CTA that holds tensor memory waits only for its cluster, whose CTAs start together, and
// for the kernel before it in the stream, all of whose CTAs hold what they need by then; so one that waits
// for the allocation waits for CTAs that come to their end.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "int8.cuh"

namespace evl {
namespace {

constexpr uint32_t kTileN = 128;                    // weight rows per tile (TMEM lanes)
constexpr uint32_t kSlice = 128;                    // K values (bytes) per stage: one swizzle atom
constexpr uint32_t kMaxStages = 12;
constexpr uint32_t kSmemCap = 200 * 1024;
constexpr uint32_t kTwoCtas = 32;                   // tokens of a tile up to which two CTAs share an SM

struct Plan {
    CUtensorMap wmap, xmap;
    I8GemmArgs a;
    uint32_t ntiles, mtiles;  // weight tiles, token tiles
    uint32_t slices;          // of K
    uint32_t split;           // CTAs (cluster) per tile
    uint32_t group;           // token tiles that share a pass over the weight tiles
    uint32_t stages;
};

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int32_t x, int32_t y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
        : "memory");
}
// K-major operand, 128-byte swizzle: 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::i8: signed 8-bit A and B, K-major, int32 D
__host__ __device__ constexpr uint32_t i8_idesc(uint32_t n, uint32_t m = 128) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16(uint32_t t, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(t)
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
__device__ __forceinline__ void tmem_ldc(uint32_t t, uint32_t (&v)[16]) { tmem_ld16(t, v); }
__device__ __forceinline__ void tmem_ldc(uint32_t t, uint32_t (&v)[32]) { tmem_ld32(t, v); }
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

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

// Tile number -> (weight tile, token tile): within a group of token tiles the tokens run fastest, so the
// CTAs at work share few weight rows and the group's tokens stay in L2.
__device__ __forceinline__ void tile_at(const Plan& P, uint32_t tile, uint32_t& nt, uint32_t& mt) {
    const uint32_t per = P.group * P.ntiles, g = tile / per, r = tile % per;
    const uint32_t here = min(P.group, P.mtiles - g * P.group);
    nt = r / here;
    mt = g * P.group + r % here;
}

// Outputs of weight row n for the tokens m0 + [c0, c1), accumulators at `at` + column: C columns at a time,
// the next ones' additions on their way meanwhile (they may share y's buffer: each is read before its
// own output is written, and no other output overlaps it).
// (Loads have no conditions and are widened where they are used: a branch or a conversion beside
// each would wait for it before the next is issued.)
template <class T, uint32_t C> struct Outputs {
    T add[C];
    __device__ __forceinline__ void fetch(const I8GemmArgs& a, uint32_t m, uint32_t count, uint32_t n, bool live) {
        if (!a.add || !live) return;
        const T* p = static_cast<const T*>(a.add) + (uint64_t)m * a.add_stride + n;
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) add[j] = p[min(j, count - 1) * a.add_stride];
    }
    __device__ __forceinline__ void put(const I8GemmArgs& a, uint32_t m, uint32_t count, uint32_t n, bool live,
                                        const uint32_t (&acc)[C], float ws) const {
        if (!live) return;
        T* p = static_cast<T*>(a.y) + (uint64_t)m * a.y_stride + n;
#pragma unroll
        for (uint32_t j = 0; j < C; ++j)
            if (j < count) {
                float y = __fmul_rn(__fmul_rn(__int2float_rn((int32_t)acc[j]), __ldg(a.xs + m + j)), ws);
                if (a.add) y = __fadd_rn(y, to_f32(add[j]));
                p[j * a.y_stride] = from_f32<T>(y);
            }
    }
};

// Outputs of token m for weight rows n .. n + 3, as far as they exist.
template <class T> __device__ __forceinline__ void put_row(const I8GemmArgs& a, uint32_t m, uint32_t n, const uint32_t (&acc)[4]) {
    const float xs = __ldg(a.xs + m);
    const T* ap = static_cast<const T*>(a.add) + (uint64_t)m * a.add_stride + n;
    T* yp = static_cast<T*>(a.y) + (uint64_t)m * a.y_stride + n;
    float add[4], ws[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        ws[j] = n + j < a.out ? __ldg(a.ws + n + j) : 0.f;
        add[j] = a.add && n + j < a.out ? to_f32(ap[j]) : 0.f;
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
        if (n + j < a.out) {
            float y = __fmul_rn(__fmul_rn(__int2float_rn((int32_t)acc[j]), xs), ws[j]);
            if (a.add) y = __fadd_rn(y, add[j]);
            yp[j] = from_f32<T>(y);
        }
}

// epilogue warps of a tile of nt tokens
__host__ __device__ constexpr uint32_t epi_warps(uint32_t nt) { return nt >= 128 ? 8 : 4; }
__host__ __device__ constexpr uint32_t gemm_threads(uint32_t nt) { return 64 + 32 * epi_warps(nt); }

template <uint32_t NT, class T>
__global__ void __launch_bounds__(gemm_threads(NT), 1) i8_gemm_kernel(const __grid_constant__ Plan P) {
    namespace cg = cooperative_groups;
    extern __shared__ uint8_t raw_smem[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], d_full[2], d_empty[2], fin;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    constexpr uint32_t kStageBytes = (kTileN + NT) * kSlice, kEpi = epi_warps(NT), kThreads = gemm_threads(NT);
    constexpr uint32_t kCols = 2 * NT < 32 ? 32 : 2 * NT;  // two accumulators (a power of two)
    const I8GemmArgs& a = P.a;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* smem = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);
    const uint32_t S = P.split, rank = blockIdx.x % S, tiles = P.ntiles * P.mtiles;
    const uint32_t s0 = (uint32_t)((uint64_t)P.slices * rank / S), s1 = (uint32_t)((uint64_t)P.slices * (rank + 1) / S);

    if (tid == 0) {
        abort_flag = 0;
        for (uint32_t i = 0; i < P.stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&d_full[i], 1);
            mbar_init(&d_empty[i], kEpi);
        }
        mbar_init(&fin, 1);
        fence_barrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = tmem_base;
    pdl_wait();
    pdl_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t n = 0;
            for (uint32_t tile = blockIdx.x / S; tile < tiles && !abort_flag; tile += gridDim.x / S) {
                uint32_t nt, mt;
                tile_at(P, tile, nt, mt);
                const int32_t w0 = (int32_t)(nt * kTileN), x0 = (int32_t)(mt * NT);
                for (uint32_t c = s0; c < s1; ++c, ++n) {
                    const uint32_t s = n % P.stages;
                    if (n >= P.stages && !bwait(&empty[s], (n / P.stages - 1) & 1, &abort_flag)) break;
                    uint8_t* dst = smem + s * kStageBytes;
                    mbar_arrive_expect_tx(&full[s], kStageBytes);
                    tma_load_2d(dst, &P.wmap, (int32_t)(c * kSlice), w0, &full[s]);
                    tma_load_2d(dst + kTileN * kSlice, &P.xmap, (int32_t)(c * kSlice), x0, &full[s]);
                }
            }
            if (abort_flag)  // copies in flight land before the CTA leaves
                for (uint32_t s = 0; s < P.stages && s < n; ++s) mbar_wait(&full[s], ((n - 1 - s) / P.stages) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t n = 0, it = 0;
            for (uint32_t tile = blockIdx.x / S; tile < tiles && !abort_flag; tile += gridDim.x / S, ++it) {
                const uint32_t acc = tm + (it & 1) * NT;
                if (it >= 2 && !bwait(&d_empty[it & 1], (it / 2 - 1) & 1, &abort_flag)) break;
                tc_after();
                for (uint32_t c = s0; c < s1; ++c, ++n) {
                    const uint32_t s = n % P.stages;
                    if (!bwait(&full[s], (n / P.stages) & 1, &abort_flag)) break;
                    tc_after();
                    const uint32_t at = smem_addr(smem + s * kStageBytes);
                    const uint64_t da = smem_desc(at), db = smem_desc(at + kTileN * kSlice);
#pragma unroll
                    for (uint32_t k = 0; k < kSlice / 32; ++k)  // 32 bytes of K further inside the swizzle atom
                        mma_i8(acc, da + 2 * k, db + 2 * k, i8_idesc(NT), c > s0 || k > 0);
                    mma_commit(&empty[s]);
                }
                mma_commit(&d_full[it & 1]);
            }
            if (abort_flag) {  // the MMAs in flight end before the tensor memory is freed
                mma_commit(&fin);
                mbar_wait(&fin, 0);
            }
        }
    } else {
        // columns of this warp: all, or half of them
        constexpr uint32_t kHalf = NT / (kEpi / 4);
        const uint32_t quad = warp & 3, r = quad * 32 + lane, c0 = (warp - 2) / 4 * kHalf;
        uint32_t it = 0;
        for (uint32_t tile = blockIdx.x / S; tile < tiles; tile += gridDim.x / S, ++it) {
            uint32_t nt, mt;
            tile_at(P, tile, nt, mt);
            const uint32_t n = nt * kTileN + r, m0 = mt * NT;
            const bool live = n < a.out;
            const float ws = live ? a.ws[n] : 0.f;
            const uint32_t cols = min(c0 + kHalf, a.rows - m0);
            constexpr uint32_t C = NT <= kTwoCtas ? 16 : 32;  // (two CTAs share the SM's registers)
            Outputs<T, C> out, next;
            if (S == 1 && c0 < cols) out.fetch(a, m0 + c0, cols - c0, n, live);
            bool ok = true;
            if (lane == 0) ok = bwait(&d_full[it & 1], (it / 2) & 1, &abort_flag);
            ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            if (!ok) break;
            tc_after();
            const uint32_t at = tm + (it & 1) * NT + ((quad * 32) << 16);
            int32_t* part = reinterpret_cast<int32_t*>(smem);  // (split: over the ring, whose slices are all read)
            for (uint32_t c = c0; c < cols; c += C) {
                uint32_t v[C];
                tmem_ldc(at + c, v);
                if (S == 1 && c + C < cols) next.fetch(a, m0 + c + C, cols - c - C, n, live);
                tmem_ld_wait();
                if (S == 1) {
                    out.put(a, m0 + c, cols - c, n, live, v, ws);
                    out = next;
                } else {  // this CTA's partial tile for the cluster
#pragma unroll
                    for (uint32_t j = 0; j < C; ++j) part[(c + j) * kTileN + r] = (int32_t)v[j];
                }
            }
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&d_empty[it & 1]);
        }
    }
    __syncwarp();
    if (S > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        uint32_t nt, mt;
        tile_at(P, blockIdx.x / S, nt, mt);
        const uint32_t n0 = nt * kTileN, m0 = mt * NT;
        const uint32_t cols = min(NT, a.rows - m0);
        const int32_t* part = reinterpret_cast<const int32_t*>(smem);
        // four neighbouring weight rows of a token per thread; every CTA's share is on its way before the
        // first is added
        for (uint32_t i = rank * kThreads + tid; i < cols * (kTileN / 4) && !abort_flag; i += S * kThreads) {
            const uint32_t c = i / (kTileN / 4), r = i % (kTileN / 4) * 4;
            int4 v[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (k < S) v[k] = *reinterpret_cast<const int4*>(cl.map_shared_rank(part + c * kTileN + r, k));
            int4 sum = v[0];
#pragma unroll
            for (uint32_t k = 1; k < 8; ++k)
                if (k < S) sum.x += v[k].x, sum.y += v[k].y, sum.z += v[k].z, sum.w += v[k].w;
            const uint32_t acc[4] = {(uint32_t)sum.x, (uint32_t)sum.y, (uint32_t)sum.z, (uint32_t)sum.w};
            put_row<T>(a, m0 + c, n0 + r, acc);
        }
        cl.sync();  // the others read this CTA's tile until here
    }
    tc_before();
    __syncthreads();
    if (tid == 0 && abort_flag) flag_error(a.err, DEV_ERR_WAIT_TIMEOUT);
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(kCols) : "memory");
}

// ------------------------------------------------------------------ two CTAs, 256 x 256
constexpr uint32_t kPairThreads = 320, kPairStage = 2 * 128 * kSlice, kPairStages = 6, kPairTokens = 256;

// the address of a shared-memory object of this CTA in the cluster's CTA `rank`
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
    return r;
}
// a load into this CTA's shared memory that completes on a barrier of the pair's first CTA
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// arrive on `bar` of both CTAs once the MMAs issued so far have ended
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_addr(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// one lane of a converged warp, in the form that tells the compiler so
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}

template <class T>
__global__ void __launch_bounds__(kPairThreads, 1) i8_gemm_pair_kernel(const __grid_constant__ Plan P) {
    namespace cg = cooperative_groups;
    extern __shared__ uint8_t raw_smem[];
    // full: of the first CTA, for both; empty, d_full: of each; d_empty: of the first CTA, from both
    __shared__ __align__(8) uint64_t full[kPairStages], empty[kPairStages], d_full[2], d_empty[2], fin;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    const I8GemmArgs& a = P.a;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    cg::cluster_group cl = cg::this_cluster();
    const uint32_t rank = cl.block_rank(), tiles = P.ntiles * P.mtiles, first = blockIdx.x / 2, stride = gridDim.x / 2;
    uint8_t* smem = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);
    if (tid == 0) {
        abort_flag = 0;
        for (uint32_t i = 0; i < kPairStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&d_full[i], 1);
            mbar_init(&d_empty[i], 16);  // eight epilogue warps of each CTA
        }
        mbar_init(&fin, 1);
        fence_barrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncwarp();
    cl.sync();  // barriers of both CTAs are there
    tc_after();
    const uint32_t tm = tmem_base;
    pdl_wait();
    pdl_launch_dependents();

    if (warp == 0) {
        if (elect_one()) {
            uint32_t n = 0;
            for (uint32_t tile = first; tile < tiles && !abort_flag; tile += stride) {
                uint32_t nt, mt;
                tile_at(P, tile, nt, mt);
                const int32_t w0 = (int32_t)(nt * 256 + rank * 128), x0 = (int32_t)(mt * kPairTokens + rank * 128);
                for (uint32_t c = 0; c < P.slices; ++c, ++n) {
                    const uint32_t s = n % kPairStages;
                    if (n >= kPairStages && !bwait(&empty[s], (n / kPairStages - 1) & 1, &abort_flag)) break;
                    uint8_t* dst = smem + s * kPairStage;
                    const uint32_t bar = in_cta(&full[s], 0);
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kPairStage);
                    tma_load_pair(dst, &P.wmap, (int32_t)(c * kSlice), w0, bar);
                    tma_load_pair(dst + 128 * kSlice, &P.xmap, (int32_t)(c * kSlice), x0, bar);
                }
            }
            if (abort_flag && rank == 0)  // copies in flight land before the CTAs leave
                for (uint32_t s = 0; s < kPairStages && s < n; ++s) mbar_wait(&full[s], ((n - 1 - s) / kPairStages) & 1);
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            uint32_t n = 0, it = 0;
            for (uint32_t tile = first; tile < tiles && !abort_flag; tile += stride, ++it) {
                const uint32_t acc = tm + (it & 1) * kPairTokens;
                if (it >= 2 && !bwait(&d_empty[it & 1], (it / 2 - 1) & 1, &abort_flag)) break;
                tc_after();
                for (uint32_t c = 0; c < P.slices; ++c, ++n) {
                    const uint32_t s = n % kPairStages;
                    if (!bwait(&full[s], (n / kPairStages) & 1, &abort_flag)) break;
                    tc_after();
                    const uint32_t at = smem_addr(smem + s * kPairStage);
                    const uint64_t da = smem_desc(at), db = smem_desc(at + 128 * kSlice);
#pragma unroll
                    for (uint32_t k = 0; k < kSlice / 32; ++k)
                        mma_i8_pair(acc, da + 2 * k, db + 2 * k, i8_idesc(kPairTokens, 256), c > 0 || k > 0);
                    commit_pair(&empty[s]);
                }
                commit_pair(&d_full[it & 1]);
            }
            if (abort_flag) {  // the MMAs in flight end before the tensor memory is freed
                commit_pair(&fin);
                mbar_wait(&fin, 0);
            }
        }
    } else {
        const uint32_t quad = warp & 3, r = quad * 32 + lane, c0 = (warp - 2) / 4 * 128;
        uint32_t it = 0;
        for (uint32_t tile = first; tile < tiles; tile += stride, ++it) {
            uint32_t nt, mt;
            tile_at(P, tile, nt, mt);
            const uint32_t n = nt * 256 + rank * 128 + r, m0 = mt * kPairTokens, cols = min(c0 + 128, a.rows - m0);
            const bool live = n < a.out;
            const float ws = live ? a.ws[n] : 0.f;
            Outputs<T, 32> out, next;
            if (c0 < cols) out.fetch(a, m0 + c0, cols - c0, n, live);
            bool ok = true;
            if (lane == 0) ok = bwait(&d_full[it & 1], (it / 2) & 1, &abort_flag);
            ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            if (!ok) break;
            tc_after();
            const uint32_t at = tm + (it & 1) * kPairTokens + ((quad * 32) << 16);
            for (uint32_t c = c0; c < cols; c += 32) {
                uint32_t v[32];
                tmem_ld32(at + c, v);
                if (c + 32 < cols) next.fetch(a, m0 + c + 32, cols - c - 32, n, live);
                tmem_ld_wait();
                out.put(a, m0 + c, cols - c, n, live, v, ws);
                out = next;
            }
            tc_before();
            __syncwarp();
            if (lane == 0) arrive_remote(in_cta(&d_empty[it & 1], 0));
        }
    }
    __syncwarp();
    tc_before();
    cl.sync();  // the pair's MMAs and copies have ended, nothing more arrives at the other's barriers
    if (tid == 0 && abort_flag) flag_error(a.err, DEV_ERR_WAIT_TIMEOUT);
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512) : "memory");
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// [rows][cols] bytes, rows `stride` apart, read in boxes of box_rows x 128 bytes; outside: zeros
bool make_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t stride, uint32_t box_rows) {
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {stride};
    const cuuint32_t box[2] = {kSlice, box_rows}, unit[2] = {1, 1};
    return encoder() && encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, unit,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// the kernel's shared memory beyond the default, once per device
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

// a launch in clusters of `cluster` CTAs that may begin while the kernel before it ends
template <auto kernel> cudaError_t go(const Plan& p, uint32_t grid, uint32_t threads, uint32_t smem, uint32_t cluster, cudaStream_t s) {
    cudaError_t e = opt_in<kernel>(kSmemCap + 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Clusters of `cluster` CTAs that the device runs at once (a cluster stays inside one GPC, so this is less
// than SMs / cluster); looked up once per device.
template <auto kernel> uint32_t clusters_at_once(uint32_t threads, uint32_t smem, uint32_t cluster) {
    static std::atomic<int> known[64][9];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || cluster > 8) return 0;
    int n = known[dev][cluster].load();
    if (!n) {
        if (opt_in<kernel>(kSmemCap + 1024) != cudaSuccess) return 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(cluster);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = cluster;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0;
        known[dev][cluster] = n ? n : -1;
    }
    return n > 0 ? (uint32_t)n : 0;
}

constexpr uint32_t kGroup = 16;  // token tiles per pass over the weights

__host__ __device__ constexpr uint32_t stage_bytes(uint32_t nt) { return (kTileN + nt) * kSlice; }
constexpr uint32_t ctas_per_sm(uint32_t nt) { return nt <= kTwoCtas ? 2 : 1; }
constexpr uint32_t ring_stages(uint32_t nt) {
    const uint32_t n = kSmemCap / ctas_per_sm(nt) / stage_bytes(nt);
    return n < kMaxStages ? n : kMaxStages;
}
// the ring; a cluster's partial tile lies over it
constexpr uint32_t gemm_smem(uint32_t nt) {
    const uint32_t ring = ring_stages(nt) * stage_bytes(nt), part = nt * kTileN * 4;
    return (ring > part ? ring : part) + 1024;
}

// How a product is cut: nt 0 is the pair kernel.
struct Cut {
    uint32_t nt = 0, split = 1;
    double cost = 1e30;
};
// Estimated SM cycles, the coefficients fitted to 105 shapes in every cut (1 to 1024 tokens, 578 to 24576
// weight rows, 200 to 25600 columns; the chosen cut is 1.5 % slower than the best one on average, 13 % at
// most): a slice costs L2 3.9 cycles per 128-byte row of the two operands or the tensor pipe 3.6 per token
// column, whichever is more; outputs 45 per column of an epilogue warp, 40 more with an addition,
// 30 more for a split's exchange; a launch 4000.
double cost_of(uint32_t nt, uint64_t tiles, uint32_t split, uint32_t slices, bool add, int sms) {
    const uint32_t cols = nt ? nt : 256, rows = nt ? kTileN + nt : 256;
    const double share = nt ? ctas_per_sm(nt) : 1;  // CTAs that share an SM's pipes and bandwidth
    const double slots = nt ? sms * share : sms / 2;
    const double per = (double)slices / split * share * std::max(3.9 * rows, 3.6 * cols);
    const double out = (45.0 + (add ? 40.0 : 0.0) + (split > 1 ? 30.0 : 0.0)) * cols / (cols >= 128 ? 2 : 1);
    const double waves = std::ceil((double)tiles * split / slots);
    // outputs of all tiles but the last are written behind the next tile's products
    return 4000.0 + waves * per + out + (waves - 1) * std::max(0.0, out - per);
}

template <uint32_t NT, class T> void consider(Cut& best, const Plan& p, int sms) {
    const uint64_t tiles = ((p.a.out + kTileN - 1) / kTileN) * (uint64_t)((p.a.rows + NT - 1) / NT);
    if (NT > 16 && p.a.rows <= NT / 2) return;  // half of the columns would be empty
    for (uint32_t k = 1; k <= 8; ++k) {
        if (k > 1) {  // a split's clusters all run at once, every CTA with four slices at least
            if (k * tiles > 2ull * sms || p.slices < 4 * k) break;
            // (the occupancy query counts one CTA per SM)
            if (tiles > (uint64_t)ctas_per_sm(NT) * clusters_at_once<i8_gemm_kernel<NT, T>>(gemm_threads(NT), gemm_smem(NT), k))
                continue;
        }
        const double c = cost_of(NT, tiles, k, p.slices, p.a.add != nullptr, sms);
        if (c < best.cost) best.nt = NT, best.split = k, best.cost = c;
    }
}

template <uint32_t NT, class T> cudaError_t launch(Plan& p, uint32_t split, int sms, cudaStream_t s) {
    const I8GemmArgs& a = p.a;
    if (!make_map(&p.wmap, a.w, a.out, a.cols, a.w_stride, kTileN) ||
        !make_map(&p.xmap, a.x, a.rows, a.cols, a.x_stride, NT))
        return cudaErrorInvalidValue;
    p.ntiles = (a.out + kTileN - 1) / kTileN;
    p.mtiles = (a.rows + NT - 1) / NT;
    p.group = kGroup;
    p.stages = ring_stages(NT);
    p.split = split;
    const uint64_t tiles = (uint64_t)p.ntiles * p.mtiles;
    if (tiles > 0x7fffffffull) return cudaErrorInvalidValue;
    const uint32_t grid = split > 1 ? (uint32_t)tiles * split : (uint32_t)std::min<uint64_t>(tiles, (uint64_t)sms * ctas_per_sm(NT));
    return go<i8_gemm_kernel<NT, T>>(p, grid, gemm_threads(NT), gemm_smem(NT), split, s);
}

template <class T> cudaError_t launch_pair(Plan& p, int sms, cudaStream_t s) {
    const I8GemmArgs& a = p.a;
    if (!make_map(&p.wmap, a.w, a.out, a.cols, a.w_stride, 128) ||
        !make_map(&p.xmap, a.x, a.rows, a.cols, a.x_stride, 128))
        return cudaErrorInvalidValue;
    p.ntiles = (a.out + 255) / 256;
    p.mtiles = (a.rows + kPairTokens - 1) / kPairTokens;
    p.group = kGroup;
    p.split = 1;
    p.stages = kPairStages;
    const uint64_t tiles = (uint64_t)p.ntiles * p.mtiles;
    if (tiles > 0x7fffffffull) return cudaErrorInvalidValue;
    static_assert(kPairStages * kPairStage <= kSmemCap, "shared memory");
    const uint32_t grid = 2 * (uint32_t)std::min<uint64_t>(tiles, sms / 2);
    return go<i8_gemm_pair_kernel<T>>(p, grid, kPairThreads, kPairStages * kPairStage + 1024, 2, s);
}

template <class T> Cut cut_for(Plan& p, int sms) {
    p.slices = (p.a.cols + kSlice - 1) / kSlice;
    Cut best;
    consider<16, T>(best, p, sms);
    consider<32, T>(best, p, sms);
    consider<64, T>(best, p, sms);
    consider<128, T>(best, p, sms);
    consider<256, T>(best, p, sms);
    if (p.a.rows > 128) {
        const uint64_t tiles = (uint64_t)((p.a.out + 255) / 256) * ((p.a.rows + 255) / 256);
        const double c = cost_of(0, tiles, 1, p.slices, p.a.add != nullptr, sms);
        if (c < best.cost) best.nt = 0, best.split = 1, best.cost = c;
    }
    return best;
}

template <class T> cudaError_t by_tokens(Plan& p, int sms, cudaStream_t s) {
    const Cut best = cut_for<T>(p, sms);
    switch (best.nt) {
        case 0: return launch_pair<T>(p, sms, s);
        case 16: return launch<16, T>(p, best.split, sms, s);
        case 32: return launch<32, T>(p, best.split, sms, s);
        case 64: return launch<64, T>(p, best.split, sms, s);
        case 128: return launch<128, T>(p, best.split, sms, s);
        default: return launch<256, T>(p, best.split, sms, s);
    }
}

}  // namespace

cudaError_t launch_i8_gemm(const I8GemmArgs& a, int sms, cudaStream_t s) {
    Plan p;
    p.a = a;
    switch (a.type) {
        case GGML_F32: return by_tokens<float>(p, sms, s);
        case GGML_F16: return by_tokens<__half>(p, sms, s);
        case GGML_BF16: return by_tokens<__nv_bfloat16>(p, sms, s);
        default: return cudaErrorInvalidValue;
    }
}

void i8_gemm_cut(const I8GemmArgs& a, int sms, uint32_t& tokens, uint32_t& split) {
    Plan p;
    p.a = a;
    const Cut c = a.type == GGML_F32 ? cut_for<float>(p, sms) : a.type == GGML_F16 ? cut_for<__half>(p, sms) : cut_for<__nv_bfloat16>(p, sms);
    tokens = c.nt, split = c.split;
}

}  // namespace evl
