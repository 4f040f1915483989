// The 8-bit floating-point product for many rows: y[m, n] = sum over blocks b of 128 k: xs[m, b] ws[n / 128, b] * (x w^T of the block), tcgen05.
//
// The tensor cores cannot apply FP32 scales, so a block's product is an accumulator of its own: four MMAs (32 k each) start it from zero, and eight warps read it back from
// tensor memory, scale it and add it to sums that they hold in registers, while the MMAs of the next block fill the other of two accumulators.  A thread has one row of x (a
// lane of tensor memory) and half the tile's columns, all of one block of weight rows, so its scale is one number a block: one read and half a packed multiply-add a column.
//
// Warp 8 brings x and w in stages of 128 k by tensor copies, warp 9 issues the MMAs.  Two forms:
//   pairs    a cluster of two CTAs has a tile of 256 x 256 (MMAs of cta_group::2: each CTA holds 128 rows of x and half the weight rows, so a stage's bytes feed twice the work);
//            pairs are persistent, the MMAs run on into the next tile while the sums of the last are stored.
//            8192 x 8192 x 4096: 230 to 240 us (2.29 to 2.40 PFLOP/s) in bursts, 276 at the power limit, copies and MMAs alone 176; FP32 rows, which leave from registers, 304.  A pair has 448 blocks of
//            some 890 cycles there (1.64 GHz), of which the tensor pipe is busy for 560: the rest is taken to be the hand-over (two accumulators, given back when the last of their columns has been read), not measured apart.
//   tiles    a CTA has a tile of 128 x 128; where tiles are few, a cluster of up to eight CTAs shares its k, and adds the parts up through distributed shared memory in rank order.
//            What bounds it is the fill from L2, some 48 bytes a clock and SM, and behind it the parts' way (150 x 2560 x 4096: 11.6 us, of them 4.2 to the first block).
// Up to 32 rows of x take a form of their own, further down.

#include "linear_f8.cuh"
#include "skinny_mma.cuh"
#include "tc_ptx.cuh"

namespace sxb {
namespace {

constexpr int kSumWarps = 8, kCopyWarp = kSumWarps, kMmaWarp = kSumWarps + 1;
constexpr int kTileM = 128;                  // rows of x of a CTA: the lanes of tensor memory
constexpr int kLine = kF8Block;              // bytes of a stage's row: a block of k
constexpr int kStages = 5;
constexpr int kTmemCols = 512;
// A third warpgroup beside the two that sum, to which most of its registers go: 40 and 232 a thread are the 168 that 384 threads were launched with.
constexpr int kThreads = 384;
constexpr int kAtOnce = 32;                  // columns of an accumulator that a thread asks for at once

template <int CTAS, int BN>
struct Shape {
    static constexpr int kBRows = BN / CTAS;                                   // weight rows that a CTA holds
    static constexpr int kStageBytes = (kTileM + kBRows) * kLine;
    static constexpr int kAccs = 512 / BN;                                     // accumulators: all of tensor memory
    static constexpr size_t kRing = (size_t)kStages * kStageBytes, kOut = (size_t)kTileM * BN * 2;  // and a tile's rows of y in BF16, on their way out
    static constexpr size_t kSmem = kRing + kOut + 1024;
    static_assert(kOut >= kSumWarps * 4096 && kSmem <= 226 * 1024 && (CTAS == 2 || (size_t)kTileM * BN * 4 <= kRing));
};

struct TcArgs8 {
    F8Args g;
    int n_m, n_n, band;  // tiles along m and n; tiles along m of a band, in which all of n is gone through
    int split;           // CTAs that share a tile's k (tiles)
    int rows;            // of x, of a tile of one CTA: up to kTileM, alike in all tiles
    int vec;             // bytes of y that may be stored at once
    int tensor_out;      // y (BF16) takes tensor copies
    int xs4;             // four scales of a row of x may be loaded at once
    uint32_t *status;
    unsigned long long wait_limit_ns;
    int test_skip_slot;
};

// Instruction descriptor of kind::f8f6f4: D FP32 (bits [4,6) = 1), A and B e4m3 (formats 0), both K-major, N >> 3 at bits [17,23), M >> 4 at bits [24,29).
__device__ inline uint32_t instr_desc_e4m3(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// D[tmem] = A[smem] * B[smem] over a stage, both 128-byte-swizzled: four MMAs of 32 k, issued by the lane with leader = 1 of a whole warp.
template <int CTAS>
__device__ inline void tc_block_e4m3(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc) {
    if constexpr (CTAS == 1)
        asm volatile(
            "{\n\t.reg .pred q, zero, one;\n\t.reg .b32 x1, x2, x3, y1, y2, y3;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t"
            "setp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 zero, 0, 0;\n\tsetp.eq.b32 one, 0, 0;\n\t"
            "add.u32 x1, %1, 2;\n\tadd.u32 x2, %1, 4;\n\tadd.u32 x3, %1, 6;\n\tadd.u32 y1, %2, 2;\n\tadd.u32 y2, %2, 4;\n\tadd.u32 y3, %2, 6;\n\t"
            "mov.b64 a0, {%1, %3};\n\tmov.b64 a1, {x1, %3};\n\tmov.b64 a2, {x2, %3};\n\tmov.b64 a3, {x3, %3};\n\t"
            "mov.b64 b0, {%2, %3};\n\tmov.b64 b1, {y1, %3};\n\tmov.b64 b2, {y2, %3};\n\tmov.b64 b3, {y3, %3};\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a0, b0, %4, zero;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a1, b1, %4, one;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a2, b2, %4, one;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a3, b3, %4, one;\n\t}" ::"r"(d),
            "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(leader)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred q, zero, one;\n\t.reg .b32 x1, x2, x3, y1, y2, y3;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t"
            "setp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 zero, 0, 0;\n\tsetp.eq.b32 one, 0, 0;\n\t"
            "add.u32 x1, %1, 2;\n\tadd.u32 x2, %1, 4;\n\tadd.u32 x3, %1, 6;\n\tadd.u32 y1, %2, 2;\n\tadd.u32 y2, %2, 4;\n\tadd.u32 y3, %2, 6;\n\t"
            "mov.b64 a0, {%1, %3};\n\tmov.b64 a1, {x1, %3};\n\tmov.b64 a2, {x2, %3};\n\tmov.b64 a3, {x3, %3};\n\t"
            "mov.b64 b0, {%2, %3};\n\tmov.b64 b1, {y1, %3};\n\tmov.b64 b2, {y2, %3};\n\tmov.b64 b3, {y3, %3};\n\t"
            "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a0, b0, %4, zero;\n\t"
            "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a1, b1, %4, one;\n\t"
            "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a2, b2, %4, one;\n\t"
            "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a3, b3, %4, one;\n\t}" ::"r"(d),
            "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(leader)
            : "memory");
}
// What was issued before has completed: an arrival at the barrier, in both CTAs of a pair.
template <int CTAS>
__device__ inline void commit_to(uint32_t leader, uint64_t *bar) {
    if constexpr (CTAS == 1) tc_commit_if(leader, bar);
    else
        asm volatile(
            "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
            "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(smem_u32(bar)),
            "r"(leader), "h"((uint16_t)3)
            : "memory");
}
// A box of x or w into this CTA's shared memory, counted at the barrier `bar` (an address in the cluster's window: the first CTA's of a pair).
template <int CTAS>
__device__ inline void load_box(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    if constexpr (CTAS == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
                     : "memory");
}
// The same place in the shared memory of the cluster's CTA `rank`.
__device__ inline uint32_t in_cta(const void *p, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ inline uint32_t in_first_cta(uint64_t *bar) { return in_cta(bar, 0); }
// What a kernel does before it may touch memory of the grid ahead: its tensor maps are fetched.
__device__ inline void fetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory"); }
__device__ inline void arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ inline void cluster_meet() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }

// 32 consecutive columns of this thread's TMEM lane: asked for, and there.  (The second names the registers, so that nothing reads them before it.)
__device__ inline void tc_ask(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
          "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ inline void tc_there(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
                   "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                   "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])::"memory");
}
__device__ inline void tc_ask(uint32_t taddr, float (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
                   "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ inline void tc_there(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
                   "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}
__device__ inline void store32(void *p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// FP32 values to y at `at`, 16-byte aligned, `left` of which lie inside the row.
template <int NV>
__device__ inline void store_run(const TcArgs8 &a, int64_t at, int left, const float (&v)[NV]) {
    float *p = static_cast<float *>(a.g.y) + at;
#pragma unroll
    for (int i = 0; i < NV; i += 8) {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(v[i + k]);
        if (i + 8 <= left && a.vec >= 32) store32(p + i, w);
        else if (i + 8 <= left) {
            reinterpret_cast<uint4 *>(p + i)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4 *>(p + i)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k < left) p[i + k] = v[i + k];
    }
}

// A place in a ring of n barriers and the parity of the phase it is in.
struct Turn {
    int at;
    uint32_t phase;
    __device__ inline void advance(int n) {
        if (++at == n) at = 0, phase ^= 1u;
    }
};

struct Tile {
    int m, n;
};
__device__ inline Tile tile_of(const TcArgs8 &a, int item) {  // at most 2^13 x 2^17 tiles
    const int per = a.band * a.n_n, b = item / per, rest = item - b * per;
    const int in_band = min(a.band, a.n_m - b * a.band);
    return Tile{b * a.band + rest % in_band, rest / in_band};
}

// TENSOR: y leaves by tensor copies, and a pair's kernel knows no other way (with all of them in one the compiler holds the sums worse: 8192 x 8192 x 4096 271 us, so 241).
template <int CTAS, int BN, bool TENSOR>
__global__ void __launch_bounds__(kThreads, 1)
    f8_tc_kernel(const TcArgs8 a, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap ymap) {
    using S = Shape<CTAS, BN>;
    constexpr int kCols = BN / 2;  // of a summing thread
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *const smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full_bar[kStages], empty_bar[kStages], acc_full[S::kAccs], acc_empty[S::kAccs], drain_bar;
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int group = CTAS == 2 ? 2 : a.split, rank = (int)blockIdx.x % group;  // of the cluster
    const int n_items = a.n_m * a.n_n, first = (int)blockIdx.x / group, step = (int)gridDim.x / group;
    const int rows = CTAS == 2 ? kTileM : a.rows;
    auto row_of = [&](const Tile &t) { return CTAS == 2 ? (t.m * 2 + rank) * kTileM : t.m * rows; };  // of x, this CTA's first
    const int kb0 = CTAS == 2 ? 0 : (int)((int64_t)a.g.kb * rank / group), kb1 = CTAS == 2 ? a.g.kb : (int)((int64_t)a.g.kb * (rank + 1) / group);
    volatile int *const abort_v = &abort_flag;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&full_bar[s], 1), mbar_init(&empty_bar[s], 1);
        for (int b = 0; b < S::kAccs; ++b) mbar_init(&acc_full[b], 1), mbar_init(&acc_empty[b], kSumWarps * CTAS);
        mbar_init(&drain_bar, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fetch_map(&xmap), fetch_map(&wmap);
    }
    if (warp == kMmaWarp) {
        if constexpr (CTAS == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_smem)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_smem)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) cluster_meet();  // the other CTA's barriers are there
    behind_grid();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_smem;

    auto raise_abort = [&](int item, int role) {
        if (atomicExch(&abort_flag, 1) == 0 && atomicCAS(&a.status[0], 0u, 2u) == 0u) {
            a.status[1] = (uint32_t)item;
            a.status[2] = (uint32_t)role;
        }
    };

    // What every warp does last.  (Called in both branches: the warps of a pair have different numbers of registers by then.)
    auto leave = [&] {
        if (*abort_v) {  // copies that a CTA issued before it gave up have landed within this time
            const unsigned long long t0 = global_ns();
            while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
        }
        tc_fence_before();
        __syncthreads();
        if (CTAS == 1 && a.split > 1) {
            cluster_meet();  // every part is there
            const Tile t = tile_of(a, first);
            const int row0 = row_of(t), col0 = t.n * BN;
            // four neighbouring columns a thread, in turn the cluster's CTAs', parts in rank order
            if (!*abort_v)
                for (int i = rank * kThreads + (int)threadIdx.x; i < rows * BN / 4; i += group * kThreads) {
                    const int r = i / (BN / 4), c = i % (BN / 4) * 4;
                    if (row0 + r >= a.g.M || col0 + c >= a.g.N) continue;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int k = 0; k < group; ++k) {
                        float4 p;
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(p.x), "=f"(p.y), "=f"(p.z), "=f"(p.w)
                                     : "r"(in_cta(smem, k) + 4u * (uint32_t)(r * BN + (c ^ (r & 7) * 4)))
                                     : "memory");
                        v.x += p.x, v.y += p.y, v.z += p.z, v.w += p.w;
                    }
                    const int64_t at = (int64_t)(row0 + r) * a.g.y_ld + col0 + c;
                    const int left = a.g.N - col0 - c;
                    if (a.g.f32) {
                        float *p = static_cast<float *>(a.g.y) + at;
                        if (left >= 4 && a.vec >= 16) *reinterpret_cast<float4 *>(p) = v;
                        else {
                            p[0] = v.x;
                            if (left > 1) p[1] = v.y;
                            if (left > 2) p[2] = v.z;
                            if (left > 3) p[3] = v.w;
                        }
                    } else {
                        uint16_t *p = static_cast<uint16_t *>(a.g.y) + at;
                        const uint32_t lo = bf16_pair(v.x, v.y), hi = bf16_pair(v.z, v.w);
                        if (left >= 4 && a.vec >= 8) *reinterpret_cast<uint2 *>(p) = make_uint2(lo, hi);
                        else {
                            p[0] = (uint16_t)lo;
                            if (left > 1) p[1] = (uint16_t)(lo >> 16);
                            if (left > 2) p[2] = (uint16_t)hi;
                            if (left > 3) p[3] = (uint16_t)(hi >> 16);
                        }
                    }
                }
            cluster_meet();  // nobody's part is read from here on
        }
        if constexpr (CTAS == 2) cluster_meet();
        if (warp == kMmaWarp) {
            tc_fence_after();
            if constexpr (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
            else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
        }
    };

    if (warp >= kSumWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == kCopyWarp) {
            // ===================== copies: one thread, as far ahead as free stages allow =====================
            if (lane == 0) {
                Turn turn{0, 1u};  // the phase before the first leaves every stage free
                int issued = 0;
                for (int item = first; item < n_items && !*abort_v; item += step) {
                    const Tile t = tile_of(a, item);
                    const int row = row_of(t), wrow = t.n * BN + (CTAS == 2 ? rank * S::kBRows : 0);
                    for (int kb = kb0; kb < kb1; ++kb, ++issued, turn.advance(kStages)) {
                        if (!mbar_wait(&empty_bar[turn.at], turn.phase, abort_v, a.wait_limit_ns)) {
                            raise_abort(item, 5);
                            break;
                        }
                        if (blockIdx.x == 0 && issued == a.test_skip_slot) continue;
                        const uint32_t dst = smem_u32(smem) + (uint32_t)(turn.at * S::kStageBytes), bar = CTAS == 2 ? in_first_cta(&full_bar[turn.at]) : smem_u32(&full_bar[turn.at]);
                        if (CTAS == 1 || rank == 0) mbar_expect_tx(&full_bar[turn.at], (uint32_t)(CTAS * (rows + S::kBRows) * kLine));
                        load_box<CTAS>(dst, &xmap, kb * kLine, row, bar);
                        load_box<CTAS>(dst + kTileM * kLine, &wmap, kb * kLine, wrow, bar);
                    }
                }
            }
            __syncwarp();
        } else if (warp == kMmaWarp) {
            // ===================== MMA issue: the pair's first CTA for both =====================
            if (CTAS == 1 || rank == 0) {
                const uint32_t leader = elect_one() ? 1u : 0u, idesc = instr_desc_e4m3(kTileM * CTAS, BN);
                const uint64_t desc0 = smem_desc(smem_u32(smem));
                const uint32_t hi = (uint32_t)(desc0 >> 32), lo0 = (uint32_t)desc0;
                Turn turn{0, 0u}, acc{0, 1u};
                bool ok = true;
                for (int item = first; item < n_items && ok; item += step)
                    for (int kb = kb0; kb < kb1; ++kb) {
                        ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[acc.at], acc.phase, abort_v, a.wait_limit_ns));
                        if (!ok) {
                            if (leader) raise_abort(item, 2);
                            break;
                        }
                        ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[turn.at], turn.phase, abort_v, a.wait_limit_ns));
                        if (!ok) {
                            if (leader) raise_abort(item, 3);
                            break;
                        }
                        tc_fence_after();
                        const uint32_t lo = lo0 + (uint32_t)(turn.at * (S::kStageBytes / 16));
                        tc_block_e4m3<CTAS>(leader, tmem_base + (uint32_t)(acc.at * BN), lo, lo + kTileM * kLine / 16, hi, idesc);
                        commit_to<CTAS>(leader, &empty_bar[turn.at]);  // the stage is free once these MMAs have read it
                        commit_to<CTAS>(leader, &acc_full[acc.at]);
                        turn.advance(kStages), acc.advance(S::kAccs);
                    }
                // every MMA has completed before shared and tensor memory are given up (not skipped while aborting)
                commit_to<CTAS>(leader, &drain_bar);
            }
            mbar_wait(&drain_bar, 0u, nullptr, a.wait_limit_ns);
            __syncwarp();
        }
        leave();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        // ===================== sums and stores =====================
        const int quad = warp & 3, half = warp >> 2;  // the TMEM lanes a warp may read: 32 (warp % 4) ..; its half of the columns
        const uint32_t lanes = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * kCols);
        const uint32_t empty_at = CTAS == 2 ? in_first_cta(&acc_empty[0]) : smem_u32(&acc_empty[0]);
        Turn acc{0, 0u};
        // A thread's scales, four blocks (a group) at a time, a group ahead of its use: next holds the factors of the group behind kb's.
        struct Four {
            float x[4], w[4];
        };
        auto group_of = [&](const Tile &t, int group) {
            const int row = row_of(t) + quad * 32 + lane, col = t.n * BN + half * kCols, kb = 4 * group;
            Four f{};
            if (row >= a.g.M || col >= a.g.N || kb >= kb1) return f;
            const float *const xs = a.g.xs + (int64_t)row * a.g.xs_ld + kb, *const ws = a.g.ws + (int64_t)(col / kF8Block) * a.g.kb + kb;
            if (a.xs4 && kb + 4 <= a.g.kb) {
                const float4 x = __ldg(reinterpret_cast<const float4 *>(xs));
                f.x[0] = x.x, f.x[1] = x.y, f.x[2] = x.z, f.x[3] = x.w;
            } else
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (kb + i < a.g.kb) f.x[i] = __ldg(xs + i);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (kb + i < a.g.kb) f.w[i] = __ldg(ws + i);
            return f;
        };
        float now[4] = {};
        Tile t = tile_of(a, first), then = t;
        Four next = group_of(t, kb0 / 4);
        for (int item = first; item < n_items; item += step, t = then) {
            const int row = row_of(t) + quad * 32 + lane, col = t.n * BN + half * kCols;
            const bool there = quad * 32 + lane < rows && row < a.g.M;
            uint64_t sum[kCols / 2];
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) sum[i] = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if ((kb & 3) == 0 || kb == kb0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) now[i] = next.x[i] * next.w[i];
                    if ((kb | 3) + 1 < kb1) next = group_of(t, kb / 4 + 1);
                    else if (item + step < n_items) then = tile_of(a, item + step), next = group_of(then, kb0 / 4);
                }
                const float s = kb & 2 ? (kb & 1 ? now[3] : now[2]) : (kb & 1 ? now[1] : now[0]);
                if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[acc.at], acc.phase, abort_v, a.wait_limit_ns))) {
                    if (lane == 0) raise_abort(item, 4);
                    break;
                }
                tc_fence_after();
                const uint64_t s2 = pair(s, s);
                constexpr int AT = kAtOnce;
                float v[2][AT];
                const uint32_t from = lanes + (uint32_t)(acc.at * BN);
                tc_ask(from, v[0]);
#pragma unroll
                for (int c = 0; c < kCols; c += AT) {
                    float(&u)[AT] = v[c / AT & 1];
                    tc_there(u);
                    if (c + AT < kCols) tc_ask(from + (uint32_t)(c + AT), v[c / AT + 1 & 1]);  // on its way under these columns' sums
                    else {  // the last columns are in registers: the accumulator may be overwritten
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive_at(empty_at + 8u * (uint32_t)acc.at);
                    }
#pragma unroll
                    for (int i = 0; i < AT / 2; ++i) sum[c / 2 + i] = fma_pair(pair(u[2 * i], u[2 * i + 1]), s2, sum[c / 2 + i]);
                }
                acc.advance(S::kAccs);
            }
            if (__any_sync(0xffffffffu, *abort_v)) break;  // as one: lanes that read it at different times would not meet again in the stores below
            if (CTAS == 1 && a.split > 1) {
                // this CTA's part to shared memory: the ring is not needed any more (its one item's MMAs have completed); sixteen bytes' place within eight of them by the row, so
                // that eight lanes' stores touch all banks
                const int r = quad * 32 + lane;
                float *const to = reinterpret_cast<float *>(smem) + r * BN;
#pragma unroll
                for (int i = 0; i < kCols / 2; i += 2) *reinterpret_cast<ulonglong2 *>(to + ((half * kCols + 2 * i) ^ (r & 7) * 4)) = make_ulonglong2(sum[i], sum[i + 1]);
            } else if (TENSOR || (CTAS == 1 && a.tensor_out)) {
                // rows of 64 columns, 128 bytes, their 16-byte pieces swizzled: eight lanes' stores touch all banks; a warp's 32 rows are a box of their own
                unsigned char *const out = smem + S::kRing + quad * 32 * 128;
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the last tile's have been read
                __syncwarp();
#pragma unroll
                for (int c = 0; c < kCols; c += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = bf16_pair(__uint_as_float((uint32_t)sum[c / 2 + i]), __uint_as_float((uint32_t)(sum[c / 2 + i] >> 32)));
                    const int at = half * kCols + c;
                    *reinterpret_cast<uint4 *>(out + (at / 64) * (kTileM * 128) + swz(lane, at % 64 / 8)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0 && there) {
#pragma unroll
                    for (int c = 0; c < kCols; c += 64)
                        if (col + c < a.g.N)
                            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(&ymap)), "r"(col + c), "r"(row),
                                         "r"(smem_u32(out + ((half * kCols + c) / 64) * (kTileM * 128)))
                                         : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            } else if (!TENSOR && a.g.f32 && a.vec >= 16) {
                if (there)
#pragma unroll
                    for (int c = 0; c < kCols; c += 32) {
                        float v[32];
#pragma unroll
                        for (int i = 0; i < 16; ++i) unpair(sum[c / 2 + i], v[2 * i], v[2 * i + 1]);
                        store_run(a, (int64_t)row * a.g.y_ld + col + c, a.g.N - col - c, v);
                    }
            } else if constexpr (!TENSOR) {
                // rows that sixteen bytes may not be stored to: 32 x 32 values change places in shared memory (the column's by the row, so that both ways touch all banks), and a row's
                // leave side by side (1049 x 2852 x 1168: 15.7 us, each thread along its own row 49.6; 4139 x 1827 x 448 23 and 89)
                float *const turned = reinterpret_cast<float *>(smem + S::kRing) + warp * 1024;
                const int n = min(32, min(rows - quad * 32, a.g.M - (row - lane)));
#pragma unroll
                for (int c = 0; c < kCols; c += 32) {
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 16; ++i) unpair(sum[c / 2 + i], turned[lane * 32 + (2 * i ^ lane)], turned[lane * 32 + (2 * i + 1 ^ lane)]);
                    __syncwarp();
                    if (!a.g.f32 && a.vec >= 4) {  // two columns a lane, two rows at once
                        const int k = 2 * (lane & 15), left = a.g.N - col - c - k;
                        uint16_t *const p = static_cast<uint16_t *>(a.g.y) + (int64_t)(row - lane) * a.g.y_ld + col + c + k;
                        if (left > 0)
#pragma unroll 8
                            for (int r = lane >> 4; r < n; r += 2) {
                                const uint32_t w = bf16_pair(turned[r * 32 + (k ^ r)], turned[r * 32 + (k + 1 ^ r)]);
                                if (left > 1) *reinterpret_cast<uint32_t *>(p + r * a.g.y_ld) = w;
                                else p[r * a.g.y_ld] = (uint16_t)w;
                            }
                    } else if (col + c + lane < a.g.N) {
                        const int64_t at = (int64_t)(row - lane) * a.g.y_ld + col + c + lane;
#pragma unroll 8
                        for (int r = 0; r < n; ++r) {
                            const float v = turned[r * 32 + (lane ^ r)];
                            if (a.g.f32) static_cast<float *>(a.g.y)[at + r * a.g.y_ld] = v;
                            else static_cast<uint16_t *>(a.g.y)[at + r * a.g.y_ld] = f32_to_bf16_bits(v);
                        }
                    }
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // what was stored from shared memory has been written
        leave();
    }
}

// CTAs that share a tile's k: a power of two that leaves every tile's their places on the machine at once (48 clusters of three did not find them: 6144 weight rows, one row of x
// 14.7 us, in pairs 9.8), two blocks each at least, and no more than pay for the parts' way through the cluster, which costs as much as `parts` blocks.
int shares(int64_t tiles, int64_t kb, int64_t parts) {
    int best = 1;
    for (int s = 2; s <= 8 && tiles * s <= (s == 8 ? 64 : sm_count()) && kb >= s * 2; s *= 2)
        if ((kb + s - 1) / s + parts < (kb + best - 1) / best + (best > 1 ? parts : 0)) best = s;
    return best;
}

template <int CTAS, int BN>
int launch_tc8(const char *fn, TcArgs8 a, cudaStream_t st) {
    using S = Shape<CTAS, BN>;
    a.n_m = (a.g.M + kTileM * CTAS - 1) / (kTileM * CTAS);
    // BF16 rows leave through shared memory, under the next tile's MMAs; a CTA's only tile too (777 x 1000 x 512: 5.4 us, from the registers 6.4)
    a.tensor_out = !a.g.f32 && a.vec >= 16 && (CTAS == 2 || a.split == 1);
    // Tiles of a CTA share the rows alike: what the fullest one has to fetch, and in a cluster to add up, bounds the call (150 x 2560 x 4096: 11.7 us, with 128 and 22 rows 13.8; 300 x
    // 4096 x 4096 14.8 for 17.4).  Tensor copies take 32 rows.
    const int even = (a.g.M + a.n_m - 1) / a.n_m, by = a.tensor_out ? 32 : 8;
    a.rows = CTAS == 2 ? kTileM : (even + by - 1) / by * by;
    CUtensorMap xmap, wmap, ymap;
    if (int rc = tensor_map_2d(fn, a.g.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)a.g.K, (uint64_t)a.g.M, (uint64_t)a.g.x_ld, kLine, (uint32_t)a.rows, CU_TENSOR_MAP_SWIZZLE_128B, &xmap))
        return rc;
    if (int rc = tensor_map_2d(fn, a.g.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)a.g.K, (uint64_t)a.g.N, (uint64_t)a.g.K, kLine, S::kBRows, CU_TENSOR_MAP_SWIZZLE_128B, &wmap))
        return rc;
    a.n_n = (a.g.N + BN - 1) / BN;
    a.band = std::min(a.n_m, 16);
    const int64_t items = (int64_t)a.n_m * a.n_n;
    const int cluster = CTAS == 2 ? 2 : a.split;
    const int64_t places = CTAS == 2 ? sm_count() / 2 : a.split > 1 ? items : (int64_t)sm_count();
    if (!a.tensor_out) ymap = xmap;  // not used
    else if (int rc = tensor_map_2d(fn, a.g.y, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)a.g.N, (uint64_t)a.g.M, (uint64_t)a.g.y_ld * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B, &ymap))
        return rc;
    auto *kern = f8_tc_kernel<CTAS, BN, false>;
    if constexpr (CTAS == 2)
        if (a.tensor_out) kern = f8_tc_kernel<CTAS, BN, true>;
    SXB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem), fn, ": reserving shared memory");
    const cudaError_t e = launch_behind(kern, dim3((unsigned)(std::min(items, places) * cluster)), dim3(kThreads), S::kSmem, st, cluster, a, xmap, wmap, ymap);
    SXB_CUDA(e, fn, ": launching M=", a.g.M, " N=", a.g.N, " K=", a.g.K);
    return SXB_OK;
}

// ---- a few rows of x: the weights on the MMAs' M side ------------------------------------------------------------------------------
//
// What bounds it is the weights' bytes, 16 KB a block of k and tile of 128 weight rows; the rows of x, 16 or 32, are the MMA's columns.  The accumulators of all stages fit tensor
// memory, so one commit a stage, of two blocks, says that its codes have been read and that its sums are there.  A lane of tensor memory is a weight row: a thread has all columns of
// one, the weight's scale is one number for the warp, and those of x go round by shuffles.  16 x 131072 x 4096: 89 us, 6.1 TB/s (128 rows' worth of MMAs, the form above: 188); 32 rows 94.
// With 64 columns a warp's shuffles and sums do not keep up (134 us, the form above 102).

template <int NB>
struct FewShape {
    static constexpr int kBlocks = 2;                                             // of k, of a stage
    static constexpr int kBlockBytes = (kTileM + NB) * kLine, kStageBytes = kBlocks * kBlockBytes;
    static constexpr int kStages = NB == 32 ? 5 : 6;
    static constexpr int kCols = kStages * kBlocks * NB, kTmem = kCols > 256 ? 512 : 256;
    static constexpr size_t kSmem = (size_t)kStages * kStageBytes + 1024;
    static_assert(kCols <= 512 && kSmem <= 226 * 1024 && NB * kTileM * 4 <= kStages * kStageBytes);
};
constexpr int kFewSumWarps = 4, kFewThreads = 32 * (kFewSumWarps + 2);

template <int NB>
__global__ void __launch_bounds__(kFewThreads, 1)
    f8_few_kernel(const TcArgs8 a, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap) {
    using S = FewShape<NB>;
    constexpr int PER = S::kBlocks;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *const smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full_bar[S::kStages], done_bar[S::kStages], drained_bar[S::kStages], drain_bar;
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int group = a.split, rank = (int)blockIdx.x % group;
    const int n_items = a.n_n, first = (int)blockIdx.x / group, step = (int)gridDim.x / group;
    const int kb0 = (int)((int64_t)a.g.kb * rank / group), kb1 = (int)((int64_t)a.g.kb * (rank + 1) / group);
    volatile int *const abort_v = &abort_flag;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) mbar_init(&full_bar[s], 1), mbar_init(&done_bar[s], 1), mbar_init(&drained_bar[s], kFewSumWarps);
        mbar_init(&drain_bar, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fetch_map(&xmap), fetch_map(&wmap);
    }
    if (warp == kFewSumWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_smem)), "r"(S::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    behind_grid();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_smem;

    auto raise_abort = [&](int item, int role) {
        if (atomicExch(&abort_flag, 1) == 0 && atomicCAS(&a.status[0], 0u, 2u) == 0u) {
            a.status[1] = (uint32_t)item;
            a.status[2] = (uint32_t)role;
        }
    };

    if (warp == kFewSumWarps) {
        // ===================== copies =====================
        if (lane == 0) {
            Turn turn{0, 1u};
            int issued = 0;
            for (int item = first; item < n_items && !*abort_v; item += step)
                for (int kb = kb0; kb < kb1; kb += PER, ++issued, turn.advance(S::kStages)) {
                    if (!mbar_wait(&done_bar[turn.at], turn.phase, abort_v, a.wait_limit_ns)) {
                        raise_abort(item, 5);
                        break;
                    }
                    if (blockIdx.x == 0 && issued == a.test_skip_slot) continue;
                    const int n = min(PER, kb1 - kb);
                    mbar_expect_tx(&full_bar[turn.at], (uint32_t)(n * S::kBlockBytes));
                    for (int i = 0; i < n; ++i) {
                        const uint32_t dst = smem_u32(smem) + (uint32_t)(turn.at * S::kStageBytes + i * S::kBlockBytes);
                        tma_load_2d(dst, &wmap, (kb + i) * kLine, item * kTileM, &full_bar[turn.at]);
                        tma_load_2d(dst + kTileM * kLine, &xmap, (kb + i) * kLine, 0, &full_bar[turn.at]);
                    }
                }
        }
        __syncwarp();
    } else if (warp == kFewSumWarps + 1) {
        // ===================== MMA issue =====================
        const uint32_t leader = elect_one() ? 1u : 0u, idesc = instr_desc_e4m3(kTileM, NB);
        const uint64_t desc0 = smem_desc(smem_u32(smem));
        const uint32_t hi = (uint32_t)(desc0 >> 32), lo0 = (uint32_t)desc0;
        Turn turn{0, 0u};
        bool ok = true;
        for (int item = first; item < n_items && ok; item += step)
            for (int kb = kb0; kb < kb1; kb += PER, turn.advance(S::kStages)) {
                ok = __all_sync(0xffffffffu, mbar_wait(&drained_bar[turn.at], turn.phase ^ 1u, abort_v, a.wait_limit_ns));
                if (!ok) {
                    if (leader) raise_abort(item, 2);
                    break;
                }
                ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[turn.at], turn.phase, abort_v, a.wait_limit_ns));
                if (!ok) {
                    if (leader) raise_abort(item, 3);
                    break;
                }
                tc_fence_after();
                for (int i = 0; i < min(PER, kb1 - kb); ++i) {
                    const uint32_t lo = lo0 + (uint32_t)(turn.at * S::kStageBytes + i * S::kBlockBytes) / 16;
                    tc_block_e4m3<1>(leader, tmem_base + (uint32_t)((turn.at * PER + i) * NB), lo, lo + kTileM * kLine / 16, hi, idesc);
                }
                commit_to<1>(leader, &done_bar[turn.at]);
            }
        // every MMA has completed before shared and tensor memory are given up (not skipped while aborting)
        commit_to<1>(leader, &drain_bar);
        mbar_wait(&drain_bar, 0u, nullptr, a.wait_limit_ns);
        __syncwarp();
    } else {
        // ===================== sums and stores =====================
        const uint32_t lanes = tmem_base + ((uint32_t)(warp * 32) << 16);
        Turn turn{0, 0u};
        // of a stage's blocks: that of the lane's row of x, and the weight's (a tile lies in one block of weight rows); asked for a stage ahead of their use
        struct Scales {
            float x[PER], w[PER];
        };
        auto scales = [&](int item, int kb) {
            Scales s;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                s.w[i] = kb + i < kb1 ? __ldg(a.g.ws + (int64_t)item * a.g.kb + kb + i) : 0.f;
                s.x[i] = lane < a.g.M && kb + i < kb1 ? __ldg(a.g.xs + lane * a.g.xs_ld + kb + i) : 0.f;
            }
            return s;
        };
        Scales next = scales(first, kb0);
        for (int item = first; item < n_items; item += step) {
            float sum[NB];
#pragma unroll
            for (int i = 0; i < NB; ++i) sum[i] = 0.f;
            for (int kb = kb0; kb < kb1; kb += PER, turn.advance(S::kStages)) {
                float now[PER];
#pragma unroll
                for (int i = 0; i < PER; ++i) now[i] = next.x[i] * next.w[i];
                if (!__all_sync(0xffffffffu, mbar_wait(&done_bar[turn.at], turn.phase, abort_v, a.wait_limit_ns))) {
                    if (lane == 0) raise_abort(item, 4);
                    break;
                }
                if (kb + PER < kb1) next = scales(item, kb + PER);
                else if (item + step < n_items) next = scales(item + step, kb0);
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    if (kb + i >= kb1) break;
                    float v[NB];
                    tc_ask(lanes + (uint32_t)((turn.at * PER + i) * NB), v);
                    tc_there(v);
                    if (i + 1 == PER || kb + i + 1 == kb1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&drained_bar[turn.at]);
                    }
#pragma unroll
                    for (int k = 0; k < NB; ++k) sum[k] = fmaf(v[k], __shfl_sync(0xffffffffu, now[i], k), sum[k]);
                }
            }
            if (__any_sync(0xffffffffu, *abort_v)) break;  // as one, see above
            const int row = warp * 32 + lane, n = item * kTileM + row;
            if (a.split > 1) {
#pragma unroll
                for (int m = 0; m < NB; ++m) reinterpret_cast<float *>(smem)[m * kTileM + row] = sum[m];  // the ring is not needed any more: all its MMAs have completed
            } else if (n < a.g.N) {
#pragma unroll
                for (int m = 0; m < NB; ++m)
                    if (m < a.g.M) {
                        if (a.g.f32) static_cast<float *>(a.g.y)[m * a.g.y_ld + n] = sum[m];
                        else static_cast<uint16_t *>(a.g.y)[m * a.g.y_ld + n] = f32_to_bf16_bits(sum[m]);
                    }
            }
        }
    }

    if (*abort_v) {  // copies that a CTA issued before it gave up have landed within this time
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    tc_fence_before();
    __syncthreads();
    if (a.split > 1) {
        cluster_meet();  // every part is there
        if (!*abort_v)
            for (int i = rank * kFewThreads + (int)threadIdx.x; i < min(NB, a.g.M) * kTileM; i += group * kFewThreads) {
                const int m = i / kTileM, n = first * kTileM + i % kTileM;
                if (n >= a.g.N) continue;
                float v = 0.f;
                for (int k = 0; k < group; ++k) {
                    float p;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p) : "r"(in_cta(smem, k) + 4u * (uint32_t)i) : "memory");
                    v += p;
                }
                if (a.g.f32) static_cast<float *>(a.g.y)[m * a.g.y_ld + n] = v;
                else static_cast<uint16_t *>(a.g.y)[m * a.g.y_ld + n] = f32_to_bf16_bits(v);
            }
        cluster_meet();  // nobody's part is read from here on
    }
    if (warp == kFewSumWarps + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(S::kTmem) : "memory");
    }
}

template <int NB>
int launch_few(const char *fn, TcArgs8 a, cudaStream_t st) {
    using S = FewShape<NB>;
    CUtensorMap xmap, wmap;
    if (int rc = tensor_map_2d(fn, a.g.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)a.g.K, (uint64_t)a.g.M, (uint64_t)a.g.x_ld, kLine, NB, CU_TENSOR_MAP_SWIZZLE_128B, &xmap)) return rc;
    if (int rc = tensor_map_2d(fn, a.g.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)a.g.K, (uint64_t)a.g.N, (uint64_t)a.g.K, kLine, kTileM, CU_TENSOR_MAP_SWIZZLE_128B, &wmap)) return rc;
    const int64_t sms = sm_count();
    a.n_n = (a.g.N + kTileM - 1) / kTileM;
    a.split = shares(a.n_n, a.g.kb, 5);
    SXB_CUDA(cudaFuncSetAttribute(f8_few_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem), fn, ": reserving shared memory");
    const int64_t places = a.split > 1 ? a.n_n : std::min<int64_t>(a.n_n, sms);
    const cudaError_t e = launch_behind(f8_few_kernel<NB>, dim3((unsigned)(places * a.split)), dim3(kFewThreads), S::kSmem, st, a.split, a, xmap, wmap);
    SXB_CUDA(e, fn, ": launching M=", a.g.M, " N=", a.g.N, " K=", a.g.K);
    return SXB_OK;
}

}  // namespace

int linear_f8_tc(const char *fn, const F8Args &g, cudaStream_t st) {
    TcArgs8 a{};
    a.g = g;
    const int64_t es = g.f32 ? 4 : 2;
    for (a.vec = 32; a.vec > 2 && (reinterpret_cast<uintptr_t>(g.y) % a.vec != 0 || g.y_ld * es % a.vec != 0); a.vec /= 2) {}
    a.xs4 = reinterpret_cast<uintptr_t>(g.xs) % 16 == 0 && g.xs_ld % 4 == 0;
    a.wait_limit_ns = wait_limit_ns(), a.test_skip_slot = test_skip_slot();
    if (int rc = library_status_words(fn, &a.status)) return rc;
    if (g.M <= 16) return launch_few<16>(fn, a, st);
    if (g.M <= 32) return launch_few<32>(fn, a, st);
    const int64_t sms = sm_count(), pairs = (int64_t)((g.M + 255) / 256) * ((g.N + 255) / 256), tiles = (int64_t)((g.M + 127) / 128) * ((g.N + 127) / 128);
    // Pairs from as many tiles on as there are places for them, whatever K is: 2304 x 2304 x 4096 (81 tiles, two rounds) 33 us, tiles of one CTA 35; 2304 x 4096 x 4096 35 and 46; 3000 x 4096 x 4096
    // 48 and 65; 600 x 8192 x 4096 33 and 34; 2048 x 4096 x 256 8.6 and 9.5; 4096 x 4096 x 512 17.7 and 17.9, but 2304 x 2304 x 448 10.5 and 9.7.  Below, few tiles share their k and pairs cannot;
    // the largest of those would gain (2048 x 2304 x 4096, 72 tiles: 20 and 26 us).
    if (g.M > 128 && pairs * 2 >= sms) return launch_tc8<2, 256>(fn, a, st);
    a.split = shares(tiles, g.kb, 11);
    return launch_tc8<1, 128>(fn, a, st);
}

}  // namespace sxb
