// Attention of a few new tokens a sequence over a paged key-value cache (sxb_attn_decode).
//
//   s_j = scale * q . k_j,   o = sum_j exp(s_j - M) v_j / sum_j exp(s_j - M),   M = max_j s_j,   lse = M + log(sum_j exp(s_j - M))
//
// One pass over the keys with a running maximum and sum.  The work is one list of units - a unit is a tile of TK keys of one (sequence, key head, tile
// of R query rows) - and every CTA takes an equal run of it, across the ends of heads and sequences: a batch of uneven lengths, or one long sequence
// alone, keeps all SMs equally busy, whatever the host knows of the lengths, and a captured graph follows them.  A segment (all units of one row tile)
// that lies in one CTA is written by it; the parts of one that several CTAs share go to the workspace, FP32 with their maxima and sums, at most two a
// CTA, and the last CTA to arrive joins them in the list's order, so that no result depends on who came last.
//
// The query heads of a key head and the new tokens of a sequence are the rows of one MMA tile: the cache is read once for all of them.  Products on
// mma.sync, whose operands come from shared memory, tiles there by cp.async from wherever the pages lie.
//   BF16 cache: exact products; weights rounded to BF16 (one rounding of 2^-9 a key, against the sum's many keys).
//   8 and 4 bits: the codes are F16 numbers exactly, q is F16 times a power of two a row (a BF16 number less than 2^28 below the row's largest is exact),
//   scale and min go on in FP32: s = scale_k * (q . code) + min_k * sum(q) a group.  For V a key's weight takes its group's scale, times a power of
//   two that follows the largest scale seen so that F16's range is no limit (one rounding of 2^-11); the mins' share, sum p * min, is FP32.

#include "attn.cuh"
#include "skinny_mma.cuh"

#include <math_constants.h>

namespace sxb {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMinRun = 2;     // units a CTA takes at least
constexpr int kMaxIds = 16;    // pages that a tile of 128 keys touches at most
constexpr int64_t kMaxRows = 1ll << 24;

template <int D_, int BITS_, int G_, int WR_> struct Shape {
    static constexpr int D = D_, BITS = BITS_, G = G_, WR = WR_;
    static constexpr int kWarps = WR == 1 ? 4 : 8, kThreads = 32 * kWarps, WK = kWarps / WR, R = 16 * WR;
    static constexpr int RB = D * BITS / 8, CR = RB / 16;  // bytes and 16-byte chunks of a cache row
    static constexpr int NG = BITS == 16 ? 0 : D / G;
    static constexpr int TK = D == 64 || (BITS == 4 && D == 128) ? 128 : 64;
    static constexpr int KI = TK / (16 * WK);  // runs of sixteen keys of a warp's share of a tile
    static constexpr int kRows = TK * RB, kScales = TK * NG * 4, kStage = 2 * (kRows + kScales);
    static constexpr int kQ = R * D * 2;
    static constexpr int kMostJoint = WK * R * 32 * 4;
    static constexpr bool kOwnJoint = kStage < kMostJoint;  // 32 columns of every warp's rows do not fit a stage
    static constexpr int kMisc = 1024 + WK * R * 8 + R * (NG + 1) * 4 + (kOwnJoint ? kMostJoint : 0);
    static constexpr int kPerSm = WR == 1 && D <= 128 ? 2 : 1;
    static constexpr int kBudget = 226 * 1024 / kPerSm;
    static constexpr int kFit = (kBudget - kMisc) / (kStage + kQ), kStages = kFit > 5 ? 5 : kFit;
    static constexpr int kSmem = kStages * (kStage + kQ) + kMisc;
    static constexpr int fit_columns() {
        int dc = D;
        while (dc > 32 && WK * R * dc * 4 > kStage) dc /= 2;
        return dc;
    }
    static constexpr int DC = fit_columns();  // columns that the warps join at a time
    static_assert(kStages >= 2 && KI >= 1 && kThreads % CR == 0, "");
};

struct Args {
    const uint16_t *q;
    int64_t q_ld;
    const int32_t *pages, *q_start, *kv_len;
    int64_t pages_ld, capacity;
    int B, T, n_q, group, window;
    float scale, softcap;
    KvView c;
    uint16_t *out;
    int64_t out_ld;
    float *lse, *partial;
    uint32_t *count, *err;
};

// What a sequence asks for.
struct Sequence {
    int q0, n, len, p0, lo, tile0, tiles, row_tiles;
    bool bad;
};
template <class S> __device__ inline Sequence sequence(const Args &a, int b) {
    Sequence s;
    s.q0 = a.q_start[b];
    const int q1 = a.q_start[b + 1];
    s.len = a.kv_len[b];
    const bool skip = s.q0 < 0 || q1 < s.q0 || q1 > a.T;
    s.n = skip ? 0 : q1 - s.q0;
    s.bad = s.len < 0 || s.len > a.capacity;
    if (s.bad) s.len = 0;
    s.p0 = s.len - s.n;
    s.lo = a.window > 0 ? max(0, s.p0 - a.window + 1) : 0;
    s.tile0 = s.lo / S::TK;
    s.tiles = max(1, (s.len + S::TK - 1) / S::TK - s.tile0);
    s.row_tiles = (int)(((int64_t)s.n * a.group + S::R - 1) / S::R);
    if (skip) s.bad = true;
    return s;
}

// A segment of the list that this CTA has units of.
struct Segment {
    int q0, n, len, p0, tile0, tiles, head, rows0, at, bad;  // rows0: first row of the tile, at: the CTA's first unit's place in the segment
};

__device__ inline uint32_t smem_of(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES> __device__ inline void copy_async(uint32_t to, const void *from, int n) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
    else if constexpr (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}
__device__ inline void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ inline void wait_async() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ inline void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ inline void load_matrices_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ inline void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ inline float exp2_fast(float v) {  // 2 ulp; exp2(-inf) = 0
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ inline uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ inline uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 1024 + code in both halves, less 1024: exact.
__device__ inline uint32_t less_1024(uint32_t v) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&v), __half2half2(__ushort_as_half(0x6400)));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// Codes two bytes (named by the selector's nibbles 0 and 2) or two nibbles (at bits 0 and 16) of a word as F16.
__device__ inline uint32_t bytes_f16(uint32_t w, uint32_t selector) { return less_1024(__byte_perm(w, 0x64646464u, selector)); }
__device__ inline uint32_t nibbles_f16(uint32_t w) { return less_1024((w & 0x000f000fu) | 0x64006400u); }

// Where chunk c of row r stands in a tile of rows of CR chunks: eight neighbouring rows' chunks of one number lie in eight different sixteenths of the
// banks' 128 bytes.
template <int CR> __device__ inline int chunk_at(int r, int c) {
    if constexpr (CR >= 8) return r * CR + (c ^ (r & 7));
    else return r * CR + (c ^ ((r / (8 / CR)) & (CR - 1)));
}
// The K rows of 8-bit codes are read eight bytes a lane, four rows a pass: pairs of chunks.
template <class S> __device__ inline int k_chunk_at(int r, int c) {
    if constexpr (S::BITS == 8 && S::CR >= 8) return r * S::CR + (c ^ (2 * (r & 3)));
    else if constexpr (S::BITS == 8) return r * S::CR + (c ^ (2 * ((r >> 1) & 1)));
    else return chunk_at<S::CR>(r, c);
}

template <class S>
__global__ void __launch_bounds__(S::kThreads, S::kPerSm) attn_decode_kernel(const __grid_constant__ Args a) {
    constexpr int D = S::D, BITS = S::BITS, NG = S::NG, TK = S::TK, KI = S::KI, R = S::R, WK = S::WK, CR = S::CR, kStages = S::kStages;
    constexpr bool kQuant = BITS != 16;
    constexpr int kThreads = S::kThreads, kWarps = S::kWarps;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *const q_ring = smem + kStages * S::kStage;
    uint8_t *const own_joint = q_ring + kStages * S::kQ, *const misc = own_joint + (S::kOwnJoint ? S::kMostJoint : 0);
    auto *const row_max = reinterpret_cast<float *>(misc);  // [WK][R]
    float *const row_sum = row_max + WK * R;                // [WK][R]
    float *const q_factor = row_sum + WK * R;               // [R]
    float *const q_sums = q_factor + R;                     // [R][NG]
    auto *const segments = reinterpret_cast<Segment *>(q_sums + R * NG);  // [kStages]
    auto *const ids = reinterpret_cast<int *>(segments + kStages);        // [2][kMaxIds]
    auto *const scan = reinterpret_cast<int64_t *>((reinterpret_cast<uintptr_t>(ids + 2 * kMaxIds) + 7) & ~(uintptr_t)7);  // [kWarps + 4]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int wr = warp % S::WR, wk = warp / S::WR;

    behind_grid();

    // ---- this CTA's run of the list ----
    int64_t total = 0;
    for (int b = tid; b < a.B; b += kThreads) {
        const Sequence s = sequence<S>(a, b);
        if (s.bad && blockIdx.x == 0) raise_error(a.err, (uint32_t)b, (uint32_t)a.kv_len[b]);
        total += (int64_t)s.tiles * s.row_tiles * a.c.n_kv;
    }
    const int64_t mine = total;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (lane == 0) scan[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += scan[w];
    const int64_t ctas = min((int64_t)gridDim.x, (total + kMinRun - 1) / kMinRun);
    if ((int64_t)blockIdx.x >= ctas) return;
    const int64_t u0 = blockIdx.x * total / ctas, u1 = (blockIdx.x + 1) * total / ctas;
    for (int64_t base = 0, before = 0; base < a.B; base += kThreads) {
        int64_t own = mine;
        if (a.B > kThreads) {
            own = 0;
            if (base + tid < a.B) {
                const Sequence s = sequence<S>(a, (int)base + tid);
                own = (int64_t)s.tiles * s.row_tiles * a.c.n_kv;
            }
        }
        int64_t upto = own;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += v;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = upto;
        __syncthreads();
        int64_t ahead = before, all = before;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) ahead += scan[w];
            all += scan[w];
        }
        upto += ahead;
        if (upto - own <= u0 && u0 < upto) scan[kWarps] = base + tid, scan[kWarps + 1] = u0 - (upto - own);
        before = all;
        if (before > u0) break;
    }
    __syncthreads();

    // ---- the cursor of the loads: kStages - 1 units ahead of the sums ----
    int l_b = (int)scan[kWarps], l_head, l_row_tile, l_at, l_segment = 0;
    Sequence l_s = sequence<S>(a, l_b);
    bool l_new = true;
    {
        const int64_t in = scan[kWarps + 1];
        const int64_t per_head = (int64_t)l_s.tiles * l_s.row_tiles;
        l_head = (int)(in / per_head);
        const int64_t rest = in - l_head * per_head;
        l_row_tile = (int)(rest / l_s.tiles), l_at = (int)(rest % l_s.tiles);
    }
    const int units = (int)(u1 - u0);
    const int page_mask = (1 << a.c.page_shift) - 1;

    // page id number tid of the tile under the cursor
    auto find_id = [&]() -> int {
        const int first = (l_s.tile0 + l_at) * TK, col = (first >> a.c.page_shift) + tid;
        const int end = min(l_s.len, first + TK);
        if (((int64_t)col << a.c.page_shift) >= end || (((int64_t)col + 1) << a.c.page_shift) <= l_s.lo) return kBadPage;
        const int id = a.pages[l_b * a.pages_ld + col];
        if ((unsigned)id < (unsigned)a.c.n_pages) return id;
        raise_error(a.err, (uint32_t)l_b, (uint32_t)id);
        return kBadPage;
    };
    auto advance = [&]() {
        l_new = false;
        if (++l_at < l_s.tiles) return;
        l_at = 0, l_new = true, ++l_segment;
        if (++l_row_tile < l_s.row_tiles) return;
        l_row_tile = 0;
        if (++l_head < a.c.n_kv) return;
        l_head = 0;
        do {
            if (++l_b >= a.B) return;
            l_s = sequence<S>(a, l_b);
        } while (l_s.n == 0);
    };
    auto load = [&](int stage, const int *id_of) {
        uint8_t *const st = smem + stage * S::kStage;
        const int first = (l_s.tile0 + l_at) * TK, col0 = first >> a.c.page_shift;
        {
            const int c = tid % CR;
            const int64_t head_rows = l_head * a.c.head_stride;
#pragma unroll 4
            for (int r = tid / CR; r < TK; r += kThreads / CR) {
                const int j = first + r, id = id_of[(j >> a.c.page_shift) - col0];
                const bool wanted = j >= l_s.lo && j < l_s.len, there = wanted && id >= 0;
                const int64_t off = there ? (id * a.c.page_stride + head_rows + (j & page_mask) * a.c.row_stride) * S::RB + c * 16 : 0;
                uint8_t *const to = st + k_chunk_at<S>(r, c) * 16;
                if (!kQuant && wanted && !there) *reinterpret_cast<uint4 *>(to) = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
                else copy_async<16>(smem_of(to), a.c.k + off, there ? 16 : 0);
                copy_async<16>(smem_of(st + S::kRows + chunk_at<CR>(r, c) * 16), a.c.v + off, there ? 16 : 0);
            }
        }
        if constexpr (kQuant) {
            constexpr int kBytes = NG * 4 > 16 ? 16 : NG * 4, kPieces = NG * 4 / kBytes;
            uint8_t *const sc = st + 2 * S::kRows;
            for (int i = tid; i < TK * kPieces; i += kThreads) {
                const int r = i / kPieces, j = first + r, id = id_of[(j >> a.c.page_shift) - col0];
                const bool wanted = j >= l_s.lo && j < l_s.len, there = wanted && id >= 0;
                const int64_t off = there ? (id * a.c.page_stride + l_head * a.c.head_stride + (j & page_mask) * a.c.row_stride) * (NG * 4) + (i % kPieces) * kBytes : 0;
                uint8_t *const to = sc + i * kBytes;
                if (wanted && !there) {
#pragma unroll
                    for (int w = 0; w < kBytes / 4; ++w) reinterpret_cast<uint32_t *>(to)[w] = 0x7fc07fc0u;
                } else {
                    copy_async<kBytes>(smem_of(to), reinterpret_cast<const uint8_t *>(a.c.k_sm) + off, there ? kBytes : 0);
                }
                copy_async<kBytes>(smem_of(to + S::kScales), reinterpret_cast<const uint8_t *>(a.c.v_sm) + off, there ? kBytes : 0);
            }
        }
        if (l_new) {
            const int slot = l_segment % kStages, rows0 = l_row_tile * R;
            uint8_t *const qs = q_ring + slot * S::kQ;
            for (int i = tid; i < R * (D / 8); i += kThreads) {
                const int r = i / (D / 8), c = i % (D / 8), row = rows0 + r, tok = row / a.group;
                const bool there = tok < l_s.n;
                const int64_t off = there ? (l_s.q0 + tok) * a.q_ld + (int64_t)(l_head * a.group + row - tok * a.group) * D + c * 8 : 0;
                copy_async<16>(smem_of(qs + chunk_at<D / 8>(r, c) * 16), a.q + off, there ? 16 : 0);
            }
            if (tid == 0)
                segments[slot] = Segment{l_s.q0, l_s.n, l_s.len, l_s.p0, l_s.tile0, l_s.tiles, l_head, rows0, l_at, (int)l_s.bad};
        }
    };

    if (tid < kMaxIds) ids[tid] = find_id();
    __syncthreads();
    for (int s = 0; s < kStages - 1; ++s) {
        if (s < units) {
            load(s, ids + (s & 1) * kMaxIds);
            if (s + 1 < units) {
                advance();
                if (tid < kMaxIds) ids[((s + 1) & 1) * kMaxIds + tid] = find_id();
            }
            __syncthreads();
        }
        commit_async();
    }

    // ---- sums ----
    const int g = lane >> 2, t4 = lane & 3;
    constexpr int kQRegs = D <= 128 ? D / 16 : 1;
    uint32_t qf[kQRegs][4];
    float o[D / 8][4];
    float o_min[2][kQuant ? NG : 1];
    float m[2], l[2], fac[2];
    int hi[2], lo[2], v_exp = 20;
    Segment sg{};
    int at = 0, segment = 0;
    bool fresh = true;

    for (int i = 0; i < units; ++i) {
        wait_async<kStages - 2>();
        __syncthreads();
        int next_id = kBadPage;
        const int ahead = i + kStages - 1;
        if (ahead < units) {
            load(ahead % kStages, ids + (ahead & 1) * kMaxIds);
            if (ahead + 1 < units) {
                advance();
                if (tid < kMaxIds) next_id = find_id();
            }
        }
        commit_async();

        uint8_t *const st = smem + (i % kStages) * S::kStage;
        uint8_t *const qs = q_ring + (segment % kStages) * S::kQ;
        if (fresh) {
            fresh = false;
            sg = segments[segment % kStages];
            at = sg.at;
            m[0] = m[1] = -CUDART_INF_F, l[0] = l[1] = 0.f, v_exp = 20;
#pragma unroll
            for (int d = 0; d < D / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
#pragma unroll
            for (int e = 0; e < (kQuant ? NG : 1); ++e) o_min[0][e] = o_min[1][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int tok = (sg.rows0 + wr * 16 + g + 8 * e) / a.group;
                hi[e] = tok < sg.n ? sg.p0 + tok : -1;
                lo[e] = a.window > 0 ? max(-1, hi[e] - a.window) : -1;
            }
            if constexpr (kQuant) {
                // q to F16 times a power of two, elements in the order that the codes come in, and each group's sum of what they then are
                constexpr int kPer = kThreads / R, kBlocks = D / 32;  // threads of a row; runs of 32 elements
                constexpr int kOwn = (kBlocks + kPer - 1) / kPer;
                const int r = tid / kPer, part = tid % kPer;
                float x[kOwn][32], most = 0.f;
#pragma unroll
                for (int b = 0; b < kOwn; ++b) {
                    const int blk = part + b * kPer;
                    if (blk < kBlocks) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint4 w = *reinterpret_cast<const uint4 *>(qs + chunk_at<D / 8>(r, blk * 4 + c) * 16);
                            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[b][c * 8 + 2 * e] = __uint_as_float(ws[e] << 16), x[b][c * 8 + 2 * e + 1] = __uint_as_float(ws[e] & 0xffff0000u);
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e) most = fmaxf(most, fabsf(x[b][e]));
                    }
                }
#pragma unroll
                for (int off = 1; off < kPer; off <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
                const int up = min(126, 14 - ((int)(__float_as_uint(most) >> 23) - 127));
                const float f = __uint_as_float((uint32_t)(up + 127) << 23);
                if (part == 0) q_factor[r] = __uint_as_float((uint32_t)(127 - up) << 23);
                float sums[kOwn];
#pragma unroll
                for (int b = 0; b < kOwn; ++b) {
                    const int blk = part + b * kPer;
                    sums[b] = 0.f;
                    if (blk < kBlocks) {
                        uint32_t w[16];  // position 16 step + 8 half + 2 lane + e of the run, as pairs
#pragma unroll
                        for (int pos = 0; pos < 32; pos += 2) {
                            const int step = pos / 16, half = pos / 8 % 2, ln = pos / 2 % 4;
                            const int d0 = BITS == 8 ? 8 * ln + 4 * step + 2 * half : 8 * ln + 2 * step + half, d1 = BITS == 8 ? d0 + 1 : d0 + 4;
                            w[pos / 2] = pack_f16(x[b][d0] * f, x[b][d1] * f);
                            const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&w[pos / 2]));
                            sums[b] += back.x + back.y;
                        }
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            *reinterpret_cast<uint4 *>(qs + chunk_at<D / 8>(r, blk * 4 + c) * 16) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
                    }
                    // groups of two or four runs: neighbouring threads, the same b (a row's threads are as many as its runs, or fewer by a power of two)
                    constexpr int kRuns = S::G / 32;
                    static_assert(kRuns <= kPer, "");
#pragma unroll
                    for (int off = 1; off < kRuns; off <<= 1) sums[b] += __shfl_xor_sync(0xffffffffu, sums[b], off);
                    if (blk < kBlocks && blk % kRuns == 0) q_sums[r * NG + blk / kRuns] = sums[b];
                }
                __syncthreads();
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) fac[e] = a.scale * (kQuant ? q_factor[wr * 16 + g + 8 * e] : 1.f);
            if constexpr (D <= 128) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    load_matrices(qf[ks], smem_of(qs + chunk_at<D / 8>(wr * 16 + (lane & 15), ks * 2 + (lane >> 4)) * 16));
            }
        }
        auto q_at = [&](int ks, uint32_t (&r)[4]) {
            if constexpr (D <= 128) {
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = qf[ks][e];
            } else {
                load_matrices(r, smem_of(qs + chunk_at<D / 8>(wr * 16 + (lane & 15), ks * 2 + (lane >> 4)) * 16));
            }
        };

        // scores
        const int first = (sg.tile0 + at) * TK;
        float s[KI][2][4];
        const auto *const k_sm = reinterpret_cast<const uint32_t *>(st + 2 * S::kRows), *const v_sm = k_sm + TK * NG;
#pragma unroll
        for (int ki = 0; ki < KI; ++ki) {
            const int key0 = (wk * KI + ki) * 16;
#pragma unroll
            for (int tl = 0; tl < 2; ++tl) s[ki][tl][0] = s[ki][tl][1] = s[ki][tl][2] = s[ki][tl][3] = 0.f;
            if constexpr (!kQuant) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    uint32_t b[4], q[4];
                    load_matrices(b, smem_of(st + k_chunk_at<S>(key0 + (lane & 7) + ((lane >> 4) & 1) * 8, ks * 2 + ((lane >> 3) & 1)) * 16));
                    q_at(ks, q);
                    mma_bf16(s[ki][0], q[0], q[1], q[2], q[3], b[0], b[1]);
                    mma_bf16(s[ki][1], q[0], q[1], q[2], q[3], b[2], b[3]);
                }
            } else {
#pragma unroll
                for (int grp = 0; grp < NG; ++grp) {
                    float part[2][4] = {};
#pragma unroll
                    for (int run = 0; run < S::G / 32; ++run) {
                        const int blk = grp * (S::G / 32) + run;
                        uint32_t q0[4], q1[4];
                        q_at(blk * 2, q0), q_at(blk * 2 + 1, q1);
#pragma unroll
                        for (int tl = 0; tl < 2; ++tl) {
                            const int key = key0 + tl * 8 + g;
                            if constexpr (BITS == 8) {
                                const uint2 w = *reinterpret_cast<const uint2 *>(st + k_chunk_at<S>(key, blk * 2 + (t4 >> 1)) * 16 + (t4 & 1) * 8);
                                mma_f16(part[tl], q0, bytes_f16(w.x, 0x4140), bytes_f16(w.x, 0x4342));
                                mma_f16(part[tl], q1, bytes_f16(w.y, 0x4140), bytes_f16(w.y, 0x4342));
                            } else {
                                const uint32_t w = *reinterpret_cast<const uint32_t *>(st + k_chunk_at<S>(key, blk) * 16 + t4 * 4);
                                mma_f16(part[tl], q0, nibbles_f16(w), nibbles_f16(w >> 4));
                                mma_f16(part[tl], q1, nibbles_f16(w >> 8), nibbles_f16(w >> 12));
                            }
                        }
                    }
                    const float qs0 = q_sums[(wr * 16 + g) * NG + grp], qs1 = q_sums[(wr * 16 + g + 8) * NG + grp];
#pragma unroll
                    for (int tl = 0; tl < 2; ++tl)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t w = k_sm[(key0 + tl * 8 + 2 * t4 + e) * NG + grp];
                            const float sc = __uint_as_float(w << 16), mn = __uint_as_float(w & 0xffff0000u);
                            s[ki][tl][e] = fmaf(sc, part[tl][e], fmaf(mn, qs0, s[ki][tl][e]));
                            s[ki][tl][2 + e] = fmaf(sc, part[tl][2 + e], fmaf(mn, qs1, s[ki][tl][2 + e]));
                        }
                }
            }
        }
        const int p_last = sg.p0 + sg.n - 1;
        const bool whole = first >= (a.window > 0 ? p_last - a.window + 1 : 0) && first + TK - 1 <= sg.p0;
        auto seen = [&](int ki, int tl, int e) {  // e: as in an accumulator
            const int j = first + (wk * KI + ki) * 16 + tl * 8 + 2 * t4 + (e & 1);
            return j <= hi[e >> 1] && j > lo[e >> 1];
        };
        float top[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
        for (int ki = 0; ki < KI; ++ki)
#pragma unroll
            for (int tl = 0; tl < 2; ++tl)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = s[ki][tl][e] * fac[e >> 1];
                    if (a.softcap > 0.f) v = a.softcap * tanhf(v / a.softcap);
                    v *= kLog2e;
                    if (!whole && !seen(ki, tl, e)) v = -CUDART_INF_F;
                    s[ki][tl][e] = v;
                    top[e >> 1] = fmaxf(top[e >> 1], v);
                }
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
            const float now = fmaxf(m[e], top[e]), base = now == -CUDART_INF_F ? 0.f : now;
            alpha[e] = exp2_fast(m[e] - base);
            m[e] = now, top[e] = base;
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int ki = 0; ki < KI; ++ki)
#pragma unroll
            for (int tl = 0; tl < 2; ++tl)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[ki][tl][e] = exp2_fast(s[ki][tl][e] - top[e >> 1]);
                    sum[e >> 1] += s[ki][tl][e];
                }
        l[0] = fmaf(l[0], alpha[0], sum[0]), l[1] = fmaf(l[1], alpha[1], sum[1]);

        // the largest scale of this warp's values, for the power of two that keeps weight times scale inside F16
        bool rescale = alpha[0] != 1.f || alpha[1] != 1.f;
        float o_scale[2] = {alpha[0], alpha[1]};
        if constexpr (kQuant) {
            int e_top = 0;
#pragma unroll
            for (int ki = 0; ki < KI; ++ki) {
                const int key = (wk * KI + ki) * 16 + (lane & 15);
#pragma unroll
                for (int grp = 0; grp < NG; ++grp) {
                    const int ex = (int)(v_sm[key * NG + grp] >> 7 & 0xffu);
                    if (ex != 255) e_top = max(e_top, ex);
                }
            }
            e_top = __reduce_max_sync(0xffffffffu, e_top);
            if (e_top > v_exp) {
                const float f = exp2_fast((float)(v_exp - e_top));
                o_scale[0] *= f, o_scale[1] *= f;
                v_exp = e_top, rescale = true;
            }
        }
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
            for (int d = 0; d < D / 8; ++d) o[d][0] *= o_scale[0], o[d][1] *= o_scale[0], o[d][2] *= o_scale[1], o[d][3] *= o_scale[1];
            if constexpr (kQuant) {
#pragma unroll
                for (int grp = 0; grp < NG; ++grp) o_min[0][grp] *= alpha[0], o_min[1][grp] *= alpha[1];
            }
        }

        // weights times values
        const uint8_t *const vt = st + S::kRows;
        if constexpr (!kQuant) {
#pragma unroll
            for (int ki = 0; ki < KI; ++ki) {
                const int key0 = (wk * KI + ki) * 16;
                // Keys that one row sees and another does not: an infinity or a NaN there must not reach the other through 0 * v.
                bool clean = true;
                if (!whole && sg.n > 1) {
                    for (int c = lane; c < 16 * CR; c += 32) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(vt + (key0 * CR + c) * 16);
                        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) clean = clean && (ws[e] & 0x7f80u) != 0x7f80u && (ws[e] & 0x7f800000u) != 0x7f800000u;
                    }
                    clean = __all_sync(0xffffffffu, clean);
                }
                if (clean) {
                    const uint32_t p0 = pack_bf16(s[ki][0][0], s[ki][0][1]), p1 = pack_bf16(s[ki][0][2], s[ki][0][3]);
                    const uint32_t p2 = pack_bf16(s[ki][1][0], s[ki][1][1]), p3 = pack_bf16(s[ki][1][2], s[ki][1][3]);
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        uint32_t b[4];
                        load_matrices_trans(b, smem_of(vt + chunk_at<CR>(key0 + (lane & 15), d * 2 + (lane >> 4)) * 16));
                        mma_bf16(o[2 * d], p0, p1, p2, p3, b[0], b[1]);
                        mma_bf16(o[2 * d + 1], p0, p1, p2, p3, b[2], b[3]);
                    }
                } else {
#pragma unroll 1
                    for (int k = 0; k < 16; ++k) {
                        const int from = (lane & ~3) | (k % 8 / 2), j = first + key0 + k;
                        float w[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float even = __shfl_sync(0xffffffffu, k < 8 ? s[ki][0][2 * e] : s[ki][1][2 * e], from);
                            const float odd = __shfl_sync(0xffffffffu, k < 8 ? s[ki][0][2 * e + 1] : s[ki][1][2 * e + 1], from);
                            w[e] = k & 1 ? odd : even;
                        }
#pragma unroll
                        for (int d = 0; d < D / 8; ++d) {
                            const uint32_t v = *reinterpret_cast<const uint32_t *>(vt + chunk_at<CR>(key0 + k, d) * 16 + t4 * 4);
                            const float v0 = __uint_as_float(v << 16), v1 = __uint_as_float(v & 0xffff0000u);
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (j <= hi[e] && j > lo[e]) o[d][2 * e] = fmaf(w[e], v0, o[d][2 * e]), o[d][2 * e + 1] = fmaf(w[e], v1, o[d][2 * e + 1]);
                        }
                    }
                }
            }
        } else {
            const float v_up = __uint_as_float((uint32_t)(141 - v_exp + 127) << 23);  // 2^(14 - (v_exp - 127))
#pragma unroll
            for (int ki = 0; ki < KI; ++ki) {
                const int key0 = (wk * KI + ki) * 16;
#pragma unroll
                for (int grp = 0; grp < NG; ++grp) {
                    float w[2][4];
#pragma unroll
                    for (int tl = 0; tl < 2; ++tl)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t x = v_sm[(key0 + tl * 8 + 2 * t4 + e) * NG + grp];
                            const float sc = __uint_as_float(x << 16) * v_up, mn = __uint_as_float(x & 0xffff0000u);
#pragma unroll
                            for (int rr = 0; rr < 2; ++rr) {
                                const float p = s[ki][tl][2 * rr + e];
                                if (whole || seen(ki, tl, 2 * rr + e)) {  // a scale or min that is none must not reach a row that does not see it
                                    w[tl][2 * rr + e] = p * sc;
                                    o_min[rr][grp] = fmaf(p, mn, o_min[rr][grp]);
                                } else {
                                    w[tl][2 * rr + e] = 0.f;
                                }
                            }
                        }
                    const uint32_t pa[4] = {pack_f16(w[0][0], w[0][1]), pack_f16(w[0][2], w[0][3]), pack_f16(w[1][0], w[1][1]), pack_f16(w[1][2], w[1][3])};
                    if constexpr (BITS == 8) {
#pragma unroll
                        for (int run = 0; run < S::G / 32; ++run) {  // two chunks of sixteen columns
                            const int c = grp * (S::G / 16) + run * 2;
                            uint32_t b[4];
                            load_matrices_trans(b, smem_of(vt + chunk_at<CR>(key0 + (lane & 15), c + (lane >> 4)) * 16));
                            mma_f16(o[2 * c], pa, bytes_f16(b[0], 0x4240), bytes_f16(b[1], 0x4240));
                            mma_f16(o[2 * c + 1], pa, bytes_f16(b[0], 0x4341), bytes_f16(b[1], 0x4341));
                            mma_f16(o[2 * c + 2], pa, bytes_f16(b[2], 0x4240), bytes_f16(b[3], 0x4240));
                            mma_f16(o[2 * c + 3], pa, bytes_f16(b[2], 0x4341), bytes_f16(b[3], 0x4341));
                        }
                    } else {
#pragma unroll
                        for (int run = 0; run < S::G / 32; ++run) {  // a chunk of 32 columns; the matrices of a second one belong to another run or group
                            const int c = grp * (S::G / 32) + run;
                            uint32_t b0, b1;
                            asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
                                         : "=r"(b0), "=r"(b1)
                                         : "r"(smem_of(vt + chunk_at<CR>(key0 + (lane & 15), c) * 16))
                                         : "memory");
#pragma unroll
                            for (int e = 0; e < 4; ++e) mma_f16(o[4 * c + e], pa, nibbles_f16(b0 >> (4 * e)), nibbles_f16(b1 >> (4 * e)));
                        }
                    }
                }
            }
        }
        if (tid < kMaxIds) ids[((ahead + 1) & 1) * kMaxIds + tid] = next_id;

        if (++at < sg.tiles && i + 1 < units) continue;

        // ---- the segment's end, or this CTA's share's: the warps' sums become one ----
        const int64_t seg0 = u0 + (i + 1) - at, seg1 = seg0 + sg.tiles;  // the segment's units in the list
        const bool split = seg0 < u0 || seg1 > u1;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
            if (t4 == 0) row_max[wk * R + wr * 16 + g + 8 * e] = m[e], row_sum[wk * R + wr * 16 + g + 8 * e] = l[e];
        }
        if constexpr (kQuant) {
            const float down = __uint_as_float((uint32_t)(v_exp - 141 + 127) << 23);
#pragma unroll
            for (int grp = 0; grp < NG; ++grp)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    o_min[e][grp] += __shfl_xor_sync(0xffffffffu, o_min[e][grp], 1);
                    o_min[e][grp] += __shfl_xor_sync(0xffffffffu, o_min[e][grp], 2);
                }
#pragma unroll
            for (int d = 0; d < D / 8; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[d][e] = fmaf(o[d][e], down, o_min[e >> 1][d * 8 / S::G]);
        }
        __syncthreads();
        auto factor = [&](int k, int r, float top_of) { return row_max[k * R + r] == -CUDART_INF_F ? 1.f : exp2_fast(row_max[k * R + r] - top_of); };
        auto top_of = [&](int r) {
            float v = row_max[r];
#pragma unroll
            for (int k = 1; k < WK; ++k) v = fmaxf(v, row_max[k * R + r]);
            return v;
        };
        float mine_f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) mine_f[e] = factor(wk, wr * 16 + g + 8 * e, top_of(wr * 16 + g + 8 * e));
        constexpr int DC = S::DC, kTurn = (DC / 8 - 1) & 7;
        auto *const joint = reinterpret_cast<float *>(S::kOwnJoint ? own_joint : st);  // [WK][R][DC], pairs of columns turned by the row
        float *const part = a.partial + (2 * (int64_t)blockIdx.x + (seg0 < u0 ? 0 : 1)) * R * (D + 2);
        const int rows = min(R, sg.n * a.group - sg.rows0);
#pragma unroll
        for (int col0 = 0; col0 < D; col0 += DC) {
            if (col0 > 0) __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = wr * 16 + g + 8 * e;
                float *const to = joint + (wk * R + r) * DC;
                auto put = [&](int col, float x, float y) {
                    *reinterpret_cast<float2 *>(to + 2 * (((col - col0) / 2) ^ ((r & kTurn) << 2))) = make_float2(x * mine_f[e], y * mine_f[e]);
                };
#pragma unroll
                for (int d = col0 / 8; d < (col0 + DC) / 8; ++d) {
                    if constexpr (BITS == 16) {
                        put(8 * d + 2 * t4, o[d][2 * e], o[d][2 * e + 1]);
                    } else if constexpr (BITS == 8) {  // accumulators 2 c, 2 c + 1: the even and the odd columns of sixteen
                        if (d % 2 == 0) {
                            put(8 * d + 4 * t4, o[d][2 * e], o[d + 1][2 * e]);
                            put(8 * d + 4 * t4 + 2, o[d][2 * e + 1], o[d + 1][2 * e + 1]);
                        }
                    } else {  // accumulator 4 c + x: columns 4 n + x of 32
                        if (d % 4 == 0) {
                            put(8 * d + 8 * t4, o[d][2 * e], o[d + 1][2 * e]);
                            put(8 * d + 8 * t4 + 2, o[d + 2][2 * e], o[d + 3][2 * e]);
                            put(8 * d + 8 * t4 + 4, o[d][2 * e + 1], o[d + 1][2 * e + 1]);
                            put(8 * d + 8 * t4 + 6, o[d + 2][2 * e + 1], o[d + 3][2 * e + 1]);
                        }
                    }
                }
            }
            __syncthreads();
            for (int x = tid; x < rows * (DC / 4); x += kThreads) {
                const int r = x / (DC / 4), c4 = x % (DC / 4);
                const float *const from = joint + r * DC + 2 * ((2 * c4) ^ ((r & kTurn) << 2));
                float4 v = *reinterpret_cast<const float4 *>(from);
                const float top_r = top_of(r);
                float sum_r = row_sum[r] * factor(0, r, top_r);
#pragma unroll
                for (int k = 1; k < WK; ++k) {
                    const float4 w = *reinterpret_cast<const float4 *>(from + k * R * DC);
                    v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
                    sum_r = fmaf(row_sum[k * R + r], factor(k, r, top_r), sum_r);
                }
                if (split) {
                    *reinterpret_cast<float4 *>(part + r * D + col0 + 4 * c4) = v;
                    if (col0 == 0 && c4 == 0) part[R * D + r] = top_r, part[R * (D + 1) + r] = sum_r;
                } else {
                    const int tok = (sg.rows0 + r) / a.group, head = sg.head * a.group + sg.rows0 + r - tok * a.group;
                    const float inv = sg.bad ? qnan_f32() : sum_r == 0.f ? 0.f : 1.f / sum_r;
                    uint2 w;
                    w.x = pack_bf16(v.x * inv, v.y * inv), w.y = pack_bf16(v.z * inv, v.w * inv);
                    *reinterpret_cast<uint2 *>(a.out + (sg.q0 + tok) * a.out_ld + (int64_t)head * D + col0 + 4 * c4) = w;
                    if (a.lse != nullptr && col0 == 0 && c4 == 0)
                        a.lse[(int64_t)(sg.q0 + tok) * a.n_q + head] = sg.bad ? qnan_f32() : sum_r == 0.f ? -CUDART_INF_F : fmaf(top_r, kLn2, logf(sum_r));
                }
            }
        }
        if (split) {
            // the CTAs that share the segment are those whose runs hold its units; the first one's number is the counter's
            auto cta_of = [&](int64_t u) { return ((u + 1) * ctas + total - 1) / total - 1; };
            const int64_t c0 = cta_of(seg0), c1 = cta_of(seg1 - 1);
            auto *const last = reinterpret_cast<int *>(scan);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const uint32_t before = atomicAdd(a.count + c0, 1u);
                *last = before == (uint32_t)(c1 - c0);
                if (*last) a.count[c0] = 0;
            }
            __syncthreads();
            if (*last) {
                __threadfence();
                for (int x = tid; x < rows * (D / 4); x += kThreads) {
                    const int r = x / (D / 4), c4 = x % (D / 4);
                    const int64_t step = 2 * (int64_t)R * (D + 2);
                    const float *const p0 = a.partial + (2 * c0 + 1) * R * (D + 2), *const p1 = a.partial + 2 * (c0 + 1) * R * (D + 2);
                    const int more = (int)(c1 - c0);
                    float top_r = __ldcg(p0 + R * D + r);
#pragma unroll 4
                    for (int k = 0; k < more; ++k) top_r = fmaxf(top_r, __ldcg(p1 + k * step + R * D + r));
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    float sum_r = 0.f;
#pragma unroll 4
                    for (int k = -1; k < more; ++k) {
                        const float *const p = k < 0 ? p0 : p1 + k * step;
                        const float top_k = __ldcg(p + R * D + r), f = top_k == -CUDART_INF_F ? 1.f : exp2_fast(top_k - top_r);
                        const float4 w = __ldcg(reinterpret_cast<const float4 *>(p + r * D + 4 * c4));
                        sum_r = fmaf(__ldcg(p + R * (D + 1) + r), f, sum_r);
                        v.x = fmaf(w.x, f, v.x), v.y = fmaf(w.y, f, v.y), v.z = fmaf(w.z, f, v.z), v.w = fmaf(w.w, f, v.w);
                    }
                    const int tok = (sg.rows0 + r) / a.group, head = sg.head * a.group + sg.rows0 + r - tok * a.group;
                    const float inv = sum_r == 0.f ? 0.f : 1.f / sum_r;
                    uint2 w;
                    w.x = pack_bf16(v.x * inv, v.y * inv), w.y = pack_bf16(v.z * inv, v.w * inv);
                    *reinterpret_cast<uint2 *>(a.out + (sg.q0 + tok) * a.out_ld + (int64_t)head * D + 4 * c4) = w;
                    if (a.lse != nullptr && c4 == 0) a.lse[(int64_t)(sg.q0 + tok) * a.n_q + head] = sum_r == 0.f ? -CUDART_INF_F : fmaf(top_r, kLn2, logf(sum_r));
                }
            }
        }
        fresh = true, ++segment;
    }
}

// The form for the rows that a key head's queries make: more query heads a key head or more drafts, more rows a tile.
inline int row_warps(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

template <class S> struct Launch {
    static int64_t ctas() { return (int64_t)sm_count() * S::kPerSm; }
    static size_t bytes() { return (size_t)((ctas() * 4 + 255) / 256 * 256 + ctas() * 2 * S::R * (S::D + 2) * 4); }
    static cudaError_t run(Args a, void *ws, int64_t most_units, cudaStream_t st) {
        const int64_t n = std::max<int64_t>(1, std::min(ctas(), (most_units + kMinRun - 1) / kMinRun));
        a.count = static_cast<uint32_t *>(ws);
        a.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + (ctas() * 4 + 255) / 256 * 256);
        const cudaError_t rc = cudaFuncSetAttribute(attn_decode_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
        if (rc != cudaSuccess) return rc;
        return launch_behind(attn_decode_kernel<S>, dim3((unsigned)n), dim3(S::kThreads), (size_t)S::kSmem, st, 1, a);
    }
};

// f(Shape) for the sizes of a call; -1 where there is none.
template <int D, int BITS, int G, class F> auto with_rows(int wr, F f) {
    if (wr == 1) return f(Shape<D, BITS, G, 1>{});
    if (wr == 2) return f(Shape<D, BITS, G, 2>{});
    return f(Shape<D, BITS, G, 4>{});
}
template <int D, class F> auto with_cache(int bits, int64_t G, int wr, F f) {
    if (bits == 16) return with_rows<D, 16, D>(wr, f);
    if (bits == 8) {
        if (G == 32) return with_rows<D, 8, 32>(wr, f);
        if (G == 64) return with_rows<D, 8, 64>(wr, f);
        return with_rows<D, 8, D < 128 ? D : 128>(wr, f);
    }
    if (G == 32) return with_rows<D, 4, 32>(wr, f);
    if (G == 64) return with_rows<D, 4, 64>(wr, f);
    return with_rows<D, 4, D < 128 ? D : 128>(wr, f);
}
template <class F> auto with_shape(int64_t D, int bits, int64_t G, int wr, F f) {
    if (D == 64) return with_cache<64>(bits, G, wr, f);
    if (D == 128) return with_cache<128>(bits, G, wr, f);
    return with_cache<256>(bits, G, wr, f);
}

}  // namespace
}  // namespace sxb

using namespace sxb;

extern "C" size_t sxb_attn_decode_workspace_bytes(int64_t n_q, int64_t n_kv, int64_t D, int bits, int64_t max_q) {
    const char *fn = "attn_decode_workspace_bytes";
    if (!(n_kv >= 1 && n_q >= n_kv && n_q <= 1024 && n_q % n_kv == 0 && (D == 64 || D == 128 || D == 256) && (bits == 16 || bits == 8 || bits == 4) &&
          max_q >= 1 && max_q <= kMaxRows)) {
        fail_check(SXB_FILE_, __LINE__, __func__, "sizes",
                   cat(fn, ": n_q = ", n_q, ", n_kv = ", n_kv, ", D = ", D, ", bits = ", bits, ", max_q = ", max_q, " unsupported"));
        return 0;
    }
    return with_shape(D, bits, 32, row_warps(max_q * (n_q / n_kv)), [](auto s) { return Launch<decltype(s)>::bytes(); });
}

extern "C" int sxb_attn_decode(const void *q, int64_t q_ld, int64_t T, int64_t n_q, const SxbKvCache *cache, const int32_t *pages, int64_t pages_ld,
                               int64_t n_cols, const int32_t *q_start, const int32_t *kv_len, int64_t B, int64_t max_q, float scale, float softcap,
                               int64_t window, void *out, int64_t out_ld, float *lse, void *ws, size_t ws_bytes, uint32_t *err, sxb_stream_t stream) {
    const char *fn = "attn_decode";
    Args a{};
    if (int rc = kv_view(fn, cache, &a.c)) return rc;
    SXB_CHECK(q != nullptr && out != nullptr && pages != nullptr && q_start != nullptr && kv_len != nullptr && ws != nullptr && err != nullptr, fn,
              ": null pointer (q=", q, ", out=", out, ", pages=", (const void *)pages, ", q_start=", (const void *)q_start, ", kv_len=",
              (const void *)kv_len, ", ws=", ws, ", err=", (const void *)err, ")");
    const int64_t D = cache->D, n_kv = cache->n_kv;
    SXB_CHECK(n_q >= n_kv && n_q <= 1024 && n_q % n_kv == 0, fn, ": n_q = ", n_q, " query heads over n_kv = ", n_kv, " key heads, expected a multiple up to 1024");
    SXB_CHECK(T >= 1 && T <= kMaxRows, fn, ": T = ", T, " rows, expected 1..2^24");
    SXB_CHECK(B >= 1 && B <= (1 << 20), fn, ": B = ", B, " sequences, expected 1..2^20");
    SXB_CHECK(max_q >= 1 && max_q <= kMaxRows, fn, ": max_q = ", max_q, ", expected 1..2^24");
    SXB_CHECK(n_cols >= 1 && pages_ld >= n_cols, fn, ": page table of ", n_cols, " columns with a stride of ", pages_ld);
    SXB_CHECK(n_cols <= ((1ll << 31) - 1024) / cache->page, fn, ": ", n_cols, " pages of ", cache->page, " tokens a sequence, positions end below 2^31 - 1024");
    SXB_CHECK(q_ld >= n_q * D && q_ld <= (1ll << 32) && q_ld % 8 == 0 && out_ld >= n_q * D && out_ld <= (1ll << 32) && out_ld % 8 == 0, fn, ": row strides ",
              q_ld, " and ", out_ld, ", expected multiples of 8, at least n_q * D = ", n_q * D);
    SXB_CHECK(aligned16(q) && aligned16(out) && aligned16(ws), fn, ": q, out and ws must be 16-byte aligned");
    SXB_CHECK(apart(q, ((T - 1) * q_ld + n_q * D) * 2, out, ((T - 1) * out_ld + n_q * D) * 2), fn, ": out [", out, "] overlaps q [", q, "]");
    SXB_CHECK(scale > -1e30f && scale < 1e30f, fn, ": scale must be finite");
    SXB_CHECK(softcap >= 0.f && softcap < 1e30f, fn, ": softcap must be finite and not negative (0: none)");
    SXB_CHECK(window >= 0 && window < (1ll << 31), fn, ": window = ", window, ", expected 0 (none) .. 2^31 - 1");
    const int wr = row_warps(max_q * (n_q / n_kv));
    const size_t need = sxb_attn_decode_workspace_bytes(n_q, n_kv, D, cache->bits, max_q);
    SXB_CHECK(ws_bytes >= need, fn, ": workspace of ", ws_bytes, " bytes, needs ", need);
    a.q = static_cast<const uint16_t *>(q), a.q_ld = q_ld, a.pages = pages, a.pages_ld = pages_ld, a.capacity = n_cols * cache->page;
    a.q_start = q_start, a.kv_len = kv_len, a.B = (int)B, a.T = (int)T, a.n_q = (int)n_q, a.group = (int)(n_q / n_kv), a.window = (int)window;
    a.scale = scale, a.softcap = softcap, a.out = static_cast<uint16_t *>(out), a.out_ld = out_ld, a.lse = lse, a.err = err;
    auto st = static_cast<cudaStream_t>(stream);
    const cudaError_t rc = with_shape(D, cache->bits, cache->G, wr, [&](auto s) {
        using S = decltype(s);
        // no list is longer than every sequence at its table's end (in a product that cannot overflow: the grid is a few hundred CTAs)
        const double most = (double)((a.capacity + S::TK - 1) / S::TK) * (double)B * n_kv * (double)((T * a.group + S::R - 1) / S::R + 1);
        return Launch<S>::run(a, ws, (int64_t)std::min(most, 1e12), st);
    });
    if (rc != cudaSuccess) return fail_cuda(SXB_FILE_, __LINE__, __func__, rc, cat(fn, " launch"));
    SXB_CHECK_LAUNCH(fn, " T=", T, " B=", B, " n_q=", n_q, " n_kv=", n_kv, " D=", D, " bits=", cache->bits);
    return SXB_OK;
}
