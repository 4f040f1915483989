// Attention of a few new tokens a sequence over a paged key-value cache (sxb_attn_decode).
//
//   s_j = scale * q . k_j,   o = sum_j exp(s_j - M) v_j / sum_j exp(s_j - M),   M = max_j s_j,   lse = M + log(sum_j exp(s_j - M))
//
// One pass over the keys with a running maximum and sum.  The work is one list of units - a unit is a tile of TK keys of one (sequence, key head, tile
// of R query rows) - and every CTA takes an equal run of it, across the ends of heads and sequences: a batch of uneven lengths, or one long sequence
// alone, keeps all SMs equally busy, whatever the host knows of the lengths, and a captured graph follows them.  A segment (all units of one row tile)
// that lies in one CTA is written by it; the parts of one that several CTAs share go to the workspace, FP32 with their maxima and sums, at most two a
// CTA, and the last CTA to arrive (or, for many rows, a second kernel) joins them in the list's order, so that no result depends on who came last.
//
// The query heads of a key head and the new tokens of a sequence are the rows of one MMA tile: the cache is read once for all of them.  Products on
// mma.sync: the rows are eight to 32, a warp's keys sixteen, and what bounds is memory (BF16) or the conversion of codes, not the tensor cores; operands
// come from shared memory, tiles there by cp.async from wherever the pages lie, each warp's by itself.
//   BF16 cache: exact products; weights rounded to BF16, as the second product's operands have one type (one rounding of 2^-9 a key, to either side, against
//   the sum's many keys; the sum of weights keeps them unrounded).
//   8 and 4 bits: the codes are F16 numbers exactly, q is F16 times a power of two a row (a BF16 number less than 2^28 below the row's largest is exact),
//   scale and min go on in FP32: s = scale_k * (q . code) + min_k * sum(q) a group.  For V a key's weight takes its group's scale, times a power of
//   two that follows the largest scale seen so that F16's range is no limit (one rounding of 2^-11); the mins' share, sum p * min, is FP32.  Sixteen keys among
//   whose scales one is far below the largest, or none, are added up by the threads in FP32 (add_values).
// Exponentials are ex2.approx (2^-22 of a weight, below either rounding).
//
// Measured (B200; us, and the time of the bytes alone at the measured copy rate): one sequence of 200001 keys, 8 key heads of 128, BF16, 129 (125); 64
// sequences of 100 to 16000 keys, 8 bits, 190 (172); 32 of 9509, 4 bits with groups of 32, 144 (59): there the bound is the integer pipe, half busy with
// codes and scales, behind it two to three warps a scheduler.  Several rows: 32 sequences x 4 rows of 8 heads x 9509 keys BF16 109 (95), 8 bits 160 (51).
// 300 keys of one sequence: 7, nothing but latencies - lengths, page table, keys, join.

#include "attn.cuh"
#include "route_pack.cuh"
#include "skinny_mma.cuh"
#include "tc_ptx.cuh"

#include <math_constants.h>

#include <atomic>
#include <type_traits>

namespace sxb {
namespace {

#define SXB_RARE(c) __builtin_expect(!!(c), 0)  // out of the loop's way

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMostPerSm = 4;
constexpr int kSlack = 8;      // powers of two that a weight may be above 1
// Powers of two that a value group's scale may be below the largest one so far.  The largest scale times a weight of 1 is 2^6 as an F16 number, one below by kSpread
// 2^-2: weights down to 2^-12 then keep F16's eleven bits, and what the smaller ones lose, 2^-25 a key at most, is 2^-23 of that group's own scale.
// Sixteen keys with a scale further down are added up in FP32 by the threads (three times their time: 32 sequences of 4009 keys, 8 bits, 35 us, 104 if all of them are).
constexpr uint32_t kSpread = 8;
constexpr uint32_t kLowestScale = (20 - kSpread) << 23;  // as a bit pattern
constexpr float kLowest = -1e30f;  // below every score; a row that sees no key keeps it
constexpr int64_t kMaxRows = 1ll << 24;

// Runs of sixteen keys that a warp takes at a time: two give it independent work and share what a step costs besides, where registers allow.  (Two in a
// loop, one after the other, are slower: 32 sequences of 9509 keys, 8 bits, 115 us side by side, 132 to 152 in turn.)
constexpr int key_runs(int D, int bits, int nt) { return nt * D <= 256 && D * bits <= 1024 ? 2 : 1; }
// R query rows, NT tiles of eight, all of them every warp's.  The four warps share a tile's keys, a run of KI times sixteen each, and every warp fetches its
// own run into its own ring: nothing but a segment's ends is the whole CTA's business.
template <int D_, int BITS_, int G_, int R_> struct Shape {
    static constexpr int D = D_, BITS = BITS_, G = G_, R = R_;
    static constexpr bool kQuant = BITS != 16;
    static constexpr int NT = R / 8, kWarps = 4, kThreads = 32 * kWarps, WK = kWarps;
    static constexpr int RB = D * BITS / 8, CR = RB / 16;  // bytes and 16-byte chunks of a cache row
    static constexpr int NG = kQuant ? D / G : 0;
    static constexpr int KI = key_runs(D, BITS, NT), RUN = 16 * KI, TK = RUN * WK;
    static constexpr int kRows = RUN * RB, kScales = RUN * NG * 4, kPart = 2 * (kRows + kScales), kStage = WK * kPart;
    static constexpr int kQ = R * D * 2;
    static constexpr int kMostJoint = WK * R * 32 * 4;
    static constexpr bool kOwnJoint = kStage < kMostJoint;  // 32 columns of every warp's rows do not fit a stage
    static constexpr int kMisc = 1024 + kWarps * 64 + WK * R * 8 + R * (2 * NG + 2) * 4 + (kOwnJoint ? kMostJoint : 0);
    // CTAs an SM: as many as registers allow (three of four warps with 168 registers a thread, two with 255), if their rings then still have 64 KB on the way
    static constexpr int kByRegisters = kQuant && NT * D <= 128 ? 3 : 2;
    static constexpr int stages(int per_sm) { return (226 * 1024 / per_sm - kMisc) / (kStage + kQ); }
    static constexpr bool fits(int per_sm) { return kByRegisters >= per_sm && stages(per_sm) >= 2 && per_sm * (stages(per_sm) - 1) * kStage >= 64 * 1024; }
    static constexpr int kPerSm = fits(3) ? 3 : fits(2) ? 2 : 1;
    static constexpr int kStages = stages(kPerSm) > 6 ? 6 : stages(kPerSm);
    static constexpr int kSmem = kStages * (kStage + kQ) + kMisc;
    static constexpr int fit_columns() {
        int dc = D;
        while (dc > 32 && WK * R * dc * 4 > kStage) dc /= 2;
        return dc;
    }
    static constexpr int DC = fit_columns();  // columns that the warps join at a time
    // Codes stay too large by so much as F16 operands, and what that adds is taken out of the sums: K's by 1024 (8 bits) or 64, V's too, but for every
    // second 4-bit code, which 1024 saves a shift - what that costs a score (an offset of a hundred times the codes) would be seen, of an output it is not
    // (where it leaves the sums every sixteen tiles: see take_out).
    static constexpr float kOffsetK = BITS == 8 ? 1024.f : 64.f, kOffset = 1024.f, kOffsetOdd = kOffsetK;
    // Few rows: the last CTA to bring its part joins them, a launch less.  Many: that CTA would read every part by itself (2 x 8 rows over 32 k keys:
    // 19 parts of 33 KB, 30 us at the end of 80), a second kernel has the rows of all segments side by side.
    static constexpr bool kJoinHere = R * D <= 8 * kThreads;  // a thread has two runs of four columns at most
    static constexpr bool kHoldQ = !kQuant && NT * D <= 256;  // q's fragments in registers
    static_assert(kStages >= 2 && KI * NT * 4 <= 32, "");
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
    struct Join *joins;
    uint32_t *status;                  // of the tcgen05 form: a wait that ran out
    unsigned long long wait_limit_ns;
    int test_skip_slot;                // >= 0: CTA 0 of that form leaves that fill of keys and values out, so that a wait runs out (tests only)
    int box_rows;
    // distances in pieces of sixteen bytes (codes) and of a row's scales: a cache has fewer than 2^32 of either
    uint32_t page_chunks, head_chunks, row_chunks, page_pieces, head_pieces, row_pieces;
};

// A split segment whose first part is the CTA's of the same number; parts = 0: that CTA began none.
struct Join {
    int q0, rows0, head, rows, parts, unused[3];
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
    s.lo = a.window > 0 ? (int)max((int64_t)0, (int64_t)s.p0 - a.window + 1) : 0;
    s.tile0 = s.lo / S::TK;
    s.tiles = max(1, (s.len + S::TK - 1) / S::TK - s.tile0);
    s.row_tiles = (int)(((int64_t)s.n * a.group + S::R - 1) / S::R);
    if (skip) s.bad = true;
    return s;
}

// A segment of the list that this CTA has units of.
struct Segment {
    int q0, n, len, p0, lo, tile0, tiles, head, rows0, at, bad;  // rows0: first row of the tile, at: the CTA's first unit's place in the segment
};

// Where a warp's loads are: in shared memory, what is looked at in the loop apart.
struct Cursor {
    Sequence s;
    int b, head, row_tile, segment;
};

__device__ inline uint32_t smem_of(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// n bytes (0: zeros instead), to a place OFF bytes behind `to`.
template <int BYTES, int OFF = 0> __device__ inline void copy_async(uint32_t to, const void *from, int n) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0 + %3], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n), "n"(OFF) : "memory");
    else if constexpr (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0 + %3], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(n), "n"(OFF) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0 + %3], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(n), "n"(OFF) : "memory");
}
template <int BYTES, int OFF = 0, int FROM = 0> __device__ inline void copy_async(uint32_t to, const void *from) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(to), "l"(from), "n"(OFF), "n"(FROM) : "memory");
    else if constexpr (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0 + %2], [%1 + %3], 8;" ::"r"(to), "l"(from), "n"(OFF), "n"(FROM) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0 + %2], [%1 + %3], 4;" ::"r"(to), "l"(from), "n"(OFF), "n"(FROM) : "memory");
}
__device__ inline void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ inline void wait_async() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Volatile: they stay behind the wait that they follow; nothing is written that the compiler knows of.
template <int OFF = 0> __device__ inline void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at), "n"(OFF));
}
template <int OFF> __device__ inline void load_matrices_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at), "n"(OFF));
}
template <int OFF> __device__ inline void load_matrices_trans(uint32_t (&r)[2], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2 + %3];" : "=r"(r[0]), "=r"(r[1]) : "r"(at), "n"(OFF));
}
template <int OFF> __device__ inline void load_shared(uint32_t (&w)[1], uint32_t at) { asm volatile("ld.shared.b32 %0, [%1 + %2];" : "=r"(w[0]) : "r"(at), "n"(OFF)); }
template <int OFF> __device__ inline void load_shared(uint32_t (&w)[2], uint32_t at) {
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2 + %3];" : "=r"(w[0]), "=r"(w[1]) : "r"(at), "n"(OFF));
}
template <int OFF> __device__ inline void load_shared(uint32_t (&w)[4], uint32_t at) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at), "n"(OFF));
}
template <int OFF> __device__ inline void load_shared(uint32_t (&w)[8], uint32_t at) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at), "n"(OFF));
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "r"(at), "n"(OFF + 16));
}
// f(integral_constant) for 0 .. N - 1: loops whose counters are immediates.
template <int N, int I = 0, class F> __device__ inline void each(F f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        each<N, I + 1>(f);
    }
}
template <bool F16> __device__ inline void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ inline float exp2_flushed(float v) {  // 2 ulp; exp2(-inf) = 0
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ inline float reciprocal_fast(float v) {  // 1 ulp
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// A score s * fac (in powers of two) under a cap: to * tanh(x), x = s * fac / to.  Below a quarter the odd series to its fourth term, x - x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315,
// as a factor of the score itself (62 x^8 / 2835 is left off: 2^-21.5 at most); above it 1 - 2 / (exp(2 x) + 1), whose cancellation is 2^-19.9 of what it gives at a quarter, and
// less further on: FP32's own error of a score, whatever the cap.  by = 2 ln 2 / to (as a power of two's exponent, 2 x is s * fac * by).
__device__ inline float capped(float s, float fac, float by, float to) {
    const float t = s * (fac * by), x2 = t * t * (0.25f * kLn2 * kLn2);
    const float near = s * fac * fmaf(x2, fmaf(x2, fmaf(x2, -17.f / 315, 2.f / 15), -1.f / 3), 1.f);
    const float far = fmaf(-2.f * to, reciprocal_fast(exp2_flushed(t) + 1.f), to);
    return fabsf(t) < 0.5f * kLog2e ? near : far;
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
// Two bytes of a word (named by the selector's nibbles 0 and 2) as F16 numbers 1024 + code; the lowest nibble of each half as 1024 + code, the next one as
// 64 + code.
__device__ inline uint32_t bytes_f16(uint32_t w, uint32_t selector) { return __byte_perm(w, 0x64646464u, selector); }
__device__ inline uint32_t low_nibbles_f16(uint32_t w) { return (w & 0x000f000fu) | 0x64006400u; }
__device__ inline uint32_t next_nibbles_f16(uint32_t w) { return (w & 0x00f000f0u) | 0x54005400u; }
__device__ inline uint32_t transposed(uint32_t v) {  // of an 8 x 8 tile of 16-bit numbers, a lane's two neighbours in a row
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

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

// The words of a lane's two keys of run KI, V's.
template <class S, int KI, int N> __device__ inline void value_words(uint32_t (&w)[2][N], uint32_t scales) {
    constexpr int kOff = S::kScales + KI * 16 * N * 4;
    load_shared<kOff>(w[0], scales), load_shared<kOff + 8 * N * 4>(w[1], scales);
}

// What the scales are multiplied by whose lowest power of two is v_low: 2^(14 - kSlack) over the largest.
__device__ inline float scale_up(uint32_t v_low) { return __uint_as_float(((2 * 127u + 14 - kSlack - kSpread) << 23) - v_low); }
// Whether a group's scale or min is an infinity or a NaN.
__device__ inline bool none_of(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

// Sixteen keys' values of codes added up by the threads in FP32, each row's for itself: weights p of the score accumulators' layout, hidden: those that do not
// count, o in the layout of the second product (less the codes' offsets).  What a group's scale or min is reaches its own columns and the rows that see the key.
template <class S, int KI>
__device__ inline void add_values(const uint8_t *values, const uint32_t (&words)[2][S::NG], const float (&p)[S::NT][4], uint32_t hidden, float v_up, int lane,
                                  float (&o)[S::D / 16][S::NT][4], float (&o_min)[S::NG][S::NT][2]) {
    constexpr int NT = S::NT, NG = S::NG, G = S::G;
    const int g = lane >> 2, t4 = lane & 3;
    const auto *const scales = reinterpret_cast<const uint32_t *>(values + S::kRows + S::kScales) + KI * 16 * NG;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if ((hidden >> (nt * 4 + e) & 1) == 0) {
#pragma unroll
                for (int grp = 0; grp < NG; ++grp) o_min[grp][nt][e & 1] = fmaf(p[nt][e], __uint_as_float(words[e >> 1][grp] & 0xffff0000u), o_min[grp][nt][e & 1]);
            }
#pragma unroll 1
    for (int k = 0; k < 16; ++k) {
        const int from = (k % 8) * 4 + t4;
        const uint32_t out_of_sight = __shfl_sync(0xffffffffu, hidden, from) >> (k < 8 ? 0 : 2);
        float w[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float low = __shfl_sync(0xffffffffu, p[nt][e], from), high = __shfl_sync(0xffffffffu, p[nt][2 + e], from);
                w[nt][e] = k < 8 ? low : high;
            }
#pragma unroll
        for (int c = 0; c < S::CR; ++c) {  // a chunk of sixteen bytes: this lane has two of them, two columns or four
            constexpr int kCols = 128 / S::BITS;
            const uint32_t code = *reinterpret_cast<const uint16_t *>(values + chunk_at<S::CR>(KI * 16 + k, c) * 16 + 2 * g);
            const float scale = __uint_as_float(scales[k * NG + c * kCols / G] << 16) * v_up;
#pragma unroll
            for (int x = 0; x < 16 / S::BITS; ++x) {
                const float v = scale * (float)(code >> (x * S::BITS) & ((1u << S::BITS) - 1));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float &to = o[c * kCols / 16 + x / 2][nt][2 * (x & 1) + e];
                        if ((out_of_sight >> (nt * 4 + e) & 1) == 0) to = fmaf(w[nt][e], v, to);
                    }
            }
        }
    }
}

// BF16 NaN throughout.
template <int BYTES> __device__ inline void store_nan(uint32_t to) {
    for (int i = 0; i < BYTES; i += 4) asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + i), "r"(0x7fc07fc0u) : "memory");
}
// Sixteen rows, PASS of them at a time, K and V.  A place in a later pass is the first one's with the turn of its rows, and a constant: a tile starts
// at a multiple of 128 bytes, and where rows are shorter than that a pass is whole turns.  Rows that follow each other in memory (NEXT) have constant
// distances there too.  Of an EDGE only the rows from .. to - 1 are there, the others become zeros.
template <class S, int PASS, int OFF, bool NEXT, bool EDGE>
__device__ inline void copy_rows(uint32_t k_to, uint32_t v_to, const uint8_t *k, const uint8_t *v, uint64_t step, int row, int from, int to) {
    static_assert((S::CR >= 8 || PASS % 8 == 0) && S::kPart % 128 == 0 && S::kRows % 128 == 0, "");
    each<16 / PASS>([&](auto i) {
        constexpr int I = decltype(i)::value, kOff = I * PASS * S::RB, kTurn = S::CR >= 8 ? I * PASS & 7 : 0, kTurnK = S::BITS == 8 ? 2 * (kTurn & 3) : kTurn;
        if constexpr (EDGE) {
            const int n = row + I * PASS >= from && row + I * PASS < to ? 16 : 0;
            copy_async<16, OFF + kOff>(k_to ^ (kTurnK << 4), k, n);
            copy_async<16, OFF + kOff>(v_to ^ (kTurn << 4), v, n);
        } else {
            copy_async<16, OFF + kOff, NEXT ? kOff : 0>(k_to ^ (kTurnK << 4), k);
            copy_async<16, OFF + kOff, NEXT ? kOff : 0>(v_to ^ (kTurn << 4), v);
        }
        if (!NEXT) k += step, v += step;
    });
}

// A run of keys with a bad page, or of pages of eight tokens: each row looks its page up.  Rows out of range become zeros, the keys of a bad page NaN.
// Out of line: the loop keeps its registers.
template <class S>
__device__ __noinline__ void load_ragged(const Args &a, const int32_t *table, uint32_t st, int run0, int lo, int len, int head, int b, int lane) {
    constexpr int CR = S::CR, NG = S::NG, RUN = S::RUN;
    constexpr int kPass = 32 / CR > RUN ? RUN : 32 / CR;
    const int page_mask = (1 << a.c.page_shift) - 1, chunk = lane % CR, row = lane / CR;
    auto place = [&](int r, bool &wanted) -> int64_t {  // of row r, -1: none
        const int j = run0 + r;
        wanted = j >= lo && j < len;
        if (!wanted) return -1;
        const int id = table[j >> a.c.page_shift];
        if ((unsigned)id < (unsigned)a.c.n_pages) return kv_row(a.c, id, head, j & page_mask);
        raise_error(a.err, (uint32_t)b, (uint32_t)id);
        return -1;
    };
    if (row < kPass) {
#pragma unroll 1
        for (int i = 0; i < RUN / kPass; ++i) {
            const int r = row + i * kPass;
            bool wanted;
            const int64_t from = place(r, wanted), off = from < 0 ? 0 : from * S::RB + chunk * 16;
            const uint32_t to = st + k_chunk_at<S>(r, chunk) * 16;
            if (!S::kQuant && wanted && from < 0) store_nan<16>(to);
            else copy_async<16>(to, a.c.k + off, from < 0 ? 0 : 16);
            copy_async<16>(st + S::kRows + chunk_at<CR>(r, chunk) * 16, a.c.v + off, from < 0 ? 0 : 16);
        }
    }
    if constexpr (S::kQuant) {
        constexpr int kBytes = NG * 4 > 16 ? 16 : NG * 4, kPieces = NG * 4 / kBytes;  // of a row's scales
#pragma unroll 1
        for (int i = lane; i < RUN * kPieces; i += 32) {
            const int r = i / kPieces, piece = i % kPieces;
            bool wanted;
            const int64_t from = place(r, wanted), off = from < 0 ? 0 : from * (NG * 4) + piece * kBytes;
            const uint32_t to = st + 2 * S::kRows + i * kBytes;
            if (wanted && from < 0) store_nan<kBytes>(to);
            else copy_async<kBytes>(to, reinterpret_cast<const uint8_t *>(a.c.k_sm) + off, from < 0 ? 0 : kBytes);
            copy_async<kBytes>(to + S::kScales, reinterpret_cast<const uint8_t *>(a.c.v_sm) + off, from < 0 ? 0 : kBytes);
        }
    }
}

// The parts of a split segment, [R][D] sums, [R] maxima, [R] sums of weights each: the first CTA's is its second one, the others' their first.
template <int R, int D> struct Parts {
    static constexpr int64_t kStep = 2 * (int64_t)R * (D + 2);
    const float *first, *rest;
    int n;
    __device__ Parts(const float *partial, int c0, int parts) : first(partial + (2 * (int64_t)c0 + 1) * R * (D + 2)), rest(partial + 2 * (int64_t)c0 * R * (D + 2)), n(parts) {}
    __device__ const float *of(int k) const { return k == 0 ? first : rest + k * kStep; }
};

// Four columns of a row out of all parts, in the parts' order, BATCH parts' loads at a time.
template <int BATCH, int R, int D> __device__ inline void join_run(const Args &a, const Parts<R, D> &from, int q0, int rows0, int key_head, int r, int c4) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f, top = kLowest;
    for (int k0 = 0; k0 < from.n; k0 += BATCH) {
        float4 w[BATCH];
        float m[BATCH], l[BATCH], now = top;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            m[k] = kLowest, l[k] = 0.f, w[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k0 + k < from.n) {
                const float *const p = from.of(k0 + k);
                w[k] = __ldcg(reinterpret_cast<const float4 *>(p + r * D + 4 * c4)), m[k] = __ldcg(p + R * D + r), l[k] = __ldcg(p + R * (D + 1) + r);
            }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) now = fmaxf(now, m[k]);
        const float before = exp2_flushed(top - now);
        v.x *= before, v.y *= before, v.z *= before, v.w *= before, sum *= before, top = now;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const float f = exp2_flushed(m[k] - top);
            sum = fmaf(l[k], f, sum), v.x = fmaf(w[k].x, f, v.x), v.y = fmaf(w[k].y, f, v.y), v.z = fmaf(w[k].z, f, v.z), v.w = fmaf(w[k].w, f, v.w);
        }
    }
    const int tok = (rows0 + r) / a.group, head = key_head * a.group + rows0 + r - tok * a.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint2 w;
    w.x = pack_bf16(v.x * inv, v.y * inv), w.y = pack_bf16(v.z * inv, v.w * inv);
    *reinterpret_cast<uint2 *>(a.out + (q0 + tok) * a.out_ld + (int64_t)head * D + 4 * c4) = w;
    if (a.lse != nullptr && c4 == 0) a.lse[(int64_t)(q0 + tok) * a.n_q + head] = sum == 0.f ? -CUDART_INF_F : fmaf(top, kLn2, logf(sum));
}

constexpr int kJoinRows = 8;
// Block (c, y): rows 8 y .. 8 y + 7 of the segment that began in CTA c, and as many again while there are more than were told of; a thread four columns.
template <class S>
__global__ void __launch_bounds__(kJoinRows * S::D / 4) attn_join_kernel(const __grid_constant__ Args a) {
    behind_grid();
    const Join j = a.joins[blockIdx.x];
    if (j.parts == 0) return;
    for (int r = blockIdx.y * kJoinRows + threadIdx.x / (S::D / 4); r < j.rows; r += gridDim.y * kJoinRows)
        join_run<8>(a, Parts<S::R, S::D>(a.partial, (int)blockIdx.x, j.parts), j.q0, j.rows0, j.head, r, threadIdx.x % (S::D / 4));
}

// The cursor of a warp at its next segment; false: there is none.
template <class S> __device__ inline bool next_segment(const Args &a, Cursor &cur, int lane) {
    Cursor c = cur;
    ++c.segment;
    if (++c.row_tile == c.s.row_tiles) {
        c.row_tile = 0;
        if (++c.head == a.c.n_kv) {
            c.head = 0;
            do {
                if (++c.b >= a.B) return false;
                c.s = sequence<S>(a, c.b);
            } while (c.s.n == 0);
        }
    }
    __syncwarp();
    if (lane == 0) cur = c;
    __syncwarp();
    return true;
}

// This CTA's run of the list: its first and last unit, all units, the CTAs that have one; the sequence of the first and the unit's number in it.  False: none.
struct Share {
    int64_t u0, u1, total, ctas;
    int b;
    int64_t in;
};
// By the whole CTA; scan: [kWarps + 2].
template <class S> __device__ inline bool find_share(const Args &a, int64_t *scan, Share &out) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int64_t total = 0;
    for (int b = tid; b < a.B; b += S::kThreads) {
        const Sequence s = sequence<S>(a, b);
        if (s.bad && blockIdx.x == 0) raise_error(a.err, (uint32_t)b, (uint32_t)a.kv_len[b]);
        total += (int64_t)s.tiles * s.row_tiles * a.c.n_kv;
    }
    if (!S::kJoinHere && tid == 0) a.joins[blockIdx.x].parts = 0;
    const int64_t mine = total;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (lane == 0) scan[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w) total += scan[w];
    const int64_t ctas = min((int64_t)gridDim.x, total);
    if ((int64_t)blockIdx.x >= ctas) return false;
    const int64_t u0 = blockIdx.x * total / ctas, u1 = (blockIdx.x + 1) * total / ctas;
    out = Share{u0, u1, total, ctas, 0, 0};
    for (int64_t base = 0, before = 0; base < a.B; base += S::kThreads) {
        int64_t own = mine;
        if (a.B > S::kThreads) {
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
        for (int w = 0; w < S::kWarps; ++w) {
            if (w < warp) ahead += scan[w];
            all += scan[w];
        }
        upto += ahead;
        if (upto - own <= u0 && u0 < upto) scan[S::kWarps] = base + tid, scan[S::kWarps + 1] = u0 - (upto - own);
        before = all;
        if (before > u0) break;
    }
    __syncthreads();
    out.b = (int)scan[S::kWarps], out.in = scan[S::kWarps + 1];
    return true;
}

template <class S>
__global__ void __launch_bounds__(S::kThreads, S::kPerSm) attn_decode_kernel(const __grid_constant__ Args a) {
    constexpr int D = S::D, BITS = S::BITS, NG = S::NG, TK = S::TK, KI = S::KI, RUN = S::RUN, R = S::R, WK = S::WK, CR = S::CR, NT = S::NT;
    constexpr int kStages = S::kStages, kThreads = S::kThreads, kWarps = S::kWarps;
    constexpr bool kQuant = S::kQuant;
    constexpr int kGroups = kQuant ? NG : 1;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *const q_ring = smem + kStages * S::kStage;
    uint8_t *const own_joint = q_ring + kStages * S::kQ, *const misc = own_joint + (S::kOwnJoint ? S::kMostJoint : 0);
    auto *const row_max = reinterpret_cast<float *>(misc);  // [WK][R]
    float *const row_sum = row_max + WK * R;                // [WK][R]
    float *const row_top = row_sum + WK * R;                // [R]
    float *const q_factor = row_top + R;                    // [R]
    float *const q_sums = q_factor + R;                     // [NG][R]: a group's sum of q, then what the codes' offsets add to its dot, less
    float *const q_extra = q_sums + NG * R;                 // [NG][R]
    auto *const scan = reinterpret_cast<int64_t *>(q_extra + R * NG);  // [kWarps + 2]
    auto *const list = scan + kWarps + 2;                                           // [4]: this CTA's first and last unit, all units, CTAs
    auto *const segments = reinterpret_cast<Segment *>(list + 4);                  // [kStages]
    Cursor &cur = reinterpret_cast<Cursor *>(segments + kStages)[threadIdx.x >> 5];  // [kWarps]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    behind_grid();

    Share share;
    if (!find_share<S>(a, scan, share)) return;
    const int64_t u0 = share.u0, u1 = share.u1, total = share.total, ctas = share.ctas, in = share.in;

    // ---- the cursor of the loads: kStages - 1 units ahead of the sums ----
    {
        Cursor c;
        c.b = share.b, c.s = sequence<S>(a, c.b), c.segment = 0;
        const int64_t per_head = (int64_t)c.s.tiles * c.s.row_tiles;
        c.head = (int)(in / per_head), c.row_tile = (int)((in - c.head * per_head) / c.s.tiles);
        if (lane == 0) cur = c;
        if (tid == 0) list[0] = u0, list[1] = u1, list[2] = total, list[3] = ctas;
    }
    __syncthreads();
    const int units = (int)(u1 - u0);
    const int page_mask = (1 << a.c.page_shift) - 1;
    constexpr int kPass = 32 / CR > 16 ? 16 : 32 / CR;  // rows that the warp fetches at a time
    constexpr int kBytes = NG * 4 > 16 ? 16 : NG * 4, kPieces = kQuant ? NG * 4 / kBytes : 1;  // of a row's scales
    constexpr int kScalePass = 32 / kPieces > 16 ? 16 : 32 / kPieces, kScalePasses = 16 / kScalePass;
    const int l_chunk = lane % CR, l_row = lane / CR, s_row = lane / kPieces, s_piece = lane % kPieces;
    const uint32_t smem0 = smem_of(smem);
    const uint32_t k_to0 = smem0 + warp * S::kPart + k_chunk_at<S>(l_row, l_chunk) * 16, v_to0 = smem0 + warp * S::kPart + S::kRows + chunk_at<CR>(l_row, l_chunk) * 16;
    const uint32_t s_to0 = smem0 + warp * S::kPart + 2 * S::kRows + lane * kBytes;
    uint32_t l_codes, l_scales;             // this lane's place in the head's first row
    int l_run0, l_lo, l_len, l_tiles;       // first key of the warp's run; the sequence's keys; tiles of the segment from here on
    const int32_t *l_table;
    bool l_new;                             // the run begins a segment
    auto at_segment = [&](int at) {         // the cursor stands at tile `at` of its segment
        l_codes = cur.head * a.head_chunks + l_row * a.row_chunks + l_chunk;
        l_scales = cur.head * a.head_pieces + s_row * a.row_pieces + s_piece;
        l_run0 = (cur.s.tile0 + at) * TK + warp * RUN, l_lo = cur.s.lo, l_len = cur.s.len, l_tiles = cur.s.tiles - at;
        l_table = a.pages + cur.b * a.pages_ld;
        l_new = true;
    };
    int l_page[KI];  // of the run's sixteens of keys: a page has sixteen or more, or load_ragged looks its ids up
    auto find_pages = [&]() {
#pragma unroll
        for (int ki = 0; ki < KI; ++ki) {
            const int first = l_run0 + 16 * ki;
            l_page[ki] = first < l_len && first + 15 >= l_lo ? l_table[first >> a.c.page_shift] : 0;
        }
    };
    auto advance = [&]() {
        l_new = false, l_run0 += TK;
        if (__builtin_expect(--l_tiles > 0, 1)) return;
        if (next_segment<S>(a, cur, lane)) at_segment(0);
    };
    auto load = [&](int stage) {
        const uint32_t by = stage * S::kStage;
        if (l_run0 >= l_len || l_run0 + RUN <= l_lo) return;  // nobody sees a key of it, and the sums leave it out
        bool fine = page_mask >= 15;
#pragma unroll
        for (int ki = 0; ki < KI; ++ki) fine = fine && (unsigned)l_page[ki] < (unsigned)a.c.n_pages;
        if (SXB_RARE(!fine)) {
            load_ragged<S>(a, l_table, smem0 + warp * S::kPart + by, l_run0, l_lo, l_len, cur.head, cur.b, lane);
            return;
        }
        const bool edge = l_run0 < l_lo || l_run0 + RUN > l_len;
        const uint64_t step = (uint64_t)a.row_chunks * (kPass * 16);
        each<KI>([&](auto kic) {
            constexpr int ki = decltype(kic)::value, kOff = ki * 16 * S::RB;
            const uint32_t in_page = (l_run0 + 16 * ki) & page_mask;
            const uint32_t chunk = (uint32_t)l_page[ki] * a.page_chunks + in_page * a.row_chunks + l_codes;
            const uint8_t *const k = a.c.k + (uint64_t)chunk * 16, *const v = a.c.v + (uint64_t)chunk * 16;
            if (kPass * CR == 32 || l_row < kPass) {
                if (SXB_RARE(edge)) copy_rows<S, kPass, kOff, false, true>(k_to0 + by, v_to0 + by, k, v, step, l_row, l_lo - l_run0 - 16 * ki, l_len - l_run0 - 16 * ki);
                else if (SXB_RARE(a.c.row_stride != 1)) copy_rows<S, kPass, kOff, false, false>(k_to0 + by, v_to0 + by, k, v, step, 0, 0, 0);
                else copy_rows<S, kPass, kOff, true, false>(k_to0 + by, v_to0 + by, k, v, 0, 0, 0, 0);
            }
            if constexpr (kQuant) {
                const uint32_t piece = (uint32_t)l_page[ki] * a.page_pieces + in_page * a.row_pieces + l_scales;
                const uint8_t *ks = reinterpret_cast<const uint8_t *>(a.c.k_sm) + (uint64_t)piece * kBytes, *vs = reinterpret_cast<const uint8_t *>(a.c.v_sm) + (uint64_t)piece * kBytes;
                each<kScalePasses>([&](auto i) {
                    constexpr int kTo = (ki * 16 + decltype(i)::value * kScalePass) * NG * 4;
                    if (kScalePass * kPieces == 32 || s_row < kScalePass) {
                        const int r = l_run0 + 16 * ki + decltype(i)::value * kScalePass + s_row, n = !edge || (r >= l_lo && r < l_len) ? kBytes : 0;
                        copy_async<kBytes, kTo>(s_to0 + by, ks, n), copy_async<kBytes, kTo + S::kScales>(s_to0 + by, vs, n);
                    }
                    ks += (uint64_t)a.row_pieces * (kScalePass * kBytes), vs += (uint64_t)a.row_pieces * (kScalePass * kBytes);
                });
            }
        });
    };
    // A segment's queries and what there is to know of it: the whole CTA's, into a ring of as many places as there are stages.
    auto load_segment = [&](int at) {
        const Sequence q = cur.s;
        const int slot = cur.segment % kStages, rows0 = cur.row_tile * R, head = cur.head;
        uint8_t *const qs = q_ring + slot * S::kQ;
#pragma unroll 1
        for (int i = tid; i < R * (D / 8); i += kThreads) {
            const int r = i / (D / 8), c = i % (D / 8), row = rows0 + r, tok = row / a.group;
            const bool there = tok < q.n;
            const int64_t off = there ? (q.q0 + tok) * a.q_ld + (int64_t)(head * a.group + row - tok * a.group) * D + c * 8 : 0;
            copy_async<16>(smem_of(qs + chunk_at<D / 8>(r, c) * 16), a.q + off, there ? 16 : 0);
        }
        if (tid == 0) segments[slot] = Segment{q.q0, q.n, q.len, q.p0, q.lo, q.tile0, q.tiles, head, rows0, at, (int)q.bad};
    };

    const int first_at = (int)(in % cur.s.tiles);
    at_segment(first_at);
    find_pages();
#pragma unroll 1
    for (int s = 0; s < kStages - 1; ++s) {
        if (s < units) {
            if (l_new) load_segment(s == 0 ? first_at : 0);
            load(s);
            if (s + 1 < units) {
                advance();
                find_pages();
            }
        }
        commit_async();
    }

    // ---- sums ----
    // Keys are the rows of the score product (A), queries its columns (B): an accumulator holds keys g and g + 8 of queries 2 t and 2 t + 1.  Of the
    // second product V's columns are the rows, its accumulators hold the same two queries, and the weights get from the first one's layout to the
    // second operand's by a transposition in registers.
    const int g = lane >> 2, t4 = lane & 3;
    // Places in a run's tiles: a lane's first, of which the others differ by the exclusive or with a chunk's number and by a constant.
    const int a_row = lane & 15, a_half = lane >> 4;  // of a fragment of sixteen rows, two chunks
    const uint32_t k_at0 = BITS == 16 ? k_chunk_at<S>(a_row, a_half) * 16 : BITS == 8 ? k_chunk_at<S>(g, t4 >> 1) * 16 + (t4 & 1) * 8 : k_chunk_at<S>(g, 0) * 16 + t4 * 4;
    const uint32_t v_at0 = S::kRows + (BITS == 16 ? chunk_at<CR>((lane & 7) + 8 * (lane >> 4), (lane >> 3) & 1) : chunk_at<CR>(a_row, BITS == 8 ? a_half : 0)) * 16;
    const uint32_t q_at0 = chunk_at<D / 8>((lane & 7), lane >> 3) * 16;
    uint32_t qf[S::kHoldQ ? NT : 1][S::kHoldQ ? D / 16 : 1][2];
    float o[D / 16][NT][4], w_sum[NT][4], o_min[kGroups][NT][2];
    float m[NT][2], l[NT][2];
    uint32_t v_low = kLowestScale;
    int at = 0, tiles = 0, whole0 = 0, whole1 = 0, segment = 0, stage = 0;
    bool fresh = true;
    auto take_out = [&]() {  // what the codes' offsets have added to the sums of their products
        if constexpr (kQuant) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int grp = 0; grp < NG; ++grp) {
                    const float sum[2] = {__shfl_sync(0xffffffffu, w_sum[nt][0], grp * 4 + t4), __shfl_sync(0xffffffffu, w_sum[nt][1], grp * 4 + t4)};
#pragma unroll
                    for (int d = grp * S::G / 16; d < (grp + 1) * S::G / 16; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[d][nt][e] = fmaf(e < 2 ? -S::kOffset : -S::kOffsetOdd, sum[e & 1], o[d][nt][e]);
                }
                w_sum[nt][0] = w_sum[nt][1] = 0.f;
            }
        }
    };

#pragma unroll 1
    for (int i = 0; i < units; ++i) {
        wait_async<kStages - 2>();
        __syncwarp();
        if (i + kStages - 1 < units) {
            if (SXB_RARE(l_new)) load_segment(0);
            load(stage == 0 ? kStages - 1 : stage - 1);
            if (i + kStages < units) {
                advance();
                find_pages();
            }
        }
        commit_async();

        const uint32_t st = smem0 + stage * S::kStage + warp * S::kPart;
        uint8_t *const qs = q_ring + (segment % kStages) * S::kQ;
        const Segment &sg = segments[segment % kStages];
        if (SXB_RARE(fresh)) {
            fresh = false;
            __syncthreads();
            at = sg.at, tiles = sg.tiles, v_low = kLowestScale;
            {   // tiles that every row sees all of
                const int p_last = sg.p0 + sg.n - 1, from = a.window > 0 ? max(0, p_last - a.window + 1) : 0;
                whole0 = (from + TK - 1) / TK - sg.tile0, whole1 = (sg.p0 + 1 + TK) / TK - 1 - sg.tile0;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                m[nt][0] = m[nt][1] = kLowest, l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) o[d][nt][0] = o[d][nt][1] = o[d][nt][2] = o[d][nt][3] = 0.f;
#pragma unroll
                for (int e = 0; e < kGroups; ++e) o_min[e][nt][0] = o_min[e][nt][1] = 0.f;
                w_sum[nt][0] = w_sum[nt][1] = w_sum[nt][2] = w_sum[nt][3] = 0.f;
            }
            if constexpr (kQuant) {
                // q to F16 times a power of two, elements in the order that the codes come in, and each group's sum of what they then are
                constexpr int kPer = kThreads / R < 32 ? kThreads / R : 32, kBlocks = D / 32;  // threads of a row; runs of 32 elements
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
                if (part == 0) q_factor[r] = fmaxf(a.scale * kLog2e * __uint_as_float((uint32_t)(127 - up) << 23), 1.2e-38f);  // not 0: it stands beside -inf
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
                    if (blk < kBlocks && blk % kRuns == 0) q_sums[blk / kRuns * R + r] = sums[b], q_extra[blk / kRuns * R + r] = -S::kOffsetK * sums[b];
                }
                __syncthreads();
            }
            if constexpr (S::kHoldQ) {
                each<NT>([&](auto nt) {
                    each<D / 32>([&](auto k2) {
                        constexpr int t = decltype(nt)::value, ks = 2 * decltype(k2)::value;
                        uint32_t r[4];
                        load_matrices<t * 8 * D * 2>(r, (smem_of(qs) + q_at0) ^ (ks * 32));
                        qf[t][ks][0] = r[0], qf[t][ks][1] = r[1], qf[t][ks + 1][0] = r[2], qf[t][ks + 1][1] = r[3];
                    });
                });
            }
        }
        const bool whole = at >= whole0 && at < whole1;
        const int run0 = (sg.tile0 + at) * TK + warp * RUN;
        if (whole || (run0 < sg.len && run0 + RUN > sg.lo)) {
        // q's fragments of two steps of sixteen elements, from step 2 K2
        auto q_at = [&](auto nt, auto k2, uint32_t (&r)[4]) {
            constexpr int t = decltype(nt)::value, ks = 2 * decltype(k2)::value;
            if constexpr (S::kHoldQ) r[0] = qf[t][ks][0], r[1] = qf[t][ks][1], r[2] = qf[t][ks + 1][0], r[3] = qf[t][ks + 1][1];
            else load_matrices<t * 8 * D * 2>(r, (smem_of(qs) + q_at0) ^ (ks * 32));
        };

        // scores
        float s[KI][NT][4];
        const uint32_t k_at = st + k_at0, s_at = st + 2 * S::kRows + g * (NG * 4);
        each<KI>([&](auto kic) {
            constexpr int ki = decltype(kic)::value, kRun = ki * 16 * S::RB;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[ki][nt][0] = s[ki][nt][1] = s[ki][nt][2] = s[ki][nt][3] = 0.f;
            if constexpr (!kQuant) {
                each<D / 32>([&](auto k2) {
                    constexpr int ks = 2 * decltype(k2)::value;
                    uint32_t k0[4], k1[4];
                    load_matrices<kRun>(k0, k_at ^ (ks * 32)), load_matrices<kRun>(k1, k_at ^ (ks * 32 + 32));
                    each<NT>([&](auto nt) {
                        uint32_t q[4];
                        q_at(nt, k2, q);
                        mma<false>(s[ki][decltype(nt)::value], k0, q[0], q[1]);
                        mma<false>(s[ki][decltype(nt)::value], k1, q[2], q[3]);
                    });
                });
            } else {
                uint32_t words[2][NG];
                load_shared<ki * 16 * NG * 4>(words[0], s_at), load_shared<(ki * 16 + 8) * NG * 4>(words[1], s_at);
                each<NG>([&](auto grpc) {
                    constexpr int grp = decltype(grpc)::value;
                    float part[NT][4];
                    float2 q_sum[NT];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        q_sum[nt] = *reinterpret_cast<const float2 *>(q_sums + grp * R + nt * 8 + 2 * t4);
                        const float2 extra = *reinterpret_cast<const float2 *>(q_extra + grp * R + nt * 8 + 2 * t4);
                        part[nt][0] = part[nt][2] = extra.x, part[nt][1] = part[nt][3] = extra.y;
                    }
                    each<S::G / 32>([&](auto run) {
                        constexpr int blk = grp * (S::G / 32) + decltype(run)::value;
                        uint32_t k0[4], k1[4];
                        if constexpr (BITS == 8) {
                            uint32_t w0[2], w1[2];
                            load_shared<kRun>(w0, k_at ^ (blk * 32)), load_shared<kRun + 8 * S::RB>(w1, k_at ^ (blk * 32));
                            k0[0] = bytes_f16(w0[0], 0x4140), k0[1] = bytes_f16(w1[0], 0x4140), k0[2] = bytes_f16(w0[0], 0x4342), k0[3] = bytes_f16(w1[0], 0x4342);
                            k1[0] = bytes_f16(w0[1], 0x4140), k1[1] = bytes_f16(w1[1], 0x4140), k1[2] = bytes_f16(w0[1], 0x4342), k1[3] = bytes_f16(w1[1], 0x4342);
                        } else {
                            uint32_t w0[1], w1[1];
                            load_shared<kRun>(w0, k_at ^ (blk * 16)), load_shared<kRun + 8 * S::RB>(w1, k_at ^ (blk * 16));
                            k0[0] = next_nibbles_f16(w0[0] << 4), k0[1] = next_nibbles_f16(w1[0] << 4), k0[2] = next_nibbles_f16(w0[0]), k0[3] = next_nibbles_f16(w1[0]);
                            k1[0] = next_nibbles_f16(w0[0] >> 4), k1[1] = next_nibbles_f16(w1[0] >> 4), k1[2] = next_nibbles_f16(w0[0] >> 8), k1[3] = next_nibbles_f16(w1[0] >> 8);
                        }
                        each<NT>([&](auto nt) {
                            uint32_t q[4];
                            q_at(nt, std::integral_constant<int, blk>{}, q);
                            mma<true>(part[decltype(nt)::value], k0, q[0], q[1]);
                            mma<true>(part[decltype(nt)::value], k1, q[2], q[3]);
                        });
                    });
                    float sc[2], mn[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        sc[e] = __uint_as_float(words[e][grp] << 16);
                        mn[e] = __uint_as_float(words[e][grp] & 0xffff0000u);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[ki][nt][e] = fmaf(sc[e >> 1], part[nt][e], fmaf(mn[e >> 1], e & 1 ? q_sum[nt].y : q_sum[nt].x, s[ki][nt][e]));
                });
            }
        });
        // a score in powers of two is s * fac
        float fac[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            fac[nt][0] = fac[nt][1] = a.scale * kLog2e;
            if constexpr (kQuant) {
                const float2 f = *reinterpret_cast<const float2 *>(q_factor + nt * 8 + 2 * t4);
                fac[nt][0] = f.x, fac[nt][1] = f.y;
            }
        }
        if (SXB_RARE(a.softcap > 0.f)) {
            const float by = 2.f / a.softcap, to = a.softcap * kLog2e;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int ki = 0; ki < KI; ++ki)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[ki][nt][e] = capped(s[ki][nt][e], fac[nt][e & 1], by, to);
                fac[nt][0] = fac[nt][1] = 1.f;
            }
        }
        uint32_t hidden = 0;  // bit (ki * NT + nt) * 4 + e: that query does not see that key
        if (SXB_RARE(!whole)) {
            const int j0 = run0 + g;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int tok = (sg.rows0 + nt * 8 + 2 * t4 + e) / a.group;
                    const int hi = tok < sg.n ? sg.p0 + tok : -1, lo = a.window > 0 ? (int)max((int64_t)-1, (int64_t)hi - a.window) : -1;
#pragma unroll
                    for (int ki = 0; ki < KI; ++ki)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int j = j0 + ki * 16 + 8 * x;
                            if (j > hi || j <= lo) {
                                s[ki][nt][2 * x + e] = -CUDART_INF_F;
                                hidden |= 1u << ((ki * NT + nt) * 4 + 2 * x + e);
                            }
                        }
                }
        }
        // The maximum that the weights are relative to is moved when a score passes it by 2^kSlack only: most tiles then need no exchange between lanes and
        // no sum is touched.  The scale that the weights of quantized values are relative to, likewise.
        float past = 0.f, top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float v = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
                for (int ki = 1; ki < KI; ++ki) v = fmaxf(v, fmaxf(s[ki][nt][e], s[ki][nt][2 + e]));
                top[nt][e] = v;
                past = fmaxf(past, fmaf(v, fac[nt][e], -m[nt][e]));
            }
        bool move = past > kSlack;
        if (SXB_RARE(__any_sync(0xffffffffu, move))) {
            float f[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float v = top[nt][e];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
                    const float now = fmaxf(m[nt][e], v * fac[nt][e]);
                    f[nt][e] = exp2_flushed(m[nt][e] - now);
                    m[nt][e] = now, l[nt][e] *= f[nt][e];
#pragma unroll
                    for (int grp = 0; grp < kGroups; ++grp) o_min[grp][nt][e] *= f[nt][e];
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int d = 0; d < D / 16; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d][nt][e] *= f[nt][e & 1];
                w_sum[nt][0] *= f[nt][0], w_sum[nt][1] *= f[nt][1];
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int ki = 0; ki < KI; ++ki)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[ki][nt][e] = exp2_flushed(fmaf(s[ki][nt][e], fac[nt][e & 1], -m[nt][e & 1]));
                    l[nt][e & 1] += s[ki][nt][e];
                }

        // weights times values
        const uint32_t v_at = st + v_at0;
        if constexpr (!kQuant) {
            // Keys that one row sees and another does not: an infinity or a NaN there must not reach the other through 0 * v.
            bool clean = true;
            if (SXB_RARE(!whole && sg.n > 1)) {
                const uint8_t *const vt = smem + stage * S::kStage + warp * S::kPart + S::kRows;
                for (int c = lane; c < RUN * CR; c += 32) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(vt + c * 16);
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) clean = clean && (ws[e] & 0x7f80u) != 0x7f80u && (ws[e] & 0x7f800000u) != 0x7f800000u;
                }
                clean = __all_sync(0xffffffffu, clean);
            }
            if (__builtin_expect(clean, 1)) {
                each<KI>([&](auto kic) {
                    constexpr int ki = decltype(kic)::value, kRun = ki * 16 * S::RB;
                    uint32_t p[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        p[nt][0] = transposed(pack_bf16(s[ki][nt][0], s[ki][nt][1]));
                        p[nt][1] = transposed(pack_bf16(s[ki][nt][2], s[ki][nt][3]));
                    }
                    each<D / 16>([&](auto d) {  // columns 0 - 7 and 8 - 15 of keys 0 - 7, then of keys 8 - 15
                        uint32_t v[4];
                        load_matrices_trans<kRun>(v, v_at ^ (decltype(d)::value * 32));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma<false>(o[decltype(d)::value][nt], v, p[nt][0], p[nt][1]);
                    });
                });
            } else {
                const uint8_t *const vt = smem + stage * S::kStage + warp * S::kPart + S::kRows;
#pragma unroll
                for (int ki = 0; ki < KI; ++ki)
#pragma unroll 1
                    for (int k = 0; k < 16; ++k) {
                        const int from = (k % 8) * 4 + t4;
                        const uint32_t out_of_sight = __shfl_sync(0xffffffffu, hidden, from) >> (ki * NT * 4 + (k < 8 ? 0 : 2));
                        float w[NT][2];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float low = __shfl_sync(0xffffffffu, s[ki][nt][e], from), high = __shfl_sync(0xffffffffu, s[ki][nt][2 + e], from);
                                w[nt][e] = k < 8 ? low : high;
                            }
#pragma unroll
                        for (int d = 0; d < D / 16; ++d) {
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const float v = bf16_bits_to_f32(*reinterpret_cast<const uint16_t *>(vt + chunk_at<CR>(ki * 16 + k, 2 * d + half) * 16 + g * 2));
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                        if ((out_of_sight >> (nt * 4 + e) & 1) == 0) o[d][nt][2 * half + e] = fmaf(w[nt][e], v, o[d][nt][2 * half + e]);
                            }
                        }
                    }
            }
        } else {
            float v_up = scale_up(v_low);
            each<KI>([&](auto kic) {
                constexpr int ki = decltype(kic)::value, kRun = ki * 16 * S::RB;
                uint32_t words[2][kGroups];
                value_words<S, ki>(words, s_at);
                // A power of two keeps the products of scales and weights inside F16; the largest scale so far sets it.  As bit patterns, less that of the lowest that goes with it,
                // what is larger, lower, an infinity, a NaN or negative is above what goes; a zero too, which changes nothing.
                uint32_t over = 0;
                bool odd = false;  // a scale or a min among them is none, and there are rows that must not hear of it
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int grp = 0; grp < NG; ++grp) over = max(over, (words[e][grp] << 16) - v_low);
                if (SXB_RARE(!whole)) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int grp = 0; grp < NG; ++grp) odd = odd || none_of(words[e][grp]);
                }
                if (SXB_RARE(__any_sync(0xffffffffu, odd || over >= (kSpread + 1) << 23))) {
                    uint32_t most = 0, least = 0xffffffffu;  // of finite scales' sizes; of all but zeros
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int grp = 0; grp < NG; ++grp) {
                            const uint32_t t = words[e][grp] << 16, size = t & 0x7f800000u;
                            if (size != 0x7f800000u) most = max(most, size);  // a scale that is none says nothing of the others
                            odd = odd || t > 0x7f7fffffu;
                            least = min(least, t - 1);
                        }
                    most = __reduce_max_sync(0xffffffffu, most);
                    if (most > v_low + (kSpread << 23)) {
                        const float down = exp2_flushed((float)((int)(v_low + (kSpread << 23) - most) >> 23));
                        v_low = most - (kSpread << 23), v_up = scale_up(v_low);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[d][nt][e] *= down;
                            w_sum[nt][0] *= down, w_sum[nt][1] *= down;
                        }
                    }
                    odd = odd || least < v_low;
                    // The matrix product would carry what is none to other columns (0 * NaN in the sums of weights) and other rows, and lose small values' weights.
                    if (__any_sync(0xffffffffu, odd)) {
                        add_values<S, ki>(smem + stage * S::kStage + warp * S::kPart + S::kRows, words, s[ki], hidden >> (ki * NT * 4), v_up, lane, o, o_min);
                        return;
                    }
                }
                float scales[2][kGroups];
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int grp = 0; grp < NG; ++grp) scales[e][grp] = __uint_as_float(words[e][grp] << 16) * v_up;
                each<NG>([&](auto grpc) {
                    constexpr int grp = decltype(grpc)::value;
                    float mn[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) mn[e] = __uint_as_float(words[e][grp] & 0xffff0000u);
                    uint32_t p[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            w[e] = s[ki][nt][e] * scales[e >> 1][grp];
                            o_min[grp][nt][e & 1] = fmaf(s[ki][nt][e], mn[e >> 1], o_min[grp][nt][e & 1]);
                        }
                        p[nt][0] = transposed(pack_f16(w[0], w[1])), p[nt][1] = transposed(pack_f16(w[2], w[3]));
                        const uint32_t one = g == grp ? 0x3c003c00u : 0u, ones[4] = {one, 0, one, 0};  // row grp of the sums
                        mma<true>(w_sum[nt], ones, p[nt][0], p[nt][1]);
                    }
                    each<S::G / 32>([&](auto runc) {
                        constexpr int run = decltype(runc)::value;
                        if constexpr (BITS == 8) {  // two chunks of sixteen columns, the even ones rows 0 - 7 of a fragment, the odd ones rows 8 - 15
                            constexpr int c = grp * (S::G / 16) + run * 2;
                            uint32_t v[4];
                            load_matrices_trans<kRun>(v, v_at ^ (c * 16));
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const uint32_t va[4] = {bytes_f16(v[2 * x], 0x4240), bytes_f16(v[2 * x], 0x4341), bytes_f16(v[2 * x + 1], 0x4240), bytes_f16(v[2 * x + 1], 0x4341)};
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) mma<true>(o[c + x][nt], va, p[nt][0], p[nt][1]);
                            }
                        } else {  // a chunk of 32 columns: 4 n and 4 n + 1 in the first fragment, 4 n + 2 and 4 n + 3 in the second
                            constexpr int c = grp * (S::G / 32) + run;
                            uint32_t v[2];
                            load_matrices_trans<kRun>(v, v_at ^ (c * 16));
                            const uint32_t va[4] = {low_nibbles_f16(v[0]), next_nibbles_f16(v[0]), low_nibbles_f16(v[1]), next_nibbles_f16(v[1])};
                            const uint32_t u0 = v[0] >> 8, u1 = v[1] >> 8;
                            const uint32_t vb[4] = {low_nibbles_f16(u0), next_nibbles_f16(u0), low_nibbles_f16(u1), next_nibbles_f16(u1)};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma<true>(o[2 * c][nt], va, p[nt][0], p[nt][1]), mma<true>(o[2 * c + 1][nt], vb, p[nt][0], p[nt][1]);
                        }
                    });
                });
            });
        }
        }
        // the accumulators' steps cut their last bit off, of sums that the offset makes 4 (8 bits) to 140 times as large: it goes before that adds up
        if constexpr (kQuant) {
            if (SXB_RARE((at & 15) == 15 || at + 1 == tiles || i + 1 == units)) take_out();
        }
        uint8_t *const stage_base = smem + stage * S::kStage;
        stage = stage + 1 == kStages ? 0 : stage + 1;
        if (__builtin_expect(++at < tiles && i + 1 < units, 1)) continue;

        // ---- the segment's end, or this CTA's share's: the warps' sums become one ----
        const int64_t u0 = list[0], u1 = list[1], total = list[2], ctas = list[3];
        const int64_t seg0 = u0 + (i + 1) - at, seg1 = seg0 + tiles;  // the segment's units in the list
        const bool split = seg0 < u0 || seg1 > u1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
                const int r = warp * R + nt * 8 + 2 * t4 + e;
                if (g == 0) row_max[r] = m[nt][e], row_sum[r] = l[nt][e];
            }
        if constexpr (kQuant) {
            const float down = __uint_as_float(2 * (127u << 23) - __float_as_uint(scale_up(v_low)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int grp = 0; grp < NG; ++grp)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) o_min[grp][nt][e] += __shfl_xor_sync(0xffffffffu, o_min[grp][nt][e], off);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int d = 0; d < D / 16; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d][nt][e] = fmaf(o[d][nt][e], down, o_min[d * 16 / S::G][nt][e & 1]);
        }
        __syncthreads();
        // what each group's sums of a row count for, the row's maximum and its sum of weights
        if (tid < R) {
            float top = row_max[tid], sum = 0.f;
#pragma unroll
            for (int k = 1; k < WK; ++k) top = fmaxf(top, row_max[k * R + tid]);
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                const float f = exp2_flushed(row_max[k * R + tid] - top);
                row_max[k * R + tid] = f, sum = fmaf(row_sum[k * R + tid], f, sum);
            }
            row_top[tid] = top, row_sum[tid] = sum;
        }
        __syncthreads();
        float mine_f[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float2 f = *reinterpret_cast<const float2 *>(row_max + warp * R + nt * 8 + 2 * t4);
            mine_f[nt][0] = f.x, mine_f[nt][1] = f.y;
        }
        constexpr int DC = S::DC;
        auto *const joint = reinterpret_cast<float *>(S::kOwnJoint ? own_joint : stage_base);  // [WK][R][DC], runs of eight columns turned by the row
        float *const part = a.partial + (2 * (int64_t)blockIdx.x + (seg0 < u0 ? 0 : 1)) * R * (D + 2);
        const int rows = min(R, sg.n * a.group - sg.rows0);
#pragma unroll
        for (int col0 = 0; col0 < D; col0 += DC) {
            if (col0 > 0) __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = nt * 8 + 2 * t4 + e;
                    float *const to = joint + (warp * R + r) * DC;
                    const float f = mine_f[nt][e];
#pragma unroll
                    for (int d = col0 / 16; d < (col0 + DC) / 16; ++d) {
                        if constexpr (BITS == 16) {
                            to[(16 * d - col0 + g) ^ (t4 << 3)] = o[d][nt][e] * f;
                            to[(16 * d - col0 + g + 8) ^ (t4 << 3)] = o[d][nt][2 + e] * f;
                        } else if constexpr (BITS == 8) {
                            *reinterpret_cast<float2 *>(to + ((16 * d - col0 + 2 * g) ^ (t4 << 3))) = make_float2(o[d][nt][e] * f, o[d][nt][2 + e] * f);
                        } else if (d % 2 == 0) {
                            *reinterpret_cast<float4 *>(to + ((16 * d - col0 + 4 * g) ^ (t4 << 3))) =
                                make_float4(o[d][nt][e] * f, o[d][nt][2 + e] * f, o[d + 1][nt][e] * f, o[d + 1][nt][2 + e] * f);
                        }
                    }
                }
            __syncthreads();
            for (int x = tid; x < rows * (DC / 4); x += kThreads) {
                const int r = x / (DC / 4), c4 = x % (DC / 4);
                const float *const from = joint + r * DC + ((4 * c4) ^ ((r >> 1 & 3) << 3));
                float4 v = *reinterpret_cast<const float4 *>(from);
                const float top_r = row_top[r], sum_r = row_sum[r];
#pragma unroll
                for (int k = 1; k < WK; ++k) {
                    const float4 w = *reinterpret_cast<const float4 *>(from + k * R * DC);
                    v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
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
            if constexpr (!S::kJoinHere) {
                if (tid == 0 && seg0 >= u0) a.joins[blockIdx.x] = Join{sg.q0, sg.rows0, sg.head, rows, (int)(c1 - c0) + 1, {}};
            } else {
                auto *const last = reinterpret_cast<int *>(scan + kWarps);
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
                    const Parts<R, D> from(a.partial, (int)c0, (int)(c1 - c0) + 1);
                    for (int x = tid; x < rows * (D / 4); x += kThreads) join_run<8>(a, from, sg.q0, sg.rows0, sg.head, x / (D / 4), x % (D / 4));
                }
            }
        }
        __syncthreads();  // the joint's place is the next loads'
        fresh = true, ++segment;
    }
}

#include "attn_decode_tc.cuh"

// The rows of a tile for those that a key head's queries make: more query heads a key head or more drafts, more rows, until registers end; what is
// above takes several tiles, and reads the keys for each.  Quantized keys' conversions are most of the work, and sixteen rows leave registers for two runs
// side by side: eight conversations of one to eight rows of eight heads, 39 us with sixteen, 48 with 32; BF16, four rows of eight heads, 200 with sixteen,
// 109 with 32.  (Tiles of 32 and 64 rows whose warps share out V's columns, the weights by way of shared memory, are slower everywhere: the first
// of these 54 to 58.)
constexpr int most_rows(int D, int bits) { return bits == 16 && D <= 128 ? 32 : 16; }
inline int tile_rows(int D, int bits, int64_t rows) { return rows <= 8 ? 8 : rows <= 16 || most_rows(D, bits) == 16 ? 16 : 32; }
// Tiles of 128 rows on tcgen05 (attn_decode_tc.cuh): more than 32 rows, and enough tiles that a table has room for, so that its start - tensor memory, a stage
// to fill before the first product - is no matter.  Rows, sequences x keys, us with tiles of 32 and with it: 64, 64 x up to 8000, 191 and 136; 2 x up to 33000, 52
// and 44; 8 x up to 9000, 35 and 35; 16 x 1000, 25 and 27; 1 x 300, 11 and 14; 128, 64 x up to 8000, 460 and 176; 16 x 1000, 35 and 36.  Chunks of 512 tokens of eight
// heads a key head on 4096 keys, 170 and 60, of 2048 on 8192, 1338 and 290.  The lengths are the device's to know; a host whose tables have room for far longer
// sequences than there are pays those 3 us, and gets by passing fewer columns what shorter tables give (the bits too: the forms add in other orders).
constexpr bool has_tc(int D, int bits) { return D == TcShape::D && bits == TcShape::BITS; }
inline bool takes_tc(int D, int bits, int64_t rows, int64_t B, int64_t n_kv, int64_t capacity) {
    if (!has_tc(D, bits) || rows <= most_rows(D, bits)) return false;
    return rows > TcShape::R || (double)B * (double)n_kv * (double)((capacity + TcShape::TK - 1) / TcShape::TK) >= 8.0 * sm_count();
}

// The counters' place is every form's: calls of different ones share a workspace.
inline size_t counter_bytes() { return ((size_t)sm_count() * kMostPerSm * (sizeof(uint32_t) + sizeof(Join)) + 255) / 256 * 256; }

template <class S> struct Kernel { static constexpr auto fn = attn_decode_kernel<S>; };
template <> struct Kernel<TcShape> { static constexpr auto fn = attn_tc_kernel<TcShape>; };

template <class S> struct Launch {
    static_assert(S::kPerSm <= kMostPerSm, "");

    static int64_t ctas() { return (int64_t)sm_count() * S::kPerSm; }
    static size_t bytes() { return counter_bytes() + (size_t)(ctas() * 2 * S::R * (S::D + 2) * 4); }
    static cudaError_t run(Args a, void *ws, int64_t most_units, int told_rows, const CUtensorMap *maps, cudaStream_t st) {
        const int64_t n = std::max<int64_t>(1, std::min(ctas(), most_units));
        a.count = static_cast<uint32_t *>(ws);
        a.joins = reinterpret_cast<Join *>(a.count + (size_t)sm_count() * kMostPerSm);
        a.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + counter_bytes());
        static std::atomic<uint64_t> told{0};  // devices that know of the kernel's shared memory, a bit each
        int dev = 0;
        if (const cudaError_t rc = cudaGetDevice(&dev); rc != cudaSuccess) return rc;
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if ((told.load(std::memory_order_acquire) & bit) == 0) {
            if (const cudaError_t rc = cudaFuncSetAttribute(Kernel<S>::fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem); rc != cudaSuccess) return rc;
            // (an SM's shared memory stays as the form wants it: it need not be empty for the next call's CTAs)
            if (const cudaError_t rc = cudaFuncSetAttribute(attn_join_kernel<S>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared); rc != cudaSuccess) return rc;
            told.fetch_or(bit, std::memory_order_release);
        }
        cudaError_t rc2;
        if constexpr (std::is_same_v<S, TcShape>) rc2 = launch_behind(Kernel<S>::fn, dim3((unsigned)n), dim3(S::kThreads), (size_t)S::kSmem, st, 1, a, maps[0], maps[1]);
        else rc2 = launch_behind(Kernel<S>::fn, dim3((unsigned)n), dim3(S::kThreads), (size_t)S::kSmem, st, 1, a);
        if (S::kJoinHere || rc2 != cudaSuccess) return rc2;
        return launch_behind(attn_join_kernel<S>, dim3((unsigned)n, (unsigned)((told_rows + kJoinRows - 1) / kJoinRows)), dim3(kJoinRows * S::D / 4), 0, st, 1, a);
    }
};

// f(Shape) for the sizes of a call.
template <int D, int BITS, int G, class F> auto with_rows(int rows, F f) {
    if (rows == 8) return f(Shape<D, BITS, G, 8>{});
    if constexpr (has_tc(D, BITS))
        if (rows == 128) return f(TcShape{});
    if constexpr (most_rows(D, BITS) == 32)
        if (rows == 32) return f(Shape<D, BITS, G, 32>{});
    return f(Shape<D, BITS, G, 16>{});
}
template <int D, class F> auto with_cache(int bits, int64_t G, int rows, F f) {
    if (bits == 16) return with_rows<D, 16, D>(rows, f);
    if (bits == 8) {
        if (G == 32) return with_rows<D, 8, 32>(rows, f);
        if (G == 64) return with_rows<D, 8, 64>(rows, f);
        return with_rows<D, 8, D < 128 ? D : 128>(rows, f);
    }
    if (G == 32) return with_rows<D, 4, 32>(rows, f);
    if (G == 64) return with_rows<D, 4, 64>(rows, f);
    return with_rows<D, 4, D < 128 ? D : 128>(rows, f);
}
template <class F> auto with_shape(int64_t D, int bits, int64_t G, int rows, F f) {
    if (D == 64) return with_cache<64>(bits, G, rows, f);
    if (D == 128) return with_cache<128>(bits, G, rows, f);
    return with_cache<256>(bits, G, rows, f);
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
    size_t most = 0;  // of a call with fewer rows too, and of any group size: how many CTAs an SM holds depends on both
    const int64_t told = max_q * (n_q / n_kv);
    for (int rows = 8; rows <= tile_rows((int)D, bits, told); rows *= 2)
        for (int G = 32; G <= D && G <= 128; G *= 2) most = std::max(most, with_shape(D, bits, G, rows, [](auto s) { return Launch<decltype(s)>::bytes(); }));
    if (has_tc((int)D, bits) && told > most_rows((int)D, bits)) most = std::max(most, Launch<TcShape>::bytes());
    return most;
}

extern "C" int sxb_attn_decode(const SxbAttnDecodeArgs *args, sxb_stream_t stream) {
    const char *fn = "attn_decode";
    SXB_CHECK(args != nullptr, fn, ": null argument block");
    const SxbKvCache *const cache = args->cache;
    const void *const q = args->q;
    void *const out = args->out, *const ws = args->ws;
    const int32_t *const pages = args->pages, *const q_start = args->q_start, *const kv_len = args->kv_len;
    const int64_t q_ld = args->q_ld, out_ld = args->out_ld, T = args->T, n_q = args->n_q, pages_ld = args->pages_ld, n_cols = args->n_cols, B = args->B;
    const int64_t max_q = args->max_q, window = args->window;
    const float scale = args->scale, softcap = args->softcap;
    uint32_t *const err = args->err;
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
    SXB_CHECK(scale > 0.f && scale < 1e30f, fn, ": scale must be finite and positive");
    SXB_CHECK(softcap == 0.f || (softcap >= 1e-6f && softcap < 1e30f), fn, ": softcap = ", softcap, ", expected 0 (none) or 1e-6 .. 1e30");
    SXB_CHECK(window >= 0 && window < (1ll << 31), fn, ": window = ", window, ", expected 0 (none) .. 2^31 - 1");
    const int64_t told = max_q * (n_q / n_kv);
    const bool tc = takes_tc((int)D, cache->bits, told, B, n_kv, n_cols * cache->page);
    const int rows = tc ? TcShape::R : tile_rows((int)D, cache->bits, told);
    const size_t need = sxb_attn_decode_workspace_bytes(n_q, n_kv, D, cache->bits, max_q);
    SXB_CHECK(args->ws_bytes >= need, fn, ": workspace of ", args->ws_bytes, " bytes, needs ", need);
    a.q = static_cast<const uint16_t *>(q), a.q_ld = q_ld, a.pages = pages, a.pages_ld = pages_ld, a.capacity = n_cols * cache->page;
    a.q_start = q_start, a.kv_len = kv_len, a.B = (int)B, a.T = (int)T, a.n_q = (int)n_q, a.group = (int)(n_q / n_kv), a.window = window >= a.capacity ? 0 : (int)window;
    a.scale = scale, a.softcap = softcap, a.out = static_cast<uint16_t *>(out), a.out_ld = out_ld, a.lse = args->lse, a.err = err;
    const uint32_t chunks = (uint32_t)(D * cache->bits / 8 / 16), words = cache->bits == 16 ? 0 : (uint32_t)(D / cache->G), pieces = words > 4 ? words / 4 : words ? 1 : 0;
    a.page_chunks = (uint32_t)cache->page_stride * chunks, a.head_chunks = (uint32_t)cache->head_stride * chunks, a.row_chunks = (uint32_t)cache->row_stride * chunks;
    a.page_pieces = (uint32_t)cache->page_stride * pieces, a.head_pieces = (uint32_t)cache->head_stride * pieces, a.row_pieces = (uint32_t)cache->row_stride * pieces;
    CUtensorMap maps[2];  // [page, head, token, column], boxes of 16 to 64 tokens of a page and 64 columns
    if (tc) {
        const uint64_t dims[4] = {(uint64_t)D, (uint64_t)cache->page, (uint64_t)n_kv, (uint64_t)cache->n_pages}, row = (uint64_t)D * 2;
        const uint64_t strides[3] = {(uint64_t)cache->row_stride * row, (uint64_t)cache->head_stride * row, (uint64_t)cache->page_stride * row};
        a.box_rows = (int)std::min<int64_t>(64, std::max<int64_t>(16, cache->page));
        const uint32_t box[4] = {64, (uint32_t)std::min<int64_t>(a.box_rows, cache->page), 1, 1};
        for (int x = 0; x < 2; ++x)
            if (int rc = tensor_map_4d(fn, x == 0 ? cache->k : cache->v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, &maps[x])) return rc;
        if (int rc = library_status_words(fn, &a.status)) return rc;
        a.wait_limit_ns = wait_limit_ns(), a.test_skip_slot = test_skip_slot();
    }
    auto st = static_cast<cudaStream_t>(stream);
    const cudaError_t rc = with_shape(D, cache->bits, cache->G, rows, [&](auto s) {
        using S = decltype(s);
        if (Launch<S>::bytes() > args->ws_bytes) return cudaErrorInvalidValue;  // nothing is written behind the workspace, whatever the sizes above say
        // no list is longer than every sequence at its table's end (in a product that cannot overflow: the grid is a few hundred CTAs)
        const double most = (double)((a.capacity + S::TK - 1) / S::TK) * (double)B * n_kv * (double)((T * a.group + S::R - 1) / S::R + 1);
        return Launch<S>::run(a, ws, (int64_t)std::min(most, 1e12), (int)std::min<int64_t>(S::R, told), maps, st);
    });
    if (rc != cudaSuccess) return fail_cuda(SXB_FILE_, __LINE__, __func__, rc, cat(fn, " launch"));
    SXB_CHECK_LAUNCH(fn, " T=", T, " B=", B, " n_q=", n_q, " n_kv=", n_kv, " D=", D, " bits=", cache->bits);
    return SXB_OK;
}
