// Verification of drafted tokens against the target's probabilities, from given random numbers (include/strix_b200.h has the rules).
//
// Two launches.  The first reads every row's logits once, a warp a chunk of 4 KB: its largest logit (and, for greedy sequences, the first token that has it) and the sum of 2^(c (x -
// max)), c = log2(e) / temperature.  A logit takes eight instructions, one of them the exponential, and issue slots, the special-function unit and memory all stand at 55 to 60 %.  The second,
// a CTA a sequence (a cluster of four or eight where the drafter gives its distribution), joins a row's chunks, tests the drafts, and draws the next token: from the chunks' sums it knows the chunk in which the random number
// falls and reads that one again; only a difference of two distributions takes the whole row of both, once more, shared by the cluster.  It is bound by its chain of loads, of which
// those that do not wait for the first launch are made ahead of its end.  Nothing is counted or left behind in the workspace: no atomics, and results do not depend on who comes first.
//
// 64 sequences of 1 to 8 rows of 131072 BF16 logits, the drafter's too (134 MB): 46 us, some 30 of them the first's (4.5 TB/s); 304 such rows in FP32 73 us (304 in BF16 48); 2 sequences of 8 rows of
// FP32 8.3 together, one row 6.3.  A CTA a chunk, its parts joined by barriers, took 108 us for the 64 sequences where a warp a chunk takes 52 (before the differences were read by batches).
//
// A border's error: a term takes c (x - max) in FP32 (2^-23 of the exponent, which is small where the term is large), one ex2 (2^-22), sums of up to sixteen
// terms and then seven more in FP32; chunks are joined in FP64, where the exponents are exact.  No finite logit is too large for either.

#include "skinny_mma.cuh"

#include <cooperative_groups.h>

namespace sxb {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kStatThreads = 128, kStatCtas = 4;       // of the first kernel; CTAs an SM
constexpr int kPieces = kThreads, kPerLane = kPieces / 32;  // of sixteen bytes, of a chunk: eight a lane of a warp, or one a thread of a CTA
constexpr int kMinRanks = 4, kMaxRanks = 8;            // CTAs that share a difference of two rows
constexpr int64_t kMaxV = 1 << 20, kMaxB = 8192;
constexpr int kMaxChunks = (int)(kMaxV / (4 * kPieces)) + 1, kMaxRun = (kMaxChunks + kMinRanks - 1) / kMinRanks;  // of a row; of a CTA's share of one
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994531;
// Of a sum of max(p - q, 0): that much may be rounding alone.  Probabilities are within 2^-19 of their size; where rows of the same numbers begin at different places in sixteen bytes or differ in
// type their chunks are not the same tokens, and their sums not the same bits.  A draft is refused with that chance at most, so what is drawn keeps its distribution to 2^-18.
constexpr double kNoDifference = 0x1p-18;

enum { kBadLogits = 1, kBadDraft = 2, kBadId = 3, kBadRandom = 4, kBadTemperature = 5, kBadRange = 6 };

struct ChunkStat {  // of 2^(c x) over a chunk
    double sum;     // relative to 2^(c best)
    float best;     // NaN: the chunk holds a NaN; +inf: an infinity
    int at;         // greedy sequences: the first token that has it
};

struct VerifyArgs {
    const void *logits, *draft;
    int64_t ld, draft_ld;
    const int32_t *ids, *q_start;
    const float *u, *u_pick, *temperature;
    int32_t *next_ids, *n_new;
    float *logp;
    ChunkStat *stats;  // [T (, T of the drafter)][pitch]
    uint32_t *err;
    int T, V, B, pitch;
    int ranks;  // CTAs of the second kernel that share a difference of two rows
};

// Tokens are read in pieces of sixteen aligned bytes.  A row may begin inside one: piece i holds the tokens i * VE - mis ..., those outside 0 .. V - 1 are none.
template <typename T>
struct Row {
    static constexpr int VE = 16 / (int)sizeof(T), kChunk = kPieces * VE;
    const T *p;
    int mis, V;
    __device__ inline Row(const void *base, int64_t ld, int64_t row, int n) : p(static_cast<const T *>(base) + row * ld), V(n) {
        mis = (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % VE);
    }
    __device__ inline int pieces() const { return (V + mis + VE - 1) / VE; }
    __device__ inline int chunks() const { return (V + mis + kChunk - 1) / kChunk; }
    __device__ inline int token(int piece) const { return piece * VE - mis; }
    __device__ inline float at(int t) const { return load_as_f32(p, t); }
    // A piece as it lies in memory, -inf where there are no tokens.
    __device__ inline uint4 raw(int piece) const {
        const int t0 = token(piece);
        return t0 >= 0 && t0 + VE <= V ? __ldg(reinterpret_cast<const uint4 *>(p + t0)) : edge(t0);
    }
    __device__ inline uint4 edge(int t0) const {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = t0 + i >= 0 && t0 + i < V ? __float_as_uint((float)p[t0 + i]) : 0xff800000u;
            else {
                const int t = t0 + 2 * i;
                w[i] = (t >= 0 && t < V ? (uint32_t)p[t] : 0xff80u) | ((t + 1 >= 0 && t + 1 < V ? (uint32_t)p[t + 1] : 0xff80u) << 16);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // The same as numbers.
    __device__ static inline void values(const uint4 &w, float (&v)[VE]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(u[i]);
            else v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
};

// The scale of a sequence's exponents; greedy sequences' log-probabilities are those of temperature 1.
__device__ inline float exponent_scale(float t) { return t == 0.f ? kLog2e : __fdiv_rn(kLog2e, t); }

// The first sequence that has the row, -1 if none has.  By a whole warp, 32 starts a step: nothing beside a row's logits for hundreds of sequences (512 of two rows of 4096: 53 us in all with a drafter's
// distribution), what bounds thousands over few tokens (8192 over 130: 260 us, with a drafter's distribution 721).
__device__ inline int sequence_of(const int32_t *q_start, int B, int row) {
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < B; b0 += 32) {
        const int b = b0 + lane;
        const bool mine = b < B && q_start[b] <= row && row < q_start[b + 1];
        const uint32_t found = __ballot_sync(0xffffffffu, mine);
        if (found) return b0 + __ffs(found) - 1;
    }
    return -1;
}

// 2^v on the special-function unit, nothing below 2^-126: with the smaller numbers that a weight this far down is not drawn by, it takes four instructions more.
__device__ inline float exp2_of(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ inline uint32_t max_nan_pair(uint32_t a, uint32_t b) {  // of two BF16
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ inline float warp_max_nan(float v) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// 2^(c (x - best)), of one and of two.  The difference is taken of halves, its factor twice c (finite: temperatures are 2^-126 at least): two logits may lie further apart than FP32 reaches and
// still both count, at temperatures as large as they are.  But for subnormal logits, whose last bit no exponent shows, halves round as the whole.
__device__ inline float weight_of(float x, float half_best, float twice_c) { return exp2_of(__fmul_rn(fmaf(x, 0.5f, -half_best), twice_c)); }
__device__ inline uint64_t weight_pair(float x0, float x1, uint64_t minus_half_best, uint64_t twice_c) {
    float e0, e1;
    unpair(mul_pair(fma_pair(pair(x0, x1), pair(0.5f, 0.5f), minus_half_best), twice_c), e0, e1);
    return pair(exp2_of(e0), exp2_of(e1));
}

// A lane's part of a chunk: piece 32 j + lane is its j-th.  Where the row does not begin or end with a piece, the tokens before the first and behind the last whole one are a lane's each.
struct Loaded {
    uint4 w[kPerLane];
    float head, tail;
};
template <typename T>
__device__ inline void load_chunk(const Row<T> &r, int chunk, Loaded &l) {
    constexpr int VE = Row<T>::VE;
    constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
    const int lane = threadIdx.x & 31, whole0 = r.mis != 0, whole1 = (r.V + r.mis) / VE, p0 = chunk * kPieces;  // the whole pieces are whole0 .. whole1 - 1
    const uint4 *const p = reinterpret_cast<const uint4 *>(r.p - r.mis);
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
        const int i = p0 + 32 * j + lane;
        l.w[j] = i >= whole0 && i < whole1 ? __ldg(p + i) : make_uint4(kNone, kNone, kNone, kNone);
    }
    l.head = l.tail = -INFINITY;
    if (p0 == 0 && whole0 && lane < min(VE - r.mis, r.V)) l.head = r.at(lane);
    const int tail = r.pieces() - 1;  // not whole, and not the head
    if (tail == whole1 && tail > 0 && tail >= p0 && tail < p0 + kPieces && lane < r.V - r.token(tail)) l.tail = r.at(r.token(tail) + lane);
    else if (tail == whole1 && tail == 0 && !whole0 && p0 == 0 && lane < r.V) l.tail = r.at(lane);
}

// A chunk's statistics, by a warp.
template <typename T>
__device__ inline ChunkStat chunk_stat(const Row<T> &r, int chunk, const Loaded &l, float c, bool greedy) {
    constexpr int VE = Row<T>::VE;
    const int lane = threadIdx.x & 31;
    const uint4(&w)[kPerLane] = l.w;
    float most = max_nan(l.head, l.tail);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < kPerLane; ++j)
            most = max_nan(most, max_nan(max_nan(__uint_as_float(w[j].x), __uint_as_float(w[j].y)), max_nan(__uint_as_float(w[j].z), __uint_as_float(w[j].w))));
    } else {
        uint32_t m = 0xff80ff80u;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) m = max_nan_pair(m, max_nan_pair(max_nan_pair(w[j].x, w[j].y), max_nan_pair(w[j].z, w[j].w)));
        most = max_nan(most, max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u)));
    }
    most = warp_max_nan(most);
    uint64_t sum[2] = {0, 0};
    int at = 0x7fffffff;
    if (most > -INFINITY && most < INFINITY) {
        const uint64_t minus = pair(-0.5f * most, -0.5f * most), cc = pair(2.f * c, 2.f * c);
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) {
            float v[VE];
            Row<T>::values(w[j], v);
#pragma unroll
            for (int i = 0; i < VE; i += 2) sum[i / 2 & 1] = add_pair(sum[i / 2 & 1], weight_pair(v[i], v[i + 1], minus, cc));
        }
        sum[0] = add_pair(sum[0], weight_pair(l.head, l.tail, minus, cc));
        if (greedy) {
            if (l.tail == most) at = r.token(r.pieces() - 1) + lane;
#pragma unroll
            for (int j = kPerLane - 1; j >= 0; --j) {
                float v[VE];
                Row<T>::values(w[j], v);
                const int t0 = r.token(chunk * kPieces + j * 32 + lane);
#pragma unroll
                for (int i = VE - 1; i >= 0; --i)
                    if (v[i] == most) at = t0 + i;
            }
            if (l.head == most) at = lane;
            at = __reduce_min_sync(0xffffffffu, at);
        }
    }
    float s, odd;
    unpair(add_pair(sum[0], sum[1]), s, odd);
    s += odd;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    return ChunkStat{(double)s, most, at};
}

// The warps' chunks: an equal run of all rows' each, the next chunk asked for ahead of the work on one.  What a row's sequence says is looked up behind its first chunk's loads, but ahead of
// the drafter's: a sequence's last row has no draft behind it, a greedy one's drafter is not asked, and those are not read.
template <typename T, bool DRAFTER>
__device__ inline void stats_run(const VerifyArgs &a, const void *base, int64_t ld, ChunkStat *out, int block, int blocks) {
    const int lane = threadIdx.x & 31, n = (a.V + Row<T>::VE - 1 + Row<T>::kChunk - 1) / Row<T>::kChunk;  // of a row that begins at a piece's last token
    const int64_t units = (int64_t)a.T * n, warps = (int64_t)blocks * (kStatThreads / 32), w = (int64_t)block * (kStatThreads / 32) + (threadIdx.x >> 5);
    const int64_t lo = units * w / warps, hi = units * (w + 1) / warps;
    if (lo >= hi) return;
    int row = (int)(lo / n), chunk = (int)(lo % n);
    float c = kLog2e;
    bool greedy = false, wanted = true, wanted2 = true;
    auto look_up = [&](int of) {  // -> wanted
        const int b = sequence_of(a.q_start, a.B, of);
        const float t = b >= 0 && a.temperature != nullptr ? a.temperature[b] : 1.f;
        c = exponent_scale(t), greedy = t == 0.f;
        return b >= 0 && !(DRAFTER && (of + 1 == a.q_start[b + 1] || greedy));
    };
    Loaded now, next;
    if (DRAFTER) wanted = look_up(row);
    if (wanted) load_chunk(Row<T>(base, ld, row, a.V), chunk, now);
    int known = DRAFTER ? row : -1;
    for (int64_t i = lo; i < hi; ++i) {
        int row2 = row, chunk2 = chunk + 1;
        if (chunk2 == n) ++row2, chunk2 = 0;
        const float c0 = c;
        if (i + 1 < hi) {
            if (DRAFTER && row2 != row) wanted2 = look_up(row2);
            else wanted2 = wanted;
            if (!DRAFTER || wanted2) load_chunk(Row<T>(base, ld, row2, a.V), chunk2, next);
        }
        if (!DRAFTER && row != known) {
            known = row;
            if (a.temperature != nullptr) wanted = look_up(row);
        }
        if (wanted) {
            const ChunkStat s = chunk_stat<T>(Row<T>(base, ld, row, a.V), chunk, now, DRAFTER ? c0 : c, !DRAFTER && greedy);
            if (lane == 0) out[(int64_t)row * a.pitch + chunk] = s;
        }
        row = row2, chunk = chunk2, now = next;
        if (DRAFTER) wanted = wanted2;
    }
}

template <typename TX, typename TD>
__global__ void __launch_bounds__(kStatThreads, kStatCtas) verify_stats_kernel(const VerifyArgs a) {
    behind_grid();
    // half the CTAs have the drafter's rows
    if (a.draft == nullptr) stats_run<TX, false>(a, a.logits, a.ld, a.stats, (int)blockIdx.x, (int)gridDim.x);
    else if ((blockIdx.x & 1) == 0) stats_run<TX, false>(a, a.logits, a.ld, a.stats, (int)blockIdx.x / 2, (int)gridDim.x / 2);
    else stats_run<TD, true>(a, a.draft, a.draft_ld, a.stats + (int64_t)a.T * a.pitch, (int)blockIdx.x / 2, (int)gridDim.x / 2);
}

// log2 of 2^(c (x - best)), exact but for FP64's rounding.
__device__ inline double exponent(float x, float best, float c) { return ((double)x - (double)best) * (double)c; }

// A chunk's sum in units of 2^(c best) of its row.  A chunk whose largest term is below 2^-125 there counts as none, so that whatever chunk is chosen has a
// term that FP32 holds (down to 2^-126: exp2_of).
__device__ inline double chunk_weight(const ChunkStat &s, float c, float best) {
    const double off = exponent(s.best, best, c);  // -inf: nothing in it
    return off < -125.0 ? 0.0 : s.sum * (double)exp2_of((float)off);
}
__device__ inline double warp_sum(double v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}
// The sum over this and the lanes below.
__device__ inline double warp_upto(double v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += o;
    }
    return v;
}

// A row's chunks joined, the sum in units of 2^(c best).  By a whole warp; a lane asks for several chunks at once.
struct RowStat {
    double sum;
    float best;
    int at, code;
};
constexpr int kHeld = 5;  // of 160 chunks: 163,840 logits in FP32 and twice as many in BF16
struct Held {
    ChunkStat k[kHeld];
};
__device__ inline void ask_stats(const ChunkStat *s, int n, Held &h) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) h.k[i] = 32 * i + lane < n ? s[32 * i + lane] : ChunkStat{0.0, -INFINITY, 0x7fffffff};
}
__device__ inline RowStat join_chunks(const ChunkStat *s, int n, const Held &h, float c, int bad_code) {
    const int lane = threadIdx.x & 31;
    float best = -INFINITY;
    int at = 0x7fffffff;
    auto larger = [&](const ChunkStat &k) {
        if (k.best > best) at = k.at;  // the first of those that are as large
        best = max_nan(best, k.best);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) larger(h.k[i]);
#pragma unroll 1
    for (int k = 32 * kHeld + lane; k < n; k += 32) larger(s[k]);
    const float most = warp_max_nan(best);
    RowStat r{0.0, most, (int)__reduce_min_sync(0xffffffffu, best == most ? at : 0x7fffffff), 0};
    if (!(most > -INFINITY && most < INFINITY)) {
        r.code = bad_code;
        return r;
    }
    double sum = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) sum += chunk_weight(h.k[i], c, most);
#pragma unroll 1
    for (int k = 32 * kHeld + lane; k < n; k += 32) sum += chunk_weight(s[k], c, most);
    r.sum = warp_sum(sum);
    return r;
}

// What is drawn from: weights of a piece's tokens.
template <typename TX>
struct OfTarget {  // 2^(c (x - best)), nothing for the token `without`
    Row<TX> r;
    float c, best;
    int without;
    static constexpr int VE = Row<TX>::VE;
    __device__ inline int token(int piece) const { return r.token(piece); }
    __device__ inline void weights(int piece, float (&w)[VE]) const {
        Row<TX>::values(r.raw(piece), w);
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = r.token(piece) + i == without ? 0.f : weight_of(w[i], 0.5f * best, 2.f * c);
    }
};
template <typename TX, typename TD>
struct OfDifference {  // max(p - q, 0)
    Row<TX> r;
    Row<TD> q;
    float c, best, inv, q_best, q_inv;
    static constexpr int VE = Row<TX>::VE;
    __device__ inline int token(int piece) const { return r.token(piece); }
    __device__ inline bool together() const { return sizeof(TX) == sizeof(TD) && r.mis == q.mis; }  // the rows' pieces hold the same tokens
    // Products and difference are rounded each by itself: equal probabilities leave nothing (a fused multiply-add would leave the other product's rounding), and a run's sum has a weight behind
    // it wherever it is computed again.
    __device__ inline void differ(float (&w)[VE], const float (&d)[VE]) const {
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = fmaxf(__fsub_rn(__fmul_rn(weight_of(w[i], 0.5f * best, 2.f * c), inv), __fmul_rn(weight_of(d[i], 0.5f * q_best, 2.f * c), q_inv)), 0.f);
    }
    __device__ inline void weights(int piece, float (&w)[VE]) const {
        float d[VE];
        const int t0 = r.token(piece);
        Row<TX>::values(r.raw(piece), w);
#pragma unroll
        for (int i = 0; i < VE; ++i) d[i] = t0 + i >= 0 && t0 + i < q.V ? q.at(t0 + i) : -INFINITY;
        differ(w, d);
    }
    // The weights' sum of one piece each of `N` chunks, kPieces apart, of rows whose pieces hold the same tokens: all are asked for before one is looked at; pieces that are not whole
    // count as nothing here.
    template <int N>
    __device__ inline void sums(int piece, int end, float (&s)[N]) const {
        const int whole0 = r.mis != 0, whole1 = min(end, (r.V + r.mis) / VE);
        const uint4 *const xp = reinterpret_cast<const uint4 *>(r.p - r.mis) + piece, *const yp = reinterpret_cast<const uint4 *>(q.p - q.mis) + piece;
        uint4 x[N], y[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (piece + i * kPieces >= whole0 && piece + i * kPieces < whole1) x[i] = __ldg(xp + i * kPieces), y[i] = __ldg(yp + i * kPieces);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = 0.f;
            if (piece + i * kPieces >= whole0 && piece + i * kPieces < whole1) {
                float w[VE], d[VE];
                Row<TX>::values(x[i], w), Row<TX>::values(y[i], d);
                differ(w, d);
#pragma unroll
                for (int k = 0; k < VE; ++k) s[i] += w[k];
            }
        }
    }
};
template <int N>
__device__ inline float sum_of(const float (&w)[N]) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) s += w[k];
    return s;
}

// Drawing, by all threads of a CTA: these have parts that lie one behind the other.
struct Draw {
    double warp_s[kWarps];
    int first, last;
};
// The sum over this and the threads before; the whole sum in *all.
__device__ inline double block_upto(Draw &sh, double v, double *all) {
    const int warp = threadIdx.x >> 5;
    double upto = warp_upto(v), sum = 0;
    __syncthreads();  // what was there before has been read
    if ((threadIdx.x & 31) == 31) sh.warp_s[warp] = upto;
    if (threadIdx.x == 0) sh.first = kThreads, sh.last = -1;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w == warp) upto += sum;
        sum += sh.warp_s[w];
    }
    *all = sum;
    return upto;
}
// After block_upto: the thread in whose part `target` falls, the last one that has any if rounding leaves none.
__device__ inline int block_find(Draw &sh, double mine, double upto, double target) {
    const uint32_t over = __ballot_sync(0xffffffffu, mine > 0 && upto > target), some = __ballot_sync(0xffffffffu, mine > 0);
    if ((threadIdx.x & 31) == 0) {
        if (over) atomicMin(&sh.first, (int)threadIdx.x + __ffs(over) - 1);
        if (some) atomicMax(&sh.last, (int)threadIdx.x + 31 - __clz(some));
    }
    __syncthreads();
    return sh.first < kThreads ? sh.first : sh.last;
}
// The first token of a piece up to which more than `target` has come, the last one with a weight if rounding leaves none.
template <typename F>
__device__ inline int pick_in_piece(const F &f, int piece, double target) {
    float w[F::VE];
    f.weights(piece, w);
    double sum = 0;
    int token = -1;
    bool found = false;
#pragma unroll
    for (int k = 0; k < F::VE; ++k) {
        sum += (double)w[k];
        if (!found && w[k] > 0.f) token = f.token(piece) + k, found = sum > target;
    }
    return token;
}

struct Decision {
    RowStat p, q;
    float x;                // the drafted token's logit
    int token, keep, code;  // the drafted token behind the row; keep: 1 kept, 0 not, -1 there is none
};
__device__ inline float log_probability(float x, const RowStat &p, float c) { return (float)(exponent(x, p.best, c) * kLn2) - logf((float)p.sum); }

template <typename TX, typename TD, bool DRAFT>
__global__ void __launch_bounds__(kThreads, 2) verify_decide_kernel(const VerifyArgs a) {
    __shared__ Decision dec[kWarps];
    __shared__ Draw draw;
    __shared__ double total_s, from_s;
    __shared__ int chunk_s;
    __shared__ float run_s[DRAFT ? kMaxRun * kWarps : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ranks = DRAFT ? a.ranks : 1, rank = (int)blockIdx.x % ranks, b = (int)blockIdx.x / ranks;
    // The caller's arrays were complete before the launch ahead, the first of the two, began its work: they are read ahead of its end.
    const int first = a.q_start[b], end = a.q_start[b + 1];
    const float t = a.temperature != nullptr ? a.temperature[b] : 1.f, u_pick = a.u_pick[b], c = exponent_scale(t);
    bool falls = false;
    for (int i = threadIdx.x; i < b; i += kThreads) falls = falls || a.q_start[i] > first;
    falls = __syncthreads_or(falls);
    if (falls || first < 0 || end < first || end > a.T || first == end) {
        behind_grid();
        if (rank == 0 && threadIdx.x == 0) {
            a.n_new[b] = 0;
            if (falls || first != end || first < 0 || end > a.T) raise_error(a.err, (uint32_t)b, kBadRange);
        }
        return;
    }
    const bool greedy = t == 0.f;
    int code = t == 0.f || (t >= 0x1p-126f && t < INFINITY) ? 0 : kBadTemperature, bad_row = first, stop = first;
    Decision d{};
    // ---- rows in order, a warp a row, up to the first whose draft is not kept
#pragma unroll 1
    for (int r0 = first;; r0 += kWarps) {
        const int row = r0 + warp;
        Decision e{};
        e.keep = -1;
        float u = 0.f, qx = 0.f;
        if (row + 1 < end) {
            e.token = a.ids[row + 1];
            u = a.u[row];
            if (e.token < 0 || e.token >= a.V) e.code = kBadId;
            else {
                e.x = Row<TX>(a.logits, a.ld, row, a.V).at(e.token);
                if constexpr (DRAFT) qx = Row<TD>(a.draft, a.draft_ld, row, a.V).at(e.token);
            }
        }
        if (r0 == first) behind_grid();
        if (code != 0) break;
        if (row < end) {
            const int bad_id = e.code, np = Row<TX>(a.logits, a.ld, row, a.V).chunks(), nq = DRAFT && row + 1 < end ? Row<TD>(a.draft, a.draft_ld, row, a.V).chunks() : 0;
            const ChunkStat *const ps = a.stats + (int64_t)row * a.pitch, *const qs = ps + (int64_t)a.T * a.pitch;
            Held hp, hq;
            ask_stats(ps, np, hp);
            if constexpr (DRAFT) ask_stats(qs, nq, hq);
            e.p = join_chunks(ps, np, hp, c, kBadLogits);
            e.code = e.p.code != 0 ? e.p.code : bad_id;
            if (row + 1 < end && e.code == 0) {
                if (greedy) e.keep = e.token == e.p.at;
                else {
                    // u q < p without the divisions: u 2^.. P < 2^.. Q
                    double q = 1.0, q_sum = 1.0;
                    if (!(u >= 0.f && u < 1.f)) e.code = kBadRandom;
                    if constexpr (DRAFT) {
                        e.q = join_chunks(qs, nq, hq, c, kBadDraft);
                        if (e.code == 0) e.code = e.q.code;
                        if (e.code == 0) q = (double)exp2_of((float)exponent(qx, e.q.best, c)), q_sum = e.q.sum;
                    }
                    if (e.code == 0) e.keep = (double)u * q * e.p.sum < (double)exp2_of((float)exponent(e.x, e.p.best, c)) * q_sum;
                }
            }
            if (lane == 0) dec[warp] = e;
        }
        __syncthreads();
        int n = 0;  // of this group, kept
        bool done = false;
        while (n < kWarps && r0 + n < end && !done) {
            if (dec[n].code != 0) code = dec[n].code, bad_row = r0 + n, done = true;
            else if (dec[n].keep != 1) d = dec[n], done = true;
            else ++n;
        }
        if (rank == 0 && warp < n && lane == 0) {
            a.next_ids[row] = e.token;
            if (a.logp != nullptr) a.logp[row] = log_probability(e.x, e.p, c);
        }
        stop = r0 + n;
        __syncthreads();
        if (done) break;
    }
    if (code == 0 && !greedy && !(u_pick >= 0.f && u_pick < 1.f)) code = kBadRandom, bad_row = stop;
    if (code != 0) {
        if (rank == 0) {
            if (threadIdx.x == 0) a.n_new[b] = 0, raise_error(a.err, (uint32_t)bad_row, (uint32_t)code);
            for (int i = first + (int)threadIdx.x; i < end; i += kThreads) {  // those of the rows before too, written ahead of the last barrier
                a.next_ids[i] = -1;
                if (a.logp != nullptr) a.logp[i] = qnan_f32();
            }
        }
        return;
    }
    if (rank == 0) {
        if (threadIdx.x == 0) a.n_new[b] = stop - first + 1;
        for (int i = stop + 1 + (int)threadIdx.x; i < end; i += kThreads) {
            a.next_ids[i] = -1;
            if (a.logp != nullptr) a.logp[i] = 0.f;
        }
    }
    const Row<TX> x(a.logits, a.ld, stop, a.V);
    const int n = x.chunks();
    auto say = [&](int token) {  // one thread
        a.next_ids[stop] = token;
        if (a.logp != nullptr) a.logp[stop] = log_probability(x.at(token), d.p, c);
    };
    if (greedy) {
        if (rank == 0 && threadIdx.x == 0) say(d.p.at);
        return;
    }
    double all;
    // ---- from the difference of two distributions: the cluster's CTAs have a run of the row's chunks each, a warp an eighth of every chunk, a thread a piece of it
    if (DRAFT && d.keep == 0) {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        const OfDifference<TX, TD> f{x, Row<TD>(a.draft, a.draft_ld, stop, a.V), c, d.p.best, (float)(1.0 / d.p.sum), d.q.best, (float)(1.0 / d.q.sum)};
        const int lo = n * rank / ranks, hi = n * (rank + 1) / ranks, parts = (hi - lo) * kWarps;
        auto lanes_sum = [](float s) {
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
            return s;
        };
        if (f.together()) {
            constexpr int kBatch = 4;
#pragma unroll 1
            for (int k = lo; k < hi; k += kBatch) {
                float sums[kBatch];
                f.sums(k * kPieces + (int)threadIdx.x, hi * kPieces, sums);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const float sum = lanes_sum(sums[i]);
                    if (lane == 0 && k + i < hi) run_s[(k + i - lo) * kWarps + warp] = sum;
                }
            }
            __syncthreads();
            // the row's first and last piece, where they are not whole
            const int last = x.pieces() - 1;
            for (int i = 0; i < 2; ++i) {
                const int piece = i ? last : 0, chunk = piece / kPieces;
                const bool part = i ? (x.V + x.mis) % Row<TX>::VE != 0 && (last > 0 || x.mis == 0) : x.mis != 0;
                if (part && chunk >= lo && chunk < hi && (int)threadIdx.x == piece % kPieces) {
                    float w[Row<TX>::VE];
                    f.weights(piece, w);
                    run_s[(chunk - lo) * kWarps + warp] += sum_of(w);
                }
                __syncwarp();
            }
        } else
#pragma unroll 1
            for (int k = warp; k < parts; k += kWarps) {
                float w[Row<TX>::VE];
                f.weights((lo + k / kWarps) * kPieces + (int)threadIdx.x, w);
                const float sum = lanes_sum(sum_of(w));
                if (lane == 0) run_s[k] = sum;
            }
        __syncthreads();
        const int per = (parts + kThreads - 1) / kThreads, k0 = min(parts, (int)threadIdx.x * per), k1 = min(parts, k0 + per);
        double mine = 0;
        for (int k = k0; k < k1; ++k) mine += (double)run_s[k];
        const double upto = block_upto(draw, mine, &all);
        if (threadIdx.x == 0) total_s = all;
        cluster.sync();
        double before = 0, total = 0, from = 0;
        int owner = -1;
        double sums[kMaxRanks];
        for (int k = 0; k < ranks; ++k) sums[k] = *cluster.map_shared_rank(&total_s, k), total += sums[k];
        cluster.sync();  // nobody's sum is read from here on
        if (total > kNoDifference) {
            const double target = (double)u_pick * total;
            bool found = false;
            for (int k = 0; k < ranks; ++k) {
                if (!found && sums[k] > 0) owner = k, from = before, found = before + sums[k] > target;
                before += sums[k];
            }
            if (owner != rank) return;
            if (block_find(draw, mine, upto, target - from) == (int)threadIdx.x) {
                double sum = upto - mine, at_from = sum;
                int at = k0;
                found = false;
                for (int k = k0; k < k1; ++k) {
                    if (!found && run_s[k] > 0.f) at = k, at_from = sum, found = sum + (double)run_s[k] > target - from;
                    sum += (double)run_s[k];
                }
                chunk_s = at, from_s = target - from - at_from;
            }
            __syncthreads();
            if (warp != 0) return;
            const int piece = (lo + chunk_s / kWarps) * kPieces + chunk_s % kWarps * 32 + lane;
            float w[Row<TX>::VE];
            f.weights(piece, w);
            const double part = (double)sum_of(w), sofar = warp_upto(part);
            const uint32_t over = __ballot_sync(0xffffffffu, part > 0 && sofar > from_s), some = __ballot_sync(0xffffffffu, part > 0);
            if (lane == (over ? __ffs(over) - 1 : 31 - __clz(some))) say(pick_in_piece(f, piece, from_s - (sofar - part)));
            return;
        }
    }
    if (rank != 0) return;
    // ---- from the target's distribution, without the refused token where the drafter gave no more than that
    const ChunkStat *const s = a.stats + (int64_t)stop * a.pitch;
    OfTarget<TX> f{x, c, d.p.best, -1};
    int refused = -1;
    double rest = 0;
    if (!DRAFT && d.keep == 0) {
        f.without = d.token, refused = (d.token + x.mis) / Row<TX>::kChunk;
        float w[Row<TX>::VE];
        f.weights(refused * kPieces + (int)threadIdx.x, w);
        block_upto(draw, (double)sum_of(w), &rest);
    }
    // chunks: a thread's run of them, one behind the other
    const int per = (n + kThreads - 1) / kThreads, k0 = min(n, (int)threadIdx.x * per), k1 = min(n, k0 + per);
    double mine = 0, upto;
#pragma unroll 1
    for (int again = 0;; ++again) {
        mine = 0;
        for (int k = k0; k < k1; ++k) mine += k == refused ? rest : chunk_weight(s[k], c, d.p.best);
        upto = block_upto(draw, mine, &all);
        if (all > 0 || again) break;
        refused = -1, f.without = -1;  // nothing but the refused token: from all of it
    }
    double target = (double)u_pick * all;
    if (block_find(draw, mine, upto, target) == (int)threadIdx.x) {
        double sum = upto - mine, from = sum;
        int at = k0;
        bool found = false;
        for (int k = k0; k < k1; ++k) {
            const double w = k == refused ? rest : chunk_weight(s[k], c, d.p.best);
            if (!found && w > 0) at = k, from = sum, found = sum + w > target;
            sum += w;
        }
        chunk_s = at, from_s = target - from;
    }
    __syncthreads();
    // pieces of the chunk: one a thread
    const int piece = chunk_s * kPieces + (int)threadIdx.x;
    target = from_s;
    float w[Row<TX>::VE];
    f.weights(piece, w);
    mine = (double)sum_of(w);
    upto = block_upto(draw, mine, &all);
    if (block_find(draw, mine, upto, target) == (int)threadIdx.x) say(pick_in_piece(f, piece, target - (upto - mine)));
}

// Chunks of a row of FP32 that begins at a piece's last token: no row has more.
int64_t most_chunks(int64_t V) { return (V + 3 + 4 * kPieces - 1) / (4 * kPieces); }

template <typename TX, typename TD>
cudaError_t launch_verify(const VerifyArgs &a, cudaStream_t st) {
    const bool draft = a.draft != nullptr;
    // a warp a chunk until the machine is full
    const int64_t chunks = (int64_t)a.T * ((a.V + 4 * kPieces - 1) / (4 * kPieces)), per = kStatThreads / 32, most = (int64_t)sm_count() * kStatCtas / 2 * 2;
    const unsigned grid = (unsigned)std::min<int64_t>((chunks + per - 1) / per * (draft ? 2 : 1), most);
    const cudaError_t e = launch_behind(verify_stats_kernel<TX, TD>, dim3(grid), dim3(kStatThreads), 0, st, 1, a);
    if (e != cudaSuccess) return e;
    return draft ? launch_behind(verify_decide_kernel<TX, TD, true>, dim3((unsigned)(a.B * a.ranks)), dim3(kThreads), 0, st, a.ranks, a)
                 : launch_behind(verify_decide_kernel<TX, TD, false>, dim3((unsigned)a.B), dim3(kThreads), 0, st, 1, a);
}

}  // namespace
}  // namespace sxb

using namespace sxb;

extern "C" {

size_t sxb_verify_drafts_workspace_bytes(int64_t T, int64_t B, int64_t V) {
    if (!(T >= 1 && T <= (1 << 20) && B >= 1 && B <= kMaxB && V >= 1 && V <= kMaxV)) {
        fail_check(SXB_FILE_, __LINE__, __func__, "1 <= T, V <= 2^20, 1 <= B <= 8192", cat("verify_drafts_workspace_bytes: T = ", T, ", B = ", B, ", V = ", V));
        return 0;
    }
    return (size_t)(2 * T * most_chunks(V)) * sizeof(ChunkStat);
}

int sxb_verify_drafts(const SxbVerifyDraftsArgs *args, sxb_stream_t stream) {
    const char *fn = "verify_drafts";
    SXB_CHECK(args != nullptr, fn, ": null argument block");
    const SxbVerifyDraftsArgs &g = *args;
    const int64_t T = g.T, V = g.V, B = g.B;
    SXB_CHECK(T >= 1 && T <= (1 << 20) && B >= 1 && B <= kMaxB && V >= 1 && V <= kMaxV, fn, ": T = ", T, " rows, B = ", B, " sequences, V = ", V, " tokens, expected 1..2^20, ",
              kMaxB, " sequences at most");
    SXB_CHECK(g.logits != nullptr && g.ids != nullptr && g.q_start != nullptr && g.u != nullptr && g.u_pick != nullptr && g.next_ids != nullptr && g.n_new != nullptr &&
                  g.ws != nullptr && g.err != nullptr,
              fn, ": null pointer (logits=", g.logits, ", ids=", (const void *)g.ids, ", q_start=", (const void *)g.q_start, ", u=", (const void *)g.u, ", u_pick=",
              (const void *)g.u_pick, ", next_ids=", (const void *)g.next_ids, ", n_new=", (const void *)g.n_new, ", ws=", g.ws, ", err=", (const void *)g.err, ")");
    SXB_CHECK(act_ok(g.act) && (g.draft_logits == nullptr || act_ok(g.draft_act)), fn, ": unsupported dtypes ", g.act, " of logits, ", g.draft_act, " of draft_logits");
    SXB_CHECK(g.ld >= V && g.ld <= (1ll << 32) && (g.draft_logits == nullptr || (g.draft_ld >= V && g.draft_ld <= (1ll << 32))), fn, ": row strides ", g.ld, " and ", g.draft_ld,
              ", rows have ", V, " tokens");
    SXB_CHECK(reinterpret_cast<uintptr_t>(g.logits) % act_bytes(g.act) == 0 &&
                  (g.draft_logits == nullptr || reinterpret_cast<uintptr_t>(g.draft_logits) % act_bytes(g.draft_act) == 0),
              fn, ": logits must be aligned to their type");
    const size_t need = sxb_verify_drafts_workspace_bytes(T, B, V);
    SXB_CHECK(g.ws_bytes >= need && aligned16(g.ws), fn, ": workspace of ", g.ws_bytes, " bytes, needs ", need, ", 16-byte aligned");
    const int64_t lb = ((T - 1) * g.ld + V) * act_bytes(g.act), db = g.draft_logits != nullptr ? ((T - 1) * g.draft_ld + V) * act_bytes(g.draft_act) : 0;
    const struct {
        const char *name;
        const void *p;
        int64_t n;
    } outs[4] = {{"next_ids", g.next_ids, 4 * T}, {"n_new", g.n_new, 4 * B}, {"logp", g.logp, g.logp != nullptr ? 4 * T : 0}, {"ws", g.ws, (int64_t)need}},
      ins[8] = {{"logits", g.logits, lb}, {"draft_logits", g.draft_logits, db}, {"ids", g.ids, 4 * T}, {"q_start", g.q_start, 4 * (B + 1)}, {"u", g.u, 4 * T},
                {"u_pick", g.u_pick, 4 * B}, {"temperature", g.temperature, 4 * B}, {"err", g.err, 12}};
    for (int o = 0; o < 4; ++o) {
        if (outs[o].p == nullptr) continue;
        for (const auto &i : ins) SXB_CHECK(i.p == nullptr || apart(outs[o].p, outs[o].n, i.p, i.n), fn, ": ", outs[o].name, " [", outs[o].p, "] overlaps ", i.name, " [", i.p, "]");
        for (int k = 0; k < o; ++k)
            SXB_CHECK(outs[k].p == nullptr || apart(outs[o].p, outs[o].n, outs[k].p, outs[k].n), fn, ": ", outs[o].name, " [", outs[o].p, "] overlaps ", outs[k].name);
    }
    VerifyArgs a{};
    a.logits = g.logits, a.draft = g.draft_logits, a.ld = g.ld, a.draft_ld = g.draft_ld, a.ids = g.ids, a.q_start = g.q_start, a.u = g.u, a.u_pick = g.u_pick;
    a.temperature = g.temperature, a.next_ids = g.next_ids, a.n_new = g.n_new, a.logp = g.logp, a.stats = static_cast<ChunkStat *>(g.ws), a.err = g.err;
    a.T = (int)T, a.V = (int)V, a.B = (int)B, a.pitch = (int)most_chunks(V);
    a.ranks = B * kMaxRanks <= 2 * (int64_t)sm_count() ? kMaxRanks : kMinRanks;  // eight while all find their places at once
    auto st = static_cast<cudaStream_t>(stream);
    const bool x32 = g.act == SXB_ACT_F32, d32 = g.draft_logits != nullptr ? g.draft_act == SXB_ACT_F32 : x32;
    const cudaError_t e = x32 ? (d32 ? launch_verify<float, float>(a, st) : launch_verify<float, uint16_t>(a, st))
                              : (d32 ? launch_verify<uint16_t, float>(a, st) : launch_verify<uint16_t, uint16_t>(a, st));
    SXB_CUDA(e, fn, ": launching T=", T, " B=", B, " V=", V);
    SXB_CHECK_LAUNCH(fn, " T=", T, " B=", B, " V=", V);
    return SXB_OK;
}

int sxb_report_verify_error(const uint32_t e[3], const char *what) {
    if (e[0] == 0) return SXB_OK;
    static const char *const said[7] = {"?", "logits that are not finite, or all masked,", "a drafter's logits that are not finite, or all masked,", "a drafted token out of range",
                                        "a random number outside [0, 1)", "a temperature out of range", "a row range that falls, overlaps or leaves the batch"};
    last_error() = cat(what, ": ", said[e[2] <= 6 ? e[2] : 0], e[2] == 6 ? " at sequence " : " at row ", e[1], "; that sequence has no new tokens");
    return SXB_ERR_DATA;
}

int sxb_check_verify_error(const uint32_t *err, const char *what) {
    uint32_t e[3];
    SXB_CHECK(err != nullptr, "check_verify_error: null pointer");
    SXB_CUDA(cudaMemcpy(e, err, sizeof(e), cudaMemcpyDeviceToHost), what, ": reading the error words");
    return sxb_report_verify_error(e, what);
}

}  // extern "C"
