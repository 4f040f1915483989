// Verification of drafted tokens against the target's probabilities, from given random numbers (include/strix_b200.h has the rules).
//
// Two launches.  The first reads every row's logits once, in chunks: a chunk's largest logit, the first token that has it, and the sum of 2^(c x - c max),
// c = log2(e) / temperature.  The second, a CTA a sequence (a cluster of eight where the drafter gives its distribution), joins a row's chunks, tests the
// drafts, and draws the next token: from the chunks' sums it knows the chunk in which the random number falls and reads that one again; only a difference of
// two distributions takes the whole row of both, once more, shared by the cluster.  Nothing is counted or left behind in the workspace: no atomics, and
// results do not depend on who comes first.
//
// A border's error: a term takes c (x - max) in FP32 (2^-23 of the exponent, which is small where the term is large), one ex2 (2^-22), sums of sixteen
// terms a thread and 256 threads in FP32; chunks are joined in FP64, where the exponents c max are exact, and no logit is too large for them.

#include "common.cuh"
#include "tc_ptx.cuh"

#include <cooperative_groups.h>

namespace sxb {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kChunk = 4096;   // tokens of a chunk: sixteen a thread, all loads at once
constexpr int kRanks = 8;      // CTAs that share a difference of two rows
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994531;

enum { kBadLogits = 1, kBadDraft = 2, kBadId = 3, kBadRandom = 4, kBadTemperature = 5, kBadRange = 6 };

struct ChunkStat {  // of 2^(c x) over a chunk
    double sum;     // relative to 2^(c best)
    float best;     // NaN: the chunk holds a NaN or +inf
    int at;
};

struct VerifyArgs {
    const void *logits, *draft;
    int64_t ld, draft_ld;
    const int32_t *ids, *q_start;
    const float *u, *u_pick, *temperature;
    int32_t *next_ids, *n_new;
    float *logp;
    ChunkStat *stats;  // [T (, T of the drafter)][n_chunks]
    uint32_t *err;
    int T, V, B, n_chunks;
};

// Tokens are read in pieces of sixteen aligned bytes.  A row may begin inside one: piece i holds the tokens i * VE - mis ..., those outside 0 .. V - 1 are none.
template <typename T>
struct Row {
    static constexpr int VE = 16 / (int)sizeof(T);
    const T *p;
    int mis, V;
    __device__ inline Row(const void *base, int64_t ld, int64_t row, int n) : p(static_cast<const T *>(base) + row * ld), V(n) {
        mis = (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % VE);
    }
    __device__ inline int pieces() const { return (V + mis + VE - 1) / VE; }
    __device__ inline int token(int piece) const { return piece * VE - mis; }
    __device__ inline float at(int t) const { return load_as_f32(p, t); }
    // The tokens t0 .. t0 + VE - 1, -inf where there are none.
    __device__ inline void load(int t0, float (&v)[VE]) const {
        if (t0 >= 0 && t0 + VE <= V && (reinterpret_cast<uintptr_t>(p + t0) & 15) == 0) {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p + t0));
            if constexpr (sizeof(T) == 4) {
                v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
            } else {
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) v[i] = t0 + i >= 0 && t0 + i < V ? load_as_f32(p, t0 + i) : -INFINITY;
        }
    }
};

// The scale of a sequence's exponents; greedy sequences' log-probabilities are those of temperature 1.
__device__ inline float exponent_scale(float t) { return t == 0.f ? kLog2e : __fdiv_rn(kLog2e, t); }

// The first sequence that has the row, -1 if none has.  By a whole warp.
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

template <typename TX>
__device__ inline void chunk_stats(const VerifyArgs &a, const void *base, int64_t ld, int64_t row, int chunk, ChunkStat *out) {
    constexpr int VE = Row<TX>::VE, NP = kChunk / VE / kThreads;
    __shared__ float most_s[kWarps], sum_s[kWarps];
    __shared__ int at_s[kWarps];
    const Row<TX> r(base, ld, row, a.V);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float v[NP][VE];
#pragma unroll
    for (int j = 0; j < NP; ++j) r.load(r.token(chunk * (kChunk / VE) + j * kThreads + (int)threadIdx.x), v[j]);
    float c = kLog2e;
    if (a.temperature != nullptr) {
        const int b = sequence_of(a.q_start, a.B, (int)row);
        if (b < 0) return;  // the same for every warp
        c = exponent_scale(a.temperature[b]);
    }
    float most = -INFINITY;
    int at = 0x7fffffff;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int t0 = r.token(chunk * (kChunk / VE) + j * kThreads + (int)threadIdx.x);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            bad = bad || !(v[j][i] < INFINITY);
            if (v[j][i] > most) most = v[j][i], at = t0 + i;
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const float m = __shfl_xor_sync(0xffffffffu, most, off);
        const int i = __shfl_xor_sync(0xffffffffu, at, off);
        if (m > most || (m == most && i < at)) most = m, at = i;
    }
    if (__any_sync(0xffffffffu, bad)) most = qnan_f32();
    if (lane == 0) most_s[warp] = most, at_s[warp] = at;
    __syncthreads();
    most = most_s[0], at = at_s[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
        const float m = most_s[w];
        if (m != m || m > most || (m == most && at_s[w] < at)) most = m, at = at_s[w];
    }
    float sum = 0.f;
    if (most > -INFINITY) {
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < VE; ++i) sum += exp2_fast((v[j][i] - most) * c);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) sum_s[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0;
        for (int w = 0; w < kWarps; ++w) total += (double)sum_s[w];
        *out = ChunkStat{total, most, at};
    }
}

template <typename TX, typename TD>
__global__ void __launch_bounds__(kThreads) verify_stats_kernel(const VerifyArgs a) {
    behind_grid();
    const int64_t row = blockIdx.x / a.n_chunks;
    const int chunk = (int)(blockIdx.x % a.n_chunks);
    ChunkStat *const out = a.stats + (blockIdx.y * (int64_t)a.T + row) * a.n_chunks + chunk;
    if (blockIdx.y == 0) chunk_stats<TX>(a, a.logits, a.ld, row, chunk, out);
    else chunk_stats<TD>(a, a.draft, a.draft_ld, row, chunk, out);
}

// A chunk's sum in units of 2^(c best) of its row.  A chunk whose largest term is below 2^-126 there counts as none, so that whatever chunk is chosen has a
// term that FP32 holds.
__device__ inline double chunk_weight(const ChunkStat &s, float c, float best) {
    const double off = ((double)s.best - (double)best) * (double)c;  // -inf: nothing in it
    return off < -126.0 ? 0.0 : s.sum * exp2(off);
}

// A row's chunks joined, the sum in units of 2^(c best).  By a whole warp.
struct RowStat {
    double sum;
    float best;
    int at, code;
};
__device__ inline RowStat join_chunks(const ChunkStat *s, int n, float c, int bad_code) {
    const int lane = threadIdx.x & 31;
    float best = -INFINITY;
    int at = 0x7fffffff;
    bool bad = false;
    for (int k = lane; k < n; k += 32) {
        const float m = s[k].best;
        bad = bad || m != m;
        if (m > best) best = m, at = s[k].at;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const float m = __shfl_xor_sync(0xffffffffu, best, off);
        const int i = __shfl_xor_sync(0xffffffffu, at, off);
        if (m > best || (m == best && i < at)) best = m, at = i;
    }
    RowStat r{0.0, best, at, 0};
    if (__any_sync(0xffffffffu, bad) || best == -INFINITY) {
        r.code = bad_code;
        return r;
    }
    double sum = 0;
    for (int k = lane; k < n; k += 32) sum += chunk_weight(s[k], c, best);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    r.sum = sum;
    return r;
}

// What is drawn from: weights of the tokens of a piece.
template <typename TX>
struct OfTarget {  // 2^(c (x - best)), nothing for the token `without`
    Row<TX> r;
    float c, best;
    int without;
    static constexpr int VE = Row<TX>::VE;
    __device__ inline int token(int piece) const { return r.token(piece); }
    __device__ inline void weights(int piece, float (&w)[VE]) const {
        const int t0 = r.token(piece);
        r.load(t0, w);
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = t0 + i == without ? 0.f : exp2_fast((w[i] - best) * c);
    }
};
template <typename TX, typename TD>
struct OfDifference {  // max(p - q, 0)
    Row<TX> r;
    Row<TD> q;
    float c, best, inv, q_best, q_inv;
    static constexpr int VE = Row<TX>::VE;
    __device__ inline int token(int piece) const { return r.token(piece); }
    __device__ inline void weights(int piece, float (&w)[VE]) const {
        const int t0 = r.token(piece);
        r.load(t0, w);
        float d[VE];
        if constexpr (Row<TD>::VE == VE) q.load(t0, d);
        else
#pragma unroll
            for (int i = 0; i < VE; ++i) d[i] = t0 + i >= 0 && t0 + i < q.V ? q.at(t0 + i) : -INFINITY;
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = fmaxf(exp2_fast((w[i] - best) * c) * inv - exp2_fast((d[i] - q_best) * c) * q_inv, 0.f);
    }
};

// The pieces lo .. hi - 1 summed, by a warp.
template <typename F>
__device__ inline double sum_pieces(const F &f, int lo, int hi) {
    const int lane = threadIdx.x & 31;
    double sum = 0;
    for (int i = lo + lane; i < hi; i += 32) {
        float w[F::VE];
        f.weights(i, w);
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < F::VE; ++k) s += w[k];
        sum += (double)s;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    return sum;
}
// The first token of these pieces up to which more than `target` has come; the last one with a weight if rounding leaves none.  By a warp, at least one weight is not zero.
template <typename F>
__device__ inline int pick_in_pieces(const F &f, int lo, int hi, double target) {
    const int lane = threadIdx.x & 31;
    double before = 0;
    int last = -1;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        float w[F::VE];
#pragma unroll
        for (int k = 0; k < F::VE; ++k) w[k] = 0.f;
        if (i < hi) f.weights(i, w);
        double mine = 0, upto;
        int my_last = -1;
#pragma unroll
        for (int k = 0; k < F::VE; ++k) {
            mine += (double)w[k];
            if (w[k] > 0.f) my_last = f.token(i) + k;
        }
        upto = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const double o = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += o;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, mine > 0 && before + upto > target);
        if (over) {
            const int src = __ffs(over) - 1;
            int token = my_last;
            double sum = before + (upto - mine);
#pragma unroll
            for (int k = F::VE - 1; k >= 0; --k) {  // from the end: the first that is over is the last one written
                double s = sum;
#pragma unroll
                for (int m = 0; m <= k; ++m) s += (double)w[m];
                if (w[k] > 0.f && s > target) token = f.token(i) + k;
            }
            return __shfl_sync(0xffffffffu, token, src);
        }
        const uint32_t some = __ballot_sync(0xffffffffu, my_last >= 0);
        if (some) last = __shfl_sync(0xffffffffu, my_last, 31 - __clz(some));
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return last;
}

// log2 of 2^(c (x - best)), exact but for FP64's rounding.
__device__ inline double exponent(float x, float best, float c) { return ((double)x - (double)best) * (double)c; }

struct Decision {
    RowStat p, q;
    double logp;
    int token, keep, code;  // the drafted token behind the row; keep: 1 kept, 0 not, -1 there is none
};

template <typename TX, typename TD, bool DRAFT>
__global__ void __launch_bounds__(kThreads) verify_decide_kernel(const VerifyArgs a) {
    behind_grid();
    __shared__ Decision dec[kWarps];
    __shared__ double part_s[kWarps], all_s[kWarps * kRanks];
    __shared__ int chosen_s[2];
    __shared__ double from_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = DRAFT ? (int)(blockIdx.x % kRanks) : 0, b = DRAFT ? (int)(blockIdx.x / kRanks) : (int)blockIdx.x;
    const int first = a.q_start[b], end = a.q_start[b + 1];
    bool falls = false;
    for (int i = threadIdx.x; i < b; i += kThreads) falls = falls || a.q_start[i] > first;
    if (__syncthreads_or(falls) || first < 0 || end < first || end > a.T) {
        if (rank == 0 && threadIdx.x == 0) a.n_new[b] = 0, raise_error(a.err, (uint32_t)b, kBadRange);
        return;
    }
    if (first == end) {
        if (rank == 0 && threadIdx.x == 0) a.n_new[b] = 0;
        return;
    }
    const float t = a.temperature != nullptr ? a.temperature[b] : 1.f, c = exponent_scale(t);
    const bool greedy = t == 0.f;
    int code = t == 0.f || (t >= 0x1p-126f && t < INFINITY) ? 0 : kBadTemperature, bad_row = first, stop = first;
    Decision d{};
    // ---- rows in order, a warp a row, up to the first whose draft is not kept
    for (int r0 = first; code == 0; r0 += kWarps) {
        const int row = r0 + warp;
        if (row < end) {
            Decision e{};
            const Row<TX> x(a.logits, a.ld, row, a.V);
            e.p = join_chunks(a.stats + (int64_t)row * a.n_chunks, a.n_chunks, c, kBadLogits);
            e.code = e.p.code;
            e.keep = -1;
            if (row + 1 < end && e.code == 0) {
                e.token = a.ids[row + 1];
                if (e.token < 0 || e.token >= a.V) e.code = kBadId;
                else if (greedy) e.keep = e.token == e.p.at;
                else {
                    const float u = a.u[row];
                    double q = 1.0;
                    if (!(u >= 0.f && u < 1.f)) e.code = kBadRandom;
                    if constexpr (DRAFT) {
                        e.q = join_chunks(a.stats + ((int64_t)a.T + row) * a.n_chunks, a.n_chunks, c, kBadDraft);
                        if (e.code == 0) e.code = e.q.code;
                        if (e.code == 0) q = exp2(exponent(Row<TD>(a.draft, a.draft_ld, row, a.V).at(e.token), e.q.best, c)) / e.q.sum;
                    }
                    const double p = exp2(exponent(x.at(e.token), e.p.best, c)) / e.p.sum;
                    e.keep = (double)u * q < p;
                }
                if (e.code == 0) e.logp = exponent(x.at(e.token), e.p.best, c) * kLn2 - log(e.p.sum);
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
        if (rank == 0 && (int)threadIdx.x < n) {
            a.next_ids[r0 + threadIdx.x] = dec[threadIdx.x].token;
            if (a.logp != nullptr) a.logp[r0 + threadIdx.x] = (float)dec[threadIdx.x].logp;
        }
        stop = r0 + n;
        __syncthreads();
        if (done) break;
    }
    float u = 0.f;
    if (code == 0 && !greedy) {
        u = a.u_pick[b];
        if (!(u >= 0.f && u < 1.f)) code = kBadRandom, bad_row = stop;
    }
    if (code != 0) {
        if (rank == 0) {
            if (threadIdx.x == 0) a.n_new[b] = 0, raise_error(a.err, (uint32_t)bad_row, (uint32_t)code);
            for (int i = first + (int)threadIdx.x; i < end; i += kThreads) {
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
    auto say = [&](int token) {  // one thread
        a.next_ids[stop] = token;
        if (a.logp != nullptr) a.logp[stop] = (float)(exponent(x.at(token), d.p.best, c) * kLn2 - log(d.p.sum));
    };
    if (greedy) {
        if (rank == 0 && threadIdx.x == 0) say(d.p.at);
        return;
    }
    // ---- from the difference of two distributions: the cluster's warps have a run of the row each
    if (DRAFT && d.keep == 0) {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        const OfDifference<TX, TD> f{x, Row<TD>(a.draft, a.draft_ld, stop, a.V), c, d.p.best, (float)(1.0 / d.p.sum), d.q.best, (float)(1.0 / d.q.sum)};
        const int pieces = x.pieces(), run = (pieces + kWarps * kRanks - 1) / (kWarps * kRanks), lo = (rank * kWarps + warp) * run, hi = min(pieces, lo + run);
        const double mine = sum_pieces(f, lo, hi);
        if (lane == 0) part_s[warp] = mine;
        cluster.sync();
        if (threadIdx.x < kWarps * kRanks) all_s[threadIdx.x] = *cluster.map_shared_rank(&part_s[threadIdx.x % kWarps], threadIdx.x / kWarps);
        cluster.sync();  // nobody's part is read from here on
        double total = 0;
        for (int i = 0; i < kWarps * kRanks; ++i) total += all_s[i];
        if (total > 0) {
            const double target = (double)u * total;
            double before = 0, from = 0;
            int at = -1;
            for (int i = 0; i < kWarps * kRanks; ++i) {
                if (all_s[i] > 0) at = i, from = before;
                before += all_s[i];
                if (at == i && before > target) break;
            }
            if (at == rank * kWarps + warp) {
                const int token = pick_in_pieces(f, lo, hi, target - from);
                if (lane == 0) say(token);
            }
            return;
        }
    }
    if (rank != 0) return;
    // ---- from the target's distribution, without the refused token where the drafter gave no more than that
    constexpr int VE = Row<TX>::VE, kPieces = kChunk / VE, kRun = kPieces / kWarps;
    const ChunkStat *const s = a.stats + (int64_t)stop * a.n_chunks;
    OfTarget<TX> f{x, c, d.p.best, -1};
    auto chunk_parts = [&](int chunk) {
        const int lo = chunk * kPieces + warp * kRun;
        const double mine = sum_pieces(f, lo, min(x.pieces(), lo + kRun));
        __syncthreads();
        if (lane == 0) part_s[warp] = mine;
        __syncthreads();
    };
    int refused = -1;
    double rest = 0;
    if (!DRAFT && d.keep == 0) {
        f.without = d.token;
        refused = (d.token + x.mis) / kChunk;
        chunk_parts(refused);
        for (int w = 0; w < kWarps; ++w) rest += part_s[w];
    }
    if (warp == 0) {
        auto of = [&](int k) { return k >= a.n_chunks ? 0.0 : k == refused ? rest : chunk_weight(s[k], c, d.p.best); };
        double total = 0;
        for (int k0 = 0; k0 < a.n_chunks; k0 += 32) total += of(k0 + lane);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
        if (!(total > 0)) {  // nothing but the refused token: from all of it
            refused = -1, total = d.p.sum;
            if (lane == 0) chosen_s[1] = 1;
        } else if (lane == 0) chosen_s[1] = 0;
        const double target = (double)u * total;
        double before = 0, from = 0;
        int at = -1;
        for (int k0 = 0; k0 < a.n_chunks; k0 += 32) {
            const double mine = of(k0 + lane);
            double upto = mine;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const double o = __shfl_up_sync(0xffffffffu, upto, off);
                if (lane >= off) upto += o;
            }
            const uint32_t over = __ballot_sync(0xffffffffu, mine > 0 && before + upto > target), some = __ballot_sync(0xffffffffu, mine > 0);
            const int src = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : -1;
            if (src >= 0) at = k0 + src, from = before + __shfl_sync(0xffffffffu, upto - mine, src);
            if (over) break;
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) chosen_s[0] = at, from_s = target - from;
    }
    __syncthreads();
    if (chosen_s[1]) f.without = -1;
    const int chunk = chosen_s[0];
    double target = from_s;
    chunk_parts(chunk);
    double from = 0, before = 0;
    int at = -1;
    for (int w = 0; w < kWarps; ++w) {
        if (part_s[w] > 0) at = w, from = before;
        before += part_s[w];
        if (at == w && before > target) break;
    }
    if (warp == at) {
        const int lo = chunk * kPieces + warp * kRun, token = pick_in_pieces(f, lo, min(x.pieces(), lo + kRun), target - from);
        if (lane == 0) say(token);
    }
}

int64_t chunks(int64_t V) { return (V + 7 + kChunk - 1) / kChunk; }  // a row may begin up to seven tokens inside a piece

template <typename TX, typename TD>
cudaError_t launch_verify(const VerifyArgs &a, cudaStream_t st) {
    const bool draft = a.draft != nullptr;
    const cudaError_t e = launch_behind(verify_stats_kernel<TX, TD>, dim3((unsigned)((int64_t)a.T * a.n_chunks), draft ? 2 : 1), dim3(kThreads), 0, st, 1, a);
    if (e != cudaSuccess) return e;
    return draft ? launch_behind(verify_decide_kernel<TX, TD, true>, dim3((unsigned)(a.B * kRanks)), dim3(kThreads), 0, st, kRanks, a)
                 : launch_behind(verify_decide_kernel<TX, TD, false>, dim3((unsigned)a.B), dim3(kThreads), 0, st, 1, a);
}

}  // namespace
}  // namespace sxb

using namespace sxb;

extern "C" {

size_t sxb_verify_drafts_workspace_bytes(int64_t T, int64_t B, int64_t V) {
    if (!(T >= 1 && T <= (1 << 20) && B >= 1 && B <= (1 << 20) && V >= 1 && V <= (1 << 20))) {
        fail_check(SXB_FILE_, __LINE__, __func__, "1 <= T, B, V <= 2^20", cat("verify_drafts_workspace_bytes: T = ", T, ", B = ", B, ", V = ", V));
        return 0;
    }
    return (size_t)(2 * T * chunks(V)) * sizeof(ChunkStat);
}

int sxb_verify_drafts(const SxbVerifyDraftsArgs *args, sxb_stream_t stream) {
    const char *fn = "verify_drafts";
    SXB_CHECK(args != nullptr, fn, ": null argument block");
    const SxbVerifyDraftsArgs &g = *args;
    const int64_t T = g.T, V = g.V, B = g.B;
    SXB_CHECK(T >= 1 && T <= (1 << 20) && B >= 1 && B <= (1 << 20) && V >= 1 && V <= (1 << 20), fn, ": T = ", T, " rows, B = ", B, " sequences, V = ", V, " tokens, expected 1..2^20");
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
      ins[6] = {{"logits", g.logits, lb}, {"draft_logits", g.draft_logits, db}, {"ids", g.ids, 4 * T}, {"q_start", g.q_start, 4 * (B + 1)}, {"u", g.u, 4 * T},
                {"u_pick", g.u_pick, 4 * B}};
    for (int o = 0; o < 4; ++o) {
        if (outs[o].p == nullptr) continue;
        for (const auto &i : ins) SXB_CHECK(i.p == nullptr || apart(outs[o].p, outs[o].n, i.p, i.n), fn, ": ", outs[o].name, " [", outs[o].p, "] overlaps ", i.name, " [", i.p, "]");
        for (int k = 0; k < o; ++k)
            SXB_CHECK(outs[k].p == nullptr || apart(outs[o].p, outs[o].n, outs[k].p, outs[k].n), fn, ": ", outs[o].name, " [", outs[o].p, "] overlaps ", outs[k].name);
    }
    VerifyArgs a{};
    a.logits = g.logits, a.draft = g.draft_logits, a.ld = g.ld, a.draft_ld = g.draft_ld, a.ids = g.ids, a.q_start = g.q_start, a.u = g.u, a.u_pick = g.u_pick;
    a.temperature = g.temperature, a.next_ids = g.next_ids, a.n_new = g.n_new, a.logp = g.logp, a.stats = static_cast<ChunkStat *>(g.ws), a.err = g.err;
    a.T = (int)T, a.V = (int)V, a.B = (int)B, a.n_chunks = (int)chunks(V);
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
