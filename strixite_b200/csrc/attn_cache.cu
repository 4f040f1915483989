// The cache side of a decode step's attention: queries and keys normed per head and rotated by their position, keys and values into their pages
// (sxb_attn_qkv_write), and rows of the cache back (sxb_kv_read).
//
//   x' = x / sqrt(mean(x^2) + eps) * w,   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = pos * inv_freq[i]
//
// One pass: a lane has eight neighbouring elements of a head, D / 8 lanes a head, a warp one to four heads; the norm's sum, the rotation's partner and a
// group's extremes go by shuffles.  All FP32, but for the angle: pos * inv_freq loses 2^-24 of a number of turns that grows with the position (a hundred
// thousand tokens: 6e-3 of a radian), so product and reduction are FP64, once a token and angle, into shared memory for all of its heads.  Norm weight
// and rotation are one pair of factors an element, the same for all heads: x'_i = inv * (x_i (w_i cos) + x_partner (w_partner +- sin)).
// The same formulas as sxb_quantize's make the codes (formats/q4.cpp:44-88), from the FP32 values: nothing is rounded on the way.
//
// Measured (B200; us, and the time of the bytes alone at the measured copy rate): 4096 tokens of 32 + 2 x 8 heads of 128 into a BF16 cache 22.2 (15.4), one
// token 3.2 (a launch and four round trips); 33000 rows of 2 x 8 heads of 128 at 8 bits read back as BF16 41 (32).  A warp a token in the first: with a warp
// for half a token 26, a CTA a token 40 (angles and factors made again for every few heads).

#include "attn.cuh"
#include "skinny_mma.cuh"

#include <type_traits>

namespace sxb {
namespace {

constexpr int kWriteWarps = 4, kWriteThreads = 32 * kWriteWarps;
constexpr int64_t kMaxTokens = 1ll << 20;

struct WriteArgs {
    const void *qkv;
    int64_t ld;
    int n_q, n_kv, rot, interleaved;
    const float *q_norm, *k_norm, *inv_freq;
    float eps;
    const int32_t *seq, *pos, *pages;
    int64_t pages_ld;
    int n_seq, n_cols, G, items_per_warp, warps_per_token;
    int64_t T;
    KvView c;
    uint16_t *q_out;
    int64_t q_ld;
    uint32_t *err;
};

// N neighbouring elements (4 to 32 bytes, aligned to them) as FP32, and back.
template <int BYTES> struct Words { uint32_t w[BYTES / 4]; };
template <int BYTES> __device__ inline Words<BYTES> load_words(const void *p) {
    Words<BYTES> r;
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4 *>(r.w)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else if constexpr (BYTES == 8) {
        *reinterpret_cast<uint2 *>(r.w) = *reinterpret_cast<const uint2 *>(p);
    } else {
        r.w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
    return r;
}
template <int BYTES> __device__ inline void store_words(void *p, const Words<BYTES> &r) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(r.w)[i];
    } else if constexpr (BYTES == 8) {
        *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(r.w);
    } else {
        *reinterpret_cast<uint32_t *>(p) = r.w[0];
    }
}
template <typename T, int N> __device__ inline void load_run(const T *p, float (&v)[N]) {
    const auto r = load_words<N * (int)sizeof(T)>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(r.w[i]);
        else v[i] = __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
    }
}
template <int N> __device__ inline void store_bf16_run(uint16_t *p, const float (&v)[N]) {
    Words<2 * N> r;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    store_words<2 * N>(p, r);
}

// A lane's eight elements of a cache row, number `part` of the row's eights.  BITS 16: rounded to BF16.  Otherwise a group's lanes find its extremes; a
// group that holds a NaN or an infinity has no code that stands for it and reads back as NaN throughout.  All lanes of the warp come here together.
template <int D, int BITS>
__device__ inline void store_run(uint8_t *rows, uint32_t *sm, int64_t row, const float (&v)[8], int part, int G, bool on) {
    if constexpr (BITS == 16) {
        if (on) store_bf16_run(reinterpret_cast<uint16_t *>(rows) + row * D + part * 8, v);
    } else {
        constexpr float kLevels = BITS == 4 ? 15.f : 255.f, kWhole = 12582912.f;
        const int lanes = G / 8;  // of a group: 4, 8 or 16
        float lo = v[0], hi = v[0];
        bool bad = !isfinite(v[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) lo = fminf(lo, v[i]), hi = fmaxf(hi, v[i]), bad = bad || !isfinite(v[i]);
        for (int off = 1; off < lanes; off <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
            bad = __shfl_xor_sync(0xffffffffu, (int)bad, off) || bad;
        }
        const uint32_t s_bits = bad ? 0x7fc0u : f32_to_bf16_bits(__fdiv_rn(__fsub_rn(hi, lo), kLevels)), m_bits = bad ? 0x7fc0u : f32_to_bf16_bits(lo);
        const float s = bf16_bits_to_f32((uint16_t)s_bits), m = bf16_bits_to_f32((uint16_t)m_bits);
        const float per = 1.f / s;
        Words<BITS> packed = {};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t code = 0;
            if (s > 0.f) {
                // (v - m) / s is within 2^-13 of the product with 1 / s below 256: where that is no nearer to a half, both round to the same code
                // (rounded by way of 1.5 * 2^23, where neighbours are one apart and the number's low bits are the code)
                const float d = __fsub_rn(v[i], m), x = d * per;
                float r = (x + kWhole) - kWhole;
                if (!(fabsf(x - r) < 0.5f - 1.f / 4096)) r = rintf(__fdiv_rn(d, s));
                code = __float_as_uint(fminf(fmaxf(r, 0.f), kLevels) + kWhole) & 0xffu;
            }
            packed.w[i * BITS / 32] |= code << (i * BITS % 32);
        }
        if (on) {
            if (part % lanes == 0) sm[row * (D / G) + part / lanes] = s_bits | m_bits << 16;
            store_words<BITS>(rows + row * (D * BITS / 8) + part * BITS, packed);
        }
    }
}

// Cache row of (sequence, position), or why there is none: 0 = found, 1 = a row to leave alone, 2 = bad.
struct Place {
    int page, at, state;
};
__device__ inline Place find_place(int seq, int pos, const int32_t *pages, int64_t pages_ld, int n_seq, int n_cols, const KvView &c) {
    Place p{0, 0, 0};
    if (seq < 0) {
        p.state = 1;
    } else if (seq >= n_seq || pos < 0 || (pos >> c.page_shift) >= n_cols) {
        p.state = 2;
    } else {
        p.page = pages[seq * pages_ld + (pos >> c.page_shift)];
        p.at = pos & ((1 << c.page_shift) - 1);
        if ((unsigned)p.page >= (unsigned)c.n_pages) p.state = 2;
    }
    return p;
}

// An item is the heads that a warp takes at once: the queries' items, then the keys', then the values'.  A warp has a run of one token's items, all of
// them where there are many tokens, and the token's angles to itself.
template <typename T, int D, int BITS>
__global__ void __launch_bounds__(kWriteThreads) qkv_write_kernel(const __grid_constant__ WriteArgs a) {
    constexpr int kLanes = D / 8, kHeads = 32 / kLanes, kBatch = sizeof(T) == 4 ? 2 : 4, kCols = D / 16;  // 64 bytes a lane on their way
    __shared__ float2 turns[kWriteWarps][D / 2];  // cos, sin of angle i at [i % 8][i / 8]: lanes have eights
    behind_grid();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane % kLanes, sub = lane / kLanes;
    const int64_t unit = (int64_t)blockIdx.x * kWriteWarps + warp, t = unit / a.warps_per_token;
    if (t >= a.T) return;
    const int first = (int)(unit - t * a.warps_per_token) * a.items_per_warp, last = first + a.items_per_warp;
    const int seq = a.seq[t], pos = a.pos[t];
    const Place place = find_place(seq, pos, a.pages, a.pages_ld, a.n_seq, a.n_cols, a.c);
    if (place.state == 1) return;
    if (place.state == 2 && lane == 0 && first == 0) raise_error(a.err, (uint32_t)t, (uint32_t)pos);
    const int half = a.rot / 2, kv_items = (a.n_kv + kHeads - 1) / kHeads, q_items = (a.n_q + kHeads - 1) / kHeads;
    float2 *const turn = turns[warp];
    if (first < q_items + kv_items) {
        for (int i = lane; i < half; i += 32) {
            // the angle less whole turns: what is left of 2^31 * inv_freq in FP64 is good to 2^-22 of a radian, of 2^20 * 1 to 2^-33
            const double angle = (double)pos * (double)a.inv_freq[i];
            const double whole = rint(angle * 0.15915494309189533577);
            float s, c;
            sincosf((float)fma(-whole, 2.4492935982947064e-16, fma(-whole, 6.283185307179586, angle)), &s, &c);
            turn[(i & 7) * kCols + (i >> 3)] = make_float2(c, s);
        }
    }
    __syncwarp();
    const bool turned = part * 8 < a.rot, low = part * 8 < half;
    const int partner = turned && !a.interleaved ? (low ? part + half / 8 : part - half / 8) : part;  // half is a multiple of 8
    // kind 0, 1, 2: queries, keys, values; `before` items and `heads_before` heads of other kinds come first
    auto take = [&](auto kindc, int before, int n_items, int heads_before, int n_heads) {
        constexpr int kind = decltype(kindc)::value;
        const int from = max(first - before, 0), to = min(last - before, n_items);
        if (from >= to) return;
        const float *const w = kind == 0 ? a.q_norm : a.k_norm;
        uint64_t by[4], cross[4];  // factors of an element and of its partner, as pairs
        if constexpr (kind != 2) {
            float x[8], y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 1.f, y[i] = 1.f;
            if (w != nullptr) load_run<float, 8>(w + part * 8, x), load_run<float, 8>(w + partner * 8, y);
            float2 cs[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = a.interleaved ? part * 4 + i / 2 : low ? part * 8 + i : part * 8 + i - half;
                cs[i] = turned ? turn[(e & 7) * kCols + (e >> 3)] : make_float2(1.f, 0.f);
                if (a.interleaved ? i % 2 == 0 : low) cs[i].y = -cs[i].y;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                by[i] = pair(x[2 * i] * cs[2 * i].x, x[2 * i + 1] * cs[2 * i + 1].x);
                cross[i] = a.interleaved ? pair(x[2 * i + 1] * cs[2 * i].y, x[2 * i] * cs[2 * i + 1].y) : pair(y[2 * i] * cs[2 * i].y, y[2 * i + 1] * cs[2 * i + 1].y);
            }
        }
        const T *src = static_cast<const T *>(a.qkv) + t * a.ld + (int64_t)(heads_before + from * kHeads + sub) * D + part * 8;
        for (int item = from; item < to; item += kBatch) {
            Words<8 * (int)sizeof(T)> raw[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (item + b < to && (item + b) * kHeads + sub < n_heads) raw[b] = load_words<8 * (int)sizeof(T)>(src + b * 32 * 8);
                else raw[b] = {};
            src += kBatch * 32 * 8;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                if (item + b >= to) break;
                const int head = (item + b) * kHeads + sub;
                const bool on = head < n_heads;
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(raw[b].w[i]);
                    else v[i] = __uint_as_float(i & 1 ? raw[b].w[i / 2] & 0xffff0000u : raw[b].w[i / 2] << 16);
                }
                if constexpr (kind != 2) {
                    uint64_t p[4], r[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] = pair(v[2 * i], v[2 * i + 1]);
                    float inv = 1.f;
                    if (w != nullptr) {
                        uint64_t sq = mul_pair(p[0], p[0]);
#pragma unroll
                        for (int i = 1; i < 4; ++i) sq = fma_pair(p[i], p[i], sq);
                        float sum, odd;
                        unpair(sq, sum, odd);
                        sum += odd;
#pragma unroll
                        for (int off = kLanes / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                        inv = rsqrtf(fmaf(sum, 1.0f / D, a.eps));
                    }
                    if (a.rot != 0) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint64_t other = a.interleaved ? pair(v[2 * i + 1], v[2 * i])
                                                                 : pair(__shfl_sync(0xffffffffu, v[2 * i], partner, kLanes), __shfl_sync(0xffffffffu, v[2 * i + 1], partner, kLanes));
                            r[i] = fma_pair(p[i], by[i], mul_pair(other, cross[i]));
                            if (!turned) r[i] = mul_pair(p[i], by[i]);  // as it is: nothing of a neighbour, not even 0 times an infinity
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) r[i] = mul_pair(p[i], by[i]);
                    }
                    const uint64_t inv2 = pair(inv, inv);
#pragma unroll
                    for (int i = 0; i < 4; ++i) unpair(mul_pair(r[i], inv2), v[2 * i], v[2 * i + 1]);
                }
                if constexpr (kind == 0) {
                    if (place.state == 2) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = qnan_f32();
                    }
                    if (on) store_bf16_run(a.q_out + t * a.q_ld + (int64_t)head * D + part * 8, v);
                } else if (place.state == 0) {
                    store_run<D, BITS>(kind == 1 ? a.c.k : a.c.v, kind == 1 ? a.c.k_sm : a.c.v_sm, kv_row(a.c, place.page, on ? head : 0, place.at), v, part, a.G, on);
                }
            }
        }
    };
    take(std::integral_constant<int, 0>{}, 0, q_items, 0, a.n_q);
    take(std::integral_constant<int, 1>{}, q_items, kv_items, a.n_q, a.n_kv);
    take(std::integral_constant<int, 2>{}, q_items + kv_items, kv_items, a.n_q + a.n_kv, a.n_kv);
}

constexpr int kReadThreads = 256, kReadTokens = 16;

struct ReadArgs {
    const int32_t *seq, *pos, *pages;
    int64_t pages_ld;
    int T, n_seq, n_cols, G, tokens;  // tokens a CTA
    KvView c;
    void *k_out, *v_out;
    uint32_t *err;
};

// The CTA's threads find the places of its tokens side by side, then read runs of sixteen elements (BF16: eight): neighbouring threads neighbouring runs of
// a row, four rows' loads in flight a thread.
template <typename T, int D, int BITS>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const __grid_constant__ ReadArgs a) {
    __shared__ int64_t rows[kReadTokens];  // row number of the token's first head; kSkip, kBad
    constexpr int64_t kSkip = -1, kBad = -2;
    constexpr int N = BITS == 16 ? 8 : 16, kBytes = N * BITS / 8, kRuns = D / N, kStep = kReadThreads / kRuns, kBatch = 4;
    behind_grid();
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
    const int tokens = (int)min((int64_t)a.tokens, a.T - t0);
    if ((int)threadIdx.x < tokens) {
        const int64_t t = t0 + threadIdx.x;
        const int pos = a.pos[t];
        const Place place = find_place(a.seq[t], pos, a.pages, a.pages_ld, a.n_seq, a.n_cols, a.c);
        if (place.state == 2) raise_error(a.err, (uint32_t)t, (uint32_t)pos);
        rows[threadIdx.x] = place.state == 0 ? kv_row(a.c, place.page, 0, place.at) : place.state == 1 ? kSkip : kBad;
    }
    __syncthreads();
    const int run = threadIdx.x % kRuns, heads = 2 * a.c.n_kv, group = run * N / a.G, groups = D / a.G;
    int token = 0, h = threadIdx.x / kRuns;
    while (h >= heads) h -= heads, ++token;
    while (token < tokens) {
        Words<kBytes> raw[kBatch];
        uint32_t sm[kBatch];
        int64_t row0[kBatch];
        T *to[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            row0[b] = token < tokens ? rows[token] : kSkip;
            const bool is_k = h < a.c.n_kv;
            const int head = is_k ? h : h - a.c.n_kv;
            to[b] = static_cast<T *>(is_k ? a.k_out : a.v_out) + (((t0 + token) * a.c.n_kv + head) * D + run * N);
            if (row0[b] >= 0) {
                const int64_t from = row0[b] + head * a.c.head_stride;
                raw[b] = load_words<kBytes>((is_k ? a.c.k : a.c.v) + from * (D * BITS / 8) + run * kBytes);
                if constexpr (BITS != 16) sm[b] = (is_k ? a.c.k_sm : a.c.v_sm)[from * groups + group];
            }
            h += kStep;
            while (h >= heads) h -= heads, ++token;
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (row0[b] == kSkip) continue;
            float v[N];
            if (row0[b] == kBad) {
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = qnan_f32();
            } else if constexpr (BITS == 16) {
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = __uint_as_float(e & 1 ? raw[b].w[e / 2] & 0xffff0000u : raw[b].w[e / 2] << 16);
            } else {
                const float s = __uint_as_float(sm[b] << 16), m = __uint_as_float(sm[b] & 0xffff0000u);
#pragma unroll
                for (int e = 0; e < N; ++e) {  // a code under the exponent of 2^23 is that number plus it
                    const uint32_t c = BITS == 8 ? __byte_perm(raw[b].w[e / 4], 0x4b000000u, 0x7540 + e % 4) : (raw[b].w[e / 8] >> (4 * (e % 8)) & 15u) | 0x4b000000u;
                    v[e] = fmaf(__uint_as_float(c) - 8388608.f, s, m);
                }
            }
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int e = 0; e < N; e += 4) *reinterpret_cast<float4 *>(to[b] + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            } else {
                store_bf16_run(to[b], v);
            }
        }
    }
}

template <typename T>
cudaError_t launch_write(const WriteArgs &a, int D, int bits, dim3 grid, cudaStream_t st) {
#define SXB_W(DD, BB) \
    if (D == DD && bits == BB) return launch_behind(qkv_write_kernel<T, DD, BB>, grid, kWriteThreads, 0, st, 1, a)
    SXB_W(64, 16); SXB_W(64, 8); SXB_W(64, 4);
    SXB_W(128, 16); SXB_W(128, 8); SXB_W(128, 4);
    SXB_W(256, 16); SXB_W(256, 8); SXB_W(256, 4);
#undef SXB_W
    return cudaErrorInvalidValue;
}
template <typename T>
cudaError_t launch_read(const ReadArgs &a, int D, int bits, unsigned grid, cudaStream_t st) {
#define SXB_R(DD, BB) \
    if (D == DD && bits == BB) return launch_behind(kv_read_kernel<T, DD, BB>, grid, kReadThreads, 0, st, 1, a)
    SXB_R(64, 16); SXB_R(64, 8); SXB_R(64, 4);
    SXB_R(128, 16); SXB_R(128, 8); SXB_R(128, 4);
    SXB_R(256, 16); SXB_R(256, 8); SXB_R(256, 4);
#undef SXB_R
    return cudaErrorInvalidValue;
}

int check_places(const char *fn, const int32_t *seq, const int32_t *pos, const int32_t *pages, int64_t pages_ld, int64_t n_cols, int64_t n_seq, int64_t T,
                 const SxbKvCache *c, const uint32_t *err) {
    SXB_CHECK(seq != nullptr && pos != nullptr && pages != nullptr && err != nullptr, fn, ": null pointer (seq=", (const void *)seq, ", pos=",
              (const void *)pos, ", pages=", (const void *)pages, ", err=", (const void *)err, ")");
    SXB_CHECK(T >= 1 && T <= kMaxTokens, fn, ": T = ", T, " tokens, expected 1..2^20");
    SXB_CHECK(n_seq >= 1 && n_seq <= (1 << 20), fn, ": n_seq = ", n_seq, ", expected 1..2^20");
    SXB_CHECK(n_cols >= 1 && pages_ld >= n_cols, fn, ": page table of ", n_cols, " columns with a stride of ", pages_ld);
    SXB_CHECK(n_cols <= ((1ll << 31) - 1024) / c->page, fn, ": ", n_cols, " pages of ", c->page, " tokens a sequence, positions end below 2^31 - 1024");
    return SXB_OK;
}

}  // namespace

int kv_view(const char *fn, const SxbKvCache *c, KvView *out) {
    SXB_CHECK(c != nullptr, fn, ": null cache");
    SXB_CHECK(c->bits == 16 || c->bits == 8 || c->bits == 4, fn, ": cache of ", c->bits, " bits unsupported (16 = BF16, 8 or 4)");
    SXB_CHECK(c->D == 64 || c->D == 128 || c->D == 256, fn, ": heads of ", c->D, " elements unsupported (64, 128 or 256)");
    SXB_CHECK(c->k != nullptr && c->v != nullptr, fn, ": null pointer (cache k=", c->k, ", v=", c->v, ")");
    SXB_CHECK(aligned16(c->k) && aligned16(c->v), fn, ": cache k and v must be 16-byte aligned");
    if (c->bits != 16) {
        SXB_CHECK((c->G == 32 || c->G == 64 || c->G == 128) && c->G <= c->D, fn, ": group size ", c->G, " unsupported (32, 64 or 128, at most D = ", c->D, ")");
        SXB_CHECK(c->k_sm != nullptr && c->v_sm != nullptr, fn, ": null pointer (cache k_sm=", (const void *)c->k_sm, ", v_sm=", (const void *)c->v_sm, ")");
        SXB_CHECK(aligned16(c->k_sm) && aligned16(c->v_sm), fn, ": cache k_sm and v_sm must be 16-byte aligned");
    }
    SXB_CHECK(c->n_pages >= 1 && c->n_pages < (1ll << 31), fn, ": n_pages = ", c->n_pages, ", expected 1..2^31 - 1");
    SXB_CHECK(c->n_kv >= 1 && c->n_kv <= 1024, fn, ": n_kv = ", c->n_kv, " heads, expected 1..1024");
    SXB_CHECK(is_pow2(c->page) && c->page >= 8 && c->page <= 4096, fn, ": pages of ", c->page, " tokens, expected a power of two of 8..4096");
    SXB_CHECK(c->page_stride >= 1 && c->head_stride >= 1 && c->row_stride >= 1 && c->page_stride < (1ll << 32) && c->head_stride < (1ll << 32) &&
                  c->row_stride <= (1ll << 22),
              fn, ": strides of ", c->page_stride, " / ", c->head_stride, " / ", c->row_stride, " rows (page / head / token), expected 1..2^32 - 1, of tokens up to 2^22");
    const int64_t last = (c->n_pages - 1) * c->page_stride + (c->n_kv - 1) * c->head_stride + (c->page - 1) * c->row_stride;
    SXB_CHECK((c->n_pages - 1) <= (1ll << 36) / c->page_stride && last < (1ll << 36) / (c->D * c->bits / 8), fn, ": keys of more than 2^36 bytes");
    *out = KvView{static_cast<uint8_t *>(c->k), static_cast<uint8_t *>(c->v), c->k_sm, c->v_sm, c->page_stride, c->head_stride, c->row_stride,
                  (int)c->n_pages, __builtin_ctzll((unsigned long long)c->page), (int)c->n_kv};
    return SXB_OK;
}

}  // namespace sxb

using namespace sxb;

extern "C" int sxb_attn_qkv_write(const SxbAttnQkvWriteArgs *args, sxb_stream_t stream) {
    const char *fn = "attn_qkv_write";
    SXB_CHECK(args != nullptr, fn, ": null argument block");
    const void *const qkv = args->qkv;
    void *const q_out = args->q_out;
    const SxbKvCache *const cache = args->cache;
    const int64_t ld = args->ld, T = args->T, n_q = args->n_q, rot = args->rot, q_ld = args->q_ld;
    const int act = args->act;
    WriteArgs a{};
    if (int rc = kv_view(fn, cache, &a.c)) return rc;
    if (int rc = check_places(fn, args->seq, args->pos, args->pages, args->pages_ld, args->n_cols, args->n_seq, T, cache, args->err)) return rc;
    SXB_CHECK(qkv != nullptr && q_out != nullptr, fn, ": null pointer (qkv=", qkv, ", q_out=", q_out, ")");
    SXB_CHECK(act_ok(act), fn, ": unsupported activation dtype ", act);
    SXB_CHECK(n_q >= 1 && n_q <= 1024, fn, ": n_q = ", n_q, " heads, expected 1..1024");
    const int64_t D = cache->D, heads = n_q + 2 * cache->n_kv, es = act_bytes(act);
    SXB_CHECK(ld >= heads * D && ld <= (1ll << 32) && q_ld >= n_q * D && q_ld <= (1ll << 32), fn, ": row strides ", ld, " and ", q_ld, ", rows have ",
              heads * D, " and ", n_q * D, " elements");
    SXB_CHECK(aligned16(qkv) && aligned16(q_out) && ld * es % 16 == 0 && q_ld % 8 == 0, fn, ": rows of qkv and q_out must be 16-byte aligned");
    SXB_CHECK(apart(qkv, ((T - 1) * ld + heads * D) * es, q_out, ((T - 1) * q_ld + n_q * D) * 2), fn, ": q_out [", q_out, "] overlaps qkv [", qkv, "]");
    SXB_CHECK(args->inv_freq != nullptr || rot == 0, fn, ": rot = ", rot, " without inv_freq");
    SXB_CHECK(rot >= 0 && rot <= D && rot % 16 == 0, fn, ": rot = ", rot, ", expected a multiple of 16 of 0..", D);
    SXB_CHECK(aligned16(args->q_norm) && aligned16(args->k_norm), fn, ": norm weights must be 16-byte aligned");
    SXB_CHECK((args->q_norm == nullptr && args->k_norm == nullptr) || (args->eps > 0.f && args->eps < 1e30f), fn, ": eps must be finite and positive");
    a.qkv = qkv, a.ld = ld, a.n_q = (int)n_q, a.n_kv = (int)cache->n_kv, a.rot = (int)rot, a.interleaved = args->interleaved != 0;
    a.q_norm = args->q_norm, a.k_norm = args->k_norm, a.inv_freq = args->inv_freq, a.eps = args->eps;
    a.seq = args->seq, a.pos = args->pos, a.pages = args->pages, a.pages_ld = args->pages_ld, a.n_seq = (int)args->n_seq, a.n_cols = (int)args->n_cols;
    a.G = (int)(cache->bits == 16 ? D : cache->G), a.q_out = static_cast<uint16_t *>(q_out), a.q_ld = q_ld, a.err = args->err;
    // few tokens: an item a warp, so that the SMs share them; many: a warp has all of its token's and computes the angles once
    const int64_t per = 256 / D, items = (n_q + per - 1) / per + 2 * ((cache->n_kv + per - 1) / per);
    a.items_per_warp = (int)std::max<int64_t>(1, std::min(items, items * T / (24 * (int64_t)sm_count())));
    a.warps_per_token = (int)((items + a.items_per_warp - 1) / a.items_per_warp), a.T = T;
    const dim3 grid((unsigned)((T * a.warps_per_token + kWriteWarps - 1) / kWriteWarps));
    auto st = static_cast<cudaStream_t>(stream);
    if (act == SXB_ACT_F32) launch_write<float>(a, (int)D, cache->bits, grid, st);
    else launch_write<uint16_t>(a, (int)D, cache->bits, grid, st);
    SXB_CHECK_LAUNCH(fn, " ", act_name(act), " T=", T, " n_q=", n_q, " n_kv=", cache->n_kv, " D=", D, " bits=", cache->bits);
    return SXB_OK;
}

extern "C" int sxb_kv_read(const SxbKvReadArgs *args, sxb_stream_t stream) {
    const char *fn = "kv_read";
    SXB_CHECK(args != nullptr, fn, ": null argument block");
    const SxbKvCache *const cache = args->cache;
    void *const k_out = args->k_out, *const v_out = args->v_out;
    const int64_t T = args->T;
    const int out_act = args->out_act;
    ReadArgs a{};
    if (int rc = kv_view(fn, cache, &a.c)) return rc;
    if (int rc = check_places(fn, args->seq, args->pos, args->pages, args->pages_ld, args->n_cols, args->n_seq, T, cache, args->err)) return rc;
    SXB_CHECK(k_out != nullptr && v_out != nullptr, fn, ": null pointer (k_out=", k_out, ", v_out=", v_out, ")");
    SXB_CHECK(act_ok(out_act), fn, ": unsupported output dtype ", out_act);
    SXB_CHECK(aligned16(k_out) && aligned16(v_out), fn, ": k_out and v_out must be 16-byte aligned");
    const int64_t D = cache->D, bytes = T * cache->n_kv * D * act_bytes(out_act);
    SXB_CHECK(apart(k_out, bytes, v_out, bytes), fn, ": v_out [", v_out, "] overlaps k_out [", k_out, "]");
    a.seq = args->seq, a.pos = args->pos, a.pages = args->pages, a.pages_ld = args->pages_ld, a.n_seq = (int)args->n_seq, a.n_cols = (int)args->n_cols;
    a.G = (int)(cache->bits == 16 ? D : cache->G), a.k_out = k_out, a.v_out = v_out, a.err = args->err;
    a.T = (int)T;
    a.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(kReadTokens, T / (8 * (int64_t)sm_count())));
    const unsigned grid = (unsigned)((T + a.tokens - 1) / a.tokens);
    auto st = static_cast<cudaStream_t>(stream);
    if (out_act == SXB_ACT_F32) launch_read<float>(a, (int)D, cache->bits, grid, st);
    else launch_read<uint16_t>(a, (int)D, cache->bits, grid, st);
    SXB_CHECK_LAUNCH(fn, " ", act_name(out_act), " T=", T, " n_kv=", cache->n_kv, " D=", D, " bits=", cache->bits);
    return SXB_OK;
}
