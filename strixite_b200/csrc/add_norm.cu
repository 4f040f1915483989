// The residual's addition and root-mean-square norm between two sublayers, with the outputs that the next product reads: s = x + y as stored, n = s /
// sqrt(mean(s^2) + eps) * weight, n as BF16 or as e4m3 codes with a scale for every block of 128 (f8.cuh).  And the same codes, in blocks of 128 x 128, of a weight.
//
// One pass: a CTA has a row in registers between the sum of its squares and its codes, so x and y are read and s and the codes written once.  The arithmetic is by pairs: one after the other,
// with divisions for what is a product here, the instructions were what bounded it (16384 x 4096: 87 us for 81).

#include "f8.cuh"
#include "skinny_mma.cuh"

#include <type_traits>

namespace sxb {
namespace {

constexpr int kVec = 8;           // elements of a thread's piece of a row: sixteen neighbouring threads have a block
constexpr int64_t kMaxD = 32768;

struct NormArgs {
    const void *x, *y;
    const float *weight;
    void *total;
    uint16_t *out;
    uint8_t *codes;
    float *scales;
    int64_t x_ld, y_ld, total_ld, out_ld, codes_ld, scales_ld;
    int64_t T;
    int d, normed;
    float eps, inv_d;
};

__device__ inline void load8(const float *p, float (&v)[kVec]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ inline void load8(const uint16_t *p, float (&v)[kVec]) {
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ inline void store8(float *p, const float (&v)[kVec]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ inline void store8(uint16_t *p, const float (&v)[kVec]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// 1 / v to the last place, for normal numbers whose reciprocals are.
__device__ inline float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// A block's values v, `most` their largest magnitude, to what its codes are rounded from: the nearest FP32 of 448 v / most (a quotient by Newton's method: v times an approximate reciprocal, put right
// by its remainder, which one multiply-add gives; 448 comes in with the correction, so that nothing is rounded before it), whatever the row's factor r.  A value that stands between two codes stays
// there and goes to the even one, as the definition says; one that is not a tie but within 2^-25 of it may round as the tie.  Where the scale is its least, v r / scale.
__device__ inline void f8_codes(float (&v)[kVec], float most, float exact, float r, float scale) {
    const bool least = !(exact >= kF8Least);  // zeros and NaN too
    const float shrink = most >= 0x1p100f ? 0x1p-40f : 1.f, by = most * shrink;
    const float inv = least ? __fdiv_rn(r, scale) : reciprocal(by), top = least ? 1.f : kF8Top * shrink, put = least ? 0.f : inv * top;
    const uint64_t tops = pair(top, top), invs = pair(inv, inv), minus = pair(least ? 0.f : -by, least ? 0.f : -by), puts = pair(put, put);
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {
        const uint64_t x = pair(v[i], v[i + 1]), q = mul_pair(x, invs);
        unpair(fma_pair(q, tops, mul_pair(fma_pair(q, minus, x), puts)), v[i], v[i + 1]);
    }
}
// The values as they are stored in TX.
template <typename TX>
__device__ inline void as_kept(float (&v)[kVec]) {
    if constexpr (sizeof(TX) == 2)
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const uint32_t w = bf16_pair(v[i], v[i + 1]);
            v[i] = __uint_as_float(w << 16), v[i + 1] = __uint_as_float(w & 0xffff0000u);
        }
}

// Eight elements as they lie in memory.
template <typename T>
struct Raw8 {
    uint4 v[sizeof(T) / 2];
    __device__ inline void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    __device__ inline void clear() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ inline float at(int i) const {
        const uint32_t w[4] = {v[i / (16 / (int)sizeof(T))].x, v[i / (16 / (int)sizeof(T))].y, v[i / (16 / (int)sizeof(T))].z, v[i / (16 / (int)sizeof(T))].w};
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i % 4]);
        else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
};

// Y: 0 = none, 1 = BF16, 2 = FP32.  NV: pieces of a row that a thread has, blockDim.x apart (a multiple of 32, so that blocks stay with sixteen lanes).  LOOP: a CTA goes on to further rows, the
// next one's x and y on their way; else it has blockDim.y rows, of a warp each if there are several.
template <typename TX, int Y, int NV, bool LOOP>
__global__ void __launch_bounds__(LOOP ? 512 : 1024) add_norm_kernel(const NormArgs a) {
    using TY = std::conditional_t<Y == 2, float, uint16_t>;
    behind_grid();
    __shared__ float parts[2][32];
    Raw8<TX> x[NV];
    Raw8<TY> y[NV];
    auto ask = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = (j * (int)blockDim.x + (int)threadIdx.x) * kVec;
            if (at < a.d) {
                x[j].load(static_cast<const TX *>(a.x) + row * a.x_ld + at);
                if constexpr (Y != 0) y[j].load(static_cast<const TY *>(a.y) + row * a.y_ld + at);
            } else {
                x[j].clear();
                if constexpr (Y != 0) y[j].clear();
            }
        }
    };
    const int64_t row0 = LOOP ? blockIdx.x : (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (!LOOP && row0 >= a.T) return;
    ask(row0);
    int turn = 0;
    for (int64_t row = row0; row < a.T; row += gridDim.x, turn ^= 1) {
        float s[NV][kVec];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = (j * (int)blockDim.x + (int)threadIdx.x) * kVec;
#pragma unroll
            for (int i = 0; i < kVec; ++i) s[j][i] = Y != 0 ? x[j].at(i) + y[j].at(i) : x[j].at(i);
            if constexpr (Y != 0) {
                as_kept<TX>(s[j]);
                if (a.total != nullptr && at < a.d) store8(static_cast<TX *>(a.total) + row * a.total_ld + at, s[j]);
            }
        }
        if (LOOP && row + gridDim.x < a.T) ask(row + gridDim.x);
        float r = 1.f;
        if (a.normed) {
            uint64_t squares[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < kVec; i += 2) {
                    const uint64_t v = pair(s[j][i], s[j][i + 1]);
                    squares[i / 2 & 1] = fma_pair(v, v, squares[i / 2 & 1]);
                }
            float sum, other;
            unpair(add_pair(squares[0], squares[1]), sum, other);
            sum += other;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if (blockDim.x > 32) {
                if ((threadIdx.x & 31) == 0) parts[turn][threadIdx.x >> 5] = sum;
                __syncthreads();
                const int warps = (int)blockDim.x >> 5, lane = threadIdx.x & 31;
                sum = lane < warps ? parts[turn][lane] : 0.f;
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            }
            r = rsqrtf(fmaf(sum, a.inv_d, a.eps));
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = (j * (int)blockDim.x + (int)threadIdx.x) * kVec;
            // s times the weight; the row's factor r, which a block's codes do not depend on, comes to the scale (and out) alone
            if (at < a.d) {
                if (a.weight != nullptr) {
                    float w[kVec];
                    load8(a.weight + at, w);
#pragma unroll
                    for (int i = 0; i < kVec; i += 2) unpair(mul_pair(pair(s[j][i], s[j][i + 1]), pair(w[i], w[i + 1])), s[j][i], s[j][i + 1]);
                }
                if (a.out != nullptr) {
                    float n[kVec];
#pragma unroll
                    for (int i = 0; i < kVec; i += 2) unpair(mul_pair(pair(s[j][i], s[j][i + 1]), pair(r, r)), n[i], n[i + 1]);
                    store8(a.out + row * a.out_ld + at, n);
                }
            }
            if (a.codes != nullptr) {
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < kVec; ++i) most = max_nan(most, fabsf(s[j][i]));
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, off));
                const float exact = __fdiv_rn(most * r, kF8Top), scale = f8_scale(exact);
                if (at < a.d) {
                    f8_codes(s[j], most, exact, r, scale);
                    const uint2 c = make_uint2(f8_quad(s[j][0], s[j][1], s[j][2], s[j][3]), f8_quad(s[j][4], s[j][5], s[j][6], s[j][7]));
                    *reinterpret_cast<uint2 *>(a.codes + row * a.codes_ld + at) = c;
                    if (at % kF8Block == 0) a.scales[row * a.scales_ld + at / kF8Block] = scale;
                }
            }
        }
        if (!LOOP) break;
    }
}

// A thread has one piece of a row, the shortest way through it; short rows are a warp's, eight of them a CTA's.  Many long rows keep the CTAs on the machine and two pieces a thread: what
// bounds a CTA that comes and goes is its chain of loads, sums and stores (16384 x 4096, BF16 x and y: 80.9 us, so 77.4, the bytes at the copy's rate 71.8; 8192 x 8192 86.9, 79.3; x alone
// 61.8, 52.1), unless y is FP32 (90.7, 93.3: the bytes take 92.4 at that rate).  16384 x 256: 17.9 with a CTA a row.
template <typename TX, int Y>
cudaError_t launch_norm(const NormArgs &a, cudaStream_t st) {
    const int pieces = a.d / kVec;
    auto go = [&](auto kern, int nv, int rows, int64_t grid) {
        return launch_behind(kern, dim3((unsigned)grid), dim3((unsigned)(((pieces + nv - 1) / nv + 31) / 32 * 32), rows), 0, st, 1, a);
    };
    if (pieces <= 32) return go(add_norm_kernel<TX, Y, 1, false>, 1, 8, (a.T + 7) / 8);
    const int64_t places = (int64_t)sm_count() * 4;
    if (Y != 2 && pieces >= 256 && pieces <= 1024 && a.T >= 4 * places) return go(add_norm_kernel<TX, Y, 2, true>, 2, 1, places);
    if (pieces > 2048) return go(add_norm_kernel<TX, Y, 4, false>, 4, 1, a.T);
    if (pieces > 1024) return go(add_norm_kernel<TX, Y, 2, false>, 2, 1, a.T);
    return go(add_norm_kernel<TX, Y, 1, false>, 1, 1, a.T);
}

// Weights are quantized once: 131072 x 4096 takes 470 to 515 us from FP32 (410 at the copy's rate) and 560 to 580 from BF16 (246); not profiled.
// A CTA has a block of 128 x 128: a thread half a row of it, in registers between the largest magnitude and the codes.
template <typename TW>
__global__ void __launch_bounds__(256) quantize_f8_kernel(const TW *__restrict__ w, int64_t N, int64_t K, int64_t kb, uint8_t *__restrict__ q,
                                                          float *__restrict__ scale, uint32_t *err) {
    __shared__ uint32_t parts[8];
    const int64_t rb = blockIdx.x / kb, cb = blockIdx.x % kb;
    // sixteen neighbouring threads read a row's 128 columns, eight rows... a thread has the columns at 8 (t % 16) of the rows t / 16, t / 16 + 16, ...
    const int64_t col = cb * kF8Block + (threadIdx.x & 15) * kVec, row0 = rb * kF8Block + (threadIdx.x >> 4);
    float v[8][kVec];
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t row = row0 + 16 * j;
        if (row < N && col < K) load8(w + row * K + col, v[j]);
        else
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[j][i] = 0.f;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            most = max(most, magnitude(v[j][i]));
            if (magnitude(v[j][i]) >= 0x7f800000u) raise_error(err, (uint32_t)row, (uint32_t)(col + i));
        }
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, parts[i]);
    const float largest = __uint_as_float(most), exact = __fdiv_rn(largest, kF8Top), s = f8_scale(exact);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t row = row0 + 16 * j;
        if (row >= N || col >= K) continue;
        f8_codes(v[j], largest, exact, 1.f, s);
        *reinterpret_cast<uint2 *>(q + row * K + col) = make_uint2(f8_quad(v[j][0], v[j][1], v[j][2], v[j][3]), f8_quad(v[j][4], v[j][5], v[j][6], v[j][7]));
    }
}

}  // namespace
}  // namespace sxb

using namespace sxb;

extern "C" int sxb_add_norm(const SxbAddNormArgs *args, sxb_stream_t stream) {
    const char *fn = "add_norm";
    SXB_CHECK(args != nullptr, fn, ": null argument block");
    const SxbAddNormArgs &g = *args;
    const int64_t T = g.T, d = g.d;
    SXB_CHECK(g.x != nullptr, fn, ": null pointer (x)");
    SXB_CHECK(act_ok(g.act) && (g.y == nullptr || act_ok(g.y_act)), fn, ": unsupported dtypes ", g.act, " of x, ", g.y_act, " of y");
    SXB_CHECK(T >= 1 && T <= (1 << 24), fn, ": T = ", T, " rows, expected 1..2^24");
    SXB_CHECK(d >= 16 && d <= kMaxD && d % 16 == 0, fn, ": d = ", d, ", expected a multiple of 16 of 16..", kMaxD);
    SXB_CHECK(g.total != nullptr || g.out != nullptr || g.codes != nullptr, fn, ": no output");
    SXB_CHECK(g.total == nullptr || g.y != nullptr, fn, ": a total without y");
    SXB_CHECK((g.codes == nullptr) == (g.scales == nullptr), fn, ": codes and scales come together (codes=", (const void *)g.codes, ", scales=", (const void *)g.scales, ")");
    SXB_CHECK(g.normed || g.weight == nullptr, fn, ": a weight without the norm");
    SXB_CHECK(!g.normed || (g.eps >= 0x1p-100f && g.eps < 1e30f), fn, ": eps must be finite and at least 2^-100");
    SXB_CHECK(aligned16(g.weight), fn, ": the weight must be 16-byte aligned");
    const int64_t es = act_bytes(g.act), ys = g.y != nullptr ? act_bytes(g.y_act) : 0, blocks = (d + kF8Block - 1) / kF8Block;
    struct Rows {
        const char *name;
        const void *p;
        int64_t ld, n, es;
        int64_t bytes(int64_t T) const { return ((T - 1) * ld + n) * es; }
    };
    const Rows rows[6] = {{"x", g.x, g.x_ld, d, es},         {"y", g.y, g.y_ld, d, ys},         {"total", g.total, g.total_ld, d, es},
                          {"out", g.out, g.out_ld, d, 2}, {"codes", g.codes, g.codes_ld, d, 1}, {"scales", g.scales, g.scales_ld, blocks, 4}};
    for (const Rows &r : rows) {
        if (r.p == nullptr) continue;
        SXB_CHECK(r.ld >= r.n && r.ld <= (1ll << 32), fn, ": row stride ", r.ld, " of ", r.name, ", rows have ", r.n, " elements");
        SXB_CHECK(r.n == blocks && r.es == 4 && r.p == (const void *)g.scales ? reinterpret_cast<uintptr_t>(r.p) % 4 == 0 : aligned16(r.p) && r.ld * r.es % 16 == 0, fn,
                  ": rows of ", r.name, " must be 16-byte aligned (scales: 4)");
    }
    // an element of total is written by the thread that has read those of x and y: it may lie on either, row for row
    for (int o = 2; o < 6; ++o)
        for (int i = 0; i < o; ++i) {
            const Rows &a = rows[o], &b = rows[i];
            if (a.p == nullptr || b.p == nullptr || (o == 2 && i < 2 && a.p == b.p && a.ld == b.ld && a.es == b.es)) continue;
            SXB_CHECK(apart(a.p, a.bytes(T), b.p, b.bytes(T)), fn, ": ", a.name, " [", a.p, "] overlaps ", b.name, " [", b.p, "]");
        }
    if (g.weight != nullptr)
        for (int o = 2; o < 6; ++o)
            SXB_CHECK(rows[o].p == nullptr || apart(rows[o].p, rows[o].bytes(T), g.weight, d * 4), fn, ": ", rows[o].name, " overlaps the weight");
    NormArgs a{};
    a.x = g.x, a.y = g.y, a.weight = g.weight, a.total = g.total, a.out = static_cast<uint16_t *>(g.out), a.codes = g.codes, a.scales = g.scales;
    a.x_ld = g.x_ld, a.y_ld = g.y_ld, a.total_ld = g.total_ld, a.out_ld = g.out_ld, a.codes_ld = g.codes_ld, a.scales_ld = g.scales_ld;
    a.T = T, a.d = (int)d, a.normed = g.normed != 0, a.eps = g.eps, a.inv_d = 1.f / (float)d;
    auto st = static_cast<cudaStream_t>(stream);
    const int y = g.y == nullptr ? 0 : g.y_act == SXB_ACT_F32 ? 2 : 1;
    cudaError_t e;
    if (g.act == SXB_ACT_F32) e = y == 0 ? launch_norm<float, 0>(a, st) : y == 1 ? launch_norm<float, 1>(a, st) : launch_norm<float, 2>(a, st);
    else e = y == 0 ? launch_norm<uint16_t, 0>(a, st) : y == 1 ? launch_norm<uint16_t, 1>(a, st) : launch_norm<uint16_t, 2>(a, st);
    SXB_CUDA(e, fn, ": launching T=", T, " d=", d);
    SXB_CHECK_LAUNCH(fn, " ", act_name(g.act), " T=", T, " d=", d);
    return SXB_OK;
}

extern "C" int sxb_quantize_f8(const void *w, int act, int64_t N, int64_t K, uint8_t *q, float *scale, uint32_t *err, sxb_stream_t stream) {
    const char *fn = "quantize_f8";
    SXB_CHECK(w != nullptr && q != nullptr && scale != nullptr && err != nullptr, fn, ": null pointer (w=", w, ", q=", (const void *)q, ", scale=", (const void *)scale,
              ", err=", (const void *)err, ")");
    SXB_CHECK(act_ok(act), fn, ": unsupported dtype ", act, " of w");
    SXB_CHECK(N >= 1 && N <= (1 << 24) && K >= 16 && K <= (1 << 20) && K % 16 == 0, fn, ": N = ", N, ", K = ", K, " (K a multiple of 16)");
    SXB_CHECK(aligned16(w) && aligned16(q) && reinterpret_cast<uintptr_t>(scale) % 4 == 0, fn, ": w and q must be 16-byte aligned, scales 4-byte");
    const int64_t kb = (K + kF8Block - 1) / kF8Block, blocks = (N + kF8Block - 1) / kF8Block * kb;
    SXB_CHECK(blocks <= 0x7fffffff, fn, ": ", blocks, " blocks");
    const struct {
        const char *name;
        const void *p;
        int64_t n;
    } of[4] = {{"w", w, N * K * act_bytes(act)}, {"err", err, 12}, {"q", q, N * K}, {"scale", scale, 4 * blocks}};
    for (int o = 1; o < 4; ++o)
        for (int i = 0; i < o; ++i) SXB_CHECK(apart(of[o].p, of[o].n, of[i].p, of[i].n), fn, ": ", of[o].name, " [", of[o].p, "] overlaps ", of[i].name, " [", of[i].p, "]");
    auto st = static_cast<cudaStream_t>(stream);
    if (act == SXB_ACT_F32) quantize_f8_kernel<<<(unsigned)blocks, 256, 0, st>>>(static_cast<const float *>(w), N, K, kb, q, scale, err);
    else quantize_f8_kernel<<<(unsigned)blocks, 256, 0, st>>>(static_cast<const uint16_t *>(w), N, K, kb, q, scale, err);
    SXB_CHECK_LAUNCH(fn, " N=", N, " K=", K);
    return SXB_OK;
}
