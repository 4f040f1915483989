// Matrix product of e4m3 codes with an FP32 scale for every block of 128 along k (activations) or 128 x 128 (weights), f8.cuh:
//   y[m, n] = sum over blocks b of k:  (xs[m, b] ws[n / 128, b]) * sum over k in b:  x[m, k] w[n, k]
// The inner sums are exact products of codes added up in FP32 by the tensor cores, from zero for every block; the threads scale them and add them up in FP32.

#include "linear_f8.cuh"

namespace sxb {
namespace {

// ---- up to eight rows of x over a weight that is not large ------------------------------------------------------------------------
//
// A CTA has 16 weight rows, its warps a run of k each: every warp asks for AHEAD blocks of k at once, codes and scales of both operands, and the parts are added up in shared
// memory in the warps' order.  What bounds it is the round trips: launch, operands, parts (6144 x 4096, one row of x: 7.8 us with the weights in HBM; the form on tcgen05 9.7, from
// 2^26 codes on that one is ahead).

constexpr int kRows = 16, kTokens = 8;  // weight rows and rows of x of an MMA

// d += 16 weight rows x 8 rows of x x 32 k of codes: exact products, FP32 sums.
__device__ inline void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ inline uint4 load16(const uint8_t *p, bool there) { return there ? __ldg(reinterpret_cast<const uint4 *>(p)) : make_uint4(0u, 0u, 0u, 0u); }
__device__ inline uint4 stream16(const uint8_t *p, bool there) {  // read once: not kept in L1
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (there) asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// k inside a block is permuted alike on both operands: lane (g = lane / 4, c = lane % 4) holds the sixteen codes at 16 c and at 64 + 16 c of its weight rows g and
// g + 8 and of its row g of x, four MMAs' worth.
struct Block {
    uint4 lo[2], hi[2], x[2];  // of weight rows g and g + 8, of x
    float ws, xs[2];           // scales: the weight's, those of rows 2 c and 2 c + 1 of x
};

template <int kWarps, int AHEAD>
__global__ void __launch_bounds__(32 * kWarps) f8_rows_kernel(const F8Args a) {
    behind_grid();
    __shared__ float parts[kWarps][kTokens][kRows + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int n0 = blockIdx.x * kRows, kb0 = (int)((int64_t)a.kb * warp / kWarps), kb1 = (int)((int64_t)a.kb * (warp + 1) / kWarps);
    const bool lo = n0 + g < a.N, hi = n0 + g + 8 < a.N, there = g < a.M;
    const uint8_t *const w = a.w + (int64_t)(n0 + g) * a.K + 16 * c, *const w8 = w + 8 * a.K, *const x = a.x + g * a.x_ld + 16 * c;
    const float *const ws = a.ws + (int64_t)(n0 / kF8Block) * a.kb, *const xs = a.xs + 2 * c * a.xs_ld;
    float acc[4] = {};
    for (int b0 = kb0; b0 < kb1; b0 += AHEAD) {
        Block k[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int64_t at = (int64_t)(b0 + i) * kF8Block;
            const bool v0 = b0 + i < kb1 && at + 16 * c < a.K, v1 = b0 + i < kb1 && at + 64 + 16 * c < a.K;
            k[i].lo[0] = stream16(w + at, lo && v0), k[i].lo[1] = stream16(w + at + 64, lo && v1);
            k[i].hi[0] = stream16(w8 + at, hi && v0), k[i].hi[1] = stream16(w8 + at + 64, hi && v1);
            k[i].x[0] = load16(x + at, there && v0), k[i].x[1] = load16(x + at + 64, there && v1);
            k[i].xs[0] = b0 + i < kb1 && 2 * c < a.M ? __ldg(xs + b0 + i) : 0.f;
            k[i].xs[1] = b0 + i < kb1 && 2 * c + 1 < a.M ? __ldg(xs + a.xs_ld + b0 + i) : 0.f;
            k[i].ws = b0 + i < kb1 ? __ldg(ws + b0 + i) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            float d[4] = {};
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                mma_e4m3(d, k[i].lo[v].x, k[i].hi[v].x, k[i].lo[v].y, k[i].hi[v].y, k[i].x[v].x, k[i].x[v].y);
                mma_e4m3(d, k[i].lo[v].z, k[i].hi[v].z, k[i].lo[v].w, k[i].hi[v].w, k[i].x[v].z, k[i].x[v].w);
            }
            const float s0 = k[i].xs[0] * k[i].ws, s1 = k[i].xs[1] * k[i].ws;
            acc[0] = fmaf(d[0], s0, acc[0]), acc[1] = fmaf(d[1], s1, acc[1]), acc[2] = fmaf(d[2], s0, acc[2]), acc[3] = fmaf(d[3], s1, acc[3]);
        }
    }
    parts[warp][2 * c][g] = acc[0], parts[warp][2 * c + 1][g] = acc[1], parts[warp][2 * c][g + 8] = acc[2], parts[warp][2 * c + 1][g + 8] = acc[3];
    __syncthreads();
    const int n = n0 + threadIdx.x % kRows, m = threadIdx.x / kRows;  // kWarps >= 4: a thread an output
    if (m < kTokens && n < a.N && m < a.M) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) sum += parts[i][m][threadIdx.x % kRows];
        if (a.f32) static_cast<float *>(a.y)[m * a.y_ld + n] = sum;
        else static_cast<uint16_t *>(a.y)[m * a.y_ld + n] = f32_to_bf16_bits(sum);
    }
}

// Warps of a CTA, and blocks that one asks for at once.  Many tiles hide a round trip behind one another: few warps a tile, few blocks (16384 x 4096, one row of x: 15.0 us, sixteen
// warps by fours 26.2; 65536 x 512: 10.0, eight by fours 28.7).  Few tiles want all their k on its way at once (1024 x 8192: 5.2 us, four warps by twos 19.1; 4096 x 4096: eight by
// fours 5.9, by ones 7.1), but no more registers than that takes (2048 x 2048: sixteen by ones 2.4, by fours 3.9; 6144 x 4096, whose 384 CTAs then are all there: eight by ones 7.8,
// by fours 8.4).
cudaError_t launch_rows(const F8Args &a, cudaStream_t st) {
    const unsigned tiles = (unsigned)((a.N + kRows - 1) / kRows);
    auto go = [&](auto kern, int warps) { return launch_behind(kern, dim3(tiles), dim3(32 * warps), 0, st, 1, a); };
    if (tiles >= 512) return a.kb <= 4 ? go(f8_rows_kernel<4, 1>, 4) : go(f8_rows_kernel<4, 2>, 4);
    if (tiles >= 320 || a.kb < 8) return go(f8_rows_kernel<8, 1>, 8);
    return a.kb >= 64 ? go(f8_rows_kernel<16, 4>, 16) : a.kb >= 24 ? go(f8_rows_kernel<8, 4>, 8) : go(f8_rows_kernel<16, 1>, 16);
}

}  // namespace
}  // namespace sxb

using namespace sxb;

extern "C" int sxb_linear_f8(const SxbLinearF8Args *args, sxb_stream_t stream) {
    const char *fn = "linear_f8";
    SXB_CHECK(args != nullptr, fn, ": null argument block");
    const SxbLinearF8Args &g = *args;
    SXB_CHECK(g.w != nullptr, fn, ": null weight");
    const int64_t M = g.M, N = g.w->N, K = g.w->K, kb = (K + kF8Block - 1) / kF8Block;
    SXB_CHECK(g.x != nullptr && g.x_scale != nullptr && g.y != nullptr && g.w->q != nullptr && g.w->scale != nullptr, fn, ": null pointer (x=", (const void *)g.x, ", x_scale=",
              (const void *)g.x_scale, ", y=", g.y, ", w->q=", (const void *)g.w->q, ", w->scale=", (const void *)g.w->scale, ")");
    SXB_CHECK(M >= 1 && M <= (1 << 20), fn, ": M (rows of x) = ", M, ", expected 1..2^20");
    SXB_CHECK(N >= 1 && N <= (1 << 24) && K >= 16 && K <= (1 << 20) && K % 16 == 0, fn, ": N = ", N, ", K = ", K, " (N up to 2^24, K a multiple of 16 up to 2^20)");
    SXB_CHECK(g.out_act == SXB_ACT_BF16 || g.out_act == SXB_ACT_F32, fn, ": output dtype ", g.out_act, " unsupported (BF16 or F32)");
    SXB_CHECK(g.x_ld >= K && g.x_ld <= (1ll << 32) && g.xs_ld >= kb && g.xs_ld <= (1ll << 32) && g.y_ld >= N && g.y_ld <= (1ll << 32), fn, ": row strides ", g.x_ld, ", ", g.xs_ld,
              " and ", g.y_ld, ", rows have ", K, ", ", kb, " and ", N, " elements");
    SXB_CHECK(aligned16(g.x) && g.x_ld % 16 == 0 && aligned16(g.w->q), fn, ": rows of x and of the weight's codes must be 16-byte aligned");
    const int64_t os = act_bytes(g.out_act);
    SXB_CHECK(reinterpret_cast<uintptr_t>(g.y) % os == 0 && reinterpret_cast<uintptr_t>(g.x_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(g.w->scale) % 4 == 0, fn,
              ": y and the scales must be aligned to their types");
    const int64_t yb = ((M - 1) * g.y_ld + N) * os;
    SXB_CHECK(apart(g.y, yb, g.x, (M - 1) * g.x_ld + K) && apart(g.y, yb, g.x_scale, ((M - 1) * g.xs_ld + kb) * 4) && apart(g.y, yb, g.w->q, N * K) &&
                  apart(g.y, yb, g.w->scale, (N + kF8Block - 1) / kF8Block * kb * 4),
              fn, ": y [", g.y, ", +", yb, " B) overlaps x, the weight or their scales");
    F8Args a{};
    a.x = g.x, a.w = g.w->q, a.xs = g.x_scale, a.ws = g.w->scale, a.y = g.y, a.x_ld = g.x_ld, a.xs_ld = g.xs_ld, a.y_ld = g.y_ld, a.K = K;
    a.M = (int)M, a.N = (int)N, a.kb = (int)kb, a.f32 = g.out_act == SXB_ACT_F32;
    auto st = static_cast<cudaStream_t>(stream);
    if (M > kTokens || N * K > (1ll << 26)) return linear_f8_tc(fn, a, st);
    const cudaError_t e = launch_rows(a, st);
    SXB_CUDA(e, fn, ": launching M=", M, " N=", N, " K=", K);
    SXB_CHECK_LAUNCH(fn, " M=", M, " N=", N, " K=", K);
    return SXB_OK;
}
