// Matrix product of e4m3 codes with an FP32 scale for every block of 128 along k (activations) or 128 x 128 (weights), f8.cuh:
//   y[m, n] = sum over blocks b of k:  (xs[m, b] ws[n / 128, b]) * sum over k in b:  x[m, k] w[n, k]
// The inner sums are exact products of codes added up in FP32 by the tensor cores, from zero for every block; the threads scale them and add them up in FP32.

#include "linear_f8.cuh"

namespace sxb {
namespace {

// ---- few rows: the weights stream through the registers -------------------------------------------------------------------------

constexpr int kRows = 16, kTokens = 8, kWarps = 8;  // weight rows and tokens of an MMA; warps of a CTA, which share out k

// d += 16 weight rows x 8 tokens x 32 k of codes: exact products, FP32 sums.
__device__ inline void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ inline uint4 load16(const uint8_t *p, bool there) { return there ? __ldg(reinterpret_cast<const uint4 *>(p)) : make_uint4(0u, 0u, 0u, 0u); }

// k inside a block is permuted alike on both operands: lane (g = lane / 4, c = lane % 4) holds the sixteen codes at 16 c and at 64 + 16 c of its weight rows g and
// g + 8 and of its token g, four MMAs' worth.
template <int NT>
__global__ void __launch_bounds__(32 * kWarps) f8_rows_kernel(const F8Args a) {
    behind_grid();
    __shared__ float parts[kWarps][kRows][NT * kTokens + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int n0 = blockIdx.x * kRows, m0 = blockIdx.y * NT * kTokens;
    float acc[NT][4] = {};
    for (int b = warp; b < a.kb; b += kWarps) {
        uint4 lo[2], hi[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int64_t k = (int64_t)b * kF8Block + v * 64 + c * 16;
            lo[v] = load16(a.w + (int64_t)(n0 + g) * a.K + k, n0 + g < a.N && k < a.K);
            hi[v] = load16(a.w + (int64_t)(n0 + g + 8) * a.K + k, n0 + g + 8 < a.N && k < a.K);
        }
        const float ws = a.ws[(int64_t)(n0 / kF8Block) * a.kb + b];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float part[4] = {};
            const int m = m0 + t * kTokens + g;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int64_t k = (int64_t)b * kF8Block + v * 64 + c * 16;
                const uint4 x = load16(a.x + m * a.x_ld + k, m < a.M && k < a.K);
                mma_e4m3(part, lo[v].x, hi[v].x, lo[v].y, hi[v].y, x.x, x.y);
                mma_e4m3(part, lo[v].z, hi[v].z, lo[v].w, hi[v].w, x.z, x.w);
            }
            const int m1 = m0 + t * kTokens + 2 * c;
            const float s0 = m1 < a.M ? a.xs[m1 * a.xs_ld + b] * ws : 0.f, s1 = m1 + 1 < a.M ? a.xs[(m1 + 1) * a.xs_ld + b] * ws : 0.f;
            acc[t][0] = fmaf(part[0], s0, acc[t][0]), acc[t][1] = fmaf(part[1], s1, acc[t][1]);
            acc[t][2] = fmaf(part[2], s0, acc[t][2]), acc[t][3] = fmaf(part[3], s1, acc[t][3]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int m = t * kTokens + 2 * c;
        parts[warp][g][m] = acc[t][0], parts[warp][g][m + 1] = acc[t][1], parts[warp][g + 8][m] = acc[t][2], parts[warp][g + 8][m + 1] = acc[t][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * NT * kTokens; i += 32 * kWarps) {
        const int row = i % kRows, m = i / kRows;
        if (n0 + row >= a.N || m0 + m >= a.M) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += parts[w][row][m];
        const int64_t at = (int64_t)(m0 + m) * a.y_ld + n0 + row;
        if (a.f32) static_cast<float *>(a.y)[at] = sum;
        else static_cast<uint16_t *>(a.y)[at] = f32_to_bf16_bits(sum);
    }
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
    if (M > 32) return linear_f8_tc(fn, a, st);
    const dim3 grid((unsigned)((N + kRows - 1) / kRows)), block(32 * kWarps);
    const cudaError_t e = M <= 8    ? launch_behind(f8_rows_kernel<1>, grid, block, 0, st, 1, a)
                          : M <= 16 ? launch_behind(f8_rows_kernel<2>, grid, block, 0, st, 1, a)
                                    : launch_behind(f8_rows_kernel<4>, grid, block, 0, st, 1, a);
    SXB_CUDA(e, fn, ": launching M=", M, " N=", N, " K=", K);
    SXB_CHECK_LAUNCH(fn, " M=", M, " N=", N, " K=", K);
    return SXB_OK;
}
