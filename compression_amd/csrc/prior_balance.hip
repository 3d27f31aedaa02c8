// The balance loss of a competition and its gradient.  With z = scale * scores, p = softmax(z) over the experts of a row
// that counts and f the share of the top_k choices that fell on an expert:
//   loss = E sum_e f_e mean_t p_te,     d loss / d score_tj = scale E / R p_tj (f_j - sum_e f_e p_te).
// One wave takes a row: lane l holds experts l, l + 64, ...  A block's waves add up p and the choices of their rows in
// registers; the blocks' sums meet in a second kernel, in a fixed order and in double.
#include "row_ops.h"

namespace {

constexpr int PB_WAVES = 4;
constexpr int PB_MAX_BLOCKS = 512;
constexpr int PB_MAX_EXPERTS = 1024;

struct Row {
    const void *scores;
    int64_t rows, row_stride, expert_stride;
    int experts;
    float scale;
    int top_k;
    const uint8_t *mask;
};

// v[i] = scores in the order of the choice (costs negated), -inf past the last expert; p[i] the row's softmax.
// Returns whether the row counts.
template <typename T, int NI>
__device__ __forceinline__ bool load_row(const Row &a, int64_t row, int lane, float (&v)[NI], float (&p)[NI]) {
    if (a.mask && !a.mask[row]) return false;
    const T *s = (const T *)a.scores + row * a.row_stride;
    const float mag = fabsf(a.scale);
    float top = -INFINITY;
    int nan = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int e = lane + 64 * i;
        float x = -INFINITY;
        if (e < a.experts) x = (float)s[e * a.expert_stride];
        v[i] = e < a.experts && a.scale < 0.0f ? -x : x;
        nan |= v[i] != v[i];
        top = fmaxf(top, v[i]);
    }
    top = wave_max(top);
    if (top == -INFINITY && __ballot(nan) == 0) return false;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        p[i] = __expf((v[i] - top) * mag);
        sum += p[i];
    }
    const float inv = 1.0f / wave_sum(sum);
#pragma unroll
    for (int i = 0; i < NI; ++i) p[i] *= inv;
    return true;
}

// partial sums of a block: [block][2 * experts + 1] words: sum of p (float), choices (int), rows (int)
template <typename T, int NI>
__global__ __launch_bounds__(64 * PB_WAVES) void prior_balance_kernel(Row a, float *__restrict__ ws) {
    __shared__ float psum[PB_WAVES][NI * 64];
    __shared__ int csum[PB_WAVES][NI * 64];
    __shared__ int rsum[PB_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float acc[NI];
    int cnt[NI], n = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) acc[i] = 0.0f, cnt[i] = 0;
    for (int64_t row = (int64_t)blockIdx.x * PB_WAVES + wave; row < a.rows; row += (int64_t)gridDim.x * PB_WAVES) {
        float v[NI], p[NI];
        if (!load_row<T, NI>(a, row, lane, v, p)) continue;
        ++n;
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[i] += p[i];
        for (int k = 0; k < a.top_k; ++k) {
            float best = -INFINITY;
            int at = PB_MAX_EXPERTS;
#pragma unroll
            for (int i = 0; i < NI; ++i)
                if (v[i] > best) best = v[i], at = lane + 64 * i;
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
                const float b = __shfl_xor(best, off, 64);
                const int o = __shfl_xor(at, off, 64);
                if (b > best || (b == best && o < at)) best = b, at = o;
            }
            if (at == PB_MAX_EXPERTS) break;                 // nothing above -inf is left
#pragma unroll
            for (int i = 0; i < NI; ++i)
                if (at == lane + 64 * i) ++cnt[i], v[i] = -INFINITY;
        }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) psum[wave][lane + 64 * i] = acc[i], csum[wave][lane + 64 * i] = cnt[i];
    if (lane == 0) rsum[wave] = n;
    __syncthreads();
    float *out = ws + (int64_t)blockIdx.x * (2 * a.experts + 1);
    for (int e = threadIdx.x; e < a.experts; e += 64 * PB_WAVES) {
        float s = 0.0f;
        int c = 0;
        for (int w = 0; w < PB_WAVES; ++w) s += psum[w][e], c += csum[w][e];
        out[e] = s;
        ((int *)out)[a.experts + e] = c;
    }
    if (threadIdx.x == 0) {
        int c = 0;
        for (int w = 0; w < PB_WAVES; ++w) c += rsum[w];
        ((int *)out)[2 * a.experts] = c;
    }
}

__global__ __launch_bounds__(1024) void prior_balance_join_kernel(const float *__restrict__ ws, int blocks, int experts, int top_k,
                                                                  float *__restrict__ loss, int32_t *__restrict__ counts,
                                                                  int32_t *__restrict__ n_rows) {
    __shared__ double part[16];
    const int e = threadIdx.x, words = 2 * experts + 1;
    int n = 0;
    for (int b = 0; b < blocks; ++b) n += ((const int *)ws)[(int64_t)b * words + 2 * experts];
    double term = 0.0;
    if (e < experts) {
        double p = 0.0;
        int c = 0;
        for (int b = 0; b < blocks; ++b) {
            p += (double)ws[(int64_t)b * words + e];
            c += ((const int *)ws)[(int64_t)b * words + experts + e];
        }
        counts[e] = c;
        if (n > 0) term = (double)c / ((double)top_k * n) * (p / n);
    }
    for (int off = 32; off > 0; off >>= 1) term += __shfl_xor(term, off, 64);
    if ((e & 63) == 0) part[e >> 6] = term;
    __syncthreads();
    if (e == 0) {
        double s = 0.0;
        for (unsigned w = 0; w < blockDim.x / 64; ++w) s += part[w];
        *loss = (float)(experts * s);
        *n_rows = n;
    }
}

template <typename T, int NI>
__global__ __launch_bounds__(64 * PB_WAVES) void prior_balance_grad_kernel(Row a, const int32_t *__restrict__ counts,
                                                                           const int32_t *__restrict__ n_rows,
                                                                           const float *__restrict__ grad_out, T *__restrict__ grad,
                                                                           int64_t grs, int64_t ges) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = *n_rows;
    // f_j - 1 / E: the difference f_j - sum_e f_e p_te is the same, and loses less where use is nearly even
    float f[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int e = lane + 64 * i;
        f[i] = e < a.experts && n > 0 ? (float)((double)counts[e] / ((double)a.top_k * n) - 1.0 / a.experts) : 0.0f;
    }
    const float g = n > 0 ? (float)((double)(grad_out ? *grad_out : 1.0f) * a.scale * a.experts / n) : 0.0f;
    for (int64_t row = (int64_t)blockIdx.x * PB_WAVES + wave; row < a.rows; row += (int64_t)gridDim.x * PB_WAVES) {
        float v[NI], p[NI], d = 0.0f;
        const bool counted = load_row<T, NI>(a, row, lane, v, p);
        if (counted) {
#pragma unroll
            for (int i = 0; i < NI; ++i) d += p[i] * f[i];
            d = wave_sum(d);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int e = lane + 64 * i;
            if (e < a.experts) grad[row * grs + e * ges] = (T)(counted ? g * p[i] * (f[i] - d) : 0.0f);
        }
    }
}

int blocks_for(int64_t rows) {
    const int64_t b = mpc_cdiv(rows, PB_WAVES);
    return (int)(b < 1 ? 1 : b > PB_MAX_BLOCKS ? PB_MAX_BLOCKS : b);
}

template <typename T, int NI>
int forward(mpc_ctx *ctx, const Row &a, float *ws, float *loss, int32_t *counts, int32_t *n_rows) {
    const int blocks = blocks_for(a.rows);
    prior_balance_kernel<T, NI><<<dim3(blocks), dim3(64 * PB_WAVES), 0, ctx->stream>>>(a, ws);
    MPC_CHECK_LAUNCH(ctx, "prior_balance");
    prior_balance_join_kernel<<<dim3(1), dim3((a.experts + 63) / 64 * 64), 0, ctx->stream>>>(ws, blocks, a.experts, a.top_k, loss, counts, n_rows);
    MPC_CHECK_LAUNCH(ctx, "prior_balance_join");
    return MPC_OK;
}

template <typename T, int NI>
int backward(mpc_ctx *ctx, const Row &a, const int32_t *counts, const int32_t *n_rows, const float *grad_out, void *grad, int64_t grs, int64_t ges) {
    const int64_t b = mpc_cdiv(a.rows, PB_WAVES);
    prior_balance_grad_kernel<T, NI><<<dim3((unsigned)(b > 4096 ? 4096 : b)), dim3(64 * PB_WAVES), 0, ctx->stream>>>(
        a, counts, n_rows, grad_out, (T *)grad, grs, ges);
    MPC_CHECK_LAUNCH(ctx, "prior_balance_grad");
    return MPC_OK;
}

int check(mpc_ctx *ctx, const void *scores, int type, int64_t rows, int experts, int64_t rs, int64_t es, float scale, int top_k) {
    MPC_REQUIRE(ctx, type == MPC_TYPE_F32 || type == MPC_TYPE_F16 || type == MPC_TYPE_BF16, "prior_balance: type %d", type);
    MPC_REQUIRE(ctx, experts > 0 && experts <= PB_MAX_EXPERTS, "prior_balance: %d experts (1..%d)", experts, PB_MAX_EXPERTS);
    MPC_REQUIRE(ctx, top_k > 0 && top_k <= experts, "prior_balance: top_k = %d of %d experts", top_k, experts);
    MPC_REQUIRE(ctx, rows >= 0 && rows < (1ll << 31) / top_k, "prior_balance: %lld rows", (long long)rows);
    MPC_REQUIRE(ctx, rs >= 0 && es >= 0, "prior_balance: negative stride");
    MPC_REQUIRE(ctx, scale != 0.0f && scale > -INFINITY && scale < INFINITY, "prior_balance: scale = %g", (double)scale);
    MPC_REQUIRE(ctx, rows == 0 || scores, "prior_balance: null pointer");
    return MPC_OK;
}

}  // namespace

#define PB_BY_EXPERTS(FN, T, ...)                             \
    do {                                                      \
        if (experts <= 64) return FN<T, 1>(__VA_ARGS__);      \
        if (experts <= 128) return FN<T, 2>(__VA_ARGS__);     \
        if (experts <= 256) return FN<T, 4>(__VA_ARGS__);     \
        if (experts <= 512) return FN<T, 8>(__VA_ARGS__);     \
        return FN<T, 16>(__VA_ARGS__);                        \
    } while (0)
#define PB_DISPATCH(FN, ...)                                             \
    do {                                                                 \
        if (type == MPC_TYPE_F32) PB_BY_EXPERTS(FN, float, __VA_ARGS__); \
        if (type == MPC_TYPE_F16) PB_BY_EXPERTS(FN, f16_t, __VA_ARGS__); \
        PB_BY_EXPERTS(FN, bf16_t, __VA_ARGS__);                          \
    } while (0)

extern "C" size_t mpc_prior_balance_workspace_bytes(int64_t rows, int experts) {
    if (rows < 0 || experts <= 0 || experts > PB_MAX_EXPERTS) return 0;
    return (size_t)blocks_for(rows) * (2 * experts + 1) * sizeof(float);
}

extern "C" int mpc_prior_balance(mpc_ctx *ctx, const void *scores, int type, int64_t rows, int experts, int64_t row_stride,
                                 int64_t expert_stride, float scale, int top_k, const uint8_t *mask, void *workspace, size_t workspace_bytes,
                                 float *loss, int32_t *counts, int32_t *n_rows) {
    MPC_ENTER(ctx);
    const int bad = check(ctx, scores, type, rows, experts, row_stride, expert_stride, scale, top_k);
    if (bad) return bad;
    MPC_REQUIRE(ctx, workspace && loss && counts && n_rows && ((uintptr_t)workspace & 3) == 0, "prior_balance: null or misaligned pointer");
    MPC_REQUIRE(ctx, workspace_bytes >= mpc_prior_balance_workspace_bytes(rows, experts), "prior_balance: workspace of %zu bytes", workspace_bytes);
    const Row a{scores, rows, row_stride, expert_stride, experts, scale, top_k, mask};
    PB_DISPATCH(forward, ctx, a, (float *)workspace, loss, counts, n_rows);
}

extern "C" int mpc_prior_balance_grad(mpc_ctx *ctx, const void *scores, int type, int64_t rows, int experts, int64_t row_stride,
                                      int64_t expert_stride, float scale, int top_k, const uint8_t *mask, const int32_t *counts,
                                      const int32_t *n_rows, const float *grad_out, void *grad, int64_t grad_row_stride,
                                      int64_t grad_expert_stride) {
    MPC_ENTER(ctx);
    const int bad = check(ctx, scores, type, rows, experts, row_stride, expert_stride, scale, top_k);
    if (bad) return bad;
    if (rows == 0) return MPC_OK;
    MPC_REQUIRE(ctx, counts && n_rows && grad, "prior_balance_grad: null pointer");
    MPC_REQUIRE(ctx, grad_row_stride >= 0 && grad_expert_stride >= 0, "prior_balance_grad: negative stride");
    const Row a{scores, rows, row_stride, expert_stride, experts, scale, top_k, mask};
    PB_DISPATCH(backward, ctx, a, counts, n_rows, grad_out, grad, grad_row_stride, grad_expert_stride);
}
