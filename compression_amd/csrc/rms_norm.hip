// Root-mean-square norm of rows with the residual's addition and, if wanted, an 8-bit output with a scale per row:
//   h = x + r,  v[c] = h[c] (mean_c h^2 + eps)^(-1/2) w[c],  y = v  or  y = e4m3(v / s), s = max_c |v| / 448.
#include "row_ops.h"

namespace {

constexpr int NORM_THREADS = 256;

template <typename T>
__global__ __launch_bounds__(NORM_THREADS) void rms_norm_rows_kernel(const T *__restrict__ x, int64_t xs, const T *__restrict__ res,
                                                                     int64_t rs, const float *__restrict__ weight, int64_t channels,
                                                                     float eps, T *__restrict__ h_out, T *__restrict__ y,
                                                                     uint8_t *__restrict__ q, float *__restrict__ scale) {
    __shared__ float part[NORM_THREADS / 64];
    __shared__ unsigned upart[NORM_THREADS / 64];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    x += row * xs;
    if (res) res += row * rs;
    auto at = [&](int64_t c) { return res ? (float)x[c] + (float)res[c] : (float)x[c]; };

    float sum = 0.0f;
    for (int64_t c = tid; c < channels; c += NORM_THREADS) {
        const float h = at(c);
        sum += h * h;
        if (h_out) h_out[row * channels + c] = (T)h;
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 0) part[tid >> 6] = sum;
    __syncthreads();
    sum = 0.0f;
    for (int i = 0; i < NORM_THREADS / 64; ++i) sum += part[i];
    const float inv = 1.0f / sqrtf(sum / (float)channels + eps);
    auto value = [&](int64_t c) { return at(c) * inv * (weight ? weight[c] : 1.0f); };
    if (!q) {
        for (int64_t c = tid; c < channels; c += NORM_THREADS) y[row * channels + c] = (T)value(c);
        return;
    }
    // largest |v| by its bits: the order of non-negative floats, with NaN above infinity
    unsigned top = 0;
    for (int64_t c = tid; c < channels; c += NORM_THREADS) {
        const unsigned b = __float_as_uint(fabsf(value(c)));
        top = b > top ? b : top;
    }
    top = wave_max(top);
    if ((tid & 63) == 0) upart[tid >> 6] = top;
    __syncthreads();
    top = 0;
    for (int i = 0; i < NORM_THREADS / 64; ++i) top = upart[i] > top ? upart[i] : top;
    float s = __uint_as_float(top) / E4M3_MAX;
    s = top == 0 ? 1.0f : s < 0x1p-126f ? 0x1p-126f : s;
    if (tid == 0) scale[row] = s;
    const float rs_ = 1.0f / s;
    for (int64_t c = tid; c < channels; c += NORM_THREADS)
        q[row * channels + c] = (uint8_t)(e4m3_pack2<false>(value(c) * rs_, 0.0f, 0) & 0xff);
}

template <typename T>
int launch(mpc_ctx *ctx, const void *x, int64_t xs, const void *res, int64_t rs, const float *weight, int64_t rows, int64_t channels,
           float eps, void *h, void *y, bool eight, float *scale) {
    rms_norm_rows_kernel<T><<<dim3((unsigned)rows), dim3(NORM_THREADS), 0, ctx->stream>>>(
        (const T *)x, xs, (const T *)res, rs, weight, channels, eps, (T *)h, eight ? nullptr : (T *)y, eight ? (uint8_t *)y : nullptr, scale);
    MPC_CHECK_LAUNCH(ctx, "rms_norm");
    return MPC_OK;
}

}  // namespace

extern "C" int mpc_rms_norm(mpc_ctx *ctx, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                            const float *weight, int64_t rows, int64_t channels, float eps, int type, void *h, void *y, int y_type,
                            float *scale) {
    MPC_ENTER(ctx);
    MPC_REQUIRE(ctx, type == MPC_TYPE_F32 || type == MPC_TYPE_F16 || type == MPC_TYPE_BF16, "rms_norm: type %d", type);
    MPC_REQUIRE(ctx, y_type == type || y_type == MPC_TYPE_E4M3, "rms_norm: output type %d from type %d", y_type, type);
    MPC_REQUIRE(ctx, rows >= 0 && rows < (1ll << 31) && channels > 0 && channels < (1ll << 31), "rms_norm: rows = %lld, channels = %lld",
                (long long)rows, (long long)channels);
    MPC_REQUIRE(ctx, eps >= 0.0f && eps < INFINITY, "rms_norm: eps = %g", (double)eps);
    if (rows == 0) return MPC_OK;
    const bool eight = y_type == MPC_TYPE_E4M3;
    MPC_REQUIRE(ctx, x && y && (scale != nullptr) == eight, "rms_norm: null pointer, or a scale without an 8-bit output");
    MPC_REQUIRE(ctx, x_stride >= 0 && residual_stride >= 0, "rms_norm: negative stride");
    if (type == MPC_TYPE_F32) return launch<float>(ctx, x, x_stride, residual, residual_stride, weight, rows, channels, eps, h, y, eight, scale);
    if (type == MPC_TYPE_F16) return launch<f16_t>(ctx, x, x_stride, residual, residual_stride, weight, rows, channels, eps, h, y, eight, scale);
    return launch<bf16_t>(ctx, x, x_stride, residual, residual_stride, weight, rows, channels, eps, h, y, eight, scale);
}
