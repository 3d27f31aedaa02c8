// Root-mean-square norm of rows with the residual's addition and, if wanted, an 8-bit output with a scale per row:
//   h = x + r,  v[c] = h[c] (mean_c h^2 + eps)^(-1/2) w[c],  y = v  or  y = e4m3(v / s), s = max_c |v| / 448.
//
// A row is read once: its threads keep h in registers (fp32) across the sum, the largest value and the output.  The kernel
// moves x, r, h and y once each and does about ten operations a value, so memory bounds it: 32768 x 4096 bf16 with residual
// to 8 bit 176 us, 5.3 TB/s; without either 99 us, 5.4 TB/s; 36864 x 192 f16 6.9 us out of L2; one row 3.4 us.
#include "row_ops.h"

namespace {

constexpr int NORM_MAX_THREADS = 1024;
constexpr int NORM_MOST = 8;                       // most 16-byte vectors of a row that a thread keeps

struct NormArgs {
    const void *x, *res;
    int64_t xs, rs, rows;
    int channels;
    float eps;
    const float *weight;
    void *h, *y;
    float *scale;
    int group;                                     // threads of a row, a power of two
};

// (mean square + eps)^(-1/2); 0 where that is 0 (eps = 0 and a row of zeros), so that the row stays one of zeros
__device__ __forceinline__ float row_inverse(float sum, int channels, float eps) {
    const float d = sum / (float)channels + eps;
    return d == 0.0f ? 0.0f : 1.0f / sqrtf(d);
}

// s = top / 448 for the row's largest |v| (by its bits: the order of non-negative floats, with NaN above infinity)
__device__ __forceinline__ float row_scale(unsigned top) {
    const float s = __uint_as_float(top) / E4M3_MAX;
    return top == 0 ? 1.0f : s < 0x1p-126f ? 0x1p-126f : s;
}

// VPT vectors of 16 bytes of x per thread: vector i * group + lane of the row, so the group's accesses are consecutive.
// Rows may start at any element; the last vector of a row may be short.
template <typename T, int VPT, bool Q>
__global__ __launch_bounds__(NORM_MAX_THREADS) void rms_norm_kernel(NormArgs a) {
    constexpr int W = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(W)));
    typedef vec vec_any __attribute__((aligned(sizeof(T))));
    typedef float fvec __attribute__((ext_vector_type(4)));
    typedef fvec fvec_any __attribute__((aligned(4)));
    typedef unsigned uvec __attribute__((ext_vector_type(W / 4)));
    typedef uvec uvec_any __attribute__((aligned(1)));
    __shared__ float part[NORM_MAX_THREADS / 64];
    __shared__ unsigned upart[NORM_MAX_THREADS / 64];

    const int G = a.group, tid = threadIdx.x, lane = tid & (G - 1);
    const int64_t at = (int64_t)blockIdx.x * (blockDim.x / G) + tid / G;
    const bool mine = at < a.rows;                                   // (the last block may have groups without a row)
    const int64_t row = mine ? at : a.rows - 1;
    const T *x = (const T *)a.x + row * a.xs, *r = a.res ? (const T *)a.res + row * a.rs : nullptr;
    const int C = a.channels;

    float v[VPT][W];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * G + lane) * W;
        vec t;
        if (c + W <= C) {
            t = *(const vec_any *)(x + c);
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j) t[j] = c + j < C ? x[c + j] : (T)0.0f;
        }
#pragma unroll
        for (int j = 0; j < W; ++j) v[i][j] = (float)t[j];
    }
    if (r) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * G + lane) * W;
            vec t;
            if (c + W <= C) {
                t = *(const vec_any *)(r + c);
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) t[j] = c + j < C ? r[c + j] : (T)0.0f;
            }
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] += (float)t[j];
        }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) sum += v[i][j] * v[i][j];
    if (a.h && mine) {
        T *h = (T *)a.h + row * C;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * G + lane) * W;
            if (c + W <= C) {
                vec t;
#pragma unroll
                for (int j = 0; j < W; ++j) t[j] = (T)v[i][j];
                *(vec_any *)(h + c) = t;
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (c + j < C) h[c + j] = (T)v[i][j];
            }
        }
    }
    for (int off = (G < 64 ? G : 64) / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (G > 64) {
        if ((tid & 63) == 0) part[tid >> 6] = sum;
        __syncthreads();
        sum = 0.0f;
        for (int i = 0; i < G / 64; ++i) sum += part[tid / G * (G / 64) + i];
    }
    const float inv = row_inverse(sum, C, a.eps);

    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * G + lane) * W;
        if (a.weight && c + W <= C) {
#pragma unroll
            for (int q = 0; q < W; q += 4) {
                const fvec w = *(const fvec_any *)(a.weight + c + q);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][q + j] = v[i][q + j] * inv * w[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] = v[i][j] * inv * (a.weight && c + j < C ? a.weight[c + j] : 1.0f);
        }
        if constexpr (Q) {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const unsigned b = __float_as_uint(v[i][j]) & 0x7fffffffu;   // (past the row's end: 0, or NaN where all of the row is)
                top = b > top ? b : top;
            }
        }
    }
    if constexpr (!Q) {
        if (!mine) return;
        T *y = (T *)a.y + row * C;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * G + lane) * W;
            if (c + W <= C) {
                vec t;
#pragma unroll
                for (int j = 0; j < W; ++j) t[j] = (T)v[i][j];
                *(vec_any *)(y + c) = t;
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (c + j < C) y[c + j] = (T)v[i][j];
            }
        }
    } else {
        for (int off = (G < 64 ? G : 64) / 2; off > 0; off >>= 1) {
            const unsigned o = __shfl_xor(top, off, 64);
            top = o > top ? o : top;
        }
        if (G > 64) {
            if ((tid & 63) == 0) upart[tid >> 6] = top;
            __syncthreads();
            for (int i = 0; i < G / 64; ++i) {
                const unsigned o = upart[tid / G * (G / 64) + i];
                top = o > top ? o : top;
            }
        }
        if (!mine) return;
        const float s = row_scale(top), back = 1.0f / s;
        if (lane == 0) a.scale[row] = s;
        uint8_t *y = (uint8_t *)a.y + row * C;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * G + lane) * W;
            uvec t;
#pragma unroll
            for (int q = 0; q < W / 4; ++q) {
                const int lo = e4m3_pack2<false>(v[i][4 * q] * back, v[i][4 * q + 1] * back, 0);
                t[q] = (unsigned)e4m3_pack2<true>(v[i][4 * q + 2] * back, v[i][4 * q + 3] * back, lo);
            }
            if (c + W <= C) {
                *(uvec_any *)(y + c) = t;
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (c + j < C) y[c + j] = (uint8_t)(t[j / 4] >> (8 * (j % 4)));
            }
        }
    }
}

// Rows too long for the registers of a block: three passes over x and r, which the L2 holds after the first.
template <typename T>
__global__ __launch_bounds__(NORM_MAX_THREADS) void rms_norm_long_kernel(NormArgs a, bool eight) {
    constexpr int NT = NORM_MAX_THREADS;
    __shared__ float part[NT / 64];
    __shared__ unsigned upart[NT / 64];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, C = a.channels;
    const T *x = (const T *)a.x + row * a.xs, *r = a.res ? (const T *)a.res + row * a.rs : nullptr;
    auto at = [&](int c) { return r ? (float)x[c] + (float)r[c] : (float)x[c]; };
    float sum = 0.0f;
    for (int64_t c = tid; c < C; c += NT) {
        const float h = at(c);
        sum += h * h;
        if (a.h) ((T *)a.h)[row * C + c] = (T)h;
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 0) part[tid >> 6] = sum;
    __syncthreads();
    sum = 0.0f;
    for (int i = 0; i < NT / 64; ++i) sum += part[i];
    const float inv = row_inverse(sum, C, a.eps);
    auto value = [&](int c) { return at(c) * inv * (a.weight ? a.weight[c] : 1.0f); };
    if (!eight) {
        for (int64_t c = tid; c < C; c += NT) ((T *)a.y)[row * C + c] = (T)value(c);
        return;
    }
    unsigned top = 0;
    for (int64_t c = tid; c < C; c += NT) {
        const unsigned b = __float_as_uint(value(c)) & 0x7fffffffu;
        top = b > top ? b : top;
    }
    top = wave_max(top);
    if ((tid & 63) == 0) upart[tid >> 6] = top;
    __syncthreads();
    top = 0;
    for (int i = 0; i < NT / 64; ++i) top = upart[i] > top ? upart[i] : top;
    const float s = row_scale(top), back = 1.0f / s;
    if (tid == 0) a.scale[row] = s;
    for (int64_t c = tid; c < C; c += NT) ((uint8_t *)a.y)[row * C + c] = (uint8_t)(e4m3_pack2<false>(value(c) * back, 0.0f, 0) & 0xff);
}

// The rows in as many launches as they take: one has fewer than 2^32 threads (`per_row` for each row).
template <typename T, bool Q, typename F>
void in_parts(const NormArgs &a, int per_row, F run) {
    const int64_t most = MPC_LAUNCH_THREADS / per_row;
    for (int64_t first = 0; first < a.rows; first += most) {
        NormArgs part = a;
        part.rows = a.rows - first < most ? a.rows - first : most;
        part.x = (const T *)a.x + first * a.xs;
        if (a.res) part.res = (const T *)a.res + first * a.rs;
        if (a.h) part.h = (T *)a.h + first * a.channels;
        part.y = (char *)a.y + first * a.channels * (Q ? 1 : sizeof(T));
        if (Q) part.scale = a.scale + first;
        run(part);
    }
}

// Vectors per thread and threads per row.  More vectors mean more loads in flight and no barrier (a row within a wave), as
// long as the card stays full of waves, a row's threads reach over 64 bytes, 512 with more than two vectors, and no more slots
// stay empty; fewer empty slots come first.  (bf16 + residual -> 8 bit, in us, one vector a thread : this rule: 50000 x 2048 138 : 137,
// 8192 x 4096 47 : 42, 100000 x 1024 136 : 129, 36864 x 192 16.2 : 10.0; always the most: 1M x 64 f16 69 : 38, 300000 x 256
// 107 : 99, 1024 x 8192 12 : 12, one row of 4096 5.6 : 3.4.)
template <typename T, bool Q>
int launch(mpc_ctx *ctx, NormArgs a) {
    constexpr int W = 16 / sizeof(T);
    const int64_t vectors = mpc_cdiv(a.channels, W);
    if (vectors > (int64_t)NORM_MOST * NORM_MAX_THREADS) {
        in_parts<T, Q>(a, NORM_MAX_THREADS, [&](const NormArgs &part) {
            rms_norm_long_kernel<T><<<dim3((unsigned)part.rows), dim3(NORM_MAX_THREADS), 0, ctx->stream>>>(part, Q);
        });
        MPC_CHECK_LAUNCH(ctx, "rms_norm_long");
        return MPC_OK;
    }
    constexpr int64_t full = 4096;                                 // waves
    int vpt = 0, group = 0;
    int64_t waste = 0;
    for (int v : {1, 2, 3, 4, NORM_MOST}) {
        int64_t g = 1;
        while (g * v < vectors) g *= 2;
        if (g > NORM_MAX_THREADS) continue;
        const int64_t lost = g * v - vectors;
        if (group && (lost * 8 > g * v + waste * 8 || (g < (v > 2 ? 32 : 4) && lost >= waste) || a.rows * g < full * 64)) continue;
        vpt = v, group = (int)g, waste = lost;
    }
    a.group = group;
    const int threads = group > 256 ? group : 256;
    in_parts<T, Q>(a, group, [&](const NormArgs &part) {
        const dim3 grid((unsigned)mpc_cdiv(part.rows, threads / group)), block(threads);
        switch (vpt) {
            case 1: rms_norm_kernel<T, 1, Q><<<grid, block, 0, ctx->stream>>>(part); break;
            case 2: rms_norm_kernel<T, 2, Q><<<grid, block, 0, ctx->stream>>>(part); break;
            case 3: rms_norm_kernel<T, 3, Q><<<grid, block, 0, ctx->stream>>>(part); break;
            case 4: rms_norm_kernel<T, 4, Q><<<grid, block, 0, ctx->stream>>>(part); break;
            default: rms_norm_kernel<T, NORM_MOST, Q><<<grid, block, 0, ctx->stream>>>(part);
        }
    });
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
    MPC_REQUIRE(ctx, rows >= 0 && rows < (1ll << 31) && channels > 0 && channels < (1ll << 31) - 65536, "rms_norm: rows = %lld, channels = %lld",
                (long long)rows, (long long)channels);
    MPC_REQUIRE(ctx, eps >= 0.0f && eps < INFINITY, "rms_norm: eps = %g", (double)eps);
    if (rows == 0) return MPC_OK;
    const bool eight = y_type == MPC_TYPE_E4M3;
    MPC_REQUIRE(ctx, x && y && (scale != nullptr) == eight, "rms_norm: null pointer, or a scale without an 8-bit output");
    MPC_REQUIRE(ctx, x_stride >= 0 && residual_stride >= 0, "rms_norm: negative stride");
    const int tb = mpc_type_bytes(type);
    MPC_REQUIRE(ctx, ((uintptr_t)x | (uintptr_t)residual | (uintptr_t)h | (eight ? 0 : (uintptr_t)y)) % tb == 0 &&
                         ((uintptr_t)weight | (uintptr_t)scale) % 4 == 0, "rms_norm: misaligned pointer");
    const NormArgs a{x, residual, x_stride, residual_stride, rows, (int)channels, eps, weight, h, y, scale, 0};
    if (type == MPC_TYPE_F32) return eight ? launch<float, true>(ctx, a) : launch<float, false>(ctx, a);
    if (type == MPC_TYPE_F16) return eight ? launch<f16_t, true>(ctx, a) : launch<f16_t, false>(ctx, a);
    return eight ? launch<bf16_t, true>(ctx, a) : launch<bf16_t, false>(ctx, a);
}
