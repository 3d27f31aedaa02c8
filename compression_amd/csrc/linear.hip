// Matrix product with its epilogue fused: out[m][n] = act(sx[m] sw[n] sum_k x[m][k] w[n][k] + b[n]) + r[m][n].
//
// Both operands lie with k innermost, which is how the matrix instructions want them: a lane of a 16x16 tile holds 16
// (16-bit operands: 8 values; e4m3: 16, two such pieces) consecutive bytes of one row.  A k-tile is 128 bytes of every
// row, 64 values of 16 bits or 128 of 8, so both widths move the same bytes and issue the same matrix cycles per tile.
// w is the instruction's first operand: a lane then holds four consecutive n of one m.  Which row of w a lane
// brings is free, so the NF tiles side by side take rows interleaved in fours: a lane ends up with 4 NF consecutive
// outputs of one row and stores them as 16-byte pieces.
#include "row_ops.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));          // a 16-byte access at any address
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));

namespace {

struct LinearArgs {
    const char *x, *w;
    int64_t M, N, K;                  // K in bytes of an operand row
    int64_t xs, ws;                   // row strides in bytes
    const float *sx, *sw, *bias;
    const char *res;
    char *out;
    int64_t rs, os;                   // in bytes
    int out_type, act;
    int vec_out, vec_res;             // 16-byte accesses are possible
    int tiles_m, tiles_n;
};

// ---- epilogue ---------------------------------------------------------------------------------------------------------
// V consecutive outputs of row m from column n on.  v: the sums.
template <int V>
__device__ __forceinline__ void activate(float (&v)[V], int act) {
    if (act == MPC_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];            // (a NaN stays)
    } else if (act == MPC_ACT_GELU) {
        // gelu(v) = max(v, 0) - |v| / 2 erfc(|v| / sqrt 2), with formula 7.1.26 of Abramowitz and Stegun (1964) for erfc, off by
        // at most 1.5e-7: erfc(u) = t (a1 + t (a2 + t (a3 + t (a4 + t a5)))) exp(-u^2), t = 1 / (1 + p u).
        // 18 issue slots a value, where the library's erfc takes several times that.
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float m = fabsf(v[i]), t = __builtin_amdgcn_rcpf(fmaf(m, 0.3275911f * 0.70710678f, 1.0f));
            float q = fmaf(t, 1.061405429f, -1.453152027f);
            q = fmaf(t, q, 1.421413741f);
            q = fmaf(t, q, -0.284496736f);
            q = fmaf(t, q, 0.254829592f);
            const float e = __builtin_amdgcn_exp2f(v[i] * v[i] * -0.72134752f);          // exp(-v^2 / 2)
            v[i] = fmaf(-0.5f * m * t * q, e, v[i] < 0.0f ? 0.0f : v[i]);
        }
    } else if (act == MPC_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v[i] * -1.44269504f));
    }
}

template <typename T, int V>
__device__ __forceinline__ void finish(const LinearArgs &a, int64_t m, int64_t n, float (&v)[V]) {
    constexpr int PER = 16 / sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(PER)));
    const bool whole = n + V <= a.N;
    if (a.res) {
        const T *r = (const T *)(a.res + m * a.rs) + n;
        if (whole && a.vec_res) {
#pragma unroll
            for (int i = 0; i < V; i += PER) {
                const vec_t t = *(const vec_t *)(r + i);
#pragma unroll
                for (int j = 0; j < PER; ++j) v[i + j] += (float)t[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (n + i < a.N) v[i] += (float)r[i];
        }
    }
    T *o = (T *)(a.out + m * a.os) + n;
    if (whole && a.vec_out) {
#pragma unroll
        for (int i = 0; i < V; i += PER) {
            vec_t t;
#pragma unroll
            for (int j = 0; j < PER; ++j) t[j] = (T)v[i + j];
            *(vec_t *)(o + i) = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (n + i < a.N) o[i] = (T)v[i];
    }
}

template <int V>
__device__ __forceinline__ void column_terms(const LinearArgs &a, int64_t n, float (&b)[V], float (&s)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        b[i] = a.bias && n + i < a.N ? a.bias[n + i] : 0.0f;
        s[i] = a.sw && n + i < a.N ? a.sw[n + i] : 1.0f;
    }
}

template <int V>
__device__ __forceinline__ void epilogue(const LinearArgs &a, int64_t m, int64_t n, float (&v)[V], const float (&b)[V], const float (&s)[V]) {
    const float sx = a.sx ? a.sx[m] : 1.0f;
    if (a.sx) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= sx * s[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += b[i];
    activate<V>(v, a.act);
    if (a.out_type == MPC_TYPE_F32) finish<float, V>(a, m, n, v);
    else if (a.out_type == MPC_TYPE_F16) finish<f16_t, V>(a, m, n, v);
    else finish<bf16_t, V>(a, m, n, v);
}

// ---- operands ---------------------------------------------------------------------------------------------------------
template <int TYPE>
struct Operand;
template <>
struct Operand<MPC_TYPE_F16> {
    static constexpr int BYTES = 2;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
};
template <>
struct Operand<MPC_TYPE_BF16> {
    static constexpr int BYTES = 2;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
    }
};
template <>
struct Operand<MPC_TYPE_E4M3> {
    static constexpr int BYTES = 1;
    // 128 values of k in one instruction; the block scales of its format are all 1 (exponent 127)
    static __device__ __forceinline__ f32x4 mma(u32x4 a0, u32x4 a1, u32x4 b0, u32x4 b1, f32x4 c) {
        const i32x8 a = {(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3], (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
        const i32x8 b = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
    }
};

// 16 bytes of an operand row of which `left` (anything) belong to the row; zeros behind them
template <int BYTES>
__device__ __forceinline__ u32x4 load_piece(const char *p, int64_t left) {
    if (left >= 16) return *(const u32x4_any *)p;
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16 / BYTES; ++i)
        if (i * BYTES < left) {
            const unsigned e = BYTES == 2 ? *(const uint16_t *)(p + 2 * i) : *(const uint8_t *)(p + i);
            v[i * BYTES / 4] |= e << (8 * (i * BYTES % 4));
        }
    return v;
}

// ---- tiles through LDS --------------------------------------------------------------------------------------------------
constexpr int KT = 128;               // bytes of a k-tile

template <int TYPE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void linear_tile_kernel(LinearArgs a) {
    constexpr int NT = 64 * (BM / WM) * (BN / WN);
    constexpr int MF = WM / 16, NF = WN / 16, V = 4 * NF;
    constexpr int XP = BM * 8 / NT, WP = BN * 8 / NT;             // 16-byte pieces per thread and tile
    extern __shared__ u32x4 lds[];                                // 2 x [BM + BN rows][8 pieces]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int j = lane & 15, g = lane >> 4;
    const int wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
    const int64_t m0 = (int64_t)(blockIdx.x % a.tiles_m) * BM, n0 = (int64_t)(blockIdx.x / a.tiles_m) * BN;

    // Piece p of row r lies at slot p ^ key(r): the 16 rows that one instruction reads at the same p then spread over the banks.
    auto xkey = [](int r) { return r & 7; };
    auto wkey = [](int r) { return (r & 3) | (r / V & 1) << 2; };

    const int p = tid & 7;
    const char *xp[XP], *wp[WP];
#pragma unroll
    for (int i = 0; i < XP; ++i) {
        const int64_t r = m0 + tid / 8 + i * (NT / 8);
        xp[i] = a.x + (r < a.M ? r : a.M - 1) * a.xs + p * 16;
    }
#pragma unroll
    for (int i = 0; i < WP; ++i) {
        const int64_t r = n0 + tid / 8 + i * (NT / 8);
        wp[i] = a.w + (r < a.N ? r : a.N - 1) * a.ws + p * 16;
    }
    u32x4 xr[XP], wr[WP];
    auto fetch = [&](int64_t k) {
        if (k + KT <= a.K) {
#pragma unroll
            for (int i = 0; i < XP; ++i) xr[i] = *(const u32x4_any *)(xp[i] + k);
#pragma unroll
            for (int i = 0; i < WP; ++i) wr[i] = *(const u32x4_any *)(wp[i] + k);
        } else {
            const int64_t left = a.K - k - p * 16;
#pragma unroll
            for (int i = 0; i < XP; ++i) xr[i] = load_piece<Operand<TYPE>::BYTES>(xp[i] + k, left);
#pragma unroll
            for (int i = 0; i < WP; ++i) wr[i] = load_piece<Operand<TYPE>::BYTES>(wp[i] + k, left);
        }
    };
    auto stash = [&](int buf) {
        u32x4 *x = lds + buf * (BM + BN) * 8, *w = x + BM * 8;
#pragma unroll
        for (int i = 0; i < XP; ++i) {
            const int r = tid / 8 + i * (NT / 8);
            x[r * 8 + (p ^ xkey(r))] = xr[i];
        }
#pragma unroll
        for (int i = 0; i < WP; ++i) {
            const int r = tid / 8 + i * (NT / 8);
            w[r * 8 + (p ^ wkey(r))] = wr[i];
        }
    };

    f32x4 acc[NF][MF];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int m = 0; m < MF; ++m) acc[f][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    fetch(0);
    stash(0);
    __syncthreads();
    int buf = 0;
    for (int64_t k = 0; k < a.K; k += KT, buf ^= 1) {
        const bool more = k + KT < a.K;
        if (more) fetch(k + KT);
        const u32x4 *x = lds + buf * (BM + BN) * 8, *w = x + BM * 8;
        auto xfrag = [&](int m, int q) {
            const int r = wm + m * 16 + j;
            return x[r * 8 + (q ^ xkey(r))];
        };
        auto wfrag = [&](int f, int q) {
            const int r = wn + (j >> 2) * V + f * 4 + (j & 3);
            return w[r * 8 + (q ^ wkey(r))];
        };
        if constexpr (TYPE == MPC_TYPE_E4M3) {
            u32x4 b0[MF], b1[MF];
#pragma unroll
            for (int m = 0; m < MF; ++m) b0[m] = xfrag(m, g), b1[m] = xfrag(m, g + 4);
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const u32x4 a0 = wfrag(f, g), a1 = wfrag(f, g + 4);
#pragma unroll
                for (int m = 0; m < MF; ++m) acc[f][m] = Operand<TYPE>::mma(a0, a1, b0[m], b1[m], acc[f][m]);
            }
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4 b[MF];
#pragma unroll
                for (int m = 0; m < MF; ++m) b[m] = xfrag(m, 4 * s + g);
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    const u32x4 w4 = wfrag(f, 4 * s + g);
#pragma unroll
                    for (int m = 0; m < MF; ++m) acc[f][m] = Operand<TYPE>::mma(w4, b[m], acc[f][m]);
                }
            }
        }
        if (more) stash(buf ^ 1);            // (the other buffer was last read before the previous barrier)
        __syncthreads();
    }

    const int64_t n = n0 + wn + g * V;
    if (n >= a.N) return;
    float b[V], s[V];
    column_terms<V>(a, n, b, s);
#pragma unroll
    for (int m = 0; m < MF; ++m) {
        const int64_t row = m0 + wm + m * 16 + j;
        if (row >= a.M) continue;
        float v[V];
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[4 * f + r] = acc[f][m][r];
        epilogue<V>(a, row, n, v, b, s);
    }
}

template <int TYPE, int BM, int BN, int WM, int WN>
int launch_tiles(mpc_ctx *ctx, LinearArgs a) {
    constexpr size_t lds = 2 * (BM + BN) * KT;
    auto kern = linear_tile_kernel<TYPE, BM, BN, WM, WN>;
    static bool attr_set[MPC_MAX_DEVICES] = {};
    bool &attr_done = attr_set[ctx->device];
    if (lds > 48 * 1024 && !attr_done) {
        MPC_HIP(ctx, hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        attr_done = true;
    }
    const int64_t tm = mpc_cdiv(a.M, BM), tn = mpc_cdiv(a.N, BN);
    MPC_REQUIRE(ctx, tm * tn < (1ll << 31), "linear: too many tiles");
    a.tiles_m = (int)tm;
    a.tiles_n = (int)tn;
    kern<<<dim3((unsigned)(tm * tn)), dim3(64 * (BM / WM) * (BN / WN)), lds, ctx->stream>>>(a);
    MPC_CHECK_LAUNCH(ctx, "linear_tile");
    return MPC_OK;
}

template <int TYPE>
int launch(mpc_ctx *ctx, const LinearArgs &a) {
    return launch_tiles<TYPE, 128, 128, 64, 64>(ctx, a);
}

bool linear_desc_ok(const mpc_linear_desc &d) {
    const bool in16 = d.in_type == MPC_TYPE_F16 || d.in_type == MPC_TYPE_BF16;
    return (in16 || d.in_type == MPC_TYPE_E4M3) &&
           (d.out_type == MPC_TYPE_F32 || d.out_type == MPC_TYPE_F16 || d.out_type == MPC_TYPE_BF16) &&
           (d.act == MPC_ACT_NONE || d.act == MPC_ACT_RELU || d.act == MPC_ACT_GELU || d.act == MPC_ACT_SILU) && d.M >= 0 &&
           d.M < (1ll << 31) && d.N > 0 && d.N < (1ll << 31) && d.K > 0 && d.K < (1ll << 31) && d.x_stride >= 0 && d.w_stride >= 0 &&
           d.residual_stride >= 0 && d.out_stride >= d.N;
}

}  // namespace

extern "C" size_t mpc_linear_workspace_bytes(const mpc_linear_desc *desc) {
    (void)desc;
    return 0;
}

extern "C" int mpc_linear_forward(mpc_ctx *ctx, const mpc_linear_desc *desc, const void *x, const float *x_scale, const void *w,
                                  const float *w_scale, const float *bias, const void *residual, void *workspace, size_t workspace_bytes,
                                  void *out) {
    MPC_ENTER(ctx);
    MPC_REQUIRE(ctx, desc, "linear: null description");
    const mpc_linear_desc &d = *desc;
    MPC_REQUIRE(ctx, linear_desc_ok(d), "linear: types %d -> %d, activation %d, M = %lld, N = %lld, K = %lld or a stride is not supported",
                d.in_type, d.out_type, d.act, (long long)d.M, (long long)d.N, (long long)d.K);
    if (d.M == 0) return MPC_OK;
    MPC_REQUIRE(ctx, x && w && out, "linear: null pointer");
    const bool eight = d.in_type == MPC_TYPE_E4M3;
    MPC_REQUIRE(ctx, (x_scale != nullptr) == eight && (w_scale != nullptr) == eight, "linear: scales go with e4m3 operands, both of them");
    MPC_REQUIRE(ctx, workspace_bytes >= mpc_linear_workspace_bytes(desc), "linear: workspace of %zu bytes", workspace_bytes);
    const int ib = mpc_type_bytes(d.in_type), ob = mpc_type_bytes(d.out_type);
    MPC_REQUIRE(ctx, ((uintptr_t)x | (uintptr_t)w) % ib == 0 && ((uintptr_t)out | (uintptr_t)residual) % ob == 0, "linear: misaligned pointer");
    LinearArgs a{};
    a.x = (const char *)x, a.w = (const char *)w;
    a.M = d.M, a.N = d.N, a.K = d.K * ib;
    a.xs = d.x_stride * ib, a.ws = d.w_stride * ib;
    a.sx = x_scale, a.sw = w_scale, a.bias = bias;
    a.res = (const char *)residual, a.out = (char *)out;
    a.rs = d.residual_stride * ob, a.os = d.out_stride * ob;
    a.out_type = d.out_type, a.act = d.act;
    a.vec_out = (uintptr_t)out % 16 == 0 && a.os % 16 == 0;
    a.vec_res = (uintptr_t)residual % 16 == 0 && a.rs % 16 == 0;
    (void)workspace;
    if (d.in_type == MPC_TYPE_F16) return launch<MPC_TYPE_F16>(ctx, a);
    if (d.in_type == MPC_TYPE_BF16) return launch<MPC_TYPE_BF16>(ctx, a);
    return launch<MPC_TYPE_E4M3>(ctx, a);
}
