// Matrix product with its epilogue fused: out[m][n] = act(sx[m] sw[n] sum_k x[m][k] w[n][k] + b[n]) + r[m][n].
//
// Both operands lie with k innermost, which is how the matrix instructions want them: a lane of a 16x16 tile holds 16
// (16-bit operands: 8 values; e4m3: 16, two such pieces) consecutive bytes of one row.  A k-tile is 128 bytes of every
// row, 64 values of 16 bits or 128 of 8, so both widths move the same bytes and issue the same matrix cycles per tile.
// w is the instruction's first operand: a lane then holds four consecutive n of one m.  Which row of w a lane brings is
// free, so two tiles take the rows of 32 columns interleaved in fours: a lane ends up with runs of 8 consecutive outputs of
// one row, 16 bytes of a 16-bit type, and the four lanes of a row with 32 consecutive ones.
//
// What bounds the four kernels, and what they take (plan_for chooses; a large copy reaches 5.17 TB/s here, a large library product
// 1574 TFLOP/s in bf16 and 3090 in e4m3): few rows, the weights' bytes: 1 x 4096 -> 4096 bf16 7.6 us, 4.4 TB/s.  64 x 64 tiles, the
// way of a k-tile through the one or two workgroups of a CU: 1537 x 1111 -> 1000 bf16 18.6 us, rows at odd addresses.  128 x 128 tiles,
// load, products and epilogue of a tile one after the other, two workgroups per CU: 36864 x 256 -> 1024 f16 with gelu 44 us, 36864 x
// 1024 -> 256 e4m3 with residual 24 us.  256 x 256 tiles, at 2.0 GHz under their load with the matrix pipes busy 56 % of the cycles:
// 8192 x 4096 -> 8192 with residual and activation, bf16 460 us, 1200 TFLOP/s; e4m3 301 us, 1830 TFLOP/s.
#include "row_ops.h"

#include <type_traits>

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x8 __attribute__((ext_vector_type(8)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));          // a 16-byte access at any address
typedef u32x4 u32x4_word __attribute__((aligned(4)));         // at any word
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
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
    int tiles_m, tiles_n;
    float *partial;                   // [splits][M][N] sums, where K is split
};

// ---- epilogue ---------------------------------------------------------------------------------------------------------
// log2 F(-m), F the normal distribution, as a polynomial in m (constant first) for gelu in 16-bit outputs: fitted as far as gelu's
// left tail stays in the type, and falling beyond.  With its roundings F is good to 2^-15.3 of itself for fp16 (m up to 5.8), 2^-12.1 for
// bf16 (13.3), a twentieth and a ninth of half a step, and to 3.5e-7 in absolute terms.
template <typename T>
struct TailExponent;
template <>
struct TailExponent<f16_t> {
    static constexpr float P[] = {-0.999999583f, -1.15112638f, -0.459036678f, -0.0529954731f, 0.0077384538f, -0.000608425296f, -1.10764704e-05f,
                                  6.52565996e-06f, -3.8450608e-07f};
};
template <>
struct TailExponent<bf16_t> {
    static constexpr float P[] = {-0.999999046f, -1.15114987f, -0.458879262f, -0.0533608608f, 0.00811367016f, -0.000794931198f, 3.39617181e-05f,
                                  1.83778775e-06f, -3.23463979e-07f, 1.63099578e-08f, -2.98272906e-10f};
};

// V consecutive outputs of row m from column n on, T their type.  v: the sums.
template <typename T, int V>
__device__ __forceinline__ void activate(float (&v)[V], int act) {
    if (act == MPC_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];            // (a NaN stays)
    } else if (act == MPC_ACT_GELU) {
        // gelu(v) = max(v, 0) - |v| F(-|v|), F the normal distribution.  gelu(inf) = inf (1e30 * 0 is subtracted); at -inf the
        // formula's -inf * 0 is NaN, here as in silu.  All fits are for the least largest error, by linear programs.
        if constexpr (sizeof(T) == 2) {
            // F(-m) = 2^P(m), one exponential and as few other instructions as the type's half step allows (TailExponent).  (36864 x 256
            // -> 1024, this : a formula good to 2^-16 for both, with a reciprocal : degree 5, good to 3e-7 of |v| but to no digit at v = -8:
            // f16 53 us : 55 : 50, bf16 48 : 50 : 44; 8192 x 4096 -> 8192 e4m3 with residual 308 : 318 : 300.)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float m = fabsf(v[i]);
                constexpr int N = sizeof(TailExponent<T>::P) / sizeof(float);
                float q = TailExponent<T>::P[N - 1];
#pragma unroll
                for (int k = N - 2; k >= 0; --k) q = fmaf(m, q, TailExponent<T>::P[k]);
                v[i] = fmaf(-fabsf(__builtin_fminf(v[i], 1e30f)), __builtin_amdgcn_exp2f(q), __builtin_fmaxf(v[i], 0.0f));
            }
        } else {
            // F(-m) = exp(-m^2 / 2) t q(t), t = 1 / (1 + 0.33 m), q of degree 8 fitted relative to F on 0 <= m <= 13.5, beyond which exp is
            // 0: t q(t) is good to 2^-21.5 with its roundings, and what those of the exponent lose is taken along: 2^-20 in all.
            constexpr float C = 0.72134752f, C_REST = 9.6298152e-9f;             // 1 / (2 ln 2)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float m = fabsf(v[i]);
                m = m > 20.0f ? 20.0f : m;                                       // (a NaN stays)
                const float m2 = m * m, z = m2 * -C;
                const float rest = fmaf(fmaf(m, m, -m2), -C, fmaf(m2, -C_REST, fmaf(m2, -C, -z)));
                float e = __builtin_amdgcn_exp2f(z);
                e = fmaf(e * rest, 0.69314718f, e);
                const float t = __builtin_amdgcn_rcpf(fmaf(m, 0.33f, 1.0f));
                float q = fmaf(t, -0.0211830456f, 0.124867819f);
                q = fmaf(t, q, -0.270793527f);
                q = fmaf(t, q, 0.228645995f);
                q = fmaf(t, q, -0.0592148937f);
                q = fmaf(t, q, 0.122923814f);
                q = fmaf(t, q, 0.110794663f);
                q = fmaf(t, q, 0.13233906f);
                q = fmaf(t, q, 0.131620139f);
                v[i] = fmaf(-fabsf(__builtin_fminf(v[i], 1e30f)), q * t * e, __builtin_fmaxf(v[i], 0.0f));
            }
        }
    } else if (act == MPC_ACT_SILU) {
        // v / (1 + exp(-v)).  exp's argument is off by 1.22 half steps, 1.22 |v| 2^-24 of the left tail: 2^-17 where silu leaves bf16's
        // range.  An fp32 output, for which that is many units, takes the steps' losses along, by e = exp(-|v|) so that nothing
        // overflows (36864 x 256 -> 1024 f16 -> fp32 49 us : 54).  Below exp's normal range it counts as 0, here 2^-119 and less.
        constexpr float L = 1.44269504f, L_REST = 1.9259630e-8f;                 // 1 / ln 2
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (sizeof(T) == 4) {
                float m = fabsf(v[i]);
                m = m > 200.0f ? 200.0f : m;                                     // (a NaN stays)
                const float z = m * -L, rest = fmaf(m, -L_REST, fmaf(m, -L, -z));
                float e = __builtin_amdgcn_exp2f(z);
                e = fmaf(e * rest, 0.69314718f, e);
                v[i] = (v[i] > 0.0f ? v[i] : v[i] * e) * __builtin_amdgcn_rcpf(1.0f + e);
            } else {
                v[i] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v[i] * -L));
            }
        }
    }
}

// One of the rows kept in registers, whose index is known only at run time: a copy for each (the empty asm keeps the copies
// from being merged into one through a pointer, which would put the rows into memory).
template <int ROWS, int P, typename Vec, int M = 0>
__device__ __forceinline__ void take_row(const Vec (&rows)[ROWS][P], int m, Vec (&out)[P]) {
    if constexpr (M + 1 < ROWS) {
        if (m != M) return take_row<ROWS, P, Vec, M + 1>(rows, m, out);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
        u32x4 t = __builtin_bit_cast(u32x4, rows[M][i]);
        asm("" : "+v"(t));
        out[i] = __builtin_bit_cast(Vec, t);
    }
}

// Eight 16-bit values to an address between words: the words in the middle as such, a value at each end.  (36864 x 256 -> 1023
// f16: 57 us with one access at such an address, 49 with these.  The residual's loads gain nothing from the like, and the 256 x 256
// tiles less than they lose in registers.)
template <typename T, typename Vec>
__device__ __forceinline__ void store_between_words(T *to, Vec t) {
    if constexpr (sizeof(T) == 2) {
        typedef unsigned u32x3 __attribute__((ext_vector_type(3)));
        typedef u32x3 u32x3_word __attribute__((aligned(4)));
        const u32x4 v = __builtin_bit_cast(u32x4, t);
        to[0] = t[0];
        *(u32x3_word *)(to + 1) = u32x3{__builtin_amdgcn_alignbyte(v[1], v[0], 2), __builtin_amdgcn_alignbyte(v[2], v[1], 2),
                                        __builtin_amdgcn_alignbyte(v[3], v[2], 2)};
        to[7] = t[7];
    }
}

// The rows of a lane: row0 + 16 m; its V columns are V / 8 runs of 8, n + 32 t .. n + 32 t + 7: the four lanes of a row then
// write 64 consecutive bytes at a time.  take(m, v) gives the sums.  One rolled loop (the sums have fixed
// registers, so take is a switch over copies): unrolled it would be tens of KB of code.
template <typename T, int MF, int V, typename Take>
__device__ __forceinline__ void finish_rows(const LinearArgs &a, int64_t row0, int64_t n, Take take) {
    constexpr int PER = 16 / sizeof(T), P = V / PER, RUN = 8 / PER;         // values of a 16-byte piece, pieces of a lane and of a run
    typedef T vec_t __attribute__((ext_vector_type(PER)));
    typedef vec_t vec_any __attribute__((aligned(sizeof(T))));              // (rows may begin at any element)
    auto col = [&](int i) { return n + (i & 7) + 32 * (i >> 3); };          // column of value i
    float b[V], s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        b[i] = a.bias && col(i) < a.N ? a.bias[col(i)] : 0.0f;
        s[i] = a.sw && col(i) < a.N ? a.sw[col(i)] : 1.0f;
    }
    const bool between = ((uintptr_t)a.out | a.os) & 3;                     // rows of the output may begin between words
    // the residual's rows: up to four at once for 16-bit types, the next one while a row is worked on for fp32
    constexpr int KEPT = sizeof(T) == 2 ? (MF < 4 ? MF : 4) : 1;
    vec_t ahead[KEPT][P];
    auto fetch = [&](int m, vec_t (&to)[P]) {
        const int64_t row = row0 + 16 * m < a.M ? row0 + 16 * m : a.M - 1;
        const T *r = (const T *)(a.res + row * a.rs);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (col(i / RUN * 8 + 7) < a.N) {
                to[i] = *(const vec_any *)(r + col(i * PER));
            } else {                                          // a run that the row ends in, or before
#pragma unroll
                for (int q = 0; q < PER; ++q) to[i][q] = col(i * PER + q) < a.N ? r[col(i * PER + q)] : (T)0.0f;
            }
        }
    };
    if (a.res && KEPT == 1) fetch(0, ahead[0]);
#pragma unroll 1
    for (int m = 0; m < MF; ++m) {
        const int64_t row = row0 + 16 * m;
        if (a.res && KEPT > 1 && m % KEPT == 0) {
#pragma unroll
            for (int i = 0; i < KEPT; ++i) fetch(m + i, ahead[i]);
        }
        float v[V];
        take(m, v);
        vec_t res[P];
        if (a.res) {
            take_row<KEPT, P>(ahead, m % KEPT, res);
            if (KEPT == 1 && m + 1 < MF) fetch(m + 1, ahead[0]);
        }
        if (row >= a.M) break;
        if (a.sx) {
            const float sx = a.sx[row];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] *= sx * s[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += b[i];
        activate<T, V>(v, a.act);
        if (a.res) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += (float)res[i / PER][i % PER];
        }
        T *o = (T *)(a.out + row * a.os);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            vec_t t;
#pragma unroll
            for (int q = 0; q < PER; ++q) t[q] = (T)v[i * PER + q];
            if (col(i / RUN * 8 + 7) < a.N) {
                T *to = o + col(i * PER);
                if (sizeof(T) == 2 && V < 32 && between && (uintptr_t)to & 2) store_between_words(to, t);
                else *(vec_any *)to = t;
            } else {
#pragma unroll
                for (int q = 0; q < PER; ++q)
                    if (col(i * PER + q) < a.N) o[col(i * PER + q)] = t[q];
            }
        }
    }
}

// V consecutive outputs of row m from column n on, whose sums have their scales and bias; for single values and the joined ones
template <typename T, int V>
__device__ __forceinline__ void finish_typed(const LinearArgs &a, int64_t m, int64_t n, float (&v)[V]) {
    activate<T, V>(v, a.act);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (n + i >= a.N) break;
        if (a.res) v[i] += (float)((const T *)(a.res + m * a.rs))[n + i];
        ((T *)(a.out + m * a.os))[n + i] = (T)v[i];
    }
}
template <int V>
__device__ __forceinline__ void finish_values(const LinearArgs &a, int64_t m, int64_t n, float (&v)[V]) {
    if (a.out_type == MPC_TYPE_F32) finish_typed<float>(a, m, n, v);
    else if (a.out_type == MPC_TYPE_F16) finish_typed<f16_t>(a, m, n, v);
    else finish_typed<bf16_t>(a, m, n, v);
}

template <int MF, int V, typename Take>
__device__ __forceinline__ void epilogue(const LinearArgs &a, int64_t row0, int64_t n, Take take) {
    if (n >= a.N) return;
    if (a.out_type == MPC_TYPE_F32) finish_rows<float, MF, V>(a, row0, n, take);
    else if (a.out_type == MPC_TYPE_F16) finish_rows<f16_t, MF, V>(a, row0, n, take);
    else finish_rows<bf16_t, MF, V>(a, row0, n, take);
}

// sums of x tile m as the V outputs of a lane's row
template <int MF, int NF, int M = 0>
__device__ __forceinline__ void take_tile(const f32x4 (&acc)[NF][MF], int m, float (&v)[4 * NF]) {
    if constexpr (M + 1 < MF) {
        if (m != M) return take_tile<MF, NF, M + 1>(acc, m, v);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float t = acc[f][M][r];
            asm("" : "+v"(t));                  // (else the copies are merged into one through a pointer, and the sums go to memory for it)
            v[4 * f + r] = t;
        }
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
    // 128 values of k in one instruction; the block scales of its format are all 1 (exponent 127).  The 8-bit instructions of
    // this GPU, this one and those of 16 and 32 k alike, add the products of eight neighbouring k on a grid of 2^-13 of the
    // largest one's power of two and the eights in fp32: 1.5e-5 of a sum of random values, an eighth of an fp16 rounding
    // and far below the operands' own 2^-4.  Products exact in fp32 take the 16-bit instructions, at half the rate: mma_exact.
    static __device__ __forceinline__ f32x4 mma(u32x4 a0, u32x4 a1, u32x4 b0, u32x4 b1, f32x4 c) {
        const i32x8 a = {(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3], (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
        const i32x8 b = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
    }
    // The same sums with products exact in fp32: every e4m3 value is an fp16 one.  For few rows, which wait for memory, the
    // conversions and twice the matrix cycles cost little (8-bit instructions : these: 7 x 4096 -> 4096 9.7 us : 9.7, 16 x 8192 -> 8192
    // 17.1 : 17.6, 32 x 8192 -> 8192 26.1 : 27.4, 16 x 512 -> 60000 20.5 : 18.1).
    static __device__ __forceinline__ half8 widen(unsigned lo, unsigned hi) {
        const half2 p[4] = {pair<false>(lo), pair<true>(lo), pair<false>(hi), pair<true>(hi)};
        return half8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
    }
    static __device__ __forceinline__ f32x4 mma_exact(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
        for (int h = 0; h < 4; h += 2) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(a[h], a[h + 1]), widen(b[h], b[h + 1]), c, 0, 0, 0);
        return c;
    }

private:
    template <bool HIGH>
    static __device__ __forceinline__ half2 pair(unsigned v) {
        return __builtin_bit_cast(half2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)v, 1.0f, HIGH));
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

__device__ __forceinline__ void lds_barrier() {               // LDS accesses done, then the barrier; memory loads stay in flight
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Tile of workgroup b: each XCD (workgroups go to the 8 in turn) gets a contiguous run of the tiles, in groups of 8 tile
// rows with the rows innermost, so that the tiles an XCD works on at a time share operands in its L2.
__device__ __forceinline__ void tile_of(int b, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int total = tiles_m * tiles_n, xcd = b & 7, per = total >> 3, rest = total & 7;
    const int i = xcd * per + (xcd < rest ? xcd : rest) + (b >> 3);
    const int group = 8 * tiles_n, first = i / group * 8, rows = tiles_m - first < 8 ? tiles_m - first : 8, in = i % group;
    tm = first + in % rows;
    tn = in / rows;
}

// 16 bytes that begin `sh` bytes before the piece wanted (0 <= sh <= 16: the row ends inside it, or before it): the piece, zeros
// behind the row
__device__ __forceinline__ u32x4 row_end(u32x4 v, int sh) {
    typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
    u64x2 t = __builtin_bit_cast(u64x2, v);
    t[0] = sh & 8 ? t[1] : t[0];
    t[1] = sh & 8 ? 0 : t[1];
    const int bits = 8 * (sh & 7);
    t[0] = t[0] >> bits | t[1] << 1 << (63 - bits);
    t[1] >>= bits;
    t[0] = sh & 16 ? 0 : t[0];
    t[1] = sh & 16 ? 0 : t[1];
    return __builtin_bit_cast(u32x4, t);
}

// The 16 bytes at an address that is `s` (0 to 3) bytes behind a multiple of 4, from the 16 at the multiple and the word behind them.
// Few rows, bound by memory: 3 x 8191 -> 8192 bf16 63 us with loads at such addresses, 34 with these.  (The tiles of the other
// kernels do not gain: 8000 x 1089 -> 4000 103 us : 130.)
__device__ __forceinline__ u32x4 from_words(u32x4 v, unsigned next, unsigned s) {
    return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], s), __builtin_amdgcn_alignbyte(v[2], v[1], s), __builtin_amdgcn_alignbyte(v[3], v[2], s),
                 __builtin_amdgcn_alignbyte(next, v[3], s)};
}

// A tile's rows of an operand as a buffer that ends with the last row: a load for a row past it gives zeros or, where rows
// overlap, values of other rows; neither reaches an output.
constexpr int64_t TILE_BYTES = 1ll << 30;                         // most that a tile's rows may span (the host checks)
typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t tile_buffer(const char *base, int rows, int64_t stride, int64_t K) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)((rows - 1) * stride + K), 0x00020000);
}
__device__ __forceinline__ u32x4 buffer_piece(rsrc_t r, unsigned offset) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0));
}

// Workgroup (tile, split): BM x BN outputs over the split's k-tiles.  DEPTH k-tiles are on their way in registers while one
// is worked on from LDS, so a tile of few rows, whose matrix instructions do not cover a memory access, is not bound by
// it.  Operand rows may begin at any element.  In the last k-tile, if the row ends inside it, a piece past the row's end is
// loaded from its last 16 bytes and shifted.
template <int TYPE, int BM, int BN, int WM, int WN, int DEPTH, int PER_SIMD>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), PER_SIMD) void linear_tile_kernel(LinearArgs a) {
    constexpr int NT = 64 * (BM / WM) * (BN / WN), TURN = DEPTH % 2 ? 2 * DEPTH : DEPTH;
    constexpr int MF = WM / 16, NF = WN / 16, V = 4 * NF;
    constexpr int XP = BM * 8 / NT, WP = BN * 8 / NT;             // 16-byte pieces per thread and tile
    extern __shared__ u32x4 lds[];                                // 2 x [BM + BN rows][8 pieces]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int j = lane & 15, g = lane >> 4;
    const int wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
    int tm, tn;
    tile_of(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int rows_x = (int)(a.M - m0 < BM ? a.M - m0 : BM), rows_w = (int)(a.N - n0 < BN ? a.N - n0 : BN);
    const rsrc_t xb = tile_buffer(a.x + m0 * a.xs, rows_x, a.xs, a.K), wb = tile_buffer(a.w + n0 * a.ws, rows_w, a.ws, a.K);
    // this split's k-tiles: T, the last split's last one being the one in which the rows end (if they end inside one)
    const int K = (int)a.K, whole = K / KT, all = (K + KT - 1) / KT;
    const int t0 = (int)((int64_t)all * blockIdx.y / gridDim.y), t1 = (int)((int64_t)all * (blockIdx.y + 1) / gridDim.y);
    const int T = K >= 16 ? t1 - t0 : 0;
    const bool ends = t1 > whole;

    // Piece p of row r lies at slot p ^ key(r): the 16 rows that one instruction reads at the same p then spread over the banks.
    auto xkey = [](int r) { return r & 7; };
    auto wkey = [](int r) { return (r & 3) | (r >> 3 & 1) << 2; };
    const int p = tid & 7, r0 = tid >> 3;
    const unsigned xo = r0 * (unsigned)a.xs, wo = r0 * (unsigned)a.ws, xstep = (unsigned)a.xs * (NT / 8), wstep = (unsigned)a.ws * (NT / 8);
    u32x4 xr[DEPTH][XP], wr[DEPTH][WP];
    auto fetch = [&](int slot, int t) {                           // (past the row's end: its last piece)
        const int at = (t0 + t) * KT + p * 16, off = at < K - 16 ? at : K - 16;
#pragma unroll
        for (int i = 0; i < XP; ++i) xr[slot][i] = buffer_piece(xb, xo + off + i * xstep);
#pragma unroll
        for (int i = 0; i < WP; ++i) wr[slot][i] = buffer_piece(wb, wo + off + i * wstep);
    };
    const int over = whole * KT + p * 16 - (K - 16), sh = over < 0 ? 0 : over > 16 ? 16 : over;
    auto finish = [&](int slot) {                                 // pieces of the tile in which the rows end
#pragma unroll
        for (int i = 0; i < XP; ++i) xr[slot][i] = row_end(xr[slot][i], sh);
#pragma unroll
        for (int i = 0; i < WP; ++i) wr[slot][i] = row_end(wr[slot][i], sh);
    };
    auto stash = [&](int slot, int buf) {
        u32x4 *x = lds + buf * (BM + BN) * 8, *w = x + BM * 8;
#pragma unroll
        for (int i = 0; i < XP; ++i) {
            const int r = r0 + i * (NT / 8);
            x[r * 8 + (p ^ xkey(r))] = xr[slot][i];
        }
#pragma unroll
        for (int i = 0; i < WP; ++i) {
            const int r = r0 + i * (NT / 8);
            w[r * 8 + (p ^ wkey(r))] = wr[slot][i];
        }
    };
    f32x4 acc[NF][MF];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int m = 0; m < MF; ++m) acc[f][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // One k-tile from LDS buffer buf.  Its operands are asked for first, all of them: their way from LDS is paid once, not once
    // per group of instructions; `beside` follows them.
    auto multiply = [&](int buf, auto beside) {
        const u32x4 *x = lds + buf * (BM + BN) * 8, *w = x + BM * 8;
        u32x4 xv[2][MF], wv[2][NF];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int m = 0; m < MF; ++m) {
                const int r = wm + m * 16 + j;
                xv[c][m] = x[r * 8 + ((4 * c + g) ^ xkey(r))];
            }
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const int r = wn + (f >> 1) * 32 + (j >> 2) * 8 + (f & 1) * 4 + (j & 3);
                wv[c][f] = w[r * 8 + ((4 * c + g) ^ wkey(r))];
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        beside();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (TYPE == MPC_TYPE_E4M3) {
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int m = 0; m < MF; ++m) acc[f][m] = Operand<TYPE>::mma(wv[0][f], wv[1][f], xv[0][m], xv[1][m], acc[f][m]);
        } else {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int f = 0; f < NF; ++f)
#pragma unroll
                    for (int m = 0; m < MF; ++m) acc[f][m] = Operand<TYPE>::mma(wv[c][f], xv[c][m], acc[f][m]);
        }
    };
    // Tile t from LDS buffer t & 1; tile t + 1 waits in slot (t + 1) % DEPTH.
    auto step = [&](int buf, int slot, int t) {
        multiply(buf, [&] {
            if (DEPTH > 1 && ends && t + 2 == T) finish(slot);
            stash(slot, buf ^ 1);                                 // (last read before the previous barrier)
            fetch(slot, t + 1 + DEPTH);
        });
        lds_barrier();
    };
    if (T > 0) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) fetch(d, d);
        if (ends && T == 1) finish(0);
        stash(0, 0);
    }
    if constexpr (DEPTH == 1) {                                   // the only tile on its way is the one waited for
        if (T > 0) {
            if (T > 1) fetch(0, 1);
            lds_barrier();
            int t = 0;
            for (; t + 2 < T; ++t) step(t & 1, 0, t);
            if (t + 1 < T) {
                multiply(t & 1, [&] {
                    if (ends) finish(0);
                    stash(0, ~t & 1);
                });
                lds_barrier();
                ++t;
            }
            multiply(t & 1, [] {});
        }
    } else if (T > 0) {
        // Tiles past the last are fetched and stored like the others, and never read: a fetch under a condition would make the
        // compiler wait for every load in flight, since it could not count on the younger ones.
        fetch(0, DEPTH);
        lds_barrier();
        for (int t = 0;; t += TURN) {
#pragma unroll
            for (int i = 0; i < TURN; ++i) {
                if (t + i >= T) goto done;
                step(i & 1, (i + 1) % DEPTH, t + i);
            }
        }
    }
done:
    if (K < 16) {                                                 // rows shorter than a piece: value by value (in one split)
#pragma unroll
        for (int i = 0; i < XP; ++i) {
            const int r = r0 + i * (NT / 8);
            xr[0][i] = load_piece<Operand<TYPE>::BYTES>(a.x + (m0 + r) * a.xs, m0 + r < a.M ? K - p * 16 : 0);
        }
#pragma unroll
        for (int i = 0; i < WP; ++i) {
            const int r = r0 + i * (NT / 8);
            wr[0][i] = load_piece<Operand<TYPE>::BYTES>(a.w + (n0 + r) * a.ws, n0 + r < a.N ? K - p * 16 : 0);
        }
        stash(0, 0);
        lds_barrier();
        multiply(0, [] {});
    }
    if (gridDim.y > 1) {                                          // the sums as they are; linear_join_kernel finishes them
        LinearArgs sums = a;
        sums.sx = sums.sw = sums.bias = nullptr;
        sums.res = nullptr;
        sums.out = (char *)(a.partial + (int64_t)blockIdx.y * a.M * a.N);
        sums.os = a.N * 4;
        sums.out_type = MPC_TYPE_F32, sums.act = MPC_ACT_NONE;
        finish_rows<float, MF, V>(sums, m0 + wm + j, n0 + wn + g * 8, [&](int m, float (&v)[V]) { take_tile<MF, NF>(acc, m, v); });
        return;
    }
    epilogue<MF, V>(a, m0 + wm + j, n0 + wn + g * 8, [&](int m, float (&v)[V]) { take_tile<MF, NF>(acc, m, v); });
}

// Adds up the splits' sums, in their order, and finishes: four columns of a row per thread.
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a, int splits) {
    const int64_t per_row = (a.N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.M * per_row) return;
    const int64_t m = i / per_row, n = i % per_row * 4, plane = a.M * a.N;
    const float *s = a.partial + m * a.N + n;
    typedef f32x4 f32x4_any __attribute__((aligned(4)));
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int z = 0; z < splits; ++z) {
        if (n + 4 <= a.N) {
            const f32x4 t = *(const f32x4_any *)(s + z * plane);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] += t[c];
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (n + c < a.N) v[c] += s[z * plane + c];
        }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (n + c >= a.N) break;
        if (a.sx) v[c] *= a.sx[m] * a.sw[n + c];
        if (a.bias) v[c] += a.bias[n + c];
    }
    finish_values(a, m, n, v);
}

// Lets a kernel use more LDS than a launch may ask for by default.  Done for all of them when a context is made (`prepare`), so
// that a first call may well be a captured one.
int allow_lds(mpc_ctx *ctx, const void *kernel, size_t bytes) {
    MPC_HIP(ctx, hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return MPC_OK;
}

// The tiles, of bm x bn outputs and a workgroup each, in as many launches as they take: one has fewer than 2^32 threads.
template <typename F>
void in_parts(const LinearArgs &a, int bm, int bn, int threads, F run) {
    const int64_t most = MPC_LAUNCH_THREADS / threads, all_n = mpc_cdiv(a.N, bn), tiles_n = all_n < most ? all_n : most;
    const int64_t rows = most / tiles_n * bm, columns = tiles_n * bn;
    const int ob = mpc_type_bytes(a.out_type);
    for (int64_t m = 0; m < a.M; m += rows) {
        for (int64_t n = 0; n < a.N; n += columns) {
            LinearArgs part = a;
            part.M = a.M - m < rows ? a.M - m : rows;
            part.N = a.N - n < columns ? a.N - n : columns;
            part.tiles_m = (int)mpc_cdiv(part.M, bm);
            part.tiles_n = (int)mpc_cdiv(part.N, bn);
            part.x = a.x + m * a.xs;
            part.w = a.w + n * a.ws;
            if (a.sx) part.sx = a.sx + m, part.sw = a.sw + n;
            if (a.bias) part.bias = a.bias + n;
            if (a.res) part.res = a.res + m * a.rs + n * ob;
            part.out = a.out + m * a.os + n * ob;
            run(part);
        }
    }
}

template <int TYPE, int BM, int BN, int WM, int WN, int DEPTH, int PER_SIMD>
int launch_tiles(mpc_ctx *ctx, const LinearArgs &a, int splits, bool prepare = false) {
    constexpr size_t lds = 2 * (BM + BN) * KT;
    auto kern = linear_tile_kernel<TYPE, BM, BN, WM, WN, DEPTH, PER_SIMD>;
    if (prepare) return allow_lds(ctx, (const void *)kern, lds);
    constexpr int NT = 64 * (BM / WM) * (BN / WN);
    in_parts(a, BM, BN, NT, [&](const LinearArgs &part) {
        kern<<<dim3((unsigned)(part.tiles_m * part.tiles_n), (unsigned)splits), dim3(NT), lds, ctx->stream>>>(part);
    });
    MPC_CHECK_LAUNCH(ctx, "linear_tile");
    if (splits > 1) {                                             // (few tiles: one part)
        linear_join_kernel<<<dim3((unsigned)mpc_cdiv(a.M * ((a.N + 3) / 4), 256)), dim3(256), 0, ctx->stream>>>(a, splits);
        MPC_CHECK_LAUNCH(ctx, "linear_join");
    }
    return MPC_OK;
}

// ---- large products: 256 x 256 tiles, one workgroup per CU -------------------------------------------------------------------
// Four waves, each 128 x 128 outputs in 256 accumulator registers: a wave then reads 32 KB of LDS per k-tile for 2048 cycles
// of matrix instructions (the four of a CU 64 bytes a cycle; waves of 64 x 64 would need all 128 that LDS delivers).  With one
// wave per SIMD nothing else hides its latencies, so they are hidden in the wave itself: a k-tile is four quadrants of
// 64 x 64, and while one multiplies, the operands of the next come from LDS, the pieces of the next k-tile go from
// registers to the other LDS buffer and those of the one after leave for memory.  The last quadrant of a tile shares no
// operand with the first of the next, so the order of the w halves alternates from tile to tile.
constexpr int BIG = 256;

// c += a b with c in accumulation registers, in place.  All 256 of them hold sums here; through the builtin the compiler moves
// sums from register to register (a result need not go where its input was), with none left to move them through: twice as
// many moves as products, and spills.  Operands come from LDS or memory reads, which the compiler waits for; two
// instructions on the same sums are at least 16 apart, and the kernel waits before it reads them.
template <int TYPE>
__device__ __forceinline__ void mma_in_place(u32x4 a, u32x4 b, f32x4 &c) {
    if constexpr (TYPE == MPC_TYPE_F16) asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <int TYPE>
__device__ __forceinline__ void mma_in_place(u32x4 a0, u32x4 a1, u32x4 b0, u32x4 b1, f32x4 &c) {
    const u32x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
    asm("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));       // (both formats default to e4m3, no block scales)
}

template <int TYPE>
__global__ __launch_bounds__(256, 1) void linear_big_kernel(LinearArgs a) {
    constexpr int V = 32;                                     // consecutive outputs of a lane
    extern __shared__ u32x4 lds[];                            // 2 x [256 rows of x, 256 of w][8 pieces]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 15, g = lane >> 4;
    const int wm = (wave & 1) * 128, wn = (wave >> 1) * 128;
    int tm, tn;
    tile_of(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * BIG, n0 = (int64_t)tn * BIG;
    const int rows_x = (int)(a.M - m0 < BIG ? a.M - m0 : BIG), rows_w = (int)(a.N - n0 < BIG ? a.N - n0 : BIG);

    const rsrc_t xr = tile_buffer(a.x + m0 * a.xs, rows_x, a.xs, a.K), wr = tile_buffer(a.w + n0 * a.ws, rows_w, a.ws, a.K);
    const int p = tid & 7, r0 = tid >> 3;
    const unsigned xo = r0 * (unsigned)a.xs + p * 16, wo = r0 * (unsigned)a.ws + p * 16;
    const unsigned xstep = 32 * (unsigned)a.xs, wstep = 32 * (unsigned)a.ws;
    u32x4 xg[8], wg[8];
    // The last k-tile, which may end early, comes first, before the loop: it takes care of its end there.  The others follow,
    // and tiles of zeros (from behind the buffer) behind them.
    const int K = (int)a.K, last = (K - 1) / KT * KT, all = last + KT;
    auto k_offset = [&](int k) { return k < all ? (unsigned)(k - KT) : 0x80000000u; };
    auto fetch_x = [&](int i, unsigned ko) { xg[i] = buffer_piece(xr, xo + ko + i * xstep); };
    auto fetch_w = [&](int i, unsigned ko) { wg[i] = buffer_piece(wr, wo + ko + i * wstep); };
    // LDS slots, as in the kernel above: piece p of row r at p ^ key(r); rows of w are read interleaved, so its
    // key takes bit 3 of the row.  [x buffer 0][x buffer 1][w buffer 0][w buffer 1], each 256 rows of 8 pieces.
    u32x4 *const xdst = lds + r0 * 8 + (p ^ (r0 & 7));
    u32x4 *const wdst = lds + 2 * BIG * 8 + r0 * 8 + (p ^ ((r0 & 3) | (r0 >> 3 & 1) << 2));
    auto stash_x = [&](int i, int buf) { xdst[buf * (BIG * 8) + i * 256] = xg[i]; };
    auto stash_w = [&](int i, int buf) { wdst[buf * (BIG * 8) + i * 256] = wg[i]; };
    // Piece n of 16 goes to LDS and the one of the tile after leaves for its registers at once: it has a whole k-tile's time to arrive.
    auto move = [&](int n, int buf, unsigned ko) {
        if (n < 8) stash_x(n, buf), fetch_x(n, ko);
        else stash_w(n - 8, buf), fetch_w(n - 8, ko);
    };
    struct Half {                                             // 64 rows: 4 tiles x 2 pieces
        u32x4 v[4][2];
    };
    const u32x4 *const xsrc[2] = {lds + (wm + j) * 8 + (g ^ (j & 7)), lds + (wm + j) * 8 + ((4 + g) ^ (j & 7))};
    const int wrow = wn + (j >> 2) * 8 + (j & 3), wkey = (j & 3) | (j >> 2 & 1) << 2;
    const u32x4 *const wsrc[2] = {lds + 2 * BIG * 8 + wrow * 8 + (g ^ wkey), lds + 2 * BIG * 8 + wrow * 8 + ((4 + g) ^ wkey)};
    auto read_x = [&](Half &h, int i, int buf, int half) { h.v[i & 3][i >> 2] = xsrc[i >> 2][buf * (BIG * 8) + (half * 4 + (i & 3)) * 128]; };
    auto read_w = [&](Half &h, int i, int buf, int half) { h.v[i & 3][i >> 2] = wsrc[i >> 2][buf * (BIG * 8) + half * 512 + (i >> 1 & 1) * 256 + (i & 1) * 32]; };

    f32x4 acc[8][8];                                          // [w tile][x tile]
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
        for (int m = 0; m < 8; ++m) acc[f][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // One quadrant in eight groups of matrix instructions; beside(i) issues what goes with group i.
    auto multiply = [&](const Half &w, const Half &x, auto wh, auto xh, auto beside) {
        constexpr int F = decltype(wh)::value * 4, M = decltype(xh)::value * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            beside(i);
            if constexpr (TYPE == MPC_TYPE_E4M3) {
#pragma unroll
                for (int m = 2 * (i & 1); m < 2 * (i & 1) + 2; ++m)
                    mma_in_place<TYPE>(w.v[i >> 1][0], w.v[i >> 1][1], x.v[m][0], x.v[m][1], acc[F + (i >> 1)][M + m]);
            } else {
#pragma unroll
                for (int m = 0; m < 4; ++m) mma_in_place<TYPE>(w.v[i & 3][i >> 2], x.v[m][i >> 2], acc[F + (i & 3)][M + m]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    using Lo = std::integral_constant<int, 0>;
    using Hi = std::integral_constant<int, 1>;
    // e4m3: the lines of the tile 2 further on are brought to the L2, by loads of a word each that nothing uses: 8 x 4 workgroups
    // of an XCD share their operands and would all wait for a line that none had yet (235 -> 225 us for 8192 x 8192 x 4096;
    // 16-bit products, which meet the power limit first, gain nothing).  Each workgroup takes its share of its tile's rows.
    constexpr int AHEAD = 2;
    const rsrc_t lr = wave & 1 ? wr : xr;
    const int half = wave >> 1;
    const unsigned lo = wave & 1 ? (unsigned)(8 * ((lane & 15) + 16 * half) + (tm & 7)) * (unsigned)a.ws
                                 : (unsigned)(4 * ((lane & 31) + 32 * half) + (tn & 3)) * (unsigned)a.xs;
    unsigned line = 0;
    Half x0, x1, w0, w1;
    // One k-tile from buffer `buf`; x0 and the first w half (wa) are in registers, the pieces of the next tile in xg, wg or on
    // their way.  k2: where the tile after the next begins (past the end: zeros are fetched, and never read).  The other
    // buffer was last read before the barrier of the tile before, this one before the barrier here: its first pieces follow
    // at once.  The pieces are spread over the whole tile, for a CU's address path takes 16 cycles for each (all in one
    // quadrant: 5 % slower).
    auto tile = [&](int buf, int k2, Half &wa, Half &wb, auto ha, auto hb) {
        constexpr int WB = decltype(hb)::value;
        const unsigned ko = k_offset(k2), ko3 = k_offset(k2 + KT);
        if constexpr (TYPE == MPC_TYPE_E4M3) {
            asm volatile("" ::"v"(line));                     // (the line asked for a tile ago; older than pieces waited for below)
            line = __builtin_amdgcn_raw_buffer_load_b32(lr, lo + k_offset(k2 + AHEAD * KT), 0, 0);
        }
        multiply(wa, x0, ha, Lo{}, [&](int i) {
            if (i < 4) read_w(wb, 2 * i, buf, WB), read_w(wb, 2 * i + 1, buf, WB);
            if (i % 2 == 0) move(4 + i / 2, buf ^ 1, ko);
        });
        multiply(wb, x0, hb, Lo{}, [&](int i) {
            if (i < 4) read_x(x1, 2 * i, buf, 1), read_x(x1, 2 * i + 1, buf, 1);
            if (i % 2 == 0) move(8 + i / 2, buf ^ 1, ko);
        });
        multiply(wb, x1, hb, Hi{}, [&](int i) {
            if (i % 2 == 0) move(12 + i / 2, buf ^ 1, ko);
        });
        lds_barrier();
        multiply(wa, x1, ha, Hi{}, [&](int i) {
            if (i < 4) {
                read_x(x0, 2 * i, buf ^ 1, 0), read_x(x0, 2 * i + 1, buf ^ 1, 0);
                read_w(wb, 2 * i, buf ^ 1, WB), read_w(wb, 2 * i + 1, buf ^ 1, WB);
            }
            if (i % 2 == 0) move(i / 2, buf, ko3);
        });
    };
    const int past = last + p * 16 - (K - 16), back = past > 0 ? past : 0;
    const unsigned k0 = last - back, k1 = k_offset(KT);
#pragma unroll
    for (int i = 0; i < 8; ++i) fetch_x(i, k0), fetch_w(i, k0);
    if (K % KT != 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) xg[i] = row_end(xg[i], back < 16 ? back : 16), wg[i] = row_end(wg[i], back < 16 ? back : 16);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) stash_x(i, 0), stash_w(i, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) fetch_x(i, k1);
#pragma unroll
    for (int i = 0; i < 8; ++i) fetch_w(i, k1);
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i) read_x(x0, i, 0, 0), read_w(w0, i, 0, 0);
    const unsigned k2 = k_offset(2 * KT);
#pragma unroll
    for (int i = 0; i < 4; ++i) move(i, 1, k2);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 7" ::: "memory");                     // (the zeros just written to the accumulators: two states before their first use)
    __builtin_amdgcn_sched_barrier(0);
    // Two tiles a turn, an odd last one beside one of zeros: its operands past K are all zero, so it adds nothing.
    int k = 0;
    do {
        tile(0, k + 2 * KT, w0, w1, Lo{}, Hi{});
        tile(1, k + 3 * KT, w1, w0, Hi{}, Lo{});
        k += 2 * KT;
    } while (k < all);
    // The compiler does not see that the last instructions above write accumulators: their results are complete behind this.
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);

    epilogue<8, V>(a, m0 + wm + j, n0 + wn + g * 8, [&](int m, float (&v)[V]) { take_tile<8, 8>(acc, m, v); });
}

template <int TYPE>
int launch_big(mpc_ctx *ctx, const LinearArgs &a, bool prepare = false) {
    constexpr size_t lds = 2 * 2 * BIG * KT;
    auto kern = linear_big_kernel<TYPE>;
    if (prepare) return allow_lds(ctx, (const void *)kern, lds);
    in_parts(a, BIG, BIG, 256, [&](const LinearArgs &part) {
        kern<<<dim3((unsigned)(part.tiles_m * part.tiles_n)), dim3(256), lds, ctx->stream>>>(part);
    });
    MPC_CHECK_LAUNCH(ctx, "linear_big");
    return MPC_OK;
}

// ---- few rows: the weights' bytes are all that counts -----------------------------------------------------------------------------
// A workgroup takes 16 rows of w, its waves every WAVES-th k-tile of them, straight from memory into the registers of the
// matrix instructions: no operand is used twice, so nothing goes through LDS but the waves' sums, which meet there in the
// order of the waves.  UNITS k-tiles of a wave are in flight at once (64 KB and more per workgroup).  More rows than
// MF tiles take more workgroups (only for rows too far apart for the other kernels: see plan_for).  ODD: rows that begin between
// words; a word that holds a byte of the row is all that is read besides it.
template <int TYPE, int MF, int WAVES, bool ODD>
__global__ __launch_bounds__(64 * WAVES) void linear_rows_kernel(LinearArgs a) {
    constexpr int UNITS = ODD && MF == 2 && WAVES == 16 ? 2 : 4, NEXT = ODD ? UNITS : 1;      // (four would not fit the registers there)
    __shared__ f32x4 part[WAVES * MF * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)(blockIdx.x % a.tiles_n) * 16, m0 = (int64_t)(blockIdx.x / a.tiles_n) * (16 * MF);
    const char *w = a.w + (n0 + j < a.N ? n0 + j : a.N - 1) * a.ws + g * 16, *x[MF];
#pragma unroll
    for (int m = 0; m < MF; ++m) x[m] = a.x + (m0 + m * 16 + j < a.M ? m0 + m * 16 + j : a.M - 1) * a.xs + g * 16;
    const unsigned wodd = (unsigned)((uintptr_t)w & 3);
    unsigned xodd[MF];
#pragma unroll
    for (int m = 0; m < MF; ++m) xodd[m] = (unsigned)((uintptr_t)x[m] & 3);
    f32x4 acc[MF];
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int units = (int)((a.K + KT - 1) / KT);
    for (int first = wave; first < units; first += WAVES * UNITS) {
        u32x4 wv[UNITS][2], xv[UNITS][MF][2];
        unsigned wnext[NEXT][2], xnext[NEXT][MF][2];
        // (the word behind the 16 bytes if it holds one of those wanted, else the last of the 16)
        auto piece = [](const char *from, unsigned odd, u32x4 &v, unsigned &next) {
            v = *(const u32x4_word *)(from - odd);
            next = *(const unsigned *)(from - odd + (odd ? 16 : 12));
        };
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int u = first + i * WAVES;
            const int64_t k = (int64_t)u * KT;
            if (k + KT <= a.K) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if constexpr (ODD) {
                        piece(w + k + c * 64, wodd, wv[i][c], wnext[i][c]);
#pragma unroll
                        for (int m = 0; m < MF; ++m) piece(x[m] + k + c * 64, xodd[m], xv[i][m][c], xnext[i][m][c]);
                    } else {
                        wv[i][c] = *(const u32x4_any *)(w + k + c * 64);
#pragma unroll
                        for (int m = 0; m < MF; ++m) xv[i][m][c] = *(const u32x4_any *)(x[m] + k + c * 64);
                    }
                }
            } else if (k >= a.K) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    wv[i][c] = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int m = 0; m < MF; ++m) xv[i][m][c] = u32x4{0, 0, 0, 0};
                }
            } else if (a.K >= 16) {                           // the row ends in this one
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int64_t at = k + c * 64, over = at + g * 16 - (a.K - 16), back = over > 0 ? over : 0;
                    const int sh = (int)(back < 16 ? back : 16);
                    auto last = [&](const char *from) {
                        if constexpr (!ODD) return row_end(*(const u32x4_any *)from, sh);
                        u32x4 v;
                        unsigned next;
                        const unsigned odd = (unsigned)((uintptr_t)from & 3);
                        piece(from, odd, v, next);
                        return row_end(from_words(v, next, odd), sh);
                    };
                    wv[i][c] = last(w + at - back);
#pragma unroll
                    for (int m = 0; m < MF; ++m) xv[i][m][c] = last(x[m] + at - back);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int64_t left = a.K - k - c * 64 - g * 16;
                    wv[i][c] = load_piece<Operand<TYPE>::BYTES>(w + k + c * 64, left);
#pragma unroll
                    for (int m = 0; m < MF; ++m) xv[i][m][c] = load_piece<Operand<TYPE>::BYTES>(x[m] + k + c * 64, left);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            if (ODD && (int64_t)(first + i * WAVES + 1) * KT <= a.K) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    wv[i][c] = from_words(wv[i][c], wnext[i % NEXT][c], wodd);
#pragma unroll
                    for (int m = 0; m < MF; ++m) xv[i][m][c] = from_words(xv[i][m][c], xnext[i % NEXT][m][c], xodd[m]);
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int m = 0; m < MF; ++m) {
                    if constexpr (TYPE == MPC_TYPE_E4M3) acc[m] = Operand<TYPE>::mma_exact(wv[i][c], xv[i][m][c], acc[m]);
                    else acc[m] = Operand<TYPE>::mma(wv[i][c], xv[i][m][c], acc[m]);
                }
            }
        }
    }
    // [wave][16 MF rows][16 columns]
#pragma unroll
    for (int m = 0; m < MF; ++m) part[(wave * MF + m) * 64 + j * 4 + g] = acc[m];
    __syncthreads();
    const float *sums = (const float *)part;
    for (int t = tid; t < MF * 256; t += 64 * WAVES) {
        const int64_t m = m0 + (t >> 4), n = n0 + (t & 15);
        if (m >= a.M || n >= a.N) continue;
        float v[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < WAVES; ++i) v[0] += sums[i * MF * 256 + t];
        if (a.sx) v[0] *= a.sx[m] * a.sw[n];
        if (a.bias) v[0] += a.bias[n];
        finish_values(a, m, n, v);
    }
}

// rows that begin between words
bool between_words(const LinearArgs &a) { return ((uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.xs | (uintptr_t)a.ws) % 4 != 0; }

template <int TYPE, int MF, bool ODD>
int launch_rows(mpc_ctx *ctx, const LinearArgs &a) {
    in_parts(a, 16 * MF, 16, 1024, [&](const LinearArgs &part) {
        const int blocks = part.tiles_m * part.tiles_n;
        // up to a workgroup per CU: 16 waves, so that the CU's whole share of w is on its way; more: 8 waves, two workgroups a CU
        if (blocks <= 256) linear_rows_kernel<TYPE, MF, 16, ODD><<<dim3((unsigned)blocks), dim3(1024), 0, ctx->stream>>>(part);
        else linear_rows_kernel<TYPE, MF, 8, ODD><<<dim3((unsigned)blocks), dim3(512), 0, ctx->stream>>>(part);
    });
    MPC_CHECK_LAUNCH(ctx, "linear_rows");
    return MPC_OK;
}

// ---- which kernel ---------------------------------------------------------------------------------------------------------------
enum { PLAN_ROWS, PLAN_SMALL, PLAN_MIDDLE, PLAN_BIG };
struct Plan {
    int kind, splits;
};

Plan plan_for(bool eight, int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws) {     // the last three in bytes
    // (rows so far apart that a tile's do not fit a buffer: the kernel that addresses each by itself)
    if (M <= 32 || BIG * xs + K > TILE_BYTES || BIG * ws + K > TILE_BYTES) return {PLAN_ROWS, 1};
    const int64_t big = mpc_cdiv(M, BIG) * mpc_cdiv(N, BIG), middle = mpc_cdiv(M, 128) * mpc_cdiv(N, 128);
    // The large tile needs most CUs busy and some k-tiles to pay for its prologue and epilogue (128 x 128 tiles against it, bf16
    // with bias and gelu: 3584 x 4096 x 4096 137 us : 105; 2048 x 4096 x 4096 77 : 99; without: 27696 x 880 -> 5504 367 : 310; 8192 x
    // 768 -> 8192 119 : 113; 8192 x 512 -> 8192 98 : 106; e4m3: 5000 x 1800 -> 3000 46 : 44; 10871 x 1500 -> 7431 261 : 307).
    // A turn of 256 of the large tiles takes as long as 0.4 + 0.62 turns of 512 middle ones, of whose last turn only a part is paid
    // (4096 x 2048 -> 4352, 272 large tiles, 103 : 91; 36864 x 2048 -> 320 101 : 75; 12000 x 3000 -> 1100 83 : 118).
    if (big >= 192 && K >= (eight ? 2048 : 1536) && (mpc_cdiv(big, 256) * 512 - 205) * 8 <= 5 * middle) return {PLAN_BIG, 1};
    // 64 x 64 tiles as long as two workgroups a CU take them all (bf16, 64 x 64 : 128 x 128: 512 x 2048 -> 4096, 512 small tiles,
    // 18.6 : 22.2; 860 x 2993 -> 2902, 644, 51 : 37; 30000 x 1024 -> 64, 469, 14.0 : 14.4; 60000 x 256 -> 64, 938, 12.0 : 10.5).
    const int64_t small = mpc_cdiv(M, 64) * mpc_cdiv(N, 64), k_tiles = mpc_cdiv(K, KT);
    if (small > 512) return {PLAN_MIDDLE, 1};
    // Split K while that gives CUs without work some, and 16 k-tiles a part: joining the parts takes 5 us and more.  (bf16, in one :
    // as here : up to two workgroups a CU: 1000 x 2048 -> 1000, 256 tiles, 13.6 : 13.6 : 18.7; 500 x 8192 -> 500 40 : 19 : 22; 64 x
    // 8192 -> 8192 40 : 29 : 29; 64 x 4096 -> 4096 22 : 13 : 13, with 32 k-tiles a part 16, with 8 15.)
    int splits = 1;
    while (splits < 16 && small * splits * 2 <= 256 && k_tiles / (splits * 2) >= 16) splits *= 2;
    return {PLAN_SMALL, splits};
}

template <int TYPE>
int launch_small(mpc_ctx *ctx, const LinearArgs &a, int splits, bool prepare = false) {
    return launch_tiles<TYPE, 64, 64, 32, 32, 4, 3>(ctx, a, splits, prepare);
}
// 8 waves of 64 x 32, two workgroups a CU: the second's products run beside the first's epilogue.  (36864 x 256 -> 1024 with
// gelu, before its gelu and its last two tiles' fetches were cut: 50 us; 4 waves of 64 x 64, with one or two tiles ahead: 53; 128 x 64
// tiles: 52; 256 x 128: 63.)
template <int TYPE>
int launch_middle(mpc_ctx *ctx, const LinearArgs &a, bool prepare = false) {
    return launch_tiles<TYPE, 128, 128, 64, 32, 1, 4>(ctx, a, 1, prepare);
}

template <int TYPE>
int launch(mpc_ctx *ctx, const LinearArgs &a) {
    const Plan plan = plan_for(TYPE == MPC_TYPE_E4M3, a.M, a.N, a.K, a.xs, a.ws);
    if (plan.kind == PLAN_ROWS) {
        if (between_words(a)) return a.M <= 16 ? launch_rows<TYPE, 1, true>(ctx, a) : launch_rows<TYPE, 2, true>(ctx, a);
        return a.M <= 16 ? launch_rows<TYPE, 1, false>(ctx, a) : launch_rows<TYPE, 2, false>(ctx, a);
    }
    if (plan.kind == PLAN_BIG) return launch_big<TYPE>(ctx, a);
    if (plan.kind == PLAN_SMALL) return launch_small<TYPE>(ctx, a, plan.splits);
    return launch_middle<TYPE>(ctx, a);
}

template <int TYPE>
int prepare(mpc_ctx *ctx) {
    const LinearArgs none{};
    int rc = launch_small<TYPE>(ctx, none, 1, true);
    if (rc == MPC_OK) rc = launch_middle<TYPE>(ctx, none, true);
    return rc == MPC_OK ? launch_big<TYPE>(ctx, none, true) : rc;
}

bool linear_desc_ok(const mpc_linear_desc &d) {
    const bool in16 = d.in_type == MPC_TYPE_F16 || d.in_type == MPC_TYPE_BF16;
    const int64_t far = 1ll << 40;             // elements: 256 rows of them are far from 63 bits of bytes
    return (in16 || d.in_type == MPC_TYPE_E4M3) &&
           (d.out_type == MPC_TYPE_F32 || d.out_type == MPC_TYPE_F16 || d.out_type == MPC_TYPE_BF16) &&
           (d.act == MPC_ACT_NONE || d.act == MPC_ACT_RELU || d.act == MPC_ACT_GELU || d.act == MPC_ACT_SILU) && d.M >= 0 &&
           d.M < (1ll << 31) && d.N > 0 && d.N < (1ll << 31) && d.K > 0 && d.K < (1ll << 31) && d.x_stride >= 0 && d.x_stride < far &&
           d.w_stride >= 0 && d.w_stride < far && d.residual_stride >= 0 && d.residual_stride < far && d.out_stride >= d.N &&
           d.out_stride < far;
}

}  // namespace

int mpc_linear_init(mpc_ctx *ctx) {
    int rc = prepare<MPC_TYPE_F16>(ctx);
    if (rc == MPC_OK) rc = prepare<MPC_TYPE_BF16>(ctx);
    return rc == MPC_OK ? prepare<MPC_TYPE_E4M3>(ctx) : rc;
}

extern "C" size_t mpc_linear_workspace_bytes(const mpc_linear_desc *desc) {
    if (!desc || !linear_desc_ok(*desc) || desc->M == 0) return 0;
    const int ib = mpc_type_bytes(desc->in_type);
    const Plan plan = plan_for(desc->in_type == MPC_TYPE_E4M3, desc->M, desc->N, desc->K * ib, desc->x_stride * ib, desc->w_stride * ib);
    return plan.splits > 1 ? (size_t)plan.splits * desc->M * desc->N * sizeof(float) : 0;
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
    const size_t need = mpc_linear_workspace_bytes(desc);
    MPC_REQUIRE(ctx, workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 16 == 0)),
                "linear: workspace of %zu bytes, %zu needed, 16-byte aligned", workspace_bytes, need);
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
    a.partial = (float *)workspace;
    if (d.in_type == MPC_TYPE_F16) return launch<MPC_TYPE_F16>(ctx, a);
    if (d.in_type == MPC_TYPE_BF16) return launch<MPC_TYPE_BF16>(ctx, a);
    return launch<MPC_TYPE_E4M3>(ctx, a);
}
