// The balance loss of a competition and its gradient.  With z = scale * scores, p = softmax(z) over the experts of a row
// that counts and f the share of the top_k choices that fell on an expert:
//   loss = E sum_e f_e mean_t p_te,     d loss / d score_tj = scale E / R p_tj (f_j - sum_e f_e p_te).
//
// A row belongs to a group of `group` lanes (a power of two), EPL consecutive experts a lane, so that the softmax's and the
// choice's reductions are a few DPP steps and a wave takes 64 / group rows at once (64 experts: 8 lanes, 8 rows).  A
// wave keeps the sums of p of its rows in registers and counts choices in LDS; the blocks' sums meet in a second kernel,
// in a fixed order and in double.  Scores whose experts are not consecutive (the competition writes its totals prior by
// prior) go through an LDS tile, read and, for the gradient, written along the rows.
//
// 1M x 64 bf16, top 2, with a mask: forward 47 us and its join 7, bound by its vector instructions (an exponential and two rounds
// of the choice per score); gradient 49 us, 5.2 TB/s.  1536 x 64 fp32, expert by expert: 5.5 us, join 3.3, gradient 5.3, latency.
#include "row_ops.h"

#include <type_traits>

namespace {

constexpr int PB_MAX_EXPERTS = 1024;
constexpr int PB_MAX_THREADS = 512;
constexpr int PB_WIDE_THREADS = 1024;   // forward kernel of consecutive experts (1M x 64 bf16, top 2: 56 us against 61 with 512)
constexpr int PB_MAX_BLOCKS = 512;
constexpr int PB_JOIN = 32;             // fewest experts of a workgroup of the join kernel
constexpr int PB_HEAD = 2 * (1 + PB_MAX_EXPERTS / PB_JOIN);      // words in front of the blocks' sums: a ticket, a double per workgroup of the join

struct Row {
    const void *scores;
    int64_t rows, row_stride, expert_stride;
    int experts;
    float scale;
    int top_k;
    const uint8_t *mask;
    int group, group_log2;
    int tile_rows;                    // staged kernels: rows of an LDS tile (a power of two)
    int tile_log2;
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
    return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, false);
}

// op over the lanes of a group; every lane gets the result.  Lane i of a quad with i ^ 1, with i ^ 2, then the mirror
// images of eight and of sixteen lanes.  LOG2: of the group's size, or -1 if that is known only at run time (`group`).
template <int LOG2, typename T, typename Op>
__device__ __forceinline__ T group_reduce(T v, int group, Op op) {
    if constexpr (LOG2 >= 0) group = 1 << LOG2;
    if (group > 1) v = op(v, dpp<0xB1>(v));
    if (group > 2) v = op(v, dpp<0x4E>(v));
    if (group > 4) v = op(v, dpp<0x141>(v));
    if (group > 8) v = op(v, dpp<0x140>(v));
    // rows of 16 lanes 0 0 2 2 and 1 1 3 3, then halves 0 0 and 1 1 (a swap reads what the instruction two before it wrote; the
    // compiler's builtins take the two results for one)
    if (group > 16) {
        T w = v;
        asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(v), "+v"(w));
        v = op(v, w);
    }
    if (group > 32) {
        T w = v;
        asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(v), "+v"(w));
        v = op(v, w);
    }
    return v;
}
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Or {
    __device__ __forceinline__ int operator()(int a, int b) const { return a | b; }
};

// What a lane brings of a row: its values as they lie in memory (the last expert's successors as the worst one), and whether
// the row's mask lets it count.
template <typename T, int EPL>
struct Raw {
    static constexpr int W = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(W)));
    typedef vec vec_any __attribute__((aligned(sizeof(T))));
    vec t[EPL / W];
    bool in, keep;

    __device__ __forceinline__ void fetch(const Row &a, int64_t row, int e0) {
        in = row < a.rows;
        const int64_t at = in ? row : 0;                      // (a group without a row reads row 0 and counts nothing)
        keep = in && (!a.mask || a.mask[at]);
        const T *s = (const T *)a.scores + at * a.row_stride;
#pragma unroll
        for (int i = 0; i < EPL / W; ++i) {
            const int e = e0 + i * W;
            if (e + W <= a.experts) {
                t[i] = *(const vec_any *)(s + e);
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) t[i][j] = e + j < a.experts ? s[e + j] : (T)(a.scale < 0.0f ? INFINITY : -INFINITY);
            }
        }
    }
    // in the order of the choice (costs negated); 0 in rows that do not count
    __device__ __forceinline__ void values(const Row &a, float (&v)[EPL]) const {
        typedef unsigned words __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int i = 0; i < EPL / W; ++i) {
            words w = __builtin_bit_cast(words, t[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = keep ? w[j] : 0u;                  // (16-bit types: two values at once)
            const vec x = __builtin_bit_cast(vec, w);
#pragma unroll
            for (int j = 0; j < W; ++j) v[i * W + j] = (float)x[j];
        }
        if (a.scale < 0.0f) {
#pragma unroll
            for (int j = 0; j < EPL; ++j) v[j] = -v[j];
        }
    }
};
template <int EPL>
__device__ __forceinline__ void staged_values(const Row &a, const float *tile_row, int e0, bool keep, float (&v)[EPL]) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        const float x = e0 + j < a.experts ? tile_row[e0 + j] : -INFINITY;
        v[j] = keep ? x : 0.0f;
    }
}

// v -> p = e * inv.  Returns whether the row counts (inv = 0 if not).  Changes v only in rows without anything above -inf.
template <int LOG2, int EPL>
__device__ __forceinline__ bool softmax(const Row &a, bool keep, float (&v)[EPL], float (&e)[EPL], float &top, float &inv) {
    const float slope = fabsf(a.scale) * 1.44269504f;
    top = v[0];
#pragma unroll
    for (int j = 1; j < EPL; ++j) top = fmaxf(top, v[j]);
    top = group_reduce<LOG2>(top, a.group, Max());
    if (__any(keep && top == -INFINITY)) {                    // rows of -inf (and NaN): rare
        int nan = 0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) nan |= v[j] != v[j];
        nan = group_reduce<LOG2>(nan, a.group, Or());
        if (top == -INFINITY && !nan) {
            keep = false;
            top = 0.0f;
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        e[j] = __builtin_amdgcn_exp2f((v[j] - top) * slope);
        sum += e[j];
    }
    sum = group_reduce<LOG2>(sum, a.group, Add());
    inv = keep ? __builtin_amdgcn_rcpf(sum) : 0.0f;
    return keep;
}

// Copies rows [first, first + tile_rows) to LDS in the order of the choice, along the rows; rows behind the last become 0.
// Consecutive rows (the competition's layout) come as 16 bytes of one expert's rows; with the tile's pitch of experts + 1
// words a wave's writes fall into different banks.  Otherwise eight loads of a thread are in flight at once.
template <typename T>
__device__ __forceinline__ void stage(const Row &a, int64_t first, float *tile) {
    constexpr int U = 8, W = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(W)));
    typedef vec vec_any __attribute__((aligned(sizeof(T))));
    const int pitch = a.experts + 1, all = a.experts << a.tile_log2, step = blockDim.x;
    const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
    const T *s = (const T *)a.scores + first * a.row_stride;
    const int64_t left = a.rows - first;
    if (a.row_stride == 1) {
        constexpr int V = 2;                                  // (tile_rows is a multiple of W)
        for (int base = threadIdx.x * W; base < all; base += V * step * W) {
            vec x[V];
#pragma unroll
            for (int u = 0; u < V; ++u) {
                const int i = base + u * step * W, r = i & (a.tile_rows - 1), e = i >> a.tile_log2;
                if (i < all && r + W <= left) {
                    x[u] = *(const vec_any *)(s + r + e * a.expert_stride);
                } else {
#pragma unroll
                    for (int j = 0; j < W; ++j) x[u][j] = i < all && r + j < left ? s[r + j + e * a.expert_stride] : (T)0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < V; ++u) {
                const int i = base + u * step * W, r = i & (a.tile_rows - 1), e = i >> a.tile_log2;
                if (i < all) {
#pragma unroll
                    for (int j = 0; j < W; ++j) tile[(r + j) * pitch + e] = (float)x[u][j] * sign;
                }
            }
        }
        return;
    }
    for (int base = threadIdx.x; base < all; base += U * step) {
        T x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + u * step, r = i & (a.tile_rows - 1), e = i >> a.tile_log2;
            x[u] = (T)0.0f;
            if (i < all && r < left) x[u] = s[r * a.row_stride + e * a.expert_stride];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + u * step;
            if (i < all) tile[(i & (a.tile_rows - 1)) * pitch + (i >> a.tile_log2)] = (float)x[u] * sign;
        }
    }
}

// words of a block in the workspace, behind the head: sum of p (float) [experts], choices (int) [experts], rows (int)
template <typename T, int EPL, int LOG2, bool STAGED>
__global__ __launch_bounds__(STAGED ? PB_MAX_THREADS : PB_WIDE_THREADS) void prior_balance_kernel(Row a, float *__restrict__ ws) {
    if constexpr (LOG2 >= 0) a.group = 1 << LOG2, a.group_log2 = LOG2;
    extern __shared__ float lds[];                            // [experts] choices | sums of the waves, or the tile
    __shared__ int rsum[PB_WIDE_THREADS / 64];
    int *hist = (int *)lds;
    float *tile = lds + a.experts;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int e0 = (lane & (a.group - 1)) * EPL, per_wave = 64 >> a.group_log2, per_block = per_wave * waves;
    if (blockIdx.x == 0 && tid == 0) *(int *)ws = 0;          // (the join's ticket)
    for (int e = tid; e < a.experts; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    float acc[EPL];
    int n = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) acc[j] = 0.0f;

    const uint64_t before = (1ull << lane) - (1ull << (lane & ~(a.group - 1)));              // the lanes in front of this one in its group
    auto one = [&](bool keep, float (&v)[EPL]) {
        float e[EPL], top, inv;
        keep = softmax<LOG2, EPL>(a, keep, v, e, top, inv);
#pragma unroll
        for (int j = 0; j < EPL; ++j) acc[j] = fmaf(e[j], inv, acc[j]);          // (rows that do not count: inv = 0, e finite)
        n += (int)__popcll(__ballot(keep && e0 == 0));
        for (int k = 0; k < a.top_k; ++k) {
            float best = top;
            if (k > 0) {
                best = v[0];
#pragma unroll
                for (int j = 1; j < EPL; ++j) best = fmaxf(best, v[j]);
                best = group_reduce<LOG2>(best, a.group, Max());
            }
            int at = EPL;
#pragma unroll
            for (int j = EPL - 1; j >= 0; --j) at = v[j] == best ? j : at;
            // the group's first lane that holds it chooses
            at = __ballot(at < EPL) & before ? EPL : at;
            if (keep && best > -INFINITY && at < EPL) atomicAdd(&hist[e0 + at], 1);
            if (k + 1 < a.top_k) {
#pragma unroll
                for (int j = 0; j < EPL; ++j) v[j] = j == at ? -INFINITY : v[j];
            }
        }
    };
    if constexpr (STAGED) {
        for (int64_t first = (int64_t)blockIdx.x * a.tile_rows; first < a.rows; first += (int64_t)gridDim.x * a.tile_rows) {
            __syncthreads();                                  // the previous tile has been read
            stage<T>(a, first, tile);
            __syncthreads();
            for (int r = wave * per_wave; r < a.tile_rows; r += per_block) {
                const int mine = r + (lane >> a.group_log2);  // (tile_rows may be less than a wave's rows)
                const bool in = mine < a.tile_rows && first + mine < a.rows;
                float v[EPL];
                const bool keep = in && (!a.mask || a.mask[first + mine]);
                staged_values<EPL>(a, tile + (in ? mine : 0) * (a.experts + 1), e0, keep, v);
                one(keep, v);
            }
        }
        __syncthreads();
    } else {
        const int64_t step = (int64_t)gridDim.x * per_block;
        int64_t first = (int64_t)blockIdx.x * per_block + wave * per_wave;
        const int mine = lane >> a.group_log2;
        Raw<T, EPL> now, next;
        if (a.rows > 0) now.fetch(a, first + mine, e0);       // (with no row at all there is none to read in a missing one's place)
        for (; first < a.rows; first += step) {               // the next rows are on their way while these are worked on
            next.fetch(a, first + step + mine, e0);
            float v[EPL];
            now.values(a, v);
            one(now.keep, v);
            now = next;
        }
    }

    // the groups of a wave, then the waves of the block
    const int width = a.group * EPL;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        for (int off = a.group; off < 64; off <<= 1) acc[j] += __shfl_xor(acc[j], off, 64);
        if (lane < a.group) tile[wave * width + e0 + j] = acc[j];
    }
    if (lane == 0) rsum[wave] = n;
    __syncthreads();
    float *out = ws + PB_HEAD + (int64_t)blockIdx.x * (2 * a.experts + 1);
    for (int e = tid; e < a.experts; e += blockDim.x) {
        float s = 0.0f;
        for (int w = 0; w < waves; ++w) s += tile[w * width + e];
        out[e] = s;
        ((int *)out)[a.experts + e] = hist[e];
    }
    if (tid == 0) {
        int c = 0;
        for (int w = 0; w < waves; ++w) c += rsum[w];
        ((int *)out)[2 * a.experts] = c;
    }
}

// A workgroup adds up the blocks' sums of J experts, 1024 / J threads an expert.  The workgroup that finishes last (the ticket
// says so) adds up their parts of the loss, in their order whichever it is.  Up to 64 experts take one workgroup, without a
// ticket, more take 32 each (forward and join, one workgroup for all experts : this: 1000 x 700 47 us : 13, 10000 x 256 25 : 13;
// one workgroup of 64 against two of 32: 1000 x 64 7.5 : 8.7; 32 against 64 at 10000 x 256: 12.6 : 14.2).
template <int J>
__global__ __launch_bounds__(1024) void prior_balance_join_kernel(float *__restrict__ ws, int blocks, int experts, int top_k,
                                                                          float *__restrict__ loss, int32_t *__restrict__ counts,
                                                                          int32_t *__restrict__ n_rows) {
    constexpr int WAVES = 16;
    __shared__ double psum[WAVES][J];
    __shared__ int csum[WAVES][J], nsum[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, words = 2 * experts + 1;
    const float *sums = ws + PB_HEAD;
    int n = 0;
    for (int b = tid; b < blocks; b += 1024) n += ((const int *)sums)[(int64_t)b * words + 2 * experts];
    const int at = tid % J, e = blockIdx.x * J + at;
    double p = 0.0;
    int c = 0;
    constexpr int U = 8, STEP = 1024 / J;               // loads of eight blocks at once
    for (int b0 = tid / J; b0 < blocks; b0 += U * STEP) {
        float x[U];
        int y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t from = (int64_t)(b0 + u * STEP < blocks ? b0 + u * STEP : b0) * words + (e < experts ? e : 0);
            x[u] = sums[from], y[u] = ((const int *)sums)[from + experts];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b0 + u * STEP < blocks) p += (double)x[u], c += y[u];
    }
    for (int off = 32; off > 0; off >>= 1) {
        n += __shfl_xor(n, off, 64);
        if (off >= J) p += __shfl_xor(p, off, 64), c += __shfl_xor(c, off, 64);
    }
    if (lane < J) psum[wave][lane] = p, csum[wave][lane] = c;
    if (lane == 0) nsum[wave] = n;
    __syncthreads();
    if (wave > 0) return;
    p = 0.0, c = 0, n = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) p += psum[w][at], c += csum[w][at], n += nsum[w];
    if (lane < J && e < experts) counts[e] = c;
    double term = lane < J && e < experts && n > 0 ? (double)c / ((double)top_k * n) * (p / n) : 0.0;
    auto total = [&] {
        for (int off = 32; off > 0; off >>= 1) term += __shfl_xor(term, off, 64);
    };
    total();
    int last = 1;
    if (gridDim.x > 1) {
        uint64_t *terms = (uint64_t *)ws + 1;
        if (lane == 0) {
            __hip_atomic_store(terms + blockIdx.x, __builtin_bit_cast(uint64_t, term), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last = __hip_atomic_fetch_add((int *)ws, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
        }
        last = __shfl(last, 0, 64);
        if (last) {
            __atomic_thread_fence(__ATOMIC_ACQUIRE);
            term = lane < (int)gridDim.x ? __builtin_bit_cast(double, __hip_atomic_load(terms + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) : 0.0;
            total();
        }
    }
    if (last && lane == 0) *loss = (float)(experts * term), *n_rows = n;
}
static_assert(PB_MAX_EXPERTS / PB_JOIN <= 64, "a wave adds up the workgroups' parts");

template <typename T, int EPL, int LOG2, bool STAGED>
__global__ __launch_bounds__(PB_MAX_THREADS) void prior_balance_grad_kernel(Row a, const int32_t *__restrict__ counts,
                                                                            const int32_t *__restrict__ n_rows,
                                                                            const float *__restrict__ grad_out, T *__restrict__ grad,
                                                                            int64_t grs, int64_t ges) {
    if constexpr (LOG2 >= 0) a.group = 1 << LOG2, a.group_log2 = LOG2;
    extern __shared__ float tile[];
    constexpr int W = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(W)));
    typedef vec vec_any __attribute__((aligned(sizeof(T))));
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int e0 = (lane & (a.group - 1)) * EPL, per_wave = 64 >> a.group_log2, per_block = per_wave * waves;
    const int n = *n_rows;
    // f_j - 1 / E: the difference f_j - sum_e f_e p_te is the same, and loses less where use is nearly even
    float f[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j)
        f[j] = e0 + j < a.experts && n > 0 ? (float)((double)counts[e0 + j] / ((double)a.top_k * n) - 1.0 / a.experts) : 0.0f;
    const float g = n > 0 ? (float)((double)(grad_out ? *grad_out : 1.0f) * a.scale * a.experts / n) : 0.0f;

    auto one = [&](int64_t row, bool in, bool keep, float (&v)[EPL], float *tile_row) {
        float e[EPL], top, inv;
        keep = softmax<LOG2, EPL>(a, keep, v, e, top, inv);
        float d = 0.0f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            e[j] *= inv;                                      // (rows that do not count: inv = 0, e finite)
            d = fmaf(e[j], f[j], d);
        }
        d = group_reduce<LOG2>(d, a.group, Add());
        const float gk = keep ? g : 0.0f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) e[j] *= gk * (f[j] - d);
        if (!in) return;
        if constexpr (STAGED) {
#pragma unroll
            for (int j = 0; j < EPL; ++j)
                if (e0 + j < a.experts) tile_row[e0 + j] = e[j];
        } else {
            T *o = grad + row * grs;
            if (ges == 1) {
#pragma unroll
                for (int i = 0; i < EPL; i += W) {
                    if (e0 + i + W <= a.experts) {
                        vec t;
#pragma unroll
                        for (int j = 0; j < W; ++j) t[j] = (T)e[i + j];
                        *(vec_any *)(o + e0 + i) = t;
                    } else {
#pragma unroll
                        for (int j = 0; j < W; ++j)
                            if (e0 + i + j < a.experts) o[e0 + i + j] = (T)e[i + j];
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < EPL; ++j)
                    if (e0 + j < a.experts) o[(e0 + j) * ges] = (T)e[j];
            }
        }
    };
    if constexpr (STAGED) {
        const int pitch = a.experts + 1;
        for (int64_t first = (int64_t)blockIdx.x * a.tile_rows; first < a.rows; first += (int64_t)gridDim.x * a.tile_rows) {
            __syncthreads();
            stage<T>(a, first, tile);
            __syncthreads();
            for (int r = wave * per_wave; r < a.tile_rows; r += per_block) {
                const int mine = r + (lane >> a.group_log2);
                const bool in = mine < a.tile_rows && first + mine < a.rows;
                float *tile_row = tile + (in ? mine : 0) * pitch;
                float v[EPL];
                const bool keep = in && (!a.mask || a.mask[first + mine]);
                staged_values<EPL>(a, tile_row, e0, keep, v);
                one(first + mine, in, keep, v, tile_row);
            }
            __syncthreads();
            if (grs == 1) {
                for (int i = tid * W; i < a.experts << a.tile_log2; i += blockDim.x * W) {
                    const int r = i & (a.tile_rows - 1), e = i >> a.tile_log2;
                    T *o = grad + first + r + e * ges;
                    vec t;
#pragma unroll
                    for (int j = 0; j < W; ++j) t[j] = (T)tile[(r + j) * pitch + e];
                    if (first + r + W <= a.rows) {
                        *(vec_any *)o = t;
                    } else {
#pragma unroll
                        for (int j = 0; j < W; ++j)
                            if (first + r + j < a.rows) o[j] = t[j];
                    }
                }
            } else {
                for (int i = tid; i < a.experts << a.tile_log2; i += blockDim.x) {
                    const int r = i & (a.tile_rows - 1), e = i >> a.tile_log2;
                    if (first + r < a.rows) grad[(first + r) * grs + e * ges] = (T)tile[r * pitch + e];
                }
            }
        }
    } else {
        const int64_t step = (int64_t)gridDim.x * per_block;
        int64_t first = (int64_t)blockIdx.x * per_block + wave * per_wave;
        Raw<T, EPL> now, next;
        if (first < a.rows) now.fetch(a, first + (lane >> a.group_log2), e0);
        for (; first < a.rows; first += step) {
            if (first + step < a.rows) next.fetch(a, first + step + (lane >> a.group_log2), e0);
            float v[EPL];
            now.values(a, v);
            one(first + (lane >> a.group_log2), now.in, now.keep, v, nullptr);
            now = next;
        }
    }
}

struct Shape {
    int epl, threads;
    int64_t passes;                   // blocks that would take every row at once
    size_t tile_bytes;
};

// Lanes per row, rows per tile, threads per block.  Few rows: small blocks (`least` threads), so that more CUs take part; not as
// small in the forward kernel, whose blocks are joined afterwards (10000 x 256, 128 threads : 512: 16.5 us : 14.5, the gradient
// 9.0 : 11.3).
Shape shape(Row &a, bool staged, int least, int most) {
    Shape s{};
    s.epl = a.experts > 8 * 64 ? 16 : 8;
    a.group = 1, a.group_log2 = 0;
    while (a.group * s.epl < a.experts) a.group *= 2, ++a.group_log2;
    const bool few = a.rows <= 64 * 256;
    int per_block;
    if (staged) {
        int r = few ? 16 : 64;
        while (r > 8 && r * (a.experts + 1) > 12288) r /= 2;
        while (!few && r * a.group < PB_MAX_THREADS && 2 * r * (a.experts + 1) <= 12288) r *= 2;    // (few experts: rows enough for the block)
        a.tile_rows = r;
        a.tile_log2 = __builtin_ctz(r);
        const int t = r * a.group;
        s.threads = t < 128 ? 128 : t > PB_MAX_THREADS ? PB_MAX_THREADS : t;
        s.tile_bytes = (size_t)r * (a.experts + 1) * sizeof(float);
        per_block = r;
    } else {
        s.threads = few ? least : most;
        per_block = s.threads / a.group;
    }
    s.passes = a.rows > 0 ? mpc_cdiv(a.rows, per_block) : 1;
    return s;
}

// f(the group's log2 as a constant): with it the reductions are straight code (1M x 64 bf16, top 2: forward 77 -> 71 us, gradient 78 -> 51)
template <typename F>
void by_group(int log2, F f) {
    switch (log2) {
        case 0: return f(std::integral_constant<int, 0>());
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        case 4: return f(std::integral_constant<int, 4>());
        case 5: return f(std::integral_constant<int, 5>());
        default: return f(std::integral_constant<int, 6>());
    }
}

template <typename T>
int forward(mpc_ctx *ctx, Row a, float *ws, float *loss, int32_t *counts, int32_t *n_rows) {
    const bool staged = a.expert_stride != 1 && a.experts > 1;
    const Shape s = shape(a, staged, 512, PB_WIDE_THREADS);
    const int blocks = (int)(s.passes > PB_MAX_BLOCKS ? PB_MAX_BLOCKS : s.passes);
    size_t sums = (size_t)(s.threads / 64) * a.group * s.epl * sizeof(float);
    if (sums < s.tile_bytes) sums = s.tile_bytes;
    const size_t lds = a.experts * sizeof(int) + sums;
    const dim3 grid(blocks), block(s.threads);
    auto run = [&](auto kernel) { kernel<<<grid, block, lds, ctx->stream>>>(a, ws); };
    if (staged) s.epl == 8 ? run(prior_balance_kernel<T, 8, -1, true>) : run(prior_balance_kernel<T, 16, -1, true>);
    else if (s.epl == 16) run(prior_balance_kernel<T, 16, 6, false>);
    else by_group(a.group_log2, [&](auto log2) { run(prior_balance_kernel<T, 8, decltype(log2)::value, false>); });
    MPC_CHECK_LAUNCH(ctx, "prior_balance");
    const dim3 all(1024);
    if (a.experts <= 64) prior_balance_join_kernel<64><<<dim3(1), all, 0, ctx->stream>>>(ws, blocks, a.experts, a.top_k, loss, counts, n_rows);
    else prior_balance_join_kernel<PB_JOIN><<<dim3((unsigned)mpc_cdiv(a.experts, PB_JOIN)), all, 0, ctx->stream>>>(ws, blocks, a.experts, a.top_k, loss,
                                                                                                                  counts, n_rows);
    MPC_CHECK_LAUNCH(ctx, "prior_balance_join");
    return MPC_OK;
}

template <typename T>
int backward(mpc_ctx *ctx, Row a, const int32_t *counts, const int32_t *n_rows, const float *grad_out, void *grad, int64_t grs, int64_t ges) {
    const bool staged = a.expert_stride != 1 && a.experts > 1;
    const Shape s = shape(a, staged, 128, PB_MAX_THREADS);
    const dim3 grid((unsigned)(s.passes > 1024 ? 1024 : s.passes)), block(s.threads);
    T *o = (T *)grad;
    auto run = [&](auto kernel) { kernel<<<grid, block, staged ? s.tile_bytes : 0, ctx->stream>>>(a, counts, n_rows, grad_out, o, grs, ges); };
    if (staged) s.epl == 8 ? run(prior_balance_grad_kernel<T, 8, -1, true>) : run(prior_balance_grad_kernel<T, 16, -1, true>);
    else if (s.epl == 16) run(prior_balance_grad_kernel<T, 16, 6, false>);
    else by_group(a.group_log2, [&](auto log2) { run(prior_balance_grad_kernel<T, 8, decltype(log2)::value, false>); });
    MPC_CHECK_LAUNCH(ctx, "prior_balance_grad");
    return MPC_OK;
}

int check(mpc_ctx *ctx, const void *scores, int type, int64_t rows, int experts, int64_t rs, int64_t es, float scale, int top_k) {
    MPC_REQUIRE(ctx, type == MPC_TYPE_F32 || type == MPC_TYPE_F16 || type == MPC_TYPE_BF16, "prior_balance: type %d", type);
    MPC_REQUIRE(ctx, experts > 0 && experts <= PB_MAX_EXPERTS, "prior_balance: %d experts (1..%d)", experts, PB_MAX_EXPERTS);
    MPC_REQUIRE(ctx, top_k > 0 && top_k <= experts, "prior_balance: top_k = %d of %d experts", top_k, experts);
    MPC_REQUIRE(ctx, rows >= 0 && rows < (1ll << 31) / top_k, "prior_balance: %lld rows", (long long)rows);
    MPC_REQUIRE(ctx, rs >= 0 && es >= 0, "prior_balance: negative stride");
    // (2^127 and more would leave fp32 with exp2's factor)
    MPC_REQUIRE(ctx, scale != 0.0f && fabsf(scale) < 0x1p127f, "prior_balance: scale = %g", (double)scale);
    MPC_REQUIRE(ctx, rows == 0 || (scores && (uintptr_t)scores % mpc_type_bytes(type) == 0), "prior_balance: null or misaligned pointer");
    return MPC_OK;
}

}  // namespace

extern "C" size_t mpc_prior_balance_workspace_bytes(int64_t rows, int experts) {
    if (rows < 0 || experts <= 0 || experts > PB_MAX_EXPERTS) return 0;
    // as many blocks as either layout's kernel may take for these rows
    const int64_t blocks = mpc_cdiv(rows, 2) + 1;
    return (PB_HEAD + (size_t)(blocks > PB_MAX_BLOCKS ? PB_MAX_BLOCKS : blocks) * (2 * experts + 1)) * sizeof(float);
}

extern "C" int mpc_prior_balance(mpc_ctx *ctx, const void *scores, int type, int64_t rows, int experts, int64_t row_stride,
                                 int64_t expert_stride, float scale, int top_k, const uint8_t *mask, void *workspace, size_t workspace_bytes,
                                 float *loss, int32_t *counts, int32_t *n_rows) {
    MPC_ENTER(ctx);
    const int bad = check(ctx, scores, type, rows, experts, row_stride, expert_stride, scale, top_k);
    if (bad) return bad;
    MPC_REQUIRE(ctx, workspace && loss && counts && n_rows && ((uintptr_t)workspace & 7) == 0, "prior_balance: null or misaligned pointer");
    MPC_REQUIRE(ctx, workspace_bytes >= mpc_prior_balance_workspace_bytes(rows, experts), "prior_balance: workspace of %zu bytes", workspace_bytes);
    const Row a{scores, rows, row_stride, expert_stride, experts, scale, top_k, mask};
    if (type == MPC_TYPE_F32) return forward<float>(ctx, a, (float *)workspace, loss, counts, n_rows);
    if (type == MPC_TYPE_F16) return forward<f16_t>(ctx, a, (float *)workspace, loss, counts, n_rows);
    return forward<bf16_t>(ctx, a, (float *)workspace, loss, counts, n_rows);
}

extern "C" int mpc_prior_balance_grad(mpc_ctx *ctx, const void *scores, int type, int64_t rows, int experts, int64_t row_stride,
                                      int64_t expert_stride, float scale, int top_k, const uint8_t *mask, const int32_t *counts,
                                      const int32_t *n_rows, const float *grad_out, void *grad, int64_t grad_row_stride,
                                      int64_t grad_expert_stride) {
    MPC_ENTER(ctx);
    const int bad = check(ctx, scores, type, rows, experts, row_stride, expert_stride, scale, top_k);
    if (bad) return bad;
    if (rows == 0) return MPC_OK;
    MPC_REQUIRE(ctx, counts && n_rows && grad && (uintptr_t)grad % mpc_type_bytes(type) == 0, "prior_balance_grad: null or misaligned pointer");
    MPC_REQUIRE(ctx, grad_row_stride >= 0 && grad_expert_stride >= 0, "prior_balance_grad: negative stride");
    const Row a{scores, rows, row_stride, expert_stride, experts, scale, top_k, mask};
    if (type == MPC_TYPE_F32) return backward<float>(ctx, a, counts, n_rows, grad_out, grad, grad_row_stride, grad_expert_stride);
    if (type == MPC_TYPE_F16) return backward<f16_t>(ctx, a, counts, n_rows, grad_out, grad, grad_row_stride, grad_expert_stride);
    return backward<bf16_t>(ctx, a, counts, n_rows, grad_out, grad, grad_row_stride, grad_expert_stride);
}
