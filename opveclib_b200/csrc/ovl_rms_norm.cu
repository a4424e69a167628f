// Root-mean-square norm of rows with the residual's addition in front of it, with an output in the tensors' type or in
// 8 bits with scales, and its backward pass.  Interface: include/ovl_b200.h.
//
// What bounds it: bytes.  A team of threads (a warp for short rows, a block for long ones) holds its row in registers
// between the reduction and the outputs, so every element is read once and written once.
#include "ovl_sequence.cuh"

namespace ovl {
namespace {

constexpr int64_t kMaxColumns = 32768;
constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 1.1754943508e-38f;   // 2^-126, the smallest normal number

struct NormParams {
    OvlRmsNorm a;
    int32_t vec;
    int32_t group_lanes, group_shift;  // 8-bit output: lanes that share a scale (a power of two; 0: through shared memory)
    float* part;                       // backward: [blocks, columns]
    float inv_columns, eps;
};

// Teams: TEAM threads work on a row; a block has THREADS / TEAM teams.
template <int TEAM>
struct TeamShape {
    static constexpr int THREADS = TEAM < 128 ? 128 : TEAM;
    static constexpr int TEAMS = THREADS / TEAM;
    static constexpr int WARPS = TEAM / 32;
};

// sums of V values over a team, in a fixed order; every thread gets them
template <int TEAM, int V>
__device__ __forceinline__ void team_sum(float (&v)[V], float (*s_sum)[32]) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int s = 16; s >= 1; s >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], s);
    if constexpr (TEAM > 32) {
        const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
        __syncthreads();                                                 // the row before has read its sums
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) s_sum[i][warp] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = lane < TeamShape<TEAM>::WARPS ? s_sum[i][lane] : 0.0f;
#pragma unroll
            for (int s = 16; s >= 1; s >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], s);
        }
    }
}

// two e4m3 values, nearest with ties to even
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

// The scale of a group whose largest magnitude has these bits (a NaN stays one): the rounded quotient by 448, from the
// rounded 1 / 448 and one correction by the remainder (equal to the division for every fraction: 2^23 of them compared).
__device__ __forceinline__ float scale_of(unsigned int bits) {
    const float x = __uint_as_float(bits);
    float scale = x * (1.0f / kE4m3Max);
    scale = fmaf(fmaf(-scale, kE4m3Max, x), 1.0f / kE4m3Max, scale);
    if (bits == 0x7f800000u) scale = x;
    return scale < kMinScale ? kMinScale : scale;
}

// Values divided by a scale, on their way to e4m3: the reciprocal with one step of Newton's method, the quotient with one
// correction by its remainder (P. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor,
// 1990).  Newton's step is not the rounded reciprocal where the scale's fraction is all ones: that one's last bit is set
// here.  The quotient may be a step of 32 bits beside the rounded one, but never on another side of a border between two
// e4m3 values, nor on one instead of beside it: compared for every fraction of a scale, every border, the 13 values nearest
// to it and a first reciprocal of up to two steps beside the right one.  So q is that of a division, which takes 123 us
// for bf16 16384 x 4096 with 128 columns a scale instead of 92 (90 with one product by an approximate reciprocal, which puts
// some values on the wrong side).  Small scales and values are taken times 2^64 (exact), so that remainders stay normal
// numbers; by an infinite scale finite values are zeros, infinite ones NaN, as all are by NaN.
struct Scale {
    float scale, up, divisor, inverse;
    __device__ __forceinline__ explicit Scale(float s) : scale(s) {
        const bool infinite = __float_as_uint(s) == 0x7f800000u;
        up = s < 0x1p-60f ? 0x1p64f : 1.0f;
        divisor = infinite ? 1.0f : s * up;
        inverse = rcp_approx(divisor);
        inverse = fmaf(fmaf(-divisor, inverse, 1.0f), inverse, inverse);
        if ((__float_as_uint(s) & 0x7fffffu) == 0x7fffffu) inverse = __uint_as_float(__float_as_uint(inverse) | 1u);
        if (infinite) inverse = 0.0f;
    }
    __device__ __forceinline__ F2 divide(F2 x) const {
        x = mul2(x, same2(up));
        const F2 q = mul2(x, same2(inverse));
        return fma2(fma2(q, same2(-divisor), x), same2(inverse), q);
    }
    __device__ __forceinline__ float divide(float x) const {
        x *= up;
        const float q = x * inverse;
        return fmaf(fmaf(-q, divisor, x), inverse, q);
    }
};

// How a thread meets its packs of 8 columns, pack k starting at column (me + k * TEAM) * 8.  VEC: columns come in whole
// packs on 16-byte boundaries; a pack behind the last column reads the last one (no load waits for a condition) and counts
// as zeros.  Otherwise element by element.
template <typename T, int TEAM, bool VEC>
struct Columns {
    int columns, me;
    __device__ __forceinline__ int at(int k) const { return (me + k * TEAM) * 8; }
    __device__ __forceinline__ bool in(int k) const { return at(k) < columns; }
    __device__ __forceinline__ int valid(int k) const {
        const int left = columns - at(k);
        return VEC || left >= 8 ? 8 : left;
    }
    __device__ __forceinline__ Pack<T, 8> load(const T* row, int k) const {
        if (VEC) return load_pack<T, 8>(row + (in(k) ? at(k) : columns - 8), true, 8);
        return load_pack<T, 8>(row + at(k), false, in(k) ? valid(k) : 0);
    }
    __device__ __forceinline__ void store(T* row, int k, const float (&x)[8]) const {
        if (in(k)) store_pack<T, 8>(row + at(k), x, VEC, valid(k));
    }
    // the weights, zeros behind the last column
    __device__ __forceinline__ void weights(float (&w)[8], const void* weight, bool f32, int k) const {
        if (f32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = in(k) && i < valid(k) ? reinterpret_cast<const float*>(weight)[at(k) + i] : 0.0f;
        } else {
            const Pack<T, 8> raw = load(reinterpret_cast<const T*>(weight), k);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = in(k) ? to_f32(raw.v[i]) : 0.0f;
        }
    }
};

template <typename T, int TEAM, int K, bool QUANT, bool VEC>
__global__ void __launch_bounds__(TeamShape<TEAM>::THREADS) norm_forward(const __grid_constant__ NormParams p) {
    using S = TeamShape<TEAM>;
    constexpr int N = 8;
    __shared__ float s_sum[1][32];
    extern __shared__ unsigned int s_max[];                              // [teams][columns / group]
    const OvlRmsNorm& a = p.a;
    const int team = threadIdx.x / TEAM, me = threadIdx.x % TEAM;
    const int64_t row = (int64_t)blockIdx.x * S::TEAMS + team;
    const bool live = row < a.rows;                                      // (a warp as a whole; blocks are whole rows)
    if (TEAM == 32 && !QUANT && !live) return;
    const int columns = (int)a.columns;
    const Columns<T, TEAM, VEC> cols{columns, me};
    const int64_t from = live ? row : a.rows - 1;
    const T* const x = reinterpret_cast<const T*>(a.x) + from * a.x_row;
    const T* const res = a.residual ? reinterpret_cast<const T*>(a.residual) + from * a.residual_row : nullptr;

    Pack<T, N> raw[K], raw_r[K];
#pragma unroll
    for (int k = 0; k < K; ++k) raw[k] = cols.load(x, k);
    if (res) {
#pragma unroll
        for (int k = 0; k < K; ++k) raw_r[k] = cols.load(res, k);
    }
    float s[K][N], sum[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) s[k][i] = to_f32(raw[k].v[i]);
    if (res) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) s[k][i] += to_f32(raw_r[k].v[i]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (VEC && !cols.in(k)) continue;                                // (element by element the rest is zeros already)
#pragma unroll
        for (int i = 0; i < N; ++i) sum[0] = fmaf(s[k][i], s[k][i], sum[0]);
    }
    if (a.residual_out && live) {
        T* const to = reinterpret_cast<T*>(a.residual_out) + row * a.columns;
#pragma unroll
        for (int k = 0; k < K; ++k) cols.store(to, k, s[k]);
    }
    team_sum<TEAM, 1>(sum, s_sum);
    const float r = rsqrtf(fmaf(sum[0], p.inv_columns, p.eps));
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float w[N];
        cols.weights(w, a.weight, a.params_f32, k);
#pragma unroll
        for (int i = 0; i < N; ++i) s[k][i] = QUANT ? s[k][i] * r * w[i] : s[k][i] * (r * w[i]);
        if (VEC && !cols.in(k)) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[k][i] = 0.0f;
        }
        if (!QUANT && live) cols.store(reinterpret_cast<T*>(a.y) + row * a.columns, k, s[k]);
    }
    if constexpr (QUANT) {
        // The largest magnitude of a group, as the largest bit pattern: a NaN stays the largest.
        const int group = (int)a.group, groups = columns / group;
        unsigned int* const maxima = s_max + team * groups;
        const bool one_scale = p.group_lanes || groups == 1;             // for the 8 values of a pack
        unsigned int top[K];
        if (one_scale) {
            unsigned int whole = 0;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                top[k] = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) top[k] = max(top[k], __float_as_uint(s[k][i]) & 0x7fffffffu);
                whole = max(whole, top[k]);
            }
            if (groups == 1) {
                whole = __reduce_max_sync(0xffffffffu, whole);
                if (me == 0) maxima[0] = 0;
                __syncthreads();
                if (me % 32 == 0) atomicMax(maxima, whole);
                __syncthreads();
                whole = maxima[0];
#pragma unroll
                for (int k = 0; k < K; ++k) top[k] = whole;
            } else {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    for (int l = 1; l < p.group_lanes; l *= 2) top[k] = max(top[k], __shfl_xor_sync(0xffffffffu, top[k], l));
            }
        } else {
            for (int i = me; i < groups; i += TEAM) maxima[i] = 0;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int col = cols.at(k);
                unsigned int run = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (col + i >= columns) continue;
                    run = max(run, __float_as_uint(s[k][i]) & 0x7fffffffu);
                    if (i == N - 1 || col + i + 1 >= columns || (col + i + 1) % group == 0) {
                        atomicMax(maxima + (col + i) / group, run);
                        run = 0;
                    }
                }
            }
            __syncthreads();
        }
        if (!live) return;
        uint8_t* const q = reinterpret_cast<uint8_t*>(a.q) + row * a.columns;
        float* const scales = a.scale + row * groups;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int col = cols.at(k);
            if (col >= columns) continue;
            float v[N];
            if (one_scale) {
                const Scale by(scale_of(top[k]));
#pragma unroll
                for (int i = 0; i < N; i += 2) unpack2(by.divide(pack2(s[k][i], s[k][i + 1])), v[i], v[i + 1]);
                const int pack = me + k * TEAM;                          // a group is group_lanes (a power of two) packs
                if (groups == 1 ? pack == 0 : (pack & (p.group_lanes - 1)) == 0) scales[groups == 1 ? 0 : pack >> p.group_shift] = by.scale;
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (col + i >= columns) continue;
                    const int g = (col + i) / group;
                    const Scale by(scale_of(maxima[g]));
                    v[i] = by.divide(s[k][i]);
                    if (col + i == g * group) scales[g] = by.scale;
                }
            }
            // (an infinite value meets an infinite scale: inf / inf is NaN)
            if (VEC) {
                uint2 bytes;
                bytes.x = e4m3_pair(v[0], v[1]) | e4m3_pair(v[2], v[3]) << 16;
                bytes.y = e4m3_pair(v[4], v[5]) | e4m3_pair(v[6], v[7]) << 16;
                *reinterpret_cast<uint2*>(q + col) = bytes;
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (col + i < columns) q[col + i] = (uint8_t)e4m3_pair(v[i], 0.0f);
            }
        }
    }
}

// With g = gy w and xhat = s r: gx = r (g - xhat mean(g xhat)) + gresidual_out; gweight = sum over the rows of gy xhat.
// Every team walks over rows with its sums for gweight in registers; as long as shared memory lasts the next row is copied
// there meanwhile, each thread what it will need itself.
template <typename T, int TEAM, int K>
struct BackRows {
    static constexpr size_t stage = sizeof(T) * 4 * K * TeamShape<TEAM>::THREADS * 8;        // x, residual, gy, gresidual_out
    static constexpr bool AHEAD = 2 * stage <= 128 * 1024;
    static constexpr size_t bytes = AHEAD ? 2 * stage : 0;
};

template <typename T, int TEAM, int K, bool VEC>
__global__ void __launch_bounds__(TeamShape<TEAM>::THREADS) norm_backward(const __grid_constant__ NormParams p) {
    using S = TeamShape<TEAM>;
    constexpr int N = 8;
    constexpr bool AHEAD = BackRows<T, TEAM, K>::AHEAD;
    __shared__ float s_sum[2][32];
    __shared__ float s_w[TEAM == 32 ? S::TEAMS : 1][TEAM == 32 ? TEAM * K * N : 1];
    extern __shared__ __align__(16) char smem[];
    const OvlRmsNorm& a = p.a;
    const int team = threadIdx.x / TEAM, me = threadIdx.x % TEAM;
    const int columns = (int)a.columns;
    const Columns<T, TEAM, VEC> cols{columns, me};
    float w[K][N], gw[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        cols.weights(w[k], a.weight, a.params_f32, k);
#pragma unroll
        for (int i = 0; i < N; ++i) gw[k][i] = 0.0f;
    }
    const int64_t first = (int64_t)blockIdx.x * S::TEAMS + team, step = (int64_t)gridDim.x * S::TEAMS;
    const bool more = a.gresidual_out != nullptr, sum_of_two = a.residual != nullptr;
    auto row_of = [&](int which, int64_t row) {
        return which == 0   ? reinterpret_cast<const T*>(a.x) + row * a.x_row
               : which == 1 ? reinterpret_cast<const T*>(a.residual) + row * a.residual_row
               : which == 2 ? reinterpret_cast<const T*>(a.gy) + row * a.gy_row
                            : reinterpret_cast<const T*>(a.gresidual_out) + row * a.gresidual_out_row;
    };
    auto slot_of = [&](int stage, int which, int k) {
        return reinterpret_cast<T*>(smem) + (((stage * 4 + which) * K + k) * S::THREADS + threadIdx.x) * 8;
    };
    auto fetch = [&](int64_t row, int stage) {
        if (row < a.rows) {
#pragma unroll
            for (int which = 0; which < 4; ++which) {
                if ((which == 1 && !sum_of_two) || (which == 3 && !more)) continue;
                const T* const from = row_of(which, row);
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (cols.in(k)) fetch_pack<T, N>(slot_of(stage, which, k), from + cols.at(k), VEC, cols.valid(k), 0);
            }
        }
        copy_commit();
    };
    auto read = [&](float (&x)[K][N], int which, int64_t row, int stage) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (AHEAD) {
                read_slot<T, N>(slot_of(stage, which, k), x[k]);
            } else {
                const Pack<T, N> raw = cols.load(row_of(which, row), k);
#pragma unroll
                for (int i = 0; i < N; ++i) x[k][i] = to_f32(raw.v[i]);
            }
            if (!cols.in(k)) {
#pragma unroll
                for (int i = 0; i < N; ++i) x[k][i] = 0.0f;
            }
        }
    };
    int stage = 0;
    if (AHEAD) fetch(first, 0);
    for (int64_t row = first; row < a.rows; row += step, stage ^= 1) {
        if (AHEAD) {
            fetch(row + step, stage ^ 1);
            copy_wait<1>();
        }
        // the sum in 32 bits, as the forward pass had it (its rounded copy would put another rounding on gweight)
        float s[K][N], g[K][N];
        read(s, 0, row, stage);
        if (sum_of_two) {
            read(g, 1, row, stage);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) s[k][i] += g[k][i];
        }
        read(g, 2, row, stage);
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                sum[0] = fmaf(s[k][i], s[k][i], sum[0]);
                sum[1] = fmaf(s[k][i] * w[k][i], g[k][i], sum[1]);
            }
        team_sum<TEAM, 2>(sum, s_sum);
        const float r = rsqrtf(fmaf(sum[0], p.inv_columns, p.eps));
        const float mean = r * r * (sum[1] * p.inv_columns);            // xhat mean(g xhat) = s mean, apart from a factor r
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                gw[k][i] = fmaf(g[k][i], s[k][i] * r, gw[k][i]);
                s[k][i] = r * fmaf(-s[k][i], mean, g[k][i] * w[k][i]);
            }
        if (more) {
            read(g, 3, row, stage);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) s[k][i] += g[k][i];
        }
#pragma unroll
        for (int k = 0; k < K; ++k) cols.store(reinterpret_cast<T*>(a.gx) + row * a.columns, k, s[k]);
    }
    float* const part = p.part + (int64_t)blockIdx.x * columns;
    if constexpr (TEAM == 32) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) s_w[team][(me + k * TEAM) * N + i] = gw[k][i];
        __syncthreads();
        for (int col = threadIdx.x; col < columns; col += S::THREADS) {
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < S::TEAMS; ++t) sum += s_w[t][col];
            part[col] = sum;
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (cols.at(k) + i < columns) part[cols.at(k) + i] = gw[k][i];
    }
}

// gweight: the blocks' parts added up in order; a warp's lanes are 32 columns, the 32 warps of a block slices of the parts
constexpr int kPartWarps = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kPartWarps) norm_backward_weight(const __grid_constant__ NormParams p, int64_t parts) {
    __shared__ float s_part[kPartWarps][32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t col = (int64_t)blockIdx.x * 32 + lane;
    float sum = 0.0f;
    if (col < p.a.columns) {
#pragma unroll 8
        for (int64_t r = warp; r < parts; r += kPartWarps) sum += p.part[r * p.a.columns + col];
    }
    s_part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && col < p.a.columns) {
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kPartWarps; ++w) sum += s_part[w][lane];
        if (p.a.params_f32) reinterpret_cast<float*>(p.a.gweight)[col] = sum;
        else reinterpret_cast<T*>(p.a.gweight)[col] = from_f32<T>(sum);
    }
}

// ---------------------------------------------------------------------------------------------------------
// host side

int check(const OvlRmsNorm* a) {
    if (!a) return OVL_ERR_NULL;
    if (a->dtype != OVL_FLOAT32 && a->dtype != OVL_FLOAT16 && a->dtype != OVL_BFLOAT16) return OVL_ERR_DTYPE;
    if (a->rows < 0 || a->columns < 1 || a->group < 0) return OVL_ERR_INVALID;
    if (a->group > 0 && a->columns % a->group != 0) return OVL_ERR_INVALID;
    if (a->columns > kMaxColumns) return OVL_ERR_TOO_LARGE;
    return OVL_OK;
}

int team_of(int64_t columns) { return columns <= 1024 ? 32 : columns <= 8192 ? 256 : 512; }
int teams_of_block(int team) { return team == 32 ? 4 : 1; }

// blocks of the backward pass: they stay for all rows, so their parts of gweight are few
int64_t backward_blocks(const OvlRmsNorm* a) {
    const int team = team_of(a->columns);
    const int64_t most = (int64_t)sequence_sm_count() * (team == 32 ? 8 : team == 256 ? 4 : 2);
    const int64_t blocks = ceil_div(a->rows, teams_of_block(team));
    return blocks < 1 ? 1 : blocks < most ? blocks : most;
}

template <typename T, int TEAM, int K, bool VEC>
int launch_forward_as(const NormParams& p, cudaStream_t stream) {
    using S = TeamShape<TEAM>;
    const int64_t blocks = ceil_div(p.a.rows, S::TEAMS);
    if (blocks > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    if (p.a.group > 0) {
        const size_t groups = p.a.columns / p.a.group;
        const size_t smem = p.group_lanes && groups > 1 ? 0 : S::TEAMS * groups * sizeof(unsigned int);
        if (smem > 24 * 1024) {                                          // up to a scale for every column
            const int st = prepare_kernel((const void*)norm_forward<T, TEAM, K, true, VEC>, sizeof(unsigned int) * S::TEAMS * TEAM * K * 8);
            if (st != OVL_OK) return st;
        }
        norm_forward<T, TEAM, K, true, VEC><<<(uint32_t)blocks, S::THREADS, smem, stream>>>(p);
    } else {
        norm_forward<T, TEAM, K, false, VEC><<<(uint32_t)blocks, S::THREADS, 0, stream>>>(p);
    }
    return launch_status();
}

template <typename T, int TEAM, int K, bool VEC>
int launch_backward_as(const NormParams& p, cudaStream_t stream) {
    constexpr size_t smem = BackRows<T, TEAM, K>::bytes;
    const int st = prepare_kernel((const void*)norm_backward<T, TEAM, K, VEC>, smem);
    if (st != OVL_OK) return st;
    norm_backward<T, TEAM, K, VEC><<<(uint32_t)backward_blocks(&p.a), TeamShape<TEAM>::THREADS, smem, stream>>>(p);
    return launch_status();
}

template <typename T, int TEAM, int K>
int launch_forward(const NormParams& p, cudaStream_t stream) {
    return p.vec ? launch_forward_as<T, TEAM, K, true>(p, stream) : launch_forward_as<T, TEAM, K, false>(p, stream);
}
template <typename T, int TEAM, int K>
int launch_backward(const NormParams& p, cudaStream_t stream) {
    return p.vec ? launch_backward_as<T, TEAM, K, true>(p, stream) : launch_backward_as<T, TEAM, K, false>(p, stream);
}
template <typename T, int TEAM, int K>
int launch(const NormParams& p, bool backward, cudaStream_t stream) {
    return backward ? launch_backward<T, TEAM, K>(p, stream) : launch_forward<T, TEAM, K>(p, stream);
}

// Columns of a thread: 8, 16 and 32 for a warp's rows (up to 1024), then forwards 16 up to 2048 and 32 up to 16384 - what a
// thread does once per row (the sum over the team, the roots and scales) weighs less than with 16 (bf16 16384 x 4096 to 8
// bits, before its quotients were corrected: 85 us, 89 with 256 threads of 16 columns).  Backwards 8 up to 2048, 16 up to
// 4096 and 32 up to 16384, and 64 above that both ways: from 8193 columns on the backward kernel spills (164 to 332 bytes of
// loads with 32 columns, 1.4 KB in 16 bits and 4.4 KB in fp32 with 64; bf16 4096 x 16384: 149 us, 2.7 TB/s, 2048 x 32768: 329
// us, 1.2 TB/s).
template <typename T>
int dispatch(const NormParams& p, bool backward, cudaStream_t stream) {
    const int64_t c = p.a.columns;
    if (c <= 256) return launch<T, 32, 1>(p, backward, stream);
    if (c <= 512) return launch<T, 32, 2>(p, backward, stream);
    if (c <= 1024) return launch<T, 32, 4>(p, backward, stream);
    if (c <= 2048) return backward ? launch_backward<T, 256, 1>(p, stream) : launch_forward<T, 128, 2>(p, stream);
    if (c <= 4096) return backward ? launch_backward<T, 256, 2>(p, stream) : launch_forward<T, 128, 4>(p, stream);
    if (c <= 8192) return launch<T, 256, 4>(p, backward, stream);
    if (c <= 16384) return launch<T, 512, 4>(p, backward, stream);
    return launch<T, 512, 8>(p, backward, stream);
}

int run(NormParams& p, bool backward, cudaStream_t stream) {
    p.inv_columns = (float)(1.0 / (double)p.a.columns);
    p.eps = (float)p.a.eps;
    if (p.a.dtype == OVL_FLOAT32) return dispatch<float>(p, backward, stream);
    if (p.a.dtype == OVL_FLOAT16) return dispatch<__half>(p, backward, stream);
    return dispatch<__nv_bfloat16>(p, backward, stream);
}

}  // namespace
}  // namespace ovl

extern "C" uint64_t ovl_rms_norm_workspace_bytes(const OvlRmsNorm* a) {
    if (ovl::check(a) != OVL_OK) return 0;
    return (uint64_t)ovl::backward_blocks(a) * a->columns * sizeof(float);
}

extern "C" int ovl_rms_norm(const OvlRmsNorm* a, void* cuda_stream) {
    const int st = ovl::check(a);
    if (st != OVL_OK) return st;
    if (a->rows == 0) return OVL_OK;
    if (!a->x || !a->weight) return OVL_ERR_NULL;
    if (a->group > 0 ? (!a->q || !a->scale) : !a->y) return OVL_ERR_NULL;
    ovl::NormParams p{};
    p.a = *a;
    p.vec = a->columns % 8 == 0 && ovl::aligned16(a->x) && a->x_row % 8 == 0 && ovl::aligned16(a->residual) &&
            (!a->residual || a->residual_row % 8 == 0) && ovl::aligned16(a->residual_out) && ovl::aligned16(a->weight) &&
            (a->group > 0 ? ovl::aligned16(a->q) : ovl::aligned16(a->y));
    const int64_t lanes = a->group / 8;
    if (a->group % 8 == 0 && lanes >= 1 && lanes <= 32 && (lanes & (lanes - 1)) == 0) {
        p.group_lanes = (int32_t)lanes;
        while ((1 << p.group_shift) < p.group_lanes) ++p.group_shift;
    }
    return ovl::run(p, false, (cudaStream_t)cuda_stream);
}

extern "C" int ovl_rms_norm_backward(const OvlRmsNorm* a, void* cuda_stream) {
    const int st = ovl::check(a);
    if (st != OVL_OK) return st;
    if (!a->weight || !a->gweight || (a->rows > 0 && (!a->x || !a->gy || !a->gx))) return OVL_ERR_NULL;
    if (!a->workspace || a->workspace_bytes < ovl_rms_norm_workspace_bytes(a) || !ovl::aligned16(a->workspace)) return OVL_ERR_SCRATCH;
    ovl::NormParams p{};
    p.a = *a;
    p.part = reinterpret_cast<float*>(a->workspace);
    p.vec = a->columns % 8 == 0 && ovl::aligned16(a->x) && a->x_row % 8 == 0 && ovl::aligned16(a->residual) &&
            (!a->residual || a->residual_row % 8 == 0) && ovl::aligned16(a->gy) && a->gy_row % 8 == 0 &&
            ovl::aligned16(a->gresidual_out) && (!a->gresidual_out || a->gresidual_out_row % 8 == 0) && ovl::aligned16(a->gx) &&
            ovl::aligned16(a->weight);
    const cudaStream_t stream = (cudaStream_t)cuda_stream;
    const int s = ovl::run(p, true, stream);
    if (s != OVL_OK) return s;
    const uint32_t grid = (uint32_t)ovl::ceil_div(a->columns, 32);
    const int64_t parts = ovl::backward_blocks(a);
    if (a->dtype == OVL_FLOAT32) ovl::norm_backward_weight<float><<<grid, 32 * ovl::kPartWarps, 0, stream>>>(p, parts);
    else if (a->dtype == OVL_FLOAT16) ovl::norm_backward_weight<__half><<<grid, 32 * ovl::kPartWarps, 0, stream>>>(p, parts);
    else ovl::norm_backward_weight<__nv_bfloat16><<<grid, 32 * ovl::kPartWarps, 0, stream>>>(p, parts);
    return ovl::launch_status();
}
