// Selective scan: h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t, out_t = (C_t . h_t + D u_t) silu(z_t), for prompts and
// training (forward and backward) and for single tokens.  Interface: include/ovl_b200.h.
//
// What bounds it.  A (token, channel) moves 8 bytes (u, delta, z, out in 16 bits) and needs one exponential per state.
// The special-function unit delivers 16 per clock and SM: with 16 states one (token, channel) per clock and SM, 2.8e11
// per second on 148 SMs, while 8 bytes at the measured copy bandwidth allow 8e11.  So the recurrence itself has to stay
// out of the way of the exponentials: it runs serially over the tokens in registers (no scan over lanes, which would
// multiply the arithmetic), and everything that is needed once per (token, channel) is computed once, in shared memory.
//
// Layout.  Prompts, forwards: a lane has 4 states of M channels (1 or 2), a channel P lanes of a warp (P = 1 ... 32: up to
// 128 states, rounded up to a power of two).  A block is 128 scanning threads = CH channels of one group of one batch, and
// 128 helping ones.  Tokens come in tiles of STEPS: while a tile is scanned the helping threads have the next ones'
// elements in flight to shared memory, each those that it will convert, mask and combine itself (softplus, dt * u) into
// what all lanes of a channel read, and finish the outputs of the tile before; double-buffered, with one barrier per tile.
// The sums over the states of V steps are formed together (reduce_lanes: less than one exchange per step).  Backwards alike,
// with 2 states (4 above 64) of 2 channels (1 above 64) a lane.
#pragma once
#include "ovl_sequence.cuh"

namespace ovl {

constexpr int kCheckpoint = 16;        // tokens between two saved states of a training step
constexpr int kMaxStates = 128;
constexpr int kMaxSegments = 32;

struct ScanDims {
    int64_t length, channels, states, groups;
    int64_t group_channels;            // channels of a group
    int64_t all_tiles, first_tile, tiles;      // channel tiles of a group; those of this launch
    int64_t segments, segment_length;  // the length cut into segments (a multiple of 32) that run side by side
    int64_t first_segment, launch_segments;   // those of this launch
    int32_t ahead;                     // the first of two launches, see below
    int32_t softplus, vec, width;      // vec: wide loads and stores of channel vectors; else copies of `width` elements
    int32_t vec_states, vec_bc;        // wide loads and stores of 4 states; of 4 elements of B and C
};

struct ScanParams {
    ScanDims d;
    OvlSelectiveScan a;
    float* seg_state;                  // [batch, segments, channels, states]: what a segment adds to the state
    float* seg_dt;                     // [batch, segments, channels]: sum of dt over the segment
    float* part_bc;                    // [batch, groups, tiles, length, 2, padded states]: gC and gB of a channel tile
    float* sum_bc;                     // [batch, groups, length, 2, padded states]: their sum over the launches before
    float* part_A;                     // [batch * segments, channels, states]
    float* part_D;                     // [batch * segments, 2, channels]: gD, gdelta_bias
};

// Lanes of a channel, pairs of states of a lane, channels of a lane.
struct ScanShape {
    int lanes, pairs, channels;
    int padded_states() const { return 2 * pairs * lanes; }
    int block_channels() const { return 128 / lanes * channels; }
};

// One source per element type (they are compiled side by side).
__attribute__((visibility("hidden"))) int scan_run_f32(const ScanParams&, const ScanShape&, bool backward, cudaStream_t);
__attribute__((visibility("hidden"))) int scan_run_f16(const ScanParams&, const ScanShape&, bool backward, cudaStream_t);
__attribute__((visibility("hidden"))) int scan_run_bf16(const ScanParams&, const ScanShape&, bool backward, cudaStream_t);
__attribute__((visibility("hidden"))) int scan_step_f32(const OvlSelectiveScanStep&, int lanes, cudaStream_t);
__attribute__((visibility("hidden"))) int scan_step_f16(const OvlSelectiveScanStep&, int lanes, cudaStream_t);
__attribute__((visibility("hidden"))) int scan_step_bf16(const OvlSelectiveScanStep&, int lanes, cudaStream_t);

namespace {

// K pairs of states from state n0 on
template <int K>
__device__ __forceinline__ void load_states(F2 (&x)[K], const float* p, int n0, int states, bool vec) {
    if (vec && n0 < states) {
        if constexpr (K == 2) {
            const float4 r = *reinterpret_cast<const float4*>(p + n0);
            x[0] = pack2(r.x, r.y);
            x[1] = pack2(r.z, r.w);
        } else {
            const float2 r = *reinterpret_cast<const float2*>(p + n0);
            x[0] = pack2(r.x, r.y);
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int n = n0 + 2 * k;
        x[k] = pack2(n < states ? p[n] : 0.0f, n + 1 < states ? p[n + 1] : 0.0f);
    }
}
template <int K>
__device__ __forceinline__ void store_states(float* p, const F2 (&x)[K], int n0, int states, bool vec) {
    float v[2 * K];
#pragma unroll
    for (int k = 0; k < K; ++k) unpack2(x[k], v[2 * k], v[2 * k + 1]);
    if (vec && n0 < states) {
        if constexpr (K == 2) *reinterpret_cast<float4*>(p + n0) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<float2*>(p + n0) = make_float2(v[0], v[1]);
        return;
    }
#pragma unroll
    for (int k = 0; k < 2 * K; ++k)
        if (n0 + k < states) p[n0 + k] = v[k];
}
// K pairs of one row of B or C in shared memory
template <int K>
__device__ __forceinline__ void read_pairs(F2 (&x)[K], const float* p) {
    if constexpr (K == 2) {
        const float4 r = *reinterpret_cast<const float4*>(p);
        x[0] = pack2(r.x, r.y);
        x[1] = pack2(r.z, r.w);
    } else {
        const float2 r = *reinterpret_cast<const float2*>(p);
        x[0] = pack2(r.x, r.y);
    }
}
// the sum over both states of K pairs of the products x y
template <int K>
__device__ __forceinline__ float dot(const F2 (&x)[K], const F2 (&y)[K]) {
    F2 r = mul2(x[0], y[0]);
#pragma unroll
    for (int k = 1; k < K; ++k) r = fma2(x[k], y[k], r);
    return sum2(r);
}

__device__ __forceinline__ int64_t used_length(const int32_t* lengths, int64_t batch, int64_t length) {
    if (!lengths) return length;
    const int64_t n = lengths[batch];
    return n < 0 ? 0 : n > length ? length : n;
}

// which piece of the problem a block works on (a launch covers the segments from first_segment and the tiles from
// first_tile on)
struct Place {
    int64_t batch, segment, group, tile, channel0, n_channels;   // tile: of the launch's; channels from channel0 on
};
__device__ __forceinline__ Place block_place(const ScanDims& d, int ch) {
    Place p;
    int64_t i = blockIdx.x;
    p.tile = i % d.tiles;
    i /= d.tiles;
    p.group = i % d.groups;
    i /= d.groups;
    p.segment = d.first_segment + i % d.launch_segments;
    p.batch = i / d.launch_segments;
    const int64_t skip = (d.first_tile + p.tile) * ch, left = d.group_channels - skip;
    p.channel0 = p.group * d.group_channels + skip;
    p.n_channels = left < ch ? left : ch;
    return p;
}

// exp(dt A) = 2^(dt A log2 e).  The special-function unit's results are 1e-8 to 2e-8 too small on average, which adds up
// over a state's memory of a thousand tokens; the same amount on the exponent takes most of it away and costs nothing
// (a multiplication becomes a multiply-add).  2^kExpBias rounds to 1, so dt = 0 still leaves a state as it is.
constexpr float kExpBias = 2e-8f;
__device__ __forceinline__ F2 decay(F2 A, F2 dt) { return exp2_pair(fma2(A, dt, same2(kExpBias))); }

// ---------------------------------------------------------------------------------------------------------
// forward

// P lanes x 4 states x M channels: a block is 128 scanning threads = 128 / P * M channels, and 128 helping threads.
template <int P, int M>
struct ForwardShape {
    static constexpr int SCAN = 128, HELP = 128, THREADS = SCAN + HELP;
    static constexpr int CH = SCAN / P * M;                              // channels of a block
    static constexpr int NP = 4 * P;                                     // states, padded
    static constexpr int STEPS = CH >= 128 ? 8 : CH >= 64 ? 16 : 32;     // tokens of a tile
    static constexpr int V = STEPS < 16 / M ? STEPS : 16 / M;            // steps whose sums are formed together
    static constexpr int ITEMS = STEPS * CH / 8;                         // 8 channels of one token
    static constexpr int IPT = (ITEMS + HELP - 1) / HELP;
    static constexpr int QUADS = STEPS * P, QPT = (QUADS + HELP - 1) / HELP;   // 4 states of one token
    static constexpr int AHEAD = 2;                                      // tiles that are fetched ahead of the scan
    static constexpr int DU = CH + CH / 8 * 2;                           // row of s_du: 16 bytes of gap after 8 channels
    static constexpr int ROW = CH + (P >= 8 ? 4 : 32 / P);               // row of s_y: lanes of different steps hit different banks
};

template <typename T, int P, int M>
struct ForwardSmem {
    using S = ForwardShape<P, M>;
    static constexpr size_t du = 0;                                                          // float2 [2][STEPS][DU]
    static constexpr size_t b = du + 2 * sizeof(float2) * S::STEPS * S::DU;                  // float [2][STEPS][NP]
    static constexpr size_t c = b + 2 * sizeof(float) * S::STEPS * S::NP;
    static constexpr size_t y = c + 2 * sizeof(float) * S::STEPS * S::NP;                    // float [2][STEPS][ROW]
    static constexpr size_t raw = y + 2 * sizeof(float) * S::STEPS * S::ROW;                 // T [AHEAD + 1][3][ITEMS][8]: u, delta, z
    static constexpr size_t raw_bc = raw + (S::AHEAD + 1) * 3 * sizeof(T) * S::STEPS * S::CH;             // T [AHEAD][2][QUADS][4]: B, C
    static constexpr size_t bytes = raw_bc + S::AHEAD * 2 * sizeof(T) * S::STEPS * S::NP;
};

// The scanning threads: nothing but the recurrence and its sums over the states.  A lane reads 16 bytes of dt and dt u
// (two channels) and 32 bytes of B and C per step and 8 states: shared memory hands out 128 bytes per clock to the SM's
// lanes whether they share addresses or not, which would make a lane with one channel wait for it (46 clocks per warp
// and step measured, 32 for the exponentials).
template <typename T, int P, int M, bool LOCAL>
__device__ __forceinline__ void scan_forward_scan(const ScanParams& p, const Place& at, char* smem, int64_t t_begin, int64_t t_used) {
    using S = ForwardShape<P, M>;
    using Mem = ForwardSmem<T, P, M>;
    constexpr int NP = S::NP, STEPS = S::STEPS, V = S::V;
    const OvlSelectiveScan& a = p.a;
    const ScanDims& d = p.d;
    const int tid = threadIdx.x, lane = tid % 32, j = lane % P, c0 = tid / P * M, n0 = 4 * j;
    const int states = (int)d.states;
    int64_t row[M];                                                      // of this channel's states in [batch, channels, states]
    bool live[M];
    F2 A[M][2], h[M][2];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        live[m] = c0 + m < at.n_channels;
        const int64_t channel = at.channel0 + (live[m] ? c0 + m : 0);
        row[m] = (at.batch * d.channels + channel) * states;
        load_states(A[m], a.A + channel * states, n0, states, d.vec_states);    // padded states have A = B = C = 0
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            A[m][k] = mul2(A[m][k], same2(kLog2e));
            h[m][k] = same2(0.0f);
        }
        if (LOCAL) continue;
        // the state in front of this segment: the one behind the first segment, then h <- exp(A sum dt) h + (what the
        // segment adds) for those between
        if (at.segment > 0) load_states(h[m], p.seg_state + (at.batch * d.segments * d.channels + channel) * states, n0, states, d.vec_states);
        else if (a.initial_state) load_states(h[m], a.initial_state + row[m], n0, states, d.vec_states);
        for (int64_t s = 1; s < at.segment; ++s) {
            const int64_t cell = (at.batch * d.segments + s) * d.channels + channel;
            const F2 sum = same2(p.seg_dt[cell]);
            F2 add[2];
            load_states(add, p.seg_state + cell * states, n0, states, d.vec_states);
#pragma unroll
            for (int k = 0; k < 2; ++k) h[m][k] = fma2(decay(A[m][k], sum), h[m][k], add[k]);
        }
    }
    const float2* const s_du = reinterpret_cast<const float2*>(smem + Mem::du) + c0 + c0 / 8 * 2;
    const float* const s_b = reinterpret_cast<const float*>(smem + Mem::b) + n0;
    const float* const s_c = reinterpret_cast<const float*>(smem + Mem::c) + n0;
    float* const s_y = reinterpret_cast<float*>(smem + Mem::y) + c0;
    const int64_t chunks = (d.length + kCheckpoint - 1) / kCheckpoint;
    float sum_dt[M] = {};
    __syncthreads();
    int buf = 0;
    for (int64_t t0 = t_begin; t0 < t_used; t0 += STEPS, buf ^= 1) {
        // The factors and addends of two steps are formed while the two before them are walked, so that a warp that is
        // alone on its scheduler does not wait for its own exponentials at every step (95 clocks per warp, step and two
        // channels against 108; 57 against 59 with one channel).
        F2 f[2][M][2], x[2][M][2], cc[2][2];
        float y[M][V];
        auto prepare = [&](int step, int i) {
            const int t = buf * STEPS + step;
            float dt[M], du[M];
            if constexpr (M == 2) {
                const float4 v = *reinterpret_cast<const float4*>(s_du + t * S::DU);
                dt[0] = v.x, du[0] = v.y, dt[1] = v.z, du[1] = v.w;
            } else {
                const float2 v = s_du[t * S::DU];
                dt[0] = v.x, du[0] = v.y;
            }
            F2 b[2];
            read_pairs(b, s_b + t * NP);
            if (!LOCAL) read_pairs(cc[i], s_c + t * NP);
#pragma unroll
            for (int m = 0; m < M; ++m) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    f[i][m][k] = decay(A[m][k], same2(dt[m]));
                    x[i][m][k] = mul2(same2(du[m]), b[k]);
                }
                if (LOCAL) sum_dt[m] += dt[m];
            }
        };
        prepare(0, 0);
        prepare(1, 1);
#pragma unroll
        for (int step = 0; step < STEPS; ++step) {
            const int i = step % 2;
            if (step % V == 0 && !LOCAL && a.checkpoints && (t0 + step) % kCheckpoint == 0 && t0 + step < d.length) {
                const int64_t skip = (at.batch * (chunks - 1) + (t0 + step) / kCheckpoint) * d.channels * states;
#pragma unroll
                for (int m = 0; m < M; ++m)
                    if (live[m]) store_states(a.checkpoints + skip + row[m], h[m], n0, states, d.vec_states);
            }
#pragma unroll
            for (int m = 0; m < M; ++m) {
#pragma unroll
                for (int k = 0; k < 2; ++k) h[m][k] = fma2(f[i][m][k], h[m][k], x[i][m][k]);
                if (!LOCAL) y[m][step % V] = dot(h[m], cc[i]);
            }
            if (step + 2 < STEPS) prepare(step + 2, i);
            if (!LOCAL && step % V == V - 1) {
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    reduce_lanes<V, P, 1>(y[m], lane);
                    if (reduced_owner<V, P>(j)) {
                        const int t = buf * STEPS + step - (V - 1) + reduced_index<V, P>(j);
#pragma unroll
                        for (int e = 0; e < reduced_count<V, P>(); ++e) s_y[(t + e) * S::ROW + m] = y[m][e];
                    }
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
        if (!live[m]) continue;
        const int64_t channel = at.channel0 + c0 + m, cell = (at.batch * d.segments + at.segment) * d.channels + channel;
        if (d.ahead) store_states(p.seg_state + cell * states, h[m], n0, states, d.vec_states);
        if (LOCAL && j == 0) p.seg_dt[cell] = sum_dt[m];
        if (!LOCAL && a.final_state && at.segment == d.segments - 1)
            store_states(a.final_state + row[m], h[m], n0, states, d.vec_states);
    }
}

// The helping threads, one tile ahead of the scan and one behind it: they fetch u, delta, z, B and C (AHEAD tiles ahead,
// each thread what it will need itself), leave dt, dt u, B and C for the scan, and finish the outputs from its sums.
template <typename T, int P, int M, bool LOCAL, bool FULL>
__device__ __forceinline__ void scan_forward_help(const ScanParams& p, const Place& at, char* smem, int64_t t_begin, int64_t t_end,
                                                  int64_t t_used) {
    using S = ForwardShape<P, M>;
    using Mem = ForwardSmem<T, P, M>;
    constexpr int CH = S::CH, NP = S::NP, STEPS = S::STEPS, IPT = S::IPT, QPT = S::QPT;
    const OvlSelectiveScan& a = p.a;
    const ScanDims& d = p.d;
    const int tid = threadIdx.x - S::SCAN;
    const int states = (int)d.states;
    float2* const s_du = reinterpret_cast<float2*>(smem + Mem::du);
    const T* const u = reinterpret_cast<const T*>(a.u) + at.batch * a.u_batch + at.channel0;
    const T* const delta = reinterpret_cast<const T*>(a.delta) + at.batch * a.delta_batch + at.channel0;
    const T* const z = a.z ? reinterpret_cast<const T*>(a.z) + at.batch * a.z_batch + at.channel0 : nullptr;
    T* const out = reinterpret_cast<T*>(a.out) + at.batch * d.length * d.channels + at.channel0;
    const T* const B = reinterpret_cast<const T*>(a.B) + at.batch * a.B_batch + at.group * a.B_group;
    const T* const C = reinterpret_cast<const T*>(a.C) + at.batch * a.C_batch + at.group * a.C_group;

    // this thread's parts of a tile: 8 channels of one token; all of them have the same channels
    static_assert(S::HELP % (CH / 8) == 0, "the parts of a thread have the same channels");
    const int item_t = tid / (CH / 8), item_c = tid % (CH / 8) * 8;
    constexpr int ITEM_STEP = S::HELP / (CH / 8);                        // tokens between two parts of a thread
    const bool has_item = tid < S::ITEMS;
    const int valid = !has_item || item_c >= at.n_channels ? 0 : at.n_channels - item_c < 8 ? (int)(at.n_channels - item_c) : 8;
    const bool vec = FULL;                                               // then valid is 8 or 0
    float skip[8], bias[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        skip[i] = !LOCAL && a.D && i < valid ? a.D[at.channel0 + item_c + i] : 0.0f;
        bias[i] = a.delta_bias && i < valid ? a.delta_bias[at.channel0 + item_c + i] : 0.0f;
    }
    auto slot_of = [&](int slot, int which, int k) {
        return reinterpret_cast<T*>(smem + Mem::raw) + ((slot * 3 + which) * S::ITEMS + tid + k * S::HELP) * 8;
    };
    auto quad_of = [&](int slot, int which, int e) {
        return reinterpret_cast<T*>(smem + Mem::raw_bc) + ((slot * 2 + which) * S::QUADS + e) * 4;
    };
    // `slot` of u, delta, z (kept until the outputs are done), `bc_slot` of B and C (until they are staged)
    auto fetch = [&](int64_t t0, int slot, int bc_slot) {
        if (t0 < t_used) {
#pragma unroll
            for (int k = 0; k < IPT; ++k) {
                const int64_t t = t0 + item_t + k * ITEM_STEP;
                if (valid > 0 && t < t_used) {
                    fetch_pack<T, 8>(slot_of(slot, 0, k), u + t * a.u_token + item_c, vec, valid, d.width);
                    fetch_pack<T, 8>(slot_of(slot, 1, k), delta + t * a.delta_token + item_c, vec, valid, d.width);
                    if (!LOCAL && z) fetch_pack<T, 8>(slot_of(slot, 2, k), z + t * a.z_token + item_c, vec, valid, d.width);
                }
            }
#pragma unroll
            for (int k = 0; k < QPT; ++k) {
                const int e = tid + k * S::HELP, n = e % P * 4;
                const int64_t t = t0 + e / P;
                if (e < S::QUADS && t < t_used && n < states) {
                    const bool wide = FULL || (d.vec_bc && n + 4 <= states);
                    fetch_pack<T, 4>(quad_of(bc_slot, 0, e), B + t * a.B_token + n, wide, states - n, 0);
                    if (!LOCAL) fetch_pack<T, 4>(quad_of(bc_slot, 1, e), C + t * a.C_token + n, wide, states - n, 0);
                }
            }
        }
        copy_commit();
    };
    auto stage = [&](int64_t t0, int slot, int bc_slot, int buf) {
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            const int it = item_t + k * ITEM_STEP;
            if (!has_item) continue;
            float x[8], dt[8];
            read_slot<T, 8>(slot_of(slot, 0, k), x);
            read_slot<T, 8>(slot_of(slot, 1, k), dt);
            float4* const to = reinterpret_cast<float4*>(s_du + (buf * STEPS + it) * S::DU + item_c + item_c / 8 * 2);
            // padding leaves the state as it is: dt = 0 makes the factor 1 and the addend 0
            const bool in = t0 + it < t_used, all = in && valid == 8;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                float e0, e1;
                dt[i] += bias[i];
                dt[i + 1] += bias[i + 1];
                if (d.softplus) softplus_pair(dt[i], dt[i + 1], e0, e1);
                float4 v = make_float4(dt[i], dt[i] * x[i], dt[i + 1], dt[i + 1] * x[i + 1]);
                if (!all) {
                    if (!in || i >= valid) v.x = v.y = 0.0f;
                    if (!in || i + 1 >= valid) v.z = v.w = 0.0f;
                }
                to[i / 2] = v;
            }
        }
#pragma unroll
        for (int k = 0; k < QPT; ++k) {
            const int e = tid + k * S::HELP;
            if (e < S::QUADS) {
                const bool in = t0 + e / P < t_used && e % P * 4 < states;
                float x[4] = {}, y[4] = {};
                if (in) {
                    read_slot<T, 4>(quad_of(bc_slot, 0, e), x);
                    if (!LOCAL) read_slot<T, 4>(quad_of(bc_slot, 1, e), y);
                }
                reinterpret_cast<float4*>(smem + Mem::b)[buf * S::QUADS + e] = make_float4(x[0], x[1], x[2], x[3]);
                if (!LOCAL) reinterpret_cast<float4*>(smem + Mem::c)[buf * S::QUADS + e] = make_float4(y[0], y[1], y[2], y[3]);
            }
        }
    };
    auto finish = [&](int64_t t0, int slot, int buf) {
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            const int it = item_t + k * ITEM_STEP;
            const int64_t t = t0 + it;
            if (valid == 0 || t >= t_end) continue;
            float o[8] = {};
            if (t < t_used) {
                const float4* const y = reinterpret_cast<const float4*>(smem + Mem::y) + ((buf * STEPS + it) * S::ROW + item_c) / 4;
                const float4 y0 = y[0], y1 = y[1];
                o[0] = y0.x, o[1] = y0.y, o[2] = y0.z, o[3] = y0.w, o[4] = y1.x, o[5] = y1.y, o[6] = y1.z, o[7] = y1.w;
                float x[8], g[8];
                read_slot<T, 8>(slot_of(slot, 0, k), x);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = fmaf(skip[i], x[i], o[i]);
                if (z) {
                    read_slot<T, 8>(slot_of(slot, 2, k), g);
#pragma unroll
                    for (int i = 0; i < 8; i += 2)
                        unpack2(mul2(pack2(o[i], o[i + 1]), silu2(pack2(g[i], g[i + 1]))), o[i], o[i + 1]);
                }
            }
            store_pack<T, 8>(out + t * d.channels + item_c, o, vec, valid, d.width);
        }
    };

#pragma unroll
    for (int k = 0; k < S::AHEAD; ++k) fetch(t_begin + k * STEPS, k, k);
    copy_wait<S::AHEAD - 1>();
    if (t_begin < t_used) stage(t_begin, 0, 0, 0);
    __syncthreads();
    int buf = 0, slot = 0, bc_slot = 0;                                  // of the tile that is being scanned
    for (int64_t t0 = t_begin; t0 < t_used; t0 += STEPS, buf ^= 1) {
        const int next = slot == S::AHEAD ? 0 : slot + 1, before = slot == 0 ? S::AHEAD : slot - 1;
        const int bc_next = bc_slot == S::AHEAD - 1 ? 0 : bc_slot + 1;
        if (!LOCAL && t0 > t_begin) finish(t0 - STEPS, before, buf ^ 1);
        fetch(t0 + S::AHEAD * STEPS, before, bc_slot);                   // (B and C of this tile are staged already)
        copy_wait<S::AHEAD - 1>();
        if (t0 + STEPS < t_used) stage(t0 + STEPS, next, bc_next, buf ^ 1);
        slot = next;
        bc_slot = bc_next;
        __syncthreads();
    }
    if (LOCAL) return;
    // the last tile, and the outputs of padding behind it
    int64_t covered = t_begin;
    if (t_used > t_begin) {
        covered += (t_used - t_begin + STEPS - 1) / STEPS * STEPS;
        finish(covered - STEPS, slot == 0 ? S::AHEAD : slot - 1, buf ^ 1);
    }
    if (valid > 0) {
        const float zero[8] = {};
        constexpr int TOKENS = S::ITEMS < S::HELP ? STEPS : ITEM_STEP;   // that the threads cover together
        for (int64_t t = covered + item_t; t < t_end; t += TOKENS)
            store_pack<T, 8>(out + t * d.channels + item_c, zero, vec, valid, d.width);
    }
}

// A length that is cut into segments takes two launches: the first does the first segment and finds out what each of
// those between the first and the last adds to the state (LOCAL: the end of a state that starts at zero, and the sum of
// dt); the second does the other segments, seeded from the segments before.
template <typename T, int P, int M, bool LOCAL, bool FULL>
__device__ __forceinline__ void scan_forward_block(const ScanParams& p, const Place& at, char* smem) {
    const ScanDims& d = p.d;
    const int64_t used = used_length(p.a.lengths, at.batch, d.length);
    const int64_t t_begin = at.segment * d.segment_length;
    const int64_t t_end = t_begin + d.segment_length < d.length ? t_begin + d.segment_length : d.length;
    const int64_t t_used = used < t_end ? used : t_end;                  // tokens of the segment that count
    if (threadIdx.x < ForwardShape<P, M>::SCAN) scan_forward_scan<T, P, M, LOCAL>(p, at, smem, t_begin, t_used);
    else scan_forward_help<T, P, M, LOCAL, FULL>(p, at, smem, t_begin, t_end, t_used);
}

template <typename T, int P, int M, bool FULL>
__global__ void __launch_bounds__(ForwardShape<P, M>::THREADS, 2) scan_forward(const __grid_constant__ ScanParams p) {
    extern __shared__ __align__(16) char smem[];
    const Place at = block_place(p.d, ForwardShape<P, M>::CH);
    if (p.d.ahead && at.segment > 0) scan_forward_block<T, P, M, true, FULL>(p, at, smem);
    else scan_forward_block<T, P, M, false, FULL>(p, at, smem);
}

// ---------------------------------------------------------------------------------------------------------
// backward
//
// The gradient of the state runs from the last token to the first: gh_t = C_t gy_t + a_{t+1} gh_{t+1} with gy = gout
// silu(z).  It meets the states h_t, which are computed again, 16 tokens at a time from the saved state in front of
// them; the 16 states and factors of a lane stay in registers, so every exponential is computed once here too.
//   gC_t = sum_d gy h_t, gB_t = sum_d gh_t dt u     sums over the channels: over the channels of a lane in registers, over
//                                                   the lanes of a warp with reduce_lanes, over the warps in shared
//                                                   memory, over the blocks in a second launch from partial sums (no
//                                                   atomics: the same bits every time)
//   w_t = a_t gh_t (handed to the token before), q = w_t h_{t-1}: gA = sum q dt, g(dt) = sum_n q A + u sum_n gh B,
//   gu = dt sum_n gh B + D gy
// Scanning and helping threads as in the forward kernel.  The scanning threads need 132 registers for the states and
// factors alone, the helping ones few: the block starts with 128 each and hands them over.

// P lanes x K pairs of states x M channels
template <int P, int K, int M>
struct BackShape {
    static constexpr int SCAN = 128, HELP = 128, THREADS = SCAN + HELP;
    static constexpr int WARPS = SCAN / 32;
    static constexpr int CH = SCAN / P * M;
    static constexpr int NP = 2 * K * P;
    static constexpr int STEPS = kCheckpoint;
    static constexpr int V = 8, G = 2;                                   // steps whose C . h, and whose gradients' sums, go together
    static constexpr int CHV = CH / 4;                                   // 4 channels of one token per item
    static constexpr int ITEMS = STEPS * CHV, IPT = (ITEMS + HELP - 1) / HELP;
    static constexpr int QUADS = STEPS * NP / 4, QPT = (QUADS + HELP - 1) / HELP;
    static constexpr int DU = CH + CH / 8 * 2;
    static constexpr int ROW = CH + (P >= 8 ? 4 : 32 / P);
    static constexpr int SLOTS = 3;
    static constexpr int SCAN_REGISTERS = 200, HELP_REGISTERS = 56;      // together 2 x 128
};

template <typename T, int P, int K, int M>
struct BackSmem {
    using S = BackShape<P, K, M>;
    static constexpr size_t du = 0;                                                          // float2 [2][STEPS][DU]
    static constexpr size_t gy = du + 2 * sizeof(float2) * S::STEPS * S::DU;                 // float [2][STEPS][CH]
    static constexpr size_t b = gy + 2 * sizeof(float) * S::STEPS * S::CH;                   // float [2][STEPS][NP]
    static constexpr size_t c = b + 2 * sizeof(float) * S::STEPS * S::NP;
    static constexpr size_t y = c + 2 * sizeof(float) * S::STEPS * S::NP;                    // float [2][STEPS][ROW]: C . h
    static constexpr size_t s = y + 2 * sizeof(float) * S::STEPS * S::ROW;                   // float [2][2][STEPS][ROW]: gh . B, q . A / ln 2
    static constexpr size_t r = s + 4 * sizeof(float) * S::STEPS * S::ROW;                   // float [2][WARPS][STEPS][2][NP]: gC, gB
    static constexpr size_t keep = r + 2 * sizeof(float) * S::WARPS * S::STEPS * 2 * S::NP;  // float4 [2][2][ITEMS]
    static constexpr size_t raw = keep + 4 * sizeof(float4) * S::ITEMS;                      // T [SLOTS][4][ITEMS][4]: u, delta, z, gout
    static constexpr size_t raw_bc = raw + S::SLOTS * 4 * sizeof(T) * S::ITEMS * 4;          // T [2][2][QUADS][4]
    static constexpr size_t bytes = raw_bc + 4 * sizeof(T) * S::QUADS * 4;
};

template <typename T, int P, int K, int M, bool LOCAL>
__device__ __forceinline__ void scan_backward_scan(const ScanParams& p, const Place& at, char* smem, int64_t t_begin, int64_t t_used) {
    using S = BackShape<P, K, M>;
    using Mem = BackSmem<T, P, K, M>;
    constexpr int NP = S::NP, STEPS = S::STEPS, V = S::V, G = S::G, R = 32 / P;
    const OvlSelectiveScan& a = p.a;
    const ScanDims& d = p.d;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, j = lane % P, c0 = tid / P * M, n0 = 2 * K * j;
    const int states = (int)d.states;
    const int64_t chunks = (d.length + kCheckpoint - 1) / kCheckpoint;
    // lanes without a channel have A = h = gh = 0: their sums over channels are zeros
    bool live[M];
    F2 A[M][K], w[M][K], start[M][K];                                    // w: a_{t+1} gh_{t+1}; start: the state in front of a tile
    const float* saved[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        live[m] = c0 + m < at.n_channels;
        const int64_t channel = at.channel0 + (live[m] ? c0 + m : 0);
        saved[m] = a.checkpoints + (at.batch * chunks * d.channels + channel) * states;
#pragma unroll
        for (int k = 0; k < K; ++k) A[m][k] = w[m][k] = start[m][k] = same2(0.0f);
        if (!live[m]) continue;
        load_states(A[m], a.A + channel * states, n0, states, d.vec_states);
#pragma unroll
        for (int k = 0; k < K; ++k) A[m][k] = mul2(A[m][k], same2(kLog2e));
        if (LOCAL) continue;
        if (at.segment < d.segments - 1)
            load_states(w[m], p.seg_state + ((at.batch * d.segments + d.segments - 1) * d.channels + channel) * states, n0, states,
                        d.vec_states);
        else if (a.gfinal)
            load_states(w[m], a.gfinal + (at.batch * d.channels + channel) * states, n0, states, d.vec_states);
        for (int64_t s = d.segments - 2; s > at.segment; --s) {
            const int64_t cell = (at.batch * d.segments + s) * d.channels + channel;
            const F2 sum = same2(p.seg_dt[cell]);
            F2 add[K];
            load_states(add, p.seg_state + cell * states, n0, states, d.vec_states);
#pragma unroll
            for (int k = 0; k < K; ++k) w[m][k] = fma2(decay(A[m][k], sum), w[m][k], add[k]);
        }
    }
    const int64_t first = t_begin, last = t_used > t_begin ? t_begin + (t_used - t_begin - 1) / STEPS * STEPS : t_begin - STEPS;
    auto fetch_start = [&](int64_t t0) {
#pragma unroll
        for (int m = 0; m < M; ++m)
            if (live[m]) load_states(start[m], saved[m] + t0 / kCheckpoint * d.channels * states, n0, states, d.vec_states);
    };
    if (!LOCAL && last >= first) fetch_start(last);
    const float2* const s_du = reinterpret_cast<const float2*>(smem + Mem::du) + c0 + c0 / 8 * 2;
    const float* const s_gy = reinterpret_cast<const float*>(smem + Mem::gy) + c0;
    const float* const s_b = reinterpret_cast<const float*>(smem + Mem::b) + n0;
    const float* const s_c = reinterpret_cast<const float*>(smem + Mem::c) + n0;
    float* const s_y = reinterpret_cast<float*>(smem + Mem::y) + c0;
    float* const s_s = reinterpret_cast<float*>(smem + Mem::s) + c0;
    float* const s_r = reinterpret_cast<float*>(smem + Mem::r) + warp * STEPS * 2 * NP + n0;
    double gA[M][2 * K] = {};
    float sum_dt[M] = {};
    const bool gated = a.z != nullptr;
    __syncthreads();
    int buf = 0;
    for (int64_t t0 = last; t0 >= first; t0 -= STEPS, buf ^= 1) {
        auto read_du = [&](int t, float (&dt)[M], float (&du)[M]) {
            if constexpr (M == 2) {
                const float4 v = *reinterpret_cast<const float4*>(s_du + (buf * STEPS + t) * S::DU);
                dt[0] = v.x, du[0] = v.y, dt[1] = v.z, du[1] = v.w;
            } else {
                const float2 v = s_du[(buf * STEPS + t) * S::DU];
                dt[0] = v.x, du[0] = v.y;
            }
        };
        F2 h[STEPS + 1][M][K], f[STEPS][M][K];                           // h[t]: the state in front of step t; factors
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < K; ++k) h[0][m][k] = start[m][k];
        if (!LOCAL && t0 > first) fetch_start(t0 - STEPS);

        // the states again, forwards
        float y[M][V];
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            float dt[M], du[M];
            F2 b[K], cc[K];
            read_du(t, dt, du);
            if (!LOCAL) {
                read_pairs(b, s_b + (buf * STEPS + t) * NP);
                read_pairs(cc, s_c + (buf * STEPS + t) * NP);
            }
#pragma unroll
            for (int m = 0; m < M; ++m) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    f[t][m][k] = decay(A[m][k], same2(dt[m]));
                    if (!LOCAL) h[t + 1][m][k] = fma2(f[t][m][k], h[t][m][k], mul2(same2(du[m]), b[k]));
                }
                if (LOCAL) sum_dt[m] += dt[m];
                else y[m][t % V] = dot(h[t + 1][m], cc);
            }
            if (!LOCAL && gated && t % V == V - 1) {
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    reduce_lanes<V, P, 1>(y[m], lane);
                    if (reduced_owner<V, P>(j)) {
                        const int tt = buf * STEPS + t - (V - 1) + reduced_index<V, P>(j);
#pragma unroll
                        for (int e = 0; e < reduced_count<V, P>(); ++e) s_y[(tt + e) * S::ROW + m] = y[m][e];
                    }
                }
            }
        }
        // the gradients, backwards
        F2 gA_tile[M][K];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < K; ++k) gA_tile[m][k] = same2(0.0f);
#pragma unroll
        for (int g = STEPS / G - 1; g >= 0; --g) {
            float s[M][2 * G], v[4 * K * G];                             // v: gC, then gB, of the steps one after the other
#pragma unroll
            for (int i = G - 1; i >= 0; --i) {
                const int t = g * G + i;
                float gy[M], dt[M], du[M];
                F2 b[K], cc[K], sum_c[K], sum_b[K];
                if constexpr (M == 2) {
                    const float2 r = *reinterpret_cast<const float2*>(s_gy + (buf * STEPS + t) * S::CH);
                    gy[0] = r.x, gy[1] = r.y;
                } else {
                    gy[0] = s_gy[(buf * STEPS + t) * S::CH];
                }
                read_pairs(cc, s_c + (buf * STEPS + t) * NP);
                if (!LOCAL) {
                    read_du(t, dt, du);
                    read_pairs(b, s_b + (buf * STEPS + t) * NP);
                }
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    F2 gh[K], q[K];
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        gh[k] = fma2(same2(gy[m]), cc[k], w[m][k]);
                        w[m][k] = mul2(f[t][m][k], gh[k]);
                        if (LOCAL) continue;
                        sum_c[k] = m == 0 ? mul2(same2(gy[m]), h[t + 1][m][k]) : fma2(same2(gy[m]), h[t + 1][m][k], sum_c[k]);
                        sum_b[k] = m == 0 ? mul2(same2(du[m]), gh[k]) : fma2(same2(du[m]), gh[k], sum_b[k]);
                        q[k] = mul2(w[m][k], h[t][m][k]);
                        gA_tile[m][k] = fma2(q[k], same2(dt[m]), gA_tile[m][k]);
                    }
                    if (!LOCAL) {
                        s[m][2 * i] = dot(gh, b);
                        s[m][2 * i + 1] = dot(q, A[m]);
                    }
                }
                if (!LOCAL) {
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        unpack2(sum_c[k], v[4 * K * i + 2 * k], v[4 * K * i + 2 * k + 1]);
                        unpack2(sum_b[k], v[4 * K * i + 2 * K + 2 * k], v[4 * K * i + 2 * K + 2 * k + 1]);
                    }
                }
            }
            // The sums of G steps are formed together: the exchanges of a sum wait for one another, those of different
            // sums do not (bf16 8 x 2048 x 2048 x 16: 993 us one step at a time, 875 us two, 917 us four: more registers).
            if (!LOCAL) {
                reduce_lanes<4 * K * G, R, P>(v, lane);
#pragma unroll
                for (int m = 0; m < M; ++m) reduce_lanes<2 * G, P, 1>(s[m], lane);
                if (reduced_owner<4 * K * G, R>(lane / P)) {
                    const int i0 = reduced_index<4 * K * G, R>(lane / P);
                    float* const to = s_r + (buf * S::WARPS * STEPS + g * G) * 2 * NP;
#pragma unroll
                    for (int e = 0; e < reduced_count<4 * K * G, R>(); ++e) {
                        const int at = i0 + e;                           // step, gC or gB, state
                        to[at / (4 * K) * 2 * NP + at / (2 * K) % 2 * NP + at % (2 * K)] = v[e];
                    }
                }
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    if (reduced_owner<2 * G, P>(j)) {
                        const int i0 = reduced_index<2 * G, P>(j);
#pragma unroll
                        for (int e = 0; e < reduced_count<2 * G, P>(); ++e)
                            s_s[((buf * 2 + (i0 + e) % 2) * STEPS + g * G + (i0 + e) / 2) * S::ROW + m] = s[m][e];
                    }
                }
            }
        }
        if (!LOCAL) {
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    float x0, x1;
                    unpack2(gA_tile[m][k], x0, x1);
                    gA[m][2 * k] += x0;
                    gA[m][2 * k + 1] += x1;
                }
        }
        __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
        if (!live[m]) continue;
        const int64_t channel = at.channel0 + c0 + m, cell = (at.batch * d.segments + at.segment) * d.channels + channel;
        if (d.ahead) store_states(p.seg_state + cell * states, w[m], n0, states, d.vec_states);
        if (LOCAL) {
            if (j == 0) p.seg_dt[cell] = sum_dt[m];
            continue;
        }
        F2 sums[K];
#pragma unroll
        for (int k = 0; k < K; ++k) sums[k] = pack2((float)gA[m][2 * k], (float)gA[m][2 * k + 1]);
        store_states(p.part_A + cell * states, sums, n0, states, d.vec_states);
        if (a.ginitial && at.segment == 0)
            store_states(a.ginitial + (at.batch * d.channels + channel) * states, w[m], n0, states, d.vec_states);
    }
}

template <typename T, int P, int K, int M, bool LOCAL, bool FULL>
__device__ __forceinline__ void scan_backward_help(const ScanParams& p, const Place& at, char* smem, int64_t t_begin, int64_t t_end,
                                                   int64_t t_used) {
    using S = BackShape<P, K, M>;
    using Mem = BackSmem<T, P, K, M>;
    constexpr int CH = S::CH, NP = S::NP, STEPS = S::STEPS, IPT = S::IPT, QPT = S::QPT, ITEMS = S::ITEMS;
    const OvlSelectiveScan& a = p.a;
    const ScanDims& d = p.d;
    const int tid = threadIdx.x - S::SCAN;
    const int states = (int)d.states;
    const int64_t first = t_begin, last = t_used > t_begin ? t_begin + (t_used - t_begin - 1) / STEPS * STEPS : t_begin - STEPS;
    const int64_t base_c = at.channel0;
    const T* const u = reinterpret_cast<const T*>(a.u) + at.batch * a.u_batch + base_c;
    const T* const delta = reinterpret_cast<const T*>(a.delta) + at.batch * a.delta_batch + base_c;
    const T* const z = a.z ? reinterpret_cast<const T*>(a.z) + at.batch * a.z_batch + base_c : nullptr;
    const T* const gout = reinterpret_cast<const T*>(a.gout) + at.batch * a.gout_batch + base_c;
    const T* const B = reinterpret_cast<const T*>(a.B) + at.batch * a.B_batch + at.group * a.B_group;
    const T* const C = reinterpret_cast<const T*>(a.C) + at.batch * a.C_batch + at.group * a.C_group;
    float2* const s_du = reinterpret_cast<float2*>(smem + Mem::du);
    float* const s_gy = reinterpret_cast<float*>(smem + Mem::gy);
    float4* const s_keep = reinterpret_cast<float4*>(smem + Mem::keep);  // derivative of dt by delta, of out by z over y

    // this thread's parts of a tile: 4 channels of one token; all of them have the same channels
    static_assert(S::HELP % S::CHV == 0, "the parts of a thread have the same channels");
    constexpr int ITEM_STEP = S::HELP / S::CHV;
    const bool has_item = tid < ITEMS;
    const int item_t = tid / S::CHV, cc = tid % S::CHV * 4;
    const int valid = !has_item || cc >= at.n_channels ? 0 : at.n_channels - cc < 4 ? (int)(at.n_channels - cc) : 4;
    const bool vec = FULL;                                               // then valid is 4 or 0
    float bias[4], skip[4], gD[4] = {}, gbias[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bias[i] = a.delta_bias && i < valid ? a.delta_bias[base_c + cc + i] : 0.0f;
        skip[i] = a.D && i < valid ? a.D[base_c + cc + i] : 0.0f;
    }
    auto slot_of = [&](int slot, int which, int k) {
        return reinterpret_cast<T*>(smem + Mem::raw) + ((slot * 4 + which) * ITEMS + tid + k * S::HELP) * 4;
    };
    auto quad_of = [&](int slot, int which, int e) {
        return reinterpret_cast<T*>(smem + Mem::raw_bc) + ((slot * 2 + which) * S::QUADS + e) * 4;
    };
    auto fetch = [&](int64_t t0, int slot, int bc_slot) {
        if (t0 >= first) {
#pragma unroll
            for (int k = 0; k < IPT; ++k) {
                const int64_t t = t0 + item_t + k * ITEM_STEP;
                if (valid > 0 && t < t_used) {
                    if (!LOCAL) fetch_pack<T, 4>(slot_of(slot, 0, k), u + t * a.u_token + cc, vec, valid, d.width);
                    fetch_pack<T, 4>(slot_of(slot, 1, k), delta + t * a.delta_token + cc, vec, valid, d.width);
                    if (z) fetch_pack<T, 4>(slot_of(slot, 2, k), z + t * a.z_token + cc, vec, valid, d.width);
                    fetch_pack<T, 4>(slot_of(slot, 3, k), gout + t * a.gout_token + cc, vec, valid, d.width);
                }
            }
#pragma unroll
            for (int k = 0; k < QPT; ++k) {
                const int e = tid + k * S::HELP, n = e % (NP / 4) * 4;
                const int64_t t = t0 + e / (NP / 4);
                if (e < S::QUADS && t < t_used && n < states) {
                    const bool wide = FULL || (d.vec_bc && n + 4 <= states);
                    if (!LOCAL) fetch_pack<T, 4>(quad_of(bc_slot, 0, e), B + t * a.B_token + n, wide, states - n, 0);
                    fetch_pack<T, 4>(quad_of(bc_slot, 1, e), C + t * a.C_token + n, wide, states - n, 0);
                }
            }
        }
        copy_commit();
    };
    auto stage = [&](int64_t t0, int slot, int buf) {
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            const int it = item_t + k * ITEM_STEP;
            if (!has_item) continue;
            const bool in = t0 + it < t_used;
            float x[4] = {}, dt[4] = {}, zz[4], g[4] = {}, slope[4], gate_slope[4] = {};
            if (in && valid > 0) {
                if (!LOCAL) read_slot<T, 4>(slot_of(slot, 0, k), x);
                read_slot<T, 4>(slot_of(slot, 1, k), dt);
                read_slot<T, 4>(slot_of(slot, 3, k), g);
            }
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                dt[i] += bias[i];
                dt[i + 1] += bias[i + 1];
                slope[i] = slope[i + 1] = 1.0f;
                if (d.softplus) {
                    const float x0 = dt[i], x1 = dt[i + 1];
                    float e0, e1;
                    softplus_pair(dt[i], dt[i + 1], e0, e1);
                    // the derivative 1 / (1 + e^-x) from e = e^-|x|
                    const float r0 = rcp_approx(1.0f + e0), r1 = rcp_approx(1.0f + e1);
                    slope[i] = x0 < 0.0f ? e0 * r0 : r0;
                    slope[i + 1] = x1 < 0.0f ? e1 * r1 : r1;
                }
            }
            if (z && in && valid > 0) {
                read_slot<T, 4>(slot_of(slot, 2, k), zz);
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const F2 zi = pack2(zz[i], zz[i + 1]), gi = pack2(g[i], g[i + 1]), sig = sigmoid2(zi), gate = mul2(zi, sig);
                    unpack2(mul2(gi, fma2(gate, fma2(sig, same2(-1.0f), same2(1.0f)), sig)), gate_slope[i], gate_slope[i + 1]);
                    unpack2(mul2(gi, gate), g[i], g[i + 1]);
                }
            }
            // padding: dt = 0 hands the gradient on as it is, gy = dt u = 0 adds nothing
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!in || i >= valid) dt[i] = g[i] = x[i] = 0.0f;
                x[i] = in && i < valid ? dt[i] * x[i] : 0.0f;
            }
            float4* const to = reinterpret_cast<float4*>(s_du + (buf * STEPS + it) * S::DU + cc + cc / 8 * 2);
            to[0] = make_float4(dt[0], x[0], dt[1], x[1]);
            to[1] = make_float4(dt[2], x[2], dt[3], x[3]);
            *reinterpret_cast<float4*>(s_gy + (buf * STEPS + it) * CH + cc) = make_float4(g[0], g[1], g[2], g[3]);
            if (!LOCAL) {
                s_keep[(buf * 2) * ITEMS + tid + k * S::HELP] = make_float4(slope[0], slope[1], slope[2], slope[3]);
                s_keep[(buf * 2 + 1) * ITEMS + tid + k * S::HELP] = make_float4(gate_slope[0], gate_slope[1], gate_slope[2], gate_slope[3]);
            }
        }
#pragma unroll
        for (int k = 0; k < QPT; ++k) {
            const int e = tid + k * S::HELP;
            if (e < S::QUADS) {
                float x[4] = {}, y[4] = {};
                if (t0 + e / (NP / 4) < t_used && e % (NP / 4) * 4 < states) {
                    if (!LOCAL) read_slot<T, 4>(quad_of(buf, 0, e), x);
                    read_slot<T, 4>(quad_of(buf, 1, e), y);
                }
                if (!LOCAL) reinterpret_cast<float4*>(smem + Mem::b)[buf * S::QUADS + e] = make_float4(x[0], x[1], x[2], x[3]);
                reinterpret_cast<float4*>(smem + Mem::c)[buf * S::QUADS + e] = make_float4(y[0], y[1], y[2], y[3]);
            }
        }
    };
    auto finish = [&](int64_t t0, int slot, int buf) {
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            const int it = item_t + k * ITEM_STEP;
            const int64_t t = t0 + it;
            if (valid == 0 || t >= t_end) continue;
            float gu[4] = {}, gd[4] = {}, gz[4] = {};
            if (t < t_used) {
                float x[4], over[4], qa[4], slope[4], gs[4], y[4] = {}, gy[4], dt[4];
                auto four = [](float (&v)[4], const float* from) {
                    const float4 r = *reinterpret_cast<const float4*>(from);
                    v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w;
                };
                read_slot<T, 4>(slot_of(slot, 0, k), x);
                four(over, reinterpret_cast<const float*>(smem + Mem::s) + ((buf * 2) * STEPS + it) * S::ROW + cc);
                four(qa, reinterpret_cast<const float*>(smem + Mem::s) + ((buf * 2 + 1) * STEPS + it) * S::ROW + cc);
                four(slope, reinterpret_cast<const float*>(s_keep + (buf * 2) * ITEMS + tid + k * S::HELP));
                four(gs, reinterpret_cast<const float*>(s_keep + (buf * 2 + 1) * ITEMS + tid + k * S::HELP));
                four(gy, s_gy + (buf * STEPS + it) * CH + cc);
                if (z) four(y, reinterpret_cast<const float*>(smem + Mem::y) + (buf * STEPS + it) * S::ROW + cc);
                const float4* const du = reinterpret_cast<const float4*>(s_du + (buf * STEPS + it) * S::DU + cc + cc / 8 * 2);
                dt[0] = du[0].x, dt[1] = du[0].z, dt[2] = du[1].x, dt[3] = du[1].z;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    gu[i] = fmaf(dt[i], over[i], skip[i] * gy[i]);
                    gd[i] = slope[i] * fmaf(x[i], over[i], kLn2 * qa[i]);
                    gz[i] = gs[i] * fmaf(skip[i], x[i], y[i]);
                    gD[i] = fmaf(gy[i], x[i], gD[i]);
                    gbias[i] += gd[i];
                }
            }
            const int64_t o = (at.batch * d.length + t) * d.channels + base_c + cc;
            store_pack<T, 4>(reinterpret_cast<T*>(a.gu) + o, gu, vec, valid, d.width);
            store_pack<T, 4>(reinterpret_cast<T*>(a.gdelta) + o, gd, vec, valid, d.width);
            if (a.gz) store_pack<T, 4>(reinterpret_cast<T*>(a.gz) + o, gz, vec, valid, d.width);
        }
        float4* const part = reinterpret_cast<float4*>(
            p.part_bc + (((at.batch * d.groups + at.group) * d.tiles + at.tile) * d.length + t0) * 2 * NP);
        const float4* const from = reinterpret_cast<const float4*>(smem + Mem::r) + buf * S::WARPS * STEPS * NP / 2;
#pragma unroll
        for (int e = tid; e < STEPS * NP / 2; e += S::HELP) {
            float4 sum = from[e];
#pragma unroll
            for (int w = 1; w < S::WARPS; ++w) {
                const float4 v = from[w * STEPS * NP / 2 + e];
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
            if (t0 + e / (NP / 2) < t_used) part[e] = sum;
        }
    };

    fetch(last, 0, 0);
    fetch(last - STEPS, 1, 1);
    copy_wait<1>();
    if (last >= first) stage(last, 0, 0);
    __syncthreads();
    int buf = 0, slot = 0;
    for (int64_t t0 = last; t0 >= first; t0 -= STEPS, buf ^= 1) {
        const int next = slot == 2 ? 0 : slot + 1, before = slot == 0 ? 2 : slot - 1;
        if (!LOCAL && t0 < last) finish(t0 + STEPS, before, buf ^ 1);
        fetch(t0 - 2 * STEPS, before, buf);                              // (B and C of this tile are staged already)
        copy_wait<1>();
        if (t0 - STEPS >= first) stage(t0 - STEPS, next, buf ^ 1);
        slot = next;
        __syncthreads();
    }
    if (LOCAL) return;
    if (last >= first) finish(first, slot == 0 ? 2 : slot - 1, buf ^ 1);
    // gradients of padding behind the last tile
    for (int64_t t0 = last + STEPS; t0 < t_end; t0 += STEPS) {
        const float zero[4] = {};
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            const int64_t t = t0 + item_t + k * ITEM_STEP;
            if (valid > 0 && t < t_end) {
                const int64_t o = (at.batch * d.length + t) * d.channels + base_c + cc;
                store_pack<T, 4>(reinterpret_cast<T*>(a.gu) + o, zero, vec, valid, d.width);
                store_pack<T, 4>(reinterpret_cast<T*>(a.gdelta) + o, zero, vec, valid, d.width);
                if (a.gz) store_pack<T, 4>(reinterpret_cast<T*>(a.gz) + o, zero, vec, valid, d.width);
            }
        }
    }
    // gD and gdelta_bias: sums over the thread's tokens; over the threads in shared memory, in thread order.  Only the
    // helping threads are still here, so they wait for one another alone.
    float* const sums = reinterpret_cast<float*>(smem + Mem::keep);      // [2][threads of a row][CH]
    constexpr int ROWS = ITEMS < S::HELP ? STEPS : ITEM_STEP;
    asm volatile("bar.sync 1, %0;" ::"n"(S::HELP) : "memory");
    if (has_item) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sums[item_t * CH + cc + i] = gD[i];
            sums[(ROWS + item_t) * CH + cc + i] = gbias[i];
        }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(S::HELP) : "memory");
    const int64_t part_row = at.batch * d.segments + at.segment;
    for (int e = tid; e < 2 * CH; e += S::HELP) {
        const int which = e / CH, ch = e % CH;
        if (ch >= at.n_channels) continue;
        float sum = 0.0f;
        for (int t = 0; t < ROWS; ++t) sum += sums[(which * ROWS + t) * CH + ch];
        p.part_D[(part_row * 2 + which) * d.channels + base_c + ch] = sum;
    }
}

template <typename T, int P, int K, int M, bool LOCAL, bool FULL>
__device__ __forceinline__ void scan_backward_block(const ScanParams& p, const Place& at, char* smem) {
    using S = BackShape<P, K, M>;
    const ScanDims& d = p.d;
    const int64_t used = used_length(p.a.lengths, at.batch, d.length);
    const int64_t t_begin = at.segment * d.segment_length;
    const int64_t t_end = t_begin + d.segment_length < d.length ? t_begin + d.segment_length : d.length;
    const int64_t t_used = used < t_end ? used : t_end;
    if (threadIdx.x < S::SCAN) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::SCAN_REGISTERS));
        scan_backward_scan<T, P, K, M, LOCAL>(p, at, smem, t_begin, t_used);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::HELP_REGISTERS));
        scan_backward_help<T, P, K, M, LOCAL, FULL>(p, at, smem, t_begin, t_end, t_used);
    }
}

// the segments from last to first, in two launches like the forward ones
template <typename T, int P, int K, int M, bool FULL>
__global__ void __launch_bounds__(BackShape<P, K, M>::THREADS, 2) scan_backward(const __grid_constant__ ScanParams p) {
    extern __shared__ __align__(16) char smem[];
    const Place at = block_place(p.d, BackShape<P, K, M>::CH);
    if (p.d.ahead && at.segment < p.d.segments - 1) scan_backward_block<T, P, K, M, true, FULL>(p, at, smem);
    else scan_backward_block<T, P, K, M, false, FULL>(p, at, smem);
}

// gB and gC: the channel tiles' parts added up, 4 values per thread; a block's 4 slices of the tiles each in order, then the
// slices, then the sum over the tiles of the launches before.  The parts of a (batch, group) and tile are one piece of
// memory, [length][2][NP].
template <typename T, int NP>
__global__ void __launch_bounds__(256) scan_backward_bc(const __grid_constant__ ScanParams p) {
    __shared__ float4 s_sum[3][64];
    const ScanDims& d = p.d;
    const int lane = threadIdx.x % 64, slice = threadIdx.x / 64;
    const int64_t quads = d.length * NP / 2, blocks = (quads + 63) / 64;
    const int64_t bg = blockIdx.x / blocks, q = blockIdx.x % blocks * 64 + lane;
    const int64_t t = q / (NP / 2), b = bg / d.groups, g = bg % d.groups;
    const bool in = q < quads && t < used_length(p.a.lengths, b, d.length);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (in) {
        const float4* const src = reinterpret_cast<const float4*>(p.part_bc) + bg * d.tiles * quads + q;
#pragma unroll 8
        for (int64_t tile = slice; tile < d.tiles; tile += 4) {
            const float4 v = src[tile * quads];
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
    }
    if (slice > 0) s_sum[slice - 1][lane] = sum;
    __syncthreads();
    if (slice > 0 || q >= quads) return;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const float4 v = s_sum[k][lane];
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    if (d.tiles < d.all_tiles && in) {
        float4* const before = reinterpret_cast<float4*>(p.sum_bc) + bg * quads + q;
        if (d.first_tile > 0) {
            const float4 v = *before;
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        *before = sum;
    }
    if (d.first_tile + d.tiles < d.all_tiles) return;
    const int part = (int)(q % (NP / 2)), n0 = part % (NP / 4) * 4;
    T* const to = reinterpret_cast<T*>(part < NP / 4 ? p.a.gC : p.a.gB) + ((b * d.length + t) * d.groups + g) * d.states;
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (n0 + k < d.states) to[n0 + k] = from_f32<T>(v[k]);
}

// gA, gD, gdelta_bias: the parts of batches and segments added up in order, by slices (see sum_slices) of one block
__global__ void __launch_bounds__(kSumThreads) scan_backward_params(const __grid_constant__ ScanParams p, int slices) {
    __shared__ double s_part[kSumThreads];
    const ScanDims& d = p.d;
    const int values = kSumThreads / slices, v = threadIdx.x % values, slice = threadIdx.x / values;
    const int64_t rows = p.a.batch * d.segments, n_A = d.channels * d.states, total = n_A + 2 * d.channels;
    const int64_t i = (int64_t)blockIdx.x * values + v;
    const bool in_A = i < n_A;
    const int64_t k = in_A ? i : i - n_A, stride = in_A ? n_A : 2 * d.channels;
    double sum = 0.0;
    if (i < total) {
        const float* const src = (in_A ? p.part_A : p.part_D) + k;
#pragma unroll 8
        for (int64_t r = slice; r < rows; r += slices) sum += src[r * stride];
    }
    s_part[threadIdx.x] = sum;
    __syncthreads();
    if (slice != 0 || i >= total) return;
    for (int s = 1; s < slices; ++s) sum += s_part[s * values + v];
    float* const to = in_A ? p.a.gA : k < d.channels ? p.a.gD : p.a.gdelta_bias;
    if (to) to[in_A || k < d.channels ? k : k - d.channels] = (float)sum;
}

// ---------------------------------------------------------------------------------------------------------
// one token

// A thread has 4 states of a channel for ROWS rows, all of whose loads are under way before the first is used; A is loaded
// once for all rows.  What is needed once per (row, channel) - softplus, the gate, the output - is shared out among the
// channel's lanes, a row (or more) each.  What bounds it: bytes, the states in and out.
// rows of a block, if that leaves enough blocks (256 rows x 4096 channels x 16 states: 31 us, 50 with a row for each block,
// which loads A 256 times)
constexpr int kStepRows = 4;

// The slot of a row: -1 for padding, -2 for one that does not exist or that an earlier row has.  All threads of the block
// call it.
__device__ __forceinline__ int64_t slot_of(const int32_t* slot_of_row, int64_t slots, int64_t row) {
    if (!slot_of_row) return row;
    const int slot = slot_of_row[row];
    int taken = 0;
    for (int r = threadIdx.x; r < row; r += blockDim.x) taken |= slot >= 0 && slot_of_row[r] == slot;
    taken = __syncthreads_or(taken);
    return slot < 0 ? -1 : slot >= slots || taken ? -2 : slot;
}

// EXACT: 4 P states, rows of A, B, C and the states on boundaries of 4 elements: no load depends on a condition.
template <typename T, int P, int ROWS, bool EXACT>
__global__ void __launch_bounds__(128) scan_step(const __grid_constant__ OvlSelectiveScanStep a, int tiles) {
    constexpr int OWN = reduced_count<ROWS, P>();                        // rows of a lane
    const int tile = blockIdx.x % tiles, tid = threadIdx.x, lane = tid % 32, j = lane % P, n0 = 4 * j;
    const int64_t row0 = (int64_t)(blockIdx.x / tiles) * ROWS;
    const int channel_at = tile * (128 / P) + tid / P, channels = (int)a.channels, states = EXACT ? 4 * P : (int)a.states;
    const bool live = channel_at < channels;
    const int channel = live ? channel_at : channels - 1;
    const int group = channel / (channels / (int)a.groups);
    const int own = reduced_index<ROWS, P>(j);
    int64_t slot[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) slot[r] = row0 + r < a.rows ? slot_of(a.slot_of_row, a.slots, row0 + r) : -3;
    float o[ROWS];
    float x[OWN];
    T z[OWN];
    if (a.slots > 0) {
        F2 A[2], h[ROWS][2];
        Pack<T, 4> b[ROWS], c[ROWS];
        // (a row without a state reads the first one's, and leaves it alone; behind the last row it is read again)
        const int64_t last = a.rows - 1;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int64_t from = slot[r] < 0 ? 0 : slot[r], row = row0 + r < last ? row0 + r : last;
            load_states(h[r], a.state + (from * channels + channel) * states, n0, states, EXACT);
            b[r] = load_pack<T, 4>(reinterpret_cast<const T*>(a.B) + row * a.B_row + group * a.B_group + n0, EXACT, states - n0);
            c[r] = load_pack<T, 4>(reinterpret_cast<const T*>(a.C) + row * a.C_row + group * a.C_group + n0, EXACT, states - n0);
        }
        float dt[OWN], du[OWN];
        T raw_u[OWN], raw_dt[OWN];
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int64_t row = row0 + own + k < last ? row0 + own + k : last;
            raw_u[k] = reinterpret_cast<const T*>(a.u)[row * a.u_row + channel];
            raw_dt[k] = reinterpret_cast<const T*>(a.delta)[row * a.delta_row + channel];
            if (a.z) z[k] = reinterpret_cast<const T*>(a.z)[row * a.z_row + channel];
        }
        load_states(A, a.A + (int64_t)channel * states, n0, states, EXACT);
        const float bias = a.delta_bias ? a.delta_bias[channel] : 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k) A[k] = mul2(A[k], same2(kLog2e));
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            x[k] = to_f32(raw_u[k]);
            dt[k] = to_f32(raw_dt[k]) + bias;
            if (a.delta_softplus) dt[k] = softplus(dt[k]);
            du[k] = dt[k] * x[k];
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float step = dt[r % OWN], add = du[r % OWN];
            if (ROWS > 1 && P > 1) {                                     // from the lane that has the row
                const int source = (lane & ~(P - 1)) + (P >= ROWS ? r * (P / ROWS) : r / OWN);
                step = __shfl_sync(0xffffffffu, step, source);
                add = __shfl_sync(0xffffffffu, add, source);
            }
            const F2 bb[2] = {pack2(to_f32(b[r].v[0]), to_f32(b[r].v[1])), pack2(to_f32(b[r].v[2]), to_f32(b[r].v[3]))};
            const F2 cc[2] = {pack2(to_f32(c[r].v[0]), to_f32(c[r].v[1])), pack2(to_f32(c[r].v[2]), to_f32(c[r].v[3]))};
#pragma unroll
            for (int k = 0; k < 2; ++k) h[r][k] = fma2(decay(A[k], same2(step)), h[r][k], mul2(same2(add), bb[k]));
            o[r] = dot(h[r], cc);
            if (live && slot[r] >= 0) store_states(a.state + (slot[r] * channels + channel) * states, h[r], n0, states, EXACT);
        }
        reduce_lanes<ROWS, P, 1>(o, lane);
    }
    if (!live || !reduced_owner<ROWS, P>(j)) return;
    const float skip = a.D ? a.D[channel] : 0.0f;
#pragma unroll
    for (int k = 0; k < OWN; ++k) {
        int64_t at = slot[k];                                            // of row own + k; slots are indexed by registers
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            if (r == own + k) at = slot[r];
        if (at == -3) continue;
        float y = at == -1 ? 0.0f : __int_as_float(0x7fffffff);
        if (at >= 0) {
            y = fmaf(skip, x[k], o[k]);
            if (a.z) y *= silu(to_f32(z[k]));
        }
        reinterpret_cast<T*>(a.out)[(row0 + own + k) * channels + channel] = from_f32<T>(y);
    }
}

// ---------------------------------------------------------------------------------------------------------
// launches

// One launch, or the two of a length that is cut into segments.
template <typename F>
int launch_segments(F kernel, ScanParams p, int threads, size_t smem, bool backward, cudaStream_t stream, int registers = 0) {
    int st = prepare_kernel((const void*)kernel, smem, threads, registers);
    if (st != OVL_OK) return st;
    const int64_t n = p.d.segments, blocks = p.a.batch * p.d.groups * p.d.tiles;
    for (int launch = n > 1 ? 0 : 1; launch < 2; ++launch) {
        p.d.ahead = launch == 0;
        p.d.launch_segments = n > 1 ? n - 1 : 1;
        p.d.first_segment = n > 1 && p.d.ahead == (backward ? 1 : 0) ? 1 : 0;
        kernel<<<(uint32_t)(blocks * p.d.launch_segments), threads, smem, stream>>>(p);
        if ((st = launch_status()) != OVL_OK) return st;
    }
    return OVL_OK;
}

template <typename T, int P, int M>
int run_forward(const ScanParams& p, cudaStream_t stream) {
    constexpr int threads = ForwardShape<P, M>::THREADS;
    constexpr size_t smem = ForwardSmem<T, P, M>::bytes;
    if (p.d.vec && p.d.vec_bc) return launch_segments(scan_forward<T, P, M, true>, p, threads, smem, false, stream);
    return launch_segments(scan_forward<T, P, M, false>, p, threads, smem, false, stream);
}

template <typename T, int P, int K, int M>
int run_backward(ScanParams p, cudaStream_t stream) {
    using S = BackShape<P, K, M>;
    // the scanning threads' registers come out of those that the block starts with: what all threads hold then
    constexpr int registers = S::SCAN * S::SCAN_REGISTERS + S::HELP * S::HELP_REGISTERS;
    constexpr size_t smem = BackSmem<T, P, K, M>::bytes;
    const int64_t bc_blocks = ceil_div(p.d.length * S::NP / 2, 64) * p.a.batch * p.d.groups;
    if (bc_blocks > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    const int64_t most = p.d.tiles;                                      // of one launch: what the work space has room for
    for (int64_t& first = p.d.first_tile; first < p.d.all_tiles; first += most) {
        p.d.tiles = p.d.all_tiles - first < most ? p.d.all_tiles - first : most;
        int st = p.d.vec && p.d.vec_bc ? launch_segments(scan_backward<T, P, K, M, true>, p, S::THREADS, smem, true, stream, registers)
                                       : launch_segments(scan_backward<T, P, K, M, false>, p, S::THREADS, smem, true, stream, registers);
        if (st != OVL_OK) return st;
        if (bc_blocks == 0) continue;
        scan_backward_bc<T, S::NP><<<(uint32_t)bc_blocks, 256, 0, stream>>>(p);
        if ((st = launch_status()) != OVL_OK) return st;
    }
    const int slices = sum_slices(p.a.batch * p.d.segments);
    const int64_t sums = ceil_div(p.d.channels * (p.d.states + 2), kSumThreads / slices);
    if (sums > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    scan_backward_params<<<(uint32_t)sums, kSumThreads, 0, stream>>>(p, slices);
    return launch_status();
}

template <typename T>
int scan_dispatch(const ScanParams& p, const ScanShape& s, bool backward, cudaStream_t stream) {
    if (backward) {
#define OVL_SCAN_CASE(P, K, M) \
    if (s.lanes == P && s.pairs == K) return run_backward<T, P, K, M>(p, stream);
        OVL_SCAN_CASE(4, 1, 2)
        OVL_SCAN_CASE(8, 1, 2)
        OVL_SCAN_CASE(16, 1, 2)
        OVL_SCAN_CASE(32, 1, 2)
        OVL_SCAN_CASE(32, 2, 1)
#undef OVL_SCAN_CASE
        return OVL_ERR_INVALID;
    }
#define OVL_SCAN_CASE(P, M) \
    if (s.lanes == P && s.channels == M) return run_forward<T, P, M>(p, stream);
    OVL_SCAN_CASE(1, 1)
    OVL_SCAN_CASE(2, 1)
    OVL_SCAN_CASE(4, 1)
    OVL_SCAN_CASE(8, 1)
    OVL_SCAN_CASE(16, 1)
    OVL_SCAN_CASE(1, 2)
    OVL_SCAN_CASE(2, 2)
    OVL_SCAN_CASE(4, 2)
    OVL_SCAN_CASE(8, 2)
    OVL_SCAN_CASE(16, 2)
    OVL_SCAN_CASE(32, 2)
#undef OVL_SCAN_CASE
    return OVL_ERR_INVALID;
}

template <typename T, int P, int ROWS>
int run_step_rows(const OvlSelectiveScanStep& a, int64_t tiles, cudaStream_t stream) {
    const int64_t blocks = tiles * ceil_div(a.rows, ROWS);
    if (blocks > 0x7fffffff || a.channels > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    const bool exact = a.states == 4 * P && aligned16(a.A) && aligned16(a.state) && aligned16(a.B) && aligned16(a.C) &&
                       a.B_row % 4 == 0 && a.C_row % 4 == 0 && a.B_group % 4 == 0 && a.C_group % 4 == 0;
    if (exact) scan_step<T, P, ROWS, true><<<(uint32_t)blocks, 128, 0, stream>>>(a, (int)tiles);
    else scan_step<T, P, ROWS, false><<<(uint32_t)blocks, 128, 0, stream>>>(a, (int)tiles);
    return launch_status();
}

template <typename T, int P>
int run_step(const OvlSelectiveScanStep& a, cudaStream_t stream) {
    const int64_t tiles = ceil_div(a.channels, 128 / P);
    if (tiles * ceil_div(a.rows, kStepRows) >= 8 * (int64_t)sequence_sm_count()) return run_step_rows<T, P, kStepRows>(a, tiles, stream);
    return run_step_rows<T, P, 1>(a, tiles, stream);
}

template <typename T>
int scan_step_dispatch(const OvlSelectiveScanStep& a, int lanes, cudaStream_t stream) {
    switch (lanes) {
        case 1: return run_step<T, 1>(a, stream);
        case 2: return run_step<T, 2>(a, stream);
        case 4: return run_step<T, 4>(a, stream);
        case 8: return run_step<T, 8>(a, stream);
        case 16: return run_step<T, 16>(a, stream);
        default: return run_step<T, 32>(a, stream);
    }
}

}  // namespace
}  // namespace ovl
