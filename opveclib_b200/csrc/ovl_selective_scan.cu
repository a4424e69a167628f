// Selective scan: h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t, out_t = (C_t . h_t + D u_t) silu(z_t), for prompts and
// training (forward and backward) and for single tokens.  Interface: include/ovl_b200.h.
//
// What bounds it.  A (token, channel) moves 8 bytes (u, delta, z, out in 16 bits) and needs one exponential per state.
// The special-function unit delivers 16 per clock and SM: with 16 states one (token, channel) per clock and SM, 2.8e11
// per second on 148 SMs, while 8 bytes at the measured copy bandwidth allow 8e11.  So the recurrence itself has to stay
// out of the way of the exponentials: it runs serially over the tokens in registers (no scan over lanes, which would
// multiply the arithmetic), and everything that is needed once per (token, channel) is computed once, in shared memory.
//
// Layout.  A channel is P lanes of a warp with 4 states each (P = 1 ... 32: up to 128 states); a block is 128 threads
// (256 for P = 32) = CH channels of one group of one batch.  Tokens come in tiles of STEPS: while a tile is scanned the
// next one's elements are in flight to registers; they are converted, masked and combined (softplus, dt * u) into
// shared memory, double-buffered, with one barrier per tile.  The sums over the states of P steps are formed together
// (reduce_lanes: less than one exchange per step), and the same threads that loaded u and z finish the outputs.
#include "ovl_sequence.cuh"

namespace ovl {
namespace {

constexpr int kCheckpoint = 16;        // tokens between two saved states of a training step
constexpr int kMaxStates = 128;
constexpr int kMaxSegments = 32;

struct ScanDims {
    int64_t length, channels, states, groups;
    int64_t group_channels, tiles;     // channels of a group, channel tiles of a group
    int64_t segments, segment_length;  // the length cut into segments (a multiple of 32) that run side by side
    int32_t softplus, vec;             // vec: wide loads and stores of channel vectors
    int32_t vec_states;                // wide loads and stores of 4 states
};

struct ScanParams {
    ScanDims d;
    OvlSelectiveScan a;
    float* seg_state;                  // [batch, segments, channels, states]: what a segment adds to the state
    float* seg_dt;                     // [batch, segments, channels]: sum of dt over the segment
    float* part_bc;                    // [batch, groups, tiles, length, 2, 4P]: gC and gB of a channel tile
    float* part_A;                     // [batch * segments, channels, states]
    float* part_D;                     // [batch * segments, 2, channels]: gD, gdelta_bias
};

template <int P>
struct Shape {
    static constexpr int THREADS = P == 32 ? 256 : 128;
    static constexpr int CH = THREADS / P;                               // channels of a block
    static constexpr int NP = 4 * P;                                     // states, padded
    static constexpr int STEPS = P == 1 ? 8 : P == 2 ? 16 : 32;          // tokens of a forward tile
    static constexpr int ROW = CH + (P >= 8 ? 4 : 32 / P);               // row of per-channel sums in shared memory:
                                                                         // lanes of different steps hit different banks
};

__device__ __forceinline__ float4 load_states(const float* p, int n0, int states, bool vec) {
    if (vec && n0 < states) return *reinterpret_cast<const float4*>(p + n0);
    float4 r;
    r.x = n0 < states ? p[n0] : 0.0f;
    r.y = n0 + 1 < states ? p[n0 + 1] : 0.0f;
    r.z = n0 + 2 < states ? p[n0 + 2] : 0.0f;
    r.w = n0 + 3 < states ? p[n0 + 3] : 0.0f;
    return r;
}
__device__ __forceinline__ void store_states(float* p, float4 x, int n0, int states, bool vec) {
    if (vec && n0 < states) {
        *reinterpret_cast<float4*>(p + n0) = x;
        return;
    }
    if (n0 < states) p[n0] = x.x;
    if (n0 + 1 < states) p[n0 + 1] = x.y;
    if (n0 + 2 < states) p[n0 + 2] = x.z;
    if (n0 + 3 < states) p[n0 + 3] = x.w;
}

__device__ __forceinline__ int64_t used_length(const int32_t* lengths, int64_t batch, int64_t length) {
    if (!lengths) return length;
    const int64_t n = lengths[batch];
    return n < 0 ? 0 : n > length ? length : n;
}

// which piece of the problem a block works on
struct Place {
    int64_t batch, segment, group, tile, channel0, n_channels;   // channels channel0 ... channel0 + n_channels - 1
};
__device__ __forceinline__ Place block_place(const ScanDims& d, int ch) {
    Place p;
    int64_t i = blockIdx.x;
    p.tile = i % d.tiles;
    i /= d.tiles;
    p.group = i % d.groups;
    i /= d.groups;
    p.segment = i % d.segments;
    p.batch = i / d.segments;
    p.channel0 = p.group * d.group_channels + p.tile * ch;
    const int64_t left = d.group_channels - p.tile * ch;
    p.n_channels = left < ch ? left : ch;
    return p;
}

// ---------------------------------------------------------------------------------------------------------
// forward

// LOCAL: only what a segment adds to a state that starts at zero, and its sum of dt (the first of two passes when the
// length is cut into segments); otherwise the whole operator, seeded from the segments before.
template <typename T, int P, bool LOCAL>
__global__ void __launch_bounds__(Shape<P>::THREADS) scan_forward(const __grid_constant__ ScanParams p) {
    using S = Shape<P>;
    constexpr int THREADS = S::THREADS, CH = S::CH, NP = S::NP, STEPS = S::STEPS, ROW = S::ROW;
    constexpr int CHV = CH / 8, ITEMS = STEPS * CHV;                     // 8 channels of one token
    constexpr int BCN = (STEPS * NP + THREADS - 1) / THREADS;
    constexpr int V = P < 16 ? P : 16;                                   // steps whose sums are formed together
    static_assert(ITEMS <= THREADS && STEPS % V == 0 && kCheckpoint % V == 0, "tile shape");
    extern __shared__ __align__(16) float smem[];
    float2* const s_du = reinterpret_cast<float2*>(smem);                // [2][STEPS][CH] (dt, dt * u)
    float* const s_b = smem + 2 * STEPS * CH * 2;                        // [2][STEPS][NP]
    float* const s_c = s_b + 2 * STEPS * NP;                             // [2][STEPS][NP]
    float* const s_y = s_c + 2 * STEPS * NP;                             // [2][STEPS][ROW]

    const OvlSelectiveScan& a = p.a;
    const ScanDims& d = p.d;
    const Place at = block_place(d, CH);
    const int tid = threadIdx.x, lane = tid % 32, j = lane % P, c = tid / P;
    const bool live = c < at.n_channels;
    const int64_t channel = at.channel0 + (live ? c : 0);
    const int states = (int)d.states;
    const int64_t used = used_length(a.lengths, at.batch, d.length);
    const int64_t t_begin = at.segment * d.segment_length;
    const int64_t t_end = t_begin + d.segment_length < d.length ? t_begin + d.segment_length : d.length;
    const int64_t t_used = used < t_end ? used : t_end;                  // tokens of the segment that count

    // this thread's part of a tile: 8 channels of one token
    const bool has_item = tid < ITEMS;
    const int item_t = tid / CHV, item_c = (tid % CHV) * 8;
    const int item_valid = has_item ? (int)(at.n_channels - item_c < 8 ? at.n_channels - item_c : 8) : 0;
    const bool item_vec = d.vec && item_valid == 8;
    const T* const u = reinterpret_cast<const T*>(a.u) + at.batch * a.u_batch + at.channel0 + item_c;
    const T* const delta = reinterpret_cast<const T*>(a.delta) + at.batch * a.delta_batch + at.channel0 + item_c;
    const T* const z = a.z ? reinterpret_cast<const T*>(a.z) + at.batch * a.z_batch + at.channel0 + item_c : nullptr;
    T* const out = reinterpret_cast<T*>(a.out) + at.batch * d.length * d.channels + at.channel0 + item_c;
    const T* const B = reinterpret_cast<const T*>(a.B) + at.batch * a.B_batch + at.group * a.B_group;
    const T* const C = reinterpret_cast<const T*>(a.C) + at.batch * a.C_batch + at.group * a.C_group;
    float skip[8], bias[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        skip[i] = a.D && i < item_valid ? a.D[at.channel0 + item_c + i] : 0.0f;
        bias[i] = a.delta_bias && i < item_valid ? a.delta_bias[at.channel0 + item_c + i] : 0.0f;
    }

    Pack<T, 8> raw_u, raw_d, raw_z, next_u, next_d, next_z;
    T raw_b[BCN], raw_c[BCN];
    auto fetch = [&](int64_t t0) {
        const int64_t t = t0 + item_t;
        const int valid = t < t_used ? item_valid : 0;
        const bool vec = item_vec && valid == 8;
        if (has_item) {
            next_u = load_pack<T, 8>(u + t * a.u_token, vec, valid);
            next_d = load_pack<T, 8>(delta + t * a.delta_token, vec, valid);
            if (!LOCAL && z) next_z = load_pack<T, 8>(z + t * a.z_token, vec, valid);
        }
#pragma unroll
        for (int k = 0; k < BCN; ++k) {
            const int e = tid + k * THREADS;
            const int64_t tt = t0 + e / NP;
            const int n = e % NP;
            const bool in = e < STEPS * NP && tt < t_used && n < states;
            raw_b[k] = in ? B[tt * a.B_token + n] : from_f32<T>(0.0f);
            if (!LOCAL) raw_c[k] = in ? C[tt * a.C_token + n] : from_f32<T>(0.0f);
        }
    };
    auto stage = [&](int64_t t0, int buf) {
        raw_u = next_u;
        raw_d = next_d;
        if (!LOCAL && z) raw_z = next_z;
        if (has_item) {
            const bool in = t0 + item_t < t_used;
            float2 du[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float dt = to_f32(raw_d.v[i]) + bias[i];
                if (d.softplus) dt = softplus(dt);
                // padding leaves the state as it is: dt = 0 makes the factor 1 and the addend 0
                du[i] = in ? make_float2(dt, dt * to_f32(raw_u.v[i])) : make_float2(0.0f, 0.0f);
            }
            float4* const to = reinterpret_cast<float4*>(s_du + (buf * STEPS + item_t) * CH + item_c);
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = make_float4(du[2 * i].x, du[2 * i].y, du[2 * i + 1].x, du[2 * i + 1].y);
        }
#pragma unroll
        for (int k = 0; k < BCN; ++k) {
            const int e = tid + k * THREADS;
            if (e < STEPS * NP) {
                s_b[buf * STEPS * NP + e] = to_f32(raw_b[k]);
                if (!LOCAL) s_c[buf * STEPS * NP + e] = to_f32(raw_c[k]);
            }
        }
    };

    // exp(dt A) = 2^(dt A log2 e); padded states have A = B = C = 0
    const float4 A4 = load_states(a.A + channel * states, 4 * j, states, d.vec_states);
    const F2 A01 = pack2(A4.x * kLog2e, A4.y * kLog2e), A23 = pack2(A4.z * kLog2e, A4.w * kLog2e);
    F2 h01 = pack2(0.0f, 0.0f), h23 = h01;
    if (t_begin < t_used) fetch(t_begin);
    if (!LOCAL) {
        const int64_t row = (at.batch * d.channels + channel) * states;
        if (a.initial_state) {
            const float4 h = load_states(a.initial_state + row, 4 * j, states, d.vec_states);
            h01 = pack2(h.x, h.y);
            h23 = pack2(h.z, h.w);
        }
        // the state in front of this segment: h <- exp(A sum dt) h + (what the segment adds), segment by segment
        for (int64_t s = 0; s < at.segment; ++s) {
            const int64_t cell = (at.batch * d.segments + s) * d.channels + channel;
            const float sum = p.seg_dt[cell];
            const float4 add = load_states(p.seg_state + cell * states, 4 * j, states, d.vec_states);
            const F2 s2 = pack2(sum, sum);
            h01 = fma2(exp2_pair(mul2(A01, s2)), h01, pack2(add.x, add.y));
            h23 = fma2(exp2_pair(mul2(A23, s2)), h23, pack2(add.z, add.w));
        }
    }
    float sum_dt = 0.0f;
    if (t_begin < t_used) stage(t_begin, 0);
    __syncthreads();

    int buf = 0;
    for (int64_t t0 = t_begin; t0 < t_used; t0 += STEPS, buf ^= 1) {
        const bool more = t0 + STEPS < t_used;
        Pack<T, 8> done_u, done_z;
        if (more) fetch(t0 + STEPS);
        const float2* const du_row = s_du + buf * STEPS * CH + c;
        const float* const b_row = s_b + buf * STEPS * NP + 4 * j;
        const float* const c_row = s_c + buf * STEPS * NP + 4 * j;
#pragma unroll 1
        for (int g = 0; g < STEPS / V; ++g) {
            if (!LOCAL && a.checkpoints && (t0 + g * V) % kCheckpoint == 0 && live && t0 + g * V < d.length) {
                float4 h;
                unpack2(h01, h.x, h.y);
                unpack2(h23, h.z, h.w);
                const int64_t chunk = (t0 + g * V) / kCheckpoint, chunks = (d.length + kCheckpoint - 1) / kCheckpoint;
                store_states(a.checkpoints + ((at.batch * chunks + chunk) * d.channels + channel) * states, h, 4 * j, states,
                             d.vec_states);
            }
            float y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int t = g * V + i;
                const float2 du = du_row[t * CH];
                const float4 b = *reinterpret_cast<const float4*>(b_row + t * NP);
                const F2 dt2 = pack2(du.x, du.x), du2 = pack2(du.y, du.y);
                h01 = fma2(exp2_pair(mul2(A01, dt2)), h01, mul2(du2, pack2(b.x, b.y)));
                h23 = fma2(exp2_pair(mul2(A23, dt2)), h23, mul2(du2, pack2(b.z, b.w)));
                if (LOCAL) {
                    sum_dt += du.x;
                } else {
                    const float4 cc = *reinterpret_cast<const float4*>(c_row + t * NP);
                    y[i] = sum2(fma2(h23, pack2(cc.z, cc.w), mul2(h01, pack2(cc.x, cc.y))));
                }
            }
            if (!LOCAL) {
                reduce_lanes<V, P, 1>(y, lane);
                if (reduced_owner<V, P>(j)) {
                    const int t = g * V + reduced_index<V, P>(j);
#pragma unroll
                    for (int i = 0; i < reduced_count<V, P>(); ++i) s_y[(buf * STEPS + t + i) * ROW + c] = y[i];
                }
            }
        }
        if (!LOCAL) {
            done_u = raw_u;
            if (z) done_z = raw_z;
        }
        if (more) stage(t0 + STEPS, buf ^ 1);
        __syncthreads();
        if (!LOCAL && has_item && t0 + item_t < t_end) {
            const int64_t t = t0 + item_t;
            const float* const y = s_y + (buf * STEPS + item_t) * ROW + item_c;
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[i] = fmaf(skip[i], to_f32(done_u.v[i]), y[i]);
                if (z) {
                    const float g = to_f32(done_z.v[i]);
                    o[i] *= g * sigmoid(g);
                }
                if (t >= t_used) o[i] = 0.0f;
            }
            store_pack<T, 8>(out + t * d.channels, o, item_vec, item_valid);
        }
    }
    if (LOCAL) {
        if (live) {
            const int64_t cell = (at.batch * d.segments + at.segment) * d.channels + channel;
            float4 h;
            unpack2(h01, h.x, h.y);
            unpack2(h23, h.z, h.w);
            store_states(p.seg_state + cell * states, h, 4 * j, states, d.vec_states);
            if (j == 0) p.seg_dt[cell] = sum_dt;
        }
        return;
    }
    // outputs of padding behind the last tile
    const int64_t covered = t_used > t_begin ? t_begin + (t_used - t_begin + STEPS - 1) / STEPS * STEPS : t_begin;
    if (has_item) {
        const float zero[8] = {};
        for (int64_t t = covered + item_t; t < t_end; t += STEPS)
            store_pack<T, 8>(out + t * d.channels, zero, item_vec, item_valid);
    }
    if (a.final_state && at.segment == d.segments - 1 && live) {
        float4 h;
        unpack2(h01, h.x, h.y);
        unpack2(h23, h.z, h.w);
        store_states(a.final_state + (at.batch * d.channels + channel) * states, h, 4 * j, states, d.vec_states);
    }
}

template <int P>
constexpr size_t forward_smem() {
    using S = Shape<P>;
    return sizeof(float) * 2 * (size_t)(S::STEPS * S::CH * 2 + 2 * S::STEPS * S::NP + S::STEPS * S::ROW);
}

// ---------------------------------------------------------------------------------------------------------
// backward
//
// The gradient of the state runs from the last token to the first: gh_t = C_t gy_t + a_{t+1} gh_{t+1} with gy = gout
// silu(z).  It meets the states h_t, which are computed again, 16 tokens at a time from the saved state in front of
// them; the 16 states and factors of a lane stay in registers, so every exponential is computed once here too.
//   gC_t = sum_d gy h_t, gB_t = sum_d gh_t dt u     sums over the channels: over the lanes of a warp with reduce_lanes,
//                                                   over the warps in shared memory, over the blocks in a second launch
//                                                   from partial sums (no atomics: the same bits every time)
//   w_t = a_t gh_t (handed to the token before), q = w_t h_{t-1}: gA = sum q dt, g(dt) = sum_n q A + u sum_n gh B,
//   gu = dt sum_n gh B + D gy
template <int P>
struct BackShape {
    using S = Shape<P>;
    static constexpr int STEPS = kCheckpoint;
    static constexpr int WARPS = S::THREADS / 32;
    static constexpr int CHV = S::CH / 4;                                // 4 channels of one token per item
    static constexpr int ITEMS = STEPS * CHV;
    static constexpr int IPT = (ITEMS + S::THREADS - 1) / S::THREADS;
    static constexpr int ROW = S::CH + (P >= 8 ? 4 : 32 / P);
    static constexpr size_t floats = STEPS * S::CH * 3 + 2 * STEPS * S::NP + 3 * STEPS * ROW + WARPS * STEPS * 2 * S::NP;
};

template <typename T, int P, bool LOCAL>
__global__ void __launch_bounds__(Shape<P>::THREADS) scan_backward(const __grid_constant__ ScanParams p) {
    using S = Shape<P>;
    using Bk = BackShape<P>;
    constexpr int THREADS = S::THREADS, CH = S::CH, NP = S::NP, STEPS = Bk::STEPS, ROW = Bk::ROW, WARPS = Bk::WARPS;
    constexpr int CHV = Bk::CHV, ITEMS = Bk::ITEMS, IPT = Bk::IPT;
    constexpr int BCN = (STEPS * NP + THREADS - 1) / THREADS;
    constexpr int R = 32 / P;                                            // channels of a warp
    extern __shared__ __align__(16) float smem[];
    float2* const s_du = reinterpret_cast<float2*>(smem);                // [STEPS][CH] (dt, dt * u)
    float* const s_gy = smem + STEPS * CH * 2;                           // [STEPS][CH]
    float* const s_b = s_gy + STEPS * CH;                                // [STEPS][NP]
    float* const s_c = s_b + STEPS * NP;                                 // [STEPS][NP]
    float* const s_y = s_c + STEPS * NP;                                 // [STEPS][ROW] C . h
    float* const s_s = s_y + STEPS * ROW;                                // [2][STEPS][ROW] sum_n gh B, sum_n q A / ln 2
    float* const s_r = s_s + 2 * STEPS * ROW;                            // [WARPS][STEPS][2][NP] gC, gB of the warps

    const OvlSelectiveScan& a = p.a;
    const ScanDims& d = p.d;
    const Place at = block_place(d, CH);
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, j = lane % P, c = tid / P;
    const bool live = c < at.n_channels;
    const int64_t channel = at.channel0 + (live ? c : 0);
    const int states = (int)d.states;
    const int64_t used = used_length(a.lengths, at.batch, d.length);
    const int64_t t_begin = at.segment * d.segment_length;
    const int64_t t_end = t_begin + d.segment_length < d.length ? t_begin + d.segment_length : d.length;
    const int64_t t_used = used < t_end ? used : t_end;
    const int64_t chunks = (d.length + kCheckpoint - 1) / kCheckpoint;
    const int64_t first = t_begin, last = t_used > t_begin ? t_begin + (t_used - t_begin - 1) / STEPS * STEPS : t_begin - STEPS;

    const int64_t base_c = at.channel0;
    const T* const u = reinterpret_cast<const T*>(a.u) + at.batch * a.u_batch + base_c;
    const T* const delta = reinterpret_cast<const T*>(a.delta) + at.batch * a.delta_batch + base_c;
    const T* const z = a.z ? reinterpret_cast<const T*>(a.z) + at.batch * a.z_batch + base_c : nullptr;
    const T* const gout = reinterpret_cast<const T*>(a.gout) + at.batch * a.gout_batch + base_c;
    const T* const B = reinterpret_cast<const T*>(a.B) + at.batch * a.B_batch + at.group * a.B_group;
    const T* const C = reinterpret_cast<const T*>(a.C) + at.batch * a.C_batch + at.group * a.C_group;

    Pack<T, 4> raw_u[IPT], raw_d[IPT], raw_z[IPT], raw_g[IPT];
    T raw_b[BCN], raw_c[BCN];
    float4 start;                                                        // the saved state in front of the tile
    auto item_of = [&](int k, int& t, int& cc, int& valid) {
        const int e = tid + k * THREADS;
        t = e / CHV;
        cc = (e % CHV) * 4;
        const int64_t left = at.n_channels - cc;
        valid = e >= ITEMS || left <= 0 ? 0 : left < 4 ? (int)left : 4;
    };
    auto fetch = [&](int64_t t0) {
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            int it, cc, valid;
            item_of(k, it, cc, valid);
            const int64_t t = t0 + it;
            if (t >= t_used) valid = 0;
            const bool vec = d.vec && valid == 4;
            if (!LOCAL) raw_u[k] = load_pack<T, 4>(u + t * a.u_token + cc, vec, valid);
            raw_d[k] = load_pack<T, 4>(delta + t * a.delta_token + cc, vec, valid);
            if (z) raw_z[k] = load_pack<T, 4>(z + t * a.z_token + cc, vec, valid);
            raw_g[k] = load_pack<T, 4>(gout + t * a.gout_token + cc, vec, valid);
        }
#pragma unroll
        for (int k = 0; k < BCN; ++k) {
            const int e = tid + k * THREADS;
            const int64_t t = t0 + e / NP;
            const int n = e % NP;
            const bool in = e < STEPS * NP && t < t_used && n < states;
            if (!LOCAL) raw_b[k] = in ? B[t * a.B_token + n] : from_f32<T>(0.0f);
            raw_c[k] = in ? C[t * a.C_token + n] : from_f32<T>(0.0f);
        }
        if (!LOCAL)
            start = load_states(a.checkpoints + ((at.batch * chunks + t0 / kCheckpoint) * d.channels + channel) * states,
                                4 * j, states, d.vec_states);
    };
    float bias[IPT][4], skip[IPT][4];
#pragma unroll
    for (int k = 0; k < IPT; ++k) {
        int it, cc, valid;
        item_of(k, it, cc, valid);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bias[k][i] = a.delta_bias && i < valid ? a.delta_bias[base_c + cc + i] : 0.0f;
            skip[k][i] = a.D && i < valid ? a.D[base_c + cc + i] : 0.0f;
        }
    }
    auto stage = [&](int64_t t0) {
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            int it, cc, valid;
            item_of(k, it, cc, valid);
            if (tid + k * THREADS < ITEMS) {
                const bool in = t0 + it < t_used;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float dt = to_f32(raw_d[k].v[i]) + bias[k][i];
                    if (d.softplus) dt = softplus(dt);
                    float gy = to_f32(raw_g[k].v[i]);
                    if (z) {
                        const float g = to_f32(raw_z[k].v[i]);
                        gy *= g * sigmoid(g);
                    }
                    const float du = LOCAL ? 0.0f : dt * to_f32(raw_u[k].v[i]);
                    s_du[it * CH + cc + i] = in ? make_float2(dt, du) : make_float2(0.0f, 0.0f);
                    s_gy[it * CH + cc + i] = in ? gy : 0.0f;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < BCN; ++k) {
            const int e = tid + k * THREADS;
            if (e < STEPS * NP) {
                if (!LOCAL) s_b[e] = to_f32(raw_b[k]);
                s_c[e] = to_f32(raw_c[k]);
            }
        }
    };

    const float4 A4 = load_states(a.A + channel * states, 4 * j, states, d.vec_states);
    const F2 A01 = pack2(A4.x * kLog2e, A4.y * kLog2e), A23 = pack2(A4.z * kLog2e, A4.w * kLog2e);
    F2 w01 = pack2(0.0f, 0.0f), w23 = w01;                               // a_{t+1} gh_{t+1}
    if (last >= first) fetch(last);
    if (!LOCAL) {
        if (a.gfinal) {
            const float4 g = load_states(a.gfinal + (at.batch * d.channels + channel) * states, 4 * j, states, d.vec_states);
            w01 = pack2(g.x, g.y);
            w23 = pack2(g.z, g.w);
        }
        for (int64_t s = d.segments - 1; s > at.segment; --s) {
            const int64_t cell = (at.batch * d.segments + s) * d.channels + channel;
            const float sum = p.seg_dt[cell];
            const float4 add = load_states(p.seg_state + cell * states, 4 * j, states, d.vec_states);
            const F2 s2 = pack2(sum, sum);
            w01 = fma2(exp2_pair(mul2(A01, s2)), w01, pack2(add.x, add.y));
            w23 = fma2(exp2_pair(mul2(A23, s2)), w23, pack2(add.z, add.w));
        }
    }
    double gA[4] = {0.0, 0.0, 0.0, 0.0};
    float gD[IPT][4] = {}, gbias[IPT][4] = {};
    float sum_dt = 0.0f;

    for (int64_t t0 = last; t0 >= first; t0 -= STEPS) {
        stage(t0);
        F2 h01[STEPS], h23[STEPS], a01[STEPS], a23[STEPS];
        const F2 s01 = pack2(start.x, start.y), s23 = pack2(start.z, start.w);
        Pack<T, 4> now_u[IPT], now_d[IPT], now_z[IPT], now_g[IPT];
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            now_u[k] = raw_u[k];
            now_d[k] = raw_d[k];
            now_z[k] = raw_z[k];
            now_g[k] = raw_g[k];
        }
        __syncthreads();
        if (t0 > first) fetch(t0 - STEPS);

        // the states again, forwards
        F2 x01 = s01, x23 = s23;
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const float2 du = s_du[t * CH + c];
            const F2 dt2 = pack2(du.x, du.x);
            a01[t] = exp2_pair(mul2(A01, dt2));
            a23[t] = exp2_pair(mul2(A23, dt2));
            if (LOCAL) {
                sum_dt += du.x;
            } else {
                const float4 b = *reinterpret_cast<const float4*>(s_b + t * NP + 4 * j);
                const F2 du2 = pack2(du.y, du.y);
                x01 = fma2(a01[t], x01, mul2(du2, pack2(b.x, b.y)));
                x23 = fma2(a23[t], x23, mul2(du2, pack2(b.z, b.w)));
                h01[t] = x01;
                h23[t] = x23;
            }
        }
        if (!LOCAL && z) {
            constexpr int V = P < 16 ? P : 16;
#pragma unroll
            for (int g = 0; g < STEPS / V; ++g) {
                float y[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float4 cc = *reinterpret_cast<const float4*>(s_c + (g * V + i) * NP + 4 * j);
                    y[i] = sum2(fma2(h23[g * V + i], pack2(cc.z, cc.w), mul2(h01[g * V + i], pack2(cc.x, cc.y))));
                }
                reduce_lanes<V, P, 1>(y, lane);
                if (reduced_owner<V, P>(j)) {
                    const int t = g * V + reduced_index<V, P>(j);
#pragma unroll
                    for (int i = 0; i < reduced_count<V, P>(); ++i) s_y[(t + i) * ROW + c] = y[i];
                }
            }
        }
        // the gradients, backwards
        F2 gA01 = pack2(0.0f, 0.0f), gA23 = gA01;
#pragma unroll
        for (int g = STEPS / 4 - 1; g >= 0; --g) {
            float s[8];
#pragma unroll
            for (int i = 3; i >= 0; --i) {
                const int t = g * 4 + i;
                const float gy = s_gy[t * CH + c];
                const F2 gy2 = pack2(gy, gy);
                const float4 cc = *reinterpret_cast<const float4*>(s_c + t * NP + 4 * j);
                const F2 g01 = fma2(gy2, pack2(cc.x, cc.y), w01), g23 = fma2(gy2, pack2(cc.z, cc.w), w23);
                w01 = mul2(a01[t], g01);
                w23 = mul2(a23[t], g23);
                if (!LOCAL) {
                    const float2 du = s_du[t * CH + c];
                    const float4 b = *reinterpret_cast<const float4*>(s_b + t * NP + 4 * j);
                    const F2 du2 = pack2(du.y, du.y), dt2 = pack2(du.x, du.x);
                    float v[8];
                    unpack2(mul2(gy2, h01[t]), v[0], v[1]);
                    unpack2(mul2(gy2, h23[t]), v[2], v[3]);
                    unpack2(mul2(du2, g01), v[4], v[5]);
                    unpack2(mul2(du2, g23), v[6], v[7]);
                    if (!live) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = 0.0f;
                    }
                    reduce_lanes<8, R, P>(v, lane);
                    if (reduced_owner<8, R>(lane / P)) {
                        const int k0 = reduced_index<8, R>(lane / P);
                        float* const to = s_r + (warp * STEPS + t) * 2 * NP + 4 * j;
#pragma unroll
                        for (int k = 0; k < reduced_count<8, R>(); ++k) to[((k0 + k) / 4) * NP + (k0 + k) % 4] = v[k];
                    }
                    s[2 * i] = sum2(fma2(g23, pack2(b.z, b.w), mul2(g01, pack2(b.x, b.y))));
                    const F2 q01 = mul2(w01, t > 0 ? h01[t > 0 ? t - 1 : 0] : s01), q23 = mul2(w23, t > 0 ? h23[t > 0 ? t - 1 : 0] : s23);
                    s[2 * i + 1] = sum2(fma2(q23, A23, mul2(q01, A01)));
                    gA01 = fma2(q01, dt2, gA01);
                    gA23 = fma2(q23, dt2, gA23);
                }
            }
            if (!LOCAL) {
                reduce_lanes<8, P, 1>(s, lane);
                if (reduced_owner<8, P>(j)) {
                    const int k0 = reduced_index<8, P>(j);
#pragma unroll
                    for (int k = 0; k < reduced_count<8, P>(); ++k)
                        s_s[(((k0 + k) % 2) * STEPS + g * 4 + (k0 + k) / 2) * ROW + c] = s[k];
                }
            }
        }
        if (!LOCAL) {
            float x, y;
            unpack2(gA01, x, y);
            gA[0] += x;
            gA[1] += y;
            unpack2(gA23, x, y);
            gA[2] += x;
            gA[3] += y;
        }
        __syncthreads();
        if (!LOCAL) {
#pragma unroll
            for (int k = 0; k < IPT; ++k) {
                int it, cc, valid;
                item_of(k, it, cc, valid);
                const int64_t t = t0 + it;
                if (valid > 0 && t < t_end) {
                    const bool in = t < t_used, vec = d.vec && valid == 4;
                    float gu[4], gd[4], gz[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float xu = to_f32(now_u[k].v[i]), go = to_f32(now_g[k].v[i]);
                        const float raw = to_f32(now_d[k].v[i]) + bias[k][i];
                        const float dt = s_du[it * CH + cc + i].x, gy = s_gy[it * CH + cc + i];
                        const float over = s_s[it * ROW + cc + i];
                        gu[i] = in ? fmaf(dt, over, skip[k][i] * gy) : 0.0f;
                        float g = fmaf(xu, over, kLn2 * s_s[(STEPS + it) * ROW + cc + i]);
                        if (d.softplus) g *= sigmoid(raw);
                        gd[i] = in ? g : 0.0f;
                        if (z) {
                            const float zz = to_f32(now_z[k].v[i]), sig = sigmoid(zz);
                            const float y = fmaf(skip[k][i], xu, s_y[it * ROW + cc + i]);
                            gz[i] = in ? go * y * sig * (1.0f + zz * (1.0f - sig)) : 0.0f;
                        }
                        gD[k][i] += in ? gy * xu : 0.0f;
                        gbias[k][i] += gd[i];
                    }
                    const int64_t o = (at.batch * d.length + t) * d.channels + base_c + cc;
                    store_pack<T, 4>(reinterpret_cast<T*>(a.gu) + o, gu, vec, valid);
                    store_pack<T, 4>(reinterpret_cast<T*>(a.gdelta) + o, gd, vec, valid);
                    if (a.gz) store_pack<T, 4>(reinterpret_cast<T*>(a.gz) + o, gz, vec, valid);
                }
            }
            float* const part =
                p.part_bc + (((at.batch * d.groups + at.group) * d.tiles + at.tile) * d.length + t0) * 2 * NP;
            for (int e = tid; e < STEPS * 2 * NP; e += THREADS) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) sum += s_r[w * STEPS * 2 * NP + e];
                if (t0 + e / (2 * NP) < t_used) part[e] = sum;
            }
            // the epilogue reads what the next stage() overwrites
            __syncthreads();
        }
    }
    if (LOCAL) {
        if (live) {
            const int64_t cell = (at.batch * d.segments + at.segment) * d.channels + channel;
            float4 w;
            unpack2(w01, w.x, w.y);
            unpack2(w23, w.z, w.w);
            store_states(p.seg_state + cell * states, w, 4 * j, states, d.vec_states);
            if (j == 0) p.seg_dt[cell] = sum_dt;
        }
        return;
    }
    // gradients of padding behind the last tile
    for (int64_t t0 = last + STEPS; t0 < t_end; t0 += STEPS) {
        const float zero[4] = {};
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            int it, cc, valid;
            item_of(k, it, cc, valid);
            if (valid > 0 && t0 + it < t_end) {
                const bool vec = d.vec && valid == 4;
                const int64_t o = (at.batch * d.length + t0 + it) * d.channels + base_c + cc;
                store_pack<T, 4>(reinterpret_cast<T*>(a.gu) + o, zero, vec, valid);
                store_pack<T, 4>(reinterpret_cast<T*>(a.gdelta) + o, zero, vec, valid);
                if (a.gz) store_pack<T, 4>(reinterpret_cast<T*>(a.gz) + o, zero, vec, valid);
            }
        }
    }
    const int64_t part_row = at.batch * d.segments + at.segment;
    if (live) {
        store_states(p.part_A + (part_row * d.channels + channel) * states,
                     make_float4((float)gA[0], (float)gA[1], (float)gA[2], (float)gA[3]), 4 * j, states, d.vec_states);
        if (a.ginitial && at.segment == 0) {
            float4 w;
            unpack2(w01, w.x, w.y);
            unpack2(w23, w.z, w.w);
            store_states(a.ginitial + (at.batch * d.channels + channel) * states, w, 4 * j, states, d.vec_states);
        }
    }
    // gD and gdelta_bias: every thread has sums over its token of each tile; over the 16 tokens in shared memory
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            int it, cc, valid;
            item_of(k, it, cc, valid);
            if (tid + k * THREADS < ITEMS) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s_y[it * ROW + cc + i] = which ? gbias[k][i] : gD[k][i];
            }
        }
        __syncthreads();
        for (int e = tid; e < at.n_channels; e += THREADS) {
            float sum = 0.0f;
            for (int t = 0; t < STEPS; ++t) sum += s_y[t * ROW + e];
            p.part_D[(part_row * 2 + which) * d.channels + base_c + e] = sum;
        }
    }
}

// gB and gC: the channel tiles' parts added up in tile order; one thread per (batch, token, group, state)
template <typename T>
__global__ void scan_backward_bc(const __grid_constant__ ScanParams p, int np) {
    const ScanDims& d = p.d;
    const int64_t per = d.length * d.groups * d.states;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < p.a.batch * per; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t b = i / per;
        int64_t k = i % per;
        const int n = (int)(k % d.states);
        k /= d.states;
        const int64_t g = k % d.groups, t = k / d.groups;
        float c = 0.0f, bb = 0.0f;
        if (t < used_length(p.a.lengths, b, d.length)) {
            const float* src = p.part_bc + ((b * d.groups + g) * d.tiles * d.length + t) * 2 * np + n;
            for (int64_t tile = 0; tile < d.tiles; ++tile) {
                c += src[tile * d.length * 2 * np];
                bb += src[tile * d.length * 2 * np + np];
            }
        }
        reinterpret_cast<T*>(p.a.gC)[i] = from_f32<T>(c);
        reinterpret_cast<T*>(p.a.gB)[i] = from_f32<T>(bb);
    }
}

// gA, gD, gdelta_bias: the parts of batches and segments added up in order
__global__ void scan_backward_params(const __grid_constant__ ScanParams p) {
    const ScanDims& d = p.d;
    const int64_t rows = p.a.batch * d.segments, n_A = d.channels * d.states, total = n_A + 2 * d.channels;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const bool in_A = i < n_A;
        const int64_t k = in_A ? i : i - n_A, stride = in_A ? n_A : 2 * d.channels;
        const float* src = (in_A ? p.part_A : p.part_D) + k;
        double sum = 0.0;
        for (int64_t r = 0; r < rows; ++r) sum += src[r * stride];
        float* const to = in_A ? p.a.gA : k < d.channels ? p.a.gD : p.a.gdelta_bias;
        if (to) to[in_A || k < d.channels ? k : k - d.channels] = (float)sum;
    }
}

// ---------------------------------------------------------------------------------------------------------
// one token

// a thread per 4 states of a (row, channel); a block works on one row
template <typename T, int P>
__global__ void __launch_bounds__(128) scan_step(const __grid_constant__ OvlSelectiveScanStep a, int64_t blocks_per_row,
                                                 int vec_states) {
    const int64_t row = blockIdx.x / blocks_per_row;
    const int tid = threadIdx.x, lane = tid % 32, j = lane % P;
    const int64_t channel_at = (blockIdx.x % blocks_per_row) * (128 / P) + tid / P;
    const bool live = channel_at < a.channels;
    const int64_t channel = live ? channel_at : a.channels - 1;
    T* const out = reinterpret_cast<T*>(a.out) + row * a.channels;
    int64_t slot = row;
    if (a.slot_of_row) {
        slot = a.slot_of_row[row];
        int taken = 0;
        for (int64_t r = tid; r < row; r += 128) taken |= slot >= 0 && a.slot_of_row[r] == slot;
        taken = __syncthreads_or(taken);
        if (slot < 0 || slot >= a.slots || taken) {
            if (live && j == 0) out[channel] = from_f32<T>(slot < 0 ? 0.0f : __int_as_float(0x7fffffff));
            return;
        }
    }
    const int states = (int)a.states;
    const int64_t group = channel / (a.channels / a.groups);
    float* const state = a.state + (slot * a.channels + channel) * states;
    float4 h = load_states(state, 4 * j, states, vec_states);
    const float4 A = load_states(a.A + channel * states, 4 * j, states, vec_states);
    const T* const B = reinterpret_cast<const T*>(a.B) + row * a.B_row + group * a.B_group;
    const T* const C = reinterpret_cast<const T*>(a.C) + row * a.C_row + group * a.C_group;
    const float u = to_f32(reinterpret_cast<const T*>(a.u)[row * a.u_row + channel]);
    float dt = to_f32(reinterpret_cast<const T*>(a.delta)[row * a.delta_row + channel]);
    const float z = a.z ? to_f32(reinterpret_cast<const T*>(a.z)[row * a.z_row + channel]) : 0.0f;
    const float skip = a.D ? a.D[channel] : 0.0f;
    if (a.delta_bias) dt += a.delta_bias[channel];
    float b[4], c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        b[i] = 4 * j + i < states ? to_f32(B[4 * j + i]) : 0.0f;
        c[i] = 4 * j + i < states ? to_f32(C[4 * j + i]) : 0.0f;
    }
    if (a.delta_softplus) dt = softplus(dt);
    const float du = dt * u, dt2 = dt * kLog2e;
    h.x = fmaf(exp2_approx(dt2 * A.x), h.x, du * b[0]);
    h.y = fmaf(exp2_approx(dt2 * A.y), h.y, du * b[1]);
    h.z = fmaf(exp2_approx(dt2 * A.z), h.z, du * b[2]);
    h.w = fmaf(exp2_approx(dt2 * A.w), h.w, du * b[3]);
    float y[1] = {fmaf(h.x, c[0], fmaf(h.y, c[1], fmaf(h.z, c[2], h.w * c[3])))};
    reduce_lanes<1, P, 1>(y, lane);
    if (!live) return;
    store_states(state, h, 4 * j, states, vec_states);
    if (j == 0) {
        float o = fmaf(skip, u, y[0]);
        if (a.z) o *= z * sigmoid(z);
        out[channel] = from_f32<T>(o);
    }
}

// ---------------------------------------------------------------------------------------------------------
// host side

int lanes_of(int64_t states) {
    int p = 1;
    while (4 * p < states) p *= 2;
    return p;
}

bool multiple_of(int64_t n, int64_t a, int64_t b) { return a % n == 0 && b % n == 0; }

int check(const OvlSelectiveScan* a, bool backward) {
    if (!a) return OVL_ERR_NULL;
    if (a->dtype != OVL_FLOAT32 && a->dtype != OVL_FLOAT16 && a->dtype != OVL_BFLOAT16) return OVL_ERR_DTYPE;
    if (a->batch < 0 || a->length < 0 || a->channels < 1 || a->groups < 1 || a->states < 1) return OVL_ERR_INVALID;
    if (a->channels % a->groups != 0) return OVL_ERR_INVALID;
    if (a->states > kMaxStates) return OVL_ERR_TOO_LARGE;
    (void)backward;
    return OVL_OK;
}

template <int P>
void shape_dims(const OvlSelectiveScan* a, ScanDims* d, bool backward) {
    d->length = a->length;
    d->channels = a->channels;
    d->states = a->states;
    d->groups = a->groups;
    d->group_channels = a->channels / a->groups;
    d->tiles = ceil_div(d->group_channels, Shape<P>::CH);
    d->softplus = a->delta_softplus != 0;
    // Segments: with fewer blocks than SMs the length is cut so that the blocks fill the device; every segment but the
    // last is then walked twice (what it adds to the state first), so a cut pays from three segments on.
    const int64_t blocks = a->batch * a->groups * d->tiles;
    const int64_t fill = sequence_sm_count() * (backward ? 2 : 3);
    int64_t s = blocks > 0 ? fill / blocks : 1;
    const int64_t most = ceil_div(a->length, 64);
    if (s > most) s = most;
    if (s > kMaxSegments) s = kMaxSegments;
    if (s < 3) s = 1;
    d->segment_length = ceil_div(ceil_div(a->length > 0 ? a->length : 1, s), 32) * 32;
    d->segments = ceil_div(a->length > 0 ? a->length : 1, d->segment_length);
}

void make_dims(const OvlSelectiveScan* a, ScanDims* d, bool backward) {
    switch (lanes_of(a->states)) {
        case 1: shape_dims<1>(a, d, backward); break;
        case 2: shape_dims<2>(a, d, backward); break;
        case 4: shape_dims<4>(a, d, backward); break;
        case 8: shape_dims<8>(a, d, backward); break;
        case 16: shape_dims<16>(a, d, backward); break;
        default: shape_dims<32>(a, d, backward); break;
    }
}

uint64_t round16(uint64_t n) { return (n + 15) / 16 * 16; }

struct Workspace {
    uint64_t state, dt, bc, A, D, total;
};
Workspace layout(const OvlSelectiveScan* a, const ScanDims& d, bool backward) {
    Workspace w{};
    uint64_t at = 0;
    auto take = [&](uint64_t floats) {
        const uint64_t here = at;
        at += round16(floats * sizeof(float));
        return here;
    };
    if (d.segments > 1) {
        w.state = take((uint64_t)a->batch * d.segments * d.channels * d.states);
        w.dt = take((uint64_t)a->batch * d.segments * d.channels);
    }
    if (backward) {
        w.bc = take((uint64_t)a->batch * d.groups * d.tiles * d.length * 8 * lanes_of(a->states));
        w.A = take((uint64_t)a->batch * d.segments * d.channels * d.states);
        w.D = take((uint64_t)a->batch * d.segments * 2 * d.channels);
    }
    w.total = at;
    return w;
}

template <typename F>
int with_smem(F kernel, size_t bytes) {
    if (bytes > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return record_cuda_error(e);
    }
    return OVL_OK;
}

template <typename T, int P>
int run_forward(const ScanParams& p, int64_t blocks, cudaStream_t stream) {
    constexpr size_t smem = forward_smem<P>();
    int st;
    if (p.d.segments > 1) {
        if ((st = with_smem(scan_forward<T, P, true>, smem)) != OVL_OK) return st;
        scan_forward<T, P, true><<<(uint32_t)blocks, Shape<P>::THREADS, smem, stream>>>(p);
        if ((st = launch_status()) != OVL_OK) return st;
    }
    if ((st = with_smem(scan_forward<T, P, false>, smem)) != OVL_OK) return st;
    scan_forward<T, P, false><<<(uint32_t)blocks, Shape<P>::THREADS, smem, stream>>>(p);
    return launch_status();
}

uint32_t grid_for(int64_t items) {
    const int64_t blocks = ceil_div(items, 256), most = 16 * 8 * (int64_t)sequence_sm_count();
    return (uint32_t)(blocks < 1 ? 1 : blocks < most ? blocks : most);
}

template <typename T, int P>
int run_backward(const ScanParams& p, int64_t blocks, cudaStream_t stream) {
    constexpr size_t smem = BackShape<P>::floats * sizeof(float);
    int st;
    if (p.d.segments > 1) {
        if ((st = with_smem(scan_backward<T, P, true>, smem)) != OVL_OK) return st;
        scan_backward<T, P, true><<<(uint32_t)blocks, Shape<P>::THREADS, smem, stream>>>(p);
        if ((st = launch_status()) != OVL_OK) return st;
    }
    if ((st = with_smem(scan_backward<T, P, false>, smem)) != OVL_OK) return st;
    scan_backward<T, P, false><<<(uint32_t)blocks, Shape<P>::THREADS, smem, stream>>>(p);
    if ((st = launch_status()) != OVL_OK) return st;
    scan_backward_bc<T><<<grid_for(p.a.batch * p.d.length * p.d.groups * p.d.states), 256, 0, stream>>>(p, Shape<P>::NP);
    if ((st = launch_status()) != OVL_OK) return st;
    scan_backward_params<<<grid_for(p.d.channels * (p.d.states + 2)), 256, 0, stream>>>(p);
    return launch_status();
}

template <typename T>
int dispatch(const ScanParams& p, bool backward, cudaStream_t stream) {
    const int64_t blocks = p.a.batch * p.d.segments * p.d.groups * p.d.tiles;
    if (blocks > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    switch (lanes_of(p.a.states)) {
        case 1: return backward ? run_backward<T, 1>(p, blocks, stream) : run_forward<T, 1>(p, blocks, stream);
        case 2: return backward ? run_backward<T, 2>(p, blocks, stream) : run_forward<T, 2>(p, blocks, stream);
        case 4: return backward ? run_backward<T, 4>(p, blocks, stream) : run_forward<T, 4>(p, blocks, stream);
        case 8: return backward ? run_backward<T, 8>(p, blocks, stream) : run_forward<T, 8>(p, blocks, stream);
        case 16: return backward ? run_backward<T, 16>(p, blocks, stream) : run_forward<T, 16>(p, blocks, stream);
        default: return backward ? run_backward<T, 32>(p, blocks, stream) : run_forward<T, 32>(p, blocks, stream);
    }
}

int run(const OvlSelectiveScan* a, bool backward, cudaStream_t stream) {
    int st = check(a, backward);
    if (st != OVL_OK) return st;
    if (a->batch == 0) return OVL_OK;
    if (!a->A) return OVL_ERR_NULL;
    if (a->length > 0 && (!a->u || !a->delta || !a->B || !a->C)) return OVL_ERR_NULL;
    if (backward) {
        if (!a->gA || (a->length > 0 && (!a->gout || !a->checkpoints || !a->gu || !a->gdelta || !a->gB || !a->gC)))
            return OVL_ERR_NULL;
        if (a->gz && !a->z) return OVL_ERR_INVALID;
    } else if (a->length > 0 && !a->out) {
        return OVL_ERR_NULL;
    }
    ScanParams p{};
    p.a = *a;
    make_dims(a, &p.d, backward);
    const Workspace w = layout(a, p.d, backward);
    if (w.total > 0 && (!a->workspace || a->workspace_bytes < w.total || !aligned16(a->workspace))) return OVL_ERR_SCRATCH;
    char* const ws = reinterpret_cast<char*>(a->workspace);
    p.seg_state = reinterpret_cast<float*>(ws + w.state);
    p.seg_dt = reinterpret_cast<float*>(ws + w.dt);
    p.part_bc = reinterpret_cast<float*>(ws + w.bc);
    p.part_A = reinterpret_cast<float*>(ws + w.A);
    p.part_D = reinterpret_cast<float*>(ws + w.D);
    // wide accesses: 8 elements at a time start on 16 bytes
    bool vec = p.d.group_channels % 8 == 0 && aligned16(a->u) && aligned16(a->delta) && aligned16(a->z) && aligned16(a->out) &&
               multiple_of(8, a->u_batch, a->u_token) && multiple_of(8, a->delta_batch, a->delta_token) &&
               (!a->z || multiple_of(8, a->z_batch, a->z_token));
    if (backward)
        vec = vec && aligned16(a->gout) && multiple_of(8, a->gout_batch, a->gout_token) && aligned16(a->gu) &&
              aligned16(a->gdelta) && aligned16(a->gz);
    p.d.vec = vec;
    p.d.vec_states = a->states % 4 == 0 && aligned16(a->A) && aligned16(a->initial_state) && aligned16(a->final_state) &&
                     aligned16(a->checkpoints) && aligned16(a->gfinal) && aligned16(a->ginitial);
    if (a->dtype == OVL_FLOAT32) return dispatch<float>(p, backward, stream);
    if (a->dtype == OVL_FLOAT16) return dispatch<__half>(p, backward, stream);
    return dispatch<__nv_bfloat16>(p, backward, stream);
}

template <typename T>
int run_step(const OvlSelectiveScanStep& a, cudaStream_t stream) {
    const int lanes = lanes_of(a.states);
    const int64_t per_row = ceil_div(a.channels, 128 / lanes), blocks = per_row * a.rows;
    if (blocks > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    const int vec = a.states % 4 == 0 && aligned16(a.A) && aligned16(a.state);
    const uint32_t grid = (uint32_t)blocks;
    switch (lanes) {
        case 1: scan_step<T, 1><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
        case 2: scan_step<T, 2><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
        case 4: scan_step<T, 4><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
        case 8: scan_step<T, 8><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
        case 16: scan_step<T, 16><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
        default: scan_step<T, 32><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
    }
    return launch_status();
}

}  // namespace
}  // namespace ovl

extern "C" uint64_t ovl_selective_scan_workspace_bytes(const OvlSelectiveScan* args, int backward) {
    if (ovl::check(args, backward != 0) != OVL_OK || args->batch == 0) return 0;
    ovl::ScanDims d;
    ovl::make_dims(args, &d, backward != 0);
    return ovl::layout(args, d, backward != 0).total;
}

extern "C" int ovl_selective_scan(const OvlSelectiveScan* args, void* cuda_stream) {
    return ovl::run(args, false, (cudaStream_t)cuda_stream);
}

extern "C" int ovl_selective_scan_backward(const OvlSelectiveScan* args, void* cuda_stream) {
    return ovl::run(args, true, (cudaStream_t)cuda_stream);
}

extern "C" int ovl_selective_scan_step(const OvlSelectiveScanStep* a, void* cuda_stream) {
    if (!a) return OVL_ERR_NULL;
    if (a->dtype != OVL_FLOAT32 && a->dtype != OVL_FLOAT16 && a->dtype != OVL_BFLOAT16) return OVL_ERR_DTYPE;
    if (a->rows < 0 || a->channels < 1 || a->groups < 1 || a->states < 1 || a->slots < 0) return OVL_ERR_INVALID;
    if (a->channels % a->groups != 0 || (!a->slot_of_row && a->slots < a->rows)) return OVL_ERR_INVALID;
    if (a->states > ovl::kMaxStates) return OVL_ERR_TOO_LARGE;
    if (a->rows == 0) return OVL_OK;
    if (!a->u || !a->delta || !a->A || !a->B || !a->C || !a->out || (!a->state && a->slots > 0)) return OVL_ERR_NULL;
    const cudaStream_t stream = (cudaStream_t)cuda_stream;
    if (a->dtype == OVL_FLOAT32) return ovl::run_step<float>(*a, stream);
    if (a->dtype == OVL_FLOAT16) return ovl::run_step<__half>(*a, stream);
    return ovl::run_step<__nv_bfloat16>(*a, stream);
}
