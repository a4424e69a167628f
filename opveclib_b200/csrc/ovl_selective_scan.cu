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
// next one's elements are in flight to shared memory, each to the thread that will convert, mask and combine them
// (softplus, dt * u) into what all lanes of a channel read; double-buffered, with one barrier per tile.  The sums over the states of P steps are formed together
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
    int32_t vec_states, vec_bc;        // wide loads and stores of 4 states; of 4 elements of B and C
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

// exp(dt A) = 2^(dt A log2 e).  The special-function unit's results are 1e-8 to 2e-8 too small on average, which adds up
// over a state's memory of a thousand tokens; the same amount on the exponent takes most of it away and costs nothing
// (a multiplication becomes a multiply-add).  2^kExpBias rounds to 1, so dt = 0 still leaves a state as it is.
constexpr float kExpBias = 2e-8f;
__device__ __forceinline__ F2 decay(F2 A, F2 dt) { return exp2_pair(fma2(A, dt, same2(kExpBias))); }

// Where (dt, dt, dt u, dt u) of channel c of a tile's token t stands, in float4: a gap after every 8 channels keeps the
// wide stores of threads with 8 (or 4) channels each off one another's banks.
template <int CH>
__device__ __forceinline__ constexpr int du_at(int t, int c) { return t * (CH + CH / 8) + c + c / 8; }

// ---------------------------------------------------------------------------------------------------------
// forward

template <typename T, int P>
struct ForwardSmem {
    using S = Shape<P>;
    static constexpr size_t du = 0;                                                          // float4 [2][du_at]
    static constexpr size_t b = du + 2 * sizeof(float4) * S::STEPS * (S::CH + S::CH / 8);    // float [2][STEPS][NP]
    static constexpr size_t c = b + 2 * sizeof(float) * S::STEPS * S::NP;
    static constexpr size_t y = c + 2 * sizeof(float) * S::STEPS * S::NP;                    // float [2][STEPS][ROW]
    static constexpr size_t raw = y + 2 * sizeof(float) * S::STEPS * S::ROW;                 // T [2][3][STEPS][CH]: u, delta, z
    static constexpr size_t raw_bc = raw + 2 * 3 * sizeof(T) * S::STEPS * S::CH;             // T [2][2][STEPS][NP]
    static constexpr size_t bytes = raw_bc + 2 * 2 * sizeof(T) * S::STEPS * S::NP;
};

// LOCAL: only what a segment adds to a state that starts at zero, and its sum of dt (the first of two passes when the
// length is cut into segments); otherwise the whole operator, seeded from the segments before.
template <typename T, int P, bool LOCAL>
__global__ void __launch_bounds__(Shape<P>::THREADS) scan_forward(const __grid_constant__ ScanParams p) {
    using S = Shape<P>;
    using M = ForwardSmem<T, P>;
    constexpr int THREADS = S::THREADS, CH = S::CH, NP = S::NP, STEPS = S::STEPS, ROW = S::ROW;
    constexpr int CHV = CH / 8, ITEMS = STEPS * CHV;                     // 8 channels of one token
    constexpr int QUADS = STEPS * P, QN = (QUADS + THREADS - 1) / THREADS;   // 4 states of one token
    constexpr int V = STEPS < 16 ? STEPS : 16;                           // steps whose sums are formed together
    static_assert(ITEMS <= THREADS && STEPS % V == 0 && kCheckpoint % V == 0, "tile shape");
    extern __shared__ __align__(16) char smem[];
    float4* const s_du = reinterpret_cast<float4*>(smem + M::du);
    float* const s_b = reinterpret_cast<float*>(smem + M::b);
    float* const s_c = reinterpret_cast<float*>(smem + M::c);
    float* const s_y = reinterpret_cast<float*>(smem + M::y);
    T* const raw = reinterpret_cast<T*>(smem + M::raw);
    T* const raw_bc = reinterpret_cast<T*>(smem + M::raw_bc);
    constexpr int DU = STEPS * (CH + CH / 8);

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
    const int item_valid = !has_item || item_c >= at.n_channels ? 0 : at.n_channels - item_c < 8 ? (int)(at.n_channels - item_c) : 8;
    const bool item_vec = d.vec && item_valid == 8;
    const T* const u = reinterpret_cast<const T*>(a.u) + at.batch * a.u_batch + at.channel0 + item_c;
    const T* const delta = reinterpret_cast<const T*>(a.delta) + at.batch * a.delta_batch + at.channel0 + item_c;
    const T* const z = a.z ? reinterpret_cast<const T*>(a.z) + at.batch * a.z_batch + at.channel0 + item_c : nullptr;
    T* const out = reinterpret_cast<T*>(a.out) + at.batch * d.length * d.channels + at.channel0 + item_c;
    const T* const B = reinterpret_cast<const T*>(a.B) + at.batch * a.B_batch + at.group * a.B_group;
    const T* const C = reinterpret_cast<const T*>(a.C) + at.batch * a.C_batch + at.group * a.C_group;
    T* const slot = raw + tid * 8;                                       // u; delta and z follow a tile's elements later
    float skip[8], bias[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        skip[i] = a.D && i < item_valid ? a.D[at.channel0 + item_c + i] : 0.0f;
        bias[i] = a.delta_bias && i < item_valid ? a.delta_bias[at.channel0 + item_c + i] : 0.0f;
    }

    auto fetch = [&](int64_t t0, int buf) {
        const int64_t t = t0 + item_t;
        if (item_valid > 0 && t < t_used) {
            T* const to = slot + buf * 3 * STEPS * CH;
            fetch_pack<T, 8>(to, u + t * a.u_token, item_vec, item_valid);
            fetch_pack<T, 8>(to + STEPS * CH, delta + t * a.delta_token, item_vec, item_valid);
            if (!LOCAL && z) fetch_pack<T, 8>(to + 2 * STEPS * CH, z + t * a.z_token, item_vec, item_valid);
        }
#pragma unroll
        for (int k = 0; k < QN; ++k) {
            const int e = tid + k * THREADS, n = e % P * 4;
            const int64_t tt = t0 + e / P;
            if (e < QUADS && tt < t_used && n < states) {
                T* const to = raw_bc + buf * 2 * STEPS * NP + e * 4;
                const bool vec = d.vec_bc && n + 4 <= states;
                fetch_pack<T, 4>(to, B + tt * a.B_token + n, vec, states - n);
                if (!LOCAL) fetch_pack<T, 4>(to + STEPS * NP, C + tt * a.C_token + n, vec, states - n);
            }
        }
        copy_commit();
    };
    auto stage = [&](int64_t t0, int buf) {
        if (has_item) {
            const bool in = t0 + item_t < t_used;
            float x[8], dt[8];
            read_slot<T, 8>(slot + buf * 3 * STEPS * CH, x);
            read_slot<T, 8>(slot + (buf * 3 + 1) * STEPS * CH, dt);
            float4* const to = s_du + buf * DU + du_at<CH>(item_t, item_c);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                float e0, e1;
                dt[i] += bias[i];
                dt[i + 1] += bias[i + 1];
                if (d.softplus) softplus_pair(dt[i], dt[i + 1], e0, e1);
#pragma unroll
                for (int k = i; k < i + 2; ++k) {
                    // padding leaves the state as it is: dt = 0 makes the factor 1 and the addend 0
                    const float s = in && k < item_valid ? dt[k] : 0.0f, su = in && k < item_valid ? dt[k] * x[k] : 0.0f;
                    to[k] = make_float4(s, s, su, su);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < QN; ++k) {
            const int e = tid + k * THREADS;
            if (e < QUADS) {
                const bool in = t0 + e / P < t_used && e % P * 4 < states;
                float x[4];
                read_slot<T, 4>(raw_bc + buf * 2 * STEPS * NP + e * 4, x);
                const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                reinterpret_cast<float4*>(s_b + buf * STEPS * NP)[e] = in ? make_float4(x[0], x[1], x[2], x[3]) : zero;
                if (!LOCAL) {
                    read_slot<T, 4>(raw_bc + (buf * 2 + 1) * STEPS * NP + e * 4, x);
                    reinterpret_cast<float4*>(s_c + buf * STEPS * NP)[e] = in ? make_float4(x[0], x[1], x[2], x[3]) : zero;
                }
            }
        }
    };

    // padded states have A = B = C = 0
    const float4 A4 = load_states(a.A + channel * states, 4 * j, states, d.vec_states);
    const F2 A01 = pack2(A4.x * kLog2e, A4.y * kLog2e), A23 = pack2(A4.z * kLog2e, A4.w * kLog2e);
    F2 h01 = same2(0.0f), h23 = h01;
    if (t_begin < t_used) fetch(t_begin, 0);
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
            const F2 sum = same2(p.seg_dt[cell]);
            const float4 add = load_states(p.seg_state + cell * states, 4 * j, states, d.vec_states);
            h01 = fma2(decay(A01, sum), h01, pack2(add.x, add.y));
            h23 = fma2(decay(A23, sum), h23, pack2(add.z, add.w));
        }
    }
    float sum_dt = 0.0f;
    copy_wait();
    if (t_begin < t_used) stage(t_begin, 0);
    __syncthreads();

    int buf = 0;
    for (int64_t t0 = t_begin; t0 < t_used; t0 += STEPS, buf ^= 1) {
        const bool more = t0 + STEPS < t_used;
        if (more) fetch(t0 + STEPS, buf ^ 1);
        const float4* const du_row = s_du + buf * DU + du_at<CH>(0, c);
        const float4* const b_row = reinterpret_cast<const float4*>(s_b + buf * STEPS * NP) + j;
        const float4* const c_row = reinterpret_cast<const float4*>(s_c + buf * STEPS * NP) + j;
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
                const float4 du = du_row[t * (CH + CH / 8)], b = b_row[t * P];
                const F2 dt2 = pack2(du.x, du.y), du2 = pack2(du.z, du.w);
                h01 = fma2(decay(A01, dt2), h01, mul2(du2, pack2(b.x, b.y)));
                h23 = fma2(decay(A23, dt2), h23, mul2(du2, pack2(b.z, b.w)));
                if (LOCAL) {
                    sum_dt += du.x;
                } else {
                    const float4 cc = c_row[t * P];
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
        if (more) {
            copy_wait();
            stage(t0 + STEPS, buf ^ 1);
        }
        __syncthreads();
        if (!LOCAL && item_valid > 0 && t0 + item_t < t_end) {
            const int64_t t = t0 + item_t;
            const float* const y = s_y + (buf * STEPS + item_t) * ROW + item_c;
            float o[8], x[8], g[8];
            read_slot<T, 8>(slot + buf * 3 * STEPS * CH, x);
            if (z) read_slot<T, 8>(slot + (buf * 3 + 2) * STEPS * CH, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[i] = fmaf(skip[i], x[i], y[i]);
                if (z) o[i] *= silu(g[i]);
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
    if (item_valid > 0) {
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
template <typename T, int P>
struct BackShape {
    using S = Shape<P>;
    static constexpr int STEPS = kCheckpoint;
    static constexpr int WARPS = S::THREADS / 32;
    static constexpr int CHV = S::CH / 4;                                // 4 channels of one token per item
    static constexpr int ITEMS = STEPS * CHV;
    static constexpr int IPT = (ITEMS + S::THREADS - 1) / S::THREADS;
    static constexpr int ROW = S::ROW;
    // shared memory
    static constexpr size_t du = 0;                                                    // float4 [du_at]
    static constexpr size_t gy = du + sizeof(float4) * STEPS * (S::CH + S::CH / 8);    // float2 [STEPS][CH] (gy, gy)
    static constexpr size_t b = gy + sizeof(float2) * STEPS * S::CH;                   // float [STEPS][NP]
    static constexpr size_t c = b + sizeof(float) * STEPS * S::NP;
    static constexpr size_t y = c + sizeof(float) * STEPS * S::NP;                     // float [STEPS][ROW]: C . h
    static constexpr size_t s = y + sizeof(float) * STEPS * ROW;                       // float [2][STEPS][ROW]: gh . B, q . A / ln 2
    static constexpr size_t r = s + 2 * sizeof(float) * STEPS * ROW;                   // float [WARPS][STEPS][2][NP]: gC, gB
    static constexpr size_t keep = r + sizeof(float) * WARPS * STEPS * 2 * S::NP;      // float4 [2][STEPS][CH / 4]
    static constexpr size_t raw = keep + 2 * sizeof(float) * STEPS * S::CH;            // T [2][4][STEPS][CH]: u, delta, z, gout
    static constexpr size_t raw_bc = raw + 2 * 4 * sizeof(T) * STEPS * S::CH;          // T [2][STEPS][NP]
    static constexpr size_t bytes = raw_bc + 2 * sizeof(T) * STEPS * S::NP;
};

template <typename T, int P, bool LOCAL>
__global__ void __launch_bounds__(Shape<P>::THREADS) scan_backward(const __grid_constant__ ScanParams p) {
    using S = Shape<P>;
    using M = BackShape<T, P>;
    constexpr int THREADS = S::THREADS, CH = S::CH, NP = S::NP, STEPS = M::STEPS, ROW = M::ROW, WARPS = M::WARPS;
    constexpr int CHV = M::CHV, ITEMS = M::ITEMS, IPT = M::IPT;
    constexpr int QUADS = STEPS * P, QN = (QUADS + THREADS - 1) / THREADS;
    constexpr int R = 32 / P;                                            // channels of a warp
    extern __shared__ __align__(16) char smem[];
    float4* const s_du = reinterpret_cast<float4*>(smem + M::du);
    float2* const s_gy = reinterpret_cast<float2*>(smem + M::gy);
    float* const s_b = reinterpret_cast<float*>(smem + M::b);
    float* const s_c = reinterpret_cast<float*>(smem + M::c);
    float* const s_y = reinterpret_cast<float*>(smem + M::y);
    float* const s_s = reinterpret_cast<float*>(smem + M::s);
    float* const s_r = reinterpret_cast<float*>(smem + M::r);
    float4* const s_keep = reinterpret_cast<float4*>(smem + M::keep);    // derivative of dt by delta, of out by z / y
    T* const raw = reinterpret_cast<T*>(smem + M::raw);
    T* const raw_bc = reinterpret_cast<T*>(smem + M::raw_bc);

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

    float4 start;                                                        // the saved state in front of the tile
    auto item_of = [&](int k, int& t, int& cc, int& valid) {
        const int e = tid + k * THREADS;
        t = e / CHV;
        cc = (e % CHV) * 4;
        const int64_t left = at.n_channels - cc;
        valid = e >= ITEMS || left <= 0 ? 0 : left < 4 ? (int)left : 4;
    };
    auto slot_of = [&](int buf, int which, int k) { return raw + ((buf * 4 + which) * ITEMS + tid + k * THREADS) * 4; };
    auto fetch = [&](int64_t t0, int buf) {
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            int it, cc, valid;
            item_of(k, it, cc, valid);
            const int64_t t = t0 + it;
            if (valid > 0 && t < t_used) {
                const bool vec = d.vec && valid == 4;
                if (!LOCAL) fetch_pack<T, 4>(slot_of(buf, 0, k), u + t * a.u_token + cc, vec, valid);
                fetch_pack<T, 4>(slot_of(buf, 1, k), delta + t * a.delta_token + cc, vec, valid);
                if (z) fetch_pack<T, 4>(slot_of(buf, 2, k), z + t * a.z_token + cc, vec, valid);
                fetch_pack<T, 4>(slot_of(buf, 3, k), gout + t * a.gout_token + cc, vec, valid);
            }
        }
#pragma unroll
        for (int k = 0; k < QN; ++k) {
            const int e = tid + k * THREADS, n = e % P * 4;
            const int64_t t = t0 + e / P;
            if (e < QUADS && t < t_used && n < states) {
                const bool vec = d.vec_bc && n + 4 <= states;
                if (!LOCAL) fetch_pack<T, 4>(raw_bc + e * 4, B + t * a.B_token + n, vec, states - n);
                fetch_pack<T, 4>(raw_bc + STEPS * NP + e * 4, C + t * a.C_token + n, vec, states - n);
            }
        }
        copy_commit();
        if (!LOCAL && live)
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
    auto stage = [&](int64_t t0, int buf) {
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
            int it, cc, valid;
            item_of(k, it, cc, valid);
            if (tid + k * THREADS < ITEMS) {
                const bool in = t0 + it < t_used;
                float x[4], dt[4], zz[4], g[4], slope[4], gate_slope[4];
                if (!LOCAL) read_slot<T, 4>(slot_of(buf, 0, k), x);
                read_slot<T, 4>(slot_of(buf, 1, k), dt);
                if (z) read_slot<T, 4>(slot_of(buf, 2, k), zz);
                read_slot<T, 4>(slot_of(buf, 3, k), g);
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    dt[i] += bias[k][i];
                    dt[i + 1] += bias[k][i + 1];
                    if (d.softplus) {
                        const float x0 = dt[i], x1 = dt[i + 1];
                        float e0, e1;
                        softplus_pair(dt[i], dt[i + 1], e0, e1);
                        // the derivative 1 / (1 + e^-x) from e = e^-|x|
                        const float r0 = rcp_approx(1.0f + e0), r1 = rcp_approx(1.0f + e1);
                        slope[i] = x0 < 0.0f ? e0 * r0 : r0;
                        slope[i + 1] = x1 < 0.0f ? e1 * r1 : r1;
                    } else {
                        slope[i] = slope[i + 1] = 1.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool ok = in && i < valid;
                    gate_slope[i] = 0.0f;
                    if (z) {
                        const float sig = sigmoid(zz[i]), gate = zz[i] * sig;
                        gate_slope[i] = g[i] * fmaf(gate, 1.0f - sig, sig);
                        g[i] *= gate;
                    }
                    const float s = ok ? dt[i] : 0.0f, su = ok && !LOCAL ? dt[i] * x[i] : 0.0f, gy = ok ? g[i] : 0.0f;
                    s_du[du_at<CH>(it, cc + i)] = make_float4(s, s, su, su);
                    s_gy[it * CH + cc + i] = make_float2(gy, gy);
                }
                if (!LOCAL) {
                    s_keep[tid + k * THREADS] = make_float4(slope[0], slope[1], slope[2], slope[3]);
                    s_keep[ITEMS + tid + k * THREADS] = make_float4(gate_slope[0], gate_slope[1], gate_slope[2], gate_slope[3]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < QN; ++k) {
            const int e = tid + k * THREADS;
            if (e < QUADS) {
                const bool in = t0 + e / P < t_used && e % P * 4 < states;
                const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float x[4];
                if (!LOCAL) {
                    read_slot<T, 4>(raw_bc + e * 4, x);
                    reinterpret_cast<float4*>(s_b)[e] = in ? make_float4(x[0], x[1], x[2], x[3]) : zero;
                }
                read_slot<T, 4>(raw_bc + STEPS * NP + e * 4, x);
                reinterpret_cast<float4*>(s_c)[e] = in ? make_float4(x[0], x[1], x[2], x[3]) : zero;
            }
        }
    };

    // lanes without a channel have A = h = gh = 0: their sums over channels are zeros
    const float4 zero4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float4 A4 = live ? load_states(a.A + channel * states, 4 * j, states, d.vec_states) : zero4;
    const F2 A01 = pack2(A4.x * kLog2e, A4.y * kLog2e), A23 = pack2(A4.z * kLog2e, A4.w * kLog2e);
    F2 w01 = same2(0.0f), w23 = w01;                                     // a_{t+1} gh_{t+1}
    start = zero4;
    if (last >= first) fetch(last, 0);
    if (!LOCAL && live) {
        if (a.gfinal) {
            const float4 g = load_states(a.gfinal + (at.batch * d.channels + channel) * states, 4 * j, states, d.vec_states);
            w01 = pack2(g.x, g.y);
            w23 = pack2(g.z, g.w);
        }
        for (int64_t s = d.segments - 1; s > at.segment; --s) {
            const int64_t cell = (at.batch * d.segments + s) * d.channels + channel;
            const F2 sum = same2(p.seg_dt[cell]);
            const float4 add = load_states(p.seg_state + cell * states, 4 * j, states, d.vec_states);
            w01 = fma2(decay(A01, sum), w01, pack2(add.x, add.y));
            w23 = fma2(decay(A23, sum), w23, pack2(add.z, add.w));
        }
    }
    double gA[4] = {0.0, 0.0, 0.0, 0.0};
    float gD[IPT][4] = {}, gbias[IPT][4] = {};
    float sum_dt = 0.0f;
    const float4* const du_row = s_du + du_at<CH>(0, c);
    const float2* const gy_row = s_gy + c;
    const float4* const b_row = reinterpret_cast<const float4*>(s_b) + j;
    const float4* const c_row = reinterpret_cast<const float4*>(s_c) + j;

    int buf = 0;
    for (int64_t t0 = last; t0 >= first; t0 -= STEPS, buf ^= 1) {
        copy_wait();
        stage(t0, buf);
        F2 h01[STEPS + 1], h23[STEPS + 1], a01[STEPS], a23[STEPS];       // h[t] is the state in front of step t
        h01[0] = pack2(start.x, start.y);
        h23[0] = pack2(start.z, start.w);
        __syncthreads();
        if (t0 > first) fetch(t0 - STEPS, buf ^ 1);

        // the states again, forwards
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const float4 du = du_row[t * (CH + CH / 8)];
            const F2 dt2 = pack2(du.x, du.y);
            a01[t] = decay(A01, dt2);
            a23[t] = decay(A23, dt2);
            if (LOCAL) {
                sum_dt += du.x;
            } else {
                const float4 b = b_row[t * P];
                const F2 du2 = pack2(du.z, du.w);
                h01[t + 1] = fma2(a01[t], h01[t], mul2(du2, pack2(b.x, b.y)));
                h23[t + 1] = fma2(a23[t], h23[t], mul2(du2, pack2(b.z, b.w)));
            }
        }
        if (!LOCAL && z) {
            float y[STEPS];
#pragma unroll
            for (int t = 0; t < STEPS; ++t) {
                const float4 cc = c_row[t * P];
                y[t] = sum2(fma2(h23[t + 1], pack2(cc.z, cc.w), mul2(h01[t + 1], pack2(cc.x, cc.y))));
            }
            reduce_lanes<STEPS, P, 1>(y, lane);
            if (reduced_owner<STEPS, P>(j)) {
                const int t = reduced_index<STEPS, P>(j);
#pragma unroll
                for (int i = 0; i < reduced_count<STEPS, P>(); ++i) s_y[(t + i) * ROW + c] = y[i];
            }
        }
        // the gradients, backwards
        F2 gA01 = same2(0.0f), gA23 = gA01;
#pragma unroll
        for (int g = STEPS / 4 - 1; g >= 0; --g) {
            float s[8];
#pragma unroll
            for (int i = 3; i >= 0; --i) {
                const int t = g * 4 + i;
                const float2 gy = gy_row[t * CH];
                const F2 gy2 = pack2(gy.x, gy.y);
                const float4 cc = c_row[t * P];
                const F2 g01 = fma2(gy2, pack2(cc.x, cc.y), w01), g23 = fma2(gy2, pack2(cc.z, cc.w), w23);
                w01 = mul2(a01[t], g01);
                w23 = mul2(a23[t], g23);
                if (!LOCAL) {
                    const float4 du = du_row[t * (CH + CH / 8)], b = b_row[t * P];
                    const F2 dt2 = pack2(du.x, du.y), du2 = pack2(du.z, du.w);
                    float v[8];
                    unpack2(mul2(gy2, h01[t + 1]), v[0], v[1]);
                    unpack2(mul2(gy2, h23[t + 1]), v[2], v[3]);
                    unpack2(mul2(du2, g01), v[4], v[5]);
                    unpack2(mul2(du2, g23), v[6], v[7]);
                    reduce_lanes<8, R, P>(v, lane);
                    if (reduced_owner<8, R>(lane / P)) {
                        const int k0 = reduced_index<8, R>(lane / P);
                        float* const to = s_r + (warp * STEPS + t) * 2 * NP + 4 * j;
#pragma unroll
                        for (int k = 0; k < reduced_count<8, R>(); ++k) to[((k0 + k) / 4) * NP + (k0 + k) % 4] = v[k];
                    }
                    s[2 * i] = sum2(fma2(g23, pack2(b.z, b.w), mul2(g01, pack2(b.x, b.y))));
                    const F2 q01 = mul2(w01, h01[t]), q23 = mul2(w23, h23[t]);
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
                    float x[4], gu[4], gd[4], gz[4];
                    read_slot<T, 4>(slot_of(buf, 0, k), x);
                    const float4 over4 = *reinterpret_cast<const float4*>(s_s + it * ROW + cc);
                    const float4 qa4 = *reinterpret_cast<const float4*>(s_s + (STEPS + it) * ROW + cc);
                    const float4 slope4 = s_keep[tid + k * THREADS], gs4 = s_keep[ITEMS + tid + k * THREADS];
                    const float over[4] = {over4.x, over4.y, over4.z, over4.w}, qa[4] = {qa4.x, qa4.y, qa4.z, qa4.w};
                    const float slope[4] = {slope4.x, slope4.y, slope4.z, slope4.w}, gs[4] = {gs4.x, gs4.y, gs4.z, gs4.w};
                    float y[4] = {};
                    if (z) {
                        const float4 y4 = *reinterpret_cast<const float4*>(s_y + it * ROW + cc);
                        y[0] = y4.x, y[1] = y4.y, y[2] = y4.z, y[3] = y4.w;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float dt = s_du[du_at<CH>(it, cc + i)].x, gy = s_gy[it * CH + cc + i].x;
                        gu[i] = in ? fmaf(dt, over[i], skip[k][i] * gy) : 0.0f;
                        gd[i] = in ? slope[i] * fmaf(x[i], over[i], kLn2 * qa[i]) : 0.0f;
                        gz[i] = in ? gs[i] * fmaf(skip[k][i], x[i], y[i]) : 0.0f;
                        gD[k][i] += in ? gy * x[i] : 0.0f;
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
    constexpr size_t smem = ForwardSmem<T, P>::bytes;
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
    constexpr size_t smem = BackShape<T, P>::bytes;
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
    // 4 elements of B and C: 8 or 16 bytes
    p.d.vec_bc = a->states % 4 == 0 && aligned16(a->B) && aligned16(a->C) && multiple_of(4, a->B_batch, a->B_token) &&
                 multiple_of(4, a->C_batch, a->C_token) && a->B_group % 4 == 0 && a->C_group % 4 == 0;
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
