// Short causal convolution along the tokens, every channel by itself, for prompts and training (forward and backward)
// and for single tokens.  Interface: include/ovl_b200.h.
//
// What bounds it: bytes.  Every element is read once and written once; a few multiplications and one silu per element
// come with it.  A thread owns some channels (one wide load per token) and walks down a strip of tokens with the last
// taps - 1 inputs in registers, so an input is loaded once but for the taps - 1 tokens in front of the strip.
#include "ovl_sequence.cuh"

namespace ovl {
namespace {

constexpr int kMaxTaps = 8;
constexpr int kStrip = 32;             // tokens of a thread, forward
constexpr int kBackStrip = 64;         // tokens of a thread, backward
constexpr int kWarps = 4;              // warps of a block: strips that follow each other

struct ConvParams {
    OvlCausalConv a;
    int64_t column_tiles, strips;      // tiles of 32 x (channels of a thread) channels, blocks of kWarps strips
    int32_t vec;
    float* part;                       // backward: [batch * strips, taps + 1, channels]
};

__device__ __forceinline__ int64_t used_length(const int32_t* lengths, int64_t batch, int64_t length) {
    if (!lengths) return length;
    const int64_t n = lengths[batch];
    return n < 0 ? 0 : n > length ? length : n;
}

// A token in front of the first one comes from the state; `t` counts from the first token, -(taps - 1) is the oldest.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_token(const OvlCausalConv& a, int64_t batch, int64_t t, int64_t used, int64_t channel,
                                                 bool vec, int valid) {
    const T* x = reinterpret_cast<const T*>(a.x) + batch * a.x_batch + t * a.x_token + channel;
    bool in = t < used;
    if (t < 0) {
        x = reinterpret_cast<const T*>(a.initial_state) + (batch * (a.taps - 1) + (a.taps - 1) + t) * a.channels + channel;
        in = a.initial_state != nullptr && t >= 1 - a.taps;
    }
    return load_pack<T, N>(x, vec && in, in ? valid : 0);
}

// TAPS: the number of taps, or 8 for any number up to 8 (`taps` says which)
template <typename T, int TAPS>
__global__ void __launch_bounds__(32 * kWarps) conv_forward(const __grid_constant__ ConvParams p) {
    constexpr int N = 8, CHUNK = 8;
    const OvlCausalConv& a = p.a;
    const int taps = TAPS == kMaxTaps ? (int)a.taps : TAPS;
    int64_t i = blockIdx.x;
    const int64_t column = (i % p.column_tiles) * 32 + threadIdx.x % 32;
    i /= p.column_tiles;
    const int64_t strip = (i % p.strips) * kWarps + threadIdx.x / 32, batch = i / p.strips;
    const int64_t channel = column * N;
    if (channel >= a.channels) return;
    const int valid = a.channels - channel < N ? (int)(a.channels - channel) : N;
    const bool vec = p.vec && valid == N;
    const int64_t used = used_length(a.lengths, batch, a.length);
    const int64_t t_begin = strip * kStrip, t_end = t_begin + kStrip < a.length ? t_begin + kStrip : a.length;

    // the state after the sequence, by the thread that has the first strip
    if (strip == 0 && a.final_state) {
        for (int64_t k = 0; k < taps - 1; ++k) {
            const int64_t t = used - (taps - 1) + k;
            float x[N];
            const Pack<T, N> raw = load_token<T, N>(a, batch, t, used, channel, vec, valid);
#pragma unroll
            for (int c = 0; c < N; ++c) x[c] = to_f32(raw.v[c]);
            store_pack<T, N>(reinterpret_cast<T*>(a.final_state) + (batch * (taps - 1) + k) * a.channels + channel, x, vec, valid);
        }
    }
    if (t_begin >= t_end) return;

    // weights of the taps, the oldest first; with TAPS = 8 the unused ones in front stay out of the sum
    float w[TAPS][N], bias[N], win[TAPS][N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
        bias[c] = a.bias && c < valid ? load_param<T>(a.bias, channel + c, a.params_f32) : 0.0f;
#pragma unroll
        for (int k = 0; k < TAPS; ++k) {
            const int kk = k - (TAPS - taps);
            w[k][c] = kk >= 0 && c < valid ? load_param<T>(a.weight, (channel + c) * taps + kk, a.params_f32) : 0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < TAPS - 1; ++k) {
        const Pack<T, N> raw = load_token<T, N>(a, batch, t_begin - (TAPS - 1) + k, used, channel, vec, valid);
#pragma unroll
        for (int c = 0; c < N; ++c) win[k][c] = to_f32(raw.v[c]);
    }
    T* const out = reinterpret_cast<T*>(a.out) + batch * a.length * a.channels + channel;
    for (int64_t t0 = t_begin; t0 < t_end; t0 += CHUNK) {
        Pack<T, N> raw[CHUNK];
#pragma unroll
        for (int s = 0; s < CHUNK; ++s) raw[s] = load_token<T, N>(a, batch, t0 + s, used < t_end ? used : t_end, channel, vec, valid);
#pragma unroll
        for (int s = 0; s < CHUNK; ++s) {
            float y[N];
#pragma unroll
            for (int c = 0; c < N; ++c) {
                win[TAPS - 1][c] = to_f32(raw[s].v[c]);
                y[c] = bias[c];
#pragma unroll
                for (int k = 0; k < TAPS; ++k)
                    if (TAPS != kMaxTaps || k >= TAPS - taps) y[c] = fmaf(w[k][c], win[k][c], y[c]);
                if (a.silu) y[c] = silu(y[c]);
                if (t0 + s >= used) y[c] = 0.0f;
            }
            if (t0 + s < t_end) store_pack<T, N>(out + (t0 + s) * a.channels, y, vec, valid);
#pragma unroll
            for (int k = 0; k < TAPS - 1; ++k)
#pragma unroll
                for (int c = 0; c < N; ++c) win[k][c] = win[k + 1][c];
        }
    }
}

// gx_t = sum_k w[k] gpre_{t + (taps - 1) - k} with gpre = gout act'(pre): the walk runs taps - 1 tokens past the strip
// (gx of the strip needs them) and starts taps - 1 tokens in front of it.  The first strip walks from token 0 and also
// has the gradient of the initial state, gx of the tokens -(taps - 1) ... -1.
template <typename T, int TAPS>
__global__ void __launch_bounds__(32 * kWarps) conv_backward(const __grid_constant__ ConvParams p) {
    constexpr int N = 4, CHUNK = 4;
    const OvlCausalConv& a = p.a;
    const int taps = TAPS == kMaxTaps ? (int)a.taps : TAPS;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int64_t i = blockIdx.x;
    const int64_t column = (i % p.column_tiles) * 32 + lane;
    i /= p.column_tiles;
    const int64_t strip_block = i % p.strips, strip = strip_block * kWarps + warp, batch = i / p.strips;
    const int64_t channel = column * N;
    const bool live = channel < a.channels;
    const int valid = !live ? 0 : a.channels - channel < N ? (int)(a.channels - channel) : N;
    const bool vec = p.vec && valid == N;
    const int64_t used = used_length(a.lengths, batch, a.length);
    const int64_t t_begin = strip * kBackStrip, t_end = t_begin + kBackStrip < a.length ? t_begin + kBackStrip : a.length;

    float w[TAPS][N], bias[N], win[TAPS][N], gp[TAPS][N], gw[TAPS][N], gb[N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
        bias[c] = a.bias && c < valid ? load_param<T>(a.bias, channel + c, a.params_f32) : 0.0f;
        gb[c] = 0.0f;
#pragma unroll
        for (int k = 0; k < TAPS; ++k) {
            const int kk = k - (TAPS - taps);
            w[k][c] = kk >= 0 && c < valid ? load_param<T>(a.weight, (channel + c) * taps + kk, a.params_f32) : 0.0f;
            gw[k][c] = gp[k][c] = 0.0f;
        }
    }
    // A zero-length batch still has its state's gradient to hand on, so the first strip always walks.
    if (valid > 0 && (t_begin < t_end || strip == 0)) {
#pragma unroll
        for (int k = 0; k < TAPS - 1; ++k) {
            const Pack<T, N> raw = load_token<T, N>(a, batch, t_begin - (TAPS - 1) + k, used, channel, vec, valid);
#pragma unroll
            for (int c = 0; c < N; ++c) win[k][c] = to_f32(raw.v[c]);
        }
        const T* const gout = reinterpret_cast<const T*>(a.gout) + batch * a.gout_batch + channel;
        const int64_t walk_end = t_end + (taps - 1);                     // gx of token t is complete at t + taps - 1
        for (int64_t t0 = t_begin; t0 < walk_end; t0 += CHUNK) {
            Pack<T, N> raw[CHUNK], rawg[CHUNK];
#pragma unroll
            for (int s = 0; s < CHUNK; ++s) {
                const int64_t t = t0 + s;
                const bool in = t < walk_end && t < used;
                raw[s] = load_token<T, N>(a, batch, t, in ? used : 0, channel, vec, valid);
                rawg[s] = load_pack<T, N>(gout + t * a.gout_token, vec && in, in ? valid : 0);
            }
#pragma unroll
            for (int s = 0; s < CHUNK; ++s) {
                const int64_t t = t0 + s;
                float gx[N];
#pragma unroll
                for (int c = 0; c < N; ++c) {
                    win[TAPS - 1][c] = to_f32(raw[s].v[c]);
                    float g = to_f32(rawg[s].v[c]);
                    if (a.silu) {
                        float pre = bias[c];
#pragma unroll
                        for (int k = 0; k < TAPS; ++k)
                            if (TAPS != kMaxTaps || k >= TAPS - taps) pre = fmaf(w[k][c], win[k][c], pre);
                        const float sig = sigmoid(pre);
                        g *= sig * fmaf(pre, 1.0f - sig, 1.0f);
                    }
                    // outside the sequence nothing comes from above, whatever the input there
                    g = t < used ? g : 0.0f;
                    gp[TAPS - 1][c] = g;
                    if (t < t_end) {
                        gb[c] += g;
#pragma unroll
                        for (int k = 0; k < TAPS; ++k)
                            if (TAPS != kMaxTaps || k >= TAPS - taps) gw[k][c] = fmaf(g, t < used ? win[k][c] : 0.0f, gw[k][c]);
                    }
                    // gp[TAPS - 1 - k] is gpre of token t - k: gx of token t - (taps - 1)
                    gx[c] = 0.0f;
#pragma unroll
                    for (int k = 0; k < TAPS; ++k)
                        if (TAPS != kMaxTaps || k >= TAPS - taps) gx[c] = fmaf(w[k][c], gp[TAPS - 1 - (k - (TAPS - taps))][c], gx[c]);
                }
                const int64_t to = t - (taps - 1);
                const bool state = to < 0;
                if (t < walk_end && (state ? strip == 0 && a.ginitial != nullptr : to >= t_begin)) {
                    // the state after the sequence holds the inputs used - (taps - 1) ... used - 1
                    const int64_t k = to - (used - (taps - 1));
                    if (a.gfinal && k >= 0 && k < taps - 1) {
                        const Pack<T, N> g = load_pack<T, N>(
                            reinterpret_cast<const T*>(a.gfinal) + (batch * (taps - 1) + k) * a.channels + channel, vec, valid);
#pragma unroll
                        for (int c = 0; c < N; ++c) gx[c] += to_f32(g.v[c]);
                    }
                    T* const dst = state ? reinterpret_cast<T*>(a.ginitial) + (batch * (taps - 1) + (taps - 1) + to) * a.channels
                                         : reinterpret_cast<T*>(a.gx) + (batch * a.length + to) * a.channels;
                    store_pack<T, N>(dst + channel, gx, vec, valid);
                }
#pragma unroll
                for (int k = 0; k < TAPS - 1; ++k)
#pragma unroll
                    for (int c = 0; c < N; ++c) {
                        win[k][c] = win[k + 1][c];
                        gp[k][c] = gp[k + 1][c];
                    }
            }
        }
    }
    // the warps' sums for the weights and the bias, added up in warp order
    __shared__ float s_part[kWarps][(TAPS + 1) * N][32];
#pragma unroll
    for (int c = 0; c < N; ++c) {
#pragma unroll
        for (int k = 0; k < TAPS; ++k) s_part[warp][k * N + c][lane] = gw[k][c];
        s_part[warp][TAPS * N + c][lane] = gb[c];
    }
    __syncthreads();
    const int64_t row = batch * p.strips + strip_block;
    for (int e = threadIdx.x; e < (TAPS + 1) * N * 32; e += 32 * kWarps) {
        const int cc = e % (N * 32), k = e / (N * 32) - (TAPS - taps);
        const int64_t ch = (blockIdx.x % p.column_tiles) * 32 * N + cc;
        if (k < 0 || ch >= a.channels) continue;
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < kWarps; ++s) sum += s_part[s][(e / (N * 32)) * N + cc % N][cc / N];
        p.part[(row * (taps + 1) + k) * a.channels + ch] = sum;
    }
}

// the strips' parts added up in order
template <typename T>
__global__ void conv_backward_params(const __grid_constant__ ConvParams p) {
    const OvlCausalConv& a = p.a;
    const int64_t total = (a.taps + 1) * a.channels, rows = a.batch * p.strips;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t k = i / a.channels, ch = i % a.channels;
        float sum = 0.0f;
        for (int64_t r = 0; r < rows; ++r) sum += p.part[r * total + i];
        void* const to = k < a.taps ? a.gweight : a.gbias;
        const int64_t at = k < a.taps ? ch * a.taps + k : ch;
        if (!to) continue;
        if (a.params_f32) reinterpret_cast<float*>(to)[at] = sum;
        else reinterpret_cast<T*>(to)[at] = from_f32<T>(sum);
    }
}

template <typename T, int TAPS>
__global__ void __launch_bounds__(128) conv_step(const __grid_constant__ OvlCausalConvStep a, int64_t blocks_per_row, int vec_ok) {
    constexpr int N = 2;
    const int taps = TAPS == kMaxTaps ? (int)a.taps : TAPS;
    const int64_t row = blockIdx.x / blocks_per_row;
    const int64_t channel = ((blockIdx.x % blocks_per_row) * 128 + threadIdx.x) * N;
    const int valid = channel >= a.channels ? 0 : a.channels - channel < N ? (int)(a.channels - channel) : N;
    const bool vec = vec_ok && valid == N;
    T* const out = reinterpret_cast<T*>(a.out) + row * a.channels + channel;
    int64_t slot = row;
    if (a.slot_of_row) {
        slot = a.slot_of_row[row];
        int taken = 0;
        for (int64_t r = threadIdx.x; r < row; r += 128) taken |= slot >= 0 && a.slot_of_row[r] == slot;
        taken = __syncthreads_or(taken);
        if (slot < 0 || slot >= a.slots || taken) {
            const float nan = __int_as_float(0x7fffffff);
            const float y[N] = {slot < 0 ? 0.0f : nan, slot < 0 ? 0.0f : nan};
            if (valid > 0) store_pack<T, N>(out, y, vec, valid);
            return;
        }
    }
    if (valid == 0) return;
    T* const state = reinterpret_cast<T*>(a.state) + slot * (taps - 1) * a.channels + channel;
    float x[TAPS][N], y[N];
#pragma unroll
    for (int k = 0; k < TAPS; ++k) {
        const int kk = k - (TAPS - taps);
        if (kk < 0) continue;
        const Pack<T, N> raw = k == TAPS - 1 ? load_pack<T, N>(reinterpret_cast<const T*>(a.x) + row * a.x_row + channel, vec, valid)
                                             : load_pack<T, N>(state + kk * a.channels, vec, valid);
#pragma unroll
        for (int c = 0; c < N; ++c) x[k][c] = to_f32(raw.v[c]);
    }
#pragma unroll
    for (int c = 0; c < N; ++c) {
        y[c] = a.bias && c < valid ? load_param<T>(a.bias, channel + c, a.params_f32) : 0.0f;
#pragma unroll
        for (int k = 0; k < TAPS; ++k) {
            const int kk = k - (TAPS - taps);
            if (kk >= 0 && c < valid) y[c] = fmaf(load_param<T>(a.weight, (channel + c) * taps + kk, a.params_f32), x[k][c], y[c]);
        }
        if (a.silu) y[c] = silu(y[c]);
    }
#pragma unroll
    for (int k = 1; k < TAPS; ++k) {
        const int kk = k - (TAPS - taps);
        if (kk >= 1) store_pack<T, N>(state + (kk - 1) * a.channels, x[k], vec, valid);
    }
    store_pack<T, N>(out, y, vec, valid);
}

// ---------------------------------------------------------------------------------------------------------
// host side

int check(const OvlCausalConv* a) {
    if (!a) return OVL_ERR_NULL;
    if (a->dtype != OVL_FLOAT32 && a->dtype != OVL_FLOAT16 && a->dtype != OVL_BFLOAT16) return OVL_ERR_DTYPE;
    if (a->batch < 0 || a->length < 0 || a->channels < 1 || a->taps < 1) return OVL_ERR_INVALID;
    if (a->taps > kMaxTaps) return OVL_ERR_TOO_LARGE;
    return OVL_OK;
}

int64_t strip_blocks(const OvlCausalConv* a, int strip) {
    const int64_t n = ceil_div(a->length, (int64_t)strip * kWarps);
    return n > 0 ? n : 1;                                                // states without tokens are passed on too
}

bool wide(const OvlCausalConv* a, int n, bool backward) {
    bool ok = a->channels % n == 0 && aligned16(a->x) && a->x_batch % n == 0 && a->x_token % n == 0 && aligned16(a->initial_state);
    if (!backward) return ok && aligned16(a->out) && aligned16(a->final_state);
    return ok && aligned16(a->gout) && a->gout_batch % n == 0 && a->gout_token % n == 0 && aligned16(a->gfinal) &&
           aligned16(a->gx) && aligned16(a->ginitial);
}

template <typename T>
int run_forward(ConvParams p, cudaStream_t stream) {
    p.column_tiles = ceil_div(p.a.channels, 32 * 8);
    p.strips = strip_blocks(&p.a, kStrip);
    p.vec = wide(&p.a, 8, false);
    const int64_t blocks = p.column_tiles * p.strips * p.a.batch;
    if (blocks > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    const uint32_t grid = (uint32_t)blocks;
    switch (p.a.taps) {
        case 2: conv_forward<T, 2><<<grid, 32 * kWarps, 0, stream>>>(p); break;
        case 3: conv_forward<T, 3><<<grid, 32 * kWarps, 0, stream>>>(p); break;
        case 4: conv_forward<T, 4><<<grid, 32 * kWarps, 0, stream>>>(p); break;
        default: conv_forward<T, kMaxTaps><<<grid, 32 * kWarps, 0, stream>>>(p); break;
    }
    return launch_status();
}

template <typename T>
int run_backward(ConvParams p, cudaStream_t stream) {
    p.column_tiles = ceil_div(p.a.channels, 32 * 4);
    p.strips = strip_blocks(&p.a, kBackStrip);
    p.vec = wide(&p.a, 4, true);
    p.part = reinterpret_cast<float*>(p.a.workspace);
    const int64_t blocks = p.column_tiles * p.strips * p.a.batch;
    if (blocks > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    const uint32_t grid = (uint32_t)blocks;
    switch (p.a.taps) {
        case 2: conv_backward<T, 2><<<grid, 32 * kWarps, 0, stream>>>(p); break;
        case 3: conv_backward<T, 3><<<grid, 32 * kWarps, 0, stream>>>(p); break;
        case 4: conv_backward<T, 4><<<grid, 32 * kWarps, 0, stream>>>(p); break;
        default: conv_backward<T, kMaxTaps><<<grid, 32 * kWarps, 0, stream>>>(p); break;
    }
    const int st = launch_status();
    if (st != OVL_OK) return st;
    conv_backward_params<T><<<(uint32_t)ceil_div((p.a.taps + 1) * p.a.channels, 128), 128, 0, stream>>>(p);
    return launch_status();
}

template <typename T>
int run_step(const OvlCausalConvStep& a, cudaStream_t stream) {
    const int64_t per_row = ceil_div(a.channels, 128 * 2), blocks = per_row * a.rows;
    if (blocks > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    const uint32_t grid = (uint32_t)blocks;
    const int vec = a.channels % 2 == 0 && a.x_row % 2 == 0 && aligned16(a.x) && aligned16(a.state) && aligned16(a.out);
    switch (a.taps) {
        case 2: conv_step<T, 2><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
        case 3: conv_step<T, 3><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
        case 4: conv_step<T, 4><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
        default: conv_step<T, kMaxTaps><<<grid, 128, 0, stream>>>(a, per_row, vec); break;
    }
    return launch_status();
}

}  // namespace
}  // namespace ovl

extern "C" uint64_t ovl_causal_conv_workspace_bytes(const OvlCausalConv* a) {
    if (ovl::check(a) != OVL_OK) return 0;
    return (uint64_t)a->batch * ovl::strip_blocks(a, ovl::kBackStrip) * (a->taps + 1) * a->channels * sizeof(float);
}

extern "C" int ovl_causal_conv(const OvlCausalConv* a, void* cuda_stream) {
    const int st = ovl::check(a);
    if (st != OVL_OK) return st;
    if (a->batch == 0) return OVL_OK;
    if (!a->weight || (a->length > 0 && (!a->x || !a->out))) return OVL_ERR_NULL;
    ovl::ConvParams p{};
    p.a = *a;
    const cudaStream_t stream = (cudaStream_t)cuda_stream;
    if (a->dtype == OVL_FLOAT32) return ovl::run_forward<float>(p, stream);
    if (a->dtype == OVL_FLOAT16) return ovl::run_forward<__half>(p, stream);
    return ovl::run_forward<__nv_bfloat16>(p, stream);
}

extern "C" int ovl_causal_conv_backward(const OvlCausalConv* a, void* cuda_stream) {
    const int st = ovl::check(a);
    if (st != OVL_OK) return st;
    if (a->batch == 0) return OVL_OK;
    if (!a->weight || !a->gweight || (a->length > 0 && (!a->x || !a->gout || !a->gx))) return OVL_ERR_NULL;
    if (!a->workspace || a->workspace_bytes < ovl_causal_conv_workspace_bytes(a) || !ovl::aligned16(a->workspace)) return OVL_ERR_SCRATCH;
    ovl::ConvParams p{};
    p.a = *a;
    const cudaStream_t stream = (cudaStream_t)cuda_stream;
    if (a->dtype == OVL_FLOAT32) return ovl::run_backward<float>(p, stream);
    if (a->dtype == OVL_FLOAT16) return ovl::run_backward<__half>(p, stream);
    return ovl::run_backward<__nv_bfloat16>(p, stream);
}

extern "C" int ovl_causal_conv_step(const OvlCausalConvStep* a, void* cuda_stream) {
    if (!a) return OVL_ERR_NULL;
    if (a->dtype != OVL_FLOAT32 && a->dtype != OVL_FLOAT16 && a->dtype != OVL_BFLOAT16) return OVL_ERR_DTYPE;
    if (a->rows < 0 || a->channels < 1 || a->taps < 1 || a->slots < 0) return OVL_ERR_INVALID;
    if (!a->slot_of_row && a->slots < a->rows) return OVL_ERR_INVALID;
    if (a->taps > ovl::kMaxTaps) return OVL_ERR_TOO_LARGE;
    if (a->rows == 0) return OVL_OK;
    if (!a->x || !a->weight || !a->out || (!a->state && a->slots > 0 && a->taps > 1)) return OVL_ERR_NULL;
    const cudaStream_t stream = (cudaStream_t)cuda_stream;
    if (a->dtype == OVL_FLOAT32) return ovl::run_step<float>(*a, stream);
    if (a->dtype == OVL_FLOAT16) return ovl::run_step<__half>(*a, stream);
    return ovl::run_step<__nv_bfloat16>(*a, stream);
}
