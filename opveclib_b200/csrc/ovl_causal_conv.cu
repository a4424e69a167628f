// Short causal convolution along the tokens, every channel by itself, for prompts and training (forward and backward)
// and for single tokens.  Interface: include/ovl_b200.h.
//
// What bounds it: bytes.  Every element is read once and written once; a few multiplications and one silu per element
// come with it.  A thread owns some channels (one wide load per token) and walks down a strip of tokens with the last
// taps - 1 inputs in registers, so an input is loaded once but for the taps - 1 tokens in front of the strip.
#include "ovl_sequence.cuh"

#include <type_traits>

namespace ovl {
namespace {

constexpr int kMaxTaps = 8;
constexpr int kMinStrip = 8, kMaxStrip = 128;   // tokens of a thread
constexpr int kForward = 8, kBackward = 4;   // channels of a thread
constexpr int kWarps = 4;              // warps of a block: strips that follow each other

struct ConvParams {
    OvlCausalConv a;
    int64_t column_tiles, strips;      // tiles of 32 x (channels of a thread) channels, blocks of kWarps strips
    int64_t strip;                     // tokens of a thread
    int32_t vec, width;                // whole packs on their boundaries; else runs of `width` elements
    float* part;                       // backward: [batch * strips, taps + 1, channels]
};

__device__ __forceinline__ int64_t used_length(const int32_t* lengths, int64_t batch, int64_t length) {
    if (!lengths) return length;
    const int64_t n = lengths[batch];
    return n < 0 ? 0 : n > length ? length : n;
}

// Which N channels a thread has: in runs of W, those of a warp's lanes next to each other, run after run.  W = N: a pack
// of its own, on its boundary.  Where rows of packs do not begin on boundaries, short runs keep what a warp touches with
// one instruction together (fp32, 1 x 2290 x 1705, forward: 14.1 us against 30.1 with 8 channels in a row for each lane,
// fetched one by one).
template <int W>
__device__ __forceinline__ constexpr int channel_of(int c) { return c / W * 32 * W + c % W; }
template <int W>
__device__ __forceinline__ int valid_channels(int64_t left, int n) {     // of the channels that are left from the thread's first
    int valid = 0;
    for (int c = 0; c < n; ++c) valid += channel_of<W>(c) < left;
    return valid;
}

template <typename T, int N, int W>
__device__ __forceinline__ Pack<T, N> load_channels(const T* __restrict__ p, int valid) {
    if constexpr (W == N) {
        return load_pack<T, N>(p, valid > 0, 0);
    } else {
        Pack<T, N> r;
#pragma unroll
        for (int c = 0; c < N; ++c) r.v[c] = c < valid ? p[channel_of<W>(c)] : from_f32<T>(0.0f);
        return r;
    }
}
template <typename T, int N, int W>
__device__ __forceinline__ void store_channels(T* __restrict__ p, const float (&x)[N], int valid) {
    if constexpr (W == N) {
        store_pack<T, N>(p, x, true, N);
    } else {
#pragma unroll
        for (int c = 0; c < N; c += W) {
            Pack<T, W> r;
#pragma unroll
            for (int k = 0; k < W; ++k) r.v[k] = from_f32<T>(x[c + k]);
            if (c < valid) *reinterpret_cast<Pack<T, W>*>(p + channel_of<W>(c)) = r;
        }
    }
}
// A token in front of the first one comes from the state; `t` counts from the first token, -(taps - 1) is the oldest.
template <typename T, int N, int W>
__device__ __forceinline__ Pack<T, N> load_token(const OvlCausalConv& a, int64_t batch, int64_t t, int64_t used, int64_t channel, int valid) {
    const T* x = reinterpret_cast<const T*>(a.x) + batch * a.x_batch + t * a.x_token + channel;
    bool in = t < used;
    if (t < 0) {
        x = reinterpret_cast<const T*>(a.initial_state) + (batch * (a.taps - 1) + (a.taps - 1) + t) * a.channels + channel;
        in = a.initial_state != nullptr && t >= 1 - a.taps;
    }
    return load_channels<T, N, W>(x, in ? valid : 0);
}

// The weights of a thread's N channels as pairs of channels, the oldest tap first; with TAPS = 8 the unused ones in front
// are zeros, which the sums leave out.
template <typename T, int TAPS, int N, int W>
__device__ __forceinline__ void load_weights(F2 (&w)[TAPS][N / 2], F2 (&bias)[N / 2], const OvlCausalConv& a, int taps, int64_t channel,
                                             int valid) {
    float v[TAPS][N], b[N];
    if (W == N && TAPS != kMaxTaps && !a.params_f32 && valid == N && aligned16(a.weight) && (N * TAPS * sizeof(T)) % 16 == 0 && channel % N == 0) {
        const Pack<T, N * TAPS> raw = load_pack<T, N * TAPS>(reinterpret_cast<const T*>(a.weight) + channel * TAPS, true, 0);
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int k = 0; k < TAPS; ++k) v[k][c] = to_f32(raw.v[c * TAPS + k]);
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int k = 0; k < TAPS; ++k) {
                const int kk = k - (TAPS - taps);
                v[k][c] = kk >= 0 && c < valid ? load_param<T>(a.weight, (channel + channel_of<W>(c)) * taps + kk, a.params_f32) : 0.0f;
            }
    }
#pragma unroll
    for (int c = 0; c < N; ++c) b[c] = a.bias && c < valid ? load_param<T>(a.bias, channel + channel_of<W>(c), a.params_f32) : 0.0f;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        bias[i] = pack2(b[2 * i], b[2 * i + 1]);
#pragma unroll
        for (int k = 0; k < TAPS; ++k) w[k][i] = pack2(v[k][2 * i], v[k][2 * i + 1]);
    }
}

template <typename T, int N>
__device__ __forceinline__ void widen(F2 (&x)[N / 2], const Pack<T, N>& raw) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) x[i] = pack2(to_f32(raw.v[2 * i]), to_f32(raw.v[2 * i + 1]));
}

__device__ __forceinline__ float half_of(uint32_t word, uint32_t upper, __half) {
    return __half2float(__ushort_as_half((unsigned short)(word >> 16 * upper)));
}
__device__ __forceinline__ float half_of(uint32_t word, uint32_t upper, __nv_bfloat16) {
    return __bfloat162float(__ushort_as_bfloat16((unsigned short)(word >> 16 * upper)));
}

// Tokens on their way while earlier ones are worked on: every thread copies what it will need itself into slots of its
// own, so nothing waits but the thread that needs a token (a register that a load may or may not fill is waited for at
// once: 197 us for the forward pass of bf16 4 x 4096 x 4096 with the next tokens in registers).
constexpr int kChunk = 4;              // tokens that are copied and worked on together
constexpr int kAhead = 3;              // chunks on their way
constexpr int kRing = kAhead + 1;

struct True {
    static constexpr bool value = true;
};
struct False {
    static constexpr bool value = false;
};

// Packs stand in the slots as they are.  Runs are copied by words of 4 bytes, a thread's words a block's width apart (next
// to each other they would meet in the same banks): pairs of 16-bit elements, or, for single ones, which no asynchronous
// copy takes, the aligned word with the element in one of its halves.  A word with an element in it is memory of the
// tensor's allocation, whose boundaries are far coarser.  bf16 8 x 2048 x 4095, forward and backward: 97 and 170 us; with
// a thread's words next to each other 138 and 223; with loads into registers that go to the slot at once 142 and 277.
template <typename T, int N, int W>
struct Ring {
    static constexpr bool kPacks = W == N;
    using Slot = std::conditional_t<kPacks, T, uint32_t>;
    static constexpr int kOfWord = sizeof(T) * W == 4 ? W : 1;           // channels of a word
    static constexpr int kSize = kPacks ? N : N / kOfWord, kStep = 32 * kWarps;
    static constexpr size_t bytes = sizeof(Slot) * kRing * kChunk * 32 * kWarps * kSize;
    Slot* base;                        // [kRing][kChunk] of: packs [threads][N], or words [kSize][threads]
    __device__ __forceinline__ explicit Ring(void* smem) : base(reinterpret_cast<Slot*>(smem) + threadIdx.x * (kPacks ? N : 1)) {}
    __device__ __forceinline__ Slot* slot(int chunk, int s) const { return base + (chunk * kChunk + s) * (32 * kWarps * kSize); }

    // into a slot of the thread's own, in flight while it goes on
    static __device__ __forceinline__ void fetch(Slot* slot, const T* __restrict__ p, int valid) {
        if constexpr (kPacks) {
            fetch_pack<T, N>(slot, p, true, N, 0);
        } else {
#pragma unroll
            for (int k = 0; k < kSize; ++k) {
                const T* const from = p + channel_of<W>(k * kOfWord);
                if (k * kOfWord < valid) copy_async<4>(slot + k * kStep, reinterpret_cast<const void*>((uintptr_t)from & ~(uintptr_t)3));
                else slot[k * kStep] = 0;
            }
        }
    }
    // `upper`: which half of its word a single element of 16 bits is in
    static __device__ __forceinline__ void widen(F2 (&x)[N / 2], const Slot* slot, uint32_t upper) {
        float v[N];
        if constexpr (kPacks) {
            read_slot<T, N>(slot, v);
        } else {
#pragma unroll
            for (int c = 0; c < N; ++c) {
                const uint32_t word = slot[c / kOfWord * kStep];
                if constexpr (sizeof(T) == 4) v[c] = __uint_as_float(word);
                else v[c] = half_of(word, kOfWord == 2 ? c % 2 : upper, T{});
            }
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) x[i] = pack2(v[2 * i], v[2 * i + 1]);
    }
};

// TAPS: the number of taps, or 8 for any number up to 8 (`taps` says which); W: see channel_of
template <typename T, int TAPS, int W>
__global__ void __launch_bounds__(32 * kWarps, TAPS == kMaxTaps ? 1 : 4) conv_forward(const __grid_constant__ ConvParams p) {
    constexpr int N = kForward, CHUNK = kChunk;
    constexpr bool FULL = W == N;
    extern __shared__ __align__(16) char smem[];
    const OvlCausalConv& a = p.a;
    const int taps = TAPS == kMaxTaps ? (int)a.taps : TAPS;
    int64_t i = blockIdx.x;
    const int64_t channel = (i % p.column_tiles) * 32 * N + threadIdx.x % 32 * W;
    i /= p.column_tiles;
    const int64_t strip = (i % p.strips) * kWarps + threadIdx.x / 32, batch = i / p.strips;
    if (channel >= a.channels) return;
    const int valid = FULL ? N : valid_channels<W>(a.channels - channel, N);
    const int64_t used = used_length(a.lengths, batch, a.length);
    const int64_t t_begin = strip * p.strip, t_end = t_begin + p.strip < a.length ? t_begin + p.strip : a.length;
    const int64_t t_used = used < t_end ? used : t_end;

    // the state after the sequence, by the thread that has the first strip
    if (strip == 0 && a.final_state) {
        for (int64_t k = 0; k < taps - 1; ++k) {
            const int64_t t = used - (taps - 1) + k;
            float x[N];
            const Pack<T, N> raw = load_token<T, N, W>(a, batch, t, used, channel, valid);
#pragma unroll
            for (int c = 0; c < N; ++c) x[c] = to_f32(raw.v[c]);
            store_channels<T, N, W>(reinterpret_cast<T*>(a.final_state) + (batch * (taps - 1) + k) * a.channels + channel, x, valid);
        }
    }
    if (t_begin >= t_end) return;

    const T* const x = reinterpret_cast<const T*>(a.x) + batch * a.x_batch + channel;
    T* const out = reinterpret_cast<T*>(a.out) + batch * a.length * a.channels + channel;
    using Tokens = Ring<T, N, W>;
    using Slot = typename Tokens::Slot;
    const Tokens ring(smem);
    const uint32_t x_at = (uint32_t)((uintptr_t)x / sizeof(T));        // which halves of words the thread's elements are in
    const T* next = x + t_begin * a.x_token;                             // of the next chunk to be fetched
    auto fetch = [&](int64_t t0, int chunk) {
        if (FULL && t0 + CHUNK <= t_used) {
#pragma unroll
            for (int s = 0; s < CHUNK; ++s) Tokens::fetch(ring.slot(chunk, s), next + s * a.x_token, N);
        } else {
#pragma unroll
            for (int s = 0; s < CHUNK; ++s)
                if (t0 + s < t_used) Tokens::fetch(ring.slot(chunk, s), next + s * a.x_token, valid);
        }
        next += CHUNK * a.x_token;
        copy_commit();
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch(t_begin + k * CHUNK, k);
    F2 w[TAPS][N / 2], bias[N / 2], win[TAPS][N / 2];
    load_weights<T, TAPS, N, W>(w, bias, a, taps, channel, valid);
#pragma unroll
    for (int k = 0; k < TAPS - 1; ++k)
        widen<T, N>(win[k], load_token<T, N, W>(a, batch, t_begin - (TAPS - 1) + k, used, channel, valid));
    const bool gated = a.silu;
    int chunk = 0;
    T* out_t = out + t_begin * a.channels;
    // one token; INSIDE: it belongs to the strip and the sequence
    auto token = [&](int64_t t, const Slot* slot, auto inside) {
        constexpr bool INSIDE = decltype(inside)::value;
        Tokens::widen(win[TAPS - 1], slot, (x_at + (uint32_t)t * (uint32_t)a.x_token) & 1);   // (behind the sequence: anything, and not used)
        float y[N];
#pragma unroll
        for (int c = 0; c < N / 2; ++c) {
            F2 sum = bias[c];
#pragma unroll
            for (int k = 0; k < TAPS; ++k)
                if (TAPS != kMaxTaps || k >= TAPS - taps) sum = fma2(w[k][c], win[k][c], sum);
            if (gated) sum = silu2(sum);
            unpack2(sum, y[2 * c], y[2 * c + 1]);
        }
        if (!INSIDE && t >= used) {
#pragma unroll
            for (int c = 0; c < N; ++c) y[c] = 0.0f;
        }
        if (INSIDE || t < t_end) store_channels<T, N, W>(out_t, y, valid);
        out_t += a.channels;
#pragma unroll
        for (int k = 0; k < TAPS - 1; ++k)
#pragma unroll
            for (int c = 0; c < N / 2; ++c) win[k][c] = win[k + 1][c];
    };
    for (int64_t t0 = t_begin; t0 < t_end; t0 += CHUNK) {
        copy_wait<kAhead - 1>();
        fetch(t0 + kAhead * CHUNK, chunk == 0 ? kAhead : chunk - 1);
        if (t0 + CHUNK <= t_used) {
#pragma unroll
            for (int s = 0; s < CHUNK; ++s) token(t0 + s, ring.slot(chunk, s), True{});
        } else {
#pragma unroll
            for (int s = 0; s < CHUNK; ++s) token(t0 + s, ring.slot(chunk, s), False{});
        }
        chunk = chunk == kAhead ? 0 : chunk + 1;
    }
}

// gx_t = sum_k w[k] gpre_{t + (taps - 1) - k} with gpre = gout act'(pre): the walk runs taps - 1 tokens past the strip
// (gx of the strip needs them).  The first strip also has the gradient of the initial state, gx of the tokens
// -(taps - 1) ... -1.
template <typename T, int TAPS, int W>
__global__ void __launch_bounds__(32 * kWarps, TAPS == kMaxTaps ? 1 : 4) conv_backward(const __grid_constant__ ConvParams p) {
    constexpr int N = kBackward, CHUNK = kChunk;
    constexpr bool FULL = W == N;
    extern __shared__ __align__(16) char smem[];
    const OvlCausalConv& a = p.a;
    const int taps = TAPS == kMaxTaps ? (int)a.taps : TAPS;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int64_t i = blockIdx.x;
    const int64_t channel = (i % p.column_tiles) * 32 * N + lane * W;
    i /= p.column_tiles;
    const int64_t strip_block = i % p.strips, strip = strip_block * kWarps + warp, batch = i / p.strips;
    const int valid = channel >= a.channels ? 0 : FULL ? N : valid_channels<W>(a.channels - channel, N);
    const int64_t used = used_length(a.lengths, batch, a.length);
    const int64_t t_begin = strip * p.strip, t_end = t_begin + p.strip < a.length ? t_begin + p.strip : a.length;

    F2 w[TAPS][N / 2], bias[N / 2], win[TAPS][N / 2], gp[TAPS][N / 2], gw[TAPS][N / 2], gb[N / 2];
#pragma unroll
    for (int c = 0; c < N / 2; ++c) {
        gb[c] = same2(0.0f);
#pragma unroll
        for (int k = 0; k < TAPS; ++k) gw[k][c] = gp[k][c] = same2(0.0f);
    }
    // A sequence without tokens still has its state's gradient to hand on, so the first strip always walks.
    if (valid > 0 && (t_begin < t_end || strip == 0)) {
        const int64_t walk_end = t_end + (taps - 1);                     // gx of token t is complete at t + taps - 1
        const int64_t walk_used = used < walk_end ? used : walk_end;
        const T* const x = reinterpret_cast<const T*>(a.x) + batch * a.x_batch + channel;
        const T* const gout = reinterpret_cast<const T*>(a.gout) + batch * a.gout_batch + channel;
        using Tokens = Ring<T, N, W>;
        using Slot = typename Tokens::Slot;
        const Tokens ring_x(smem), ring_g(smem + Tokens::bytes);
        const uint32_t x_at = (uint32_t)((uintptr_t)x / sizeof(T)), g_at = (uint32_t)((uintptr_t)gout / sizeof(T));
        const T* next_x = x + t_begin * a.x_token;                       // of the next chunk to be fetched
        const T* next_g = gout + t_begin * a.gout_token;
        auto fetch = [&](int64_t t0, int chunk) {
            if (FULL && t0 + CHUNK <= walk_used) {
#pragma unroll
                for (int s = 0; s < CHUNK; ++s) {
                    Tokens::fetch(ring_x.slot(chunk, s), next_x + s * a.x_token, N);
                    Tokens::fetch(ring_g.slot(chunk, s), next_g + s * a.gout_token, N);
                }
            } else {
#pragma unroll
                for (int s = 0; s < CHUNK; ++s) {
                    if (t0 + s < walk_used) {
                        Tokens::fetch(ring_x.slot(chunk, s), next_x + s * a.x_token, valid);
                        Tokens::fetch(ring_g.slot(chunk, s), next_g + s * a.gout_token, valid);
                    }
                }
            }
            next_x += CHUNK * a.x_token;
            next_g += CHUNK * a.gout_token;
            copy_commit();
        };
#pragma unroll
        for (int k = 0; k < kAhead; ++k) fetch(t_begin + k * CHUNK, k);
        load_weights<T, TAPS, N, W>(w, bias, a, taps, channel, valid);
#pragma unroll
        for (int k = 0; k < TAPS - 1; ++k)
            widen<T, N>(win[k], load_token<T, N, W>(a, batch, t_begin - (TAPS - 1) + k, used, channel, valid));
        const bool gated = a.silu;
        int chunk = 0;
        T* gx_t = reinterpret_cast<T*>(a.gx) + (batch * a.length + t_begin - (taps - 1)) * a.channels + channel;   // of token t - (taps - 1)
        // one token; INSIDE: it belongs to the strip and the sequence, and so does the one whose gx it completes
        auto token = [&](int64_t t, const Slot* slot_x, const Slot* slot_g, auto inside) {
            constexpr bool INSIDE = decltype(inside)::value;
            F2 g[N / 2];
            Tokens::widen(win[TAPS - 1], slot_x, (x_at + (uint32_t)t * (uint32_t)a.x_token) & 1);
            Tokens::widen(g, slot_g, (g_at + (uint32_t)t * (uint32_t)a.gout_token) & 1);
            if (gated) {
#pragma unroll
                for (int c = 0; c < N / 2; ++c) {
                    F2 pre = bias[c];
#pragma unroll
                    for (int k = 0; k < TAPS; ++k)
                        if (TAPS != kMaxTaps || k >= TAPS - taps) pre = fma2(w[k][c], win[k][c], pre);
                    // the derivative of silu: sig + silu (1 - sig)
                    const F2 sig = sigmoid2(pre);
                    g[c] = mul2(g[c], fma2(mul2(pre, sig), fma2(sig, same2(-1.0f), same2(1.0f)), sig));
                }
            }
            // outside the sequence nothing comes from above, whatever the inputs there
            const bool in = INSIDE || t < used;
#pragma unroll
            for (int c = 0; c < N / 2; ++c) gp[TAPS - 1][c] = in ? g[c] : same2(0.0f);
            if (INSIDE || (in && t < t_end)) {
#pragma unroll
                for (int c = 0; c < N / 2; ++c) {
                    gb[c] = add2(gb[c], gp[TAPS - 1][c]);
#pragma unroll
                    for (int k = 0; k < TAPS; ++k)
                        if (TAPS != kMaxTaps || k >= TAPS - taps) gw[k][c] = fma2(gp[TAPS - 1][c], win[k][c], gw[k][c]);
                }
            }
            // gp[TAPS - 1 - k] is gpre of token t - k: gx of token t - (taps - 1)
            const int64_t to = t - (taps - 1);
            const bool state = !INSIDE && to < 0;
            if (INSIDE || (t < walk_end && (state ? strip == 0 && a.ginitial != nullptr : to >= t_begin))) {
                float gx[N];
#pragma unroll
                for (int c = 0; c < N / 2; ++c) {
                    F2 sum = same2(0.0f);
#pragma unroll
                    for (int k = 0; k < TAPS; ++k)
                        if (TAPS != kMaxTaps || k >= TAPS - taps) {
                            if constexpr (TAPS != kMaxTaps) {
                                sum = fma2(w[k][c], gp[TAPS - 1 - k][c], sum);
                            } else {
                                // tap k - (8 - taps): gp is indexed by registers, so every possible one is compared
#pragma unroll
                                for (int m = 0; m < TAPS; ++m)
                                    if (m == k - (TAPS - taps)) sum = fma2(w[k][c], gp[TAPS - 1 - m][c], sum);
                            }
                        }
                    unpack2(sum, gx[2 * c], gx[2 * c + 1]);
                }
                if (!INSIDE && a.gfinal) {
                    // the state after the sequence holds the inputs used - (taps - 1) ... used - 1
                    const int64_t k = to - (used - (taps - 1));
                    if (k >= 0 && k < taps - 1) {
                        const Pack<T, N> gf = load_channels<T, N, W>(
                            reinterpret_cast<const T*>(a.gfinal) + (batch * (taps - 1) + k) * a.channels + channel, valid);
#pragma unroll
                        for (int c = 0; c < N; ++c) gx[c] += to_f32(gf.v[c]);
                    }
                }
                T* dst = gx_t;
                if (state) dst = reinterpret_cast<T*>(a.ginitial) + (batch * (taps - 1) + (taps - 1) + to) * a.channels + channel;
                store_channels<T, N, W>(dst, gx, valid);
            }
            gx_t += a.channels;
#pragma unroll
            for (int k = 0; k < TAPS - 1; ++k)
#pragma unroll
                for (int c = 0; c < N / 2; ++c) {
                    win[k][c] = win[k + 1][c];
                    gp[k][c] = gp[k + 1][c];
                }
        };
        for (int64_t t0 = t_begin; t0 < walk_end; t0 += CHUNK) {
            copy_wait<kAhead - 1>();
            fetch(t0 + kAhead * CHUNK, chunk == 0 ? kAhead : chunk - 1);
            // (gfinal belongs to tokens that the walk completes at t >= used)
            if (t0 >= t_begin + (taps - 1) && t0 + CHUNK <= t_end && t0 + CHUNK <= used) {
#pragma unroll
                for (int s = 0; s < CHUNK; ++s) token(t0 + s, ring_x.slot(chunk, s), ring_g.slot(chunk, s), True{});
            } else {
#pragma unroll 1
                for (int s = 0; s < CHUNK; ++s) token(t0 + s, ring_x.slot(chunk, s), ring_g.slot(chunk, s), False{});
            }
            chunk = chunk == kAhead ? 0 : chunk + 1;
        }
    }
    // the warps' sums for the weights and the bias, added up in warp order
    __shared__ float s_part[kWarps][(TAPS + 1) * N][32];
#pragma unroll
    for (int c = 0; c < N / 2; ++c) {
        float x0, x1;
#pragma unroll
        for (int k = 0; k < TAPS; ++k) {
            unpack2(gw[k][c], x0, x1);
            s_part[warp][k * N + 2 * c][lane] = x0;
            s_part[warp][k * N + 2 * c + 1][lane] = x1;
        }
        unpack2(gb[c], x0, x1);
        s_part[warp][TAPS * N + 2 * c][lane] = x0;
        s_part[warp][TAPS * N + 2 * c + 1][lane] = x1;
    }
    __syncthreads();
    const int64_t row = batch * p.strips + strip_block;
    for (int e = threadIdx.x; e < (TAPS + 1) * N * 32; e += 32 * kWarps) {
        const int cc = e % (N * 32), k = e / (N * 32) - (TAPS - taps);
        const int64_t ch = (blockIdx.x % p.column_tiles) * 32 * N + cc;
        if (k < 0 || ch >= a.channels) continue;
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < kWarps; ++s) sum += s_part[s][(e / (N * 32)) * N + cc / (32 * W) * W + cc % W][cc / W % 32];
        p.part[(row * (taps + 1) + k) * a.channels + ch] = sum;
    }
}

// the strips' parts added up in order, by slices (see sum_slices) of one block
template <typename T>
__global__ void __launch_bounds__(kSumThreads) conv_backward_params(const __grid_constant__ ConvParams p, int slices) {
    __shared__ float s_part[kSumThreads];
    const OvlCausalConv& a = p.a;
    const int values = kSumThreads / slices, v = threadIdx.x % values, slice = threadIdx.x / values;
    const int64_t total = (a.taps + 1) * a.channels, rows = a.batch * p.strips, i = (int64_t)blockIdx.x * values + v;
    float sum = 0.0f;
    if (i < total) {
#pragma unroll 8
        for (int64_t r = slice; r < rows; r += slices) sum += p.part[r * total + i];
    }
    s_part[threadIdx.x] = sum;
    __syncthreads();
    if (slice != 0 || i >= total) return;
    for (int s = 1; s < slices; ++s) sum += s_part[s * values + v];
    const int64_t k = i / a.channels, ch = i % a.channels;
    void* const to = k < a.taps ? a.gweight : a.gbias;
    const int64_t at = k < a.taps ? ch * a.taps + k : ch;
    if (!to) return;
    if (a.params_f32) reinterpret_cast<float*>(to)[at] = sum;
    else reinterpret_cast<T*>(to)[at] = from_f32<T>(sum);
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

// The strips' length: a block of k on one SM costs its tokens (and what it does before the first, as much as 12 tokens)
// times k + 3/4, which fits the times of strips of 8 to 256 tokens over the sizes below to a tenth, so the length of least
// cost is taken.  Measured (us; forward, backward) against other lengths, bf16:
//   4 x 4096 x 4096    64 tokens: 52.3, 103.7   128: 57.6, 97.5    48: 55.3, 112.5   16: 70.3, 160.1
//   1 x 2048 x 4096    20 tokens: 13.1, 23.5     40: 14.9, 19.8     8: 14.3, 32.6    64: 16.6, 20.9
//   1 x 512 x 2048      8 tokens:  5.9,  7.9     16:  8.1,  8.7    64: 15.6, 16.3
void cut(const OvlCausalConv* a, int channels_of_thread, ConvParams* p) {
    p->column_tiles = ceil_div(a->channels, 32 * channels_of_thread);
    const int64_t columns = a->batch * p->column_tiles, sms = sequence_sm_count();
    double least = 0;
    for (int64_t strip = kMinStrip; strip <= kMaxStrip; strip += kChunk) {
        const int64_t strips = ceil_div(a->length, strip * kWarps);
        const double cost = (double)(strip + 12) * (ceil_div(columns * strips, sms) + 0.75);
        if (strip == kMinStrip || cost < least) {
            least = cost;
            p->strip = strip;
            p->strips = strips;
        }
        if (strips <= 1) break;
    }
    if (p->strips < 1) p->strips = 1;                                    // states without tokens are passed on too
}

bool wide(const OvlCausalConv* a, int n, bool backward) {
    bool ok = a->channels % n == 0 && aligned16(a->x) && a->x_batch % n == 0 && a->x_token % n == 0 && aligned16(a->initial_state);
    if (!backward) return ok && aligned16(a->out) && aligned16(a->final_state);
    return ok && aligned16(a->gout) && a->gout_batch % n == 0 && a->gout_token % n == 0 && aligned16(a->gfinal) &&
           aligned16(a->gx) && aligned16(a->ginitial);
}

// `full`: whole packs of channels on 16-byte boundaries (the kernel has no other path then); `pairs`: two elements of 16
// bits on 4-byte boundaries; `single`: what is left
template <typename F>
int launch(const ConvParams& p, size_t smem, cudaStream_t stream, F full, F pairs, F single) {
    F kernel = p.vec ? full : p.width >= 2 ? pairs : single;
    const int64_t blocks = p.column_tiles * p.strips * p.a.batch;
    if (blocks > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    const int st = prepare_kernel((const void*)kernel, smem);
    if (st != OVL_OK) return st;
    kernel<<<(uint32_t)blocks, 32 * kWarps, smem, stream>>>(p);
    return launch_status();
}

template <typename T>
constexpr int kPairs = sizeof(T) == 2 ? 2 : 1;

template <typename T>
int run_forward(ConvParams p, cudaStream_t stream) {
    cut(&p.a, kForward, &p);
    p.vec = wide(&p.a, kForward, false);
    p.width = copy_width<T>({p.a.x, p.a.out, p.a.initial_state, p.a.final_state}, {p.a.channels, p.a.x_batch, p.a.x_token});
    const size_t smem = p.vec || p.width >= 1 ? Ring<T, kForward, kForward>::bytes : Ring<T, kForward, 1>::bytes;
    switch (p.a.taps) {
        case 2: return launch(p, smem, stream, conv_forward<T, 2, kForward>, conv_forward<T, 2, kPairs<T>>, conv_forward<T, 2, 1>);
        case 3: return launch(p, smem, stream, conv_forward<T, 3, kForward>, conv_forward<T, 3, kPairs<T>>, conv_forward<T, 3, 1>);
        case 4: return launch(p, smem, stream, conv_forward<T, 4, kForward>, conv_forward<T, 4, kPairs<T>>, conv_forward<T, 4, 1>);
        default: return launch(p, smem, stream, conv_forward<T, kMaxTaps, kForward>, conv_forward<T, kMaxTaps, kPairs<T>>, conv_forward<T, kMaxTaps, 1>);
    }
}

template <typename T>
int run_backward(ConvParams p, cudaStream_t stream) {
    cut(&p.a, kBackward, &p);
    p.vec = wide(&p.a, kBackward, true);
    p.width = copy_width<T>({p.a.x, p.a.gout, p.a.gx, p.a.initial_state, p.a.gfinal, p.a.ginitial},
                            {p.a.channels, p.a.x_batch, p.a.x_token, p.a.gout_batch, p.a.gout_token});
    p.part = reinterpret_cast<float*>(p.a.workspace);
    const size_t smem = 2 * (p.vec || p.width >= 1 ? Ring<T, kBackward, kBackward>::bytes : Ring<T, kBackward, 1>::bytes);
    int st;
    switch (p.a.taps) {
        case 2: st = launch(p, smem, stream, conv_backward<T, 2, kBackward>, conv_backward<T, 2, kPairs<T>>, conv_backward<T, 2, 1>); break;
        case 3: st = launch(p, smem, stream, conv_backward<T, 3, kBackward>, conv_backward<T, 3, kPairs<T>>, conv_backward<T, 3, 1>); break;
        case 4: st = launch(p, smem, stream, conv_backward<T, 4, kBackward>, conv_backward<T, 4, kPairs<T>>, conv_backward<T, 4, 1>); break;
        default: st = launch(p, smem, stream, conv_backward<T, kMaxTaps, kBackward>, conv_backward<T, kMaxTaps, kPairs<T>>, conv_backward<T, kMaxTaps, 1>); break;
    }
    if (st != OVL_OK) return st;
    const int slices = sum_slices(p.a.batch * p.strips);
    conv_backward_params<T><<<(uint32_t)ceil_div((p.a.taps + 1) * p.a.channels, kSumThreads / slices), kSumThreads, 0, stream>>>(p, slices);
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
    ovl::ConvParams p{};
    ovl::cut(a, ovl::kBackward, &p);
    return (uint64_t)a->batch * p.strips * (a->taps + 1) * a->channels * sizeof(float);
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
