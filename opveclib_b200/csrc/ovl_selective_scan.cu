// Selective scan: what its entry points check, how a problem is cut, and where the work space lies.  The kernels are in
// ovl_selective_scan.cuh; interface: include/ovl_b200.h.
#include <mutex>
#include <set>
#include <utility>
#include "ovl_selective_scan.cuh"

namespace ovl {

int prepare_kernel(const void* kernel, size_t smem, int threads, int registers) {
    static std::mutex mutex;
    static std::set<std::pair<const void*, int>> done;
    if (smem <= 24 * 1024 && registers == 0) return OVL_OK;              // (with the 18 KB that some have beside it: 48 KB need no leave)
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return record_cuda_error(e);
    const std::pair<const void*, int> key(kernel, device);
    std::lock_guard<std::mutex> lock(mutex);
    if (done.count(key)) return OVL_OK;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (registers > 0) {
        cudaFuncAttributes attributes;
        e = cudaFuncGetAttributes(&attributes, kernel);
        if (e != cudaSuccess) return record_cuda_error(e);
        if (attributes.numRegs * threads < registers) return OVL_ERR_INVALID;
    }
    done.insert(key);
    return OVL_OK;
}

namespace {

bool multiple_of(int64_t n, int64_t a, int64_t b) { return a % n == 0 && b % n == 0; }

int check(const OvlSelectiveScan* a) {
    if (!a) return OVL_ERR_NULL;
    if (a->dtype != OVL_FLOAT32 && a->dtype != OVL_FLOAT16 && a->dtype != OVL_BFLOAT16) return OVL_ERR_DTYPE;
    if (a->batch < 0 || a->length < 0 || a->channels < 1 || a->groups < 1 || a->states < 1) return OVL_ERR_INVALID;
    if (a->channels % a->groups != 0) return OVL_ERR_INVALID;
    if (a->states > kMaxStates) return OVL_ERR_TOO_LARGE;
    return OVL_OK;
}

int lanes_for(int64_t states, int per_lane, int least) {
    int p = least;
    while (per_lane * p < states) p *= 2;
    return p;
}

// Two channels per lane need less shared memory bandwidth and fewer instructions for each, one channel gives twice the
// blocks.  bf16, 16 states, 2048 channels: with 256 blocks of 64 channels (8 x 2048 tokens) 238 us against 268 us, with
// 128 of them (4 x 2048 tokens) 152 against 138 us.
ScanShape forward_shape(const OvlSelectiveScan* a) {
    ScanShape s{lanes_for(a->states, 4, 1), 2, 2};
    const int64_t blocks = a->batch * a->groups * ceil_div(a->channels / a->groups, s.block_channels());
    if (s.lanes < 32 && 2 * blocks < 3 * (int64_t)sequence_sm_count()) s.channels = 1;
    return s;
}

ScanShape backward_shape(const OvlSelectiveScan* a) {
    if (a->states > 64) return ScanShape{32, 2, 1};
    return ScanShape{lanes_for(a->states, 2, 4), 1, 2};
}

constexpr int64_t kMostParts = (int64_t)1 << 30;
// bytes of one channel tile's parts of gB and gC, over all batches and groups
int64_t part_bytes(const OvlSelectiveScan* a, const ScanShape& shape) {
    return a->batch * a->groups * a->length * 2 * shape.padded_states() * (int64_t)sizeof(float);
}

void make_dims(const OvlSelectiveScan* a, ScanDims* d, ScanShape* shape, bool backward) {
    d->length = a->length;
    d->channels = a->channels;
    d->states = a->states;
    d->groups = a->groups;
    d->group_channels = a->channels / a->groups;
    d->softplus = a->delta_softplus != 0;
    *shape = backward ? backward_shape(a) : forward_shape(a);
    d->all_tiles = d->tiles = ceil_div(d->group_channels, shape->block_channels());
    d->first_tile = 0;
    // Segments that run side by side in two launches (one less than there are segments in each): as many as two blocks per
    // SM hold, from four segments on - with S segments the two launches walk 2 / S of the length.  bf16, one sequence, 16
    // states: 2048 tokens x 2048 channels (64 blocks) 82 us in one piece, 59 us in 5 segments; 16384 x 4096 (128 blocks)
    // 625 us in one piece, 637 us in 3 segments, 723 us in 4.
    const int64_t blocks = a->batch * a->groups * d->tiles;
    int64_t s = blocks > 0 ? 1 + 2 * (int64_t)sequence_sm_count() / blocks : 1;
    const int64_t most = ceil_div(a->length, 64);
    if (s > most) s = most;
    if (s > kMaxSegments) s = kMaxSegments;
    if (s < 4) s = 1;
    d->segment_length = ceil_div(ceil_div(a->length > 0 ? a->length : 1, s), 32) * 32;
    d->segments = ceil_div(a->length > 0 ? a->length : 1, d->segment_length);
    if (!backward || a->batch == 0) return;
    // The parts of gB and gC are 8 bytes per token, padded state and tile, and tiles have fewer channels the more states there
    // are (32 with 16 states, 8 with 64, 4 with 128): 4, 64 and 256 bytes per token and channel, 34 GB for 8 x 4096 x 4096 x
    // 128.  What is more than kMostParts goes through the same memory in several launches, each with as many blocks as
    // the SMs hold at a time (two each, one above 64 states: shared memory), or a multiple of them.  The backward pass of
    // bf16 4 x 2048 x 4096 x 128: 10.7 ms with 1.2 GB allocated, 10.4 ms with 8.9 GB in one piece.
    const int64_t bytes = part_bytes(a, *shape), at_a_time = (a->states > 64 ? 1 : 2) * (int64_t)sequence_sm_count();
    if (d->all_tiles <= 1 || bytes * d->all_tiles <= kMostParts) return;
    const int64_t wave = ceil_div(at_a_time, a->batch * a->groups * (d->segments > 1 ? d->segments - 1 : 1));
    const int64_t waves = kMostParts / (bytes * wave);
    d->tiles = wave * (waves > 1 ? waves : 1);
    if (d->tiles > d->all_tiles) d->tiles = d->all_tiles;
}

uint64_t round16(uint64_t n) { return (n + 15) / 16 * 16; }

struct Workspace {
    uint64_t state, dt, bc, sum, A, D, total;
};
Workspace layout(const OvlSelectiveScan* a, const ScanDims& d, const ScanShape& shape, bool backward) {
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
        w.bc = take(part_bytes(a, shape) / sizeof(float) * d.tiles);
        if (d.tiles < d.all_tiles) w.sum = take(part_bytes(a, shape) / sizeof(float));
        w.A = take((uint64_t)a->batch * d.segments * d.channels * d.states);
        w.D = take((uint64_t)a->batch * d.segments * 2 * d.channels);
    }
    w.total = at;
    return w;
}

int run(const OvlSelectiveScan* a, bool backward, cudaStream_t stream) {
    int st = check(a);
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
    ScanShape shape;
    make_dims(a, &p.d, &shape, backward);
    if (a->batch * p.d.segments * p.d.groups * p.d.tiles > 0x7fffffff) return OVL_ERR_TOO_LARGE;
    const Workspace w = layout(a, p.d, shape, backward);
    if (w.total > 0 && (!a->workspace || a->workspace_bytes < w.total || !aligned16(a->workspace))) return OVL_ERR_SCRATCH;
    char* const ws = reinterpret_cast<char*>(a->workspace);
    p.seg_state = reinterpret_cast<float*>(ws + w.state);
    p.seg_dt = reinterpret_cast<float*>(ws + w.dt);
    p.part_bc = reinterpret_cast<float*>(ws + w.bc);
    p.sum_bc = reinterpret_cast<float*>(ws + w.sum);
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
    auto width = [&](auto one) {
        using T = decltype(one);
        const bool b = backward;
        return copy_width<T>({a->u, a->delta, a->z, b ? a->gout : nullptr, b ? a->gu : a->out, b ? a->gdelta : nullptr, b ? a->gz : nullptr},
                             {p.d.group_channels, a->u_batch, a->u_token, a->delta_batch, a->delta_token, a->z ? a->z_batch : 0,
                              a->z ? a->z_token : 0, b ? a->gout_batch : 0, b ? a->gout_token : 0});
    };
    p.d.width = a->dtype == OVL_FLOAT32 ? width(float()) : width(__half());
    if (a->dtype == OVL_FLOAT32) return scan_run_f32(p, shape, backward, stream);
    if (a->dtype == OVL_FLOAT16) return scan_run_f16(p, shape, backward, stream);
    return scan_run_bf16(p, shape, backward, stream);
}

}  // namespace
}  // namespace ovl

extern "C" uint64_t ovl_selective_scan_workspace_bytes(const OvlSelectiveScan* args, int backward) {
    if (ovl::check(args) != OVL_OK || args->batch == 0) return 0;
    ovl::ScanDims d;
    ovl::ScanShape shape;
    ovl::make_dims(args, &d, &shape, backward != 0);
    return ovl::layout(args, d, shape, backward != 0).total;
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
    const int lanes = ovl::lanes_for(a->states, 4, 1);
    if (a->dtype == OVL_FLOAT32) return ovl::scan_step_f32(*a, lanes, stream);
    if (a->dtype == OVL_FLOAT16) return ovl::scan_step_f16(*a, lanes, stream);
    return ovl::scan_step_bf16(*a, lanes, stream);
}
