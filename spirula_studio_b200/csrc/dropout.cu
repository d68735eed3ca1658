// Dropout of splat parameters from a counter-based generator: the decision for a group of values is one 32-bit word of
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) at the group's own
// number, so forward and backward regenerate the same mask and none is ever stored.
#include "ssb_common.cuh"

namespace ssb {

constexpr float kDroppedLogit = SSB_DROPPED_LOGIT;

struct DropArgs {
    uint32_t k0[10], k1[10];       // the rounds' keys (added up in the kernel instead: 57 and 172 us where these take 56 and 169)
    uint64_t offset;
    const uint64_t* d_offset;
    uint32_t threshold;        // a group is dropped when its word is below it
    float scale;               // 1 / (1 - rate)
};

__device__ __forceinline__ uint4 philox4x32_10(uint4 c, const uint32_t* k0, const uint32_t* k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = (uint64_t)c.x * 0xD2511F53u, q = (uint64_t)c.z * 0xCD9E8D57u;
        c = make_uint4((uint32_t)(q >> 32) ^ c.y ^ k0[r], (uint32_t)q, (uint32_t)(p >> 32) ^ c.w ^ k1[r], (uint32_t)p);
    }
    return c;
}

__device__ __forceinline__ uint64_t drop_offset(const DropArgs& a) { return a.offset + (a.d_offset ? *a.d_offset : 0); }

// The four words of block b: the decisions of groups 4b .. 4b + 3.
__device__ __forceinline__ uint4 drop_words(const DropArgs& a, uint64_t offset, uint64_t block) {
    return philox4x32_10(make_uint4((uint32_t)block, (uint32_t)(block >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)), a.k0, a.k1);
}
// Four consecutive values at p[i], of which only those with 0 <= i + k < count exist.  VEC: p + i is 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p, int64_t i, int64_t count) {
    if (VEC && i >= 0 && i + 3 < count) return *(const float4*)(p + i);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i >= 0 && i < count) v.x = p[i];
    if (i + 1 >= 0 && i + 1 < count) v.y = p[i + 1];
    if (i + 2 >= 0 && i + 2 < count) v.z = p[i + 2];
    if (i + 3 >= 0 && i + 3 < count) v.w = p[i + 3];
    return v;
}
template <bool VEC>
__device__ __forceinline__ void store4(float* p, int64_t i, int64_t count, float4 v) {
    if (VEC && i >= 0 && i + 3 < count) { *(float4*)(p + i) = v; return; }
    if (i >= 0 && i < count) p[i] = v.x;
    if (i + 1 >= 0 && i + 1 < count) p[i + 1] = v.y;
    if (i + 2 >= 0 && i + 2 < count) p[i + 2] = v.z;
    if (i + 3 >= 0 && i + 3 < count) p[i + 3] = v.w;
}

constexpr int kDropThreads = 256;
constexpr int kDropChunks = 4;                                     // chunks of four values per thread, all loads in flight
constexpr int kDropTile = kDropThreads * kDropChunks * 4;          // values per block

// Every value decides for itself: a thread's four values are the four words of one generator block, so the decisions never
// leave registers.  Chunks start on multiples of four of the whole array's numbering.  Bound by memory, 8 bytes a value: 135M values in
// 167 us, 6.5 TB/s, 99 % of the copy bandwidth; the generator's ten rounds fit behind it.  Arrays off the numbering's 16-byte
// boundaries (VEC = false) take four 4-byte accesses per chunk: 45M values 82 us where 16-byte ones take 56.
// One chunk a thread less or more: 167 (two) and 160 us (eight) where four took 157 on the same day.
template <bool VEC>
__global__ void __launch_bounds__(kDropThreads) dropout_values_kernel(const float* x, float* y, int64_t first, int64_t count, DropArgs a) {
    const uint64_t offset = drop_offset(a);
    const int64_t chunk0 = (int64_t)blockIdx.x * (kDropThreads * kDropChunks) + threadIdx.x;
    const int64_t i0 = 4 * chunk0 - (first & 3);
    float4 v[kDropChunks];
#pragma unroll
    for (int c = 0; c < kDropChunks; ++c) v[c] = load4<VEC>(x, i0 + 4 * kDropThreads * c, count);
#pragma unroll
    for (int c = 0; c < kDropChunks; ++c) {
        const uint4 w = drop_words(a, offset, (uint64_t)(first >> 2) + (uint64_t)(chunk0 + kDropThreads * c));
        v[c].x = w.x < a.threshold ? 0.0f : v[c].x * a.scale;
        v[c].y = w.y < a.threshold ? 0.0f : v[c].y * a.scale;
        v[c].z = w.z < a.threshold ? 0.0f : v[c].z * a.scale;
        v[c].w = w.w < a.threshold ? 0.0f : v[c].w * a.scale;
        store4<VEC>(y, i0 + 4 * kDropThreads * c, count, v[c]);
    }
}

// Groups of several values: the decisions of the groups that a block's tile touches are made once, one generator block per
// four groups, and kept as one byte each in shared memory while the tile's values are on their way.  45M values in groups of three: 55 us,
// 6.5 TB/s, 99 % of the copy bandwidth (75 where the two arrays lie differently in their 16 bytes); with a 64-bit place per value it was
// 69 us and bound by integer arithmetic.
struct GroupArgs {
    uint32_t group, magic;
    uint32_t first_rem;        // place of the first value in its group
    int32_t shift;             // tile 0 starts this many values before the array, on a 16-byte boundary
    uint64_t first_group;      // group of the first value
};
// p / group for places p counted from the start of a tile's first group
__device__ __forceinline__ uint32_t group_of(const GroupArgs& ga, uint32_t p) { return ga.magic ? __umulhi(p, ga.magic) : (p >= ga.group ? 1u : 0u); }

template <bool VEC>
__global__ void __launch_bounds__(kDropThreads) dropout_groups_kernel(const float* x, float* y, int64_t count, GroupArgs ga, DropArgs a) {
    __shared__ uint32_t keep_s[(kDropTile / 2 + 8) / 4 + 2];
    const uint64_t offset = drop_offset(a);
    const int64_t tile = (int64_t)blockIdx.x * kDropTile - ga.shift;            // the tile's first value; may lie before the array
    const int64_t i0 = tile + 4 * threadIdx.x;
    float4 v[kDropChunks];
#pragma unroll
    for (int c = 0; c < kDropChunks; ++c) v[c] = load4<VEC>(x, i0 + 4 * kDropThreads * c, count);
    const int64_t lo = max(tile, (int64_t)0), hi = min(tile + kDropTile, count) - 1;
    const uint64_t at = (uint64_t)lo + ga.first_rem, g = at / ga.group;
    const uint64_t g0 = ga.first_group + g;
    const uint32_t r0 = (uint32_t)(at - g * ga.group);                          // place of value lo in its group, g0
    const uint32_t last = (uint32_t)(hi - lo) + r0;                             // place of value hi, counted from the start of g0
    const uint32_t n_groups = group_of(ga, last) + 1;
    const uint32_t lead = (uint32_t)(g0 & 3);
    for (uint32_t b = threadIdx.x; 4 * b < lead + n_groups; b += kDropThreads) {
        const uint4 w = drop_words(a, offset, (g0 >> 2) + b);
        keep_s[b] = (w.x < a.threshold ? 0u : 1u) | (w.y < a.threshold ? 0u : 1u << 8) | (w.z < a.threshold ? 0u : 1u << 16) |
                    (w.w < a.threshold ? 0u : 1u << 24);
    }
    __syncthreads();
    const uint8_t* keep = (const uint8_t*)keep_s + lead;
    const uint32_t p0 = (uint32_t)(i0 - lo) + r0;
#pragma unroll
    for (int c = 0; c < kDropChunks; ++c) {
        float* e = &v[c].x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            // a value outside the array takes some decision of the tile: it is not stored
            const uint32_t p = min(p0 + (uint32_t)(4 * kDropThreads * c + k), last);
            e[k] = keep[group_of(ga, p)] ? e[k] * a.scale : 0.0f;
        }
        store4<VEC>(y, i0 + 4 * kDropThreads * c, count, v[c]);
    }
}

// A kept splat's opacity s = sigmoid(x) becomes z = s / (1 - r).  With d = ln((1 - r) / r) - x and w = 1 - e^-d, logit(z) is
// x - ln(1 - r) - ln w and its slope 1 / w; both stay accurate where z approaches one, since d is the difference the
// cancellation happens in and w = -expm1(-d).
struct OpacityArgs {
    float x0_hi, x0_lo;        // ln((1 - r) / r) as a sum of two floats
    float a;                   // -ln(1 - r)
    float x_cap;               // largest x whose compensated opacity stays below the cap
    float capped;              // logit of the cap
};


// 1 - e^-d for d > 0 to within 2^-22.  Below 1.375 as d P(d), P the polynomial of degree seven that fits (1 - e^-d) / d there
// (Chebyshev nodes; with fp32 coefficients 2^-24.9 off, 2.7 half-ulps as evaluated); above it the hardware exponential, whose 2 ulp and the
// argument's rounding weigh e^-d / (1 - e^-d) <= 0.34 of themselves.  Other d are not used (the opacity is then limited).  expm1f
// instead made the two calls take 68 instead of 55 us for 10M opacities.
__device__ __forceinline__ float one_minus_exp_neg(float d) {
    float p = -1.36514881887706e-05f;
    p = fmaf(p, d, 0.0001761570747476071f);
    p = fmaf(p, d, -0.0013644357677549124f);
    p = fmaf(p, d, 0.008318103849887848f);
    p = fmaf(p, d, -0.04166145622730255f);
    p = fmaf(p, d, 0.16666579246520996f);
    p = fmaf(p, d, -0.4999999403953552f);
    p = fmaf(p, d, 1.0f);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * -1.4426950408889634f));
    return d >= 1.375f ? 1.0f - e : p * d;
}

template <bool BWD>
__device__ __forceinline__ float drop_opacity(float x, float v, bool dropped, const OpacityArgs& o) {
    const float w = one_minus_exp_neg((o.x0_hi - x) + o.x0_lo);
    if (BWD) return (dropped || x > o.x_cap) ? 0.0f : __fdividef(v, w);
    // the hardware logarithm: off by 2^-22 where w is above 1/2 and by 2^-22 of itself below, against w's own 2^-22; logf made
    // the forward call take 29 instead of 21 us for 10M opacities
    float l;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(l) : "f"(w));
    return dropped ? kDroppedLogit : (x > o.x_cap ? o.capped : fmaf(-0.6931471805599453f, l, x + o.a));
}

// Two chunks of loads in flight per thread; one took 31 + 27 us where two took 29 + 25, four 29 + 30 (forward + backward, before the
// hardware logarithm).
constexpr int kOpacityChunks = 2;

// 8 bytes a splat forward, 12 backward.  10M splats: 20.8 to 22.9 and 23.7 us (23.0 and 27.1 with VEC = false); ssb_dropout, which moves the
// forward call's bytes with a third of its arithmetic, takes 16.4 at that size, a device copy of torch's 20.9.  The forward call issues 48
// instructions a value on 74 % of the cycles.

template <bool BWD, bool VEC>
__global__ void __launch_bounds__(kDropThreads) dropout_opacity_kernel(const float* x, const float* v, float* out, int64_t first, int64_t count,
                                                                       DropArgs a, OpacityArgs o) {
    const uint64_t offset = drop_offset(a);
    const int64_t chunk0 = (int64_t)blockIdx.x * (kDropThreads * kOpacityChunks) + threadIdx.x;
    const int64_t i0 = 4 * chunk0 - (first & 3);
    float4 xv[kOpacityChunks], vv[kOpacityChunks];
#pragma unroll
    for (int c = 0; c < kOpacityChunks; ++c) {
        xv[c] = load4<VEC>(x, i0 + 4 * kDropThreads * c, count);
        if (BWD) vv[c] = load4<VEC>(v, i0 + 4 * kDropThreads * c, count);
    }
#pragma unroll
    for (int c = 0; c < kOpacityChunks; ++c) {
        const uint4 w = drop_words(a, offset, (uint64_t)(first >> 2) + (uint64_t)(chunk0 + kDropThreads * c));
        float4 r;
        r.x = drop_opacity<BWD>(xv[c].x, BWD ? vv[c].x : 0.f, w.x < a.threshold, o);
        r.y = drop_opacity<BWD>(xv[c].y, BWD ? vv[c].y : 0.f, w.y < a.threshold, o);
        r.z = drop_opacity<BWD>(xv[c].z, BWD ? vv[c].z : 0.f, w.z < a.threshold, o);
        r.w = drop_opacity<BWD>(xv[c].w, BWD ? vv[c].w : 0.f, w.w < a.threshold, o);
        store4<VEC>(out, i0 + 4 * kDropThreads * c, count, r);
    }
}

static int drop_args(const SsbDropout* d, const char* who, DropArgs* a) {
    SSB_REQUIRE(d, "%s: NULL dropout description", who);
    SSB_REQUIRE(d->rate >= 0.0f && d->rate < 1.0f, "%s: the rate must be in [0, 1) (got %g)", who, (double)d->rate);
    SSB_REQUIRE(d->reserved == 0, "%s: reserved must be 0", who);
    SSB_REQUIRE(((uintptr_t)d->d_offset & 7) == 0, "%s: d_offset must be 8-byte aligned", who);
    for (int r = 0; r < 10; ++r) {
        a->k0[r] = (uint32_t)d->seed + (uint32_t)r * 0x9E3779B9u;
        a->k1[r] = (uint32_t)(d->seed >> 32) + (uint32_t)r * 0xBB67AE85u;
    }
    a->offset = d->offset;
    a->d_offset = d->d_offset;
    a->threshold = (uint32_t)floor((double)d->rate * 4294967296.0);
    a->scale = (float)(1.0 / (1.0 - (double)d->rate));
    return SSB_OK;
}

static int check_range(int64_t first, int64_t count, const char* who) {
    SSB_REQUIRE(first >= 0 && count >= 0 && first <= ((int64_t)1 << 62) && count <= ((int64_t)1 << 40), "%s: bad range", who);
    return SSB_OK;
}

static int check_floats(const char* who, const void* a, const void* b, const void* c) {
    SSB_REQUIRE(a && b && c, "%s: NULL argument", who);
    SSB_REQUIRE((((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 3) == 0, "%s: arrays must lie on 4-byte boundaries", who);
    return SSB_OK;
}

static OpacityArgs opacity_args(float rate) {
    const double r = rate, cap = 0.999;
    const double x0 = log((1.0 - r) / r);
    OpacityArgs o;
    o.x0_hi = (float)x0;
    o.x0_lo = (float)(x0 - (double)o.x0_hi);
    o.a = (float)-log1p(-r);
    // s = cap (1 - r): the opacity whose compensated value is the cap
    const double xc = log(cap * (1.0 - r) / (1.0 - cap * (1.0 - r)));
    o.x_cap = (float)xc;
    if ((double)o.x_cap >= xc) o.x_cap = nextafterf(o.x_cap, -INFINITY);
    o.capped = (float)log(cap / (1.0 - cap));
    return o;
}

// Whether value `first` being at p leaves the multiples of four of the numbering on 16-byte boundaries: then chunks travel as 16-byte
// accesses, otherwise as 4-byte ones (the kernels' comments have both times).
static bool chunk_aligned(const void* p, int64_t first) { return (((uintptr_t)p >> 2) & 3) == (uintptr_t)(first & 3); }

static int launch_opacity(bool bwd, const float* x, const float* v, float* out, int64_t first, int64_t count, const SsbDropout* d, const DropArgs& a,
                          cudaStream_t st) {
    const unsigned blocks = (unsigned)ceil_div(count + (first & 3), 4 * kDropThreads * kOpacityChunks);
    const OpacityArgs o = opacity_args(d->rate);
    const bool vec = chunk_aligned(x, first) && chunk_aligned(out, first) && (!bwd || chunk_aligned(v, first));
    if (bwd && vec) dropout_opacity_kernel<true, true><<<blocks, kDropThreads, 0, st>>>(x, v, out, first, count, a, o);
    else if (bwd) dropout_opacity_kernel<true, false><<<blocks, kDropThreads, 0, st>>>(x, v, out, first, count, a, o);
    else if (vec) dropout_opacity_kernel<false, true><<<blocks, kDropThreads, 0, st>>>(x, v, out, first, count, a, o);
    else dropout_opacity_kernel<false, false><<<blocks, kDropThreads, 0, st>>>(x, v, out, first, count, a, o);
    SSB_LAUNCHED("dropout_opacity_kernel");
    return SSB_OK;
}

}  // namespace ssb

extern "C" {

int ssb_dropout(const float* d_x, int64_t first, int64_t count, int32_t group, const SsbDropout* dropout, float* d_y, void* stream) {
    using namespace ssb;
    DropArgs a;
    if (int e = drop_args(dropout, "ssb_dropout", &a)) return e;
    if (int e = check_range(first, count, "ssb_dropout")) return e;
    SSB_REQUIRE(group >= 1, "ssb_dropout: group must be at least 1 (got %d)", group);
    if (count == 0) return SSB_OK;
    if (int e = check_floats("ssb_dropout", d_x, d_x, d_y)) return e;
    cudaStream_t st = (cudaStream_t)stream;
    if (group == 1) {
        const unsigned blocks = (unsigned)ceil_div(count + (first & 3), kDropTile);
        if (chunk_aligned(d_x, first) && chunk_aligned(d_y, first)) dropout_values_kernel<true><<<blocks, kDropThreads, 0, st>>>(d_x, d_y, first, count, a);
        else dropout_values_kernel<false><<<blocks, kDropThreads, 0, st>>>(d_x, d_y, first, count, a);
        SSB_LAUNCHED("dropout_values_kernel");
        return SSB_OK;
    }
    // p / group = umulhi(p, ceil(2^32 / group)) for p < group + kDropTile as long as group (group + kDropTile) < 2^32; a tile
    // touches at most two larger groups
    const bool vec = (((uintptr_t)d_x ^ (uintptr_t)d_y) & 15) == 0;
    GroupArgs ga;
    ga.group = (uint32_t)group;
    ga.magic = group <= 32768 ? (uint32_t)(((uint64_t)1 << 32) / (uint32_t)group + 1) : 0;
    ga.first_group = (uint64_t)first / (uint32_t)group;
    ga.first_rem = (uint32_t)((uint64_t)first % (uint32_t)group);
    ga.shift = vec ? (int32_t)(((uintptr_t)d_x >> 2) & 3) : 0;
    const unsigned blocks = (unsigned)ceil_div(count + ga.shift, kDropTile);
    if (vec) dropout_groups_kernel<true><<<blocks, kDropThreads, 0, st>>>(d_x, d_y, count, ga, a);
    else dropout_groups_kernel<false><<<blocks, kDropThreads, 0, st>>>(d_x, d_y, count, ga, a);
    SSB_LAUNCHED("dropout_groups_kernel");
    return SSB_OK;
}

int ssb_dropout_opacities(const float* d_opacities, int64_t first, int64_t count, const SsbDropout* dropout, float* d_out, void* stream) {
    using namespace ssb;
    DropArgs a;
    if (int e = drop_args(dropout, "ssb_dropout_opacities", &a)) return e;
    if (int e = check_range(first, count, "ssb_dropout_opacities")) return e;
    if (count == 0) return SSB_OK;
    if (int e = check_floats("ssb_dropout_opacities", d_opacities, d_opacities, d_out)) return e;
    if (dropout->rate == 0.0f) {
        if (d_out != d_opacities) SSB_CUDA(cudaMemcpyAsync(d_out, d_opacities, (size_t)count * sizeof(float), cudaMemcpyDeviceToDevice, (cudaStream_t)stream));
        return SSB_OK;
    }
    return launch_opacity(false, d_opacities, nullptr, d_out, first, count, dropout, a, (cudaStream_t)stream);
}

int ssb_dropout_opacities_bwd(const float* d_opacities, const float* d_v_out, int64_t first, int64_t count, const SsbDropout* dropout,
                              float* d_v_opacities, void* stream) {
    using namespace ssb;
    DropArgs a;
    if (int e = drop_args(dropout, "ssb_dropout_opacities_bwd", &a)) return e;
    if (int e = check_range(first, count, "ssb_dropout_opacities_bwd")) return e;
    if (count == 0) return SSB_OK;
    if (int e = check_floats("ssb_dropout_opacities_bwd", d_opacities, d_v_out, d_v_opacities)) return e;
    if (dropout->rate == 0.0f) {
        if (d_v_out != d_v_opacities) SSB_CUDA(cudaMemcpyAsync(d_v_opacities, d_v_out, (size_t)count * sizeof(float), cudaMemcpyDeviceToDevice, (cudaStream_t)stream));
        return SSB_OK;
    }
    return launch_opacity(true, d_opacities, d_v_out, d_v_opacities, first, count, dropout, a, (cudaStream_t)stream);
}

}  // extern "C"
