// Dropout of splat parameters from a counter-based generator: the decision for a group of values is one 32-bit word of
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) at the group's own
// number, so forward and backward regenerate the same mask and none is ever stored.
#include "ssb_common.cuh"

namespace ssb {

constexpr float kDroppedLogit = SSB_DROPPED_LOGIT;

struct DropArgs {
    uint32_t key0, key1;
    uint64_t offset;
    const uint64_t* d_offset;
    uint32_t threshold;        // a group is dropped when its word is below it
    float scale;               // 1 / (1 - rate)
};

__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = (uint64_t)c.x * 0xD2511F53u, q = (uint64_t)c.z * 0xCD9E8D57u;
        c = make_uint4((uint32_t)(q >> 32) ^ c.y ^ k0, (uint32_t)q, (uint32_t)(p >> 32) ^ c.w ^ k1, (uint32_t)p);
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    return c;
}

__device__ __forceinline__ uint64_t drop_offset(const DropArgs& a) { return a.offset + (a.d_offset ? *a.d_offset : 0); }

// The four words of block b: the decisions of groups 4b .. 4b + 3.
__device__ __forceinline__ uint4 drop_words(const DropArgs& a, uint64_t offset, uint64_t block) {
    return philox4x32_10(make_uint4((uint32_t)block, (uint32_t)(block >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)), a.key0, a.key1);
}
__device__ __forceinline__ uint32_t word_of(const uint4& w, int k) { return k == 0 ? w.x : (k == 1 ? w.y : (k == 2 ? w.z : w.w)); }

__global__ void __launch_bounds__(256) dropout_kernel(const float* x, float* y, int64_t first, int64_t count, int32_t group,
                                                      DropArgs a) {
    const uint64_t offset = drop_offset(a);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const uint64_t g = (uint64_t)(first + i) / (uint32_t)group;
        const uint32_t w = word_of(drop_words(a, offset, g >> 2), (int)(g & 3));
        y[i] = w < a.threshold ? 0.0f : x[i] * a.scale;
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

template <bool BWD>
__global__ void __launch_bounds__(256) dropout_opacity_kernel(const float* x, const float* v, float* out,
                                                              int64_t first, int64_t count, DropArgs a, OpacityArgs o) {
    const uint64_t offset = drop_offset(a);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const uint64_t g = (uint64_t)(first + i);
        const bool dropped = word_of(drop_words(a, offset, g >> 2), (int)(g & 3)) < a.threshold;
        const float xi = x[i];
        const float w = -expm1f(-((o.x0_hi - xi) + o.x0_lo));
        if (BWD) out[i] = (dropped || xi > o.x_cap) ? 0.0f : v[i] / w;
        else out[i] = dropped ? kDroppedLogit : (xi > o.x_cap ? o.capped : (xi + o.a) - logf(w));
    }
}

static int drop_args(const SsbDropout* d, const char* who, DropArgs* a) {
    SSB_REQUIRE(d, "%s: NULL dropout description", who);
    SSB_REQUIRE(d->rate >= 0.0f && d->rate < 1.0f, "%s: the rate must be in [0, 1) (got %g)", who, (double)d->rate);
    SSB_REQUIRE(d->reserved == 0, "%s: reserved must be 0", who);
    SSB_REQUIRE(((uintptr_t)d->d_offset & 7) == 0, "%s: d_offset must be 8-byte aligned", who);
    a->key0 = (uint32_t)d->seed; a->key1 = (uint32_t)(d->seed >> 32);
    a->offset = d->offset;
    a->d_offset = d->d_offset;
    a->threshold = (uint32_t)floor((double)d->rate * 4294967296.0);
    a->scale = (float)(1.0 / (1.0 - (double)d->rate));
    return SSB_OK;
}

static int check_range(int64_t first, int64_t count, const char* who) {
    SSB_REQUIRE(first >= 0 && count >= 0 && first <= ((int64_t)1 << 62) && count <= ((int64_t)1 << 62) - first, "%s: bad range", who);
    return SSB_OK;
}

static int check_floats(const char* who, const void* a, const void* b, const void* c) {
    SSB_REQUIRE(a && b && c, "%s: NULL argument", who);
    SSB_REQUIRE((((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 3) == 0, "%s: arrays must lie on 4-byte boundaries", who);
    return SSB_OK;
}

static unsigned drop_blocks(int64_t count) { return (unsigned)(count > 148 * 8 * 256 ? 148 * 8 : ceil_div(count, 256)); }

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
    dropout_kernel<<<drop_blocks(count), 256, 0, (cudaStream_t)stream>>>(d_x, d_y, first, count, group, a);
    SSB_LAUNCHED("dropout_kernel");
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
    dropout_opacity_kernel<false><<<drop_blocks(count), 256, 0, (cudaStream_t)stream>>>(d_opacities, nullptr, d_out, first, count, a, opacity_args(dropout->rate));
    SSB_LAUNCHED("dropout_opacity_kernel");
    return SSB_OK;
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
    dropout_opacity_kernel<true><<<drop_blocks(count), 256, 0, (cudaStream_t)stream>>>(d_opacities, d_v_out, d_v_opacities, first, count, a, opacity_args(dropout->rate));
    SSB_LAUNCHED("dropout_opacity_kernel");
    return SSB_OK;
}

}  // extern "C"
