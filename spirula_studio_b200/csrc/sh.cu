// Spherical harmonics on their own: 4-bit rows with band scales (encode, decode), and the product of every splat's 3 x 15
// coefficient matrix with the basis of its viewing directions, forward and backward.
#include "sh_device.cuh"

#include <algorithm>

namespace ssb {

// ---- 4-bit rows -------------------------------------------------------------
// A band's scale is the smallest bf16 s with 7 s >= the largest finite magnitude m of the band (zero below 2^-100, where s
// and its multiples would lose bits, and one step smaller where 7 s would overflow); a value's code is v / s rounded to the nearest integer, ties to even, so that
// decode(encode(v)) is within s / 2.  The quotient is not formed: q = rint(v * (1 / s)) is off by one at most next to a
// midpoint, and the remainder v - q s, exact in one fused multiply-add (it has at most the bits of v below s), tells.
__device__ __forceinline__ float row_scale(float m) {
    if (!(m >= 7.8886090522101181e-31f)) return 0.0f;                                      // 2^-100
    float s = __uint_as_float(__float_as_uint(m * (1.0f / 7.0f)) & 0xffff0000u);            // within one bf16 step of the answer
    if (7.0f * s < m) s = __uint_as_float(__float_as_uint(s) + 0x10000u);                   // 7 s is exact (eleven bits)
    if (7.0f * s < m) s = __uint_as_float(__float_as_uint(s) + 0x10000u);
    const float below = __uint_as_float(__float_as_uint(s) - 0x10000u);
    return 7.0f * below >= m || isinf(7.0f * s) ? below : s;
}

__device__ __forceinline__ int row_code(float v, float s, float inv) {
    if (!(s > 0.0f) || v != v) return 0;
    v = fminf(fmaxf(v, -7.0f * s), 7.0f * s);                                               // infinities
    float q = rintf(v * inv);
    const float r = fmaf(-q, s, v), h = 0.5f * s;
    if (fabsf(r) > h || (fabsf(r) == h && ((int)q & 1))) q += copysignf(1.0f, r);
    return (int)q;
}

// The row's six words of codes, value by value as row_code defines them; `sh` holds the splat's 45 values.
__device__ __noinline__ void encode_row_checked(const float* sh, uint32_t w[6], const float s[3], const float inv[3]) {
    for (int j = 0; j < kNumSh; ++j)
        for (int ch = 0; ch < 3; ++ch) {
            const int k = 2 * ch + (j >> 3);
            w[k] = ((j & 7) ? w[k] : 0u) | (uint32_t)(row_code(sh[3 * j + ch], s[sh_band(j)], inv[sh_band(j)]) + 8) << (4 * (j & 7));
        }
}

// Per value: t = v / s + 8 + 1.5 2^23 rounds to the code and leaves it in the low bits of t, so a word is a sum of shifted t's less
// a constant.  The remainder decides whether the rounding was the right one (see row_code); rows with a value next to a midpoint,
// an infinity or a NaN -- one splat in a hundred thousand of ordinary ones -- take the checked way.
__global__ void __launch_bounds__(kProjBlock) sh_rows_encode_kernel(const float* __restrict__ sh, int64_t n, uint4* __restrict__ rows) {
    __shared__ __align__(16) float sh_s[kProjBlock * kShPerSplat];
    const int64_t first = (int64_t)blockIdx.x * kProjBlock;
    const int64_t i = first + threadIdx.x;
    stage_sh(sh_s, nullptr, sh, nullptr, nullptr, 32, 256, first, n);
    __syncthreads();
    if (i >= n) return;
    float v[kShPerSplat];
#pragma unroll
    for (int k = 0; k < kShPerSplat; ++k) v[k] = sh_s[threadIdx.x * kShPerSplat + k];
    float m[3] = {0.0f, 0.0f, 0.0f}, s[3], inv[3], half[3], odd = 0.0f;
#pragma unroll
    for (int k = 0; k < kShPerSplat; ++k) {
        m[sh_band(k / 3)] = fmaxf(m[sh_band(k / 3)], fabsf(v[k]));
        odd = fmaf(v[k], 0.0f, odd);                     // NaN as soon as one value is not finite
    }
    bool checked = odd != 0.0f;
    if (checked) {
        m[0] = m[1] = m[2] = 0.0f;
        for (int k = 0; k < kShPerSplat; ++k) {
            const float a = fabsf(sh_s[threadIdx.x * kShPerSplat + k]), f = a <= 3.402823466e38f ? a : 0.0f;
            if (k < 9) m[0] = fmaxf(m[0], f); else if (k < 24) m[1] = fmaxf(m[1], f); else m[2] = fmaxf(m[2], f);
        }
    }
#pragma unroll
    for (int b = 0; b < 3; ++b) {
        s[b] = row_scale(m[b]);
        inv[b] = s[b] > 0.0f ? 1.0f / s[b] : 0.0f;
        half[b] = s[b] > 0.0f ? 0.5f * s[b] : INFINITY;
    }
    constexpr float kMagic = 12582912.0f + 8.0f;
    uint32_t w[8] = {};
#pragma unroll
    for (int j = 0; j < kNumSh; ++j)
#pragma unroll
        for (int ch = 0; ch < 3; ++ch) {
            const float x = v[3 * j + ch], t = fmaf(x, inv[sh_band(j)], kMagic);
            checked |= fabsf(fmaf(kMagic - t, s[sh_band(j)], x)) >= half[sh_band(j)];
            w[2 * ch + (j >> 3)] += __float_as_uint(t) << (4 * (j & 7));
        }
#pragma unroll
    for (int ch = 0; ch < 3; ++ch) { w[2 * ch] -= 0x4b400000u * 0x11111111u; w[2 * ch + 1] -= 0x4b400000u * 0x01111111u; }
    if (checked) {
        uint32_t c[6];
        encode_row_checked(sh_s + threadIdx.x * kShPerSplat, c, s, inv);
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = c[k];
    }
    w[6] = (__float_as_uint(s[0]) >> 16) | (__float_as_uint(s[1]) & 0xffff0000u);
    w[7] = __float_as_uint(s[2]) >> 16;
    rows[2 * i] = make_uint4(w[0], w[1], w[2], w[3]);
    rows[2 * i + 1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// Writes a block's contiguous span of `count` floats from shared memory (16-byte aligned there) to global memory.  A full span
// on a 16-byte boundary leaves as one bulk copy (or, when added to what is there, one bulk reduction: every address belongs to one
// thread block, so the sum has one order); anything else takes coalesced 4-byte stores.  All threads call it between the barrier
// after the span was written and bulk_done().
__device__ __forceinline__ void store_span(float* dst, const float* span_s, int count, int full, bool add) {
    if (count == full && ((uintptr_t)dst & 15) == 0) {
        if (threadIdx.x == 0) {
            const uint32_t src = (uint32_t)__cvta_generic_to_shared(span_s);
            if (add) asm volatile("cp.reduce.async.bulk.global.shared::cta.bulk_group.add.f32 [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(4 * full) : "memory");
            else asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(4 * full) : "memory");
        }
    } else if (add) for (int k = threadIdx.x; k < count; k += kProjBlock) dst[k] += span_s[k];
    else for (int k = threadIdx.x; k < count; k += kProjBlock) dst[k] = span_s[k];
}
// The thread's writes to shared memory become visible to bulk copies issued after the next barrier.
__device__ __forceinline__ void span_written() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Waits until the block's bulk copies have read their spans (the spans may then be written again, or the block may end).
__device__ __forceinline__ void bulk_done() {
    if (threadIdx.x == 0) asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
}

__global__ void __launch_bounds__(kProjBlock) sh_rows_decode_kernel(const void* __restrict__ rows, int64_t n, float* __restrict__ sh) {
    __shared__ __align__(16) float sh_s[kProjBlock * kShPerSplat];
    const int64_t first = (int64_t)blockIdx.x * kProjBlock;
    const int64_t i = first + threadIdx.x;
    if (i < n) decode_sh_row(load_sh_row(rows, i), sh_s + threadIdx.x * kShPerSplat);
    span_written();
    __syncthreads();
    store_span(sh + first * kShPerSplat, sh_s, (int)min((int64_t)kProjBlock, n - first) * kShPerSplat, kProjBlock * kShPerSplat, false);
    bulk_done();
}

int launch_sh_rows_encode(const float* d_values, int64_t n, void* d_rows, cudaStream_t st) {
    if (n == 0) return SSB_OK;
    sh_rows_encode_kernel<<<(unsigned)ceil_div(n, kProjBlock), kProjBlock, 0, st>>>(d_values, n, (uint4*)d_rows);
    SSB_LAUNCHED("sh_rows_encode_kernel");
    return SSB_OK;
}

int launch_sh_rows_decode(const void* d_rows, int64_t n, float* d_values, cudaStream_t st) {
    if (n == 0) return SSB_OK;
    sh_rows_decode_kernel<<<(unsigned)ceil_div(n, kProjBlock), kProjBlock, 0, st>>>(d_rows, n, d_values);
    SSB_LAUNCHED("sh_rows_decode_kernel");
    return SSB_OK;
}

// ---- the product ------------------------------------------------------------
// value[v][i] = C0 dc_i + sum_j b_j(dir) W_i[j], dir = (mean_i - centre_v) / |mean_i - centre_v|.  The difference is what
// loses bits when a camera is close to a splat far from the origin, so the centre is kept as a sum of two floats.
struct ViewCentre { float hi[3], lo[3]; };     // -centre = R^T t

__device__ __forceinline__ ViewCentre view_centre(const float* __restrict__ viewmats, int v) {
    const float* m = viewmats + 16 * v;
    ViewCentre c;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        const double s = (double)m[j] * m[3] + (double)m[4 + j] * m[7] + (double)m[8 + j] * m[11];
        c.hi[j] = (float)s;
        c.lo[j] = (float)(s - (double)c.hi[j]);
    }
    return c;
}

struct Direction { float x, y, z, inv; };      // unit vector and 1 / distance

// The direction of a splat at the camera's own position is undefined: the bands then contribute nothing (all components 0).
__device__ __noinline__ Direction direction_rescaled(float dx, float dy, float dz) {
    const float m = fmaxf(fabsf(dx), fmaxf(fabsf(dy), fabsf(dz)));
    if (dx == 0.0f && dy == 0.0f && dz == 0.0f) return {0.0f, 0.0f, 0.0f, 0.0f};
    const int e = isfinite(m) ? ilogbf(m) : 0;
    dx = scalbnf(dx, -e); dy = scalbnf(dy, -e); dz = scalbnf(dz, -e);
    const float inv = rsqrtf(dx * dx + dy * dy + dz * dz);
    return {dx * inv, dy * inv, dz * inv, scalbnf(inv, -e)};
}

__device__ __forceinline__ Direction view_direction(const ViewCentre& c, const float mean[3]) {
    const float dx = (mean[0] + c.hi[0]) + c.lo[0], dy = (mean[1] + c.hi[1]) + c.lo[1], dz = (mean[2] + c.hi[2]) + c.lo[2];
    const float d2 = dx * dx + dy * dy + dz * dz;
    if (!(d2 > 1e-30f && d2 < 1e30f)) return direction_rescaled(dx, dy, dz);
    float inv = rsqrtf(d2);
    inv = inv * fmaf(-0.5f * d2, inv * inv, 1.5f);
    return {dx * inv, dy * inv, dz * inv, inv};
}

constexpr int kCentreChunk = 32;      // views whose centres a block keeps at a time

__device__ __forceinline__ void stage_centres(ViewCentre* centres_s, const float* __restrict__ viewmats, int v0, int views) {
    const int v = v0 + threadIdx.x;
    if (threadIdx.x < kCentreChunk && v < views) centres_s[threadIdx.x] = view_centre(viewmats, v);
}

// The SH values of the thread's splat: in registers from its 4-bit row, or from the block's staged span.
template <bool ROWS>
__device__ __forceinline__ void read_sh(float sh[kShPerSplat], const float* sh_s, const SsbShQuant& shq, int64_t i, int n_sh) {
    if (n_sh == 0) {
#pragma unroll
        for (int k = 0; k < kShPerSplat; ++k) sh[k] = 0.0f;
    } else if (ROWS) {
        decode_sh_row(load_sh_row(shq.packed, i), sh);
    } else {
#pragma unroll
        for (int k = 0; k < kShPerSplat; ++k) sh[k] = sh_s[threadIdx.x * kShPerSplat + k];
    }
}

template <bool ROWS>
__global__ void __launch_bounds__(kProjBlock) sh_eval_fwd_kernel(SsbSplats sp, SsbShQuant shq, int64_t n, int views, const float* __restrict__ viewmats,
                                                                 int n_sh, float* __restrict__ out) {
    __shared__ __align__(16) float sh_s[ROWS ? 4 : kProjBlock * kShPerSplat];
    __shared__ __align__(16) unsigned char raw_s[ROWS ? 16 : kShRawBytes];
    __shared__ ViewCentre centres_s[kCentreChunk];
    stage_centres(centres_s, viewmats, 0, views);
    __syncthreads();
    for (int64_t first = (int64_t)blockIdx.x * kProjBlock; first < n; first += (int64_t)gridDim.x * kProjBlock) {
        const int64_t i = first + threadIdx.x;
        if (!ROWS && n_sh > 0) {
            __syncthreads();
            stage_sh(sh_s, raw_s, sp.features_sh, shq.packed, shq.bounds, shq.bits, shq.bounds_stride, first, n);
            __syncthreads();
        }
        const int64_t il = min(i, n - 1);
        const float mean[3] = {sp.means[3 * il], sp.means[3 * il + 1], sp.means[3 * il + 2]};
        float dc[3] = {0.f, 0.f, 0.f};
        if (sp.features_dc)
#pragma unroll
            for (int ch = 0; ch < 3; ++ch) dc[ch] = kShC0 * sp.features_dc[3 * il + ch];
        float sh[kShPerSplat];
        read_sh<ROWS>(sh, sh_s, shq, il, n_sh);
        for (int v0 = 0; v0 < views; v0 += kCentreChunk) {
            if (views > kCentreChunk) {
                __syncthreads();
                stage_centres(centres_s, viewmats, v0, views);
                __syncthreads();
            }
            const int v1 = min(views - v0, kCentreChunk);
            for (int v = 0; v < v1; ++v) {
                const Direction d = view_direction(centres_s[v], mean);
                float b[kNumSh];
                sh_basis(d.x, d.y, d.z, b);
                if (d.inv == 0.0f) b[5] = 0.0f;            // no direction: the one basis function that does not vanish by itself
                float c[3] = {dc[0], dc[1], dc[2]};
#pragma unroll
                for (int j = 0; j < kNumSh; ++j)
                    if (j < n_sh)
#pragma unroll
                        for (int ch = 0; ch < 3; ++ch) c[ch] += b[j] * sh[3 * j + ch];
                if (i < n) {
                    float* o = out + 3 * ((int64_t)(v0 + v) * n + i);
                    o[0] = c[0]; o[1] = c[1]; o[2] = c[2];
                }
            }
        }
    }
}

template <bool ROWS>
__global__ void __launch_bounds__(kProjBlock) sh_eval_bwd_kernel(SsbSplats sp, SsbShQuant shq, int64_t n, int views, const float* __restrict__ viewmats,
                                                                 int n_sh, const float* __restrict__ v_out, SsbSplats gr, int accumulate) {
    __shared__ __align__(16) float sh_s[kProjBlock * kShPerSplat];       // values on the way in, their gradients on the way out
    __shared__ __align__(16) float mean_s[kProjBlock * 3];
    __shared__ __align__(16) float dc_s[kProjBlock * 3];
    __shared__ __align__(16) unsigned char raw_s[ROWS ? 16 : kShRawBytes];
    __shared__ ViewCentre centres_s[kCentreChunk];
    stage_centres(centres_s, viewmats, 0, views);
    for (int64_t first = (int64_t)blockIdx.x * kProjBlock; first < n; first += (int64_t)gridDim.x * kProjBlock) {
        const int64_t i = first + threadIdx.x, il = min(i, n - 1);
        __syncthreads();
        if (!ROWS && n_sh > 0) {
            stage_sh(sh_s, raw_s, sp.features_sh, shq.packed, shq.bounds, shq.bits, shq.bounds_stride, first, n);
            __syncthreads();
        }
        const float mean[3] = {sp.means[3 * il], sp.means[3 * il + 1], sp.means[3 * il + 2]};
        float sh[kShPerSplat], g_mean[3] = {0.f, 0.f, 0.f}, g_dc[3] = {0.f, 0.f, 0.f}, g_sh[kShPerSplat];
        read_sh<ROWS>(sh, sh_s, shq, il, n_sh);
#pragma unroll
        for (int k = 0; k < kShPerSplat; ++k) g_sh[k] = 0.f;
        for (int v0 = 0; v0 < views; v0 += kCentreChunk) {
            if (views > kCentreChunk) {
                __syncthreads();
                stage_centres(centres_s, viewmats, v0, views);
                __syncthreads();
            }
            const int v1 = min(views - v0, kCentreChunk);
            for (int v = 0; v < v1; ++v) {
                const float* gp = v_out + 3 * ((int64_t)(v0 + v) * n + il);
                const float g[3] = {gp[0], gp[1], gp[2]};
                const Direction d = view_direction(centres_s[v], mean);
                float b[kNumSh], w[kNumSh];
                sh_basis(d.x, d.y, d.z, b);
                if (d.inv == 0.0f) b[5] = 0.0f;
#pragma unroll
                for (int j = 0; j < kNumSh; ++j) {
                    w[j] = 0.0f;
                    if (j < n_sh) {
#pragma unroll
                        for (int ch = 0; ch < 3; ++ch) { w[j] += sh[3 * j + ch] * g[ch]; g_sh[3 * j + ch] += b[j] * g[ch]; }
                    }
                }
#pragma unroll
                for (int ch = 0; ch < 3; ++ch) g_dc[ch] += kShC0 * g[ch];
                float vn[3];
                sh_basis_vjp(d.x, d.y, d.z, w, vn);
                const float dn = d.x * vn[0] + d.y * vn[1] + d.z * vn[2];
                g_mean[0] += (vn[0] - d.x * dn) * d.inv;
                g_mean[1] += (vn[1] - d.y * dn) * d.inv;
                g_mean[2] += (vn[2] - d.z * dn) * d.inv;
            }
        }
        bulk_done();
        __syncthreads();          // the previous tile's copies have left, and every thread has read its values
#pragma unroll
        for (int k = 0; k < 3; ++k) { mean_s[3 * threadIdx.x + k] = g_mean[k]; dc_s[3 * threadIdx.x + k] = g_dc[k]; }
#pragma unroll
        for (int k = 0; k < kShPerSplat; ++k) sh_s[kShPerSplat * threadIdx.x + k] = g_sh[k];
        span_written();
        __syncthreads();
        const int count = (int)min((int64_t)kProjBlock, n - first);
        if (gr.means) store_span(gr.means + 3 * first, mean_s, 3 * count, 3 * kProjBlock, accumulate != 0);
        if (gr.features_dc) store_span(gr.features_dc + 3 * first, dc_s, 3 * count, 3 * kProjBlock, accumulate != 0);
        if (gr.features_sh) store_span(gr.features_sh + kShPerSplat * first, sh_s, kShPerSplat * count, kProjBlock * kShPerSplat, accumulate != 0);
        if (!ROWS) bulk_done();   // the next tile is staged into the same span
    }
    bulk_done();
}

// Checks shared by the two directions; on success q is the SH source and *n_sh the coefficients past DC in use.
static int check_eval(const SsbSplats* splats, const SsbShQuant* shq, int64_t n, const SsbCameras* cams, const char* who, SsbShQuant* q, int* n_sh) {
    SSB_REQUIRE(splats && cams, "%s: NULL argument", who);
    SSB_REQUIRE(n >= 0 && n <= (int64_t)kProjBlock * 0x7fffffff && cams->count >= 0, "%s: bad sizes", who);
    SSB_REQUIRE(cams->sh_degree_plus1 >= 0 && cams->sh_degree_plus1 <= 4, "%s: sh_degree_plus1 must be 0 (all bands) or 1..4", who);
    *n_sh = active_sh_count(cams);
    *q = SsbShQuant{nullptr, nullptr, 32, 0, 256};
    if (n == 0) return SSB_OK;
    SSB_REQUIRE(splats->means, "%s: means are NULL", who);
    SSB_REQUIRE(cams->d_viewmats || cams->count == 0, "%s: d_viewmats is NULL", who);
    SSB_REQUIRE((((uintptr_t)splats->means | (uintptr_t)splats->features_dc | (uintptr_t)splats->features_sh | (uintptr_t)cams->d_viewmats) & 3) == 0,
                "%s: arrays must lie on 4-byte boundaries", who);
    if (*n_sh > 0) return check_shq(splats, shq, *q);
    return SSB_OK;
}

}  // namespace ssb

extern "C" {

int ssb_sh_eval_fwd(const SsbSplats* splats, const SsbShQuant* shq, int64_t n, const SsbCameras* cams, float* d_values, void* stream) {
    using namespace ssb;
    SsbShQuant q;
    int n_sh;
    if (int e = check_eval(splats, shq, n, cams, "ssb_sh_eval_fwd", &q, &n_sh)) return e;
    if (n == 0 || cams->count == 0) return SSB_OK;
    SSB_REQUIRE(d_values && ((uintptr_t)d_values & 3) == 0, "ssb_sh_eval_fwd: d_values is NULL or not on a 4-byte boundary");
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(n, kProjBlock), 148 * 8);
    if (q.bits == 4) sh_eval_fwd_kernel<true><<<blocks, kProjBlock, 0, (cudaStream_t)stream>>>(*splats, q, n, cams->count, cams->d_viewmats, n_sh, d_values);
    else sh_eval_fwd_kernel<false><<<blocks, kProjBlock, 0, (cudaStream_t)stream>>>(*splats, q, n, cams->count, cams->d_viewmats, n_sh, d_values);
    SSB_LAUNCHED("sh_eval_fwd_kernel");
    return SSB_OK;
}

int ssb_sh_eval_bwd(const SsbSplats* splats, const SsbShQuant* shq, int64_t n, const SsbCameras* cams, const float* d_v_values,
                    const SsbSplats* grads, int accumulate, void* stream) {
    using namespace ssb;
    SsbShQuant q;
    int n_sh;
    SSB_REQUIRE(grads, "ssb_sh_eval_bwd: NULL argument");
    if (int e = check_eval(splats, shq, n, cams, "ssb_sh_eval_bwd", &q, &n_sh)) return e;
    if (n == 0) return SSB_OK;
    SSB_REQUIRE(d_v_values || cams->count == 0, "ssb_sh_eval_bwd: NULL argument");
    SSB_REQUIRE((((uintptr_t)d_v_values | (uintptr_t)grads->means | (uintptr_t)grads->features_dc | (uintptr_t)grads->features_sh) & 3) == 0,
                "ssb_sh_eval_bwd: arrays must lie on 4-byte boundaries");
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(n, kProjBlock), 148 * 8);
    if (q.bits == 4) sh_eval_bwd_kernel<true><<<blocks, kProjBlock, 0, (cudaStream_t)stream>>>(*splats, q, n, cams->count, cams->d_viewmats, n_sh, d_v_values, *grads, accumulate);
    else sh_eval_bwd_kernel<false><<<blocks, kProjBlock, 0, (cudaStream_t)stream>>>(*splats, q, n, cams->count, cams->d_viewmats, n_sh, d_v_values, *grads, accumulate);
    SSB_LAUNCHED("sh_eval_bwd_kernel");
    return SSB_OK;
}

}  // extern "C"
