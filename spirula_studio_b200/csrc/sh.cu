// Spherical harmonics on their own: 4-bit rows with band scales (encode, decode), and the product of every splat's 3 x 15
// coefficient matrix with the basis of its viewing directions, forward and backward.
#include "sh_device.cuh"

#include <algorithm>
#include <cooperative_groups.h>

namespace ssb {

// ---- 4-bit rows -------------------------------------------------------------
// A band's scale is the smallest bf16 s with 7 s >= the largest finite magnitude m of the band (zero below 2^-100, where s and its
// multiples would lose bits, and one step smaller where 7 s would overflow); a value's code is v / s rounded to the nearest
// integer, ties to even, so that decode(encode(v)) is within s / 2.  The scale is rounded up to bf16's eight bits before the codes
// are taken: that widens a step by less than 1/128 and makes every decoded value an exact float (eleven bits).
// The quotient is not formed: q = rint(v * (1 / s)) is off by one at most next to a midpoint, and the remainder v - q s, exact in
// one fused multiply-add (it has at most the bits of v below s), tells.
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
// an infinity or a NaN -- a few splats in a hundred thousand of ordinary ones -- take the checked way.
// Bound by memory: a block's 128 rows of values come in as 16-byte asynchronous copies, its rows leave as two 16-byte stores per
// splat.  5M splats: 156 us for 1.06 GB, at the copy bandwidth; one value at a time with a conversion to integer it was 282 us.
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

// Bound by memory: one row per thread, the block's values leave as one bulk copy.  5M splats: 160 us for 1.06 GB.
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
// value[v][i] = C0 dc_i + sum_j b_j(dir) W_i[j], dir = (mean_i - centre_v) / |mean_i - centre_v|.
//
// The basis functions are taken as polynomials p_j of the direction without their constants k_j (b_j = k_j p_j); the constants go
// into the coefficients or into their gradients, once per splat.
//
// One view is bound by memory: a thread per splat, nothing kept, codes decoded where they are multiplied.  Several views (the *_views
// kernels) are bound by arithmetic: a thread works on two
// splats at once, 128 apart, with the coefficients in registers, and all its arithmetic is on pairs, one packed single-precision
// instruction for two results.  What limits that is the register file: a packed multiply-add on three different register pairs was
// measured at three cycles per scheduler, a scalar one at 1.9, so a pair costs less than two scalars; one splat per thread, scalar or
// packed over coefficients, took 76 and 81 us where this form takes 64 (1M splats, 16 views, forward) and 157 against 153 backward.
// The active degree is no part of the kernels' types: below degree 3 they do the same work on zeros (degree 0: 60 and 143 us, degrees 1 and 2 as 3).
typedef float2 Pair;
__device__ __forceinline__ Pair operator+(Pair a, Pair b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ Pair operator*(Pair a, Pair b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ Pair operator*(float a, Pair b) { return __fmul2_rn(make_float2(a, a), b); }
__device__ __forceinline__ Pair fma_(Pair a, Pair b, Pair c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ Pair fma_(float a, Pair b, Pair c) { return __ffma2_rn(make_float2(a, a), b, c); }
__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
template <class T> __device__ __forceinline__ T all(float a);
template <> __device__ __forceinline__ float all<float>(float a) { return a; }
template <> __device__ __forceinline__ Pair all<Pair>(float a) { return make_float2(a, a); }

// b_j = sh_constant(j) p_j.  The polynomials are scaled so that none of them, nor a component of a gradient, needs a constant
// factor (a constant costs a packed instruction two registers or two moves):
//   y, z, x | 2xy, 2yz, z^2 - 1/3, 2xz, x^2 - y^2 | y(3x^2 - y^2), 2xyz, y(z^2 - 1/5), z(z^2 - 3/5), x(z^2 - 1/5), z(x^2 - y^2),
//   x(x^2 - 3y^2)
__device__ __forceinline__ constexpr float sh_constant(int j) {
    constexpr float k[kNumSh] = {-0.4886025119029199f, 0.4886025119029199f, -0.4886025119029199f,
                                 0.5462742152960396f, -0.5462742152960396f, 0.94617469575756f, -0.5462742152960396f, 0.5462742152960396f,
                                 -0.5900435899266435f, 1.445305721320277f, -2.285228997322329f, 1.865881662950577f, -2.285228997322329f,
                                 1.445305721320277f, -0.5900435899266435f};
    return k[j];
}
// What coefficient j is multiplied by in the sums w_j that sh_polynomials_vjp takes: b_j's constant times the constant that its
// gradient's components share.
__device__ __forceinline__ constexpr float sh_grad_constant(int j) {
    constexpr float k[kNumSh] = {-0.4886025119029199f, 0.4886025119029199f, -0.4886025119029199f,
                                 1.0925484305920792f, -1.0925484305920792f, 1.89234939151512f, -1.0925484305920792f, 1.0925484305920792f,
                                 -1.7701307697799304f, 1.445305721320277f, -2.285228997322329f, 5.597644988851731f, -2.285228997322329f,
                                 1.445305721320277f, -1.7701307697799304f};
    return k[j];
}

// The difference mean - centre is what loses bits when a camera is close to a splat far from the origin, so the centre is kept as
// a sum of two floats.
template <class T> struct ViewCentre { T hi[3], lo[3]; };      // -centre = R^T t

// Component j of R^T t.
__device__ __forceinline__ double centre_component(const float* __restrict__ viewmats, int v, int j) {
    const float* m = viewmats + 16 * (int64_t)v;
    return (double)m[j] * m[3] + (double)m[4 + j] * m[7] + (double)m[8 + j] * m[11];
}

template <class T>
struct Directions { T x, y, z, inv; };         // unit vectors and 1 / distance

// d2 leaves the caller to notice squares that left the range of floats (see eval_checked).
template <class T>
__device__ __forceinline__ Directions<T> view_directions(const ViewCentre<T>& c, const T mean[3], T& d2) {
    const T dx = (mean[0] + c.hi[0]) + c.lo[0], dy = (mean[1] + c.hi[1]) + c.lo[1], dz = (mean[2] + c.hi[2]) + c.lo[2];
    d2 = fma_(dx, dx, fma_(dy, dy, dz * dz));
    T inv;
    if constexpr (sizeof(T) == 8) inv = make_float2(rsqrtf(d2.x), rsqrtf(d2.y)); else inv = rsqrtf(d2);
    return {dx * inv, dy * inv, dz * inv, inv};
}
constexpr float kSquareMin = 1e-30f, kSquareMax = 1e30f;
// The largest of three, NaN if one is (fmaxf drops them): a square that is not a number left the range too.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <class T>
struct Polynomials { T p[kNumSh], ny, x2, t; };        // -y, 2x, z^2 - 1/5

template <class T>
__device__ __forceinline__ Polynomials<T> sh_polynomials(const Directions<T>& d) {
    Polynomials<T> o;
    const T x = d.x, y = d.y, z = d.z, zz = z * z, y2 = y + y;
    o.ny = -1.0f * y; o.x2 = x + x; o.t = zz + all<T>(-0.2f);
    o.p[0] = y; o.p[1] = z; o.p[2] = x;
    o.p[3] = o.x2 * y; o.p[4] = y2 * z; o.p[5] = zz + all<T>(-1.0f / 3.0f); o.p[6] = o.x2 * z; o.p[7] = fma_(x, x, o.ny * y);
    o.p[8] = y * fma_(o.x2, x, o.p[7]); o.p[9] = o.p[3] * z; o.p[10] = y * o.t; o.p[11] = z * (zz + all<T>(-0.6f));
    o.p[12] = x * o.t; o.p[13] = z * o.p[7]; o.p[14] = x * fma_(y2, o.ny, o.p[7]);
    return o;
}

// Gradient with respect to the mean of sum_j b_j W_j, given w_j = sh_grad_constant(j) W_j: the polynomials' gradient, made tangent
// to the sphere; what is left is to divide by the distance.
template <class T>
__device__ __forceinline__ void sh_polynomials_vjp(const Directions<T>& d, const Polynomials<T>& o, const T w[kNumSh], T v[3]) {
    const T x = d.x, y = d.y, z = d.z, xy2 = o.p[3], yz2 = o.p[4], xz2 = o.p[6], c1 = o.p[7], nyz2 = -1.0f * yz2;
    T gx = fma_(y, w[3], w[2]), gy = fma_(x, w[3], w[0]), gz = fma_(y, w[4], w[1]);
    gx = fma_(z, w[6], gx); gx = fma_(x, w[7], gx); gx = fma_(xy2, w[8], gx); gx = fma_(yz2, w[9], gx);
    gx = fma_(o.t, w[12], gx); gx = fma_(xz2, w[13], gx); gx = fma_(c1, w[14], gx);
    gy = fma_(z, w[4], gy); gy = fma_(o.ny, w[7], gy); gy = fma_(c1, w[8], gy); gy = fma_(xz2, w[9], gy);
    gy = fma_(o.t, w[10], gy); gy = fma_(nyz2, w[13], gy); gy = fma_(o.x2 * o.ny, w[14], gy);
    gz = fma_(z, w[5], gz); gz = fma_(x, w[6], gz); gz = fma_(xy2, w[9], gz); gz = fma_(yz2, w[10], gz);
    gz = fma_(o.t, w[11], gz); gz = fma_(xz2, w[12], gz); gz = fma_(c1, w[13], gz);
    const T nd = -1.0f * fma_(x, gx, fma_(y, gy, z * gz));
    v[0] = fma_(x, nd, gx); v[1] = fma_(y, nd, gy); v[2] = fma_(z, nd, gz);
}

// ---- coefficients ----
// A code is read in place: the four bits at position 4 p of a word, or-ed into 2^23, are 2^23 + code 2^4p as a float, and the 2^-4p
// goes into a constant; only the positions 5..7 need the word shifted first.
__device__ __forceinline__ constexpr int code_shift(int j) { return (j & 7) > 4 ? 4 * (j & 7) - 16 : 4 * (j & 7); }
__device__ __forceinline__ constexpr float code_unit(int j) { return 1.0f / (float)(1 << code_shift(j)); }
__device__ __forceinline__ constexpr float code_bias(int j) { return -(8388608.0f + (float)(8 << code_shift(j))); }
__device__ __forceinline__ float code_bits(const ShRow& r, int j, int ch) {
    const uint32_t w = r.w[2 * ch + (j >> 3)];
    float f;       // (w & mask) | 2^23 in one instruction: left to the compiler it took two
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=f"(f) : "r"((j & 7) > 4 ? w >> 16 : w), "r"(15u << code_shift(j)), "r"(0x4b000000u));
    return f;
}
// (code - 8) / code_unit(j), exact
__device__ __forceinline__ float code_of(const ShRow& r, int j, int ch) { return code_bits(r, j, ch) + code_bias(j); }
__device__ __forceinline__ Pair code_of(const ShRow& a, const ShRow& b, int j, int ch) {
    return make_float2(code_bits(a, j, ch), code_bits(b, j, ch)) + all<Pair>(code_bias(j));
}
// A band's scale, zero above the active degree.
__device__ __forceinline__ float active_scale(const ShRow& r, int band, int n_sh) { return n_sh > (band + 1) * (band + 1) - 1 ? sh_row_scale(r, band) : 0.0f; }

// Everything about one splat by the definition, with the direction in double precision, whose range the square of a distance cannot
// leave: for splats that are nearer to a camera than 1e-15 or farther than 1e15.  A splat at the camera's own position has no
// direction: the bands contribute nothing, and at degree 0 no position matters, not even one that is not finite.  Forward (v_out NULL): the values of all views at out.  Backward: g receives the
// gradients of the mean (3), of DC (3) and of the coefficients (45).
__device__ __noinline__ void eval_checked(const SsbSplats sp, const float* sh, const void* rows, int64_t i, int64_t n, int views,
                                          const float* viewmats, int n_sh, float* out, const float* v_out, float* g) {
    float W[kShPerSplat];
    if (rows) decode_sh_row(load_sh_row(rows, i), W);
    else for (int k = 0; k < 3 * n_sh; ++k) W[k] = sh[k];
    if (v_out) for (int k = 0; k < 6 + kShPerSplat; ++k) g[k] = 0.0f;
    for (int v = 0; v < views; ++v) {
        double d[3], r2 = 0.0;
        for (int k = 0; k < 3; ++k) { d[k] = (double)sp.means[3 * i + k] + centre_component(viewmats, v, k); r2 += d[k] * d[k]; }
        const double inv = r2 == 0.0 ? 0.0 : 1.0 / sqrt(r2);
        const Directions<float> dir = {(float)(d[0] * inv), (float)(d[1] * inv), (float)(d[2] * inv), (float)inv};
        Polynomials<float> o = sh_polynomials(dir);
        if (r2 == 0.0) o.p[5] = 0.0f;
        if (!v_out) {
            for (int ch = 0; ch < 3; ++ch) {
                float c = sp.features_dc ? kShC0 * sp.features_dc[3 * i + ch] : 0.0f;
                for (int j = 0; j < n_sh; ++j) c += o.p[j] * sh_constant(j) * W[3 * j + ch];
                out[3 * ((int64_t)v * n + i) + ch] = c;
            }
        } else {
            const float* go = v_out + 3 * ((int64_t)v * n + i);
            float w[kNumSh] = {}, vm[3];
            for (int ch = 0; ch < 3; ++ch) {
                g[3 + ch] += kShC0 * go[ch];
                for (int j = 0; j < n_sh; ++j) {
                    w[j] += sh_grad_constant(j) * W[3 * j + ch] * go[ch];
                    g[6 + 3 * j + ch] += o.p[j] * sh_constant(j) * go[ch];
                }
            }
            if (n_sh == 0) continue;
            sh_polynomials_vjp(dir, o, w, vm);
            for (int k = 0; k < 3; ++k) g[k] += vm[k] * dir.inv;
        }
    }
}

// ---- one view ----
constexpr int kRowBlock = kProjBlock;
// 10M splats: with 8 blocks (64 registers) 121 us, 6 (79) 112, 5 (93) 121, 4 (107) 131: fewer registers cost moves, fewer blocks loads
// under way.
constexpr int kRowBlocksPerSm = 6;

// Components of -centre of view 0 as two floats each, by the block's first three threads; a barrier follows.
__device__ __forceinline__ void stage_centre(ViewCentre<float>& c, const float* __restrict__ viewmats) {
    if (threadIdx.x < 3) {
        const double s = centre_component(viewmats, 0, threadIdx.x);
        c.hi[threadIdx.x] = (float)s;
        c.lo[threadIdx.x] = (float)(s - (double)(float)s);
    }
}

// A splat's inputs; the next tile's are loaded before the current one is worked on.
struct RowInputs { ShRow r; float mean[3], dc[3]; };
__device__ __forceinline__ void load_row_inputs(RowInputs& in, const char* rows, const float* means, const float* dc, uint32_t t) {
    if (rows) in.r = load_sh_row(rows, t);
#pragma unroll
    for (int k = 0; k < 3; ++k) in.mean[k] = means[3 * t + k];
    if (dc)
#pragma unroll
        for (int k = 0; k < 3; ++k) in.dc[k] = dc[3 * t + k];
}

// 68 bytes a splat (row, mean, DC, value) and 280 instructions.  10M splats: 112 us, 6.1 TB/s, 93 % of the copy bandwidth, in a short
// run; called without a pause the GPU reaches its power limit, lowers its clock to 1.7 GHz, and it is 130 us.  The blocks stay for all
// their tiles: the camera's centre is taken once, and the next tile's loads are under way while a tile is worked on (one tile per
// block: 137 us, 158 with the outputs staged).  Multiply-adds and the codes' offsets on pairs of coefficients: 330 instructions before.
__global__ void __launch_bounds__(kRowBlock, kRowBlocksPerSm) sh_eval_fwd_row_kernel(SsbSplats sp, const void* __restrict__ rows, int64_t n,
                                                                                     const float* __restrict__ viewmats, int n_sh, float* __restrict__ out) {
    __shared__ ViewCentre<float> centre_s;
    const int64_t first = (int64_t)blockIdx.x * kRowBlock, step = (int64_t)gridDim.x * kRowBlock;
    // pointers to the tile being loaded, and the splats from its start on
    const char* rp = n_sh > 0 ? (const char*)rows + kShRowBytes * first : nullptr;
    const float* mp = sp.means + 3 * first;
    const float* dp = sp.features_dc ? sp.features_dc + 3 * first : nullptr;
    float* op = out + 3 * first;
    int64_t left = n - first;
    RowInputs in = {};
    load_row_inputs(in, rp, mp, dp, (uint32_t)min((int64_t)threadIdx.x, left - 1));
    stage_centre(centre_s, viewmats);
    __syncthreads();
    const ViewCentre<float> centre = centre_s;
    while (left > 0) {
        const RowInputs now = in;
        const bool mine = threadIdx.x < left;
        left -= step;
        if (left > 0) {
            mp += 3 * step;
            if (rp) rp += kShRowBytes * step;
            if (dp) dp += 3 * step;
            load_row_inputs(in, rp, mp, dp, (uint32_t)min((int64_t)threadIdx.x, left - 1));
        }
        float d2, c[3];
        const Polynomials<float> o = sh_polynomials(view_directions(centre, now.mean, d2));
#pragma unroll
        for (int ch = 0; ch < 3; ++ch) c[ch] = kShC0 * now.dc[ch];
        // coefficients (2k, 2k + 1) side by side; the last pair's second half is coefficient 14 again, times zero
        const float sc[3] = {active_scale(now.r, 0, n_sh), active_scale(now.r, 1, n_sh), active_scale(now.r, 2, n_sh)};
        Pair sum[3] = {make_float2(c[0], 0.0f), make_float2(c[1], 0.0f), make_float2(c[2], 0.0f)};
#pragma unroll
        for (int j = 0; j < kNumSh; j += 2) {
            const int j1 = j + 1 < kNumSh ? j + 1 : j;
            const Pair f = make_float2((sh_constant(j) * code_unit(j)) * o.p[j], (sh_constant(j1) * code_unit(j1)) * o.p[j1]) *
                           make_float2(sc[sh_band(j)], j1 > j ? sc[sh_band(j1)] : 0.0f);
#pragma unroll
            for (int ch = 0; ch < 3; ++ch)
                sum[ch] = fma_(f, make_float2(code_bits(now.r, j, ch), code_bits(now.r, j1, ch)) + make_float2(code_bias(j), code_bias(j1)), sum[ch]);
        }
#pragma unroll
        for (int ch = 0; ch < 3; ++ch) c[ch] = sum[ch].x + sum[ch].y;
        if (mine) {
#pragma unroll
            for (int ch = 0; ch < 3; ++ch) op[3 * threadIdx.x + ch] = c[ch];
            if (!(d2 > kSquareMin && d2 < kSquareMax))
                eval_checked(sp, nullptr, n_sh ? rows : nullptr, (op - out) / 3 + threadIdx.x, n, 1, viewmats, n_sh, out, nullptr, nullptr);
        }
        op += 3 * step;
    }
}

// The same for values in another form: a block's 128 splats' values are staged in shared memory as the projection does.  3M splats: fp32
// 99 us, the copy bandwidth; 16-bit codes 134 and 8-bit ones 148, bound by decoding.  On the kernel of several views: 109, 196, 177.
__global__ void __launch_bounds__(kRowBlock) sh_eval_fwd_staged_kernel(SsbSplats sp, SsbShQuant shq, int64_t n, const float* __restrict__ viewmats, int n_sh,
                                                                       float* __restrict__ out) {
    __shared__ __align__(16) float sh_s[kRowBlock * kShPerSplat];
    __shared__ __align__(16) unsigned char raw_s[kShRawBytes];
    __shared__ ViewCentre<float> centre_s;
    const int64_t first = (int64_t)blockIdx.x * kRowBlock, i = first + threadIdx.x, il = min(i, n - 1);
    const float mean[3] = {sp.means[3 * il], sp.means[3 * il + 1], sp.means[3 * il + 2]};
    float c[3] = {0.f, 0.f, 0.f};
    if (sp.features_dc) { c[0] = sp.features_dc[3 * il]; c[1] = sp.features_dc[3 * il + 1]; c[2] = sp.features_dc[3 * il + 2]; }
    stage_centre(centre_s, viewmats);
    stage_sh(sh_s, raw_s, sp.features_sh, shq.packed, shq.bounds, shq.bits, shq.bounds_stride, first, n);
    __syncthreads();
    if (i >= n) return;
    const float* W = sh_s + threadIdx.x * kShPerSplat;
    float d2;
    const Polynomials<float> o = sh_polynomials(view_directions(centre_s, mean, d2));
#pragma unroll
    for (int ch = 0; ch < 3; ++ch) c[ch] *= kShC0;
#pragma unroll
    for (int j = 0; j < kNumSh; ++j)
        if (j < n_sh) {
            const float f = sh_constant(j) * o.p[j];
#pragma unroll
            for (int ch = 0; ch < 3; ++ch) c[ch] = fmaf(f, W[3 * j + ch], c[ch]);
        }
#pragma unroll
    for (int ch = 0; ch < 3; ++ch) out[3 * i + ch] = c[ch];
    if (!(d2 > kSquareMin && d2 < kSquareMax)) eval_checked(sp, W, nullptr, i, n, 1, viewmats, n_sh, out, nullptr, nullptr);
}

// 260 bytes a splat from 4-bit rows, 204 of them written.  3M splats: 121 us, 6.4 TB/s, 98 % of the copy bandwidth.  A tile's three
// arrays of gradients are contiguous spans, written to shared memory at a stride of 45 words (no bank conflicts) and sent off as three
// bulk copies; with direct stores it was 699 us.  Values in another form are staged in the span that their gradients leave from: fp32 183 us,
// 16-bit codes 211, 8-bit 217 (266, 389, 343 on the kernel of several views).
template <bool ROWS>
__global__ void __launch_bounds__(kRowBlock) sh_eval_bwd_one_kernel(SsbSplats sp, SsbShQuant shq, int64_t n, const float* __restrict__ viewmats, int n_sh,
                                                                    const float* __restrict__ v_out, SsbSplats gr, int accumulate) {
    __shared__ __align__(16) float sh_s[kRowBlock * kShPerSplat];
    __shared__ __align__(16) float mean_s[kRowBlock * 3];
    __shared__ __align__(16) float dc_s[kRowBlock * 3];
    __shared__ __align__(16) unsigned char raw_s[ROWS ? 16 : kShRawBytes];
    __shared__ ViewCentre<float> centre_s;
    const int64_t first = (int64_t)blockIdx.x * kRowBlock, i = first + threadIdx.x, il = min(i, n - 1);
    const void* rows = ROWS && n_sh > 0 ? shq.packed : nullptr;
    ShRow r = {};
    if (rows) r = load_sh_row(rows, il);
    const float mean[3] = {sp.means[3 * il], sp.means[3 * il + 1], sp.means[3 * il + 2]};
    const float g[3] = {v_out[3 * il], v_out[3 * il + 1], v_out[3 * il + 2]};
    stage_centre(centre_s, viewmats);
    if (!ROWS) stage_sh(sh_s, raw_s, sp.features_sh, shq.packed, shq.bounds, shq.bits, shq.bounds_stride, first, n);
    __syncthreads();
    float* W = sh_s + threadIdx.x * kShPerSplat;              // the splat's values, then their gradients
    float d2, w[kNumSh], vm[3];
    const Directions<float> d = view_directions(centre_s, mean, d2);
    const Polynomials<float> o = sh_polynomials(d);
    const bool checked = !(d2 > kSquareMin && d2 < kSquareMax) && i < n;
    float e[6 + kShPerSplat];
    if (checked) eval_checked(sp, W, rows, i, n, 1, viewmats, n_sh, nullptr, v_out, e);
#pragma unroll
    for (int j = 0; j < kNumSh; ++j) {
        const bool active = n_sh > (sh_band(j) + 1) * (sh_band(j) + 1) - 1;
        if (ROWS) {
            const float t = fmaf(code_of(r, j, 2), g[2], fmaf(code_of(r, j, 1), g[1], code_of(r, j, 0) * g[0]));
            w[j] = active ? ((sh_grad_constant(j) * code_unit(j)) * sh_row_scale(r, sh_band(j))) * t : 0.0f;
        } else {
            w[j] = active ? sh_grad_constant(j) * fmaf(W[3 * j + 2], g[2], fmaf(W[3 * j + 1], g[1], W[3 * j] * g[0])) : 0.0f;
        }
#pragma unroll
        for (int ch = 0; ch < 3; ++ch) W[3 * j + ch] = active ? sh_constant(j) * o.p[j] * g[ch] : 0.0f;
    }
    sh_polynomials_vjp(d, o, w, vm);
#pragma unroll
    for (int k = 0; k < 3; ++k) { mean_s[3 * threadIdx.x + k] = vm[k] * d.inv; dc_s[3 * threadIdx.x + k] = kShC0 * g[k]; }
    if (checked) {
        for (int k = 0; k < 3; ++k) { mean_s[3 * threadIdx.x + k] = e[k]; dc_s[3 * threadIdx.x + k] = e[3 + k]; }
        for (int k = 0; k < kShPerSplat; ++k) W[k] = e[6 + k];
    }
    span_written();
    __syncthreads();
    const int count = (int)min((int64_t)kRowBlock, n - first);
    if (gr.features_sh) store_span(gr.features_sh + kShPerSplat * first, sh_s, kShPerSplat * count, kShPerSplat * kRowBlock, accumulate != 0);
    if (gr.means) store_span(gr.means + 3 * first, mean_s, 3 * count, 3 * kRowBlock, accumulate != 0);
    if (gr.features_dc) store_span(gr.features_dc + 3 * first, dc_s, 3 * count, 3 * kRowBlock, accumulate != 0);
    bulk_done();
}

// ---- several views ----
constexpr int kEvalTile = 2 * kProjBlock;      // splats per block and step
constexpr int kCentreChunk = 32;               // views whose centres a block keeps at a time
constexpr int kEvalShBytes = kEvalTile * kShPerSplat * (int)sizeof(float);

__device__ __forceinline__ void stage_centres(ViewCentre<Pair>* centres_s, const float* __restrict__ viewmats, int v0, int views) {
    const int v = threadIdx.x / 3, j = threadIdx.x - 3 * v;
    if (v < kCentreChunk && v0 + v < views) {
        const double s = centre_component(viewmats, v0 + v, j);
        centres_s[v].hi[j] = all<Pair>((float)s);
        centres_s[v].lo[j] = all<Pair>((float)(s - (double)(float)s));
    }
}
static_assert(3 * kCentreChunk <= kProjBlock, "one thread per component of a chunk's centres");

__device__ __forceinline__ void stage_tile(float* sh_s, unsigned char* raw_s, const SsbSplats& sp, const SsbShQuant& shq, int64_t first, int64_t n) {
    stage_sh(sh_s, raw_s, sp.features_sh, shq.packed, shq.bounds, shq.bits, shq.bounds_stride, first, n);
    __syncthreads();
    stage_sh(sh_s + kProjBlock * kShPerSplat, raw_s, sp.features_sh, shq.packed, shq.bounds, shq.bits, shq.bounds_stride, first + kProjBlock, n);
    __syncthreads();
}

// With few splats and many views the views are split over the grid's second dimension: block (., y) takes its share of them, which
// is as if it had been given that many views and the arrays from its first one on.
__device__ __forceinline__ int64_t share_of_views(int& views) {
    const int from = (int)((int64_t)views * blockIdx.y / gridDim.y), to = (int)((int64_t)views * (blockIdx.y + 1) / gridDim.y);
    views = to - from;
    return from;
}

// A tile's inputs travel to shared memory while the tile before is worked on: each thread copies and reads its own two splats', so
// no barrier is needed.
struct TileInputs { uint4 row[4][kProjBlock]; Pair mean[3][kProjBlock], dc[3][kProjBlock]; };
__device__ __forceinline__ void fetch_pairs(const Pair* dst, const float* __restrict__ p, int64_t l0, int64_t l1) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(dst);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s + 8 * kProjBlock * k), "l"(p + 3 * l0 + k) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s + 8 * kProjBlock * k + 4), "l"(p + 3 * l1 + k) : "memory");
    }
}
template <bool ROWS>
__device__ __forceinline__ void fetch_inputs(TileInputs& in, const SsbSplats& sp, bool want_dc, const void* __restrict__ rows, int n_sh, int64_t first, int64_t n) {
    // a thread whose second splat is beyond the array takes its first one twice, one with neither leaves its slots as they are (what
    // it then computes is not stored); clamping to the last splat made the blocks of a split over views queue for one address
    const int64_t l0 = first + threadIdx.x, l1 = l0 + kProjBlock < n ? l0 + kProjBlock : l0;
    if (l0 < n) {
        if (ROWS && n_sh > 0) {
            const uint32_t s = (uint32_t)__cvta_generic_to_shared(&in.row[0][threadIdx.x]);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s + 16 * kProjBlock * k),
                             "l"((const char*)rows + kShRowBytes * (k < 2 ? l0 : l1) + 16 * (k & 1)) : "memory");
        }
        fetch_pairs(&in.mean[0][threadIdx.x], sp.means, l0, l1);
        if (want_dc) fetch_pairs(&in.dc[0][threadIdx.x], sp.features_dc, l0, l1);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ ShRow input_row(const TileInputs& in, int which) {
    const uint4 a = in.row[2 * which][threadIdx.x], b = in.row[2 * which + 1][threadIdx.x];
    return ShRow{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}

// W[j][ch] of both splats times sh_constant(j) or, for the backward pass, sh_grad_constant(j); zero above the active degree.
template <bool ROWS, bool GRAD>
__device__ __forceinline__ void read_coefficients(Pair W[kShPerSplat], const float* sh_s, const TileInputs& in, int n_sh) {
    if (ROWS) {
        const ShRow a = input_row(in, 0), b = input_row(in, 1);
#pragma unroll
        for (int j = 0; j < kNumSh; ++j) {
            const Pair f = ((GRAD ? sh_grad_constant(j) : sh_constant(j)) * code_unit(j)) * make_float2(active_scale(a, sh_band(j), n_sh), active_scale(b, sh_band(j), n_sh));
#pragma unroll
            for (int ch = 0; ch < 3; ++ch) W[3 * j + ch] = f * code_of(a, b, j, ch);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kNumSh; ++j)
#pragma unroll
            for (int ch = 0; ch < 3; ++ch) {
                const int k = 3 * j + ch;
                W[k] = j < n_sh ? (GRAD ? sh_grad_constant(j) : sh_constant(j)) * make_float2(sh_s[threadIdx.x * kShPerSplat + k], sh_s[(threadIdx.x + kProjBlock) * kShPerSplat + k])
                                : all<Pair>(0.0f);
            }
    }
}

// The sum over j as a polynomial in z whose coefficients belong to the azimuthal functions 1, x, y, x^2 - y^2, 2xy, x^3 - 3xy^2 and
// 3x^2 y - y^3: fifteen multiply-adds like the sum itself, but the fifteen p_j need not be formed, only the azimuthal functions.
// W comes in as sh_constant(j) W_j and leaves as: [0] z^3 [1] z^2 [2] z [3] 1 (with dc) | [4] x z^2 [5] x z [6] x | [7] y z^2 [8] y z
// [9] y | [10] (x^2 - y^2) z [11] x^2 - y^2 | [12] 2xy z [13] 2xy | [14] x^3 - 3xy^2 [15] 3x^2 y - y^3, of channel ch at 3 * k + ch.
__device__ __forceinline__ void to_azimuthal(Pair A[16 * 3], const Pair W[kShPerSplat], const Pair dc[3]) {
#pragma unroll
    for (int ch = 0; ch < 3; ++ch) {
        A[0 + ch] = W[33 + ch]; A[3 + ch] = W[15 + ch]; A[6 + ch] = fma_(-0.6f, W[33 + ch], W[3 + ch]); A[9 + ch] = fma_(-1.0f / 3.0f, W[15 + ch], dc[ch]);
        A[12 + ch] = W[36 + ch]; A[15 + ch] = W[18 + ch] + W[18 + ch]; A[18 + ch] = fma_(-0.2f, W[36 + ch], W[6 + ch]);
        A[21 + ch] = W[30 + ch]; A[24 + ch] = W[12 + ch] + W[12 + ch]; A[27 + ch] = fma_(-0.2f, W[30 + ch], W[0 + ch]);
        A[30 + ch] = W[39 + ch]; A[33 + ch] = W[21 + ch];
        A[36 + ch] = W[27 + ch]; A[39 + ch] = W[9 + ch];
        A[42 + ch] = W[42 + ch]; A[45 + ch] = W[24 + ch];
    }
}

// What the registers allow (156 forward; backward 252 from rows, 255 and 24 bytes of spills from other storages); the grids are this many
// blocks, which walk the tiles.  Four forward blocks make the compiler spill: 73 us against 64.
constexpr int kFwdBlocksPerSm = 3, kBwdBlocksPerSm = 2;
constexpr int kMaxSplit = 8;                   // blocks that share a tile's views in the backward pass, a cluster

// Per (splat, view): the direction (12 operations), the azimuthal functions (7) and 45 multiply-adds.  1M splats, 16 views: 64 us;
// 20.1M packed instructions at the three cycles of the register file are 52 us, the bytes (248 MB) 38 us.
template <bool ROWS>
__global__ void __launch_bounds__(kProjBlock, kFwdBlocksPerSm) sh_eval_fwd_views_kernel(SsbSplats sp, SsbShQuant shq, int64_t n, int views,
                                                                                        const float* __restrict__ viewmats, int n_sh,
                                                                                        float* __restrict__ out) {
    extern __shared__ __align__(16) unsigned char dyn_s[];
    __shared__ ViewCentre<Pair> centres_s[kCentreChunk];
    __shared__ TileInputs in;
    float* sh_s = (float*)dyn_s;
    const bool with_dc = sp.features_dc != nullptr;
    const int64_t stride = (int64_t)gridDim.x * kEvalTile, from = share_of_views(views);
    viewmats += 16 * from;
    out += 3 * from * n;
    fetch_inputs<ROWS>(in, sp, with_dc, shq.packed, n_sh, (int64_t)blockIdx.x * kEvalTile, n);
    stage_centres(centres_s, viewmats, 0, views);
    __syncthreads();
    for (int64_t first = (int64_t)blockIdx.x * kEvalTile; first < n; first += stride) {
        const int64_t i0 = first + threadIdx.x, i1 = i0 + kProjBlock;
        if (!ROWS) {
            __syncthreads();
            stage_tile(sh_s, dyn_s + kEvalShBytes, sp, shq, first, n);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        Pair mean[3], dc[3], W[kShPerSplat];
#pragma unroll
        for (int k = 0; k < 3; ++k) { mean[k] = in.mean[k][threadIdx.x]; dc[k] = with_dc ? kShC0 * in.dc[k][threadIdx.x] : all<Pair>(0.f); }
        read_coefficients<ROWS, false>(W, sh_s, in, n_sh);
        Pair A[16 * 3];
        to_azimuthal(A, W, dc);
        fetch_inputs<ROWS>(in, sp, with_dc, shq.packed, n_sh, first + stride, n);
        float least = kSquareMax, most = kSquareMin;
        for (int v0 = 0; v0 < views; v0 += kCentreChunk) {
            if (views > kCentreChunk) {
                __syncthreads();
                stage_centres(centres_s, viewmats, v0, views);
                __syncthreads();
            }
            const int v1 = min(views - v0, kCentreChunk);
            float* o0 = out + 3 * ((int64_t)v0 * n + i0);
            for (int v = 0; v < v1; ++v, o0 += 3 * n) {
                Pair d2, c[3];
                const Directions<Pair> d = view_directions(centres_s[v], mean, d2);
                least = fminf(least, fminf(d2.x, d2.y)); most = max_nan(most, d2.x, d2.y);
                const Pair ny = -1.0f * d.y, c1 = fma_(d.x, d.x, ny * d.y), s1 = (d.x + d.x) * d.y;
                const Pair c3 = fma_(d.x, c1, ny * s1), s3 = fma_(d.x, s1, d.y * c1);
#pragma unroll
                for (int ch = 0; ch < 3; ++ch) {
                    Pair t = fma_(d.z, fma_(d.z, fma_(d.z, A[ch], A[3 + ch]), A[6 + ch]), A[9 + ch]);
                    t = fma_(d.x, fma_(d.z, fma_(d.z, A[12 + ch], A[15 + ch]), A[18 + ch]), t);
                    t = fma_(d.y, fma_(d.z, fma_(d.z, A[21 + ch], A[24 + ch]), A[27 + ch]), t);
                    t = fma_(c1, fma_(d.z, A[30 + ch], A[33 + ch]), t);
                    t = fma_(s1, fma_(d.z, A[36 + ch], A[39 + ch]), t);
                    c[ch] = fma_(s3, A[45 + ch], fma_(c3, A[42 + ch], t));
                }
#pragma unroll
                for (int ch = 0; ch < 3; ++ch) {
                    if (i0 < n) o0[ch] = c[ch].x;
                    if (i1 < n) o0[3 * kProjBlock + ch] = c[ch].y;
                }
            }
        }
        if (!(least > kSquareMin && most < kSquareMax)) {
            const void* rows = ROWS && n_sh > 0 ? shq.packed : nullptr;
            if (i0 < n) eval_checked(sp, sh_s + threadIdx.x * kShPerSplat, rows, i0, n, views, viewmats, n_sh, out, nullptr, nullptr);
            if (i1 < n) eval_checked(sp, sh_s + (threadIdx.x + kProjBlock) * kShPerSplat, rows, i1, n, views, viewmats, n_sh, out, nullptr, nullptr);
        }
    }
}

// The gradients of the next views travel to shared memory while a view is worked on: each thread copies and reads its own six
// numbers, so no barrier is needed.
constexpr int kGradAhead = 3;
struct GradRing { Pair g[kGradAhead + 1][3][kProjBlock]; };
// What the ring fetches next: view after view of a tile, then on into the block's next tile.
struct GradCursor { const float* p0; const float* p1; int64_t first; int view; };
__device__ __forceinline__ void cursor_tile(GradCursor& c, const float* v_out, int64_t n, int64_t first) {
    c.first = first;
    c.view = 0;
    c.p0 = v_out + 3 * min(first + threadIdx.x, n - 1);
    c.p1 = v_out + 3 * min(first + threadIdx.x + kProjBlock, n - 1);
}
__device__ __forceinline__ void fetch_grads(GradRing& ring, int slot, GradCursor& c, const float* v_out, int64_t n, int views, int64_t stride) {
    if (c.first < n) {
        const uint32_t s = (uint32_t)__cvta_generic_to_shared(&ring.g[slot][0][threadIdx.x]);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s + 8 * kProjBlock * k), "l"(c.p0 + k) : "memory");
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s + 8 * kProjBlock * k + 4), "l"(c.p1 + k) : "memory");
        }
        c.p0 += 3 * n;
        c.p1 += 3 * n;
        if (++c.view == views) cursor_tile(c, v_out, n, c.first + stride);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// dst[k] = the sum over the cluster's blocks of their span[k], for this block's share of k; spans are 16-byte aligned.  The loads of
// a step are independent: one float at a time the join of 24 tiles took 12 us.
__device__ __forceinline__ void join_span(float* dst, float* span_s, int count, bool add) {
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int blocks = (int)gridDim.y, quads = (count + 3) / 4, from = quads * (int)blockIdx.y / blocks, to = quads * ((int)blockIdx.y + 1) / blocks;
#pragma unroll 4
    for (int k = from + threadIdx.x; k < to; k += kProjBlock) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 0; q < kMaxSplit; ++q)
            if (q < blocks) {
                const float4 b = *(const float4*)cluster.map_shared_rank(span_s + 4 * k, q);
                a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
            }
        const float e[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (4 * k + j < count) dst[4 * k + j] = add ? dst[4 * k + j] + e[j] : e[j];
    }
}

// Per (splat, view): direction and polynomials (35 operations), 45 multiply-adds for the coefficients' gradients, 45 for the sums w_j
// and 40 for the mean's.  The 45 gradients of both splats stay in registers over all views, so nothing is added in memory and the sum
// has one order.  1M splats, 16 views: 153 us; 47.1M packed instructions at three cycles are 122 us, the bytes (440 MB) 67 us.
template <bool ROWS>
__global__ void __launch_bounds__(kProjBlock, kBwdBlocksPerSm) sh_eval_bwd_views_kernel(SsbSplats sp, SsbShQuant shq, int64_t n, int views,
                                                                                        const float* __restrict__ viewmats, int n_sh,
                                                                                        const float* __restrict__ v_out, SsbSplats gr, int accumulate) {
    extern __shared__ __align__(16) unsigned char dyn_s[];
    __shared__ __align__(16) float mean_s[kEvalTile * 3];
    __shared__ __align__(16) float dc_s[kEvalTile * 3];
    __shared__ GradRing ring;
    __shared__ TileInputs in;
    __shared__ ViewCentre<Pair> centres_s[kCentreChunk];
    float* sh_s = (float*)dyn_s;                 // values on the way in, their gradients on the way out
    const int64_t stride = (int64_t)gridDim.x * kEvalTile, from = share_of_views(views);
    viewmats += 16 * from;
    v_out += 3 * from * n;
    GradCursor ahead;
    int slot = 0;
    cursor_tile(ahead, v_out, n, (int64_t)blockIdx.x * kEvalTile);
    fetch_inputs<ROWS>(in, sp, false, shq.packed, n_sh, (int64_t)blockIdx.x * kEvalTile, n);
    for (int k = 0; k < kGradAhead && views > 0; ++k) fetch_grads(ring, k, ahead, v_out, n, views, stride);
    stage_centres(centres_s, viewmats, 0, views);
    for (int64_t first = (int64_t)blockIdx.x * kEvalTile; first < n; first += stride) {
        const int64_t i0 = first + threadIdx.x, i1 = i0 + kProjBlock;
        __syncthreads();
        if (!ROWS) stage_tile(sh_s, dyn_s + kEvalShBytes, sp, shq, first, n);
        // at least `views` groups were begun after the tile's inputs, the last kGradAhead of which may be under way
        if (views >= kGradAhead) asm volatile("cp.async.wait_group %0;" ::"n"(kGradAhead) : "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
        Pair mean[3], g_mean[3], g_dc[3], g_sh[kShPerSplat], W[kShPerSplat];
#pragma unroll
        for (int k = 0; k < 3; ++k) mean[k] = in.mean[k][threadIdx.x];
        read_coefficients<ROWS, true>(W, sh_s, in, n_sh);
        fetch_inputs<ROWS>(in, sp, false, shq.packed, n_sh, first + stride, n);
#pragma unroll
        for (int k = 0; k < 3; ++k) g_mean[k] = g_dc[k] = all<Pair>(0.f);
#pragma unroll
        for (int k = 0; k < kShPerSplat; ++k) g_sh[k] = all<Pair>(0.f);
        float least = kSquareMax, most = kSquareMin;
        for (int v0 = 0; v0 < views; v0 += kCentreChunk) {
            if (views > kCentreChunk) {
                __syncthreads();
                stage_centres(centres_s, viewmats, v0, views);
                __syncthreads();
            }
            const int v1 = min(views - v0, kCentreChunk);
            for (int v = 0; v < v1; ++v) {
                Pair d2, g[3], w[kNumSh], vm[3];
                fetch_grads(ring, (slot + kGradAhead) & kGradAhead, ahead, v_out, n, views, stride);
                asm volatile("cp.async.wait_group %0;" ::"n"(kGradAhead) : "memory");
#pragma unroll
                for (int k = 0; k < 3; ++k) g[k] = ring.g[slot][k][threadIdx.x];
                slot = (slot + 1) & kGradAhead;
                const Directions<Pair> d = view_directions(centres_s[v], mean, d2);
                const Polynomials<Pair> o = sh_polynomials(d);
                least = fminf(least, fminf(d2.x, d2.y)); most = max_nan(most, d2.x, d2.y);
#pragma unroll
                for (int j = 0; j < kNumSh; ++j) {
                    w[j] = W[3 * j] * g[0];
                    w[j] = fma_(W[3 * j + 1], g[1], w[j]);
                    w[j] = fma_(W[3 * j + 2], g[2], w[j]);
#pragma unroll
                    for (int ch = 0; ch < 3; ++ch) g_sh[3 * j + ch] = fma_(o.p[j], g[ch], g_sh[3 * j + ch]);
                }
                sh_polynomials_vjp(d, o, w, vm);
#pragma unroll
                for (int k = 0; k < 3; ++k) { g_dc[k] = g_dc[k] + g[k]; g_mean[k] = fma_(vm[k], d.inv, g_mean[k]); }
            }
        }
        float e0[6 + kShPerSplat], e1[6 + kShPerSplat];
        const bool checked = !(least > kSquareMin && most < kSquareMax) && i0 < n;
        if (checked) {
            const void* rows = ROWS && n_sh > 0 ? shq.packed : nullptr;
            eval_checked(sp, sh_s + threadIdx.x * kShPerSplat, rows, i0, n, views, viewmats, n_sh, nullptr, v_out, e0);
            if (i1 < n) eval_checked(sp, sh_s + (threadIdx.x + kProjBlock) * kShPerSplat, rows, i1, n, views, viewmats, n_sh, nullptr, v_out, e1);
        }
        bulk_done();
        __syncthreads();          // the previous tile's copies have left, and every thread has read its values
        const int t0 = threadIdx.x, t1 = threadIdx.x + kProjBlock;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            mean_s[3 * t0 + k] = g_mean[k].x; mean_s[3 * t1 + k] = g_mean[k].y;
            dc_s[3 * t0 + k] = kShC0 * g_dc[k].x; dc_s[3 * t1 + k] = kShC0 * g_dc[k].y;
        }
#pragma unroll
        for (int j = 0; j < kNumSh; ++j)
#pragma unroll
            for (int ch = 0; ch < 3; ++ch) {
                const Pair t = j < n_sh ? sh_constant(j) * g_sh[3 * j + ch] : all<Pair>(0.0f);
                sh_s[kShPerSplat * t0 + 3 * j + ch] = t.x; sh_s[kShPerSplat * t1 + 3 * j + ch] = t.y;
            }
        if (checked) {
            for (int k = 0; k < 3; ++k) { mean_s[3 * t0 + k] = e0[k]; mean_s[3 * t1 + k] = e1[k]; dc_s[3 * t0 + k] = e0[3 + k]; dc_s[3 * t1 + k] = e1[3 + k]; }
            for (int k = 0; k < kShPerSplat; ++k) { sh_s[kShPerSplat * t0 + k] = e0[6 + k]; sh_s[kShPerSplat * t1 + k] = e1[6 + k]; }
        }
        const int count = (int)min((int64_t)kEvalTile, n - first);
        if (gridDim.y > 1) {      // the tile's blocks form a cluster: each adds up its part of the spans over all of them, in view order
            cooperative_groups::this_cluster().sync();
            if (gr.means) join_span(gr.means + 3 * first, mean_s, 3 * count, accumulate != 0);
            if (gr.features_dc) join_span(gr.features_dc + 3 * first, dc_s, 3 * count, accumulate != 0);
            if (gr.features_sh) join_span(gr.features_sh + kShPerSplat * first, sh_s, kShPerSplat * count, accumulate != 0);
            cooperative_groups::this_cluster().sync();      // nobody leaves, or writes its spans again, while they are being read
            continue;
        }
        span_written();
        __syncthreads();
        if (gr.means) store_span(gr.means + 3 * first, mean_s, 3 * count, 3 * kEvalTile, accumulate != 0);
        if (gr.features_dc) store_span(gr.features_dc + 3 * first, dc_s, 3 * count, 3 * kEvalTile, accumulate != 0);
        if (gr.features_sh) store_span(gr.features_sh + kShPerSplat * first, sh_s, kShPerSplat * count, kShPerSplat * kEvalTile, accumulate != 0);
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
    cudaStream_t st = (cudaStream_t)stream;
    const bool rows = q.bits == 4 || n_sh == 0;
    const unsigned tiles = (unsigned)ceil_div(n, kRowBlock);
    if (rows && cams->count == 1) {
        sh_eval_fwd_row_kernel<<<std::min(tiles, 148u * kRowBlocksPerSm), kRowBlock, 0, st>>>(*splats, q.packed, n, cams->d_viewmats, n_sh, d_values);
    } else if (cams->count == 1) {
        sh_eval_fwd_staged_kernel<<<tiles, kRowBlock, 0, st>>>(*splats, q, n, cams->d_viewmats, n_sh, d_values);
    } else {
        const unsigned resident = 148 * kFwdBlocksPerSm, tiles2 = (unsigned)std::min<int64_t>(ceil_div(n, kEvalTile), resident);
        // few tiles: their views over the blocks that fit beside them (1 splat and 1 000 views 157 -> 3.9 us, 6 007 and 16 5.2 -> 4.1)
        const dim3 blocks(tiles2, std::max(1u, std::min((unsigned)cams->count, resident / tiles2)));
        constexpr int smem = kEvalShBytes + kShRawBytes;
        if (rows) sh_eval_fwd_views_kernel<true><<<blocks, kProjBlock, 0, st>>>(*splats, q, n, cams->count, cams->d_viewmats, n_sh, d_values);
        else {
            if (int e = ensure_dynamic_smem((const void*)sh_eval_fwd_views_kernel<false>, smem)) return e;
            sh_eval_fwd_views_kernel<false><<<blocks, kProjBlock, smem, st>>>(*splats, q, n, cams->count, cams->d_viewmats, n_sh, d_values);
        }
    }
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
    cudaStream_t st = (cudaStream_t)stream;
    const bool rows = q.bits == 4 || n_sh == 0;
    if (cams->count == 1) {
        const unsigned tiles = (unsigned)ceil_div(n, kRowBlock);
        if (rows) sh_eval_bwd_one_kernel<true><<<tiles, kRowBlock, 0, st>>>(*splats, q, n, cams->d_viewmats, n_sh, d_v_values, *grads, accumulate);
        else sh_eval_bwd_one_kernel<false><<<tiles, kRowBlock, 0, st>>>(*splats, q, n, cams->d_viewmats, n_sh, d_v_values, *grads, accumulate);
    } else {
        const unsigned resident = 148 * kBwdBlocksPerSm, tiles = (unsigned)std::min<int64_t>(ceil_div(n, kEvalTile), resident);
        // Few tiles and many views: a tile's views over a cluster of blocks.  A view costs a tile about 0.4 us, the join 3.5: 300 splats
        // and 70 views 37 -> 10 us, 6 007 and 16 10.8 -> 8.8, but 6 007 and 4 6.0 -> 8.5.
        unsigned split = 1;
        while (cams->count >= 16 && split < kMaxSplit && 2 * split * tiles <= resident && 2 * (int64_t)split <= cams->count / 2) split *= 2;
        auto* kernel = rows ? sh_eval_bwd_views_kernel<true> : sh_eval_bwd_views_kernel<false>;
        const int smem = kEvalShBytes + (rows ? 0 : kShRawBytes);
        if (int e = ensure_dynamic_smem((const void*)kernel, smem)) return e;
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = 1; cluster.val.clusterDim.y = split; cluster.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(tiles, split); cfg.blockDim = dim3(kProjBlock); cfg.dynamicSmemBytes = (size_t)smem; cfg.stream = st;
        cfg.attrs = &cluster; cfg.numAttrs = split > 1 ? 1 : 0;
        SSB_CUDA(cudaLaunchKernelEx(&cfg, kernel, *splats, q, n, (int)cams->count, cams->d_viewmats, n_sh, d_v_values, *grads, accumulate));
    }
    SSB_LAUNCHED("sh_eval_bwd_kernel");
    return SSB_OK;
}

}  // extern "C"
