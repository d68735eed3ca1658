// Spherical harmonics on the device: the basis and its gradient, and the ways a block of splats' SH coefficients are read
// (fp32, 16- and 8-bit codes against shared bounds, 4-bit rows).  Used by the projection kernels (project.cu) and by the
// product on its own (sh.cu).
#pragma once

#include "ssb_common.cuh"

namespace ssb {

constexpr int kProjBlock = 128;
constexpr int kShPerSplat = 3 * kNumSh;  // 45

// Real SH basis, bands 1..3, at a unit direction (src/shaders/harmonics.slang:154-251).
__device__ __forceinline__ void sh_basis(float x, float y, float z, float b[kNumSh]) {
    const float c1 = 0.48860251190292f;
    b[0] = -c1 * y; b[1] = c1 * z; b[2] = -c1 * x;
    float z2 = z * z;
    float t0b = -1.092548430592079f * z;
    const float c2a = 0.5462742152960395f;
    float fC1 = x * x - y * y, fS1 = 2.f * x * y;
    b[3] = c2a * fS1; b[4] = t0b * y; b[5] = 0.9461746957575601f * z2 - 0.3153915652525201f;
    b[6] = t0b * x; b[7] = c2a * fC1;
    float t0c = -2.285228997322329f * z2 + 0.4570457994644658f;
    float t1b = 1.445305721320277f * z;
    const float c3a = -0.5900435899266435f;
    float fC2 = x * fC1 - y * fS1, fS2 = x * fS1 + y * fC1;
    b[8] = c3a * fS2; b[9] = t1b * fS1; b[10] = t0c * y;
    b[11] = z * (1.865881662950577f * z2 - 1.119528997770346f);
    b[12] = t0c * x; b[13] = t1b * fC1; b[14] = c3a * fC2;
}

// Gradient of the SH basis with respect to the (unit) direction, contracted
// with the per-coefficient weights w[j] = sum_ch sh[j][ch] * vc[ch].
__device__ __forceinline__ void sh_basis_vjp(float x, float y, float z, const float w[kNumSh], float v[3]) {
    const float c1 = 0.48860251190292f, c2a = 0.5462742152960395f, c2b = 1.092548430592079f;
    const float c3a = -0.5900435899266435f, c3b = 1.445305721320277f, c3c = 2.285228997322329f;
    float z2 = z * z;
    float t0c = -c3c * z2 + 0.4570457994644658f;
    float fC1 = x * x - y * y, fS1 = 2.f * x * y;
    float vx = -c1 * w[2], vy = -c1 * w[0], vz = c1 * w[1];
    vx += 2.f * c2a * y * w[3] - c2b * z * w[6] + 2.f * c2a * x * w[7];
    vy += 2.f * c2a * x * w[3] - c2b * z * w[4] - 2.f * c2a * y * w[7];
    vz += -c2b * y * w[4] + 2.f * 0.9461746957575601f * z * w[5] - c2b * x * w[6];
    vx += c3a * 3.f * fS1 * w[8] + 2.f * c3b * y * z * w[9] + t0c * w[12] + 2.f * c3b * z * x * w[13] + c3a * 3.f * fC1 * w[14];
    vy += c3a * 3.f * fC1 * w[8] + 2.f * c3b * x * z * w[9] + t0c * w[10] - 2.f * c3b * z * y * w[13] - c3a * 3.f * fS1 * w[14];
    vz += c3b * fS1 * w[9] - 2.f * c3c * z * y * w[10] + (3.f * 1.865881662950577f * z2 - 1.119528997770346f) * w[11]
        - 2.f * c3c * z * x * w[12] + c3b * fC1 * w[13];
    v[0] = vx; v[1] = vy; v[2] = vz;
}

// ---- 4-bit rows (SsbShQuant::bits = 4) --------------------------------------
// One 32-byte row per splat, so a splat's coefficients are one DRAM sector.  Words 2c and 2c + 1 hold channel c: coefficient
// j's code q + 8 (q in -7..7) in bits 4 (j % 8) of word 2c + j / 8.  Words 6 and 7 hold the bf16 scales of bands 1, 2 | 3.
constexpr int kShRowBytes = 32;

struct ShRow { uint32_t w[8]; };

__device__ __forceinline__ ShRow load_sh_row(const void* __restrict__ rows, int64_t splat) {
    ShRow r;
    const uint4* p = (const uint4*)((const char*)rows + kShRowBytes * splat);
    const uint4 a = p[0], b = p[1];
    r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
    r.w[4] = b.x; r.w[5] = b.y; r.w[6] = b.z; r.w[7] = b.w;
    return r;
}
__device__ __forceinline__ float sh_row_scale(const ShRow& r, int band) {       // band 0..2
    return __uint_as_float(band == 1 ? r.w[6] & 0xffff0000u : (band == 0 ? r.w[6] : r.w[7]) << 16);
}
__device__ __forceinline__ constexpr int sh_band(int j) { return j < 3 ? 0 : (j < 8 ? 1 : 2); }
// The code of coefficient j, channel ch, as a float: the four bits become the low mantissa bits of 2^23.
__device__ __forceinline__ float sh_row_code(const ShRow& r, int j, int ch) {
    return __uint_as_float(((r.w[2 * ch + (j >> 3)] >> (4 * (j & 7))) & 15u) | 0x4b000000u) - 8388616.0f;
}

// The row's 45 values (coefficient-major, colour-minor), exact: a code times a bf16 scale has eleven significant bits.
__device__ __forceinline__ void decode_sh_row(const ShRow& r, float* __restrict__ out) {
#pragma unroll
    for (int j = 0; j < kNumSh; ++j) {
        const float s = sh_row_scale(r, sh_band(j));
#pragma unroll
        for (int ch = 0; ch < 3; ++ch) out[3 * j + ch] = s * sh_row_code(r, j, ch);
    }
}

// Loads the block's SH span into shared memory as fp32 (decoding packed codes).
// A full block's span starts on a 16-byte boundary in every format (128 * 45 cells), so it is
// brought in with 16-byte asynchronous copies (global -> shared without passing through
// registers, all of a thread's copies in flight at once): fp32 coefficients straight into
// sh_s, packed codes into raw_s, from where they are decoded 8 (16-bit) or 16 (8-bit) at a
// time -- the codes of one vector share a bounds entry whenever the bounds stride is a
// multiple of the vector's cell count.  Register-staged 16-byte loads were measured slower
// than 4-byte ones here; the asynchronous copies are a quarter faster than either.
// Partial blocks and unaligned arrays take 4-byte loads.
__device__ __forceinline__ void async_copy_span(void* smem_dst, const void* gmem_src, int n_vec16) {
    const uint32_t sdst = (uint32_t)__cvta_generic_to_shared(smem_dst);
    const uint4* src = (const uint4*)gmem_src;
    for (int v = threadIdx.x; v < n_vec16; v += kProjBlock)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sdst + 16u * (uint32_t)v), "l"(src + v) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ void async_copy_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

constexpr int kShRawBytes = kProjBlock * kShPerSplat * 2;   // a block's 16-bit codes

__device__ __forceinline__ void stage_sh(
    float* sh_s, unsigned char* raw_s, const float* __restrict__ sh_f32, const void* __restrict__ packed, const float* __restrict__ bounds,
    int bits, int64_t bounds_stride, int64_t first_splat, int64_t n) {
    if (bits == 4) {        // a thread decodes its own splat's row: two 16-byte loads instead of a share of the block's span
        if (first_splat + threadIdx.x < n) decode_sh_row(load_sh_row(packed, first_splat + threadIdx.x), sh_s + threadIdx.x * kShPerSplat);
        return;
    }
    const int64_t base = first_splat * kShPerSplat;
    const int count = (int)min((int64_t)kProjBlock, n - first_splat) * kShPerSplat;
    const bool quant = bits == 8 || bits == 16;
    const void* arr = quant ? packed : (const void*)sh_f32;
    const bool full = count == kProjBlock * kShPerSplat && ((uintptr_t)arr & 15) == 0;
    if (full && !quant) {
        async_copy_span(sh_s, sh_f32 + base, kProjBlock * kShPerSplat / 4);
        async_copy_wait();
    } else if (full && bits == 16 && (bounds_stride & 7) == 0) {
        async_copy_span(raw_s, (const uint16_t*)packed + base, kProjBlock * kShPerSplat / 8);
        const int64_t b0 = base / bounds_stride;
        const unsigned r0 = (unsigned)(base - b0 * bounds_stride), stride = (unsigned)min(bounds_stride, (int64_t)0x7fffffff);
        const float inv = 1.0f / 65535.0f;
        async_copy_wait();
        __syncthreads();
        for (int v = threadIdx.x; v < kProjBlock * kShPerSplat / 8; v += kProjBlock) {
            const uint4 c = ((const uint4*)raw_s)[v];
            const float2 mm = ((const float2*)bounds)[b0 + (r0 + 8u * v) / stride];
            const float d = mm.y - mm.x;
            float4 lo, hi;
            lo.x = mm.x + d * ((float)(c.x & 0xffffu) * inv); lo.y = mm.x + d * ((float)(c.x >> 16) * inv);
            lo.z = mm.x + d * ((float)(c.y & 0xffffu) * inv); lo.w = mm.x + d * ((float)(c.y >> 16) * inv);
            hi.x = mm.x + d * ((float)(c.z & 0xffffu) * inv); hi.y = mm.x + d * ((float)(c.z >> 16) * inv);
            hi.z = mm.x + d * ((float)(c.w & 0xffffu) * inv); hi.w = mm.x + d * ((float)(c.w >> 16) * inv);
            ((float4*)sh_s)[2 * v] = lo; ((float4*)sh_s)[2 * v + 1] = hi;
        }
    } else if (full && bits == 8 && (bounds_stride & 15) == 0) {
        async_copy_span(raw_s, (const uint8_t*)packed + base, kProjBlock * kShPerSplat / 16);
        const int64_t b0 = base / bounds_stride;
        const unsigned r0 = (unsigned)(base - b0 * bounds_stride), stride = (unsigned)min(bounds_stride, (int64_t)0x7fffffff);
        const float inv = 1.0f / 255.0f;
        async_copy_wait();
        __syncthreads();
        for (int v = threadIdx.x; v < kProjBlock * kShPerSplat / 16; v += kProjBlock) {
            const uint4 c = ((const uint4*)raw_s)[v];
            const float2 mm = ((const float2*)bounds)[b0 + (r0 + 16u * v) / stride];
            const float d = mm.y - mm.x;
            const unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float4 o;
                o.x = mm.x + d * ((float)(w[k] & 0xffu) * inv); o.y = mm.x + d * ((float)((w[k] >> 8) & 0xffu) * inv);
                o.z = mm.x + d * ((float)((w[k] >> 16) & 0xffu) * inv); o.w = mm.x + d * ((float)(w[k] >> 24) * inv);
                ((float4*)sh_s)[4 * v + k] = o;
            }
        }
    } else if (quant) {
        const float inv = bits == 8 ? (1.0f / 255.0f) : (1.0f / 65535.0f);
        for (int i = threadIdx.x; i < count; i += kProjBlock) {
            int64_t cell = base + i;
            float q = bits == 8 ? (float)((const uint8_t*)packed)[cell] : (float)((const uint16_t*)packed)[cell];
            float2 mm = ((const float2*)bounds)[cell / bounds_stride];
            sh_s[i] = mm.x + (mm.y - mm.x) * (q * inv);
        }
    } else {
        for (int i = threadIdx.x; i < count; i += kProjBlock) sh_s[i] = sh_f32[base + i];
    }
}

}  // namespace ssb
