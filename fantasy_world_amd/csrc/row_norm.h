// Row statistics and the normalise / modulate arithmetic of the wave-per-row norm kernels (elementwise.hip, residual_norm.hip): one
// definition, so that a fused pass returns the bits of the separate ones.
#pragma once
#include "fw_common.h"

// The normalise / modulate arithmetic of BOTH LayerNorm wave kernels, spelled out operation by operation (no contraction, no
// reassociation): u = (v - mean) * rstd;  [u = u * w (+ b)];  u = fma(u, scale, u) = u * (1 + scale) in one rounding;  u = u + shift.
// A sequence shard (few rows per rank: one-wave-per-row kernel) and the unsharded forward (LDS-staged kernel) must agree bit for bit.
__device__ __forceinline__ f32x4_t ln_finish(f32x4_t v, float mean, float rstd, bool has_w, f32x4_t w4, bool has_b, f32x4_t b4,
                                             bool has_scale, f32x4_t sc, bool has_shift, f32x4_t sh) {
    // Every fusion is spelled out (explicit fma) and every place where the back end could still contract or reassociate under
    // -ffast-math (it honours the function-level unsafe-fp-math attribute, not the per-statement pragmas) is fenced by an empty asm:
    // the two LayerNorm kernels must emit the same arithmetic whatever their surrounding code looks like.
    f32x4_t t;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float u = v[j] - mean;
        asm volatile("" : "+v"(u));
        u = u * rstd;
        asm volatile("" : "+v"(u));
        if (has_w) u = has_b ? __builtin_fmaf(u, w4[j], b4[j]) : u * w4[j];
        if (has_scale) u = __builtin_fmaf(u, sc[j], u);
        if (has_shift) { asm volatile("" : "+v"(u)); u = u + sh[j]; }
        t[j] = u;
    }
    return t;
}

// Row statistics of BOTH LayerNorm wave kernels, with the summation order pinned (no reassociation under -ffast-math): the LDS-staged
// kernel (unsharded forward) and the one-wave-per-row kernel (a sequence shard's few rows) must produce the same mean / rstd bits.
// (Round 3: with VPL = 4 the compiler associated the two kernels' sums differently -- caught by the sharded-vs-unsharded bit test.)
template <int VPL>
__device__ __forceinline__ void ln_stats(const f32x4_t (&v)[VPL], int C, float eps, float& mean, float& rstd) {
    // pinned order: chunk sums (a + b) + (c + d) accumulated left to right, squares by explicit fma, 1 / C as one reciprocal used
    // by both statistics; the asm fences keep the back end from re-associating / contracting across statements
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        float a = v[i][0] + v[i][1], b = v[i][2] + v[i][3];
        asm volatile("" : "+v"(a), "+v"(b));
        float c = a + b;
        asm volatile("" : "+v"(c));
        s = s + c;
        asm volatile("" : "+v"(s));
    }
    float inv_c = 1.0f / (float)C;
    asm volatile("" : "+v"(inv_c));
    mean = wave_sum(s) * inv_c;
    asm volatile("" : "+v"(mean));
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float d = v[i][j] - mean;
            asm volatile("" : "+v"(d));
            q = __builtin_fmaf(d, d, q);
        }
    rstd = rsqrtf(__builtin_fmaf(wave_sum(q), inv_c, eps));
}
