// The seam between two halves of a transformer block in one pass over the stream (fw_residual_norm):
//     t  = y + bias;  [t = norm(t) * post_w];  x' = x + t * g1 + g0;  h = norm(x') [* w + b] [* (1 + scale) + shift]
// x' goes back to the stream, h leaves in bf16 or as MXFP4 rows for the linear that follows.  Run apart (fw_residual_add, then
// fw_layernorm_mod, then fw_mxfp4_quant_rows) the stream is read twice and h written and read once more.  Bound by HBM.
// One wave per row, the row in registers (VPL float4 a lane, C <= 256 VPL), statistics by wave shuffles in row_norm.h's pinned order:
// with LayerNorm, no post norm and 1024, 2048 or 5120 columns (one wave a row there too) the results are the bits of fw_residual_add followed
// by fw_layernorm_mod.
#include "mxfp4.h"
#include "row_norm.h"

namespace {

struct RnArgs {
    const void* x; int64_t ldx; void* xo; int64_t ldxo; int x_dtype;
    const void* y; int64_t ldy; int y_dtype;
    const float* bias; const float* g1; const float* g0; int post; const float* post_w;
    int norm; const float* w; const float* b; const float* scale; const float* shift; float eps;
    void* h; int64_t ldh; uint8_t* hs; int mx, slabs;
    int rows, C, rows_per_mod;
};

// MODE of a row access: 0 four at a time at any alignment, the row's last ones singly (any C), 1 four at a time, aligned (C % 4 == 0), 2 four at a time and C = 256 VPL, known at
// compile time (no lane is ever past the row: per-chunk predicates cost registers and branches).
// Chunk i of a row: lane l holds elements 4 l .. 4 l + 3 of its 256.  Everything below works on groups of G chunks, so that what a call has
// or has not (a type, a vector) is one uniform branch a group.
constexpr int rn_group(int vpl) { return vpl < 4 ? vpl : 4; }

// PAST: a stream larger than the memory-side cache (256 MB) is read and written past the caches -- what a row leaves there is gone before
// anybody comes back for it, and it costs the rows that follow.  32760 x 5120 in place, fp32 stream, bf16 y: bf16 h 397 us, 376 so; MXFP4 h
// 364 and 308.  A smaller stream finds part of itself there (8190 x 5120: 90 us, 95 past the caches).
template <int MODE, bool PAST, int G>
__device__ __forceinline__ void rn_load(const char* row, bool f32, int lane, int i0, int C, f32x4_t (&t)[G]) {
#pragma unroll
    for (int i = 0; i < G; ++i) t[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (f32) {
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const int c = (lane + 64 * (i0 + i)) * 4;
            if (MODE == 2 || (MODE == 1 && c < C)) t[i] = fw_load<PAST, f32x4_t>(row + lane * 16 + (i0 + i) * 1024);
            else if (MODE == 0 && c + 4 <= C) t[i] = *(const f32x4_odd_t*)(row + lane * 16 + (i0 + i) * 1024);
            else if (MODE == 0) {
#pragma unroll
                for (int j = 0; j < 3; ++j) if (c + j < C) t[i][j] = ((const float*)row)[c + j];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const int c = (lane + 64 * (i0 + i)) * 4;
            if (MODE == 2 || (MODE == 1 ? c < C : c + 4 <= C)) {
                u32x2_t r;
                if constexpr (MODE == 0) r = *(const u32x2_odd_t*)(row + lane * 8 + (i0 + i) * 512);
                else r = fw_load<PAST, u32x2_t>(row + lane * 8 + (i0 + i) * 512);
                t[i] = f32x4_t{__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xffff0000u), __uint_as_float(r[1] << 16), __uint_as_float(r[1] & 0xffff0000u)};
            } else if (MODE == 0) {
#pragma unroll
                for (int j = 0; j < 3; ++j) if (c + j < C) t[i][j] = bf16_bits_to_f32(((const uint16_t*)row)[c + j]);
            }
        }
    }
}
// 4 bf16 (two dwords) of chunk i
template <int MODE, bool PAST>
__device__ __forceinline__ void rn_store_bf16(char* row, int lane, int i, int C, u32x2_t r) {
    const int c = (lane + 64 * i) * 4;
    if (MODE == 2 || (MODE == 1 && c < C)) fw_store<PAST>(row + lane * 8 + i * 512, r);
    else if (MODE == 0 && c + 4 <= C) *(u32x2_odd_t*)(row + lane * 8 + i * 512) = r;
    else if (MODE == 0) {
#pragma unroll
        for (int j = 0; j < 3; ++j) if (c + j < C) ((uint16_t*)row)[c + j] = (uint16_t)(r[j >> 1] >> (16 * (j & 1)));
    }
}

// mean and 1 / sqrt(var + eps) (layer) or 0 and 1 / sqrt(mean square + eps) (rms) over the C live elements of the row
template <int VPL>
__device__ __forceinline__ void rn_stats(const f32x4_t (&v)[VPL], int lane, int C, bool layer, float eps, float& mean, float& rstd) {
    if (layer && C == VPL * 256) { ln_stats<VPL>(v, C, eps, mean, rstd); return; }
    const float inv_c = 1.0f / (float)C;
    mean = 0.f;
    if (layer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; ++i) s += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
        mean = wave_sum(s) * inv_c;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float d = v[i][j] - mean;
            if ((lane + 64 * i) * 4 + j < C) q = __builtin_fmaf(d, d, q);
        }
    rstd = rsqrtf(__builtin_fmaf(wave_sum(q), inv_c, eps));
}

// which parameter vectors a call has, and their place among the staged ones
enum { RN_BIAS, RN_POST_W, RN_W, RN_B, RN_G1, RN_G0, RN_SCALE, RN_SHIFT, RN_VECS };      // from RN_G1 on: one vector per run of rows

__device__ __forceinline__ const float* rn_ptr(const RnArgs& p, int k) {
    return k == RN_BIAS ? p.bias : k == RN_POST_W ? p.post_w : k == RN_W ? p.w : k == RN_B ? p.b : k == RN_G1 ? p.g1 : k == RN_G0 ? p.g0 : k == RN_SCALE ? p.scale : p.shift;
}

template <int VPL, int MODE, bool STAGE>
struct RnParams {
    const RnArgs& p;
    const f32x4_t* sm;                                    // [vector][VPL * 64] where staged
    int lane;
    int64_t mo;                                           // this row's modulation vectors
    // group i0 of vector k, if the call has it
    template <int G>
    __device__ __forceinline__ bool get(int k, int i0, f32x4_t (&t)[G]) const {
        const float* v = rn_ptr(p, k);
        if (!v) return false;
        if (STAGE) {
            int slot = 0;
#pragma unroll
            for (int j = 0; j < RN_VECS; ++j) slot += j < k && rn_ptr(p, j) ? 1 : 0;
#pragma unroll
            for (int i = 0; i < G; ++i) t[i] = sm[slot * VPL * 64 + 64 * (i0 + i) + lane];
        } else {
            rn_load<MODE, false, G>((const char*)(v + (k >= RN_G1 ? mo : 0)), true, lane, i0, MODE == 2 ? VPL * 256 : p.C, t);
        }
        return true;
    }
};

// x' of a group from x (v) and the finished y term (t): stored, and left in v as the norm reads it
template <int VPL, int MODE, bool STAGE, bool PAST, int G>
__device__ __forceinline__ void rn_update(const RnArgs& p, const RnParams<VPL, MODE, STAGE>& par, f32x4_t* v, f32x4_t (&t)[G], int i0, char* xo, bool xf) {
    const int lane = par.lane, C = MODE == 2 ? VPL * 256 : p.C;
    f32x4_t a[G], o[G];
    if (!par.get(RN_G1, i0, a)) {
#pragma unroll
        for (int i = 0; i < G; ++i) a[i] = f32x4_t{1.f, 1.f, 1.f, 1.f};
    }
    if (!par.get(RN_G0, i0, o)) {
#pragma unroll
        for (int i = 0; i < G; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[i][j] += fw_affine(t[i][j], a[i][j], o[i][j]);
            if (MODE != 2 && (lane + 64 * (i0 + i)) * 4 + j >= C) v[i][j] = 0.f;      // lanes past C carry g0 and bias: the statistics expect zeros
        }
    if (xf) {
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const int c = (lane + 64 * (i0 + i)) * 4;
            if (MODE == 2 || (MODE == 1 && c < C)) fw_store<PAST>(xo + lane * 16 + (i0 + i) * 1024, v[i]);
            else if (MODE == 0 && c + 4 <= C) *(f32x4_odd_t*)(xo + lane * 16 + (i0 + i) * 1024) = v[i];
            else if (MODE == 0) {
#pragma unroll
                for (int j = 0; j < 3; ++j) if (c + j < C) ((float*)xo)[c + j] = v[i][j];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const u32x2_t r = {pack_bf16x2(v[i][0], v[i][1]), pack_bf16x2(v[i][2], v[i][3])};
            rn_store_bf16<MODE, PAST>(xo, lane, i0 + i, C, r);
            v[i] = f32x4_t{__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xffff0000u), __uint_as_float(r[1] << 16), __uint_as_float(r[1] & 0xffff0000u)};
        }
    }
}

// a row's offset as the scalar it is: left to the compiler, the loop over rows keeps a 64-bit address per access in vector registers
__device__ __forceinline__ int64_t rn_uniform(int64_t off) {
    int lo = __builtin_amdgcn_readfirstlane((int)off), hi = __builtin_amdgcn_readfirstlane((int)(off >> 32));
    asm volatile("" : "+s"(lo), "+s"(hi));
    return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}

template <int VPL, int MODE, bool POST, bool STAGE, bool PAST>
__device__ __forceinline__ void rn_row(const RnArgs& p, const RnParams<VPL, MODE, STAGE>& par, int row) {
    constexpr int G = rn_group(VPL);
    const int C = MODE == 2 ? VPL * 256 : p.C, lane = par.lane;
    const bool xf = p.x_dtype == FW_DT_F32, yf = p.y_dtype == FW_DT_F32;
    const char* xr = (const char*)p.x + rn_uniform((int64_t)row * p.ldx * (xf ? 4 : 2));
    const char* yr = (const char*)p.y + rn_uniform((int64_t)row * p.ldy * (yf ? 4 : 2));
    char* xo = (char*)p.xo + rn_uniform((int64_t)row * p.ldxo * (xf ? 4 : 2));
    f32x4_t v[VPL];
#pragma unroll
    for (int i0 = 0; i0 < VPL; i0 += G) rn_load<MODE, PAST, G>(xr, xf, lane, i0, C, *(f32x4_t(*)[G])(v + i0));
    float mean, rstd;
    if (POST) {                                           // the statistics need all of y + bias
        f32x4_t t[VPL];
#pragma unroll
        for (int i0 = 0; i0 < VPL; i0 += G) rn_load<MODE, PAST, G>(yr, yf, lane, i0, C, *(f32x4_t(*)[G])(t + i0));
#pragma unroll
        for (int i0 = 0; i0 < VPL; i0 += G) {
            f32x4_t u[G];
            if (par.get(RN_BIAS, i0, u)) {
#pragma unroll
                for (int i = 0; i < G; ++i) t[i0 + i] += u[i];
            }
        }
        rn_stats<VPL>(t, lane, C, p.post == FW_RNORM_LAYER, p.eps, mean, rstd);
#pragma unroll
        for (int i0 = 0; i0 < VPL; i0 += G) {
            f32x4_t u[G], w[G];
#pragma unroll
            for (int i = 0; i < G; ++i) u[i] = (t[i0 + i] - mean) * rstd;
            if (par.get(RN_POST_W, i0, w)) {
#pragma unroll
                for (int i = 0; i < G; ++i) u[i] *= w[i];
            }
            rn_update<VPL, MODE, STAGE, PAST, G>(p, par, v + i0, u, i0, xo, xf);
        }
    } else if (p.y) {                                     // a group of y at a time, the next one on its way: the row of x is all that stays
        f32x4_t t[2][G];
        rn_load<MODE, PAST, G>(yr, yf, lane, 0, C, t[0]);
#pragma unroll
        for (int i0 = 0; i0 < VPL; i0 += G) {
            f32x4_t (&u)[G] = t[(i0 / G) & 1];
            if (i0 + G < VPL) rn_load<MODE, PAST, G>(yr, yf, lane, i0 + G, C, t[(i0 / G + 1) & 1]);
            f32x4_t b[G];
            if (par.get(RN_BIAS, i0, b)) {
#pragma unroll
                for (int i = 0; i < G; ++i) u[i] += b[i];
            }
            rn_update<VPL, MODE, STAGE, PAST, G>(p, par, v + i0, u, i0, xo, xf);
        }
    }
    rn_stats<VPL>(v, lane, C, p.norm == FW_RNORM_LAYER, p.eps, mean, rstd);
    char* hr = (char*)p.h + rn_uniform((int64_t)row * p.ldh * (p.mx ? 1 : 2));
    uint8_t* hs = p.hs + rn_uniform((int64_t)(row >> 5) * p.slabs * 256 + (row & 31) * 8);
#pragma unroll
    for (int i0 = 0; i0 < VPL; i0 += G) {
        // ln_finish's operations (row_norm.h) in ln_finish's order, a vector at a time
        f32x4_t o[G], u[G], w[G];
#pragma unroll
        for (int i = 0; i < G; ++i) o[i] = ln_finish(v[i0 + i], mean, rstd, false, o[i], false, o[i], false, o[i], false, o[i]);
        if (par.get(RN_W, i0, w)) {
            if (par.get(RN_B, i0, u)) {
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[i][j] = __builtin_fmaf(o[i][j], w[i][j], u[i][j]);
            } else {
#pragma unroll
                for (int i = 0; i < G; ++i) o[i] *= w[i];
            }
        }
        if (par.get(RN_SCALE, i0, w)) {
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][j] = __builtin_fmaf(o[i][j], w[i][j], o[i][j]);
        }
        if (par.get(RN_SHIFT, i0, u)) {
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) { float a = o[i][j]; asm volatile("" : "+v"(a)); o[i][j] = a + u[i][j]; }
        }
        u32x2_t r[G];
#pragma unroll
        for (int i = 0; i < G; ++i) r[i] = u32x2_t{pack_bf16x2(o[i][0], o[i][1]), pack_bf16x2(o[i][2], o[i][3])};
        if (p.mx) {
#pragma unroll
            for (int i = 0; i < G; ++i) {
                // 8 lanes hold a block of 32; both dwords carry two bf16
                if (MODE != 2) {
                    const int c = (lane + 64 * (i0 + i)) * 4;
#pragma unroll
                    for (int j = 0; j < 4; ++j) if (c + j >= C) r[i][j >> 1] &= (j & 1) ? 0x0000ffffu : 0xffff0000u;
                }
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 2; ++j) { top = max(top, r[i][j] & 0x7fff0000u); top = max(top, (r[i][j] << 16) & 0x7fff0000u); }
                top = mx_quad_max(top);
                top = max(top, (uint32_t)__builtin_amdgcn_ds_swizzle((int)top, 0x101F));                // lane ^ 4
                const uint32_t byte = mx_scale_byte(top);
                const float sc = mx_scale_f32(byte);
                uint32_t q = 0;
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, mx_pair(r[i][0]), sc, 0);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, mx_pair(r[i][1]), sc, 1);
                if (MODE == 2 || i0 + i < p.slabs) {
                    *(uint16_t*)(hr + lane * 2 + (i0 + i) * 128) = (uint16_t)q;
                    if ((lane & 7) == 0) hs[(i0 + i) * 256 + (lane >> 3)] = (uint8_t)byte;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < G; ++i) rn_store_bf16<MODE, PAST>(hr, lane, i0 + i, C, r[i]);
        }
    }
}

// Few rows: four of them a work-group, parameter vectors from the caches.
template <int VPL, int MODE, bool POST>
__global__ __launch_bounds__(256) void residual_norm_kernel(RnArgs p) {
    const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));      // uniform: addresses in scalar registers
    if (row >= p.rows) return;
    const RnParams<VPL, MODE, false> par{p, nullptr, (int)threadIdx.x & 63, (int64_t)(row / p.rows_per_mod) * p.C};
    rn_row<VPL, MODE, POST, false, false>(p, par, row);
}

// Many rows: a work-group stages the parameter vectors of one run of rows in LDS and walks that run with the run's other work-groups.
// Through the caches the vectors cost more than the row itself (bias, g1, scale, shift: 80 KiB per 60 KiB row at C = 5120): 32760 x 5120
// takes 923 us that way.  The work-groups walk side by side: with a contiguous block of rows for each, their equal strides of 2^18 bytes
// and more fall on the same memory channels (522 us).
template <int VPL, int MODE, bool POST, bool PAST>
__global__ __launch_bounds__(POST ? 256 : 512, POST ? 1 : 2) void residual_norm_staged_kernel(RnArgs p, int wgs_per_run) {
    extern __shared__ f32x4_t rn_smem[];
    constexpr int T = POST ? 256 : 512;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = blockIdx.x / wgs_per_run, w = blockIdx.x - g * wgs_per_run;
    int slot = 0;
#pragma unroll
    for (int k = 0; k < RN_VECS; ++k) {
        const float* src = rn_ptr(p, k);
        if (!src) continue;
        src += k >= RN_G1 ? (int64_t)g * p.C : 0;
        for (int i = threadIdx.x; i < VPL * 64; i += T) {
            f32x4_t t = {0.f, 0.f, 0.f, 0.f};
            if (MODE > 0 ? i * 4 < p.C : i * 4 + 4 <= p.C) t = MODE > 0 ? *(const f32x4_t*)(src + i * 4) : (f32x4_t)*(const f32x4_odd_t*)(src + i * 4);
            else if (MODE == 0) {
#pragma unroll
                for (int j = 0; j < 3; ++j) if (i * 4 + j < p.C) t[j] = src[i * 4 + j];
            }
            rn_smem[slot * VPL * 64 + i] = t;
        }
        ++slot;
    }
    __syncthreads();
    const unsigned last = (unsigned)min((int64_t)p.rows, (int64_t)(g + 1) * p.rows_per_mod);
    for (unsigned r = (unsigned)(g * p.rows_per_mod) + w * (T / 64) + wave; r < last; r += wgs_per_run * (T / 64)) {
        // the vectors stay in LDS: as invariants of this loop the compiler keeps them in 320 registers and spills
        int z = 0;
        asm volatile("" : "+s"(z));
        rn_row<VPL, MODE, POST, true, PAST>(p, RnParams<VPL, MODE, true>{p, rn_smem + z, lane, 0}, __builtin_amdgcn_readfirstlane((int)r));
    }
}

template <int VPL, int MODE, bool POST>
int rn_launch(const RnArgs& p, hipStream_t st) {
    // staged from 4096 rows on (a chip full of work-groups walks at least two rows a wave there; below, filling LDS costs more than it
    // saves), if the vectors leave room for it.  Rows past 5120 columns do not fit a wave's registers next to the addressing.
    // Unaligned rows: from 2049 columns on (20001 x 5117: 406 us, 333 staged; 9000 x 1283: 45, 50 staged).
    if constexpr (VPL <= 20 && (MODE > 0 || VPL == 20)) {
        int vecs = 0;
        for (const float* v : {p.bias, p.post_w, p.w, p.b, p.g1, p.g0, p.scale, p.shift}) vecs += v != nullptr;
        const int lds = vecs * VPL * 64 * 16;
        const int runs = (p.rows - 1) / p.rows_per_mod + 1;
        if (vecs && p.rows >= 4096 && runs <= 64 && lds <= 160 * 1024) {
            constexpr int waves = POST ? 4 : 8;
            const int per_cu = POST ? (lds <= 40 * 1024 ? 4 : lds <= 80 * 1024 ? 2 : 1) : (lds <= 80 * 1024 ? 2 : 1);
            const int wgs_per_run = min(256 * per_cu / runs, (p.rows_per_mod - 1) / waves + 1);
            const bool past = MODE == 2 && (int64_t)p.rows * p.C * (p.x_dtype == FW_DT_F32 ? 4 : 2) > FW_CACHE_BYTES;
            const auto f = past ? residual_norm_staged_kernel<VPL, MODE, POST, MODE == 2> : residual_norm_staged_kernel<VPL, MODE, POST, false>;
            if (lds > 64 * 1024) {
                const int rc = (int)hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
                if (rc) return rc;
            }
            hipLaunchKernelGGL(f, dim3((unsigned)(runs * wgs_per_run)), dim3(waves * 64), lds, st, p, wgs_per_run);
            return (int)hipGetLastError();
        }
    }
    hipLaunchKernelGGL((residual_norm_kernel<VPL, MODE, POST>), dim3((unsigned)((p.rows - 1) / 4 + 1)), dim3(256), 0, st, p);
    return (int)hipGetLastError();
}

template <int VPL>
int rn_dispatch(const RnArgs& p, bool vec, hipStream_t st) {
    if (vec && p.C == VPL * 256) return p.post ? rn_launch<VPL, 2, true>(p, st) : rn_launch<VPL, 2, false>(p, st);
    if (vec) return p.post ? rn_launch<VPL, 1, true>(p, st) : rn_launch<VPL, 1, false>(p, st);
    return p.post ? rn_launch<VPL, 0, true>(p, st) : rn_launch<VPL, 0, false>(p, st);
}

}  // namespace

extern "C" int fw_residual_norm(const void* x, int64_t ldx, void* x_out, int64_t ldxo, int x_dtype, const void* y, int64_t ldy, int y_dtype,
                                const float* bias, const float* g1, const float* g0, int post, const float* post_w,
                                int norm, const float* w, const float* b, const float* scale, const float* shift, float eps,
                                void* h, int64_t ldh, int h_dtype, uint8_t* h_scale, int rows, int C, int rows_per_mod, void* stream) {
    if (rows <= 0) return 0;
    const int xe = x_dtype == FW_DT_F32 ? 4 : 2, ye = y_dtype == FW_DT_F32 ? 4 : 2;
    if (!x || !h || C <= 0 || C > 8192 || ldx < C || (x_dtype != FW_DT_F32 && x_dtype != FW_DT_BF16) || (((uintptr_t)x) & (xe - 1)) || rows_per_mod <= 0) {
        fw_set_error("fw_residual_norm: f32 / bf16 x, 0 < C <= 8192, ldx >= C, rows_per_mod > 0 required"); return FW_E_BADARG; }
    if (y && ((y_dtype != FW_DT_F32 && y_dtype != FW_DT_BF16) || ldy < C || (((uintptr_t)y) & (ye - 1)) || !x_out || ldxo < C || (((uintptr_t)x_out) & (xe - 1)))) {
        fw_set_error("fw_residual_norm: f32 / bf16 y with ldy >= C and an x_out with ldxo >= C required"); return FW_E_BADARG; }
    if (!y && (bias || g1 || g0 || post || post_w)) { fw_set_error("fw_residual_norm: bias / g1 / g0 / post need y"); return FW_E_BADARG; }
    if ((norm != FW_RNORM_LAYER && norm != FW_RNORM_RMS) || (post != FW_RNORM_NONE && post != FW_RNORM_LAYER && post != FW_RNORM_RMS) || (post_w && !post) || (b && !w)) {
        fw_set_error("fw_residual_norm: norm is layer or rms; post none, layer or rms; post_w needs post, b needs w"); return FW_E_BADARG; }
    const int slabs = mx_slabs(C);
    if (h_dtype == FW_DT_MXFP4 ? (!h_scale || ldh < (int64_t)slabs * 128 || (ldh % 16) || (((uintptr_t)h) & 15) || (((uintptr_t)h_scale) & 3))
                               : (h_dtype != FW_DT_BF16 || ldh < C || (((uintptr_t)h) & 1))) {
        fw_set_error("fw_residual_norm: bf16 h with ldh >= C, or MXFP4 h with h_scale, 16-byte aligned rows and ldh >= roundup(C, 256) / 2"); return FW_E_BADARG; }
    const uintptr_t pv = ((uintptr_t)bias) | ((uintptr_t)g1) | ((uintptr_t)g0) | ((uintptr_t)post_w) | ((uintptr_t)w) | ((uintptr_t)b) | ((uintptr_t)scale) | ((uintptr_t)shift);
    if (pv & 3) { fw_set_error("fw_residual_norm: misaligned parameter vector"); return FW_E_BADARG; }
    // A row is whole in its wave's registers before its outputs are stored, so an output may be an input -- the same rows in the same type --
    // but shares no byte with any other operand, which other waves still read.
    {
        const int64_t runs = (rows - 1) / rows_per_mod + 1;
        const bool mx = h_dtype == FW_DT_MXFP4;
        const FwSpan xs(x, ldx * xe, (int64_t)C * xe, rows), ys(y, ldy * ye, (int64_t)C * ye, rows), xos(y ? x_out : nullptr, ldxo * xe, (int64_t)C * xe, rows);
        const FwSpan hs(h, mx ? ldh : ldh * 2, mx ? (int64_t)slabs * 128 : (int64_t)C * 2, rows), ss(mx ? h_scale : nullptr, ((int64_t)rows + 31) / 32 * slabs * 256);
        auto clash = [](const FwSpan& in, bool same_type, const FwSpan& out) { return fw_overlap(in, out) && !(same_type && in.same(out)); };
        bool bad = clash(xs, true, xos) || clash(ys, x_dtype == y_dtype, xos) || clash(xs, x_dtype == h_dtype, hs) || clash(ys, y_dtype == h_dtype, hs) ||
                   fw_overlap(xos, hs) || fw_overlap(xs, ss) || fw_overlap(ys, ss) || fw_overlap(xos, ss) || fw_overlap(hs, ss);
        const float* vec[] = {bias, post_w, w, b, g1, g0, scale, shift};
        for (int i = 0; i < 8; ++i) {
            const FwSpan v(vec[i], (i < 4 ? 1 : runs) * C * 4);
            bad = bad || fw_overlap(v, xos) || fw_overlap(v, hs) || fw_overlap(v, ss);
        }
        if (bad) { fw_set_error("fw_residual_norm: an output overlaps another operand (it may be x or y: the same rows in the same type)"); return FW_E_BADARG; }
    }
    RnArgs p;
    p.x = x; p.ldx = ldx; p.xo = x_out; p.ldxo = ldxo; p.x_dtype = x_dtype; p.y = y; p.ldy = ldy; p.y_dtype = y_dtype;
    p.bias = bias; p.g1 = g1; p.g0 = g0; p.post = post; p.post_w = post_w; p.norm = norm; p.w = w; p.b = b; p.scale = scale; p.shift = shift;
    p.eps = eps; p.h = h; p.ldh = ldh; p.hs = h_scale; p.mx = h_dtype == FW_DT_MXFP4; p.slabs = slabs; p.rows = rows; p.C = C;
    p.rows_per_mod = min(rows_per_mod, rows);            // one vector for all: any value from rows on, the largest int too; sums with it stay in 32 bits
    // 4 values at a time: every row of every operand starts on the access size (16 bytes in fp32, 8 in bf16)
    auto rows_ok = [](const void* q, int64_t ld, int e) { return (((uintptr_t)q) & (4 * e - 1)) == 0 && (ld % 4) == 0; };
    const bool vec = (C % 4) == 0 && (pv & 15) == 0 && rows_ok(x, ldx, xe) && (!y || (rows_ok(y, ldy, ye) && rows_ok(x_out, ldxo, xe))) && (p.mx || rows_ok(h, ldh, 2));
    hipStream_t st = (hipStream_t)stream;
    const int n = (C + 255) / 256;
    if (n <= 1) return rn_dispatch<1>(p, vec, st);
    if (n <= 2) return rn_dispatch<2>(p, vec, st);
    if (n <= 4) return rn_dispatch<4>(p, vec, st);
    if (n <= 8) return rn_dispatch<8>(p, vec, st);
    if (n <= 20) return rn_dispatch<20>(p, vec, st);
    return rn_dispatch<32>(p, vec, st);
}
