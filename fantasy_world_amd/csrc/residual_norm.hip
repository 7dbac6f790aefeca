// The seam between two halves of a transformer block in one pass over the stream (fw_residual_norm):
//     t  = y + bias;  [t = norm(t) * post_w];  x' = x + t * g1 + g0;  h = norm(x') [* w + b] [* (1 + scale) + shift]
// x' goes back to the stream, h leaves in bf16 or as MXFP4 rows for the linear that follows.  Run apart (fw_residual_add, then
// fw_layernorm_mod, then fw_mxfp4_quant_rows) the stream is read twice and h written and read once more.  Bound by HBM.
// One wave per row, the row in registers (VPL float4 a lane, C <= 256 VPL), statistics by wave shuffles in row_norm.h's pinned order:
// with LayerNorm, no post norm and C = 256 VPL the results are the bits of fw_residual_add followed by fw_layernorm_mod.
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

// 4 consecutive values at element c of a row; VEC: c + 3 < C and aligned.  Elements past C are 0.
template <bool VEC>
__device__ __forceinline__ f32x4_t rn_load(const void* p, int64_t off, int c, int C, bool f32) {
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    if (VEC) {
        if (c >= C) return v;
        if (f32) return *(const f32x4_t*)((const float*)p + off + c);
        const u32x2_t r = *(const u32x2_t*)((const uint16_t*)p + off + c);
        return f32x4_t{__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xffff0000u), __uint_as_float(r[1] << 16), __uint_as_float(r[1] & 0xffff0000u)};
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < C) v[j] = f32 ? ((const float*)p)[off + c + j] : bf16_bits_to_f32(((const uint16_t*)p)[off + c + j]);
    return v;
}
template <bool VEC>
__device__ __forceinline__ f32x4_t rn_vec(const float* p, int c, int C) { return rn_load<VEC>(p, 0, c, C, true); }

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

template <int VPL, bool VEC>
__global__ __launch_bounds__(256) void residual_norm_kernel(RnArgs p) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.rows) return;
    const int C = p.C;
    const int64_t mo = (int64_t)(row / p.rows_per_mod) * C;            // this row's modulation vectors
    f32x4_t v[VPL];
    const bool xf = p.x_dtype == FW_DT_F32;
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = rn_load<VEC>(p.x, (int64_t)row * p.ldx, (lane + 64 * i) * 4, C, xf);
    float mean, rstd;
    if (p.y) {
        f32x4_t t[VPL];
        const bool yf = p.y_dtype == FW_DT_F32;
#pragma unroll
        for (int i = 0; i < VPL; ++i) t[i] = rn_load<VEC>(p.y, (int64_t)row * p.ldy, (lane + 64 * i) * 4, C, yf);
        if (p.bias) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) t[i] += rn_vec<VEC>(p.bias, (lane + 64 * i) * 4, C);
        }
        if (p.post) {
            rn_stats<VPL>(t, lane, C, p.post == FW_RNORM_LAYER, p.eps, mean, rstd);
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                t[i] = (t[i] - mean) * rstd;
                if (p.post_w) t[i] *= rn_vec<VEC>(p.post_w, (lane + 64 * i) * 4, C);
            }
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int c = (lane + 64 * i) * 4;
            const f32x4_t one = {1.f, 1.f, 1.f, 1.f}, zero = {0.f, 0.f, 0.f, 0.f};
            const f32x4_t a = p.g1 ? rn_vec<VEC>(p.g1 + mo, c, C) : one, o = p.g0 ? rn_vec<VEC>(p.g0 + mo, c, C) : zero;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] += fw_affine(t[i][j], a[j], o[j]);
            if (c < C) {
                if (xf) {
                    float* d = (float*)p.xo + (int64_t)row * p.ldxo + c;
                    if (VEC) *(f32x4_t*)d = v[i];
                    else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) if (c + j < C) d[j] = v[i][j];
                    }
                } else {
                    uint16_t* d = (uint16_t*)p.xo + (int64_t)row * p.ldxo + c;
                    const u32x2_t r = {pack_bf16x2(v[i][0], v[i][1]), pack_bf16x2(v[i][2], v[i][3])};
                    if (VEC) *(u32x2_t*)d = r;
                    else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) if (c + j < C) d[j] = (uint16_t)(r[j >> 1] >> (16 * (j & 1)));
                    }
                    // the norm reads the stream as it is stored
                    v[i] = f32x4_t{__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xffff0000u), __uint_as_float(r[1] << 16), __uint_as_float(r[1] & 0xffff0000u)};
                }
            }
            if (!VEC || c >= C) {                       // lanes past C carry g0 and bias: back to the zeros that the statistics expect
#pragma unroll
                for (int j = 0; j < 4; ++j) if (c + j >= C) v[i][j] = 0.f;
            }
        }
    }
    rn_stats<VPL>(v, lane, C, p.norm == FW_RNORM_LAYER, p.eps, mean, rstd);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int c = (lane + 64 * i) * 4;
        const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
        const f32x4_t o = ln_finish(v[i], mean, rstd, p.w != nullptr, p.w ? rn_vec<VEC>(p.w, c, C) : zero, p.b != nullptr, p.b ? rn_vec<VEC>(p.b, c, C) : zero,
                                    p.scale != nullptr, p.scale ? rn_vec<VEC>(p.scale + mo, c, C) : zero,
                                    p.shift != nullptr, p.shift ? rn_vec<VEC>(p.shift + mo, c, C) : zero);
        u32x2_t r = {pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
        if (p.mx) {
            // 8 lanes hold a block of 32; both dwords carry two bf16
            if (c >= C) r = u32x2_t{0, 0};
            else if (!VEC) {
#pragma unroll
                for (int j = 0; j < 4; ++j) if (c + j >= C) r[j >> 1] &= (j & 1) ? 0x0000ffffu : 0xffff0000u;
            }
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) { top = max(top, r[j] & 0x7fff0000u); top = max(top, (r[j] << 16) & 0x7fff0000u); }
            top = mx_quad_max(top);
            top = max(top, (uint32_t)__builtin_amdgcn_ds_swizzle((int)top, 0x101F));                // lane ^ 4
            const uint32_t byte = mx_scale_byte(top);
            const float sc = mx_scale_f32(byte);
            uint32_t q = 0;
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, mx_pair(r[0]), sc, 0);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, mx_pair(r[1]), sc, 1);
            if (i < p.slabs) {
                *(uint16_t*)((uint8_t*)p.h + (int64_t)row * p.ldh + (c >> 1)) = (uint16_t)q;
                if ((lane & 7) == 0) p.hs[((int64_t)(row >> 5) * p.slabs + i) * 256 + (row & 31) * 8 + (lane >> 3)] = (uint8_t)byte;
            }
        } else if (c < C) {
            uint16_t* d = (uint16_t*)p.h + (int64_t)row * p.ldh + c;
            if (VEC) *(u32x2_t*)d = r;
            else {
#pragma unroll
                for (int j = 0; j < 4; ++j) if (c + j < C) d[j] = (uint16_t)(r[j >> 1] >> (16 * (j & 1)));
            }
        }
    }
}

template <int VPL>
void rn_launch(const RnArgs& p, bool vec, hipStream_t st) {
    const dim3 g((unsigned)((p.rows + 3) / 4)), b(256);
    if (vec) hipLaunchKernelGGL((residual_norm_kernel<VPL, true>), g, b, 0, st, p);
    else hipLaunchKernelGGL((residual_norm_kernel<VPL, false>), g, b, 0, st, p);
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
    RnArgs p;
    p.x = x; p.ldx = ldx; p.xo = x_out; p.ldxo = ldxo; p.x_dtype = x_dtype; p.y = y; p.ldy = ldy; p.y_dtype = y_dtype;
    p.bias = bias; p.g1 = g1; p.g0 = g0; p.post = post; p.post_w = post_w; p.norm = norm; p.w = w; p.b = b; p.scale = scale; p.shift = shift;
    p.eps = eps; p.h = h; p.ldh = ldh; p.hs = h_scale; p.mx = h_dtype == FW_DT_MXFP4; p.slabs = slabs; p.rows = rows; p.C = C; p.rows_per_mod = rows_per_mod;
    // 4 values at a time: every row of every operand starts on the access size (16 bytes in fp32, 8 in bf16)
    auto rows_ok = [](const void* q, int64_t ld, int e) { return (((uintptr_t)q) & (4 * e - 1)) == 0 && (ld % 4) == 0; };
    const bool vec = (C % 4) == 0 && (pv & 15) == 0 && rows_ok(x, ldx, xe) && (!y || (rows_ok(y, ldy, ye) && rows_ok(x_out, ldxo, xe))) && (p.mx || rows_ok(h, ldh, 2));
    hipStream_t st = (hipStream_t)stream;
    const int n = (C + 255) / 256;
    if (n <= 1) rn_launch<1>(p, vec, st);
    else if (n <= 2) rn_launch<2>(p, vec, st);
    else if (n <= 4) rn_launch<4>(p, vec, st);
    else if (n <= 8) rn_launch<8>(p, vec, st);
    else if (n <= 20) rn_launch<20>(p, vec, st);
    else rn_launch<32>(p, vec, st);
    return (int)hipGetLastError();
}
