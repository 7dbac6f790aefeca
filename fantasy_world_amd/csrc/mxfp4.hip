// MXFP4 rows: quantiser and dequantiser (encoding and storage: mxfp4.h).  Both are bound by HBM: 2 + 17/32 bytes a value.
// 32760 x 13824 bf16: 174 us = 6.6 TB/s there and 161 us = 7.1 TB/s back; 203 and 210 with the wide side passing through the caches.
// A work-group owns one scale tile -- 32 rows x 256 values -- so its 256 scale bytes leave as one contiguous write and nobody else touches
// them; a half-wave reads 512 contiguous bytes of a row (8 values a lane), four rows one after another so that four loads are in flight.
#include "mxfp4.h"

namespace {

template <bool F32, bool VEC, bool PAST>
__device__ __forceinline__ void load8(const void* x, int64_t off, int k, int K, float* f, u32x4_t& raw) {
    if (F32) {
        if (VEC) {
            const f32x4_t a = fw_load<PAST, f32x4_t>((const float*)x + off), b = fw_load<PAST, f32x4_t>((const float*)x + off + 4);
            f[0] = a[0]; f[1] = a[1]; f[2] = a[2]; f[3] = a[3]; f[4] = b[0]; f[5] = b[1]; f[6] = b[2]; f[7] = b[3];
        } else if (k + 8 <= K) {
            const f32x4_t a = *(const f32x4_odd_t*)((const float*)x + off), b = *(const f32x4_odd_t*)((const float*)x + off + 4);
            f[0] = a[0]; f[1] = a[1]; f[2] = a[2]; f[3] = a[3]; f[4] = b[0]; f[5] = b[1]; f[6] = b[2]; f[7] = b[3];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = k + j < K ? ((const float*)x)[off + j] : 0.f;
        }
    } else if (VEC) {
        raw = fw_load<PAST, u32x4_t>((const uint16_t*)x + off);
    } else if (k + 8 <= K) {
        raw = *(const u32x4_odd_t*)((const uint16_t*)x + off);
    } else {
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = k + j < K ? ((const uint16_t*)x)[off + j] : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[j] = h[2 * j] | (h[2 * j + 1] << 16);
    }
}

template <bool F32, bool VEC, bool PAST>
__global__ __launch_bounds__(256) void mxfp4_quant_rows_kernel(const void* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq,
                                                               uint8_t* __restrict__ s, int M, int K, int slabs) {
    __shared__ uint8_t tile[32 * 8];
    const int rb = blockIdx.x / slabs, ks = blockIdx.x % slabs;
    const int l = threadIdx.x & 31, hw = threadIdx.x >> 5;             // lane of the half-wave, half-wave 0..7
    const int k = ks * MX_SLAB + l * 8;
    float f[4][8];
    u32x4_t raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = rb * 32 + i * 8 + hw;
        raw[i] = u32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
        if (row < M && k < K) load8<F32, VEC, PAST>(x, (int64_t)row * ldx + k, k, K, f[i], raw[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int rl = i * 8 + hw, row = rb * 32 + rl;
        uint32_t top = 0;
        if (F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[i][j]) & 0x7fffffffu);
        } else {
            top = mx_top8_bf16(raw[i]);
        }
        const uint32_t byte = mx_scale_byte(mx_quad_max(top));
        const float scale = mx_scale_f32(byte);
        const uint32_t codes = F32 ? mx_pack8_f32(f[i], scale) : mx_pack8_bf16(raw[i], scale);
        if (row < M) *(uint32_t*)(q + (int64_t)row * ldq + (k >> 1)) = codes;
        if ((l & 3) == 0) tile[rl * 8 + (l >> 2)] = (uint8_t)byte;
    }
    __syncthreads();
    if (threadIdx.x < 64) ((uint32_t*)(s + (int64_t)blockIdx.x * 256))[threadIdx.x] = ((const uint32_t*)tile)[threadIdx.x];
}

template <bool F32, bool VEC, bool PAST>
__global__ __launch_bounds__(256) void mxfp4_dequant_rows_kernel(const uint8_t* __restrict__ q, int64_t ldq, const uint8_t* __restrict__ s,
                                                                 void* __restrict__ y, int64_t ldy, int M, int K, int slabs) {
    const int rb = blockIdx.x / slabs, ks = blockIdx.x % slabs;
    const int l = threadIdx.x & 31, hw = threadIdx.x >> 5;
    const int k = ks * MX_SLAB + l * 8;
    uint32_t codes[4], byte[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int rl = i * 8 + hw, row = rb * 32 + rl;
        codes[i] = row < M && k < K ? *(const uint32_t*)(q + (int64_t)row * ldq + (k >> 1)) : 0u;
        byte[i] = s[(int64_t)blockIdx.x * 256 + rl * 8 + (l >> 2)];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = rb * 32 + i * 8 + hw;
        if (row >= M || k >= K) continue;
        // level * 2^(byte - 127): exact in both output types (the smallest, 2^-128, is a subnormal of each)
        typedef __attribute__((ext_vector_type(2))) float f32x2_t;
        const f32x2_t p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 1),
                              __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 3)};
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            f[j] = byte[i] == 255u ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(p[j >> 1][j & 1], (int)byte[i] - 127);
        const int64_t off = (int64_t)row * ldy + k;
        if (F32) {
            if (VEC) {
                fw_store<PAST>((float*)y + off, f32x4_t{f[0], f[1], f[2], f[3]});
                fw_store<PAST>((float*)y + off + 4, f32x4_t{f[4], f[5], f[6], f[7]});
            } else if (k + 8 <= K) {
                *(f32x4_odd_t*)((float*)y + off) = f32x4_t{f[0], f[1], f[2], f[3]};
                *(f32x4_odd_t*)((float*)y + off + 4) = f32x4_t{f[4], f[5], f[6], f[7]};
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) if (k + j < K) ((float*)y)[off + j] = f[j];
            }
        } else {
            if (VEC) {
                fw_store<PAST>((uint16_t*)y + off, u32x4_t{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])});
            } else if (k + 8 <= K) {
                *(u32x4_odd_t*)((uint16_t*)y + off) = u32x4_t{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) if (k + j < K) ((uint16_t*)y)[off + j] = f32_to_bf16_bits(f[j]);
            }
        }
    }
}

}  // namespace

extern "C" int fw_mxfp4_quant_rows(const void* x, int64_t ldx, int x_dtype, uint8_t* q, int64_t ldq, uint8_t* s, int M, int K, void* stream) {
    if (M <= 0) return 0;
    const int slabs = mx_slabs(K);
    if (!x || !q || !s || K <= 0 || K > MX_MAX || ldx < K || ldq < (int64_t)slabs * 128 || (ldq % 16) || (((uintptr_t)q) & 15) || (((uintptr_t)s) & 3) ||
        (x_dtype != FW_DT_BF16 && x_dtype != FW_DT_F32) || (((uintptr_t)x) & (x_dtype == FW_DT_F32 ? 3 : 1))) {
        fw_set_error("fw_mxfp4_quant_rows: bf16 / f32 x with ldx >= K, 0 < K < 2^31 - 256, q 16-byte aligned with ldq % 16 == 0 and ldq >= roundup(K, 256) / 2, s 4-byte aligned required");
        return FW_E_BADARG; }
    const int64_t nwg = ((int64_t)M + 31) / 32 * slabs;
    if (nwg > 0x7fffffff) { fw_set_error("fw_mxfp4_quant_rows: grid too large"); return FW_E_BADARG; }
    const FwSpan xs(x, ldx * (x_dtype == FW_DT_F32 ? 4 : 2), (int64_t)K * (x_dtype == FW_DT_F32 ? 4 : 2), M), qs(q, ldq, (int64_t)slabs * 128, M);
    const FwSpan ss(s, ((int64_t)M + 31) / 32 * slabs * 256);
    if (fw_overlap(xs, qs) || fw_overlap(xs, ss) || fw_overlap(qs, ss)) { fw_set_error("fw_mxfp4_quant_rows: x, q and s must not overlap"); return FW_E_BADARG; }
    const bool vec = (K % 8) == 0 && ((((uintptr_t)x) & 15) == 0) && (ldx % (x_dtype == FW_DT_F32 ? 4 : 8)) == 0;
    const bool past = (int64_t)M * K * (x_dtype == FW_DT_F32 ? 4 : 2) > FW_CACHE_BYTES;
    const dim3 g((unsigned)nwg), b(256);
    hipStream_t st = (hipStream_t)stream;
    if (x_dtype == FW_DT_F32) {
        if (vec && past) hipLaunchKernelGGL((mxfp4_quant_rows_kernel<true, true, true>), g, b, 0, st, x, ldx, q, ldq, s, M, K, slabs);
        else if (vec) hipLaunchKernelGGL((mxfp4_quant_rows_kernel<true, true, false>), g, b, 0, st, x, ldx, q, ldq, s, M, K, slabs);
        else hipLaunchKernelGGL((mxfp4_quant_rows_kernel<true, false, false>), g, b, 0, st, x, ldx, q, ldq, s, M, K, slabs);
    } else {
        if (vec && past) hipLaunchKernelGGL((mxfp4_quant_rows_kernel<false, true, true>), g, b, 0, st, x, ldx, q, ldq, s, M, K, slabs);
        else if (vec) hipLaunchKernelGGL((mxfp4_quant_rows_kernel<false, true, false>), g, b, 0, st, x, ldx, q, ldq, s, M, K, slabs);
        else hipLaunchKernelGGL((mxfp4_quant_rows_kernel<false, false, false>), g, b, 0, st, x, ldx, q, ldq, s, M, K, slabs);
    }
    return (int)hipGetLastError();
}

extern "C" int fw_mxfp4_dequant_rows(const uint8_t* q, int64_t ldq, const uint8_t* s, void* y, int64_t ldy, int y_dtype, int M, int K, void* stream) {
    if (M <= 0) return 0;
    const int slabs = mx_slabs(K);
    if (!q || !s || !y || K <= 0 || K > MX_MAX || ldy < K || ldq < (int64_t)slabs * 128 || (ldq % 16) || (((uintptr_t)q) & 15) ||
        (y_dtype != FW_DT_BF16 && y_dtype != FW_DT_F32) || (((uintptr_t)y) & (y_dtype == FW_DT_F32 ? 3 : 1))) {
        fw_set_error("fw_mxfp4_dequant_rows: bf16 / f32 y with ldy >= K, 0 < K < 2^31 - 256, q 16-byte aligned with ldq % 16 == 0 and ldq >= roundup(K, 256) / 2 required");
        return FW_E_BADARG; }
    const int64_t nwg = ((int64_t)M + 31) / 32 * slabs;
    if (nwg > 0x7fffffff) { fw_set_error("fw_mxfp4_dequant_rows: grid too large"); return FW_E_BADARG; }
    const FwSpan ys(y, ldy * (y_dtype == FW_DT_F32 ? 4 : 2), (int64_t)K * (y_dtype == FW_DT_F32 ? 4 : 2), M);
    if (fw_overlap(ys, FwSpan(q, ldq, (int64_t)slabs * 128, M)) || fw_overlap(ys, FwSpan(s, ((int64_t)M + 31) / 32 * slabs * 256))) {
        fw_set_error("fw_mxfp4_dequant_rows: y must not overlap q or s"); return FW_E_BADARG; }
    const bool vec = (K % 8) == 0 && ((((uintptr_t)y) & 15) == 0) && (ldy % (y_dtype == FW_DT_F32 ? 4 : 8)) == 0;
    const bool past = (int64_t)M * K * (y_dtype == FW_DT_F32 ? 4 : 2) > FW_CACHE_BYTES;
    const dim3 g((unsigned)nwg), b(256);
    hipStream_t st = (hipStream_t)stream;
    if (y_dtype == FW_DT_F32) {
        if (vec && past) hipLaunchKernelGGL((mxfp4_dequant_rows_kernel<true, true, true>), g, b, 0, st, q, ldq, s, y, ldy, M, K, slabs);
        else if (vec) hipLaunchKernelGGL((mxfp4_dequant_rows_kernel<true, true, false>), g, b, 0, st, q, ldq, s, y, ldy, M, K, slabs);
        else hipLaunchKernelGGL((mxfp4_dequant_rows_kernel<true, false, false>), g, b, 0, st, q, ldq, s, y, ldy, M, K, slabs);
    } else {
        if (vec && past) hipLaunchKernelGGL((mxfp4_dequant_rows_kernel<false, true, true>), g, b, 0, st, q, ldq, s, y, ldy, M, K, slabs);
        else if (vec) hipLaunchKernelGGL((mxfp4_dequant_rows_kernel<false, true, false>), g, b, 0, st, q, ldq, s, y, ldy, M, K, slabs);
        else hipLaunchKernelGGL((mxfp4_dequant_rows_kernel<false, false, false>), g, b, 0, st, q, ldq, s, y, ldy, M, K, slabs);
    }
    return (int)hipGetLastError();
}
