// MXFP4 x MXFP4 MFMA GEMM:  C = epi(A[M,K] W[N,K]^T), both operands e2m1 codes with one E8M0 scale per 32 values along K (mxfp4.h).
//
// v_mfma_scale_f32_32x32x64_f8f6f4 with both format selectors at fp4 multiplies 64 values of K per instruction in the time an fp8 MFMA
// takes for 32 and applies both block scales itself; products of e2m1 values and their sums inside an instruction are exact in fp32.
// Lane l supplies row l & 31 of an operand and one 16-byte chunk = one block of 32 values.  The four k-steps of a 256-value slab are
// assigned to the chunks so that lane (r, h = l >> 5) takes chunks 4h .. 4h + 3 in order: its four scale bytes are then one aligned
// dword of the scale tile, selected by the instruction's byte selector, and never pass through LDS.  Any assignment of blocks to k-steps
// is right as long as both operands use the same one.
// LDS image: a row of a slab is 128 bytes (8 chunks); chunk c of row r is stored at c ^ ((r >> 1) & 7), applied to the source address of
// the LDS-DMA and again on the read, which makes the 16-byte fragment reads conflict-free.
#include "mxfp4.h"
#include <type_traits>

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;

struct MxArgs {
    const uint8_t* A; int64_t lda; const uint8_t* sa;
    const uint8_t* W; int64_t ldw; const uint8_t* sw;
    void* C; int64_t ldc; int out_dtype; uint8_t* cs;
    int M, N, slabs;
    const float* bias; int act; const float* g1; const float* g0;
    const void* res; int64_t ldr; int res_dtype;
    int tiles_m, tiles_n, vec, cslabs;
};

// the upper half of the 8-register operand type is not read for fp4
#define FWX_MFMA(A, B, C, J, SA, SB) __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4( \
    i32x8_t{(A)[0], (A)[1], (A)[2], (A)[3], 0, 0, 0, 0}, i32x8_t{(B)[0], (B)[1], (B)[2], (B)[3], 0, 0, 0, 0}, C, 4, 4, J, SA, J, SB)
#define FWX_BLDS16(rs, voff, soff, ldsptr) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, FW_LDS_PTR(ldsptr), 16, voff, soff, 0, 0)

// descriptor over the rows from `base` on: an access past `bytes` reads zeros (a tile that lies in a quantised row's padding has no rows at all)
__device__ __forceinline__ auto mx_rsrc(const uint8_t* base, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)(unsigned)(bytes > 0xffffffffLL ? 0xffffffffLL : bytes < 0 ? 0 : bytes), 0x00020000);
}

// tile of this work-group: XCD-contiguous tile ranges (bijective), groups of GROUP row tiles walked column by column inside them
__device__ __forceinline__ void mx_tile(const MxArgs& p, int& tm, int& tn) {
    const int nwg = p.tiles_m * p.tiles_n;
    const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, q = nwg >> 3, r = nwg & 7;
    const int wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + slot;
    const int GROUP = p.tiles_n >= 20 ? 4 : 8;
    const int per_group = GROUP * p.tiles_n, gid = wg / per_group, first_m = gid * GROUP;
    const int gsz = min(p.tiles_m - first_m, GROUP), in_g = wg - gid * per_group;
    tm = first_m + in_g % gsz;
    tn = in_g / gsz;
}

// One 64 x 64 quadrant of a wave: accumulators [2][2] -> LDS (16 KiB of this wave's own) -> rows -> bias, activation, per-column affine,
// residual, store.  A lane owns 8 consecutive columns of one row at a time, 8 rows per step: 16-byte stores in bf16, and with MXFP4 output
// a block of 32 columns is the 4 lanes of a quad.
template <int ACT>
__device__ __forceinline__ void mx_epilogue64(const MxArgs& p, char* reg, const f32x16_t& a00, const f32x16_t& a01, const f32x16_t& a10,
                                              const f32x16_t& a11, int lane, int m0, int n0) {
    const int fi = lane & 31, hi = lane >> 5;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int row_l = (r & 3) + 8 * (r >> 2) + 4 * hi;
        *(float*)(reg + row_l * 256 + fi * 4) = a00[r];
        *(float*)(reg + row_l * 256 + (32 + fi) * 4) = a01[r];
        *(float*)(reg + (32 + row_l) * 256 + fi * 4) = a10[r];
        *(float*)(reg + (32 + row_l) * 256 + (32 + fi) * 4) = a11[r];
    }
    const int c8 = (lane & 7) * 8, rl = lane >> 3;
    const int col = n0 + c8;
    float bias[8], g1[8], g0[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bool in = col + j < p.N;
        bias[j] = p.bias && in ? p.bias[col + j] : 0.f;
        g1[j] = p.g1 && in ? p.g1[col + j] : 1.f;
        g0[j] = p.g0 && in ? p.g0[col + j] : 0.f;
    }
#pragma unroll 2
    for (int it = 0; it < 8; ++it) {
        const int row_l = it * 8 + rl, row = m0 + row_l;
        const f32x4_t lo = *(const f32x4_t*)(reg + row_l * 256 + c8 * 4), up = *(const f32x4_t*)(reg + row_l * 256 + c8 * 4 + 16);
        float v[8] = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = fw_apply_act(v[j] + bias[j], ACT);
            if (p.g1 || p.g0) v[j] = fw_affine(v[j], g1[j], g0[j]);
        }
        const bool live = row < p.M;
        if (p.res_dtype != FW_DT_NONE && live) {
            const int64_t o = (int64_t)row * p.ldr + col;
            if (p.vec && col < p.N) {
                if (p.res_dtype == FW_DT_F32) {
                    const f32x4_t x = *(const f32x4_t*)((const float*)p.res + o), y = *(const f32x4_t*)((const float*)p.res + o + 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) { v[j] += x[j]; v[4 + j] += y[j]; }
                } else {
                    const u32x4_t w = *(const u32x4_t*)((const uint16_t*)p.res + o);
#pragma unroll
                    for (int j = 0; j < 4; ++j) { v[2 * j] += __uint_as_float(w[j] << 16); v[2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u); }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (col + j < p.N) v[j] += p.res_dtype == FW_DT_F32 ? ((const float*)p.res)[o + j] : bf16_bits_to_f32(((const uint16_t*)p.res)[o + j]);
            }
        }
        if (p.out_dtype == FW_DT_MXFP4) {
            // the value is rounded to bf16 first: a fused quantisation returns the bytes of fw_mxfp4_quant_rows on the bf16 output.
            // Columns past N are zeros of the padded row (the launcher's grid covers all of it).
            u32x4_t h;
#pragma unroll
            for (int j = 0; j < 4; ++j) h[j] = pack_bf16x2(col + 2 * j < p.N ? v[2 * j] : 0.f, col + 2 * j + 1 < p.N ? v[2 * j + 1] : 0.f);
            const uint32_t byte = mx_scale_byte(mx_quad_max(mx_top8_bf16(h)));
            const uint32_t codes = mx_pack8_bf16(h, mx_scale_f32(byte));
            if (live && col < p.cslabs * MX_SLAB) {
                *(uint32_t*)((uint8_t*)p.C + (int64_t)row * p.ldc + (col >> 1)) = codes;
                if ((lane & 3) == 0) p.cs[((int64_t)(row >> 5) * p.cslabs + (col >> 8)) * 256 + (row & 31) * 8 + ((col >> 5) & 7)] = (uint8_t)byte;
            }
        } else if (live) {
            const int64_t o = (int64_t)row * p.ldc + col;
            if (p.out_dtype == FW_DT_F32) {
                if (p.vec && col < p.N) {
                    *(f32x4_t*)((float*)p.C + o) = f32x4_t{v[0], v[1], v[2], v[3]};
                    *(f32x4_t*)((float*)p.C + o + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) if (col + j < p.N) ((float*)p.C)[o + j] = v[j];
                }
            } else {
                if (p.vec && col < p.N) {
                    *(u32x4_t*)((uint16_t*)p.C + o) = u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) if (col + j < p.N) ((uint16_t*)p.C)[o + j] = f32_to_bf16_bits(v[j]);
                }
            }
        }
    }
}

template <typename F>
__device__ __forceinline__ void mx_by_act(int act, F&& f) {
    switch (act) {
        case FW_ACT_RELU: f(std::integral_constant<int, FW_ACT_RELU>{}); break;
        case FW_ACT_GELU_TANH: f(std::integral_constant<int, FW_ACT_GELU_TANH>{}); break;
        case FW_ACT_GELU_ERF: f(std::integral_constant<int, FW_ACT_GELU_ERF>{}); break;
        case FW_ACT_SILU: f(std::integral_constant<int, FW_ACT_SILU>{}); break;
        default: f(std::integral_constant<int, FW_ACT_NONE>{}); break;
    }
}

// ---------------------------------------------------------------------------------------------------------------
// 128 x 128 tile, 4 waves (2 x 2, wave tile 64 x 64), K slabs of 256 in two 32 KiB stages: two work-groups per CU.
// ---------------------------------------------------------------------------------------------------------------
constexpr int SM = 128, SN = 128, SSTAGE = (SM + SN) * 128;

__global__ __launch_bounds__(256, 2) void gemm_mxfp4_128_kernel(MxArgs p) {
    __shared__ __attribute__((aligned(16))) char smem[2 * SSTAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, fi = lane & 31, hi = lane >> 5;
    int tm, tn;
    mx_tile(p, tm, tn);
    const int m0 = tm * SM, n0 = tn * SN;
    const auto ars = mx_rsrc(p.A + (int64_t)m0 * p.lda, (long long)(p.M - m0) * p.lda);
    const auto wrs = mx_rsrc(p.W + (int64_t)n0 * p.ldw, (long long)(p.N - n0) * p.ldw);
    // a DMA piece = 8 rows x 128 bytes; this wave's pieces of a slab: rows 32 wave .. 32 wave + 31 of both operands
    const int pr = lane >> 3, pc = lane & 7;
    const int va[2] = {pr * (int)p.lda + ((pc ^ (pr >> 1)) << 4), pr * (int)p.lda + ((pc ^ ((pr >> 1) | 4)) << 4)};
    const int vw[2] = {pr * (int)p.ldw + ((pc ^ (pr >> 1)) << 4), pr * (int)p.ldw + ((pc ^ ((pr >> 1) | 4)) << 4)};
    const int astep = __builtin_amdgcn_readfirstlane((int)p.lda * 8), wstep = __builtin_amdgcn_readfirstlane((int)p.ldw * 8);
    auto issue = [&](int st, int kt) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) FWX_BLDS16(ars, va[j & 1], kt * 128 + (wave * 4 + j) * astep, smem + st * SSTAGE + (wave * 4 + j) * 1024);
#pragma unroll
        for (int j = 0; j < 4; ++j) FWX_BLDS16(wrs, vw[j & 1], kt * 128 + (wave * 4 + j) * wstep, smem + st * SSTAGE + SM * 128 + (wave * 4 + j) * 1024);
    };
    // scale dwords: one per 32 rows and slab; row blocks past the end repeat the last one (their rows are zeros and are never stored)
    const int rba = (p.M + 31) / 32 - 1, rbw = (p.N + 31) / 32 - 1;
    const uint8_t* sap[2];
    const uint8_t* swp[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        sap[i] = p.sa + (int64_t)min((m0 >> 5) + wm * 2 + i, rba) * p.slabs * 256 + fi * 8 + hi * 4;
        swp[i] = p.sw + (int64_t)min((n0 >> 5) + wn * 2 + i, rbw) * p.slabs * 256 + fi * 8 + hi * 4;
    }
    int sca[2], scw[2];
    auto scales = [&](int kt) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) { sca[i] = *(const int*)(sap[i] + (int64_t)kt * 256); scw[i] = *(const int*)(swp[i] + (int64_t)kt * 256); }
    };
    f32x16_t acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const int swz = (fi >> 1) & 7;
    scales(0);
    issue(0, 0);
    for (int kt = 0; kt < p.slabs; ++kt) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's pieces of slab kt ...
        __syncthreads();                                  // ... and everybody's; nobody reads the other stage any more
        const char* a = smem + (kt & 1) * SSTAGE + (wm * 64 + fi) * 128;
        const char* w = smem + (kt & 1) * SSTAGE + SM * 128 + (wn * 64 + fi) * 128;
        const int ca[2] = {sca[0], sca[1]}, cw[2] = {scw[0], scw[1]};
        if (kt + 1 < p.slabs) { scales(kt + 1); issue((kt + 1) & 1, kt + 1); }
#define FWX_STEP(J) do { \
            const int off = ((4 * hi + (J)) ^ swz) << 4; \
            const i32x4_t a0 = *(const i32x4_t*)(a + off), a1 = *(const i32x4_t*)(a + 32 * 128 + off); \
            const i32x4_t w0 = *(const i32x4_t*)(w + off), w1 = *(const i32x4_t*)(w + 32 * 128 + off); \
            acc[0][0] = FWX_MFMA(a0, w0, acc[0][0], J, ca[0], cw[0]); \
            acc[0][1] = FWX_MFMA(a0, w1, acc[0][1], J, ca[0], cw[1]); \
            acc[1][0] = FWX_MFMA(a1, w0, acc[1][0], J, ca[1], cw[0]); \
            acc[1][1] = FWX_MFMA(a1, w1, acc[1][1], J, ca[1], cw[1]); } while (0)
        FWX_STEP(0); FWX_STEP(1); FWX_STEP(2); FWX_STEP(3);
#undef FWX_STEP
    }
    __syncthreads();                                      // everybody has read the last slab: the stages become the epilogue's space
    mx_by_act(p.act, [&](auto act) __attribute__((always_inline)) {
        mx_epilogue64<decltype(act)::value>(p, smem + wave * 16384, acc[0][0], acc[0][1], acc[1][0], acc[1][1], lane, m0 + wm * 64, n0 + wn * 64);
    });
}

}  // namespace

extern "C" int fw_gemm_mxfp4(const uint8_t* A, int64_t lda, const uint8_t* sa, const uint8_t* W, int64_t ldw, const uint8_t* sw,
                             void* C, int64_t ldc, int out_dtype, uint8_t* cs, int M, int N, int K,
                             const float* bias, int act, const float* g1, const float* g0,
                             const void* res, int64_t ldr, int res_dtype, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    const int slabs = mx_slabs(K);
    if (!A || !sa || !W || !sw || !C || K <= 0 || lda < (int64_t)slabs * 128 || ldw < (int64_t)slabs * 128 || (lda % 16) || (ldw % 16) ||
        lda >= (1 << 23) || ldw >= (1 << 23) || ((((uintptr_t)A) | ((uintptr_t)W)) & 15) || ((((uintptr_t)sa) | ((uintptr_t)sw)) & 3)) {
        fw_set_error("fw_gemm_mxfp4: K > 0; A / W 16-byte aligned with roundup(K, 256) / 2 <= ld < 2^23, ld % 16 == 0; scales 4-byte aligned"); return FW_E_BADARG; }
    if (act < FW_ACT_NONE || act > FW_ACT_SILU) { fw_set_error("fw_gemm_mxfp4: bad act"); return FW_E_BADARG; }
    const int cslabs = mx_slabs(N);
    if (out_dtype == FW_DT_MXFP4) {
        if (!cs || ldc < (int64_t)cslabs * 128 || (ldc % 16) || (((uintptr_t)C) & 15) || (((uintptr_t)cs) & 3)) {
            fw_set_error("fw_gemm_mxfp4: MXFP4 output needs c_scale, C 16-byte aligned, ldc % 16 == 0 and ldc >= roundup(N, 256) / 2"); return FW_E_BADARG; }
    } else if ((out_dtype != FW_DT_BF16 && out_dtype != FW_DT_F32) || ldc < N || (((uintptr_t)C) & (out_dtype == FW_DT_F32 ? 3 : 1))) {
        fw_set_error("fw_gemm_mxfp4: out_dtype bf16 / f32 / mxfp4, ldc >= N and an aligned C required"); return FW_E_BADARG; }
    if (res_dtype != FW_DT_NONE && (!res || (res_dtype != FW_DT_BF16 && res_dtype != FW_DT_F32) || ldr < N || (((uintptr_t)res) & (res_dtype == FW_DT_F32 ? 3 : 1)))) {
        fw_set_error("fw_gemm_mxfp4: res_dtype set but res NULL, misaligned, of another type or ldr < N"); return FW_E_BADARG; }
    if ((((uintptr_t)bias) | ((uintptr_t)g1) | ((uintptr_t)g0)) & 3) { fw_set_error("fw_gemm_mxfp4: misaligned bias / g1 / g0"); return FW_E_BADARG; }
    MxArgs p;
    p.A = A; p.lda = lda; p.sa = sa; p.W = W; p.ldw = ldw; p.sw = sw; p.C = C; p.ldc = ldc; p.out_dtype = out_dtype; p.cs = cs;
    p.M = M; p.N = N; p.slabs = slabs; p.bias = bias; p.act = act; p.g1 = g1; p.g0 = g0;
    p.res = res; p.ldr = ldr; p.res_dtype = res_dtype; p.cslabs = cslabs;
    // 16-byte accesses of 8 columns in the epilogue
    const int ce = out_dtype == FW_DT_F32 ? 4 : 8, re = res_dtype == FW_DT_F32 ? 4 : 8;
    p.vec = (N % 8) == 0 && (out_dtype == FW_DT_MXFP4 || ((ldc % ce) == 0 && (((uintptr_t)C) & 15) == 0)) &&
            (res_dtype == FW_DT_NONE || ((ldr % re) == 0 && (((uintptr_t)res) & 15) == 0));
    const int n_cover = out_dtype == FW_DT_MXFP4 ? cslabs * MX_SLAB : N;       // the padding of a quantised row is written too
    p.tiles_m = (M + SM - 1) / SM; p.tiles_n = (n_cover + SN - 1) / SN;
    const int64_t nwg = (int64_t)p.tiles_m * p.tiles_n;
    if (nwg > 0x7fffffff) { fw_set_error("fw_gemm_mxfp4: grid too large"); return FW_E_BADARG; }
    hipLaunchKernelGGL(gemm_mxfp4_128_kernel, dim3((unsigned)nwg), dim3(256), 0, (hipStream_t)stream, p);
    return (int)hipGetLastError();
}
