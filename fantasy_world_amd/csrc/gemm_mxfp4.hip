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
    int tiles_m, tiles_n, vec, cslabs, past;
};

// the upper half of the 8-register operand type is not read for fp4
#define FWX_MFMA(A, B, C, J, SA, SB) __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4( \
    i32x8_t{(A)[0], (A)[1], (A)[2], (A)[3], 0, 0, 0, 0}, i32x8_t{(B)[0], (B)[1], (B)[2], (B)[3], 0, 0, 0, 0}, C, 4, 4, J, SA, J, SB)
#define FWX_BLDS16(rs, voff, soff, ldsptr) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, FW_LDS_PTR(ldsptr), 16, voff, soff, 0, 0)

#define FWX_BARRIER() do { __builtin_amdgcn_sched_barrier(0); asm volatile("s_barrier" ::: "memory"); __builtin_amdgcn_sched_barrier(0); } while (0)
template <int N> __device__ __forceinline__ void mx_wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// descriptor over the rows from `base` on: an access past `bytes` reads zeros (a tile that lies in a quantised row's padding has no rows at all)
__device__ __forceinline__ auto mx_rsrc(const uint8_t* base, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)(unsigned)(bytes > 0xffffffffLL ? 0xffffffffLL : bytes < 0 ? 0 : bytes), 0x00020000);
}

// the same over `rows` rows of `slabs` slabs, to the last byte of the last one: the stride's tail behind it need not be anybody's memory
__device__ __forceinline__ auto mx_rows_rsrc(const uint8_t* base, int rows, int64_t ld, int slabs) {
    return mx_rsrc(base, rows <= 0 ? 0 : (long long)(rows - 1) * ld + slabs * 128);
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

// GELU with erf:  x Phi(x) = max(x, 0) - |x| / 2 * erfc(|x| / sqrt 2),  no cancellation on either side.  log2 erfc(z / sqrt 2) is smooth and 0 at 0:
// a polynomial of degree 10 without constant term, fitted to 64-bit values on [0, 6] by least squares reweighted towards the smallest
// largest error, each point weighted by erfc itself down to 1e-3.  Error of erfc 6e-9 + fp32 rounding: 3.3e-8 of N(0, 0.3^2) and 2.8e-8 of N(0, 1) in the
// 2-norm, where 0.5 x (1 + erf) in fp32 is 4e-8 off.  Past 6 it falls on (the leading term is negative).  erff in its place costs 14 us per
// 128 x 256 tile.  Past 8 the value is x itself in fp32 (1 - Phi(8) = 6e-16), infinity included, where the difference below would be
// inf - inf * 0; at -infinity the formula is -inf * 0, a NaN, here as there.
__device__ __forceinline__ float mx_gelu_erf(float x) {
    const float z = fabsf(x);
    float q = -2.8891838e-8f;
    q = __builtin_fmaf(q, z, 8.6283444e-7f);
    q = __builtin_fmaf(q, z, -1.1020638e-5f);
    q = __builtin_fmaf(q, z, 7.6711956e-5f);
    q = __builtin_fmaf(q, z, -2.7991601e-4f);
    q = __builtin_fmaf(q, z, -1.5661665e-6f);
    q = __builtin_fmaf(q, z, 6.9519272e-3f);
    q = __builtin_fmaf(q, z, -5.2446816e-2f);
    q = __builtin_fmaf(q, z, -4.5921841e-1f);
    q = __builtin_fmaf(q, z, -1.1511044f);
    const float v = __builtin_fmaf(-0.5f * z, __builtin_amdgcn_exp2f(q * z), fmaxf(x, 0.f));
    return x > 8.f ? x : v;
}
template <int ACT>
__device__ __forceinline__ float mx_act(float v) {
    // a block with a NaN makes its products NaN, and a ReLU keeps them: (v > 0 ? v : 0) would answer 0
    if (ACT == FW_ACT_RELU) return __builtin_elementwise_maximum(v, 0.f);
    return ACT == FW_ACT_GELU_ERF ? mx_gelu_erf(v) : fw_apply_act(v, ACT);
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

// Epilogue of NQ quadrants (32 RBK x 64 each, stacked along M) of a wave: bias and activation on the accumulators (a lane holds one column
// of each 32 x 32 block), then through LDS (16 KiB of the wave's own) to rows, per-column affine, residual, store.  There a lane owns 8
// consecutive columns of a row, 8 rows per step: 16-byte accesses in bf16, and with MXFP4 output a block of 32 columns is the 4 lanes of a
// quad.
// LDS image: 16-byte chunk c of row r lies at (c >> 1) + 8 ((c ^ r) & 1) of the row's 16: the 16 lanes of a read (chunk 2q or 2q + 1 of two
// neighbouring rows) then hit 16 different chunks of the 64 banks.
// VEC: every row of C and of the residual is 16-byte accessible and N % 8 == 0; otherwise (and RES < 0) element by element.
// With a residual and no activation all of a quadrant's residual rows are in flight before the transpose and the next quadrant's are issued
// as registers free up; with an activation as well (ACT_TOO) they follow the transpose, in the registers that the accumulators leave.
// HALVES (fp32 residual and fp32 output): a lane's 8 columns are 4 + 4, one half of the 64 each, so that the 8 lanes of a row touch 128
// contiguous bytes in every access; 8 consecutive fp32 are two accesses that each touch all 256 bytes.  Which half is first alternates
// with the row: the LDS reads then stay free of conflicts.  32760 x 5120 x 5120 with gate and residual in place:
// 566 us, 594 with 8 consecutive ones.
template <int RES, bool VEC, bool ACT_TOO, bool HALVES, bool PAST, int RBK, int NQ, typename Acc>
__device__ __forceinline__ void mx_epilogue(const MxArgs& p, char* reg, const Acc& acc, int lane, int m0, int n0) {
    const int fi = lane & 31, hi = lane >> 5, q = lane & 7, rl = lane >> 3;
    // this lane's columns: col .. + 3 and col2 .. + 3
    const int lc = HALVES ? 32 * (rl & 1) + q * 4 : q * 8, lc2 = HALVES ? lc ^ 32 : lc + 4;
    const int col = n0 + lc, col2 = n0 + lc2;
    const bool in = col < p.N, in2 = HALVES ? col2 < p.N : in;
    // and where they lie in a row of the LDS image
    const int at_lo = HALVES ? (lc >> 3) * 16 + ((q ^ rl) & 1) * 128 : q * 16 + (rl & 1) * 128;
    const int at_up = HALVES ? (lc2 >> 3) * 16 + ((q ^ rl) & 1) * 128 : q * 16 + ((rl & 1) ^ 1) * 128;
    const int res_dtype = RES < 0 ? p.res_dtype : RES;
    constexpr int IT = 4 * RBK;                           // steps of 8 rows
    u32x4_t rv[IT][RES == FW_DT_F32 ? 2 : 1];
    auto load_res = [&](int it, int row0) __attribute__((always_inline)) {
        const int row = row0 + rl;
        if (VEC && RES > 0 && (HALVES || in) && row < p.M) {
            // a scalar row address and a 32-bit lane offset: 64-bit addresses of 16 loads do not fit next to the accumulators
            const char* r = (const char*)p.res + ((int64_t)row0 * p.ldr + n0) * (RES == FW_DT_F32 ? 4 : 2) + (unsigned)(rl * (int)p.ldr + lc) * (RES == FW_DT_F32 ? 4u : 2u);
            if (!HALVES || in) rv[it][0] = fw_load<PAST, u32x4_t>(r);
            if (RES == FW_DT_F32 && (!HALVES || in2)) rv[it][RES == FW_DT_F32 ? 1 : 0] = fw_load<PAST, u32x4_t>(r + (lc2 - lc) * 4);
        }
    };
    if (VEC && RES > 0 && !ACT_TOO) {
#pragma unroll
        for (int it = 0; it < IT; ++it) load_res(it, m0 + it * 8);
    }
    float g1[8], g0[8], bias[2];
    const bool affine = p.g1 || p.g0;
#pragma unroll
    for (int j = 0; j < 2; ++j) bias[j] = p.bias && n0 + j * 32 + fi < p.N ? p.bias[n0 + j * 32 + fi] : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int c = j < 4 ? col + j : col2 + j - 4;
        g1[j] = p.g1 && c < p.N ? p.g1[c] : 1.f;
        g0[j] = p.g0 && c < p.N ? p.g0[c] : 0.f;
    }
    auto quadrant = [&](auto q_tag) __attribute__((always_inline)) {
        constexpr int Q = decltype(q_tag)::value;
        // chunk of column fi: fi >> 2, of column 32 + fi: 8 + (fi >> 2); rows of a register pair alternate in parity
        const int c = fi >> 2, base = (4 * hi) * 256 + (fi & 3) * 4 + (c >> 1) * 16;
        const int at[2] = {base + (c & 1) * 128, base + ((c & 1) ^ 1) * 128};
        mx_by_act(ACT_TOO ? p.act : FW_ACT_NONE, [&](auto act_tag) __attribute__((always_inline)) {
            constexpr int ACT = decltype(act_tag)::value;
#pragma unroll
            for (int rb = 0; rb < RBK; ++rb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row_l = rb * 32 + (r & 3) + 8 * (r >> 2);
                    *(float*)(reg + row_l * 256 + at[r & 1]) = mx_act<ACT>(acc[RBK * Q + rb][0][r] + bias[0]);
                    *(float*)(reg + row_l * 256 + at[r & 1] + 64) = mx_act<ACT>(acc[RBK * Q + rb][1][r] + bias[1]);
                }
        });
        if (VEC && RES > 0 && ACT_TOO) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int it = 0; it < IT; ++it) load_res(it, m0 + Q * 32 * RBK + it * 8);
        }
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int row_l = it * 8 + rl, row = m0 + Q * 32 * RBK + row_l;
            const f32x4_t lo = *(const f32x4_t*)(reg + row_l * 256 + at_lo), up = *(const f32x4_t*)(reg + row_l * 256 + at_up);
            float v[8] = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
            if (affine) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = fw_affine(v[j], g1[j], g0[j]);
            }
            const bool live = row < p.M;
            if (VEC && RES > 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (RES == FW_DT_F32) { v[j] += __uint_as_float(rv[it][0][j]); v[4 + j] += __uint_as_float(rv[it][RES == FW_DT_F32 ? 1 : 0][j]); }
                    else { v[2 * j] += __uint_as_float(rv[it][0][j] << 16); v[2 * j + 1] += __uint_as_float(rv[it][0][j] & 0xffff0000u); }
                }
                if (Q + 1 < NQ && !ACT_TOO) load_res(it, m0 + (Q + 1) * 32 * RBK + it * 8);
            } else if (res_dtype != FW_DT_NONE && live) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int64_t o = (int64_t)row * p.ldr + col + j;
                    if (col + j < p.N) v[j] += res_dtype == FW_DT_F32 ? ((const float*)p.res)[o] : bf16_bits_to_f32(((const uint16_t*)p.res)[o]);
                }
            }
            if (HALVES) {
                const int64_t o = (int64_t)row * p.ldc;
                if (live && in) fw_store<PAST>((float*)p.C + o + col, f32x4_t{v[0], v[1], v[2], v[3]});
                if (live && in2) fw_store<PAST>((float*)p.C + o + col2, f32x4_t{v[4], v[5], v[6], v[7]});
            } else if (p.out_dtype == FW_DT_MXFP4) {
                // the value is rounded to bf16 first: a fused quantisation returns the bytes of fw_mxfp4_quant_rows on the bf16 output.
                // Columns past N are zeros of the padded row (the launcher's grid covers all of it).
                u32x4_t h;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    h[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
                    if (VEC) { if (!in) h[j] = 0; }
                    else h[j] &= (col + 2 * j < p.N ? 0xffffu : 0u) | (col + 2 * j + 1 < p.N ? 0xffff0000u : 0u);
                }
                const uint32_t byte = mx_scale_byte(mx_quad_max(mx_top8_bf16(h)));
                const uint32_t codes = mx_pack8_bf16(h, mx_scale_f32(byte));
                if (live && col < p.cslabs * MX_SLAB) {
                    *(uint32_t*)((uint8_t*)p.C + (int64_t)row * p.ldc + (col >> 1)) = codes;
                    if ((lane & 3) == 0) p.cs[((int64_t)(row >> 5) * p.cslabs + (col >> 8)) * 256 + (row & 31) * 8 + ((col >> 5) & 7)] = (uint8_t)byte;
                }
            } else if (live && in) {
                const int64_t o = (int64_t)row * p.ldc + col;
                if (VEC) {
                    if (p.out_dtype == FW_DT_F32) {
                        *(f32x4_t*)((float*)p.C + o) = f32x4_t{v[0], v[1], v[2], v[3]};
                        *(f32x4_t*)((float*)p.C + o + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
                    } else {
                        fw_store<PAST>((uint16_t*)p.C + o, u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])});
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (col + j < p.N) {
                            if (p.out_dtype == FW_DT_F32) ((float*)p.C)[o + j] = v[j];
                            else ((uint16_t*)p.C)[o + j] = f32_to_bf16_bits(v[j]);
                        }
                }
            }
        }
    };
    quadrant(std::integral_constant<int, 0>{});
    if constexpr (NQ > 1) quadrant(std::integral_constant<int, 1>{});
}

// BIG: with outputs larger than the memory-side cache (256 MB; p.past), which are stored past the caches, the residual read the same way: they
// would only push the operands out (32760 x 5120 x 5120 with gate and fp32 residual: 573 us, 507 so; with the norm that reads it 758 and
// 702).  A smaller output stays where its reader finds it (8190 rows: 139 us, 156 past the caches).
template <bool BIG, int RBK, int NQ, typename Acc>
__device__ __forceinline__ void mx_finish(const MxArgs& p, char* reg, const Acc& acc, int lane, int m0, int n0) {
    const bool act = p.act != FW_ACT_NONE;
    if constexpr (BIG) {
        if (p.past && p.vec) {
            if (p.res_dtype == FW_DT_NONE) { mx_epilogue<FW_DT_NONE, true, true, false, true, RBK, NQ>(p, reg, acc, lane, m0, n0); return; }
            if (p.res_dtype == FW_DT_F32 && p.out_dtype == FW_DT_F32 && !act) { mx_epilogue<FW_DT_F32, true, false, true, true, RBK, NQ>(p, reg, acc, lane, m0, n0); return; }
            if (p.res_dtype == FW_DT_BF16 && !act) { mx_epilogue<FW_DT_BF16, true, false, false, true, RBK, NQ>(p, reg, acc, lane, m0, n0); return; }
        }
    }
    if (!p.vec) mx_epilogue<-1, false, true, false, false, RBK, NQ>(p, reg, acc, lane, m0, n0);
    else if (p.res_dtype == FW_DT_NONE) mx_epilogue<FW_DT_NONE, true, true, false, false, RBK, NQ>(p, reg, acc, lane, m0, n0);
    else if (p.res_dtype == FW_DT_F32) {
        if (act) mx_epilogue<FW_DT_F32, true, true, false, false, RBK, NQ>(p, reg, acc, lane, m0, n0);
        else if (p.out_dtype == FW_DT_F32) mx_epilogue<FW_DT_F32, true, false, true, false, RBK, NQ>(p, reg, acc, lane, m0, n0);
        else mx_epilogue<FW_DT_F32, true, false, false, false, RBK, NQ>(p, reg, acc, lane, m0, n0);
    } else if (act) mx_epilogue<FW_DT_BF16, true, true, false, false, RBK, NQ>(p, reg, acc, lane, m0, n0);
    else mx_epilogue<FW_DT_BF16, true, false, false, false, RBK, NQ>(p, reg, acc, lane, m0, n0);
}

// ---------------------------------------------------------------------------------------------------------------
// BM x BN tiles, K slabs of 256 values in a ring of ST stages: four waves multiply (wave tile 32 x 64 at 64 x 128, 64 x 64 at 64 x 256, 128 x 64
// at 128 x 256), four others do nothing but request codes and scale bytes by LDS-DMA, ST - 1 slabs ahead; one barrier a slab.  Nothing is
// requested past the last slab: the wait for it is the one for everything.
// Why loaders of their own: a wave that requests its slab is held until the CU's path from L2 (64 bytes a clock) has taken the request, and
// with one multiplying wave on a SIMD nobody multiplies meanwhile -- 257 x 5120 x 13824 took 39 us with four waves doing both, at two stages
// as at four, and takes 21.7 with loaders.  What bounds it now is LDS (the waves' fragment reads and the DMA's writes: 574, 840 and 1150
// clocks a slab of the three tiles, against 256, 512 and 1024 of the matrix pipe) and, per slab, the latency from the barrier to the first
// fragments.  Time of a slab with one tile a CU: 0.37, 0.58 and 0.93 us.
// ---------------------------------------------------------------------------------------------------------------
template <int BM, int BN, int ST>
__global__ __launch_bounds__(512, ST * (BM + BN) * 136 <= 80 * 1024 ? 4 : 2) void gemm_mxfp4_ring_kernel(MxArgs p) {
    constexpr int WAVES_N = BN / 64, WAVES_M = 4 / WAVES_N;
    constexpr int WM = BM / WAVES_M / 32;                 // 32-row blocks of a wave; it has two 32-column blocks
    constexpr int APC = BM / 32, WPC = BN / 32;           // DMA pieces (8 rows x 128 bytes) of a wave and slab
    constexpr int RB = (BM + BN) / 32;                    // 32-row groups of a slab = 256-byte scale tiles
    constexpr int SPC = (RB + 3) / 4;                     // scale pieces of a wave (a wave past the last group repeats it)
    constexpr int STAGE = (BM + BN) * 136;
    constexpr int LDS = ST * STAGE > 4 * 16384 ? ST * STAGE : 4 * 16384;
    __shared__ __attribute__((aligned(16))) char smem[LDS];
    const int lane = threadIdx.x & 63, wave8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = wave8 & 3;
    const int wm = wave / WAVES_N, wn = wave % WAVES_N, fi = lane & 31, hi = lane >> 5;
    int tm, tn;
    mx_tile(p, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const auto ars = mx_rows_rsrc(p.A + (int64_t)m0 * p.lda, min(p.M - m0, BM), p.lda, p.slabs);
    const auto wrs = mx_rows_rsrc(p.W + (int64_t)n0 * p.ldw, min(p.N - n0, BN), p.ldw, p.slabs);
    const int sstride = __builtin_amdgcn_readfirstlane(p.slabs * 256);
    const auto sars = mx_rsrc(p.sa + (int64_t)(m0 >> 5) * sstride, (long long)min((p.M + 31) / 32 - (m0 >> 5), BM / 32) * sstride);
    const auto swrs = mx_rsrc(p.sw + (int64_t)(n0 >> 5) * sstride, (long long)min((p.N + 31) / 32 - (n0 >> 5), BN / 32) * sstride);
    const int pr = lane >> 3, pc = lane & 7;
    const int va[2] = {pr * (int)p.lda + ((pc ^ (pr >> 1)) << 4), pr * (int)p.lda + ((pc ^ ((pr >> 1) | 4)) << 4)};
    const int vw[2] = {pr * (int)p.ldw + ((pc ^ (pr >> 1)) << 4), pr * (int)p.ldw + ((pc ^ ((pr >> 1) | 4)) << 4)};
    const int astep = __builtin_amdgcn_readfirstlane((int)p.lda * 8), wstep = __builtin_amdgcn_readfirstlane((int)p.ldw * 8);
    auto issue = [&](char* st, int kt) __attribute__((always_inline)) {
        const int k0 = kt * 128, s0 = kt * 256;
#pragma unroll
        for (int j = 0; j < APC; ++j) FWX_BLDS16(ars, va[j & 1], k0 + (wave * APC + j) * astep, st + (wave * APC + j) * 1024);
#pragma unroll
        for (int j = 0; j < WPC; ++j) FWX_BLDS16(wrs, vw[j & 1], k0 + (wave * WPC + j) * wstep, st + BM * 128 + (wave * WPC + j) * 1024);
#pragma unroll
        for (int j = 0; j < SPC; ++j) {
            const int g = min(wave + 4 * j, RB - 1);
            char* d = st + (BM + BN) * 128 + g * 256;
            if (g < BM / 32) __builtin_amdgcn_raw_ptr_buffer_load_lds(sars, FW_LDS_PTR(d), 4, lane * 4, s0 + g * sstride, 0, 0);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(swrs, FW_LDS_PTR(d), 4, lane * 4, s0 + (g - BM / 32) * sstride, 0, 0);
        }
    };
    const int swz = (fi >> 1) & 7;
    const int a_row = (wm * WM * 32 + fi) * 128, w_row = BM * 128 + (wn * 64 + fi) * 128;
    const int s_a = (BM + BN) * 128 + wm * WM * 256 + fi * 8 + hi * 4, s_w = (BM + BN) * 128 + (BM / 32 + wn * 2) * 256 + fi * 8 + hi * 4;

    if (wave8 >= 4) {
        static_assert(ST == 3, "a wait leaves the one slab after its own in flight");
        issue(smem, 0);
        if (p.slabs > 1) issue(smem + STAGE, 1);
        int nxt = 2;                                      // stage of slab kt + 2: that of kt - 1
        for (int kt = 0; kt < p.slabs; ++kt) {
            if (kt + 1 < p.slabs) mx_wait_vm<APC + WPC + SPC>();      // this wave's pieces of slab kt ...
            else mx_wait_vm<0>();
            FWX_BARRIER();                                // ... and every loader's; the others have read slab kt - 1
            if (kt + 2 < p.slabs) issue(smem + nxt * STAGE, kt + 2);
            nxt = nxt == 2 ? 0 : nxt + 1;
        }
        FWX_BARRIER();
        return;
    }
    f32x16_t acc[WM][2];                                  // [32-row block][32-column block]
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    int cur = 0;
    for (int kt = 0; kt < p.slabs; ++kt) {
        FWX_BARRIER();
        const char* st = smem + cur * STAGE;
        int ca[WM], cw[2];
#pragma unroll
        for (int i = 0; i < WM; ++i) ca[i] = *(const int*)(st + s_a + i * 256);
        cw[0] = *(const int*)(st + s_w);
        cw[1] = *(const int*)(st + s_w + 256);
#define FWX_STEP(J) do { \
            const int off = ((4 * hi + (J)) ^ swz) << 4; \
            const i32x4_t w0 = *(const i32x4_t*)(st + w_row + off), w1 = *(const i32x4_t*)(st + w_row + 32 * 128 + off); \
            _Pragma("unroll") for (int i = 0; i < WM; ++i) { \
                const i32x4_t a0 = *(const i32x4_t*)(st + a_row + i * 32 * 128 + off); \
                acc[i][0] = FWX_MFMA(a0, w0, acc[i][0], J, ca[i], cw[0]); \
                acc[i][1] = FWX_MFMA(a0, w1, acc[i][1], J, ca[i], cw[1]); } } while (0)
        FWX_STEP(0); FWX_STEP(1); FWX_STEP(2); FWX_STEP(3);
#undef FWX_STEP
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        cur = cur + 1 == ST ? 0 : cur + 1;
    }
    FWX_BARRIER();                                        // everybody has read the last slab: the stages become the epilogue's space
    mx_finish<false, (WM < 2 ? 1 : 2), (WM < 2 ? 1 : WM / 2)>(p, smem + wave * 16384, acc, lane, m0 + wm * WM * 32, n0 + wn * 64);
}

// ---------------------------------------------------------------------------------------------------------------
// 256 x 256 tile, 8 waves = 2 (M) x 4 (N) with wave tiles of 128 x 64, the two 4-wave groups one barrier slot apart:
//     slot:        2t          2t+1         2t+2         2t+3
//     group A:   LOAD(t)     MFMA(t)      LOAD(t+1)    MFMA(t+1)          LOAD(t): W fragments and A rows 0..63 of the wave tile, then this
//     group B:   MFMA(t-1)   LOAD(t)      MFMA(t)      LOAD(t+1)          wave's scale dwords and 8 DMA pieces; MFMA(t): 32 MFMAs in one
//                                                                         burst, A rows 64..127 re-read into the registers it has consumed
// so a SIMD always has one wave in its burst while the other one reads.  A in two 32 KiB stages, W in three (160 KiB): with the third, W(t+2)
// can be requested while W(t+1) waits.  Scale dwords go from memory to registers one slab ahead; they are requested ahead of the slab's
// pieces, so the counted wait for the pieces covers them.  Waits: a wave's requests in LOAD(t) are S(t+1) 6, A(t+1) 4, W(t+2) 4;
// vmcnt(4) at the end of the burst = everything but W(t+2) has landed; group B's W(t+1) is read one slot after its LOAD(t) by group A, so it
// waits vmcnt(14) there = all but this LOAD's own.
// ---------------------------------------------------------------------------------------------------------------
constexpr int LM = 256, LN = 256;
constexpr int L_A_STAGE = LM * 128, L_W_BASE = 2 * L_A_STAGE, L_W_STAGE = LN * 128, L_LDS = L_W_BASE + 3 * L_W_STAGE;

__global__ __launch_bounds__(512, 2) void gemm_mxfp4_256_kernel(MxArgs p) {
    __shared__ __attribute__((aligned(16))) char smem[L_LDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = wave >> 2, wn = wave & 3, fi = lane & 31, hi = lane >> 5;
    int tm, tn;
    mx_tile(p, tm, tn);
    const int m0 = tm * LM, n0 = tn * LN;
    const auto ars = mx_rows_rsrc(p.A + (int64_t)m0 * p.lda, min(p.M - m0, LM), p.lda, p.slabs);
    const auto wrs = mx_rows_rsrc(p.W + (int64_t)n0 * p.ldw, min(p.N - n0, LN), p.ldw, p.slabs);
    // scale tiles of this wave's 4 + 2 groups of 32 rows; groups past the end read zeros
    const int sstride = __builtin_amdgcn_readfirstlane(p.slabs * 256);
    const int ab = (m0 >> 5) + grp * 4, wb = (n0 >> 5) + wn * 2;
    const auto sars = mx_rsrc(p.sa + (int64_t)ab * sstride, (long long)((p.M + 31) / 32 - ab) * sstride);
    const auto swrs = mx_rsrc(p.sw + (int64_t)wb * sstride, (long long)((p.N + 31) / 32 - wb) * sstride);
    const int svo = fi * 8 + hi * 4;
    // a piece = 8 rows x 128 bytes; this wave's pieces: tile rows (grp * 128 + 32 wn) .. + 31 of both operands
    const int pr = lane >> 3, pc = lane & 7;
    const int va[2] = {pr * (int)p.lda + ((pc ^ (pr >> 1)) << 4), pr * (int)p.lda + ((pc ^ ((pr >> 1) | 4)) << 4)};
    const int vw[2] = {pr * (int)p.ldw + ((pc ^ (pr >> 1)) << 4), pr * (int)p.ldw + ((pc ^ ((pr >> 1) | 4)) << 4)};
    const int astep = __builtin_amdgcn_readfirstlane((int)p.lda * 8), wstep = __builtin_amdgcn_readfirstlane((int)p.ldw * 8);
    const int q0 = grp * 16 + 4 * wn;
    auto issue_a = [&](int as, int kt) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) FWX_BLDS16(ars, va[j & 1], kt * 128 + (q0 + j) * astep, smem + as * L_A_STAGE + (q0 + j) * 1024);
    };
    auto issue_w = [&](int ws, int kt) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) FWX_BLDS16(wrs, vw[j & 1], kt * 128 + (q0 + j) * wstep, smem + L_W_BASE + ws * L_W_STAGE + (q0 + j) * 1024);
    };
    auto load_scales = [&](int (&sa)[4], int (&sw)[2], int kt) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sa[i] = (int)__builtin_amdgcn_raw_buffer_load_b32(sars, svo, i * sstride + kt * 256, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) sw[i] = (int)__builtin_amdgcn_raw_buffer_load_b32(swrs, svo, i * sstride + kt * 256, 0);
    };
    const int swz = (fi >> 1) & 7;
    int co[4];                             // byte offset of k-step j's chunk inside a row
#pragma unroll
    for (int j = 0; j < 4; ++j) co[j] = ((4 * hi + j) ^ swz) << 4;
    const int a_row = (grp * 128 + fi) * 128, w_row = L_W_BASE + (wn * 64 + fi) * 128;

    f32x16_t acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    i32x4_t af[2][4], wf[2][4];            // [row / column block][k-step]
    int sa[4], sw[2], na[4], nw[2];        // scales of this slab and of the next

    const int nk = p.slabs;                // >= 4 (launcher)
    load_scales(sa, sw, 0);
    load_scales(na, nw, 1);
    issue_a(0, 0); issue_w(0, 0);
    issue_a(1, 1); issue_w(1, 1);
    issue_w(2, 2);
    mx_wait_vm<12>();
    FWX_BARRIER();
    if (grp == 1) FWX_BARRIER();

    int kt = 0, ws = 0;                    // ws = kt % 3
    // One slab.  The peeling is compile-time (first / steady / second-last / last), so LOAD and MFMA are one basic block each; the
    // accumulators are pinned by empty asm, which keeps the burst on its side of the barrier behind it.
    auto slab = [&](auto g_tag, auto first_tag, auto n1_tag, auto n2_tag) __attribute__((always_inline)) {
        constexpr int G = decltype(g_tag)::value;
        constexpr bool FIRST = decltype(first_tag)::value, N1 = decltype(n1_tag)::value, N2 = decltype(n2_tag)::value;   // kt == 0; kt + 1 < nk; kt + 2 < nk
        const int as = kt & 1;
        const char* ab_ = smem + as * L_A_STAGE + a_row;
        const char* wb_ = smem + ws * L_W_STAGE + w_row;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            wf[0][j] = *(const i32x4_t*)(wb_ + co[j]);
            wf[1][j] = *(const i32x4_t*)(wb_ + 32 * 128 + co[j]);
            af[0][j] = *(const i32x4_t*)(ab_ + co[j]);
            af[1][j] = *(const i32x4_t*)(ab_ + 32 * 128 + co[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (!FIRST && N1) {
            load_scales(na, nw, kt + 1);
            __builtin_amdgcn_sched_barrier(0);
            issue_a(as ^ 1, kt + 1);
            if (N2) issue_w(ws == 0 ? 2 : ws - 1, kt + 2);
        }
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (G == 1 && N1) {
            if (FIRST) mx_wait_vm<4>(); else if (N2) mx_wait_vm<14>(); else mx_wait_vm<10>();
        }
        FWX_BARRIER();
        __builtin_amdgcn_s_setprio(1);
#define FWX_LOWER(J) do { \
            acc[0][0] = FWX_MFMA(af[0][J], wf[0][J], acc[0][0], J, sa[0], sw[0]); \
            acc[0][1] = FWX_MFMA(af[0][J], wf[1][J], acc[0][1], J, sa[0], sw[1]); \
            __builtin_amdgcn_sched_barrier(0); \
            af[0][J] = *(const i32x4_t*)(ab_ + 64 * 128 + co[J]); \
            __builtin_amdgcn_sched_barrier(0); \
            acc[1][0] = FWX_MFMA(af[1][J], wf[0][J], acc[1][0], J, sa[1], sw[0]); \
            acc[1][1] = FWX_MFMA(af[1][J], wf[1][J], acc[1][1], J, sa[1], sw[1]); \
            __builtin_amdgcn_sched_barrier(0); \
            af[1][J] = *(const i32x4_t*)(ab_ + 96 * 128 + co[J]); \
            __builtin_amdgcn_sched_barrier(0); } while (0)
#define FWX_UPPER(J) do { \
            acc[2][0] = FWX_MFMA(af[0][J], wf[0][J], acc[2][0], J, sa[2], sw[0]); \
            acc[2][1] = FWX_MFMA(af[0][J], wf[1][J], acc[2][1], J, sa[2], sw[1]); \
            acc[3][0] = FWX_MFMA(af[1][J], wf[0][J], acc[3][0], J, sa[3], sw[0]); \
            acc[3][1] = FWX_MFMA(af[1][J], wf[1][J], acc[3][1], J, sa[3], sw[1]); } while (0)
        FWX_LOWER(0); FWX_LOWER(1); FWX_LOWER(2); FWX_LOWER(3);
        FWX_UPPER(0); FWX_UPPER(1); FWX_UPPER(2); FWX_UPPER(3);
#undef FWX_LOWER
#undef FWX_UPPER
        __builtin_amdgcn_s_setprio(0);
        asm volatile("" : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1]));
        asm volatile("" : "+v"(acc[2][0]), "+v"(acc[2][1]), "+v"(acc[3][0]), "+v"(acc[3][1]));
        if (N1) {
            if (N2) mx_wait_vm<4>(); else mx_wait_vm<0>();
#pragma unroll
            for (int i = 0; i < 4; ++i) sa[i] = na[i];
            sw[0] = nw[0]; sw[1] = nw[1];
        }
        FWX_BARRIER();
        ++kt;
        ws = ws == 2 ? 0 : ws + 1;
    };
    using T = std::true_type;
    using F = std::false_type;
    auto mainloop = [&](auto g_tag) __attribute__((always_inline)) {
        // (distinct opaque markers at both ends of an arm keep the compiler from hoisting the arms' common head above the group branch
        //  and from merging their tails)
        asm volatile("; mxfp4 two-slot mainloop, group %0: begin" ::"n"(decltype(g_tag)::value) : "memory");
        slab(g_tag, T{}, T{}, T{});
        while (kt < nk - 2) slab(g_tag, F{}, T{}, T{});
        slab(g_tag, F{}, T{}, F{});                           // kt = nk - 2
        slab(g_tag, F{}, F{}, F{});                           // kt = nk - 1
        asm volatile("; mxfp4 two-slot mainloop, group %0: end" ::"n"(decltype(g_tag)::value) : "memory");
    };
    if (grp == 0) { mainloop(std::integral_constant<int, 0>{}); FWX_BARRIER(); }
    else mainloop(std::integral_constant<int, 1>{});
    mx_finish<true, 2, 2>(p, smem + wave * 16384, acc, lane, m0 + grp * 128, n0 + wn * 64);
}

// ---------------------------------------------------------------------------------------------------------------
// Up to 32 rows: the weights are all there is to read, so the split is made for them.  A work-group takes 16 NB columns (W rows) and all
// rows of A (16 MT), its 8 waves a run of K each, v_mfma_scale_f32_16x16x128_f8f6f4 (lane l: row l & 15, block l >> 4 of four); a wave requests all
// W of its next 2 to 8 instructions (UB) before it multiplies, which keeps the whole matrix in flight across the chip.  The eight partial sums are added
// in LDS, in wave order: no atomics, no workspace, the same bits every time.
// FUSED: A is bf16 and the work-group quantises all of it into LDS, a block of 32 a lane, while its first W is on the way;
// every work-group repeats that, which costs less than a launch and a round trip through memory.  LDS rows are padded by one 16-byte chunk,
// so the fragment reads of 16 rows hit 16 different chunks.
// ---------------------------------------------------------------------------------------------------------------
#define FWX_MFMA16(A, B, C, SA, SB) __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4( \
    i32x8_t{(A)[0], (A)[1], (A)[2], (A)[3], 0, 0, 0, 0}, i32x8_t{(B)[0], (B)[1], (B)[2], (B)[3], 0, 0, 0, 0}, C, 4, 4, 0, SA, 0, SB)

template <int MT, int NB, bool FUSED>
__global__ __launch_bounds__(512, 4) void gemm_mxfp4_rows_kernel(MxArgs p, int blocks) {
    constexpr int UB = MT * NB == 1 ? 8 : NB == 4 ? 2 : 4;      // instructions (of 128 values of K) whose operands are requested together
    __shared__ float red[8][MT * NB * 4][64];
    extern __shared__ u32x4_t mx_rows[];                  // FUSED: codes [M][slabs * 8 + 1] chunks, then scale bytes [M][slabs * 8]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, h = lane >> 4;
    const int n0 = blockIdx.x * 16 * NB;
    const int units = p.slabs * 2, u0 = wave * units / 8, u1 = (wave + 1) * units / 8;
    // rows past the end repeat the last one: their results are never stored
    const uint8_t* wp[NB];
    const uint8_t* swp[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int n = min(n0 + b * 16 + r, p.N - 1);
        wp[b] = p.W + (int64_t)n * p.ldw + h * 16;
        swp[b] = p.sw + (int64_t)(n >> 5) * p.slabs * 256 + (n & 31) * 8 + h;
    }
    const int chunks = p.slabs * 8;                       // 16-byte chunks = blocks of a padded row
    uint8_t* smem_s = (uint8_t*)(mx_rows + p.M * (chunks + 1));
    const uint8_t* ap[MT];
    const uint8_t* sap[MT];
    f32x4_t acc[MT][NB];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = min(m * 16 + r, p.M - 1);
        ap[m] = FUSED ? (const uint8_t*)(mx_rows + row * (chunks + 1) + h) : p.A + (int64_t)row * p.lda + h * 16;
        sap[m] = FUSED ? smem_s + row * chunks + h : p.sa + row * 8 + h;
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[m][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    i32x4_t w[UB][NB], a[UB][MT];
    int sw[UB][NB], sa[UB][MT];
    auto load_w = [&](int u) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < UB; ++i)
            if (u + i < u1) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    w[i][b] = *(const i32x4_t*)(wp[b] + (int64_t)(u + i) * 64);
                    sw[i][b] = swp[b][(int64_t)((u + i) >> 1) * 256 + ((u + i) & 1) * 4];
                }
            }
    };
    load_w(u0);
    if (FUSED) {
        for (int i = threadIdx.x; i < p.M * chunks; i += 512) {
            const int row = i / chunks, c = i - row * chunks;
            u32x4_t x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = c < blocks ? *(const u32x4_t*)(p.A + (int64_t)row * p.lda + c * 64 + j * 16) : u32x4_t{0, 0, 0, 0};
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) top = max(top, mx_top8_bf16(x[j]));
            const uint32_t byte = mx_scale_byte(top);
            u32x4_t q;
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = mx_pack8_bf16(x[j], mx_scale_f32(byte));
            mx_rows[row * (chunks + 1) + c] = q;
            smem_s[i] = (uint8_t)byte;
        }
        __syncthreads();
    }
    for (int u = u0; u < u1; u += UB) {
        if (u != u0) load_w(u);
#pragma unroll
        for (int i = 0; i < UB; ++i)
            if (u + i < u1) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    a[i][m] = *(const i32x4_t*)(ap[m] + (int64_t)(u + i) * 64);
                    sa[i][m] = FUSED ? sap[m][(u + i) * 4] : sap[m][(int64_t)((u + i) >> 1) * 256 + ((u + i) & 1) * 4];
                }
            }
#pragma unroll
        for (int i = 0; i < UB; ++i)
            if (u + i < u1) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int b = 0; b < NB; ++b) acc[m][b] = FWX_MFMA16(a[i][m], w[i][b], acc[m][b], sa[i][m], sw[i][b]);
            }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[wave][(m * NB + b) * 4 + i][lane] = acc[m][b][i];
    __syncthreads();
    // lane l of a fragment holds column l & 15 of rows 4 (l >> 4) .. + 3
    constexpr int COLS = 16 * NB;
#pragma unroll
    for (int e = threadIdx.x; e < 16 * MT * COLS; e += 512) {      // whole waves: 256, 512 or 1024 results
        const int row = e / COLS, c = e % COLS, col = n0 + c;
        const int slot = ((row >> 4) * NB + (c >> 4)) * 4 + (row & 3), at = ((row >> 2) & 3) * 16 + (c & 15);
        float v = red[0][slot][at];
#pragma unroll
        for (int k = 1; k < 8; ++k) v += red[k][slot][at];
        const bool in = col < p.N, live = row < p.M;
        if (p.bias && in) v += p.bias[col];
        mx_by_act(p.act, [&](auto act) __attribute__((always_inline)) { v = mx_act<decltype(act)::value>(v); });
        if ((p.g1 || p.g0) && in) v = fw_affine(v, p.g1 ? p.g1[col] : 1.f, p.g0 ? p.g0[col] : 0.f);
        if (p.res_dtype != FW_DT_NONE && in && live) {
            const int64_t o = (int64_t)row * p.ldr + col;
            v += p.res_dtype == FW_DT_F32 ? ((const float*)p.res)[o] : bf16_bits_to_f32(((const uint16_t*)p.res)[o]);
        }
        if (NB > 1 && p.out_dtype == FW_DT_MXFP4) {      // 32 lanes hold a block
            const uint32_t b16 = in ? f32_to_bf16_bits(v) : 0;
            uint32_t top = (b16 & 0x7fffu) << 16;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
            const uint32_t byte = mx_scale_byte(top);
            uint32_t q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, mx_pair(b16), mx_scale_f32(byte), 0) & 15u;
            q <<= 4 * (c & 7);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) q |= (uint32_t)__shfl_xor((int)q, o, 64);
            if (live && (c & 7) == 0) *(uint32_t*)((uint8_t*)p.C + (int64_t)row * p.ldc + (col >> 1)) = q;
            if (live && (c & 31) == 0) p.cs[((int64_t)(row >> 5) * p.cslabs + (col >> 8)) * 256 + (row & 31) * 8 + ((col >> 5) & 7)] = (uint8_t)byte;
        } else if (live && in) {
            const int64_t o = (int64_t)row * p.ldc + col;
            if (p.out_dtype == FW_DT_F32) ((float*)p.C)[o] = v;
            else ((uint16_t*)p.C)[o] = f32_to_bf16_bits(v);
        }
    }
}

template <int BM, int BN, int ST>
int mx_launch_ring(MxArgs& p, int n_cover, hipStream_t st) {
    p.tiles_m = (p.M + BM - 1) / BM; p.tiles_n = (n_cover + BN - 1) / BN;
    const int64_t nwg = (int64_t)p.tiles_m * p.tiles_n;
    if (nwg > 0x7fffffff) { fw_set_error("fw_gemm_mxfp4: grid too large"); return FW_E_BADARG; }
    hipLaunchKernelGGL((gemm_mxfp4_ring_kernel<BM, BN, ST>), dim3((unsigned)nwg), dim3(512), 0, st, p);
    return (int)hipGetLastError();
}

// Which tile: the one whose rounds over the 256 CUs, at its measured time of a slab and of the rest of a tile (ns), end first.  A slab takes
// half as long on a nearly empty chip as on a full one (clock, L2); 64 x 128 tiles run two to a CU from 257 of them on.
//     tile        slab   rest      512 x 10240 x 5120   1565 x 5120 x 13824   2047 x 15360 x 5120   32760 x 15360 x 5120   (us measured)
//     64 x 128     300   2500            24.0                 82.2                 116.6                 1873
//     64 x 256     560   5000            28.6                 75.5                 119.6                 1830
//     128 x 256    950   7500            22.3                103.5                  95.2                 1453
//     256 x 256   1550  11000            31.5                102.7                  82.0                 1190
// All of them add the same instructions in the same order per output element: a row's bits do not depend on the choice.
int mx_tile_choice(int M, int n_cover, int slabs) {
    static const int shape[4][4] = {{64, 128, 300, 2500}, {64, 256, 560, 5000}, {128, 256, 950, 7500}, {256, 256, 1550, 11000}};
    int best = 0;
    int64_t least = INT64_MAX;
    for (int i = 0; i < (slabs >= 4 ? 4 : 3); ++i) {      // the 256 x 256 schedule needs four slabs
        const int64_t tiles = (int64_t)((M + shape[i][0] - 1) / shape[i][0]) * ((n_cover + shape[i][1] - 1) / shape[i][1]);
        const int64_t rounds = (tiles + 255) / 256;
        const int64_t slab = i > 0 ? shape[i][2] * (rounds * 256 + tiles) / (rounds * 512) : tiles > 256 ? 300 : 370;
        const int64_t t = rounds * (slabs * slab + shape[i][3]);
        if (t < least) { least = t; best = i; }
    }
    return best;
}

// Columns of a work-group: as few as give every CU one (16 NB, the whole K each), then wider rather than a second round.  Same bits each.
//     us, NB = 1 / 2 / 4     1 x 5120 x 5120    16 x 5120 x 5120    32 x 4096 x 1024    16 x 13824 x 5120    16 x 30000 x 2048
//     from MXFP4 rows         5.4 / 5.5 / 8.5     7.5 / 6.2 / 9.4     3.0 / 3.6 / 5.0    14.0 / 11.1 / 10.5    14.0 / 10.2 / 8.9
//     from bf16 rows          5.5 / 5.6 / 8.1    11.3 / 9.0 / 12.0    4.1 / 4.7 / 6.2    21.2 / 16.0 / 13.4    18.9 / 13.2 / 10.8
template <int MT, bool FUSED>
int mx_launch_rows(const MxArgs& p, int n_cover, int blocks, hipStream_t st) {
    const int lds = FUSED ? p.M * (p.slabs * 8 + 1) * 16 + p.M * p.slabs * 8 : 0;
    int nb = p.out_dtype == FW_DT_MXFP4 ? 2 : 1;
    while (nb < 4 && n_cover > 256 * 16 * nb) nb *= 2;
    const dim3 grid((unsigned)((n_cover + 16 * nb - 1) / (16 * nb)));
    if (nb == 4) hipLaunchKernelGGL((gemm_mxfp4_rows_kernel<MT, 4, FUSED>), grid, dim3(512), lds, st, p, blocks);
    else if (nb == 2) hipLaunchKernelGGL((gemm_mxfp4_rows_kernel<MT, 2, FUSED>), grid, dim3(512), lds, st, p, blocks);
    else hipLaunchKernelGGL((gemm_mxfp4_rows_kernel<MT, 1, FUSED>), grid, dim3(512), lds, st, p, blocks);
    return (int)hipGetLastError();
}

// Rows that fw_linear_mxfp4 quantises inside the product: at most 32, in whole 16-byte accessible blocks, that take at most 48 KiB of LDS.
// 21 x 4096 x 1024: 3.6 us, in two launches 8.3; 16 x 5120 x 5120: 9.0, in two launches 9.3 -- and 3 us less of the host's time each.
bool mx_rows_fused(const void* x, int64_t ldx, int M, int K) {
    return M <= 32 && K > 0 && (K % 32) == 0 && (ldx % 8) == 0 && (((uintptr_t)x) & 15) == 0 && (int64_t)M * (mx_slabs(K) * 136 + 16) <= 48 * 1024;
}

}  // namespace

// Work-groups read all of the operands while others store: an output shares no byte with any of them.  The residual is read by the lane
// that stores in its place, so C may be the residual -- the same rows in the same type.
static bool mx_overlap(const MxArgs& p, const FwSpan& a, const FwSpan& a_scale) {
    const int ce = p.out_dtype == FW_DT_F32 ? 4 : 2, re = p.res_dtype == FW_DT_F32 ? 4 : 2;
    const bool mx = p.out_dtype == FW_DT_MXFP4;
    const FwSpan c = mx ? FwSpan(p.C, p.ldc, (int64_t)p.cslabs * 128, p.M) : FwSpan(p.C, p.ldc * ce, (int64_t)p.N * ce, p.M);
    const FwSpan cs(mx ? p.cs : nullptr, ((int64_t)p.M + 31) / 32 * p.cslabs * 256), res(p.res_dtype == FW_DT_NONE ? nullptr : p.res, p.ldr * re, (int64_t)p.N * re, p.M);
    const FwSpan in[] = {a, a_scale, FwSpan(p.W, p.ldw, (int64_t)p.slabs * 128, p.N), FwSpan(p.sw, ((int64_t)p.N + 31) / 32 * p.slabs * 256),
                         FwSpan(p.bias, (int64_t)p.N * 4), FwSpan(p.g1, (int64_t)p.N * 4), FwSpan(p.g0, (int64_t)p.N * 4)};
    for (const FwSpan& i : in) if (fw_overlap(i, c) || fw_overlap(i, cs)) return true;
    return fw_overlap(c, cs) || fw_overlap(res, cs) || (fw_overlap(res, c) && !(res.same(c) && p.res_dtype == p.out_dtype));
}
static int mx_refuse_overlap() {
    fw_set_error("fw_gemm_mxfp4: the output overlaps an operand (it may be the residual: the same rows in the same type)");
    return FW_E_BADARG;
}

// Everything but A: the checks that fw_gemm_mxfp4 and fw_linear_mxfp4 share, and the arguments.  0, or the error code with its message set.
static int mx_args(MxArgs& p, const uint8_t* W, int64_t ldw, const uint8_t* sw, void* C, int64_t ldc, int out_dtype, uint8_t* cs, int M, int N, int K,
                   const float* bias, int act, const float* g1, const float* g0, const void* res, int64_t ldr, int res_dtype) {
    if (M > MX_MAX || N > MX_MAX || K > MX_MAX) { fw_set_error("fw_gemm_mxfp4: M, N and K below 2^31 - 256 required"); return FW_E_BADARG; }
    const int slabs = mx_slabs(K), cslabs = mx_slabs(N);
    if (!W || !sw || !C || K <= 0 || ldw < (int64_t)slabs * 128 || (ldw % 16) || ldw >= (1 << 23) || (((uintptr_t)W) & 15) || (((uintptr_t)sw) & 3)) {
        fw_set_error("fw_gemm_mxfp4: K > 0; W 16-byte aligned with roundup(K, 256) / 2 <= ldw < 2^23, ldw % 16 == 0; scales 4-byte aligned"); return FW_E_BADARG; }
    if (act < FW_ACT_NONE || act > FW_ACT_SILU) { fw_set_error("fw_gemm_mxfp4: bad act"); return FW_E_BADARG; }
    if (out_dtype == FW_DT_MXFP4) {
        if (!cs || ldc < (int64_t)cslabs * 128 || (ldc % 16) || (((uintptr_t)C) & 15) || (((uintptr_t)cs) & 3)) {
            fw_set_error("fw_gemm_mxfp4: MXFP4 output needs c_scale, C 16-byte aligned, ldc % 16 == 0 and ldc >= roundup(N, 256) / 2"); return FW_E_BADARG; }
    } else if ((out_dtype != FW_DT_BF16 && out_dtype != FW_DT_F32) || ldc < N || (((uintptr_t)C) & (out_dtype == FW_DT_F32 ? 3 : 1))) {
        fw_set_error("fw_gemm_mxfp4: out_dtype bf16 / f32 / mxfp4, ldc >= N and an aligned C required"); return FW_E_BADARG; }
    if (res_dtype != FW_DT_NONE && (!res || (res_dtype != FW_DT_BF16 && res_dtype != FW_DT_F32) || ldr < N || (((uintptr_t)res) & (res_dtype == FW_DT_F32 ? 3 : 1)))) {
        fw_set_error("fw_gemm_mxfp4: res_dtype set but res NULL, misaligned, of another type or ldr < N"); return FW_E_BADARG; }
    if ((((uintptr_t)bias) | ((uintptr_t)g1) | ((uintptr_t)g0)) & 3) { fw_set_error("fw_gemm_mxfp4: misaligned bias / g1 / g0"); return FW_E_BADARG; }
    p.W = W; p.ldw = ldw; p.sw = sw; p.C = C; p.ldc = ldc; p.out_dtype = out_dtype; p.cs = cs;
    p.M = M; p.N = N; p.slabs = slabs; p.bias = bias; p.act = act; p.g1 = g1; p.g0 = g0;
    p.res = res; p.ldr = ldr; p.res_dtype = res_dtype; p.cslabs = cslabs;
    // 16-byte accesses of 8 columns in the epilogue
    const int ce = out_dtype == FW_DT_F32 ? 4 : 8, re = res_dtype == FW_DT_F32 ? 4 : 8;
    p.vec = (N % 8) == 0 && (out_dtype == FW_DT_MXFP4 || ((ldc % ce) == 0 && (((uintptr_t)C) & 15) == 0)) &&
            (res_dtype == FW_DT_NONE || ((ldr % re) == 0 && (((uintptr_t)res) & 15) == 0 && ldr < (1 << 26)));
    p.past = out_dtype != FW_DT_MXFP4 && (int64_t)M * N * (out_dtype == FW_DT_F32 ? 4 : 2) > FW_CACHE_BYTES;
    return 0;
}

extern "C" int fw_gemm_mxfp4(const uint8_t* A, int64_t lda, const uint8_t* sa, const uint8_t* W, int64_t ldw, const uint8_t* sw,
                             void* C, int64_t ldc, int out_dtype, uint8_t* cs, int M, int N, int K,
                             const float* bias, int act, const float* g1, const float* g0,
                             const void* res, int64_t ldr, int res_dtype, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    MxArgs p;
    if (const int rc = mx_args(p, W, ldw, sw, C, ldc, out_dtype, cs, M, N, K, bias, act, g1, g0, res, ldr, res_dtype)) return rc;
    const int slabs = p.slabs, cslabs = p.cslabs;
    if (!A || !sa || lda < (int64_t)slabs * 128 || (lda % 16) || lda >= (1 << 23) || (((uintptr_t)A) & 15) || (((uintptr_t)sa) & 3)) {
        fw_set_error("fw_gemm_mxfp4: A 16-byte aligned with roundup(K, 256) / 2 <= lda < 2^23, lda % 16 == 0; scales 4-byte aligned"); return FW_E_BADARG; }
    p.A = A; p.lda = lda; p.sa = sa;
    if (mx_overlap(p, FwSpan(A, lda, (int64_t)slabs * 128, M), FwSpan(sa, ((int64_t)M + 31) / 32 * slabs * 256))) return mx_refuse_overlap();
    const int n_cover = out_dtype == FW_DT_MXFP4 ? cslabs * MX_SLAB : N;       // the padding of a quantised row is written too
    hipStream_t st = (hipStream_t)stream;
    if (M <= 16) return mx_launch_rows<1, false>(p, n_cover, 0, st);
    if (M <= 32) return mx_launch_rows<2, false>(p, n_cover, 0, st);
    int choice = mx_tile_choice(M, n_cover, slabs);
    if (choice == 3) {
        // a tail of at most 128 rows past the last full tile does not get a round of 256-row tiles: it goes by the same rule on its own
        const int tail = M % LM, m_big = tail > 0 && tail <= 128 && M > LM ? M - tail : M;
        MxArgs b = p;
        b.M = m_big;
        b.tiles_m = (m_big + LM - 1) / LM; b.tiles_n = (n_cover + LN - 1) / LN;
        const int64_t nwg = (int64_t)b.tiles_m * b.tiles_n;
        if (nwg > 0x7fffffff) { fw_set_error("fw_gemm_mxfp4: grid too large"); return FW_E_BADARG; }
        hipLaunchKernelGGL(gemm_mxfp4_256_kernel, dim3((unsigned)nwg), dim3(512), 0, st, b);
        const int rc = (int)hipGetLastError();
        if (rc || m_big == M) return rc;
        // whole scale tiles (32 rows) lie behind, so the rest's scales and quantised output start on a tile of their own
        p.A = A + (int64_t)m_big * lda; p.sa = sa + (int64_t)(m_big / 32) * slabs * 256; p.M = tail;
        if (out_dtype == FW_DT_MXFP4) { p.C = (uint8_t*)C + (int64_t)m_big * ldc; p.cs = cs + (int64_t)(m_big / 32) * cslabs * 256; }
        else p.C = (char*)C + (int64_t)m_big * ldc * (out_dtype == FW_DT_F32 ? 4 : 2);
        if (res_dtype != FW_DT_NONE) p.res = (const char*)res + (int64_t)m_big * ldr * (res_dtype == FW_DT_F32 ? 4 : 2);
        choice = min(mx_tile_choice(tail, n_cover, slabs), 2);
    }
    switch (choice) {
        case 0: return mx_launch_ring<64, 128, 3>(p, n_cover, st);
        case 1: return mx_launch_ring<64, 256, 3>(p, n_cover, st);
        default: return mx_launch_ring<128, 256, 3>(p, n_cover, st);
    }
}

extern "C" int64_t fw_linear_mxfp4_workspace_bytes(int M, int K) {
    if (M <= 0 || K <= 0) return 0;
    const int64_t slabs = mx_slabs(K);
    return (int64_t)M * slabs * 128 + ((int64_t)M + 31) / 32 * slabs * 256;
}

extern "C" int fw_linear_mxfp4(const uint16_t* x, int64_t ldx, const uint8_t* W, int64_t ldw, const uint8_t* sw,
                               void* C, int64_t ldc, int out_dtype, uint8_t* cs, int M, int N, int K,
                               const float* bias, int act, const float* g1, const float* g0,
                               const void* res, int64_t ldr, int res_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || ldx < K || (((uintptr_t)x) & 1)) { fw_set_error("fw_linear_mxfp4: bf16 x with ldx >= K required"); return FW_E_BADARG; }
    if (mx_rows_fused(x, ldx, M, K)) {
        MxArgs p;
        if (const int rc = mx_args(p, W, ldw, sw, C, ldc, out_dtype, cs, M, N, K, bias, act, g1, g0, res, ldr, res_dtype)) return rc;
        p.A = (const uint8_t*)x; p.lda = ldx * 2; p.sa = nullptr;
        if (mx_overlap(p, FwSpan(x, ldx * 2, (int64_t)K * 2, M), FwSpan(nullptr, 0))) return mx_refuse_overlap();
        const int n_cover = out_dtype == FW_DT_MXFP4 ? p.cslabs * MX_SLAB : N;
        return M <= 16 ? mx_launch_rows<1, true>(p, n_cover, K / 32, (hipStream_t)stream) : mx_launch_rows<2, true>(p, n_cover, K / 32, (hipStream_t)stream);
    }
    if (!workspace || workspace_bytes < fw_linear_mxfp4_workspace_bytes(M, K) || (((uintptr_t)workspace) & 15)) {
        fw_set_error("fw_linear_mxfp4: a 16-byte aligned workspace of fw_linear_mxfp4_workspace_bytes(M, K) required"); return FW_E_BADARG; }
    const int64_t lda = (int64_t)mx_slabs(K) * 128;
    uint8_t* q = (uint8_t*)workspace;
    uint8_t* s = q + (int64_t)M * lda;
    // the product's arguments first: nothing is launched for a call that is refused
    MxArgs p;
    if (const int rc = mx_args(p, W, ldw, sw, C, ldc, out_dtype, cs, M, N, K, bias, act, g1, g0, res, ldr, res_dtype)) return rc;
    if (mx_overlap(p, FwSpan(x, ldx * 2, (int64_t)K * 2, M), FwSpan(workspace, fw_linear_mxfp4_workspace_bytes(M, K)))) return mx_refuse_overlap();
    if (const int rc = fw_mxfp4_quant_rows(x, ldx, FW_DT_BF16, q, lda, s, M, K, stream)) return rc;
    return fw_gemm_mxfp4(q, lda, s, W, ldw, sw, C, ldc, out_dtype, cs, M, N, K, bias, act, g1, g0, res, ldr, res_dtype, stream);
}
