// MXFP4 device helpers (OCP Microscaling Formats v1.0): 32 consecutive e2m1 values share one E8M0 scale, a power of two.
//
// Encoding rule of this library.  With top = the largest magnitude of the block and E = its binary exponent,
//     scale = 2^(E - 2),  one binade more where top's mantissa is 1.75 or above,  within 2^-127 .. 2^125;
//     value -> e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6) of value / scale, to nearest, ties to the even code.
// A top of 1.75 * 2^E would round to 8 units of 2^(E - 2) and e2m1 ends at 6: with the plain 2^(E - 2) such a block clips its largest
// values by up to a quarter; a whole binade for every top above 1.5 costs the other 31 values a bit.  Relative error of 2^20 values with
// the rule / the plain floor / the bump from 1.5: normal 0.1119 / 0.1148 / 0.1154, Laplace 0.1241 / 0.1267 / 0.1320, behind a GELU
// 0.1390 / 0.1394 / 0.1474.
// (2^125 and not 2^126: 4 * 2^126 would decode to an infinity.)
// Infinities and NaN have no e2m1 form: their block's scale byte is 0xff (NaN), which makes every product with the block NaN.
//
// Storage.  Rows are packed two values a byte (the first in the low half), K padded with zeros to a multiple of 256 (Kp): q [rows][ldq],
// ldq >= Kp / 2.  Scale bytes: s [rows / 32][Kp / 256][32][8] -- the 8 bytes a row needs for 256 values next to those of its 31 neighbours,
// so that the dword lane (r, h) of a 32x32x64 scaled MFMA needs for four k-steps (blocks 4h .. 4h + 3 of the slab) is one coalesced
// 256-byte read per 32 rows and slab.
#pragma once
#include "fw_common.h"

constexpr int MX_SLAB = 256;                 // values of one padded K slab = 128 bytes of codes + 8 scale bytes a row

// largest number of values of a row (and of rows of a product): whole slabs and tiles of it are still counted in 32 bits
constexpr int MX_MAX = 0x7fffffff - MX_SLAB;

static inline int mx_slabs(int K) { return (int)(((int64_t)K + MX_SLAB - 1) / MX_SLAB); }

// Operands as the host sees them: `rows` rows of `width` bytes, `pitch` bytes apart (pitch >= width).  Absent ones have no rows.
struct FwSpan {
    uintptr_t at; int64_t pitch, width, rows;
    FwSpan(const void* p, int64_t pitch_, int64_t width_, int64_t rows_) : at((uintptr_t)p), pitch(pitch_), width(width_), rows(p && width_ > 0 ? rows_ : 0) {}
    FwSpan(const void* p, int64_t bytes) : FwSpan(p, bytes, bytes, 1) {}
    bool same(const FwSpan& o) const { return at == o.at && width == o.width && rows == o.rows && (pitch == o.pitch || rows == 1); }
    int64_t end() const { return (int64_t)at + (rows - 1) * pitch + width; }
};

// Do two operands share a byte?  Column slices of one buffer interleave without sharing any: equal pitches are decided by the distance
// modulo the pitch, others row by row.
static inline bool fw_overlap(const FwSpan& a, const FwSpan& b) {
    if (a.rows <= 0 || b.rows <= 0 || a.end() <= (int64_t)b.at || b.end() <= (int64_t)a.at) return false;
    if (a.rows > b.rows) return fw_overlap(b, a);
    const int64_t d = (int64_t)a.at - (int64_t)b.at, P = b.pitch;
    auto floor_div = [](int64_t n, int64_t m) { return n / m - (n % m < 0 ? 1 : 0); };
    if (a.pitch == P) {
        // row i of a starts r bytes into pitch i + k of b
        const int64_t k = floor_div(d, P), r = d - k * P;
        auto meet = [&](int64_t s) { return (s > 0 ? s : 0) < (b.rows < a.rows + s ? b.rows : a.rows + s); };      // some i with 0 <= i + s < b.rows
        return (r < b.width && meet(k)) || (r + a.width > P && meet(k + 1));
    }
    for (int64_t i = 0; i < a.rows; ++i) {
        const int64_t s = d + i * a.pitch, j = floor_div(s - b.width, P) + 1;                     // the first row of b that ends behind s
        if ((j > 0 ? j : 0) < b.rows && (j > 0 ? j : 0) * P < s + a.width) return true;
    }
    return false;
}

// scale byte from the fp32 bits of the largest magnitude (taken by integer compare: NaN sorts above infinity)
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    const int b = (int)e - 2 + ((top & 0x7fffffu) >= 0x600000u ? 1 : 0);
    return e == 255u ? 255u : (uint32_t)min(max(b, 0), 252);
}
// the scale as the conversion instructions take it: an fp32 whose exponent field is the byte (a field of 0 counts as 2^-127 there)
__device__ __forceinline__ float mx_scale_f32(uint32_t byte) { return __uint_as_float(byte << 23); }

// largest magnitude of 8 bf16 in four dwords, as fp32 bits
__device__ __forceinline__ uint32_t mx_top8_bf16(u32x4_t v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) { m = max(m, v[i] & 0x7fff0000u); m = max(m, (v[i] << 16) & 0x7fff0000u); }
    return m;
}
// maximum over the 4 lanes of a quad: 8 values a lane = one block of 32
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t m) {
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));      // lane ^ 1
    return max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));   // lane ^ 2
}
// a dword as two bf16, BY VALUE: hipcc's __builtin_bit_cast of a vector's element expression reads the vector's first element
__device__ __forceinline__ bf16x2_t mx_pair(uint32_t v) { return __builtin_bit_cast(bf16x2_t, v); }
// 8 bf16 -> 8 codes (one dword).  The conversion rounds to nearest, ties to the even code (checked against the definition for every bf16)
__device__ __forceinline__ uint32_t mx_pack8_bf16(u32x4_t v, float scale) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, mx_pair(v[0]), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, mx_pair(v[1]), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, mx_pair(v[2]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, mx_pair(v[3]), scale, 3);
}
__device__ __forceinline__ uint32_t mx_pack8_f32(const float* f, float scale) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[0], f[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[2], f[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[4], f[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[6], f[7], scale, 3);
}

// An array larger than the memory-side cache gains nothing from passing through the caches and costs what else lies there: PAST accesses go
// past them.
constexpr int64_t FW_CACHE_BYTES = (int64_t)256 << 20;
template <bool PAST, typename V>
__device__ __forceinline__ V fw_load(const void* a) {
    if constexpr (PAST) return __builtin_nontemporal_load((const V*)a);
    else return *(const V*)a;
}
template <bool PAST, typename V>
__device__ __forceinline__ void fw_store(void* a, V v) {
    if constexpr (PAST) __builtin_nontemporal_store(v, (V*)a);
    else *(V*)a = v;
}

// Vectors at any alignment of their element (the hardware takes them so): rows of an odd length or from an odd column on.
typedef f32x4_t __attribute__((aligned(4))) f32x4_odd_t;
typedef u32x2_t __attribute__((aligned(2))) u32x2_odd_t;
typedef u32x4_t __attribute__((aligned(2))) u32x4_odd_t;
