// Device-side pieces shared by the block-scaled product kernels.
#pragma once

#include "scaled.hpp"

namespace ctc {
namespace scaled {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// eight 8-bit codes (FMT 0 e4m3, 1 e5m2) to bf16, exactly
template <int FMT> __device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi)
{
    bf16x2 a, b, c, d;
    if constexpr (FMT) {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, 1.f, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, 1.f, true);
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
    }
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A lane's 32 codes of a block of 128 as an operand of the matrix core.  FAST: the codes themselves, for one
// v_mfma_f32_16x16x128_f8f6f4.  That is four times the rate of the bf16 form, but the 8-bit forms of the matrix core (the
// 16x16x32 ones too) align the products of each group of eight k to the largest one and drop what lies below its 2^-13 (measured:
// 2^16 + 2^3 in one group is exact, 2^16 + 2^2 gives 2^16; between groups the sum is f32).  On normal operands that is
// 1.5e-5 of the result's norm: far below the 2^-9 of a bf16 result, far above the 2^-24 of an f32 one.  Otherwise: the codes
// widened to bf16 (exactly) for four v_mfma_f32_16x16x32_bf16, which sum in f32.
template <int FMT, bool FAST> struct BlockOperand;
template <int FMT> struct BlockOperand<FMT, true> {
    v8i v;
    __device__ __forceinline__ void set(const v4i &lo, const v4i &hi) { v = v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}; }
};
template <int FMT> struct BlockOperand<FMT, false> {
    bf16x8 v[4];
    __device__ __forceinline__ void set(const v4i &lo, const v4i &hi)
    {
        v[0] = widen<FMT>(lo[0], lo[1]);
        v[1] = widen<FMT>(lo[2], lo[3]);
        v[2] = widen<FMT>(hi[0], hi[1]);
        v[3] = widen<FMT>(hi[2], hi[3]);
    }
};
// the 16 x 16 sums of a block's products: NT row tiles of B by one of A
template <int FA, bool FAST, int NT> __device__ __forceinline__ void block_sums(const BlockOperand<0, FAST> (&b)[NT], const BlockOperand<FA, FAST> &a, v4f (&d)[NT])
{
    const v4f zero = {0.f, 0.f, 0.f, 0.f};
    if constexpr (FAST) {
#pragma unroll
        for (int j = 0; j < NT; ++j) d[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j].v, a.v, zero, 0, FA, 0, 0, 0, 0);
    } else {
        // a quarter of every tile before the next quarter: the MFMAs of one tile depend on each other
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < NT; ++j) d[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j].v[q], a.v[q], q ? d[j] : zero, 0, 0, 0);
    }
}

// The product of a block's two scales as f * 2^e, f of 1 to 4 in magnitude: as one f32 number it can be subnormal or infinite
// (scales of 2^-109 and 2^-30, of 2^64 and 2^100) where the block's term is neither.  Zeros, infinities and NaNs stay in f.
struct ScalePair {
    float f;
    int e;
};
__device__ __forceinline__ ScalePair scale_pair(float sa, float sb)
{
    return {4.f * (__builtin_amdgcn_frexp_mantf(sa) * __builtin_amdgcn_frexp_mantf(sb)), __builtin_amdgcn_frexp_expf(sa) + __builtin_amdgcn_frexp_expf(sb) - 2};
}
// acc + d * f * 2^e.  A power of two scales d without rounding, so these are the bits of fma(d, sa * sb, acc) wherever sa * sb is a normal number.
__device__ __forceinline__ float add_scaled(float d, ScalePair s, float acc) { return __builtin_fmaf(__builtin_ldexpf(d, s.e), s.f, acc); }

__device__ __forceinline__ v4i load16(const uint8_t *q)  // any alignment
{
    v4i v;
    __builtin_memcpy(&v, q, 16);
    return v;
}
// 16 bytes of a row from byte k on, zeros from byte k_end on; any alignment.  Nothing behind k_end is read: a chunk that the
// row ends in is the shifted end of the 16 bytes in front of k_end where the row has 16 (long_row), bytes otherwise.
__device__ __forceinline__ uint4 load_chunk(const uint8_t *row, int64_t k, int64_t k_end, bool long_row)
{
    uint4 u = make_uint4(0, 0, 0, 0);
    const int64_t left = k_end - k;
    if (left >= 16) {
        __builtin_memcpy(&u, row + k, 16);
    } else if (left > 0 && long_row) {
        uint64_t w[2];
        __builtin_memcpy(w, row + k_end - 16, 16);
        const int bits = 8 * (16 - (int)left);  // 8 .. 120
        const uint64_t lo = bits < 64 ? w[0] >> bits | w[1] << (64 - bits) : w[1] >> (bits - 64), hi = bits < 64 ? w[1] >> bits : 0;
        u = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
    } else if (left > 0) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i >> 2] |= (i < left ? (uint32_t)row[k + (i < left ? i : 0)] : 0u) << (8 * (i & 3));
        u = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return u;
}

__device__ __forceinline__ int64_t min64(int64_t a, int64_t b) { return a < b ? a : b; }
__device__ __forceinline__ int64_t clamp_offset(int64_t o, int64_t hi) { return o < 0 ? 0 : (o > hi ? hi : o); }


__device__ __forceinline__ uint16_t to_bf16(float f)
{
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);  // NaN stays one
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}
__device__ __forceinline__ float from_bf16(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }

// four consecutive n of row m, alpha and beta applied in f32, rounded once
__device__ __forceinline__ void store4(const ScaledGemmParams &p, int64_t at, int64_t n, v4f v, bool vec)
{
    if (p.c_f32) {
        float *c = static_cast<float *>(p.C) + at;
        if (vec && n + 4 <= p.N) {
            v4f o = v * p.alpha;
            if (p.beta != 0.f) o += p.beta * *reinterpret_cast<const v4f *>(c);
            *reinterpret_cast<v4f *>(c) = o;
            return;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < p.N) c[r] = p.alpha * v[r] + (p.beta != 0.f ? p.beta * c[r] : 0.f);
        return;
    }
    uint16_t *c = static_cast<uint16_t *>(p.C) + at;
    if (vec && n + 4 <= p.N) {
        uint2 old = make_uint2(0, 0);
        if (p.beta != 0.f) old = *reinterpret_cast<const uint2 *>(c);
        const uint16_t h[4] = {(uint16_t)old.x, (uint16_t)(old.x >> 16), (uint16_t)old.y, (uint16_t)(old.y >> 16)};
        uint16_t o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = to_bf16(p.alpha * v[r] + (p.beta != 0.f ? p.beta * from_bf16(h[r]) : 0.f));
        *reinterpret_cast<uint2 *>(c) = make_uint2((uint32_t)o[0] | (uint32_t)o[1] << 16, (uint32_t)o[2] | (uint32_t)o[3] << 16);
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (n + r < p.N) c[r] = to_bf16(p.alpha * v[r] + (p.beta != 0.f ? p.beta * from_bf16(c[r]) : 0.f));
}

// One block of 128 contracted elements of 16 rows of codes in a wave's registers, 32 bytes a lane.
//
// As the matrix core takes it, lane (fr = l % 16, fg = l / 16) holds bytes 16 fg .. and 64 + 16 fg .. of row fr.  Loaded that
// way, sixteen neighbouring lanes touch sixteen rows and the L1's tag lookups, one per 16 bytes, bound the kernel at 4.4 TB/s.  So
// the lanes load four abreast along a row (lane l: row l / 4, bytes 16 (l % 4) .. and 64 further: 64-byte pieces, a quarter of the
// lookups), and `turn` passes the block through 2 KB of LDS that belong to the wave alone.
//
// The loads have no branch: those of several blocks stay in flight together, where a branch per block makes the compiler wait for each.
struct Codes {
    v4i lo, hi;
};
// row: the lane's row + 16 (l % 4)
__device__ __forceinline__ Codes load_codes(const uint8_t *row, int64_t k)
{
    Codes c;
    c.lo = load16(row + k);
    c.hi = load16(row + k + 64);
    return c;
}
__device__ __forceinline__ Codes turn(const Codes &c, uint8_t *scratch, int lane)
{
    // [half][row][four 16-byte chunks], chunk c of row r at c ^ (r / 4 & 3): rows four apart share their banks
    const int wr = lane >> 2, wc = lane & 3, rr = lane & 15, rc = lane >> 4;
    uint8_t *to = scratch + wr * 64 + ((wc ^ ((wr >> 2) & 3)) << 4);
    const uint8_t *from = scratch + rr * 64 + ((rc ^ ((rr >> 2) & 3)) << 4);
    *reinterpret_cast<v4i *>(to) = c.lo;
    *reinterpret_cast<v4i *>(to + 1024) = c.hi;
    // other lanes' bytes are read: one wave's LDS accesses complete in order, the compiler is kept from moving them
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    Codes o;
    o.lo = *reinterpret_cast<const v4i *>(from);
    o.hi = *reinterpret_cast<const v4i *>(from + 1024);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    return o;
}
// the block that the rows end in, as the matrix core takes it (row: the lane's row fr + 16 fg, k_end counted from there): zeros from k_end on
__device__ __forceinline__ Codes load_last_codes(const uint8_t *row, int64_t k, int64_t k_end, bool long_row)
{
    Codes c;
    c.lo = __builtin_bit_cast(v4i, load_chunk(row, k, k_end, long_row));
    c.hi = __builtin_bit_cast(v4i, load_chunk(row, k + 64, k_end, long_row));
    return c;
}

}  // namespace scaled
}  // namespace ctc
