// Block quantiser on gfx950: x (bf16 or f32) to 8-bit codes with one f32 scale per block, and, in the same pass over x,
// the transposed matrix with blocks along the other index.
//
//   top = max(2^-100, largest finite |x| of the block),  scale = top / L,  q = rne8(x * (L / top)),
//   L = 448 (e4m3) or 57344 (e5m2), both quotients rounded to f32 once (IEEE division).
// The product x * (L / top) is rounded to f32 in front of the conversion; codes differ from those of the unrounded
// product only where the f32 value falls on a tie of the 8-bit grid by that rounding (one in 2^20 of the elements).  The floor keeps L / top and scale normal f32
// numbers; a block below it (an all-zero one among them) is coded on the floor's grid.  Infinities and NaNs do not
// count in `top`: they turn into the format's own NaN (e4m3 has no infinity) or infinity, and their block's other
// elements keep their codes.
//
// Both kernels are bound by HBM: x is read once, each output written once.
#include "scaled.hpp"

namespace ctc {

namespace {

constexpr float kFloor = 7.8886090522101181e-31f;  // 2^-100

template <int FMT> constexpr float largest() { return FMT ? 57344.f : 448.f; }

template <int FMT> __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d)
{
    int v = 0;
    if constexpr (FMT) {
        v = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, v, false);
        v = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, v, true);
    } else {
        v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, v, false);
        v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
    }
    return (uint32_t)v;
}

// Eight consecutive elements of a row as they lie in memory.  Magnitudes are compared as integers, two bf16 at a time:
// without their signs, finite numbers order like their bits and infinities and NaNs stand above them.
template <int SRC> struct Row8;
template <> struct Row8<2> {
    static constexpr int W = 4;
    static constexpr uint32_t kSigns = 0x80008000u;
    uint32_t w[4];
    static __device__ __forceinline__ uint32_t pmax(uint32_t a, uint32_t b)
    {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
    }
    static __device__ __forceinline__ uint32_t fold(uint32_t m) { return max(m & 0xffffu, m >> 16); }  // of both halves
    static __device__ __forceinline__ uint32_t finite(uint32_t m)
    {
        return ((m & 0xffffu) < 0x7f80u ? m & 0xffffu : 0u) | (m < 0x7f800000u ? m & 0xffff0000u : 0u);
    }
    static __device__ __forceinline__ bool special(uint32_t m) { return fold(m) >= 0x7f80u; }
    static __device__ __forceinline__ float value(uint32_t m) { return __uint_as_float(m << 16); }  // of a folded maximum
    __device__ __forceinline__ float at(int j) const { return __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16); }
    __device__ __forceinline__ void load(const void *x, int64_t at, int64_t left)
    {
        const uint16_t *p = static_cast<const uint16_t *>(x) + at;
        if (left >= 8) {
            __builtin_memcpy(w, p, 16);
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (2 * i < left ? (uint32_t)p[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)p[2 * i + 1] << 16 : 0u);
    }
};
template <> struct Row8<1> {
    static constexpr int W = 8;
    static constexpr uint32_t kSigns = 0x80000000u;
    uint32_t w[8];
    static __device__ __forceinline__ uint32_t pmax(uint32_t a, uint32_t b) { return max(a, b); }
    static __device__ __forceinline__ uint32_t fold(uint32_t m) { return m; }
    static __device__ __forceinline__ uint32_t finite(uint32_t m) { return m < 0x7f800000u ? m : 0u; }
    static __device__ __forceinline__ bool special(uint32_t m) { return m >= 0x7f800000u; }
    static __device__ __forceinline__ float value(uint32_t m) { return __uint_as_float(m); }
    __device__ __forceinline__ float at(int j) const { return __uint_as_float(w[j]); }
    __device__ __forceinline__ void load(const void *x, int64_t at, int64_t left)
    {
        const uint32_t *p = static_cast<const uint32_t *>(x) + at;
        if (left >= 8) {
            __builtin_memcpy(w, p, 32);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = i < left ? p[i] : 0u;
    }
};

// eight codes to q[0 .. 8), those with an index below n only
__device__ __forceinline__ void store8(uint8_t *q, uint32_t lo, uint32_t hi, int64_t n)
{
    if (n >= 8) {
        const uint2 u = make_uint2(lo, hi);
        __builtin_memcpy(q, &u, 8);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
}

// the maximum over the sixteen lanes of a DPP row, in all of them
template <typename R> __device__ __forceinline__ uint32_t max16(uint32_t m)
{
    m = R::pmax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x128, 0xf, 0xf, false));  // row_ror 8, 4, 2, 1
    m = R::pmax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x124, 0xf, 0xf, false));
    m = R::pmax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x122, 0xf, 0xf, false));
    return R::pmax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x121, 0xf, 0xf, false));
}

// One scale per row and 128 columns, no transpose: sixteen lanes own a group and load it whole (16 or 32 bytes a lane),
// so the maximum is four exchanges inside sixteen lanes and nothing passes through LDS.  bf16: 8192 x 4096 28.6 us, 3.5 TB/s,
// 4096 x 8192 25.7 us; 512 x 4096 and below the call's 8 to 9 us.
template <int SRC, int FMT> __global__ void __launch_bounds__(256) quantize_rows_kernel(QuantizeParams p, int64_t nblk, int64_t total)
{
    typedef Row8<SRC> R;
    const int64_t first = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
    const int64_t step = (int64_t)gridDim.x * 16;
    const int lane = threadIdx.x & 15;
    for (int64_t g = first; g < total; g += step) {
        const int64_t blk = g % nblk, rest = g / nblk;
        const int64_t row = rest % p.rows, b = rest / p.rows;
        const int64_t c = blk * kScaleBlock + lane * 8;
        R v;
        v.load(p.x, b * p.x_batch + row * p.ldx + c, p.cols - c);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < R::W; ++i) m = R::pmax(m, v.w[i] & ~R::kSigns);
        if (__any(R::special(m))) {
            m = 0;
#pragma unroll
            for (int i = 0; i < R::W; ++i) m = R::pmax(m, R::finite(v.w[i] & ~R::kSigns));
        }
        const float top = fmaxf(R::value(R::fold(max16<R>(m))), kFloor);
        const float r = largest<FMT>() / top;
        const uint32_t lo = pack4<FMT>(v.at(0) * r, v.at(1) * r, v.at(2) * r, v.at(3) * r);
        const uint32_t hi = pack4<FMT>(v.at(4) * r, v.at(5) * r, v.at(6) * r, v.at(7) * r);
        store8(p.out.q + b * p.out.batch + row * p.out.ld + c, lo, hi, p.cols - c);
        if (lane == 0) p.out.scale[b * p.out.s_batch + row * p.out.s_row + blk * p.out.s_blk] = top / largest<FMT>();
    }
}

// A 128 x 128 tile per workgroup, held in registers as it was loaded: thread (rg, cg) owns an 8 x 8 block (rows 8 rg ..,
// columns 8 cg ..), so a row's maximum is an exchange inside sixteen lanes, a column's one between the four row groups of
// a wave and one pass through LDS between the waves, and a block's eight column slices are the eight bytes that the
// transposed row takes: one 8-byte LDS store each, no byte shuffles through memory.  The transposed tile leaves LDS in
// 16-byte rows.  bf16: at most 128 registers, four workgroups a CU,
// whose loads, exchanges and stores cover each other (8192 x 4096, both ways: 29.4 us, 4.7 TB/s; with two workgroups 44);
// f32 spills there and takes three (5001 x 4104 tiles, both ways: 31 us, 3.9 TB/s; with four and spills 45).
template <int SRC, int FMT, bool TILES> __global__ void __launch_bounds__(256, SRC == 2 ? 4 : 3) quantize_tile_kernel(QuantizeParams p, unsigned nblk)
{
    typedef Row8<SRC> R;
    __shared__ __attribute__((aligned(16))) uint8_t image[128 * 128];
    __shared__ uint32_t part[4][16 * R::W];
    __shared__ uint32_t part_tile[4];
    const int t = threadIdx.x, cg = t & 15, rg = t >> 4, wave = t >> 6;
    const int64_t cblk = blockIdx.x % nblk, rblk = blockIdx.x / nblk;
    const int64_t c0 = cblk * 128 + cg * 8, r0 = rblk * 128 + rg * 8;
    const int64_t b = blockIdx.z;
    const bool rowwise = p.out.q != nullptr, transposed = p.out_t.q != nullptr;

    R v[8];
    const int64_t x0 = b * p.x_batch + r0 * p.ldx + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load(p.x, x0 + i * p.ldx, r0 + i < p.rows ? p.cols - c0 : 0);
    uint32_t rmax[8], cmax[R::W];
    auto maxima = [&](auto filter) {
#pragma unroll
        for (int j = 0; j < R::W; ++j) cmax[j] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            rmax[i] = 0;
#pragma unroll
            for (int j = 0; j < R::W; ++j) {
                const uint32_t m = filter(v[i].w[j] & ~R::kSigns);
                rmax[i] = R::pmax(rmax[i], m);
                cmax[j] = R::pmax(cmax[j], m);
            }
        }
    };
    maxima([](uint32_t m) { return m; });
    uint32_t all = 0;
#pragma unroll
    for (int j = 0; j < R::W; ++j) all = R::pmax(all, cmax[j]);
    if (__any(R::special(all))) {
        maxima([](uint32_t m) { return R::finite(m); });
        all = 0;
#pragma unroll
        for (int j = 0; j < R::W; ++j) all = R::pmax(all, cmax[j]);
    }
    float tile_top = kFloor;
    if constexpr (TILES) {
        uint32_t m = R::fold(max16<R>(all));
        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
        if ((t & 63) == 0) part_tile[wave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) tile_top = fmaxf(tile_top, R::value(part_tile[w]));
    }
    if (rowwise) {
        float top = tile_top;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (!TILES) top = fmaxf(R::value(R::fold(max16<R>(rmax[i]))), kFloor);
            const float r = largest<FMT>() / top;
            const int64_t row = r0 + i;
            if (row < p.rows && c0 < p.cols) {
                const uint32_t lo = pack4<FMT>(v[i].at(0) * r, v[i].at(1) * r, v[i].at(2) * r, v[i].at(3) * r);
                const uint32_t hi = pack4<FMT>(v[i].at(4) * r, v[i].at(5) * r, v[i].at(6) * r, v[i].at(7) * r);
                store8(p.out.q + b * p.out.batch + row * p.out.ld + c0, lo, hi, p.cols - c0);
            }
            if (!TILES && cg == 0 && row < p.rows) p.out.scale[b * p.out.s_batch + row * p.out.s_row + cblk * p.out.s_blk] = top / largest<FMT>();
        }
        if (TILES && t == 0) p.out.scale[b * p.out.s_batch + rblk * p.out.s_row + cblk * p.out.s_blk] = tile_top / largest<FMT>();
    }
    if (!transposed) return;
    if constexpr (!TILES) {
#pragma unroll
        for (int j = 0; j < R::W; ++j) {
            cmax[j] = R::pmax(cmax[j], (uint32_t)__shfl_xor((int)cmax[j], 16));
            cmax[j] = R::pmax(cmax[j], (uint32_t)__shfl_xor((int)cmax[j], 32));
        }
        if ((t & 48) == 0) {
#pragma unroll
            for (int j = 0; j < R::W; ++j) part[wave][cg * R::W + j] = cmax[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < R::W; ++j)
            cmax[j] = R::pmax(R::pmax(part[0][cg * R::W + j], part[1][cg * R::W + j]), R::pmax(part[2][cg * R::W + j], part[3][cg * R::W + j]));
    } else if (t == 0) {
        p.out_t.scale[b * p.out_t.s_batch + cblk * p.out_t.s_row + rblk * p.out_t.s_blk] = tile_top / largest<FMT>();
    }
    // image [column][128 rows], 16-byte chunk k of a line at k ^ (line / 8 & 7): the sixteen lanes of a row group write
    // column 8 cg + j, lines a kilobyte apart, and would all meet in the same banks without it
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float top = tile_top;
        if constexpr (!TILES) {
            top = fmaxf(R::value(SRC == 2 ? (j & 1 ? cmax[j >> 1] >> 16 : cmax[j >> 1] & 0xffffu) : cmax[j % R::W]), kFloor);
            if (rg == 0 && c0 + j < p.cols) p.out_t.scale[b * p.out_t.s_batch + (c0 + j) * p.out_t.s_row + rblk * p.out_t.s_blk] = top / largest<FMT>();
        }
        const float r = largest<FMT>() / top;
        const uint32_t lo = pack4<FMT>(v[0].at(j) * r, v[1].at(j) * r, v[2].at(j) * r, v[3].at(j) * r);
        const uint32_t hi = pack4<FMT>(v[4].at(j) * r, v[5].at(j) * r, v[6].at(j) * r, v[7].at(j) * r);
        *reinterpret_cast<uint2 *>(image + (cg * 8 + j) * 128 + (((rg >> 1) ^ (cg & 7)) << 4) + ((rg & 1) << 3)) = make_uint2(lo, hi);
    }
    __syncthreads();
    // eight lanes write one line
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int line = i * 32 + (t >> 3), chunk = t & 7;
        const int64_t col = cblk * 128 + line, row = rblk * 128 + chunk * 16;
        if (col >= p.cols || row >= p.rows) continue;
        const uint4 u = *reinterpret_cast<const uint4 *>(image + line * 128 + ((chunk ^ ((line >> 3) & 7)) << 4));
        uint8_t *dst = p.out_t.q + b * p.out_t.batch + col * p.out_t.ld + row;
        if (p.rows - row >= 16) {
            __builtin_memcpy(dst, &u, 16);
        } else {
            store8(dst, u.x, u.y, p.rows - row);
            if (p.rows - row > 8) store8(dst + 8, u.z, u.w, p.rows - row - 8);
        }
    }
}

template <int SRC, int FMT> void launch_fmt(const QuantizeParams &p, bool tiles, hipStream_t stream)
{
    const int64_t nblk = (p.cols + 127) / 128;
    if (!tiles && !p.out_t.q) {
        const int64_t total = nblk * p.rows * p.batch;
        int64_t blocks = (total + 15) / 16;
        if (blocks > 256 * 16) blocks = 256 * 16;
        hipLaunchKernelGGL((quantize_rows_kernel<SRC, FMT>), dim3((unsigned)blocks), dim3(256), 0, stream, p, nblk, total);
        return;
    }
    const dim3 grid((unsigned)(nblk * ((p.rows + 127) / 128)), 1, (unsigned)p.batch);
    if (tiles) hipLaunchKernelGGL((quantize_tile_kernel<SRC, FMT, true>), grid, dim3(256), 0, stream, p, (unsigned)nblk);
    else hipLaunchKernelGGL((quantize_tile_kernel<SRC, FMT, false>), grid, dim3(256), 0, stream, p, (unsigned)nblk);
}

}  // namespace

hipError_t launch_block_quantize(const QuantizeParams &p, hipStream_t stream)
{
    const ScaledMatrix &m = p.out.q ? p.out : p.out_t;
    const bool tiles = m.shift != 0;
    if (p.src == 2) {
        if (m.e5m2) launch_fmt<2, 1>(p, tiles, stream);
        else launch_fmt<2, 0>(p, tiles, stream);
    } else {
        if (m.e5m2) launch_fmt<1, 1>(p, tiles, stream);
        else launch_fmt<1, 0>(p, tiles, stream);
    }
    return hipGetLastError();
}

}  // namespace ctc
