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

// |x| of a finite x, 0 otherwise
__device__ __forceinline__ float finite_mag(float x)
{
    const float a = __builtin_fabsf(x);
    return a < __builtin_inff() ? a : 0.f;  // false for NaN
}

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

// eight consecutive elements of a row from column c on, zeros beyond `cols`
template <int SRC> __device__ __forceinline__ void load8(const void *x, int64_t at, int64_t c, int64_t cols, float (&v)[8])
{
    if (c + 8 <= cols) {
        if constexpr (SRC == 2) {
            uint4 u;
            __builtin_memcpy(&u, static_cast<const uint16_t *>(x) + at, 16);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
            __builtin_memcpy(v, static_cast<const float *>(x) + at, 32);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = 0.f;
        if (c + i < cols) {
            if constexpr (SRC == 2) v[i] = __uint_as_float((uint32_t)static_cast<const uint16_t *>(x)[at + i] << 16);
            else v[i] = static_cast<const float *>(x)[at + i];
        }
    }
}

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

__device__ __forceinline__ float max16(float m)
{
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    return m;
}

// One scale per row and 128 columns, no transpose: sixteen lanes own a group and load it whole (16 or 32 bytes a lane),
// so the maximum is four exchanges inside sixteen lanes and nothing passes through LDS.
template <int SRC, int FMT> __global__ void __launch_bounds__(256) quantize_rows_kernel(QuantizeParams p, int64_t nblk, int64_t total)
{
    const int64_t first = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
    const int64_t step = (int64_t)gridDim.x * 16;
    const int lane = threadIdx.x & 15;
    for (int64_t g = first; g < total; g += step) {
        const int64_t blk = g % nblk, rest = g / nblk;
        const int64_t row = rest % p.rows, b = rest / p.rows;
        const int64_t c = blk * kScaleBlock + lane * 8;
        float v[8];
        load8<SRC>(p.x, b * p.x_batch + row * p.ldx + c, c, p.cols, v);
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_mag(v[i]));
        const float top = fmaxf(max16(m), kFloor);
        const float r = largest<FMT>() / top;
        const uint32_t lo = pack4<FMT>(v[0] * r, v[1] * r, v[2] * r, v[3] * r);
        const uint32_t hi = pack4<FMT>(v[4] * r, v[5] * r, v[6] * r, v[7] * r);
        store8(p.out.q + b * p.out.batch + row * p.out.ld + c, lo, hi, p.cols - c);
        if (lane == 0) p.out.scale[b * p.out.s_batch + row * p.out.s_row + blk * p.out.s_blk] = top / largest<FMT>();
    }
}

// A 128 x 128 tile per workgroup, held in registers: thread (rg, cg) owns an 8 x 8 block (rows 8 rg .., columns 8 cg ..),
// so a row's maximum is an exchange inside sixteen lanes, a column's one between the four row groups of a wave and one
// pass through LDS between the waves, and a block's eight column slices are the eight bytes that the transposed
// row takes: one 8-byte LDS store each, no byte shuffles through memory.  The transposed tile leaves LDS in 16-byte rows.
template <int SRC, int FMT, bool TILES> __global__ void __launch_bounds__(256) quantize_tile_kernel(QuantizeParams p, unsigned nblk)
{
    __shared__ __attribute__((aligned(16))) uint8_t image[128 * 128];
    __shared__ float part[4][128];
    __shared__ float part_tile[4];
    const int t = threadIdx.x, cg = t & 15, rg = t >> 4, wave = t >> 6;
    const int64_t cblk = blockIdx.x % nblk, rblk = blockIdx.x / nblk;
    const int64_t c0 = cblk * 128 + cg * 8, r0 = rblk * 128 + rg * 8;
    const int64_t b = blockIdx.z;
    const bool rowwise = p.out.q != nullptr, transposed = p.out_t.q != nullptr;

    float v[8][8];  // [row][column]
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = r0 + i;
        if (row < p.rows && c0 < p.cols) {
            load8<SRC>(p.x, b * p.x_batch + row * p.ldx + c0, c0, p.cols, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        }
    }
    float rmax[8], cmax[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) cmax[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        rmax[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float m = finite_mag(v[i][j]);
            rmax[i] = fmaxf(rmax[i], m);
            cmax[j] = fmaxf(cmax[j], m);
        }
    }
    float tile_top = kFloor;
    if constexpr (TILES) {
        float m = rmax[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = fmaxf(m, rmax[i]);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
        if ((t & 63) == 0) part_tile[wave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) tile_top = fmaxf(tile_top, part_tile[w]);
    }
    if (rowwise) {
        float top = tile_top;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (!TILES) top = fmaxf(max16(rmax[i]), kFloor);
            const float r = largest<FMT>() / top;
            const int64_t row = r0 + i;
            if (row < p.rows && c0 < p.cols) {
                const uint32_t lo = pack4<FMT>(v[i][0] * r, v[i][1] * r, v[i][2] * r, v[i][3] * r);
                const uint32_t hi = pack4<FMT>(v[i][4] * r, v[i][5] * r, v[i][6] * r, v[i][7] * r);
                store8(p.out.q + b * p.out.batch + row * p.out.ld + c0, lo, hi, p.cols - c0);
            }
            if (!TILES && cg == 0 && row < p.rows)
                p.out.scale[b * p.out.s_batch + row * p.out.s_row + cblk * p.out.s_blk] = top / largest<FMT>();
        }
        if (TILES && t == 0)
            p.out.scale[b * p.out.s_batch + rblk * p.out.s_row + cblk * p.out.s_blk] = tile_top / largest<FMT>();
    }
    if (!transposed) return;
    if constexpr (!TILES) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cmax[j] = fmaxf(cmax[j], __shfl_xor(cmax[j], 16));
            cmax[j] = fmaxf(cmax[j], __shfl_xor(cmax[j], 32));
        }
        if ((t & 48) == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) part[wave][cg * 8 + j] = cmax[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j)
            cmax[j] = fmaxf(fmaxf(fmaxf(part[0][cg * 8 + j], part[1][cg * 8 + j]), fmaxf(part[2][cg * 8 + j], part[3][cg * 8 + j])), kFloor);
        if (rg == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + j < p.cols)
                    p.out_t.scale[b * p.out_t.s_batch + (c0 + j) * p.out_t.s_row + rblk * p.out_t.s_blk] = cmax[j] / largest<FMT>();
        }
    } else if (t == 0) {
        p.out_t.scale[b * p.out_t.s_batch + cblk * p.out_t.s_row + rblk * p.out_t.s_blk] = tile_top / largest<FMT>();
    }
    // image [column][128 rows], 16-byte chunk k of a line at k ^ (line / 8 & 7): the sixteen lanes of a row group write
    // column 8 cg + j, lines a kilobyte apart, and would all meet in the same banks without it
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float r = largest<FMT>() / (TILES ? tile_top : cmax[j]);
        const uint32_t lo = pack4<FMT>(v[0][j] * r, v[1][j] * r, v[2][j] * r, v[3][j] * r);
        const uint32_t hi = pack4<FMT>(v[4][j] * r, v[5][j] * r, v[6][j] * r, v[7][j] * r);
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
