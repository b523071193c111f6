// Block-scaled 8-bit products with few rows of A (one token, or a few per expert): B is read once and is nearly all
// there is to read, so the kernel is bound by HBM, or by latency where B is small.
//
// A workgroup owns 16 columns of C (rows of B); its waves take the blocks of 128 contracted elements in turn and hold the
// operands in registers: the lanes of one load instruction cover 64 contiguous bytes of 16 rows, two instructions the
// whole 128-byte block, and nothing passes through LDS before the waves' partial sums do (in wave order: the same
// bits on every run).  Four blocks are in flight per wave: with eight waves 64 KB per CU, more than the 24 KB that
// a microsecond of latency at 6 TB/s takes.
#include "scaled_device.hpp"

namespace ctc {

using namespace scaled;

namespace {

struct Codes {
    v4i lo, hi;
};
__device__ __forceinline__ Codes load_codes(const uint8_t *row, int64_t k, int64_t k_end, bool whole)
{
    Codes c;
    if (whole) {
        __builtin_memcpy(&c.lo, row + k, 16);
        __builtin_memcpy(&c.hi, row + k + 64, 16);
    } else {
        c.lo = __builtin_bit_cast(v4i, load_chunk(row, k, k_end));
        c.hi = __builtin_bit_cast(v4i, load_chunk(row, k + 64, k_end));
    }
    return c;
}

// MT: row tiles of 16 in one pass; a group with more rows takes several passes over its part of B
template <int FA, bool BUNI, int MT, int NW> __global__ void __launch_bounds__(NW * 64) scaled_skinny_kernel(ScaledGemmParams p)
{
    constexpr int U = MT == 1 ? 4 : 2;  // blocks in flight
    __shared__ __attribute__((aligned(16))) float part[NW][MT * 256];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    const int64_t entry = blockIdx.x / (unsigned)p.nbn, n0 = (int64_t)(blockIdx.x % (unsigned)p.nbn) * 16;
    int64_t m_begin = 0, m_end = p.M;
    const uint8_t *A = p.a.q;
    const float *SA = p.a.scale;
    if (p.mode == kScaledRows) {
        m_begin = clamp_offset(p.offsets[entry], p.M);
        m_end = clamp_offset(p.offsets[entry + 1], p.M);
    } else {
        A += entry * p.a.batch;
        SA += entry * p.a.s_batch;
    }
    const int64_t n_lane = n0 + fr < p.N ? n0 + fr : p.N - 1;
    const uint8_t *b_row = p.b.q + entry * p.b.batch + n_lane * p.b.ld;
    const float *SB = p.b.scale + entry * p.b.s_batch;
    const float *sb_ptr[BUNI ? 1 : 4];
#pragma unroll
    for (int r = 0; r < (BUNI ? 1 : 4); ++r) {
        const int64_t n = BUNI ? n0 : n0 + fg * 4 + r;
        sb_ptr[r] = SB + ((n < p.N ? n : p.N - 1) >> p.b.shift) * p.b.s_row;
    }
    const int steps = (int)((p.K + kScaleBlock - 1) / kScaleBlock);
    const int64_t c_entry = p.mode == kScaledRows ? 0 : entry * p.c_batch;
    const bool vec = ((p.ldc | p.c_batch) & 3) == 0 && (reinterpret_cast<uintptr_t>(p.C) & (p.c_f32 ? 15 : 7)) == 0;

    for (int64_t m0 = m_begin; m0 < m_end; m0 += MT * 16) {
        const uint8_t *a_row[MT];
        const float *sa_ptr[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            int64_t m = m0 + i * 16 + fr;
            m = m < m_end ? m : m_end - 1;
            a_row[i] = A + m * p.a.ld;
            sa_ptr[i] = SA + (m >> p.a.shift) * p.a.s_row;
        }
        const int64_t rows = m_end - m0;
        v4f acc[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
        for (int s0 = wave; s0 < steps; s0 += NW * U) {
            Codes fb[U], fa[U][MT];
            float sb[U][BUNI ? 1 : 4], sa[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u * NW;
                if (s >= steps) break;
                const int64_t k = (int64_t)s * kScaleBlock + fg * 16;
                const bool whole = (int64_t)(s + 1) * kScaleBlock <= p.K;
                fb[u] = load_codes(b_row, k, p.K, whole);
#pragma unroll
                for (int r = 0; r < (BUNI ? 1 : 4); ++r) sb[u][r] = sb_ptr[r][(int64_t)s * p.b.s_blk];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (i > 0 && rows <= i * 16) break;
                    fa[u][i] = load_codes(a_row[i], k, p.K, whole);
                    sa[u][i] = sa_ptr[i][(int64_t)s * p.a.s_blk];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (s0 + u * NW >= steps) break;
                BlockOperand<0, false> ob[1];
                ob[0].set(fb[u].lo, fb[u].hi);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (i > 0 && rows <= i * 16) break;
                    BlockOperand<FA, false> oa;
                    oa.set(fa[u][i].lo, fa[u][i].hi);
                    v4f d[1];
                    block_sums<FA, false, 1>(ob, oa, d);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][r] = __builtin_fmaf(d[0][r], sa[u][i] * sb[u][BUNI ? 0 : r], acc[i][r]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) *reinterpret_cast<v4f *>(&part[wave][(i * 16 + fr) * 16 + fg * 4]) = acc[i];
        __syncthreads();
        // four consecutive columns of a row per thread
        for (int q = t; q < MT * 64; q += NW * 64) {
            const int64_t m = m0 + (q >> 2), n = n0 + (q & 3) * 4;
            v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) v += *reinterpret_cast<const v4f *>(&part[w][q * 4]);
            if (m < m_end && n < p.N) store4(p, c_entry + m * p.ldc + n, n, v, vec);
        }
        __syncthreads();
    }
}

template <int FA, bool BUNI, int MT> void launch_rows(const ScaledGemmParams &p, int waves, unsigned grid, hipStream_t stream)
{
    if (waves == 16) hipLaunchKernelGGL((scaled_skinny_kernel<FA, BUNI, MT, 16>), dim3(grid), dim3(1024), 0, stream, p);
    else if (waves == 8) hipLaunchKernelGGL((scaled_skinny_kernel<FA, BUNI, MT, 8>), dim3(grid), dim3(512), 0, stream, p);
    else hipLaunchKernelGGL((scaled_skinny_kernel<FA, BUNI, MT, 4>), dim3(grid), dim3(256), 0, stream, p);
}
template <int FA, bool BUNI> void launch_b(const ScaledGemmParams &p, int waves, unsigned grid, hipStream_t stream)
{
    const int64_t rows = p.mode == kScaledRows ? (p.M + p.batch - 1) / p.batch : p.M;
    if (rows <= 16) launch_rows<FA, BUNI, 1>(p, waves, grid, stream);
    else launch_rows<FA, BUNI, 2>(p, waves, grid, stream);
}

}  // namespace

hipError_t launch_scaled_skinny(const ScaledGemmParams &pp, const ScaledSchedule &s, hipStream_t stream)
{
    ScaledGemmParams p = pp;
    p.nbn = (int)((p.N + 15) / 16);
    const int64_t grid = (int64_t)p.nbn * p.batch;
    if (grid > 0x3fffff) return hipErrorInvalidValue;
    const bool uni = p.b.shift == 7;
    if (p.a.e5m2) {
        if (uni) launch_b<1, true>(p, s.waves, (unsigned)grid, stream);
        else launch_b<1, false>(p, s.waves, (unsigned)grid, stream);
    } else {
        if (uni) launch_b<0, true>(p, s.waves, (unsigned)grid, stream);
        else launch_b<0, false>(p, s.waves, (unsigned)grid, stream);
    }
    return hipGetLastError();
}

}  // namespace ctc
