// Block-scaled 8-bit products with few rows of A (one token, or a few per expert): B is read once and is nearly all
// there is to read, so the kernel is bound by HBM, or by latency where B is small.
//
// A workgroup owns 16 columns of C (rows of B); its waves take the blocks of 128 contracted elements in turn, two or four
// in flight each, hold the operands in registers (turned through LDS of the wave's own: see Codes) and meet once, in the
// sum of their partial results, in wave order: the same bits on every run.  A wave that met a product of scales outside the normal
// numbers takes its blocks once more (see ScalePair); looking costs nothing up to 16 rows and 4 % at 32 x 8192 x 8192 (16.6 -> 17.5 us).  1 x 131072 x 8192: 163 us, 6.6 TB/s; 16 rows x 131072 x
// 4096: 114 us, 4.7 TB/s (A is as many bytes as B for every workgroup then, out of the L2).
#include "scaled_device.hpp"

namespace ctc {

using namespace scaled;

namespace {

// MT: row tiles of 16 in one pass; a group with more rows takes several passes over its part of B.  U: blocks in flight a wave
template <int FA, bool BUNI, int MT, int NW, int U> __global__ void __launch_bounds__(NW * 64) scaled_skinny_kernel(ScaledGemmParams p)
{
    constexpr int S = BUNI ? 1 : 4;
    __shared__ __attribute__((aligned(16))) float part[NW][MT * 256];
    __shared__ __attribute__((aligned(16))) uint8_t scratch[NW][2048];
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
    const uint8_t *B = p.b.q + entry * p.b.batch;
    const int lr = lane >> 2, lc = (lane & 3) * 16;  // the row and the bytes that the lane loads
    const uint8_t *b_row = B + min64(n0 + lr, p.N - 1) * p.b.ld + lc;
    const float *SB = p.b.scale + entry * p.b.s_batch;
    const float *sb_ptr[S];
#pragma unroll
    for (int r = 0; r < S; ++r) {
        const int64_t n = BUNI ? n0 : n0 + fg * 4 + r;
        sb_ptr[r] = SB + ((n < p.N ? n : p.N - 1) >> p.b.shift) * p.b.s_row;
    }
    const int whole = (int)(p.K / kScaleBlock);
    const int64_t c_entry = p.mode == kScaledRows ? 0 : entry * p.c_batch;
    const bool vec = ((p.ldc | p.c_batch) & 3) == 0 && (reinterpret_cast<uintptr_t>(p.C) & (p.c_f32 ? 15 : 7)) == 0;

    for (int64_t m0 = m_begin; m0 < m_end; m0 += MT * 16) {
        const uint8_t *a_row[MT];
        const float *sa_ptr[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            a_row[i] = A + min64(m0 + i * 16 + lr, m_end - 1) * p.a.ld + lc;
            sa_ptr[i] = SA + (min64(m0 + i * 16 + fr, m_end - 1) >> p.a.shift) * p.a.s_row;
        }
        v4f acc[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
        bool odd = false;  // a product of scales is no normal number
        // `mine` chooses and does not branch: loads would sink into the branches, one wait each
        auto multiply = [&](const Codes &cb, const Codes(&ca)[MT], const float(&sb)[S], const float(&sa)[MT], bool mine) {
            BlockOperand<0, false> ob[1];
            ob[0].set(cb.lo, cb.hi);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                BlockOperand<FA, false> oa;
                oa.set(ca[i].lo, ca[i].hi);
                v4f d[1];
                block_sums<FA, false, 1>(ob, oa, d);
                float f[S];
#pragma unroll
                for (int r = 0; r < S; ++r) {
                    f[r] = sa[i] * sb[r];
                    odd |= !__builtin_isnormal(f[r]);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][r] = mine ? __builtin_fmaf(d[0][r], f[BUNI ? 0 : r], acc[i][r]) : acc[i][r];
            }
        };
        for (int s0 = wave; s0 < whole; s0 += NW * U) {
            Codes cb[U], ca[U][MT];
            float sb[U][S], sa[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) {  // beyond the last block: that one again, not added
                const int64_t s = s0 + u * NW < whole ? s0 + u * NW : whole - 1;
                cb[u] = load_codes(b_row, s * kScaleBlock);
#pragma unroll
                for (int i = 0; i < MT; ++i) ca[u][i] = load_codes(a_row[i], s * kScaleBlock);
#pragma unroll
                for (int r = 0; r < S; ++r) sb[u][r] = sb_ptr[r][s * p.b.s_blk];
#pragma unroll
                for (int i = 0; i < MT; ++i) sa[u][i] = sa_ptr[i][s * p.a.s_blk];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                Codes tb = turn(cb[u], scratch[wave], lane), ta[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) ta[i] = turn(ca[u][i], scratch[wave], lane);
                multiply(tb, ta, sb[u], sa[u], s0 + u * NW < whole);
            }
        }
        // The block that K ends in; and where a product of scales was no normal number all of the wave's blocks once more: with the scales'
        // exponents apart from their product
        const bool again = __ballot(odd) != 0;
        if (__builtin_expect(again, 0)) {
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
        }
        const int blocks = (int)((p.K + kScaleBlock - 1) / kScaleBlock);
#pragma unroll 1
        for (int s = again ? wave : wave == whole % NW ? whole : blocks; s < blocks; s += NW) {
            int l = lane;
            asm volatile("" : "+v"(l));  // addresses made here: held in front of the loop they cost the one above its registers
            const int row = l & 15, col = (l >> 4) * 16;
            const int64_t k = (int64_t)s * kScaleBlock, k_end = p.K - col;
            BlockOperand<0, false> ob[1];
            const Codes cb = load_last_codes(B + min64(n0 + row, p.N - 1) * p.b.ld + col, k, k_end, p.K >= 16);
            ob[0].set(cb.lo, cb.hi);
            float sb[S];
#pragma unroll
            for (int r = 0; r < S; ++r) sb[r] = sb_ptr[r][s * p.b.s_blk];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const Codes ca = load_last_codes(A + min64(m0 + i * 16 + row, m_end - 1) * p.a.ld + col, k, k_end, p.K >= 16);
                const float sa = sa_ptr[i][s * p.a.s_blk];
                BlockOperand<FA, false> oa;
                oa.set(ca.lo, ca.hi);
                v4f d[1];
                block_sums<FA, false, 1>(ob, oa, d);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][r] = add_scaled(d[0][r], scale_pair(sa, sb[BUNI ? 0 : r]), acc[i][r]);
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

// Waves of a workgroup: two where there are workgroups enough and K is short (a wave then has eight blocks or more of its
// own, and less of its life goes into starting and into the sum over the waves: 64 groups, 96 rows spread over them, 2048 x 2048 weights
// 66 -> 38 us, 4096 x 1024 ones 112 -> 36), eight where there are few workgroups or K is long (1 x 4096 x 8192: 10.5 us against 14.0,
// 1 x 131072 x 8192: 163 against 184).
struct SkinnyForm {
    bool two_waves, two_row_tiles;
};
SkinnyForm choose_form(const ScaledGemmParams &p)
{
    const int64_t rows = p.mode == kScaledRows ? (p.M + p.batch - 1) / p.batch : p.M;
    const int64_t grid = (p.N + 15) / 16 * p.batch, blocks = p.K / kScaleBlock;
    return {(grid >= 1024 && blocks <= 32) || (grid >= 512 && blocks <= 16), rows > 16};
}
template <int FA, bool BUNI> void launch_b(const ScaledGemmParams &p, SkinnyForm form, unsigned grid, hipStream_t stream)
{
    const bool two = form.two_waves;
    if (form.two_row_tiles) {
        if (two) hipLaunchKernelGGL((scaled_skinny_kernel<FA, BUNI, 2, 2, 2>), dim3(grid), dim3(128), 0, stream, p);
        else hipLaunchKernelGGL((scaled_skinny_kernel<FA, BUNI, 2, 8, 2>), dim3(grid), dim3(512), 0, stream, p);
    } else {
        if (two) hipLaunchKernelGGL((scaled_skinny_kernel<FA, BUNI, 1, 2, 2>), dim3(grid), dim3(128), 0, stream, p);
        else hipLaunchKernelGGL((scaled_skinny_kernel<FA, BUNI, 1, 8, 4>), dim3(grid), dim3(512), 0, stream, p);
    }
}

// one launch
hipError_t launch_part(ScaledGemmParams p, SkinnyForm form, hipStream_t stream)
{
    p.nbn = (int)((p.N + 15) / 16);
    const unsigned grid = (unsigned)p.nbn * (unsigned)p.batch;
    const bool uni = p.b.shift == 7;
    if (p.a.e5m2) {
        if (uni) launch_b<1, true>(p, form, grid, stream);
        else launch_b<1, false>(p, form, grid, stream);
    } else {
        if (uni) launch_b<0, true>(p, form, grid, stream);
        else launch_b<0, false>(p, form, grid, stream);
    }
    return hipGetLastError();
}

}  // namespace

// A launch holds fewer than 2^32 threads, of which a workgroup has up to 512: entries beyond 2^22 workgroups, and columns beyond as many,
// take launches of their own, all of one form.
hipError_t launch_scaled_skinny(const ScaledGemmParams &p, hipStream_t stream)
{
    constexpr int64_t kMostGroups = 0x3fffff, kMostColumns = kMostGroups * 16 / kScaleBlock * kScaleBlock;  // whole tiles of B's scales
    const SkinnyForm form = choose_form(p);
    const int64_t size = p.c_f32 ? 4 : 2;
    for (int64_t n0 = 0; n0 < p.N; n0 += kMostColumns) {
        ScaledGemmParams columns = p;
        columns.N = p.N - n0 < kMostColumns ? p.N - n0 : kMostColumns;
        columns.b.q += n0 * p.b.ld;
        columns.b.scale += (n0 >> p.b.shift) * p.b.s_row;
        columns.C = static_cast<char *>(p.C) + n0 * size;
        const int64_t entries = kMostGroups / ((columns.N + 15) / 16);
        for (int64_t e = 0; e < p.batch; e += entries) {
            ScaledGemmParams part = columns;
            part.batch = (int)(p.batch - e < entries ? p.batch - e : entries);
            part.b.q += e * p.b.batch;
            part.b.scale += e * p.b.s_batch;
            if (p.mode == kScaledRows) {
                part.offsets += e;
            } else {
                part.a.q += e * p.a.batch;
                part.a.scale += e * p.a.s_batch;
                part.C = static_cast<char *>(columns.C) + e * p.c_batch * size;
            }
            const hipError_t err = launch_part(part, form, stream);
            if (err != hipSuccess) return err;
        }
    }
    return hipSuccess;
}

}  // namespace ctc
