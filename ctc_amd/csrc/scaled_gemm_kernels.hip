// Block-scaled 8-bit products on gfx950:
//   C(m, n) = alpha * sum_g sa(m, g) sb(n, g) * (sum over the 128 k of block g of A(m, k) B(n, k)) + beta * C(m, n)
// with one f32 scale per row (or 128-row tile) and block of 128 contracted elements.
//
// One v_mfma_f32_16x16x128_f8f6f4 is exactly one block of a 16 x 16 piece: it starts from zero, and its four results
// per lane are added to the f32 accumulators with one FMA each, times sa * sb.  That FMA is the price of scales that are
// no powers of two: 4 vector-ALU cycles per 64 products' sums against the matrix core's 8, so both pipes have to run
// side by side (two waves per SIMD).  The MFMA's first operand is B, so a lane holds four consecutive n of one m:
// one A scale per lane and 16 rows, and a B scale that is uniform where B carries 128 x 128 tiles.
#include "scaled_device.hpp"
#include "lds_dma.hpp"

namespace ctc {

using namespace scaled;

namespace {

__device__ __attribute__((aligned(16))) const uint8_t zero_chunk[16] = {};

// What a workgroup multiplies: rows [m0, m_end) x columns [n0, N) over the contracted [k_begin, k_end), written to C
struct Item {
    int64_t m0, m_end, n0, k_begin, k_end;
    int64_t entry;  // batch entry or group: selects B, and C where the result has one matrix per entry
    int chunk;      // split-K chunk
};

// Tile `id` of the groups' row tiles, group after group; returns false beyond the last one.  Every wave scans the offsets
// 64 groups at a time, so that no workgroup waits for another and nothing is prepared on the host.  Offsets outside
// [0, rows] count as the nearer end and a group that ends before it starts as empty: no access leaves the operands.
__device__ __forceinline__ bool find_group_tile(const int32_t *offsets, int groups, int64_t rows, int bm, int64_t id, int &group, int64_t &m0, int64_t &m_end)
{
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < groups; base += 64) {
        const int g = base + lane;
        int64_t lo = 0, hi = 0;
        if (g < groups) {
            lo = clamp_offset(offsets[g], rows);
            hi = clamp_offset(offsets[g + 1], rows);
        }
        int n = hi > lo ? (int)((hi - lo + bm - 1) / bm) : 0;
        int sum = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        const unsigned long long past = __ballot(sum > id);
        if (past) {
            const int l = __ffsll((long long)past) - 1;
            const int before = __shfl(sum - n, l);
            const int64_t glo = __shfl((int)lo, l), ghi = __shfl((int)hi, l);
            group = base + l;
            m0 = glo + (id - before) * bm;
            m_end = ghi;
            return true;
        }
        id -= __shfl(sum, 63);
    }
    return false;
}
__device__ __forceinline__ int64_t count_group_tiles(const int32_t *offsets, int groups, int64_t rows, int bm)
{
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int g = lane; g < groups; g += 64) {
        const int64_t lo = clamp_offset(offsets[g], rows), hi = clamp_offset(offsets[g + 1], rows);
        n += hi > lo ? (int)((hi - lo + bm - 1) / bm) : 0;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
    return n;
}

// XCD-contiguous runs of tile ids (workgroup i runs on XCD i % 8): neighbouring tiles share operand panels in one L2
__device__ __forceinline__ int64_t xcd_run(int64_t id, int64_t total)
{
    const int64_t q = total >> 3, r = total & 7, x = id & 7;
    return x * q + (x < r ? x : r) + (id >> 3);
}
// tiles in groups of 8 tile rows, row index fastest: a run of ids covers a compact block of C
__device__ __forceinline__ void grouped_order(int64_t id, int64_t nbm, int64_t nbn, int64_t &tm, int64_t &tn)
{
    const int64_t per = 8 * nbn, g = id / per, first = g * 8;
    const int64_t h = nbm - first < 8 ? nbm - first : 8;
    const int64_t in = id - g * per;
    tm = first + in % h;
    tn = in / h;
}

template <int BM, int BN> __device__ __forceinline__ bool find_item(const ScaledGemmParams &p, Item &it)
{
    int64_t id = blockIdx.x, tm, tn;
    it.chunk = 0;
    it.k_begin = 0;
    it.k_end = p.K;
    if (p.mode == kScaledRows) {
        const int64_t rows = count_group_tiles(p.offsets, p.batch, p.M, BM);
        const int64_t total = rows * p.nbn;
        if (id >= total) return false;
        grouped_order(xcd_run(id, total), rows, p.nbn, tm, tn);
        int g = 0;
        if (!find_group_tile(p.offsets, p.batch, p.M, BM, tm, g, it.m0, it.m_end)) return false;
        // one value for the whole workgroup: kept in scalar registers
        it.entry = __builtin_amdgcn_readfirstlane(g);
        it.m0 = __builtin_amdgcn_readfirstlane((int)it.m0);
        it.m_end = __builtin_amdgcn_readfirstlane((int)it.m_end);
        it.n0 = (int64_t)__builtin_amdgcn_readfirstlane((int)tn) * BN;
        return true;
    }
    const int64_t per_entry = (int64_t)p.nbm * p.nbn, total = per_entry * p.batch * p.split;
    id = xcd_run(id, total);
    it.entry = id / (per_entry * p.split);
    id -= it.entry * per_entry * p.split;
    it.chunk = (int)(id / per_entry);
    id -= it.chunk * per_entry;
    grouped_order(id, p.nbm, p.nbn, tm, tn);
    it.m0 = tm * BM;
    it.m_end = p.M;
    it.n0 = tn * BN;
    if (p.mode == kScaledContracted) {
        // groups start at whole blocks; an offset that does not is taken at the block it falls into (the last one may be the ragged end of K)
        int64_t lo = clamp_offset(p.offsets[it.entry], p.K), hi = clamp_offset(p.offsets[it.entry + 1], p.K);
        if (lo < p.K) lo &= ~(int64_t)(kScaleBlock - 1);
        if (hi < p.K) hi &= ~(int64_t)(kScaleBlock - 1);
        it.k_begin = lo;
        it.k_end = hi > lo ? hi : lo;
    } else if (p.split > 1) {
        it.k_begin = (int64_t)it.chunk * p.steps_per * kScaleBlock;
        const int64_t end = it.k_begin + (int64_t)p.steps_per * kScaleBlock;
        it.k_end = end < p.K ? end : p.K;
    }
    return true;
}

// BM x BN tile, WM x WN waves.  FA: A holds e5m2.  BUNI: B's scale is one per 128 x 128 tile, hence uniform in a wave.
// DMA: both operands 16-byte aligned with row pitches that are multiples of 16: their blocks go global -> LDS by DMA;
// otherwise every chunk passes through registers (byte-exact at any alignment).
//
// LDS, two stages of a block each: rows of 128 bytes, 16-byte chunk c of row r at c ^ (r / 2 & 7).  A fragment is the
// chunks g and g + 4 of row l % 16 (g = l / 16), for both operands alike, so that the k order inside the MFMA's block
// does not matter; with the XOR sixteen lanes that ds_read_b128 serves together fall on sixteen different 16-byte slots.
template <int FA, bool FAST, bool BUNI, int BM, int BN, int WM, int WN, bool DMA>
__global__ void __launch_bounds__(WM *WN * 64) scaled_gemm_kernel(ScaledGemmParams p)
{
    constexpr int T = WM * WN * 64;
    constexpr int WTM = BM / WM, WTN = BN / WN, MT = WTM / 16, NT = WTN / 16;
    constexpr int STAGE = (BM + BN) * 128;
    constexpr int NA = BM * 8 / T, NB = BN * 8 / T;  // chunks a thread stages
    static_assert(BM * 8 % T == 0 && BN * 8 % T == 0 && (!BUNI || (128 % WTN == 0 && BN % WTN == 0)), "tile");
    static_assert(T / 8 % 16 == 0, "a thread's rows are 16 or more apart: one swizzle term for all of them");
    __shared__ __attribute__((aligned(16))) uint8_t image[2][STAGE];
    __shared__ __attribute__((aligned(16))) float scales[2][BM + BN];

    Item it;
    if (!find_item<BM, BN>(p, it)) return;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int64_t a_entry = p.mode == kScaledDense ? it.entry : 0, b_entry = p.mode == kScaledContracted ? 0 : it.entry;
    const uint8_t *A = p.a.q + a_entry * p.a.batch, *B = p.b.q + b_entry * p.b.batch;
    const float *SA = p.a.scale + a_entry * p.a.s_batch, *SB = p.b.scale + b_entry * p.b.s_batch;

    // staging: thread t owns chunk slot t % 8 of rows t / 8 + i * T / 8; rows beyond the operand repeat its last one
    const int srow = t >> 3, slot = t & 7, schunk = slot ^ ((srow >> 1) & 7);
    int64_t a_off[NA], b_off[NB];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        int64_t r = it.m0 + srow + i * (T / 8);
        a_off[i] = (r < it.m_end ? r : it.m_end - 1) * p.a.ld;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        int64_t r = it.n0 + srow + i * (T / 8);
        b_off[i] = (r < p.N ? r : p.N - 1) * p.b.ld;
    }
    const int64_t steps = (it.k_end - it.k_begin + kScaleBlock - 1) / kScaleBlock;
    const int64_t blk0 = it.k_begin / kScaleBlock;

    auto stage = [&](int64_t s, int buf) {
        const int64_t k = it.k_begin + s * kScaleBlock + schunk * 16;
        const int64_t left = it.k_end - k;
        if constexpr (DMA) {
            const unsigned base = lds_dma::lds_addr(&image[buf][0]) + wave * 1024;
            const bool whole = left >= 16;
#pragma unroll
            for (int i = 0; i < NA; ++i) {
                const void *src = whole ? A + a_off[i] + k : zero_chunk;
                asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(base + i * (T * 16)) : "memory");
            }
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const void *src = whole ? B + b_off[i] + k : zero_chunk;
                asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(base + BM * 128 + i * (T * 16)) : "memory");
            }
        } else {
#pragma unroll
            for (int i = 0; i < NA; ++i)
                *reinterpret_cast<uint4 *>(&image[buf][(srow + i * (T / 8)) * 128 + slot * 16]) = load_chunk(A + a_off[i], k, it.k_end);
#pragma unroll
            for (int i = 0; i < NB; ++i)
                *reinterpret_cast<uint4 *>(&image[buf][BM * 128 + (srow + i * (T / 8)) * 128 + slot * 16]) = load_chunk(B + b_off[i], k, it.k_end);
        }
    };
    // behind the DMA's wait: the chunk that K ends inside of, byte by byte, by the lane whose transfer wrote zeros there
    auto mend_tail = [&](int64_t s, int buf) {
        if constexpr (DMA) {
            const int64_t k = it.k_begin + s * kScaleBlock + schunk * 16;
            const int64_t left = it.k_end - k;
            if (left > 0 && left < 16) {
#pragma unroll 1
                for (int i = 0; i < NA; ++i)
                    *reinterpret_cast<uint4 *>(&image[buf][(srow + i * (T / 8)) * 128 + slot * 16]) = load_chunk(A + a_off[i], k, it.k_end);
#pragma unroll 1
                for (int i = 0; i < NB; ++i)
                    *reinterpret_cast<uint4 *>(&image[buf][BM * 128 + (srow + i * (T / 8)) * 128 + slot * 16]) = load_chunk(B + b_off[i], k, it.k_end);
            }
        }
    };
    // scales: thread t owns entry t (+ T) of the tile's BM rows and BN columns
    constexpr int NS = (BM + BN + T - 1) / T;
    const float *s_ptr[NS];
    int64_t s_blk[NS];
    float s_val[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int e = t + i * T;
        if (e < BM) {
            int64_t r = it.m0 + e;
            r = r < it.m_end ? r : it.m_end - 1;
            s_ptr[i] = SA + (r >> p.a.shift) * p.a.s_row + blk0 * p.a.s_blk;
            s_blk[i] = p.a.s_blk;
        } else {
            int64_t r = it.n0 + e - BM;
            r = r < p.N ? r : p.N - 1;
            s_ptr[i] = SB + (r >> p.b.shift) * p.b.s_row + blk0 * p.b.s_blk;
            s_blk[i] = p.b.s_blk;
        }
    }
    auto scale_load = [&](int64_t s) {
#pragma unroll
        for (int i = 0; i < NS; ++i) s_val[i] = s_ptr[i][s * s_blk[i]];
    };
    auto scale_store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (NS * T == BM + BN || t + i * T < BM + BN) scales[buf][t + i * T] = s_val[i];
    };

    v4f acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

    if (steps > 0) {
        scale_load(0);
        stage(0, 0);
        scale_store(0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (steps == 1) mend_tail(0, 0);
        __syncthreads();
    }
    const int fr = lane & 15, fg = lane >> 4;
    // fragment addresses: row base + fr, chunks fg and fg + 4 under the row's swizzle (fr / 2 & 7: row bases are multiples of 16)
    const int sw = (fr >> 1) & 7;
    const int off0 = fr * 128 + ((fg ^ sw) << 4), off1 = fr * 128 + (((fg + 4) ^ sw) << 4);
    auto frag = [&](auto &f, const uint8_t *base) { f.set(*reinterpret_cast<const v4i *>(base + off0), *reinterpret_cast<const v4i *>(base + off1)); };
#pragma unroll 1
    for (int64_t s = 0; s < steps; ++s) {
        const int buf = (int)(s & 1);
        const bool more = s + 1 < steps;
        if (more) {
            scale_load(s + 1);
            stage(s + 1, buf ^ 1);
        }
        const uint8_t *ia = &image[buf][wm * WTM * 128], *ib = &image[buf][BM * 128 + wn * WTN * 128];
        const float *fs = scales[buf];
        BlockOperand<0, FAST> fb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) frag(fb[j], ib + j * 16 * 128);
        v4f sb[BUNI ? 1 : NT];
        if constexpr (BUNI) {
            sb[0][0] = fs[BM + wn * WTN];
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) sb[j] = *reinterpret_cast<const v4f *>(fs + BM + wn * WTN + j * 16 + fg * 4);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            BlockOperand<FA, FAST> fa;
            frag(fa, ia + i * 16 * 128);
            float sa = fs[wm * WTM + i * 16 + fr];
            if constexpr (BUNI) sa *= sb[0][0];
            v4f d[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j)
                d[j] = block_sums<FA, FAST>(fb[j], fa);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f = BUNI ? sa : sa * sb[BUNI ? 0 : j][r];
                    acc[i][j][r] = __builtin_fmaf(d[j][r], f, acc[i][j][r]);
                }
            }
        }
        if (more) {
            scale_store(buf ^ 1);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (s + 2 == steps) mend_tail(s + 1, buf ^ 1);
        }
        __syncthreads();
    }

    const int64_t n_base = it.n0 + wn * WTN + fg * 4;
    if (p.split > 1) {
        float *w = p.ws + ((int64_t)it.chunk * p.batch + it.entry) * p.M * p.N;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int64_t m = it.m0 + wm * WTM + i * 16 + fr;
            if (m >= it.m_end) continue;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int64_t n = n_base + j * 16;
                float *c = w + m * p.N + n;
                if ((p.N & 3) == 0 && n < p.N) *reinterpret_cast<v4f *>(c) = acc[i][j];
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < p.N) c[r] = acc[i][j][r];
            }
        }
        return;
    }
    const int64_t c_entry = p.mode == kScaledRows ? 0 : it.entry * p.c_batch;
    const bool vec = ((p.ldc | p.c_batch) & 3) == 0 && (reinterpret_cast<uintptr_t>(p.C) & (p.c_f32 ? 15 : 7)) == 0;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = it.m0 + wm * WTM + i * 16 + fr;
        if (m >= it.m_end) continue;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int64_t n = n_base + j * 16;
            if (n < p.N) store4(p, c_entry + m * p.ldc + n, n, acc[i][j], vec);
        }
    }
}

// Sums the chunks' partial results in the order of the chunks (the same on every run) and stores C.
__global__ void __launch_bounds__(256) scaled_split_sum_kernel(ScaledGemmParams p)
{
    const int64_t per = p.M * p.N, total = per * p.batch;
    const int64_t quads = (p.N + 3) >> 2, items = quads * p.M * p.batch;
    const bool vec = ((p.ldc | p.c_batch) & 3) == 0 && (reinterpret_cast<uintptr_t>(p.C) & (p.c_f32 ? 15 : 7)) == 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
        const int64_t n = (i % quads) * 4, rest = i / quads, m = rest % p.M, b = rest / p.M;
        const float *w = p.ws + b * per + m * p.N + n;
        v4f v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < p.split; ++s, w += total) {
            if ((p.N & 3) == 0) {
                v += *reinterpret_cast<const v4f *>(w);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < p.N) v[r] += w[r];
            }
        }
        store4(p, b * p.c_batch + m * p.ldc + n, n, v, vec);
    }
}

template <int FA, bool FAST, bool BUNI> hipError_t launch_tiles(const ScaledGemmParams &p, int kind, bool dma, unsigned grid, hipStream_t stream)
{
    if (FAST && kind == 2)
        hipLaunchKernelGGL((scaled_gemm_kernel<FA, FAST, BUNI, 256, 256, 2, 4, true>), dim3(grid), dim3(512), 0, stream, p);
    else if (dma)
        hipLaunchKernelGGL((scaled_gemm_kernel<FA, FAST, BUNI, 128, 128, 2, 2, true>), dim3(grid), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((scaled_gemm_kernel<FA, FAST, BUNI, 128, 128, 2, 2, false>), dim3(grid), dim3(256), 0, stream, p);
    return hipGetLastError();
}

bool dma_ready(const ScaledMatrix &m) { return ((reinterpret_cast<uintptr_t>(m.q) | (uintptr_t)m.ld | (uintptr_t)m.batch) & 15) == 0; }

}  // namespace

ScaledSchedule schedule_scaled(const ScaledGemmParams &p, int cus, size_t ws_limit)
{
    ScaledSchedule s;
    const int64_t rows = p.mode == kScaledRows ? (p.M + p.batch - 1) / p.batch : p.M;
    if (p.mode != kScaledContracted && rows <= 32) return s;
    const int64_t entries = p.mode == kScaledRows ? 1 : p.batch;
    const auto tiles = [&](int64_t b) {
        const int64_t nbm = (p.M + b - 1) / b + (p.mode == kScaledRows ? p.batch / 2 : 0);
        return nbm * ((p.N + b - 1) / b) * entries;
    };
    s.kind = !p.c_f32 && dma_ready(p.a) && dma_ready(p.b) && tiles(256) >= cus * 3 / 4 ? 2 : 1;
    if (s.kind == 1 && p.mode == kScaledDense && tiles(128) < cus) {
        const int64_t steps = (p.K + kScaleBlock - 1) / kScaleBlock;
        int64_t split = 2 * cus / tiles(128);
        if (split > steps / 4) split = steps / 4;
        const size_t one = (size_t)p.M * p.N * p.batch * 4;
        if (split > 1 && (size_t)split * one > ws_limit) split = (int64_t)(ws_limit / one);
        if (split > 1) {
            const int64_t per = (steps + split - 1) / split;
            s.split = (int)((steps + per - 1) / per);
            s.ws_bytes = s.split > 1 ? (size_t)s.split * one : 0;
        }
    }
    return s;
}

hipError_t launch_scaled_gemm(ScaledGemmParams p, const ScaledSchedule &s, hipStream_t stream)
{
    const int b = s.kind == 2 ? 256 : 128;
    p.nbm = (int)((p.M + b - 1) / b);
    p.nbn = (int)((p.N + b - 1) / b);
    p.split = s.split;
    const int64_t steps = (p.K + kScaleBlock - 1) / kScaleBlock;
    p.steps_per = (int)((steps + s.split - 1) / s.split);
    int64_t grid = (int64_t)p.nbm * p.nbn * p.batch * p.split;
    // row tiles of ragged groups: each group adds at most one partly filled tile
    if (p.mode == kScaledRows) grid = (p.M / b + (p.batch < p.M ? p.batch : p.M)) * (int64_t)p.nbn;
    if (grid > 0x7fffff) return hipErrorInvalidValue;
    const bool uni = p.b.shift == 7, dma = dma_ready(p.a) && dma_ready(p.b);
    const bool fast = !p.c_f32;  // an f32 result takes f32 sums (see block_sums)
    typedef hipError_t (*launcher)(const ScaledGemmParams &, int, bool, unsigned, hipStream_t);
    static const launcher table[2][2][2] = {{{launch_tiles<0, false, false>, launch_tiles<0, false, true>}, {launch_tiles<0, true, false>, launch_tiles<0, true, true>}},
                                            {{launch_tiles<1, false, false>, launch_tiles<1, false, true>}, {launch_tiles<1, true, false>, launch_tiles<1, true, true>}}};
    const hipError_t e = table[p.a.e5m2][fast][uni](p, s.kind, dma, (unsigned)grid, stream);
    if (e != hipSuccess || p.split == 1) return e;
    int64_t blocks = (((p.N + 3) >> 2) * p.M * p.batch + 255) / 256;
    if (blocks > 256 * 16) blocks = 256 * 16;
    hipLaunchKernelGGL(scaled_split_sum_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace ctc
