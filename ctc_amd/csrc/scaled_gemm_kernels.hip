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

// What a workgroup multiplies: rows [m0, m_end) x columns [n0, N) over the contracted [k_begin, k_end), written to C
struct Item {
    int64_t m0, m_end, n0, k_begin, k_end;
    int64_t entry;  // batch entry or group: selects B, and C where the result has one matrix per entry
    int chunk;      // split-K chunk
};

// Row tiles of a group of `rows` rows: all of them, those of more than BM / 2 rows ("full"), or the one that is not, if there is one
enum Which { kAll, kFull, kLight };
template <int BM, Which W> __device__ __forceinline__ int row_tiles(int64_t rows)
{
    if (rows <= 0) return 0;
    const int all = (int)((rows + BM - 1) / BM);
    const int light = (rows - 1) % BM < BM / 2;
    return W == kAll ? all : W == kLight ? light : all - light;
}

// Tile `id` of the groups' row tiles, group after group; returns false beyond the last one.  Every wave scans the offsets
// 64 groups at a time, so that no workgroup waits for another and nothing is prepared on the host.  Offsets outside
// [0, rows] count as the nearer end and a group that ends before it starts as empty: no access leaves the operands.
template <int BM, Which W> __device__ __forceinline__ bool find_group_tile(const int32_t *offsets, int groups, int64_t rows, int64_t id, int &group, int64_t &m0, int64_t &m_end)
{
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < groups; base += 64) {
        const int g = base + lane;
        int64_t lo = 0, hi = 0;
        if (g < groups) {
            lo = clamp_offset(offsets[g], rows);
            hi = clamp_offset(offsets[g + 1], rows);
        }
        const int n = row_tiles<BM, W>(hi - lo);
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
            m0 = glo + (W == kLight ? (ghi - glo - 1) / BM : id - before) * BM;
            m_end = ghi;
            return true;
        }
        id -= __shfl(sum, 63);
    }
    return false;
}
template <int BM, Which W> __device__ __forceinline__ uint32_t count_group_tiles(const int32_t *offsets, int groups, int64_t rows)
{
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int g = lane; g < groups; g += 64) {
        const int64_t lo = clamp_offset(offsets[g], rows), hi = clamp_offset(offsets[g + 1], rows);
        n += row_tiles<BM, W>(hi - lo);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
    return (uint32_t)__builtin_amdgcn_readfirstlane(n);
}

// XCD-contiguous runs of tile ids (workgroup i runs on XCD i % 8): neighbouring tiles share operand panels in one L2.
// Ids are below 2^23: 32-bit divisions, a fraction of the 64-bit ones' instructions.
__device__ __forceinline__ uint32_t xcd_run(uint32_t id, uint32_t total)
{
    const uint32_t q = total >> 3, r = total & 7, x = id & 7;
    return x * q + (x < r ? x : r) + (id >> 3);
}
// tiles in groups of 8 tile rows, row index fastest: a run of ids covers a compact block of C
__device__ __forceinline__ void grouped_order(uint32_t id, uint32_t nbm, uint32_t nbn, uint32_t &tm, uint32_t &tn)
{
    const uint32_t per = 8 * nbn, g = id / per, first = g * 8;
    const uint32_t h = nbm - first < 8 ? nbm - first : 8;
    const uint32_t in = id - g * per;
    tn = in / h;
    tm = first + in - tn * h;
}

// a value that is the same in all lanes, into scalar registers
__device__ __forceinline__ int64_t uniform(int64_t v)
{
    const int lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}

// The group that is `place` in the order of falling lengths (ties by index); beyond 64 groups, a wave's lanes, the order as it is
__device__ __forceinline__ int longest_first(const int32_t *offsets, int groups, int64_t k, int place)
{
    if (groups > 64) return place;
    const int lane = threadIdx.x & 63;
    int len = -1;
    if (lane < groups) len = (int)(clamp_offset(offsets[lane + 1], k) - clamp_offset(offsets[lane], k));
    int rank = 0;
    for (int j = 0; j < groups; ++j) {
        const int other = __builtin_amdgcn_readlane(len, j);
        rank += other > len || (other == len && j < lane);
    }
    return __ffsll((long long)__ballot(lane < groups && rank == place)) - 1;
}

// The order of the large tile's kernel where it tells full tiles from light ones (at most BM / 2 rows, two thirds of a full one's
// time): the full ones, then, if the last round of full tiles would keep less than half of the compute units busy, its tiles in halves
// (4096 x 5120 x 4096, 320 tiles: 125 -> 106 us), then the light ones (4200 x 4096 x 4096: 123 -> 103).
struct Place {
    uint32_t id;
    int kind;  // -1 nothing, 0 full, 1 upper half, 2 lower half, 3 light
};
__device__ __forceinline__ Place place_of(uint32_t id, uint32_t full, uint32_t light, uint32_t cus)
{
    uint32_t rest = full % cus;
    if (2 * rest + light > cus) rest = 0;
    const uint32_t whole = full - rest;
    if (id < whole) return {xcd_run(id, whole), 0};
    id -= whole;
    if (id < 2 * rest) {
        id = xcd_run(id, 2 * rest);
        return {whole + (id >> 1), 1 + (int)(id & 1)};
    }
    id -= 2 * rest;
    if (id < light) return {xcd_run(id, light), 3};
    return {0, -1};
}

template <int BM, int BN, bool LIGHT> __device__ __forceinline__ bool find_item(const ScaledGemmParams &p, Item &it)
{
    uint32_t id = blockIdx.x, tm, tn;
    it.chunk = 0;
    it.k_begin = 0;
    it.k_end = p.K;
    if constexpr (LIGHT) {
        const bool ragged = p.mode == kScaledRows;
        const uint32_t nbn = (uint32_t)p.nbn, entries = ragged ? 1 : (uint32_t)p.batch;
        uint32_t full_rows, light_rows;
        if (ragged) {
            full_rows = count_group_tiles<BM, kFull>(p.offsets, p.batch, p.M);
            light_rows = count_group_tiles<BM, kLight>(p.offsets, p.batch, p.M);
        } else {
            full_rows = row_tiles<BM, kFull>(p.M);
            light_rows = row_tiles<BM, kLight>(p.M);
        }
        const Place at = place_of(id, full_rows * nbn * entries, light_rows * nbn * entries, (uint32_t)p.cus);
        if (at.kind < 0) return false;
        const uint32_t rows = at.kind == 3 ? light_rows : full_rows, entry = at.id / (rows * nbn);
        grouped_order(at.id - entry * (rows * nbn), rows, nbn, tm, tn);
        it.n0 = (int64_t)tn * BN;
        if (ragged) {
            int g = 0;
            const bool found = at.kind == 3 ? find_group_tile<BM, kLight>(p.offsets, p.batch, p.M, tm, g, it.m0, it.m_end)
                                            : find_group_tile<BM, kFull>(p.offsets, p.batch, p.M, tm, g, it.m0, it.m_end);
            if (!found) return false;
            it.entry = g;
        } else {
            it.entry = entry;
            it.m0 = (int64_t)(at.kind == 3 ? full_rows : tm) * BM;
            it.m_end = p.M;
        }
        it.m_end = min64(it.m_end, it.m0 + BM);
        if (at.kind == 1) it.m_end = it.m0 + BM / 2;  // (a full tile has rows beyond)
        if (at.kind == 2) it.m0 += BM / 2;
        return true;
    }
    if (p.mode == kScaledRows) {
        const uint32_t rows = count_group_tiles<BM, kAll>(p.offsets, p.batch, p.M), total = rows * (uint32_t)p.nbn;
        if (id >= total) return false;
        grouped_order(xcd_run(id, total), rows, p.nbn, tm, tn);
        int g = 0;
        if (!find_group_tile<BM, kAll>(p.offsets, p.batch, p.M, tm, g, it.m0, it.m_end)) return false;
        it.entry = g;
        it.n0 = (int64_t)tn * BN;
        return true;
    }
    const uint32_t per_entry = (uint32_t)p.nbm * (uint32_t)p.nbn, per = per_entry * (uint32_t)p.split;
    // Groups of the contracted index differ in length: each is spread over all XCDs, and the longest come first.  Entries of a
    // batch are equal and stay together.
    const bool spread = p.mode == kScaledContracted;
    if (!spread) id = xcd_run(id, per * (uint32_t)p.batch);
    const uint32_t entry = id / per;
    id -= entry * per;
    if (spread) id = xcd_run(id, per);
    const uint32_t chunk = id / per_entry;
    id -= chunk * per_entry;
    it.entry = spread ? longest_first(p.offsets, p.batch, p.K, (int)entry) : (int)entry;
    it.chunk = (int)chunk;
    grouped_order(id, p.nbm, p.nbn, tm, tn);
    it.n0 = (int64_t)tn * BN;
    it.m0 = (int64_t)tm * BM;
    it.m_end = p.M;
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

__device__ __forceinline__ void store_partial(float *w, int64_t left, v4f v, bool vec)
{
    if (vec) {
        *reinterpret_cast<v4f *>(w) = v;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (r < left) w[r] = v[r];
}

// BM x BN tile, WM x WN waves.  FA: A holds e5m2.  FAST: see BlockOperand.  BUNI: B's scale is one per 128 x 128 tile, hence
// uniform in a wave.  DMA: both operands 16-byte aligned with row pitches that are multiples of 16: their blocks go
// global -> LDS by DMA; otherwise they pass through registers, requested a block ahead (byte-exact at any alignment).
//
// LDS, two stages (light tiles, and workgroups alone on a CU: three) of a block each: rows of 128 bytes, 16-byte chunk c of row r at c ^ (r / 2 & 7).  A fragment is the
// chunks g and g + 4 of row l % 16 (g = l / 16), for both operands alike, so that the k order inside the MFMA's block
// does not matter; with the XOR sixteen lanes that ds_read_b128 serves together fall on sixteen different 16-byte slots.
//
// A wave walks its row tiles with one tile's results in hand while the next one's MFMAs run: fragment i + 1 is
// requested, tile i multiplied, tile i - 1 scaled and added.  The order is pinned (sched_barrier): left alone, the
// compiler requests every fragment first and spills.
template <int FA, bool FAST, bool BUNI, int BM, int BN, int WM, int WN, bool DMA, int STAGES>
__device__ __forceinline__ void multiply_tile(const ScaledGemmParams &p, const Item &it, uint8_t *image, float *scales, int *again)
{
    constexpr int T = WM * WN * 64;
    constexpr int WTM = BM / WM, WTN = BN / WN, MT = WTM / 16, NT = WTN / 16;
    constexpr int STAGE = (BM + BN) * 128;
    constexpr int NA = BM * 8 / T, NB = BN * 8 / T;  // chunks a thread stages
    static_assert(BM * 8 % T == 0 && BN * 8 % T == 0 && (!BUNI || (128 % WTN == 0 && BN % WTN == 0)), "tile");
    static_assert(T / 8 % 16 == 0, "a thread's rows are 16 or more apart: one swizzle term for all of them");
    static_assert(T >= BM + BN && BM % 64 == 0 && BN % 64 == 0, "a thread loads one scale a step, a wave those of one operand");
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int64_t a_entry = p.mode == kScaledDense ? it.entry : 0, b_entry = p.mode == kScaledContracted ? 0 : it.entry;
    const int64_t blk0 = it.k_begin / kScaleBlock;

    // staging: thread t owns chunk slot t % 8 of rows t / 8 + i * T / 8; rows beyond the operand repeat its last one
    const int srow = t >> 3, slot = t & 7, schunk = slot ^ ((srow >> 1) & 7);
    const uint8_t *A = p.a.q + a_entry * p.a.batch + it.m0 * p.a.ld + it.k_begin;
    const uint8_t *B = p.b.q + b_entry * p.b.batch + it.n0 * p.b.ld + it.k_begin;
    uint32_t a_off[NA], b_off[NB];  // from the tile's corner: at most 255 rows of at most 2^22 bytes where DMA is set
    const int a_last = (int)((it.m_end - it.m0 < BM ? it.m_end - it.m0 : BM) - 1), b_last = (int)((p.N - it.n0 < BN ? p.N - it.n0 : BN) - 1);
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        a_off[i] = (uint32_t)min(srow + i * (T / 8), a_last) * (uint32_t)p.a.ld + schunk * 16;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        b_off[i] = (uint32_t)min(srow + i * (T / 8), b_last) * (uint32_t)p.b.ld + schunk * 16;
    }
    const unsigned lds0 = lds_dma::lds_addr(image) + wave * 1024;
    const int64_t k_len = it.k_end - it.k_begin;

    v4i held[DMA ? 1 : NA + NB];
    // requests the whole block s
    auto stage = [&](int64_t s, int buf) {
        if constexpr (DMA) {
            const unsigned base = lds0 + buf * STAGE;
#pragma unroll
            for (int i = 0; i < NA; ++i) lds_dma::dma16_spaced(A + s * kScaleBlock, a_off[i], base + i * (T * 16));
#pragma unroll
            for (int i = 0; i < NB; ++i) lds_dma::dma16_spaced(B + s * kScaleBlock, b_off[i], base + BM * 128 + i * (T * 16));
        } else {
            int row = srow;
            asm volatile("" : "+v"(row));  // each row's address anew: eight of them held through the loop spill
            const int64_t k = s * kScaleBlock + schunk * 16;
#pragma unroll
            for (int i = 0; i < NA; ++i) held[i] = load16(A + (int64_t)min(row + i * (T / 8), a_last) * p.a.ld + k);
#pragma unroll
            for (int i = 0; i < NB; ++i) held[NA + i] = load16(B + (int64_t)min(row + i * (T / 8), b_last) * p.b.ld + k);
        }
    };
    // without DMA: the block that stage() requested, into LDS
    auto put = [&](int buf) {
        uint8_t *to = image + buf * STAGE + srow * 128 + slot * 16;
#pragma unroll
        for (int i = 0; i < NA; ++i) *reinterpret_cast<v4i *>(to + i * (T * 16)) = held[i];
#pragma unroll
        for (int i = 0; i < NB; ++i) *reinterpret_cast<v4i *>(to + BM * 128 + i * (T * 16)) = held[NA + i];
    };
    // block s is in LDS when this has run in every wave
    auto land = [&](int buf) {
        if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else put(buf);
    };
    // block s through registers, chunk by chunk, zeros beyond the end; any alignment
    auto put_chunks = [&](int64_t s, int buf) {
        uint8_t *to = image + buf * STAGE + srow * 128 + slot * 16;
        const int64_t k = s * kScaleBlock + schunk * 16;
        const bool long_row = it.k_end >= 16;
#pragma unroll
        for (int i = 0; i < NA; ++i)
            *reinterpret_cast<uint4 *>(to + i * (T * 16)) = load_chunk(A + (int64_t)min(srow + i * (T / 8), a_last) * p.a.ld, k, k_len, long_row);
#pragma unroll
        for (int i = 0; i < NB; ++i)
            *reinterpret_cast<uint4 *>(to + BM * 128 + i * (T * 16)) = load_chunk(B + (int64_t)min(srow + i * (T / 8), b_last) * p.b.ld, k, k_len, long_row);
    };
    const int64_t whole = k_len / kScaleBlock;  // blocks in front of the one K ends in, if it ends in one
    // scales: thread t owns entry t of the tile's BM rows and BN columns
    const bool a_scale = wave < BM / 64, has_scale = T == BM + BN || wave < (BM + BN) / 64;
    const float *s_ptr;
    int64_t s_step;
    if (a_scale) {
        s_ptr = p.a.scale + a_entry * p.a.s_batch + ((it.m0 + min(t, a_last)) >> p.a.shift) * p.a.s_row + blk0 * p.a.s_blk;
        s_step = p.a.s_blk;
    } else {
        s_ptr = p.b.scale + b_entry * p.b.s_batch + ((it.n0 + min(t - BM, b_last)) >> p.b.shift) * p.b.s_row + blk0 * p.b.s_blk;
        s_step = p.b.s_blk;
    }

    v4f acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

    // a wave whose rows all lie behind the last one only stages
    const bool active = it.m0 + wm * WTM < it.m_end;
    const int fr = lane & 15, fg = lane >> 4;
    // fragment addresses: row base + fr, chunks fg and fg + 4 under the row's swizzle (fr / 2 & 7: row bases are multiples of 16)
    const int sw = (fr >> 1) & 7;
    const int off0 = fr * 128 + ((fg ^ sw) << 4), off1 = fr * 128 + (((fg + 4) ^ sw) << 4);
    // Scales of 2^-63 to 2^64 multiply to normal numbers.  A thread looks at the one it stages (`odd`: the lanes of the wave whose scale is
    // another); then this, on the block in stage `buf`: does a product of one of them leave the normal numbers where it matters?  It does
    // not if the scale or, under a small one, all codes are zeros: a masked row, weights that are not used.
    const auto outside = [](float f) { return (__float_as_uint(f) & 0x7fffffffu) - (64u << 23) >= (127u << 23); };
    auto matters = [&](int buf) {
        auto counts = [&](int line, float f) {  // f: the scale's magnitude
            if (f == 0.f) return false;
            if (!(f < 0x1p-63f)) return true;
            const v4i *q = reinterpret_cast<const v4i *>(image + buf * STAGE + line * 128);
            int any = 0;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) any |= q[c][0] | q[c][1] | q[c][2] | q[c][3];
            return (any & 0x7f7f7f7f) != 0;
        };
        const float *fs = scales + buf * (BM + BN);
        const float f = fabsf(fs[t]);
        const bool mine = outside(f) && counts(t, f);
        if (__ballot(mine) == 0) return false;
        if (__ballot(mine && !(f < INFINITY)) != 0) return true;
        // the smallest and the largest scale: of mine, and of the other side
        float lo = mine ? f : INFINITY, hi = mine ? f : 0.f, other_lo = INFINITY, other_hi = 0.f;
#pragma unroll 1
        for (int l = (a_scale ? BM : 0) + lane; l < (a_scale ? BM + BN : BM); l += 64) {
            const float o = fabsf(fs[l]);
            if (counts(l, o)) other_lo = fminf(other_lo, o), other_hi = fmaxf(other_hi, o);
        }
#pragma unroll 1
        for (int d = 1; d < 64; d <<= 1) {
            lo = fminf(lo, __shfl_xor(lo, d));
            hi = fmaxf(hi, __shfl_xor(hi, d));
            other_lo = fminf(other_lo, __shfl_xor(other_lo, d));
            other_hi = fmaxf(other_hi, __shfl_xor(other_hi, d));
        }
        return __ballot(other_hi > 0.f && !(__builtin_isnormal(lo * other_lo) && __builtin_isnormal(hi * other_hi))) != 0;
    };
    // multiplies the block in stage `buf`
    auto multiply = [&](int buf) {
        const uint8_t *stage_base = image + buf * STAGE;
        const uint8_t *ia0 = stage_base + wm * WTM * 128 + off0, *ia1 = stage_base + wm * WTM * 128 + off1;
        const uint8_t *ib0 = stage_base + (BM + wn * WTN) * 128 + off0, *ib1 = stage_base + (BM + wn * WTN) * 128 + off1;
        const float *fs = scales + buf * (BM + BN);
        BlockOperand<0, FAST> fb[NT];
        BlockOperand<FA, FAST> fa[2];
        fa[0].set(*reinterpret_cast<const v4i *>(ia0), *reinterpret_cast<const v4i *>(ia1));
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[j].set(*reinterpret_cast<const v4i *>(ib0 + j * 2048), *reinterpret_cast<const v4i *>(ib1 + j * 2048));
        v4f sb[BUNI ? 1 : NT];
        if constexpr (BUNI) {
            sb[0][0] = fs[BM + wn * WTN];
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) sb[j] = *reinterpret_cast<const v4f *>(fs + BM + wn * WTN + j * 16 + fg * 4);
        }
        float sa[MT];
        sa[0] = fs[wm * WTM + fr];
        v4f d[2][NT];
        auto add = [&](int i, const v4f(&v)[NT], float f) {
            if constexpr (BUNI) f *= sb[0][0];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(v[j][r], BUNI ? f : f * sb[BUNI ? 0 : j][r], acc[i][j][r]);
            // here and not where the sums are next used: the compiler would move the additions behind the whole block's MFMAs,
            // with every tile's results live until then
#pragma unroll
            for (int j = 0; j < NT; ++j) asm volatile("" : "+v"(acc[i][j]));
        };
        if constexpr (!FAST) __builtin_amdgcn_s_setprio(1);  // (4 % here, nothing for the 8-bit form)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if (i + 1 < MT) {
                fa[(i + 1) & 1].set(*reinterpret_cast<const v4i *>(ia0 + (i + 1) * 2048), *reinterpret_cast<const v4i *>(ia1 + (i + 1) * 2048));
                sa[i + 1] = fs[wm * WTM + (i + 1) * 16 + fr];
            }
            block_sums<FA, FAST, NT>(fb, fa[i & 1], d[i & 1]);
            if (i > 0) add(i - 1, d[(i - 1) & 1], sa[i - 1]);
            // one MFMA, then additions: a wave that waits for the matrix core has work, and the core always a request
#pragma unroll
            for (int j = 0; j < (FAST ? NT : 4 * NT); ++j) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, FAST ? (BUNI ? 5 : 8) : (BUNI ? 2 : 3), 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!FAST) __builtin_amdgcn_s_setprio(0);
        add(MT - 1, d[(MT - 1) & 1], sa[MT - 1]);
    };
    // multiplies the block in stage `buf` with the scales' exponents apart from their product (see ScalePair), one 16 x 16 piece after the other
    auto multiply_apart = [&](int buf) {
        const float *fs = scales + buf * (BM + BN);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint8_t *ia = image + buf * STAGE + (wm * WTM + i * 16) * 128, *ib = image + buf * STAGE + (BM + wn * WTN + j * 16) * 128;
                BlockOperand<FA, FAST> a;
                BlockOperand<0, FAST> b[1];
                a.set(*reinterpret_cast<const v4i *>(ia + off0), *reinterpret_cast<const v4i *>(ia + off1));
                b[0].set(*reinterpret_cast<const v4i *>(ib + off0), *reinterpret_cast<const v4i *>(ib + off1));
                v4f d[1];
                block_sums<FA, FAST, 1>(b, a, d);
                const float sa = fs[wm * WTM + i * 16 + fr];
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = add_scaled(d[0][r], scale_pair(sa, fs[BM + wn * WTN + (BUNI ? 0 : j * 16 + fg * 4 + r)]), acc[i][j][r]);
                asm volatile("" : "+v"(acc[i][j])::"memory");
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    // Where such a product matters, the whole tile is multiplied once more behind the loop.  There and not in it: a second form of the block's
    // product spills 90 of the large tile's registers, a precise look at every pair of scales costs it 2 to 4 %, this one 0 to 2.  4096^3,
    // e5m2 A: bf16 79 us, with masked rows 76; f32 118 and 141; with rows of 1e-38 280 and 430 to 520.
    unsigned long long odd = 0;
    auto look = [&](int buf) {
        if (__builtin_expect(odd != 0, 0) && matters(buf)) *again = 1;
    };
    if (t == 0) *again = 0;
    if constexpr (STAGES > 2) {
        // Two blocks under way, scales included.  Every wave waits for its own share of block s; behind the barrier all shares are
        // there, and everyone is done with block s - 1, whose stage takes block s + 2.
        constexpr int PER = NA + NB + 1;  // transfers of a block and wave
        // (waves that own no scale fetch one all the same, behind the stages: all count the same transfers)
        const unsigned scales0 = lds_dma::lds_addr(scales) + (has_scale ? wave * 256 : STAGES * (BM + BN) * 4 + (wave - (BM + BN) / 64) * 256);
        const unsigned scales_step = has_scale ? (BM + BN) * 4 : 0;
        int next = 0;
        auto request = [&](int64_t s) {
            stage(s, next);
            lds_dma::dma4_spaced(s_ptr + s * s_step, scales0 + next * scales_step);
            next = next == STAGES - 1 ? 0 : next + 1;
        };
        if (whole > 0) request(0);
        if (whole > 1) request(1);
        int buf = 0;
#pragma unroll 1
        for (int64_t s = 0; s < whole; ++s) {
            if (s + 1 < whole) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (s + 2 < whole) request(s + 2);
            const float s_mine = scales[buf * (BM + BN) + (has_scale ? t : 0)];
            if (active) multiply(buf);
            odd = __ballot(has_scale && outside(s_mine));
            look(buf);
            buf = buf == STAGES - 1 ? 0 : buf + 1;
        }
        s_ptr += whole * s_step;
        __syncthreads();
    } else {
    if (whole > 0) {
        stage(0, 0);
        const float s_first = *s_ptr;
        if (has_scale) scales[t] = s_first;
        odd = __ballot(has_scale && outside(s_first));
        land(0);
        __syncthreads();
    }
#pragma unroll 1
    for (int64_t s = 0; s < whole; ++s) {
        const int buf = (int)(s & 1);
        const bool more = s + 1 < whole;
        float s_next = 0.f;
        if (more) {
            s_ptr += s_step;
            s_next = *s_ptr;
            stage(s + 1, buf ^ 1);
        }
        if (active) multiply(buf);
        look(buf);
        if (more) {
            if (has_scale) scales[(buf ^ 1) * (BM + BN) + t] = s_next;
            odd = __ballot(has_scale && outside(s_next));
            land(buf ^ 1);
        }
        __syncthreads();
    }
    }
    // The block that K ends in, behind the loop (inside it, its branches cost the loop its registers): through registers, chunk
    // by chunk, zeros beyond the end.
    if (k_len % kScaleBlock != 0) {
        const int buf = (int)(whole % STAGES);
        if (STAGES == 2 && whole > 0) s_ptr += s_step;
        const float s_last = *s_ptr;
        if (has_scale) scales[buf * (BM + BN) + t] = s_last;
        odd = __ballot(has_scale && outside(s_last));
        put_chunks(whole, buf);
        __syncthreads();
        if (active) multiply(buf);
        look(buf);
        __syncthreads();
    }

    // Every block once more, with the scales' exponents apart.  (`again` was cleared in front of the first barrier and is read behind the last one.)
    if (k_len > 0 && __builtin_expect(__builtin_amdgcn_readfirstlane(*again), 0)) {
        const int64_t blocks = (k_len + kScaleBlock - 1) / kScaleBlock;
        s_ptr -= (STAGES > 2 || k_len % kScaleBlock != 0 ? whole : whole - 1) * s_step;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int64_t s = 0; s < blocks; ++s, s_ptr += s_step) {
            put_chunks(s, 0);
            if (has_scale) scales[t] = *s_ptr;
            __syncthreads();
            if (active) multiply_apart(0);
            __syncthreads();
        }
    }

    // The finished tile passes through LDS (the operands' stages are free) in pieces of 32 rows of every wave row, and
    // leaves in runs of whole rows: 16 bytes or more per lane, a row's columns along the lanes.
    constexpr int PITCH = BN + 4;  // the sixteen rows of a wave's store start on sixteen different 16-byte slots
    static_assert(WM * 32 * PITCH * 4 <= 2 * STAGE && MT % 2 == 0, "a piece fits the stages");
    float *piece = reinterpret_cast<float *>(image);
    const int64_t c_entry = p.split > 1 ? 0 : p.mode == kScaledRows ? 0 : it.entry * p.c_batch;
    float *ws = p.ws + ((int64_t)it.chunk * p.batch + it.entry) * p.M * p.N;
    const bool vec = p.split > 1 ? (p.N & 3) == 0
                                 : ((p.ldc | p.c_batch) & 3) == 0 && (reinterpret_cast<uintptr_t>(p.C) & (p.c_f32 ? 15 : 7)) == 0;
    // f32: a lane's four columns are 16 bytes and a row's four lanes 64, whole sectors without the pass through LDS
    if (vec && (p.N & 3) == 0 && (p.split > 1 || (p.c_f32 && p.beta == 0.f))) {
        float *c = p.split > 1 ? ws : static_cast<float *>(p.C) + c_entry;
        const int64_t ld = p.split > 1 ? p.N : p.ldc;
        const float alpha = p.split > 1 ? 1.f : p.alpha;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int64_t m = it.m0 + wm * WTM + i * 16 + fr, n = it.n0 + wn * WTN + fg * 4;
#pragma unroll
            for (int j = 0; j < NT; ++j)
                if (m < it.m_end && n + j * 16 < p.N) *reinterpret_cast<v4f *>(c + m * ld + n + j * 16) = acc[i][j] * alpha;
        }
        return;
    }
#pragma unroll
    for (int h = 0; h < MT / 2; ++h) {
        if (h > 0) __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                *reinterpret_cast<v4f *>(piece + (wm * 32 + i * 16 + fr) * PITCH + wn * WTN + j * 16 + fg * 4) = acc[2 * h + i][j];
        __syncthreads();
        constexpr int QUADS = BN / 4, STEP = T / QUADS;
        const int q = t % QUADS;
        const int64_t n = it.n0 + q * 4;
#pragma unroll 2
        for (int r = t / QUADS; r < WM * 32; r += STEP) {
            const int64_t m = it.m0 + (r >> 5) * WTM + h * 32 + (r & 31);
            if (m >= it.m_end || n >= p.N) continue;
            const v4f v = *reinterpret_cast<const v4f *>(piece + r * PITCH + q * 4);
            if (p.split > 1) store_partial(ws + m * p.N + n, p.N - n, v, vec);
            else store4(p, c_entry + m * p.ldc + n, n, v, vec);
        }
    }
}

// LIGHT: tiles of at most BM / 2 rows run on waves of half the rows; three of their blocks fit in LDS, which is worth another tenth
// (64 groups, 16384 rows, 2048 x 2048: 165 us without light tiles, 157 with two stages, 150 with three).  A second copy of the kernel,
// since the other tiles' presence costs the full ones 1 % (4096 x 8192 x 4096).
template <int FA, bool FAST, bool BUNI, int BM, int BN, int WM, int WN, bool DMA, bool LIGHT, int STAGES>
__global__ void __launch_bounds__(WM *WN * 64, STAGES > 2 ? 1 : 2) scaled_gemm_kernel(ScaledGemmParams p)
{
    __shared__ __attribute__((aligned(16))) uint8_t image[LIGHT ? 3 * (BM / 2 + BN) * 128 : STAGES * (BM + BN) * 128];
    __shared__ __attribute__((aligned(16))) float scales[LIGHT ? 3 * (BM / 2 + BN) + 128 : STAGES * (BM + BN)];
    __shared__ int again;
    Item it;
    if (!find_item<BM, BN, LIGHT>(p, it)) return;
    it.m0 = uniform(it.m0);
    it.m_end = uniform(it.m_end);
    it.n0 = uniform(it.n0);
    it.k_begin = uniform(it.k_begin);
    it.k_end = uniform(it.k_end);
    it.entry = uniform(it.entry);
    if constexpr (LIGHT) {
        if (it.m_end - it.m0 <= BM / 2) {
            multiply_tile<FA, FAST, BUNI, BM / 2, BN, WM, WN, DMA, 3>(p, it, image, scales, &again);
            return;
        }
    }
    multiply_tile<FA, FAST, BUNI, BM, BN, WM, WN, DMA, STAGES>(p, it, image, scales, &again);
}

// Sums the chunks' partial results in the order of the chunks (the same on every run) and stores C.  A split result has fewer
// tiles than the device compute units, hence indexes of 32 bits.  Four chunks are requested at a time: one by one, each would wait
// for the one before it.
__global__ void __launch_bounds__(256) scaled_split_sum_kernel(ScaledGemmParams p)
{
    const uint32_t rows = (uint32_t)p.M, quads = (uint32_t)((p.N + 3) >> 2), items = quads * rows * (uint32_t)p.batch;
    const int64_t total = p.M * p.N * p.batch;
    const bool vec = ((p.ldc | p.c_batch) & 3) == 0 && (reinterpret_cast<uintptr_t>(p.C) & (p.c_f32 ? 15 : 7)) == 0;
    const bool whole = (p.N & 3) == 0;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < items; i += gridDim.x * 256) {
        const uint32_t line = i / quads, b = line / rows;
        const int64_t n = (int64_t)(i - line * quads) * 4, m = line - b * rows;
        const float *w = p.ws + (int64_t)line * p.N + n;
        v4f v = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < p.split; s0 += 4) {
            v4f part[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {  // beyond the last chunk: that one again, not added
                const float *from = w + (s0 + u < p.split ? s0 + u : p.split - 1) * total;
                if (whole) {
                    part[u] = *reinterpret_cast<const v4f *>(from);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) part[u][r] = from[n + r < p.N ? r : 0];
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = s0 + u < p.split ? v[r] + part[u][r] : v[r];
        }
        store4(p, b * p.c_batch + m * p.ldc + n, n, v, vec);
    }
}

template <int FA, bool FAST, bool BUNI> hipError_t launch_tiles(const ScaledGemmParams &p, int kind, bool dma, unsigned grid, hipStream_t stream)
{
    if constexpr (FAST) {  // (two fragments of bf16 do not fit the registers beside 128 accumulators)
        if (kind == 2) {
            if (p.cus > 0)
                hipLaunchKernelGGL((scaled_gemm_kernel<FA, FAST, BUNI, 256, 256, 2, 4, true, true, 2>), dim3(grid), dim3(512), 0, stream, p);
            else
                hipLaunchKernelGGL((scaled_gemm_kernel<FA, FAST, BUNI, 256, 256, 2, 4, true, false, 2>), dim3(grid), dim3(512), 0, stream, p);
            return hipGetLastError();
        }
    }
    if (dma && kind == 3)
        hipLaunchKernelGGL((scaled_gemm_kernel<FA, FAST, BUNI, 128, 128, 2, 2, true, false, 3>), dim3(grid), dim3(256), 0, stream, p);
    else if (dma)
        hipLaunchKernelGGL((scaled_gemm_kernel<FA, FAST, BUNI, 128, 128, 2, 2, true, false, 2>), dim3(grid), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((scaled_gemm_kernel<FA, FAST, BUNI, 128, 128, 2, 2, false, false, 2>), dim3(grid), dim3(256), 0, stream, p);
    return hipGetLastError();
}

// (2^22: the DMA's offsets inside a tile are 32-bit, 255 rows and a row's length)
bool dma_ready(const ScaledMatrix &m, int64_t k) { return ((reinterpret_cast<uintptr_t>(m.q) | (uintptr_t)m.ld | (uintptr_t)m.batch) & 15) == 0 && m.ld <= 1 << 22 && k >= 16; }

}  // namespace

ScaledSchedule schedule_scaled(const ScaledGemmParams &p, int cus, size_t ws_limit)
{
    ScaledSchedule s;
    // Few rows: B is read for them alone, straight into registers.  Dense products up to 32 rows; groups up to a mean of 8, since
    // shares are uneven and a group of more than 16 rows passes over its weights again (32 groups, weights 2048 x 4096:
    // 54 us against 64 on the 128 tile at a mean of 8 rows, 73 against 67 at 12, 83 against 67 at 16).
    if (p.mode == kScaledDense && p.M <= 32) return s;
    if (p.mode == kScaledRows && p.M <= 8 * (int64_t)p.batch) return s;
    const int64_t entries = p.mode == kScaledRows ? 1 : p.batch;
    const auto tiles = [&](int64_t b) -> double {  // (the product of three 31-bit counts)
        const int64_t nbm = (p.M + b - 1) / b + (p.mode == kScaledRows ? p.batch / 2 : 0);
        return (double)nbm * (double)((p.N + b - 1) / b) * (double)entries;
    };
    s.kind = !p.c_f32 && dma_ready(p.a, p.K) && dma_ready(p.b, p.K) && tiles(256) >= cus * 3 / 4 ? 2 : 1;
    if (s.kind == 1 && p.mode == kScaledDense && tiles(128) < cus) {
        const int64_t steps = (p.K + kScaleBlock - 1) / kScaleBlock;
        // chunks of eight blocks or more, 64 at most: a second launch has to pay (150 x 260 x 16384: 20 us in chunks of four, 16 of
        // eight, 18 of sixteen, 84 whole; 128 x 128 x 131072: 80 in 256 chunks, 47 in 128, 35 in 64, 614 whole)
        // With DMA one workgroup a compute unit and three stages: longer chunks, fewer partial sums (512 x 4096 x 4096: 26.1 -> 23.3 us;
        // 128 x 8192 x 8192: 31.0 -> 26.3; 48 x 4096 x 4096: 13.2 -> 12.8); without, two workgroups.
        const bool dma = dma_ready(p.a, p.K) && dma_ready(p.b, p.K);
        int64_t split = (int64_t)((dma ? 1 : 2) * cus / tiles(128));
        if (split > steps / 8) split = steps / 8;
        if (split > 64) split = 64;
        const size_t one = (size_t)p.M * p.N * p.batch * 4;
        if (split > 1 && (size_t)split * one > ws_limit) split = (int64_t)(ws_limit / one);
        if (split > 1) {
            const int64_t per = (steps + split - 1) / split;
            s.split = (int)((steps + per - 1) / per);
            s.ws_bytes = s.split > 1 ? (size_t)s.split * one : 0;
        }
        if (dma && tiles(128) * s.split <= cus) s.kind = 3;
    }
    return s;
}

hipError_t launch_scaled_gemm(ScaledGemmParams p, const ScaledSchedule &s, int cus, hipStream_t stream)
{
    const int b = s.kind == 2 ? 256 : 128;
    p.nbm = (int)((p.M + b - 1) / b);
    p.nbn = (int)((p.N + b - 1) / b);
    p.split = s.split;
    const int64_t steps = (p.K + kScaleBlock - 1) / kScaleBlock;
    p.steps_per = (int)((steps + s.split - 1) / s.split);
    double count = (double)p.nbm * p.nbn * p.batch * p.split;
    // row tiles of ragged groups: each group adds at most one partly filled tile
    if (p.mode == kScaledRows) count = (double)(p.M / b + (p.batch < p.M ? p.batch : p.M)) * p.nbn;
    if (count > 0x7fffff - cus) return hipErrorInvalidValue;  // (512 threads each: a launch holds fewer than 2^32)
    if (s.kind == 2) {
        // Groups always have light tiles (32 groups, 16384 rows, 2048 x 4096: 205 -> 197 us; 64 groups, 4096 rows, 4096 x 2048: 163 -> 140).
        // A dense product may have a light last row or a last round to halve; beyond eight rounds neither pays the full tiles' 1 %.
        const bool light = (p.M - 1) % b < b / 2;
        const int tiles = (int)count, full = light ? tiles / p.nbm * (p.nbm - 1) : tiles, rest = full % cus;
        const bool halves = rest > 0 && 2 * rest + (tiles - full) <= cus;
        if (p.mode == kScaledRows || (p.mode == kScaledDense && (light || halves) && tiles <= 8 * cus)) {
            p.cus = cus;
            count += cus / 2;  // a tile in halves is one workgroup more
        }
    }
    const unsigned grid = (unsigned)count;
    const bool uni = p.b.shift == 7, dma = dma_ready(p.a, p.K) && dma_ready(p.b, p.K);
    const bool fast = !p.c_f32;  // an f32 result takes f32 sums (see block_sums)
    typedef hipError_t (*launcher)(const ScaledGemmParams &, int, bool, unsigned, hipStream_t);
    static const launcher table[2][2][2] = {{{launch_tiles<0, false, false>, launch_tiles<0, false, true>}, {launch_tiles<0, true, false>, launch_tiles<0, true, true>}},
                                            {{launch_tiles<1, false, false>, launch_tiles<1, false, true>}, {launch_tiles<1, true, false>, launch_tiles<1, true, true>}}};
    const hipError_t e = table[p.a.e5m2][fast][uni](p, s.kind, dma, grid, stream);
    if (e != hipSuccess || p.split == 1) return e;
    int64_t blocks = (((p.N + 3) >> 2) * p.M * p.batch + 255) / 256;
    if (blocks > 256 * 16) blocks = 256 * 16;
    hipLaunchKernelGGL(scaled_split_sum_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace ctc
