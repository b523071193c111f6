// A whole mixture-of-experts layer for a few tokens on gfx950, in two kernels:
//   y[t] = sum_j gate[t, j] * D_e ( silu(G_e x_t) * (U_e x_t) ),  e = pick[t, j],
// weights in e4m3 with one f32 scale per 128 x 128 tile ([G_e; U_e] is one matrix of 2 * inner rows), x and y in bf16.
//
// All there is to read is the picked experts' weights, each once: HBM (or, for one token, latency) bounds both kernels.
// The matrix core multiplies in bf16: e4m3 codes are exact in bf16 and x is bf16 already, so nothing is rounded on the way in;
// sums are f32 and a block of 128 is scaled in f32 before it is added.  The tokens of an expert are the MFMA's columns,
// packed from the router's picks by one ballot (lane = token): a token that did not pick the expert is in no column, so
// that nothing an expert's weights hold (NaN among it) reaches a token that did not pick it.
// Between the kernels h = gate * silu(G x) * (U x) is rounded to bf16, as an activation between two layers is: the second
// kernel's MFMA takes 16 bits.  Its error in y is the size of y's own rounding (0.0024 of the norm together, 0.0017 alone).
// Kept as two bf16 numbers, with two MFMAs, h costs as many bytes out of the L2 as the weights out of HBM: measured 116 us
// against 80 for the second kernel of 32 tokens, 64 experts, 4096 x 1536.
#include "scaled_device.hpp"

namespace ctc {

using namespace scaled;

namespace {

static_assert(kExpertMaxTokens == 64, "a token is a lane of a wave");
static_assert(kExpertMaxExperts / 32 == 128, "a lane of the listing wave reads two words of the experts' bits");

// the bf16 elements at the places of a lane's Codes
struct Halves {
    uint4 v[4];
};
__device__ __forceinline__ Halves load_halves(const uint8_t *row, int64_t k)
{
    Halves h;
#pragma unroll
    for (int q = 0; q < 4; ++q) __builtin_memcpy(&h.v[q], row + 2 * (k + (q & 1) * 8 + (q >> 1) * 64), 16);
    return h;
}
__device__ __forceinline__ Halves load_last_halves(const uint8_t *row, int64_t k, int64_t k_end, bool long_row)
{
    Halves h;
#pragma unroll
    for (int q = 0; q < 4; ++q) h.v[q] = load_chunk(row, 2 * (k + (q & 1) * 8 + (q >> 1) * 64), 2 * k_end, long_row);
    return h;
}
__device__ __forceinline__ v4f block_product(const Codes &c, const Halves &h)
{
    v4f d = {0.f, 0.f, 0.f, 0.f};
    const uint32_t w[8] = {(uint32_t)c.lo[0], (uint32_t)c.lo[1], (uint32_t)c.lo[2], (uint32_t)c.lo[3], (uint32_t)c.hi[0], (uint32_t)c.hi[1], (uint32_t)c.hi[2], (uint32_t)c.hi[3]};
#pragma unroll
    for (int q = 0; q < 4; ++q)
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen<0>(w[2 * q], w[2 * q + 1]), __builtin_bit_cast(bf16x8, h.v[q]), d, 0, 0, 0);
    return d;
}

// the picks of one token, held by the token's lane; -1 beyond `top` and for lanes beyond the tokens
struct Picks {
    int e[kExpertMaxTop];
};
__device__ __forceinline__ Picks load_picks(const ExpertParams &p, int lane)
{
    Picks k;
#pragma unroll
    for (int j = 0; j < kExpertMaxTop; ++j) k.e[j] = j < p.top && lane < p.tokens ? p.pick[lane * p.ld_pick + j] : -1;
    return k;
}
// the first place of `e` among the token's picks, -1: none
__device__ __forceinline__ int place_of(const Picks &k, int e)
{
    int at = -1;
#pragma unroll
    for (int j = kExpertMaxTop - 1; j >= 0; --j)
        if (k.e[j] == e) at = j;
    return at;
}

// h = gate * silu(G x) * (U x) for 16 of an expert's inner rows and all its tokens.  Workgroup (slice, y): y is a pair
// (token, place) where there are fewer pairs than experts, and only the first pair of an expert works; else y is the expert.
// The waves share the contracted blocks, U in flight each; their partial sums meet in LDS, in wave order.
template <bool UNI, int NW, int U> __global__ void __launch_bounds__(NW * 64) expert_up_kernel(ExpertParams p, int by_pair)
{
    __shared__ __attribute__((aligned(16))) float part[NW][2][256];
    __shared__ __attribute__((aligned(16))) uint8_t scratch[NW][2048];
    __shared__ int token_of[64], row_of[64];
    __shared__ float gate_of[64];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    const int64_t i0 = (int64_t)blockIdx.x * 16;
    int e = blockIdx.y;
    if (by_pair) e = p.pick[(blockIdx.y / p.top) * p.ld_pick + blockIdx.y % p.top];
    e = __builtin_amdgcn_readfirstlane(e);
    if (e < 0 || e >= p.experts) return;
    const Picks picks = load_picks(p, lane);
    const int place = place_of(picks, e);
    const unsigned long long mask = __ballot(place >= 0);
    if (mask == 0) return;
    if (by_pair) {  // the expert's first pair: the first token's first place
        const int first = __ffsll((long long)mask) - 1;
        if ((unsigned)(first * p.top + __shfl(place, first)) != blockIdx.y) return;
    }
    const int count = __popcll(mask);
    if (wave == 0 && place >= 0) {
        float g = 0.f;  // a token may name an expert twice: its weights add
#pragma unroll
        for (int j = 0; j < kExpertMaxTop; ++j)
            if (picks.e[j] == e) g += p.gate[lane * p.ld_gate + j];
        const int c = __popcll(mask & ((1ull << lane) - 1));
        token_of[c] = lane;
        row_of[c] = lane * p.top + place;
        gate_of[c] = g;
    }
    __syncthreads();

    constexpr int S = UNI ? 1 : 4;
    const uint8_t *W = p.up.q + e * p.up.batch;
    const int64_t to_up = p.inner * p.up.ld;
    const uint8_t *w_gate = W + min64(i0 + (lane >> 2), p.inner - 1) * p.up.ld + (lane & 3) * 16, *w_up = w_gate + to_up;
    const float *scale = p.up.scale + e * p.up.s_batch;
    const float *s_gate[S], *s_up[S];
#pragma unroll
    for (int r = 0; r < S; ++r) {
        int64_t i = UNI ? i0 : i0 + fg * 4 + r;
        i = i < p.inner ? i : p.inner - 1;
        s_gate[r] = scale + (i >> 7) * p.up.s_row;
        s_up[r] = scale + ((p.inner + i) >> 7) * p.up.s_row;
    }
    const int whole = (int)(p.hidden / kScaleBlock);
    for (int c0 = 0; c0 < count; c0 += 16) {
        const int c = c0 + fr < count ? c0 + fr : count - 1;
        const uint8_t *x = static_cast<const uint8_t *>(p.x) + 2 * (token_of[c] * p.ldx + fg * 16);
        v4f ag = {0.f, 0.f, 0.f, 0.f}, au = {0.f, 0.f, 0.f, 0.f};
        // `mine` chooses and does not branch: loads would sink into the branches, one wait each
        auto multiply = [&](const Codes &cg, const Codes &cu, const Halves &h, const float(&fgate)[S], const float(&fup)[S], bool mine) {
            const v4f dg = block_product(cg, h), du = block_product(cu, h);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                ag[r] = mine ? __builtin_fmaf(dg[r], fgate[UNI ? 0 : r], ag[r]) : ag[r];
                au[r] = mine ? __builtin_fmaf(du[r], fup[UNI ? 0 : r], au[r]) : au[r];
            }
        };
        for (int s0 = wave; s0 < whole; s0 += NW * U) {
            Codes cg[U], cu[U];
            Halves h[U];
            float fgate[U][S], fup[U][S];
#pragma unroll
            for (int u = 0; u < U; ++u) {  // beyond the last block: that one again, not added
                const int64_t s = s0 + u * NW < whole ? s0 + u * NW : whole - 1;
                cg[u] = load_codes(w_gate, s * kScaleBlock);
                cu[u] = load_codes(w_up, s * kScaleBlock);
                h[u] = load_halves(x, s * kScaleBlock);
#pragma unroll
                for (int r = 0; r < S; ++r) {
                    fgate[u][r] = s_gate[r][s * p.up.s_blk];
                    fup[u][r] = s_up[r][s * p.up.s_blk];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) multiply(turn(cg[u], scratch[wave], lane), turn(cu[u], scratch[wave], lane), h[u], fgate[u], fup[u], s0 + u * NW < whole);
        }
        if (p.hidden % kScaleBlock != 0 && wave == whole % NW) {  // the block that the rows end in
            const int64_t k = (int64_t)whole * kScaleBlock, k_end = p.hidden - fg * 16;
            float fgate[S], fup[S];
#pragma unroll
            for (int r = 0; r < S; ++r) {
                fgate[r] = s_gate[r][whole * p.up.s_blk];
                fup[r] = s_up[r][whole * p.up.s_blk];
            }
            const uint8_t *row = W + min64(i0 + fr, p.inner - 1) * p.up.ld + fg * 16;
            multiply(load_last_codes(row, k, k_end, p.hidden >= 16), load_last_codes(row + to_up, k, k_end, p.hidden >= 16), load_last_halves(x, k, k_end, p.hidden >= 8), fgate, fup, true);
        }
        *reinterpret_cast<v4f *>(&part[wave][0][fr * 16 + fg * 4]) = ag;
        *reinterpret_cast<v4f *>(&part[wave][1][fr * 16 + fg * 4]) = au;
        __syncthreads();
        for (int q = t; q < 256; q += NW * 64) {  // (column, row)
            const int col = c0 + (q >> 4), row = q & 15;
            float g = 0.f, u = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                g += part[w][0][q];
                u += part[w][1][q];
            }
            if (col < count && i0 + row < p.inner) {
                const float h = g / (1.f + expf(-g)) * u * gate_of[col];
                static_cast<uint16_t *>(p.h)[row_of[col] * p.inner + i0 + row] = to_bf16(h);
            }
        }
        __syncthreads();
    }
}

// y for 16 of the hidden rows and all tokens: the waves share the picked experts (several waves an expert's contracted
// blocks where there are few), add an expert's columns to their own LDS copy of the 16 x tokens result, and the
// copies are summed in wave order: no atomics on values, the same bits on every run.
template <int NW, int U> __global__ void __launch_bounds__(NW * 64) expert_down_kernel(ExpertParams p, int k_parts)
{
    extern __shared__ __attribute__((aligned(16))) float y_part[];  // [wave][token][16]
    __shared__ uint32_t bits[kExpertMaxExperts / 32];
    __shared__ int list[kExpertMaxPairs];
    __shared__ int listed;
    __shared__ int columns[NW][64];
    __shared__ __attribute__((aligned(16))) uint8_t scratch[NW][2048];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    const int64_t r0 = (int64_t)blockIdx.x * 16;
    const int per_wave = p.tokens * 16;
    for (int i = t; i < NW * per_wave; i += NW * 64) y_part[i] = 0.f;
    if (t < kExpertMaxExperts / 32) bits[t] = 0;
    __syncthreads();
    for (int i = t; i < p.tokens * p.top; i += NW * 64) {
        const int e = p.pick[(i / p.top) * p.ld_pick + i % p.top];
        if (e >= 0 && e < p.experts) atomicOr(&bits[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
    if (wave == 0) {  // the experts in ascending order
        const uint32_t w0 = bits[2 * lane], w1 = bits[2 * lane + 1];
        const int n = __popc(w0) + __popc(w1);
        int sum = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        int at = sum - n;
        for (uint32_t b = w0; b; b &= b - 1) list[at++] = 64 * lane + __ffs((int)b) - 1;
        for (uint32_t b = w1; b; b &= b - 1) list[at++] = 64 * lane + 32 + __ffs((int)b) - 1;
        if (lane == 63) listed = sum;
    }
    const Picks picks = load_picks(p, lane);
    __syncthreads();
    const int experts = listed, lanes = NW / k_parts;
    const int part = wave / lanes, whole = (int)(p.inner / kScaleBlock);
    float *own_y = y_part + wave * per_wave;
    const uint8_t *w0 = p.down.q + min64(r0 + (lane >> 2), p.hidden - 1) * p.down.ld + (lane & 3) * 16;
    const uint8_t *last0 = p.down.q + min64(r0 + fr, p.hidden - 1) * p.down.ld + fg * 16;
    const float *scale0 = p.down.scale + (r0 >> 7) * p.down.s_row;
    const uint8_t *h0 = static_cast<const uint8_t *>(p.h) + 2 * fg * 16;
    for (int u = wave % lanes; u < experts; u += lanes) {
        const int e = __builtin_amdgcn_readfirstlane(list[u]);
        const uint8_t *w = w0 + e * p.down.batch;
        const float *scale = scale0 + e * p.down.s_batch;
        const int place = place_of(picks, e);
        const unsigned long long mask = __ballot(place >= 0);
        const int count = __popcll(mask);
        if (place >= 0) columns[wave][__popcll(mask & ((1ull << lane) - 1))] = lane * p.top + place;
        __builtin_amdgcn_wave_barrier();  // one wave's LDS accesses are in order
        for (int c0 = 0; c0 < count; c0 += 16) {
            const int pair = columns[wave][c0 + fr < count ? c0 + fr : count - 1];
            const uint8_t *h = h0 + 2 * pair * p.inner;
            v4f acc = {0.f, 0.f, 0.f, 0.f};
            for (int s0 = part; s0 < whole; s0 += k_parts * U) {
                Codes c[U];
                Halves v[U];
                float f[U];
#pragma unroll
                for (int q = 0; q < U; ++q) {  // beyond the last block: that one again, not added
                    const int64_t s = s0 + q * k_parts < whole ? s0 + q * k_parts : whole - 1;
                    c[q] = load_codes(w, s * kScaleBlock);
                    v[q] = load_halves(h, s * kScaleBlock);
                    f[q] = scale[s * p.down.s_blk];
                }
#pragma unroll
                for (int q = 0; q < U; ++q) {  // chosen, not branched over: loads would sink into the branches, one wait each
                    const v4f d = block_product(turn(c[q], scratch[wave], lane), v[q]);
                    const bool mine = s0 + q * k_parts < whole;
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[r] = mine ? __builtin_fmaf(d[r], f[q], acc[r]) : acc[r];
                }
            }
            if (p.inner % kScaleBlock != 0 && part == whole % k_parts) {  // the block that the rows end in
                const int64_t k = (int64_t)whole * kScaleBlock, k_end = p.inner - fg * 16;
                const v4f d = block_product(load_last_codes(last0 + e * p.down.batch, k, k_end, p.inner >= 16), load_last_halves(h, k, k_end, p.inner >= 8));
                const float f = scale[whole * p.down.s_blk];
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(d[r], f, acc[r]);
            }
            if (c0 + fr < count) {
                v4f *dst = reinterpret_cast<v4f *>(own_y + (pair / p.top) * 16 + fg * 4);
                *dst += acc;
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (int i = t; i < per_wave; i += NW * 64) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += y_part[w * per_wave + i];
        const int64_t r = r0 + (i & 15);
        if (r < p.hidden) static_cast<uint16_t *>(p.y)[(i >> 4) * p.ldy + r] = to_bf16(v);
    }
}

}  // namespace

hipError_t launch_expert_layer(const ExpertParams &p, hipStream_t stream)
{
    const int pairs = p.tokens * p.top;
    const int by_pair = pairs < p.experts;
    const dim3 up((unsigned)((p.inner + 15) / 16), (unsigned)(by_pair ? pairs : p.experts));
    const bool uni = p.inner % 16 == 0;
    // four waves with two blocks in flight (32 tokens, 4096 and 1536: 161 us, as with two waves; eight take 172 and more.  One token's layer
    // of 128 experts of 4096 and 1536: 42.6 us; eight waves with one block take 45.9, with two 49.2, sixteen 51.6)
    if (uni) hipLaunchKernelGGL((expert_up_kernel<true, 4, 2>), up, dim3(4 * 64), 0, stream, p, by_pair);
    else hipLaunchKernelGGL((expert_up_kernel<false, 4, 2>), up, dim3(4 * 64), 0, stream, p, by_pair);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // Eight waves with two blocks in flight (sixteen waves, or four blocks: 0 to 1 us more).  At most `pairs` experts: with fewer than the
    // waves, several waves share one expert's contracted blocks
    int k_parts = 1;
    while (k_parts < 8 && pairs * k_parts < 8) k_parts *= 2;
    hipLaunchKernelGGL((expert_down_kernel<8, 2>), dim3((unsigned)((p.hidden + 15) / 16)), dim3(512), (size_t)8 * p.tokens * 16 * 4, stream, p, k_parts);
    return hipGetLastError();
}

}  // namespace ctc
