// Block-scaled 8-bit operators: what the C ABI (scaled_api.cpp) and the kernel files share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ctc {

constexpr int kScaleBlock = 128;  // contracted elements (and, for tiles, rows) under one scale

// q(r, c) * scale(r >> shift, c / 128): shift 0 for one scale per row and block, 7 for 128 x 128 tiles.  Element strides.
struct ScaledMatrix {
    uint8_t *q = nullptr;
    int64_t ld = 0, batch = 0;
    float *scale = nullptr;
    int64_t s_row = 0, s_blk = 0, s_batch = 0;
    int shift = 0;
    int e5m2 = 0;
};

// ---- quantiser (scaled_quantize_kernels.hip) ----
struct QuantizeParams {
    const void *x = nullptr;
    int64_t rows = 0, cols = 0, ldx = 0, x_batch = 0;
    int batch = 1;
    int src = 0;  // 1 f32, 2 bf16 (ctc_tc_dtype)
    ScaledMatrix out, out_t;  // q == nullptr: not wanted
};
hipError_t launch_block_quantize(const QuantizeParams &p, hipStream_t stream);

// ---- products (scaled_gemm_kernels.hip, scaled_skinny_kernels.hip) ----
enum ScaledMode { kScaledDense = 0, kScaledRows = 1, kScaledContracted = 2 };

struct ScaledGemmParams {
    ScaledMatrix a, b;  // [M][K], [N][K]
    void *C = nullptr;
    int64_t ldc = 0, c_batch = 0;
    int64_t M = 0, N = 0, K = 0;
    int batch = 1;  // dense: entries; grouped: groups
    float alpha = 1.f, beta = 0.f;
    int c_f32 = 0;
    int mode = kScaledDense;
    const int32_t *offsets = nullptr;  // grouped: batch + 1 offsets of rows (of contracted elements), on the device
    // schedule
    int nbm = 0, nbn = 0;
    int cus = 0;  // compute units where the large tile's kernel tells full tiles from light ones, else 0
    int split = 1, steps_per = 0;  // dense: K blocks of a chunk; partial sums of chunk s at ws + s * batch * M * N
    float *ws = nullptr;
};

struct ScaledSchedule {
    int kind = 0;  // 0 skinny (no LDS staging), 1 the 128 tile, 2 the 256 tile, 3 the 128 tile with three stages
    int split = 1;
    size_t ws_bytes = 0;
};
// cus: compute units of the device; ws_limit: bytes of workspace the caller has
ScaledSchedule schedule_scaled(const ScaledGemmParams &p, int cus, size_t ws_limit);
hipError_t launch_scaled_gemm(ScaledGemmParams p, const ScaledSchedule &s, int cus, hipStream_t stream);
hipError_t launch_scaled_skinny(const ScaledGemmParams &p, hipStream_t stream);

// ---- the experts' layer for a few tokens (expert_kernels.hip) ----
constexpr int kExpertMaxTokens = 64;
constexpr int kExpertMaxTop = 16;
constexpr int kExpertMaxPairs = kExpertMaxTokens * kExpertMaxTop;
constexpr int kExpertMaxExperts = 4096;
struct ExpertParams {
    const void *x = nullptr;  // bf16
    int64_t ldx = 0;
    ScaledMatrix up, down;
    const int32_t *pick = nullptr;
    const float *gate = nullptr;
    int64_t ld_pick = 0, ld_gate = 0;
    void *y = nullptr;  // bf16
    int64_t ldy = 0;
    int tokens = 0, top = 0, experts = 0;
    int64_t hidden = 0, inner = 0;
    void *h = nullptr;  // workspace: tokens * top rows of `inner` bf16 numbers
};
hipError_t launch_expert_layer(const ExpertParams &p, hipStream_t stream);

}  // namespace ctc
