// C ABI of the block-scaled 8-bit operators (declared in include/ctc_tc.h): argument checks, schedules, launches.
#include "ctc_tc.h"

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstring>
#include <string>
#include <utility>

#include "api_internal.hpp"
#include "scaled.hpp"

namespace {

using ctc_internal::set_last_error;
using ctc_internal::set_last_hip_error;

std::atomic<int64_t> g_skinny{0}, g_tile128{0}, g_tile256{0}, g_split{0};

// elements that an operand may span: offsets, in bytes as well, stay far inside 64 bits
constexpr double kMaxSpan = 70368744177664.0;  // 2^46
double span(int64_t batch, int64_t batch_stride, int64_t rows, int64_t ld, int64_t cols)
{
    return (double)(batch - 1) * (double)batch_stride + (double)(rows - 1) * (double)ld + (double)cols;
}
constexpr int64_t kMaxDim = 0x7fffffff - 4096;  // row, column and block indexes are 32-bit inside a launch

int refuse(const char *what, const char *why) { return set_last_error(CTC_TC_EINVAL, std::string(what) + ": " + why); }
int unsupported(const char *what, const char *why) { return set_last_error(CTC_TC_EUNSUPPORTED, std::string(what) + ": " + why); }

int64_t blocks_of(int64_t n) { return (n + ctc::kScaleBlock - 1) / ctc::kScaleBlock; }

// of the current device; asked for once per device
int compute_units()
{
    static std::atomic<int> known[64];
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess) {
        (void)hipGetLastError();
        return 256;
    }
    if (dev >= 0 && dev < 64 && (cus = known[dev].load(std::memory_order_relaxed)) > 0) return cus;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1) {
        (void)hipGetLastError();
        return 256;
    }
    if (dev >= 0 && dev < 64) known[dev].store(cus, std::memory_order_relaxed);
    return cus;
}

ctc::ScaledMatrix matrix(const ctc_tc_scaled_matrix &m)
{
    ctc::ScaledMatrix o;
    o.q = static_cast<uint8_t *>(m.q);
    o.ld = m.ld;
    o.batch = m.batch_stride;
    o.scale = m.scale;
    o.s_row = m.scale_row;
    o.s_blk = m.scale_block;
    o.s_batch = m.scale_batch;
    o.shift = m.block == CTC_TC_BLOCK_TILES ? 7 : 0;
    o.e5m2 = m.dtype == CTC_TC_F8E5M2;
    return o;
}

// rows x cols 8-bit matrix `m`, `batch` of them; its message carries the operand's name
int check_matrix(const char *what, const char *name, const ctc_tc_scaled_matrix *m, int64_t rows, int64_t cols, int64_t batch, bool e5m2_ok)
{
    const std::string w = std::string(what) + ": " + name;
    if (!m) return set_last_error(CTC_TC_EINVAL, w + " is null");
    if (m->dtype != CTC_TC_F8E4M3 && m->dtype != CTC_TC_F8E5M2) return set_last_error(CTC_TC_EINVAL, w + " must be e4m3 or e5m2");
    if (m->dtype == CTC_TC_F8E5M2 && !e5m2_ok) return set_last_error(CTC_TC_EUNSUPPORTED, w + " must be e4m3");
    if (m->block != CTC_TC_BLOCK_ROWS && m->block != CTC_TC_BLOCK_TILES) return set_last_error(CTC_TC_EINVAL, w + " has an unknown block kind");
    if (rows == 0 || cols == 0 || batch == 0) return CTC_TC_OK;
    if (!m->q || !m->scale) return set_last_error(CTC_TC_EINVAL, w + " has a null pointer");
    if (reinterpret_cast<uintptr_t>(m->scale) & 3) return set_last_error(CTC_TC_EALIGN, w + " has scales off a 4-byte boundary");
    if (m->ld < cols) return set_last_error(CTC_TC_EINVAL, w + " has a leading dimension below its row length");
    if (m->batch_stride < 0 || m->scale_row < 0 || m->scale_block < 0 || m->scale_batch < 0)
        return set_last_error(CTC_TC_EINVAL, w + " has a negative stride");
    if (span(batch, m->batch_stride, rows, m->ld, cols) > kMaxSpan ||
        span(batch, m->scale_batch, rows, m->scale_row, 1) + (double)blocks_of(cols) * (double)m->scale_block > kMaxSpan)
        return set_last_error(CTC_TC_EUNSUPPORTED, w + " spans too much memory");
    return CTC_TC_OK;
}

// `batch` matrices of rows x cols at these strides that would write to the same place: neither whole matrices nor the
// matrices' rows (a batch index between the two) stand apart
bool overlap(int64_t rows, int64_t cols, int64_t ld, int64_t batch, int64_t stride)
{
    if (batch <= 1) return false;
    const bool whole = (double)stride >= span(1, 0, rows, ld, cols);
    const bool between = stride >= cols && (rows <= 1 || (double)ld >= span(1, 0, batch, stride, cols));
    return !whole && !between;
}

// a matrix that the quantiser writes: nothing of it twice
int check_written(const char *what, const char *name, const ctc_tc_scaled_matrix &m, int64_t rows, int64_t cols, int64_t batch)
{
    const int64_t r = m.block == CTC_TC_BLOCK_TILES ? blocks_of(rows) : rows, c = blocks_of(cols);
    // the scales' three strides in rising order, each past the extent of those below it
    int64_t stride[3] = {m.scale_row, m.scale_block, m.scale_batch}, n[3] = {r, c, batch};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (stride[j] < stride[i]) {
                std::swap(stride[i], stride[j]);
                std::swap(n[i], n[j]);
            }
    double extent = 1;
    bool twice = overlap(rows, cols, m.ld, batch, m.batch_stride);
    for (int i = 0; i < 3; ++i) {
        if (n[i] == 1) continue;
        twice = twice || (double)stride[i] < extent;
        extent += (double)(n[i] - 1) * (double)stride[i];
    }
    return twice ? set_last_error(CTC_TC_EINVAL, std::string(what) + ": " + name + " overlaps itself") : CTC_TC_OK;
}

int check_result(const char *what, const void *C, int64_t ldc, int64_t c_batch, int64_t rows, int64_t n, int64_t batch, int dtype)
{
    if (dtype != CTC_TC_F32 && dtype != CTC_TC_BF16) return unsupported(what, "the result is f32 or bf16");
    if (rows == 0 || n == 0 || batch == 0) return CTC_TC_OK;
    if (!C) return refuse(what, "the result is null");
    if (reinterpret_cast<uintptr_t>(C) & (dtype == CTC_TC_F32 ? 3 : 1)) return set_last_error(CTC_TC_EALIGN, std::string(what) + ": the result is not aligned to its elements");
    if (ldc < n) return refuse(what, "the result's leading dimension is below its row length");
    if (batch > 1 && c_batch < 0) return refuse(what, "a stride of the result is negative");
    if (span(batch, batch > 1 ? c_batch : 0, rows, ldc, n) > kMaxSpan) return unsupported(what, "the result spans too much memory");
    if (overlap(rows, n, ldc, batch, c_batch)) return refuse(what, "the result's matrices overlap");
    return CTC_TC_OK;
}

int run_product(const char *what, ctc::ScaledGemmParams &p, void *workspace, int64_t workspace_bytes, hipStream_t stream)
{
    const size_t room = workspace ? (size_t)workspace_bytes : 0;
    const int cus = compute_units();
    const ctc::ScaledSchedule s = ctc::schedule_scaled(p, cus, room);
    p.ws = static_cast<float *>(workspace);
    hipError_t e = s.kind == 0 ? ctc::launch_scaled_skinny(p, stream) : ctc::launch_scaled_gemm(p, s, cus, stream);
    if (e == hipErrorInvalidValue) return unsupported(what, "too many tiles for one launch");
    if (e != hipSuccess) return set_last_hip_error(e, what);
    (s.kind == 0 ? g_skinny : s.kind == 2 ? g_tile256 : g_tile128).fetch_add(1, std::memory_order_relaxed);
    if (s.split > 1) g_split.fetch_add(1, std::memory_order_relaxed);
    return CTC_TC_OK;
}

}  // namespace

namespace ctc_internal {
int64_t scaled_counter(const char *name)
{
    if (!strcmp(name, "launches_scaled_skinny")) return g_skinny.load();
    if (!strcmp(name, "launches_scaled_128")) return g_tile128.load();
    if (!strcmp(name, "launches_scaled_256")) return g_tile256.load();
    if (!strcmp(name, "launches_scaled_split")) return g_split.load();
    return -1;
}
}  // namespace ctc_internal

extern "C" {

int ctc_tc_block_quantize(const void *x, int64_t rows, int64_t cols, int64_t ldx, int64_t batch, int64_t batch_stride_x, int src_dtype,
                          const ctc_tc_scaled_matrix *out, const ctc_tc_scaled_matrix *out_t, void *stream)
{
    CTC_ABI_TRY
    const char *what = "block_quantize";
    if (rows < 0 || cols < 0 || batch < 0) return refuse(what, "negative size");
    if (src_dtype != CTC_TC_F32 && src_dtype != CTC_TC_BF16) return unsupported(what, "the input is f32 or bf16");
    if (!out && !out_t) return refuse(what, "no result is wanted");
    if (out && out_t && (out->dtype != out_t->dtype || out->block != out_t->block)) return refuse(what, "the two results differ in type or block kind");
    if (out) {
        if (int rc = check_matrix(what, "the result", out, rows, cols, batch, true)) return rc;
    }
    if (out_t) {
        if (int rc = check_matrix(what, "the transposed result", out_t, cols, rows, batch, true)) return rc;
    }
    if (rows == 0 || cols == 0 || batch == 0) return CTC_TC_OK;
    if (!x) return refuse(what, "the input is null");
    if (reinterpret_cast<uintptr_t>(x) & (src_dtype == CTC_TC_F32 ? 3 : 1)) return set_last_error(CTC_TC_EALIGN, "block_quantize: the input is not aligned to its elements");
    if (ldx < cols || batch_stride_x < 0) return refuse(what, "the input's leading dimension is below its row length, or a stride is negative");
    if (span(batch, batch_stride_x, rows, ldx, cols) > kMaxSpan) return unsupported(what, "the input spans too much memory");
    if (out) {
        if (int rc = check_written(what, "the result", *out, rows, cols, batch)) return rc;
    }
    if (out_t) {
        if (int rc = check_written(what, "the transposed result", *out_t, cols, rows, batch)) return rc;
    }
    if (rows > kMaxDim || cols > kMaxDim || batch > 65535 || blocks_of(rows) * blocks_of(cols) > (1 << 23)) return unsupported(what, "too large for one launch");
    ctc::QuantizeParams p;
    p.x = x;
    p.rows = rows;
    p.cols = cols;
    p.ldx = ldx;
    p.x_batch = batch_stride_x;
    p.batch = (int)batch;
    p.src = src_dtype;
    if (out) p.out = matrix(*out);
    if (out_t) p.out_t = matrix(*out_t);
    hipError_t e = ctc::launch_block_quantize(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return set_last_hip_error(e, "block_quantize kernel launch");
    return CTC_TC_OK;
    CTC_ABI_CATCH
}

int64_t ctc_tc_scaled_workspace_bytes(int64_t m, int64_t n, int64_t k, int64_t batch)
{
    CTC_ABI_TRY
    const char *what = "scaled_workspace_bytes";
    if (m < 0 || n < 0 || k < 0 || batch < 0) return refuse(what, "negative size");
    if (m > kMaxDim || n > kMaxDim || k > kMaxDim || batch > 65535) return unsupported(what, "an extent is too large");
    if (m == 0 || n == 0 || batch == 0) return 0;
    ctc::ScaledGemmParams p;
    p.M = m;
    p.N = n;
    p.K = k;
    p.batch = (int)batch;
    p.a.ld = 1;  // operands off 16 bytes split the furthest
    return (int64_t)ctc::schedule_scaled(p, compute_units(), (size_t)1 << 62).ws_bytes;
    CTC_ABI_CATCH
}

int ctc_tc_scaled_contract(int64_t m, int64_t n, int64_t k, int64_t batch, const ctc_tc_scaled_matrix *a, const ctc_tc_scaled_matrix *b,
                           double alpha, double beta, void *C, int64_t ldc, int64_t batch_stride_c, int c_dtype, void *workspace,
                           int64_t workspace_bytes, void *stream)
{
    CTC_ABI_TRY
    const char *what = "scaled_contract";
    if (m < 0 || n < 0 || k < 0 || batch < 0 || workspace_bytes < 0) return refuse(what, "negative size");
    if (m > kMaxDim || n > kMaxDim || k > kMaxDim || batch > 65535) return unsupported(what, "an extent is too large");
    if (int rc = check_matrix(what, "A", a, m, k, batch, true)) return rc;
    if (int rc = check_matrix(what, "B", b, n, k, batch, false)) return rc;
    if (int rc = check_result(what, C, ldc, batch_stride_c, m, n, batch, c_dtype)) return rc;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return set_last_error(CTC_TC_EALIGN, "scaled_contract: the workspace is not 16-byte aligned");
    if (m == 0 || n == 0 || batch == 0) return CTC_TC_OK;
    ctc::ScaledGemmParams p;
    p.a = matrix(*a);
    p.b = matrix(*b);
    p.C = C;
    p.ldc = ldc;
    p.c_batch = batch > 1 ? batch_stride_c : 0;
    p.M = m;
    p.N = n;
    p.K = k;
    p.batch = (int)batch;
    p.alpha = (float)alpha;
    p.beta = (float)beta;
    p.c_f32 = c_dtype == CTC_TC_F32;
    return run_product(what, p, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
    CTC_ABI_CATCH
}

int ctc_tc_scaled_grouped_contract(int along, int64_t groups, const int32_t *offsets, int64_t m, int64_t n, int64_t k,
                                   const ctc_tc_scaled_matrix *a, const ctc_tc_scaled_matrix *b, double alpha, double beta, void *C,
                                   int64_t ldc, int64_t group_stride_c, int c_dtype, void *stream)
{
    CTC_ABI_TRY
    const char *what = "scaled_grouped_contract";
    if (along != CTC_TC_GROUPS_ROWS && along != CTC_TC_GROUPS_CONTRACTED) return refuse(what, "unknown kind of groups");
    const bool rows = along == CTC_TC_GROUPS_ROWS;
    if (m < 0 || n < 0 || k < 0 || groups < 0) return refuse(what, "negative size");
    if (m > kMaxDim || n > kMaxDim || k > kMaxDim || groups > 65535) return unsupported(what, "an extent is too large");
    if (int rc = check_matrix(what, "A", a, m, k, 1, true)) return rc;
    if (int rc = check_matrix(what, "B", b, n, k, rows ? groups : 1, false)) return rc;
    if (int rc = check_result(what, C, ldc, group_stride_c, m, n, rows ? 1 : groups, c_dtype)) return rc;
    if (m == 0 || n == 0 || groups == 0) return CTC_TC_OK;
    if (!offsets) return refuse(what, "the offsets are null");
    if (reinterpret_cast<uintptr_t>(offsets) & 3) return set_last_error(CTC_TC_EALIGN, "scaled_grouped_contract: the offsets are off a 4-byte boundary");
    ctc::ScaledGemmParams p;
    p.a = matrix(*a);
    p.b = matrix(*b);
    p.a.batch = p.a.s_batch = 0;
    if (!rows) p.b.batch = p.b.s_batch = 0;
    p.C = C;
    p.ldc = ldc;
    p.c_batch = !rows && groups > 1 ? group_stride_c : 0;
    p.M = m;
    p.N = n;
    p.K = k;
    p.batch = (int)groups;
    p.alpha = (float)alpha;
    p.beta = (float)beta;
    p.c_f32 = c_dtype == CTC_TC_F32;
    p.mode = rows ? ctc::kScaledRows : ctc::kScaledContracted;
    p.offsets = offsets;
    return run_product(what, p, nullptr, 0, static_cast<hipStream_t>(stream));
    CTC_ABI_CATCH
}

int64_t ctc_tc_expert_workspace_bytes(int64_t tokens, int64_t top, int64_t inner)
{
    CTC_ABI_TRY
    const char *what = "expert_workspace_bytes";
    if (tokens < 0 || top < 0 || inner < 0) return refuse(what, "negative size");
    if (tokens > ctc::kExpertMaxTokens) return refuse(what, "at most 64 tokens");
    if (top > ctc::kExpertMaxTop) return refuse(what, "at most 16 experts a token");
    if (inner > kMaxDim) return refuse(what, "an extent is too large");
    return tokens * top * inner * 2;
    CTC_ABI_CATCH
}

int ctc_tc_expert_layer(int64_t tokens, int64_t top, int64_t experts, int64_t hidden, int64_t inner, const void *x, int64_t ldx,
                        const ctc_tc_scaled_matrix *up, const ctc_tc_scaled_matrix *down, const int32_t *pick, int64_t ld_pick,
                        const float *gate, int64_t ld_gate, void *y, int64_t ldy, void *workspace, int64_t workspace_bytes, void *stream)
{
    CTC_ABI_TRY
    const char *what = "expert_layer";
    if (tokens < 0 || top < 1 || experts < 1 || hidden < 1 || inner < 1 || workspace_bytes < 0) return refuse(what, "a size is too small");
    if (tokens > ctc::kExpertMaxTokens) return unsupported(what, "at most 64 tokens (more: the products over groups of rows)");
    if (top > ctc::kExpertMaxTop || experts > ctc::kExpertMaxExperts) return unsupported(what, "at most 16 experts a token, 4096 in all");
    if (hidden > kMaxDim / 2 || inner > 16 * 65535 * 8 || inner > kMaxDim / 4) return unsupported(what, "an extent is too large");
    if (int rc = check_matrix(what, "the up weights", up, 2 * inner, hidden, experts, false)) return rc;
    if (int rc = check_matrix(what, "the down weights", down, hidden, inner, experts, false)) return rc;
    if (up->block != CTC_TC_BLOCK_TILES || down->block != CTC_TC_BLOCK_TILES) return unsupported(what, "the weights carry one scale per 128 x 128 tile");
    if (tokens == 0) return CTC_TC_OK;
    if (!x || !pick || !gate || !y) return refuse(what, "a null pointer");
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 1 || (reinterpret_cast<uintptr_t>(pick) | reinterpret_cast<uintptr_t>(gate)) & 3)
        return set_last_error(CTC_TC_EALIGN, "expert_layer: an argument is not aligned to its elements");
    if (ldx < hidden || ldy < hidden || ld_pick < top || ld_gate < top) return refuse(what, "a leading dimension is below its row length");
    for (int64_t ld : {ldx, ldy, ld_pick, ld_gate})
        if (span(1, 0, tokens, ld, hidden) > kMaxSpan) return unsupported(what, "an argument spans too much memory");
    if (!workspace || workspace_bytes < tokens * top * inner * 2) return refuse(what, "the workspace is smaller than expert_workspace_bytes says");
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return set_last_error(CTC_TC_EALIGN, "expert_layer: the workspace is not 16-byte aligned");
    ctc::ExpertParams p;
    p.x = x;
    p.ldx = ldx;
    p.up = matrix(*up);
    p.down = matrix(*down);
    p.pick = pick;
    p.gate = gate;
    p.ld_pick = ld_pick;
    p.ld_gate = ld_gate;
    p.y = y;
    p.ldy = ldy;
    p.tokens = (int)tokens;
    p.top = (int)top;
    p.experts = (int)experts;
    p.hidden = hidden;
    p.inner = inner;
    p.h = workspace;
    hipError_t e = ctc::launch_expert_layer(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return set_last_hip_error(e, "expert_layer kernel launch");
    return CTC_TC_OK;
    CTC_ABI_CATCH
}

}  // extern "C"
