// block_api.hip -- the extern "C" surface of the trainable block operators (include/iffnerf_hip.h): argument checking and error reporting.
#include "../../../include/iffnerf_hip.h"
#include "block_launch.h"

#include <cstdarg>
#include <cstdio>

int iff_report(int code, const char* message);          // api.hip

static int fail(int code, const char* fmt, ...) {
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    return iff_report(code, text);
}
#define IFF_HIP(call)                                                                                                       \
    do {                                                                                                                    \
        hipError_t e__ = (call);                                                                                            \
        if (e__ != hipSuccess) return fail((int)e__, "%s: %s (%s)", #call, hipGetErrorString(e__), hipGetErrorName(e__)); \
    } while (0)
#define IFF_REQUIRE(cond, ...)                                           \
    do {                                                                 \
        if (!(cond)) return fail(IFF_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
    } while (0)

static bool block_type(int32_t t) { return t == IFF_TYPE_F32 || t == IFF_TYPE_BF16 || t == IFF_TYPE_F16; }

static int check_norm(const char* who, int32_t x_type, int64_t n0, int64_t n1, int32_t width, int32_t par_type) {
    IFF_REQUIRE(block_type(x_type), "%s: type %d is not one of IFF_TYPE_F32 / BF16 / F16", who, x_type);
    IFF_REQUIRE(par_type == IFF_TYPE_F32 || par_type == x_type, "%s: parameters of type %d with activations of type %d (fp32 or the same)", who, par_type, x_type);
    IFF_REQUIRE(n0 >= 0 && n1 >= 0 && (n1 == 0 || n0 <= INT32_MAX / n1), "%s: bad row counts %lld x %lld", who, (long long)n0, (long long)n1);
    IFF_REQUIRE(width >= 1 && width <= (1 << 24), "%s: bad width %d", who, width);
    return 0;
}
static NormArgs norm_args(const void* x, int32_t x_type, int64_t n0, int64_t n1, int64_t stride0, int64_t stride1, int32_t width, const void* w,
                          int32_t par_type) {
    NormArgs a{};
    a.dt = x_type; a.x = x; a.s0 = stride0; a.s1 = stride1; a.n1 = (uint32_t)(n1 ? n1 : 1); a.rows = (uint32_t)(n0 * n1); a.D = width;
    a.w = w; a.wk = !w ? 0 : par_type == IFF_TYPE_F32 ? 1 : 2;
    return a;
}
extern "C" int iff_layer_norm_forward(const void* x, int32_t x_type, int64_t n0, int64_t n1, int64_t stride0, int64_t stride1, int32_t width,
                                      const void* w_opt, const void* b_opt, int32_t par_type, float eps, void* y, float* stats_opt, void* stream) {
    if (const int rc = check_norm("iff_layer_norm_forward", x_type, n0, n1, width, par_type)) return rc;
    IFF_REQUIRE(eps >= 0.0f, "iff_layer_norm_forward: eps must not be negative");
    if (n0 * n1 == 0) return 0;
    IFF_REQUIRE(x && y, "iff_layer_norm_forward: null buffer");
    IFF_REQUIRE(((uintptr_t)stats_opt & 7) == 0, "iff_layer_norm_forward: stats must be 8-byte aligned");
    NormArgs a = norm_args(x, x_type, n0, n1, stride0, stride1, width, w_opt, par_type);
    a.b = b_opt; a.bk = !b_opt ? 0 : par_type == IFF_TYPE_F32 ? 1 : 2;
    a.eps = eps; a.y = y; a.stats = stats_opt;
    IFF_HIP(launch_layernorm_fwd(a, (hipStream_t)stream));
    return 0;
}
extern "C" size_t iff_layer_norm_backward_workspace(int64_t rows, int32_t width) {
    if (rows <= 0 || rows > INT32_MAX || width < 1) return 0;
    return (size_t)norm_bwd_groups((uint32_t)rows) * 2 * (size_t)width * 4;
}
extern "C" int iff_layer_norm_backward(const void* x, int32_t x_type, int64_t n0, int64_t n1, int64_t stride0, int64_t stride1, int32_t width,
                                       const void* w_opt, int32_t par_type, const float* stats, const void* dy, void* dx_opt, void* dw_opt,
                                       void* db_opt, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_norm("iff_layer_norm_backward", x_type, n0, n1, width, par_type)) return rc;
    const int64_t rows = n0 * n1;
    if (!dx_opt && !dw_opt && !db_opt) return 0;
    IFF_REQUIRE(rows == 0 || (x && stats && dy), "iff_layer_norm_backward: null buffer");
    IFF_REQUIRE(((uintptr_t)stats & 7) == 0, "iff_layer_norm_backward: stats must be 8-byte aligned");
    const bool params = dw_opt || db_opt;
    const size_t need = params ? iff_layer_norm_backward_workspace(rows, width) : 0;
    if (need && (!workspace || workspace_bytes < need))
        return fail(IFF_ERR_WORKSPACE, "iff_layer_norm_backward: workspace %zu < %zu bytes", workspace_bytes, need);
    NormArgs a = norm_args(x, x_type, n0, n1, stride0, stride1, width, w_opt, par_type);
    a.stats = const_cast<float*>(stats); a.dy = dy; a.dx = dx_opt; a.dw = dw_opt; a.db = db_opt;
    a.dwk = par_type == IFF_TYPE_F32 ? 1 : 2;
    IFF_HIP(launch_layernorm_bwd(a, (float*)workspace, (hipStream_t)stream));
    return 0;
}

static int64_t ffn_limit() { return (int64_t)1 << 21; }          // 2 H and the operand rows of the tile kernel stay below 2^22

static int check_ffn(const char* who, int32_t type, int64_t M, int32_t D, int32_t H, int32_t O) {
    IFF_REQUIRE(block_type(type), "%s: type %d is not one of IFF_TYPE_F32 / BF16 / F16", who, type);
    IFF_REQUIRE(M >= 0 && M <= INT32_MAX, "%s: bad row count %lld", who, (long long)M);
    IFF_REQUIRE(D >= 1 && H >= 1 && O >= 1 && D <= ffn_limit() && H <= ffn_limit() / 2 && O <= ffn_limit(), "%s: bad widths D %d H %d O %d", who, D, H, O);
    return 0;
}
static bool ffn_ok(int32_t type, int64_t M, int32_t D, int32_t H, int32_t O) {
    return block_type(type) && M > 0 && M <= INT32_MAX && D >= 1 && H >= 1 && O >= 1 && D <= ffn_limit() && H <= ffn_limit() / 2 && O <= ffn_limit();
}
static FfnArgs ffn_args(int32_t type, int64_t M, int32_t D, int32_t H, int32_t O) {
    FfnArgs a{};
    a.dt = type; a.M = M; a.D = D; a.H = H; a.O = O;
    return a;
}
extern "C" size_t iff_gated_mlp_kept_bytes(int32_t type, int64_t M, int32_t D, int32_t H, int32_t O) {
    return ffn_ok(type, M, D, H, O) ? ffn_kept_bytes(ffn_args(type, M, D, H, O)) : 0;
}
extern "C" size_t iff_gated_mlp_forward_workspace(int32_t type, int64_t M, int32_t D, int32_t H, int32_t O) {
    return ffn_ok(type, M, D, H, O) ? ffn_forward_workspace(ffn_args(type, M, D, H, O)) : 0;
}
extern "C" int iff_gated_mlp_forward(const void* x, int32_t type, int64_t M, int32_t D, int32_t H, int32_t O, const void* w12,
                                     const void* b12_opt, const void* w3, const void* b3_opt, int32_t activation, void* y, void* kept_opt,
                                     size_t kept_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_ffn("iff_gated_mlp_forward", type, M, D, H, O)) return rc;
    IFF_REQUIRE(activation == IFF_ACT_SILU || activation == IFF_ACT_GELU, "iff_gated_mlp_forward: activation %d is neither IFF_ACT_SILU nor IFF_ACT_GELU", activation);
    if (M == 0) return 0;
    IFF_REQUIRE(x && w12 && w3 && y, "iff_gated_mlp_forward: null buffer");
    FfnArgs a = ffn_args(type, M, D, H, O);
    if (kept_opt && kept_bytes < ffn_kept_bytes(a))
        return fail(IFF_ERR_WORKSPACE, "iff_gated_mlp_forward: kept %zu < %zu bytes", kept_bytes, ffn_kept_bytes(a));
    const size_t need = ffn_forward_workspace(a);
    if (!workspace || workspace_bytes < need)
        return fail(IFF_ERR_WORKSPACE, "iff_gated_mlp_forward: workspace %zu < %zu bytes", workspace_bytes, need);
    IFF_REQUIRE((((uintptr_t)workspace | (uintptr_t)kept_opt) & 15) == 0, "iff_gated_mlp_forward: workspace and kept must be 16-byte aligned");
    a.act = activation; a.x = x; a.w12 = w12; a.b12 = b12_opt; a.w3 = w3; a.b3 = b3_opt; a.y = y; a.kept = kept_opt;
    IFF_HIP(launch_ffn_forward(a, workspace, (hipStream_t)stream));
    return 0;
}
extern "C" size_t iff_gated_mlp_backward_workspace(int32_t type, int64_t M, int32_t D, int32_t H, int32_t O) {
    if (M == 0) return ffn_ok(type, 1, D, H, O) ? ffn_backward_workspace(ffn_args(type, 0, D, H, O)) : 0;
    return ffn_ok(type, M, D, H, O) ? ffn_backward_workspace(ffn_args(type, M, D, H, O)) : 0;
}
extern "C" int iff_gated_mlp_backward(const void* x, int32_t type, int64_t M, int32_t D, int32_t H, int32_t O, const void* w12,
                                      const void* w3, const void* kept, const void* dy, void* dx_opt, void* dw12_opt, void* db12_opt,
                                      void* dw3_opt, void* db3_opt, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_ffn("iff_gated_mlp_backward", type, M, D, H, O)) return rc;
    IFF_REQUIRE(M == 0 || (x && w12 && w3 && kept && dy), "iff_gated_mlp_backward: null buffer");
    const size_t need = iff_gated_mlp_backward_workspace(type, M, D, H, O);
    if (!workspace || workspace_bytes < need)
        return fail(IFF_ERR_WORKSPACE, "iff_gated_mlp_backward: workspace %zu < %zu bytes", workspace_bytes, need);
    IFF_REQUIRE((((uintptr_t)workspace | (uintptr_t)kept) & 15) == 0, "iff_gated_mlp_backward: workspace and kept must be 16-byte aligned");
    FfnArgs a = ffn_args(type, M, D, H, O);
    a.x = x; a.w12 = w12; a.w3 = w3; a.kept = const_cast<void*>(kept); a.dy = dy;
    a.dx = dx_opt; a.dw12 = dw12_opt; a.db12 = db12_opt; a.dw3 = dw3_opt; a.db3 = db3_opt;
    IFF_HIP(launch_ffn_backward(a, workspace, (hipStream_t)stream));
    return 0;
}

extern "C" int iff_dropout(const void* x, int32_t type, int64_t n, const void* residual_opt, int32_t threshold, uint64_t seed,
                           const uint64_t* seed_dev_opt, uint64_t offset, void* y, void* stream) {
    IFF_REQUIRE(block_type(type), "iff_dropout: type %d is not one of IFF_TYPE_F32 / BF16 / F16", type);
    IFF_REQUIRE(n >= 0, "iff_dropout: bad size %lld", (long long)n);
    IFF_REQUIRE(threshold >= 0 && threshold <= 65536, "iff_dropout: threshold %d is not in 0 .. 65536", threshold);
    if (n == 0) return 0;
    IFF_REQUIRE(x && y, "iff_dropout: null buffer");
    const float scale = threshold == 65536 ? 0.0f : 65536.0f / (float)(65536 - threshold);
    IFF_HIP(launch_dropout(type, x, residual_opt, y, n, (uint32_t)threshold, scale, seed, seed_dev_opt, offset, (hipStream_t)stream));
    return 0;
}
