// block_launch.h -- host-side launcher prototypes of the trainable block operators, shared between their kernels and block_api.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// block_kernels.hip -- layer norm with its gradients, dropout (the backbone's trainable blocks, pose_estimation/train.py:97-119)
struct NormArgs {
    int dt;                               // IFF_TYPE_*: type of x, y, dy, dx
    const void* x; int64_t s0, s1; uint32_t n1, rows;      // row (i, j) of x at i s0 + j s1 elements, j < n1, rows in all
    int D;
    const void* w; const void* b; int wk, bk;              // 0 absent, 1 fp32, 2 the type of x
    float eps;
    void* y; void* stats;                 // stats [rows][2] = (mean, 1 / sqrt(var + eps))
    const void* dy; void* dx; void* dw; void* db;          // backward only; dx, dw, db nullable
    int dwk;                              // 1: dw, db in fp32, 2: in the type of x
};
int norm_bwd_groups(uint32_t rows);       // workgroups of the backward pass: the shares of dw / db are [groups][2][D] floats
hipError_t launch_layernorm_fwd(const NormArgs& a, hipStream_t s);
hipError_t launch_layernorm_bwd(const NormArgs& a, float* part, hipStream_t s);
hipError_t launch_dropout(int dt, const void* x, const void* res, void* y, int64_t n, uint32_t threshold, float scale, uint64_t seed,
                          const uint64_t* seed_dev, uint64_t offset, hipStream_t s);

// ffn_kernels.hip -- the gated feed-forward block with its gradients
struct FfnArgs {
    int dt, act;                          // IFF_TYPE_*, IFF_ACT_*
    int64_t M; int D, H, O;
    const void* x; const void* w12; const void* b12; const void* w3; const void* b3;
    void* y;
    void* kept;                           // what the backward pass reads (ffn_kept_bytes), null when there is none
    const void* dy; void* dx; void* dw12; void* db12; void* dw3; void* db3;
};
size_t ffn_kept_bytes(const FfnArgs& a);
size_t ffn_forward_workspace(const FfnArgs& a);
size_t ffn_backward_workspace(const FfnArgs& a);
hipError_t launch_ffn_forward(const FfnArgs& a, void* ws, hipStream_t s);
hipError_t launch_ffn_backward(const FfnArgs& a, void* ws, hipStream_t s);
