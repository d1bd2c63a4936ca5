// block_kernels.hip -- the memory-bound operators of a trainable transformer block (the backbone that pose_estimation/train.py:97-119
// back-propagates through, pose_estimation/backbone.py:12-14): layer norm with its gradients, and dropout from a counter-based generator.
//
// Layer norm over the last axis of rows x [D]:
//     mean = sum x / D,  var = sum (x - mean)^2 / D,  r = 1 / sqrt(var + eps),  xh = (x - mean) r,  y = xh w + b
//     e = dy w,   dx = r (e - mean(e) - xh mean(e xh)),   dw = sum_rows dy xh,   db = sum_rows dy
// A row is read once into registers (the variance is the second pass over the REGISTERS: no cancellation of E[x^2] - mean^2), so the
// forward pass moves x and y and nothing else; the backward pass moves x, dy and dx.  Both are bound by memory: 65 792 x 1024 bf16 forward
// 54 us (5.0 TB/s), backward 82 us (4.9 TB/s) and 5 for the join of the parameters' shares, where a copy of 2 GB reaches 4.86 TB/s.
#include "block_launch.h"
#include "block_types.h"

#include <algorithm>

namespace {

struct RowView {                       // rows r = (i, j), i < n0, j < n1, at i s0 + j s1 elements: a contiguous tensor, or tokens[:, 1:]
    int64_t s0, s1;
    uint32_t n1;
    __device__ __forceinline__ int64_t at(uint32_t r) const {
        const uint32_t i = r / n1;
        return (int64_t)i * s0 + (int64_t)(r - i * n1) * s1;
    }
};

// weight / bias vector: absent, fp32, or the activations' own type
enum { W_NONE = 0, W_F32 = 1, W_SAME = 2 };
template <class T, int V>
__device__ __forceinline__ void load_par(const void* p, int kind, int c, float v[V], float absent) {
    if (kind == W_SAME) Pack<T, V>::load(reinterpret_cast<const T*>(p) + c, v);
    else if (kind == W_F32) {
        const float* q = reinterpret_cast<const float*>(p) + c;
        if constexpr (V == 1) v[0] = q[0];
        else {
#pragma unroll
            for (int i = 0; i < V; i += 4) Pack<float, 4>::load(q + i, v + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = absent;
    }
}

// sum over the WPR waves that share a row (WPR 1: one wave; 4: the workgroup), every lane gets it.  `s`: 4 floats of LDS per call site
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* s) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    if constexpr (WPR == 4) {
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (s[0] + s[1]) + (s[2] + s[3]);
        __syncthreads();
    }
    return v;
}

// WPR waves per row, NCH chunks of V elements per lane: chunk c of lane t holds columns (c 64 WPR + t) V ...
template <class T, int V, int NCH, int WPR>
__global__ void __launch_bounds__(256) k_layernorm_fwd(const T* __restrict__ x, RowView xv, uint32_t M, int D, const void* __restrict__ w,
                                                       const void* __restrict__ b, int wk, int bk, float eps, T* __restrict__ y,
                                                       float2* __restrict__ stats) {
    constexpr int TPR = 64 * WPR;
    __shared__ float s[4];
    const int t = threadIdx.x % TPR;
    constexpr uint32_t RPB = 4 / WPR;
    for (uint32_t row = blockIdx.x * RPB + (WPR == 1 ? threadIdx.x >> 6 : 0); row < M; row += gridDim.x * RPB) {
        const T* xr = x + xv.at(row);
        float v[NCH][V];
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = (c * TPR + t) * V;
            if (col < D) Pack<T, V>::load(xr + col, v[c]);
            else
#pragma unroll
                for (int i = 0; i < V; ++i) v[c][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) sum += v[c][i];
        }
        const float mean = row_sum<WPR>(sum, s) / (float)D;
        float sq = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
            if ((c * TPR + t) * V < D) {
#pragma unroll
                for (int i = 0; i < V; ++i) { const float d = v[c][i] - mean; sq = fmaf(d, d, sq); }
            }
        const float r = 1.0f / sqrtf(row_sum<WPR>(sq, s) / (float)D + eps);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = (c * TPR + t) * V;
            if (col >= D) continue;
            float g[V], h[V], o[V];
            load_par<T, V>(w, wk, col, g, 1.0f);
            load_par<T, V>(b, bk, col, h, 0.0f);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = fmaf((v[c][i] - mean) * r, g[i], h[i]);
            Pack<T, V>::store(y + (int64_t)row * D + col, o);
        }
        if (stats && t == 0) stats[row] = make_float2(mean, r);
    }
}

// rows of any width: one workgroup per row, the row read three times (from the L2 after the first)
template <class T>
__global__ void __launch_bounds__(256) k_layernorm_fwd_any(const T* __restrict__ x, RowView xv, uint32_t M, int D, const void* __restrict__ w,
                                                           const void* __restrict__ b, int wk, int bk, float eps, T* __restrict__ y,
                                                           float2* __restrict__ stats) {
    __shared__ float s[4];
    for (uint32_t row = blockIdx.x; row < M; row += gridDim.x) {
        const T* xr = x + xv.at(row);
        float sum = 0.0f, sq = 0.0f;
        for (int c = threadIdx.x; c < D; c += 256) sum += (float)xr[c];
        const float mean = row_sum<4>(sum, s) / (float)D;
        for (int c = threadIdx.x; c < D; c += 256) { const float d = (float)xr[c] - mean; sq = fmaf(d, d, sq); }
        const float r = 1.0f / sqrtf(row_sum<4>(sq, s) / (float)D + eps);
        for (int c = threadIdx.x; c < D; c += 256) {
            float g[1], h[1];
            load_par<T, 1>(w, wk, c, g, 1.0f);
            load_par<T, 1>(b, bk, c, h, 0.0f);
            y[(int64_t)row * D + c] = (T)fmaf(((float)xr[c] - mean) * r, g[0], h[0]);
        }
        if (stats && threadIdx.x == 0) stats[row] = make_float2(mean, r);
    }
}

// dx of the rows a workgroup takes (every gridDim-th), and its share of dw / db: part[blockIdx][0] = sum dy xh, [1] = sum dy over its
// rows in increasing order -- k_layernorm_params adds the workgroups' shares in a fixed order, so dw and db are the same bits every run.
template <class T, int V, int NCH, int WPR>
__global__ void __launch_bounds__(256) k_layernorm_bwd(const T* __restrict__ x, RowView xv, const T* __restrict__ dy, uint32_t M, int D,
                                                       const void* __restrict__ w, int wk, const float2* __restrict__ stats,
                                                       T* __restrict__ dx, float* __restrict__ part) {
    constexpr int TPR = 64 * WPR, RPB = 4 / WPR;
    __shared__ float s[4];
    __shared__ float sacc[WPR == 1 ? 4 * 64 * V : 1];
    const int t = threadIdx.x % TPR, wave = threadIdx.x >> 6;
    float aw[NCH][V], ab[NCH][V];
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) aw[c][i] = ab[c][i] = 0.0f;
    // the next row's values are on their way while this one is reduced (raw: half the registers of a 16-bit type's fp32 values)
    typename Raw<T, V>::t rx[NCH], rg[NCH];
    float2 nst = make_float2(0.0f, 0.0f);
    const auto fetch = [&](uint32_t r) {
        const T* xr = x + xv.at(r);
        const T* gr = dy + (int64_t)r * D;
        nst = stats[r];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = (c * TPR + t) * V;
            if (col < D) {
                rx[c] = *reinterpret_cast<const typename Raw<T, V>::t*>(xr + col);
                rg[c] = *reinterpret_cast<const typename Raw<T, V>::t*>(gr + col);
            }
        }
    };
    uint32_t row = blockIdx.x * RPB + (WPR == 1 ? wave : 0);
    if (row < M) fetch(row);
    for (; row < M; row += gridDim.x * RPB) {
        const float2 st = nst;
        float xh[NCH][V], e[NCH][V];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
            if ((c * TPR + t) * V < D) { Raw<T, V>::unpack(rx[c], xh[c]); Raw<T, V>::unpack(rg[c], e[c]); }
        if (row + gridDim.x * RPB < M) fetch(row + gridDim.x * RPB);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = (c * TPR + t) * V;
            if (col < D) {
                float g[V];
                load_par<T, V>(w, wk, col, g, 1.0f);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    xh[c][i] = (xh[c][i] - st.x) * st.y;
                    aw[c][i] = fmaf(e[c][i], xh[c][i], aw[c][i]);
                    ab[c][i] += e[c][i];
                    e[c][i] *= g[i];
                    s1 += e[c][i];
                    s2 = fmaf(e[c][i], xh[c][i], s2);
                }
            }
        }
        if (dx) {
            const float m1 = row_sum<WPR>(s1, s) / (float)D, m2 = row_sum<WPR>(s2, s) / (float)D;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int col = (c * TPR + t) * V;
                if (col >= D) continue;
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = st.y * (e[c][i] - m1 - xh[c][i] * m2);
                Pack<T, V>::store(dx + (int64_t)row * D + col, o);
            }
        }
    }
    if (!part) return;
    float* pw = part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const float* a = which ? ab[c] : aw[c];
            if constexpr (WPR == 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < V; ++i) sacc[wave * 64 * V + t * V + i] = a[i];
                __syncthreads();
                for (int j = threadIdx.x; j < 64 * V; j += 256) {
                    const int col = c * 64 * V + j;
                    if (col < D) pw[which * D + col] = (sacc[j] + sacc[64 * V + j]) + (sacc[2 * 64 * V + j] + sacc[3 * 64 * V + j]);
                }
            } else {
                const int col = (c * TPR + t) * V;
                if (col < D)
#pragma unroll
                    for (int i = 0; i < V; ++i) pw[which * D + col + i] = a[i];
            }
        }
}

// any width: dx one workgroup per row
template <class T>
__global__ void __launch_bounds__(256) k_layernorm_dx_any(const T* __restrict__ x, RowView xv, const T* __restrict__ dy, uint32_t M, int D,
                                                          const void* __restrict__ w, int wk, const float2* __restrict__ stats,
                                                          T* __restrict__ dx) {
    __shared__ float s[4];
    for (uint32_t row = blockIdx.x; row < M; row += gridDim.x) {
        const T* xr = x + xv.at(row);
        const T* gr = dy + (int64_t)row * D;
        const float2 st = stats[row];
        float s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < D; c += 256) {
            float g[1];
            load_par<T, 1>(w, wk, c, g, 1.0f);
            const float e = (float)gr[c] * g[0];
            s1 += e;
            s2 = fmaf(e, ((float)xr[c] - st.x) * st.y, s2);
        }
        const float m1 = row_sum<4>(s1, s) / (float)D, m2 = row_sum<4>(s2, s) / (float)D;
        for (int c = threadIdx.x; c < D; c += 256) {
            float g[1];
            load_par<T, 1>(w, wk, c, g, 1.0f);
            const float xh = ((float)xr[c] - st.x) * st.y;
            dx[(int64_t)row * D + c] = (T)(st.y * ((float)gr[c] * g[0] - m1 - xh * m2));
        }
    }
}
// any width: the shares of dw / db, a thread per column, the rows of block y in increasing order
template <class T>
__global__ void __launch_bounds__(256) k_layernorm_part_any(const T* __restrict__ x, RowView xv, const T* __restrict__ dy, uint32_t M, int D,
                                                            const float2* __restrict__ stats, float* __restrict__ part) {
    const int64_t col = blockIdx.x * (int64_t)256 + threadIdx.x;
    if (col >= D) return;
    float aw = 0.0f, ab = 0.0f;
    for (uint32_t row = blockIdx.y; row < M; row += gridDim.y) {
        const float2 st = stats[row];
        const float g = (float)dy[(int64_t)row * D + col];
        aw = fmaf(g, ((float)x[xv.at(row) + col] - st.x) * st.y, aw);
        ab += g;
    }
    part[(int64_t)blockIdx.y * 2 * D + col] = aw;
    part[(int64_t)blockIdx.y * 2 * D + D + col] = ab;
}

template <class T>
__device__ __forceinline__ void put_par(void* p, int kind, int64_t c, float v) {
    if (kind == W_F32) reinterpret_cast<float*>(p)[c] = v;
    else reinterpret_cast<T*>(p)[c] = (T)v;
}
// dw[c], db[c] = sum over the G shares: 16 columns x 64 groups of shares per workgroup, groups joined in order (a thread then waits for
// G / 64 loads: 11 us with 16 groups of 512 shares, 5 with 64)
template <class T>
__global__ void __launch_bounds__(1024) k_layernorm_params(const float* __restrict__ part, int G, int D, void* __restrict__ dw,
                                                           void* __restrict__ db, int kind) {
    __shared__ float s[64][17];
    const int c16 = threadIdx.x & 15, grp = threadIdx.x >> 4;
    const int64_t c = blockIdx.x * (int64_t)16 + c16;          // over dw's columns, then db's
    const int64_t W = 2 * (int64_t)D;
    float a = 0.0f;
    if (c < W)
#pragma unroll 8
        for (int g = grp; g < G; g += 64) a += part[g * W + c];
    s[grp][c16] = a;
    __syncthreads();
    if (grp == 0 && c < W) {
        float v = s[0][c16];
        for (int j = 1; j < 64; ++j) v += s[j][c16];
        if (c < D) { if (dw) put_par<T>(dw, kind, c, v); }
        else if (db) put_par<T>(db, kind, c - D, v);
    }
}

// ------------------------------------------------------------------------------------------------ dropout
// Philox 4x32, 10 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): counter (block, block >> 32,
// offset, offset >> 32), key (seed, seed >> 32).  Value i takes 16 bits of block i / 8 -- bits 16 (i % 2) ... of word (i % 8) / 2 -- and is
// kept where they are >= threshold = round(65536 p): 16 bits set p to 2^-17 and halve the generator's 20 wide multiplications per value, which
// keeps the launch bound by memory (16448 x 1536 fp32 with residual: forward and backward 48 us each on average, 5.2 TB/s).
__device__ __forceinline__ void philox10(uint64_t block, uint64_t offset, uint64_t seed, uint32_t out[4]) {
    uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32), c = (uint32_t)offset, d = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t pa = (uint64_t)a * 0xD2511F53u, pc = (uint64_t)c * 0xCD9E8D57u;
        a = (uint32_t)(pc >> 32) ^ b ^ k0; b = (uint32_t)pc;
        c = (uint32_t)(pa >> 32) ^ d ^ k1; d = (uint32_t)pa;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    out[0] = a; out[1] = b; out[2] = c; out[3] = d;
}

// y = residual + keep x scale: a thread takes one block of the generator, 8 values.  A dropped value is never multiplied (an infinity or
// a NaN there does not reach y).  VECTOR: 16-byte accesses (every pointer 16-byte aligned)
template <class T, bool VECTOR>
__global__ void __launch_bounds__(256) k_dropout(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y, int64_t n,
                                                 uint32_t threshold, float scale, uint64_t seed, const uint64_t* __restrict__ seed_dev,
                                                 uint64_t offset) {
    constexpr int V = VECTOR ? 16 / (int)sizeof(T) : 1;
    if (seed_dev) seed = *seed_dev;
    const int64_t blocks = (n + 7) >> 3;
    for (int64_t k = blockIdx.x * (int64_t)256 + threadIdx.x; k < blocks; k += (int64_t)gridDim.x * 256) {
        uint32_t r[4];
        philox10((uint64_t)k, offset, seed, r);
        const int64_t i0 = k * 8;
        if (i0 + 8 <= n) {
            float v[8], q[8];
#pragma unroll
            for (int i = 0; i < 8; i += V) {
                Pack<T, V>::load(x + i0 + i, v + i);
                if (res) Pack<T, V>::load(res + i0 + i, q + i);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t bits = (r[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
                const float base = res ? q[i] : 0.0f;
                v[i] = bits >= threshold ? (res ? fmaf(v[i], scale, base) : v[i] * scale) : base;
            }
#pragma unroll
            for (int i = 0; i < 8; i += V) Pack<T, V>::store(y + i0 + i, v + i);
        } else {
            for (int i = 0; i0 + i < n; ++i) {
                const uint32_t word = i < 2 ? r[0] : i < 4 ? r[1] : i < 6 ? r[2] : r[3];
                const uint32_t bits = (word >> (16 * (i & 1))) & 0xFFFFu;
                const float xv = (float)x[i0 + i], base = res ? (float)res[i0 + i] : 0.0f;
                y[i0 + i] = (T)(bits >= threshold ? (res ? fmaf(xv, scale, base) : xv * scale) : base);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ launchers
// The widest row a variant holds in registers is 32 elements per lane: 16-byte chunks where D and every pointer and stride allow,
// single elements otherwise; one wave per row while 4 (16-byte) chunks per lane reach, the workgroup's four waves after that.
struct NormShape { bool vec; int wpr, nch; };              // nch 0: no register form (k_layernorm_*_any)
inline NormShape norm_shape(int dt, int D, bool aligned) {
    const int V = 16 / (int)dt_size(dt);
    const bool vec = aligned && D % V == 0;
    const int v = vec ? V : 1, most = vec ? 32 / V : 16;
    for (int wpr = 1; wpr <= 4; wpr += 3)
        for (int nch = vec ? 1 : 2; nch <= most; nch *= 2)
            if ((int64_t)64 * wpr * v * nch >= D && !(wpr == 4 && nch * 4 < most)) return {vec, wpr, nch};
    return {false, 4, 0};
}

inline uint32_t norm_grid(uint32_t wgs) { return std::min<uint32_t>(wgs, 1u << 22); }      // (a launch has fewer than 2^32 threads)

template <class T, int V, int NCH, int WPR>
void fwd_go(const NormArgs& a, RowView xv, hipStream_t s) {
    k_layernorm_fwd<T, V, NCH, WPR><<<norm_grid(WPR == 1 ? (a.rows + 3) / 4 : a.rows), 256, 0, s>>>((const T*)a.x, xv, a.rows, a.D, a.w, a.b, a.wk, a.bk, a.eps,
                                                                                     (T*)a.y, (float2*)a.stats);
}
template <class T, int V, int NCH, int WPR>
void bwd_go(const NormArgs& a, RowView xv, int G, float* part, hipStream_t s) {
    k_layernorm_bwd<T, V, NCH, WPR><<<G, 256, 0, s>>>((const T*)a.x, xv, (const T*)a.dy, a.rows, a.D, a.w, a.wk, (const float2*)a.stats, (T*)a.dx, part);
}
// GO(V, NCH, WPR) over the forms norm_shape can return
#define NORM_FORMS(T, sh, GO)                                                                       \
    do {                                                                                            \
        constexpr int VV = 16 / (int)sizeof(T);                                                     \
        if (sh.vec) {                                                                               \
            if (sh.wpr == 1) {                                                                      \
                if (sh.nch == 1) GO(VV, 1, 1); else if (sh.nch == 2) GO(VV, 2, 1); else if (sh.nch == 4) GO(VV, 4, 1); else GO(VV, 32 / VV, 1); \
            } else { if (sh.nch == 32 / VV) GO(VV, 32 / VV, 4); else if (sh.nch == 16 / VV) GO(VV, 16 / VV, 4); else GO(VV, 8 / VV, 4); } \
        } else if (sh.wpr == 1) {                                                                   \
            if (sh.nch == 2) GO(1, 2, 1); else if (sh.nch == 4) GO(1, 4, 1); else if (sh.nch == 8) GO(1, 8, 1); else GO(1, 16, 1); \
        } else { if (sh.nch == 16) GO(1, 16, 4); else if (sh.nch == 8) GO(1, 8, 4); else GO(1, 4, 4); } \
    } while (0)

template <class T>
hipError_t norm_fwd(const NormArgs& a, hipStream_t s) {
    const RowView xv{a.s0, a.s1, a.n1};
    const int V = 16 / (int)sizeof(T);
    const bool al = aligned16(a.x) && aligned16(a.y) && aligned16(a.w) && aligned16(a.b) && a.s0 % V == 0 && a.s1 % V == 0;
    const NormShape sh = norm_shape(a.dt, a.D, al);
    if (!sh.nch) k_layernorm_fwd_any<T><<<norm_grid(a.rows), 256, 0, s>>>((const T*)a.x, xv, a.rows, a.D, a.w, a.b, a.wk, a.bk, a.eps, (T*)a.y, (float2*)a.stats);
    else {
#define GO(v, n, p) fwd_go<T, v, n, p>(a, xv, s)
        NORM_FORMS(T, sh, GO);
#undef GO
    }
    return hipGetLastError();
}
template <class T>
hipError_t norm_bwd(const NormArgs& a, float* part, hipStream_t s) {
    const RowView xv{a.s0, a.s1, a.n1};
    const int V = 16 / (int)sizeof(T);
    const bool al = aligned16(a.x) && aligned16(a.dy) && aligned16(a.dx) && aligned16(a.w) && a.s0 % V == 0 && a.s1 % V == 0;
    const NormShape sh = norm_shape(a.dt, a.D, al);
    const bool params = a.dw || a.db;
    const int G = norm_bwd_groups(a.rows);
    if (a.rows) {
        if (!sh.nch) {
            if (a.dx) k_layernorm_dx_any<T><<<norm_grid(a.rows), 256, 0, s>>>((const T*)a.x, xv, (const T*)a.dy, a.rows, a.D, a.w, a.wk, (const float2*)a.stats, (T*)a.dx);
            if (params)
                k_layernorm_part_any<T><<<dim3((a.D + 255) / 256, G), 256, 0, s>>>((const T*)a.x, xv, (const T*)a.dy, a.rows, a.D,
                                                                                   (const float2*)a.stats, part);
        } else {
#define GO(v, n, p) bwd_go<T, v, n, p>(a, xv, G, params ? part : nullptr, s)
            NORM_FORMS(T, sh, GO);
#undef GO
        }
    }
    if (params)
        k_layernorm_params<T><<<(int)((2 * (int64_t)a.D + 15) / 16), 1024, 0, s>>>(part, a.rows ? G : 0, a.D, a.dw, a.db, a.dwk);
    return hipGetLastError();
}

template <class T>
hipError_t dropout_go(const void* x, const void* res, void* y, int64_t n, uint32_t threshold, float scale, uint64_t seed, const uint64_t* seed_dev,
                      uint64_t offset, hipStream_t s) {
    const int64_t blocks = (n + 7) / 8;
    const int grid = (int)std::min<int64_t>((blocks + 255) / 256, 8192);
    if (aligned16(x) && aligned16(res) && aligned16(y))
        k_dropout<T, true><<<grid, 256, 0, s>>>((const T*)x, (const T*)res, (T*)y, n, threshold, scale, seed, seed_dev, offset);
    else
        k_dropout<T, false><<<grid, 256, 0, s>>>((const T*)x, (const T*)res, (T*)y, n, threshold, scale, seed, seed_dev, offset);
    return hipGetLastError();
}

}  // namespace

// four workgroups per CU (65 792 x 1024 bf16: 82 us, 91 with two), each with at least 8 rows (3724 x 1001 fp16: 17 us with 512, 22 with 1024)
int norm_bwd_groups(uint32_t rows) { return (int)std::min<uint32_t>((rows + 7) / 8, 1024); }

hipError_t launch_layernorm_fwd(const NormArgs& a, hipStream_t s) {
    if (!a.rows || !a.D) return hipSuccess;
    return a.dt == IFF_DT_F32 ? norm_fwd<float>(a, s) : a.dt == IFF_DT_BF16 ? norm_fwd<__bf16>(a, s) : norm_fwd<_Float16>(a, s);
}
hipError_t launch_layernorm_bwd(const NormArgs& a, float* part, hipStream_t s) {
    return a.dt == IFF_DT_F32 ? norm_bwd<float>(a, part, s) : a.dt == IFF_DT_BF16 ? norm_bwd<__bf16>(a, part, s) : norm_bwd<_Float16>(a, part, s);
}
hipError_t launch_dropout(int dt, const void* x, const void* res, void* y, int64_t n, uint32_t threshold, float scale, uint64_t seed,
                          const uint64_t* seed_dev, uint64_t offset, hipStream_t s) {
    if (!n) return hipSuccess;
    return dt == IFF_DT_F32 ? dropout_go<float>(x, res, y, n, threshold, scale, seed, seed_dev, offset, s)
         : dt == IFF_DT_BF16 ? dropout_go<__bf16>(x, res, y, n, threshold, scale, seed, seed_dev, offset, s)
                             : dropout_go<_Float16>(x, res, y, n, threshold, scale, seed, seed_dev, offset, s);
}
