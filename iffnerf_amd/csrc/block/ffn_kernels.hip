// ffn_kernels.hip -- the gated feed-forward block of a trainable backbone (pose_estimation/train.py:97-119 back-propagates through
// pose_estimation/backbone.py:12-14), forward and backward:
//     [g | u] = x W12^T + b12,   h = act(g) u,   y = h W3^T + b3                    x [M][D], W12 [2H][D], W3 [O][H]
//     q = act(g), p = u act'(g):  dh = dy W3,  dg = dh p,  du = dh q
//     dx = [dg | du] W12,  dW12 = [dg | du]^T x,  dW3 = dy^T h,  db12 = sum_m [dg | du],  db3 = sum_m dy
// Six matrix products on one tile kernel; both projections, the activation and the product of the first are ONE launch (the gate and the
// up column of a hidden unit sit in the same lane's accumulators), and so are dh and the products with its two factors.
// The forward pass keeps h in the operand type (it is the second product's operand) and p, q in fp32: rounding them too would add a
// third rounding between dy and dx (against 64 bits: 2.1 roundings' worth instead of 1.4).
#include "block_launch.h"
#include "block_types.h"
#include "ffn_plan.h"

#include <algorithm>
#include <type_traits>

namespace {

enum { ACT_SILU = 0, ACT_GELU = 1 };

// act(g) and act'(g)
template <bool EXACT>
__device__ __forceinline__ void activation(int act, float g, float& f, float& df) {
    if (act == ACT_SILU) {                         // s = 1 / (1 + e^-g), act = g s, act' = s + g s (1 - s)
        const float s = EXACT ? 1.0f / (1.0f + expf(-g)) : __builtin_amdgcn_rcpf(1.0f + __expf(-g));
        f = g * s;
        df = fmaf(f, 1.0f - s, s);
    } else {                                       // c = (1 + erf(g / sqrt 2)) / 2, act = g c, act' = c + g e^(-g^2/2) / sqrt(2 pi)
        const float c = 0.5f * erfcf(-0.70710678118654752440f * g);
        f = g * c;
        df = fmaf(g * 0.39894228040143267794f, EXACT ? expf(-0.5f * g * g) : __expf(-0.5f * g * g), c);
    }
}

// ------------------------------------------------------------------------------------------------ operands
// The matrix cores' element of a type and the number of planes an operand of it has.  fp32 is multiplied as three bf16 planes
// a = a0 + a1 + a2 (8 bits of the significand each, by truncation: exact) and the six plane products whose weight is above 2^-24.
template <class T> struct Mat { typedef __bf16 e; static constexpr int P = 3; };
template <> struct Mat<__bf16> { typedef __bf16 e; static constexpr int P = 1; };
template <> struct Mat<_Float16> { typedef _Float16 e; static constexpr int P = 1; };
template <class E> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 t; };
template <> struct Vec8<_Float16> { typedef f16x8 t; };
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float trunc_bf16(float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); }
template <class T>
__device__ __forceinline__ void pieces(float v, typename Mat<T>::e out[Mat<T>::P]) {
    if constexpr (Mat<T>::P == 1) out[0] = (typename Mat<T>::e)v;
    else {
        // An infinity is (the largest finite value, 0, infinity) with its sign: the third piece meets one other piece alone, the first of the
        // other operand, which is 0 only where that operand is -- in the first piece it would meet pieces of 0 and end as a NaN.  The finite
        // first piece brings another infinity's third to bear (inf x inf); all its products have the sign of the infinite one.  NaN likewise.
        const bool ok = __builtin_isfinite(v);
        const float a = ok ? trunc_bf16(v) : copysignf(__uint_as_float(0x7F7F0000u), v), r = ok ? v - a : 0.0f, b = trunc_bf16(r);
        out[0] = (__bf16)a; out[1] = (__bf16)b; out[2] = (__bf16)(ok ? r - b : v);
    }
}

// A row-major operand as the tile kernel reads it: planes of [rows][ld] elements, ld a multiple of 8, 16-byte aligned; the columns behind
// its width (fewer than 8) are zero.  A 16-bit tensor of such a shape is its own operand; any other is packed into the workspace first.
struct Operand { const void* p; int64_t ld, plane; };

// four consecutive values of a row as operand planes / as T
template <class T>
__device__ __forceinline__ void store_planes(typename Mat<T>::e* o, int64_t plane, const float v[4]) {
    typedef typename Mat<T>::e E;
    typedef E E4 __attribute__((ext_vector_type(4)));
    constexpr int P = Mat<T>::P;
    E4 t[P];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        E e[P];
        pieces<T>(v[i], e);
#pragma unroll
        for (int p = 0; p < P; ++p) t[p][i] = e[p];
    }
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<E4*>(o + p * plane) = t[p];
}
// what store_planes of a 16-bit type left of four values (nothing of an infinity or a NaN)
template <class T>
__device__ __forceinline__ void store_rest(T* o, const float v[4]) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float r = (float)(T)v[i];
        t[i] = (T)(__builtin_isfinite(r) ? v[i] - r : 0.0f);
    }
    *reinterpret_cast<T4*>(o) = t;
}
template <class T>
__device__ __forceinline__ void store4(T* o, const float v[4]) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<T4*>(o) = T4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
}

// Up to six matrices in one launch, job j from workgroup first[j] on: src [halves x R][C] -> planes [P][halves x RP][CP], zeros behind
// column C and behind row R of a half; 8 columns per thread
// With `finite` infinities and NaN leave as zeros.
struct PackJob { const void* src; void* dst; int64_t R, RP, C, CP, rows_out; int vec, finite; };
struct PackJobs { PackJob job[6]; unsigned first[7]; int n; };
template <class T>
__global__ void __launch_bounds__(256) k_ffn_pack(PackJobs jobs) {
    typedef typename Mat<T>::e E;
    typedef typename Vec8<E>::t E8;
    constexpr int P = Mat<T>::P;
    int k = 0;
    while (k + 1 < jobs.n && blockIdx.x >= jobs.first[k + 1]) ++k;
    const PackJob j = jobs.job[k];
    const unsigned wgs = jobs.first[k + 1] - jobs.first[k];
    const int64_t cols8 = j.CP / 8, n = j.rows_out * cols8;
    E* const dst = reinterpret_cast<E*>(j.dst);
    for (int64_t t = (blockIdx.x - jobs.first[k]) * (int64_t)256 + threadIdx.x; t < n; t += (int64_t)wgs * 256) {
        const int64_t row = n < (1ll << 31) ? (int64_t)((uint32_t)t / (uint32_t)cols8) : t / cols8, c0 = (t - row * cols8) * 8;
        const int64_t half = row >= j.RP, r = row - half * j.RP;
        float v[8];
        const T* s = reinterpret_cast<const T*>(j.src) + (half * j.R + r) * j.C + c0;
        if (j.vec && r < j.R) {
#pragma unroll
            for (int i = 0; i < 8; i += 16 / (int)sizeof(T)) Pack<T, 16 / sizeof(T)>::load(s + i, v + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = r < j.R && c0 + i < j.C ? (float)s[i] : 0.0f;
        }
        if (j.finite)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __builtin_isfinite(v[i]) ? v[i] : 0.0f;
        E8 o[P];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            E e[P];
            pieces<T>(v[i], e);
#pragma unroll
            for (int p = 0; p < P; ++p) o[p][i] = e[p];
        }
#pragma unroll
        for (int p = 0; p < P; ++p) *reinterpret_cast<E8*>(dst + p * j.rows_out * j.CP + row * j.CP + c0) = o[p];
    }
}

// ------------------------------------------------------------------------------------------------ the tile kernel
// C[m][n] = sum_k A(m, k) B(n, k).  KC: an operand's rows are m (or n) and its columns k; KS: its rows are k and its columns m (or n).
enum { KC = 0, KS = 1 };
enum { EPI_OUT = 0, EPI_GATE = 1, EPI_DH = 2 };
struct Prod {
    Operand a, b;
    int64_t ra, rb;                       // rows of a KC operand (reads are clamped to them)
    int64_t M, N, K, k_per_split, m_base;      // a launch covers the rows m_base .. M - 1 of C
    // EPI_OUT: out[row(m)][n] = acc + bias[n], ld N; row(m) = m, or with two halves of `half_pad` padded rows each, of which `half` exist.
    // With `part`: the fp32 share of a split over k instead, part[z][row][n] of rows_out rows
    void* out; const void* bias; float* part; int64_t half_pad, half, rows_out; bool vec_out;
    // EPI_GATE: N = H; B rows n (gate) and up_row + n (up).  out = h planes of ld ldo; factors p, q [M][HP = pad8(H)] or null; bias b12
    // EPI_DH: out = [dg | du] planes of ld ldo, du at column HP
    // and with `sums`: [M / 32 MR][2H] column sums of dg and du (fp32, before they are rounded) over a wave's rows
    int64_t up_row, HP, ldo, plane_o; float* p; float* q; int act; float* sums;
    // EPI_GATE and EPI_DH of a 16-bit type: what rounding row m leaves, itself rounded, this many elements behind it (0: not kept)
    int64_t rest;
};

__device__ __attribute__((aligned(16))) const unsigned int g_zeros[4] = {0, 0, 0, 0};

// 16 bytes per lane from `src` to LDS, lane-linear from byte `lds` on.  TR: as assembly -- behind the builtin the compiler drains the memory
// queue before every transposed LDS read (it takes the two for aliases), which serialised the products with a k-strided operand (dW12 at
// 16448 x 1536 x 4096: 745 against 369 us); beside plain reads the builtin is the faster form (F2: 219 against 245 us).  Nothing is
// returned to a register; the waits are the kernel's own counted ones.  m0 is reserved: a clobber of it means nothing to the compiler, which
// writes it right before each use of its own.  (That there is none in these kernels is tested on the built code.)
template <bool TR>
__device__ __forceinline__ void dma16(const char* src, uint32_t lds) {
    if constexpr (TR) asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory");
    else __builtin_amdgcn_global_load_lds((const void*)src, (__attribute__((address_space(3))) void*)(uintptr_t)lds, 16, 0, 0);
}

// Workgroups are dealt round-robin over the 8 XCDs, each with its own L2.  The ones that share an XCD (ids equal mod 8) take a contiguous
// range of tiles, and that range runs down columns of 8 tiles of m before it moves on in n: what is in flight on an XCD shares operands.
__device__ __forceinline__ void tile_of(unsigned id, unsigned gm, unsigned gn, unsigned& tm, unsigned& tn) {
    const unsigned total = gm * gn, xcd = id & 7, q = total >> 3, r = total & 7;
    unsigned t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (id >> 3);
    const unsigned group = t / (8 * gn), first = group * 8, rows = min(gm - first, 8u);
    t -= group * 8 * gn;
    tm = first + t % rows;
    tn = t / rows;
}

// Tiles of 32 MR WM x 32 NR WN, 64 deep, WM x WN waves of 32 MR x 32 NR.  Operand tiles go from memory to LDS by DMA (16 bytes per lane,
// 1 KB per instruction, lane-linear in LDS) into a ring of NBUF buffers.  A KC tile is rows of 64 k (128 B), its 16-byte chunk c in
// slot c ^ (row / 2 & 7); a KS tile is rows of one k, chunk c in slot c ^ 4 (k & 3) (64 and 192 columns, whose rows are not whole
// 256-byte bank rows: c ^ 2 (k & 2)), and its fragments are read transposed (ds_read_b64_tr_b16).  Both swizzles are applied to the
// lanes' SOURCE addresses and keep the LDS reads free of bank conflicts.  What bounds it: the fill of LDS from L2 (a build that does
// nothing else needs 0.6 - 0.8 of a launch) beside the matrix pipe (0.47 of F2's clocks at 16448 x 1536 x 4096, 217 us).  32-deep rings of
// three to five buffers measured the same or slower, four waves of 128 x 128 17 % slower.
template <class T, int AK, int BK, int EPI, int WM, int WN, int MR, int NR, int NBUF>
__global__ void __launch_bounds__(64 * WM * WN, NBUF > 2 && MR * NR == 4 ? 1 : 2) k_ffn_product(Prod g, unsigned gm, unsigned gn) {
    typedef typename Mat<T>::e E;
    typedef typename Vec8<E>::t E8;
    constexpr int P = Mat<T>::P, NW = WM * WN, BM = 32 * MR * WM, BN = 32 * NR * WN;
    constexpr int KT = 64, ROW = KT * 2, PA = BM * ROW / 1024 / NW, PB = BN * ROW / 1024 / NW;      // 1-KB pieces per wave and step
    constexpr int TILE = (BM + BN) * ROW, GW = 16 * NR;
    constexpr int OLD = 32 * NR + 4;                                  // floats per row of a wave's output tile in LDS: conflict-free 16-byte writes down a column
    constexpr int POOL = NBUF * TILE > NW * 32 * OLD * 4 ? NBUF * TILE : NW * 32 * OLD * 4;
    __shared__ __attribute__((aligned(1024))) char s_all[POOL];
    const uint32_t s_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_all;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 31, lh = lane >> 5;
    const int wm = (wave / WN) * 32 * MR, wn = (wave % WN) * 32 * NR;
    unsigned tm, tn;
    tile_of(blockIdx.x, gm, gn, tm, tn);
    constexpr int NT = EPI == EPI_GATE ? BN / 2 : BN;                 // columns of C per tile (a gate tile: as many gate as up columns)
    const int64_t m0 = g.m_base + (int64_t)tm * BM, n0 = (int64_t)tn * NT;
    const int64_t k_lo = blockIdx.y * g.k_per_split, k_hi = min(g.K, k_lo + g.k_per_split);
    const E* const A = reinterpret_cast<const E*>(g.a.p);
    const E* const B = reinterpret_cast<const E*>(g.b.p);

    const auto swizzle = [](int r) { return (r >> 1) & 7; };
    const auto turn = [](int r, int width) { return width % 128 ? (r & 2) << 1 : (r & 3) << 2; };

    // the lane's source of each piece, in bytes from the tile's corner at the step's k (ld < 2^22: 256 rows stay below 2^31), and its first k
    uint32_t oa[PA], ob[PB];
    int ka[PA], kb[PB];
#pragma unroll
    for (int i = 0; i < PA; ++i) {
        const int at = (wave + NW * i) * 1024 + lane * 16;
        const int r = at / (AK == KC ? ROW : BM * 2), c = ((at % (AK == KC ? ROW : BM * 2)) >> 4) ^ (AK == KC ? swizzle(r) : turn(r, BM));
        if (AK == KC) { oa[i] = (uint32_t)((min(m0 + r, g.ra - 1) - m0) * g.a.ld + c * 8) * 2; ka[i] = c * 8; }
        else { oa[i] = (uint32_t)(r * g.a.ld + min(m0 + c * 8, g.a.ld - 8) - m0) * 2; ka[i] = r; }
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
        const int at = (wave + NW * i) * 1024 + lane * 16;
        const int r = at / (BK == KC ? ROW : BN * 2), c = ((at % (BK == KC ? ROW : BN * 2)) >> 4) ^ (BK == KC ? swizzle(r) : turn(r, BN));
        if (BK == KC) {
            // a gate tile's rows, per wave: GW gate rows, then the up rows of the same hidden units
            const int64_t row = EPI == EPI_GATE ? min(n0 + r / (2 * GW) * GW + r % GW, g.N - 1) : min(n0 + r, g.rb - 1);
            ob[i] = (uint32_t)((row - n0) * g.b.ld + c * 8) * 2;
            kb[i] = c * 8;
        } else { ob[i] = (uint32_t)(r * g.b.ld + min(n0 + c * 8, g.b.ld - 8) - n0) * 2; kb[i] = r; }
    }
    const int64_t sa = AK == KC ? KT : KT * g.a.ld, sb = BK == KC ? KT : KT * g.b.ld;            // elements per step
    const E* const a0 = A + (AK == KC ? m0 * g.a.ld + k_lo : k_lo * g.a.ld + m0);
    const E* const b0 = B + (BK == KC ? n0 * g.b.ld + k_lo : k_lo * g.b.ld + n0);
    const int steps_k = (int)((k_hi - k_lo + KT - 1) / KT), steps = k_hi > k_lo ? steps_k * (P == 3 ? 6 : 1) : 0;

    // the next step to request: planes of the six products, smallest first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0); k values from it on.  Behind the
    // last step `left` is not positive and the pieces are zeros: the queue holds the same number of pieces at every step
    const char* as = reinterpret_cast<const char*>(a0);
    const char* bs = reinterpret_cast<const char*>(b0);
    int pair = 0, kt = 0, head = 0;
    int left = steps ? (int)(k_hi - k_lo) : 0;
    const auto planes = [&]() {
        const int pa = P == 1 ? 0 : pair == 0 ? 2 : pair == 2 || pair == 3 ? 1 : 0, pb = P == 1 ? 0 : pair == 1 ? 2 : pair == 2 || pair == 4 ? 1 : 0;
        as = reinterpret_cast<const char*>(a0 + pa * g.a.plane);
        bs = reinterpret_cast<const char*>(b0 + pb * g.b.plane);
    };
    planes();
    const auto piece = [&](int i) {                                   // i < PA: of A, else of B
        const bool isa = i < PA;
        const int j = isa ? i : i - PA;
        const char* base = isa ? as : bs;
        if (EPI == EPI_GATE && !isa && (((wave + NW * j) * (1024 / ROW) / GW) & 1)) base += g.up_row * g.b.ld * 2;
        const char* src = base + (isa ? oa[j] : ob[j]);
        src = (isa ? ka[j] : kb[j]) < left ? src : reinterpret_cast<const char*>(g_zeros);
        dma16<AK == KS || BK == KS>(src, s_base + (uint32_t)(head * TILE + (isa ? 0 : BM * ROW) + (wave + j * NW) * 1024));
    };
    const auto requested = [&]() {                                    // all pieces of the step are out
        head = head + 1 == NBUF ? 0 : head + 1;
        left -= KT; as += sa * 2; bs += sb * 2;
        if (P == 3 && ++kt == steps_k) {
            kt = 0; ++pair;
            left = pair < 6 ? (int)(k_hi - k_lo) : 0;
            planes();
        }
    };

    // where this lane's fragments are in a tile: KC one 16-byte read per 16 k, KS two transposed 8-byte reads
    constexpr int ROWA = AK == KC ? ROW : BM * 2, ROWB = BK == KC ? ROW : BN * 2;
    const int sw = swizzle(lr), trow = 8 * lh + ((lane & 15) >> 2);
    const int tcol = (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;
    auto frag = [&](const char* tile, int kind, int rowbytes, int base, int j, int ks) -> E8 {
        if (kind == KC) return *reinterpret_cast<const E8*>(tile + (base + 32 * j + lr) * ROW + (((2 * ks + lh) ^ sw) << 4));
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const char* at = tile + (16 * ks + trow) * rowbytes + (((base / 8 + 4 * j) ^ turn(trow, rowbytes / 2)) << 4) + tcol;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 4 * rowbytes));
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        return __builtin_bit_cast(E8, v);
    };

    f32x16 acc[NR][MR];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[n][m][r] = 0.0f;
    // A ring of NBUF buffers.  While a block of 16 k is multiplied the fragments of the next one are read, across the step's border too: before
    // the last block of step t everybody's pieces of step t + 1 have landed (a counted wait -- a __syncthreads would drain the queue -- and
    // the barrier) and step t has been read by everybody, so step t + NBUF is requested into its buffer.  The pieces go out BETWEEN the products
    // of two blocks: a CU drains about 32 bytes per clock into LDS, and a burst of them would hold up the waves' matrix instructions
    struct Frags { E8 a[MR], b[NR]; };
    constexpr int PIECES = PA + PB, FIRST = PIECES / 2;               // pieces of a step before / after the step's border
    const auto read = [&](Frags& f, int i, int buf, int ks) {          // fragment i of the MR + NR of a block
        const char* const ta = s_all + buf * TILE;
        if (i < NR) f.b[i] = frag(ta + BM * ROW, BK, ROWB, wn, i, ks);
        else f.a[i - NR] = frag(ta, AK, ROWA, wm, i - NR, ks);
    };
    // the products of one block; between them, in this order, the reads of the next block (ks of buffer buf) and the pieces p0 .. p1 - 1
    const auto block = [&](const Frags& f, Frags& next, int buf, int ks, int p0, int p1) {
        constexpr int N = MR * NR, R = MR + NR;
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int j = R * i / N; j < R * (i + 1) / N; ++j) read(next, j, buf, ks);
#pragma unroll
            for (int j = p0 + (p1 - p0) * i / N; j < p0 + (p1 - p0) * (i + 1) / N; ++j) piece(j);
            acc[i % NR][i / NR] = mfma(f.b[i % NR], f.a[i / NR], acc[i % NR][i / NR]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    Frags f0, f1;
    if (steps) {
#pragma unroll
        for (int i = 0; i < NBUF; ++i) {
#pragma unroll
            for (int j = 0; j < PIECES; ++j)
                if (i < NBUF - 1 || j < FIRST) piece(j);
            if (i < NBUF - 1) requested();
        }
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NBUF - 2) * PIECES + FIRST) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < MR + NR; ++i) read(f0, i, 0, 0);
    }
    int cur = 0;
    for (int t = 0; t < steps; ++t) {
#pragma unroll
        for (int ks = 0; ks < KT / 16 - 1; ++ks) {
            block(ks & 1 ? f1 : f0, ks & 1 ? f0 : f1, cur, ks + 1, FIRST, ks == 0 ? PIECES : FIRST);      // (the rest of step t + NBUF - 1)
            if (ks == 0) requested();
        }
        const int nxt = cur + 1 == NBUF ? 0 : cur + 1;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NBUF - 2) * PIECES) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        block(f1, f0, nxt, 0, 0, FIRST);                              // (behind the last step: reads of zeros, not used)
        cur = nxt;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                  // the last pieces, before the buffers are used again

    // A lane holds row m = lr of C and columns (reg & 3) + 8 (reg >> 2) + 4 lh of each 32 x 32 block: stored from there an instruction
    // touches 32 rows with 16 bytes each.  Every wave turns its 32-row slices over in LDS instead and works along the rows, 4 columns per lane:
    // whole 128- to 512-byte runs (the direct form cost 76 us of F2's 271, 371 of the gate product's 735 at 16448 x 1536 x 4096)
    const T* const bias = reinterpret_cast<const T*>(g.bias);
    float* const tile = reinterpret_cast<float*>(s_all) + wave * 32 * OLD;
    constexpr int CPL = EPI == EPI_GATE ? GW / 4 : 8 * NR, RPI = 64 / CPL;          // lanes per row, rows per pass
    const int col = (lane % CPL) * 4;
    const int64_t n = n0 + (EPI == EPI_GATE ? wn / 2 : wn) + col;
    float bi[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = bias && n + i < g.N;
        bi[0][i] = in ? (float)bias[n + i] : 0.0f;
        bi[1][i] = in && EPI == EPI_GATE ? (float)bias[g.N + n + i] : 0.0f;
    }
    float sg[4] = {0.0f, 0.0f, 0.0f, 0.0f}, su[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool whole = m0 + BM <= g.M && n0 + NT <= g.N && !g.half_pad && (EPI != EPI_OUT || g.vec_out);
    const auto slice = [&](int mb, int it, auto all_inside, const float* pre) {
        constexpr bool IN = decltype(all_inside)::value;
        const int r = it * RPI + lane / CPL;
        if (64 % CPL && lane >= RPI * CPL) return;                    // (192 columns: 48 lanes work)
        const int64_t m = m0 + wm + 32 * mb + r;
        float v[4];
        Pack<float, 4>::load(tile + r * OLD + col, v);
        if (!IN && m >= g.M) return;
        if constexpr (EPI == EPI_GATE) {
            if (!IN && n >= g.HP) return;
            float u[4], hv[4], pv[4];
            Pack<float, 4>::load(tile + r * OLD + GW + col, u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = IN || n + i < g.N;
                const float gv = v[i] + bi[0][i], uv = u[i] + bi[1][i];
                float f, df;
                activation<P == 3>(g.act, gv, f, df);
                hv[i] = in ? f * uv : 0.0f;
                pv[i] = in ? uv * df : 0.0f;
                v[i] = in ? f : 0.0f;
            }
            E* o = reinterpret_cast<E*>(g.out) + m * g.ldo + n;
            store_planes<T>(o, g.plane_o, hv);
            if (P == 1 && !IN && g.rest) store_rest<E>(o + g.rest, hv);          // (the rows it is kept for never fill a tile)
            if (g.p) {
                Pack<float, 4>::store(g.p + m * g.HP + n, pv);
                Pack<float, 4>::store(g.q + m * g.HP + n, v);
            }
        } else if constexpr (EPI == EPI_DH) {
            if (!IN && n >= g.HP) return;
            float p[4], q[4];
            if (IN) {
#pragma unroll
                for (int i = 0; i < 4; ++i) { p[i] = pre[i]; q[i] = pre[4 + i]; }
            } else {
                Pack<float, 4>::load(g.p + m * g.HP + n, p);
                Pack<float, 4>::load(g.q + m * g.HP + n, q);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = IN || n + i < g.N;
                p[i] = in ? v[i] * p[i] : 0.0f;
                q[i] = in ? v[i] * q[i] : 0.0f;
                sg[i] += p[i];
                su[i] += q[i];
            }
            E* o = reinterpret_cast<E*>(g.out) + m * g.ldo + n;
            store_planes<T>(o, g.plane_o, p);
            store_planes<T>(o + g.HP, g.plane_o, q);
            if (P == 1 && !IN && g.rest) { store_rest<E>(o + g.rest, p); store_rest<E>(o + g.rest + g.HP, q); }
        } else {
            int64_t row = m;
            if (!IN && g.half_pad) {
                const int64_t hf = m >= g.half_pad;
                if (m - hf * g.half_pad >= g.half) return;
                row = hf * g.half + m - hf * g.half_pad;
            }
            const bool vec = IN || (g.vec_out && n < g.N);
            if (g.part) {
                float* o = g.part + (blockIdx.y * g.rows_out + row - g.m_base) * g.N + n;
                if (vec) Pack<float, 4>::store(o, v);
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < g.N) o[i] = v[i];
            } else {
                T* o = reinterpret_cast<T*>(g.out) + row * g.N + n;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += bi[0][i];
                if (vec) store4<T>(o, v);
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < g.N) o[i] = (T)v[i];
            }
        }
    };
    float ahead[4][8];
    const auto factors = [&](int mb, int it) {                        // p and q of four passes from pass `it` on
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t at = (m0 + wm + 32 * mb + (it + i) * RPI + lane / CPL) * g.HP + n;
            Pack<float, 4>::load(g.p + at, ahead[i]);
            Pack<float, 4>::load(g.q + at, ahead[i] + 4);
        }
    };
    if (EPI == EPI_DH && whole) factors(0, 0);
    __syncthreads();                                                  // everybody has read the last fragments
#pragma unroll
    for (int mb = 0; mb < MR; ++mb) {
#pragma unroll
        for (int nb = 0; nb < NR; ++nb)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<f32x4*>(tile + lr * OLD + 32 * nb + 8 * q4 + 4 * lh) =
                    f32x4{acc[nb][mb][4 * q4], acc[nb][mb][4 * q4 + 1], acc[nb][mb][4 * q4 + 2], acc[nb][mb][4 * q4 + 3]};
        // a tile that lies wholly inside C: no checks between the passes, so that their reads and stores overlap; the factors of the next
        // passes are on their way while these are worked on
        constexpr int ITS = 32 / RPI, GROUP = 4;
        if (whole && EPI == EPI_DH) {
#pragma unroll
            for (int g0 = 0; g0 < ITS; g0 += GROUP) {
                float now[GROUP][8];
#pragma unroll
                for (int i = 0; i < GROUP; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) now[i][j] = ahead[i][j];
                const bool last = g0 + GROUP >= ITS;
                if (!last || mb + 1 < MR) factors(last ? mb + 1 : mb, last ? 0 : g0 + GROUP);
#pragma unroll
                for (int i = 0; i < GROUP; ++i) slice(mb, g0 + i, std::true_type{}, now[i]);
            }
        } else if (whole) {
#pragma unroll 4
            for (int it = 0; it < ITS; ++it) slice(mb, it, std::true_type{}, nullptr);
        } else {
#pragma unroll 1
            for (int it = 0; it < ITS; ++it) slice(mb, it, std::false_type{}, nullptr);
        }
    }
    if constexpr (EPI == EPI_DH) {
        if (!g.sums || m0 + wm >= g.M) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int off = CPL; off < 64; off <<= 1) { sg[i] += __shfl_xor(sg[i], off, 64); su[i] += __shfl_xor(su[i], off, 64); }
            if (lane < CPL && n + i < g.N) {
                float* o = g.sums + (m0 + wm) / (32 * MR) * 2 * g.N + n + i;
                o[0] = sg[i];
                o[g.N] = su[i];
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ a few tokens
// At most 8 rows and no gradients (serving token by token): the weights are read once and that is all the time there is, so the products are
// vector dot products -- a wave per RW rows of the weight matrix, its lanes over k, 16 bytes per load, fp32 sums joined across the lanes --
// and not tiles of which 8 of 128 rows would be used.  GATE: RW / 2 hidden units, their gate and their up row; else RW outputs.  The hidden
// activation stays fp32 between the two launches.  One token, 1536 x 4096 bf16: 6 + 4 us, 3.9 TB/s of weights (partly
// from the Infinity Cache where they are read again at once).
template <class T, int V, int MM, int RW, bool GATE, class TX, class TO>
__global__ void __launch_bounds__(256) k_ffn_few(const TX* __restrict__ x, int M, int64_t K, const T* __restrict__ w, int64_t N, const T* __restrict__ bias,
                                                 int act, TO* __restrict__ out) {
    constexpr int VX = V == 1 ? 1 : 16 / (int)sizeof(TX) < V ? 16 / (int)sizeof(TX) : V;
    constexpr int U = GATE ? RW / 2 : RW;                            // columns of the output per wave
    const int lane = threadIdx.x & 63;
    const int64_t n0 = (blockIdx.x * (int64_t)4 + (threadIdx.x >> 6)) * U;
    if (n0 >= N) return;
    const T* row[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) {
        const int64_t n = min(n0 + r % U, N - 1);
        row[r] = w + (GATE && r >= U ? N + n : n) * K;
    }
    float acc[RW][MM];
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int m = 0; m < MM; ++m) acc[r][m] = 0.0f;
#pragma unroll 2
    for (int64_t k = lane * V; k < K; k += 64 * V) {
        float a[RW][V];
#pragma unroll
        for (int r = 0; r < RW; ++r) Pack<T, V>::load(row[r] + k, a[r]);
#pragma unroll
        for (int m = 0; m < MM; ++m) {
            float b[V];
#pragma unroll
            for (int i = 0; i < V; i += VX) Pack<TX, VX>::load(x + min(m, M - 1) * K + k + i, b + i);
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[r][m] = fmaf(a[r][i], b[i], acc[r][m]);
        }
    }
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int m = 0; m < MM; ++m)
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) acc[r][m] += __shfl_xor(acc[r][m], off, 64);
    // lane u MM + m writes output column n0 + u of row m
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < MM; ++m) {
            const int64_t n = n0 + u;
            if (lane != u * MM + m || m >= M || n >= N) continue;
            float v = acc[u][m] + (bias ? (float)bias[n] : 0.0f);
            if constexpr (GATE) {
                const float up = acc[U + u][m] + (bias ? (float)bias[N + n] : 0.0f);
                float f, df;
                activation<Mat<T>::P == 3>(act, v, f, df);
                v = f * up;
            }
            out[m * N + n] = (TO)v;
        }
}

// Sums of shares, every one a call leaves in one launch (a launch of its own costs each of them 5 us of GPU time and 4 of the host's): job j
// from workgroup first[j] on.  Elements: out[i] = sum_z part[z][i] (+ bias of the column) in increasing z.  Columns (many shares, few sums):
// 16 columns x 64 groups of shares per workgroup, a group in increasing order, the groups joined in order.  PAIRS: elements whose odd shares
// are products of what roundings left (product_of_pairs): where the sum is an infinity or a NaN, it is that of the even ones alone.
enum { JOIN_ELEMENTS = 0, JOIN_COLUMNS = 1, JOIN_ELEMENTS4 = 2 };      // (the last: four at a time, where N and out allow it)
struct JoinJob { const float* part; void* out; const void* bias; int64_t n, N; int Z, kind; bool pairs; };
struct JoinJobs { JoinJob job[6]; unsigned first[7]; int n; };
__device__ __forceinline__ float even_shares(const JoinJob& j, int64_t i) {
    float v = j.part[i];
    for (int z = 2; z < j.Z; z += 2) v += j.part[z * j.n + i];
    return v;
}
template <class T>
__global__ void __launch_bounds__(1024) k_ffn_join(JoinJobs jobs) {
    __shared__ float s[64][17];
    int k = 0;
    while (k + 1 < jobs.n && blockIdx.x >= jobs.first[k + 1]) ++k;
    const JoinJob j = jobs.job[k];
    const unsigned wg = blockIdx.x - jobs.first[k], wgs = jobs.first[k + 1] - jobs.first[k];
    T* const out = reinterpret_cast<T*>(j.out);
    if (j.kind == JOIN_ELEMENTS4) {
        const T* const bias = reinterpret_cast<const T*>(j.bias);
        for (int64_t i = (wg * (int64_t)1024 + threadIdx.x) * 4; i < j.n; i += (int64_t)wgs * 4096) {
            float v[4], t[4];
            Pack<float, 4>::load(j.part + i, v);
#pragma unroll 4
            for (int z = 1; z < j.Z; ++z) {
                Pack<float, 4>::load(j.part + z * j.n + i, t);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += t[e];
            }
            if (j.pairs && !(__builtin_isfinite(v[0]) & __builtin_isfinite(v[1]) & __builtin_isfinite(v[2]) & __builtin_isfinite(v[3])))
#pragma unroll 1
                for (int e = 0; e < 4; ++e) {                         // (one loop, not four: the code it sits in is 8 % slower with those)
                    const float even = even_shares(j, i + e);
                    v[0] = e == 0 && !__builtin_isfinite(v[0]) ? even : v[0];
                    v[1] = e == 1 && !__builtin_isfinite(v[1]) ? even : v[1];
                    v[2] = e == 2 && !__builtin_isfinite(v[2]) ? even : v[2];
                    v[3] = e == 3 && !__builtin_isfinite(v[3]) ? even : v[3];
                }
            if (bias)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += (float)bias[i % j.N + e];
            store4<T>(out + i, v);
        }
        return;
    }
    if (j.kind == JOIN_ELEMENTS) {
        const T* const bias = reinterpret_cast<const T*>(j.bias);
        for (int64_t i = wg * (int64_t)1024 + threadIdx.x; i < j.n; i += (int64_t)wgs * 1024) {
            float v = j.part[i];
            for (int z = 1; z < j.Z; ++z) v += j.part[z * j.n + i];
            if (j.pairs && !__builtin_isfinite(v)) v = even_shares(j, i);
            out[i] = (T)(bias ? v + (float)bias[i % j.N] : v);
        }
        return;
    }
    const int c16 = threadIdx.x & 15, grp = threadIdx.x >> 4;
    const int64_t c = wg * (int64_t)16 + c16;
    float a = 0.0f;
    if (c < j.n)
#pragma unroll 8
        for (int g = grp; g < j.Z; g += 64) a += j.part[g * j.n + c];
    s[grp][c16] = a;
    __syncthreads();
    if (grp == 0 && c < j.n) {
        for (int i = 1; i < 64; ++i) a += s[i][c16];
        out[c] = (T)a;
    }
}

// shares of the column sums of a [M][N] matrix: part[y][n] over the rows of block y (every gridDim.y-th group of 8); V columns per thread
template <class T, int V>
__global__ void __launch_bounds__(256) k_ffn_colsum(const T* __restrict__ a, int64_t M, int64_t N, float* __restrict__ part) {
    __shared__ float s[8][32 * V + 1];
    const int c = (threadIdx.x & 31) * V, r8 = threadIdx.x >> 5;
    const int64_t n = blockIdx.x * (int64_t)(32 * V) + c;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.0f;
    if (n < N)
#pragma unroll 4
        for (int64_t m = blockIdx.y * (int64_t)8 + r8; m < M; m += (int64_t)gridDim.y * 8) {
            float t[V];
            Pack<T, V>::load(a + m * N + n, t);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += t[i];
        }
#pragma unroll
    for (int i = 0; i < V; ++i) s[r8][c + i] = v[i];
    __syncthreads();
    for (int j = threadIdx.x; j < 32 * V; j += 256) {
        float t = s[0][j];
        for (int r = 1; r < 8; ++r) t += s[r][j];
        if (blockIdx.x * (int64_t)(32 * V) + j < N) part[blockIdx.y * N + blockIdx.x * (int64_t)(32 * V) + j] = t;
    }
}

// ------------------------------------------------------------------------------------------------ launches

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// the workspace, handed out front to back; with base null only its size is counted and nothing is launched
struct Work {
    char* base; size_t used; hipStream_t s;
    void* take(size_t bytes) { void* p = base ? base + used : nullptr; used += up256(bytes); return p; }
    bool counting() const { return !base; }
};
#define FFN_TRY(call) do { const hipError_t e__ = (call); if (e__ != hipSuccess) return e__; } while (0)

template <class T> inline size_t planes_bytes(int64_t rows, int64_t ld) { return (size_t)rows * ld * Mat<T>::P * 2; }

// the matrices a call multiplies, each as itself or packed by one launch for all of them
template <class T>
struct Packer {
    Work& w;
    PackJobs jobs{};
    explicit Packer(Work& work) : w(work) {}
    // src [halves x R][C]; where the size is counted the copy is too (whether a start is 16-byte aligned must not change it).  `times`: the
    // rows that many times over (16-bit types), finite values alone after the first: what they are multiplied with there is what a rounding
    // left, often 0, and an infinity's product is the first copy's to give
    Operand add(const void* src, int64_t halves, int64_t R, int64_t C, int times = 1) {
        const int64_t RP = halves > 1 ? pad8(R) : R, CP = pad8(C), rows = halves * RP;
        if (Mat<T>::P == 1 && CP == C && RP == R && times == 1 && !w.counting() && aligned16(src)) return {src, CP, rows * CP};
        char* dst = (char*)w.take(planes_bytes<T>(times * rows, CP));
        for (int i = 0; i < times && !w.counting() && rows; ++i) {
            const int64_t n = rows * CP / 8;
            jobs.job[jobs.n] = {src, dst + i * planes_bytes<T>(rows, CP), R, RP, C, CP, rows, aligned16(src) && CP == C, i > 0};
            jobs.first[jobs.n + 1] = jobs.first[jobs.n] + (unsigned)std::min<int64_t>((n + 255) / 256, 4096);
            ++jobs.n;
        }
        return {dst, CP, times * rows * CP};
    }
    hipError_t go() {
        if (!jobs.n) return hipSuccess;
        k_ffn_pack<T><<<jobs.first[jobs.n], 256, 0, w.s>>>(jobs);
        return hipGetLastError();
    }
};

template <class T, int AK, int BK, int EPI, int WM, int WN, int MR, int NR, int NBUF>
hipError_t tiles(Prod g, int splits, hipStream_t s) {
    constexpr int BM = 32 * MR * WM, NT = EPI == EPI_GATE ? 16 * NR * WN : 32 * NR * WN;
    const int64_t N = EPI == EPI_OUT ? g.N : g.HP, gm = (g.M - g.m_base + BM - 1) / BM, gn = (N + NT - 1) / NT;
    if (gm <= 0 || !gn) return hipSuccess;
    if (gm * gn >= (1ll << 32) / (64 * WM * WN)) return hipErrorInvalidConfiguration;      // (a launch has fewer than 2^32 threads)
    g.k_per_split = splits > 1 ? ((g.K + splits - 1) / splits + 63) / 64 * 64 : std::max<int64_t>(g.K, 64);
    k_ffn_product<T, AK, BK, EPI, WM, WN, MR, NR, NBUF><<<dim3((unsigned)(gm * gn), splits), 64 * WM * WN, 0, s>>>(g, (unsigned)gm, (unsigned)gn);
    return hipGetLastError();
}
template <class T, int AK, int BK, int EPI>
hipError_t launch_shape(int shape, const Prod& g, int splits, hipStream_t s) {
    switch (shape) {
    case SHAPE_256: return tiles<T, AK, BK, EPI, 4, 2, 2, 4, 2>(g, splits, s);
    case SHAPE_192:
        if constexpr (AK == KS) return tiles<T, AK, BK, EPI, 4, 2, 2, 3, 2>(g, splits, s);
        else return hipErrorInvalidConfiguration;
    case SHAPE_128: return tiles<T, AK, BK, EPI, 2, 2, 2, 2, 2>(g, splits, s);
    case SHAPE_128_DEEP: return tiles<T, AK, BK, EPI, 2, 2, 2, 2, 4>(g, splits, s);
    default: return tiles<T, AK, BK, EPI, 2, 2, 1, 1, 4>(g, splits, s);
    }
}
// the sums of shares that a call's launches leave, taken by one launch at its end
template <class T>
struct Joins {
    Work& w;
    JoinJobs jobs{};
    explicit Joins(Work& work) : w(work) {}
    void add(JoinJob j, int64_t wgs) {
        if (!j.n) return;
        jobs.job[jobs.n] = j;
        jobs.first[jobs.n + 1] = jobs.first[jobs.n] + (unsigned)wgs;
        ++jobs.n;
    }
    void elements(const float* part, int z, int64_t rows, int64_t N, const void* bias, void* out, bool pairs = false) {
        const int64_t n = rows * N;
        const bool four = N % 4 == 0 && aligned16(out);
        const int64_t per = four ? 4096 : 1024;
        add({part, out, bias, n, N, z, four ? JOIN_ELEMENTS4 : JOIN_ELEMENTS, pairs}, std::min<int64_t>((n + per - 1) / per, 2048));
    }
    void columns(const float* part, int64_t shares, int64_t N, void* out) { add({part, out, nullptr, N, N, (int)shares, JOIN_COLUMNS, false}, (N + 15) / 16); }
    hipError_t go() {
        if (!jobs.n || w.counting()) return hipSuccess;
        k_ffn_join<T><<<jobs.first[jobs.n], 1024, 0, w.s>>>(jobs);
        return hipGetLastError();
    }
};
// rows `from` .. M - 1 of a product, over `splits` shares of k
template <class T, int AK, int BK, int EPI>
hipError_t rows_of(Work& w, Joins<T>& joins, Prod g, int64_t from, int shape, int splits) {
    float* part = splits > 1 ? (float*)w.take((size_t)splits * (g.M - from) * g.N * 4) : nullptr;
    if (w.counting() || from == g.M) return hipSuccess;
    g.m_base = from;
    if (!part) return launch_shape<T, AK, BK, EPI>(shape, g, 1, w.s);
    g.part = part; g.rows_out = g.M - from; g.vec_out = g.N % 4 == 0;
    FFN_TRY((launch_shape<T, AK, BK, EPI>(shape, g, splits, w.s)));
    joins.elements(part, splits, g.M - from, g.N, g.bias, (T*)g.out + from * g.N);
    return hipSuccess;
}
template <class T, int EPI>
Plan product_plan(const Prod& g) {
    constexpr int es = sizeof(T), pairs = Mat<T>::P == 3 ? 6 : 1;
    return EPI == EPI_GATE ? gate_plan(g.M, g.HP, g.K, es, pairs, g.p) : EPI == EPI_DH ? dh_plan(g.M, g.HP, g.K, es, pairs) : rows_plan(g.M, g.N, g.K, es, pairs);
}
// a product over the rows of a batch
template <class T, int AK, int BK, int EPI>
hipError_t product(Work& w, Joins<T>& joins, Prod g) {
    const Plan p = product_plan<T, EPI>(g);
    const int64_t M = g.M;
    g.M = p.main_rows;
    FFN_TRY((rows_of<T, AK, BK, EPI>(w, joins, g, 0, p.shape, p.splits)));
    g.M = M;
    return rows_of<T, AK, BK, EPI>(w, joins, g, p.main_rows, p.rest_shape, p.rest_splits);
}
// a product over the rows of a batch whose A holds them twice, rounded and what the rounding left: both halves are shares of one sum
template <class T, int BK>
hipError_t product_of_pairs(Work& w, Joins<T>& joins, Prod g) {
    g.ra = g.rows_out = 2 * g.M;
    const int64_t M = g.M;
    g.M *= 2;
    const Plan p = product_plan<T, EPI_OUT>(g);                       // (at most 2 FEW rows: one launch)
    g.part = (float*)w.take((size_t)p.splits * g.M * g.N * 4);
    if (w.counting()) return hipSuccess;
    g.vec_out = g.N % 4 == 0;
    FFN_TRY((launch_shape<T, KC, BK, EPI_OUT>(p.shape, g, p.splits, w.s)));
    joins.elements(g.part, 2 * p.splits, M, g.N, g.bias, g.out, true);
    return hipSuccess;
}
template <class T>
hipError_t weight_gradient(Work& w, Joins<T>& joins, Prod g, int64_t rows_out) {
    const Plan p = weight_plan(g.M, g.N, g.K, sizeof(T), Mat<T>::P == 3 ? 6 : 1);
    g.rows_out = rows_out;
    if (p.splits > 1) g.part = (float*)w.take((size_t)p.splits * rows_out * g.N * 4);
    if (w.counting()) return hipSuccess;
    g.vec_out = g.N % 4 == 0 && (p.splits > 1 || aligned16(g.out));
    FFN_TRY((launch_shape<T, KS, KS, EPI_OUT>(p.shape, g, p.splits, w.s)));
    if (p.splits > 1) joins.elements(g.part, p.splits, rows_out, g.N, nullptr, g.out);
    return hipSuccess;
}
// shares: enough workgroups for the chip, each at least 64 rows
template <class T>
hipError_t colsum(Work& w, Joins<T>& joins, const void* a, int64_t M, int64_t N, void* out) {
    constexpr int V = 16 / (int)sizeof(T);
    const int64_t shares = std::max<int64_t>(1, std::min<int64_t>((M + 63) / 64, 128));
    float* part = (float*)w.take((size_t)shares * N * 4);
    if (w.counting()) return hipSuccess;
    if (N % V == 0 && aligned16(a))
        k_ffn_colsum<T, V><<<dim3((unsigned)((N + 32 * V - 1) / (32 * V)), (unsigned)shares), 256, 0, w.s>>>((const T*)a, M, N, part);
    else
        k_ffn_colsum<T, 1><<<dim3((unsigned)((N + 31) / 32), (unsigned)shares), 256, 0, w.s>>>((const T*)a, M, N, part);
    joins.columns(part, shares, N, out);
    return hipGetLastError();
}

// A few rows' h and [dg | du] keep what their rounding leaves next to them, as that many more rows: with so few, the error of rounding h is not
// averaged (1 to 3 rows of fp16: up to 1.55 of the result's own rounding in y and dW3, 1.41 with many), and twice the rows fit in the same tile.
constexpr int FEW = 8;
template <class T> inline bool in_pairs(int64_t M) { return Mat<T>::P == 1 && M <= FEW; }

// what the forward pass keeps: h planes, then p and q
template <class T> inline size_t kept_h(int64_t M, int64_t H) { return up256(planes_bytes<T>(in_pairs<T>(M) ? 2 * M : M, pad8(H))); }

template <class T, int V, int MM, int RW>
hipError_t few_go(const FfnArgs& f, float* h, hipStream_t s) {
    const int64_t units = ((int64_t)f.H + RW / 2 - 1) / (RW / 2), outs = ((int64_t)f.O + RW / 2 - 1) / (RW / 2);
    k_ffn_few<T, V, MM, RW, true, T, float><<<(unsigned)((units + 3) / 4), 256, 0, s>>>((const T*)f.x, (int)f.M, f.D, (const T*)f.w12, f.H, (const T*)f.b12, f.act, h);
    k_ffn_few<T, V, MM, RW / 2, false, float, T><<<(unsigned)((outs + 3) / 4), 256, 0, s>>>(h, (int)f.M, f.H, (const T*)f.w3, f.O, (const T*)f.b3, f.act, (T*)f.y);
    return hipGetLastError();
}
template <class T, int V>
hipError_t few(const FfnArgs& f, float* h, hipStream_t s) {
    return f.M == 1 ? few_go<T, V, 1, 2>(f, h, s) : f.M == 2 ? few_go<T, V, 2, 2>(f, h, s) : f.M <= 4 ? few_go<T, V, 4, 4>(f, h, s) : few_go<T, V, 8, 4>(f, h, s);
}

template <class T>
hipError_t forward(const FfnArgs& f, Work& w) {
    const int64_t HP = pad8(f.H);
    if (f.M <= FEW && !f.kept) {
        float* h = (float*)w.take((size_t)f.M * f.H * 4);
        if (!w.counting()) {
            constexpr int V = 16 / (int)sizeof(T);
            const bool vec = f.D % V == 0 && f.H % V == 0 && aligned16(f.x) && aligned16(f.w12) && aligned16(f.w3);
            return vec ? few<T, V>(f, h, w.s) : few<T, 1>(f, h, w.s);
        }
    }
    Packer<T> pack(w);
    Joins<T> joins(w);
    const Operand x = pack.add(f.x, 1, f.M, f.D), w12 = pack.add(f.w12, 2, f.H, f.D), w3 = pack.add(f.w3, 1, f.O, f.H);
    FFN_TRY(pack.go());
    char* h = (char*)f.kept;
    if (!h) h = (char*)w.take(kept_h<T>(f.M, f.H));
    Prod g{};
    g.a = x; g.b = w12; g.ra = f.M; g.M = f.M; g.N = f.H; g.K = f.D; g.out = h; g.bias = f.b12; g.act = f.act; g.HP = HP; g.ldo = HP; g.plane_o = f.M * HP; g.up_row = HP;
    if (f.kept) { g.p = (float*)(h + kept_h<T>(f.M, f.H)); g.q = g.p + f.M * HP; }
    if (in_pairs<T>(f.M)) g.rest = f.M * HP;
    FFN_TRY((product<T, KC, KC, EPI_GATE>(w, joins, g)));
    Prod d{};
    d.a = {h, HP, f.M * HP}; d.b = w3; d.ra = f.M; d.rb = f.O; d.M = f.M; d.N = f.O; d.K = f.H; d.out = f.y; d.bias = f.b3;
    d.vec_out = f.O % 4 == 0 && aligned16(f.y);
    if (in_pairs<T>(f.M)) FFN_TRY((product_of_pairs<T, KC>(w, joins, d)));
    else FFN_TRY((product<T, KC, KC, EPI_OUT>(w, joins, d)));
    return joins.go();
}

template <class T>
hipError_t backward(const FfnArgs& f, Work& w) {
    const int64_t HP = pad8(f.H);
    const bool all = w.counting(), hidden = all || f.dx || f.dw12 || f.db12;
    const int times = in_pairs<T>(f.M) ? 2 : 1;
    char* h = (char*)f.kept;
    const float* p = (const float*)(h + (all ? 0 : kept_h<T>(f.M, f.H)));
    Packer<T> pack(w);
    Joins<T> joins(w);
    Operand dy{}, w3{}, w12{}, x{};
    if (hidden || f.dw3) dy = pack.add(f.dy, 1, f.M, f.O, times);
    if (hidden) w3 = pack.add(f.w3, 1, f.O, f.H);
    if (all || f.dx) w12 = pack.add(f.w12, 2, f.H, f.D);
    if (all || f.dw12) x = pack.add(f.x, 1, f.M, f.D, times);
    FFN_TRY(pack.go());
    const Operand dgu{hidden ? w.take(planes_bytes<T>(times * f.M, 2 * HP)) : nullptr, 2 * HP, f.M * 2 * HP};
    if (hidden) {
        Prod g{};
        g.a = dy; g.b = w3; g.ra = f.M; g.M = f.M; g.N = f.H; g.K = f.O; g.out = const_cast<void*>(dgu.p); g.HP = HP; g.ldo = 2 * HP; g.plane_o = dgu.plane;
        g.p = const_cast<float*>(p); g.q = g.p + f.M * HP; g.rest = times == 2 ? dgu.plane : 0;
        const int slice = product_plan<T, EPI_DH>(g).shape == SHAPE_64 ? 32 : 64;
        const int64_t slices = (f.M + slice - 1) / slice;
        if (all || f.db12) g.sums = (float*)w.take((size_t)slices * 2 * f.H * 4);
        FFN_TRY((product<T, KC, KS, EPI_DH>(w, joins, g)));
        if (!all && f.db12) joins.columns(g.sums, slices, 2 * (int64_t)f.H, f.db12);
    }
    if (all || f.dx) {
        Prod g{};
        g.a = dgu; g.b = w12; g.ra = f.M; g.M = f.M; g.N = f.D; g.K = 2 * HP; g.out = f.dx; g.vec_out = f.D % 4 == 0 && aligned16(f.dx);
        if (times == 2) FFN_TRY((product_of_pairs<T, KS>(w, joins, g)));
        else FFN_TRY((product<T, KC, KS, EPI_OUT>(w, joins, g)));
    }
    if (all || f.dw12) {
        Prod g{};
        g.a = dgu; g.b = x; g.M = 2 * HP; g.N = f.D; g.K = times * f.M; g.out = f.dw12; g.half_pad = HP; g.half = f.H;
        FFN_TRY(weight_gradient<T>(w, joins, g, 2 * (int64_t)f.H));
    }
    if (all || f.dw3) {
        Prod g{};
        g.a = dy; g.b = {h, HP, f.M * HP}; g.M = f.O; g.N = f.H; g.K = times * f.M; g.out = f.dw3;
        FFN_TRY(weight_gradient<T>(w, joins, g, f.O));
    }
    if (all || f.db3) FFN_TRY(colsum<T>(w, joins, f.dy, f.M, f.O, f.db3));
    return joins.go();
}

template <class F>
auto by_type(int dt, F f) { return dt == IFF_DT_F32 ? f(float{}) : dt == IFF_DT_BF16 ? f(__bf16{}) : f(_Float16{}); }

}  // namespace

size_t ffn_kept_bytes(const FfnArgs& a) {
    return by_type(a.dt, [&](auto t) { return kept_h<decltype(t)>(a.M, a.H) + (size_t)2 * a.M * pad8(a.H) * 4; });
}
size_t ffn_forward_workspace(const FfnArgs& a) {
    Work w{nullptr, 0, nullptr};
    (void)by_type(a.dt, [&](auto t) { return forward<decltype(t)>(a, w); });
    return w.used;
}
size_t ffn_backward_workspace(const FfnArgs& a) {
    Work w{nullptr, 0, nullptr};
    (void)by_type(a.dt, [&](auto t) { return backward<decltype(t)>(a, w); });
    return w.used;
}
hipError_t launch_ffn_forward(const FfnArgs& a, void* ws, hipStream_t s) {
    Work w{(char*)ws, 0, s};
    return by_type(a.dt, [&](auto t) { return forward<decltype(t)>(a, w); });
}
hipError_t launch_ffn_backward(const FfnArgs& a, void* ws, hipStream_t s) {
    Work w{(char*)ws, 0, s};
    return by_type(a.dt, [&](auto t) { return backward<decltype(t)>(a, w); });
}
