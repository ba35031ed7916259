// Orthogonalised updates: Newton-Schulz products over stacks of weight matrices (s3d_orthogonalize) and the optimizer step built on them
// (s3d_muon_step).
//
// Mathematics.  X0 = U / max(|U|_F, eps); with m the smaller side, `steps` times
//     A = X X^T (wide) or X^T X (tall),   P = a I + b A + c A^2 (m x m, symmetric),   X <- P X (wide) or X P (tall)
// i.e. every singular value s of X0 becomes p(p(..p(s))) with p(s) = a s + b s^3 + c s^5, the singular vectors stay.  A matrix keeps its
// orientation from the gradient to the update, so nothing is ever transposed in memory: the Gram product of a wide matrix and the product of a
// tall one read k-contiguous rows; the other two operands are k-major tiles, read from LDS with the transposing reads.  The two symmetric
// products compute the lower triangle of tiles and store the mirror image.
//
// Precision.  A step multiplies a small singular value by a = 3.4 and with it every rounding that fell into its direction: five steps
// turn one rounding of the operands to bf16 into 3.4^5 * 2^-9 = 90 % of a direction, to fp16 into 10 %.  Operands are therefore PAIRS of fp16 planes
// (hi = rne(x s), lo = rne(x s - hi), 22 bits; s a power of two that keeps the largest possible entry below 2^15) multiplied as
// hi lo + lo hi + hi hi with fp32 accumulation: an fp32 product at a third of the fp16 matrix rate, five times that of the fp32 matrix
// instructions.  fp16 planes rather than bf16: all entries are bounded by the spectral norm, so the exponent range is not needed and
// the six extra bits are.  Results in bf16 take the same products and are rounded once, at the end: the last two steps on the hi planes alone would save
// a fifth of 4 x 2048^2 (2110 us to 1646) and cost up to another rounding of the result (2 * 2^-12 (a^2 + a): 0.7 % for a = 3.44, more for a larger a).
//
// Bound: the matrix cores for large stacks (4 x 2048^2: P X 161 - 200 us = 1030 - 1280 TF of fp16 products, a large library product 1095), the balance of uneven
// k over the CUs for a model's (48 matrices, 384 wide: Gram 48 us of 30, P X 63 of 45, the last product HBM: 425 MB in 87 us), what one CU can fetch and
// the latency of dependent launches for few small ones (192 x 192: twelve launches of 4 - 9 us, 74 us).
#include <math.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "kmajor.h"
#include "ranges.h"

namespace {

typedef _Float16 half_t;
typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(4))) _Float16 half4;

constexpr int NS_ITEMS = 16;          // stacks of one launch (kernel-argument table); more are worked in several rounds

struct NsDims {
    int count, rows, cols;            // the caller's matrices
    int rp, cp, mp;                   // rows, columns and smaller side padded to the tile
    int tall;                         // rows > cols
    int chunks;                       // partial sums of squares per matrix
    long ws, wsz;                     // first matrix's tensors in the workspace / size of one matrix's (in halves)
    long part;                        // first matrix's partial sums
    int per; unsigned per_inv;        // this launch: workgroups of a matrix, 2^32 / per
};
struct NsTable {
    int n;
    unsigned wgs[NS_ITEMS];           // workgroups of every stack in this launch, 0 behind the last
    NsDims d[NS_ITEMS];
};
struct NsPtrs {
    const void* x[NS_ITEMS]; long xs[NS_ITEMS], xld[NS_ITEMS];      // ortho: input.  muon: gradient
    void* o[NS_ITEMS]; long os[NS_ITEMS], old[NS_ITEMS];            // ortho: output.  muon: parameters
    float* m[NS_ITEMS]; long ms[NS_ITEMS], mld[NS_ITEMS];           // muon: momentum
    bf16_t* hi[NS_ITEMS]; bf16_t* lo[NS_ITEMS];                     // muon: planes of the parameters (strides of p)
    float scale[NS_ITEMS];
};
enum { SRC_F32 = 0, SRC_BF16 = 1, SRC_MUON = 2 };
enum { EPI_GRAM = 0, EPI_POLY = 1, EPI_MULT = 2, EPI_OUT_F32 = 3, EPI_OUT_BF16 = 4, EPI_UPDATE = 5, EPI_GRAM_ROWS = 6 };      // _ROWS: no stack is tall

// Workgroups go round robin over the eight XCDs, each with an L2 of its own: XCD x takes the x-th eighth of every stack's workgroups, so that the
// tiles of one matrix share an L2 and the XCDs have equal shares of long and short products.  The grid is 8 * sum of ceil(wgs / 8): false for
// what is over.
struct NsPlace { int it, mat, tile; };
__device__ __forceinline__ bool ns_place(const NsTable& t, NsPlace& w) {
    const unsigned per0 = t.d[0].per, inv0 = t.d[0].per_inv;
    const unsigned x = blockIdx.x & 7, i = blockIdx.x >> 3;
    unsigned c = 0, r = 0;
    int it = -1;
#pragma unroll
    for (int k = 0; k < NS_ITEMS; ++k) {                             // (straight line, counts behind the last stack are 0: one load instead of a chain)
        const unsigned n = t.wgs[k], lo = (x * n) >> 3, size = ((x + 1) * n >> 3) - lo;
        const bool here = i - c < size;
        it = here ? k : it;
        r = here ? lo + (i - c) : r;
        c += size;
    }
    if (it < 0) return false;
    unsigned per = per0, inv = inv0;
    if (it) { per = t.d[it].per; inv = t.d[it].per_inv; }
    unsigned q = (unsigned)(((unsigned long long)r * inv) >> 32);    // r / per, at most two short
    if (r - q * per >= per) ++q;
    if (r - q * per >= per) ++q;
    w.it = it; w.mat = (int)q; w.tile = (int)(r - q * per);
    return true;
}
// tensors of one matrix, in halves from its base: X [rp][cp] twice (read one, write the other), A [mp][mp], P [mp][mp], each with room for a pair
__device__ __forceinline__ long off_x(const NsDims& d, int which) { return 2L * d.rp * d.cp * which; }
__device__ __forceinline__ long off_a(const NsDims& d) { return 4L * d.rp * d.cp; }
__device__ __forceinline__ long off_p(const NsDims& d) { return 4L * d.rp * d.cp + 2L * d.mp * d.mp; }

// Pairs in memory: blocks of 32 columns, [hi 32 | lo 32] = one 128-byte line, so that a stage of 32 k of a row is ONE line (with two separate planes
// every line was fetched twice, half of it each time: 12 TB/s of useful L2 traffic instead of 20).
__device__ __forceinline__ long ns_at(long r, int c, int ld) { return r * 2 * ld + ((c >> 5) << 6) + (c & 31); }

__device__ __forceinline__ void split_half(float v, half_t& hi, half_t& lo) {
    hi = (half_t)v;
    lo = (half_t)(v - (float)hi);
}

// momentum and the direction of the step, elementwise: m' = mu m + (1 - mu) g, u = nesterov ? (1 - mu) g + mu m' : m'
__device__ __forceinline__ float muon_mix(float g, float m, float mu) { return fmaf(mu, m, (1.f - mu) * g); }

// 8 consecutive elements (n of them inside the row, the rest 0) in 16-byte accesses, whatever the row's alignment: rows of odd length are
// not aligned, and global memory takes 16-byte accesses at the element's alignment
typedef f32x4 __attribute__((aligned(4))) f32x4_any;
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
__device__ __forceinline__ void load8f(const float* p, int n, float* v) {
    if (n == 8) {
        const f32x4 a = *reinterpret_cast<const f32x4_any*>(p), b = *reinterpret_cast<const f32x4_any*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
    }
}
__device__ __forceinline__ void store8f(float* p, int n, const float* v) {
    if (n == 8) {
        *reinterpret_cast<f32x4_any*>(p) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_any*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = v[i];
    }
}
__device__ __forceinline__ void load8b(const bf16_t* p, int n, float* v) {
    if (n == 8) {
        U128 a;
        a.u = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = bf2f(a.h[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? bf2f(p[i]) : 0.f;
    }
}

__device__ __forceinline__ void store8b(bf16_t* p, int n, const float* v) {
    if (n == 8) {
        *reinterpret_cast<u32x4_any*>(p) = u32x4{f2bf2(v[0], v[1]), f2bf2(v[2], v[3]), f2bf2(v[4], v[5]), f2bf2(v[6], v[7])};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = f2bf(v[i]);
    }
}

// ---- 1. (momentum and) the sum of squares of every matrix: d.chunks partial sums in 64 bits, added in order by the next kernel ----
template <int SRC>
__global__ __launch_bounds__(256) void ns_sumsq_kernel(const NsTable t, const NsPtrs p, const float* __restrict__ hyper, int nesterov,
                                                       double* __restrict__ part) {
    NsPlace w;
    if (!ns_place(t, w)) return;
    const int it = w.it, mat = w.mat, chunk = w.tile;
    const NsDims& d = t.d[it];
    const unsigned upr = (d.cols + 7) / 8, total = upr * d.rows;              // units of 8 columns (at most 2^29)
    const unsigned per = (total + d.chunks - 1) / d.chunks, lo = chunk * per, hi = lo + per < total ? lo + per : total;
    float mu = 0.f, gs = 1.f;
    if constexpr (SRC == SRC_MUON) { mu = hyper[1]; gs = hyper[3]; }
    double s = 0.;
    for (unsigned e = lo + threadIdx.x; e < hi; e += 256) {
        const unsigned r = e / upr, c = (e - r * upr) * 8;
        const int n = d.cols - (int)c < 8 ? d.cols - (int)c : 8;
        const long xi = mat * p.xs[it] + (long)r * p.xld[it] + c;
        float u[8];
        if constexpr (SRC == SRC_BF16) load8b((const bf16_t*)p.x[it] + xi, n, u);
        else load8f((const float*)p.x[it] + xi, n, u);
        if constexpr (SRC == SRC_MUON) {
            float* mp = p.m[it] + mat * p.ms[it] + (long)r * p.mld[it] + c;
            float m[8];
            load8f(mp, n, m);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float g = u[i] * gs;
                m[i] = muon_mix(g, m[i], mu);
                u[i] = nesterov ? muon_mix(g, m[i], mu) : m[i];
            }
            store8f(mp, n, m);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) s += (double)u[i] * u[i];
    }
    __shared__ double red[256];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if (threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0) part[d.part + (long)mat * d.chunks + chunk] = red[0];
}

// ---- 2. X0 = U / max(|U|, eps) as pairs, padding cleared: 2048 elements of [rp][cp] per workgroup ----
template <int SRC>
__global__ __launch_bounds__(256) void ns_load_kernel(const NsTable t, const NsPtrs p, const float* __restrict__ hyper, int nesterov,
                                                      const double* __restrict__ part, float eps, float sx, half_t* __restrict__ ws) {
    NsPlace w;
    if (!ns_place(t, w)) return;
    const int it = w.it, mat = w.mat, blk = w.tile;
    const NsDims& d = t.d[it];
    __shared__ double red[256];
    {
        double s = 0.;
        for (int k = threadIdx.x; k < d.chunks; k += 256) s += part[d.part + (long)mat * d.chunks + k];
        red[threadIdx.x] = s;
    }
    const unsigned cpu = d.cp / 8, e = (unsigned)blk * 256 + threadIdx.x, r = e / cpu, c = (e - r * cpu) * 8;
    float mu = 0.f, gs = 1.f;
    if constexpr (SRC == SRC_MUON) { mu = hyper[1]; gs = hyper[3]; }
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = 0.f;
    const int n = (int)r < d.rows ? (d.cols - (int)c < 8 ? d.cols - (int)c : 8) : 0;
    if (n > 0) {
        const long xi = mat * p.xs[it] + (long)r * p.xld[it] + c;
        if constexpr (SRC == SRC_BF16) load8b((const bf16_t*)p.x[it] + xi, n, u);
        else if constexpr (SRC == SRC_F32) load8f((const float*)p.x[it] + xi, n, u);
        else {
            float m[8];
            load8f(p.m[it] + mat * p.ms[it] + (long)r * p.mld[it] + c, n, m);
            if (nesterov) load8f((const float*)p.x[it] + xi, n, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = nesterov ? muon_mix(u[i] * gs, m[i], mu) : m[i];
        }
    }
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if (threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
        __syncthreads();
    }
    const double nrm = sqrt(red[0]);
    // 1 / |U| in two parts: rounded to fp32 it moves all singular values together
    const double exact = (double)sx / (nrm > (double)eps ? nrm : (nrm == nrm ? (double)eps : nrm));
    const float inv = (float)exact, inv_low = (float)(exact - (double)inv);
    half8 h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        half_t a, b;
        split_half(i < n ? fmaf(u[i], inv, u[i] * inv_low) : 0.f, a, b);
        h[i] = a;
        l[i] = b;
    }
    half_t* X = ws + d.ws + mat * d.wsz + ns_at(r, c, d.cp);
    *reinterpret_cast<half8*>(X) = h;
    *reinterpret_cast<half8*>(X + 32) = l;
}

// ---- 3. the products ----
// One operand of a product, i the tile's side: element (i, k) at row i, column k (KM false) or at row k, column i (KM true) of a tensor with ld columns;
// the tile starts at i = at.
struct NsOperand { const half_t* p; int ld, at; };

// One stage of an operand is T x 128 bytes of LDS: T rows of one line (k-contiguous), or 32 k rows of the tile's columns (k-major).
// Piece q of it is 1 KB = one DMA instruction of a wave; every lane brings 16 bytes, the slot swizzle is applied here.  A lane's byte offset from ns_base is
// (ns_lane_source ^ ns_flip(q)) + q * rows of a piece * row: the swizzles are linear in the row's bits and a row is a multiple of what they permute, so a
// wave keeps one register for all its pieces.
template <int T, bool KM>
struct NsPieces {
    static constexpr int W = 2 * T, WK = W / 8;                     // k-major: halves / 16-byte slots of a row
    static constexpr int ROWS = KM ? 64 / WK : 8;                    // of a piece
};
template <int T, bool KM>
__device__ __forceinline__ unsigned ns_lane_source(const NsOperand& o, int lane) {
    using P = NsPieces<T, KM>;
    const int r = KM ? lane / P::WK : lane >> 3, chunk = KM ? (lane % P::WK) ^ kmajor_swz<P::W>(r) : (lane & 7) ^ dma_swz64(r);
    return (unsigned)(r * 2 * o.ld + chunk * 8) * 2;
}
template <int T, bool KM>
__device__ __forceinline__ unsigned ns_flip(int piece) {
    using P = NsPieces<T, KM>;
    return (KM ? kmajor_swz<P::W>(piece * P::ROWS) : dma_swz64(piece * P::ROWS)) * 16;
}
template <int T, bool KM>
__device__ __forceinline__ int ns_advance(const NsOperand& o, int piece) { return piece * NsPieces<T, KM>::ROWS * 2 * o.ld; }      // in halves
template <int T, bool KM>
__device__ __forceinline__ unsigned ns_source(const NsOperand& o, int piece, int lane) {           // (at most 192 rows)
    return (ns_lane_source<T, KM>(o, lane) ^ ns_flip<T, KM>(piece)) + (unsigned)ns_advance<T, KM>(o, piece) * 2;
}
template <bool KM>
__device__ __forceinline__ const half_t* ns_base(const NsOperand& o) { return o.p + (KM ? 2L * o.at : 2L * o.at * o.ld); }
template <bool KM>
__device__ __forceinline__ long ns_step(const NsOperand& o) { return KM ? 64L * o.ld : 64; }      // halves from stage to stage (32 rows of 2 ld, or one line)
// one piece: every lane's 16 bytes at base + off land lane-linear at LDS byte address dst (all but off wave-uniform).  The compiler does not count the
// load: it is retired with a counted wait before anything reads the piece.
__device__ __forceinline__ void ns_dma(const half_t* base, unsigned off, unsigned dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(dst), "s"(base)
                 : "memory");
}
// s_waitcnt vmcnt(vm) [lgkmcnt(0)] as the compiler's own instruction: its count of outstanding LDS reads stays right
template <int VM, bool LGKM>
__device__ __forceinline__ void ns_wait() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((VM & 15) | (7 << 4) | ((LGKM ? 0 : 15) << 8) | ((VM >> 4) << 14));
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void ns_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A lane's LDS address of the fragments whose rows / columns begin at w0 (a multiple of 32, of 16 for a single one), of an operand's tile at `tile`
// (a multiple of 512); fragment (q, i), plane q of rows / columns w0 + 16 i .. + 15, is a constant away.  Both
// swizzles depend on the lane alone, so that one register per operand is kept instead of one per fragment.
template <int T, bool KM>
__device__ __forceinline__ unsigned ns_lane(const unsigned char* tile, int w0, int lane) {
    if constexpr (!KM) {
        const int r = w0 + (lane & 15);
        return (unsigned)(uintptr_t)tile + r * 128 + (((lane >> 4) ^ dma_swz64(r)) << 4);
    } else return kmajor_addr<2 * T>(tile, (w0 >> 5) * 64 + (w0 & 31), (lane >> 4) * 8, lane);
}
template <int T, bool KM>
__device__ __forceinline__ half8 ns_frag(unsigned at, int q, int i) {
    if constexpr (!KM) {
        typedef __attribute__((address_space(3))) half8 lds_half8;
        return *(const lds_half8*)(uintptr_t)((at ^ (q * 64)) + i * 2048);
    } else {
        typedef __attribute__((ext_vector_type(4))) short short4v;
        typedef __attribute__((address_space(3))) short4v lds_short4;
        constexpr int ROW = 4 * T;                                                   // bytes
        struct { short4v a, b; } u;
        const unsigned ad = at ^ ((i >> 1) * 128 + q * 64 + (i & 1) * 32);
        u.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)ad);
        u.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)(ad + 4 * ROW));
        return __builtin_bit_cast(half8, u);
    }
}
template <int FR, int FC>
struct NsFrags { half8 l[2][FR], r[2][FC]; };
// the fragments of a stage, and the products [from, to) of its 3 FR FC (hi lo, lo hi, hi hi): numbered so that they can be dealt out between the other
// instructions of a stage
template <int T, int F, bool KM>
__device__ __forceinline__ void ns_read(half8 (&f)[2][F], unsigned at) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < F; ++i) f[q][i] = ns_frag<T, KM>(at, q, i);
}
// Sums of a tile.  The matrix cores' accumulation rounds towards zero at the size of what is there, so one running sum of three products per 32 k is
// off to one side, for all singular values together (results of orthogonalize 1.1e-6 .. 2.3e-6 off in the 2-norm; 0.5e-6 .. 0.7e-6 with these and the shift of A below).
// SPLIT (the short sums of a wave that has a part of k): hi hi in one sum, the two products 2^11 smaller in another.  Else: two stages begin at zero,
// small products first, and are added to a total that rounds to nearest.
template <int FR, int FC, bool SPLIT>
struct NsSums {
    f32x4 sum[FR][FC], more[FR][FC];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < FR; ++i)
#pragma unroll
            for (int j = 0; j < FC; ++j) sum[i][j] = more[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void flush() {
        if constexpr (!SPLIT) {
#pragma unroll
            for (int i = 0; i < FR; ++i)
#pragma unroll
                for (int j = 0; j < FC; ++j) more[i][j] += sum[i][j];
        }
    }
    __device__ __forceinline__ f32x4 get(int i, int j) const {
        if constexpr (SPLIT) return sum[i][j] + more[i][j];
        else return more[i][j];
    }
};
// FIRST: the first of two stages
template <bool FIRST, int FR, int FC, bool SPLIT>
__device__ __forceinline__ void ns_mfma(const NsFrags<FR, FC>& f, NsSums<FR, FC, SPLIT>& acc, int from = 0, int to = 3 * FR * FC) {
#pragma unroll
    for (int e = from; e < to; ++e) {
        const int q = e / (FR * FC), i = e / FC % FR, j = e % FC, ql = q == 1, qr = q == 0;
        f32x4& a = SPLIT && q < 2 ? acc.more[i][j] : acc.sum[i][j];
        const f32x4 c = !SPLIT && FIRST && q == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : a;
        a = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.r[qr][j], f.l[ql][i], c, 0, 0, 0);
    }
}

// acc = sum over k of L(i, k) R(j, k) for a TR x TC tile by 2 x 2 waves of TR/2 x TC/2: a ring of
// RING stages filled by LDS-DMA; the fragments of the next stage are read while the matrix cores work on this one (a SIMD has
// two waves: without that the LDS time of a stage adds to its MFMA time).  K is a multiple of 64, a stage 32 of it.  acc.get(i, j)[e] = C[wr + 16 i + (lane & 15)][wc + 16 j + 4 (lane >> 4) + e].
template <int TR, int TC, int RING, bool LK, bool RK>
__device__ __forceinline__ void ns_product(const NsOperand& L, const NsOperand& R, int K, unsigned char* smem, NsSums<TR / 32, TC / 32, false>& acc) {
    constexpr int STAGE = (TR + TC) * 128;                           // bytes: L, R
    constexpr int PIECES = STAGE / 1024 / 4;                         // 1 KB DMA pieces per wave and stage: wave w brings w PIECES .. of L's and R's
    constexpr int LEFT = TR / 8, FR = TR / 32, FC = TC / 32;         // L's pieces; 16-row fragments per wave
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int left = LEFT - wave * PIECES;                           // this wave's pieces below `left` are L's
    const long step_l = ns_step<LK>(L), step_r = ns_step<RK>(R);
    const half_t *src_l = ns_base<LK>(L), *src_r = ns_base<RK>(R);
    const unsigned off_l = ns_lane_source<TR, LK>(L, lane), off_r = ns_lane_source<TC, RK>(R, lane);
    auto bring = [&](unsigned at) {                                  // this wave's pieces of the next stage
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int ql = wave * PIECES + i, qr = ql - LEFT;
            const half_t* src = i < left ? src_l + ns_advance<TR, LK>(L, ql) : src_r + ns_advance<TC, RK>(R, qr);
            const unsigned off = i < left ? off_l ^ ns_flip<TR, LK>(ql) : off_r ^ ns_flip<TC, RK>(qr);
            ns_dma(src, off, at + i * 1024);
        }
    };
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)smem + wave * PIECES * 1024);
    const int KT = K / 32;
    unsigned slot_in = 0, slot = 0;                                  // in bytes
    auto advance = [](unsigned& s) { s = s == (RING - 1) * STAGE ? 0 : s + STAGE; };
    acc.clear();
    for (int k = 0; k < RING && k < KT; ++k) {
        bring(lds0 + slot_in);
        src_l += step_l;
        src_r += step_r;
        advance(slot_in);
    }
    const int wr = (wave >> 1) * (TR / 2), wc = (wave & 1) * (TC / 2);
    // stage 0 has landed when at most the later stages' pieces are outstanding
    if (RING <= KT) ns_wait<(RING - 1) * PIECES, false>();
    else ns_wait<0, false>();
    ns_barrier();
    NsFrags<FR, FC> fa, fb;
    const unsigned lane_l = ns_lane<TR, LK>(smem, wr, lane), lane_r = ns_lane<TC, RK>(smem + TR * 128, wc, lane);
    ns_read<TR, FR, LK>(fa.l, lane_l);
    ns_read<TC, FC, RK>(fa.r, lane_r);
    auto body = [&](auto first, int kt, NsFrags<FR, FC>& now, NsFrags<FR, FC>& next) {
        constexpr bool FIRST = decltype(first)::value;
        // this wave holds stage kt in registers (lgkmcnt) and its pieces of stage kt + 1 have landed; behind the barrier that is true of every wave:
        // the slot of stage kt can be refilled, stage kt + 1 can be read (behind the last stage: old data that nobody uses)
        if (RING == 2 || kt + RING > KT) ns_wait<0, true>();
        else ns_wait<(RING - 2) * PIECES, true>();
        ns_barrier();
        const bool more = kt + RING < KT;
        advance(slot);
        // the reads lie under the products (finer interleavings of loads, reads and products measured the same or slower)
        constexpr int M = 3 * FR * FC;
        if (more) bring(lds0 + slot_in);
        ns_mfma<FIRST>(now, acc, 0, M / 3);
        ns_read<TR, FR, LK>(next.l, lane_l + slot);
        ns_mfma<FIRST>(now, acc, M / 3, 2 * M / 3);
        ns_read<TC, FC, RK>(next.r, lane_r + slot);              // (lo of either side is done: all at once are 32 registers more)
        ns_mfma<FIRST>(now, acc, 2 * M / 3, M);
        src_l += step_l;
        src_r += step_r;
        advance(slot_in);
    };
    for (int kt = 0; kt < KT; kt += 2) {
        body(std::true_type(), kt, fa, fb);
        if (kt + 1 < KT) body(std::false_type(), kt + 1, fb, fa);
        acc.flush();
    }
}

// The same for a 64 x 64 or 32 x 32 tile with the k range dealt to the four waves (stage s to wave s % 4): every wave works the whole tile on its own
// stages, brought by itself, so nothing is waited for but its own loads; a quarter of the serial length and half the LDS reads per product.  The
// four partial sums are added through LDS in the order of the waves.  64: out[j][e] = C[16 wave + (lane & 15)][16 j + 4 (lane >> 4) + e]; 32: out[0][e] =
// C[16 (wave >> 1) + (lane & 15)][16 (wave & 1) + 4 (lane >> 4) + e].
template <int T, int RING, bool LK, bool RK>
__device__ __forceinline__ void ns_product_ksplit(const NsOperand& L, const NsOperand& R, int K, unsigned char* smem, f32x4 (&out)[T * T / 1024]) {
    constexpr int STAGE = 2 * T * 128, PIECES = STAGE / 1024, F = T / 16, MINE = F * F / 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    unsigned char* mine = smem + wave * RING * STAGE;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)mine);
    const int KT = (K / 32 - wave + 3) / 4;         // stages wave, wave + 4, ..
    const long step_l = ns_step<LK>(L), step_r = ns_step<RK>(R);
    const half_t *src_l = ns_base<LK>(L) + wave * step_l, *src_r = ns_base<RK>(R) + wave * step_r;
    unsigned off[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) off[i] = i >= PIECES / 2 ? ns_source<T, RK>(R, i - PIECES / 2, lane) : ns_source<T, LK>(L, i, lane);
    unsigned slot = 0;                                               // in bytes
    auto issue = [&](unsigned at) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) ns_dma(i >= PIECES / 2 ? src_r : src_l, off[i], lds0 + at + i * 1024);
        src_l += 4 * step_l;
        src_r += 4 * step_r;
    };
    NsSums<F, F, true> acc;
    acc.clear();
    const unsigned lane_l = ns_lane<T, LK>(mine, 0, lane), lane_r = ns_lane<T, RK>(mine + T * 128, 0, lane);
    for (int k = 0; k < RING && k < KT; ++k) issue(k * STAGE);
    for (int kt = 0; kt < KT; ++kt) {
        if (kt + RING <= KT) ns_wait<(RING - 1) * PIECES, false>();
        else ns_wait<0, false>();
        NsFrags<F, F> f;
        ns_read<T, F, LK>(f.l, lane_l + slot);
        ns_read<T, F, RK>(f.r, lane_r + slot);
        ns_wait<63, true>();                                         // the slot is in registers: refill it
        if (kt + RING < KT) issue(slot);
        slot = slot == (RING - 1) * STAGE ? 0 : slot + STAGE;
        ns_mfma<false>(f, acc);
    }
    // partial sums: T x T per wave in its own ring (read by nobody any more), then a quarter of the tile from all four
    f32x4* red = reinterpret_cast<f32x4*>(mine);
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) red[(i * F + j) * 64 + lane] = acc.get(i, j);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) v += reinterpret_cast<const f32x4*>(smem + w * RING * STAGE)[(wave * MINE + j) * 64 + lane];
        out[j] = v;
    }
}

// How a tile is worked.  TILE_128: 128 x 128, four waves, 66 KB of LDS: two workgroups share a CU, one's start and epilogue lie under the other's
// products.  TILE_HALF: 128 x 64, 48 KB, three on a CU: half the granularity for half again the LDS traffic per product.  TILE_64: 64 x 64, the
// k range over the four waves: launches with too few tiles for the CUs.  TILE_32 the same with 32 x 32, 70 KB, two on a CU: launches with so few that
// what one CU can fetch is the bound.
enum { TILE_128 = 0, TILE_64 = 1, TILE_HALF = 2, TILE_32 = 3 };
template <int KIND>
struct NsTile {
    static constexpr bool KSPLIT = KIND == TILE_64 || KIND == TILE_32;
    static constexpr int TR = KIND == TILE_64 ? 64 : KIND == TILE_32 ? 32 : 128, TC = KIND == TILE_HALF ? 64 : TR, PITCH = TC + 4;
    static constexpr int RING = 2;
    static constexpr int SUM_BYTES = TR * PITCH * 4;                 // the tile in fp32
    static constexpr int RING_BYTES = (KSPLIT ? 4 : 1) * RING * (TR + TC) * 128;
    static constexpr int SUM_AT = KSPLIT ? RING_BYTES : 0;           // over the ring, except where the ring still holds partial sums
    static constexpr int BYTES = KSPLIT ? RING_BYTES + SUM_BYTES : SUM_BYTES > RING_BYTES ? SUM_BYTES : RING_BYTES;
};

// 8 elements of a tensor of the iteration at column c (a multiple of 8)
__device__ __forceinline__ void ns_store8(half_t* base, long r, int c, int ld, const float* v) {
    half8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) { half_t a, b; split_half(v[e], a, b); h[e] = a; l[e] = b; }
    half_t* o = base + ns_at(r, c, ld);
    *reinterpret_cast<half8*>(o) = h;
    *reinterpret_cast<half8*>(o + 32) = l;
}

// the last product's epilogue for n <= 8 elements of a row: the result, or the parameters' step
template <int EPI>
__device__ __forceinline__ void ns_finish8(const NsPtrs& p, int it, int mat, int r, int c, int n, float lr, float keep, int zero_grad, float* v) {
    const long oi = mat * p.os[it] + (long)r * p.old[it] + c;
    if constexpr (EPI == EPI_OUT_F32) store8f((float*)p.o[it] + oi, n, v);
    if constexpr (EPI == EPI_OUT_BF16) store8b((bf16_t*)p.o[it] + oi, n, v);
    if constexpr (EPI == EPI_UPDATE) {
        float q[8];
        load8f((const float*)p.o[it] + oi, n, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(-lr, v[e], q[e] * keep);
        store8f((float*)p.o[it] + oi, n, v);
        if (p.hi[it]) {
            store8b(p.hi[it] + oi, n, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] -= bf2f(f2bf(v[e]));
            store8b(p.lo[it] + oi, n, v);
        }
        if (zero_grad) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
            store8f((float*)p.x[it] + mat * p.xs[it] + (long)r * p.xld[it] + c, n, v);
        }
    }
}

// f0 .. f2: scale factors of the epilogue (below)
struct NsScale { float f0, f1, f2; int zero_grad; };
__device__ __forceinline__ float ns_poly(const NsScale& f, float square, float a, bool diagonal) { return fmaf(f.f1, a, f.f0 * square) + (diagonal ? f.f2 : 0.f); }

template <int KIND, int EPI>
__global__ __launch_bounds__(256, KIND == TILE_64 ? 1 : KIND == TILE_HALF && EPI != EPI_GRAM ? 3 : 2) void ns_gemm_kernel(
    const NsTable t, const NsPtrs p, half_t* __restrict__ ws, const float* __restrict__ hyper, int which, const NsScale f) {
    extern __shared__ __attribute__((aligned(512))) unsigned char smem[];
    using Tile = NsTile<KIND>;
    constexpr int TR = Tile::TR, TC = Tile::TC, PITCH = Tile::PITCH, Q = TR / TC;
    constexpr bool GRAM = EPI == EPI_GRAM || EPI == EPI_GRAM_ROWS, SYM = GRAM || EPI == EPI_POLY;
    NsPlace w;
    if (!ns_place(t, w)) return;
    const int it = w.it, mat = w.mat, tile = w.tile;
    NsDims d = t.d[0];                                               // (loaded with the counts; the others cost a second round trip)
    if (it) d = t.d[it];
    int ti, tj;
    if constexpr (SYM) {                                             // lower triangle, row by row: tile = Q ti (ti + 1) / 2 + tj
        const int t1 = tile / Q;
        ti = __builtin_amdgcn_readfirstlane((int)((__builtin_amdgcn_sqrtf(8.f * t1 + 1.f) - 1.f) * 0.5f));
        if (ti * (ti + 1) / 2 > t1) --ti;
        if ((ti + 1) * (ti + 2) / 2 <= t1) ++ti;
        tj = tile - Q * (ti * (ti + 1) / 2);
    } else {
        const int tc = d.cp / TC;
        ti = tile / tc;
        tj = tile - ti * tc;
    }
    half_t* base = ws + d.ws + mat * d.wsz;
    const half_t* X = base + off_x(d, which);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float* S = reinterpret_cast<float*>(smem + Tile::SUM_AT);        // the tile, [TR][PITCH]
    auto product = [&](auto lk, auto rk, const NsOperand& L, const NsOperand& R, int K) {
        constexpr bool LK = decltype(lk)::value, RK = decltype(rk)::value;
        if constexpr (KIND == TILE_32) {
            f32x4 acc[1];
            ns_product_ksplit<TR, Tile::RING, LK, RK>(L, R, K, smem, acc);
            *reinterpret_cast<f32x4*>(S + ((wave >> 1) * 16 + (lane & 15)) * PITCH + (wave & 1) * 16 + (lane >> 4) * 4) = acc[0];
        } else if constexpr (KIND == TILE_64) {
            f32x4 acc[4];
            ns_product_ksplit<TR, Tile::RING, LK, RK>(L, R, K, smem, acc);
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4*>(S + (wave * 16 + (lane & 15)) * PITCH + j * 16 + (lane >> 4) * 4) = acc[j];
        } else {
            NsSums<TR / 32, TC / 32, false> acc;
            ns_product<TR, TC, Tile::RING, LK, RK>(L, R, K, smem, acc);
            float* mine = S + ((wave >> 1) * (TR / 2) + (lane & 15)) * PITCH + (wave & 1) * (TC / 2) + (lane >> 4) * 4;
            __syncthreads();                                         // every wave has read its last stage: the ring is free
#pragma unroll
            for (int i = 0; i < TR / 32; ++i)
#pragma unroll
                for (int j = 0; j < TC / 32; ++j) *reinterpret_cast<f32x4*>(mine + i * 16 * PITCH + j * 16) = acc.get(i, j);
        }
        __syncthreads();
    };
    const std::false_type rows;                                      // operand stored as rows of k
    const std::true_type kmajor;
    if constexpr (EPI == EPI_GRAM_ROWS) product(rows, rows, NsOperand{X, d.cp, ti * TR}, NsOperand{X, d.cp, tj * TC}, d.cp);
    else if constexpr (EPI == EPI_GRAM) {
        const NsOperand L = {X, d.cp, ti * TR}, R = {X, d.cp, tj * TC};
        if (!d.tall) product(rows, rows, L, R, d.cp);
        else product(kmajor, kmajor, L, R, d.rp);
    } else if constexpr (EPI == EPI_POLY) {
        const NsOperand L = {base + off_a(d), d.mp, ti * TR}, R = {base + off_a(d), d.mp, tj * TC};
        product(rows, rows, L, R, d.mp);
    } else {
        const half_t* P = base + off_p(d);
        if (!d.tall) product(rows, kmajor, NsOperand{P, d.mp, ti * TR}, NsOperand{X, d.cp, tj * TC}, d.mp);
        else product(rows, rows, NsOperand{X, d.cp, ti * TR}, NsOperand{P, d.mp, tj * TC}, d.mp);
    }
    float lr = 0.f, keep = 1.f;
    if constexpr (EPI == EPI_UPDATE) { lr = hyper[0]; keep = 1.f - lr * hyper[2]; lr *= p.scale[it]; }
    half_t* O = base + (GRAM ? off_a(d) : EPI == EPI_POLY ? off_p(d) : off_x(d, which ^ 1));
    const int ld = SYM ? d.mp : d.cp;
    // rows of the tile, 8 columns per thread
#pragma unroll 4
    for (int u = tid; u < TR * TC / 8; u += 256) {
        const int lrow = u / (TC / 8), lcol = (u % (TC / 8)) * 8, r = ti * TR + lrow, c = tj * TC + lcol;
        float* sp = S + lrow * PITCH + lcol;
        float v[8];
        {
            const f32x4 a = *reinterpret_cast<const f32x4*>(sp), b = *reinterpret_cast<const f32x4*>(sp + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
        }
        // GRAM: f0 = sA / sX^2, f2 = -shift sA.  POLY: f0 = c sP / sA^2, f1 = b' sP / sA, f2 = a' sP.  MULT: f0 = sX' / (sP sX).  Last: 1 / (sP sX)
        if constexpr (EPI == EPI_POLY) {
            const half_t* A = base + off_a(d) + ns_at(r, c, d.mp);
            const half8 ah = *reinterpret_cast<const half8*>(A), al = *reinterpret_cast<const half8*>(A + 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ns_poly(f, v[e], (float)ah[e] + (float)al[e], r == c + e);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= f.f0;
        }
        if constexpr (GRAM) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r == c + e ? f.f2 : 0.f;
        }
        if constexpr (SYM) {
            if (tj / Q != ti) {                                         // for the mirror image
                *reinterpret_cast<f32x4*>(sp) = f32x4{v[0], v[1], v[2], v[3]};
                *reinterpret_cast<f32x4*>(sp + 4) = f32x4{v[4], v[5], v[6], v[7]};
            }
        }
        if constexpr (SYM || EPI == EPI_MULT) ns_store8(O, r, c, ld, v);
        else {
            const int n = r < d.rows ? (d.cols - c < 8 ? d.cols - c : 8) : 0;
            if (n > 0) ns_finish8<EPI>(p, it, mat, r, c, n, lr, keep, f.zero_grad, v);
        }
    }
    if constexpr (SYM) {
        if (tj / Q == ti) return;
        __syncthreads();
        // the mirror image: 4 x 16 (8 columns of the output) x (rows of the output) per wave: one line per 4 lanes, LDS columns two lanes a bank
#pragma unroll 2
        for (int u = tid; u < TR * TC / 8; u += 256) {
            const int g = u >> 6, lcol8 = (g % (TR / 32)) * 4 + (u & 3), lrow = (g / (TR / 32)) * 16 + ((u >> 2) & 15);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = S[(lcol8 * 8 + e) * PITCH + lrow];
            ns_store8(O, (long)tj * TC + lrow, ti * TR + lcol8 * 8, ld, v);
        }
    }
}

// Polynomial and P X in one launch for smaller sides up to 192: a workgroup forms the 64 rows of P that its 64 x 64 tile needs by itself.  All of A
// (147 KB) is on its way to LDS at once; the band of P never leaves it.  Launches of this size last as long as their latencies
// (start, first load, store, gap: 4 of 5.5 us), so a third of the launches saved is worth the products done m / 64 times over.
// Eight waves: 2 x 4 over the band's 64 rows and A's m columns, then 2 x 4 over the 64 x 64 tile.
constexpr int SMALL_M = 192, SMALL_BYTES = SMALL_M * SMALL_M * 4, SMALL_PITCH = 68;
template <int MT>
__device__ __forceinline__ void ns_small_product(const half_t* A, const half_t* X, const NsDims& d, int ti, int tj, const NsScale& poly, unsigned char* smem) {
    constexpr int SK = 32, KT = MT * 64 / SK, STAGE = MT * 64 * 128, X_STAGE = 64 * 128;      // k of a stage, stages, bytes of A's and X's
    // X's tile takes the place of the first half of A's stages as soon as they are read, the band of P that of the second half; a 64-wide A leaves
    // them room behind it
    constexpr int HALF = (KT + 1) / 2;
    constexpr unsigned X_AT = MT == 1 ? KT * STAGE : 0, P_AT = MT == 1 ? KT * (STAGE + X_STAGE) : HALF * STAGE;
    static_assert(MT == 1 || (KT * X_STAGE <= HALF * STAGE && P_AT + KT * X_STAGE <= SMALL_BYTES && KT * STAGE <= SMALL_BYTES), "the tiles fit");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)smem);
    const int band = (d.tall ? tj : ti) * 64;
    {
        const NsOperand op = {A, MT * 64, 0};
        unsigned off[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) off[i] = ns_source<64, false>(op, wave * MT + i, lane);
#pragma unroll
        for (int s = 0; s < KT; ++s)
#pragma unroll
            for (int i = 0; i < MT; ++i) ns_dma(A + s * 64, off[i], lds0 + s * STAGE + (wave * MT + i) * 1024);
    }
    const int wr = (wave >> 2) * 32, wc = (wave & 3) * MT * 16;
    half4 ah[2][MT], al[2][MT];                                       // A's own elements under this wave's part of the band
    NsSums<2, MT, true> acc;
    acc.clear();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) ah[i][j] = al[i][j] = half4{0, 0, 0, 0};
    auto place = [&](int r, int c, int q) {                           // 4 elements at row r, column c of a stage: byte offset of plane q
        return r * 128 + (((4 * q + ((c % SK) >> 3)) ^ dma_swz64(r)) << 4) + (c & 7) * 2;
    };
    const unsigned lane_l = ns_lane<64, false>(smem, band + wr, lane), lane_r = ns_lane<64, false>(smem, wc, lane);
    auto square = [&](int s) {
        const unsigned char* st = smem + s * STAGE;
        NsFrags<2, MT> f;
        ns_read<64, 2, false>(f.l, lane_l + s * STAGE);
        ns_read<64, MT, false>(f.r, lane_r + s * STAGE);
#pragma unroll
        for (int j = 0; j < MT; ++j)
            if ((wc + j * 16) / SK == s) {                            // uniform
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int rr = band + wr + i * 16 + (lane & 15), c = wc + j * 16 + (lane >> 4) * 4;
                    ah[i][j] = *reinterpret_cast<const half4*>(st + place(rr, c, 0));
                    al[i][j] = *reinterpret_cast<const half4*>(st + place(rr, c, 1));
                }
            }
        ns_mfma<false>(f, acc);
    };
    // stage s has landed when at most what was issued behind it is outstanding
    auto first_half = [&](auto self, auto at) {
        constexpr int S = decltype(at)::value;
        if constexpr (S < HALF) {
            ns_wait<(KT - 1 - S) * MT, false>();
            ns_barrier();
            square(S);
            self(self, std::integral_constant<int, S + 1>());
        }
    };
    first_half(first_half, std::integral_constant<int, 0>());
    ns_wait<63, true>();
    ns_barrier();
    {
        const NsOperand op = {X, d.cp, (d.tall ? ti : tj) * 64};
        const half_t* src = d.tall ? ns_base<false>(op) : ns_base<true>(op);
        const long step = d.tall ? ns_step<false>(op) : ns_step<true>(op);
        const unsigned off = d.tall ? ns_source<64, false>(op, wave, lane) : ns_source<64, true>(op, wave, lane);
#pragma unroll
        for (int s = 0; s < KT; ++s) {
            ns_dma(src, off, lds0 + X_AT + s * X_STAGE + wave * 1024);
            src += step;
        }
    }
    auto second_half = [&](auto self, auto at) {
        constexpr int S = decltype(at)::value;
        if constexpr (S < KT) {
            ns_wait<KT + (KT - 1 - S) * MT, false>();
            ns_barrier();
            square(S);
            self(self, std::integral_constant<int, S + 1>());
        }
    };
    second_half(second_half, std::integral_constant<int, HALF>());
    ns_wait<63, true>();
    ns_barrier();                                                     // A has been read
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int r = wr + i * 16 + (lane & 15), c = wc + j * 16 + (lane >> 4) * 4;
            const f32x4 sq = acc.get(i, j);
            half4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                half_t x, y;
                split_half(ns_poly(poly, sq[e], (float)ah[i][j][e] + (float)al[i][j][e], band + r == c + e), x, y);
                h[e] = x;
                l[e] = y;
            }
            unsigned char* o = smem + P_AT + (c / SK) * X_STAGE;
            *reinterpret_cast<half4*>(o + place(r, c, 0)) = h;
            *reinterpret_cast<half4*>(o + place(r, c, 1)) = l;
        }
    ns_wait<0, true>();                                               // X's tile has landed, the band is written
    ns_barrier();
    NsSums<2, 1, true> out;
    out.clear();
    const int o_r = (wave >> 2) * 32, o_c = (wave & 3) * 16;
    auto last = [&](auto tall) {
        constexpr bool TALL = decltype(tall)::value;
        const unsigned ol = ns_lane<64, false>(smem + (TALL ? X_AT : P_AT), o_r, lane), o_right = ns_lane<64, !TALL>(smem + (TALL ? P_AT : X_AT), o_c, lane);
#pragma unroll
        for (int s = 0; s < KT; ++s) {
            NsFrags<2, 1> f;
            ns_read<64, 2, false>(f.l, ol + s * X_STAGE);
            ns_read<64, 1, !TALL>(f.r, o_right + s * X_STAGE);
            ns_mfma<false>(f, out);
        }
    };
    if (d.tall) last(std::true_type());
    else last(std::false_type());
    ns_wait<63, true>();
    ns_barrier();                                                     // the operands have been read: the tile in fp32 goes to the front
    float* S = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<f32x4*>(S + (o_r + i * 16 + (lane & 15)) * SMALL_PITCH + o_c + (lane >> 4) * 4) = out.get(i, 0);
    __syncthreads();
}
template <int EPI>
__global__ __launch_bounds__(512, 1) void ns_small_kernel(
    const NsTable t, const NsPtrs p, half_t* __restrict__ ws, const float* __restrict__ hyper, int which, const NsScale poly,
    const NsScale f) {
    extern __shared__ __attribute__((aligned(512))) unsigned char smem[];
    NsPlace w;
    if (!ns_place(t, w)) return;
    const int it = w.it, mat = w.mat, tile = w.tile;
    NsDims d = t.d[0];
    if (it) d = t.d[it];
    const int tc = d.cp / 64, ti = tile / tc, tj = tile - ti * tc, tid = threadIdx.x;
    half_t* base = ws + d.ws + mat * d.wsz;
    const half_t *A = base + off_a(d), *X = base + off_x(d, which);
    if (d.mp == 192) ns_small_product<3>(A, X, d, ti, tj, poly, smem);
    else if (d.mp == 128) ns_small_product<2>(A, X, d, ti, tj, poly, smem);
    else ns_small_product<1>(A, X, d, ti, tj, poly, smem);
    float lr = 0.f, keep = 1.f;
    if constexpr (EPI == EPI_UPDATE) { lr = hyper[0]; keep = 1.f - lr * hyper[2]; lr *= p.scale[it]; }
    const int lrow = tid >> 3, lcol = (tid & 7) * 8, r = ti * 64 + lrow, c = tj * 64 + lcol;
    float v[8];
    {
        const float* sp = reinterpret_cast<const float*>(smem) + lrow * SMALL_PITCH + lcol;
        const f32x4 a = *reinterpret_cast<const f32x4*>(sp), b = *reinterpret_cast<const f32x4*>(sp + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = a[e] * f.f0; v[4 + e] = b[e] * f.f0; }
    }
    if constexpr (EPI == EPI_MULT) ns_store8(base + off_x(d, which ^ 1), r, c, d.cp, v);
    else {
        const int n = r < d.rows ? (d.cols - c < 8 ? d.cols - c : 8) : 0;
        if (n > 0) ns_finish8<EPI>(p, it, mat, r, c, n, lr, keep, f.zero_grad, v);
    }
}

// ------------------------------------------------------------------------------------------------ host side
struct NsPlan {
    NsTable t;
    int pad;                          // sides are padded to multiples of it: 64 or 128
    long parts;                       // partial sums in front of the planes
    size_t bytes;
};
inline int up(int x, int to) { return (x + to - 1) / to * to; }

// Padding of a round: multiples of 128 allow the 128 x 128 tiles; not for sides that would grow by much or rounds too small to use them.
int pad_of(long padded64, long padded128) { return padded128 / (128 * 128) >= 128 && padded128 <= padded64 + padded64 / 4 ? 128 : 64; }
// the stacks [0, n) of one round: orientation, padding, workspace layout (partial sums first, then the planes)
bool ns_plan(NsPlan& pl, int n, const int* count, const int* rows, const int* cols) {
    memset(&pl, 0, sizeof(pl));
    pl.t.n = n;
    long padded[2] = {0, 0}, units = 0;
    for (int i = 0; i < n; ++i) {
        for (int k = 0; k < 2; ++k) padded[k] += (long)count[i] * up(rows[i], 64 << k) * up(cols[i], 64 << k);
        units += ((long)cols[i] + 7) / 8 * rows[i] * count[i];
    }
    // units of one partial sum: one per thread while that leaves few workgroups, else four (sum of squares, us with 256 / 1024 units: a 192-wide block
    // 5.5 / 7.2, ragged stacks of 309 k units 9.2 / 10.5, 12 x 1536 x 384 11.3 / 8.6)
    const long chunk = units <= 1024 * 512 ? 256 : 1024;
    pl.pad = pad_of(padded[0], padded[1]);
    long off = 0;
    for (int i = 0; i < n; ++i) {
        NsDims& d = pl.t.d[i];
        d.count = count[i]; d.rows = rows[i]; d.cols = cols[i];
        d.tall = rows[i] > cols[i];
        d.rp = up(rows[i], pl.pad); d.cp = up(cols[i], pl.pad); d.mp = d.tall ? d.cp : d.rp;
        const long chunks = (((long)cols[i] + 7) / 8 * rows[i] + chunk - 1) / chunk;
        d.chunks = (int)(chunks > 512 ? 512 : chunks);
        d.part = pl.parts;
        pl.parts += (long)d.count * d.chunks;
        d.wsz = 4L * d.rp * d.cp + 4L * d.mp * d.mp;
        d.ws = off;
        off += d.wsz * d.count;
    }
    pl.parts = (pl.parts + 31) / 32 * 32;
    pl.bytes = (size_t)pl.parts * sizeof(double) + (size_t)off * sizeof(half_t);
    return true;
}
enum { TILES_SUMSQ, TILES_LOAD, TILES_SYM, TILES_MULT };
// workgroups of every stack for one kind of launch on tiles of tr x tc; the size of the grid, -1: more than a grid holds
long ns_grid(NsTable& t, int kind, int tr = 64, int tc = 64) {
    long at = 0;
    for (int i = 0; i < t.n; ++i) {
        NsDims& d = t.d[i];
        const long tm = d.mp / tr;
        const long per = kind == TILES_SUMSQ ? d.chunks : kind == TILES_LOAD ? (long)d.rp * d.cp / 2048 : kind == TILES_SYM ? tr / tc * (tm * (tm + 1) / 2) : (long)(d.rp / tr) * (d.cp / tc);
        if (per * d.count >= (1L << 28)) return -1;
        d.per = (int)per;
        d.per_inv = per > 1 ? (unsigned)((1ULL << 32) / per) : 0xffffffffu;
        t.wgs[i] = (unsigned)(per * d.count);
        at += (t.wgs[i] + 7) / 8 * 8;
    }
    return at < (1L << 31) ? at : -1;
}
float pow2_under(double top, double bound) {     // largest power of two s with s * bound <= top
    int e;
    (void)frexp(top / bound, &e);
    return (float)ldexp(1., e - 1);
}
// bounds of |X| and |P| over the spectrum [0, bound] of one step; returns the next step's bound
double ns_bounds(double bound, double a, double b, double c, double& pmax) {
    double xmax = 0.;
    pmax = 0.;
    for (int i = 0; i <= 2048; ++i) {
        const double s = bound * i / 2048, q = fabs(a + (b + c * s * s) * s * s);
        if (q > pmax) pmax = q;
        if (q * s > xmax) xmax = q * s;
    }
    pmax = pmax > 1e-3 ? pmax * 1.01 : 1e-3;
    return xmax > 1e-3 ? xmax * 1.01 : 1e-3;
}

// Which tile a launch takes.  32 x 32, two on a CU, for products of pairs whose tiles fit on the CUs once over: a 64 x 64 tile of k = 768 fetches 393 KB
// through one CU (64 / 32, us for one Gram launch: 192 x 192, 6 / 21 tiles, 7.0 / 4.9; the four matrices of a 192-wide block, 24 / 84, 10.9 / 6.6.  Whole
// chains: 2 x 384^2 116 / 90, 512^2 128 / 92, 768^2 169 / 142, 700 x 3000 280 / 250), or nearly so if k is short (513 .. 560 tiles: k = 576 163 / 153, ragged
// stacks 178 / 170; k = 1024 190 / 204, k = 4000 371 / 445).
// Else the shortest estimate (Gram products of pairs with tall stacks among them, two k-major operands, need 268 / 177 registers: no 128 x 128 tiles, two
// 128 x 64 on a CU: 761 us for a 384-wide model's step, 788 with three and registers in scratch, 784 on 64 x 64) from times measured on pairs of planes, in us: 5 for a tile's start and end, plus per 32 k
// (n tiles on 256 CUs)                 64 x 64: 0.225, alone on its CU
//   128 x 128: 0.85 alone, 1.15 for two on a CU             128 x 64: 0.5 alone, 0.75 for two, 1.1 for three.
// Measured, 64 / 128 for the whole chain of five steps (tiles of 128 in the symmetric products / in P X): 12 x 384^2 (72 / 108) 166 / 236, 16 x 384^2
// (96 / 144) 251 / 239, 4 x 768^2 (84 / 144) 326 / 354, 12 x 768^2 (252 / 432) 657 / 469, 8 x 384 x 1536 (48 / 288) 277 / 374, 16 x (96 / 576) 493 / 439.
// 128 x 128 / 128 x 64 for one launch: the four products of twelve 384-wide blocks, Gram 52 / 48, polynomial 27 / 25, P X 63 / 67; 4 x 2048^2, Gram
// 126 / 121, polynomial 130 / 123, P X 179 / 197; ragged stacks of 192 tiles, P X 15 / 12.
int tile_kind(const NsTable& t, bool large, bool gram, bool sym, bool tall) {
    struct Sum { double n = 0., alone = 0., two = 0., three = 0.; } s64, s128, half;
    double n32 = 0.;
    auto add = [](Sum& s, double n, double stages, double alone, double two, double three) {
        s.n += n;
        s.two += n * (5. + two * stages);
        s.three += n * (5. + three * stages);
        s.alone = fmax(s.alone, 5. + alone * stages);
    };
    for (int i = 0; i < t.n; ++i) {
        const NsDims& d = t.d[i];
        const double stages = (gram ? (d.tall ? d.rp : d.cp) : d.mp) / 32;
        const double m3 = d.mp / 32, m6 = d.mp / 64, m12 = d.mp / 128;
        const double a = d.count * (sym ? m6 * (m6 + 1) / 2 : (double)(d.rp / 64) * (d.cp / 64));
        const double b = d.count * (sym ? m12 * (m12 + 1) / 2 : (double)(d.rp / 128) * (d.cp / 128));
        n32 += d.count * (sym ? m3 * (m3 + 1) / 2 : (double)(d.rp / 32) * (d.cp / 32));
        add(s64, a, stages, 0.225, 0.225, 0.);
        add(s128, b, stages, 0.85, 1.15, 0.);
        add(half, 2. * b, stages, 0.5, 0.75, 1.1);
    }
    if (n32 <= 512 || (n32 <= 640 && s64.two <= 12. * s64.n)) return TILE_32;
    const double t64 = ceil(s64.n / 256) * s64.two / s64.n;
    if (!large) return TILE_64;
    const double t128 = s128.n <= 256 ? s128.alone : ceil(s128.n / 512) * s128.two / s128.n;
    if (gram && tall) return (half.n <= 256 ? half.alone : fmax(half.alone, fmax(1., half.n / 512) * half.two / half.n)) < t64 ? TILE_HALF : TILE_64;
    const double th = half.n <= 256 ? half.alone : half.n <= 512 ? fmax(half.alone, half.two / half.n) : ceil(half.n / 768) * half.three / half.n;
    return th < t64 && th < t128 ? TILE_HALF : t128 < t64 ? TILE_128 : TILE_64;
}
template <int KIND, int EPI>
int launch_gemm_v(NsTable& t, const NsPtrs& p, half_t* ws, const float* hyper, int which, const NsScale& f, hipStream_t s) {
    using Tile = NsTile<KIND>;
    const long grid = ns_grid(t, EPI == EPI_GRAM || EPI == EPI_GRAM_ROWS || EPI == EPI_POLY ? TILES_SYM : TILES_MULT, Tile::TR, Tile::TC);
    S3D_REQUIRE(grid >= 0, "newton_schulz: too many tiles");
    auto k = ns_gemm_kernel<KIND, EPI>;
    if (Tile::BYTES > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, Tile::BYTES);
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(256), Tile::BYTES, s, t, p, ws, hyper, which, f);
    S3D_CHECK_LAUNCH_V("newton_schulz", KIND * 10 + EPI);
    return 0;
}
template <int EPI>
int launch_gemm(NsPlan& pl, const NsPtrs& p, half_t* ws, const float* hyper, int which, const NsScale& f, hipStream_t s) {
    bool tall = false;
    for (int i = 0; i < pl.t.n; ++i) tall |= pl.t.d[i].tall != 0;
    const int kind = tile_kind(pl.t, pl.pad == 128, EPI == EPI_GRAM, EPI == EPI_GRAM || EPI == EPI_POLY, tall);
    constexpr int ROWS = EPI == EPI_GRAM ? EPI_GRAM_ROWS : EPI;
    if (kind == TILE_32) return launch_gemm_v<TILE_32, EPI>(pl.t, p, ws, hyper, which, f, s);
    if (kind == TILE_64) return launch_gemm_v<TILE_64, EPI>(pl.t, p, ws, hyper, which, f, s);
    if (kind == TILE_128) return launch_gemm_v<TILE_128, ROWS>(pl.t, p, ws, hyper, which, f, s);
    return tall ? launch_gemm_v<TILE_HALF, EPI>(pl.t, p, ws, hyper, which, f, s) : launch_gemm_v<TILE_HALF, ROWS>(pl.t, p, ws, hyper, which, f, s);
}

// Polynomial and P X in one launch?  Sides that fit, tiles of P X on the CUs once over.  Whole call, two launches / one, us: 192 x 192 93 / 76, the
// four matrices of a 192-wide block 130 / 112.
bool small_sides(const NsTable& t) {
    long n = 0;
    for (int i = 0; i < t.n; ++i) {
        const NsDims& d = t.d[i];
        if (d.mp > SMALL_M) return false;
        n += (long)d.count * (d.rp / 64) * (d.cp / 64);
    }
    return n <= 256;
}
template <int EPI>
int launch_small(NsPlan& pl, const NsPtrs& p, half_t* ws, const float* hyper, int which, const NsScale& poly, const NsScale& mult, hipStream_t s) {
    const long grid = ns_grid(pl.t, TILES_MULT);
    S3D_REQUIRE(grid >= 0, "newton_schulz: too many tiles");
    auto k = ns_small_kernel<EPI>;
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, SMALL_BYTES);
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(512), SMALL_BYTES, s, pl.t, p, ws, hyper, which, poly, mult);
    S3D_CHECK_LAUNCH_V("newton_schulz_small", EPI);
    return 0;
}

template <int SRC, int LAST>
int ns_run(NsPlan& pl, const NsPtrs& p, const S3dNsArgs& a, const float* hyper, void* workspace, hipStream_t s) {
    double* part = reinterpret_cast<double*>(workspace);
    half_t* ws = reinterpret_cast<half_t*>(part + pl.parts);
    NsTable& t = pl.t;
    long at = ns_grid(t, TILES_SUMSQ);
    S3D_REQUIRE(at >= 0, "newton_schulz: too many matrices");
    hipLaunchKernelGGL(ns_sumsq_kernel<SRC>, dim3((unsigned)at), dim3(256), 0, s, t, p, hyper, a.nesterov, part);
    S3D_CHECK_LAUNCH_V("newton_schulz_sumsq", SRC);
    const bool small = small_sides(t);
    double bound = 1.001;
    float sx = pow2_under(32768., bound);
    at = ns_grid(t, TILES_LOAD);
    S3D_REQUIRE(at >= 0, "newton_schulz: too many tiles");
    hipLaunchKernelGGL(ns_load_kernel<SRC>, dim3((unsigned)at), dim3(256), 0, s, t, p, hyper, a.nesterov, part, a.eps, sx, ws);
    S3D_CHECK_LAUNCH_V("newton_schulz_load", SRC);
    for (int k = 0; k < a.steps; ++k) {
        double pmax;
        const double next = ns_bounds(bound, a.a, a.b, a.c, pmax);
        // What is kept of A and squared is A - shift I, in the middle of the spectrum: P = c (A - shift)^2 + b' (A - shift) + a'.  Near the end, where the
        // singular values are about 1, that square is a tenth of A^2 and so is what its sum loses (the whole result: a third less).
        const double shift = 0.375 * bound * bound, a1 = a.a + (a.b + a.c * shift) * shift, b1 = a.b + 2. * a.c * shift;
        const float sa = pow2_under(32768., bound * bound - shift), sp = pow2_under(32768., pmax), sn = pow2_under(32768., next);
        if (int rc = launch_gemm<EPI_GRAM>(pl, p, ws, hyper, k & 1, {sa / (sx * sx), 0.f, -(float)shift * sa, 0}, s)) return rc;
        const NsScale poly = {a.c * sp / (sa * sa), (float)b1 * sp / sa, (float)a1 * sp, 0}, mult = {sn / (sp * sx), 0.f, 0.f, 0}, last = {1.f / (sp * sx), 0.f, 0.f, a.zero_grad};
        const bool end = k + 1 == a.steps;
        int rc;
        if (small) {
            rc = end ? launch_small<LAST>(pl, p, ws, hyper, k & 1, poly, last, s) : launch_small<EPI_MULT>(pl, p, ws, hyper, k & 1, poly, mult, s);
        } else {
            rc = launch_gemm<EPI_POLY>(pl, p, ws, hyper, k & 1, poly, s);
            if (!rc) rc = end ? launch_gemm<LAST>(pl, p, ws, hyper, k & 1, last, s) : launch_gemm<EPI_MULT>(pl, p, ws, hyper, k & 1, mult, s);
        }
        if (rc) return rc;
        sx = sn;
        bound = next;
    }
    return 0;
}

int ns_check(const S3dNsArgs* a, const char* who) {
    S3D_REQUIRE(a != nullptr, "%s: null args", who);
    S3D_REQUIRE(a->steps >= 1 && a->steps <= 32, "%s: %d steps (1 .. 32)", who, a->steps);
    S3D_REQUIRE(isfinite(a->a) && isfinite(a->b) && isfinite(a->c), "%s: non-finite coefficients", who);
    S3D_REQUIRE(a->eps >= 1e-30f && isfinite(a->eps), "%s: eps must be at least 1e-30", who);
    double bound = 1.001, pmax;
    for (int k = 0; k < a->steps; ++k) {
        bound = ns_bounds(bound, a->a, a->b, a->c, pmax);
        S3D_REQUIRE(bound < 64. && pmax < 4096., "%s: the polynomial leaves the range of the products (a singular value may grow to %g at step %d)", who, bound, k);
    }
    return 0;
}
int ns_check_shape(const char* who, int i, int count, int rows, int cols) {
    S3D_REQUIRE(count >= 0 && rows >= 0 && cols >= 0, "%s: item %d has a negative size", who, i);
    S3D_REQUIRE(rows <= 65536 && cols <= 65536 && count <= (1 << 20), "%s: item %d is too large (%d x %d x %d)", who, i, count, rows, cols);
    return 0;
}
// The non-empty items in rounds of up to NS_ITEMS stacks, the longest products first (the workgroups that start last are then short ones):
// run(indices, number, rows, cols, count) until it returns non-zero.
template <typename Item, typename Run>
int ns_rounds(const Item* items, int n, Run run) {
    int idx[NS_ITEMS], k = 0;
    for (int i = 0; i <= n; ++i) {
        if (k == NS_ITEMS || (i == n && k > 0)) {
            NsPlan pl;
            int count[NS_ITEMS], rows[NS_ITEMS], cols[NS_ITEMS];
            for (int j = 0; j < k; ++j) { count[j] = items[idx[j]].count; rows[j] = items[idx[j]].rows; cols[j] = items[idx[j]].cols; }
            ns_plan(pl, k, count, rows, cols);
            if (int rc = run(pl, idx, k)) return rc;
            k = 0;
        }
        if (i == n) break;
        const Item& q = items[i];
        if (q.count == 0 || q.rows == 0 || q.cols == 0) continue;
        const int len = q.rows > q.cols ? q.rows : q.cols;
        int at = k++;
        for (; at > 0; --at) {
            const Item& o = items[idx[at - 1]];
            if ((o.rows > o.cols ? o.rows : o.cols) >= len) break;
            idx[at] = idx[at - 1];
        }
        idx[at] = i;
    }
    return 0;
}
template <typename Item>
size_t ns_workspace(const Item* items, int n) {
    size_t most = 256;
    for (int i = 0; i < n; ++i)
        if (ns_check_shape("newton_schulz", i, items[i].count, items[i].rows, items[i].cols)) return 0;
    ns_rounds(items, n, [&](const NsPlan& pl, const int*, int) {
        if (pl.bytes > most) most = pl.bytes;
        return 0;
    });
    return most;
}

// No tensor that is written may share elements with another one: the workgroups of a launch run in any order, and stacks beyond the sixteenth in
// later launches.  Sorted by address, each compared with those that begin inside it.
struct NsRanges {
    MatRange* v;
    long n = 0;
    explicit NsRanges(long most) : v((MatRange*)malloc(sizeof(MatRange) * (most > 0 ? most : 1))) {}
    ~NsRanges() { free(v); }
    NsRanges(const NsRanges&) = delete;
    NsRanges& operator=(const NsRanges&) = delete;
    void add(const void* p, int size, long stride, long ld, int count, int rows, int cols, bool write, int item) {
        uintptr_t at = (uintptr_t)p;
        if (count == 1) stride = 0;                                  // (says nothing)
        if (stride < 0) {                                            // an input may run backwards: the same matrices from the lowest one up
            at += (uintptr_t)((count - 1) * stride * size);
            stride = -stride;
        }
        v[n++] = MatRange{at, size, stride, ld, count, rows, cols, write, item};
    }
    // same_item: also tensors of one item
    int check(const char* who, bool same_item) {
        std::sort(v, v + n, [](const MatRange& a, const MatRange& b) { return a.at < b.at; });
        for (long i = 0; i < n; ++i) {
            const uintptr_t end = v[i].end();
            for (long j = i + 1; j < n && v[j].at < end; ++j) {
                if (!(v[i].write || v[j].write) || (!same_item && v[i].item == v[j].item)) continue;
                S3D_REQUIRE(!ranges_meet(v[i], v[j]), "%s: a tensor of item %d that is written shares memory with one of item %d", who, v[i].item, v[j].item);
            }
        }
        return 0;
    }
};

}  // namespace

size_t s3d_ortho_workspace(const S3dOrthoItem* items, int n) { return ns_workspace(items, n); }
size_t s3d_muon_workspace(const S3dMuonItem* items, int n) { return ns_workspace(items, n); }

int s3d_launch_orthogonalize(const S3dOrthoItem* items, int n, const S3dNsArgs* a, void* workspace, size_t bytes, hipStream_t s) {
    const char* who = "s3d_orthogonalize";
    if (int rc = ns_check(a, who)) return rc;
    S3D_REQUIRE(n >= 0 && (items || n == 0), "%s: null items", who);
    for (int i = 0; i < n; ++i) {
        const S3dOrthoItem& q = items[i];
        if (int rc = ns_check_shape(who, i, q.count, q.rows, q.cols)) return rc;
        if (q.count == 0 || q.rows == 0 || q.cols == 0) continue;
        S3D_REQUIRE(q.x && q.out, "%s: item %d has a null pointer", who, i);
        S3D_REQUIRE(q.x_ld >= q.cols && q.out_ld >= q.cols, "%s: item %d: row pitch below %d columns", who, i, q.cols);
        S3D_REQUIRE(q.count == 1 || q.out_stride >= (long)(q.rows - 1) * q.out_ld + q.cols, "%s: item %d: output matrices overlap", who, i);
    }
    if (n == 0) return 0;
    const size_t need = ns_workspace(items, n);
    S3D_REQUIRE(workspace && bytes >= need && ((uintptr_t)workspace & 15) == 0, "%s: the workspace needs %zu bytes, 16-byte aligned", who, need);
    NsRanges used(2L * n);
    S3D_REQUIRE(used.v, "%s: no host memory for %d items", who, n);
    for (int i = 0; i < n; ++i) {
        const S3dOrthoItem& q = items[i];
        if (q.count == 0 || q.rows == 0 || q.cols == 0) continue;
        used.add(q.x, a->x_bf16 ? 2 : 4, q.x_stride, q.x_ld, q.count, q.rows, q.cols, false, i);
        used.add(q.out, a->out_bf16 ? 2 : 4, q.out_stride, q.out_ld, q.count, q.rows, q.cols, true, i);
    }
    if (int rc = used.check(who, false)) return rc;
    return ns_rounds(items, n, [&](NsPlan& pl, const int* idx, int k) {
        NsPtrs p;
        memset(&p, 0, sizeof(p));
        for (int j = 0; j < k; ++j) {
            const S3dOrthoItem& q = items[idx[j]];
            p.x[j] = q.x; p.xs[j] = q.x_stride; p.xld[j] = q.x_ld;
            p.o[j] = q.out; p.os[j] = q.out_stride; p.old[j] = q.out_ld;
        }
        if (a->x_bf16) return a->out_bf16 ? ns_run<SRC_BF16, EPI_OUT_BF16>(pl, p, *a, nullptr, workspace, s) : ns_run<SRC_BF16, EPI_OUT_F32>(pl, p, *a, nullptr, workspace, s);
        return a->out_bf16 ? ns_run<SRC_F32, EPI_OUT_BF16>(pl, p, *a, nullptr, workspace, s) : ns_run<SRC_F32, EPI_OUT_F32>(pl, p, *a, nullptr, workspace, s);
    });
}

int s3d_launch_muon(const S3dMuonItem* items, int n, const S3dNsArgs* a, const float* hyper, void* workspace, size_t bytes, hipStream_t s) {
    const char* who = "s3d_muon_step";
    if (int rc = ns_check(a, who)) return rc;
    S3D_REQUIRE(n >= 0 && (items || n == 0), "%s: null items", who);
    S3D_REQUIRE(hyper, "%s: null hyper", who);
    for (int i = 0; i < n; ++i) {
        const S3dMuonItem& q = items[i];
        if (int rc = ns_check_shape(who, i, q.count, q.rows, q.cols)) return rc;
        if (q.count == 0 || q.rows == 0 || q.cols == 0) continue;
        S3D_REQUIRE(q.p && q.g && q.m, "%s: item %d has a null pointer", who, i);
        S3D_REQUIRE((q.hi == nullptr) == (q.lo == nullptr), "%s: item %d: both weight planes or none", who, i);
        S3D_REQUIRE(q.p_ld >= q.cols && q.g_ld >= q.cols && q.m_ld >= q.cols, "%s: item %d: row pitch below %d columns", who, i, q.cols);
        const long last = (long)(q.rows - 1);
        S3D_REQUIRE(q.count == 1 || (q.p_stride >= last * q.p_ld + q.cols && q.m_stride >= last * q.m_ld + q.cols && q.g_stride >= last * q.g_ld + q.cols),
                    "%s: item %d: matrices of the stack overlap", who, i);
        S3D_REQUIRE(isfinite(q.scale), "%s: item %d: non-finite scale", who, i);
    }
    if (n == 0) return 0;
    const size_t need = ns_workspace(items, n);
    S3D_REQUIRE(workspace && bytes >= need && ((uintptr_t)workspace & 15) == 0, "%s: the workspace needs %zu bytes, 16-byte aligned", who, need);
    NsRanges used(5L * n);
    S3D_REQUIRE(used.v, "%s: no host memory for %d items", who, n);
    for (int i = 0; i < n; ++i) {
        const S3dMuonItem& q = items[i];
        if (q.count == 0 || q.rows == 0 || q.cols == 0) continue;
        used.add(q.p, 4, q.p_stride, q.p_ld, q.count, q.rows, q.cols, true, i);
        used.add(q.m, 4, q.m_stride, q.m_ld, q.count, q.rows, q.cols, true, i);
        used.add(q.g, 4, q.g_stride, q.g_ld, q.count, q.rows, q.cols, a->zero_grad != 0, i);
        if (q.hi) {
            used.add(q.hi, 2, q.p_stride, q.p_ld, q.count, q.rows, q.cols, true, i);
            used.add(q.lo, 2, q.p_stride, q.p_ld, q.count, q.rows, q.cols, true, i);
        }
    }
    if (int rc = used.check(who, true)) return rc;
    return ns_rounds(items, n, [&](NsPlan& pl, const int* idx, int k) {
        NsPtrs p;
        memset(&p, 0, sizeof(p));
        for (int j = 0; j < k; ++j) {
            const S3dMuonItem& q = items[idx[j]];
            p.x[j] = q.g; p.xs[j] = q.g_stride; p.xld[j] = q.g_ld;
            p.o[j] = q.p; p.os[j] = q.p_stride; p.old[j] = q.p_ld;
            p.m[j] = q.m; p.ms[j] = q.m_stride; p.mld[j] = q.m_ld;
            p.hi[j] = q.hi; p.lo[j] = q.lo; p.scale[j] = q.scale;
        }
        return ns_run<SRC_MUON, EPI_UPDATE>(pl, p, *a, hyper, workspace, s);
    });
}
