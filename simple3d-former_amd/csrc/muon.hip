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
// hi hi + hi lo + lo hi with fp32 accumulation: an fp32 product at a third of the fp16 matrix rate, five times that of the fp32 matrix
// instructions.  fp16 planes rather than bf16: all entries are bounded by the spectral norm, so the exponent range is not needed and
// the six extra bits are.
#include <math.h>
#include <string.h>

#include "kernels.h"
#include "kmajor.h"

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
    long ws, wsz;                     // first matrix's planes in the workspace / planes per matrix (in halves)
    long part;                        // first matrix's partial sums
};
struct NsTable {
    int n;
    int tile0[NS_ITEMS + 1];          // first workgroup of every stack in this launch
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
enum { EPI_GRAM = 0, EPI_POLY = 1, EPI_MULT = 2, EPI_OUT_F32 = 3, EPI_OUT_BF16 = 4, EPI_UPDATE = 5 };

// Workgroups go round robin over the eight XCDs, each with an L2 of its own: XCD x takes the x-th eighth of the tile list, so that the
// tiles of one matrix share an L2.
__device__ __forceinline__ int xcd_order(int wg, int total) {
    const int q = total >> 3, r = total & 7, x = wg & 7;
    return x * q + (x < r ? x : r) + (wg >> 3);
}
__device__ __forceinline__ int ns_find(const NsTable& t, int wg) {
    int i = 0;
    while (i + 1 < t.n && wg >= t.tile0[i + 1]) ++i;
    return i;
}
// planes of one matrix, in halves from its base: X hi | lo [rp][cp] twice (read one, write the other), A hi | lo [mp][mp], P hi | lo [mp][mp]
__device__ __forceinline__ long off_x(const NsDims& d, int which) { return 2L * d.rp * d.cp * which; }
__device__ __forceinline__ long off_a(const NsDims& d) { return 4L * d.rp * d.cp; }
__device__ __forceinline__ long off_p(const NsDims& d) { return 4L * d.rp * d.cp + 2L * d.mp * d.mp; }

__device__ __forceinline__ void split_half(float v, half_t& hi, half_t& lo) {
    hi = (half_t)v;
    lo = (half_t)(v - (float)hi);
}

// momentum and the direction of the step, elementwise: m' = mu m + (1 - mu) g, u = nesterov ? (1 - mu) g + mu m' : m'
__device__ __forceinline__ float muon_mix(float g, float m, float mu) { return fmaf(mu, m, (1.f - mu) * g); }

// 8 consecutive elements (n of them inside the row, the rest 0); 16-byte loads where the address allows them
__device__ __forceinline__ void load8f(const float* p, int n, float* v) {
    if (n == 8 && ((uintptr_t)p & 15) == 0) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
    }
}
__device__ __forceinline__ void store8f(float* p, int n, const float* v) {
    if (n == 8 && ((uintptr_t)p & 15) == 0) {
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = v[i];
    }
}
__device__ __forceinline__ void load8b(const bf16_t* p, int n, float* v) {
    if (n == 8 && ((uintptr_t)p & 15) == 0) {
        U128 a;
        a.u = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = bf2f(a.h[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? bf2f(p[i]) : 0.f;
    }
}

// ---- 1. (momentum and) the sum of squares of every matrix: d.chunks partial sums in 64 bits, added in order by the next kernel ----
template <int SRC>
__global__ __launch_bounds__(256) void ns_sumsq_kernel(const NsTable t, const NsPtrs p, const float* __restrict__ hyper, int nesterov,
                                                       double* __restrict__ part) {
    const int it = ns_find(t, blockIdx.x);
    const NsDims& d = t.d[it];
    const int mat = (blockIdx.x - t.tile0[it]) / d.chunks, chunk = (blockIdx.x - t.tile0[it]) - mat * d.chunks;
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

// ---- 2. X0 = U / max(|U|, eps) as planes, padding cleared: 2048 elements of [rp][cp] per workgroup ----
template <int SRC>
__global__ __launch_bounds__(256) void ns_load_kernel(const NsTable t, const NsPtrs p, const float* __restrict__ hyper, int nesterov,
                                                      const double* __restrict__ part, float eps, float sx, half_t* __restrict__ ws) {
    const int it = ns_find(t, blockIdx.x);
    const NsDims& d = t.d[it];
    const int per = (int)((long)d.rp * d.cp / 2048);
    const int mat = (blockIdx.x - t.tile0[it]) / per, blk = (blockIdx.x - t.tile0[it]) - mat * per;
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
    const float inv = (float)(1. / (nrm > (double)eps ? nrm : (nrm == nrm ? (double)eps : nrm)));
    half8 h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        half_t a, b;
        split_half(i < n ? u[i] * inv * sx : 0.f, a, b);
        h[i] = a;
        l[i] = b;
    }
    half_t* X = ws + d.ws + mat * d.wsz + (long)r * d.cp + c;
    *reinterpret_cast<half8*>(X) = h;
    *reinterpret_cast<half8*>(X + (long)d.rp * d.cp) = l;
}

// ---- 3. the products ----
// One operand of a product: rows of k (KM false: element (i, k) at p + i ld + k) or columns (KM true: at p + k ld + i); the tile starts at i = at.
struct NsOperand { const half_t* p; long plane; int ld, at; };

template <int T, bool KM>
__device__ __forceinline__ half8 ns_frag(const unsigned char* tile, int i16, int lane) {
    if constexpr (!KM) {
        const int r = i16 + (lane & 15);
        return *reinterpret_cast<const half8*>(tile + r * 64 + (((lane >> 4) ^ dma_swz32(r)) << 4));
    } else {
        typedef __attribute__((ext_vector_type(4))) short short4v;
        typedef __attribute__((address_space(3))) short4v lds_short4;
        struct { short4v a, b; } u;
        const unsigned ad = kmajor_addr<T>(tile, i16, (lane >> 4) * 8, lane);
        u.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)ad);
        u.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)(ad + 4 * T * 2));
        return __builtin_bit_cast(half8, u);
    }
}

// acc = sum over k of L(i, k) R(j, k) for a T x T tile: 256 threads = 2 x 2 waves of T/2 x T/2, 32 k per stage, a ring of RING stages filled by
// LDS-DMA.  PL planes (2: hi hi + hi lo + lo hi).  acc[i][j][e] = C[wr + 16 i + (lane & 15)][wc + 16 j + 4 (lane >> 4) + e].
template <int T, int RING, int PL, bool LK, bool RK>
__device__ __forceinline__ void ns_product(const NsOperand& L, const NsOperand& R, int K, unsigned char* smem, f32x4 (&acc)[T / 32][T / 32]) {
    constexpr int PLANE = T * 64, STAGE = 2 * PL * PLANE;            // bytes; L hi (lo), R hi (lo)
    constexpr int PIECES = STAGE / 1024 / 4;                         // 1 KB DMA pieces per wave and stage
    constexpr int F = T / 32;                                        // 16-row fragments per wave and side
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const bf16_t* src[PIECES];
    long step[PIECES];                                               // (two values; constant per piece after unrolling)
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int q = wave * PIECES + i, plane = q / (T / 16), piece = q % (T / 16);
        const bool right = plane >= PL;
        const NsOperand& o = right ? R : L;
        const bool km = right ? RK : LK;
        const int wk = T / 8;                                        // 16-byte slots of a k-major row
        const int r = km ? piece * (64 / wk) + lane / wk : piece * 16 + (lane >> 2);
        const int chunk = km ? (lane % wk) ^ kmajor_swz<T>(r) : (lane & 3) ^ dma_swz32(r);
        const half_t* pl = o.p + (plane - (right ? PL : 0)) * o.plane;
        src[i] = reinterpret_cast<const bf16_t*>(km ? pl + (long)r * o.ld + o.at + chunk * 8 : pl + ((long)o.at + r) * o.ld + chunk * 8);
        step[i] = km ? 32L * o.ld : 32;
    }
    const unsigned lds0 = (unsigned)(uintptr_t)smem + wave * PIECES * 1024;
    const int KT = K / 32;
    int slot_in = 0, slot = 0;
    auto issue = [&]() {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            glds16(src[i], __builtin_amdgcn_readfirstlane(lds0 + slot_in * STAGE + i * 1024));
            src[i] += step[i];
        }
        slot_in = slot_in + 1 == RING ? 0 : slot_in + 1;
    };
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < RING - 1 && k < KT; ++k) issue();
    const int wr = (wave >> 1) * (T / 2), wc = (wave & 1) * (T / 2);
    for (int kt = 0; kt < KT; ++kt) {
        // stage kt has landed when at most the later stages' pieces are outstanding; the barrier also tells that every wave has read
        // stage kt - 1, whose slot is refilled next
        if (kt + RING - 2 < KT) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RING - 2) * PIECES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (kt + RING - 1 < KT) issue();
        const unsigned char* st = smem + slot * STAGE;
        slot = slot + 1 == RING ? 0 : slot + 1;
        half8 l[PL][F], r[PL][F];
#pragma unroll
        for (int q = 0; q < PL; ++q)
#pragma unroll
            for (int i = 0; i < F; ++i) {
                l[q][i] = ns_frag<T, LK>(st + q * PLANE, wr + i * 16, lane);
                r[q][i] = ns_frag<T, RK>(st + (PL + q) * PLANE, wc + i * 16, lane);
            }
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(r[0][j], l[0][i], acc[i][j], 0, 0, 0);
        if constexpr (PL == 2) {
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(r[1][j], l[0][i], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(r[0][j], l[1][i], acc[i][j], 0, 0, 0);
        }
    }
}

// f0 .. f2: scale factors of the epilogue; low: the planes written are pairs (0: the next product takes the hi plane only)
template <int T, int RING, int PL, int EPI>
__global__ __launch_bounds__(256) void ns_gemm_kernel(const NsTable t, const NsPtrs p, half_t* __restrict__ ws, const float* __restrict__ hyper,
                                                      int which, float f0, float f1, float f2, int low, int zero_grad) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr int F = T / 32;
    constexpr bool SYM = EPI == EPI_GRAM || EPI == EPI_POLY;
    const int wg = xcd_order(blockIdx.x, gridDim.x);
    const int it = ns_find(t, wg);
    const NsDims& d = t.d[it];
    const int tm = d.mp / T, tc = d.cp / T;
    const int per = SYM ? tm * (tm + 1) / 2 : (d.rp / T) * tc;
    const int mat = (wg - t.tile0[it]) / per, tile = (wg - t.tile0[it]) - mat * per;
    int ti, tj;
    if constexpr (SYM) {                                             // lower triangle, row by row: tile = ti (ti + 1) / 2 + tj
        ti = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
        while (ti * (ti + 1) / 2 > tile) --ti;
        while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
        tj = tile - ti * (ti + 1) / 2;
    } else {
        ti = tile / tc;
        tj = tile - ti * tc;
    }
    half_t* base = ws + d.ws + mat * d.wsz;
    const long xx = (long)d.rp * d.cp, mm = (long)d.mp * d.mp;
    const half_t* X = base + off_x(d, which);
    f32x4 acc[F][F];
    if constexpr (EPI == EPI_GRAM) {
        const NsOperand L = {X, xx, d.cp, ti * T}, R = {X, xx, d.cp, tj * T};
        if (!d.tall) ns_product<T, RING, PL, false, false>(L, R, d.cp, smem, acc);
        else ns_product<T, RING, PL, true, true>(L, R, d.rp, smem, acc);
    } else if constexpr (EPI == EPI_POLY) {
        const NsOperand L = {base + off_a(d), mm, d.mp, ti * T}, R = {base + off_a(d), mm, d.mp, tj * T};
        ns_product<T, RING, PL, false, false>(L, R, d.mp, smem, acc);
    } else {
        const half_t* P = base + off_p(d);
        if (!d.tall) {
            const NsOperand L = {P, mm, d.mp, ti * T}, R = {X, xx, d.cp, tj * T};
            ns_product<T, RING, PL, false, true>(L, R, d.mp, smem, acc);
        } else {
            const NsOperand L = {X, xx, d.cp, ti * T}, R = {P, mm, d.mp, tj * T};
            ns_product<T, RING, PL, false, false>(L, R, d.mp, smem, acc);
        }
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int row = ti * T + (wave >> 1) * (T / 2) + (lane & 15), col = tj * T + (wave & 1) * (T / 2) + (lane >> 4) * 4;
    float lr = 0.f, keep = 1.f;
    if constexpr (EPI == EPI_UPDATE) { lr = hyper[0]; keep = 1.f - lr * hyper[2]; lr *= p.scale[it]; }
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
            const int r = row + i * 16, c = col + j * 16;
            f32x4 v = acc[i][j];
            if constexpr (SYM || EPI == EPI_MULT) {
                half_t* O;
                long ld, pl;
                if constexpr (EPI == EPI_GRAM) {                     // f0 = sA / sX^2
                    v *= f0;
                    O = base + off_a(d); ld = d.mp; pl = mm;
                } else if constexpr (EPI == EPI_POLY) {              // v = (a I + b A + c A^2) sP: f0 = c sP / sA^2, f1 = b sP / sA, f2 = a sP
                    const half_t* A = base + off_a(d) + (long)r * d.mp + c;
                    const half4 ah = *reinterpret_cast<const half4*>(A);
                    half4 al = {0, 0, 0, 0};
                    if constexpr (PL == 2) al = *reinterpret_cast<const half4*>(A + mm);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = fmaf(v[e], f0, f1 * ((float)ah[e] + (float)al[e])) + (r == c + e ? f2 : 0.f);
                    O = base + off_p(d); ld = d.mp; pl = mm;
                } else {                                             // f0 = sX' / (sP sX)
                    v *= f0;
                    O = base + off_x(d, which ^ 1); ld = d.cp; pl = xx;
                }
                half4 h, l;
#pragma unroll
                for (int e = 0; e < 4; ++e) { half_t a, b; split_half(v[e], a, b); h[e] = a; l[e] = b; }
                *reinterpret_cast<half4*>(O + (long)r * ld + c) = h;
                if (low) *reinterpret_cast<half4*>(O + pl + (long)r * ld + c) = l;
                if (SYM && ti != tj) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) O[(long)(c + e) * ld + r] = h[e];
                    if (low) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) O[pl + (long)(c + e) * ld + r] = l[e];
                    }
                }
            } else {                                                 // f0 = 1 / (sP sX)
                if (r >= d.rows || c >= d.cols) continue;
                v *= f0;
                const long oi = mat * p.os[it] + (long)r * p.old[it] + c;
                const int n = d.cols - c < 4 ? d.cols - c : 4;
                if constexpr (EPI == EPI_OUT_BF16) {
                    bf16_t* o = (bf16_t*)p.o[it] + oi;
                    if (n == 4 && ((uintptr_t)o & 7) == 0) *reinterpret_cast<u32x2*>(o) = u32x2{f2bf2(v[0], v[1]), f2bf2(v[2], v[3])};
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (e < n) o[e] = f2bf(v[e]);
                    continue;
                }
                float* o = (float*)p.o[it] + oi;
                const bool vec = n == 4 && ((uintptr_t)o & 15) == 0;
                if constexpr (EPI == EPI_UPDATE) {
                    f32x4 w = {0.f, 0.f, 0.f, 0.f};
                    if (vec) w = *reinterpret_cast<const f32x4*>(o);
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (e < n) w[e] = o[e];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = fmaf(-lr, v[e], w[e] * keep);
                    if (p.hi[it]) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (e < n) {
                                bf16_t h, l;
                                split_bf16(v[e], h, l);
                                p.hi[it][oi + e] = h;
                                p.lo[it][oi + e] = l;
                            }
                    }
                    if (zero_grad) {
                        float* g = (float*)p.x[it] + mat * p.xs[it] + (long)r * p.xld[it] + c;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (e < n) g[e] = 0.f;
                    }
                }
                if (vec) *reinterpret_cast<f32x4*>(o) = v;
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < n) o[e] = v[e];
            }
        }
}

// ------------------------------------------------------------------------------------------------ host side
struct NsPlan {
    NsTable t;
    int T;                            // tile
    long parts;                       // partial sums in front of the planes
    size_t bytes;
};
inline int up(int x, int to) { return (x + to - 1) / to * to; }

// Tile of a round by its padded elements: 128 x 128 tiles halve the LDS and L2 traffic of a product, 64 x 64 tiles pad less and spread over more CUs.
int tile_of(long padded64, long padded128) {
    return padded128 / (128 * 128) >= 256 && padded128 <= padded64 + padded64 / 4 ? 128 : 64;
}
// the stacks [0, n) of one round: orientation, padding, workspace layout (partial sums first, then the planes)
bool ns_plan(NsPlan& pl, int n, const int* count, const int* rows, const int* cols) {
    memset(&pl, 0, sizeof(pl));
    pl.t.n = n;
    long padded[2] = {0, 0};
    for (int i = 0; i < n; ++i)
        for (int k = 0; k < 2; ++k) padded[k] += (long)count[i] * up(rows[i], 64 << k) * up(cols[i], 64 << k);
    pl.T = tile_of(padded[0], padded[1]);
    long off = 0;
    for (int i = 0; i < n; ++i) {
        NsDims& d = pl.t.d[i];
        d.count = count[i]; d.rows = rows[i]; d.cols = cols[i];
        d.tall = rows[i] > cols[i];
        d.rp = up(rows[i], pl.T); d.cp = up(cols[i], pl.T); d.mp = d.tall ? d.cp : d.rp;
        const long units = ((long)cols[i] + 7) / 8 * rows[i], chunks = (units + 1023) / 1024;
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
// first workgroup of every stack for one kind of launch; the number of workgroups, -1: more than a grid holds
long ns_tiles(NsTable& t, int T, int kind) {
    long at = 0;
    for (int i = 0; i < t.n; ++i) {
        t.tile0[i] = (int)at;
        const NsDims& d = t.d[i];
        const long tm = d.mp / T;
        const long per = kind == TILES_SUMSQ ? d.chunks : kind == TILES_LOAD ? (long)d.rp * d.cp / 2048 : kind == TILES_SYM ? tm * (tm + 1) / 2 : (long)(d.rp / T) * (d.cp / T);
        at += per * d.count;
        if (at > 0x7fffffffL) return -1;
    }
    t.tile0[t.n] = (int)at;
    return at;
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

template <int EPI, int T, int RING, int PL>
int launch_gemm_v(const NsTable& t, const NsPtrs& p, half_t* ws, const float* hyper, int which, float f0, float f1, float f2, int low, int zero_grad,
                  long tiles, hipStream_t s) {
    constexpr int bytes = RING * 2 * PL * T * 64;
    auto k = ns_gemm_kernel<T, RING, PL, EPI>;
    if (bytes > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(256), bytes, s, t, p, ws, hyper, which, f0, f1, f2, low, zero_grad);
    S3D_CHECK_LAUNCH_V("newton_schulz", T * 100 + PL * 10 + EPI);
    return 0;
}
template <int EPI>
int launch_gemm(int T, int pl, const NsTable& t, const NsPtrs& p, half_t* ws, const float* hyper, int which, float f0, float f1, float f2, int low,
                int zero_grad, long tiles, hipStream_t s) {
    if (T == 128) {
        if (pl == 2) return launch_gemm_v<EPI, 128, 2, 2>(t, p, ws, hyper, which, f0, f1, f2, low, zero_grad, tiles, s);
        return launch_gemm_v<EPI, 128, 4, 1>(t, p, ws, hyper, which, f0, f1, f2, low, zero_grad, tiles, s);
    }
    if (pl == 2) return launch_gemm_v<EPI, 64, 4, 2>(t, p, ws, hyper, which, f0, f1, f2, low, zero_grad, tiles, s);
    return launch_gemm_v<EPI, 64, 4, 1>(t, p, ws, hyper, which, f0, f1, f2, low, zero_grad, tiles, s);
}

template <int SRC, int LAST>
int ns_run(NsPlan& pl, const NsPtrs& p, const S3dNsArgs& a, const float* hyper, void* workspace, hipStream_t s) {
    double* part = reinterpret_cast<double*>(workspace);
    half_t* ws = reinterpret_cast<half_t*>(part + pl.parts);
    NsTable& t = pl.t;
    long at = ns_tiles(t, pl.T, TILES_SUMSQ);
    S3D_REQUIRE(at >= 0, "newton_schulz: too many matrices");
    hipLaunchKernelGGL(ns_sumsq_kernel<SRC>, dim3((unsigned)at), dim3(256), 0, s, t, p, hyper, a.nesterov, part);
    S3D_CHECK_LAUNCH_V("newton_schulz_sumsq", SRC);
    double bound = 1.001;
    float sx = pow2_under(32768., bound);
    at = ns_tiles(t, pl.T, TILES_LOAD);
    S3D_REQUIRE(at >= 0, "newton_schulz: too many tiles");
    hipLaunchKernelGGL(ns_load_kernel<SRC>, dim3((unsigned)at), dim3(256), 0, s, t, p, hyper, a.nesterov, part, a.eps, sx, ws);
    S3D_CHECK_LAUNCH_V("newton_schulz_load", SRC);
    const long sym = ns_tiles(t, pl.T, TILES_SYM);
    // Results kept in bf16: the last two steps run on the hi planes alone.  What they round (2^-12) is multiplied by at most a and 1 before the
    // result, which adds about 1e-3 to the 1.7e-3 (2-norm) of the result's own rounding, whatever the spectrum; a third such step would triple it.
    const int plain_from = LAST == EPI_OUT_BF16 ? a.steps - 2 : a.steps;
    for (int k = 0; k < a.steps; ++k) {
        double pmax;
        const double next = ns_bounds(bound, a.a, a.b, a.c, pmax);
        const float sa = pow2_under(32768., bound * bound), sp = pow2_under(32768., pmax), sn = pow2_under(32768., next);
        const int planes = k >= plain_from ? 1 : 2, low = planes == 2, low_x = k + 1 < plain_from;
        ns_tiles(t, pl.T, TILES_SYM);
        if (int rc = launch_gemm<EPI_GRAM>(pl.T, planes, t, p, ws, hyper, k & 1, sa / (sx * sx), 0.f, 0.f, low, 0, sym, s)) return rc;
        if (int rc = launch_gemm<EPI_POLY>(pl.T, planes, t, p, ws, hyper, k & 1, a.c * sp / (sa * sa), a.b * sp / sa, a.a * sp, low, 0, sym, s)) return rc;
        at = ns_tiles(t, pl.T, TILES_MULT);
        if (k + 1 < a.steps) {
            if (int rc = launch_gemm<EPI_MULT>(pl.T, planes, t, p, ws, hyper, k & 1, sn / (sp * sx), 0.f, 0.f, low_x, 0, at, s)) return rc;
        } else {
            if (int rc = launch_gemm<LAST>(pl.T, planes, t, p, ws, hyper, k & 1, 1.f / (sp * sx), 0.f, 0.f, 0, a.zero_grad, at, s)) return rc;
        }
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
template <typename Item>
size_t ns_workspace(const Item* items, int n) {
    size_t most = 0;
    int count[NS_ITEMS], rows[NS_ITEMS], cols[NS_ITEMS], k = 0;
    NsPlan pl;
    for (int i = 0; i <= n; ++i) {
        if (k == NS_ITEMS || (i == n && k > 0)) {
            ns_plan(pl, k, count, rows, cols);
            if (pl.bytes > most) most = pl.bytes;
            k = 0;
        }
        if (i == n) break;
        if (ns_check_shape("newton_schulz", i, items[i].count, items[i].rows, items[i].cols)) return 0;
        if (items[i].count == 0 || items[i].rows == 0 || items[i].cols == 0) continue;
        count[k] = items[i].count; rows[k] = items[i].rows; cols[k] = items[i].cols;
        ++k;
    }
    return most ? most : 256;
}

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
    const size_t need = ns_workspace(items, n);
    S3D_REQUIRE(workspace && bytes >= need && ((uintptr_t)workspace & 15) == 0, "%s: the workspace needs %zu bytes, 16-byte aligned", who, need);
    int count[NS_ITEMS], rows[NS_ITEMS], cols[NS_ITEMS], k = 0;
    NsPlan pl;
    NsPtrs p;
    memset(&p, 0, sizeof(p));
    for (int i = 0; i <= n; ++i) {
        if (k == NS_ITEMS || (i == n && k > 0)) {
            ns_plan(pl, k, count, rows, cols);
            int rc;
            if (a->x_bf16) rc = a->out_bf16 ? ns_run<SRC_BF16, EPI_OUT_BF16>(pl, p, *a, nullptr, workspace, s) : ns_run<SRC_BF16, EPI_OUT_F32>(pl, p, *a, nullptr, workspace, s);
            else rc = a->out_bf16 ? ns_run<SRC_F32, EPI_OUT_BF16>(pl, p, *a, nullptr, workspace, s) : ns_run<SRC_F32, EPI_OUT_F32>(pl, p, *a, nullptr, workspace, s);
            if (rc) return rc;
            k = 0;
        }
        if (i == n) break;
        const S3dOrthoItem& q = items[i];
        if (q.count == 0 || q.rows == 0 || q.cols == 0) continue;
        count[k] = q.count; rows[k] = q.rows; cols[k] = q.cols;
        p.x[k] = q.x; p.xs[k] = q.x_stride; p.xld[k] = q.x_ld;
        p.o[k] = q.out; p.os[k] = q.out_stride; p.old[k] = q.out_ld;
        ++k;
    }
    return 0;
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
    const size_t need = ns_workspace(items, n);
    S3D_REQUIRE(workspace && bytes >= need && ((uintptr_t)workspace & 15) == 0, "%s: the workspace needs %zu bytes, 16-byte aligned", who, need);
    int count[NS_ITEMS], rows[NS_ITEMS], cols[NS_ITEMS], k = 0;
    NsPlan pl;
    NsPtrs p;
    memset(&p, 0, sizeof(p));
    for (int i = 0; i <= n; ++i) {
        if (k == NS_ITEMS || (i == n && k > 0)) {
            ns_plan(pl, k, count, rows, cols);
            if (int rc = ns_run<SRC_MUON, EPI_UPDATE>(pl, p, *a, hyper, workspace, s)) return rc;
            k = 0;
        }
        if (i == n) break;
        const S3dMuonItem& q = items[i];
        if (q.count == 0 || q.rows == 0 || q.cols == 0) continue;
        count[k] = q.count; rows[k] = q.rows; cols[k] = q.cols;
        p.x[k] = q.g; p.xs[k] = q.g_stride; p.xld[k] = q.g_ld;
        p.o[k] = q.p; p.os[k] = q.p_stride; p.old[k] = q.p_ld;
        p.m[k] = q.m; p.ms[k] = q.m_stride; p.mld[k] = q.m_ld;
        p.hi[k] = q.hi; p.lo[k] = q.lo; p.scale[k] = q.scale;
        ++k;
    }
    return 0;
}
