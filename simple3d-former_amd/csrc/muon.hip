// Orthogonalised updates: Newton-Schulz products over stacks of weight matrices (s3d_orthogonalize) and the optimizer step built on them
// (s3d_muon_step).
//
// Mathematics.  X0 = U / max(|U|_F, eps) with the smaller side as rows (m <= n); `steps` times
//     A = X X^T (m x m),   P = a I + b A + c A^2 (m x m),   X <- P X
// i.e. every singular value s of X0 becomes p(p(..p(s))) with p(s) = a s + b s^3 + c s^5, the singular vectors stay.  All products are
// "row by row" (C = L R^T with both operands k-contiguous): the Gram product reads X, the square reads the symmetric A twice, and P X
// reads P and the transpose of X, so X is kept in both orientations ([m][n] for the Gram product, [n][m] for P X).  The two symmetric
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

#include "dma_tile.h"
#include "kernels.h"

namespace {

typedef _Float16 half_t;
typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(4))) _Float16 half4;

constexpr int NS_ITEMS = 16;          // stacks of one launch (kernel-argument table); more are worked in several rounds
constexpr int NS_CHUNKS = 64;         // partial sums of squares per matrix

struct NsDims {
    int count, rows, cols;            // the caller's matrices
    int m, n, mp, np;                 // working orientation m <= n, padded to the tile
    long ws, wsz;                     // first matrix's planes in the workspace / planes per matrix (in halves)
    int mat0;                         // global index of the stack's first matrix (partial sums)
};
struct NsTable {
    NsDims d[NS_ITEMS];
    int tile0[NS_ITEMS + 1];          // first workgroup of every stack in this launch
    int n;
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

__device__ __forceinline__ int ns_find(const NsTable& t, int wg, int per, int& mat, int& tile) {
    int i = 0;
    while (i + 1 < t.n && wg >= t.tile0[i + 1]) ++i;
    const int r = wg - t.tile0[i];
    mat = r / per;
    tile = r - mat * per;
    return i;
}
// planes of one matrix, in halves from its base: X hi | lo [mp][np], XT hi | lo [np][mp] twice, A hi | lo [mp][mp], B hi | lo [mp][mp]
__device__ __forceinline__ long off_xt(const NsDims& d, int which) { return 2L * d.mp * d.np * (1 + which); }
__device__ __forceinline__ long off_a(const NsDims& d) { return 6L * d.mp * d.np; }
__device__ __forceinline__ long off_b(const NsDims& d) { return 6L * d.mp * d.np + 2L * d.mp * d.mp; }

__device__ __forceinline__ void split_half(float v, half_t& hi, half_t& lo) {
    hi = (half_t)v;
    lo = (half_t)(v - (float)hi);
}

// momentum and the direction of the step, elementwise: m' = mu m + (1 - mu) g, u = nesterov ? (1 - mu) g + mu m' : m'
__device__ __forceinline__ float muon_mix(float g, float m, float mu) { return fmaf(mu, m, (1.f - mu) * g); }

// ---- 1. (momentum and) the sum of squares of every matrix: NS_CHUNKS partial sums in 64 bits, added in order by the next kernel ----
template <int SRC>
__global__ __launch_bounds__(256) void ns_sumsq_kernel(const NsTable t, const NsPtrs p, const float* __restrict__ hyper, int nesterov,
                                                       double* __restrict__ part) {
    int mat, chunk;
    const int it = ns_find(t, blockIdx.x, NS_CHUNKS, mat, chunk);
    const NsDims& d = t.d[it];
    const long total = (long)d.rows * d.cols, per = (total + NS_CHUNKS - 1) / NS_CHUNKS;
    const long lo = chunk * per, hi = lo + per < total ? lo + per : total;
    float mu = 0.f, gs = 1.f;
    if constexpr (SRC == SRC_MUON) { mu = hyper[1]; gs = hyper[3]; }
    double s = 0.;
    for (long e = lo + threadIdx.x; e < hi; e += 256) {
        const long r = e / d.cols, c = e - r * d.cols;
        float u;
        const long xi = mat * p.xs[it] + r * p.xld[it] + c;
        if constexpr (SRC == SRC_BF16) u = bf2f(((const bf16_t*)p.x[it])[xi]);
        else u = ((const float*)p.x[it])[xi];
        if constexpr (SRC == SRC_MUON) {
            float* mp = p.m[it] + mat * p.ms[it] + r * p.mld[it] + c;
            const float g = u * gs, mn = muon_mix(g, *mp, mu);
            *mp = mn;
            u = nesterov ? muon_mix(g, mn, mu) : mn;
        }
        s += (double)u * u;
    }
    __shared__ double red[256];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if (threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0) part[(long)(d.mat0 + mat) * NS_CHUNKS + chunk] = red[0];
}

// ---- 2. X0 = U / max(|U|, eps) as planes in both orientations, padding cleared: one workgroup per 64 x 64 tile of [mp][np] ----
template <int SRC>
__global__ __launch_bounds__(256) void ns_load_kernel(const NsTable t, const NsPtrs p, const float* __restrict__ hyper, int nesterov,
                                                      const double* __restrict__ part, float eps, float sx, half_t* __restrict__ ws) {
    int mat, tile;
    int it = 0;
    while (it + 1 < t.n && (int)blockIdx.x >= t.tile0[it + 1]) ++it;
    const NsDims& d = t.d[it];
    const int tn = d.np / 64, per = (d.mp / 64) * tn;
    {
        const int r = blockIdx.x - t.tile0[it];
        mat = r / per;
        tile = r - mat * per;
    }
    const int ti = tile / tn, tj = tile - ti * tn;
    __shared__ float buf[64][65];
    double s = 0.;
    for (int k = 0; k < NS_CHUNKS; ++k) s += part[(long)(d.mat0 + mat) * NS_CHUNKS + k];
    const double nrm = sqrt(s);
    const float inv = (float)(1. / (nrm > (double)eps ? nrm : (nrm == nrm ? (double)eps : nrm)));
    float mu = 0.f, gs = 1.f;
    if constexpr (SRC == SRC_MUON) { mu = hyper[1]; gs = hyper[3]; }
    const bool tall = d.rows > d.cols;
    // source tile: rows r0.., columns c0.. of the caller's matrix
    const int r0 = tall ? tj * 64 : ti * 64, c0 = tall ? ti * 64 : tj * 64;
    for (int e = threadIdx.x; e < 4096; e += 256) {
        const int r = e >> 6, c = e & 63;
        float u = 0.f;
        if (r0 + r < d.rows && c0 + c < d.cols) {
            const long xi = mat * p.xs[it] + (long)(r0 + r) * p.xld[it] + c0 + c;
            if constexpr (SRC == SRC_BF16) u = bf2f(((const bf16_t*)p.x[it])[xi]);
            else u = ((const float*)p.x[it])[xi];
            if constexpr (SRC == SRC_MUON) {
                const float mn = p.m[it][mat * p.ms[it] + (long)(r0 + r) * p.mld[it] + c0 + c];
                u = nesterov ? muon_mix(u * gs, mn, mu) : mn;
            }
            u *= inv;
        }
        buf[r][c] = u * sx;
    }
    __syncthreads();
    half_t* base = ws + d.ws + mat * d.wsz;
    half_t* X = base + (long)ti * 64 * d.np + tj * 64;                         // [mp][np]
    half_t* XT = base + off_xt(d, 0) + (long)tj * 64 * d.mp + ti * 64;         // [np][mp]
    const long plane = (long)d.mp * d.np;
    for (int e = threadIdx.x; e < 4096; e += 256) {
        const int r = e >> 6, c = e & 63;
        half_t hi, lo;
        split_half(tall ? buf[c][r] : buf[r][c], hi, lo);                      // X[r][c]
        X[(long)r * d.np + c] = hi;
        X[plane + (long)r * d.np + c] = lo;
        split_half(tall ? buf[r][c] : buf[c][r], hi, lo);                      // XT[r][c]
        XT[(long)r * d.mp + c] = hi;
        XT[plane + (long)r * d.mp + c] = lo;
    }
}

// ---- 3. the products ----
// C = L R^T on T x T tiles: 256 threads = 2 x 2 waves of T/2 x T/2, 32 k per stage, a ring of RING stages filled by LDS-DMA.
template <int T, int RING, int EPI>
__global__ __launch_bounds__(256) void ns_gemm_kernel(const NsTable t, const NsPtrs p, half_t* __restrict__ ws, const float* __restrict__ hyper,
                                                      int which, float f0, float f1, float f2, float f3, int zero_grad) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr int PLANE = T * 64, STAGE = 4 * PLANE;                 // bytes: T rows of 32 halves; L hi, L lo, R hi, R lo
    constexpr int PIECES = STAGE / 1024 / 4;                         // 1 KB DMA pieces per wave and stage
    constexpr int F = T / 32;                                        // 16-row fragments per wave and side
    constexpr bool SYM = EPI == EPI_GRAM || EPI == EPI_POLY;
    int it = 0;
    while (it + 1 < t.n && (int)blockIdx.x >= t.tile0[it + 1]) ++it;
    const NsDims& d = t.d[it];
    const int tm = d.mp / T, tn = d.np / T;
    const int per = SYM ? tm * (tm + 1) / 2 : tm * tn;
    int mat = (blockIdx.x - t.tile0[it]) / per, tile = (blockIdx.x - t.tile0[it]) - mat * per;
    const bool tall = d.rows > d.cols;
    int ti, tj;
    if constexpr (SYM) {                                             // lower triangle, row by row: tile = ti (ti + 1) / 2 + tj
        ti = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
        while (ti * (ti + 1) / 2 > tile) --ti;
        while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
        tj = tile - ti * (ti + 1) / 2;
    } else if (EPI == EPI_MULT || !tall) {
        ti = tile / tn; tj = tile - ti * tn;
    } else {
        ti = tile / tm; tj = tile - ti * tm;
    }
    half_t* base = ws + d.ws + mat * d.wsz;
    const long mn = (long)d.mp * d.np, mm = (long)d.mp * d.mp;
    // operands (row pitch = K, both k-contiguous), planes lo behind hi
    const half_t *Lp, *Rp;
    long lpl, rpl;
    int K;
    if constexpr (EPI == EPI_GRAM) { Lp = Rp = base; lpl = rpl = mn; K = d.np; }
    else if constexpr (EPI == EPI_POLY) { Lp = Rp = base + off_a(d); lpl = rpl = mm; K = d.mp; }
    else {
        K = d.mp;
        const half_t* b = base + off_b(d);
        const half_t* xt = base + off_xt(d, which);
        if (EPI == EPI_MULT || !tall) { Lp = b; lpl = mm; Rp = xt; rpl = mn; }
        else { Lp = xt; lpl = mn; Rp = b; rpl = mm; }
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // DMA sources: piece q of the stage = 16 rows of one plane; lane -> row lane >> 2, physical 16-byte slot lane & 3
    const bf16_t* src[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int q = wave * PIECES + i, plane = q / (T / 16), r = (q % (T / 16)) * 16 + (lane >> 2);
        const int chunk = (lane & 3) ^ dma_swz32(r);
        const half_t* pl = plane < 2 ? Lp + plane * lpl + ((long)ti * T + r) * K : Rp + (plane - 2) * rpl + ((long)tj * T + r) * K;
        src[i] = reinterpret_cast<const bf16_t*>(pl + chunk * 8);
    }
    const unsigned lds0 = (unsigned)(uintptr_t)smem;
    const int KT = K / 32;
    auto issue = [&](int kt) {
        const unsigned dst = lds0 + (kt % RING) * STAGE + wave * PIECES * 1024;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) glds16(src[i] + kt * 32, __builtin_amdgcn_readfirstlane(dst + i * 1024));
    };
    f32x4 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < RING - 1 && k < KT; ++k) issue(k);
    const int wr = (wave >> 1) * (T / 2), wc = (wave & 1) * (T / 2);
    const int fr = lane & 15, fk = lane >> 4;
    for (int kt = 0; kt < KT; ++kt) {
        // stage kt has landed when at most the later stages' pieces are outstanding; the barrier also tells that every wave has read
        // stage kt - 1, whose slot is refilled next
        if (kt + RING - 2 < KT) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RING - 2) * PIECES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (kt + RING - 1 < KT) issue(kt + RING - 1);
        const unsigned char* st = smem + (kt % RING) * STAGE;
        half8 lh[F], ll[F], rh[F], rl[F];
#pragma unroll
        for (int i = 0; i < F; ++i) {
            const int r = wr + i * 16 + fr, o = r * 64 + ((fk ^ dma_swz32(r)) << 4);
            lh[i] = *reinterpret_cast<const half8*>(st + o);
            ll[i] = *reinterpret_cast<const half8*>(st + PLANE + o);
            const int c = wc + i * 16 + fr, oc = c * 64 + ((fk ^ dma_swz32(c)) << 4);
            rh[i] = *reinterpret_cast<const half8*>(st + 2 * PLANE + oc);
            rl[i] = *reinterpret_cast<const half8*>(st + 3 * PLANE + oc);
        }
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rh[j], ll[i], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rl[j], lh[i], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rh[j], lh[i], acc[i][j], 0, 0, 0);
            }
    }
    // acc[i][j][e] = C[row + 16 i][col + 16 j + e]
    const int row = ti * T + wr + fr, col = tj * T + wc + fk * 4;
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
            const int r = row + i * 16, c = col + j * 16;
            f32x4 v = acc[i][j];
            if constexpr (SYM || EPI == EPI_MULT) {
                half_t *O, *OT;
                long ld, ldt, pl, plt;
                if constexpr (EPI == EPI_GRAM) {                     // f0 = sA / sX^2
                    v *= f0;
                    O = OT = base + off_a(d); ld = ldt = d.mp; pl = plt = mm;
                } else if constexpr (EPI == EPI_POLY) {              // v = (a I + b A + c A^2) sB: f0 = c sB / sA^2, f1 = b sB / sA, f2 = a sB
                    const half_t* A = base + off_a(d) + (long)r * d.mp + c;
                    const half4 ah = *reinterpret_cast<const half4*>(A), al = *reinterpret_cast<const half4*>(A + mm);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = fmaf(v[e], f0, f1 * ((float)ah[e] + (float)al[e])) + (r == c + e ? f2 : 0.f);
                    O = OT = base + off_b(d); ld = ldt = d.mp; pl = plt = mm;
                } else {                                             // f0 = sX' / (sB sX)
                    v *= f0;
                    O = base; ld = d.np; pl = mn;
                    OT = base + off_xt(d, which ^ 1); ldt = d.mp; plt = mn;
                }
                half4 h, l;
#pragma unroll
                for (int e = 0; e < 4; ++e) { half_t a, b; split_half(v[e], a, b); h[e] = a; l[e] = b; }
                *reinterpret_cast<half4*>(O + (long)r * ld + c) = h;
                *reinterpret_cast<half4*>(O + pl + (long)r * ld + c) = l;
                if (!SYM || ti != tj) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        OT[(long)(c + e) * ldt + r] = h[e];
                        OT[plt + (long)(c + e) * ldt + r] = l[e];
                    }
                }
            } else {
                if (r >= d.rows) continue;
                float lr = 0.f, keep = 1.f;
                if constexpr (EPI == EPI_UPDATE) { lr = hyper[0]; keep = 1.f - lr * hyper[2]; lr *= p.scale[it]; }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (c + e >= d.cols) continue;
                    const float o = v[e] * f0;                       // f0 = 1 / (sB sX)
                    const long oi = mat * p.os[it] + (long)r * p.old[it] + c + e;
                    if constexpr (EPI == EPI_OUT_F32) ((float*)p.o[it])[oi] = o;
                    if constexpr (EPI == EPI_OUT_BF16) ((bf16_t*)p.o[it])[oi] = f2bf(o);
                    if constexpr (EPI == EPI_UPDATE) {
                        float* pp = (float*)p.o[it] + oi;
                        const float np = fmaf(-lr, o, *pp * keep);
                        *pp = np;
                        if (p.hi[it]) {
                            bf16_t h, l;
                            split_bf16(np, h, l);
                            p.hi[it][oi] = h;
                            p.lo[it][oi] = l;
                        }
                        if (zero_grad) ((float*)p.x[it])[mat * p.xs[it] + (long)r * p.xld[it] + c + e] = 0.f;
                    }
                }
            }
        }
}

// ------------------------------------------------------------------------------------------------ host side
struct NsPlan {
    NsTable t;
    int T;                            // tile
    long mats;
    size_t bytes;
};
inline int up(int x, int to) { return (x + to - 1) / to * to; }

// the stacks [0, n) of one round: orientation, padding, workspace layout (partial sums first, then the planes)
bool ns_plan(NsPlan& pl, int n, const int* count, const int* rows, const int* cols) {
    memset(&pl, 0, sizeof(pl));
    pl.t.n = n;
    pl.T = 64;
    long off = 0;
    for (int i = 0; i < n; ++i) {
        NsDims& d = pl.t.d[i];
        d.count = count[i]; d.rows = rows[i]; d.cols = cols[i];
        d.m = rows[i] < cols[i] ? rows[i] : cols[i];
        d.n = rows[i] < cols[i] ? cols[i] : rows[i];
        d.mp = up(d.m, pl.T); d.np = up(d.n, pl.T);
        d.mat0 = (int)pl.mats;
        pl.mats += d.count;
        d.wsz = 6L * d.mp * d.np + 4L * d.mp * d.mp;
        d.ws = off;
        off += d.wsz * d.count;
    }
    pl.bytes = (size_t)pl.mats * NS_CHUNKS * sizeof(double) + (size_t)off * sizeof(half_t);
    return true;
}
long ns_tiles(NsTable& t, int T, bool sym) {
    long at = 0;
    for (int i = 0; i < t.n; ++i) {
        t.tile0[i] = (int)at;
        const long tm = t.d[i].mp / T, tn = t.d[i].np / T;
        at += (sym ? tm * (tm + 1) / 2 : tm * tn) * t.d[i].count;
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

template <int EPI, int T, int RING>
int launch_gemm(const NsTable& t, const NsPtrs& p, half_t* ws, const float* hyper, int which, float f0, float f1, float f2, int zero_grad, long tiles,
                hipStream_t s) {
    constexpr int bytes = RING * 4 * T * 64;
    auto k = ns_gemm_kernel<T, RING, EPI>;
    if (bytes > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(256), bytes, s, t, p, ws, hyper, which, f0, f1, f2, 0.f, zero_grad);
    S3D_CHECK_LAUNCH_V("newton_schulz", T * 10 + EPI);
    return 0;
}

template <int SRC, int LAST>
int ns_run(NsPlan& pl, const NsPtrs& p, const S3dNsArgs& a, const float* hyper, void* workspace, hipStream_t s) {
    double* part = reinterpret_cast<double*>(workspace);
    half_t* ws = reinterpret_cast<half_t*>(part + pl.mats * NS_CHUNKS);
    NsTable& t = pl.t;
    long at = 0;
    for (int i = 0; i < t.n; ++i) { t.tile0[i] = (int)at; at += (long)t.d[i].count * NS_CHUNKS; }
    t.tile0[t.n] = (int)at;
    S3D_REQUIRE(at <= 0x7fffffffL, "newton_schulz: too many matrices");
    hipLaunchKernelGGL(ns_sumsq_kernel<SRC>, dim3((unsigned)at), dim3(256), 0, s, t, p, hyper, a.nesterov, part);
    S3D_CHECK_LAUNCH_V("newton_schulz_sumsq", SRC);
    double bound = 1.001;
    float sx = pow2_under(32768., bound);
    at = ns_tiles(t, 64, false);
    S3D_REQUIRE(at >= 0, "newton_schulz: too many tiles");
    hipLaunchKernelGGL(ns_load_kernel<SRC>, dim3((unsigned)at), dim3(256), 0, s, t, p, hyper, a.nesterov, part, a.eps, sx, ws);
    S3D_CHECK_LAUNCH_V("newton_schulz_load", SRC);
    for (int k = 0; k < a.steps; ++k) {
        double pmax;
        const double next = ns_bounds(bound, a.a, a.b, a.c, pmax);
        const float sa = pow2_under(32768., bound * bound), sb = pow2_under(32768., pmax), sn = pow2_under(32768., next);
        at = ns_tiles(t, 64, true);
        if (int rc = launch_gemm<EPI_GRAM, 64, 4>(t, p, ws, hyper, k & 1, sa / (sx * sx), 0.f, 0.f, 0, at, s)) return rc;
        if (int rc = launch_gemm<EPI_POLY, 64, 4>(t, p, ws, hyper, k & 1, a.c * sb / (sa * sa), a.b * sb / sa, a.a * sb, 0, at, s)) return rc;
        at = ns_tiles(t, 64, false);
        if (k + 1 < a.steps) {
            if (int rc = launch_gemm<EPI_MULT, 64, 4>(t, p, ws, hyper, k & 1, sn / (sb * sx), 0.f, 0.f, 0, at, s)) return rc;
        } else {
            if (int rc = launch_gemm<LAST, 64, 4>(t, p, ws, hyper, k & 1, 1.f / (sb * sx), 0.f, 0.f, a.zero_grad, at, s)) return rc;
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
