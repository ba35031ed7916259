// Norms of queries and keys for each head with the position rotation in the same pass (s3d_qk_norm_rope_fwd / _bwd): the step between the
// qkv product and the attention kernels, on the packed [rows][(H | Hkv | Hkv) hd] tensor both of them use.
//
// Forward, per token and q / k head: r = 1 / sqrt(mean(x^2) + eps), z = x r g, y = R z with R the rotation of the pairs (i, i + hd/2) --
// or (2i, 2i + 1) -- by the token's angles.  Backward: dz = R^T dy, dg += dz x r, d = dz g, dx = r (d - x r mean(d x r)).
// Nothing but x is kept for the backward: r is one reduction over values it reads anyway.
//
// Bound: HBM (188160 tokens of 9 heads of 256: forward 1.73 GB in 357 us = 4.85 TB/s, backward 2.6 GB in 480 us = 5.4 TB/s with the gains' reduction, a
// large copy runs at 4.73), launch and host for few tokens (26: 4 us of kernel).  One pass, every element read and written once in 16-byte pieces; the angles come from a table of [positions][hd/2] cosines and
// sines that stays in the caches.  A head is worked by G = 1 .. 16 lanes (hd / 16 rounded up to a power of two): each holds 8 elements of
// either half, i.e. 8 whole pairs, so the rotation needs no exchange and the mean is log2(G) lane exchanges.  A workgroup works the query, the
// key or the value heads of a range of rows (blockIdx.y): one gain and one gain gradient in registers, no divergence, and three times the
// workgroups when there are few rows.
#include "kernels.h"
#include "ranges.h"

namespace {

struct QkPlan {
    int rows_per_wg;
    unsigned h_inv[2], st_inv, T_inv;  // 2^32 / heads (queries, keys), / st, / T
};

// a / b with inv = 2^32 / b (b >= 2; 0xffffffff for 1): the product's high word is at most two short
__device__ __forceinline__ unsigned div_by(unsigned a, unsigned b, unsigned inv) {
    unsigned q = __umulhi(a, inv);
    if (a - q * b >= b) ++q;
    if (a - q * b >= b) ++q;
    return q;
}

// sum over aligned groups of G lanes (within a row of 16): exchanges between halves that already agree
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#define S3D_QK_STEP(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
    if constexpr (G >= 2) S3D_QK_STEP(0xB1);        // quad_perm:[1,0,3,2]
    if constexpr (G >= 4) S3D_QK_STEP(0x4E);        // quad_perm:[2,3,0,1]
    if constexpr (G >= 8) S3D_QK_STEP(0x141);       // row_half_mirror
    if constexpr (G >= 16) S3D_QK_STEP(0x140);      // row_mirror
#undef S3D_QK_STEP
    return v;
}
struct Piece { u32x4 hi, lo; };
__device__ __forceinline__ Piece load8(const bf16_t* hi, const bf16_t* lo, long at) {
    Piece p;
    p.hi = *reinterpret_cast<const u32x4*>(hi + at);
    p.lo = lo ? *reinterpret_cast<const u32x4*>(lo + at) : u32x4{0, 0, 0, 0};
    return p;
}
__device__ __forceinline__ void unpack8(const Piece& p, bool pair, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(p.hi[i] << 16);
        x[2 * i + 1] = __uint_as_float(p.hi[i] & 0xffff0000u);
    }
    if (pair) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] += __uint_as_float(p.lo[i] << 16);
            x[2 * i + 1] += __uint_as_float(p.lo[i] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ void store8(bf16_t* hi, bf16_t* lo, long at, const float* x) {
    U128 a, b;
    if (lo) {
#pragma unroll
        for (int i = 0; i < 4; ++i) split_bf16x2(x[2 * i], x[2 * i + 1], a.w[i], b.w[i]);
        *reinterpret_cast<u32x4*>(lo + at) = b.u;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) a.w[i] = f2bf2(x[2 * i], x[2 * i + 1]);
    }
    *reinterpret_cast<u32x4*>(hi + at) = a.u;
}

// the value heads: planes copied bit for bit, or converted where one side has a low plane and the other has not
__device__ __forceinline__ void copy_values(const bf16_t* sh, const bf16_t* sl, long lds, bf16_t* oh, bf16_t* ol, long ldo, int nrow, long row0, int first, int width) {
    const unsigned per = width / 8, units = nrow * per;
    for (unsigned u = threadIdx.x; u < units; u += 256) {
        const unsigned r = u / per, c = (u - r * per) * 8;
        const long s = (row0 + r) * lds + first + c, o = (row0 + r) * ldo + first + c;
        const Piece p = load8(sh, sl, s);
        if ((sl == nullptr) == (ol == nullptr)) {
            *reinterpret_cast<u32x4*>(oh + o) = p.hi;
            if (ol) *reinterpret_cast<u32x4*>(ol + o) = p.lo;
        } else {
            float x[8];
            unpack8(p, sl != nullptr, x);
            store8(oh, ol, o, x);
        }
    }
}

// x[16]: the lane's two pieces; pair p = (x[p], x[p + 8]) with split halves, (x[2p], x[2p + 1]) interleaved
template <bool INTER> __device__ __forceinline__ constexpr int pa(int p) { return INTER ? 2 * p : p; }
template <bool INTER> __device__ __forceinline__ constexpr int pb(int p) { return INTER ? 2 * p + 1 : p + 8; }

template <int G, bool INTER, bool BWD>
__global__ __launch_bounds__(256) void qk_norm_kernel(const S3dQkNormArgs a, const QkPlan q) {
    constexpr int GROUPS = 256 / G;
    const int role = blockIdx.y;                             // 0: queries, 1: keys, 2: values
    const long row0 = (long)blockIdx.x * q.rows_per_wg;
    const int nrow = (int)(row0 + q.rows_per_wg < a.rows ? q.rows_per_wg : a.rows - row0);
    const bf16_t *sh = BWD ? a.dout : a.qkv_hi, *sl = BWD ? a.dout_lo : a.qkv_lo;
    bf16_t *oh = BWD ? a.dqkv : a.out_hi, *ol = BWD ? a.dqkv_lo : a.out_lo;
    const long lds = BWD ? a.lddo : a.ld, ldo = BWD ? a.lddq : a.ldo;
    const int hd = a.hd, half = hd >> 1;
    if (role == 2) {
        copy_values(sh, sl, lds, oh, ol, ldo, nrow, row0, (a.H + a.Hkv) * hd, a.Hkv * hd);
        return;
    }
    const int heads = role ? a.Hkv : a.H, first = role ? a.H * hd : 0;
    const float* gain = role ? a.k_gain : a.q_gain;
    const int c = threadIdx.x % G, grp = threadIdx.x / G;
    const bool on = c * 16 < hd;
    const int o0 = on ? (INTER ? 16 * c : 8 * c) : 0, o1 = on ? (INTER ? 16 * c + 8 : half + 8 * c) : 0;      // the two 8-element pieces within a head
    float g[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        g[i] = gain ? gain[o0 + i] : 1.f;
        g[8 + i] = gain ? gain[o1 + i] : 1.f;
    }
    float acc[16];                                           // backward: this lane's part of the gain's gradient
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    const float inv_hd = 1.f / (float)hd;
    const unsigned units = (unsigned)nrow * heads;
    for (unsigned u = grp; u < units; u += GROUPS) {         // (the lanes of a group stay together)
        const unsigned row_l = div_by(u, heads, q.h_inv[role]);
        const long row = row0 + row_l;
        const int at_h = first + (int)(u - row_l * heads) * hd;
        const long at = row * a.ld + at_h;
        Piece x0, x1, y0, y1;
        x0 = load8(a.qkv_hi, a.qkv_lo, at + o0);
        x1 = load8(a.qkv_hi, a.qkv_lo, at + o1);
        if constexpr (BWD) {
            y0 = load8(sh, sl, row * lds + at_h + o0);
            y1 = load8(sh, sl, row * lds + at_h + o1);
        }
        f32x4 cs[2], sn[2];
        cs[0] = cs[1] = f32x4{1.f, 1.f, 1.f, 1.f};
        sn[0] = sn[1] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (a.cos_t) {
            int t;
            if (a.pos) t = a.pos[row];
            else {
                const unsigned s = div_by((unsigned)row, a.st, q.st_inv);
                t = (int)(s - div_by(s, a.T, q.T_inv) * a.T);
            }
            if (t >= 0 && t < a.T) {
                const long k = (long)t * half + (on ? 8 * c : 0);
                cs[0] = *reinterpret_cast<const f32x4*>(a.cos_t + k);
                cs[1] = *reinterpret_cast<const f32x4*>(a.cos_t + k + 4);
                sn[0] = *reinterpret_cast<const f32x4*>(a.sin_t + k);
                sn[1] = *reinterpret_cast<const f32x4*>(a.sin_t + k + 4);
            }
        }
        float x[16], y[16];
        unpack8(x0, a.qkv_lo != nullptr, x);
        unpack8(x1, a.qkv_lo != nullptr, x + 8);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
        const float r = rsqrtf(group_sum<G>(on ? ss : 0.f) * inv_hd + a.eps);
        if constexpr (!BWD) {
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                const int i = pa<INTER>(p), j = pb<INTER>(p);
                const float z0 = x[i] * r * g[i], z1 = x[j] * r * g[j], cp = cs[p >> 2][p & 3], sp = sn[p >> 2][p & 3];
                y[i] = z0 * cp - z1 * sp;
                y[j] = z1 * cp + z0 * sp;
            }
        } else {
            unpack8(y0, sl != nullptr, y);
            unpack8(y1, sl != nullptr, y + 8);
            float dot = 0.f;
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                const int i = pa<INTER>(p), j = pb<INTER>(p);
                const float cp = cs[p >> 2][p & 3], sp = sn[p >> 2][p & 3];
                const float d0 = y[i] * cp + y[j] * sp, d1 = y[j] * cp - y[i] * sp;
                x[i] *= r;
                x[j] *= r;
                acc[i] = fmaf(d0, x[i], acc[i]);
                acc[j] = fmaf(d1, x[j], acc[j]);
                y[i] = d0 * g[i];
                y[j] = d1 * g[j];
                dot = fmaf(y[i], x[i], dot);
                dot = fmaf(y[j], x[j], dot);
            }
            dot = group_sum<G>(on ? dot : 0.f) * inv_hd;
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = r * (y[i] - x[i] * dot);
        }
        if (on) {
            store8(oh, ol, row * ldo + at_h + o0, y);
            store8(oh, ol, row * ldo + at_h + o1, y + 8);
        }
    }
    if constexpr (BWD) {
        // this workgroup's sums over its rows and heads, added in the order of the groups: partial[q | k][wg][hd]
        __shared__ float red[256 * 17];
#pragma unroll
        for (int i = 0; i < 16; ++i) red[threadIdx.x * 17 + i] = acc[i];
        __syncthreads();
        for (int e = threadIdx.x; e < hd; e += 256) {
            const int cc = INTER ? e >> 4 : (e < half ? e : e - half) >> 3, i = INTER ? e & 15 : ((e < half ? e : e - half) & 7) + (e < half ? 0 : 8);
            float s = 0.f;
            for (int k = 0; k < GROUPS; ++k) s += red[(k * G + cc) * 17 + i];
            a.partial[((long)role * gridDim.x + blockIdx.x) * hd + e] = s;
        }
    }
}

// gradients of the gains: the workgroups' rows [q | k][blocks][hd] added in a fixed order (64 bits), one workgroup per 16 columns
__global__ __launch_bounds__(1024) void qk_gain_reduce_kernel(const float* __restrict__ partial, int blocks, int hd, float* dq, float* dk, int accumulate) {
    const int which = blockIdx.y, col = blockIdx.x * 16 + (threadIdx.x & 15);          // hd is a multiple of 16
    const float* p = partial + (long)which * blocks * hd + col;
    __shared__ double red[1024];
    double s = 0.;
    for (int b0 = threadIdx.x >> 4; b0 < blocks; b0 += 512) {                          // eight rows in flight: a chain of single loads took 60 us for 2048 rows
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int b = b0 + 64 * k;
            v[k] = b < blocks ? p[(long)b * hd] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) s += (double)v[k];
    }
    red[threadIdx.x] = s;
    __syncthreads();
    for (int k = 32; k > 0; k >>= 1) {
        if ((threadIdx.x >> 4) < k) red[threadIdx.x] += red[threadIdx.x + 16 * k];
        __syncthreads();
    }
    if (threadIdx.x < 16) {
        float* o = (which ? dk : dq) + col;
        *o = (accumulate ? *o : 0.f) + (float)red[threadIdx.x];
    }
}

int lanes_of(int hd) {
    int g = 1;
    while (g * 16 < hd) g <<= 1;
    return g;
}
// Rows of one workgroup: one pass of its groups over the heads while there are few rows, about 2048 row ranges (x 3 roles) when there are many.
// Backward: a workgroup ends by adding its groups' gain gradients through LDS, and every row range is a row of the reduction behind it, so up to four
// passes as long as 900 workgroups are left.  One / two / four passes, us with the reduction: 1203 ranges of 80-wide heads 23.4 / 17.7 / 16.7,
// 747 ranges of 64-wide heads 19.6 / 16.6 / 17.3.
int rows_per_wg(long rows, int H, int hd, bool bwd) {
    const int groups = 256 / lanes_of(hd);
    long r = (groups + H - 1) / H;
    const long cap = (rows + 2047) / 2048;
    if (bwd) {
        const long passes = (rows + r - 1) / r / 300;
        r *= passes < 1 ? 1 : passes > 4 ? 4 : passes;
    }
    return (int)(r < cap ? cap : r);
}
unsigned inv_of(int b) { return b > 1 ? (unsigned)((1ULL << 32) / (unsigned)b) : 0xffffffffu; }

template <bool BWD>
int launch(const S3dQkNormArgs& a, hipStream_t s) {
    QkPlan q;
    q.rows_per_wg = rows_per_wg(a.rows, a.H, a.hd, BWD);
    q.h_inv[0] = inv_of(a.H);
    q.h_inv[1] = inv_of(a.Hkv);
    q.st_inv = inv_of(a.st);
    q.T_inv = inv_of(a.T);
    const unsigned wgs = (unsigned)((a.rows + q.rows_per_wg - 1) / q.rows_per_wg);
    const int G = lanes_of(a.hd);
    const bool in_place = BWD ? a.dqkv == a.dout : a.out_hi == a.qkv_hi;      // the value heads are where they belong
    const dim3 grid(wgs, in_place ? 2 : 3);
#define S3D_QK_CASE(g)                                                                                                  \
    if (G == g) {                                                                                                       \
        if (a.interleaved) hipLaunchKernelGGL((qk_norm_kernel<g, true, BWD>), grid, dim3(256), 0, s, a, q);             \
        else hipLaunchKernelGGL((qk_norm_kernel<g, false, BWD>), grid, dim3(256), 0, s, a, q);                          \
    }
    S3D_QK_CASE(1) S3D_QK_CASE(2) S3D_QK_CASE(4) S3D_QK_CASE(8) S3D_QK_CASE(16)
#undef S3D_QK_CASE
    S3D_CHECK_LAUNCH_V("qk_norm", G * 4 + (BWD ? 2 : 0) + (a.interleaved ? 1 : 0));
    if (BWD) {
        hipLaunchKernelGGL(qk_gain_reduce_kernel, dim3(a.hd / 16, 2), dim3(1024), 0, s, a.partial, (int)wgs, a.hd, a.dq_gain, a.dk_gain, a.accumulate);
        S3D_CHECK_LAUNCH("qk_gain_reduce");
    }
    return 0;
}

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check(const S3dQkNormArgs& a, bool bwd) {
    const char* who = bwd ? "s3d_qk_norm_rope_bwd" : "s3d_qk_norm_rope_fwd";
    S3D_REQUIRE(a.rows >= 0 && a.rows < (1L << 31), "%s: %ld rows", who, a.rows);
    S3D_REQUIRE(a.H >= 1 && a.Hkv >= 1 && a.H <= 1024 && a.Hkv <= 1024, "%s: %d query and %d key heads (1 .. 1024)", who, a.H, a.Hkv);
    S3D_REQUIRE(a.hd >= 16 && a.hd <= 256 && a.hd % 16 == 0, "%s: head dim %d (a multiple of 16 up to 256)", who, a.hd);
    const long W = (long)(a.H + 2 * a.Hkv) * a.hd;
    S3D_REQUIRE(a.qkv_hi && aligned(a.qkv_hi) && aligned(a.qkv_lo), "%s: qkv must be set and 16-byte aligned", who);
    S3D_REQUIRE(a.ld >= W && a.ld % 8 == 0, "%s: qkv row pitch %ld (at least %ld, a multiple of 8)", who, a.ld, W);
    S3D_REQUIRE(a.eps >= 0.f && a.eps < 1e30f, "%s: eps %g", who, (double)a.eps);
    S3D_REQUIRE((a.cos_t == nullptr) == (a.sin_t == nullptr), "%s: both tables or none", who);
    S3D_REQUIRE(!a.cos_t || (a.T >= 1 && aligned(a.cos_t) && aligned(a.sin_t)), "%s: the tables need rows and 16-byte alignment", who);
    S3D_REQUIRE(!a.cos_t || a.pos || a.st >= 1, "%s: token stride %d", who, a.st);
    if (!bwd) {
        S3D_REQUIRE(a.out_hi != a.qkv_hi || (a.ldo == a.ld && a.out_lo == a.qkv_lo), "%s: in place needs the same planes and pitch", who);
        S3D_REQUIRE(a.out_hi && aligned(a.out_hi) && aligned(a.out_lo), "%s: out must be set and 16-byte aligned", who);
        S3D_REQUIRE(a.ldo >= W && a.ldo % 8 == 0, "%s: out row pitch %ld (at least %ld, a multiple of 8)", who, a.ldo, W);
    } else {
        S3D_REQUIRE(a.dqkv != a.dout || (a.lddq == a.lddo && a.dqkv_lo == a.dout_lo), "%s: in place needs the same planes and pitch", who);
        S3D_REQUIRE(a.dout && aligned(a.dout) && aligned(a.dout_lo) && a.dqkv && aligned(a.dqkv) && aligned(a.dqkv_lo), "%s: dout and dqkv must be set and 16-byte aligned", who);
        S3D_REQUIRE(a.lddo >= W && a.lddo % 8 == 0 && a.lddq >= W && a.lddq % 8 == 0, "%s: gradient row pitch (at least %ld, a multiple of 8)", who, W);
        S3D_REQUIRE(a.dq_gain && a.dk_gain, "%s: dq_gain and dk_gain must be set", who);
        const int need = s3d_qk_norm_blocks(a.rows, a.H, a.Hkv, a.hd);
        S3D_REQUIRE(a.partial && a.partial_blocks >= need, "%s: partial needs %d blocks", who, need);
        S3D_REQUIRE(a.dq_gain + a.hd <= a.dk_gain || a.dk_gain + a.hd <= a.dq_gain, "%s: dq_gain and dk_gain overlap (one gain for both: add the two)", who);
    }
    if (a.rows > 0) {
        // what is written may be what is read in place (same plane and pitch: every element is read and written by one lane), never a shifted part of it
        const bf16_t *out[2] = {bwd ? a.dqkv : a.out_hi, bwd ? a.dqkv_lo : a.out_lo}, *in[4] = {a.qkv_hi, a.qkv_lo, bwd ? a.dout : nullptr, bwd ? a.dout_lo : nullptr};
        const long ldo = bwd ? a.lddq : a.ldo, ldi[4] = {a.ld, a.ld, a.lddo, a.lddo};
        auto range = [&](const bf16_t* p, long ld) { return MatRange{(uintptr_t)p, 2, 0, ld, 1, a.rows, (int)W, true, 0}; };
        for (int i = 0; i < 2; ++i)
            for (int k = 0; k < 4 && out[i]; ++k)
                S3D_REQUIRE(!in[k] || (in[k] == out[i] && ldi[k] == ldo && (k & 1) == i) || !ranges_meet(range(out[i], ldo), range(in[k], ldi[k])),
                            "%s: an output plane overlaps an input plane", who);
        S3D_REQUIRE(!out[1] || !ranges_meet(range(out[0], ldo), range(out[1], ldo)), "%s: the output planes overlap", who);
        // nor may what is written share memory with the gains, tables and positions, nor the gains' gradients and their partial sums with anything
        auto flat = [](const void* p, size_t n) { return FlatRange{(uintptr_t)p, p ? n * 4 : 0}; };
        const FlatRange read[5] = {flat(a.q_gain, a.hd), flat(a.k_gain, a.hd), flat(a.cos_t, a.cos_t ? (size_t)a.T * (a.hd / 2) : 0),
                                   flat(a.sin_t, a.cos_t ? (size_t)a.T * (a.hd / 2) : 0), flat(a.cos_t ? a.pos : nullptr, a.rows)};
        const size_t sums = bwd ? (size_t)s3d_qk_norm_blocks(a.rows, a.H, a.Hkv, a.hd) * 2 * a.hd : 0;
        const FlatRange written[3] = {flat(bwd ? a.dq_gain : nullptr, a.hd), flat(bwd ? a.dk_gain : nullptr, a.hd), flat(bwd ? a.partial : nullptr, sums)};
        for (const FlatRange& f : read) {
            if (!f.bytes) continue;
            for (int i = 0; i < 2; ++i) S3D_REQUIRE(!out[i] || !ranges_meet(range(out[i], ldo), f), "%s: an output plane overlaps a gain, a table or the positions", who);
            for (const FlatRange& w : written) S3D_REQUIRE(!ranges_meet(w, f), "%s: a gain's gradient or partial overlaps a gain, a table or the positions", who);
        }
        for (const FlatRange& w : written) {
            if (!w.bytes) continue;
            for (int i = 0; i < 2; ++i) S3D_REQUIRE(!out[i] || !ranges_meet(range(out[i], ldo), w), "%s: a gain's gradient or partial overlaps an output plane", who);
            for (int k = 0; k < 4; ++k) S3D_REQUIRE(!in[k] || !ranges_meet(range(in[k], ldi[k]), w), "%s: a gain's gradient or partial overlaps an input plane", who);
        }
        S3D_REQUIRE(!ranges_meet(written[0], written[2]) && !ranges_meet(written[1], written[2]), "%s: partial overlaps a gain's gradient", who);
    }
    return 0;
}

}  // namespace

int s3d_qk_norm_blocks(long rows, int H, int Hkv, int hd) {
    if (rows <= 0 || H < 1 || Hkv < 1 || hd < 16 || hd > 256) return 0;
    const int r = rows_per_wg(rows, H, hd, true);
    return (int)((rows + r - 1) / r);
}
int s3d_launch_qk_norm_fwd(const S3dQkNormArgs& a, hipStream_t s) {
    if (int rc = check(a, false)) return rc;
    return a.rows == 0 ? 0 : launch<false>(a, s);
}
int s3d_launch_qk_norm_bwd(const S3dQkNormArgs& a, hipStream_t s) {
    if (int rc = check(a, true)) return rc;
    if (a.rows == 0) {                                       // no rows: nothing to add, the gradients of an overwriting call are zero
        if (!a.accumulate) {
            hipLaunchKernelGGL(qk_gain_reduce_kernel, dim3(a.hd / 16, 2), dim3(1024), 0, s, a.partial, 0, a.hd, a.dq_gain, a.dk_gain, 0);
            S3D_CHECK_LAUNCH("qk_gain_reduce");
        }
        return 0;
    }
    return launch<true>(a, s);
}
