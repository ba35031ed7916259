// Norms of queries and keys for each head with the position rotation in the same pass (s3d_qk_norm_rope_fwd / _bwd): the step between the
// qkv product and the attention kernels, on the packed [rows][(H | Hkv | Hkv) hd] tensor both of them use.
//
// Forward, per token and q / k head: r = 1 / sqrt(mean(x^2) + eps), z = x r g, y = R z with R the rotation of the pairs (i, i + hd/2) --
// or (2i, 2i + 1) -- by the token's angles.  Backward: dz = R^T dy, dg += dz x r, d = dz g, dx = r (d - x r mean(d x r)).
// Nothing but x is kept for the backward: r is one reduction over values it reads anyway.
//
// Bound: HBM.  One pass, every element read and written once in 16-byte pieces; the angles come from a table of [positions][hd/2] cosines and
// sines that stays in the caches.  A head is worked by G = 1 .. 16 lanes (hd / 16 rounded up to a power of two): each holds 8 elements of
// either half, i.e. 8 whole pairs, so the rotation needs no exchange and the mean is log2(G) lane exchanges.
#include "kernels.h"

namespace {

struct QkUnits {
    int rows_per_wg;                  // rows of one workgroup
    int HT;                           // H + 2 Hkv
};

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int k = 1; k < G; k <<= 1) v += __shfl_xor(v, k, 64);
    return v;
}
__device__ __forceinline__ void load8(const bf16_t* hi, const bf16_t* lo, long at, float* x) {
    U128 a;
    a.u = *reinterpret_cast<const u32x4*>(hi + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = bf2f(a.h[i]);
    if (lo) {
        a.u = *reinterpret_cast<const u32x4*>(lo + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += bf2f(a.h[i]);
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

// x[16]: the lane's two pieces; pair p = (x[p], x[p + 8]) with split halves, (x[2p], x[2p + 1]) interleaved
template <bool INTER> __device__ __forceinline__ int pa(int p) { return INTER ? 2 * p : p; }
template <bool INTER> __device__ __forceinline__ int pb(int p) { return INTER ? 2 * p + 1 : p + 8; }

template <int G, bool INTER, bool BWD>
__global__ __launch_bounds__(256) void qk_norm_kernel(const S3dQkNormArgs a, const QkUnits q) {
    constexpr int GROUPS = 256 / G;
    const int hd = a.hd, half = hd >> 1;
    const int c = threadIdx.x % G, grp = threadIdx.x / G;
    const bool on = c * 16 < hd;
    const int o0 = INTER ? 16 * c : 8 * c, o1 = INTER ? 16 * c + 8 : half + 8 * c;      // the two 8-element pieces within a head
    float gq[16], gk[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        gq[i] = on && a.q_gain ? a.q_gain[o0 + i] : 1.f;
        gq[8 + i] = on && a.q_gain ? a.q_gain[o1 + i] : 1.f;
        gk[i] = on && a.k_gain ? a.k_gain[o0 + i] : 1.f;
        gk[8 + i] = on && a.k_gain ? a.k_gain[o1 + i] : 1.f;
    }
    float aq[16], ak[16];                                    // backward: sums of the gains' gradients
#pragma unroll
    for (int i = 0; i < 16; ++i) aq[i] = ak[i] = 0.f;
    const float inv_hd = 1.f / (float)hd;
    const long row0 = (long)blockIdx.x * q.rows_per_wg;
    const int nrow = (int)(row0 + q.rows_per_wg < a.rows ? q.rows_per_wg : a.rows - row0);
    const int units = nrow * q.HT;
    const bool copy_v = BWD ? a.dout != a.dqkv || a.dout_lo != a.dqkv_lo : a.qkv_hi != a.out_hi || a.qkv_lo != a.out_lo;
    for (int u0 = 0; u0 < units; u0 += GROUPS) {
        const int u = u0 + grp;
        const bool live = u < units && on;
        const int row_l = u / q.HT, h = u - row_l * q.HT;
        const long row = row0 + row_l;
        const bool isq = h < a.H, isv = h >= a.H + a.Hkv;
        const long at = row * a.ld + (long)h * hd;
        float x[16], y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = y[i] = 0.f;
        const bf16_t *sh = BWD ? a.dout : a.qkv_hi, *sl = BWD ? a.dout_lo : a.qkv_lo;
        bf16_t *oh = BWD ? a.dqkv : a.out_hi, *ol = BWD ? a.dqkv_lo : a.out_lo;
        const long at_s = row * (BWD ? a.lddo : a.ld) + (long)h * hd, at_o = row * (BWD ? a.lddq : a.ldo) + (long)h * hd;
        if (live && isv && copy_v && (sl == nullptr) == (ol == nullptr)) {       // values: the planes bit for bit
            const u32x4 v0 = *reinterpret_cast<const u32x4*>(sh + at_s + o0), v1 = *reinterpret_cast<const u32x4*>(sh + at_s + o1);
            *reinterpret_cast<u32x4*>(oh + at_o + o0) = v0;
            *reinterpret_cast<u32x4*>(oh + at_o + o1) = v1;
            if (sl) {
                const u32x4 w0 = *reinterpret_cast<const u32x4*>(sl + at_s + o0), w1 = *reinterpret_cast<const u32x4*>(sl + at_s + o1);
                *reinterpret_cast<u32x4*>(ol + at_o + o0) = w0;
                *reinterpret_cast<u32x4*>(ol + at_o + o1) = w1;
            }
        }
        const bool raw_v = isv && (!copy_v || (sl == nullptr) == (ol == nullptr));   // nothing left to do for this head
        if (live && !raw_v) {
            if (!BWD || !isv) {
                load8(a.qkv_hi, a.qkv_lo, at + o0, x);
                load8(a.qkv_hi, a.qkv_lo, at + o1, x + 8);
            }
            if (BWD) {
                load8(sh, sl, at_s + o0, y);
                load8(sh, sl, at_s + o1, y + 8);
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
        const float r = rsqrtf(group_sum<G>(ss) * inv_hd + a.eps);
        float cs[8], sn[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) { cs[i] = 1.f; sn[i] = 0.f; }
        if (live && !isv && a.cos_t) {
            const int t = a.pos ? a.pos[row] : (int)((row / a.st) % a.T);
            if (t >= 0 && t < a.T) {
                const long k = (long)t * half + 8 * c;
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const f32x4 cv = *reinterpret_cast<const f32x4*>(a.cos_t + k + i), sv = *reinterpret_cast<const f32x4*>(a.sin_t + k + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { cs[i + e] = cv[e]; sn[i + e] = sv[e]; }
                }
            }
        }
        if constexpr (!BWD) {
            if (!isv) {
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    const int i = pa<INTER>(p), j = pb<INTER>(p);
                    const float z0 = x[i] * r * (isq ? gq[i] : gk[i]), z1 = x[j] * r * (isq ? gq[j] : gk[j]);
                    x[i] = z0 * cs[p] - z1 * sn[p];
                    x[j] = z1 * cs[p] + z0 * sn[p];
                }
            }
            if (live && !raw_v) {
                store8(oh, ol, at_o + o0, x);
                store8(oh, ol, at_o + o1, x + 8);
            }
        } else {
            float dot = 0.f;
            if (!isv) {
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    const int i = pa<INTER>(p), j = pb<INTER>(p);
                    const float d0 = y[i] * cs[p] + y[j] * sn[p], d1 = y[j] * cs[p] - y[i] * sn[p];
                    x[i] *= r;
                    x[j] *= r;
                    if (isq) { aq[i] = fmaf(d0, x[i], aq[i]); aq[j] = fmaf(d1, x[j], aq[j]); }
                    else { ak[i] = fmaf(d0, x[i], ak[i]); ak[j] = fmaf(d1, x[j], ak[j]); }
                    y[i] = d0 * (isq ? gq[i] : gk[i]);
                    y[j] = d1 * (isq ? gq[j] : gk[j]);
                    dot = fmaf(y[i], x[i], dot);
                    dot = fmaf(y[j], x[j], dot);
                }
            }
            dot = group_sum<G>(dot) * inv_hd;
            if (!isv) {
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = r * (y[i] - x[i] * dot);
            }
            if (live && !raw_v) {
                store8(oh, ol, at_o + o0, y);
                store8(oh, ol, at_o + o1, y + 8);
            }
        }
    }
    if constexpr (BWD) {
        // this workgroup's sums over its rows and heads, added in the order of the groups: partial[wg][q | k][hd]
        __shared__ float red[256 * 16];
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 16; ++i) red[(grp * G + c) * 16 + i] = which ? ak[i] : aq[i];
            __syncthreads();
            for (int e = threadIdx.x; e < hd; e += 256) {
                const int cc = INTER ? e >> 4 : (e % half) >> 3, i = INTER ? e & 15 : (e % half & 7) + (e >= half ? 8 : 0);
                float s = 0.f;
                for (int g = 0; g < GROUPS; ++g) s += red[(g * G + cc) * 16 + i];
                a.partial[((long)blockIdx.x * 2 + which) * hd + e] = s;
            }
        }
    }
}

// gradients of the gains: the workgroups' rows added in order (64 bits), one workgroup per 4 columns of [q | k][hd]
__global__ __launch_bounds__(256) void qk_gain_reduce_kernel(const float* __restrict__ partial, int blocks, int hd, float* dq, float* dk, int accumulate) {
    const int col = blockIdx.x * 4 + (threadIdx.x & 3);
    __shared__ double red[256];
    double s = 0.;
    if (col < 2 * hd)
        for (int b = threadIdx.x >> 2; b < blocks; b += 64) s += (double)partial[(long)b * 2 * hd + col];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int k = 32; k > 0; k >>= 1) {
        if ((threadIdx.x >> 2) < k) red[threadIdx.x] += red[threadIdx.x + 4 * k];
        __syncthreads();
    }
    if (threadIdx.x < 4 && col < 2 * hd) {
        float* o = col < hd ? dq + col : dk + col - hd;
        *o = (accumulate ? *o : 0.f) + (float)red[threadIdx.x];
    }
}

int lanes_of(int hd) {
    int g = 1;
    while (g * 16 < hd) g <<= 1;
    return g;
}
// rows of one workgroup: at least four passes of its groups, at most about 2048 workgroups (8 per CU)
int rows_per_wg(long rows, int HT, int hd) {
    const int groups = 256 / lanes_of(hd);
    long r = (4L * groups + HT - 1) / HT;
    const long cap = (rows + 2047) / 2048;
    if (r < cap) r = cap;
    return (int)r;
}

template <bool BWD>
int launch(const S3dQkNormArgs& a, hipStream_t s) {
    QkUnits q;
    q.HT = a.H + 2 * a.Hkv;
    q.rows_per_wg = rows_per_wg(a.rows, q.HT, a.hd);
    const unsigned wgs = (unsigned)((a.rows + q.rows_per_wg - 1) / q.rows_per_wg);
    const int G = lanes_of(a.hd);
#define S3D_QK_CASE(g)                                                                                                  \
    if (G == g) {                                                                                                       \
        if (a.interleaved) hipLaunchKernelGGL((qk_norm_kernel<g, true, BWD>), dim3(wgs), dim3(256), 0, s, a, q);        \
        else hipLaunchKernelGGL((qk_norm_kernel<g, false, BWD>), dim3(wgs), dim3(256), 0, s, a, q);                     \
    }
    S3D_QK_CASE(1) S3D_QK_CASE(2) S3D_QK_CASE(4) S3D_QK_CASE(8) S3D_QK_CASE(16)
#undef S3D_QK_CASE
    S3D_CHECK_LAUNCH_V("qk_norm", G * 4 + (BWD ? 2 : 0) + (a.interleaved ? 1 : 0));
    if (BWD) {
        hipLaunchKernelGGL(qk_gain_reduce_kernel, dim3((2 * a.hd + 3) / 4), dim3(256), 0, s, a.partial, (int)wgs, a.hd, a.dq_gain, a.dk_gain, a.accumulate);
        S3D_CHECK_LAUNCH("qk_gain_reduce");
    }
    return 0;
}

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check(const S3dQkNormArgs& a, bool bwd) {
    const char* who = bwd ? "s3d_qk_norm_rope_bwd" : "s3d_qk_norm_rope_fwd";
    S3D_REQUIRE(a.rows >= 0 && a.rows < (1L << 31), "%s: %ld rows", who, a.rows);
    S3D_REQUIRE(a.H >= 1 && a.Hkv >= 1 && a.H <= 4096 && a.Hkv <= 4096, "%s: %d query and %d key heads", who, a.H, a.Hkv);
    S3D_REQUIRE(a.hd >= 16 && a.hd <= 256 && a.hd % 16 == 0, "%s: head dim %d (a multiple of 16 up to 256)", who, a.hd);
    const long W = (long)(a.H + 2 * a.Hkv) * a.hd;
    S3D_REQUIRE(a.qkv_hi && aligned(a.qkv_hi) && aligned(a.qkv_lo), "%s: qkv must be set and 16-byte aligned", who);
    S3D_REQUIRE(a.ld >= W && a.ld % 8 == 0, "%s: qkv row pitch %ld (at least %ld, a multiple of 8)", who, a.ld, W);
    S3D_REQUIRE(a.eps >= 0.f && a.eps < 1e30f, "%s: eps %g", who, (double)a.eps);
    S3D_REQUIRE((a.cos_t == nullptr) == (a.sin_t == nullptr), "%s: both tables or none", who);
    S3D_REQUIRE(!a.cos_t || (a.T >= 1 && aligned(a.cos_t) && aligned(a.sin_t)), "%s: the tables need rows and 16-byte alignment", who);
    S3D_REQUIRE(!a.cos_t || a.pos || a.st >= 1, "%s: token stride %d", who, a.st);
    S3D_REQUIRE((long)rows_per_wg(a.rows, a.H + 2 * a.Hkv, a.hd) * (a.H + 2 * a.Hkv) < (1L << 30), "%s: %ld rows of %d heads", who, a.rows, a.H + 2 * a.Hkv);
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
    }
    return 0;
}

}  // namespace

int s3d_qk_norm_blocks(long rows, int H, int Hkv, int hd) {
    if (rows <= 0 || H < 1 || Hkv < 1 || hd < 16 || hd > 256) return 0;
    const int r = rows_per_wg(rows, H + 2 * Hkv, hd);
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
            hipLaunchKernelGGL(qk_gain_reduce_kernel, dim3((2 * a.hd + 3) / 4), dim3(256), 0, s, a.partial, 0, a.hd, a.dq_gain, a.dk_gain, 0);
            S3D_CHECK_LAUNCH("qk_gain_reduce");
        }
        return 0;
    }
    return launch<true>(a, s);
}
