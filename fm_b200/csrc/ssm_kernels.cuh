// Device code of the selective state-space scan (fms_ssm_*): forward, backward and one-token step.
//
//   h_t[n] = a_t[n] h_{t-1}[n] + u_t B_t[n]     a_t[n] = exp(dt_t A[n])    u_t = dt_t x_t
//   y_t    = sum_n C_t[n] h_t[n] + D x_t
//
// A warp walks some channels of one sequence along time in tiles of 64 positions.  Its lanes form a
// grid of 8 time lanes x 4 state lanes; a lane holds 8 consecutive positions of 4 states, so the 16
// states of a block and the 64 positions of a tile are spread over the warp, and B and C of the tile
// stay in registers while the warp goes through its channels.  Per channel and state a lane
//   1. forms its 8 decays (one exponential each) and its aggregate (P, S): P = exp(A * sum dt) of its
//      positions, S their state from a zero start,
//   2. takes part in a 3-step shuffle scan of the pairs over the 8 time lanes, seeded with the carry,
//   3. runs its 8 positions again from the state that enters them, in registers.
// Each decay is thus computed once and the sequence is parallel over positions, channels and states;
// a thread per channel that walks time alone needs 64 x fewer positions in flight but fills the
// machine only from some 40000 channels on, and its two-pass split along time computes every decay
// twice.  The exponentials bound the forward: 16 per clock and SM.
#pragma once

#include "scan_kernels.cuh"

namespace fms {

constexpr int kSsmE = 8;                       // consecutive positions of a lane
constexpr int kSsmTimeLanes = 8;
constexpr int kSsmTile = kSsmE * kSsmTimeLanes;  // positions of a tile
constexpr int kSsmNL = 4;                      // states of a lane
constexpr int kSsmNB = 16;                     // states of a block (4 lanes x 4)
constexpr int kSsmFwdWarps = 4;
constexpr int kSsmBwdWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename S>
struct SsmProblem {
    const S *x, *delta, *z, *B, *C;
    int64_t xs[2], ds[2], zs[2], Bs[3], Cs[3];  // element strides: batch, channel | batch, group, state
    const float *A, *D, *bias, *h0;
    const int64_t *lengths;
    int64_t batch, channels, groups;
    int T, N, NP;       // NP: states rounded up to whole blocks
    int per_group;      // channels of a group
    int cw;             // channels of a warp
    int chunks;         // CTAs along the channels of a group
    int tiles;
    int softplus;
};

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float sigmoid_f(float v) { return __fdividef(1.f, 1.f + ex2(-kLog2e * v)); }

// log(1 + exp(v)); beyond 20 the two agree to fp32's last bit.  Once per position, not per state, so
// the accurate library functions cost little; sigmoid_f is its derivative.
__device__ __forceinline__ float softplus_f(float v) { return v > 20.f ? v : log1pf(expf(v)); }

template <typename S>
__device__ __forceinline__ S from_float(float f);
template <>
__device__ __forceinline__ float from_float<float>(float f) { return f; }
template <>
__device__ __forceinline__ __half from_float<__half>(float f) { return __float2half_rn(f); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float f) { return __float2bfloat16_rn(f); }

// Positions [t, t + 8) of a row as floats; positions from `lim` on are zero and not read.  ALIGNED: the
// row starts on a 16-byte boundary and t is a multiple of 8.
template <typename S, bool ALIGNED>
__device__ __forceinline__ void load8(const S *__restrict__ row, int t, int lim, float (&f)[8]) {
    if (ALIGNED && t + 8 <= lim) {
        if constexpr (sizeof(S) == 4) {
            const float4 p = __ldg(reinterpret_cast<const float4 *>(row + t));
            const float4 q = __ldg(reinterpret_cast<const float4 *>(row + t) + 1);
            f[0] = p.x, f[1] = p.y, f[2] = p.z, f[3] = p.w;
            f[4] = q.x, f[5] = q.y, f[6] = q.z, f[7] = q.w;
        } else {
            const uint4 p = __ldg(reinterpret_cast<const uint4 *>(row + t));
            Store<S>::unpack(p, f);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = t + i < lim ? Store<S>::to_float(row[t + i]) : 0.f;
    }
}

// Stores positions [t, t + 8) of a row, those below `T` only.
template <typename S, bool ALIGNED>
__device__ __forceinline__ void store8(S *__restrict__ row, int t, int T, const float (&f)[8]) {
    if (ALIGNED && t + 8 <= T) {
        if constexpr (sizeof(S) == 4) {
            float4 *o = reinterpret_cast<float4 *>(row + t);
            o[0] = make_float4(f[0], f[1], f[2], f[3]);
            o[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4 *>(row + t) = Store<S>::pack(f);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (t + i < T) row[t + i] = from_float<S>(f[i]);
    }
}

// A tile's 64 floats in shared memory: time lane s keeps positions 8s ... 8s+3 at [4s] and the other
// four at [32 + 4s], so that 8 time lanes read or write 128 contiguous bytes.
__device__ __forceinline__ void tile_get(const float *base, int s, float (&f)[8]) {
    const float4 p = *reinterpret_cast<const float4 *>(base + 4 * s);
    const float4 q = *reinterpret_cast<const float4 *>(base + 32 + 4 * s);
    f[0] = p.x, f[1] = p.y, f[2] = p.z, f[3] = p.w;
    f[4] = q.x, f[5] = q.y, f[6] = q.z, f[7] = q.w;
}
__device__ __forceinline__ void tile_put(float *base, int s, const float (&f)[8]) {
    *reinterpret_cast<float4 *>(base + 4 * s) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4 *>(base + 32 + 4 * s) = make_float4(f[4], f[5], f[6], f[7]);
}

// Sum of v over the 4 state lanes, spread so that each of them keeps two positions: state lane q gets
// positions 4 * (q & 1) + 2 * (q >> 1) and the next.  `fresh`: the pair replaces what the tile holds.
__device__ __forceinline__ void tile_sum(float *base, int s, int q, const float (&v)[8], bool fresh) {
    const bool hi = q & 1, hi2 = q >> 1;
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float keep = hi ? v[i + 4] : v[i], give = hi ? v[i] : v[i + 4];
        r[i] = keep + __shfl_xor_sync(kFullMask, give, 8);
    }
    float2 o;
    {
        const float k0 = hi2 ? r[2] : r[0], g0 = hi2 ? r[0] : r[2];
        const float k1 = hi2 ? r[3] : r[1], g1 = hi2 ? r[1] : r[3];
        o.x = k0 + __shfl_xor_sync(kFullMask, g0, 16);
        o.y = k1 + __shfl_xor_sync(kFullMask, g1, 16);
    }
    float2 *at = reinterpret_cast<float2 *>(base + (hi ? 32 : 0) + 4 * s + (hi2 ? 2 : 0));
    if (!fresh) {
        const float2 old = *at;
        o.x += old.x;
        o.y += old.y;
    }
    *at = o;
}

// Inclusive scan of (P, S) over the 8 time lanes; lane 0's S is already the true state.
__device__ __forceinline__ float scan_up(float P, float S, int s) {
#pragma unroll
    for (int k = 1; k < 8; k *= 2) {
        const float Sp = __shfl_up_sync(kFullMask, S, k, 8);
        const float Pp = k < 4 ? __shfl_up_sync(kFullMask, P, k, 8) : 0.f;
        if (s >= k) {
            S = fmaf(P, Sp, S);
            P *= Pp;
        }
    }
    return S;
}
__device__ __forceinline__ float scan_down(float P, float S, int s) {
#pragma unroll
    for (int k = 1; k < 8; k *= 2) {
        const float Sp = __shfl_down_sync(kFullMask, S, k, 8);
        const float Pp = k < 4 ? __shfl_down_sync(kFullMask, P, k, 8) : 0.f;
        if (s + k < 8) {
            S = fmaf(P, Sp, S);
            P *= Pp;
        }
    }
    return S;
}

// Which channels a warp has: [c0, c0 + nc) of group g of sequence b; nc may be <= 0.
struct SsmPlace {
    int64_t b, d0;  // sequence; first channel counted over all groups
    int g, chunk, nc;
};
template <typename S>
__device__ __forceinline__ SsmPlace ssm_place(const SsmProblem<S> &p, int warps) {
    SsmPlace w;
    const int per = p.chunks;
    int64_t k = blockIdx.x;
    w.chunk = static_cast<int>(k % per);
    k /= per;
    w.g = static_cast<int>(k % p.groups);
    w.b = k / p.groups;
    const int c0 = (w.chunk * warps + static_cast<int>(threadIdx.x >> 5)) * p.cw;
    w.nc = min(p.cw, p.per_group - c0);
    w.d0 = static_cast<int64_t>(w.g) * p.per_group + c0;
    return w;
}
template <typename S>
__device__ __forceinline__ int ssm_length(const SsmProblem<S> &p, int64_t b) {
    if (!p.lengths) return p.T;
    const int64_t n = p.lengths[b];
    return static_cast<int>(n < 0 ? 0 : n > p.T ? p.T : n);
}

// dt of 8 raw values; positions from lim on get 0, which makes them the identity step.
template <typename S>
__device__ __forceinline__ void time_steps(const SsmProblem<S> &p, float bias, int t, int lim, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float r = v[i] + bias;
        v[i] = t + i < lim ? (p.softplus ? softplus_f(r) : r) : 0.f;
    }
}

// floats of shared memory a warp needs
inline __host__ __device__ int ssm_fwd_floats(int cw, int NP) { return cw * (3 * kSsmTile + 2 * NP); }
inline __host__ __device__ int ssm_bwd_floats(int cw, int NP) { return cw * (6 * kSsmTile + 4 * NP + 4); }

template <typename S, bool ALIGNED>
__global__ void __launch_bounds__(kSsmFwdWarps * 32)
ssm_forward_kernel(const SsmProblem<S> p, S *__restrict__ out, float *__restrict__ h_last,
                   float *__restrict__ checkpoints) {
    extern __shared__ __align__(16) float ssm_smem[];
    const int lane = threadIdx.x & 31, s = lane & 7, q = lane >> 3;
    const SsmPlace w = ssm_place(p, kSsmFwdWarps);
    if (w.nc <= 0) return;
    float *dt_ = ssm_smem + (threadIdx.x >> 5) * ssm_fwd_floats(p.cw, p.NP);
    float *u_ = dt_ + p.cw * kSsmTile, *y_ = u_ + p.cw * kSsmTile;
    float *h_ = y_ + p.cw * kSsmTile, *A_ = h_ + p.cw * p.NP;
    const int len = ssm_length(p, w.b);
    const int64_t row0 = w.b * p.channels + w.d0;

    for (int i = lane; i < w.nc * p.NP; i += 32) {
        const int c = i / p.NP, n = i - c * p.NP;
        A_[i] = n < p.N ? p.A[(w.d0 + c) * p.N + n] * kLog2e : 0.f;
        h_[i] = n < p.N && p.h0 ? p.h0[(row0 + c) * p.N + n] : 0.f;
    }
    __syncwarp();

    for (int tile = 0; tile < p.tiles; ++tile) {
        const int t = tile * kSsmTile + s * kSsmE;
        if (tile * kSsmTile >= len) {  // behind the sequence: zeros
            const float zero[8] = {};
            for (int c = q; c < w.nc; c += 4) store8<S, ALIGNED>(out + (row0 + c) * p.T, t, p.T, zero);
            continue;
        }
        if (checkpoints) {
            float *ck = checkpoints + ((w.b * p.tiles + tile) * p.channels + w.d0) * p.N;
            for (int i = lane; i < w.nc * p.N; i += 32) ck[i] = h_[i / p.N * p.NP + i % p.N];
        }
        for (int c = q; c < w.nc; c += 4) {
            float x[8], dt[8];
            load8<S, ALIGNED>(p.x + w.b * p.xs[0] + (w.d0 + c) * p.xs[1], t, len, x);
            load8<S, ALIGNED>(p.delta + w.b * p.ds[0] + (w.d0 + c) * p.ds[1], t, len, dt);
            time_steps(p, p.bias ? p.bias[w.d0 + c] : 0.f, t, len, dt);
            tile_put(dt_ + c * kSsmTile, s, dt);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= dt[i];
            tile_put(u_ + c * kSsmTile, s, x);
        }
        __syncwarp();

        for (int n0 = q * kSsmNL; n0 < p.NP; n0 += kSsmNB) {
            float B[kSsmNL][8], C[kSsmNL][8];
#pragma unroll
            for (int j = 0; j < kSsmNL; ++j) {
                const int lim = n0 + j < p.N ? len : 0;
                load8<S, ALIGNED>(p.B + w.b * p.Bs[0] + w.g * p.Bs[1] + (n0 + j) * p.Bs[2], t, lim, B[j]);
                load8<S, ALIGNED>(p.C + w.b * p.Cs[0] + w.g * p.Cs[1] + (n0 + j) * p.Cs[2], t, lim, C[j]);
            }
            for (int c = 0; c < w.nc; ++c) {
                float dt[8], u[8], y[8], sum = 0.f;
                tile_get(dt_ + c * kSsmTile, s, dt);
                tile_get(u_ + c * kSsmTile, s, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum += dt[i];
                    y[i] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < kSsmNL; ++j) {
                    const float A = A_[c * p.NP + n0 + j], carry = h_[c * p.NP + n0 + j];
                    float a[8], S0 = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        a[i] = ex2(dt[i] * A);
                        S0 = fmaf(a[i], S0, u[i] * B[j][i]);
                    }
                    const float P = ex2(sum * A);
                    if (s == 0) S0 = fmaf(P, carry, S0);
                    S0 = scan_up(P, S0, s);
                    float h = __shfl_up_sync(kFullMask, S0, 1, 8);
                    if (s == 0) h = carry;
                    if (s == 7) h_[c * p.NP + n0 + j] = S0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        h = fmaf(a[i], h, u[i] * B[j][i]);
                        y[i] = fmaf(C[j][i], h, y[i]);
                    }
                }
                tile_sum(y_ + c * kSsmTile, s, q, y, n0 < kSsmNB);
            }
        }
        __syncwarp();

        for (int c = q; c < w.nc; c += 4) {
            float y[8], x[8];
            tile_get(y_ + c * kSsmTile, s, y);
            if (p.D) {
                const float D = p.D[w.d0 + c];
                load8<S, ALIGNED>(p.x + w.b * p.xs[0] + (w.d0 + c) * p.xs[1], t, len, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = fmaf(D, x[i], y[i]);
            }
            if (p.z) {
                float z[8];
                load8<S, ALIGNED>(p.z + w.b * p.zs[0] + (w.d0 + c) * p.zs[1], t, len, z);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] *= z[i] * sigmoid_f(z[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = t + i < len ? y[i] : 0.f;
            store8<S, ALIGNED>(out + (row0 + c) * p.T, t, p.T, y);
        }
        __syncwarp();
    }
    if (h_last)
        for (int i = lane; i < w.nc * p.N; i += 32) h_last[row0 * p.N + i] = h_[i / p.N * p.NP + i % p.N];
}

// What the backward writes; the partial sums live in the caller's workspace.
template <typename S>
struct SsmGrads {
    const float *checkpoints;
    const S *grad_out;
    const float *grad_last;
    S *dx, *ddelta, *dz;
    float *dh0;
    float *bc_part;  // [batch][group][chunk][B | C][N][tiles * 64]
    float *a_part;   // [batch][D][N]
    float *d_part;   // [batch][2][D]: grad of D, grad of delta_bias
};

// g_t = C_t dy_t + c_{t+1},  c_t = a_t g_t;  with q_t = c_t h_{t-1}:
//   ddt_t = sum_n A q_t + x_t sum_n g_t B_t,  dx_t = dt_t sum_n g_t B_t + D dy_t,
//   dA = sum_t dt_t q_t,  dB_t = sum_d g_t u_t,  dC_t = sum_d dy_t h_t.
// The tiles are walked from the last to the first; the states of a tile are recomputed in registers
// from the checkpoint in front of it, the adjoint is scanned in the other direction with the same
// decays.  Sums over states cross the 4 state lanes; dB and dC add up in registers over the warp's
// channels and, once per tile, over the warps of the CTA in a fixed order; what is left (CTAs along the
// channels, sequences for dA) goes through partial sums in the workspace, so no atomics.
template <typename S, bool ALIGNED, bool GATED>
__global__ void __launch_bounds__(kSsmBwdWarps * 32, 1)
ssm_backward_kernel(const SsmProblem<S> p, const SsmGrads<S> o) {
    extern __shared__ __align__(16) float ssm_smem[];
    constexpr int W = kSsmBwdWarps;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, s = lane & 7, q = lane >> 3;
    const SsmPlace w = ssm_place(p, W);
    float *red = ssm_smem;  // [warp][64][lane]
    float *dt_ = red + W * 64 * 32 + warp * ssm_bwd_floats(p.cw, p.NP);
    const int ct = p.cw * kSsmTile, cn = p.cw * p.NP;
    float *u_ = dt_ + ct, *dy_ = u_ + ct, *gB_ = dy_ + ct, *q_ = gB_ + ct, *y_ = q_ + ct;
    float *A_ = y_ + ct, *h_ = A_ + cn, *c_ = h_ + cn, *dA_ = c_ + cn, *dD_ = dA_ + cn, *db_ = dD_ + p.cw;
    const int len = ssm_length(p, w.b);
    const int64_t row0 = w.b * p.channels + w.d0;
    const int Tpad = p.tiles * kSsmTile;
    float *bc = o.bc_part + ((w.b * p.groups + w.g) * p.chunks + w.chunk) * 2 * p.N * static_cast<int64_t>(Tpad);

    for (int i = lane; i < w.nc * p.NP; i += 32) {
        const int c = i / p.NP, n = i - c * p.NP;
        A_[i] = n < p.N ? p.A[(w.d0 + c) * p.N + n] * kLog2e : 0.f;
        c_[i] = n < p.N && o.grad_last ? o.grad_last[(row0 + c) * p.N + n] : 0.f;
        h_[i] = 0.f;
        dA_[i] = 0.f;
    }
    for (int i = lane; i < w.nc; i += 32) dD_[i] = db_[i] = 0.f;

    for (int tile = p.tiles - 1; tile >= 0; --tile) {
        const int t = tile * kSsmTile + s * kSsmE;
        if (tile * kSsmTile >= len) {
            const float zero[8] = {};
            for (int c = q; c < w.nc; c += 4) {
                store8<S, ALIGNED>(o.dx + (row0 + c) * p.T, t, p.T, zero);
                store8<S, ALIGNED>(o.ddelta + (row0 + c) * p.T, t, p.T, zero);
                if (GATED) store8<S, ALIGNED>(o.dz + (row0 + c) * p.T, t, p.T, zero);
            }
            for (int i = threadIdx.x; i < 2 * p.N * kSsmTile; i += W * 32)
                bc[static_cast<int64_t>(i / kSsmTile) * Tpad + tile * kSsmTile + i % kSsmTile] = 0.f;
            continue;
        }
        __syncwarp();
        {
            const float *ck = o.checkpoints + ((w.b * p.tiles + tile) * p.channels + w.d0) * p.N;
            for (int i = lane; i < w.nc * p.N; i += 32) h_[i / p.N * p.NP + i % p.N] = ck[i];
        }
        for (int c = q; c < w.nc; c += 4) {
            float x[8], dt[8], dy[8];
            load8<S, ALIGNED>(p.x + w.b * p.xs[0] + (w.d0 + c) * p.xs[1], t, len, x);
            load8<S, ALIGNED>(p.delta + w.b * p.ds[0] + (w.d0 + c) * p.ds[1], t, len, dt);
            load8<S, ALIGNED>(o.grad_out + (row0 + c) * p.T, t, len, dy);
            time_steps(p, p.bias ? p.bias[w.d0 + c] : 0.f, t, len, dt);
            if (GATED) {
                float z[8];
                load8<S, ALIGNED>(p.z + w.b * p.zs[0] + (w.d0 + c) * p.zs[1], t, len, z);
#pragma unroll
                for (int i = 0; i < 8; ++i) dy[i] = t + i < len ? dy[i] * z[i] * sigmoid_f(z[i]) : 0.f;
            }
            tile_put(dt_ + c * kSsmTile, s, dt);
            tile_put(dy_ + c * kSsmTile, s, dy);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= dt[i];
            tile_put(u_ + c * kSsmTile, s, x);
        }
        __syncwarp();

        for (int nb = 0; nb < p.NP; nb += kSsmNB) {
            const int n0 = nb + q * kSsmNL;
            float B[kSsmNL][8], C[kSsmNL][8], dB[kSsmNL][8], dC[kSsmNL][8];
#pragma unroll
            for (int j = 0; j < kSsmNL; ++j) {
                const int lim = n0 + j < p.N ? len : 0;
                load8<S, ALIGNED>(p.B + w.b * p.Bs[0] + w.g * p.Bs[1] + (n0 + j) * p.Bs[2], t, lim, B[j]);
                load8<S, ALIGNED>(p.C + w.b * p.Cs[0] + w.g * p.Cs[1] + (n0 + j) * p.Cs[2], t, lim, C[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) dB[j][i] = dC[j][i] = 0.f;
            }
            for (int c = 0; c < w.nc; ++c) {
                float dt[8], u[8], dy[8], gB[8], Q[8], y[8], dA[kSsmNL], sum = 0.f;
                tile_get(dt_ + c * kSsmTile, s, dt);
                tile_get(u_ + c * kSsmTile, s, u);
                tile_get(dy_ + c * kSsmTile, s, dy);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum += dt[i];
                    gB[i] = Q[i] = y[i] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < kSsmNL; ++j) {
                    const int at = c * p.NP + n0 + j;
                    const float A = A_[at], first = h_[at], carry = c_[at];
                    float a[8], h[8], S0 = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        a[i] = ex2(dt[i] * A);
                        S0 = fmaf(a[i], S0, u[i] * B[j][i]);
                    }
                    const float P = ex2(sum * A);
                    if (s == 0) S0 = fmaf(P, first, S0);
                    S0 = scan_up(P, S0, s);
                    float hin = __shfl_up_sync(kFullMask, S0, 1, 8);
                    if (s == 0) hin = first;
                    float R0 = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        h[i] = fmaf(a[i], i ? h[i - 1] : hin, u[i] * B[j][i]);
                        dC[j][i] = fmaf(dy[i], h[i], dC[j][i]);
                        if (GATED) y[i] = fmaf(C[j][i], h[i], y[i]);
                    }
#pragma unroll
                    for (int i = 7; i >= 0; --i) R0 = a[i] * fmaf(C[j][i], dy[i], R0);
                    if (s == 7) R0 = fmaf(P, carry, R0);
                    R0 = scan_down(P, R0, s);
                    float cc = __shfl_down_sync(kFullMask, R0, 1, 8);
                    if (s == 7) cc = carry;
                    if (s == 0) c_[at] = R0;
                    dA[j] = 0.f;
#pragma unroll
                    for (int i = 7; i >= 0; --i) {
                        const float g = fmaf(C[j][i], dy[i], cc);
                        cc = a[i] * g;
                        const float qq = cc * (i ? h[i - 1] : hin);
                        Q[i] = fmaf(A, qq, Q[i]);
                        dA[j] = fmaf(dt[i], qq, dA[j]);
                        gB[i] = fmaf(g, B[j][i], gB[i]);
                        dB[j][i] = fmaf(g, u[i], dB[j][i]);
                    }
                }
                {  // dA over the 8 time lanes: lane s < 4 keeps state 2 * (s & 1) + (s >> 1)
                    const bool hi = s & 1, hi2 = s & 2;
                    const float k0 = hi ? dA[2] : dA[0], g0 = hi ? dA[0] : dA[2];
                    const float k1 = hi ? dA[3] : dA[1], g1 = hi ? dA[1] : dA[3];
                    const float r0 = k0 + __shfl_xor_sync(kFullMask, g0, 1);
                    const float r1 = k1 + __shfl_xor_sync(kFullMask, g1, 1);
                    float v = (hi2 ? r1 : r0) + __shfl_xor_sync(kFullMask, hi2 ? r0 : r1, 2);
                    v += __shfl_xor_sync(kFullMask, v, 4);
                    if (s < 4) dA_[c * p.NP + n0 + 2 * (s & 1) + (s >> 1)] += v;
                }
                tile_sum(gB_ + c * kSsmTile, s, q, gB, nb == 0);
                tile_sum(q_ + c * kSsmTile, s, q, Q, nb == 0);
                if (GATED) tile_sum(y_ + c * kSsmTile, s, q, y, nb == 0);
            }
            // dB, dC over the warps of the CTA
            float *mine = red + warp * 64 * 32 + lane;
#pragma unroll
            for (int j = 0; j < kSsmNL; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    mine[(j * 8 + i) * 32] = dB[j][i];
                    mine[((4 + j) * 8 + i) * 32] = dC[j][i];
                }
            __syncthreads();
            {
                static_assert(W == 2 * kSsmNL, "a warp sums the values of one state of dB or dC");
                const int n = nb + q * kSsmNL + (warp & 3);
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[i] = 0.f;
#pragma unroll
                    for (int k = 0; k < W; ++k) v[i] += red[(k * 64 + warp * 8 + i) * 32 + lane];
                }
                if (n < p.N) {
                    float4 *to = reinterpret_cast<float4 *>(bc + (static_cast<int64_t>(warp >> 2) * p.N + n) * Tpad + t);
                    to[0] = make_float4(v[0], v[1], v[2], v[3]);
                    to[1] = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
            __syncthreads();
        }

        for (int c = q; c < w.nc; c += 4) {
            float x[8], raw[8], dy[8], dt[8], gB[8], Q[8], out[8];
            tile_get(dt_ + c * kSsmTile, s, dt);
            tile_get(dy_ + c * kSsmTile, s, dy);
            tile_get(gB_ + c * kSsmTile, s, gB);
            tile_get(q_ + c * kSsmTile, s, Q);
            const float D = p.D ? p.D[w.d0 + c] : 0.f, bias = p.bias ? p.bias[w.d0 + c] : 0.f;
            load8<S, ALIGNED>(p.x + w.b * p.xs[0] + (w.d0 + c) * p.xs[1], t, len, x);
            load8<S, ALIGNED>(p.delta + w.b * p.ds[0] + (w.d0 + c) * p.ds[1], t, len, raw);
            float sD = 0.f, sb = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                out[i] = t + i < len ? fmaf(dt[i], gB[i], D * dy[i]) : 0.f;
                sD = fmaf(dy[i], x[i], sD);
            }
            store8<S, ALIGNED>(o.dx + (row0 + c) * p.T, t, p.T, out);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = fmaf(kLn2, Q[i], x[i] * gB[i]);
                if (p.softplus && raw[i] + bias <= 20.f) v *= sigmoid_f(raw[i] + bias);
                out[i] = t + i < len ? v : 0.f;
                sb += out[i];
            }
            store8<S, ALIGNED>(o.ddelta + (row0 + c) * p.T, t, p.T, out);
            if (GATED) {
                float z[8], y[8], up[8];
                tile_get(y_ + c * kSsmTile, s, y);
                load8<S, ALIGNED>(p.z + w.b * p.zs[0] + (w.d0 + c) * p.zs[1], t, len, z);
                load8<S, ALIGNED>(o.grad_out + (row0 + c) * p.T, t, len, up);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float sg = sigmoid_f(z[i]);
                    out[i] = t + i < len ? up[i] * fmaf(D, x[i], y[i]) * sg * fmaf(z[i], 1.f - sg, 1.f) : 0.f;
                }
                store8<S, ALIGNED>(o.dz + (row0 + c) * p.T, t, p.T, out);
            }
            // the lanes of one state-lane row hold one channel: they are the active ones
            const unsigned row = 0xffu << (q * 8);
#pragma unroll
            for (int k = 1; k < 8; k *= 2) {
                sD += __shfl_xor_sync(row, sD, k);
                sb += __shfl_xor_sync(row, sb, k);
            }
            if (s == 0) {
                dD_[c] += sD;
                db_[c] += sb;
            }
        }
    }
    __syncwarp();
    for (int i = lane; i < w.nc * p.N; i += 32) {
        const int c = i / p.N, k = c * p.NP + i % p.N;
        o.a_part[row0 * p.N + i] = dA_[k];
        if (o.dh0) o.dh0[row0 * p.N + i] = c_[k];
    }
    for (int i = lane; i < w.nc; i += 32) {
        o.d_part[(w.b * 2) * p.channels + w.d0 + i] = dD_[i];
        o.d_part[(w.b * 2 + 1) * p.channels + w.d0 + i] = db_[i];
    }
}

// grad_B, grad_C: the chunks' partial sums in order, rounded once.
template <typename S>
__global__ void ssm_bc_kernel(const float *__restrict__ part, S *__restrict__ dB, S *__restrict__ dC, int64_t groups,
                              int chunks, int N, int T, int Tpad) {
    const int64_t row = blockIdx.x;  // (batch * group, which, n)
    const int n = static_cast<int>(row % N), which = static_cast<int>(row / N % 2);
    const int64_t bg = row / N / 2;
    const float *src = part + ((bg * chunks) * 2 + which) * N * static_cast<int64_t>(Tpad) + n * static_cast<int64_t>(Tpad);
    S *dst = (which ? dC : dB) + (bg * N + n) * T;
    const int64_t step = 2 * static_cast<int64_t>(N) * Tpad;
    for (int t = blockIdx.y * blockDim.x + threadIdx.x; t < T; t += gridDim.y * blockDim.x) {
        float v = 0.f;
        for (int k = 0; k < chunks; ++k) v += src[k * step + t];
        dst[t] = from_float<S>(v);
    }
}

// out[i] = sum over `count` slices of `stride` floats, in order
__global__ void sum_slices_kernel(const float *__restrict__ part, float *__restrict__ out, int64_t n, int64_t count,
                                  int64_t stride) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n) return;
    float v = 0.f;
    for (int64_t k = 0; k < count; ++k) v += part[k * stride + i];
    out[i] = v;
}

// ---------------------------------------------------------------- one token ------------------
// Row b's place in the pool, or -1 for padding.  A slot that an earlier row names belongs to that row:
// every thread looks at its share of the earlier rows and the block votes, while the loads of the
// state that the caller issued before are on their way.
__device__ __forceinline__ int64_t step_slot(const int64_t *slots, int64_t b, int64_t pool) {
    const int64_t v = slots ? slots[b] : b;
    return v >= 0 && v < pool ? v : -1;
}
__device__ __forceinline__ bool slot_taken(const int64_t *slots, int64_t b, int64_t slot) {
    bool seen = false;
    if (slots && slot >= 0)
        for (int64_t k = threadIdx.x; k < b; k += blockDim.x) seen |= slots[k] == slot;
    return __syncthreads_or(seen);
}

// L lanes share a channel, a lane has 4 consecutive states at a time.  Bound by the states' bytes
// (8 per state) and, for a few rows, by latency: all loads are issued before the first use.
template <typename S, bool VEC>
__global__ void __launch_bounds__(128)
ssm_step_kernel(const SsmProblem<S> p, float *__restrict__ state, int64_t pool, const int64_t *__restrict__ slots,
                S *__restrict__ out, int L, int blocks) {
    const int64_t b = blockIdx.x / blocks;
    const int l = threadIdx.x % L;
    const int64_t d = static_cast<int64_t>(blockIdx.x % blocks) * (blockDim.x / L) + threadIdx.x / L;
    const bool live = d < p.channels;
    const int64_t slot = step_slot(slots, b, pool);
    const bool use = live && slot >= 0;
    const int64_t g = live ? d / p.per_group : 0;
    float x = 0.f, dt = 0.f, z = 0.f, D = 0.f;
    float h[4] = {}, A[4] = {}, B[4] = {}, C[4] = {};
    float *hp = state + (slot * p.channels + d) * p.N;
    const float *Ap = p.A + d * p.N;
    const S *Bp = p.B + b * p.Bs[0] + g * p.Bs[1], *Cp = p.C + b * p.Cs[0] + g * p.Cs[1];
    auto fetch = [&](int n) {
        if constexpr (VEC) {
            const float4 hv = *reinterpret_cast<const float4 *>(hp + n);
            const float4 av = __ldg(reinterpret_cast<const float4 *>(Ap + n));
            h[0] = hv.x, h[1] = hv.y, h[2] = hv.z, h[3] = hv.w;
            A[0] = av.x, A[1] = av.y, A[2] = av.z, A[3] = av.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = n + i < p.N;
            if (!VEC) {
                h[i] = in ? hp[n + i] : 0.f;
                A[i] = in ? Ap[n + i] : 0.f;
            }
            B[i] = in ? Store<S>::to_float(Bp[n + i]) : 0.f;
            C[i] = in ? Store<S>::to_float(Cp[n + i]) : 0.f;
        }
    };
    if (use) {
        x = Store<S>::to_float(p.x[b * p.xs[0] + d]);
        dt = Store<S>::to_float(p.delta[b * p.ds[0] + d]) + (p.bias ? p.bias[d] : 0.f);
        if (p.z) z = Store<S>::to_float(p.z[b * p.zs[0] + d]);
        if (p.D) D = p.D[d];
        if (4 * l < p.N) fetch(4 * l);
    }
    const bool taken = slot_taken(slots, b, slot);
    float y = 0.f;
    if (use && !taken) {
        if (p.softplus) dt = softplus_f(dt);
        const float u = dt * x;
        for (int n = 4 * l; n < p.N; n += 4 * L) {
            if (n != 4 * l) fetch(n);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] = fmaf(ex2(dt * (A[i] * kLog2e)), h[i], u * B[i]);
                y = fmaf(C[i], h[i], y);
            }
            if constexpr (VEC) {
                *reinterpret_cast<float4 *>(hp + n) = make_float4(h[0], h[1], h[2], h[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.N) hp[n + i] = h[i];
            }
        }
    }
    for (int k = 1; k < L; k *= 2) y += __shfl_xor_sync(kFullMask, y, k);
    if (live && l == 0) {
        y = fmaf(D, x, y);
        if (p.z) y *= z * sigmoid_f(z);
        out[b * p.channels + d] = from_float<S>(use && !taken ? y : 0.f);
    }
}

}  // namespace fms
