// Device code of the short causal filter (fms_conv_*): forward, backward and one-token step.
//
//   pre_t = bias + sum_k w_k x_{t-K+1+k}      out_t = act(pre_t)
//   dpre_t = dout_t act'(pre_t)               dx_t = sum_k w_k dpre_{t+K-1-k}
//   dw_k = sum_{b,t} dpre_t x_{t-K+1+k}       dbias = sum dpre
//
// K is 2 to 8 and the filter is a few operations per byte, so HBM bounds it: every input is loaded
// once, 16 bytes a lane, with the loads of a whole unit (4 vectors a lane and tensor) issued before the
// first use.  A lane holds 8 consecutive positions; the K - 1 positions in front of them (for dx: the
// K - 1 values of dpre behind them) come from the neighbouring lane by shuffle, across tiles from the
// tile walked before, and only at a unit's border from memory.  Rows shorter than a warp's 256
// positions share a warp.
#pragma once

#include "ssm_kernels.cuh"

namespace fms {

constexpr int kConvUnroll = 4;  // tiles of a unit
constexpr int kConvWarps = 4;

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

template <typename S>
struct ConvProblem {
    const S *x;
    int64_t xs[2];
    const float *weight, *bias;
    const S *x0;
    const int64_t *lengths;
    int64_t batch, channels, chunks;  // chunks: units along a row
    int T, lpr, silu;                 // lpr: lanes of a row (power of two)
};

template <typename S>
struct ConvPlace {
    int64_t row, b, d, chunk;
    int l, len;
    bool live;
};
template <typename S>
__device__ __forceinline__ ConvPlace<S> conv_place(const ConvProblem<S> &p) {
    ConvPlace<S> w;
    const int lane = threadIdx.x & 31, rows = 32 / p.lpr;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kConvWarps + (threadIdx.x >> 5);
    w.chunk = unit % p.chunks;
    w.row = unit / p.chunks * rows + lane / p.lpr;
    w.l = lane % p.lpr;
    w.live = w.row < p.batch * p.channels;
    w.b = w.live ? w.row / p.channels : 0;
    w.d = w.live ? w.row - w.b * p.channels : 0;
    w.len = 0;
    if (w.live) {
        const int64_t n = p.lengths ? p.lengths[w.b] : p.T;
        w.len = static_cast<int>(n < 0 ? 0 : n > p.T ? p.T : n);
    }
    return w;
}

// Input at position t of the sequence, t < 0 reaching into x0.
template <typename S, int K>
__device__ __forceinline__ float conv_at(const ConvProblem<S> &p, const ConvPlace<S> &w, const S *row, int t) {
    if (t >= 0) return t < w.len ? Store<S>::to_float(row[t]) : 0.f;
    return p.x0 && w.live ? Store<S>::to_float(p.x0[w.row * (K - 1) + K - 1 + t]) : 0.f;
}

__device__ __forceinline__ float silu_f(float v) { return v * sigmoid_f(v); }
__device__ __forceinline__ float dsilu_f(float v) {
    const float g = sigmoid_f(v);
    return g * fmaf(v, 1.f - g, 1.f);
}

// the K - 1 inputs in front of a lane's 8 positions of tile u
template <typename S, int K, int U>
__device__ __forceinline__ void conv_halo(const ConvProblem<S> &p, const ConvPlace<S> &w, const S *row, int t0,
                                          const float (&f)[U][8], int u, float (&halo)[K - 1]) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        const float side = __shfl_up_sync(kFullMask, f[u][8 - (K - 1) + j], 1, p.lpr);
        float front;
        if (u > 0) front = __shfl_sync(kFullMask, f[u > 0 ? u - 1 : 0][8 - (K - 1) + j], p.lpr - 1, p.lpr);
        else front = w.l == 0 ? conv_at<S, K>(p, w, row, t0 - (K - 1) + j) : 0.f;
        halo[j] = w.l == 0 ? front : side;
    }
}

template <int K>
__device__ __forceinline__ float conv_tap(const float (&halo)[K - 1], const float (&f)[8], int i) {
    return i < K - 1 ? halo[i < K - 1 ? i : 0] : f[i < K - 1 ? 0 : i - (K - 1)];
}

template <typename S, int K, bool ALIGNED>
__global__ void __launch_bounds__(kConvWarps * 32)
conv_forward_kernel(const ConvProblem<S> p, S *__restrict__ out, S *__restrict__ x_last) {
    constexpr int U = kConvUnroll;
    const ConvPlace<S> w = conv_place(p);
    const S *row = p.x + w.b * p.xs[0] + w.d * p.xs[1];
    const int span = p.lpr * 8, t0 = static_cast<int>(w.chunk) * span * U + w.l * 8;
    float f[U][8], wt[K], bias = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) load8<S, ALIGNED>(row, t0 + u * span, w.len, f[u]);
#pragma unroll
    for (int k = 0; k < K; ++k) wt[k] = w.live ? p.weight[w.d * K + k] : 0.f;
    if (p.bias && w.live) bias = p.bias[w.d];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int t = t0 + u * span;
        float halo[K - 1], y[8];
        conv_halo<S, K, U>(p, w, row, t, f, u, halo);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v = bias;
#pragma unroll
            for (int k = 0; k < K; ++k) v = fmaf(wt[k], conv_tap<K>(halo, f[u], i + k), v);
            if (p.silu) v = silu_f(v);
            y[i] = t + i < w.len ? v : 0.f;
        }
        if (w.live) store8<S, ALIGNED>(out + w.row * p.T, t, p.T, y);
    }
    if (x_last && w.live && w.chunk == 0)
        for (int j = w.l; j < K - 1; j += p.lpr) {
            const int t = w.len - (K - 1) + j;
            x_last[w.row * (K - 1) + j] = from_float<S>(conv_at<S, K>(p, w, row, t));
        }
}

// part: [chunk][row][K + 1], the sums over a unit's positions of dpre * x (K of them) and of dpre.
template <typename S, int K, bool ALIGNED>
__global__ void __launch_bounds__(kConvWarps * 32)
conv_backward_kernel(const ConvProblem<S> p, const S *__restrict__ dout, const S *__restrict__ dlast,
                     S *__restrict__ dx, S *__restrict__ dx0, float *__restrict__ part) {
    constexpr int U = kConvUnroll;
    const ConvPlace<S> w = conv_place(p);
    const S *row = p.x + w.b * p.xs[0] + w.d * p.xs[1];
    const S *grow = dout + w.row * p.T;
    const int span = p.lpr * 8, t0 = static_cast<int>(w.chunk) * span * U + w.l * 8;
    float f[U][8], g[U][8], wt[K], bias = 0.f, dw[K], db = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        load8<S, ALIGNED>(row, t0 + u * span, w.len, f[u]);
        load8<S, ALIGNED>(grow, t0 + u * span, w.len, g[u]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        wt[k] = w.live ? p.weight[w.d * K + k] : 0.f;
        dw[k] = 0.f;
    }
    if (p.bias && w.live) bias = p.bias[w.d];
    // dpre of the K - 1 positions behind the unit, one a lane (a unit of fewer lanes ends its row)
    float behind[K - 1];
    {
        const int t = static_cast<int>(w.chunk + 1) * span * U + w.l;
        float v = 0.f;
        if (w.l < K - 1 && t < w.len) {
            v = Store<S>::to_float(grow[t]);
            if (p.silu) {
                float pre = bias;
#pragma unroll
                for (int k = 0; k < K; ++k) pre = fmaf(wt[k], conv_at<S, K>(p, w, row, t - (K - 1) + k), pre);
                v *= dsilu_f(pre);
            }
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            const float r = __shfl_sync(kFullMask, v, j, p.lpr);
            behind[j] = j < p.lpr ? r : 0.f;
        }
    }
#pragma unroll
    for (int u = U - 1; u >= 0; --u) {
        const int t = t0 + u * span;
        float halo[K - 1], dp[8 + K - 1], o[8];
        conv_halo<S, K, U>(p, w, row, t, f, u, halo);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v = g[u][i];
            if (p.silu) {
                float pre = bias;
#pragma unroll
                for (int k = 0; k < K; ++k) pre = fmaf(wt[k], conv_tap<K>(halo, f[u], i + k), pre);
                v *= dsilu_f(pre);
            }
            dp[i] = t + i < w.len ? v : 0.f;
            db += dp[i];
#pragma unroll
            for (int k = 0; k < K; ++k) dw[k] = fmaf(dp[i], conv_tap<K>(halo, f[u], i + k), dw[k]);
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            const float side = __shfl_down_sync(kFullMask, dp[j], 1, p.lpr);
            dp[8 + j] = w.l == p.lpr - 1 ? behind[j] : side;
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) behind[j] = __shfl_sync(kFullMask, dp[j], 0, p.lpr);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) v = fmaf(wt[k], dp[i + K - 1 - k], v);
            const int j = t + i - (w.len - (K - 1));
            if (dlast && j >= 0 && t + i < w.len) v += Store<S>::to_float(dlast[w.row * (K - 1) + j]);
            o[i] = t + i < w.len ? v : 0.f;
        }
        if (w.live) store8<S, ALIGNED>(dx + w.row * p.T, t, p.T, o);
        if (u == 0 && dx0 && w.live && w.chunk == 0 && w.l == 0) {
#pragma unroll
            for (int j = 0; j < K - 1; ++j) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k <= j; ++k) v = fmaf(wt[k], dp[j - k], v);
                if (dlast && j >= w.len) v += Store<S>::to_float(dlast[w.row * (K - 1) + j - w.len]);
                dx0[w.row * (K - 1) + j] = from_float<S>(v);
            }
        }
    }
    for (int k = 1; k < p.lpr; k *= 2) {
#pragma unroll
        for (int j = 0; j < K; ++j) dw[j] += __shfl_xor_sync(kFullMask, dw[j], k);
        db += __shfl_xor_sync(kFullMask, db, k);
    }
    if (w.live && w.l == 0) {
        float *to = part + (w.chunk * p.batch * p.channels + w.row) * (K + 1);
#pragma unroll
        for (int k = 0; k < K; ++k) to[k] = dw[k];
        to[K] = db;
    }
}

// One warp per channel: the partial sums of all units of its rows, in a fixed order.
template <int K>
__global__ void __launch_bounds__(128)
conv_weight_kernel(const float *__restrict__ part, float *__restrict__ dw, float *__restrict__ db, int64_t batch,
                   int64_t channels, int64_t chunks) {
    const int64_t d = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (d >= channels) return;
    const int lane = threadIdx.x & 31;
    float v[K + 1] = {};
    for (int64_t i = lane; i < batch * chunks; i += 32) {
        const float *src = part + (i * channels + d) * (K + 1);  // unit (chunk, b) is number chunk * batch + b
#pragma unroll
        for (int k = 0; k <= K; ++k) v[k] += src[k];
    }
#pragma unroll
    for (int o = 16; o; o /= 2)
#pragma unroll
        for (int k = 0; k <= K; ++k) v[k] += __shfl_xor_sync(kFullMask, v[k], o);
    if (lane == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) dw[d * K + k] = v[k];
        if (db) db[d] = v[K];
    }
}

template <typename S, int K>
__global__ void __launch_bounds__(128)
conv_step_kernel(const ConvProblem<S> p, S *__restrict__ state, int64_t pool, const int64_t *__restrict__ slots,
                 S *__restrict__ out, int blocks) {
    const int64_t b = blockIdx.x / blocks, d = static_cast<int64_t>(blockIdx.x % blocks) * blockDim.x + threadIdx.x;
    const int64_t slot = step_slot(slots, b, pool);
    const bool use = d < p.channels && slot >= 0;
    S *st = state + (slot * p.channels + d) * (K - 1);
    S v[K];
    float wt[K], y = 0.f;
    if (use) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) v[k] = st[k];
        v[K - 1] = p.x[b * p.xs[0] + d];
#pragma unroll
        for (int k = 0; k < K; ++k) wt[k] = p.weight[d * K + k];
        if (p.bias) y = p.bias[d];
    }
    const bool taken = slot_taken(slots, b, slot);
    if (use && !taken) {
#pragma unroll
        for (int k = 0; k < K; ++k) y = fmaf(wt[k], Store<S>::to_float(v[k]), y);
        if (p.silu) y = silu_f(y);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) st[k] = v[k + 1];
    } else {
        y = 0.f;
    }
    if (d < p.channels) out[b * p.channels + d] = from_float<S>(y);
}

}  // namespace fms
