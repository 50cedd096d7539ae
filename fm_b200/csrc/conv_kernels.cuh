// Device code of the short causal filter (fms_conv_*): forward, backward and one-token step.
//
//   pre_t = bias + sum_k w_k x_{t-K+1+k}      out_t = act(pre_t)
//   dpre_t = dout_t act'(pre_t)               dx_t = sum_k w_k dpre_{t+K-1-k}
//   dw_k = sum_{b,t} dpre_t x_{t-K+1+k}       dbias = sum dpre
//
// K is 2 to 8 and the filter is a few operations per byte, so HBM bounds it as long as there are few
// instructions per position: every input is loaded once, 16 bytes a lane, with the loads of a group (4
// vectors a lane and tensor) issued before the first is unpacked, and a warp walks several groups of its
// row.  A lane holds 8 consecutive positions, laid on the 16-byte grid of the row it writes, so rows of any
// length are stored in vectors, and loaded in vectors where they have the same offset from the grid.
// The K - 1 positions in front of a lane's (for dx: the K - 1 values of dpre behind them) come from the
// neighbouring lane by shuffle, across tiles from the tile walked before, and only at a unit's border from
// memory.  Rows shorter than a group share a warp.  What happens at a row's ends is kept out of line.
//
// Measured at (8,2048,4096) bf16, 4 taps, SiLU: forward 62 us = 4.3 TB/s, backward 117 us = 3.4 TB/s (bytes alone:
// 42 and 62 us at the measured copy rate); issue slots bound it, some 170 and 320 instructions for a warp's
// 256 positions.  Rows of odd length, (3,768,16385) fp16: 39 us = 3.9 TB/s.
#pragma once

#include "ssm_kernels.cuh"

namespace fms {

constexpr int kConvUnroll = 4;  // tiles of a group
constexpr int kConvWarps = 4;

template <typename S>
struct ConvProblem {
    const S *x;
    int64_t xs[2];
    const float *weight, *bias;
    const S *x0;
    const int64_t *lengths;
    int64_t batch, channels;
    int T, lpr, silu;             // lpr: lanes of a row (power of two)
    int groups, per_unit, units;  // groups of a row, of a unit; units of a row
};

template <typename S>
struct ConvPlace {
    const S *x, *x0;  // the row at t = 0; the K - 1 inputs in front of it, or null
    int64_t row, d;
    int unit, l, len, t0, first, last;  // t0: the lane's first position of group 0; groups [first, last)
    bool live;
};
// Grid: x = unit of a row + units * block of channels, y = sequence.  `lead`: positions that the row's grid
// starts in front of t = 0, on top of the row's offset from it.
template <typename S, int K>
__device__ __forceinline__ ConvPlace<S> conv_place(const ConvProblem<S> &p, int64_t b, const S *written, int lead) {
    ConvPlace<S> w;
    const int block = static_cast<int>(blockIdx.x) / p.units;
    const int lane = threadIdx.x & 31, log = 31 - __clz(p.lpr);
    w.unit = static_cast<int>(blockIdx.x) - block * p.units;
    w.first = w.unit * p.per_unit;
    w.last = min(p.groups, w.first + p.per_unit);
    w.d = ((static_cast<int64_t>(block) * kConvWarps + (threadIdx.x >> 5)) << (5 - log)) + (lane >> log);
    w.l = lane & (p.lpr - 1);
    w.live = w.d < p.channels;
    if (!w.live) w.d = 0;
    w.row = b * p.channels + w.d;
    w.x = p.x + b * p.xs[0] + w.d * p.xs[1];
    w.x0 = p.x0 ? p.x0 + w.row * (K - 1) : nullptr;
    w.len = 0;
    if (w.live) {
        const int64_t n = p.lengths ? p.lengths[b] : p.T;
        w.len = static_cast<int>(n < 0 ? 0 : n > p.T ? p.T : n);
    }
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(written + w.row * p.T) & 15) / sizeof(S));
    w.t0 = w.l * 8 - off - lead;
    return w;
}

// Input at position t of the sequence, t < 0 reaching into x0.
template <typename S, int K>
__device__ __forceinline__ S conv_in(const ConvPlace<S> &w, int t) {
    if (t >= 0) return t < w.len ? w.x[t] : from_float<S>(0.f);
    return w.x0 && w.live && t >= 1 - K ? w.x0[K - 1 + t] : from_float<S>(0.f);
}
template <typename S, int K>
__device__ __forceinline__ float conv_at(const ConvPlace<S> &w, int t) {
    return Store<S>::to_float(conv_in<S, K>(w, t));
}

// Eight values as they are stored.
template <typename S>
union Raw8 {
    uint4 v[sizeof(S) / 2];
    S s[8];
};
struct Eight {
    float f[8];
};
// Issued where `on`, without a branch: nothing waits for the value until it is used.
template <typename S>
__device__ __forceinline__ Raw8<S> load8(const S *__restrict__ p, bool on) {
    Raw8<S> r;
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(S)) / 2; ++k)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.s32 q, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\t"
                     "mov.b32 %3, 0;\n\t@q ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                     : "=&r"(r.v[k].x), "=&r"(r.v[k].y), "=&r"(r.v[k].z), "=&r"(r.v[k].w)
                     : "l"(reinterpret_cast<const uint4 *>(p) + k), "r"(static_cast<int>(on)));
    return r;
}
// positions t ... t + 7 where a vector will not do: zeros from `len` on; `back` inputs lie in front of t = 0
template <typename S>
__device__ __noinline__ Raw8<S> load8_edge(const S *row, const S *x0, int t, int len, int back) {
    Raw8<S> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int at = t + i;
        r.s[i] = at >= 0 ? (at < len ? row[at] : from_float<S>(0.f)) : (x0 && at >= -back ? x0[back + at] : from_float<S>(0.f));
    }
    return r;
}
template <typename S>
__device__ __forceinline__ void unpack8(const Raw8<S> &r, float (&f)[8]) {
    if constexpr (sizeof(S) == 4) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            f[4 * k] = __uint_as_float(r.v[k].x), f[4 * k + 1] = __uint_as_float(r.v[k].y);
            f[4 * k + 2] = __uint_as_float(r.v[k].z), f[4 * k + 3] = __uint_as_float(r.v[k].w);
        }
    } else {
        Store<S>::unpack(r.v[0], f);
    }
}
template <typename S>
__device__ __noinline__ void store8_edge(S *row, int t, int len, int T, Eight e) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (t + i >= 0 && t + i < T) row[t + i] = from_float<S>(t + i < len ? e.f[i] : 0.f);
}
// Eight outputs: in one vector where all belong to the sequence, else those that do, and zeros behind it.
template <typename S>
__device__ __forceinline__ void store8(S *__restrict__ row, int t, int len, int T, const Eight &e) {
    if (t >= 0 && t + 8 <= len) {
        if constexpr (sizeof(S) == 4) {
            reinterpret_cast<float4 *>(row + t)[0] = make_float4(e.f[0], e.f[1], e.f[2], e.f[3]);
            reinterpret_cast<float4 *>(row + t)[1] = make_float4(e.f[4], e.f[5], e.f[6], e.f[7]);
        } else {
            *reinterpret_cast<uint4 *>(row + t) = Store<S>::pack(e.f);
        }
    } else if (t < T) {
        store8_edge(row, t, len, T, e);
    }
}

__device__ __forceinline__ float silu_f(float v) { return v * sigmoid_f(v); }
__device__ __forceinline__ float dsilu_f(float v) {
    const float g = sigmoid_f(v);
    return g * fmaf(v, 1.f - g, 1.f);
}

template <int K>
__device__ __forceinline__ float conv_sum(const float (&wt)[K], float v, const float (&halo)[K - 1], const float (&f)[8], int i) {
#pragma unroll
    for (int k = 0; k < K; ++k) v = fmaf(wt[k], i + k < K - 1 ? halo[i + k < K - 1 ? i + k : 0] : f[i + k < K - 1 ? 0 : i + k - (K - 1)], v);
    return v;
}

// Seven CTAs an SM where the loads of a group are few registers: 68 -> 62 us at (8,2048,4096) bf16.
template <typename S, int K>
__global__ void __launch_bounds__(kConvWarps * 32, sizeof(S) == 4 ? 4 : K <= 4 ? 7 : 6)
conv_forward_kernel(const ConvProblem<S> p, S *__restrict__ out, S *__restrict__ x_last) {
    constexpr int U = kConvUnroll;
    const int span = p.lpr * 8;
    for (int64_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
        const ConvPlace<S> w = conv_place<S, K>(p, b, out, 0);
        S *to = out + w.row * p.T;
        const bool same = same_phase16(w.x, to);
        Raw8<S> raw[U];
        float wt[K], bias = 0.f, prev[K - 1];
        auto fetch = [&](int group) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = w.t0 + (group * U + u) * span;
                raw[u] = load8(w.x + t, same && t >= 0 && t + 8 <= w.len);
            }
        };
#pragma unroll
        for (int k = 0; k < K; ++k) wt[k] = w.live ? p.weight[w.d * K + k] : 0.f;
        if (p.bias && w.live) bias = p.bias[w.d];
#pragma unroll
        for (int j = 0; j < K - 1; ++j) prev[j] = w.l == 0 ? conv_at<S, K>(w, w.t0 + w.first * U * span - (K - 1) + j) : 0.f;
        for (int group = w.first; group < w.last; ++group) {
            fetch(group);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = w.t0 + (group * U + u) * span;
                float f[8], halo[K - 1];
                Eight y;
                if (!same || t < 0 || t + 8 > w.len) raw[u] = load8_edge(w.x, w.live ? w.x0 : nullptr, t, w.len, K - 1);
                unpack8(raw[u], f);
#pragma unroll
                for (int j = 0; j < K - 1; ++j) {  // lane 0 gets the last lane's, for the next tile
                    const float side = __shfl_sync(kFullMask, f[8 - (K - 1) + j], w.l + p.lpr - 1, p.lpr);
                    halo[j] = w.l == 0 ? prev[j] : side;
                    prev[j] = side;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) y.f[i] = conv_sum<K>(wt, bias, halo, f, i);
                if (p.silu) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) y.f[i] = silu_f(y.f[i]);
                }
                if (w.live) store8(to, t, w.len, p.T, y);
            }
        }
        if (x_last && w.live && w.unit == 0)
            for (int j = w.l; j < K - 1; j += p.lpr) x_last[w.row * (K - 1) + j] = conv_in<S, K>(w, w.len - (K - 1) + j);
    }
}

// What a row's ends add to the gradient of positions t ... t + 7: that of the last K - 1 inputs; and the
// positions in front of t = 0 go to x0.
template <typename S, int K>
__device__ __noinline__ Eight conv_ends(Eight v, const S *dlast, S *dx0, int t, int len) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int at = t + i, j = at - (len - (K - 1));
        if (dlast && j >= 0 && j < K - 1 && at >= 1 - K) v.f[i] += Store<S>::to_float(dlast[j]);
        if (dx0 && at < 0 && at >= 1 - K) dx0[K - 1 + at] = from_float<S>(v.f[i]);
    }
    return v;
}
__device__ __noinline__ inline Eight keep_inside(Eight v, int t, int len) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (t + i < 0 || t + i >= len) v.f[i] = 0.f;
    return v;
}

// part: [unit][row][K + 1], the sums over a unit's positions of dpre * x (K of them) and of dpre.  The groups
// are walked from the last to the first.
template <typename S, int K>
__global__ void __launch_bounds__(kConvWarps * 32, sizeof(S) == 4 ? 3 : 4)
conv_backward_kernel(const ConvProblem<S> p, const S *__restrict__ dout, const S *__restrict__ dlast,
                     S *__restrict__ dx, S *__restrict__ dx0, float *__restrict__ part) {
    constexpr int U = kConvUnroll;
    const int span = p.lpr * 8;
    for (int64_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
        const ConvPlace<S> w = conv_place<S, K>(p, b, dx, dx0 ? 8 : 0);  // the grid takes the positions of x0 in
        const S *grow = dout + w.row * p.T;
        S *to = dx + w.row * p.T;
        const bool same_x = same_phase16(w.x, to), same_g = same_phase16(grow, to);
        float wt[K], bias = 0.f, dw[K], db = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            wt[k] = w.live ? p.weight[w.d * K + k] : 0.f;
            dw[k] = 0.f;
        }
        if (p.bias && w.live) bias = p.bias[w.d];
        // dpre of the K - 1 positions behind the unit, one a lane (a unit of fewer lanes ends its row)
        float behind[K - 1];
        {
            const int t = w.t0 - w.l * 7 + span * U * w.last;  // the l-th position behind
            float v = 0.f;
            if (w.l < K - 1 && t < w.len) {
                v = Store<S>::to_float(grow[t]);
                if (p.silu) {
                    float pre = bias;
#pragma unroll
                    for (int k = 0; k < K; ++k) pre = fmaf(wt[k], conv_at<S, K>(w, t - (K - 1) + k), pre);
                    v *= dsilu_f(pre);
                }
            }
#pragma unroll
            for (int j = 0; j < K - 1; ++j) {
                const float r = __shfl_sync(kFullMask, v, j, p.lpr);
                behind[j] = j < p.lpr ? r : 0.f;
            }
        }
        for (int group = w.last - 1; group >= w.first; --group) {
            const int tg = w.t0 + group * U * span;
            Raw8<S> fr[U], gr[U];
            S front[K - 1];  // lane 0: the inputs in front of the group
            float turn[K - 1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = tg + u * span;
                const bool inside = t >= 0 && t + 8 <= w.len;
                fr[u] = load8(w.x + t, same_x && inside);
                gr[u] = load8(grow + t, same_g && inside);
            }
#pragma unroll
            for (int j = 0; j < K - 1; ++j) front[j] = w.l == 0 ? conv_in<S, K>(w, tg - (K - 1) + j) : from_float<S>(0.f);
#pragma unroll
            for (int u = U - 1; u >= 0; --u) {
                const int t = tg + u * span;
                float f[8 + K - 1], dp[8 + K - 1];  // inputs from t - K + 1 on; dpre from t on
                {
                    float a[8], g[8], halo[K - 1];
                    if (u == U - 1) {  // the rest of the group that did not come in vectors
#pragma unroll
                        for (int k = 0; k < U; ++k) {
                            const int tk = tg + k * span;
                            const bool inside = tk >= 0 && tk + 8 <= w.len;
                            if (!same_x || !inside) fr[k] = load8_edge(w.x, w.live ? w.x0 : nullptr, tk, w.len, K - 1);
                            if (!same_g || !inside) gr[k] = load8_edge(grow, static_cast<const S *>(nullptr), tk, w.len, 0);
                        }
                    }
                    unpack8(fr[u], a);
                    unpack8(gr[u], g);
#pragma unroll
                    for (int j = 0; j < K - 1; ++j) {  // lane 0 gets the last lane's of the tile in front
                        if (u == U - 1) turn[j] = __shfl_sync(kFullMask, a[8 - (K - 1) + j], w.l + p.lpr - 1, p.lpr);
                        const float side = turn[j];
                        turn[j] = u ? __shfl_sync(kFullMask, Store<S>::to_float(fr[u ? u - 1 : 0].s[8 - (K - 1) + j]), w.l + p.lpr - 1, p.lpr)
                                    : Store<S>::to_float(front[j]);
                        f[j] = halo[j] = w.l == 0 ? turn[j] : side;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        f[K - 1 + i] = a[i];
                        dp[i] = p.silu ? g[i] * dsilu_f(conv_sum<K>(wt, bias, halo, a, i)) : g[i];
                    }
                }
                if (p.silu && (t < 0 || t + 8 > w.len)) {  // a zero there times a slope that may not be finite
                    Eight v;
#pragma unroll
                    for (int i = 0; i < 8; ++i) v.f[i] = dp[i];
                    v = keep_inside(v, t, w.len);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dp[i] = v.f[i];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    db += dp[i];
#pragma unroll
                    for (int k = 0; k < K; ++k) dw[k] = fmaf(dp[i], f[i + k], dw[k]);
                }
#pragma unroll
                for (int j = 0; j < K - 1; ++j) {
                    const float side = __shfl_sync(kFullMask, dp[j], w.l + 1, p.lpr);  // the last lane gets lane 0's
                    dp[8 + j] = w.l == p.lpr - 1 ? behind[j] : side;
                    behind[j] = side;
                }
                Eight v;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v.f[i] = wt[K - 1] * dp[i];
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) v.f[i] = fmaf(wt[k], dp[i + K - 1 - k], v.f[i]);
                }
                if (w.live) {
                    if ((dlast || dx0) && (t < 0 || t + 8 > w.len - (K - 1)))
                        v = conv_ends<S, K>(v, dlast ? dlast + w.row * (K - 1) : nullptr, dx0 ? dx0 + w.row * (K - 1) : nullptr, t, w.len);
                    store8(to, t, w.len, p.T, v);
                }
            }
        }
        for (int k = 1; k < p.lpr; k *= 2) {
#pragma unroll
            for (int j = 0; j < K; ++j) dw[j] += __shfl_xor_sync(kFullMask, dw[j], k);
            db += __shfl_xor_sync(kFullMask, db, k);
        }
        if (w.live && w.l == 0) {
            float *sums = part + (static_cast<int64_t>(w.unit) * p.batch * p.channels + w.row) * (K + 1);
#pragma unroll
            for (int k = 0; k < K; ++k) sums[k] = dw[k];
            sums[K] = db;
        }
    }
}

// One warp per channel: the partial sums of all units of its rows, in a fixed order.
template <int K>
__global__ void __launch_bounds__(128)
conv_weight_kernel(const float *__restrict__ part, float *__restrict__ dw, float *__restrict__ db, int64_t batch,
                   int64_t channels, int units) {
    const int64_t d = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (d >= channels) return;
    const int lane = threadIdx.x & 31;
    float v[K + 1] = {};
    for (int64_t i = lane; i < batch * units; i += 32) {
        const float *src = part + (i * channels + d) * (K + 1);  // (unit, b) is number unit * batch + b
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
    const bool taken = __syncthreads_or(slot_seen(slots, b, slot));
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
