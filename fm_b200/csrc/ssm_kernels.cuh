// Device code of the selective state-space scan (fms_ssm_*): forward, backward and one-token step.
//
//   h_t[n] = a_t[n] h_{t-1}[n] + u_t B_t[n]     a_t[n] = exp(dt_t A[n])    u_t = dt_t x_t
//   y_t    = sum_n C_t[n] h_t[n] + D x_t
//
// A warp walks some channels of one sequence along time in tiles of 64 positions.  Its lanes form a
// grid of 8 time lanes x 4 state lanes; a lane holds 8 consecutive positions of 4 states, so the 16
// states of a block and the 64 positions of a tile are spread over the warp, and B and C of the tile
// stay in registers while the warp goes through its channels.  Per channel and state a lane
//   1. forms its 8 decays (one exponential each) and its aggregate (P, S): P = exp(A * sum dt), one more
//      exponential, which unlike the product of the decays does not add up their roundings over a long
//      memory; S the state of its positions from a zero start,
//   2. takes part in a 3-step shuffle scan of the pairs over the 8 time lanes, seeded with the carry,
//   3. runs its 8 positions again from the state that enters them, in registers.
// Each decay is thus computed once and the sequence is parallel over positions, channels and states;
// a thread per channel that walks time alone needs 64 x fewer positions in flight but fills the
// machine only from some 40000 channels on, and its two-pass split along time computes every decay
// twice.
//
// Rates that shape the code, measured per SM quarter: an exponential takes 8 cycles per warp, a
// shuffle 4, a packed pair of fp32 multiply-adds 2 (one issue slot instead of two), a 16-byte
// shared-memory load 16 for the SM's four quarters together whatever its lanes share.  Hence B and C stay in
// registers; work that is the same for all states of a position (time step, gate) is done once per
// position, four positions a lane; multiply-adds are packed in pairs (of states forward, of positions
// backward, where pairs of states would take twice the registers for what they share); two channels
// forward and two states backward go side by side, since a warp alone issues once in four to five cycles;
// and the tile's inputs come through shared memory, copied asynchronously one tile ahead: B and C once for
// the CTA, the rows once per warp.
//
// Measured at (8,1024,4096) bf16, N = 16, with gate: forward 0.44 ms, of which the exponentials alone would
// take 0.12 ms and the bytes 0.04 ms; backward 1.21 ms (0.12 ms, 0.07 ms).  What bounds them are the
// latencies of the scan's dependent steps at 8 warps an SM (registers): per channel's tile of 64 positions
// a warp of the forward issues some 280 instructions for the states and 100 for the positions, plus 550
// per tile; the backward about two and a half times as many.
#pragma once

#include "scan_kernels.cuh"

namespace fms {

constexpr int kSsmE = 8;                       // consecutive positions of a lane
constexpr int kSsmTimeLanes = 8;
constexpr int kSsmTile = kSsmE * kSsmTimeLanes;  // positions of a tile
constexpr int kSsmNL = 4;                      // states of a lane
constexpr int kSsmNB = 16;                     // states of a block (4 lanes x 4)
constexpr int kSsmFwdWarps = 4;
constexpr int kSsmStages = 2;                  // tiles in shared memory; three and four were no faster
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
    int segs, seg_tiles;  // time is cut into segs pieces of seg_tiles tiles, each with CTAs of its own
};

// ------------------------------------------------------------------------------ arithmetic ----
__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float sigmoid_f(float v) { return rcp(1.f + ex2(-kLog2e * v)); }

// two fp32 values in one 64-bit register pair; one instruction works on both
using f2 = unsigned long long;
__device__ __forceinline__ f2 pk(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float lo(f2 v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float hi(f2 v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// log(1 + exp(v)) = max(v, 0) + log1p(e) with e = exp(-|v|) in (0, 1].  The argument |v| log2(e) is taken to
// twice the precision (its rounding would cost e up to |v| roundings, and a state adds up the time steps of
// its whole memory).  log1p(e) = 2 artanh(r) with r = e / (2 + e) <= 1/3, so small e keep their relative
// precision; artanh(r) / r is a polynomial of degree 4 in r^2, fitted at Chebyshev points of [0, 1/9] and off
// by at most 8e-9.  sigmoid_f is its derivative.
__device__ __forceinline__ float softplus_f(float v) {
    constexpr float kLog2eLow = 1.925963033500e-8f, kLn2f = 0.6931471805599453f;  // log2(e) - kLog2e
    const float w = -fabsf(v), t = w * kLog2e, low = fmaf(w, kLog2e, -t) + w * kLog2eLow;
    float e = ex2(t);
    e = fmaf(e, low * kLn2f, e);
    const float r = e * rcp(2.f + e), q = r * r;
    float s = fmaf(0.14087329f, q, 0.13980709f);
    s = fmaf(s, q, 0.20012427f);
    s = fmaf(s, q, 0.33333158f);
    s = fmaf(s, q, 1.f);
    const float y = fmaf(r + r, s, v > 0.f ? v : v != v ? v : 0.f);
    return w < -80.f ? fmaxf(v, 0.f) : y;  // beyond, e is not a normal number and its correction no number
}

template <typename S>
__device__ __forceinline__ S from_float(float f);
template <>
__device__ __forceinline__ float from_float<float>(float f) { return f; }
template <>
__device__ __forceinline__ __half from_float<__half>(float f) { return __float2half_rn(f); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float f) { return __float2bfloat16_rn(f); }

template <typename S>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// --------------------------------------------------------------------- a row's tile, staged ----
// 64 positions of a row lie in shared memory as they are in global memory: whole 16-byte granules,
// from the one that holds the first position; rows that do not start on a 16-byte boundary need one
// granule more.  What lies behind `lim` is filled with zeros and not read.
template <typename S>
__host__ __device__ constexpr int row_bytes() { return kSsmTile * static_cast<int>(sizeof(S)) + 16; }

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All of this thread's copies but those of the N newest groups have arrived.
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Thread `i` of `n` (a multiple of 32) copies its granules of `rows` rows; src(row) gives a row's first
// position (t = 0), or null for a row of zeros.  `any`: some valid address, named by copies that read nothing.
template <typename S, bool ALIGNED, typename Src>
__device__ __forceinline__ void stage_rows(unsigned char *to, int rows, int t0, int lim, int i, int n, const void *any,
                                           Src src) {
    constexpr int G = kSsmTile * static_cast<int>(sizeof(S)) / 16 + (ALIGNED ? 0 : 1);
    const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    for (int k = i; k < rows * G; k += n) {
        const int row = k / G, g = k - row * G;  // G is a constant: a shift where the rows are aligned
        const S *first = src(row);
        const uint32_t dst = base + row * row_bytes<S>() + g * 16;
        const unsigned char *from = reinterpret_cast<const unsigned char *>(first + t0);
        if (!ALIGNED) from -= reinterpret_cast<uintptr_t>(from) & 15;
        from += g * 16;
        if (first && t0 + kSsmTile + 16 / static_cast<int>(sizeof(S)) <= lim) {  // wholly inside the row
            copy16(dst, from, 16);
        } else {
            const int64_t d = first ? reinterpret_cast<const unsigned char *>(first + lim) - from : 0;
            const int left = d < 0 ? 0 : d > 16 ? 16 : static_cast<int>(d);
            copy16(dst, left ? static_cast<const void *>(from) : any, left);
        }
    }
}

// The same where every granule lies inside the row (tile_inside): lane `i` of `n` keeps one granule of every
// n / G-th row, so its addresses advance by constants, and the last one of a row that does not start on a
// boundary also copies the one behind.  `from`: its granule of row i / G.
template <typename S>
constexpr int granules = kSsmTile * static_cast<int>(sizeof(S)) / 16;
template <typename S, bool ALIGNED>
__device__ __forceinline__ bool tile_inside(int t0, int len) {
    return t0 + kSsmTile + (ALIGNED ? 0 : 16 / static_cast<int>(sizeof(S))) <= len;
}
template <typename S, bool ALIGNED>
__device__ __forceinline__ void stage_whole(uint32_t dst, const S *from, int64_t stride, int rows, int i, int n) {
    const int step = n / granules<S>;
    const bool behind = !ALIGNED && i % granules<S> == granules<S> - 1;
    for (int r = i / granules<S>; r < rows; r += step) {
        const unsigned char *at = reinterpret_cast<const unsigned char *>(from);
        if (!ALIGNED) at -= reinterpret_cast<uintptr_t>(at) & 15;
        copy16(dst, at, 16);
        if (behind) copy16(dst + 16, at + 16, 16);
        dst += step * row_bytes<S>();
        from += step * stride;
    }
}
template <typename S>
__device__ __forceinline__ uint32_t whole_dst(const void *to, int i) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(to)) + i / granules<S> * row_bytes<S>() + i % granules<S> * 16;
}
template <typename S>
__device__ __forceinline__ const S *whole_src(const S *row, int64_t stride, int i) {
    return row + i / granules<S> * stride + i % granules<S> * (16 / static_cast<int>(sizeof(S)));
}

// Element offset of a staged row's first position inside its first granule.
template <typename S, bool ALIGNED>
__device__ __forceinline__ int row_shift(const S *first) {
    return ALIGNED ? 0 : static_cast<int>((reinterpret_cast<uintptr_t>(first) & 15) / sizeof(S));
}

// N words from the word `at` (< 4) of the 16-byte granules at `from` on.  Whole granules are read and the
// words picked: loads of single words, 16 or 32 bytes apart from lane to lane, would meet the same few banks
// (a training forward of (4,1024,4097) fp32: 442 us with them, 351 us so).
template <int N>
__device__ __forceinline__ void words_at(const unsigned char *from, int at, uint32_t (&w)[N]) {
    constexpr int G = (N + 6) / 4;
    const uint4 *q = reinterpret_cast<const uint4 *>(from);
    uint32_t v[4 * G];
#pragma unroll
    for (int k = 0; k < G; ++k) {
        const uint4 a = q[k];
        v[4 * k] = a.x, v[4 * k + 1] = a.y, v[4 * k + 2] = a.z, v[4 * k + 3] = a.w;
    }
    const bool two = at & 2, one = at & 1;
#pragma unroll
    for (int k = 0; k < N + 1; ++k) v[k] = two ? v[k + 2] : v[k];
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = one ? v[k + 1] : v[k];
}

// positions 4g ... 4g + 3 of a staged row
template <typename S, bool ALIGNED>
__device__ __forceinline__ void row_four(const unsigned char *row, int shift, int g, float (&f)[4]) {
    const S *p = reinterpret_cast<const S *>(row) + shift + 4 * g;
    if constexpr (!ALIGNED && sizeof(S) == 4) {
        uint32_t w[4];
        words_at(row + 16 * g, shift, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    } else if constexpr (!ALIGNED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = Store<S>::to_float(p[i]);
    } else if constexpr (sizeof(S) == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        const float2 a = unpack2<S>(v.x), b = unpack2<S>(v.y);
        f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
    }
}

// positions 8s ... 8s + 7 of a staged row, as 4 packed pairs
template <typename S, bool ALIGNED>
__device__ __forceinline__ void row_eight(const unsigned char *row, int shift, int s, f2 (&o)[4]) {
    const S *p = reinterpret_cast<const S *>(row) + shift + 8 * s;
    if constexpr (sizeof(S) == 4) {
        if constexpr (ALIGNED) {
            const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
            o[0] = pk(a.x, a.y), o[1] = pk(a.z, a.w), o[2] = pk(b.x, b.y), o[3] = pk(b.z, b.w);
        } else {
            uint32_t w[8];
            words_at(row + 32 * s, shift, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = pk(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
        }
    } else {
        uint32_t w[4];
        if constexpr (ALIGNED) {
            const uint4 a = *reinterpret_cast<const uint4 *>(p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {  // five of the six words around the eight halfwords, shifted by one halfword where they start
                  // odd; in 8-byte loads, which meet fewer banks twice than words do ((3,768,16386): 736 -> 692 us)
            const uint2 *q = reinterpret_cast<const uint2 *>(row + 16 * s + (shift >> 2) * 8);
            const uint2 a = q[0], b = q[1], c = q[2];
            const bool one = shift & 2;
            const uint32_t v[5] = {one ? a.y : a.x, one ? b.x : a.y, one ? b.y : b.x, one ? c.x : b.y, one ? c.y : c.x};
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(v[k], v[k + 1], (shift & 1) * 16);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = unpack2<S>(w[k]);
            o[k] = pk(f.x, f.y);
        }
    }
}

// A tile's 64 floats in shared memory: time lane s keeps positions 8s ... 8s+3 at [4s] and the other
// four at [32 + 4s], so that 8 time lanes read or write 128 contiguous bytes.
__device__ __forceinline__ float4 &tile_four(float *base, int g) {  // positions 4g ... 4g + 3
    return *reinterpret_cast<float4 *>(base + (g & 1) * 32 + (g >> 1) * 4);
}
__device__ __forceinline__ void tile_put(float *base, int g, const float (&f)[4]) { tile_four(base, g) = make_float4(f[0], f[1], f[2], f[3]); }
__device__ __forceinline__ void tile_take(float *base, int g, float (&f)[4]) {
    const float4 v = tile_four(base, g);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
}
__device__ __forceinline__ void tile_get(const float *base, int s, f2 (&f)[4]) {
    const float4 p = *reinterpret_cast<const float4 *>(base + 4 * s);
    const float4 q = *reinterpret_cast<const float4 *>(base + 32 + 4 * s);
    f[0] = pk(p.x, p.y), f[1] = pk(p.z, p.w), f[2] = pk(q.x, q.y), f[3] = pk(q.z, q.w);
}

// the same, every value twice in a pair
__device__ __forceinline__ void tile_get_twice(const float *base, int s, f2 (&f)[8]) {
    const float4 p = *reinterpret_cast<const float4 *>(base + 4 * s);
    const float4 q = *reinterpret_cast<const float4 *>(base + 32 + 4 * s);
    f[0] = pk(p.x, p.x), f[1] = pk(p.y, p.y), f[2] = pk(p.z, p.z), f[3] = pk(p.w, p.w);
    f[4] = pk(q.x, q.x), f[5] = pk(q.y, q.y), f[6] = pk(q.z, q.z), f[7] = pk(q.w, q.w);
}
// two rows of 8 positions as 8 pairs (first row, second row)
__device__ __forceinline__ void zip8(const f2 (&a)[4], const f2 (&b)[4], f2 (&o)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[2 * k] = pk(lo(a[k]), lo(b[k])), o[2 * k + 1] = pk(hi(a[k]), hi(b[k]));
}

// Sum of v over the 4 state lanes, spread so that each of them keeps two positions: state lane q gets
// positions 4 * (q & 1) + 2 * (q >> 1) and the next.  `fresh`: the pair replaces what the tile holds.
__device__ __forceinline__ void tile_sum(float *base, int s, int q, const f2 (&v)[4], bool fresh) {
    const bool up = q & 1, up2 = q >> 1;
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = i & 1 ? hi(v[i >> 1]) : lo(v[i >> 1]), b = i & 1 ? hi(v[2 + (i >> 1)]) : lo(v[2 + (i >> 1)]);
        r[i] = (up ? b : a) + __shfl_xor_sync(kFullMask, up ? a : b, 8);
    }
    float2 o;
    o.x = (up2 ? r[2] : r[0]) + __shfl_xor_sync(kFullMask, up2 ? r[0] : r[2], 16);
    o.y = (up2 ? r[3] : r[1]) + __shfl_xor_sync(kFullMask, up2 ? r[1] : r[3], 16);
    float2 *at = reinterpret_cast<float2 *>(base + (up ? 32 : 0) + 4 * s + (up2 ? 2 : 0));
    if (!fresh) {
        const float2 old = *at;
        o.x += old.x;
        o.y += old.y;
    }
    *at = o;
}

// Inclusive scans of M pairs (P, S) over the 8 time lanes, towards higher or lower lanes, side by side;
// `carry` enters the first lane.  in: the state that enters the lane; S becomes the one that leaves it.
template <bool UP, int M>
__device__ __forceinline__ void lane_scan(const float (&P0)[M], float (&S)[M], const float (&carry)[M], float (&in)[M], int s) {
    const int r = UP ? s : 7 - s;
    float P[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        P[m] = P0[m];
        if (r == 0) S[m] = fmaf(P[m], carry[m], S[m]);
    }
#pragma unroll
    for (int k = 1; k < 8; k *= 2) {
        float Sp[M], Pp[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            Sp[m] = UP ? __shfl_up_sync(kFullMask, S[m], k, 8) : __shfl_down_sync(kFullMask, S[m], k, 8);
            if (k < 4) Pp[m] = UP ? __shfl_up_sync(kFullMask, P[m], k, 8) : __shfl_down_sync(kFullMask, P[m], k, 8);
        }
#pragma unroll
        for (int m = 0; m < M; ++m)
            if (r >= k) {
                S[m] = fmaf(P[m], Sp[m], S[m]);
                if (k < 4) P[m] *= Pp[m];
            }
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
        const float v = UP ? __shfl_up_sync(kFullMask, S[m], 1, 8) : __shfl_down_sync(kFullMask, S[m], 1, 8);
        in[m] = r == 0 ? carry[m] : v;
    }
}
// The same for two states at once, packed.
template <bool UP>
__device__ __forceinline__ f2 lane_move(f2 v, int k) {
    return UP ? pk(__shfl_up_sync(kFullMask, lo(v), k, 8), __shfl_up_sync(kFullMask, hi(v), k, 8))
              : pk(__shfl_down_sync(kFullMask, lo(v), k, 8), __shfl_down_sync(kFullMask, hi(v), k, 8));
}
// M scans side by side: P, S as in lane_scan; carry[k][j] goes in, and the state after all lanes' positions
// comes out in the last lane's; in[k] is the state that enters the lane.
template <int M>
struct Count {
    static constexpr int value = M;
};
template <bool UP, int M>
__device__ __forceinline__ void lane_scan2(f2 (&P)[M], f2 (&S)[M], f2 (&carry)[M][2], int j, f2 (&in)[M], int s) {
    const int r = UP ? s : 7 - s;
#pragma unroll
    for (int k = 0; k < M; ++k)
        if (r == 0) S[k] = fma2(P[k], carry[k][j], S[k]);
#pragma unroll
    for (int d = 1; d < 8; d *= 2) {
        f2 Sp[M], Pp[M];
#pragma unroll
        for (int k = 0; k < M; ++k) {
            Sp[k] = lane_move<UP>(S[k], d);
            if (d < 4) Pp[k] = lane_move<UP>(P[k], d);
        }
#pragma unroll
        for (int k = 0; k < M; ++k)
            if (r >= d) {
                S[k] = fma2(P[k], Sp[k], S[k]);
                if (d < 4) P[k] = mul2(P[k], Pp[k]);
            }
    }
#pragma unroll
    for (int k = 0; k < M; ++k) {
        const f2 v = lane_move<UP>(S[k], 1);
        in[k] = r == 0 ? carry[k][j] : v;
        carry[k][j] = S[k];
    }
}

// Which channels a warp has: [c0, c0 + nc) of group g of sequence b; nc may be <= 0.
struct SsmPlace {
    int64_t b, d0;  // sequence; first channel counted over all groups
    int g, chunk, nc;
    int seg, first, last;  // piece of time: tiles [first, last)
};
template <typename S>
__device__ __forceinline__ SsmPlace ssm_place(const SsmProblem<S> &p, int warps) {
    SsmPlace w;
    int64_t k = blockIdx.x;
    w.seg = static_cast<int>(k % p.segs);
    k /= p.segs;
    w.first = w.seg * p.seg_tiles;
    w.last = min(p.tiles, w.first + p.seg_tiles);
    w.chunk = static_cast<int>(k % p.chunks);
    k /= p.chunks;
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

// Zeros at the positions of t ... t + 3 that are not below `len`.
__device__ __forceinline__ void cut_four(float (&f)[4], int t, int len) {
    if (t + 4 > len) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (t + i >= len) f[i] = 0.f;
    }
}

// Time steps of four raw values; positions behind the sequence get 0, which makes them identity steps.
__device__ __forceinline__ void time_steps(float (&f)[4], float bias, int softplus, int t, int len) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] += bias;
        if (softplus) f[i] = softplus_f(f[i]);
    }
    cut_four(f, t, len);
}

// Positions t ... t + 3 of an output row, those below T only.
template <typename S, bool ALIGNED>
__device__ __forceinline__ void store_four(S *__restrict__ row, int t, int T, const float (&f)[4]) {
    if (ALIGNED && t + 4 <= T) {
        if constexpr (sizeof(S) == 4) {
            *reinterpret_cast<float4 *>(row + t) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
            union {
                S h[4];
                uint2 w;
            } v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v.h[i] = from_float<S>(f[i]);
            *reinterpret_cast<uint2 *>(row + t) = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (t + i < T) row[t + i] = from_float<S>(f[i]);
    }
}

// `count` floats, copied by the lanes of a warp between rows of NP floats in shared memory and rows of N in
// global memory (N == NP: one run of whole vectors).
__device__ __forceinline__ void states_out(float *__restrict__ to, const float *from, int rows, int N, int NP, int lane) {
    if (N == NP && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
        for (int i = lane; i < rows * N / 4; i += 32) reinterpret_cast<float4 *>(to)[i] = reinterpret_cast<const float4 *>(from)[i];
    } else {
        for (int c = 0; c < rows; ++c)
            for (int n = lane; n < N; n += 32) to[static_cast<int64_t>(c) * N + n] = from[c * NP + n];
    }
}

// bytes of shared memory: B and C of a CTA; the rest of a warp, forward and backward
template <typename S>
inline __host__ __device__ size_t ssm_bc_bytes() { return kSsmStages * 2 * kSsmNB * row_bytes<S>(); }
template <typename S>
inline __host__ __device__ size_t ssm_fwd_warp_bytes(int cw, int NP) {
    return cw * (2 * 3 * row_bytes<S>() + sizeof(float) * (3 * kSsmTile + 2 * NP + 4));
}
template <typename S>
inline __host__ __device__ size_t ssm_bwd_warp_bytes(int cw, int NP) {
    return cw * (kSsmStages * (4 * row_bytes<S>() + sizeof(float) * NP) + sizeof(float) * (6 * kSsmTile + 3 * NP + 36));
}

// Position in the walk of (tile, block of states) steps, and the places of its copies in their rings.
struct SsmWalk {
    int tile, nb, slot, row_slot;
    __device__ __forceinline__ void next(int blocks, int dir) {
        slot ^= 1;
        if (++nb == blocks) {
            nb = 0;
            tile += dir;
            row_slot ^= 1;
        }
    }
};

template <typename S, bool ALIGNED>
__global__ void __launch_bounds__(kSsmFwdWarps * 32, 2)
ssm_forward_kernel(const SsmProblem<S> p, const float *__restrict__ carries, S *__restrict__ out,
                   float *__restrict__ h_last, float *__restrict__ checkpoints) {
    extern __shared__ __align__(16) unsigned char ssm_smem[];
    constexpr int RB = row_bytes<S>();
    const int lane = threadIdx.x & 31, s = lane & 7, q = lane >> 3;
    const SsmPlace w = ssm_place(p, kSsmFwdWarps);
    unsigned char *raw = ssm_smem + ssm_bc_bytes<S>() + (threadIdx.x >> 5) * ssm_fwd_warp_bytes<S>(p.cw, p.NP);
    float *dt_ = reinterpret_cast<float *>(raw + 2 * 3 * p.cw * RB);
    float *u_ = dt_ + p.cw * kSsmTile, *y_ = u_ + p.cw * kSsmTile;
    float *h_ = y_ + p.cw * kSsmTile, *A_ = h_ + p.cw * p.NP, *bias_ = A_ + p.cw * p.NP, *D_ = bias_ + p.cw;
    const int len = ssm_length(p, w.b);
    const int64_t row0 = w.b * p.channels + w.d0;
    const S *xrow = p.x + w.b * p.xs[0] + w.d0 * p.xs[1], *drow = p.delta + w.b * p.ds[0] + w.d0 * p.ds[1];
    const S *zrow = p.z ? p.z + w.b * p.zs[0] + w.d0 * p.zs[1] : nullptr;
    const S *Brow = p.B + w.b * p.Bs[0] + w.g * p.Bs[1], *Crow = p.C + w.b * p.Cs[0] + w.g * p.Cs[1];

    for (int c = 0; c < w.nc; ++c)
        for (int n = lane; n < p.NP; n += 32) {
            A_[c * p.NP + n] = n < p.N ? p.A[(w.d0 + c) * p.N + n] * kLog2e : 0.f;
            // a piece of time starts from the state that the pieces before it leave
            const float *h0 = carries ? carries + ((w.b * p.segs + w.seg) * p.channels + w.d0) * p.N
                                      : p.h0 ? p.h0 + row0 * p.N : nullptr;
            h_[c * p.NP + n] = n < p.N && h0 ? h0[c * p.N + n] : 0.f;
        }
    if (lane < w.nc) {  // at most 8 channels
        bias_[lane] = p.bias ? p.bias[w.d0 + lane] : 0.f;
        D_[lane] = p.D ? p.D[w.d0 + lane] : 0.f;
    }

    const int blocks = p.NP / kSsmNB, live_tiles = min(w.last, (len + kSsmTile - 1) / kSsmTile);
    const void *any = reinterpret_cast<const void *>(reinterpret_cast<uintptr_t>(p.x) & ~uintptr_t{15});
    const S *xw = whole_src(xrow, p.xs[1], lane), *dw = whole_src(drow, p.ds[1], lane);
    const S *zw = p.z ? whole_src(zrow, p.zs[1], lane) : nullptr;
    const S *Bw = whole_src(Brow, p.Bs[2], threadIdx.x), *Cw = whole_src(Crow, p.Cs[2], threadIdx.x);
    auto stage = [&](int tile, int nb, int step) {
        const int t0 = tile * kSsmTile;
        unsigned char *bc = ssm_smem + (step & 1) * (2 * kSsmNB * RB), *to = raw + (tile & 1) * (3 * p.cw * RB);
        if (ALIGNED && tile_inside<S, ALIGNED>(t0, len)) {  // unaligned rows too: 50 -> 54 us at (3,768,1001) fp16
            constexpr int n = kSsmFwdWarps * 32;
            if ((nb + 1) * kSsmNB <= p.N) {
                stage_whole<S, ALIGNED>(whole_dst<S>(bc, threadIdx.x), Bw + nb * kSsmNB * p.Bs[2] + t0, p.Bs[2], kSsmNB, threadIdx.x, n);
                stage_whole<S, ALIGNED>(whole_dst<S>(bc + kSsmNB * RB, threadIdx.x), Cw + nb * kSsmNB * p.Cs[2] + t0, p.Cs[2], kSsmNB, threadIdx.x, n);
            }
            if (nb == 0) {
                stage_whole<S, ALIGNED>(whole_dst<S>(to, lane), xw + t0, p.xs[1], w.nc, lane, 32);
                stage_whole<S, ALIGNED>(whole_dst<S>(to + p.cw * RB, lane), dw + t0, p.ds[1], w.nc, lane, 32);
                if (p.z) stage_whole<S, ALIGNED>(whole_dst<S>(to + 2 * p.cw * RB, lane), zw + t0, p.zs[1], w.nc, lane, 32);
            }
        } else if (nb == 0) {
            stage_rows<S, ALIGNED>(to, w.nc, t0, len, lane, 32, any, [&](int c) { return xrow + c * p.xs[1]; });
            stage_rows<S, ALIGNED>(to + p.cw * RB, w.nc, t0, len, lane, 32, any, [&](int c) { return drow + c * p.ds[1]; });
            if (p.z)
                stage_rows<S, ALIGNED>(to + 2 * p.cw * RB, w.nc, t0, len, lane, 32, any, [&](int c) { return zrow + c * p.zs[1]; });
        }
        if (!ALIGNED || !tile_inside<S, ALIGNED>(t0, len) || (nb + 1) * kSsmNB > p.N)
            stage_rows<S, ALIGNED>(bc, 2 * kSsmNB, t0, len, threadIdx.x, kSsmFwdWarps * 32, any, [&](int r) -> const S * {
                const int n = nb * kSsmNB + (r & (kSsmNB - 1));
                return n >= p.N ? nullptr : r < kSsmNB ? Brow + n * p.Bs[2] : Crow + n * p.Cs[2];
            });
        copies_commit();
    };
    if (live_tiles > w.first) stage(w.first, 0, 0);

    for (int tile = w.first, step = 0; tile < live_tiles; ++tile) {
        const int g = lane & 15, t = tile * kSsmTile + 4 * g;  // outside the state loop a lane has four positions of a channel
        const unsigned char *mine = raw + (tile & 1) * (3 * p.cw * RB);
        for (int nb = 0; nb < blocks; ++nb, ++step) {
            copies_wait<0>();
            __syncthreads();
            if (nb + 1 < blocks) stage(tile, nb + 1, step + 1);
            else if (tile + 1 < live_tiles) stage(tile + 1, 0, step + 1);
            const unsigned char *bc = ssm_smem + (step & 1) * (2 * kSsmNB * RB);
            if (nb == 0) {
                for (int c = lane >> 4; c < w.nc; c += 2) {
                    float x[4], dt[4];
                    row_four<S, ALIGNED>(mine + c * RB, row_shift<S, ALIGNED>(xrow + c * p.xs[1]), g, x);
                    row_four<S, ALIGNED>(mine + (p.cw + c) * RB, row_shift<S, ALIGNED>(drow + c * p.ds[1]), g, dt);
                    time_steps(dt, bias_[c], p.softplus, t, len);
                    tile_put(dt_ + c * kSsmTile, g, dt);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] *= dt[i];
                    tile_put(u_ + c * kSsmTile, g, x);
                }
                if (checkpoints)
                    states_out(checkpoints + ((w.b * p.tiles + tile) * p.channels + w.d0) * p.N, h_, w.nc, p.N, p.NP, lane);
                __syncwarp();
            }
            const int n0 = nb * kSsmNB + q * kSsmNL;
            f2 B[2][8], C[2][8];  // [pair of states][position]
            {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = q * kSsmNL + 2 * j, n = n0 + 2 * j;
                    f2 e[4], o[4];
                    row_eight<S, ALIGNED>(bc + r * RB, row_shift<S, ALIGNED>(Brow + n * p.Bs[2]), s, e);
                    row_eight<S, ALIGNED>(bc + (r + 1) * RB, row_shift<S, ALIGNED>(Brow + (n + 1) * p.Bs[2]), s, o);
                    zip8(e, o, B[j]);
                    row_eight<S, ALIGNED>(bc + (kSsmNB + r) * RB, row_shift<S, ALIGNED>(Crow + n * p.Cs[2]), s, e);
                    row_eight<S, ALIGNED>(bc + (kSsmNB + r + 1) * RB, row_shift<S, ALIGNED>(Crow + (n + 1) * p.Cs[2]), s, o);
                    zip8(e, o, C[j]);
                }
            }
            // M channels side by side, whose chains of multiply-adds and shuffles overlap: 385 -> 330 us for a prompt of
            // (1,2048,8192) bf16, although at 255 registers only 8 warps fit an SM instead of 12
            auto channels = [&](int c, auto m) {
                constexpr int M = decltype(m)::value;
                f2 dt[M][8], u[M][8], Av[M][2], hv[M][2], span[M];
                float y[M][8];
#pragma unroll
                for (int k = 0; k < M; ++k) {
                    tile_get_twice(dt_ + (c + k) * kSsmTile, s, dt[k]);
                    tile_get_twice(u_ + (c + k) * kSsmTile, s, u[k]);
                    const float4 A4 = *reinterpret_cast<const float4 *>(A_ + (c + k) * p.NP + n0);
                    const float4 h4 = *reinterpret_cast<const float4 *>(h_ + (c + k) * p.NP + n0);
                    Av[k][0] = pk(A4.x, A4.y), Av[k][1] = pk(A4.z, A4.w);
                    hv[k][0] = pk(h4.x, h4.y), hv[k][1] = pk(h4.z, h4.w);
                    span[k] = add2(add2(add2(dt[k][0], dt[k][1]), add2(dt[k][2], dt[k][3])),
                                   add2(add2(dt[k][4], dt[k][5]), add2(dt[k][6], dt[k][7])));
                }
                __syncwarp();  // the carries are read before the last time lane replaces them
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    f2 a[M][8], b[M][8], P[M], S0[M], h[M];
#pragma unroll
                    for (int k = 0; k < M; ++k) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const f2 e = mul2(dt[k][i], Av[k][j]);
                            a[k][i] = pk(ex2(lo(e)), ex2(hi(e)));
                            b[k][i] = mul2(u[k][i], B[j][i]);
                        }
                        const f2 e = mul2(span[k], Av[k][j]);
                        P[k] = pk(ex2(lo(e)), ex2(hi(e)));
                        S0[k] = b[k][0];
                    }
#pragma unroll
                    for (int i = 1; i < 8; ++i)
#pragma unroll
                        for (int k = 0; k < M; ++k) S0[k] = fma2(a[k][i], S0[k], b[k][i]);
                    lane_scan2<true, M>(P, S0, hv, j, h, s);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int k = 0; k < M; ++k) {
                            h[k] = fma2(a[k][i], h[k], b[k][i]);
                            y[k][i] = j ? fmaf(lo(C[j][i]), lo(h[k]), y[k][i]) : lo(C[j][i]) * lo(h[k]);
                            y[k][i] = fmaf(hi(C[j][i]), hi(h[k]), y[k][i]);
                        }
                }
#pragma unroll
                for (int k = 0; k < M; ++k) {
                    if (s == 7)
                        *reinterpret_cast<float4 *>(h_ + (c + k) * p.NP + n0) =
                            make_float4(lo(hv[k][0]), hi(hv[k][0]), lo(hv[k][1]), hi(hv[k][1]));
                    const f2 sum[4] = {pk(y[k][0], y[k][1]), pk(y[k][2], y[k][3]), pk(y[k][4], y[k][5]), pk(y[k][6], y[k][7])};
                    tile_sum(y_ + (c + k) * kSsmTile, s, q, sum, nb == 0);
                }
            };
            int c = 0;
            for (; c + 1 < w.nc; c += 2) channels(c, Count<2>{});
            if (c < w.nc) channels(c, Count<1>{});
        }
        __syncwarp();
        for (int c = lane >> 4; c < w.nc; c += 2) {
            float y[4], v[4];
            tile_take(y_ + c * kSsmTile, g, y);
            if (p.D) {
                row_four<S, ALIGNED>(mine + c * RB, row_shift<S, ALIGNED>(xrow + c * p.xs[1]), g, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = fmaf(D_[c], v[i], y[i]);
            }
            if (p.z) {
                row_four<S, ALIGNED>(mine + (2 * p.cw + c) * RB, row_shift<S, ALIGNED>(zrow + c * p.zs[1]), g, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] *= v[i] * sigmoid_f(v[i]);
            }
            cut_four(y, t, len);
            store_four<S, ALIGNED>(out + (row0 + c) * p.T, t, p.T, y);
        }
    }
    __syncwarp();
    const float zero[4] = {};
    for (int tile = max(w.first, live_tiles); tile < w.last; ++tile)  // behind the sequence: zeros
        for (int c = lane >> 4; c < w.nc; c += 2)
            store_four<S, ALIGNED>(out + (row0 + c) * p.T, tile * kSsmTile + 4 * (lane & 15), p.T, zero);
    if (h_last && w.nc > 0 && w.seg == p.segs - 1) states_out(h_last + row0 * p.N, h_, w.nc, p.N, p.NP, lane);
}

// What the backward writes; the partial sums live in the caller's workspace.
template <typename S>
struct SsmGrads {
    const float *checkpoints;
    const S *grad_out;
    const float *grad_last, *carries;
    S *dx, *ddelta, *dz;
    float *dh0;
    float *bc_part;  // [batch][group][chunk][B | C][N][tiles * 64]
    float *a_part;   // [batch][segment][D][N]
    float *d_part;   // [batch][segment][2][D]: grad of D, grad of delta_bias
};

// With e_t = C_t dy_t:  c_t = a_t (e_t + c_{t+1}) is what reaches the state before t, g_t = e_t + c_{t+1},
// q_t = c_t h_{t-1};
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
    extern __shared__ __align__(16) unsigned char ssm_smem[];
    constexpr int W = kSsmBwdWarps, RB = row_bytes<S>(), NL = 2;  // states of a lane, side by side
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, s = lane & 7, q = lane >> 3;
    const SsmPlace w = ssm_place(p, W);
    float *red = reinterpret_cast<float *>(ssm_smem + ssm_bc_bytes<S>());  // [2][warp][32][lane]
    unsigned char *raw = reinterpret_cast<unsigned char *>(red + W * 64 * 32) + warp * ssm_bwd_warp_bytes<S>(p.cw, p.NP);
    const int ct = p.cw * kSsmTile, cn = p.cw * p.NP;
    float *ck_ = reinterpret_cast<float *>(raw + kSsmStages * 4 * p.cw * RB), *dt_ = ck_ + kSsmStages * cn;
    float *u_ = dt_ + ct, *dy_ = u_ + ct, *gB_ = dy_ + ct, *q_ = gB_ + ct, *y_ = q_ + ct;
    float *A_ = y_ + ct, *c_ = A_ + cn, *dA_ = c_ + cn, *dD_ = dA_ + cn, *bias_ = dD_ + 32 * p.cw, *D_ = bias_ + p.cw;
    const int len = ssm_length(p, w.b);
    const int64_t row0 = w.b * p.channels + w.d0;
    const int Tpad = p.tiles * kSsmTile;
    float *bc_out = o.bc_part + ((w.b * p.groups + w.g) * p.chunks + w.chunk) * 2 * p.N * static_cast<int64_t>(Tpad);
    const S *xrow = p.x + w.b * p.xs[0] + w.d0 * p.xs[1], *drow = p.delta + w.b * p.ds[0] + w.d0 * p.ds[1];
    const S *zrow = GATED ? p.z + w.b * p.zs[0] + w.d0 * p.zs[1] : nullptr, *grow = o.grad_out + row0 * p.T;
    const S *Brow = p.B + w.b * p.Bs[0] + w.g * p.Bs[1], *Crow = p.C + w.b * p.Cs[0] + w.g * p.Cs[1];

    for (int c = 0; c < w.nc; ++c) {
        for (int n = lane; n < p.NP; n += 32) {
            const int i = c * p.NP + n;
            A_[i] = n < p.N ? p.A[(w.d0 + c) * p.N + n] * kLog2e : 0.f;
            const float *c0 = o.carries ? o.carries + ((w.b * p.segs + w.seg) * p.channels + w.d0) * p.N
                                        : o.grad_last ? o.grad_last + row0 * p.N : nullptr;
            c_[i] = n < p.N && c0 ? c0[c * p.N + n] : 0.f;
            for (int k = 0; k < kSsmStages; ++k) ck_[k * cn + i] = 0.f;
            dA_[i] = 0.f;
        }
        dD_[c * 32 + lane] = 0.f;
        if (lane == 0) {
            bias_[c] = p.bias ? p.bias[w.d0 + c] : 0.f;
            D_[c] = p.D ? p.D[w.d0 + c] : 0.f;
        }
    }

    const int blocks = p.NP / kSsmNB, live_tiles = min(w.last, (len + kSsmTile - 1) / kSsmTile);
    const void *any = reinterpret_cast<const void *>(reinterpret_cast<uintptr_t>(p.x) & ~uintptr_t{15});
    const int64_t T = p.T;
    const S *xw = whole_src(xrow, p.xs[1], lane), *dw = whole_src(drow, p.ds[1], lane), *gw = whole_src(grow, T, lane);
    const S *zw = GATED ? whole_src(zrow, p.zs[1], lane) : nullptr;
    const S *Bw = whole_src(Brow, p.Bs[2], threadIdx.x), *Cw = whole_src(Crow, p.Cs[2], threadIdx.x);
    SsmWalk ahead{live_tiles - 1, 0, 0, 0}, at = ahead;
    const bool ck_whole = p.N == p.NP && (reinterpret_cast<uintptr_t>(o.checkpoints) & 15) == 0;
    auto stage = [&]() {  // the copies of the next step; past the end an empty group, which keeps the count
        if (ahead.tile < w.first) {
            copies_commit();
            return;
        }
        const int nb = ahead.nb, t0 = ahead.tile * kSsmTile;
        unsigned char *bc = ssm_smem + ahead.slot * (2 * kSsmNB * RB), *to = raw + ahead.row_slot * (4 * p.cw * RB);
        if (nb == 0) {  // the states in front of the tile
            const float *ck = o.checkpoints + ((w.b * p.tiles + ahead.tile) * p.channels + w.d0) * p.N;
            const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(ck_ + ahead.row_slot * cn));
            if (ck_whole) {
                for (int i = lane; i < w.nc * p.N / 4; i += 32) copy16(dst + i * 16, ck + i * 4, 16);
            } else {
                for (int c = 0; c < w.nc; ++c)
                    for (int n = lane; n < p.N; n += 32) copy4(dst + (c * p.NP + n) * 4, ck + c * p.N + n);
            }
        }
        if (tile_inside<S, ALIGNED>(t0, len)) {
            constexpr int n = W * 32;
            if ((nb + 1) * kSsmNB <= p.N) {
                stage_whole<S, ALIGNED>(whole_dst<S>(bc, threadIdx.x), Bw + nb * kSsmNB * p.Bs[2] + t0, p.Bs[2], kSsmNB, threadIdx.x, n);
                stage_whole<S, ALIGNED>(whole_dst<S>(bc + kSsmNB * RB, threadIdx.x), Cw + nb * kSsmNB * p.Cs[2] + t0, p.Cs[2], kSsmNB, threadIdx.x, n);
            }
            if (nb == 0) {
                stage_whole<S, ALIGNED>(whole_dst<S>(to, lane), xw + t0, p.xs[1], w.nc, lane, 32);
                stage_whole<S, ALIGNED>(whole_dst<S>(to + p.cw * RB, lane), dw + t0, p.ds[1], w.nc, lane, 32);
                stage_whole<S, ALIGNED>(whole_dst<S>(to + 2 * p.cw * RB, lane), gw + t0, T, w.nc, lane, 32);
                if (GATED) stage_whole<S, ALIGNED>(whole_dst<S>(to + 3 * p.cw * RB, lane), zw + t0, p.zs[1], w.nc, lane, 32);
            }
        } else if (nb == 0) {
            stage_rows<S, ALIGNED>(to, w.nc, t0, len, lane, 32, any, [&](int c) { return xrow + c * p.xs[1]; });
            stage_rows<S, ALIGNED>(to + p.cw * RB, w.nc, t0, len, lane, 32, any, [&](int c) { return drow + c * p.ds[1]; });
            stage_rows<S, ALIGNED>(to + 2 * p.cw * RB, w.nc, t0, len, lane, 32, any, [&](int c) { return grow + c * T; });
            if (GATED)
                stage_rows<S, ALIGNED>(to + 3 * p.cw * RB, w.nc, t0, len, lane, 32, any, [&](int c) { return zrow + c * p.zs[1]; });
        }
        if (!tile_inside<S, ALIGNED>(t0, len) || (nb + 1) * kSsmNB > p.N)
            stage_rows<S, ALIGNED>(bc, 2 * kSsmNB, t0, len, threadIdx.x, W * 32, any, [&](int r) -> const S * {
                const int n = nb * kSsmNB + (r & (kSsmNB - 1));
                return n >= p.N ? nullptr : r < kSsmNB ? Brow + n * p.Bs[2] : Crow + n * p.Cs[2];
            });
        copies_commit();
        ahead.next(blocks, -1);
    };
    const int g4 = lane & 15;  // outside the state loop a lane has four positions of a channel
    auto row_at = [&](const unsigned char *mine, int kind, int c, float (&f)[4]) {
        const S *first = kind == 0   ? xrow + c * p.xs[1]
                         : kind == 1 ? drow + c * p.ds[1]
                         : kind == 2 ? grow + c * T
                                     : zrow + c * p.zs[1];
        row_four<S, ALIGNED>(mine + (kind * p.cw + c) * RB, row_shift<S, ALIGNED>(first), g4, f);
    };

    for (int tile = max(w.first, live_tiles); tile < w.last; ++tile) {  // behind the sequence: zeros
        const int t = tile * kSsmTile + 4 * g4;
        const float zero[4] = {};
        for (int c = lane >> 4; c < w.nc; c += 2) {
            store_four<S, ALIGNED>(o.dx + (row0 + c) * T, t, p.T, zero);
            store_four<S, ALIGNED>(o.ddelta + (row0 + c) * T, t, p.T, zero);
            if (GATED) store_four<S, ALIGNED>(o.dz + (row0 + c) * T, t, p.T, zero);
        }
        for (int i = threadIdx.x; i < 2 * p.N * kSsmTile; i += W * 32)
            bc_out[static_cast<int64_t>(i / kSsmTile) * Tpad + tile * kSsmTile + i % kSsmTile] = 0.f;
    }
    __syncwarp();  // the states' places are cleared
    for (int k = 1; k < kSsmStages; ++k) stage();

    for (int tile = live_tiles - 1; tile >= w.first; --tile) {
        const int t = tile * kSsmTile + 4 * g4;
        const unsigned char *mine = raw + at.row_slot * (4 * p.cw * RB);
        const float *h_ = ck_ + at.row_slot * cn;
        for (int nb = 0; nb < blocks; ++nb) {
            copies_wait<0>();
            __syncthreads();
            stage();
            const unsigned char *bc = ssm_smem + at.slot * (2 * kSsmNB * RB);
            at.next(blocks, -1);
            if (nb == 0) {
                for (int c = lane >> 4; c < w.nc; c += 2) {
                    float x[4], dt[4], dy[4];
                    row_at(mine, 0, c, x);
                    row_at(mine, 1, c, dt);
                    row_at(mine, 2, c, dy);
                    if (GATED) {
                        float z[4];
                        row_at(mine, 3, c, z);
#pragma unroll
                        for (int i = 0; i < 4; ++i) dy[i] *= z[i] * sigmoid_f(z[i]);
                    }
                    time_steps(dt, bias_[c], p.softplus, t, len);
                    tile_put(dt_ + c * kSsmTile, g4, dt);
                    tile_put(dy_ + c * kSsmTile, g4, dy);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] *= dt[i];
                    tile_put(u_ + c * kSsmTile, g4, x);
                }
                __syncwarp();
            }
            for (int sub = 0; sub < kSsmNB && nb * kSsmNB + sub < p.N; sub += 4 * NL) {  // 8 states at a time
                const int n0 = nb * kSsmNB + sub + q * NL;
                const bool fresh = nb == 0 && sub == 0;
                f2 B[NL][4], C[NL][4], dB[NL][4], dC[NL][4];
#pragma unroll
                for (int j = 0; j < NL; ++j) {
                    const int r = sub + q * NL + j;
                    row_eight<S, ALIGNED>(bc + r * RB, row_shift<S, ALIGNED>(Brow + (n0 + j) * p.Bs[2]), s, B[j]);
                    row_eight<S, ALIGNED>(bc + (kSsmNB + r) * RB, row_shift<S, ALIGNED>(Crow + (n0 + j) * p.Cs[2]), s, C[j]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) dB[j][k] = dC[j][k] = 0;
                }
                for (int c = 0; c < w.nc; ++c) {
                    f2 dt[4], u[4], dy[4], gB[4], Q[4], y[4];
                    float dA[NL];
                    tile_get(dt_ + c * kSsmTile, s, dt);
                    tile_get(u_ + c * kSsmTile, s, u);
                    tile_get(dy_ + c * kSsmTile, s, dy);
                    const f2 both = add2(add2(dt[0], dt[1]), add2(dt[2], dt[3]));
                    const float sum = lo(both) + hi(both);
                    const int at = c * p.NP + n0;
                    const float2 A2 = *reinterpret_cast<const float2 *>(A_ + at), h2 = *reinterpret_cast<const float2 *>(h_ + at);
                    const float2 c2 = *reinterpret_cast<const float2 *>(c_ + at);
                    __syncwarp();  // the carries are read before the first time lane replaces them
                    const float Av[NL] = {A2.x, A2.y}, hv[NL] = {h2.x, h2.y};
                    float cv[NL] = {c2.x, c2.y};
                    f2 a[NL][4], v[NL][4], h[NL][4], e[NL][4];
                    float P[NL], S0[NL], hin[NL], after[NL];
#pragma unroll
                    for (int k = 0; k < 4; ++k) gB[k] = Q[k] = y[k] = 0;
#pragma unroll
                    for (int j = 0; j < NL; ++j) {
                        const f2 Ad = pk(Av[j], Av[j]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const f2 x = mul2(dt[k], Ad);
                            a[j][k] = pk(ex2(lo(x)), ex2(hi(x)));
                            v[j][k] = mul2(u[k], B[j][k]);
                        }
                        P[j] = ex2(sum * Av[j]);
                        S0[j] = lo(v[j][0]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int j = 0; j < NL; ++j) {
                            if (k) S0[j] = fmaf(lo(a[j][k]), S0[j], lo(v[j][k]));
                            S0[j] = fmaf(hi(a[j][k]), S0[j], hi(v[j][k]));
                        }
                    lane_scan<true, NL>(P, S0, hv, hin, s);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int j = 0; j < NL; ++j) {
                            const float h1 = fmaf(lo(a[j][k]), k ? hi(h[j][k ? k - 1 : 0]) : hin[j], lo(v[j][k]));
                            h[j][k] = pk(h1, fmaf(hi(a[j][k]), h1, hi(v[j][k])));
                            dC[j][k] = fma2(dy[k], h[j][k], dC[j][k]);
                            if (GATED) y[k] = fma2(C[j][k], h[j][k], y[k]);
                            e[j][k] = mul2(C[j][k], dy[k]);
                            v[j][k] = mul2(a[j][k], e[j][k]);
                        }
#pragma unroll
                    for (int j = 0; j < NL; ++j) S0[j] = hi(v[j][3]);
#pragma unroll
                    for (int k = 3; k >= 0; --k)
#pragma unroll
                        for (int j = 0; j < NL; ++j) {
                            if (k < 3) S0[j] = fmaf(hi(a[j][k]), S0[j], hi(v[j][k]));
                            S0[j] = fmaf(lo(a[j][k]), S0[j], lo(v[j][k]));
                        }
                    lane_scan<false, NL>(P, S0, cv, after, s);  // c of the position behind
                    if (s == 0) *reinterpret_cast<float2 *>(c_ + at) = make_float2(S0[0], S0[1]);
                    f2 dAj[NL] = {0, 0};
#pragma unroll
                    for (int k = 3; k >= 0; --k)
#pragma unroll
                        for (int j = 0; j < NL; ++j) {
                            const float c1 = fmaf(hi(a[j][k]), after[j], hi(v[j][k])), c0 = fmaf(lo(a[j][k]), c1, lo(v[j][k]));
                            const f2 g = add2(e[j][k], pk(c1, after[j]));
                            const f2 qq = pk(c0 * (k ? hi(h[j][k ? k - 1 : 0]) : hin[j]), c1 * lo(h[j][k]));
                            after[j] = c0;
                            Q[k] = fma2(pk(Av[j], Av[j]), qq, Q[k]);
                            dAj[j] = fma2(dt[k], qq, dAj[j]);
                            gB[k] = fma2(g, B[j][k], gB[k]);
                            dB[j][k] = fma2(g, u[k], dB[j][k]);
                        }
#pragma unroll
                    for (int j = 0; j < NL; ++j) dA[j] = lo(dAj[j]) + hi(dAj[j]);
                    {  // dA over the 8 time lanes: lane s < 2 keeps state s
                        float d = ((s & 1) ? dA[1] : dA[0]) + __shfl_xor_sync(kFullMask, (s & 1) ? dA[0] : dA[1], 1);
                        d += __shfl_xor_sync(kFullMask, d, 2);
                        d += __shfl_xor_sync(kFullMask, d, 4);
                        if (s < 2) dA_[at + s] += d;
                    }
                    tile_sum(gB_ + c * kSsmTile, s, q, gB, fresh);
                    tile_sum(q_ + c * kSsmTile, s, q, Q, fresh);
                    if (GATED) tile_sum(y_ + c * kSsmTile, s, q, y, fresh);
                }
                // dB, dC over the warps of the CTA; the two halves of `red` take turns
                float *half = red + ((sub / (4 * NL)) & 1) * W * 32 * 32, *slot = half + warp * 32 * 32 + lane;
#pragma unroll
                for (int j = 0; j < NL; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        slot[(j * 8 + 2 * k) * 32] = lo(dB[j][k]);
                        slot[(j * 8 + 2 * k + 1) * 32] = hi(dB[j][k]);
                        slot[((NL + j) * 8 + 2 * k) * 32] = lo(dC[j][k]);
                        slot[((NL + j) * 8 + 2 * k + 1) * 32] = hi(dC[j][k]);
                    }
                __syncthreads();
                {
                    static_assert(W == 4 * NL, "a warp sums four positions of one state of dB or dC");
                    const int n = n0 + ((warp >> 1) & (NL - 1)), which = warp / (2 * NL);
                    float x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = 0.f;
#pragma unroll
                        for (int k = 0; k < W; ++k) x[i] += half[(k * 32 + warp * 4 + i) * 32 + lane];
                    }
                    if (n < p.N)
                        *reinterpret_cast<float4 *>(bc_out + (static_cast<int64_t>(which) * p.N + n) * Tpad + tile * kSsmTile +
                                                    s * kSsmE + 4 * (warp & 1)) = make_float4(x[0], x[1], x[2], x[3]);
                }
            }
        }

        for (int c = lane >> 4; c < w.nc; c += 2) {
            const int at = c * kSsmTile;
            float dt[4], dy[4], gB[4], Q[4], x[4], r[4], v[4], sD = 0.f, sb = 0.f;
            tile_take(dt_ + at, g4, dt);
            tile_take(dy_ + at, g4, dy);
            tile_take(gB_ + at, g4, gB);
            tile_take(q_ + at, g4, Q);
            row_at(mine, 0, c, x);
            row_at(mine, 1, c, r);
            const float D = D_[c], bias = bias_[c];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = fmaf(dt[i], gB[i], D * dy[i]);
                sD = fmaf(dy[i], x[i], sD);
            }
            cut_four(v, t, len);
            store_four<S, ALIGNED>(o.dx + (row0 + c) * T, t, p.T, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = fmaf(kLn2, Q[i], x[i] * gB[i]);
                if (p.softplus) v[i] *= sigmoid_f(r[i] + bias);
            }
            cut_four(v, t, len);
            store_four<S, ALIGNED>(o.ddelta + (row0 + c) * T, t, p.T, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) sb += v[i];
            if (GATED) {
                float z[4], up[4];
                tile_take(y_ + at, g4, v);
                row_at(mine, 3, c, z);
                row_at(mine, 2, c, up);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float sg = sigmoid_f(z[i]);
                    v[i] = up[i] * fmaf(D, x[i], v[i]) * sg * fmaf(z[i], 1.f - sg, 1.f);
                }
                cut_four(v, t, len);
                store_four<S, ALIGNED>(o.dz + (row0 + c) * T, t, p.T, v);
            }
            float2 *sums = reinterpret_cast<float2 *>(dD_) + c * 16 + g4;  // this lane's share of grad D, grad delta_bias
            *sums = make_float2(sums->x + sD, sums->y + sb);
        }
    }
    __syncwarp();
    const int64_t part = w.b * p.segs + w.seg;
    for (int c = 0; c < w.nc; ++c) {
        for (int n = lane; n < p.N; n += 32) {
            const int k = c * p.NP + n;
            o.a_part[(part * p.channels + w.d0 + c) * p.N + n] = dA_[k];
            if (o.dh0 && w.seg == 0) o.dh0[(row0 + c) * p.N + n] = c_[k];
        }
        if (lane < 2) {  // grad D, grad delta_bias: the 16 lanes' shares in order
            float v = 0.f;
            for (int i = 0; i < 16; ++i) v += dD_[(c * 16 + i) * 2 + lane];
            o.d_part[(part * 2 + lane) * p.channels + w.d0 + c] = v;
        }
    }
}

// First pass over a time that is cut into pieces: what each piece leaves to the next from a zero start.
// Forward the state h at its end, REVERSE the adjoint c at its beginning; with both the sum of its time
// steps, whose exponential is the piece's product of decays.  The second pass is the kernels above.
template <typename S>
inline __host__ __device__ size_t ssm_carry_warp_bytes(int cw, int NP) {
    return cw * (kSsmStages * 3 * row_bytes<S>() + sizeof(float) * (2 * kSsmTile + 2 * NP + 20));
}
template <typename S, bool ALIGNED, bool REVERSE>
__global__ void __launch_bounds__(kSsmFwdWarps * 32, 3)
ssm_carry_kernel(const SsmProblem<S> p, const S *__restrict__ grad_out, float *__restrict__ carries,
                 float *__restrict__ sums) {
    extern __shared__ __align__(16) unsigned char ssm_smem[];
    constexpr int RB = row_bytes<S>(), n_threads = kSsmFwdWarps * 32;
    const int lane = threadIdx.x & 31, s = lane & 7, q = lane >> 3, g = lane & 15;
    const SsmPlace w = ssm_place(p, kSsmFwdWarps);
    unsigned char *raw = ssm_smem + ssm_bc_bytes<S>() + (threadIdx.x >> 5) * ssm_carry_warp_bytes<S>(p.cw, p.NP);
    float *dt_ = reinterpret_cast<float *>(raw + kSsmStages * 3 * p.cw * RB), *u_ = dt_ + p.cw * kSsmTile;  // u_: REVERSE dy
    float *h_ = u_ + p.cw * kSsmTile, *A_ = h_ + p.cw * p.NP, *sum_ = A_ + p.cw * p.NP, *bias_ = sum_ + 16 * p.cw;
    const int len = ssm_length(p, w.b);
    const int64_t row0 = w.b * p.channels + w.d0, T = p.T;
    // rows: delta; tokens, or reverse grad_out and z.  Reverse reads C, forward B.
    const S *drow = p.delta + w.b * p.ds[0] + w.d0 * p.ds[1];
    const S *xrow = REVERSE ? grad_out + row0 * T : p.x + w.b * p.xs[0] + w.d0 * p.xs[1];
    const S *zrow = REVERSE && p.z ? p.z + w.b * p.zs[0] + w.d0 * p.zs[1] : nullptr;
    const int64_t xs = REVERSE ? T : p.xs[1], vs = REVERSE ? p.Cs[2] : p.Bs[2];
    const S *vrow = REVERSE ? p.C + w.b * p.Cs[0] + w.g * p.Cs[1] : p.B + w.b * p.Bs[0] + w.g * p.Bs[1];

    for (int c = 0; c < w.nc; ++c) {
        for (int n = lane; n < p.NP; n += 32) {
            A_[c * p.NP + n] = n < p.N ? p.A[(w.d0 + c) * p.N + n] * kLog2e : 0.f;
            h_[c * p.NP + n] = 0.f;
        }
        if (lane < 16) sum_[c * 16 + lane] = 0.f;
        if (lane == 0) bias_[c] = p.bias ? p.bias[w.d0 + c] : 0.f;
    }

    const int blocks = p.NP / kSsmNB, live_tiles = min(w.last, (len + kSsmTile - 1) / kSsmTile);
    const void *any = reinterpret_cast<const void *>(reinterpret_cast<uintptr_t>(p.x) & ~uintptr_t{15});
    const int dir = REVERSE ? -1 : 1, end = REVERSE ? w.first - 1 : max(w.first, live_tiles);
    SsmWalk ahead{REVERSE ? max(w.first, live_tiles) - 1 : w.first, 0, 0, 0}, at = ahead;
    auto stage = [&]() {  // the copies of the next step; past the end an empty group, which keeps the count
        if (ahead.tile == end) {
            copies_commit();
            return;
        }
        const int nb = ahead.nb, t0 = ahead.tile * kSsmTile;
        unsigned char *to = raw + ahead.row_slot * (3 * p.cw * RB);
        if (nb == 0) {
            stage_rows<S, ALIGNED>(to, w.nc, t0, len, lane, 32, any, [&](int c) { return drow + c * p.ds[1]; });
            stage_rows<S, ALIGNED>(to + p.cw * RB, w.nc, t0, len, lane, 32, any, [&](int c) { return xrow + c * xs; });
            if (zrow)
                stage_rows<S, ALIGNED>(to + 2 * p.cw * RB, w.nc, t0, len, lane, 32, any, [&](int c) { return zrow + c * p.zs[1]; });
        }
        stage_rows<S, ALIGNED>(ssm_smem + ahead.slot * (kSsmNB * RB), kSsmNB, t0, len, threadIdx.x, n_threads, any,
                               [&](int r) -> const S * {
                                   const int n = nb * kSsmNB + r;
                                   return n < p.N ? vrow + n * vs : nullptr;
                               });
        copies_commit();
        ahead.next(blocks, dir);
    };
    for (int k = 1; k < kSsmStages; ++k) stage();
    while (at.tile != end) {
        const int nb = at.nb, t = at.tile * kSsmTile + 4 * g;
        const unsigned char *mine = raw + at.row_slot * (3 * p.cw * RB), *bc = ssm_smem + at.slot * (kSsmNB * RB);
        copies_wait<0>();
        __syncthreads();
        stage();
        at.next(blocks, dir);
        if (nb == 0) {
            for (int c = lane >> 4; c < w.nc; c += 2) {
                float x[4], dt[4];
                row_four<S, ALIGNED>(mine + c * RB, row_shift<S, ALIGNED>(drow + c * p.ds[1]), g, dt);
                row_four<S, ALIGNED>(mine + (p.cw + c) * RB, row_shift<S, ALIGNED>(xrow + c * xs), g, x);
                time_steps(dt, bias_[c], p.softplus, t, len);
                if (REVERSE) {
                    if (zrow) {
                        float z[4];
                        row_four<S, ALIGNED>(mine + (2 * p.cw + c) * RB, row_shift<S, ALIGNED>(zrow + c * p.zs[1]), g, z);
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] *= z[k] * sigmoid_f(z[k]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] *= dt[k];
                }
                tile_put(dt_ + c * kSsmTile, g, dt);
                tile_put(u_ + c * kSsmTile, g, x);
                sum_[c * 16 + g] += (dt[0] + dt[1]) + (dt[2] + dt[3]);
            }
            __syncwarp();
        }
        const int n0 = nb * kSsmNB + q * kSsmNL;
        f2 V[2][8];
        {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = q * kSsmNL + 2 * j, n = n0 + 2 * j;
                f2 e[4], o[4];
                row_eight<S, ALIGNED>(bc + r * RB, row_shift<S, ALIGNED>(vrow + n * vs), s, e);
                row_eight<S, ALIGNED>(bc + (r + 1) * RB, row_shift<S, ALIGNED>(vrow + (n + 1) * vs), s, o);
                zip8(e, o, V[j]);
            }
        }
        for (int c = 0; c < w.nc; ++c) {
            f2 dt[8], u[8];
            tile_get_twice(dt_ + c * kSsmTile, s, dt);
            tile_get_twice(u_ + c * kSsmTile, s, u);
            const f2 span = add2(add2(add2(dt[0], dt[1]), add2(dt[2], dt[3])), add2(add2(dt[4], dt[5]), add2(dt[6], dt[7])));
            const float4 A4 = *reinterpret_cast<const float4 *>(A_ + c * p.NP + n0);
            const float4 h4 = *reinterpret_cast<const float4 *>(h_ + c * p.NP + n0);
            __syncwarp();
            const f2 Av[2] = {pk(A4.x, A4.y), pk(A4.z, A4.w)};
            f2 hv[1][2] = {{pk(h4.x, h4.y), pk(h4.z, h4.w)}};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f2 all = mul2(span, Av[j]);
                f2 P[1] = {pk(ex2(lo(all)), ex2(hi(all)))}, S0[1] = {0}, in[1];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int i8 = REVERSE ? 7 - k : k;
                    const f2 e = mul2(dt[i8], Av[j]), a = pk(ex2(lo(e)), ex2(hi(e))), b = mul2(u[i8], V[j][i8]);
                    // h = a h + u B;  reverse c = a (C dy + c)
                    S0[0] = REVERSE ? mul2(a, k ? add2(S0[0], b) : b) : (k ? fma2(a, S0[0], b) : b);
                }
                lane_scan2<!REVERSE, 1>(P, S0, hv, j, in, s);
            }
            if (s == (REVERSE ? 0 : 7))
                *reinterpret_cast<float4 *>(h_ + c * p.NP + n0) = make_float4(lo(hv[0][0]), hi(hv[0][0]), lo(hv[0][1]), hi(hv[0][1]));
        }
    }
    __syncwarp();
    if (w.nc > 0) {
        const int64_t row = (w.b * p.segs + w.seg) * p.channels + w.d0;
        states_out(carries + row * p.N, h_, w.nc, p.N, p.NP, lane);
        if (lane < w.nc) {
            float v = 0.f;
            for (int i = 0; i < 16; ++i) v += sum_[lane * 16 + i];
            sums[row + lane] = v;
        }
    }
}

// In place: what each piece leaves becomes what enters it, in the order of the scan from `first` on.
static __global__ void __launch_bounds__(128)
ssm_fold_kernel(float *__restrict__ carries, const float *__restrict__ sums, const float *__restrict__ A,
                const float *__restrict__ first, int64_t batch, int64_t channels, int N, int segs, int reverse) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x, per = channels * N;
    if (i >= batch * per) return;
    const int64_t b = i / per, k = i - b * per, d = k / N;
    const float a = A[k] * kLog2e;
    float carry = first ? first[i] : 0.f;
    constexpr int M = 8;  // loads ahead of the serial fold
    for (int j0 = 0; j0 < segs; j0 += M) {
        float c[M], t[M];
#pragma unroll
        for (int j = 0; j < M; ++j)
            if (j0 + j < segs) {
                const int64_t seg = b * segs + (reverse ? segs - 1 - j0 - j : j0 + j);
                c[j] = carries[seg * per + k];
                t[j] = sums[seg * channels + d];
            }
#pragma unroll
        for (int j = 0; j < M; ++j)
            if (j0 + j < segs) {
                const int64_t seg = b * segs + (reverse ? segs - 1 - j0 - j : j0 + j);
                carries[seg * per + k] = carry;
                carry = fmaf(ex2(a * t[j]), carry, c[j]);
            }
    }
}

// The last sums of the backward in one launch, each in a fixed order.  Blocks below `bc_blocks`: grad_B and
// grad_C over the CTAs along the channels, 256 positions of a row (sequence, group, B | C, state) each; the
// others: grad_A, grad_D and grad_delta_bias over the sequences and pieces of time.
template <typename S>
__global__ void __launch_bounds__(256)
ssm_finish_kernel(const SsmProblem<S> p, const SsmGrads<S> o, S *__restrict__ dB, S *__restrict__ dC, float *__restrict__ dA,
                  float *__restrict__ dD, float *__restrict__ dbias, unsigned bc_blocks, int row_blocks) {
    if (blockIdx.x < bc_blocks) {
        const int Tpad = p.tiles * kSsmTile;
        const int64_t row = blockIdx.x / row_blocks, bg = row / (2 * p.N);
        const int r = static_cast<int>(row - bg * 2 * p.N), which = r >= p.N, n = r - which * p.N;
        const int t = static_cast<int>(blockIdx.x - row * row_blocks) * 256 + threadIdx.x;
        if (t >= p.T) return;
        const int64_t step = 2 * static_cast<int64_t>(p.N) * Tpad;
        const float *src = o.bc_part + bg * p.chunks * step + r * static_cast<int64_t>(Tpad) + t;
        float v = 0.f;
#pragma unroll 4
        for (int k = 0; k < p.chunks; ++k) v += src[k * step];
        (which ? dC : dB)[(bg * p.N + n) * p.T + t] = from_float<S>(v);
        return;
    }
    int64_t i = static_cast<int64_t>(blockIdx.x - bc_blocks) * 256 + threadIdx.x;
    const int64_t nA = p.channels * p.N, parts = p.batch * p.segs;
    const float *src = o.a_part;
    int64_t step = nA;
    float *dst = dA;
    if (i >= nA) {
        i -= nA;
        if (i >= 2 * p.channels) return;
        src = o.d_part, step = 2 * p.channels;
        dst = i < p.channels ? dD : dbias ? dbias - p.channels : nullptr;
        if (!dst) return;
    }
    float v = 0.f;
#pragma unroll 4
    for (int64_t k = 0; k < parts; ++k) v += src[k * step + i];
    dst[i] = v;
}

// ---------------------------------------------------------------- one token ------------------
// Row b's place in the pool, or -1 for padding.  A slot that an earlier row names belongs to that row:
// every thread looks at its share of the earlier rows, on loads that need not wait for its own slot, and the
// block votes.
__device__ __forceinline__ int64_t step_slot(const int64_t *slots, int64_t b, int64_t pool) {
    const int64_t v = slots ? slots[b] : b;
    return v >= 0 && v < pool ? v : -1;
}
__device__ __forceinline__ bool slot_seen(const int64_t *slots, int64_t b, int64_t slot) {
    bool seen = false;
    if (slots && slot >= 0)
        for (int64_t k = threadIdx.x; k < b; k += blockDim.x) seen |= slots[k] == slot;
    return seen;
}

// Eight consecutive values; `vec`: they are whole and start on a 16-byte boundary.
template <typename S>
__device__ __forceinline__ void load_eight(const S *__restrict__ p, bool vec, int left, float (&f)[8]) {
    if (vec) {
        if constexpr (sizeof(S) == 4) {
            const float4 v = reinterpret_cast<const float4 *>(p)[0], w = reinterpret_cast<const float4 *>(p)[1];
            f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w, f[4] = w.x, f[5] = w.y, f[6] = w.z, f[7] = w.w;
        } else {
            Store<S>::unpack(*reinterpret_cast<const uint4 *>(p), f);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < left ? Store<S>::to_float(p[i]) : 0.f;
    }
}

// A block has 128 / L channels of one row and group.  What a channel needs once (time step, gate) is
// prepared by one thread per channel in shared memory while the states, asked for before, are on their
// way; then L lanes share a channel, 8 states a lane.  Bound by the states' bytes (8 per state) for many
// rows, by the latency of one pass for a few.  Two channels a thread, or a block that walks several rows with
// the next one's states on their way, were no faster (256 rows x 2048 channels x 16 states: 24 us of 11 us
// for the bytes alone).  VEC: states and A come in vectors.
template <typename S, bool VEC>
__global__ void __launch_bounds__(128)
ssm_step_kernel(const SsmProblem<S> p, float *__restrict__ state, int64_t pool, const int64_t *__restrict__ slots,
                S *__restrict__ out, int log_L, bool bc_vec) {
    __shared__ float4 once[128];  // dt log2(e), dt x, D x, gate
    __shared__ float y_[128];
    const int L = 1 << log_L, per = 128 >> log_L, l = threadIdx.x & (L - 1), c = threadIdx.x >> log_L;
    const int first = blockIdx.x * per, nc = min(per, p.per_group - first), g = blockIdx.y;
    const int64_t d0 = static_cast<int64_t>(g) * p.per_group + first;
    for (int64_t b = blockIdx.z; b < p.batch; b += gridDim.z) {
        const int64_t slot = step_slot(slots, b, pool);
        const S *Bp = p.B + b * p.Bs[0] + g * p.Bs[1], *Cp = p.C + b * p.Cs[0] + g * p.Cs[1];
        float *hp = state + (slot * p.channels + d0 + c) * p.N;
        const float *Ap = p.A + (d0 + c) * p.N;
        float h[8], A[8], B[8], C[8], y = 0.f;
        auto fetch = [&](int n) {
            load_eight(hp + n, VEC, p.N - n, h);
            load_eight(Ap + n, VEC, p.N - n, A);
            load_eight(Bp + n, bc_vec, p.N - n, B);
            load_eight(Cp + n, bc_vec, p.N - n, C);
        };
        const bool seen = slot_seen(slots, b, slot);
        if (slot >= 0) {
            if (c < nc && 8 * l < p.N) fetch(8 * l);
            if (static_cast<int>(threadIdx.x) < nc) {
                const int64_t d = d0 + threadIdx.x;
                const float x = Store<S>::to_float(p.x[b * p.xs[0] + d]), z = p.z ? Store<S>::to_float(p.z[b * p.zs[0] + d]) : 0.f;
                float dt = Store<S>::to_float(p.delta[b * p.ds[0] + d]) + (p.bias ? p.bias[d] : 0.f);
                if (p.softplus) dt = softplus_f(dt);
                once[threadIdx.x] = make_float4(dt * kLog2e, dt * x, p.D ? p.D[d] * x : 0.f, p.z ? z * sigmoid_f(z) : 1.f);
            }
        }
        const bool use = !__syncthreads_or(seen) && slot >= 0;
        if (use) {
            if (c < nc) {
                const float2 v = *reinterpret_cast<const float2 *>(&once[c]);
                for (int n = 8 * l; n < p.N; n += 8 * L) {
                    if (n != 8 * l) fetch(n);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        h[i] = fmaf(ex2(v.x * A[i]), h[i], v.y * B[i]);
                        y = fmaf(C[i], h[i], y);
                    }
                    if constexpr (VEC) {
                        reinterpret_cast<float4 *>(hp + n)[0] = make_float4(h[0], h[1], h[2], h[3]);
                        reinterpret_cast<float4 *>(hp + n)[1] = make_float4(h[4], h[5], h[6], h[7]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (n + i < p.N) hp[n + i] = h[i];
                    }
                }
            }
            for (int i = 1; i < L; i *= 2) y += __shfl_xor_sync(kFullMask, y, i);
            if (l == 0) y_[c] = y;
        }
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < nc)
            out[b * p.channels + d0 + threadIdx.x] = from_float<S>(use ? (y_[threadIdx.x] + once[threadIdx.x].z) * once[threadIdx.x].w : 0.f);
        __syncthreads();
    }
}

}  // namespace fms
