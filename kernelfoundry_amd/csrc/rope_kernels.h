// rope_kernels.h -- RMS norm of every query and key head, then rotary
// positions, in one pass over Q and K.
//
//   y = x / sqrt(mean(x^2) + eps) * w              (over the D channels; only with weights)
//   angle_i = position * freqs[i],  i < rot / 2
//   (a, b) -> scale * (a cos - b sin, b cos + a sin)
// for the channel pairs (i, i + rot / 2), or (2 i, 2 i + 1) interleaved; the
// channels from rot on keep y.  Everything in fp32, rounded once; the angle
// is reduced to a fraction of a turn in fp64, since position * freq reaches
// 2^20 radians, of which fp32 would keep 2^-4.
#pragma once

#include "elem.h"

namespace kf {

struct RopeParams {
    const uint16_t* x[2];    // Q, K
    uint16_t* y[2];
    const uint16_t* w[2];    // [D] or null: no norm
    long long token[2], head[2];  // strides of x in elements
    long long y_token[2], y_head[2];
    int heads_q, heads;      // H_q, H_q + H_kv
    int tokens;
    const int* positions;
    const double* freqs;     // [rot / 2], radians per position
    int rot;
    int interleaved;
    float eps, scale;
};

constexpr int kRopeWaves = 4;

// sin and cos of 2 pi f, |f| <= 1/2, to a few units in the last place of 1: the
// nearest quarter turn is taken off exactly, and for the rest, |x| <= pi / 4,
// the Taylor series end below 2^-29 (sin, x^11 / 11!) and 2^-25 (cos, x^10 / 10!).
// (v_sin_f32 and v_cos_f32 promise no such bound.)
__device__ __forceinline__ void sincos_turns(float f, float& sn, float& cs) {
    const float quarter = __builtin_rintf(4.0f * f);
    const float x = (f - 0.25f * quarter) * 6.283185307179586f, z = x * x;
    const float s = x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), 1.f);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.f / 40320, -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const int k = (int)quarter;                // -2 .. 2
    sn = (k & 1) ? c : s;
    cs = (k & 1) ? s : c;
    if (k & 2) sn = -sn;
    if ((k + 1) & 2) cs = -cs;
}

// Workgroup: 4 waves, kTokens (1 or 4) tokens.  The angles' sines and cosines
// are computed once per token, a thread per pair, and shared by all heads
// through LDS; then a token's rows (heads) go through one wave (kTokens = 4)
// or are dealt to all four, D / 8 lanes of 8 channels each to a row, so a wave
// moves 64 16-byte chunks an instruction and a lane's channels, weights, sines
// and cosines are the same for all its rows.
template <bool kBF, int D, int kTokens>
__global__ __launch_bounds__(64 * kRopeWaves)
void kf_qk_norm_rope_kernel(RopeParams p) {
    using X8 = typename Elem<kBF>::x8;
    constexpr int kLanes = D / 8;               // lanes of a row
    constexpr int kRows = 64 / kLanes;          // rows of a wave's pass
    __shared__ float2 turn[kTokens * (D / 2)];  // scale cos, scale sin

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int half = p.rot / 2;
    for (int k = tid; k < kTokens * half; k += 64 * kRopeWaves) {
        const int t = blockIdx.x * kTokens + k / half;
        if (t < p.tokens) {
            const double turns = (double)p.positions[t] * p.freqs[k % half] * 0.15915494309189535;
            const float f = (float)(turns - __builtin_rint(turns));  // within half a turn
            float sn, cs;
            sincos_turns(f, sn, cs);
            turn[k] = make_float2(p.scale * cs, p.scale * sn);
        }
    }
    __syncthreads();

    const int t = blockIdx.x * kTokens + (kTokens == 1 ? 0 : wave);
    if (t >= p.tokens) return;
    const float2* tt = turn + (kTokens == 1 ? 0 : wave) * half;
    const int c = lane % kLanes;                // this lane's chunk of 8 channels
    const bool turned = 8 * c < p.rot;
    const bool first = p.interleaved || 16 * c < p.rot;
    // The lane that holds the pairs' other channels (half layout).
    const int other = lane + (first ? p.rot / 16 : -(p.rot / 16));
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int i = p.interleaved ? (8 * c + e) / 2 : first ? 8 * c + e : 8 * c + e - half;
        const float2 v = turned ? tt[i] : make_float2(1.f, 0.f);
        cs[e] = v.x;
        // The sign with which the other channel of the pair comes in.
        sn[e] = (p.interleaved ? (e & 1) == 0 : first) ? -v.y : v.y;
    }
    for (int r0 = (kTokens == 1 ? wave : 0) * kRows; r0 < p.heads; r0 += kRows * (kTokens == 1 ? kRopeWaves : 1)) {
        const int r = min(r0 + lane / kLanes, p.heads - 1);  // (the last pass' spare lanes repeat a row)
        const int s = r >= p.heads_q;
        const int h = s ? r - p.heads_q : r;
        const u32x4 raw = *reinterpret_cast<const u32x4*>(p.x[s] + (size_t)t * p.token[s] +
                                                          (size_t)h * p.head[s] + 8 * c);
        f32x8 v = widen8<kBF>(raw);
        f32x8 wt;
        float norm = 1.f;
        if (p.w[s]) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
#pragma unroll
            for (int m = 1; m < kLanes; m *= 2) sum += __shfl_xor(sum, m);
            norm = 1.0f / __builtin_sqrtf(sum * (1.0f / D) + p.eps);
            wt = widen8<kBF>(*reinterpret_cast<const u32x4*>(p.w[s] + 8 * c));
            v *= wt * norm;
        }
        f32x8 y;
        if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = fmaf(v[e ^ 1], sn[e], v[e] * cs[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = fmaf(__shfl(v[e], other), sn[e], v[e] * cs[e]);
        }
        if (!turned) y = v;
        if (r0 + lane / kLanes < p.heads)
            *reinterpret_cast<X8*>(p.y[s] + (size_t)t * p.y_token[s] + (size_t)h * p.y_head[s] + 8 * c) =
                round8<kBF>(y);
    }
}

}  // namespace kf
