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

// v of the lane whose index differs in bit kBit, for lanes whose values agree
// below it (4: i -> 7 - i within 8 lanes, 8: i -> 15 - i within 16).
template <int kBit>
__device__ __forceinline__ float from_xor(float v) {
    static_assert(kBit == 1 || kBit == 2 || kBit == 4 || kBit == 8, "within a DPP row");
    constexpr int kCtrl = kBit == 1 ? 0xB1 : kBit == 2 ? 0x4E : kBit == 4 ? 0x141 : 0x140;
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xF, 0xF, false));
}

// Sum over the kLanes (2 to 32) neighbouring lanes of a row, on the VALU.
template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
    v += from_xor<1>(v);
    if constexpr (kLanes > 2) v += from_xor<2>(v);
    if constexpr (kLanes > 4) v += from_xor<4>(v);
    if constexpr (kLanes > 8) v += from_xor<8>(v);
    if constexpr (kLanes > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// Workgroup: 4 waves, kTokens (1 or 4) tokens.  The angles' sines and cosines
// are computed once per token, a thread per pair, and shared by all heads
// through LDS; then a token's rows (heads) go through one wave (kTokens = 4)
// or are dealt to all four, D / 8 lanes of 8 channels each to a row, so a wave
// moves 64 16-byte chunks an instruction and a lane's channels, weights, sines
// and cosines are the same for all its rows.  Bound by memory: kAhead passes' rows
// are requested together, the first ones before the angles; the stores, which
// nothing here reads again, go past the caches.  17918 tokens of 32 + 8 heads, D =
// 128 (367 MB): 76.5 us, 4.8 TB/s, as a copy reaches.  Where this form took 79.5,
// one pass ahead took 94, three 89 (registers), cached stores 84.6.
template <bool kBF, int D, int kTokens>
__global__ __launch_bounds__(64 * kRopeWaves)
void kf_qk_norm_rope_kernel(RopeParams p) {
    constexpr int kLanes = D / 8;               // lanes of a row
    constexpr int kRows = 64 / kLanes;          // rows of a wave's pass
    constexpr int kAhead = 2;
    constexpr int kStep = kRows * (kTokens == 1 ? kRopeWaves : 1);
    __shared__ float2 turn[kTokens * (D / 2)];  // scale cos, scale sin

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t = blockIdx.x * kTokens + (kTokens == 1 ? 0 : wave);
    const int c = lane % kLanes;                // this lane's chunk of 8 channels
    const int first_row = kTokens == 1 ? wave * kRows : 0;
    // Row r0 + lane / kLanes of the token; past the last head, the last one again.
    const int tc = min(t, p.tokens - 1);
    const uint16_t* const xq = p.x[0] + (size_t)tc * p.token[0];
    const uint16_t* const xk = p.x[1] + (size_t)tc * p.token[1];
    auto row_of = [&](int r0) { return min(r0 + lane / kLanes, p.heads - 1); };
    auto load = [&](int r0) {
        const int r = row_of(r0);
        const uint16_t* x = r >= p.heads_q ? xk + (size_t)(r - p.heads_q) * p.head[1] : xq + (size_t)r * p.head[0];
        return *reinterpret_cast<const u32x4*>(x + 8 * c);
    };
    u32x4 raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) raw[u] = load(first_row + u * kStep);

    const int half = p.rot / 2;
    for (int k = tid; k < kTokens * half; k += 64 * kRopeWaves) {
        const int tt = min((int)blockIdx.x * kTokens + k / half, p.tokens - 1);
        const double turns = (double)p.positions[tt] * p.freqs[k % half] * 0.15915494309189535;
        const float f = (float)(turns - __builtin_rint(turns));  // within half a turn
        float sn, cs;
        sincos_turns(f, sn, cs);
        turn[k] = make_float2(p.scale * cs, p.scale * sn);
    }
    __syncthreads();
    if (t >= p.tokens) return;

    const float2* tt = turn + (kTokens == 1 ? 0 : wave) * half;
    const bool turned = 8 * c < p.rot;
    const bool first = p.interleaved || 16 * c < p.rot;
    // The lane that holds the pairs' other channels (half layout).
    const int other = turned ? lane + (first ? p.rot / 16 : -(p.rot / 16)) : lane;
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int i = p.interleaved ? (8 * c + e) / 2 : first ? 8 * c + e : 8 * c + e - half;
        const float2 v = turned ? tt[i] : make_float2(1.f, 0.f);
        cs[e] = v.x;
        // The sign with which the other channel of the pair comes in.
        sn[e] = (p.interleaved ? (e & 1) == 0 : first) ? -v.y : v.y;
    }
    // Weights of this lane's channels, of 1 where there are none.
    const uint32_t one = kBF ? 0x3f803f80u : 0x3c003c00u;
    u32x4 wt[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
        wt[s] = p.w[s] ? *reinterpret_cast<const u32x4*>(p.w[s] + 8 * c) : u32x4{one, one, one, one};

    for (int r0 = first_row; r0 < p.heads; r0 += kAhead * kStep) {
        u32x4 now[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) now[u] = raw[u];
        if (r0 + kAhead * kStep < p.heads) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) raw[u] = load(r0 + (kAhead + u) * kStep);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int r = row_of(r0 + u * kStep);
            const int s = r >= p.heads_q;
            f32x8 v = widen8<kBF>(now[u]);
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
            sum = row_sum<kLanes>(sum);
            const bool normed = s ? p.w[1] != nullptr : p.w[0] != nullptr;
            const float norm = normed ? 1.0f / __builtin_sqrtf(sum * (1.0f / D) + p.eps) : 1.0f;
            const f32x8 w = widen8<kBF>(s ? wt[1] : wt[0]);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= w[e] * norm;
            f32x8 y;
            if (p.interleaved) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = fmaf(v[e ^ 1], sn[e], v[e] * cs[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = fmaf(__shfl(v[e], other), sn[e], v[e] * cs[e]);
            }
            if (!turned) y = v;
            if (r0 + u * kStep + lane / kLanes < p.heads) {
                uint16_t* out = p.y[s] + (size_t)t * p.y_token[s] + (size_t)(s ? r - p.heads_q : r) * p.y_head[s];
                __builtin_nontemporal_store(__builtin_bit_cast(u32x4, round8<kBF>(y)), reinterpret_cast<u32x4*>(out + 8 * c));
            }
        }
    }
}

}  // namespace kf
