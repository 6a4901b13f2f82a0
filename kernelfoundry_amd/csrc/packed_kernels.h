// packed_kernels.h -- attention over packed sequences: queries, keys and
// values of all sequences one after the other, [tokens][heads][D] with any
// token and head strides, as the projections write them.
//
// The query rows that read a KV head are (token, head of its group), token
// major: row r of a sequence is query r / ratio of group head r % ratio.  A
// workgroup takes a tile of consecutive rows of one sequence and KV head, so
// grouped heads share every K and V stage, and a tile's rows cover few
// tokens, which keeps the part of the causal triangle that a tile computes
// for nothing small.  The work inside a tile is the wide prefill's: S^T = K Q^T,
// online softmax, O^T += V^T P^T with the 32x32x16 MFMA, K and V stages HBM
// -> LDS by LDS-DMA, P^T straight from the score registers.
//
// Bound by the matrix units and the softmax between their products: causal, 32 / 8
// heads, D = 128, 1 x 8192 takes 507 to 518 us in bf16 and 545 in fp16, 1.0 to 1.1
// PFLOP/s (a library product 1.2), MFMA busy 59 % of the SIMD cycles, LDS 30 %, next to
// no bank conflicts; 16 sequences of 16 to 4096 111 to 119 us (0.77 to 0.82 PFLOP/s), of
// which a workgroup's first loads and its store (191 MB in all, 38 us of memory time)
// hide behind other workgroups' products in part; 4 x 512 queries against 4096
// keys, 16 / 4 heads, D = 256, 146 to 154 (0.84 to 0.88).  1 x 4096 in fp16: 144 us at 32
// / 8 heads of 128 (0.95; with fp32 output 146), 91 at 32 / 1 of 64 (0.76), 165 to 169
// at 16 / 4 of 256 (0.81 to 0.83), 276 at 32 / 8 of 256 (0.99); without the mask 283 at 32 / 8 of
// 128 (0.97), 164 at 32 / 8 of 64 (0.84), 268 at 16 / 4 of 256 (1.03).  What bounds
// D = 64 is not measured.  Tried: 64 rows a wave on 8 waves
// (4 to 6 % faster at 8192, 5 to 40 % slower at the others), the scores of the next
// stage beside this one's products (its third buffer costs a workgroup a CU: no gain),
// stages requested two tiles ahead (no change), two V tiles before the softmax at
// D = 128 (spills).
#pragma once

#include "elem.h"

namespace kf {

struct PackedParams : AttnParams {  // Q, K, V, O, Mi (LSE), scales, causal, heads_kv, out_dtype, xcds
    long long q_token, k_token, v_token;  // strides in elements
    long long q_head, k_head, v_head;
    const int* q_starts;                  // [n_seqs + 1]
    const int* k_starts;
    int n_seqs, tokens_q, tokens_k, ratio;
    int level_tiles;                      // see packed_find
};

// A workgroup is NW waves of 32 query rows each; with KS > 1 they form KS
// groups that take the same rows and a share of the keys each, merged through
// LDS at the end.
template <int D, int NW, int KS> struct PackedCfg {
    static constexpr int kThreads = 64 * NW;
    static constexpr int kRowWaves = NW / KS;             // waves per KV group
    static constexpr int kRows = 32 * kRowWaves;          // query rows per workgroup
    static constexpr int BC = 32;                         // keys per MFMA tile and LDS stage
    // Waves per SIMD that the registers have to allow: three workgroups of 4 waves
    // a CU at D = 128 (four at D = 64, two at D = 256), two of 8 waves at D = 64.
    static constexpr int kWavesPerSimd = D == 64 ? 4 : D == 128 && KS == 1 ? 3 : 2;
    // LDS reads that are issued together, ahead of the MFMAs that need them: K
    // fragments (16 channels each), and V^T tiles of 32 channels before the
    // softmax, which does not need them.  As many as the registers leave: with one
    // or two waves on a SIMD nothing else hides an LDS read's latency (512 queries
    // against 4096 keys, 32 / 8 heads, D = 128: KS = 1 105.7 -> 96.6 us, KS = 2
    // 74.3 -> 65.3; full grids lose 1 %).
    static constexpr int kBatch = D == 256 ? 4 : KS == 1 ? 2 : D / 16;
    static constexpr int kAhead = D == 256 ? 0 : KS == 1 ? 1 : D / 32;
    // Kept apart from the scheduler; without KV groups it does as well by itself (1 x 8192,
    // 32 / 8 heads, D = 128: bf16 518 and 514 us, no more than two runs differ by).
    static constexpr bool kOrder = KS > 1 && D < 256;
    // Stages copied in asm, from a scalar row and lane offsets that stay in registers; the
    // builtin's offsets, computed for every stage, cost 2 to 3 % (1 x 8192, 32 / 8 heads,
    // D = 128, bf16 524 -> 512 us; 1 x 4096, 32 / 1 heads, D = 64, 93.2 -> 90.2). At
    // D = 256 there are no registers for them: spills, and no gain without.
    static constexpr bool kAsmCopy = D < 256;
    // The per-lane LDS offsets of a tile derived from one, for want of registers.
    static constexpr bool kXorOff = D >= 128;
};

// One sequence's tokens and keys.
struct PackedSeq {
    int q0, qn, k0, kn;
};
__device__ __forceinline__ PackedSeq packed_seq(const PackedParams& p, int i) {
    PackedSeq s;
    s.q0 = min(max(p.q_starts[i], 0), p.tokens_q);
    s.qn = min(max(p.q_starts[i + 1], s.q0), p.tokens_q) - s.q0;
    s.k0 = min(max(p.k_starts[i], 0), p.tokens_k);
    s.kn = min(max(p.k_starts[i + 1], s.k0), p.tokens_k) - s.k0;
    return s;
}

// Workgroup tile j of a KV head -> sequence and row tile in it; false past the
// last.  Up to 64 sequences (one to a lane) the tiles are numbered by their keys,
// longest first: the dispatcher starts workgroups in order, and short tiles then fill
// the CUs that finish early.  A tile's level is its keys in units of level_tiles tiles'
// rows, up to a constant: a sequence that is not causal has one, a causal one
// level_tiles of its tiles in each, its last ones first.  Against tiles
// numbered sequence by sequence (us, 32 / 8 heads of 128 where not stated, causal):
// 1 x 8192 bf16 559 -> 510, 16 sequences of 16 to 4096 122 -> 116, 8 x 1024 with
// 16 / 16 heads of 64 40.4 -> 28.3, 1 x 4096 with 16 / 4 of 256 198 -> 160; 1 x 512 and
// 32 x 128, of which all workgroups run at once, 12.6 -> 13.1 and 20.8 -> 21.2.
// More than 64 sequences, a lane each, are numbered one after the other: the more
// there are, the less the order does (64 of 16 to 2048, heads of 64, 122 -> 117).
template <int kRows>
__device__ __forceinline__ bool packed_find(const PackedParams& p, int lane, int j, int& seq, int& tile) {
    const auto tiles_of = [&](const PackedSeq& s) { return (int)(((long long)s.qn * p.ratio + kRows - 1) / kRows); };
    if (p.n_seqs <= 64) {
        PackedSeq s{0, 0, 0, 0};
        if (lane < p.n_seqs) s = packed_seq(p, lane);
        const int n = tiles_of(s);
        const int low = (int)((long long)max(p.causal ? s.kn - s.qn : s.kn, 0) * p.ratio / kRows);
        const auto from = [&](int k) {   // this lane's tiles of level k or more
            return p.causal ? min(max(low + n - k * p.level_tiles, 0), n) : low >= k * p.level_tiles ? n : 0;
        };
        if (__builtin_amdgcn_readlane(wave_scan(n), 63) <= j) return false;
        // The largest level of which, with those above it, there are more than j.
        int lo = 0, hi = (low + n) / p.level_tiles + 1;  // hi: none from there on, once it is the wave's largest
#pragma unroll
        for (int m = 1; m < 64; m *= 2) hi = max(hi, __shfl_xor(hi, m));
        hi = __builtin_amdgcn_readfirstlane(hi);
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (__builtin_amdgcn_readlane(wave_scan(from(mid)), 63) > j) lo = mid; else hi = mid;
        }
        const int longer = from(lo + 1), here = from(lo) - longer;
        const int above = __builtin_amdgcn_readlane(wave_scan(longer), 63);
        const int inc = wave_scan(here);
        const uint64_t mine = __ballot(inc > j - above);
        seq = __builtin_ctzll(mine);
        // Of the sequence's tiles the last one above which `longer` lie.
        tile = __builtin_amdgcn_readlane(n - 1 - longer + inc - here, seq) - (j - above);
        return true;
    }
    // 64 runs of consecutive sequences, then the sequences of the run.
    const int per = (p.n_seqs + 63) / 64;
    int sum = 0;
    for (int i = lane * per; i < min((lane + 1) * per, p.n_seqs); ++i) sum += tiles_of(packed_seq(p, i));
    int inc = wave_scan(sum);
    uint64_t past = __ballot(inc > j);
    if (past == 0) return false;
    const int run = __builtin_ctzll(past);
    int left = j - (__builtin_amdgcn_readlane(inc, run) - __builtin_amdgcn_readlane(sum, run));
    for (int i0 = run * per;; i0 += 64) {
        const int i = i0 + lane;
        sum = i < min((run + 1) * per, p.n_seqs) ? tiles_of(packed_seq(p, i)) : 0;
        inc = wave_scan(sum);
        past = __ballot(inc > left);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            seq = i0 + at;
            tile = left - (__builtin_amdgcn_readlane(inc, at) - __builtin_amdgcn_readlane(sum, at));
            return true;
        }
        left -= __builtin_amdgcn_readlane(inc, 63);
        if (i0 + 64 >= min((run + 1) * per, p.n_seqs)) return false;  // not reached
    }
}

// exp2 and 16-bit pack of a 32-row score block.  The product with V takes 16-bit
// operands, so the weights are rounded (relative 2^-11 or 2^-8: with O's own
// rounding 1.2 to 1.4 times the error of weights kept in fp32); the fp32 values are
// summed, so that the log-sum-exp has their precision.
template <bool kBF>
__device__ __forceinline__ void packed_exp(const f32x16& s, float scale_log2, float neg_m,
                                           typename Elem<kBF>::x8 (&p)[2], float& acc) {
    f32x8 e0, e1;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        e0[r] = exp2_hw(fmaf(s[r], scale_log2, neg_m));
        e1[r] = exp2_hw(fmaf(s[8 + r], scale_log2, neg_m));
    }
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        a += e0[r];
        b += e1[r];
    }
    acc += a + b;
    p[0] = round8<kBF>(e0);
    p[1] = round8<kBF>(e1);
}

// Store a wave's 32-row block of O, scaled by inv, as kOut, through kBytes of
// LDS of the wave's own.  From the accumulators a lane would write 8 or 16 bytes
// of its row, 32 rows to an instruction; as it lies in LDS the wave writes whole
// rows, 16 bytes a lane (32 prompts of 128 tokens, 32 / 8 heads, D = 128: 31.6 us -> 22.5).
// Row r's 16-byte chunk c is at chunk c ^ (r & 15 or fewer), against bank
// conflicts; as many 32-channel tiles at a time as fit.  `at`: lane r's row in O.
template <int kOut, int D, int kBytes>
__device__ __forceinline__ void packed_store(const AttnParams& p, const f32x16 (&o)[D / 32], float inv, char* lds, int at,
                                             int nrows, int lane) {
    constexpr int kSize = kOut == kOutF32 ? 4 : 2;
    constexpr int kTiles = kBytes / (32 * 32 * kSize) < D / 32 ? kBytes / (32 * 32 * kSize) : D / 32;
    constexpr int kChunks = kTiles * 32 * kSize / 16;     // of a row, at a time
    constexpr int kMask = (kChunks < 16 ? kChunks : 16) - 1;
    static_assert(kTiles >= 1 && (D / 32) % kTiles == 0 && (kChunks & kMask) == 0, "whole passes");
    const int row = lane & 31, g = lane >> 5;
    char* const mine = lds + row * kChunks * 16;
#pragma unroll
    for (int t0 = 0; t0 < D / 32; t0 += kTiles) {
#pragma unroll
        for (int td = 0; td < kTiles; ++td)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 32 * td + 8 * i + 4 * g;    // of the pass
                const f32x4 v = f32x4{o[t0 + td][4 * i], o[t0 + td][4 * i + 1], o[t0 + td][4 * i + 2],
                                      o[t0 + td][4 * i + 3]} * inv;
                if constexpr (kOut == kOutF32) {
                    *reinterpret_cast<f32x4*>(mine + ((d / 4) ^ (row & kMask)) * 16) = v;
                } else {
                    char* const dst = mine + ((d / 8) ^ (row & kMask)) * 16 + g * 8;
                    if constexpr (kOut == kOutF16)
                        *reinterpret_cast<f16x4*>(dst) = __builtin_convertvector(v, f16x4);
                    else
                        *reinterpret_cast<bf16x4*>(dst) = __builtin_convertvector(v, bf16x4);
                }
            }
        wave_lds_sync();
        char* const out = reinterpret_cast<char*>(p.O) + t0 * 32 * kSize;
#pragma unroll 4
        for (int k = 0; k < kChunks / 2; ++k) {           // 32 kChunks chunks, 64 at a time
            const int r = (k * 64 + lane) / kChunks, c = (k * 64 + lane) % kChunks;
            const u32x4 v = *reinterpret_cast<const u32x4*>(lds + (r * kChunks + (c ^ (r & kMask))) * 16);
            const int to = __shfl(at, r);
            if (r < nrows) *reinterpret_cast<u32x4*>(out + (size_t)to * (D * kSize) + c * 16) = v;
        }
        wave_lds_sync();
    }
}

// LDS-DMA in asm as lds_copy16_nt's, but kept in the L2: other tiles read the same keys.
__device__ __forceinline__ void lds_copy16(uint32_t lds, const void* base, uint32_t off) {
    const uint64_t b = (uint64_t)(uintptr_t)base;
    base = (const void*)(uintptr_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) |
                                    (uint32_t)__builtin_amdgcn_readfirstlane((int)b));
    lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
                 ::"{m0}"(lds), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void lds_copy16(uint32_t lds, const void* lane_src) {
    lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, off"
                 ::"{m0}"(lds), "v"(lane_src) : "memory");
}

template <bool kBF, int D, int NW, int KS>
__global__ __launch_bounds__((PackedCfg<D, NW, KS>::kThreads), (PackedCfg<D, NW, KS>::kWavesPerSimd))
void kf_attn_packed_kernel(PackedParams p) {
    using Cfg = PackedCfg<D, NW, KS>;
    using E = Elem<kBF>;
    using X8 = typename E::x8;
    using SW = SwizzleRow<D>;
    constexpr int BC = Cfg::BC, kRows = Cfg::kRows;
    constexpr int kRowBytes = D * 2, kChunks = D / 8, kRowsPerInstr = 1024 / kRowBytes;
    constexpr int kInstr = BC * kRowBytes / 1024;         // LDS-DMA instructions per tensor and stage
    constexpr int kTensorBytes = BC * kRowBytes;
    constexpr int kRowWaves = Cfg::kRowWaves;
    constexpr int kPerWave = 2 * kInstr / kRowWaves;
    static_assert(2 * kInstr % kRowWaves == 0 && kInstr % kPerWave == 0, "a wave copies K or V");
    constexpr int kNKK = D / 16, kNTD = D / 32;
    constexpr int kBuf = KS * 2 * kTensorBytes;           // a stage of every group
    __shared__ __attribute__((aligned(1024))) char buf0[kBuf];
    __shared__ __attribute__((aligned(1024))) char buf1[kBuf];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave_id = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 5;
    // KV heads next to each other: with ids dealt round-robin over the XCDs, 8
    // heads have an XCD, and its L2, each.
    const int hk = blockIdx.x % p.heads_kv;
    int seq, rt;
    if (!packed_find<kRows>(p, lane, blockIdx.x / p.heads_kv, seq, rt)) return;
    PackedSeq sq = packed_seq(p, seq);
    sq.q0 = __builtin_amdgcn_readfirstlane(sq.q0);
    sq.qn = __builtin_amdgcn_readfirstlane(sq.qn);
    sq.k0 = __builtin_amdgcn_readfirstlane(sq.k0);
    sq.kn = __builtin_amdgcn_readfirstlane(sq.kn);
    const int ratio = p.ratio, R = sq.qn * ratio, klen = sq.kn;
    const float c = p.scale_log2;
    const int wave = KS > 1 ? wave_id % kRowWaves : wave_id;
    const int kgrp = KS > 1 ? wave_id / kRowWaves : 0;
    // (Of starts in no order the sums by which the tile was found may wrap.)
    if ((unsigned)rt * (unsigned)kRows >= (unsigned)R) return;
    const auto limit = [&](int row) {  // keys that the row sees
        return p.causal ? min(max(row / ratio + klen - sq.qn + 1, 0), klen) : klen;
    };
    const int r0 = rt * kRows, w0 = r0 + wave * 32;
    const int blk_lim = limit(min(R, r0 + kRows) - 1);
    // Group kgrp has keys [kv_base, kv_end), as many tiles as every other;
    // row limits count from kv_base.
    const int ntiles = ((blk_lim + BC - 1) / BC + KS - 1) / KS;
    const int kv_base = kgrp * ntiles * BC, kv_end = min(kv_base + ntiles * BC, blk_lim);
    const auto own = [&](int lim) { return KS > 1 ? min(lim, kv_end) - kv_base : lim; };
    const int wave_min = own(w0 < R ? limit(w0) : blk_lim);
    const int wave_max = own(w0 < R ? limit(min(R, w0 + 32) - 1) : 0);
    const int nt_w = (wave_max + BC - 1) / BC;            // the wave's tiles (none if not positive); it skips the others

    const int lim = own(limit(min(w0 + (lane & 31), R - 1)));
    const int nrows = R - w0;                             // rows of the wave, if any
    // The row of O (below tokens_q H_q, an int) of this lane; rows past R
    // compute on the last one and are not stored.  From an opaque lane, so that
    // none of it lives across the tiles.
    auto out_row = [&]() {
        int l = lane;
        asm volatile("" : "+v"(l));
        const int r = min(w0 + (l & 31), R - 1);
        return ((sq.q0 + r / ratio) * p.heads_kv + hk) * ratio + r % ratio;
    };
    if (ntiles == 0) {                                    // no key for any row
        const int at = out_row();
        if ((lane & 31) < nrows && kgrp == 0) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) store_out4(p, (size_t)at * D + 8 * i + 4 * g, f32x4{0.f, 0.f, 0.f, 0.f});
            if (g == 0) store_stats(p, at, -INFINITY, 0.f);
        }
        return;
    }

    const char* Kh = reinterpret_cast<const char*>(p.K + (size_t)sq.k0 * p.k_token + (size_t)hk * p.k_head);
    const char* Vh = reinterpret_cast<const char*>(p.V + (size_t)sq.k0 * p.v_token + (size_t)hk * p.v_head);
    // LDS-DMA: wave w of a group copies the KiB instructions w kPerWave + i of
    // its stage, all of K or all of V.  Lane l of one fills row l / kChunks of
    // its rows, physical chunk l % kChunks.
    const int copier = wave_id % kRowWaves;
    const bool is_v = copier * kPerWave >= kInstr;
    const char* src = is_v ? Vh : Kh;
    const uint32_t row_stride = 2 * (uint32_t)(is_v ? p.v_token : p.k_token);  // at most 2^29 (the host sees to it)
    const int ii0 = copier * kPerWave % kInstr;
    const int lr = lane / kChunks;
    // The swizzle depends on row & 15: the lane offsets of an instruction
    // within its rows repeat.
    constexpr int kPeriod = kRowsPerInstr >= 16 ? 1 : 16 / kRowsPerInstr < kPerWave ? 16 / kRowsPerInstr : kPerWave;
    uint32_t chunk_off[kPeriod];
#pragma unroll
    for (int i = 0; i < kPeriod; ++i)
        chunk_off[i] = (((lane % kChunks) ^ SW::h((ii0 + i) * kRowsPerInstr + lr)) % kChunks) * 16;
    auto issue_stage = [&](char* dst, int kv0) {
        char* d = dst + (is_v ? kTensorBytes : 0) + ii0 * 1024;
        const uint32_t d_lds = (uint32_t)(uintptr_t)(lds_void*)d;
        const int kv = kv_base + kv0 + ii0 * kRowsPerInstr;
        if (kv_base + kv0 + BC <= klen) {
            // Whole stage: wave-uniform row base and a 32-bit lane offset.
#pragma unroll
            for (int i = 0; i < kPerWave; ++i) {
                uint32_t off = lr * row_stride + chunk_off[i % kPeriod];
                if constexpr (Cfg::kAsmCopy) {
                    lds_copy16(d_lds + i * 1024, src + (size_t)(kv + i * kRowsPerInstr) * row_stride, off);
                } else {
                    asm volatile("" : "+v"(off));  // computed here, so that the address stays their sum
                    const char* a = src + (size_t)(kv + i * kRowsPerInstr) * row_stride + off;
                    __builtin_amdgcn_global_load_lds(a, (lds_void*)(d + i * 1024), 16, 0, 0);
                }
            }
        } else {
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = 0; i < kPerWave; ++i) {
                // Rows past the keys re-read the last one (finite data whose scores are masked).
                const int row = min(kv + i * kRowsPerInstr + lr, klen - 1);
                const char* a = src + (size_t)row * row_stride + chunk_off[i % kPeriod];
                if constexpr (Cfg::kAsmCopy)
                    lds_copy16(d_lds + i * 1024, a);
                else
                    __builtin_amdgcn_global_load_lds(a, (lds_void*)(d + i * 1024), 16, 0, 0);
            }
        }
    };

    // LDS reads, as in the prefill kernels.
    // (With D >= 128's swizzle the offset of k-step kk is that of the first ^ 32 kk,
    // of V^T tile td ^ 64 td, of its second 8 rows ^ 128 and 8 rows on: derived
    // at each tile where registers for them are short.)
    constexpr bool kXorOff = Cfg::kXorOff;
    static_assert(!kXorOff || D >= 128, "XOR offsets use the D >= 128 swizzle");
    int koff[kNKK];
#pragma unroll
    for (int kk = 0; kk < kNKK; ++kk) {
        const int r = lane & 31;
        koff[kk] = r * kRowBytes + (((2 * kk + g) ^ SW::h(r)) % kChunks) * 16;
    }
    int voff[kNTD][2];
    {
        const int G = lane >> 4, w = lane & 15;
#pragma unroll
        for (int td = 0; td < kNTD; ++td)
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2) {
                const int r = 4 * (G >> 1) + (w >> 2) + 8 * h2;
                const int d = 32 * td + 16 * (G & 1) + 4 * (w & 3);
                voff[td][h2] = kTensorBytes + r * kRowBytes + (((d >> 3) ^ SW::h(r)) % kChunks) * 16 + ((d >> 2) & 1) * 8;
            }
    }

    char* const b0 = buf0 + kgrp * 2 * kTensorBytes;      // this group's stages
    char* const b1 = buf1 + kgrp * 2 * kTensorBytes;
    issue_stage(b0, 0);
    X8 q[kNKK];
    {
        const int rc = min(w0 + (lane & 31), R - 1);
        const uint16_t* Qr = p.Q + (size_t)(sq.q0 + rc / ratio) * p.q_token + (size_t)(hk * ratio + rc % ratio) * p.q_head;
#pragma unroll
        for (int kk = 0; kk < kNKK; ++kk) q[kk] = *reinterpret_cast<const X8*>(Qr + (2 * kk + g) * 8);
    }

    RowState st{-INFINITY, -INFINITY, 0.f, -INFINITY};
    f32x16 o[kNTD];
    const float inv_c = 1.0f / c;
#pragma unroll
    for (int td = 0; td < kNTD; ++td) o[td] = f32x16{};
    // V^T of 32 channels and 16 keys, V rows at stage + kTensorBytes.
    auto v_frag = [&](const char* stage, int vb, int td, int jj) {
        const int vo0 = kXorOff ? vb ^ (64 * td) : voff[td][0];
        const int vo1 = kXorOff ? (vb ^ (64 * td) ^ 128) + 8 * kRowBytes : voff[td][1];
        const f16x4 lo = lds_read_tr16(stage + vo0 + jj * 16 * kRowBytes);
        const f16x4 hi = lds_read_tr16(stage + vo1 + jj * 16 * kRowBytes);
        return __builtin_bit_cast(X8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto tile = [&](const char* stage, int t) {
        if (t >= nt_w) return;
        constexpr int kBatch = Cfg::kBatch, kAhead = Cfg::kAhead;
        static_assert(kNKK % kBatch == 0 && kAhead <= kNTD, "whole batches");
        int kb = koff[0], vb = voff[0][0];
        if constexpr (kXorOff) asm volatile("" : "+v"(kb), "+v"(vb));  // derived per tile
        f32x16 s[1] = {f32x16{}};
#pragma unroll
        for (int k0 = 0; k0 < kNKK; k0 += kBatch) {
            X8 kf[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                kf[i] = *reinterpret_cast<const X8*>(stage + (kXorOff ? kb ^ (32 * (k0 + i)) : koff[k0 + i]));
            if constexpr (Cfg::kOrder) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kBatch; ++i) s[0] = E::mfma32(kf[i], q[k0 + i], s[0]);
        }
        X8 vf[kAhead > 0 ? kAhead : 1][2];
#pragma unroll
        for (int td = 0; td < kAhead; ++td)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) vf[td][jj] = v_frag(stage, vb, td, jj);
        if constexpr (Cfg::kOrder) __builtin_amdgcn_sched_barrier(0);
        if ((t + 1) * BC > wave_min) {      // keys that a row does not see -> -inf
            asm volatile("" ::: "memory");  // a branch, not selects in every tile
            const int lg = lim - t * BC - 4 * g;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (8 * (r >> 2) + (r & 3) >= lg) s[0][r] = -INFINITY;
        }
        X8 pp[2];
        block_update_max<kNTD>(st, block_rowmax<1>(s), c, inv_c, o);
        // A row that has seen no key yet keeps m = -inf and must get P = 0, not NaN.
        packed_exp<kBF>(s[0], c, st.m == -INFINITY ? 0.f : -st.m, pp, st.l);
#pragma unroll
        for (int td = 0; td < kNTD; ++td)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj)
                o[td] = E::mfma32(td < kAhead ? vf[td < kAhead ? td : 0][jj] : v_frag(stage, vb, td, jj), pp[jj], o[td]);
    };
    for (int t0 = 0; t0 < ntiles; t0 += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int t = t0 + u;
            if (t >= ntiles) break;
            char* cur = u == 0 ? b0 : b1;
            char* nxt = u == 0 ? b1 : b0;
            // Stage t has landed for every wave; every wave is done with
            // stage t - 1 (in nxt).
            if constexpr (Cfg::kAsmCopy) {
                // (A wait that the compiler sees, so that the first tile's loads
                // of Q do not make it wait for a stage in every tile.)
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
            }
            if (t + 1 < ntiles) issue_stage(nxt, (t + 1) * BC);
            tile(cur, t);
        }
    }
    if constexpr (KS > 1) {
        // Merge slot k: 1 KiB of the then free stage buffers.
        static_assert(kRowWaves * kNTD * 4 * (KS - 1) * 1024 <= 2 * kBuf, "merge slots");
        __shared__ float merge_ml[2 * NW * 64];
        const auto slot_base = [&](int k) { return k < kBuf / 1024 ? buf0 + k * 1024 : buf1 + (k * 1024 - kBuf); };
        merge_kv_groups<D, KS, kRowWaves>(p, st, o, slot_base, merge_ml, wave, kgrp, lane, g, out_row(), 0,
                                          (lane & 31) < nrows);
        return;
    }
    __syncthreads();  // every wave is done with the stages
    char* const mine = (wave_id < NW / 2 ? buf0 : buf1) + wave_id % (NW / 2) * (2 * kBuf / NW);
    const float l = sum_xor32(st.l);
    const bool empty = !(l > 0.f);                        // causal: no visible key
    const float inv = empty ? 0.f : 1.0f / l;
    const int at = out_row();
    if (p.out_dtype == kOutF16)
        packed_store<kOutF16, D, 2 * kBuf / NW>(p, o, inv, mine, at, nrows, lane);
    else if (p.out_dtype == kOutBF16)
        packed_store<kOutBF16, D, 2 * kBuf / NW>(p, o, inv, mine, at, nrows, lane);
    else
        packed_store<kOutF32, D, 2 * kBuf / NW>(p, o, inv, mine, at, nrows, lane);
    if (g == 0 && (lane & 31) < nrows)
        store_stats(p, at, st.rmax * p.scale, empty ? 0.f : l * rebase_factor(st.m, st.rmax, c));
}

}  // namespace kf
