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
#pragma once

#include "elem.h"

namespace kf {

struct PackedParams : AttnParams {  // Q, K, V, O, Mi (LSE), scales, causal, heads_kv, out_dtype, xcds
    long long q_token, k_token, v_token;  // strides in elements
    long long q_head, k_head, v_head;
    const int* q_starts;                  // [n_seqs + 1]
    const int* k_starts;
    int n_seqs, tokens_q, tokens_k, ratio;
};

template <int D, int NW, int RB> struct PackedCfg {
    static constexpr int kThreads = 64 * NW;
    static constexpr int kRows = 32 * RB * NW;            // query rows per workgroup
    static constexpr int BC = 32;                         // keys per MFMA tile
    static constexpr int kStageRows = D >= 256 ? 32 : 64; // keys per LDS stage
    static constexpr bool kQ1Lds = RB == 2 && D == 128;   // block-1 Q^T read from LDS
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
// last.  Up to 64 sequences (one to a lane) the tiles are numbered by
// their keys, longest first: the dispatcher starts workgroups in order, and
// short tiles then fill the CUs that finish early.  A tile's level is its
// keys in units of a tile's rows, up to a constant: consecutive for
// the tiles of a causal sequence, the same for all of one that is not.  More
// sequences, of which any order spreads the work, are numbered one after the other.
template <int kRows>
__device__ __forceinline__ bool packed_find(const PackedParams& p, int lane, int j, int& seq, int& tile) {
    const auto tiles_of = [&](const PackedSeq& s) { return (int)(((long long)s.qn * p.ratio + kRows - 1) / kRows); };
    if (p.n_seqs <= 64) {
        PackedSeq s{0, 0, 0, 0};
        if (lane < p.n_seqs) s = packed_seq(p, lane);
        const int n = tiles_of(s);
        const int low = (int)((long long)max(p.causal ? s.kn - s.qn : s.kn, 0) * p.ratio / kRows);
        const auto from = [&](int k) {   // this lane's tiles of level k or more
            return p.causal ? min(max(low + n - k, 0), n) : low >= k ? n : 0;
        };
        if (__builtin_amdgcn_readlane(wave_scan(n), 63) <= j) return false;
        // The largest level of which, with those above it, there are more than j.
        int lo = 0, hi = low + n + 1;    // hi: none from there on, once it is the wave's largest
#pragma unroll
        for (int m = 1; m < 64; m *= 2) hi = max(hi, __shfl_xor(hi, m));
        hi = __builtin_amdgcn_readfirstlane(hi);
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (__builtin_amdgcn_readlane(wave_scan(from(mid)), 63) > j) lo = mid; else hi = mid;
        }
        const int above = __builtin_amdgcn_readlane(wave_scan(from(lo + 1)), 63);
        const int here = from(lo) - from(lo + 1);
        const int inc = wave_scan(here);
        const uint64_t mine = __ballot(inc > j - above);
        seq = __builtin_ctzll(mine);
        tile = p.causal ? lo - __builtin_amdgcn_readlane(low, seq)
                        : j - above - (__builtin_amdgcn_readlane(inc, seq) - __builtin_amdgcn_readlane(here, seq));
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

// exp2 and 16-bit pack of a 32-row score block; the fp32 values are summed, so
// that the log-sum-exp has their precision.
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

template <bool kBF, int D, int NW, int RB>
__global__ __launch_bounds__((PackedCfg<D, NW, RB>::kThreads), 2)
void kf_attn_packed_kernel(PackedParams p) {
    using Cfg = PackedCfg<D, NW, RB>;
    using E = Elem<kBF>;
    using X8 = typename E::x8;
    using SW = SwizzleRow<D>;
    constexpr int BC = Cfg::BC, SR = Cfg::kStageRows, kRows = Cfg::kRows;
    constexpr int kRowBytes = D * 2, kChunks = D / 8, kRowsPerInstr = 1024 / kRowBytes;
    constexpr int kInstr = SR * kRowBytes / 1024;         // LDS-DMA instructions per tensor and stage
    constexpr int kTensorBytes = SR * kRowBytes;
    constexpr int kPerWave = 2 * kInstr / NW;
    static_assert(2 * kInstr % NW == 0 && kInstr % kPerWave == 0, "a wave copies K or V");
    constexpr int kNKK = D / 16, kNTD = D / 32;
    constexpr bool kQ1Lds = Cfg::kQ1Lds;
    __shared__ __attribute__((aligned(1024))) char buf0[2 * kTensorBytes];
    __shared__ __attribute__((aligned(1024))) char buf1[2 * kTensorBytes];
    __shared__ __attribute__((aligned(256))) char q1_lds[kQ1Lds ? NW * 32 * kRowBytes : 16];

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
    // Causal: waves w and w + 4 share a SIMD; blocks w and 7 - w.
    const int wave = (NW == 8 && p.causal && wave_id >= 4) ? 11 - wave_id : wave_id;
    const auto limit = [&](int row) {  // keys that the row sees
        return p.causal ? min(max(row / ratio + klen - sq.qn + 1, 0), klen) : klen;
    };
    const int r0 = rt * kRows, w0 = r0 + wave * 32 * RB;
    const int blk_lim = limit(min(R, r0 + kRows) - 1);
    const int wave_min = w0 < R ? limit(w0) : blk_lim;
    const int wave_max = w0 < R ? limit(min(R, w0 + 32 * RB) - 1) : 0;
    const int ntiles = (blk_lim + BC - 1) / BC;
    const int nstages = (blk_lim + SR - 1) / SR;
    const int nt_w = (wave_max + BC - 1) / BC;            // the wave's tiles; it skips the others

    int rows[RB], lim[RB];
    size_t out_row[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        rows[b] = w0 + 32 * b + (lane & 31);
        const int rc = min(rows[b], R - 1);               // rows past R compute on it, unstored
        lim[b] = limit(rc);
        out_row[b] = ((size_t)(sq.q0 + rc / ratio) * p.heads_kv + hk) * ratio + rc % ratio;
    }
    if (ntiles == 0) {                                    // no key for any row
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            if (rows[b] >= R) continue;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) store_out4(p, out_row[b] * D + 8 * i + 4 * g, f32x4{0.f, 0.f, 0.f, 0.f});
            if (g == 0) store_stats(p, out_row[b], -INFINITY, 0.f);
        }
        return;
    }

    const char* Kh = reinterpret_cast<const char*>(p.K + (size_t)sq.k0 * p.k_token + (size_t)hk * p.k_head);
    const char* Vh = reinterpret_cast<const char*>(p.V + (size_t)sq.k0 * p.v_token + (size_t)hk * p.v_head);
    // LDS-DMA: wave w copies the KiB instructions w kPerWave + i of the
    // stage, all of K or all of V.  Lane l of one fills row l / kChunks of
    // its rows, physical chunk l % kChunks.
    const bool is_v = wave_id * kPerWave >= kInstr;
    const char* src = is_v ? Vh : Kh;
    const size_t row_stride = 2 * (size_t)(is_v ? p.v_token : p.k_token);
    const int ii0 = wave_id * kPerWave % kInstr;
    const int lr = lane / kChunks;
    auto issue_stage = [&](char* dst, int kv0) {
        char* d = dst + (is_v ? kTensorBytes : 0) + ii0 * 1024;
#pragma unroll
        for (int i = 0; i < kPerWave; ++i) {
            const int r = (ii0 + i) * kRowsPerInstr + lr;
            const int kv = min(kv0 + r, klen - 1);        // rows past the keys re-read the last
            const char* a = src + (size_t)kv * row_stride + (((lane % kChunks) ^ SW::h(r)) % kChunks) * 16;
            __builtin_amdgcn_global_load_lds(a, (lds_void*)(d + i * 1024), 16, 0, 0);
        }
    };

    // LDS reads, as in the prefill kernels.
    // (With D >= 128's swizzle the offset of k-step kk is that of the first ^ 32 kk,
    // of V^T tile td ^ 64 td, of its second 8 rows ^ 128 and 8 rows on: derived
    // at each tile where registers for them are short.)
    constexpr bool kXorOff = D >= 256;
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

    issue_stage(buf0, 0);
    X8 q[RB == 2 && !kQ1Lds ? 2 : 1][kNKK];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int rc = min(rows[b], R - 1);
        const uint16_t* Qr = p.Q + (size_t)(sq.q0 + rc / ratio) * p.q_token + (size_t)(hk * ratio + rc % ratio) * p.q_head;
#pragma unroll
        for (int kk = 0; kk < kNKK; ++kk) {
            const X8 v = *reinterpret_cast<const X8*>(Qr + (2 * kk + g) * 8);
            if (kQ1Lds && b == 1)
                *reinterpret_cast<X8*>(q1_lds + wave * 32 * kRowBytes + koff[kk]) = v;
            else
                q[b][kk] = v;
        }
    }
    const char* q1w = q1_lds + wave * 32 * kRowBytes;

    RowState st[RB];
    f32x16 o[RB][kNTD];
    const float inv_c = 1.0f / c;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        st[b] = RowState{-INFINITY, -INFINITY, 0.f, -INFINITY};
#pragma unroll
        for (int td = 0; td < kNTD; ++td) o[b][td] = f32x16{};
    }
    auto tile = [&](const char* stage, int t) {
        if (t >= nt_w) return;
        f32x16 s[RB][1];
#pragma unroll
        for (int b = 0; b < RB; ++b) s[b][0] = f32x16{};
        int kb = koff[0], vb = voff[0][0];
        if constexpr (kXorOff) asm volatile("" : "+v"(kb), "+v"(vb));  // derived per tile
#pragma unroll
        for (int kk = 0; kk < kNKK; ++kk) {
            const X8 kf = *reinterpret_cast<const X8*>(stage + (kXorOff ? kb ^ (32 * kk) : koff[kk]));
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                if (kQ1Lds && b == 1)
                    s[b][0] = E::mfma32(kf, *reinterpret_cast<const X8*>(q1w + koff[kk]), s[b][0]);
                else
                    s[b][0] = E::mfma32(kf, q[b][kk], s[b][0]);
            }
        }
        if ((t + 1) * BC > wave_min) {
            asm volatile("" ::: "memory");  // a branch, not selects in every tile
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const int lg = lim[b] - t * BC - 4 * g;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (8 * (r >> 2) + (r & 3) >= lg) s[b][0][r] = -INFINITY;
            }
        }
        X8 pp[RB][2];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            block_update_max<kNTD>(st[b], block_rowmax<1>(s[b]), c, inv_c, o[b]);
            packed_exp<kBF>(s[b][0], c, st[b].m == -INFINITY ? 0.f : -st[b].m, pp[b], st[b].l);
        }
#pragma unroll
        for (int td = 0; td < kNTD; ++td) {
            const int vo0 = kXorOff ? vb ^ (64 * td) : voff[td][0];
            const int vo1 = kXorOff ? (vb ^ (64 * td) ^ 128) + 8 * kRowBytes : voff[td][1];
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                const f16x4 lo = lds_read_tr16(stage + vo0 + jj * 16 * kRowBytes);
                const f16x4 hi = lds_read_tr16(stage + vo1 + jj * 16 * kRowBytes);
                const X8 a = __builtin_bit_cast(X8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int b = 0; b < RB; ++b) o[b][td] = E::mfma32(a, pp[b][jj], o[b][td]);
            }
        }
    };
    constexpr int kSub = SR / BC;
    for (int js = 0; js < nstages; js += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int j = js + u;
            if (j >= nstages) break;
            char* cur = u == 0 ? buf0 : buf1;
            char* nxt = u == 0 ? buf1 : buf0;
            // Stage j has landed for every wave; every wave is done with
            // stage j - 1 (in nxt).
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (j + 1 < nstages) issue_stage(nxt, (j + 1) * SR);
            tile(cur, kSub * j);
            if (kSub == 2 && 2 * j + 1 < ntiles) tile(cur + BC * kRowBytes, 2 * j + 1);
        }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const float l = sum_xor32(st[b].l);
        if (rows[b] >= R) continue;
        const bool empty = !(l > 0.f);                    // causal: no visible key
        store_o_row_any<D>(p, out_row[b], o[b], empty ? 0.f : 1.0f / l, g);
        if (g == 0)
            store_stats(p, out_row[b], st[b].rmax * p.scale,
                        empty ? 0.f : l * rebase_factor(st[b].m, st[b].rmax, c));
    }
}

}  // namespace kf
