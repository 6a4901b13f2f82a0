// paged_kernels.h -- attention of packed new tokens over a paged 16-bit K/V cache,
// and the attention weight that each of its keys gathers.
//
// Pools are [num_pages][H_kv][page_size][D] (attn_decode_paged's); sequence b's new
// tokens are the packed ones q_starts[b] .. q_starts[b + 1] - 1 and the last of its
// kv_lens[b] keys.  The query rows that read a KV head are (token, head of its group),
// token major: row r of a sequence is query r / ratio of group head r % ratio.
#pragma once

#include <cfloat>

#include "elem.h"
#include "packed_kernels.h"

namespace kf {

struct PagedParams : AttnParams {  // Q, K, V, O, Mi (LSE), scales, causal, heads_kv, out_dtype, pages, kv_lens
    long long q_token, q_head;     // strides in elements
    const int* q_starts;           // [n_seqs + 1]
    int n_seqs, tokens_q, ratio;
    // Tiles are cut into parts where there are too few of them for the device (see
    // paged_find): `target` parts of a KV head are aimed at (0: no cuts), none smaller
    // than min_share units.
    int target, min_share, unit_shift;
    const uint32_t* row_lse;       // kf_kv_weigh: [tokens_q][H_q], bits of fp32
    float* weights;                // kf_kv_weigh: [num_pages][H_kv][page_size]
    int cut;                       // where shares cut a line: whether they cut tiles of it, too
};

// One sequence's new tokens and keys.
struct PagedSeq {
    int q0, qn, kn;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int i) {
    PagedSeq s;
    s.q0 = min(max(p.q_starts[i], 0), p.tokens_q);
    s.qn = min(max(p.q_starts[i + 1], s.q0), p.tokens_q) - s.q0;
    s.kn = min(max(p.kv_lens[i], 0), p.kv_len);
    return s;
}

// The work of a sequence in a KV head: tiles, and how many units each could be cut into.
struct PagedCount {
    int tiles, units;
};
// Attention: tiles of kRows query rows, units of 32 << unit_shift keys.
template <int kRows>
__device__ __forceinline__ PagedCount paged_count(const PagedParams& p, int i) {
    const PagedSeq s = paged_seq(p, i);
    return PagedCount{(int)(((long long)s.qn * p.ratio + kRows - 1) / kRows),
                      (key_stages(s.kn) + (1 << p.unit_shift) - 1) >> p.unit_shift};
}

// A part of a tile: its sequence, tile and part in it, of how many, and, where there
// are several, the partial that it writes.
struct PagedItem {
    int seq, tile, part, parts, slot;
};

// Item j of a KV head, by the lanes of a wave; false past the last.  Every tile of a
// sequence has the same number of parts, so many that one has at most `share`
// units; `share` is the work of all tiles over p.target.  So no more than target + tiles
// parts come out, and 2 target of tiles that are cut: more than one part means more
// than `share` units, and fewer than twice as many parts as shares.  Up to 64 sequences have a
// lane each, of more a lane has a run of consecutive ones.  kCut: j counts the tiles
// that are cut, not the parts; of the parts, a sequence's last tiles, which see the most keys, come first.
// Of starts in no order the counts have no bound: a lane's stop at kFindMost, which no j reaches (a grid
// has less than 2^32 threads, 256 a workgroup), so that all in front of an item that is found are exact.
constexpr int kFindMost = 1 << 24;
template <bool kCut, class CountOf>
__device__ __forceinline__ bool paged_find(const PagedParams& p, int lane, int j, PagedItem& it, const CountOf& count) {
    using Count = PagedCount;
    const int per = (p.n_seqs + 63) / 64, first = min(lane * per, p.n_seqs), last = min(first + per, p.n_seqs);
    Count mine{0, 0};
    if (per == 1 && first < last) mine = count(first);
    int share = 0;
    if (p.target > 0) {
        unsigned sum = (unsigned)mine.tiles * (unsigned)mine.units;
        if (per > 1)
            for (int i = first; i < last; ++i) {
                const Count c = count(i);
                sum += (unsigned)c.tiles * (unsigned)c.units;
            }
        const unsigned total = (unsigned)__builtin_amdgcn_readlane(wave_scan((int)sum), 63);
        share = max((int)((total + (unsigned)p.target - 1u) / (unsigned)p.target), p.min_share);
    }
    const auto parts_of = [&](const Count& c) { return share > 0 ? max((c.units + share - 1) / share, 1) : 1; };
    const auto all_parts = [](const Count& c, int parts) { return (int)min((long long)c.tiles * parts, (long long)kFindMost); };
    const auto items_of = [&](const Count& c, int parts) { return kCut ? (parts > 1 ? c.tiles : 0) : all_parts(c, parts); };
    const auto slots_of = [&](const Count& c, int parts) { return parts > 1 ? all_parts(c, parts) : 0; };
    int parts = parts_of(mine), items = items_of(mine, parts), slots = slots_of(mine, parts);
    if (per > 1) {
        items = slots = 0;
        for (int i = first; i < last; ++i) {
            const Count c = count(i);
            parts = parts_of(c);
            items = min(items + items_of(c, parts), kFindMost);
            slots = min(slots + slots_of(c, parts), kFindMost);
        }
    }
    const int inc = wave_scan(items), slot_inc = wave_scan(slots);
    const uint64_t past = __ballot(inc > j);
    if (past == 0) return false;
    const int run = __builtin_ctzll(past);
    int left = j - (__builtin_amdgcn_readlane(inc, run) - __builtin_amdgcn_readlane(items, run));
    long long slot = __builtin_amdgcn_readlane(slot_inc, run) - __builtin_amdgcn_readlane(slots, run);
    int tiles;
    if (per == 1) {
        it.seq = run;
        it.parts = __builtin_amdgcn_readlane(parts, run);
        tiles = __builtin_amdgcn_readlane(mine.tiles, run);
    } else {
        const int end = min((run + 1) * per, p.n_seqs);
        for (int i0 = run * per;; i0 += 64) {
            if (i0 >= end) return false;  // not reached
            mine = i0 + lane < end ? count(i0 + lane) : Count{0, 0};
            parts = parts_of(mine);
            items = items_of(mine, parts);
            slots = slots_of(mine, parts);
            const int in = wave_scan(items), sl = wave_scan(slots);
            const uint64_t over = __ballot(in > left);
            if (over != 0) {
                const int at = __builtin_ctzll(over);
                it.seq = i0 + at;
                it.parts = __builtin_amdgcn_readlane(parts, at);
                tiles = __builtin_amdgcn_readlane(mine.tiles, at);
                left -= __builtin_amdgcn_readlane(in, at) - __builtin_amdgcn_readlane(items, at);
                slot += __builtin_amdgcn_readlane(sl, at) - __builtin_amdgcn_readlane(slots, at);
                break;
            }
            left -= __builtin_amdgcn_readlane(in, 63);
            slot += __builtin_amdgcn_readlane(sl, 63);
        }
    }
    if (kCut) {
        it.part = 0;
        it.tile = left;
    } else {
        it.part = left % it.parts;
        it.tile = tiles - 1 - left / it.parts;
    }
    slot += (long long)it.tile * it.parts + it.part;
    it.slot = (int)slot;
    // (Of starts in no order there may be more partials than the workspace holds.)
    return it.parts == 1 || slot + (kCut ? it.parts : 1) <= 2LL * p.target;
}

// The work of a KV head as a line of units, its sequences one after the other, of which every
// workgroup has an equal share.  Share j: from unit u0 of the line on to u1; the sequence
// of u0 and its place among the sequence's units.  By the lanes of a wave; false past the last
// unit.  (A sequence has at most 2^52 units, rows and keys being ints; of starts in no order a lane's
// stop at kLineMost, so that 64 of them do not pass 63 bits.)
constexpr long long kLineMost = 1LL << 56;
struct LineShare {
    long long u0, u1, share, at;
    int seq;
};
__device__ __forceinline__ long long line_scan(long long v, int lane) {
    if (__all(v < 1 << 24)) return wave_scan((int)v);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
__device__ __forceinline__ long long line_lane(long long v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
    return (long long)((uint64_t)hi << 32 | lo);
}
// a / b, a not negative, mostly by 32 bits.
__device__ __forceinline__ long long line_div(long long a, int b) {
    return a < INT_MAX ? (int)((unsigned)a / (unsigned)b) : a / b;
}
template <class UnitsOf>
__device__ __forceinline__ bool line_find(const PagedParams& p, int lane, int j, LineShare& w, const UnitsOf& units_of) {
    const int per = (p.n_seqs + 63) / 64, first = min(lane * per, p.n_seqs), last = min(first + per, p.n_seqs);
    long long mine = 0;
    for (int i = first; i < last; ++i) mine = min(mine + units_of(i), kLineMost);
    long long inc = line_scan(mine, lane);
    const long long total = line_lane(inc, 63);
    w.share = max(line_div(total + p.target - 1, p.target), (long long)p.min_share);
    w.u0 = j * w.share;
    w.u1 = min(w.u0 + w.share, total);
    if (w.u0 >= total) return false;
    const int run = __builtin_ctzll(__ballot(inc > w.u0));
    w.at = w.u0 - (line_lane(inc, run) - line_lane(mine, run));
    w.seq = run;
    if (per == 1) return true;
    const int end = min((run + 1) * per, p.n_seqs);
    for (int i0 = run * per; i0 < end; i0 += 64) {
        mine = i0 + lane < end ? units_of(i0 + lane) : 0;
        inc = line_scan(mine, lane);
        const uint64_t over = __ballot(inc > w.at);
        if (over != 0) {
            const int at = __builtin_ctzll(over);
            w.seq = i0 + at;
            w.at -= line_lane(inc, at) - line_lane(mine, at);
            return true;
        }
        w.at -= line_lane(inc, 63);
    }
    return false;  // not reached
}
// Where share `share` begins inside a tile, `in_front` of whose units lie in front of it and `behind`
// from it on, and is the first that does: how many parts the tile has, else 0.  The
// parts' slots: the last one of the share in front, the first of this and the later ones.
__device__ __forceinline__ int line_parts(const LineShare& w, long long in_front, long long behind) {
    if (in_front <= 0 || in_front > w.share) return 0;
    return 1 + (int)((behind + w.share - 1) / w.share);
}
__device__ __forceinline__ int line_slot(int share, int k) { return k == 0 ? 2 * share - 1 : 2 * (share + k - 1); }

// Attention of tiles of 32 rows: every tile of a sequence has its 32-key stages, and what
// starting on one costs, as units (32 contexts of 512 to 8192 keys, 32 / 8 heads of 128, 80 us with
// none, 74, 69 and 66 with 3, 6 and 12; 64 of 16 to 512 39, 29, 28 and 27; with up to 8 tokens over 64
// to 1024 33, 28, 26 and 26).
constexpr int kLineStart = 6;
__device__ __forceinline__ int line_stages(const PagedSeq& s) { return kLineStart + key_stages(s.kn); }
__device__ __forceinline__ long long line_units(const PagedParams& p, int i) {
    const PagedSeq s = paged_seq(p, i);
    return ((long long)s.qn * p.ratio + 31) / 32 * line_stages(s);
}

// Chunks are bound by the matrix unit and the softmax, which overlap in part only: 4 x 512
// tokens over 8192 keys, 32 / 8 heads of 128, 327 us, 866 TFLOPS, 2048 over 65536 at D = 256 2100 us,
// 1064.  Steps wait half of their cycles and read at 5.4 TB/s (32 contexts of 512 to 8192 keys), the
// matrix unit is busy for 6 %.
// A workgroup is NW waves of 32 query rows each; with KS > 1 they form KS groups that
// take the same rows and a share of the keys each, merged through LDS at the end.
template <int D, int NW, int KS> struct PagedCfg {
    static constexpr int kThreads = 64 * NW;
    static constexpr int kRowWaves = NW / KS;             // waves per KV group
    static constexpr int kRows = 32 * kRowWaves;          // query rows per workgroup
    static constexpr int BC = 32;                         // keys per MFMA tile and LDS stage
    // Waves per SIMD that the registers have to allow.
    static constexpr int kWavesPerSimd =
        D == 64 ? (KS == 4 ? 2 : 4) : D == 128 ? (KS == 1 ? 3 : KS == 2 ? 2 : 1) : KS == 1 ? 2 : 1;
};

// What a masked key's V row is read from, so that its weight 0 meets finite values: 16
// rows of zeros.
static __device__ const u32x4 paged_zeros[16 * 256 * 2 / 16] = {};

// One tile, or the part of it from stage s0 on to s1 (of a line's: else those of it.part).
template <bool kBF, int D, int NW, int KS>
__device__ __forceinline__ void paged_tile(const PagedParams& p, const PagedItem& it, int hk, int lane, int line_s0,
                                           int line_s1) {
    using Cfg = PagedCfg<D, NW, KS>;
    using E = Elem<kBF>;
    using X8 = typename E::x8;
    using SW = SwizzleRow<D>;
    constexpr int BC = Cfg::BC, kRows = Cfg::kRows, kRowWaves = Cfg::kRowWaves;
    constexpr int kRowBytes = D * 2, kChunks = D / 8, kRowsPerInstr = 1024 / kRowBytes;
    constexpr int kTensorBytes = BC * kRowBytes;
    // A unit of copying: 16 rows of K or V, which lie in one page.
    constexpr int kUnitInstr = 16 / kRowsPerInstr, kUnitsPerWave = 4 / kRowWaves;
    static_assert(kRowWaves == 1 || kRowWaves == 2 || kRowWaves == 4, "whole units");
    constexpr int kNKK = D / 16, kNTD = D / 32;
    constexpr int kBuf = KS * 2 * kTensorBytes;           // a stage of every group
    __shared__ __attribute__((aligned(1024))) char buf0[kBuf];
    __shared__ __attribute__((aligned(1024))) char buf1[kBuf];

    const int wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 5;
    PagedSeq sq = paged_seq(p, it.seq);
    sq.q0 = __builtin_amdgcn_readfirstlane(sq.q0);
    sq.qn = __builtin_amdgcn_readfirstlane(sq.qn);
    sq.kn = __builtin_amdgcn_readfirstlane(sq.kn);
    const int ratio = p.ratio, R = sq.qn * ratio, klen = sq.kn, sh = p.page_shift;
    const float c = p.scale_log2;
    const int wave = KS > 1 ? wave_id % kRowWaves : wave_id;
    const int kgrp = KS > 1 ? wave_id / kRowWaves : 0;
    if ((unsigned)it.tile * (unsigned)kRows >= (unsigned)R) return;   // not reached
    const auto limit = [&](int row) {  // keys that the row sees
        return p.causal ? min(max(klen - sq.qn + row / ratio + 1, 0), klen) : klen;
    };
    const int r0 = it.tile * kRows, w0 = r0 + wave * 32;
    const int blk_lim = limit(min(R, r0 + kRows) - 1);
    // This part's stages of those that the tile sees, and the groups' of these, as many
    // as any other's; row limits count from kv_base.
    const int seen = key_stages(blk_lim), per_part = (seen + it.parts - 1) / it.parts;
    const int s0 = min(kRows == 32 ? line_s0 : it.part * per_part, seen);
    const int s1 = min(kRows == 32 ? line_s1 : s0 + per_part, seen);
    const int ntiles = (s1 - s0 + KS - 1) / KS;
    const int kv_base = (s0 + kgrp * ntiles) * BC, kv_end = min(min(kv_base + ntiles * BC, s1 * BC), blk_lim);
    const auto own = [&](int lim) { return min(lim, kv_end) - kv_base; };
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
    // The partial of this lane's row.
    const auto part_row = [&]() {
        return ((size_t)it.slot * p.heads_kv + hk) * kRows + wave * 32 + (lane & 31);
    };
    if (ntiles == 0) {                                    // no key for any row
        if ((lane & 31) < nrows && kgrp == 0) {
            if (it.parts > 1) {
                if (g == 0) {
                    p.Mpart[part_row()] = -INFINITY;
                    p.Lpart[part_row()] = 0.f;
                }
            } else {
                const int at = out_row();
#pragma unroll
                for (int i = 0; i < D / 8; ++i) store_out4(p, (size_t)at * D + 8 * i + 4 * g, f32x4{0.f, 0.f, 0.f, 0.f});
                if (g == 0) store_stats(p, at, -INFINITY, 0.f);
            }
        }
        return;
    }

    // The ids of 64 pages from page0 on, one to a lane; stages come in order.
    const int* const table = p.block_table + (size_t)it.seq * p.max_pages;
    int page0 = kv_base >> sh;
    int ids = table[min(page0 + lane, p.max_pages - 1)];
    auto page_of = [&](int key) {                         // of a key below klen
        if ((key >> sh) - page0 >= 64) {
            page0 = key >> sh;
            ids = table[min(page0 + lane, p.max_pages - 1)];
        }
        return __builtin_amdgcn_readlane(ids, (key >> sh) - page0);
    };
    const char* const Kp = reinterpret_cast<const char*>(p.K);
    const char* const Vp = reinterpret_cast<const char*>(p.V);
    // LDS-DMA: lane l of an instruction fills row l / kChunks of its rows, physical chunk
    // l % kChunks.  The swizzle depends on row & 15: the units' lane offsets are alike.
    const int copier = wave_id % kRowWaves;
    const int lr = lane / kChunks;
    uint32_t chunk_off[kUnitInstr];
#pragma unroll
    for (int i = 0; i < kUnitInstr; ++i)
        chunk_off[i] = (((lane % kChunks) ^ SW::h(i * kRowsPerInstr + lr)) % kChunks) * 16;
    // Requests the stage that begins at key kv_base + kv0; returns which of its halves lie on
    // no valid page, bit 0 keys 0 .. 15, bit 1 the others.
    // kWhat: 1 K, 2 V, 3 both.
    auto issue_stage = [&](char* dst, int kv0, auto what) {
        constexpr int kWhat = decltype(what)::value;
        const int kv = kv_base + kv0;
        int id[2], bad = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            id[h] = kv + 16 * h < klen ? page_of(kv + 16 * h) : -1;
            bad |= (unsigned)id[h] < (unsigned)p.num_pages ? 0 : 1 << h;
        }
#pragma unroll
        for (int u = 0; u < kUnitsPerWave; ++u) {
            const int unit = copier * kUnitsPerWave + u, h = unit & 1;
            const bool is_v = unit >= 2;
            if (kRowWaves == 1 && (kWhat >> (u >> 1) & 1) == 0) continue;
            const uint32_t d_lds = (uint32_t)(uintptr_t)(lds_void*)(dst + unit * (kTensorBytes / 2));
            const int key = kv + 16 * h;
            const int page = h ? id[1] : id[0];
            const bool ok = (bad >> h & 1) == 0;
            const size_t row = (((size_t)(ok ? page : 0) * p.heads_kv + hk) << sh) + (key & ((1 << sh) - 1));
            const char* src = (is_v ? Vp : Kp) + row * kRowBytes;
            if (!ok) src = reinterpret_cast<const char*>(paged_zeros);
            if (!ok || key + 16 <= klen) {
#pragma unroll
                for (int i = 0; i < kUnitInstr; ++i)
                    lds_copy16(d_lds + i * 1024, src + i * 1024, lr * kRowBytes + chunk_off[i]);
            } else {
                // Rows past the keys re-read the last one (finite data whose scores are masked).
#pragma unroll
                for (int i = 0; i < kUnitInstr; ++i)
                    lds_copy16(d_lds + i * 1024, src, min(i * kRowsPerInstr + lr, klen - 1 - key) * kRowBytes + chunk_off[i]);
            }
        }
        return bad;
    };

    // LDS reads, as in the packed kernel.
    constexpr bool kXorOff = D >= 128;
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
    constexpr std::integral_constant<int, 1> kK{};
    constexpr std::integral_constant<int, 2> kV{};
    constexpr std::integral_constant<int, 3> kBoth{};
    int bad_next = issue_stage(b0, 0, kBoth);
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
    // S of a tile, masked and rebased to the running maximum, and then O.
    f32x16 s[1];
    const auto scores = [&](const char* stage) {
        int kb = koff[0];
        if constexpr (kXorOff) asm volatile("" : "+v"(kb));  // derived per tile
        s[0] = f32x16{};
#pragma unroll
        for (int kk = 0; kk < kNKK; ++kk) {
            const X8 kf = *reinterpret_cast<const X8*>(stage + (kXorOff ? kb ^ (32 * kk) : koff[kk]));
            s[0] = E::mfma32(kf, q[kk], s[0]);
        }
    };
    X8 pp[2];
    const auto weights = [&](int t, int bad) {
        if ((t + 1) * BC > wave_min || bad != 0) {      // keys that a row does not see -> -inf
            asm volatile("" ::: "memory");              // a branch, not selects in every tile
            const int lg = lim - t * BC - 4 * g;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (8 * (r >> 2) + (r & 3) >= lg || (bad >> (r >> 3) & 1)) s[0][r] = -INFINITY;
        }
        block_update_max<kNTD>(st, block_rowmax<1>(s), c, inv_c, o);
        // A row that has seen no key yet keeps m = -inf and must get P = 0, not NaN.
        packed_exp<kBF>(s[0], c, st.m == -INFINITY ? 0.f : -st.m, pp, st.l);
    };
    const auto outputs = [&](const char* stage) {
        int vb = voff[0][0];
        if constexpr (kXorOff) asm volatile("" : "+v"(vb));
#pragma unroll
        for (int td = 0; td < kNTD; ++td)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) o[td] = E::mfma32(v_frag(stage, vb, td, jj), pp[jj], o[td]);
    };
    if constexpr (kRowWaves == 1) {
        // The wave copies its stages itself and waits for itself alone: K of the stage after the
        // next as soon as this one's has been read, and V likewise (64 contexts of 2048 keys,
        // 32 / 8 heads of 128: 112 us with one stage on its way, 108 so).  As compiled, a
        // stage's first products also wait for q's loads, and page ids for their own, by the
        // counter that all copies are in, so that fewer than three of four half stages are.
        constexpr int kHalf = 2 * kUnitInstr;             // copies of K or V of a stage
        const auto landed = [](int halves) {              // but for so many younger halves
            asm volatile("" ::: "memory");
            const auto wait = [](auto n) {
                constexpr int v = decltype(n)::value * kHalf;
                static_assert(v < 64, "vmcnt");
                __builtin_amdgcn_s_waitcnt(0x0f70 | (v & 15) | (v >> 4) << 14);
            };
            if (halves == 3) wait(std::integral_constant<int, 3>{});
            else if (halves == 2) wait(std::integral_constant<int, 2>{});
            else if (halves == 1) wait(std::integral_constant<int, 1>{});
            else wait(std::integral_constant<int, 0>{});
            asm volatile("" ::: "memory");
        };
        const auto read = [] {                            // all LDS reads have returned
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xc07f);
            asm volatile("" ::: "memory");
        };
        int bad = bad_next;
        if (ntiles > 1) bad_next = issue_stage(b1, BC, kBoth);
        for (int t = 0; t < ntiles; ++t) {
            char* const stage = t & 1 ? b1 : b0;
            const int later = min(ntiles - 1 - t, 2);     // stages behind this one, up to two
            int bad_after = 0;
            landed(later > 0 ? 3 : 1);
            if (t < nt_w) scores(stage);
            read();
            if (later > 1) bad_after = issue_stage(stage, (t + 2) * BC, kK);
            if (t < nt_w) weights(t, bad);
            landed(later == 0 ? 0 : later + 1);
            if (t < nt_w) outputs(stage);
            read();
            if (later > 1) issue_stage(stage, (t + 2) * BC, kV);
            bad = bad_next;
            bad_next = bad_after;
        }
    } else {
        for (int t0 = 0; t0 < ntiles; t0 += 2) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int t = t0 + u;
                if (t >= ntiles) break;
                char* cur = u == 0 ? b0 : b1;
                char* nxt = u == 0 ? b1 : b0;
                // Stage t has landed for every wave; every wave is done with stage t - 1 (in nxt).
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                const int bad = bad_next;
                if (t + 1 < ntiles) bad_next = issue_stage(nxt, (t + 1) * BC, kBoth);
                if (t >= nt_w) continue;
                scores(cur);
                weights(t, bad);
                outputs(cur);
            }
        }
    }
    if constexpr (KS > 1) {
        // Merge slot k: 1 KiB of the then free stage buffers.
        static_assert(kRowWaves * kNTD * 4 * (KS - 1) * 1024 <= 2 * kBuf, "merge slots");
        __shared__ float merge_ml[2 * NW * 64];
        const auto slot_base = [&](int k) { return k < kBuf / 1024 ? buf0 + k * 1024 : buf1 + (k * 1024 - kBuf); };
        AttnParams to = p;
        to.n_splits = it.parts;
        merge_kv_groups<D, KS, kRowWaves>(to, st, o, slot_base, merge_ml, wave, kgrp, lane, g, out_row(), part_row(),
                                          (lane & 31) < nrows);
        return;
    }
    __syncthreads();  // every wave is done with the stages
    char* const mine = (wave_id < NW / 2 ? buf0 : buf1) + wave_id % (NW / 2) * (2 * kBuf / NW);
    const float l = sum_xor32(st.l);
    if (it.parts > 1) {
        // Rebased to the rows' true maxima, for the merge.
        const bool none = st.rmax == -INFINITY;
        const float beta = none ? 0.f : rebase_factor(st.m, st.rmax, c);
        const size_t at = part_row();
        AttnParams to = p;
        to.O = p.Opart + (at - (lane & 31)) * D;
        packed_store<kOutF32, D, 2 * kBuf / NW>(to, o, beta, mine, lane & 31, nrows, lane);
        if (g == 0 && (lane & 31) < nrows) {
            p.Mpart[at] = none ? -INFINITY : st.rmax * p.scale;
            p.Lpart[at] = l * beta;
        }
        return;
    }
    const bool empty = !(l > 0.f);                        // no visible key
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

template <bool kBF, int D, int NW, int KS>
__global__ __launch_bounds__((PagedCfg<D, NW, KS>::kThreads), (PagedCfg<D, NW, KS>::kWavesPerSimd))
void kf_attn_paged_kernel(PagedParams p) {
    constexpr int kRows = PagedCfg<D, NW, KS>::kRows;
    // KV heads next to each other: with ids dealt round-robin over the XCDs, 8
    // heads have an XCD, and its L2, each.
    const int hk = blockIdx.x % p.heads_kv, share = blockIdx.x / p.heads_kv;
    int lane = threadIdx.x & 63;
    PagedItem it;
    if constexpr (kRows > 32) {
        if (paged_find<false>(p, lane, share, it, [&](int i) { return paged_count<kRows>(p, i); }))
            paged_tile<kBF, D, NW, KS>(p, it, hk, lane, 0, 0);
    } else {
        LineShare w;
        if (!line_find(p, lane, share, w, [&](int i) { return line_units(p, i); })) return;
        int seq = w.seq;
        long long at = w.at, left = w.u1 - w.u0;
        while (left > 0 && seq < p.n_seqs) {
            // (An opaque lane: nothing that is derived from it lives across the tiles.)
            lane = threadIdx.x & 63;
            asm volatile("" : "+v"(lane));
            const PagedSeq sq = paged_seq(p, seq);
            const int stages = line_stages(sq);
            const long long all = ((long long)sq.qn * p.ratio + 31) / 32 * stages;
            if (at >= all) {
                at -= all;
                ++seq;
                continue;
            }
            it.seq = seq;
            it.tile = __builtin_amdgcn_readfirstlane((int)line_div(at, stages));
            const int a = __builtin_amdgcn_readfirstlane((int)(at - (long long)it.tile * stages));
            // Without a second kernel a tile goes to the share of its first unit.
            const int b = p.cut ? (int)min((long long)stages, a + left) : stages;
            if (!p.cut && a > 0) {
                at += b - a;
                left -= b - a;
                continue;
            }
            it.part = 0;
            it.parts = b - a == stages ? 1 : 2;
            it.slot = 2 * share + (a == 0 ? 1 : 0);
            paged_tile<kBF, D, NW, KS>(p, it, hk, lane, max(a - kLineStart, 0), max(b - kLineStart, 0));
            __syncthreads();  // every wave is done with the stages
            at += b - a;
            left -= b - a;
        }
    }
}

// The parts of the tiles that were cut, joined: a workgroup per KV head and 32 rows of a
// tile (32 contexts with 1 to 512 new tokens, 32 / 8 heads of 128, 9.4 us; 128 rows 18.8),
// a lane per 4 channels of a row.  O = sum_i w_i O_i / L, L = sum_i w_i l_i, w_i = exp(m_i - max m), in
// the order of the keys; a part in which a row saw no key (m_i = -inf) wrote no O.
constexpr int kPagedMergeThreads = 256;
template <int D, int kRows>
__global__ __launch_bounds__(kPagedMergeThreads)
void kf_attn_paged_merge_kernel(PagedParams p) {
    const int lane = threadIdx.x & 63, hk = blockIdx.x % p.heads_kv, share = blockIdx.x / p.heads_kv + 1;
    PagedItem it;
    if constexpr (kRows > 32) {
        if (!paged_find<true>(p, lane, share - 1, it, [&](int i) { return paged_count<kRows>(p, i); })) return;
    } else {
        LineShare w;
        if (!line_find(p, lane, share, w, [&](int i) { return line_units(p, i); })) return;
        const int stages = line_stages(paged_seq(p, w.seq));
        it.seq = w.seq;
        it.tile = (int)line_div(w.at, stages);
        const long long in_front = w.at - (long long)it.tile * stages;
        it.parts = line_parts(w, in_front, stages - in_front);
        if (it.parts == 0) return;
    }
    const PagedSeq sq = paged_seq(p, it.seq);
    const int R = sq.qn * p.ratio, r0 = it.tile * kRows;
    if ((unsigned)it.tile * (unsigned)kRows >= (unsigned)R) return;
    constexpr int kUnroll = 4;
    // Rows 32 blockIdx.y and the next 31.
    const int first = blockIdx.y * 32 * (D / 4), n = min(min(kRows, R - r0) * (D / 4), first + 32 * (D / 4));
    for (int i = first + threadIdx.x; i < n; i += kPagedMergeThreads) {
        const int r = i / (D / 4), c4 = i % (D / 4) * 4;
        const auto at = [&](int k) {
            return ((size_t)(kRows > 32 ? it.slot + k : line_slot(share, k)) * p.heads_kv + hk) * kRows + r;
        };
        float m = -INFINITY, l = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < it.parts; k0 += kUnroll) {
            float mv[kUnroll], lv[kUnroll];
            f32x4 ov[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const size_t pi = at(min(k0 + u, it.parts - 1));
                mv[u] = p.Mpart[pi];
                lv[u] = p.Lpart[pi];
                ov[u] = *reinterpret_cast<const f32x4*>(p.Opart + pi * D + c4);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (k0 + u >= it.parts || mv[u] == -INFINITY) continue;
                const float top = fmaxf(m, mv[u]);
                const float keep = m == -INFINITY ? 0.f : exp2_hw((m - top) * kLog2e);
                const float w = exp2_hw((mv[u] - top) * kLog2e);
                l = l * keep + w * lv[u];
                acc = acc * keep + ov[u] * w;
                m = top;
            }
        }
        const int row = r0 + r, to = ((sq.q0 + row / p.ratio) * p.heads_kv + hk) * p.ratio + row % p.ratio;
        store_out4(p, (size_t)to * D + c4, acc * (l > 0.f ? 1.0f / l : 0.f));
        if (c4 == 0) store_stats(p, to, m, l);
    }
}

// ---------------------------------------------------------------------------
// The attention weight that keys gather: weights[j] += sum over the query rows of
// exp(s_rj - lse_r), r over the new tokens that see key j and the heads of its group.
//
// S^T = K Q^T by the 32x32x16 MFMA: a wave holds 64 keys as the A operand, straight
// from the pages, and the query rows go by as the B operand, 32 at a time, in LDS
// stages of 64 that the workgroup's waves share; lane l has row l % 32 of 16 keys a
// product, and adds their weights up in registers.  At the end the lanes' sums of a
// key are added, and the one wave that has the key adds them to its weight: no
// atomics, always the same order.
//
// A sequence of up to 32 rows, a step's, is read once from the pages: there the wave
// holds the rows, and its keys go by through LDS stages of its own (weigh_step).
//
// The work of a KV head is a line of units, 64 rows that meet a block of keys or a
// run of a step's keys, of which every workgroup has an equal share.  Where a block's
// units lie in several shares, their sums go through the workspace and a second kernel.
// Chunks keep neither unit busy: of 421K cycles a SIMD the VALU issues for 195K, an exponential, a
// multiply-add and an addition a score, and the matrix unit works for 136K, while waves, two a
// SIMD, wait for 31 % of theirs, for stages at the one barrier of each (4 x 512 tokens over 8192
// keys, 32 / 8 heads of 128, 198 us).  Steps wait for 75 % and read at 5.2 TB/s (32 contexts of 512
// to 8192 keys 31.5 us).
// ---------------------------------------------------------------------------
constexpr int kWeighRows = 64;                                      // query rows of a stage
template <int D> struct WeighCfg {
    static constexpr int kThreads = 256, kWaves = kThreads / 64;
    // 32-key tiles of a wave: two of 256 channels would not fit its registers.
    static constexpr int kTiles = D == 256 ? 1 : 2;
    static constexpr int kWaveKeys = 32 * kTiles;
    static constexpr int kKeys = kWaveKeys * kWaves;                // of a block
    static constexpr int kWavesPerSimd = 2;
    // Steps: a run has a tile of 32 keys for every wave, and counts as much as so many
    // units (steps alone take the same by 1, 2 and 4, 34 us for 32 contexts of 512 to 8192
    // keys; with 1 to 256 new tokens each 123, 145 and 180); channels of an LDS stage
    // and the stages of a wave; tiles whose sums wait in LDS.
    static constexpr int kStepKeys = 32 * kWaves, kStepUnits = 2;
    static constexpr int kStepWidth = D < 128 ? D : 128, kRing = D == 64 ? 4 : 2;
    static constexpr int kStepStage = 32 * kStepWidth * 2, kStepSums = 16;
    static constexpr int kRowsBytes = 2 * kWeighRows * 2 * D, kRingBytes = kWaves * kRing * kStepStage;
    static constexpr int kLds = kRowsBytes > kRingBytes ? kRowsBytes : kRingBytes;
};

// The blocks of one sequence's keys.  Causal: query i sees keys j <= i + before, and the rows in
// front of the first that sees any of a block's have no units there.
template <int D> struct WeighSeq {
    int q0, qn, kn, rows, stages;
    bool step;
    __device__ __forceinline__ WeighSeq(const PagedParams& p, int i) {
        const PagedSeq s = paged_seq(p, i);
        q0 = s.q0, qn = s.qn, kn = s.kn;
        rows = qn * p.ratio;
        stages = (int)(((unsigned)rows + kWeighRows - 1) / kWeighRows);
        step = rows <= 32;
    }
    __device__ __forceinline__ int before() const { return kn - qn; }
    __device__ __forceinline__ int tiles() const {
        const int keys = step ? WeighCfg<D>::kStepKeys : WeighCfg<D>::kKeys;
        return rows == 0 ? 0 : (kn + keys - 1) / keys;
    }
    // The first stage of block t, and the units of the t blocks in front of it.
    __device__ __forceinline__ int first(const PagedParams& p, int t) const {
        return !p.causal || step ? 0 : (int)((long long)max(t * WeighCfg<D>::kKeys - before(), 0) * p.ratio / kWeighRows);
    }
    __device__ __forceinline__ long long units(const PagedParams& p, int t) const {
        if (step) return (long long)t * WeighCfg<D>::kStepUnits;
        long long u = (long long)t * stages;
        // From block t0 on first() is m t - c: a block has a whole number m of stages' rows.
        const int t0 = before() < 0 ? 0 : before() / WeighCfg<D>::kKeys + 1;
        if (p.causal && t > t0) {
            const long long m = WeighCfg<D>::kKeys / kWeighRows * p.ratio, b = (long long)before() * p.ratio;
            const long long c = b >= 0 ? (b + kWeighRows - 1) / kWeighRows : -(-b / kWeighRows);
            u -= m * (((long long)t * (t - 1) - (long long)t0 * (t0 - 1)) / 2) - c * (t - t0);
        }
        return u;
    }
    __device__ __forceinline__ long long units(const PagedParams& p) const { return units(p, tiles()); }
    // The block of unit u.
    __device__ __forceinline__ int tile_of(const PagedParams& p, long long u) const {
        int lo = 0, hi = tiles();   // units(lo) <= u < units(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (units(p, mid) <= u) lo = mid; else hi = mid;
        }
        return lo;
    }
};

// A row's log-sum-exp, as bits: the compiler takes comparisons of floats to have no NaN.  -inf, of a
// row that adds nothing whatever it and the keys hold; NaN; neither a number nor +inf; and what the
// row's exponents are less by.
__device__ __forceinline__ bool lse_none(uint32_t e) { return e == 0xff800000u; }
__device__ __forceinline__ bool lse_nan(uint32_t e) { return (e & 0x7fffffffu) > 0x7f800000u; }
__device__ __forceinline__ bool lse_strange(uint32_t e) { return lse_none(e) || lse_nan(e); }
constexpr uint32_t kLseLow = 0xff300000u;   // -2.34e38; from -2.36e38 down lse_less passes fp32's range
__device__ __forceinline__ float lse_less(uint32_t e) { return -__uint_as_float(e) * kLog2e; }

// Runs r0 .. r1 - 1 of a step's keys.  S = Q K^T: lane l has key l % 32 and 16 of the
// rows, the sum over which needs one exchange; of fewer rows only those groups of eight
// that there are have exponentials.  Every wave copies its own stages, 32 keys or half of
// their 256 channels, and waits for itself alone.
template <bool kBF, int D>
__device__ __forceinline__ void weigh_step(const PagedParams& p, const WeighSeq<D>& sq, int seq, int r0, int r1, int hk,
                                           int wave, int lane, char* lds, float* sums) {
    using Cfg = WeighCfg<D>;
    using E = Elem<kBF>;
    using X8 = typename E::x8;
    constexpr int W = Cfg::kStepWidth, kChunks = W / 8, kRowBytes = 2 * W, kRowsPerInstr = 1024 / kRowBytes;
    using SW = SwizzleRow<W>;
    constexpr int kNKK = D / 16, kStageKK = W / 16, kHalves = D / W, kHalfInstr = 16 / kRowsPerInstr;
    const int g = lane >> 5, sh = p.page_shift, ratio = p.ratio, R = sq.rows;
    // Tile t of the wave begins at key k0 + t kStepKeys.
    const int k0 = r0 * Cfg::kStepKeys + wave * 32, left = min(r1 * Cfg::kStepKeys, sq.kn) - k0;
    if (left <= 0) return;
    const int ntiles = (left + Cfg::kStepKeys - 1) / Cfg::kStepKeys, nst = ntiles * kHalves;
    // The ids of 64 pages from page0 on, one to a lane; stages come in order.
    const int* const table = p.block_table + (size_t)seq * p.max_pages;
    const int last_page = (sq.kn - 1) >> sh;
    int page0 = k0 >> sh, ids = table[min(page0 + lane, last_page)];
    const int lr = lane / kChunks;
    uint32_t lane_off[kHalfInstr];
#pragma unroll
    for (int i = 0; i < kHalfInstr; ++i) {
        const int r = i * kRowsPerInstr + lr;
        lane_off[i] = (uint32_t)(r * 2 * D) + (((lane % kChunks) ^ SW::h(r)) % kChunks) * 16;
    }
    char* const ring = lds + wave * (Cfg::kRing * Cfg::kStepStage);
    const auto issue = [&](int s) {
        const uint32_t d_lds = (uint32_t)(uintptr_t)(lds_void*)(ring + s % Cfg::kRing * Cfg::kStepStage);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // (Rows behind the keys lie in their page still, or are those of page 0.)
            const int key = k0 + s / kHalves * Cfg::kStepKeys + 16 * h;
            int id = -1;
            if (key < sq.kn) {
                if ((key >> sh) - page0 >= 64) {
                    page0 = key >> sh;
                    ids = table[min(page0 + lane, last_page)];
                }
                id = __builtin_amdgcn_readlane(ids, (key >> sh) - page0);
            }
            const size_t row = (((size_t)((unsigned)id < (unsigned)p.num_pages ? id : 0) * p.heads_kv + hk) << sh) +
                               (key & ((1 << sh) - 1));
            const char* const src = reinterpret_cast<const char*>(p.K) + row * (2 * D) + s % kHalves * kRowBytes;
#pragma unroll
            for (int i = 0; i < kHalfInstr; ++i)
                lds_copy16(d_lds + (h * kHalfInstr + i) * 1024, src, lane_off[i]);
        }
    };
    // The rows, those past the last as the last, and what their exponents are less by: those and
    // rows without a key add nothing.
    X8 q[kNKK];
    const int row = min(lane & 31, R - 1);
    {
        const uint16_t* Qr = p.Q + (size_t)(sq.q0 + row / ratio) * p.q_token + (size_t)(hk * ratio + row % ratio) * p.q_head;
#pragma unroll
        for (int kk = 0; kk < kNKK; ++kk) q[kk] = *reinterpret_cast<const X8*>(Qr + (2 * kk + g) * 8);
    }
    const uint32_t e = p.row_lse[((size_t)(sq.q0 + row / ratio) * p.heads_kv + hk) * ratio + row % ratio];
#pragma unroll
    for (int s = 0; s < Cfg::kRing - 1; ++s)
        if (s < nst) issue(s);
    // (NaN stays NaN: the weights of keys that a row does not see, and those of rows that add nothing,
    // are 0 whatever they would be.)
    const float less_row = (lane & 31) >= R ? -INFINITY : __uint_as_float(lse_nan(e) ? e : __float_as_uint(lse_less(e)));
    // The last key to which a row adds something: all of them up to one, or none.
    const int last_row = lse_none(e) ? -1 : p.causal ? sq.before() + (lane & 31) / ratio : sq.kn;
    const int clear = __any(lse_none(e)) ? 0 : p.causal ? sq.before() + 1 : INT_MAX;   // in front of it all rows do
    float less[16];
    int last[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        less[r] = __shfl(less_row, 8 * (r >> 2) + (r & 3) + 4 * g);
        last[r] = __shfl(last_row, 8 * (r >> 2) + (r & 3) + 4 * g);
    }
    int koff[kStageKK];
#pragma unroll
    for (int kk = 0; kk < kStageKK; ++kk) {
        const int r = lane & 31;
        koff[kk] = r * kRowBytes + (((2 * kk + g) ^ SW::h(r)) % kChunks) * 16;
    }
    for (int t0 = 0; t0 < ntiles; t0 += Cfg::kStepSums) {
        const int n = min(Cfg::kStepSums, ntiles - t0);
        for (int t = t0; t < t0 + n; ++t) {
            f32x16 x = {};
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf) {
                const int s = t * kHalves + hf;
                if (s + Cfg::kRing - 1 < nst) {
                    asm volatile("" ::: "memory");
                    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the stage there has been read
                    issue(s + Cfg::kRing - 1);
                }
                // This stage has landed where no more than the later ones' copies are on their way.
                const int ahead = min(Cfg::kRing - 1, nst - 1 - s);
                asm volatile("" ::: "memory");
                if (ahead >= 3) __builtin_amdgcn_s_waitcnt(0x0f70 | (6 * kHalfInstr & 15) | (6 * kHalfInstr >> 4) << 14);
                else if (ahead == 2) __builtin_amdgcn_s_waitcnt(0x0f70 | (4 * kHalfInstr & 15) | (4 * kHalfInstr >> 4) << 14);
                else if (ahead == 1) __builtin_amdgcn_s_waitcnt(0x0f70 | (2 * kHalfInstr & 15) | (2 * kHalfInstr >> 4) << 14);
                else __builtin_amdgcn_s_waitcnt(0x0f70);
                asm volatile("" ::: "memory");
                const char* const stage = ring + s % Cfg::kRing * Cfg::kStepStage;
#pragma unroll
                for (int kk = 0; kk < kStageKK; ++kk)
                    x = E::mfma32(q[hf * kStageKK + kk], *reinterpret_cast<const X8*>(stage + koff[kk]), x);
            }
            const int kt = k0 + t * Cfg::kStepKeys, key = kt + (lane & 31);
            const bool whole = kt + 31 < clear;
            float add = 0.f;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (8 * b >= R) break;
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = exp2_hw(fmaf(x[4 * b + i], p.scale_log2, less[4 * b + i]));
                if (!whole) {
                    asm volatile("" ::: "memory");       // a branch, not selects in every tile
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key > last[4 * b + i]) w[i] = 0.f;
                }
                add += (w[0] + w[1]) + (w[2] + w[3]);
            }
            add += __shfl_xor(add, 32);
            if (g == 0) sums[(t - t0) * 32 + lane] = add;
        }
        // The wave's own sums, two tiles at a time.
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        for (int t = t0 + g; t < t0 + n; t += 2) {
            const int key = k0 + t * Cfg::kStepKeys + (lane & 31);
            const int id = key < sq.kn ? table[key >> sh] : -1;
            if ((unsigned)id < (unsigned)p.num_pages)
                p.weights[(((size_t)id * p.heads_kv + hk) << sh) + (key & ((1 << sh) - 1))] += sums[(t - t0) * 32 + (lane & 31)];
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): later waits count copies alone
        asm volatile("" ::: "memory");
    }
}

template <bool kBF, int D>
__global__ __launch_bounds__(WeighCfg<D>::kThreads, WeighCfg<D>::kWavesPerSimd)
void kf_kv_weigh_kernel(PagedParams p) {
    using Cfg = WeighCfg<D>;
    using E = Elem<kBF>;
    using X8 = typename E::x8;
    using SW = SwizzleRow<D>;
    constexpr int kNKK = D / 16, kChunks = D / 8, kRowBytes = 2 * D, kRowsPerInstr = 1024 / kRowBytes;
    constexpr int kWaves = Cfg::kWaves, kInstr = kWeighRows / kRowsPerInstr / kWaves;  // of a wave and stage
    constexpr int kTiles = Cfg::kTiles, kWaveKeys = Cfg::kWaveKeys, kKeys = Cfg::kKeys;
    constexpr bool kXorOff = D >= 128;
    __shared__ __attribute__((aligned(1024))) char lds[Cfg::kLds];
    __shared__ float step_sums[kWaves][Cfg::kStepSums * 32];
    __shared__ uint32_t off[kInstr][Cfg::kThreads];       // this thread's offsets of a whole stage
    const auto buf = [&](int s) { return lds + (s & 1) * (kWeighRows * kRowBytes); };
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hk = blockIdx.x % p.heads_kv, sh = p.page_shift, ratio = p.ratio, share = blockIdx.x / p.heads_kv;
    // LDS-DMA, as in the attention kernels: lane l of an instruction fills row l / kChunks of
    // its rows, physical chunk l % kChunks.
    const auto row_of = [&](int l, int i) { return (wave * kInstr + i) * kRowsPerInstr + l / kChunks; };
    const auto chunk_off = [&](int l, int i) { return (uint32_t)((((l % kChunks) ^ SW::h(row_of(l, i))) % kChunks) * 16); };
    // Whole stages begin at a token, and their lanes' offsets from it have 32 bits.
    const bool plain = kWeighRows % ratio == 0 && kWeighRows / ratio * p.q_token + ratio * p.q_head < (1LL << 30);
    const size_t stage_bytes = (size_t)(kWeighRows / ratio) * p.q_token * 2;
    LineShare w;
    {
        const int l = threadIdx.x & 63;
        if (!line_find(p, l, share, w, [&](int i) { return WeighSeq<D>(p, i).units(p); })) return;
#pragma unroll
        for (int i = 0; i < kInstr; ++i) {
            const int row = row_of(l, i), q = row / ratio;
            off[i][threadIdx.x] = (uint32_t)((q * p.q_token + (row - q * ratio) * p.q_head) * 2) + chunk_off(l, i);
        }
    }
    int seq = w.seq;
    long long at = w.at, left = w.u1 - w.u0;
    while (left > 0 && seq < p.n_seqs) {
        // (An opaque lane: nothing that is derived from it lives across the blocks.)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int g = lane >> 5;
        WeighSeq<D> sq(p, seq);
        sq.q0 = __builtin_amdgcn_readfirstlane(sq.q0);
        sq.qn = __builtin_amdgcn_readfirstlane(sq.qn);
        sq.kn = __builtin_amdgcn_readfirstlane(sq.kn);
        sq.rows = __builtin_amdgcn_readfirstlane(sq.rows);
        sq.stages = __builtin_amdgcn_readfirstlane(sq.stages);
        sq.step = sq.rows <= 32;
        const long long all = sq.units(p);
        if (at >= all) {
            at -= all;
            ++seq;
            continue;
        }
        if (sq.step) {
            // The runs that begin in this share.
            const long long n = min(all - at, left);
            const int r0 = (int)((at + Cfg::kStepUnits - 1) / Cfg::kStepUnits);
            const int r1 = (int)((at + n + Cfg::kStepUnits - 1) / Cfg::kStepUnits);
            if (r0 < r1) weigh_step<kBF, D>(p, sq, seq, r0, r1, hk, wave, lane, lds, step_sums[wave]);
            at += n;
            left -= n;
            __syncthreads();  // every wave is done with its stages
            continue;
        }
        const int R = sq.rows, tile = __builtin_amdgcn_readfirstlane(sq.tile_of(p, at));
        const long long begin = sq.units(p, tile);
        const int s_first = sq.first(p, tile), n_units = sq.stages - s_first;
        // Stages of this share.  Without a second kernel a block goes to the share of its first unit.
        int s0 = s_first + (int)(at - begin), s1 = (int)min((long long)sq.stages, s0 + left);
        const int skip = s0;
        if (!p.cut) {
            s1 = sq.stages;
            if (s0 > s_first) s0 = s1;
        }
        const bool whole_block = s0 == s_first && s1 == sq.stages;
        const int slot = 2 * share + (s0 == s_first ? 1 : 0);
        at = begin + (s1 - s_first);
        left -= s1 - skip;
        if (s0 >= s1 || n_units <= 0) continue;
        const int kb = tile * kKeys, k0 = kb + wave * kWaveKeys, before = sq.before();
        const int* const table = p.block_table + (size_t)seq * p.max_pages;
        const auto page_of = [&](int key) { return key < sq.kn ? table[key >> sh] : -1; };
        const auto valid = [&](int id) { return (unsigned)id < (unsigned)p.num_pages; };
        // The keys of the A operand.  Past the last, or on no valid page, any row will do: it
        // reaches no other key's sum, and its own is dropped.
        X8 kf[kTiles][kNKK];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int key = k0 + 32 * t + (lane & 31), id = page_of(key);
            const uint16_t* Kr = p.K + ((((size_t)(valid(id) ? id : 0) * p.heads_kv + hk) << sh) + (key & ((1 << sh) - 1))) * D;
#pragma unroll
            for (int kk = 0; kk < kNKK; ++kk) kf[t][kk] = *reinterpret_cast<const X8*>(Kr + (2 * kk + g) * 8);
        }
        int koff[kNKK];
#pragma unroll
        for (int kk = 0; kk < kNKK; ++kk) {
            const int r = lane & 31;
            koff[kk] = r * kRowBytes + (((2 * kk + g) ^ SW::h(r)) % kChunks) * 16;
        }
        const char* const Qh = reinterpret_cast<const char*>(p.Q + (size_t)sq.q0 * p.q_token + (size_t)hk * ratio * p.q_head);
        const uint32_t* const lse = p.row_lse + ((size_t)sq.q0 * p.heads_kv + hk) * ratio;
        const uint32_t lse_off = (uint32_t)(lane / ratio * p.heads_kv * ratio + lane % ratio) * 4;
        // Requests a stage, and the log-sum-exp of a row of it.  (Other stages than whole ones
        // from an opaque lane.)
        const auto issue_stage = [&](int s, uint32_t& e) {
            const int r0 = s * kWeighRows;
            const uint32_t d_lds = (uint32_t)(uintptr_t)(lds_void*)(buf(s) + wave * kInstr * 1024);
            if (plain && r0 + kWeighRows <= R) {
                const char* const src = Qh + s * stage_bytes;
#pragma unroll
                for (int i = 0; i < kInstr; ++i) lds_copy16(d_lds + i * 1024, src, off[i][threadIdx.x]);
                e = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(lse + (size_t)r0 * p.heads_kv) + lse_off);
            } else {
                int l = lane;
                asm volatile("" : "+v"(l));
#pragma unroll
                for (int i = 0; i < kInstr; ++i) {
                    const int row = min(r0 + row_of(l, i), R - 1), q = row / ratio;
                    lds_copy16(d_lds + i * 1024, Qh + ((size_t)q * p.q_token + (size_t)(row - q * ratio) * p.q_head) * 2 +
                                                     chunk_off(l, i));
                }
                const int row = min(r0 + l, R - 1), q = row / ratio;
                e = lse[(size_t)q * p.heads_kv * ratio + (row - q * ratio)];
            }
        };
        // Rows in front of `first` see no key of the wave, those in front of `whole` not all.
        const auto rows_to = [&](int key) { return (int)min((long long)max(key - before, 0) * ratio, (long long)R); };
        const int first = p.causal ? rows_to(k0) : 0, whole = p.causal ? rows_to(k0 + kWaveKeys - 1) : 0;
        f32x16 sum[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) sum[t] = f32x16{};
        // The scores x of 32 rows, and beside their products the exponentials of `old` ones, the
        // instructions in this order: a wave overlaps them only as they stand in its stream.
        // Rows are read kAhead steps before they are used, also the first of the next 32.
        constexpr int kAhead = 3;
        X8 q[kAhead + 1];
        int kb0 = koff[0];
        const auto read = [&](const char* rows, int kk) {
            return *reinterpret_cast<const X8*>(rows + (kXorOff ? kb0 ^ (32 * kk) : koff[kk]));
        };
        const auto scores = [&](const char* rows, const char* next, f32x16 (&x)[kTiles], const f32x16 (&old)[kTiles], float less) {
            constexpr int kPer = 16 * kTiles / kNKK;
            if constexpr (kXorOff) asm volatile("" : "+v"(kb0));  // derived per tile
#pragma unroll
            for (int kk = 0; kk < kNKK; ++kk) {
                if (kk + kAhead < kNKK) q[(kk + kAhead) % (kAhead + 1)] = read(rows, kk + kAhead);
                else if (next) q[(kk + kAhead) % (kAhead + 1)] = read(next, kk + kAhead - kNKK);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) x[t] = E::mfma32(kf[t][kk], q[kk % (kAhead + 1)], kk == 0 ? f32x16{} : x[t]);
#pragma unroll
                for (int e = kk * kPer; e < (kk + 1) * kPer; ++e) {
                    float v = sum[e / 16][e % 16] + exp2_hw(fmaf(old[e / 16][e % 16], p.scale_log2, less));
                    asm volatile("" : "+v"(v));                   // here, not behind later branches
                    sum[e / 16][e % 16] = v;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // The rows `half` of the 64 that lane l has row l's log-sum-exp e of: where e is NaN or -inf
        // (`strange`: there may be such) -> e, and then keys that a row does not see -> -inf.
        const auto hide = [&](f32x16 (&x)[kTiles], int r0, bool strange, uint32_t e, int half) {
            if (strange) {
                asm volatile("" ::: "memory");
                const uint32_t mine = __shfl(e, 32 * half + (lane & 31));
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        x[t][r] = __uint_as_float(lse_strange(mine) ? mine : __float_as_uint(x[t][r]));
            }
            if (r0 >= whole) return;
            asm volatile("" ::: "memory");                        // a branch, not selects in every tile
            const int lim = min(r0 + (lane & 31), R - 1) / ratio + before + 1 - k0 - 4 * g;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * t + 8 * (r >> 2) + (r & 3) >= lim) x[t][r] = -INFINITY;
        };
        uint32_t e_next = 0;
        if (s0 < s1) issue_stage(s0, e_next);
        // The second half's scores wait for their exponentials until the next products.
        f32x16 x[kTiles], late[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) late[t] = f32x16{};
        float late_less = -INFINITY;
        for (int s = s0; s < s1; ++s) {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const uint32_t e = e_next;
            if (s + 1 < s1) issue_stage(s + 1, e_next);
            const char* const rows = buf(s);
            const int r0 = s * kWeighRows;
            if (min(r0 + kWeighRows, R) <= first) continue;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) q[i] = read(rows, i);
            // What the exponents of the stage's row `lane` are less by; rows past the last add nothing.  (NaN
            // and -inf are in the scores that the row sees: here a NaN would reach all.)
            const bool strange = __any(e >= kLseLow || lse_nan(e));
            float less = r0 + lane >= R ? -INFINITY : lse_less(e);
            if (strange) less = lse_strange(e) ? 0.f : fminf(less, FLT_MAX);   // -inf + inf would be NaN
            scores(rows, rows + 32 * kRowBytes, x, late, late_less);
            hide(x, r0, strange, e, 0);
            scores(rows + 32 * kRowBytes, nullptr, late, x, __shfl(less, lane & 31));
            hide(late, r0 + 32, strange, e, 1);
            late_less = __shfl(less, 32 + (lane & 31));
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[t][r] += exp2_hw(fmaf(late[t][r], p.scale_log2, late_less));
        // Over the 32 rows: with every exchange a lane keeps half of its keys, in the end
        // lane l (and l ^ 16) the one of register l % 16.
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
            for (int b = 3; b >= 0; --b)
#pragma unroll
                for (int r = 0; r < 1 << b; ++r) {
                    const bool up = (lane >> b & 1) != 0;
                    const float give = up ? sum[t][r] : sum[t][r + (1 << b)];
                    sum[t][r] = (up ? sum[t][r + (1 << b)] : sum[t][r]) + __shfl_xor(give, 1 << b);
                }
            const float total = sum[t][0] + __shfl_xor(sum[t][0], 16);
            const int place = wave * kWaveKeys + 32 * t + acc_row(lane & 15, lane), key = kb + place, id = page_of(key);
            if ((lane & 16) != 0) continue;
            if (!whole_block)
                p.Opart[((size_t)slot * p.heads_kv + hk) * kKeys + place] = total;
            else if (valid(id))
                p.weights[(((size_t)id * p.heads_kv + hk) << sh) + (key & ((1 << sh) - 1))] += total;
        }
        __syncthreads();  // every wave is done with the stages
    }
}

// The sums of the blocks that were cut, added up: the first share that begins inside a
// block sees to it.  A thread per key and quarter of the parts, eight loads on their
// way, and the quarters in order.
template <int D>
__global__ __launch_bounds__(4 * WeighCfg<D>::kKeys)
void kf_kv_weigh_merge_kernel(PagedParams p) {
    constexpr int kKeys = WeighCfg<D>::kKeys, kRuns = 4;
    __shared__ float sums[kRuns][kKeys];
    const int lane = threadIdx.x & 63, hk = blockIdx.x % p.heads_kv, share = blockIdx.x / p.heads_kv + 1, sh = p.page_shift;
    LineShare w;
    if (!line_find(p, lane, share, w, [&](int i) { return WeighSeq<D>(p, i).units(p); })) return;
    const WeighSeq<D> sq(p, w.seq);
    if (sq.step) return;
    const int tile = sq.tile_of(p, w.at);
    const long long in_front = w.at - sq.units(p, tile), behind = sq.units(p, tile + 1) - w.at;
    const int parts = line_parts(w, in_front, behind);
    if (parts == 0) return;
    const int at = threadIdx.x % kKeys, run = threadIdx.x / kKeys, key = tile * kKeys + at;
    const int per = (parts + kRuns - 1) / kRuns, k1 = min((run + 1) * per, parts);
    float total = 0.f;
    for (int k = run * per; k < k1; k += 8) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            v[u] = p.Opart[((size_t)line_slot(share, min(k + u, k1 - 1)) * p.heads_kv + hk) * kKeys + at];
#pragma unroll
        for (int u = 0; u < 8; ++u) total += k + u < k1 ? v[u] : 0.f;
    }
    sums[run][at] = total;
    __syncthreads();
    if (run > 0 || key >= sq.kn) return;
    const int id = p.block_table[(size_t)w.seq * p.max_pages + (key >> sh)];
    if ((unsigned)id >= (unsigned)p.num_pages) return;
#pragma unroll
    for (int r = 1; r < kRuns; ++r) total += sums[r][at];
    p.weights[(((size_t)id * p.heads_kv + hk) << sh) + (key & ((1 << sh) - 1))] += total;
}

}  // namespace kf
