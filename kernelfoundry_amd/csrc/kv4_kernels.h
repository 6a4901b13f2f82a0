// kv4_kernels.h -- a paged K/V cache in 4 bits: quantised as it is written,
// read back, and attended to.
//
// The format is the Open Compute Project's microscaling one with 4-bit
// elements: every block of 32 consecutive channels of a row shares a scale
// 2^(E - 127), E one byte, and each channel is a code of 4 bits (sign, 2
// exponent bits, 1 mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6).  E is the
// exponent field of the block's largest magnitude (as fp32) less 2, at least
// 1; x / 2^(E - 127) is rounded to the nearest code, ties to the even one (5
// to 4), and magnitudes above 5 give 6 (the largest is below 8).  Dividing by a
// power of two is exact, so a code does not depend on the precision it is
// computed in, and a code times its scale is exact in fp16 and bf16 (of fp16
// inputs, and of bf16 ones).  A block that holds an infinity or a NaN gets E =
// 255 and reads back as NaN, also where the decode reads it.
//
// A pool is [num_pages][H_kv][page_size * 17 D / 32] bytes: per page and KV
// head the codes of the page's rows, [page_size][D / 2] (channel 2 i in the
// low half of byte i), then their scale bytes, [page_size][D / 32].
#pragma once

#include "elem.h"

namespace kf {

struct Kv4Params {
    const uint16_t* x[2];       // K, V in 16 bits (append)
    uint16_t* y[2];             // K, V in 16 bits (read)
    uint8_t* pages[2];
    long long token[2], head[2];  // strides of x in elements
    const int* block_table;     // [n_seqs][max_pages]
    const int* starts;          // [n_seqs + 1]
    const int* kv_lens;         // [n_seqs]
    int n_seqs, tokens, heads;
    int max_pages, page_shift, num_pages;
    size_t page_bytes;          // of one head
    int tile;                   // tokens of a workgroup, at most kKv4MaxTile
};

// Where token t's row lies: its page's bytes and the row in it, or a page of
// -1.  Sequence b's packed tokens are its last n_b = starts[b + 1] - starts[b]
// of kv_lens[b] keys.
struct Kv4Row {
    int page, row;
};
__device__ __forceinline__ Kv4Row kv4_row(const Kv4Params& p, int t) {
    Kv4Row r{-1, 0};            // (row 0: readers without a page read the pool's first row)
    if (t < p.starts[0] || t >= p.starts[p.n_seqs]) return r;
    const int b = sequence_of(p.starts, p.n_seqs, t);
    const long long at = (long long)p.kv_lens[b] - p.starts[b + 1] + t;
    if (at < 0 || at >= ((long long)p.max_pages << p.page_shift)) return r;
    const int id = p.block_table[(size_t)b * p.max_pages + (at >> p.page_shift)];
    if ((unsigned)id >= (unsigned)p.num_pages) return r;
    r.page = id;
    r.row = (int)(at & ((1 << p.page_shift) - 1));
    return r;
}

constexpr int kKv4Threads = 256;
constexpr int kKv4MaxTile = 256;   // tokens of a workgroup

// Both kernels: a workgroup takes p.tile consecutive tokens.  A thread per token
// finds its place (a binary search and four dependent loads, once for all heads), then the
// threads go through the items (token, head, 8 channels of K and of V) side by
// side, so that a wave's loads and stores are contiguous, kKv4Ahead items
// of a thread requested together.  Bound by memory: 30000 tokens of 8 heads, D =
// 128 (156 MB) 38 us written (4.1 TB/s; a copy 4.8), 26 read back (5.9 TB/s);
// with a thread per item that found its own place 40 and 48.
constexpr int kKv4Ahead = 2;

// The items of a thread: every 256th of the tile's.
struct Kv4Item {
    int t, rest;               // token of the tile; head and chunk in it
};
struct Kv4Walk {
    int per, dt, drest;        // items of a token; a step of 256 items
    __device__ __forceinline__ explicit Kv4Walk(int per_token)
        : per(per_token), dt(kKv4Threads / per_token), drest(kKv4Threads % per_token) {}
    __device__ __forceinline__ Kv4Item first(int tid) const { return Kv4Item{tid / per, tid % per}; }
    __device__ __forceinline__ void next(Kv4Item& i) const {
        i.t += dt;
        i.rest += drest;
        if (i.rest >= per) {
            i.rest -= per;
            ++i.t;
        }
    }
};

// Four neighbouring lanes hold a block, 8 channels (16 bytes in, 4 out) each.
template <bool kBF, int D>
__global__ __launch_bounds__(kKv4Threads)
void kf_kv4_append_kernel(Kv4Params p) {
    using E = Elem<kBF>;
    constexpr int kChunks = D / 8;
    __shared__ Kv4Row places[kKv4MaxTile];
    const int tid = threadIdx.x, t0 = blockIdx.x * p.tile, n = min(p.tile, p.tokens - t0);
    const Kv4Walk walk(p.heads * kChunks);
    Kv4Item it = walk.first(tid);
    bool placed = false;
    // The same trips for all threads, which meet at the barrier in the first.
    for (int left = (n * walk.per + kKv4Threads - 1) / kKv4Threads; left > 0; left -= kKv4Ahead) {
        Kv4Item its[kKv4Ahead];
        u32x4 raw[kKv4Ahead][2];
#pragma unroll
        for (int u = 0; u < kKv4Ahead; ++u) {
            its[u] = it;
            const int t = t0 + min(it.t, n - 1), h = it.rest / kChunks, c = it.rest % kChunks;
#pragma unroll
            for (int s = 0; s < 2; ++s)
                raw[u][s] = *reinterpret_cast<const u32x4*>(p.x[s] + (size_t)t * p.token[s] + (size_t)h * p.head[s] + 8 * c);
            walk.next(it);
        }
        if (!placed) {
            if (tid < n) places[tid] = kv4_row(p, t0 + tid);
            __syncthreads();
            placed = true;
        }
#pragma unroll
        for (int u = 0; u < kKv4Ahead; ++u) {
            const Kv4Row at = places[min(its[u].t, n - 1)];
            if (its[u].t >= n || at.page < 0) continue;    // the same for the lanes of a block
            const int h = its[u].rest / kChunks, c = its[u].rest % kChunks;
            const size_t base = ((size_t)at.page * p.heads + h) * p.page_bytes;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                // The largest magnitude by the bits: for one sign they order as the
                // values do, infinity and NaN above all.
                const u32x4 x = raw[u][s];
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, max(x[e] & 0x7fffu, (x[e] >> 16) & 0x7fffu));
                top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, false));  // lanes 1 0 3 2
                top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, false));  // lanes 2 3 0 1
                uint32_t exp;
                if constexpr (kBF) {
                    exp = top >> 7;
                } else {
                    exp = __float_as_uint((float)__builtin_bit_cast(f16, (uint16_t)top)) >> 23;
                }
                const bool bad = top >= E::kExpBits;
                exp = exp < 3 ? 1 : exp - 2;
                const float scale = __uint_as_float(exp << 23);
                const auto v = __builtin_bit_cast(typename E::x8, x);
                uint32_t code = 0;
                code = E::template to_fp4<0>(code, __builtin_shufflevector(v, v, 0, 1), scale);
                code = E::template to_fp4<1>(code, __builtin_shufflevector(v, v, 2, 3), scale);
                code = E::template to_fp4<2>(code, __builtin_shufflevector(v, v, 4, 5), scale);
                code = E::template to_fp4<3>(code, __builtin_shufflevector(v, v, 6, 7), scale);
                uint8_t* page = p.pages[s] + base;
                *reinterpret_cast<uint32_t*>(page + (size_t)at.row * (D / 2) + 4 * c) = bad ? 0u : code;
                // The scales of up to four blocks (16 lanes) by one lane.
                uint32_t bytes = bad ? 255 : exp;
                bytes |= (uint32_t)__builtin_amdgcn_mov_dpp((int)bytes, 0x104, 0xF, 0xF, true) << 8;  // of lane + 4
                uint8_t* const scales = page + ((size_t)(D / 2) << p.page_shift) + (size_t)at.row * (D / 32) + c / 4;
                if constexpr (D == 64) {
                    if (c == 0) *reinterpret_cast<uint16_t*>(scales) = (uint16_t)bytes;
                } else {
                    bytes |= (uint32_t)__builtin_amdgcn_mov_dpp((int)bytes, 0x108, 0xF, 0xF, true) << 16;  // of lane + 8
                    if (c % 16 == 0) *reinterpret_cast<uint32_t*>(scales) = bytes;
                }
            }
        }
    }
}

// The inverse: rows in 16 bits, [tokens][H_kv][D], of the same places; zeros
// for a token whose page is invalid, and nothing for one outside the
// sequences.
template <bool kBF, int D>
__global__ __launch_bounds__(kKv4Threads)
void kf_kv4_read_kernel(Kv4Params p) {
    using X8 = typename Elem<kBF>::x8;
    constexpr int kChunks = D / 8;
    __shared__ Kv4Row places[kKv4MaxTile];
    const int tid = threadIdx.x, t0 = blockIdx.x * p.tile, n = min(p.tile, p.tokens - t0);
    const int begin = p.starts[0], end = p.starts[p.n_seqs];
    if (tid < n) places[tid] = kv4_row(p, t0 + tid);
    const Kv4Walk walk(p.heads * kChunks);
    Kv4Item it = walk.first(tid);
    __syncthreads();
    while (it.t < n) {
        Kv4Item its[kKv4Ahead];
        uint32_t code[kKv4Ahead][2], exp[kKv4Ahead][2];
        bool ok[kKv4Ahead];
#pragma unroll
        for (int u = 0; u < kKv4Ahead; ++u) {
            its[u] = it;
            const Kv4Row at = places[min(it.t, n - 1)];
            const int h = it.rest / kChunks, c = it.rest % kChunks;
            ok[u] = at.page >= 0;
            // (A token without a page reads the pool's first row.)
            const size_t base = ((size_t)max(at.page, 0) * p.heads + h) * p.page_bytes;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint8_t* page = p.pages[s] + base;
                code[u][s] = *reinterpret_cast<const uint32_t*>(page + (size_t)at.row * (D / 2) + 4 * c);
                exp[u][s] = page[((size_t)(D / 2) << p.page_shift) + (size_t)at.row * (D / 32) + c / 4];
            }
            walk.next(it);
        }
#pragma unroll
        for (int u = 0; u < kKv4Ahead; ++u) {
            const int t = t0 + its[u].t;
            if (its[u].t >= n || t < begin || t >= end) continue;
            const int h = its[u].rest / kChunks, c = its[u].rest % kChunks;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4 v = __builtin_bit_cast(u32x4, from_fp4x8<kBF>(code[u][s], __uint_as_float(exp[u][s] << 23)));
                const uint32_t nan = kBF ? 0x7fc07fc0u : 0x7e007e00u;
                if (exp[u][s] == 255) v = u32x4{nan, nan, nan, nan};
                if (!ok[u]) v = u32x4{0u, 0u, 0u, 0u};
                __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p.y[s] + ((size_t)t * p.heads + h) * D + 8 * c));
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Decode over the 4-bit cache: <= 32 query rows per KV head.  The 32-key
// stages that the sequences hold are shared evenly over the waves of the
// grid, as in kf_attn_decode_ragged_kernel, whose map of the stages, partials
// and merge kernel this kernel uses.
//
// A stage is 32 keys x 17 D / 32 bytes of K and the same of V: a quarter of
// the fp16 cache's, so it waits in registers.  S^T = K Q^T by the 16x16x32
// MFMA: A is 16 keys, lane l holding key l % 16 and D / 4 consecutive channels
// from (l / 16) D / 4 on, its own codes and one or two scales, loaded straight
// from the page and converted in registers; any order of the channels does
// for the contraction as long as Q's operand has the same one.  V's rows
// arrive the same way, are converted (exactly) and go through LDS, from which
// ds_read_b64_tr_b16 brings them as V^T; P^T comes from the score registers:
// lane group q holds keys 4 q .. + 3 of both halves of the stage, and V^T is
// read in that order of the keys.  K(t + 1) is requested when the score MFMAs
// have consumed K(t), V(t + 1) when V(t) has gone to LDS.
//
// Bound by memory: with the loads alone it takes as long.  32 / 8 heads, D = 128, both
// launches: 32 x 8192 keys (285 MB) 58 us, 4.9 TB/s, the stages themselves at 6.2
// (63 with pages of 16 rows); 8 x 50000 to 65536, 4 queries each, bf16 (506 MB) 88 to
// 93, 5.4 to 5.7; 32 x 512 to 8192 (84 MB) 25; 1 x 4096 (4.5 MB) 9.  About 10 us are fixed: the launch
// 2.3, key counts, page ids and first rows one after the other 1.3 to 3.3, the
// LDS merge 2, the merge launch 3 to 5.  The scale bytes, a row's 4 to 16, cost 2
// to 10 % of the stages' time.  Tried: 64 keys a trip (spills with three
// workgroups a CU; with two, 25 -> 29 us for the 84 MB), two stages in flight
// with Q in LDS (slower), cached instead of non-temporal loads (slower from 84 MB on).
// ---------------------------------------------------------------------------
// NQ: 16-row blocks of queries.  Two for more than 16 rows alone: their registers and
// LDS leave a third fewer workgroups (16 rows on two blocks 58 -> 72 us, 93 -> 123).
// With 32 rows, 8 queries a sequence, 32 x 8192 keys take 77 to 79 us and 8 x 57000 (496
// MB) 123 to 129; with 32 / 1 heads 64 x 8192 (71 MB) 32 and 8 x 16384 (18 MB) 20, of
// which a wave's share is two stages and the partials half as many bytes as the keys.
template <int D, int NQ> struct Kv4Cfg {
    static constexpr int kWaves = 4;                          // workers per workgroup
    static constexpr int kThreads = 64 * kWaves;
    // Workgroups per CU, as many as registers and LDS hold (16 rows, D = 128: one
    // fewer, two, 58.0 -> 60.7 us for 32 x 8192 and 93 -> 104 for the 506 MB above; calls
    // whose share is a few stages a wave run up to 20 % faster or 12 % slower,
    // by how the shares fall on the heads).
    static constexpr int kPerCU = D == 64 ? (NQ == 1 ? 4 : 3) : D == 128 ? (NQ == 1 ? 3 : 2) : NQ == 1 ? 2 : 1;
    static constexpr int kSlot = NQ * 64 * D;                 // a wave's V rows in 16 bits; its partial
};
inline int kv4_workgroups(int D, int R, int cus) {
    const int one = D == 64 ? Kv4Cfg<64, 1>::kPerCU : D == 128 ? Kv4Cfg<128, 1>::kPerCU : Kv4Cfg<256, 1>::kPerCU;
    const int two = D == 64 ? Kv4Cfg<64, 2>::kPerCU : D == 128 ? Kv4Cfg<128, 2>::kPerCU : Kv4Cfg<256, 2>::kPerCU;
    return cus * (R <= 16 ? one : two);
}

template <bool kBF, int D, int NQ>
__global__ __launch_bounds__((Kv4Cfg<D, NQ>::kThreads), (Kv4Cfg<D, NQ>::kPerCU))
void kf_attn_decode_kv4_kernel(AttnParams p) {
    using Cfg = Kv4Cfg<D, NQ>;
    using E = Elem<kBF>;
    using X8 = typename E::x8;
    using SW = SwizzleRow<D>;
    constexpr int NW = Cfg::kWaves;
    constexpr int kWords = D / 32;                 // code words of a lane's row
    constexpr int kScales = D >= 256 ? 2 : 1;      // blocks of a lane's row
    constexpr int kChunks = D / 8;                 // 16-byte chunks of a V row in LDS
    constexpr int kRowBytes = 2 * D;
    constexpr int kNT = D / 16;                    // 16-row O^T tiles
    __shared__ __attribute__((aligned(1024))) char slots[NW * Cfg::kSlot];
    __shared__ float tail_m[NW * 16 * NQ], tail_l[NW * 16 * NQ];
    __shared__ int tail_grp[NW], tail_slot[NW], tail_ends[NW];
    __shared__ int blocks[64];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, q4 = lane >> 4;
    const int R = p.rows_per_group;
    const int wg = blockIdx.x;
    RaggedMap map;
    map.init(p, lane, wave, NW, blocks);
    const StageSplit parts = StageSplit::even(map.total, max(min((int)gridDim.x, map.total / NW), 1));
    const int wg_first = parts.first(wg), wg_stages = parts.first(wg + 1) - wg_first;
    if (wg_stages <= 0) return;    // workgroup-uniform
    const StageSplit waves = StageSplit::even(wg_stages, NW);
    const int first_pos = wg_first + waves.first(wave), end = wg_first + waves.first(wave + 1);
    const int worker = wg * NW + wave;

    char* const vs = slots + wave * Cfg::kSlot;
    const uint8_t* const Kp = reinterpret_cast<const uint8_t*>(p.K);
    const uint8_t* const Vp = reinterpret_cast<const uint8_t*>(p.V);
    const int sh = p.page_shift;
    const size_t page_bytes = (size_t)(17 * D / 32) << sh;
    const uint32_t scales_at = (uint32_t)(D / 2) << sh;
    const uint32_t code_off = col * (D / 2) + q4 * (D / 8);
    const uint32_t scale_off = col * (D / 32) + q4 * (D / 32) / 4;

    struct Stage {
        size_t at[2];       // the (page, head) of keys 0..15 and 16..31
        int row[2];         // their first row in it
        int k0, k1;         // first key; end of the keys
        int bad;            // invalid pages: bit 0 keys 0..15, bit 1 keys 16..31
    };
    struct PageIds {
        int id0, id1;
    };
    auto page_ids = [&](const RaggedSeg& s, int j) {
        const int k0 = s.key(j), pi = k0 >> sh;
        const int* tbl = p.block_table + (size_t)s.b * p.max_pages;
        // 16-row pages: the second half is the next page, if it has keys.
        return PageIds{uniform_load(tbl, pi), uniform_load(tbl, sh == 4 && k0 + 16 < s.kvb ? pi + 1 : pi)};
    };
    auto stage_at = [&](const RaggedSeg& s, int j, const PageIds& ids) {
        Stage st;
        st.k0 = s.key(j);
        st.k1 = min(s.kvb, st.k0 + kDecodeStage);
        const bool ok0 = (unsigned)ids.id0 < (unsigned)p.num_pages;
        const bool ok1 = (unsigned)ids.id1 < (unsigned)p.num_pages;
        // An invalid page reads the pool's first page.
        st.at[0] = ((size_t)(ok0 ? ids.id0 : 0) * p.heads_kv + s.h) * page_bytes;
        st.at[1] = ((size_t)(ok1 ? ids.id1 : 0) * p.heads_kv + s.h) * page_bytes;
        st.row[0] = st.k0 & ((1 << sh) - 1);
        st.row[1] = sh == 4 ? 0 : st.row[0] + 16;
        st.bad = (ok0 ? 0 : 1) | (ok1 ? 0 : 2);
        return st;
    };
    // A stage's K or V: pages hold whole halves, so every address is inside
    // the pool, also past the keys.
    struct Rows {
        uint32_t code[2][kWords];
        uint32_t scale[2];
    };
    auto load_rows = [&](const uint8_t* pool, const Stage& st, Rows& r) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint8_t* codes = pool + st.at[t] + (uint32_t)(st.row[t] * (D / 2));
            const uint8_t* scales = pool + st.at[t] + scales_at + (uint32_t)(st.row[t] * (D / 32));
            if constexpr (D == 64) {
                const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(codes + code_off));
                r.code[t][0] = v.x;
                r.code[t][1] = v.y;
            } else {
#pragma unroll
                for (int w = 0; w < kWords; w += 4) {
                    const u32x4 v = __builtin_nontemporal_load(
                        reinterpret_cast<const u32x4*>(codes + code_off + 4 * w));
#pragma unroll
                    for (int e = 0; e < 4; ++e) r.code[t][w + e] = v[e];
                }
            }
            if constexpr (kScales == 2)
                r.scale[t] = *reinterpret_cast<const uint16_t*>(scales + scale_off);
            else
                r.scale[t] = scales[scale_off];
        }
    };
    // (Exponent byte 255: the conversion takes the scale for a NaN, whatever the code, so
    // a block that held no finite values makes its scores, or its channels of O, NaN.)
    auto scale_of = [&](const Rows& r, int t, int j) {
        return __uint_as_float((j < 4 ? r.scale[t] & 0xffu : r.scale[t] >> 8) << 23);
    };

    X8 qf[NQ][kWords];
    f32x4 o[NQ][kNT];
    RowState st[NQ];
    int lim_min, lim_lane[NQ];   // keys that every row, and this lane's rows, see
    auto open_segment = [&](const RaggedSeg& c) {
        const uint16_t* Qg = p.Q + (size_t)(c.b * p.heads_kv + c.h) * R * D;
        lim_min = p.causal ? max(c.kvb - p.q_len + 1, 0) : c.kvb;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int row = min(16 * n + col, R - 1);
#pragma unroll
            for (int j = 0; j < kWords; ++j)
                qf[n][j] = *reinterpret_cast<const X8*>(Qg + (size_t)row * D + q4 * (D / 4) + 8 * j);
            lim_lane[n] = row_kv_limit(p, c.kvb, row % p.q_len);
            st[n] = RowState{-INFINITY, -INFINITY, 0.f, -INFINITY};
#pragma unroll
            for (int i = 0; i < kNT; ++i) o[n][i] = f32x4{};
        }
    };
    const float c = p.scale_log2, inv_c = 1.0f / c;

    Rows kr, vr;
    // One stage, cs, whose rows are on their way into kr and vr; with `more`,
    // the next one, which it returns, is requested as they become free.
    auto stage = [&](const Stage& cs, bool more, const RaggedSeg& nseg, int nj) {
        const PageIds ids = page_ids(nseg, nj);
        f32x4 s[NQ][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[n][t] = f32x4{};
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const X8 a = from_fp4x8<kBF>(kr.code[t][j], scale_of(kr, t, j));
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[n][t] = E::mfma16(a, qf[n][j], s[n][t]);
            }
        }
        const Stage ns = stage_at(nseg, nj, ids);
        if (more) load_rows(Kp, ns, kr);
        if (cs.k1 < cs.k0 + kDecodeStage || cs.k1 > lim_min || cs.bad) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int lim = min(cs.k1, lim_lane[n]) - cs.k0;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * t + 4 * q4 + r >= lim || (cs.bad >> t & 1)) s[n][t][r] = -INFINITY;
            }
            // V rows past the keys or of an invalid page may hold anything:
            // zeros, so that P = 0 meets finite values.
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (cs.k0 + 16 * t + col >= cs.k1 || (cs.bad >> t & 1)) {
#pragma unroll
                    for (int w = 0; w < kWords; ++w) vr.code[t][w] = 0;
                    vr.scale[t] = 0x7f7f;
                }
        }
        X8 pb[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float mx = s[n][0][0];
#pragma unroll
            for (int r = 1; r < 8; ++r) mx = fmaxf(mx, s[n][r >> 2][r & 3]);
            mx = reduce_mod<16, true>(mx);
            RowState& rs = st[n];
            rs.rmax = fmaxf(rs.rmax, mx);
            const bool need = mx > rs.thr;
            if (__any(need)) {
                const float mt = mx * c;
                const float mnew = need ? mt : rs.m;
                const float alpha = need ? exp2_hw(rs.m - mt) : 1.0f;
                rs.l *= alpha;
#pragma unroll
                for (int i = 0; i < kNT; ++i) o[n][i] *= alpha;
                rs.m = mnew;
                rs.thr = (mnew + kLazyRescaleLog2) * inv_c;
            }
            // A row without a key so far keeps m = -inf and gets P = 0.
            const float neg_m = rs.m == -INFINITY ? 0.f : -rs.m;
            f32x8 e;
#pragma unroll
            for (int r = 0; r < 8; ++r) e[r] = exp2_hw(fmaf(s[n][r >> 2][r & 3], c, neg_m));
            rs.l += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
            pb[n] = round8<kBF>(e);    // as the product takes it (see packed_exp); summed in fp32
        }
        // V rows to LDS (chunks XOR-swizzled by the row), back as V^T.
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int row = 16 * t + col;
#pragma unroll
            for (int j = 0; j < kWords; ++j)
                *reinterpret_cast<X8*>(vs + row * kRowBytes + (((q4 * kWords + j) ^ SW::h(row)) % kChunks) * 16) =
                    from_fp4x8<kBF>(vr.code[t][j], scale_of(vr, t, j));
        }
        if (more) load_rows(Vp, ns, vr);
        wave_lds_sync();
        const int v_row = 4 * q4 + (col >> 2);
#pragma unroll
        for (int i = 0; i < kNT; ++i) {
            const int d = 16 * i + 4 * (col & 3);
            const int off = v_row * kRowBytes + (((d >> 3) ^ SW::h(v_row)) % kChunks) * 16 + ((d >> 2) & 1) * 8;
            const f16x4 lo = lds_read_tr16(vs + off), hi = lds_read_tr16(vs + off + 16 * kRowBytes);
            const X8 a = __builtin_bit_cast(X8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int n = 0; n < NQ; ++n) o[n][i] = E::mfma16(a, pb[n], o[n][i]);
        }
        wave_lds_sync();
        return ns;
    };

    int tgrp = -1, tslot = 0, tends = 0;  // the worker's partial last segment
    if (first_pos < end) {
        int pos = first_pos;     // global stage at which `cur` starts
        RaggedSeg cur = map.find(p, lane, pos, end);
        Stage cs = stage_at(cur, 0, page_ids(cur, 0));
        load_rows(Kp, cs, kr);
        load_rows(Vp, cs, vr);
        open_segment(cur);
        int j = 0;
        for (int left = end - first_pos; left > 0; --left) {
            const bool seg_end = j + 1 == cur.n;
            // The stage after this one; past the segment's last it is the
            // next head's first, or the next sequence's that has keys (after
            // the share's last, this one again, not requested).
            RaggedSeg nxt = cur;
            if (seg_end && left > 1) {
                const int npos = pos + cur.n;
                if (cur.h + 1 < p.heads_kv)
                    nxt = RaggedSeg{cur.b, cur.h + 1, 0, min(cur.T, end - npos), cur.T, cur.kvb, 0};
                else
                    nxt = map.find(p, lane, npos, end);
            }
            cs = stage(cs, left > 1, nxt, left == 1 ? j : seg_end ? 0 : j + 1);
            ++j;
            if (!seg_end) continue;

            const int grp = cur.b * p.heads_kv + cur.h;
            const int slot = 2 * worker + (pos != first_pos ? 1 : 0);
            const bool whole = cur.n == cur.T;
            // The worker of a head's first stage tells the merge where the
            // head's partials are (see kf_attn_decode_ragged_kernel).
            if (cur.t0 == 0 && lane == 0) {
                const int z = pos + cur.T;                  // end of the head
                const int ep = parts.part_of(z - 1);        // part of its last stage
                int groups = 1;
                uint32_t alone = ~0u;
                if (!whole) {
                    const int elo = parts.first(ep);
                    const StageSplit ew = StageSplit::even(parts.first(ep + 1) - elo, NW);
                    const int ewave = ew.part_of(z - 1 - elo);
                    const bool tail = z == elo + ew.first(ewave + 1);  // that wave's last segment
                    groups = ep - wg + (tail || ewave > 0 ? 1 : 0);
                    if (!tail) alone = 2 * (ep * NW + ewave);
                }
                p.ragged_heads[grp] = u32x4{(uint32_t)slot, (uint32_t)groups, alone, 2u * NW};
            }
            if (!whole && left == 1) {
                tgrp = grp;
                tslot = slot;
                tends = (cur.t0 == 0 ? 1 : 0) | (cur.t0 + cur.n == cur.T ? 2 : 0);
            } else {
                // A whole head's final rows, or the partial of a head that
                // ended with this worker's first segment.
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const float l = reduce_mod<16, false>(st[n].l);
                    const bool none = st[n].rmax == -INFINITY;
                    const float beta = none ? 0.f : rebase_factor(st[n].m, st[n].rmax, c);
                    const float m_nat = none ? -INFINITY : st[n].rmax * p.scale;
                    const int row = 16 * n + col;
                    if (row >= R) continue;
                    const size_t ri = (size_t)grp * R + row, pi = (size_t)slot * R + row;
                    const float f = !whole ? beta : l > 0.f ? 1.0f / l : 0.f;
#pragma unroll
                    for (int i = 0; i < kNT; ++i) {
                        const int d = 16 * i + 4 * q4;
                        if (whole)
                            store_out4(p, ri * D + d, o[n][i] * f);
                        else
                            store_out4_as<kOutPartial>(p, pi * D + d, o[n][i] * f);
                    }
                    if (q4 == 0) {
                        if (whole) {
                            store_stats(p, ri, m_nat, l * beta);
                        } else {
                            p.Mpart[pi] = m_nat;
                            p.Lpart[pi] = l * beta;
                        }
                    }
                }
            }
            if (left > 1) {
                pos += cur.n;
                cur = nxt;
                j = 0;
                open_segment(cur);
            }
        }
    }

    // ---- The workers' last segments, merged per head. ----
    constexpr int kRowsQ = 16 * NQ;
    if (tgrp >= 0) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float l = reduce_mod<16, false>(st[n].l);
            const bool none = st[n].rmax == -INFINITY;
            const float beta = none ? 0.f : rebase_factor(st[n].m, st[n].rmax, c);
            const int row = 16 * n + col;
            if (row >= R) continue;
            float* dst = reinterpret_cast<float*>(vs) + row * D;
#pragma unroll
            for (int i = 0; i < kNT; ++i)   // chunks XOR-ed by the row, against bank conflicts
                *reinterpret_cast<f32x4*>(dst + ((4 * i + q4) ^ (row & 7)) * 4) = o[n][i] * beta;
            if (q4 == 0) {
                tail_m[wave * kRowsQ + row] = none ? -INFINITY : st[n].rmax * p.scale;
                tail_l[wave * kRowsQ + row] = l * beta;
            }
        }
    }
    if (lane == 0) {
        tail_grp[wave] = tgrp;
        tail_slot[wave] = tslot;
        tail_ends[wave] = tends;
    }
    __syncthreads();
    // Runs of workers on one head: bit w of `live` where worker w has a
    // partial, of `heads` where a run starts (a worker without one ends it).
    const int tg = lane < NW ? tail_grp[lane] : -1;
    const int tg_before = __shfl_up(tg, 1);
    const uint32_t live = (uint32_t)__ballot(tg >= 0);
    const uint32_t heads = (uint32_t)__ballot(tg >= 0 && (lane == 0 || tg != tg_before));
    for (uint32_t left = heads; left;) {
        const int w0 = __builtin_ctz(left);
        left &= left - 1;
        const uint32_t run = live & ((left ? left & -left : 1u << NW) - 1) & ~((1u << w0) - 1);
        const int w1 = w0 + __builtin_popcount(run);  // past the run's last
        const int grp = __builtin_amdgcn_readlane(tg, w0);
        // The run holds the whole head: final rows.
        const bool whole = ((tail_ends[w0] & 1) != 0) && ((tail_ends[w1 - 1] & 2) != 0);
        const int slot = tail_slot[w0];
        for (int i = tid; i < R * (D / 4); i += Cfg::kThreads) {
            const int mrow = i / (D / 4), cc = i % (D / 4);
            float mw[NW], lw[NW];
            f32x4 ow[NW];
            // Every worker's, so that the loads are in flight together; those
            // outside the run count for nothing.
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const bool in = w >= w0 && w < w1;
                mw[w] = in ? tail_m[w * kRowsQ + mrow] : -INFINITY;
                lw[w] = tail_l[w * kRowsQ + mrow];
                ow[w] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(slots + w * Cfg::kSlot) +
                                                        mrow * D + (cc ^ (mrow & 7)) * 4);
            }
            float m = mw[0];
#pragma unroll
            for (int w = 1; w < NW; ++w) m = fmaxf(m, mw[w]);
            float l = 0.f;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w)
                if (w >= w0 && w < w1) {
                    // Weight 0 for a row without a key here, whose sums are 0.
                    const float wt = mw[w] == -INFINITY ? 0.f : exp2_hw((mw[w] - m) * kLog2e);
                    l += wt * lw[w];
                    acc += wt * ow[w];
                }
            const size_t ri = (size_t)grp * R + mrow, pi = (size_t)slot * R + mrow;
            if (whole) {
                store_out4(p, ri * D + 4 * cc, acc * (l > 0.f ? 1.0f / l : 0.f));
                if (cc == 0) store_stats(p, ri, m, l);
            } else {
                *reinterpret_cast<f32x4*>(p.Opart + pi * D + 4 * cc) = acc;
                if (cc == 0) {
                    p.Mpart[pi] = m;
                    p.Lpart[pi] = l;
                }
            }
        }
    }
}

}  // namespace kf
