// cache_kernels.h -- a paged K/V cache in 16 bits: new tokens written into it, and
// keys evicted from it by the attention weight that they have gathered.
//
// Pools are [num_pages][H_kv][page_size][D] (attn_decode_paged's) and the weights
// [num_pages][H_kv][page_size] in fp32.
#pragma once

#include <utility>

#include "kv4_kernels.h"

namespace kf {

// ---------------------------------------------------------------------------
// New tokens into the pages: copies of 16 bytes, the places found and the items walked
// through as in the 4-bit cache's kernels.  Bound by HBM: 16 prompts of 32 to 4096 tokens, 8
// heads of 128, 91 MB in 16.3 us, a copy's rate; one token of each of 64 sequences 4.2.
// ---------------------------------------------------------------------------
struct KvAppendParams : Kv4Params {  // x, pages, strides; page_bytes of the 16-bit page
    float* weights;                  // null: none
};

template <int D>
__global__ __launch_bounds__(kKv4Threads)
void kf_kv_append_kernel(KvAppendParams p) {
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
            if (its[u].t >= n) continue;
            const Kv4Row to = places[its[u].t];
            if (to.page < 0) continue;
            const int h = its[u].rest / kChunks, c = its[u].rest % kChunks;
            const size_t at = ((size_t)to.page * p.heads + h) * p.page_bytes;
#pragma unroll
            for (int s = 0; s < 2; ++s)
                *reinterpret_cast<u32x4*>(p.pages[s] + at + (size_t)to.row * (2 * D) + 16 * c) = raw[u][s];
            if (p.weights && c == 0) p.weights[(((size_t)to.page * p.heads + h) << p.page_shift) + to.row] = 0.f;
        }
    }
}

// ---------------------------------------------------------------------------
// Eviction.  Sequence b is cut from n keys to m = min(n, budgets[b]); of every KV head the last r =
// min(recent, m) stay, and of the n - r old ones the k = m - r of largest weight.
// Attention does not depend on the order of the keys, so that of the old ones only those
// move that have to: the kept ones in places from k on go to the places below k that were
// freed, the i-th to the i-th, and the last r to k .. m - 1, in order.  (Closing
// the gaps in order would move half a head's keys where one of them goes.)
//
// Select: a workgroup per (sequence, KV head) finds the k-th largest weight by three
// counts of 12, 10 and 10 bits and writes the moves to the workspace.  Bound by round
// trips and barriers for few keys (4097 keys of 256 heads 13 us), by instructions of one
// CU for many (65537 keys of one head 62 us).  Move: the rows of K and V and the weights, by these
// lists, at a copy's rate (16 sequences of 4096 to 32768 keys, 8 heads of 128, to half: 467 MB in
// 95 us).
// ---------------------------------------------------------------------------
struct EvictParams {
    uint8_t* pages[2];          // K, V
    uint32_t* weights;          // bits of fp32
    const int* block_table;     // [n_seqs][max_pages]
    const int* kv_lens;         // [n_seqs]
    const int* budgets;         // [n_seqs]
    int* kept;                  // [n_seqs], may be kv_lens or budgets
    int n_seqs, heads, recent, max_pages, page_shift, num_pages, capacity;
    int parts;                  // workgroups of a head that move keys behind the new end
    int* cuts;                  // [n_seqs * heads][4]: n, m, moves among the old keys (-1: none of the head's
                                // rows move), how many of them are from places below m
    int* moves;                 // [n_seqs * heads][capacity]: where to, from the middle on where from
};

// One sequence's table: the place of a key.
struct EvictTable {
    const int* table;
    int heads, head, shift;
    __device__ __forceinline__ size_t at(int page, int key) const {   // of a pool seen as [rows]
        return (((size_t)page * heads + head) << shift) + (key & ((1 << shift) - 1));
    }
    __device__ __forceinline__ size_t row(int key) const { return at(table[key >> shift], key); }
    // Of a key that the workspace names, one of n (of weights that change while they are
    // looked through, it may hold none).
    __device__ __forceinline__ size_t listed(int key, int n) const { return row(min(max(key, 0), n - 1)); }
};

// A weight's place in the order, as an unsigned number: larger weights larger, NaN
// above all, -0 as 0.
__device__ __forceinline__ uint32_t evict_order(uint32_t u) {
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if (u == 0x80000000u) u = 0;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;

// Bits of lanes below this one.
__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}
// f(std::integral_constant<int, i>) for i = 0 .. n - 1, whatever the size of f.
template <class F, int... I>
__device__ __forceinline__ void evict_unrolled(const F& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}

constexpr int kSelectHist = (1 << 12) + 2 * (1 << 10) + 3 * 256;   // the bins of all three counts
constexpr int kSelectMost = 72, kSelectPages = kSelectMost * kSelectThreads / 16;
struct EvictShared {
    __attribute__((aligned(16))) int hist[kSelectHist];
    int pages[kSelectPages];          // of the first keys
    int wave_sums[4][kSelectWaves];
};

// The cut of one head from n to m keys.  kPer: up to so many old keys of a thread are read
// once, into registers; 0: read anew by every pass.
template <int kPer>
__device__ __forceinline__ void evict_select(const EvictParams& p, const EvictTable& tb, EvictShared& sh, int grp, int n, int m) {
    constexpr int kHeld = kPer > 0 ? kPer : 1, kSelectAhead = 8;   // weights of a thread on their way at a time
    static_assert(kPer <= kSelectMost && kPer % kSelectAhead == 0, "whole batches");
    int* const hist = sh.hist;
    const int* const pages = sh.pages;
    auto& wave_sums = sh.wave_sums;
    // (Opaque: nothing that is derived from it is made for the forms that are not taken.)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = min(p.recent, m), k = m - r, old = n - r;
    int* const cuts = p.cuts + 4 * (size_t)grp;
    // Every wave has a run of the old keys, 64 at a time.
    const int its = (old + kSelectThreads - 1) / kSelectThreads, i0 = wave * its * 64;
    const auto place = [&](int i) { return i0 + 64 * i + lane; };
    uint32_t held[kHeld];
    if constexpr (kPer > 0) {
        evict_unrolled([&](auto batch) {
            constexpr int j = decltype(batch)::value * kSelectAhead;
            if (j >= its) return;
            uint32_t raw[kSelectAhead];
#pragma unroll
            for (int u = 0; u < kSelectAhead; ++u) {
                raw[u] = 0;
                if (j + u < its) {
                    const int at = min(place(j + u), old - 1);
                    raw[u] = p.weights[tb.at(pages[at >> p.page_shift], at)];
                }
            }
#pragma unroll
            for (int u = 0; u < kSelectAhead; ++u) held[j + u] = place(j + u) < old ? evict_order(raw[u]) : 0;
        }, std::make_integer_sequence<int, kPer / kSelectAhead>{});
    }
    // f(place of lane 0, a weight's order) for all of the wave's keys, 64 at a time and in order.  Lanes
    // past the last key have 0, less than any weight's order.
    const auto each = [&](auto f) {
        if constexpr (kPer > 0) {
            evict_unrolled([&](auto index) {
                constexpr int i = decltype(index)::value;
                if (i < its) f(i0 + 64 * i, held[i]);
            }, std::make_integer_sequence<int, kPer>{});
        } else {
            for (int i = 0; i < its; ++i) {
                const int at = min(place(i), old - 1);
                f(i0 + 64 * i, place(i) < old ? evict_order(p.weights[tb.row(at)]) : 0);
            }
        }
    };

    // The k-th largest of the old weights: `top` so far of its bits, `need` how many of
    // those that share them are kept, of `alike`.
    uint32_t top = 0xffffffffu;
    int need = 0, alike = 1;
    if (k > 0) {
        top = 0;
        need = k;
        const auto count_digit = [&](auto shift_c, auto bits_c, int* hist) {
            // Bins lie in 64 runs, each padded by four: the reads below go to all banks.
            constexpr int shift = decltype(shift_c)::value, bits = decltype(bits_c)::value, kBins = 1 << bits;
            constexpr int kRun = kBins / 64;
            const auto slot = [](int bin) { return bin + bin / kRun * 4; };
            each([&](int, uint32_t u) {
                const int bin = u >> shift & (kBins - 1);
                if constexpr (shift + bits < 32) {
                    if ((u >> (shift + bits)) == (top >> (shift + bits))) atomicAdd(&hist[slot(bin)], 1);
                } else if (const int lead = __builtin_amdgcn_readfirstlane(bin); __all(bin == lead)) {
                    if (lane == 0) atomicAdd(&hist[slot(lead)], 64);       // one place for 64 lanes is slow
                } else {
                    atomicAdd(&hist[slot(bin)], 1);
                }
            });
            __syncthreads();
            // Every wave finds the bin: its run, of which lane l has the one 63 - l, and then it in the run.
            int sum = 0;
#pragma unroll
            for (int e = 0; e < kRun; e += 4) {
                const int4 v = *reinterpret_cast<const int4*>(&hist[slot((63 - lane) * kRun) + e]);
                sum += (v.x + v.y) + (v.z + v.w);
            }
            int inc = wave_scan(sum);
            // (Of weights that change meanwhile there may be none.)
            const int run = __builtin_ctzll(__ballot(inc >= need) | 1ull << 63);
            need -= __builtin_amdgcn_readlane(inc, run) - __builtin_amdgcn_readlane(sum, run);
            sum = lane < kRun ? hist[slot((63 - run) * kRun) + kRun - 1 - lane] : 0;
            inc = wave_scan(sum);
            const int e = __builtin_ctzll(__ballot(inc >= need) | 1ull << (kRun - 1));
            alike = __builtin_amdgcn_readlane(sum, e);
            need -= __builtin_amdgcn_readlane(inc, e) - alike;
            top |= (uint32_t)((63 - run) * kRun + kRun - 1 - e) << shift;
        };
        count_digit(std::integral_constant<int, 20>{}, std::integral_constant<int, 12>{}, hist);
        count_digit(std::integral_constant<int, 10>{}, std::integral_constant<int, 10>{}, hist + (1 << 12) + 256);
        count_digit(std::integral_constant<int, 0>{}, std::integral_constant<int, 10>{}, hist + (1 << 12) + (1 << 10) + 512);
    }
    // Of the keys of the k-th weight the first `need` are kept; mostly that is all of them.
    const bool tie = need < alike;
    int before = 0;
    if (tie) {
        int equal = 0;
        each([&](int, uint32_t u) { equal += __popcll(__ballot(u == top)); });
        if (lane == 0) wave_sums[0][wave] = equal;
        __syncthreads();
        for (int w = 0; w < wave; ++w) before += wave_sums[0][w];
    }
    // Of 64 keys which are kept; `ties` counts those of the k-th weight.
    const auto kept_of = [&](uint32_t u, int& ties) {
        if (!tie) return (uint64_t)__ballot(u >= top);
        const uint64_t same = __ballot(u == top);
        const uint64_t keep = __ballot(u > top || (u == top && ties + lanes_below(same) < need));
        ties += __popcll(same);
        return keep;
    };
    // Those of 64 places from c on that are below x.
    const auto low = [](int c, int x) { return c + 64 <= x ? ~0ull : c >= x ? 0ull : (1ull << (x - c)) - 1; };
    // The places that are freed, the keys that move, and those of them below the new end.
    int freed = 0, moved = 0, near = 0, ties = before;
    each([&](int c, uint32_t u) {
        const uint64_t keep = kept_of(u, ties), front = low(c, k);
        freed += __popcll(front & ~keep);
        moved += __popcll(keep & ~front);
        near += __popcll(keep & ~front & low(c, m));
    });
    if (lane == 0) {
        wave_sums[1][wave] = freed;
        wave_sums[2][wave] = moved;
        wave_sums[3][wave] = near;
    }
    __syncthreads();
    int to = 0, from = 0, all_freed = 0, all_moved = 0, all_near = 0;
    for (int w = 0; w < kSelectWaves; ++w) {
        if (w < wave) {
            to += wave_sums[1][w];
            from += wave_sums[2][w];
        }
        all_freed += wave_sums[1][w];
        all_moved += wave_sums[2][w];
        all_near += wave_sums[3][w];
    }
    // As many places are freed as keys move, no more than half of the old keys (of weights
    // that change meanwhile, as of a page that two sequences share, perhaps not).
    const int half = p.capacity / 2, count = min(min(all_freed, all_moved), half);
    int* const list = p.moves + (size_t)grp * p.capacity;
    int* const sources = list + half;
    ties = before;
    each([&](int c, uint32_t u) {
        const uint64_t keep = kept_of(u, ties), front = low(c, k), fs = front & ~keep, vs = keep & ~front;
        const int f_at = to + lanes_below(fs), v_at = from + lanes_below(vs);
        if ((fs >> lane & 1) && f_at < half) list[f_at] = c + lane;
        if ((vs >> lane & 1) && v_at < half) sources[v_at] = c + lane;
        to += __popcll(fs);
        from += __popcll(vs);
    });
    if (tid == 0) {
        cuts[2] = count;
        cuts[3] = min(all_near, count);
    }
}

// By how many old keys a thread has: up to 16 or 72 in registers (4097 keys of 256 heads 13.3 us
// by 16 and 22.5 by 80 once, whose passes step over what they do not need; 65537 keys of one head 62,
// and 135 without registers).
__global__ __launch_bounds__(kSelectThreads)
void kf_kv_evict_select_kernel(EvictParams p) {
    __shared__ EvictShared sh;
    const int tid = threadIdx.x;
    const int grp = blockIdx.x, b = grp / p.heads, head = grp % p.heads;
    const EvictTable tb{p.block_table + (size_t)b * p.max_pages, p.heads, head, p.page_shift};
    const int n = __builtin_amdgcn_readfirstlane(min(max(p.kv_lens[b], 0), p.capacity));
    const int m = __builtin_amdgcn_readfirstlane(min(max(p.budgets[b], 0), n));
    for (int i = tid; i < kSelectHist; i += kSelectThreads) sh.hist[i] = 0;
    // A key on no valid page has no place: the sequence is left as it is.
    bool bad = false;
    if (m < n)
        for (int i = tid; i <= (n - 1) >> p.page_shift; i += kSelectThreads) {
            const int id = tb.table[i];
            bad |= (unsigned)id >= (unsigned)p.num_pages;
            if (i < kSelectPages) sh.pages[i] = id;
        }
    const bool left = __syncthreads_or(bad) != 0 || m == n;
    int* const cuts = p.cuts + 4 * (size_t)grp;
    if (tid == 0) {
        cuts[0] = n;
        cuts[1] = m;
        if (left) cuts[2] = -1;
    }
    // (kept may be the array that the other heads' workgroups still read: the mover
    // writes it.)
    if (left) return;
    const int per = (n - min(p.recent, m) + kSelectThreads - 1) / kSelectThreads;
    if (per <= 16)
        evict_select<16>(p, tb, sh, grp, n, m);
    else if (per <= kSelectMost)
        evict_select<kSelectMost>(p, tb, sh, grp, n, m);
    else
        evict_select<0>(p, tb, sh, grp, n, m);
}

// Keys from below the new end m have to be read before the last r are written over them:
// these, and the last r in order, are moved by a workgroup per (sequence, KV head), tensor and
// 128 bytes of a row, in which rows of other segments lie elsewhere.  The others are
// from places that are not written and go to freed ones that are not read: whole rows
// by `parts` more workgroups of the head, in any order.
constexpr int kMoveThreads = 256;
constexpr int kMoveAhead = 4;          // rows of a thread on their way

template <int D>
__global__ __launch_bounds__(kMoveThreads)
void kf_kv_evict_move_kernel(EvictParams p) {
    constexpr int kSegments = 2 * (D / 64);
    const int tid = threadIdx.x, groups = p.n_seqs * p.heads;
    const bool bulk = blockIdx.x >= (unsigned)(groups * kSegments);
    const int item = bulk ? blockIdx.x - groups * kSegments : blockIdx.x, of = bulk ? p.parts : kSegments;
    const int grp = item / of, seg = item % of, b = grp / p.heads, head = grp % p.heads;
    const int* const cuts = p.cuts + 4 * (size_t)grp;
    const int n = cuts[0], m = cuts[1], count = cuts[2];
    if (!bulk && head == 0 && seg == 0 && tid == 0) p.kept[b] = count < 0 ? n : m;
    if (count < 0) return;
    const int near = cuts[3];
    const EvictTable tb{p.block_table + (size_t)b * p.max_pages, p.heads, head, p.page_shift};
    const int r = min(p.recent, m), k = m - r, old = n - r;
    const int* const list = p.moves + (size_t)grp * p.capacity;
    const int* const sources = list + p.capacity / 2;
    if (bulk) {
        constexpr int kLanes = D / 8, kRows = kMoveThreads / kLanes, kStep = kRows * kMoveAhead;
        const int chunk = tid % kLanes;
        const auto at = [&](int s, size_t row) { return reinterpret_cast<u32x4*>(p.pages[s] + row * (2 * D)) + chunk; };
        for (int i0 = near + seg * kStep; i0 < count; i0 += p.parts * kStep) {
            size_t from[kMoveAhead], to[kMoveAhead];
            u32x4 v[kMoveAhead][2];
            uint32_t w[kMoveAhead];
#pragma unroll
            for (int u = 0; u < kMoveAhead; ++u) {
                const int i = min(i0 + u * kRows + tid / kLanes, count - 1);
                from[u] = tb.listed(sources[i], n);
                to[u] = tb.listed(list[i], n);
            }
#pragma unroll
            for (int u = 0; u < kMoveAhead; ++u) {
                v[u][0] = *at(0, from[u]);
                v[u][1] = *at(1, from[u]);
                w[u] = chunk == 0 ? p.weights[from[u]] : 0;
            }
#pragma unroll
            for (int u = 0; u < kMoveAhead; ++u) {
                if (i0 + u * kRows + tid / kLanes >= count) continue;
                *at(0, to[u]) = v[u][0];
                *at(1, to[u]) = v[u][1];
                if (chunk == 0) p.weights[to[u]] = w[u];
            }
        }
        return;
    }
    constexpr int kRows = kMoveThreads / 8, kStep = kRows * kMoveAhead;   // 8 lanes of 16 bytes a row
    uint8_t* const pool = p.pages[seg / (D / 64)] + seg % (D / 64) * 128 + tid % 8 * 16;
    const auto at = [&](size_t row) { return reinterpret_cast<u32x4*>(pool + row * (2 * D)); };
    const bool weigh = seg == 0 && tid % 8 == 0;          // moves the weights too
    // `count` rows, from and to of the i-th; a place is written when all that is in front of it in
    // the list, and kStep rows from it on, has been read.
    const auto move = [&](int count, auto from_of, auto to_of) {
        for (int i0 = 0; i0 < count; i0 += kStep) {
            u32x4 v[kMoveAhead];
            uint32_t w[kMoveAhead];
#pragma unroll
            for (int u = 0; u < kMoveAhead; ++u) {
                const size_t from = from_of(min(i0 + u * kRows + tid / 8, count - 1));
                v[u] = *at(from);
                w[u] = weigh ? p.weights[from] : 0;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kMoveAhead; ++u) {
                const int i = i0 + u * kRows + tid / 8;
                if (i >= count) continue;
                const size_t to = to_of(i);
                *at(to) = v[u];
                if (weigh) p.weights[to] = w[u];
            }
        }
    };
    move(near, [&](int i) { return tb.listed(sources[i], n); }, [&](int i) { return tb.listed(list[i], n); });
    __syncthreads();
    move(r, [&](int i) { return tb.row(old + i); }, [&](int i) { return tb.row(k + i); });
}

}  // namespace kf
