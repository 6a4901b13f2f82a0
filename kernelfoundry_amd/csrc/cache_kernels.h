// cache_kernels.h -- a paged K/V cache in 16 bits: new tokens written into it, and
// keys evicted from it by the attention weight that they have gathered.
//
// Pools are [num_pages][H_kv][page_size][D] (attn_decode_paged's) and the weights
// [num_pages][H_kv][page_size] in fp32.
#pragma once

#include "kv4_kernels.h"

namespace kf {

// ---------------------------------------------------------------------------
// New tokens into the pages: copies of 16 bytes, the places found and the items walked
// through as in the 4-bit cache's kernels.
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
// Attention does not depend on the order of the old keys, so that only those move
// that have to: the kept ones in places from k on go to the places below k that were
// freed, the i-th to the i-th, and the last r to k .. m - 1, in order.  (Closing
// the gaps in order would move half a head's keys where one of them goes.)
//
// Select: a workgroup per (sequence, KV head) finds the k-th largest weight by four
// counts of 8 bits each, writes the moves to the workspace and moves the weights.
// Move: the rows of K and V, by these lists.
// ---------------------------------------------------------------------------
struct EvictParams {
    uint8_t* pages[2];          // K, V
    uint32_t* weights;          // bits of fp32
    const int* block_table;     // [n_seqs][max_pages]
    const int* kv_lens;         // [n_seqs]
    const int* budgets;         // [n_seqs]
    int* kept;                  // [n_seqs], may be kv_lens or budgets
    int n_seqs, heads, recent, max_pages, page_shift, num_pages, capacity;
    int* counts;                // [n_seqs * heads]: moves among the old keys, -1: none of the head's rows move
    int* cuts;                  // [n_seqs * heads][2]: n, m
    int* moves;                 // [n_seqs * heads][capacity]: where to, from the middle on where from
};

// One sequence's table: the place of a key.
struct EvictTable {
    const int* table;
    int heads, head, shift;
    __device__ __forceinline__ size_t row(int key) const {   // of a pool seen as [rows]
        return (((size_t)table[key >> shift] * heads + head) << shift) + (key & ((1 << shift) - 1));
    }
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

__global__ __launch_bounds__(kSelectThreads)
void kf_kv_evict_select_kernel(EvictParams p) {
    __shared__ int hist[kSelectWaves][256];
    __shared__ int wave_sums[3][kSelectWaves];
    __shared__ int found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = blockIdx.x, b = grp / p.heads, head = grp % p.heads;
    const EvictTable tb{p.block_table + (size_t)b * p.max_pages, p.heads, head, p.page_shift};
    const int n = min(max(p.kv_lens[b], 0), p.capacity), m = min(max(p.budgets[b], 0), n);
    // A key on no valid page has no place: the sequence is left as it is.
    bool bad = false;
    if (m < n)
        for (int i = tid; i <= (n - 1) >> p.page_shift; i += kSelectThreads)
            bad |= (unsigned)tb.table[i] >= (unsigned)p.num_pages;
    const bool left = __syncthreads_or(bad) != 0 || m == n;
    const int r = min(p.recent, m), k = m - r, old = n - r;
    if (tid == 0) {
        p.cuts[2 * grp] = n;
        p.cuts[2 * grp + 1] = m;
        if (left) p.counts[grp] = -1;
    }
    // (kept may be the array that the other heads' workgroups still read: the mover
    // writes it.)
    if (left) return;
    const auto order_at = [&](int i) { return evict_order(p.weights[tb.row(i)]); };

    // The k-th largest of the old weights: `top` so far of its bits, `need` how many of
    // those that share them are kept.
    uint32_t top = 0;
    int need = k;
    if (k > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < kSelectWaves * 256; i += kSelectThreads) (&hist[0][0])[i] = 0;
            __syncthreads();
            for (int i = tid; i < old; i += kSelectThreads) {
                const uint32_t u = order_at(i);
                if (shift == 24 || (u >> (shift + 8)) == (top >> (shift + 8))) atomicAdd(&hist[wave][u >> shift & 255], 1);
            }
            __syncthreads();
            if (wave == 0) {
                // Lane l has the bins 255 - 4 l down to 252 - 4 l.
                int bins[4], sum = 0;
                for (int e = 0; e < 4; ++e) {
                    bins[e] = 0;
                    for (int w = 0; w < kSelectWaves; ++w) bins[e] += hist[w][255 - 4 * lane - e];
                    sum += bins[e];
                }
                int above = wave_scan(sum) - sum;
                if (above < need && above + sum >= need) {
                    int e = 0;
                    while (above + bins[e] < need) above += bins[e++];
                    found[0] = 255 - 4 * lane - e;
                    found[1] = need - above;
                }
            }
            __syncthreads();
            top |= (uint32_t)found[0] << shift;
            need = found[1];
        }
    }
    // Every wave has a run of the old keys.  First the ones of the k-th weight, of which the
    // first `need` are kept, then the places that are freed and the keys that move.
    const int run = (old + kSelectThreads - 1) / kSelectThreads * 64, i0 = min(wave * run, old), i1 = min(i0 + run, old);
    int equal = 0;
    if (k > 0)
        for (int i = i0; i < i1; i += 64) {
            const bool in = i + lane < i1;
            equal += __popcll(__ballot(in && order_at(min(i + lane, old - 1)) == top));
        }
    if (lane == 0) wave_sums[0][wave] = equal;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; ++w) before += wave_sums[0][w];
    const uint64_t below = (1ull << lane) - 1;
    // Of 64 keys which are kept; `ties` counts those of the k-th weight.
    const auto kept_of = [&](int i, int& ties) {
        const bool in = i + lane < i1;
        const uint32_t u = k > 0 ? order_at(min(i + lane, old - 1)) : 0;
        const uint64_t same = __ballot(in && u == top);
        const bool keep = in && k > 0 && (u > top || (u == top && ties + __popcll(same & below) < need));
        ties += __popcll(same);
        return keep;
    };
    int freed = 0, moved = 0, ties = before;
    for (int i = i0; i < i1; i += 64) {
        const bool keep = kept_of(i, ties);
        freed += __popcll(__ballot(i + lane < min(i1, k) && !keep));
        moved += __popcll(__ballot(i + lane >= k && keep));
    }
    if (lane == 0) {
        wave_sums[1][wave] = freed;
        wave_sums[2][wave] = moved;
    }
    __syncthreads();
    int to = 0, from = 0, all_freed = 0, all_moved = 0;
    for (int w = 0; w < kSelectWaves; ++w) {
        if (w < wave) {
            to += wave_sums[1][w];
            from += wave_sums[2][w];
        }
        all_freed += wave_sums[1][w];
        all_moved += wave_sums[2][w];
    }
    // As many places are freed as keys move, no more than half of the old keys (of weights
    // that change meanwhile, as of a page that two sequences share, perhaps not).
    const int half = p.capacity / 2, count = min(min(all_freed, all_moved), half);
    int* const list = p.moves + (size_t)grp * p.capacity;
    int* const sources = list + half;
    ties = before;
    for (int i = i0; i < i1; i += 64) {
        const bool keep = kept_of(i, ties);
        const bool f = i + lane < min(i1, k) && !keep, v = i + lane >= k && keep;
        const uint64_t fs = __ballot(f), vs = __ballot(v);
        const int f_at = to + __popcll(fs & below), v_at = from + __popcll(vs & below);
        if (f && f_at < half) list[f_at] = i + lane;
        if (v && v_at < half) sources[v_at] = i + lane;
        to += __popcll(fs);
        from += __popcll(vs);
    }
    if (tid == 0) p.counts[grp] = count;
    __syncthreads();
    // The weights: first the moves, whose places lie in front of all sources, then the last r.
    for (int i = tid; i < count; i += kSelectThreads) p.weights[tb.listed(list[i], n)] = p.weights[tb.listed(sources[i], n)];
    __syncthreads();
    for (int i = 0; i < r; i += kSelectThreads) {
        const uint32_t w = i + tid < r ? p.weights[tb.row(old + i + tid)] : 0;
        __syncthreads();
        if (i + tid < r) p.weights[tb.row(k + i + tid)] = w;
    }
}

// A workgroup per (sequence, KV head), tensor and 128 bytes of a row; rows of other
// segments lie elsewhere, so that only its own loads and stores have to be in order.
constexpr int kMoveThreads = 256;
constexpr int kMoveAhead = 4;          // rows of a thread in flight

template <int D>
__global__ __launch_bounds__(kMoveThreads)
void kf_kv_evict_move_kernel(EvictParams p) {
    constexpr int kSegments = D / 64, kRows = kMoveThreads / 8;   // 8 lanes of 16 bytes a row
    const int tid = threadIdx.x, seg = blockIdx.x % (2 * kSegments), grp = blockIdx.x / (2 * kSegments);
    const int b = grp / p.heads, head = grp % p.heads;
    const int count = p.counts[grp], n = p.cuts[2 * grp], m = p.cuts[2 * grp + 1];
    if (head == 0 && seg == 0 && tid == 0) p.kept[b] = count < 0 ? n : m;
    if (count < 0) return;
    const EvictTable tb{p.block_table + (size_t)b * p.max_pages, p.heads, head, p.page_shift};
    uint8_t* const pool = p.pages[seg / kSegments] + seg % kSegments * 128 + tid % 8 * 16;
    const auto at = [&](size_t row) { return reinterpret_cast<u32x4*>(pool + row * (2 * D)); };
    const int r = min(p.recent, m), k = m - r, old = n - r;
    const int* const list = p.moves + (size_t)grp * p.capacity;
    const int* const sources = list + p.capacity / 2;
    for (int i0 = tid / 8; i0 < count; i0 += kRows * kMoveAhead) {
        u32x4 v[kMoveAhead];
#pragma unroll
        for (int u = 0; u < kMoveAhead; ++u) v[u] = *at(tb.listed(sources[min(i0 + u * kRows, count - 1)], n));
#pragma unroll
        for (int u = 0; u < kMoveAhead; ++u)
            if (i0 + u * kRows < count) *at(tb.listed(list[i0 + u * kRows], n)) = v[u];
    }
    // The last r keys, over places that the moves have read.
    __syncthreads();
    for (int i = 0; i < r; i += kRows * kMoveAhead) {
        u32x4 v[kMoveAhead];
#pragma unroll
        for (int u = 0; u < kMoveAhead; ++u) v[u] = *at(tb.row(old + min(i + u * kRows + tid / 8, r - 1)));
        // A place is written when it has been read; later rows are read behind all of these.
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveAhead; ++u)
            if (const int j = i + u * kRows + tid / 8; j < r) *at(tb.row(k + j)) = v[u];
    }
}

}  // namespace kf
