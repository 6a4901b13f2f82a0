// serve_capi.hip -- C ABI of what stands beside the attention forward in a
// server: packed prompts, head norms with rotary positions, the 4-bit cache
// and decode over it, the 16-bit cache with attention of new tokens over it, the
// weights that its keys gather and eviction by them.  Entry points are declared in include/kf/attn.h; as in
// attn_capi.hip, every argument check runs before the first HIP call.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "cache_kernels.h"
#include "capi_internal.h"
#include "kv4_kernels.h"
#include "packed_kernels.h"
#include "paged_kernels.h"
#include "rope_kernels.h"

namespace {

using namespace kf_capi;

bool aligned4(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 3u) == 0; }

constexpr int64_t kMaxKvTokenStride = 1 << 28;
// Rows and keys have int indexes, and the kernels round them up to whole tiles.
constexpr long long kMaxIndex = INT_MAX - 1024;

// Strides of 16-byte chunks, not negative; n of them.
int check_strides(const int64_t* s, int n) {
    for (int i = 0; i < n; ++i) {
        if (s[i] < 0) return KF_ERR_SIZE;
        if (s[i] % 8 != 0) return KF_ERR_ALIGN;
    }
    return KF_OK;
}

// Whether no two rows of D elements overlap, of which `tokens` lie `token` apart
// and in each `heads` lie `head` apart.
bool distinct_rows(int tokens, int64_t token, int heads, int64_t head, int D) {
    if (tokens == 1) return heads == 1 || head >= D;
    if (heads == 1) return token >= D;
    const int64_t inner = std::min(token, head), outer = std::max(token, head);
    const int n = token < head ? tokens : heads;  // rows `inner` apart
    return inner >= D && outer / inner >= n - 1 && outer - inner * (n - 1) >= D;
}

int check_heads(int H_q, int H_kv) {
    if (H_q <= 0 || H_kv <= 0 || H_q % H_kv != 0) return KF_ERR_GQA;
    return KF_OK;
}

// Sizes that the entry points with packed tokens share: a head dimension of
// whole 32-channel MFMA tiles, counts within the kernels' int indexing.
int check_packed(long long tokens, int heads, int D) {
    if (D != 64 && D != 128 && D != 256) return KF_ERR_HEAD_DIM;
    if (tokens <= 0 || heads <= 0) return KF_ERR_SIZE;
    if (tokens * heads > kMaxIndex) return KF_ERR_SIZE;
    return KF_OK;
}

// Whether a grid's threads have 32-bit numbers, as the hardware needs.
bool fits_grid(long long workgroups, int threads) { return workgroups * threads <= (long long)UINT_MAX; }

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KF_OK : hip_fail(e);
}

void set_scales(kf::AttnParams& prm, int D) {
    prm.scale = 1.0f / __builtin_sqrtf((float)D);
    prm.scale_log2 = (float)(1.0 / __builtin_sqrt((double)D) * 1.4426950408889634);
}

int out_dtype(int flags) {
    return (flags & KF_ATTN_OUT_F16) ? kf::kOutF16 : (flags & KF_ATTN_OUT_BF16) ? kf::kOutBF16 : kf::kOutF32;
}

int check_attn_flags(int flags) {
    constexpr int kKnown = KF_ATTN_CAUSAL | KF_ATTN_OUT_F16 | KF_ATTN_OUT_BF16 | KF_ATTN_LSE | KF_BF16;
    if ((flags & ~kKnown) != 0) return KF_ERR_FLAGS;
    if ((flags & KF_ATTN_OUT_F16) && (flags & KF_ATTN_OUT_BF16)) return KF_ERR_FLAGS;
    return KF_OK;
}

// ---- Packed attention. ----

template <bool kBF, int D, int NW, int KS>
int launch_packed(kf::PackedParams& prm, long long rows, hipStream_t stream) {
    using Cfg = kf::PackedCfg<D, NW, KS>;
    // Tiles of all sequences: a partial one for each at most.
    const long long tiles = rows / Cfg::kRows + std::min<long long>(prm.n_seqs, prm.tokens_q);
    if (!fits_grid(tiles * prm.heads_kv, Cfg::kThreads)) return KF_ERR_SIZE;
    // Strictly by length, the tiles that share keys run far apart, and their keys come
    // from beyond the L2 each time.  Many workgroups a CU even out by themselves, so
    // that coarser levels do: 64 x 256 queries, 32 / 8 heads, D = 128 (16 a CU), 97 us
    // in levels of one tile, 89 of two; 64 of 16 to 4096 (46 a CU) 747 and, of four to
    // eight, 735 to 729; 8 x 1024, 16 / 16 heads, D = 64 (4 a CU), 28.3 and, of four, 32.0.
    prm.level_tiles = (int)std::clamp<long long>(tiles * prm.heads_kv / (8LL * current_device_shape().cus), 1, 8);
    (void)hipGetLastError();
    kf::kf_attn_packed_kernel<kBF, D, NW, KS>
        <<<dim3((unsigned)(tiles * prm.heads_kv)), dim3(Cfg::kThreads), 0, stream>>>(prm);
    return launched();
}

// The layouts of the packed kernel: 128 rows on 4 waves, of which the CU holds
// several workgroups, is the cheapest for work enough; KV groups cut the
// longest chain of key tiles, which bounds a grid that leaves CUs idle.
// Cost in us of a call of equal sequences, by the averages that the host knows:
// the longest chain, start + chain per 32-key tile of a KV group, and the grid's
// work, each workgroup + tile over the device's CUs, joined by their 4-norm.
// Fitted to 158 shapes a head dimension (1 to 64 sequences of 32 to 8192
// queries against as many keys or eight times as many; rms 6 to 11 %, and the
// layout it picks is 1.1 % slower than the best of these at the geometric mean,
// 14 % at worst).  Always the first layout would be 16 % slower: 1 x 512 queries
// against 4096 keys, 32 / 8 heads, D = 128, take 96, 58 and 53 us in the three.
// The averages say little of a batch of very unequal lengths, whose longest chain is
// then underrated: 1 x 2048 queries beside 31 x 1, 8 / 8 heads, D = 128, take 50 us in
// the first layout, where the 2048 alone get KV groups and take 28.
struct PackedLayout {
    int rows, kv_groups;
    double start, chain, workgroup, tile;
};
constexpr PackedLayout kPacked64[3] = {{128, 1, 3.63, 0.504, 1.734, 0.321},
                                       {64, 2, 3.78, 0.570, 1.628, 0.362},
                                       {64, 4, 4.40, 0.784, 3.032, 0.731}};
constexpr PackedLayout kPacked128[3] = {{128, 1, 4.57, 0.739, 3.546, 0.535},
                                        {64, 2, 4.73, 0.803, 3.518, 0.652},
                                        {64, 4, 5.63, 1.235, 6.639, 1.397}};
constexpr PackedLayout kPacked256[2] = {{128, 1, 6.42, 1.309, 7.246, 1.011}, {128, 2, 9.87, 1.849, 12.804, 2.290}};

int packed_layout(const kf::PackedParams& prm, int D) {
    const PackedLayout* layouts = D == 64 ? kPacked64 : D == 128 ? kPacked128 : kPacked256;
    const double queries = std::max(1.0, (double)prm.tokens_q / prm.n_seqs);
    const double keys = (double)prm.tokens_k / prm.n_seqs;
    const double cus = current_device_shape().cus;
    int best = 0;
    double least = 0.0;
    for (int i = 0; i < (D == 256 ? 2 : 3); ++i) {
        const PackedLayout& l = layouts[i];
        const double tiles = std::ceil(queries * prm.ratio / l.rows);
        double seen = keys;  // by a row tile, on average
        if (prm.causal && tiles > 1.0) seen = std::min(keys, keys - (queries - 1.0) / 2 + l.rows / (2.0 * prm.ratio));
        const double key_tiles = std::max(seen, 0.0) / 32 + 0.5 + (l.kv_groups > 1 ? 0.5 * l.kv_groups : 0.0);
        const double chain = l.start + l.chain * std::ceil(std::ceil(keys / 32) / l.kv_groups);
        const double work = prm.n_seqs * (double)prm.heads_kv * tiles *
                            (l.workgroup + l.tile * key_tiles / l.kv_groups) / cus;
        const double cost = std::sqrt(std::sqrt(chain * chain * chain * chain + work * work * work * work));
        if (i == 0 || cost < least) {
            best = i;
            least = cost;
        }
    }
    return best;
}

template <bool kBF>
int launch_packed_dim(kf::PackedParams& prm, int D, hipStream_t stream) {
    const long long rows = (long long)prm.tokens_q * prm.ratio;
    const int layout = packed_layout(prm, D);
    switch (D) {
        case 64:
            return layout == 0   ? launch_packed<kBF, 64, 4, 1>(prm, rows, stream)
                   : layout == 1 ? launch_packed<kBF, 64, 4, 2>(prm, rows, stream)
                                 : launch_packed<kBF, 64, 8, 4>(prm, rows, stream);
        case 128:
            return layout == 0   ? launch_packed<kBF, 128, 4, 1>(prm, rows, stream)
                   : layout == 1 ? launch_packed<kBF, 128, 4, 2>(prm, rows, stream)
                                 : launch_packed<kBF, 128, 8, 4>(prm, rows, stream);
        default:
            return layout == 0 ? launch_packed<kBF, 256, 4, 1>(prm, rows, stream)
                               : launch_packed<kBF, 256, 8, 2>(prm, rows, stream);
    }
}

// ---- 4-bit decode. ----

struct Kv4Plan {
    int R, groups, wgs, merge_waves, cap, shift;
    size_t parts, o_bytes, s_bytes, ws_bytes;
};

int kv4_plan(int B, int q_len, int H_q, int H_kv, int D, int page_size, int max_pages, int num_pages, Kv4Plan* pl) {
    if (D != 64 && D != 128 && D != 256) return KF_ERR_HEAD_DIM;
    if (const int st = check_heads(H_q, H_kv); st != KF_OK) return st;
    if (B <= 0 || q_len <= 0) return KF_ERR_SIZE;
    if (const int st = paged_geometry(page_size, max_pages, num_pages, &pl->shift, &pl->cap); st != KF_OK) return st;
    const long long R = (long long)(H_q / H_kv) * q_len, groups = (long long)B * H_kv;
    if (R > 32 || pl->cap > kMaxIndex) return KF_ERR_SIZE;
    const long long stages = groups * ((pl->cap + 31LL) / 32);
    if (groups > INT_MAX || stages > (1LL << 30) || groups * R * (D / 4) > INT_MAX) return KF_ERR_SIZE;
    pl->R = (int)R;
    pl->groups = (int)groups;
    // No workgroup without a stage for each of its waves.
    pl->wgs = (int)std::min<long long>(kf::kv4_workgroups(D, (int)R, current_device_shape().cus),
                                       std::max<long long>(stages / kf::Kv4Cfg<64, 1>::kWaves, 1));
    pl->parts = (size_t)2 * pl->wgs * kf::Kv4Cfg<64, 1>::kWaves * (size_t)R;
    pl->o_bytes = align_up(pl->parts * D * sizeof(float), kWsAlign);
    pl->s_bytes = align_up(pl->parts * sizeof(float), kWsAlign);
    pl->ws_bytes = pl->o_bytes + 2 * pl->s_bytes + align_up((size_t)groups * sizeof(kf::u32x4), kWsAlign);
    pl->merge_waves = ragged_merge_waves(pl->R, pl->groups, D);
    // (A wave per head at least, in workgroups of kRaggedMergeWaves.)
    if (!fits_grid(groups * pl->merge_waves + kf::kRaggedMergeWaves - 1, 64)) return KF_ERR_SIZE;
    return KF_OK;
}

template <bool kBF, int D>
int launch_kv4(const Kv4Plan& pl, const kf::AttnParams& prm, hipStream_t stream) {
    (void)hipGetLastError();
    if (pl.R <= 16)
        kf::kf_attn_decode_kv4_kernel<kBF, D, 1><<<dim3(pl.wgs), dim3(kf::Kv4Cfg<D, 1>::kThreads), 0, stream>>>(prm);
    else
        kf::kf_attn_decode_kv4_kernel<kBF, D, 2><<<dim3(pl.wgs), dim3(kf::Kv4Cfg<D, 2>::kThreads), 0, stream>>>(prm);
    if (const int st = launched(); st != KF_OK) return st;
    const hipError_t e = merge_ragged(D, pl.groups, prm, stream);
    return e == hipSuccess ? KF_OK : hip_fail(e);
}

// ---- The 4-bit cache. ----

int check_kv4(int tokens, int n_seqs, int H_kv, int D, int page_size, int max_pages, int num_pages, int flags,
              const int* table, const int* starts, const int* lens, kf::Kv4Params* prm) {
    if (const int st = check_packed(tokens, H_kv, D); st != KF_OK) return st;
    if (n_seqs <= 0) return KF_ERR_SIZE;
    int cap;
    if (const int st = paged_geometry(page_size, max_pages, num_pages, &prm->page_shift, &cap); st != KF_OK) return st;
    if ((flags & ~KF_BF16) != 0) return KF_ERR_FLAGS;
    if (!table || !starts || !lens) return KF_ERR_NULL;
    if (!aligned4(table) || !aligned4(starts) || !aligned4(lens)) return KF_ERR_ALIGN;
    if ((long long)H_kv * (D / 8) * kf::kKv4MaxTile > INT_MAX) return KF_ERR_SIZE;
    prm->block_table = table;
    prm->starts = starts;
    prm->kv_lens = lens;
    prm->n_seqs = n_seqs;
    prm->tokens = tokens;
    prm->heads = H_kv;
    prm->max_pages = max_pages;
    prm->num_pages = num_pages;
    prm->page_bytes = kf_kv4_page_bytes(page_size, D);
    return KF_OK;
}

// Tokens of a workgroup: enough to give its threads an item each, and up to four
// while that leaves two workgroups a CU (16 x 1000 tokens, 8 heads, D = 128, 19.3 us
// written in 4 bits; eight items and four workgroups 21.6).
int cache_tile(const kf::Kv4Params& prm, int D) {
    const int per_token = prm.heads * (D / 8), fill = (kf::kKv4Threads + per_token - 1) / per_token;
    const long long share = prm.tokens / (2LL * current_device_shape().cus);
    return (int)std::min<long long>(std::max<long long>(fill, std::min<long long>(share, 4LL * fill)), kf::kKv4MaxTile);
}

template <bool kBF, int D>
int launch_cache(bool append, kf::Kv4Params& prm, hipStream_t stream) {
    prm.tile = cache_tile(prm, D);
    const dim3 grid((prm.tokens + prm.tile - 1) / prm.tile), block(kf::kKv4Threads);
    if (!fits_grid(grid.x, kf::kKv4Threads)) return KF_ERR_SIZE;
    (void)hipGetLastError();
    if (append)
        kf::kf_kv4_append_kernel<kBF, D><<<grid, block, 0, stream>>>(prm);
    else
        kf::kf_kv4_read_kernel<kBF, D><<<grid, block, 0, stream>>>(prm);
    return launched();
}

template <bool kBF>
int launch_cache_dim(bool append, kf::Kv4Params& prm, int D, hipStream_t stream) {
    switch (D) {
        case 64: return launch_cache<kBF, 64>(append, prm, stream);
        case 128: return launch_cache<kBF, 128>(append, prm, stream);
        default: return launch_cache<kBF, 256>(append, prm, stream);
    }
}

// ---- Norm and rotary positions. ----

template <bool kBF, int D>
int launch_rope(const kf::RopeParams& prm, hipStream_t stream) {
    (void)hipGetLastError();
    const dim3 block(64 * kf::kRopeWaves);
    // A wave per token while that gives every CU ten, else a workgroup: 512 tokens of 32 + 8 heads,
    // D = 128, 6.3 us by workgroups and 9.5 by waves, 2048 12.9 and 13.8, 3000
    // 16.7 and 16.1, 6000 30.9 and 27.0; of 32 + 1 heads of 64, 2048 8.9 and 8.9, 8192 24.6 and 19.0.
    if (prm.tokens >= 10 * current_device_shape().cus) {
        const int grid = (prm.tokens + 3) / 4;
        if (!fits_grid(grid, 64 * kf::kRopeWaves)) return KF_ERR_SIZE;
        kf::kf_qk_norm_rope_kernel<kBF, D, 4><<<dim3(grid), block, 0, stream>>>(prm);
    } else {
        kf::kf_qk_norm_rope_kernel<kBF, D, 1><<<dim3(prm.tokens), block, 0, stream>>>(prm);
    }
    return launched();
}

template <bool kBF>
int launch_rope_dim(const kf::RopeParams& prm, int D, hipStream_t stream) {
    switch (D) {
        case 16: return launch_rope<kBF, 16>(prm, stream);
        case 64: return launch_rope<kBF, 64>(prm, stream);
        case 128: return launch_rope<kBF, 128>(prm, stream);
        default: return launch_rope<kBF, 256>(prm, stream);
    }
}

// ---- Attention over the paged 16-bit cache. ----

struct PagedPlan {
    int rows, slots;                      // rows of a tile (PagedCfg)
    long long items, cut_tiles;           // at most, of a KV head
    size_t o_bytes, s_bytes, ws_bytes;
    kf::PagedParams prm;
};

int check_paged(int n_seqs, int tokens, int H_q, int H_kv, int D, int page_size, int max_pages, int num_pages,
                kf::PagedParams* prm) {
    if (D != 64 && D != 128 && D != 256) return KF_ERR_HEAD_DIM;
    if (const int st = check_heads(H_q, H_kv); st != KF_OK) return st;
    if (n_seqs <= 0) return KF_ERR_SIZE;
    if (const int st = check_packed(tokens, H_q, D); st != KF_OK) return st;
    if (const int st = paged_geometry(page_size, max_pages, num_pages, &prm->page_shift, &prm->kv_len); st != KF_OK)
        return st;
    return prm->kv_len > kMaxIndex ? KF_ERR_SIZE : KF_OK;
}

void paged_sizes(int D, int H_kv, PagedPlan* pl) {
    const size_t parts = (size_t)pl->slots * H_kv * pl->rows;
    pl->o_bytes = align_up(parts * D * sizeof(float), kWsAlign);
    pl->s_bytes = align_up(parts * sizeof(float), kWsAlign);
    pl->ws_bytes = pl->o_bytes + 2 * pl->s_bytes;
}

int paged_plan(int n_seqs, int tokens, int H_q, int H_kv, int D, int page_size, int max_pages, int num_pages,
               PagedPlan* pl) {
    kf::PagedParams& prm = pl->prm;
    if (const int st = check_paged(n_seqs, tokens, H_q, H_kv, D, page_size, max_pages, num_pages, &prm); st != KF_OK)
        return st;
    const long long rows = (long long)tokens * (H_q / H_kv);
    // By the rows that a sequence has on average.  us with 32, 64 and 128 rows, 32 / 8 heads of 128:
    //   32 x 4 tokens over 2048 keys 52, 53, 53  x 12 92, 59, 61  x 24 134, 64, 70  x 64 338, 117, 102
    //   4 x 4 over 8192 36, 36, 36               x 12 50, 45, 46  x 24  69, 42, 48  x 64 129,  64,  65
    //   32 x 1 over 512 to 8192 69, 73, 67       x 1 to 4 71, 76, 71;  8 x 1 over 512 to 32768 54, 62, 54
    // and with 32 and 128 rows, 16 / 4 heads of 256,
    //   32 x 4 over 2048 70, 60                  x 12 102, 69;  4 x 4 over 8192 53, 59  x 12 76, 86
    //   32 x 1 over 512 to 8192 74, 88           x 1 to 16 94, 105  x 1 to 64 136, 115
    // At D = 64, 64 rows would be the best up to 96, too (32 x 2 over 2048 33, 29, 34, x 24 67, 40, 42;
    // 32 x 1 over 512 to 8192 36, 35, 40).  Averages say little of steps beside a prompt or of empty
    // sequences: 1 x 4096 alone takes 169 us, among 999 empty ones, in tiles of 32, 996.
    const double avg = (double)rows / n_seqs;
    pl->rows = D == 256 ? (avg > 32 ? 128 : 32) : avg > 64 ? 128 : avg > 32 ? 64 : 32;
    if (pl->rows == 32) {
        // Equal shares of a line, for every workgroup that the device holds; no fewer than 8
        // units each (one step over 4096 keys, 32 / 8 heads of 128, 17.6, 16.4 and 18.7 us by 4, 8 and
        // 16; 40 of 1 to 4 tokens over 16 to 300 20, 20 and 23).
        prm.target = std::max(1, current_device_shape().cus * (D == 64 ? 2 : 1) / H_kv);
        prm.min_share = 8;
        // Few keys: no second launch (by the table's places: the host knows no lengths).  us without and
        // with one: 1 step over 256 keys 10.6, 13.3, over 512 14.1, 13.4, over 1024 21.5, 14.0; 32 steps
        // 12.6, 14.5, 18.3, 20.3, and over 2048 48, 50.
        prm.cut = prm.target > 1 && prm.kv_len > 256 ? 1 : 0;
        pl->items = prm.target;
        pl->cut_tiles = prm.cut ? prm.target - 1 : 0;
        pl->slots = prm.cut ? 2 * prm.target : 0;
        paged_sizes(D, H_kv, pl);
        return fits_grid(pl->items * H_kv, 256) ? KF_OK : KF_ERR_SIZE;
    }
    const long long least = (rows + pl->rows - 1) / pl->rows;
    const long long tiles = rows / pl->rows + std::min<long long>(n_seqs, tokens);
    const long long stages = ((long long)prm.kv_len + 31) / 32;
    // No cuts where tiles fill the device twice, or of few keys (us without and with cuts, 64 tokens: 1 x over
    // 256 keys 14.0, 15.8, over 512 21.0, 20.0, over 1024 35, 21; 16 x 16.3, 18.4, 23.9, 32.0, 38, 42, and
    // over 2048 66, 63).
    const int wanted = std::max(1, 2 * current_device_shape().cus / H_kv);
    prm.target = least >= 2 * wanted || stages <= 8 ? 0 : wanted;
    prm.unit_shift = 0;
    while (tiles * ((stages >> prm.unit_shift) + 1) > INT_MAX) ++prm.unit_shift;
    // (1 x 64 tokens over 2048 keys 33, 26 and 28 us by 4, 8 and 16, 4 x 64 over 512 25, 21, 23.)
    prm.min_share = std::max(1, 8 >> prm.unit_shift);
    pl->items = tiles + prm.target;
    pl->cut_tiles = std::min<long long>(tiles, prm.target);
    pl->slots = 2 * prm.target;
    paged_sizes(D, H_kv, pl);
    if (!fits_grid(pl->items * H_kv, 256)) return KF_ERR_SIZE;
    return KF_OK;
}

template <bool kBF, int D, int NW, int KS>
int launch_paged(const PagedPlan& pl, hipStream_t stream) {
    using Cfg = kf::PagedCfg<D, NW, KS>;
    const kf::PagedParams& prm = pl.prm;
    (void)hipGetLastError();
    kf::kf_attn_paged_kernel<kBF, D, NW, KS>
        <<<dim3((unsigned)(pl.items * prm.heads_kv)), dim3(Cfg::kThreads), 0, stream>>>(prm);
    if (const int st = launched(); st != KF_OK || pl.cut_tiles == 0) return st;
    kf::kf_attn_paged_merge_kernel<D, Cfg::kRows>
        <<<dim3((unsigned)(pl.cut_tiles * prm.heads_kv), Cfg::kRows / 32), dim3(kf::kPagedMergeThreads), 0, stream>>>(prm);
    return launched();
}

template <bool kBF>
int launch_paged_dim(const PagedPlan& pl, int D, hipStream_t stream) {
    switch (D) {
        case 64:
            return pl.rows == 128  ? launch_paged<kBF, 64, 4, 1>(pl, stream)
                   : pl.rows == 64 ? launch_paged<kBF, 64, 4, 2>(pl, stream)
                                   : launch_paged<kBF, 64, 4, 4>(pl, stream);
        case 128:
            return pl.rows == 128  ? launch_paged<kBF, 128, 4, 1>(pl, stream)
                   : pl.rows == 64 ? launch_paged<kBF, 128, 4, 2>(pl, stream)
                                   : launch_paged<kBF, 128, 4, 4>(pl, stream);
        default: return pl.rows == 128 ? launch_paged<kBF, 256, 4, 1>(pl, stream) : launch_paged<kBF, 256, 2, 2>(pl, stream);
    }
}

// What the paged attention and the gathered weights have in common, the sizes apart.
void set_paged(kf::PagedParams& prm, const void* Q, const int64_t* strides, const void* K_pages, const int* block_table,
               const int* seq_starts, const int* kv_lens, int n_seqs, int tokens, int H_q, int H_kv, int D,
               int max_pages, int num_pages, int flags) {
    prm.Q = static_cast<const uint16_t*>(Q);
    prm.K = static_cast<const uint16_t*>(K_pages);
    prm.q_token = strides ? strides[0] : (int64_t)H_q * D;
    prm.q_head = strides ? strides[1] : D;
    prm.q_starts = seq_starts;
    prm.kv_lens = kv_lens;
    prm.block_table = block_table;
    prm.max_pages = max_pages;
    prm.num_pages = num_pages;
    prm.n_seqs = n_seqs;
    prm.tokens_q = tokens;
    prm.heads_kv = H_kv;
    prm.ratio = H_q / H_kv;
    prm.causal = (flags & KF_ATTN_CAUSAL) ? 1 : 0;
    prm.n_splits = 1;
    set_scales(prm, D);
}

// ---- Gathered weights. ----

struct WeighPlan {
    size_t ws_bytes;
    kf::PagedParams prm;
};

int weigh_plan(int n_seqs, int tokens, int H_q, int H_kv, int D, int page_size, int max_pages, int num_pages,
               WeighPlan* pl) {
    kf::PagedParams& prm = pl->prm;
    if (const int st = check_paged(n_seqs, tokens, H_q, H_kv, D, page_size, max_pages, num_pages, &prm); st != KF_OK)
        return st;
    const int keys = D == 256 ? kf::WeighCfg<256>::kKeys : kf::WeighCfg<128>::kKeys;
    const long long rows = (long long)tokens * (H_q / H_kv);
    // A share for every workgroup that the device holds, of 4 units at least (us by 2, 4 and 8: 1 x 64
    // tokens over 8192 keys 29.4, 26.5, 28.9, over 512 16.4, 20.3, 26.9; 32 steps over 512 12.2, 12.1, 14.8).
    prm.target = std::max(1, 2 * current_device_shape().cus / H_kv);
    prm.min_share = 4;
    // Blocks are cut where sequences have, on average, more than a stage of rows; a
    // batch of steps is spared the second launch.  us without and with cuts, 32 / 8 heads of 128: 1 x 32
    // tokens over 2048 keys 19, 22 |  x 64 17, 21 |  x 128 25, 21 |  x 512 79, 35; 4 x 64 over 8192 45, 48 |
    // x 128 67, 67 |  x 512 209, 198.  (1 x 1000 alone 32 us; among 63 empty sequences, by the average not
    // cut, 96.)
    prm.cut = rows / n_seqs > kf::kWeighRows ? 1 : 0;
    pl->ws_bytes = prm.cut ? align_up((size_t)2 * prm.target * H_kv * keys * sizeof(float), kWsAlign) : 0;
    return fits_grid((long long)prm.target * H_kv, 4 * keys) ? KF_OK : KF_ERR_SIZE;
}

template <bool kBF, int D>
int launch_weigh(const WeighPlan& pl, hipStream_t stream) {
    using Cfg = kf::WeighCfg<D>;
    const kf::PagedParams& prm = pl.prm;
    (void)hipGetLastError();
    kf::kf_kv_weigh_kernel<kBF, D>
        <<<dim3((unsigned)(prm.target * prm.heads_kv)), dim3(Cfg::kThreads), 0, stream>>>(prm);
    if (const int st = launched(); st != KF_OK || !prm.cut || prm.target == 1) return st;
    kf::kf_kv_weigh_merge_kernel<D>
        <<<dim3((unsigned)((prm.target - 1) * prm.heads_kv)), dim3(4 * Cfg::kKeys), 0, stream>>>(prm);
    return launched();
}

template <bool kBF>
int launch_weigh_dim(const WeighPlan& pl, int D, hipStream_t stream) {
    switch (D) {
        case 64: return launch_weigh<kBF, 64>(pl, stream);
        case 128: return launch_weigh<kBF, 128>(pl, stream);
        default: return launch_weigh<kBF, 256>(pl, stream);
    }
}

// ---- The 16-bit cache: new tokens, eviction. ----

template <int D>
int launch_append(kf::KvAppendParams& prm, hipStream_t stream) {
    prm.tile = cache_tile(prm, D);
    const dim3 grid((prm.tokens + prm.tile - 1) / prm.tile), block(kf::kKv4Threads);
    if (!fits_grid(grid.x, kf::kKv4Threads)) return KF_ERR_SIZE;
    (void)hipGetLastError();
    kf::kf_kv_append_kernel<D><<<grid, block, 0, stream>>>(prm);
    return launched();
}

struct EvictPlan {
    int shift, capacity, parts;
    size_t cuts_bytes, ws_bytes;
};

int evict_plan(int n_seqs, int H_kv, int D, int page_size, int max_pages, int num_pages, EvictPlan* pl) {
    if (D != 64 && D != 128 && D != 256) return KF_ERR_HEAD_DIM;
    if (n_seqs <= 0 || H_kv <= 0) return KF_ERR_SIZE;
    if (const int st = paged_geometry(page_size, max_pages, num_pages, &pl->shift, &pl->capacity); st != KF_OK) return st;
    const long long groups = (long long)n_seqs * H_kv;
    // Up to 32 workgroups a CU that move keys, each with a few rounds at least (16 contexts of 4096 to
    // 32768 keys to half 145, 138 and 137 us by 16, 32 and 64; one key of 32 contexts in tables of 65536
    // places 28.5, 28.9, 32.8).
    const long long rounds = pl->capacity / 2 / (kf::kMoveThreads * 8 / D * kf::kMoveAhead);
    pl->parts = (int)std::max<long long>(1, std::min(32LL * current_device_shape().cus / groups, rounds / 4));
    if (pl->capacity > kMaxIndex || !fits_grid(groups, kf::kSelectThreads) ||
        !fits_grid(groups * (D / 32 + pl->parts), kf::kMoveThreads))
        return KF_ERR_SIZE;
    pl->cuts_bytes = align_up((size_t)groups * 4 * sizeof(int), kWsAlign);
    pl->ws_bytes = pl->cuts_bytes + align_up((size_t)groups * pl->capacity * sizeof(int), kWsAlign);
    return KF_OK;
}

template <int D>
int launch_evict(const kf::EvictParams& prm, hipStream_t stream) {
    const int groups = prm.n_seqs * prm.heads;
    const dim3 grid(groups), block(kf::kSelectThreads);
    (void)hipGetLastError();
    kf::kf_kv_evict_select_kernel<<<grid, block, 0, stream>>>(prm);
    if (const int st = launched(); st != KF_OK) return st;
    kf::kf_kv_evict_move_kernel<D><<<dim3(groups * (D / 32 + prm.parts)), dim3(kf::kMoveThreads), 0, stream>>>(prm);
    return launched();
}

}  // namespace

extern "C" {

int kf_attn_packed(const void* Q, const void* K, const void* V, void* O, float* row_max, float* row_sumexp,
                   const int64_t* strides, const int* q_starts, const int* kv_starts, int n_seqs, int tokens_q,
                   int tokens_kv, int H_q, int H_kv, int D, int flags, void* stream) {
    if (D != 64 && D != 128 && D != 256) return KF_ERR_HEAD_DIM;
    if (const int st = check_heads(H_q, H_kv); st != KF_OK) return st;
    if (n_seqs <= 0) return KF_ERR_SIZE;
    if (const int st = check_packed(tokens_q, H_q, D); st != KF_OK) return st;
    if (const int st = check_packed(tokens_kv, H_kv, D); st != KF_OK) return st;
    if ((long long)tokens_kv * (H_q / H_kv) > kMaxIndex) return KF_ERR_SIZE;
    if (const int st = check_attn_flags(flags); st != KF_OK) return st;
    if (!Q || !K || !V || !O || !q_starts || !kv_starts) return KF_ERR_NULL;
    if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || !aligned16(O)) return KF_ERR_ALIGN;
    if (!aligned4(q_starts) || !aligned4(kv_starts)) return KF_ERR_ALIGN;
    const int64_t packed[6] = {(int64_t)H_q * D, D, (int64_t)H_kv * D, D, (int64_t)H_kv * D, D};
    if (!strides) strides = packed;
    if (const int st = check_strides(strides, 6); st != KF_OK) return st;
    // (A lane's offset within an LDS-DMA instruction, up to 7 rows, has 32 bits.)
    if (strides[2] > kMaxKvTokenStride || strides[4] > kMaxKvTokenStride) return KF_ERR_SIZE;
    kf::PackedParams prm{};
    prm.Q = static_cast<const uint16_t*>(Q);
    prm.K = static_cast<const uint16_t*>(K);
    prm.V = static_cast<const uint16_t*>(V);
    prm.O = static_cast<float*>(O);
    prm.Mi = row_max;
    prm.Li = row_sumexp;
    prm.lse = (flags & KF_ATTN_LSE) ? 1 : 0;
    prm.out_dtype = out_dtype(flags);
    prm.causal = (flags & KF_ATTN_CAUSAL) ? 1 : 0;
    prm.heads_kv = H_kv;
    prm.n_splits = 1;
    set_scales(prm, D);
    prm.q_token = strides[0];
    prm.q_head = strides[1];
    prm.k_token = strides[2];
    prm.k_head = strides[3];
    prm.v_token = strides[4];
    prm.v_head = strides[5];
    prm.q_starts = q_starts;
    prm.k_starts = kv_starts;
    prm.n_seqs = n_seqs;
    prm.tokens_q = tokens_q;
    prm.tokens_k = tokens_kv;
    prm.ratio = H_q / H_kv;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return (flags & KF_BF16) ? launch_packed_dim<true>(prm, D, s) : launch_packed_dim<false>(prm, D, s);
}

int kf_qk_norm_rope(const void* Q, const void* K, void* Q_out, void* K_out, const int64_t* strides,
                    const void* q_weight, const void* k_weight, const int* positions, const double* freqs, int tokens,
                    int H_q, int H_kv, int D, int rot, float eps, float scale, int flags, void* stream) {
    if (D != 16 && D != 64 && D != 128 && D != 256) return KF_ERR_HEAD_DIM;
    if (tokens <= 0 || tokens > kMaxIndex || H_q <= 0 || H_kv <= 0 || rot < 0 || rot > D || rot % 16 != 0) return KF_ERR_SIZE;
    if ((long long)H_q + H_kv > INT_MAX / 2) return KF_ERR_SIZE;
    if ((flags & ~(KF_BF16 | KF_ROPE_INTERLEAVED)) != 0) return KF_ERR_FLAGS;
    if (!Q || !K || !Q_out || !K_out || (rot > 0 && (!positions || !freqs))) return KF_ERR_NULL;
    if (!aligned16(Q) || !aligned16(K) || !aligned16(Q_out) || !aligned16(K_out) || !aligned16(q_weight) ||
        !aligned16(k_weight) || !aligned4(positions) || (reinterpret_cast<uintptr_t>(freqs) & 7u) != 0)
        return KF_ERR_ALIGN;
    const int64_t packed[8] = {(int64_t)H_q * D, D, (int64_t)H_kv * D, D, (int64_t)H_q * D, D, (int64_t)H_kv * D, D};
    if (!strides) strides = packed;
    if (const int st = check_strides(strides, 8); st != KF_OK) return st;
    if (!distinct_rows(tokens, strides[4], H_q, strides[5], D) || !distinct_rows(tokens, strides[6], H_kv, strides[7], D))
        return KF_ERR_SIZE;
    kf::RopeParams prm{};
    prm.x[0] = static_cast<const uint16_t*>(Q);
    prm.x[1] = static_cast<const uint16_t*>(K);
    prm.y[0] = static_cast<uint16_t*>(Q_out);
    prm.y[1] = static_cast<uint16_t*>(K_out);
    prm.w[0] = static_cast<const uint16_t*>(q_weight);
    prm.w[1] = static_cast<const uint16_t*>(k_weight);
    for (int i = 0; i < 2; ++i) {
        prm.token[i] = strides[2 * i];
        prm.head[i] = strides[2 * i + 1];
        prm.y_token[i] = strides[4 + 2 * i];
        prm.y_head[i] = strides[5 + 2 * i];
    }
    prm.heads_q = H_q;
    prm.heads = H_q + H_kv;
    prm.tokens = tokens;
    prm.positions = positions;
    prm.freqs = freqs;
    prm.rot = rot;
    prm.interleaved = (flags & KF_ROPE_INTERLEAVED) ? 1 : 0;
    prm.eps = eps;
    prm.scale = scale;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return (flags & KF_BF16) ? launch_rope_dim<true>(prm, D, s) : launch_rope_dim<false>(prm, D, s);
}

size_t kf_kv4_page_bytes(int page_size, int D) {
    int sh, cap;
    if ((D != 64 && D != 128 && D != 256) || paged_geometry(page_size, 1, 1, &sh, &cap) != KF_OK) return 0;
    return (size_t)page_size * (17 * D / 32);
}

int kf_kv4_append(const void* K, const void* V, const int64_t* strides, void* K_pages, void* V_pages,
                  const int* block_table, const int* seq_starts, const int* kv_lens, int n_seqs, int tokens, int H_kv,
                  int D, int page_size, int max_pages_per_seq, int num_pages, int flags, void* stream) {
    kf::Kv4Params prm{};
    if (const int st = check_kv4(tokens, n_seqs, H_kv, D, page_size, max_pages_per_seq, num_pages, flags, block_table,
                                 seq_starts, kv_lens, &prm);
        st != KF_OK)
        return st;
    if (!K || !V || !K_pages || !V_pages) return KF_ERR_NULL;
    if (!aligned16(K) || !aligned16(V) || !aligned16(K_pages) || !aligned16(V_pages)) return KF_ERR_ALIGN;
    const int64_t packed[4] = {(int64_t)H_kv * D, D, (int64_t)H_kv * D, D};
    if (!strides) strides = packed;
    if (const int st = check_strides(strides, 4); st != KF_OK) return st;
    prm.x[0] = static_cast<const uint16_t*>(K);
    prm.x[1] = static_cast<const uint16_t*>(V);
    prm.pages[0] = static_cast<uint8_t*>(K_pages);
    prm.pages[1] = static_cast<uint8_t*>(V_pages);
    for (int i = 0; i < 2; ++i) {
        prm.token[i] = strides[2 * i];
        prm.head[i] = strides[2 * i + 1];
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    return (flags & KF_BF16) ? launch_cache_dim<true>(true, prm, D, s) : launch_cache_dim<false>(true, prm, D, s);
}

int kf_kv4_read(const void* K_pages, const void* V_pages, const int* block_table, const int* seq_starts,
                const int* kv_lens, void* K, void* V, int n_seqs, int tokens, int H_kv, int D, int page_size,
                int max_pages_per_seq, int num_pages, int flags, void* stream) {
    kf::Kv4Params prm{};
    if (const int st = check_kv4(tokens, n_seqs, H_kv, D, page_size, max_pages_per_seq, num_pages, flags, block_table,
                                 seq_starts, kv_lens, &prm);
        st != KF_OK)
        return st;
    if (!K || !V || !K_pages || !V_pages) return KF_ERR_NULL;
    if (!aligned16(K) || !aligned16(V) || !aligned16(K_pages) || !aligned16(V_pages)) return KF_ERR_ALIGN;
    prm.y[0] = static_cast<uint16_t*>(K);
    prm.y[1] = static_cast<uint16_t*>(V);
    prm.pages[0] = static_cast<uint8_t*>(const_cast<void*>(K_pages));
    prm.pages[1] = static_cast<uint8_t*>(const_cast<void*>(V_pages));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return (flags & KF_BF16) ? launch_cache_dim<true>(false, prm, D, s) : launch_cache_dim<false>(false, prm, D, s);
}

size_t kf_attn_decode_kv4_workspace_bytes(int B, int q_len, int H_q, int H_kv, int D, int page_size,
                                          int max_pages_per_seq) {
    Kv4Plan pl;
    if (kv4_plan(B, q_len, H_q, H_kv, D, page_size, max_pages_per_seq, 1, &pl) != KF_OK) return 0;
    return pl.ws_bytes;
}

int kf_attn_decode_kv4(const void* Q, const void* K_pages, const void* V_pages, const int* block_table,
                       const int* kv_lens, void* O, float* row_max, float* row_sumexp, int B, int q_len, int H_q,
                       int H_kv, int D, int page_size, int max_pages_per_seq, int num_pages, int flags,
                       void* workspace, size_t workspace_bytes, void* stream) {
    Kv4Plan pl;
    if (const int st = kv4_plan(B, q_len, H_q, H_kv, D, page_size, max_pages_per_seq, num_pages, &pl); st != KF_OK)
        return st;
    if (const int st = check_attn_flags(flags); st != KF_OK) return st;
    if (!Q || !K_pages || !V_pages || !O || !block_table || !kv_lens) return KF_ERR_NULL;
    if (!aligned16(Q) || !aligned16(K_pages) || !aligned16(V_pages) || !aligned16(O)) return KF_ERR_ALIGN;
    if (!aligned4(block_table) || !aligned4(kv_lens)) return KF_ERR_ALIGN;
    if (!workspace || workspace_bytes < pl.ws_bytes) return KF_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & (kWsAlign - 1)) != 0) return KF_ERR_ALIGN;
    kf::AttnParams prm{};
    prm.Q = static_cast<const uint16_t*>(Q);
    prm.K = static_cast<const uint16_t*>(K_pages);
    prm.V = static_cast<const uint16_t*>(V_pages);
    prm.O = static_cast<float*>(O);
    prm.Mi = row_max;
    prm.Li = row_sumexp;
    char* ws = static_cast<char*>(workspace);
    prm.Opart = reinterpret_cast<float*>(ws);
    prm.Mpart = reinterpret_cast<float*>(ws + pl.o_bytes);
    prm.Lpart = reinterpret_cast<float*>(ws + pl.o_bytes + pl.s_bytes);
    prm.ragged_heads = reinterpret_cast<kf::u32x4*>(ws + pl.o_bytes + 2 * pl.s_bytes);
    prm.rows_per_group = pl.R;
    prm.kv_len = pl.cap;
    prm.rows_total = pl.groups * pl.R;
    set_scales(prm, D);
    prm.kv_lens = kv_lens;
    prm.causal = (flags & KF_ATTN_CAUSAL) ? 1 : 0;
    prm.q_len = q_len;
    prm.heads_kv = H_kv;
    prm.block_table = block_table;
    prm.max_pages = max_pages_per_seq;
    prm.page_shift = pl.shift;
    prm.num_pages = num_pages;
    prm.out_dtype = out_dtype(flags);
    prm.lse = (flags & KF_ATTN_LSE) ? 1 : 0;
    prm.batch = B;
    prm.merge_waves = pl.merge_waves;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (flags & KF_BF16) {
        switch (D) {
            case 64: return launch_kv4<true, 64>(pl, prm, s);
            case 128: return launch_kv4<true, 128>(pl, prm, s);
            default: return launch_kv4<true, 256>(pl, prm, s);
        }
    }
    switch (D) {
        case 64: return launch_kv4<false, 64>(pl, prm, s);
        case 128: return launch_kv4<false, 128>(pl, prm, s);
        default: return launch_kv4<false, 256>(pl, prm, s);
    }
}

int kf_kv_append(const void* K, const void* V, const int64_t* strides, void* K_pages, void* V_pages, float* weights,
                 const int* block_table, const int* seq_starts, const int* kv_lens, int n_seqs, int tokens, int H_kv,
                 int D, int page_size, int max_pages_per_seq, int num_pages, int flags, void* stream) {
    kf::KvAppendParams prm{};
    if (const int st = check_kv4(tokens, n_seqs, H_kv, D, page_size, max_pages_per_seq, num_pages, flags, block_table,
                                 seq_starts, kv_lens, &prm);
        st != KF_OK)
        return st;
    if (!K || !V || !K_pages || !V_pages) return KF_ERR_NULL;
    if (!aligned16(K) || !aligned16(V) || !aligned16(K_pages) || !aligned16(V_pages) || !aligned4(weights))
        return KF_ERR_ALIGN;
    const int64_t packed[4] = {(int64_t)H_kv * D, D, (int64_t)H_kv * D, D};
    if (!strides) strides = packed;
    if (const int st = check_strides(strides, 4); st != KF_OK) return st;
    prm.x[0] = static_cast<const uint16_t*>(K);
    prm.x[1] = static_cast<const uint16_t*>(V);
    prm.pages[0] = static_cast<uint8_t*>(K_pages);
    prm.pages[1] = static_cast<uint8_t*>(V_pages);
    for (int i = 0; i < 2; ++i) {
        prm.token[i] = strides[2 * i];
        prm.head[i] = strides[2 * i + 1];
    }
    prm.page_bytes = (size_t)page_size * D * 2;
    prm.weights = weights;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: return launch_append<64>(prm, s);
        case 128: return launch_append<128>(prm, s);
        default: return launch_append<256>(prm, s);
    }
}

size_t kf_attn_paged_workspace_bytes(int n_seqs, int tokens, int H_q, int H_kv, int D, int page_size,
                                     int max_pages_per_seq) {
    PagedPlan pl{};
    return paged_plan(n_seqs, tokens, H_q, H_kv, D, page_size, max_pages_per_seq, 1, &pl) == KF_OK ? pl.ws_bytes : 0;
}

int kf_attn_paged(const void* Q, const int64_t* strides, const void* K_pages, const void* V_pages,
                  const int* block_table, const int* seq_starts, const int* kv_lens, void* O, float* row_max,
                  float* row_sumexp, int n_seqs, int tokens, int H_q, int H_kv, int D, int page_size,
                  int max_pages_per_seq, int num_pages, int flags, void* workspace, size_t workspace_bytes,
                  void* stream) {
    PagedPlan pl{};
    if (const int st = paged_plan(n_seqs, tokens, H_q, H_kv, D, page_size, max_pages_per_seq, num_pages, &pl);
        st != KF_OK)
        return st;
    if (const int st = check_attn_flags(flags); st != KF_OK) return st;
    if (!Q || !K_pages || !V_pages || !O || !block_table || !seq_starts || !kv_lens) return KF_ERR_NULL;
    if (!aligned16(Q) || !aligned16(K_pages) || !aligned16(V_pages) || !aligned16(O)) return KF_ERR_ALIGN;
    if (!aligned4(block_table) || !aligned4(seq_starts) || !aligned4(kv_lens)) return KF_ERR_ALIGN;
    if (strides)
        if (const int st = check_strides(strides, 2); st != KF_OK) return st;
    if (pl.ws_bytes > 0) {
        if (!workspace || workspace_bytes < pl.ws_bytes) return KF_ERR_WORKSPACE;
        if ((reinterpret_cast<uintptr_t>(workspace) & (kWsAlign - 1)) != 0) return KF_ERR_ALIGN;
    }
    kf::PagedParams& prm = pl.prm;
    set_paged(prm, Q, strides, K_pages, block_table, seq_starts, kv_lens, n_seqs, tokens, H_q, H_kv, D,
              max_pages_per_seq, num_pages, flags);
    prm.V = static_cast<const uint16_t*>(V_pages);
    prm.O = static_cast<float*>(O);
    prm.Mi = row_max;
    prm.Li = row_sumexp;
    prm.lse = (flags & KF_ATTN_LSE) ? 1 : 0;
    prm.out_dtype = out_dtype(flags);
    char* ws = static_cast<char*>(workspace);
    prm.Opart = reinterpret_cast<float*>(ws);
    prm.Mpart = reinterpret_cast<float*>(ws + pl.o_bytes);
    prm.Lpart = reinterpret_cast<float*>(ws + pl.o_bytes + pl.s_bytes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return (flags & KF_BF16) ? launch_paged_dim<true>(pl, D, s) : launch_paged_dim<false>(pl, D, s);
}

size_t kf_kv_weigh_workspace_bytes(int n_seqs, int tokens, int H_q, int H_kv, int D, int page_size,
                                   int max_pages_per_seq) {
    WeighPlan pl{};
    return weigh_plan(n_seqs, tokens, H_q, H_kv, D, page_size, max_pages_per_seq, 1, &pl) == KF_OK ? pl.ws_bytes : 0;
}

int kf_kv_weigh(const void* Q, const int64_t* strides, const void* K_pages, float* weights, const int* block_table,
                const int* seq_starts, const int* kv_lens, const float* lse, int n_seqs, int tokens, int H_q, int H_kv,
                int D, int page_size, int max_pages_per_seq, int num_pages, int flags, void* workspace,
                size_t workspace_bytes, void* stream) {
    WeighPlan pl{};
    if (const int st = weigh_plan(n_seqs, tokens, H_q, H_kv, D, page_size, max_pages_per_seq, num_pages, &pl);
        st != KF_OK)
        return st;
    if ((flags & ~(KF_ATTN_CAUSAL | KF_BF16)) != 0) return KF_ERR_FLAGS;
    if (!Q || !K_pages || !weights || !block_table || !seq_starts || !kv_lens || !lse) return KF_ERR_NULL;
    if (!aligned16(Q) || !aligned16(K_pages)) return KF_ERR_ALIGN;
    if (!aligned4(weights) || !aligned4(block_table) || !aligned4(seq_starts) || !aligned4(kv_lens) || !aligned4(lse))
        return KF_ERR_ALIGN;
    if (strides)
        if (const int st = check_strides(strides, 2); st != KF_OK) return st;
    if (pl.ws_bytes > 0) {
        if (!workspace || workspace_bytes < pl.ws_bytes) return KF_ERR_WORKSPACE;
        if ((reinterpret_cast<uintptr_t>(workspace) & (kWsAlign - 1)) != 0) return KF_ERR_ALIGN;
    }
    set_paged(pl.prm, Q, strides, K_pages, block_table, seq_starts, kv_lens, n_seqs, tokens, H_q, H_kv, D,
              max_pages_per_seq, num_pages, flags);
    pl.prm.row_lse = reinterpret_cast<const uint32_t*>(lse);
    pl.prm.weights = weights;
    pl.prm.Opart = static_cast<float*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return (flags & KF_BF16) ? launch_weigh_dim<true>(pl, D, s) : launch_weigh_dim<false>(pl, D, s);
}

size_t kf_kv_evict_workspace_bytes(int n_seqs, int H_kv, int D, int page_size, int max_pages_per_seq) {
    EvictPlan pl;
    return evict_plan(n_seqs, H_kv, D, page_size, max_pages_per_seq, 1, &pl) == KF_OK ? pl.ws_bytes : 0;
}

int kf_kv_evict(void* K_pages, void* V_pages, float* weights, const int* block_table, const int* kv_lens,
                const int* budgets, int* kept, int n_seqs, int H_kv, int D, int page_size, int max_pages_per_seq,
                int num_pages, int recent, void* workspace, size_t workspace_bytes, void* stream) {
    EvictPlan pl;
    if (const int st = evict_plan(n_seqs, H_kv, D, page_size, max_pages_per_seq, num_pages, &pl); st != KF_OK) return st;
    if (recent < 0) return KF_ERR_SIZE;
    if (!K_pages || !V_pages || !weights || !block_table || !kv_lens || !budgets || !kept) return KF_ERR_NULL;
    if (!aligned16(K_pages) || !aligned16(V_pages)) return KF_ERR_ALIGN;
    if (!aligned4(weights) || !aligned4(block_table) || !aligned4(kv_lens) || !aligned4(budgets) || !aligned4(kept))
        return KF_ERR_ALIGN;
    if (!workspace || workspace_bytes < pl.ws_bytes) return KF_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & (kWsAlign - 1)) != 0) return KF_ERR_ALIGN;
    kf::EvictParams prm{};
    prm.pages[0] = static_cast<uint8_t*>(K_pages);
    prm.pages[1] = static_cast<uint8_t*>(V_pages);
    prm.weights = reinterpret_cast<uint32_t*>(weights);
    prm.block_table = block_table;
    prm.kv_lens = kv_lens;
    prm.budgets = budgets;
    prm.kept = kept;
    prm.n_seqs = n_seqs;
    prm.heads = H_kv;
    prm.recent = recent;
    prm.max_pages = max_pages_per_seq;
    prm.page_shift = pl.shift;
    prm.num_pages = num_pages;
    prm.capacity = pl.capacity;
    char* ws = static_cast<char*>(workspace);
    prm.parts = pl.parts;
    prm.cuts = reinterpret_cast<int*>(ws);
    prm.moves = reinterpret_cast<int*>(ws + pl.cuts_bytes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: return launch_evict<64>(prm, s);
        case 128: return launch_evict<128>(prm, s);
        default: return launch_evict<256>(prm, s);
    }
}

}  // extern "C"
