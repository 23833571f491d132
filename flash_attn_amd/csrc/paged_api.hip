// C entry points of rotary positions and of the paged cache (include/flash_attn_mi355.h): argument checks, split count, launches.
#include "flash_attn_mi355.h"

#include <cmath>
#include <cstring>

#include "api_common.h"
#include "paged_kernel.h"
#include "rotary_kernels.h"

namespace {

using fa::device_usable;
using fa::misaligned;
using fa::record_hip;

constexpr int kNumCU = 256;  // MI355X
constexpr int kMostTokens = 1 << 25;
constexpr long long kMostOfToken = 1LL << 30;  // elements of a token's heads: the kernels count them in an int, with a launch's step on top

// strides of rows that are moved 16 bytes at a time
inline bool odd_stride(int64_t s) { return (s & 7) != 0; }

// ---------------------------------------------------------------------------------------------- rotary

int run_rotary(const flash_rotary_params* p, hipStream_t st)
{
    if (!p) return FLASH_EINVAL;
    if (p->dtype != FLASH_FP16 && p->dtype != FLASH_BF16 && p->dtype != FLASH_FP32) return FLASH_EINVAL;
    if (p->B < 0 || p->H < 0 || p->N < 0 || p->d <= 0) return FLASH_EINVAL;
    if (p->rot < 2 || (p->rot & 1) || p->rot > p->d || p->rot > 512) return FLASH_EINVAL;
    // (a wave per row of a batch: a launch is limited to 2^32 threads)
    if ((long long)p->B * p->N > kMostTokens || (long long)p->H * p->d > kMostOfToken) return FLASH_EINVAL;
    if (!std::isfinite(p->factor)) return FLASH_EINVAL;
    for (int64_t s : {p->x_batch, p->x_head, p->x_row, p->y_batch, p->y_head, p->y_row, p->positions_batch})
        if (s < 0) return FLASH_EINVAL;
    if (p->B == 0 || p->H == 0 || p->N == 0) return FLASH_OK;
    if (!p->X || !p->Y || !p->positions || !p->inv_freq) return FLASH_EINVAL;
    // (in place: the same rows, not others of the same memory)
    if (p->X == p->Y && ((p->B > 1 && p->x_batch != p->y_batch) || (p->H > 1 && p->x_head != p->y_head) || (p->N > 1 && p->x_row != p->y_row)))
        return FLASH_EINVAL;
    // (rows that are one and the same cannot be written)
    if ((p->B > 1 && p->y_batch == 0) || (p->H > 1 && p->y_head == 0) || (p->N > 1 && p->y_row == 0)) return FLASH_EINVAL;
    const size_t size = p->dtype == FLASH_FP32 ? 4 : 2;
    if (misaligned(p->X, size) || misaligned(p->Y, size) || misaligned(p->positions, p->positions_64 ? 8 : 4) || misaligned(p->inv_freq, 4))
        return FLASH_EALIGN;
    if (const int rc = device_usable(); rc != FLASH_OK) return rc;
    int wide = 8;  // elements at once, as far as addresses and strides allow
    while (wide > 1) {
        bool fits = !misaligned(p->X, wide * size) && !misaligned(p->Y, wide * size);
        for (int64_t s : {p->B > 1 ? p->x_batch : 0, p->B > 1 ? p->y_batch : 0, p->H > 1 ? p->x_head : 0, p->H > 1 ? p->y_head : 0, p->N > 1 ? p->x_row : 0,
                          p->N > 1 ? p->y_row : 0})
            fits = fits && s % wide == 0;
        if (fits) break;
        wide /= 2;
    }
    fa::RotaryArgs a{};
    a.X = p->X, a.Y = p->Y, a.positions = p->positions, a.inv_freq = p->inv_freq;
    a.x_batch = p->x_batch, a.x_head = p->x_head, a.x_row = p->x_row;
    a.y_batch = p->y_batch, a.y_head = p->y_head, a.y_row = p->y_row, a.positions_batch = p->positions_batch;
    a.factor = p->factor;
    a.B = p->B, a.H = p->H, a.N = p->N, a.d = p->d, a.rot = p->rot;
    a.positions_64 = p->positions_64 != 0, a.interleaved = p->interleaved != 0, a.inverse = p->inverse != 0;
    return record_hip(fa::launch_rotary(a, p->dtype, wide, st));
}

// ---------------------------------------------------------------------------------------------- paged cache

// sizes, types and strides that both entry points share; *empty: nothing to do
int validate_paged(const flash_paged_params* p, bool* empty)
{
    *empty = false;
    if (!p) return FLASH_EINVAL;
    if (p->dtype != FLASH_FP16 && p->dtype != FLASH_BF16) return FLASH_EINVAL;
    if (p->B < 0 || p->H <= 0 || p->H_kv <= 0 || p->H % p->H_kv != 0 || p->d <= 0) return FLASH_EINVAL;
    if (p->d > FLASH_MAX_HEAD_DIM) return FLASH_EHEADDIM;
    if (p->d % 8 != 0) return FLASH_EINVAL;
    if (p->total_q < 0 || p->num_pages < 0 || p->max_pages < 0 || p->page_size <= 0 || p->page_size % 16 != 0) return FLASH_EINVAL;
    if (p->max_seqlen_q < 0 || p->max_seqlen_k < 0 || p->block_table_stride < 0) return FLASH_EINVAL;
    // (positions and keys stay far below 2^31 in the kernels' int arithmetic)
    if ((long long)p->page_size * p->max_pages > (1LL << 30) || p->total_q > kMostTokens || p->B > (1 << 24)) return FLASH_EINVAL;
    if ((long long)p->total_q * p->H > 0x7fffffffLL - 0x1000000 || (long long)p->H * p->d > kMostOfToken) return FLASH_EINVAL;
    if (p->num_splits > FLASH_MAX_SPLITS) return FLASH_ESPLITS;
    if (p->B == 0 || p->total_q == 0) *empty = true;
    return FLASH_OK;
}

// the cache's strides, bases and index tensors; `launch` alone has pointers
int validate_cache(const flash_paged_params* p)
{
    for (int64_t s : {p->kc_page, p->kc_head, p->kc_row, p->vc_page, p->vc_head, p->vc_row})
        if (s < 0 || odd_stride(s)) return FLASH_EINVAL;
    // (the kernels address the 16 rows of a request with 32 bits, and multiply a page's number by 32 bits)
    if (p->kc_row > (1 << 26) || p->vc_row > (1 << 26) || p->kc_page > 0x7fffffffLL || p->vc_page > 0x7fffffffLL) return FLASH_EINVAL;
    if (!p->seqlens_k || !p->cu_seqlens_q) return FLASH_EINVAL;
    if (p->max_pages > 0 && !p->block_table) return FLASH_EINVAL;
    if (misaligned(p->seqlens_k, 4) || misaligned(p->cu_seqlens_q, 4) || misaligned(p->block_table, 4)) return FLASH_EALIGN;
    if (p->num_pages > 0) {
        if (!p->K_cache || !p->V_cache) return FLASH_EINVAL;
        if (misaligned(p->K_cache, 16) || misaligned(p->V_cache, 16)) return FLASH_EALIGN;
    }
    return FLASH_OK;
}

// rows [tokens, heads, d] that are written: no two of them the same
bool apart(int64_t token, int64_t head, int tokens, int heads) { return (tokens <= 1 || token != 0) && (heads <= 1 || head != 0); }

int rows_strides(int64_t token, int64_t head, const void* base)
{
    if (token < 0 || head < 0 || odd_stride(token) || odd_stride(head)) return FLASH_EINVAL;
    if (!base) return FLASH_EINVAL;
    return misaligned(base, 16) ? FLASH_EALIGN : FLASH_OK;
}

int group_of(const flash_paged_params* p) { return p->H / p->H_kv; }
int longest_chunk(const flash_paged_params* p) { return p->max_seqlen_q > 0 && p->max_seqlen_q < p->total_q ? p->max_seqlen_q : p->total_q; }
int capacity_of(const flash_paged_params* p) { return p->num_pages > 0 ? p->page_size * p->max_pages : 0; }

long long blocks_of(const flash_paged_params* p, int br)
{
    const int G = group_of(p);
    const long long each = ((long long)longest_chunk(p) * G + br - 1) / br;
    const long long all = (long long)p->total_q * G / br + p->B;
    return each * p->B < all ? each * p->B : all;
}

// bounds that can never cut are none: the kernels' position + right stays in an int
int window_left_of(const flash_paged_params* p) { return p->window_left >= capacity_of(p) ? -1 : p->window_left; }
// (the last row stands at the last key, and no row more than a chunk in front of it)
int window_right_of(const flash_paged_params* p) { return p->window_right >= p->total_q ? -1 : p->window_right; }

// keys of the longest sequence
int keys_of(const flash_paged_params* p)
{
    const int cap = capacity_of(p);
    return p->max_seqlen_k > 0 && p->max_seqlen_k < cap ? p->max_seqlen_k : cap;
}

// tiles of 64 keys that the masks leave a block of br rows, at most
int window_tiles(const flash_paged_params* p, int br)
{
    const int wl = window_left_of(p), wr = window_right_of(p);
    if (wl < 0 || (!p->is_causal && wr < 0)) return 0x7fffffff;
    return (int)(((long long)wl + 1 + (p->is_causal ? 0 : wr) + (br + group_of(p) - 1) / group_of(p) + 63 + 63) / 64);
}
// ... and that it sees
int most_tiles(const flash_paged_params* p, int br)
{
    const int keys = keys_of(p), w = window_tiles(p, br);
    return w < (keys + 63) / 64 ? w : (keys + 63) / 64;
}

// Rows of a work-group, which says which form: 32 or 256.  Up to 64 rows per K/V head and sequence 32 are the faster ones at every length: their
// waves stream tiles of their own (B64 H_kv8 500 keys, 40 rows 21.7 us against 31.4; B8 H_kv8 4000 keys, 64 rows 27.9 / 31.6).  Longer
// chunks take them while the launch is short and its work-groups are on the GPU together: a work-group of 256 rows walks its tiles at up to 2 us
// each whether or not it is alone, where one of 32 rows has four waves at it.  In units of 32 rows x 64 keys the small ones, each of which
// asks the L2 for its tiles, cost 2 ns at d = 128 and 1 ns at d = 64 once the GPU is full, the large ones 1 and 0.7 ns.
// 32 rows / 256 rows, one MI355X: d128 H8 1000 causal rows (2000 units) 16.0 / 26.1 us, 512 rows on 1000 keys (2600) 19.2 / 26.0, 1000 on 1000
// (6100) 26.0 / 28.8, 100 on 16000 (8000) 30.9 / 26.1, 256 on 16000 (16000) 49.9 / 36.5; d64 H16 2000 (16000) 26.9 / 37.2, 4096 (68000)
// 77 / 68; more than 1024 work-groups: d128 B8 H32 H_kv8 up to 256 (3400 units, 1136 work-groups) 22.3 / 14.5.  (128 rows, four waves that share
// tiles, two work-groups per CU, were the fastest by more than 5 % on 3 of 94 such launches, 13.6 us against 14.5 at best.)
constexpr int kShortRows = 64, kShortUnits = 7000, kShortUnits64 = 30000, kShortGroups = 1024;
int rows_per_group(const flash_paged_params* p)
{
    const long long chunk = longest_chunk(p), groups = blocks_of(p, fa::kPagedFewRows) * p->H_kv;
    if (chunk * group_of(p) <= kShortRows) return fa::kPagedFewRows;
    long long tiles = most_tiles(p, fa::kPagedFewRows);
    const long long keys = keys_of(p);
    if (p->is_causal && tiles > (keys - chunk / 2) / 64 + 1) tiles = (keys > chunk / 2 ? keys - chunk / 2 : 0) / 64 + 1;  // (the mean row's)
    return groups <= kShortGroups && groups * tiles <= (p->d <= 64 ? kShortUnits64 : kShortUnits) ? fa::kPagedFewRows : fa::kPagedTallRows;
}

// Whether the work-groups of a launch in splits are the pieces that its row blocks have, one after the other (PagedArgs::pieces): where the mask cuts
// the ends of the ranges alone, and a wave has a lane for each split of each sequence.  (32 rows in long caches, where nearly all pieces are
// there, stay in the order that leaves row blocks of the same keys to the same XCD.)
bool real_pieces(const flash_paged_params* p, int br, int splits)
{
    if (splits < 2 || (long long)p->B * splits > 64 || window_left_of(p) >= 0 || (!p->is_causal && window_right_of(p) < 0)) return false;
    return br == fa::kPagedTallRows || ((long long)longest_chunk(p) * group_of(p) > br && keys_of(p) / 2 <= longest_chunk(p));
}

// Splits by an estimate, for launches with several row blocks per sequence:
//     begin + tiles of a piece * t + [splits > 1] (merge + partial results written and read at 7 TB/s)
// as long as the pieces have a CU each, or half of one (32 rows, d <= 64: t grows by half then; at d = 128 two on a CU take twice as long).  Under
// a causal mask the first row blocks have fewer pieces than the last, so there may be more splits than places per row block.  One MI355X, splits that a
// CU for every row block and split would allow / by this rule, us: 4096 causal rows H4 d128 4: 47.7, 7: 40.7; H8 2: 72.4, 3: 63.0; 2 x 3000 rows
// H4 2: 57.4, 4: 44.0; 1500 rows H16 H_kv2 2: 41.4, 4: 34.8; 8192 rows H4 d64 2: 80.0, 3: 63.5; where nothing is gained: 2048 rows in a window of 600, H16
// H_kv8, 26.5 whole, 36.6 in 2.  32 rows: 2839 causal rows H1 d128 2: 24.1, 5: 19.3; 2 x up to 2359 rows H1 d96 1: 29.4, 2: 23.2; 875 rows on 4989 keys
// H4 d64 2: 25.4, 4: 20.8; the worst of 130 random launches 367 rows on 8324 keys H2 d96 11: 19.3, 8: 21.0.
constexpr double kPartialBytesPerUs = 7e6;
int splits_by_estimate(const flash_paged_params* p, int br, int nt)
{
    // row blocks of a chunk of mean length behind the longest sequence's keys
    const bool tall = br == fa::kPagedTallRows, narrow = p->d <= 64;
    const int G = group_of(p), keys = keys_of(p), reach = p->is_causal ? 0 : window_right_of(p);
    const int mean = (p->total_q + p->B - 1) / p->B, chunk = mean < longest_chunk(p) ? mean : longest_chunk(p);
    const long long n = ((long long)chunk * G + br - 1) / br, parts = (long long)p->B * p->H_kv;
    const double begin_us = tall ? 7.0 : 4.5, merge_us = tall ? 8.0 : 3.0, tile_us = tall ? (narrow ? 0.95 : p->d <= 96 ? 1.35 : 1.53) : narrow ? 0.365 : 0.6;
    const double split_us = 8.0 * p->d * p->total_q * p->H / kPartialBytesPerUs;
    const long long places = !tall && narrow ? 2 * kNumCU : kNumCU + kNumCU / 32;  // (a few more find a CU that short pieces have left)
    double best = begin_us + nt * tile_us;
    int chosen = 1;
    for (int s = 2; s <= nt && s <= FLASH_MAX_SPLITS; ++s) {
        const int per = (nt + s - 1) / s;
        if ((nt + per - 1) / per != s) continue;  // (a smaller count says the same)
        long long pieces = n * s;
        if (real_pieces(p, br, s)) {
            pieces = n;
            if (s <= n) {
                for (int k = 1; k < s; ++k) {
                    const long long key = 64LL * per * k, x = key - (keys - chunk) - reach;
                    pieces += keys <= key || x >= chunk ? 0 : n - (x > 0 ? x * G / br : 0);
                }
            } else {
                for (long long m = 0; m < n; ++m) {
                    const long long last = ((m + 1) * br < (long long)chunk * G ? (m + 1) * br : (long long)chunk * G) - 1, hi = keys - chunk + last / G + 1 + reach;
                    const long long tiles = ((hi < keys ? hi : keys) + 63) / 64;
                    pieces += tiles > per ? (tiles + per - 1) / per - 1 : 0;
                }
            }
        } else if (!tall && (long long)s * p->H_kv > 8 && (long long)s * p->H_kv % 8 != 0) {
            continue;  // (row blocks that read the same keys would lie on different XCDs: 80 rows on 13400 keys, B 8, H 1, 10 splits 34.7 us, 8 27.1)
        }
        if (pieces * parts > places) break;
        const double us = begin_us + per * tile_us * (!tall && pieces * parts > kNumCU ? 1.5 : 1.0) + merge_us + split_us * pieces / n;
        if (us < best) best = us, chosen = s;
    }
    return chosen;
}

// Split count that the library chooses.  One row block of 32 rows per sequence: a work-group per CU at least, as long as each split has two tiles; and
// where there are several sequences, whose lengths nobody here knows, pieces of some kFewestTiles tiles, so that the long sequences of a batch do not
// outlast the others.  The merge reads 8 B H d bytes per split and token more, which is little next to the keys of a piece.  Its launch costs 3 us, in
// which a work-group of 32 rows walks some tiles: shorter ranges stay whole.  Whole / in splits, single tokens, H 8, H_kv 2, one MI355X: d = 128
// 256 keys 6.3 / 9.3 us, 512 keys 8.6 / 9.3, 1024 keys 13.6 / 9.2; d = 64, G = 1: 512 keys 6.3 / 9.5, 1024 keys 8.9 / 9.5, 2048 keys 14.7 / 9.1.
constexpr int kFewestTiles = 32, kMostGroups = 2048, kWholeTiles = 8, kWholeTiles64 = 16;
int splits_of(const flash_paged_params* p)
{
    const int br = rows_per_group(p), nt = most_tiles(p, br);
    if (nt <= 1 || (long long)p->total_q * p->H >= 1LL << 26) return 1;  // (the merge has a wave per row: 2^32 threads)
    long long s = p->num_splits;
    if (s <= 0) {
        const long long groups = blocks_of(p, br) * p->H_kv;
        if (br == fa::kPagedTallRows) return groups >= kNumCU ? 1 : splits_by_estimate(p, br, nt);
        if (nt <= (p->d <= 64 ? kWholeTiles64 : kWholeTiles)) return 1;
        if ((long long)longest_chunk(p) * group_of(p) > br) {
            s = splits_by_estimate(p, br, nt);
        } else {
            s = groups >= kNumCU ? 1 : kNumCU / groups;
            if (s > nt / 2) s = nt / 2;
        }
        if (p->B > 1) {
            long long more = kFewestTiles;
            more = nt / more < kMostGroups / groups ? nt / more : kMostGroups / groups;
            if (more > s) s = more;
        }
    }
    if (s > nt) s = nt;
    if (s > FLASH_MAX_SPLITS) s = FLASH_MAX_SPLITS;
    if (s < 1) s = 1;
    const int per = (int)((nt + s - 1) / s);
    return (nt + per - 1) / per;
}

// Whether the row blocks of all sequences are started by the end of their keys, heaviest first under a causal mask, instead of sequence by sequence:
// work-groups are dealt to the XCDs strictly in turn, so that behind the light ones at a sequence's end the heavy ones of the next wait for
// one XCD while others have room, and the launch's last ones may be heavy.  For it the work-groups of a sequence are less often at the same
// keys together, and a work-group's look for its place takes 0.3 us more.  In order of sequences / of ends, one MI355X: 900 causal rows, B 3, H 24, d 128
// (288 work-groups) 37.8 / 29.8 us; 789 rows, B 18, H 8, d 64 (576) 48.7 / 35.8; up to 2942, B 34, H 2, d 64 (458) 66.3 / 49.4; up to 3 x 8192, H 8,
// H_kv 1, d 128 270 / 227; up to 1885, B 19, H 8, d 128 (736) 92.0 / 80.2; worst 837 rows on 1902 keys, B 4, H 64, H_kv 16, d 80 (896) 220 / 229.
// Long launches even out by themselves: 1300 to 8600 work-groups gained 8 % at best and lost 14 % (442 rows, B 14, H 64, H_kv 32, d 128, 1792
// work-groups, 99.2 / 112.2); short sequences in many work-groups lost too (203 rows, B 5, H 256, H_kv 32, d 64, 1120 work-groups 31.3 / 33.9).
constexpr int kOrderedGroups = 1300, kOrderedShort = 900, kShortKeys = 256;
bool ordered(const flash_paged_params* p, int br)
{
    if (br != fa::kPagedTallRows || p->B < 2 || p->B > 64) return false;
    const long long groups = blocks_of(p, br) * p->H_kv;  // (a CU for each: nothing to order)
    return groups > kNumCU && groups <= (keys_of(p) > kShortKeys ? kOrderedGroups : kOrderedShort);
}

int run_forward(const flash_paged_params* p, hipStream_t st)
{
    bool empty;
    int rc = validate_paged(p, &empty);
    if (rc != FLASH_OK) return rc;
    if (!(p->softmax_scale > 0.0f) || std::isinf(p->softmax_scale)) return FLASH_EINVAL;
    if (empty) return FLASH_OK;
    if ((rc = validate_cache(p)) != FLASH_OK) return rc;
    if ((rc = rows_strides(p->q_token, p->q_head, p->Q)) != FLASH_OK || (rc = rows_strides(p->o_token, p->o_head, p->O)) != FLASH_OK) return rc;
    if (!p->LSE || !apart(p->o_token, p->o_head, p->total_q, p->H)) return FLASH_EINVAL;
    if (misaligned(p->LSE, 4)) return FLASH_EALIGN;
    const int br = rows_per_group(p), splits = splits_of(p), nt = most_tiles(p, br);
    if (splits > 1) {
        if (!p->O_partial || !p->LSE_partial) return FLASH_EWORKSPACE;
        if (misaligned(p->O_partial, 16) || misaligned(p->LSE_partial, 4)) return FLASH_EALIGN;
    }
    const long long blocks = blocks_of(p, br) * p->H_kv * splits;
    if (blocks * fa::paged_threads(br) >= 1LL << 32) return FLASH_EINVAL;
    if ((rc = device_usable()) != FLASH_OK) return rc;
    fa::PagedArgs a{};
    a.Q = static_cast<const char*>(p->Q), a.K = static_cast<const char*>(p->K_cache), a.V = static_cast<const char*>(p->V_cache);
    a.O = static_cast<char*>(p->O), a.LSE = p->LSE, a.O_partial = p->O_partial, a.LSE_partial = p->LSE_partial;
    a.table = p->block_table, a.lens = p->seqlens_k, a.cu = p->cu_seqlens_q;
    a.q_token = 2 * p->q_token, a.q_head = 2 * p->q_head, a.o_token = 2 * p->o_token, a.o_head = 2 * p->o_head;
    a.k_page = (uint32_t)(2 * p->kc_page), a.k_head = 2 * p->kc_head, a.v_page = (uint32_t)(2 * p->vc_page), a.v_head = 2 * p->vc_head;
    a.k_row = (uint32_t)(2 * p->kc_row), a.v_row = (uint32_t)(2 * p->vc_row);
    a.table_stride = p->block_table_stride;
    a.B = p->B, a.H = p->H, a.Hk = p->H_kv, a.G = group_of(p), a.d = p->d, a.tokens = p->total_q, a.num_pages = p->num_pages, a.page = p->page_size;
    a.capacity = capacity_of(p);
    a.causal = p->is_causal != 0, a.wl = window_left_of(p), a.wr = window_right_of(p);
    a.scale_log2 = p->softmax_scale * fa::kLog2e;
    a.num_splits = splits, a.tiles_per_split = (nt + splits - 1) / splits, a.window_tiles = window_tiles(p, br);
    a.direct = (long long)longest_chunk(p) * a.G <= br;
    a.ordered = splits == 1 && ordered(p, br) ? (keys_of(p) + 8) / 9 : 0;
    a.pieces = real_pieces(p, br, splits);
    a.by_heads = fa::fast_div(a.Hk), a.by_group = fa::fast_div(a.G), a.by_page = fa::fast_div(a.page);
    a.by_splits = fa::fast_div(splits);
    const bool bf16 = p->dtype == FLASH_BF16;
    rc = record_hip(p->d <= 64 ? fa::launch_paged_d64(a, bf16, br, blocks, st) : fa::launch_paged_d128(a, bf16, br, blocks, st));
    if (rc != FLASH_OK || splits == 1) return rc;
    return record_hip(fa::launch_paged_merge(a, bf16, st));
}

int run_append(const flash_paged_params* p, hipStream_t st)
{
    bool empty;
    int rc = validate_paged(p, &empty);
    if (rc != FLASH_OK) return rc;
    const bool turns = p->inv_freq != nullptr, queries = turns && p->Q != nullptr;
    if (turns) {
        if (p->rot < 2 || (p->rot & 1) || p->rot > p->d || !std::isfinite(p->factor)) return FLASH_EINVAL;
        if (misaligned(p->inv_freq, 4)) return FLASH_EALIGN;
        if (p->positions && misaligned(p->positions, p->positions_64 ? 8 : 4)) return FLASH_EALIGN;
    }
    if (empty) return FLASH_OK;
    if ((rc = validate_cache(p)) != FLASH_OK) return rc;
    if ((rc = rows_strides(p->k_token, p->k_head, p->K)) != FLASH_OK || (rc = rows_strides(p->v_token, p->v_head, p->V)) != FLASH_OK) return rc;
    if (p->num_pages > 0 && (!apart(p->kc_page, p->kc_head, p->num_pages, p->H_kv) || p->kc_row == 0 || !apart(p->vc_page, p->vc_head, p->num_pages, p->H_kv) ||
                             p->vc_row == 0))
        return FLASH_EINVAL;
    if (queries) {
        if ((rc = rows_strides(p->q_token, p->q_head, p->Q)) != FLASH_OK || (rc = rows_strides(p->o_token, p->o_head, p->O)) != FLASH_OK) return rc;
        if (!apart(p->o_token, p->o_head, p->total_q, p->H)) return FLASH_EINVAL;
        if (p->Q == p->O && ((p->total_q > 1 && p->q_token != p->o_token) || (p->H > 1 && p->q_head != p->o_head))) return FLASH_EINVAL;
    }
    if ((rc = device_usable()) != FLASH_OK) return rc;
    fa::AppendArgs a{};
    a.Q = p->Q, a.K = p->K, a.V = p->V, a.O = p->O, a.K_cache = p->K_cache, a.V_cache = p->V_cache, a.positions = p->positions;
    a.table = p->block_table, a.lens = p->seqlens_k, a.cu = p->cu_seqlens_q, a.inv_freq = p->inv_freq;
    a.q_token = p->q_token, a.q_head = p->q_head, a.o_token = p->o_token, a.o_head = p->o_head;
    a.k_token = p->k_token, a.k_head = p->k_head, a.v_token = p->v_token, a.v_head = p->v_head;
    a.kc_page = p->kc_page, a.kc_head = p->kc_head, a.kc_row = p->kc_row, a.vc_page = p->vc_page, a.vc_head = p->vc_head, a.vc_row = p->vc_row;
    a.table_stride = p->block_table_stride;
    a.factor = p->factor;
    a.B = p->B, a.H = queries ? p->H : 0, a.Hk = p->H_kv, a.d = p->d, a.rot = turns ? p->rot : 0, a.tokens = p->total_q, a.num_pages = p->num_pages;
    a.page = p->page_size, a.capacity = capacity_of(p), a.positions_64 = p->positions_64 != 0, a.interleaved = turns && p->interleaved != 0;
    return record_hip(fa::launch_append(a, p->dtype, st));
}

}  // namespace

#define FLASH_EXPORT __attribute__((visibility("default")))

extern "C" {

FLASH_EXPORT int flash_rotary(const flash_rotary_params* p, void* stream) { return run_rotary(p, static_cast<hipStream_t>(stream)); }

FLASH_EXPORT int flash_append_paged(const flash_paged_params* p, void* stream) { return run_append(p, static_cast<hipStream_t>(stream)); }

FLASH_EXPORT int flash_forward_paged(const flash_paged_params* p, void* stream) { return run_forward(p, static_cast<hipStream_t>(stream)); }

FLASH_EXPORT int flash_forward_paged_resolve_splits(const flash_paged_params* p)
{
    bool empty;
    const int rc = validate_paged(p, &empty);
    if (rc != FLASH_OK) return rc;
    return empty ? 1 : splits_of(p);
}

FLASH_EXPORT int flash_forward_paged_workspace_bytes(const flash_paged_params* p, size_t* o_partial_bytes, size_t* lse_partial_bytes)
{
    bool empty;
    const int rc = validate_paged(p, &empty);
    if (rc != FLASH_OK) return rc;
    const int splits = empty ? 1 : splits_of(p);
    const size_t rows = splits > 1 ? (size_t)p->total_q * p->H * splits : 0;
    if (o_partial_bytes) *o_partial_bytes = rows * p->d * sizeof(float);
    if (lse_partial_bytes) *lse_partial_bytes = rows * sizeof(float);
    return FLASH_OK;
}

FLASH_EXPORT void flash_rotary_params_init(flash_rotary_params* p)
{
    if (!p) return;
    std::memset(p, 0, sizeof(*p));
    p->factor = 1.0f;
}

FLASH_EXPORT void flash_paged_params_init(flash_paged_params* p)
{
    if (!p) return;
    std::memset(p, 0, sizeof(*p));
    p->window_left = p->window_right = -1;
    p->factor = 1.0f;
}

FLASH_EXPORT size_t flash_rotary_params_size(void) { return sizeof(flash_rotary_params); }
FLASH_EXPORT size_t flash_paged_params_size(void) { return sizeof(flash_paged_params); }

}  // extern "C"
