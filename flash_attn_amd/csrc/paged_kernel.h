// Attention of ragged chunks of new tokens over a paged K/V cache (flash_forward_paged), fp16 and bf16, d a multiple of 8 up to 128.
//
//   O_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that row i sees, LSE_i = log sum_j exp(scale q_i . k_j)
//
// Sequence b has the query rows cu[b] ... cu[b + 1] - 1 of Q [tokens, H, d] and lens[b] keys; key j lies in row j % page of page
// table[b][j / page].  The chunk's rows are the last of the sequence: row i stands at position i + len - rows.
// The G query heads of a K/V head are the rows of one problem over it: row r is query r / G of head r % G, so that K and V
// are read once per K/V head, whatever G is.
//
// Pages.  A request of the tile loads (global_load_lds_dwordx4, one KiB) covers 4 rows of 256 bytes or 8 of 128.  Tiles begin at multiples of
// 32 keys and pages hold multiples of 16, so the rows of a request lie in one page: its place is worked out on the scalar unit (an
// entry of the table by s_load, one tile ahead of its use, and two 32 x 32 -> 64-bit products) and the lanes' own offsets never change.
// No vector instruction goes into paging, and with it no page size costs more than another: 119 scalar instructions per tile and
// wave of the tall form beside 194 vector instructions and 32 MFMAs (185 with every address worked out where it is used).
//
// Two forms share the mathematics of fwd_kernel.h (S^T = K Q^T and O^T += V^T P^T on 32x32x16 MFMA, one query row per lane, scores
// scaled inside the exponent, a running maximum that is raised only when some row outgrows it by 2^8).  Scores, maxima, sums and O are held in
// 32 bits, partial results of splits and waves too; the probabilities are rounded once, to nearest, to the type of V, whose matrix product takes
// no other, behind the sum of the denominator, which has them as they are:
//   paged_tall_kernel  256 rows per work-group, eight waves that share the tiles, the schedule of fwd_pp_kernel.h: on every SIMD one
//                      wave is at its MFMAs while the other is at its softmax.  Bound by MFMA and softmax (and by the clock that the
//                      power management leaves them): 8192 causal rows H32 H_kv8 d128 bf16 505-537 us, 1.02-1.09 PFLOP/s.
//   paged_few_kernel   32 rows, four waves that share out the tiles, each with LDS stages of its own and no barrier in the loop;
//                      the four results are merged through LDS.  Bound by HBM: single tokens B16 H32 H_kv32 on 4096 keys d128 163 us,
//                      6.6 TB/s.
// Either form may split the key range (num_splits): partial results in fp32, merged by paged_merge_kernel.  Which one a call gets:
// rows_per_group in paged_api.hip.
//
// What is not in the sequence must not reach the result: keys past its end are not read, columns d ... D - 1 of the tiles in LDS are zeroed once and
// never requested, and a product of a masked probability, 0, with a V that is not finite is taken back out at the end (rescue).  Rows of a tile past the
// sequence's end repeat the last key's in K, whose scores are masked.  In V they have to be finite whatever the last key holds, which its row may
// see: in the 32-row form they come from a row of zeroes (kPagedZeroes), in the 256-row form they are cleared if need be (paged_clear_past).
#pragma once
#include <type_traits>

#include "combine.h"
#include "common.h"

namespace fa {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kPagedTallRows = 256, kPagedMidRows = 128, kPagedFewRows = 32;  // rows of a work-group
constexpr int kPagedCus = 256;                                                      // of an MI355X
constexpr int paged_threads(int rows) { return rows == kPagedTallRows ? 512 : 256; }

struct PagedArgs {
    // what a work-group needs to find its place comes first
    const int32_t *table, *lens, *cu;
    FastDiv by_heads;
    int Hk, num_splits, B, direct;     // direct: every sequence has one row block
    int pieces;                        // != 0: of the splits only those that a row block has
    int ordered;                       // > 0: row blocks of all sequences by the end of their keys, in pieces of so many
    int tiles_per_split, window_tiles; // window_tiles: tiles of 64 keys that the masks leave a row block at most
    FastDiv by_splits, by_group, by_page;
    int H, G, d, tokens, num_pages, page, capacity;  // capacity: keys that a row of the table can name
    int causal, wl, wr;                // wl / wr < 0: unbounded
    const char *Q, *K, *V;
    char* O;
    float* LSE;                        // [tokens, H]
    float *O_partial, *LSE_partial;    // [tokens, H, S, d] and [tokens, H, S]
    int64_t q_token, q_head, o_token, o_head, k_head, v_head, table_stride;  // bytes (table_stride: entries)
    uint32_t k_page, v_page, k_row, v_row;                                   // bytes
    float scale_log2;
};

// Scores and masks beside those of flash_forward (flash_paged_params: softcap, alibi_slopes, prefix_lens, tree_mask); instances of their own, kScores:
enum { kScoresPlain, kScoresMasked, kScoresCapped, kScoresSloped, kScoresBoth };  // kScoresMasked: a prefix or a tree alone, which all but kScoresPlain take
constexpr bool has_cap(int scores) { return scores == kScoresCapped || scores == kScoresBoth; }
constexpr bool has_slopes(int scores) { return scores == kScoresSloped || scores == kScoresBoth; }

// With a bias by distance the tiles come last first: the nearest keys' scores are the largest, and the running maximum hardly ever moves behind them, where from
// the front it is raised, and O scaled, tile by tile (six prompts up to 2048 H16 d64 53.7 -> 49.5 us).
constexpr bool last_first(int scores) { return has_slopes(scores); }
// Tile of the range that comes in place t, for places past the end too
template <int kScores>
__device__ __forceinline__ int tile_of(int t, int ntiles) { return last_first(kScores) ? max(ntiles - 1 - t, 0) : t; }

constexpr int kTreeTokens = 256;  // drafted tokens of a sequence that a mask can name
struct ScoredExtras {
    const uint64_t* tree;       // [tokens, tree_words], or null.  With a tree `causal` is 0 and `wr` is -1
    const int32_t* prefix;      // [B], or null
    const float* slopes;        // [H]
    int64_t tree_stride;
    float cap_in, cap;          // exp2 of cap_in times a product is e^(2 score / cap)
    float slope_unit;           // of the slopes, to the units of what they are added to
    int tree_words;
};
// (in front: the line of arguments that is read first has them, and nobody waits for another)
struct ScoredArgs : ScoredExtras, PagedArgs {};
template <int kScores>
using ArgsOf = std::conditional_t<kScores == kScoresPlain, PagedArgs, ScoredArgs>;

// A kernel's own arguments, read once more where they stand: what is used behind the loop, or seldom, would otherwise lie in scalar registers all along, of which there
// are too few for all (60 of them went into lanes of a vector register and back: 250 instructions of the 1200 in front of the first product).
__device__ __forceinline__ const PagedArgs& read_again(const PagedArgs& a) { return a; }
__device__ __forceinline__ const ScoredArgs& read_again(const ScoredArgs&)
{
    uintptr_t at = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const ScoredArgs*)reinterpret_cast<const __attribute__((address_space(4))) ScoredArgs*>(at);
}

// What the merge needs of them (short arguments launch faster: common.h)
struct PagedMergeArgs {
    char* O;
    float* LSE;
    const float *O_partial, *LSE_partial;
    const int32_t* cu;
    int64_t o_token, o_head;
    int B, H, d, tokens, num_splits;
};

// An int that nobody writes during the launch at an address that is the same in all lanes: a load of the scalar unit.
__device__ __forceinline__ int read_uniform_int(const int32_t* p)
{
    return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

template <bool kBf16>
struct Elem {
    static __device__ __forceinline__ v16f mfma(v8h a, v8h b, v16f c)
    {
        if constexpr (kBf16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    // two floats rounded to nearest even, packed
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        const v2f t = {a, b};
        if constexpr (kBf16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(t, v2bf));
        else return __builtin_bit_cast(uint32_t, __builtin_convertvector(t, v2h));
    }
    static __device__ __forceinline__ float low(uint32_t u)
    {
        if constexpr (kBf16) return __uint_as_float(u << 16);
        else return (float)__builtin_bit_cast(v2h, u)[0];
    }
    static __device__ __forceinline__ float high(uint32_t u)
    {
        if constexpr (kBf16) return __uint_as_float(u & 0xffff0000u);
        else return (float)__builtin_bit_cast(v2h, u)[1];
    }
    // whether one of the two is infinite or not a number
    static __device__ __forceinline__ bool not_finite(uint32_t u)
    {
        constexpr uint32_t e = kBf16 ? 0x7f80u : 0x7c00u;
        return (u & e) == e || (u >> 16 & e) == e;
    }
};

// ---------------------------------------------------------------------------------------------- work of a work-group

struct PagedItem {
    int b, hk, split;
    int tok0, rows;   // first token of the chunk; query rows of the problem (tokens times heads per K/V head)
    int row0;         // first row of the work-group
    int len, shift;   // keys; position of query 0
    int splits, per;  // of the sequence (a.pieces: of the row block); tiles of a split
};

// Lengths come from device memory: whatever they hold, nothing outside the tensors is touched.
__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// inclusive sum over the lanes of a wave: inside rows of 16 lanes by DPP shifts, then the rows' last lanes
__device__ __forceinline__ int wave_prefix(int v, int lane)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr by 1, 2, 4, 8, nothing shifted in
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = r0 + __builtin_amdgcn_readlane(v, 31), r2 = r1 + __builtin_amdgcn_readlane(v, 47);
    return v + (lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r1 : r2);
}

// Tiles of a split of a sequence of `len` keys (*per), and its splits: pieces of as many tiles as the launch was sized for, or more, should
// the sequence be longer than the caller said.  a.window_tiles: tiles that the masks leave a row block at most.
__device__ __forceinline__ int splits_of_sequence(const PagedArgs& a, int len, int* per)
{
    const int nt = min((len + 63) >> 6, a.window_tiles);
    const int each = max(a.tiles_per_split, a.by_splits.quotient(nt + a.num_splits - 1));
    *per = each;
    if (a.num_splits == 1) return 1;
    return nt <= each ? 1 : (int)((uint32_t)(nt + each - 1) / (uint32_t)each);
}

// Keys at the begin of sequence b that all its tokens see
template <class A>
__device__ __forceinline__ int prefix_of(const A& a, int b)
{
    if constexpr (std::is_same_v<A, ScoredArgs>) return a.prefix ? clamp_int(a.prefix[b], 0, a.capacity) : 0;
    else return 0;
}

// Of a sequence's n row blocks those that see key c or one behind it: its last ones, as ends do not fall.
template <int BR, class A>
__device__ __forceinline__ int blocks_behind(const A& a, int tokens, int keys, int n, int c, int prefix)
{
    const int reach = a.causal ? 0 : a.wr;
    int x = max(c - (keys - tokens), -(1 << 30)) - reach;  // the first token that sees key c
    x = reach < 0 ? 0 : max(x, 0);
    if constexpr (std::is_same_v<A, ScoredArgs>) x = c < prefix ? 0 : x;
    return keys <= c || x >= tokens ? 0 : n - x * a.G / BR;
}

// Work-group -> (sequence, row block, split, K/V head); false where there is nothing to do.  K/V heads vary fastest, so that with a multiple
// of 8 of them the work-groups that read the same keys share an XCD's L2.  Behind that all pieces that the launch has come first, and the
// work-groups that there are too many of (lengths are known on the device alone) last: work-groups are started in order and dealt to the parts of an
// XCD in turn, and a launch with idle ones in between waits for one part with others empty.  Row blocks of a sequence come last first, which
// under a causal mask is heaviest first; a.ordered: those of all sequences, by the piece of nine of the longest length in which their keys end,
// the last piece first, a piece's sequences in turn.  a.pieces: first splits of a sequence's row blocks, second splits of those that have one, ...: under a
// causal mask the others would stand between them with nothing to do, and what comes behind the places of the GPU waits for a round.
template <int BR, class A>
__device__ __forceinline__ bool paged_item(const A& a, int lane, PagedItem* it)
{
    const int block = blockIdx.x, w = a.by_heads.quotient(block);
    it->hk = block - w * a.Hk;
    int b = 0, m = 0, c0, c1, len;
    if (a.direct && (a.num_splits == 1 || a.B == 1)) {  // one row block per sequence, and one split or sequence
        if (a.num_splits == 1) b = w, it->split = 0;
        else it->split = w;
        c0 = clamp_int(read_uniform_int(a.cu + b), 0, a.tokens), c1 = clamp_int(read_uniform_int(a.cu + b + 1), c0, a.tokens);
        len = clamp_int(read_uniform_int(a.lens + b), 0, a.capacity);
    } else if (a.ordered) {
        // A lane per sequence, B <= 64.  Two looks at two ends each find the piece of the work-group's row block.
        int first = 0, end = 0, keys = 0;
        if (lane < a.B) {
            first = a.cu[lane], end = a.cu[lane + 1], keys = a.lens[lane];
            first = clamp_int(first, 0, a.tokens), end = clamp_int(end, first, a.tokens), keys = clamp_int(keys, 0, a.capacity);
        }
        const int n = ((end - first) * a.G + BR - 1) / BR;
        const int prefix = prefix_of(a, lane < a.B ? lane : 0);
        auto ends_behind = [&](int t) { return blocks_behind<BR>(a, end - first, keys, n, a.ordered * t, prefix); };
        int t0 = 0, f0 = n, f1 = 0, before = 0;  // blocks behind the piece's begin (0: all) and behind its end (none behind the last); f1 of all lanes
#pragma unroll
        for (int step = 3; step > 0; step -= 2) {
            const int near = ends_behind(t0 + step), far = ends_behind(t0 + 2 * step);
            const uint32_t all = (uint32_t)__builtin_amdgcn_readlane(wave_prefix((int)((uint32_t)near + ((uint32_t)far << 16)), lane), 63);  // (kOrderedGroups: 16 bits hold each)
            const int all_near = (int)(all & 0xffffu), all_far = (int)(all >> 16);
            if (all_far > w) t0 += 2 * step, f0 = far;
            else if (all_near > w) t0 += step, f0 = near, f1 = far, before = all_far;
            else f1 = near, before = all_near;
        }
        const int upto = wave_prefix(f0 - f1, lane), local = w - before;
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > local);
        if (past == 0) return false;
        b = wave_uniform(__builtin_ctzll(past));
        const int block_of = __builtin_amdgcn_readlane(f1, b) + local - (__builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(f0 - f1, b));
        const int blocks = __builtin_amdgcn_readlane(n, b);
        if ((uint32_t)block_of >= (uint32_t)blocks) return false;  // (sums of offsets that make no sense may overflow)
        m = wave_uniform(blocks - 1 - block_of);
        it->split = 0;
        c0 = __builtin_amdgcn_readlane(first, b), c1 = __builtin_amdgcn_readlane(end, b), len = __builtin_amdgcn_readlane(keys, b);
    } else if (a.pieces) {
        // a lane per sequence and split, B * num_splits <= 64, windows without a left end: what is there of a split is the last row blocks
        const int bl = a.by_splits.quotient(lane), s = lane - bl * a.num_splits;
        int first = 0, end = 0, keys = 0, each = 1;
        if (bl < a.B) {
            first = a.cu[bl], end = a.cu[bl + 1], keys = a.lens[bl];
            first = clamp_int(first, 0, a.tokens), end = clamp_int(end, first, a.tokens), keys = clamp_int(keys, 0, a.capacity);
            splits_of_sequence(a, keys, &each);
        }
        const int n = ((end - first) * a.G + BR - 1) / BR;
        const int there = s == 0 ? n : blocks_behind<BR>(a, end - first, keys, n, (int)min((int64_t)s * each * 64, (int64_t)keys), prefix_of(a, bl < a.B ? bl : 0));
        const int upto = wave_prefix(there, lane);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > w);
        if (past == 0) return false;
        const int at = wave_uniform(__builtin_ctzll(past));
        const int block_of = w - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(there, at)), blocks = __builtin_amdgcn_readlane(n, at);
        if ((uint32_t)block_of >= (uint32_t)blocks) return false;
        b = wave_uniform(a.by_splits.quotient(at));
        it->split = at - b * a.num_splits;
        m = wave_uniform(blocks - 1 - block_of);
        c0 = __builtin_amdgcn_readlane(first, at), c1 = __builtin_amdgcn_readlane(end, at), len = __builtin_amdgcn_readlane(keys, at);
    } else {
        // 64 sequences at a time, a lane each
        int before = 0;
        bool found = false;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            const int mine = b0 + lane;
            int blocks = 0, splits = 1, per, first = 0, end = 0, keys = 0;
            if (mine < a.B) {
                first = a.cu[mine], end = a.cu[mine + 1], keys = a.lens[mine];
                first = clamp_int(first, 0, a.tokens), end = clamp_int(end, first, a.tokens), keys = clamp_int(keys, 0, a.capacity);
                blocks = ((end - first) * a.G + BR - 1) / BR;
                splits = splits_of_sequence(a, keys, &per);
            }
            const int upto = wave_prefix(blocks * splits, lane);
            const uint64_t past = __builtin_amdgcn_ballot_w64(before + upto > w);
            if (past != 0) {
                const int at = __builtin_ctzll(past);
                const int n = __builtin_amdgcn_readlane(blocks, at), each = __builtin_amdgcn_readlane(splits, at);
                const int local = w - (before + __builtin_amdgcn_readlane(upto, at) - n * each);
                const int block_of = each == 1 ? local : (int)((uint32_t)local / (uint32_t)each);
                b = wave_uniform(b0 + at);
                m = wave_uniform(n - 1 - block_of);
                it->split = wave_uniform(local - block_of * each);
                c0 = __builtin_amdgcn_readlane(first, at), c1 = __builtin_amdgcn_readlane(end, at), len = __builtin_amdgcn_readlane(keys, at);
                found = (uint32_t)block_of < (uint32_t)n;  // (sums of offsets that make no sense may overflow)
                break;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
        if (!found) return false;
    }
    it->b = b;
    it->tok0 = c0;
    it->rows = (c1 - c0) * a.G;
    it->row0 = m * BR;
    it->len = len;
    it->shift = len - (c1 - c0);
    it->splits = splits_of_sequence(a, len, &it->per);
    if (a.pieces) {  // of the row block
        const int last = min(it->row0 + BR, it->rows) - 1, reach = a.causal ? 0 : a.wr;
        int hi = reach < 0 ? len : min(len, a.by_group.quotient(last) + it->shift + reach + 1);
        if constexpr (std::is_same_v<A, ScoredArgs>) hi = max(hi, min(len, prefix_of(a, b)));
        it->splits = hi <= it->per * 64 ? 1 : (int)((uint32_t)((hi + 63) / 64 + it->per - 1) / (uint32_t)it->per);
    }
    return it->row0 < it->rows && it->split < it->splits;
}

// keys [kmin, kmax) that some row of the work-group sees, of those its split's share: the range of the row block is cut, not the
// sequence, so that windows and short chunks in long caches divide evenly
template <int BR, class A>
__device__ __forceinline__ void paged_range(const A& a, const PagedItem& it, int* kmin, int* kmax)
{
    const int last = it.row0 + BR < it.rows ? it.row0 + BR - 1 : it.rows - 1;
    const int p0 = a.by_group.quotient(it.row0) + it.shift, p1 = a.by_group.quotient(last) + it.shift;
    int lo = 0, hi = it.len;
    if (a.wl >= 0) lo = max(0, p0 - a.wl);
    if (a.causal) hi = min(hi, p1 + 1);
    if (a.wr >= 0) hi = min(hi, p1 + a.wr + 1);
    if constexpr (std::is_same_v<A, ScoredArgs>) {
        if (a.tree && a.wl >= 0) lo = max(0, it.shift - a.wl);  // (no token of a tree stands in front of the first one's place)
        hi = max(hi, min(it.len, prefix_of(a, it.b)));
    }
    if (it.splits > 1) {
        const int64_t s0 = ((int64_t)(lo >> 6) + (int64_t)it.split * it.per) * 64;
        lo = (int)max((int64_t)lo, min(s0, (int64_t)max(hi, lo)));
        if (it.split < it.splits - 1) hi = (int)min((int64_t)hi, s0 + (int64_t)it.per * 64);
    }
    *kmin = lo;
    *kmax = hi;
}

// The first split's work-group says of the splits that its sequence does not have that there is nothing in them.
template <int BR, int kThreads>
__device__ __forceinline__ void paged_mark_missing(const PagedArgs& a, const PagedItem& it, int tid)
{
    const int missing = a.num_splits - it.splits;
    if (it.split != 0 || missing == 0) return;
    const int n = min(BR, it.rows - it.row0);
    for (int r = tid / 16; r < n; r += kThreads / 16) {
        const int i = a.by_group.quotient(it.row0 + r), head = it.hk * a.G + (it.row0 + r - i * a.G);
        float* const lse = a.LSE_partial + ((size_t)(it.tok0 + i) * a.H + head) * a.num_splits + it.splits;
        for (int s = tid % 16; s < missing; s += 16) lse[s] = -INFINITY;
    }
}

// first and last key that row r (of the problem) sees; [lo, hi] may be empty
__device__ __forceinline__ void paged_bounds(const PagedArgs& a, const PagedItem& it, int r, int kmin, int kmax, int* lo, int* hi)
{
    const int p = a.by_group.quotient(r < it.rows ? r : it.rows - 1) + it.shift;
    int l = kmin, h = kmax - 1;
    if (a.wl >= 0) l = max(l, p - a.wl);
    if (a.causal) h = min(h, p);
    if (a.wr >= 0) h = min(h, p + a.wr);
    *lo = l;
    *hi = h;
}

__device__ __forceinline__ int row_token(const PagedArgs& a, const PagedItem& it, int r, int* head)
{
    const int i = a.by_group.quotient(r);
    *head = it.hk * a.G + (r - i * a.G);
    return it.tok0 + i;
}

// Where rows of the sequence lie: entry of the table and row within the page, asked for a tile ahead of their use.  Keys from len on
// stand for the last one.  The entry is kept inside the cache whatever the table holds.
struct PagedPlace {
    int entry, row;
    __device__ __forceinline__ void ask(const PagedArgs& a, const int32_t* table_row, int len, int j)
    {
        const int jj = j < len ? j : len - 1, pg = a.by_page.quotient(jj);
        row = jj - pg * a.page;
        entry = read_uniform_int(table_row + pg);
    }
    // 32 x 32 -> 64-bit products on the scalar unit (the host sees to it that strides fit)
    __device__ __forceinline__ const char* in(const PagedArgs& a, const char* head, uint32_t page_bytes, uint32_t row_bytes) const
    {
        const uint32_t e = (uint32_t)entry < (uint32_t)a.num_pages ? (uint32_t)entry : 0u;
        return head + (uint64_t)e * page_bytes + (uint64_t)(uint32_t)row * row_bytes;
    }
};

// rows of the work-group that see no key: O = 0, LSE = -inf, or the same as partial results
template <int BR, int kThreads>
__device__ __forceinline__ void paged_store_empty(const PagedArgs& a, const PagedItem& it, int tid)
{
    const int n = min(BR, it.rows - it.row0);
    for (int k = tid; k < n * 16; k += kThreads) {
        const int r = it.row0 + (k >> 4), c = k & 15;
        int head;
        const int tok = row_token(a, it, r, &head);
        const size_t row = (size_t)tok * a.H + head;
        if (a.num_splits > 1) {  // (a partial result of weight 0 is not read)
            if (c == 0) a.LSE_partial[row * a.num_splits + it.split] = -INFINITY;
        } else {
            const v4u z = {0u, 0u, 0u, 0u};
            if (c * 8 < a.d) *reinterpret_cast<v4u*>(a.O + (size_t)tok * a.o_token + (size_t)head * a.o_head + c * 16) = z;
            if (c == 0) a.LSE[row] = -INFINITY;
        }
    }
}

// ---------------------------------------------------------------------------------------------- tiles in LDS
//
// A stage holds BC keys row-major, D * 2 bytes each, with the 16-byte chunks of a row permuted so that the fragment reads are free of
// bank conflicts:
//   K: chunk c of key r in slot c ^ (r % 16) (256-byte rows) or c ^ (r / 2 % 8) (128-byte rows)
//   V: 32-byte chunk c in slot c ^ (2 (r % 4) + r / 4 % 2), or the two halves of a 128-byte row exchanged in rows 2, 3 mod 4
template <int D, int kKeys = 64>
struct PagedTile {
    static constexpr int BC = kKeys, KB = BC / 32, KS = D / 16, MB = D / 32, ROW = D * 2, BUF = BC * ROW;
    static constexpr int RPB = 1024 / ROW;   // rows of a request
    static constexpr int REQ = BUF / 1024;   // requests of a tile
    static constexpr int CPR = ROW / 16;     // chunks of a row
    static __device__ __forceinline__ int k_chunk(int slot, int r) { return D == 128 ? slot ^ (r & 15) : slot ^ ((r >> 1) & 7); }
    static __device__ __forceinline__ int v_chunk(int slot, int r)
    {
        return D == 128 ? ((((slot >> 1) ^ (2 * (r & 3) + ((r >> 2) & 1))) << 1) | (slot & 1)) : slot ^ (((r >> 1) & 1) << 2);
    }
    // lane part of a K fragment's address: key l32, chunk 2 ks + g -> k_lane ^ (ks << 5), + 32 ROW for the second 32 keys
    static __device__ __forceinline__ int k_lane(int lane)
    {
        const int l32 = lane & 31, g = lane >> 5, z = D == 128 ? l32 & 15 : (l32 >> 1) & 7;
        return l32 * ROW + ((g ^ (z & 1)) << 4) + ((z >> 1) << 5);
    }
    // of a V fragment's: keys 16 st + 8 h + 4 (lane / 32) + e, columns 32 mb + 16 (lane / 16 % 2) + 4 j ... + 3
    // -> v_lane ^ (mb << 6), + (16 st + 8 h) ROW
    static __device__ __forceinline__ int v_lane(int lane)
    {
        const int G = lane >> 4, e = (lane >> 2) & 3, j = lane & 3;
        if (D == 128) return (4 * (G >> 1) + e) * ROW + (((G & 1) ^ (G >> 1)) << 5) + 8 * j + (e << 6);
        return (4 * (G >> 1) + e) * ROW + ((G & 1) << 5) + 8 * j + ((e >> 1) << 6);
    }
};

__device__ __forceinline__ FA_LDS const char* lds_at(uint32_t addr) { return reinterpret_cast<FA_LDS const char*>(static_cast<uintptr_t>(addr)); }

// The sum of the register and the lane part, kept as one register (written out, the compiler keeps one per fragment).
__device__ __forceinline__ uint32_t fragment_base(FA_LDS const char* stage, int lane_part)
{
    uint32_t v = (uint32_t)(uintptr_t)stage + (uint32_t)lane_part;
    asm volatile("" : "+v"(v));
    return v;
}

template <int D>
__device__ __forceinline__ v8h v_fragment(uint32_t vbase, int st, int mb)
{
    FA_LDS const char* p0 = lds_at(vbase ^ (uint32_t)(mb << 6)) + st * 16 * PagedTile<D>::ROW;
    union { v4hp p[2]; v8h v; } f;
    f.p[0] = __builtin_amdgcn_ds_read_tr16_b64_v4f16((FA_LDS v4hp*)(p0));
    f.p[1] = __builtin_amdgcn_ds_read_tr16_b64_v4f16((FA_LDS v4hp*)(p0 + 8 * PagedTile<D>::ROW));
    return f.v;
}
template <int D>
__device__ __forceinline__ v8h k_fragment(uint32_t kbase, int ks, int kb)
{
    return *reinterpret_cast<FA_LDS const v8h*>(lds_at(kbase ^ (uint32_t)(ks << 5)) + kb * (32 * PagedTile<D>::ROW));
}

// Reads of LDS and MFMAs in turn, kAhead fragments (of kReads reads each) in front: left to itself the compiler waits for every fragment where it is used, 120
// cycles for an MFMA of 32.  Stands behind the code that it orders.
template <int kFragments, int kReads, int kAhead, bool kFirstAreThere = false>
__device__ __forceinline__ void order_reads_and_mfmas()
{
    constexpr int ahead = kAhead < kFragments ? kAhead : kFragments;
    if constexpr (!kFirstAreThere) __builtin_amdgcn_sched_group_barrier(0x100, kReads * ahead, 0);
#pragma unroll
    for (int x = 0; x < kFragments; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (x + ahead < kFragments) __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
    }
}

constexpr float kPagedTau = 8.0f;                       // powers of two by which a row may outgrow its running maximum
constexpr float kPagedNothing = -3.402823466e38f;       // running maximum of a row that has seen no key

// Online softmax of one tile of KB * 32 keys: scores in s (unscaled), P^T packed into p as the B operand of the second product.
// sides != 0: some row does not see all of the tile, but keys lo_rel ... hi_rel, counted from the tile's first plus the lane's 4 g
template <bool kBf16, int MB, int KB>
struct PagedSoftmax {
    float m_ref = kPagedNothing, m_thr = -INFINITY, l_run = 0.0f;
    // kOffset: all scores of the row are larger by `off`
    template <bool kOffset = false>
    __device__ __forceinline__ void tile(v16f (&s)[KB], v16f (&oacc)[MB], uint32_t (&p)[KB][2][4], float c2, float inv_c2, int sides, int lo_rel, int hi_rel, float off = 0.0f)
    {
        if (__builtin_expect(sides != 0, 0)) {
            if constexpr (KB == 2) {
                mask_tile<false>(s[0], s[1], wave_uniform(mask_modes_general(sides)), lo_rel, hi_rel, -INFINITY);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = 8 * (r >> 2) + (r & 3);
                    s[0][r] = key < lo_rel || key > hi_rel ? -INFINITY : s[0][r];
                }
            }
        }
        float mk[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) mk[kb] = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) mk[kb] = fmaxf(mk[kb], s[kb][r]);
        float mx = fmaxf(mk[0], mk[KB - 1]);
        if constexpr (kOffset) mx += off;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(mx > m_thr) != 0ull, 0)) {
            const float m_new = fmaxf(m_ref, xhalf_max(mx) * c2);  // c2 > 0
            float alpha = fast_exp2(m_ref - m_new);
            asm volatile("; raise running max" : "+v"(alpha));
            m_ref = m_new;
            m_thr = (m_new + kPagedTau) * inv_c2;
            l_run *= alpha;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int r = 0; r < 16; ++r) oacc[mb][r] *= alpha;
        }
        float rs = 0.0f, from = m_ref;
        if constexpr (kOffset) from = __builtin_fmaf(-off, c2, m_ref);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float p0 = fast_exp2(__builtin_fmaf(s[kb][r], c2, -from)), p1 = fast_exp2(__builtin_fmaf(s[kb][r + 1], c2, -from));
                rs = kb == 0 && r == 0 ? p0 + p1 : rs + p0 + p1;
                p[kb][r >> 3][(r & 7) >> 1] = Elem<kBf16>::pack(p0, p1);
            }
        l_run += rs;
    }
};

// ---------------------------------------------------------------------------------------------- scores and masks of other kinds
//
// A cap turns a score x into c tanh(x / c).  tanh(z) = 1 + 2 t with t = -1 / (1 + e^(2 z)), which grows with z from -1 to 0: the softmax goes by t in place
// of the product, in units of 2 c log2 e, and the constant c that is missing is added to the LSE.  That is a product, two transcendental
// instructions and a subtraction per score in front of the usual fma and exp2, 24 cycles of a SIMD beside the 24 that a plain score takes and the 32 of its
// MFMAs at d = 128.  t is off by at most 4.5 half steps of 2^-24 (the argument's two roundings and v_exp_f32, of which at most a quarter arrives, below 1.5; the
// subtraction 1; v_rcp_f32 2), a score by 9 c 2^-24, 16 c 2^-24 with what the softmax rounds behind it; a polynomial for small z that
// stays relative takes as many cycles (measured: v_exp_f32 and v_rcp_f32 8 cycles a wave, other instructions 4).
// A bias by distance, -slope |p - j|, begins as slope (j - p), which a product of its own and an offset of the tile work out; tiles with keys that stand
// otherwise and may be seen get the difference.  The sums of a score begin with slope (j - first of the tile), so that what they round grows with 64 |slope|.  Behind a cap it is added to t, one instruction per score.
// A tree's tokens see the keys in front of the chunk, and of the chunk's those whose bit is set; they stand at the chunk's begin plus their depth, the number
// of tokens that they see in the chunk less one.  The masks of the sequence's tokens and the depths lie in LDS; all they touch is the last tile or
// the last few of a sequence, which take a mask of 64 bits per row.

struct TreeTable {
    FA_LDS uint64_t* words;  // [kTreeTokens][tree_words]
    FA_LDS int* depth;       // [kTreeTokens]
    int tokens;              // of the sequence, that have a row here
};
constexpr int kTreeLds = kTreeTokens * (kTreeTokens / 64) * 8 + kTreeTokens * 4;

// Word w of the mask of the chunk's token i, of n: bits of tokens that there are not cleared
__device__ __forceinline__ uint64_t tree_word(const ScoredArgs& a, const PagedItem& it, int i, int w, int n)
{
    const int left = n - 64 * w;
    const uint64_t there = left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
    return a.tree[(int64_t)(it.tok0 + i) * a.tree_stride + w] & there;
}

// Called by all threads of a work-group whose keys reach the chunk's own, where there is a tree: behind the requests for its first tiles, so that what
// is loaded here is on its way together with them.  depths: whether they are asked for
template <int kThreads>
__device__ __forceinline__ void tree_setup(const ScoredArgs& a, const PagedItem& it, int tid, FA_LDS char* lds, bool depths, TreeTable* tree)
{
    const int W = a.tree_words, n = min(it.len - it.shift, 64 * W);
    tree->words = (FA_LDS uint64_t*)lds;
    tree->depth = (FA_LDS int*)(lds + kTreeTokens * (kTreeTokens / 64) * 8);
    tree->tokens = n;
    for (int k = tid; k < n * W; k += kThreads) {
        const int i = (int)((uint32_t)k / (uint32_t)W);
        tree->words[k] = tree_word(a, it, i, k - i * W, n);
    }
    __syncthreads();
    if (!depths) return;
    for (int i = tid; i < n; i += kThreads) {
        int c = -1;
        for (int w = 0; w < W; ++w) c += __builtin_popcountll(tree->words[i * W + w]);
        tree->depth[i] = max(c, 0);
    }
    __syncthreads();
}

// Keys lo ... hi of the 64 that a tile begins with, counted from its first
__device__ __forceinline__ uint64_t range_bits(int lo, int hi)
{
    const uint64_t below = hi < 0 ? 0ull : hi >= 63 ? ~0ull : (2ull << hi) - 1;
    return below & (lo <= 0 ? ~0ull : lo > 63 ? 0ull : ~0ull << lo);
}

// What a lane knows of its row, and its wave of its rows
template <int kScores>
struct RowScores {
    TreeTable tree = {nullptr, nullptr, 0};  // (none: keys in front of the chunk alone)
    int token, base;      // its index in the chunk; the chunk's first key
    int kmin, kmax;       // keys of the work-group
    int place;            // position
    int bent;             // first key whose bias may not be slope (key - place)
    float slope;

    // keys [lo, hi] that row r sees, but for the chunk's own of a tree, whose table must be there where the work-group's keys reach them
    __device__ __forceinline__ void set(const ScoredArgs& a, const PagedItem& it, int r, int kmin_, int kmax_, int* lo, int* hi)
    {
        const int rr = r < it.rows ? r : it.rows - 1, i = a.by_group.quotient(rr);
        kmin = kmin_, kmax = kmax_, base = it.shift, token = i;
        place = i + it.shift;
        int l = kmin, h = kmax - 1;
        if (a.tree) {
            place = base;
            const int n = min(it.len - it.shift, 64 * a.tree_words);
            if ((has_slopes(kScores) || a.wl >= 0) && i < n) {
                int c = -1;
                for (int w = 0; w < a.tree_words; ++w) c += __builtin_popcountll(tree_word(a, it, i, w, n));
                place += max(c, 0);
            }
            h = min(h, base - 1);
        }
        if (a.wl >= 0) l = max(l, place - a.wl);
        if (a.causal) h = min(h, place);
        if (a.wr >= 0) h = min(h, place + a.wr);
        if (a.prefix) h = max(h, min(prefix_of(a, it.b), kmax) - 1);
        *lo = l;
        *hi = h;
        if constexpr (has_slopes(kScores)) {
            slope = a.slopes[it.hk * a.G + (rr - i * a.G)] * a.slope_unit;
            if constexpr (!has_cap(kScores)) set_slant(threadIdx.x & 31, (threadIdx.x & 63) >> 5);
            bent = a.tree ? base : a.causal && !a.prefix ? 0x7fffffff : __builtin_amdgcn_readfirstlane(place) + 1;  // (under a causal mask alone nobody sees one)
        }
    }
    // the chunk's own keys among the 64 from kb0 on that the row sees
    __device__ __forceinline__ uint64_t drafted_bits(const ScoredArgs& a, int kb0) const
    {
        if (token >= tree.tokens) return 0;
        const int o = kb0 - base, W = a.tree_words, w = o >> 6, sh = o & 63;
        const FA_LDS uint64_t* const row = tree.words + token * W;
        const uint64_t w0 = w >= 0 && w < W ? row[w] : 0ull, w1 = w + 1 >= 0 && w + 1 < W ? row[w + 1] : 0ull;
        return ((w0 >> sh) | (sh ? w1 << (64 - sh) : 0ull)) & range_bits(kmin - kb0, kmax - 1 - kb0);
    }
    __device__ __forceinline__ bool sees(const ScoredArgs& a, int j, int lo, int hi) const
    {
        return (j >= lo && j <= hi) || (a.tree && j >= base && (drafted_bits(a, j) & 1));
    }
    __device__ __forceinline__ float distance(const ScoredArgs& a, int j) const
    {
        int at = j;
        if (a.tree && j >= base) at = base + (j - base < tree.tokens ? tree.depth[j - base] : 0);
        return (float)(at - place);
    }
    // Bias of keys in front of the row, slope (key - place): the tile's part, slope (kb0 - place), is the softmax's offset; what the keys' places in the tile
    // add comes out of a product of its own, 16 columns of which three are used: the slope in three parts of eight bits (bf16, whatever the caches hold)
    // times the place, 0 ... 63, which is exact.  One MFMA per 32 keys, 32 cycles, where sixteen additions per lane would take 64 of the softmax's.
    v8h q_slant, k_slant[2];
    __device__ __forceinline__ void set_slant(int l32, int g)
    {
        const float hi = Elem<true>::low(Elem<true>::pack(slope, slope)), mid = Elem<true>::low(Elem<true>::pack(slope - hi, slope - hi)), lo = slope - hi - mid;
        const float on = g == 0 ? 1.0f : 0.0f;
        const uint32_t q[4] = {Elem<true>::pack(hi * on, mid * on), Elem<true>::pack(lo * on, 0.0f), 0u, 0u};
        q_slant = fragment_of(q);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const float key = (float)(l32 + 32 * kb) * on;
            const uint32_t k[4] = {Elem<true>::pack(key, key), Elem<true>::pack(key, 0.0f), 0u, 0u};
            k_slant[kb] = fragment_of(k);
        }
    }
    __device__ __forceinline__ v16f slant(int kb) const
    {
        const v16f z = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        return Elem<true>::mfma(k_slant[kb], q_slant, z);
    }
    static __device__ __forceinline__ v8h fragment_of(const uint32_t (&p)[4])
    {
        const v4u t = {p[0], p[1], p[2], p[3]};
        return __builtin_bit_cast(v8h, t);
    }
    // (behind a cap the two halves of the lanes, whose keys are 4 apart, have offsets of their own: the larger score of a row is looked for with them)
    __device__ __forceinline__ float offset(int kb0, int g) const
    {
        return !has_slopes(kScores) ? 0.0f : has_cap(kScores) ? slope * (float)(kb0 + 4 * g - place) : slope * (float)(kb0 - place);
    }
    // ... and what makes it that of the others, as far as a row may see them: keys behind it, and a tree's, which stand at their depths
    template <int KB>
    __device__ __forceinline__ void bend(const ScoredArgs& a, v16f (&s)[KB], int kb0, int g) const
    {
        const int k0 = kb0 + 4 * g;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = k0 + 32 * kb + 8 * (r >> 2) + (r & 3);
                s[kb][r] -= slope * (__builtin_fabsf(distance(a, key)) + (float)(key - place));  // (0 for the others)
                asm volatile("" : "+v"(s[kb][r]));  // (one after the other: 32 distances at once do not fit in the registers)
            }
    }
    // t of a product
    __device__ __forceinline__ float capped(const ScoredArgs& a, float s) const { return __builtin_amdgcn_rcpf(-1.0f - fast_exp2(s * a.cap_in)); }
    // From products to what the softmax goes by, masks applied.  sides: as in PagedSoftmax::tile
    template <int KB>
    __device__ __forceinline__ void finish(const ScoredArgs& a, v16f (&s)[KB], int kb0, int g, int sides, int lo, int hi) const
    {
        if constexpr (has_cap(kScores)) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kb][r] = capped(a, s[kb][r]);
            if constexpr (has_slopes(kScores)) {  // (to t, and the lane's 4 g)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kb][r] = __builtin_fmaf(slope, (float)(32 * kb + 8 * (r >> 2) + (r & 3)), s[kb][r]);
            }
        }
        if (has_slopes(kScores) && __builtin_expect(kb0 + 32 * KB > bent, 0)) bend(read_again(a), s, kb0, g);
        if (__builtin_expect(sides != 0, 0)) {
            const ScoredArgs& again = read_again(a);
            if (again.tree) {
                const uint64_t seen = (range_bits(lo - kb0, hi - kb0) | drafted_bits(again, kb0)) >> (4 * g);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const uint32_t bits = (uint32_t)(seen >> (32 * kb));
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kb][r] = bits >> (8 * (r >> 2) + (r & 3)) & 1 ? s[kb][r] : -INFINITY;
                }
            } else if constexpr (KB == 2) {
                mask_tile<false>(s[0], s[1], wave_uniform(mask_modes_general(sides)), lo - kb0 - 4 * g, hi - kb0 - 4 * g, -INFINITY);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = kb0 + 4 * g + 8 * (r >> 2) + (r & 3);
                    s[0][r] = key < lo || key > hi ? -INFINITY : s[0][r];
                }
            }
        }
    }
    // The same of one key's product, unmasked
    __device__ __forceinline__ float one(const ScoredArgs& a, float s, int j) const
    {
        if constexpr (has_cap(kScores)) s = capped(a, s);
        if constexpr (has_slopes(kScores)) s -= slope * __builtin_fabsf(distance(a, j));
        return s;
    }
};
template <>
struct RowScores<kScoresPlain> {};

template <int kScores>
__device__ __forceinline__ float lse_of(const ArgsOf<kScores>& a, float m, float l)
{
    const float lse = __builtin_fmaf(m, kLn2, fast_log2(l) * kLn2);
    if constexpr (has_cap(kScores)) return lse + a.cap;
    else return lse;
}

// of a wave's 32 rows (lanes 0 ... 31 and again 32 ... 63)
__device__ __forceinline__ int rows_min(int v)
{
#pragma unroll
    for (int m = 1; m < 32; m *= 2) v = min(v, __shfl_xor(v, m));
    return wave_uniform(v);
}

__device__ __forceinline__ v8h as_fragment(const uint32_t (&p)[4])
{
    const v4u t = {p[0], p[1], p[2], p[3]};
    return __builtin_bit_cast(v8h, t);
}

// Q fragments (B operand): lane holds row r's columns 16 ks + 8 g ... + 7; zeroes past d
template <int KS>
__device__ __forceinline__ void load_q(const PagedArgs& a, const PagedItem& it, int r, int g, v8h (&qf)[KS])
{
    int head;
    const int tok = row_token(a, it, r < it.rows ? r : it.rows - 1, &head);
    const char* const q = a.Q + (size_t)tok * a.q_token + (size_t)head * a.q_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int c = 16 * ks + 8 * g;
        v4u v = *reinterpret_cast<const v4u*>(q + 2 * (c < a.d ? c : 0));
        const v4u z = {0u, 0u, 0u, 0u};
        v = c < a.d ? v : z;
        qf[ks] = __builtin_bit_cast(v8h, v);
    }
}

// A masked probability is 0, and 0 times a V that is not finite is not: such a product has spoilt the row's sum if V has one in a tile of
// which the row sees a part, or none.  Called once per wave, behind its loop, where some sum is not finite: looks for such
// values among the wave's partly masked tiles and, if there are any, works out the rows in question once more key by key, visible
// keys alone.  (Tiles first, first + step, ... of the range from key kb_first on.)
template <int BC, int MB, bool kBf16, int kScores>
__device__ __forceinline__ void paged_rescue(const ArgsOf<kScores>& a, const PagedItem& it, int r, int kmin, int kmax, int tile0, int ntiles, int first,
                                                       int step, float m_ref, v16f (&oacc)[MB], RowScores<kScores>& row)
{
    const int lane = threadIdx.x & 63, g = lane >> 5;
    const int32_t* const table_row = a.table + (size_t)it.b * a.table_stride;
    int lo, hi;
    if constexpr (kScores == kScoresPlain) paged_bounds(a, it, r, kmin, kmax, &lo, &hi);
    else row.set(a, it, r, kmin, kmax, &lo, &hi);
    auto row_of = [&](const char* base, uint32_t page_bytes, int64_t head_bytes, uint32_t row_bytes, int j) {
        const int pg = a.by_page.quotient(j);
        const PagedPlace at = {table_row[pg], j - pg * a.page};
        return at.in(a, base + it.hk * head_bytes, page_bytes, row_bytes);
    };
    // lane j: key j of the tile; masked for some row of the wave, and not finite somewhere?
    bool spoilt = false;
    for (int t = first; t < ntiles; t += step) {
        const int kb0 = (tile0 + t) * BC, j = kb0 + (lane & (BC - 1));
        bool some = false;  // of the lanes' rows does one not see key j?  (the key is told to all rows in turn)
        for (int q = 0; q < 32; ++q) {
            const int l = __builtin_amdgcn_readlane(lo, q), h = __builtin_amdgcn_readlane(hi, q);
            some |= j < l || j > h;  // (of a tree's own tokens all are looked at)
        }
        if (some && j < it.len) {
            const char* const v = row_of(a.V, a.v_page, a.v_head, a.v_row, j);
            for (int c = 0; c < a.d; c += 2) spoilt |= Elem<kBf16>::not_finite(*reinterpret_cast<const uint32_t*>(v + 2 * c));
        }
    }
    if (__builtin_amdgcn_ballot_w64(spoilt) == 0) return;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[mb][e] = 0.0f;
    int head;
    const int tok = row_token(a, it, r < it.rows ? r : it.rows - 1, &head);
    const char* const q = a.Q + (size_t)tok * a.q_token + (size_t)head * a.q_head;
    for (int t = first; t < ntiles; t += step) {
        const int kb0 = (tile0 + t) * BC;
        int j0 = max(kb0, lo), j1 = min(kb0 + BC - 1, hi);
        if constexpr (kScores != kScoresPlain)
            if (a.tree) j0 = max(kb0, kmin), j1 = min(kb0 + BC, kmax) - 1;
        for (int j = j0; j <= j1; ++j) {
            if constexpr (kScores != kScoresPlain)
                if (!row.sees(a, j, lo, hi)) continue;
            const char* const k = row_of(a.K, a.k_page, a.k_head, a.k_row, j);
            const char* const v = row_of(a.V, a.v_page, a.v_head, a.v_row, j);
            float s = 0.0f;
            for (int c = 0; c < a.d; c += 2) {
                const uint32_t x = *reinterpret_cast<const uint32_t*>(q + 2 * c), y = *reinterpret_cast<const uint32_t*>(k + 2 * c);
                s = __builtin_fmaf(Elem<kBf16>::low(x), Elem<kBf16>::low(y), s);
                s = __builtin_fmaf(Elem<kBf16>::high(x), Elem<kBf16>::high(y), s);
            }
            if constexpr (kScores != kScoresPlain) s = row.one(a, s, j);
            const float e = fast_exp2(__builtin_fmaf(s, a.scale_log2, -m_ref)), p = Elem<kBf16>::low(Elem<kBf16>::pack(e, e));
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int rg = 0; rg < 4; ++rg) {
                    const int c = 32 * mb + 8 * rg + 4 * g;
                    if (c < a.d) {
                        const v2u w = *reinterpret_cast<const v2u*>(v + 2 * c);
                        oacc[mb][4 * rg] = __builtin_fmaf(p, Elem<kBf16>::low(w[0]), oacc[mb][4 * rg]);
                        oacc[mb][4 * rg + 1] = __builtin_fmaf(p, Elem<kBf16>::high(w[0]), oacc[mb][4 * rg + 1]);
                        oacc[mb][4 * rg + 2] = __builtin_fmaf(p, Elem<kBf16>::low(w[1]), oacc[mb][4 * rg + 2]);
                        oacc[mb][4 * rg + 3] = __builtin_fmaf(p, Elem<kBf16>::high(w[1]), oacc[mb][4 * rg + 3]);
                    }
                }
        }
    }
}

template <int MB>
__device__ __forceinline__ bool any_not_finite(const v16f (&oacc)[MB])
{
    float z = 0.0f;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) z = __builtin_fmaf(oacc[mb][r], 0.0f, z);
    return __builtin_amdgcn_ballot_w64(!(z == 0.0f)) != 0ull;
}

// One KiB into LDS from an address of each lane's own (dma_kib and dma_kib_nt in common.h).
template <bool kNt>
__device__ __forceinline__ void dma_kib_lanes(const char* at, FA_LDS char* lds_dst)
{
    const uint32_t m0v = (uint32_t)(uintptr_t)lds_dst;
    if constexpr (kNt) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" : : "s"(m0v), "v"(at) : "memory", "m0");
    else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(m0v), "v"(at) : "memory", "m0");
}

// ---------------------------------------------------------------------------------------------- few rows

// Where rows of V past a sequence's end come from.  (Rows that repeat the last key's and are looked over in LDS, as in the 256-row form, cost 0.3-1 us more at
// the end of these short work-groups: 58 single tokens H64 H_kv16 d80 11.4 us with rows that nobody clears, 11.5 so, 12.5 looked over.)
static __device__ const v4u kPagedZeroes = {0u, 0u, 0u, 0u};

// A wave has one stage of 8 KiB for K and for V each: tiles of 32 keys (256-byte rows) or 64.  K of the next tile is requested as soon as the scores
// of this one have read theirs, V behind the second product; requests are non-temporal, since nobody else asks for the keys.  With 64 to
// 68 KiB per work-group two share a CU: one streams while the other begins, merges or ends.  Tiles of 64 keys at d = 128, two stages at
// d = 64, one work-group per CU -> so: single tokens B64 H32 H_kv8 up to 500 keys 24.2 -> 15.0 us, up to 16384 391 -> 375 (unsplit), B64 H16 d64
// 2000 keys 89.8 -> 79.7 (6.6 TB/s), B1 H32 H_kv8 32000 in 32 splits 27.9 -> 26.7.
template <int D>
struct FewCfg {
    static constexpr int kWaves = 4, BC = D == 128 ? 32 : 64;
    static constexpr int WAVE = 2 * PagedTile<D, BC>::BUF;    // LDS of a wave's stages
    static constexpr int OROW = D + 4;                        // floats of a row of partial O
    static constexpr int MERGE = kWaves * (32 * OROW + 64) * 4;
    static constexpr int SMEM = kWaves * WAVE > MERGE ? kWaves * WAVE : MERGE;
    static_assert(2 * SMEM <= 160 * 1024, "two work-groups per CU");
};

template <int D, bool kBf16, int kScores>
__device__ __forceinline__ void few_rows(const ArgsOf<kScores> a)
{
    using C = FewCfg<D>;
    constexpr int BC = C::BC;
    using T = PagedTile<D, BC>;
    constexpr int KS = T::KS, MB = T::MB, KB = T::KB, REQ = T::REQ, GROUPS = BC / 16;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6), l32 = lane & 31, g = lane >> 5;

    PagedItem it;
    if (!paged_item<kPagedFewRows, ArgsOf<kScores>>(a, lane, &it)) return;
    paged_mark_missing<kPagedFewRows, 256>(a, it, tid);
    int kmin, kmax;
    paged_range<kPagedFewRows>(a, it, &kmin, &kmax);
    if (kmax <= kmin) {
        paged_store_empty<kPagedFewRows, 256>(a, it, tid);
        return;
    }
    const int tile0 = kmin / BC, ntiles = (kmax + BC - 1) / BC - tile0;
    const int len = it.len;
    RowScores<kScores> row;
    const int32_t* const table_row = a.table + (size_t)it.b * a.table_stride;

    FA_LDS char* const kst = (FA_LDS char*)smem + wave * C::WAVE;
    FA_LDS char* const vst = kst + T::BUF;
    if (a.d != D) {  // columns that no request writes
        const v4u z = {0u, 0u, 0u, 0u};
        for (int k = lane; k < C::WAVE / 16; k += 64) *reinterpret_cast<FA_LDS v4u*>(kst + 16 * k) = z;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }

    // ---- requests: request x of a tile covers its rows RPB x ... ; one table entry for each 16 keys
    const int lrow = lane / T::CPR, slot = lane % T::CPR;
    constexpr int kPer = REQ / GROUPS;  // requests per 16 keys
    uint32_t koff[kPer], voff[kPer];
    bool kok[kPer], vok[kPer];
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
        const int r = T::RPB * x + lrow, ck = T::k_chunk(slot, r), cv = T::v_chunk(slot, r);
        koff[x] = (uint32_t)r * a.k_row + ck * 16;
        voff[x] = (uint32_t)r * a.v_row + cv * 16;
        kok[x] = ck * 8 < a.d;
        vok[x] = cv * 8 < a.d;
    }
    const char* const Kh = a.K + it.hk * a.k_head;
    const char* const Vh = a.V + it.hk * a.v_head;
    PagedPlace place[GROUPS];  // of the tile to request next
    auto ask = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < GROUPS; ++s) place[s].ask(a, table_row, len, (tile0 + tile_of<kScores>(t, ntiles)) * BC + 16 * s);
    };
    // the rows of tile t (its places asked for) of K or V
    auto request = [&](auto is_v_c, int t, const char* head, uint32_t page_bytes, uint32_t row_bytes, const uint32_t (&off)[kPer], const bool (&ok)[kPer],
                       FA_LDS char* dst) __attribute__((always_inline)) {
        constexpr bool kIsV = decltype(is_v_c)::value;
        const int kb0 = (tile0 + tile_of<kScores>(t, ntiles)) * BC;
        const bool whole = kb0 + BC <= len;
        if constexpr (kScores != kScoresPlain) {
            if (__builtin_expect(whole && a.d == D, 1)) {  // (nearly all tiles, and nearly all others: no branch per request)
#pragma unroll
                for (int s = 0; s < GROUPS; ++s) {
                    const char* const at = place[s].in(a, head, page_bytes, row_bytes);
#pragma unroll
                    for (int x = 0; x < kPer; ++x) dma_kib_nt(at, off[x], dst + (s * kPer + x) * 1024);
                }
                return;
            }
            if (__builtin_expect(a.d == D, 1)) {
#pragma unroll
                for (int s = 0; s < GROUPS; ++s) {
                    const char* const at = place[s].in(a, head, page_bytes, row_bytes);
#pragma unroll
                    for (int x = 0; x < kPer; ++x) {
                        const int r = T::RPB * x + lrow, past = r - (len - 1 - (kb0 + 16 * s));
                        if constexpr (kIsV) dma_kib_lanes<true>(past <= 0 ? at + off[x] : reinterpret_cast<const char*>(&kPagedZeroes), dst + (s * kPer + x) * 1024);
                        else dma_kib_nt(at, off[x] - (uint32_t)min(max(past, 0), r) * row_bytes, dst + (s * kPer + x) * 1024);
                    }
                }
                return;
            }
        }
#pragma unroll
        for (int s = 0; s < GROUPS; ++s) {
            const char* const at = place[s].in(a, head, page_bytes, row_bytes);
#pragma unroll
            for (int x = 0; x < kPer; ++x) {
                uint32_t o = off[x];
                if (!whole) {  // rows past the last key: of K they repeat it, of V they are zeroes
                    const int r = T::RPB * x + lrow, most = max(len - 1 - (kb0 + 16 * s), 0);
                    if constexpr (kIsV) {
                        const char* const from = kb0 + 16 * s + r < len ? at + o : reinterpret_cast<const char*>(&kPagedZeroes);
                        if (ok[x]) dma_kib_lanes<true>(from, dst + (s * kPer + x) * 1024);
                        continue;
                    }
                    if (r > most) o -= (uint32_t)(r - most) * row_bytes;
                }
                if (ok[x]) dma_kib_nt(at, o, dst + (s * kPer + x) * 1024);
            }
        }
    };
    auto request_k = [&](int t) { request(std::false_type{}, t, Kh, a.k_page, a.k_row, koff, kok, kst); };
    auto request_v = [&](int t) { request(std::true_type{}, t, Vh, a.v_page, a.v_row, voff, vok, vst); };

    const int r = it.row0 + l32;
    v8h qf[KS];
    v16f oacc[MB];
    PagedSoftmax<kBf16, MB, KB> soft;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[mb][e] = 0.0f;

    int lo, hi;
    if constexpr (kScores == kScoresPlain) paged_bounds(a, it, r, kmin, kmax, &lo, &hi);
    else lo = hi = 0;
    int lo_max = lo, hi_min = hi;
    if (wave < ntiles) {
        ask(wave);
        load_q<KS>(a, it, r, g, qf);
        request_k(wave);
        request_v(wave);
        if constexpr (kScores == kScoresPlain) {
            lo_max = __builtin_amdgcn_readlane(lo, 31);  // (bounds do not fall from row to row)
            hi_min = __builtin_amdgcn_readlane(hi, 0);
        }
    }
    if constexpr (kScores != kScoresPlain) {
        const ScoredArgs& again = read_again(a);
        if (again.tree && kmax > it.shift) tree_setup<256>(again, it, tid, (FA_LDS char*)smem + C::SMEM, has_slopes(kScores), &row.tree);
        row.set(again, it, r, kmin, kmax, &lo, &hi);
        lo_max = again.tree ? -rows_min(-lo) : __builtin_amdgcn_readlane(lo, 31);  // (a tree's bounds may fall)
        hi_min = __builtin_amdgcn_readlane(hi, 0);
    }
    const float c2 = a.scale_log2, inv_c2 = __builtin_amdgcn_rcpf(c2);
    const int k_rd = T::k_lane(lane), v_rd = T::v_lane(lane);
    for (int t = wave; t < ntiles; t += 4) {
        const int kb0 = (tile0 + tile_of<kScores>(t, ntiles)) * BC;
        const bool more = t + 4 < ntiles;
        if (more) ask(t + 4);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(REQ) : "memory");  // K of this tile is there
        if (t == wave) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
        }
        v16f s[KB];
        {
            const uint32_t kbase = fragment_base(kst, k_rd);
            const v16f z = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
            if constexpr (kScores == kScoresSloped) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) s[kb] = row.slant(kb);
            }
            if constexpr (kScores != kScoresPlain) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
                    s[kb] = Elem<kBf16>::mfma(k_fragment<D>(kbase, ks, kb), qf[ks], ks == 0 && kScores != kScoresSloped ? z : s[kb]);
            if constexpr (kScores != kScoresPlain) order_reads_and_mfmas<KS * KB, 1, 6>();
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the fragments have been read
        if (more) request_k(t + 4);
        uint32_t p[KB][2][4];
        const int sides = is_negative(kb0 - lo_max) | is_negative(hi_min - (BC - 1) - kb0) << 1;
        if constexpr (kScores == kScoresPlain) {
            soft.tile(s, oacc, p, c2, inv_c2, sides, lo - kb0 - 4 * g, hi - kb0 - 4 * g);
        } else {
            row.finish(a, s, kb0, g, sides, lo, hi);
            soft.template tile<has_slopes(kScores)>(s, oacc, p, c2, inv_c2, 0, 0, 0, row.offset(kb0, g));
        }
        if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(REQ) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        {
            const uint32_t vbase = fragment_base(vst, v_rd);
            if constexpr (kScores != kScoresPlain) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int st = 0; st < 2 * KB; ++st)
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) oacc[mb] = Elem<kBf16>::mfma(v_fragment<D>(vbase, st, mb), as_fragment(p[st >> 1][st & 1]), oacc[mb]);
            if constexpr (kScores != kScoresPlain) order_reads_and_mfmas<2 * KB * MB, 2, 4>();
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) request_v(t + 4);
    }
    if (wave < ntiles && __builtin_expect(any_not_finite<MB>(oacc), 0))
        paged_rescue<BC, MB, kBf16, kScores>(read_again(a), it, r, kmin, kmax, tile0, ntiles, last_first(kScores) ? (ntiles - 1 - wave) & 3 : wave, 4, soft.m_ref, oacc, row);

    // ---- merge of the four waves: reference of a row = the largest of theirs
    const int nrows = min(kPagedFewRows, it.rows - it.row0);
    FA_LDS float* const xo = (FA_LDS float*)smem;                       // [4][32][OROW]
    FA_LDS float* const xm = xo + 4 * 32 * C::OROW;                     // [4][32] reference, then [4][32] sum
    __syncthreads();  // every wave is done with its stages
    {
        const float l = xhalf_sum(soft.l_run);
        if (l32 < nrows) {
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int rg = 0; rg < 4; ++rg) {
                    const v4f o = {oacc[mb][4 * rg], oacc[mb][4 * rg + 1], oacc[mb][4 * rg + 2], oacc[mb][4 * rg + 3]};
                    *reinterpret_cast<FA_LDS v4f*>(xo + (wave * 32 + l32) * C::OROW + 32 * mb + 8 * rg + 4 * g) = o;
                }
            if (g == 0) {
                xm[wave * 32 + l32] = soft.m_ref;
                xm[128 + wave * 32 + l32] = l;
            }
        }
    }
    __syncthreads();
    constexpr int CO = D / 8;  // eight columns per thread
    const ArgsOf<kScores>& end = read_again(a);
    for (int k = tid; k < nrows * CO; k += 256) {
        const int row = k / CO, c = (k % CO) * 8;
        float m = xm[row];
#pragma unroll
        for (int w = 1; w < 4; ++w) m = fmaxf(m, xm[w * 32 + row]);
        float l = 0.0f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float lw = xm[128 + w * 32 + row], f = lw == 0.0f ? 0.0f : fast_exp2(xm[w * 32 + row] - m);
            l += f * lw;
            const FA_LDS float* const src = xo + (w * 32 + row) * C::OROW + c;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __builtin_fmaf(f, src[e], o[e]);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const float lse = l == 0.0f ? -INFINITY : lse_of<kScores>(end, m, l);
        int head;
        const int tok = row_token(end, it, it.row0 + row, &head);
        const size_t at = (size_t)tok * end.H + head;
        if (c >= end.d) continue;
        if (end.num_splits > 1) {
            const size_t part = at * end.num_splits + it.split;
            float* const op = end.O_partial + part * end.d + c;
            const v4f o0 = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv}, o1 = {o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv};
            *reinterpret_cast<v4f*>(op) = o0;
            *reinterpret_cast<v4f*>(op + 4) = o1;
            if (c == 0) end.LSE_partial[part] = lse;
        } else {
            const v4u w = {Elem<kBf16>::pack(o[0] * inv, o[1] * inv), Elem<kBf16>::pack(o[2] * inv, o[3] * inv),
                           Elem<kBf16>::pack(o[4] * inv, o[5] * inv), Elem<kBf16>::pack(o[6] * inv, o[7] * inv)};
            *reinterpret_cast<v4u*>(end.O + (size_t)tok * end.o_token + (size_t)head * end.o_head + c * 2) = w;
            if (c == 0) end.LSE[at] = lse;
        }
    }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(256, 2) paged_few_kernel(const PagedArgs a)
{
    few_rows<D, kBf16, kScoresPlain>(a);
}
template <int D, bool kBf16, int kScores>
__global__ void __launch_bounds__(256, 2) scored_few_kernel(const ScoredArgs a)
{
    few_rows<D, kBf16, kScores>(a);
}

// ---------------------------------------------------------------------------------------------- tiles that waves share

// What one of kWaves waves requests of the work-group's tiles: KiB blocks wave, wave + kWaves, ... of each.
template <int D, int kWaves>
struct PagedRequests {
    using T = PagedTile<D>;
    static constexpr int NL = T::REQ / kWaves, STEP = T::RPB * kWaves;  // blocks, and rows from one to the next
    static_assert(STEP % 16 == 0, "the permutations of the chunks repeat");
    const int32_t* table_row;
    const char *Kh, *Vh;
    int len, tile0, wave, brow, lrow;
    uint32_t koff, voff;
    bool kok, vok;
    PagedPlace place[NL];   // of the tile of K to request next
    const char* vnext[NL];  // rows of the tile of V to request next: where K's were

    __device__ __forceinline__ void set(const PagedArgs& a, const PagedItem& it, int first_tile, int wave_, int lane)
    {
        table_row = a.table + (size_t)it.b * a.table_stride;
        Kh = a.K + it.hk * a.k_head;
        Vh = a.V + it.hk * a.v_head;
        len = it.len, tile0 = first_tile, wave = wave_;
        lrow = lane / T::CPR;
        brow = T::RPB * wave;
        const int slot = lane % T::CPR, ck = T::k_chunk(slot, brow + lrow), cv = T::v_chunk(slot, brow + lrow);
        koff = (uint32_t)lrow * a.k_row + ck * 16, voff = (uint32_t)lrow * a.v_row + cv * 16;
        kok = ck * 8 < a.d, vok = cv * 8 < a.d;
    }
    __device__ __forceinline__ void ask(const PagedArgs& a, int t)
    {
#pragma unroll
        for (int x = 0; x < NL; ++x) place[x].ask(a, table_row, len, (tile0 + t) * T::BC + brow + STEP * x);
    }
    __device__ __forceinline__ void request(int t, int x, const char* at, uint32_t row_bytes, uint32_t off, bool ok, FA_LDS char* stage) const
    {
        const int kb0 = (tile0 + t) * T::BC;
        uint32_t o = off;
        if (kb0 + T::BC > len) {  // rows past the last key repeat it
            const int most = max(len - 1 - (kb0 + brow + STEP * x), 0);
            if (lrow > most) o -= (uint32_t)(lrow - most) * row_bytes;
        }
        if (ok) dma_kib(at, o, stage + (wave + kWaves * x) * 1024);
    }
    __device__ __forceinline__ void load_k(const PagedArgs& a, int t, FA_LDS char* stage) const
    {
#pragma unroll
        for (int x = 0; x < NL; ++x) request(t, x, place[x].in(a, Kh, a.k_page, a.k_row), a.k_row, koff, kok, stage);
    }
    // Tile t of K and V, branches once for all requests: tiles that are not the last, rows without a gap behind them
    __device__ __forceinline__ void load(const PagedArgs& a, int t, FA_LDS char* k_stage, FA_LDS char* v_stage)
    {
        if (__builtin_expect((tile0 + t + 1) * T::BC <= len && a.d == D, 1)) {
#pragma unroll
            for (int x = 0; x < NL; ++x) dma_kib(place[x].in(a, Kh, a.k_page, a.k_row), koff, k_stage + (wave + kWaves * x) * 1024);
#pragma unroll
            for (int x = 0; x < NL; ++x) dma_kib(place[x].in(a, Vh, a.v_page, a.v_row), voff, v_stage + (wave + kWaves * x) * 1024);
        } else {
            load_k(a, t, k_stage);
            find_v(a);
            load_v(a, t, v_stage);
        }
    }
    __device__ __forceinline__ void find_v(const PagedArgs& a)
    {
#pragma unroll
        for (int x = 0; x < NL; ++x) vnext[x] = place[x].in(a, Vh, a.v_page, a.v_row);
    }
    __device__ __forceinline__ void load_v(const PagedArgs& a, int t, FA_LDS char* stage) const
    {
#pragma unroll
        for (int x = 0; x < NL; ++x) request(t, x, vnext[x], a.v_row, voff, vok, stage);
    }
};

// LDS-only barrier: requests in flight are not waited for, and nothing moves across.
__device__ __forceinline__ void paged_barrier()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// The same with the last kReads reads of LDS left in flight.
template <int kReads>
__device__ __forceinline__ void paged_barrier_keep()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(%0)\n\ts_barrier" ::"n"(kReads < 15 ? kReads : 15) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Results of a wave's 32 rows from first_row on (r: the lane's).  `ost`: LDS of the wave's own, 32 rows of D columns.
template <int D, int MB, bool kBf16, int kScores>
__device__ __forceinline__ void paged_store_rows(const ArgsOf<kScores>& a, const PagedItem& it, int first_row, int r, int lane, int g, float m_ref, float l_run,
                                                 const v16f (&oacc)[MB], FA_LDS char* ost)
{
    using T = PagedTile<D>;
    using E = Elem<kBf16>;
    const int l32 = lane & 31;
    const float l = xhalf_sum(l_run);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float lse = l == 0.0f ? -INFINITY : lse_of<kScores>(a, m_ref, l);
    int head;
    const int tok = row_token(a, it, r < it.rows ? r : it.rows - 1, &head);
    const size_t at = (size_t)tok * a.H + head;
    if (a.num_splits > 1) {
        if (r < it.rows) {
            const size_t part = at * a.num_splits + it.split;
            if (g == 0) a.LSE_partial[part] = lse;
            float* const op = a.O_partial + part * a.d;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int rg = 0; rg < 4; ++rg) {
                    const int c = 32 * mb + 8 * rg + 4 * g;
                    const v4f o = {oacc[mb][4 * rg] * inv, oacc[mb][4 * rg + 1] * inv, oacc[mb][4 * rg + 2] * inv, oacc[mb][4 * rg + 3] * inv};
                    if (c < a.d) *reinterpret_cast<v4f*>(op + c) = o;
                }
        }
        return;
    }
    if (r < it.rows && g == 0) a.LSE[at] = lse;
    // O^T is turned round in LDS and leaves as whole rows
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int rg = 0; rg < 4; ++rg) {
            const v2u w = {E::pack(oacc[mb][4 * rg] * inv, oacc[mb][4 * rg + 1] * inv), E::pack(oacc[mb][4 * rg + 2] * inv, oacc[mb][4 * rg + 3] * inv)};
            *reinterpret_cast<FA_LDS v2u*>(ost + l32 * T::ROW + T::k_chunk(4 * mb + rg, l32) * 16 + g * 8) = w;
        }
#pragma unroll
    for (int x = 0; x < 32 / T::RPB; ++x) {
        const int rl = T::RPB * x + lane / T::CPR, c = T::k_chunk(lane % T::CPR, rl);
        const v4u val = *reinterpret_cast<FA_LDS const v4u*>(ost + x * 1024 + lane * 16);
        if (first_row + rl < it.rows && c * 8 < a.d) {
            int oh;
            const int ot = row_token(a, it, first_row + rl, &oh);
            __builtin_nontemporal_store(val, reinterpret_cast<v4u*>(a.O + (size_t)ot * a.o_token + (size_t)oh * a.o_head + c * 16));
        }
    }
}

// ---------------------------------------------------------------------------------------------- many rows

template <int D>
struct TallCfg {
    static constexpr int kWaves = 8, NST = 4;                 // LDS stages per tensor
    // 128 or 64 KiB of stages, and room for the Q rows of two waves; those of the others lie in stages that are empty at the start
    static constexpr int QBUF = 32 * PagedTile<D>::ROW, SMEM = NST * 2 * PagedTile<D>::BUF + 2 * QBUF;
    static_assert(2 * QBUF == PagedTile<D>::BUF, "Q rows of two waves per stage");
};

// Rows of a tile of V from `left` on lie past the sequence's end and repeat the last key's.  Their probabilities are 0, but 0 times a value that is not
// finite is not, and the wave's rows may see the last key: if it has such a value these rows become 0.  Each wave does so in front of its own reads, all
// write the same, and all go by the last key's own row, which nobody writes: a row that another wave has cleared says nothing of those behind it.
// (Requests that take the rows from a row of zeroes, as in the 32-row form, make the loop longer: 640 rows on 28339 keys B4 H5 H_kv1 d80
// 113.1 -> 118.2 us; so 113.5.)
__host__ __device__ constexpr int paged_asked_row(int left) { return left - 1; }
template <int D, bool kBf16>
__device__ __forceinline__ void paged_clear_past(FA_LDS char* stage, int left, int lane)
{
    using T = PagedTile<D>;
    const v4u row = *reinterpret_cast<FA_LDS const v4u*>(stage + paged_asked_row(left) * T::ROW + (lane % T::CPR) * 16);
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= Elem<kBf16>::not_finite(row[e]);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd) == 0, 1)) return;
    const v4u z = {0u, 0u, 0u, 0u};
    for (int at = left * T::ROW + lane * 16; at < T::BUF; at += 1024) *reinterpret_cast<FA_LDS v4u*>(stage + at) = z;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// Waves 0-3 and 4-7 run half an iteration apart (the second group passes one more barrier in front of the loop): while one wave of a
// SIMD is at its softmax, the other is at its MFMAs.  A tile of 256 rows x 64 keys at d = 128 takes a CU 1.97 us, as in fwd_pp_kernel, 90 % of
// what that mix of MFMAs and softmax reaches without any waits; ragged prompts up to 4096 H32 H_kv4 fp16 362-372 us, 0.92-0.95 PFLOP/s.  V(t + 2) is
// requested at the start of iteration t and waited for at its end, K(t + 3) at its end and waited for at the next one's; their slots were last
// read two barriers before.
// DU: columns that are worked on, a multiple of 16 from d on, the scores in steps of 16, O in blocks of 32 (rows in LDS have D): with DU = D the
// products of d = 80 meet zeroes in every third MFMA (a window of 512 keys B3 H12 N1777, DU 128, 96, 80: 32.1, 29.8, 29.3 us; 8 x up to 2000 rows H16
// 69.9 -> 67.0 with 80; d = 40 on 8000 keys 89.7 -> 86.6 with 48; d = 112 138.0 -> 136.2 with 112).
template <int D, int DU, bool kBf16, int kScores>
__device__ __forceinline__ void tall_rows(const ArgsOf<kScores> a)
{
    using T = PagedTile<D>;
    using C = TallCfg<D>;
    using E = Elem<kBf16>;
    constexpr int KS = DU / 16, MB = (DU + 31) / 32, NST = C::NST, NL = PagedRequests<D, C::kWaves>::NL, BC = T::BC;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    FA_LDS char* const Ks = (FA_LDS char*)smem;
    FA_LDS char* const Vs = Ks + NST * T::BUF;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6), grp = wave >> 2, l32 = lane & 31, g = lane >> 5;

    PagedItem it;
    if (!paged_item<kPagedTallRows, ArgsOf<kScores>>(a, lane, &it)) return;
    paged_mark_missing<kPagedTallRows, 512>(a, it, tid);
    int kmin, kmax;
    paged_range<kPagedTallRows>(a, it, &kmin, &kmax);
    if (kmax <= kmin) {
        paged_store_empty<kPagedTallRows, 512>(a, it, tid);
        return;
    }
    const int tile0 = kmin >> 6, ntiles = ((kmax + 63) >> 6) - tile0;
    if (a.d != D) {  // columns that no request writes
        const v4u z = {0u, 0u, 0u, 0u};
        for (int k = tid; k < C::SMEM / 16; k += 512) *reinterpret_cast<FA_LDS v4u*>(Ks + 16 * k) = z;
        paged_barrier();
    }

    // (row blocks s and 7 - s on SIMD s: evens out the diagonal)
    const int rblk = wave < 4 ? wave : 11 - wave;
    const int first_row = it.row0 + rblk * 32, r = first_row + l32;

    PagedRequests<D, C::kWaves> req;
    req.set(a, it, tile0, wave, lane);

    // ---- what the rows of this wave see
    int lo, hi, lo_max, hi_min, lo_min, hi_max;
    RowScores<kScores> row;
    if constexpr (kScores == kScoresPlain) {
        paged_bounds(a, it, r, kmin, kmax, &lo, &hi);
        lo_min = __builtin_amdgcn_readlane(lo, 0);
        hi_min = __builtin_amdgcn_readlane(hi, 0);
        lo_max = __builtin_amdgcn_readlane(lo, 31);  // (bounds do not fall from row to row)
        hi_max = __builtin_amdgcn_readlane(hi, 31);
    }

    v8h qf[KS];
    v16f oacc[MB], s[2];
    uint32_t p[2][2][4];
    PagedSoftmax<kBf16, MB, 2> soft;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[mb][e] = 0.0f;
    const float c2 = a.scale_log2, inv_c2 = __builtin_amdgcn_rcpf(c2);
    const int k_rd = T::k_lane(lane), v_rd = T::v_lane(lane);

    // ---- fragments of the MFMA phase, one software-pipelined stream of LDS reads and MFMAs (fwd_pp_kernel.h)
    v8h vf[4][MB];
    constexpr int VPD = 2, KPD = KS < 3 ? KS : 3;  // steps of V and K in flight
    v8h kf[KS][2];
    auto v_read = [&](uint32_t vbase, int st) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) vf[st][mb] = v_fragment<D>(vbase, st, mb);
    };
    auto k_read = [&](uint32_t kbase, int ks) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) kf[ks][kb] = k_fragment<D>(kbase, ks, kb);
    };
    auto pv_mfma = [&](int st) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) oacc[mb] = E::mfma(vf[st][mb], as_fragment(p[st >> 1][st & 1]), oacc[mb]);
    };
    auto qk_mfma = [&](int ks) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) s[kb] = E::mfma(kf[ks][kb], qf[ks], s[kb]);
    };
    auto s_clear = [&]() {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            if constexpr (kScores == kScoresSloped) {
                s[kb] = row.slant(kb);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kb][e] = 0.0f;
            }
        }
    };
    auto mfma_phase = [&](auto last_c, uint32_t vbase, uint32_t kbase) __attribute__((always_inline)) {
        constexpr bool kLast = decltype(last_c)::value;
        // step st: reads of V step st + VPD (behind the last ones: of K), MFMAs of step st
        pv_mfma(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 1; st < 4; ++st) {
            if (st + VPD - 1 < 4) v_read(vbase, st + VPD - 1);
            if (st == 3 && !kLast) {
#pragma unroll
                for (int ks = 0; ks < KPD; ++ks) k_read(kbase, ks);
            }
            pv_mfma(st);
        }
        if constexpr (!kLast) {
            s_clear();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + KPD < KS) k_read(kbase, ks + KPD);
                qk_mfma(ks);
            }
        }
#pragma unroll
        for (int st = 1; st < 4; ++st) {
            if (st + VPD - 1 < 4) __builtin_amdgcn_sched_group_barrier(0x100, 2 * MB, 0);
            if (st == 3 && !kLast) __builtin_amdgcn_sched_group_barrier(0x100, 2 * KPD, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, MB, 0);
        }
        if constexpr (!kLast) {
            if constexpr (kScores == kScoresSloped) __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + KPD < KS) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
            }
        }
    };
    // what has to have landed at the end of iteration t, and the requests for what is to come
    auto tail_requests = [&](int t, FA_LDS char* wrk) __attribute__((always_inline)) {
        if (t + 3 < ntiles) {
            req.load_k(a, tile_of<kScores>(t + 3, ntiles), wrk);
            req.find_v(a);
            req.ask(a, tile_of<kScores>(t + 4, ntiles));
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
    };
    auto iteration = [&](auto last_c, FA_LDS const char* __restrict__ rdv, FA_LDS const char* __restrict__ rdk, FA_LDS char* __restrict__ wrk,
                         FA_LDS char* __restrict__ wrv, int t) __attribute__((always_inline)) {
        const int kb0 = (tile0 + tile_of<kScores>(t, ntiles)) * BC;
        if (t + 2 < ntiles) req.load_v(a, tile_of<kScores>(t + 2, ntiles), wrv);
        if constexpr (kScores == kScoresPlain) {
            soft.tile(s, oacc, p, c2, inv_c2, mask_sides(kb0, lo_max, hi_min), lo - kb0 - 4 * g, hi - kb0 - 4 * g);
        } else {
            row.finish(a, s, kb0, g, mask_sides(kb0, lo_max, hi_min), lo, hi);
            soft.template tile<has_slopes(kScores)>(s, oacc, p, c2, inv_c2, 0, 0, 0, row.offset(kb0, g));
        }
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t vbase = fragment_base(rdv, v_rd);
        const uint32_t kbase = fragment_base(rdk, k_rd);
        v_read(vbase, 0);
        __builtin_amdgcn_sched_barrier(0);
        v_read(vbase, 1);
        paged_barrier_keep<2 * VPD * MB>();
        __builtin_amdgcn_s_setprio(1);
        mfma_phase(last_c, vbase, kbase);
        __builtin_amdgcn_s_setprio(0);
        tail_requests(t, wrk);
        paged_barrier();
    };

    // ---- prologue: Q, K(0), V(0), K(1), V(1), K(2) are requested in this order, and the first scores wait for Q and K(0) alone: 80 KiB
    // per CU (D = 128), against 144 KiB for all.  Q takes the way of the tiles, whole rows per request, through LDS of the
    // wave's own.  Before (Q by lanes into registers, one wait for everything) -> so: 1024 causal rows, B 8, H 32, d = 64 71.6 -> 67.8 us,
    // 256 rows on 512 keys, B 128, H 8, d = 128 106.2 -> 103.0 us, 2048 rows, B 2, H 16, d = 80 51.8 -> 50.6 us.  What is
    // left before the first scores, about 3 us, is these bytes' way from L2 into the CU: the page numbers of all three tiles asked
    // for at once changed nothing.
    req.ask(a, tile_of<kScores>(0, ntiles));
    FA_LDS char* const qst = wave < 2   ? Ks + 2 * NST * T::BUF + wave * C::QBUF
                             : wave < 4 ? Vs + 2 * T::BUF + (wave - 2) * C::QBUF
                             : wave < 6 ? Ks + 3 * T::BUF + (wave - 4) * C::QBUF
                                        : Vs + 3 * T::BUF + (wave - 6) * C::QBUF;
#pragma unroll
    for (int x = 0; x < 32 / T::RPB; ++x) {
        const int rl = T::RPB * x + lane / T::CPR, c = T::k_chunk(lane % T::CPR, rl), row = first_row + rl;
        int head;
        const int tok = row_token(a, it, row < it.rows ? row : it.rows - 1, &head);
        if (c * 8 < a.d) dma_kib_lanes<false>(a.Q + (size_t)tok * a.q_token + (size_t)head * a.q_head + c * 16, qst + x * 1024);
    }
#pragma unroll
    for (int t = 0; t < 3; ++t) {
        if (t < ntiles) {
            if (t > 0) req.ask(a, tile_of<kScores>(t, ntiles));
            req.load_k(a, tile_of<kScores>(t, ntiles), Ks + t * T::BUF);
            req.find_v(a);
            if (t < 2) req.load_v(a, tile_of<kScores>(t, ntiles), Vs + t * T::BUF);
        }
    }
    req.ask(a, tile_of<kScores>(3, ntiles));  // (vnext: of tile 2)
    if constexpr (kScores != kScoresPlain) {
        const ScoredArgs& again = read_again(a);
        if (again.tree && kmax > it.shift) tree_setup<512>(again, it, tid, (FA_LDS char*)smem + C::SMEM, has_slopes(kScores), &row.tree);
        row.set(again, it, r, kmin, kmax, &lo, &hi);
        lo_min = __builtin_amdgcn_readlane(lo, 0);
        hi_min = __builtin_amdgcn_readlane(hi, 0);
        lo_max = __builtin_amdgcn_readlane(lo, 31);
        hi_max = __builtin_amdgcn_readlane(hi, 31);
        if (again.tree) lo_min = rows_min(lo), lo_max = -rows_min(-lo), hi_max = kmax - 1;  // (a tree's bounds may fall)
    }
    if (ntiles > 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * NL) : "memory");
    else if (ntiles == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * NL) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");
    {
        const uint32_t qbase = fragment_base(qst, k_rd);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = k_fragment<D>(qbase, ks, 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));  // in registers before the loop
    }
    paged_barrier();  // K(0) is there for all, and every wave has read its Q
    {
        const uint32_t kbase = fragment_base(Ks, k_rd);
#pragma unroll
        for (int ks = 0; ks < KPD; ++ks) k_read(kbase, ks);
        s_clear();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (ks + KPD < KS) k_read(kbase, ks + KPD);
            qk_mfma(ks);
        }
    }
    if (ntiles > 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NL) : "memory");
    else if (ntiles == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    paged_barrier();  // V(0) and K(1) too
    if (grp == 1) {
        // V(1): the first group reads it before the barrier that ends this group's first iteration, behind which alone the second group's part of it
        // would be sure to have landed
        if (ntiles > 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        paged_barrier();
    }

    // Tiles of which no row of this wave sees a key: only the wave's share of the requests and the barriers.
    auto idle_iteration = [&](int t) {
        if (t + 2 < ntiles) req.load_v(a, tile_of<kScores>(t + 2, ntiles), Vs + ((t + 2) % NST) * T::BUF);
        paged_barrier();
        tail_requests(t, Ks + ((t + 3) % NST) * T::BUF);
        paged_barrier();
    };
    int t_lo = 0, t_hi = 0;
    if (first_row < it.rows && hi_max >= lo_min) {
        t_lo = max(0, (lo_min >> 6) - tile0 - 1);  // (the tile in front of the first visible one brings that one's scores)
        t_hi = min(ntiles, (hi_max >> 6) - tile0 + 1);
        if constexpr (last_first(kScores)) {
            t_lo = max(0, ntiles - 1 - t_hi);
            t_hi = ntiles - max(0, (lo_min >> 6) - tile0);
        }
        t_lo = min(t_lo, t_hi);
    }
    int t = 0;
    if constexpr (last_first(kScores))  // (the last tile's V is there)
        if (const int left = it.len - (tile0 + ntiles - 1) * BC; t_lo == 0 && t_hi > 0 && left < BC) paged_clear_past<D, kBf16>(Vs, left, lane);
    for (; t < t_lo; ++t) idle_iteration(t);
    for (; t < t_hi - 1; ++t)
        iteration(std::false_type{}, Vs + (t % NST) * T::BUF, Ks + ((t + 1) % NST) * T::BUF, Ks + ((t + 3) % NST) * T::BUF, Vs + ((t + 2) % NST) * T::BUF, t);
    if (t < t_hi) {
        if (const int left = it.len - (tile0 + t) * BC; !last_first(kScores) && left < BC) paged_clear_past<D, kBf16>(Vs + (t % NST) * T::BUF, left, lane);
        iteration(std::true_type{}, Vs + (t % NST) * T::BUF, Ks + ((t + 1) % NST) * T::BUF, Ks + ((t + 3) % NST) * T::BUF, Vs + ((t + 2) % NST) * T::BUF, t);
        ++t;
    }
    for (; t < ntiles; ++t) idle_iteration(t);
    if (grp == 0) paged_barrier();
    if (first_row >= it.rows) return;

    // ---- epilogue
    if (__builtin_expect(any_not_finite<MB>(oacc), 0)) paged_rescue<BC, MB, kBf16, kScores>(read_again(a), it, r, kmin, kmax, tile0, ntiles, 0, 1, soft.m_ref, oacc, row);
    paged_store_rows<D, MB, kBf16, kScores>(read_again(a), it, first_row, r, lane, g, soft.m_ref, soft.l_run, oacc, Ks + wave * (32 * T::ROW));
}

template <int D, int DU, bool kBf16>
__global__ void __launch_bounds__(512, DU == 32 ? 4 : 2) paged_tall_kernel(const PagedArgs a)
{
    tall_rows<D, DU, kBf16, kScoresPlain>(a);
}
template <int D, int DU, bool kBf16, int kScores>
__global__ void __launch_bounds__(512, 2) scored_tall_kernel(const ScoredArgs a)
{
    tall_rows<D, DU, kBf16, kScores>(a);
}

// ---------------------------------------------------------------------------------------------- rows between few and many
//
// 128 rows, four waves that share tiles of 64 keys: a chunk of some thirty to 128 tokens times heads, as a tree of drafted tokens is, leaves half of a
// 256-row work-group's waves without rows, and in 32-row ones each row block asks the L2 for the tiles by itself.  One barrier per tile: behind it the
// tile is there, and the stage that the one NST - 1 tiles ahead goes to has been read.  Two stages leave room for two work-groups per CU at D = 128, whose
// waves fill in for each other: one wave alone on a SIMD takes 1.45 us per tile, bound by the issue of its instructions (four stages: the same), two
// take 2.0.  Where there is a CU for each work-group it has a second group of waves instead, with every other tile and stages of its own; the two merge in LDS.
template <int D, int NSTAGES, int GROUPS>
struct MidCfg {
    static constexpr int kWaves = 4, NST = NSTAGES, STAGE = 2 * PagedTile<D>::BUF, SMEM = GROUPS * NST * STAGE;  // a stage: K, then V
    static_assert(kWaves * 32 * PagedTile<D>::ROW <= STAGE, "Q lies in the last stage at first, O in the first one at last");
    static_assert(GROUPS == 1 || kWaves * 64 * 4 * (D / 2 + 2) <= SMEM, "the second group's results");
};

template <int D, int DU, int NSTAGES, int GROUPS, bool kBf16, int kScores>
__global__ void __launch_bounds__(256 * GROUPS, 2) scored_mid_kernel(const ScoredArgs a)
{
    using T = PagedTile<D>;
    using C = MidCfg<D, NSTAGES, GROUPS>;
    using E = Elem<kBf16>;
    constexpr int KS = DU / 16, MB = (DU + 31) / 32, BC = T::BC, NST = C::NST, NL = PagedRequests<D, C::kWaves>::NL, kThreads = 256 * GROUPS;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6) & 3, grp = wave_uniform(tid >> 8), l32 = lane & 31, g = lane >> 5;
    FA_LDS char* const stages = (FA_LDS char*)smem + grp * (C::NST * C::STAGE);  // of the group

    PagedItem it;
    if (!paged_item<kPagedMidRows>(a, lane, &it)) return;
    paged_mark_missing<kPagedMidRows, kThreads>(a, it, tid);
    int kmin, kmax;
    paged_range<kPagedMidRows>(a, it, &kmin, &kmax);
    if (kmax <= kmin) {
        paged_store_empty<kPagedMidRows, kThreads>(a, it, tid);
        return;
    }
    const int tile0 = kmin >> 6, ntiles = ((kmax + 63) >> 6) - tile0;
    if (a.d != D) {  // columns that no request writes
        const v4u z = {0u, 0u, 0u, 0u};
        for (int k = tid; k < C::SMEM / 16; k += kThreads) *reinterpret_cast<FA_LDS v4u*>((FA_LDS char*)smem + 16 * k) = z;
        paged_barrier();
    }
    const int first_row = it.row0 + wave * 32, r = first_row + l32;

    // ---- Q, then the group's first NST - 1 tiles: grp, grp + GROUPS, ... in their order
    const int mine = (ntiles - grp + GROUPS - 1) / GROUPS, steps = (ntiles + GROUPS - 1) / GROUPS;
    auto tile_at = [&](int i) __attribute__((always_inline)) { return tile_of<kScores>(min(i * GROUPS + grp, ntiles - 1), ntiles); };
    PagedRequests<D, C::kWaves> req;
    req.set(a, it, tile0, wave, lane);
    req.ask(a, tile_at(0));
    FA_LDS char* const qst = stages + (NST - 1) * C::STAGE + wave * (32 * T::ROW);
#pragma unroll
    for (int x = 0; x < 32 / T::RPB; ++x) {
        const int rl = T::RPB * x + lane / T::CPR, c = T::k_chunk(lane % T::CPR, rl), row = first_row + rl;
        int head;
        const int tok = row_token(a, it, row < it.rows ? row : it.rows - 1, &head);
        if (c * 8 < a.d) dma_kib_lanes<false>(a.Q + (size_t)tok * a.q_token + (size_t)head * a.q_head + c * 16, qst + x * 1024);
    }
    auto request = [&](int i) __attribute__((always_inline)) {  // the group's tile i, whose places have been asked for
        FA_LDS char* const st = stages + (i % NST) * C::STAGE;
        req.load(a, tile_at(i), st, st + T::BUF);
    };
#pragma unroll
    for (int i = 0; i < NST - 1; ++i) {
        if (i < mine) {
            if (i > 0) req.ask(a, tile_at(i));
            request(i);
        }
    }
    req.ask(a, tile_at(NST - 1));
    RowScores<kScores> row;
    const ScoredArgs& again = read_again(a);
    if (again.tree && kmax > it.shift) tree_setup<kThreads>(again, it, tid, (FA_LDS char*)smem + C::SMEM, has_slopes(kScores), &row.tree);
    int lo, hi;
    row.set(again, it, r, kmin, kmax, &lo, &hi);
    int lo_min = __builtin_amdgcn_readlane(lo, 0), hi_min = __builtin_amdgcn_readlane(hi, 0);
    int lo_max = __builtin_amdgcn_readlane(lo, 31), hi_max = __builtin_amdgcn_readlane(hi, 31);  // (bounds do not fall from row to row)
    if (again.tree) lo_min = rows_min(lo), lo_max = -rows_min(-lo), hi_max = kmax - 1;           // (but a tree's do)

    v8h qf[KS];
    v16f oacc[MB];
    PagedSoftmax<kBf16, MB, 2> soft;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[mb][e] = 0.0f;
    const float c2 = a.scale_log2, inv_c2 = __builtin_amdgcn_rcpf(c2);
    const int k_rd = T::k_lane(lane), v_rd = T::v_lane(lane);
    for (int i = 0; i < steps; ++i) {
        const int kb0 = (tile0 + tile_at(i)) * BC;
        FA_LDS char* const kst = stages + (i % NST) * C::STAGE;
        FA_LDS char* const vst = kst + T::BUF;
        // tile i has landed when no more than the requests of those behind it are on their way (of each K and V, NL)
        const int behind = min(NST - 2, mine - 1 - i);
        if (NST > 3 && behind == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * NL) : "memory");
        else if (NST > 2 && behind == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NL) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (i == 0) {  // (Q came in front of it)
            const uint32_t qbase = fragment_base(qst, k_rd);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qf[ks] = k_fragment<D>(qbase, ks, 0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
        }
        paged_barrier();
        if (i + NST - 1 < mine) {
            request(i + NST - 1);
            req.ask(a, tile_at(i + NST));
        }
        if (i >= mine) continue;
        if (first_row >= it.rows || kb0 > hi_max || kb0 + BC <= lo_min) continue;  // nothing that this wave's rows see
        if (const int left = it.len - kb0; left < BC) paged_clear_past<D, kBf16>(vst, left, lane);
        v16f s[2];
        uint32_t p[2][2][4];
        {
            const uint32_t kbase = fragment_base(kst, k_rd);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                if constexpr (kScores == kScoresSloped) {
                    s[kb] = row.slant(kb);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[kb][e] = 0.0f;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) s[kb] = E::mfma(k_fragment<D>(kbase, ks, kb), qf[ks], s[kb]);
            order_reads_and_mfmas<2 * KS, 1, 6>();
            __builtin_amdgcn_sched_barrier(0);
        }
        const uint32_t vbase = fragment_base(vst, v_rd);
        v8h vf[4][MB];  // (the first step's are read while the softmax is worked out)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) vf[0][mb] = v_fragment<D>(vbase, 0, mb);
        __builtin_amdgcn_sched_barrier(0);
        row.finish(a, s, kb0, g, mask_sides(kb0, lo_max, hi_min), lo, hi);
        soft.template tile<has_slopes(kScores)>(s, oacc, p, c2, inv_c2, 0, 0, 0, row.offset(kb0, g));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ps = 0; ps < 4; ++ps)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                if (ps > 0) vf[ps][mb] = v_fragment<D>(vbase, ps, mb);
                oacc[mb] = E::mfma(vf[ps][mb], as_fragment(p[ps >> 1][ps & 1]), oacc[mb]);
            }
        order_reads_and_mfmas<4 * MB, 2, MB, true>();
        __builtin_amdgcn_sched_barrier(0);
    }
    if (first_row < it.rows && __builtin_expect(any_not_finite<MB>(oacc), 0))
        paged_rescue<BC, MB, kBf16, kScores>(read_again(a), it, r, kmin, kmax, tile0, ntiles, last_first(kScores) ? (ntiles - 1 - grp) % GROUPS : grp, GROUPS, soft.m_ref, oacc, row);
    paged_barrier();  // every wave is done with the stages
    FA_LDS char* ost = (FA_LDS char*)smem + wave * (32 * T::ROW);
    if constexpr (GROUPS == 2) {
        // the second group's results to the first, lane by lane: reference, sum, O
        FA_LDS float* const x = (FA_LDS float*)smem + wave * (64 * (16 * MB + 2)) + lane;
        ost = (FA_LDS char*)((FA_LDS float*)smem + wave * (64 * (16 * MB + 2)));  // (what the wave itself reads here)
        if (grp == 1) {
            x[0] = soft.m_ref, x[64] = soft.l_run;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[64 * (2 + 16 * mb + e)] = oacc[mb][e];
        }
        paged_barrier();
        if (grp == 1) return;
        const float m1 = x[0], m = fmaxf(soft.m_ref, m1), f0 = fast_exp2(soft.m_ref - m), f1 = fast_exp2(m1 - m);
        soft.l_run = f0 * soft.l_run + f1 * x[64];
        soft.m_ref = m;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[mb][e] = f0 * oacc[mb][e] + f1 * x[64 * (2 + 16 * mb + e)];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (read before O goes there)
    }
    if (first_row >= it.rows) return;
    paged_store_rows<D, MB, kBf16, kScores>(read_again(a), it, first_row, r, lane, g, soft.m_ref, soft.l_run, oacc, ost);
}

// ---------------------------------------------------------------------------------------------- merge of splits

// O = sum_s w_s O_s, LSE = log sum_s exp LSE_s with w_s = exp(LSE_s - LSE): one or (kWaves = 4, few rows with many splits) four waves per
// row.  Half a wave reads one split's row, 16 bytes per lane.  Bound by latency where there are few rows (32 rows x 27 splits of 128 columns
// 3.3 us): the first rows are requested before their weights are known; by memory where there are many (16384 x 4: 9.8 us, 38 MB): there a
// wave waits for the weights, and what a split that found nothing has in its place is not read (4096 causal rows H4 d128 in 7 splits, of which 4
// are there on average, 40.7 -> 36.9 us with the attention itself).
template <bool kBf16, int kWaves>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedMergeArgs a)
{
    __shared__ float xs[kWaves == 4 ? 4 * 2 * 32 * 5 : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6), half = lane >> 5, l32 = lane & 31;
    const int64_t row = kWaves == 4 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    const int tok = (int)(row / a.H);
    if (tok >= a.tokens) return;
    const int head = (int)(row - (int64_t)tok * a.H), S = a.num_splits, d = a.d;
    const float* const op = a.O_partial + (size_t)row * S * d + 4 * l32;
    const int first = kWaves == 4 ? 2 * wave : 0, step = 2 * kWaves;
    constexpr int U = 4;  // rows in flight per half wave
    v4f x[U];
    uint64_t there0 = 0, there1 = 0;  // splits that have found something
    auto request = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int s = s0 + k * step + half;
            const v4f z = {0.0f, 0.0f, 0.0f, 0.0f};
            x[k] = z;
            if (s < S && 4 * l32 < d && (kWaves == 4 || (s < 64 ? there0 >> s : there1 >> (s - 64)) & 1)) x[k] = *reinterpret_cast<const v4f*>(op + (size_t)s * d);
        }
    };
    const float* const lse = a.LSE_partial + (size_t)row * S;
    if constexpr (kWaves == 4) request(first);
    const float l0 = lane < S ? lse[lane] : -INFINITY, l1 = lane + 64 < S ? lse[lane + 64] : -INFINITY;
    if constexpr (kWaves == 1) {
        there0 = __builtin_amdgcn_ballot_w64(l0 != -INFINITY), there1 = __builtin_amdgcn_ballot_w64(l1 != -INFINITY);
        request(first);
    }
    // rows in front of the first sequence and behind the last one are nobody's
    if (tok < read_uniform_int(a.cu) || tok >= read_uniform_int(a.cu + a.B)) return;
    const float m = wave_max(fmaxf(l0, l1));
    const float m0 = m == -INFINITY ? 0.0f : m;
    const float w0 = fast_exp2((l0 - m0) * kLog2e), w1 = fast_exp2((l1 - m0) * kLog2e);
    const float sum = wave_sum(w0 + w1);
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = first; s0 < S; s0 += U * step) {
        if (s0 != first) request(s0);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int s = s0 + k * step + half;
            const float w = s < 64 ? __shfl(w0, s & 63) : __shfl(w1, s & 63);
            if (s < S && !(w == 0.0f)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(w, x[k][e], o[e]);
            }
        }
    }
    if constexpr (kWaves == 4) {
        float* const mine = xs + ((wave * 2 + half) * 32 + l32) * 5;  // (five words apart: no bank conflicts)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[e] = o[e];
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o[e] = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) o[e] += xs[((k * 2 + half) * 32 + l32) * 5 + e];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = xhalf_sum(o[e]);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (half == 0 && 4 * l32 < d) {
        const v2u w = {Elem<kBf16>::pack(o[0] * inv, o[1] * inv), Elem<kBf16>::pack(o[2] * inv, o[3] * inv)};
        *reinterpret_cast<v2u*>(a.O + (size_t)tok * a.o_token + (size_t)head * a.o_head + 8 * l32) = w;
    }
    if (lane == 0) a.LSE[row] = sum == 0.0f ? -INFINITY : m0 + fast_log2(sum) * kLn2;
}

// ---------------------------------------------------------------------------------------------- launches

template <int D, int DU, bool kBf16, int kRows>
inline hipError_t launch_paged_instance(const PagedArgs& a, long long blocks, hipStream_t st)
{
    const auto kern = [] {
        if constexpr (kRows == kPagedFewRows) return paged_few_kernel<D, kBf16>;
        else return paged_tall_kernel<D, DU, kBf16>;
    }();
    constexpr int smem = kRows == kPagedFewRows ? FewCfg<D>::SMEM : TallCfg<D>::SMEM;
    static DeviceFlags attr_done;  // per instantiation and device
    if (hipError_t e = ensure_dynamic_lds(reinterpret_cast<const void*>(kern), smem, attr_done); e != hipSuccess) return e;
    return launch_kernel(kern, dim3((unsigned)blocks), dim3(paged_threads(kRows)), smem, st, a);
}

// rows: of a work-group, which says which form
template <int D, bool kBf16>
inline int launch_paged_type(const PagedArgs& a, int rows, long long blocks, hipStream_t st)
{
    if (rows == kPagedFewRows) return (int)launch_paged_instance<D, D, kBf16, kPagedFewRows>(a, blocks, st);
    if constexpr (D == 128)
        if (a.d <= 80) return (int)launch_paged_instance<D, 80, kBf16, kPagedTallRows>(a, blocks, st);
    if (a.d <= D - 32) return (int)launch_paged_instance<D, D - 32, kBf16, kPagedTallRows>(a, blocks, st);
    if (a.d <= D - 16) return (int)launch_paged_instance<D, D - 16, kBf16, kPagedTallRows>(a, blocks, st);
    return (int)launch_paged_instance<D, D, kBf16, kPagedTallRows>(a, blocks, st);
}
template <int D>
inline int launch_paged_bucket(const PagedArgs& a, bool bf16, int rows, long long blocks, hipStream_t st)
{
    return bf16 ? launch_paged_type<D, true>(a, rows, blocks, st) : launch_paged_type<D, false>(a, rows, blocks, st);
}

template <int kRows>
inline hipError_t launch_scored_kernel(void (*kern)(ScoredArgs), int tiles, DeviceFlags& attr_done, const ScoredArgs& a, long long blocks, hipStream_t st, int threads = paged_threads(kRows))
{
    if (hipError_t e = ensure_dynamic_lds(reinterpret_cast<const void*>(kern), tiles + kTreeLds, attr_done); e != hipSuccess) return e;
    return launch_kernel(kern, dim3((unsigned)blocks), dim3(threads), a.tree ? tiles + kTreeLds : tiles, st, a);
}
template <int D, int DU, bool kBf16, int kScores, int kRows, int NSTAGES = 4, int GROUPS = 1>
inline hipError_t launch_scored_instance(const ScoredArgs& a, long long blocks, hipStream_t st)
{
    static DeviceFlags attr_done;  // per instantiation and device
    if constexpr (kRows == kPagedFewRows) {
        static_assert(2 * (FewCfg<D>::SMEM + kTreeLds) <= 160 * 1024, "two work-groups per CU");
        return launch_scored_kernel<kRows>(scored_few_kernel<D, kBf16, kScores>, FewCfg<D>::SMEM, attr_done, a, blocks, st);
    } else if constexpr (kRows == kPagedMidRows) {
        static_assert((3 - GROUPS) * (MidCfg<D, NSTAGES, GROUPS>::SMEM + kTreeLds) <= 160 * 1024, "two work-groups per CU, or one of two groups");
        return launch_scored_kernel<kRows>(scored_mid_kernel<D, DU, NSTAGES, GROUPS, kBf16, kScores>, MidCfg<D, NSTAGES, GROUPS>::SMEM, attr_done, a, blocks, st, 256 * GROUPS);
    } else {
        static_assert(TallCfg<D>::SMEM + kTreeLds <= 160 * 1024, "a work-group per CU");
        return launch_scored_kernel<kRows>(scored_tall_kernel<D, DU, kBf16, kScores>, TallCfg<D>::SMEM, attr_done, a, blocks, st);
    }
}
template <int kScores, bool kBf16>
inline int launch_scored_type(const ScoredArgs& a, int rows, long long blocks, hipStream_t st)
{
    if (rows == kPagedFewRows)
        return (int)(a.d <= 64 ? launch_scored_instance<64, 64, kBf16, kScores, kPagedFewRows>(a, blocks, st)
                               : launch_scored_instance<128, 128, kBf16, kScores, kPagedFewRows>(a, blocks, st));
    if (rows == kPagedMidRows) {
        // a CU for each work-group: two groups of waves where there are tiles enough (one group / two, pieces of 10 to 30 tiles 1.21 on average, more than 30
        // 1.39, 5 to 10 1.08, of one tile 0.92; a window of 1023 on 2900 keys H12 H_kv4 d64 29.8 -> 25.3 us)
        if (blocks <= kPagedCus && a.tiles_per_split >= 6)
            return (int)(a.d <= 64 ? launch_scored_instance<64, 64, kBf16, kScores, kPagedMidRows, 4, 2>(a, blocks, st)
                                   : launch_scored_instance<128, 128, kBf16, kScores, kPagedMidRows, 2, 2>(a, blocks, st));
        if (a.d <= 64) return (int)launch_scored_instance<64, 64, kBf16, kScores, kPagedMidRows>(a, blocks, st);
        return (int)launch_scored_instance<128, 128, kBf16, kScores, kPagedMidRows, 2>(a, blocks, st);
    }
    if (a.d <= 64) return (int)launch_scored_instance<64, 64, kBf16, kScores, kPagedTallRows>(a, blocks, st);
    if (a.d <= 96) return (int)launch_scored_instance<128, 96, kBf16, kScores, kPagedTallRows>(a, blocks, st);
    return (int)launch_scored_instance<128, 128, kBf16, kScores, kPagedTallRows>(a, blocks, st);
}
template <int kScores>
inline int launch_scored_kind(const ScoredArgs& a, bool bf16, int rows, long long blocks, hipStream_t st)
{
    return bf16 ? launch_scored_type<kScores, true>(a, rows, blocks, st) : launch_scored_type<kScores, false>(a, rows, blocks, st);
}
int launch_scored_masked(const ScoredArgs& a, bool bf16, int rows, long long blocks, hipStream_t st);
int launch_scored_capped(const ScoredArgs& a, bool bf16, int rows, long long blocks, hipStream_t st);
int launch_scored_sloped(const ScoredArgs& a, bool bf16, int rows, long long blocks, hipStream_t st);
int launch_scored_both(const ScoredArgs& a, bool bf16, int rows, long long blocks, hipStream_t st);

int launch_paged_d64(const PagedArgs& a, bool bf16, int rows, long long blocks, hipStream_t st);
int launch_paged_d128(const PagedArgs& a, bool bf16, int rows, long long blocks, hipStream_t st);
int launch_paged_merge(const PagedArgs& a, bool bf16, hipStream_t st);

}  // namespace fa
