// Attention over the paged 4-bit cache on the matrix cores: the kernel of every form, which differ in who sees what.
//
//   y = sum_t softmax_t(scale * q . k_t [+ bias of t - p]) v_t over the tokens t <= p (the last `window` of them) of a sequence, or over all of its tokens.
//
// Work.  An item is 16 or 32 rows (some new tokens x the query heads that share a key/value head) against the
// tokens they see, in tiles of 64 tokens.  All tiles of all items lie in one line, head by head, and the workgroups of one round
// take equal stretches of it, whatever the lengths of the sequences are: a stretch ends inside an item where it has to, its
// sums go to the workspace, and either the workgroup that writes the last part of an item adds them, or, where there are
// many parts, a second kernel.  Items that are all short stay whole.  The line is laid out
// on the device (a scan over the lengths in every workgroup), so that a captured call follows the lengths.  Inside a
// workgroup the four waves take tiles in turn, each with its own running maximum, sum and result; they meet once, at the
// end of an item.  No barrier in the loop over tiles.  (Rows of several sequences that share tokens, and waves with rows of their own: see
// PrefixArgs and rows_apart.)
//
// A tile.  v_mfma_f32_16x16x32_f16 with tokens (then dimensions) as rows and queries as columns, so that a lane's column is
// one query throughout: row statistics are a lane's own, and the probabilities come out of the first product in the
// order in which the second takes them.
//   scores   acc = sum over a block of 32 of (n - 8) * q, in fp32; S += d_k * acc.  A word of eight codes becomes halves in a shift,
//            four and-ors (1024 + n, or 1024 + 16 n for a nibble in bits 4..7) and four subtractions or fmas.  (Left as the subnormals
//            that nibbles are as they stand, with 8 sum(q) taken off apart, they cost half of that, and 1 to 2% of the time less:
//            but the matrix cores line products up by their factors' exponents, a subnormal's being 2^-14, and drop what lies 24 bits
//            below the largest.  Results were off by 1.5e-5 of their size, now by 3e-7.)
//            q is scaled by a power of two of its row and split into two halves: 22 bits, two products.
//   values   codes become n - 8 (1024 + n as half bits, less 1032), times the block's d: product and remainder of one
//            multiplication are two halves that hold it exactly (4 x 11 bits), the largest d of a tile brought to 2^11..2^12 by a power
//            of two that the result is kept in.  Probabilities split into two halves too: three products (low x low is under 2^-22).
//   A lane needs eight tokens' codes of one dimension, memory holds one token's of all: ds_read_b64_tr_b4 turns 16 x 16 nibbles.
// The running maximum of a row moves only when a score passes it by 2^2.5; until then nothing is rescaled.  Weights are 2^13 at
// the maximum, so that as pairs of halves they keep 22 bits down to 2^-26 of it, and steps of 2^-37 of it below.  A weight's
// exponent is its score less (the maximum less 13), in one fma.  From maxima of 2^20 on fp32 would round what is in parentheses by too much (from 2^26 on
// 13 may become 16, and weights pass fp16): there the maximum is taken off first, then 13 is added.  Such rows are rescaled every tile, and that branch does it, so
// that others pay for it with the compiler's registers only (0.3 % in the mean of 12 calls, 1.3 % at most; as a branch of its own up to 3.5 %).
//
// Weights, sums, maxima and results are fp32; every value that goes to the matrix cores has 22 bits.
//
// What bounds it, 32 heads of 128 on 8 (us a call): a token behind 131072 others 45, 151 MB of cache (3.3 TB/s; a copy moves
// 5.1), 48 sequences of 100 to 8191 tokens 62, 232 MB (3.8 TB/s), 4096 prompt tokens 386, 137 Gflop (356 Tflop/s): the vector
// units' and the matrix cores' issue slots.  A tile of 64 tokens and 16 (32) rows takes about 690 (870) vector instructions of four
// cycles, two thirds of them to unpack its codes, and 80 (160) products of sixteen.  A short chat's token 11.5: the chain of
// arguments, lengths, page, codes, one tile (2.2), the waves' meeting and the joining of two parts.
#pragma once

#include "kv_cache.h"
#include "lds_direct.h"
#include "qproj_internal.h"

#include <algorithm>
#include <cmath>

namespace qproj {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTile = 64;            // tokens of a tile
constexpr float kBias = 13.f;        // weights are 2^kBias at the running maximum
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kSlack = 2.5f;       // a score may pass it by this before the row is rescaled: 2^15.5 < 65504
constexpr float kFar = 0x1p20f;      // a running maximum this large is taken off the scores before kBias is added

// Who sees what.  A kernel is compiled for one of the argument types below.
enum Sees {
    kBefore,     // a row at position p: tokens up to p, the last `window` of them
    kAll,        // every row: all tokens of its sequence
    kBiased,     // either, with a bias of the distance added to the scores
    kPrefix,     // tokens up to p; several sequences an item, which share their first tokens
};

struct AttentionArgs {
    static constexpr Sees kSees = kBefore;
    static constexpr bool kApart = false;     // every wave has rows of its own and goes through all tiles of an item, instead of some tiles of rows that are all waves'
    KvView kv;
    const float *q;
    float *y;
    int64_t q_stride, y_stride, pages_stride;
    const int32_t *q_start, *kv_len, *pages;
    int32_t *error;
    float *parts;            // [workgroups][2] sums of items that were cut (part_floats each)
    uint32_t *calls;         // [slots] how many calls have counted parts; a workgroup's own and those no workgroup has go on by one in every such call
    uint64_t *arrived;       // [2][slots] parts written of the item that a stretch begins and does not end, and above them the call that counts them;
                             // calls use either half in turn.  Null: attention_join_kernel adds the parts
    int32_t *joins;          // [heads][n_seq][row_tiles][2] for it: of every item its first stretch (-1: nothing to join) and its last
    float scale;             // times log2(e) / kScoreBits
    int32_t n_tokens, n_seq, max_q, window;
    int32_t group;           // query heads of a key/value head
    int32_t splits, split;   // they are served `split` at a time, in `splits` goes
    uint32_t split_part;     // 2^16 / split, rounded up
    int32_t tokens;          // new tokens of an item
    int32_t row_tiles;       // items of a sequence, at most
    int32_t slots;           // workgroups that a grid can have
    int32_t slots_each;      // of those that this grid does not have, a workgroup's share
    int32_t most_items;      // of a head: as many as sequences that share no rows can have.  Their turns can be counted in 32 bits
    int32_t young;           // workgroups from this one on go first every other tile
};

struct AllArgs : AttentionArgs {
    static constexpr Sees kSees = kAll;
};

struct BiasArgs : AttentionArgs {
    static constexpr Sees kSees = kBiased;
    const float *bias;       // [query heads][2 * reach + 1], of tokens `reach` before a row to `reach` behind it
    int32_t reach;
    int32_t all;             // rows see all tokens
};

struct AllApartArgs : AllArgs {
    static constexpr bool kApart = true;
};

struct BiasApartArgs : BiasArgs {
    static constexpr bool kApart = true;
};

struct PrefixArgs : AttentionArgs {
    static constexpr Sees kSees = kPrefix;
    const int32_t *group_start, *shared_len;
    int32_t n_groups, max_group;
    int32_t together;        // sequences of an item
    uint32_t row_part;       // 2^16 / max_q, rounded up
};

// Scores, their maxima and biases are in powers of 2^kScoreBits: log2(e) takes the largest biases of fp32 past it otherwise.
template <typename A>
constexpr float kScoreBits = A::kSees == kBiased ? 4.f : 1.f;

// The kernel's arguments, loaded where they are used from here on.  Kept in registers from the start they are more scalars than there are, and
// the kernel's phases use different ones.
template <typename A>
__device__ __forceinline__ const A &fresh_arguments() {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef const A __attribute__((address_space(4))) *arguments;
    arguments p = (arguments)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const A *)p;
#else
    static A none;   // device-only; the host pass just has to parse it
    return none;
#endif
}

constexpr int part_floats(int dim, int cols) { return 16 * cols * (dim + 2); }

// workgroups of a compute unit, waves of a SIMD (a third would fit where dim * cols <= 128, with the 168 registers that leaves: a token of
// 131072 took 59 us instead of 48, of 64-wide heads 34 instead of 29; the vector units are busy with two)
constexpr int kPerCu = 2;

// a row's token: slot / split, of slots under 64 (the fraction is off by less than 2^-10, the quotient's distance from the next is 2^-5 at least)
__device__ __forceinline__ int token_of(const AttentionArgs &a, int slot) { return (int)((uint32_t)slot * a.split_part >> 16); }

// a / b of numbers under 2^31: a quotient in fp32, off by 2^-22 of itself, then what it misses by, then one (a third of the instructions of /)
__host__ __device__ __forceinline__ uint32_t quotient(uint32_t a, uint32_t b) {
#if defined(__HIP_DEVICE_COMPILE__)
    const float part = __builtin_amdgcn_rcpf((float)b);
    uint32_t q = (uint32_t)((float)a * part);
    q += (uint32_t)(int)floorf((float)(int)(a - q * b) * part);
    const int left = (int)(a - q * b);
    return q + (left >= (int)b) - (left < 0);
#else
    return a / b;
#endif
}

struct Sequence {
    int start, count, len;   // first row, rows, tokens in the cache; count 0 where there is nothing to do
};

__host__ __device__ __forceinline__ Sequence sequence(const AttentionArgs &a, int s, bool &bad) {
    Sequence q;
    q.start = a.q_start[s];
    const int end = a.q_start[s + 1];
    q.len = a.kv_len[s];
    q.count = end - q.start;
    bad = q.start < 0 || end < q.start || end > a.n_tokens || q.count > a.max_q || q.len < 0 || (int64_t)q.len > a.pages_stride << a.kv.page_shift;
    if (bad) q.count = 0;
    return q;
}

// the rows of an item and the tokens that any of them sees
struct Item {
    int seq, first, count;   // first row, its tokens
    int lo, hi;              // positions of its first and last token; tokens [see, hi] are seen (hi < 0: none).  Where all are: both the last one
    int see;
    int at;                  // kBiased: position of its first token
};

template <typename A>
__host__ __device__ __forceinline__ Item item_of(const A &a, int s, const Sequence &q, int row_tile) {
    Item it;
    it.seq = s;
    it.first = q.start + row_tile * a.tokens;
    it.count = min(a.tokens, q.count - row_tile * a.tokens);
    it.lo = q.len - q.count + row_tile * a.tokens;
    it.hi = it.lo + it.count - 1;
    it.see = a.window && it.lo >= a.window ? it.lo - a.window + 1 : 0;     // (lo is negative where a sequence has more rows than tokens)
    if constexpr (A::kSees == kPrefix) {     // (of a group: its first sequence, sequences, tokens they share)
        it.seq = q.start + row_tile * a.together;
        it.count = min(a.together, q.count - row_tile * a.together);
        it.first = it.lo = it.hi = 0;
        it.see = q.len;
    }
    if constexpr (A::kSees == kAll) it.lo = it.hi = q.len - 1;
    if constexpr (A::kSees == kBiased) {
        it.at = it.lo;
        if (a.all) it.lo = it.hi = q.len - 1;
    }
    return it;
}

__host__ __device__ __forceinline__ int item_tiles(const Item &it) { return it.hi < 0 ? 1 : it.hi / kTile - it.see / kTile + 1; }
// what an item takes of the line: a turn of the waves for every kWaves tiles, or where they are apart for every one
template <typename A>
__host__ __device__ __forceinline__ int item_turns(const Item &it) { return it.count <= 0 ? 0 : A::kApart ? item_tiles(it) : (item_tiles(it) + kWaves - 1) / kWaves; }
// a wave's rows of an item where they are apart
template <typename A>
__device__ __forceinline__ Item item_of_wave(const A &a, const Item &it, int wave) {
    Item mine = it;
    if constexpr (A::kApart) {
        const int skip = wave * (a.tokens / kWaves);
        mine.count = max(0, min(a.tokens / kWaves, it.count - skip));
        if (mine.count) mine.first += skip;      // (otherwise a row that there is: queries are loaded all the same)
        if constexpr (A::kSees == kBiased) {
            mine.at += skip;
            if (!a.all) mine.lo += skip, mine.hi = mine.lo + mine.count - 1;
        }
    }
    return mine;
}

// What lies behind the line's places: sequences, or groups of them.  Of a group: its first sequence, sequences, the tokens that they share.
template <typename A>
__host__ __device__ __forceinline__ int units_of(const A &a) {
    if constexpr (A::kSees == kPrefix) return a.n_groups * a.row_tiles;
    else return a.n_seq * a.row_tiles;
}
template <typename A>
__host__ __device__ __forceinline__ int each_of(const A &a) {     // what an item takes of a unit
    if constexpr (A::kSees == kPrefix) return a.together;
    else return a.tokens;
}
template <typename A>
__host__ __device__ __forceinline__ Sequence unit_of(const A &a, int s, bool &bad) {
    if constexpr (A::kSees == kPrefix) {
        Sequence g;
        g.start = a.group_start[s];
        const int end = a.group_start[s + 1];
        g.len = a.shared_len[s];
        g.count = end - g.start;
        bad = g.start < 0 || end < g.start || end > a.n_seq || g.count > a.max_group || g.len < 0;
        if (bad) g.count = 0;
        bad = bad || (s == 0 && g.start != 0) || (s == a.n_groups - 1 && end != a.n_seq);     // (sequences of no group: reported, left out)
        return g;
    } else {
        return sequence(a, s, bad);
    }
}

// Tiles of an item of several sequences: those that they share, then every sequence's own.  A sequence shares no more than lies before its rows, and
// whole tiles only.
__host__ __device__ __forceinline__ int shared_tiles(int shared, int before) { return max(0, min(shared, before)) / kTile; }
__host__ __device__ __forceinline__ int tiles_of(int len) { return len > 0 ? (len - 1) / kTile + 1 : 0; }
template <typename A>
__host__ __device__ __forceinline__ int turns_of(const A &a, int s, const Sequence &q, int row_tile) {
    const Item it = item_of(a, s, q, row_tile);
    if constexpr (A::kSees == kPrefix) {
        int before = 0x7fffffff, tiles = 0, with_rows = 0;
        for (int i = 0; i < it.count; ++i) {
            bool bad;
            const Sequence m = sequence(a, it.seq + i, bad);
            if (m.count == 0) continue;
            before = min(before, m.len - m.count);
            tiles += tiles_of(m.len);
            ++with_rows;
        }
        const int shared = with_rows ? shared_tiles(it.see, before) : 0;
        tiles -= (with_rows - 1) * shared;
        return (max(1, tiles) + kWaves - 1) / kWaves;
    } else {
        return item_turns<A>(it);
    }
}

// Thread `id`'s places of the line of one head's items, `per` of them: f(sequence, row tile, rows, turns) of those that hold an item (a sequence has
// as many places as max_q allows), until one returns true.  outside(sequence) of sequences that break the bounds.
template <typename A, typename F, typename G>
__host__ __device__ __forceinline__ void each_item(const A &a, int id, int units, int per, F &&f, G &&outside) {
    for (int u = id * per; u < min(units, (id + 1) * per);) {
        const int s = a.row_tiles == 1 ? u : (int)quotient(u, a.row_tiles), tile0 = u - s * a.row_tiles, tile1 = min(a.row_tiles, tile0 + min(units, (id + 1) * per) - u);
        bool bad;
        const Sequence q = unit_of(a, s, bad);
        if (bad && tile0 == 0) outside(s);
        for (int tile = tile0; tile < tile1 && tile * each_of(a) < q.count; ++tile)
            if (f(s, tile, q, turns_of(a, s, q, tile))) return;
        u += tile1 - tile0;
    }
}

// What a call's workgroups share out: the turns of all heads' items in one line, head by head.
struct Line {
    int start;               // what beginning an item counts as, in turns
    bool whole;              // items stay whole: the line is one of items
    int head_length;         // of one head
    uint32_t total, active;  // of all; stretches, as many as workgroups have one
    uint32_t length, longer; // a stretch's; the first `longer` have one more
};

// (spread: of the forms other than the causal one; apart: of items whose waves are, which stay whole)
__host__ __device__ __forceinline__ Line line_of(int head_turns, int head_items, int longest, uint32_t heads, uint32_t groups, bool spread, bool apart) {
    // Where there are more turns than workgroups, beginning an item (staging its queries, adding its sums) counts as two turns.  Where no item
    // is longer than a workgroup's share, items stay whole and are dealt out, forwards and backwards in turn: an item is as long as its
    // rows are far from the start of their sequence, so that long ones meet short ones.  Otherwise every workgroup has a stretch of the
    // line, of one length or one more; those of an XCD are neighbours.  (Without the charge 48 sequences took 67 us instead of 64.5, four
    // with eight new tokens 32.6 instead of 28.3, heads of 64 behind 100000 tokens 31 instead of 29.4, but 64 of 2000 tokens 14.3 instead of
    // 16.2; always charged, one of 8000 13.4 instead of 12.0; half of it, or from two turns a workgroup on, 1% more over 60 drawn
    // calls.  Cut where they could stay whole, 512 prompt tokens took 27.5 us instead of 23.3, 4096 410 instead of 402.)
    Line l;
    l.start = (uint32_t)head_turns * heads > groups ? 2 : 0;
    // (as long as a share: ceil(line / groups))
    l.whole = (uint64_t)(uint32_t)(longest + l.start - 1) * groups < (uint32_t)(head_turns + l.start * head_items) * heads;
    // The other forms cut items too where whole ones, a few a workgroup, would leave most workgroups waiting for those that have one more: where that is
    // over two turns of the average item.  (616 items on 512 workgroups, rows over five images' states: 60.8 us instead of 71.8; prompts
    // with a bias 64.9 instead of 67.8, a drawn one 124 instead of 177; where it is less than two, level.)
    if (apart) {
        l.whole = true;
    } else if (spread && l.whole && l.start) {
        const uint32_t items = (uint32_t)head_items * heads, turns = (uint32_t)(head_turns + l.start * head_items) * heads, rounds = (items + groups - 1) / groups;
        l.whole = (float)rounds * (float)turns / (float)items - (float)turns / (float)groups <= 2.f;
    }
    l.head_length = l.whole ? head_items : head_turns + l.start * head_items;
    l.total = (uint32_t)l.head_length * heads;
    l.active = l.total < groups ? l.total : groups;
    l.length = l.active ? quotient(l.total, l.active) : 0;
    l.longer = l.total - l.length * l.active;
    return l;
}

// The stretch of a workgroup; those with none get a number behind the last.  Workgroups b, b + 8, ... are on one XCD: they have neighbours, and
// those before `active` have every stretch once whatever the grid is.
__host__ __device__ __forceinline__ uint32_t stretch_of_block(uint32_t block, uint32_t active) {
    const uint32_t xcd = block % 8, rest = active % 8;
    return block < active ? xcd * (active / 8) + (xcd < rest ? xcd : rest) + block / 8 : active;
}

// the stretch that has position p of the line (the last one of what lies behind: where lengths change during a call, an item may seem to reach there)
__host__ __device__ __forceinline__ uint32_t stretch_at(const Line &l, uint32_t p) {
    const uint32_t edge = l.longer * (l.length + 1), last = l.active - 1;
    const uint32_t at = p < edge ? quotient(p, l.length + 1) : l.longer + quotient(p - edge, l.length);
    return at < last ? at : last;
}

// what a stretch takes of an item that it reaches at place `skip`, with `left` of the stretch to go: turns [from, to); none where it ends within
// the item's start (to <= 0)
struct Piece {
    int take, from, to;
};
__host__ __device__ __forceinline__ Piece piece_of(const Line &l, int skip, int turns, uint32_t left) {
    Piece p;
    const uint32_t rest = (uint32_t)(turns + l.start - skip);
    p.take = (int)(rest < left ? rest : left);
    p.from = l.whole ? 0 : max(0, skip - l.start);
    p.to = l.whole ? turns : skip + p.take - l.start;
    return p;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ void wave_sync() {   // LDS of one wave: its operations go in order, the compiler has to keep to it
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ uint32_t half_pair(float a, float b) {   // to nearest
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2v));
}
__device__ __forceinline__ float low_half(uint32_t v) { return (float)__builtin_bit_cast(half2v, v)[0]; }
__device__ __forceinline__ float high_half(uint32_t v) { return (float)__builtin_bit_cast(half2v, v)[1]; }

__device__ __forceinline__ float max_xor(float v) {   // over the lanes of a column: xor 16, xor 32
    uint32_t x, y;
    swap16(__float_as_uint(v), x, y);
    v = fmaxf(__uint_as_float(x), __uint_as_float(y));
    swap32(__float_as_uint(v), x, y);
    return fmaxf(__uint_as_float(x), __uint_as_float(y));
}

// 16 bytes a lane from `g` to l + 16 * lane, as global_to_lds16, but unseen by the compiler, which would wait for all loads in flight before
// any read of that memory.  Loads come back in order: what follows a wait for a later load of the same wave finds the bytes there.
__device__ __forceinline__ void global_to_lds16_unseen(const void *g, const void *l) {
    const uint32_t to = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)l;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(g) : "memory");   // (m0: nothing else here reads it)
}

// the same of 4 bytes, to l + 4 * lane
__device__ __forceinline__ void global_to_lds4_unseen(const void *g, const void *l) {
    const uint32_t to = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)l;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(g) : "memory");
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(v))));   // each row of 16 lanes
    uint32_t x, y;
    swap16(v, x, y);
    v = max(x, y);
    swap32(v, x, y);
    return (uint32_t)uniform((int)max(x, y));
}

// sums over the lanes up to each one
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);    // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
    return v;
}

// keeps a value where it is computed: the compiler otherwise moves whole chains behind the next branch, and what feeds them stays
// in registers that long
__device__ __forceinline__ void pin(f32x4 &v) { asm volatile("" : "+v"(v)); }
// an offset that the block it is used in sees as 32 bits: loads take it beside a scalar base
__device__ __forceinline__ uint32_t local(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Where the transposing read finds 16-byte chunk `chunk` of a token's value codes: the rows that one read takes together are 16 tokens
// apart, their chunks are turned so that they fall into different banks.  chunk_at is the chunk that lies at a place.
template <int D>
__device__ __forceinline__ int chunk_turn(int token) {
    const int turn = (token >> 4) & 3;
    return D == 128 ? turn : D == 256 ? turn | ((token >> 1) & 1) << 2 : D == 64 ? turn & 1 : turn % 3;
}
template <int D>
__device__ __forceinline__ int value_at(int token, int chunk) {
    const int turn = chunk_turn<D>(token);
    return token * (D / 2) + (D == 96 ? (chunk + turn) % 3 : chunk ^ turn) * 16;
}
template <int D>
__device__ __forceinline__ int chunk_at(int token, int place) {
    const int turn = chunk_turn<D>(token);
    return D == 96 ? (place + 3 - turn) % 3 : place ^ turn;
}

// Value codes go from memory to LDS directly.  Two tiles' worth of room where the rest leaves it: the next tile's codes are then asked for
// while this tile's are still read, otherwise behind the scores.
constexpr bool values_ahead(int dim) { return dim <= 128; }

template <int D, int NQ>
struct WaveLds {
    uint8_t v[values_ahead(D) ? 2 : 1][kTile * D / 2];
    uint16_t k_scale[D / 32][kTile];
    uint16_t v_scale[D / 32][kTile];
};

constexpr int meet_rounds(int dim) { return dim > 128 ? 2 : 1; }   // (so that two workgroups' LDS fit)

// What a kind of attention keeps beside.
template <Sees S>
struct KindLds {};

// Biases of the item's heads by distance, from reach + kBiasPad tokens before a row to as many behind it, those beyond reach the last ones repeated: a
// tile of 64 tokens that some row of an item is within reach of finds all its biases at one address a lane and constant offsets.
constexpr int kBiasPad = 96, kBiasFloats = 3600;     // (pad: 63 tokens of the tile, 31 rows of the item.  Room: eight heads at a reach of 128)
constexpr int bias_room(int reach) { return 2 * reach + 1 + 2 * kBiasPad; }
template <>
struct KindLds<kBiased> {
    float bias[kBiasFloats + 64];     // (loads write 64 at a time)
};

// The item's sequences, a copy for every wave, which keeps itself in order.
constexpr int kTogether = 32;        // at most
template <>
struct KindLds<kPrefix> {
    int32_t first[kWaves][kTogether], count[kWaves][kTogether], before[kWaves][kTogether];   // first row, rows, tokens before them
    int32_t newest[kWaves][64];      // its last token
    int32_t ends[kWaves][64];        // tiles of the item up to the sequence's last one
};

template <int D, int NQ, typename A>
struct SharedLds : KindLds<A::kSees> {
    union {
        WaveLds<D, NQ> wave[kWaves];
        struct {
            f32x4 o[kWaves][D / 16 / meet_rounds(D)][64];
            float m[kWaves][16], l[kWaves][16];
        } meet;
    };
    u32x4 q[A::kApart ? kWaves : 1][D / 32][NQ][2][64];   // the item's queries as the matrix cores take them: high halves, low halves
    float q_most[kWaves][NQ][16]; // of the waves' blocks, the rows' largest queries
    int32_t line[kThreads][2];    // a thread's items on a head's line: turns before them, theirs
    int32_t only[6][kThreads];    // where a thread has one place of the line: its item, as in `found`
    int32_t waves[kWaves][3];     // a wave's: turns, items, the longest
    int32_t last;                 // whether the workgroup wrote the last part of an item
    uint32_t call;                // the call's number, where parts are counted, less kFirstCall; for the first wave
    int32_t found[2][7];          // this item and the next one in turn: sequence, row tile, its turns, the sequence's first row, rows, tokens, and what is before the item (-1: it is gone)
};

// what a wave holds of an item
template <int D, int NQ>
struct Running {
    f32x4 o[D / 16][NQ];   // [16 dimensions][16 queries]: lane's column is query lane % 16, rows 4 * (lane / 16) + r
    float m[NQ], l[NQ];    // of the lane's column; l of the lane's own tokens only until the end
};

// kPrefix: what is the same for all lanes of the item's sequences
struct Members {
    int lead;            // a sequence whose pages hold what is shared
    int shared, tiles;   // tiles that are shared, all of them
};

template <int D, int NQ, typename A>
__device__ __forceinline__ Members members(const A &a, const Item &it, SharedLds<D, NQ, A> &lds, int wave, int lane) {
    Members m{};
    if constexpr (A::kSees == kPrefix) {
        Sequence q{0, 0, 0};
        bool bad = false;
        if (lane < it.count) q = sequence(a, it.seq + lane, bad);
        if (bad) atomicOr(a.error, kKvBadRows);
        const uint64_t rows = __ballot(q.count > 0);
        const int before = 0x7fffffff - (int)wave_max(q.count > 0 ? 0x7fffffffu - (uint32_t)max(0, q.len - q.count) : 0u);
        m.shared = rows ? shared_tiles(it.see, before) : 0;
        m.lead = it.seq + (rows ? __builtin_ctzll(rows) : 0);
        const int ends = wave_scan(q.count > 0 ? tiles_of(q.len) - m.shared : 0) + m.shared;
        m.tiles = __builtin_amdgcn_readlane(ends, 63);
        if (lane < kTogether) {
            lds.first[wave][lane] = q.count > 0 ? q.start : 0;     // (a row that there is: columns without one load it)
            lds.count[wave][lane] = q.count;
            lds.before[wave][lane] = q.len - q.count;
        }
        lds.newest[wave][lane] = q.len - 1;
        lds.ends[wave][lane] = ends;
        wave_sync();
    }
    return m;
}

// A column's row: whether there is one, its number, and of kPrefix the sequence within the item and the last token that it sees.
struct Row {
    bool live;
    int row, head, seq, last;
};
template <int D, int NQ, typename A>
__device__ __forceinline__ Row row_of(const A &a, const Item &it, int heads, int slot, const SharedLds<D, NQ, A> &lds, int wave) {
    Row r{};
    const int token = token_of(a, slot);
    r.head = slot - token * a.split;
    if constexpr (A::kSees == kPrefix) {
        const int seq = token < a.tokens ? (int)((uint32_t)token * a.row_part >> 16) : 0, i = token - seq * a.max_q;
        r.live = token < a.tokens && i < lds.count[wave][seq] && r.head < heads;
        r.row = lds.first[wave][seq] + (r.live ? i : 0);
        r.seq = r.live ? seq : -1;
        r.last = r.live ? lds.before[wave][seq] + i : -1;
    } else {
        r.live = token < it.count && r.head < heads;
        r.row = it.first + (r.live ? token : 0);
    }
    return r;
}

// 16 queries of an item for the matrix cores: 22 bits of q * scale * log2(e), the row scaled by a power of two.  A wave takes the blocks
// wave, wave + 4, ... of all rows.  (All blocks in every wave, for want of a meeting about the rows' largest values, kept the loads of
// keys and values waiting: 512 prompt tokens took 23.5 us instead of 21.7, 4096 402 instead of 388.)
template <int D, int NQ, typename A>
struct Queries {
    static constexpr int kEvery = A::kApart ? 1 : kWaves, kMine = (D / 32 + kEvery - 1) / kEvery;
    f32x4 x[NQ][kMine][2];
};

template <int D, int NQ, typename A>
__device__ __forceinline__ void load_queries(const A &a, const Item &it, int head0, int heads, Queries<D, NQ, A> &q, const SharedLds<D, NQ, A> &lds, int wave, int lane) {
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
        const Row r = row_of(a, it, heads, g * 16 + (lane & 15), lds, wave);
        const float *row = a.q + (int64_t)r.row * a.q_stride + (int64_t)(head0 + (r.live ? r.head : 0)) * D + 8 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < q.kMine; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) q.x[g][i][k] = *reinterpret_cast<const f32x4 *>(row + 32 * min((A::kApart ? 0 : wave) + q.kEvery * i, D / 32 - 1) + 4 * k);
    }
}

// One barrier, about the rows' largest values; the staged queries need another.  q_unit: what sums are multiplied by, of the lane's columns.
template <int D, int NQ, typename A>
__device__ __forceinline__ void stage_queries(const A &a, const Item &it, int heads, Queries<D, NQ, A> &q, SharedLds<D, NQ, A> &lds, float (&q_unit)[NQ], int wave,
                                              int lane) {
    const int col = lane & 15;
    float mosts[NQ];
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
        const bool live = row_of(a, it, heads, g * 16 + col, lds, wave).live;
        float most = 0.f;
        bool whole = true;
#pragma unroll
        for (int i = 0; i < q.kMine; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = live ? q.x[g][i][k][j] * a.scale : 0.f;
                    q.x[g][i][k][j] = x;
                    most = fmaxf(most, fabsf(x));
                    whole = whole && fabsf(x) <= 3.402823466e38f;
                }
        most = max_xor(whole ? most : INFINITY);
        if (A::kApart) mosts[g] = most;
        else if (lane < 16) lds.q_most[wave][g][lane] = most;
    }
    if (!A::kApart) __syncthreads();
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
        float most = 0.f;
        if (A::kApart) {
            most = mosts[g];
        } else {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) most = fmaxf(most, lds.q_most[w][g][col]);
        }
        // (frexp: most = f * 2^e with f in [0.5, 1); where a value is not finite the row stays as it is: NaN comes of it)
        const int e = most > 0.f && most < INFINITY ? __builtin_amdgcn_frexp_expf(most) : 0;
        q_unit[g] = ldexpf(1.f, max(e - 15, -126));    // (not 0, which masked scores are multiplied by; such scores are 0)
#pragma unroll
        for (int i = 0; i < q.kMine; ++i) {
            const int b = (A::kApart ? 0 : wave) + q.kEvery * i;
            if (b >= D / 32) continue;
            u32x4 hi, lo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float u = ldexpf(q.x[g][i][0][j], 15 - e), v = ldexpf(q.x[g][i][1][j], 15 - e);
                hi[j] = half_pair(u, v);
                lo[j] = half_pair(u - low_half(hi[j]), v - high_half(hi[j]));
            }
            lds.q[A::kApart ? wave : 0][b][g][0][lane] = hi;
            lds.q[A::kApart ? wave : 0][b][g][1][lane] = lo;
        }
    }
}

// Tiles [from, to) of an item (in tiles from token 0 on), every kWaves-th of them (all of them where the waves are apart).  Two barriers of the workgroup, before and
// behind the staged queries (the second alone where the waves are apart), whatever there is to do.
template <int D, int NQ, typename A>
__device__ __forceinline__ void walk(const A &a, const Item &it, const Members &members, int kv_head, int head0, int heads, int from, int to, SharedLds<D, NQ, A> &shared,
                                     int wave, Running<D, NQ> &st, int lane) {
    WaveLds<D, NQ> &lds = shared.wave[wave];
    constexpr int B = D / 32, RB = D / 2, T = D / 16;
    constexpr bool kAhead = values_ahead(D);
    constexpr int kEvery = A::kApart ? 1 : kWaves;
    const int col = lane & 15, part = lane >> 4;
    const KvView &kv = a.kv;
    const int shift = kv.page_shift, mask = (1 << shift) - 1;

#pragma unroll
    for (int g = 0; g < NQ; ++g) {
        st.m[g] = -INFINITY;
        st.l[g] = 0.f;
#pragma unroll
        for (int t = 0; t < T; ++t) st.o[t][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const bool work = from < to && (A::kSees == kPrefix ? members.tiles > 0 : it.hi >= 0) && (!A::kApart || it.count > 0);

    // Where a tile's tokens are: whose (of the item's sequences; -1: shared, or the only one's), which pages, its first token, the first and the last one that is seen.
    struct Place {
        int own, seq, t0, see, hi;
    };
    const auto find = [&](int tile) {
        if constexpr (A::kSees == kPrefix) {
            if (tile < members.shared) return Place{-1, members.lead, tile * kTile, 0, members.shared * kTile - 1};
            const int ends = shared.ends[wave][lane], last = shared.newest[wave][lane];
            const int own = min((int)__popcll(__ballot(ends <= tile)), it.count - 1);
            const int start = own ? __builtin_amdgcn_readlane(ends, max(own - 1, 0)) : members.shared;
            return Place{own, it.seq + own, (members.shared + tile - start) * kTile, 0, __builtin_amdgcn_readlane(last, own)};
        } else {
            return Place{-1, it.seq, tile * kTile, it.see, it.hi};
        }
    };
    // page of the lane's token of a tile (a token outside what is seen: of the nearest one that is)
    const int32_t *table = a.pages + (int64_t)it.seq * a.pages_stride;
    const auto page_of = [&](const Place &p) {
        const int t = min(max(p.t0 + lane, p.see), p.hi);
        return (A::kSees == kPrefix ? a.pages + (int64_t)p.seq * a.pages_stride : table)[t >> shift];
    };
    const int last_tile = work ? from + (to - 1 - from) / kEvery * kEvery : from;   // of this wave
    Place now{}, next{};        // kPrefix: this tile's and the wave's next one's (otherwise known from their numbers)
    if (A::kSees == kPrefix && work) now = find(from), next = find(min(from + kEvery, last_tile));
    int page = work ? page_of(A::kSees == kPrefix ? now : find(from)) : 0, page_next = work ? page_of(A::kSees == kPrefix ? next : find(min(from + kEvery, last_tile))) : 0;
    bool bad_page = false;

    uint32_t k_raw[4][B];
    uint32_t ks_raw[(B + 1) / 2], vs_raw[(B + 1) / 2];
    int bad_groups;      // of the tile whose loads are in flight
    uint32_t rows[4];    // first row of its groups of 16 tokens

    const auto place = [&](const Place &p) {   // rows of the tile whose pages have come
        const int own = p.t0 + lane, t = min(max(own, p.see), p.hi);
        const bool bad = (uint32_t)page >= (uint32_t)kv.n_pages;
        bad_page = bad_page || (bad && t == own);
        bad_groups = 0;
        const uint32_t row = (((bad ? 0u : (uint32_t)page) * kv.n_head + kv_head) << shift) + (own & mask);
        const uint64_t bad_lanes = __ballot(bad);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            rows[g] = __builtin_amdgcn_readlane(row, 16 * g);
            bad_groups |= (int)(bad_lanes >> (16 * g) & 1) << g;
        }
    };
    // chunk i * 64 + lane of the tile's value codes, in the order in which they lie in LDS
    const uint32_t k_off = (uint32_t)(col * RB + part * B * 4), s_off = (uint32_t)(col * B * 2);
    const auto chunk_offset = [&](int i) {
        const int chunk = i * 64 + lane, token = chunk / B;
        return (uint32_t)((token & 15) * RB + chunk_at<D>(token, chunk - token * B) * 16);
    };
    uint32_t v_off[D == 128 ? 1 : B];
#pragma unroll
    for (int i = 0; i < (D == 128 ? 1 : B); ++i) v_off[i] = chunk_offset(i);
    const auto offset = [&](int i) { return D == 128 ? local(v_off[0]) ^ (uint32_t)(16 * i) : v_off[D == 128 ? 0 : i]; };   // (of 128: the turn alone)
    const auto load_v = [&](int to_buffer, const uint32_t (&rows)[4]) {
        uint8_t *const to = lds.v[to_buffer];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (B >= 4) {            // 64 chunks are within one group of 16 tokens
                global_to_lds16_unseen(kv.v_codes + (uint64_t)rows[i * 64 / (16 * B)] * RB + offset(i), to + i * 1024);
            } else {                 // of two
                const int group = (i * 64 + lane) / (16 * B);
                const uint32_t row = group == 0 ? rows[0] : group == 1 ? rows[1] : group == 2 ? rows[2] : rows[3];
                global_to_lds16_unseen(kv.v_codes + (uint64_t)row * RB + offset(i), to + i * 1024);
            }
        }
    };
    const auto load_scales = [&]() {
        const uint64_t row = part == 0 ? rows[0] : part == 1 ? rows[1] : part == 2 ? rows[2] : rows[3];
        const uint8_t *ks = reinterpret_cast<const uint8_t *>(kv.k_scales) + row * (B * 2) + s_off;
        const uint8_t *vs = reinterpret_cast<const uint8_t *>(kv.v_scales) + row * (B * 2) + s_off;
        if (B == 3) {
            const uint16_t *k3 = reinterpret_cast<const uint16_t *>(ks), *v3 = reinterpret_cast<const uint16_t *>(vs);
            ks_raw[0] = k3[0] | (uint32_t)k3[1] << 16, ks_raw[1] = k3[2];
            vs_raw[0] = v3[0] | (uint32_t)v3[1] << 16, vs_raw[1] = v3[2];
        } else {
#pragma unroll
            for (int i = 0; i < B / 2; ++i) {
                ks_raw[i] = reinterpret_cast<const uint32_t *>(ks)[i];
                vs_raw[i] = reinterpret_cast<const uint32_t *>(vs)[i];
            }
        }
    };
    const auto load_k = [&]() {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const auto base = scalar_global(kv.k_codes + (uint64_t)rows[g] * RB);
            if constexpr (B == 2) {
                const u32x2 w = load_global<u32x2>(base, local(k_off));
                k_raw[g][0] = w[0], k_raw[g][1] = w[1];
            } else if constexpr (B == 3) {
#pragma unroll
                for (int b = 0; b < B; ++b) k_raw[g][b] = load_global<uint32_t>(base, local(k_off) + 4 * b);
            } else {
#pragma unroll
                for (int b = 0; b < B; b += 4) {
                    const u32x4 w = load_global<u32x4>(base, local(k_off) + 4 * b);
#pragma unroll
                    for (int i = 0; i < 4; ++i) k_raw[g][b + i] = w[i];
                }
            }
        }
    };
    // (loads come back in order: pages, then queries, then keys and values)
    // Of two waves of a SIMD the older one issues first whenever it can, and the younger one is left over: of 4096 prompt tokens the first
    // 256 workgroups were done after 290 us, the others after 420.  So the younger ones go first every other tile; apart from that whoever
    // multiplies values goes before whoever multiplies keys, which keeps the two in different phases, and what the waves meet for
    // before everything.  (No wave up 403.5 us, the younger ones 386.7, all of them 391; 512 prompt tokens 22.6, 21.5, 22.1; 48 sequences 66, 64, 64.5.
    // Where one item is cut into many parts, all of them: a token of 131072 46.0 us against 46.9, of 32768 24.1 against 24.8.)
    __builtin_amdgcn_s_setprio(3);
    if constexpr (A::kSees == kBiased) {     // (before the queries: where those are waited for, these have come)
        const int span = 2 * a.reach + 1, room = bias_room(a.reach);
        for (int i = wave * 64; i < heads * room; i += kThreads) {
            const int h = min((int)quotient(i + lane, room), heads - 1), at = i + lane - h * room;
            global_to_lds4_unseen(a.bias + (int64_t)(head0 + h) * span + min(max(at - kBiasPad, 0), span - 1), shared.bias + i);
        }
    }
    Queries<D, NQ, A> queries;
    load_queries<D, NQ>(a, it, head0, heads, queries, shared, wave, lane);
    if (work) {
        place(A::kSees == kPrefix ? now : find(from));
        if (kAhead) load_v(0, rows);
        load_scales();
        load_k();
    }
    float q_unit[NQ];
    stage_queries<D, NQ>(a, it, heads, queries, shared, q_unit, wave, lane);
    __syncthreads();
    if (!work) return;

    int pos[NQ];                // what the column's row sees, up to this token, -1: no row
    int own_bias[NQ];           // kBiased: its bias of token 0 is there, had the row one that far away
    int own_seq[NQ];            // kPrefix: of the item's sequences
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
        const int slot = g * 16 + col, token = token_of(a, slot);
        const bool live = token < it.count && slot - token * a.split < heads;
        pos[g] = live ? (A::kSees == kAll ? it.hi : it.lo + token) : -1;
        if constexpr (A::kSees == kPrefix) {
            const Row r = row_of(a, it, heads, slot, shared, wave);
            pos[g] = r.last;
            own_seq[g] = r.seq;
        }
        if constexpr (A::kSees == kBiased) {
            if (live && a.all) pos[g] = it.hi;
            own_bias[g] = (live ? slot - token * a.split : 0) * bias_room(a.reach) + kBiasPad + a.reach - (it.at + (live ? token : 0));
        }
    }

    // (in registers, and unknown to the compiler: and-or in one instruction, half times -1 plus float in one)
    uint32_t mask0 = 0x000f000fu, mask1 = 0x00f000f0u, magic = 0x64006400u;
    float minus = -1.f;
    asm volatile("" : "+v"(mask0), "+v"(mask1), "+s"(magic), "+s"(minus));

    int unit = 0;               // results are in units of 2^unit
    float limit[NQ];            // a row is rescaled where a score passes this
    float base[NQ];             // what is taken off a score
    uint32_t poison = 0;        // blocks of values that are not finite and were seen, 8 bits a column
#pragma unroll
    for (int g = 0; g < NQ; ++g) base[g] = -kBias, limit[g] = -INFINITY;

    int buffer = 0;
    const bool young = (int)blockIdx.x >= a.young;
    bool up = false;
    for (int tile = from; tile < to; tile += kEvery) {
        const Place here = A::kSees == kPrefix ? now : find(tile);
        const int t0 = here.t0;
        const int bad_now = bad_groups;
        up = young && !up;
        if (up) __builtin_amdgcn_s_setprio(2); else __builtin_amdgcn_s_setprio(0);
        // ---- scales to LDS ----
        const int t = t0 + lane;
        const bool live = t >= here.see && t <= here.hi && !((bad_now >> part) & 1);
        uint32_t most = 0;
        bool tiny = false;
        uint16_t vs[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            lds.k_scale[b][lane] = (uint16_t)(ks_raw[b / 2] >> (16 * (b & 1)));
            vs[b] = live ? (uint16_t)(vs_raw[b / 2] >> (16 * (b & 1))) : 0;
            const uint32_t size = (uint32_t)vs[b] & 0x7fffu;
            most = max(most, size);
            tiny = tiny || size - 1 < 0x3ffu;       // (zero is not)
        }
        uint64_t strange = __ballot(most >= 0x7c00u);
        if (strange) {           // blocks that are not finite count as zeros here; who sees them gets NaN below
            most = 0;
#pragma unroll
            for (int b = 0; b < B; ++b)
                if ((vs[b] & 0x7fffu) < 0x7c00u) most = max(most, (uint32_t)vs[b] & 0x7fffu);
        }
        // scales within 2^-14 .. 2^12 are taken as they are; otherwise the tile's largest goes to 2^11 .. 2^12
        int unit_now = 0;
        if (__ballot(most >= 0x6c00u || tiny)) {
            const uint32_t top = wave_max(most);
            unit_now = top ? __builtin_amdgcn_frexp_expf(h2f(top)) - 12 : unit;     // top < 2^(unit + 12)
        }
        const float shrink = unit_now == unit ? 1.f : ldexpf(1.f, unit - unit_now);  // of what has been summed
        unit = unit_now;
        if (unit == 0 && !strange) {
#pragma unroll
            for (int b = 0; b < B; ++b) lds.v_scale[b][lane] = vs[b];
        } else {
#pragma unroll
            for (int b = 0; b < B; ++b) lds.v_scale[b][lane] = (vs[b] & 0x7fffu) < 0x7c00u ? f2h(ldexpf(h2f(vs[b]), -unit)) : 0;
        }
        uint64_t strange_of[B];
        if (strange) {
#pragma unroll
            for (int b = 0; b < B; ++b) strange_of[b] = __ballot((vs[b] & 0x7fffu) >= 0x7c00u);
        }
        wave_sync();
        const uint32_t rows_now[4] = {rows[0], rows[1], rows[2], rows[3]};
        // ---- the next tile's values and scales, and the page of the one behind ----
        // (behind the wave's last tile that tile again: loads that no branch surrounds are waited for one by one)
        page = page_next;
        if constexpr (A::kSees == kPrefix) {
            now = next;
            next = find(min(tile + 2 * kEvery, last_tile));
            page_next = page_of(next);
            place(now);
        } else {
            page_next = page_of(find(min(tile + 2 * kEvery, last_tile)));
            place(find(min(tile + kEvery, last_tile)));
        }
        load_scales();
        // ---- scores ----
        f32x4 s[4][NQ];
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int c = 0; c < NQ; ++c) s[g][c] = f32x4{0.f, 0.f, 0.f, 0.f};
        // A step is a block of kStep groups of tokens.  Behind each of its products goes a piece of the next step's codes or of the
        // previous step's sums, so that the matrix cores and the vector unit work at once; the barriers keep that order.
        constexpr int kStep = NQ == 1 ? 4 : 2, kSteps = B * 4 / kStep;
        {
            half8 codes[2][kStep];
            f32x4 acc[2][kStep][NQ];
            u32x2 d[2][kStep];
            half8 qh[NQ], ql[NQ];
            const auto code = [&](int step, int g) {
                const uint32_t w = k_raw[step % (4 / kStep) * kStep + g][step / (4 / kStep)], w8 = w >> 8;
                const half2v k1032 = {(_Float16)1032.f, (_Float16)1032.f}, k72 = {(_Float16)72.f, (_Float16)72.f}, k16th = {(_Float16)0.0625f, (_Float16)0.0625f};
                const auto even = [&](uint32_t x) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (x & mask0) | magic) - k1032); };
                const auto odd = [&](uint32_t x) {
                    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2v, (x & mask1) | magic), k16th, -k72));
                };
                codes[step & 1][g] = __builtin_bit_cast(half8, u32x4{even(w), odd(w), even(w8), odd(w8)});
            };
            const auto add = [&](int step, int g, int c) {
                f32x4 &to = s[step % (4 / kStep) * kStep + g][c];
                const u32x2 dk = d[step & 1][g];
#pragma unroll
                for (int r = 0; r < 4; ++r) to[r] = fmaf(r & 1 ? high_half(dk[r / 2]) : low_half(dk[r / 2]), acc[step & 1][g][c][r], to[r]);
            };
            const auto fetch = [&](int step) {
                const int b = step / (4 / kStep), g0 = step % (4 / kStep) * kStep;
                if (g0 == 0) {
#pragma unroll
                    for (int c = 0; c < NQ; ++c) {
                        qh[c] = __builtin_bit_cast(half8, shared.q[A::kApart ? wave : 0][b][c][0][lane]);
                        ql[c] = __builtin_bit_cast(half8, shared.q[A::kApart ? wave : 0][b][c][1][lane]);
                    }
                }
#pragma unroll
                for (int g = 0; g < kStep; ++g) d[step & 1][g] = *reinterpret_cast<const u32x2 *>(&lds.k_scale[b][16 * (g0 + g) + 4 * part]);
            };
#pragma unroll
            for (int g = 0; g < kStep; ++g) code(0, g);
#pragma unroll
            for (int step = 0; step < kSteps; ++step) {
                fetch(step);
                constexpr int kProducts = 2 * kStep * NQ, kPieces = kStep + kStep * NQ;
#pragma unroll
                for (int i = 0; i < kProducts; ++i) {
                    const int half = i / (kStep * NQ), g = i % (kStep * NQ) / NQ, c = i % NQ;
                    f32x4 &to = acc[step & 1][g][c];
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes[step & 1][g], half ? qh[c] : ql[c], half ? to : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                    for (int x = i * kPieces / kProducts; x < (i + 1) * kPieces / kProducts; ++x) {
                        if (x < kStep) {
                            if (step + 1 < kSteps) code(step + 1, x);
                        } else if (step > 0) {
                            add(step - 1, (x - kStep) / NQ, (x - kStep) % NQ);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int x = 0; x < kStep * NQ; ++x) add(kSteps - 1, x / NQ, x % NQ);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int c = 0; c < NQ; ++c) pin(s[g][c]);
        // The keys' codes have come, so the values' have, which were asked for before them.
        if (kAhead) load_v(buffer ^ 1, rows);
        else load_v(0, rows_now);
        load_k();
        // ---- weights ----
        const bool edge = A::kSees == kPrefix ? here.own >= 0 || bad_now
                                              : t0 + kTile - 1 > it.lo || (a.window && t0 <= it.hi - a.window) || t0 < it.see || bad_now;
        u32x4 p_hi[2][NQ], p_lo[2][NQ];
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
            float times = q_unit[c], plus = 0.f, lift = 0.f;     // a score is s * times + plus; lift: plus in powers of two, under infinity
            if constexpr (A::kSees == kBiased) {
                const bool before = t0 + kTile - 1 - it.at <= -a.reach, behind = t0 - (it.at + it.count - 1) >= a.reach;
                if (before || behind) {              // out of reach of all rows: one bias a head
                    const int slot = c * 16 + col, token = token_of(a, slot), head = token < it.count ? min(slot - token * a.split, heads - 1) : 0;
                    plus = shared.bias[head * bias_room(a.reach) + (before ? 0 : bias_room(a.reach) - 1)] * (kLog2e / kScoreBits<A>);
                    if (__ballot(plus == -INFINITY)) {
#pragma unroll
                        for (int g = 0; g < 4; ++g)
#pragma unroll
                            for (int r = 0; r < 4; ++r) s[g][c][r] = plus == -INFINITY ? -INFINITY : s[g][c][r];
                        plus = plus == -INFINITY ? 0.f : plus;
                    }
                    lift = plus * kScoreBits<A>;         // (a row with a larger bias that has seen any of its tokens is far, see below; of others all are masked here)
                    lift = lift > 3.402823466e38f ? 3.402823466e38f : lift;
                } else {
                    const float *const bias = shared.bias + (own_bias[c] + t0 + 4 * part);
#pragma unroll
                    for (int g = 0; g < 4; ++g)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float b = bias[16 * g + r];
                            s[g][c][r] = b == -INFINITY ? b : fmaf(b, kLog2e / kScoreBits<A>, s[g][c][r] * times);
                        }
                    times = 1.f;
                }
            }
            if (edge) {
                int last = pos[c] - t0 - 4 * part;                             // of the lane's tokens 16 g + r
                if constexpr (A::kSees == kPrefix) last = here.own >= 0 && own_seq[c] != here.own ? -1 : last;
                const int behind = A::kSees != kPrefix && a.window ? last - a.window : -kTile;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const bool there = !((bad_now >> g) & 1);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        s[g][c][r] = 16 * g + r <= last && 16 * g + r > behind && there ? s[g][c][r] : -INFINITY;
                }
            }
            if (strange) {
                uint32_t seen = 0;      // bit 4 g + r: the lane's token r of group g
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int r = 0; r < 4; ++r) seen |= (s[g][c][r] != -INFINITY ? 1u : 0u) << (4 * g + r);
#pragma unroll
                for (int b = 0; b < B; ++b) {
                    const uint64_t own = strange_of[b] >> (4 * part);     // bit 16 g + r
                    const uint32_t bits = (uint32_t)(own & 15) | (uint32_t)(own >> 12 & 0xf0) | (uint32_t)(own >> 24 & 0xf00) | (uint32_t)(own >> 36 & 0xf000);
                    poison |= (seen & bits ? 1u : 0u) << (8 * c + b);
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; ++g) top = fmaxf(top, fmaxf(fmaxf(s[g][c][0], s[g][c][1]), fmaxf(s[g][c][2], s[g][c][3])));
            if constexpr (A::kSees == kBiased) top = fmaf(top, times, plus);
            else top *= q_unit[c];
            float back = shrink;
            if (__ballot(top > limit[c])) {
                const float m = fmaxf(st.m[c], max_xor(top));
                const float f = m == st.m[c] ? 1.f : __builtin_amdgcn_exp2f((st.m[c] - m) * kScoreBits<A>);
                st.l[c] *= f;
                back *= f;
                st.m[c] = m;
                const bool plain = fabsf(m) < kFar / kScoreBits<A>, far = !plain && m != -INFINITY;
                base[c] = plain ? m * kScoreBits<A> - kBias : -kBias;
                limit[c] = plain ? m + kSlack / kScoreBits<A> : -INFINITY;
                if (__builtin_expect(__ballot(far) != 0, 0)) {
#pragma unroll
                    for (int g = 0; g < 4; ++g)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            // (plus - m is exact where it matters.  m is rounded, scores beside a large bias are not: they may pass it by half a step of fp32)
                            const float x = fmaf(s[g][c][r], times, plus - m);
                            s[g][c][r] = !far ? s[g][c][r] : x > kSlack / kScoreBits<A> ? kSlack / kScoreBits<A> : x;
                        }
                    times = far ? 1.f : times;
                    lift = far ? 0.f : lift;
                }
            }
            if (__ballot(back != 1.f)) {
#pragma unroll
                for (int x = 0; x < T; ++x)
#pragma unroll
                    for (int r = 0; r < 4; ++r) st.o[x][c][r] *= back;
            }
            const float off = A::kSees == kBiased ? lift - base[c] : -base[c], by = times * kScoreBits<A>;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s[g][c][r] = __builtin_amdgcn_exp2f(fmaf(s[g][c][r], by, off));
                st.l[c] += (s[g][c][0] + s[g][c][1]) + (s[g][c][2] + s[g][c][3]);
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const uint32_t hi = half_pair(s[g][c][r], s[g][c][r + 1]);
                    p_hi[g / 2][c][(g & 1) * 2 + r / 2] = hi;
                    p_lo[g / 2][c][(g & 1) * 2 + r / 2] = half_pair(fmaf(low_half(hi), minus, s[g][c][r]), fmaf(high_half(hi), minus, s[g][c][r + 1]));
                }
            }
        }
        if (!up) __builtin_amdgcn_s_setprio(1);
        // ---- values ----
        // The lane's dimension is lane % 16 of 16; its eight tokens of either half of the tile are those of its scores.  It names the
        // row that nibble lane % 16 of the result comes from: nibbles i and i + 4 of a word, which one and takes together, are neighbours.
        if (!kAhead) {           // the keys' loads, which went out behind the values', may still be on their way
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(B) : "memory");
        }
        const int jj = col & 7, k = (jj & 3) * 2 + (jj >> 2);
        const int from_token = 32 * (col >> 3) + 16 * (k >> 2) + 4 * part + (k & 3);
        // A step is kWide times 16 dimensions; behind each of its products goes a piece of the next step's values, made of codes and
        // scales that were asked of LDS a step earlier.  A piece is one register of both halves in four instructions, and overlaps
        // with its neighbours: none waits for the one before it.
        constexpr int kWide = NQ == 1 ? 2 : 1, kRounds = T / kWide, kUnits = 8 * kWide;
        {
            u32x4 v_hi[2][kWide][2], v_lo[2][kWide][2];
            i32x2 raw[2][kWide];
            u32x2 d[2][4];       // scales of the lane's tokens of a group of 16
            uint32_t big[kUnits];
            half2v code[kUnits];
            const auto fetch = [&](int step) {
                const int b = step * kWide / 2;
#pragma unroll
                for (int k = 0; k < kWide; ++k)
                    raw[step & 1][k] = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                        (__attribute__((address_space(3))) i32x2 *)(lds.v[buffer] + value_at<D>(from_token, b) + 8 * ((step * kWide + k) & 1)));
#pragma unroll
                for (int g = 0; g < 4; ++g) d[step & 1][g] = *reinterpret_cast<const u32x2 *>(&lds.v_scale[b][16 * g + 4 * part]);
            };
            // unit u: register u % 4 of half u / 4 % 2 of 16 dimensions u / 8
            const auto lift = [&](int step, int u) {
                const uint32_t w = (uint32_t)raw[step & 1][u / 8][u / 4 % 2];
                big[u] = (((u & 2) ? w >> 8 : w) & ((u & 1) ? mask1 : mask0)) | magic;         // 1024 + n, or 1024 + 16 n
            };
            const auto center = [&](int u) {
                const half2v b = __builtin_bit_cast(half2v, big[u]);
                code[u] = u & 1 ? __builtin_elementwise_fma(b, half2v{(_Float16)0.0625f, (_Float16)0.0625f}, half2v{(_Float16)-72.f, (_Float16)-72.f})
                                : b - half2v{(_Float16)1032.f, (_Float16)1032.f};
            };
            const auto scale = [&](int step, int u) { return __builtin_bit_cast(half2v, (uint32_t)d[step & 1][2 * (u / 4 % 2) + (u % 4 >> 1)][u & 1]); };
            const auto high = [&](int step, int u) { v_hi[step & 1][u / 8][u / 4 % 2][u % 4] = __builtin_bit_cast(uint32_t, code[u] * scale(step, u)); };
            const auto low = [&](int step, int u) {
                v_lo[step & 1][u / 8][u / 4 % 2][u % 4] =
                    __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code[u], scale(step, u), -__builtin_bit_cast(half2v, (uint32_t)v_hi[step & 1][u / 8][u / 4 % 2][u % 4])));
            };
            const auto piece = [&](int step, int u) {
                if (u == 0) {
                    lift(step, 0);
                    lift(step, 1);
                    center(0);
                }
                if (u + 2 < kUnits) lift(step, u + 2);
                high(step, u);
                if (u + 1 < kUnits) center(u + 1);
                low(step, u);
            };
            fetch(0);
            fetch(1);
#pragma unroll
            for (int u = 0; u < kUnits; ++u) piece(0, u);
#pragma unroll
            for (int step = 0; step < kRounds; ++step) {
                if (step + 2 < kRounds) fetch(step + 2);
                __builtin_amdgcn_sched_barrier(0);
                constexpr int kProducts = 6 * kWide * NQ;
#pragma unroll
                for (int x = 0; x < kProducts; ++x) {
                    const int c = x % NQ, k = x / NQ % kWide, i = x / (NQ * kWide) % 3, h = x / (NQ * kWide * 3);
                    const half8 v = __builtin_bit_cast(half8, i == 0 ? v_lo[step & 1][k][h] : v_hi[step & 1][k][h]);
                    const half8 p = __builtin_bit_cast(half8, i == 1 ? p_lo[h][c] : p_hi[h][c]);
                    f32x4 &o = st.o[step * kWide + k][c];
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p, o, 0, 0, 0);
                    if (step + 1 < kRounds) {
#pragma unroll
                        for (int u = x * kUnits / kProducts; u < (x + 1) * kUnits / kProducts; ++u) piece(step + 1, u);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        wave_sync();
        if (kAhead) buffer ^= 1;
    }
    __builtin_amdgcn_s_setprio(3);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last codes asked for have to be in LDS before it is used for something else
    if (bad_page) atomicOr(a.error, kKvBadPage);
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        st.l[c] = add_xor32(add_xor16(st.l[c]));
        uint32_t p = poison >> (8 * c) & 0xffu, u, w;
        swap16(p, u, w);
        p = u | w;
        swap32(p, u, w);
        p = u | w;
#pragma unroll
        for (int x = 0; x < T; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) st.o[x][c][r] = (p >> (x / 2)) & 1 ? NAN : ldexpf(st.o[x][c][r], unit);
    }
}

// Parts go from one workgroup to another past the caches of their XCDs: stores and loads of device scope, which reach the memory that all of
// them share.  (With ordinary ones and fences, every fence writes back or drops a whole L2: a token of 131072 took 149 us, like this 45.)
__device__ __forceinline__ void store_part(float *p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void store_part(f32x4 *p, f32x4 v) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        __hip_atomic_store(reinterpret_cast<uint64_t *>(p) + i, __builtin_bit_cast(uint64_t, f32x2{v[2 * i], v[2 * i + 1]}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_part(const float *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ f32x4 load_part(const f32x4 *p) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x2 x = __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<const uint64_t *>(p) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        v[2 * i] = x[0], v[2 * i + 1] = x[1];
    }
    return v;
}

// One more part of an item is written; how many there are.  The call before has left the word at this call's number and no part.  A word that holds
// anything else (calls of one context that ran at once, lengths that changed during a call) is begun anew by whoever meets it first, and each
// part is counted once all the same: those that met the old word come here again, those that come later find the new one.
__device__ __forceinline__ uint32_t arrive(uint64_t *word, uint32_t call) {
    const uint64_t was = __hip_atomic_fetch_add(word, (uint64_t)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if ((uint32_t)(was >> 32) == call) return (uint32_t)was + 1;
    uint64_t now = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), next;
    do {
        next = (uint32_t)(now >> 32) == call ? now + 1 : ((uint64_t)call << 32) + 1;
    } while (!__hip_atomic_compare_exchange_strong(word, &now, next, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    return (uint32_t)next;
}

// What a workgroup of a call that counts parts does once: the next call's words, in the half that this call does not use, and the calls' number.  Its
// slots are its own and its share of those that the grid has no workgroup for, so that every slot goes on whatever the grids are; and by an addition,
// so that calls which ran at once, and may have spoiled each other's results, leave all numbers alike.
template <typename A>
__device__ __forceinline__ void advance(const A &a, uint32_t call) {
    uint64_t *const next = a.arrived + (call & 1 ? 0 : a.slots);
    for (uint32_t i = threadIdx.x; i <= (uint32_t)a.slots_each; i += 64) {
        const uint32_t slot = i ? gridDim.x + blockIdx.x * a.slots_each + i - 1 : blockIdx.x;
        if (slot >= (uint32_t)a.slots) break;
        __hip_atomic_store(next + slot, (uint64_t)(call + 1) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_fetch_add(a.calls + slot, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
constexpr uint32_t kFirstCall = 0x9e3779b9u;     // (the number of a call that finds zeros: no word of zeros is taken for counted)

// rows of an item from sums: lane's column of 16 queries, 4 dimensions of 16
template <int D, int NQ, typename A>
__device__ __forceinline__ float *out_row(const A &a, const Row &r, int head0, int lane) {
    return a.y + (int64_t)r.row * a.y_stride + (int64_t)(head0 + (r.live ? r.head : 0)) * D + 4 * (lane >> 4);
}

// The waves' sums of an item: every wave adds a quarter of the dimensions, and writes rows of the result, or a part of one.
template <int D, int NQ, typename A>
__device__ __forceinline__ void meet(const A &a, const Item &it, int head0, int heads, const Running<D, NQ> &st, bool whole, float *part, SharedLds<D, NQ, A> &lds,
                                     int wave, int lane) {
    constexpr int T = D / 16, kMeet = T / meet_rounds(D);
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
        const Row r = row_of(a, it, heads, g * 16 + (lane & 15), lds, wave);
        const bool live = r.live;
        float *y = out_row<D, NQ>(a, r, head0, lane);
#pragma unroll
        for (int t0 = 0; t0 < T; t0 += kMeet) {
            __syncthreads();
            if (lane < 16) {
                lds.meet.m[wave][lane] = st.m[g];
                lds.meet.l[wave][lane] = st.l[g];
            }
#pragma unroll
            for (int t = 0; t < kMeet; ++t) lds.meet.o[wave][t][lane] = st.o[t0 + t][g];
            __syncthreads();
            if (live) {
                float m = -INFINITY, l = 0.f, f[kWaves];
#pragma unroll
                for (int w = 0; w < kWaves; ++w) m = fmaxf(m, lds.meet.m[w][lane & 15]);
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const float mw = lds.meet.m[w][lane & 15];
                    f[w] = mw == m ? 1.f : __builtin_amdgcn_exp2f((mw - m) * kScoreBits<A>);
                    l += lds.meet.l[w][lane & 15] * f[w];
                }
                const float unit = whole ? (l != 0.f ? 1.f / l : 0.f) : 1.f;
                for (int t = wave; t < kMeet; t += kWaves) {
                    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) {
                        const f32x4 x = lds.meet.o[w][t][lane];
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] += x[r] * f[w];
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] *= unit;
                    if (whole) *reinterpret_cast<f32x4 *>(y + 16 * (t0 + t)) = v;
                    else store_part(reinterpret_cast<f32x4 *>(part) + ((t0 + t) * NQ + g) * 64 + lane, v);
                }
                if (!whole && wave == 0 && lane < 16) {
                    store_part(part + 16 * NQ * D + g * 16 + lane, m);
                    store_part(part + 16 * NQ * D + (NQ + g) * 16 + lane, l);
                }
            }
        }
    }
}

// Rows of a wave that is apart.
template <int D, int NQ, typename A>
__device__ __forceinline__ void finish(const A &a, const Item &it, int head0, int heads, const Running<D, NQ> &st, SharedLds<D, NQ, A> &lds, int wave, int lane) {
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
        const Row r = row_of(a, it, heads, g * 16 + (lane & 15), lds, wave);
        float *const y = out_row<D, NQ>(a, r, head0, lane);
        const float unit = st.l[g] != 0.f ? 1.f / st.l[g] : 0.f;
        if (!r.live) continue;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) *reinterpret_cast<f32x4 *>(y + 16 * t) = f32x4{st.o[t][g][0] * unit, st.o[t][g][1] * unit, st.o[t][g][2] * unit, st.o[t][g][3] * unit};
    }
}

// An item that was cut into a few parts, which stretches first .. first + parts - 1 wrote: their sums.  The waves share the dimensions; a part
// comes from far away, so several are asked for at a time.
template <int D, int NQ, typename A>
__device__ __forceinline__ void join_parts(const A &a, const Item &it, int head0, int heads, int first, int parts, SharedLds<D, NQ, A> &lds, int wave, int lane) {
    constexpr int T = D / 16, kMine = (T + kWaves - 1) / kWaves, kBatch = 4, kM = 16 * NQ * D, kL = kM + 16 * NQ;
    const int col = lane & 15;
    const int64_t size = part_floats(D, NQ);
    const auto part = [&](int w) { return a.parts + ((int64_t)(first + w) * 2 + (w ? 0 : 1)) * size; };   // (the first is a stretch's second)
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
        const Row r = row_of(a, it, heads, g * 16 + (lane & 15), lds, wave);
        const bool live = r.live;
        float *y = out_row<D, NQ>(a, r, head0, lane);
        float m = -INFINITY;
        for (int w = wave * 4 + (lane >> 4); live && w < parts; w += 4 * kWaves) m = fmaxf(m, load_part(part(w) + kM + g * 16 + col));
        m = max_xor(m);
        __syncthreads();
        if (lane < 16) lds.meet.m[wave][lane] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, lds.meet.m[w][col]);
        if (live) {
            float l = 0.f;
            f32x4 o[kMine];
#pragma unroll
            for (int t = 0; t < kMine; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int w0 = 0; w0 < parts; w0 += kBatch) {
                float mw[kBatch], lw[kBatch];
                f32x4 v[kBatch][kMine];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {       // (behind the last part that part again, with no weight)
                    const float *p = part(min(w0 + k, parts - 1));
                    mw[k] = load_part(p + kM + g * 16 + col);
                    lw[k] = load_part(p + kL + g * 16 + col);
#pragma unroll
                    for (int t = 0; t < kMine; ++t) v[k][t] = load_part(reinterpret_cast<const f32x4 *>(p) + (min(t * kWaves + wave, T - 1) * NQ + g) * 64 + lane);
                }
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    if (w0 + k >= parts) break;
                    const float f = mw[k] == m ? 1.f : __builtin_amdgcn_exp2f((mw[k] - m) * kScoreBits<A>);
                    l += lw[k] * f;
#pragma unroll
                    for (int t = 0; t < kMine; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[t][r] += v[k][t][r] * f;
                }
            }
            const float unit = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
            for (int t = 0; t < kMine; ++t)
                if (t * kWaves + wave < T)
                    *reinterpret_cast<f32x4 *>(y + 16 * (t * kWaves + wave)) = f32x4{o[t][0] * unit, o[t][1] * unit, o[t][2] * unit, o[t][3] * unit};
        }
    }
}

template <int D, int NQ, typename A>
__global__ __launch_bounds__(kThreads, kPerCu) void attention_kernel(const A) {
    const A &a = fresh_arguments<A>();
    fetch_arguments<void(A), sizeof(A)>();
    __shared__ __align__(16) SharedLds<D, NQ, A> lds;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), id = threadIdx.x;
    const int units = units_of(a), per = (units + kThreads - 1) / kThreads;
    // ---- the line of turns ----
    int turns_mine = 0, items_mine = 0, longest = 0;
    each_item(a, id, units, per, [&](int s, int tile, const Sequence &q, int n) {
        const int item[6] = {s, tile, n, q.start, q.count, q.len};
        if (per == 1) {
#pragma unroll
            for (int i = 0; i < 6; ++i) lds.only[i][id] = item[i];
        }
        turns_mine += n;
        ++items_mine;
        longest = max(longest, n);
        return A::kSees == kPrefix && items_mine > a.most_items;     // (groups that do not ascend could have any number of items, whose sequences are looked at)
    }, [&](int) {
        if (blockIdx.x == 0) atomicOr(a.error, A::kSees == kPrefix ? kKvBadGroups : kKvBadRows);
    });
    int turns_before = wave_scan(turns_mine), items_before = wave_scan(items_mine);
    longest = (int)wave_max((uint32_t)longest);
    if (lane == 63) {
        lds.waves[wave][0] = turns_before;
        lds.waves[wave][1] = items_before;
        lds.waves[wave][2] = longest;
    }
    // (behind the lengths, which would be waited for with it, and to LDS, where it takes no register while tiles are worked on)
    const bool counted = a.arrived != nullptr;
    if (counted && id == 0) global_to_lds4_unseen(a.calls + blockIdx.x, &lds.call);
    const auto call = [&]() {     // behind a wait for the wave's loads
        return (uint32_t)uniform((int)*(volatile __attribute__((address_space(3))) uint32_t *)&lds.call) + kFirstCall;
    };
    bool advanced = !counted || wave != 0;
    const auto leave = [&](const A &a) {
        if (advanced) return;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        advance(a, call());
        advanced = true;
    };
    turns_before -= turns_mine, items_before -= items_mine;
    __syncthreads();
    int head_turns = 0, head_items = 0;
    longest = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) turns_before += lds.waves[w][0], items_before += lds.waves[w][1];
        head_turns += lds.waves[w][0];
        head_items += lds.waves[w][1];
        longest = max(longest, lds.waves[w][2]);
    }
    head_turns = uniform(head_turns), head_items = uniform(head_items), longest = uniform(longest);
    if (__builtin_expect(head_items > a.most_items, 0)) {      // (q_start falls somewhere: reported above)
        const A &a = fresh_arguments<A>();
        if (!a.arrived)                                        // nothing is to be joined
            for (int i = id; i < units_of(a) * a.kv.n_head * a.splits; i += kThreads) a.joins[2 * i] = -1;
        return leave(a);
    }
    const Line line = line_of(head_turns, head_items, longest, a.kv.n_head * a.splits, gridDim.x, A::kSees != kBefore, A::kApart);
    lds.line[id][0] = line.whole ? items_before : turns_before + line.start * items_before;   // (each thread's own: kept out of the registers
    lds.line[id][1] = line.whole ? items_mine : turns_mine + line.start * items_mine;         // that the tiles want)
    const uint32_t me = line.whole ? blockIdx.x : stretch_of_block(blockIdx.x, line.active);
    if (me >= line.active) return leave(a);
    uint32_t at = line.whole ? me : me * line.length + std::min(me, line.longer);
    const uint32_t end = line.whole ? line.total : at + line.length + (me < line.longer ? 1 : 0);
    uint32_t round = 0;

    // whoever has the place `at` writes down its item
    const auto seek = [&](uint32_t at, int32_t *found) {
        const int off = (int)(at - quotient(at, (uint32_t)line.head_length) * line.head_length);
        const int before = lds.line[id][0], mine = lds.line[id][1];
        if (off < before || off >= before + mine) return;     // one thread
        int b = before;
        if (per == 1) {
            int item[6];        // (read before any is written: one trip instead of six)
#pragma unroll
            for (int i = 0; i < 6; ++i) item[i] = lds.only[i][id];
#pragma unroll
            for (int i = 0; i < 6; ++i) found[i] = item[i];
        } else {
            bool there = false;
            each_item(a, id, units, per, [&](int s, int tile, const Sequence &q, int n) {
                const int weight = line.whole ? 1 : n + line.start;
                if (off >= b + weight) {
                    b += weight;
                    return false;
                }
                const int item[6] = {s, tile, n, q.start, q.count, q.len};
#pragma unroll
                for (int i = 0; i < 6; ++i) found[i] = item[i];
                there = true;
                return true;
            }, [](int) {});
            if (!there) b = -1;      // (lengths that another stream changes meanwhile)
        }
        found[6] = b;
    };
    // Of 32 rows an item the next one is looked for before this one's tiles, so that nothing waits for it behind them: two prompts of 500 behind 100 to
    // 900, heads of 96 with a bias, 60.8 us instead of 65.0, 512 prompt tokens 20.9 instead of 21.5, drawn ones up to 3% less.  Of 16 it is not: the second copy of
    // the search costs tokens, which have one item a workgroup, 1%.
    constexpr bool kEarly = NQ == 2;
    int turn = 0;
    if (kEarly) {
        if (at < end) seek(at, lds.found[0]);
        __syncthreads();
    }
    while (at < end) {
        const int hv = (int)quotient(at, (uint32_t)line.head_length), off = (int)(at - (uint32_t)hv * line.head_length);
        if (!kEarly) {
            seek(at, lds.found[0]);
            __syncthreads();
        }
        const int32_t *const found = lds.found[kEarly ? turn : 0];
        const int seq = uniform(found[0]), row_tile = uniform(found[1]), turns = uniform(found[2]), first = uniform(found[6]);
        if (first < 0) break;
        const Sequence q = {uniform(found[3]), uniform(found[4]), uniform(found[5])};
        const Item it = item_of(a, seq, q, row_tile);
        const A &a = fresh_arguments<A>();
        const int kv_head = a.splits == 1 ? hv : hv / a.splits, go = hv - kv_head * a.splits;
        const int head0 = kv_head * a.group + go * a.split, heads = min(a.split, a.group - go * a.split);
        const int skip = off - first;
        const uint32_t begin = at - skip;     // of the item
        const Piece piece = piece_of(line, skip, turns, end - at);
        if (piece.to <= 0) break;
        const auto move_on = [&]() {
            ++round, turn ^= 1;
            at = line.whole ? round * line.active + (round & 1 ? line.active - 1 - me : me) : at + piece.take;
        };
        if (kEarly) {
            move_on();
            if (at < end) seek(at, lds.found[turn]);
        }
        const Members seqs = members<D, NQ>(a, it, lds, wave, lane);
        const int tile0 = A::kSees == kPrefix || it.hi < 0 ? 0 : it.see / kTile;
        const int tile1 = tile0 + min(piece.to * kWaves, A::kSees == kPrefix ? max(1, seqs.tiles) : item_tiles(it));

        Running<D, NQ> st;
        if constexpr (A::kApart) {      // whole items only
            const Item mine = item_of_wave(a, it, wave);
            walk<D, NQ>(a, mine, seqs, kv_head, head0, heads, tile0, min(tile0 + turns, mine.hi / kTile + 1), lds, wave, st, lane);
            leave(a);
            finish<D, NQ>(fresh_arguments<A>(), mine, head0, heads, st, lds, wave, lane);
        } else {
            walk<D, NQ>(a, it, seqs, kv_head, head0, heads, tile0 + piece.from * kWaves + wave, tile1, lds, wave, st, lane);
            leave(a);                       // (here, so that nothing waits for it)
            // ---- the waves' sums ----
            const bool starts = piece.from == 0, ends = piece.to == turns;
            meet<D, NQ>(fresh_arguments<A>(), it, head0, heads, st, starts && ends, fresh_arguments<A>().parts + ((int64_t)me * 2 + (starts ? 1 : 0)) * part_floats(D, NQ), lds, wave, lane);
            const A &c = fresh_arguments<A>();
            if (!c.arrived) {            // whoever writes an item's end says what is to be joined
                if (ends && id == 0) {
                    int32_t *const join = c.joins + 2 * ((int64_t)hv * units_of(c) + seq * c.row_tiles + row_tile);
                    join[0] = starts ? -1 : (int32_t)stretch_at(line, begin + line.start);
                    join[1] = (int32_t)me;
                }
            } else if (!(starts && ends)) {
                // The part is in memory before it is counted (the wait is for the stores); whoever counts the last one loads them after that.
                const int first = (int)stretch_at(line, begin + line.start), parts = (int)stretch_at(line, begin + line.start + turns - 1) - first + 1;
                const uint32_t number = call();
                uint64_t *const word = c.arrived + (number & 1 ? c.slots : 0) + first;
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (id == 0) lds.last = arrive(word, number) == (uint32_t)parts;
                __syncthreads();
                if (lds.last) join_parts<D, NQ>(c, it, head0, heads, first, parts, lds, wave, lane);
            }
        }
        if (!kEarly) move_on();
        if (at < end) __syncthreads();
    }
    leave(fresh_arguments<A>());
}

// Items that were cut into many parts: the sums of stretches first .. last.  A workgroup takes 16 queries and 16
// dimensions; its waves take the parts in turn, four at a time (their loads go out together: a part comes from another XCD's memory), and meet once.
constexpr int kJoinWaves = 8;

template <int D, int NQ, typename A>
__global__ __launch_bounds__(64 * kJoinWaves) void attention_join_kernel(const A a) {
    constexpr int kBatch = 4, kM = 16 * NQ * D, kL = kM + 16 * NQ;
    __shared__ __align__(16) f32x4 sums[kJoinWaves][64];
    __shared__ float tops[kJoinWaves][16], weights[kJoinWaves][16];
    const int32_t *j = a.joins + 2 * (int64_t)blockIdx.x;
    const int first = j[0], last = j[1], units = units_of(a);
    const int hv = blockIdx.x / units, s = (blockIdx.x - hv * units) / a.row_tiles, row_tile = blockIdx.x - hv * units - s * a.row_tiles;
    bool bad;
    const Item it = item_of(a, s, unit_of(a, s, bad), row_tile);
    if (it.count <= 0 || first < 0) return;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15;
    const int x = blockIdx.y / NQ, g = blockIdx.y % NQ, parts = last - first + 1;
    const auto part = [&](int w) { return a.parts + ((int64_t)(first + w) * 2 + (w ? 0 : 1)) * part_floats(D, NQ); };   // (the first is a stretch's second)
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    for (int w0 = wave; w0 < parts; w0 += kBatch * kJoinWaves) {
        float mw[kBatch], lw[kBatch];
        f32x4 v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {       // (behind the last part the first of the batch again, with no weight)
            const int w = w0 + k * kJoinWaves;
            const float *p = part(w < parts ? w : w0);
            mw[k] = p[kM + g * 16 + col];
            lw[k] = p[kL + g * 16 + col];
            v[k] = reinterpret_cast<const f32x4 *>(p)[(x * NQ + g) * 64 + lane];
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) top = fmaxf(top, mw[k]);
        const float back = m == top ? 1.f : __builtin_amdgcn_exp2f((m - top) * kScoreBits<A>);
        m = top;
        l *= back;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] *= back;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (w0 + k * kJoinWaves >= parts) break;
            const float f = mw[k] == m ? 1.f : __builtin_amdgcn_exp2f((mw[k] - m) * kScoreBits<A>);
            l += lw[k] * f;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] += v[k][r] * f;
        }
    }
    if (lane < 16) tops[wave][lane] = m, weights[wave][lane] = l;
    sums[wave][lane] = o;
    __syncthreads();
    if (wave != 0) return;
    const int kv_head = hv / a.splits, go = hv - kv_head * a.splits, heads = min(a.split, a.group - go * a.split);
    const int token = token_of(a, g * 16 + col);
    Row r{};
    r.head = g * 16 + col - token * a.split;
    if constexpr (A::kSees == kPrefix) {
        const int member = (int)((uint32_t)token * a.row_part >> 16), i = token - member * a.max_q;
        if (token >= a.tokens || member >= it.count || r.head >= heads) return;
        const Sequence q = sequence(a, it.seq + member, bad);
        r.live = i < q.count;
        r.row = q.start + i;
    } else {
        r.live = token < it.count && r.head < heads;
        r.row = it.first + token;
    }
    if (!r.live) return;
    float *y = out_row<D, NQ>(a, r, kv_head * a.group + go * a.split, lane);
    const int used = min(kJoinWaves, parts);
    m = -INFINITY, l = 0.f;
    for (int w = 0; w < used; ++w) m = fmaxf(m, tops[w][col]);
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < used; ++w) {
        const float f = tops[w][col] == m ? 1.f : __builtin_amdgcn_exp2f((tops[w][col] - m) * kScoreBits<A>);
        const f32x4 v = sums[w][lane];
        l += weights[w][col] * f;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] += v[r] * f;
    }
    const float unit = l != 0.f ? 1.f / l : 0.f;
    *reinterpret_cast<f32x4 *>(y + 16 * x) = f32x4{o[0] * unit, o[1] * unit, o[2] * unit, o[3] * unit};
}

template <int D, int NQ, typename A>
hipError_t launch(const A &a, int groups, int places, hipStream_t s) {
    hipLaunchKernelGGL((attention_kernel<D, NQ, A>), dim3(groups), dim3(kThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    if constexpr (!A::kApart) {      // (whose items stay whole)
        if (e != hipSuccess || a.arrived) return e;
        hipLaunchKernelGGL((attention_join_kernel<D, NQ, A>), dim3(places, D / 16 * NQ), dim3(64 * kJoinWaves), 0, s, a);
        return hipGetLastError();
    }
    return e;
}

// numbers of calls and counts of parts, what the joining kernel is to do, then the parts; zeros before the first call
inline size_t counts_bytes(int cus) { return (size_t)cus * kPerCu * 2 * 8; }
inline size_t calls_bytes(int cus) { return ((size_t)cus * kPerCu * 4 + 255) / 256 * 256; }
inline size_t joins_bytes(int cus) { return (size_t)cus * kPerCu * 8; }
inline size_t head_bytes(int cus) { return counts_bytes(cus) + calls_bytes(cus) + joins_bytes(cus); }

template <typename A>
hipError_t launch_as(const AttentionJob &j, A a, hipStream_t s) {
    if (j.n_tokens == 0 || j.n_seq == 0) return hipSuccess;     // (max_q 0: any row of a sequence is one too many, which the kernel reports)
    a.kv = *j.kv;
    a.q = j.q;
    a.y = j.y;
    a.q_stride = j.q_stride;
    a.y_stride = j.y_stride;
    a.pages_stride = j.pages_stride;
    a.n_tokens = (int32_t)j.n_tokens;
    a.n_seq = (int32_t)j.n_seq;
    a.max_q = (int32_t)j.max_q;
    a.q_start = j.q_start;
    a.kv_len = j.kv_len;
    a.pages = j.pages;
    a.error = j.error;
    a.scale = j.scale * kLog2e / kScoreBits<A>;
    a.window = j.window;
    a.group = j.n_head / j.kv->n_head;
    // 16 rows an item, or 32 of them that share the work of unpacking the codes.  Few rows of work leave most of the chip waiting for a turn of
    // 32, which takes half as long again: 16 up to six turns of 16 rows (and two for their start) a workgroup.  Eight rows behind 4000
    // tokens 14.1 us in sixteens and 17.7 in 32s, 64 rows 28.3 and 33.5; 128 rows 41.3 and 40.7, 128 behind 16000 122 and 103, 512
    // prompt tokens 25.4 and 24.3, 1000 64 and 53.  Heads of 256 leave no registers for 32 at two waves a SIMD, and at one they were slower
    // from 8 rows behind 1000 tokens (28 against 18.5 us) to 512 behind 32000 (838 against 804).
    const int groups_most = kPerCu * j.cus;
    const int64_t most_len = j.pages_stride << j.kv->page_shift;
    double items = 0;
    int cols = A::kApart && a.kv.dim == 64 ? 2 : 1;
    for (;; ++cols) {
        const int rows = 16 * cols;
        a.splits = (a.group + rows - 1) / rows;
        a.split = (a.group + a.splits - 1) / a.splits;
        if constexpr (A::kSees == kBiased) {     // as many heads as there is room for the biases of
            const int most = kBiasFloats / bias_room(a.reach);
            a.splits = std::max(a.splits, (a.group + most - 1) / most);
            a.split = (a.group + a.splits - 1) / a.splits;
            a.splits = (a.group + a.split - 1) / a.split;
        }
        a.split_part = (65536 + a.split - 1) / a.split;
        a.tokens = (A::kApart ? kWaves : 1) * (rows / a.split);
        a.row_tiles = (int32_t)std::max<int64_t>(1, (j.max_q + a.tokens - 1) / a.tokens);
        a.most_items = a.n_tokens / a.tokens + a.n_seq;
        items = std::min((double)a.n_seq * a.row_tiles, (double)a.n_tokens / a.tokens + a.n_seq) * j.kv->n_head * a.splits;
        if constexpr (A::kSees == kPrefix) {     // sequences that an item has the rows of, alike for all items of the largest group
            a.together = std::min({(int32_t)(a.tokens / j.max_q), a.max_group, (int32_t)kTogether});
            if (a.together < 2 && cols == 1 && a.kv.dim <= 128) continue;
            a.row_tiles = (a.max_group + a.together - 1) / a.together;
            a.together = (a.max_group + a.row_tiles - 1) / a.row_tiles;
            a.tokens = a.together * a.max_q;
            a.row_part = (65536 + a.max_q - 1) / a.max_q;
            a.most_items = a.n_seq / a.together + a.n_groups;
            items = std::min((double)a.n_groups * a.row_tiles, (double)a.most_items) * j.kv->n_head * a.splits;
            // 16 columns, where they hold two sequences: a tile of 32 takes 1.77 times as long, and of a sequence's own tokens only its columns are any use.  32
            // save where what is shared is about 26 times as long as what is not (four heads a key/value head, one row).  The host knows neither, only how
            // wide the table is: taken for so where a sequence can have 32768 tokens, so that short ones in such a table pay for the width.  48 sequences behind 8192 tokens with 30 to 1500 of their own 45.0 us in sixteens and 50.2 in 32s, four groups of
            // nine with up to four rows 26.8 and 31.4, 32 sequences behind 65536 with 10 to 400 of their own 126 and 105.
            if (a.max_group * a.max_q * a.group <= 16 || (a.together >= 2 && most_len < 32768)) break;
        }
        const int64_t seen = j.window ? std::min<int64_t>(most_len, (int64_t)j.window + a.tokens) : most_len;
        if (A::kApart || cols == 2 || a.kv.dim > 128 || (A::kSees != kPrefix && j.max_q * a.group <= 16) || items * ((double)seen / (kWaves * kTile) + 2) <= 6. * groups_most) break;
    }
    // no more workgroups than there can be turns
    const int64_t most = (most_len + kTile - 1) / kTile + 1;
    const int64_t places = (int64_t)units_of(a) * j.kv->n_head * a.splits;
    int groups;
    if constexpr (A::kSees == kPrefix) {
        // (an item's sequences may share next to nothing; where they share nearly everything its turns are one's, and if eight parts an item are enough
        // for those, one launch does: two sequences behind 1024 tokens 13.6 us instead of 14.4)
        groups = (int)std::max(1., std::min<double>(groups_most, items * ((double)most * a.together / kWaves + 1)));
        if (groups > 8 * places && items * ((double)most / kWaves + 1) <= 8. * places) groups = (int)(8 * places);
    } else {
        groups = (int)std::max(1., std::min<double>(groups_most, items * (A::kApart ? 1. : (double)most / kWaves + 1)));
    }
    a.parts = reinterpret_cast<float *>(j.scratch + head_bytes(j.cus));
    a.slots = groups_most;
    a.slots_each = (groups_most - groups + groups - 1) / groups;
    // An item is cut into as many parts as there are workgroups for it, one or two more at its ends.  Up to eight, whoever writes the last part
    // adds them: one launch.  More are added by a kernel whose workgroups share the work: for a token of 131072 (64 parts) 45 us against 56,
    // of 8192 13.8 against 19.0, for eight rows behind 6000 17.2 against 22.1; a short chat's token, with two, 14.0 against 11.9.  (Up to five
    // instead of eight: 0.6% more over 50 drawn calls, up to three 2%.)
    // (the joins' list has a place for every item there could be, fewer than groups / 8)
    const bool few_parts = A::kApart || groups <= 8 * places;
    a.arrived = few_parts ? reinterpret_cast<uint64_t *>(j.scratch) : nullptr;
    a.calls = reinterpret_cast<uint32_t *>(j.scratch + counts_bytes(j.cus));
    a.young = few_parts ? j.cus : 0;      // (the second workgroups of the compute units, or all: see walk)
    a.joins = reinterpret_cast<int32_t *>(j.scratch + counts_bytes(j.cus) + calls_bytes(j.cus));
    if (dry_run()) {
        const char *const sees[] = {"", ", all", ", biased", ", prefix"};
        plan_note("attention_kernel<%d, %d%s%s>: %d heads in %d x %d of %d, %d tokens x %d a sequence of rows, grid %d x %d, first from %d on", a.kv.dim, cols, sees[A::kSees], A::kApart ? ", apart" : "", j.n_head,
                  a.kv.n_head, a.splits, a.split, a.tokens, a.row_tiles, groups, kThreads, a.young);
        return hipSuccess;
    }
    if constexpr (A::kApart) {
        if (a.kv.dim == 64) return launch<64, 2, A>(a, groups, (int)places, s);
        if (a.kv.dim == 96) return launch<96, 1, A>(a, groups, (int)places, s);
        if constexpr (A::kSees == kAll) return launch<128, 1, A>(a, groups, (int)places, s);
        return hipErrorInvalidValue;
    } else {
        if (cols == 1) {
            if (a.kv.dim == 64) return launch<64, 1, A>(a, groups, (int)places, s);
            if (a.kv.dim == 96) return launch<96, 1, A>(a, groups, (int)places, s);
            if (a.kv.dim == 128) return launch<128, 1, A>(a, groups, (int)places, s);
            return launch<256, 1, A>(a, groups, (int)places, s);
        }
        if (a.kv.dim == 64) return launch<64, 2, A>(a, groups, (int)places, s);
        if (a.kv.dim == 96) return launch<96, 2, A>(a, groups, (int)places, s);
        return launch<128, 2, A>(a, groups, (int)places, s);
    }
}

// Whether every wave is to have rows of its own, 32 of an item of 128 (of heads wider than 64 16 of one of 64), and go through all tiles.  Otherwise four waves
// share the rows and the tiles, and meet: an item of a short sequence is one or two tiles a wave between finding it, staging its queries and adding the
// waves' sums, some 10000 cycles of 17000.  Apart the queries are found and staged once for four times the rows and nothing is added; an item is as
// long as the tokens it sees, though, stays whole, and there are a quarter as many.  So: where there are items enough for how long they can be, at least
// 32 for every tile, and beyond eight tiles four times as many as tiles for each.  Over 125 batches inside the rule (heads of 64, a bias on both sides or
// causal and cross attention, rows alike and of all lengths) 1.32 times as fast in the mean, 2.07 at best, 0.90 at worst: 64 sequences of 128 on 8 heads 40.4 us ->
// 19.9, 16 of 512 on 16 98 -> 72, 8 of up to 512 on 16 39.5 -> 34.7; outside it 2 of 1024 on 8 24.0 -> 47.4.
// The queries of four waves have to leave room in LDS for a second workgroup: 32 rows a wave of heads of 64, 16 of 96 and, without biases, of 128.  Those tiles' codes are
// unpacked twice as often, which pays up to six tiles: 1.29 times as fast in the mean of 116 batches, 1.04 to 1.77 (64 sequences of 128 on 8 heads of 128 52.8 us ->
// 35.6, 32 of 384 on 16 193 -> 143); of eight tiles 0.8 to 1.34.
inline bool rows_apart(const AttentionJob &j, bool biased) {
    if (j.n_tokens == 0 || j.n_seq == 0 || j.kv->dim > (biased ? 96 : 128)) return false;
    const double rows = (double)j.n_tokens * j.n_head / j.kv->n_head, tiles = std::ceil((double)(j.pages_stride << j.kv->page_shift) / kTile);
    if (j.kv->dim > 64 && tiles > 6) return false;
    return rows >= (j.kv->dim > 64 ? 16. : 32.) * j.n_seq && rows * j.kv->n_head / 128 >= tiles * std::max(32., 4 * tiles);
}

// For the tests: the pieces of the line that every workgroup of a call takes, in the order in which it takes them, worked out on the host by the
// kernel's own arithmetic.  A piece is {workgroup, head, sequence, row tile, its turns from, to, all the item's turns, first and last stretch of the item}.
// Their number, or -1 where a workgroup would not come to an end.  kv_len_later: what the lengths are when an item is looked for.
template <typename A>
int64_t pieces_of(A a, const int32_t *kv_len_later, int heads, int groups, int32_t *out, int64_t room) {
    const int units = units_of(a), per = (units + kThreads - 1) / kThreads;
    struct Thread { int turns_before, items_before, turns, items, only[3]; } threads[kThreads];
    int head_turns = 0, head_items = 0, longest = 0;
    for (int id = 0; id < kThreads; ++id) {
        Thread &t = threads[id];
        t = Thread{head_turns, head_items, 0, 0, {0, 0, 0}};
        each_item(a, id, units, per, [&](int s, int tile, const Sequence &, int n) {
            t.only[0] = s, t.only[1] = tile, t.only[2] = n;
            t.turns += n;
            ++t.items;
            longest = max(longest, n);
            return A::kSees == kPrefix && t.items > a.most_items;
        }, [](int) {});
        head_turns += t.turns, head_items += t.items;
    }
    if (head_items > a.most_items) return 0;
    const Line line = line_of(head_turns, head_items, longest, heads, groups, A::kSees != kBefore, A::kApart);
    a.kv_len = kv_len_later;
    int64_t pieces = 0;
    for (int block = 0; block < groups; ++block) {
        const uint32_t me = line.whole ? block : stretch_of_block(block, line.active);
        if (me >= line.active) continue;
        uint32_t at = line.whole ? me : me * line.length + std::min(me, line.longer);
        const uint32_t end = line.whole ? line.total : at + line.length + (me < line.longer ? 1 : 0);
        uint32_t round = 0;
        int found[4] = {0, 0, 0, 0};
        for (int64_t steps = 0; at < end; ++steps) {
            if (steps > line.total) return -1;
            const int hv = (int)quotient(at, (uint32_t)line.head_length), off = (int)(at - (uint32_t)hv * line.head_length);
            for (int id = 0; id < kThreads; ++id) {
                const Thread &t = threads[id];
                int b = line.whole ? t.items_before : t.turns_before + line.start * t.items_before;
                if (off < b || off >= b + (line.whole ? t.items : t.turns + line.start * t.items)) continue;
                if (per == 1) {
                    found[0] = t.only[0], found[1] = t.only[1], found[2] = t.only[2];
                } else {
                    bool there = false;
                    each_item(a, id, units, per, [&](int s, int tile, const Sequence &, int n) {
                        const int weight = line.whole ? 1 : n + line.start;
                        if (off >= b + weight) {
                            b += weight;
                            return false;
                        }
                        found[0] = s, found[1] = tile, found[2] = n;
                        there = true;
                        return true;
                    }, [](int) {});
                    if (!there) b = -1;
                }
                found[3] = b;
            }
            if (found[3] < 0) break;
            const int turns = found[2], skip = off - found[3];
            const Piece piece = piece_of(line, skip, turns, end - at);
            if (piece.to <= 0) break;
            const uint32_t first = line.whole ? me : stretch_at(line, at - skip + line.start), last = line.whole ? me : stretch_at(line, at - skip + line.start + turns - 1);
            if (pieces < room) {
                const int32_t row[9] = {block, hv, found[0], found[1], piece.from, piece.to, turns, (int32_t)first, (int32_t)last};
                for (int i = 0; i < 9; ++i) out[9 * pieces + i] = row[i];
            }
            ++pieces;
            if (line.whole) {
                ++round;
                at = round * line.active + (round & 1 ? line.active - 1 - me : me);
            } else {
                at += piece.take;
            }
        }
    }
    return pieces;
}

}  // namespace

}  // namespace qproj
