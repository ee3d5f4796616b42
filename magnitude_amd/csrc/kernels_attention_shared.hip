// Causal attention of a batch whose sequences share their first tokens.
//
// An item has the rows of several sequences of a group as its columns.  Its tiles are those that the sequences share, which all columns see, then
// every sequence's own, which the others' columns are masked in: weights, sums and the joining of parts are the other kinds' own,
// and what is shared is read and unpacked once for up to 32 columns instead of once a sequence.  A tile of a sequence's own costs what it costs in an item
// of that sequence alone and as many columns.
//
// What bounds it, as of every kind: the vector units' and the matrix cores' issue slots, 690 vector instructions and 80 products a tile and 16 columns.  48
// sequences behind 8192 tokens with 30 to 1500 of their own (32 heads of 128 on 8, one row) 45.7 us, 54 MB that have to be read; 48 % of a SIMD's
// cycles issue vector instructions, 17 % matrix ones.  The causal kernel, which reads what is shared 48 times, takes 98 us (and where nothing is shared 98 against 107).  32
// behind 65536 with 10 to 400 of their own 106 us (84 MB, 34 Gflop); two behind 1024 13.8; four groups of nine, up to four rows,
// 14 heads of 64 on 7, 26.8.  (Batches of the loads of an item's sequences in the scan, four or eight at a time: level or up to 5 % more.)
#include "attention_device.h"

namespace qproj {

// Whether an item can have the rows of two sequences at least: otherwise they fill it by themselves, and the causal kernel takes them as well.  A layer
// with a window sees nothing of a long prefix.
static bool sharing_pays(const AttentionJob &j, const SharedGroups &g) {
    if (j.window || j.max_q <= 0 || g.max_group < 2 || g.n_groups < 1) return false;
    const int rows = j.kv->dim > 128 ? 16 : 32, group = j.n_head / j.kv->n_head;
    const int splits = (group + rows - 1) / rows, split = (group + splits - 1) / splits;
    if (j.max_q > rows / split / 2) return false;
    if ((double)g.n_groups * (g.max_group + 1) > 2e9) return false;      // places of the line, in 32 bits
    // the line's turns are counted in 32 bits: groups that do not ascend may have any item hold the most sequences
    const double turns = ((double)(j.pages_stride << j.kv->page_shift) / (kWaves * kTile) + 4) * ((double)j.n_seq + (double)kTogether * g.n_groups);
    return turns * j.n_head <= 2e9;
}

hipError_t launch_attention_shared(const AttentionJob &j, const SharedGroups &g, hipStream_t s) {
    if (!sharing_pays(j, g)) return launch_attention(j, s);
    PrefixArgs a{};
    a.group_start = g.start;
    a.shared_len = g.shared;
    a.n_groups = (int32_t)g.n_groups;
    a.max_group = (int32_t)g.max_group;
    return launch_as(j, a, s);
}

// For the tests: as attention_pieces, of groups; `together` sequences an item.  A piece's "sequence" is its group.
int64_t attention_shared_pieces(const AttentionJob &j, const SharedGroups &g, const int32_t *kv_len_later, int64_t most_len, int together, int heads, int groups, int32_t *out,
                                int64_t room) {
    PrefixArgs a{};
    a.group_start = g.start, a.shared_len = g.shared, a.n_groups = (int32_t)g.n_groups, a.max_group = (int32_t)g.max_group;
    a.pages_stride = most_len;      // (pages of one token)
    a.n_tokens = (int32_t)j.n_tokens, a.n_seq = (int32_t)j.n_seq, a.max_q = (int32_t)j.max_q;
    a.q_start = j.q_start, a.kv_len = j.kv_len;
    a.together = together;
    a.row_tiles = std::max(1, (a.max_group + together - 1) / together);
    a.most_items = a.n_seq / together + a.n_groups;
    return pieces_of(a, kv_len_later, heads, groups, out, room);
}

}  // namespace qproj
