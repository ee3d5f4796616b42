// Causal attention over the paged 4-bit cache: attention_device.h's kernel for rows that see what lies before them.
#include "attention_device.h"

namespace qproj {

size_t attention_scratch_bytes(int cus) {
    return head_bytes(cus) + (size_t)cus * kPerCu * 2 * std::max(part_floats(256, 1), part_floats(128, 2)) * 4;
}
size_t attention_counts_bytes(int cus) { return counts_bytes(cus); }


hipError_t launch_attention(const AttentionJob &j, hipStream_t s) { return launch_as(j, AttentionArgs{}, s); }

// For the tests: the pieces of the line that every workgroup of a call takes, in the order in which it takes them, worked out on the host by the
// kernel's own arithmetic.  A piece is {workgroup, head, sequence, row tile, its turns from, to, all the item's turns, first and last stretch of the item}.
// Their number, or -1 where a workgroup would not come to an end.  kv_len_later: what the lengths are when an item is looked for.
int64_t attention_pieces(const AttentionJob &j, const int32_t *kv_len_later, int64_t most_len, int tokens, int heads, int groups, int32_t *out, int64_t room) {
    AttentionArgs a{};
    a.pages_stride = most_len;      // (pages of one token)
    a.n_tokens = (int32_t)j.n_tokens, a.n_seq = (int32_t)j.n_seq, a.max_q = (int32_t)j.max_q, a.window = j.window;
    a.q_start = j.q_start, a.kv_len = j.kv_len;
    a.tokens = tokens;
    a.row_tiles = std::max(1, (a.max_q + tokens - 1) / tokens);
    a.most_items = a.n_tokens / tokens + a.n_seq;
    const int units = a.n_seq * a.row_tiles, per = (units + kThreads - 1) / kThreads;
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
            return false;
        }, [](int) {});
        head_turns += t.turns, head_items += t.items;
    }
    if (head_items > a.most_items) return 0;
    const Line line = line_of(head_turns, head_items, longest, heads, groups);
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

}  // namespace qproj
