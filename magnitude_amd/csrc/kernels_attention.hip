// Causal attention over the paged 4-bit cache: attention_device.h's kernel for rows that see what lies before them.
#include "attention_device.h"

namespace qproj {

size_t attention_scratch_bytes(int cus) {
    return head_bytes(cus) + (size_t)cus * kPerCu * 2 * std::max(part_floats(256, 1), part_floats(128, 2)) * 4;
}
size_t attention_counts_bytes(int cus) { return counts_bytes(cus); }


hipError_t launch_attention(const AttentionJob &j, hipStream_t s) { return launch_as(j, AttentionArgs{}, s); }

// For the tests, of a causal call: see pieces_of.  kv_len_later: what the lengths are when an item is looked for.
int64_t attention_pieces(const AttentionJob &j, const int32_t *kv_len_later, int64_t most_len, int tokens, int heads, int groups, int32_t *out, int64_t room) {
    AttentionArgs a{};
    a.pages_stride = most_len;      // (pages of one token)
    a.n_tokens = (int32_t)j.n_tokens, a.n_seq = (int32_t)j.n_seq, a.max_q = (int32_t)j.max_q, a.window = j.window;
    a.q_start = j.q_start, a.kv_len = j.kv_len;
    a.tokens = tokens;
    a.row_tiles = std::max(1, (a.max_q + tokens - 1) / tokens);
    a.most_items = a.n_tokens / tokens + a.n_seq;
    return pieces_of(a, kv_len_later, heads, groups, out, room);
}

}  // namespace qproj
