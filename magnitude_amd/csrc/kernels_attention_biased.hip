// Attention with a bias of the distance between a token and a row, learned by buckets, and the layout of such biases.
//
// A softmax's exponent is scale * q . k + bias, in powers of two one fma of the score: scale, the bias times log2(e) and what is taken off.  Biases of an item's
// heads lie by distance in LDS, a padded row a head, so that no tile looks for a bucket: a tile within reach of some row reads 16 of them a lane and 16 columns
// at constant offsets from one address, any other tile has one a head.  (A bias of -infinity hides its token, also where the key is not finite: the choice costs 1 to 2 %.)
//
// What bounds it, as of every kind: issue slots, and where sequences are short the finding and staging of items.  Encoders of 16 heads of 64, reach 128: eight
// texts of up to 512 tokens 35.0 us; one of 4096 233 us, 68.7 Gflop (2.5 times that on the matrix cores, as pairs of halves: 735 Tflop/s).  Two prompts of 500 behind
// 100 to 900, 24 heads of 96 on 8, reach 400, 61.2 us, of which the biases are some 5.  A token of 16 sequences of up to
// 512, 16 heads of 64, 11.0.
#include "attention_device.h"

namespace qproj {

namespace {

// out[h][i] = table[buckets[i]][h]: a thread each
__global__ __launch_bounds__(256) void bias_by_distance_kernel(const float *table, int n_buckets, int n_head, const int32_t *buckets, int distances, float *out, int32_t *error) {
    const int at = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
    if (at >= distances) return;
    const int b = buckets[at];
    if ((uint32_t)b >= (uint32_t)n_buckets && h == 0) atomicOr(error, kKvBadBucket);
    out[(int64_t)h * distances + at] = (uint32_t)b < (uint32_t)n_buckets ? table[(int64_t)b * n_head + h] : 0.f;
}

}  // namespace

int attention_most_reach() { return (kBiasFloats - 1 - 2 * kBiasPad) / 2; }

hipError_t launch_bias_by_distance(const float *table, int n_buckets, int n_head, const int32_t *buckets, int reach, float *out, int32_t *error, hipStream_t s) {
    const int distances = 2 * reach + 1;
    if (dry_run()) {
        plan_note("bias_by_distance_kernel: %d heads x %d distances", n_head, distances);
        return hipSuccess;
    }
    hipLaunchKernelGGL(bias_by_distance_kernel, dim3((distances + 255) / 256, n_head), dim3(256), 0, s, table, n_buckets, n_head, buckets, distances, out, error);
    return hipGetLastError();
}

hipError_t launch_attention_biased(const AttentionJob &j, const float *bias, int reach, bool all, hipStream_t s) {
    const auto with = [&](auto a) {
        a.bias = bias;
        a.reach = reach;
        a.all = all;
        return launch_as(j, a, s);
    };
    return rows_apart(j, true) ? with(BiasApartArgs{}) : with(BiasArgs{});
}

// For the tests: as attention_pieces, where every wave has rows of its own; rows see what lies before them, or all.
int64_t attention_apart_pieces(const AttentionJob &j, bool all, const int32_t *kv_len_later, int64_t most_len, int tokens, int heads, int groups, int32_t *out, int64_t room) {
    BiasApartArgs a{};
    a.all = all;
    a.pages_stride = most_len;      // (pages of one token)
    a.n_tokens = (int32_t)j.n_tokens, a.n_seq = (int32_t)j.n_seq, a.max_q = (int32_t)j.max_q;
    a.q_start = j.q_start, a.kv_len = j.kv_len;
    a.tokens = tokens;
    a.row_tiles = std::max(1, (a.max_q + tokens - 1) / tokens);
    a.most_items = a.n_tokens / tokens + a.n_seq;
    return pieces_of(a, kv_len_later, heads, groups, out, room);
}

}  // namespace qproj
