// Attention over the paged 4-bit cache.
//
//   y = sum_t softmax_t(scale * q . k_t) v_t over the tokens t <= p (the last `window` of them) of a sequence.
//
// A wave serves one row of one head: it goes over the tokens once with the running maximum and sum of the softmax.
#include "kv_cache.h"
#include "qproj_internal.h"

namespace qproj {

namespace {

constexpr int kMostDims = 256;

struct AttentionArgs {
    KvView kv;
    const float *q;
    float *y;
    int64_t q_stride, y_stride, pages_stride, n_tokens, n_seq, max_q;
    const int32_t *q_start, *kv_len, *pages;
    int32_t *error;
    float scale;
    int32_t window, group;
};

__global__ __launch_bounds__(64) void attention_kernel(const AttentionArgs a) {
    constexpr int kHeld = kMostDims / 64;
    const int lane = threadIdx.x, head = blockIdx.y, kv_head = head / a.group, dim = a.kv.dim, blocks = dim / 32;
    const int64_t row = blockIdx.x;
    const auto bad = [&](int64_t s) {
        const int64_t b = a.q_start[s], e = a.q_start[s + 1], n = a.kv_len[s];
        return b < 0 || e < b || e > a.n_tokens || e - b > a.max_q || n < 0 || n > a.pages_stride << a.kv.page_shift;
    };
    if (row == 0 && head == 0)
        for (int64_t s = lane; s < a.n_seq; s += 64)
            if (bad(s)) atomicOr(a.error, kKvBadRows);
    int64_t seq = 0, start = 0, end = 0;
    for (; seq < a.n_seq; ++seq) {
        start = a.q_start[seq], end = a.q_start[seq + 1];
        if (row >= start && row < end) break;
    }
    if (seq == a.n_seq || bad(seq)) return;
    const int64_t len = a.kv_len[seq];
    const int64_t p = len - (end - row);
    float q[kHeld], o[kHeld];
    for (int i = 0; i < kHeld; ++i) {
        const int d = lane + 64 * i;
        q[i] = d < dim ? a.q[row * a.q_stride + (int64_t)head * dim + d] * a.scale : 0.f;
        o[i] = 0.f;
    }
    float m = -3e38f, l = 0.f;
    for (int64_t t = a.window ? max((int64_t)0, p - a.window + 1) : 0; t <= p; ++t) {
        const int64_t page = a.pages[seq * a.pages_stride + (t >> a.kv.page_shift)];
        if (page < 0 || page >= a.kv.n_pages) {
            if (lane == 0) atomicOr(a.error, kKvBadPage);
            continue;
        }
        const int64_t at = kv_row(a.kv, page, kv_head, (int)(t & ((1 << a.kv.page_shift) - 1)));
        float s = 0.f, v[kHeld];
        for (int i = 0; i < kHeld; ++i) {
            const int d = lane + 64 * i;
            v[i] = 0.f;
            if (d >= dim) continue;
            const int b = d / 32, e = d / 8 % 4, j = d % 8;
            const uint32_t kw = reinterpret_cast<const uint32_t *>(a.kv.k_codes + at * (dim / 2))[key_word(blocks, b, e)];
            const uint32_t vw = reinterpret_cast<const uint32_t *>(a.kv.v_codes + at * (dim / 2))[value_word(b, e)];
            s = fmaf(q[i], h2f(a.kv.k_scales[at * blocks + b]) * (float)((int)((kw >> (4 * j)) & 15) - 8), s);
            v[i] = h2f(a.kv.v_scales[at * blocks + b]) * (float)((int)((vw >> (4 * j)) & 15) - 8);
        }
        s = wave_sum(s);
        const float top = fmaxf(m, s), back = expf(m - top), w = expf(s - top);
        l = fmaf(l, back, w);
        for (int i = 0; i < kHeld; ++i) o[i] = fmaf(o[i], back, w * v[i]);
        m = top;
    }
    for (int i = 0; i < kHeld; ++i) {
        const int d = lane + 64 * i;
        if (d < dim) a.y[row * a.y_stride + (int64_t)head * dim + d] = l != 0.f ? o[i] / l : 0.f;
    }
}

}  // namespace

hipError_t launch_attention(const AttentionJob &j, hipStream_t s) {
    if (j.n_tokens == 0 || j.n_seq == 0) return hipSuccess;
    AttentionArgs a{};
    a.kv = *j.kv;
    a.q = j.q;
    a.y = j.y;
    a.q_stride = j.q_stride;
    a.y_stride = j.y_stride;
    a.pages_stride = j.pages_stride;
    a.n_tokens = j.n_tokens;
    a.n_seq = j.n_seq;
    a.max_q = j.max_q;
    a.q_start = j.q_start;
    a.kv_len = j.kv_len;
    a.pages = j.pages;
    a.error = j.error;
    a.scale = j.scale;
    a.window = j.window;
    a.group = j.n_head / j.kv->n_head;
    if (dry_run()) {
        plan_note("attention_kernel: %lld tokens x %d heads, a wave each", (long long)j.n_tokens, j.n_head);
        return hipSuccess;
    }
    hipLaunchKernelGGL(attention_kernel, dim3((unsigned)j.n_tokens, (unsigned)j.n_head), dim3(64), 0, s, a);
    return hipGetLastError();
}

}  // namespace qproj
