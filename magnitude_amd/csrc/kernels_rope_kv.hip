// Rotary positions, and keys and values into the paged 4-bit cache with the rotation on the way.
//
//   angle = pos * freq_i;  (a, b) -> magnitude * (a cos - b sin, a sin + b cos)   for pair i of a head: neighbours, or
//   values i and i + n_dims / 2; values from n_dims on stay.
//   a block of 32 values: d = (its value of largest magnitude, the first of them) / -8, kept as fp16;
//   n = min(15, trunc(x / d + 8.5)) with 1 / d and both steps rounded to fp32, as ggml's quantize_row_q4_0 takes them.
//
// Angles and products are taken in 64 bits and rounded to fp32 once: at position a million an fp32 angle is 0.06 rad off, and a
// key that is the nearest fp32 value lands on the code that any other correct program gives it, also next to a border
// between two codes.  A workgroup serves one token: its cosines and sines are one turn of sincospi a pair, shared by
// all heads through LDS; the products are two 64-bit operations a value, hidden behind the rows (4 bytes in, 4 or 0.56 out).
// Bound: the rows' bytes for prompts, the launch itself for a token.  2048 tokens of 40 heads of 128, half of each rotated: 14.7 us,
// 84 MB, 5.7 TB/s; 4096 tokens' append with 32 heads of queries beside 8 of keys and values 37.5, 172 MB, 4.6 TB/s; what they wrote
// read again 10.3, 38 MB, 3.7 TB/s; one token 3.1 and 2.0 us.
#include "kv_cache.h"
#include "qproj_internal.h"

#include <algorithm>

namespace qproj {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kUnit = 8;   // values a thread takes
constexpr int64_t kMostGrid = (int64_t)1 << 23;   // tokens of a launch: a grid has fewer than 2^32 threads in a direction

struct RotateArgs {
    const int32_t *pos;
    const double *freqs;
    int32_t half;          // pairs; 0: no rotation
    int32_t halves;        // pairs are values i and i + half (otherwise neighbours)
    float magnitude;
};

struct RopeKvArgs {
    RotateArgs r;
    const float *q;
    float *q_out;
    int64_t q_stride, q_out_stride;
    int32_t q_units, q_dim;      // units of a token's queries, values of a head
    const float *k, *v;
    int64_t k_stride, v_stride;
    const int64_t *slots;
    int32_t kv_units;            // units of a token's keys (and as many of its values); 0: queries only
    int32_t *error;
    KvView kv;
};

__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }

__device__ __forceinline__ void turn(float &a, float &b, double2 cs) {
    const double x = a, y = b;
    a = (float)fma(x, cs.x, -(y * cs.y));
    b = (float)fma(x, cs.y, y * cs.x);
}

// 8 queries' worth of values: in pairs mode 8 neighbours, in halves mode 4 pairs of values (the thread owns both values of
// every pair, so x and y may be the same rows), behind the rotated part a copy of 8
__device__ __forceinline__ void rotate_unit(const RopeKvArgs &a, const double2 *cs, int64_t token, int unit) {
    const int per_head = a.q_dim / kUnit, head = unit / per_head, u = unit - head * per_head;
    const float *x = a.q + token * a.q_stride + (int64_t)head * a.q_dim;
    float *y = a.q_out + token * a.q_out_stride + (int64_t)head * a.q_dim;
    const int half = a.r.half;
    const bool split = a.r.halves && u * kUnit < 2 * half;
    const int d0 = split ? u * 4 : u * kUnit, d1 = split ? d0 + half : d0 + 4;
    float4 lo = load4(x + d0), hi = load4(x + d1);
    if (split) {
        turn(lo.x, hi.x, cs[d0]);
        turn(lo.y, hi.y, cs[d0 + 1]);
        turn(lo.z, hi.z, cs[d0 + 2]);
        turn(lo.w, hi.w, cs[d0 + 3]);
    } else if (u * kUnit < 2 * half) {
        const double2 *c = cs + u * 4;
        turn(lo.x, lo.y, c[0]);
        turn(lo.z, lo.w, c[1]);
        turn(hi.x, hi.y, c[2]);
        turn(hi.z, hi.w, c[3]);
    }
    *reinterpret_cast<float4 *>(y + d0) = lo;
    *reinterpret_cast<float4 *>(y + d1) = hi;
}

// values d .. d + 3 of a key, rotated (half is a multiple of 4: they lie in one half)
__device__ __forceinline__ float4 rotated4(const RotateArgs &r, const double2 *cs, const float *row, int d) {
    float4 v = load4(row + d);
    if (d >= 2 * r.half) return v;
    if (!r.halves) {
        turn(v.x, v.y, cs[d / 2]);
        turn(v.z, v.w, cs[d / 2 + 1]);
        return v;
    }
    const bool second = d >= r.half;
    const int i = second ? d - r.half : d;
    float4 o = load4(row + (second ? i : d + r.half));
    float *pv = &v.x, *po = &o.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (second) turn(po[j], pv[j], cs[i + j]);
        else turn(pv[j], po[j], cs[i + j]);
    }
    return v;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_bits(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}

// The codes of 8 values of a block and the block's scale; four neighbouring lanes hold the block.  A block with a value that
// is not finite, or too large for an fp16 scale, is NaN as a whole.
__device__ __forceinline__ uint32_t quantize_unit(float4 lo, float4 hi, int eighth, uint16_t &scale) {
    const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t most = 0, top = __float_as_uint(x[0]);   // magnitudes compare as their bits do; NaN and infinity are the largest
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t b = __float_as_uint(x[j]), m = b & 0x7fffffffu;
        if (m > most) most = m, top = b;
    }
    uint32_t om = dpp_bits<0xB1>(most), ot = dpp_bits<0xB1>(top);   // the lane beside
    if (om > most || (om == most && (eighth & 1))) most = om, top = ot;
    om = dpp_bits<0x4E>(most), ot = dpp_bits<0x4E>(top);            // the pair beside
    if (om > most || (om == most && (eighth & 2))) most = om, top = ot;
    const float d = __uint_as_float(top) * -0.125f, inv = 1.0f / d;
    scale = f2h(d);
    const uint32_t mag = scale & 0x7fffu;
    if (mag >= 0x7c00u) scale = 0x7e00u;
    if (mag == 0 || mag >= 0x7c00u) return 0x88888888u;
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int n = (int)__fadd_rn(__fmul_rn(x[j], inv), 8.5f);
        word |= (uint32_t)min(15, max(0, n)) << (4 * j);
    }
    return word;
}

__global__ __launch_bounds__(kRopeThreads) void rope_kv_kernel(const RopeKvArgs a) {
    extern __shared__ __align__(16) double2 cs[];
    const int64_t token = blockIdx.x;
    if (a.r.half) {
        const double pos = (double)a.r.pos[token], mag = (double)a.r.magnitude;
        for (int i = threadIdx.x; i < a.r.half; i += kRopeThreads) {
            double turns = pos * a.r.freqs[i] * 0.15915494309189533577;   // 1 / 2 pi
            turns -= rint(turns);
            double s, c;
            sincospi(2.0 * turns, &s, &c);
            cs[i] = make_double2(c * mag, s * mag);
        }
        __syncthreads();
    }
    int unit = blockIdx.y * kRopeThreads + threadIdx.x;
    if (unit < a.q_units) {
        rotate_unit(a, cs, token, unit);
        return;
    }
    unit -= a.q_units;
    if (unit >= 2 * a.kv_units) return;
    const bool key = unit < a.kv_units;
    if (!key) unit -= a.kv_units;
    const int64_t slot = a.slots[token];
    const bool outside = slot >= a.kv.n_pages << a.kv.page_shift;
    if (outside && unit == 0) atomicOr(a.error, kKvBadSlot);
    if (slot < 0 || outside) return;
    // four neighbouring lanes take a block: q_units, kv_units and the workgroup are multiples of 4
    const int blocks = a.kv.dim / 32, eighth = unit & 3, block = (unit >> 2) % blocks, head = (unit >> 2) / blocks;
    const int d = 32 * block + 8 * eighth;
    const float *row = (key ? a.k + token * a.k_stride : a.v + token * a.v_stride) + (int64_t)head * a.kv.dim;
    float4 lo, hi;
    if (key) {
        lo = rotated4(a.r, cs, row, d);
        hi = rotated4(a.r, cs, row, d + 4);
    } else {
        lo = load4(row + d);
        hi = load4(row + d + 4);
    }
    uint16_t scale;
    const uint32_t word = quantize_unit(lo, hi, eighth, scale);
    const int64_t at = kv_row(a.kv, slot >> a.kv.page_shift, head, (int)(slot & ((1 << a.kv.page_shift) - 1)));
    uint8_t *codes = (key ? a.kv.k_codes : a.kv.v_codes) + at * (a.kv.dim / 2);
    reinterpret_cast<uint32_t *>(codes)[key ? key_word(blocks, block, eighth) : value_word(block, eighth)] = word;
    if (eighth == 0) (key ? a.kv.k_scales : a.kv.v_scales)[at * blocks + block] = scale;
}

// rows of the cache as fp32 values; places outside it (and negative ones) are zeros
__global__ __launch_bounds__(kRopeThreads) void kv_read_kernel(const KvView kv, const int64_t *slots, float *k_out, float *v_out,
                                                               int kv_units, int32_t *error) {
    const int64_t token = blockIdx.x;
    int unit = blockIdx.y * kRopeThreads + threadIdx.x;
    if (unit >= 2 * kv_units) return;
    const bool key = unit < kv_units;
    if (!key) unit -= kv_units;
    float *out = key ? k_out : v_out;
    if (!out) return;
    const int64_t slot = slots[token];
    const bool outside = slot >= kv.n_pages << kv.page_shift;
    if (outside && unit == 0) atomicOr(error, kKvBadSlot);
    const int blocks = kv.dim / 32, eighth = unit & 3, block = (unit >> 2) % blocks, head = (unit >> 2) / blocks;
    float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
    if (slot >= 0 && !outside) {
        const int64_t at = kv_row(kv, slot >> kv.page_shift, head, (int)(slot & ((1 << kv.page_shift) - 1)));
        const uint8_t *codes = (key ? kv.k_codes : kv.v_codes) + at * (kv.dim / 2);
        const uint32_t w = reinterpret_cast<const uint32_t *>(codes)[key ? key_word(blocks, block, eighth) : value_word(block, eighth)];
        const float d = h2f((key ? kv.k_scales : kv.v_scales)[at * blocks + block]);
        const auto value = [&](int j) { return d * (float)((int)((w >> (4 * j)) & 15u) - 8); };
        lo = make_float4(value(0), value(1), value(2), value(3));
        hi = make_float4(value(4), value(5), value(6), value(7));
    }
    float *y = out + (token * kv.n_head + head) * kv.dim + 32 * block + 8 * eighth;
    *reinterpret_cast<float4 *>(y) = lo;
    *reinterpret_cast<float4 *>(y + 4) = hi;
}

}  // namespace

hipError_t launch_rope_kv(const RopeKvJob &j, hipStream_t s) {
    if (j.n_tokens == 0) return hipSuccess;
    RopeKvArgs a{};
    a.r.pos = j.pos;
    a.r.freqs = j.freqs;
    a.r.half = j.n_dims / 2;
    a.r.halves = j.halves;
    a.r.magnitude = j.magnitude;
    a.q = j.q;
    a.q_out = j.q_out;
    a.q_stride = j.q_stride;
    a.q_out_stride = j.q_out_stride;
    a.q_dim = j.q_dim;
    a.q_units = (int)((int64_t)j.n_head * j.q_dim / kUnit);
    a.k = j.k;
    a.v = j.v;
    a.k_stride = j.k_stride;
    a.v_stride = j.v_stride;
    a.slots = j.slots;
    a.error = j.error;
    if (j.kv) {
        a.kv = *j.kv;
        a.kv_units = j.kv->n_head * j.kv->dim / kUnit;
    }
    if (j.kv && a.q_units % 4) return hipErrorInvalidValue;   // a block of the cache is four lanes of a quad
    const int units = a.q_units + 2 * a.kv_units;
    for (int64_t left = j.n_tokens; left > 0; left -= kMostGrid) {
        const dim3 grid((unsigned)std::min(left, kMostGrid), (unsigned)((units + kRopeThreads - 1) / kRopeThreads));
        if (dry_run()) {
            plan_note("rope_kv_kernel: %u tokens, %d units of queries + 2 x %d of keys and values, grid %u x %u x %d", grid.x, a.q_units, a.kv_units, grid.x,
                      grid.y, kRopeThreads);
        } else {
            hipLaunchKernelGGL(rope_kv_kernel, grid, dim3(kRopeThreads), (size_t)a.r.half * sizeof(double2), s, a);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        a.r.pos += a.r.half ? kMostGrid : 0;
        a.q += kMostGrid * (a.q ? a.q_stride : 0);
        a.q_out += kMostGrid * (a.q ? a.q_out_stride : 0);
        a.k += kMostGrid * (a.k ? a.k_stride : 0);
        a.v += kMostGrid * (a.v ? a.v_stride : 0);
        a.slots += a.slots ? kMostGrid : 0;
    }
    return hipSuccess;
}

hipError_t launch_kv_read(const KvView &kv, const int64_t *slots, int64_t n, float *k_out, float *v_out, int32_t *error, hipStream_t s) {
    if (n == 0) return hipSuccess;
    const int units = kv.n_head * kv.dim / kUnit;
    const int64_t row = (int64_t)kv.n_head * kv.dim;
    for (int64_t at = 0; at < n; at += kMostGrid) {
        const dim3 grid((unsigned)std::min(n - at, kMostGrid), (unsigned)((2 * units + kRopeThreads - 1) / kRopeThreads));
        if (dry_run()) {
            plan_note("kv_read_kernel: %u places, 2 x %d units, grid %u x %u x %d", grid.x, units, grid.x, grid.y, kRopeThreads);
            continue;
        }
        hipLaunchKernelGGL(kv_read_kernel, grid, dim3(kRopeThreads), 0, s, kv, slots + at, k_out ? k_out + at * row : nullptr,
                           v_out ? v_out + at * row : nullptr, units, error);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace qproj
