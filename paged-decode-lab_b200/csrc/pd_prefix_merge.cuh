// pd_prefix_merge.cuh — one output row of shared-prefix attention from its parts.
#pragma once

#include <cuda_fp16.h>

#include "paged_decode.h"
#include "pd_device.cuh"
#include "pd_prefix_args.cuh"

namespace pd {

// Eight elements of 16-byte aligned memory, in FP32.
__device__ __forceinline__ void load8(float (&x)[8], const float *src) {
    const float4 u = __ldcg(reinterpret_cast<const float4 *>(src)), v = __ldcg(reinterpret_cast<const float4 *>(src) + 1);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
}
__device__ __forceinline__ void load8(float (&x)[8], const __half *src) {
    const uint4 u = __ldcg(reinterpret_cast<const uint4 *>(src));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = unpack_half2(w[i]);
        x[2 * i] = v.x, x[2 * i + 1] = v.y;
    }
}

// (m, l) of one row over tokens from .. to of sequence b's live table, kWalk of every `step`
// (from: the start of kWalk tokens of a page), and in `o` eight dims of it: for a dynamic
// launch's pieces that the group's matrix does not describe.  D / 8 neighbouring lanes.  Tokens of pages
// outside the cache are skipped and flagged, as in the decode kernel.
constexpr int kWalk = 4;
template <typename Elt, int D>
__device__ __noinline__ float2 walk(const PrefixArgs &a, int64_t row, int kv_head, int b, int from, int to, int step,
                                    int lane, float (&o)[8]) {
    constexpr int LANES = D / 8;
    const unsigned mates = ((1u << LANES) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));
    const int32_t *pages = a.table + b * a.width;
    float q[8], m = -INFINITY, l = 0.f;
    load8(q, static_cast<const Elt *>(a.q) + row * D + lane * 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] *= a.scale_log2, o[i] = 0.f;
    for (int t = from; t < to; t += step) {
        const int64_t page = __ldcg(pages + t / a.page_size);
        if (page < 0 || page >= a.P) {
            if (lane == 0) atomicOr(a.error, PD_DEVERR_BAD_PAGE);
            continue;
        }
        const int64_t at = ((page * a.page_size + t % a.page_size) * a.Hkv + kv_head) * D + lane * 8;
        const int64_t row_step = int64_t(a.Hkv) * D;
        float s[kWalk], top = m;
#pragma unroll
        for (int j = 0; j < kWalk; ++j) {           // (the rest of a page is there, whatever it holds)
            float x[8];
            load8(x, static_cast<const Elt *>(a.k) + at + j * row_step);
            s[j] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s[j] = fmaf(q[i], x[i], s[j]);
        }
#pragma unroll
        for (int j = 0; j < kWalk; ++j) {
#pragma unroll
            for (int x = LANES / 2; x > 0; x >>= 1) s[j] += __shfl_xor_sync(mates, s[j], x);
            if (t + j >= to) s[j] = -INFINITY;
            top = fmaxf(top, s[j]);
        }
        const float base = top == -INFINITY ? 0.f : top, shrink = exp2f(m - base);
        m = top;
        l *= shrink;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] *= shrink;
#pragma unroll
        for (int j = 0; j < kWalk; ++j) {
            if (t + j >= to) break;
            float x[8];
            load8(x, static_cast<const Elt *>(a.v) + at + j * row_step);
            const float p = exp2f(s[j] - base);
            l += p;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = fmaf(p, x[i], o[i]);
        }
    }
    return make_float2(m, l);
}

// Eight FP32 values to eight elements, one rounding each.
__device__ __forceinline__ void store8(float *dst, const float (&x)[8]) {
    *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__half *dst, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(dst) =
        make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]), pack_half2(x[6], x[7]));
}

// A row's sums over its parts, this thread's eight dims: parts (m, l, o), o not
// normalised, are brought to the common maximum `top` of their m.  Parts without a
// token have l = 0; a NaN denominator stays one.
struct RowSum {
    float top, den = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ explicit RowSum(float top) : top(top) {}
    __device__ __forceinline__ void add(float2 ml, const float (&x)[8]) {
        const float w = ml.y != 0.f ? exp2f(ml.x - top) : 0.f;
        if (w == 0.f && ml.y == ml.y) return;       // (o of an empty part was never written)
        den = fmaf(w, ml.y, den);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = fmaf(w, x[i], o[i]);
    }
    __device__ __forceinline__ void add(float2 ml, float4 u, float4 v) {
        const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        add(ml, x);
    }
};

// What counts for the maximum.
__device__ __forceinline__ float top_of(float2 ml) { return ml.y != 0.f ? ml.x : -INFINITY; }

// Two parts' sum, each with a maximum of its own.
__device__ __forceinline__ RowSum joined(const RowSum &x, float2 ml, const float (&o)[8]) {
    RowSum sum(fmaxf(top_of(make_float2(x.top, x.den)), top_of(ml)));
    sum.add(make_float2(x.top, x.den), x.o);
    sum.add(ml, o);
    return sum;
}

// The suffix decode's (m, l) of a row, and its normalised row as a part.
__device__ __forceinline__ float2 suffix_stats(const PrefixArgs &a, int64_t row) {
    return a.rows ? __ldcg(reinterpret_cast<const float2 *>(a.stats) + row) : make_float2(-INFINITY, 0.f);
}
template <int D>
__device__ __forceinline__ void add_suffix(RowSum &sum, const PrefixArgs &a, float2 ml, int64_t row, int lane) {
    if (ml.y == 0.f) return;
    const float4 *x = reinterpret_cast<const float4 *>(a.rows + row * D + lane * 8);
    const float4 u = __ldcg(x), v = __ldcg(x + 1);
    sum.add(ml, make_float4(u.x * ml.y, u.y * ml.y, u.z * ml.y, u.w * ml.y),
            make_float4(v.x * ml.y, v.y * ml.y, v.z * ml.y, v.w * ml.y));
}

template <typename Elt, int D>
__device__ __forceinline__ void store_row(RowSum &sum, const PrefixArgs &a, int64_t row, int lane) {
    const float inv = sum.den != 0.f ? 1.f / sum.den : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum.o[i] *= inv;
    store8(static_cast<Elt *>(a.out) + row * D + lane * 8, sum.o);
}

// The first token of piece p of `count`, as the plan cuts them.
__device__ __forceinline__ int piece_start(const PrefixArgs &a, int prefix_pages, int count, int p) {
    const int steps = (prefix_pages + a.step_pages - 1) / a.step_pages;
    return min(prefix_pages, p * steps / count * a.step_pages) * a.page_size;
}

// A dynamic launch's pieces that the group's matrix does not describe, token by token: of the first
// `whole` those whose pages are others now (each by the set that has it), and the one that the
// sequence ends in, at token `live` (by all sets).
template <typename Elt, int D>
__device__ __noinline__ void add_others(RowSum &sum, const PrefixArgs &a, int64_t row, int kv_head, int b,
                                        const float2 *ml, int prefix_pages, int count, int whole, int live, int way,
                                        int ways, int lane) {
    float o[8];
    for (int p = way; p < whole; p += ways)
        if (__ldcg(ml + int64_t(p) * a.tile_rows).y == kPieceMoved) {
            const float2 st = walk<Elt, D>(a, row, kv_head, b, piece_start(a, prefix_pages, count, p),
                                           piece_start(a, prefix_pages, count, p + 1), kWalk, lane, o);
            sum = joined(sum, st, o);
        }
    if (whole < count) {
        const float2 st = walk<Elt, D>(a, row, kv_head, b, piece_start(a, prefix_pages, count, whole) + way * kWalk, live,
                                       kWalk * ways, lane, o);
        sum = joined(sum, st, o);
    }
}

}  // namespace pd
