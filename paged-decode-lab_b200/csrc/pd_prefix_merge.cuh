// pd_prefix_merge.cuh — one output row of shared-prefix attention from its parts.
#pragma once

#include <cuda_fp16.h>

#include "pd_device.cuh"
#include "pd_prefix_args.cuh"

namespace pd {

// (m, l) of one row over the first `limit` tokens of its prefix, and in `o`
// eight dims of it: for a dynamic launch's sequence that ends inside its prefix,
// whose row in the group's matrix covers the whole prefix.  D / 8 neighbouring
// lanes, a token at a time: such lengths are rare, and most of them 0.
template <typename Elt, int D>
__device__ __forceinline__ float2 prefix_row(const PrefixArgs &a, int64_t row, int kv_head, const int32_t *pages,
                                          int limit, int lane, float (&o)[8]) {
    constexpr int LANES = D / 8;
    const unsigned mates = ((1u << LANES) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));
    float q[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        q[i] = float(static_cast<const Elt *>(a.q)[row * D + lane * 8 + i]) * a.scale_log2;
        o[i] = 0.f;
    }
    for (int t = 0; t < limit; ++t) {
        const int64_t at = ((int64_t(pages[t / a.page_size]) * a.page_size + t % a.page_size) * a.Hkv + kv_head) * D +
                           lane * 8;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(q[i], float(static_cast<const Elt *>(a.k)[at + i]), s);
#pragma unroll
        for (int x = LANES / 2; x > 0; x >>= 1) s += __shfl_xor_sync(mates, s, x);
        const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
        const float shrink = exp2f(m - base), p = exp2f(s - base);
        l = fmaf(l, shrink, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = fmaf(o[i], shrink, p * float(static_cast<const Elt *>(a.v)[at + i]));
        m = top;
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

// The whole row of a sequence that ends inside its prefix (a dynamic launch).
template <typename Elt, int D>
__device__ __noinline__ void row_inside(const PrefixArgs &a, int64_t row, int kv_head, const int32_t *pages, int b,
                                        int lane) {
    float o[8];
    const float2 ml = prefix_row<Elt, D>(a, row, kv_head, pages, __ldcg(a.lengths + b), lane, o);
    const float2 suffix = suffix_stats(a, row);
    RowSum sum(fmaxf(top_of(ml), top_of(suffix)));
    add_suffix<D>(sum, a, suffix, row, lane);
    sum.add(ml, o);
    store_row<Elt, D>(sum, a, row, lane);
}

}  // namespace pd
