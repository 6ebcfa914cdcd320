// pd_rotary.cu — RMS norm and position rotation of query and key heads, alone
// or on the way into the paged cache.
//
// A head row x[D] with weight w and rotary_dim r:
//   y = x * rsqrt(mean(x^2) + eps) * w                                  (skipped without a weight)
//   pairs (a, b) of y[:r] -> (a cos - b sin, b cos + a sin), cos | sin = table[position]
// where a pair is (y[i], y[i + r/2]) or, interleaved, (y[2i], y[2i + 1]);
// y[r:] passes.  Everything in FP32, one rounding at the store.  Appended
// values are copied bit for bit.
#include <algorithm>
#include <cmath>
#include <string>

#include "paged_decode.h"
#include "pd_device.cuh"
#include "pd_plan.hpp"

#define PD_API extern "C" __attribute__((visibility("default")))

namespace pd {
namespace {

struct HeadRows {
    const void *data;       // [tokens][heads][D], the last dim contiguous; NULL: no such rows
    void *out;
    int64_t token_stride, head_stride;           // in elements
    int64_t out_token_stride, out_head_stride;
    int32_t heads;
};

struct RotaryArgs {
    HeadRows q, k, v;       // v only when appending
    const float *table;     // [max_positions][rotary]: cos | sin; NULL: no rotation
    const float *q_weight, *k_weight;            // FP32 [D]; NULL: no norm
    float eps;
    int32_t rotary, interleaved;
    int64_t max_positions;
    int64_t tokens;
    const int32_t *positions;                    // [tokens] (rotation alone)
    // append: k.out and v.out are the caches [P, T, kv_heads, D]
    const int32_t *page_table, *lengths, *indptr;   // [B, W], [B], [B + 1] or NULL (one token per sequence)
    int64_t width, pages;
    int32_t batch, page_size;
    uint32_t *error;
};

constexpr int kRows = 4;              // rows a thread loads before it works on the first
constexpr int kMaxThreads = 512;
constexpr uint32_t kErrBadPage = PD_DEVERR_BAD_PAGE, kErrLength = PD_DEVERR_LENGTH, kErrPosition = PD_DEVERR_POSITION;

template <typename Elt>
__device__ __forceinline__ float to_float(Elt x) {
    return float(x);
}
template <>
__device__ __forceinline__ float to_float<__half>(__half x) {
    return __half2float(x);
}

template <typename Elt>
__device__ __forceinline__ Elt from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float x) {
    return __float2half_rn(x);
}

// One thread's part of a row: 16 bytes, moved whole when everything is
// 16-byte aligned (VECTOR), else element by element.
template <typename Elt>
struct alignas(16) Part {
    static constexpr int N = 16 / int(sizeof(Elt));
    Elt e[N];
};

template <typename Elt, bool VECTOR>
__device__ __forceinline__ Part<Elt> load_part(const Elt *p) {
    Part<Elt> r;
    if constexpr (VECTOR) {
        *reinterpret_cast<uint4 *>(&r) = *reinterpret_cast<const uint4 *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < Part<Elt>::N; ++i) r.e[i] = p[i];
    }
    return r;
}

template <typename Elt, bool VECTOR>
__device__ __forceinline__ void store_part(Elt *p, const Part<Elt> &r) {
    if constexpr (VECTOR) {
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(&r);
    } else {
#pragma unroll
        for (int i = 0; i < Part<Elt>::N; ++i) p[i] = r.e[i];
    }
}

// The sequence of token i: the last b with indptr[b] <= i (a binary search;
// stays inside [0, batch) whatever indptr holds).
__device__ __forceinline__ int sequence_of(const int32_t *indptr, int batch, int64_t i) {
    int lo = 0, hi = batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (int64_t(__ldg(indptr + mid)) <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One CTA per token (grid-stride).  A row is D / N lanes of one warp, 16 bytes
// each; a CTA holds blockDim / lanes row slots, and row slot s takes rows s, s
// + slots, .. of [queries][keys][values].  The first kRows rows of a thread are
// in flight before it looks up where the token goes.
template <typename Elt, int D, bool VECTOR, bool APPEND>
__global__ void __launch_bounds__(kMaxThreads) rotary_kernel(const RotaryArgs a) {
    using P = Part<Elt>;
    constexpr int N = P::N, LANES = D / N;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int slots = blockDim.x / LANES;
    const int slot = threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    const int e0 = lane * N;                    // first element of this thread's part
    const int kq = a.q.heads, kk = kq + a.k.heads, rows = kk + a.v.heads;   // ends of queries, keys, values
    const int half = a.rotary / 2, half_lanes = half / N;
    const bool turns = a.table && lane < a.rotary / N;
    const bool first = lane < half_lanes;       // half-split: this thread holds the pairs' first elements
    // the lane with the pairs' other elements
    const int mate = (threadIdx.x & 31) + (!turns || a.interleaved ? 0 : first ? half_lanes : -half_lanes);

    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
        P part[kRows];
        const auto load = [&](int base) {
#pragma unroll
            for (int u = 0; u < kRows; ++u) {
                const int row = base + slot + u * slots;
                if (row >= rows) continue;
                const bool is_q = row < kq, is_k = row < kk;
                const void *data = is_q ? a.q.data : is_k ? a.k.data : a.v.data;
                const int64_t ts = is_q ? a.q.token_stride : is_k ? a.k.token_stride : a.v.token_stride;
                const int64_t hs = is_q ? a.q.head_stride : is_k ? a.k.head_stride : a.v.head_stride;
                const int head = row - (is_q ? 0 : is_k ? kq : kk);
                part[u] = load_part<Elt, VECTOR>(static_cast<const Elt *>(data) + token * ts + head * hs + e0);
            }
        };
        load(0);

        // ---- where the token goes
        int64_t position, cache_row = 0;        // cache_row: row (page * T + offset) of the cache
        bool live = true;                       // false: its query rows are zeros, nothing is appended
        if constexpr (APPEND) {
            int b;
            int64_t to_end;                     // tokens from this one to the sequence's end
            if (a.indptr) {
                b = sequence_of(a.indptr, a.batch, token);
                to_end = __ldg(a.indptr + b + 1) - token;   // <= 0: padding past the last sequence
            } else {
                b = int(token);
                to_end = 1;
            }
            const int64_t length = __ldg(a.lengths + b);
            position = length - to_end;
            if (to_end <= 0 || (!a.indptr && length == 0)) {
                live = false;                   // padding, or a sequence that is not in use
            } else if (position < 0 || position >= a.width * a.page_size) {
                live = false;
                if (threadIdx.x == 0) atomicOr(a.error, kErrLength);
            } else {
                const int32_t page = __ldg(a.page_table + int64_t(b) * a.width + position / a.page_size);
                if (page >= 0 && page < a.pages) {
                    cache_row = int64_t(page) * a.page_size + position % a.page_size;
                } else {
                    live = false;
                    if (threadIdx.x == 0) atomicOr(a.error, kErrBadPage);
                }
            }
        } else {
            position = __ldg(a.positions + token);
        }
        if (live && a.table && (position < 0 || position >= a.max_positions)) {
            live = false;
            if (threadIdx.x == 0) atomicOr(a.error, kErrPosition);
        }
        float c[N], s[N];                       // cos and sin of the thread's pairs (interleaved: the first N / 2)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            c[i] = 1.f;
            s[i] = 0.f;
        }
        if (turns && live) {
            const float *t = a.table + position * a.rotary + (a.interleaved ? e0 / 2 : first ? e0 : e0 - half);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                if (a.interleaved && i >= N / 2) continue;
                const float2 cc = __ldg(reinterpret_cast<const float2 *>(t + i));
                const float2 ss = __ldg(reinterpret_cast<const float2 *>(t + half + i));
                c[i] = cc.x, c[i + 1] = cc.y;
                s[i] = ss.x, s[i + 1] = ss.y;
            }
        }

        for (int base = 0;;) {
#pragma unroll
            for (int u = 0; u < kRows; ++u) {
                // The row's lanes are neighbours in one warp, whose other rows may be of another
                // kind or past the end: every lane takes part in the exchanges.
                const int row = base + slot + u * slots;
                const bool is_q = row < kq, is_k = !is_q && row < kk;
                const float *weight = is_q ? a.q_weight : is_k ? a.k_weight : nullptr;
                float x[N];
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = row < rows ? to_float<Elt>(part[u].e[i]) : 0.f;
                if (a.q_weight || a.k_weight) {
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < N; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
                    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
                    if (weight) {
                        const float scale = rsqrtf(sum / float(D) + a.eps);
#pragma unroll
                        for (int i = 0; i < N; ++i) x[i] = x[i] * scale * __ldg(weight + e0 + i);
                    }
                }
                if (a.table) {
                    if (a.interleaved) {
                        if (turns) {
#pragma unroll
                            for (int i = 0; i < N; i += 2) {
                                const float p = x[i], q = x[i + 1];
                                x[i] = fmaf(p, c[i / 2], -q * s[i / 2]);
                                x[i + 1] = fmaf(q, c[i / 2], p * s[i / 2]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const float m = __shfl_sync(kFullMask, x[i], mate);
                            if (turns) x[i] = fmaf(x[i], c[i], first ? -m * s[i] : m * s[i]);
                        }
                    }
                }
                if (row >= rows) continue;
                P r = part[u];                  // values stay as they are
                if (is_q || is_k) {
#pragma unroll
                    for (int i = 0; i < N; ++i) r.e[i] = from_float<Elt>(live ? x[i] : 0.f);
                }
                Elt *dst;
                if (is_q) {
                    dst = static_cast<Elt *>(a.q.out) + token * a.q.out_token_stride + row * a.q.out_head_stride;
                } else if constexpr (APPEND) {
                    if (!live) continue;
                    dst = static_cast<Elt *>(is_k ? a.k.out : a.v.out) +
                          (cache_row * a.k.heads + (row - (is_k ? kq : kk))) * D;
                } else {
                    dst = static_cast<Elt *>(a.k.out) + token * a.k.out_token_stride + (row - kq) * a.k.out_head_stride;
                }
                store_part<Elt, VECTOR>(dst + e0, r);
            }
            base += slots * kRows;
            if (base >= rows) break;
            load(base);
        }
    }
}

template <typename Elt, int D>
cudaError_t launch_rotary(const RotaryArgs &a, bool vector, bool append, cudaStream_t stream) {
    constexpr int LANES = D * int(sizeof(Elt)) / 16;
    const int rows = a.q.heads + a.k.heads + a.v.heads;
    // row slots: a thread's kRows rows cover the token, in whole warps
    int threads = (rows + kRows - 1) / kRows * LANES;
    threads = std::min(kMaxThreads, (threads + 31) / 32 * 32);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(std::min<int64_t>(a.tokens, 1 << 30)));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (append)
        return vector ? cudaLaunchKernelEx(&cfg, rotary_kernel<Elt, D, true, true>, a)
                      : cudaLaunchKernelEx(&cfg, rotary_kernel<Elt, D, false, true>, a);
    return vector ? cudaLaunchKernelEx(&cfg, rotary_kernel<Elt, D, true, false>, a)
                  : cudaLaunchKernelEx(&cfg, rotary_kernel<Elt, D, false, false>, a);
}

// Rows, strides and pointers of one operand; `vector` turns false when its
// parts are not 16-byte aligned.
pd_status check_rows(const pd_heads *h, const char *name, int elt, bool needs_out, bool *vector, HeadRows *rows) {
    *rows = HeadRows{};
    if (!h) return PD_OK;
    if (h->heads < 0 || h->heads > 65535) return fail(PD_ERR_VALUE, std::string(name) + ": heads must be in [0, 65535]");
    if (h->heads == 0) return PD_OK;
    if (!h->data || (needs_out && !h->out)) return fail(PD_ERR_VALUE, std::string(name) + " must not be NULL");
    const uintptr_t at = reinterpret_cast<uintptr_t>(h->data) | reinterpret_cast<uintptr_t>(needs_out ? h->out : nullptr);
    if (at & uintptr_t(elt - 1)) return fail(PD_ERR_VALUE, std::string(name) + " must be aligned to its element size");
    int64_t strides = h->token_stride | h->head_stride;
    if (needs_out) strides |= h->out_token_stride | h->out_head_stride;
    if ((at & 15) || ((strides * elt) & 15)) *vector = false;
    *rows = HeadRows{h->data, h->out, h->token_stride, h->head_stride, h->out_token_stride, h->out_head_stride, h->heads};
    return PD_OK;
}

pd_status check_rotation(const pd_rotation *r, int head_dim, RotaryArgs *a) {
    if (!r) return PD_OK;
    if (r->head_dim != head_dim) return fail(PD_ERR_VALUE, "rotation and layout differ in head_dim");
    if (r->table) {
        if (r->rotary_dim < 16 || r->rotary_dim > r->head_dim || r->rotary_dim % 16)
            return fail(PD_ERR_VALUE, "rotary_dim must be a multiple of 16 up to head_dim");
        if (r->max_positions < 1) return fail(PD_ERR_VALUE, "max_positions must be positive");
        if (reinterpret_cast<uintptr_t>(r->table) & 15) return fail(PD_ERR_VALUE, "the rotation table must be 16-byte aligned");
        a->table = r->table;
        a->rotary = r->rotary_dim;
        a->max_positions = r->max_positions;
        a->interleaved = r->interleaved ? 1 : 0;
    }
    if ((reinterpret_cast<uintptr_t>(r->q_weight) | reinterpret_cast<uintptr_t>(r->k_weight)) & 15)
        return fail(PD_ERR_VALUE, "norm weights must be 16-byte aligned");
    if (!(r->eps >= 0.f) || std::isinf(r->eps)) return fail(PD_ERR_VALUE, "eps must be finite and not negative");
    a->q_weight = r->q_weight;
    a->k_weight = r->k_weight;
    a->eps = r->eps;
    return PD_OK;
}

pd_status run_rotary(const RotaryArgs &a, int head_dim, pd_dtype dtype, bool vector, bool append, int32_t device,
                     void *stream) {
    if (a.tokens == 0 || a.q.heads + a.k.heads + a.v.heads == 0) return PD_OK;
    int prev = -1;
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    cudaError_t err = prev == device ? cudaSuccess : cudaSetDevice(device);
    if (err != cudaSuccess) return fail(PD_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(err));
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == PD_FLOAT16)
        err = head_dim == 64 ? launch_rotary<__half, 64>(a, vector, append, st)
                             : launch_rotary<__half, 128>(a, vector, append, st);
    else
        err = head_dim == 64 ? launch_rotary<float, 64>(a, vector, append, st)
                             : launch_rotary<float, 128>(a, vector, append, st);
    if (prev >= 0 && prev != device) cudaSetDevice(prev);
    if (err != cudaSuccess) return fail(PD_ERR_CUDA, std::string("rotary launch: ") + cudaGetErrorString(err));
    return PD_OK;
}

pd_status check_common(int head_dim, pd_dtype dtype, int64_t tokens, const uint32_t *error) {
    if (dtype != PD_FLOAT16 && dtype != PD_FLOAT32) return fail(PD_ERR_TYPE, "heads must be float16 or float32");
    if (head_dim != 64 && head_dim != 128) return fail(PD_ERR_VALUE, "head_dim must be 64 or 128");
    if (tokens < 0) return fail(PD_ERR_VALUE, "tokens must not be negative");
    if (!error || (reinterpret_cast<uintptr_t>(error) & 3))
        return fail(PD_ERR_VALUE, "the error word must be a 4-byte aligned device pointer");
    return PD_OK;
}

}  // namespace
}  // namespace pd

using namespace pd;

PD_API pd_status pd_rotate_heads(const pd_rotation *rotation, const pd_heads *q, const pd_heads *k, int64_t tokens,
                                 const int32_t *positions, pd_dtype dtype, uint32_t *error, int32_t device,
                                 void *stream) {
    if (!rotation) return fail(PD_ERR_VALUE, "rotation must not be NULL");
    pd_status s = check_common(rotation->head_dim, dtype, tokens, error);
    if (s != PD_OK) return s;
    RotaryArgs a{};
    if ((s = check_rotation(rotation, rotation->head_dim, &a)) != PD_OK) return s;
    const int elt = dtype == PD_FLOAT16 ? 2 : 4;
    bool vector = true;
    if (tokens == 0) return PD_OK;
    if ((s = check_rows(q, "q", elt, true, &vector, &a.q)) != PD_OK) return s;
    if ((s = check_rows(k, "k", elt, true, &vector, &a.k)) != PD_OK) return s;
    if (!positions || (reinterpret_cast<uintptr_t>(positions) & 3))
        return fail(PD_ERR_VALUE, "positions must be a 4-byte aligned device pointer");
    a.tokens = tokens;
    a.positions = positions;
    a.error = error;
    return run_rotary(a, rotation->head_dim, dtype, vector, false, device, stream);
}

PD_API pd_status pd_cache_append(const pd_layout *layout, const pd_rotation *rotation, const pd_heads *q,
                                 const pd_heads *k, const pd_heads *v, int64_t tokens, void *k_cache, void *v_cache,
                                 pd_dtype dtype, const int32_t *table, int64_t table_width, const int32_t *lengths,
                                 const int32_t *indptr, uint32_t *error, int32_t device, void *stream) {
    if (!layout) return fail(PD_ERR_VALUE, "layout must not be NULL");
    const pd_layout &L = *layout;
    if (L.batch <= 0 || L.kv_heads <= 0 || L.physical_pages <= 0 || L.batch > 65535)
        return fail(PD_ERR_VALUE, "layout dimensions must be positive, batch at most 65535");
    if (L.page_size != 16 && L.page_size != 32) return fail(PD_ERR_VALUE, "page_size must be 16 or 32");
    pd_status s = check_common(L.head_dim, dtype, tokens, error);
    if (s != PD_OK) return s;
    RotaryArgs a{};
    if ((s = check_rotation(rotation, L.head_dim, &a)) != PD_OK) return s;
    if (!k || !v || k->heads != L.kv_heads || v->heads != L.kv_heads || (q && q->heads && q->heads != L.query_heads))
        return fail(PD_ERR_VALUE, "head counts must match the layout");
    if (!indptr && tokens != L.batch) return fail(PD_ERR_VALUE, "without indptr there is one token per sequence");
    if (table_width < 1 || table_width > INT32_MAX) return fail(PD_ERR_VALUE, "page table must have at least one column");
    if (tokens == 0) return PD_OK;
    const int elt = dtype == PD_FLOAT16 ? 2 : 4;
    bool vector = true;
    if ((s = check_rows(q, "q", elt, true, &vector, &a.q)) != PD_OK) return s;
    if ((s = check_rows(k, "k", elt, false, &vector, &a.k)) != PD_OK) return s;
    if ((s = check_rows(v, "v", elt, false, &vector, &a.v)) != PD_OK) return s;
    if (!k_cache || !v_cache || !table || !lengths) return fail(PD_ERR_VALUE, "pointers must not be NULL");
    if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15)
        return fail(PD_ERR_VALUE, "k_cache and v_cache must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(indptr)) & 3)
        return fail(PD_ERR_VALUE, "table, lengths and indptr must be 4-byte aligned");
    a.k.out = k_cache;
    a.v.out = v_cache;
    a.tokens = tokens;
    a.page_table = table;
    a.lengths = lengths;
    a.indptr = indptr;
    a.width = table_width;
    a.pages = L.physical_pages;
    a.batch = L.batch;
    a.page_size = L.page_size;
    a.error = error;
    return run_rotary(a, L.head_dim, dtype, vector, true, device, stream);
}
