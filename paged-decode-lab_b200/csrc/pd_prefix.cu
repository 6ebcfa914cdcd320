// pd_prefix.cu — shared-prefix decode attention: kernels and C ABI.
//
// For a group of n sequences that share P leading pages, the queries of one KV
// head are a matrix Q of n * G rows.  One pass over the prefix's tokens gives
// each row its (m, l, o):  s = Q K^T / sqrt(D),  m = max s,  l = sum 2^(s - m),
// o = sum 2^(s - m) v  (base 2: scores carry log2(e)).  The tokens behind the
// prefix go through the decode kernel, which gives (m', l', o'), and
// out = (2^(m-M) o + 2^(m'-M) l' o') / (2^(m-M) l + 2^(m'-M) l'),  M = max(m, m').
#include <cmath>
#include <cstring>
#include <new>
#include <string>

#include "paged_decode.h"
#include "pd_device.cuh"
#include "pd_prefix.hpp"
#include "pd_prefix_args.cuh"
#include "pd_prefix_merge.cuh"
#include "pd_prefix_mma.cuh"

#define PD_API extern "C" __attribute__((visibility("default")))

namespace pd {
namespace {

constexpr int kSimtRows = 16, kSimtTokens = 32, kSimtThreads = 128;

// Four elements as FP32, past L1: another kernel may have written them since this SM last read them.
template <typename Elt>
__device__ __forceinline__ float4 load4(const Elt *p);
template <>
__device__ __forceinline__ float4 load4<float>(const float *p) {
    return __ldcg(reinterpret_cast<const float4 *>(p));
}
// One CTA per work item: 16 query rows of one KV head against a piece of the
// prefix, 32 tokens a step.  Eight threads per row: each scores every eighth
// token, then adds up its eighth of the head's dims.
template <typename Elt, int D>
__global__ void __launch_bounds__(kSimtThreads) prefix_simt_kernel(const PrefixArgs a) {
    constexpr int R = kSimtRows, N = kSimtTokens, KS = D + 4;   // KS: K row stride, rows 4 banks apart
    __shared__ __align__(16) float qs[R * D], ks[N * KS], vs[N * D], ps[R * N];
    // With a suffix decode in front, q, the caches and the lengths are complete (it waited for
    // their writers before any of this grid's CTAs could start) and only its rows are not.
    if (!a.rows) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 i0 = a.items[2 * blockIdx.x], i1 = a.items[2 * blockIdx.x + 1];
    const int T = a.page_size, tid = threadIdx.x, r = tid >> 3, c = tid & 7;
    const int row = i0.w * R + r;                               // row of the group's matrix
    const int member = row / a.group;
    const bool on = member < i0.y;
    const int b = on ? a.members[i0.x + member] : 0;
    const int head = i0.z * a.group + row % a.group;
    const int limit = on ? __ldcg(a.lengths + b) : 0;                  // live tokens of the row's sequence
    const Elt *q = static_cast<const Elt *>(a.q) + (int64_t(b) * a.Hq + head) * D;
    for (int d = 4 * c; d < D; d += 32) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on) x = load4<Elt>(q + d);
        *reinterpret_cast<float4 *>(qs + r * D + d) = x;
    }
    float m = -INFINITY, l = 0.f, o[D / 8];
#pragma unroll
    for (int d = 0; d < D / 8; ++d) o[d] = 0.f;
    for (int t0 = i1.y * T; t0 < i1.z * T; t0 += N) {
        __syncthreads();
        for (int e = tid; e < N * (D / 4); e += kSimtThreads) {
            const int n = e / (D / 4), d = e % (D / 4) * 4, t = t0 + n;
            float4 kx = make_float4(0.f, 0.f, 0.f, 0.f), vx = kx;
            if (t < i1.z * T) {
                const int64_t at = ((int64_t(a.pages[i1.x + t / T]) * T + t % T) * a.Hkv + i0.z) * D + d;
                kx = load4<Elt>(static_cast<const Elt *>(a.k) + at);
                vx = load4<Elt>(static_cast<const Elt *>(a.v) + at);
            }
            *reinterpret_cast<float4 *>(ks + n * KS + d) = kx;
            *reinterpret_cast<float4 *>(vs + n * D + d) = vx;
        }
        __syncthreads();
        const int live = min(limit, i1.z * T) - t0;             // tokens of this step the row sees (<= 0: none)
        float s[N / 8], top = m;
#pragma unroll
        for (int k = 0; k < N / 8; ++k) {
            const float *kr = ks + (c + 8 * k) * KS;
            float x = 0.f;
#pragma unroll 8
            for (int d = 0; d < D; d += 4) {
                const float4 qa = *reinterpret_cast<const float4 *>(qs + r * D + d);
                const float4 ka = *reinterpret_cast<const float4 *>(kr + d);
                x = fmaf(qa.x, ka.x, fmaf(qa.y, ka.y, fmaf(qa.z, ka.z, fmaf(qa.w, ka.w, x))));
            }
            s[k] = c + 8 * k < live ? x * a.scale_log2 : -INFINITY;
            top = fmaxf(top, s[k]);
        }
#pragma unroll
        for (int x = 4; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, x));
        const float base = top == -INFINITY ? 0.f : top;        // a row that sees nothing yet
        const float shrink = exp2f(m - base);
        l *= shrink;
#pragma unroll
        for (int k = 0; k < N / 8; ++k) {
            const float p = exp2f(s[k] - base);
            l += p;
            ps[r * N + c + 8 * k] = p;
        }
        m = top;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) o[d] *= shrink;
        __syncwarp();
        const int seen = min(live, N);                          // rows past it may hold anything, NaN too
        for (int n = 0; n < seen; ++n) {
            const float p = ps[r * N + n];
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                const float4 x = *reinterpret_cast<const float4 *>(vs + n * D + 32 * d + 4 * c);
                o[4 * d] = fmaf(p, x.x, o[4 * d]);
                o[4 * d + 1] = fmaf(p, x.y, o[4 * d + 1]);
                o[4 * d + 2] = fmaf(p, x.z, o[4 * d + 2]);
                o[4 * d + 3] = fmaf(p, x.w, o[4 * d + 3]);
            }
        }
    }
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) l += __shfl_xor_sync(kFullMask, l, x);
    if (on) {
        float *po = a.part_o + int64_t(i1.w) * R * D + r * 8 + c % 2 * 4;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
            *reinterpret_cast<float4 *>(po + (4 * d + c / 2) * (R * 8)) =
                make_float4(o[4 * d], o[4 * d + 1], o[4 * d + 2], o[4 * d + 3]);
        if (c == 0) a.part_ml[int64_t(i1.w) * R + r] = make_float2(m, l);
    }
    // the suffix decode's rows are complete when this grid is
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Each output row from the suffix's normalised row and the prefix pieces: D / 8
// threads per row, eight dims each, and `ways` such sets per row that take every
// ways-th piece (several where rows are few and pieces many); the sets' parts are
// merged in order.  What a row needs to know is looked up before the
// prefix kernel is waited for; pieces are loaded four at a time.
constexpr int kMergeThreads = 256;
template <typename Elt, int D>
__global__ void __launch_bounds__(kMergeThreads) prefix_merge_kernel(const PrefixArgs a, int ways) {
    constexpr int LANES = D / 8, BATCH = 4;
    __shared__ float sums[kMergeThreads][10];
    const int per_cta = kMergeThreads / LANES / ways;
    const int set = threadIdx.x / LANES, way = set % ways, lane = threadIdx.x % LANES;
    const int64_t out_row = int64_t(blockIdx.x) * per_cta + set / ways;
    bool on = out_row < int64_t(a.B) * a.Hq;
    const int b = on ? int(out_row / a.Hq) : 0, head = int(out_row % a.Hq);
    const int4 sq = on ? __ldg(a.seqs + 2 * b) : make_int4(-1, 0, 0, 0);
    int pieces = 0, prefix_pages = 0;
    const float2 *ml = a.part_ml;
    const float *po = a.part_o;
    if (sq.x >= 0) {
        const int row = sq.x * a.group + head % a.group;
        const int2 tile = __ldg(a.tiles + sq.y + int64_t(head / a.group) * sq.z + row / a.tile_rows);
        prefix_pages = __ldg(a.seqs + 2 * b + 1).x;
        pieces = tile.y;
        ml += int64_t(tile.x) * a.tile_rows + row % a.tile_rows;
        po += int64_t(tile.x) * a.tile_rows * D + lane * (a.tile_rows * 8) + row % a.tile_rows * 8;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // a dynamic launch's sequence that ends inside its prefix
    if (sizeof(Elt) == 2 && prefix_pages > 0 && __ldcg(a.lengths + b) < prefix_pages * a.page_size) {
        if (way == 0) row_inside<Elt, D>(a, out_row, head / a.group, a.pages + sq.w, b, lane);
        pieces = 0;
        on = false;
    }
    const int64_t ml_step = a.tile_rows, o_step = int64_t(a.tile_rows) * D;
    const float2 suffix = on && way == 0 ? suffix_stats(a, out_row) : make_float2(-INFINITY, 0.f);
    float top = top_of(suffix);
    for (int p = way; p < pieces; p += ways) top = fmaxf(top, top_of(__ldcg(ml + p * ml_step)));
    RowSum sum(top);
    add_suffix<D>(sum, a, suffix, out_row, lane);
    for (int p0 = way; p0 < pieces; p0 += ways * BATCH) {
        float2 st[BATCH];
        float4 u[BATCH], v[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const int p = p0 + j * ways;
            st[j] = make_float2(-INFINITY, 0.f);
            if (p < pieces) {
                st[j] = __ldcg(ml + p * ml_step);
                const float4 *x = reinterpret_cast<const float4 *>(po + p * o_step);
                u[j] = __ldcg(x);
                v[j] = __ldcg(x + 1);
            }
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) sum.add(st[j], u[j], v[j]);
    }
    if (ways > 1) {
        float *mine = sums[threadIdx.x];
        mine[0] = sum.top, mine[1] = sum.den;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[2 + i] = sum.o[i];
        __syncthreads();
        if (way != 0) return;
        float all = -INFINITY;
        for (int w = 0; w < ways; ++w)
            if (sums[threadIdx.x + w * LANES][1] != 0.f) all = fmaxf(all, sums[threadIdx.x + w * LANES][0]);
        sum = RowSum(all);
        for (int w = 0; w < ways; ++w) {
            const float *x = sums[threadIdx.x + w * LANES];
            sum.add(make_float2(x[0], x[1]), make_float4(x[2], x[3], x[4], x[5]), make_float4(x[6], x[7], x[8], x[9]));
        }
    }
    if (on) store_row<Elt, D>(sum, a, out_row, lane);
}

template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), int64_t grid, unsigned threads, size_t smem,
                             cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(grid));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

using MmaKernel = void (*)(const CUtensorMap, const CUtensorMap, const PrefixArgs);
struct MmaEntry {
    MmaKernel kernel;
    unsigned threads;
    size_t smem;
};
template <int D, int T>
MmaEntry mma_entry() {
    return {prefix_mma_kernel<D, T>, PrefixShape<D, T>::THREADS, PrefixShape<D, T>::SMEM};
}
MmaEntry mma_entry_for(const pd_layout &L) {
    if (L.head_dim == 64) return L.page_size == 16 ? mma_entry<64, 16>() : mma_entry<64, 32>();
    return L.page_size == 16 ? mma_entry<128, 16>() : mma_entry<128, 32>();
}

template <int D>
cudaError_t launch_prefix(const pd_prefix_plan &p, const PrefixArgs &a, const CUtensorMap &map_k,
                          const CUtensorMap &map_v, cudaStream_t stream) {
    cudaError_t err = cudaSuccess;
    const int64_t items = int64_t(p.items.size()) / p.item_words;
    if (items && p.dtype == PD_FLOAT16) {
        const MmaEntry e = mma_entry_for(p.layout);
        err = launch_dependent(e.kernel, items, e.threads, e.smem, stream, map_k, map_v, a);
        if (p.direct) return err;
    } else if (items) {
        err = launch_dependent(prefix_simt_kernel<float, D>, items, kSimtThreads, 0, stream, a);
    }
    if (err != cudaSuccess) return err;
    const int64_t rows = int64_t(a.B) * a.Hq, per_cta = kMergeThreads / (D / 8) / p.merge_ways;
    const int64_t grid = (rows + per_cta - 1) / per_cta;
    return p.dtype == PD_FLOAT16
               ? launch_dependent(prefix_merge_kernel<__half, D>, grid, kMergeThreads, 0, stream, a, p.merge_ways)
               : launch_dependent(prefix_merge_kernel<float, D>, grid, kMergeThreads, 0, stream, a, p.merge_ways);
}

pd_status decode_impl(pd_prefix_plan *p, const void *q, const void *k, const void *v, pd_dtype dtype,
                      const int32_t *table, const int32_t *lengths, void *out, void *stream) {
    if (!p) return fail(PD_ERR_VALUE, "plan must not be NULL");
    if (p->device < 0) return fail(PD_ERR_VALUE, "host-only plan (device < 0) cannot launch");
    if (!p->dev) return fail(PD_ERR_UNBOUND, "plan has no device buffer: call pd_prefix_plan_bind first");
    if (dtype != p->dtype) return fail(PD_ERR_TYPE, "input dtype differs from the plan's dtype");
    if (!q || !k || !v || !out) return fail(PD_ERR_VALUE, "q, k, v and out must not be NULL");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
         reinterpret_cast<uintptr_t>(out)) & 15)
        return fail(PD_ERR_VALUE, "q, k, v and out must be 16-byte aligned");
    int prev = -1;
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    cudaError_t err = prev == p->device ? cudaSuccess : cudaSetDevice(p->device);
    if (err != cudaSuccess) return fail(PD_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(err));
    const PrefixImage &im = p->image;
    PrefixArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.items = reinterpret_cast<const int4 *>(p->dev + im.off_items);
    a.seqs = reinterpret_cast<const int4 *>(p->dev + im.off_seqs);
    a.tiles = reinterpret_cast<const int2 *>(p->dev + im.off_tiles);
    a.members = reinterpret_cast<const int32_t *>(p->dev + im.off_members);
    a.pages = reinterpret_cast<const int32_t *>(p->dev + im.off_pages);
    a.lengths = lengths ? lengths : reinterpret_cast<const int32_t *>(p->dev + im.off_lengths);
    a.part_o = reinterpret_cast<float *>(p->dev + im.off_part_o);
    a.part_ml = reinterpret_cast<float2 *>(p->dev + im.off_part_ml);
    a.out = out;
    a.error = reinterpret_cast<uint32_t *>(p->dev + im.off_error);
    a.B = p->layout.batch;
    a.Hq = p->layout.query_heads;
    a.Hkv = p->layout.kv_heads;
    a.group = p->group;
    a.page_size = p->layout.page_size;
    a.tile_rows = p->tile_rows;
    a.direct = p->direct ? 1 : 0;
    a.P = p->layout.physical_pages;
    a.scale_log2 = float(1.4426950408889634 / std::sqrt(double(p->layout.head_dim)));
    pd_status s = PD_OK;
    alignas(64) CUtensorMap map_k, map_v;
    if (dtype == PD_FLOAT16 && !p->items.empty()) s = encode_prefix_maps(*p->suffix, k, v, &map_k, &map_v);
    if (s == PD_OK && !p->suffix_empty) {
        float *rows = reinterpret_cast<float *>(p->dev + im.off_rows);
        float *stats = reinterpret_cast<float *>(p->dev + im.off_stats);
        s = table ? pd_decode_dynamic(p->suffix, q, k, v, dtype, table, lengths, rows, stats, stream)
                  : pd_decode_with_stats(p->suffix, q, k, v, dtype, rows, stats, stream);
        a.rows = rows;
        a.stats = stats;
    }
    if (s == PD_OK) {
        const auto st = static_cast<cudaStream_t>(stream);
        err = p->layout.head_dim == 64 ? launch_prefix<64>(*p, a, map_k, map_v, st)
                                       : launch_prefix<128>(*p, a, map_k, map_v, st);
        if (err != cudaSuccess) s = fail(PD_ERR_CUDA, std::string("prefix launch: ") + cudaGetErrorString(err));
    }
    if (prev >= 0 && prev != p->device) cudaSetDevice(prev);
    return s;
}

pd_status create_impl(const pd_layout *layout, const int32_t *table, int64_t width, const int32_t *lengths,
                      const int32_t *max_lengths, int32_t group_count, const int32_t *indptr, const int32_t *members,
                      const int32_t *pages, pd_dtype dtype, int32_t device, pd_prefix_plan &p) {
    // the decode plan's own checks of layout, table and lengths, before the groups look at them
    pd_plan *whole = nullptr;
    pd_status s = create_suffix_plan(layout, table, width, lengths, max_lengths, nullptr, dtype, -1, &whole);
    if (s != PD_OK) return s;
    pd_plan_destroy(whole);
    p.layout = *layout;
    p.dtype = dtype;
    p.device = device;
    p.width = width;
    p.dynamic = max_lengths != nullptr;
    if (group_count < 0) {
        find_prefix_groups(p.layout, table, width, lengths, 0, p.groups);
    } else {
        if (group_count > 0 && (!indptr || !members || !pages))
            return fail(PD_ERR_VALUE, "group arrays must not be NULL");
        for (int g = 0; g < group_count; ++g) {
            if (indptr[g] < 0 || indptr[g + 1] < indptr[g] || indptr[g + 1] - indptr[0] > layout->batch)
                return fail(PD_ERR_VALUE, "group indptr must not decrease, and name at most batch members");
            PrefixGroup group;
            group.pages = pages[g];
            group.members.assign(members + indptr[g], members + indptr[g + 1]);
            p.groups.push_back(std::move(group));
        }
        if ((s = check_prefix_groups(p.layout, table, width, lengths, p.groups)) != PD_OK) return s;
    }
    std::vector<int32_t> first(layout->batch, 0);
    for (const PrefixGroup &g : p.groups)
        for (const int32_t b : g.members) first[b] = g.pages;
    s = create_suffix_plan(layout, table, width, lengths, max_lengths, first.data(), dtype, device, &p.suffix);
    if (s != PD_OK) return s;
    p.suffix_empty = p.suffix->total_pages == 0;
    return build_prefix_plan(p, table, lengths, p.suffix->sm_count);
}

}  // namespace
}  // namespace pd

using namespace pd;

PD_API pd_status pd_prefix_plan_create(const pd_layout *layout, const int32_t *table, int64_t table_width,
                                       const int32_t *lengths, const int32_t *max_lengths, int32_t group_count,
                                       const int32_t *indptr, const int32_t *members, const int32_t *pages,
                                       pd_dtype dtype, int32_t device, pd_prefix_plan **out_plan) {
    if (!out_plan) return fail(PD_ERR_VALUE, "out_plan must not be NULL");
    *out_plan = nullptr;
    pd_prefix_plan *p = nullptr;
    try {
        p = new pd_prefix_plan();
        const pd_status s = pd::create_impl(layout, table, table_width, lengths, max_lengths, group_count, indptr,
                                            members, pages, dtype, device, *p);
        if (s != PD_OK) {
            delete p;
            return s;
        }
    } catch (const std::bad_alloc &) {
        delete p;
        return fail(PD_ERR_VALUE, "out of host memory");
    }
    *out_plan = p;
    return PD_OK;
}

PD_API void pd_prefix_plan_destroy(pd_prefix_plan *plan) { delete plan; }

PD_API pd_status pd_prefix_plan_get_info(const pd_prefix_plan *p, pd_prefix_info *info) {
    if (!p || !info) return fail(PD_ERR_VALUE, "plan and info must not be NULL");
    *info = pd_prefix_info{};
    info->groups = int32_t(p->groups.size());
    for (const PrefixGroup &g : p->groups) {
        info->members += int32_t(g.members.size());
        info->shared_pages += int64_t(g.members.size() - 1) * g.pages;
    }
    info->tile_rows = p->tile_rows;
    info->items = int32_t(p->items.size() / p->item_words);
    info->suffix_launch = p->suffix_empty ? 0 : 1;
    info->dynamic = p->dynamic ? 1 : 0;
    info->device_bytes = int64_t(p->image.bytes);
    return PD_OK;
}

PD_API pd_status pd_prefix_plan_copy_groups(const pd_prefix_plan *p, int32_t *group, int32_t *pages) {
    if (!p) return fail(PD_ERR_VALUE, "plan must not be NULL");
    if (group)
        for (int b = 0; b < p->layout.batch; ++b) group[b] = -1;
    for (size_t g = 0; g < p->groups.size(); ++g) {
        if (pages) pages[g] = p->groups[g].pages;
        if (group)
            for (const int32_t b : p->groups[g].members) group[b] = int32_t(g);
    }
    return PD_OK;
}

PD_API size_t pd_prefix_plan_device_bytes(const pd_prefix_plan *p) { return p ? p->image.bytes : 0; }

PD_API pd_status pd_prefix_plan_bind(pd_prefix_plan *p, void *buffer, size_t bytes, void *stream) {
    if (!p) return fail(PD_ERR_VALUE, "plan must not be NULL");
    if (p->device < 0) return fail(PD_ERR_VALUE, "host-only plan (device < 0) cannot be bound");
    if (!buffer || bytes < p->image.bytes)
        return fail(PD_ERR_VALUE, "device buffer is NULL or smaller than the plan needs");
    if (reinterpret_cast<uintptr_t>(buffer) & 255) return fail(PD_ERR_VALUE, "device buffer must be 256-byte aligned");
    uint8_t *dev = static_cast<uint8_t *>(buffer);
    pd_status s = pd_plan_bind(p->suffix, dev + p->image.off_suffix, p->image.off_rows - p->image.off_suffix, stream);
    if (s != PD_OK) return s;
    int prev = -1;
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    cudaError_t err = prev == p->device ? cudaSuccess : cudaSetDevice(p->device);
    const auto st = static_cast<cudaStream_t>(stream);
    if (err == cudaSuccess && p->dtype == PD_FLOAT16) {
        const MmaEntry e = mma_entry_for(p->layout);
        err = cudaFuncSetAttribute(reinterpret_cast<const void *>(e.kernel), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   int(e.smem));
    }
    if (err == cudaSuccess)
        err = cudaMemcpyAsync(dev, p->host_image.data(), p->host_image.size(), cudaMemcpyHostToDevice, st);
    if (err == cudaSuccess) err = cudaStreamSynchronize(st);
    if (prev >= 0 && prev != p->device) cudaSetDevice(prev);
    if (err != cudaSuccess) return fail(PD_ERR_CUDA, std::string("plan upload: ") + cudaGetErrorString(err));
    p->dev = dev;
    return PD_OK;
}

PD_API pd_status pd_prefix_decode(pd_prefix_plan *p, const void *q, const void *k, const void *v, pd_dtype dtype,
                                  void *out, void *stream) {
    return pd::decode_impl(p, q, k, v, dtype, nullptr, nullptr, out, stream);
}

PD_API pd_status pd_prefix_decode_dynamic(pd_prefix_plan *p, const void *q, const void *k, const void *v,
                                          pd_dtype dtype, const int32_t *table, const int32_t *lengths, void *out,
                                          void *stream) {
    if (p && !p->dynamic) return fail(PD_ERR_VALUE, "plan was built without max_lengths");
    if (!table || !lengths) return fail(PD_ERR_VALUE, "table and lengths must not be NULL");
    if ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(lengths)) & 3)
        return fail(PD_ERR_VALUE, "table and lengths must be 4-byte aligned");
    return pd::decode_impl(p, q, k, v, dtype, table, lengths, out, stream);
}

PD_API pd_status pd_prefix_plan_read_errors(pd_prefix_plan *p, uint32_t *error_word, void *stream) {
    if (!p || !error_word) return fail(PD_ERR_VALUE, "plan and error_word must not be NULL");
    if (!p->dev) return fail(PD_ERR_UNBOUND, "plan has no device buffer: call pd_prefix_plan_bind first");
    uint32_t suffix = 0, own = 0;
    pd_status s = pd_plan_read_errors(p->suffix, &suffix, stream);
    if (s != PD_OK) return s;
    int prev = -1;
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    cudaError_t err = prev == p->device ? cudaSuccess : cudaSetDevice(p->device);
    const auto st = static_cast<cudaStream_t>(stream);
    if (err == cudaSuccess) err = cudaMemcpyAsync(&own, p->dev + p->image.off_error, 4, cudaMemcpyDeviceToHost, st);
    if (err == cudaSuccess) err = cudaMemsetAsync(p->dev + p->image.off_error, 0, 4, st);
    if (err == cudaSuccess) err = cudaStreamSynchronize(st);
    if (prev >= 0 && prev != p->device) cudaSetDevice(prev);
    if (err != cudaSuccess) return fail(PD_ERR_CUDA, std::string("error readback: ") + cudaGetErrorString(err));
    *error_word = suffix | own;
    return PD_OK;
}
