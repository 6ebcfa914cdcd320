// pd_prefix.cu — shared-prefix decode attention: kernels and C ABI.
//
// For a group of n sequences that share P leading pages, the queries of one KV
// head are a matrix Q of n * G rows.  One pass over the prefix's tokens gives
// each row its (m, l, o):  s = Q K^T / sqrt(D),  m = max s,  l = sum 2^(s - m),
// o = sum 2^(s - m) v  (base 2: scores carry log2(e)).  The tokens behind the
// prefix go through the decode kernel, which gives (m', l', o'), and
// out = (2^(m-M) o + 2^(m'-M) l' o') / (2^(m-M) l + 2^(m'-M) l'),  M = max(m, m').
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <string>

#include "paged_decode.h"
#include "pd_device.cuh"
#include "pd_launch.cuh"
#include "pd_prefix.hpp"
#include "pd_prefix_args.cuh"
#include "pd_prefix_merge.cuh"
#include "pd_prefix_mma.cuh"

#define PD_API extern "C" __attribute__((visibility("default")))

namespace pd {
namespace {

constexpr int kSimtThreads = 128, kSimtTokens = 32;

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// Shared memory of the FP32 kernel, in floats: queries [R][D + 4], two stages of
// K [32][D + 4] and V [32][D], weights [R][36], rescale factors [R].  (Row strides
// 4 floats over a multiple of 32: the rows a warp reads side by side lie 4 banks apart.)
template <int R, int D>
struct SimtShape {
    static constexpr int QS = D + 4, KS = D + 4, PS = kSimtTokens + 4;
    static constexpr int Q = 0, K = Q + R * QS, V = K + 2 * kSimtTokens * KS, P = V + 2 * kSimtTokens * D,
                         F = P + R * PS, FLOATS = F + R;
};

// FP32 prefix kernel: one CTA per work item, R query rows of one KV head against
// a piece of the prefix, 32 tokens a step, the next step's K and V on their way
// (cp.async).  CUDA cores, two FMAs to an instruction: the scores in R/16 x 4
// blocks per thread, the output in R/8 x D/16 ones, so that an operand read from
// shared memory serves several products.  The online softmax of a row is shared
// by the eight threads that hold its scores.  Rows of sequences that end inside
// their prefix (dynamic launches) are dropped by the merge kernel, so only the
// piece's end needs a mask.  Bound by the FMAs: 27 TFLOP/s of 74 on a B200 with 64
// rows (32:8 heads of 128), shared memory reads and two barriers a step being the
// rest; 16-row tiles (one query head per KV head) reach 15.
// LIVE: a dynamic launch.
template <int R, int D, bool LIVE>
__global__ void __launch_bounds__(kSimtThreads) prefix_simt_kernel(const __grid_constant__ PrefixArgs a) {
    using S = SimtShape<R, D>;
    constexpr int N = kSimtTokens, TR = R / 16, OR = R / 8, OD = D / 16;   // rows and dims of a thread's blocks
    extern __shared__ __align__(16) float sm[];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 i0 = a.items[2 * blockIdx.x], i1 = a.items[2 * blockIdx.x + 1];
    const int T = a.page_size, tid = threadIdx.x, end = i1.z * T;
    const uint32_t base = smem_u32(sm);
    for (int e = tid; e < R * (D / 4); e += kSimtThreads) {
        const int r = e / (D / 4), d = e % (D / 4) * 4, row = i0.w * R + r, member = row / a.group;
        const bool on = member < i0.y;
        const int64_t b = on ? __ldg(a.members + i0.x + member) : 0;
        copy16(base + (S::Q + r * S::QS + d) * 4,
               static_cast<const float *>(a.q) + (b * a.Hq + i0.z * a.group + row % a.group) * D + d, on);
    }
    const auto load = [&](int t0, int stage) {
        for (int e = tid; e < N * (D / 4); e += kSimtThreads) {
            const int n = e / (D / 4), d = e % (D / 4) * 4, t = t0 + n;
            const bool on = t < end;
            const int64_t page = on ? __ldg(a.pages + i1.x + t / T) : 0;
            const int64_t at = ((page * T + t % T) * a.Hkv + i0.z) * D + d;
            copy16(base + (S::K + (stage * N + n) * S::KS + d) * 4, static_cast<const float *>(a.k) + at, on);
            copy16(base + (S::V + (stage * N + n) * D + d) * 4, static_cast<const float *>(a.v) + at, on);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // scores: tokens tg + 8 j of rows rg + 16 i;  output: rows og + 8 i, dims 4 dg + 64 k + [0, 4)
    const int tg = tid & 7, rg = tid >> 3, dg = tid & 15, og = tid >> 4;
    float m[TR], l[TR];
    f32x2 o[OR][OD / 2];
#pragma unroll
    for (int i = 0; i < TR; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int i = 0; i < OR; ++i)
#pragma unroll
        for (int k = 0; k < OD / 2; ++k) o[i][k] = 0;
    load(i1.y * T, 0);
    // A dynamic launch: whether a row's live table has other pages in this piece.  kSimtThreads / R threads
    // share a row's pages of each step, whose ids come while its scores are formed.
    __shared__ int moved[R];
    const int32_t *live_ids = nullptr;
    if (LIVE) {
        const int member = (i0.w * R + tid % R) / a.group;
        if (member < i0.y) live_ids = a.table + __ldg(a.members + i0.x + member) * a.width;
        if (tid < R) moved[tid] = 0;                    // (ordered by the barriers below)
    }
    for (int t0 = i1.y * T, stage = 0; t0 < end; t0 += N, stage ^= 1) {
        if (t0 + N < end) {
            load(t0 + N, stage ^ 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        const int seen = t0 / T + tid / R;              // at most two pages a step, at least two threads a row
        const bool looks = LIVE && live_ids && tid / R < N / T && seen < i1.z;
        const int32_t id = looks ? __ldg(live_ids + seen) ^ __ldg(a.pages + i1.x + seen) : 0;
        // ---- scores
        const float *ks = sm + S::K + (stage * N + tg) * S::KS, *qs = sm + S::Q + rg * S::QS;
        f32x2 acc[TR][4];
#pragma unroll
        for (int i = 0; i < TR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0;
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
            ulonglong2 q[TR], k[4];
#pragma unroll
            for (int i = 0; i < TR; ++i) q[i] = *reinterpret_cast<const ulonglong2 *>(qs + 16 * i * S::QS + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const ulonglong2 *>(ks + 8 * j * S::KS + d);
#pragma unroll
            for (int i = 0; i < TR; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fma_f32x2(q[i].y, k[j].y, fma_f32x2(q[i].x, k[j].x, acc[i][j]));
        }
        // ---- softmax
#pragma unroll
        for (int i = 0; i < TR; ++i) {
            float s[4], top = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 x = unpack_f32x2(acc[i][j]);
                s[j] = t0 + tg + 8 * j < end ? (x.x + x.y) * a.scale_log2 : -INFINITY;
                top = fmaxf(top, s[j]);
            }
#pragma unroll
            for (int x = 4; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, x));
            const float ref = top == -INFINITY ? 0.f : top;
            const float shrink = exp2f(m[i] - ref);
            m[i] = top;
            l[i] *= shrink;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(s[j] - ref);
                l[i] += p;
                sm[S::P + (rg + 16 * i) * S::PS + tg + 8 * j] = p;
            }
            if (tg == 0) sm[S::F + rg + 16 * i] = shrink;
        }
        if (LIVE && id != 0) moved[tid % R] = 1;
        __syncthreads();
        // ---- output
        const float *vs = sm + S::V + stage * N * D + 4 * dg;
#pragma unroll
        for (int i = 0; i < OR; ++i) {
            const float f = sm[S::F + og + 8 * i];
            if (f != 1.f)
#pragma unroll
                for (int k = 0; k < OD / 2; ++k) o[i][k] = mul_f32x2(o[i][k], pack_f32x2(f, f));
        }
#pragma unroll 2
        for (int n = 0; n < N; n += 4) {
            float4 p[OR];
#pragma unroll
            for (int i = 0; i < OR; ++i) p[i] = *reinterpret_cast<const float4 *>(sm + S::P + (og + 8 * i) * S::PS + n);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                ulonglong2 v[OD / 4];
#pragma unroll
                for (int k = 0; k < OD / 4; ++k) v[k] = *reinterpret_cast<const ulonglong2 *>(vs + (n + u) * D + 64 * k);
#pragma unroll
                for (int i = 0; i < OR; ++i) {
                    const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
                    const f32x2 w2 = pack_f32x2(w, w);
#pragma unroll
                    for (int k = 0; k < OD / 4; ++k) {
                        o[i][2 * k] = fma_f32x2(w2, v[k].x, o[i][2 * k]);
                        o[i][2 * k + 1] = fma_f32x2(w2, v[k].y, o[i][2 * k + 1]);
                    }
                }
            }
        }
        __syncthreads();        // the stage, the weights and the factors may be overwritten
    }
#pragma unroll
    for (int i = 0; i < TR; ++i) {
#pragma unroll
        for (int x = 4; x > 0; x >>= 1) l[i] += __shfl_xor_sync(kFullMask, l[i], x);
        if (tg == 0) {
            const bool usable = !LIVE || !moved[rg + 16 * i];
            a.part_ml[int64_t(i1.w) * R + rg + 16 * i] = make_float2(m[i], usable ? l[i] : kPieceMoved);
        }
    }
    float *po = a.part_o + int64_t(i1.w) * R * D;
#pragma unroll
    for (int i = 0; i < OR; ++i)
#pragma unroll
        for (int k = 0; k < OD / 4; ++k) {
            const int d = 4 * dg + 64 * k;
            *reinterpret_cast<ulonglong2 *>(po + (d / 8 * R + og + 8 * i) * 8 + d % 8) =
                make_ulonglong2(o[i][2 * k], o[i][2 * k + 1]);
        }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Each output row from the suffix's normalised row and the prefix pieces: D / 8
// threads per row, eight dims each, and `ways` such sets per row that take every
// ways-th piece (several where rows are few and pieces many); the sets' parts are
// merged in order.  What a row needs to know is looked up before the
// kernels in front are waited for; pieces are loaded four at a time.  Bound by
// latency: 17 us for 16384 rows of head_dim 128 when profiled alone on cold caches.
// LIVE: a dynamic launch; pieces that its lengths or table do not bear out are left to add_others.
constexpr int kMergeThreads = 256;
template <typename Elt, int D, bool LIVE>
__global__ void __launch_bounds__(kMergeThreads, 3) prefix_merge_kernel(const __grid_constant__ PrefixArgs a, int ways) {
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
    // The decode kernel flags live lengths past the plan's; where it has nothing to do, this one does.
    if (!a.rows && on && way == 0 && lane == 0 && __ldcg(a.lengths + b) > __ldg(a.seqs + 2 * b + 1).y)
        atomicOr(a.error, PD_DEVERR_LENGTH);
    // A dynamic launch's sequence that ends inside its prefix: pieces before its end count.
    const int count = pieces;
    int live = prefix_pages * a.page_size;
    if (LIVE && count > 0) {
        const int length = __ldcg(a.lengths + b);
        if (length < live) {
            live = length;
            while (pieces > 0 && piece_start(a, prefix_pages, count, pieces) > live) --pieces;
        }
    }
    bool moved = false;                     // a piece whose pages are others in the live table
    const int64_t ml_step = a.tile_rows, o_step = int64_t(a.tile_rows) * D;
    const float2 suffix = on && way == 0 ? suffix_stats(a, out_row) : make_float2(-INFINITY, 0.f);
    float top = top_of(suffix);
    for (int p = way; p < pieces; p += ways) {
        const float2 st = __ldcg(ml + p * ml_step);
        if (LIVE && st.y == kPieceMoved) moved = true;
        else top = fmaxf(top, top_of(st));
    }
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
        for (int j = 0; j < BATCH; ++j) {
            if (LIVE && st[j].y == kPieceMoved) st[j] = make_float2(-INFINITY, 0.f);
            sum.add(st[j], u[j], v[j]);
        }
    }
    if (LIVE && (moved || pieces < count)) {
        RowSum all = sum;
        add_others<Elt, D>(all, a, out_row, head / a.group, b, ml, prefix_pages, count, pieces, live, way, ways, lane);
        sum = all;
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

using MmaKernel = void (*)(const CUtensorMap, const CUtensorMap, const PrefixArgs);
struct MmaEntry {
    MmaKernel kernel;
    unsigned threads;
    size_t smem;
};
template <int D, int T>
MmaEntry mma_entry(bool live) {
    return {live ? prefix_mma_kernel<D, T, true> : prefix_mma_kernel<D, T, false>, PrefixShape<D, T>::THREADS,
            PrefixShape<D, T>::SMEM};
}
MmaEntry mma_entry_for(const pd_layout &L, bool live) {
    if (L.head_dim == 64) return L.page_size == 16 ? mma_entry<64, 16>(live) : mma_entry<64, 32>(live);
    return L.page_size == 16 ? mma_entry<128, 16>(live) : mma_entry<128, 32>(live);
}

using SimtKernel = void (*)(const PrefixArgs);
struct SimtEntry {
    SimtKernel kernel;
    size_t smem;
};
template <int R, int D>
SimtEntry simt_entry(bool live) {
    return {live ? prefix_simt_kernel<R, D, true> : prefix_simt_kernel<R, D, false>, SimtShape<R, D>::FLOATS * 4};
}
SimtEntry simt_entry_for(const pd_prefix_plan &p, bool live) {
    if (p.layout.head_dim == 64) return p.tile_rows == 16 ? simt_entry<16, 64>(live) : simt_entry<64, 64>(live);
    return p.tile_rows == 16 ? simt_entry<16, 128>(live) : simt_entry<64, 128>(live);
}

// Allow the prefix kernels of this plan their shared memory.
cudaError_t allow_smem(const pd_prefix_plan &p) {
    for (const bool live : {false, true}) {
        if (live && !p.dynamic) break;
        const void *kernel;
        size_t smem;
        if (p.dtype == PD_FLOAT16) {
            const MmaEntry e = mma_entry_for(p.layout, live);
            kernel = reinterpret_cast<const void *>(e.kernel), smem = e.smem;
        } else {
            const SimtEntry e = simt_entry_for(p, live);
            kernel = reinterpret_cast<const void *>(e.kernel), smem = e.smem;
        }
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        if (err != cudaSuccess) return err;
    }
    return cudaSuccess;
}

cudaError_t launch_prefix(const pd_prefix_plan &p, const PrefixArgs &a, const CUtensorMap &map_k,
                          const CUtensorMap &map_v, cudaStream_t stream) {
    const int64_t items = int64_t(p.items.size()) / p.item_words;
    if (p.dtype == PD_FLOAT16) {
        const MmaEntry e = mma_entry_for(p.layout, a.table != nullptr);
        return launch_dependent(e.kernel, items, e.threads, e.smem, stream, map_k, map_v, a);
    }
    const SimtEntry e = simt_entry_for(p, a.table != nullptr);
    return launch_dependent(e.kernel, items, kSimtThreads, e.smem, stream, a);
}

template <int D>
cudaError_t launch_merge(const pd_prefix_plan &p, const PrefixArgs &a, cudaStream_t stream) {
    const int64_t rows = int64_t(a.B) * a.Hq, per_cta = kMergeThreads / (D / 8) / p.merge_ways;
    const int64_t grid = (rows + per_cta - 1) / per_cta;
    const auto kernel = p.dtype == PD_FLOAT16
                            ? (a.table ? prefix_merge_kernel<__half, D, true> : prefix_merge_kernel<__half, D, false>)
                            : (a.table ? prefix_merge_kernel<float, D, true> : prefix_merge_kernel<float, D, false>);
    return launch_dependent(kernel, grid, kMergeThreads, 0, stream, a, p.merge_ways);
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
    a.table = table;
    a.width = p->width;
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
    a.P = p->layout.physical_pages;
    a.step_pages = p->step_pages;
    a.scale_log2 = float(1.4426950408889634 / std::sqrt(double(p->layout.head_dim)));
    // The prefix kernel goes first: it lets the suffix's decode start beside it as soon as its own
    // CTAs have (FP16, on the SMs it leaves), and the merge waits for both.
    pd_status s = PD_OK;
    const auto st = static_cast<cudaStream_t>(stream);
    const bool wide = p->layout.head_dim == 128;
    if (!p->items.empty()) {
        alignas(64) CUtensorMap map_k, map_v;
        if (dtype == PD_FLOAT16) s = encode_prefix_maps(*p->suffix, k, v, &map_k, &map_v);
        if (s == PD_OK) {
            err = launch_prefix(*p, a, map_k, map_v, st);
            if (err != cudaSuccess) s = fail(PD_ERR_CUDA, std::string("prefix launch: ") + cudaGetErrorString(err));
        }
    }
    const bool merges = !p->items.empty() || dtype == PD_FLOAT16;     // (else: nothing shared, nothing to convert)
    if (s == PD_OK && (!p->suffix_empty || !merges)) {
        float *rows = merges ? reinterpret_cast<float *>(p->dev + im.off_rows) : static_cast<float *>(out);
        float *stats = reinterpret_cast<float *>(p->dev + im.off_stats);
        s = decode_suffix(p->suffix, q, k, v, table, lengths, rows, stats, !p->items.empty() && p->suffix_ctas > 0, stream);
        a.rows = rows;
        a.stats = stats;
    }
    if (s == PD_OK && merges) {
        err = wide ? launch_merge<128>(*p, a, st) : launch_merge<64>(*p, a, st);
        if (err != cudaSuccess) s = fail(PD_ERR_CUDA, std::string("merge launch: ") + cudaGetErrorString(err));
    }
    if (prev >= 0 && prev != p->device) cudaSetDevice(prev);
    return s;
}

pd_status create_impl(const pd_layout *layout, const int32_t *table, int64_t width, const int32_t *lengths,
                      const int32_t *max_lengths, int32_t group_count, const int32_t *indptr, const int32_t *members,
                      const int32_t *pages, pd_dtype dtype, int32_t device, pd_prefix_plan &p) {
    if (group_count < -2) return fail(PD_ERR_VALUE, "group_count must be -2, -1 or a number of groups");
    // the decode plan's own checks of layout, table and lengths, before the groups look at them
    pd_plan *whole = nullptr;
    pd_status s = create_suffix_plan(layout, table, width, lengths, max_lengths, nullptr, dtype, -1, 0, &whole);
    if (s != PD_OK) return s;
    pd_plan_destroy(whole);
    p.layout = *layout;
    p.dtype = dtype;
    p.device = device;
    p.width = width;
    p.dynamic = max_lengths != nullptr;
    if (group_count < 0) {
        find_prefix_groups(p.layout, table, width, lengths, p.groups);
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
    int sm_count = 148;
    if (device >= 0) {
        const cudaError_t err = cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, device);
        if (err != cudaSuccess) return fail(PD_ERR_CUDA, std::string("device query: ") + cudaGetErrorString(err));
    }
    std::vector<int32_t> first(layout->batch, 0);
    const int32_t *span = max_lengths ? max_lengths : lengths;
    const auto suffix_pages = [&]() {       // the pages outside of all groups
        std::fill(first.begin(), first.end(), 0);
        for (const PrefixGroup &g : p.groups)
            for (const int32_t b : g.members) first[b] = g.pages;
        int64_t pages = 0;
        for (int b = 0; b < layout->batch; ++b)
            pages += std::max<int64_t>(0, (int64_t(span[b]) + layout->page_size - 1) / layout->page_size - first[b]);
        return pages;
    };
    set_shape(p);
    if (group_count == -1) keep_paying_groups(p, suffix_pages(), sm_count);
    const int64_t rest = suffix_pages();
    p.suffix_empty = rest == 0;
    choose_pieces(p, rest, sm_count);
    s = create_suffix_plan(layout, table, width, lengths, max_lengths, first.data(), dtype, device, p.suffix_ctas,
                           &p.suffix);
    if (s != PD_OK) return s;
    return build_prefix_plan(p, table, lengths, max_lengths ? max_lengths : lengths, sm_count);
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
    info->item_words = p->item_words;
    info->suffix_ctas = p->suffix_ctas;
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

PD_API pd_status pd_prefix_plan_copy_items(const pd_prefix_plan *p, int32_t *items) {
    if (!p || !items) return fail(PD_ERR_VALUE, "plan and items must not be NULL");
    std::copy(p->items.begin(), p->items.end(), items);
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
    if (err == cudaSuccess) err = allow_smem(*p);
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
