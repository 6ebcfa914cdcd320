// pd_rotary.cu — RMS norm and position rotation of query and key heads, alone
// or on the way into the paged cache.
//
// A head row x[D] with weight w and rotary_dim r:
//   y = x * rsqrt(mean(x^2) + eps) * w                                  (skipped without a weight)
//   pairs (a, b) of y[:r] -> (a cos - b sin, b cos + a sin), cos | sin = table[position]
// where a pair is (y[i], y[i + r/2]) or, interleaved, (y[2i], y[2i + 1]);
// y[r:] passes.  Everything in FP32, one rounding at the store.  Appended
// values are copied bit for bit.
//
// Bound by memory: each head row is read and written once.  Measured on a B200
// (graph replay): 16384 tokens of 32:8 FP16 heads of 128 62.5 us (344 MB, 5.5
// TB/s), 24k tokens of 64:8 into the cache 155 to 164 us (971 MB, 5.9 to 6.3
// TB/s), 4099 of
// 32:32 FP32 heads of 64 21.6 us (135 MB, 6.2 TB/s); 64 tokens of 32:1 3.2 us
// and 4 tokens into the cache 3.5 us, a launch and three trips to memory.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "paged_decode.h"
#include "pd_device.cuh"
#include "pd_launch.cuh"
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
    int32_t batch, page_shift;                   // log2 of the page size
    uint32_t *error;
};

// The direct kernel: rows that a lane holds at once, and the largest CTA.
constexpr int kRows = 4, kMaxThreads = 512;
// The streaming kernel: consumer warps beside one producer warp, CTAs per SM and
// the shared memory of each one's stages.
constexpr int kConsumers = 8, kStreamCtas = 3, kStreamThreads = 32 * (kConsumers + 1);
constexpr int kMaxStages = 8, kMinStages = 3;
constexpr int kRingBytes[kStreamCtas + 1] = {0, 208 * 1024, 104 * 1024, 70 * 1024};   // by CTAs per SM
constexpr uint32_t kErrBadPage = PD_DEVERR_BAD_PAGE, kErrLength = PD_DEVERR_LENGTH, kErrPosition = PD_DEVERR_POSITION;

// One thread's part of a row: two pieces of 8 bytes, each moved whole when
// everything is 8-byte aligned (VECTOR), else element by element.
template <typename Elt>
struct alignas(8) Piece {
    static constexpr int H = 8 / int(sizeof(Elt));   // elements
    Elt e[H];
};
template <typename Elt>
struct Part {
    Piece<Elt> lo, hi;
};

template <typename Elt, bool VECTOR>
__device__ __forceinline__ void load_piece(Piece<Elt> &r, const Elt *p) {
    if constexpr (VECTOR) {
        *reinterpret_cast<uint2 *>(&r) = *reinterpret_cast<const uint2 *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < Piece<Elt>::H; ++i) r.e[i] = p[i];
    }
}

template <typename Elt, bool VECTOR>
__device__ __forceinline__ void store_piece(Elt *p, const Piece<Elt> &r) {
    if constexpr (VECTOR) {
        *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(&r);
    } else {
#pragma unroll
        for (int i = 0; i < Piece<Elt>::H; ++i) p[i] = r.e[i];
    }
}

// A piece in FP32, two elements to a register pair, and back (one rounding).
__device__ __forceinline__ void widen(f32x2 (&x)[2], const Piece<__half> &p) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&p.e[2 * i]));
        x[i] = pack_f32x2(v.x, v.y);
    }
}
__device__ __forceinline__ void widen(f32x2 (&x)[1], const Piece<float> &p) { x[0] = pack_f32x2(p.e[0], p.e[1]); }
__device__ __forceinline__ void narrow(Piece<__half> &p, const f32x2 (&x)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 v = unpack_f32x2(x[i]);
        *reinterpret_cast<__half2 *>(&p.e[2 * i]) = __floats2half2_rn(v.x, v.y);
    }
}
__device__ __forceinline__ void narrow(Piece<float> &p, const f32x2 (&x)[1]) {
    const float2 v = unpack_f32x2(x[0]);
    p.e[0] = v.x, p.e[1] = v.y;
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

// Where a token goes.
struct Place {
    int64_t position;
    int64_t cache_row;      // row (page * T + offset) of the cache
    bool live;              // false: its query rows are zeros, nothing is appended
};

// `report`: this thread flags a token that is skipped.
template <bool APPEND>
__device__ __forceinline__ Place place_of(const RotaryArgs &a, int64_t token, bool report) {
    Place p{0, 0, true};
    uint32_t flag = 0;
    if constexpr (APPEND) {
        int b;
        int64_t to_end;     // tokens from this one to the sequence's end
        bool before = false;                            // of the first sequence's range
        if (a.indptr) {
            before = token < __ldg(a.indptr);
            b = sequence_of(a.indptr, a.batch, token);
            to_end = __ldg(a.indptr + b + 1) - token;   // <= 0: padding past the last sequence
        } else {
            b = int(token);
            to_end = 1;
        }
        const int64_t length = __ldg(a.lengths + b);
        p.position = length - to_end;
        if (to_end <= 0 || (!a.indptr && length == 0)) {
            p.live = false;                             // padding, or a sequence that is not in use
        } else if (before || p.position < 0 || p.position >= (a.width << a.page_shift)) {
            flag = kErrLength;
        } else {
            const int at = int(p.position);
            const int32_t page = __ldg(a.page_table + int64_t(b) * a.width + (at >> a.page_shift));
            if (page >= 0 && page < a.pages)
                p.cache_row = (int64_t(page) << a.page_shift) + (at & ((1 << a.page_shift) - 1));
            else flag = kErrBadPage;
        }
    } else {
        p.position = __ldg(a.positions + token);
    }
    if (p.live && !flag && a.table && (p.position < 0 || p.position >= a.max_positions)) flag = kErrPosition;
    if (flag) {
        p.live = false;
        if (report) atomicOr(a.error, flag);
    }
    return p;
}

// The cosines and sines of a lane's pairs, as its two pieces x and y meet them:
//   half-split    x' = x c + y t, y' = y c + x t2        with t = -s, t2 = s
//   interleaved   x' = x c + swap(x) t, y' = y c2 + swap(y) t2   with (c, c), (-s, s) per pair
template <int W>
struct Turn {
    f32x2 c[W], t[W], c2[W], t2[W];
};

// From the table's cosines and sines of the lane's H = 2 W pairs.
template <int W, bool INTERLEAVED>
__device__ __forceinline__ void load_turn(Turn<W> &r, const float *c, const float *s) {
    float cc[2 * W], ss[2 * W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float2 x = *reinterpret_cast<const float2 *>(c + 2 * i), y = *reinterpret_cast<const float2 *>(s + 2 * i);
        cc[2 * i] = x.x, cc[2 * i + 1] = x.y;
        ss[2 * i] = y.x, ss[2 * i + 1] = y.y;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (INTERLEAVED) {      // pair i in x, pair W + i in y
            r.c[i] = pack_f32x2(cc[i], cc[i]);
            r.t[i] = pack_f32x2(-ss[i], ss[i]);
            r.c2[i] = pack_f32x2(cc[W + i], cc[W + i]);
            r.t2[i] = pack_f32x2(-ss[W + i], ss[W + i]);
        } else {
            r.c[i] = pack_f32x2(cc[2 * i], cc[2 * i + 1]);
            r.t[i] = pack_f32x2(-ss[2 * i], -ss[2 * i + 1]);
            r.t2[i] = pack_f32x2(ss[2 * i], ss[2 * i + 1]);
        }
    }
}

// 2 W floats from 8-byte aligned memory.
template <int W>
__device__ __forceinline__ void load_floats(f32x2 (&r)[W], const float *p) {
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = *reinterpret_cast<const f32x2 *>(p + 2 * i);
}

// One lane's part of a row: the norm, then the rotation.  With `sums` every lane
// of the warp takes part in its rows' sums; `norms`: this row uses them.
template <typename Elt, int LANES, bool INTERLEAVED>
__device__ __forceinline__ void norm_rotate(Part<Elt> &part, bool sums, bool norms, const f32x2 (&wlo)[Piece<Elt>::H / 2],
                                            const f32x2 (&whi)[Piece<Elt>::H / 2], float eps, bool turns,
                                            const Turn<Piece<Elt>::H / 2> &r) {
    constexpr int W = Piece<Elt>::H / 2;
    f32x2 x[W], y[W];
    widen(x, part.lo);
    widen(y, part.hi);
    if (sums) {
        f32x2 sum2 = mul_f32x2(x[0], x[0]);
#pragma unroll
        for (int i = 1; i < W; ++i) sum2 = fma_f32x2(x[i], x[i], sum2);
#pragma unroll
        for (int i = 0; i < W; ++i) sum2 = fma_f32x2(y[i], y[i], sum2);
        float sum = unpack_f32x2(sum2).x + unpack_f32x2(sum2).y;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
        if (norms) {
            const float scale = rsqrtf(fmaf(sum, 1.f / float(LANES * 4 * W), eps));
            const f32x2 scale2 = pack_f32x2(scale, scale);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                x[i] = mul_f32x2(x[i], mul_f32x2(wlo[i], scale2));
                y[i] = mul_f32x2(y[i], mul_f32x2(whi[i], scale2));
            }
        }
    }
    if (turns) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (INTERLEAVED) {
                const float2 u = unpack_f32x2(x[i]), v = unpack_f32x2(y[i]);
                x[i] = fma_f32x2(x[i], r.c[i], mul_f32x2(pack_f32x2(u.y, u.x), r.t[i]));
                y[i] = fma_f32x2(y[i], r.c2[i], mul_f32x2(pack_f32x2(v.y, v.x), r.t2[i]));
            } else {
                const f32x2 u = mul_f32x2(y[i], r.t[i]), v = mul_f32x2(x[i], r.t2[i]);
                x[i] = fma_f32x2(x[i], r.c[i], u);
                y[i] = fma_f32x2(y[i], r.c[i], v);
            }
        }
    }
    narrow(part.lo, x);
    narrow(part.hi, y);
}

// A row is D / N lanes of one warp.  A lane holds both elements of each of its
// pairs, so that the rotation needs no exchange and half the cosines: pieces
// [H lane, +H) and r/2 further on in half-split rows, neighbouring pieces in
// interleaved ones and past the rotation.
template <typename Elt, int D, bool INTERLEAVED>
struct Lane {
    static constexpr int H = Piece<Elt>::H, W = H / 2, N = 2 * H, LANES = D / N, PER_WARP = 32 / LANES;
    int lane, lo, hi;
    bool turns;
    __device__ __forceinline__ explicit Lane(const RotaryArgs &a) {
        lane = threadIdx.x % LANES;
        turns = lane < a.rotary / N;
        const bool apart = turns && !INTERLEAVED;
        lo = apart ? H * lane : N * lane;
        hi = apart ? lo + a.rotary / 2 : lo + H;
    }
};

// Direct kernel: any strides, alignment and size.  One CTA per token; its
// row slots take rows slot, slot + slots, .. of [queries][keys][values], kRows of
// them in flight before the token's place is looked up.
template <typename Elt, int D, bool VECTOR, bool APPEND, bool INTERLEAVED>
__global__ void __launch_bounds__(kMaxThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
    using P = Part<Elt>;
    using L = Lane<Elt, D, INTERLEAVED>;
    constexpr int H = L::H, W = L::W, LANES = L::LANES;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const L l(a);
    const int slots = blockDim.x / LANES, slot = threadIdx.x / LANES;
    const int kq = a.q.heads, kk = kq + a.k.heads, rows = kk + a.v.heads;   // ends of queries, keys, values
    const int64_t token = blockIdx.x;
    P part[kRows];
    const auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            const int row = base + slot + u * slots;
            if (row >= rows) continue;
            const bool is_q = row < kq, is_k = row < kk;
            const Elt *p = static_cast<const Elt *>(is_q ? a.q.data : is_k ? a.k.data : a.v.data);
            const int64_t ts = is_q ? a.q.token_stride : is_k ? a.k.token_stride : a.v.token_stride;
            const int64_t hs = is_q ? a.q.head_stride : is_k ? a.k.head_stride : a.v.head_stride;
            p += token * ts + (row - (is_q ? 0 : is_k ? kq : kk)) * hs;
            load_piece<Elt, VECTOR>(part[u].lo, p + l.lo);
            load_piece<Elt, VECTOR>(part[u].hi, p + l.hi);
        }
    };
    load(0);
    const Place at = place_of<APPEND>(a, token, threadIdx.x == 0);
    Turn<W> turn;
    if (l.turns && at.live) {
        const float *t = a.table + at.position * a.rotary + H * l.lane;
        load_turn<W, INTERLEAVED>(turn, t, t + a.rotary / 2);
    }
    for (int base = 0;;) {
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            const int row = base + slot + u * slots;
            const bool is_q = row < kq, is_k = !is_q && row < kk;
            if (__any_sync(kFullMask, is_q || is_k)) {
                f32x2 wlo[W], whi[W];
                Part<Elt> r = part[u];
                const float *weight = is_q ? a.q_weight : is_k ? a.k_weight : nullptr;
                if (weight) {
                    load_floats<W>(wlo, weight + l.lo);
                    load_floats<W>(whi, weight + l.hi);
                }
                norm_rotate<Elt, LANES, INTERLEAVED>(r, a.q_weight || a.k_weight, weight != nullptr, wlo, whi, a.eps,
                                                     l.turns && at.live, turn);
                if (is_q || is_k) part[u] = at.live ? r : Part<Elt>{};      // values stay as they are
            }
            if (row >= rows) continue;
            Elt *dst;
            if (is_q) {
                dst = static_cast<Elt *>(a.q.out) + token * a.q.out_token_stride + row * a.q.out_head_stride;
            } else if constexpr (APPEND) {
                if (!at.live) continue;
                dst = static_cast<Elt *>(is_k ? a.k.out : a.v.out) +
                      (at.cache_row * a.k.heads + (row - (is_k ? kq : kk))) * D;
            } else {
                dst = static_cast<Elt *>(a.k.out) + token * a.k.out_token_stride + (row - kq) * a.k.out_head_stride;
            }
            store_piece<Elt, VECTOR>(dst + l.lo, part[u].lo);
            store_piece<Elt, VECTOR>(dst + l.hi, part[u].hi);
        }
        base += slots * kRows;
        if (base >= rows) break;
        load(base);
    }
}

// ---------------------------------------------------------------- streaming kernel
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

__device__ __forceinline__ void bulk_store(void *dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

// Shared memory: [stages][q | k | v | table row] barriers.
struct StreamShape {
    int q_bytes, k_bytes, v_bytes, stage_bytes, stages;
    size_t smem;
};

// Streaming kernel: tokens whose rows lie one after another (16-byte aligned).
// The bulk copies keep three stages per CTA in flight without registers (loads
// into registers reached 2.8 TB/s), and three CTAs per SM of eight consumer warps
// leave enough of them to hide the norm's exchanges (two CTAs 4.5 TB/s, four 5.0).
// A persistent CTA takes every gridDim-th token through a ring of stages: the
// producer warp brings a token's queries, keys, values and its row of the rotation
// table by bulk copies, the consumer warps norm and rotate the rows where they are,
// and the producer sends the whole token on by bulk stores.  Places are looked up
// by the producer's lanes, 32 tokens at a time.
template <typename Elt, int D, bool APPEND, bool INTERLEAVED>
__global__ void __launch_bounds__(kStreamThreads, kStreamCtas)
    rotary_stream_kernel(const __grid_constant__ RotaryArgs a, const __grid_constant__ StreamShape sh) {
    using L = Lane<Elt, D, INTERLEAVED>;
    constexpr int H = L::H, W = L::W, LANES = L::LANES, PER_WARP = L::PER_WARP;
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + size_t(sh.stages) * sh.stage_bytes);
    uint64_t *done = full + kMaxStages;
    int64_t *cache_rows = reinterpret_cast<int64_t *>(done + kMaxStages);
    volatile int *lives = reinterpret_cast<volatile int *>(cache_rows + kMaxStages);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stages = sh.stages;
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(smem_u32(full + i), 1);
            mbar_init(smem_u32(done + i), kConsumers);
        }
        mbar_init_fence();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __syncthreads();
    // this CTA's tokens; tokens fit 31 bits
    const int n = (int(a.tokens) - int(blockIdx.x) + int(gridDim.x) - 1) / int(gridDim.x);
    const auto token_of = [&](int j) { return blockIdx.x + int64_t(j) * gridDim.x; };
    // token j is in stage j % stages, whose barriers are then in phase j / stages
    struct Turnstile {
        int stage = 0, phase = 0;
        __device__ __forceinline__ void next(int stages) {
            if (++stage == stages) stage = 0, phase ^= 1;
        }
    };

    if (warp == kConsumers) {
        Place batch{};
        int loaded = 0;                 // tokens whose loads were issued
        int load_stage = 0;
        const auto load = [&]() {       // the next token's
            const int j = loaded++, st = load_stage;
            if (++load_stage == stages) load_stage = 0;
            if ((j & 31) == 0 && j + lane < n) batch = place_of<APPEND>(a, token_of(j + lane), true);
            const int from = j & 31;
            const int64_t position = __shfl_sync(kFullMask, batch.position, from);
            const int64_t cache_row = __shfl_sync(kFullMask, batch.cache_row, from);
            const bool live = __shfl_sync(kFullMask, int(batch.live), from) != 0;
            if (lane != 0) return;
            cache_rows[st] = cache_row;
            lives[st] = live;
            const uint32_t bar = smem_u32(full + st), dst = smem_u32(smem + size_t(st) * sh.stage_bytes);
            const int turn_bytes = a.table && live ? a.rotary * 4 : 0;
            mbar_arrive_expect_tx(bar, uint32_t(sh.q_bytes + sh.k_bytes + sh.v_bytes + turn_bytes));
            const int64_t token = token_of(j);
            if (sh.q_bytes) bulk_load(dst, static_cast<const Elt *>(a.q.data) + token * a.q.token_stride, sh.q_bytes, bar);
            if (sh.k_bytes)
                bulk_load(dst + sh.q_bytes, static_cast<const Elt *>(a.k.data) + token * a.k.token_stride, sh.k_bytes, bar);
            if (sh.v_bytes)
                bulk_load(dst + sh.q_bytes + sh.k_bytes, static_cast<const Elt *>(a.v.data) + token * a.v.token_stride,
                          sh.v_bytes, bar);
            if (turn_bytes)
                bulk_load(dst + sh.q_bytes + sh.k_bytes + sh.v_bytes, a.table + position * a.rotary, turn_bytes, bar);
        };
        while (loaded < min(n, stages)) load();
        Turnstile at;
        for (int j = 0; j < n; ++j, at.next(stages)) {
            const int st = at.stage;
            if (!__all_sync(kFullMask, mbar_wait(smem_u32(done + st), at.phase))) {
                if (lane == 0) atomicOr(a.error, PD_DEVERR_TIMEOUT);
                break;
            }
            if (lane == 0) {
                const int64_t token = token_of(j);
                const uint32_t src = smem_u32(smem + size_t(st) * sh.stage_bytes);
                if (sh.q_bytes) bulk_store(static_cast<Elt *>(a.q.out) + token * a.q.out_token_stride, src, sh.q_bytes);
                if constexpr (APPEND) {
                    if (lives[st]) {
                        const int64_t at = cache_rows[st] * a.k.heads * D;
                        bulk_store(static_cast<Elt *>(a.k.out) + at, src + sh.q_bytes, sh.k_bytes);
                        bulk_store(static_cast<Elt *>(a.v.out) + at, src + sh.q_bytes + sh.k_bytes, sh.v_bytes);
                    }
                } else if (sh.k_bytes) {
                    bulk_store(static_cast<Elt *>(a.k.out) + token * a.k.out_token_stride, src + sh.q_bytes, sh.k_bytes);
                }
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                // all but the newest store have read their stages: token j - 1's is free
                asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            }
            __syncwarp();
            if (j > 0 && loaded < n) load();
        }
        // no copy is in flight when the CTA ends
        for (int j = max(0, loaded - stages); j < loaded; ++j)
            if (!mbar_wait(smem_u32(full + j % stages), (j / stages) & 1) && lane == 0) atomicOr(a.error, PD_DEVERR_TIMEOUT);
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    } else {
        const L l(a);
        f32x2 q_lo[W], q_hi[W], k_lo[W], k_hi[W];
        if (a.q_weight) {
            load_floats<W>(q_lo, a.q_weight + l.lo);
            load_floats<W>(q_hi, a.q_weight + l.hi);
        }
        if (a.k_weight) {
            load_floats<W>(k_lo, a.k_weight + l.lo);
            load_floats<W>(k_hi, a.k_weight + l.hi);
        }
        Turnstile at;
        for (int j = 0; j < n; ++j, at.next(stages)) {
            const int st = at.stage;
            if (!__all_sync(kFullMask, mbar_wait(smem_u32(full + st), at.phase))) {
                if (lane == 0) atomicOr(a.error, PD_DEVERR_TIMEOUT);
                break;
            }
            uint8_t *stage = smem + size_t(st) * sh.stage_bytes;
            const bool live = lives[st] != 0;
            Turn<W> turn;
            if (l.turns) {
                const float *t = reinterpret_cast<const float *>(stage + sh.q_bytes + sh.k_bytes + sh.v_bytes) + H * l.lane;
                load_turn<W, INTERLEAVED>(turn, t, t + a.rotary / 2);
            }
            // rows of one kind: PER_WARP for each warp at a time, beginning with warp `first`
            const auto work = [&](Elt *rows, int heads, int first, bool norms, const f32x2 (&lo)[W], const f32x2 (&hi)[W]) {
                if (!norms && !a.table && live) return;
#pragma unroll 2
                for (int base = first * PER_WARP; base < heads; base += kConsumers * PER_WARP) {
                    const int row = base + lane / LANES;
                    Elt *x = rows + row * D;
                    Part<Elt> part{};
                    if (row < heads) {
                        load_piece<Elt, true>(part.lo, x + l.lo);
                        load_piece<Elt, true>(part.hi, x + l.hi);
                    }
                    norm_rotate<Elt, LANES, INTERLEAVED>(part, norms, norms, lo, hi, a.eps, l.turns, turn);
                    if (!live) part = Part<Elt>{};
                    if (row < heads) {
                        store_piece<Elt, true>(x + l.lo, part.lo);
                        store_piece<Elt, true>(x + l.hi, part.hi);
                    }
                }
            };
            work(reinterpret_cast<Elt *>(stage), a.q.heads, warp, a.q_weight != nullptr, q_lo, q_hi);
            work(reinterpret_cast<Elt *>(stage + sh.q_bytes), a.k.heads, kConsumers - 1 - warp, a.k_weight != nullptr, k_lo,
                 k_hi);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");    // before the bulk stores read it
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(done + st));
        }
    }
}

// What a call's operands allow: whole 8-byte pieces, whole 16-byte aligned rows one after another.
struct Alignment {
    bool pieces = true, rows = true;
};

template <typename Elt, int D, bool APPEND, bool INTERLEAVED>
cudaError_t launch_rotary(const RotaryArgs &a, Alignment align, int device, cudaStream_t stream) {
    constexpr int LANES = D * int(sizeof(Elt)) / 16;
    int sms = 148;
    cudaError_t err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (err != cudaSuccess) return err;
    // Streaming wherever the rows allow it and three tokens fit an SM, in as many CTAs as then have
    // three stages.  Against the direct kernel, us at 16 / 148 / 600 / 2000 tokens: rotating 32:8 FP16
    // heads of 128 3.1 / 3.2 / 5.7 / 10.9 against 4.3 / 4.5 / 7.1 / 14.0, appending 64:8 of them
    // 4.2 / 4.4 / 8.1 / 16.0 against 5.2 / 5.3 / 11.0 / 28.3.
    StreamShape sh{};
    const int row = D * int(sizeof(Elt));
    const int64_t token_bytes = (int64_t(a.q.heads + a.k.heads + a.v.heads) * row + a.rotary * 4 + 127) / 128 * 128;
    int ctas = kStreamCtas;
    while (ctas > 0 && token_bytes * kMinStages > kRingBytes[ctas]) --ctas;
    if (align.rows && ctas > 0) {
        sh.q_bytes = a.q.heads * row;
        sh.k_bytes = a.k.heads * row;
        sh.v_bytes = a.v.heads * row;
        sh.stage_bytes = int(token_bytes);
        sh.stages = std::min(kMaxStages, kRingBytes[ctas] / sh.stage_bytes);
        sh.smem = size_t(sh.stages) * sh.stage_bytes + kMaxStages * (8 + 8 + 8 + 4);
        const auto kernel = rotary_stream_kernel<Elt, D, APPEND, INTERLEAVED>;
        static std::atomic<uint64_t> allowed{0};    // devices on which this kernel may use its shared memory
        const uint64_t bit = unsigned(device) < 64 ? uint64_t(1) << device : 0;
        if (!(allowed.load(std::memory_order_relaxed) & bit)) {
            err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes[1] + 1024);
            if (err != cudaSuccess) return err;
            allowed.fetch_or(bit, std::memory_order_relaxed);
        }
        return launch_dependent(kernel, std::min<int64_t>(a.tokens, int64_t(ctas) * sms), kStreamThreads, sh.smem,
                                stream, a, sh);
    }
    // row slots: a thread's kRows rows cover the token, in whole warps
    const int rows = a.q.heads + a.k.heads + a.v.heads;
    int threads = (rows + kRows - 1) / kRows * LANES;
    threads = std::min(kMaxThreads, (threads + 31) / 32 * 32);
    const auto kernel = align.pieces ? rotary_kernel<Elt, D, true, APPEND, INTERLEAVED>
                                     : rotary_kernel<Elt, D, false, APPEND, INTERLEAVED>;
    return launch_dependent(kernel, a.tokens, threads, 0, stream, a);
}

template <typename Elt, int D>
cudaError_t launch_rotary(const RotaryArgs &a, Alignment align, bool append, int device, cudaStream_t stream) {
    const auto launch = append ? (a.interleaved ? launch_rotary<Elt, D, true, true> : launch_rotary<Elt, D, true, false>)
                               : (a.interleaved ? launch_rotary<Elt, D, false, true> : launch_rotary<Elt, D, false, false>);
    return launch(a, align, device, stream);
}

// Rows, strides and pointers of one operand, and what they allow.
pd_status check_rows(const pd_heads *h, const char *name, int elt, int head_dim, bool needs_out, Alignment *align,
                     HeadRows *rows) {
    *rows = HeadRows{};
    if (!h) return PD_OK;
    if (h->heads < 0 || h->heads > 65535) return fail(PD_ERR_VALUE, std::string(name) + ": heads must be in [0, 65535]");
    if (h->heads == 0) return PD_OK;
    if (!h->data || (needs_out && !h->out)) return fail(PD_ERR_VALUE, std::string(name) + " must not be NULL");
    const uintptr_t at = reinterpret_cast<uintptr_t>(h->data) | reinterpret_cast<uintptr_t>(needs_out ? h->out : nullptr);
    if (at & uintptr_t(elt - 1)) return fail(PD_ERR_VALUE, std::string(name) + " must be aligned to its element size");
    int64_t strides = h->token_stride | h->head_stride;
    if (needs_out) strides |= h->out_token_stride | h->out_head_stride;
    if ((at & 7) || ((strides * elt) & 7)) align->pieces = false;
    if ((at & 15) || ((strides * elt) & 15) || h->head_stride != head_dim || (needs_out && h->out_head_stride != head_dim))
        align->rows = false;
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

pd_status run_rotary(const RotaryArgs &a, int head_dim, pd_dtype dtype, Alignment align, bool append, int32_t device,
                     void *stream) {
    if (a.tokens > INT32_MAX) return fail(PD_ERR_VALUE, "too many tokens");
    if (a.tokens == 0 || a.q.heads + a.k.heads + a.v.heads == 0) return PD_OK;
    int prev = -1;
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    cudaError_t err = prev == device ? cudaSuccess : cudaSetDevice(device);
    if (err != cudaSuccess) return fail(PD_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(err));
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == PD_FLOAT16)
        err = head_dim == 64 ? launch_rotary<__half, 64>(a, align, append, device, st)
                             : launch_rotary<__half, 128>(a, align, append, device, st);
    else
        err = head_dim == 64 ? launch_rotary<float, 64>(a, align, append, device, st)
                             : launch_rotary<float, 128>(a, align, append, device, st);
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
    Alignment align;
    if (tokens == 0) return PD_OK;
    if ((s = check_rows(q, "q", elt, rotation->head_dim, true, &align, &a.q)) != PD_OK) return s;
    if ((s = check_rows(k, "k", elt, rotation->head_dim, true, &align, &a.k)) != PD_OK) return s;
    if (!positions || (reinterpret_cast<uintptr_t>(positions) & 3))
        return fail(PD_ERR_VALUE, "positions must be a 4-byte aligned device pointer");
    a.tokens = tokens;
    a.positions = positions;
    a.error = error;
    return run_rotary(a, rotation->head_dim, dtype, align, false, device, stream);
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
    Alignment align;
    if ((s = check_rows(q, "q", elt, L.head_dim, true, &align, &a.q)) != PD_OK) return s;
    if ((s = check_rows(k, "k", elt, L.head_dim, false, &align, &a.k)) != PD_OK) return s;
    if ((s = check_rows(v, "v", elt, L.head_dim, false, &align, &a.v)) != PD_OK) return s;
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
    a.page_shift = L.page_size == 16 ? 4 : 5;
    a.error = error;
    return run_rotary(a, L.head_dim, dtype, align, true, device, stream);
}
