// pd_prefix_mma.cuh — the FP16 shared-prefix kernel on the 5th-generation tensor cores.
//
// One CTA per work item.  An item has up to two streams, each one tile of 128
// query rows against a run of prefix pages, 128 tokens a step:
//   * paired: two row tiles of one (group, KV head) over the same pages; each
//     K and V step is loaded once and used by both;
//   * split: one row tile whose pages are cut in two runs; each stream loads
//     its own steps (few rows: the prefix's bytes bound the kernel, and two
//     streams keep both the loads and the softmax busy).
// Roles (10 warps):
//   * warps 0-3 / 4-7: softmax of stream 0 / 1, one thread per query row
//     (tensor-memory lane).  S is read from tensor memory, the weights go back
//     as FP16 over the scores' own columns, where the PV product reads them as
//     its A operand;
//   * warp 8, two lanes: TMA loads of K and V steps into one ring (one lane its
//     even slots, one its odd slots), one box per page;
//   * warp 9, one thread: the MMAs.  S = Q K^T (M 128, N 128), O += P V (M 128,
//     N = head dim).  While one stream's softmax works, the other's products run.
// The scores of step i + 1 overwrite the weights of step i, so they are issued
// once the PV product of step i has completed.
//
// Softmax in base 2 with a reference m that moves only when a score passes it
// by more than 2^15 (then O is rescaled in tensor memory): a fresh reference is
// 2^7 below the step's maximum, so weights stay within (0, 2^15] and FP16 keeps
// its full precision down to 2^-21 of the largest.  The denominator sums the
// FP32 weights.  Rows are either in use for the whole prefix or their results
// are dropped (a live length inside the prefix: the merge kernel's slow path),
// so no scores need masks; a last step of fewer pages takes fewer columns.
//
// Every wait is bounded; on a timeout the CTA records PD_DEVERR_TIMEOUT,
// unwinds, waits for its own MMAs and frees its tensor memory.
#pragma once

#include "paged_decode.h"
#include "pd_device.cuh"
#include "pd_prefix_args.cuh"
#include "pd_tcgen05.cuh"

namespace pd {

template <int D, int T>
struct PrefixShape {
    static constexpr int M = 128, NS = 128;             // rows of a tile, tokens of a step
    static constexpr int NP = NS / T;                   // pages of a step
    static constexpr int NBOX = D * 2 / 128;            // 128-byte boxes per row
    static constexpr int PAGE_BYTES = T * D * 2;        // K (or V) rows of one page and head
    static constexpr int STEP_BYTES = NP * PAGE_BYTES;
    static constexpr int Q_BOX = M * 128;
    static constexpr int Q_BYTES = NBOX * Q_BOX;
    static constexpr int SLOTS = D == 128 ? 5 : 8;      // ring slots of one K or V step
    static constexpr int SOFTMAX_WARPS = 8, W_LOAD = 8, W_MMA = 9;
    static constexpr int THREADS = 320;
    static constexpr int S_COL = 0, O_COL = 2 * NS;     // tensor memory: [S0 | P0][S1 | P1][O0][O1]
    static constexpr int TMEM_COLS = 512;
    static constexpr int NBARS = 2 * SLOTS + 2 * 4 + 1;
    static constexpr size_t SMEM = 1024 + 2 * size_t(Q_BYTES) + size_t(SLOTS) * STEP_BYTES + NBARS * 8 + 16;
    static_assert(O_COL + 2 * D <= TMEM_COLS, "tensor memory budget");
    static_assert(SMEM <= 232448 && SMEM > 116 * 1024, "one CTA per SM: tensor memory is never contended");
};

__device__ __forceinline__ float ex2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// One stream of a work item.
struct PrefixStream {
    int tile, first, end, slot;     // row tile, page run within the group's prefix, partial slot
    __device__ __forceinline__ int steps(int np) const { return (end - first + np - 1) / np; }
};

struct PrefixItem {
    int member0, members, head, paired;
    int page0;
    PrefixStream s0, s1;            // an absent stream has end == first
    __device__ __forceinline__ PrefixStream s(int t) const {
        return PrefixStream{t ? s1.tile : s0.tile, t ? s1.first : s0.first, t ? s1.end : s0.end, t ? s1.slot : s0.slot};
    }
};

__device__ __forceinline__ PrefixItem prefix_item(const PrefixArgs &a, int i) {
    const int4 x = __ldg(a.items + 4 * i), y = __ldg(a.items + 4 * i + 1);
    const int4 z = __ldg(a.items + 4 * i + 2), w = __ldg(a.items + 4 * i + 3);
    PrefixItem it;
    it.member0 = x.x, it.members = x.y, it.head = x.z, it.paired = x.w;
    it.page0 = y.x;
    it.s0 = PrefixStream{z.x, z.y, z.z, z.w};
    it.s1 = PrefixStream{w.x, w.y, w.z, w.w};
    return it;
}

// The order in which the MMA thread uses the ring: the first K of each stream,
// then per step and stream V and the next K; paired streams share stream 0's.
// use(position, stream, is_v, step) is called for each.
template <typename Use>
__device__ __forceinline__ void ring_order(int n0, int n1, bool paired, Use use) {
    const int streams = paired ? 1 : 2;
    int pos = 0;
    for (int t = 0; t < streams; ++t)
        if ((t ? n1 : n0) > 0 && !use(pos++, t, false, 0)) return;
    for (int i = 0; i < n0; ++i)
        for (int t = 0; t < streams; ++t) {
            const int n = t ? n1 : n0;
            if (i < n && !use(pos++, t, true, i)) return;
            if (i + 1 < n && !use(pos++, t, false, i + 1)) return;
        }
}

template <int D, int T>
__global__ void __launch_bounds__(PrefixShape<D, T>::THREADS, 1)
    prefix_mma_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const PrefixArgs a) {
    using S = PrefixShape<D, T>;
    constexpr int NP = S::NP, SLOTS = S::SLOTS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *qbuf = smem;                                   // [2][box][128 rows][128 B]
    uint8_t *ring = qbuf + 2 * S::Q_BYTES;                  // [SLOTS][STEP_BYTES]
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + size_t(SLOTS) * S::STEP_BYTES);
    uint64_t *empty = full + SLOTS;
    uint64_t *q_full = empty + SLOTS;       // [2] query rows written (4 warps)
    uint64_t *s_full = q_full + 2;          // [2] scores done
    uint64_t *p_full = s_full + 2;          // [2] weights written (4 warps)
    uint64_t *o_done = p_full + 2;          // [2] PV product done
    uint64_t *mma_done = o_done + 2;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(mma_done + 1);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1) + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(smem_u32(full + s), 1);
            mbar_init(smem_u32(empty + s), 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(smem_u32(q_full + t), 4);
            mbar_init(smem_u32(s_full + t), 1);
            mbar_init(smem_u32(p_full + t), 4);
            mbar_init(smem_u32(o_done + t), 1);
        }
        mbar_init(smem_u32(mma_done), 1);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == S::W_MMA) {
        tc::alloc(smem_u32(tmem_slot), S::TMEM_COLS);
        tc::relinquish_alloc_permit();
        tc::fence_before_sync();
    }
    const PrefixItem it = prefix_item(a, blockIdx.x);
    const int n0 = it.s0.steps(NP), n1 = it.s1.steps(NP);   // n1 <= n0; paired: n1 == n0
    const bool paired = it.paired != 0;
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // With a suffix decode in front, q, the caches and the lengths are complete (it waited for
    // their writers before any CTA of this grid could start) and only its rows are not.
    if (!a.rows) asm volatile("griddepcontrol.wait;" ::: "memory");

    const auto fail_wait = [&]() {
        if (!*abort_flag) atomicOr(a.error, PD_DEVERR_TIMEOUT);
        *abort_flag = 1;
    };

    if (warp == S::W_LOAD) {
        // ------------------------------------------------------------ loads
        if (lane < 2) {
            tma_prefetch_descriptor(lane == 0 ? &tm_k : &tm_v);
            int last = -1;              // the last position this lane loaded
            ring_order(n0, n1, paired, [&](int pos, int t, bool is_v, int step) {
                if ((pos % SLOTS & 1) != lane) return true;
                const int p0 = it.s(t).first + step * NP, n = min(NP, it.s(t).end - p0);
                int ids[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) ids[p] = p < n ? __ldg(a.pages + it.page0 + p0 + p) : 0;
                const int slot = pos % SLOTS, use = pos / SLOTS;
                if (use > 0) {      // both lanes are of one warp: poll without suspending it
                    const unsigned long long t0 = global_ns();
                    while (!mbar_test_wait(smem_u32(empty + slot), (use - 1) & 1)) {
                        if (*abort_flag) return false;
                        if (global_ns() - t0 > kWaitTimeoutNs) {
                            fail_wait();
                            return false;
                        }
                    }
                }
                last = pos;
                const uint32_t bar = smem_u32(full + slot), dst = smem_u32(ring + size_t(slot) * S::STEP_BYTES);
                mbar_arrive_expect_tx(bar, uint32_t(n) * S::PAGE_BYTES);
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    if (p >= n) continue;
                    if (is_v) tma_load_5d(dst + p * S::PAGE_BYTES, &tm_v, 0, 0, 0, it.head, ids[p], bar);
                    else tma_load_5d(dst + p * S::PAGE_BYTES, &tm_k, 0, 0, it.head * S::NBOX, 0, ids[p], bar);
                }
                return true;
            });
            // no copy of this lane is in flight when the CTA ends, whatever became of its readers
            for (int pos = last; pos >= 0 && pos > last - SLOTS; --pos)
                if ((pos % SLOTS & 1) == lane && !mbar_wait(smem_u32(full + pos % SLOTS), (pos / SLOTS) & 1)) fail_wait();
        }
        __syncwarp();
    } else if (warp == S::W_MMA) {
        // ------------------------------------------------------------ MMAs (one thread)
        if (lane == 0) {
            constexpr uint32_t ID_S = tc::idesc_f16_f32(S::M, S::NS, false, false);   // Q, K: K-major
            constexpr uint32_t ID_O = tc::idesc_f16_f32(S::M, D, false, true);        // V: MN-major
            bool ok = true;
            int pos = 0;                // ring positions used
            const auto take = [&]() {   // wait for the next position's data
                ok = ok && mbar_wait(smem_u32(full + pos % SLOTS), (pos / SLOTS) & 1);
                return smem_u32(ring + size_t(pos % SLOTS) * S::STEP_BYTES);
            };
            const auto give = [&]() { tc::commit(smem_u32(empty + pos++ % SLOTS)); };
            const auto scores = [&](int t, uint32_t kb) {
                const uint32_t qa = smem_u32(qbuf + (paired ? t : 0) * S::Q_BYTES);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint64_t ad =
                        tc::smem_desc(qa + (kk >> 2) * S::Q_BOX + (kk & 3) * 32, 16, 1024, tc::kSwizzle128);
                    const uint64_t bd =
                        tc::smem_desc(kb + (kk >> 2) * 1024 + (kk & 3) * 32, 16, S::NBOX * 1024, tc::kSwizzle128);
                    tc::mma_f16(tmem + S::S_COL + t * S::NS, ad, bd, ID_S, kk > 0 ? 1u : 0u);
                }
                tc::commit(smem_u32(s_full + t));
            };
            const auto products = [&](int t, uint32_t vb, int tokens, bool first) {
#pragma unroll 1
                for (int kk = 0; kk < tokens / 16; ++kk) {
                    const uint32_t page = vb + kk * 16 / T * S::PAGE_BYTES;
                    const uint64_t bd = tc::smem_desc(page + kk * 16 % T * 128, T * 128, 1024, tc::kSwizzle128);
                    tc::mma_f16_ta(tmem + S::O_COL + t * D, tmem + S::S_COL + t * S::NS + kk * 8, bd, ID_O,
                                   first && kk == 0 ? 0u : 1u);
                }
                tc::commit(smem_u32(o_done + t));
            };
            const int streams = n1 > 0 ? 2 : 1;
            uint32_t kb = 0, vb = 0;
            for (int t = 0; t < streams && ok; ++t) {
                const bool own = t == 0 || !paired;     // this stream's first use of its ring position
                if (own) kb = take();
                if (t == 0 || paired) ok = ok && mbar_wait(smem_u32(q_full + t), 0);
                if (!ok) break;
                tc::fence_after_sync();
                scores(t, kb);
                if (!paired || t == streams - 1) give();
            }
            // Paired: positions K0, V0, K1, V1, ..; a step's V and the next step's K are
            // taken by stream 0 and given back by stream 1, so both are open at once.
            for (int i = 0; i < n0 && ok; ++i) {
                const int base = pos;
                for (int t = 0; t < streams && ok; ++t) {
                    const int n = t ? n1 : n0;
                    if (i >= n) continue;
                    if (paired) pos = base;
                    const int p0 = it.s(t).first + i * NP;
                    if (t == 0 || !paired) vb = take();
                    ok = ok && !*abort_flag && mbar_wait(smem_u32(p_full + t), i & 1);
                    if (!ok) break;
                    tc::fence_after_sync();
                    products(t, vb, min(NP, it.s(t).end - p0) * T, i == 0);
                    if (!paired || t == streams - 1) give();
                    else ++pos;
                    if (i + 1 >= n) continue;
                    if (t == 0 || !paired) kb = take();
                    // the next scores overwrite the weights that this product reads
                    ok = ok && mbar_wait(smem_u32(o_done + t), i & 1);
                    if (!ok) break;
                    tc::fence_after_sync();
                    scores(t, kb);
                    if (!paired || t == streams - 1) give();
                    else ++pos;
                }
            }
            if (!ok) fail_wait();
            // every MMA has finished before shared and tensor memory go
            tc::commit(smem_u32(mma_done));
            if (!mbar_wait(smem_u32(mma_done), 0)) fail_wait();
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax, one thread per row
        const int t = warp >> 2, quad = warp & 3, r = 32 * quad + lane;
        const PrefixStream st = it.s(t);
        const int n = t ? n1 : n0;
        if (t == 0 || paired) {
            // the tile's query rows, 16-byte chunks XORed by row % 8 (K-major, 128-byte swizzle)
            constexpr int CPR = D / 8;
            uint8_t *qs = qbuf + t * S::Q_BYTES;
#pragma unroll 4
            for (int e = threadIdx.x & 127; e < S::M * CPR; e += 128) {
                const int row = e / CPR, c = e % CPR, gr = st.tile * S::M + row, member = gr / a.group;
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (member < it.members) {
                    const int64_t b = __ldg(a.members + it.member0 + member);
                    const int64_t at = (b * a.Hq + it.head * a.group + gr % a.group) * D;
                    x = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const __half *>(a.q) + at) + c);
                }
                *reinterpret_cast<uint4 *>(qs + swz128<S::M>(row, c)) = x;
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(q_full + t));
        }
        const uint32_t lanes = uint32_t(32 * quad) << 16;
        const uint32_t ts = tmem + lanes + S::S_COL + t * S::NS, to = tmem + lanes + S::O_COL + t * D;
        const auto warp_wait = [&](uint64_t *bar, int parity) {
            return __all_sync(kFullMask, mbar_wait(smem_u32(bar), uint32_t(parity)));
        };
        float m = -INFINITY;                            // the row's reference
        unsigned long long l2 = 0;                      // two partial denominators
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            if (!warp_wait(s_full + t, i & 1)) {
                ok = false;
                break;
            }
            tc::fence_after_sync();
            // columns past the run's last page hold scores of stale rows
            const int live = min(NP, st.end - st.first - i * NP) * T;
            uint32_t x[32], y[32];
            const auto load = [&](uint32_t (&v)[32], int c) { tc::ld_32x32b_x32(ts + 32 * c, v); };
            const auto mask = [&](uint32_t (&v)[32], int c) {
                if (live < S::NS)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * c + e >= live) v[e] = __float_as_uint(-INFINITY);
            };
            float top0 = -INFINITY, top1 = -INFINITY;
            const auto raise = [&]() {
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    top0 = max3(top0, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
                    top1 = max3(top1, __uint_as_float(y[e]), __uint_as_float(y[e + 1]));
                }
            };
            // Two passes over the 128 scores, 64 of them held in registers: the upper half is
            // read twice.  (All 128 at once spill.)
            load(x, 2);
            load(y, 3);
            tc::wait_ld();
            mask(x, 2);
            mask(y, 3);
            raise();
            load(x, 0);
            load(y, 1);
            tc::wait_ld();
            mask(x, 0);
            mask(y, 1);
            raise();
            const float peak = fmaxf(top0, top1) * a.scale_log2;
            const bool moves = peak > m + 15.f;
            if (__any_sync(kFullMask, moves)) {
                const float next = moves ? peak - 7.f : m;
                const float f = next == -INFINITY ? 1.f : ex2_approx(m - next);
                if (i > 0) {
                    if (!warp_wait(o_done + t, (i - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    tc::fence_after_sync();
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tc::ld_32x32b_x32(to + c, o);
                        tc::wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tc::st_32x32b_x32(to + c, o);
                    }
                    tc::wait_st();
                }
                const float2 l = unpack_f32x2(l2);
                l2 = pack_f32x2(l.x * f, l.y * f);
                m = next;
            }
            const float base = m == -INFINITY ? 0.f : m;
            const unsigned long long scale2 = pack_f32x2(a.scale_log2, a.scale_log2), base2 = pack_f32x2(-base, -base);
            // 32 weights into columns [16 c, 16 c + 16), where the scores have been read
            const auto emit = [&](const uint32_t (&v)[32], int c) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float2 z = unpack_f32x2(fma_f32x2(
                        pack_f32x2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), scale2, base2));
                    const float w0 = ex2_approx(z.x), w1 = ex2_approx(z.y);
                    l2 = add_f32x2(l2, pack_f32x2(w0, w1));
                    p[e] = pack_half2(w0, w1);
                }
                tc::st_32x32b_x16(ts + 16 * c, p);
            };
            emit(x, 0);
            load(x, 2);
            emit(y, 1);
            load(y, 3);
            tc::wait_ld();
            mask(x, 2);
            mask(y, 3);
            emit(x, 2);
            emit(y, 3);
            tc::wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(p_full + t));
        }
        if (!ok && lane == 0) fail_wait();
        // ------------------------------------------------------------ partial
        if (n > 0 && ok) {
            ok = warp_wait(o_done + t, (n - 1) & 1);
            if (!ok && lane == 0) fail_wait();
        }
        if (n > 0 && ok) {
            tc::fence_after_sync();
            const float2 l = unpack_f32x2(l2);
            const int64_t row = int64_t(st.slot) * S::M + r;
            const bool on = (st.tile * S::M + r) / a.group < it.members;
            float *dst = a.part_o + row * D;
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tc::ld_32x32b_x32(to + c, o);
                tc::wait_ld();
                if (on)
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4 *>(dst + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
            if (on) a.part_ml[row] = make_float2(m, l.x + l.y);
            tc::fence_before_sync();
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __syncthreads();
    tc::fence_after_sync();
    if (warp == S::W_MMA) tc::dealloc(tmem, S::TMEM_COLS);
    // the suffix decode's rows are complete when this grid is
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace pd
