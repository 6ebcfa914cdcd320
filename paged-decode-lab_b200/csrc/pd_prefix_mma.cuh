// pd_prefix_mma.cuh — the FP16 shared-prefix kernel on the 5th-generation tensor cores.
//
// One CTA per work item.  An item has up to two streams, each one tile of 128
// query rows against a run of prefix pages, 64 tokens a step:
//   * paired: two row tiles of one (group, KV head) over the same pages; each
//     K and V step is loaded once and used by both;
//   * split: one row tile whose pages are cut in two runs; each stream loads
//     its own steps (few rows: the prefix's bytes bound the kernel, and two
//     streams keep both the loads and the softmax busy).
// Roles (12 warps):
//   * warps 0-3 / 4-7: softmax of stream 0 / 1, one thread per query row
//     (tensor-memory lane).  S is read from tensor memory, the weights go back
//     as FP16 over the scores' own columns, where the PV product reads them as
//     its A operand;
//   * warps 8 / 9, one elected lane each: the MMAs of stream 0 / 1.  S = Q K^T
//     (M 128, N 64), O += P V (M 128, N = head dim);
//   * warps 10 / 11, one elected lane each: TMA loads of K and V steps into rings
//     of shared memory, one box per page.
// Each stream has two score blocks, so that a softmax finds its next scores
// ready: those of step i + 2 are issued once the PV product of step i, whose
// weights lie in the same block, has completed.  (Steps of 128 tokens leave
// tensor memory for one block per stream: every step then waited for PV, QK and
// softmax one after another; 188 us against 180 with 256 sequences of 64:8 heads.)
//
// Softmax in base 2 with a reference m that moves only when a score passes it
// by more than 2^15 (then O is rescaled in tensor memory): a fresh reference is
// 2^7 below the step's maximum, so weights stay within (0, 2^15] and FP16 keeps
// its full precision down to 2^-21 of the largest.  The denominator sums the
// rounded weights, as the warp-level decode kernel does, so that o / l stays an average
// of the values (both in FP32).  Rows are either in use for the whole prefix or their results
// are dropped (a live length inside the prefix, or other pages there: the merge kernel's slow path),
// so no scores need masks; a last step of fewer pages takes fewer columns.
//
// Each stream leaves its rows' (m, l, o) as a partial for the merge kernel.  The
// grid is kept smaller than the device: once its CTAs have started, the suffix's decode
// kernel runs beside it on the other SMs.
//
// Bound by the tensor core and the exponentials alike: a 64-token step of both
// streams counts 1280 cycles of MMAs (if scores of N 64 read shared memory at its
// limit) and 1024 of ex2.  Measured on a B200, between lengths of 16384 and 65536
// tokens (256 sequences of 64:8 heads of 128, 128 CTAs): 0.95 us a step of both streams, 1.13
// PFLOP/s (0.87 and 1.23 with the unrounded weights' sum, two of which take one addition; up
// to 12288 tokens the times are alike); with few rows the loads bound it: 8 sequences of 32:8 heads behind
// 131072 tokens 91 us with the merge, 5.9 TB/s.
//
// Every wait is bounded; on a timeout the CTA records PD_DEVERR_TIMEOUT,
// unwinds, waits for its own MMAs and copies and frees its tensor memory.
#pragma once

#include "paged_decode.h"
#include "pd_device.cuh"
#include "pd_prefix_args.cuh"
#include "pd_tcgen05.cuh"

namespace pd {

template <int D, int T>
struct PrefixShape {
    static constexpr int M = 128, NS = 64;              // rows of a tile, tokens of a step
    static constexpr int NP = NS / T;                   // pages of a step
    static constexpr int NBOX = D * 2 / 128;            // 128-byte boxes per row
    static constexpr int PAGE_BYTES = T * D * 2;        // K (or V) rows of one page and head
    static constexpr int STEP_BYTES = NP * PAGE_BYTES;
    static constexpr int Q_BOX = M * 128;
    static constexpr int Q_BYTES = NBOX * Q_BOX;
    static constexpr int K_SLOTS = D == 128 ? 2 : 4, V_SLOTS = D == 128 ? 3 : 4;   // of one step, per stream
    static constexpr int SLOTS = 2 * (K_SLOTS + V_SLOTS);
    static constexpr int SOFTMAX_WARPS = 8, W_MMA = 8, W_LOAD = 10;     // and one more of each kind
    static constexpr int THREADS = 384;
    // tensor memory: score blocks (weights in their first half) [stream][2], outputs [stream]
    static constexpr int S_COL = 0, O_COL = 4 * NS;
    static constexpr int TMEM_COLS = 512;
    static constexpr int NBARS = 2 * SLOTS + 2 + 4 + 4 + 2 + 2 + 1;
    static constexpr size_t SMEM = 1024 + 2 * size_t(Q_BYTES) + size_t(SLOTS) * STEP_BYTES + NBARS * 8 + 16 + 2 * M * 4;
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

// x += the low FP16 of v, y += the high one, in FP32.
__device__ __forceinline__ void add_halves(float &x, float &y, uint32_t v) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tadd.rn.f32.f16 %0, a, %0;\n\tadd.rn.f32.f16 %1, b, %1;\n\t}"
        : "+f"(x), "+f"(y)
        : "r"(v));
}

// A read-only load that stays where it is written: its result is used much later.
__device__ __forceinline__ int32_t load_here(const int32_t *p) {
    int32_t r;
    asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(r) : "l"(p));
    return r;
}

// 32 bytes: a whole sector by one thread.
__device__ __forceinline__ void store_sector(void *p, const uint32_t *r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// One stream of a work item.
struct PrefixStream {
    int tile, first, end, slot;     // row tile, page run within the group's prefix, partial slot
    __device__ __forceinline__ int steps(int np) const { return (end - first + np - 1) / np; }
};

struct PrefixItem {
    int member0, members, head, kind;
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
    it.member0 = x.x, it.members = x.y, it.head = x.z, it.kind = x.w;
    it.page0 = y.x;
    it.s0 = PrefixStream{z.x, z.y, z.z, z.w};
    it.s1 = PrefixStream{w.x, w.y, w.z, w.w};
    return it;
}

// Cursor over a run of ring slots; `phase` is the parity of the slot's current use.
struct RingCursor {
    int first, count, slot, phase;
    __device__ __forceinline__ void next() {
        if (++slot == first + count) {
            slot = first;
            phase ^= 1;
        }
    }
};

// K and V steps have slots of their own: paired streams share 2 K_SLOTS and 2
// V_SLOTS of them, split streams have half each.
template <typename S>
__device__ __forceinline__ RingCursor k_cursor(int t, bool paired) {
    const int first = paired ? 0 : t * S::K_SLOTS;
    return RingCursor{first, paired ? 2 * S::K_SLOTS : S::K_SLOTS, first, 0};
}
template <typename S>
__device__ __forceinline__ RingCursor v_cursor(int t, bool paired) {
    const int first = 2 * S::K_SLOTS + (paired ? 0 : t * S::V_SLOTS);
    return RingCursor{first, paired ? 2 * S::V_SLOTS : S::V_SLOTS, first, 0};
}

// LIVE: a dynamic launch.
template <int D, int T, bool LIVE>
__global__ void __launch_bounds__(PrefixShape<D, T>::THREADS, 1)
    prefix_mma_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ PrefixArgs a) {
    using S = PrefixShape<D, T>;
    constexpr int NP = S::NP, SLOTS = S::SLOTS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *qbuf = smem;                                   // [2][box][128 rows][128 B]
    uint8_t *ring = qbuf + 2 * S::Q_BYTES;                  // [SLOTS][STEP_BYTES]
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + size_t(SLOTS) * S::STEP_BYTES);
    uint64_t *empty = full + SLOTS;
    uint64_t *q_full = empty + SLOTS;       // [2] query rows written (4 warps)
    uint64_t *s_full = q_full + 2;          // [stream][block] scores done
    uint64_t *p_full = s_full + 4;          // [stream][block] weights written (4 warps)
    uint64_t *o_done = p_full + 4;          // [stream] PV product done
    uint64_t *o_last = o_done + 2;          // [stream] the last PV product done
    uint64_t *mma_done = o_last + 2;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(mma_done + 1);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1) + 1;
    int *moved = reinterpret_cast<int *>(mma_done + 1) + 4;     // [stream][a member's first row of the tile]

    const int warp = int(__reduce_max_sync(kFullMask, threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const PrefixItem it = prefix_item(a, blockIdx.x);
    const int n0 = it.s0.steps(NP), n1 = it.s1.steps(NP);   // n1 <= n0; paired: n1 == n0
    const bool paired = it.kind == kItemPaired;
    // Warps 8 to 11 stay converged, and what they hand to the hardware is the same in all lanes
    // (reductions over the warp give the compiler the proof): operands then live in uniform registers.
    const auto uniform = [](int x) { return __reduce_max_sync(kFullMask, x); };
    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(smem_u32(full + s), 1);
            mbar_init(smem_u32(empty + s), 1 + (paired ? 1 : 0));   // a commit per stream that reads it
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(smem_u32(q_full + t), 4);
            mbar_init(smem_u32(o_done + t), 1);
            mbar_init(smem_u32(o_last + t), 1);
            for (int b = 0; b < 2; ++b) {
                mbar_init(smem_u32(s_full + 2 * t + b), 1);
                mbar_init(smem_u32(p_full + 2 * t + b), 4);
            }
        }
        mbar_init(smem_u32(mma_done), 2);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == S::W_MMA) {
        tc::alloc(smem_u32(tmem_slot), S::TMEM_COLS);
        tc::relinquish_alloc_permit();
        tc::fence_before_sync();
    }
    if (LIVE && threadIdx.x < 2 * S::M) moved[threadIdx.x] = 0;
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const auto fail_wait = [&]() {
        if (!*abort_flag) atomicOr(a.error, PD_DEVERR_TIMEOUT);
        *abort_flag = 1;
    };

    if (warp >= S::W_LOAD) {
        // ------------------------------------------------------------ loads
        const int w = warp - S::W_LOAD;
        const bool upaired = uniform(it.kind) == kItemPaired;
        const int head = uniform(it.head);
        // one sequence of steps: K or V of a stream, with page ids 32 at a time, one per lane
        struct Feed {
            RingCursor at;
            int first, end, steps, done, window, base;
        };
        const auto feed = [&](RingCursor at, const PrefixStream &st) {
            return Feed{at, uniform(st.first), uniform(st.end), uniform(st.steps(NP)), 0, 0, -64};
        };
        bool ok = true;
        const auto load = [&](Feed &f, bool is_v) {
            if (!ok || f.done >= f.steps) return;
            const int p0 = f.first + f.done * NP, n = min(NP, f.end - p0);
            if (p0 + NP > f.base + 32) {
                f.base = p0;
                f.window = p0 + lane < f.end ? __ldg(a.pages + it.page0 + p0 + lane) : 0;
            }
            // (a fresh barrier's preceding phase counts as complete: the first pass does not wait)
            ok = __all_sync(kFullMask, mbar_wait(smem_u32(empty + f.at.slot), uint32_t(f.at.phase ^ 1))) &&
                 !__any_sync(kFullMask, *abort_flag != 0);
            if (!ok) return;
            const uint32_t bar = smem_u32(full + f.at.slot);
            const uint32_t dst = smem_u32(ring) + uint32_t(f.at.slot) * S::STEP_BYTES;
            if (lane == 0) mbar_arrive_expect_tx(bar, uint32_t(n) * S::PAGE_BYTES);
            __syncwarp();
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                if (p >= n) continue;
                const int id = uniform(__shfl_sync(kFullMask, f.window, p0 - f.base + p));
                if (is_v) tma_load_5d_warp(dst + p * S::PAGE_BYTES, &tm_v, 0, 0, 0, head, id, bar);
                else tma_load_5d_warp(dst + p * S::PAGE_BYTES, &tm_k, 0, 0, head * S::NBOX, 0, id, bar);
            }
            f.at.next();
            ++f.done;
        };
        // paired streams: one warp brings K, the other V; split streams: a warp each, K two steps ahead
        Feed fk = feed(k_cursor<S>(upaired ? 0 : w, upaired), it.s(upaired ? 0 : w));
        Feed fv = feed(v_cursor<S>(upaired ? 0 : w, upaired), it.s(upaired ? 0 : w));
        if (upaired && w == 0) fv.steps = 0;
        if (upaired && w == 1) fk.steps = 0;
        load(fk, false);
        load(fk, false);
        while (ok && (fk.done < fk.steps || fv.done < fv.steps)) {
            load(fv, true);
            load(fk, false);
        }
        if (!ok && lane == 0) fail_wait();
        // no copy is in flight when the CTA ends, whatever became of its readers
        const auto drain = [&](const Feed &f) {
            for (int i = 0; i < min(f.at.count, f.done); ++i) {
                const int slot = f.at.first + i;
                const int phase = slot < f.at.slot ? f.at.phase : f.at.phase ^ 1;    // of its last use
                if (!mbar_wait(smem_u32(full + slot), uint32_t(phase)) && lane == 0) fail_wait();
            }
        };
        drain(fk);
        drain(fv);
        __syncwarp();
    } else if (warp >= S::W_MMA) {
        // ------------------------------------------------------------ MMAs of one stream (one elected lane)
        const int t = warp - S::W_MMA;
        const bool upaired = uniform(it.kind) == kItemPaired;
        const int un = uniform(t ? n1 : n0);
        const int pages = uniform(t ? it.s1.end - it.s1.first : it.s0.end - it.s0.first);
        const uint32_t utmem = __reduce_max_sync(kFullMask, tmem);
        constexpr uint32_t ID_S = tc::idesc_f16_f32(S::M, S::NS, false, false);   // Q, K: K-major
        constexpr uint32_t ID_O = tc::idesc_f16_f32(S::M, D, false, true);        // V: MN-major
        const uint64_t q_desc =
            tc::smem_desc(smem_u32(qbuf) + (upaired && t ? S::Q_BYTES : 0), 16, 1024, tc::kSwizzle128);
        const uint64_t k_desc = tc::smem_desc(smem_u32(ring), 16, S::NBOX * 1024, tc::kSwizzle128);
        const uint64_t v_desc = tc::smem_desc(smem_u32(ring), T * 128, 1024, tc::kSwizzle128);
        const uint32_t s_block = utmem + S::S_COL + 2 * t * S::NS, o_block = utmem + S::O_COL + t * D;
        RingCursor kr = k_cursor<S>(t, upaired), vr = v_cursor<S>(t, upaired);
        bool ok = true;
        const auto wait_for = [&](uint64_t *bar, int phase) {
            ok = ok && __all_sync(kFullMask, mbar_wait(smem_u32(bar), uint32_t(phase & 1)));
        };
        // scores of step j into block j % 2
        const auto scores = [&](int j) {
            wait_for(full + kr.slot, kr.phase);
            if (!ok) return;
            tc::fence_after_sync();
            const uint64_t bd = k_desc + uint32_t(kr.slot) * (S::STEP_BYTES >> 4);
            const uint32_t d = s_block + (j & 1) * S::NS;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
                tc::mma_f16_warp(d, q_desc + (((kk >> 2) * S::Q_BOX + (kk & 3) * 32) >> 4),
                                 bd + (((kk >> 2) * 1024 + (kk & 3) * 32) >> 4), ID_S, kk > 0 ? 1u : 0u);
            tc::commit_warp(smem_u32(s_full + 2 * t + (j & 1)));
            tc::commit_warp(smem_u32(empty + kr.slot));
            kr.next();
        };
        if (un > 0) wait_for(q_full + (upaired ? t : 0), 0);
        for (int j = 0; j < min(un, 2) && ok; ++j) scores(j);
        for (int i = 0; i < un && ok; ++i) {
            wait_for(full + vr.slot, vr.phase);
            wait_for(p_full + 2 * t + (i & 1), i >> 1);
            if (!ok) break;
            tc::fence_after_sync();
            const uint64_t bd = v_desc + uint32_t(vr.slot) * (S::STEP_BYTES >> 4);
            const uint32_t p = s_block + (i & 1) * S::NS;
            const int blocks = min(NP, pages - i * NP) * (T / 16);    // of 16 tokens
#pragma unroll
            for (int kk = 0; kk < S::NS / 16; ++kk)
                if (kk < blocks)
                    tc::mma_f16_ta_warp(o_block, p + kk * 8,
                                        bd + ((kk * 16 / T * S::PAGE_BYTES + kk * 16 % T * 128) >> 4), ID_O,
                                        i == 0 && kk == 0 ? 0u : 1u);
            tc::commit_warp(smem_u32(i + 1 < un ? o_done + t : o_last + t));
            tc::commit_warp(smem_u32(empty + vr.slot));
            vr.next();
            if (i + 2 < un) {
                wait_for(o_done + t, i);    // the next scores overwrite this step's weights
                if (ok) scores(i + 2);
                ok = ok && !__any_sync(kFullMask, *abort_flag != 0);
            }
        }
        if (!ok && lane == 0) fail_wait();
        // every MMA has finished before shared and tensor memory go
        tc::commit_warp(smem_u32(mma_done));
        if (!mbar_wait(smem_u32(mma_done), 0) && lane == 0) fail_wait();
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
#pragma unroll
            for (int j = 0; j < CPR; ++j) {
                const int e = j * 128 + (threadIdx.x & 127), row = e / CPR, c = e % CPR;
                const int gr = st.tile * S::M + row, member = gr / a.group;
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
        // A dynamic launch: whether the live table of the row's member has other pages in this run.  The threads of
        // a member's rows share the pages of each step, whose ids come while its scores do.
        const int row = st.tile * S::M + r, member = row / a.group;
        const int first_row = max(0, member * a.group - st.tile * S::M);
        const int32_t *live_ids = nullptr, *planned_ids = a.pages + it.page0 + st.first;
        const int mate = r - first_row, mates = min(S::M, (member + 1) * a.group - st.tile * S::M) - first_row;
        bool other = false;
        if (LIVE && member < it.members && mate < NP)
            live_ids = a.table + __ldg(a.members + it.member0 + member) * a.width + st.first;
        if (LIVE && live_ids)           // a member with fewer rows than a step has pages: the others at once
            for (int p = mate + mates; p < NP; p += mates)
#pragma unroll 4
                for (int at = p; at < st.end - st.first; at += NP)
                    other = other | (__ldg(live_ids + at) != __ldg(planned_ids + at));
        const uint32_t lanes = uint32_t(32 * quad) << 16;
        const uint32_t ts = tmem + lanes + S::S_COL + 2 * t * S::NS, to = tmem + lanes + S::O_COL + t * D;
        const auto warp_wait = [&](uint64_t *bar, int parity) {
            return __all_sync(kFullMask, mbar_wait(smem_u32(bar), uint32_t(parity)));
        };
        float m = -INFINITY;                            // the row's reference
        float l[4] = {0.f, 0.f, 0.f, 0.f};              // partial denominators
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            int32_t id = 0, planned = 0;                // of page `mate` of the step; compared at its end
            if (LIVE && live_ids) {
                const int end = min((i + 1) * NP, st.end - st.first), at = i * NP + mate;
                if (at < end) id = load_here(live_ids + at), planned = load_here(planned_ids + at);
            }
            if (!warp_wait(s_full + 2 * t + (i & 1), i >> 1 & 1)) {
                ok = false;
                break;
            }
            tc::fence_after_sync();
            const uint32_t block = ts + (i & 1) * S::NS;
            uint32_t x[32], y[32];
            tc::ld_32x32b_x32(block, x);
            tc::ld_32x32b_x32(block + 32, y);
            tc::wait_ld();
            // columns past the run's last page hold scores of stale rows
            const int live = min(NP, st.end - st.first - i * NP) * T;
            if (live < S::NS) {
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    if (e >= live) x[e] = __float_as_uint(-INFINITY);
                    if (32 + e >= live) y[e] = __float_as_uint(-INFINITY);
                }
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                top[0] = max3(top[0], __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
                top[1] = max3(top[1], __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
                top[2] = max3(top[2], __uint_as_float(y[e]), __uint_as_float(y[e + 1]));
                top[3] = max3(top[3], __uint_as_float(y[e + 2]), __uint_as_float(y[e + 3]));
            }
            const float peak = fmaxf(max3(top[0], top[1], top[2]), top[3]) * a.scale_log2;
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
#pragma unroll
                for (int c = 0; c < 4; ++c) l[c] *= f;
                m = next;
            }
            const float base = m == -INFINITY ? 0.f : m;
            const unsigned long long scale2 = pack_f32x2(a.scale_log2, a.scale_log2), base2 = pack_f32x2(-base, -base);
            // 32 weights of x or y into columns [16 c, 16 c + 16) of the block
            uint32_t px[16], py[16];
            const auto emit = [&](const uint32_t (&v)[32], int c, uint32_t (&p)[16]) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float2 z = unpack_f32x2(fma_f32x2(
                        pack_f32x2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), scale2, base2));
                    p[e] = pack_half2(ex2_approx(z.x), ex2_approx(z.y));
                }
                tc::st_32x32b_x16(block + 16 * c, p);
            };
            emit(x, 0, px);
            emit(y, 1, py);
            tc::wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(p_full + 2 * t + (i & 1)));
            // the denominator, of the weights as the product has them, while that runs
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                add_halves(l[0], l[1], px[e]);
                add_halves(l[2], l[3], py[e]);
            }
            if (LIVE) other = other || id != planned;
        }
        if (LIVE) {
            if (other) moved[t * S::M + first_row] = 1;
            named_barrier_sync(1 + t, S::M);
        }
        if (!ok && lane == 0) fail_wait();
        // ------------------------------------------------------------ the row's part
        if (n > 0 && ok) {
            // (its own barrier: by now o_done may be more than one phase past what a parity can tell)
            ok = warp_wait(o_last + t, 0);
            if (!ok && lane == 0) fail_wait();
        }
        tc::fence_after_sync();
        const bool on = n > 0 && ok && member < it.members;
        if (n > 0) {
            // partials lie [D / 8][rows][8]: a row's reads take whole sectors, as do a thread's stores
            float *dst = a.part_o + (int64_t(st.slot) * D * S::M + r * 8);
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                tc::ld_32x32b_x16(to + c, o);
                tc::wait_ld();
                if (on) {
                    store_sector(dst + c / 8 * (S::M * 8), o);
                    store_sector(dst + (c / 8 + 1) * (S::M * 8), o + 8);
                }
            }
            const bool usable = !LIVE || !moved[t * S::M + first_row];
            if (on) a.part_ml[int64_t(st.slot) * S::M + r] = make_float2(m, usable ? (l[0] + l[2]) + (l[1] + l[3]) : kPieceMoved);
        }
        tc::fence_before_sync();
    }
    __syncthreads();
    tc::fence_after_sync();
    if (warp == S::W_MMA) tc::dealloc(tmem, S::TMEM_COLS);
}

}  // namespace pd
