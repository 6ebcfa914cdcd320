// pd_prefix_args.cuh — what the shared-prefix kernels are given.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace pd {

struct PrefixArgs {
    const void *q;              // [B, Hq, D]
    const void *k, *v;          // [P, T, Hkv, D]
    const int4 *items;          // 2 per work item: {first member, members, KV head, tile},
                                // {first page in `pages`, first and end page of the piece, slot}
    const int4 *seqs;           // per sequence: {member index or -1, first slot, tiles, pieces} of its group
    const int32_t *members;     // sequences of the groups, one after another
    const int32_t *pages;       // shared pages of the groups, one after another
    const int32_t *lengths;     // [B]
    const float *rows;          // the suffix decode: FP32 [B, Hq, D] and (m, l) [B, Hq, 2]; NULL: no suffix
    const float *stats;
    float *part_o;              // [slots][tile rows][D]
    float2 *part_ml;            // [slots][tile rows]
    void *out;                  // [B, Hq, D]
    uint32_t *error;
    int32_t B, Hq, Hkv, group, page_size, tile_rows;
    int64_t P;
    float scale_log2;           // log2(e) / sqrt(D)
};

}  // namespace pd
