// attn.cuh — what the two attention kernels share (attn_stream.cu, attn_tile.cu).
#pragma once

#include "kv.cuh"

namespace tq {

struct AttnArgs {
    KvArgs kv;
    const uint16_t *q;
    void *out;
    size_t ldo;
    int q_heads, group;          // group = q_heads / kv heads
    float c;                     // scale * log2(e) (times k_scale)
    int out_bf16;
    float *part;                 // partial tiles, two per CTA
    int *arrived;                // per CTA: parts of the tile that starts in it
    unsigned long long limit_ns; // of a wait (attn_tile.cu)
    int rows, box;               // TMA copies (attn_tile.cu): rows of a pool, of a copy
};

// attn_tile.cu: tiles of 128 query rows on tcgen05
void launch_attn_tile(const AttnArgs &a, bool e4m3, int sms);
size_t attn_tile_part_floats(int sms);       // of a.part

}  // namespace tq
