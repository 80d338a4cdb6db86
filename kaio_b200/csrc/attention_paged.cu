// Attention over the paged 8-bit cache: which kernels take a call.
#include "kernels.h"

namespace kaio {

// The few-row kernel takes up to 16 rows (new tokens x query heads of a key/value head), what its MMAs have columns for.
// Measured in us, few-row / tile kernel, 64 and 16 sequences of 4000 tokens, one of 32000, one of 1000:
//   head size 128  64 query heads over 8, 16 rows  150 / 212, 51 / 59, 29 / 36, 13.1 / 15.4
//                  16 over 1, 16 rows               34 / 37, 17.0 / 17.5, 20 / 25, 12.4 / 14.1
//                  24 over 8, 9 rows               145 / 211, 48 / 60, 27 / 37, 11.8 / 16.2
//   head size 64   64 over 8, 16 rows              101 / 183, 34 / 50, 21 / 31, 10.6 / 14.3
//                  16 over 1, 16 rows               24 / 32, 13.2 / 15.8, 16 / 22, 10.3 / 13.0
//                  24 over 8, 9 rows                97 / 182, 32 / 50, 20 / 31, 9.7 / 14.9
// For 17 rows and more it would have to read the cache once for every 16: at 64 over 8, head size 128, 32 rows take the tile
// kernel as long as 16 do.
// A call that may hold both kinds of sequences (some have less than max_new new tokens) launches both kernels and each takes
// its own: one token of a sequence among prompts would otherwise walk its whole cache on one SM.
struct Cut {
    bool few, tiles;
    uint32_t most_new;  // new tokens of a sequence that is the few-row kernel's
};

static Cut cut_of(uint32_t batch, uint32_t tokens, uint32_t max_new, uint32_t heads, uint32_t kv_heads)
{
    if (attention_paged_decode_ok(max_new, heads, kv_heads))
        return {true, false, max_new};
    // in a mixed call only what its form of 8 rows takes, or one token
    const uint32_t group = heads / kv_heads, most = group <= 8 ? 8 / group : 1;
    const bool mixed = (uint64_t)batch * max_new > tokens && batch > 1 && attention_paged_decode_ok(most, heads, kv_heads);
    return {mixed, true, mixed ? most : 0};
}

static size_t up4(size_t n)
{
    return (n + 3) / 4 * 4;
}

size_t attention_paged_scratch_floats(uint32_t batch, uint32_t tokens, uint32_t max_new, uint32_t heads,
                                      uint32_t kv_heads, uint32_t head_dim)
{
    const Cut cut = cut_of(batch, tokens, max_new, heads, kv_heads);
    return (cut.few ? up4(attention_paged_decode_scratch(cut.most_new, heads, kv_heads, head_dim)) : 0) +
           (cut.tiles ? attention_paged_chunk_scratch(batch, tokens, heads, kv_heads, head_dim) : 0);
}

cudaError_t launch_attention_paged(const DeviceCtx& ctx, const KvParams& kp, const __half* q, __half* out,
                                   uint32_t q_stride, uint32_t max_new, bool causal, float* scratch,
                                   cudaStream_t stream, const char** variant)
{
    const Cut cut = cut_of(kp.batch, kp.rows, max_new, kp.heads, kp.kv_heads);
    *variant = !cut.tiles ? "attention_paged_decode" : cut.few ? "attention_paged_tcgen05_and_decode" : "attention_paged_tcgen05";
    if (cut.few) {
        const cudaError_t err = launch_attention_paged_decode(ctx, kp, q, out, q_stride, max_new, cut.most_new, causal, cut.tiles,
                                                              scratch, stream);
        if (err != cudaSuccess || !cut.tiles)
            return err;
        scratch += up4(attention_paged_decode_scratch(cut.most_new, kp.heads, kp.kv_heads, kp.head_dim));
    }
    return launch_attention_paged_chunk(ctx, kp, q, out, q_stride, max_new, cut.most_new + 1, causal, cut.few, scratch, stream);
}

}  // namespace kaio
