// Attention over the paged 8-bit cache: which kernel takes a call.
#include "kernels.h"

namespace kaio {

// Up to 32 rows (new tokens x query heads of a key/value head) a sequence the few-row kernel, which reads every cached byte
// once and multiplies 16 rows at a time; above that the tile kernel, whose 128 rows it would fill to a quarter at most.
static bool few_rows(uint32_t batch, uint32_t max_new, uint32_t heads, uint32_t kv_heads)
{
    return attention_paged_decode_ok(batch, max_new, heads, kv_heads);
}

size_t attention_paged_scratch_floats(uint32_t batch, uint32_t tokens, uint32_t max_new, uint32_t heads,
                                      uint32_t kv_heads, uint32_t head_dim)
{
    return few_rows(batch, max_new, heads, kv_heads)
               ? attention_paged_decode_scratch(batch, max_new, heads, kv_heads, head_dim)
               : attention_paged_chunk_scratch(batch, tokens, heads, kv_heads, head_dim);
}

cudaError_t launch_attention_paged(const DeviceCtx& ctx, const KvParams& kp, const __half* q, __half* out,
                                   uint32_t q_stride, uint32_t max_new, bool causal, float* scratch,
                                   cudaStream_t stream, const char** variant)
{
    if (few_rows(kp.batch, max_new, kp.heads, kp.kv_heads)) {
        *variant = "attention_paged_decode";
        return launch_attention_paged_decode(ctx, kp, q, out, q_stride, max_new, causal, scratch, stream);
    }
    *variant = "attention_paged_tcgen05";
    return launch_attention_paged_chunk(ctx, kp, q, out, q_stride, max_new, causal, scratch, stream);
}

}  // namespace kaio
