// Attention over the paged 8-bit cache: one warp per (new token, query head), 32 keys at a time with an online softmax.
#include "kernels.h"
#include "kv_cache.cuh"

namespace kaio {
namespace apaged {

constexpr int WARPS = 4;

struct Params {
    const __half* q;
    __half* out;
    const int32_t *q_start, *kv_len;
    uint32_t batch, tokens, heads, q_stride, max_new;
    float scale;
    int causal;
};

template <int D>
__global__ void __launch_bounds__(WARPS * 32) attention_paged_kernel(const KvCache c, const Params p)
{
    constexpr int VPL = D / 32;  // value dims per lane
    __shared__ float qs[WARPS][D];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t head = blockIdx.y * WARPS + warp;
    if (head >= p.heads)
        return;
    const uint32_t kvh = head / (p.heads / c.kv_heads);
    uint32_t local;
    const uint32_t b = kv_find_sequence<0, 0>(p.q_start, p.batch, 1, blockIdx.x, &local);
    const int32_t q0 = p.q_start[b];
    const KvSequence s = kv_sequence(q0, p.q_start[b + 1], p.kv_len[b], p.tokens, p.max_new, c.max_pages * c.page_size);
    if (s.bad)
        kv_report(c, s.bad, KERNEL_ATTN_PAGED);
    const uint32_t row = blockIdx.x;
    if (row - (uint32_t)q0 >= s.new_tokens)
        return;
    const uint32_t seen = kv_visible(s, row - (uint32_t)q0, p.causal != 0);
    for (int i = lane; i < D; i += 32)
        qs[warp][i] = __half2float(p.q[(size_t)row * p.q_stride + (size_t)head * D + i]) * p.scale;
    __syncwarp();
    float m = -INFINITY, sum = 0.0f, acc[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i)
        acc[i] = 0.0f;
    for (uint32_t key0 = 0; key0 < seen; key0 += 32) {
        const uint32_t key = key0 + lane;
        uint32_t page = KV_NO_PAGE;
        if (key < seen)
            page = kv_page(c, b, key, KERNEL_ATTN_PAGED);
        float x = -INFINITY, vs = 0.0f;
        size_t vrow = 0;
        if (page != KV_NO_PAGE) {
            const size_t at = kv_row(c, page, kvh, key);
            const size_t sat = kv_scale_row(c, page, kvh, key);
            float dot = 0.0f;
            for (int i = 0; i < D; ++i)
                dot = fmaf(qs[warp][i], (float)c.k[at * D + i], dot);
            x = dot * fmaxf(c.ks[sat], KV_SCALE_MIN);
            vs = fmaxf(c.vs[sat], KV_SCALE_MIN);
            vrow = at;
        }
        float top = x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m, top);
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = exp2f(m - ref), pr = exp2f(x - ref);
        m = m_new;
        sum = sum * alpha + pr;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            acc[i] *= alpha;
        for (int j = 0; j < 32; ++j) {
            const float w = __shfl_sync(0xffffffffu, pr * vs, j);
            const size_t at = __shfl_sync(0xffffffffu, vrow, j);
#pragma unroll
            for (int i = 0; i < VPL; ++i)
                acc[i] = fmaf(w, (float)c.v[at * D + lane + 32 * i], acc[i]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
        p.out[((size_t)row * p.heads + head) * D + lane + 32 * i] = __float2half_rn(acc[i] * inv);
}

}  // namespace apaged

size_t attention_paged_scratch_floats(uint32_t batch, uint32_t tokens, uint32_t max_new, uint32_t heads,
                                      uint32_t kv_heads, uint32_t head_dim)
{
    (void)tokens;
    return attention_paged_decode_ok(batch, max_new, heads, kv_heads)
               ? attention_paged_decode_scratch(batch, max_new, heads, kv_heads, head_dim)
               : 0;
}

cudaError_t launch_attention_paged(const DeviceCtx& ctx, const KvParams& kp, const __half* q, __half* out,
                                   uint32_t q_stride, uint32_t max_new, bool causal, float* scratch,
                                   cudaStream_t stream, const char** variant)
{
    if (attention_paged_decode_ok(kp.batch, max_new, kp.heads, kp.kv_heads)) {
        *variant = "attention_paged_decode";
        return launch_attention_paged_decode(ctx, kp, q, out, q_stride, max_new, causal, scratch, stream);
    }
    using namespace apaged;
    const KvCache c = kv_cache_of(ctx, kp);
    const Params p = {q, out, kp.start, kp.kv_len, kp.batch, kp.rows, kp.heads, q_stride, max_new,
                      1.4426950408889634f / sqrtf((float)kp.head_dim), causal ? 1 : 0};
    const dim3 grid(kp.rows, (kp.heads + WARPS - 1) / WARPS);
    *variant = "attention_paged_warp";
    if (kp.head_dim == 128)
        attention_paged_kernel<128><<<grid, WARPS * 32, 0, stream>>>(c, p);
    else
        attention_paged_kernel<64><<<grid, WARPS * 32, 0, stream>>>(c, p);
    return cudaGetLastError();
}

}  // namespace kaio
