// Appending keys and values to the paged 8-bit cache, with the position rotation applied on the way, and reading the
// cache back.
//
// rope_append_kv: token t of the call is token pos = kv_len[b] - new[b] + (t - q_start[b]) of its sequence b.
//   rotation  y0 = x0 c - x1 s, y1 = x1 c + x0 s over the first rot_dim dims, c and s from row pos of f32 tables, in f32
//             with every product and sum rounded (no fused multiply-add), so the same bits come out of any plain f32 code
//   q         rotated and rounded to f16 once
//   k, v      quantised per block of 16 tokens and head: s = max(max |y| / 127, the block's stored scale unless the call
//             writes the block from its first slot, 2^-40); tokens that were in the block already move to the larger
//             scale, q = rint(q * (s_old / s)); new ones are q = rint(y * (1 / s)) in [-127, 127]
//   An infinity counts as +-131008 (twice the largest f16), a NaN as 0: one bad value costs its block precision and
//   reaches no other.
//
// A warp has one head of one 16-token block, as f32 in registers between the maximum and the quantisation, so a value
// is read once and written once.  Lane l of a token takes 8 dims: 4 pairs, or 8 dims beside the rotated ones.
#include "kernels.h"
#include "kv_cache.cuh"

namespace kaio {
namespace kvapp {

constexpr int WARPS = 8;

struct Params {
    const __half *q, *k, *v;
    const float *cos, *sin;
    __half* q_out;
    const int32_t *q_start, *kv_len;
    uint32_t batch, tokens, heads, q_stride, kv_stride, rot_dim, max_pos;
    int interleaved;
};

__device__ __forceinline__ void load4(const __half* p, float* x)
{
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    x[0] = a.x;
    x[1] = a.y;
    x[2] = b.x;
    x[3] = b.y;
}

__device__ __forceinline__ void store4(__half* p, const float* x)
{
    const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
    uint2 w;
    w.x = *reinterpret_cast<const uint32_t*>(&a);
    w.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(p) = w;
}

__device__ __forceinline__ void rotate(float& x0, float& x1, float c, float s)
{
    const float y0 = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
    x1 = __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, s));
    x0 = y0;
}

// clamp(rint(x), -127, 127), NaN -> 0 (the conversion's result for it)
__device__ __forceinline__ uint32_t quant(float x)
{
    return (uint32_t)max(-127, min(127, __float2int_rn(x))) & 0xffu;
}

__device__ __forceinline__ uint32_t quant4(const float* x, float f)
{
    return quant(__fmul_rn(x[0], f)) | quant(__fmul_rn(x[1], f)) << 8 | quant(__fmul_rn(x[2], f)) << 16 |
           quant(__fmul_rn(x[3], f)) << 24;
}

__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f)
{
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x[i] = (float)(int8_t)(w >> (8 * i));
    return quant4(x, f);
}

template <int D>
__global__ void __launch_bounds__(WARPS * 32) rope_append_kernel(const KvCache c, const Params p)
{
    constexpr uint32_t LPT = D / 8;       // lanes of a token
    constexpr uint32_t TPI = 32 / LPT;    // tokens of a step
    constexpr int STEPS = KV_BLOCK / TPI;
    const uint32_t lane = threadIdx.x & 31, l = lane % LPT, tok = lane / LPT;
    uint32_t slot = blockIdx.y * WARPS + (threadIdx.x >> 5);  // a key/value head, then a query head
    const bool is_q = slot >= c.kv_heads;
    const uint32_t head = is_q ? slot - c.kv_heads : slot;
    if (is_q && head >= p.heads)
        return;

    uint32_t local;
    const uint32_t b = kv_find_sequence<4, 2>(p.q_start, p.batch, 1, blockIdx.x, &local);
    const KvSpan span = kv_append_span(p.q_start[b], p.q_start[b + 1], p.kv_len[b], p.tokens, local);
    const uint32_t base = span.base, begin = span.begin, end = span.end, row0 = span.row0;
    if (span.bad || end == 0) {
        if (span.bad)
            kv_report(c, span.bad, KERNEL_KV_APPEND);
        return;
    }
    if (p.rot_dim && base + end > p.max_pos) {
        kv_report(c, KV_SITE_POSITION, KERNEL_KV_APPEND);
        return;
    }

    const uint32_t rot_lanes = p.rot_dim / 8;
    const bool turns = l < rot_lanes;
    // this lane's dims: [da, da + 4) and [db, db + 4)
    const uint32_t da = turns && !p.interleaved ? 4 * l : 8 * l;
    const uint32_t db = turns && !p.interleaved ? p.rot_dim / 2 + 4 * l : 8 * l + 4;
    const uint32_t half = p.rot_dim / 2;

    auto load_rotated = [&](const __half* row, uint32_t pos, float (&x)[8]) {
        load4(row + da, x);
        load4(row + db, x + 4);
        if (turns) {
            const float4 cs = *reinterpret_cast<const float4*>(p.cos + (size_t)pos * half + 4 * l);
            const float4 sn = *reinterpret_cast<const float4*>(p.sin + (size_t)pos * half + 4 * l);
            if (p.interleaved) {
                rotate(x[0], x[1], cs.x, sn.x);
                rotate(x[2], x[3], cs.y, sn.y);
                rotate(x[4], x[5], cs.z, sn.z);
                rotate(x[6], x[7], cs.w, sn.w);
            } else {
                rotate(x[0], x[4], cs.x, sn.x);
                rotate(x[1], x[5], cs.y, sn.y);
                rotate(x[2], x[6], cs.z, sn.z);
                rotate(x[3], x[7], cs.w, sn.w);
            }
        }
    };

    if (is_q) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const uint32_t s = i * TPI + tok;
            if (s >= begin && s < end) {
                float x[8];
                load_rotated(p.q + (size_t)(row0 + s) * p.q_stride + (size_t)head * D, base + s, x);
                __half* out = p.q_out + ((size_t)(row0 + s) * p.heads + head) * D;
                store4(out + da, x);
                store4(out + db, x + 4);
            }
        }
        return;
    }

    const uint32_t page = kv_page(c, b, base, KERNEL_KV_APPEND);
    if (page == KV_NO_PAGE)
        return;
    const size_t row = kv_row(c, page, head, base);
    const size_t srow = kv_scale_row(c, page, head, base);
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        int8_t* cache = (which ? c.v : c.k) + row * D;
        float* scale = (which ? c.vs : c.ks) + srow;
        const float s_old = begin > 0 ? *scale : 0.0f;
        const uint32_t a = which ? 8 * l : da, bb = which ? 8 * l + 4 : db;
        float x[STEPS][8];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const uint32_t s = i * TPI + tok;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[i][e] = 0.0f;
            if (s >= begin && s < end) {
                const size_t at = (size_t)(row0 + s) * p.kv_stride + (size_t)head * D;
                if (which) {
                    load4(p.v + at + a, x[i]);
                    load4(p.v + at + bb, x[i] + 4);
                } else {
                    load_rotated(p.k + at, base + s, x[i]);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                top = fmaxf(top, fabsf(x[i][e]));  // a NaN is passed over
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float s = fmaxf(fmaxf(__fdiv_rn(fminf(top, KV_LARGEST), 127.0f), s_old), KV_SCALE_MIN);
        const float inv = __fdiv_rn(1.0f, s);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const uint32_t t = i * TPI + tok;
            if (t >= begin && t < end) {
                *reinterpret_cast<uint32_t*>(cache + (size_t)t * D + a) = quant4(x[i], inv);
                *reinterpret_cast<uint32_t*>(cache + (size_t)t * D + bb) = quant4(x[i] + 4, inv);
            }
        }
        if (begin > 0 && s > s_old) {
            const float ratio = __fdiv_rn(s_old, s);
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const uint32_t t = i * TPI + tok;
                if (t < begin) {
                    uint2* w = reinterpret_cast<uint2*>(cache + (size_t)t * D + 8 * l);
                    const uint2 old = *w;
                    *w = make_uint2(rescale4(old.x, ratio), rescale4(old.y, ratio));
                }
            }
        }
        __syncwarp();  // every lane has read the old scale
        if (lane == 0)
            *scale = s;
    }
}

struct GatherParams {
    const int32_t* kv_start;
    __half *k_out, *v_out;
    uint32_t batch, total;
};

// out[kv_start[b] + j] = f16(s8 * scale): a warp has one head of one 16-token block.
template <int D>
__global__ void __launch_bounds__(WARPS * 32) gather_kernel(const KvCache c, const GatherParams p)
{
    constexpr uint32_t LPT = D / 8, TPI = 32 / LPT;
    constexpr int STEPS = KV_BLOCK / TPI;
    const uint32_t lane = threadIdx.x & 31, l = lane % LPT, tok = lane / LPT;
    const uint32_t head = blockIdx.y * WARPS + (threadIdx.x >> 5);
    if (head >= c.kv_heads)
        return;
    uint32_t local;
    const uint32_t b = kv_find_sequence<4, 1>(p.kv_start, p.batch, 1, blockIdx.x, &local);
    const int32_t r0 = p.kv_start[b], r1 = p.kv_start[b + 1];
    const KvSpan span = kv_append_span(r0, r1, (int32_t)((uint32_t)r1 - (uint32_t)r0), p.total, local);  // the rows are the positions from 0 on
    const uint32_t base = span.base;
    if (span.bad || span.end == 0) {
        if (span.bad)
            kv_report(c, span.bad, KERNEL_KV_GATHER);
        return;
    }
    const uint32_t page = kv_page(c, b, base, KERNEL_KV_GATHER);
    if (page == KV_NO_PAGE)
        return;
    const size_t row = kv_row(c, page, head, base);
    const size_t srow = kv_scale_row(c, page, head, base);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int8_t* cache = (which ? c.v : c.k) + row * D;
        const float s = fmaxf((which ? c.vs : c.ks)[srow], KV_SCALE_MIN);
        __half* out = which ? p.v_out : p.k_out;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const uint32_t t = i * TPI + tok;
            if (t < span.end) {
                const uint2 w = *reinterpret_cast<const uint2*>(cache + (size_t)t * D + 8 * l);
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[e] = s * (float)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
                __half* o = out + ((size_t)(span.row0 + t) * c.kv_heads + head) * D + 8 * l;
                store4(o, x);
                store4(o + 4, x + 4);
            }
        }
    }
}

}  // namespace kvapp

cudaError_t launch_rope_append_kv(const DeviceCtx& ctx, const KvParams& kp, const __half* q, const __half* k,
                                  const __half* v, const float* cos, const float* sin, __half* q_out,
                                  uint32_t q_stride, uint32_t kv_stride, uint32_t rot_dim, bool interleaved,
                                  uint32_t max_pos, cudaStream_t stream)
{
    using namespace kvapp;
    const KvCache c = kv_cache_of(ctx, kp);
    Params p = {};
    p.q = q;
    p.k = k;
    p.v = v;
    p.cos = cos;
    p.sin = sin;
    p.q_out = q_out;
    p.q_start = kp.start;
    p.kv_len = kp.kv_len;
    p.batch = kp.batch;
    p.tokens = kp.rows;
    p.heads = q ? kp.heads : 0;
    p.q_stride = q_stride;
    p.kv_stride = kv_stride;
    p.rot_dim = rot_dim;
    p.max_pos = max_pos;
    p.interleaved = interleaved ? 1 : 0;
    const dim3 grid(kp.rows / KV_BLOCK + 2 * kp.batch, (p.heads + kp.kv_heads + WARPS - 1) / WARPS);
    if (kp.head_dim == 128)
        rope_append_kernel<128><<<grid, WARPS * 32, 0, stream>>>(c, p);
    else
        rope_append_kernel<64><<<grid, WARPS * 32, 0, stream>>>(c, p);
    return cudaGetLastError();
}

cudaError_t launch_gather_kv(const DeviceCtx& ctx, const KvParams& kp, __half* k_out, __half* v_out, cudaStream_t stream)
{
    using namespace kvapp;
    const KvCache c = kv_cache_of(ctx, kp);
    const GatherParams p = {kp.start, k_out, v_out, kp.batch, kp.rows};
    const dim3 grid(kp.rows / KV_BLOCK + kp.batch, (kp.kv_heads + WARPS - 1) / WARPS);
    if (kp.head_dim == 128)
        gather_kernel<128><<<grid, WARPS * 32, 0, stream>>>(c, p);
    else
        gather_kernel<64><<<grid, WARPS * 32, 0, stream>>>(c, p);
    return cudaGetLastError();
}

}  // namespace kaio
