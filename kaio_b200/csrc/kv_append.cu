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
// Both kernels are bound by HBM at prompts and by latency at single tokens, so all loads of a warp are issued before the
// first is used, and what depends on the page comes last; steps without a new token are passed over by the whole warp.
//  * A warp has one head of q, k or v of one 16-token block.  Keys and values stay in registers as f16 between the maximum
//    and the quantisation (the rotation is made twice, which is cheaper than 64 registers of its results): a value is read
//    once and written once.
//  * Lane l of a token takes 8 dims: 4 pairs, or 8 dims beside the rotated ones.
//
// Measured at head size 128, 64 query heads over 8: three prompts of 1777, 1657 and 1558 tokens, 197 MB, appended in 47 us (4.2
// TB/s: the index arithmetic and the rotation, issue slots 55 % busy, share the blame with HBM; a warp that keeps the angles and
// takes several heads spilled or was as fast); three ragged ones of up to 1777, 161 MB, appended and read back in 51.  One token each of 64 sequences, appended and their
// caches of up to 120 tokens read back: 15 us.  Reading back eight ragged caches of up to 2000 tokens, 32 heads, 303 MB: 53 us = 5.7 TB/s, 0.87 of
// the copy rate.
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

__device__ __forceinline__ void widen4(uint2 w, float* x)
{
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
__global__ void __launch_bounds__(WARPS * 32, 3) rope_append_kernel(const KvCache c, const Params p)
{
    constexpr uint32_t LPT = D / 8;       // lanes of a token
    constexpr uint32_t TPI = 32 / LPT;    // tokens of a step
    constexpr int STEPS = KV_BLOCK / TPI;
    kv_begin();
    const uint32_t lane = threadIdx.x & 31, l = lane % LPT, tok = lane / LPT;
    // the warp's part: K of a head, V of a head, a query head
    const uint32_t slot = blockIdx.y * WARPS + (threadIdx.x >> 5);
    const bool is_q = slot >= 2 * c.kv_heads, is_v = !is_q && slot >= c.kv_heads;
    const uint32_t head = is_q ? slot - 2 * c.kv_heads : is_v ? slot - c.kv_heads : slot;
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

    const bool turns = l < p.rot_dim / 8;
    const uint32_t half = p.rot_dim / 2;
    // this lane's dims of q and k: [da, da + 4) and [db, db + 4)
    const uint32_t da = turns && !p.interleaved ? 4 * l : 8 * l;
    const uint32_t db = turns && !p.interleaved ? half + 4 * l : 8 * l + 4;
    // whether step i has new tokens, which slot this lane reads in it (its own, or another new token's), and whether its own
    // is new
    auto live = [&](int i) { return (i + 1) * TPI > begin && i * TPI < end; };
    auto place = [&](int i) {
        const uint32_t s = i * TPI + tok;
        return s < begin ? begin : s < end ? s : end - 1;
    };
    auto mine = [&](int i) {
        const uint32_t s = i * TPI + tok;
        return s >= begin && s < end;
    };
    auto load_angles = [&](int i, float4& cs, float4& sn) {
        if (live(i) && turns) {
            const size_t at = (size_t)(base + place(i)) * half + 4 * l;
            cs = kv_load(reinterpret_cast<const float4*>(p.cos + at));
            sn = kv_load(reinterpret_cast<const float4*>(p.sin + at));
        }
    };
    auto turn = [&](float (&x)[8], const float4& cs, const float4& sn) {
        if (turns) {
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

    // the lane's values are at the dims [a, a + 4) and [bb, bb + 4)
    const uint32_t a = is_v ? 8 * l : da, bb = is_v ? 8 * l + 4 : db;
    const __half* from = (is_q ? p.q : is_v ? p.v : p.k) + (size_t)head * D;
    const uint32_t stride = is_q ? p.q_stride : p.kv_stride;
    uint2 wa[STEPS], wb[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
        if (live(i)) {
            const __half* row = from + (size_t)(row0 + place(i)) * stride;
            wa[i] = *reinterpret_cast<const uint2*>(row + a);
            wb[i] = *reinterpret_cast<const uint2*>(row + bb);
        }
    // step i's values, rotated
    auto values = [&](int i, float (&x)[8]) {
        float4 cs, sn;
        if (!is_v)
            load_angles(i, cs, sn);
        widen4(wa[i], x);
        widen4(wb[i], x + 4);
        if (!is_v)
            turn(x, cs, sn);
    };

    if (is_q) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
            if (live(i)) {
                float x[8];
                values(i, x);
                if (mine(i)) {
                    __half* out = p.q_out + ((size_t)(row0 + i * TPI + tok) * p.heads + head) * D;
                    store4(out + da, x);
                    store4(out + db, x + 4);
                }
            }
        return;
    }

    const uint32_t page = kv_page(c, b, base, KERNEL_KV_APPEND);
    if (page == KV_NO_PAGE)
        return;
    int8_t* cache = (is_v ? c.v : c.k) + kv_row(c, page, head, base) * D;
    float* scale = (is_v ? c.vs : c.ks) + kv_scale_row(c, page, head, base);
    const float s_old = begin > 0 ? *scale : 0.0f;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
        if (live(i)) {
            float x[8];
            values(i, x);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                top = fmaxf(top, fabsf(x[e]));  // a NaN is passed over
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float s = fmaxf(fmaxf(__fdiv_rn(fminf(top, KV_LARGEST), 127.0f), s_old), KV_SCALE_MIN);
    const float inv = __fdiv_rn(1.0f, s);
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
        if (live(i)) {
            float x[8];
            values(i, x);
            if (mine(i)) {
                int8_t* to = cache + (size_t)(i * TPI + tok) * D;
                if (bb == a + 4) {
                    *reinterpret_cast<uint2*>(to + a) = make_uint2(quant4(x, inv), quant4(x + 4, inv));
                } else {
                    *reinterpret_cast<uint32_t*>(to + a) = quant4(x, inv);
                    *reinterpret_cast<uint32_t*>(to + bb) = quant4(x + 4, inv);
                }
            }
        }
    if (begin > 0 && s > s_old) {
        const float ratio = __fdiv_rn(s_old, s);
        uint2 old[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
            if (i * TPI < begin && i * TPI + tok < begin)
                old[i] = *reinterpret_cast<const uint2*>(cache + (size_t)(i * TPI + tok) * D + 8 * l);
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
            if (i * TPI < begin && i * TPI + tok < begin)
                *reinterpret_cast<uint2*>(cache + (size_t)(i * TPI + tok) * D + 8 * l) =
                    make_uint2(rescale4(old[i].x, ratio), rescale4(old[i].y, ratio));
    }
    __syncwarp();  // every lane has read the old scale
    if (lane == 0)
        *scale = s;
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
    constexpr uint32_t LPT = D / 8, TPI = 32 / LPT;  // 8 dims a lane: 16 bytes out, so that every store fills its sectors
    constexpr int STEPS = KV_BLOCK / TPI;
    kv_begin();
    const uint32_t lane = threadIdx.x & 31, l = lane % LPT, tok = lane / LPT;
    const uint32_t head = blockIdx.y * WARPS + (threadIdx.x >> 5);
    if (head >= c.kv_heads)
        return;
    uint32_t local;
    const uint32_t b = kv_find_sequence<4, 1>(p.kv_start, p.batch, 1, blockIdx.x, &local);
    const int32_t r0 = p.kv_start[b], r1 = p.kv_start[b + 1];
    // the rows are the positions from 0 on
    const KvSpan span = kv_append_span(r0, r1, (int32_t)((uint32_t)r1 - (uint32_t)r0), p.total, local);
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
    uint2 w[2][STEPS];  // slots behind the last token are in the page too
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const size_t at = (row + i * TPI + tok) * D + 8 * l;
        w[0][i] = __ldcs(reinterpret_cast<const uint2*>(c.k + at));
        w[1][i] = __ldcs(reinterpret_cast<const uint2*>(c.v + at));
    }
    const float s[2] = {fmaxf(c.ks[srow], KV_SCALE_MIN), fmaxf(c.vs[srow], KV_SCALE_MIN)};
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const uint32_t t = i * TPI + tok;
            uint32_t h[4], out[4];
            s8x4_to_f16(w[which][i].x, h[0], h[1]);
            s8x4_to_f16(w[which][i].y, h[2], h[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
                const __half2 y = __floats2half2_rn(f.x * s[which], f.y * s[which]);
                out[e] = *reinterpret_cast<const uint32_t*>(&y);
            }
            if (t < span.end)
                __stcs(reinterpret_cast<uint4*>((which ? p.v_out : p.k_out) + ((size_t)(span.row0 + t) * c.kv_heads + head) * D + 8 * l),
                       make_uint4(out[0], out[1], out[2], out[3]));
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
    const dim3 grid(kp.rows / KV_BLOCK + 2 * kp.batch, (p.heads + 2 * kp.kv_heads + WARPS - 1) / WARPS);
    return kv_launch(kp.head_dim == 128 ? rope_append_kernel<128> : rope_append_kernel<64>, grid, WARPS * 32, 0, true, stream, c, p);
}

cudaError_t launch_gather_kv(const DeviceCtx& ctx, const KvParams& kp, __half* k_out, __half* v_out, cudaStream_t stream)
{
    using namespace kvapp;
    const KvCache c = kv_cache_of(ctx, kp);
    const GatherParams p = {kp.start, k_out, v_out, kp.batch, kp.rows};
    const dim3 grid(kp.rows / KV_BLOCK + kp.batch, (kp.kv_heads + WARPS - 1) / WARPS);
    return kv_launch(kp.head_dim == 128 ? gather_kernel<128> : gather_kernel<64>, grid, WARPS * 32, 0, true, stream, c, p);
}

}  // namespace kaio
