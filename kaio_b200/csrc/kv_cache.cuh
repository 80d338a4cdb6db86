// The paged 8-bit key/value cache: its layout and the lookups its kernels share.
//
//   k, v     s8  [num_pages][kv_heads][page_size][head_dim]
//   ks, vs   f32 [num_pages][kv_heads][page_size / 16]   one scale per 16 tokens and head
//   table    s32 [batch][max_pages]: token j of sequence b is slot j % page_size of page table[b][j / page_size]
//
// A value is s8 * max(scale, KV_SCALE_MIN).  What the device reads out of table, q_start and kv_len is checked here
// before it becomes an address: a page, a row or a position outside its buffer is reported in the status block and
// the access left out.
#pragma once

#include "common.cuh"
#include "kernels.h"
#include "kv_index.cuh"

namespace kaio {

// The smallest scale.  Without a floor an all-zero block would have to keep a scale of zero (the attention kernels
// divide by the values' scale) or of one (which later tokens of the block would inherit).
constexpr float KV_SCALE_MIN = 0x1p-40f;
// What an infinity is held as: above every finite rotated f16 pair (65504 * sqrt(2)).
constexpr float KV_LARGEST = 131008.0f;

// The attention kernels hold P = 2^(x - ref) as f16, with a reference this far (a power of two) below the largest x that it was
// taken from.  The largest P is then 2^7 at least, and one that is 2^21 smaller still has all of f16's bits (2^14 with the
// maximum itself: behind a first key with nearly all the weight, 15 above the others in the natural exponent, their
// P were rounded to subnormal steps and outputs off by 1e-2 of their value).
constexpr float KV_P_TOP = 7.0f;

struct KvCache {
    int8_t *k, *v;
    float *ks, *vs;
    const int32_t* table;
    uint32_t kv_heads, head_dim, page_size, page_shift, num_pages, max_pages, batch;
    uint32_t* status;
};

// Programmatic dependent launch: a kernel of the cache is set up while the one in front of it still runs, whatever that is.
// kv_begin() waits until the one in front is done: nothing that it may have written is read, and nothing that it may read is
// written, before.  Only then it lets the next one be set up: a W4A16 call behind this one reads its weights without waiting,
// and may count on what was in front of this one.  Calls one after the other, plain launches / these: one token over
// 500 10.2 / 8.2 us, of 64 sequences appended and read back 16.4 / 14.6.
__device__ __forceinline__ void kv_begin()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <class... Formal, class... Actual>
cudaError_t kv_launch(void (*kernel)(Formal...), dim3 grid, uint32_t threads, uint32_t smem, bool early, cudaStream_t stream,
                      const Actual&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = early && pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Loads that stay behind kv_begin(): the compiler may move __ldg in front of it.  Not by way of the read-only path (.nc), which
// is for memory that nothing writes during the kernel: the one in front may, while this one is set up.
__device__ __forceinline__ int32_t kv_load(const int32_t* p)
{
    return *p;
}

__device__ __forceinline__ float4 kv_load(const float4* p)
{
    float4 v;
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ void kv_report(const KvCache& c, uint32_t site, uint32_t kernel_id)
{
    report_status(c.status + STATUS_INDEX, DEV_BAD_INDEX, site, kernel_id);
}

// The page of token `pos` of sequence b; KV_NO_PAGE (reported) when there is none.
__device__ __forceinline__ uint32_t kv_page(const KvCache& c, uint32_t b, uint32_t pos, uint32_t kernel_id)
{
    const uint64_t none = (uint64_t)c.max_pages * c.batch;
    const uint64_t at = kv_table_entry(b, pos, c.page_shift, c.max_pages, c.batch);
    const uint32_t page = at < none ? kv_checked_page(kv_load(c.table + at), c.num_pages) : KV_NO_PAGE;
    if (page == KV_NO_PAGE)
        kv_report(c, KV_SITE_PAGE, kernel_id);
    return page;
}

// Cache row (of head_dim values) of token `pos` of a sequence, whose page this is, and the scale of its block.
__device__ __forceinline__ size_t kv_row(const KvCache& c, uint32_t page, uint32_t head, uint32_t pos)
{
    return (((size_t)page * c.kv_heads + head) << c.page_shift) + (pos & (c.page_size - 1));
}

__device__ __forceinline__ size_t kv_scale_row(const KvCache& c, uint32_t page, uint32_t head, uint32_t pos)
{
    return kv_row(c, page, head, pos) / KV_BLOCK;
}

// The sequence that work unit u belongs to (see kv_first_unit); its number inside the sequence in *local.  Warp-wide.
template <uint32_t SHIFT, uint32_t EXTRA>
__device__ __forceinline__ uint32_t kv_find_sequence(const int32_t* start, uint32_t batch, uint32_t scale, uint32_t u,
                                                     uint32_t* local)
{
    const uint32_t lane = threadIdx.x & 31;
    KvSearch s = {0, batch};
    while (s.n > 1) {
        const uint32_t at = lane * s.step();
        bool hit = at < s.n;
        if (hit)
            hit = kv_first_unit(kv_load(start + s.lo + at), s.lo + at, scale, SHIFT, EXTRA) <= u;
        s.narrow(__ballot_sync(0xffffffffu, hit));
    }
    *local = u - kv_first_unit(kv_load(start + s.lo), s.lo, scale, SHIFT, EXTRA);
    return s.lo;
}

inline KvCache kv_cache_of(const DeviceCtx& ctx, const KvParams& p)
{
    return {p.k, p.v, p.ks, p.vs, p.table, p.kv_heads, p.head_dim, p.page_size, (uint32_t)__builtin_ctz(p.page_size),
            p.num_pages, p.max_pages, p.batch, ctx.status};
}

// s8 x 4 -> two f16 pairs, exact: the byte with its sign bit flipped is x + 128; as the low byte of 0x6400 it is the
// f16 1024 + 128 + x, and subtracting 1152 is exact.  `lo` gets bytes 0 and 1, `hi` bytes 2 and 3.
__device__ __forceinline__ void s8x4_to_f16(uint32_t x, uint32_t& lo, uint32_t& hi)
{
    const uint32_t u = x ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 x0 = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 x1 = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x0);
    hi = *reinterpret_cast<const uint32_t*>(&x1);
}

}  // namespace kaio
