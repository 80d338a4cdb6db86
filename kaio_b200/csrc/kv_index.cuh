// What the kernels of the paged cache compute from numbers they find on the device (row starts, lengths, pages), apart
// from the kernels so that it is compiled and tested on the host too: none of it may lead outside a buffer, whatever
// the numbers are.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define KAIO_KV_FN __host__ __device__ __forceinline__
#else
#define KAIO_KV_FN inline
#endif

namespace kaio {

constexpr uint32_t KV_BLOCK = 16;  // tokens that share a scale
constexpr uint32_t KV_NO_PAGE = 0xffffffffu;
// The most that batch * max_pages * page_size * kv_heads of an attention call may be: pages may be shared, so the cache's own
// size bounds nothing, and a CTA counts the units of its share in 32 bits.
constexpr uint64_t KV_MOST_KEYS = 1ull << 43;

// Sites of DEV_BAD_INDEX (0: nothing wrong).
enum : uint32_t {
    KV_SITE_PAGE = 1,      // a page outside the cache, or a token past the table's last page
    KV_SITE_POSITION = 2,  // a token at a position outside the rotation table
    KV_SITE_LENGTH = 3,    // kv_len below the call's new tokens, negative, or past the table's last page
    KV_SITE_ROWS = 4,      // q_start / kv_start not ascending inside [0, rows]
    KV_SITE_MAX_NEW = 5,   // a sequence with more new tokens than the call's max_new
};

// Work units of a ragged batch without a prefix sum: sequence b has the units from
// floor(start[b] * scale / 2^shift) + extra * b on.  Its rows [start[b], start[b + 1]) cut into groups of 2^shift need
// ceil(rows * scale / 2^shift) of them, or one more when they begin inside a group (extra = 2), and the next
// sequence's first unit is never nearer than that.  A grid of floor(rows * scale / 2^shift) + extra * batch units
// covers every split of the rows into sequences.
KAIO_KV_FN uint32_t kv_first_unit(int32_t start, uint32_t b, uint32_t scale, uint32_t shift, uint32_t extra)
{
    return (uint32_t)(((uint64_t)(uint32_t)start * scale) >> shift) + extra * b;
}

// One step of the search for the last sequence whose first unit is <= u: 32 lanes look at the sequences lo + lane * step
// of the n that are left; bit `lane` of `hits` is set where lane * step < n and the sequence's first unit is <= u.
struct KvSearch {
    uint32_t lo, n;

    KAIO_KV_FN uint32_t step() const { return (n + 31) / 32; }
    KAIO_KV_FN void narrow(uint32_t hits)
    {
        const uint32_t s = step();
#ifdef __CUDA_ARCH__
        const uint32_t last = hits ? 31 - __clz(hits) : 0;
#else
        const uint32_t last = hits ? 31 - __builtin_clz(hits) : 0;
#endif
        lo += last * s;
        n = n - last * s < s ? n - last * s : s;
    }
};

// The slots [begin, end) of the 16-token block at position `base` that get the rows row0 + slot (modulo 2^32: the sum is a
// row of the sequence for every slot of the range).  bad: site, and then nothing is to be done.
struct KvSpan {
    uint32_t base, begin, end, row0, bad;
};

// Unit `local` of a sequence with the rows [q0, q1) of `rows`, which become its positions [kv - (q1 - q0), kv).
KAIO_KV_FN KvSpan kv_append_span(int32_t q0, int32_t q1, int32_t kv, uint32_t rows, uint32_t local)
{
    KvSpan s = {0, 0, 0, 0, 0};
    if (q0 < 0 || q1 < q0 || (uint32_t)q1 > rows) {
        s.bad = KV_SITE_ROWS;
        return s;
    }
    if (q1 == q0)
        return s;
    if (kv < q1 - q0) {
        s.bad = KV_SITE_LENGTH;
        return s;
    }
    const uint32_t first = (uint32_t)(kv - (q1 - q0));
    const uint64_t base = ((uint64_t)(first / KV_BLOCK) + local) * KV_BLOCK;
    if (base >= (uint64_t)kv)
        return s;
    s.base = (uint32_t)base;
    s.begin = first > s.base ? first - s.base : 0;
    s.end = (uint32_t)kv - s.base < KV_BLOCK ? (uint32_t)kv - s.base : KV_BLOCK;
    s.row0 = (uint32_t)q0 + s.base - first;
    return s;
}

// New tokens and cached tokens of a sequence as the attention kernels take them; new_tokens == 0: nothing is to be done for it.
struct KvSequence {
    uint32_t new_tokens, kv, bad;
};

KAIO_KV_FN KvSequence kv_sequence(int32_t q0, int32_t q1, int32_t kv, uint32_t rows, uint32_t max_new, uint32_t room)
{
    KvSequence s = {0, 0, 0};
    if (q0 < 0 || q1 < q0 || (uint32_t)q1 > rows)
        s.bad = KV_SITE_ROWS;
    else if (q1 == q0)
        return s;
    else if (kv < 0 || (uint32_t)kv > room)
        s.bad = KV_SITE_LENGTH;
    else if ((uint32_t)(q1 - q0) > max_new)
        s.bad = KV_SITE_MAX_NEW;
    if (s.bad == 0) {
        s.new_tokens = (uint32_t)(q1 - q0);
        s.kv = (uint32_t)kv;
    }
    return s;
}

// Keys that new token i of a sequence sees.
KAIO_KV_FN uint32_t kv_visible(const KvSequence& s, uint32_t i, bool causal)
{
    if (!causal)
        return s.kv;
    return s.kv + i + 1 > s.new_tokens ? s.kv + i + 1 - s.new_tokens : 0;
}

// An even cut of `units` work units over at most `workers` workers, and back: worker w has the units
// [begin(w), begin(w + 1)).  With fewer units than workers the first `units` workers have one each.
struct KvCut {
    uint64_t units;
    uint32_t workers;

    KAIO_KV_FN KvCut(uint64_t u, uint32_t w) : units(u), workers(u < w ? (uint32_t)u : w) {}
    KAIO_KV_FN uint64_t begin(uint32_t w) const { return w * units / workers; }
    KAIO_KV_FN uint32_t owner(uint64_t u) const { return (uint32_t)(((u + 1) * workers - 1) / units); }
};

// The table entry that holds token `pos` of sequence b, or max_pages * batch when there is none.
KAIO_KV_FN uint64_t kv_table_entry(uint32_t b, uint32_t pos, uint32_t page_shift, uint32_t max_pages, uint32_t batch)
{
    const uint32_t at = pos >> page_shift;
    return at < max_pages && b < batch ? (uint64_t)b * max_pages + at : (uint64_t)max_pages * batch;
}

KAIO_KV_FN uint32_t kv_checked_page(int32_t entry, uint32_t num_pages)
{
    return (uint32_t)entry < num_pages ? (uint32_t)entry : KV_NO_PAGE;
}

}  // namespace kaio
