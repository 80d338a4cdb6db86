// Attention of a few new tokens per sequence over the paged 8-bit cache (decode steps, drafted tokens): up to 16 rows
// (new tokens x query heads of a key/value head) per (sequence, key/value head).
//
// out = O / l with  x_j = (q . kint_j) ks_j log2(e) / sqrt(d) + log2(vs_j),  P_j = 2^(x_j - ref),
//                   O = sum_j P_j vint_j,  l = sum_j P_j / vs_j.
// ks and vs are constant over 16 keys, so neither scale costs work per cached value, the 8-bit integers are exact as f16
// operands, and P (rounded to f16 for the product, f32 in l) is largest where it weighs most, whatever the scales are.
//
// What bounds it: HBM, every cached byte is read once.  Per byte an SM has 5.6 issue slots of a lane, so what is done per
// byte decides, and the products are warp-level MMAs (16 rows; tcgen05's 128 would be padding).
//  * Both products with the cached side as the 16-row operand and the rows of q as the 8 columns (two column tiles for 9 to
//    16 rows): S^T = K Q^T, O^T = V^T P^T.  P^T is turned from one to the other by movmatrix.
//  * S^T on the integer tensor cores: q is cut into three signed digits of 7 bits, q = sq (2^14 h + 2^7 m + l), exact to
//    2^-22 of the row's largest value, and K is an operand as it lies in shared memory.  (Converting K to f16 took 5
//    instructions for 4 values, a sixth of all.)
//  * O^T in f16: two keys of a dim make one operand word, 1.5 instructions a value, shared by all rows.
//  * A unit is 128 keys of one (sequence, head), 32 for each of four warps; a fifth warp fetches K and V by TMA, 16 rows a
//    box, into a ring of three tiles.  The boxes' swizzle keeps the row-wise reads of K and the column-wise ones of V free
//    of bank conflicts.  (With a ring a warp, loaded by itself, the bookkeeping was half of all instructions.)
//  * All units of the call are cut evenly over the CTAs, whatever the lengths of the sequences: a long sequence is spread
//    over the GPU, short ones are put together.  A CTA that holds a part of a (sequence, head) leaves (O, ref, l) in
//    scratch; a second launch, resident before the first ends, adds the parts in ascending order.
//
// Measured (both launches, caches from HBM, head size 128): 64 ragged sequences of up to 7000 tokens, 64 query heads over 8,
// 500 MB in 101 us = 5.0 TB/s, 0.76 of the copy rate (the first launch alone 5.4 to 5.9); eight of 2000 tokens, 32 heads, 131 MB
// in 31 us; one of 100001 tokens, 64 heads over 8, 205 MB in 45 us; one of 500 tokens 8 us, nearly all of it the two
// launches.  ptxas spills 196 bytes a thread in the form of 9 to 16 rows at head size 128 (168 registers, two CTAs an SM), and none in
// the other three; what that costs has not been measured.
#include "kernels.h"
#include "kv_cache.cuh"
#include "mma_sync.cuh"

namespace kaio {
namespace apdec {

constexpr int WARPS = 4;             // that compute; one more loads
constexpr int THREADS = (WARPS + 1) * 32;
constexpr uint32_t MAX_SMS = 160;
constexpr uint32_t MAX_WORKERS = MAX_SMS * 3;
constexpr uint32_t UNIT = 32 * WARPS;  // keys of a unit
constexpr uint32_t BLOCKS = UNIT / KV_BLOCK;
constexpr uint32_t ROWS = 16;        // the most rows
constexpr uint32_t MAX_GROUPS = 1024;  // groups of 32 sequences
constexpr float WINDOW = 15.0f;      // P may grow to 2^15 before O and l are rescaled

constexpr uint32_t NO_PAIR = 0xffffffffu;

enum : uint32_t { SITE_FULL = 1, SITE_EMPTY = 2 };

struct Params {
    const __half* q;
    __half* out;
    const int32_t *q_start, *kv_len;
    float *part_o, *part_ml;  // [2 * workers][rows][D], [2 * workers][rows][2]
    uint2* meta;              // [workers]: the pair whose first part is the worker's last one, and its last worker
    uint32_t tokens, heads, group, q_stride, max_new, room;
    uint32_t most_new;  // sequences with more new tokens are another kernel's,
    int follows;        // which follows in the same call and needs nothing of this one's
    uint32_t part_rows;
    float scale_log2;
    int causal;
};

// A tile is K or V of a unit; the ring takes them in turn.  NB column tiles of 8 rows.
template <int D, int NB>
struct Shape {
    static constexpr int CTAS = NB == 1 ? 3 : 2;              // an SM: by registers, 128 a thread and 168
    static constexpr uint32_t BLOCK_BYTES = 16 * D;           // 16 keys of K or V
    static constexpr uint32_t TILE_BYTES = BLOCKS * BLOCK_BYTES;
    static constexpr uint32_t TILES = (NB == 1 ? 3 : 4) * (128 / D);
    static constexpr uint32_t MERGE_FLOATS = NB * (D / 4 + 4) * 32;  // O, ref and l of a warp
    static constexpr uint32_t SMEM = 1024 + TILES * TILE_BYTES + 2 * MERGE_FLOATS * 4;
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void imma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void imma_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                           uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// The 8 x 8 transpose of 16-bit values: lane (g, t) holds the row g, columns 2t and 2t + 1.
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// The three digits of four values x (scaled to [-127 * 2^14, 127 * 2^14]), packed a digit a word.
__device__ __forceinline__ void digits(const float (&x)[4], uint32_t (&w)[3])
{
    w[0] = w[1] = w[2] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int v = __float2int_rn(x[i]);
        const int h = (v + 8192) >> 14, r = v - (h << 14);  // r in [-8192, 8191]
        const int m = (r + 64) >> 7, l = r - (m << 7);      // m in [-64, 64], l in [-64, 63]
        w[0] |= (uint32_t)(h & 0xff) << (8 * i);
        w[1] |= (uint32_t)(m & 0xff) << (8 * i);
        w[2] |= (uint32_t)(l & 0xff) << (8 * i);
    }
}

__device__ __forceinline__ uint4 lds128(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

__device__ __forceinline__ uint2 lds64(uint32_t addr)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}

// Where a walk over the units stands: unit `un` of (sequence b, head).
struct Cursor {
    uint32_t b, head, un, units;
    KvSequence s;
    int32_t q0;
};

__device__ __forceinline__ uint32_t units_of(const KvCache& c, const Params& p, uint32_t b, KvSequence& s, int32_t& q0)
{
    q0 = kv_load(p.q_start + b);
    s = kv_sequence(q0, kv_load(p.q_start + b + 1), kv_load(p.kv_len + b), p.tokens, p.max_new, p.room);
    if (s.bad)
        kv_report(c, s.bad, KERNEL_ATTN_PAGED);
    if (s.new_tokens > p.most_new)
        s.new_tokens = 0;
    return s.new_tokens == 0 ? 0 : (s.kv == 0 ? 1 : (s.kv + UNIT - 1) / UNIT);
}

// Warp-wide: the sequences without new tokens (free places of a batch) are passed over 32 at a time.
__device__ __forceinline__ void advance(Cursor& x, const KvCache& c, const Params& p)
{
    if (++x.un < x.units)
        return;
    x.un = 0;
    if (++x.head < c.kv_heads)
        return;
    x.head = 0;
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t first = x.b + 1; first < c.batch; first += 32) {
        KvSequence s = {0, 0, 0};
        int32_t q0 = 0;
        const uint32_t n = first + lane < c.batch ? units_of(c, p, first + lane, s, q0) : 0;
        const uint32_t found = __ballot_sync(0xffffffffu, n != 0);
        if (found) {
            const uint32_t src = __ffs(found) - 1;
            x.b = first + src;
            x.units = __shfl_sync(0xffffffffu, n, src);
            x.s.new_tokens = __shfl_sync(0xffffffffu, s.new_tokens, src);
            x.s.kv = __shfl_sync(0xffffffffu, s.kv, src);
            x.q0 = __shfl_sync(0xffffffffu, q0, src);
            return;
        }
    }
}

// NB: up to 8 * NB rows.
template <int D, int NB>
__global__ void __launch_bounds__(THREADS, Shape<D, NB>::CTAS)
attention_paged_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                              const KvCache c, const Params p)
{
    using S = Shape<D, NB>;
    constexpr int KC = D / 64;       // 16-byte chunks of a key row per lane
    constexpr int STEPS = D / 32;    // MMA steps along d of the scores
    constexpr int MT = D / 16;       // row tiles of O^T
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2][S::TILES];
    __shared__ alignas(16) float scales[S::TILES][2 * BLOCKS];  // with a K tile: ks of its blocks, then vs; read in pairs
    __shared__ uint32_t valid[S::TILES];            // with a K tile: a bit for each block that is there
    __shared__ uint32_t group_first[MAX_GROUPS + 1];
    __shared__ volatile uint32_t abort_flag;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    auto full = [&](uint32_t i) { return smem_u32(&bars[0][i]); };
    auto empty = [&](uint32_t i) { return smem_u32(&bars[1][i]); };

    if (threadIdx.x < S::TILES) {
        mbar_init(full(threadIdx.x), 1 + 2 * BLOCKS);  // the bytes' arrive and the lanes that fetch scales
        mbar_init(empty(threadIdx.x), WARPS);
    }
    if (threadIdx.x == 0)
        abort_flag = 0;
    fence_barrier_init();
    kv_begin();
    if (threadIdx.x == 0)
        p.meta[blockIdx.x] = make_uint2(NO_PAIR, 0);

    // ---- units of every sequence.  Up to 32 sequences: a lane each, in every warp.  More: sums of 32 at a time, then a running
    // sum over those.
    const uint32_t groups = (c.batch + 31) / 32;
    KvSequence s = {0, 0, 0};
    int32_t q0 = 0;
    uint32_t mine = 0, total;  // of sequence 32 * lo + lane
    auto count = [&](uint32_t b) { return b < c.batch ? units_of(c, p, b, s, q0) : 0; };
    if (groups == 1) {
        mine = count(lane);
        total = __reduce_add_sync(0xffffffffu, mine);
        __syncthreads();  // the barriers are there
    } else {
        for (uint32_t i = warp; i < groups; i += WARPS + 1) {
            const uint32_t n = __reduce_add_sync(0xffffffffu, count(i * 32 + lane));
            if (lane == 0)
                group_first[i] = n;
        }
        __syncthreads();
        if (warp == 0) {
            uint32_t sum = 0;
            for (uint32_t i = 0; i < groups; i += 32) {
                const uint32_t n = i + lane < groups ? group_first[i + lane] : 0;
                uint32_t incl = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
                    incl += lane >= o ? x : 0;
                }
                if (i + lane < groups)
                    group_first[i + lane] = sum + incl - n;
                sum += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (lane == 0)
                group_first[groups] = sum;
        }
        __syncthreads();
        total = group_first[groups];
    }
    const KvCut cut((uint64_t)total * c.kv_heads, gridDim.x);
    const uint32_t worker = blockIdx.x;
    if (worker >= cut.workers)
        return;
    uint32_t left = (uint32_t)(cut.begin(worker + 1) - cut.begin(worker));  // see KV_MOST_KEYS

    // ---- the sequence, head and unit that the CTA begins with
    Cursor at;
    {
        const uint64_t begin = cut.begin(worker);
        uint32_t lo = 0, before = 0;
        if (groups > 1) {
            for (uint32_t n = groups; n > 1;) {
                const uint32_t step = (n + 31) / 32;
                const uint32_t hit = __ballot_sync(0xffffffffu, lane * step < n &&
                                                   (uint64_t)group_first[lo + (lane * step < n ? lane * step : 0)] * c.kv_heads <= begin);
                const uint32_t last = 31 - __clz(hit);
                lo += last * step;
                n = n - last * step < step ? n - last * step : step;
            }
            mine = count(lo * 32 + lane);
            before = group_first[lo];
        }
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
            incl += lane >= o ? x : 0;
        }
        const uint64_t first = ((uint64_t)before + incl - mine) * c.kv_heads;
        const uint32_t src =
            __ffs(__ballot_sync(0xffffffffu, mine != 0 && begin >= first && begin < first + (uint64_t)mine * c.kv_heads)) - 1;
        at.b = lo * 32 + src;
        const uint64_t local = __shfl_sync(0xffffffffu, (unsigned long long)(begin - first), src);
        at.s.new_tokens = __shfl_sync(0xffffffffu, s.new_tokens, src);
        at.s.kv = __shfl_sync(0xffffffffu, s.kv, src);
        at.s.bad = 0;
        at.q0 = __shfl_sync(0xffffffffu, q0, src);
        at.units = __shfl_sync(0xffffffffu, mine, src);
        at.head = (uint32_t)(local / at.units);
        at.un = (uint32_t)(local - (uint64_t)at.head * at.units);
    }

    if (warp == WARPS) {
        // ------------------------------------------------------------ loader: lane i has block i % 8 of a unit
        auto lookup = [&]() {
            const uint32_t pos = at.un * UNIT + (lane % BLOCKS) * KV_BLOCK;
            return lane < 2 * BLOCKS && pos < at.s.kv ? kv_page(c, at.b, pos, KERNEL_ATTN_PAGED) : KV_NO_PAGE;
        };
        uint32_t page = lookup();
        uint32_t tile = 0, phase = 1;
        bool ok = true;
        for (; ok && left; --left) {
            const bool there = page != KV_NO_PAGE;
            const uint32_t mask = __ballot_sync(0xffffffffu, there) & ((1u << BLOCKS) - 1);
            const size_t row = there ? kv_row(c, page, at.head, at.un * UNIT + (lane % BLOCKS) * KV_BLOCK) : 0;
            if (left > 1) {
                advance(at, c, p);
                page = lookup();  // of the next unit, while this one is asked for
            }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                ok = ok && mbar_wait_bounded(empty(tile), phase, &abort_flag, c.status, SITE_EMPTY, KERNEL_ATTN_PAGED);
                if (!ok)
                    break;
                const uint32_t bar = full(tile);
                if (lane == 0) {
                    if (v == 0)
                        valid[tile] = mask;
                    mbar_expect_tx(bar, __popc(mask) * S::BLOCK_BYTES);
                }
                __syncwarp();
                if (lane < 2 * BLOCKS) {
                    if (there && lane < BLOCKS)
                        tma_load_2d(ring + tile * S::TILE_BYTES + lane * S::BLOCK_BYTES, v ? &v_map : &k_map, bar, 0, (int32_t)row);
                    if (there && v == 0)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&scales[tile][lane])),
                                     "l"((lane < BLOCKS ? c.ks : c.vs) + row / KV_BLOCK) : "memory");
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
                }
                __syncwarp();
                if (++tile == S::TILES) {
                    tile = 0;
                    phase ^= 1u;
                }
            }
        }
        if (abort_flag)
            for (uint32_t spin = 0; spin < 2000; ++spin)
                __nanosleep(100);  // the copies in flight land before the shared memory is given up
        return;
    }

    // ---------------------------------------------------------------- the walk
    // A wait that has given up ends no loop here (the warps meet at barriers): the rest is run through without waiting.
    const uint32_t g = lane >> 2, t = lane & 3u;
    float* merge = reinterpret_cast<float*>(smem_raw + (ring - smem_u32(smem_raw)) + S::TILES * S::TILE_BYTES);
    uint32_t bq[NB][STEPS][6];  // q's digits: h, m, l
    float sq[NB][2];            // and their unit, times log2(e) / sqrt(d)
    float o[NB][MT][4];         // a lane's rows are 8 nb + 2t and 8 nb + 2t + 1
    float ref[NB][2], l[NB][2];
    uint32_t seen[NB][2];
    uint32_t seen_least = 0;
    bool open = false, from_start = false, ok = true;
    uint32_t tile = 0, phase = 0;
    auto wait = [&]() {
        if (ok)
            ok = mbar_wait_bounded(full(tile), phase, &abort_flag, c.status, SITE_FULL, KERNEL_ATTN_PAGED);
    };
    auto next_tile = [&]() {
        __syncwarp();  // every lane has read the tile
        if (lane == 0)
            mbar_arrive(empty(tile));
        if (++tile == S::TILES) {
            tile = 0;
            phase ^= 1u;
        }
    };
    // Row g of a tile of 8 keys is key gp.  At 128 dims they are numbered so that the eight lanes of a shared-memory phase
    // read eight different chunks of 16 bytes, of K (one row, four chunks) and of V (four rows, chunk gp).
    const uint32_t gp = D == 128 ? (g >> 1) + (g & 1u) * 4 : g;
    auto key_of = [&](uint32_t e) { return D == 128 ? t + 4 * e : 2 * t + e; };  // that of row 2t + e
    for (; left; --left) {
        if (!open) {
            // ---- a new (sequence, head): its rows of q, what each sees
            open = true;
            from_start = at.un == 0;
            const uint32_t rows = at.s.new_tokens * p.group;
            seen_least = 0xffffffffu;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const uint32_t row = nb * 8 + g;
                const uint32_t i = row / p.group;
                const bool there = row < rows;
                const uint32_t sees = there ? kv_visible(at.s, i, p.causal != 0) : 0xffffffffu;
                seen_least = min(seen_least, sees);
                const __half* src = p.q + (size_t)((uint32_t)at.q0 + i) * p.q_stride +
                                    (size_t)(at.head * p.group + row - i * p.group) * D + 16 * t;
                uint4 w[KC][2];
                __half2 top = __float2half2_rn(0.0f);
#pragma unroll
                for (int ch = 0; ch < KC; ++ch)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        w[ch][h] = make_uint4(0, 0, 0, 0);
                        if (there)
                            w[ch][h] = *reinterpret_cast<const uint4*>(src + ch * 64 + h * 8);
                        const __half2* x = reinterpret_cast<const __half2*>(&w[ch][h]);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            top = __hmax2_nan(top, __habs2(x[e]));
                    }
                top = __hmax2_nan(top, __lowhigh2highlow(top));
                top = __hmax2_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = __hmax2_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float most = __low2float(top);
                // a row with an infinity or a NaN in it has no digits: all its scores are NaN
                const bool finite = most < INFINITY;
                const float unit = finite ? 127.0f * 16384.0f / fmaxf(most, 1e-30f) : 0.0f;
                const float mine = finite ? p.scale_log2 * most * (1.0f / (127.0f * 16384.0f)) : NAN;
#pragma unroll
                for (int ch = 0; ch < KC; ++ch)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int k2 = 0; k2 < 2; ++k2) {  // dims 16 (t + 4 ch) + 8 h + 4 k2 ...
                            const __half2* x = reinterpret_cast<const __half2*>(&w[ch][h]) + 2 * k2;
                            const float2 x0 = __half22float2(x[0]), x1 = __half22float2(x[1]);
                            const float v[4] = {x0.x * unit, x0.y * unit, x1.x * unit, x1.y * unit};
                            uint32_t dg[3];
                            digits(v, dg);
#pragma unroll
                            for (int e = 0; e < 3; ++e)
                                bq[nb][ch * 2 + h][2 * e + k2] = dg[e];
                        }
#pragma unroll
                for (int e = 0; e < 2; ++e) {  // from the lanes that hold row 2t + e as their g
                    sq[nb][e] = __shfl_sync(0xffffffffu, mine, 8 * t + 4 * e);
                    seen[nb][e] = __shfl_sync(0xffffffffu, sees, 8 * t + 4 * e);
                    ref[nb][e] = -INFINITY;
                    l[nb][e] = 0.0f;
                }
#pragma unroll
                for (int i2 = 0; i2 < MT; ++i2)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[nb][i2][e] = 0.0f;
            }
            seen_least = __reduce_min_sync(0xffffffffu, seen_least);
        }
        wait();
        const uint32_t key0 = at.un * UNIT + warp * 32;
        const uint32_t mask = valid[tile] >> (2 * warp) & 3u;
        const float2 k_sc = *reinterpret_cast<const float2*>(&scales[tile][2 * warp]);
        const float2 v_sc = *reinterpret_cast<const float2*>(&scales[tile][BLOCKS + 2 * warp]);
        const uint32_t k_src = ring + tile * S::TILE_BYTES + 2 * warp * S::BLOCK_BYTES;
        if (mask == 0) {  // past the sequence's end
            next_tile();
            wait();
            next_tile();
        } else {
            // ---- scores: two blocks of 16 keys x the rows; x[.][.][e]: key gp + 8 (e / 2), row 2t + e % 2
            float x[2][NB][4];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                int acc[NB][3][4];
                const uint32_t row = k_src + kb * S::BLOCK_BYTES + gp * D;
#pragma unroll
                for (int ch = 0; ch < KC; ++ch) {
                    const uint32_t chunk = 16 * (D == 128 ? ((t + 4 * ch) ^ gp) : (t ^ ((gp >> 1) & 3u)));  // gp + 8 has the same
                    const uint4 w0 = lds128(row + chunk), w1 = lds128(row + 8 * D + chunk);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int e = 0; e < 3; ++e) {
                            if (ch == 0)
                                imma_first(acc[nb][e], w0.x, w1.x, w0.y, w1.y, bq[nb][0][2 * e], bq[nb][0][2 * e + 1]);
                            else
                                imma(acc[nb][e], w0.x, w1.x, w0.y, w1.y, bq[nb][2 * ch][2 * e], bq[nb][2 * ch][2 * e + 1]);
                            imma(acc[nb][e], w0.z, w1.z, w0.w, w1.w, bq[nb][2 * ch + 1][2 * e], bq[nb][2 * ch + 1][2 * e + 1]);
                        }
                }
                // each digit's sum stays below 127 * 127 * 128 = 2^21
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[kb][nb][e] = fmaf((float)acc[nb][0][e], 16384.0f, (float)(acc[nb][1][e] * 128 + acc[nb][2][e]));
            }
            next_tile();
            // ---- scale, mask, maximum
            const float vs[2] = {fmaxf(v_sc.x, KV_SCALE_MIN), fmaxf(v_sc.y, KV_SCALE_MIN)};
            const float ks[2] = {fmaxf(k_sc.x, KV_SCALE_MIN), fmaxf(k_sc.y, KV_SCALE_MIN)};
            const float lv[2] = {__log2f(vs[0]), __log2f(vs[1])};
            float iv[2] = {__fdividef(1.0f, vs[0]), __fdividef(1.0f, vs[1])};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[kb][nb][e] = fmaf(x[kb][nb][e], ks[kb] * sq[nb][e & 1], lv[kb]);
            if (mask != 3u || key0 + 32 > seen_least) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!(mask >> kb & 1u) || key0 + kb * 16 + gp + 8 * (e >> 1) >= seen[nb][e & 1])
                                x[kb][nb][e] = -INFINITY;
                // a block that is not there has no scale either
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    iv[kb] = (mask >> kb & 1u) ? iv[kb] : 0.0f;
            }
            float top[NB][2];
            bool grow = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float m = fmaxf(fmaxf(x[0][nb][e], x[0][nb][e + 2]), fmaxf(x[1][nb][e], x[1][nb][e + 2]));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    top[nb][e] = m;
                    grow = grow || m - ref[nb][e] > WINDOW;  // the sum would be rounded
                }
            // ---- a new reference where the old one has become too small
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float next = fmaxf(ref[nb][e], top[nb][e] - KV_P_TOP);
                        const float alpha = next == -INFINITY ? 1.0f : ex2(ref[nb][e] - next);
                        ref[nb][e] = next;
                        l[nb][e] *= alpha;
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            o[nb][i][e] *= alpha;
                            o[nb][i][e + 2] *= alpha;
                        }
                    }
            }
            // ---- P: the sum in f32, as f16 operands turned round
            uint32_t pb[2][NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float base[2] = {ref[nb][0] == -INFINITY ? 0.0f : ref[nb][0], ref[nb][1] == -INFINITY ? 0.0f : ref[nb][1]};
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    float pr[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        pr[e] = ex2(x[kb][nb][e] - base[e & 1]);
                    l[nb][0] = fmaf(pr[0] + pr[2], iv[kb], l[nb][0]);
                    l[nb][1] = fmaf(pr[1] + pr[3], iv[kb], l[nb][1]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const __half2 pk = __floats2half2_rn(pr[2 * h], pr[2 * h + 1]);
                        pb[kb][nb][h] = transpose8(*reinterpret_cast<const uint32_t*>(&pk));
                    }
                }
            }
            wait();
            const uint32_t v_src = ring + tile * S::TILE_BYTES + 2 * warp * S::BLOCK_BYTES;
            // ---- O^T += V^T P^T, 16 keys a step: lane (g, t) reads the keys of the rows 2t and 2t + 1 of both tiles of 8, and
            // of each the D / 8 dims from (D / 8) gp on, two for each row tile
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const uint32_t blk = v_src + kb * S::BLOCK_BYTES;
                uint32_t w[4][D / 32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t key = (i >> 1) * 8 + key_of(i & 1);
                    if constexpr (D == 128) {
                        const uint4 v = lds128(blk + key * D + (gp ^ (key & 7u)) * 16);
                        w[i][0] = v.x;
                        w[i][1] = v.y;
                        w[i][2] = v.z;
                        w[i][3] = v.w;
                    } else {
                        const uint2 v = lds64(blk + key * D + ((g >> 1) ^ ((key >> 1) & 3u)) * 16 + (g & 1u) * 8);
                        w[i][0] = v.x;
                        w[i][1] = v.y;
                    }
                }
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    uint32_t a[4], a8[4];  // dims 4i ... 4i + 3 of the lane, keys of the first and of the second tile
                    s8x4_to_f16(__byte_perm(w[0][i], w[1][i], 0x5140), a[0], a[1]);
                    s8x4_to_f16(__byte_perm(w[0][i], w[1][i], 0x7362), a[2], a[3]);
                    s8x4_to_f16(__byte_perm(w[2][i], w[3][i], 0x5140), a8[0], a8[1]);
                    s8x4_to_f16(__byte_perm(w[2][i], w[3][i], 0x7362), a8[2], a8[3]);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        mma_m16n8k16_f16(o[nb][2 * i], a[0], a[1], a8[0], a8[1], pb[kb][nb][0], pb[kb][nb][1]);
                        mma_m16n8k16_f16(o[nb][2 * i + 1], a[2], a[3], a8[2], a8[3], pb[kb][nb][0], pb[kb][nb][1]);
                    }
                }
            }
            next_tile();
        }

        const bool last = at.un + 1 == at.units;
        if (last || left == 1) {
            // ---- the end of this (sequence, head), or of this CTA's part of it: the warps' sums are added in
            // two steps, 2 to 0 and 3 to 1, then 1 to 0
            open = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int k = 4; k < 32; k <<= 1)
                        l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], k);
            auto give = [&](uint32_t buf) {
                float* m = merge + buf * S::MERGE_FLOATS + lane;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            m[((nb * MT + i) * 4 + e) * 32] = o[nb][i][e];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        m[((NB * MT + nb) * 4 + e) * 32] = ref[nb][e];
                        m[((NB * MT + nb) * 4 + 2 + e) * 32] = l[nb][e];
                    }
                }
            };
            auto take = [&](uint32_t buf) {
                const float* m = merge + buf * S::MERGE_FLOATS + lane;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float other = m[((NB * MT + nb) * 4 + e) * 32];
                        const float next = fmaxf(ref[nb][e], other), base = next == -INFINITY ? 0.0f : next;
                        const float f0 = ex2(ref[nb][e] - base), f1 = ex2(other - base);
                        ref[nb][e] = next;
                        l[nb][e] = l[nb][e] * f0 + m[((NB * MT + nb) * 4 + 2 + e) * 32] * f1;
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int k = e; k < 4; k += 2)
                                o[nb][i][k] = o[nb][i][k] * f0 + m[((nb * MT + i) * 4 + k) * 32] * f1;
                    }
            };
            auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); };
            if (warp >= 2)
                give(warp - 2);
            meet();
            if (warp < 2)
                take(warp);
            meet();
            if (warp == 1)
                give(1);
            meet();
            if (warp == 0) {
                take(1);
                const uint32_t rows = at.s.new_tokens * p.group;
                const uint32_t pair = at.b * c.kv_heads + at.head;
                const bool whole = from_start && last;
                constexpr int DL = D / 8;  // a lane's dims of its two rows, from DL * gp on
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t row = nb * 8 + 2 * t + e;
                        if (row >= rows)
                            continue;
                        float y[DL];
#pragma unroll
                        for (int i = 0; i < DL; ++i)
                            y[i] = o[nb][i >> 1][(i & 1) * 2 + e];
                        if (whole) {
                            const uint32_t i = row / p.group;
                            const float inv = l[nb][e] == 0.0f ? 0.0f : __fdividef(1.0f, l[nb][e]);
                            __half* dst = p.out + ((size_t)((uint32_t)at.q0 + i) * p.heads + at.head * p.group + row - i * p.group) * D + DL * gp;
#pragma unroll
                            for (int k = 0; k < DL; k += 8) {
                                uint32_t h[4];
#pragma unroll
                                for (int k2 = 0; k2 < 4; ++k2) {
                                    const __half2 v = __floats2half2_rn(y[k + 2 * k2] * inv, y[k + 2 * k2 + 1] * inv);
                                    h[k2] = *reinterpret_cast<const uint32_t*>(&v);
                                }
                                *reinterpret_cast<uint4*>(dst + k) = make_uint4(h[0], h[1], h[2], h[3]);
                            }
                        } else {
                            const uint32_t slot = 2 * worker + (from_start ? 1u : 0u);
                            const size_t prow = (size_t)slot * p.part_rows + row;
#pragma unroll
                            for (int k = 0; k < DL; k += 4)
                                *reinterpret_cast<float4*>(p.part_o + prow * D + DL * gp + k) =
                                    make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]);
                            if (g == 0)
                                *reinterpret_cast<float2*>(p.part_ml + prow * 2) = make_float2(ref[nb][e], l[nb][e]);
                        }
                    }
                if (from_start && !whole && lane == 0) {
                    const uint64_t end = cut.begin(worker + 1) - left + (at.units - at.un);  // of the pair's units
                    p.meta[worker] = make_uint2(pair, cut.owner(end - 1));
                }
            }
            meet();  // the buffers are free again
        }
        if (left > 1)
            advance(at, c, p);
    }
}

// Adds the parts of the (sequence, head) whose first part the worker blockIdx.x left, a row a CTA (or several
// in turn): its warps take the row's parts in turn, each in ascending order, a lane D / 32 dims, and their sums are added in the warps' order.
constexpr int COMBINE_WARPS = 8;

template <int D>
__global__ void __launch_bounds__(COMBINE_WARPS * 32) attention_paged_combine_kernel(const KvCache c, const Params p)
{
    constexpr int V = D / 32;
    __shared__ float sum_o[COMBINE_WARPS][D];
    __shared__ float sum_ml[COMBINE_WARPS][2];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // The tile kernel may start beside this one.  The next call's first launch may not: its CTAs would take the places of
    // this one's that have not started (33 -> 41 us for one token of eight sequences).
    if (p.follows)
        asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t first = blockIdx.x;
    const uint2 meta = p.meta[first];
    if (meta.x == NO_PAIR)
        return;
    const uint32_t pair = meta.x, n = meta.y - first + 1;
    const uint32_t b = pair / c.kv_heads, head = pair - b * c.kv_heads;
    const uint32_t q0 = (uint32_t)kv_load(p.q_start + b);
    const uint32_t new_tokens = (uint32_t)kv_load(p.q_start + b + 1) - q0;  // the pair has parts, so its numbers are good
    for (uint32_t row = blockIdx.y; row < p.part_rows && row < new_tokens * p.group; row += gridDim.y) {
        float ref = -INFINITY, l = 0.0f, acc[V];
#pragma unroll
        for (int e = 0; e < V; ++e)
            acc[e] = 0.0f;
#pragma unroll 8
        for (uint32_t i = warp; i < n; i += COMBINE_WARPS) {
            // part 0 is the first worker's last, the others are their workers' first
            const size_t slot = (size_t)(2 * (first + i) + (i == 0 ? 1u : 0u)) * p.part_rows + row;
            const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot * 2);
            alignas(16) float v[V];
            if constexpr (V == 4)
                *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p.part_o + slot * D + lane * V);
            else
                *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(p.part_o + slot * D + lane * V);
            const float next = fmaxf(ref, ml.x), base = next == -INFINITY ? 0.0f : next;
            const float f0 = ex2(ref - base), f1 = ex2(ml.x - base);
            ref = next;
            l = l * f0 + ml.y * f1;
#pragma unroll
            for (int e = 0; e < V; ++e)
                acc[e] = acc[e] * f0 + v[e] * f1;
        }
#pragma unroll
        for (int e = 0; e < V; ++e)
            sum_o[warp][lane * V + e] = acc[e];
        if (lane == 0) {
            sum_ml[warp][0] = ref;
            sum_ml[warp][1] = l;
        }
        __syncthreads();
        if (warp == 0) {
            float top = -INFINITY;
            for (int w = 0; w < COMBINE_WARPS; ++w)
                top = fmaxf(top, sum_ml[w][0]);
            const float base = top == -INFINITY ? 0.0f : top;
            float total = 0.0f, out[V];
#pragma unroll
            for (int e = 0; e < V; ++e)
                out[e] = 0.0f;
            for (int w = 0; w < COMBINE_WARPS; ++w) {
                const float f = ex2(sum_ml[w][0] - base);
                total = fmaf(f, sum_ml[w][1], total);
#pragma unroll
                for (int e = 0; e < V; ++e)
                    out[e] = fmaf(f, sum_o[w][lane * V + e], out[e]);
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            const uint32_t i = row / p.group;
            __half* dst = p.out + ((size_t)(q0 + i) * p.heads + head * p.group + row - i * p.group) * D + lane * V;
#pragma unroll
            for (int e = 0; e < V; e += 2)
                *reinterpret_cast<__half2*>(dst + e) = __floats2half2_rn(out[e] * inv, out[e + 1] * inv);
        }
        __syncthreads();  // the sums have been read
    }
}

struct Layout {
    uint32_t part_rows;
    size_t part_o, part_ml, meta, floats;  // offsets and the whole length, in floats
};

static Layout layout(uint32_t most_new, uint32_t heads, uint32_t kv_heads, uint32_t head_dim)
{
    Layout a;
    a.part_rows = most_new * (heads / kv_heads);
    const size_t slots = 2 * MAX_WORKERS;
    a.part_o = 0;
    a.part_ml = slots * a.part_rows * head_dim;
    a.meta = a.part_ml + (slots * a.part_rows * 2 + 3) / 4 * 4;
    a.floats = a.meta + 2 * MAX_WORKERS;
    return a;
}

template <int D, int NB>
static cudaError_t launch(const DeviceCtx& ctx, const KvCache& c, const Params& p, const CUtensorMap& km,
                          const CUtensorMap& vm, cudaStream_t stream)
{
    using S = Shape<D, NB>;
    auto kernel = attention_paged_decode_kernel<D, NB>;
    static bool set[64] = {};
    if (!set[ctx.device]) {
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
        if (err != cudaSuccess)
            return err;
        set[ctx.device] = true;
    }
    const uint32_t sms = (uint32_t)ctx.num_sms < MAX_SMS ? (uint32_t)ctx.num_sms : MAX_SMS;
    // in front of the tile kernel, which starts beside the second launch and does not wait for what is in front of this one,
    // only when all that is done
    const cudaError_t err = kv_launch(kernel, dim3(sms * S::CTAS), THREADS, S::SMEM, !p.follows, stream, km, vm, c, p);
    if (err != cudaSuccess)
        return err;
    // beside another kernel, whose calls seldom leave much to add: fewer CTAs, which loop over the rows
    return kv_launch(attention_paged_combine_kernel<D>, dim3(sms * S::CTAS, p.follows && p.part_rows > 2 ? 2 : p.part_rows),
                     COMBINE_WARPS * 32, 0, true, stream, c, p);
}

}  // namespace apdec

bool attention_paged_decode_ok(uint32_t most_new, uint32_t heads, uint32_t kv_heads)
{
    const uint64_t rows = (uint64_t)most_new * (heads / kv_heads);
    return rows > 0 && rows <= apdec::ROWS;  // a batch of 32768 over 4096 heads: 2^27 (sequence, head)
}

size_t attention_paged_decode_scratch(uint32_t most_new, uint32_t heads, uint32_t kv_heads,
                                      uint32_t head_dim)
{
    return apdec::layout(most_new, heads, kv_heads, head_dim).floats;
}

cudaError_t launch_attention_paged_decode(const DeviceCtx& ctx, const KvParams& kp, const __half* q, __half* out,
                                          uint32_t q_stride, uint32_t max_new, uint32_t most_new, bool causal,
                                          bool follows, float* scratch, cudaStream_t stream)
{
    using namespace apdec;
    const KvCache c = kv_cache_of(ctx, kp);
    const Layout a = layout(most_new, kp.heads, kp.kv_heads, kp.head_dim);
    Params p = {};
    p.q = q;
    p.out = out;
    p.q_start = kp.start;
    p.kv_len = kp.kv_len;
    p.part_o = scratch + a.part_o;
    p.part_ml = scratch + a.part_ml;
    p.meta = reinterpret_cast<uint2*>(scratch + a.meta);
    p.tokens = kp.rows;
    p.heads = kp.heads;
    p.group = kp.heads / kp.kv_heads;
    p.q_stride = q_stride;
    p.max_new = max_new;
    p.most_new = most_new;
    p.follows = follows ? 1 : 0;
    p.room = kp.max_pages * kp.page_size;
    p.part_rows = a.part_rows;
    p.scale_log2 = 1.4426950408889634f / sqrtf((float)kp.head_dim);
    p.causal = causal ? 1 : 0;
    CUtensorMap km, vm;
    const uint64_t rows = (uint64_t)kp.num_pages * kp.kv_heads * kp.page_size;
    const CUtensorMapSwizzle sw = kp.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    cudaError_t err = encode_tensor_map_2d(&km, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, kp.k, kp.head_dim, rows, kp.head_dim,
                                           kp.head_dim, KV_BLOCK, sw);
    if (err != cudaSuccess)
        return err;
    err = encode_tensor_map_2d(&vm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, kp.v, kp.head_dim, rows, kp.head_dim, kp.head_dim,
                               KV_BLOCK, sw);
    if (err != cudaSuccess)
        return err;
    const bool one = a.part_rows <= 8;
    if (kp.head_dim == 128)
        return one ? launch<128, 1>(ctx, c, p, km, vm, stream) : launch<128, 2>(ctx, c, p, km, vm, stream);
    return one ? launch<64, 1>(ctx, c, p, km, vm, stream) : launch<64, 2>(ctx, c, p, km, vm, stream);
}

}  // namespace kaio
