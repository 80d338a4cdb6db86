// Attention of a few new tokens per sequence over the paged 8-bit cache (decode steps, drafted tokens): up to 32 rows
// (new tokens x query heads of a key/value head) per (sequence, key/value head).
//
// out = O / l with  x_j = (q . kint_j) ks_j log2(e) / sqrt(d) + log2(vs_j),  P_j = 2^(x_j - ref),
//                   O = sum_j P_j vint_j,  l = sum_j P_j / vs_j.
// ks and vs are constant over 16 keys, so neither scale costs work per cached value, the 8-bit integers are exact as f16
// operands, and P (rounded to f16 for the product, f32 in l) is largest where it weighs most, whatever the scales are.
//
// What bounds it: HBM, every cached byte is read once.  Per byte an SM has 5.6 issue slots of a lane; the conversion to
// f16 takes 1.25 to 1.5, the products are warp-level MMAs (16 rows; tcgen05's 128 would be padding).
//  * A unit is 32 keys of one (sequence, head): K and V by TMA, 16 rows a box, into a ring that belongs to one warp,
//    which loads, waits, multiplies and reloads on its own: no barrier between warps, three units in flight a warp.
//    The box's swizzle makes the row-wise reads of K and the column-wise ones of V free of bank conflicts.
//  * All units of the call are cut evenly over all warps of the grid, whatever the lengths of the sequences: a long
//    sequence is spread over the GPU, short ones are put together.  A warp that holds a part of a (sequence, head)
//    leaves (O, ref, l) in scratch; a second launch, resident before the first ends, adds the parts in ascending order.
#include "kernels.h"
#include "kv_cache.cuh"
#include "mma_sync.cuh"

namespace kaio {
namespace apdec {

constexpr int WARPS = 4;
constexpr int CTAS_PER_SM = 2;
constexpr uint32_t MAX_SMS = 160;
constexpr uint32_t MAX_WORKERS = MAX_SMS * CTAS_PER_SM * WARPS;
constexpr uint32_t UNIT = 32;        // keys of a unit
constexpr uint32_t ROWS = 16;        // rows of a row block
constexpr uint32_t MAX_GROUPS = 1024;  // groups of 32 sequences
constexpr float LAZY = 8.0f;         // P may grow to 2^8 before O and l are rescaled

enum : uint32_t { SITE_FULL = 1 };

struct Params {
    const __half* q;
    __half* out;
    const int32_t *q_start, *kv_len;
    float *part_o, *part_ml;  // [2 * workers][rows][D], [2 * workers][rows][2]
    uint32_t* meta;           // [pairs][2]: first and last worker
    uint32_t tokens, heads, group, q_stride, max_new, room;
    uint32_t row_blocks, part_rows;
    float scale_log2;
    int causal;
};

template <int D>
struct Shape {
    static constexpr uint32_t BLOCK_BYTES = 16 * D;            // 16 keys of K or V
    static constexpr uint32_t STAGE_BYTES = 4 * BLOCK_BYTES;   // K0 K1 V0 V1
    static constexpr uint32_t STAGES = D == 128 ? 3 : 6;
    static constexpr uint32_t SMEM = 1024 + WARPS * STAGES * STAGE_BYTES;
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The rows g of the tile only: rows g + 8 are not there.
__device__ __forceinline__ void mma_half(float& c0, float& c1, uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1)
{
    float d2, d3;
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%0, %1, %9, %9};"
        : "+f"(c0), "+f"(c1), "=f"(d2), "=f"(d3)
        : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1), "f"(0.0f));
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

// Where a walk over the units stands: unit `un` of (sequence b, head and row block pr).
struct Cursor {
    uint32_t b, pr, un, units;
    KvSequence s;
    int32_t q0;
};

__device__ __forceinline__ uint32_t units_of(const KvCache& c, const Params& p, uint32_t b, KvSequence& s, int32_t& q0)
{
    q0 = __ldg(p.q_start + b);
    s = kv_sequence(q0, __ldg(p.q_start + b + 1), __ldg(p.kv_len + b), p.tokens, p.max_new, p.room);
    if (s.bad)
        kv_report(c, s.bad, KERNEL_ATTN_PAGED);
    return s.new_tokens == 0 ? 0 : (s.kv == 0 ? 1 : (s.kv + UNIT - 1) / UNIT);
}

__device__ __forceinline__ void advance(Cursor& x, const KvCache& c, const Params& p)
{
    if (++x.un < x.units)
        return;
    x.un = 0;
    if (++x.pr < c.kv_heads * p.row_blocks)
        return;
    x.pr = 0;
    do {
        if (++x.b >= c.batch)
            return;
        x.units = units_of(c, p, x.b, x.s, x.q0);
    } while (x.units == 0);
}

// HALF: no row block has more than 8 rows.
template <int D, bool HALF>
__global__ void __launch_bounds__(WARPS * 32, CTAS_PER_SM)
attention_paged_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                              const KvCache c, const Params p)
{
    using S = Shape<D>;
    constexpr int KC = D / 64;       // 16-byte chunks of a key row per lane
    constexpr int STEPS = D / 16;    // MMA steps along d
    constexpr int NT = D / 8;        // column tiles of the output
    constexpr int RH = HALF ? 1 : 2; // row halves
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[WARPS][S::STAGES];
    __shared__ float4 scales[WARPS][S::STAGES];  // ks0 ks1 vs0 vs1
    __shared__ uint32_t valid[WARPS][S::STAGES];
    __shared__ uint32_t group_first[MAX_GROUPS + 1];
    __shared__ volatile uint32_t abort_flag;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3u;
    const uint32_t ring = ((smem_u32(smem_raw) + 1023u) & ~1023u) + warp * S::STAGES * S::STAGE_BYTES;
    const uint32_t bar0 = smem_u32(&bars[warp][0]);
    asm volatile("griddepcontrol.launch_dependents;");

    // ---- units of every sequence: sums of 32 at a time, then a running sum over those
    const uint32_t groups = (c.batch + 31) / 32;
    for (uint32_t i = warp; i < groups; i += WARPS) {
        KvSequence s;
        int32_t q0;
        uint32_t n = i * 32 + lane < c.batch ? units_of(c, p, i * 32 + lane, s, q0) : 0;
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0)
            group_first[i] = n;
    }
    if (lane < S::STAGES)
        mbar_init(bar0 + 8 * lane, 1 + 4);  // the bytes' arrive and the four lanes that fetch scales
    if (threadIdx.x == 0)
        abort_flag = 0;
    fence_barrier_init();
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
    const uint32_t hr = c.kv_heads * p.row_blocks;
    const KvCut cut((uint64_t)group_first[groups] * hr, gridDim.x * WARPS);
    const uint32_t worker = warp * gridDim.x + blockIdx.x;  // few units: one SM each before a second
    if (worker >= cut.workers)
        return;
    const uint64_t begin = cut.begin(worker);
    uint64_t left = cut.begin(worker + 1) - begin;

    // ---- the sequence, head and unit that `begin` is
    Cursor load;
    {
        uint32_t lo = 0, n = groups;
        while (n > 1) {
            const uint32_t step = (n + 31) / 32;
            const uint32_t hit = __ballot_sync(0xffffffffu, lane * step < n &&
                                               (uint64_t)group_first[lo + (lane * step < n ? lane * step : 0)] * hr <= begin);
            const uint32_t last = 31 - __clz(hit);
            lo += last * step;
            n = n - last * step < step ? n - last * step : step;
        }
        KvSequence s = {0, 0, 0};
        int32_t q0 = 0;
        const uint32_t b = lo * 32 + lane;
        const uint32_t mine = b < c.batch ? units_of(c, p, b, s, q0) : 0;
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
            incl += lane >= o ? x : 0;
        }
        const uint64_t first = ((uint64_t)group_first[lo] + incl - mine) * hr;
        const uint32_t src = __ffs(__ballot_sync(0xffffffffu, mine != 0 && begin >= first && begin < first + (uint64_t)mine * hr)) - 1;
        load.b = lo * 32 + src;
        load.units = __shfl_sync(0xffffffffu, mine, src);
        const uint64_t local = __shfl_sync(0xffffffffu, (unsigned long long)(begin - first), src);
        load.s.new_tokens = __shfl_sync(0xffffffffu, s.new_tokens, src);
        load.s.kv = __shfl_sync(0xffffffffu, s.kv, src);
        load.s.bad = 0;
        load.q0 = __shfl_sync(0xffffffffu, q0, src);
        load.pr = (uint32_t)(local / load.units);
        load.un = (uint32_t)(local - (uint64_t)load.pr * load.units);
    }
    Cursor at = load;
    uint64_t to_load = left;
    // Lanes 0 and 1 fetch the two blocks of a unit, lanes 0 to 3 the scales ks0 ks1 vs0 vs1.  The page of the unit
    // after the next to be loaded is looked up a unit ahead.
    auto lookup = [&]() {
        const uint32_t pos = load.un * UNIT + (lane & 1u) * KV_BLOCK;
        uint32_t page = KV_NO_PAGE;
        if (lane < 4 && pos < load.s.kv)
            page = kv_page(c, load.b, pos, KERNEL_ATTN_PAGED);
        return page;
    };
    uint32_t page = lookup();
    auto issue = [&](uint32_t stage) {
        const uint32_t bar = bar0 + 8 * stage, dst = ring + stage * S::STAGE_BYTES;
        const bool ok = page != KV_NO_PAGE;
        const uint32_t mask = __ballot_sync(0xffffffffu, ok) & 3u;
        if (lane == 0) {
            valid[warp][stage] = mask;
            mbar_expect_tx(bar, __popc(mask) * 2 * S::BLOCK_BYTES);
        }
        __syncwarp();
        if (lane < 4) {
            const uint32_t pos = load.un * UNIT + (lane & 1u) * KV_BLOCK;
            const uint32_t head = load.pr / p.row_blocks;
            if (ok) {
                if (lane < 2) {
                    const int32_t y = (int32_t)(kv_row(c, page, head) + pos % c.page_size);
                    tma_load_2d(dst + lane * S::BLOCK_BYTES, &k_map, bar, 0, y);
                    tma_load_2d(dst + (2 + lane) * S::BLOCK_BYTES, &v_map, bar, 0, y);
                }
                const float* src = (lane < 2 ? c.ks : c.vs) + kv_scale_row(c, page, head) + pos % c.page_size / KV_BLOCK;
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(
                                 smem_u32(&scales[warp][stage]) + 4 * lane), "l"(src) : "memory");
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
        }
        __syncwarp();
        if (--to_load) {
            advance(load, c, p);
            page = lookup();
        }
    };
#pragma unroll 1
    for (uint32_t s = 0; s < S::STAGES && to_load; ++s)
        issue(s);

    // ---- the walk
    uint32_t aq[STEPS][2 * RH];
    float o[NT][2 * RH];
    float ref[RH], l[RH];
    uint32_t seen[RH];
    uint32_t seen_least = 0;
    bool open = false, from_start = false;
    uint32_t stage = 0, phase = 0;
    // Key of this lane's score columns 2t and 2t + 1 inside a tile of 8.  At 128 dims the keys (and the output's dims)
    // of a tile are numbered so that the eight lanes of a shared-memory phase read eight different chunks of 16 bytes.
    auto column = [&](uint32_t e) { return D == 128 ? t + 4 * e : 2 * t + e; };
    // First of the NT dims in this lane's output columns 2t + e.
    auto dims = [&](uint32_t e) { return D == 128 ? 16 * t + 64 * e : 16 * t + 8 * e; };
    for (; left; --left) {
        if (!open) {
            // ---- a new (sequence, head, row block): its rows of q, what each sees
            open = true;
            from_start = at.un == 0;
            const uint32_t head = at.pr / p.row_blocks, rb = at.pr - head * p.row_blocks;
            const uint32_t rows = at.s.new_tokens * p.group;
            seen_least = 0xffffffffu;
#pragma unroll
            for (int r = 0; r < RH; ++r) {
                const uint32_t row = rb * ROWS + r * 8 + g;
                const uint32_t i = row / p.group;
                const bool there = row < rows;
                seen[r] = there ? kv_visible(at.s, i, p.causal != 0) : 0xffffffffu;
                seen_least = min(seen_least, seen[r]);
                const __half* src = p.q + (size_t)((uint32_t)at.q0 + i) * p.q_stride +
                                    (size_t)(head * p.group + row - i * p.group) * D + 16 * t;
#pragma unroll
                for (int ch = 0; ch < KC; ++ch)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint4 x = make_uint4(0, 0, 0, 0);
                        if (there)
                            x = *reinterpret_cast<const uint4*>(src + ch * 64 + h * 8);
                        const int st = ch * 4 + h * 2;
                        aq[st][r] = x.x;
                        aq[st][RH + r] = x.y;
                        aq[st + 1][r] = x.z;
                        aq[st + 1][RH + r] = x.w;
                    }
                ref[r] = -INFINITY;
                l[r] = 0.0f;
            }
            seen_least = __reduce_min_sync(0xffffffffu, seen_least);
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 2 * RH; ++e)
                    o[i][e] = 0.0f;
        }
        if (!mbar_wait_bounded(bar0 + 8 * stage, phase, &abort_flag, c.status, SITE_FULL, KERNEL_ATTN_PAGED))
            break;
        const uint32_t src = ring + stage * S::STAGE_BYTES;
        const uint32_t mask = valid[warp][stage];
        const float4 sc = scales[warp][stage];

        // ---- scores: rows x 32 keys
        float x[4][2 * RH];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t key = (j & 1) * 8 + (D == 128 ? (g >> 1) + (g & 1u) * 4 : g);  // row of the 16-row box
            const uint32_t row = src + (j >> 1) * S::BLOCK_BYTES + key * D;
#pragma unroll
            for (int e = 0; e < 2 * RH; ++e)
                x[j][e] = 0.0f;
#pragma unroll
            for (int ch = 0; ch < KC; ++ch) {
                const uint32_t chunk = D == 128 ? ((t + 4 * ch) ^ (key & 7u)) : (t ^ ((key >> 1) & 3u));
                const uint4 w = lds128(row + chunk * 16);
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t b0, b1;
                    s8x4_to_f16(ws[i], b0, b1);
                    const int st = ch * 4 + i;
                    if constexpr (HALF)
                        mma_half(x[j][0], x[j][1], aq[st][0], aq[st][1], b0, b1);
                    else
                        mma_m16n8k16_f16(x[j], aq[st][0], aq[st][1], aq[st][2], aq[st][3], b0, b1);
                }
            }
        }
        // ---- scale, mask, maximum
        const float vs[2] = {fmaxf(sc.z, KV_SCALE_MIN), fmaxf(sc.w, KV_SCALE_MIN)};
        float ck[2] = {fmaxf(sc.x, KV_SCALE_MIN) * p.scale_log2, fmaxf(sc.y, KV_SCALE_MIN) * p.scale_log2};
        float lv[2] = {__log2f(vs[0]), __log2f(vs[1])}, iv[2] = {__frcp_rn(vs[0]), __frcp_rn(vs[1])};
        const bool all = mask == 3u && (at.un + 1) * UNIT <= seen_least;
        float top[RH];
#pragma unroll
        for (int r = 0; r < RH; ++r)
            top[r] = -INFINITY;
        if (!all) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < RH; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t key = at.un * UNIT + j * 8 + column(e);
                        const bool live = (mask >> (j >> 1) & 1u) && key < seen[r];
                        x[j][2 * r + e] = live ? fmaf(x[j][2 * r + e], ck[j >> 1], lv[j >> 1]) : -INFINITY;
                    }
            // a block that is not there has no scale either
#pragma unroll
            for (int i = 0; i < 2; ++i)
                iv[i] = (mask >> i & 1u) ? iv[i] : 0.0f;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2 * RH; ++e)
                    x[j][e] = fmaf(x[j][e], ck[j >> 1], lv[j >> 1]);
        }
#pragma unroll
        for (int r = 0; r < RH; ++r) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                top[r] = fmaxf(top[r], fmaxf(x[j][2 * r], x[j][2 * r + 1]));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
        }
        // ---- a new reference where the old one has become too small
        bool grow = top[0] > ref[0] + LAZY;
        if (RH == 2)
            grow = grow || top[RH - 1] > ref[RH - 1] + LAZY;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int r = 0; r < RH; ++r) {
                const float next = fmaxf(ref[r], top[r]);
                const float alpha = next == -INFINITY ? 1.0f : ex2(ref[r] - next);
                ref[r] = next;
                l[r] *= alpha;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    o[i][2 * r] *= alpha;
                    o[i][2 * r + 1] *= alpha;
                }
            }
        }
        // ---- P: the sum in f32, the pairs of keys as f16 operands
        uint32_t pa[2][2 * RH];
#pragma unroll
        for (int r = 0; r < RH; ++r) {
            const float base = ref[r] == -INFINITY ? 0.0f : ref[r];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                float part = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float p0 = ex2(x[2 * ks + h][2 * r] - base), p1 = ex2(x[2 * ks + h][2 * r + 1] - base);
                    part += p0 + p1;
                    const __half2 pk = __floats2half2_rn(p0, p1);
                    pa[ks][h * RH + r] = *reinterpret_cast<const uint32_t*>(&pk);
                }
                l[r] = fmaf(part, iv[ks], l[r]);
            }
        }
        // ---- O += P V: 16 keys a step; lane (g, t) reads the keys of its two columns in both tiles, and of each the
        // D / 8 dims that are its column of every output tile
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const uint32_t blk = src + (2 + ks) * S::BLOCK_BYTES;
            uint32_t w[4][D / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t key = (i >> 1) * 8 + column(i & 1);
                if constexpr (D == 128) {
                    const uint4 v = lds128(blk + key * D + (((g >> 1) + (g & 1u) * 4) ^ (key & 7u)) * 16);
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
                uint32_t b0[4], b1[4];
                s8x4_to_f16(__byte_perm(w[0][i], w[1][i], 0x5140), b0[0], b0[1]);
                s8x4_to_f16(__byte_perm(w[0][i], w[1][i], 0x7362), b0[2], b0[3]);
                s8x4_to_f16(__byte_perm(w[2][i], w[3][i], 0x5140), b1[0], b1[1]);
                s8x4_to_f16(__byte_perm(w[2][i], w[3][i], 0x7362), b1[2], b1[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (HALF)
                        mma_half(o[4 * i + e][0], o[4 * i + e][1], pa[ks][0], pa[ks][1], b0[e], b1[e]);
                    else
                        mma_m16n8k16_f16(o[4 * i + e], pa[ks][0], pa[ks][1], pa[ks][2], pa[ks][3], b0[e], b1[e]);
                }
            }
        }
        __syncwarp();  // every lane has read the stage
        if (to_load)
            issue(stage);
        if (++stage == S::STAGES) {
            stage = 0;
            phase ^= 1u;
        }

        const bool last = at.un + 1 == at.units;
        if (last || left == 1) {
            // ---- the end of this (sequence, head, row block), or of this warp's part of it
            open = false;
            const uint32_t head = at.pr / p.row_blocks, rb = at.pr - head * p.row_blocks;
            const uint32_t rows = at.s.new_tokens * p.group;
            const uint32_t pair = at.b * hr + at.pr;
            const bool whole = from_start && last;
#pragma unroll
            for (int r = 0; r < RH; ++r) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
                const uint32_t row = rb * ROWS + r * 8 + g;
                if (row < rows) {
                    if (whole) {
                        const uint32_t i = row / p.group;
                        const float inv = l[r] == 0.0f ? 0.0f : __fdividef(1.0f, l[r]);
                        __half* dst = p.out + ((size_t)((uint32_t)at.q0 + i) * p.heads + head * p.group + row - i * p.group) * D;
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int i8 = 0; i8 < NT; i8 += 8) {
                                uint32_t h[4];
#pragma unroll
                                for (int k2 = 0; k2 < 4; ++k2) {
                                    const __half2 v = __floats2half2_rn(o[i8 + 2 * k2][2 * r + e] * inv, o[i8 + 2 * k2 + 1][2 * r + e] * inv);
                                    h[k2] = *reinterpret_cast<const uint32_t*>(&v);
                                }
                                *reinterpret_cast<uint4*>(dst + dims(e) + i8) = make_uint4(h[0], h[1], h[2], h[3]);
                            }
                    } else {
                        const uint32_t slot = 2 * worker + (from_start ? 1u : 0u);
                        const size_t prow = (size_t)slot * p.part_rows + r * 8 + g;
                        float* dst = p.part_o + prow * D;
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int i4 = 0; i4 < NT; i4 += 4)
                                *reinterpret_cast<float4*>(dst + dims(e) + i4) =
                                    make_float4(o[i4][2 * r + e], o[i4 + 1][2 * r + e], o[i4 + 2][2 * r + e], o[i4 + 3][2 * r + e]);
                        if (t == 0)
                            *reinterpret_cast<float2*>(p.part_ml + prow * 2) = make_float2(ref[r], l[r]);
                    }
                }
            }
            if (from_start && lane == 0) {
                const uint64_t end = (begin + (cut.begin(worker + 1) - begin - left)) + (at.units - at.un);
                p.meta[2 * pair] = worker;
                p.meta[2 * pair + 1] = whole ? worker : cut.owner(end - 1);
            }
        }
        advance(at, c, p);
    }
    if (abort_flag)
        for (uint32_t spin = 0; spin < 2000; ++spin)
            __nanosleep(100);  // the copies in flight land before the shared memory is given up
}

// Adds the parts of one row of one (sequence, head, row block).
template <int D>
__global__ void __launch_bounds__(D) attention_paged_combine_kernel(const KvCache c, const Params p)
{
    __shared__ float weight[MAX_WORKERS];
    __shared__ float red[D / 32], red2[D / 32];
    const uint32_t hr = c.kv_heads * p.row_blocks;
    const uint32_t pair = blockIdx.x, r = blockIdx.y;
    const uint32_t b = pair / hr, pr = pair - b * hr, head = pr / p.row_blocks, rb = pr - head * p.row_blocks;
    const int32_t q0 = __ldg(p.q_start + b);
    const KvSequence s = kv_sequence(q0, __ldg(p.q_start + b + 1), __ldg(p.kv_len + b), p.tokens, p.max_new, p.room);
    const uint32_t row = rb * ROWS + r;
    if (row >= s.new_tokens * p.group)
        return;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t first = p.meta[2 * pair], n = p.meta[2 * pair + 1] - first + 1;
    if (n == 1)
        return;
    // part 0 is the first worker's last, the others are their workers' first
    auto slot = [&](uint32_t i) { return (size_t)(2 * (first + i) + (i == 0 ? 1u : 0u)) * p.part_rows + r; };
    float top = -INFINITY;
    for (uint32_t i = threadIdx.x; i < n; i += D)
        top = fmaxf(top, p.part_ml[slot(i) * 2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0)
        red[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        top = fmaxf(top, red[i]);
    const float base = top == -INFINITY ? 0.0f : top;
    float l = 0.0f;
    for (uint32_t i = threadIdx.x; i < n; i += D) {
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot(i) * 2);
        const float w = ex2(ml.x - base);
        weight[i] = w;
        l = fmaf(w, ml.y, l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        l += __shfl_xor_sync(0xffffffffu, l, o);
    if ((threadIdx.x & 31) == 0)
        red2[threadIdx.x >> 5] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        l += red2[i];
    float acc = 0.0f;
#pragma unroll 8
    for (uint32_t i = 0; i < n; ++i)
        acc = fmaf(weight[i], p.part_o[slot(i) * D + threadIdx.x], acc);
    const uint32_t i = row / p.group;
    p.out[((size_t)((uint32_t)q0 + i) * p.heads + head * p.group + row - i * p.group) * D + threadIdx.x] =
        __float2half_rn(l == 0.0f ? 0.0f : acc / l);
}

struct Layout {
    uint32_t row_blocks, part_rows;
    size_t part_o, part_ml, meta, floats;  // offsets and the whole length, in floats
};

static Layout layout(uint32_t batch, uint32_t max_new, uint32_t heads, uint32_t kv_heads, uint32_t head_dim)
{
    const uint32_t rows = max_new * (heads / kv_heads);
    Layout a;
    a.row_blocks = (rows + ROWS - 1) / ROWS;
    a.part_rows = rows < ROWS ? rows : ROWS;
    const size_t slots = 2 * MAX_WORKERS;
    a.part_o = 0;
    a.part_ml = slots * a.part_rows * head_dim;
    a.meta = a.part_ml + (slots * a.part_rows * 2 + 3) / 4 * 4;
    a.floats = a.meta + (size_t)batch * kv_heads * a.row_blocks * 2;
    return a;
}

template <int D>
static cudaError_t launch(const DeviceCtx& ctx, const KvCache& c, const Params& p, const CUtensorMap& km,
                          const CUtensorMap& vm, bool half, cudaStream_t stream)
{
    using S = Shape<D>;
    auto kernel = half ? attention_paged_decode_kernel<D, true> : attention_paged_decode_kernel<D, false>;
    static bool set[64][2] = {};
    if (!set[ctx.device][half]) {
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
        if (err != cudaSuccess)
            return err;
        set[ctx.device][half] = true;
    }
    const uint32_t sms = (uint32_t)ctx.num_sms < MAX_SMS ? (uint32_t)ctx.num_sms : MAX_SMS;
    kernel<<<sms * CTAS_PER_SM, WARPS * 32, S::SMEM, stream>>>(km, vm, c, p);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess)
        return err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c.batch * c.kv_heads * p.row_blocks, p.part_rows);
    cfg.blockDim = dim3(D);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attention_paged_combine_kernel<D>, c, p);
}

}  // namespace apdec

bool attention_paged_decode_ok(uint32_t batch, uint32_t max_new, uint32_t heads, uint32_t kv_heads)
{
    const uint64_t rows = (uint64_t)max_new * (heads / kv_heads);
    return rows <= 32 && (uint64_t)batch * kv_heads * ((rows + 15) / 16) <= 0x7fffffffu;
}

size_t attention_paged_decode_scratch(uint32_t batch, uint32_t max_new, uint32_t heads, uint32_t kv_heads,
                                      uint32_t head_dim)
{
    return apdec::layout(batch, max_new, heads, kv_heads, head_dim).floats;
}

cudaError_t launch_attention_paged_decode(const DeviceCtx& ctx, const KvParams& kp, const __half* q, __half* out,
                                          uint32_t q_stride, uint32_t max_new, bool causal, float* scratch,
                                          cudaStream_t stream)
{
    using namespace apdec;
    const KvCache c = kv_cache_of(ctx, kp);
    const Layout a = layout(kp.batch, max_new, kp.heads, kp.kv_heads, kp.head_dim);
    Params p = {};
    p.q = q;
    p.out = out;
    p.q_start = kp.start;
    p.kv_len = kp.kv_len;
    p.part_o = scratch + a.part_o;
    p.part_ml = scratch + a.part_ml;
    p.meta = reinterpret_cast<uint32_t*>(scratch + a.meta);
    p.tokens = kp.rows;
    p.heads = kp.heads;
    p.group = kp.heads / kp.kv_heads;
    p.q_stride = q_stride;
    p.max_new = max_new;
    p.room = kp.max_pages * kp.page_size;
    p.row_blocks = a.row_blocks;
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
    const bool half = a.part_rows <= 8;
    return kp.head_dim == 128 ? launch<128>(ctx, c, p, km, vm, half, stream) : launch<64>(ctx, c, p, km, vm, half, stream);
}

}  // namespace kaio
