// Attention of chunks of new tokens (prompts, parts of prompts) over the paged 8-bit cache on the 5th-generation tensor
// cores.  The mathematics is that of attention_paged_decode.cu: integer keys and values as exact f16 operands, both
// scales, constant over 16 keys, applied to the scores (the values' as log2 in the exponent):
//   x_j = (q . kint_j) ck + lv,  ck = ks log2(e) / sqrt(d),  lv = log2(vs);  P_j = 2^(x_j - ref);
//   O = sum_j P_j vint_j,  l = sum_j P_j / vs_j,  out = O / l.
//
// An item = 256 rows of (sequence, key/value head): new token x query head of the group, so that a group's heads share
// every converted key and value.  16 warps, one CTA per SM, which stays: the items are the blocks of the grid, a sequence's
// heaviest first, and a CTA that is at work takes over blocks that have not started (clusterlaunchcontrol), so that tensor memory
// and barriers are set up once, and keys, values and Q of the next item arrive beside the softmax and the output of the
// last one.
//   warp 0       issues the MMAs, for row tiles t in {0, 1} of 128 rows:  S_t = Q_t K_j^T (tcgen05.mma kind::f16
//                M128 N128 K16, both from shared memory), O_t += P_t V_j (P_t from tensor memory); PV_t(j), QK_t(j+1) in
//                turn, so that one tile's softmax runs beside the other's products
//   warp 1       items; looks up pages and fetches their rows by TMA, 16 a box, a block of K and one of V ahead
//   warps 2, 3   fetch Q (cp.async into the MMAs' swizzle)
//   warps 4-11   softmax of tile 0 / 1, thread = row: the score row in registers, block maxima scaled by the block's
//                constants, lazy rescale (P may grow to 2^15), P packed to f16 in tensor memory in two halves
//   warps 13-15  s8 -> f16, stored in the 128-byte swizzle that the MMAs read; two stages each of K and V; the blocks'
//                constants go to a ring of four beside them.  None of them is on the MMA warp's scheduler, whose chain of
//                waits is the longest of all (warp 12, which would be, rests: 198 -> 174 us for the chunk below)
// An item of one tile's rows (the last of a sequence, short chunks, drafted tokens) gives both tiles its keys in turn and adds
// the two sums at the end, so that two chains of softmax and products run all the same.  A call that has no others (SHORT) is
// bound by the conversion, of a block of keys for one tile: warp 12 takes part there, and the place of the second tile's Q
// holds a second stage of raw bytes.  64 sequences of 4000 tokens, 8 key heads, 32 rows: 355 us with one tile at work, 277 with
// two, 241 with the raw stage and without masks for rows that are not there, 212 with the fourth warp.
// Registers are moved from the first and last four warps to the softmax ones (setmaxnreg: 72 + 2 x 168 + 104 = 4 x 128);
// ptxas still spills 28 to 52 bytes a thread.
// Few items: the keys of an item are cut over several CTAs, whose (O, ref, l) a second launch adds in ascending order.
// Q comes by TMA where a group's heads divide a tile's 128 rows, else row by row (154 -> 150 us for the prompts below).
//
// What bounds it: the chain S -> softmax -> P -> O of a block, 4000 cycles for both tiles where the products need 2400 on the
// tensor pipe and the exponentials 2048 on MUFU.  Measured at head size 128: 512 tokens behind 8192 cached ones, 64 query
// heads over 8, 173 us = 0.82 PFLOP/s (128 items of equal weight, one round on 128 of 148 SMs); four ragged prompts of up to
// 2048 tokens, 32 heads, 151 us = 0.51 PFLOP/s (half of every diagonal block is masked, and a mixed call's other launches take
// 9 us of it).
#include "kernels.h"
#include "kv_cache.cuh"
#include "softmax_tile.cuh"

#include <type_traits>

namespace kaio {
namespace apchunk {

constexpr uint32_t BQ = 128;    // rows of a tile (two tiles per item)
constexpr uint32_t BKV = 128;   // keys of a block
constexpr uint32_t STAGES = 2;  // of K and of V
constexpr uint32_t Q_SUB = 128 * 128;  // one [128 rows][64 f16] sub-tile
constexpr uint32_t KV_SUB = BKV * 128;
constexpr int NUM_THREADS = 512;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t TMEM_S = 0;    // per tile: 128 columns of f32 scores; P (f16 pairs) reuses the first 64
constexpr uint32_t TMEM_O = 256;  // per tile: 128 columns (f32 output accumulator)
constexpr float RESCALE_WINDOW = 15.0f;  // P = 2^(x - ref) may reach f16's 2^15 before O and l are rescaled
constexpr uint32_t TARGET_CTAS = 148;  // SMs of a B200: how many CTAs a call with few items is cut into
constexpr uint32_t MAX_SPLITS = 32;
constexpr uint32_t CONST_RING = 4;
constexpr uint32_t ITEM_RING = 2;
constexpr uint32_t NO_ITEM = 0xffffffffu;
// Cached tokens of a sequence: half a second for an item, and some roles wait from one item to the next (their waits give up
// after one).
constexpr uint32_t LONGEST = 1u << 25;

enum : uint32_t {
    SITE_Q_FULL = 1, SITE_K_FULL = 2, SITE_V_FULL = 3, SITE_K_EMPTY = 4, SITE_V_EMPTY = 5, SITE_S_FULL = 6,
    SITE_P_FULL = 7, SITE_PV_DONE = 8, SITE_Q_EMPTY = 9, SITE_ITEM_FULL = 10, SITE_ITEM_EMPTY = 11,
    SITE_RAW_FULL = 12, SITE_RAW_EMPTY = 13, SITE_DUAL = 14
};

// SHORT: no sequence of the call has more rows than a tile, so the second tile's place for Q goes to the raw bytes: a block's
// are then asked for while those of the block in front wait for the converting warps.
template <int D, bool SHORT>
struct Shape {
    static constexpr uint32_t Q_TILES = SHORT ? 1 : 2;
    static constexpr uint32_t CW = SHORT ? 4 : 3;  // converting warps, the last of the block
    static constexpr uint32_t READERS = 11 + CW;  // warps that take items: all but the one that hands them out and one that may rest
    static constexpr uint32_t RAW_STAGES = SHORT ? 256 / D : 128 / D;
    static constexpr uint32_t Q_BYTES = D / 64 * Q_SUB;    // 128 rows
    static constexpr uint32_t KV_BYTES = D / 64 * KV_SUB;  // a block of K or V
    static constexpr uint32_t K_OFF = Q_TILES * Q_BYTES, V_OFF = K_OFF + STAGES * KV_BYTES;
    static constexpr uint32_t BLOCK_BYTES = KV_BLOCK * D;  // 16 keys of K or V in 8 bits
    static constexpr uint32_t RAW_BYTES = BKV * D;         // a block of K or V in 8 bits
    static constexpr uint32_t RAW_OFF = V_OFF + STAGES * KV_BYTES, END = RAW_OFF + 2 * RAW_STAGES * RAW_BYTES;
    static constexpr uint32_t SMEM = 1024 + END;
    static_assert(RAW_STAGES <= CONST_RING, "a block's ks waits in the ring of constants");
    static constexpr uint32_t IDESC_QK = make_idesc(1, 0, 0, /*a K-major*/ 0, /*b K-major*/ 0, BQ, BKV);
    static constexpr uint32_t IDESC_PV = make_idesc(1, 0, 0, /*a K-major*/ 0, /*b MN-major*/ 1, BQ, D);
};

struct Params {
    const __half* q;
    __half* out;
    const int32_t *q_start, *kv_len;
    float *part_o, *part_ml;  // [splits][tokens * heads][D], [splits][tokens * heads][2]
    uint32_t tokens, heads, group, q_stride, max_new, room, items, splits;
    uint32_t least_new;  // sequences with fewer new tokens are another kernel's,
    int beside;          // which was launched in front and may still be running
    float scale_log2;
    int causal;
    int q_boxes;  // Q by TMA
};

// A value that all lanes of the warp have anyway, in a form the compiler knows it by: the MMAs' addresses are then kept in
// uniform registers from the start, instead of being moved there in front of every MMA.
__device__ __forceinline__ uint32_t uniform(uint32_t v)
{
    return __reduce_max_sync(0xffffffffu, v);
}

template <uint32_t N>
__device__ __forceinline__ void regs_up()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <uint32_t N>
__device__ __forceinline__ void regs_down()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

// One item: its sequence and rows, and what this CTA has of its keys, the blocks [j0, j0 + n).  Of those tile t has the
// first n_t, or, in an item of one tile's rows (dual), every second one from block t on: both tiles are then of the same rows.
struct Item {
    KvSequence s;
    uint32_t b, q0, head, split, row0, rows;
    uint32_t n0, n1, n, j0, dual;
};

// false: block x of the grid stands for nothing.  Made by one warp and handed to the others in shared memory: the search, the
// loads and the divisions are 300 instructions, and every role would stand still for them between two items.
__device__ __forceinline__ bool make_item(const KvCache& c, const Params& p, uint32_t x, Item& im)
{
    im.split = x % p.splits;
    const uint32_t rest = x / p.splits;
    im.head = rest % c.kv_heads;
    // from the last item down: a sequence's last rows see the most keys (of several sequences the last comes first)
    uint32_t local;
    im.b = kv_find_sequence<8, 1>(p.q_start, c.batch, p.group, p.items - 1 - rest / c.kv_heads, &local);
    im.q0 = (uint32_t)kv_load(p.q_start + im.b);
    const uint32_t q1 = (uint32_t)kv_load(p.q_start + im.b + 1);
    im.s = kv_sequence((int32_t)im.q0, (int32_t)q1, kv_load(p.kv_len + im.b), p.tokens, p.max_new, p.room);
    // a sequence of the other kernel's is that one's to report: it may have more tokens than this one takes
    if (im.s.bad && !(p.beside && q1 - im.q0 < p.least_new))
        kv_report(c, im.s.bad, KERNEL_ATTN_PAGED);
    im.rows = im.s.new_tokens < p.least_new ? 0 : im.s.new_tokens * p.group;
    if ((uint64_t)local * 2 * BQ >= im.rows)
        return false;
    im.row0 = local * 2 * BQ;
    // key blocks of a tile: what its last row sees
    auto blocks = [&](uint32_t first) -> uint32_t {
        if (first >= im.rows)
            return 0;
        const uint32_t last = (first + BQ < im.rows ? first + BQ : im.rows) - 1;
        return (kv_visible(im.s, last / p.group, p.causal != 0) + BKV - 1) / BKV;
    };
    const uint32_t all0 = blocks(im.row0), all1 = blocks(im.row0 + BQ), all = all0 > all1 ? all0 : all1;
    im.j0 = (uint32_t)((uint64_t)all * im.split / p.splits);
    const uint32_t j1 = (uint32_t)((uint64_t)all * (im.split + 1) / p.splits);
    const uint32_t e0 = all0 < j1 ? all0 : j1, e1 = all1 < j1 ? all1 : j1;
    im.n0 = e0 > im.j0 ? e0 - im.j0 : 0;
    im.n1 = e1 > im.j0 ? e1 - im.j0 : 0;
    im.n = im.n0 > im.n1 ? im.n0 : im.n1;
    im.dual = im.row0 + BQ >= im.rows && im.n > 1 ? 1 : 0;
    if (im.dual) {
        im.n0 = (im.n + 1) / 2;
        im.n1 = im.n / 2;
    }
    return true;
}

// Asks the hardware for a block of this grid that has not started; the 16-byte answer arrives on `bar`.
__device__ __forceinline__ void ask_for_block(uint32_t answer, uint32_t bar)
{
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     answer), "r"(bar) : "memory");
}

// The block that an answer gives, NO_ITEM when there was none left.
__device__ __forceinline__ uint32_t block_of(uint32_t answer)
{
    uint32_t x;
    asm volatile(
        "{\n"
        ".reg .b128 h;\n"
        ".reg .pred p;\n"
        "ld.shared.b128 h, [%1];\n"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
        "mov.u32 %0, %2;\n"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n"
        "}\n"
        : "=r"(x)
        : "r"(answer), "n"(NO_ITEM)
        : "memory");
    return x;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <int D, bool SHORT>
__global__ void __launch_bounds__(NUM_THREADS, 1)
attention_paged_chunk_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                             const __grid_constant__ CUtensorMap v_map, const KvCache c, const Params p)
{
    using S = Shape<D, SHORT>;
    constexpr uint32_t RS = S::RAW_STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 + 4 * STAGES + 15 + 4 * RS];
    __shared__ float2 dual_ml[BQ];  // ref and l of a dual item's tile 1
    __shared__ float4 consts[CONST_RING][BKV / KV_BLOCK];  // ck, lv, 1 / vs of a block of 16 keys; in front of that, .w is its ks
    __shared__ float raw_vs[RS][BKV / KV_BLOCK];
    __shared__ uint32_t raw_valid[RS];  // a bit for each block of 16 that is there
    __shared__ alignas(16) uint8_t answer[16];
    __shared__ Item items[ITEM_RING];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t abort_flag;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto bar = [&](uint32_t i) { return smem_u32(&bars[i]); };
    const uint32_t q_full = bar(0), q_empty = bar(1);
    auto k_full = [&](uint32_t g) { return bar(2 + g % STAGES); };
    auto k_empty = [&](uint32_t g) { return bar(2 + STAGES + g % STAGES); };
    auto v_full = [&](uint32_t g) { return bar(2 + 2 * STAGES + g % STAGES); };
    auto v_empty = [&](uint32_t g) { return bar(2 + 3 * STAGES + g % STAGES); };
    auto use = [](uint32_t g) { return g / STAGES & 1u; };  // parity of a stage's use by block g
    constexpr uint32_t REST = 2 + 4 * STAGES;
    auto s_full = [&](uint32_t t) { return bar(REST + t); };
    auto p_lo = [&](uint32_t t) { return bar(REST + 2 + t); };  // P of keys 0-63 stored
    auto p_hi = [&](uint32_t t) { return bar(REST + 4 + t); };  // P of keys 64-127 stored
    auto pv_done = [&](uint32_t t) { return bar(REST + 6 + t); };
    auto item_full = [&](uint32_t s) { return bar(REST + 8 + s); };
    auto item_empty = [&](uint32_t s) { return bar(REST + 10 + s); };
    const uint32_t answer_full = bar(REST + 12);
    const uint32_t dual_full = bar(REST + 13), dual_empty = bar(REST + 14);  // O_1, ref and l of tile 1 for tile 0's warps
    auto raw_full = [&](uint32_t v, uint32_t g) { return bar(REST + 15 + v * RS + g % RS); };  // of K (0) and of V (1)
    auto raw_empty = [&](uint32_t v, uint32_t g) { return bar(REST + 15 + (2 + v) * RS + g % RS); };
    auto raw_use = [](uint32_t g) { return g / RS & 1u; };

    if (threadIdx.x == 0) {
        mbar_init(q_full, p.q_boxes ? 1 : 2);
        mbar_init(q_empty, 1);
        for (uint32_t i = 0; i < STAGES; ++i) {
            mbar_init(k_full(i), S::CW);
            mbar_init(k_empty(i), 1);
            mbar_init(v_full(i), S::CW);
            mbar_init(v_empty(i), 1);
        }
        for (uint32_t i = 0; i < RS; ++i) {
            mbar_init(raw_full(0, i), 1 + 16);  // the bytes' arrive and the lanes that fetch scales
            mbar_init(raw_full(1, i), 1);
            mbar_init(raw_empty(0, i), S::CW);
            mbar_init(raw_empty(1, i), S::CW);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(s_full(i), 1);
            mbar_init(p_lo(i), 4);
            mbar_init(p_hi(i), 4);
            mbar_init(pv_done(i), 1);
            mbar_init(item_full(i), 1);
            mbar_init(item_empty(i), S::READERS);
        }
        mbar_init(answer_full, 1);
        mbar_init(dual_full, 4);
        mbar_init(dual_empty, 4);
        abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0) {
        tmem_alloc<TMEM_COLS>(smem_u32(&tmem_slot));
        tmem_relinquish();
    }
    if (!p.beside)
        asm volatile("griddepcontrol.wait;" ::: "memory");
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *const_cast<volatile uint32_t*>(&tmem_slot);

    // The next item for a warp that takes them in order; false: there is none.
    uint32_t taken = 0;
    auto next_item = [&](Item& im) {
        const uint32_t slot = taken % ITEM_RING, use_of = taken / ITEM_RING & 1u;
        ++taken;
        if (!mbar_wait_bounded(item_full(slot), use_of, &abort_flag, c.status, SITE_ITEM_FULL, KERNEL_ATTN_PAGED))
            return false;
        im = items[slot];
        __syncwarp();
        if (lane == 0)
            mbar_arrive(item_empty(slot));
        return im.rows != 0;
    };

    if (warp < 4) {
        regs_down<72>();
        if (warp == 0) {
            // ------------------------------------------------------------ MMA issuer
            uint32_t gave_up = 0;  // site of a wait that did
            auto wait = [&](uint32_t bar_addr, uint32_t parity, uint32_t site) {
                const bool ok = mbar_wait_light(bar_addr, parity, &abort_flag);
                tc_fence_after_sync();
                gave_up = ok ? gave_up : site;
                return ok;
            };
            const uint32_t tmem = uniform(tmem_base), smem = uniform(smem_base);
            uint32_t g0 = 0;            // key blocks of the items before: a block's number selects its stage
            uint32_t done[2] = {0, 0};  // blocks each tile's softmax has handed over
            uint32_t q_items = 0;
            bool ok = true;
            for (Item im; ok && next_item(im);) {
                const uint32_t n0 = uniform(im.n0), n1 = uniform(im.n1), n = uniform(im.n), dual = uniform(im.dual);
                if (n == 0)
                    continue;
                // as_dual: std::true_type in a dual item (the two forms have code of their own, this warp is the slowest)
                auto issue_qk = [&](auto as_dual, uint32_t t, uint32_t j) {
                    constexpr bool DUAL = decltype(as_dual)::value;
                    const uint32_t k = smem + S::K_OFF + (g0 + j) % STAGES * S::KV_BYTES;
                    const uint32_t q = smem + (DUAL ? 0 : t * S::Q_BYTES);
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t kk = 0; kk < D / 16; ++kk) {
                            const uint32_t off = (kk >> 2) * Q_SUB + (kk & 3u) * 32;
                            umma_f16(tmem + TMEM_S + t * BKV, make_smem_desc_sw128(q + off, 16, 1024),
                                     make_smem_desc_sw128(k + off, 16, 1024), S::IDESC_QK, kk != 0 ? 1u : 0u);
                        }
                        umma_commit(s_full(t));
                        if (DUAL || t == 1 || j >= n1) {
                            umma_commit(k_empty(g0 + j));  // the last reader of this K
                            if (j + 1 == n)
                                umma_commit(q_empty);  // and of Q
                        }
                    }
                    __syncwarp();
                };
                auto issue_pv = [&](auto as_dual, uint32_t t, uint32_t j, uint32_t k0) {
                    constexpr bool DUAL = decltype(as_dual)::value;
                    const uint32_t v = smem + S::V_OFF + (g0 + j) % STAGES * S::KV_BYTES;
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t kk = k0; kk < k0 + BKV / 32; ++kk)
                            umma_f16_ts(tmem + TMEM_O + t * 128, tmem + TMEM_S + t * BKV + kk * 8,
                                        make_smem_desc_sw128(v + kk * 2048, KV_SUB, 1024), S::IDESC_PV,
                                        ((DUAL ? j >> 1 : j) | kk) != 0 ? 1u : 0u);
                        if (k0) {
                            umma_commit(pv_done(t));
                            if (DUAL || t == 1 || j >= n1)
                                umma_commit(v_empty(g0 + j));
                        }
                    }
                    __syncwarp();
                };
                ok = wait(q_full, q_items++ & 1u, SITE_Q_FULL) && wait(k_full(g0), use(g0), SITE_K_FULL);
                if (dual) {
                    if (ok)
                        issue_qk(std::true_type(), 0, 0);
                    ok = ok && wait(k_full(g0 + 1), use(g0 + 1), SITE_K_FULL);
                    if (ok)
                        issue_qk(std::true_type(), 1, 1);
                    for (uint32_t j = 0; ok && j < n; ++j) {
                        const uint32_t t = j & 1u, g = g0 + j, parity = (t ? done[1] : done[0]) & 1u;
                        ok = wait(v_full(g), use(g), SITE_V_FULL) && wait(p_lo(t), parity, SITE_P_FULL);
                        if (ok)
                            issue_pv(std::true_type(), t, j, 0);
                        ok = ok && wait(p_hi(t), parity, SITE_P_FULL);
                        if (ok)
                            issue_pv(std::true_type(), t, j, BKV / 32);
                        done[0] += t ^ 1u;
                        done[1] += t;
                        if (ok && j + 2 < n) {
                            ok = wait(k_full(g + 2), use(g + 2), SITE_K_FULL);
                            if (ok)
                                issue_qk(std::true_type(), t, j + 2);
                        }
                    }
                    g0 += n;
                    continue;
                }
                if (ok) {
                    if (n0 > 0)
                        issue_qk(std::false_type(), 0, 0);
                    if (n1 > 0)
                        issue_qk(std::false_type(), 1, 0);
                }
                for (uint32_t j = 0; ok && j < n; ++j) {
                    const uint32_t g = g0 + j;
                    bool v_ready = false, k_ready = false;
#pragma unroll
                    for (uint32_t t = 0; t < 2; ++t) {
                        const uint32_t nt = t ? n1 : n0;
                        if (ok && j < nt) {
                            if (!v_ready)
                                ok = v_ready = wait(v_full(g), use(g), SITE_V_FULL);
                            ok = ok && wait(p_lo(t), done[t] & 1u, SITE_P_FULL);
                            if (ok)
                                issue_pv(std::false_type(), t, j, 0);
                            ok = ok && wait(p_hi(t), done[t] & 1u, SITE_P_FULL);
                            if (ok)
                                issue_pv(std::false_type(), t, j, BKV / 32);
                            ++done[t];
                        }
                        if (ok && j + 1 < nt) {
                            // behind its P V, so that the other tile's softmax overlaps it; in-order execution on the
                            // tensor pipe makes the overwrite of P_t by S_t safe
                            if (!k_ready)
                                ok = k_ready = wait(k_full(g + 1), use(g + 1), SITE_K_FULL);
                            if (ok)
                                issue_qk(std::false_type(), t, j + 1);
                        }
                    }
                }
                g0 += n;
            }
            if (gave_up)
                report_wait(&abort_flag, c.status, gave_up, KERNEL_ATTN_PAGED);
        } else if (warp == 1) {
            // ------------------------------------------------------------ items, pages, rows
            // lane i has the 16 tokens i % 8 of a block, K in lanes 0-7 and V in lanes 8-15
            uint32_t g = 0;
            bool ok = true;
            uint32_t asked = 0, given = 0;
            // the last item is followed by one without rows
            auto give = [&](const Item& im) {
                const uint32_t slot = given % ITEM_RING, use_of = given / ITEM_RING & 1u;
                ++given;
                if (!mbar_wait_bounded(item_empty(slot), use_of ^ 1u, &abort_flag, c.status, SITE_ITEM_EMPTY, KERNEL_ATTN_PAGED))
                    return false;
                if (lane == 0) {
                    items[slot] = im;
                    mbar_arrive(item_full(slot));
                }
                __syncwarp();
                return true;
            };
            for (uint32_t x = blockIdx.x;;) {
                Item im;
                if (x == NO_ITEM) {
                    im.rows = 0;
                    give(im);
                    break;
                }
                const bool valid = make_item(c, p, x, im);
                if (valid)
                    ok = give(im);
                auto find = [&](uint32_t j) {
                    const uint32_t pos = (im.j0 + j) * BKV + (lane & 7u) * KV_BLOCK;
                    return lane < 16 && j < im.n && pos < im.s.kv ? kv_page(c, im.b, pos, KERNEL_ATTN_PAGED) : KV_NO_PAGE;
                };
                uint32_t page = valid ? find(0) : KV_NO_PAGE;
                for (uint32_t j = 0; ok && valid && j < im.n; ++j, ++g) {
                    const bool there = page != KV_NO_PAGE;
                    const uint32_t mask = __ballot_sync(0xffffffffu, there) & 0xffu;
                    const size_t row = there ? kv_row(c, page, im.head, (im.j0 + j) * BKV + (lane & 7u) * KV_BLOCK) : 0;
                    page = find(j + 1);
#pragma unroll
                    for (uint32_t v = 0; v < 2; ++v) {
                        ok = ok && mbar_wait_bounded(raw_empty(v, g), raw_use(g) ^ 1u, &abort_flag, c.status, SITE_RAW_EMPTY, KERNEL_ATTN_PAGED);
                        if (!ok)
                            break;
                        if (lane == 0) {
                            if (v == 0)
                                raw_valid[g % RS] = mask;
                            mbar_expect_tx(raw_full(v, g), __popc(mask) * S::BLOCK_BYTES);
                        }
                        __syncwarp();
                        if (lane < 16) {
                            if (there && lane >> 3 == v)
                                tma_load_2d(smem_base + S::RAW_OFF + g % RS * 2 * S::RAW_BYTES + lane * S::BLOCK_BYTES,
                                            v ? &v_map : &k_map, raw_full(v, g), 0, (int32_t)row);
                            if (v == 0) {
                                if (there)
                                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(lane < 8 ? &consts[g & (CONST_RING - 1)][lane].w : &raw_vs[g % RS][lane - 8])),
                                                 "l"((lane < 8 ? c.ks : c.vs) + row / KV_BLOCK) : "memory");
                                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(raw_full(0, g)) : "memory");
                            }
                        }
                        __syncwarp();
                    }
                }
                if (!ok)
                    break;
                // Asked for only now, a few blocks before the MMAs are done with this one: what a CTA has claimed no other
                // can take.
                if (lane == 0) {
                    mbar_expect_tx(answer_full, 16);
                    ask_for_block(smem_u32(answer), answer_full);
                }
                __syncwarp();
                if (!mbar_wait_bounded(answer_full, asked++ & 1u, &abort_flag, c.status, SITE_ITEM_FULL, KERNEL_ATTN_PAGED))
                    break;
                x = block_of(smem_u32(answer));
                fence_proxy_async_smem();  // read before the next answer is written there
                __syncwarp();
            }
            if (abort_flag)
                for (uint32_t spin = 0; spin < 2000; ++spin)
                    __nanosleep(100);  // what is in flight lands before the shared memory is given up
        } else {
            // ------------------------------------------------------------ Q
            constexpr uint32_t TPR = D / 8;             // threads of a row, 16 bytes each
            constexpr uint32_t STRIDE = 64 / TPR;       // rows of a step
            const uint32_t tid = threadIdx.x - 64, ch = tid % TPR;
            const uint32_t step_tok = STRIDE / p.group, step_head = STRIDE % p.group;
            uint32_t q_items = 0;
            // A group whose heads divide a tile's 128 rows: whole tokens to a tile, one box for 64 of its dims (rows past the
            // sequence's are its neighbour's; no row of the products looks at another).  Other groups row by row.
            if (p.q_boxes) {
                for (Item im; next_item(im);) {
                    if (im.n == 0 || warp == 3)
                        continue;
                    if (!mbar_wait_bounded(q_empty, (q_items++ & 1u) ^ 1u, &abort_flag, c.status, SITE_Q_EMPTY, KERNEL_ATTN_PAGED))
                        break;
                    if (lane == 0) {
                        const uint32_t tiles = im.n1 && !im.dual ? 2 : 1;
                        mbar_expect_tx(q_full, tiles * S::Q_BYTES);
                        for (uint32_t t = 0; t < tiles; ++t)
#pragma unroll
                            for (uint32_t s = 0; s < D / 64; ++s)
                                tma_load_3d(smem_base + t * S::Q_BYTES + s * Q_SUB, &q_map, q_full, s * 64, im.head * p.group,
                                            im.q0 + (im.row0 + t * BQ) / p.group);
                    }
                    __syncwarp();
                }
            }
            for (Item im; !p.q_boxes && next_item(im);) {
                if (im.n == 0)
                    continue;
                if (!mbar_wait_bounded(q_empty, (q_items & 1u) ^ 1u, &abort_flag, c.status, SITE_Q_EMPTY, KERNEL_ATTN_PAGED))
                    break;
                ++q_items;
                uint32_t r = tid / TPR, row = im.row0 + r;
                uint32_t tok = row / p.group, h = row - tok * p.group;
                const __half* src = p.q + (size_t)im.head * p.group * D + ch * 8;
                const uint32_t dst = smem_base + (ch >> 3) * Q_SUB;
#pragma unroll 4
                for (; r < S::Q_TILES * BQ; r += STRIDE) {
                    const bool there = im.row0 + r < im.rows;  // the others are zeros
                    cp_async16(dst + (r / BQ) * S::Q_BYTES + sw128_offset(r % BQ, ch & 7u),
                               there ? src + (size_t)(im.q0 + tok) * p.q_stride + h * D : p.q, there ? 16 : 0);
                    tok += step_tok;
                    h += step_head;
                    if (h >= p.group) {
                        h -= p.group;
                        ++tok;
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(q_full);
            }
        }
    } else if (warp < 12) {
        regs_up<168>();
        // ------------------------------------------------------------ softmax, output
        const uint32_t t = (warp - 4) >> 2, quarter = warp & 3u;
        const uint32_t lane_sel = (quarter * 32u) << 16;
        const uint32_t s_tmem = tmem_base + TMEM_S + t * BKV + lane_sel;
        const uint32_t o_tmem = tmem_base + TMEM_O + t * 128 + lane_sel;
        uint32_t g0 = 0, cnt = 0;  // key blocks of the items before, blocks of this tile
        uint32_t duals = 0;
        bool ok = true;
        for (Item im; ok && next_item(im);) {
            const uint32_t n_t = t ? im.n1 : im.n0;
            const uint32_t row = im.row0 + (im.dual ? 0 : t * BQ) + quarter * 32 + lane;
            const uint32_t tok = row / p.group;
            const uint32_t seen = row < im.rows ? kv_visible(im.s, tok, p.causal != 0) : 0xffffffffu;  // no need to mask the others
            const uint32_t seen_least = __reduce_min_sync(0xffffffffu, seen);  // of the warp's rows
            float m_ref = -INFINITY, l_sum = 0.0f;
            const uint32_t first = im.dual ? t : 0, step = 1 + im.dual, end = im.dual ? im.n : n_t;
            for (uint32_t j = first; j < end; j += step, ++cnt) {
                if (!mbar_wait_bounded(s_full(t), cnt & 1u, &abort_flag, c.status, SITE_S_FULL, KERNEL_ATTN_PAGED)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const float4* cst = consts[(g0 + j) & (CONST_RING - 1)];
                const uint32_t col_base = (im.j0 + j) * BKV;
                uint32_t r[4][32];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    tmem_ld_32x32b_x32(s_tmem + 32 * k, r[k]);
                tmem_ld_wait();
                if (col_base + BKV > seen_least) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (col_base + 32 * k + i >= seen)
                                r[k][i] = 0xff800000u;  // -inf
                }
                // ---- maximum of each block of 16 keys, scaled (the scale is positive: scale after)
                float m_blk = -INFINITY;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t(&x)[32] = r[k >> 1];
                    const int at = (k & 1) * 16;
                    float m0 = __uint_as_float(x[at]), m1 = __uint_as_float(x[at + 1]);
#pragma unroll
                    for (int i = 2; i < 16; i += 4) {
                        m0 = max3_f32(m0, __uint_as_float(x[at + i]), __uint_as_float(x[at + i + 1]));
                        if (i + 2 < 16)
                            m1 = max3_f32(m1, __uint_as_float(x[at + i + 2]), __uint_as_float(x[at + i + 3]));
                    }
                    m_blk = fmaxf(m_blk, fmaf(fmaxf(m0, m1), cst[k].x, cst[k].y));
                }
                // ---- lazy rescale; the first block only sets the reference, KV_P_TOP below its maximum
                float alpha = 1.0f;
                bool rescale = false;
                if (j == first) {
                    m_ref = m_blk - KV_P_TOP;
                } else {
                    rescale = __any_sync(0xffffffffu, m_blk - m_ref > RESCALE_WINDOW);  // the sum would be rounded
                    const float next = m_blk - KV_P_TOP;
                    if (rescale && next > m_ref) {
                        alpha = ex2_approx(m_ref - next);
                        m_ref = next;
                        l_sum *= alpha;
                    }
                }
                const float base = m_ref == -INFINITY ? 0.0f : m_ref;
                // ---- P = 2^((x ck + lv) - ref), two per instruction; the sums of a block of 16 keys are divided by its vs.  Rounded as
                // the maximum was and only then subtracted from: x ck + (lv - ref) in one FMA would be off by up to a step of
                // ref, and from scores of 2^24 on P past f16's largest value.
                const uint64_t minus_base = pack_f32x2(-base, -base);
                auto exp_chunk = [&](const uint32_t (&x)[32], uint32_t k) {
                    uint32_t pk[16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float4 cc = cst[2 * k + h];
                        const uint64_t scale2 = pack_f32x2(cc.x, cc.x), lv2 = pack_f32x2(cc.y, cc.y);
                        uint64_t sa = 0, sb = 0;
#pragma unroll
                        for (int i = 16 * h; i < 16 * h + 16; i += 4) {
                            float x0, x1, x2, x3;
                            unpack_f32x2(add_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), scale2, lv2), minus_base), x0, x1);
                            unpack_f32x2(add_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), scale2, lv2), minus_base), x2, x3);
                            const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                            const float p2 = ex2_approx(x2), p3 = ex2_approx(x3);
                            sa = add_f32x2(sa, pack_f32x2(p0, p1));
                            sb = add_f32x2(sb, pack_f32x2(p2, p3));
                            const __half2 h01 = __floats2half2_rn(p0, p1);
                            const __half2 h23 = __floats2half2_rn(p2, p3);
                            pk[i >> 1] = *reinterpret_cast<const uint32_t*>(&h01);
                            pk[(i >> 1) + 1] = *reinterpret_cast<const uint32_t*>(&h23);
                        }
                        float a0, a1;
                        unpack_f32x2(add_f32x2(sa, sb), a0, a1);
                        l_sum = fmaf(a0 + a1, cc.z, l_sum);
                    }
                    tmem_st_32x32b_x16(s_tmem + k * 16, pk);
                };
                exp_chunk(r[0], 0);
                exp_chunk(r[1], 1);
                if (!rescale) {
                    // first half of P handed over: its P V steps run while the second half is computed
                    tmem_st_wait();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(p_lo(t));
                    // keep the second half's arithmetic behind the hand-over
#pragma unroll
                    for (int k = 2; k < 4; ++k)
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
                            asm volatile("" : "+r"(r[k][i]), "+r"(r[k][i + 1]), "+r"(r[k][i + 2]), "+r"(r[k][i + 3]),
                                              "+r"(r[k][i + 4]), "+r"(r[k][i + 5]), "+r"(r[k][i + 6]), "+r"(r[k][i + 7])
                                         :: "memory");
                }
                exp_chunk(r[2], 2);
                exp_chunk(r[3], 3);
                tmem_st_wait();
                if (rescale) {
                    // O_t (last written by the P V of block j - 1, complete since S_j was issued behind it) is scaled before any
                    // P V of this block may start, so this block hands both halves over at the end
                    if (!mbar_wait_bounded(pv_done(t), (cnt - 1) & 1u, &abort_flag, c.status, SITE_PV_DONE, KERNEL_ATTN_PAGED)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) {
                        tmem_ld_32x32b_x32(o_tmem + 32 * k, r[k]);
                    }
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            r[k][i] = __float_as_uint(__uint_as_float(r[k][i]) * alpha);
                        tmem_st_32x32b_x32(o_tmem + 32 * k, r[k]);
                    }
                    tmem_st_wait();
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (rescale)
                        mbar_arrive(p_lo(t));
                    mbar_arrive(p_hi(t));
                }
            }
            // ---- O / l, or this CTA's part of it
            if (ok && n_t > 0)
                ok = mbar_wait_bounded(pv_done(t), (cnt - 1) & 1u, &abort_flag, c.status, SITE_PV_DONE, KERNEL_ATTN_PAGED);
            float own = 1.0f, other = 0.0f;  // what O_0 and O_1 count of a dual item
            if (ok && im.dual) {
                if (t == 1) {
                    dual_ml[quarter * 32 + lane] = make_float2(m_ref, l_sum);
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(dual_full);
                    // O_1 may be written again once it has been read
                    ok = mbar_wait_bounded(dual_empty, duals++ & 1u, &abort_flag, c.status, SITE_DUAL, KERNEL_ATTN_PAGED);
                } else {
                    ok = mbar_wait_bounded(dual_full, duals++ & 1u, &abort_flag, c.status, SITE_DUAL, KERNEL_ATTN_PAGED);
                    const float2 ml = dual_ml[quarter * 32 + lane];
                    const float next = fmaxf(m_ref, ml.x), base = next == -INFINITY ? 0.0f : next;
                    own = ex2_approx(m_ref - base);
                    other = ex2_approx(ml.x - base);
                    m_ref = next;
                    l_sum = l_sum * own + ml.y * other;
                }
            }
            if (ok && !(im.dual && t == 1)) {
                tc_fence_after_sync();
                const float inv = l_sum == 0.0f ? 0.0f : 1.0f / l_sum;
                const size_t at = (size_t)(im.q0 + tok) * p.heads + im.head * p.group + row - tok * p.group;
#pragma unroll 1
                for (uint32_t k = 0; k < D / 32; ++k) {
                    uint32_t r[32];
                    if (n_t > 0) {
                        tmem_ld_32x32b_x32(o_tmem + k * 32, r);
                        tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            r[i] = 0;
                    }
                    if (im.dual) {
                        uint32_t r1[32];
                        tmem_ld_32x32b_x32(o_tmem + 128 + k * 32, r1);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            r[i] = __float_as_uint(__uint_as_float(r[i]) * own + __uint_as_float(r1[i]) * other);
                    }
                    if (row < im.rows) {
                        if (p.splits == 1) {
                            uint4* dst = reinterpret_cast<uint4*>(p.out + at * D + k * 32);
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                uint32_t h[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const __half2 v = __floats2half2_rn(__uint_as_float(r[i + 2 * e]) * inv, __uint_as_float(r[i + 2 * e + 1]) * inv);
                                    h[e] = *reinterpret_cast<const uint32_t*>(&v);
                                }
                                dst[i >> 3] = make_uint4(h[0], h[1], h[2], h[3]);
                            }
                        } else {
                            const size_t part = (size_t)im.split * p.tokens * p.heads + at;
                            uint4* dst = reinterpret_cast<uint4*>(p.part_o + part * D + k * 32);
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                dst[i >> 2] = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
                            if (k == 0)
                                *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(n_t > 0 ? m_ref : -INFINITY, l_sum);
                        }
                    }
                }
            }
            // O_t has been read before this warp arrives for the next item's first block
            tc_fence_before_sync();
            if (im.dual && t == 0) {
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(dual_empty);
            }
            g0 += im.n;
        }
    } else if (warp < 16 - S::CW) {
        regs_down<104>();
    } else {
        regs_down<104>();
        // ------------------------------------------------------------ K and V: s8 -> f16
        constexpr uint32_t CHUNKS = BKV * D / 512;  // of 32 x 16 bytes in a block of K or V
        constexpr uint32_t TPR = D / 16;            // threads of a row
        const uint32_t cw = warp - (16 - S::CW), c8 = lane % TPR, row = lane / TPR;
        // where the 16 values of this thread's chunk go: two 16-byte chunks of its f16 row.  At head size 128 the threads of
        // the second sub-tile store their odd chunk first, so that eight threads never meet in a bank.
        const bool swap = D == 128 && c8 >= 4;
        const uint32_t src = smem_base + S::RAW_OFF + lane * 16;
        const uint32_t dst = smem_base + (c8 >> 2) * KV_SUB;
        auto convert = [&](uint32_t from, uint32_t off) {
            constexpr uint32_t ROWS = 512 / D;  // of a chunk
            for (uint32_t i0 = cw; i0 < CHUNKS; i0 += 4 * S::CW) {
                uint4 w[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    if (i0 + S::CW * i < CHUNKS)
                        w[i] = lds128(src + from + (i0 + S::CW * i) * 512);
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (i0 + S::CW * i >= CHUNKS)
                        break;
                    const uint32_t r = (i0 + S::CW * i) * ROWS + row;
                    uint32_t h[8];
                    s8x4_to_f16(swap ? w[i].z : w[i].x, h[0], h[1]);
                    s8x4_to_f16(swap ? w[i].w : w[i].y, h[2], h[3]);
                    s8x4_to_f16(swap ? w[i].x : w[i].z, h[4], h[5]);
                    s8x4_to_f16(swap ? w[i].y : w[i].w, h[6], h[7]);
                    sts128(dst + off + sw128_offset(r, ((2 * c8) & 7u) + (swap ? 1 : 0)), h[0], h[1], h[2], h[3]);
                    sts128(dst + off + sw128_offset(r, ((2 * c8) & 7u) + (swap ? 0 : 1)), h[4], h[5], h[6], h[7]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
        };
        uint32_t g = 0;  // number of the key block: it selects the stages
        bool ok = true;
        for (Item im; ok && next_item(im);) {
            for (uint32_t j = 0; j < im.n; ++j, ++g) {
                const uint32_t parity = use(g) ^ 1u;
                ok = mbar_wait_bounded(raw_full(0, g), raw_use(g), &abort_flag, c.status, SITE_RAW_FULL, KERNEL_ATTN_PAGED) &&
                     mbar_wait_bounded(k_empty(g), parity, &abort_flag, c.status, SITE_K_EMPTY, KERNEL_ATTN_PAGED);
                if (!ok)
                    break;
                if (warp == 15 && lane < 8) {
                    // 16 tokens that are not there: every score of them is -inf.  The ring of four: this block's K is stored
                    // once block g - 2's has been read, by when the softmax has done with block g - 3.
                    float4& constant = consts[g & (CONST_RING - 1)][lane];
                    const float ks = fmaxf(constant.w, KV_SCALE_MIN), vs = fmaxf(raw_vs[g % RS][lane], KV_SCALE_MIN);
                    constant =
                        raw_valid[g % RS] >> lane & 1u ? make_float4(ks * p.scale_log2, __log2f(vs), __fdividef(1.0f, vs), 0.0f)
                                               : make_float4(1.0f, -INFINITY, 0.0f, 0.0f);
                }
                convert(g % RS * 2 * S::RAW_BYTES, S::K_OFF + g % STAGES * S::KV_BYTES);
                if (lane == 0) {
                    mbar_arrive(k_full(g));
                    mbar_arrive(raw_empty(0, g));
                }
                ok = mbar_wait_bounded(raw_full(1, g), raw_use(g), &abort_flag, c.status, SITE_RAW_FULL, KERNEL_ATTN_PAGED) &&
                     mbar_wait_bounded(v_empty(g), parity, &abort_flag, c.status, SITE_V_EMPTY, KERNEL_ATTN_PAGED);
                if (!ok)
                    break;
                convert((g % RS * 2 + 1) * S::RAW_BYTES, S::V_OFF + g % STAGES * S::KV_BYTES);
                if (lane == 0) {
                    mbar_arrive(v_full(g));
                    mbar_arrive(raw_empty(1, g));
                }
            }
        }
    }

    // ---------------------------------------------------------------- teardown
    if (p.beside)
        asm volatile("griddepcontrol.wait;" ::: "memory");  // what follows this launch follows that one too
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after_sync();
        tmem_dealloc<TMEM_COLS>(tmem_base);
    }
}

// Adds the parts of a token's rows: a warp has one query head, a lane D / 32 dims.
template <int D>
__global__ void __launch_bounds__(256) attention_paged_chunk_combine_kernel(const KvCache c, const Params p)
{
    constexpr int V = D / 32;
    const uint32_t lane = threadIdx.x & 31, token = blockIdx.x;
    kv_begin();
    uint32_t local;
    const uint32_t b = kv_find_sequence<0, 0>(p.q_start, c.batch, 1, token, &local);
    const int32_t q0 = kv_load(p.q_start + b);
    const KvSequence s = kv_sequence(q0, kv_load(p.q_start + b + 1), kv_load(p.kv_len + b), p.tokens, p.max_new, p.room);
    if (token - (uint32_t)q0 >= s.new_tokens || s.new_tokens < p.least_new)
        return;
    const uint32_t h = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (h < p.heads) {
        const size_t row = (size_t)token * p.heads + h, rows = (size_t)p.tokens * p.heads;
        float top = -INFINITY;
        for (uint32_t i = 0; i < p.splits; ++i)
            top = fmaxf(top, p.part_ml[(i * rows + row) * 2]);
        const float base = top == -INFINITY ? 0.0f : top;
        float l = 0.0f, acc[V];
#pragma unroll
        for (int e = 0; e < V; ++e)
            acc[e] = 0.0f;
#pragma unroll 4
        for (uint32_t i = 0; i < p.splits; ++i) {
            const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (i * rows + row) * 2);
            alignas(16) float v[V];
            if constexpr (V == 4)
                *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p.part_o + (i * rows + row) * D + lane * V);
            else
                *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(p.part_o + (i * rows + row) * D + lane * V);
            const float f = ex2_approx(ml.x - base);
            l = fmaf(f, ml.y, l);
#pragma unroll
            for (int e = 0; e < V; ++e)
                acc[e] = fmaf(f, v[e], acc[e]);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        __half* dst = p.out + row * D + lane * V;
#pragma unroll
        for (int e = 0; e < V; e += 2)
            *reinterpret_cast<__half2*>(dst + e) = __floats2half2_rn(acc[e] * inv, acc[e + 1] * inv);
    }
}

static uint64_t items_of(uint32_t batch, uint32_t tokens, uint32_t group)
{
    return (((uint64_t)tokens * group) >> 8) + batch;
}

// Few items: as many parts of each as bring the CTAs up to one per SM.
static uint32_t splits_of(uint32_t batch, uint32_t tokens, uint32_t heads, uint32_t kv_heads)
{
    const uint64_t ctas = items_of(batch, tokens, heads / kv_heads) * kv_heads;
    if (2 * ctas > TARGET_CTAS)
        return 1;
    const uint32_t s = (uint32_t)(TARGET_CTAS / ctas);
    return s < MAX_SPLITS ? s : MAX_SPLITS;
}

template <int D, bool SHORT>
static cudaError_t launch(const DeviceCtx& ctx, const KvCache& c, const Params& p, const CUtensorMap& qm,
                          const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t stream)
{
    using S = Shape<D, SHORT>;
    static bool set[64] = {};
    if (!set[ctx.device]) {
        const cudaError_t err = cudaFuncSetAttribute(attention_paged_chunk_kernel<D, SHORT>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
        if (err != cudaSuccess)
            return err;
        set[ctx.device] = true;
    }
    const cudaError_t err = kv_launch(attention_paged_chunk_kernel<D, SHORT>, dim3(p.items * c.kv_heads * p.splits), NUM_THREADS,
                                      S::SMEM, true, stream, qm, km, vm, c, p);
    if (err != cudaSuccess || p.splits == 1)
        return err;
    return kv_launch(attention_paged_chunk_combine_kernel<D>, dim3(p.tokens, (p.heads + 7) / 8), 256, 0, true, stream, c, p);
}

}  // namespace apchunk

bool attention_paged_chunk_ok(uint32_t batch, uint32_t tokens, uint32_t heads, uint32_t kv_heads)
{
    return apchunk::items_of(batch, tokens, heads / kv_heads) * kv_heads <= 0x7fffffffu;
}

size_t attention_paged_chunk_scratch(uint32_t batch, uint32_t tokens, uint32_t heads, uint32_t kv_heads,
                                     uint32_t head_dim)
{
    const uint32_t s = apchunk::splits_of(batch, tokens, heads, kv_heads);
    return s == 1 ? 0 : (size_t)s * tokens * heads * (head_dim + 2);
}

cudaError_t launch_attention_paged_chunk(const DeviceCtx& ctx, const KvParams& kp, const __half* q, __half* out,
                                         uint32_t q_stride, uint32_t max_new, uint32_t least_new, bool causal,
                                         bool beside, float* scratch, cudaStream_t stream)
{
    using namespace apchunk;
    const KvCache c = kv_cache_of(ctx, kp);
    Params p = {};
    p.q = q;
    p.out = out;
    p.q_start = kp.start;
    p.kv_len = kp.kv_len;
    p.tokens = kp.rows;
    p.heads = kp.heads;
    p.group = kp.heads / kp.kv_heads;
    p.q_stride = q_stride;
    p.max_new = max_new;
    p.least_new = least_new;
    p.beside = beside ? 1 : 0;
    p.room = kp.max_pages * kp.page_size < LONGEST ? kp.max_pages * kp.page_size : LONGEST;
    p.items = (uint32_t)items_of(kp.batch, kp.rows, p.group);
    p.splits = splits_of(kp.batch, kp.rows, kp.heads, kp.kv_heads);
    p.scale_log2 = 1.4426950408889634f / sqrtf((float)kp.head_dim);
    p.causal = causal ? 1 : 0;
    p.part_o = scratch;
    p.part_ml = scratch + (size_t)p.splits * kp.rows * kp.heads * kp.head_dim;
    CUtensorMap km, vm;
    const uint64_t rows = (uint64_t)kp.num_pages * kp.kv_heads * kp.page_size;
    cudaError_t err = encode_tensor_map_2d(&km, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, kp.k, kp.head_dim, rows, kp.head_dim,
                                           kp.head_dim, KV_BLOCK, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (err != cudaSuccess)
        return err;
    err = encode_tensor_map_2d(&vm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, kp.v, kp.head_dim, rows, kp.head_dim, kp.head_dim,
                               KV_BLOCK, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (err != cudaSuccess)
        return err;
    CUtensorMap qm = km;
    p.q_boxes = BQ % p.group == 0;
    if (p.q_boxes) {
        err = encode_tensor_map_3d_f16(&qm, q, {kp.head_dim, kp.heads, kp.rows}, {kp.head_dim * 2, (uint64_t)q_stride * 2},
                                       {64, p.group, BQ / p.group});
        if (err != cudaSuccess)
            return err;
    }
    if ((uint64_t)max_new * p.group <= BQ)
        return kp.head_dim == 128 ? launch<128, true>(ctx, c, p, qm, km, vm, stream) : launch<64, true>(ctx, c, p, qm, km, vm, stream);
    return kp.head_dim == 128 ? launch<128, false>(ctx, c, p, qm, km, vm, stream) : launch<64, false>(ctx, c, p, qm, km, vm, stream);
}

}  // namespace kaio
