// mx_tc.cu -- products with MX4 weights on the block-scaled tensor cores (include/unoq_mx.h).
//
// D[weight row][column] += sum over blocks b of 2^(sa + sb) * (codes of W) . (codes of X), tcgen05 with
// one scale per row and 32 values on both sides, accumulators in TMEM. The 128 weight rows of a tile
// are the M side whatever the number of tokens, so a single token streams the same weight tiles
// as a prompt does, and its column count N is the multiple of 8 that holds it. Two kinds:
//
//   KIND 4  kind::mxf4: both sides e2m1, 64 values per instruction, 256 to a stage.
//   KIND 8  kind::mxf8f6f4: weights e2m1 (TMA unpacks each 4-bit code to a byte of shared memory),
//           activations e4m3, 128 values to a stage. A 16-bit activation is not rounded to e4m3: it is
//           split into P pieces of four significant bits, x = 2^s (p0 + p1 / 16 + p2 / 256) (P = 2 holds
//           bf16's 8 bits, 3 f16's 11), each piece a column of its own whose block scale carries its
//           power of 16; the epilogue adds the P columns in 32 bits. Few tokens leave the columns unused
//           otherwise, and a 16-bit tensor-core product would need the weights expanded in registers.
//
// In either kind a stage is 128 weight rows of 128 bytes and N columns of 128 bytes in shared memory
// (SWIZZLE_128B) and takes four MMAs.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "device_state.hpp"
#include "mx.cuh"
#include "mx_mma.cuh"

namespace uq {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxStages = 16;
constexpr int kThreads = 224;      // warp 0: weight copies, warp 1: MMA, warps 2-5: epilogue, warp 6: activation copies
constexpr int kCtrlBytes = 1024;   // barriers, TMEM slot and, for the experts, the token list
constexpr int kItemWords = 2 + 32; // an item: expert, tokens, the pairs (a lane each)
// Most tokens of one expert that one CTA takes: two accumulators of 32 tokens' hidden pieces would fill its 256 columns
// of TMEM.
constexpr int kChunk = 24;
constexpr uint32_t kA = 16384;     // one weight tile in shared memory

__host__ __device__ constexpr uint32_t up_to(uint32_t v, uint32_t to) { return (v + to - 1) / to * to; }

enum Mode { kDense = 0, kGateUp = 1, kDown = 2, kFused = 3 };   // kFused: dense, 16-bit activations split in the kernel

struct TcArgs {
    uint32_t m, n;            // tokens, weight rows of one matrix
    uint32_t steps, kw;       // stages along K (256 values in KIND 4, 128 in KIND 8), code tiles along K
    uint32_t nt;              // tokens of a full CTA tile
    uint32_t group;           // tokens per 256 rows of pieces (KIND 8, kDense)
    uint32_t stages, split;   // ring depth; CTAs of a cluster that share a tile's K
    uint32_t stage_bytes, b_bytes, tmem_cols, d_cols, ring_bytes, row_tiles;
    const uint8_t *w_scales, *x_scales;
    void *y;
    int type;
    uint64_t stride;
    // kFused
    const void *x;
    uint32_t k;
    uint64_t x_stride;
    bool x_vec;
    // experts
    uint32_t top_k, per_cta, chunk, head_bytes;   // per_cta: row tiles (kSome); head: the choices, the columns' scales, gate and up values
    bool shared;              // kShared
    const int32_t *chosen;
    const float *weight;
    uint32_t *arrived;
    uint32_t *items;          // the gate / up product's work items, for the down product
    uint8_t *h_pieces, *h_scales;
    uint32_t h_steps;         // scale words along a hidden row
    float *partial;
    bool combine;             // the down product adds the pairs' parts itself
};

struct Ctrl {
    unsigned long long full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
    unsigned long long rows_ready, scales_ready, spare;
    uint32_t tmem;
    int abort;
    uint32_t pairs[32], found[4];
    float weights[kChunk];
    alignas(16) int32_t rows[kChunk * kMxHiddenPieces];   // of pieces
};
static_assert(sizeof(Ctrl) <= kCtrlBytes, "control block");

// DEAL: which row tiles a CTA of the experts takes: one, or up to per_cta, of an item, the grid being tiles, item, K; or
// its part of all items' tiles in a row (grid.x). A kernel each: the loops cost the one-tile kernel 0.3 us of 17.
enum Deal { kOne = 0, kSome = 1, kShared = 2 };
template <int KIND, int P, int MODE, int DEAL>
__global__ void __launch_bounds__(kThreads) mx_tc_kernel(const __grid_constant__ CUtensorMap wmap,
                                                         const __grid_constant__ CUtensorMap xmap, const TcArgs a) {
    constexpr bool kExperts = MODE == kGateUp || MODE == kDown, kDealt = DEAL == kShared;
    constexpr uint32_t kSub = KIND == 8 ? 1 : 2;                  // scale tiles of a stage, per 128 rows
    constexpr uint32_t kSf = kSub * kMxScaleTile;
    constexpr uint32_t kWeightTx = (KIND == 8 ? kMxCodeTile / 2 : kMxCodeTile) + kSf;  // an unpacking copy counts what it reads
    extern __shared__ uint8_t raw[];
    uint8_t *base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    Ctrl &c = *reinterpret_cast<Ctrl *>(base);
    // experts: tokens of each, the chosen expert of every pair, the columns' scales, gate and up values
    uint32_t *counts = reinterpret_cast<uint32_t *>(base + kCtrlBytes);
    uint8_t *ids = base + kCtrlBytes + 1024;
    uint8_t *sfb_all = ids + (MODE == kGateUp ? up_to(a.m * a.top_k, kMxScaleTile) : 0);
    uint8_t *ring = base + kCtrlBytes + (kExperts ? a.head_bytes : 0);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = blockIdx.z;
    volatile int *abort = &c.abort;

    auto init_barriers = [&] {
        for (uint32_t i = 0; i < kMaxStages; i++) {
            mbar_init(smem_u32(&c.full[i]), 2);
            mbar_init(smem_u32(&c.empty[i]), 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_u32(&c.acc_full[i]), 1);
            mbar_init(smem_u32(&c.acc_empty[i]), 4);
        }
        mbar_init(smem_u32(&c.spare), 1);
        mbar_init(smem_u32(&c.rows_ready), 128);
        mbar_init(smem_u32(&c.scales_ready), 128);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    };
    auto drop_barriers = [&] {   // before they are set up anew
        for (uint32_t b = smem_u32(&c.full[0]); b <= smem_u32(&c.spare); b += 8)
            asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(b) : "memory");
    };
    if (threadIdx.x == 0) {
        init_barriers();
        c.abort = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&xmap)) : "memory");
    }

    // ---- what this CTA computes ----
    uint32_t tile0 = DEAL == kSome ? blockIdx.x * a.per_cta : blockIdx.x, w_tile = tile0;
    uint32_t tiles = DEAL == kSome ? min(a.per_cta, a.row_tiles - tile0) : 1;
    uint32_t tokens = 0, tok0 = 0, expert = 0, chunk = 0;   // columns: tokens, or a chunk of one expert's pairs
    uint32_t mine = 0;                                 // lanes (pairs) of the expert, where one warp holds all pairs
    const uint32_t k0 = a.steps * rank / a.split, k1 = a.steps * (rank + 1) / a.split;
    const uint32_t pairs = kExperts ? a.m * a.top_k : 0;
    const bool one_warp = MODE == kGateUp && pairs <= 32 && a.m <= a.chunk;
    // Work items: every chosen expert's tokens in chunks. The gate / up product finds its items from the
    // choices themselves and leaves the list to the down product. kShared: a CTA takes the tiles [unit, unit_end) of
    // all items' tiles in a row, one item after another.
    uint32_t item = blockIdx.y, unit = 0, unit_end = 0, total = 0;
    uint32_t id = 0, same = 0, firsts = 0;             // one_warp: the lane's choice, the lanes of the same and of firsts
    if constexpr (!kExperts) {
        tok0 = blockIdx.y * a.nt;
        tokens = min(a.nt, a.m - tok0);
    } else {
        if (MODE == kDown) {
            grid_dep_wait();  // the items and the hidden vectors
            total = __ldcg(a.items);
        } else if (one_warp) {
            // few pairs: a lane each in every warp, experts in the order of their first choice
            grid_dep_wait();  // the router's choice
            id = (uint32_t)lane < pairs ? (uint32_t)__ldcg(a.chosen + lane) : 0xFFFFu;
            same = __match_any_sync(~0u, id);
            firsts = __ballot_sync(~0u, (uint32_t)lane < pairs && __ffs(same) - 1 == lane);
            total = __popc(firsts);
        } else {
            // experts in order, counted in shared memory
            for (uint32_t i = threadIdx.x; i < 256; i += kThreads) counts[i] = 0;
            __syncthreads();
            grid_dep_wait();
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < pairs; i += kThreads) {
                const uint32_t e = (uint32_t)__ldcg(a.chosen + i);
                ids[i] = (uint8_t)e;
                atomicAdd(&counts[e % 256], 1u);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; i++) total += (counts[lane * 8 + i] + a.chunk - 1) / a.chunk;
            total = __reduce_add_sync(~0u, total);
        }
        if (MODE == kGateUp && blockIdx.x == 0 && blockIdx.y == 0 && rank == 0 && threadIdx.x == 0) a.items[0] = total;
    }
    auto find = [&] {   // the item's expert and tokens
        if (MODE == kDown) {
            const uint32_t *it = a.items + kItemWords * (1 + item);
            const uint32_t of = __ldcg(it), pair = __ldcg(it + 2 + lane);
            tokens = __ldcg(it + 1);
            expert = of;
            if (warp == 2) c.pairs[lane] = pair;
        } else if (one_warp) {
            const int first = (int)__fns(firsts, 0, (int)item + 1);
            expert = __shfl_sync(~0u, id, first);
            mine = __shfl_sync(~0u, same, first);
            tokens = __popc(mine);
        } else {   // every warp on its own: a lane has eight experts
            uint32_t n[8], items = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                n[i] = counts[lane * 8 + i];
                items += (n[i] + a.chunk - 1) / a.chunk;
            }
            uint32_t upto = items;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t below = __shfl_up_sync(~0u, upto, o);
                if (lane >= o) upto += below;
            }
            const int holder = __ffs(__ballot_sync(~0u, item < upto)) - 1;   // there is one: item < total
            uint32_t left = item - (upto - items), found = 0, here = 0;
            bool open = true;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t chunks = (n[i] + a.chunk - 1) / a.chunk;
                if (open && left < chunks) {
                    found = lane * 8 + i;
                    here = n[i];
                    open = false;
                }
                if (open) left -= chunks;
            }
            expert = __shfl_sync(~0u, found, holder);
            chunk = __shfl_sync(~0u, left, holder);
            tokens = min(__shfl_sync(~0u, here, holder) - chunk * a.chunk, a.chunk);
        }
        w_tile = expert * a.row_tiles + tile0;
    };
    auto next_item = [&] {
        item = unit / a.row_tiles;
        tile0 = unit - item * a.row_tiles;
        tiles = min(a.row_tiles - tile0, unit_end - unit);
        unit += tiles;
        find();
    };
    if (kDealt) {
        const uint32_t units = total * a.row_tiles;
        unit = units * blockIdx.x / gridDim.x;
        unit_end = units * (blockIdx.x + 1) / gridDim.x;
        if (unit == unit_end) return;
        next_item();
    } else if (kExperts) {
        if (MODE == kDown) find();   // its loads go out with the total's; past that they read the list's unused places
        if (item >= total) return;   // the same in the whole cluster
        if (MODE != kDown) find();
    }
    constexpr uint32_t accs = DEAL == kOne ? 1 : 2;   // accumulators: the epilogue reads one while the next fills
    uint32_t n_cols, b_bytes, stage_bytes, stages;
    const uint32_t sfb_cols = KIND == 8 && a.nt * P > 128 ? 8 : 4, sf_cols = kSub * (4 + sfb_cols);
    auto shape_ring = [&] {   // the experts' ring is as deep as this expert's few tokens allow
        n_cols = (tokens * P + 7) / 8 * 8;
        b_bytes = kExperts ? n_cols * 128 : a.b_bytes;
        stage_bytes = kExperts ? kA + b_bytes + 1024 : a.stage_bytes;
        stages = kExperts ? min(a.stages, a.ring_bytes / stage_bytes) : a.stages;
    };
    shape_ring();
    const uint32_t col_tiles = kExperts ? 1 : (n_cols + 127) / 128;

    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem)),
                     "r"(a.tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (kExperts) grid_dep_launch();  // every CTA holds its TMEM: the next kernel's may come
    const uint32_t tmem = c.tmem, steps = k1 - k0;

    // a column's row of pieces; columns past the last token repeat it
    auto row_of = [&](uint32_t i) {
        const uint32_t pair = c.pairs[min(i / P, tokens - 1)];
        return (MODE == kGateUp ? pair / a.top_k : pair) * P + (i / P < tokens ? i % P : 0);
    };
    // no copy may land after this CTA has left: the last round's barriers, on the way out of an abort
    auto drain = [&](uint32_t issued) {
        for (uint32_t it = issued > stages ? issued - stages : 0; it < issued; it++)
            for (int i = 0; i < 100 && !mbar_try_wait(smem_u32(&c.full[it % stages]), it / stages & 1, 1000000); i++) {
            }
    };

    for (;;) {   // items (a dense product is one); the body is not indented for it
    if (warp == 0 && elect_one()) {
        // ---- weight tiles and their scales, in the order of memory ----
        // The kernel before may be any, one that writes the weights too; but the one that makes pieces has seen
        // all earlier work done.
        if (MODE == kFused || (MODE == kDense && KIND == 4)) grid_dep_wait();
        const uint32_t st0 = smem_u32(ring), full0 = smem_u32(&c.full[0]), empty0 = smem_u32(&c.empty[0]);
        uint32_t st = st0, full = full0, empty = empty0, s = 0, phase = 1, issued = 0;   // phase 1: not yet used
        for (uint32_t tile = 0; tile < tiles; tile++) {
            const uint32_t wt = w_tile + tile;
            int x = KIND == 8 ? (int)(k0 % 2 * 128) : 0;   // KIND 8: a half of a code tile
            int y = (int)((wt * a.kw + (KIND == 8 ? k0 / 2 : k0)) * 128);
            const uint8_t *sf = a.w_scales + ((size_t)wt * 2 * a.kw + kSub * k0) * kMxScaleTile;
            for (uint32_t step = 0; step < steps; step++, sf += kSf) {
                if (!mbar_poll(empty, phase, abort, 601)) goto weights_out;
                mbar_expect(full, kWeightTx);
                tma_2d(st, &wmap, x, y, full);
                bulk_copy(st + kA + b_bytes, sf, kSf, full);
                if (KIND == 8) x ^= 128;
                if (x == 0) y += 128;
                issued++;
                st += stage_bytes, full += 8, empty += 8;
                if (++s == stages) s = 0, phase ^= 1, st = st0, full = full0, empty = empty0;
            }
        }
        // before a next item sets the barriers up anew: the MMAs' arrivals on all of these
        for (uint32_t i = 0; kDealt && unit != unit_end && i < stages; i++) {
            if (!mbar_poll(empty, phase, abort, 603)) break;
            empty += 8;
            if (++s == stages) s = 0, phase ^= 1, empty = empty0;
        }
    weights_out:
        if (*abort) drain(issued);
    } else if (warp == 6 && MODE != kFused) {
        // ---- activation columns and, for dense products, their scales ----
        const bool listed = !kExperts || mbar_poll(smem_u32(&c.rows_ready), 0, abort, 605);
        if (kExperts && listed)
            for (uint32_t i = lane; i < n_cols; i += 32) c.rows[i] = (int32_t)row_of(i);
        __syncwarp();
        if (listed && elect_one()) {
            if (MODE == kDense) grid_dep_wait();  // the pieces, or codes
            const uint32_t st0 = smem_u32(ring) + kA, full0 = smem_u32(&c.full[0]), empty0 = smem_u32(&c.empty[0]);
            uint32_t st = st0, full = full0, empty = empty0, s = 0, phase = 1, issued = 0;
            if (MODE == kDense) {
                const bool two = KIND == 8 && col_tiles > 1;   // more than 128 columns (three pieces): a second tile of scales
                const uint32_t tx = a.b_bytes + (two ? 2 : 1) * kSf;
                const uint32_t row = KIND == 8 ? tok0 / a.group * 256 + tok0 % a.group * P : tok0;
                const uint32_t row_sf = (KIND == 8 ? a.steps : 2 * a.kw) * kMxScaleTile;   // scales of 128 rows
                const uint8_t *sf = a.x_scales + (size_t)(row / 128) * row_sf + k0 * kSf;
                int x = KIND == 8 ? (int)(k0 * 128) : (int)((row / 128 * a.kw + k0) * 128);
                for (uint32_t step = 0; step < steps; step++, x += 128, sf += kSf) {
                    if (!mbar_poll(empty, phase, abort, 608)) goto columns_out;
                    mbar_expect(full, tx);
                    if (KIND == 8) tma_2d(st, &xmap, x, (int)row, full);
                    else tma_2d(st, &xmap, 0, x, full);
                    bulk_copy(st + b_bytes + kSf, sf, kSf, full);
                    if (two) bulk_copy(st + b_bytes + 2 * kSf, sf + row_sf, kSf, full);
                    issued++;
                    st += stage_bytes, full += 8, empty += 8;
                    if (++s == stages) s = 0, phase ^= 1, st = st0, full = full0, empty = empty0;
                }
            } else {
                const int4 *rows = reinterpret_cast<const int4 *>(c.rows);
                const int4 r0 = rows[0], r1 = rows[1], r2 = rows[2], r3 = rows[3];   // most experts' columns
                for (uint32_t tile = 0; tile < tiles; tile++) {
                    int x = (int)(k0 * 128);
                    for (uint32_t step = 0; step < steps; step++, x += 128) {
                        if (!mbar_poll(empty, phase, abort, 608)) goto columns_out;
                        mbar_expect(full, n_cols * 128);
                        tma_gather4(st, &xmap, x, r0, full);
                        tma_gather4(st + 512, &xmap, x, r1, full);
                        if (n_cols > 8) {
                            tma_gather4(st + 1024, &xmap, x, r2, full);
                            tma_gather4(st + 1536, &xmap, x, r3, full);
                        }
                        for (uint32_t i = 16; i < n_cols; i += 4) tma_gather4(st + i * 128, &xmap, x, rows[i / 4], full);
                        issued++;
                        st += stage_bytes, full += 8, empty += 8;
                        if (++s == stages) s = 0, phase ^= 1, st = st0, full = full0, empty = empty0;
                    }
                }
            }
        columns_out:
            if (*abort) drain(issued);
        }
    } else if (warp == 1 && elect_one()) {
        // ---- MMA ----
        const uint32_t sf_tmem = tmem + a.d_cols * accs, idesc = scaled_instr_desc<KIND>(128, n_cols);
        const uint32_t st0 = smem_u32(ring), full0 = smem_u32(&c.full[0]), empty0 = smem_u32(&c.empty[0]);
        // each stage has scale columns of its own: they are rewritten only after its MMAs are done
        uint32_t st = st0, full = full0, empty = empty0, sfa = sf_tmem, s = 0, phase = 0;
        bool ok = !kExperts || mbar_poll(smem_u32(&c.scales_ready), 0, abort, 606);
        for (uint32_t tile = 0; ok && tile < tiles; tile++) {
            if (tile >= 2 && !mbar_poll(smem_u32(&c.acc_empty[tile & 1]), (tile / 2 & 1) ^ 1, abort, 607)) {
                ok = false;
                break;
            }
            const uint32_t d = tmem + (tile & 1) * a.d_cols;
            uint32_t sfb_smem = smem_u32(sfb_all);
            for (uint32_t step = 0; step < steps; step++) {
                if (!mbar_poll(full, phase, abort, 602)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t b = st + kA, sf = b + b_bytes, sfb = sfa + 4 * kSub;
#pragma unroll
                for (uint32_t h = 0; h < kSub; h++) {
                    scales_to_tmem(sfa + 4 * h, sf + h * kMxScaleTile);
                    if (!kExperts) {
                        scales_to_tmem(sfb + sfb_cols * h, sf + kSf + h * kMxScaleTile);
                        if (KIND == 8 && col_tiles > 1) scales_to_tmem(sfb + sfb_cols * h + 4, sf + 2 * kSf + h * kMxScaleTile);
                    } else {
                        scales_to_tmem(sfb, sfb_smem);
                    }
                }
                sfb_smem += kMxScaleTile;
                const uint64_t ad = smem_desc(st), bd = smem_desc(b);
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {   // 32 bytes of each row at a time
                    const uint32_t h = KIND == 8 ? 0 : j / 2, id = KIND == 8 ? j : j % 2 * 2;   // which scale bytes
                    mma_scaled<KIND>(d, ad + 2 * j, bd + 2 * j, idesc | id << 4 | id << 29, sfa + 4 * h, sfb + sfb_cols * h,
                                     step | j);
                }
                mma_commit(empty);
                st += stage_bytes, full += 8, empty += 8, sfa += sf_cols;
                if (++s == stages) s = 0, phase ^= 1, st = st0, full = full0, empty = empty0, sfa = sf_tmem;
            }
            mma_commit(smem_u32(&c.acc_full[tile & 1]));
        }
        if (!ok) {   // the MMAs that were issued end before TMEM is freed
            mma_commit(smem_u32(&c.spare));
            for (int i = 0; i < 100 && !mbar_try_wait(smem_u32(&c.spare), 0, 1000000); i++) {
            }
        }
    }
    __syncwarp();
    const bool epi = warp >= 2 && warp < 6;
    if constexpr (MODE == kFused) {
        // ---- the columns of at most 32 pieces, made here (a launch of its own for them costs 2.5 us of the host's
        // time): a warp to every fourth stage, 16 lanes to a token's 128 values of it ----
        using T = typename std::conditional<P == 2, __nv_bfloat16, __half>::type;
        constexpr uint32_t kPasses = 32 / P / 2;   // two tokens each
        if (epi) {
            grid_dep_wait();
            const uint32_t l16 = lane % 16, passes = (tokens + 1) / 2;
            MxRaw<T> raw[kPasses];   // of the warp's next stage
            auto load = [&](uint32_t step, uint32_t n) {
                const uint32_t j = (k0 + step) * 128 + l16 * 8, left = step < steps && j < a.k ? a.k - j : 0;
                const uint32_t t = n * 2 + lane / 16;
                const T *p = static_cast<const T *>(a.x) + t * a.x_stride + j;
                if (a.x_vec && left >= 8 && t < tokens) raw[n].load(p);
                else raw[n].load_some(p, t < tokens ? left : 0);
            };
            const uint32_t w = warp - 2;
#pragma unroll
            for (uint32_t n = 0; n < kPasses; n++)
                if (n < passes) load(w, n);
            uint32_t s = w, phase = 1;
            while (s >= stages) s -= stages, phase ^= 1;
            for (uint32_t step = w; step < steps; step += 4) {
                if (!__all_sync(~0u, mbar_poll(smem_u32(&c.empty[s]), phase, abort, 609))) break;
                const uint32_t b = smem_u32(ring + s * stage_bytes) + kA, sf = b + b_bytes + kSf;
#pragma unroll
                for (uint32_t n = 0; n < kPasses; n++) {
                    if (n >= passes) break;
                    const uint32_t t = n * 2 + lane / 16;
                    uint32_t top = raw[n].top();
                    top = max(top, __shfl_xor_sync(~0u, top, 1));
                    top = max(top, __shfl_xor_sync(~0u, top, 2));
                    const uint32_t sc = mx_piece_scale(__uint_as_float(raw[n].top_bits(top)), P);
                    float v[8];
                    raw[n].values(v, __uint_as_float((254u - min(sc, 253u)) << 23));
                    load(step + 4, n);
#pragma unroll
                    for (uint32_t p = 0; p < P; p++) {
                        uint32_t h[4];
                        mx_piece8(v, h);
                        if (t >= tokens) continue;
                        if (sc == 255) h[0] = h[1] = h[2] = h[3] = 0;
                        const uint32_t r = t * P + p;   // column; SWIZZLE_128B: its 16-byte chunks by its place in eight
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(b + r * 128 + ((l16 / 2 ^ (r & 7)) << 4) + l16 % 2 * 8),
                                     "r"(h[0] | h[1] << 16), "r"(h[2] | h[3] << 16)
                                     : "memory");
                        if (l16 % 4 == 0)
                            asm volatile("st.shared.u8 [%0], %1;" ::"r"(sf + r * 16 + l16 / 4), "r"(mx_piece_scale_of(sc, p)) : "memory");
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&c.full[s]));
                s += 4;
                while (s >= stages) s -= stages, phase ^= 1;
            }
        }
        __syncwarp();
    }
    if (kExperts && epi) {
        // ---- the item's tokens, and all their scales of this CTA's share of K ----
        const uint32_t at = threadIdx.x - 64;
        if (MODE == kGateUp && one_warp) {
            if (warp == 2 && (mine >> lane & 1)) c.pairs[__popc(mine & ((1u << lane) - 1))] = lane;
        } else if (MODE == kGateUp) {   // its pairs, in order: every warp looks through a quarter of them
            const uint32_t quarter = up_to(pairs, 128) / 4, w = warp - 2, from = w * quarter, to = min(from + quarter, pairs);
            uint32_t seen = 0;
            for (uint32_t i = from; i < to; i += 32) seen += __popc(__ballot_sync(~0u, i + lane < to && ids[i + lane] == expert));
            if (lane == 0) c.found[w] = seen;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            seen = 0;
            for (uint32_t i = 0; i < w; i++) seen += c.found[i];
            for (uint32_t i = from; i < to; i += 32) {
                const bool hit = i + lane < to && ids[i + lane] == expert;
                const uint32_t mask = __ballot_sync(~0u, hit), nth = seen + __popc(mask & ((1u << lane) - 1)) - chunk * a.chunk;
                if (hit && nth < a.chunk) c.pairs[nth] = i + lane;
                seen += __popc(mask);
            }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        mbar_arrive(smem_u32(&c.rows_ready));
#pragma unroll 4
        for (uint32_t j = at; j < n_cols * steps; j += 128) {
            const uint32_t i = j / steps, t = j - i * steps;
            *reinterpret_cast<uint32_t *>(sfb_all + t * kMxScaleTile + i % 32 * 16 + i / 32 * 4) =
                __ldcg(reinterpret_cast<const uint32_t *>(a.x_scales) + (size_t)row_of(i) * a.steps + k0 + t);
        }
        fence_proxy_async();  // read by the tensor core's scale copy
        mbar_arrive(smem_u32(&c.scales_ready));
        if (MODE == kDown) {
            if (at < tokens) c.weights[at] = __ldcg(a.weight + c.pairs[at]);
            asm volatile("bar.sync 1, 128;" ::: "memory");
        }
        if (MODE == kGateUp && tile0 == 0 && rank == 0 && warp == 2) {
            uint32_t *it = a.items + kItemWords * (1 + item);
            if (lane < tokens) it[2 + lane] = c.pairs[lane];
            if (lane == 0) it[0] = expert, it[1] = tokens;
        }
    }

    // ---- epilogue: thread = weight row ----
    const uint32_t q = warp % 4;
    uint32_t tile = tile0, row = tile0 * 128 + q * 32 + lane;   // of the tile being read
    // [token][128]: a cluster's partial sums, and the gate and up values, which lie in different warps' rows
    // (at the same place in every CTA of the cluster, whose shares of K may differ by a step)
    float *red =
        reinterpret_cast<float *>(MODE == kGateUp ? sfb_all + (a.steps + a.split - 1) / a.split * kMxScaleTile : ring);

    // The hidden value of one of the tile's 64 and its pieces. A warp's 32 are one block along the next
    // product's K. Four pieces hold it to 2^-19 of itself, or 2^-29 of its block's largest: where the sums in 32 bits
    // are off by as much. Three hold it to 2^-14, which outputs in f16 show. One token through 4 of 32 experts, and 64
    // through 8 of 128: three pieces 17.0 and 96.4 us, four 17.1 and 99.1, five (2^-24) 17.1 and 104.3.
    auto hidden = [&](uint32_t i, float g, float u) {
        const float h = g / (1.0f + expf(-g)) * u;
        const uint32_t top = __reduce_max_sync(~0u, __float_as_uint(h) & 0x7FFFFFFFu);
        const uint32_t s = mx_piece_scale(__uint_as_float(top), kMxHiddenPieces);
        float left = h * __uint_as_float((254u - min(s, 253u)) << 23);
        const uint32_t at = tile * kMxHalf + q % 2 * 32 + lane;
        const bool pad = tile + 1 == a.row_tiles && a.row_tiles % 2;   // the next product's tiles are 128 wide
        const size_t r = (size_t)c.pairs[i] * kMxHiddenPieces;
#pragma unroll
        for (int p = 0; p < kMxHiddenPieces; p++) {
            float back;
            const uint32_t code = mx_e4m3(left, &back);
            left = (left - back) * 16.0f;
            uint8_t *to = a.h_pieces + (r + p) * a.h_steps * 128 + at;
            uint8_t *sf = a.h_scales + (r + p) * a.h_steps * 4 + at / 32;
            *to = s == 255 ? 0 : (uint8_t)code;
            if (lane == 0) *sf = (uint8_t)mx_piece_scale_of(s, p);
            if (pad) {
                to[kMxHalf] = 0;
                if (lane == 0) sf[kMxHalf / 32] = 0;
            }
        }
    };
    // Down products go, weighted, to their pairs' own places. The warp that brings a token's last pair of
    // 32 rows adds the token's top_k parts in their order, so the sum does not depend on who that is.
    // This is done once for all tiles of the CTA: one fence, and a lane to each (tile, token)
    // (a fence and a round of atomics after every tile took 4.4 us a tile, its MMAs 2.2).
    auto part = [&](uint32_t i, float v) {
        if (row < a.n) a.partial[(size_t)c.pairs[i] * a.n + row] = v * c.weights[i];
    };
    auto combine = [&](uint32_t first, uint32_t step) {
        __threadfence();
        __syncwarp();
        const uint32_t each = (tokens - first + step - 1) / step, all = first < tokens ? tiles * each : 0;
        for (uint32_t j0 = 0; j0 < all; j0 += 32) {
            const uint32_t j = j0 + lane, of = j / each, i = first + (j - of * each) * step;
            const uint32_t t = j < all ? c.pairs[i] / a.top_k : 0;
            const bool last =
                j < all && atomicAdd(a.arrived + ((size_t)t * a.row_tiles + tile0 + of) * 4 + q, 1u) == a.top_k - 1;
            uint32_t mask = __ballot_sync(~0u, last);
            __threadfence();
            while (mask) {
                const int from = __ffs(mask) - 1;
                const uint32_t to = __shfl_sync(~0u, t, from), at = (tile0 + __shfl_sync(~0u, of, from)) * 128 + q * 32 + lane;
                mask &= mask - 1;
                if (at < a.n) {
                    const float *parts = a.partial + (size_t)to * a.top_k * a.n + at;
                    float sum = 0.0f;
#pragma unroll 8
                    for (uint32_t p = 0; p < a.top_k; p++) sum += __ldcg(parts + (size_t)p * a.n);
                    put_as(a.y, a.type, to * a.stride + at, sum);
                }
            }
        }
    };

    for (uint32_t nth = 0; epi && nth < tiles; nth++) {
        tile = tile0 + nth;
        row = tile * 128 + q * 32 + lane;
        mbar_poll(smem_u32(&c.acc_full[nth & 1]), nth / 2 & 1, abort, 604);
        tc_fence_after();
        const uint32_t taddr = tmem + (q * 32 << 16) + (nth & 1) * a.d_cols;
        if (!kExperts && a.split == 1) {
            constexpr uint32_t kAt = P == 1 ? 32 : P == 2 ? 16 : 8;   // tokens at a time: up to 32 columns
            uint32_t i0 = 0;
            for (; i0 + kAt <= up_to(tokens, 8); i0 += kAt) {
                float v[kAt];
                load_tokens<P>(taddr + i0 * P, v);
                if (row < a.n) put_tokens_as(a.y, a.type, (tok0 + i0) * a.stride + row, a.stride, v, tokens - i0);
            }
            for (; i0 < tokens; i0 += 8) {
                float v[8];
                load_tokens<P>(taddr + i0 * P, v);
                if (row < a.n) put_tokens_as(a.y, a.type, (tok0 + i0) * a.stride + row, a.stride, v, tokens - i0);
            }
        } else {
            if (MODE == kGateUp && nth) asm volatile("bar.sync 1, 128;" ::: "memory");   // the last tile's values are read
            for (uint32_t i0 = 0; i0 < tokens; i0 += 8) {
                float v[8];
                load_tokens<P>(taddr + i0 * P, v);
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) {
                    if (i0 + i >= tokens) break;
                    if (MODE == kDown && a.split == 1) part(i0 + i, v[i]);
                    else red[(i0 + i) * 128 + q * 32 + lane] = v[i];
                }
            }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&c.acc_empty[nth & 1]));
        if (MODE == kGateUp && a.split == 1) {
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (uint32_t i = q / 2; i < tokens; i += 2) {   // a warp: half of the tokens, half of the tile's 64 values
                const float *v = red + i * 128 + q % 2 * 32 + lane;
                hidden(i, v[0], v[kMxHalf]);
            }
        }
    }
    if (MODE == kDown && epi && a.split == 1 && a.combine) combine(0, 1);
    if (a.split > 1) {
        // the cluster's partial tiles, added in rank order through distributed shared memory
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (epi) {
            const uint32_t first = MODE == kGateUp ? rank * 2 + q / 2 : rank, every = MODE == kGateUp ? 2 * a.split : a.split;
            const uint32_t at = MODE == kGateUp ? q % 2 * 32 + lane : q * 32 + lane;
            for (uint32_t i0 = first; i0 < tokens; i0 += 4 * every) {
                float g[4] = {}, u[4] = {};   // four tokens' loads go out before the first sum
#pragma unroll
                for (uint32_t r = 0; r < 8; r++) {
                    if (r >= a.split) break;
                    const float *other = cluster.map_shared_rank(red, r) + at;
                    float v[4], w[4];
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) {
                        const uint32_t i = min(i0 + j * every, tokens - 1);
                        v[j] = other[i * 128];
                        if (MODE == kGateUp) w[j] = other[i * 128 + kMxHalf];
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) {
                        g[j] += v[j];
                        if (MODE == kGateUp) u[j] += w[j];
                    }
                }
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const uint32_t i = i0 + j * every;
                    if (i >= tokens) break;
                    if (MODE == kGateUp) hidden(i, g[j], u[j]);
                    else if (MODE == kDown) part(i, g[j]);
                    else if (row < a.n) put_as(a.y, a.type, (tok0 + i) * a.stride + row, g[j]);
                }
            }
        }
        __syncwarp();
        cluster.barrier_arrive();   // this CTA reads the others' shared memory no more
        if (MODE == kDown && epi && a.combine) combine(rank, a.split);
        __syncwarp();
        cluster.barrier_wait();
    }
    if (!kDealt || unit == unit_end) break;
    // The next item, once this one's tiles are out. All its copies and MMAs have been waited for, or the CTA gives up.
    __syncthreads();
    tc_fence_after();
    const bool give_up = *abort;
    if (threadIdx.x == 0) {
        drop_barriers();
        init_barriers();
    }
    next_item();
    shape_ring();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (give_up) break;
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols));
    }
}

// ---- activation pieces of a dense product ---------------------------------------------------------
//
// The quantiser's division of work (k_mx.cu): a warp takes 256 columns of ROWS tokens and writes P
// rows of e4m3 for each. Token t's pieces are rows t / group * 256 + t % group * P + p, so that a
// full tile of tokens starts on a scale tile.

template <typename T, int P, int ROWS>
__global__ void __launch_bounds__(256) pieces_kernel(const T *x, uint32_t m, uint32_t k, uint64_t stride, uint32_t kt,
                                                     uint32_t chunks, uint32_t group, uint8_t *pieces, uint8_t *scales, bool vec) {
    grid_dep_wait();
    grid_dep_launch();  // the product may start on its weights
    const uint32_t lane = threadIdx.x % 32, w = blockIdx.x * 8 + threadIdx.x / 32;
    const uint32_t tokens = w / chunks, chunk = w - tokens * chunks, t0 = tokens * ROWS;
    if (t0 >= m) return;
    const uint32_t n = min((uint32_t)ROWS, m - t0), j = chunk * 256 + lane * 8;
    MxRaw<T> raw[ROWS];
    mx_load_rows<T, ROWS>(raw, x + t0 * stride + j, stride, n, j < k ? k - j : 0, vec && chunk * 256 + 256 <= k);
    uint32_t r = t0 / group * 256 + t0 % group * P;   // ROWS divides the group: the rows follow each other
    uint8_t *to = pieces + (size_t)r * kt * 128 + j;
    const bool mine = j / kMxTile < kt;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        if ((uint32_t)i >= n) break;
        uint32_t top = raw[i].top();
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        const uint32_t s = mx_piece_scale(__uint_as_float(raw[i].top_bits(top)), P);
        float v[8];
        raw[i].values(v, __uint_as_float((254u - min(s, 253u)) << 23));
#pragma unroll
        for (int p = 0; p < P; p++, r++, to += (size_t)kt * 128) {
            uint32_t h[4];
            mx_piece8(v, h);
            if (mine) {
                *reinterpret_cast<uint2 *>(to) = s == 255 ? make_uint2(0, 0) : make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
                if (lane % 4 == 0) scales[mx_scale_at(r, j / 32, kt)] = (uint8_t)mx_piece_scale_of(s, p);
            }
        }
    }
}

// ---- the parts of every token's pairs, added in their order --------------------------------------
//
// For many pairs: in the down product nearly every CTA near the end brings last pairs, and its sums, one after
// another, kept 64 tokens of 8 pairs 13 us longer than this kernel. Few pairs' sums cost less there.

__global__ void __launch_bounds__(128) combine_kernel(const float *partial, uint32_t d, uint32_t top_k, void *y, int type,
                                                      uint64_t stride) {
    grid_dep_wait();
    const uint32_t at = blockIdx.x * 128 + threadIdx.x, t = blockIdx.y;
    if (at >= d) return;
    const float *parts = partial + (size_t)t * top_k * d + at;
    float sum = 0.0f;
#pragma unroll 8
    for (uint32_t p = 0; p < top_k; p++) sum += __ldcg(parts + (size_t)p * d);
    put_as(y, type, t * stride + at, sum);
}

// ---- host -----------------------------------------------------------------------------------------

cudaError_t encode(CUtensorMap *map, CUtensorMapDataType type, const void *ptr, uint64_t inner, uint64_t rows, uint64_t pitch,
                   uint32_t box0, uint32_t box1, CUtensorMapSwizzle swizzle) {
    const cuuint64_t dims[2] = {inner, rows}, strides[1] = {pitch};
    const cuuint32_t box[2] = {box0, box1}, ones[2] = {1, 1};
    EncodeTiled fn = encoder();
    if (!fn || fn(map, type, 2, const_cast<void *>(ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    return cudaSuccess;
}

// Weight tiles: 128 bytes of codes a row, tiles of 128 rows one after another. KIND 8 unpacks half a row at a time.
template <int KIND>
cudaError_t encode_weights(CUtensorMap *map, const uint8_t *codes, uint64_t tiles) {
    if (KIND == 8)
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, codes, 256, tiles * 128, 128, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, 128, tiles * 128, 128, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
}

uint32_t pow2_cols(uint32_t v) {
    uint32_t c = 32;
    while (c < v) c *= 2;
    return c;
}

#include "mx_pair.cuh"

template <int KIND, int P, int MODE, int DEAL = kOne>
cudaError_t launch(const CUtensorMap &wmap, const CUtensorMap &xmap, const TcArgs &a, dim3 grid, uint32_t smem, cudaStream_t s) {
    // A CTA waits for its TMEM without a limit, and a cluster's for each other: with kernels on several streams, CTAs
    // of two clusters could each hold what the other's lack. So an SM has no more CTAs of clusters than its 512
    // columns serve: shared memory for two with up to 256 each, or for one.
    if (a.split > 1) smem = std::max(smem, (a.tmem_cols > 256 ? 116u : 112u) * 1024);
    if (!a.stages || a.tmem_cols > 512 || smem > 227 * 1024) return cudaErrorInvalidConfiguration;
    auto kernel = mx_tc_kernel<KIND, P, MODE, DEAL>;
    if (!once_per_device(100 + DEAL * 200 + KIND * 16 + P * 4 + MODE, [&] {
            return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) == cudaSuccess;
        }))
        return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = kThreads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled(kPdlMx) ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = a.split;
    cfg.attrs = attr;
    cfg.numAttrs = a.split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, wmap, xmap, a);
}

// Ring depth and shared memory for one or two (`per_sm`) CTAs on an SM.
template <int KIND, int P, int MODE>
uint32_t plan_ring(TcArgs &a, uint32_t per_sm) {
    const uint32_t n = up_to(a.nt * P, 8), sub = KIND == 8 ? 1 : 2;
    const bool experts = MODE == kGateUp || MODE == kDown;
    a.b_bytes = n * 128;
    a.stage_bytes = kA + a.b_bytes + up_to(kMxScaleTile * sub * (1 + (experts ? 0 : (n + 127) / 128)), 1024);
    a.d_cols = up_to(a.nt, 8) * P;
    const uint32_t sf_cols = sub * (4 + (a.nt * P > 128 ? 8 : 4));
    const uint32_t extra = 1024 + kCtrlBytes + a.head_bytes;
    const uint32_t budget = (per_sm == 1 ? 226 : 112) * 1024 - extra, cols = per_sm == 1 ? 512 : 256;
    const uint32_t acc_cols = a.d_cols * (a.shared || a.per_cta > 1 ? 2 : 1);
    a.stages = std::min((cols - acc_cols) / sf_cols, (uint32_t)kMaxStages);
    if (!a.shared) a.stages = std::min(a.stages, (a.steps + a.split - 1) / a.split * a.per_cta);
    if (!experts) {
        a.stages = std::min(a.stages, budget / a.stage_bytes);
        a.ring_bytes = a.stages * a.stage_bytes;
    } else {   // the kernel fits its stages into this by its expert's number of tokens
        a.ring_bytes = std::max(std::min(budget, a.stages * a.stage_bytes), a.stage_bytes);
        a.stages = std::min(a.stages, a.ring_bytes / (kA + 2048));
    }
    a.tmem_cols = pow2_cols(acc_cols + a.stages * sf_cols);
    const uint32_t red = MODE != kGateUp && a.split > 1 ? a.nt * 128 * 4 : 0;
    return extra + std::max(a.ring_bytes, red);
}

// x, x_scales: MX4 codes (KIND 4) or pieces (KIND 8), or null for MODE kFused.
template <int KIND, int P, int MODE>
cudaError_t dense(const MxProductArgs &p, const uint8_t *x, const uint8_t *x_scales, cudaStream_t s) {
    const uint32_t rt = mx_tiles(p.n), kw = mx_ktiles(p.k) / 2;
    constexpr uint32_t kGroup = P == 1 ? 256 : P == 2 ? 128 : 64;   // tokens that fill 256 columns (P = 3: 192)
    // Pairs of CTAs once their tiles go round most of the 74, whatever the form. Against single CTAs, K 4096 and 4096 weight
    // rows: 4 bits, 128 tiles 16.2 us and 20.0, 64 10.7 and 10.8, 32 10.3 and 6.7; bf16 28.8 and 33.5, 17.2 and 18.3, 15.2 and
    // 11.6; f16 22.0 and 25.2, 13.4 and 13.5, 12.2 and 12.4. With K 1024, 128 and 64 tiles: 4 bits 9.8 and 10.8, 7.1 and 6.2;
    // bf16 11.5 and 14.2, 8.2 and 8.4; f16 9.6 and 12.6, 7.0 and 7.2.
    if (MODE == kDense && p.m > kGroup / 2 && (rt + 1) / 2 * ((p.m + kGroup - 1) / kGroup) >= 64)
        return pair_product<KIND, P>(p, x, x_scales, s);
    TcArgs a{};
    a.m = p.m;
    a.n = p.n;
    a.kw = kw;
    a.steps = KIND == 8 ? mx_tiles(p.k) : kw;
    a.group = kGroup;
    a.row_tiles = rt;
    a.per_cta = 1;
    // 128 columns to a single CTA, two of which share an SM, rather than 256 (bf16 x, 128 x 4096 x 4096: 10.5 us, 15.1);
    // the pieces of f16 start on scale tiles every 64 tokens
    constexpr uint32_t kMost = P == 1 ? 128 : 64;
    a.nt = p.m < kMost ? p.m : kMost;
    const uint32_t tt = (p.m + a.nt - 1) / a.nt;
    // K over a cluster while that leaves a CTA an SM to itself, and once more where each still streams more than 200 KB
    // of weights (one token, 8192 x 8192: 2: 11.3 us, 4: 10.0, 8: 15.4; 16 tokens in 4 bits, 4096 x 4096: 2: 6.7, 4: 6.0,
    // 8: 8.5). More than 32 tokens' sums cost what they save (48 x 4096 x 4096: 1: 9.9, 2: 11.0, 4: 9.5).
    a.split = 1;
    while (a.split < 8 && rt * tt * a.split * 2 <= 148 && a.steps / (a.split * 2) >= 2 && a.nt <= 32) a.split *= 2;
    if (a.split < 8 && rt * tt * a.split * 2 <= 2 * 148 && a.steps / a.split > 24 && a.nt <= 32) a.split *= 2;
    const uint32_t per_sm = rt * tt * a.split > 148 && up_to(a.nt, 8) * P <= 128 ? 2 : 1;
    a.w_scales = p.w_scales;
    a.x_scales = x_scales;
    a.y = p.y;
    a.type = p.type;
    a.stride = p.stride;
    a.x = p.x;
    a.k = p.k;
    a.x_stride = p.x_stride;
    a.x_vec = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.x_stride % 8 == 0;
    const uint32_t smem = plan_ring<KIND, P, MODE>(a, per_sm);
    CUtensorMap wmap, xmap;
    cudaError_t e = encode_weights<KIND>(&wmap, p.w_codes, (uint64_t)rt * kw);
    if (e != cudaSuccess) return e;
    if (MODE == kFused)
        xmap = wmap;   // not read
    else if (KIND == 8)
        e = encode(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, (uint64_t)a.steps * 128, mx_piece_rows(p.m, p.x_type),
                   (uint64_t)a.steps * 128, 128, a.b_bytes / 128, CU_TENSOR_MAP_SWIZZLE_128B);
    else
        e = encode(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, 128, (uint64_t)mx_tiles(p.m) * kw * 128, 128, 128, a.b_bytes / 128,
                   CU_TENSOR_MAP_SWIZZLE_128B);
    if (e != cudaSuccess) return e;
    return launch<KIND, P, MODE>(wmap, xmap, a, dim3(rt, tt, a.split), smem, s);
}

template <typename T, int P>
cudaError_t dense_x16(const MxProductArgs &p, cudaStream_t s) {
    if (mx_fused(p.m, p.k, p.x_type)) return dense<8, P, kFused>(p, nullptr, nullptr, s);
    const uint32_t kt = mx_tiles(p.k), chunks = (p.k + 255) / 256;
    constexpr uint32_t kGroup = P == 2 ? 128 : 64;
    uint8_t *pieces = static_cast<uint8_t *>(p.workspace);
    const size_t rows = mx_piece_rows(p.m, p.x_type);
    uint8_t *scales = pieces + (rows * kt * 128 + 255) / 256 * 256;
    const bool vec = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.x_stride % 8 == 0;
    const bool many = (uint64_t)(p.m / 4) * chunks >= 148 * 32;   // as the quantiser's rule
    const uint64_t warps = many ? (uint64_t)((p.m + 3) / 4) * chunks : (uint64_t)p.m * chunks;
    auto kernel = many ? pieces_kernel<T, P, 4> : pieces_kernel<T, P, 1>;
    const cudaError_t e = launch_pdl(kPdlMx, kernel, (unsigned)((warps + 7) / 8), 256, 0, s, static_cast<const T *>(p.x), p.m, p.k,
                                     p.x_stride, kt, chunks, kGroup, pieces, scales, vec);
    return e != cudaSuccess ? e : dense<8, P, kDense>(p, pieces, scales, s);
}

// Whether the down product adds the pairs' parts: 32 pairs or fewer.
bool mx_combines(const MxExpertsArgs &e) { return e.tokens * e.top_k <= 32; }

template <int P, int MODE>
cudaError_t expert_product(const MxExpertsArgs &e, cudaStream_t s) {
    const uint32_t width = MODE == kGateUp ? e.d : e.f;
    TcArgs a{};
    a.m = e.tokens;
    a.n = e.d;
    a.steps = mx_tiles(width);
    a.kw = mx_ktiles(width) / 2;
    a.h_steps = mx_tiles(e.f);
    a.row_tiles = MODE == kGateUp ? (e.f + kMxHalf - 1) / kMxHalf : mx_tiles(e.d);
    a.top_k = e.top_k;
    a.chosen = e.ws.chosen;
    a.weight = e.ws.weight;
    a.arrived = e.ws.arrived;
    a.items = e.ws.items;
    a.h_pieces = e.ws.h_pieces;
    a.h_scales = e.ws.h_scales;
    a.partial = e.ws.partial;
    a.x_scales = MODE == kGateUp ? e.ws.x_scales : e.ws.h_scales;
    a.w_scales = MODE == kGateUp ? e.gate_up_scales : e.down_scales;
    a.y = e.y;
    a.type = e.type;
    a.stride = e.y_stride;
    a.combine = mx_combines(e);
    // Tokens to a CTA: 24 where that spares the experts their second or third item, else 16, whose columns cost less (16 of
    // 64 experts, d 2048, f 1024: 12 pairs to an expert on average 75.5 us with 16, 78.3 with 24; 14: 101, 87.5; 20: 131, 105;
    // 24: 138, 137; 28: 145, 163; 4 of 16, d 4096, f 2048: 13: 77.5, 79.1; 16: 107, 87.7; 32: 157, 168).
    const uint32_t pairs = e.tokens * e.top_k, slots = std::min(e.experts, pairs);
    a.chunk = pairs > e.experts * 13 && pairs <= e.experts * kChunk ? kChunk : 16;
    a.nt = std::min(e.tokens, a.chunk);
    // as many items as there can be: one to each chosen expert, one more for every further chunk of pairs
    const uint32_t items = slots + (pairs - slots) / a.chunk;
    // K is split over a cluster only so that its scales fit: a cluster's launch and sums cost more than they
    // save (one token, 4 of 32 experts: 18.1 us without, 18.4 to 19.5 with 2 or 4)
    a.split = 1;
    while (a.split < 8 && a.steps / a.split > 32) a.split *= 2;
    // A round of CTAs is two to an SM. Up to four tiles of an item to each while one round holds all items there can be;
    // more tiles are dealt out evenly, from one item on to the next, which costs 4 us for each change of items
    // (bf16, 4 of 32 experts, d 2048, f 1024, two tiles to a CTA: 16 tokens 31 us, dealt out 37; 8 of 128, four tiles: 8
    // tokens 46, dealt out 49; seven: 16 tokens 66 dealt out, 77 in rounds of four tiles, and 64 tokens 98 and 101).
    const uint32_t ctas = 2 * (uint32_t)current_sm_count(), each = (a.row_tiles * slots + ctas - 1) / ctas;
    a.shared = a.split == 1 && each > 4;
    a.per_cta = a.split == 1 && !a.shared ? each : 1;
    a.head_bytes = 1024 + (a.steps + a.split - 1) / a.split * kMxScaleTile +
                   (MODE == kGateUp ? up_to(pairs, kMxScaleTile) + a.nt * 512 : 0);
    a.head_bytes = up_to(a.head_bytes, 1024);
    const uint32_t smem = plan_ring<8, P, MODE>(a, 2);
    CUtensorMap wmap, xmap;
    cudaError_t r = encode_weights<8>(&wmap, MODE == kGateUp ? e.gate_up_codes : e.down_codes,
                                      (uint64_t)e.experts * a.row_tiles * a.kw);
    if (r != cudaSuccess) return r;
    const uint64_t piece_rows = MODE == kGateUp ? (uint64_t)e.tokens * P : (uint64_t)pairs * P;
    r = encode(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, MODE == kGateUp ? e.ws.x_pieces : e.ws.h_pieces, (uint64_t)a.steps * 128,
               piece_rows, (uint64_t)a.steps * 128, 128, 1, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != cudaSuccess) return r;
    if (a.shared) return launch<8, P, MODE, kShared>(wmap, xmap, a, dim3(ctas), smem, s);
    if (a.per_cta == 1) return launch<8, P, MODE>(wmap, xmap, a, dim3(a.row_tiles, items, a.split), smem, s);
    return launch<8, P, MODE, kSome>(wmap, xmap, a, dim3((a.row_tiles + a.per_cta - 1) / a.per_cta, items), smem, s);
}

}  // namespace

size_t mx_piece_rows(uint32_t m, int x_type) {
    const uint32_t p = mx_pieces(x_type), group = p == 2 ? 128 : 64;
    return (size_t)(m / group) * 256 + m % group * p;
}

cudaError_t launch_mx4_product(const MxProductArgs &a, cudaStream_t s) {
    if (!a.x) return dense<4, 1, kDense>(a, a.a_codes, a.a_scales, s);
    if (a.x_type == 1) return dense_x16<__half, 3>(a, s);
    return dense_x16<__nv_bfloat16, 2>(a, s);
}

cudaError_t launch_mx4_expert_products(const MxExpertsArgs &a, cudaStream_t s) {
    cudaError_t e = a.type == 1 ? expert_product<3, kGateUp>(a, s) : expert_product<2, kGateUp>(a, s);
    if (e == cudaSuccess) e = expert_product<kMxHiddenPieces, kDown>(a, s);
    if (e != cudaSuccess || mx_combines(a)) return e;
    return launch_pdl(kPdlMx, combine_kernel, dim3((a.d + 127) / 128, a.tokens), 128, 0, s, (const float *)a.ws.partial, a.d, a.top_k,
                      a.y, a.type, a.y_stride);
}

int mx_tc_error(bool reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tc_error, sizeof(int)) != cudaSuccess) return 0;
    if (v && reset) {
        const int z = 0;
        cudaMemcpyToSymbol(g_tc_error, &z, sizeof(int));
    }
    return v;
}

}  // namespace uq
