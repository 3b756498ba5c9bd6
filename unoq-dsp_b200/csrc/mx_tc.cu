// mx_tc.cu -- products with MX4 weights on the block-scaled tensor cores (include/unoq_mx.h).
//
// D[weight row][column] += sum over blocks b of 2^(sa + sb) * (codes of W) . (codes of X), tcgen05 with
// one scale per row and 32 values on both sides, accumulators in TMEM. The 128 weight rows of a tile
// are the M side whatever the number of tokens, so a single token streams the same weight tiles
// as a prompt does, and its column count N is the multiple of 8 that holds it. Two kinds:
//
//   KIND 4  kind::mxf4: both sides e2m1, 64 values per instruction.
//   KIND 8  kind::mxf8f6f4: weights e2m1 (TMA unpacks each 4-bit code to a byte of shared memory),
//           activations e4m3. A 16-bit activation is not rounded to e4m3: it is split into P pieces of
//           four significant bits, x = 2^s (p0 + p1 / 16 + p2 / 256) (P = 2 holds bf16's 8 bits, 3
//           f16's 11), each piece a column of its own whose block scale carries its power of 16;
//           the epilogue adds the P columns in 32 bits. Few tokens leave the columns unused
//           otherwise, and a 16-bit tensor-core product would need the weights expanded in registers.
#include <cooperative_groups.h>

#include <algorithm>

#include "device_state.hpp"
#include "mx.cuh"
#include "tc_common.cuh"

namespace uq {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxStages = 12;
constexpr int kThreads = 192;      // warp 0: TMA, warp 1: MMA, warps 2-5: epilogue
constexpr int kCtrlBytes = 2048;   // barriers, TMEM slot and, for the experts, the token list
constexpr int kChunk = 32;         // tokens of one expert that one CTA takes

enum Mode { kDense = 0, kGateUp = 1, kDown = 2 };

struct TcArgs {
    uint32_t m, n, kt;        // tokens, weight rows of one matrix, tiles along K
    uint32_t nt;              // tokens of a full CTA tile
    uint32_t group;           // tokens per 256 rows of pieces (KIND 8, kDense)
    uint32_t stages, split;   // ring depth; CTAs of a cluster that share a tile's K
    uint32_t stage_bytes, b_bytes, b_box_bytes, tmem_cols, d_cols;
    const uint8_t *w_scales, *x_scales;
    void *y;
    int type;
    uint64_t stride;
    // experts
    uint32_t experts, top_k, chunks, row_tiles, sfb_bytes;
    const int32_t *chosen;
    const float *weight;
    uint32_t *arrived;
    uint8_t *h_pieces, *h_scales;
    float *partial;
};

struct Ctrl {
    unsigned long long full[kMaxStages], empty[kMaxStages], done;
    uint32_t tmem;
    int abort;
    uint32_t chosen_bits[8];
    uint32_t pairs[kChunk];
    uint32_t count;
    alignas(16) int32_t rows[kChunk * 4];
};
static_assert(sizeof(Ctrl) <= kCtrlBytes, "control block");

__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
// Four rows of 128 bytes from anywhere in the matrix (the map's box is one row high).
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap *map, int c0, int4 r, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

// One 512-byte scale tile (128 rows x 4 blocks) into 4 TMEM columns, repeated for the four lane quarters.
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint32_t smem) {
    const uint64_t desc = (uint64_t)((smem >> 4) & 0x3FFF) | (1ull << 16) | (8ull << 32) | (1ull << 46);
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc));
}

template <int KIND>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    if (KIND == 8) return smem_desc(addr);  // 128-byte rows, SWIZZLE_128B
    // 64-byte rows, SWIZZLE_64B, 8-row atoms 512 bytes apart
    return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | (32ull << 32) | (1ull << 46) | (4ull << 61);
}

template <int KIND>
__device__ __forceinline__ uint32_t scaled_instr_desc(uint32_t n) {
    const uint32_t types = KIND == 8 ? (5u << 7) | (0u << 10) : (1u << 7) | (1u << 10);  // e2m1 x e4m3 | e2m1 x e2m1
    return types | (n >> 3) << 17 | 1u << 23 | 1u << 27;                                 // e8m0 scales, M = 128
}

template <int KIND>
__device__ __forceinline__ void mma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                           uint32_t acc) {
    if (KIND == 8)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc));
}

__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(r[i]));  // no use moves above the wait
}

// Eight tokens' values of this thread's weight row: the P columns of each, added in 32 bits, the
// smallest piece first.
template <int P>
__device__ __forceinline__ void load_tokens(uint32_t addr, float (&v)[8]) {
    uint32_t r[8 * P];
#pragma unroll
    for (int p = 0; p < P; p++) tmem_ld8(addr + 8 * p, r + 8 * p);
    tmem_wait(r);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = __uint_as_float(r[i * P + P - 1]);
#pragma unroll
        for (int p = P - 2; p >= 0; p--) v[i] += __uint_as_float(r[i * P + p]);
    }
}

__device__ __forceinline__ void put_as(void *y, int type, size_t at, float v) {
    if (type == 0) static_cast<float *>(y)[at] = v;
    else if (type == 1) static_cast<__half *>(y)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(y)[at] = __float2bfloat16_rn(v);
}

template <int KIND, int P, int MODE>
__global__ void __launch_bounds__(kThreads) mx_tc_kernel(const __grid_constant__ CUtensorMap wmap,
                                                         const __grid_constant__ CUtensorMap xmap, const TcArgs a) {
    constexpr uint32_t kA = KIND == 8 ? 16384 : 8192;   // one weight tile in shared memory
    constexpr uint32_t kMats = MODE == kGateUp ? 2 : 1;  // weight tiles per stage: gate and up
    extern __shared__ uint8_t raw[];
    uint8_t *base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    Ctrl &c = *reinterpret_cast<Ctrl *>(base);
    uint8_t *sfb_all = base + kCtrlBytes;
    uint8_t *ring = sfb_all + (MODE == kDense ? 0 : a.sfb_bytes);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = blockIdx.z;
    volatile int *abort = &c.abort;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < a.stages; i++) {
            mbar_init(smem_u32(&c.full[i]), 1);
            mbar_init(smem_u32(&c.empty[i]), 1);
        }
        mbar_init(smem_u32(&c.done), 1);
        c.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&xmap)) : "memory");
    }

    // ---- what this CTA computes ----
    uint32_t w_tile = blockIdx.x;           // first weight tile along the rows
    uint32_t tokens, tok0 = 0, expert = 0;  // columns: tokens, or pairs of one expert
    const uint32_t kt0 = a.kt * rank / a.split, kt1 = a.kt * (rank + 1) / a.split;
    if (MODE == kDense) {
        tok0 = blockIdx.y * a.nt;
        tokens = min(a.nt, a.m - tok0);
    } else {
        const uint32_t slot = blockIdx.y / a.chunks, chunk = blockIdx.y % a.chunks, pairs = a.m * a.top_k;
        if (threadIdx.x < 8) c.chosen_bits[threadIdx.x] = 0;
        __syncthreads();
        grid_dep_wait();  // the router's choice, or the hidden vectors, of the kernel before
        for (uint32_t i = threadIdx.x; i < pairs; i += kThreads) {
            const uint32_t e = (uint32_t)__ldcg(a.chosen + i);
            atomicOr(&c.chosen_bits[e / 32 % 8], 1u << (e % 32));
        }
        __syncthreads();
        // the slot-th chosen expert
        uint32_t left = slot;
        expert = 0xFFFFFFFFu;
        for (int w = 0; w < 8 && expert == 0xFFFFFFFFu; w++) {
            const uint32_t bits = c.chosen_bits[w], here = __popc(bits);
            if (left < here) expert = w * 32 + __fns(bits, 0, left + 1);
            else left -= here;
        }
        if (expert == 0xFFFFFFFFu) return;  // the same in the whole cluster
        if (warp == 0) {  // its pairs, in order
            uint32_t found = 0;
            for (uint32_t i = 0; i < pairs; i += 32) {
                const bool hit = i + lane < pairs && (uint32_t)__ldcg(a.chosen + i + lane) == expert;
                const uint32_t mask = __ballot_sync(~0u, hit);
                const uint32_t at = found + __popc(mask & ((1u << lane) - 1));
                if (hit && at / kChunk == chunk) c.pairs[at % kChunk] = i + lane;
                found += __popc(mask);
            }
            if (lane == 0) c.count = found > chunk * kChunk ? min(found - chunk * kChunk, (uint32_t)kChunk) : 0;
        }
        __syncthreads();
        tokens = c.count;
        if (!tokens) return;
        w_tile = (expert * a.row_tiles + blockIdx.x) * kMats;
    }
    const uint32_t n_cols = (tokens * P + 7) / 8 * 8;
    const uint32_t sfb_tiles = MODE == kDense ? (n_cols + 127) / 128 : 1;
    const uint32_t sf_cols = 4 * kMats + (a.nt * P > 128 ? 8 : 4);

    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem)),
                     "r"(a.tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (MODE != kDense) {
        // the columns' rows of pieces, and all their scales of this CTA's share of K
        for (uint32_t i = threadIdx.x; i < n_cols; i += kThreads) {
            const uint32_t t = min(i / P, tokens - 1);  // columns past the last token repeat it
            const uint32_t src = MODE == kGateUp ? c.pairs[t] / a.top_k : c.pairs[t];
            const uint32_t row = src * P + (i / P < tokens ? i % P : 0);
            c.rows[i] = (int32_t)row;
            const uint32_t *s = reinterpret_cast<const uint32_t *>(a.x_scales) + (size_t)row * a.kt;
            for (uint32_t t2 = kt0; t2 < kt1; t2++)
                *reinterpret_cast<uint32_t *>(sfb_all + (t2 - kt0) * kMxScaleTile + i % 32 * 16 + i / 32 * 4) = __ldcg(s + t2);
        }
        fence_proxy_async();  // read by the tensor core's scale copy
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (MODE == kGateUp) grid_dep_launch();  // every CTA holds its TMEM: the next kernel's may come
    const uint32_t tmem = c.tmem;
    const uint32_t iters = kt1 - kt0;

    if (warp == 0 && lane == 0) {
        // ---- TMA ----
        // a copy that unpacks counts the bytes that it read, 64 a row, for either kind
        const uint32_t stage_tx = kMats * (kMxCodeTile + kMxScaleTile) +
                                  (MODE == kDense ? (KIND == 8 ? a.b_box_bytes : sfb_tiles * a.b_box_bytes) + sfb_tiles * kMxScaleTile
                                                  : n_cols * 128);
        auto load_w = [&](uint32_t it) {
            const uint32_t s = it % a.stages, bar = smem_u32(&c.full[s]);
            const uint32_t st = smem_u32(ring + s * a.stage_bytes), sf = st + kMats * kA + a.b_bytes;
            mbar_expect(bar, stage_tx);
#pragma unroll
            for (uint32_t i = 0; i < kMats; i++) {
                const size_t t = (size_t)(w_tile + i) * a.kt + kt0 + it;
                tma_2d(st + i * kA, &wmap, 0, (int)(t * 128), bar);
                bulk_copy(sf + i * kMxScaleTile, a.w_scales + t * kMxScaleTile, kMxScaleTile, bar);
            }
        };
        auto load_x = [&](uint32_t it) {
            const uint32_t s = it % a.stages, bar = smem_u32(&c.full[s]);
            const uint32_t st = smem_u32(ring + s * a.stage_bytes), b = st + kMats * kA, sf = b + a.b_bytes + kMats * kMxScaleTile;
            const uint32_t k = kt0 + it;
            if (MODE != kDense) {
                for (uint32_t i = 0; i < n_cols; i += 4)
                    tma_gather4(b + i * 128, &xmap, (int)(k * 128), *reinterpret_cast<const int4 *>(&c.rows[i]), bar);
            } else if (KIND == 8) {
                const uint32_t row = tok0 / a.group * 256 + tok0 % a.group * P;
                tma_2d(b, &xmap, (int)(k * 128), (int)row, bar);
                for (uint32_t i = 0; i < sfb_tiles; i++)
                    bulk_copy(sf + i * kMxScaleTile, a.x_scales + ((size_t)(row / 128 + i) * a.kt + k) * kMxScaleTile, kMxScaleTile, bar);
            } else {
                for (uint32_t i = 0; i < sfb_tiles; i++) {
                    const size_t t = (size_t)(tok0 / 128 + i) * a.kt + k;
                    tma_2d(b + i * a.b_box_bytes, &xmap, 0, (int)(t * 128), bar);
                    bulk_copy(sf + i * kMxScaleTile, a.x_scales + t * kMxScaleTile, kMxScaleTile, bar);
                }
            }
        };
        // weights do not depend on the kernel before: the ring's first round of them goes out at once
        const uint32_t ahead = min(a.stages, iters);
        uint32_t issued = ahead;
        for (uint32_t it = 0; it < ahead; it++) load_w(it);
        if (MODE == kDense && KIND == 8) grid_dep_wait();  // the pieces
        for (uint32_t it = 0; it < ahead; it++) load_x(it);
        for (uint32_t it = ahead; it < iters; it++) {
            if (!mbar_wait(smem_u32(&c.empty[it % a.stages]), (it / a.stages & 1) ^ 1, abort, 601)) break;
            load_w(it);
            load_x(it);
            issued = it + 1;
        }
        if (*abort)  // no copy may land after this CTA has left
            for (uint32_t it = issued > a.stages ? issued - a.stages : 0; it < issued; it++)
                for (int i = 0; i < 1000 && !mbar_try_wait(smem_u32(&c.full[it % a.stages]), it / a.stages & 1, 1000000); i++) {
                }
    } else if (warp == 1 && lane == 0) {
        // ---- MMA ----
        const uint32_t sf_tmem = tmem + a.d_cols * kMats;
        bool ok = true;
        for (uint32_t it = 0; it < iters; it++) {
            const uint32_t s = it % a.stages;
            if (!mbar_wait(smem_u32(&c.full[s]), it / a.stages & 1, abort, 602)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t st = smem_u32(ring + s * a.stage_bytes), b = st + kMats * kA, sf = b + a.b_bytes;
            // each stage has scale columns of its own: they are rewritten only after its MMAs are done
            const uint32_t sfa = sf_tmem + s * sf_cols, sfb = sfa + 4 * kMats;
#pragma unroll
            for (uint32_t i = 0; i < kMats; i++) scales_to_tmem(sfa + 4 * i, sf + i * kMxScaleTile);
            if (MODE == kDense)
                for (uint32_t i = 0; i < sfb_tiles; i++) scales_to_tmem(sfb + 4 * i, sf + (kMats + i) * kMxScaleTile);
            else
                scales_to_tmem(sfb, smem_u32(sfb_all + it * kMxScaleTile));
            const uint64_t bd = operand_desc<KIND>(b);
            const uint32_t idesc = scaled_instr_desc<KIND>(n_cols);
#pragma unroll
            for (uint32_t i = 0; i < kMats; i++) {
                const uint64_t ad = operand_desc<KIND>(st + i * kA);
#pragma unroll
                for (uint32_t j = 0; j < (KIND == 8 ? 4 : 2); j++) {   // 32 bytes of each row at a time
                    const uint32_t id = KIND == 8 ? j : 2 * j;         // which of the four scale bytes
                    mma_scaled<KIND>(tmem + i * a.d_cols, ad + 2 * j, bd + 2 * j, idesc | id << 4 | id << 29, sfa + 4 * i, sfb,
                                     it | j);
                }
            }
            mma_commit(smem_u32(&c.empty[s]));
        }
        mma_commit(smem_u32(&c.done));
        if (!ok) mbar_wait(smem_u32(&c.done), 0, &c.abort, 603);
    }
    __syncwarp();

    // ---- epilogue: thread = weight row ----
    const uint32_t q = warp % 4, row = blockIdx.x * 128 + q * 32 + lane;
    const bool epi = warp >= 2;
    float *red = reinterpret_cast<float *>(ring);   // [token][128] per matrix, once the ring is idle

    auto finish = [&](uint32_t i, float g, float u) {
        if (MODE == kDense) {
            if (row < a.n) put_as(a.y, a.type, (tok0 + i) * a.stride + row, g);
        } else if (MODE == kGateUp) {
            // The hidden value and its pieces. A warp's 32 rows are one block along the next
            // product's K. Three pieces keep 12 bits of it: past what x and y hold in either type.
            const float h = g / (1.0f + expf(-g)) * u;
            const uint32_t top = __reduce_max_sync(~0u, __float_as_uint(h) & 0x7FFFFFFFu);
            const uint32_t s = mx_piece_scale(__uint_as_float(top), kMxHiddenPieces);
            float left = h * __uint_as_float((254u - min(s, 253u)) << 23);
            const size_t r = (size_t)c.pairs[i] * kMxHiddenPieces, kt = a.row_tiles;
#pragma unroll
            for (int p = 0; p < kMxHiddenPieces; p++) {
                float back;
                const uint32_t code = mx_e4m3(left, &back);
                left = (left - back) * 16.0f;
                a.h_pieces[(r + p) * kt * 128 + row] = s == 255 ? 0 : (uint8_t)code;
                if (lane == 0) a.h_scales[(r + p) * kt * 4 + row / 32] = (uint8_t)mx_piece_scale_of(s, p);
            }
        } else {
            // Weighted, to the pair's own place; the warp whose pair comes last for a token adds the
            // token's top_k parts in their order, so the sum does not depend on who that is.
            const uint32_t pair = c.pairs[i], t = pair / a.top_k;
            if (row < a.n) a.partial[(size_t)pair * a.n + row] = g * __ldcg(a.weight + pair);
            __threadfence();
            __syncwarp();
            uint32_t before = 0;
            if (lane == 0) before = atomicAdd(a.arrived + ((size_t)t * a.row_tiles + blockIdx.x) * 4 + q, 1u);
            if (__shfl_sync(~0u, before, 0) == a.top_k - 1) {
                __threadfence();
                if (row < a.n) {
                    float sum = 0.0f;
                    for (uint32_t j = 0; j < a.top_k; j++) sum += __ldcg(a.partial + (size_t)(t * a.top_k + j) * a.n + row);
                    put_as(a.y, a.type, t * a.stride + row, sum);
                }
            }
        }
    };

    if (epi) {
        mbar_wait(smem_u32(&c.done), 0, abort, 604);
        tc_fence_after();
        const uint32_t taddr = tmem + (q * 32 << 16);
        for (uint32_t i0 = 0; i0 < tokens; i0 += 8) {
            float g[8], u[8];
            load_tokens<P>(taddr + i0 * P, g);
            if (MODE == kGateUp) load_tokens<P>(taddr + a.d_cols + i0 * P, u);
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
                if (i0 + i >= tokens) break;
                if (a.split == 1) {
                    finish(i0 + i, g[i], MODE == kGateUp ? u[i] : 0.0f);
                } else {
                    red[(i0 + i) * 128 + q * 32 + lane] = g[i];
                    if (MODE == kGateUp) red[(a.nt + i0 + i) * 128 + q * 32 + lane] = u[i];
                }
            }
        }
        tc_fence_before();
    }
    if (a.split > 1) {
        // the cluster's partial tiles, added in rank order through distributed shared memory
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (epi)
            for (uint32_t i = rank; i < tokens; i += a.split) {
                float g = 0.0f, u = 0.0f;
                for (uint32_t r = 0; r < a.split; r++) {
                    const float *other = cluster.map_shared_rank(red, r);
                    g += other[i * 128 + q * 32 + lane];
                    if (MODE == kGateUp) u += other[(a.nt + i) * 128 + q * 32 + lane];
                }
                finish(i, g, u);
            }
        __syncwarp();
        cluster.sync();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols));
    }
}

// ---- activation pieces of a dense product ---------------------------------------------------------
//
// 16 lanes take one row's 128 values, 8 each (as the quantiser does), and write P rows of e4m3.
// Token t's pieces are rows t / group * 256 + t % group * P + p, so that a full tile of tokens
// starts on a scale tile.

template <typename T, int P>
__global__ void __launch_bounds__(256) pieces_kernel(const T *x, uint32_t m, uint32_t k, uint64_t stride, uint32_t kt,
                                                     uint32_t group, uint8_t *pieces, uint8_t *scales, bool vec) {
    grid_dep_launch();  // the product may start on its weights
    const uint32_t lane = threadIdx.x % 16, units = m * kt;
    const uint32_t step = gridDim.x * (blockDim.x / 16), first = (blockIdx.x * blockDim.x + threadIdx.x) / 16;
    for (uint32_t base = first & ~1u; base < units; base += step) {
        const uint32_t un = base + (first & 1u);
        const bool live = un < units;
        const uint32_t t = live ? un / kt : 0, tile = live ? un - t * kt : 0, j = tile * kMxTile + lane * 8;
        const uint32_t left = live && j < k ? k - j : 0;
        const T *src = x + t * stride + j;
        float v[8];
        if (vec && left >= 8) {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(src));
            const T *h = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = mx_float(h[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = (uint32_t)i < left ? mx_float(src[i]) : 0.0f;
        }
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);  // NaN above infinity above all
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        const uint32_t s = mx_piece_scale(__uint_as_float(top), P);
        const float inverse = __uint_as_float((254u - min(s, 253u)) << 23);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= inverse;
        const uint32_t row = t / group * 256 + t % group * P;
#pragma unroll
        for (int p = 0; p < P; p++) {
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float back;
                w[i / 4] |= mx_e4m3(v[i], &back) << (i % 4 * 8);
                v[i] = (v[i] - back) * 16.0f;
            }
            const uint32_t sp = mx_piece_scale_of(s, p);
            uint32_t all = sp | __shfl_down_sync(~0u, sp, 4) << 8;
            all |= __shfl_down_sync(~0u, all, 8) << 16;
            if (live) {
                const uint32_t r = row + p;
                *reinterpret_cast<uint2 *>(pieces + ((size_t)r * kt + tile) * 128 + lane * 8) =
                    s == 255 ? make_uint2(0, 0) : make_uint2(w[0], w[1]);
                if (lane == 0) *reinterpret_cast<uint32_t *>(scales + mx_scale_at(r, tile * 4, kt)) = all;
            }
        }
    }
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

// Weight tiles: 64 bytes of codes a row, tiles of 128 rows one after another.
template <int KIND>
cudaError_t encode_weights(CUtensorMap *map, const uint8_t *codes, uint64_t tiles) {
    if (KIND == 8)
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, codes, 128, tiles * 128, 64, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, 64, tiles * 128, 64, 64, 128, CU_TENSOR_MAP_SWIZZLE_64B);
}

uint32_t up_to(uint32_t v, uint32_t to) { return (v + to - 1) / to * to; }
uint32_t pow2_cols(uint32_t v) {
    uint32_t c = 32;
    while (c < v) c *= 2;
    return c;
}

template <int KIND, int P, int MODE>
cudaError_t launch(const CUtensorMap &wmap, const CUtensorMap &xmap, const TcArgs &a, dim3 grid, uint32_t smem, bool dependent,
                   cudaStream_t s) {
    auto kernel = mx_tc_kernel<KIND, P, MODE>;
    if (!once_per_device(100 + KIND * 16 + P * 4 + MODE, [&] {
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
    attr[0].val.programmaticStreamSerializationAllowed = dependent ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = a.split;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, wmap, xmap, a);
}

// Ring depth and shared memory for `per_sm` CTAs on an SM.
template <int KIND, int P, int MODE>
uint32_t plan_ring(TcArgs &a, uint32_t per_sm) {
    const uint32_t mats = MODE == kGateUp ? 2 : 1, n = up_to(a.nt * P, 8);
    // KIND 4 copies whole boxes of 128 rows past the first 128 columns
    a.b_bytes = KIND == 8 ? n * 128 : n <= 128 ? up_to(n * 64, 1024) : up_to(n, 128) * 64;
    const uint32_t sf = kMxScaleTile * (mats + (MODE == kDense ? (n + 127) / 128 : 0));
    a.stage_bytes = up_to(mats * (KIND == 8 ? 16384 : 8192) + a.b_bytes + sf, 1024);
    a.d_cols = up_to(a.nt, 8) * P;
    const uint32_t sf_cols = 4 * mats + (a.nt * P > 128 ? 8 : 4);
    const uint32_t extra = 1024 + kCtrlBytes + a.sfb_bytes;
    const uint32_t budget = (per_sm == 1 ? 226 : per_sm == 2 ? 112 : 74) * 1024 - extra;
    const uint32_t cols = per_sm == 1 ? 512 : per_sm == 2 ? 256 : 128;
    a.stages = std::min<uint32_t>({budget / a.stage_bytes, (cols - a.d_cols * mats) / sf_cols, (uint32_t)kMaxStages,
                                   std::max(1u, (a.kt + a.split - 1) / a.split)});
    a.tmem_cols = pow2_cols(a.d_cols * mats + a.stages * sf_cols);
    const uint32_t red = a.split > 1 ? mats * a.nt * 128 * 4 : 0;
    return extra + std::max(a.stages * a.stage_bytes, red);
}

template <int KIND, int P>
cudaError_t dense(const MxProductArgs &p, const uint8_t *x, const uint8_t *x_scales, cudaStream_t s) {
    const uint32_t kt = mx_tiles(p.k), rt = mx_tiles(p.n);
    constexpr uint32_t kGroup = P == 1 ? 256 : P == 2 ? 128 : 64;   // tokens that fill 256 columns (P = 3: 192)
    TcArgs a{};
    a.m = p.m;
    a.n = p.n;
    a.kt = kt;
    a.group = kGroup;
    a.nt = p.m < kGroup ? p.m : kGroup;
    const uint32_t tt = (p.m + a.nt - 1) / a.nt;
    const uint32_t per_sm = up_to(a.nt, 8) * P <= 128 ? 2 : 1;
    a.split = 1;
    while (a.split < 8 && rt * tt * a.split * 2 <= 148 * per_sm && kt / (a.split * 2) >= 2 && a.nt <= 64) a.split *= 2;
    a.w_scales = p.w_scales;
    a.x_scales = x_scales;
    a.y = p.y;
    a.type = p.type;
    a.stride = p.stride;
    const uint32_t smem = plan_ring<KIND, P, kDense>(a, per_sm);
    CUtensorMap wmap, xmap;
    cudaError_t e = encode_weights<KIND>(&wmap, p.w_codes, (uint64_t)rt * kt);
    if (e != cudaSuccess) return e;
    const uint32_t n = up_to(a.nt * P, 8);
    if (KIND == 8) {
        const uint64_t rows = (uint64_t)(p.m / kGroup) * 256 + p.m % kGroup * P;
        a.b_box_bytes = n * 128;
        e = encode(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, (uint64_t)kt * 128, rows, (uint64_t)kt * 128, 128, n,
                   CU_TENSOR_MAP_SWIZZLE_128B);
    } else {
        const uint32_t box = n < 128 ? n : 128;
        a.b_box_bytes = box * 64;
        e = encode(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, 64, (uint64_t)mx_tiles(p.m) * kt * 128, 64, 64, box,
                   CU_TENSOR_MAP_SWIZZLE_64B);
    }
    if (e != cudaSuccess) return e;
    return launch<KIND, P, kDense>(wmap, xmap, a, dim3(rt, tt, a.split), smem, KIND == 8, s);
}

template <typename T, int P>
cudaError_t dense_x16(const MxProductArgs &p, cudaStream_t s) {
    const uint32_t kt = mx_tiles(p.k), units = p.m * kt;
    constexpr uint32_t kGroup = P == 2 ? 128 : 64;
    uint8_t *pieces = static_cast<uint8_t *>(p.workspace);
    const size_t rows = mx_piece_rows(p.m, p.x_type);
    uint8_t *scales = pieces + (rows * kt * 128 + 255) / 256 * 256;
    const bool vec = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.x_stride % 8 == 0;
    const unsigned grid = std::min<unsigned>((units + 15) / 16, 148 * 8);
    pieces_kernel<T, P><<<grid, 256, 0, s>>>(static_cast<const T *>(p.x), p.m, p.k, p.x_stride, kt, kGroup, pieces, scales, vec);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : dense<8, P>(p, pieces, scales, s);
}

template <int P, int MODE>
cudaError_t expert_product(const MxExpertsArgs &e, cudaStream_t s) {
    const uint32_t width = MODE == kGateUp ? e.d : e.f, rows = MODE == kGateUp ? e.f : e.d;
    TcArgs a{};
    a.m = e.tokens;
    a.n = rows;
    a.kt = mx_tiles(width);
    a.row_tiles = mx_tiles(rows);
    a.nt = std::min<uint32_t>(e.tokens, kChunk);
    a.chunks = (e.tokens + kChunk - 1) / kChunk;
    a.experts = e.experts;
    a.top_k = e.top_k;
    a.chosen = e.ws.chosen;
    a.weight = e.ws.weight;
    a.arrived = e.ws.arrived;
    a.h_pieces = e.ws.h_pieces;
    a.h_scales = e.ws.h_scales;
    a.partial = e.ws.partial;
    a.x_scales = MODE == kGateUp ? e.ws.x_scales : e.ws.h_scales;
    a.w_scales = MODE == kGateUp ? e.gate_up_scales : e.down_scales;
    a.y = e.y;
    a.type = e.type;
    a.stride = e.y_stride;
    const uint32_t slots = std::min(e.experts, e.tokens * e.top_k);
    a.split = 1;
    while (a.split < 8 && a.kt / (a.split * 2) >= 2 &&
           (a.row_tiles * slots * a.split * 2 <= 148 * 2 || a.kt / a.split > 32))
        a.split *= 2;
    a.sfb_bytes = up_to((a.kt + a.split - 1) / a.split * kMxScaleTile, 1024);
    const uint32_t smem = plan_ring<8, P, MODE>(a, 2);
    const uint32_t mats = MODE == kGateUp ? 2 : 1;
    CUtensorMap wmap, xmap;
    cudaError_t r = encode_weights<8>(&wmap, MODE == kGateUp ? e.gate_up_codes : e.down_codes,
                                      (uint64_t)e.experts * a.row_tiles * mats * a.kt);
    if (r != cudaSuccess) return r;
    const uint64_t piece_rows = MODE == kGateUp ? (uint64_t)e.tokens * P : (uint64_t)e.tokens * e.top_k * P;
    r = encode(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, MODE == kGateUp ? e.ws.x_pieces : e.ws.h_pieces, (uint64_t)a.kt * 128,
               piece_rows, (uint64_t)a.kt * 128, 128, 1, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != cudaSuccess) return r;
    return launch<8, P, MODE>(wmap, xmap, a, dim3(a.row_tiles, slots * a.chunks, a.split), smem, true, s);
}

}  // namespace

size_t mx_piece_rows(uint32_t m, int x_type) {
    const uint32_t p = mx_pieces(x_type), group = p == 2 ? 128 : 64;
    return (size_t)(m / group) * 256 + m % group * p;
}

cudaError_t launch_mx4_product(const MxProductArgs &a, cudaStream_t s) {
    if (!a.x) return dense<4, 1>(a, a.a_codes, a.a_scales, s);
    if (a.x_type == 1) return dense_x16<__half, 3>(a, s);
    return dense_x16<__nv_bfloat16, 2>(a, s);
}

cudaError_t launch_mx4_expert_products(const MxExpertsArgs &a, cudaStream_t s) {
    const cudaError_t e = a.type == 1 ? expert_product<3, kGateUp>(a, s) : expert_product<2, kGateUp>(a, s);
    return e != cudaSuccess ? e : expert_product<kMxHiddenPieces, kDown>(a, s);
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
