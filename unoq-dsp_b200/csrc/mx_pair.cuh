// mx_pair.cuh -- the MX4 product of many tokens (included by mx_tc.cu): pairs of CTAs.
//
// At 256 columns a tile of mx_tc_kernel reads 26 KB of operands per 128 x 256 x 128 block, 102 bytes a
// cycle and SM at the rate of the 4-bit tensor cores; the L2 delivers 64 (18.3 TB/s measured).
// A pair of CTAs (tcgen05 cta_group::2) multiplies 256 weight rows by 256 columns: each CTA loads its own
// 128 rows and half of the columns, both tensor cores read both halves, and the traffic falls to
// 17 KB for as much work of an SM. The kernel is persistent, one pair to two SMs. Its epilogue (8 warps) first
// takes a tile's accumulators into registers, which gives TMEM back to the MMAs within some hundred
// cycles, and writes them while the next tile is multiplied.
#pragma once

struct PairArgs {
    uint32_t m, n, steps, kw, rt;         // tokens, weight rows, stages and code tiles along K, row tiles
    uint32_t row_pairs, tiles;            // pairs of row tiles; times token tiles
    uint32_t stages, stage_bytes, group;
    void *y;
    int type;
    uint64_t stride;
    bool wide;                            // 16-bit y whose rows start on 16 bytes
};

struct PairCtrl {
    unsigned long long full[kMaxStages], empty[kMaxStages], acc_full, acc_empty, spare;
    uint32_t tmem;
    int abort;
};

constexpr uint32_t kPairOut = 32 * 256;   // 32 tokens of a tile's 128 16-bit values, for each half of the epilogue
constexpr int kPairThreads = 352;   // warp 0: weight copies, 1: MMA, 2-9: epilogue, 10: activation copies

__device__ __forceinline__ uint32_t in_leader(uint32_t smem) {   // the same place in the pair's first CTA
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem));
    return a;
}
// An arrival in the other CTA that orders nothing but TMEM reads (by the tcgen05 fences around it): one with
// release semantics waits for the warp's earlier stores, 1500 cycles and more.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Copies that complete on a barrier of the pair's first CTA, whichever CTA of the two they are issued in and written to.
__device__ __forceinline__ void pair_tma_2d(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::
            "r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void pair_tma_3d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}
// Arrives on the barriers at this place in both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void pair_commit(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void pair_scales_to_tmem(uint32_t tmem, uint32_t smem) {
    const uint64_t desc = (uint64_t)((smem >> 4) & 0x3FFF) | (1ull << 16) | (8ull << 32) | (1ull << 46);
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc));
}
template <int KIND>
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t acc) {
    if (KIND == 8)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc));
}

template <int KIND, int P>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    mx_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                   const __grid_constant__ CUtensorMap wsmap, const __grid_constant__ CUtensorMap xsmap, const PairArgs a) {
    constexpr uint32_t kTokens = P == 1 ? 256 : P == 2 ? 128 : 64, kN = kTokens * P;
    constexpr uint32_t kB = kN / 2 * 128;                          // this CTA's half of the columns
    constexpr uint32_t kSub = KIND == 8 ? 1 : 2, kSf = kSub * kMxScaleTile;   // scales of a stage, per 128 rows
    constexpr uint32_t kSfCols = kSub * (4 + 8);
    extern __shared__ uint8_t raw[];
    uint8_t *base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    PairCtrl &c = *reinterpret_cast<PairCtrl *>(base);
    uint8_t *out = base + kCtrlBytes, *ring = out + 2 * kPairOut;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = blockIdx.x % 2, pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    volatile int *abort = &c.abort;
    cg::cluster_group cluster = cg::this_cluster();

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kMaxStages; i++) {
            mbar_init(smem_u32(&c.full[i]), 2);
            mbar_init(smem_u32(&c.empty[i]), 1);
        }
        mbar_init(smem_u32(&c.acc_full), 1);
        mbar_init(smem_u32(&c.acc_empty), 16);   // the epilogue warps of both CTAs
        mbar_init(smem_u32(&c.spare), 1);
        c.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&xmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wsmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&xsmap)) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem)), "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    tc_fence_before();
    cluster.sync();
    tc_fence_after();
    const uint32_t tmem = c.tmem, stages = a.stages, stage_bytes = a.stage_bytes;
    // On the way out of an abort no copy may land after this CTA has left, and the barriers are the first
    // CTA's: about a millisecond is a thousand times what the last ones take.
    auto drain = [&]() {
        for (const long long start = clock64(); clock64() - start < 2000000;) {
        }
    };

    if (warp == 0 && elect_one()) {
        // ---- weight tiles and their scales: both CTAs' complete on the first one's barriers, which it alone arms ----
        if (KIND == 4) grid_dep_wait();   // the kernel before may have written them; KIND 8's is the one that makes pieces
        const uint32_t st0 = smem_u32(ring), full0 = in_leader(smem_u32(&c.full[0])), empty0 = smem_u32(&c.empty[0]);
        uint32_t st = st0, full = full0, empty = empty0, s = 0, phase = 1;
        for (uint32_t t = pair; t < a.tiles; t += pairs) {
            // the row tile past an odd number of them: past the matrix, zeros
            const uint32_t tile = 2 * (t % a.row_pairs) + rank;
            int x = 0, y = (int)(tile * a.kw * 128), sf = (int)(tile * 2 * a.kw);
            for (uint32_t k = 0; k < a.steps; k++, sf += kSub) {
                if (!mbar_poll(empty, phase, abort, 611)) goto weights_out;
                // an unpacking copy counts what it reads
                if (rank == 0) mbar_expect(smem_u32(&c.full[s]), 2 * ((KIND == 8 ? kMxCodeTile / 2 : kMxCodeTile) + kSf));
                pair_tma_2d(st, &wmap, x, y, full);
                pair_tma_2d(st + kA + kB, &wsmap, 0, sf, full);
                if (KIND == 8) x ^= 128;
                if (x == 0) y += 128;
                st += stage_bytes, full += 8, empty += 8;
                if (++s == stages) s = 0, phase ^= 1, st = st0, full = full0, empty = empty0;
            }
        }
    weights_out:
        if (*abort) drain();
    } else if (warp == 10 && elect_one()) {
        // ---- this CTA's half of the columns, and the scales of all of them ----
        grid_dep_wait();
        const uint32_t st0 = smem_u32(ring) + kA, full0 = in_leader(smem_u32(&c.full[0])), empty0 = smem_u32(&c.empty[0]);
        uint32_t st = st0, full = full0, empty = empty0, s = 0, phase = 1;
        for (uint32_t t = pair; t < a.tiles; t += pairs) {
            const int tt = (int)(t / a.row_pairs);   // 256 rows of codes or pieces, two scale tiles, to a token tile
            const int row = tt * 256 + (int)rank * (int)(kN / 2);
            int x = KIND == 8 ? 0 : (2 * tt + (int)rank) * (int)a.kw * 128;
            for (uint32_t k = 0; k < a.steps; k++, x += 128) {
                if (!mbar_poll(empty, phase, abort, 618)) goto columns_out;
                if (rank == 0) mbar_expect(smem_u32(&c.full[s]), 2 * (kB + 2 * kSf));
                if (KIND == 8) pair_tma_2d(st, &xmap, x, row, full);
                else pair_tma_2d(st, &xmap, 0, x, full);
                pair_tma_3d(st + kB + kSf, &xsmap, 0, (int)(k * kSub), 2 * tt, full);
                st += stage_bytes, full += 8, empty += 8;
                if (++s == stages) s = 0, phase ^= 1, st = st0, full = full0, empty = empty0;
            }
        }
    columns_out:
        if (*abort) drain();
    } else if (warp == 1 && rank == 0 && elect_one()) {
        // ---- MMA of the pair ----
        const uint32_t idesc = scaled_instr_desc<KIND>(256, kN);
        const uint32_t st0 = smem_u32(ring), full0 = smem_u32(&c.full[0]), empty0 = smem_u32(&c.empty[0]);
        const uint32_t sf0 = tmem + kN;
        uint32_t st = st0, full = full0, empty = empty0, sfa = sf0, s = 0, phase = 0, nth = 0;
        bool ok = true;
        for (uint32_t t = pair; ok && t < a.tiles; t += pairs, nth++) {
            if (nth && !mbar_poll(smem_u32(&c.acc_empty), (nth - 1) & 1, abort, 617)) break;
            for (uint32_t k = 0; k < a.steps; k++) {
                if (!mbar_poll(full, phase, abort, 612)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t b = st + kA, sf = b + kB, sfb = sfa + 4 * kSub;
#pragma unroll
                for (uint32_t h = 0; h < kSub; h++) {
                    pair_scales_to_tmem(sfa + 4 * h, sf + h * kMxScaleTile);
                    pair_scales_to_tmem(sfb + 8 * h, sf + kSf + h * kMxScaleTile);
                    pair_scales_to_tmem(sfb + 8 * h + 4, sf + 2 * kSf + h * kMxScaleTile);
                }
                const uint64_t ad = smem_desc(st), bd = smem_desc(b);
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {   // 32 bytes of each row at a time
                    const uint32_t h = KIND == 8 ? 0 : j / 2, id = KIND == 8 ? j : j % 2 * 2;   // which scale bytes
                    pair_mma<KIND>(tmem, ad + 2 * j, bd + 2 * j, idesc | id << 4 | id << 29, sfa + 4 * h, sfb + 8 * h, k | j);
                }
                pair_commit(empty);
                st += stage_bytes, full += 8, empty += 8, sfa += kSfCols;
                if (++s == stages) s = 0, phase ^= 1, st = st0, full = full0, empty = empty0, sfa = sf0;
            }
            pair_commit(smem_u32(&c.acc_full));
        }
        if (!ok || *abort) {   // the MMAs that were issued end before TMEM is freed
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&c.spare))
                         : "memory");
            for (int i = 0; i < 100 && !mbar_try_wait(smem_u32(&c.spare), 0, 1000000); i++) {
            }
        }
    } else if (warp >= 2 && warp < 10) {
        // ---- epilogue: thread = weight row, half of the tile's tokens ----
        constexpr uint32_t kMine = kTokens / 2, kAt = P == 3 ? 8 : 32 / P;
        const uint32_t q = warp % 4, half = (warp - 2) / 4;
        uint32_t nth = 0;
        for (uint32_t t = pair; t < a.tiles; t += pairs, nth++) {
            const uint32_t rp = t % a.row_pairs, tt = t / a.row_pairs;
            if (!mbar_poll(smem_u32(&c.acc_full), nth & 1, abort, 615)) break;
            tc_fence_after();
            const uint32_t taddr = tmem + (q * 32 << 16) + half * kMine * P;
            float v[kMine];
#pragma unroll
            for (uint32_t i = 0; i < kMine; i += kAt) {
                float w[kAt];
                load_tokens<P>(taddr + i * P, w);
#pragma unroll
                for (uint32_t j = 0; j < kAt; j++) v[i + j] = w[j];
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(in_leader(smem_u32(&c.acc_empty)));
            const uint32_t row = (2 * rp + rank) * 128 + q * 32 + lane, tok = tt * kTokens + half * kMine;
            if (!a.wide) {
                if (row < a.n && tok < a.m) put_tokens_as(a.y, a.type, tok * a.stride + row, a.stride, v, a.m - tok);
                continue;
            }
            // 32 tokens at a time through shared memory, so that 16 lanes write a token's 256 bytes: a warp's own 32
            // rows would go out as half lines, which took the loads 10 us of 4096 x 8192 x 4096's 62
            constexpr uint32_t kOut = kMine < 32 ? kMine : 32;
            const uint32_t row0 = (2 * rp + rank) * 128, at = q * 32 + lane;
            uint16_t *to = reinterpret_cast<uint16_t *>(out + half * kPairOut);
#pragma unroll
            for (uint32_t i0 = 0; i0 < kMine; i0 += kOut) {
                if (tok + i0 >= a.m) break;   // the same for all of the half
                asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");   // the tokens before are out
#pragma unroll
                for (uint32_t j = 0; j < kOut; j++) {
                    const float f = v[i0 + j];
                    to[j * 128 + at] = a.type == 1 ? __half_as_ushort(__float2half_rn(f)) : __bfloat16_as_ushort(__float2bfloat16_rn(f));
                }
                asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
#pragma unroll
                for (uint32_t j = at / 16; j < kOut; j += 8) {
                    const uint32_t t = tok + i0 + j, r = row0 + at % 16 * 8;
                    if (t >= a.m || r >= a.n) continue;
                    const uint16_t *from = to + j * 128 + at % 16 * 8;
                    uint16_t *y = static_cast<uint16_t *>(a.y) + t * a.stride + r;
                    if (r + 8 <= a.n) *reinterpret_cast<uint4 *>(y) = *reinterpret_cast<const uint4 *>(from);
                    else
                        for (uint32_t b = 0; r + b < a.n; b++) y[b] = from[b];
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    cluster.sync();   // no arrival or copy goes to a CTA that has left
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

template <int KIND, int P>
cudaError_t pair_product(const MxProductArgs &p, const uint8_t *x, const uint8_t *x_scales, cudaStream_t s) {
    constexpr uint32_t kTokens = P == 1 ? 256 : P == 2 ? 128 : 64, kN = kTokens * P, kB = kN / 2 * 128, kSub = KIND == 8 ? 1 : 2;
    PairArgs a{};
    a.m = p.m;
    a.n = p.n;
    a.kw = mx_ktiles(p.k) / 2;
    a.steps = KIND == 8 ? mx_tiles(p.k) : a.kw;
    a.rt = mx_tiles(p.n);
    a.row_pairs = (a.rt + 1) / 2;
    a.tiles = a.row_pairs * ((p.m + kTokens - 1) / kTokens);
    a.stage_bytes = kA + kB + up_to(3 * kSub * kMxScaleTile, 1024);
    a.wide = p.type != 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 && p.stride % 8 == 0;
    const uint32_t extra = 1024 + kCtrlBytes + 2 * kPairOut;
    a.stages = std::min<uint32_t>({(226 * 1024 - extra) / a.stage_bytes, (512 - kN) / (12 * kSub), (uint32_t)kMaxStages});
    a.y = p.y;
    a.type = p.type;
    a.stride = p.stride;
    CUtensorMap wmap, xmap, wsmap, xsmap;
    const uint64_t rows = KIND == 8 ? mx_piece_rows(p.m, p.x_type) : (uint64_t)mx_tiles(p.m) * 128;
    cudaError_t e = encode_weights<KIND>(&wmap, p.w_codes, (uint64_t)a.rt * a.kw);
    if (e != cudaSuccess) return e;
    if (KIND == 8)
        e = encode(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, (uint64_t)a.steps * 128, rows, (uint64_t)a.steps * 128, 128, kN / 2,
                   CU_TENSOR_MAP_SWIZZLE_128B);
    else
        e = encode(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, 128, rows * a.kw, 128, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (e != cudaSuccess) return e;
    // scale tiles as rows of 128 words; a stage's for both tiles of columns in one copy
    e = encode(&wsmap, CU_TENSOR_MAP_DATA_TYPE_UINT32, p.w_scales, 128, (uint64_t)a.rt * 2 * a.kw, kMxScaleTile, 128, kSub,
               CU_TENSOR_MAP_SWIZZLE_NONE);
    if (e != cudaSuccess) return e;
    const cuuint64_t along = a.steps * kSub;
    const cuuint64_t dims[3] = {128, along, (rows + 127) / 128}, strides[2] = {kMxScaleTile, along * kMxScaleTile};
    const cuuint32_t box[3] = {128, kSub, 2}, ones[3] = {1, 1, 1};
    if (encoder()(&xsmap, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<uint8_t *>(x_scales), dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    auto kernel = mx_pair_kernel<KIND, P>;
    if (!once_per_device(90 + P, [&] {
            return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) == cudaSuccess;
        }))
        return cudaErrorInvalidValue;
    const uint32_t sms = (uint32_t)current_sm_count() / 2 * 2;
    return launch_pdl(kPdlMx, kernel, dim3(std::min(2 * a.tiles, sms)), dim3(kPairThreads),
                      (size_t)extra + a.stages * a.stage_bytes, s, wmap, xmap, wsmap, xsmap, a);
}
