// mx_mma.cuh -- device helpers of the MX4 products (mx_tc.cu, mx_pair.cuh): copies, bounded polling,
// block-scaled MMAs, TMEM reads and output rows.
#pragma once
#include "mx.cuh"
#include "tc_common.cuh"

namespace uq {
namespace {

// One thread of a converged warp. The copy and MMA threads are chosen so, and not by their lane number: the
// compiler then knows that one thread runs, and issues a copy in about 15 cycles, not 55.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// Bounded wait that polls: what is waited for is mostly there, or comes within some hundred cycles, and a
// wait with a suspension limit costs 63 cycles even then, a plain one 27, and wakes later.
__device__ __forceinline__ bool mbar_poll(uint32_t bar, uint32_t parity, volatile int *abort, int code) {
    long long start = 0;
    for (uint32_t i = 0;; i++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok)
                     : "r"(bar), "r"(parity)
                     : "memory");
        if (ok) return true;
        if (i % 64 != 63) continue;
        if (*abort) return false;
        if (!start) start = clock64();
        if (clock64() - start > kTimeoutCycles) {
            *abort = 1;
            atomicCAS(&g_tc_error, 0, code);
            return false;
        }
    }
}
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

// Instruction descriptor without the scale bytes' numbers: e8m0 scales, M = 128 or 256 rows.
template <int KIND>
__device__ __forceinline__ uint32_t scaled_instr_desc(uint32_t m, uint32_t n) {
    const uint32_t types = KIND == 8 ? (5u << 7) | (0u << 10) : (1u << 7) | (1u << 10);  // e2m1 x e4m3 | e2m1 x e2m1
    return types | (n >> 3) << 17 | 1u << 23 | (m >> 7) << 27;
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

// N tokens' values of this thread's weight row: the P columns of each, added in 32 bits, the
// smallest piece first.
template <int P, int N>
__device__ __forceinline__ void load_tokens(uint32_t addr, float (&v)[N]) {
    uint32_t r[N * P];
#pragma unroll
    for (int p = 0; p < N * P / 8; p++) tmem_ld8(addr + 8 * p, r + 8 * p);
    tmem_wait(r);
#pragma unroll
    for (int i = 0; i < N; i++) {
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

// `count` tokens' values of one weight row (this thread's), rows of y `stride` apart: the 32 lanes of a
// warp write 32 neighbouring values of a token.
template <typename T, int N>
__device__ __forceinline__ void put_tokens(T *p, uint64_t stride, const float (&v)[N], uint32_t count) {
    if (count >= N) {
#pragma unroll
        for (int i = 0; i < N; i++, p += stride) *p = mx_to<T>(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++, p += stride)
            if ((uint32_t)i < count) *p = mx_to<T>(v[i]);
    }
}
template <int N>
__device__ __forceinline__ void put_tokens_as(void *y, int type, size_t at, uint64_t stride, const float (&v)[N], uint32_t count) {
    if (type == 0) put_tokens(static_cast<float *>(y) + at, stride, v, count);
    else if (type == 1) put_tokens(static_cast<__half *>(y) + at, stride, v, count);
    else put_tokens(static_cast<__nv_bfloat16 *>(y) + at, stride, v, count);
}

}  // namespace
}  // namespace uq
