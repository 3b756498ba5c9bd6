// mx.cuh -- microscaled 4-bit (MX4) operators: layouts, number conversions and launchers shared by
// k_mx.cu (quantisation, packing, activation pieces, router), mx_tc.cu (products) and mx_abi.cu.
//
// Types are UgMxType (0 f32, 1 f16, 2 bf16). Operand layout: code tiles of 128 rows x 256 values, 128
// contiguous bytes a row (copies of 128-byte rows run at 18.3 TB/s from L2, of 64-byte rows at 13.7),
// and scale tiles of 128 rows x 128 values, 512 bytes in the order that the tensor cores' scale copy
// takes (unoq_mx.h).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace uq {

constexpr int kMxTile = 128;          // rows of a tile, values of a scale tile
constexpr int kMxCodeTile = 16384;    // bytes of a code tile, 128 x 256
constexpr int kMxScaleTile = 512;     // bytes of a scale tile, 128 x 128
constexpr int kMxHalf = 64;           // gate rows, and up rows, of a tile of paired matrices
constexpr int kMxHiddenPieces = 4;    // pieces of the hidden vector of ug_mx4_experts
constexpr int kMxRouterCluster = 8;   // CTAs that share one token's router product

__host__ __device__ inline uint32_t mx_tiles(uint32_t n) { return (n + kMxTile - 1) / kMxTile; }
// Scale tiles along a row of k values, two to a code tile.
__host__ __device__ inline uint32_t mx_ktiles(uint32_t k) { return (k + 255) / 256 * 2; }
// Pieces of a 16-bit value: 4 significant bits each, so two hold a bf16 (8) and three an f16 (11).
__host__ __device__ inline int mx_pieces(int type) { return type == 2 ? 2 : 3; }
// Whether the product splits m tokens itself: up to 32 columns of pieces (16 bf16 or 10 f16 tokens), for long rows fewer.
// That is one launch for two, but every CTA splits its share of the rows anew. bf16, a call, in the product and before it:
// 4096 x 4096, 1 token 8.8 us and 13.3, 16 tokens 11.3 and 13.3 (the GPU's time alone 6.6 and 6.2, 11.2 and 6.7);
// 2048 x 8192, 2 tokens 12.1 and 13.1, 4 13.5 and 13.2, 8 16.6 and 13.2; 8192 x 8192, 4 tokens 9.9 and 13.4, 16 18.0 and
// 13.3; 8192 x 16384, 2 tokens 12.5 and 13.1, 6 16.3 and 13.3; 4096 x 65536, 2 tokens 26.7 and 27.8, 6 35.5 and 29.7.
inline bool mx_fused(uint32_t m, uint32_t k, int type) {
    return (uint64_t)m * mx_pieces(type) <= (k <= 4096 ? 32 : 65536 / k);
}

#ifdef __CUDACC__
__device__ __forceinline__ size_t mx_code_at(uint32_t r, uint32_t j, uint32_t kt) {
    return ((size_t)(r / kMxTile) * (kt / 2) + j / 256) * kMxCodeTile + (r % kMxTile) * 128 + j % 256 / 2;
}
__device__ __forceinline__ size_t mx_scale_at(uint32_t r, uint32_t b, uint32_t kt) {
    return ((size_t)(r / kMxTile) * kt + b / 4) * kMxScaleTile + (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4;
}

// 2^(code - 127) of a scale byte; 255 is NaN and 0 the subnormal 2^-127.
__device__ __forceinline__ float mx_scale_value(uint32_t code) {
    return code == 255 ? __int_as_float(0x7FC00000) : __uint_as_float(code ? code << 23 : 0x00400000u);
}

// Eight floats (already divided by the scale) to eight e2m1 codes, the first in the low nibble:
// round to nearest even, saturating at 6.
__device__ __forceinline__ uint32_t mx_pack8(const float (&v)[8]) {
    uint32_t d;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(d)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return d;
}

// Eight e2m1 codes to floats (exact: f16 holds every e2m1 value).
__device__ __forceinline__ void mx_unpack8(uint32_t codes, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// The e2m1 value of the low four bits.
__device__ __forceinline__ float mx_unpack1(uint32_t code) {
    uint32_t h;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(code));
    return __low2float(*reinterpret_cast<const __half2 *>(&h));
}

// Two floats rounded to a pair of 16-bit values, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t mx_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t mx_pair<__half>(float a, float b) {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}
template <>
__device__ __forceinline__ uint32_t mx_pair<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}

// Eight values of a row as they are in memory.
template <typename T>
struct MxRaw {   // 16-bit types, two to a word
    uint32_t w[4];
    // largest magnitude as its 16 bits (NaN above infinity above every number), and that in 32 bits
    __device__ __forceinline__ uint32_t top() const {
        const uint32_t m = __vimax3_u16x2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu,
                                          __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
        return max(m >> 16, m & 0xFFFFu);
    }
    __device__ __forceinline__ static uint32_t top_bits(uint32_t t) {
        return sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? t << 16 : __float_as_uint(__half2float(__ushort_as_half((uint16_t)t)));
    }
    __device__ __forceinline__ void values(float (&v)[8], float scale) const {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float2 f;
            if (__is_same(T, __nv_bfloat16)) {
                f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
            } else {
                f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            }
            v[2 * i] = f.x * scale;
            v[2 * i + 1] = f.y * scale;
        }
    }
    __device__ __forceinline__ void load(const T *p) {
        const uint4 q = *reinterpret_cast<const uint4 *>(p);
        w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    }
    __device__ __forceinline__ void load_some(const T *p, uint32_t left) {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
            w[i] = (2 * i < left ? h[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)h[2 * i + 1] << 16 : 0u);
    }
};
template <>
struct MxRaw<float> {
    uint32_t w[8];
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) m = max(m, w[i] & 0x7FFFFFFFu);
        return m;
    }
    __device__ __forceinline__ static uint32_t top_bits(uint32_t t) { return t; }
    __device__ __forceinline__ void values(float (&v)[8], float scale) const {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __uint_as_float(w[i]) * scale;
    }
    __device__ __forceinline__ void load(const float *p) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p), b = reinterpret_cast<const uint4 *>(p)[1];
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    }
    __device__ __forceinline__ void load_some(const float *p, uint32_t left) {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) w[i] = i < left ? __float_as_uint(p[i]) : 0u;
    }
};

// The same eight columns of n <= ROWS rows, zeros past `left` columns and n rows; `whole`: 16-byte
// aligned and all inside.
template <typename T, int ROWS>
__device__ __forceinline__ void mx_load_rows(MxRaw<T> (&raw)[ROWS], const T *p, uint64_t stride, uint32_t n, uint32_t left,
                                             bool whole) {
    if (whole) {
#pragma unroll
        for (int i = 0; i < ROWS; i++, p += stride) {
            if ((uint32_t)i < n) raw[i].load(p);
            else raw[i].load_some(p, 0);
        }
    } else {
#pragma unroll
        for (int i = 0; i < ROWS; i++, p += stride) raw[i].load_some(p, (uint32_t)i < n ? left : 0);
    }
}

// Two floats to two e4m3 bytes (nearest even, saturating), the first in the low byte; their values
// come back too.
__device__ __forceinline__ uint32_t mx_e4m3x2(float a, float b, float2 *back) {
    uint16_t p;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(b), "f"(a));
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(p));
    *back = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    return p;
}

// The next piece of eight values, as four pairs of e4m3; what it leaves of them, 16 times as large, in v.
__device__ __forceinline__ void mx_piece8(float (&v)[8], uint32_t (&h)[4]) {
#pragma unroll
    for (int b = 0; b < 4; b++) {
        float2 back;
        h[b] = mx_e4m3x2(v[2 * b], v[2 * b + 1], &back);
        v[2 * b] = (v[2 * b] - back.x) * 16.0f;
        v[2 * b + 1] = (v[2 * b + 1] - back.y) * 16.0f;
    }
}

// One float to e4m3 (nearest even, saturating) and the value that it stands for.
__device__ __forceinline__ uint32_t mx_e4m3(float v, float *back) {
    uint16_t p;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(0.0f), "f"(v));
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(p));
    *back = __low2float(*reinterpret_cast<const __half2 *>(&h));
    return p & 0xFFu;
}

// Scale byte of the first piece of a block whose largest magnitude is `top`: top / 2^(s - 127) lies
// in [128, 256), under e4m3's 448, so no piece saturates. Piece p of the block has scale byte
// s - 4p: a piece leaves at most half a step, 8 of these units, which the next, 16 times finer,
// holds as 128. s is at least 4 (pieces - 1) so that every s - 4p is a scale. NaN and infinity: 255.
__device__ __forceinline__ uint32_t mx_piece_scale(float top, int pieces) {
    const uint32_t e = __float_as_uint(top) >> 23, least = 4 * (pieces - 1);
    return e == 255 ? 255u : max(e < 7 ? 0u : e - 7u, least);
}
__device__ __forceinline__ uint32_t mx_piece_scale_of(uint32_t s, int p) { return s == 255 ? 255u : s - 4 * p; }

template <typename T>
__device__ __forceinline__ float mx_float(T v);
template <>
__device__ __forceinline__ float mx_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float mx_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T mx_to(float v);
template <>
__device__ __forceinline__ float mx_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half mx_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 mx_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
#endif

// The kernels below but pack_kernel, which is launched in full stream order, are launched programmatically (common.cuh):
// a kernel's first access to memory follows grid_dep_wait(), and it lets the next one start only after that, so a
// kernel that has started early never meets memory of one before the last. The exception are the weight copies of
// a product that follows pieces_kernel: that kernel has waited for all before it and writes no weights, so they
// need not wait for it. Loads are plain ones, not __ldg: those are for memory
// that nobody writes while the kernel runs, and the kernel before may still write when this one starts.
cudaError_t launch_mx4_quantize(const void *x, int type, uint32_t rows, uint32_t k, uint64_t stride, int layout,
                                uint8_t *codes, uint8_t *scales, cudaStream_t s);
cudaError_t launch_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, int layout, uint32_t rows, uint32_t k,
                                  void *y, int type, uint64_t stride, cudaStream_t s);
cudaError_t launch_mx4_pack(const uint8_t *codes, const uint8_t *scales, uint32_t count, uint32_t rows, uint32_t k,
                            int paired, uint8_t *out_codes, uint8_t *out_scales, cudaStream_t s);

// The router's results and the scratch of one ug_mx4_experts call, carved from its workspace.
struct MxExpertsScratch {
    int32_t *chosen;      // tokens x top_k
    float *weight;        // tokens x top_k
    uint32_t *items;      // the work items of the products: mx_experts_items of 34 words, after one for their number
    uint32_t *arrived;    // tokens x 4 mx_tiles(d): pairs whose 32 values are written
    uint8_t *x_pieces;    // (tokens * pieces) x 128 mx_tiles(d), e4m3
    uint8_t *x_scales;    // (tokens * pieces) x 4 mx_tiles(d)
    uint8_t *h_pieces;    // (tokens * top_k * 4) x 128 mx_tiles(f), e4m3
    uint8_t *h_scales;    // (tokens * top_k * 4) x 4 mx_tiles(f)
    float *partial;       // (tokens * top_k) x d: weighted down products
};

// The most work items that `pairs` (token, choice) pairs over `experts` can make, in the smallest chunks of 16.
inline size_t mx_experts_items(size_t pairs, size_t experts) {
    const size_t slots = pairs < experts ? pairs : experts;
    return slots + (pairs - slots) / 16;
}

struct MxExpertsArgs {
    uint32_t experts, top_k, d, f, tokens;
    int normalize, type;
    const void *router;
    const float *bias;
    const uint8_t *gate_up_codes, *gate_up_scales, *down_codes, *down_scales;
    const void *x;
    uint64_t x_stride;
    void *y;
    uint64_t y_stride;
    int32_t *chosen;      // the caller's copies, or null
    float *weights;
    MxExpertsScratch ws;
};

cudaError_t launch_mx4_router(const MxExpertsArgs &a, cudaStream_t s);

struct MxProductArgs {
    const void *x;            // 16-bit activations (x16), or null
    int x_type;
    uint64_t x_stride;
    const uint8_t *a_codes, *a_scales;   // MX4 activations, or null
    uint32_t m;
    const uint8_t *w_codes, *w_scales;
    uint32_t n, k;
    void *y;
    int type;
    uint64_t stride;
    void *workspace;          // x16: pieces and their scales
};

// Rows of e4m3 pieces of m 16-bit tokens (x16).
size_t mx_piece_rows(uint32_t m, int x_type);
// Site code of a product kernel's wait that ran out of time on the current device since the last reset.
int mx_tc_error(bool reset);
cudaError_t launch_mx4_product(const MxProductArgs &a, cudaStream_t s);
cudaError_t launch_mx4_expert_products(const MxExpertsArgs &a, cudaStream_t s);

}  // namespace uq
