// k_mx.cu -- MX4 quantisation, its inverse, packing into the operand layout, and the router of the
// expert layer (include/unoq_mx.h). The products are in mx_tc.cu.
#include <cooperative_groups.h>

#include "common.cuh"
#include "mx.cuh"

namespace uq {
namespace {

namespace cg = cooperative_groups;

// ---- quantise / dequantise -------------------------------------------------------------------
//
// 16 lanes take one row's 128 values (one operand tile's width), 8 each: four lanes to a block of
// 32, whose largest magnitude is found by two shuffles. Bound by memory: in bf16 a value is 2 bytes
// read and 17/32 written.

template <typename T>
__device__ __forceinline__ void load8(const T *p, uint32_t left, bool vec, float (&v)[8]) {
    if (vec && left >= 8) {
        if (sizeof(T) == 4) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint16_t h = (uint16_t)(w[i / 2] >> (i % 2 * 16));
                v[i] = mx_float(*reinterpret_cast<const T *>(&h));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (uint32_t)i < left ? mx_float(p[i]) : 0.0f;
    }
}

template <typename T, bool OPERAND>
__global__ void __launch_bounds__(256) quantize_kernel(const T *x, uint32_t rows, uint32_t k, uint64_t stride,
                                                       uint32_t kt, uint32_t units, uint8_t *codes, uint8_t *scales,
                                                       bool vec_in, bool vec_out) {
    const uint32_t lane = threadIdx.x % 16;
    const uint32_t step = gridDim.x * (blockDim.x / 16);
    const uint32_t first = (blockIdx.x * blockDim.x + threadIdx.x) / 16;
    // every lane of a warp runs the same number of rounds: the two halves differ by one unit
    for (uint32_t base = first & ~1u; base < units; base += step) {
        const uint32_t u = base + (first & 1u);
        const bool live = u < units;
        const uint32_t r = live ? u / kt : 0, tile = live ? u - r * kt : 0;
        const uint32_t j = tile * kMxTile + lane * 8;
        float v[8];
        load8(x + r * stride + j, live && j < k ? k - j : 0, vec_in, v);
        float top = 0.0f;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            top = fmaxf(top, fabsf(v[i]));   // fmaxf drops NaN: kept apart
            nan |= v[i] != v[i];
        }
        uint32_t bits = nan ? 0x7FC00000u : __float_as_uint(top);  // orders as the magnitudes do
        bits = max(bits, __shfl_xor_sync(~0u, bits, 1));
        bits = max(bits, __shfl_xor_sync(~0u, bits, 2));
        const uint32_t e = bits >> 23;                  // biased exponent; subnormal and zero: 0
        const uint32_t s = e == 255 ? 255u : (e < 2 ? 0u : e - 2);
        const float inverse = __uint_as_float((254u - min(s, 253u)) << 23);   // 2^(127 - s), exact
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= inverse;
        const uint32_t c = s == 255 ? 0u : mx_pack8(v);
        if (OPERAND) {
            uint32_t all = s | __shfl_down_sync(~0u, s, 4) << 8;
            all |= __shfl_down_sync(~0u, all, 8) << 16;
            if (live) {
                *reinterpret_cast<uint32_t *>(codes + mx_code_at(r, j, kt)) = c;
                if (lane == 0) *reinterpret_cast<uint32_t *>(scales + mx_scale_at(r, tile * 4, kt)) = all;
            }
        } else if (live && j < k) {
            const uint32_t row_bytes = (k + 1) / 2;
            uint8_t *dst = codes + (size_t)r * row_bytes + j / 2;
            if (vec_out && j + 8 <= k)
                *reinterpret_cast<uint32_t *>(dst) = c;
            else
                for (uint32_t i = 0; i < 4 && j / 2 + i < row_bytes; i++) dst[i] = (uint8_t)(c >> (8 * i));
            if (lane % 4 == 0) scales[(size_t)r * ((k + 31) / 32) + j / 32] = (uint8_t)s;
        }
    }
}

template <typename T, bool OPERAND>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t *codes, const uint8_t *scales, uint32_t rows,
                                                         uint32_t k, uint32_t kt, uint32_t units, T *y, uint64_t stride,
                                                         bool vec_in, bool vec_out) {
    const uint32_t lane = threadIdx.x % 16;
    const uint32_t step = gridDim.x * (blockDim.x / 16);
    for (uint32_t u = (blockIdx.x * blockDim.x + threadIdx.x) / 16; u < units; u += step) {
        const uint32_t r = u / kt, tile = u - r * kt;
        const uint32_t j = tile * kMxTile + lane * 8;
        if (j >= k) continue;
        uint32_t c = 0, s;
        if (OPERAND) {
            c = __ldg(reinterpret_cast<const uint32_t *>(codes + mx_code_at(r, j, kt)));
            s = __ldg(scales + mx_scale_at(r, j / 32, kt));
        } else {
            const uint32_t row_bytes = (k + 1) / 2;
            const uint8_t *src = codes + (size_t)r * row_bytes + j / 2;
            if (vec_in && j + 8 <= k)
                c = __ldg(reinterpret_cast<const uint32_t *>(src));
            else
                for (uint32_t i = 0; i < 4 && j / 2 + i < row_bytes; i++) c |= (uint32_t)src[i] << (8 * i);
            s = __ldg(scales + (size_t)r * ((k + 31) / 32) + j / 32);
        }
        float v[8];
        mx_unpack8(c, v);
        const float scale = mx_scale_value(s);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= scale;
        T *dst = y + r * stride + j;
        if (vec_out && j + 8 <= k) {
            if (sizeof(T) == 4) {
                reinterpret_cast<float4 *>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4 *>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    T p[2] = {mx_to<T>(v[2 * i]), mx_to<T>(v[2 * i + 1])};
                    w[i] = *reinterpret_cast<const uint32_t *>(p);
                }
                *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            for (uint32_t i = 0; i < 8 && j + i < k; i++) dst[i] = mx_to<T>(v[i]);
        }
    }
}

// ---- stored -> operand layout ------------------------------------------------------------------
//
// Once per weight, not per call. 16 lanes write the 64 code bytes and the four scales of one
// (row, tile), the padding rows and columns with zeros.

__global__ void __launch_bounds__(256) pack_kernel(const uint8_t *codes, const uint8_t *scales, uint32_t rows,
                                                   uint32_t k, int paired, uint32_t padded, uint32_t kt, uint64_t units,
                                                   uint8_t *out_codes, uint8_t *out_scales) {
    const uint32_t lane = threadIdx.x % 16;
    const uint64_t step = (uint64_t)gridDim.x * (blockDim.x / 16);
    const uint32_t row_bytes = (k + 1) / 2, blocks = (k + 31) / 32;
    for (uint64_t u = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) / 16; u < units; u += step) {
        const uint64_t out_row = u / kt;
        const uint32_t tile = (uint32_t)(u - out_row * kt);
        const uint32_t matrix = (uint32_t)(out_row / padded), pr = (uint32_t)(out_row - (uint64_t)matrix * padded);
        uint32_t r = pr;   // source row, or `rows` for padding
        if (paired) {
            const uint32_t half = rows / 2, i = pr / 256 * 128 + pr % 128;
            r = i < half ? i + (pr / 128 % 2 ? half : 0) : rows;
        }
        uint32_t c = 0;
        if (r < rows) {
            const uint8_t *src = codes + ((size_t)matrix * rows + r) * row_bytes;
            const uint32_t at = tile * 64 + lane * 4;
            for (uint32_t i = 0; i < 4; i++) {
                if (at + i >= row_bytes) break;
                uint32_t b = src[at + i];
                if (k % 2 && at + i == row_bytes - 1) b &= 15;  // the nibble past the last value
                c |= b << (8 * i);
            }
        }
        const size_t t = out_row / kMxTile * kt + tile;
        const uint32_t tr = (uint32_t)(out_row % kMxTile);
        *reinterpret_cast<uint32_t *>(out_codes + t * kMxCodeTile + tr * 64 + lane * 4) = c;
        if (lane < 4) {
            const uint32_t b = tile * 4 + lane;
            out_scales[t * kMxScaleTile + tr % 32 * 16 + tr / 32 * 4 + lane] =
                r < rows && b < blocks ? scales[((size_t)matrix * rows + r) * blocks + b] : 0;
        }
    }
}

// ---- router ------------------------------------------------------------------------------------
//
// A cluster of 8 CTAs per token: each holds the token's row in shared memory and takes every eighth
// expert, one warp to an expert's product (32 lanes across d, fixed order, so logits do not depend
// on timing). The logits meet in the first CTA's shared memory, whose first warp selects. The same
// CTAs split the row into the pieces that the gate / up product reads.

template <typename T>
__global__ void __cluster_dims__(kMxRouterCluster, 1, 1) __launch_bounds__(256) router_kernel(MxExpertsArgs a, bool vec) {
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ float logits[256];
    T *row = reinterpret_cast<T *>(raw);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = blockIdx.x, t = blockIdx.y;
    grid_dep_launch();  // the products' set-up may begin; they wait for this kernel's results
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const T *x = static_cast<const T *>(a.x) + t * a.x_stride;
    for (uint32_t i = threadIdx.x; i < a.d; i += blockDim.x) row[i] = x[i];
    cluster.sync();  // the row is staged, and the first CTA's shared memory exists for the others

    float *remote = cluster.map_shared_rank(logits, 0);
    for (uint32_t e = rank + kMxRouterCluster * warp; e < a.experts; e += kMxRouterCluster * 8) {
        const T *w = static_cast<const T *>(a.router) + (size_t)e * a.d;
        float sum = 0.0f;
        if (vec) {
#pragma unroll 4
            for (uint32_t i = lane * 8; i < a.d; i += 256) {
                const uint4 p = __ldg(reinterpret_cast<const uint4 *>(w + i)), q = *reinterpret_cast<const uint4 *>(row + i);
                const T *ph = reinterpret_cast<const T *>(&p), *qh = reinterpret_cast<const T *>(&q);
#pragma unroll
                for (int j = 0; j < 8; j++) sum = fmaf(mx_float(ph[j]), mx_float(qh[j]), sum);
            }
        } else {
            for (uint32_t i = lane; i < a.d; i += 32) sum = fmaf(mx_float(w[i]), mx_float(row[i]), sum);
        }
#pragma unroll
        for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane == 0) remote[e] = sum + (a.bias ? a.bias[e] : 0.0f);
    }

    // the row's pieces: one warp to a block of 32 values
    const uint32_t kt = mx_tiles(a.d);
    const int pieces = mx_pieces(a.type);
    for (uint32_t b = rank * 8 + warp; b < kt * 4; b += kMxRouterCluster * 8) {
        const uint32_t i = b * 32 + lane;
        const float v = i < a.d ? mx_float(row[i]) : 0.0f;
        // infinity and NaN order above every number here
        const uint32_t top = __reduce_max_sync(~0u, __float_as_uint(v) & 0x7FFFFFFFu);
        const uint32_t s = mx_piece_scale(__uint_as_float(top), pieces);
        float left = v * __uint_as_float((254u - min(s, 253u)) << 23);
        for (int p = 0; p < pieces; p++) {
            float back;
            const uint32_t code = mx_e4m3(left, &back);
            left = (left - back) * 16.0f;
            const size_t r = (size_t)t * pieces + p;
            a.ws.x_pieces[r * kt * 128 + i] = s == 255 ? 0 : (uint8_t)code;
            if (lane == 0) a.ws.x_scales[r * kt * 4 + b] = (uint8_t)mx_piece_scale_of(s, p);
        }
    }
    if (rank == 0)
        for (uint32_t i = threadIdx.x; i < kt * 4; i += blockDim.x) a.ws.arrived[(size_t)t * kt * 4 + i] = 0;

    cluster.sync();
    if (rank != 0 || warp != 0) return;
    // selection: keys order as the logits do; a NaN is below every number, a taken expert is 0
    uint32_t key[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t e = lane + 32 * i;
        key[i] = 0;
        if (e < a.experts) {
            const float l = logits[e];
            const uint32_t bits = __float_as_uint(l);
            key[i] = l != l ? 1u : (bits & 0x80000000u ? ~bits : bits | 0x80000000u);
            if (l == 0.0f) key[i] = 0x80000000u;  // -0 and 0 tie
        }
    }
    float chosen_logit = 0.0f, first = 0.0f;
    uint32_t chosen = 0;
    for (uint32_t j = 0; j < a.top_k; j++) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) best = max(best, key[i]);
        best = __reduce_max_sync(~0u, best);
        uint32_t at = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 7; i >= 0; i--)
            if (key[i] == best) at = lane + 32 * i;
        at = __reduce_min_sync(~0u, at);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (at == lane + 32u * i) key[i] = 0;
        const float l = logits[at];
        if (j == 0) first = l;
        if (lane == (int)j) {
            chosen = at;
            chosen_logit = l;
        }
    }
    const bool mine = lane < (int)a.top_k;
    const float p = mine ? expf(chosen_logit - first) : 0.0f;
    float total = p;
    if (!a.normalize) {
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t e = lane + 32 * i;
            if (e < a.experts) total += expf(logits[e] - first);
        }
    }
#pragma unroll
    for (int o = 16; o; o /= 2) total += __shfl_xor_sync(~0u, total, o);
    if (mine) {
        const size_t at = (size_t)t * a.top_k + lane;
        a.ws.chosen[at] = (int32_t)chosen;
        a.ws.weight[at] = p / total;
        if (a.chosen) a.chosen[at] = (int32_t)chosen;
        if (a.weights) a.weights[at] = p / total;
    }
}

bool aligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Blocks of 256 threads (16 units) to fill the GPU a few times over, no more than the units need.
unsigned unit_grid(uint64_t units) {
    const uint64_t need = (units + 15) / 16;
    return (unsigned)(need < 148 * 16 ? need : 148 * 16);
}

template <typename T>
cudaError_t quantize(const void *x, uint32_t rows, uint32_t k, uint64_t stride, int layout, uint8_t *codes,
                     uint8_t *scales, cudaStream_t s) {
    const uint32_t kt = mx_tiles(k), units = rows * kt;
    const bool vec_in = aligned(x, 16) && stride * sizeof(T) % 16 == 0;
    const bool vec_out = aligned(codes, 4) && (k + 1) / 2 % 4 == 0;
    auto kernel = layout ? quantize_kernel<T, true> : quantize_kernel<T, false>;
    kernel<<<unit_grid(units), 256, 0, s>>>(static_cast<const T *>(x), rows, k, stride, kt, units, codes, scales, vec_in,
                                           vec_out);
    return cudaGetLastError();
}

template <typename T>
cudaError_t dequantize(const uint8_t *codes, const uint8_t *scales, int layout, uint32_t rows, uint32_t k, void *y,
                       uint64_t stride, cudaStream_t s) {
    const uint32_t kt = mx_tiles(k), units = rows * kt;
    const bool vec_in = aligned(codes, 4) && (k + 1) / 2 % 4 == 0;
    const bool vec_out = aligned(y, 16) && stride * sizeof(T) % 16 == 0;
    auto kernel = layout ? dequantize_kernel<T, true> : dequantize_kernel<T, false>;
    kernel<<<unit_grid(units), 256, 0, s>>>(codes, scales, rows, k, kt, units, static_cast<T *>(y), stride, vec_in,
                                           vec_out);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mx4_quantize(const void *x, int type, uint32_t rows, uint32_t k, uint64_t stride, int layout,
                                uint8_t *codes, uint8_t *scales, cudaStream_t s) {
    if (type == 0) return quantize<float>(x, rows, k, stride, layout, codes, scales, s);
    if (type == 1) return quantize<__half>(x, rows, k, stride, layout, codes, scales, s);
    return quantize<__nv_bfloat16>(x, rows, k, stride, layout, codes, scales, s);
}

cudaError_t launch_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, int layout, uint32_t rows, uint32_t k,
                                  void *y, int type, uint64_t stride, cudaStream_t s) {
    if (type == 0) return dequantize<float>(codes, scales, layout, rows, k, y, stride, s);
    if (type == 1) return dequantize<__half>(codes, scales, layout, rows, k, y, stride, s);
    return dequantize<__nv_bfloat16>(codes, scales, layout, rows, k, y, stride, s);
}

cudaError_t launch_mx4_pack(const uint8_t *codes, const uint8_t *scales, uint32_t count, uint32_t rows, uint32_t k,
                            int paired, uint8_t *out_codes, uint8_t *out_scales, cudaStream_t s) {
    const uint32_t padded = (paired ? 2 * mx_tiles(rows / 2) : mx_tiles(rows)) * kMxTile, kt = mx_tiles(k);
    const uint64_t units = (uint64_t)count * padded * kt;
    pack_kernel<<<unit_grid(units), 256, 0, s>>>(codes, scales, rows, k, paired, padded, kt, units, out_codes, out_scales);
    return cudaGetLastError();
}

cudaError_t launch_mx4_router(const MxExpertsArgs &a, cudaStream_t s) {
    const bool vec = aligned(a.router, 16) && a.d % 8 == 0;
    const dim3 grid(kMxRouterCluster, a.tokens);
    const size_t smem = (a.d * 2 + 15) / 16 * 16;
    if (a.type == 1)
        router_kernel<__half><<<grid, 256, smem, s>>>(a, vec);
    else
        router_kernel<__nv_bfloat16><<<grid, 256, smem, s>>>(a, vec);
    return cudaGetLastError();
}

}  // namespace uq
