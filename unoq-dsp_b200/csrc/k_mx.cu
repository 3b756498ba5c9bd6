// k_mx.cu -- MX4 quantisation, its inverse, packing into the operand layout, and the router of the
// expert layer (include/unoq_mx.h). The products are in mx_tc.cu.
#include <cooperative_groups.h>

#include <utility>

#include "common.cuh"
#include "mx.cuh"

namespace uq {
namespace {

namespace cg = cooperative_groups;

// ---- quantise / dequantise -------------------------------------------------------------------
//
// A warp takes 256 columns (a code tile's width, 8 values to a lane, four lanes to a block of
// 32) of ROWS consecutive rows: the loads of all of them go out first, and a row's addresses are the
// one before's plus a constant. What bounds it is memory, once the instructions are few: with one
// row to a thread and its indices by division, 168 instructions a thread held a matrix of 8192 x 8192
// bf16 to 50 us of issue time.

template <typename T, bool OPERAND, int ROWS>
__global__ void __launch_bounds__(256) quantize_kernel(const T *x, uint32_t rows, uint32_t k, uint64_t stride, uint32_t kt,
                                                       uint32_t chunks, uint8_t *codes, uint8_t *scales, bool vec_in,
                                                       bool vec_out) {
    grid_dep_wait();
    grid_dep_launch();
    const uint32_t lane = threadIdx.x % 32, w = blockIdx.x * 8 + threadIdx.x / 32;
    const uint32_t group = w / chunks, chunk = w - group * chunks, r0 = group * ROWS;
    if (r0 >= rows) return;
    const uint32_t n = min((uint32_t)ROWS, rows - r0), j = chunk * 256 + lane * 8;
    MxRaw<T> raw[ROWS];
    mx_load_rows<T, ROWS>(raw, x + r0 * stride + j, stride, n, j < k ? k - j : 0, vec_in && chunk * 256 + 256 <= k);
    const uint32_t row_bytes = (k + 1) / 2, blocks = (k + 31) / 32;
    uint8_t *to = codes + (OPERAND ? mx_code_at(r0, j, kt) : (size_t)r0 * row_bytes + j / 2);
    uint8_t *st = scales + (OPERAND ? mx_scale_at(r0, j / 32, kt) : (size_t)r0 * blocks + j / 32);
    const bool mine = OPERAND || j < k;   // a code tile is written whole
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        if ((uint32_t)i >= n) break;
        uint32_t top = raw[i].top();
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        const uint32_t e = raw[i].top_bits(top) >> 23;  // biased exponent; subnormal and zero: 0
        const uint32_t s = e == 255 ? 255u : (e < 2 ? 0u : e - 2);
        float v[8];
        raw[i].values(v, __uint_as_float((254u - min(s, 253u)) << 23));   // times 2^(127 - s), exact
        const uint32_t c = s == 255 ? 0u : mx_pack8(v);
        if (mine) {
            if (OPERAND || (vec_out && j + 8 <= k)) {
                *reinterpret_cast<uint32_t *>(to) = c;
            } else {
                for (uint32_t b = 0; b < 4 && j / 2 + b < row_bytes; b++) to[b] = (uint8_t)(c >> (8 * b));
            }
            if (lane % 4 == 0) *st = (uint8_t)s;
        }
        to += OPERAND ? 128 : row_bytes;
        st += OPERAND ? 16 : blocks;
    }
}

template <typename T, bool OPERAND, int ROWS>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t *codes, const uint8_t *scales, uint32_t rows, uint32_t k,
                                                         uint32_t kt, uint32_t chunks, T *y, uint64_t stride, bool vec_in,
                                                         bool vec_out) {
    grid_dep_wait();
    grid_dep_launch();
    const uint32_t lane = threadIdx.x % 32, w = blockIdx.x * 8 + threadIdx.x / 32;
    const uint32_t group = w / chunks, chunk = w - group * chunks, r0 = group * ROWS;
    const uint32_t j = chunk * 256 + lane * 8;
    if (r0 >= rows) return;
    const uint32_t n = j < k ? min((uint32_t)ROWS, rows - r0) : 0, row_bytes = (k + 1) / 2, blocks = (k + 31) / 32;
    const uint8_t *from = codes + (OPERAND ? mx_code_at(r0, j, kt) : (size_t)r0 * row_bytes + j / 2);
    const uint8_t *sf = scales + (OPERAND ? mx_scale_at(r0, j / 32, kt) : (size_t)r0 * blocks + j / 32);
    uint32_t c[ROWS], s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        c[i] = s[i] = 0;
        if ((uint32_t)i < n) {
            if (OPERAND || (vec_in && j + 8 <= k)) {
                c[i] = *reinterpret_cast<const uint32_t *>(from);
            } else {
                for (uint32_t b = 0; b < 4 && j / 2 + b < row_bytes; b++) c[i] |= (uint32_t)from[b] << (8 * b);
            }
            s[i] = *sf;
        }
        from += OPERAND ? 128 : row_bytes;
        sf += OPERAND ? 16 : blocks;
    }
    if (!vec_out) {
        // rows that start anywhere: lane l writes values l, l + 32, ..., neighbours side by side
        T *to = y + r0 * stride + chunk * 256;
        const uint32_t inside = k - chunk * 256;
        for (uint32_t i = 0; i < min((uint32_t)ROWS, rows - r0); i++, to += stride) {
            uint32_t word = 0, code = 0;
#pragma unroll
            for (int b = 0; b < ROWS; b++)
                if ((uint32_t)b == i) word = c[b], code = s[b];
            const float scale = mx_scale_value(code);
#pragma unroll
            for (uint32_t b = 0; b < 8; b++) {
                const uint32_t at = b * 32 + lane;
                const uint32_t w8 = __shfl_sync(~0u, word, at / 8);
                const float sc = __shfl_sync(~0u, scale, at / 8);
                if (at < inside) to[at] = mx_to<T>(mx_unpack1(w8 >> (at % 8 * 4)) * sc);
            }
        }
        return;
    }
    T *to = y + r0 * stride + j;
#pragma unroll
    for (int i = 0; i < ROWS; i++, to += stride) {
        if ((uint32_t)i >= n) break;
        float v[8];
        mx_unpack8(c[i], v);
        const float scale = mx_scale_value(s[i]);
#pragma unroll
        for (int b = 0; b < 8; b++) v[b] *= scale;
        if (j + 8 <= k) {
            if constexpr (sizeof(T) == 4) {
                reinterpret_cast<float4 *>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4 *>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                uint32_t p[4];
#pragma unroll
                for (int b = 0; b < 4; b++) p[b] = mx_pair<T>(v[2 * b], v[2 * b + 1]);
                *reinterpret_cast<uint4 *>(to) = make_uint4(p[0], p[1], p[2], p[3]);
            }
        } else {
            for (uint32_t b = 0; b < 8 && j + b < k; b++) to[b] = mx_to<T>(v[b]);
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
            const uint32_t half = rows / 2, i = pr / kMxTile * kMxHalf + pr % kMxHalf;
            r = i < half ? i + (pr % kMxTile < kMxHalf ? 0 : half) : rows;
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
        const size_t row_tile = out_row / kMxTile, t = row_tile * kt + tile;
        const uint32_t tr = (uint32_t)(out_row % kMxTile);
        *reinterpret_cast<uint32_t *>(out_codes + (row_tile * (kt / 2) + tile / 2) * kMxCodeTile + tr * 128 + tile % 2 * 64 +
                                      lane * 4) = c;
        if (lane < 4) {
            const uint32_t b = tile * 4 + lane;
            out_scales[t * kMxScaleTile + tr % 32 * 16 + tr / 32 * 4 + lane] =
                r < rows && b < blocks ? scales[((size_t)matrix * rows + r) * blocks + b] : 0;
        }
    }
}

// ---- router ------------------------------------------------------------------------------------
//
// A cluster of 8 CTAs per token: each takes every eighth expert, one warp to an expert's product (32
// lanes across d, fixed order, so logits do not depend on timing). The logits meet in the first CTA's
// shared memory, whose first warp selects. The same CTAs split the token's row into the pieces that the
// gate / up product reads. It is a chain of latencies: 4.4 us for one token and 32 experts of 2048, 2 of
// them for the products, 0.7 for the cluster's barrier and 0.6 for the selection. Four tokens to a
// cluster, sharing the router rows that they read, took longer at 64 tokens (13.6 us).

template <typename T>
__global__ void __cluster_dims__(kMxRouterCluster, 1, 1) __launch_bounds__(256) router_kernel(MxExpertsArgs a, bool vec) {
    __shared__ float logits[256];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = blockIdx.x, t = blockIdx.y;
    auto started = cluster.barrier_arrive();  // the first CTA's shared memory exists for the others after the wait
    grid_dep_wait();
    grid_dep_launch();  // the products' set-up may begin; they wait for this kernel's results
    bool waited = false;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const T *x = static_cast<const T *>(a.x) + t * a.x_stride;

    // A row's loads go out together before the first product: eight of 16 bytes, or sixteen single values
    // where rows do not start on 16 bytes (1447 wide: 10.9 -> 6.1 us).
    float *remote = cluster.map_shared_rank(logits, 0);
    for (uint32_t e = rank + kMxRouterCluster * warp; e < a.experts; e += kMxRouterCluster * 8) {
        const T *w = static_cast<const T *>(a.router) + (size_t)e * a.d;
        float sum = 0.0f;
        if (vec) {
            for (uint32_t i0 = lane * 8; i0 < a.d; i0 += 2048) {
                uint4 p[8], q[8];
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const uint32_t i = i0 + c * 256;
                    p[c] = i < a.d ? *reinterpret_cast<const uint4 *>(w + i) : make_uint4(0, 0, 0, 0);
                    q[c] = i < a.d ? *reinterpret_cast<const uint4 *>(x + i) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const T *ph = reinterpret_cast<const T *>(&p[c]), *qh = reinterpret_cast<const T *>(&q[c]);
#pragma unroll
                    for (int j = 0; j < 8; j++) sum = fmaf(mx_float(ph[j]), mx_float(qh[j]), sum);
                }
            }
        } else {
            for (uint32_t i0 = lane; i0 < a.d; i0 += 512) {
                T p[16], q[16];
#pragma unroll
                for (int c = 0; c < 16; c++) {
                    const uint32_t i = i0 + c * 32;
                    p[c] = i < a.d ? w[i] : mx_to<T>(0.0f);
                    q[c] = i < a.d ? x[i] : mx_to<T>(0.0f);
                }
#pragma unroll
                for (int c = 0; c < 16; c++) sum = fmaf(mx_float(p[c]), mx_float(q[c]), sum);
            }
        }
#pragma unroll
        for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
        if (!waited) {
            cluster.barrier_wait(std::move(started));
            waited = true;
        }
        if (lane == 0) remote[e] = sum + (a.bias ? a.bias[e] : 0.0f);
    }
    if (!waited) cluster.barrier_wait(std::move(started));

    // the row's pieces: one warp to a block of 32 values
    const uint32_t kt = mx_tiles(a.d);
    const int pieces = mx_pieces(a.type);
    for (uint32_t b = rank * 8 + warp; b < kt * 4; b += kMxRouterCluster * 8) {
        const uint32_t i = b * 32 + lane;
        const float v = i < a.d ? mx_float(x[i]) : 0.0f;
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
    // selection: keys order as the logits do; a NaN is above every number, so that it is chosen and shows in the weights
    // and the output whichever softmax is taken; a taken expert is 0
    uint32_t key[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t e = lane + 32 * i;
        key[i] = 0;
        if (e < a.experts) {
            const float l = logits[e];
            const uint32_t bits = __float_as_uint(l);
            key[i] = l != l ? 0xFFFFFFFFu : (bits & 0x80000000u ? ~bits : bits | 0x80000000u);
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

// Blocks of 256 threads (16 units each) to fill the GPU a few times over, no more than the units need.
unsigned unit_grid(uint64_t units) {
    const uint64_t need = (units + 15) / 16;
    return (unsigned)(need < 148 * 16 ? need : 148 * 16);
}

// Rows to a warp: 8 (4 in 32 bits) once that still leaves every SM 32 warps, else one,
// so that small matrices spread over the GPU.
bool many_rows(uint32_t rows, uint32_t chunks, int each) { return (uint64_t)(rows / each) * chunks >= 148 * 32; }
unsigned row_grid(uint32_t rows, uint32_t chunks, int each) {
    return (unsigned)((((uint64_t)rows + each - 1) / each * chunks + 7) / 8);
}

template <typename T>
cudaError_t quantize(const void *x, uint32_t rows, uint32_t k, uint64_t stride, int layout, uint8_t *codes,
                     uint8_t *scales, cudaStream_t s) {
    constexpr int kRows = sizeof(T) == 4 ? 4 : 8;
    const uint32_t kt = mx_ktiles(k), chunks = (k + 255) / 256;
    const bool vec_in = aligned(x, 16) && stride * sizeof(T) % 16 == 0;
    const bool vec_out = aligned(codes, 4) && (k + 1) / 2 % 4 == 0;
    const bool many = many_rows(rows, chunks, kRows);
    auto kernel = layout ? (many ? quantize_kernel<T, true, kRows> : quantize_kernel<T, true, 1>)
                         : (many ? quantize_kernel<T, false, kRows> : quantize_kernel<T, false, 1>);
    return launch_pdl(kPdlMx, kernel, row_grid(rows, chunks, many ? kRows : 1), 256, 0, s, static_cast<const T *>(x), rows, k,
                      stride, kt, chunks, codes, scales, vec_in, vec_out);
}

template <typename T>
cudaError_t dequantize(const uint8_t *codes, const uint8_t *scales, int layout, uint32_t rows, uint32_t k, void *y,
                       uint64_t stride, cudaStream_t s) {
    constexpr int kRows = 8;
    const uint32_t kt = mx_ktiles(k), chunks = (k + 255) / 256;
    const bool vec_in = aligned(codes, 4) && (k + 1) / 2 % 4 == 0;
    const bool vec_out = aligned(y, 16) && stride * sizeof(T) % 16 == 0;
    const bool many = many_rows(rows, chunks, kRows);
    auto kernel = layout ? (many ? dequantize_kernel<T, true, kRows> : dequantize_kernel<T, true, 1>)
                         : (many ? dequantize_kernel<T, false, kRows> : dequantize_kernel<T, false, 1>);
    return launch_pdl(kPdlMx, kernel, row_grid(rows, chunks, many ? kRows : 1), 256, 0, s, codes, scales, rows, k, kt, chunks,
                      static_cast<T *>(y), stride, vec_in, vec_out);
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
    const uint32_t padded = (paired ? (rows / 2 + kMxHalf - 1) / kMxHalf : mx_tiles(rows)) * kMxTile, kt = mx_ktiles(k);
    const uint64_t units = (uint64_t)count * padded * kt;
    pack_kernel<<<unit_grid(units), 256, 0, s>>>(codes, scales, rows, k, paired, padded, kt, units, out_codes, out_scales);
    return cudaGetLastError();
}

cudaError_t launch_mx4_router(const MxExpertsArgs &a, cudaStream_t s) {
    const bool vec = aligned(a.router, 16) && a.d % 8 == 0 && aligned(a.x, 16) && a.x_stride % 8 == 0;
    return launch_pdl(kPdlMx, a.type == 1 ? router_kernel<__half> : router_kernel<__nv_bfloat16>,
                      dim3(kMxRouterCluster, a.tokens), 256, 0, s, a, vec);
}

}  // namespace uq
