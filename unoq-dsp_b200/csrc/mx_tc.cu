// mx_tc.cu -- products with MX4 weights (include/unoq_mx.h).
#include "mx.cuh"

namespace uq {
namespace {

__device__ __forceinline__ float mx_at(const uint8_t *codes, const uint8_t *scales, uint32_t r, uint32_t j, uint32_t kt) {
    float v[8];
    mx_unpack8(codes[mx_code_at(r, j, kt)] >> (j % 2 * 4), v);
    return v[0] * mx_scale_value(scales[mx_scale_at(r, j / 32, kt)]);
}

template <typename T>
__device__ __forceinline__ void put(void *y, size_t at, float v) { static_cast<T *>(y)[at] = mx_to<T>(v); }
__device__ __forceinline__ void put_as(void *y, int type, size_t at, float v) {
    if (type == 0) put<float>(y, at, v);
    else if (type == 1) put<__half>(y, at, v);
    else put<__nv_bfloat16>(y, at, v);
}
__device__ __forceinline__ float get_as(const void *x, int type, size_t at) {
    const float v = type == 1 ? __half2float(static_cast<const __half *>(x)[at])
                              : __bfloat162float(static_cast<const __nv_bfloat16 *>(x)[at]);
    return v + (v - v);  // an infinity counts as NaN
}

__global__ void product_kernel(MxProductArgs a) {
    const uint32_t j = blockIdx.x * blockDim.x + threadIdx.x, kt = mx_tiles(a.k);
    if (j >= a.n) return;
    for (uint32_t i = blockIdx.y; i < a.m; i += gridDim.y) {
        float sum = 0.0f;
        for (uint32_t t = 0; t < a.k; t++) {
            const float x = a.x ? get_as(a.x, a.x_type, i * a.x_stride + t) : mx_at(a.a_codes, a.a_scales, i, t, kt);
            sum = fmaf(x, mx_at(a.w_codes, a.w_scales, j, t, kt), sum);
        }
        put_as(a.y, a.type, i * a.stride + j, sum);
    }
}

// h of one (token, choice) pair, in the partial buffer's place
__global__ void hidden_kernel(MxExpertsArgs a, float *h) {
    const uint32_t j = blockIdx.x * blockDim.x + threadIdx.x, pair = blockIdx.y, kt = mx_tiles(a.d);
    if (j >= a.f) return;
    const uint32_t e = a.ws.chosen[pair], t = pair / a.top_k;
    const uint32_t r = (e * mx_tiles(a.f) + j / 128) * 256 + j % 128;
    float g = 0.0f, u = 0.0f;
    for (uint32_t i = 0; i < a.d; i++) {
        const float x = get_as(a.x, a.type, t * a.x_stride + i);
        g = fmaf(x, mx_at(a.gate_up_codes, a.gate_up_scales, r, i, kt), g);
        u = fmaf(x, mx_at(a.gate_up_codes, a.gate_up_scales, r + 128, i, kt), u);
    }
    h[(size_t)pair * a.f + j] = g / (1.0f + expf(-g)) * u;
}

__global__ void down_kernel(MxExpertsArgs a, const float *h) {
    const uint32_t j = blockIdx.x * blockDim.x + threadIdx.x, t = blockIdx.y, kt = mx_tiles(a.f);
    if (j >= a.d) return;
    float y = 0.0f;
    for (uint32_t c = 0; c < a.top_k; c++) {
        const uint32_t pair = t * a.top_k + c, r = a.ws.chosen[pair] * mx_tiles(a.d) * 128 + j;
        float sum = 0.0f;
        for (uint32_t i = 0; i < a.f; i++)
            sum = fmaf(h[(size_t)pair * a.f + i], mx_at(a.down_codes, a.down_scales, r, i, kt), sum);
        y += a.ws.weight[pair] * sum;
    }
    put_as(a.y, a.type, t * a.y_stride + j, y);
}

}  // namespace

cudaError_t launch_mx4_product(const MxProductArgs &a, cudaStream_t s) {
    product_kernel<<<dim3((a.n + 127) / 128, a.m < 65535 ? a.m : 65535), 128, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_mx4_expert_products(const MxExpertsArgs &a, cudaStream_t s) {
    float *h = reinterpret_cast<float *>(a.ws.h_pieces);
    hidden_kernel<<<dim3((a.f + 127) / 128, a.tokens * a.top_k), 128, 0, s>>>(a, h);
    down_kernel<<<dim3((a.d + 127) / 128, a.tokens), 128, 0, s>>>(a, h);
    return cudaGetLastError();
}

}  // namespace uq
