// mx_abi.cu -- the C ABI of the MX4 operators (include/unoq_mx.h): argument checks, workspace
// layout and launches on the caller's stream. Nothing here allocates, waits or keeps state between
// calls, so calls on several threads, streams and devices do not meet, and all may be captured.
#include <cuda_runtime.h>

#include <initializer_list>
#include <string>

#include "engine.hpp"
#include "mx.cuh"
#include "unoq_mx.h"

namespace {

int fail(int code, const char *what) {
    try {
        uq::set_error(what);
    } catch (...) {  // out of host memory: the code alone
    }
    return code;
}

size_t type_bytes(int type) { return type == UG_F32 ? 4 : 2; }
bool is_type(int type) { return type == UG_F32 || type == UG_F16 || type == UG_BF16; }
bool is_half(int type) { return type == UG_F16 || type == UG_BF16; }
bool is_aligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// The device of a call's arrays, made current for the call and put back after it.
class OnDevice {
  public:
    ~OnDevice() {
        if (was_ >= 0) cudaSetDevice(was_);
    }
    int enter(std::initializer_list<const void *> ptrs) {
        int count = 0;
        if (cudaGetDeviceCount(&count) != cudaSuccess || count <= 0) {
            cudaGetLastError();
            return fail(2002, "no CUDA device");
        }
        int device = -1;
        for (const void *p : ptrs) {
            if (!p) continue;
            cudaPointerAttributes at{};
            if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
                cudaGetLastError();
                return fail(22, "MX4: a data pointer is not device memory");
            }
            if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
                return fail(22, "MX4: a data pointer is not device memory");
            if (device >= 0 && at.device != device) return fail(22, "MX4: data pointers of two devices");
            device = at.device;
        }
        int current = 0;
        if (cudaGetDevice(&current) != cudaSuccess) return fail(2001, "cudaGetDevice");
        if (current != device) {
            if (cudaSetDevice(device) != cudaSuccess) return fail(2001, "cudaSetDevice");
            was_ = current;
        }
        return 0;
    }

  private:
    int was_ = -1;
};

int launched(cudaError_t e) {
    if (e == cudaSuccess) return 0;
    return fail(2001, cudaGetErrorString(e));
}

// A launcher's result; its host bookkeeping may run out of memory, and no exception leaves a C function.
template <typename F>
int launch(const F &f) {
    try {
        return launched(f());
    } catch (...) {
        return fail(2001, "out of host memory");
    }
}

// rows x k with so many tiles each: counted in 32 bits by the kernels (unoq_mx.h states the limit)
bool sizes_ok(uint64_t rows, uint32_t k) { return k >= 1 && k <= (1u << 30) && rows * uq::mx_ktiles(k) < (1ull << 31); }

size_t up(size_t v) { return (v + 255) / 256 * 256; }

size_t experts_scratch(const UgMx4Experts &l, uint32_t tokens, uint8_t *base, uq::MxExpertsScratch *ws) {
    const size_t pairs = (size_t)tokens * l.top_k, dt = uq::mx_tiles(l.d), ft = uq::mx_tiles(l.f);
    const size_t xr = (size_t)tokens * uq::mx_pieces(l.type), hr = pairs * uq::kMxHiddenPieces;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t *p = base + at;
        at += up(bytes);
        return p;
    };
    uq::MxExpertsScratch w;
    w.chosen = reinterpret_cast<int32_t *>(take(pairs * 4));
    w.weight = reinterpret_cast<float *>(take(pairs * 4));
    w.items = reinterpret_cast<uint32_t *>(take((1 + uq::mx_experts_items(pairs, l.experts)) * 34 * 4));
    w.arrived = reinterpret_cast<uint32_t *>(take(tokens * dt * 16));
    w.x_pieces = take(xr * dt * 128);
    w.x_scales = take(xr * dt * 4);
    w.h_pieces = take(hr * ft * 128);
    w.h_scales = take(hr * ft * 4);
    w.partial = reinterpret_cast<float *>(take(pairs * l.d * 4));
    if (ws) *ws = w;
    return at;
}

int check_layer(const UgMx4Experts *l) {
    if (!l) return fail(22, "ug_mx4_experts: null layer");
    if (!is_half(l->type)) return fail(18, "ug_mx4_experts: type must be UG_F16 or UG_BF16");
    if (l->experts < 1 || l->experts > UG_MX4_MAX_EXPERTS || l->top_k < 1 || l->top_k > UG_MX4_MAX_TOP_K ||
        l->top_k > l->experts)
        return fail(18, "ug_mx4_experts: experts must be 1..256 and top_k 1..16, at most the experts");
    if (l->d < 1 || l->d > UG_MX4_MAX_WIDTH || l->f < 1 || l->f > UG_MX4_MAX_WIDTH)
        return fail(18, "ug_mx4_experts: widths must be 1..16384");
    return 0;
}

}  // namespace

extern "C" {

size_t ug_mx4_codes_bytes(int layout, uint32_t rows, uint32_t k) {
    if (layout == UG_MX4_STORED) return (size_t)rows * ((k + 1ull) / 2);
    if (layout == UG_MX4_OPERAND) return (size_t)((rows + 127ull) / 128) * ((k + 255ull) / 256) * uq::kMxCodeTile;
    return 0;
}

size_t ug_mx4_scales_bytes(int layout, uint32_t rows, uint32_t k) {
    if (layout == UG_MX4_STORED) return (size_t)rows * ((k + 31ull) / 32);
    if (layout == UG_MX4_OPERAND) return (size_t)((rows + 127ull) / 128) * ((k + 255ull) / 256) * 2 * uq::kMxScaleTile;
    return 0;
}

int ug_mx4_quantize(const void *x, int type, uint32_t rows, uint32_t k, uint64_t stride, int layout, uint8_t *codes,
                    uint8_t *scales, void *stream) {
    if (!is_type(type) || (layout != UG_MX4_STORED && layout != UG_MX4_OPERAND))
        return fail(18, "ug_mx4_quantize: unknown type or layout");
    if (!sizes_ok(rows, k) || stride < k) return fail(18, "ug_mx4_quantize: sizes out of range or stride below k");
    if (!rows) return 0;
    if (!x || !codes || !scales || !is_aligned(x, type_bytes(type))) return fail(22, "ug_mx4_quantize: null or misaligned pointer");
    if (layout == UG_MX4_OPERAND && (!is_aligned(codes, 128) || !is_aligned(scales, 16)))
        return fail(22, "ug_mx4_quantize: operand codes need 128-byte and scales 16-byte alignment");
    OnDevice on;
    if (int rc = on.enter({x, codes, scales})) return rc;
    return launch([&] { return uq::launch_mx4_quantize(x, type, rows, k, stride, layout, codes, scales, static_cast<cudaStream_t>(stream)); });
}

int ug_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, int layout, uint32_t rows, uint32_t k, void *y,
                      int type, uint64_t stride, void *stream) {
    if (!is_type(type) || (layout != UG_MX4_STORED && layout != UG_MX4_OPERAND))
        return fail(18, "ug_mx4_dequantize: unknown type or layout");
    if (!sizes_ok(rows, k) || stride < k) return fail(18, "ug_mx4_dequantize: sizes out of range or stride below k");
    if (!rows) return 0;
    if (!y || !codes || !scales || !is_aligned(y, type_bytes(type)))
        return fail(22, "ug_mx4_dequantize: null or misaligned pointer");
    if (layout == UG_MX4_OPERAND && (!is_aligned(codes, 128) || !is_aligned(scales, 16)))
        return fail(22, "ug_mx4_dequantize: operand codes need 128-byte and scales 16-byte alignment");
    OnDevice on;
    if (int rc = on.enter({codes, scales, y})) return rc;
    return launch([&] { return uq::launch_mx4_dequantize(codes, scales, layout, rows, k, y, type, stride, static_cast<cudaStream_t>(stream)); });
}

uint32_t ug_mx4_pack_rows(uint32_t count, uint32_t rows, int paired) {
    const uint64_t per = paired ? 128ull * ((rows / 2 + 63ull) / 64) : 128ull * ((rows + 127ull) / 128);
    const uint64_t all = per * count;
    return all < (1ull << 32) ? (uint32_t)all : 0;
}

int ug_mx4_pack(const uint8_t *codes, const uint8_t *scales, uint32_t count, uint32_t rows, uint32_t k, int paired,
                uint8_t *packed_codes, uint8_t *packed_scales, void *stream) {
    if (paired != 0 && paired != 1) return fail(18, "ug_mx4_pack: paired must be 0 or 1");
    if (paired && rows % 2) return fail(18, "ug_mx4_pack: paired matrices need an even number of rows");
    const uint32_t all = ug_mx4_pack_rows(count, rows, paired);
    if (!count || !rows) {
        if (k < 1) return fail(18, "ug_mx4_pack: sizes out of range");
        return 0;
    }
    if (!all || !sizes_ok(all, k)) return fail(18, "ug_mx4_pack: sizes out of range");
    if (!codes || !scales || !packed_codes || !packed_scales) return fail(22, "ug_mx4_pack: null pointer");
    if (!is_aligned(packed_codes, 128) || !is_aligned(packed_scales, 16))
        return fail(22, "ug_mx4_pack: packed codes need 128-byte and scales 16-byte alignment");
    OnDevice on;
    if (int rc = on.enter({codes, scales, packed_codes, packed_scales})) return rc;
    return launch([&] {
        return uq::launch_mx4_pack(codes, scales, count, rows, k, paired, packed_codes, packed_scales, static_cast<cudaStream_t>(stream));
    });
}

static int product(uq::MxProductArgs &p, bool pieces, void *stream, const char *name) {
    if (!is_type(p.type)) return fail(18, name);
    // rows counted with their padding: whole tiles of m and n, up to four rows of pieces to a 16-bit token of m
    if (p.k < 1 || p.k > UG_MX4_MAX_K || p.m > UG_MX4_MAX_M || !sizes_ok(pieces ? (uint64_t)p.m * 4 + 256 : (uint64_t)p.m + 255, p.k) ||
        !sizes_ok((uint64_t)p.n + 127, p.k) || p.stride < p.n)
        return fail(18, name);
    if (!p.m || !p.n) return 0;
    const void *x = p.x ? p.x : p.a_codes;
    if (!p.w_codes || !p.w_scales || !p.y || !is_aligned(p.w_codes, 128) || !is_aligned(p.w_scales, 16) ||
        !is_aligned(p.y, type_bytes(p.type)))
        return fail(22, name);
    OnDevice on;
    if (int rc = on.enter({x, p.a_scales, p.w_codes, p.w_scales, p.y, p.workspace})) return rc;
    return launch([&] { return uq::launch_mx4_product(p, static_cast<cudaStream_t>(stream)); });
}

int ug_mx4_matmul(const uint8_t *a_codes, const uint8_t *a_scales, uint32_t m, const uint8_t *w_codes,
                  const uint8_t *w_scales, uint32_t n, uint32_t k, void *y, int type, uint64_t stride, void *stream) {
    if (m && n && (!a_codes || !a_scales || !is_aligned(a_codes, 128) || !is_aligned(a_scales, 16)))
        return fail(22, "ug_mx4_matmul: null or misaligned activations");
    uq::MxProductArgs p{};
    p.a_codes = a_codes;
    p.a_scales = a_scales;
    p.m = m;
    p.w_codes = w_codes;
    p.w_scales = w_scales;
    p.n = n;
    p.k = k;
    p.y = y;
    p.type = type;
    p.stride = stride;
    return product(p, false, stream, "ug_mx4_matmul: type, sizes, stride or pointers out of range");
}

size_t ug_mx4_matmul_x16_workspace(uint32_t m, uint32_t k, int x_type) {
    if (!is_half(x_type) || !k || uq::mx_fused(m, k, x_type)) return 0;
    const size_t rows = uq::mx_piece_rows(m, x_type), kt = (k + 127ull) / 128;
    return up(rows * kt * 128) + up((rows + 127) / 128 * kt * uq::kMxScaleTile);
}

int ug_mx4_matmul_x16(const void *x, int x_type, uint64_t x_stride, uint32_t m, const uint8_t *w_codes,
                      const uint8_t *w_scales, uint32_t n, uint32_t k, void *y, int type, uint64_t stride,
                      void *workspace, size_t workspace_bytes, void *stream) {
    if (!is_half(x_type) || x_stride < k) return fail(18, "ug_mx4_matmul_x16: x must be 16-bit with rows k apart or more");
    const size_t need = ug_mx4_matmul_x16_workspace(m, k, x_type);
    if (m && n && (!x || !is_aligned(x, 2) || (need && (!workspace || !is_aligned(workspace, 256)))))
        return fail(22, "ug_mx4_matmul_x16: null or misaligned x or workspace");
    if (m && n && workspace_bytes < need) return fail(22, "ug_mx4_matmul_x16: workspace too small");
    uq::MxProductArgs p{};
    p.x = x;
    p.x_type = x_type;
    p.x_stride = x_stride;
    p.m = m;
    p.w_codes = w_codes;
    p.w_scales = w_scales;
    p.n = n;
    p.k = k;
    p.y = y;
    p.type = type;
    p.stride = stride;
    p.workspace = need ? workspace : nullptr;
    return product(p, true, stream, "ug_mx4_matmul_x16: type, sizes, stride or pointers out of range");
}

size_t ug_mx4_experts_workspace(const UgMx4Experts *layer, uint32_t tokens) {
    if (check_layer(layer) || tokens > UG_MX4_MAX_TOKENS) return 0;
    return experts_scratch(*layer, tokens, nullptr, nullptr);
}

int ug_mx4_experts(const UgMx4Experts *layer, const void *x, uint64_t x_stride, uint32_t tokens, void *y,
                   uint64_t y_stride, int32_t *chosen, float *weights, void *workspace, size_t workspace_bytes,
                   void *stream) {
    if (int rc = check_layer(layer)) return rc;
    const UgMx4Experts &l = *layer;
    if (tokens > UG_MX4_MAX_TOKENS || x_stride < l.d || y_stride < l.d)
        return fail(18, "ug_mx4_experts: at most 128 tokens, strides of d or more");
    if (!tokens) return 0;
    if (!x || !y || !l.router || !l.gate_up_codes || !l.gate_up_scales || !l.down_codes || !l.down_scales || !workspace)
        return fail(22, "ug_mx4_experts: null pointer");
    if (!is_aligned(x, 2) || !is_aligned(y, 2) || !is_aligned(l.router, 2) || !is_aligned(l.bias, 4) ||
        !is_aligned(l.gate_up_codes, 128) || !is_aligned(l.gate_up_scales, 16) || !is_aligned(l.down_codes, 128) ||
        !is_aligned(l.down_scales, 16) || !is_aligned(chosen, 4) || !is_aligned(weights, 4) || !is_aligned(workspace, 256))
        return fail(22, "ug_mx4_experts: misaligned pointer");
    if (workspace_bytes < experts_scratch(l, tokens, nullptr, nullptr)) return fail(22, "ug_mx4_experts: workspace too small");
    OnDevice on;
    if (int rc = on.enter({x, y, l.router, l.bias, l.gate_up_codes, l.gate_up_scales, l.down_codes, l.down_scales, chosen,
                           weights, workspace}))
        return rc;
    uq::MxExpertsArgs a{};
    a.experts = l.experts;
    a.top_k = l.top_k;
    a.d = l.d;
    a.f = l.f;
    a.tokens = tokens;
    a.normalize = l.normalize;
    a.type = l.type;
    a.router = l.router;
    a.bias = l.bias;
    a.gate_up_codes = l.gate_up_codes;
    a.gate_up_scales = l.gate_up_scales;
    a.down_codes = l.down_codes;
    a.down_scales = l.down_scales;
    a.x = x;
    a.x_stride = x_stride;
    a.y = y;
    a.y_stride = y_stride;
    a.chosen = chosen;
    a.weights = weights;
    experts_scratch(l, tokens, static_cast<uint8_t *>(workspace), &a.ws);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (int rc = launch([&] { return uq::launch_mx4_router(a, s); })) return rc;
    return launch([&] { return uq::launch_mx4_expert_products(a, s); });
}

int ug_mx4_check(int device) {
    int count = 0, current = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count <= 0) {
        cudaGetLastError();
        return fail(2002, "no CUDA device");
    }
    if (device < 0 || device >= count) return fail(2002, "device index out of range");
    if (cudaGetDevice(&current) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return fail(2001, "cudaSetDevice");
    const cudaError_t e = cudaDeviceSynchronize();
    const int late = e == cudaSuccess ? uq::mx_tc_error(true) : 0;
    cudaSetDevice(current);
    if (late) return fail(2003, "MX4: a device-side wait timed out");
    return launched(e);
}

}  // extern "C"
