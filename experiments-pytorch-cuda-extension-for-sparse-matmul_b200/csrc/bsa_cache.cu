// Paged key / value cache: writing the keys and values of new tokens, and reading places back.
//
// The cache is [pages, heads, page, head_dim]; a token lives at slot = page_id * page + place.  Two forms:
//   * 16 bits: the tokens' own type, copied;
//   * e4m3 with one fp32 scale per token, head and side:
//         a = max(max_d |x_d|, 2^-100)     scale = a / 448     code_d = e4m3(x_d * (448 / a))
//     (round to nearest even; 448 is e4m3's largest value).  The floor keeps 448 / a finite; a row that holds an
//     infinity or a NaN gets a scale that is none either, so it never reads back as ordinary numbers.
//     Reading gives round16(code * scale): one rounding to 16 bits, of the product held in fp32.
//
// One 16-byte chunk (8 elements) of a token's head per thread: head_dim / 8 neighbouring lanes hold one row, its maximum
// is log2(head_dim / 8) shuffles, every load is 16 bytes and every store 8 (codes) or 16.  Both kernels move each byte
// once: bound by DRAM at prompt sizes, by the launch at decoding sizes.
#include <cuda_fp8.h>

#include "bsa_common.cuh"

namespace bsa {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxFloor = 0x1p-100f;

struct CacheParams {
    const void* src[2];             // write: the tokens' keys / values; read: the cache's
    void* dst[2];
    float* scales[2];               // e4m3 only
    int64_t token_stride[2], head_stride[2];      // of the tokens' tensors, in elements
    const int64_t* slots;
    int64_t slot_count;             // pages * page
    uint32_t rows, heads;           // rows = tokens * heads
    int page_shift;
    uint32_t* status;
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Scalar<T>::to_float(e[i]);
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// A slot behind the cache's end is reported and skipped like a negative one.
__device__ __forceinline__ int64_t checked_slot(const CacheParams& p, uint32_t token) {
    const int64_t slot = p.slots[token];
    if (slot < p.slot_count) return slot;
    atomicExch(p.status, (uint32_t)BSA_ERR_BAD_SHAPE);
    return -1;
}

// Row of the cache that holds `slot` of `head`.
__device__ __forceinline__ int64_t cache_row(const CacheParams& p, int64_t slot, uint32_t head) {
    return (((slot >> p.page_shift) * p.heads + head) << p.page_shift) + (slot & ((1 << p.page_shift) - 1));
}

// kRows: rows of a lane group, 1 where the grid is small (a decoding step), 4 at prompt sizes, so that four loads are in
// flight per thread.
template <typename T, bool kE4m3, int kDim, int kRows>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheParams p) {
    constexpr int kLanes = kDim / 8;
    constexpr uint32_t kStep = 256 / kLanes;
    const int side = blockIdx.y, lane = threadIdx.x % kLanes;
    const uint32_t first = blockIdx.x * (kRows * kStep) + threadIdx.x / kLanes;
    uint4 w[kRows];
    int64_t at[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t row = first + i * kStep;
        at[i] = -1;
        w[i] = make_uint4(0, 0, 0, 0);
        if (row >= p.rows) continue;
        const uint32_t token = row / p.heads, head = row - token * p.heads;
        w[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.src[side]) + token * p.token_stride[side] +
                                               head * p.head_stride[side] + lane * 8);
        const int64_t slot = checked_slot(p, token);
        if (slot >= 0) at[i] = cache_row(p, slot, head);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (kE4m3) {
            float x[8];
            unpack8<T>(w[i], x);
            // magnitudes compared as integers: the order of the bit patterns puts NaN above infinity, so neither is lost
            uint32_t top = __float_as_uint(kAmaxFloor);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
            for (int s = kLanes / 2; s > 0; s >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
            const float amax = __uint_as_float(top), inv = __fdiv_rn(kE4m3Max, amax);
            if (at[i] < 0) continue;
            uint2 c;
            c.x = codes4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
            c.y = codes4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.dst[side]) + at[i] * kDim + lane * 8) = c;
            if (lane == 0) p.scales[side][at[i]] = __fdiv_rn(amax, kE4m3Max);
        } else if (at[i] >= 0) {
            *reinterpret_cast<uint4*>(static_cast<T*>(p.dst[side]) + at[i] * kDim + lane * 8) = w[i];
        }
    }
}

__device__ __forceinline__ float2 values2(uint32_t codes) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <typename T, bool kE4m3, int kDim, int kRows>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheParams p) {
    constexpr int kLanes = kDim / 8;
    constexpr uint32_t kStep = 256 / kLanes;
    const int side = blockIdx.y, lane = threadIdx.x % kLanes;
    const uint32_t first = blockIdx.x * (kRows * kStep) + threadIdx.x / kLanes;
    int64_t at[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t row = first + i * kStep;
        at[i] = -1;
        if (row >= p.rows) continue;
        const uint32_t token = row / p.heads;
        const int64_t slot = checked_slot(p, token);
        if (slot >= 0) at[i] = cache_row(p, slot, row - token * p.heads);
    }
    uint4 w[kRows];
    float scale[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        w[i] = make_uint4(0, 0, 0, 0);
        scale[i] = 0.0f;
        if (at[i] < 0) continue;
        if (kE4m3) {
            const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.src[side]) + at[i] * kDim + lane * 8);
            w[i].x = c.x; w[i].y = c.y;
            scale[i] = p.scales[side][at[i]];
        } else {
            w[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.src[side]) + at[i] * kDim + lane * 8);
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t row = first + i * kStep;
        if (row >= p.rows) continue;
        if (kE4m3) {
            const uint32_t c[4] = {w[i].x & 0xffffu, w[i].x >> 16, w[i].y & 0xffffu, w[i].y >> 16};
            uint4 out;
            T* e = reinterpret_cast<T*>(&out);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float2 v = values2(c[u]);
                e[2 * u] = Scalar<T>::from_float(v.x * scale[i]);
                e[2 * u + 1] = Scalar<T>::from_float(v.y * scale[i]);
            }
            w[i] = out;
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(p.dst[side]) + (size_t)row * kDim + lane * 8) = w[i];
    }
}

template <typename T, bool kE4m3, int kDim>
int launch(bool write, const CacheParams& p, cudaStream_t stream) {
    constexpr uint32_t kStep = 256 / (kDim / 8);
    // 4 rows per lane group once even that grid fills the SMs (148 x 8 CTAs)
    const bool wide = p.rows >= 2u * 1184u * kStep;
    const uint32_t per_cta = kStep * (wide ? 4 : 1);
    const dim3 grid((p.rows + per_cta - 1) / per_cta, 2);
    if (write) {
        if (wide) cache_write_kernel<T, kE4m3, kDim, 4><<<grid, 256, 0, stream>>>(p);
        else cache_write_kernel<T, kE4m3, kDim, 1><<<grid, 256, 0, stream>>>(p);
    } else {
        if (wide) cache_read_kernel<T, kE4m3, kDim, 4><<<grid, 256, 0, stream>>>(p);
        else cache_read_kernel<T, kE4m3, kDim, 1><<<grid, 256, 0, stream>>>(p);
    }
    return launch_status();
}

template <typename T>
int launch_typed(bool write, int store, int64_t dim, const CacheParams& p, cudaStream_t stream) {
    if (store == BSA_CACHE_E4M3)
        return dim == 64 ? launch<T, true, 64>(write, p, stream) : launch<T, true, 128>(write, p, stream);
    return dim == 64 ? launch<T, false, 64>(write, p, stream) : launch<T, false, 128>(write, p, stream);
}

int run_cache(bool write, int dtype, int store, CacheParams& p, int64_t tokens, int64_t pages, int64_t heads, int64_t page,
              int64_t dim, void* workspace, size_t workspace_bytes, void* stream) {
    const int checked = check_cache(dtype, store, p.scales[0], p.scales[1], pages, heads, page, dim);
    if (checked != BSA_OK) return checked;
    if (tokens < 0) return BSA_ERR_BAD_SHAPE;
    if (!workspace || workspace_bytes < BSA_WORKSPACE_BYTES) return BSA_ERR_WORKSPACE;
    if (tokens == 0) return BSA_OK;
    for (int side = 0; side < 2; ++side) {
        if (!p.src[side] || !p.dst[side]) return BSA_ERR_NULL_POINTER;
        if (!aligned16(p.src[side]) || !aligned16(p.dst[side])) return BSA_ERR_ALIGNMENT;
        if (p.token_stride[side] < 0 || p.head_stride[side] < 0) return BSA_ERR_BAD_SHAPE;
        if (p.token_stride[side] % 8 != 0 || p.head_stride[side] % 8 != 0) return BSA_ERR_ALIGNMENT;
    }
    if (!p.slots) return BSA_ERR_NULL_POINTER;
    if (tokens > (int64_t)INT32_MAX / (heads * (dim / 8))) return BSA_ERR_TOO_LARGE;       // 32-bit chunk numbers
    p.slot_count = pages * page;
    p.rows = (uint32_t)(tokens * heads);
    p.heads = (uint32_t)heads;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page) ++p.page_shift;
    p.status = static_cast<uint32_t*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == BSA_DTYPE_F16 ? launch_typed<__half>(write, store, dim, p, s)
                                  : launch_typed<__nv_bfloat16>(write, store, dim, p, s);
}

}  // namespace

int check_cache(int dtype, int store, const float* key_scales, const float* value_scales, int64_t pages, int64_t heads,
                int64_t page, int64_t dim) {
    if (dtype != BSA_DTYPE_F16 && dtype != BSA_DTYPE_BF16) return BSA_ERR_BAD_DTYPE;
    if (store != BSA_CACHE_SAME && store != BSA_CACHE_E4M3) return BSA_ERR_BAD_MODE;
    if (store == BSA_CACHE_E4M3 && (!key_scales || !value_scales)) return BSA_ERR_NULL_POINTER;
    if (page != 16 && page != 32 && page != 64 && page != 128) return BSA_ERR_BAD_BLOCK;
    if (pages <= 0 || heads <= 0 || (dim != 64 && dim != 128)) return BSA_ERR_BAD_SHAPE;
    if (heads > 65535 || pages > (int64_t)INT32_MAX / (heads * page)) return BSA_ERR_TOO_LARGE;      // 32-bit row numbers
    return BSA_OK;
}

}  // namespace bsa

extern "C" int bsa_cache_write(int dtype, int store, const void* k, const void* v, int64_t k_token_stride,
                               int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots,
                               int64_t tokens, void* keys, void* values, float* key_scales, float* value_scales,
                               int64_t pages, int64_t heads, int64_t page, int64_t head_dim, void* workspace,
                               size_t workspace_bytes, void* stream) {
    bsa::CacheParams p{};
    p.src[0] = k; p.src[1] = v;
    p.dst[0] = keys; p.dst[1] = values;
    p.scales[0] = key_scales; p.scales[1] = value_scales;
    p.token_stride[0] = k_token_stride; p.token_stride[1] = v_token_stride;
    p.head_stride[0] = k_head_stride; p.head_stride[1] = v_head_stride;
    p.slots = slots;
    return bsa::run_cache(true, dtype, store, p, tokens, pages, heads, page, head_dim, workspace, workspace_bytes, stream);
}

extern "C" int bsa_cache_read(int dtype, int store, const int64_t* slots, int64_t tokens, const void* keys,
                              const void* values, const float* key_scales, const float* value_scales, void* k, void* v,
                              int64_t pages, int64_t heads, int64_t page, int64_t head_dim, void* workspace,
                              size_t workspace_bytes, void* stream) {
    bsa::CacheParams p{};
    p.src[0] = keys; p.src[1] = values;
    p.dst[0] = k; p.dst[1] = v;
    p.scales[0] = const_cast<float*>(key_scales); p.scales[1] = const_cast<float*>(value_scales);
    p.slots = slots;
    return bsa::run_cache(false, dtype, store, p, tokens, pages, heads, page, head_dim, workspace, workspace_bytes, stream);
}
