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
// 16 elements of a token's head per thread: head_dim / 16 neighbouring lanes hold a row, whose maximum is that of packed
// 16-bit magnitudes and two or three shuffles; a lane group takes one token and two of its heads, keys and values,
// so a token's place is computed once and four 32-byte loads are in flight.  Both kernels move each byte once:
// bound by DRAM at prompt sizes (16,000 tokens of 8 heads x 128 into e4m3: 20.4 us, 4.9 TB/s; read back: 20.6 us), by the
// launch at decoding sizes (1.7 us for 512 rows in a graph, 5 us as a call).  (One row and side per group of 16 lanes spent
// its time on addresses: 36 us; four heads per group on registers: 24 us.)
#include <cuda_fp8.h>

#include "bsa_common.cuh"

namespace bsa {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxFloor = 0x1p-100f;

constexpr int kWideHeads = 2;                   // at prompt sizes: 20.4 us, with 4: 24.4
// Tokens x heads below which a lane group takes one row.  8-bit writes of 8 heads x 128, one row / two heads of both sides, in
// a replayed graph: 512 rows 1.7 / 2.4 us, 4096 2.2 / 2.8, 8192 2.6 / 2.9, 16384 3.4 / 3.5, 32768 5.0 / 4.8, 128000 16.8 / 15.0.
constexpr int64_t kNarrowRows = 16384;

struct CacheParams {
    const void* src[2];             // write: the tokens' keys / values; read: the cache's
    void* dst[2];
    float* scales[2];               // e4m3 only
    int64_t token_stride[2], head_stride[2];      // of the tokens' tensors, in elements
    const int64_t* slots;
    int64_t slot_count;             // pages * page
    int tokens, heads, page_shift;
    int wide[2];                    // the tokens' rows start on 32 bytes
    uint32_t* status;
};

struct Words { uint32_t w[8]; };    // 16 elements of 16 bits

__device__ __forceinline__ Words load_words(const void* p, bool wide) {
    Words r;
    if (wide) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7]) : "l"(p));
    } else {
        *reinterpret_cast<uint4*>(r.w) = static_cast<const uint4*>(p)[0];
        *reinterpret_cast<uint4*>(r.w + 4) = static_cast<const uint4*>(p)[1];
    }
    return r;
}
__device__ __forceinline__ void store_words(void* p, const Words& r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7]) : "memory");
}

// The slot of a token; one behind the cache's end is reported and skipped like a negative one.
__device__ __forceinline__ int64_t checked_slot(const CacheParams& p, int token) {
    const int64_t slot = p.slots[token];
    if (slot < p.slot_count) return slot;
    atomicExch(p.status, (uint32_t)BSA_ERR_BAD_SHAPE);
    return -1;
}

template <typename T> __device__ __forceinline__ float2 unpack_word(uint32_t w);
template <> __device__ __forceinline__ float2 unpack_word<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 unpack_word<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// (an index that is not known when compiling would put the parameters into local memory)
template <typename A>
__device__ __forceinline__ A of(const A (&pair)[2], int side) { return side ? pair[1] : pair[0]; }

// kHeads heads and kSides of keys and values per lane group: 1 and 1 (the side in blockIdx.z) where the grid is small.
template <typename T, bool kE4m3, int kDim, int kHeads, int kSides>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheParams p) {
    constexpr int kLanes = kDim / 16, kTokens = 256 / kLanes;
    const int lane = threadIdx.x % kLanes, token = blockIdx.x * kTokens + threadIdx.x / kLanes;
    const int head0 = blockIdx.y * kHeads, heads = min(kHeads, p.heads - head0);
    const int side0 = kSides == 2 ? 0 : blockIdx.z;
    const int64_t slot = token < p.tokens ? checked_slot(p, token) : -1;
    // row of the cache: page, head, place
    const int64_t row = (((slot >> p.page_shift) * p.heads + head0) << p.page_shift) + (slot & ((1 << p.page_shift) - 1));
    Words x[kHeads][kSides];
    if (slot >= 0) {
#pragma unroll
        for (int i = 0; i < kSides; ++i) {
            const int side = side0 + i;
            const T* from = static_cast<const T*>(of(p.src, side)) + token * of(p.token_stride, side) + head0 * of(p.head_stride, side) + lane * 16;
#pragma unroll
            for (int h = 0; h < kHeads; ++h)
                if (h < heads) x[h][i] = load_words(from + h * of(p.head_stride, side), of(p.wide, side) != 0);
        }
    }
    if (!kE4m3) {
        if (slot < 0) return;
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
#pragma unroll
            for (int i = 0; i < kSides; ++i)
                if (h < heads) store_words(static_cast<T*>(of(p.dst, side0 + i)) + ((row + ((int64_t)h << p.page_shift)) * kDim + lane * 16), x[h][i]);
        return;
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
        if (h >= heads) break;
        const int64_t at = row + ((int64_t)h << p.page_shift);
#pragma unroll
        for (int i = 0; i < kSides; ++i) {
            const int side = side0 + i;
            const Words& v = x[h][i];
            // magnitudes compared as integers: the order of the bit patterns puts NaN above infinity, so neither is lost
            uint32_t top = v.w[0] & 0x7fff7fffu;
#pragma unroll
            for (int e = 1; e < 8; ++e) top = __vmaxu2(top, v.w[e] & 0x7fff7fffu);
#pragma unroll
            for (int s = kLanes / 2; s > 0; s >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, s));
            const float2 both = unpack_word<T>(top);
            const float amax = __uint_as_float(max(max(__float_as_uint(both.x), __float_as_uint(both.y)), __float_as_uint(kAmaxFloor)));
            const float inv = __fdiv_rn(kE4m3Max, amax);
            uint32_t codes[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 a = unpack_word<T>(v.w[2 * e]), b = unpack_word<T>(v.w[2 * e + 1]);
                codes[e] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a.x * inv, a.y * inv), __NV_SATFINITE, __NV_E4M3) |
                           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(b.x * inv, b.y * inv), __NV_SATFINITE, __NV_E4M3) << 16;
            }
            if (slot < 0) continue;
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(of(p.dst, side)) + at * kDim + lane * 16) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
            if (lane == 0) of(p.scales, side)[at] = __fdiv_rn(amax, kE4m3Max);
        }
    }
}

// Two codes (low 16 bits), scaled and rounded once to the 16-bit type.
template <typename T>
__device__ __forceinline__ uint32_t values2(uint32_t codes, float scale) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
    T r[2] = {Scalar<T>::from_float(v.x * scale), Scalar<T>::from_float(v.y * scale)};
    return *reinterpret_cast<const uint32_t*>(r);
}

template <typename T, bool kE4m3, int kDim, int kHeads, int kSides>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheParams p) {
    constexpr int kLanes = kDim / 16, kTokens = 256 / kLanes;
    const int lane = threadIdx.x % kLanes, token = blockIdx.x * kTokens + threadIdx.x / kLanes;
    if (token >= p.tokens) return;
    const int head0 = blockIdx.y * kHeads, heads = min(kHeads, p.heads - head0);
    const int side0 = kSides == 2 ? 0 : blockIdx.z;
    const int64_t slot = checked_slot(p, token);
    const int64_t row = (((slot >> p.page_shift) * p.heads + head0) << p.page_shift) + (slot & ((1 << p.page_shift) - 1));
    Words x[kHeads][kSides];
    float scale[kHeads][kSides];
#pragma unroll
    for (int i = 0; i < kSides; ++i)
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const int side = side0 + i;
            scale[h][i] = 0.0f;
            x[h][i] = Words{};
            if (h >= heads || slot < 0) continue;
            const int64_t at = row + ((int64_t)h << p.page_shift);
            if (kE4m3) {
                *reinterpret_cast<uint4*>(x[h][i].w) = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(of(p.src, side)) + at * kDim + lane * 16);
                scale[h][i] = of(p.scales, side)[at];
            } else {
                x[h][i] = load_words(static_cast<const T*>(of(p.src, side)) + at * kDim + lane * 16, true);
            }
        }
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
        for (int i = 0; i < kSides; ++i) {
            if (h >= heads) continue;
            Words v = x[h][i];
            if (kE4m3) {
#pragma unroll
                for (int e = 3; e >= 0; --e) {
                    const uint32_t c = v.w[e];
                    v.w[2 * e] = values2<T>(c & 0xffffu, scale[h][i]);
                    v.w[2 * e + 1] = values2<T>(c >> 16, scale[h][i]);
                }
            }
            store_words(static_cast<T*>(of(p.dst, side0 + i)) + ((int64_t)token * p.heads + head0 + h) * kDim + lane * 16, v);
        }
}

template <typename T, bool kE4m3, int kDim, int kHeads, int kSides>
int launch_shape(bool write, const CacheParams& p, cudaStream_t stream) {
    constexpr int kTokens = 256 / (kDim / 16);
    const dim3 grid((unsigned)((p.tokens + kTokens - 1) / kTokens), (unsigned)((p.heads + kHeads - 1) / kHeads), 2 / kSides);
    if (write) cache_write_kernel<T, kE4m3, kDim, kHeads, kSides><<<grid, 256, 0, stream>>>(p);
    else cache_read_kernel<T, kE4m3, kDim, kHeads, kSides><<<grid, 256, 0, stream>>>(p);
    return launch_status();
}
template <typename T, bool kE4m3, int kDim>
int launch(bool write, const CacheParams& p, cudaStream_t stream) {
    // few rows: one load per thread is the shortest way; many: four in flight
    const int64_t rows = (int64_t)p.tokens * p.heads;
    return rows < kNarrowRows ? launch_shape<T, kE4m3, kDim, 1, 1>(write, p, stream)
                              : launch_shape<T, kE4m3, kDim, kWideHeads, 2>(write, p, stream);
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
        // the cache is read and written 32 bytes at a time, and so is the output of a read
        if (!aligned16(p.src[side]) || (reinterpret_cast<uintptr_t>(p.dst[side]) & 31)) return BSA_ERR_ALIGNMENT;
        if (!write && (reinterpret_cast<uintptr_t>(p.src[side]) & 31)) return BSA_ERR_ALIGNMENT;
        if (p.token_stride[side] < 0 || p.head_stride[side] < 0) return BSA_ERR_BAD_SHAPE;
        if (p.token_stride[side] % 8 != 0 || p.head_stride[side] % 8 != 0) return BSA_ERR_ALIGNMENT;
        p.wide[side] = (reinterpret_cast<uintptr_t>(p.src[side]) & 31) == 0 && p.token_stride[side] % 16 == 0 && p.head_stride[side] % 16 == 0;
    }
    if (!p.slots) return BSA_ERR_NULL_POINTER;
    if (tokens > (int64_t)INT32_MAX - 256) return BSA_ERR_TOO_LARGE;                        // 32-bit token numbers
    p.slot_count = pages * page;
    p.tokens = (int)tokens;
    p.heads = (int)heads;
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
