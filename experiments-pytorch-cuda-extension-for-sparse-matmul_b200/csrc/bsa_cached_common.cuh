// What the kernels of attention over a paged cache share: their parameters, and how the tiles of a batch are shared out.
#pragma once
#include "bsa_tc_common.cuh"

namespace bsa {

struct CachedParams {
    const void* q;
    void* o;
    int64_t q_batch, q_draft, q_head;           // strides of q in elements
    const float* scales[2];
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* counts;                      // may be null
    const int64_t* tree;                        // may be null
    const uint8_t* pattern;                     // may be null: [pattern_rows, pattern_cols] of 1 << pattern_shift tokens
    int pattern_rows, pattern_cols, pattern_shift;
    int batch, drafts, group, kv_heads, row_tiles, table_width, pages, page_shift;
    float scale_log2;                           // scale * log2 e
    float* partial;                             // [ctas][2][rows][head_dim], then [ctas][2][rows][2] of (m, l)
    int ctas;
    uint32_t* status;
};

struct Share {
    int64_t per, first, end;        // units per CTA; this CTA's range
    int b, hm, tile;                // where the range starts
};

namespace {

// The lowest n bits.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }

__device__ __forceinline__ int cached_length(const CachedParams& p, int b) {
    return min(max(p.lengths[b], 0), p.table_width << p.page_shift);
}
template <int kTile>
__device__ __forceinline__ int cached_tiles(const CachedParams& p, int b) {
    return max(1, (cached_length(p, b) + kTile - 1) / kTile);
}

// Units of one head and row tile of the whole batch, and of the sequences before `part` (in `before`), by one warp.
template <int kTile, int kBegin>
__device__ __forceinline__ int64_t total_cost(const CachedParams& p, int part, int64_t& before, int lane) {
    int64_t sum = 0, some = 0;
#pragma unroll 4
    for (int b = lane; b < p.batch; b += 32) {
        const int cost = cached_tiles<kTile>(p, b) + kBegin;
        sum += cost;
        if (b < part) some += cost;
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, s);
        some += __shfl_xor_sync(0xffffffffu, some, s);
    }
    before = some;
    return sum;
}
// a / b; the units fit 32 bits unless a batch holds more keys than the device's memory
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// A (sequence, head, row tile) takes kBegin + tiles units of the list, its tiles last.  Finds where this CTA's share
// starts; a share that starts inside the first kBegin units starts at tile 0.
template <int kTile, int kBegin>
__device__ __forceinline__ Share find_share(const CachedParams& p, int cta, int lane) {
    Share s;
    const int hms = p.kv_heads * p.row_tiles;
    // (the first 32 sequences stay in registers: with no more than those there is one load on the way to the first tile)
    const int first = lane < p.batch ? cached_tiles<kTile>(p, lane) + kBegin : 0;
    int64_t sum = first;
    for (int b = 32 + lane; b < p.batch; b += 32) sum += cached_tiles<kTile>(p, b) + kBegin;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const int64_t units = sum * hms;
    s.per = quotient(units + p.ctas - 1, p.ctas);
    s.first = min((int64_t)cta * s.per, units);
    s.end = min(s.first + s.per, units);
    s.b = s.hm = s.tile = 0;
    if (s.first >= s.end) return s;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int mine = b0 == 0 ? first : (b0 + lane < p.batch ? cached_tiles<kTile>(p, b0 + lane) + kBegin : 0);
        int64_t upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, s.first < (before + upto) * hms);
        if (past) {
            const int l = __ffs(past) - 1;
            const int cost = __shfl_sync(0xffffffffu, mine, l);
            const int64_t start = before + __shfl_sync(0xffffffffu, upto, l) - cost;
            const int64_t off = s.first - start * hms;
            s.b = b0 + l;
            s.hm = (int)quotient(off, cost);
            const int within = (int)(off - (int64_t)s.hm * cost);
            s.tile = max(within - kBegin, 0);
            s.first += max(kBegin - within, 0);             // the unit of that tile
            return s;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return s;
}

// Map of a side of the cache as rows of head_dim elements, one page (at most a tile of it) per box.
bool make_cache_map(CUtensorMap* map, int store, int dtype, const void* base, int64_t rows, int64_t dim, int piece) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const int es = store == BSA_CACHE_E4M3 ? 1 : 2, row_bytes = (int)dim * es, panel = row_bytes < 128 ? row_bytes : 128;
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)rows, 1};
    const cuuint64_t strides[2] = {(cuuint64_t)row_bytes, (cuuint64_t)row_bytes * (cuuint64_t)rows};
    const cuuint32_t box[3] = {(cuuint32_t)(panel / es), (cuuint32_t)piece, 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUtensorMapDataType type = es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                             : (dtype == BSA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
    return fn(map, type, 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              panel == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

// The variant for many query rows over a 16-bit cache (tcgen05): scratch bytes, and the two launches.
size_t cached_wide_scratch(int64_t head_dim);
int cached_wide(const CachedParams& p, int dtype, int64_t head_dim, const void* keys, const void* values, int64_t page,
                cudaStream_t stream);

}  // namespace bsa
