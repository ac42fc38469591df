// What the packed attention kernels share: finding a CTA's rows, 128-row operand tiles, TMEM accesses of one row per
// thread, tensor maps over [tokens, heads, head_dim] with strides.
#pragma once
#include "bsa_tc_common.cuh"

namespace bsa {
namespace {

constexpr int kRowsTile = 128;                              // query rows / keys of a tile: the M of an MMA
constexpr int kPanelBytes = kRowsTile * 128;                // 128 rows x 64 elements of 16 bits, 128-byte swizzle
constexpr float kPackedLog2e = 1.4426950408889634f;

// One sequence's tile, or (b == batch) a tile of the rows behind the last sequence, which hold zeros.
struct PackedItem {
    int start, length, tile, b;                             // first row and rows of the sequence; length 0: nothing to do
};

__device__ __forceinline__ int warp_sum(int x) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
// Item `rank` of the list of all tiles of `per_tile` rows, called by one warp; nothing about the offsets is known on the
// host.  The list goes by the number of a tile in its sequence, the largest first (of a causal sequence the later tiles
// are the longer ones, so this is longest first over all sequences), and by the sequence's number among equals; the tiles of the
// rows behind the last sequence come last.  F(t) = sum_b max(0, tiles_b - t) items have a number of t or more, so the
// item's number is the largest t with F(t) > rank, found by bisection.
// Offsets that are not 0 = o_0 <= o_1 <= .. <= rows are reported, and clamped so that nothing outside the tensors is
// touched.
__device__ __forceinline__ PackedItem packed_locate(const int32_t* offsets, int batch, int rows, int per_tile, int rank,
                                                    int lane, uint32_t* status) {
    const auto span = [&](int b, int& start) {              // rows of sequence b
        start = 0;
        if (b >= batch) return 0;
        start = min(max(offsets[b], 0), rows);
        return min(max(offsets[b + 1], start), rows) - start;
    };
    int most = 0, all = 0;
    for (int b = lane; b < batch; b += 32) {
        int start;
        const int length = span(b, start), tiles = (length + per_tile - 1) / per_tile;
        if (offsets[b] != start || offsets[b + 1] != start + length || (b == 0 && start != 0)) atomicExch(status, (uint32_t)BSA_ERR_BAD_SHAPE);
        most = max(most, tiles);
        all += tiles;
    }
    most = (int)__reduce_max_sync(0xffffffffu, (uint32_t)most);
    all = warp_sum(all);
    PackedItem item{0, 0, 0, 0};
    if (rank >= all) {
        const int behind = min(max(offsets[batch], 0), rows);
        if (rank - all < (rows - behind + per_tile - 1) / per_tile) item = PackedItem{behind, rows - behind, rank - all, batch};
        return item;
    }
    int t = 0, end = most, above = 0;                       // F(t) > rank >= F(end) = above
    while (end - t > 1) {
        const int mid = (t + end) / 2;
        int f = 0;
        for (int b = lane; b < batch; b += 32) {
            int start;
            f += max((span(b, start) + per_tile - 1) / per_tile - mid, 0);
        }
        f = warp_sum(f);
        if (f > rank) t = mid;
        else { end = mid; above = f; }
    }
    int nth = rank - above;                                 // among the sequences that have a tile t
    for (int b0 = 0; b0 < batch; b0 += 32) {
        int start;
        const int length = span(b0 + lane, start);
        uint32_t has = __ballot_sync(0xffffffffu, (length + per_tile - 1) / per_tile > t);
        if (nth >= __popc(has)) { nth -= __popc(has); continue; }
        for (; nth > 0; --nth) has &= has - 1;
        const int l = __ffs(has) - 1;
        item.start = __shfl_sync(0xffffffffu, start, l);
        item.length = __shfl_sync(0xffffffffu, length, l);
        item.tile = t;
        item.b = b0 + l;
        break;
    }
    return item;
}

// Operand descriptor of a 128-row tile in 64-element panels: K-major (a row is one M / N index) or MN-major (a row is
// one K index; the leading offset is the distance of the panels, which hold consecutive 64-wide ranges of M / N).
__device__ __forceinline__ uint64_t panel_desc(uint32_t smem_addr, bool mn_major) {
    uint64_t d = (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(mn_major ? (kPanelBytes >> 4) : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// D[128 x 128] = A B^T over head_dim, both operands K-major in shared memory.
template <int kDim>
__device__ __forceinline__ void mma_rows(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
    for (int kk = 0; kk < kDim / 16; ++kk) {
        const uint64_t at = (uint64_t)((kk / 4) * (kPanelBytes >> 4) + (kk % 4) * 2);
        tc_mma_f16(tmem_d, a + at, b + at, idesc, kk > 0 ? 1u : 0u);
    }
}
// D[128 x head_dim] (+)= A B over half of a tile's keys, A in tensor memory as 16-bit pairs, B MN-major.  kPart 0: keys
// 0-63, 1: keys 64-127.
template <int kPart>
__device__ __forceinline__ void mma_keys(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, bool accumulate) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int kk = 4 * kPart + i;
        tc_mma_f16_ts(tmem_d, tmem_a + (uint32_t)(8 * kk), b + (uint64_t)(kk * (2048 >> 4)), idesc, accumulate || i > 0 ? 1u : 0u);
    }
}
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, int* abort_flag, uint32_t* status) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status)) != 0;
}
__device__ __forceinline__ void arrive_warp(uint64_t* bar, int lane) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}
__device__ __forceinline__ void tc_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
// the first 16 words of r
__device__ __forceinline__ void tc_st_32x32b_x16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tc_st_32x32b_x32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}

__device__ __forceinline__ void tc_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

__device__ __forceinline__ uint64_t f2_of(uint32_t lo, uint32_t hi) { return f2_pack(__uint_as_float(lo), __uint_as_float(hi)); }

// Zeroes rows [from, 128) of a tile in shared memory (all lanes of a warp), for the tensor cores to read: what TMA
// brought there belongs to another sequence, and 0 times a NaN of it would be NaN.
template <int kDim>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from, int lane) {
#pragma unroll
    for (int panel = 0; panel < kDim / 64; ++panel)
        for (int at = from * 128 + lane * 16; at < kPanelBytes; at += 512)
            *reinterpret_cast<uint4*>(tile + panel * kPanelBytes + at) = make_uint4(0u, 0u, 0u, 0u);
    fence_async_shared();
    __syncwarp();
}

// 32 fp32 values of a row, rounded, to global memory (64 bytes, 32-byte aligned).
template <bool kBf16>
__device__ __forceinline__ void store_row32(void* to, const uint32_t (&r)[32], float by) {
    uint32_t w[8];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i] = pack2<kBf16>(__uint_as_float(r[16 * half + 2 * i]) * by, __uint_as_float(r[16 * half + 2 * i + 1]) * by);
        st_global_v8(static_cast<uint8_t*>(to) + 32 * half, w);
    }
}

// Rows of a warp to global memory, 64 columns at a time: through shared memory (`stage`: 32 rows x 128 bytes of this warp,
// swizzled) and a TMA store where all 32 rows belong to the sequence, else row by row.  (A row per thread stored straight
// from registers touches 32 lines per instruction: an epilogue of 128 x 128 took 3000-4000 cycles.)
__device__ __forceinline__ void store_done() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_rows64(uint8_t* stage, const CUtensorMap* map, const uint32_t (&w)[32], int column, int head,
                                             int row, int lane) {
    if (lane == 0) store_done();                // the last store has read the stage
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 8; ++u)
        *reinterpret_cast<uint4*>(stage + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
    fence_async_shared();
    __syncwarp();
    if (lane == 0)
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];\n\tcp.async.bulk.commit_group;"
                     ::"l"(map), "r"(smem_u32(stage)), "r"(column), "r"(head), "r"(row) : "memory");
}
// The same 64 columns of one row from its thread (32-byte aligned).
__device__ __forceinline__ void store_row64(void* to, const uint32_t (&w)[32]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t part[8] = {w[8 * q], w[8 * q + 1], w[8 * q + 2], w[8 * q + 3], w[8 * q + 4], w[8 * q + 5], w[8 * q + 6], w[8 * q + 7]};
        st_global_v8(static_cast<uint8_t*>(to) + 32 * q, part);
    }
}
// Two values that a word of 16-bit values stands for.
template <bool kBf16>
__device__ __forceinline__ float2 word_values(uint32_t w) {
    if (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Zero rows [from, to) of a contiguous 16-bit [rows, heads, head_dim] tensor, one head, by thread `me` of `threads`.
__device__ __forceinline__ void zero_tail(void* base, int from, int to, int head, int heads, int dim, int me, int threads) {
    const int chunks = dim / 8;
    for (int i = me; i < (to - from) * chunks; i += threads) {
        const int row = from + i / chunks, c = i % chunks;
        reinterpret_cast<uint4*>(base)[((size_t)row * heads + head) * chunks + c] = make_uint4(0u, 0u, 0u, 0u);
    }
}

// Tensor map over [tokens, heads, head_dim] (16 bits, strides in elements): boxes of 64 elements x 1 head x box_rows tokens.
// Rows behind the last read as zero.
bool make_packed_map(CUtensorMap* map, int dtype, const void* base, int64_t tokens, int64_t heads, int64_t dim,
                     int64_t token_stride, int64_t head_stride, int box_rows = kRowsTile) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUtensorMapDataType type = dtype == BSA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return fn(map, type, 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The driver's encoder needs the device's context bound to the calling thread.
bool bind_device() {
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) return true;
    cudaGetLastError();
    return false;
}

// Checks of the types and sizes of both directions.
int check_packed(int dtype, int64_t rows, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim) {
    if (dtype != BSA_DTYPE_F16 && dtype != BSA_DTYPE_BF16) return BSA_ERR_BAD_DTYPE;
    if (dim != 64 && dim != 128) return BSA_ERR_BAD_SHAPE;
    if (rows < 0 || batch < 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0) return BSA_ERR_BAD_SHAPE;
    // Every item looks through the offsets of all sequences, so the time grows with the square of their number: sequences of
    // one row, 4 heads of 64, forward: 1.4 ms for 4,096, 19 ms for 16,384, 0.57 s for 65,536.  A million would hold the
    // device for minutes.
    if (batch > 65536) return BSA_ERR_TOO_LARGE;
    // 32-bit rows, tiles and CTA numbers
    if (rows > (int64_t)INT32_MAX - 256 || q_heads > 65535) return BSA_ERR_TOO_LARGE;
    if ((rows / kRowsTile + batch + 2) * q_heads > (int64_t)INT32_MAX) return BSA_ERR_TOO_LARGE;
    return BSA_OK;
}
int check_strides(int64_t token_stride, int64_t head_stride) {
    if (token_stride <= 0 || head_stride <= 0 || token_stride >= (1ll << 38) || head_stride >= (1ll << 38)) return BSA_ERR_BAD_SHAPE;
    return token_stride % 8 || head_stride % 8 ? BSA_ERR_ALIGNMENT : BSA_OK;
}

}  // namespace
}  // namespace bsa
