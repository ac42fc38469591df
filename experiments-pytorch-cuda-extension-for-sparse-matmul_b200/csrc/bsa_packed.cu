// Attention inside the sequences of a packed batch, forward (sm_100a only):
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i),  j in the sequence of i, and j <= i if causal
// with q [rows, q_heads, D], k and v [rows, kv_heads, D], D 64 or 128, q_heads a multiple of kv_heads.
//
// One pass over the keys with the running row maximum m and sum l: S = Q K^T on the tensor cores into TMEM, one thread
// per row turns it into P = 2^(c S - m) (c = scale log2 e), 16 bits, back into TMEM as the A operand of O += P V, which
// stays in TMEM; O / l goes out at the end.  m is raised only when a tile's maximum exceeds it by more than 8 (then O is
// scaled by 2^(m_old - m_new) in TMEM), so P <= 2^8 and O and l carry the same factor whatever m is.
//
// A CTA (one per SM) works on two Q tiles of 128 rows that read the same K and V tiles, so that the tensor cores work
// on one while the other is in its softmax: two heads of one key head where the group is even (every K / V tile serves
// both, and rows go in steps of 128), else two neighbouring tiles of one head.  Per tile of 128 keys that is
// 8 x 128 x 128 x D operations, 1024 x D / 64 cycles of the tensor pipe at its peak, and 2 x 128 x 128 exponentials,
// 2048 cycles of the four MUFU units: at D = 128 the two balance, at D = 64 the exponentials bind.
//
//   warps 0-3, 4-7   softmax of tile 0 / 1, one row per thread; the epilogue
//   warp 8           TMA producer: Q, then K and V tiles through a ring of 4 stages
//   warp 9           MMA issuer: S0 S1 | PV0 S0' PV1 S1' | ..
// The last K / V tile of a sequence may hold rows of the next one; its V rows are zeroed before use (see zero_rows).
// All waits are bounded.
#include "bsa_packed_common.cuh"

namespace bsa {
namespace {

constexpr int kFwdStages = 4;
constexpr int kFwdThreads = 384;                // 10 warps work; 3 warpgroups are needed to hand out registers

struct PackedParams {
    void* o;
    float* lse;                                 // [q_heads, rows], in units of log2, scale included; may be null
    const int32_t* offsets;
    int batch, rows, q_heads, kv_heads, group, causal;
    int pair;                                   // the two tiles: heads 2 h, 2 h + 1 of a group (1), or rows (0)
    float scale_log2;                           // |scale| log2 e
    int negative;                               // scale < 0
    uint32_t* status;
};

struct __align__(8) FwdBarriers {
    uint64_t q_full, full[kFwdStages], empty[kFwdStages];
    uint64_t s_full[2], p_full[2], o_full[2];
    uint64_t drain;
    PackedItem item;
    uint32_t tmem_base;
    int abort_flag;
};

template <int kDim>
constexpr int fwd_smem() { return (2 + kFwdStages) * (kDim / 64) * kPanelBytes + (int)sizeof(FwdBarriers); }

template <bool kBf16, int kDim>
__global__ void __launch_bounds__(kFwdThreads, 1)
packed_forward_kernel(const PackedParams p, const __grid_constant__ CUtensorMap map_q,
                      const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    constexpr int kPanels = kDim / 64, kTileBytes_ = kPanels * kPanelBytes;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* ring = smem + 2 * kTileBytes_;
    FwdBarriers* bars = reinterpret_cast<FwdBarriers*>(ring + kFwdStages * kTileBytes_);
    int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_tile = p.pair ? kRowsTile : 2 * kRowsTile;
    const int head_items = p.pair ? p.q_heads / 2 : p.q_heads;
    const int rank = (int)blockIdx.x / head_items, head_item = (int)blockIdx.x - rank * head_items;

    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 8) {
        const PackedItem found = packed_locate(p.offsets, p.batch, p.rows, per_tile, rank, lane, p.status);
        if (lane == 0) {
            bars->item = found;
            *abort_flag = 0;
            mbar_init(&bars->q_full, 1);
            for (int i = 0; i < kFwdStages; ++i) { mbar_init(&bars->full[i], 1); mbar_init(&bars->empty[i], 1); }
            for (int i = 0; i < 2; ++i) { mbar_init(&bars->s_full[i], 1); mbar_init(&bars->p_full[i], 128); mbar_init(&bars->o_full[i], 1); }
            mbar_init(&bars->drain, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            fence_async_shared();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&bars->tmem_base;
    const PackedItem item = bars->item;
    const int head0 = p.pair ? 2 * head_item : head_item;       // tile s: head head0 + s (pair) or rows + 128 s
    const int tiles = (item.length + per_tile - 1) / per_tile;
    // the later tiles of a causal sequence are the longer ones: they go first
    const int tile = tiles - 1 - item.tile;
    const int row0 = tile * per_tile;                           // in the sequence
    const bool work = item.length > 0 && item.b < p.batch;
    // K / V tiles of each Q tile
    int steps[2] = {0, 0};
    if (work) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int first = p.pair ? row0 : row0 + s * kRowsTile;
            if (first < item.length) {
                const int keys = p.causal ? min(first + kRowsTile, item.length) : item.length;
                steps[s] = (keys + kRowsTile - 1) / kRowsTile;
            }
        }
    }
    const int all_steps = max(steps[0], steps[1]);
    const uint32_t fmt = kBf16 ? 1u : 0u;
    const uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRowsTile >> 4) << 24);

    if (item.length > 0 && item.b == p.batch) {                 // rows behind the last sequence
        const int from = item.start + item.tile * per_tile, to = min(from + per_tile, p.rows);
        for (int h = head0; h <= head0 + p.pair; ++h) {
            zero_tail(p.o, from, to, h, p.q_heads, kDim);
            if (p.lse)
                for (int r = from + (int)threadIdx.x; r < to; r += blockDim.x) p.lse[(size_t)h * p.rows + r] = -INFINITY;
        }
    }
    if (warp == 8) {
        // ------------------------------------------------------------ producer
        if (all_steps > 0) {
            const int kv_head = head0 / p.group;
            bool ok = true;
            if (elect_one()) {
                mbar_expect_tx(&bars->q_full, (uint32_t)(2 * kTileBytes_));
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int c = 0; c < kPanels; ++c)
                        tma_load_3d(smem + s * kTileBytes_ + c * kPanelBytes, &map_q, &bars->q_full, 64 * c,
                                    p.pair ? head0 + s : head0, item.start + row0 + (p.pair ? 0 : s * kRowsTile));
            }
            __syncwarp();
            for (int t = 0; ok && t < 2 * all_steps; ++t) {     // K of step t / 2, then V
                const int stage = t % kFwdStages;
                ok = __all_sync(0xffffffffu, mbar_wait(&bars->empty[stage], ((uint32_t)(t / kFwdStages) & 1u) ^ 1u, abort_flag, p.status)) != 0;
                if (ok && elect_one()) {
                    mbar_expect_tx(&bars->full[stage], (uint32_t)kTileBytes_);
                    const CUtensorMap* map = t & 1 ? &map_v : &map_k;
#pragma unroll
                    for (int c = 0; c < kPanels; ++c)
                        tma_load_3d(ring + stage * kTileBytes_ + c * kPanelBytes, map, &bars->full[stage], 64 * c, kv_head,
                                    item.start + (t / 2) * kRowsTile);
                }
                __syncwarp();
            }
            if (lane == 0 && *(volatile int*)abort_flag) let_copies_land();
            __syncwarp();
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------ MMA issuer
        if (all_steps > 0) {
            const uint32_t idesc_s = common | ((uint32_t)(kRowsTile >> 3) << 17);
            const uint32_t idesc_o = common | (1u << 16) | ((uint32_t)(kDim >> 3) << 17);
            const uint64_t q_desc[2] = {panel_desc(smem_u32(smem), false), panel_desc(smem_u32(smem + kTileBytes_), false)};
            bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->q_full, 0, abort_flag, p.status)) != 0;
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bars->full[0], 0, abort_flag, p.status)) != 0;
            if (ok) {
                tc_fence_after();
                const uint64_t k_desc = panel_desc(smem_u32(ring), false);
                if (elect_one()) {
#pragma unroll
                    for (int s = 0; s < 2; ++s)
                        if (steps[s] > 0) {
                            mma_rows<kDim>(tmem + (uint32_t)(s * 128), q_desc[s], k_desc, idesc_s);
                            tc_commit(&bars->s_full[s]);
                        }
                    tc_commit(&bars->empty[0]);
                }
                __syncwarp();
            }
            for (int j = 0; ok && j < all_steps; ++j) {
                const int v_no = 2 * j + 1, k_no = 2 * j + 2, v_stage = v_no % kFwdStages, k_stage = k_no % kFwdStages;
                const bool more = j + 1 < all_steps;
                ok = __all_sync(0xffffffffu, mbar_wait(&bars->full[v_stage], (uint32_t)(v_no / kFwdStages) & 1u, abort_flag, p.status)) != 0;
                if (ok && more)
                    ok = __all_sync(0xffffffffu, mbar_wait(&bars->full[k_stage], (uint32_t)(k_no / kFwdStages) & 1u, abort_flag, p.status)) != 0;
                if (!ok) break;
                const int valid = item.length - j * kRowsTile;
                if (valid < kRowsTile) zero_rows<kDim>(ring + v_stage * kTileBytes_, valid, lane);
                const uint64_t v_desc = panel_desc(smem_u32(ring + v_stage * kTileBytes_), true);
                const uint64_t k_desc = panel_desc(smem_u32(ring + k_stage * kTileBytes_), false);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (!ok || j >= steps[s]) continue;
                    ok = __all_sync(0xffffffffu, mbar_wait(&bars->p_full[s], (uint32_t)j & 1u, abort_flag, p.status)) != 0;
                    if (!ok) continue;
                    tc_fence_after();
                    if (elect_one()) {
                        mma_keys(tmem + (uint32_t)(256 + s * kDim), tmem + (uint32_t)(s * 128), v_desc, idesc_o, j > 0);
                        if (j + 1 < steps[s]) {
                            mma_rows<kDim>(tmem + (uint32_t)(s * 128), q_desc[s], k_desc, idesc_s);
                            tc_commit(&bars->s_full[s]);
                        } else {
                            tc_commit(&bars->o_full[s]);
                        }
                    }
                    __syncwarp();
                }
                if (ok && elect_one()) {
                    tc_commit(&bars->empty[v_stage]);
                    if (more) tc_commit(&bars->empty[k_stage]);
                }
                __syncwarp();
            }
            // all MMAs issued by the elected lane must have retired before TMEM is freed
            if (elect_one()) {
                tc_commit(&bars->drain);
                mbar_wait(&bars->drain, 0, abort_flag, p.status);
            }
            __syncwarp();
        }
    } else if (warp < 8) {
        // ------------------------------------------------------------ softmax of tile s, one row per thread
        const int s = warp >> 2, r = (warp & 3) * 32 + lane;
        const int n = steps[s];
        const int row = row0 + (p.pair ? 0 : s * kRowsTile) + r;        // in the sequence
        const int last = p.causal ? min(row, item.length - 1) : item.length - 1;      // the last key the row sees
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_tmem = tmem + lanes + (uint32_t)(s * 128), o_tmem = tmem + lanes + (uint32_t)(256 + s * kDim);
        const float c = p.scale_log2;
        float m = -INFINITY, l = 0.0f;                                  // m in units of c S
        bool ok = true;
        for (int j = 0; ok && j < n; ++j) {
            ok = mbar_wait(&bars->s_full[s], (uint32_t)j & 1u, abort_flag, p.status);
            ok = __all_sync(0xffffffffu, ok) != 0;
            if (!ok) break;
            tc_fence_after();
            uint32_t x[4][32];
#pragma unroll
            for (int i = 0; i < 4; ++i) tc_ld_32x32b_x32(s_tmem + (uint32_t)(32 * i), x[i]);
            tc_wait_ld();
            if (p.negative) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[i][e] ^= 0x80000000u;
            }
            const int see = last - j * kRowsTile;                       // columns 0 .. see of the tile are seen
            if (__any_sync(0xffffffffu, see < kRowsTile - 1)) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * i + e > see) x[i][e] = 0xff800000u;
            }
            float top[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                top[i] = __uint_as_float(x[i][0]);
#pragma unroll
                for (int e = 1; e < 31; e += 2) top[i] = fmax3(top[i], __uint_as_float(x[i][e]), __uint_as_float(x[i][e + 1]));
                top[i] = fmaxf(top[i], __uint_as_float(x[i][31]));
            }
            const float mt = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
            if (__any_sync(0xffffffffu, mt > m + 8.0f)) {
                const float higher = fmaxf(m, mt);
                const float fall = higher == -INFINITY ? 1.0f : attn_exp2(m - higher);
                m = higher;
                l *= fall;
                if (j > 0) {
                    // (rare; 8 columns at a time, beside the 128 scores that are in registers)
#pragma unroll 1
                    for (int i = 0; i < kDim; i += 8) {
                        uint32_t acc[8];
                        tc_ld_32x32b_x8(o_tmem + (uint32_t)i, acc);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[e] = __float_as_uint(__uint_as_float(acc[e]) * fall);
                        tc_st_32x32b_x8(o_tmem + (uint32_t)i, acc);
                    }
                }
            }
            const float ref = m == -INFINITY ? 0.0f : -m;
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float a = attn_exp2(fmaf(__uint_as_float(x[i][e]), c, ref));
                    const float b = attn_exp2(fmaf(__uint_as_float(x[i][e + 1]), c, ref));
                    sum[0] += a;
                    sum[1] += b;
                    x[i / 2][(i & 1) * 16 + e / 2] = pack2<kBf16>(a, b);
                }
                if (i & 1) tc_st_32x32b_x32(s_tmem + (uint32_t)(32 * (i / 2)), x[i / 2]);
            }
            l += sum[0] + sum[1];
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&bars->p_full[s]);
        }
        if (n > 0) {
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_full[s], 0, abort_flag, p.status)) != 0;
            tc_fence_after();
            const int head = p.pair ? head0 + s : head0;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint8_t* to = static_cast<uint8_t*>(p.o) + (((size_t)(item.start + row) * p.q_heads + head) * kDim) * 2;
#pragma unroll
            for (int i = 0; i < kDim / 32; ++i) {
                uint32_t acc[32];
                tc_ld_32x32b_x32(o_tmem + (uint32_t)(32 * i), acc);
                tc_wait_ld();
                if (ok && row < item.length) store_row32<kBf16>(to + 64 * i, acc, inv);
            }
            if (ok && row < item.length && p.lse) p.lse[(size_t)head * p.rows + item.start + row] = m + __log2f(l);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <bool kBf16, int kDim>
int launch_forward(const PackedParams& p, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
    auto kernel = packed_forward_kernel<kBf16, kDim>;
    constexpr int smem = fwd_smem<kDim>();
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return BSA_ERR_LAUNCH;
    // an upper bound of the tiles: every sequence and the rows behind the last one may end inside a tile
    const int per_tile = p.pair ? kRowsTile : 2 * kRowsTile;
    const unsigned grid = (unsigned)((p.rows / per_tile + p.batch + 1) * (p.pair ? p.q_heads / 2 : p.q_heads));
    kernel<<<grid, kFwdThreads, smem, stream>>>(p, mq, mk, mv);
    return launch_status();
}

}  // namespace
}  // namespace bsa

extern "C" int bsa_packed_forward(int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                  int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                  int64_t v_head_stride, void* o, float* lse, const int32_t* offsets, int64_t rows,
                                  int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, float scale, int causal,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    using namespace bsa;
    int checked = check_packed(dtype, rows, batch, q_heads, kv_heads, head_dim);
    if (checked != BSA_OK) return checked;
    if (!workspace || workspace_bytes < BSA_WORKSPACE_BYTES) return BSA_ERR_WORKSPACE;
    if (rows == 0) return BSA_OK;
    if (!q || !k || !v || !o || !offsets) return BSA_ERR_NULL_POINTER;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || (reinterpret_cast<uintptr_t>(o) & 31)) return BSA_ERR_ALIGNMENT;
    if ((checked = check_strides(q_token_stride, q_head_stride)) != BSA_OK || (checked = check_strides(k_token_stride, k_head_stride)) != BSA_OK ||
        (checked = check_strides(v_token_stride, v_head_stride)) != BSA_OK) return checked;
    PackedParams p{};
    p.o = o; p.lse = lse; p.offsets = offsets;
    p.batch = (int)batch; p.rows = (int)rows; p.q_heads = (int)q_heads; p.kv_heads = (int)kv_heads;
    p.group = (int)(q_heads / kv_heads); p.causal = causal != 0;
    p.pair = p.group % 2 == 0;
    p.negative = scale < 0.0f;
    // a scale of 0 stays a factor that keeps masked scores at -infinity
    p.scale_log2 = fmaxf(fabsf(scale) * kPackedLog2e, 1e-37f);
    p.status = static_cast<uint32_t*>(workspace);
    CUtensorMap mq, mk, mv;
    if (!bind_device()) return BSA_ERR_LAUNCH;
    if (!make_packed_map(&mq, dtype, q, rows, q_heads, head_dim, q_token_stride, q_head_stride) ||
        !make_packed_map(&mk, dtype, k, rows, kv_heads, head_dim, k_token_stride, k_head_stride) ||
        !make_packed_map(&mv, dtype, v, rows, kv_heads, head_dim, v_token_stride, v_head_stride)) return BSA_ERR_DRIVER;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == BSA_DTYPE_BF16)
        return head_dim == 64 ? launch_forward<true, 64>(p, mq, mk, mv, s) : launch_forward<true, 128>(p, mq, mk, mv, s);
    return head_dim == 64 ? launch_forward<false, 64>(p, mq, mk, mv, s) : launch_forward<false, 128>(p, mq, mk, mv, s);
}
