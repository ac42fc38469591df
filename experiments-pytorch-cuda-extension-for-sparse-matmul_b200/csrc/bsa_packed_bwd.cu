// Gradients of the packed attention (sm_100a only).  With P = exp(scale Q K^T - lse) recomputed on chip:
//   dV = P^T dO        dP = dO V^T        dS = P o (dP - delta),  delta = rowsum(dO o O)
//   dQ = scale dS K    dK = scale dS^T Q
// dK and dV of a key head are the sums over the query heads of its group.
//
// Three launches, none with atomics, so the results do not depend on timing:
//   packed_stats_kernel   (lse, delta) per row and head
//   packed_keys_kernel    dK, dV: a CTA holds 128 keys and walks the query tiles that see them, head after head of the
//                         group; both sums stay in TMEM to the end
//   packed_queries_kernel dQ: a CTA holds 128 queries of a head and walks the key tiles that they see
// S and dP are computed in both (7 products of 128 x 128 x D per pair of tiles where 5 would do with dQ summed in memory).
//
// Both walk 128 x 128 tiles: S (or S^T) and dP from shared memory into TMEM, two warpgroups turn them into P and dS
// (each thread one row, 64 of the 128 columns), 16 bits, written over the scores as the A operand of the products that
// accumulate.  The issue order keeps the tensor cores busy while the warps work: by keys  dV(i) S(i+1) | dK(i) dP(i+1),
// the first pair while the warps make dS(i), the second while they make P(i + 1); by queries S(j+1) | dP(j+1) dQ(j).
// At the tensor pipe's peak a pair of tiles costs 4 (3) x 4 D cycles, its 16384 exponentials 1024 on the MUFU units.
//
// P and dS are rounded to the inputs' type before the accumulating products, everything else is fp32.
#include "bsa_packed_common.cuh"

namespace bsa {
namespace {

constexpr int kBwdThreads = 384;
constexpr int kStatBytes = kRowsTile * 8;

struct PackedBwdParams {
    const void* o;
    const void* dout;
    int64_t dout_token, dout_head;              // strides in elements
    const float* lse;
    float2* stats;                              // [q_heads, rows] of (lse, delta)
    void* dq;
    void* dk;
    void* dv;
    const int32_t* offsets;
    int batch, rows, q_heads, kv_heads, group, causal;
    float scale, scale_log2;
    uint32_t* status;
};

// One row and head per D / 8 lanes.
template <typename T, int kDim>
__global__ void __launch_bounds__(256) packed_stats_kernel(const PackedBwdParams p) {
    constexpr int kLanes = kDim / 8;
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kLanes;      // row * q_heads + head
    const int lane = threadIdx.x % kLanes;
    float sum = 0.0f;
    const bool in = at < (int64_t)p.rows * p.q_heads;
    const int64_t row = at / p.q_heads;
    const int head = (int)(at - row * p.q_heads);
    if (in) {
        const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.o) + at * kDim + lane * 8);
        const uint4 b = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.dout) + row * p.dout_token + head * p.dout_head + lane * 8);
        const T* x = reinterpret_cast<const T*>(&a);
        const T* y = reinterpret_cast<const T*>(&b);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(Scalar<T>::to_float(x[e]), Scalar<T>::to_float(y[e]), sum);
    }
#pragma unroll
    for (int s = kLanes / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if (in && lane == 0) {
        const int64_t to = (int64_t)head * p.rows + row;
        const float lse = p.lse[to];
        p.stats[to] = make_float2(lse == -INFINITY ? INFINITY : lse, sum);      // a row without keys: P = 2^-inf = 0
    }
}

struct __align__(8) BwdBarriers {
    uint64_t x_full, y_full[2], y_empty[2], st_full[2], st_empty[2];
    uint64_t s_full[2], dp_full, p_full, ds_full, done, drain;
    PackedItem item;
    uint32_t tmem_base;
    int abort_flag;
};
template <int kDim>
constexpr int bwd_smem() { return 6 * (kDim / 64) * kPanelBytes + 2 * kStatBytes + (int)sizeof(BwdBarriers); }

// A in TMEM as two halves of 64 elements, 64 columns apart (each warpgroup writes over the scores that it has read).
__device__ __forceinline__ void mma_halves(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, bool accumulate) {
#pragma unroll
    for (int kk = 0; kk < kRowsTile / 16; ++kk)
        tc_mma_f16_ts(tmem_d, tmem_a + (uint32_t)((kk / 4) * 64 + (kk % 4) * 8), b + (uint64_t)(kk * (2048 >> 4)), idesc,
                      accumulate || kk > 0 ? 1u : 0u);
}

__device__ __forceinline__ void bwd_begin(BwdBarriers* bars, const PackedBwdParams& p, int rank, int warp, int lane) {
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 8) {
        const PackedItem found = packed_locate(p.offsets, p.batch, p.rows, kRowsTile, rank, lane, p.status);
        if (lane == 0) {
            bars->item = found;
            bars->abort_flag = 0;
            mbar_init(&bars->x_full, 1);
            for (int i = 0; i < 2; ++i) {
                mbar_init(&bars->y_full[i], 1); mbar_init(&bars->y_empty[i], 1);
                mbar_init(&bars->st_full[i], 1); mbar_init(&bars->st_empty[i], 8);
                mbar_init(&bars->s_full[i], 1);
            }
            mbar_init(&bars->dp_full, 1);
            mbar_init(&bars->p_full, 8);
            mbar_init(&bars->ds_full, 8);
            mbar_init(&bars->done, 1);
            mbar_init(&bars->drain, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            fence_async_shared();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
}
__device__ __forceinline__ void bwd_end(uint32_t tmem, int warp) {
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}
template <int kDim>
__device__ __forceinline__ void load_tile(uint8_t* to, const CUtensorMap* map, uint64_t* bar, int head, int row) {
#pragma unroll
    for (int c = 0; c < kDim / 64; ++c) tma_load_3d(to + c * kPanelBytes, map, bar, 64 * c, head, row);
}

// ------------------------------------------------------------------------------------------------ dK, dV
template <bool kBf16, int kDim>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_keys_kernel(const PackedBwdParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do) {
    constexpr int kTile_ = (kDim / 64) * kPanelBytes;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* k_smem = smem;
    uint8_t* v_smem = smem + kTile_;
    uint8_t* y_smem = smem + 2 * kTile_;                        // stage i: Q, dO
    float4* st_smem = reinterpret_cast<float4*>(smem + 6 * kTile_);
    BwdBarriers* bars = reinterpret_cast<BwdBarriers*>(smem + 6 * kTile_ + 2 * kStatBytes);
    int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x / p.kv_heads, kv_head = (int)blockIdx.x - rank * p.kv_heads;
    bwd_begin(bars, p, rank, warp, lane);
    const uint32_t tmem = *(volatile uint32_t*)&bars->tmem_base;
    const PackedItem item = bars->item;
    const bool work = item.length > 0 && item.b < p.batch;
    const int tiles = (item.length + kRowsTile - 1) / kRowsTile;
    const int key_tile = tiles - 1 - item.tile;                 // (the first keys are seen by the most queries)
    const int first_q = p.causal ? key_tile : 0;                // the query tiles that see these keys: first_q .. tiles - 1
    const int per_head = tiles - first_q, n = work ? per_head * p.group : 0;
    const uint32_t s_tmem = tmem, dp_tmem = tmem + 128u, dv_tmem = tmem + 256u, dk_tmem = tmem + 256u + kDim;

    if (item.length > 0 && item.b == p.batch) {                 // rows behind the last sequence
        const int from = item.start + item.tile * kRowsTile, to = min(from + kRowsTile, p.rows);
        zero_tail(p.dk, from, to, kv_head, p.kv_heads, kDim, threadIdx.x, blockDim.x);
        zero_tail(p.dv, from, to, kv_head, p.kv_heads, kDim, threadIdx.x, blockDim.x);
    }
    if (warp == 8) {
        // ------------------------------------------------------------ producer
        if (n > 0) {
            bool ok = true;
            if (elect_one()) {
                mbar_expect_tx(&bars->x_full, (uint32_t)(2 * kTile_));
                load_tile<kDim>(k_smem, &map_k, &bars->x_full, kv_head, item.start + key_tile * kRowsTile);
                load_tile<kDim>(v_smem, &map_v, &bars->x_full, kv_head, item.start + key_tile * kRowsTile);
            }
            __syncwarp();
            int head = kv_head * p.group, qt = first_q;
            for (int i = 0; ok && i < n; ++i) {
                const int st = i & 1;
                ok = wait_all(&bars->y_empty[st], ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag, p.status);
                if (ok && elect_one()) {
                    mbar_expect_tx(&bars->y_full[st], (uint32_t)(2 * kTile_));
                    load_tile<kDim>(y_smem + 2 * st * kTile_, &map_q, &bars->y_full[st], head, item.start + qt * kRowsTile);
                    load_tile<kDim>(y_smem + (2 * st + 1) * kTile_, &map_do, &bars->y_full[st], head, item.start + qt * kRowsTile);
                }
                __syncwarp();
                if (++qt == tiles) { qt = first_q; ++head; }
            }
            if (lane == 0 && *(volatile int*)abort_flag) let_copies_land();
            __syncwarp();
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------ MMA issuer
        if (n > 0) {
            const uint32_t fmt = kBf16 ? 1u : 0u;
            const uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRowsTile >> 4) << 24);
            const uint32_t idesc_t = common | ((uint32_t)(kRowsTile >> 3) << 17);
            const uint32_t idesc_acc = common | (1u << 16) | ((uint32_t)(kDim >> 3) << 17);
            const uint64_t k_desc = panel_desc(smem_u32(k_smem), false), v_desc = panel_desc(smem_u32(v_smem), false);
            int qt = first_q;                                   // of the stage that is waited for next
            bool ok = wait_all(&bars->x_full, 0, abort_flag, p.status);
            // a stage's rows behind the sequence's end must not reach the sums over rows
            auto stage_ready = [&](int i) {
                const int st = i & 1;
                if (!wait_all(&bars->y_full[st], (uint32_t)(i >> 1) & 1u, abort_flag, p.status)) return false;
                const int valid = item.length - qt * kRowsTile;
                if (valid < kRowsTile) {
                    zero_rows<kDim>(y_smem + 2 * st * kTile_, valid, lane);
                    zero_rows<kDim>(y_smem + (2 * st + 1) * kTile_, valid, lane);
                }
                if (++qt == tiles) qt = first_q;
                return true;
            };
            if (ok) ok = stage_ready(0);
            if (ok) {
                tc_fence_after();
                if (elect_one()) {
                    mma_rows<kDim>(s_tmem, k_desc, panel_desc(smem_u32(y_smem), false), idesc_t);
                    tc_commit(&bars->s_full[0]);
                    mma_rows<kDim>(dp_tmem, v_desc, panel_desc(smem_u32(y_smem + kTile_), false), idesc_t);
                    tc_commit(&bars->dp_full);
                }
                __syncwarp();
            }
            for (int i = 0; ok && i < n; ++i) {
                const int st = i & 1, next = st ^ 1;
                const bool more = i + 1 < n;
                const uint8_t* y = y_smem + 2 * st * kTile_;
                const uint8_t* y_next = y_smem + 2 * next * kTile_;
                ok = wait_all(&bars->p_full, (uint32_t)i & 1u, abort_flag, p.status);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) mma_halves(dv_tmem, s_tmem, panel_desc(smem_u32(y + kTile_), true), idesc_acc, i > 0);
                __syncwarp();
                if (more) {
                    ok = stage_ready(i + 1);
                    if (!ok) break;
                    if (elect_one()) {
                        mma_rows<kDim>(s_tmem, k_desc, panel_desc(smem_u32(y_next), false), idesc_t);
                        tc_commit(&bars->s_full[0]);
                    }
                    __syncwarp();
                }
                ok = wait_all(&bars->ds_full, (uint32_t)i & 1u, abort_flag, p.status);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    mma_halves(dk_tmem, dp_tmem, panel_desc(smem_u32(y), true), idesc_acc, i > 0);
                    tc_commit(&bars->y_empty[st]);
                    if (more) {
                        mma_rows<kDim>(dp_tmem, v_desc, panel_desc(smem_u32(y_next + kTile_), false), idesc_t);
                        tc_commit(&bars->dp_full);
                    } else {
                        tc_commit(&bars->done);
                    }
                }
                __syncwarp();
            }
            if (elect_one()) {
                tc_commit(&bars->drain);
                mbar_wait(&bars->drain, 0, abort_flag, p.status);
            }
            __syncwarp();
        }
    } else if (warp == 10) {
        // ------------------------------------------------------------ statistics of the query tiles
        bool ok = true;
        int head = kv_head * p.group, qt = first_q;
        for (int i = 0; ok && i < n; ++i) {
            const int st = i & 1, row = item.start + qt * kRowsTile + 4 * lane;
            float2 s[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s[e] = row + e < p.rows ? p.stats[(size_t)head * p.rows + row + e] : make_float2(0.0f, 0.0f);
            ok = wait_all(&bars->st_empty[st], ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag, p.status);
            if (!ok) break;
            st_smem[st * (kRowsTile / 2) + 2 * lane] = make_float4(s[0].x, s[0].y, s[1].x, s[1].y);
            st_smem[st * (kRowsTile / 2) + 2 * lane + 1] = make_float4(s[2].x, s[2].y, s[3].x, s[3].y);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->st_full[st]);
            if (++qt == tiles) { qt = first_q; ++head; }
        }
    } else if (warp < 8 && n > 0) {
        // ------------------------------------------------------------ P and dS: one key per thread, 64 queries
        const int half = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(64 * half);
        const float c = p.scale_log2;
        bool ok = true;
        int qt = first_q;
        for (int i = 0; i < n; ++i) {
            const int st = i & 1;
            const float4* stat = st_smem + st * (kRowsTile / 2) + 32 * half;
            // columns (queries of this half) from `from` up to `to` see the key
            const int from = (p.causal && qt == key_tile ? r : 0) - 64 * half, to = item.length - qt * kRowsTile - 64 * half;
            const bool masked = __any_sync(0xffffffffu, from > 0 || to < 64) != 0;
            ok = ok && wait_all(&bars->st_full[st], (uint32_t)(i >> 1) & 1u, abort_flag, p.status);
            ok = ok && wait_all(&bars->s_full[0], (uint32_t)i & 1u, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            uint32_t x[2][32], w[32];
            tc_ld_32x32b_x32(s_tmem + lanes, x[0]);
            tc_ld_32x32b_x32(s_tmem + lanes + 32u, x[1]);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
                const float4 s2 = stat[e / 2];
                float a = attn_exp2(fmaf(__uint_as_float(x[e / 32][e % 32]), c, -s2.x));
                float b = attn_exp2(fmaf(__uint_as_float(x[e / 32][e % 32 + 1]), c, -s2.z));
                if (masked) {
                    if (e < from || e >= to) a = 0.0f;
                    if (e + 1 < from || e + 1 >= to) b = 0.0f;
                }
                x[e / 32][e % 32] = __float_as_uint(a);
                x[e / 32][e % 32 + 1] = __float_as_uint(b);
                w[e / 2] = pack2<kBf16>(a, b);
            }
            tc_st_32x32b_x32(s_tmem + lanes, w);
            tc_wait_st();
            arrive_warp(&bars->p_full, lane);
            ok = wait_all(&bars->dp_full, (uint32_t)i & 1u, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t d[32];
                tc_ld_32x32b_x32(dp_tmem + lanes + (uint32_t)(32 * h), d);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float4 s2 = stat[16 * h + e / 2];
                    float a = __uint_as_float(x[h][e]) * (__uint_as_float(d[e]) - s2.y);
                    float b = __uint_as_float(x[h][e + 1]) * (__uint_as_float(d[e + 1]) - s2.w);
                    if (masked) {                               // (0 times what a row behind the end holds)
                        if (32 * h + e < from || 32 * h + e >= to) a = 0.0f;
                        if (32 * h + e + 1 < from || 32 * h + e + 1 >= to) b = 0.0f;
                    }
                    w[16 * h + e / 2] = pack2<kBf16>(a, b);
                }
            }
            tc_st_32x32b_x32(dp_tmem + lanes, w);
            tc_wait_st();
            arrive_warp(&bars->ds_full, lane);
            if (lane == 0) mbar_arrive(&bars->st_empty[st]);
            if (++qt == tiles) qt = first_q;
        }
        ok = ok && wait_all(&bars->done, 0, abort_flag, p.status);
        tc_fence_after();
        const int key = key_tile * kRowsTile + r;
        const size_t at = ((size_t)(item.start + key) * p.kv_heads + kv_head) * kDim;
#pragma unroll
        for (int i = 0; i < kDim / 64; ++i) {                   // this half's columns of both
            const int col = half * (kDim / 2) + 32 * i;
            uint32_t acc[32];
            tc_ld_32x32b_x32(dv_tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)col, acc);
            tc_wait_ld();
            if (ok && key < item.length) store_row32<kBf16>(static_cast<uint8_t*>(p.dv) + (at + col) * 2, acc, 1.0f);
            tc_ld_32x32b_x32(dk_tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)col, acc);
            tc_wait_ld();
            if (ok && key < item.length) store_row32<kBf16>(static_cast<uint8_t*>(p.dk) + (at + col) * 2, acc, p.scale);
        }
    }
    bwd_end(tmem, warp);
}

// ------------------------------------------------------------------------------------------------ dQ
template <bool kBf16, int kDim>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_queries_kernel(const PackedBwdParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do) {
    constexpr int kTile_ = (kDim / 64) * kPanelBytes;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_smem = smem;
    uint8_t* do_smem = smem + kTile_;
    uint8_t* y_smem = smem + 2 * kTile_;                        // stage j: K, V
    BwdBarriers* bars = reinterpret_cast<BwdBarriers*>(smem + 6 * kTile_ + 2 * kStatBytes);
    int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x / p.q_heads, head = (int)blockIdx.x - rank * p.q_heads, kv_head = head / p.group;
    bwd_begin(bars, p, rank, warp, lane);
    const uint32_t tmem = *(volatile uint32_t*)&bars->tmem_base;
    const PackedItem item = bars->item;
    const bool work = item.length > 0 && item.b < p.batch;
    const int tiles = (item.length + kRowsTile - 1) / kRowsTile;
    const int tile = item.tile;
    const int n = work ? (p.causal ? tile + 1 : tiles) : 0;
    const uint32_t dp_tmem = tmem + 256u, dq_tmem = tmem + 384u;

    if (item.length > 0 && item.b == p.batch) {
        const int from = item.start + item.tile * kRowsTile, to = min(from + kRowsTile, p.rows);
        zero_tail(p.dq, from, to, head, p.q_heads, kDim, threadIdx.x, blockDim.x);
    }
    if (warp == 8) {
        // ------------------------------------------------------------ producer
        if (n > 0) {
            bool ok = true;
            if (elect_one()) {
                mbar_expect_tx(&bars->x_full, (uint32_t)(2 * kTile_));
                load_tile<kDim>(q_smem, &map_q, &bars->x_full, head, item.start + tile * kRowsTile);
                load_tile<kDim>(do_smem, &map_do, &bars->x_full, head, item.start + tile * kRowsTile);
            }
            __syncwarp();
            for (int j = 0; ok && j < n; ++j) {
                const int st = j & 1;
                ok = wait_all(&bars->y_empty[st], ((uint32_t)(j >> 1) & 1u) ^ 1u, abort_flag, p.status);
                if (ok && elect_one()) {
                    mbar_expect_tx(&bars->y_full[st], (uint32_t)(2 * kTile_));
                    load_tile<kDim>(y_smem + 2 * st * kTile_, &map_k, &bars->y_full[st], kv_head, item.start + j * kRowsTile);
                    load_tile<kDim>(y_smem + (2 * st + 1) * kTile_, &map_v, &bars->y_full[st], kv_head, item.start + j * kRowsTile);
                }
                __syncwarp();
            }
            if (lane == 0 && *(volatile int*)abort_flag) let_copies_land();
            __syncwarp();
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------ MMA issuer
        if (n > 0) {
            const uint32_t fmt = kBf16 ? 1u : 0u;
            const uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRowsTile >> 4) << 24);
            const uint32_t idesc_t = common | ((uint32_t)(kRowsTile >> 3) << 17);
            const uint32_t idesc_acc = common | (1u << 16) | ((uint32_t)(kDim >> 3) << 17);
            const uint64_t q_desc = panel_desc(smem_u32(q_smem), false), do_desc = panel_desc(smem_u32(do_smem), false);
            bool ok = wait_all(&bars->x_full, 0, abort_flag, p.status);
            auto stage_ready = [&](int j) {
                const int st = j & 1, valid = item.length - j * kRowsTile;
                if (!wait_all(&bars->y_full[st], (uint32_t)(j >> 1) & 1u, abort_flag, p.status)) return false;
                if (valid < kRowsTile) zero_rows<kDim>(y_smem + 2 * st * kTile_, valid, lane);      // K: summed over keys
                return true;
            };
            if (ok) ok = stage_ready(0);
            if (ok) {
                tc_fence_after();
                if (elect_one()) {
                    mma_rows<kDim>(tmem, q_desc, panel_desc(smem_u32(y_smem), false), idesc_t);
                    tc_commit(&bars->s_full[0]);
                    mma_rows<kDim>(dp_tmem, do_desc, panel_desc(smem_u32(y_smem + kTile_), false), idesc_t);
                    tc_commit(&bars->dp_full);
                }
                __syncwarp();
            }
            for (int j = 0; ok && j < n; ++j) {
                const int st = j & 1, next = st ^ 1;
                const bool more = j + 1 < n;
                if (more) {
                    ok = stage_ready(j + 1);
                    if (!ok) break;
                    if (elect_one()) {
                        mma_rows<kDim>(tmem + (uint32_t)(128 * next), q_desc, panel_desc(smem_u32(y_smem + 2 * next * kTile_), false), idesc_t);
                        tc_commit(&bars->s_full[next]);
                    }
                    __syncwarp();
                }
                ok = wait_all(&bars->ds_full, (uint32_t)j & 1u, abort_flag, p.status);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    if (more) {
                        mma_rows<kDim>(dp_tmem, do_desc, panel_desc(smem_u32(y_smem + (2 * next + 1) * kTile_), false), idesc_t);
                        tc_commit(&bars->dp_full);
                    }
                    mma_halves(dq_tmem, tmem + (uint32_t)(128 * st), panel_desc(smem_u32(y_smem + 2 * st * kTile_), true), idesc_acc, j > 0);
                    tc_commit(&bars->y_empty[st]);
                    if (!more) tc_commit(&bars->done);
                }
                __syncwarp();
            }
            if (elect_one()) {
                tc_commit(&bars->drain);
                mbar_wait(&bars->drain, 0, abort_flag, p.status);
            }
            __syncwarp();
        }
    } else if (warp < 8 && n > 0) {
        // ------------------------------------------------------------ P and dS: one query per thread, 64 keys
        const int half = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lane_part = (uint32_t)((warp & 3) * 32) << 16, lanes = lane_part + (uint32_t)(64 * half);
        const float c = p.scale_log2;
        const int row = tile * kRowsTile + r;
        const int last = p.causal ? min(row, item.length - 1) : item.length - 1;
        const float2 stat = row < item.length ? p.stats[(size_t)head * p.rows + item.start + row] : make_float2(INFINITY, 0.0f);
        bool ok = true;
        for (int j = 0; j < n; ++j) {
            const int see = last - j * kRowsTile - 64 * half;               // columns 0 .. see of this half are seen
            const bool masked = __any_sync(0xffffffffu, see < 63) != 0;
            const uint32_t s_tmem = tmem + (uint32_t)(128 * (j & 1)) + lanes;
            ok = wait_all(&bars->s_full[j & 1], (uint32_t)(j >> 1) & 1u, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            uint32_t x[2][32], w[32];
            tc_ld_32x32b_x32(s_tmem, x[0]);
            tc_ld_32x32b_x32(s_tmem + 32u, x[1]);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 64; ++e) {
                const float a = attn_exp2(fmaf(__uint_as_float(x[e / 32][e % 32]), c, -stat.x));
                x[e / 32][e % 32] = __float_as_uint(a);
            }
            ok = wait_all(&bars->dp_full, (uint32_t)j & 1u, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t d[32];
                tc_ld_32x32b_x32(dp_tmem + lanes + (uint32_t)(32 * h), d);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float a = __uint_as_float(x[h][e]) * (__uint_as_float(d[e]) - stat.y);
                    float b = __uint_as_float(x[h][e + 1]) * (__uint_as_float(d[e + 1]) - stat.y);
                    if (masked) {
                        if (32 * h + e > see) a = 0.0f;
                        if (32 * h + e + 1 > see) b = 0.0f;
                    }
                    w[16 * h + e / 2] = pack2<kBf16>(a, b);
                }
            }
            tc_st_32x32b_x32(s_tmem, w);
            tc_wait_st();
            arrive_warp(&bars->ds_full, lane);
        }
        ok = ok && wait_all(&bars->done, 0, abort_flag, p.status);
        tc_fence_after();
        const size_t at = ((size_t)(item.start + row) * p.q_heads + head) * kDim;
#pragma unroll
        for (int i = 0; i < kDim / 64; ++i) {
            const int col = half * (kDim / 2) + 32 * i;
            uint32_t acc[32];
            tc_ld_32x32b_x32(dq_tmem + lane_part + (uint32_t)col, acc);
            tc_wait_ld();
            if (ok && row < item.length) store_row32<kBf16>(static_cast<uint8_t*>(p.dq) + (at + col) * 2, acc, p.scale);
        }
    }
    bwd_end(tmem, warp);
}

template <bool kBf16, int kDim>
int launch_backward(const PackedBwdParams& p, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                    const CUtensorMap& mdo, cudaStream_t stream) {
    using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
    auto keys = packed_keys_kernel<kBf16, kDim>;
    auto queries = packed_queries_kernel<kBf16, kDim>;
    constexpr int smem = bwd_smem<kDim>();
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(keys), smem) ||
        !ensure_dynamic_smem(reinterpret_cast<const void*>(queries), smem)) return BSA_ERR_LAUNCH;
    const int64_t rows_heads = (int64_t)p.rows * p.q_heads, per_cta = 256 / (kDim / 8);
    packed_stats_kernel<T, kDim><<<(unsigned)((rows_heads + per_cta - 1) / per_cta), 256, 0, stream>>>(p);
    const unsigned items = (unsigned)(p.rows / kRowsTile + p.batch + 1);
    keys<<<items * p.kv_heads, kBwdThreads, smem, stream>>>(p, mq, mk, mv, mdo);
    queries<<<items * p.q_heads, kBwdThreads, smem, stream>>>(p, mq, mk, mv, mdo);
    return launch_status();
}

}  // namespace
}  // namespace bsa

extern "C" int bsa_packed_backward(int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                   int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                   int64_t v_head_stride, const void* o, const void* dout, int64_t dout_token_stride,
                                   int64_t dout_head_stride, const float* lse, void* dq, void* dk, void* dv,
                                   const int32_t* offsets, int64_t rows, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                   int64_t head_dim, float scale, int causal, void* stats, size_t stats_bytes,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    using namespace bsa;
    int checked = check_packed(dtype, rows, batch, q_heads, kv_heads, head_dim);
    if (checked != BSA_OK) return checked;
    if (!workspace || workspace_bytes < BSA_WORKSPACE_BYTES) return BSA_ERR_WORKSPACE;
    if (rows == 0) return BSA_OK;
    if (!q || !k || !v || !o || !dout || !lse || !dq || !dk || !dv || !offsets || !stats) return BSA_ERR_NULL_POINTER;
    for (const void* ptr : {q, k, v, o, dout, static_cast<const void*>(stats)})
        if (!aligned16(ptr)) return BSA_ERR_ALIGNMENT;
    for (const void* ptr : {dq, dk, dv})
        if (reinterpret_cast<uintptr_t>(ptr) & 31) return BSA_ERR_ALIGNMENT;
    if ((checked = check_strides(q_token_stride, q_head_stride)) != BSA_OK || (checked = check_strides(k_token_stride, k_head_stride)) != BSA_OK ||
        (checked = check_strides(v_token_stride, v_head_stride)) != BSA_OK ||
        (checked = check_strides(dout_token_stride, dout_head_stride)) != BSA_OK) return checked;
    if (stats_bytes < (size_t)rows * q_heads * sizeof(float2)) return BSA_ERR_WORKSPACE;
    PackedBwdParams p{};
    p.o = o; p.dout = dout; p.dout_token = dout_token_stride; p.dout_head = dout_head_stride;
    p.lse = lse; p.stats = static_cast<float2*>(stats);
    p.dq = dq; p.dk = dk; p.dv = dv; p.offsets = offsets;
    p.batch = (int)batch; p.rows = (int)rows; p.q_heads = (int)q_heads; p.kv_heads = (int)kv_heads;
    p.group = (int)(q_heads / kv_heads); p.causal = causal != 0;
    p.scale = scale; p.scale_log2 = scale * kPackedLog2e;
    p.status = static_cast<uint32_t*>(workspace);
    CUtensorMap mq, mk, mv, mdo;
    if (!bind_device()) return BSA_ERR_LAUNCH;
    if (!make_packed_map(&mq, dtype, q, rows, q_heads, head_dim, q_token_stride, q_head_stride) ||
        !make_packed_map(&mk, dtype, k, rows, kv_heads, head_dim, k_token_stride, k_head_stride) ||
        !make_packed_map(&mv, dtype, v, rows, kv_heads, head_dim, v_token_stride, v_head_stride) ||
        !make_packed_map(&mdo, dtype, dout, rows, q_heads, head_dim, dout_token_stride, dout_head_stride)) return BSA_ERR_DRIVER;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == BSA_DTYPE_BF16)
        return head_dim == 64 ? launch_backward<true, 64>(p, mq, mk, mv, mdo, s) : launch_backward<true, 128>(p, mq, mk, mv, mdo, s);
    return head_dim == 64 ? launch_backward<false, 64>(p, mq, mk, mv, mdo, s) : launch_backward<false, 128>(p, mq, mk, mv, mdo, s);
}
