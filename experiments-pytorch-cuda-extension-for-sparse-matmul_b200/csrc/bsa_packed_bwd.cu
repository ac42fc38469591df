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
// Both walk 128 x 128 tiles: S (or S^T) and dP on the tensor cores into TMEM; warps turn them into P and dS, 16 bits, the
// A operands of the products that accumulate.  Two warpgroups take alternate tiles, one row of 128 per thread, so that
// one is in its exponentials (1024 cycles of the MUFU units per tile) while the other multiplies and stores.  (With both
// on the same tile, half a row per thread, a tile took 3500 cycles by keys and 3400 by queries.)  At its peak the tensor
// pipe takes 16 D (keys) or 12 D (queries) cycles per tile, which is what binds at D = 128.
//   by keys     S(i+1) as soon as S(i) is in registers | dV(i), P from shared memory | dK(i), dS over dP in TMEM | dP(i+1)
//   by queries  S(j+1) into the other S buffer | dP(j+1) as soon as dP(j) is in registers | dQ(j), dS over S in TMEM
// By keys, where a key head serves an even number of query heads, a cluster of two CTAs shares a key tile, half of the
// heads each, and the second hands its sums to the first through distributed shared memory: a key tile's work is the
// product of the group and the query tiles behind it, too much for one SM beside the others.
//
// P and dS are rounded to the inputs' type before the accumulating products, everything else is fp32.
//
// 8,192 rows of 7 sequences, 16 / 4 heads x 128, bf16: statistics 24 us, keys 234, queries 177 (each alone,
// cold).  A tile takes 2400 cycles by queries and 3500 by keys, bound by shared memory: a product of two operands there reads 128 bytes per cycle at the
// tensor pipe's peak, all that an SM has, and the copies of the next tiles want 64 KB more.
#include "bsa_packed_common.cuh"

namespace bsa {
namespace {

constexpr int kBwdThreads = 384;

struct PackedBwdParams {
    const void* o;
    const void* o_low;                          // what rounding took from o
    const void* dout;
    int64_t dout_token, dout_head;              // strides in elements
    const float* lse;
    float2* stats;                              // [q_heads, rows] of (lse, delta)
    void* dq;
    void* dk;
    void* dv;
    const int32_t* offsets;
    int batch, rows, q_heads, kv_heads, group, causal;
    int split;                                  // CTAs per key tile and key head: 2 where the group is even, else 1
    float scale, scale_log2;
    uint32_t* status;
};

// One row and head per D / 8 lanes.  delta is made from o as it was before its rounding: with the rounded o alone the gradients' error against 64 bits is 1.5 times that of fp32 arithmetic rounded at the end.
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
        const uint4 low = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.o_low) + at * kDim + lane * 8);
        const T* x = reinterpret_cast<const T*>(&a);
        const T* z = reinterpret_cast<const T*>(&low);
        const T* y = reinterpret_cast<const T*>(&b);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(Scalar<T>::to_float(x[e]) + Scalar<T>::to_float(z[e]), Scalar<T>::to_float(y[e]), sum);
    }
#pragma unroll
    for (int s = kLanes / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if (in && lane == 0) {
        const int64_t to = (int64_t)head * p.rows + row;
        const float lse = p.lse[to];
        p.stats[to] = make_float2(lse == -INFINITY ? INFINITY : lse, sum);      // a row without keys: P = 2^-inf = 0
    }
}

struct __align__(16) BwdBarriers {
    uint64_t x_full, a_full[3], a_empty[3], b_full[2], b_empty[2];      // rings of the two moving tiles
    uint64_t st_full[2], st_empty[2];
    uint64_t s_full[2], s_read[2], dp_full[2], dp_read[2], p_full[2], p_empty[2], ds_full[2], done, drain;
    PackedItem item;
    uint32_t tmem_base;
    int abort_flag;
};
constexpr int kStatFloats = 2 * kRowsTile;      // -lse, then -delta, of a tile's queries
template <int kDim>
constexpr int bwd_smem() { return 7 * (kDim / 64) * kPanelBytes + (int)sizeof(BwdBarriers); }
template <int kDim>
constexpr int bwd_smem_keys() { return (6 * (kDim / 64) + (kDim == 128 ? 2 : 0)) * kPanelBytes + 2 * kStatFloats * 4 + (int)sizeof(BwdBarriers); }

// All threads of a cluster; every role ends in bounded time and comes here.
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(uint32_t addr, uint32_t cta) {
    uint32_t d;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(addr), "r"(cta));
    return d;
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
            for (int i = 0; i < 3; ++i) { mbar_init(&bars->a_full[i], 1); mbar_init(&bars->a_empty[i], 1); }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&bars->b_full[i], 1); mbar_init(&bars->b_empty[i], 1);
                mbar_init(&bars->st_full[i], 1); mbar_init(&bars->st_empty[i], 4);
                mbar_init(&bars->s_full[i], 1); mbar_init(&bars->s_read[i], 4);
                mbar_init(&bars->dp_full[i], 1); mbar_init(&bars->dp_read[i], 4);
                mbar_init(&bars->p_full[i], 4); mbar_init(&bars->p_empty[i], 1);
                mbar_init(&bars->ds_full[i], 4);
            }
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
    if (elect_one()) {
        mbar_expect_tx(bar, (uint32_t)((kDim / 64) * kPanelBytes));
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) tma_load_3d(to + c * kPanelBytes, map, bar, 64 * c, head, row);
    }
    __syncwarp();
}
// Completion n of a pair of barriers that take turns: barrier n & 1, its phase n / 2.
__device__ __forceinline__ bool wait_turn(uint64_t (&bars)[2], int n, int* abort_flag, uint32_t* status) {
    return wait_all(&bars[n & 1], (uint32_t)(n >> 1) & 1u, abort_flag, status);
}

// ------------------------------------------------------------------------------------------------ dK, dV
template <bool kBf16, int kDim>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_keys_kernel(const PackedBwdParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do) {
    constexpr int kTile_ = (kDim / 64) * kPanelBytes;
    // Where P goes: at head dim 64 the sums leave room in TMEM for two buffers of scores, P is written over its own; at 128
    // there is one, and P goes through shared memory so that S(i+1) need not wait for dV(i).
    constexpr bool kPInSmem = kDim == 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* k_smem = smem;
    uint8_t* v_smem = smem + kTile_;
    uint8_t* q_smem = smem + 2 * kTile_;                        // two stages
    uint8_t* do_smem = smem + 4 * kTile_;                       // two stages
    uint8_t* p_smem = smem + 6 * kTile_;                        // P^T: 128 keys x 128 queries
    constexpr int kAfterP = 6 * kTile_ + (kPInSmem ? 2 * kPanelBytes : 0);
    float* st_smem = reinterpret_cast<float*>(smem + kAfterP);
    BwdBarriers* bars = reinterpret_cast<BwdBarriers*>(smem + kAfterP + 2 * kStatFloats * 4);
    int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // with p.split CTAs per item (a cluster), this one takes heads from `first_head` on
    const int part = (int)blockIdx.x % p.split, number = (int)blockIdx.x / p.split;
    const int rank = number / p.kv_heads, kv_head = number - rank * p.kv_heads;
    const int heads = p.group / p.split, first_head = kv_head * p.group + part * heads;
    bwd_begin(bars, p, rank, warp, lane);
    const uint32_t tmem = *(volatile uint32_t*)&bars->tmem_base;
    const PackedItem item = bars->item;
    const bool work = item.length > 0 && item.b < p.batch;
    const int tiles = (item.length + kRowsTile - 1) / kRowsTile;
    const int key_tile = tiles - 1 - item.tile;                 // (the first keys are seen by the most queries)
    const int first_q = p.causal ? key_tile : 0;                // the query tiles that see these keys: first_q .. tiles - 1
    const int n = work ? (tiles - first_q) * heads : 0;
    const uint32_t s_tmem = tmem, dp_tmem = tmem + (kPInSmem ? 128u : 256u), dv_tmem = dp_tmem + 128u, dk_tmem = dv_tmem + kDim;
    bool ok = true;

    if (item.length > 0 && item.b == p.batch && part == 0) {    // rows behind the last sequence
        const int from = item.start + item.tile * kRowsTile, to = min(from + kRowsTile, p.rows);
        zero_tail(p.dk, from, to, kv_head, p.kv_heads, kDim, threadIdx.x, blockDim.x);
        zero_tail(p.dv, from, to, kv_head, p.kv_heads, kDim, threadIdx.x, blockDim.x);
    }
    if (warp == 8 && n > 0) {
        // ------------------------------------------------------------ producer
        if (elect_one()) {
            mbar_expect_tx(&bars->x_full, (uint32_t)(2 * kTile_));
#pragma unroll
            for (int c = 0; c < kDim / 64; ++c) {
                tma_load_3d(k_smem + c * kPanelBytes, &map_k, &bars->x_full, 64 * c, kv_head, item.start + key_tile * kRowsTile);
                tma_load_3d(v_smem + c * kPanelBytes, &map_v, &bars->x_full, 64 * c, kv_head, item.start + key_tile * kRowsTile);
            }
        }
        __syncwarp();
        int head = first_head, qt = first_q;
        for (int i = 0; ok && i < n; ++i) {
            const int st = i & 1;
            const uint32_t parity = ((uint32_t)(i >> 1) & 1u) ^ 1u;
            ok = wait_all(&bars->a_empty[st], parity, abort_flag, p.status);
            if (ok) load_tile<kDim>(q_smem + st * kTile_, &map_q, &bars->a_full[st], head, item.start + qt * kRowsTile);
            ok = ok && wait_all(&bars->b_empty[st], parity, abort_flag, p.status);
            if (ok) load_tile<kDim>(do_smem + st * kTile_, &map_do, &bars->b_full[st], head, item.start + qt * kRowsTile);
            if (++qt == tiles) { qt = first_q; ++head; }
        }
        if (lane == 0 && *(volatile int*)abort_flag) let_copies_land();
        __syncwarp();
    } else if (warp == 9 && n > 0) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t fmt = kBf16 ? 1u : 0u;
        const uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRowsTile >> 4) << 24);
        const uint32_t idesc_t = common | ((uint32_t)(kRowsTile >> 3) << 17);
        const uint32_t idesc_acc = common | (1u << 16) | ((uint32_t)(kDim >> 3) << 17);
        const uint64_t k_desc = panel_desc(smem_u32(k_smem), false), v_desc = panel_desc(smem_u32(v_smem), false);
        const uint64_t p_desc = panel_desc(smem_u32(p_smem), false);
        int q_tile = first_q, do_tile = first_q;                // of the tiles that are waited for next
        // a tile's rows behind the sequence's end must not reach the sums over rows
        auto ready = [&](uint64_t* full, uint8_t* base, int i, int& qt) {
            ok = wait_all(&full[i & 1], (uint32_t)(i >> 1) & 1u, abort_flag, p.status);
            if (!ok) return false;
            const int valid = item.length - qt * kRowsTile;
            if (valid < kRowsTile) zero_rows<kDim>(base + (i & 1) * kTile_, valid, lane);
            if (++qt == tiles) qt = first_q;
            return true;
        };
        auto scores = [&](int i) {
            if (elect_one()) {
                mma_rows<kDim>(s_tmem + (kPInSmem ? 0u : (uint32_t)(128 * (i & 1))), k_desc, panel_desc(smem_u32(q_smem + (i & 1) * kTile_), false), idesc_t);
                tc_commit(&bars->s_full[i & 1]);
            }
            __syncwarp();
        };
        auto products = [&](int i) {
            if (elect_one()) {
                mma_rows<kDim>(dp_tmem, v_desc, panel_desc(smem_u32(do_smem + (i & 1) * kTile_), false), idesc_t);
                tc_commit(&bars->dp_full[i & 1]);
            }
            __syncwarp();
        };
        ok = wait_all(&bars->x_full, 0, abort_flag, p.status);
        if (ok && ready(bars->a_full, q_smem, 0, q_tile)) {
            tc_fence_after();
            scores(0);
        }
        if (ok && ready(bars->b_full, do_smem, 0, do_tile)) {
            tc_fence_after();
            products(0);
        }
        for (int i = 0; ok && i < n; ++i) {
            const int st = i & 1;
            const bool more = i + 1 < n;
            if (more) {
                if (kPInSmem) ok = wait_turn(bars->s_read, i, abort_flag, p.status);
                if (!ok || !ready(bars->a_full, q_smem, i + 1, q_tile)) break;
                tc_fence_after();
                scores(i + 1);
            }
            ok = wait_turn(bars->p_full, i, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t do_desc = panel_desc(smem_u32(do_smem + st * kTile_), true);
#pragma unroll
                for (int kk = 0; kk < kRowsTile / 16; ++kk)
                    if (!kPInSmem)
                        tc_mma_f16_ts(dv_tmem, s_tmem + (uint32_t)(128 * st + 8 * kk), do_desc + (uint64_t)(kk * (2048 >> 4)), idesc_acc, i > 0 || kk > 0 ? 1u : 0u);
                    else
                        tc_mma_f16(dv_tmem, p_desc + (uint64_t)((kk / 4) * (kPanelBytes >> 4) + (kk % 4) * 2), do_desc + (uint64_t)(kk * (2048 >> 4)),
                               idesc_acc, i > 0 || kk > 0 ? 1u : 0u);
                tc_commit(&bars->p_empty[st]);
                tc_commit(&bars->b_empty[st]);
            }
            __syncwarp();
            ok = wait_turn(bars->ds_full, i, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                mma_keys<0>(dk_tmem, dp_tmem, panel_desc(smem_u32(q_smem + st * kTile_), true), idesc_acc, i > 0);
                mma_keys<1>(dk_tmem, dp_tmem, panel_desc(smem_u32(q_smem + st * kTile_), true), idesc_acc, true);
                tc_commit(&bars->a_empty[st]);
                if (!more) tc_commit(&bars->done);
            }
            __syncwarp();
            if (more) {
                if (!ready(bars->b_full, do_smem, i + 1, do_tile)) break;
                products(i + 1);
            }
        }
        if (elect_one()) {
            tc_commit(&bars->drain);
            mbar_wait(&bars->drain, 0, abort_flag, p.status);
        }
        __syncwarp();
    } else if (warp == 10) {
        // ------------------------------------------------------------ statistics of the query tiles
        int head = first_head, qt = first_q;
        for (int i = 0; ok && i < n; ++i) {
            const int st = i & 1, row = qt * kRowsTile + 4 * lane;
            float2 s[4];                                        // negated; behind the sequence's end P = 2^-inf = 0 and dS = 0
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[e] = row + e < item.length ? p.stats[(size_t)head * p.rows + item.start + row + e] : make_float2(INFINITY, 0.0f);
                s[e].x = -s[e].x;
                s[e].y = -s[e].y;
            }
            ok = wait_all(&bars->st_empty[st], ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag, p.status);
            if (!ok) break;
            float4* to = reinterpret_cast<float4*>(st_smem + st * kStatFloats);
            to[lane] = make_float4(s[0].x, s[1].x, s[2].x, s[3].x);
            to[32 + lane] = make_float4(s[0].y, s[1].y, s[2].y, s[3].y);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->st_full[st]);
            if (++qt == tiles) { qt = first_q; ++head; }
        }
    } else if (warp < 8 && n > 0) {
        // ------------------------------------------------------------ P and dS of every second tile: one key per thread
        const int mine = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const float c = p.scale_log2;
        uint8_t* p_row = p_smem + r * 128;
        const float4* lse4 = reinterpret_cast<const float4*>(st_smem + mine * kStatFloats);
        const float4* delta4 = lse4 + kRowsTile / 4;
        const uint64_t c2 = f2_pack(c, c);
        int qt = first_q;
        for (int i = 0; i < n; ++i) {
            const bool diagonal = p.causal && qt == key_tile;       // queries from r on see the key
            if (++qt == tiles) qt = first_q;
            if ((i & 1) != mine) continue;
            ok = wait_turn(bars->st_full, i, abort_flag, p.status) && wait_turn(bars->s_full, i, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_at = s_tmem + lanes + (kPInSmem ? 0u : (uint32_t)(128 * mine));
            uint32_t x[4][32];
#pragma unroll
            for (int q = 0; q < 4; ++q) tc_ld_32x32b_x32(s_at + (uint32_t)(32 * q), x[q]);
            tc_wait_ld();
            if (kPInSmem) {
                arrive_warp(&bars->s_read[mine], lane);
                if (i > 0) ok = wait_turn(bars->p_empty, i - 1, abort_flag, p.status);
                if (!ok) break;
            }
            if (diagonal) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * q + e < r) x[q][e] = p.scale_log2 < 0.0f ? 0x7f800000u : 0xff800000u;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 lse = lse4[8 * q + e / 4];
                    float y[4];
                    f2_unpack(f2_fma(f2_of(x[q][e], x[q][e + 1]), c2, f2_pack(lse.x, lse.y)), y[0], y[1]);
                    f2_unpack(f2_fma(f2_of(x[q][e + 2], x[q][e + 3]), c2, f2_pack(lse.z, lse.w)), y[2], y[3]);
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[q][e + u] = __float_as_uint(attn_exp2(y[u]));
                    w[e / 2] = pack2<kBf16>(__uint_as_float(x[q][e]), __uint_as_float(x[q][e + 1]));
                    w[e / 2 + 1] = pack2<kBf16>(__uint_as_float(x[q][e + 2]), __uint_as_float(x[q][e + 3]));
                }
                if (kPInSmem) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int chunk = 4 * q + u;
                        *reinterpret_cast<uint4*>(p_row + (chunk >> 3) * kPanelBytes + (((chunk & 7) ^ (r & 7)) << 4)) =
                            make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
                    }
                } else {
                    tc_st_32x32b_x16(s_at + (uint32_t)(16 * q), w);
                }
            }
            if (kPInSmem) fence_async_shared();
            else tc_wait_st();
            arrive_warp(&bars->p_full[mine], lane);
            ok = wait_turn(bars->dp_full, i, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            uint32_t d[2][16];
            tc_ld_32x32b_x16(dp_tmem + lanes, d[0]);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                tc_wait_ld();
                if (q < 7) tc_ld_32x32b_x16(dp_tmem + lanes + (uint32_t)(16 * (q + 1)), d[(q + 1) & 1]);
                uint32_t (&h)[16] = d[q & 1];
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 delta = delta4[4 * q + e / 4];
                    const uint32_t* at = &x[q / 2][16 * (q & 1) + e];
                    float y[4];
                    f2_unpack(f2_mul(f2_of(at[0], at[1]), f2_add(f2_of(h[e], h[e + 1]), f2_pack(delta.x, delta.y))), y[0], y[1]);
                    f2_unpack(f2_mul(f2_of(at[2], at[3]), f2_add(f2_of(h[e + 2], h[e + 3]), f2_pack(delta.z, delta.w))), y[2], y[3]);
                    x[q / 2][8 * (q & 1) + e / 2] = pack2<kBf16>(y[0], y[1]);
                    x[q / 2][8 * (q & 1) + e / 2 + 1] = pack2<kBf16>(y[2], y[3]);
                }
                // 16 words over columns of dP that have been read
                if (q & 1) tc_st_32x32b_x16(dp_tmem + lanes + (uint32_t)(8 * (q - 1)), x[q / 2]);
            }
            tc_wait_st();
            arrive_warp(&bars->ds_full[mine], lane);
            if (lane == 0) mbar_arrive(&bars->st_empty[mine]);
        }
        ok = ok && wait_all(&bars->done, 0, abort_flag, p.status);
        tc_fence_after();
    }
    // Sums: warps 0-3 store dV, 4-7 dK.  In a cluster the second CTA hands its own to the first: 128 x D floats of each, into
    // the stages of Q and dO, which are free once both are done.
    if (n > 0 && p.split == 2) cluster_sync();
    if (warp < 8 && n > 0) {
        const int which = warp >> 2, r = (warp & 3) * 32 + lane, key = key_tile * kRowsTile + r;
        const uint32_t from = (which ? dk_tmem : dv_tmem) + ((uint32_t)((warp & 3) * 32) << 16);
        const float by = which ? p.scale : 1.0f;
        float4* here = reinterpret_cast<float4*>(q_smem) + which * (kRowsTile * kDim / 4) + r;
        if (part == 1) {
            const uint32_t there = peer_address(smem_u32(here), 0);
#pragma unroll
            for (int i = 0; i < kDim / 32; ++i) {
                uint32_t acc[32];
                tc_ld_32x32b_x32(from + (uint32_t)(32 * i), acc);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};"
                                 ::"r"(there + (uint32_t)((8 * i + e / 4) * kRowsTile * 16)), "r"(acc[e]), "r"(acc[e + 1]), "r"(acc[e + 2]), "r"(acc[e + 3]) : "memory");
            }
        }
        if (p.split == 2) cluster_sync();
        if (part == 0) {
            uint8_t* to = static_cast<uint8_t*>(which ? p.dk : p.dv) + ((size_t)(item.start + key) * p.kv_heads + kv_head) * kDim * 2;
#pragma unroll
            for (int i = 0; i < kDim / 32; ++i) {
                uint32_t acc[32];
                tc_ld_32x32b_x32(from + (uint32_t)(32 * i), acc);
                tc_wait_ld();
                if (p.split == 2) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 other = here[(8 * i + e / 4) * kRowsTile];
                        acc[e] = __float_as_uint(__uint_as_float(acc[e]) + other.x);
                        acc[e + 1] = __float_as_uint(__uint_as_float(acc[e + 1]) + other.y);
                        acc[e + 2] = __float_as_uint(__uint_as_float(acc[e + 2]) + other.z);
                        acc[e + 3] = __float_as_uint(__uint_as_float(acc[e + 3]) + other.w);
                    }
                }
                if (ok && key < item.length) store_row32<kBf16>(to + 64 * i, acc, by);
            }
        }
    } else if (n > 0 && p.split == 2) {
        cluster_sync();
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
    uint8_t* k_smem = smem + 2 * kTile_;                        // three stages: K(j) is read until dQ(j)
    uint8_t* v_smem = smem + 5 * kTile_;                        // two stages
    BwdBarriers* bars = reinterpret_cast<BwdBarriers*>(smem + 7 * kTile_);
    int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x / p.q_heads, head = (int)blockIdx.x - rank * p.q_heads, kv_head = head / p.group;
    bwd_begin(bars, p, rank, warp, lane);
    const uint32_t tmem = *(volatile uint32_t*)&bars->tmem_base;
    const PackedItem item = bars->item;
    const bool work = item.length > 0 && item.b < p.batch;
    const int tiles = (item.length + kRowsTile - 1) / kRowsTile, tile = item.tile;
    const int n = work ? (p.causal ? tile + 1 : tiles) : 0;
    const uint32_t dp_tmem = tmem + 256u, dq_tmem = tmem + 384u;
    bool ok = true;

    if (item.length > 0 && item.b == p.batch) {
        const int from = item.start + item.tile * kRowsTile, to = min(from + kRowsTile, p.rows);
        zero_tail(p.dq, from, to, head, p.q_heads, kDim, threadIdx.x, blockDim.x);
    }
    if (warp == 8 && n > 0) {
        // ------------------------------------------------------------ producer
        if (elect_one()) {
            mbar_expect_tx(&bars->x_full, (uint32_t)(2 * kTile_));
#pragma unroll
            for (int c = 0; c < kDim / 64; ++c) {
                tma_load_3d(q_smem + c * kPanelBytes, &map_q, &bars->x_full, 64 * c, head, item.start + tile * kRowsTile);
                tma_load_3d(do_smem + c * kPanelBytes, &map_do, &bars->x_full, 64 * c, head, item.start + tile * kRowsTile);
            }
        }
        __syncwarp();
        for (int j = 0, st = 0; ok && j < n; ++j, st = st == 2 ? 0 : st + 1) {
            ok = wait_all(&bars->a_empty[st], ((uint32_t)(j / 3) & 1u) ^ 1u, abort_flag, p.status);
            if (ok) load_tile<kDim>(k_smem + st * kTile_, &map_k, &bars->a_full[st], kv_head, item.start + j * kRowsTile);
            ok = ok && wait_all(&bars->b_empty[j & 1], ((uint32_t)(j >> 1) & 1u) ^ 1u, abort_flag, p.status);
            if (ok) load_tile<kDim>(v_smem + (j & 1) * kTile_, &map_v, &bars->b_full[j & 1], kv_head, item.start + j * kRowsTile);
        }
        if (lane == 0 && *(volatile int*)abort_flag) let_copies_land();
        __syncwarp();
    } else if (warp == 9 && n > 0) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t fmt = kBf16 ? 1u : 0u;
        const uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRowsTile >> 4) << 24);
        const uint32_t idesc_t = common | ((uint32_t)(kRowsTile >> 3) << 17);
        const uint32_t idesc_acc = common | (1u << 16) | ((uint32_t)(kDim >> 3) << 17);
        const uint64_t q_desc = panel_desc(smem_u32(q_smem), false), do_desc = panel_desc(smem_u32(do_smem), false);
        auto scores = [&](int j) {
            const int st = j % 3, valid = item.length - j * kRowsTile;
            ok = wait_all(&bars->a_full[st], (uint32_t)(j / 3) & 1u, abort_flag, p.status);
            if (!ok) return;
            if (valid < kRowsTile) zero_rows<kDim>(k_smem + st * kTile_, valid, lane);       // summed over keys in dQ
            tc_fence_after();
            if (elect_one()) {
                mma_rows<kDim>(tmem + (uint32_t)(128 * (j & 1)), q_desc, panel_desc(smem_u32(k_smem + st * kTile_), false), idesc_t);
                tc_commit(&bars->s_full[j & 1]);
            }
            __syncwarp();
        };
        auto products = [&](int j) {
            ok = wait_turn(bars->b_full, j, abort_flag, p.status);
            if (!ok) return;
            // (dP of keys behind the end is 0 and meets P = 0; it could be NaN otherwise)
            const int valid = item.length - j * kRowsTile;
            if (valid < kRowsTile) zero_rows<kDim>(v_smem + (j & 1) * kTile_, valid, lane);
            tc_fence_after();
            if (elect_one()) {
                mma_rows<kDim>(dp_tmem, do_desc, panel_desc(smem_u32(v_smem + (j & 1) * kTile_), false), idesc_t);
                tc_commit(&bars->dp_full[j & 1]);
                tc_commit(&bars->b_empty[j & 1]);
            }
            __syncwarp();
        };
        ok = wait_all(&bars->x_full, 0, abort_flag, p.status);
        if (ok) scores(0);
        if (ok) products(0);
        for (int j = 0; ok && j < n; ++j) {
            const bool more = j + 1 < n;
            if (more) scores(j + 1);
            if (!ok) break;
            if (more) {
                ok = wait_turn(bars->dp_read, j, abort_flag, p.status);
                if (!ok) break;
                products(j + 1);
                if (!ok) break;
            }
            ok = wait_turn(bars->ds_full, j, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t a = tmem + (uint32_t)(128 * (j & 1));
                const uint64_t k_desc = panel_desc(smem_u32(k_smem + j % 3 * kTile_), true);
                mma_keys<0>(dq_tmem, a, k_desc, idesc_acc, j > 0);
                mma_keys<1>(dq_tmem, a, k_desc, idesc_acc, true);
                tc_commit(&bars->a_empty[j % 3]);
                if (!more) tc_commit(&bars->done);
            }
            __syncwarp();
        }
        if (elect_one()) {
            tc_commit(&bars->drain);
            mbar_wait(&bars->drain, 0, abort_flag, p.status);
        }
        __syncwarp();
    } else if (warp < 8 && n > 0) {
        // ------------------------------------------------------------ P and dS of every second tile: one query per thread
        const int mine = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const float c = p.scale_log2;
        const int row = tile * kRowsTile + r;
        const int last = p.causal ? min(row, item.length - 1) : item.length - 1;
        const float2 stat = row < item.length ? p.stats[(size_t)head * p.rows + item.start + row] : make_float2(INFINITY, 0.0f);
        const uint64_t c2 = f2_pack(c, c), lse2 = f2_pack(-stat.x, -stat.x), delta2 = f2_pack(-stat.y, -stat.y);
        const uint32_t s_tmem = tmem + (uint32_t)(128 * mine) + lanes;
        for (int j = mine; j < n; j += 2) {
            const int see = last - j * kRowsTile;                           // columns 0 .. see of the tile are seen
            const bool masked = __any_sync(0xffffffffu, see < kRowsTile - 1) != 0;
            ok = wait_turn(bars->s_full, j, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            uint32_t x[4][32];
#pragma unroll
            for (int q = 0; q < 4; ++q) tc_ld_32x32b_x32(s_tmem + (uint32_t)(32 * q), x[q]);
            tc_wait_ld();
            if (masked) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * q + e > see) x[q][e] = p.scale_log2 < 0.0f ? 0x7f800000u : 0xff800000u;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float a, b;
                    f2_unpack(f2_fma(f2_of(x[q][e], x[q][e + 1]), c2, lse2), a, b);
                    x[q][e] = __float_as_uint(attn_exp2(a));
                    x[q][e + 1] = __float_as_uint(attn_exp2(b));
                }
            ok = wait_turn(bars->dp_full, j, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            uint32_t d[2][16];
            tc_ld_32x32b_x16(dp_tmem + lanes, d[0]);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                tc_wait_ld();
                if (q < 7) tc_ld_32x32b_x16(dp_tmem + lanes + (uint32_t)(16 * (q + 1)), d[(q + 1) & 1]);
                else arrive_warp(&bars->dp_read[mine], lane);
                uint32_t (&h)[16] = d[q & 1];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const uint32_t* at = &x[q / 2][16 * (q & 1) + e];
                    float a, b;
                    f2_unpack(f2_mul(f2_of(at[0], at[1]), f2_add(f2_of(h[e], h[e + 1]), delta2)), a, b);
                    x[q / 2][8 * (q & 1) + e / 2] = pack2<kBf16>(a, b);
                }
                if (q & 1) tc_st_32x32b_x16(s_tmem + (uint32_t)(8 * (q - 1)), x[q / 2]);
            }
            tc_wait_st();
            arrive_warp(&bars->ds_full[mine], lane);
        }
        ok = ok && wait_all(&bars->done, 0, abort_flag, p.status);
        tc_fence_after();
        const size_t at = ((size_t)(item.start + row) * p.q_heads + head) * kDim;
#pragma unroll
        for (int i = 0; i < kDim / 64; ++i) {                   // each warpgroup stores half of the columns
            const int col = mine * (kDim / 2) + 32 * i;
            uint32_t acc[32];
            tc_ld_32x32b_x32(dq_tmem + lanes + (uint32_t)col, acc);
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
    constexpr int smem = bwd_smem<kDim>(), smem_keys = bwd_smem_keys<kDim>();
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(keys), smem_keys) ||
        !ensure_dynamic_smem(reinterpret_cast<const void*>(queries), smem)) return BSA_ERR_LAUNCH;
    const int64_t rows_heads = (int64_t)p.rows * p.q_heads, per_cta = 256 / (kDim / 8);
    packed_stats_kernel<T, kDim><<<(unsigned)((rows_heads + per_cta - 1) / per_cta), 256, 0, stream>>>(p);
    const unsigned items = (unsigned)(p.rows / kRowsTile + p.batch + 1);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(items * p.kv_heads * p.split);
    config.blockDim = dim3(kBwdThreads);
    config.dynamicSmemBytes = smem_keys;
    config.stream = stream;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = (unsigned)p.split;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, keys, p, mq, mk, mv, mdo) != cudaSuccess) { cudaGetLastError(); return BSA_ERR_LAUNCH; }
    queries<<<items * p.q_heads, kBwdThreads, smem, stream>>>(p, mq, mk, mv, mdo);
    return launch_status();
}

}  // namespace
}  // namespace bsa

extern "C" int bsa_packed_backward(int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                   int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                   int64_t v_head_stride, const void* o, const void* o_low, const void* dout, int64_t dout_token_stride,
                                   int64_t dout_head_stride, const float* lse, void* dq, void* dk, void* dv,
                                   const int32_t* offsets, int64_t rows, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                   int64_t head_dim, float scale, int causal, void* stats, size_t stats_bytes,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    using namespace bsa;
    int checked = check_packed(dtype, rows, batch, q_heads, kv_heads, head_dim);
    if (checked != BSA_OK) return checked;
    if (!workspace || workspace_bytes < BSA_WORKSPACE_BYTES) return BSA_ERR_WORKSPACE;
    if (rows == 0) return BSA_OK;
    if (!q || !k || !v || !o || !o_low || !dout || !lse || !dq || !dk || !dv || !offsets || !stats) return BSA_ERR_NULL_POINTER;
    for (const void* ptr : {q, k, v, o, o_low, dout, static_cast<const void*>(stats)})
        if (!aligned16(ptr)) return BSA_ERR_ALIGNMENT;
    for (const void* ptr : {dq, dk, dv})
        if (reinterpret_cast<uintptr_t>(ptr) & 31) return BSA_ERR_ALIGNMENT;
    if ((checked = check_strides(q_token_stride, q_head_stride)) != BSA_OK || (checked = check_strides(k_token_stride, k_head_stride)) != BSA_OK ||
        (checked = check_strides(v_token_stride, v_head_stride)) != BSA_OK ||
        (checked = check_strides(dout_token_stride, dout_head_stride)) != BSA_OK) return checked;
    if (stats_bytes < (size_t)rows * q_heads * sizeof(float2)) return BSA_ERR_WORKSPACE;
    PackedBwdParams p{};
    p.o = o; p.o_low = o_low; p.dout = dout; p.dout_token = dout_token_stride; p.dout_head = dout_head_stride;
    p.lse = lse; p.stats = static_cast<float2*>(stats);
    p.dq = dq; p.dk = dk; p.dv = dv; p.offsets = offsets;
    p.batch = (int)batch; p.rows = (int)rows; p.q_heads = (int)q_heads; p.kv_heads = (int)kv_heads;
    p.group = (int)(q_heads / kv_heads); p.causal = causal != 0;
    p.split = p.group % 2 == 0 ? 2 : 1;
    p.scale = scale;
    p.scale_log2 = scale * kPackedLog2e;
    if (fabsf(p.scale_log2) < 1e-37f) p.scale_log2 = 1e-37f;     // a factor that keeps masked scores at -infinity
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
