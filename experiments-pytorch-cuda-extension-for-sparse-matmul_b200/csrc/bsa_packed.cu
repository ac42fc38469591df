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
// The CTAs are persistent (one per SM): a CTA takes over the places of CTAs of the grid that have not started (cluster
// launch control), so the list of tiles, longest first, is shared out as SMs come free; while the softmax warps end one
// item, the producer already loads the next one's Q and K and its first scores are computed.
//   warps 0-3, 4-7   softmax of tile 0 / 1, one row per thread; the epilogue
//   warp 8           TMA producer: items, Q, then K and V tiles through a ring of 4 stages
//   warp 9           MMA issuer: S0 S1 | PV0 S0' PV1 S1' | ..; each PV in two parts, the first while the second half of P is made
// The last K / V tile of a sequence may hold rows of the next one; its V rows are zeroed before use (see zero_rows).
// All waits are bounded.
//
// 16,127 rows of 8 sequences, 16 / 4 heads x 128, bf16: 219 to 227 us, 930 to 960 TFLOP/s (194 us replayed on the
// same inputs).  A pair of tiles takes 3100 cycles where the tensor pipe needs 2048: the chain of one tile (waiting for
// its MMAs 1130 cycles, 400 until its maximum, 1330 of exponentials) is half hidden behind the other's.
#include <climits>
#include <type_traits>

#include "bsa_packed_common.cuh"

namespace bsa {
namespace {

constexpr int kFwdStages = 4;
constexpr int kFwdThreads = 320;

struct PackedParams {
    void* o;
    void* o_low;                                // what rounding took from o, in o's type
    float* lse;                                 // [q_heads, rows], in units of log2, scale included
    const int32_t* offsets;
    int batch, rows, q_heads, kv_heads, group, causal;
    int items;                                  // upper bound of the work items
    int pair;                                   // the two tiles: heads 2 h, 2 h + 1 of a group (1), or rows (0)
    float scale_log2;                           // |scale| log2 e
    int negative;                               // scale < 0
    uint32_t* status;
};

struct __align__(16) FwdBarriers {
    uint64_t item_full[2], item_empty[2];
    uint64_t q_full[2], q_empty[2], full[kFwdStages], empty[kFwdStages];
    uint64_t s_full[2], p_full[2][2], o_full[2];
    uint64_t drain, stolen;
    uint4 response;                             // of the request for another CTA's place
    int4 items[2];                              // first row of the sequence, its length, the tile, the first head; length 0: no more
    uint32_t tmem_base;
    int abort_flag;
};

constexpr int kStoreBytes = 8 * 32 * 128;       // a store stage per softmax warp
template <int kDim>
constexpr int fwd_smem() { return (2 + kFwdStages) * (kDim / 64) * kPanelBytes + kStoreBytes + (int)sizeof(FwdBarriers); }

// What an item means: K / V tiles of each of its two Q tiles.
struct FwdItem {
    int start, length, row0, head0, steps[2];
    __device__ __forceinline__ FwdItem(const int4& v, const PackedParams& p) {
        start = v.x; length = v.y; head0 = v.w;
        row0 = v.z * (p.pair ? kRowsTile : 2 * kRowsTile);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int first = p.pair ? row0 : row0 + s * kRowsTile;
            const int keys = p.causal ? min(first + kRowsTile, length) : length;
            steps[s] = first < length ? (keys + kRowsTile - 1) / kRowsTile : 0;
        }
    }
};

// kKeep: what a backward needs is kept (the rest of o, lse).
template <bool kBf16, int kDim, bool kKeep>
__global__ void __launch_bounds__(kFwdThreads, 1)
packed_forward_kernel(const PackedParams p, const __grid_constant__ CUtensorMap map_q,
                      const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_low) {
    constexpr int kPanels = kDim / 64, kTile_ = kPanels * kPanelBytes;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* ring = smem + 2 * kTile_;
    uint8_t* store_smem = ring + kFwdStages * kTile_;
    FwdBarriers* bars = reinterpret_cast<FwdBarriers*>(store_smem + kStoreBytes);
    int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int i = 0; i < kFwdStages; ++i) { mbar_init(&bars->full[i], 1); mbar_init(&bars->empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars->item_full[i], 1); mbar_init(&bars->item_empty[i], 9);
            mbar_init(&bars->q_full[i], 1); mbar_init(&bars->q_empty[i], 1);
            mbar_init(&bars->s_full[i], 1); mbar_init(&bars->o_full[i], 1);
            mbar_init(&bars->p_full[i][0], 4); mbar_init(&bars->p_full[i][1], 4);
        }
        mbar_init(&bars->drain, 1);
        mbar_init(&bars->stolen, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&bars->tmem_base;
    bool ok = true;
    // the next item, for every warp but the producer; false: no more
    int item_no = 0;
    auto next_item = [&](int4& v) {
        const int slot = item_no & 1;
        ok = wait_all(&bars->item_full[slot], (uint32_t)(item_no >> 1) & 1u, abort_flag, p.status);
        if (!ok) return false;
        v = bars->items[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->item_empty[slot]);
        ++item_no;
        return v.y > 0;
    };

    if (warp == 8) {
        // ------------------------------------------------------------ producer
        const int per_tile = p.pair ? kRowsTile : 2 * kRowsTile;
        const int head_items = p.pair ? p.q_heads / 2 : p.q_heads;
        int posted = 0, t = 0, q_no[2] = {0, 0};
        auto post = [&](const int4& v) {
            const int slot = posted & 1;
            ok = wait_all(&bars->item_empty[slot], ((uint32_t)(posted >> 1) & 1u) ^ 1u, abort_flag, p.status);
            if (ok && lane == 0) {
                bars->items[slot] = v;
                mbar_arrive(&bars->item_full[slot]);
            }
            __syncwarp();
            ++posted;
        };
        auto load = [&](uint8_t* to, const CUtensorMap* map, uint64_t* bar, int head, int row) {
            if (elect_one()) {
                mbar_expect_tx(bar, (uint32_t)kTile_);
#pragma unroll
                for (int c = 0; c < kPanels; ++c) tma_load_3d(to + c * kPanelBytes, map, bar, 64 * c, head, row);
            }
            __syncwarp();
        };
        bool more = true;
        int behind = INT_MAX;                                   // the smallest rank found to lie behind the list's end
        int at = (int)blockIdx.x, next = 0;
        for (int round = 0; ok && more; ++round, at = next) {
            // The next item: the place of a CTA that has not started yet.  Asked for once this one's loads are out, about two
            // steps before its end: earlier, an SM with a long item would hold back another one.
            auto take = [&]() {
                if (lane == 0) {
                    mbar_expect_tx(&bars->stolen, 16);
                    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                                 ::"r"(smem_u32(&bars->response)), "r"(smem_u32(&bars->stolen)) : "memory");
                }
                __syncwarp();
                if (!wait_all(&bars->stolen, (uint32_t)round & 1u, abort_flag, p.status)) { ok = false; return; }
                uint32_t canceled;
                asm volatile("{\n\t.reg .b128 r;\n\t.reg .pred c;\n\tld.shared.b128 r, [%2];\n\t"
                             "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 c, r;\n\tselp.u32 %0, 1, 0, c;\n\t"
                             "mov.u32 %1, 0;\n\t@c clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
                             : "=r"(canceled), "=r"(next) : "r"(smem_u32(&bars->response)) : "memory");
                fence_async_shared();
                __syncwarp();
                more = canceled != 0;
            };
            const int rank = at / head_items, head_item = at - rank * head_items, head0 = p.pair ? 2 * head_item : head_item;
            PackedItem found{0, 0, 0, 0};
            if (rank < behind) found = packed_locate(p.offsets, p.batch, p.rows, per_tile, rank, lane, p.status);
            if (found.length == 0) {                            // behind the list's end, and so is every larger rank (a place
                behind = min(behind, rank);                     // that is taken over later may have a smaller one)
                take();
                continue;
            }
            if (found.b == p.batch) {                           // rows behind the last sequence
                const int from = found.start + found.tile * per_tile, to = min(from + per_tile, p.rows);
                for (int h = head0; h <= head0 + p.pair; ++h) {
                    zero_tail(p.o, from, to, h, p.q_heads, kDim, lane, 32);
                    if (kKeep) zero_tail(p.o_low, from, to, h, p.q_heads, kDim, lane, 32);
                    if (kKeep)
                        for (int r = from + lane; r < to; r += 32) p.lse[(size_t)h * p.rows + r] = -INFINITY;
                }
                take();
                continue;
            }
            const int4 v = make_int4(found.start, found.length, found.tile, head0);
            post(v);
            const FwdItem item(v, p);
            const int all_steps = max(item.steps[0], item.steps[1]), kv_head = head0 / p.group;
            for (int j = 0; ok && j < 2 * all_steps; ++j, ++t) {        // K of step j / 2, then V; the Q tiles around the first
                if (j < 2 && item.steps[j] > 0) {
                    ok = wait_all(&bars->q_empty[j], ((uint32_t)q_no[j] & 1u) ^ 1u, abort_flag, p.status);
                    if (!ok) break;
                    ++q_no[j];
                    load(smem + j * kTile_, &map_q, &bars->q_full[j], p.pair ? head0 + j : head0,
                         item.start + item.row0 + (p.pair ? 0 : j * kRowsTile));
                }
                const int stage = t % kFwdStages;
                ok = wait_all(&bars->empty[stage], ((uint32_t)(t / kFwdStages) & 1u) ^ 1u, abort_flag, p.status);
                if (ok) load(ring + stage * kTile_, j & 1 ? &map_v : &map_k, &bars->full[stage], kv_head, item.start + (j / 2) * kRowsTile);
            }
            if (ok) take();
        }
        if (ok) post(make_int4(0, 0, 0, 0));
        if (lane == 0 && *(volatile int*)abort_flag) let_copies_land();
        __syncwarp();
    } else if (warp == 9) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t fmt = kBf16 ? 1u : 0u;
        const uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRowsTile >> 4) << 24);
        const uint32_t idesc_s = common | ((uint32_t)(kRowsTile >> 3) << 17);
        const uint32_t idesc_o = common | (1u << 16) | ((uint32_t)(kDim >> 3) << 17);
        const uint64_t q_desc[2] = {panel_desc(smem_u32(smem), false), panel_desc(smem_u32(smem + kTile_), false)};
        int t = 0, q_no[2] = {0, 0}, p_no[2] = {0, 0};          // tiles of the ring, Q tiles and P tiles so far
        auto stage_ready = [&](int no) {
            ok = wait_all(&bars->full[no % kFwdStages], (uint32_t)(no / kFwdStages) & 1u, abort_flag, p.status);
            return ok;
        };
        int4 v;
        while (next_item(v)) {
            const FwdItem item(v, p);
            const int all_steps = max(item.steps[0], item.steps[1]);
            if (!stage_ready(t)) break;
            {
                const uint64_t k_desc = panel_desc(smem_u32(ring + t % kFwdStages * kTile_), false);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (!ok || item.steps[s] == 0) continue;
                    ok = wait_all(&bars->q_full[s], (uint32_t)q_no[s]++ & 1u, abort_flag, p.status);
                    if (!ok) continue;
                    tc_fence_after();
                    if (elect_one()) {
                        mma_rows<kDim>(tmem + (uint32_t)(s * 128), q_desc[s], k_desc, idesc_s);
                        tc_commit(&bars->s_full[s]);
                        if (item.steps[s] == 1) tc_commit(&bars->q_empty[s]);
                    }
                    __syncwarp();
                }
                if (ok && elect_one()) tc_commit(&bars->empty[t % kFwdStages]);
                __syncwarp();
            }
            for (int j = 0; ok && j < all_steps; ++j) {
                const int v_stage = (t + 2 * j + 1) % kFwdStages, k_stage = (t + 2 * j + 2) % kFwdStages;
                const bool more = j + 1 < all_steps;
                if (!stage_ready(t + 2 * j + 1) || (more && !stage_ready(t + 2 * j + 2))) break;
                const int valid = item.length - j * kRowsTile;
                if (valid < kRowsTile) zero_rows<kDim>(ring + v_stage * kTile_, valid, lane);
                const uint64_t v_desc = panel_desc(smem_u32(ring + v_stage * kTile_), true);
                const uint64_t k_desc = panel_desc(smem_u32(ring + k_stage * kTile_), false);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (!ok || j >= item.steps[s]) continue;
                    const uint32_t s_tmem = tmem + (uint32_t)(s * 128), o_tmem = tmem + (uint32_t)(256 + s * kDim);
                    ok = wait_all(&bars->p_full[s][0], (uint32_t)p_no[s] & 1u, abort_flag, p.status);
                    if (!ok) continue;
                    tc_fence_after();
                    if (elect_one()) mma_keys<0>(o_tmem, s_tmem, v_desc, idesc_o, j > 0);
                    __syncwarp();
                    ok = wait_all(&bars->p_full[s][1], (uint32_t)p_no[s]++ & 1u, abort_flag, p.status);
                    if (!ok) continue;
                    tc_fence_after();
                    if (elect_one()) {
                        mma_keys<1>(o_tmem, s_tmem, v_desc, idesc_o, true);
                        if (j + 1 < item.steps[s]) {
                            mma_rows<kDim>(s_tmem, q_desc[s], k_desc, idesc_s);
                            tc_commit(&bars->s_full[s]);
                            if (j + 2 == item.steps[s]) tc_commit(&bars->q_empty[s]);
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
            t += 2 * all_steps;
            if (!ok) break;
        }
        // all MMAs issued by the elected lane must have retired before TMEM is freed
        if (elect_one()) {
            tc_commit(&bars->drain);
            mbar_wait(&bars->drain, 0, abort_flag, p.status);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax of tile s, one row per thread
        const int s = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_tmem = tmem + lanes + (uint32_t)(s * 128), o_tmem = tmem + lanes + (uint32_t)(256 + s * kDim);
        const float c = p.scale_log2;
        int s_no = 0, o_no = 0;
        int4 v;
        while (next_item(v)) {
            const FwdItem item(v, p);
            const int n = item.steps[s];
            if (n == 0) continue;
            const int row = item.row0 + (p.pair ? 0 : s * kRowsTile) + r;           // in the sequence
            const int last = p.causal ? min(row, item.length - 1) : item.length - 1;      // the last key the row sees
            float m = -INFINITY, l = 0.0f;                                          // m in units of c S
            for (int j = 0; j < n; ++j) {
                ok = wait_all(&bars->s_full[s], (uint32_t)s_no++ & 1u, abort_flag, p.status);
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
                const int see = last - j * kRowsTile;                               // columns 0 .. see of the tile are seen
                const bool masked = __any_sync(0xffffffffu, see < kRowsTile - 1) != 0;
                if (masked) {
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
                        // rare; 8 columns at a time, beside the 128 scores that are in registers
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
                const uint64_t c2 = f2_pack(c, c), ref2 = f2_pack(ref, ref);
                uint64_t sum[2] = {0ull, 0ull};
                // The first half of P goes out before the second is made: its products run meanwhile.
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int i = 2 * half; i < 2 * half + 2; ++i)
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float a, b;
                            f2_unpack(f2_fma(f2_of(x[i][e], x[i][e + 1]), c2, ref2), a, b);
                            a = attn_exp2(a);
                            b = attn_exp2(b);
                            sum[(e / 2) & 1] = f2_add(sum[(e / 2) & 1], f2_pack(a, b));
                            x[half][(i & 1) * 16 + e / 2] = pack2<kBf16>(a, b);
                        }
                    tc_st_32x32b_x32(s_tmem + (uint32_t)(32 * half), x[half]);
                    tc_wait_st();
                    arrive_warp(&bars->p_full[s][half], lane);
                }
                float a, b;
                f2_unpack(f2_add(sum[0], sum[1]), a, b);
                l += a + b;
            }
            if (!ok) break;
            ok = wait_all(&bars->o_full[s], (uint32_t)o_no++ & 1u, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            const int head = p.pair ? item.head0 + s : item.head0;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const bool full = row - lane + 32 <= item.length;                       // all 32 rows of the warp
            const size_t at = ((size_t)(item.start + row) * p.q_heads + head) * kDim;
            uint8_t* stage = store_smem + warp * 4096;
#pragma unroll
            for (int i = 0; i < kDim / 64; ++i) {
                uint32_t acc[2][32], w[32];
                tc_ld_32x32b_x32(o_tmem + (uint32_t)(64 * i), acc[0]);
                tc_ld_32x32b_x32(o_tmem + (uint32_t)(64 * i + 32), acc[1]);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 64; e += 2) {
                    acc[e / 32][e % 32] = __float_as_uint(__uint_as_float(acc[e / 32][e % 32]) * inv);
                    acc[e / 32][e % 32 + 1] = __float_as_uint(__uint_as_float(acc[e / 32][e % 32 + 1]) * inv);
                    w[e / 2] = pack2<kBf16>(__uint_as_float(acc[e / 32][e % 32]), __uint_as_float(acc[e / 32][e % 32 + 1]));
                }
                if (full) store_rows64(stage, &map_o, w, 64 * i, head, item.start + row - lane, lane);
                else if (row < item.length) store_row64(static_cast<uint8_t*>(p.o) + (at + 64 * i) * 2, w);
                if (kKeep) {
#pragma unroll
                    for (int e = 0; e < 64; e += 2) {
                        const float2 v = word_values<kBf16>(w[e / 2]);
                        w[e / 2] = pack2<kBf16>(__uint_as_float(acc[e / 32][e % 32]) - v.x, __uint_as_float(acc[e / 32][e % 32 + 1]) - v.y);
                    }
                    if (full) store_rows64(stage, &map_low, w, 64 * i, head, item.start + row - lane, lane);
                    else if (row < item.length) store_row64(static_cast<uint8_t*>(p.o_low) + (at + 64 * i) * 2, w);
                }
            }
            if (kKeep && row < item.length) p.lse[(size_t)head * p.rows + item.start + row] = m + __log2f(l);
        }
        if (lane == 0) store_done();
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <bool kBf16, int kDim, bool kKeep>
int launch_forward(PackedParams p, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mo,
                   const CUtensorMap& ml, cudaStream_t stream) {
    auto kernel = packed_forward_kernel<kBf16, kDim, kKeep>;
    constexpr int smem = fwd_smem<kDim>();
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return BSA_ERR_LAUNCH;
    // an upper bound of the tiles: every sequence and the rows behind the last one may end inside a tile
    const int per_tile = p.pair ? kRowsTile : 2 * kRowsTile;
    p.items = (p.rows / per_tile + p.batch + 1) * (p.pair ? p.q_heads / 2 : p.q_heads);
    kernel<<<p.items, kFwdThreads, smem, stream>>>(p, mq, mk, mv, mo, ml);
    return launch_status();
}

}  // namespace
}  // namespace bsa

extern "C" int bsa_packed_forward(int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                  int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                  int64_t v_head_stride, void* o, void* o_low, float* lse, const int32_t* offsets, int64_t rows,
                                  int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, float scale, int causal,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    using namespace bsa;
    int checked = check_packed(dtype, rows, batch, q_heads, kv_heads, head_dim);
    if (checked != BSA_OK) return checked;
    if (!workspace || workspace_bytes < BSA_WORKSPACE_BYTES) return BSA_ERR_WORKSPACE;
    if (rows == 0) return BSA_OK;
    if (!q || !k || !v || !o || !offsets || (lse != nullptr) != (o_low != nullptr)) return BSA_ERR_NULL_POINTER;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || (reinterpret_cast<uintptr_t>(o) & 31) || (reinterpret_cast<uintptr_t>(o_low) & 31)) return BSA_ERR_ALIGNMENT;
    if ((checked = check_strides(q_token_stride, q_head_stride)) != BSA_OK || (checked = check_strides(k_token_stride, k_head_stride)) != BSA_OK ||
        (checked = check_strides(v_token_stride, v_head_stride)) != BSA_OK) return checked;
    PackedParams p{};
    p.o = o; p.o_low = o_low; p.lse = lse; p.offsets = offsets;
    p.batch = (int)batch; p.rows = (int)rows; p.q_heads = (int)q_heads; p.kv_heads = (int)kv_heads;
    p.group = (int)(q_heads / kv_heads); p.causal = causal != 0;
    p.pair = p.group % 2 == 0;
    p.negative = scale < 0.0f;
    // a scale of 0 stays a factor that keeps masked scores at -infinity
    p.scale_log2 = fmaxf(fabsf(scale) * kPackedLog2e, 1e-37f);
    p.status = static_cast<uint32_t*>(workspace);
    CUtensorMap mq, mk, mv, mo, ml;
    if (!bind_device()) return BSA_ERR_LAUNCH;
    if (!make_packed_map(&mq, dtype, q, rows, q_heads, head_dim, q_token_stride, q_head_stride) ||
        !make_packed_map(&mk, dtype, k, rows, kv_heads, head_dim, k_token_stride, k_head_stride) ||
        !make_packed_map(&mv, dtype, v, rows, kv_heads, head_dim, v_token_stride, v_head_stride) ||
        !make_packed_map(&mo, dtype, o, rows, q_heads, head_dim, q_heads * head_dim, head_dim, 32) ||
        !make_packed_map(&ml, dtype, o_low ? o_low : o, rows, q_heads, head_dim, q_heads * head_dim, head_dim, 32)) return BSA_ERR_DRIVER;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const auto launch = [&](auto bf16, auto dim) {
        constexpr bool kBf16 = decltype(bf16)::value;
        constexpr int kDim = decltype(dim)::value;
        return lse ? launch_forward<kBf16, kDim, true>(p, mq, mk, mv, mo, ml, s) : launch_forward<kBf16, kDim, false>(p, mq, mk, mv, mo, ml, s);
    };
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (dtype == BSA_DTYPE_BF16) return head_dim == 64 ? launch(std::true_type{}, D64{}) : launch(std::true_type{}, D128{});
    return head_dim == 64 ? launch(std::false_type{}, D64{}) : launch(std::false_type{}, D128{});
}
