// Attention over a paged 16-bit cache for many query rows per key head (drafts x group above 32): the same sums as
// bsa_cached_attention.cu, on tcgen05.
//
// With that many rows the m16n8k16 kernel is bound by its own instructions (24 drafts x 4 heads over 46,000 tokens: 70 us,
// of which the cache's 94 MB take 14; here 40.5 us).  Here the rows of a key head, up to 128, are one M = 128
// tile; keys go in tiles of 128, and two streams of tiles, even and odd, each with its own scores, maximum, sum and O in TMEM, take turns on the
// tensor cores and in the softmax, as the two query tiles of the packed forward do; at the end the second hands its O to
// the first.  The units (tiles of a sequence, key head and row tile) are shared out evenly over the SMs as in the other
// kernel; a CTA that holds all of a sequence's tiles writes the output, the others leave (O, m, l) in fp32, columns by
// rows so that a warp writes whole lines, and a second kernel joins them in the order of the tiles.
//
//   warps 0-3, 4-7   softmax of the even / odd tiles of a share, one row per thread; 0-3 also bring the queries
//   warp 8           TMA producer: one lane per page and panel, K and V through rings of 3 stages
//   warp 9           MMA issuer
// All waits are bounded.
#include <algorithm>
#include <type_traits>

#include "bsa_cached_common.cuh"
#include "bsa_packed_common.cuh"

namespace bsa {
namespace {

constexpr int kWideBegin = 3;                   // what beginning and ending a (sequence, head) costs, in tiles
constexpr int kWideStages = 3;
constexpr int kWideThreads = 320;
constexpr int kJoinCols = 4;

struct __align__(16) WideBarriers {
    uint64_t q_full, q_empty, k_full[kWideStages], k_empty[kWideStages], v_full[kWideStages], v_empty[kWideStages];
    uint64_t s_full[2], p_full[2][2], o_full[2], drain;
    uint64_t m_full, m_empty;                   // half of the second stream's O (in the queries' place), handed to the first
    float2 ml[kRowsTile];                       // the second stream's (m, l)
    uint32_t ok[8];                             // by tile: bit i: page i of it was loaded
    Share share;
    uint32_t tmem_base;
    int abort_flag;
};
template <int kDim>
constexpr int wide_smem() { return (1 + 2 * kWideStages) * (kDim / 64) * kPanelBytes + (int)sizeof(WideBarriers); }

// The share of a CTA, segment by segment: tiles of one (sequence, head, row tile).
struct Walk {
    int64_t u, end;
    int b, hm, tile, hms, length, tiles;
    __device__ __forceinline__ Walk(const CachedParams& p, const Share& s) : u(s.first), end(s.end), b(s.b), hm(s.hm), tile(s.tile), hms(p.kv_heads * p.row_tiles), length(0), tiles(0) {
        if (u < end) enter(p);
    }
    __device__ __forceinline__ void enter(const CachedParams& p) {
        length = cached_length(p, b);
        tiles = max(1, (length + kRowsTile - 1) / kRowsTile);
    }
    __device__ __forceinline__ bool more() const { return u < end; }
    __device__ __forceinline__ int count() const { return (int)min((int64_t)(tiles - tile), end - u); }
    __device__ __forceinline__ void next(const CachedParams& p) {
        const int n = count();
        u += n;
        tile += n;
        if (tile == tiles) {
            tile = 0;
            u += kWideBegin;
            if (++hm == hms) {
                hm = 0;
                ++b;
                if (u < end) enter(p);
            }
        }
    }
};

template <bool kBf16, int kDim>
__global__ void __launch_bounds__(kWideThreads, 1)
cached_wide_kernel(const CachedParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   int negative, float scale_log2) {
    constexpr int kPanels = kDim / 64, kTile_ = kPanels * kPanelBytes;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* k_ring = smem + kTile_;
    uint8_t* v_ring = k_ring + kWideStages * kTile_;
    WideBarriers* bars = reinterpret_cast<WideBarriers*>(v_ring + kWideStages * kTile_);
    int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 8) {
        const Share mine = find_share<kRowsTile, kWideBegin>(p, (int)blockIdx.x, lane);
        if (lane == 0) bars->share = mine;
    }
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        mbar_init(&bars->q_full, 4); mbar_init(&bars->q_empty, 1);
        for (int i = 0; i < kWideStages; ++i) {
            mbar_init(&bars->k_full[i], 1); mbar_init(&bars->k_empty[i], 1);
            mbar_init(&bars->v_full[i], 1); mbar_init(&bars->v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars->s_full[i], 1); mbar_init(&bars->o_full[i], 1);
            mbar_init(&bars->p_full[i][0], 4); mbar_init(&bars->p_full[i][1], 4);
        }
        mbar_init(&bars->drain, 1);
        mbar_init(&bars->m_full, 4); mbar_init(&bars->m_empty, 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&bars->tmem_base;
    const int piece = min(1 << p.page_shift, kRowsTile), piece_shift = min(p.page_shift, 7), pieces = kRowsTile >> piece_shift;
    bool ok = true;
    Walk w(p, bars->share);
    int t = 0;                                  // tiles so far, of the whole share

    if (warp == 8) {
        // ------------------------------------------------------------ producer
        const int my_piece = lane & 7, my_panel = lane >> 3;
        for (; ok && w.more(); w.next(p)) {
            if (lane == 0 && p.lengths[w.b] != w.length) atomicExch(p.status, (uint32_t)BSA_ERR_BAD_SHAPE);
            const int head = w.hm / p.row_tiles, n = w.count();
            auto look = [&](int i) {                            // this lane's page of a tile, fetched a tile ahead
                const int key = (w.tile + i) * kRowsTile + my_piece * piece;
                return my_piece < pieces && i < n && key < w.length ? p.table[(int64_t)w.b * p.table_width + (key >> p.page_shift)] : 0;
            };
            int next = look(0);
            for (int i = 0; ok && i < n; ++i, ++t) {
                const int key = (w.tile + i) * kRowsTile + my_piece * piece, id = next;
                next = look(i + 1);
                bool there = my_piece < pieces && key < w.length;
                int row = 0;
                if (there) {
                    if ((uint32_t)id >= (uint32_t)p.pages) {
                        atomicExch(p.status, (uint32_t)BSA_ERR_BAD_SHAPE);
                        there = false;
                    } else {
                        row = ((id * p.kv_heads + head) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
                    }
                }
                const uint32_t loaded = __ballot_sync(0xffffffffu, there) & 255u;
                const int stage = t % kWideStages;
                const uint32_t parity = ((uint32_t)(t / kWideStages) & 1u) ^ 1u, bytes = (uint32_t)(__popc(loaded) * piece * kDim * 2);
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    uint64_t* full = side ? &bars->v_full[stage] : &bars->k_full[stage];
                    ok = ok && wait_all(side ? &bars->v_empty[stage] : &bars->k_empty[stage], parity, abort_flag, p.status);
                    if (!ok) break;
                    if (lane == 0) {
                        bars->ok[t & 7] = loaded;
                        mbar_expect_tx(full, bytes);
                    }
                    __syncwarp();
                    if (there && my_panel < kPanels)
                        tma_load_3d((side ? v_ring : k_ring) + stage * kTile_ + my_panel * kPanelBytes + my_piece * piece * 128,
                                    side ? &map_v : &map_k, full, 64 * my_panel, row, 0);
                    __syncwarp();
                }
            }
        }
        if (lane == 0 && *(volatile int*)abort_flag) let_copies_land();
        __syncwarp();
    } else if (warp == 9) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t fmt = kBf16 ? 1u : 0u;
        const uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRowsTile >> 4) << 24);
        const uint32_t idesc_s = common | ((uint32_t)(kRowsTile >> 3) << 17);
        const uint32_t idesc_o = common | (1u << 16) | ((uint32_t)(kDim >> 3) << 17);
        const uint64_t q_desc = panel_desc(smem_u32(smem), false);
        int segment = 0, p_no[2] = {0, 0};
        for (; ok && w.more(); w.next(p), ++segment) {
            const int n = w.count();
            auto scores = [&](int i) {
                const int no = t + i, stage = no % kWideStages, s = i & 1;
                ok = wait_all(&bars->k_full[stage], (uint32_t)(no / kWideStages) & 1u, abort_flag, p.status);
                if (!ok) return;
                tc_fence_after();
                if (elect_one()) {
                    mma_rows<kDim>(tmem + (uint32_t)(128 * s), q_desc, panel_desc(smem_u32(k_ring + stage * kTile_), false), idesc_s);
                    tc_commit(&bars->s_full[s]);
                    tc_commit(&bars->k_empty[stage]);
                    if (i == n - 1) tc_commit(&bars->q_empty);
                }
                __syncwarp();
            };
            ok = wait_all(&bars->q_full, (uint32_t)segment & 1u, abort_flag, p.status);
            if (ok) scores(0);
            if (ok && n > 1) scores(1);
            for (int i = 0; ok && i < n; ++i) {
                const int no = t + i, stage = no % kWideStages, s = i & 1;
                ok = wait_all(&bars->v_full[stage], (uint32_t)(no / kWideStages) & 1u, abort_flag, p.status);
                if (!ok) break;
                // V of keys that are not there: zero, for their weight is
                const int valid = w.length - (w.tile + i) * kRowsTile;
                const uint32_t loaded = bars->ok[no & 7];
                if (valid < kRowsTile || __popc(loaded) != pieces) {
                    uint8_t* v = v_ring + stage * kTile_;
                    for (int row = lane; row < kRowsTile; row += 32)
                        if (row >= valid || !(loaded >> (row >> piece_shift) & 1u))
#pragma unroll
                            for (int c = 0; c < kPanels * 8; ++c)
                                *reinterpret_cast<uint4*>(v + (c >> 3) * kPanelBytes + row * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    fence_async_shared();
                    __syncwarp();
                }
                const uint64_t v_desc = panel_desc(smem_u32(v_ring + stage * kTile_), true);
                const uint32_t s_tmem = tmem + (uint32_t)(128 * s), o_tmem = tmem + (uint32_t)(256 + s * kDim);
                ok = wait_all(&bars->p_full[s][0], (uint32_t)p_no[s] & 1u, abort_flag, p.status);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) mma_keys<0>(o_tmem, s_tmem, v_desc, idesc_o, i > 1);
                __syncwarp();
                ok = wait_all(&bars->p_full[s][1], (uint32_t)p_no[s]++ & 1u, abort_flag, p.status);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    mma_keys<1>(o_tmem, s_tmem, v_desc, idesc_o, true);
                    tc_commit(&bars->v_empty[stage]);
                    if (i + 2 >= n) tc_commit(&bars->o_full[s]);
                }
                __syncwarp();
                if (i + 2 < n) scores(i + 2);
            }
            t += n;
        }
        if (elect_one()) {
            tc_commit(&bars->drain);
            mbar_wait(&bars->drain, 0, abort_flag, p.status);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax of every second tile, one row per thread
        const int s = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_tmem = tmem + lanes + (uint32_t)(128 * s), o_tmem = tmem + lanes + (uint32_t)(256 + s * kDim);
        const float c = scale_log2;
        int s_no = 0, o_no = 0, segment = 0, m_no = 0;
        float* merge = reinterpret_cast<float*>(smem);          // [column of a half][row]
        for (; ok && w.more(); w.next(p), ++segment) {
            const int n = w.count(), head = w.hm / p.row_tiles, row = (w.hm - head * p.row_tiles) * kRowsTile + r;
            const int draft = row / p.group, count = p.counts ? min(max(p.counts[w.b], 0), p.drafts) : p.drafts;
            const int prefix = w.length - count;
            const bool row_on = draft < count;
            const uint64_t sees = !row_on ? 0ull : (p.tree ? (uint64_t)p.tree[(int64_t)w.b * p.drafts + draft] : ~0ull >> (63 - draft));
            if (s == 0) {                       // the queries, 16-byte chunks where the swizzle wants them
                const uint16_t* q = static_cast<const uint16_t*>(p.q) + (w.b * p.q_batch + draft * p.q_draft + (head * p.group + row - draft * p.group) * p.q_head);
                uint4 x[kDim / 8];
#pragma unroll
                for (int i = 0; i < kDim / 8; ++i) x[i] = row_on ? *reinterpret_cast<const uint4*>(q + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
                if (negative) {                 // a negative scale: the queries' signs
#pragma unroll
                    for (int i = 0; i < kDim / 8; ++i) x[i] = make_uint4(x[i].x ^ 0x80008000u, x[i].y ^ 0x80008000u, x[i].z ^ 0x80008000u, x[i].w ^ 0x80008000u);
                }
                // their place is free once the last scores are made, and all of this stream have read what the other left there
                ok = wait_all(&bars->q_empty, ((uint32_t)segment & 1u) ^ 1u, abort_flag, p.status) &&
                     wait_all(&bars->m_empty, ((uint32_t)m_no & 1u) ^ 1u, abort_flag, p.status);
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < kDim / 8; ++i)
                    *reinterpret_cast<uint4*>(smem + (i >> 3) * kPanelBytes + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = x[i];
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->q_full);
            }
            float m = -INFINITY, l = 0.0f;
            for (int i = s; i < n; i += 2) {
                ok = wait_all(&bars->s_full[s], (uint32_t)s_no++ & 1u, abort_flag, p.status);
                if (!ok) break;
                tc_fence_after();
                uint32_t x[4][32];
#pragma unroll
                for (int q = 0; q < 4; ++q) tc_ld_32x32b_x32(s_tmem + (uint32_t)(32 * q), x[q]);
                tc_wait_ld();
                const int key0 = (w.tile + i) * kRowsTile;
                const uint32_t loaded = bars->ok[(t + i) & 7];
                if (key0 + kRowsTile > prefix || __popc(loaded) != pieces) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {               // which of 32 keys the row sees, as bits
                        const int from = key0 + 32 * q, d = from - prefix;
                        uint32_t there = piece_shift >= 5 ? (loaded >> ((32 * q) >> piece_shift) & 1u ? 0xffffffffu : 0u)
                                                          : ((loaded >> (2 * q) & 1u ? 0xffffu : 0u) | (loaded >> (2 * q + 1) & 1u ? 0xffff0000u : 0u));
                        there &= below(w.length - from);
                        const uint32_t drafts = d >= 64 || d <= -32 ? 0u : (d >= 0 ? (uint32_t)(sees >> d) : (uint32_t)sees << -d);
                        const uint32_t seen = row_on ? there & (below(-d) | drafts) : 0u;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(seen >> e & 1u)) x[q][e] = 0xff800000u;
                    }
                }
                float top[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    top[q] = __uint_as_float(x[q][0]);
#pragma unroll
                    for (int e = 1; e < 31; e += 2) top[q] = fmax3(top[q], __uint_as_float(x[q][e]), __uint_as_float(x[q][e + 1]));
                    top[q] = fmaxf(top[q], __uint_as_float(x[q][31]));
                }
                const float mt = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
                if (__any_sync(0xffffffffu, mt > m + 8.0f)) {
                    const float higher = fmaxf(m, mt);
                    const float fall = higher == -INFINITY ? 1.0f : attn_exp2(m - higher);
                    m = higher;
                    l *= fall;
                    if (i > 1) {
#pragma unroll 1
                        for (int k = 0; k < kDim; k += 8) {
                            uint32_t acc[8];
                            tc_ld_32x32b_x8(o_tmem + (uint32_t)k, acc);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 8; ++e) acc[e] = __float_as_uint(__uint_as_float(acc[e]) * fall);
                            tc_st_32x32b_x8(o_tmem + (uint32_t)k, acc);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : -m;
                const uint64_t c2 = f2_pack(c, c), ref2 = f2_pack(ref, ref);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int q = 2 * half; q < 2 * half + 2; ++q)
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float a, b;
                            f2_unpack(f2_fma(f2_of(x[q][e], x[q][e + 1]), c2, ref2), a, b);
                            a = attn_exp2(a);
                            b = attn_exp2(b);
                            sum[(e / 2) & 1] = f2_add(sum[(e / 2) & 1], f2_pack(a, b));
                            x[half][(q & 1) * 16 + e / 2] = pack2<kBf16>(a, b);
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
            if (s >= n) { t += n; continue; }
            ok = wait_all(&bars->o_full[s], (uint32_t)o_no++ & 1u, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            constexpr int kHalf = kDim / 2;
            float mine = 1.0f, theirs = 0.0f;
            const bool whole = w.tile == 0 && n == w.tiles;
            bool any = false;
            const int64_t part = (int64_t)blockIdx.x * 2 + (w.tile == 0 ? 1 : 0);
            uint8_t* out = static_cast<uint8_t*>(p.o) +
                (((int64_t)w.b * p.drafts + draft) * (p.kv_heads * p.group) + head * p.group + row - draft * p.group) * kDim * 2;
            if (s == 1) bars->ml[r] = make_float2(m, l);
            // (short loops: this code runs once per segment, and unrolled its instructions took longer to fetch than to run)
#pragma unroll 1
            for (int h = 0; ok && h < 2; ++h) {
                const bool joined = n > 1;
                if (s == 1) ok = wait_all(&bars->m_empty, ((uint32_t)m_no++ & 1u) ^ 1u, abort_flag, p.status);
                else if (joined) ok = wait_all(&bars->m_full, (uint32_t)m_no++ & 1u, abort_flag, p.status);
                if (!ok) break;
                if (s == 0 && h == 0) {
                    if (joined) {
                        const float2 other = bars->ml[r];
                        const float higher = fmaxf(m, other.x), ref = higher == -INFINITY ? 0.0f : higher;
                        mine = attn_exp2(m - ref);
                        theirs = attn_exp2(other.x - ref);
                        m = higher;
                        l = l * mine + other.y * theirs;
                    }
                    any = row_on && l != 0.0f;                  // false: the row sees nothing, and is zero whatever V holds
                    if (whole) {
                        const float inv = any ? 1.0f / l : 0.0f;
                        mine *= inv;
                        theirs *= inv;
                    } else {
                        reinterpret_cast<float2*>(p.partial + (int64_t)p.ctas * 2 * kRowsTile * kDim)[part * kRowsTile + r] =
                            any ? make_float2(m, l) : make_float2(-INFINITY, 0.0f);
                    }
                }
#pragma unroll 1
                for (int at = 0; at < kHalf; at += 16) {
                    const int col = h * kHalf + at;
                    uint32_t acc[16];
                    tc_ld_32x32b_x16(o_tmem + (uint32_t)col, acc);
                    tc_wait_ld();
                    float* shared = merge + at * kRowsTile + r;
                    if (s == 1) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) shared[e * kRowsTile] = __uint_as_float(acc[e]);
                        continue;
                    }
                    float x[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {              // (a stream that saw nothing has weight 0, and may hold anything)
                        x[e] = mine != 0.0f ? __uint_as_float(acc[e]) * mine : 0.0f;
                        if (theirs != 0.0f) x[e] += shared[e * kRowsTile] * theirs;
                        if (!any) x[e] = 0.0f;
                    }
                    if (whole) {
                        uint32_t words[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) words[e] = pack2<kBf16>(x[2 * e], x[2 * e + 1]);
                        if (draft < p.drafts) st_global_v8(out + col * 2, words);
                    } else {
                        float* to = p.partial + part * (kRowsTile * kDim) + col * kRowsTile + r;
#pragma unroll
                        for (int e = 0; e < 16; ++e) to[e * kRowsTile] = x[e];
                    }
                }
                __syncwarp();
                if (lane == 0 && joined) mbar_arrive(s == 1 ? &bars->m_full : &bars->m_empty);
            }
            if (!ok) break;
            t += n;
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Joins the parts of one (sequence, key head, row tile), kCols columns: one row per thread, many small CTAs whose loads
// travel together.
template <typename T, int kDim>
__global__ void __launch_bounds__(kRowsTile) cached_wide_join_kernel(const CachedParams p) {
    constexpr int kCols = kJoinCols;
    const int lane = threadIdx.x & 31, r = threadIdx.x, hms = p.kv_heads * p.row_tiles;
    const int item = blockIdx.x / (kDim / kCols), col0 = (blockIdx.x - item * (kDim / kCols)) * kCols;
    const int b = item / hms, hm = item - b * hms, head = hm / p.row_tiles;
    const int row = (hm - head * p.row_tiles) * kRowsTile + r, draft = row / p.group;
    int64_t before;
    const int64_t per = quotient(total_cost<kRowsTile, kWideBegin>(p, b, before, lane) * hms + p.ctas - 1, p.ctas);
    const int tiles = cached_tiles<kRowsTile>(p, b);
    const int64_t start = before * hms + (int64_t)hm * (tiles + kWideBegin) + kWideBegin, end = start + tiles;
    const int first = (int)quotient(start, per), last = (int)quotient(end - 1, per);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (draft >= p.drafts || first == last) return;         // one CTA had all of it and wrote the output
    const float2* ml = reinterpret_cast<const float2*>(p.partial + (int64_t)p.ctas * 2 * kRowsTile * kDim);
    constexpr int kBatch = 8;
    float sum[kCols], l = 0.0f, top = -INFINITY;
#pragma unroll
    for (int e = 0; e < kCols; ++e) sum[e] = 0.0f;
    for (int i0 = first; i0 <= last; i0 += kBatch) {
        float2 w[kBatch];
        float x[kBatch][kCols];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = min(i0 + k, last);
            const int64_t part = (int64_t)i * 2 + (i == first);
            w[k] = ml[part * kRowsTile + r];
            if (i0 + k > last) w[k] = make_float2(-INFINITY, 0.0f);
            const float* from = p.partial + part * (kRowsTile * kDim) + col0 * kRowsTile + r;       // (zeros where it saw nothing)
#pragma unroll
            for (int e = 0; e < kCols; ++e) x[k][e] = from[e * kRowsTile];
        }
        float higher = top;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) higher = fmaxf(higher, w[k].x);
        const float ref = higher == -INFINITY ? 0.0f : higher, fall = attn_exp2(top - ref);
        top = higher;
        l *= fall;
#pragma unroll
        for (int e = 0; e < kCols; ++e) sum[e] *= fall;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float weight = attn_exp2(w[k].x - ref);
            l += w[k].y * weight;
#pragma unroll
            for (int e = 0; e < kCols; ++e) sum[e] += x[k][e] * weight;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    __align__(8) T out[kCols];
#pragma unroll
    for (int e = 0; e < kCols; ++e) out[e] = Scalar<T>::from_float(sum[e] * inv);
    T* to = static_cast<T*>(p.o) + (((int64_t)b * p.drafts + draft) * (p.kv_heads * p.group) + head * p.group + (row - draft * p.group)) * kDim + col0;
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(out);
}

template <bool kBf16, int kDim>
int launch_wide(const CachedParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t stream) {
    using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
    auto kernel = cached_wide_kernel<kBf16, kDim>;
    constexpr int smem = wide_smem<kDim>();
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return BSA_ERR_LAUNCH;
    // a scale of 0 stays a factor that keeps masked scores at -infinity
    kernel<<<p.ctas, kWideThreads, smem, stream>>>(p, map_k, map_v, p.scale_log2 < 0.0f, fmaxf(fabsf(p.scale_log2), 1e-37f));
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(p.batch * p.kv_heads * p.row_tiles * (kDim / kJoinCols)));
    config.blockDim = dim3(kRowsTile);
    config.stream = stream;
    cudaLaunchAttribute overlap{};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &overlap;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, cached_wide_join_kernel<T, kDim>, p) != cudaSuccess) { cudaGetLastError(); return BSA_ERR_LAUNCH; }
    return launch_status();
}

}  // namespace

size_t cached_wide_scratch(int64_t head_dim) {
    return (size_t)std::max(sm_count(), 1) * 2 * kRowsTile * (size_t)(head_dim + 2) * 4;
}

int cached_wide(const CachedParams& given, int dtype, int64_t head_dim, const void* keys, const void* values, int64_t page,
                cudaStream_t stream) {
    CachedParams p = given;
    p.row_tiles = (p.drafts * p.group + kRowsTile - 1) / kRowsTile;
    p.ctas = sm_count();
    if (p.ctas <= 0) return BSA_ERR_LAUNCH;
    if ((int64_t)p.row_tiles * p.kv_heads > (int64_t)INT32_MAX / p.batch / 32) return BSA_ERR_TOO_LARGE;
    CUtensorMap map_k, map_v;
    const int64_t rows = (int64_t)p.pages * p.kv_heads * page;
    const int piece = (int)std::min<int64_t>(page, kRowsTile);
    if (!make_cache_map(&map_k, BSA_CACHE_SAME, dtype, keys, rows, head_dim, piece) ||
        !make_cache_map(&map_v, BSA_CACHE_SAME, dtype, values, rows, head_dim, piece)) return BSA_ERR_DRIVER;
    if (dtype == BSA_DTYPE_BF16)
        return head_dim == 64 ? launch_wide<true, 64>(p, map_k, map_v, stream) : launch_wide<true, 128>(p, map_k, map_v, stream);
    return head_dim == 64 ? launch_wide<false, 64>(p, map_k, map_v, stream) : launch_wide<false, 128>(p, map_k, map_v, stream);
}

}  // namespace bsa
