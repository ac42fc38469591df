// Attention of drafted tokens over a paged key / value cache (sm_100a only):
//   o_i = sum_j p_ij v_j,   p_ij = exp(scale q_i k_j - lse_i)   over the keys j that draft i sees:
// every cached token before the sequence's drafts, and among the drafts those whose bit is set in word i of `tree`
// (none given: the drafts up to i itself).  A block layout, where given, takes away the keys of the blocks it lacks.
//
// One token of a sequence is a handful of query rows (drafts x the heads that share a key head), so the work is the
// cache read once: bound by DRAM from a few thousand cached tokens on, below that by the two launches.
//
// Split.  The unit is a tile of 64 keys of one (sequence, key head, row tile), and each of those begins with kBegin empty
// units for what its first and last steps cost; the units of the whole batch are one list, and 2 x #SM persistent CTAs
// take equal contiguous shares of it, whatever the lengths are: nothing about the lengths is known on the host.  A CTA that holds all tiles of a (sequence, head) writes its output; the others leave (O, m, l) in
// fp32, at most two per CTA, and a second small kernel joins them in the order of the tiles (no atomics: the result does
// not depend on timing).
//
// A CTA is a producer warp (TMA boxes of the pages, swizzled, into a ring of stages; one lane per page of the tile) and
// four warps that each take 16 * G of the 64 keys for 16 of the 16 * G rows (G = 1, 2, 4 row groups): with few rows every
// stored byte is read from shared memory once.  Products are m16n8k16 with the operands where ldmatrix leaves them:
// at these row counts the tensor pipe idles either way, and a 128-row tcgen05 tile would be 7/8 padding.
//
// e4m3 caches.  Codes are exact in fp16, so the products run in fp16 on the codes themselves and the scales go where they
// are cheap: the key's into the score, the value's into the weight: P_ij = 2^(s_ij - m_i) as ever, l += P_ij, and
// O += (P_ij sv_j / r) code.  r is a power of two per warp, raised lazily to the power of two under the largest finite |sv|
// of the keys so far (as m is), so the weights stay below 2^8 x 16; O r is what goes out, so nothing outside the loop
// knows of r.  l never sees a value's scale: a scale may be 0, negative, or 2^-109 (a row of zeros) beside 2^119.  A
// weight below 2^-14 of r is rounded to steps of 2^-24 of it, so a row's error is relative to the largest stored values
// of its sequence, as it is where fp16 holds the values themselves.  bf16 queries are brought to fp16 by a power of two
// per row (exact but for values below 2^-14 of the row's largest).  The 8-bit elements are paired by ldmatrix as 16-bit
// units, which permutes the contraction axis of Q K^T (the query is loaded in the same order) and the columns of O
// (undone at the store).
//
// The weights are rounded to the products' 16-bit type (half a step: relative 2^-8 in bf16, 2^-11 in fp16), l, m and O are
// fp32.
//
// 32 sequences of 1 to 8192 tokens, 8 heads x 128, e4m3 (94 MB): 32.8 us, 2.9 TB/s; bound by the latency of a warp's
// step of 32 keys (2100 cycles with 2 consumer warps per scheduler) and what begins a share (2,800 cycles) and ends it
// (2,200 to 5,400).  One token over 391: 10.3 us a call, 9.2 in a graph.
//
// A layout takes keys away from the softmax, not from the work: every page is brought and multiplied all the same, and a
// step looks its blocks up besides.  One sequence of 32,768 tokens, 4 heads x 128, whose last row keeps 5 of 512 blocks,
// 16 bits: one token 38.9 us with and without; 16 tokens of 16 query heads 65.4 us here, 38.9 without it in the kernel for
// many rows, which takes no layout; e4m3 36.9 and 32.8, 67.6 and 53.2.
#include <algorithm>
#include <type_traits>

#include "bsa_cached_common.cuh"

namespace bsa {
namespace {

constexpr int kTileKeys = 64;
constexpr int kConsumers = 4;                   // warps
constexpr int kBegin = 6;                       // what beginning and ending a (sequence, head) costs a CTA, in tiles.  Found on one
                                                // batch (32 of 1 to 8192 tokens, e4m3: with 3 37.1 us, 5 32.5, 6 32.8, 7 32.9,
                                                // 10 34.8) and used for every type; one token of one sequence does not feel it
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kExponent = 1u << 23;        // one step of an fp32 number's exponent
// Query rows of a key head above which a 16-bit cache goes to the tcgen05 kernel.  8 x 4000 tokens of 4 heads x 128: 32 rows
// 26.7 us here, 30.0 us there; 40 rows 38.8 and 30.7, 128 rows 56.3 and 34.8.  16 x 300 tokens: 16.4 and 18.4; 20.5 and 18.4.
constexpr int64_t kWideRows = 32;

// Barriers go by the number of the tile, modulo kBars, and so belong to one stream of tiles each: a warp that skips the
// other stream's tiles sees every phase of the barriers that it waits for.  (With a barrier per stage and an odd number of
// stages it saw every second one, and could take a phase that had not begun for the one before it.)
template <int kBars>
struct __align__(8) CachedBarriers {
    uint64_t full[kBars], empty[kBars];
    uint32_t ok[kBars];             // bit i: page i of the tile was loaded
    Share share;
    int abort_flag;
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (kBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four e4m3 codes as fp16 values: codes 0, 1 and codes 2, 3.
__device__ __forceinline__ void halves4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(codes));
}

template <bool kE4m3, int kDim, int kGroups>
struct CachedShape {
    static constexpr int kRowBytes = kDim * (kE4m3 ? 1 : 2);
    static constexpr int kPanelBytes = kRowBytes < 128 ? kRowBytes : 128;       // width of a TMA box
    static constexpr int kPanels = kRowBytes / kPanelBytes;
    static constexpr int kSideBytes = kTileKeys * kRowBytes;
    static constexpr int kScaleBytes = kE4m3 ? 2 * kTileKeys * 4 : 0;
    static constexpr int kStageBytes = 2 * kSideBytes;
    static constexpr int kStages = kStageBytes >= 32768 ? 3 : (kStageBytes >= 16384 ? 5 : 8);
    static constexpr int kStreams = kGroups == 1 ? 2 : 1;       // of tiles, see the kernel
    static constexpr int kBars = kStages * (kStages % kStreams == 0 ? 1 : kStreams);
    // columns of O that the warps of a row group join at a time (the 8-bit layout stores pairs of 8-column tiles)
    static constexpr int kJoin = kE4m3 ? 64 : 32;
    static constexpr int kJoinFloats = kGroups == 4 ? 0 : kConsumers * 16 * (kJoin + 2);
    static constexpr int kRows = 16 * kGroups;
    static constexpr int kQueryBytes = kRows * (kDim * 2 + 4);                  // fragments, and a factor per row
    static constexpr int kKeyBytes = kE4m3 ? kConsumers * 32 * 8 : 0;           // the scales of the warps' keys, the value's over r
    static constexpr int kSmem = kStages * (kStageBytes + kScaleBytes) + kKeyBytes + kQueryBytes + kJoinFloats * 4 + (int)sizeof(CachedBarriers<kBars>);
    static_assert(2 * (kSmem + 1024) <= 233472, "two CTAs per SM");
};

// Where the TMA swizzle leaves 16-byte chunk `chunk` of row `row` (of 8 or 16 rows that start on a multiple of 8).
template <int kPanelBytes>
__device__ __forceinline__ uint32_t chunk_offset(int row, int chunk) {
    if (kPanelBytes == 128)
        return (uint32_t)((chunk >> 3) * (kTileKeys * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
    return (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
}

// How many other drafts a draft sees (its own bit may be set or not).
__device__ __forceinline__ int ancestors(uint64_t word, int draft) { return __popcll(word & ~(1ull << draft)); }

// Of 32 keys from key0 on, those (of `wanted`) whose block is in the layout, seen from block row `row`.  Whole blocks before
// the drafts are one lookup per 16 keys; a draft stands behind the prefix and its ancestors.
// (`at`: the row of the pattern; `tree`: the sequence's words, or null)
__device__ __noinline__ uint32_t in_pattern(const uint8_t* at, int cols, int shift, const int64_t* tree, int key0, int prefix, uint32_t wanted) {
    uint32_t bits = 0u;
#pragma unroll 1
    for (int k = 0; k < 32; ++k) {
        const int key = key0 + k, draft = key - prefix;
        if ((k & 15) == 0 && key + 16 <= prefix) {
            const int block = key >> shift;
            if (block < cols && at[block]) bits |= 0xffffu << k;
            k += 15;
            continue;
        }
        if (!(wanted >> k & 1u)) continue;
        int place = key;
        if (draft >= 0) {
            const uint64_t w = tree ? (uint64_t)tree[draft] : ~0ull >> (63 - draft);
            place = max(prefix, 0) + ancestors(w, draft);
        }
        const int block = place >> shift;
        if (block < cols && at[block]) bits |= 1u << k;
    }
    return bits;
}

// T: type of q and o; kGroups: groups of 16 rows (1, 2 or 4).
template <typename T, bool kE4m3, int kDim, int kGroups>
__global__ void __launch_bounds__((kConsumers + 1) * 32, 2)
cached_attention_kernel(const CachedParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using S = CachedShape<kE4m3, kDim, kGroups>;
    using Bars = CachedBarriers<S::kBars>;
    constexpr bool kTBf16 = std::is_same_v<T, __nv_bfloat16>;
    constexpr bool kBf16 = !kE4m3 && kTBf16;                // type of the products
    constexpr int kRows = 16 * kGroups;
    constexpr int kSplit = kConsumers / kGroups;            // warps that share a row group
    // With one row group the warps work as two pairs on alternate tiles, 32 keys each: 16 keys per warp and tile leave
    // too few independent instructions between the tile's barriers.
    constexpr int kStreams = S::kStreams;
    constexpr int kWarpKeys = kTileKeys * kStreams / kSplit;            // keys of a tile per warp
    constexpr int kStepKeys = 32;                           // keys of a step of the warp (registers)
    constexpr int kNT = kStepKeys / 8;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* scale_smem = smem + S::kStages * S::kStageBytes;
    float* key_smem = reinterpret_cast<float*>(scale_smem + S::kStages * S::kScaleBytes);
    uint32_t* q_smem = reinterpret_cast<uint32_t*>(scale_smem + S::kStages * S::kScaleBytes + S::kKeyBytes);     // [row group][k step][lane][4]
    float* q_factor = reinterpret_cast<float*>(q_smem + kRows * kDim / 2);
    float* merge = q_factor + kRows;
    Bars* bars = reinterpret_cast<Bars*>(merge + S::kJoinFloats);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        const Share mine = find_share<kTileKeys, kBegin>(p, (int)blockIdx.x, lane);
        if (lane == 0) bars->share = mine;
    } else if (warp == kConsumers && lane == 0) {
        bars->abort_flag = 0;
        for (int i = 0; i < S::kBars; ++i) {
            mbar_init(&bars->full[i], 1);
            mbar_init(&bars->empty[i], kConsumers / kStreams);
        }
        fence_async_shared();
    }
    __syncthreads();
    const Share share = bars->share;
    int b = share.b, hm = share.hm, tile = share.tile;
    const int hms = p.kv_heads * p.row_tiles;
    uint32_t turn = 0;                                      // tiles so far

    if (warp == kConsumers) {                               // ---- producer
        // One lane per copy of a tile, so that all leave with one instruction: pages (at most 4) x sides x panels of the
        // keys and values in lanes 0-15, pages x sides of the scales in lanes 16-23.  (Issued one after another by the
        // pages' lanes they took longer than the tile's arithmetic: 49 against 43 us.)
        const int page = 1 << p.page_shift, piece = min(page, kTileKeys), pieces = kTileKeys / piece;
        const int my_piece = lane & 3, my_side = (lane >> 2) & 1, my_panel = (lane >> 3) & 1;
        const bool my_scale = kE4m3 && lane >= 16 && lane < 24, my_tile = lane < 8 * S::kPanels;
        const CUtensorMap* my_map = my_side == 0 ? &map_k : &map_v;
        bool dead = false;
        int64_t u = share.first;
        int length = 0, tiles = 0, id = 0;
        auto enter = [&]() {                                // a new sequence
            length = cached_length(p, b);
            tiles = max(1, (length + kTileKeys - 1) / kTileKeys);
            if (lane == 0 && p.lengths[b] != length) atomicExch(p.status, (uint32_t)BSA_ERR_BAD_SHAPE);
        };
        auto look = [&]() {                                 // this lane's page of the tile
            const int key = tile * kTileKeys + my_piece * piece;
            id = 0;
            if (my_piece < pieces && key < length) id = p.table[(int64_t)b * p.table_width + (key >> p.page_shift)];
        };
        if (u < share.end) { enter(); look(); }
        while (u < share.end) {
            const int head = hm / p.row_tiles;
            const int key = tile * kTileKeys + my_piece * piece;
            bool ok = my_piece < pieces && key < length;
            if (ok && (uint32_t)id >= (uint32_t)p.pages) {  // not a page of this cache: its keys are left out, and reported
                atomicExch(p.status, (uint32_t)BSA_ERR_BAD_SHAPE);
                ok = false;
            }
            const int row = ok ? ((id * p.kv_heads + head) << p.page_shift) + (key & (page - 1)) : 0;
            // on to the next tile: its page numbers travel while this one waits for its stage
            ++u;
            if (++tile == tiles) {
                tile = 0;
                u += kBegin;
                if (++hm == hms) {
                    hm = 0;
                    ++b;
                    if (u < share.end) enter();
                }
            }
            if (u < share.end) look();
            const uint32_t loaded = __ballot_sync(0xffffffffu, ok) & 15u;
            const uint32_t stage = turn % S::kStages, bar = turn % S::kBars;
            if (turn >= (uint32_t)S::kStages) {             // the stage's last tile has been read
                const uint32_t last = turn - S::kStages;
                dead = !mbar_wait(&bars->empty[last % S::kBars], last / S::kBars & 1u, &bars->abort_flag, p.status);
            }
            if (dead) break;
            if (lane == 0) {
                bars->ok[bar] = loaded;
                mbar_expect_tx(&bars->full[bar], (uint32_t)(__popc(loaded) * piece * (2 * S::kRowBytes + (kE4m3 ? 8 : 0))));
            }
            __syncwarp();
            if (ok && my_tile)
                tma_load_3d(smem + stage * S::kStageBytes + my_side * S::kSideBytes + my_panel * (kTileKeys * S::kPanelBytes) +
                            my_piece * piece * S::kPanelBytes, my_map, &bars->full[bar],
                            my_panel * (S::kPanelBytes / (kE4m3 ? 1 : 2)), row, 0);
            if (ok && my_scale)
                bulk_load_1d(scale_smem + stage * S::kScaleBytes + my_side * (kTileKeys * 4) + my_piece * piece * 4,
                             p.scales[my_side] + row, (uint32_t)(piece * 4), &bars->full[bar]);
            __syncwarp();
            ++turn;
        }
        if (dead) let_copies_land();
        return;
    }

    // ---- consumers
    const int rg = warp / kSplit, part = warp % kSplit;     // row group; number among its warps
    const int stream = part % kStreams, first_key = part / kStreams * kWarpKeys;        // which tiles, which keys of them
    const int g = lane >> 2, c = lane & 3;
    // addresses of this lane's ldmatrix rows inside 8 keys (K) and 16 keys (V)
    uint32_t k_lane[S::kRowBytes / 64];
#pragma unroll
    for (int x = 0; x < S::kRowBytes / 64; ++x) k_lane[x] = chunk_offset<S::kPanelBytes>(lane & 7, 4 * x + (lane >> 3));
    const uint32_t v_lane = chunk_offset<S::kPanelBytes>(lane & 15, lane >> 4);
    bool dead = false;
    int64_t u = share.first;
    // The queries of the next (sequence, head, row tile) are fetched before the one at hand is joined and stored, so that
    // they travel meanwhile; they go to shared memory in the order of the fragments.
    constexpr int kChunks = kDim / 8, kLoads = (kRows * kChunks + kConsumers * 32 - 1) / (kConsumers * 32);
    int at_b = -1, length = 0, tiles = 0, count = 0;
    uint64_t sees[2];                                       // of this thread's two rows: the drafts that it sees,
    int row_block[2];                                       // its block row in the pattern,
    bool row_on[2];                                         // and whether it is one of the sequence's drafts
    uint4 fetched[kLoads];
    auto fetch = [&]() {
        if (b != at_b) {
            at_b = b;
            length = cached_length(p, b);
            count = p.counts ? min(max(p.counts[b], 0), p.drafts) : p.drafts;
            tiles = max(1, (length + kTileKeys - 1) / kTileKeys);
        }
        const int head = hm / p.row_tiles, row_tile = hm - head * p.row_tiles;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int chunk = (int)threadIdx.x + i * kConsumers * 32;
            const int row = row_tile * kRows + chunk / kChunks, draft = row / p.group, h = head * p.group + row - draft * p.group;
            fetched[i] = make_uint4(0u, 0u, 0u, 0u);
            if (chunk < kRows * kChunks && draft < count)   // (drafts behind the sequence's own are zeros, and masked)
                fetched[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.q_batch + draft * p.q_draft + h * p.q_head + chunk % kChunks * 8);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int draft = (row_tile * kRows + rg * 16 + g + 8 * r) / p.group;
            row_on[r] = draft < count;
            sees[r] = 0;
            row_block[r] = -1;
            if (row_on[r]) {
                sees[r] = p.tree ? (uint64_t)p.tree[(int64_t)b * p.drafts + draft] : ~0ull >> (63 - draft);
                // a draft stands behind the prefix and its ancestors
                if (p.pattern) row_block[r] = (max(length - count, 0) + ancestors(sees[r], draft)) >> p.pattern_shift;
            }
        }
    };
    auto put = [&]() {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int chunk = (int)threadIdx.x + i * kConsumers * 32, row = chunk / kChunks, at = chunk % kChunks;
            uint32_t w[4] = {fetched[i].x, fetched[i].y, fetched[i].z, fetched[i].w};
            if (kE4m3 && kTBf16) {                          // bf16 queries to fp16 by a power of two per row
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7fff0000u, w[e] << 16 & 0x7fff0000u));
#pragma unroll
                for (int d = kChunks / 2; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
                const int e = min(max((int)(top >> 23), 1), 253);                // biased exponent of the row's largest
                const float down = __uint_as_float((uint32_t)(254 - e) << 23);    // 2^-(e - 127)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    w[x] = pack2<false>(__uint_as_float(w[x] << 16) * down, __uint_as_float(w[x] & 0xffff0000u) * down);
                if (at == 0 && row < kRows) q_factor[row] = p.scale_log2 * __uint_as_float((uint32_t)e << 23);
            }
            if (row < kRows) {
                // k step at / 2; the fragment of lane 4 (row % 8) + c holds the words (row, row + 8) x (first, second pair)
                uint32_t* to = q_smem + (((row / 16) * (kDim / 16) + at / 2) * 32 + (row & 7) * 4) * 4 + ((row >> 3) & 1);
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    to[kE4m3 ? (2 * (at & 1) + x / 2) * 4 + 2 * (x & 1) : x * 4 + 2 * (at & 1)] = w[x];
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
    };
    if (u < share.end) fetch();
    while (u < share.end) {
        put();
        const int prefix = length - count;                  // negative where a sequence has fewer tokens than drafts
        const int todo = (int)min((int64_t)(tiles - tile), share.end - u);
        const bool from_start = tile == 0, whole = from_start && todo == tiles;
        const uint4* q_frag = reinterpret_cast<const uint4*>(q_smem) + rg * (kDim / 16) * 32 + lane;
        const float row_scale[2] = {kE4m3 && kTBf16 ? q_factor[rg * 16 + g] : p.scale_log2, kE4m3 && kTBf16 ? q_factor[rg * 16 + g + 8] : p.scale_log2};

        float out[kDim / 8][4];
#pragma unroll
        for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) out[i][e] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        uint32_t r_bits = kExponent;                        // e4m3: r, a power of two from 2^-126 to 2^126; O is in units of it

        for (int i = 0; i < todo; ++i, ++tile, ++turn) {
            if (kStreams == 2 && (int)(turn & 1) != stream) continue;
            const uint32_t stage = turn % S::kStages, bar = turn % S::kBars;
            if (!dead) dead = !mbar_wait(&bars->full[bar], turn / S::kBars & 1u, &bars->abort_flag, p.status);
            const uint32_t k_base = smem_u32(smem) + stage * S::kStageBytes, v_base = k_base + S::kSideBytes;
            const uint32_t loaded = bars->ok[bar];
#pragma unroll 1
            for (int base = first_key; base < first_key + kWarpKeys; base += kStepKeys) {
            const int key0 = tile * kTileKeys + base, tile_end = (tile + 1) * kTileKeys;
            const bool all_loaded = loaded == (1u << (kTileKeys >> min(p.page_shift, 6))) - 1u;
            const bool masked = tile_end > prefix || !all_loaded || p.pattern != nullptr;
            // The step's 32 keys as bits: what each of the two rows sees, and what any row of the warp does: the other keys may
            // hold anything.  (Written out per element this was most of the kernel's code, and a short sequence, all of whose
            // steps are masked, waited for it to be fetched.)
            uint32_t seen[2] = {0xffffffffu, 0xffffffffu}, used = 0xffffffffu;
            if (masked) {
                const int shift = min(p.page_shift, 6), d = key0 - prefix;
                uint32_t there = shift >= 5 ? (loaded >> (base >> shift) & 1u ? 0xffffffffu : 0u)
                                            : ((loaded >> (base >> 4) & 1u ? 0xffffu : 0u) | (loaded >> ((base >> 4) + 1) & 1u ? 0xffff0000u : 0u));
                there &= below(length - key0);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t drafts = d >= 64 || d <= -32 ? 0u : (d >= 0 ? (uint32_t)(sees[r] >> d) : (uint32_t)sees[r] << -d);
                    seen[r] = row_on[r] ? there & (below(-d) | drafts) : 0u;
                    if (p.pattern)
                        seen[r] = row_block[r] < 0 || row_block[r] >= p.pattern_rows ? 0u :
                            seen[r] & in_pattern(p.pattern + (int64_t)row_block[r] * p.pattern_cols, p.pattern_cols, p.pattern_shift,
                                                 p.tree ? p.tree + (int64_t)b * p.drafts : nullptr, key0, prefix, seen[r]);
                }
                __syncwarp();
                used = __reduce_or_sync(0xffffffffu, seen[0] | seen[1]);
            }
            // e4m3: a lane brings the scales of one key, the warp shares them (the key's, and the value's over r)
            if (kE4m3) {
                const float* scales = reinterpret_cast<const float*>(scale_smem + stage * S::kScaleBytes) + base + lane;
                const float sv = used >> lane & 1u ? scales[kTileKeys] : 0.0f;
                const uint32_t size = __float_as_uint(sv) & 0x7fffffffu;
                const bool finite = size < 0x7f800000u;
                if (__any_sync(0xffffffffu, finite && size >= r_bits + 4 * kExponent)) {
                    const uint32_t top = min(__reduce_max_sync(0xffffffffu, finite ? size : 0u) & 0x7f800000u, 253 * kExponent);
                    // 2^-(steps of the exponent), 0 where that is no normal number (of O nothing is left beside the new r)
                    const uint32_t steps = top - r_bits;
                    const float fall = __uint_as_float(127 * kExponent - min(steps, 127 * kExponent));
                    r_bits = top;
#pragma unroll
                    for (int d = 0; d < kDim / 8; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) out[d][e] *= fall;
                }
                __syncwarp();                               // the last step's have been read
                key_smem[warp * 64 + lane] = scales[0];
                key_smem[warp * 64 + 32 + lane] = sv * __uint_as_float(254 * kExponent - r_bits);
                __syncwarp();
            }
            float s[kNT][4];
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
            // Q K^T
            const uint32_t rows8 = k_base + (uint32_t)(base * S::kPanelBytes);
#pragma unroll
            for (int x = 0; x < S::kRowBytes / 64; ++x) {
                constexpr int kSteps = kE4m3 ? 4 : 2;       // k steps of 64 bytes of a key
                uint32_t qf[kSteps][4];
#pragma unroll
                for (int e = 0; e < kSteps; ++e) {
                    const uint4 w = q_frag[(kSteps * x + e) * 32];
                    qf[e][0] = w.x; qf[e][1] = w.y; qf[e][2] = w.z; qf[e][3] = w.w;
                }
#pragma unroll
                for (int n = 0; n < kNT; ++n) {
                    uint32_t kf[4];
                    ldsm_x4(rows8 + (uint32_t)(n * 8 * S::kPanelBytes) + k_lane[x], kf);
                    if (!kE4m3) {
                        mma_16816<kBf16>(s[n], qf[0], kf[0], kf[1]);
                        mma_16816<kBf16>(s[n], qf[kSteps / 2], kf[2], kf[3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < kSteps; ++e) {
                            uint32_t b0, b1;
                            halves4(kf[e], b0, b1);
                            mma_16816<false>(s[n], qf[e], b0, b1);
                        }
                    }
                }
            }
            // scores in units of log2
#pragma unroll
            for (int n = 0; n < kNT; ++n) {
                if (kE4m3) {
                    const float2 both = *reinterpret_cast<const float2*>(key_smem + warp * 64 + n * 8 + 2 * c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = s[n][e] * ((e & 1) ? both.y : both.x) * row_scale[e >> 1];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] *= row_scale[e >> 1];
                }
            }
            uint32_t keep[kNT];                             // per n-tile: which of this thread's two keys are used
            if (masked) {
#pragma unroll
                for (int n = 0; n < kNT; ++n) {
                    const int at = 8 * n + 2 * c;
                    keep[n] = (used >> at & 1u ? 0x0000ffffu : 0u) | (used >> (at + 1) & 1u ? 0xffff0000u : 0u);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(seen[e >> 1] >> (at + (e & 1)) & 1u)) s[n][e] = -INFINITY;
                }
            }
            // The running maximum is raised only where a score exceeds it by more than 8 (units of log2): P stays below
            // 2^8, and O and l carry the same factor whatever it is.
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
            float ref[2];
            if (__any_sync(0xffffffffu, top[0] > m[0] + 8.0f || top[1] > m[1] + 8.0f)) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                    const float higher = fmaxf(m[r], top[r]);
                    const float fall = higher == -INFINITY ? 1.0f : attn_exp2(m[r] - higher);
                    m[r] = higher;
                    l[r] *= fall;
#pragma unroll
                    for (int d = 0; d < kDim / 8; ++d) {
                        out[d][2 * r] *= fall;
                        out[d][2 * r + 1] *= fall;
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) ref[r] = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
            for (int n = 0; n < kNT; ++n) {
                const float2 over = kE4m3 ? *reinterpret_cast<const float2*>(key_smem + warp * 64 + 32 + n * 8 + 2 * c) : make_float2(1.0f, 1.0f);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][e] = attn_exp2(s[n][e] - ref[e >> 1]);
                    l[e >> 1] += s[n][e];
                    if (kE4m3) s[n][e] *= (e & 1) ? over.y : over.x;
                }
            }
            // P V
#pragma unroll
            for (int ks = 0; ks < kStepKeys / 16; ++ks) {
                const uint32_t pf[4] = {pack2<kBf16>(s[2 * ks][0], s[2 * ks][1]), pack2<kBf16>(s[2 * ks][2], s[2 * ks][3]),
                                        pack2<kBf16>(s[2 * ks + 1][0], s[2 * ks + 1][1]), pack2<kBf16>(s[2 * ks + 1][2], s[2 * ks + 1][3])};
                // lanes 0-7: keys 0-7 of the step, chunk a; 8-15: keys 8-15, chunk a; 16-31: the same of chunk a + 1
                const uint32_t rows16 = v_base + (uint32_t)((base + ks * 16) * S::kPanelBytes) + v_lane;
#pragma unroll
                for (int a = 0; a < S::kRowBytes / 16; a += 2) {
                    uint32_t vf[4];
                    // (a is even, so the chunk's number goes into the swizzled address as an exclusive or)
                    ldsm_x4_trans((rows16 ^ (uint32_t)((a & 7) << 4)) + (uint32_t)((a >> 3) * (kTileKeys * 128)), vf);
                    if (masked) {                           // what no row sees may be anything, a NaN too
                        vf[0] &= keep[2 * ks]; vf[1] &= keep[2 * ks + 1];
                        vf[2] &= keep[2 * ks]; vf[3] &= keep[2 * ks + 1];
                    }
                    if (!kE4m3) {
                        mma_16816<kBf16>(out[a], pf, vf[0], vf[1]);
                        mma_16816<kBf16>(out[a + 1], pf, vf[2], vf[3]);
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {       // bytes (0, 2): even columns of the chunk, (1, 3): odd ones
                            const uint32_t w0 = __byte_perm(vf[2 * x], 0, 0x3120), w1 = __byte_perm(vf[2 * x + 1], 0, 0x3120);
                            uint32_t even0, odd0, even1, odd1;
                            halves4(w0, even0, odd0);
                            halves4(w1, even1, odd1);
                            mma_16816<false>(out[2 * (a + x)], pf, even0, even1);
                            mma_16816<false>(out[2 * (a + x) + 1], pf, odd0, odd1);
                        }
                    }
                }
            }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->empty[bar]);
        }
        if (kE4m3) {
#pragma unroll
            for (int d = 0; d < kDim / 8; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) out[d][e] *= __uint_as_float(r_bits);
        }
        // the quad's four partial sums of a row
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        const int b_now = b, hm_now = hm;
        const bool on_now[2] = {row_on[0], row_on[1]};
        u += todo;
        if (tile == tiles) {
            tile = 0;
            u += kBegin;
            if (++hm == hms) { hm = 0; ++b; }
        }
        if (u < share.end) fetch();

        // The warps that share a row group put their O side by side, kJoin columns at a time, and each joins and stores its
        // part of the columns.
        constexpr int kTiles = S::kJoin / 8;
        float weight[kSplit][2];
#pragma unroll
        for (int h = 0; h < kDim / S::kJoin; ++h) {
            if (kSplit > 1) {
                float* ml = merge + kConsumers * 16 * S::kJoin;
#pragma unroll
                for (int d = 0; d < kTiles; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) merge[((warp * kTiles + d) * 4 + e) * 32 + lane] = out[kTiles * h + d][e];
                if (h == 0 && c == 0) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) { ml[warp * 32 + r * 8 + g] = m[r]; ml[warp * 32 + 16 + r * 8 + g] = l[r]; }
                }
                asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
                if (h == 0) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float of[kSplit], top = -INFINITY, sum = 0.0f;
#pragma unroll
                        for (int w = 0; w < kSplit; ++w) {
                            of[w] = ml[(rg * kSplit + w) * 32 + r * 8 + g];
                            top = fmaxf(top, of[w]);
                        }
                        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
                        for (int w = 0; w < kSplit; ++w) {
                            weight[w][r] = attn_exp2(of[w] - ref);
                            sum += weight[w][r] * ml[(rg * kSplit + w) * 32 + 16 + r * 8 + g];
                        }
                        m[r] = top;
                        l[r] = sum;
                    }
                }
            }
            constexpr int kOwn = kTiles / kSplit;           // n-tiles of these columns that this warp stores
            float x[kOwn][4];
#pragma unroll
            for (int d = 0; d < kOwn; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (kSplit == 1) {
                        x[d][e] = out[kTiles * h + d][e];
                    } else {
                        x[d][e] = 0.0f;
#pragma unroll
                        for (int w = 0; w < kSplit; ++w)
                            x[d][e] += merge[(((rg * kSplit + w) * kTiles + part * kOwn + d) * 4 + e) * 32 + lane] * weight[w][e >> 1];
                    }
                }
            // (also before the next queries overwrite these)
            if (kSplit > 1 || h == 0) asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
            const int64_t part_row = ((int64_t)blockIdx.x * 2 + (from_start ? 1 : 0)) * kRows + rg * 16 + g;
            float* ml = p.partial + (int64_t)p.ctas * 2 * kRows * kDim;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int head = hm_now / p.row_tiles, row = (hm_now - head * p.row_tiles) * kRows + rg * 16 + g + 8 * r;
                const int draft = row / p.group;
                if (draft >= p.drafts) continue;
                const int64_t o_at = (((int64_t)b_now * p.drafts + draft) * (p.kv_heads * p.group) + head * p.group + row - draft * p.group) * kDim;
                const bool any = on_now[r] && l[r] != 0.0f;         // false: the row sees nothing, and is zero whatever V holds
                const float by = !any ? 0.0f : (whole ? 1.0f / l[r] : 1.0f);
                if (!whole && h == 0 && part == 0 && c == 0) {
                    ml[(part_row + 8 * r) * 2] = any ? m[r] : -INFINITY;
                    ml[(part_row + 8 * r) * 2 + 1] = any ? l[r] : 0.0f;
                }
#pragma unroll
                for (int d = 0; d < kOwn; d += (kE4m3 ? 2 : 1)) {
                    // e4m3: tiles d, d + 1 hold the even and odd columns of a chunk of 16, this thread's are 4 c .. 4 c + 3
                    const int col = S::kJoin * h + 8 * (part * kOwn + d) + (kE4m3 ? 4 * c : 2 * c);
                    const int d1 = kE4m3 ? d + 1 : d;
                    float v[4] = {x[d][2 * r], kE4m3 ? x[d1][2 * r] : x[d][2 * r + 1], x[d][2 * r + 1], x[d1][2 * r + 1]};
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = any ? v[e] * by : 0.0f;
                    if (whole) {
                        T* to = static_cast<T*>(p.o) + o_at + col;
                        if (kE4m3) *reinterpret_cast<uint2*>(to) = make_uint2(pack2<kTBf16>(v[0], v[1]), pack2<kTBf16>(v[2], v[3]));
                        else *reinterpret_cast<uint32_t*>(to) = pack2<kTBf16>(v[0], v[1]);
                    } else {
                        float* to = p.partial + (part_row + 8 * r) * kDim + col;
                        if (kE4m3) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
                        else *reinterpret_cast<float2*>(to) = make_float2(v[0], v[1]);
                    }
                }
            }
        }
    }
    // the join may be scheduled once every CTA is here (it waits for their memory itself)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Joins what several CTAs left of one (sequence, key head, row tile): one warp per row, kDim / 32 columns per lane.
template <typename T, int kDim>
__global__ void __launch_bounds__(128)
cached_join_kernel(const CachedParams p, int rows) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hms = p.kv_heads * p.row_tiles;
    const int in_tile = rows / 4, item = blockIdx.x / in_tile, r = (blockIdx.x - item * in_tile) * 4 + warp;
    const int b = item / hms, hm = item - b * hms;
    const int head = hm / p.row_tiles, row = (hm - head * p.row_tiles) * rows + r, draft = row / p.group;
    // which CTAs hold this item's tiles follows from the lengths alone: found while the main kernel still runs
    int64_t before;
    const int64_t per = quotient(total_cost<kTileKeys, kBegin>(p, b, before, lane) * hms + p.ctas - 1, p.ctas);
    const int tiles = cached_tiles<kTileKeys>(p, b);
    const int64_t start = before * hms + (int64_t)hm * (tiles + kBegin) + kBegin;       // the unit of tile 0
    const int first = (int)quotient(start, per), last = (int)quotient(start + tiles - 1, per);
    // (also where there is nothing to do: the stream's next kernel waits for this grid, which must not end before the main one)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (draft >= p.drafts || first == last) return;         // one CTA had all of it and wrote the output
    const float* ml = p.partial + (int64_t)p.ctas * 2 * rows * kDim;
    constexpr int kCols = kDim / 32, kBatch = 8;
    float sum[kCols], l = 0.0f, top = -INFINITY;
#pragma unroll
    for (int e = 0; e < kCols; ++e) sum[e] = 0.0f;
    for (int i0 = first; i0 <= last; i0 += kBatch) {        // loads of 8 parts at a time, in the order of the tiles
        float2 w[kBatch];
        float v[kBatch][kCols];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {                  // (slot 1: the CTA that has tile 0; slot 0: the ones after it)
            const int i = min(i0 + k, last);
            const int64_t at = ((int64_t)i * 2 + (i == first)) * rows + r;
            w[k] = *reinterpret_cast<const float2*>(ml + at * 2);
            if (i0 + k > last) w[k] = make_float2(-INFINITY, 0.0f);
            const float* x = p.partial + at * kDim + lane * kCols;      // (zeros where this part saw nothing)
#pragma unroll
            for (int e = 0; e < kCols; e += 2) *reinterpret_cast<float2*>(v[k] + e) = *reinterpret_cast<const float2*>(x + e);
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
            for (int e = 0; e < kCols; ++e) sum[e] += v[k][e] * weight;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* to = static_cast<T*>(p.o) + (((int64_t)b * p.drafts + draft) * (p.kv_heads * p.group) + head * p.group + (row - draft * p.group)) * kDim + lane * kCols;
#pragma unroll
    for (int e = 0; e < kCols; ++e) to[e] = Scalar<T>::from_float(sum[e] * inv);
}

int row_groups(int64_t rows) { return rows <= 16 ? 1 : (rows <= 32 ? 2 : 4); }

template <typename T, bool kE4m3, int kDim, int kGroups>
int launch_cached(const CachedParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t stream) {
    auto kernel = cached_attention_kernel<T, kE4m3, kDim, kGroups>;
    constexpr int smem = CachedShape<kE4m3, kDim, kGroups>::kSmem;
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return BSA_ERR_LAUNCH;
    kernel<<<p.ctas, (kConsumers + 1) * 32, smem, stream>>>(p, map_k, map_v);
    // the join's CTAs may start while the last ones above end; they wait for all of them before they read
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(p.batch * p.kv_heads * p.row_tiles * 4 * kGroups));
    config.blockDim = dim3(128);
    config.stream = stream;
    cudaLaunchAttribute overlap{};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &overlap;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, cached_join_kernel<T, kDim>, p, 16 * kGroups) != cudaSuccess) { cudaGetLastError(); return BSA_ERR_LAUNCH; }
    return launch_status();
}
template <typename T, bool kE4m3, int kDim>
int launch_groups(int groups, const CachedParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t stream) {
    if (groups == 1) return launch_cached<T, kE4m3, kDim, 1>(p, map_k, map_v, stream);
    if (groups == 2) return launch_cached<T, kE4m3, kDim, 2>(p, map_k, map_v, stream);
    return launch_cached<T, kE4m3, kDim, 4>(p, map_k, map_v, stream);
}
template <typename T>
int launch_cached_typed(int store, int64_t dim, int groups, const CachedParams& p, const CUtensorMap& map_k,
                        const CUtensorMap& map_v, cudaStream_t stream) {
    if (store == BSA_CACHE_E4M3)
        return dim == 64 ? launch_groups<T, true, 64>(groups, p, map_k, map_v, stream)
                         : launch_groups<T, true, 128>(groups, p, map_k, map_v, stream);
    return dim == 64 ? launch_groups<T, false, 64>(groups, p, map_k, map_v, stream)
                     : launch_groups<T, false, 128>(groups, p, map_k, map_v, stream);
}

}  // namespace
}  // namespace bsa

extern "C" size_t bsa_cached_attention_scratch(int64_t drafts, int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
    if (drafts <= 0 || kv_heads <= 0 || q_heads < kv_heads || head_dim <= 0) return 0;
    const int64_t rows = drafts * (q_heads / kv_heads), tile = 16 * bsa::row_groups(rows);
    const size_t wide = rows > bsa::kWideRows ? bsa::cached_wide_scratch(head_dim) : 0;
    return std::max(wide, (size_t)std::max(bsa::sm_count(), 1) * 2 * 2 * tile * (size_t)(head_dim + 2) * 4);
}

extern "C" int bsa_cached_attention(int dtype, int store, const void* q, int64_t q_batch_stride, int64_t q_draft_stride,
                                    int64_t q_head_stride, const void* keys, const void* values, const float* key_scales,
                                    const float* value_scales, void* o, const int32_t* table, const int32_t* lengths,
                                    const int32_t* counts, const int64_t* tree, const uint8_t* pattern,
                                    int64_t pattern_rows, int64_t pattern_cols, int64_t pattern_block, int64_t batch,
                                    int64_t drafts, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t pages,
                                    int64_t page, int64_t table_width, float scale, void* scratch, size_t scratch_bytes,
                                    void* workspace, size_t workspace_bytes, void* stream) {
    using namespace bsa;
    const int checked = check_cache(dtype, store, key_scales, value_scales, pages, kv_heads, page, head_dim);
    if (checked != BSA_OK) return checked;
    if (batch < 0 || drafts <= 0 || q_heads <= 0 || q_heads % kv_heads != 0 || table_width <= 0) return BSA_ERR_BAD_SHAPE;
    if (drafts > 64) return BSA_ERR_TOO_LARGE;              // one bit of a tree word per draft
    // every CTA of the join looks through all lengths: 16 tokens of each sequence, 2 key heads of 64, take 0.5 ms for 4,096
    // sequences, 5.6 ms for 16,384 and 83 ms for 65,536
    if (batch > 65536) return BSA_ERR_TOO_LARGE;
    if (!workspace || workspace_bytes < BSA_WORKSPACE_BYTES) return BSA_ERR_WORKSPACE;
    if (pattern && (!valid_block((int)pattern_block) || pattern_block > 128)) return BSA_ERR_BAD_BLOCK;
    if (pattern && (pattern_rows <= 0 || pattern_cols <= 0 || pattern_rows > 65535 || pattern_cols > 65535)) return BSA_ERR_BAD_SHAPE;
    if (batch == 0) return BSA_OK;
    if (!q || !keys || !values || !o || !table || !lengths || !scratch) return BSA_ERR_NULL_POINTER;
    if (!aligned16(q) || !aligned16(keys) || !aligned16(values) || !aligned16(o) || !aligned16(scratch)) return BSA_ERR_ALIGNMENT;
    if (store == BSA_CACHE_E4M3 && (!aligned16(key_scales) || !aligned16(value_scales))) return BSA_ERR_ALIGNMENT;
    if (q_batch_stride < 0 || q_draft_stride < 0 || q_head_stride < 0) return BSA_ERR_BAD_SHAPE;
    if (q_batch_stride % 8 || q_draft_stride % 8 || q_head_stride % 8) return BSA_ERR_ALIGNMENT;
    if (table_width > (int64_t)(INT32_MAX - 256) / page) return BSA_ERR_TOO_LARGE;      // 32-bit positions in a sequence
    // the kernel for many rows stores 32 bytes at a time; asked of every call, so that it does not depend on the number of rows
    if (reinterpret_cast<uintptr_t>(o) & 31) return BSA_ERR_ALIGNMENT;
    CachedParams p{};
    const int64_t group = q_heads / kv_heads;
    const int groups = row_groups(drafts * group);
    const int64_t row_tiles = (drafts * group + 16 * groups - 1) / (16 * groups);
    if (row_tiles * kv_heads > (int64_t)INT32_MAX / batch / (4 * groups) || q_heads > 65535) return BSA_ERR_TOO_LARGE;
    p.q = q; p.o = o;
    p.q_batch = q_batch_stride; p.q_draft = q_draft_stride; p.q_head = q_head_stride;
    p.scales[0] = key_scales; p.scales[1] = value_scales;
    p.table = table; p.lengths = lengths; p.counts = counts; p.tree = tree;
    p.pattern = pattern;
    p.pattern_rows = (int)pattern_rows; p.pattern_cols = (int)pattern_cols;
    while (pattern && (1 << p.pattern_shift) < pattern_block) ++p.pattern_shift;
    p.batch = (int)batch; p.drafts = (int)drafts; p.group = (int)group; p.kv_heads = (int)kv_heads;
    p.row_tiles = (int)row_tiles; p.table_width = (int)table_width; p.pages = (int)pages;
    while ((1 << p.page_shift) < page) ++p.page_shift;
    p.scale_log2 = scale * kLog2e;
    p.partial = static_cast<float*>(scratch);
    p.ctas = 2 * sm_count();
    p.status = static_cast<uint32_t*>(workspace);
    if (p.ctas <= 0) return BSA_ERR_LAUNCH;
    if (scratch_bytes < bsa_cached_attention_scratch(drafts, q_heads, kv_heads, head_dim)) return BSA_ERR_WORKSPACE;
    // the driver's encoder needs the device's context bound to this thread
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) { cudaGetLastError(); return BSA_ERR_LAUNCH; }
    if (drafts * group > kWideRows && store == BSA_CACHE_SAME && !pattern)
        return cached_wide(p, dtype, head_dim, keys, values, page, static_cast<cudaStream_t>(stream));
    CUtensorMap map_k, map_v;
    const int64_t rows = pages * kv_heads * page;
    const int piece = (int)std::min<int64_t>(page, kTileKeys);
    if (!make_cache_map(&map_k, store, dtype, keys, rows, head_dim, piece) ||
        !make_cache_map(&map_v, store, dtype, values, rows, head_dim, piece)) return BSA_ERR_DRIVER;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == BSA_DTYPE_F16 ? launch_cached_typed<__half>(store, head_dim, groups, p, map_k, map_v, s)
                                  : launch_cached_typed<__nv_bfloat16>(store, head_dim, groups, p, map_k, map_v, s);
}
