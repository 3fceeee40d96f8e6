// Attention of one new token a row where rows share a prefix (epq_paged_attend_shared): the plan,
// the shared tokens and the join.  (The rest: k_paged_attn_shared.cu; what they hand on: epq_shared.cuh.)
//
// Rows of a group that see tokens [0, L) all alike are one attention of many query rows over one
// set of keys: with r rows and g query heads a key head, r g rows over L tokens, 4 r g flops a
// cached value.  So it is the tensor cores' (tcgen05) work, and what is read once is read for
// r rows.
//
// Plan (one CTA): groups are cut into tiles of up to 256 query rows (128 where head_dim > 128);
// L of a tile is its prefix, or the shortest of its rows' lengths.  No score needs a mask by row
// then: what a row sees beyond L is its own part, and a value there that is not finite stays in
// the rows that see it.  A tile shares where reading its tokens row by row is reckoned to take
// longer than its blocks here (Reckoning below), a batch where its tiles save more than kFixed.
//
// Shared part.  Blocks of 128 tokens of all units (tile, key head) are dealt out to the CTAs in
// equal runs, one CTA an SM, and each piece of a unit leaves its sums as records.  In a CTA:
//   * one warp looks up pages and copies Q and the rows of K and V (TMA boxes of up to 128 rows
//     of a page, a lane a box) into shared memory in the 128-byte swizzle; rows of 8-bit caches
//     pass through four more warps that widen them to 16 bits (exact);
//   * one thread issues the products: S = Q K^T (Q, K in shared memory) and O += P V (P in tensor
//     memory, V as the MN-major operand);
//   * 8 warps a slot take half a row a thread: maximum, weights, sum; P goes back in place of S.
// Two slots (S and O in tensor memory: all of its 512 columns) keep the products of one under
// the softmax of the other: two tiles of 128 rows over the same block, or, for units of up to
// 128 rows, one tile whose blocks alternate.
//
// Precision.  Weights are the sum of two 16-bit values, as in k_paged_attn.cu: one rounding of
// them is as large as the result's own (products with P cost twice as much, 3 units of tensor
// time a block instead of 2).  8-bit caches: keys are exact in q's type, values and weights are
// bf16, whose range takes any scale; a key's scale multiplies its score, a value's its weight.
// The running maximum moves only when a score passes it by 2^8.
//
// Measured (B200, device time in a graph of calls, all four launches): 64 rows behind 8,192 tokens, 32 / 8
// heads of 128, bf16: 67 us (row by row 211); 256 rows behind 32,768, 64 / 8 heads, e4m3: 628 us, 552 of
// them the shared tokens (row by row 2,152).  What bounds it is a slot's chain of product, softmax and product, about
// 4 us a block of 128 tokens for 1.7 us of tensor time with two slots: a softmax thread reads its half row of S from
// tensor memory twice, 32 columns at a time and each time to the end, and the 8-bit forms, built for 22 warps at 80
// registers, spill (88 to 92 bytes stored, 300 to 308 loaded a thread).  A tile whose shortest row is of 5 tokens goes row by
// row: 64 rows behind 8,192 take 211 us with one such row.
#include "epq_attend.cuh"
#include "epq_sm100.cuh"
#include <cuda.h>

namespace epq {
namespace paged {

int attend_behind_shared(const AttendArgs& A, int cols, cudaStream_t st);
int attend_shared_read_device_error(int* flag);

namespace {

__device__ int g_shared_error = 0;         // kBadPosition, kBadPage
__device__ int g_shared_timeout = 0;       // a bounded wait gave up

constexpr unsigned kWarpAll = 0xffffffffu;
constexpr int kPlanThreads = 512;
constexpr int kHeldTiles = 512;            // tiles that the plan keeps in shared memory
constexpr uint32_t kWaitLimit = 1u << 22;
constexpr int kSmemLimit = 232448;         // 227 KB a CTA

// What is reckoned with, in ns, from both sides measured (B200, graphs of calls; 2 to 64 rows a
// group, 1 to 16 groups, 1024 to 65536 tokens, 32 / 8, 64 / 8 and 8 / 1 heads of 64 and 128,
// 16 / 4 of 256).  Row by row: 10 us and 9.0 to 10.3 TB/s of 16-bit caches (6.2 for heads of 256), 5.6
// to 6.9 of 8-bit ones; what several rows read comes from L2.  Shared: 30 to 41 us, and a block of 128
// tokens and 128 rows 1.65 us (64 dims), 2.0 (128) or 4.1 (256), 8-bit ones 2.6 and 3.1.  So 2
// rows of 32 / 8 heads do not share before 2 x 16 groups x 16k tokens (222 us for 326; 16 x 4k:
// 81 for 80), 4 groups of 4 with int8 not at all (354 us for 309 at 64k), and 64 rows always
// from 4k tokens on.  What the plan then leaves row by row costs its launches, 9 us.
constexpr float kFixed = 25000.f;
struct Reckoning {
    float row_token;                       // a token of all key heads, row by row, on the whole card
    float block;                           // 128 tokens of 128 rows and a key head, on one SM
};
Reckoning reckon(const PagesD& P) {
    const int64_t token_bytes = 2LL * P.kv_heads * (P.format == EPQ_CACHE_SAME ? P.head_dim * 2 : P.head_dim + 4);
    if (P.format != EPQ_CACHE_SAME) return {(float)token_bytes / 6900.f, P.head_dim <= 64 ? 2600.f : 3100.f};
    if (P.head_dim > 128) return {(float)token_bytes / 6200.f, 4100.f};
    return {(float)token_bytes / 9300.f, P.head_dim <= 64 ? 1650.f : 2050.f};
}

struct SharedArgs {
    PagesD pages;
    SharedD s;
    const int32_t* seq;
    const int64_t* lengths;
    const int32_t* starts;
    const int64_t* prefix;
    Reckoning cost;
    bool always;                           // share whatever can be
    int batch, groups, heads, group, max_tiles, grid, box_rows;
    float scale_log2;
};
struct Maps {                              // q [batch][heads][head_dim], the pools [pages][heads, slots][head_dim]
    CUtensorMap q, k, v;
};

// ---------------------------------------------------------------- plan
// Inclusive sum over the CTA's threads; `total` gets the whole sum.  (Two barriers.)
__device__ int64_t block_scan(int64_t v, int64_t* shared, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(kWarpAll, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) shared[warp] = v;
    __syncthreads();
    int64_t w = lane < kPlanThreads / 32 ? shared[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(kWarpAll, w, o);
        if (lane >= o) w += u;
    }
    *total = __shfl_sync(kWarpAll, w, 31);
    const int64_t before = __shfl_sync(kWarpAll, w, warp ? warp - 1 : 0);
    __syncthreads();
    return warp ? v + before : v;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const SharedArgs A) {
    __shared__ int64_t scratch[32];
    __shared__ SharedTile held[kHeldTiles];
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const PagesD& P = A.pages;
    const int64_t cap = (int64_t)P.max_pages * P.page_size;
    const int tile_rows = A.s.slots * A.s.lane_rows;
    SharedTile* const tile = A.max_tiles <= kHeldTiles ? held : A.s.tiles;     // (written out at the end)
    // rows that are neither empty nor bad (which the last launch reports)
    auto counts = [&](int b) {
        const int64_t n = A.lengths[b];
        const int s = A.seq ? A.seq[b] : b;
        return n > 0 && n <= cap && s >= 0 && s < P.seqs;
    };
    for (int b = tid; b < A.batch; b += kPlanThreads) {
        A.s.row_tile[b] = -1;
        A.s.row_from[b] = 0;
    }
    // groups to tiles
    bool good = true;
    for (int g = tid; g < A.groups; g += kPlanThreads) {
        const int from = A.starts[g], to = A.starts[g + 1];
        const int64_t p = A.prefix[g];
        good = good && from >= 0 && from <= to && to <= A.batch && p >= 0 && p <= cap;
    }
    good = __syncthreads_and(good);
    if (!good && tid == 0) atomicOr(&g_shared_error, kBadPosition);
    int64_t tiles = 0;
    for (int g0 = 0; good && g0 < A.groups; g0 += kPlanThreads) {
        const int g = g0 + tid;
        const int from = g < A.groups ? A.starts[g] : 0, rows = g < A.groups ? A.starts[g + 1] - from : 0;
        const int count = rows >= 2 ? (rows + tile_rows - 1) / tile_rows : 0;
        int64_t all;
        int64_t at = tiles + block_scan(count, scratch, &all) - count;
        for (int i = 0; i < count && at < A.max_tiles; ++i, ++at) {
            SharedTile T = {};
            T.row0 = from + i * tile_rows;
            T.rows = min(tile_rows, from + rows - T.row0);
            T.tokens = (int)A.prefix[g];
            tile[at] = T;
        }
        tiles += all;
    }
    tiles = min(tiles, (int64_t)A.max_tiles);
    __syncthreads();
    // what each tile's rows share
    int64_t saved = 0;
    for (int t = warp; t < tiles; t += kPlanThreads / 32) {
        const SharedTile T = tile[t];
        int active = 0, first = INT32_MAX, least = T.tokens;
        for (int r = lane; r < T.rows; r += 32) {
            if (!counts(T.row0 + r)) continue;
            ++active;
            first = min(first, r);
            least = (int)min((int64_t)least, A.lengths[T.row0 + r]);
        }
        active = __reduce_add_sync(kWarpAll, active);
        first = __reduce_min_sync(kWarpAll, first);
        least = active < 2 ? 0 : __reduce_min_sync(kWarpAll, least);
        if (lane == 0) {
            const int b = T.row0 + first;
            tile[t].seq = active < 2 ? 0 : A.seq ? A.seq[b] : b;
            const int blocks = (least + kSharedTokens - 1) / kSharedTokens;
            const int tile_slots = T.rows > A.s.lane_rows ? 2 : 1;              // (of up to 128 query rows)
            const float gain = (float)active * (float)least * A.cost.row_token -
                               (float)blocks * (float)(P.kv_heads * tile_slots) * A.cost.block / (float)A.grid;
            const bool shares = A.always || gain > 0.f;
            tile[t].tokens = shares ? least : 0;
            saved += shares ? (int64_t)gain : 0;
        }
    }
    int64_t all_saved;
    block_scan(saved, scratch, &all_saved);
    const bool worth = A.always || all_saved > (int64_t)kFixed;
    // places of the units
    int64_t total = 0;
    for (int t0 = 0; t0 < tiles; t0 += kPlanThreads) {
        const int t = t0 + tid;
        const int blocks = worth && t < tiles ? (tile[t].tokens + kSharedTokens - 1) / kSharedTokens : 0;
        const int64_t mine = (int64_t)blocks * P.kv_heads;
        int64_t all;
        const int64_t at = total + block_scan(mine, scratch, &all) - mine;
        if (t < tiles) {
            SharedTile T = tile[t];
            T.blocks = blocks;
            T.first = at;
            A.s.tiles[t] = T;
        }
        total += all;
    }
    if (tid == 0) *A.s.head = {total, (int)max((int64_t)1, (total + A.grid - 1) / A.grid), (int)tiles};
    for (int t = warp; worth && t < tiles; t += kPlanThreads / 32) {
        const SharedTile T = tile[t];                                  // (what it needs of T is there since the first part)
        for (int r = lane; T.tokens && r < T.rows; r += 32) {
            A.s.row_tile[T.row0 + r] = t;
            A.s.row_from[T.row0 + r] = counts(T.row0 + r) ? T.tokens : 0;
        }
    }
}

// ---------------------------------------------------------------- the shared tokens
enum Codes { kNone = 0, kInts = 1, kFloats = 2 };

template <int kCodes, int kDim> struct Cfg {
    static constexpr int kSlots = kDim == 256 ? 1 : 2;
    static constexpr int kConvertWarps = kCodes ? 4 : 0;
    static constexpr int kSoftmaxWarps = kSlots * 8, kMmaWarp = kSoftmaxWarps + kConvertWarps, kLoadWarp = kMmaWarp + 1;
    static constexpr int kThreads = (kLoadWarp + 1) * 32;
    static constexpr int kBuf = kSharedTokens * kDim * 2;              // K or V of a block
    static constexpr int kSlab = kSharedTokens * 128;                  // 64 values of each of its rows
    static constexpr int kQ = kSlots * kSharedLanes * kDim * 2;
    static constexpr int kRaw = kCodes ? kSharedTokens * kDim : 0;     // codes of K or V of a block
    static constexpr int kRawStages = kCodes ? 3 : 0;
    // Blocks whose masks and scales are kept: a block's are written once its K has a stage, when the items that are
    // kStages stages back have been multiplied, and so the softmax of all before them is done.
    static constexpr int kRing = kCodes ? 4 : 8;
    static constexpr int kScales = kCodes ? kRing * 2 * kSharedTokens * 4 : 0;
    static constexpr int kMasksAt = kScales, kTopsAt = kMasksAt + kRing * 16, kBarsAt = kTopsAt + kSlots * 2 * kSharedLanes * 4;
    static constexpr int kMisc = kBarsAt + 352;
    static constexpr int kFit = (kSmemLimit - 1024 - kMisc - kQ - kRawStages * kRaw) / kBuf, kMost = kCodes ? 4 : 8;
    static constexpr int kStages = kFit > kMost ? kMost : kFit;
    static constexpr int kQAt = kStages * kBuf, kRawAt = kQAt + kQ, kMiscAt = kRawAt + kRawStages * kRaw;
    static constexpr int kSmem = 1024 + kMiscAt + kMisc;
    static_assert(kStages >= (kSlots == 2 ? 3 : 2) && kSmem <= kSmemLimit, "shared memory");
};

// A unit's piece in this CTA: blocks [i, i + n) of tile T for key head h.
struct Piece {
    SharedTile T;
    int t, h, i, n, c;                     // c: pieces of this CTA before it
    int64_t at, end;
};
__device__ __forceinline__ bool piece_at(const SharedArgs& A, Piece& p) {
    if (p.at >= p.end) return false;
    p.T = A.s.tiles[p.t];
    p.i = (int)(p.at - p.T.first - (int64_t)p.h * p.T.blocks);
    p.n = (int)min((int64_t)p.T.blocks - p.i, p.end - p.at);
    return true;
}
__device__ __forceinline__ void next_piece(const SharedArgs& A, Piece& p) {
    p.at += p.n;
    ++p.c;
    if (p.at >= p.end) return;
    if (++p.h == A.pages.kv_heads) {
        p.h = 0;
        while (A.s.tiles[++p.t].blocks == 0) {}                        // (there is one: its blocks are dealt out)
    }
}

// Codes of 8-bit caches as 16-bit values, exactly: four of them as two pairs.
template <int kCodes, bool kBf> __device__ __forceinline__ void widen(uint32_t x, uint32_t& p0, uint32_t& p1) {
    if constexpr (kCodes == kInts && kBf) {
        // 0x43 above a byte is 128 + its low 7 bits, or 256 + them; taking off 128, or 256 where the byte's top bit is
        // set, leaves its low 7 bits, less 128 where it is
        const uint32_t w0 = __byte_perm(x, 0x43434343u, 0x4140), w1 = __byte_perm(x, 0x43434343u, 0x4342);
        auto value = [](uint32_t w) {
            const uint32_t a = w & 0xff7fff7fu, b = w & 0xff80ff80u;
            const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
            return *reinterpret_cast<const uint32_t*>(&r);
        };
        p0 = value(w0);
        p1 = value(w1);
    } else {
        codes_f16<kCodes == kInts ? kInt8 : kFp8, false>(x, p0, p1);
        if (kBf) {
            const float2 a = unpack2<__half>(p0), b = unpack2<__half>(p1);
            p0 = pack2<__nv_bfloat16>(a.x, a.y);
            p1 = pack2<__nv_bfloat16>(b.x, b.y);
        }
    }
}

// Weights as pairs of 16-bit values and of what these leave.  bf16: the first part is the upper half of the float32, without
// its lower bits, which takes no conversion; the second, of what that leaves exactly, is rounded to the nearest.  Both
// together are off by at most 2^-16, and by nothing on average; a second part that is cut off too (256 rows x 32k, e4m3:
// 621 us, rounded 628) is 2^-17 too small on average, and the sum that the result is divided by is of whole weights.
template <bool kBf> __device__ __forceinline__ void split(const float (&w)[32], uint32_t (&hi)[16], uint32_t (&lo)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float a = w[2 * i], b = w[2 * i + 1];
        if (kBf) {
            const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
            hi[i] = __byte_perm(x, y, 0x7632);
            const float c = a - __uint_as_float(x & 0xffff0000u), d = b - __uint_as_float(y & 0xffff0000u);
            lo[i] = pack2<__nv_bfloat16>(c, d);
        } else {
            hi[i] = pack2<__half>(a, b);
            const float2 back = unpack2<__half>(hi[i]);
            lo[i] = pack2<__half>(a - back.x, b - back.y);
        }
    }
}

// kBfQ: S in bf16 (else f16); kBfV: P and V in bf16 (else f16).
template <int kCodes, bool kBfQ, bool kBfV, int kDim>
__global__ void __launch_bounds__(Cfg<kCodes, kDim>::kThreads, 1)
    shared_kernel(const SharedArgs A, const __grid_constant__ Maps maps) {
    using C = Cfg<kCodes, kDim>;
    using namespace sm100;
    constexpr int S_ = C::kStages, kSlots = C::kSlots;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PagesD& P = A.pages;
    const int hd = P.head_dim, gh = A.group, ps = P.page_size;

    const uint32_t raw = sm100::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* const gen = smem_raw + (base - raw);
    uint8_t* const misc = gen + C::kMiscAt;
    float* const scales = reinterpret_cast<float*>(misc);              // [kRing][2][128]: of keys, of values
    uint32_t* const masks = reinterpret_cast<uint32_t*>(misc + C::kMasksAt);           // [kRing][4]
    float* const tops = reinterpret_cast<float*>(misc + C::kTopsAt);   // [slots][halves][128]
    const uint32_t bars = base + C::kMiscAt + C::kBarsAt;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 64u + 8u * s; };
    auto raw_full = [&](int s) { return bars + 128u + 8u * s; };
    auto raw_empty = [&](int s) { return bars + 160u + 8u * s; };
    auto s_full = [&](int s) { return bars + 192u + 8u * s; };
    auto p_full = [&](int s) { return bars + 208u + 8u * s; };
    auto o_done = [&](int s) { return bars + 224u + 8u * s; };
    const uint32_t q_full = bars + 240u, q_free = bars + 248u, over = bars + 256u, part_full = bars + 264u, tslot = bars + 272u;
    auto pair_full = [&](int i) { return bars + 288u + 8u * i; };
    volatile int* const abortp = reinterpret_cast<volatile int*>(misc + C::kBarsAt + 280);
    volatile int* const where = reinterpret_cast<volatile int*>(misc + C::kBarsAt + 284);
    auto wait = [&](uint32_t bar, uint32_t parity) {
        return mbar_wait_bounded(bar, parity & 1u, abortp, &g_shared_timeout, kWaitLimit);
    };
    // every lane, or none
    auto wait_all = [&](uint32_t bar, uint32_t parity) { return __all_sync(kWarpAll, wait(bar, parity)); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < S_; ++s) {
            mbar_init(full(s), kCodes ? C::kConvertWarps * 32 : 1);
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < C::kRawStages; ++s) {
            mbar_init(raw_full(s), 1);
            mbar_init(raw_empty(s), C::kConvertWarps * 32);
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(s_full(s), 2);                                   // the products' end, and the issuing thread
            mbar_init(p_full(s), 256);
            for (int i = 0; i < 4; ++i) mbar_init(pair_full(4 * s + i), 64);
            mbar_init(o_done(s), 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_free, 1);
        mbar_init(over, 1);
        mbar_init(part_full, 1);
        *abortp = 0;
        mbar_init_fence();
    }
    if (warp == C::kLoadWarp && lane == 0) {
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
    }
    if (warp == C::kMmaWarp) tmem_alloc(tslot, 512);
    pdl_enter();                                                       // (nothing above reads what the plan writes)
    const SharedHead head = *A.s.head;
    Piece first;
    first.at = (int64_t)blockIdx.x * head.run;
    first.end = min(head.total, first.at + head.run);
    if (warp == 0) {                                                   // the tile of the first piece
        int t = 0;
        for (int t0 = 0; t0 < head.tiles; t0 += 32) {
            const bool here = t0 + lane < head.tiles && A.s.tiles[t0 + lane].first <= first.at;
            const unsigned below = __ballot_sync(kWarpAll, here);
            if (below) t = t0 + 31 - __clz(below);
            if (below != kWarpAll) break;
        }
        if (lane == 0) *where = t;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(kWarpAll, *reinterpret_cast<volatile uint32_t*>(misc + C::kBarsAt + 272), 0);
    first.t = *where;
    first.c = 0;
    first.h = 0;
    if (first.at < first.end) {
        const SharedTile T = A.s.tiles[first.t];
        first.h = (int)((first.at - T.first) / T.blocks);
    }
    const uint32_t q_at = base + C::kQAt;
    constexpr uint32_t kOCol = kSlots * 128u;                          // S and P of slot s in columns 128 s, O behind them
    auto alternates = [&](const SharedTile& T) { return kSlots == 1 || shared_alternates(T.rows, A.s.lane_rows, kSlots); };

    if (warp >= C::kMmaWarp) {
        if (warp == C::kLoadWarp) {
            // -------------------------------------------------------- loads: a lane a box of rows of one page
            const int R = A.box_rows, boxes = kSharedTokens / R;
            constexpr int kSlabs = kDim / 64;
            const bool mine = lane < boxes;
            int fills = 0, parts = 0;                                  // stages filled; blocks that end inside
            bool ok = true;
            int32_t next_page = -1;
            auto look_up = [&](const SharedTile& T, int block) {       // the page of this lane's box; it is on its way
                const int t = block * kSharedTokens + lane * R;
                next_page = mine && t < T.tokens ? P.table[(int64_t)T.seq * P.table_stride + P.page_of(t)] : -1;
            };
            auto open = [&](uint32_t bar, int f, int ring) {           // fill f's stage of a ring, once it is free
                ok = f < ring || wait_all(bar, f / ring - 1);
                return ok;
            };
            Piece p = first;
            for (; ok && piece_at(A, p); next_piece(A, p)) {
                look_up(p.T, p.i);
                for (int k = 0; ok && k < p.n; ++k) {
                    const int block = p.i + k, t0 = block * kSharedTokens + lane * R;
                    const bool inside = mine && t0 < p.T.tokens;
                    const int32_t page = next_page;
                    const bool there = inside && page >= 0 && page < P.pages;
                    if (inside && !there) atomicOr(&g_shared_error, kBadPage);
                    if (k + 1 < p.n) look_up(p.T, block + 1);
                    const int y = there ? p.h * ps + t0 - P.page_of(t0) * ps : 0;
                    const int count = __popc(__ballot_sync(kWarpAll, there));
                    // (an 8-bit block's rows that are no tokens are zeroed where the codes are widened)
                    const bool whole = kCodes || (count == boxes && (block + 1) * kSharedTokens <= p.T.tokens);
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const CUtensorMap* const map = kv ? &maps.v : &maps.k;
                        if constexpr (kCodes) {
                            const int s = fills % C::kRawStages;
                            if (!open(raw_empty(s), fills, C::kRawStages)) break;
                            if (lane == 0) mbar_expect_tx(raw_full(s), count * R * hd);
                            __syncwarp();
                            if (there) tma_load_3d(base + C::kRawAt + s * C::kRaw + lane * R * hd, map, raw_full(s), 0, y, page);
                        } else {
                            const int s = fills % S_;
                            if (!open(empty(s), fills, S_)) break;
                            const uint32_t to = base + s * C::kBuf;
                            if (kv == 0) {                             // which rows are tokens
                                const int seen = there ? min(R, p.T.tokens - t0) : 0;
                                if (whole) {
                                    if (lane < 4) masks[(fills / 2 % C::kRing) * 4 + lane] = kWarpAll;
                                } else {
                                    for (int w = 0; w < 4; ++w) {      // (boxes of 8 to 128 rows)
                                        uint32_t bits = 0;
                                        const int r0 = lane * R - 32 * w, r1 = r0 + seen;
                                        if (seen && r1 > 0 && r0 < 32) {
                                            bits = r1 >= 32 ? kWarpAll : (1u << r1) - 1;
                                            if (r0 > 0) bits &= ~((1u << r0) - 1);
                                        }
                                        bits = __reduce_or_sync(kWarpAll, bits);
                                        if (lane == 0) masks[(fills / 2 % C::kRing) * 4 + w] = bits;
                                    }
                                }
                            }
                            // a value of a row that is no token must be finite: such a block's V is patched first
                            const uint32_t bar = kv && !whole ? part_full : full(s);
                            __syncwarp();
                            if (lane == 0) mbar_expect_tx(bar, count * R * 128 * kSlabs);
                            __syncwarp();
                            if (there)
#pragma unroll
                                for (int x = 0; x < kSlabs; ++x)
                                    tma_load_3d(to + x * C::kSlab + lane * R * 128, map, bar, 64 * x, y, page);
                            if (kv && !whole) {
                                ok = wait_all(part_full, parts++);
                                if (!ok) break;
                                const unsigned good = __ballot_sync(kWarpAll, there);
                                for (int r = lane; r < kSharedTokens; r += 32)
                                    if (!(good >> (r / R) & 1) || block * kSharedTokens + r >= p.T.tokens)
                                        for (int x = 0; x < kSlabs * 8; ++x)
                                            *reinterpret_cast<uint4*>(gen + s * C::kBuf + (x / 8) * C::kSlab + r * 128 + (x % 8) * 16) =
                                                make_uint4(0, 0, 0, 0);
                                fence_async_smem();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(full(s));
                            }
                        }
                        ++fills;
                        if (k == 0 && kv == 0) {                       // q, behind the first keys
                            if (p.c) {
                                ok = wait_all(q_free, p.c - 1);
                                if (!ok) break;
                            }
                            const int tiles = alternates(p.T) ? 1 : kSlots;
                            if (lane == 0) {
                                mbar_expect_tx(q_full, tiles * kSlabs * A.s.lane_rows * gh * 128);
                                for (int t = 0; t < tiles; ++t)
                                    for (int x = 0; x < kSlabs; ++x)
                                        tma_load_3d(q_at + t * (128 * kDim * 2) + x * C::kSlab, &maps.q, q_full, 64 * x, p.h * gh,
                                                    p.T.row0 + t * A.s.lane_rows);
                            }
                        }
                    }
                }
            }
            // the copies in flight land before the CTA ends (their barriers are those that the others wait for; after
            // a wait that gave up nobody may have)
            if (!ok) {
                for (int s = 0; s < (kCodes ? C::kRawStages : S_); ++s)
                    for (int f = fills - 1; f >= 0 && f >= fills - (kCodes ? C::kRawStages : S_); --f)
                        if (f % (kCodes ? C::kRawStages : S_) == s)
                            for (uint32_t i = 0; i < kWaitLimit; ++i)
                                if (mbar_try_wait(kCodes ? raw_full(s) : full(s), (f / (kCodes ? C::kRawStages : S_)) & 1)) break;
            }
        } else {
            // -------------------------------------------------------- products
            constexpr uint32_t s_idesc = idesc_f16<kBfQ, 128, kSharedTokens>();
            constexpr uint32_t o_idesc = idesc_f16<kBfV, 128, kDim, false, true>();
            const uint64_t q_desc = desc_kmajor_sw128(q_at), k_desc = desc_kmajor_sw128(base);
            const uint64_t v_desc = desc_mnmajor_sw128(base, C::kSlab, 1024);
            int count0 = 0, count1 = 0;                                // products with P that the slots have had
            int fills = 0;                                             // stages before this piece
            bool ok = true;
            Piece p = first;
            for (; ok && piece_at(A, p); next_piece(A, p)) {
                const bool alternate = alternates(p.T);
                const int items = alternate ? p.n : 2 * p.n;
                ok = wait_all(q_full, p.c);
                // item w is block w (alternate) or w / 2, of slot w % kSlots
                auto scores = [&](int w) {
                    const int slot = w % kSlots, block = alternate ? w : w >> 1, f = fills + 2 * block, s = f % S_;
                    ok = ok && wait_all(full(s), f / S_);
                    // P of the slot's last item lies where S goes
                    const int had = slot ? count1 : count0;
                    if (had) ok = ok && wait_all(o_done(slot), had - 1);
                    if (!ok) return;
                    tc_fence_after();
                    if (!elect_one()) return;
                    const uint64_t q = q_desc + (alternate ? 0 : slot * (128 * kDim * 2 / 16)), k = k_desc + s * (C::kBuf / 16);
                    auto step = [&](int d) {                           // 16 dims
                        const uint32_t off = (d / 4) * (C::kSlab / 16) + 2 * (d % 4);
                        mma_f16_ss(tmem + slot * 128, q + off, k + off, s_idesc, d != 0);
                    };
                    if (hd == kDim) {
#pragma unroll
                        for (int d = 0; d < kDim / 16; ++d) step(d);
                    } else {
#pragma unroll 1
                        for (int d = 0; d < hd / 16; ++d) step(d);
                    }
                    mma_commit(s_full(slot));
                    mbar_arrive(s_full(slot));
                    if (alternate || slot == 1) mma_commit(empty(s));
                    if (w == items - 1) mma_commit(q_free);
                };
                auto sums = [&](int w) {
                    const int slot = w % kSlots, block = alternate ? w : w >> 1, f = fills + 2 * block + 1, s = f % S_;
                    const int had = slot ? count1 : count0;
                    ok = ok && wait_all(full(s), f / S_) && wait_all(p_full(slot), had);
                    (slot ? count1 : count0) = had + 1;
                    if (!ok) return;
                    tc_fence_after();
                    if (!elect_one()) return;
                    const uint64_t v = v_desc + s * (C::kBuf / 16);
                    const uint32_t o = tmem + kOCol + slot * kDim, p_at = tmem + slot * 128;
#pragma unroll
                    for (int t = 0; t < kSharedTokens / 16; ++t) {     // 16 tokens: 8 columns of each part of P
                        const uint32_t at = p_at + 32 * (t / 2) + 8 * (t % 2);
                        mma_f16_ts(o, at, v + t * (2048 / 16), o_idesc, w >= kSlots || t != 0);
                        mma_f16_ts(o, at + 16, v + t * (2048 / 16), o_idesc, 1);
                    }
                    mma_commit(o_done(slot));
                    if (alternate || slot == 1) mma_commit(empty(s));
                };
                for (int w = 0; w < kSlots && w < items && ok; ++w) {
                    scores(w);
                    __syncwarp();
                }
                for (int w = 0; w < items && ok; ++w) {
                    sums(w);
                    __syncwarp();
                    if (ok && w + kSlots < items) scores(w + kSlots);
                    __syncwarp();
                }
                fills += 2 * p.n;
            }
            // every product is complete before tensor memory is released
            if (elect_one()) mma_commit(over);
            for (uint32_t i = 0; i < kWaitLimit; ++i)
                if (mbar_try_wait(over, 0)) break;
        }
        __syncwarp();
    } else if (kCodes && warp >= C::kSoftmaxWarps) {
        // ------------------------------------------------------------ 8-bit rows to 16 bits: a thread a row
        if constexpr (kCodes != kNone) {
            const int row = threadIdx.x - C::kSoftmaxWarps * 32, chunks = hd / 16;
            const int ch0 = row % chunks;                              // lanes begin at different chunks: no bank conflicts
            int fills = 0;
            bool ok = true;
            int32_t next_page = -1;
            auto look_up = [&](const SharedTile& T, int block) {
                const int t = block * kSharedTokens + row;
                next_page = t < T.tokens ? P.table[(int64_t)T.seq * P.table_stride + P.page_of(t)] : -1;
            };
            Piece p = first;
            for (; ok && piece_at(A, p); next_piece(A, p)) {
                look_up(p.T, p.i);
                for (int k = 0; ok && k < p.n; ++k) {
                    const int block = p.i + k, entry = fills / 2 % C::kRing;
                    const int32_t page = next_page;
                    const bool there = page >= 0 && page < P.pages;    // (others are reported by the loads)
                    float ks = 0.f, vs = 0.f;
                    if (there) {
                        const int t = block * kSharedTokens + row;
                        const int64_t at = page * P.scale_stride + (int64_t)p.h * ps + t - P.page_of(t) * ps;
                        ks = P.k_scale[at];
                        vs = P.v_scale[at];
                    }
                    if (k + 1 < p.n) look_up(p.T, block + 1);
                    const unsigned seen = __ballot_sync(kWarpAll, there);
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const int s = fills % S_, rs = fills % C::kRawStages;
                        ok = wait_all(raw_full(rs), fills / C::kRawStages) && (fills < S_ || wait_all(empty(s), fills / S_ - 1));
                        if (!ok) break;
                        if (kv == 0) {
                            if (lane == 0) masks[entry * 4 + row / 32] = seen;
                            scales[entry * 2 * kSharedTokens + row] = ks;
                            scales[(entry * 2 + 1) * kSharedTokens + row] = vs;
                        }
                        const uint4* const from = reinterpret_cast<const uint4*>(gen + C::kRawAt + rs * C::kRaw + row * hd);
                        uint8_t* const to = gen + s * C::kBuf + row * 128;
                        int ch = ch0;
#pragma unroll 4
                        for (int c = 0; c < chunks; ++c) {
                            const uint4 x = there ? from[ch] : make_uint4(0, 0, 0, 0);
                            uint32_t o[8];
                            if (kv) {
                                widen<kCodes, kBfV>(x.x, o[0], o[1]);
                                widen<kCodes, kBfV>(x.y, o[2], o[3]);
                                widen<kCodes, kBfV>(x.z, o[4], o[5]);
                                widen<kCodes, kBfV>(x.w, o[6], o[7]);
                            } else {
                                widen<kCodes, kBfQ>(x.x, o[0], o[1]);
                                widen<kCodes, kBfQ>(x.y, o[2], o[3]);
                                widen<kCodes, kBfQ>(x.z, o[4], o[5]);
                                widen<kCodes, kBfQ>(x.w, o[6], o[7]);
                            }
                            uint8_t* const slab = to + (ch / 4) * C::kSlab;
                            const int place = 2 * (ch % 4);
                            *reinterpret_cast<uint4*>(slab + ((place ^ (row & 7)) * 16)) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4*>(slab + (((place + 1) ^ (row & 7)) * 16)) = make_uint4(o[4], o[5], o[6], o[7]);
                            if (++ch == chunks) ch = 0;
                        }
                        fence_async_smem();
                        mbar_arrive(full(s));
                        mbar_arrive(raw_empty(rs));
                        ++fills;
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------------------ softmax: two threads a query row (TMEM lane), each
        // with half of a block's tokens
        const int slot = warp / 8, half = warp / 4 % 2, quarter = warp % 4, row = quarter * 32 + lane;
        const uint32_t both = pair_full(4 * slot + quarter);
        const uint32_t lane_at = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_at = lane_at + slot * 128, o_at = lane_at + kOCol + slot * kDim;
        constexpr float kRowLift = kBfV ? 0.f : kLift;
        const bool down = A.scale_log2 < 0.f;
        const int my_b = row / gh, my_j = row - my_b * gh;             // row of the tile's part, head of the group
        int count = 0, blocks = 0, met = 0;                            // blocks of the slot, of all; with the pair's maximum
        bool ok = true;
        Piece p = first;
        for (; ok && piece_at(A, p); next_piece(A, p)) {
            const bool alternate = alternates(p.T);
            const int step = alternate ? kSlots : 1;
            // warps whose rows are none pass on at once: what is in their lanes stays in their lanes
            const bool active = quarter * 32 < min(A.s.lane_rows, p.T.rows - (alternate ? 0 : slot * A.s.lane_rows)) * gh;
            float m = -FLT_MAX, l = 0.f;
            bool begun = false;
            for (int k = alternate ? slot : 0; k < p.n; k += step) {
                const int entry = (blocks + k) % C::kRing;
                ok = wait_all(s_full(slot), count);
                if (!ok) break;
                if (!active) {
                    mbar_arrive(p_full(slot));
                    ++count;
                    continue;
                }
                tc_fence_after();
                const uint4 mask = *reinterpret_cast<const uint4*>(masks + entry * 4);
                const bool part = (mask.x & mask.y & mask.z & mask.w) != kWarpAll;     // some rows are no tokens
                const float* const ks = scales + entry * 2 * kSharedTokens;
                const float* const vs = ks + kSharedTokens;
                // the scores of 32 tokens, times the sign of the scale
                auto scores = [&](int c, float (&v)[32]) {
                    uint32_t x[32];
                    tmem_ld_32x32b_x32(s_at + 32 * c, x);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(x[i]);
                    if (kCodes) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(ks + 32 * c + i);
                            mul2(v[i], v[i + 1], v[i], v[i + 1], f.x, f.y);
                            mul2(v[i + 2], v[i + 3], v[i + 2], v[i + 3], f.z, f.w);
                        }
                    }
                    if (down) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = -v[i];
                    }
                    return masks[entry * 4 + c];
                };
                float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // fmaxf passes over NaN, which reaches the sums
#pragma unroll 1
                for (int c = 2 * half; c < 2 * half + 2; ++c) {
                    float v[32];
                    const uint32_t tokens = scores(c, v);
                    if (part) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(tokens >> i & 1)) v[i] = -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) most[i & 3] = fmaxf(most[i & 3], v[i]);
                }
                const float scale = fabsf(A.scale_log2);
                const float mine = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
                tops[(2 * slot + half) * kSharedLanes + row] = mine;
                mbar_arrive(both);
                ok = wait_all(both, met++);
                if (!ok) break;
                const float top = fmaxf(mine, tops[(2 * slot + 1 - half) * kSharedLanes + row]) * scale;
                const bool moved = top > m + kSlack;
                if (!begun) {
                    if (moved) m = top;
                    begun = true;
                } else if (__any_sync(kWarpAll, moved)) {
                    // the sums so far come down; the last products with P are complete
                    ok = wait_all(o_done(slot), count - 1);
                    if (!ok) break;
                    tc_fence_after();
                    const float turn = moved ? ex2(m - top) : 1.f;
                    if (moved) {
                        m = top;
                        l *= turn;
                    }
#pragma unroll 1
                    for (int d = 16 * half; d < hd; d += 32) {
                        uint32_t o[16];
                        tmem_ld_32x32b_x16(o_at + d, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * turn);
                        tmem_st_32x32b_x16(o_at + d, o);
                    }
                }
                // weights, 32 tokens at a time: their first parts and their second ones go where these tokens' scores were
                const float less = m - kRowLift;
                float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                for (int c = 2 * half; c < 2 * half + 2; ++c) {
                    float w[32];
                    const uint32_t tokens = scores(c, w);
#pragma unroll
                    for (int i = 0; i < 32; ++i) w[i] = ex2(fmaf(w[i], scale, -less));
                    if (part) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(tokens >> i & 1)) w[i] = 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) sums[i & 3] += w[i];
                    if (kCodes) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(vs + 32 * c + i);
                            mul2(w[i], w[i + 1], w[i], w[i + 1], f.x, f.y);
                            mul2(w[i + 2], w[i + 3], w[i + 2], w[i + 3], f.z, f.w);
                        }
                    }
                    uint32_t hi[16], lo[16];
                    split<kBfV>(w, hi, lo);
                    tmem_st_32x32b_x16(s_at + 32 * c, hi);
                    tmem_st_32x32b_x16(s_at + 32 * c + 16, lo);
                }
                l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(p_full(slot));
                ++count;
            }
            if (!ok) break;
            // ---- the piece's records
            float* rec = nullptr;
            const int b = (alternate ? 0 : slot * A.s.lane_rows) + my_b;
            if (my_b < A.s.lane_rows && b < p.T.rows)
                rec = p.i == 0 ? A.s.own + ((alternate ? slot * A.s.own_records : 0) + (int64_t)(p.T.row0 + b) * A.heads + p.h * gh + my_j) *
                                               A.s.pitch
                               : A.s.cut + (((int64_t)blockIdx.x * 2 + slot) * kSharedLanes + row) * A.s.pitch;
            if (begun) {
                ok = wait_all(o_done(slot), count - 1);
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int d = 32 * half; d < hd; d += 64) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(o_at + d, o);
                    if (rec) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (d + i < hd) *reinterpret_cast<uint4*>(rec + d + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
            }
            tc_fence_before();
            if (rec) {
                if (half == 0) rec[A.s.pitch - 4] = m == -FLT_MAX ? m : m - kRowLift;
                rec[A.s.pitch - 3 + half] = l;
            }
            blocks += p.n;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == C::kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------- the join
// kTeam warps a row's head: the records of its unit's pieces and of its other tokens, in the order of the pieces, so that
// results do not depend on timing.  Bound: the records' bytes (from L2), 8 records at a time and warp.  Up to
// 4 query rows an SM, of many pieces each, get a CTA each: 16 rows of 8 heads behind one prefix of 64k
// 45 us in all, with a warp each 86; 64 rows of 32 heads behind 4k 58 and 42, so they get a warp.
constexpr int kJoinWarps = 8;

template <bool kBf, int kTeam, bool kWide>
__global__ void __launch_bounds__(kJoinWarps * 32, kWide ? 2 : 3) join_kernel(const AttendArgs A) {
    constexpr int kVals = kWide ? 8 : 4;                               // a lane's: dims 4 lane on, and with kWide 128 + 4 lane on
    pdl_enter();
    const SharedD& S = A.shared;
    const int lane = threadIdx.x & 31, hd = A.pages.head_dim, pitch = S.pitch;
    __shared__ float parts[kTeam > 1 ? kTeam : 1][kTeam > 1 ? 2 + kVals : 1][32];
    const int member = threadIdx.x / 32 % kTeam;
    const int64_t place = (int64_t)blockIdx.x * (kJoinWarps / kTeam) + threadIdx.x / 32 / kTeam;
    if (place >= S.own_records) return;
    const int b = (int)(place / A.heads), h = (int)(place - (int64_t)b * A.heads);
    const int tile = S.row_tile[b];
    if (S.row_from[b] == 0) return;                                    // it shares nothing and is written already
    const float* const rest = S.rest + place * pitch;
    const SharedTile T = S.tiles[tile];
    const int head = h / A.group, part = (b - T.row0) / S.lane_rows;
    const int at = (b - T.row0 - part * S.lane_rows) * A.group + h - head * A.group;
    const int64_t first = T.first + (int64_t)head * T.blocks, run = S.head->run, c0 = first / run;
    const int two = shared_alternates(T.rows, S.lane_rows, S.slots) ? 2 : 1;
    const int pieces = (int)((first + T.blocks - 1) / run - c0 + 1) * two;
    auto record = [&](int p) -> const float* {                          // p = pieces: the rest
        if (p >= pieces) return rest;
        const int64_t c = c0 + (two == 2 ? p >> 1 : p);
        const int slot = two == 2 ? p & 1 : part;
        return c == c0 ? S.own + ((two == 2 ? slot * S.own_records : 0) + place) * pitch
                       : S.cut + ((c * 2 + slot) * kSharedLanes + at) * pitch;
    };
    const bool second = kWide && lane * 4 + 128 < hd;
    float top = -FLT_MAX, sum = 0.f, v[kVals];
#pragma unroll
    for (int i = 0; i < kVals; ++i) v[i] = 0.f;
    const int per = (pieces + kTeam) / kTeam, end = min(pieces + 1, per * (member + 1));
    for (int p0 = per * member; p0 < end; p0 += 32) {
        // a lane a record: its maximum and sum; one without a score above -inf holds no values
        const int p = p0 + lane;
        float4 ml = make_float4(-FLT_MAX, 0.f, 0.f, 0.f);
        if (p < end) ml = __ldcg(reinterpret_cast<const float4*>(record(p) + pitch - 4));
        float m = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kWarpAll, m, o));
        const float now = fmaxf(top, m), turn = now == top ? 1.f : ex2(top - now);
        const bool empty = ml.x == -FLT_MAX && ml.y + ml.z == 0.f;     // (a sum can be NaN without a maximum)
        const float weight = empty ? 0.f : ex2(ml.x - now);
        float l = empty ? 0.f : (ml.y + ml.z) * weight;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(kWarpAll, l, o);
        sum = sum * turn + l;
#pragma unroll
        for (int i = 0; i < kVals; ++i) v[i] *= turn;
        top = now;
        const unsigned there = __ballot_sync(kWarpAll, !empty);
        const int count = min(32, end - p0);
        constexpr int kAtOnce = 8;
        for (int q0 = 0; q0 < count; q0 += kAtOnce) {
            float4 x[kAtOnce], y[kWide ? kAtOnce : 1];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                x[i] = y[kWide ? i : 0] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (q0 + i < count && there >> (q0 + i) & 1 && lane * 4 < hd) {
                    const float* rec = record(p0 + q0 + i);
                    x[i] = __ldcg(reinterpret_cast<const float4*>(rec) + lane);
                    if (second) y[kWide ? i : 0] = __ldcg(reinterpret_cast<const float4*>(rec + 128) + lane);
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const float w = __shfl_sync(kWarpAll, weight, q0 + i);
                v[0] += x[i].x * w, v[1] += x[i].y * w, v[2] += x[i].z * w, v[3] += x[i].w * w;
                if (kWide) {
                    const float4 z = y[kWide ? i : 0];
                    v[kVals - 4] += z.x * w, v[kVals - 3] += z.y * w, v[kVals - 2] += z.z * w, v[kVals - 1] += z.w * w;
                }
            }
        }
    }
    if (kTeam > 1) {
        parts[member][0][lane] = top;
        parts[member][1][lane] = sum;
#pragma unroll
        for (int i = 0; i < kVals; ++i) parts[member][2 + i][lane] = v[i];
        __syncthreads();
        if (member) return;
#pragma unroll
        for (int w = 1; w < kTeam; ++w) top = fmaxf(top, parts[w][0][lane]);
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < kVals; ++i) v[i] = 0.f;
#pragma unroll
        for (int w = 0; w < kTeam; ++w) {                              // (a warp without a score has zeros)
            const float turn = ex2(parts[w][0][lane] - top);
            sum += parts[w][1][lane] * turn;
#pragma unroll
            for (int i = 0; i < kVals; ++i) v[i] += parts[w][2 + i][lane] * turn;
        }
    }
    using H = typename Half<kBf>::type;
    const float gain = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* const out = static_cast<uint16_t*>(A.out) + place * hd + lane * 4;
    if (lane * 4 < hd) *reinterpret_cast<uint2*>(out) = make_uint2(pack2<H>(v[0] * gain, v[1] * gain), pack2<H>(v[2] * gain, v[3] * gain));
    if (second)
        *reinterpret_cast<uint2*>(out + 128) =
            make_uint2(pack2<H>(v[kVals - 4] * gain, v[kVals - 3] * gain), pack2<H>(v[kVals - 2] * gain, v[kVals - 1] * gain));
    if (A.lse && lane == 0) A.lse[place] = sum == 0.f ? -INFINITY : (top + log2f(sum)) / kLog2e;
}

template <int kCodes, bool kBfQ, bool kBfV, int kDim> int launch_shared(const SharedArgs& A, const Maps& maps, cudaStream_t st) {
    using C = Cfg<kCodes, kDim>;
    return launch(shared_kernel<kCodes, kBfQ, kBfV, kDim>, dim3((unsigned)A.grid), dim3(C::kThreads), (size_t)C::kSmem, st,
                  "epq_paged_attend_shared", A, maps);
}
template <int kCodes, bool kBfQ, bool kBfV> int launch_shared_d(const SharedArgs& A, const Maps& maps, cudaStream_t st) {
    const int hd = A.pages.head_dim;
    if (hd <= 64) return launch_shared<kCodes, kBfQ, kBfV, 64>(A, maps, st);
    if (hd <= 128) return launch_shared<kCodes, kBfQ, kBfV, 128>(A, maps, st);
    if constexpr (kCodes == kNone) return launch_shared<kCodes, kBfQ, kBfV, 256>(A, maps, st);
    return EPQ_EUNSUPPORTED;               // (may_share)
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Where things lie in the workspace, behind the attention's own part.
struct Layout {
    int lane_rows, max_tiles, slots, pitch;
    int64_t head, tiles, row_tile, row_from, rest, own, cut, bytes;
};
Layout layout_of(const PagesD& P, int64_t batch, int heads, int64_t groups, int64_t behind) {
    Layout L;
    const int dim = P.head_dim <= 64 ? 64 : P.head_dim <= 128 ? 128 : 256, group = heads / P.kv_heads;
    L.slots = dim == 256 ? 1 : 2;
    L.pitch = dim + 4;
    L.lane_rows = kSharedLanes / group;
    const int64_t some = groups < batch / 2 ? groups : batch / 2;      // groups of two rows or more
    L.max_tiles = (int)(batch / (L.slots * L.lane_rows) + some + 1);
    L.head = behind;
    L.tiles = L.head + 256;
    L.row_tile = align256(L.tiles + L.max_tiles * (int64_t)sizeof(SharedTile));
    L.row_from = align256(L.row_tile + batch * 4);
    L.rest = align256(L.row_from + batch * 4);
    L.own = align256(L.rest + batch * heads * L.pitch * 4);
    L.cut = align256(L.own + 2 * batch * heads * L.pitch * 4);
    L.bytes = L.cut + (int64_t)device_sms() * 2 * kSharedLanes * L.pitch * 4;
    return L;
}

// Whether a batch can share anything (that is worth it): groups of two rows or more whose query heads fit a tile, enough
// tokens that the tables could hold, and pages that the copies of rows take: boxes of 8 rows or more, which lie side by
// side in the 128-byte swizzle.  8-bit heads above 128 have no room for their 16-bit form.
bool may_share(const PagesD& P, int64_t batch, int heads, int64_t groups, bool always) {
    const int64_t most = (int64_t)P.max_pages * P.page_size;
    const int64_t pool = P.pages > (1LL << 40) / P.page_size ? 1LL << 40 : P.pages * P.page_size;   // (all tables together)
    const int64_t tokens = most < pool ? most : pool;
    return groups > 0 && batch > 1 && heads / P.kv_heads <= kSharedLanes && P.page_size % 8 == 0 &&
           (P.format == EPQ_CACHE_SAME || P.head_dim <= 128) &&
           (always || (double)batch * (double)tokens * (double)reckon(P).row_token > (double)kFixed);
}
// Whether rows of q can be copied as boxes (other views take the plain form).
bool boxes_of(const epq_heads& q, int64_t batch) {
    auto good = [](int64_t stride) { return stride > 0 && stride % 8 == 0 && stride < (1LL << 36); };
    return (uintptr_t)q.data % 16 == 0 && good(q.stride_row) && (q.heads == 1 || good(q.stride_head));
}

}  // namespace

int shared_read_device_error(int* flag) {
    int bad = 0, behind = 0;
    if (cudaMemcpyFromSymbol(&bad, g_shared_error, sizeof(int)) != cudaSuccess)
        return check_launch("read shared attention error flag");
    const int rc = attend_shared_read_device_error(&behind);
    *flag = bad | behind;
    return rc;
}
int shared_read_timeout(int* flag) {
    if (cudaMemcpyFromSymbol(flag, g_shared_timeout, sizeof(int)) != cudaSuccess)
        return check_launch("read shared attention error flag");
    return EPQ_OK;
}

}  // namespace paged
}  // namespace epq

using namespace epq;
using namespace epq::paged;

extern "C" {

int64_t epq_paged_attend_shared_workspace_bytes(const epq_pages* pages, int64_t batch, int32_t heads, int64_t groups,
                                                int32_t always) {
    const char* const who = "epq_paged_attend_shared_workspace_bytes";
    if (groups < 0) return set_error(EPQ_EINVAL, "%s: groups=%lld", who, (long long)groups);
    const int64_t behind = attend_bytes(who, pages, batch, heads);
    if (behind < 0) return behind;
    PagesD P;
    make_pages(pages, &P, who);
    if (batch > 65536) return set_error(EPQ_EUNSUPPORTED, "%s: batch=%lld", who, (long long)batch);
    if (!may_share(P, batch, heads, groups, always != 0)) return behind;
    return layout_of(P, batch, heads, groups, align256(behind)).bytes;
}

int epq_paged_attend_shared(const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                            int64_t batch, const int32_t* starts, const int64_t* prefix, int64_t groups, int32_t always,
                            float scale, void* out, float* lse, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* const who = "epq_paged_attend_shared";
    if (groups < 0 || groups > INT32_MAX - 1 || (groups && (!starts || !prefix)))
        return set_error(EPQ_EINVAL, "%s: groups=%lld, or NULL starts or prefix", who, (long long)groups);
    AttendArgs A = {};
    int cols;
    bool ready;
    const int rc = make_attend(who, pages, q, seq, lengths, batch, scale, out, lse, dtype, workspace, workspace_bytes, &A, &cols,
                               &ready);
    if (rc != EPQ_OK || !ready) return rc;
    const PagesD& P = A.pages;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!may_share(P, batch, A.heads, groups, always != 0) || !boxes_of(*q, batch)) {
        A.starts = starts;
        A.prefix = prefix;
        A.groups = (int)groups;
        return launch_attend_plain(A, cols, st);
    }
    const int64_t behind = align256(attend_bytes(who, pages, batch, A.heads));
    const Layout L = layout_of(P, batch, A.heads, groups, behind);
    if (workspace_bytes < L.bytes)
        return set_error(EPQ_EWORKSPACE, "%s: workspace of %lld bytes (need %lld)", who, (long long)workspace_bytes,
                         (long long)L.bytes);
    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    SharedArgs S = {};
    S.pages = P;
    S.s.head = reinterpret_cast<SharedHead*>(ws + L.head);
    S.s.tiles = reinterpret_cast<SharedTile*>(ws + L.tiles);
    S.s.row_tile = reinterpret_cast<int32_t*>(ws + L.row_tile);
    S.s.row_from = reinterpret_cast<int32_t*>(ws + L.row_from);
    S.s.rest = reinterpret_cast<float*>(ws + L.rest);
    S.s.own = reinterpret_cast<float*>(ws + L.own);
    S.s.cut = reinterpret_cast<float*>(ws + L.cut);
    S.s.own_records = batch * A.heads;
    S.s.pitch = L.pitch;
    S.s.slots = L.slots;
    S.s.lane_rows = L.lane_rows;
    S.seq = seq;
    S.lengths = lengths;
    S.starts = starts;
    S.prefix = prefix;
    S.cost = reckon(P);
    S.always = always != 0;
    S.batch = (int)batch;
    S.groups = (int)groups;
    S.heads = A.heads;
    S.group = A.group;
    S.max_tiles = L.max_tiles;
    S.grid = device_sms();
    S.scale_log2 = A.scale_log2;
    S.box_rows = kSharedTokens;
    while (P.page_size % S.box_rows) S.box_rows /= 2;
    Maps maps;
    const bool codes = P.format != EPQ_CACHE_SAME;
    int e = make_tmap_3d(&maps.q, q->data, 2, {P.head_dim, q->heads, batch}, q->heads > 1 ? q->stride_head : P.head_dim,
                         q->stride_row, {64, A.group, L.lane_rows}, true, who);
    for (int i = 0; e == EPQ_OK && i < 2; ++i)
        e = make_tmap_3d(i ? &maps.v : &maps.k, i ? P.v : P.k, codes ? 1 : 2,
                         {P.head_dim, (int64_t)P.kv_heads * P.page_size, P.pages}, P.head_dim, P.page_stride,
                         {codes ? P.head_dim : 64, S.box_rows, 1}, !codes, who);
    if (e != EPQ_OK) return e;
    e = launch(plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, who, S);
    if (e != EPQ_OK) return e;
    const bool bf = dtype == EPQ_BF16;
    if (P.format == EPQ_CACHE_INT8)
        e = bf ? launch_shared_d<kInts, true, true>(S, maps, st) : launch_shared_d<kInts, false, true>(S, maps, st);
    else if (P.format == EPQ_CACHE_FP8)
        e = bf ? launch_shared_d<kFloats, true, true>(S, maps, st) : launch_shared_d<kFloats, false, true>(S, maps, st);
    else
        e = bf ? launch_shared_d<kNone, true, true>(S, maps, st) : launch_shared_d<kNone, false, false>(S, maps, st);
    if (e != EPQ_OK) return e;
    A.shared = S.s;
    e = attend_behind_shared(A, cols, st);
    if (e != EPQ_OK) return e;
    const bool teams = S.s.own_records <= 4LL * S.grid;
    const dim3 grid((unsigned)cdiv(S.s.own_records, teams ? 1 : kJoinWarps)), threads(kJoinWarps * 32);
    auto join = [&](auto kern) { return launch(kern, grid, threads, 0, st, who, A); };
    if (P.head_dim > 128) {
        if (teams) return bf ? join(join_kernel<true, kJoinWarps, true>) : join(join_kernel<false, kJoinWarps, true>);
        return bf ? join(join_kernel<true, 1, true>) : join(join_kernel<false, 1, true>);
    }
    if (teams) return bf ? join(join_kernel<true, kJoinWarps, false>) : join(join_kernel<false, kJoinWarps, false>);
    return bf ? join(join_kernel<true, 1, false>) : join(join_kernel<false, 1, false>);
}

}  // extern "C"
