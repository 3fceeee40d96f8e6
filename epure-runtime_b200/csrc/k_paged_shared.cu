// Attention of one new token a row where rows share a prefix (epq_paged_attend_shared): the plan
// and the shared tokens.  (The rest: k_paged_attn_shared.cu; what they hand on: epq_shared.cuh.)
//
// Rows of a group that see tokens [0, L) all alike are one attention of many query rows over one
// set of keys: with r rows and g query heads a key head, r g rows over L tokens, 4 r g flops a
// cached value.  So it is the tensor cores' (tcgen05) work, and what is read once is read for
// r rows.
//
// Plan (one CTA): groups are cut into tiles of up to 256 query rows (128 where head_dim > 128);
// L of a tile is its prefix, or the shortest of its rows' lengths.  No score needs a mask by row
// then: what a row sees beyond L is its own part, and a value there that is not finite stays in
// the rows that see it.  Where the whole batch would save less than kWorth bytes of reading,
// nothing is shared.
//
// Shared part.  Blocks of 128 tokens of all units (tile, key head) are dealt out to the CTAs in
// equal runs, one CTA an SM, and each piece of a unit leaves its sums as records.  In a CTA:
//   * 4 loader warps look up pages and bring rows of K and V into a ring of shared-memory stages
//     in the 128-byte swizzle, 16-bit rows by cp.async, codes of 8-bit caches through registers
//     to 16 bits (exact);
//   * one thread issues the products: S = Q K^T (Q, K in shared memory) and O += P V (P in tensor
//     memory, V as the MN-major operand);
//   * 4 warps a slot take a row a thread: maximum, weights, sum; P goes back in place of S.
// Two slots (S and O in tensor memory: all of its 512 columns) keep the products of one under
// the softmax of the other: two tiles of 128 rows over the same block, or, for units of up to
// 128 rows, one tile whose blocks alternate.
//
// Precision.  Weights are the sum of two 16-bit values, as in k_paged_attn.cu: one rounding of
// them is as large as the result's own (products with P cost twice as much, 3 units of tensor
// time a block instead of 2).  8-bit caches: keys are exact in q's type, values and weights are
// bf16, whose range takes any scale; a key's scale multiplies its score, a value's its weight.
// The running maximum moves only when a score passes it by 2^8.
#include "epq_attend.cuh"
#include "epq_sm100.cuh"

namespace epq {
namespace paged {

int attend_behind_shared(const AttendArgs& A, int cols, cudaStream_t st);
int attend_shared_read_device_error(int* flag);

namespace {

__device__ int g_shared_error = 0;         // kBadPosition, kBadPage
__device__ int g_shared_timeout = 0;       // a bounded wait gave up

constexpr unsigned kWarpAll = 0xffffffffu;
constexpr int kPlanThreads = 1024;
constexpr uint32_t kWaitLimit = 1u << 22;
constexpr int kSmemLimit = 232448;         // 227 KB a CTA
// Bytes of reading that sharing has to save: the plan and the shared part's launch cost about as
// much as these take from HBM.
constexpr int64_t kWorth = 32 << 20;

struct SharedArgs {
    PagesD pages;
    SharedD s;
    const void* q;
    int64_t q_row, q_head;
    const int32_t* seq;
    const int64_t* lengths;
    const int32_t* starts;
    const int64_t* prefix;
    int64_t token_bytes;                   // of one cached token: keys, values, scales
    int batch, groups, heads, group, tile_rows, max_tiles, grid, q_aligned;
    float scale_log2;
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
    int64_t w = shared[lane];
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
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const PagesD& P = A.pages;
    const int64_t cap = (int64_t)P.max_pages * P.page_size;
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
    for (int g = tid; g < A.groups; g += kPlanThreads)
        good = good && A.starts[g] >= 0 && A.starts[g] <= A.starts[g + 1] && A.starts[g + 1] <= A.batch && A.prefix[g] >= 0 &&
               A.prefix[g] <= cap;
    good = __syncthreads_and(good);
    if (!good && tid == 0) atomicOr(&g_shared_error, kBadPosition);
    int64_t tiles = 0;
    for (int g0 = 0; good && g0 < A.groups; g0 += kPlanThreads) {
        const int g = g0 + tid;
        const int from = g < A.groups ? A.starts[g] : 0, rows = g < A.groups ? A.starts[g + 1] - from : 0;
        const int count = rows >= 2 ? (rows + A.tile_rows - 1) / A.tile_rows : 0;
        int64_t all;
        int64_t at = tiles + block_scan(count, scratch, &all) - count;
        for (int i = 0; i < count && at < A.max_tiles; ++i, ++at) {
            SharedTile T = {};
            T.row0 = from + i * A.tile_rows;
            T.rows = min(A.tile_rows, from + rows - T.row0);
            T.group = g;
            A.s.tiles[at] = T;
        }
        tiles += all;
    }
    tiles = min(tiles, (int64_t)A.max_tiles);
    __syncthreads();
    // what each tile's rows share
    int64_t saved = 0;
    for (int t = warp; t < tiles; t += kPlanThreads / 32) {
        SharedTile T = A.s.tiles[t];
        int active = 0, first = INT32_MAX;
        int64_t least = A.prefix[T.group];
        for (int r = lane; r < T.rows; r += 32) {
            if (!counts(T.row0 + r)) continue;
            ++active;
            first = min(first, r);
            least = min(least, A.lengths[T.row0 + r]);
        }
        active = __reduce_add_sync(kWarpAll, active);
        first = __reduce_min_sync(kWarpAll, first);
        least = __reduce_min_sync(kWarpAll, (int)least);
        if (lane == 0) {
            const int b = T.row0 + first;
            T.seq = active < 2 ? 0 : A.seq ? A.seq[b] : b;
            T.tokens = active < 2 ? 0 : (int)least;
            T.blocks = (T.tokens + kSharedTokens - 1) / kSharedTokens;
            A.s.tiles[t] = T;
            saved += (int64_t)(active - 1) * T.tokens;
        }
    }
    int64_t all_saved;
    block_scan(saved, scratch, &all_saved);
    const bool worth = all_saved * A.token_bytes >= kWorth;
    // places of the units
    int64_t total = 0;
    for (int t0 = 0; t0 < tiles; t0 += kPlanThreads) {
        const int t = t0 + tid;
        const int64_t mine = worth && t < tiles ? (int64_t)A.s.tiles[t].blocks * P.kv_heads : 0;
        int64_t all;
        const int64_t at = total + block_scan(mine, scratch, &all) - mine;
        if (t < tiles) {
            A.s.tiles[t].first = at;
            if (!worth) A.s.tiles[t].blocks = 0;
        }
        total += all;
    }
    if (tid == 0) *A.s.head = {total, (int)max((int64_t)1, (total + A.grid - 1) / A.grid), (int)tiles};
    __syncthreads();
    for (int t = warp; worth && t < tiles; t += kPlanThreads / 32) {
        const SharedTile T = A.s.tiles[t];
        for (int r = lane; T.blocks && r < T.rows; r += 32) {
            const int b = T.row0 + r;
            A.s.row_tile[b] = t;
            A.s.row_from[b] = counts(b) ? T.tokens : 0;
        }
    }
}

// ---------------------------------------------------------------- the shared tokens
enum Codes { kNone = 0, kInts = 1, kFloats = 2 };

template <int kCodes, int kDim> struct Cfg {
    static constexpr int kSlots = kDim == 256 ? 1 : 2;
    static constexpr int kLoaderWarps = 4;
    static constexpr int kMmaWarp = kSlots * 4;
    static constexpr int kThreads = (kMmaWarp + 1 + kLoaderWarps) * 32;
    static constexpr int kBuf = kSharedTokens * kDim * 2;              // K or V of a block
    static constexpr int kSlab = kSharedTokens * 128;                  // 64 values of each of its rows
    static constexpr int kQ = kSlots * kSharedLanes * kDim * 2;
    static constexpr int kRing = 8;                                    // blocks whose masks and scales are kept
    static constexpr int kScales = kCodes ? kRing * 2 * kSharedTokens * 4 : 0;
    static constexpr int kPagesAt = kScales, kMasksAt = kPagesAt + 2 * kSharedTokens * 4, kBarsAt = kMasksAt + kRing * 16;
    static constexpr int kMisc = kBarsAt + 224;
    static constexpr int kFit = (kSmemLimit - 1024 - kMisc - kQ) / kBuf;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kQAt = kStages * kBuf, kMiscAt = kQAt + kQ, kSmem = 1024 + kMiscAt + kMisc;
    static_assert(kStages >= 2 && kSmem <= kSmemLimit, "shared memory");
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

__device__ __forceinline__ void cp_wait_all_but(int left) {            // groups that may still be on their way
    switch (left) {
        case 0: cp_wait<0>(); break;
        case 1: cp_wait<1>(); break;
        case 2: cp_wait<2>(); break;
        default: cp_wait<3>(); break;
    }
}

// kBfQ: S in bf16 (else f16); kBfV: P and V in bf16 (else f16).
template <int kCodes, bool kBfQ, bool kBfV, int kDim>
__global__ void __launch_bounds__(Cfg<kCodes, kDim>::kThreads, 1) shared_kernel(const SharedArgs A) {
    using C = Cfg<kCodes, kDim>;
    using namespace sm100;
    using TQ = typename Half<kBfQ>::type;
    using TV = typename Half<kBfV>::type;
    constexpr int S_ = C::kStages, kSlots = C::kSlots;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PagesD& P = A.pages;
    const int hd = P.head_dim, gh = A.group, ps = P.page_size;

    const SharedHead head = *A.s.head;
    Piece first;
    first.at = (int64_t)blockIdx.x * head.run;
    first.end = min(head.total, first.at + head.run);
    if (first.at >= head.total) return;

    const uint32_t raw = sm100::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* const gen = smem_raw + (base - raw);
    uint8_t* const misc = gen + C::kMiscAt;
    float* const scales = reinterpret_cast<float*>(misc);              // [kRing][2][128]: of keys, of values
    int32_t* const page_of_row = reinterpret_cast<int32_t*>(misc + C::kPagesAt);       // [2][128], -1: no token
    uint32_t* const masks = reinterpret_cast<uint32_t*>(misc + C::kMasksAt);           // [kRing][4]
    const uint32_t bars = base + C::kMiscAt + C::kBarsAt;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 64u + 8u * s; };
    auto s_full = [&](int s) { return bars + 128u + 8u * s; };
    auto p_full = [&](int s) { return bars + 144u + 8u * s; };
    auto o_done = [&](int s) { return bars + 160u + 8u * s; };
    const uint32_t q_free = bars + 176u, over = bars + 184u, tslot = bars + 192u, looked_up = bars + 208u;
    volatile int* const abortp = reinterpret_cast<volatile int*>(misc + C::kBarsAt + 196);
    volatile int* const where = reinterpret_cast<volatile int*>(misc + C::kBarsAt + 200);
    auto wait = [&](uint32_t bar, uint32_t parity) {
        return mbar_wait_bounded(bar, parity & 1u, abortp, &g_shared_timeout, kWaitLimit);
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < S_; ++s) {
            mbar_init(full(s), C::kLoaderWarps * 32);
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(s_full(s), 2);                                   // the products' end, and the issuing thread
            mbar_init(p_full(s), 128);
            mbar_init(o_done(s), 1);
        }
        mbar_init(q_free, 1);
        mbar_init(over, 1);
        mbar_init(looked_up, C::kLoaderWarps * 32);
        *abortp = 0;
        mbar_init_fence();
    }
    if (warp == C::kMmaWarp) tmem_alloc(tslot, 512);
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
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(misc + C::kBarsAt + 192);
    first.t = *where;
    first.c = 0;
    {
        const SharedTile T = A.s.tiles[first.t];
        first.h = (int)((first.at - T.first) / T.blocks);
    }
    const uint32_t q_at = base + C::kQAt;
    constexpr uint32_t kOCol = kSlots * 128u;                          // S and P of slot s in columns 128 s, O behind them

    if (warp > C::kMmaWarp) {
        // ------------------------------------------------------------ loaders
        const int tid = threadIdx.x - (C::kMmaWarp + 1) * 32;          // 0..127
        // a thread's chunks (16 bytes of a row of the cache): chunk ch of rows row0, row0 + kStep, ...
        constexpr int kChunks = kDim * (kCodes ? 1 : 2) / 16, kStep = 128 / kChunks, kEach = 128 / kStep;
        const int ch = tid % kChunks, row0 = tid / kChunks;
        const bool on = ch * 16 < hd * (kCodes ? 1 : 2);
        int filled = 0, arrived = 0;                                   // stages
        constexpr int kLag = S_ - 2 < 3 ? S_ - 2 : 3;
        bool ok = true;
        auto arrive_to = [&](int most) {                               // all but `most` of the filled stages are there
            if (filled - arrived <= most) return;
            cp_wait_all_but(most);
            fence_async_smem();
            while (filled - arrived > most) mbar_arrive(full(arrived++ % S_));
        };
        auto open = [&]() {                                            // the next stage, once it is free
            const int s = filled % S_;
            bool got = true;
            if (filled >= S_ && !mbar_try_wait(empty(s), ((filled / S_) - 1) & 1)) {
                if (!kCodes) arrive_to(0);                             // (the one that frees it may wait for them)
                got = wait(empty(s), (filled / S_) - 1);
            }
            ok = __all_sync(kWarpAll, got);
            return base + s * C::kBuf;
        };
        // this thread's row of the next block: its page's number is on its way
        int32_t next_page = -1;
        auto look_up = [&](const SharedTile& T, int block) {
            const int t = block * kSharedTokens + tid;
            next_page = t < T.tokens ? P.table[(int64_t)T.seq * P.table_stride + P.page_of(t)] : -1;
            return t < T.tokens;
        };
        bool next_on = false;
        Piece p = first;
        int blocks = 0;                                                // before this piece
        for (; ok && piece_at(A, p); next_piece(A, p)) {
            const int q_rows = p.T.rows * gh;
            if (p.c) {
                if (!kCodes) arrive_to(0);
                ok = __all_sync(kWarpAll, wait(q_free, p.c - 1));
                if (!ok) break;
            }
            // q, with the first keys: rows (row of the batch, head of the group)
            {
                constexpr int kQChunks = kDim / 8, kQStep = 128 / kQChunks;
                const int qc = tid % kQChunks, inv = (65536 + gh - 1) / gh;
                const int rows = kSlots == 2 && !shared_alternates(q_rows, kSlots) ? 256 : 128;
                const bool dims = qc * 8 < hd;
                for (int r = tid / kQChunks; r < rows; r += kQStep) {
                    const int b = (r * inv) >> 16, j = r - b * gh;
                    const bool there = dims && r < q_rows;
                    const uint16_t* from = static_cast<const uint16_t*>(A.q) +
                                           (there ? (p.T.row0 + b) * A.q_row + (p.h * gh + j) * A.q_head + qc * 8 : 0);
                    const uint32_t to = q_at + (r / 128) * (128 * kDim * 2) + (qc / 8) * C::kSlab + (r % 128) * 128 +
                                        (((qc % 8) ^ (r & 7)) * 16);
                    if (A.q_aligned) {
                        cp16(to, from, there ? 16 : 0);
                    } else {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = there ? reinterpret_cast<const uint32_t*>(from)[i] : 0u;
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                                     : "memory");
                    }
                }
                if (kCodes) {
                    cp_commit();
                    cp_wait<0>();
                }
            }
            next_on = look_up(p.T, p.i);
            for (int k = 0; ok && k < p.n; ++k) {
                const int block = p.i + k, entry = (blocks + k) % C::kRing;
                // pages of the block's rows for all loaders; which rows are tokens for the softmax
                int32_t page = next_page;
                if (next_on && (page < 0 || page >= P.pages)) {
                    atomicOr(&g_shared_error, kBadPage);
                    page = -1;
                }
                int32_t* const table = page_of_row + ((blocks + k) & 1) * kSharedTokens;
                table[tid] = page;
                const unsigned seen = __ballot_sync(kWarpAll, page >= 0);
                float ks = 0.f, vs = 0.f;
                if (kCodes && page >= 0) {
                    const int t = block * kSharedTokens + tid, slot = t - P.page_of(t) * ps;
                    const int64_t at = page * P.scale_stride + (int64_t)p.h * ps + slot;
                    ks = P.k_scale[at];
                    vs = P.v_scale[at];
                }
                mbar_arrive(looked_up);
                ok = __all_sync(kWarpAll, wait(looked_up, blocks + k));
                if (!ok) break;
                if (k + 1 < p.n) next_on = look_up(p.T, block + 1);
                auto row_at = [&](int r, bool& there) -> int64_t {     // first value of row r of this head
                    const int32_t pg = table[r];
                    const int t = block * kSharedTokens + r, slot = t - P.page_of(t) * ps;
                    there = pg >= 0 && on;
                    return there ? pg * P.page_stride + ((int64_t)p.h * ps + slot) * hd : 0;
                };
                if constexpr (kCodes == kNone) {
                    uint32_t to[2];
                    to[0] = open();
                    if (!ok) break;
                    if (lane == 0) masks[entry * 4 + tid / 32] = seen;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        if (kv) to[1] = open();
                        if (!ok) break;
                        const uint8_t* const pool = kv ? P.v : P.k;
#pragma unroll 4
                        for (int e = 0; e < kEach; ++e) {
                            const int r = row0 + e * kStep;
                            bool there;
                            const int64_t at = row_at(r, there);
                            if (on)
                                cp16(to[kv] + (ch / 8) * C::kSlab + r * 128 + (((ch % 8) ^ (r & 7)) * 16), pool + at * 2 + (there ? ch * 16 : 0),
                                     there ? 16 : 0);
                        }
                        cp_commit();
                        ++filled;
                        arrive_to(kLag);
                    }
                } else {
                    constexpr int kHalf = kEach > 8 ? 8 : kEach;       // chunks in registers at once
                    uint4 x[2][kHalf];
                    auto fetch = [&](int kv, int e0) {
                        const uint8_t* const pool = kv ? P.v : P.k;
#pragma unroll
                        for (int e = 0; e < kHalf; ++e) {
                            bool there;
                            const int64_t at = row_at(row0 + (e0 + e) * kStep, there);
                            x[kv][e] = there ? __ldg(reinterpret_cast<const uint4*>(pool + at) + ch) : make_uint4(0, 0, 0, 0);
                        }
                    };
                    auto put = [&](int kv, int e0, uint32_t to) {
#pragma unroll
                        for (int e = 0; e < kHalf; ++e) {
                            const int r = row0 + (e0 + e) * kStep;
                            const uint32_t w[4] = {x[kv][e].x, x[kv][e].y, x[kv][e].z, x[kv][e].w};
                            uint32_t o[8];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                codes_f16<kCodes == kInts ? kInt8 : kFp8, false>(w[i], o[2 * i], o[2 * i + 1]);
                                if (kv ? kBfV : kBfQ) {                // exact: codes have at most 8 significant bits
#pragma unroll
                                    for (int j = 0; j < 2; ++j) {
                                        const float2 f = unpack2<__half>(o[2 * i + j]);
                                        o[2 * i + j] = pack2<__nv_bfloat16>(f.x, f.y);
                                    }
                                }
                            }
                            if (on) {
                                const uint32_t row = to + (ch / 4) * C::kSlab + r * 128;
#pragma unroll
                                for (int i = 0; i < 2; ++i)
                                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(row + ((((2 * ch + i) % 8) ^ (r & 7)) * 16)),
                                                 "r"(o[4 * i]), "r"(o[4 * i + 1]), "r"(o[4 * i + 2]), "r"(o[4 * i + 3]) : "memory");
                            }
                        }
                    };
                    fetch(0, 0);
                    if (kEach == kHalf) fetch(1, 0);
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const uint32_t to = open();
                        if (!ok) break;
                        if (kv == 0) {
                            if (lane == 0) masks[entry * 4 + tid / 32] = seen;
                            scales[(entry * 2) * kSharedTokens + tid] = ks;
                            scales[(entry * 2 + 1) * kSharedTokens + tid] = vs;
                        }
#pragma unroll
                        for (int e0 = 0; e0 < kEach; e0 += kHalf) {
                            if (kEach != kHalf && (kv || e0)) fetch(kv, e0);
                            put(kv, e0, to);
                        }
                        fence_async_smem();
                        mbar_arrive(full(filled % S_));
                        ++filled;
                    }
                }
            }
            blocks += p.n;
        }
        if (!kCodes) arrive_to(0);
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == C::kMmaWarp) {
        // ------------------------------------------------------------ products
        if (lane == 0) {
            constexpr uint32_t s_desc = idesc_f16<kBfQ, 128, kSharedTokens>();
            constexpr uint32_t o_desc = idesc_f16<kBfV, 128, kDim, false, true>();
            int count[2] = {0, 0};                                     // products with P that a slot has had
            int fills = 0;                                             // stages before this piece
            bool ok = true;
            Piece p = first;
            for (; ok && piece_at(A, p); next_piece(A, p)) {
                const bool alternate = kSlots == 1 || shared_alternates(p.T.rows * gh, kSlots);
                const int items = alternate ? p.n : 2 * p.n;
                // item w is block w (alternate) or w / 2, of slot w % kSlots
                auto scores = [&](int w) {
                    const int slot = w % kSlots, block = alternate ? w : w >> 1, f = fills + 2 * block, s = f % S_;
                    ok = ok && wait(full(s), f / S_);
                    // P of the slot's last item lies where S goes
                    if (count[slot]) ok = ok && wait(o_done(slot), count[slot] - 1);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t q = q_at + (alternate ? 0 : slot * 128 * kDim * 2), k = base + s * C::kBuf;
                    for (int d = 0; d < hd / 16; ++d)
                        mma_f16_ss(tmem + slot * 128, desc_kmajor_sw128(q + (d / 4) * C::kSlab) + 2 * (d % 4),
                                   desc_kmajor_sw128(k + (d / 4) * C::kSlab) + 2 * (d % 4), s_desc, d != 0);
                    mma_commit(s_full(slot));
                    mbar_arrive(s_full(slot));
                    if (alternate || slot == 1) mma_commit(empty(s));
                    if (w == items - 1) mma_commit(q_free);
                };
                auto sums = [&](int w) {
                    const int slot = w % kSlots, block = alternate ? w : w >> 1, f = fills + 2 * block + 1, s = f % S_;
                    ok = ok && wait(full(s), f / S_) && wait(p_full(slot), count[slot]);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t v = base + s * C::kBuf, o = tmem + kOCol + slot * kDim;
                    for (int t = 0; t < kSharedTokens / 16; ++t) {     // 16 tokens: 8 columns of each part of P
                        const uint32_t at = tmem + slot * 128 + 32 * (t / 2) + 8 * (t % 2);
                        const uint64_t d = desc_mnmajor_sw128(v + t * 2048, C::kSlab, 1024);
                        mma_f16_ts(o, at, d, o_desc, w >= kSlots || t != 0);
                        mma_f16_ts(o, at + 16, d, o_desc, 1);
                    }
                    mma_commit(o_done(slot));
                    ++count[slot];
                    if (alternate || slot == 1) mma_commit(empty(s));
                };
                for (int w = 0; w < kSlots && w < items && ok; ++w) scores(w);
                for (int w = 0; w < items && ok; ++w) {
                    sums(w);
                    if (ok && w + kSlots < items) scores(w + kSlots);
                }
                fills += 2 * p.n;
            }
            // every product is complete before tensor memory is released
            mma_commit(over);
            for (uint32_t i = 0; i < kWaitLimit; ++i)
                if (mbar_try_wait(over, 0)) break;
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax: thread = query row = TMEM lane
        const int slot = warp / 4, part = warp & 3, row = part * 32 + lane;
        const uint32_t lane_at = tmem + ((uint32_t)(part * 32) << 16);
        const uint32_t s_at = lane_at + slot * 128, o_at = lane_at + kOCol + slot * kDim;
        constexpr float kRowLift = kBfV ? 0.f : kLift;
        const bool down = A.scale_log2 < 0.f;
        int count = 0, blocks = 0;
        bool ok = true;
        Piece p = first;
        for (; ok && piece_at(A, p); next_piece(A, p)) {
            const int q_rows = p.T.rows * gh;
            const bool alternate = kSlots == 1 || shared_alternates(q_rows, kSlots);
            const int step = alternate ? kSlots : 1;
            float m = -FLT_MAX, l = 0.f;
            bool begun = false;
            for (int k = alternate ? slot : 0; k < p.n; k += step) {
                const int entry = (blocks + k) % C::kRing;
                ok = __all_sync(kWarpAll, wait(s_full(slot), count));
                if (!ok) break;
                tc_fence_after();
                const float* const ks = scales + entry * 2 * kSharedTokens;
                const float* const vs = ks + kSharedTokens;
                // the scores of 32 tokens, without the softmax's scale; those that are no tokens are -inf
                auto scores = [&](int c, float (&v)[32]) {
                    uint32_t x[32];
                    tmem_ld_32x32b_x32(s_at + 32 * c, x);
                    const uint32_t mask = masks[entry * 4 + c];
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float4 f = make_float4(1.f, 1.f, 1.f, 1.f);
                        if (kCodes) f = *reinterpret_cast<const float4*>(ks + 32 * c + i);
                        v[i] = __uint_as_float(x[i]) * f.x;
                        v[i + 1] = __uint_as_float(x[i + 1]) * f.y;
                        v[i + 2] = __uint_as_float(x[i + 2]) * f.z;
                        v[i + 3] = __uint_as_float(x[i + 3]) * f.w;
                    }
                    return mask;
                };
                float top = -INFINITY;                                 // fmaxf passes over NaN, which reaches the sums
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    float v[32];
                    const uint32_t mask = scores(c, v);
                    if (mask == kWarpAll && !down) {
                        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 32; i += 2) t0 = fmaxf(t0, v[i]), t1 = fmaxf(t1, v[i + 1]);
                        top = fmaxf(top, fmaxf(t0, t1));
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (mask >> i & 1) top = fmaxf(top, down ? -v[i] : v[i]);
                    }
                }
                top *= fabsf(A.scale_log2);
                const bool moved = top > m + kSlack;
                if (!begun) {
                    if (moved) m = top;
                    begun = true;
                } else if (__any_sync(kWarpAll, moved)) {
                    // the sums so far come down; the last products with P are complete
                    ok = __all_sync(kWarpAll, wait(o_done(slot), count - 1));
                    if (!ok) break;
                    tc_fence_after();
                    const float turn = moved ? ex2(m - top) : 1.f;
                    if (moved) {
                        m = top;
                        l *= turn;
                    }
#pragma unroll 1
                    for (int d = 0; d < hd; d += 32) {
                        uint32_t x[32];
                        tmem_ld_32x32b_x32(o_at + d, x);
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * turn);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint32_t half[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) half[j] = x[16 * i + j];
                            tmem_st_32x32b_x16(o_at + d + 16 * i, half);
                        }
                    }
                }
                const float less = m - kRowLift;
                float part_l = 0.f;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    float v[32];
                    const uint32_t mask = scores(c, v);
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = ex2(fmaf(v[i], A.scale_log2, -less));
                    if (mask != kWarpAll) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(mask >> i & 1)) v[i] = 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[i & 3] += v[i];
                    part_l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    if (kCodes) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(vs + 32 * c + i);
                            v[i] *= f.x, v[i + 1] *= f.y, v[i + 2] *= f.z, v[i + 3] *= f.w;
                        }
                    }
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        hi[i] = pack2<TV>(v[2 * i], v[2 * i + 1]);
                        const float2 back = unpack2<TV>(hi[i]);
                        lo[i] = pack2<TV>(v[2 * i] - back.x, v[2 * i + 1] - back.y);
                    }
                    tmem_st_32x32b_x16(s_at + 32 * c, hi);
                    tmem_st_32x32b_x16(s_at + 32 * c + 16, lo);
                }
                l += part_l;
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(p_full(slot));
                ++count;
            }
            if (!ok) break;
            // ---- the piece's records
            const int at_row = alternate ? row : slot * kSharedLanes + row;
            if (begun) {
                ok = __all_sync(kWarpAll, wait(o_done(slot), count - 1));
                if (!ok) break;
                tc_fence_after();
            }
            float* rec = nullptr;
            if (at_row < q_rows) {
                const int b = at_row / gh, h = p.h * gh + at_row - b * gh;
                rec = p.i == 0 ? A.s.own + ((alternate ? slot * A.s.own_records : 0) + (int64_t)(p.T.row0 + b) * A.heads + h) * A.s.pitch
                               : A.s.cut + (((int64_t)blockIdx.x * 2 + slot) * kSharedLanes + row) * A.s.pitch;
            }
            if (begun) {
#pragma unroll 1
                for (int d = 0; d < hd; d += 32) {
                    uint32_t x[32];
                    tmem_ld_32x32b_x32(o_at + d, x);
                    if (rec) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (d + i < hd)
                                *reinterpret_cast<uint4*>(rec + d + i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                    }
                }
            }
            tc_fence_before();
            if (rec) *reinterpret_cast<float2*>(rec + A.s.pitch - 4) = make_float2(m == -FLT_MAX ? m : m - kRowLift, l);
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

template <int kCodes, bool kBfQ, bool kBfV, int kDim> int launch_shared(const SharedArgs& A, cudaStream_t st) {
    using C = Cfg<kCodes, kDim>;
    return launch(shared_kernel<kCodes, kBfQ, kBfV, kDim>, dim3((unsigned)A.grid), dim3(C::kThreads), (size_t)C::kSmem, st,
                  "epq_paged_attend_shared", A);
}
template <int kCodes, bool kBfQ, bool kBfV> int launch_shared_d(const SharedArgs& A, cudaStream_t st) {
    const int hd = A.pages.head_dim;
    if (hd <= 64) return launch_shared<kCodes, kBfQ, kBfV, 64>(A, st);
    if (hd <= 128) return launch_shared<kCodes, kBfQ, kBfV, 128>(A, st);
    return launch_shared<kCodes, kBfQ, kBfV, 256>(A, st);
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Where things lie in the workspace, behind the attention's own part.
struct Layout {
    int tile_rows, max_tiles, slots, pitch;
    int64_t head, tiles, row_tile, row_from, own, cut, bytes;
};
Layout layout_of(const PagesD& P, int64_t batch, int heads, int64_t groups, int64_t behind) {
    Layout L;
    const int dim = P.head_dim <= 64 ? 64 : P.head_dim <= 128 ? 128 : 256, group = heads / P.kv_heads;
    L.slots = dim == 256 ? 1 : 2;
    L.pitch = dim + 4;
    L.tile_rows = L.slots * kSharedLanes / group;
    const int64_t some = groups < batch / 2 ? groups : batch / 2;      // groups of two rows or more
    L.max_tiles = (int)(batch / (L.tile_rows ? L.tile_rows : 1) + some + 1);
    L.head = behind;
    L.tiles = L.head + 256;
    L.row_tile = align256(L.tiles + L.max_tiles * (int64_t)sizeof(SharedTile));
    L.row_from = align256(L.row_tile + batch * 4);
    L.own = align256(L.row_from + batch * 4);
    L.cut = align256(L.own + 2 * batch * heads * L.pitch * 4);
    L.bytes = L.cut + (int64_t)device_sms() * 2 * kSharedLanes * L.pitch * 4;
    return L;
}

// Whether a batch can share anything that is worth it: groups of two rows or more whose query heads fit a tile, and
// enough tokens that the tables could hold.
bool may_share(const PagesD& P, int64_t batch, int heads, int64_t groups, int64_t token_bytes) {
    const int64_t most = (int64_t)P.max_pages * P.page_size;
    const int64_t pool = P.pages > (1LL << 40) / P.page_size ? 1LL << 40 : P.pages * P.page_size;   // (all tables together)
    const int64_t tokens = most < pool ? most : pool;
    return groups > 0 && batch > 1 && heads / P.kv_heads <= kSharedLanes &&
           (double)(batch - 1) * (double)tokens * (double)token_bytes >= (double)kWorth;
}
int64_t bytes_of_token(const PagesD& P, int dtype_bytes) {
    return 2LL * P.kv_heads * (P.format == EPQ_CACHE_SAME ? P.head_dim * dtype_bytes : P.head_dim + 4);
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

int64_t epq_paged_attend_shared_workspace_bytes(const epq_pages* pages, int64_t batch, int32_t heads, int64_t groups) {
    const char* const who = "epq_paged_attend_shared_workspace_bytes";
    if (groups < 0) return set_error(EPQ_EINVAL, "%s: groups=%lld", who, (long long)groups);
    const int64_t behind = attend_bytes(who, pages, batch, heads);
    if (behind < 0) return behind;
    PagesD P;
    make_pages(pages, &P, who);
    if (batch > 65536) return set_error(EPQ_EUNSUPPORTED, "%s: batch=%lld", who, (long long)batch);
    if (!may_share(P, batch, heads, groups, bytes_of_token(P, 2))) return behind;
    return layout_of(P, batch, heads, groups, align256(behind)).bytes;
}

int epq_paged_attend_shared(const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                            int64_t batch, const int32_t* starts, const int64_t* prefix, int64_t groups, float scale, void* out,
                            float* lse, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
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
    const int64_t token_bytes = bytes_of_token(P, 2);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!may_share(P, batch, A.heads, groups, token_bytes)) return launch_attend_plain(A, cols, st);
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
    S.s.own = reinterpret_cast<float*>(ws + L.own);
    S.s.cut = reinterpret_cast<float*>(ws + L.cut);
    S.s.own_records = batch * A.heads;
    S.s.pitch = L.pitch;
    S.s.slots = L.slots;
    S.q = q->data;
    S.q_row = q->stride_row;
    S.q_head = q->stride_head;
    S.q_aligned = heads_aligned(*q, 2, 16);
    S.seq = seq;
    S.lengths = lengths;
    S.starts = starts;
    S.prefix = prefix;
    S.token_bytes = token_bytes;
    S.batch = (int)batch;
    S.groups = (int)groups;
    S.heads = A.heads;
    S.group = A.group;
    S.tile_rows = L.tile_rows;
    S.max_tiles = L.max_tiles;
    S.grid = device_sms();
    S.scale_log2 = A.scale_log2;
    int e = launch(plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, who, S);
    if (e != EPQ_OK) return e;
    const bool bf = dtype == EPQ_BF16;
    if (P.format == EPQ_CACHE_INT8)
        e = bf ? launch_shared_d<kInts, true, true>(S, st) : launch_shared_d<kInts, false, true>(S, st);
    else if (P.format == EPQ_CACHE_FP8)
        e = bf ? launch_shared_d<kFloats, true, true>(S, st) : launch_shared_d<kFloats, false, true>(S, st);
    else
        e = bf ? launch_shared_d<kNone, true, true>(S, st) : launch_shared_d<kNone, false, false>(S, st);
    if (e != EPQ_OK) return e;
    A.shared = S.s;
    return attend_behind_shared(A, cols, st);
}

}  // extern "C"
