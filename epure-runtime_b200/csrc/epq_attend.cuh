// The attention kernel of one new token a row over a paged cache, for every form of it: all
// tokens of a row's sequence (k_paged_attn.cu, which holds the description), those of selected
// blocks (k_paged_attn_blocks.cu), or those behind a shared prefix (k_paged_attn_shared.cu).
// Each file instantiates its own form.
#pragma once

#include <cfloat>

#include "epq_paged.cuh"
#include "epq_shared.cuh"

namespace epq {
namespace paged {

struct AttendArgs {
    PagesD pages;
    const void* q;
    int64_t q_row, q_head;
    const int32_t* seq;
    const int64_t* lengths;
    void* out;
    float* lse;
    float* records;
    unsigned* counters;
    int64_t window;
    const int32_t* blocks;   // kListed: [batch][kv_heads][count] pages of the sequence, -1: none
    int count;
    SharedD shared;          // kBehindShared
    const int32_t* starts;   // kAllTokens, for a batch that could share but does not: its groups, which are looked
    const int64_t* prefix;   // at for their errors alone
    int groups;
    int batch, heads, group, chunks, dtype;
    float scale_log2;
};

// Which tokens a row attends over.
enum Mode {
    kAllTokens = 0,      // the first lengths[b] of its sequence (the last `window` of them)
    kListed = 1,         // those of the blocks (pages) that a list of each row and key head names
    kBehindShared = 2    // those from row_from[b] on, left as sums
};

namespace {

__device__ int g_attend_error = 0;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16;                  // tokens of a tensor-core tile; a warp's block is one or two
constexpr int kMinBlocks = 4;              // a CTA's run is at least this long
constexpr int kWhole = 12;                 // and a unit of at most this many is not cut for latency
// What a unit costs besides its blocks (its q, joining its warps), in blocks: 64 x 8k fp8
// took 104 us with 2, 101 with 4, 97 with 8 to 16.
constexpr int kUnitCost = 12;
constexpr int kMaxUnits = 65536;           // counters in the workspace
constexpr int kMaxGrid = 512;              // CTAs of a launch
constexpr float kSlack = 8.f;              // how far (log2) a score may pass the running maximum
// Weights in f16 are 2^kLift of those that the maximum stands for, which is as high as f16
// goes (2^(8 + 7)): what is below 2^-32 of the maximum is lost, not what is below 2^-25.
constexpr float kLift = 7.f;
constexpr float kLog2e = 1.4426950408889634f;

// Element kinds of the cache: what the tensor cores multiply.
enum Kind { kBf16 = 0, kF16 = 1, kInt8 = 2, kFp8 = 3 };

template <int kKind> constexpr int kind_bytes() { return kKind <= kF16 ? 2 : 1; }

// ---------------------------------------------------------------- PTX
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {   // bytes 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool kIsBf16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (kIsBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <bool kIsBf16> struct Half { using type = __half; };
template <> struct Half<true> { using type = __nv_bfloat16; };
template <bool kIsBf16> __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return pack2<typename Half<kIsBf16>::type>(lo, hi);
}

// The four 8-bit codes of x as two pairs of f16: its bytes (0, 1) and (2, 3), or with
// kAcross (0, 2) and (1, 3).  An int8 byte comes with 0x64 above it, 1024 + (code ^ 0x80),
// and 1152 is taken off; e4m3 has an instruction of its own.
template <int kKind, bool kAcross> __device__ __forceinline__ void codes_f16(uint32_t x, uint32_t& p0, uint32_t& p1) {
    if (kKind == kInt8) {
        const uint32_t u = x ^ 0x80808080u, off = 0x64806480u;
        const uint32_t u0 = __byte_perm(u, 0x64646464u, kAcross ? 0x4240 : 0x4140);
        const uint32_t u1 = __byte_perm(u, 0x64646464u, kAcross ? 0x4341 : 0x4342);
        const __half2 v0 = __hsub2(*reinterpret_cast<const __half2*>(&u0), *reinterpret_cast<const __half2*>(&off));
        const __half2 v1 = __hsub2(*reinterpret_cast<const __half2*>(&u1), *reinterpret_cast<const __half2*>(&off));
        p0 = *reinterpret_cast<const uint32_t*>(&v0);
        p1 = *reinterpret_cast<const uint32_t*>(&v1);
    } else {
        const uint32_t u = kAcross ? __byte_perm(x, 0u, 0x3120) : x;
        asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %2;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n cvt.rn.f16x2.e4m3x2 %1, hi;\n}\n"
            : "=r"(p0), "=r"(p1) : "r"(u));
    }
}

// Byte offset of 16-byte chunk `ch` of row `row` in a stage of rows of kPitch bytes: the
// chunk's place within 128 bytes is turned by the line's number, so the 8 rows of an
// ldmatrix fall into different banks.
template <int kPitch> __device__ __forceinline__ uint32_t swizzled(int row, int ch) {
    const uint32_t at = (uint32_t)(row * kPitch + ch * 16);
    return at ^ ((at >> 7 & 7u) << 4);
}

// ---------------------------------------------------------------- units and blocks
struct Span {
    int lo, first, n, blocks;   // tokens [lo, n) in blocks of kTok from `first` on
    int limit;                  // kListed: the sequence's own length (lo to n count places in the list)
};

template <int kMode, int kTok> __device__ __forceinline__ Span span_of(const AttendArgs& A, int b, bool report) {
    const int64_t cap = (int64_t)A.pages.max_pages * A.pages.page_size;
    int64_t n = A.lengths[b];
    bool bad = n < 0 || n > cap;
    if (A.seq && (A.seq[b] < 0 || A.seq[b] >= A.pages.seqs)) bad = n != 0 || bad;
    if (bad) {
        if (report) atomicOr(&g_attend_error, kBadPosition);
        n = 0;
    }
    Span s;
    s.limit = s.n = (int)n;
    s.lo = 0;
    if (kMode == kAllTokens && A.window > 0 && n > A.window) s.lo = (int)(n - A.window);
    if (kMode == kBehindShared) s.lo = min(A.shared.row_from[b], s.n);
    if (kMode == kListed && s.n > 0) s.n = min(A.count, A.pages.page_of(s.n - 1) + 1) * A.pages.page_size;
    s.first = s.lo & ~(kTok - 1);
    s.blocks = (s.n - s.first + kTok - 1) / kTok;
    if (kMode == kBehindShared && s.lo == s.n) s.blocks = 0;
    return s;
}

// A place in the dealt-out order: block i of unit u of sequence b.
template <int kMode, int kTok> struct Cursor {
    int b, u, i, units;
    Span s;
    __device__ __forceinline__ void next_sequence(const AttendArgs& A) {
        u = 0;
        do {
            if (b + 1 >= A.batch) {                    // never, unless lengths change under the kernel: nothing more is read
                s.n = 0;
                s.blocks = 1 << 28;
                return;
            }
            ++b;
            s = span_of<kMode, kTok>(A, b, false);
        } while (s.blocks == 0);
    }
    // Moves on by `step` blocks; the caller knows that they exist.
    __device__ __forceinline__ void advance(const AttendArgs& A, int step) {
        i += step;
        while (i >= s.blocks) {
            i -= s.blocks;
            if (++u == units) next_sequence(A);
        }
    }
};

template <int kKind, int kDim, int kCols>
struct Shape {
    static constexpr int kBytes = kind_bytes<kKind>();
    static constexpr int kPitch = kDim * kBytes;
    // Two tiles a block where a tile is at most 2 KB and its accumulators leave the registers
    // for them: the block's control flow then counts half (64 x 8k fp8: 119 us with one).
    static constexpr int kTiles = kPitch <= 128 && kDim * kCols <= 128 ? 2 : 1;
    static constexpr int kTok = kTiles * kTile;
    static constexpr int kRows = kTok * kPitch;                          // one of K, V
    static constexpr int kScales = kBytes == 1 ? 2 * kTok * 4 : 0;
    static constexpr int kStage = 2 * kRows + kScales;
    // (Two columns of heads of 256 spill 216 to 448 bytes at 255 registers: 24 / 2 heads over
    // 32 sequences of up to 8192 tokens take 80 us in bf16, where 16 / 2 heads, which do not, take 64.)
    static constexpr int kCtas = kPitch > 256 ? 1 : kPitch == 64 && kCols == 1 ? 3 : 2;       // an SM
    static constexpr int kMergePitch = kDim + 4;                         // floats; spreads a column's heads over the banks
    static constexpr int kMerge = kWarps * 8 * kMergePitch * 4;
    // a warp's ring: its share of what 228 KB leave a CTA (1 KB is the system's, 512 bytes are static)
    static constexpr int kBudget = (228 * 1024 / kCtas - 1024 - 512 - kMerge) / kWarps;
    static constexpr int kFit = kBudget / kStage;
    static constexpr int kStages = kFit > 6 ? 6 : kFit;
    static constexpr int kRing = kStages * kStage;
    static constexpr int kSmem = kWarps * kRing + kMerge;
    static constexpr int kRecord = kCols * 8 * kMergePitch;              // floats: accumulators, then m, M, l in the padding
    static_assert(kStages >= 2, "ring");
};

// a / b of the dealt-out order: 32-bit wherever it is enough.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// Four values of a row's head: sums `val` of weights relative to 2^at and their sum `sum` relative to 2^to, divided
// and written; sum = 0: every score was -inf.  Behind a shared prefix the sums go to the join as they are.
template <int kMode, bool kQuant>
__device__ __forceinline__ void emit_row(const AttendArgs& A, int b, int h, int d, const float (&val)[4], float at, float to,
                                         float sum) {
    const int64_t place = (int64_t)b * A.heads + h;
    if (kMode == kBehindShared && A.shared.row_from[b] > 0) {
        const float turn = kQuant && sum != 0.f ? ex2(at - to) : 1.f;
        float* const rec = A.shared.rest + place * A.shared.pitch;
        *reinterpret_cast<float4*>(rec + d) = make_float4(val[0] * turn, val[1] * turn, val[2] * turn, val[3] * turn);
        if (d == 0) *reinterpret_cast<float4*>(rec + A.shared.pitch - 4) = make_float4(sum == 0.f ? -FLT_MAX : to, sum, 0.f, 0.f);
        return;
    }
    float gain = sum == 0.f ? 0.f : 1.f / sum;
    if (kQuant) gain *= ex2(at - to);
    uint2 o;
    if (A.dtype == EPQ_BF16) {
        o = make_uint2(pack<true>(val[0] * gain, val[1] * gain), pack<true>(val[2] * gain, val[3] * gain));
    } else {
        o = make_uint2(pack<false>(val[0] * gain, val[1] * gain), pack<false>(val[2] * gain, val[3] * gain));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(A.out) + place * A.pages.head_dim + d) = o;
    if (A.lse && d == 0) A.lse[place] = sum == 0.f ? -INFINITY : (to + log2f(sum)) / kLog2e;
}

template <int kMode, int kKind, int kDim, int kCols>
__global__ void __launch_bounds__(kThreads, Shape<kKind, kDim, kCols>::kCtas) attend_kernel(const AttendArgs A) {
    using S = Shape<kKind, kDim, kCols>;
    constexpr bool kQuant = kKind >= kInt8;
    constexpr bool kIsBf16 = kKind == kBf16;
    constexpr int kTok = S::kTok, kTiles = S::kTiles;
    constexpr float kSumLift = kKind == kF16 ? kLift : 0.f;      // 8-bit caches lift the values' weights alone
    constexpr unsigned kAll = 0xffffffffu;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t seen[kWarps][S::kStages];     // bit r: row r of the stage is a token of the span
    __shared__ bool last;
    pdl_enter();

    const PagesD& P = A.pages;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hd = P.head_dim, units = P.kv_heads * A.chunks;
    const int hd_chunks = hd * S::kBytes / 16;

    // ---- this CTA's run of blocks.  Every warp works it out for itself: lane i looks at the
    // sequences [i per, (i + 1) per)
    const int per = (A.batch + 31) / 32;
    const int b0 = min(A.batch, lane * per), b1 = min(A.batch, b0 + per);
    auto weight = [&](int blocks) { return blocks ? blocks + kUnitCost : 0; };
    auto scan = [&](int v) {                           // inclusive, over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(kAll, v, o);
            if (lane >= o) v += u;
        }
        return v;
    };
    const bool looks = kMode == kAllTokens && A.groups > 0 && blockIdx.x == gridDim.x - 1;
    int from = 0, to = 0;                              // a thread's first group, on its way with the lengths
    int64_t prefix = 0;
    if (looks && tid < A.groups) {
        from = A.starts[tid];
        to = A.starts[tid + 1];
        prefix = A.prefix[tid];
    }
    const int first_blocks = b0 < b1 ? span_of<kMode, kTok>(A, b0, blockIdx.x == 0).blocks : 0;
    int mine = weight(first_blocks), some_empty = b0 < b1 && first_blocks == 0;
    for (int b = b0 + 1; b < b1; ++b) {
        const int blocks = span_of<kMode, kTok>(A, b, blockIdx.x == 0).blocks;
        mine += weight(blocks);
        some_empty |= blocks == 0;
    }
    if (looks) {
        auto bad_group = [&]() { return from < 0 || from > to || to > A.batch || prefix < 0 || prefix > (int64_t)P.max_pages * P.page_size; };
        bool bad = bad_group();
        for (int g = tid + kThreads; g < A.groups; g += kThreads) {
            from = A.starts[g];
            to = A.starts[g + 1];
            prefix = A.prefix[g];
            bad |= bad_group();
        }
        if (bad) atomicOr(&g_attend_error, kBadPosition);
    }
    const int64_t total = (int64_t)__reduce_add_sync(kAll, mine) * units;
    const int run = max(kMinBlocks, (int)quotient(total + gridDim.x - 1, gridDim.x));
    // Where cutting every long unit into pieces of at most `run` blocks makes no more pieces
    // than there are CTAs, each CTA takes one piece; else runs go over unit boundaries.
    auto pieces_of = [&](int blocks) { return blocks > kWhole ? (blocks + run - 1) / run : blocks > 0; };
    int pieces = pieces_of(first_blocks);
    for (int b = b0 + 1; b < b1; ++b) pieces += pieces_of(span_of<kMode, kTok>(A, b, false).blocks);
    const int64_t all_pieces = (int64_t)__reduce_add_sync(kAll, pieces) * units;
    const bool one_each = all_pieces <= gridDim.x;
    const int share = one_each ? pieces : mine, upto = scan(share);    // of the lane's sequences, and up to them
    const int64_t f0 = one_each ? blockIdx.x : blockIdx.x * (int64_t)run;    // piece, or place in the dealt-out order
    // sequences without a token
    some_empty = __any_sync(kAll, some_empty);
    for (int b = blockIdx.x; some_empty && b < A.batch; b += gridDim.x) {
        if (span_of<kMode, kTok>(A, b, false).blocks) continue;
        if (kMode == kBehindShared && A.shared.row_from[b] > 0) {      // nothing but the shared tokens, if any
            for (int h = tid; h < A.heads; h += kThreads)
                *reinterpret_cast<float4*>(A.shared.rest + ((int64_t)b * A.heads + h + 1) * A.shared.pitch - 4) =
                    make_float4(-FLT_MAX, 0.f, 0.f, 0.f);
            continue;
        }
        for (int e = tid; e < A.heads * hd; e += kThreads)
            static_cast<uint16_t*>(A.out)[(int64_t)b * A.heads * hd + e] = 0;
        if (A.lse)
            for (int h = tid; h < A.heads; h += kThreads) A.lse[(int64_t)b * A.heads + h] = -INFINITY;
    }
    if (f0 >= (one_each ? all_pieces : total)) return;
    Cursor<kMode, kTok> unit;                                 // of the unit that the CTA is at
    unit.units = units;
    {
        const int64_t lo = (int64_t)(upto - share) * units, hi = (int64_t)upto * units;
        const bool here = f0 >= lo && f0 < hi;
        int at_b = 0, at_u = 0, at_i = 0;
        if (here) {
            int64_t at = f0 - lo;
            for (int b = b0; b < b1; ++b) {
                const int blocks = b == b0 ? first_blocks : span_of<kMode, kTok>(A, b, false).blocks;
                const int each = one_each ? pieces_of(blocks) : weight(blocks);
                if (at < (int64_t)each * units) {
                    at_b = b;
                    at_u = (int)quotient(at, each);
                    at_i = (int)(at - (int64_t)at_u * each);
                    break;
                }
                at -= (int64_t)each * units;
            }
        }
        const int from = __ffs(__ballot_sync(kAll, here)) - 1;
        unit.b = __shfl_sync(kAll, at_b, from);
        unit.u = __shfl_sync(kAll, at_u, from);
        unit.i = __shfl_sync(kAll, at_i, from);
    }
    unit.s = span_of<kMode, kTok>(A, unit.b, false);
    int count, piece = 0, piece_count = 1;             // blocks of this CTA; its place among its unit's pieces
    int64_t unit_at = f0 - unit.i;                     // where the unit begins in the dealt-out order
    if (one_each) {
        piece = unit.i;
        piece_count = pieces_of(unit.s.blocks);
        unit.i = (int)((int64_t)unit.s.blocks * piece / piece_count);
        count = (int)((int64_t)unit.s.blocks * (piece + 1) / piece_count) - unit.i;
    } else {
        // a unit's first kUnitCost places stand for its own cost, the others are its blocks
        const int at = unit.i;
        unit.i = max(0, at - kUnitCost);
        count = 0;
        int left = (int)min((int64_t)run, total - f0), begun = at;
        Cursor<kMode, kTok> to = unit;
        for (;;) {
            const int all = weight(to.s.blocks), take = min(left, all - begun);
            count += max(0, begun + take - kUnitCost) - max(0, begun - kUnitCost);
            left -= take;
            if (left == 0) break;
            const int same = min(units - 1 - to.u, left / all);    // whole units of the same sequence
            count += same * to.s.blocks;
            left -= same * all;
            if (left == 0) break;
            to.u += same;
            begun = 0;
            if (++to.u == units) to.next_sequence(A);
        }
        if (count == 0) return;
    }
    uint8_t* ring = smem + warp * S::kRing;
    const uint32_t ring_at = smem_u32(ring);
    if (hd < kDim) {                                   // chunks past the head's end stay zero
        for (int e = lane; e < S::kRing / 16; e += 32) reinterpret_cast<uint4*>(ring)[e] = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }

    // ---- loads, kStages - 1 blocks ahead
    const bool straight = P.page_size % kTile == 0 && hd == kDim;      // a tile's rows lie side by side in one page
    Cursor<kMode, kTok> ahead = unit;
    int f_load = warp;                                 // blocks are counted from the run's start
    // of the next block's row `lane & (kTok - 1)`: table entry, slot, whether it is a token
    int next_page = 0, next_slot = 0;
    bool next_on = false;                              // (the entry may still be on its way)
    auto look_up = [&]() {
        const int t = ahead.s.first + ahead.i * kTok + (lane & (kTok - 1));
        next_on = t >= ahead.s.lo && t < ahead.s.n;
        if (next_on) {
            int col = P.page_of(t);
            const int s = A.seq ? A.seq[ahead.b] : ahead.b;
            next_slot = t - col * P.page_size;
            if (kMode == kListed) {                    // the place's page by its list, and whether the slot is a token
                const int head = A.chunks == 1 ? ahead.u : ahead.u / A.chunks;
                col = A.blocks[((int64_t)ahead.b * P.kv_heads + head) * A.count + col];
                next_on = col >= 0 && (col >= P.max_pages || col * P.page_size + next_slot < ahead.s.limit);
                if (next_on && col >= P.max_pages) {
                    atomicOr(&g_attend_error, kBadPosition);
                    next_on = false;
                }
            }
            if (kMode == kAllTokens || next_on) next_page = P.table[(int64_t)s * P.table_stride + col];
        }
    };
    if (f_load < count) {
        ahead.advance(A, warp);
        look_up();
    }
    const int g = lane >> 2, c = lane & 3;             // row and column pair of the tensor fragments
    // q as B fragments: column g is the unit's query head 8 n + g.  16-bit caches: dims 2c, 2c+1
    // and 2c+8, 2c+9 of every 16; 8-bit ones: 4c .. 4c+3
    uint32_t qf[kCols][kDim / 16][2];
    auto load_q = [&](const Cursor<kMode, kTok>& u) {
        const int head = A.chunks == 1 ? u.u : u.u / A.chunks, chunk = u.u - head * A.chunks;
        const int h0 = head * A.group + chunk * 8 * kCols, n_heads = min(8 * kCols, A.group - chunk * 8 * kCols);
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
            const bool on = 8 * n + g < n_heads;
            const uint16_t* q = static_cast<const uint16_t*>(A.q) + u.b * A.q_row + (h0 + 8 * n + g) * A.q_head;
#pragma unroll
            for (int k = 0; k < kDim / 16; ++k) {
                const int d0 = 16 * k + (kQuant ? 4 * c : 2 * c), d1 = d0 + (kQuant ? 2 : 8);
                const bool there = on && 16 * k < hd;
                qf[n][k][0] = there ? *reinterpret_cast<const uint32_t*>(q + d0) : 0u;
                qf[n][k][1] = there ? *reinterpret_cast<const uint32_t*>(q + d1) : 0u;
            }
        }
    };
    load_q(unit);                                      // (on its way with the first table entry)
    constexpr int kChunks = S::kPitch / 16;            // of a row
    constexpr int kCopies = kTile * kChunks / 32;      // chunks a lane and tile
    const int my_row = lane / kChunks, my_ch = lane % kChunks;     // a lane's chunks: rows my_row, my_row + 32 / kChunks, ...
    // its place in a stage: 512 bytes further each time, with bit 6 turned (see swizzled)
    const uint32_t my_at = swizzled<S::kPitch>(my_row, my_ch);
    int load_stage = 0;
    auto load = [&]() {
        if (f_load < count) {
            if (next_on && (next_page < 0 || next_page >= P.pages)) {
                atomicOr(&g_attend_error, kBadPage);
                next_on = false;
            }
            const int head = A.chunks == 1 ? ahead.u : ahead.u / A.chunks;
            const int slot_at = head * P.page_size + next_slot;
            const int64_t at = (next_page * P.page_stride + (int64_t)slot_at * hd) * S::kBytes;
            const uint32_t k_at = ring_at + load_stage * S::kStage, v_at = k_at + S::kRows;
            const uint32_t mask = __ballot_sync(kAll, next_on);
            if (lane == 0) seen[warp][load_stage] = mask;
            if (straight && mask == kAll) {            // the ordinary block: every row is a token (with 16 rows, lanes repeat)
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) {
                    const int64_t off = __shfl_sync(kAll, at, tile * kTile) + lane * 16;
                    const uint8_t* k_from = P.k + off;
                    const uint8_t* v_from = P.v + off;
#pragma unroll
                    for (int e = 0; e < kCopies; ++e) {
                        const uint32_t to = tile * kTile * S::kPitch + (my_at ^ (e & 1) * 64) + e * 512;
                        cp16(k_at + to, k_from + e * 512);
                        cp16(v_at + to, v_from + e * 512);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < kTiles * kCopies; ++e) {
                    const int row = my_row + e * (32 / kChunks);
                    const int64_t from = __shfl_sync(kAll, at, row);
                    const bool on = mask >> row & 1;
                    if (my_ch < hd_chunks) {
                        const int64_t off = on ? from + my_ch * 16 : 0;
                        const uint32_t to = (my_at ^ (e & 1) * 64) + e * 512;
                        cp16(k_at + to, P.k + off, on ? 16 : 0);
                        cp16(v_at + to, P.v + off, on ? 16 : 0);
                    }
                }
            }
            if (kQuant) {
                const int64_t off = next_on ? next_page * P.scale_stride + slot_at : 0;
                const int bytes = next_on ? 4 : 0;
                if (kTiles == 2) {
                    cp4(v_at + S::kRows + lane * 4, P.k_scale + off, bytes);
                    cp4(v_at + S::kRows + kTok * 4 + lane * 4, P.v_scale + off, bytes);
                } else {                               // lanes 0-15: key scales, 16-31: value scales
                    cp4(v_at + S::kRows + lane * 4, (lane < 16 ? P.k_scale : P.v_scale) + off, bytes);
                }
            }
            f_load += kWarps;
            if (f_load < count) {
                ahead.advance(A, kWarps);
                look_up();
            }
        }
        cp_commit();
        if (++load_stage == S::kStages) load_stage = 0;
    };
#pragma unroll
    for (int e = 0; e < S::kStages - 1; ++e) load();

    // ---- units
    int f = warp, stage = 0;
    for (int at = 0; at < count;) {
        const int unit_start = at - unit.i, unit_end = unit_start + unit.s.blocks;   // unit_start < 0: begun before this run
        const int end = min(count, unit_end);
        const int head = A.chunks == 1 ? unit.u : unit.u / A.chunks, chunk = unit.u - head * A.chunks;
        const int h_first = head * A.group + chunk * 8 * kCols;               // query heads of this unit
        const int h_count = min(8 * kCols, A.group - chunk * 8 * kCols);
        const int seq_b = unit.b, unit_index = unit.b * units + unit.u;

        float q_gain[kCols][2];                        // what scores of heads 2c, 2c + 1 are multiplied by
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
            q_gain[n][0] = q_gain[n][1] = A.scale_log2;
            if (kQuant) {                              // q to f16, times a power of two
                const bool bf = A.dtype == EPQ_BF16;
                auto value = [&](uint32_t two, int hi) {
                    const uint16_t h = hi ? two >> 16 : two & 0xffff;
                    return bf ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
                };
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < kDim / 16; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        top = max(top, __float_as_uint(value(qf[n][k][r >> 1], r & 1)) & 0x7fffffffu);
                top = max(top, __shfl_xor_sync(kAll, top, 1));
                top = max(top, __shfl_xor_sync(kAll, top, 2));
                // the largest value's exponent becomes 14; zeros, infinities and NaN stay
                int shift = top == 0 || top >= 0x7f800000u ? 0 : 14 - ((int)(top >> 23) - 127);
                shift = max(-120, min(120, shift));
                const float up = __uint_as_float((uint32_t)(127 + shift) << 23);
                const float down = __uint_as_float((uint32_t)(127 - shift) << 23);
#pragma unroll
                for (int k = 0; k < kDim / 16; ++k)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        qf[n][k][r] = pack<false>(value(qf[n][k][r], 0) * up, value(qf[n][k][r], 1) * up);
                q_gain[n][0] *= __shfl_sync(kAll, down, 8 * c);
                q_gain[n][1] *= __shfl_sync(kAll, down, 8 * c + 4);
            }
        }

        float m[kCols][2], M[kCols][2], l[kCols][2], acc[kCols][kDim / 16][4];
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                m[n][r] = M[n][r] = -FLT_MAX;
                l[n][r] = 0.f;
            }
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[n][d][r] = 0.f;
        }

        for (; f < end; f += kWarps) {
            cp_wait<S::kStages - 2>();
            __syncwarp();
            load();                                    // into the stage of the block before this one
            const uint32_t k_at = ring_at + stage * S::kStage;
            const uint32_t mask = seen[warp][stage];
            constexpr int kLoads = kDim * S::kBytes / 32;          // ldmatrix a block and operand
            constexpr int kBatch = kLoads < 8 ? kLoads : 8;        // of which so many are in registers

            // scores: even and odd steps into accumulators of their own
            float sc[kTiles][kCols][4];
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                float sc2[kCols][4];
#pragma unroll
                for (int n = 0; n < kCols; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[tile][n][r] = sc2[n][r] = 0.f;
                // rows 0-15, 16-byte chunks 2 k and 2 k + 1 of them: the four 8 x 8 parts lie tokens first
#pragma unroll
                for (int k0 = 0; k0 < kLoads; k0 += kBatch) {
                    uint32_t x[kBatch][4];
#pragma unroll
                    for (int k = 0; k < kBatch; ++k)
                        ldsm(x[k], k_at + tile * kTile * S::kPitch + swizzled<S::kPitch>(lane & 15, 2 * (k0 + k) + (lane >> 4)));
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        if (!kQuant) {
#pragma unroll
                            for (int n = 0; n < kCols; ++n)
                                mma<kIsBf16>(k & 1 ? sc2[n] : sc[tile][n], x[k], qf[n][k0 + k][0], qf[n][k0 + k][1]);
                        } else {
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                uint32_t a[4];
                                codes_f16<kKind, false>(x[k][2 * r], a[0], a[2]);
                                codes_f16<kKind, false>(x[k][2 * r + 1], a[1], a[3]);
#pragma unroll
                                for (int n = 0; n < kCols; ++n)
                                    mma<false>(r ? sc2[n] : sc[tile][n], a, qf[n][2 * (k0 + k) + r][0], qf[n][2 * (k0 + k) + r][1]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < kCols; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[tile][n][r] += sc2[n][r];
            }
            // the first values are on their way while the weights are formed
            uint32_t y[kTiles][kBatch][4];
            auto load_values = [&](int tile, int d0) {
#pragma unroll
                for (int d = 0; d < kBatch; ++d) {
                    // 16-bit: chunks first, the order of the fragment; 8-bit: tokens first, the codes are paired below
                    const int row = kQuant ? lane & 15 : (lane >> 4) * 8 + (lane & 7);
                    const int ch = 2 * (d0 + d) + (kQuant ? lane >> 4 : lane >> 3 & 1);
                    ldsm_t(y[tile][d], k_at + S::kRows + tile * kTile * S::kPitch + swizzled<S::kPitch>(row, ch));
                }
            };
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) load_values(tile, 0);
            float ks[kTiles][2], lv[kTiles][2];
            if (kQuant) {
                const float* scales = reinterpret_cast<const float*>(ring + stage * S::kStage + 2 * S::kRows);
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        ks[tile][r] = scales[tile * kTile + g + 8 * r];
                        lv[tile][r] = __log2f(scales[kTok + tile * kTile + g + 8 * r]);
                    }
            }
            // weights; r: token g + 8 (r >> 1) of the tile, head 2c + (r & 1)
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
                for (int n = 0; n < kCols; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        sc[tile][n][r] *= kQuant ? q_gain[n][r & 1] * ks[tile][r >> 1] : q_gain[n][r & 1];
            if (mask != kAll) {
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
                    for (int n = 0; n < kCols; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!(mask >> (tile * kTile + g + 8 * (r >> 1)) & 1)) sc[tile][n][r] = -INFINITY;
            }
            float over = -INFINITY;                    // fmaxf passes over NaN, which reaches the sums through the weights
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
                for (int n = 0; n < kCols; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        over = fmaxf(over, sc[tile][n][r] - m[n][r & 1]);
                        if (kQuant) over = fmaxf(over, sc[tile][n][r] + (lv[tile][r >> 1] - M[n][r & 1]));
                    }
            if (__any_sync(kAll, over > kSlack)) {
#pragma unroll
                for (int n = 0; n < kCols; ++n) {
                    float turn_acc[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float top = -FLT_MAX, topM = -FLT_MAX;
#pragma unroll
                        for (int tile = 0; tile < kTiles; ++tile) {
                            top = fmaxf(top, fmaxf(sc[tile][n][r], sc[tile][n][r + 2]));
                            if (kQuant) topM = fmaxf(topM, fmaxf(sc[tile][n][r] + lv[tile][0], sc[tile][n][r + 2] + lv[tile][1]));
                        }
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) {
                            top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
                            if (kQuant) topM = fmaxf(topM, __shfl_xor_sync(kAll, topM, o));
                        }
                        const float mn = fmaxf(m[n][r], top);
                        const float turn_l = mn == m[n][r] ? 1.f : ex2(m[n][r] - mn);
                        l[n][r] *= turn_l;
                        m[n][r] = mn;
                        turn_acc[r] = turn_l;
                        if (kQuant) {
                            const float Mn = fmaxf(M[n][r], topM);
                            turn_acc[r] = Mn == M[n][r] ? 1.f : ex2(M[n][r] - Mn);
                            M[n][r] = Mn;
                        }
                    }
#pragma unroll
                    for (int d = 0; d < kDim / 16; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[n][d][r] *= turn_acc[r & 1];
                }
            }
            // A weight is the sum of two values of the type (16 bits of it in bf16, 22 in f16): one
            // rounding of it alone is as large as the result's in bf16 or f16 caches, and in 8-bit
            // ones as large as an f16 result's (error of 2-norm 2.7e-4 instead of 2.1e-4 off 64 bits;
            // the second part takes 64 x 8k e4m3 from 97.1 to 97.5 us, 16 x 4k int8 from 20.3 to 21.1).
            constexpr int kParts = 2;
            uint32_t pf[kTiles][kCols][kParts][2];
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
                for (int n = 0; n < kCols; ++n) {
                    float w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        w[r] = ex2(sc[tile][n][r] - (m[n][r & 1] - kSumLift));
                        l[n][r & 1] += w[r];
                        if (kQuant) w[r] = ex2(sc[tile][n][r] + (lv[tile][r >> 1] - (M[n][r & 1] - kLift)));
                    }
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const uint32_t two = pack<kIsBf16>(w[2 * r], w[2 * r + 1]);
                            pf[tile][n][part][r] = transpose8x8(two);
                            if (part + 1 < kParts) {
                                const float2 back = unpack2<typename Half<kIsBf16>::type>(two);
                                w[2 * r] -= back.x;
                                w[2 * r + 1] -= back.y;
                            }
                        }
                    }
                }
            // O^T += V^T P^T
#pragma unroll
            for (int d0 = 0; d0 < kLoads; d0 += kBatch)
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) {
                    if (d0) load_values(tile, d0);
#pragma unroll
                    for (int d = 0; d < kBatch; ++d) {
                        const uint32_t (&v)[4] = y[tile][d];
                        if (!kQuant) {
#pragma unroll
                            for (int n = 0; n < kCols; ++n)
#pragma unroll
                                for (int part = 0; part < kParts; ++part)
                                    mma<kIsBf16>(acc[n][d0 + d], v, pf[tile][n][part][0], pf[tile][n][part][1]);
                        } else {
#pragma unroll
                            for (int r = 0; r < 2; ++r) {  // rows 0-7: the even dims of 16, rows 8-15: the odd ones
                                uint32_t a[4];
                                codes_f16<kKind, true>(v[2 * r], a[0], a[1]);
                                codes_f16<kKind, true>(v[2 * r + 1], a[2], a[3]);
#pragma unroll
                                for (int n = 0; n < kCols; ++n)
#pragma unroll
                                    for (int part = 0; part < kParts; ++part)
                                        mma<false>(acc[n][2 * (d0 + d) + r], a, pf[tile][n][part][0], pf[tile][n][part][1]);
                            }
                        }
                    }
                }
            if (++stage == S::kStages) stage = 0;
        }

        // ---- the unit's piece: the four warps' states to one
        const bool cut_before = unit_start < 0, cut = cut_before || unit_end > count;
        const int64_t unit_from = unit_at + kUnitCost, unit_to = unit_from + unit.s.blocks;
        at = end;
        if (at < count) {                              // the next unit's q is on its way meanwhile
            unit_at = unit_to;
            unit.advance(A, unit.s.blocks - unit.i);
            load_q(unit);
        }
        float* const merge = reinterpret_cast<float*>(smem + kWarps * S::kRing);
        constexpr int kQuads = kDim / 4;               // of a head's dims
        auto emit = [&](int h, int d, const float (&val)[4], float mx, float Mx, float sum) {
            emit_row<kMode, kQuant>(A, seq_b, h_first + h, d, val, kQuant ? Mx - kLift : mx - kSumLift, mx - kSumLift, sum);
        };
        // none where the unit is whole; else where the piece's record goes
        float* const record = !cut ? nullptr
                                   : A.records + ((int64_t)blockIdx.x * 2 + (cut_before && !one_each ? 0 : 1)) * S::kRecord;
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
            if (8 * n < h_count) {
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int dim = 16 * d + (kQuant ? 2 * g + (r >> 1) : g + 8 * (r >> 1));
                        merge[(warp * 8 + 2 * c + (r & 1)) * S::kMergePitch + dim] = acc[n][d][r];
                    }
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {          // (m, M, l) behind the head's accumulators
                    float s = l[n][r];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) s += __shfl_xor_sync(kAll, s, o);
                    if (lane < 4)
                        *reinterpret_cast<float4*>(merge + (warp * 8 + 2 * c + r) * S::kMergePitch + kDim) =
                            make_float4(m[n][r], kQuant ? M[n][r] : m[n][r], s, 0.f);
                }
                __syncthreads();
                for (int e = tid; e < 8 * kQuads; e += kThreads) {
                    const int j = e / kQuads, d = e % kQuads * 4, h = 8 * n + j;
                    if (h >= h_count) break;
                    if (d >= hd) continue;
                    float4 of[kWarps];
                    float mx = -FLT_MAX, Mx = -FLT_MAX;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        of[w] = *reinterpret_cast<const float4*>(merge + (w * 8 + j) * S::kMergePitch + kDim);
                        mx = fmaxf(mx, of[w].x);
                        Mx = fmaxf(Mx, of[w].y);
                    }
                    float sum = 0.f, val[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        // a warp that saw nothing has m = M = -FLT_MAX and zeros; NaN passes through
                        const float fl = ex2(of[w].x - mx);
                        const float fa = kQuant ? ex2(of[w].y - Mx) : fl;
                        const float4 a = *reinterpret_cast<const float4*>(merge + (w * 8 + j) * S::kMergePitch + d);
                        sum += of[w].z * fl;
                        val[0] += a.x * fa;
                        val[1] += a.y * fa;
                        val[2] += a.z * fa;
                        val[3] += a.w * fa;
                    }
                    if (!record) {
                        emit(h, d, val, mx, Mx, sum);
                    } else {
                        float* rec = record + h * S::kMergePitch;
                        *reinterpret_cast<float4*>(rec + d) = make_float4(val[0], val[1], val[2], val[3]);
                        if (d == 0) *reinterpret_cast<float4*>(rec + kDim) = make_float4(mx, Mx, sum, 0.f);
                    }
                }
                __syncthreads();
            }
        }

        // ---- a unit cut over several CTAs: the last of them joins the records
        if (record) {
            int first, parts;
            if (one_each) {
                first = (int)blockIdx.x - piece;
                parts = piece_count;
            } else {
                first = (int)quotient(unit_from, run);
                parts = (int)quotient(unit_to - 1, run) - first + 1;
            }
            if (tid == 0) {
                // releases the CTA's record (complete at the barrier above), acquires the others'
                unsigned before;
                asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                             : "=r"(before) : "l"(A.counters + unit_index) : "memory");
                last = before == (unsigned)parts - 1;
                if (last) A.counters[unit_index] = 0u;
            }
            __syncthreads();
            if (last) {
                for (int e = tid; e < 8 * kCols * kQuads; e += kThreads) {
                    const int h = e / kQuads, d = e % kQuads * 4;
                    if (h >= h_count) break;
                    if (d >= hd) continue;
                    float mx = -FLT_MAX, Mx = -FLT_MAX, sum = 0.f, val[4] = {0.f, 0.f, 0.f, 0.f};
                    constexpr int kAtOnce = 8;
                    for (int p0 = 0; p0 < parts; p0 += kAtOnce) {
                        float4 of[kAtOnce], a[kAtOnce];
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) {
                            const int p = min(p0 + i, parts - 1);
                            // where runs go over boundaries, only the first part is its CTA's last piece
                            const float* rec = A.records + ((int64_t)(first + p) * 2 + (one_each || p == 0 ? 1 : 0)) * S::kRecord +
                                               h * S::kMergePitch;
                            of[i] = __ldcg(reinterpret_cast<const float4*>(rec + kDim));
                            a[i] = __ldcg(reinterpret_cast<const float4*>(rec + d));
                        }
                        float mn = mx, Mn = Mx;
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) {
                            mn = fmaxf(mn, of[i].x);
                            Mn = fmaxf(Mn, of[i].y);
                        }
                        const float fl = mn == mx ? 1.f : ex2(mx - mn), fa = Mn == Mx ? 1.f : ex2(Mx - Mn);
                        sum *= fl;
#pragma unroll
                        for (int i = 0; i < 4; ++i) val[i] *= fa;
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) {
                            if (p0 + i < parts) {
                                const float w = ex2(of[i].y - Mn);
                                sum += of[i].z * ex2(of[i].x - mn);
                                val[0] += a[i].x * w;
                                val[1] += a[i].y * w;
                                val[2] += a[i].z * w;
                                val[3] += a[i].w * w;
                            }
                        }
                        mx = mn;
                        Mx = Mn;
                    }
                    emit(h, d, val, mx, Mx, sum);
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int kMode, int kKind, int kDim, int kCols>
int launch_attend(const AttendArgs& A, cudaStream_t st) {
    using S = Shape<kKind, kDim, kCols>;
    const int grid = device_sms() * S::kCtas;
    return launch(attend_kernel<kMode, kKind, kDim, kCols>, dim3((unsigned)(grid < kMaxGrid ? grid : kMaxGrid)), dim3(kThreads),
                  (size_t)S::kSmem, st, "epq_paged_attend", A);
}
template <int kMode, int kKind, int kDim>
int launch_attend_d(const AttendArgs& A, int cols, cudaStream_t st) {
    return cols == 1 ? launch_attend<kMode, kKind, kDim, 1>(A, st) : launch_attend<kMode, kKind, kDim, 2>(A, st);
}
template <int kMode, int kKind>
int launch_attend_k(const AttendArgs& A, int cols, cudaStream_t st) {
    const int hd = A.pages.head_dim;
    if (hd <= 64) return launch_attend_d<kMode, kKind, 64>(A, cols, st);
    if (hd <= 128) return launch_attend_d<kMode, kKind, 128>(A, cols, st);
    return launch_attend_d<kMode, kKind, 256>(A, cols, st);
}
template <int kMode> int launch_attend_mode(const AttendArgs& A, int cols, cudaStream_t st) {
    switch (A.pages.format) {
        case EPQ_CACHE_INT8: return launch_attend_k<kMode, kInt8>(A, cols, st);
        case EPQ_CACHE_FP8: return launch_attend_k<kMode, kFp8>(A, cols, st);
        default:
            return A.dtype == EPQ_BF16 ? launch_attend_k<kMode, kBf16>(A, cols, st) : launch_attend_k<kMode, kF16>(A, cols, st);
    }
}
int read_attend_error(int* flag) {
    if (cudaMemcpyFromSymbol(flag, g_attend_error, sizeof(int)) != cudaSuccess)
        return check_launch("read paged attention error flag");
    return EPQ_OK;
}

}  // namespace

// Checks the arguments that the forms have in common and fills what does not depend on the
// form; *cols: columns of 8 query heads a unit has.  *ready is false for an empty batch.
int make_attend(const char* who, const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                int64_t batch, float scale, void* out, float* lse, int32_t dtype, void* workspace, int64_t workspace_bytes,
                AttendArgs* A, int* cols, bool* ready);
// The form over all of a row's tokens (k_paged_attn.cu).
int launch_attend_plain(const AttendArgs& A, int cols, cudaStream_t st);
// Bytes of an attention's workspace: counters and records.
int64_t attend_bytes(const char* who, const epq_pages* pages, int64_t batch, int32_t heads);

}  // namespace paged
}  // namespace epq
