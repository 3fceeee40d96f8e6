// What a cheap score needs and chooses of a paged cache: the bounds of every page's keys
// (epq_paged_bounds) and, for each row and key head, the blocks (pages) to attend over
// (epq_paged_select).
//
//   lo[d], hi[d] = min, max over the page's tokens of K[t, d]
//   score = max over the key head's query heads of  sum_d max(q_d lo_d, q_d hi_d)
//
// which no q . K[t] of the page passes (16-bit caches, finite keys, up to the sums' rounding; the
// bounds of 8-bit ones are rounded to the nearest bf16).  A product of two 16-bit values is exact in float32
// and the sum's order is fixed (neighbours, then neighbours of their sums), so which blocks
// are chosen is the same wherever it is computed in float32.
//
// Bounds.  Bound: HBM, one read of the keys; for the pages of a decode step the chain of length,
// page and keys.  Up to 8 warps share one head of one page, so that a page is two accesses deep;
// a warp's lanes hold 16 bytes of a row each, the rows of an access side by side.
//
// Selection.  Bound: HBM, 4 head_dim bytes a block and head.  The defined sums would be bound by the
// issue rate (185 instructions a block of 8 heads of 128: 64 x 32k took 104 us for 21 us of bytes),
// so they are formed for few blocks only.  As max(q lo, q hi) = max(q, 0) hi + min(q, 0) lo (lo <= hi)
// the scores of 16 blocks and 8 heads are a product on the tensor cores (m16n8k16: a group's heads are
// its 8 columns; tcgen05's tiles of 128 rows would be read from shared memory, where these operands
// come from HBM straight into the registers that multiply them).  Its float32 sums have another
// order than the defined ones.  Together they are taken to be off by less than E = (1.5 head_dim + 8) 2^-23 |q|_1
// max|bounds| (3 head_dim over f16 bounds, and for an f16 q over bf16 bounds, which has two parts): head_dim
// products and twice head_dim / 8 sums of them, each off by at most 2^-23 of the sum of all |q_d bound_d|, in
// the one, log2 of that in the other.  That assumes of the tensor cores, whose sums no document specifies, that
// addends keep 24 bits from the largest of their sum's values on.
// The CTAs of a unit (row, key head) leave their scores as integers in the order of the floats;
// the last of them finds the count-th largest, T, by counting in 1,024 bins of the scores' range and then
// of the bin that it is in.  A block more than 2 E above T is chosen and one more than 2 E below is not,
// whatever the order; where those between are more than are still wanted, their defined scores decide.
//
// Measured (B200, graphs of calls): selection of 64 rows of up to 32,768 tokens in pages of 32, 64 / 8 heads: 51 us for 137 MB
// (3 CTAs an SM with half the loads: 48, but 1 us more for small calls); 1 x 131,072 in pages of 64: 14.4 us, a chain
// of accesses.  Bounds of 8 prompts of 8,191, 4 heads of 80: 15.9 us; of the pages of a step's new tokens 3.4 to 7.2.
#include "epq_paged.cuh"
#include <cfloat>

namespace epq {
namespace paged {
namespace {

__device__ int g_sparse_error = 0;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxUnits = 65536;               // counters in the workspace
constexpr int kMaxBlocks = (1 << 21) - 1;      // of a sequence, in a selection

// ---------------------------------------------------------------- bounds
struct BoundsArgs {
    PagesD pages;
    const int32_t* seq;
    const int64_t* first;
    const int64_t* lengths;
    uint16_t* bounds;
    int64_t stride;                            // values between pages
    int parts;                                 // CTAs a row
    int team;                                  // warps a head of a page
};

enum Kind { kBf16 = 0, kF16 = 1, kInt8 = 2, kFp8 = 3 };

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <typename T2> __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    const T2 r = __hmin2_nan(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T2> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const T2 r = __hmax2_nan(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Running bounds of a 16-byte chunk of a row: 8 values of a 16-bit cache as packed pairs...
template <int kKind> struct Chunk {
    using T2 = typename std::conditional<kKind == kBf16, __nv_bfloat162, __half2>::type;
    static constexpr int kBytes = 2;
    static constexpr uint32_t kInf = kKind == kBf16 ? 0x7f807f80u : 0x7c007c00u;
    uint32_t lo[4], hi[4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[i] = kInf, hi[i] = kInf | 0x80008000u;
    }
    __device__ __forceinline__ void add(const uint4& x, float) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[i] = min2<T2>(lo[i], w[i]), hi[i] = max2<T2>(hi[i], w[i]);
    }
    static constexpr int kWords = 8;
    __device__ __forceinline__ uint32_t word(int i) const { return i < 4 ? lo[i] : hi[i - 4]; }
    __device__ __forceinline__ void join(int i, uint32_t x) {          // word i of another
        if (i < 4) lo[i] = min2<T2>(lo[i], x);
        else hi[i - 4] = max2<T2>(hi[i - 4], x);
    }
    // infinities as the largest finite value
    __device__ __forceinline__ void store(uint16_t* to_lo, uint16_t* to_hi) const {
        constexpr uint32_t top = kInf - 0x00010001u, bottom = top | 0x80008000u;
        uint32_t l[4], h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            l[i] = max2<T2>(min2<T2>(lo[i], top), bottom);
            h[i] = max2<T2>(min2<T2>(hi[i], top), bottom);
        }
        *reinterpret_cast<uint4*>(to_lo) = make_uint4(l[0], l[1], l[2], l[3]);
        *reinterpret_cast<uint4*>(to_hi) = make_uint4(h[0], h[1], h[2], h[3]);
    }
};
// ... or 16 codes of an 8-bit one as the float32 values that they stand for, rounded to bf16 at the end.
template <int kKind> struct Codes {
    static constexpr int kBytes = 1;
    float lo[16], hi[16];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 16; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
    }
    __device__ __forceinline__ void add(const uint4& x, float scale) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float f[4];
            if (kKind == kInt8) {
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = (float)(int8_t)(w[i] >> (8 * j));
            } else {
                uint32_t p0, p1;
                asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %2;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n cvt.rn.f16x2.e4m3x2 %1, hi;\n}\n"
                    : "=r"(p0), "=r"(p1) : "r"(w[i]));
                const float2 a = unpack2<__half>(p0), b = unpack2<__half>(p1);
                f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = __fmul_rn(f[j], scale);
                lo[4 * i + j] = min_nan(lo[4 * i + j], v);
                hi[4 * i + j] = max_nan(hi[4 * i + j], v);
            }
        }
    }
    static constexpr int kWords = 32;
    __device__ __forceinline__ uint32_t word(int i) const { return __float_as_uint(i < 16 ? lo[i] : hi[i - 16]); }
    __device__ __forceinline__ void join(int i, uint32_t x) {
        if (i < 16) lo[i] = min_nan(lo[i], __uint_as_float(x));
        else hi[i - 16] = max_nan(hi[i - 16], __uint_as_float(x));
    }
    __device__ __forceinline__ void store(uint16_t* to_lo, uint16_t* to_hi) const {
        constexpr uint32_t top = 0x7f7f7f7fu, bottom = top | 0x80008000u;
        uint32_t l[8], h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            l[i] = max2<__nv_bfloat162>(min2<__nv_bfloat162>(pack2<__nv_bfloat16>(lo[2 * i], lo[2 * i + 1]), top), bottom);
            h[i] = max2<__nv_bfloat162>(min2<__nv_bfloat162>(pack2<__nv_bfloat16>(hi[2 * i], hi[2 * i + 1]), top), bottom);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            reinterpret_cast<uint4*>(to_lo)[i] = make_uint4(l[4 * i], l[4 * i + 1], l[4 * i + 2], l[4 * i + 3]);
            reinterpret_cast<uint4*>(to_hi)[i] = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
        }
    }
};

// Length and sequence of row b, or a length of 0 with the error noted.
__device__ __forceinline__ int row_length(const PagesD& P, const int32_t* seq, const int64_t* lengths, int b, int* s, bool report) {
    const int64_t n = lengths[b];
    *s = seq ? seq[b] : b;
    if (n < 0 || n > (int64_t)P.max_pages * P.page_size || (n > 0 && (*s < 0 || *s >= P.seqs))) {
        if (report) atomicOr(&g_sparse_error, kBadPosition);
        return 0;
    }
    return (int)n;
}

template <int kKind>
__global__ void __launch_bounds__(kThreads) bounds_kernel(const BoundsArgs A) {
    using C = typename std::conditional<kKind <= kF16, Chunk<kKind>, Codes<kKind>>::type;
    __shared__ uint32_t shared[C::kWords][kWarps][32];
    pdl_enter();
    const PagesD& P = A.pages;
    const int b = blockIdx.x / A.parts, part = blockIdx.x - b * A.parts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int s;
    const int n = row_length(P, A.seq, A.lengths, b, &s, threadIdx.x == 0 && part == 0);
    const int64_t from = A.first ? A.first[b] : 0;
    if (from < 0) {
        if (threadIdx.x == 0 && part == 0) atomicOr(&g_sparse_error, kBadPosition);
        return;
    }
    if (n == 0 || from >= n) return;
    const int ps = P.page_size, hd = P.head_dim, team = A.team, teams = kWarps / team;
    const int member = warp % team, first = part * teams + warp / team;        // the team's first item
    const int c0 = P.page_of((int)from), cols = P.page_of(n - 1) + 1 - c0;
    const int chunks = hd * C::kBytes / 16, rows = 32 / chunks;        // of a row; rows an access
    const int row = lane / chunks, ch = lane - row * chunks;
    const bool on = row < rows;
    const int items = cols * P.kv_heads;                               // (below 2^31: a page has at least its heads' tokens)
    auto together = [&]() {                                            // the team's warps
        if (team > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / team), "r"(team * 32) : "memory");
    };
    for (int i = first; i < items; i += A.parts * teams) {
        const int col = c0 + i / P.kv_heads, head = i % P.kv_heads;
        const int64_t page = P.table[(int64_t)s * P.table_stride + col];
        if (page < 0 || page >= P.pages) {
            if (lane == 0 && member == 0) atomicOr(&g_sparse_error, kBadPage);
            continue;
        }
        const int tokens = min(ps, n - col * ps);
        const int64_t at = page * P.page_stride + (int64_t)head * ps * hd;
        const uint4* k = reinterpret_cast<const uint4*>(P.k + at * C::kBytes) + ch;
        const float* scale = kKind >= kInt8 ? P.k_scale + page * P.scale_stride + (int64_t)head * ps : nullptr;
        C c;
        c.clear();
        constexpr int kAtOnce = 8;
        for (int t = on ? member * rows + row : tokens; t < tokens; t += kAtOnce * team * rows) {
            uint4 x[kAtOnce];
            float f[kAtOnce];
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) {
                const int u = min(t + e * team * rows, tokens - 1);    // (a row twice changes no bound)
                x[e] = __ldg(k + (int64_t)u * chunks);
                f[e] = kKind >= kInt8 ? __ldg(scale + u) : 1.f;
            }
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) c.add(x[e], f[e]);
        }
        __syncwarp();
        for (int r = rows; r > 1;) {                                   // the upper rows' lanes into the lower ones'
            const int half = (r + 1) / 2, other = (lane + half * chunks) & 31;
            const bool take = row + half < r;
#pragma unroll
            for (int w = 0; w < C::kWords; ++w) {
                const uint32_t x = __shfl_sync(kAll, c.word(w), other);
                if (take) c.join(w, x);
            }
            r = half;
        }
        if (team > 1) {                                                // the other warps into the first
            if (member && row == 0)
#pragma unroll
                for (int w = 0; w < C::kWords; ++w) shared[w][warp][lane] = c.word(w);
            together();
            if (!member && row == 0)
                for (int m = 1; m < team; ++m)
#pragma unroll
                    for (int w = 0; w < C::kWords; ++w) c.join(w, shared[w][warp + m][lane]);
        }
        if (row == 0 && !member) {
            uint16_t* to = A.bounds + page * A.stride + (int64_t)head * 2 * hd + ch * (16 / C::kBytes);
            c.store(to, to + hd);
        }
        together();                                                    // (the words are read)
    }
}

// ---------------------------------------------------------------- selection
struct SelectArgs {
    PagesD pages;
    const uint16_t* bounds;
    int64_t stride;
    const void* q;
    int64_t q_row, q_head;
    const int32_t* seq;
    const int64_t* lengths;
    int32_t* chosen;
    uint32_t* keys;                            // [units][max_pages]
    float* largest;                            // [units][parts]: max|bounds|
    unsigned* counters;
    int heads, group, dtype, q_aligned, count, sinks, recent, parts;
};

// Integers in the order of the floats; -0 is 0 and NaN the largest.
__device__ __forceinline__ uint32_t key_of(float s) {
    if (s != s) return kAll;
    const uint32_t u = __float_as_uint(s + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

// Where the `need`-th largest of some keys lies (1 <= need <= their number): in [low, high], with `above` of them past high.
// Counted in 1024 bins of the range, then in 1024 of the bin it is in, until `stop` or fewer keys are left or low = high.
constexpr int kBins = 1024;
struct Place {
    uint32_t low, high;
    int above;
};
template <typename F> __device__ Place find_place(int need, int stop, int j0, int j1, const F& key_at) {
    __shared__ int bins[kBins], sums[kWarps], found[3];
    __shared__ uint32_t ends[2][kWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    Place at = {kAll, 0u, 0};
    for (int j = j0 + tid; j < j1; j += kThreads) {
        const uint32_t key = key_at(j);
        at.low = min(at.low, key);
        at.high = max(at.high, key);
    }
    at.low = __reduce_min_sync(kAll, at.low);
    at.high = __reduce_max_sync(kAll, at.high);
    __syncthreads();                                                   // (an earlier call's are read)
    if (lane == 0) ends[0][warp] = at.low, ends[1][warp] = at.high;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) at.low = min(at.low, ends[0][w]), at.high = max(at.high, ends[1][w]);
    while (true) {
        const int shift = max(0, 22 - __clz(at.high - at.low));        // (the range's bits less 10)
        constexpr int kMine = kBins / kThreads;
#pragma unroll
        for (int i = 0; i < kMine; ++i) bins[tid + i * kThreads] = 0;
        __syncthreads();
        for (int j = j0 + tid; j < j1; j += kThreads) {
            const uint32_t key = key_at(j);
            if (key >= at.low && key <= at.high) atomicAdd(&bins[(key - at.low) >> shift], 1);
        }
        __syncthreads();
        // thread 0 has the last bins
        int have[kMine], all = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) all += have[i] = bins[kBins - 1 - tid * kMine - i];
        int upto = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(kAll, upto, o);
            if (lane >= o) upto += u;
        }
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        int before = at.above + upto - all;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) before += w < warp ? sums[w] : 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            if (before < need && before + have[i] >= need) found[0] = kBins - 1 - tid * kMine - i, found[1] = before, found[2] = have[i];
            before += have[i];
        }
        __syncthreads();
        at.low += (uint32_t)found[0] << shift;
        at.high = at.low + min(at.high - at.low, (1u << shift) - 1u);  // (a bin of NaN's key may end past 2^32)
        at.above = found[1];
        if (found[2] <= stop || shift == 0) return at;
        __syncthreads();                                               // (found and sums are read)
    }
}

// 8 values of a row of q from dim on.
__device__ __forceinline__ void load_q(const SelectArgs& A, int b, int h, int dim, float (&f)[8]) {
    const uint16_t* q = static_cast<const uint16_t*>(A.q) + b * A.q_row + h * A.q_head + dim;
    if (A.dtype == EPQ_BF16) {
        Eight<__nv_bfloat16> x;
        x.load(reinterpret_cast<const __nv_bfloat16*>(q), A.q_aligned);
        x.get(f);
    } else {
        Eight<__half> x;
        x.load(reinterpret_cast<const __half*>(q), A.q_aligned);
        x.get(f);
    }
}

// The defined score of a block of row b's key head, by a warp: as many lanes a query head as hold its dims, 8 each;
// neighbours' sums first.
template <typename T> __device__ float defined_score(const SelectArgs& A, int b, int head, const T* bounds) {
    const int lane = threadIdx.x & 31, hd = A.pages.head_dim;
    int lanes = 2;
    while (lanes * 8 < hd) lanes *= 2;
    const int dim = lane % lanes * 8;
    float lo[8], hi[8], score = -INFINITY;
    const bool on = dim < hd;
    if (on) {
        load_v<T, 8>(lo, bounds + dim);
        load_v<T, 8>(hi, bounds + hd + dim);
    }
#pragma unroll 4
    for (int h0 = 0; h0 < A.group; h0 += 32 / lanes) {
        const int h = h0 + lane / lanes;
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = 0.f;
        if (on && h < A.group) {
            load_q(A, b, head * A.group + h, dim, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = max_nan(__fmul_rn(t[i], lo[i]), __fmul_rn(t[i], hi[i]));
        }
        float v = __fadd_rn(__fadd_rn(__fadd_rn(t[0], t[1]), __fadd_rn(t[2], t[3])),
                            __fadd_rn(__fadd_rn(t[4], t[5]), __fadd_rn(t[6], t[7])));
        for (int o = 1; o < lanes; o <<= 1) v = __fadd_rn(v, __shfl_xor_sync(kAll, v, o));
        if (h < A.group) score = max_nan(score, v);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) score = max_nan(score, __shfl_xor_sync(kAll, score, o));
    return score;
}

// The unit's list: the first `sinks` and last `recent` of its n > count blocks and the best of
// the others, ties to the lowest block, in ascending order.  The keys' scores are off by at most `err`;
// NaN: by any amount.
constexpr int kLocal = 4096;                                           // keys that shared memory holds
template <typename T>
__device__ void choose(const SelectArgs& A, uint32_t* keys, int n, int b, int head, const int32_t* table, float err, int32_t* out) {
    constexpr int kListed = 1024, kFew = 8;
    __shared__ int before[kWarps][3];
    __shared__ uint32_t local[kLocal];
    __shared__ int list[kListed], listed;
    __shared__ uint32_t defined[kListed];
    const PagesD& P = A.pages;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int first = A.sinks, past = n - A.recent;
    const int need = A.count - A.sinks - A.recent;                     // n > count: the two do not meet
    const bool here = n <= kLocal;
    if (here)
        for (int j = tid; j < n; j += kThreads) local[j] = __ldcg(keys + j);
    if (tid == 0) listed = 0;
    __syncthreads();
    auto key_at = [&](int j) { return here ? local[j] : __ldcg(keys + j); };
    auto set_key = [&](int j, uint32_t key) { (here ? local : keys)[j] = key; };
    auto defined_key = [&](int j) {                                    // (of a block with a page: its key is not 0)
        const T* bounds = reinterpret_cast<const T*>(A.bounds) + table[j] * A.stride + (int64_t)head * 2 * P.head_dim;
        return key_of(defined_score<T>(A, b, head, bounds));
    };
    // chosen: keys above `over`, and of those that equal it as many as are still wanted
    uint32_t over = kAll;
    if (need > 0) {
        Place at = find_place(need, kFew, first, past, key_at);
        bool few = false;
        for (int attempt = 0; attempt < 2; ++attempt) {
            // those that are in the place, or that the error may bring there
            const float from = score_of(at.low) - 2.f * err, to = score_of(at.high) + 2.f * err;
            const bool sure = from > -FLT_MAX && to < FLT_MAX;         // (false with NaN)
            const uint32_t low = key_of(from), high = key_of(to);
            if (!sure && err != 0.f) break;
            if (attempt == 0 && err == 0.f) {                          // scores of no error: nothing to look up
                at = find_place(need, 0, first, past, key_at);
                break;
            }
            int above = 0;
            for (int j = first + tid; j < past; j += kThreads) {
                const uint32_t key = key_at(j);
                above += key > high;
                if (key >= low && key <= high) {
                    const int i = atomicAdd(&listed, 1);               // (in any order: they are ranked below)
                    if (i < kListed) list[i] = j;
                }
            }
            above = __reduce_add_sync(kAll, above);
            if (lane == 0) before[warp][0] = above;
            __syncthreads();
            int all_above = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) all_above += before[w][0];
            const int count = listed, wanted = need - all_above;       // (1 <= wanted <= count)
            few = count <= kListed;
            if (few) {
                over = high;
                for (int i = warp; i < count && count > wanted; i += kWarps) {
                    const uint32_t key = defined_key(list[i]);
                    if (lane == 0) defined[i] = key;
                }
                __syncthreads();
                for (int i = tid; i < count; i += kThreads) {
                    int better = 0;
                    for (int e = 0; e < count && count > wanted; ++e)
                        better += defined[e] > defined[i] || (defined[e] == defined[i] && list[e] < list[i]);
                    set_key(list[i], better < wanted ? kAll : 0u);
                }
                __syncthreads();
                break;
            }
            __syncthreads();
            if (tid == 0) listed = 0;
            at = find_place(need, 0, first, past, key_at);
        }
        if (!few) {
            if (err != 0.f) {                                          // every score anew
                __syncthreads();
                for (int j = first + warp; j < past; j += kWarps) {
                    if (key_at(j) == 0u) continue;                     // (no page)
                    const uint32_t key = defined_key(j);
                    __syncwarp();
                    if (lane == 0) set_key(j, key);
                }
                __syncthreads();
                at = find_place(need, 0, first, past, key_at);
            }
            over = at.low;
        }
    }
    // a warp an eighth of the blocks: how many are above, how many equal
    const int each = (n + kThreads - 1) / kThreads * 32, w0 = min(n, warp * each), w1 = min(n, w0 + each);
    int sure = 0, ties = 0, forced = 0;
    auto look = [&](int j0, unsigned* above, unsigned* equal) {
        const int j = j0 + lane;
        const bool edge = j < w1 && (j < first || j >= past), in = j < w1 && !edge && need > 0;
        const uint32_t key = in ? key_at(j) : 0u;
        *above = __ballot_sync(kAll, edge || (in && key > over));
        *equal = __ballot_sync(kAll, in && key == over);
        return __popc(__ballot_sync(kAll, edge));
    };
    for (int j0 = w0; j0 < w1; j0 += 32) {
        unsigned above, equal;
        forced += look(j0, &above, &equal);
        sure += __popc(above);
        ties += __popc(equal);
    }
    __syncthreads();
    if (lane == 0) before[warp][0] = sure, before[warp][1] = ties, before[warp][2] = forced;
    __syncthreads();
    int all_sure = 0, all_forced = 0, sure_to = 0, ties_to = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        all_sure += before[w][0];
        all_forced += before[w][2];
        if (w < warp) sure_to += before[w][0], ties_to += before[w][1];
    }
    const int take = need - (all_sure - all_forced);                   // ties that are chosen
    for (int j0 = w0; j0 < w1; j0 += 32) {
        unsigned above, equal;
        look(j0, &above, &equal);
        const unsigned below = (1u << lane) - 1u;
        const int s = sure_to + __popc(above & below), t = ties_to + __popc(equal & below);
        if (above >> lane & 1) out[s + min(t, take)] = j0 + lane;
        else if ((equal >> lane & 1) && t < take) out[s + t] = j0 + lane;
        sure_to += __popc(above);
        ties_to += __popc(equal);
    }
}

template <bool kIsBf16>
__device__ __forceinline__ void multiply(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (kIsBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Heads of up to 32 kSteps.  Lane 4 g + c holds 8 dims from 32 i + 8 c on of rows g and g + 8 (blocks) and of column g (a
// head): any order of the dims is one, if it is the same in both.
constexpr int kRows = 16, kColumns = 8;

template <bool kIsBf16, int kSteps>
__global__ void __launch_bounds__(kThreads, 2) select_kernel(const SelectArgs A) {
    using T = typename std::conditional<kIsBf16, __nv_bfloat16, __half>::type;   // of the bounds
    using T2 = typename std::conditional<kIsBf16, __nv_bfloat162, __half2>::type;
    constexpr int kAtOnce = kSteps < 4 ? kSteps : 4;                   // steps whose loads are under way together
    // max(q, 0) and min(q, 0) as T, and what that leaves of an f16 q over bf16 bounds (as bf16, exact)
    __shared__ uint4 columns[2][2][kSteps][32];
    __shared__ float norms[kColumns], peaks[kColumns], largest[kWarps];
    __shared__ bool last;
    pdl_enter();
    const PagesD& P = A.pages;
    const int unit = blockIdx.x / A.parts, part = blockIdx.x - unit * A.parts;
    const int b = unit / P.kv_heads, head = unit - b * P.kv_heads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int hd = P.head_dim;
    int s;
    const int length = row_length(P, A.seq, A.lengths, b, &s, tid == 0 && part == 0 && head == 0);
    const int n = length ? P.page_of(length - 1) + 1 : 0;
    int32_t* out = A.chosen + (int64_t)unit * A.count;
    if (n <= A.count) {
        if (part == 0)
            for (int j = tid; j < A.count; j += kThreads) out[j] = j < n ? j : -1;
        return;
    }
    uint32_t* keys = A.keys + (int64_t)unit * P.max_pages;
    const int per = (n + A.parts - 1) / A.parts, begin = min(n, part * per), end = min(n, begin + per);
    const int32_t* table = P.table + (int64_t)s * P.table_stride;
    // the first blocks' pages: on their way while q is read
    auto page_at = [&](int j) { return j < end ? table[j] : -1; };
    const int first0 = page_at(begin + warp * kRows + g), first1 = page_at(begin + warp * kRows + g + 8);
    const bool two = kIsBf16 && A.dtype == EPQ_F16;
    float norm = 0.f;                                                  // the largest head's |q|_1
    T2 most;                                                           // of |bounds|
    most.x = most.y = T(0.f);
    for (int h0 = 0; h0 < A.group; h0 += kColumns) {
        __syncthreads();                                               // (the last heads' columns are read)
        {                                                              // a warp a head: |q|_1, max|q|
            float sum = 0.f, top = 0.f;
            if (h0 + warp < A.group)
                for (int d = lane * 8; d < hd; d += 256) {
                    float f[8];
                    load_q(A, b, head * A.group + h0 + warp, d, f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum += fabsf(f[i]), top = max_nan(top, fabsf(f[i]));
                }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                sum += __shfl_xor_sync(kAll, sum, o);
                top = max_nan(top, __shfl_xor_sync(kAll, top, o));
            }
            if (lane == 0) norms[warp] = sum, peaks[warp] = top;
        }
        __syncthreads();
        // a bf16 q over f16 bounds is brought to f16 by a power of two
        auto lift_of = [&](int h) {
            const float top = peaks[h];
            return !kIsBf16 && A.dtype == EPQ_BF16 && top >= 1e-33f && top < INFINITY ? ldexpf(1.f, -ilogbf(top)) : 1.f;
        };
#pragma unroll
        for (int h = 0; h < kColumns; ++h) norm = max_nan(norm, norms[h]);
        for (int e = tid; e < kSteps * 32; e += kThreads) {
            const int i = e / 32, h = e % 32 >> 2, dim = 32 * i + 8 * (e & 3);
            float f[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = 0.f;
            if (dim < hd && h0 + h < A.group) load_q(A, b, head * A.group + h0 + h, dim, f);
            const float lift = lift_of(h);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t w[2][4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    float v[2], rest[2];
                    T2 near, left;
#pragma unroll
                    for (int y = 0; y < 2; ++y) v[y] = half ? min_nan(f[2 * x + y] * lift, 0.f) : max_nan(f[2 * x + y] * lift, 0.f);
                    near.x = T(v[0]), near.y = T(v[1]);
#pragma unroll
                    for (int y = 0; y < 2; ++y) rest[y] = v[y] - (float)(y ? near.y : near.x);
                    left.x = T(rest[0]), left.y = T(rest[1]);
                    w[0][x] = *reinterpret_cast<uint32_t*>(&near);
                    w[1][x] = *reinterpret_cast<uint32_t*>(&left);
                }
                columns[0][half][i][e % 32] = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
                columns[1][half][i][e % 32] = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
            }
        }
        __syncthreads();
        const bool is0 = h0 + 2 * c < A.group, is1 = h0 + 2 * c + 1 < A.group;
        const float back0 = 1.f / lift_of(2 * c), back1 = 1.f / lift_of(2 * c + 1);
        const int stride = kWarps * kRows;
        int next0 = first0, next1 = first1;
        for (int j = begin + warp * kRows; j < end; j += stride) {
            const int page0 = next0, page1 = next1;
            const bool good0 = page0 >= 0 && page0 < P.pages, good1 = page1 >= 0 && page1 < P.pages;
            next0 = page_at(j + stride + g);
            next1 = page_at(j + stride + g + 8);
            const uint16_t* from0 = A.bounds + (good0 ? page0 : 0) * A.stride + (int64_t)head * 2 * hd + 8 * c;
            const uint16_t* from1 = A.bounds + (good1 ? page1 : 0) * A.stride + (int64_t)head * 2 * hd + 8 * c;
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i0 = 0; i0 < kSteps; i0 += kAtOnce) {
                uint4 x[2][kAtOnce], y[2][kAtOnce];                    // rows g and g + 8; hi, lo
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const int dim = 32 * (i0 + i), at = (half ? 0 : hd) + dim;
                        x[half][i] = y[half][i] = make_uint4(0, 0, 0, 0);
                        if (good0 && dim + 8 * c < hd) x[half][i] = __ldg(reinterpret_cast<const uint4*>(from0 + at));
                        if (good1 && dim + 8 * c < hd) y[half][i] = __ldg(reinterpret_cast<const uint4*>(from1 + at));
                    }
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const uint4 u = x[half][i], v = y[half][i], w = columns[0][half][i0 + i][lane];
                        multiply<kIsBf16>(d, u.x, v.x, u.y, v.y, w.x, w.y);
                        multiply<kIsBf16>(d, u.z, v.z, u.w, v.w, w.z, w.w);
                        if (two) {
                            const uint4 z = columns[1][half][i0 + i][lane];
                            multiply<kIsBf16>(d, u.x, v.x, u.y, v.y, z.x, z.y);
                            multiply<kIsBf16>(d, u.z, v.z, u.w, v.w, z.z, z.w);
                        }
                        if (h0 == 0) {
                            const uint32_t words[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int e = 0; e < 8; ++e) most = __hmax2_nan(most, __habs2(*reinterpret_cast<const T2*>(&words[e])));
                        }
                    }
            }
            float score0 = max_nan(is0 ? d[0] * back0 : -INFINITY, is1 ? d[1] * back1 : -INFINITY);
            float score1 = max_nan(is0 ? d[2] * back0 : -INFINITY, is1 ? d[3] * back1 : -INFINITY);
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                score0 = max_nan(score0, __shfl_xor_sync(kAll, score0, o));
                score1 = max_nan(score1, __shfl_xor_sync(kAll, score1, o));
            }
            const int mine = j + g + 8 * c;                            // lanes c = 0 and 1 write
            if (c < 2 && mine < end) {
                const bool good = c ? good1 : good0;
                if (!good) atomicOr(&g_sparse_error, kBadPage);
                const uint32_t key = good ? key_of(c ? score1 : score0) : 0u;
                keys[mine] = h0 ? max(keys[mine], key) : key;
            }
        }
    }
    {
        float top = max_nan((float)most.x, (float)most.y);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(kAll, top, o));
        if (lane == 0) largest[warp] = top;
    }
    __syncthreads();
    if (tid == 0) {
        float top = 0.f;
        for (int w = 0; w < kWarps; ++w) top = max_nan(top, largest[w]);
        A.largest[blockIdx.x] = top;
        // releases the CTA's keys (complete at the barrier above), acquires the others'
        unsigned done;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(done) : "l"(A.counters + unit) : "memory");
        last = done == (unsigned)A.parts - 1;
        if (last) A.counters[unit] = 0u;
    }
    __syncthreads();
    if (!last) return;
    float top = 0.f;
    for (int p = lane; p < A.parts; p += 32) top = max_nan(top, __ldcg(A.largest + unit * A.parts + p));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(kAll, top, o));
    // Exact where all is zero; values that the tensor cores may take for zeros are nothing beside 1e-30.  Each product is
    // cut off once and each of the head_dim / 8 sums twice; an f16 q over bf16 bounds has two parts, a lifted bf16 q is off by 2^-25 of
    // its largest value.
    float err = NAN;
    if (top < INFINITY && norm < INFINITY) {
        const float steps = (two || !kIsBf16 ? 3.f : 1.5f) * (float)hd + 8.f;
        if (top == 0.f || norm == 0.f) err = 0.f;
        else if (top >= 1e-30f && norm >= 1e-30f && norm * top < 1e37f) err = steps * 0x1p-23f * 1.05f * (norm * top) + 1e-35f;
    }
    choose<T>(A, keys, n, b, head, table, err, out);
}

template <bool kIsBf16> int launch_select(const SelectArgs& A, unsigned grid, cudaStream_t st) {
    auto go = [&](auto kern) { return launch(kern, dim3(grid), dim3(kThreads), 0, st, "epq_paged_select", A); };
    const int hd = A.pages.head_dim;
    if (hd <= 64) return go(select_kernel<kIsBf16, 2>);
    if (hd <= 128) return go(select_kernel<kIsBf16, 4>);
    return go(select_kernel<kIsBf16, 8>);
}

// Bounds are held in the cache's own 16-bit type, or in bf16 for 8-bit caches.
int check_bounds(const epq_pages* pages, PagesD* P, const void* bounds, int64_t stride, int dtype, const char* who) {
    const int rc = make_pages(pages, P, who);
    if (rc != EPQ_OK) return rc;
    if (dtype != EPQ_BF16 && dtype != EPQ_F16) return set_error(EPQ_EDTYPE, "%s: bounds of dtype %d (f16 or bf16)", who, dtype);
    if (P->format != EPQ_CACHE_SAME && dtype != EPQ_BF16)
        return set_error(EPQ_EDTYPE, "%s: the bounds of an 8-bit cache are bf16", who);
    if (!bounds) return set_error(EPQ_EINVAL, "%s: bounds is NULL", who);
    if ((uintptr_t)bounds % 16 || stride % 8)
        return set_error(EPQ_EALIGN, "%s: bounds must be 16-byte aligned, pages a multiple of 8 values apart", who);
    if (stride < (int64_t)P->kv_heads * 2 * P->head_dim)
        return set_error(EPQ_ESHAPE, "%s: bounds of pages %lld values apart", who, (long long)stride);
    return EPQ_OK;
}

}  // namespace

int sparse_read_device_error(int* flag) {
    if (cudaMemcpyFromSymbol(flag, g_sparse_error, sizeof(int)) != cudaSuccess)
        return check_launch("read paged selection error flag");
    return EPQ_OK;
}

}  // namespace paged
}  // namespace epq

using namespace epq;
using namespace epq::paged;

extern "C" {

int epq_paged_bounds(const epq_pages* pages, void* bounds, int64_t bounds_stride, int32_t dtype, const int32_t* seq,
                     const int64_t* first, const int64_t* lengths, int64_t batch, void* stream) {
    BoundsArgs A = {};
    const int rc = check_bounds(pages, &A.pages, bounds, bounds_stride, dtype, "epq_paged_bounds");
    if (rc != EPQ_OK) return rc;
    const PagesD& P = A.pages;
    if (batch < 0 || batch > kMaxUnits) return set_error(EPQ_EINVAL, "epq_paged_bounds: batch=%lld", (long long)batch);
    if ((int64_t)P.max_pages * P.kv_heads > INT32_MAX / 2)
        return set_error(EPQ_EUNSUPPORTED, "epq_paged_bounds: %d pages of %d heads a sequence", P.max_pages, P.kv_heads);
    if (!seq && batch > P.seqs)
        return set_error(EPQ_ESHAPE, "epq_paged_bounds: batch=%lld of a table of %d sequences", (long long)batch, P.seqs);
    if (batch == 0) return EPQ_OK;
    if (!lengths) return set_error(EPQ_EINVAL, "epq_paged_bounds: lengths is NULL");
    A.seq = seq;
    A.first = first;
    A.lengths = lengths;
    A.bounds = static_cast<uint16_t*>(bounds);
    A.stride = bounds_stride;
    // warps a head of a page: 8 accesses of 512 bytes each
    const int64_t bytes = (int64_t)P.page_size * P.head_dim * (P.format == EPQ_CACHE_SAME ? 2 : 1);
    A.team = 1;
    while (A.team < kWarps && A.team * 4096 < bytes) A.team *= 2;
    // enough CTAs a row to fill the card where all of its pages are new
    const int64_t most = cdiv((int64_t)P.max_pages * P.kv_heads * A.team, kWarps), fill = cdiv(8LL * device_sms(), batch);
    A.parts = (int)(most < fill ? most : fill);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto kern) {
        return launch(kern, dim3((unsigned)(batch * A.parts)), dim3(kThreads), 0, st, "epq_paged_bounds", A);
    };
    if (P.format == EPQ_CACHE_INT8) return go(bounds_kernel<kInt8>);
    if (P.format == EPQ_CACHE_FP8) return go(bounds_kernel<kFp8>);
    return dtype == EPQ_BF16 ? go(bounds_kernel<kBf16>) : go(bounds_kernel<kF16>);
}

int64_t epq_paged_select_workspace_bytes(const epq_pages* pages, int64_t batch) {
    PagesD P;
    const int rc = make_pages(pages, &P, "epq_paged_select_workspace_bytes");
    if (rc != EPQ_OK) return rc;
    if (P.max_pages > kMaxBlocks)
        return set_error(EPQ_EUNSUPPORTED, "epq_paged_select: %d pages a sequence (at most %d)", P.max_pages, kMaxBlocks);
    if (batch < 0 || batch * P.kv_heads > kMaxUnits)
        return set_error(EPQ_EUNSUPPORTED, "epq_paged_select: batch=%lld of %d key heads (at most %d units)", (long long)batch,
                         P.kv_heads, kMaxUnits);
    // counters, keys, the parts' largest bounds
    return (int64_t)kMaxUnits * 4 + batch * P.kv_heads * ((int64_t)P.max_pages + cdiv(P.max_pages, kRows * kWarps)) * 4;
}

int epq_paged_select(const epq_pages* pages, const void* bounds, int64_t bounds_stride, int32_t bounds_dtype,
                     const epq_heads* q, int32_t dtype, const int32_t* seq, const int64_t* lengths, int64_t batch,
                     int32_t count, int32_t sinks, int32_t recent, int32_t* chosen, void* workspace, int64_t workspace_bytes,
                     void* stream) {
    SelectArgs A = {};
    const int rc = check_bounds(pages, &A.pages, bounds, bounds_stride, bounds_dtype, "epq_paged_select");
    if (rc != EPQ_OK) return rc;
    const PagesD& P = A.pages;
    if (!q || batch < 0 || count < 1 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > count)
        return set_error(EPQ_EINVAL, "epq_paged_select: count=%d, sinks=%d, recent=%d (sinks + recent <= count)", count, sinks,
                         recent);
    if (dtype != EPQ_BF16 && dtype != EPQ_F16)
        return set_error(EPQ_EDTYPE, "epq_paged_select: dtype %d (f16 or bf16)", dtype);
    if (q->heads <= 0 || q->heads % P.kv_heads)
        return set_error(EPQ_ESHAPE, "epq_paged_select: %d query heads over %d key heads", q->heads, P.kv_heads);
    if (!seq && batch > P.seqs)
        return set_error(EPQ_ESHAPE, "epq_paged_select: batch=%lld of a table of %d sequences", (long long)batch, P.seqs);
    const int64_t need = epq_paged_select_workspace_bytes(pages, batch);
    if (need < 0) return (int)need;
    if (batch == 0) return EPQ_OK;
    if (!q->data || !lengths || !chosen) return set_error(EPQ_EINVAL, "epq_paged_select: NULL q, lengths or chosen");
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
        return set_error(EPQ_EWORKSPACE, "epq_paged_select: workspace of %lld bytes (need %lld, 256-aligned)",
                         (long long)workspace_bytes, (long long)need);
    A.bounds = static_cast<const uint16_t*>(bounds);
    A.stride = bounds_stride;
    A.q = q->data;
    A.q_row = q->stride_row;
    A.q_head = q->stride_head;
    A.q_aligned = heads_aligned(*q, 2, 16);
    A.seq = seq;
    A.lengths = lengths;
    A.chosen = chosen;
    A.counters = static_cast<unsigned*>(workspace);
    A.keys = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + (int64_t)kMaxUnits * 4);
    A.heads = q->heads;
    A.group = q->heads / P.kv_heads;
    A.dtype = dtype;
    A.count = count;
    A.sinks = sinks;
    A.recent = recent;
    // CTAs a unit: enough to fill the card twice (lengths differ), each with a step of its warps
    const int64_t units = batch * P.kv_heads, fill = cdiv(4LL * device_sms(), units), most = cdiv(P.max_pages, kRows * kWarps);
    A.parts = (int)(fill < most ? fill : most);
    A.largest = reinterpret_cast<float*>(A.keys + units * P.max_pages);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)(units * A.parts);
    return bounds_dtype == EPQ_BF16 ? launch_select<true>(A, grid, st) : launch_select<false>(A, grid, st);
}

}  // extern "C"
