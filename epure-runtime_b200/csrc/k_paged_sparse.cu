// What a cheap score needs and chooses of a paged cache: the bounds of every page's keys
// (epq_paged_bounds) and, for each row and key head, the blocks (pages) to attend over
// (epq_paged_select).
//
//   lo[d], hi[d] = min, max over the page's tokens of K[t, d]
//   score = max over the key head's query heads of  sum_d max(q_d lo_d, q_d hi_d)
//
// which no q . K[t] of the page passes.  A product of two 16-bit values is exact in float32
// and the sum's order is fixed (neighbours, then neighbours of their sums), so which blocks
// are chosen is the same wherever it is computed in float32.
//
// Bounds.  Bound: HBM, one read of the keys; for the pages of a decode step the chain of length,
// page and keys.  Up to 8 warps share one head of one page, so that a page is two accesses deep;
// a warp's lanes hold 16 bytes of a row each, the rows of an access side by side.
//
// Selection.  Bound: HBM, 4 head_dim bytes a block and head; next to it the issue rate, about
// 1.5 instructions a dim, block and query head.  A lane holds 8 dims of two blocks; q lies in
// shared memory as max(q, 0) and min(q, 0), so that max(q lo, q hi) = max(q, 0) hi + min(q, 0) lo
// is a product and a fused product of two dims at once (one of the two is zero: nothing is
// rounded).  The lanes of a block then add up all its heads together: each step halves the heads
// a lane holds.  The CTAs of a unit (row, key head) leave its scores as integers in the order of
// the floats; the last of them finds the count-th largest, two bits at a time, and writes the list.
#include "epq_paged.cuh"

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
    unsigned* counters;
    int heads, group, dtype, q_aligned, count, sinks, recent, parts;
};

__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float add_halves(uint64_t a) {
    float x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a));
    return x + y;
}

// Integers in the order of the floats; -0 is 0 and NaN the largest.
__device__ __forceinline__ uint32_t key_of(float s) {
    if (s != s) return kAll;
    const uint32_t u = __float_as_uint(s + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// The unit's list: the first `sinks` and last `recent` of its n > count blocks and the best of
// the others, ties to the lowest block, in ascending order.
__device__ void choose(const SelectArgs& A, const uint32_t* keys, int n, int32_t* out) {
    constexpr int kHeld = 16;                                          // keys of a thread that stay in registers
    __shared__ int64_t sums[2][kWarps];
    __shared__ int before[kWarps][3];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int each = (n + kThreads - 1) / kThreads, j0 = min(n, tid * each), j1 = min(n, j0 + each);
    const int past = n - A.recent;
    const int need = A.count - A.sinks - A.recent;                     // n > count: the two do not meet
    auto free_key = [&](int j) { return j < A.sinks || j >= past ? 0u : __ldcg(keys + j); };
    uint32_t held[kHeld];
    const bool in_registers = each <= kHeld;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = in_registers && j0 + i < j1 ? free_key(j0 + i) : 0u;
    // the largest value that at least `need` keys reach, two bits at a time: of the three next values the largest that
    // so many reach (their counts in 21 bits each; a unit has below 2^21 blocks)
    uint32_t at = 0;
    for (int bit = 30; bit >= 0; bit -= 2) {
        const uint32_t to1 = at | 1u << bit, to2 = at | 2u << bit, to3 = at | 3u << bit;
        int have1 = 0, have2 = 0, have3 = 0;
        auto count = [&](uint32_t key) { have1 += key >= to1, have2 += key >= to2, have3 += key >= to3; };
        if (in_registers) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (i >= each) break;
                count(held[i]);
            }
        } else {
            for (int j = j0; j < j1; ++j) count(free_key(j));
        }
        const int h1 = __reduce_add_sync(kAll, have1), h2 = __reduce_add_sync(kAll, have2), h3 = __reduce_add_sync(kAll, have3);
        int64_t* const mine = sums[bit / 2 & 1];
        if (lane == 0) mine[warp] = h1 | (int64_t)h2 << 21 | (int64_t)h3 << 42;
        __syncthreads();
        int64_t total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) total += mine[w];
        constexpr int kMask = (1 << 21) - 1;
        if ((int)(total >> 42) >= need) at = to3;
        else if ((int)(total >> 21 & kMask) >= need) at = to2;
        else if ((int)(total & kMask) >= need) at = to1;
    }
    // sure ones and ties before this thread's blocks
    int sure = 0, ties = 0, above = 0;
    for (int j = j0; j < j1; ++j) {
        const bool forced = j < A.sinks || j >= past;
        const uint32_t key = free_key(j);
        above += !forced && key > at;
        sure += forced || key > at;
        ties += !forced && key == at;
    }
    int sure_to = sure, ties_to = ties;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(kAll, sure_to, o), c = __shfl_up_sync(kAll, ties_to, o);
        if (lane >= o) sure_to += a, ties_to += c;
    }
    above = __reduce_add_sync(kAll, above);
    if (lane == 31) before[warp][0] = sure_to, before[warp][1] = ties_to, before[warp][2] = above;
    __syncthreads();
    int all_above = 0;
    sure_to -= sure;
    ties_to -= ties;
    for (int w = 0; w < kWarps; ++w) {
        all_above += before[w][2];
        if (w < warp) sure_to += before[w][0], ties_to += before[w][1];
    }
    const int take = need - all_above;                                 // ties that are chosen
    for (int j = j0; j < j1; ++j) {
        const bool forced = j < A.sinks || j >= past;
        const uint32_t key = free_key(j);
        if (forced || key > at) {
            out[sure_to + min(ties_to, take)] = j;
            ++sure_to;
        } else if (key == at) {
            if (ties_to < take) out[sure_to + ties_to] = j;
            ++ties_to;
        }
    }
}

// kLanes lanes a block, 8 dims each; kHeads query heads at once.
template <bool kIsBf16, int kLanes, int kHeads>
__global__ void __launch_bounds__(kThreads, 2) select_kernel(const SelectArgs A) {
    using T = typename std::conditional<kIsBf16, __nv_bfloat16, __half>::type;   // of the bounds
    // of a head and a lane's dims (i, i + 4): max(q, 0) of i = 0, 1 and 2, 3, min(q, 0) of the same
    __shared__ float4 split[kHeads][4][kLanes];
    __shared__ bool last;
    pdl_enter();
    const PagesD& P = A.pages;
    const int unit = blockIdx.x / A.parts, part = blockIdx.x - unit * A.parts;
    const int b = unit / P.kv_heads, head = unit - b * P.kv_heads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hd = P.head_dim;
    int s;
    const int length = row_length(P, A.seq, A.lengths, b, &s, threadIdx.x == 0 && part == 0 && head == 0);
    const int n = length ? P.page_of(length - 1) + 1 : 0;
    int32_t* out = A.chosen + (int64_t)unit * A.count;
    if (n <= A.count) {
        if (part == 0)
            for (int j = threadIdx.x; j < A.count; j += kThreads) out[j] = j < n ? j : -1;
        return;
    }
    uint32_t* keys = A.keys + (int64_t)unit * P.max_pages;
    constexpr int kGroups = 32 / kLanes, kEach = 2, kStep = kGroups * kEach;   // blocks of a warp's step
    const int sub = lane / kLanes, mine = lane % kLanes, dim = mine * 8;
    const bool on = dim < hd;
    const int per = (n + A.parts - 1) / A.parts, end = min(n, (part + 1) * per);
    const int32_t* table = P.table + (int64_t)s * P.table_stride;
    for (int h0 = 0; h0 < A.group; h0 += kHeads) {
        if (h0) __syncthreads();
        for (int e = threadIdx.x; e < kHeads * kLanes; e += kThreads) {
            const int h = e / kLanes, l = e % kLanes;
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = 0.f;
            if (8 * l < hd && h0 + h < A.group) {
                const uint16_t* q = static_cast<const uint16_t*>(A.q) + b * A.q_row + (head * A.group + h0 + h) * A.q_head + 8 * l;
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
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                split[h][i][l] = make_float4(max_nan(f[2 * i], 0.f), max_nan(f[2 * i + 4], 0.f), max_nan(f[2 * i + 1], 0.f),
                                             max_nan(f[2 * i + 5], 0.f));
                split[h][2 + i][l] = make_float4(min_nan(f[2 * i], 0.f), min_nan(f[2 * i + 4], 0.f), min_nan(f[2 * i + 1], 0.f),
                                                 min_nan(f[2 * i + 5], 0.f));
            }
        }
        __syncthreads();
        // the head that this lane is left with, and whether there is one
        int left = 0;
#pragma unroll
        for (int o = 1, half = kHeads / 2; half > 0; o <<= 1, half >>= 1) left += lane & o ? half : 0;
        const bool is_head = h0 + left < A.group;

        const uint4 none = make_uint4(0, 0, 0, 0);
        const int stride = kWarps * kStep;
        int j = part * per + warp * kStep + sub;                       // this lane's first block of the step; the others kGroups apart
        auto page_at = [&](int i) { return i < end ? table[i] : 0; };
        auto fetch = [&](int i, int page, uint4& l, uint4& h) {        // a block's bounds, zeros where there are none
            l = h = none;
            if (i < end && page >= 0 && page < P.pages && on) {
                const uint16_t* from = A.bounds + page * A.stride + (int64_t)head * 2 * hd + dim;
                l = __ldg(reinterpret_cast<const uint4*>(from));
                h = __ldg(reinterpret_cast<const uint4*>(from + hd));
            }
        };
        // bounds one step ahead, page numbers two
        int page[kEach], next_page[kEach];
        uint4 lo[kEach], hi[kEach];
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            page[x] = page_at(j + x * kGroups);
            next_page[x] = page_at(j + stride + x * kGroups);
        }
#pragma unroll
        for (int x = 0; x < kEach; ++x) fetch(j + x * kGroups, page[x], lo[x], hi[x]);
        for (; __any_sync(kAll, j < end); j += stride) {
            uint64_t l[kEach][4], h[kEach][4];
            int now[kEach];
#pragma unroll
            for (int x = 0; x < kEach; ++x) {
                const uint32_t lw[4] = {lo[x].x, lo[x].y, lo[x].z, lo[x].w}, hw[4] = {hi[x].x, hi[x].y, hi[x].z, hi[x].w};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 a = unpack2<T>(lw[i]), c = unpack2<T>(lw[i + 2]);
                    l[x][2 * i] = pair(a.x, c.x);
                    l[x][2 * i + 1] = pair(a.y, c.y);
                    const float2 d = unpack2<T>(hw[i]), e = unpack2<T>(hw[i + 2]);
                    h[x][2 * i] = pair(d.x, e.x);
                    h[x][2 * i + 1] = pair(d.y, e.y);
                }
                now[x] = page[x];
                page[x] = next_page[x];
                next_page[x] = page_at(j + 2 * stride + x * kGroups);
                fetch(j + stride + x * kGroups, page[x], lo[x], hi[x]);
            }
            float v[kEach][kHeads];
#pragma unroll
            for (int e = 0; e < kHeads; ++e) {
                uint64_t up[4], down[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 a = split[e][i][mine], c = split[e][2 + i][mine];
                    up[2 * i] = pair(a.x, a.y);
                    up[2 * i + 1] = pair(a.z, a.w);
                    down[2 * i] = pair(c.x, c.y);
                    down[2 * i + 1] = pair(c.z, c.w);
                }
#pragma unroll
                for (int x = 0; x < kEach; ++x) {
                    uint64_t t[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) t[i] = fma_pair(up[i], h[x][i], mul_pair(down[i], l[x][i]));
                    v[x][e] = add_halves(add_pair(add_pair(t[0], t[1]), add_pair(t[2], t[3])));
                }
            }
#pragma unroll
            for (int x = 0; x < kEach; ++x) {
                // each step joins two lanes' sums; while a lane holds several heads it passes on half of them
                int held = kHeads;
#pragma unroll
                for (int o = 1; o < kLanes; o <<= 1) {
                    if (held > 1) {
                        held /= 2;
#pragma unroll
                        for (int e = 0; e < kHeads / 2; ++e)
                            if (e < held) {
                                const float give = lane & o ? v[x][e] : v[x][e + held], keep = lane & o ? v[x][e + held] : v[x][e];
                                v[x][e] = keep + __shfl_xor_sync(kAll, give, o);
                            }
                    } else {
                        v[x][0] += __shfl_xor_sync(kAll, v[x][0], o);
                    }
                }
                float score = is_head ? v[x][0] : -INFINITY;
#pragma unroll
                for (int o = 1; o < kHeads; o <<= 1) score = max_nan(score, __shfl_xor_sync(kAll, score, o));
                const int i = j + x * kGroups;
                if (mine == 0 && i < end) {
                    const bool good = now[x] >= 0 && now[x] < P.pages;
                    if (!good) atomicOr(&g_sparse_error, kBadPage);
                    const uint32_t key = good ? key_of(score) : 0u;
                    keys[i] = h0 ? max(keys[i], key) : key;
                }
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        // releases the CTA's keys (complete at the barrier above), acquires the others'
        unsigned done;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(done) : "l"(A.counters + unit) : "memory");
        last = done == (unsigned)A.parts - 1;
        if (last) A.counters[unit] = 0u;
    }
    __syncthreads();
    if (last) choose(A, keys, n, out);
}

template <bool kIsBf16, int kLanes>
int launch_select_h(const SelectArgs& A, unsigned grid, cudaStream_t st) {
    auto go = [&](auto kern) { return launch(kern, dim3(grid), dim3(kThreads), 0, st, "epq_paged_select", A); };
    if (A.group == 1) return go(select_kernel<kIsBf16, kLanes, 1>);
    if (A.group == 2) return go(select_kernel<kIsBf16, kLanes, 2>);
    if (A.group <= 4) return go(select_kernel<kIsBf16, kLanes, 4>);
    return go(select_kernel<kIsBf16, kLanes, 8>);
}
template <bool kIsBf16> int launch_select(const SelectArgs& A, unsigned grid, cudaStream_t st) {
    const int hd = A.pages.head_dim;
    if (hd <= 64) return launch_select_h<kIsBf16, 8>(A, grid, st);
    if (hd <= 128) return launch_select_h<kIsBf16, 16>(A, grid, st);
    return launch_select_h<kIsBf16, 32>(A, grid, st);
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
    return (int64_t)kMaxUnits * 4 + batch * P.kv_heads * P.max_pages * 4;
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
    // CTAs a unit: enough to fill the card twice (lengths differ), each with at least two steps of its warps
    const int64_t units = batch * P.kv_heads, fill = cdiv(4LL * device_sms(), units), most = cdiv(P.max_pages, 64);
    A.parts = (int)(fill < most ? fill : most);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)(units * A.parts);
    return bounds_dtype == EPQ_BF16 ? launch_select<true>(A, grid, st) : launch_select<false>(A, grid, st);
}

}  // extern "C"
