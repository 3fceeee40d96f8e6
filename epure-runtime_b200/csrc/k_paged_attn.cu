// Attention of one new token a sequence over a paged cache (epq_paged_attend):
//   out[b, h] = sum_t softmax_t(scale q[b, h] . K[t]) V[t],  t in [max(0, n - window), n).
//
// Bound: HBM.  Every cached key and value is read once: 2 flops a value and query head,
// 8 flops a byte at 8 heads a key head in bf16, far below what the tensor cores need.
// The work is to keep enough loads in flight on every SM, whatever the lengths are.
//
// Split.  A unit is (sequence, key head, up to 8 or 16 of its query heads); its tokens
// are cut into blocks of 16.  The blocks of all units, in order, are dealt out to the
// CTAs in equal runs, so ragged lengths load every SM alike; a unit that a run's ends
// cut is joined from (maximum, sum, accumulator) records by the last of its CTAs to
// finish, in the order of the CTAs, which keeps results independent of timing.  Within
// a CTA warp w takes the blocks w, w + 4, ... of the run; each warp has its own ring of
// shared-memory stages filled by 16-byte asynchronous copies that run ahead over unit
// boundaries.
//
// Mathematics of a block: S^T = K Q^T as m16n8k16 products with the 16 tokens as rows
// and the query heads as the 8 columns, so a group of up to 8 heads fills the tile (with
// heads as rows half of it or more would be padding); O^T = V^T P^T likewise, with the
// head's dims as rows.  At one column of 8 heads tcgen05's 128-row tiles would be
// 15/16 padding, and the tensor pipe is not what limits this kernel.  The running
// maximum moves only when a score passes it by 2^8; sums are float32.
//
// 8-bit caches: codes are converted to f16 (exact: int8 and e4m3 fit its 11 bits); a
// head's q is brought to f16 by a power of two (exact but for values below 2^-38 of the
// largest); the key's scale multiplies the score, and the value's scale enters the
// weight as 2^(s + log2 scale - M) with a running maximum M of its own, so that neither
// large nor small scales leave f16's range.
#include "epq_paged.cuh"

namespace epq {
namespace paged {
namespace {

__device__ int g_attend_error = 0;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kBlock = 16;                 // tokens of a warp's block
constexpr int kMinBlocks = 4;              // a CTA's run is at least this long
constexpr int kMaxUnits = 65536;           // counters in the workspace
constexpr float kSlack = 8.f;              // how far (log2) a score may pass the running maximum
constexpr float kLog2e = 1.4426950408889634f;

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
    int batch, heads, group, chunks, dtype;
    float scale_log2;
};

// Element kinds of the cache: what the tensor cores multiply.
enum Kind { kBf16 = 0, kF16 = 1, kInt8 = 2, kFp8 = 3 };

template <int kKind> constexpr int kind_bytes() { return kKind <= kF16 ? 2 : 1; }

// ---------------------------------------------------------------- PTX
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
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
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool kIsBf16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (kIsBf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <bool kIsBf16> __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    if (kIsBf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Two f16 values from the 8-bit codes that `sel` picks from x (bytes of an int8 pair
// come with 0x64 above them: 1024 + (code ^ 0x80), so 1152 is taken off).
template <int kKind, uint32_t kSel> __device__ __forceinline__ uint32_t codes_f16(uint32_t x) {
    if (kKind == kInt8) {
        const uint32_t u = __byte_perm(x, 0x64646464u, kSel);
        const uint32_t off = 0x64806480u;
        const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&off));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    constexpr uint32_t kPair = (kSel & 0xf) | (kSel >> 4 & 0xf0);   // the two codes' bytes side by side
    const uint32_t two = __byte_perm(x, 0u, kPair);
    uint32_t r;
    asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(r) : "r"(two));
    return r;
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
    int lo, lo16, n, blocks;   // tokens [lo, n) in blocks from lo16 on
};

__device__ __forceinline__ Span span_of(const AttendArgs& A, int b, bool report) {
    const int64_t cap = (int64_t)A.pages.max_pages * A.pages.page_size;
    int64_t n = A.lengths[b];
    bool bad = n < 0 || n > cap;
    if (A.seq && (A.seq[b] < 0 || A.seq[b] >= A.pages.seqs)) bad = n != 0 || bad;
    if (bad) {
        if (report) atomicOr(&g_attend_error, kBadPosition);
        n = 0;
    }
    Span s;
    s.n = (int)n;
    s.lo = A.window > 0 && n > A.window ? (int)(n - A.window) : 0;
    s.lo16 = s.lo & ~(kBlock - 1);
    s.blocks = (s.n - s.lo16 + kBlock - 1) / kBlock;
    return s;
}

// A place in the dealt-out order: block i of unit u of sequence b.
struct Cursor {
    int b, u, i, units;
    Span s;
    __device__ __forceinline__ void next_sequence(const AttendArgs& A) {
        do {
            ++b;
            s = span_of(A, b, false);
        } while (s.blocks == 0);
        u = 0;
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
    static constexpr int kRows = kBlock * kPitch;                        // one of K, V
    static constexpr int kScales = kBytes == 1 ? 2 * kBlock * 4 : 0;
    static constexpr int kStage = 2 * kRows + kScales;
    static constexpr int kBudget = kDim == 256 && kBytes == 2 ? 48 * 1024 : 24 * 1024;   // a warp's ring
    static constexpr int kFit = kBudget / kStage;
    static constexpr int kStages = kFit > 6 ? 6 : kFit;
    static constexpr int kRing = kStages * kStage;
    static constexpr int kMergePitch = kDim + 4;                         // floats; spreads a column's heads over the banks
    static constexpr int kMerge = kWarps * 8 * kMergePitch * 4;
    static constexpr int kSmem = kWarps * kRing + kMerge;
    static constexpr int kCtas = kDim == 256 && kBytes == 2 ? 1 : 2;     // an SM
    static constexpr int kRecord = kCols * 8 * kMergePitch;              // floats: accumulators, then m, M, l in the padding
    static_assert(kStages >= 2, "ring");
};

template <int kKind, int kDim, int kCols>
__global__ void __launch_bounds__(kThreads, Shape<kKind, kDim, kCols>::kCtas) attend_kernel(const AttendArgs A) {
    using S = Shape<kKind, kDim, kCols>;
    constexpr bool kQuant = kKind >= kInt8;
    constexpr bool kIsBf16 = kKind == kBf16;
    constexpr unsigned kAll = 0xffffffffu;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float wm[kWarps][8 * kCols], wM[kWarps][8 * kCols], wl[kWarps][8 * kCols];
    __shared__ uint32_t seen[kWarps][S::kStages];     // bit r: row r of the stage is a token of the span
    __shared__ int64_t sums[kWarps];
    __shared__ int start_b;
    __shared__ int64_t start_at;
    __shared__ bool last;
    pdl_enter();

    const PagesD& P = A.pages;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hd = P.head_dim, KV = P.kv_heads, units = KV * A.chunks;
    const int hd_chunks = hd * S::kBytes / 16;

    // ---- this CTA's run of blocks [f0, f1)
    const int per = (A.batch + kThreads - 1) / kThreads;
    const int b0 = min(A.batch, tid * per), b1 = min(A.batch, b0 + per);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += span_of(A, b, blockIdx.x == 0).blocks;
    int64_t before = mine;                             // inclusive scan over the threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(kAll, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sums[w];
        total += sums[w];
    }
    before -= mine;
    total *= units;
    int64_t run = (total + gridDim.x - 1) / gridDim.x;
    if (run < kMinBlocks) run = kMinBlocks;
    const int64_t f0 = min(total, blockIdx.x * run), f1 = min(total, f0 + run);
    if (f0 < f1 && f0 >= before * units && f0 < (before + mine) * units) {
        int64_t at = f0 - before * units;
        int b = b0;
        for (;;) {
            const int64_t here = (int64_t)span_of(A, b, false).blocks * units;
            if (at < here) break;
            at -= here;
            ++b;
        }
        start_b = b;
        start_at = at;
    }
    // sequences without a token
    for (int b = blockIdx.x; b < A.batch; b += gridDim.x) {
        if (span_of(A, b, false).blocks) continue;
        for (int e = tid; e < A.heads * hd; e += kThreads)
            static_cast<uint16_t*>(A.out)[(int64_t)b * A.heads * hd + e] = 0;
        if (A.lse)
            for (int h = tid; h < A.heads; h += kThreads) A.lse[(int64_t)b * A.heads + h] = -INFINITY;
    }
    uint8_t* ring = smem + warp * S::kRing;
    const uint32_t ring_at = smem_u32(ring);
    if (hd < kDim)                                     // chunks past the head's end stay zero
        for (int e = lane; e < S::kRing / 16; e += 32) reinterpret_cast<uint4*>(ring)[e] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (f0 >= f1) return;

    Cursor unit;                                       // of the unit that the CTA is at
    unit.units = units;
    unit.b = start_b;
    unit.s = span_of(A, start_b, false);
    unit.u = (int)(start_at / unit.s.blocks);
    unit.i = (int)(start_at - (int64_t)unit.u * unit.s.blocks);

    // ---- loads, kStages - 1 blocks ahead
    Cursor ahead = unit;
    int64_t f_load = f0 + warp;
    int next_page = 0;                                 // table entry of row `lane & 15` of the next block to load
    bool next_on = false;                              // whether that row is a token (the entry may still be on its way)
    auto look_up = [&]() {
        const int t = ahead.s.lo16 + ahead.i * kBlock + (lane & 15);
        next_on = t >= ahead.s.lo && t < ahead.s.n;
        if (next_on) {
            const int s = A.seq ? A.seq[ahead.b] : ahead.b;
            next_page = P.table[(int64_t)s * P.table_stride + t / P.page_size];
        }
    };
    if (f_load < f1) {
        ahead.advance(A, warp);
        look_up();
    }
    int load_stage = 0;
    auto load = [&]() {
        if (f_load < f1) {
            const int t = ahead.s.lo16 + ahead.i * kBlock + (lane & 15);
            const int head = ahead.u / A.chunks;
            if (next_on && (next_page < 0 || next_page >= P.pages)) {
                atomicOr(&g_attend_error, kBadPage);
                next_on = false;
            }
            const int slot = t - t / P.page_size * P.page_size;
            const int64_t slot_at = (int64_t)head * P.page_size + slot;
            const int64_t at = next_on ? next_page * P.page_stride + slot_at * hd : -1;
            const uint32_t k_at = ring_at + load_stage * S::kStage, v_at = k_at + S::kRows;
            const uint32_t mask = __ballot_sync(kAll, next_on) & 0xffffu;
            if (lane == 0) seen[warp][load_stage] = mask;
            constexpr int kChunks = S::kPitch / 16;
#pragma unroll
            for (int e = 0; e < kBlock * kChunks / 32; ++e) {
                const int idx = e * 32 + lane, row = idx / kChunks, ch = idx % kChunks;
                const int64_t from = __shfl_sync(kAll, at, row);
                if (ch < hd_chunks) {
                    const int64_t off = from < 0 ? 0 : (from * S::kBytes + ch * 16);
                    const int bytes = from < 0 ? 0 : 16;
                    cp16(k_at + swizzled<S::kPitch>(row, ch), P.k + off, bytes);
                    cp16(v_at + swizzled<S::kPitch>(row, ch), P.v + off, bytes);
                }
            }
            if (kQuant) {                              // lanes 0-15: key scales, 16-31: value scales
                const float* sc = lane < 16 ? P.k_scale : P.v_scale;
                const int64_t off = next_on ? next_page * P.scale_stride + slot_at : 0;
                cp4(v_at + S::kRows + lane * 4, sc + off, next_on ? 4 : 0);
            }
            f_load += kWarps;
            if (f_load < f1) {
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
    const int g = lane >> 2, c = lane & 3;             // row and column pair of the tensor fragments
    int64_t f = f0 + warp;
    int stage = 0;
    for (int64_t at = f0; at < f1;) {
        const int64_t unit_start = at - unit.i, unit_end = unit_start + unit.s.blocks;
        const int64_t end = min(f1, unit_end);
        const int head = unit.u / A.chunks, chunk = unit.u - head * A.chunks;
        const int h_first = head * A.group + chunk * 8 * kCols;               // query heads of this unit
        const int h_count = min(8 * kCols, A.group - chunk * 8 * kCols);

        // q as B fragments: column g is head h_first + 8 n + g
        uint32_t qf[kCols][kDim / 16][2];
        float q_gain[kCols][2];                        // what scores of heads 2c, 2c + 1 are multiplied by
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
            const bool on = 8 * n + g < h_count;
            const uint16_t* q = static_cast<const uint16_t*>(A.q) + unit.b * A.q_row + (h_first + 8 * n + g) * A.q_head;
#pragma unroll
            for (int k = 0; k < kDim / 16; ++k) {
                // 16-bit caches: dims 2c, 2c+1 and 2c+8, 2c+9; 8-bit ones: 4c .. 4c+3
                const int d0 = 16 * k + (kQuant ? 4 * c : 2 * c), d1 = d0 + (kQuant ? 2 : 8);
                const bool there = on && 16 * k < hd;
                qf[n][k][0] = there ? *reinterpret_cast<const uint32_t*>(q + d0) : 0u;
                qf[n][k][1] = there ? *reinterpret_cast<const uint32_t*>(q + d1) : 0u;
            }
            q_gain[n][0] = q_gain[n][1] = A.scale_log2;
            if (kQuant) {                              // to f16, times a power of two
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
                m[n][r] = M[n][r] = -INFINITY;
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
            const uint32_t k_at = ring_at + stage * S::kStage, v_at = k_at + S::kRows;
            const uint32_t mask = seen[warp][stage];

            // scores
            float sc[kCols][4];
#pragma unroll
            for (int n = 0; n < kCols; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[n][r] = 0.f;
            if (!kQuant) {
#pragma unroll
                for (int k = 0; k < kDim / 16; ++k) {
                    if (16 * k < hd) {
                        uint32_t a[4];
                        ldsm(a, k_at + swizzled<S::kPitch>(lane & 15, 2 * k + (lane >> 4)));
#pragma unroll
                        for (int n = 0; n < kCols; ++n) mma<kIsBf16>(sc[n], a, qf[n][k][0], qf[n][k][1]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < kDim / 32; ++k) {
                    if (32 * k < hd) {
                        uint32_t x[4];
                        ldsm(x, k_at + swizzled<S::kPitch>((lane >> 3 & 1) * 8 + (lane & 7), 2 * k + (lane >> 4)));
                        if (kKind == kInt8) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) x[r] ^= 0x80808080u;
                        }
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const uint32_t a[4] = {codes_f16<kKind, 0x4140>(x[2 * r]), codes_f16<kKind, 0x4140>(x[2 * r + 1]),
                                                   codes_f16<kKind, 0x4342>(x[2 * r]), codes_f16<kKind, 0x4342>(x[2 * r + 1])};
#pragma unroll
                            for (int n = 0; n < kCols; ++n)
                                mma<false>(sc[n], a, qf[n][2 * k + r][0], qf[n][2 * k + r][1]);
                        }
                    }
                }
            }
            float ks[2] = {1.f, 1.f}, lv[2] = {0.f, 0.f};
            if (kQuant) {
                const float* scales = reinterpret_cast<const float*>(ring + stage * S::kStage + 2 * S::kRows);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    ks[r] = scales[g + 8 * r];
                    lv[r] = __log2f(scales[16 + g + 8 * r]);
                }
            }
            // weights
            bool rise = false;
#pragma unroll
            for (int n = 0; n < kCols; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {          // r: token g + 8 (r >> 1), head 2c + (r & 1)
                    const bool on = mask >> (g + 8 * (r >> 1)) & 1;
                    sc[n][r] = on ? sc[n][r] * (kQuant ? q_gain[n][r & 1] * ks[r >> 1] : q_gain[n][r & 1]) : -INFINITY;
                    rise |= sc[n][r] > m[n][r & 1] + kSlack;
                    if (kQuant) rise |= sc[n][r] + lv[r >> 1] > M[n][r & 1] + kSlack;
                }
            if (__any_sync(kAll, rise)) {
#pragma unroll
                for (int n = 0; n < kCols; ++n) {
                    float turn_acc[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        // fmaxf passes over NaN, which then reaches the sums through the weights
                        float top = fmaxf(sc[n][r], sc[n][r + 2]);
                        float topM = kQuant ? fmaxf(sc[n][r] + lv[0], sc[n][r + 2] + lv[1]) : 0.f;
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
            uint32_t pf[kCols][2];
#pragma unroll
            for (int n = 0; n < kCols; ++n) {
                float w[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = sc[n][r] == -INFINITY ? 0.f : ex2(sc[n][r] - m[n][r & 1]);
                    l[n][r & 1] += p;
                    w[r] = p;
                    if (kQuant) {
                        const float x = sc[n][r] + lv[r >> 1];
                        w[r] = x == -INFINITY ? 0.f : ex2(x - M[n][r & 1]);
                    }
                }
                pf[n][0] = transpose8x8(pack<kIsBf16>(w[0], w[1]));
                pf[n][1] = transpose8x8(pack<kIsBf16>(w[2], w[3]));
            }
            // O^T += V^T P^T
            if (!kQuant) {
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
                    if (16 * d < hd) {
                        uint32_t a[4];
                        ldsm_t(a, v_at + swizzled<S::kPitch>((lane >> 4) * 8 + (lane & 7), 2 * d + (lane >> 3 & 1)));
#pragma unroll
                        for (int n = 0; n < kCols; ++n) mma<kIsBf16>(acc[n][d], a, pf[n][0], pf[n][1]);
                    }
                }
            } else {
#pragma unroll
                for (int d = 0; d < kDim / 32; ++d) {
                    if (32 * d < hd) {
                        uint32_t x[4];
                        ldsm_t(x, v_at + swizzled<S::kPitch>((lane >> 3 & 1) * 8 + (lane & 7), 2 * d + (lane >> 4)));
                        if (kKind == kInt8) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) x[r] ^= 0x80808080u;
                        }
#pragma unroll
                        for (int r = 0; r < 2; ++r) {  // rows 0-7: the even dims of 16, rows 8-15: the odd ones
                            const uint32_t a[4] = {codes_f16<kKind, 0x4240>(x[2 * r]), codes_f16<kKind, 0x4341>(x[2 * r]),
                                                   codes_f16<kKind, 0x4240>(x[2 * r + 1]), codes_f16<kKind, 0x4341>(x[2 * r + 1])};
#pragma unroll
                            for (int n = 0; n < kCols; ++n) mma<false>(acc[n][2 * d + r], a, pf[n][0], pf[n][1]);
                        }
                    }
                }
            }
            if (++stage == S::kStages) stage = 0;
        }

        // ---- the unit's piece: the four warps' states to one
        float* const merge = reinterpret_cast<float*>(smem + kWarps * S::kRing);
        const bool whole = at == unit_start && end == unit_end;
        float* const record = A.records + ((int64_t)blockIdx.x * 2 + (unit_start < f0 ? 0 : 1)) * S::kRecord;
        const int unit_index = unit.b * units + unit.u;

        // m, M and l of a warp to shared memory (l summed over the lanes of a column)
        auto put_sums = [&](const float (&m_)[kCols][2], const float (&M_)[kCols][2], const float (&l_)[kCols][2]) {
#pragma unroll
            for (int n = 0; n < kCols; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float s = l_[n][r];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) s += __shfl_xor_sync(kAll, s, o);
                    if (lane < 4) {
                        wm[warp][8 * n + 2 * c + r] = m_[n][r];
                        wM[warp][8 * n + 2 * c + r] = kQuant ? M_[n][r] : m_[n][r];
                        wl[warp][8 * n + 2 * c + r] = s;
                    }
                }
        };
        // Joins the warps' states of column n and hands (head in unit, dim, value, m, M, l) on.
        auto join = [&](int n, bool final) {
            for (int e = tid; e < 8 * hd; e += kThreads) {
                const int j = e / hd, d = e - j * hd, h = 8 * n + j;
                if (h >= h_count) break;
                float mx = -INFINITY, Mx = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    mx = fmaxf(mx, wm[w][h]);
                    Mx = fmaxf(Mx, wM[w][h]);
                }
                float sum = 0.f, val = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    // a warp that saw nothing has l = 0 and zeros; NaN must pass through
                    sum += wm[w][h] == -INFINITY ? wl[w][h] : wl[w][h] * ex2(wm[w][h] - mx);
                    const float a = merge[(w * 8 + j) * S::kMergePitch + d];
                    val += wM[w][h] == -INFINITY ? a : a * ex2(wM[w][h] - Mx);
                }
                if (final) {
                    // l = 0: every score was -inf.  2^(M - m) is 1 for 16-bit caches.
                    float o = sum == 0.f ? 0.f : val / sum;
                    if (kQuant && Mx != -INFINITY) o *= ex2(Mx - mx);
                    const int64_t to = ((int64_t)unit.b * A.heads + h_first + h) * hd + d;
                    if (A.dtype == EPQ_BF16) static_cast<__nv_bfloat16*>(A.out)[to] = __float2bfloat16_rn(o);
                    else static_cast<__half*>(A.out)[to] = __float2half_rn(o);
                    if (A.lse && d == 0)
                        A.lse[(int64_t)unit.b * A.heads + h_first + h] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) / kLog2e;
                } else {
                    float* rec = record + (int64_t)h * S::kMergePitch;
                    rec[d] = val;
                    if (d == 0) {
                        rec[kDim] = mx;
                        rec[kDim + 1] = Mx;
                        rec[kDim + 2] = sum;
                    }
                }
            }
        };
        put_sums(m, M, l);
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
            if (8 * n < h_count) {
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int dim = 16 * d + (kQuant ? 2 * g + (r >> 1) : g + 8 * (r >> 1));
                        merge[(warp * 8 + 2 * c + (r & 1)) * S::kMergePitch + dim] = acc[n][d][r];
                    }
                __syncthreads();
                join(n, whole);
                __syncthreads();
            }
        }

        // ---- a unit cut over several CTAs: the last of them joins the records
        if (!whole) {
            __threadfence();
            __syncthreads();
            const int first = (int)(unit_start / run), pieces = (int)((unit_end - 1) / run) - first + 1;
            if (tid == 0) last = atomicAdd(&A.counters[unit_index], 1u) == (unsigned)pieces - 1;
            __syncthreads();
            if (last) {
                __threadfence();
                auto record_of = [&](int p) {
                    return A.records + ((int64_t)(first + p) * 2 + (unit_start < (first + p) * run ? 0 : 1)) * S::kRecord;
                };
                constexpr int kPer = kDim / 32;        // dims a lane
#pragma unroll
                for (int n = 0; n < kCols; ++n) {
                    if (8 * n < h_count) {
                        for (int j = 0; j < 8 && 8 * n + j < h_count; ++j) {
                            const int64_t off = (int64_t)(8 * n + j) * S::kMergePitch;
                            float mx = -INFINITY, Mx = -INFINITY;
                            for (int p = warp + kWarps * lane; p < pieces; p += kWarps * 32) {
                                const float* rec = record_of(p) + off;
                                mx = fmaxf(mx, __ldcg(rec + kDim));
                                Mx = fmaxf(Mx, __ldcg(rec + kDim + 1));
                            }
#pragma unroll
                            for (int o = 16; o > 0; o >>= 1) {
                                mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, o));
                                Mx = fmaxf(Mx, __shfl_xor_sync(kAll, Mx, o));
                            }
                            float sum = 0.f, val[kPer];
#pragma unroll
                            for (int i = 0; i < kPer; ++i) val[i] = 0.f;
#pragma unroll 4
                            for (int p = warp; p < pieces; p += kWarps) {
                                const float* rec = record_of(p) + off;
                                const float pm = __ldcg(rec + kDim), pM = __ldcg(rec + kDim + 1);
                                const float fl = pm == -INFINITY ? 1.f : ex2(pm - mx);
                                const float fa = pM == -INFINITY ? 1.f : ex2(pM - Mx);
                                sum += __ldcg(rec + kDim + 2) * fl;
#pragma unroll
                                for (int i = 0; i < kPer; ++i)
                                    if (i * 32 + lane < hd) val[i] += __ldcg(rec + i * 32 + lane) * fa;
                            }
#pragma unroll
                            for (int i = 0; i < kPer; ++i)
                                merge[(warp * 8 + j) * S::kMergePitch + i * 32 + lane] = val[i];
                            if (lane == 0) {
                                wm[warp][8 * n + j] = mx;
                                wM[warp][8 * n + j] = Mx;
                                wl[warp][8 * n + j] = sum;
                            }
                        }
                        __syncthreads();
                        join(n, true);
                        __syncthreads();
                    }
                }
                if (tid == 0) A.counters[unit_index] = 0u;
            }
        }
        at = end;
        if (at < f1) unit.advance(A, unit.s.blocks - unit.i);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int kKind, int kDim, int kCols>
int launch_attend(const AttendArgs& A, cudaStream_t st) {
    using S = Shape<kKind, kDim, kCols>;
    return launch(attend_kernel<kKind, kDim, kCols>, dim3((unsigned)(device_sms() * S::kCtas)), dim3(kThreads),
                  (size_t)S::kSmem, st, "epq_paged_attend", A);
}
template <int kKind, int kDim>
int launch_attend_d(const AttendArgs& A, int cols, cudaStream_t st) {
    return cols == 1 ? launch_attend<kKind, kDim, 1>(A, st) : launch_attend<kKind, kDim, 2>(A, st);
}
template <int kKind>
int launch_attend_k(const AttendArgs& A, int cols, cudaStream_t st) {
    const int hd = A.pages.head_dim;
    if (hd <= 64) return launch_attend_d<kKind, 64>(A, cols, st);
    if (hd <= 128) return launch_attend_d<kKind, 128>(A, cols, st);
    return launch_attend_d<kKind, 256>(A, cols, st);
}

// Columns of 8 query heads a unit has: one, or two for groups above 8.
int cols_of(int group) { return group <= 8 ? 1 : 2; }

int64_t records_bytes(int hd, int group) {
    const int dim = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    return (int64_t)device_sms() * 2 * 2 * cols_of(group) * 8 * (dim + 4) * 4;
}

}  // namespace

int attend_read_device_error(int* flag) {
    if (cudaMemcpyFromSymbol(flag, g_attend_error, sizeof(int)) != cudaSuccess)
        return check_launch("read paged attention error flag");
    return EPQ_OK;
}

}  // namespace paged
}  // namespace epq

using namespace epq;
using namespace epq::paged;

extern "C" {

int64_t epq_paged_attend_workspace_bytes(const epq_pages* pages, int64_t batch, int32_t heads) {
    PagesD P;
    const int rc = make_pages(pages, &P, "epq_paged_attend_workspace_bytes");
    if (rc != EPQ_OK) return rc;
    if (batch < 0 || heads <= 0 || heads % P.kv_heads)
        return set_error(EPQ_ESHAPE, "epq_paged_attend_workspace_bytes: %d query heads over %d key heads", heads,
                         P.kv_heads);
    return (int64_t)kMaxUnits * 4 + records_bytes(P.head_dim, heads / P.kv_heads);
}

int epq_paged_attend(const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                     int64_t batch, float scale, int64_t window, void* out, float* lse, int32_t dtype,
                     void* workspace, int64_t workspace_bytes, void* stream) {
    AttendArgs A = {};
    const int rc = make_pages(pages, &A.pages, "epq_paged_attend");
    if (rc != EPQ_OK) return rc;
    const int KV = A.pages.kv_heads;
    if (!q || batch < 0 || window < 0) return set_error(EPQ_EINVAL, "epq_paged_attend: bad arguments");
    if (dtype != EPQ_BF16 && dtype != EPQ_F16)
        return set_error(EPQ_EDTYPE, "epq_paged_attend: dtype %d (f16 or bf16)", dtype);
    if (q->heads <= 0 || q->heads % KV)
        return set_error(EPQ_ESHAPE, "epq_paged_attend: %d query heads over %d key heads", q->heads, KV);
    A.group = q->heads / KV;
    const int cols = cols_of(A.group);
    A.chunks = (A.group + 8 * cols - 1) / (8 * cols);
    if (batch * KV * A.chunks > kMaxUnits)
        return set_error(EPQ_EUNSUPPORTED, "epq_paged_attend: batch=%lld of %d key heads (at most %d units)",
                         (long long)batch, KV, kMaxUnits);
    if (!seq && batch > A.pages.seqs)
        return set_error(EPQ_ESHAPE, "epq_paged_attend: batch=%lld of a table of %d sequences", (long long)batch,
                         A.pages.seqs);
    if (batch == 0) return EPQ_OK;
    if (!q->data || !lengths || !out) return set_error(EPQ_EINVAL, "epq_paged_attend: NULL q, lengths or out");
    if (!heads_aligned(*q, 2, 4))
        return set_error(EPQ_EALIGN, "epq_paged_attend: q must be 4-byte aligned with even strides");
    const int64_t need = epq_paged_attend_workspace_bytes(pages, batch, q->heads);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
        return set_error(EPQ_EWORKSPACE, "epq_paged_attend: workspace of %lld bytes (need %lld, 256-aligned)",
                         (long long)workspace_bytes, (long long)need);
    A.q = q->data;
    A.q_row = q->stride_row;
    A.q_head = q->stride_head;
    A.seq = seq;
    A.lengths = lengths;
    A.out = out;
    A.lse = lse;
    A.counters = static_cast<unsigned*>(workspace);
    A.records = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (int64_t)kMaxUnits * 4);
    A.window = window;
    A.batch = (int)batch;
    A.heads = q->heads;
    A.dtype = dtype;
    A.scale_log2 = scale * kLog2e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (A.pages.format) {
        case EPQ_CACHE_INT8: return launch_attend_k<kInt8>(A, cols, st);
        case EPQ_CACHE_FP8: return launch_attend_k<kFp8>(A, cols, st);
        default:
            return dtype == EPQ_BF16 ? launch_attend_k<kBf16>(A, cols, st) : launch_attend_k<kF16>(A, cols, st);
    }
}

}  // extern "C"
