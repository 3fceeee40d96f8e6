// The paged key-value cache: rows written with the norm, the rotation and the 8-bit
// quantisation of the step fused in (epq_paged_write), and read back (epq_paged_read).
//
//   a = max|x| over a head's row, scale = a * (1 / top), code = round(x * (top / a)),
//   top = 127 (int8, rounded to even) or 448 (e4m3); read: code * scale.
//
// Bound: HBM.  A row is read once in its own type and written once in the cache's; the
// arithmetic (one division a row, about ten operations a value) stays below that.
//
// Split: one warp takes (a share of) one token's rows -- q heads, k heads, v heads --
// with 8 values a lane, so a row is 8, 16 or 32 lanes, its maximum and sum of squares a
// few shuffles, and the token's page, cos and sin are found once.  16-bit rows stay
// packed two values a word for loads, shuffles and the maximum, and products go two an
// instruction: at 110 instructions a row of 128 the kernel is as near to its issue rate
// as to HBM's.
//
// Measured (B200): 65536 tokens of 32 + 8 + 8 heads of 128, bf16 to int8, rotated and
// written: 258 us (1.48 GB, 5.7 TB/s, 89% of the measured copy rate); read back: 75 us
// (0.41 GB, 5.4 TB/s).  16 tokens: 2.6 us and 2.0 us, the chain position, page, row.
#include "epq_paged.cuh"

namespace epq {
namespace paged {
namespace {

__device__ int g_cache_error = 0;

constexpr int kCacheThreads = 128;

struct Rows {
    const void* p;
    int64_t row, head;   // strides, in elements
};

template <int N> struct Const {
    static constexpr int value = N;
};

// How a lane comes by the values that its own turn with: from the lane that holds them,
// from its own, or from memory (where neither fits).
enum Turn { kNoTurn = 0, kHalfLanes = 1, kNeighbours = 2, kHalfLoads = 3 };

struct WriteArgs {
    PagesD pages;
    Rows q, k, v;
    void* q_out;
    int64_t qo_row, qo_head;
    const int32_t* seq;
    const int64_t* pos;
    const float* cos_t;
    const float* sin_t;
    int64_t m, max_len;
    int heads, r, turn, qk_norm, splits, aligned, out_aligned;
    float eps;
};

template <int kFormat> constexpr float kTop = kFormat == EPQ_CACHE_INT8 ? 127.f : 448.f;    // the largest code

// Eight values times `inv` (= top / max, at most top (1 + 2^-23) in magnitude), as codes.
template <int kFormat>
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float inv, float scale) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) mul2(y[i], y[i + 1], x[i], x[i + 1], inv, inv);
    if (inv == INFINITY) {          // a row whose maximum is so small that top / max overflows is divided instead
#pragma unroll
        for (int i = 0; i < 8; ++i)
            y[i] = scale > 0.f ? fmaxf(-kTop<kFormat>, fminf(kTop<kFormat>, __fdiv_rn(x[i], scale))) : 0.f;
    }
    uint32_t b[8];
    if (kFormat == EPQ_CACHE_INT8) {
        // 1.5 2^23 + y: float32 rounds to the integer (ties to even), which is its low byte
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(__fadd_rn(y[i], 12582912.f));
        return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                          __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            b[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i], y[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
        return make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
    }
}

constexpr int kAtOnce = 2;          // rows of a lane in flight

// What a kernel takes for granted.  kExact: heads fill their lanes and passes, the whole
// head turns (or none of it); kLanesOnly: partners are whole lanes; both: 16-byte loads
// and stores.  kAny: nothing.  (8192 tokens of 32 + 8 + 8 heads of 128 to int8, us: kExact
// 36 in bf16 and 64 in float32; kAny, bf16, interleaved 46, unaligned 58, 50 values turned 84.)
enum Class { kExact = 0, kLanesOnly = 1, kAny = 2 };

// Registers for 7 CTAs (28 warps) an SM: 64k rows of 48 heads took 376 us (with their
// reading back) at the 88 registers that the compiler would use, 340 at 72, 337 at 64.
// At 72 the 16-bit instances spill at most 24 bytes.
template <typename T, int kFormat, int kLanes, int kClass>
__global__ void __launch_bounds__(kCacheThreads, sizeof(T) == 2 && kClass != kAny ? 7 : 1)
    write_kernel(const WriteArgs A) {
    pdl_enter();
    constexpr unsigned kAll = 0xffffffffu;
    constexpr int kFit = 32 / kLanes, kStep = kFit * kAtOnce;      // heads of a warp side by side, and a pass
    const int warp = blockIdx.x * (kCacheThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int64_t row = warp / A.splits;
    if (row >= A.m) return;
    const int split = warp - (int)row * A.splits;
    const PagesD& P = A.pages;
    const int hd = kClass == kExact ? kLanes * 8 : P.head_dim, KV = P.kv_heads;
    const int sub = lane / kLanes, chunk = lane & (kLanes - 1), e0 = chunk * 8;
    const bool in_row = kClass == kExact || e0 < hd;
    const bool aligned = kClass != kAny || A.aligned, out_aligned = kClass != kAny || A.out_aligned;

    // A pass is kStep heads of q, k or v; this warp's are [p0, p1).  A pass's rows are
    // fetched while the one before it (first: the token's place) is worked on.  Lanes past
    // the last head or value fetch what another lane does.
    const int of_q = (A.heads + kStep - 1) / kStep, of_kv = (KV + kStep - 1) / kStep, passes = of_q + 2 * of_kv;
    const int p0 = passes * split / A.splits, p1 = passes * (split + 1) / A.splits;
    Eight<T> next[kAtOnce];
    auto fetch = [&](const Rows& src, int heads, int h0) {
        const T* const from = static_cast<const T*>(src.p) + row * src.row + (in_row ? e0 : 0);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int h = h0 + sub + i * kFit;
            next[i].load(from + (kClass == kExact ? h : min(h, heads - 1)) * src.head, aligned);
        }
    };
    auto fetch_pass = [&](int p) {
        if (p < of_q) fetch(A.q, A.heads, p * kStep);
        else if (p < of_q + of_kv) fetch(A.k, KV, (p - of_q) * kStep);
        else fetch(A.v, KV, (p - of_q - of_kv) * kStep);
    };
    if (p0 < p1) fetch_pass(p0);

    const int64_t pos = A.pos[row];
    const int seq = A.seq[row];
    // cos and the signed sin of this lane's 8 values, y = x c + partner s, on their way with
    // the page's number (of some position of the table, where the row's is outside it)
    float c[8], s[8];
    int partner = lane;                                // kHalfLanes: the lane that holds the other halves
    if (A.turn != kNoTurn) {
        const int half = A.r >> 1;
        const int64_t at_row = (pos < 0 ? 0 : pos < A.max_len ? pos : A.max_len - 1) * half;
        if (kClass != kAny || A.turn == kHalfLanes) {
            const int part = half >> 3;
            const bool second = chunk >= part;
            if (kClass == kExact || e0 < A.r) {
                partner = second ? lane - part : lane + part;
                const int64_t at = at_row + (second ? e0 - half : e0);
                load_v<float, 8>(c, A.cos_t + at);
                load_v<float, 8>(s, A.sin_t + at);
                if (!second) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[i] = -s[i];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = e0 + i;
                if (e < A.r) {
                    const bool second = A.turn == kNeighbours ? e & 1 : e >= half;
                    const int64_t at = at_row + (A.turn == kNeighbours ? e >> 1 : second ? e - half : e);
                    c[i] = A.cos_t[at];
                    s[i] = second ? A.sin_t[at] : -A.sin_t[at];
                }
            }
        }
    }
    int64_t page = 0;
    int slot = 0, bad = 0;
    bool live = pos >= 0;
    if (live) {
        live = find_slot(P, seq, pos, &page, &slot, &bad);
        if (live && A.turn != kNoTurn && pos >= A.max_len) {
            live = false;
            bad = kBadPosition;
        }
        if (bad && lane == 0) atomicOr(&g_cache_error, bad);
    }
    T* const q_to = static_cast<T*>(A.q_out) + row * A.qo_row + e0;
    if (!live) {                                       // a padding row's q is zero
        for (int h = p0 * kStep + sub; h < min(p1 * kStep, A.heads); h += kFit) {
            Eight<T> zero;
            zero.clear();
            if (in_row) zero.store(q_to + h * A.qo_head, out_aligned);
        }
        return;
    }

    const int64_t cached = page * P.page_stride + (int64_t)slot * hd + e0, scaled = page * P.scale_stride + slot;
    const int64_t head_step = (int64_t)P.page_size * hd;

    // Works on the pass's rows x: heads h0 + sub, h0 + sub + kFit, ... of q (kWhich = 0), k (1) or v (2)
    auto work = [&](auto which, int h0, Eight<T> (&x)[kAtOnce]) {
        constexpr int kWhich = decltype(which)::value;
        const int heads = kWhich == 0 ? A.heads : KV;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int h = h0 + sub + i * kFit;
            const bool on = kClass == kExact || (in_row && h < heads);
            if (kClass != kExact && !in_row) x[i].clear();
            if (kWhich < 2) {
                float f[8], gain = 1.f;
                if (A.qk_norm) {                       // RMSNorm of the head, rounded to T
                    x[i].get(f);
                    float ss = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
#pragma unroll
                    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(kAll, ss, o);
                    gain = rsqrtf(ss / (float)hd + A.eps);
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] *= gain;
                    x[i].set(f);
                }
                if (A.turn != kNoTurn) {
                    float other[8];
                    x[i].get(f);
                    if (kClass != kAny || A.turn == kHalfLanes) {
                        x[i].from_lane(partner).get(other);
                        if (kClass == kExact || e0 < A.r) {        // (rotary_dim is a multiple of 16: all 8 or none)
#pragma unroll
                            for (int j = 0; j < 8; j += 2) {
                                mul2(f[j], f[j + 1], f[j], f[j + 1], c[j], c[j + 1]);
                                mul2(other[j], other[j + 1], other[j], other[j + 1], s[j], s[j + 1]);
                            }
#pragma unroll
                            for (int j = 0; j < 8; ++j) f[j] = __fadd_rn(f[j], other[j]);
                            x[i].set(f);
                        }
                    } else {
                        if (A.turn == kNeighbours) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) other[j] = f[j ^ 1];
                        } else {
                            const Rows& src = kWhich == 0 ? A.q : A.k;
                            const T* const from = static_cast<const T*>(src.p) + row * src.row + h * src.head + e0;
                            const int half = A.r >> 1;
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const int e = e0 + j;
                                other[j] = 0.f;
                                if (on && e < A.r) {
                                    other[j] = to_f<T>(from[(e < half ? half : -half) + j]);
                                    if (A.qk_norm) other[j] = to_f<T>(from_f<T>(other[j] * gain));
                                }
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (e0 + j < A.r) f[j] = __fadd_rn(__fmul_rn(f[j], c[j]), __fmul_rn(other[j], s[j]));
                        x[i].set(f);
                    }
                }
            }
            if (kWhich == 0) {
                if (on) x[i].store(q_to + h * A.qo_head, out_aligned);
            } else {
                uint8_t* const pool = kWhich == 1 ? P.k : P.v;
                const int64_t at = cached + h * head_step;
                if (kFormat == EPQ_CACHE_SAME) {
                    if (on) x[i].store(reinterpret_cast<T*>(pool) + at, true);
                } else {
                    const float a = x[i].template largest<kLanes>();
                    // (a row that is not finite reads back as NaN, whatever its codes are)
                    const float scale = a < INFINITY ? __fmul_rn(a, 1.f / kTop<kFormat>) : NAN;
                    const float inv = a > 0.f ? __fdiv_rn(kTop<kFormat>, a) : 0.f;
                    if (on) {
                        float f[8];
                        x[i].get(f);
                        *reinterpret_cast<uint2*>(pool + at) = codes8<kFormat>(f, inv, scale);
                        if (chunk == 0) (kWhich == 1 ? P.k_scale : P.v_scale)[scaled + (int64_t)h * P.page_size] = scale;
                    }
                }
            }
        }
    };
    for (int p = p0; p < p1; ++p) {
        Eight<T> x[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) x[i] = next[i];
        if (p + 1 < p1) fetch_pass(p + 1);
        if (p < of_q) work(Const<0>(), p * kStep, x);
        else if (p < of_q + of_kv) work(Const<1>(), (p - of_q) * kStep, x);
        else work(Const<2>(), (p - of_q - of_kv) * kStep, x);
    }
}

struct ReadArgs {
    PagesD pages;
    const int32_t* seq;
    const int64_t* pos;
    void* k_out;
    void* v_out;
    int64_t m;
    int splits;
};

// 16 values an item: 16 bytes of codes, or two loads of a cache in T.
template <typename T, int kFormat>
__global__ void __launch_bounds__(kCacheThreads) read_kernel(const ReadArgs A) {
    pdl_enter();
    const int warp = blockIdx.x * (kCacheThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int64_t row = warp / A.splits;
    if (row >= A.m) return;
    const int split = warp - (int)row * A.splits;
    const PagesD& P = A.pages;
    const int hd = P.head_dim, KV = P.kv_heads, per_head = hd >> 4, items = 2 * KV * per_head;
    const int64_t pos = A.pos[row];
    int64_t page = 0;
    int slot = 0, bad = 0;
    const bool live = pos >= 0 && find_slot(P, A.seq[row], pos, &page, &slot, &bad);
    if (bad && lane == 0) atomicOr(&g_cache_error, bad);
    for (int it = split * 32 + lane; it < items; it += 32 * A.splits) {
        const int j = it / per_head, e0 = (it - j * per_head) * 16;
        const bool is_v = j >= KV;
        const int head = is_v ? j - KV : j;
        const int64_t slot_at = (int64_t)head * P.page_size + slot, at = page * P.page_stride + slot_at * hd + e0;
        const uint8_t* from = is_v ? P.v : P.k;
        T* to = static_cast<T*>(is_v ? A.v_out : A.k_out) + (row * KV + head) * hd + e0;
        float f[2][8];
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i >> 3][i & 7] = 0.f;
        if (live) {
            if (kFormat == EPQ_CACHE_SAME) {
                load_v<T, 8>(f[0], reinterpret_cast<const T*>(from) + at);
                load_v<T, 8>(f[1], reinterpret_cast<const T*>(from) + at + 8);
            } else {
                const uint4 w = *reinterpret_cast<const uint4*>(from + at);
                const float scale = (is_v ? P.v_scale : P.k_scale)[page * P.scale_stride + slot_at];
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float(&g)[8] = f[i >> 1];
                    const int j = 4 * (i & 1);
                    if (kFormat == EPQ_CACHE_INT8) {
                        // a byte b = code + 128 below 2^23 as bits, less 2^23 + 128
                        const uint32_t v = u[i] ^ 0x80808080u;
                        g[j] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7650)) - 8388736.f;
                        g[j + 1] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7651)) - 8388736.f;
                        g[j + 2] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7652)) - 8388736.f;
                        g[j + 3] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7653)) - 8388736.f;
                    } else {
                        const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u[i] & 0xffffu), __NV_E4M3);
                        const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u[i] >> 16), __NV_E4M3);
                        const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
                        g[j] = a.x, g[j + 1] = a.y, g[j + 2] = b.x, g[j + 3] = b.y;
                    }
                    mul2(g[j], g[j + 1], g[j], g[j + 1], scale, scale);
                    mul2(g[j + 2], g[j + 3], g[j + 2], g[j + 3], scale, scale);
                }
            }
        }
        store_v<T, 8>(to, f[0]);
        store_v<T, 8>(to + 8, f[1]);
    }
}

template <typename T, int kFormat, int kLanes>
int launch_write_l(const WriteArgs& A, unsigned blocks, cudaStream_t st) {
    constexpr int kStep = 32 / kLanes * kAtOnce;
    const int hd = A.pages.head_dim;
    const bool plain = A.aligned && (A.heads == 0 || A.out_aligned) && (A.turn == kNoTurn || A.turn == kHalfLanes);
    const bool exact = plain && hd == kLanes * 8 && A.heads % kStep == 0 && A.pages.kv_heads % kStep == 0 &&
                       (A.turn == kNoTurn || A.r == hd);
    const char* who = "epq_paged_write";
    if (exact) return launch(write_kernel<T, kFormat, kLanes, kExact>, dim3(blocks), dim3(kCacheThreads), 0, st, who, A);
    if (plain) return launch(write_kernel<T, kFormat, kLanes, kLanesOnly>, dim3(blocks), dim3(kCacheThreads), 0, st, who, A);
    return launch(write_kernel<T, kFormat, kLanes, kAny>, dim3(blocks), dim3(kCacheThreads), 0, st, who, A);
}
template <typename T, int kFormat>
int launch_write(const WriteArgs& A, unsigned blocks, cudaStream_t st) {
    const int hd = A.pages.head_dim;
    if (hd <= 64) return launch_write_l<T, kFormat, 8>(A, blocks, st);
    return hd <= 128 ? launch_write_l<T, kFormat, 16>(A, blocks, st) : launch_write_l<T, kFormat, 32>(A, blocks, st);
}
template <typename T>
int launch_write_t(const WriteArgs& A, unsigned blocks, cudaStream_t st) {
    if (A.pages.format == EPQ_CACHE_SAME) return launch_write<T, EPQ_CACHE_SAME>(A, blocks, st);
    if (A.pages.format == EPQ_CACHE_INT8) return launch_write<T, EPQ_CACHE_INT8>(A, blocks, st);
    return launch_write<T, EPQ_CACHE_FP8>(A, blocks, st);
}
template <typename T>
int launch_read_t(const ReadArgs& A, unsigned blocks, cudaStream_t st) {
    const char* who = "epq_paged_read";
    if (A.pages.format == EPQ_CACHE_SAME)
        return launch(read_kernel<T, EPQ_CACHE_SAME>, dim3(blocks), dim3(kCacheThreads), 0, st, who, A);
    if (A.pages.format == EPQ_CACHE_INT8)
        return launch(read_kernel<T, EPQ_CACHE_INT8>, dim3(blocks), dim3(kCacheThreads), 0, st, who, A);
    return launch(read_kernel<T, EPQ_CACHE_FP8>, dim3(blocks), dim3(kCacheThreads), 0, st, who, A);
}

// Warps a token: one, or as many as it has passes while there are too few tokens to give
// every SM 32 warps.  (The bounded write kernels hold 28 of them, so some sizes end with a
// round of their own: 2048 tokens of 16 + 8 + 8 heads have 3 warps each, 1.5 rounds.)
int share_out(int64_t m, int64_t passes) {
    int64_t splits = cdiv((int64_t)device_sms() * 32, m);
    return (int)(splits < passes ? splits : passes);
}

}  // namespace

int make_pages(const epq_pages* in, PagesD* d, const char* who) {
    if (!in) return set_error(EPQ_EINVAL, "%s: pages is NULL", who);
    if (in->kv_heads <= 0 || in->page_size <= 0 || in->seqs <= 0 || in->max_pages <= 0 || in->pages <= 0)
        return set_error(EPQ_EINVAL, "%s: kv_heads=%d, page_size=%d, seqs=%d, max_pages=%d, pages=%lld", who,
                         in->kv_heads, in->page_size, in->seqs, in->max_pages, (long long)in->pages);
    if (!in->k || !in->v || !in->table) return set_error(EPQ_EINVAL, "%s: k, v and table must be non-NULL", who);
    if (in->head_dim < 16 || in->head_dim > 256 || in->head_dim % 16)
        return set_error(EPQ_EUNSUPPORTED, "%s: head_dim=%d (a multiple of 16 up to 256)", who, in->head_dim);
    if (in->format < EPQ_CACHE_SAME || in->format > EPQ_CACHE_FP8)
        return set_error(EPQ_EINVAL, "%s: format=%d", who, in->format);
    if (in->format != EPQ_CACHE_SAME && (!in->k_scale || !in->v_scale))
        return set_error(EPQ_EINVAL, "%s: an 8-bit cache needs k_scale and v_scale", who);
    // positions and a page's rows are 32-bit in the kernels, with room for a block past the end
    const int64_t rows = (int64_t)in->kv_heads * in->page_size;
    if ((int64_t)in->max_pages * in->page_size > INT32_MAX - 64 || rows > INT32_MAX - 64 || in->kv_heads > 65536)
        return set_error(EPQ_EUNSUPPORTED, "%s: %d pages of %d tokens a sequence, %d kv heads", who, in->max_pages,
                         in->page_size, in->kv_heads);
    if (in->page_stride < rows * in->head_dim || in->table_stride < in->max_pages ||
        (in->format != EPQ_CACHE_SAME && in->scale_stride < rows))
        return set_error(EPQ_ESHAPE, "%s: strides of pages (%lld), scales (%lld) or table (%lld) are too small", who,
                         (long long)in->page_stride, (long long)in->scale_stride, (long long)in->table_stride);
    if (((uintptr_t)in->k | (uintptr_t)in->v) % 16 || in->page_stride % 16)
        return set_error(EPQ_EALIGN, "%s: k, v and page_stride must be multiples of 16 bytes / values", who);
    d->k = static_cast<uint8_t*>(in->k);
    d->v = static_cast<uint8_t*>(in->v);
    d->k_scale = in->k_scale;
    d->v_scale = in->v_scale;
    d->table = in->table;
    d->page_stride = in->page_stride;
    d->scale_stride = in->scale_stride;
    d->table_stride = in->table_stride;
    d->pages = in->pages;
    d->seqs = in->seqs;
    d->max_pages = in->max_pages;
    d->page_size = in->page_size;
    d->kv_heads = in->kv_heads;
    d->head_dim = in->head_dim;
    d->format = in->format;
    // t / page_size = (mulhi(t, page_mul) + t) >> page_shift, exact for all t < 2^31
    d->page_shift = 0;
    while ((1u << d->page_shift) < (uint32_t)in->page_size) ++d->page_shift;
    d->page_mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << d->page_shift) - in->page_size)) / in->page_size + 1);
    return EPQ_OK;
}

int cache_read_device_error(int* flag) {
    if (cudaMemcpyFromSymbol(flag, g_cache_error, sizeof(int)) != cudaSuccess)
        return check_launch("read paged cache error flag");
    return EPQ_OK;
}

}  // namespace paged
}  // namespace epq

using namespace epq;
using namespace epq::paged;

extern "C" {

int epq_paged_write(const epq_pages* pages, const epq_heads* q, const epq_heads* q_out, const epq_heads* k,
                    const epq_heads* v, const int32_t* seq, const int64_t* pos, int64_t m, const float* cos_tab,
                    const float* sin_tab, int64_t max_len, int32_t rotary_dim, int32_t interleaved,
                    int32_t qk_norm, float eps, int32_t dtype, void* stream) {
    WriteArgs A = {};
    const int rc = make_pages(pages, &A.pages, "epq_paged_write");
    if (rc != EPQ_OK) return rc;
    if (!k || !v || m < 0 || (!q) != (!q_out) || (!cos_tab) != (!sin_tab))
        return set_error(EPQ_EINVAL, "epq_paged_write: bad arguments");
    if (!dtype_ok(dtype)) return set_error(EPQ_EDTYPE, "epq_paged_write: dtype %d", dtype);
    const int hd = A.pages.head_dim, KV = A.pages.kv_heads, elem = dtype_size(dtype);
    if (k->heads != KV || v->heads != KV || (q && (q->heads <= 0 || q->heads != q_out->heads || q->heads > 65536)))
        return set_error(EPQ_ESHAPE, "epq_paged_write: %d k heads and %d v heads for a cache of %d", k->heads,
                         v->heads, KV);
    if (cos_tab && (rotary_dim < 2 || rotary_dim > hd || rotary_dim % 2 || max_len <= 0))
        return set_error(EPQ_EUNSUPPORTED, "epq_paged_write: rotary_dim=%d (even, 2..%d)", rotary_dim, hd);
    if (m == 0) return EPQ_OK;
    if (!seq || !pos || !k->data || !v->data || (q && (!q->data || !q_out->data)))
        return set_error(EPQ_EINVAL, "epq_paged_write: NULL rows, seq or pos");
    if (q && (heads_overlap(*q_out, m, hd) || moved_in_place(*q, *q_out, m)))
        return set_error(EPQ_ESHAPE, "epq_paged_write: rows or heads of q_out overlap (strides %lld, %lld)",
                         (long long)q_out->stride_row, (long long)q_out->stride_head);
    A.k = {k->data, k->stride_row, k->stride_head};
    A.v = {v->data, v->stride_row, v->stride_head};
    A.aligned = heads_aligned(*k, elem, 16) && heads_aligned(*v, elem, 16);
    if (q) {
        A.q = {q->data, q->stride_row, q->stride_head};
        A.aligned = A.aligned && heads_aligned(*q, elem, 16);
        A.q_out = q_out->data;
        A.qo_row = q_out->stride_row;
        A.qo_head = q_out->stride_head;
        A.out_aligned = heads_aligned(*q_out, elem, 16);
        A.heads = q->heads;
    }
    A.seq = seq;
    A.pos = pos;
    A.cos_t = cos_tab;
    A.sin_t = sin_tab;
    A.m = m;
    A.max_len = max_len;
    A.r = rotary_dim;
    const bool whole = rotary_dim % 16 == 0 && ((uintptr_t)cos_tab | (uintptr_t)sin_tab) % 16 == 0;
    A.turn = !cos_tab ? kNoTurn : interleaved ? kNeighbours : whole ? kHalfLanes : kHalfLoads;
    // In place, a lane's loads of its partner's values would race with that lane's store.
    if (A.turn == kHalfLoads && q && q->data == q_out->data)
        return set_error(EPQ_EUNSUPPORTED, "epq_paged_write: q in place needs rotary_dim %% 16 == 0 (got %d) and aligned tables",
                         rotary_dim);
    A.qk_norm = qk_norm != 0;
    A.eps = eps;
    const int fit = hd <= 64 ? 4 : hd <= 128 ? 2 : 1;
    A.splits = share_out(m, cdiv(A.heads, fit * kAtOnce) + 2 * cdiv(KV, fit * kAtOnce));
    if (m * A.splits > (int64_t)1 << 30)
        return set_error(EPQ_EUNSUPPORTED, "epq_paged_write: m=%lld rows", (long long)m);
    const unsigned blocks = (unsigned)cdiv(m * A.splits * 32, kCacheThreads);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == EPQ_F32) return launch_write_t<float>(A, blocks, st);
    if (dtype == EPQ_F16) return launch_write_t<__half>(A, blocks, st);
    return launch_write_t<__nv_bfloat16>(A, blocks, st);
}

int epq_paged_read(const epq_pages* pages, const int32_t* seq, const int64_t* pos, int64_t m, void* k_out,
                   void* v_out, int32_t dtype, void* stream) {
    ReadArgs A = {};
    const int rc = make_pages(pages, &A.pages, "epq_paged_read");
    if (rc != EPQ_OK) return rc;
    if (m < 0) return set_error(EPQ_EINVAL, "epq_paged_read: m=%lld", (long long)m);
    if (!dtype_ok(dtype)) return set_error(EPQ_EDTYPE, "epq_paged_read: dtype %d", dtype);
    if (m == 0) return EPQ_OK;
    if (!seq || !pos || !k_out || !v_out) return set_error(EPQ_EINVAL, "epq_paged_read: NULL rows, seq or pos");
    if (((uintptr_t)k_out | (uintptr_t)v_out) % 16)
        return set_error(EPQ_EALIGN, "epq_paged_read: k_out and v_out must be 16-byte aligned");
    A.seq = seq;
    A.pos = pos;
    A.k_out = k_out;
    A.v_out = v_out;
    A.m = m;
    A.splits = share_out(m, cdiv(2 * A.pages.kv_heads * (A.pages.head_dim / 16), 32));
    if (m * A.splits > (int64_t)1 << 30)
        return set_error(EPQ_EUNSUPPORTED, "epq_paged_read: m=%lld rows", (long long)m);
    const unsigned blocks = (unsigned)cdiv(m * A.splits * 32, kCacheThreads);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == EPQ_F32) return launch_read_t<float>(A, blocks, st);
    if (dtype == EPQ_F16) return launch_read_t<__half>(A, blocks, st);
    return launch_read_t<__nv_bfloat16>(A, blocks, st);
}

}  // extern "C"
