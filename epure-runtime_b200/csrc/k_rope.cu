// Rotary positions (epq_rope): y_a = x_a cos - x_b sin, y_b = x_b cos + x_a sin for the
// pairs (a, b) of the first rotary_dim values of every head, in the half layout
// (j, j + r/2) or the interleaved one (2j, 2j + 1); the rest is copied.  The inverse
// turn (sin negated) is the gradient.
//
// Bound: HBM.  Every value is read and written once (2 elem bytes a value, 3 flops);
// cos / sin are 4 r bytes a token, shared by its heads.
//
// Split: one warp takes (a share of) one token's heads.  A lane keeps one item of a
// head -- V pairs of the half layout, or V neighbouring values -- over all heads it
// visits, so its cos / sin stay in registers and the table is read once a token.  The
// rows of the next heads are fetched while the last ones are turned, the first while the
// position and the table are on their way: 16384 tokens of 24 heads in bf16, forward and
// gradient, take 70 us (404 MB, 89% of the copy rate; 94 us without fetching ahead).
#include "epq_paged.cuh"

namespace epq {
namespace paged {
namespace {

__device__ int g_rope_error = 0;

struct RopeArgs {
    const void* x[2];
    void* y[2];
    int64_t xr[2], xh[2], yr[2], yh[2];   // row and head strides, in elements
    int heads[2];
    const int64_t* pos;
    const float* cos_t;
    const float* sin_t;
    int64_t m, max_len;
    int hd, r, lanes, splits, inverse, wide_table;
};

// N values of a table; `wide`: the address is a multiple of their size, 16 bytes at most.
template <int N> __device__ __forceinline__ void load_table(float (&f)[N], const float* p, int wide) {
    if (N > 1 && wide) {
        load_v<float, N>(f, p);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = p[i];
    }
}

constexpr int kRopeThreads = 128;

// Heads of one lane in flight: as many as keep about 64 bytes of it under way, and 32 of
// single 16-bit values and of interleaved float32.  (Half
// layout in bf16, 16384 tokens: 83 us with 1, 70 with 2 and 4; interleaved 77 with 2, 68
// with 4; single values, 8192 tokens: 139 with 2, 105 with 4.)
template <typename T, int V, bool kInterleaved> constexpr int rope_heads() {
    return V <= 2 ? 8 : kInterleaved && sizeof(T) == 2 ? 4 : 2;
}

// V: values a load (V = 1: any alignment and size).  An item holds V pairs (half
// layout) or max(V, 2) neighbouring values (interleaved), or is V copied values.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs A) {
    pdl_enter();
    constexpr int kRopeHeads = rope_heads<T, V, kInterleaved>();
    constexpr int kNear = V > 1 ? V : 2;                    // values of an interleaved item
    constexpr int kPairs = kInterleaved ? kNear / 2 : V;
    using W = typename Word<V * (int)sizeof(T)>::type;
    const int warp = blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int64_t row = warp / A.splits;
    if (row >= A.m) return;
    const int split = warp - (int)row * A.splits;
    const int half = A.r >> 1;
    const int turns = kInterleaved ? A.r / kNear : half / V;
    const int items = turns + (A.hd - A.r) / V;
    const int fit = 32 / A.lanes;                           // heads side by side in the warp
    const int sub = lane / A.lanes, first = lane - sub * A.lanes;
    // A pass is kRopeHeads groups of `fit` heads of one tensor; this warp's are [p0, p1).  A
    // pass is fetched while the one before it (first: the position) is worked on.
    const int step = kRopeHeads * fit;
    const int passes0 = (A.heads[0] + step - 1) / step, passes = passes0 + (A.heads[1] + step - 1) / step;
    const int p0 = passes * split / A.splits, p1 = passes * (split + 1) / A.splits;
    for (int it = first; it < items; it += A.lanes) {
        const bool copied = it >= turns;
        const int a0 = copied ? A.r + (it - turns) * V : kInterleaved ? it * kNear : it * V;
        // the second value or word of a pair that is not side by side with the first
        const int apart = copied ? 0 : kInterleaved ? (V > 1 ? 0 : 1) : half;
        W next_a[kRopeHeads], next_b[kRopeHeads];
        auto fetch = [&](int p) {
            const int t = p >= passes0, h0 = (t ? p - passes0 : p) * step + sub;
            const T* x = static_cast<const T*>(A.x[t]) + row * A.xr[t] + a0;
#pragma unroll
            for (int e = 0; e < kRopeHeads; ++e) {
                const T* at = x + min(h0 + e * fit, A.heads[t] - 1) * A.xh[t];  // past the end: the last head again
                next_a[e] = *reinterpret_cast<const W*>(at);
                if (apart) next_b[e] = *reinterpret_cast<const W*>(at + apart);
            }
        };
        if (sub < fit && p0 < p1) fetch(p0);
        const int64_t pos = A.pos[row];
        const bool inside = pos >= 0 && pos < A.max_len;
        if (!inside && lane == 0) atomicOr(&g_rope_error, kBadPosition);
        if (sub >= fit) return;
        float c[kPairs], s[kPairs];
        if (inside && !copied) {
            const int64_t at = pos * half + (kInterleaved ? a0 >> 1 : a0);
            load_table<kPairs>(c, A.cos_t + at, A.wide_table);
            load_table<kPairs>(s, A.sin_t + at, A.wide_table);
            if (A.inverse) {
#pragma unroll
                for (int i = 0; i < kPairs; ++i) s[i] = -s[i];
            }
        }
        for (int p = p0; p < p1; ++p) {
            W u[kRopeHeads], w[kRopeHeads];
#pragma unroll
            for (int e = 0; e < kRopeHeads; ++e) {
                u[e] = next_a[e];
                w[e] = next_b[e];
            }
            if (p + 1 < p1) fetch(p + 1);
            const int t = p >= passes0, h0 = (t ? p - passes0 : p) * step + sub;
            T* const y = static_cast<T*>(A.y[t]) + row * A.yr[t] + a0;
#pragma unroll
            for (int e = 0; e < kRopeHeads; ++e) {
                const int h = h0 + e * fit;
                if (h >= A.heads[t]) break;
                if (!inside) {
                    u[e] = W{};
                    w[e] = W{};
                } else if (!copied) {
                    float a[V], b[V];
                    load_v<T, V>(a, reinterpret_cast<const T*>(&u[e]));
                    if (apart) load_v<T, V>(b, reinterpret_cast<const T*>(&w[e]));
                    if constexpr (kInterleaved && V > 1) {
#pragma unroll
                        for (int i = 0; i < V / 2; ++i) turn(a[2 * i], a[2 * i + 1], c[i], s[i]);
                    } else if constexpr (V == 1) {
                        turn(a[0], b[0], c[0], s[0]);
                    } else {
#pragma unroll
                        for (int i = 0; i < V; i += 2) turn2(a[i], a[i + 1], b[i], b[i + 1], c[i], c[i + 1], s[i], s[i + 1]);
                    }
                    store_v<T, V>(reinterpret_cast<T*>(&u[e]), a);
                    if (apart) store_v<T, V>(reinterpret_cast<T*>(&w[e]), b);
                }
                T* const at = y + h * A.yh[t];
                *reinterpret_cast<W*>(at) = u[e];
                if (apart) *reinterpret_cast<W*>(at + apart) = w[e];
            }
        }
    }
}

template <typename T, int V, bool kInterleaved>
int launch_rope_l(RopeArgs A, cudaStream_t st) {
    const int step = rope_heads<T, V, kInterleaved>() * (32 / A.lanes);
    const int64_t passes = cdiv(A.heads[0], step) + cdiv(A.heads[1], step);
    // A token's heads are shared out to several warps while there are too few tokens to
    // give every SM 16 warps (4096 tokens of 10 heads of 64, both directions: 9.9 us, 12.1
    // with 32; 16384 tokens with up to 128: 80 instead of 70).
    int64_t splits = cdiv((int64_t)device_sms() * 16, A.m);
    if (splits > passes) splits = passes;
    A.splits = (int)splits;
    if (A.m * splits > (int64_t)1 << 30)
        return set_error(EPQ_EUNSUPPORTED, "epq_rope: m=%lld rows", (long long)A.m);
    const unsigned blocks = (unsigned)cdiv(A.m * splits * 32, kRopeThreads);
    return launch(rope_kernel<T, V, kInterleaved>, dim3(blocks), dim3(kRopeThreads), 0, st, "epq_rope", A);
}
template <typename T, int V> int launch_rope_v(const RopeArgs& A, bool interleaved, cudaStream_t st) {
    return interleaved ? launch_rope_l<T, V, true>(A, st) : launch_rope_l<T, V, false>(A, st);
}

}  // namespace

int rope_read_device_error(int* flag) {
    if (cudaMemcpyFromSymbol(flag, g_rope_error, sizeof(int)) != cudaSuccess)
        return check_launch("read rotary error flag");
    return EPQ_OK;
}

}  // namespace paged
}  // namespace epq

using namespace epq;
using namespace epq::paged;

extern "C" int epq_rope(const epq_heads* x, const epq_heads* y, int32_t count, const int64_t* pos, int64_t m,
                        int32_t head_dim, int32_t rotary_dim, const float* cos_tab, const float* sin_tab,
                        int64_t max_len, int32_t interleaved, int32_t inverse, int32_t dtype, void* stream) {
    if (!x || !y || (m > 0 && !pos) || !cos_tab || !sin_tab || count < 1 || count > 2 || m < 0 || max_len <= 0)
        return set_error(EPQ_EINVAL, "epq_rope: bad arguments");
    if (!dtype_ok(dtype)) return set_error(EPQ_EDTYPE, "epq_rope: dtype %d", dtype);
    if (head_dim < 2 || head_dim > 1024 || rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2)
        return set_error(EPQ_EUNSUPPORTED, "epq_rope: rotary_dim=%d (even, 2..head_dim) of head_dim=%d (2..1024)",
                         rotary_dim, head_dim);
    const int elem = dtype_size(dtype);
    RopeArgs A = {};
    int64_t heads = 0;
    for (int i = 0; i < count; ++i) {
        if (x[i].heads < 0 || x[i].heads != y[i].heads)
            return set_error(EPQ_ESHAPE, "epq_rope: %d heads in, %d out", x[i].heads, y[i].heads);
        if (m > 0 && x[i].heads > 0 && (!x[i].data || !y[i].data))
            return set_error(EPQ_EINVAL, "epq_rope: tensor %d is NULL", i);
        A.x[i] = x[i].data;
        A.y[i] = y[i].data;
        A.xr[i] = x[i].stride_row;
        A.xh[i] = x[i].stride_head;
        A.yr[i] = y[i].stride_row;
        A.yh[i] = y[i].stride_head;
        A.heads[i] = x[i].heads;
        heads += x[i].heads;
    }
    if (heads > 65536) return set_error(EPQ_EUNSUPPORTED, "epq_rope: %lld heads > 65536", (long long)heads);
    if (m == 0 || heads == 0) return EPQ_OK;
    for (int i = 0; i < count; ++i)
        if (heads_overlap(y[i], m, head_dim) || moved_in_place(x[i], y[i], m))
            return set_error(EPQ_ESHAPE, "epq_rope: rows or heads of output %d overlap (strides %lld, %lld)", i,
                             (long long)y[i].stride_row, (long long)y[i].stride_head);
    A.pos = pos;
    A.cos_t = cos_tab;
    A.sin_t = sin_tab;
    A.m = m;
    A.max_len = max_len;
    A.hd = head_dim;
    A.r = rotary_dim;
    A.inverse = inverse != 0;
    // The widest load that every row, head and part of a head is a multiple of: 16
    // bytes, else pairs of values, else single ones.
    const int part = interleaved ? rotary_dim : rotary_dim / 2;
    auto fits = [&](int v) {
        if (part % v || head_dim % v || (head_dim - rotary_dim) % v) return false;
        for (int i = 0; i < count; ++i)
            if (x[i].heads && (!heads_aligned(x[i], elem, v * elem) || !heads_aligned(y[i], elem, v * elem)))
                return false;
        return true;
    };
    const int wide = 16 / elem;
    const int v = fits(wide) ? wide : fits(2) ? 2 : 1;
    const int turns = interleaved ? rotary_dim / (v > 1 ? v : 2) : rotary_dim / 2 / v;
    const int items = turns + (head_dim - rotary_dim) / v;
    // Lanes a head: each has one item of it, or up to 4, where that leaves fewer of the
    // warp's lanes without work (20 items: 2 a lane of 3 heads at once, 60 of 64 places).
    double best = 0;
    for (int n = 1; n <= 4 || A.lanes == 0; ++n) {
        const int lanes = (items + n - 1) / n;
        if (lanes > 32) continue;
        const double used = (double)items * (32 / lanes) / (32.0 * n);
        if (used > best * 1.1) {
            best = used;
            A.lanes = lanes;
        }
    }
    const int pairs = interleaved ? (v > 1 ? v / 2 : 1) : v;
    A.wide_table = ((uintptr_t)cos_tab | (uintptr_t)sin_tab) % 16 == 0 && rotary_dim / 2 % (pairs < 4 ? pairs : 4) == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool il = interleaved != 0;
    if (dtype == EPQ_F32) {
        if (v == 4) return launch_rope_v<float, 4>(A, il, st);
        return v == 2 ? launch_rope_v<float, 2>(A, il, st) : launch_rope_v<float, 1>(A, il, st);
    }
    if (dtype == EPQ_F16) {
        if (v == 8) return launch_rope_v<__half, 8>(A, il, st);
        return v == 2 ? launch_rope_v<__half, 2>(A, il, st) : launch_rope_v<__half, 1>(A, il, st);
    }
    if (v == 8) return launch_rope_v<__nv_bfloat16, 8>(A, il, st);
    return v == 2 ? launch_rope_v<__nv_bfloat16, 2>(A, il, st)
                  : launch_rope_v<__nv_bfloat16, 1>(A, il, st);
}
