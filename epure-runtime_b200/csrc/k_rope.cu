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
// visits, so its cos / sin stay in registers and the table is read once a token.
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
    int hd, r, splits, inverse;
};

constexpr int kRopeThreads = 128;
constexpr int kRopeHeads = 2;   // heads of one lane in flight

// V: values a load (V = 1: any alignment and size).  An item holds V pairs (half
// layout) or max(V, 2) neighbouring values (interleaved), or is V copied values.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs A) {
    pdl_enter();
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
    const int fit = items < 32 ? 32 / items : 1;            // heads side by side in the warp
    const int sub = items < 32 ? lane / items : 0;
    const int first = items < 32 ? lane - sub * items : lane;
    // this split's share [g0, g1) of the two tensors' groups of `fit` heads
    const int groups0 = (A.heads[0] + fit - 1) / fit, groups = groups0 + (A.heads[1] + fit - 1) / fit;
    const int g0 = (int)((int64_t)groups * split / A.splits), g1 = (int)((int64_t)groups * (split + 1) / A.splits);
    const int64_t p = A.pos[row];
    const bool inside = p >= 0 && p < A.max_len;
    if (!inside && lane == 0) atomicOr(&g_rope_error, kBadPosition);
    if (sub >= fit) return;
    for (int it = first; it < items; it += 32) {
        const bool copied = it >= turns;
        const int a0 = copied ? A.r + (it - turns) * V : kInterleaved ? it * kNear : it * V;
        // the second value or word of a pair that is not side by side with the first
        const int apart = copied ? 0 : kInterleaved ? (V > 1 ? 0 : 1) : half;
        float c[kPairs], s[kPairs];
        if (inside && !copied) {
            const int64_t at = p * half + (kInterleaved ? a0 >> 1 : a0);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                c[i] = A.cos_t[at + i];
                s[i] = A.inverse ? -A.sin_t[at + i] : A.sin_t[at + i];
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int from = (t ? max(g0 - groups0, 0) : g0) * fit + sub;
            const int to = min(A.heads[t], (t ? g1 - groups0 : min(g1, groups0)) * fit);
            const T* x = static_cast<const T*>(A.x[t]) + row * A.xr[t] + a0;
            T* y = static_cast<T*>(A.y[t]) + row * A.yr[t] + a0;
            for (int h0 = from; h0 < to; h0 += kRopeHeads * fit) {
                W u[kRopeHeads], w[kRopeHeads];
#pragma unroll
                for (int e = 0; e < kRopeHeads; ++e) {
                    const T* at = x + min(h0 + e * fit, to - 1) * A.xh[t];      // past the end: some head again
                    u[e] = *reinterpret_cast<const W*>(at);
                    if (apart) w[e] = *reinterpret_cast<const W*>(at + apart);
                }
#pragma unroll
                for (int e = 0; e < kRopeHeads; ++e) {
                    const int h = h0 + e * fit;
                    if (h >= to) break;
                    T* at = y + h * A.yh[t];
                    if (!inside) {
                        u[e] = W{};
                        w[e] = W{};
                    } else if (!copied) {
                        float a[V], b[V];
                        load_v<T, V>(a, reinterpret_cast<const T*>(&u[e]));
                        if (apart) load_v<T, V>(b, reinterpret_cast<const T*>(&w[e]));
                        if (!kInterleaved || V == 1) {
#pragma unroll
                            for (int i = 0; i < V; ++i) turn(a[i], b[i], c[i], s[i]);
                        } else {
#pragma unroll
                            for (int i = 0; i < V / 2; ++i) turn(a[2 * i], a[2 * i + 1], c[i], s[i]);
                        }
                        store_v<T, V>(reinterpret_cast<T*>(&u[e]), a);
                        if (apart) store_v<T, V>(reinterpret_cast<T*>(&w[e]), b);
                    }
                    *reinterpret_cast<W*>(at) = u[e];
                    if (apart) *reinterpret_cast<W*>(at + apart) = w[e];
                }
            }
        }
    }
}

template <typename T, int V>
int launch_rope_v(const RopeArgs& A, bool interleaved, unsigned blocks, cudaStream_t st) {
    return interleaved ? launch(rope_kernel<T, V, true>, dim3(blocks), dim3(kRopeThreads), 0, st, "epq_rope", A)
                       : launch(rope_kernel<T, V, false>, dim3(blocks), dim3(kRopeThreads), 0, st, "epq_rope", A);
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
    const int fit = items < 32 ? 32 / items : 1;
    const int64_t groups = cdiv(A.heads[0], fit) + cdiv(A.heads[1], fit);
    // A token's heads are shared out to several warps while there are too few tokens to
    // give every SM 16 warps.
    int64_t splits = cdiv((int64_t)device_sms() * 16, m);
    if (splits > groups) splits = groups;
    A.splits = (int)splits;
    if (m * splits > (int64_t)1 << 30) return set_error(EPQ_EUNSUPPORTED, "epq_rope: m=%lld rows", (long long)m);
    const unsigned blocks = (unsigned)cdiv(m * splits * 32, kRopeThreads);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool il = interleaved != 0;
    if (dtype == EPQ_F32) {
        if (v == 4) return launch_rope_v<float, 4>(A, il, blocks, st);
        return v == 2 ? launch_rope_v<float, 2>(A, il, blocks, st) : launch_rope_v<float, 1>(A, il, blocks, st);
    }
    if (dtype == EPQ_F16) {
        if (v == 8) return launch_rope_v<__half, 8>(A, il, blocks, st);
        return v == 2 ? launch_rope_v<__half, 2>(A, il, blocks, st) : launch_rope_v<__half, 1>(A, il, blocks, st);
    }
    if (v == 8) return launch_rope_v<__nv_bfloat16, 8>(A, il, blocks, st);
    return v == 2 ? launch_rope_v<__nv_bfloat16, 2>(A, il, blocks, st)
                  : launch_rope_v<__nv_bfloat16, 1>(A, il, blocks, st);
}
