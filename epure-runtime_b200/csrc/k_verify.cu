// Verification of drafted tokens against the target's probabilities (epq_verify_drafts).
//
// Bound: HBM for a batch, latency for a row: of each row one step's probabilities are read
// once, target and draft, and a chain of dependent accesses remains (drafts, their
// probabilities, the weights, the place of the drawn token).
//
// Split.  A row is a thread-block cluster; each of its warps sums the weights of one run of the
// vocabulary in 64 bits.  The sums of all warps are scanned in distributed shared memory by
// every CTA alike, and the one warp whose run holds the drawn token goes through it a second
// time (from L2).  So results depend neither on timing nor on another row.
// 64 bits, because the drawn token is where a cumulative sum passes a number: float32 sums of
// 128k weights would move it in about one draw of a hundred.
#include "epq_common.cuh"
#include "epq_paged.cuh"
#include "epq_sampling.h"

namespace epq {
namespace sampling {
namespace {

__device__ int g_verify_error = 0;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;
constexpr int kRuns = kCluster * kWarps;       // runs of the vocabulary
static_assert(kRuns % 32 == 0, "a warp scans the runs");

struct VerifyArgs {
    epq_probs p, q;                            // q.data NULL: drafts of probability 1
    const int64_t* tokens;
    const float* uniforms;
    int64_t tokens_stride, uniforms_stride, vocab;
    int64_t* out;
    int64_t* accepted;
    int drafts;
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ double cluster_load(const double* mine, unsigned rank) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(mine);
    uint32_t there;
    double v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(there) : "memory");
    return v;
}

// kV values of a row from element e on, as they count: those of [0, n) and 0 outside.  With
// kV > 1 the address of element e is a multiple of their size.
template <typename T, int kV> __device__ __forceinline__ void fetch(float (&f)[kV], const T* row, int64_t e, int64_t n) {
    if (kV > 1 && e >= 0 && e + kV <= n) {
        paged::load_v<T, kV>(f, row + e);
    } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) f[i] = e + i >= 0 && e + i < n ? paged::to_f<T>(row[e + i]) : 0.f;
    }
}

// Inclusive sums over the lanes.
__device__ __forceinline__ double scan(double v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(kAll, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

template <typename T, int kV>
__global__ void __launch_bounds__(kThreads) verify_kernel(const VerifyArgs A) {
    __shared__ int taken_at;                   // accepted drafts, times 2, and whether the next one was refused
    __shared__ double sums[kWarps];
    paged::pdl_enter();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t b = blockIdx.x / kCluster;
    const int rank = blockIdx.x % kCluster;
    const T* p0 = static_cast<const T*>(A.p.data) + b * A.p.stride_row;
    const T* q0 = static_cast<const T*>(A.q.data) + b * A.q.stride_row;
    const int64_t* x = A.tokens + b * A.tokens_stride;
    const float* u = A.uniforms + b * A.uniforms_stride;
    const int64_t V = A.vocab;

    // ---- accepted drafts (every CTA finds them alike)
    if (warp == 0) {
        int n = A.drafts, refused = 0;
        for (int i0 = 0; i0 < A.drafts; i0 += 32) {
            const int i = i0 + lane;
            bool keep = false, there = false;
            if (i < A.drafts) {
                const int64_t t = x[i];
                if (t >= V && rank == 0) atomicOr(&g_verify_error, 1);
                there = t >= 0 && t < V;
                if (there) {
                    const double px = paged::to_f<T>(p0[i * A.p.stride_step + t]);
                    const double qx = A.q.data ? (double)paged::to_f<T>(q0[i * A.q.stride_step + t]) : 1.0;
                    keep = (double)u[i] * qx < px;
                }
            }
            const unsigned stop = __ballot_sync(kAll, !keep && i < A.drafts);
            if (stop) {
                const int at = __ffs(stop) - 1;
                n = i0 + at;
                refused = __shfl_sync(kAll, (int)there, at);
                break;
            }
        }
        if (lane == 0) taken_at = 2 * n + refused;
    }
    __syncthreads();
    const int n = taken_at >> 1;
    const T* p = p0 + n * A.p.stride_step;
    const T* q = q0 + n * A.q.stride_step;
    const double draw = (double)u[A.drafts];

    // ---- weights; elements are counted from a 16-byte boundary of p's row
    const int64_t head = kV > 1 ? (int64_t)((uintptr_t)p % 16 / sizeof(T)) : 0;
    constexpr int kTile = 32 * kV;
    const int64_t tiles = (head + V + kTile - 1) / kTile, per = (tiles + kRuns - 1) / kRuns;
    const int run = rank * kWarps + warp;
    const int64_t t0 = min(tiles, run * per), t1 = min(tiles, t0 + per);
    // 0: the whole row; 1: max(p - q, 0); 2: all but the drafted token
    int how = taken_at & 1 ? (A.q.data ? 1 : 2) : 0;
    const int64_t without = how == 2 ? x[n] : -1;
    auto weights = [&](int64_t tile, double (&w)[kV]) {
        const int64_t e = tile * kTile + lane * kV - head;
        float f[kV], g[kV];
        fetch<T, kV>(f, p, e, V);
        if (how == 1) fetch<T, kV>(g, q, e, V);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            double v = how == 1 ? (double)f[i] - (double)g[i] : (double)f[i];
            if (e + i == without) v = 0.0;
            w[i] = v > 0.0 ? v : 0.0;          // (NaN too)
        }
    };
    double total = 0.0, target = 0.0, upto = 0.0, mine = 0.0;
    int from = -1, last_with = -1;
    for (int pass = 0;; ++pass) {              // (all CTAs go through it equally often, whatever they read)
        mine = 0.0;
        constexpr int kAtOnce = kV > 1 ? 4 : 8;
        for (int64_t t = t0; t < t1; t += kAtOnce) {
            double w[kAtOnce][kV];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (t + i < t1) {
                    weights(t + i, w[i]);
                } else {
#pragma unroll
                    for (int k = 0; k < kV; ++k) w[i][k] = 0.0;
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                for (int k = 0; k < kV; ++k) mine += w[i][k];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(kAll, mine, o);
        if (lane == 0) sums[warp] = mine;
        cluster_sync();
        // every warp scans the runs' sums: lane l those of kRuns / 32 runs
        constexpr int kEach = kRuns / 32;
        double part[kEach], own = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = lane * kEach + i;
            part[i] = cluster_load(sums + r % kWarps, r / kWarps);
            own += part[i];
        }
        const double to = scan(own, lane);
        total = __shfl_sync(kAll, to, 31);
        target = draw * total;
        double at = to - own;
        int hit = kRuns, with = -1;            // first run that passes the target, last run with a weight
        double before = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (part[i] > 0.0) {
                with = lane * kEach + i;
                if (hit == kRuns && at + part[i] > target) {
                    hit = lane * kEach + i;
                    before = at;
                }
            }
            at += part[i];
        }
        const int first = __reduce_min_sync(kAll, hit);
        last_with = __reduce_max_sync(kAll, with);
        from = first < kRuns ? first : last_with;
        upto = __shfl_sync(kAll, before, first < kRuns ? first / kEach : 0);
        if (first == kRuns) target = INFINITY;                         // the last token with a weight
        cluster_sync();                        // nobody reads the sums any more
        if (last_with >= 0 || pass) break;
        how = 0;                               // nothing is left of the residual: p itself
    }

    // ---- the drawn token, by the warp whose run it is in (-1: by the first)
    if (run != max(from, 0)) return;
    int64_t token = -1;
    if (from >= 0) {
        for (int64_t t = t0; t < t1; ++t) {
            double w[kV], own = 0.0;
            weights(t, w);
#pragma unroll
            for (int k = 0; k < kV; ++k) own += w[k];
            const double to = scan(own, lane);
            double at = upto + (to - own);
            int64_t found = -1, with = -1;
#pragma unroll
            for (int k = 0; k < kV; ++k) {
                at += w[k];
                if (w[k] > 0.0) {
                    with = t * kTile + lane * kV + k - head;
                    if (found < 0 && at > target) found = with;
                }
            }
            const unsigned any = __ballot_sync(kAll, found >= 0), some = __ballot_sync(kAll, with >= 0);
            if (any) {
                token = __shfl_sync(kAll, found, __ffs(any) - 1);
                break;
            }
            // where the two orders of summing differ in the last bit, the run's last token with a weight
            if (some) token = __shfl_sync(kAll, with, 31 - __clz(some));
            upto += __shfl_sync(kAll, to, 31);
        }
    }
    int64_t* out = A.out + b * (A.drafts + 1);
    for (int i = lane; i <= A.drafts; i += 32) out[i] = i < n ? x[i] : i == n ? token : -1;
    if (lane == 0) A.accepted[b] = n;
}

template <typename T, int kV>
int launch_verify(const VerifyArgs& A, int64_t batch, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * kCluster));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kCluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, verify_kernel<T, kV>, A);
    return check_launch("epq_verify_drafts");
}

template <typename T> int launch_verify_t(const VerifyArgs& A, int64_t batch, cudaStream_t st) {
    constexpr int kV = 16 / (int)sizeof(T);
    // wide loads where p and q of every row and step have the same place within 16 bytes
    const bool wide = !A.q.data || (((uintptr_t)A.p.data - (uintptr_t)A.q.data) % 16 == 0 &&
                                    (A.p.stride_row - A.q.stride_row) * (int64_t)sizeof(T) % 16 == 0 &&
                                    (A.p.stride_step - A.q.stride_step) * (int64_t)sizeof(T) % 16 == 0);
    return wide ? launch_verify<T, kV>(A, batch, st) : launch_verify<T, 1>(A, batch, st);
}

}  // namespace

int verify_read_device_error(int* flag) {
    if (cudaMemcpyFromSymbol(flag, g_verify_error, sizeof(int)) != cudaSuccess)
        return check_launch("read draft verification error flag");
    return EPQ_OK;
}

}  // namespace sampling
}  // namespace epq

using namespace epq;
using namespace epq::sampling;

extern "C" int epq_verify_drafts(const epq_probs* target, const epq_probs* draft, const int64_t* tokens, int64_t tokens_stride,
                                 const float* uniforms, int64_t uniforms_stride, int64_t batch, int32_t drafts, int64_t vocab,
                                 int32_t dtype, int64_t* out, int64_t* accepted, void* stream) {
    if (!target || batch < 0 || drafts < 0 || vocab < 1)
        return set_error(EPQ_EINVAL, "epq_verify_drafts: batch=%lld, drafts=%d, vocab=%lld", (long long)batch, drafts,
                         (long long)vocab);
    if (!dtype_ok(dtype)) return set_error(EPQ_EDTYPE, "epq_verify_drafts: dtype %d", dtype);
    if (batch > INT32_MAX / kCluster || drafts > (1 << 20) || vocab > INT32_MAX)
        return set_error(EPQ_EUNSUPPORTED, "epq_verify_drafts: batch=%lld, drafts=%d, vocab=%lld", (long long)batch, drafts,
                         (long long)vocab);
    if (batch == 0) return EPQ_OK;
    if (!target->data || (draft && drafts && !draft->data) || (!tokens && drafts) || !uniforms || !out || !accepted)
        return set_error(EPQ_EINVAL, "epq_verify_drafts: NULL probabilities, tokens, uniforms or outputs");
    const int elem = dtype_size(dtype);
    if ((uintptr_t)target->data % elem || (draft && (uintptr_t)draft->data % elem))
        return set_error(EPQ_EALIGN, "epq_verify_drafts: probabilities must have the alignment of their type");
    VerifyArgs A = {};
    A.p = *target;
    if (draft && drafts) A.q = *draft;         // without drafts there is nothing to refuse
    A.tokens = tokens;
    A.uniforms = uniforms;
    A.tokens_stride = tokens_stride;
    A.uniforms_stride = uniforms_stride;
    A.vocab = vocab;
    A.out = out;
    A.accepted = accepted;
    A.drafts = drafts;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == EPQ_F32) return launch_verify_t<float>(A, batch, st);
    if (dtype == EPQ_F16) return launch_verify_t<__half>(A, batch, st);
    return launch_verify_t<__nv_bfloat16>(A, batch, st);
}
