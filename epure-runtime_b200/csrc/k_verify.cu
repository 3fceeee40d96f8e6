// Verification of drafted tokens against the target's probabilities (epq_verify_drafts).
//
// Bound: HBM for a batch, latency for a row: of each row one step's probabilities are read
// once, target and draft, and a chain of dependent accesses remains (drafts, their
// probabilities, the weights, the place of the drawn token).
//
// Split.  A row is a thread-block cluster; each of its warps sums the weights of one run of the
// vocabulary.  The runs' sums are scanned in distributed shared memory by every CTA alike; the
// CTA whose run holds the drawn token goes through that run a second time (from L2), a part of it
// a warp, and the warp whose part holds it a third time.  So results depend neither on timing nor
// on another row.
//
// Precision.  The drawn token is where a cumulative sum passes a number: float32 sums of 128k
// weights would move it in about one draw of a hundred.  64-bit additions, and above all the
// conversions to 64 bits, are what the first pass would spend its time on, so it sums in pairs of
// float32: each sum and difference with what its rounding left over, which keeps about 46 bits.
// All that follows is 64-bit.
//
// Measured (B200, graphs of calls): 64 x 4 drafts over 128,256 tokens, float32: 16.8 us (10.2 at the copy rate); 1 x 4 over
// 151,936: 9.9 us; 33 x 7 looked up over 32,001, bf16: 6.9 us.  With 64-bit sums in the first pass 1 x 4 took 21 us.
#include "epq_common.cuh"
#include "epq_paged.cuh"
#include "epq_sampling.h"

namespace epq {
namespace sampling {
namespace {

__device__ int g_verify_error = 0;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kCluster = 8;
// Threads a CTA: few rows have the most warps on each of them, many rows all CTAs of a row of 64
// sequences on the card at once (4 an SM).
constexpr int kFew = 1024, kMany = 256;

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
template <typename T, int kV> __device__ __forceinline__ void fetch(float (&f)[kV], const T* row, int e, int n) {
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

// A sum in two floats: values that were added, and what the additions' roundings left over.
struct Sum {
    float s = 0.f, rest = 0.f;
    __device__ __forceinline__ void add(float x, float left) {
        const float t = s + x, z = t - s;
        rest += (s - (t - z)) + (x - z) + left;
        s = t;
    }
    __device__ __forceinline__ double value() const { return isinf(s) ? (double)s : (double)s + (double)rest; }
};

template <typename T, int kV, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == kMany ? 4 : 1) verify_kernel(const VerifyArgs A) {
    constexpr int kWarps = kThreads / 32, kRuns = kCluster * kWarps;   // runs of the vocabulary
    static_assert(kRuns % 32 == 0, "a warp scans the runs");
    __shared__ int taken_at;                   // accepted drafts, times 2, and whether the next one was refused
    __shared__ double sums[kWarps], parts[kWarps], found_target, found_upto;
    __shared__ int found_run;
    paged::pdl_enter();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t b = blockIdx.x / kCluster;
    const int rank = blockIdx.x % kCluster;
    const T* p0 = static_cast<const T*>(A.p.data) + b * A.p.stride_row;
    const T* q0 = static_cast<const T*>(A.q.data) + b * A.q.stride_row;
    const int64_t* x = A.tokens + b * A.tokens_stride;
    const float* u = A.uniforms + b * A.uniforms_stride;
    const int64_t V = A.vocab;
    const double draw = (double)u[A.drafts];

    // ---- accepted drafts (every CTA finds them alike)
    if (warp == 0) {
        int n = A.drafts, refused = 0;
        for (int i0 = 0; i0 < A.drafts; i0 += 32) {
            const int i = i0 + lane;
            bool keep = false, there = false;
            if (i < A.drafts) {
                const int64_t t = x[i];
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
    } else if (warp == 1 && rank == 0) {       // what ends the row's drafts: a negative token, or one to report
        for (int i0 = 0; i0 < A.drafts; i0 += 32) {
            const int64_t t = i0 + lane < A.drafts ? x[i0 + lane] : 0;
            const unsigned past = __ballot_sync(kAll, t >= V), ends = __ballot_sync(kAll, t < 0) | past;
            if (ends) {
                if (lane == 0 && past >> (__ffs(ends) - 1) & 1) atomicOr(&g_verify_error, 1);
                break;
            }
        }
    }
    __syncthreads();
    const int n = taken_at >> 1;
    const T* p = p0 + n * A.p.stride_step;
    const T* q = q0 + n * A.q.stride_step;

    // ---- weights; elements are counted from a 16-byte boundary of p's row
    const int head = kV > 1 ? (int)((uintptr_t)p % 16 / sizeof(T)) : 0;
    constexpr int kTile = 32 * kV;
    const int vocab = (int)V, tiles = (head + vocab + kTile - 1) / kTile, per = (tiles + kRuns - 1) / kRuns;
    // 0: the whole row; 1: max(p - q, 0); 2: all but the drafted token
    int how = taken_at & 1 ? (A.q.data ? 1 : 2) : 0;
    int without = how == 2 ? (int)x[n] : -1;
    auto load = [&](int tile, float (&f)[kV], float (&g)[kV]) {
        const int e = tile * kTile + lane * kV - head;
        fetch<T, kV>(f, p, e, vocab);
        if (how == 1) fetch<T, kV>(g, q, e, vocab);
    };
    auto weights = [&](int tile, double (&w)[kV]) {
        const int e = tile * kTile + lane * kV - head;
        float f[kV], g[kV];
        load(tile, f, g);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            const double v = how == 1 ? (double)f[i] - (double)g[i] : (double)f[i];
            w[i] = v > 0.0 && e + i != without ? v : 0.0;              // (NaN is none)
        }
    };
    auto added = [&](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
        return v;
    };
    double target = 0.0, upto = 0.0;
    int from = -1;
    for (int pass = 0;; ++pass) {              // (all CTAs go through it equally often, whatever they read)
        const int t0 = min(tiles, (rank * kWarps + warp) * per), t1 = min(tiles, t0 + per);
        Sum lanes[kV];
        constexpr int kAtOnce = kV > 4 ? 2 : kV > 1 ? 4 : 8;
        for (int t = t0; t < t1; t += kAtOnce) {
            float f[kAtOnce][kV], g[kAtOnce][kV];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) load(t + i < t1 ? t + i : tiles, f[i], g[i]);   // (tile `tiles` lies outside)
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                for (int k = 0; k < kV; ++k) {
                    const float a = f[i][k];
                    float d = a, left = 0.f;
                    if (how == 1) {
                        const float c = g[i][k];
                        d = a - c;
                        const float z = d - a;
                        left = (a - (d - z)) - (c + z);
                    } else if (how == 2 && (t + i) * kTile + lane * kV - head + k == without) {
                        d = 0.f;
                    }
                    const bool some = d > 0.f;                         // (NaN is none)
                    lanes[k].add(some ? d : 0.f, some ? left : 0.f);
                }
        }
        double mine = 0.0;
#pragma unroll
        for (int k = 0; k < kV; ++k) mine += lanes[k].value();
        mine = added(mine);
        if (lane == 0) sums[warp] = mine;
        cluster_sync();
        // a warp of each CTA scans the runs' sums: lane l those of kRuns / 32 runs
        if (warp == 0) {
            constexpr int kEach = kRuns / 32;
            double part[kEach], own = 0.0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int r = lane * kEach + i;
                part[i] = cluster_load(sums + r % kWarps, r / kWarps);
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i) own += part[i];
            const double to = scan(own, lane);
            target = draw * __shfl_sync(kAll, to, 31);
            double at = to - own;
            int hit = kRuns, with = -1;        // first run that passes the target, last run with a weight
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
            const int first = __reduce_min_sync(kAll, hit), last_with = __reduce_max_sync(kAll, with);
            upto = __shfl_sync(kAll, before, first < kRuns ? first / kEach : 0);
            if (lane == 0) {
                found_run = first < kRuns ? first : last_with;
                found_target = first < kRuns ? target : INFINITY;      // (else the last token with a weight)
                found_upto = upto;
            }
        }
        cluster_sync();                        // nobody reads the sums any more
        from = found_run;
        target = found_target;
        upto = found_upto;
        if (from >= 0 || pass) break;
        __syncthreads();                       // (the three are read)
        how = 0;                               // nothing is left of the residual: p itself, the drafted token too
        without = -1;
    }

    // ---- the drawn token, by the CTA whose run it is in (-1: by the first)
    if (rank != max(from, 0) / kWarps) return;
    int64_t* out = A.out + b * (A.drafts + 1);
    auto write = [&](int64_t token) {
        for (int i = lane; i <= A.drafts; i += 32) out[i] = i < n ? x[i] : i == n ? token : -1;
        if (lane == 0) A.accepted[b] = n;
    };
    if (from < 0) {
        if (warp == 0) write(-1);
        return;
    }
    const int r0 = min(tiles, from * per), r1 = min(tiles, r0 + per), each = (r1 - r0 + kWarps - 1) / kWarps;
    const int t0 = min(r1, r0 + warp * each), t1 = min(r1, t0 + each);
    double mine = 0.0;
    for (int t = t0; t < t1; ++t) {
        double w[kV];
        weights(t, w);
#pragma unroll
        for (int k = 0; k < kV; ++k) mine += w[k];
    }
    mine = added(mine);
    if (lane == 0) parts[warp] = mine;
    __syncthreads();
    const double own = lane < kWarps ? parts[lane] : 0.0, to = scan(own, lane);
    const unsigned some = __ballot_sync(kAll, own > 0.0), past = __ballot_sync(kAll, own > 0.0 && upto + to > target);
    // (where two orders of summing differ in the last bits, the run's last part with a weight)
    const int chosen = past ? __ffs(past) - 1 : some ? 31 - __clz(some) : 0;
    if (warp != chosen) return;
    upto += __shfl_sync(kAll, to - own, chosen);
    int64_t token = -1;
    for (int t = t0; t < t1; ++t) {
        double w[kV], sum = 0.0;
        weights(t, w);
#pragma unroll
        for (int k = 0; k < kV; ++k) sum += w[k];
        const double end = scan(sum, lane);
        double at = upto + (end - sum);
        int found = -1, with = -1;
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            at += w[k];
            if (w[k] > 0.0) {
                with = t * kTile + lane * kV + k - head;
                if (found < 0 && at > target) found = with;
            }
        }
        const unsigned any = __ballot_sync(kAll, found >= 0), weighed = __ballot_sync(kAll, with >= 0);
        if (any) {
            token = __shfl_sync(kAll, found, __ffs(any) - 1);
            break;
        }
        if (weighed) token = __shfl_sync(kAll, with, 31 - __clz(weighed));     // (the part's last, as above)
        upto += __shfl_sync(kAll, end, 31);
    }
    write(token);
}

template <typename T, int kV, int kThreads>
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
    cudaLaunchKernelEx(&cfg, verify_kernel<T, kV, kThreads>, A);
    return check_launch("epq_verify_drafts");
}

template <typename T> int launch_verify_t(const VerifyArgs& A, int64_t batch, cudaStream_t st) {
    constexpr int kV = 16 / (int)sizeof(T);
    // wide loads where p and q of every row and step have the same place within 16 bytes
    const bool wide = !A.q.data || (((uintptr_t)A.p.data - (uintptr_t)A.q.data) % 16 == 0 &&
                                    (A.p.stride_row - A.q.stride_row) * (int64_t)sizeof(T) % 16 == 0 &&
                                    (A.p.stride_step - A.q.stride_step) * (int64_t)sizeof(T) % 16 == 0);
    const bool few = batch * kCluster <= device_sms();
    if (wide) return few ? launch_verify<T, kV, kFew>(A, batch, st) : launch_verify<T, kV, kMany>(A, batch, st);
    return few ? launch_verify<T, 1, kFew>(A, batch, st) : launch_verify<T, 1, kMany>(A, batch, st);
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
    if (batch > INT32_MAX / kCluster || drafts > (1 << 20) || vocab > INT32_MAX / 2)
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
