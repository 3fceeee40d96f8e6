// Attention of one new token a row where rows share a prefix (epq_paged_attend_shared).  Each
// row goes through all of its tokens by itself.
#include "epq_attend.cuh"

namespace epq {
namespace paged {
namespace {

__device__ int g_shared_error = 0;

}  // namespace

int shared_read_device_error(int* flag) {
    if (cudaMemcpyFromSymbol(flag, g_shared_error, sizeof(int)) != cudaSuccess)
        return check_launch("read shared attention error flag");
    return EPQ_OK;
}

}  // namespace paged
}  // namespace epq

using namespace epq;
using namespace epq::paged;

extern "C" {

int64_t epq_paged_attend_shared_workspace_bytes(const epq_pages* pages, int64_t batch, int32_t heads, int64_t groups) {
    if (groups < 0) return set_error(EPQ_EINVAL, "epq_paged_attend_shared: groups=%lld", (long long)groups);
    return attend_bytes("epq_paged_attend_shared", pages, batch, heads);
}

int epq_paged_attend_shared(const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                            int64_t batch, const int32_t* starts, const int64_t* prefix, int64_t groups, float scale, void* out,
                            float* lse, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    if (groups < 0 || (groups && (!starts || !prefix)))
        return set_error(EPQ_EINVAL, "epq_paged_attend_shared: groups=%lld, or NULL starts or prefix", (long long)groups);
    return epq_paged_attend(pages, q, seq, lengths, batch, scale, 0, out, lse, dtype, workspace, workspace_bytes, stream);
}

}  // extern "C"
