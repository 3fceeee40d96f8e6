// Of epq_paged_attend_shared: each row's own tokens, behind those that it shares (epq_shared.cuh),
// by the kernel of k_paged_attn.cu.  Its sums are joined with those over the shared tokens.
#include "epq_attend.cuh"

namespace epq {
namespace paged {

int attend_behind_shared(const AttendArgs& A, int cols, cudaStream_t st) { return launch_attend_mode<kBehindShared>(A, cols, st); }
int attend_shared_read_device_error(int* flag) { return read_attend_error(flag); }

}  // namespace paged
}  // namespace epq
