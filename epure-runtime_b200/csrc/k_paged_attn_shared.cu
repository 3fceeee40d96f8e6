// The last launch of epq_paged_attend_shared: each row's own tokens, behind those that it shares
// (epq_shared.cuh), by the kernel of k_paged_attn.cu.  Where a row's result is written its sums
// are joined with the records that the shared part left, in the order of the pieces, so results
// do not depend on timing.
#include "epq_attend.cuh"

namespace epq {
namespace paged {

int attend_behind_shared(const AttendArgs& A, int cols, cudaStream_t st) { return launch_attend_mode<kBehindShared>(A, cols, st); }
int attend_shared_read_device_error(int* flag) { return read_attend_error(flag); }

}  // namespace paged
}  // namespace epq
