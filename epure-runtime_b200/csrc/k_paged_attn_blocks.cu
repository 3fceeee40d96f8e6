// Attention of one new token a row over the blocks that a list of each row and key head
// names (epq_paged_attend_blocks): the kernel of k_paged_attn.cu with one more access between
// a block's place and its page.  A place in the list is a page's worth of tokens; the list
// entry of the next block is looked up while the block before it is copied, as the page's
// number is (one block earlier: no change).
//
// Measured (B200, graphs of calls): 64 rows x 8 key heads x 64 blocks of 32 tokens, 64 heads of 128, e4m3: 64 us, 4.2 TB/s (units
// are short, so their joins and starts count); 1 x 8 x 64 blocks of 64, bf16: 12.6 us.
#include "epq_attend.cuh"

namespace epq {
namespace paged {

int attend_blocks_read_device_error(int* flag) { return read_attend_error(flag); }

}  // namespace paged
}  // namespace epq

using namespace epq;
using namespace epq::paged;

extern "C" int epq_paged_attend_blocks(const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                                       int64_t batch, const int32_t* blocks, int32_t count, float scale, void* out, float* lse,
                                       int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    AttendArgs A = {};
    int cols;
    bool ready;
    if (count < 0) return set_error(EPQ_EINVAL, "epq_paged_attend_blocks: count=%d", count);
    const int rc = make_attend("epq_paged_attend_blocks", pages, q, seq, lengths, batch, scale, out, lse, dtype, workspace,
                               workspace_bytes, &A, &cols, &ready);
    if (rc != EPQ_OK || !ready) return rc;
    if (!blocks && count) return set_error(EPQ_EINVAL, "epq_paged_attend_blocks: blocks is NULL");
    A.blocks = blocks;
    A.count = count;
    return launch_attend_mode<kListed>(A, cols, static_cast<cudaStream_t>(stream));
}
