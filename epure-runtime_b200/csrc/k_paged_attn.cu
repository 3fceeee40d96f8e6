// Attention of one new token a sequence over a paged cache (epq_paged_attend):
//   out[b, h] = sum_t softmax_t(scale q[b, h] . K[t]) V[t],  t in [max(0, n - window), n).
//
// Bound: HBM.  Every cached key and value is read once: 2 flops a value and query head,
// 8 flops a byte at 8 heads a key head in bf16, far below what the tensor cores need.
// The work is to keep enough loads in flight on every SM, whatever the lengths are.
//
// Split.  A unit is (sequence, key head, up to 8 or 16 of its query heads); its tokens
// are cut into blocks of 16 or 32.  The blocks of all units, in order, are dealt out to
// the CTAs in equal runs, each unit counting for its own cost too, so ragged lengths load
// every SM alike; where there are few units each CTA takes one piece of one instead.  A
// unit that is cut is joined from (m, M, l, accumulator) records by the last of its CTAs
// to finish, in the order of the CTAs, so results do not depend on timing.  Within a CTA
// warp w takes the blocks w, w + 4, ... of the run; each warp has its own ring of
// shared-memory stages filled by 16-byte asynchronous copies that run ahead over unit
// boundaries, 64 to 130 KB in flight an SM.
//
// Mathematics of a block: S^T = K Q^T as m16n8k16 products with 16 tokens as rows and
// the query heads as the 8 columns, so a group of up to 8 heads fills the tile (with
// heads as rows half of it or more would be padding); O^T = V^T P^T likewise, with the
// head's dims as rows.  tcgen05's tiles have 128 rows and at most 8 columns would be
// used; the tensor pipe is not what limits this kernel.  The running maximum moves only
// when a score passes it by 2^8; sums are float32.
//
// Measured (B200, device time in a graph of calls): 1 x 131072 tokens, 32 / 8 heads of
// 128, bf16: 90 us, 6.0 TB/s (93% of the measured copy rate); 64 sequences of up to 8192,
// 64 / 8 heads, e4m3: 98 us, 5.7 TB/s; 16 of up to 4096, 32 / 8 heads, int8: 21 us, of
// which 3 are the plan and first loads and 4 the last joins; 1 x 145: 6.4 us, a chain of
// five dependent memory accesses and one join of warps.
//
// 8-bit caches: codes are converted to f16 (exact: int8 and e4m3 fit its 11 bits); a
// head's q is brought to f16 by a power of two (exact for values down to 2^-28 of the
// largest, the others to 2^-39 of the largest's power of two); the key's scale multiplies
// the score, and the value's scale enters the weight as 2^(s + log2 scale - M) with a
// running maximum M of its own, so that neither large nor small scales leave f16's range.
#include "epq_attend.cuh"

namespace epq {
namespace paged {
namespace {

// Columns of 8 query heads a unit has: one, or two for groups above 8.
int cols_of(int group) { return group <= 8 ? 1 : 2; }

int64_t records_bytes(int hd, int group) {
    const int dim = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    return (int64_t)kMaxGrid * 2 * cols_of(group) * 8 * (dim + 4) * 4;
}

}  // namespace

int attend_read_device_error(int* flag) { return read_attend_error(flag); }

int launch_attend_plain(const AttendArgs& A, int cols, cudaStream_t st) { return launch_attend_mode<kAllTokens>(A, cols, st); }

int64_t attend_bytes(const char* who, const epq_pages* pages, int64_t batch, int32_t heads) {
    PagesD P;
    const int rc = make_pages(pages, &P, who);
    if (rc != EPQ_OK) return rc;
    if (batch < 0 || heads <= 0 || heads % P.kv_heads)
        return set_error(EPQ_ESHAPE, "%s: %d query heads over %d key heads", who, heads, P.kv_heads);
    return (int64_t)kMaxUnits * 4 + records_bytes(P.head_dim, heads / P.kv_heads);
}

int make_attend(const char* who, const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                int64_t batch, float scale, void* out, float* lse, int32_t dtype, void* workspace, int64_t workspace_bytes,
                AttendArgs* A, int* cols, bool* ready) {
    *ready = false;
    const int rc = make_pages(pages, &A->pages, who);
    if (rc != EPQ_OK) return rc;
    const int KV = A->pages.kv_heads;
    if (!q || batch < 0) return set_error(EPQ_EINVAL, "%s: bad arguments", who);
    if (dtype != EPQ_BF16 && dtype != EPQ_F16) return set_error(EPQ_EDTYPE, "%s: dtype %d (f16 or bf16)", who, dtype);
    if (q->heads <= 0 || q->heads % KV)
        return set_error(EPQ_ESHAPE, "%s: %d query heads over %d key heads", who, q->heads, KV);
    A->group = q->heads / KV;
    *cols = cols_of(A->group);
    A->chunks = (A->group + 8 * *cols - 1) / (8 * *cols);
    if (batch * KV * A->chunks > kMaxUnits)
        return set_error(EPQ_EUNSUPPORTED, "%s: batch=%lld of %d key heads (at most %d units)", who, (long long)batch, KV,
                         kMaxUnits);
    if (!seq && batch > A->pages.seqs)
        return set_error(EPQ_ESHAPE, "%s: batch=%lld of a table of %d sequences", who, (long long)batch, A->pages.seqs);
    // a batch's blocks are counted in 32 bits, and a CTA's run of all units' blocks too (at least 64 CTAs share them)
    const int64_t most = batch * ((int64_t)A->pages.max_pages * A->pages.page_size / kTile + 1 + kUnitCost);
    if (most > INT32_MAX || most * KV * A->chunks > (int64_t)INT32_MAX * 64)
        return set_error(EPQ_EUNSUPPORTED, "%s: batch=%lld of up to %lld tokens each", who, (long long)batch,
                         (long long)A->pages.max_pages * A->pages.page_size);
    if (batch == 0) return EPQ_OK;
    if (!q->data || !lengths || !out) return set_error(EPQ_EINVAL, "%s: NULL q, lengths or out", who);
    if (!heads_aligned(*q, 2, 4) || (uintptr_t)out % 16)
        return set_error(EPQ_EALIGN, "%s: q must be 4-byte aligned with even strides, out 16-byte aligned", who);
    const int64_t need = attend_bytes(who, pages, batch, q->heads);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
        return set_error(EPQ_EWORKSPACE, "%s: workspace of %lld bytes (need %lld, 256-aligned)", who,
                         (long long)workspace_bytes, (long long)need);
    A->q = q->data;
    A->q_row = q->stride_row;
    A->q_head = q->stride_head;
    A->seq = seq;
    A->lengths = lengths;
    A->out = out;
    A->lse = lse;
    A->counters = static_cast<unsigned*>(workspace);
    A->records = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (int64_t)kMaxUnits * 4);
    A->batch = (int)batch;
    A->heads = q->heads;
    A->dtype = dtype;
    A->scale_log2 = scale * kLog2e;
    *ready = true;
    return EPQ_OK;
}

}  // namespace paged
}  // namespace epq

using namespace epq;
using namespace epq::paged;

extern "C" {

int64_t epq_paged_attend_workspace_bytes(const epq_pages* pages, int64_t batch, int32_t heads) {
    return attend_bytes("epq_paged_attend_workspace_bytes", pages, batch, heads);
}

int epq_paged_attend(const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                     int64_t batch, float scale, int64_t window, void* out, float* lse, int32_t dtype,
                     void* workspace, int64_t workspace_bytes, void* stream) {
    AttendArgs A = {};
    int cols;
    bool ready;
    if (window < 0) return set_error(EPQ_EINVAL, "epq_paged_attend: bad arguments");
    const int rc = make_attend("epq_paged_attend", pages, q, seq, lengths, batch, scale, out, lse, dtype, workspace,
                               workspace_bytes, &A, &cols, &ready);
    if (rc != EPQ_OK || !ready) return rc;
    A.window = window;
    return launch_attend_plain(A, cols, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
