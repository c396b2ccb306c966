// Attention of new tokens over a paged key/value cache:
//   out_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r k_j - max_j),
// over the rows j that row r = (token, query head) sees: the sequence's cached rows, and those of its new
// rows that a bit mask (a drafted tree) or the order (a chain) lets it see.
//
// The keys of a sequence are cut into ranges, one workgroup each, where the rows alone leave the chip idle; a
// range's maximum (base 2), sum and unnormalised output are joined by a second kernel in the order of the ranges,
// so a call repeats itself to the bit.  Its bits go by what chooses the kernel and the cut: all sequences' lengths,
// max_new, alignment, the workgroups that the device runs at once, and, on the vector ALUs, the table's width.  How long a range is, every workgroup works out from all
// sequences' lengths, which only the device knows (CallPlan in qmm_paged_attention.h): the host sees no more than the width of the table.
#include "qmm_paged_attention.h"

namespace qmm {
namespace paged {

int tree_attention(const qmm_paged_kv* kv, const qmm_paged_query* in, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    View v;
    const int rc = check_query(kv, in, &v);
    if (rc != QMM_OK) return rc;
    if (in->tokens == 0 || v.c.batch == 0 || in->max_new == 0) return QMM_OK;
    const Plan p = plan<Tree>(v, *in);
    std::unique_lock<std::mutex> held;  // until the merge is enqueued
    if (p.bytes > 0) {
        if (workspace) {
            if (workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
                return bad("the workspace must be 16-byte aligned and hold qmm_paged_attention_workspace() bytes.");
        } else {
            const hipError_t e = take_workspace(WorkspaceKind::kAttention, stream, p.bytes, held, &workspace);
            if (e != hipSuccess) return launched(e, "paged attention workspace");
        }
    }
    const AttnArgs a = attention_args(v, *in, p, workspace);
    const int launch = launch_attention<Tree>(v, a, p, stream);
    if (launch != QMM_OK || !p.merge) return launch;
    return launch_merge<Tree>(v, a, p.kind != Kind::kLanes, p.most_ranges, stream);
}

}  // namespace paged
}  // namespace qmm

extern "C" {

size_t qmm_paged_attention_workspace(const qmm_paged_kv* kv, const qmm_paged_query* in) {
    size_t bytes = 0;
    qmm::paged::entry([&] {
        qmm::paged::View v;
        const int rc = qmm::paged::check_query(kv, in, &v);
        if (rc == QMM_OK && in->tokens > 0) bytes = qmm::paged::plan<qmm::paged::Tree>(v, *in).bytes;
        return rc;
    });
    return bytes;
}

int qmm_paged_tree_attention(const qmm_paged_kv* kv, const qmm_paged_query* in, void* workspace, size_t workspace_bytes, void* stream) {
    return qmm::paged::entry([&] {
        return qmm::paged::tree_attention(kv, in, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
