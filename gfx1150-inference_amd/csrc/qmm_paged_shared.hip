// Attention of a batch whose groups of sequences begin with the same rows (a system prompt, a document, the prompt of
// a beam search): the group's tokens attend to the shared rows together, as the new tokens of one sequence that has
// these rows, and every token to the rest of its own sequence's; the partial rows of both, each with its maximum and sum,
// are joined as those of any two ranges are,
//   m = max(m1, m2),  out = (2^(m1 - m) o1 + 2^(m2 - m) o2) / (2^(m1 - m) l1 + 2^(m2 - m) l2).
#include "qmm_paged_attention.h"

namespace qmm {
namespace paged {
namespace {

// What the launches read of the groups.
struct Groups {
    const int32_t *first, *shared;
    int count;
    int32_t *starts, *cu, *ctx, *lead;  // [count + 1], [count + 1], [count], [count]
    int32_t* from;                      // [batch]
};

constexpr int kGroupThreads = 1024;

// One workgroup: where groups begin (made ascending, so that no sequence is in two), the rows that a group shares (no more than any
// of its sequences has cached, whole blocks of 16, which lie in one page; none where it has one sequence), and the row that every sequence
// goes on from.
__global__ __launch_bounds__(kGroupThreads) void groups_kernel(View v, Groups g) {
    const int tid = threadIdx.x, batch = v.c.batch;
    if (tid < 64) {
        int most = 0;
        for (int i0 = 0; i0 <= g.count; i0 += 64) {
            const int i = i0 + tid;
            int x = i <= g.count ? min(max(g.first[i], 0), batch) : 0;
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(x, o, 64);
                if (tid >= o) x = max(x, y);
            }
            x = max(x, most);
            most = __shfl(x, 63, 64);
            if (i <= g.count) {
                g.starts[i] = x;
                g.cu[i] = v.c.cu[x];
            }
        }
    }
    __syncthreads();
    const int64_t room = static_cast<int64_t>(v.c.table_width) << v.page_shift;
    for (int i = tid; i < g.count; i += kGroupThreads) {
        const int members = g.starts[i + 1] - g.starts[i];
        g.ctx[i] = members > 1 ? static_cast<int>(min(static_cast<int64_t>(max(g.shared[i], 0)), room)) : 0;
        g.lead[i] = min(g.starts[i], batch - 1);
    }
    __syncthreads();
    // the group of a sequence: the count of starts at or below it, less one
    auto group_of = [&](int b) {
        int lo = 0, hi = g.count + 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (g.starts[mid] <= b) lo = mid + 1;
            else hi = mid;
        }
        return lo - 1;
    };
    for (int b = tid; b < batch; b += kGroupThreads) {
        const int i = group_of(b);
        if (i >= 0 && i < g.count) atomicMin(&g.ctx[i], cached_rows(v, b));
    }
    __syncthreads();
    for (int i = tid; i < g.count; i += kGroupThreads) g.ctx[i] &= ~15;
    __syncthreads();
    for (int b = tid; b < batch; b += kGroupThreads) {
        const int i = group_of(b);
        g.from[b] = i >= 0 && i < g.count ? g.ctx[i] : 0;
    }
}

struct SharedPlan {
    Plan lead, rest;
    size_t groups, cut, ml, o, bytes;  // where the workspace's parts begin
    int64_t parts;                     // in rows
};

size_t whole(size_t bytes) { return (bytes + 15) / 16 * 16; }

int check_groups(const qmm_paged_groups* g) {
    if (!g) return bad("groups must be non-null.");
    if (g->count < 0 || g->count > 65535) return bad("the count of groups must be between 0 and 65535.");
    if (g->count > 0 && (!g->first || !g->shared)) return bad("first and shared must be non-null.");
    return QMM_OK;
}

// What groups share is taken apart where the matrix kernels serve the call; the others read every row for itself.
bool shares(const View& v, const qmm_paged_query& in, const qmm_paged_groups& g) {
    return g.count > 0 && matrix_operands(v, in) && static_cast<int64_t>(in.tokens) * (in.heads / v.c.kv_heads) <= (1 << 28);
}

View lead_view(const View& v, const qmm_paged_groups& g) {
    View u = v;
    u.c.batch = g.count;
    return u;
}

qmm_paged_query lead_query(const qmm_paged_query& in) {
    qmm_paged_query q = in;
    q.mask = nullptr;
    q.mask_words = 0;
    q.max_new = in.tokens;  // of a group
    return q;
}

SharedPlan shared_plan(const View& v, const qmm_paged_query& in, const qmm_paged_groups& g) {
    SharedPlan p{};
    p.rest = plan<Part>(v, in);
    p.lead = plan<Part>(lead_view(v, g), lead_query(in));
    p.parts = p.rest.parts + p.lead.parts;
    p.cut = whole((3 * static_cast<size_t>(g.count) + 2 + g.count + v.c.batch) * sizeof(int32_t));
    p.ml = p.cut + 2 * static_cast<size_t>(in.tokens) * sizeof(int4);
    p.o = p.ml + whole(static_cast<size_t>(p.parts) * sizeof(float2));
    p.bytes = p.o + static_cast<size_t>(p.parts) * v.c.head_dim * sizeof(float);
    return p;
}

int shared_attention(const qmm_paged_kv* kv, const qmm_paged_query* in, const qmm_paged_groups* groups, void* workspace,
                     size_t workspace_bytes, hipStream_t stream) {
    View v;
    int rc = check_query(kv, in, &v);
    if (rc == QMM_OK) rc = check_groups(groups);
    if (rc != QMM_OK) return rc;
    if (in->tokens == 0 || v.c.batch == 0 || in->max_new == 0) return QMM_OK;
    if (!shares(v, *in, *groups)) return tree_attention(kv, in, workspace, workspace_bytes, stream);
    const SharedPlan p = shared_plan(v, *in, *groups);
    std::unique_lock<std::mutex> held;  // until the join is enqueued
    if (workspace) {
        if (workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return bad("the workspace must be 16-byte aligned and hold qmm_paged_shared_workspace() bytes.");
    } else {
        const hipError_t e = take_workspace(WorkspaceKind::kAttention, stream, p.bytes, held, &workspace);
        if (e != hipSuccess) return launched(e, "paged attention workspace");
    }
    char* base = static_cast<char*>(workspace);
    Groups g{groups->first, groups->shared, groups->count, reinterpret_cast<int32_t*>(base), nullptr, nullptr, nullptr, nullptr};
    g.cu = g.starts + g.count + 1;
    g.ctx = g.cu + g.count + 1;
    g.lead = g.ctx + g.count;
    g.from = g.lead + g.count;
    hipLaunchKernelGGL(groups_kernel, dim3(1), dim3(kGroupThreads), 0, stream, v, g);
    rc = launched(hipGetLastError(), "paged groups kernel launch");
    if (rc != QMM_OK) return rc;

    AttnArgs rest{};
    rest.in = *in;
    rest.scale_log2 = score_scale(v, *in);
    rest.v_scale = v.c.v_scale;
    rest.slots = p.rest.slots;
    rest.part_o = reinterpret_cast<float*>(base + p.o);
    rest.part_ml = reinterpret_cast<float2*>(base + p.ml);
    rest.parts = p.rest.parts / in->heads;
    rest.cut = reinterpret_cast<int4*>(base + p.cut);
    rest.from = g.from;
    AttnArgs lead = rest;
    lead.in = lead_query(*in);
    lead.slots = p.lead.slots;
    lead.part_o = rest.part_o + rest.parts * in->heads * v.c.head_dim;
    lead.part_ml = rest.part_ml + rest.parts * in->heads;
    lead.parts = p.lead.parts / in->heads;
    lead.cut = rest.cut + in->tokens;
    lead.from = nullptr;
    lead.lead = g.lead;
    View u = lead_view(v, *groups);
    u.c.cu = g.cu;
    u.c.ctx = g.ctx;
    rc = launch_attention<Part>(u, lead, p.lead, stream);
    if (rc == QMM_OK) rc = launch_attention<Part>(v, rest, p.rest, stream);
    if (rc != QMM_OK) return rc;
    AttnArgs join = rest;
    join.lead_cut = lead.cut;
    join.lead_part = rest.parts;
    join.all_parts = rest.parts + lead.parts;
    return launch_merge<Part>(v, join, true, p.rest.most_ranges + p.lead.most_ranges, stream);
}

}  // namespace
}  // namespace paged
}  // namespace qmm

extern "C" {

size_t qmm_paged_shared_workspace(const qmm_paged_kv* kv, const qmm_paged_query* in, const qmm_paged_groups* groups) {
    size_t bytes = 0;
    qmm::paged::entry([&] {
        qmm::paged::View v;
        int rc = qmm::paged::check_query(kv, in, &v);
        if (rc == QMM_OK) rc = qmm::paged::check_groups(groups);
        if (rc == QMM_OK && in->tokens > 0 && v.c.batch > 0)
            bytes = qmm::paged::shares(v, *in, *groups) ? qmm::paged::shared_plan(v, *in, *groups).bytes : qmm_paged_attention_workspace(kv, in);
        return rc;
    });
    return bytes;
}

int qmm_paged_shared_attention(const qmm_paged_kv* kv, const qmm_paged_query* in, const qmm_paged_groups* groups, void* workspace,
                               size_t workspace_bytes, void* stream) {
    return qmm::paged::entry([&] {
        return qmm::paged::shared_attention(kv, in, groups, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
