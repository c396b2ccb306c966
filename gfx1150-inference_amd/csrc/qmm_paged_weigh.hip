// Attention that also tells what every cached row was worth: beside the outputs, for each kv head and row j of a sequence,
//   sum over the new tokens i that see j and the query heads h of the kv head of  exp(scale q_ih k_j - log sum_j' exp(scale q_ih k_j')),
// on top of what the row has gathered before.  The attention's kernels leave the logarithms of the rows' sums, and a
// second pass over the keys forms the weights from them: every sum belongs to one thread group, which adds in a fixed
// order, so that a call repeats itself to the bit.
#include "qmm_paged_attention.h"

namespace qmm {
namespace paged {
namespace {

struct WeighArgs {
    qmm_paged_weights w;
    int blocks;  // along the rows
};

// The rows of a sequence that have a sum.
__device__ __forceinline__ int summed_rows(const WeighArgs& wa, const Span& s) {
    return static_cast<int>(min(static_cast<int64_t>(s.ctx) + s.n, static_cast<int64_t>(wa.w.rows)));
}

// Every head size and alignment: groups of `lpk` lanes take a key each and go through the sequence's queries.
// Block (x, y, z): keys, kv head, sequence.
template <class T, class C>
__global__ __launch_bounds__(kThreads) void weigh_lanes_kernel(View v, AttnArgs a, WeighArgs wa, int aligned) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, D = v.c.head_dim, g = blockIdx.y, group = a.in.heads / v.c.kv_heads;
    const Span s = span_of<Lse>(v, a, blockIdx.z);
    const int lpk = lanes_per_key(D), sub = lane % lpk, d0 = 8 * sub, per_wave = 64 / lpk;
    const int held = summed_rows(wa, s), tokens = min(s.n, a.in.max_new);
    const float* from = wa.w.old_sums + blockIdx.z * wa.w.old_batch + g * wa.w.old_head;
    float* to = wa.w.new_sums + blockIdx.z * wa.w.new_batch + g * wa.w.new_head;
    for (int64_t k0 = static_cast<int64_t>(blockIdx.x) * 4 * per_wave; k0 < held; k0 += static_cast<int64_t>(wa.blocks) * 4 * per_wave) {
        const int64_t at = k0 + w * per_wave + lane / lpk;
        const int k = static_cast<int>(min(at, static_cast<int64_t>(held) - 1));
        const bool live = at < held;
        const int page = live && k < s.total ? page_of(v, s.seq, k) : -1;
        float x[8], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0f;
        if (page >= 0 && d0 < D)
            load8f(static_cast<const C*>(v.c.k) + page * v.c.k_page + g * v.c.k_head + (k & (v.c.page_size - 1)) * v.c.k_slot + d0, aligned, x);
        for (int r = 0; r < tokens * group; ++r) {
            const int i = r / group, head = g * group + r % group;
            const T* qp = static_cast<const T*>(a.in.q) + static_cast<int64_t>(s.first + i) * a.in.q_token + head * a.in.q_head;
            float dot = 0.0f;
            if (d0 < D)
#pragma unroll
                for (int e = 0; e < 8; ++e) dot += to_float(qp[d0 + e]) * x[e];
            for (int o = lpk / 2; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
            if (page >= 0 && (k < s.ctx || sees_new(a, s, i, k - s.ctx)))
                sum += __builtin_amdgcn_exp2f(dot * a.scale_log2 - a.lse[static_cast<int64_t>(s.first + i) * a.in.heads + head]);
        }
        if (live && sub == 0) to[k] = k < s.ctx ? from[k] + sum : sum;
    }
}

struct WeighPlan {
    Plan attend;
    size_t lse, bytes;  // where the logarithms begin
};

WeighPlan weigh_plan(const View& v, const qmm_paged_query& in) {
    WeighPlan p{};
    p.attend = plan<Lse>(v, in);
    p.lse = (p.attend.bytes + 15) / 16 * 16;
    p.bytes = p.lse + (static_cast<size_t>(in.tokens) * in.heads * sizeof(float) + 15) / 16 * 16;
    return p;
}

int check_weights(const View& v, const qmm_paged_weights* w) {
    if (!w) return bad("weights must be non-null.");
    if (w->rows < 0) return bad("rows must be non-negative.");
    if (w->rows > 0 && v.c.batch > 0 && (!w->old_sums || !w->new_sums)) return bad("old_sums and new_sums must be non-null.");
    if ((reinterpret_cast<uintptr_t>(w->old_sums) | reinterpret_cast<uintptr_t>(w->new_sums)) % 4 != 0) return bad("old_sums and new_sums must be aligned to their elements.");
    if (w->old_sums == w->new_sums && (w->old_batch != w->new_batch || w->old_head != w->new_head)) return bad("sums in place need the same strides.");
    if (v.c.kv_heads > 65535) return bad("too many heads.");
    return QMM_OK;
}

int weighted_attention(const qmm_paged_kv* kv, const qmm_paged_query* in, const qmm_paged_weights* weights, void* workspace,
                       size_t workspace_bytes, hipStream_t stream) {
    View v;
    int rc = check_query(kv, in, &v);
    if (rc == QMM_OK) rc = check_weights(v, weights);
    if (rc != QMM_OK) return rc;
    if (v.c.batch == 0) return QMM_OK;
    const bool attends = in->tokens > 0 && in->max_new > 0;
    const WeighPlan p = weigh_plan(v, *in);
    std::unique_lock<std::mutex> held;  // until the last launch is enqueued
    if (workspace) {
        if (workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return bad("the workspace must be 16-byte aligned and hold qmm_paged_weighted_workspace() bytes.");
    } else if (attends) {
        const hipError_t e = take_workspace(WorkspaceKind::kAttention, stream, p.bytes, held, &workspace);
        if (e != hipSuccess) return launched(e, "paged attention workspace");
    }
    AttnArgs a = attention_args(v, *in, p.attend, workspace);
    a.lse = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.lse);
    if (attends) {
        rc = launch_attention<Lse>(v, a, p.attend, stream);
        if (rc == QMM_OK && p.attend.merge) rc = launch_merge<Lse>(v, a, p.attend.kind != Kind::kLanes, p.attend.most_ranges, stream);
        if (rc != QMM_OK) return rc;
    }
    // a row of no sequence has no sum; what the table can hold bounds the cached ones that have been given pages
    WeighArgs wa{*weights, 1};
    if (weights->rows == 0) return QMM_OK;
    const int keys = 4 * (64 / (v.c.head_dim <= 64 ? 8 : v.c.head_dim <= 128 ? 16 : 32));
    wa.blocks = static_cast<int>(std::min<int64_t>((weights->rows + keys - 1) / keys, 1024));
    const dim3 grid(static_cast<unsigned>(wa.blocks), static_cast<unsigned>(v.c.kv_heads), static_cast<unsigned>(v.c.batch));
    const int aligned = operands_aligned(v) ? 1 : 0;
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, stream, v, a, wa, aligned); };
    const bool fp8 = v.c.dtype == QMM_DTYPE_E4M3;
    if (in->dtype == QMM_DTYPE_F16) fp8 ? go(weigh_lanes_kernel<_Float16, Fp8>) : go(weigh_lanes_kernel<_Float16, _Float16>);
    else fp8 ? go(weigh_lanes_kernel<__bf16, Fp8>) : go(weigh_lanes_kernel<__bf16, __bf16>);
    return launched(hipGetLastError(), "paged weights kernel launch");
}

}  // namespace
}  // namespace paged
}  // namespace qmm

extern "C" {

size_t qmm_paged_weighted_workspace(const qmm_paged_kv* kv, const qmm_paged_query* in, const qmm_paged_weights* weights) {
    size_t bytes = 0;
    qmm::paged::entry([&] {
        qmm::paged::View v;
        int rc = qmm::paged::check_query(kv, in, &v);
        if (rc == QMM_OK) rc = qmm::paged::check_weights(v, weights);
        if (rc == QMM_OK && in->tokens > 0 && v.c.batch > 0) bytes = qmm::paged::weigh_plan(v, *in).bytes;
        return rc;
    });
    return bytes;
}

int qmm_paged_weighted_attention(const qmm_paged_kv* kv, const qmm_paged_query* in, const qmm_paged_weights* weights, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    return qmm::paged::entry([&] {
        return qmm::paged::weighted_attention(kv, in, weights, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
