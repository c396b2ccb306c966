// Attention of new tokens over a paged key/value cache:
//   out_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r k_j - max_j),
// over the rows j that row r = (token, query head) sees: the sequence's cached rows, and those of its new
// rows that a bit mask (a drafted tree) or the order (a chain) lets it see.
//
// The keys of a sequence are cut into ranges of `kps`, one workgroup each, where the rows alone leave the
// chip idle; a range's maximum (base 2), sum and unnormalised output are joined by a second kernel in the
// order of the ranges, so a result depends on the call's sizes alone.
#include "qmm_paged.h"

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

namespace qmm {
namespace paged {
namespace {

constexpr int kThreads = 256;

struct AttnArgs {
    qmm_paged_query in;
    float scale_log2;  // scale * k_scale * log2 e
    float v_scale;
    int splits, kps;   // ranges of keys in the grid, keys per range
    float* part_o;     // [split][token][head][D]
    float2* part_ml;   // [split][token][head]: maximum, sum
};

// The new tokens of one sequence.
struct Span {
    int seq, first, n, ctx, total;  // first token, count, cached rows, rows that the table can hold of both
};

__device__ __forceinline__ Span span_of(const View& v, const AttnArgs& a, int seq) {
    Span s;
    s.seq = seq;
    s.first = max(v.c.cu[seq], 0);
    s.n = max(min(v.c.cu[seq + 1], a.in.tokens) - s.first, 0);
    s.ctx = min(max(v.c.ctx[seq], 0), 1 << 30);
    s.total = static_cast<int>(min(static_cast<int64_t>(s.ctx) + s.n, static_cast<int64_t>(v.c.table_width) << v.page_shift));
    return s;
}

// Does new token i of the sequence see its new token j?
__device__ __forceinline__ bool sees_new(const AttnArgs& a, const Span& s, int i, int j) {
    if (a.in.mask == nullptr) return j <= i;
    const int word = j >> 5;
    return word < a.in.mask_words && ((a.in.mask[(s.first + i) * a.in.mask_stride + word] >> (j & 31)) & 1);
}

template <class C>
__device__ __forceinline__ void load8f(const C* p, bool aligned, float (&x)[8]) {
    if (!aligned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to_float(p[e]);
    } else if constexpr (std::is_same_v<C, Fp8>) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), false);
            const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), true);
            x[4 * i] = lo[0];
            x[4 * i + 1] = lo[1];
            x[4 * i + 2] = hi[0];
            x[4 * i + 3] = hi[1];
        }
    } else {
        using V = std::conditional_t<std::is_same_v<C, _Float16>, f16x8, bf16x8>;
        const V w = *reinterpret_cast<const V*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(w[e]);
    }
}

// One row over the keys [begin, end) on the vector ALUs, one wave: groups of `lpk` lanes take every
// (64 / lpk)-th key, 8 dimensions a lane, each with an online softmax of its own; the groups are joined at the
// end.  A key that the row does not see is not read, and a weight of 0 takes nothing from its value, so that
// an infinite or NaN row reaches no output that does not see it.
struct RowState {
    float m, l, o[8];
};

template <class T, class C>
__device__ __forceinline__ RowState scan_row(const View& v, const AttnArgs& a, const Span& s, int i, int head, int begin, int end,
                                             int lane, int lpk, bool aligned) {
    const int D = v.c.head_dim, g = head / (a.in.heads / v.c.kv_heads);
    const int sub = lane % lpk, d0 = 8 * sub;
    const bool own = d0 < D;
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = 0.0f;
    const T* qp = static_cast<const T*>(a.in.q) + static_cast<int64_t>(s.first + i) * a.in.q_token + head * a.in.q_head;
    if (own)
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = to_float(qp[d0 + e]);
    RowState r;
    r.m = -INFINITY;
    r.l = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.o[e] = 0.0f;
    const int groups = 64 / lpk;
#pragma unroll 1
    for (int kb = begin; kb < end; kb += groups) {
        const int k = kb + lane / lpk;
        int page = -1;
        if (k < end && (k < s.ctx || sees_new(a, s, i, k - s.ctx))) page = page_of(v, s.seq, k);
        const int slot = k & (v.c.page_size - 1);
        float x[8], y[8], dot = 0.0f;
        if (page >= 0 && own) {
            load8f(static_cast<const C*>(v.c.k) + page * v.c.k_page + g * v.c.k_head + slot * v.c.k_slot + d0, aligned, x);
            load8f(static_cast<const C*>(v.c.v) + page * v.c.v_page + g * v.c.v_head + slot * v.c.v_slot + d0, aligned, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot += q[e] * x[e];
        }
        for (int o = lpk / 2; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
        if (page >= 0) {
            const float sc = dot * a.scale_log2;
            const float mn = fmaxf(r.m, sc);
            if (mn > r.m) {
                const float f = __builtin_amdgcn_exp2f(r.m - mn);
                r.l *= f;
#pragma unroll
                for (int e = 0; e < 8; ++e) r.o[e] = f > 0.0f ? r.o[e] * f : 0.0f;
                r.m = mn;
            }
            const float p = sc == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sc - r.m);
            r.l += p;
            if (own && !(p <= 0.0f))
#pragma unroll
                for (int e = 0; e < 8; ++e) r.o[e] += p * y[e];
        }
    }
    for (int o = lpk; o < 64; o <<= 1) {
        const float om = __shfl_xor(r.m, o, 64), ol = __shfl_xor(r.l, o, 64);
        const float mn = fmaxf(r.m, om);
        const float f = r.m == mn ? 1.0f : __builtin_amdgcn_exp2f(r.m - mn);
        const float g2 = om == mn ? 1.0f : __builtin_amdgcn_exp2f(om - mn);
        r.l = r.l * f + ol * g2;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float oo = __shfl_xor(r.o[e], o, 64);
            r.o[e] = (f > 0.0f ? r.o[e] * f : 0.0f) + (g2 > 0.0f ? oo * g2 : 0.0f);
        }
        r.m = mn;
    }
    return r;
}

__device__ __forceinline__ int lanes_per_key(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// Every head size and alignment: one wave per row and range.  Block (x, y, z): head, range, token.
template <class T, class C>
__global__ __launch_bounds__(kThreads) void attention_lanes_kernel(View v, AttnArgs a, int aligned) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x, split = blockIdx.y, head = blockIdx.z * 4 + w;
    const int seq = sequence_of(v, t, lane);
    if (seq >= v.c.batch || t < v.c.cu[seq] || head >= a.in.heads) return;
    const Span s = span_of(v, a, seq);
    const int begin = split * a.kps;
    if (begin >= s.total && split > 0) return;  // the first range of a sequence without rows writes zeros
    const int lpk = lanes_per_key(v.c.head_dim);
    const RowState r = scan_row<T, C>(v, a, s, t - s.first, head, begin, min(s.total, begin + a.kps), lane, lpk, aligned != 0);
    const int d0 = 8 * lane;
    if (a.splits == 1) {
        if (d0 >= v.c.head_dim) return;
        T* out = static_cast<T*>(a.in.out) + static_cast<int64_t>(t) * a.in.out_token + head * a.in.out_head;
        const float inv = r.l == 0.0f ? 0.0f : a.v_scale / r.l;
#pragma unroll
        for (int e = 0; e < 8; ++e) out[d0 + e] = static_cast<T>(r.l == 0.0f ? 0.0f : r.o[e] * inv);
    } else {
        const int64_t at = (static_cast<int64_t>(split) * a.in.tokens + t) * a.in.heads + head;
        if (lane == 0) a.part_ml[at] = float2{r.m, r.l};
        if (d0 < v.c.head_dim)
#pragma unroll
            for (int e = 0; e < 8; ++e) a.part_o[at * v.c.head_dim + d0 + e] = r.o[e];
    }
}

// Joins the ranges of each row in their order: D / 4 threads a row, 4 ranges requested at once.
// Block (x, y): token, heads.
template <class T>
__global__ __launch_bounds__(kThreads) void attention_merge_kernel(View v, AttnArgs a) {
    const int t = blockIdx.x, D = v.c.head_dim, per = D / 4, rows = kThreads / per;
    const int seq = sequence_of(v, t, threadIdx.x & 63);
    if (seq >= v.c.batch || t < v.c.cu[seq]) return;
    const Span s = span_of(v, a, seq);
    const int slot = threadIdx.x / per, d0 = 4 * (threadIdx.x % per), head = blockIdx.y * rows + slot;
    if (slot >= rows || head >= a.in.heads) return;
    const int n = max((s.total + a.kps - 1) / a.kps, 1);
    const int64_t row = static_cast<int64_t>(t) * a.in.heads + head, step = static_cast<int64_t>(a.in.tokens) * a.in.heads;
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < n; c0 += 4) {
        float2 ml[4];
        f32x4 po[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t at = row + min(c0 + i, n - 1) * step;
            ml[i] = a.part_ml[at];
            po[i] = *reinterpret_cast<const f32x4*>(a.part_o + at * D + d0);
            if (c0 + i >= n) ml[i] = float2{-INFINITY, 0.0f};
        }
        const float mn = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), m);
        const float f = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
        if (f > 0.0f) o *= f;
        else o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m = mn;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (ml[i].y == 0.0f) continue;  // a range of which the row sees nothing: its output may be unwritten
            const float w = ml[i].x == mn ? 1.0f : __builtin_amdgcn_exp2f(ml[i].x - mn);
            l += ml[i].y * w;
            if (!(w <= 0.0f)) o += po[i] * w;
        }
    }
    T h[4];
    const float inv = a.v_scale / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = static_cast<T>(l == 0.0f ? 0.0f : o[i] * inv);
    T* out = static_cast<T*>(a.in.out) + static_cast<int64_t>(t) * a.in.out_token + head * a.in.out_head + d0;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = h[i];
}

// ---- host side -------------------------------------------------------------------------------
struct Plan {
    int splits, kps;
    size_t o_bytes, bytes;
};

Plan plan(const View& v, const qmm_paged_query& in) {
    Plan p{};
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(static_cast<int64_t>(v.c.table_width) * v.c.page_size, INT32_MAX - 4096));
    const int64_t rows = static_cast<int64_t>(in.tokens) * in.heads;
    int64_t kps = 64;
    while (kps < most && (rows * ((most + kps - 1) / kps) > 16384 || (most + kps - 1) / kps > 1024)) kps *= 2;
    p.kps = static_cast<int>(kps);
    p.splits = static_cast<int>((most + kps - 1) / kps);
    if (p.splits > 1) {
        p.o_bytes = static_cast<size_t>(p.splits) * rows * v.c.head_dim * sizeof(float);
        p.bytes = p.o_bytes + static_cast<size_t>(p.splits) * rows * sizeof(float2);
    }
    return p;
}

int check_query(const qmm_paged_kv* kv, const qmm_paged_query* in, View* v) {
    const int rc = check_view(kv, true, v);
    if (rc != QMM_OK) return rc;
    if (!in) return bad("in must be non-null.");
    if (in->dtype != QMM_DTYPE_F16 && in->dtype != QMM_DTYPE_BF16) return bad("the queries' dtype must be F16 or BF16.");
    if (v->c.dtype != QMM_DTYPE_E4M3 && v->c.dtype != in->dtype) return bad("the cache must be E4M3 or of the queries' dtype.");
    if (in->heads <= 0 || in->heads % v->c.kv_heads != 0) return bad("heads must be divisible by kv_heads.");
    if (in->tokens < 0 || in->max_new < 0 || in->mask_words < 0) return bad("tokens, max_new and mask_words must be non-negative.");
    if (!std::isfinite(in->scale)) return bad("scale must be finite.");
    if (in->tokens > 0 && v->c.batch > 0 && (!in->q || !in->out)) return bad("q and out must be non-null.");
    if ((reinterpret_cast<uintptr_t>(in->q) | reinterpret_cast<uintptr_t>(in->out)) % 2 != 0) return bad("q and out must be aligned to their elements.");
    if (in->heads > 65535) return bad("too many heads.");
    return QMM_OK;
}

bool operands_aligned(const View& v, const qmm_paged_query& in) {
    const bool fp8 = v.c.dtype == QMM_DTYPE_E4M3;
    const uint64_t els = static_cast<uint64_t>(v.c.k_page | v.c.k_head | v.c.k_slot | v.c.v_page | v.c.v_head | v.c.v_slot);
    const uint64_t ptr = reinterpret_cast<uintptr_t>(v.c.k) | reinterpret_cast<uintptr_t>(v.c.v);
    return els % 8 == 0 && ptr % (fp8 ? 8 : 16) == 0;
}

int tree_attention(const qmm_paged_kv* kv, const qmm_paged_query* in, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    View v;
    const int rc = check_query(kv, in, &v);
    if (rc != QMM_OK) return rc;
    if (in->tokens == 0 || v.c.batch == 0 || in->max_new == 0) return QMM_OK;
    const Plan p = plan(v, *in);
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
    AttnArgs a{};
    a.in = *in;
    const float scale = in->scale != 0.0f ? in->scale : 1.0f / std::sqrt(static_cast<float>(v.c.head_dim));
    a.scale_log2 = scale * v.c.k_scale * 1.4426950408889634f;
    a.v_scale = v.c.v_scale;
    a.splits = p.splits;
    a.kps = p.kps;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + p.o_bytes);
    const int aligned = operands_aligned(v, *in) ? 1 : 0;
    const dim3 grid(static_cast<unsigned>(in->tokens), static_cast<unsigned>(p.splits), static_cast<unsigned>((in->heads + 3) / 4));
    auto go = [&](auto tc, auto cc) {
        using T = decltype(tc);
        using C = decltype(cc);
        hipLaunchKernelGGL((attention_lanes_kernel<T, C>), grid, dim3(kThreads), 0, stream, v, a, aligned);
    };
    const bool fp8 = v.c.dtype == QMM_DTYPE_E4M3;
    if (in->dtype == QMM_DTYPE_F16) fp8 ? go(_Float16{}, Fp8{}) : go(_Float16{}, _Float16{});
    else fp8 ? go(__bf16{}, Fp8{}) : go(__bf16{}, __bf16{});
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return launched(e, "paged attention kernel launch");
    if (p.splits > 1) {
        const int rows = kThreads / (v.c.head_dim / 4);
        const dim3 mgrid(static_cast<unsigned>(in->tokens), static_cast<unsigned>((in->heads + rows - 1) / rows));
        if (in->dtype == QMM_DTYPE_F16) hipLaunchKernelGGL(attention_merge_kernel<_Float16>, mgrid, dim3(kThreads), 0, stream, v, a);
        else hipLaunchKernelGGL(attention_merge_kernel<__bf16>, mgrid, dim3(kThreads), 0, stream, v, a);
        e = hipGetLastError();
    }
    return launched(e, "paged attention merge kernel launch");
}

}  // namespace
}  // namespace paged
}  // namespace qmm

extern "C" {

size_t qmm_paged_attention_workspace(const qmm_paged_kv* kv, const qmm_paged_query* in) {
    size_t bytes = 0;
    qmm::paged::entry([&] {
        qmm::paged::View v;
        const int rc = qmm::paged::check_query(kv, in, &v);
        if (rc == QMM_OK && in->tokens > 0) bytes = qmm::paged::plan(v, *in).bytes;
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
