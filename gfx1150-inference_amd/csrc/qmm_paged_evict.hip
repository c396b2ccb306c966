// Eviction from a paged cache: for every layer, sequence and kv head the rows that have gathered the most attention stay, with the
// first and the last ones, and are copied in their order into fresh pages (the old ones may be shared with other
// sequences).
#include "qmm_paged.h"

#include <algorithm>

namespace qmm {
namespace paged {
namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kThreads = 256;

struct EvictArgs {
    qmm_paged_evict_args e;
    int32_t* list;  // [layer][sequence][kv head][keep]: the kept rows, ascending
};

// Rows of a sequence that its table has places for.
__device__ __forceinline__ int table_rows(const View& v, int seq) {
    return static_cast<int>(min(static_cast<int64_t>(cached_rows(v, seq)), static_cast<int64_t>(v.c.table_width) << v.page_shift));
}

// The order of the weights as that of unsigned numbers: -0 as 0, NaN as -inf.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = x != x ? 0xFF800000u : x == 0.0f ? 0u : __float_as_uint(x);
    return b >> 31 ? ~b : b | 0x80000000u;
}

// Block (x, y, z): kv head, sequence, layer.  The m-th largest weight of the rows in between is found bit by bit from the
// top, each bit by a count of the weights at or above the number so far with the bit set; then the kept rows are
// listed in order, those equal to it as far as there is room.
__global__ __launch_bounds__(kSelectThreads) void select_kernel(View v, EvictArgs a) {
    __shared__ int counts[2][kSelectWaves];
    __shared__ int2 scan[kSelectWaves];
    const int g = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = table_rows(v, b), keep = a.e.keep;
    const float* weights = a.e.weights + layer * a.e.w_layer + b * a.e.w_batch + g * a.e.w_head;
    float* out = a.e.weights_out + layer * a.e.wo_layer + b * a.e.wo_batch + g * a.e.wo_head;
    if (g == 0 && layer == 0) {
        const int pages = (keep + v.c.page_size - 1) >> v.page_shift;
        for (int p = tid; p < v.c.table_width; p += kSelectThreads)
            a.e.table_out[static_cast<int64_t>(b) * v.c.table_width + p] = n <= keep ? v.c.table[b * v.c.table_stride + p]
                                                                           : p < pages ? a.e.fresh[b * a.e.fresh_stride + p] : -1;
        if (tid == 0) a.e.lens_out[b] = min(n, keep);
    }
    if (n <= keep) {
        for (int j = tid; j < a.e.rows; j += kSelectThreads) out[j] = j < n ? weights[j] : 0.0f;
        return;
    }
    for (int j = keep + tid; j < a.e.rows; j += kSelectThreads) out[j] = 0.0f;
    const int first = a.e.sinks, last = n - a.e.recent, need = keep - a.e.sinks - a.e.recent;
    auto rank = [&](int j) { return ordered(j < a.e.rows ? weights[j] : -INFINITY); };
    uint32_t limit = 0;
    int above = 0;  // weights above the limit
    if (need > 0) {
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t probe = limit | (1u << bit);
            int count = 0;
            for (int j0 = first; j0 < last; j0 += kSelectThreads) {
                const int j = j0 + tid;
                count += static_cast<int>(__popcll(__ballot(j < last && rank(j) >= probe)));
            }
            if (lane == 0) counts[bit & 1][w] = count;
            __syncthreads();
            int total = 0;
            for (int i = 0; i < kSelectWaves; ++i) total += counts[bit & 1][i];
            if (total >= need) limit = probe;
            else above = total;
        }
    }
    // kept rows of a step of 1024: those above the limit, and the first of those at it
    int32_t* list = a.list + ((static_cast<int64_t>(layer) * v.c.batch + b) * v.c.kv_heads + g) * keep;
    const int at_limit = need - above;
    int taken = 0, equal = 0;
    for (int j0 = 0; j0 < n; j0 += kSelectThreads) {
        const int j = j0 + tid;
        const bool outer = j < n && (j < first || j >= last);
        const uint32_t r = j < n && !outer ? rank(j) : 0;
        const bool inner = j < n && !outer && need > 0;
        const uint64_t below = (uint64_t{1} << lane) - 1;
        const uint64_t over = __ballot(outer || (inner && r > limit)), same = __ballot(inner && r == limit);
        if (lane == 0) scan[w] = int2{static_cast<int>(__popcll(over)), static_cast<int>(__popcll(same))};
        __syncthreads();
        int o = taken, e = equal;
        for (int i = 0; i < kSelectWaves; ++i) {
            if (i < w) {
                o += scan[i].x;
                e += scan[i].y;
            }
            taken += scan[i].x;
            equal += scan[i].y;
        }
        e += static_cast<int>(__popcll(same & below));
        o += static_cast<int>(__popcll(over & below));
        const bool keeps = (over >> lane) & 1 || ((same >> lane) & 1 && e < at_limit);
        const int place = o + min(e, at_limit);
        if (keeps && place < keep) {
            list[place] = j;
            if (place < a.e.rows) out[place] = j < a.e.rows ? weights[j] : 0.0f;
        }
        __syncthreads();
    }
}

// Copies the kept rows.  Block (x, y, z): 256 units of (row, piece) a pass, sequence and kv head, layer.
constexpr int kRowsAtOnce = 4;  // of K and of V, per thread

template <int B>
__global__ __launch_bounds__(kThreads) void gather_kernel(View v, Strides st, EvictArgs a) {
    using U = typename Unit<B>::type;
    const int b = blockIdx.y / v.c.kv_heads, g = blockIdx.y % v.c.kv_heads, layer = blockIdx.z, keep = a.e.keep;
    if (table_rows(v, b) <= keep) return;
    const int32_t* list = a.list + ((static_cast<int64_t>(layer) * v.c.batch + b) * v.c.kv_heads + g) * keep;
    U* k = static_cast<U*>(v.c.k) + layer * st.k_layer + g * st.k_head;
    U* x = static_cast<U*>(v.c.v) + layer * st.v_layer + g * st.v_head;
    const int64_t total = static_cast<int64_t>(keep) * st.per_row, step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; at < total; at += kRowsAtOnce * step) {
        U rk[kRowsAtOnce], rv[kRowsAtOnce];
        int64_t to_k[kRowsAtOnce], to_v[kRowsAtOnce];
#pragma unroll
        for (int i = 0; i < kRowsAtOnce; ++i) {
            const int64_t u = at + i * step;
            to_k[i] = -1;
            if (u >= total) continue;
            const int row = static_cast<int>(u / st.per_row), piece = static_cast<int>(u % st.per_row);
            const int from = list[row], page = page_of(v, b, from), slot = from & (v.c.page_size - 1);
            const int target = a.e.fresh[b * a.e.fresh_stride + (row >> v.page_shift)], to = row & (v.c.page_size - 1);
            if (page < 0 || static_cast<uint32_t>(target) >= static_cast<uint32_t>(v.c.num_pages)) continue;
            rk[i] = k[page * st.k_page + slot * st.k_slot + piece];
            rv[i] = x[page * st.v_page + slot * st.v_slot + piece];
            to_k[i] = target * st.k_page + to * st.k_slot + piece;
            to_v[i] = target * st.v_page + to * st.v_slot + piece;
        }
#pragma unroll
        for (int i = 0; i < kRowsAtOnce; ++i) {
            if (to_k[i] < 0) continue;
            k[to_k[i]] = rk[i];
            x[to_v[i]] = rv[i];
        }
    }
}

size_t list_bytes(const View& v, const qmm_paged_evict_args& e) {
    return (static_cast<size_t>(v.c.num_layers) * v.c.batch * v.c.kv_heads * e.keep * sizeof(int32_t) + 15) / 16 * 16;
}

int check_evict(const qmm_paged_kv* kv, const qmm_paged_evict_args* e, View* v) {
    const int rc = check_view(kv, false, v);
    if (rc != QMM_OK) return rc;
    if (!e) return bad("args must be non-null.");
    if (e->keep < 1) return bad("keep must be positive.");
    if (e->recent < 0 || e->sinks < 0 || static_cast<int64_t>(e->recent) + e->sinks > e->keep) return bad("recent and sinks must be non-negative, keep at least their sum.");
    if (e->rows < 0) return bad("rows must be non-negative.");
    if (e->fresh_width < 0 || static_cast<int64_t>(e->fresh_width) * v->c.page_size < e->keep) return bad("the fresh pages must have places for keep rows.");
    if (v->c.batch > 0 && (!e->fresh || !e->lens_out || (v->c.table_width > 0 && !e->table_out) || (e->rows > 0 && (!e->weights || !e->weights_out))))
        return bad("weights, weights_out, fresh, table_out and lens_out must be non-null.");
    if ((reinterpret_cast<uintptr_t>(e->weights) | reinterpret_cast<uintptr_t>(e->weights_out)) % 4 != 0) return bad("weights must be aligned to their elements.");
    if (v->c.batch > 0 && (e->weights_out == e->weights && e->rows > 0)) return bad("weights_out must not be weights.");
    if (v->c.batch > 0 && (e->table_out == v->c.table || e->lens_out == v->c.ctx)) return bad("table_out and lens_out must not be the inputs.");
    if (v->c.kv_heads > 65535 || v->c.num_layers > 65535 || static_cast<int64_t>(v->c.batch) * v->c.kv_heads > 65535) return bad("too many layers, sequences and heads.");
    return QMM_OK;
}

int evict(const qmm_paged_kv* kv, const qmm_paged_evict_args* e, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    View v;
    const int rc = check_evict(kv, e, &v);
    if (rc != QMM_OK || v.c.batch == 0) return rc;
    const size_t need = list_bytes(v, *e);
    std::unique_lock<std::mutex> held;  // until the last launch is enqueued
    if (workspace) {
        if (workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return bad("the workspace must be 16-byte aligned and hold qmm_paged_evict_workspace() bytes.");
    } else {
        const hipError_t err = take_workspace(WorkspaceKind::kAttention, stream, need, held, &workspace);
        if (err != hipSuccess) return launched(err, "paged evict workspace");
    }
    const EvictArgs a{*e, static_cast<int32_t*>(workspace)};
    const dim3 grid(static_cast<unsigned>(v.c.kv_heads), static_cast<unsigned>(v.c.batch), static_cast<unsigned>(v.c.num_layers));
    hipLaunchKernelGGL(select_kernel, grid, dim3(kSelectThreads), 0, stream, v, a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return launched(err, "paged evict kernel launch");
    Strides st;
    const int unit = copy_unit(v.c, &st);
    const int64_t units = static_cast<int64_t>(e->keep) * st.per_row, each = kThreads * kRowsAtOnce;
    const dim3 rows(static_cast<unsigned>(std::min<int64_t>((units + each - 1) / each, 1 << 20)), static_cast<unsigned>(v.c.batch * v.c.kv_heads),
                    static_cast<unsigned>(v.c.num_layers));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, rows, dim3(kThreads), 0, stream, v, st, a); };
    unit == 16 ? go(gather_kernel<16>) : unit == 4 ? go(gather_kernel<4>) : go(gather_kernel<1>);
    return launched(hipGetLastError(), "paged evict kernel launch");
}

}  // namespace
}  // namespace paged
}  // namespace qmm

extern "C" {

size_t qmm_paged_evict_workspace(const qmm_paged_kv* kv, const qmm_paged_evict_args* args) {
    size_t bytes = 0;
    qmm::paged::entry([&] {
        qmm::paged::View v;
        const int rc = qmm::paged::check_evict(kv, args, &v);
        if (rc == QMM_OK && v.c.batch > 0) bytes = qmm::paged::list_bytes(v, *args);
        return rc;
    });
    return bytes;
}

int qmm_paged_evict(const qmm_paged_kv* kv, const qmm_paged_evict_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    return qmm::paged::entry([&] { return qmm::paged::evict(kv, args, workspace, workspace_bytes, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
