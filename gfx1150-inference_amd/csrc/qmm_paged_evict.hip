// Eviction from a paged cache: for every layer, sequence and kv head the rows that have gathered the most attention stay, with the
// first and the last ones, and are copied in their order into fresh pages (the old ones may be shared with other
// sequences).
#include "qmm_paged.h"

#include <algorithm>
#include <type_traits>

namespace qmm {
namespace paged {
namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
static_assert(kSelectWaves == 16, "a row of lanes adds up the waves' counts");
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

// Block (x, y, z): kv head, sequence, layer.  The m-th largest weight of the rows in between is found from the top, two bits at a
// time, by counts of the weights at or above the three numbers that the bits so far begin; where a count is m, those are
// the rows.  Then the kept rows are listed in order, of those equal to the m-th largest the first ones.  Weights of up to
// kHeld 1024 rows wait in registers (a count is a comparison and a scalar population count for each 64 of them, with no atomics to
// meet on); of longer sequences (kHeld 0) they are read for each count.  Bound by the chain of counts: 256 workgroups of 3000 rows 14 us;
// 768 of up to 8192, of which two thirds choose, 44.
// A row without a page is no row: nothing of it could be copied, and its place in a fresh page would show what the page held before.
// Where fewer rows than `keep` have pages the sequence ends with them; past them only places without a fresh page, which show
// nothing either, count for rows without one.
template <int kHeld>
__global__ __launch_bounds__(kSelectThreads, kHeld <= 16 ? 8 : 4) void select_kernel(View v, EvictArgs a) {
    __shared__ int counts[2][4][kSelectWaves];  // [turn][number][wave]
    __shared__ int2 scan[kHeld ? kHeld : 1][kSelectWaves];
    __shared__ int none[2];  // rows without a page: of the first and last ones, of those in between
    const int g = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int keep = a.e.keep;
    const float* weights = a.e.weights + layer * a.e.w_layer + b * a.e.w_batch + g * a.e.w_head;
    float loaded[kHeld ? kHeld : 1];  // requested ahead of the sequence's length
    if constexpr (kHeld > 0)
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int j = i * kSelectThreads + tid;
            loaded[i] = j < a.e.rows ? weights[j] : -INFINITY;
        }
    const int n = table_rows(v, b);
    float* out = a.e.weights_out + layer * a.e.wo_layer + b * a.e.wo_batch + g * a.e.wo_head;
    const int32_t* fresh = a.e.fresh + b * a.e.fresh_stride;
    auto put_table = [&](int length) {
        if (g != 0 || layer != 0) return;
        const int pages = (length + v.c.page_size - 1) >> v.page_shift;
        for (int p = tid; p < v.c.table_width; p += kSelectThreads)
            a.e.table_out[static_cast<int64_t>(b) * v.c.table_width + p] = n <= keep ? v.c.table[b * v.c.table_stride + p] : p < pages ? fresh[p] : -1;
        if (tid == 0) a.e.lens_out[b] = length;
    };
    if (n <= keep) {
        put_table(n);
        for (int j = tid; j < a.e.rows; j += kSelectThreads) out[j] = j < n ? weights[j] : 0.0f;
        return;
    }
    const int first = a.e.sinks, last = n - a.e.recent, pages = ((n - 1) >> v.page_shift) + 1;
    bool misses = false;
    for (int p = tid; p < pages; p += kSelectThreads) misses |= page_of(v, b, p << v.page_shift) < 0;
    if (tid < 2) none[tid] = 0;
    const bool gap = __syncthreads_or(misses);
    int need = keep - a.e.sinks - a.e.recent, kept = keep, length = keep;  // rows to choose, rows that stay, the new length
    if (gap) {
        for (int p = tid; p < pages; p += kSelectThreads) {
            if (page_of(v, b, p << v.page_shift) >= 0) continue;
            const int from = p << v.page_shift, to = min(from + v.c.page_size, n), inner = max(min(to, last) - max(from, first), 0);
            atomicAdd(&none[0], to - from - inner);
            atomicAdd(&none[1], inner);
        }
        __syncthreads();
        const int ends = a.e.sinks + a.e.recent - none[0];
        need = min(keep - ends, last - first - none[1]);
        kept = ends + need;
        for (int p = kept >> v.page_shift; kept < keep && p <= (keep - 1) >> v.page_shift; ++p) {
            if (static_cast<uint32_t>(fresh[p]) >= static_cast<uint32_t>(v.c.num_pages)) continue;
            length = max(kept, p << v.page_shift);
            break;
        }
    }
    put_table(length);
    // Of a row in between its weight's, at least ordered(-inf).  Of the others, which no count meets, kAway where there is no page and
    // the row does not stay in any case, else 0.
    constexpr uint32_t kAway = 1;
    auto between = [&](int j) { return j >= first && j < last; };
    auto away = [&](int j) { return gap && j < n && page_of(v, b, j) < 0; };
    auto rank = [&](int j) { return away(j) ? (between(j) ? 0u : kAway) : between(j) ? ordered(j < a.e.rows ? weights[j] : -INFINITY) : 0u; };
    uint32_t held[kHeld ? kHeld : 1];
    if constexpr (kHeld > 0) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) held[i] = between(i * kSelectThreads + tid) ? ordered(loaded[i]) : 0u;
        if (gap)
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (const int j = i * kSelectThreads + tid; away(j)) held[i] = between(j) ? 0u : kAway;
    }
    for (int j = length + tid; j < a.e.rows; j += kSelectThreads) out[j] = 0.0f;
    uint32_t limit = 0;     // rows above it stay, and the first at_limit of those at it
    int above = 0;          // rows above
    if (need == 0) limit = 0xFFFFFFFFu;
    for (int bit = 30; bit >= 0 && need > 0; bit -= 2) {
        int count[3] = {0, 0, 0};
        auto add = [&](uint32_t r) {
#pragma unroll
            for (int c = 0; c < 3; ++c) count[c] += static_cast<int>(__popcll(__ballot(r >= (limit | static_cast<uint32_t>(c + 1) << bit))));
        };
        if constexpr (kHeld > 0) {
#pragma unroll
            for (int i = 0; i < kHeld; i += 4)
                if (i * kSelectThreads < last)
#pragma unroll
                    for (int k = 0; k < 4; ++k) add(held[i + k]);
        } else {
            for (int j0 = first; j0 < last; j0 += kSelectThreads) add(rank(j0 + tid));
        }
        if (lane < 3) counts[(bit >> 1) & 1][lane][w] = lane == 0 ? count[0] : lane == 1 ? count[1] : count[2];
        __syncthreads();
        // 16 lanes add up a number's counts (the last 16 read what is never written)
        int all = counts[(bit >> 1) & 1][lane / kSelectWaves][lane % kSelectWaves];
        auto fold = [&](auto ctrl) { all += __builtin_amdgcn_update_dpp(0, all, decltype(ctrl)::value, 0xF, 0xF, false); };
        fold(std::integral_constant<int, 0xB1>{});   // lane ^ 1
        fold(std::integral_constant<int, 0x4E>{});   // lane ^ 2
        fold(std::integral_constant<int, 0x141>{});  // the mirrored lane of 8
        fold(std::integral_constant<int, 0x140>{});  // .. and of 16
        const int total[3] = {__builtin_amdgcn_readlane(all, 0), __builtin_amdgcn_readlane(all, 16), __builtin_amdgcn_readlane(all, 32)};
        int most = 0;  // the largest two bits that leave enough
#pragma unroll
        for (int c = 0; c < 3; ++c) {
            if (total[c] >= need) most = c + 1;
        }
        if (most < 3) above = total[most];
        if (most > 0) limit |= static_cast<uint32_t>(most) << bit;
        if (most > 0 && total[most - 1] == need) {  // these are the rows
            --limit;
            above = need;
            break;
        }
    }
    const int at_limit = need - above;
    int32_t* list = a.list + ((static_cast<int64_t>(layer) * v.c.batch + b) * v.c.kv_heads + g) * keep;
    const uint64_t below = (uint64_t{1} << lane) - 1;
    auto stays = [&](int j, uint32_t r) { return j < n && (between(j) ? r > limit : r != kAway); };
    auto equal = [&](int j, uint32_t r) { return at_limit > 0 && r == limit && between(j); };
    auto put_at = [&](int place, int j) {
        list[place] = j;
        if (place < a.e.rows) out[place] = j < a.e.rows ? weights[j] : 0.0f;
    };
    auto put = [&](int j, uint64_t over, uint64_t same, int2 ahead) {
        const int o = ahead.x + static_cast<int>(__popcll(over & below)), e = ahead.y + static_cast<int>(__popcll(same & below));
        if (!((over >> lane) & 1) && !((same >> lane) & 1 && e < at_limit)) return;
        const int place = o + min(e, at_limit);
        if (place < kept) put_at(place, j);
    };
    auto number = [](uint64_t over, uint64_t same) { return int2{static_cast<int>(__popcll(over)), static_cast<int>(__popcll(same))}; };
    if constexpr (kHeld > 0) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int j = i * kSelectThreads + tid;
            const uint64_t over = __ballot(stays(j, held[i])), same = __ballot(equal(j, held[i]));
            if (lane == 0) scan[i][w] = number(over, same);
        }
        __syncthreads();
        if (w == 0) {  // what is ahead of every 64 rows
            int2 base{0, 0};
            for (int i0 = 0; i0 < kHeld * kSelectWaves; i0 += 64) {
                int2* at = &scan[0][0] + i0 + lane;
                const int2 x = i0 + lane < kHeld * kSelectWaves ? *at : int2{0, 0};
                int2 s = x;
                for (int o = 1; o < 64; o <<= 1) {
                    const int sx = __shfl_up(s.x, o, 64), sy = __shfl_up(s.y, o, 64);
                    if (lane >= o) s = int2{s.x + sx, s.y + sy};
                }
                if (i0 + lane < kHeld * kSelectWaves) *at = int2{base.x + s.x - x.x, base.y + s.y - x.y};
                base = int2{base.x + __shfl(s.x, 63, 64), base.y + __shfl(s.y, 63, 64)};
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int j = i * kSelectThreads + tid;
            if (i * kSelectThreads < n) put(j, __ballot(stays(j, held[i])), __ballot(equal(j, held[i])), scan[i][w]);
        }
    } else {
        int2 ahead{0, 0};
        for (int j0 = 0; j0 < n; j0 += kSelectThreads) {
            const int j = j0 + tid;
            const uint32_t r = rank(j);
            const uint64_t over = __ballot(stays(j, r)), same = __ballot(equal(j, r));
            if (lane == 0) scan[0][w] = number(over, same);
            __syncthreads();
            int2 mine = ahead;
            for (int i = 0; i < kSelectWaves; ++i) {
                const int2 x = scan[0][i];
                if (i < w) mine = int2{mine.x + x.x, mine.y + x.y};
                ahead = int2{ahead.x + x.x, ahead.y + x.y};
            }
            put(j, over, same, mine);
            __syncthreads();
        }
    }
    if (length == kept) return;
    for (int j = tid; j < n; j += kSelectThreads) {
        if (!away(j)) continue;
        int place = kept + (j & (v.c.page_size - 1));
        for (int p = 0; p < j >> v.page_shift; ++p) place += page_of(v, b, p << v.page_shift) < 0 ? v.c.page_size : 0;
        if (place < length) put_at(place, j);
    }
}

// Copies the kept rows.  Block (x, y, z): a run of rows, sequence and kv head, layer; a thread keeps its piece of a row and takes every
// (kThreads / per_row)-th row, kRowsAtOnce of K and of V at once.  At the rate of a copy: 1.45 GB read and written in 289 us, 5.0 TB/s (297 where the rows stay in the
// caches).
constexpr int kRowsAtOnce = 4;

template <int B>
__global__ __launch_bounds__(kThreads) void gather_kernel(View v, Strides st, EvictArgs a, int rows_each) {
    using U = typename Unit<B>::type;
    const int b = blockIdx.y / v.c.kv_heads, g = blockIdx.y % v.c.kv_heads, layer = blockIdx.z, keep = a.e.keep;
    const int length = a.e.lens_out[b];  // `keep`, or less where rows have no page
    if (table_rows(v, b) <= keep) return;
    const int abreast = max(kThreads / st.per_row, 1), sub = static_cast<int>(threadIdx.x) / st.per_row;
    if (sub >= abreast) return;
    const int32_t* list = a.list + ((static_cast<int64_t>(layer) * v.c.batch + b) * v.c.kv_heads + g) * keep;
    const int32_t* fresh = a.e.fresh + b * a.e.fresh_stride;
    U* k = static_cast<U*>(v.c.k) + layer * st.k_layer + g * st.k_head;
    U* x = static_cast<U*>(v.c.v) + layer * st.v_layer + g * st.v_head;
    const int begin = blockIdx.x * rows_each, end = min(begin + min(rows_each, keep - begin), length);
    if (begin >= end) return;
    for (int piece = static_cast<int>(threadIdx.x) % st.per_row; piece < st.per_row; piece += kThreads) {
        for (int row = begin + sub; row < end; row += kRowsAtOnce * abreast) {
            U rk[kRowsAtOnce], rv[kRowsAtOnce];
            int page[kRowsAtOnce], from[kRowsAtOnce], target[kRowsAtOnce];
#pragma unroll
            for (int i = 0; i < kRowsAtOnce; ++i) from[i] = list[min(row + i * abreast, end - 1)];
#pragma unroll
            for (int i = 0; i < kRowsAtOnce; ++i) {
                const int to = min(row + i * abreast, end - 1);
                page[i] = page_of(v, b, from[i]);
                target[i] = fresh[to >> v.page_shift];
                if (row + i * abreast >= end || static_cast<uint32_t>(target[i]) >= static_cast<uint32_t>(v.c.num_pages)) page[i] = -1;
            }
#pragma unroll
            for (int i = 0; i < kRowsAtOnce; ++i) {
                if (page[i] < 0) continue;
                const int slot = from[i] & (v.c.page_size - 1);
                rk[i] = __builtin_nontemporal_load(k + page[i] * st.k_page + slot * st.k_slot + piece);
                rv[i] = __builtin_nontemporal_load(x + page[i] * st.v_page + slot * st.v_slot + piece);
            }
#pragma unroll
            for (int i = 0; i < kRowsAtOnce; ++i) {
                if (page[i] < 0) continue;
                const int slot = (row + i * abreast) & (v.c.page_size - 1);
                __builtin_nontemporal_store(rk[i], k + target[i] * st.k_page + slot * st.k_slot + piece);
                __builtin_nontemporal_store(rv[i], x + target[i] * st.v_page + slot * st.v_slot + piece);
            }
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
    if (e->rows > 0 && !apart({{v->c.kv_heads, e->wo_head}, {v->c.batch, e->wo_batch}, {v->c.num_layers, e->wo_layer}}, e->rows))
        return bad("weights_out must not overlap itself.");
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
    auto select = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kSelectThreads), 0, stream, v, a); };
    const int64_t room = static_cast<int64_t>(v.c.table_width) * v.c.page_size;  // of a sequence
    if (room <= 4 * kSelectThreads) select(select_kernel<4>);
    else if (room <= 8 * kSelectThreads) select(select_kernel<8>);
    else if (room <= 16 * kSelectThreads) select(select_kernel<16>);
    else if (room <= 32 * kSelectThreads) select(select_kernel<32>);
    else select(select_kernel<0>);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return launched(err, "paged evict kernel launch");
    Strides st;
    const int unit = copy_unit(v.c, &st);
    const int rows_each = std::max(kThreads / st.per_row, 1) * kRowsAtOnce;
    const dim3 rows(static_cast<unsigned>((e->keep + static_cast<int64_t>(rows_each) - 1) / rows_each), static_cast<unsigned>(v.c.batch * v.c.kv_heads),
                    static_cast<unsigned>(v.c.num_layers));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, rows, dim3(kThreads), 0, stream, v, st, a, rows_each); };
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
