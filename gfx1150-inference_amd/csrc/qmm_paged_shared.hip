// Attention of a batch whose groups of sequences begin with the same rows (a system prompt, a document, the prompt of
// a beam search): the group's tokens attend to the shared rows together, as the new tokens of one sequence that has
// these rows, and every token to the rest of its own sequence's; the partial rows of both, each with its maximum and sum,
// are joined as those of any two ranges are,
//   m = max(m1, m2),  out = (2^(m1 - m) o1 + 2^(m2 - m) o2) / (2^(m1 - m) l1 + 2^(m2 - m) l2).
// Shared rows meet many queries and are bound by the matrix cores (64 tokens of 64 heads behind 16384 rows, 34 GFLOP: 47 us), a
// sequence's own by their reading (197 MB: 40 us).
#include "qmm_paged_attention.h"

namespace qmm {
namespace paged {
namespace {

// How a part is cut; the rest of it is as CallPlan says.
struct CutArgs {
    int tile_shift, step_shift, min_steps;  // rows of a row tile (-1: one for all), keys of a step; the least steps of a range
    int slots;                  // workgroups that run at once
    PartSeq* seqs;
    int32_t* first_block;
};

struct Groups {
    const int32_t *first, *shared;
    int count;
    int32_t *starts, *ctx;  // [count + 1], [count], for more groups than fit LDS
    CutArgs lead, rest;
};

constexpr int kPlanThreads = 256, kPlanWaves = kPlanThreads / 64, kTries = 4;

// One workgroup cuts the call: where groups begin (made ascending, so that no sequence is in two), the rows that a group shares (no
// more than any of its sequences has cached, whole blocks of 16, which lie in one page; none where it has one sequence), and
// for both parts, by the rules of CallPlan, the ranges of every sequence and the workgroups ahead of it.  The attention's
// workgroups look theirs up: worked out by each of them, the cut of 128 sequences took most of the time of short contexts.
__global__ __launch_bounds__(kPlanThreads) void cut_kernel(View v, qmm_paged_query in, Groups g) {
    __shared__ int starts_lds[kPlanThreads], ctx_lds[kPlanThreads], shared_lds[kPlanThreads], cu_lds[kPlanThreads];
    __shared__ float sums[2 * kTries][kPlanWaves];
    __shared__ int4 scans[kPlanWaves];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, batch = v.c.batch, group = in.heads / v.c.kv_heads, kvh = v.c.kv_heads;
    int* starts = g.count < kPlanThreads ? starts_lds : g.starts;
    int* ctx = g.count < kPlanThreads ? ctx_lds : g.ctx;
    // what a thread's sequence and group have, requested together: one round trip where there are no more of them than threads
    const bool small = batch < kPlanThreads && g.count < kPlanThreads;
    int own_ctx = 0;
    if (small) {
        const int first = tid <= g.count ? g.first[tid] : 0, shared = tid < g.count ? g.shared[tid] : 0, cu = tid <= batch ? v.c.cu[tid] : 0;
        if (tid < batch) own_ctx = cached_rows(v, tid);
        starts_lds[tid] = first;
        shared_lds[tid] = shared;
        cu_lds[tid] = cu;
        __syncthreads();
    }
    auto ctx_of = [&](int b) { return small ? own_ctx : cached_rows(v, b); };  // of the thread's own sequence
    auto cu_of = [&](int b) { return small ? cu_lds[b] : v.c.cu[b]; };
    if (w == 0) {
        int most = 0;
        for (int i0 = 0; i0 <= g.count; i0 += 64) {
            const int i = i0 + tid;
            int x = i <= g.count ? min(max(small ? starts_lds[i] : g.first[i], 0), batch) : 0;
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(x, o, 64);
                if (tid >= o) x = max(x, y);
            }
            x = max(x, most);
            most = __shfl(x, 63, 64);
            if (i <= g.count) starts[i] = x;
        }
    }
    __syncthreads();
    const int64_t room = static_cast<int64_t>(v.c.table_width) << v.page_shift;
    for (int i = tid; i < g.count; i += kPlanThreads)
        ctx[i] = starts[i + 1] - starts[i] > 1 ? static_cast<int>(min(static_cast<int64_t>(max(small ? shared_lds[i] : g.shared[i], 0)), room)) : 0;
    __syncthreads();
    // the group of a sequence: the count of starts at or below it, less one
    auto group_of = [&](int b) {
        int lo = 0, hi = g.count + 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (starts[mid] <= b) lo = mid + 1;
            else hi = mid;
        }
        return lo - 1 < g.count ? lo - 1 : -1;
    };
    int own_group = -1;
    for (int b = tid; b < batch; b += kPlanThreads) {
        own_group = group_of(b);
        if (own_group >= 0) atomicMin(&ctx[own_group], ctx_of(b));
    }
    __syncthreads();

    // rows that group i shares; past the caches, which may hold what an entry was before the minima
    auto shared_of = [&](int i) { return __hip_atomic_load(&ctx[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & ~15; };
    struct Own {
        PartSeq s;
        int steps;
        float work;
    };
    auto token = [&](int b) { return min(max(cu_of(b), 0), in.tokens); };
    // sequence b of the rest, group b of what is shared
    auto own_of = [&](const CutArgs& c, bool lead, int b) {
        Own x{};
        PartSeq& s = x.s;
        if (b >= (lead ? g.count : batch)) return x;
        if (lead) {
            s.table_row = min(starts[b], batch - 1);
            s.first = token(starts[b]);
            s.n = max(token(starts[b + 1]) - s.first, 0);
            s.total = s.ctx = shared_of(b);
            s.rows = s.ctx > 0 ? s.n : 0;
        } else {
            const int i = small ? own_group : group_of(b);
            s.table_row = b;
            s.first = max(cu_of(b), 0);
            s.n = max(token(b + 1) - s.first, 0);
            s.ctx = ctx_of(b);
            s.total = static_cast<int>(min(static_cast<int64_t>(s.ctx) + s.n, room));
            s.from = i >= 0 ? shared_of(i) : 0;
            s.rows = min(s.n, in.max_new);
        }
        s.tiles = c.tile_shift < 0 ? s.rows > 0 : static_cast<int>((static_cast<int64_t>(s.rows) * group + (1 << c.tile_shift) - 1) >> c.tile_shift);
        auto steps = [&](int keys) { return (max(keys - 1, 0) >> c.step_shift) + 1; };
        x.steps = s.rows > 0 ? steps(s.total - s.from) : 0;
        const int seen = (lead || in.mask ? s.total : min(s.total, s.ctx + (s.n + 1) / 2)) - s.from;
        x.work = static_cast<float>(steps(seen)) * static_cast<float>(s.tiles);
        return x;
    };
    const int chunks = (max(batch, g.count) + kPlanThreads - 1) / kPlanThreads;
    auto total_of = [&](int row) {
        float x = lane < kPlanWaves ? sums[row][lane] : 0.0f;
        return wave_total(x);
    };
    Own rest{}, lead{};
    double work[2] = {0.0, 0.0};
    for (int c = 0; c < chunks; ++c) {
        rest = own_of(g.rest, false, c * kPlanThreads + tid);
        lead = own_of(g.lead, true, c * kPlanThreads + tid);
        work[0] += static_cast<double>(rest.work);
        work[1] += static_cast<double>(lead.work);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float x = wave_total(static_cast<float>(work[k]));
        if (lane == 0) sums[k][w] = x;
    }
    __syncthreads();
    int u[2][kTries];
    float count[2 * kTries];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const CutArgs& c = k ? g.lead : g.rest;
        const float shortest = total_of(k) * static_cast<float>(kvh) / static_cast<float>(c.slots) * 1.00001f;  // as in CallPlan
#pragma unroll
        for (int t = 0; t < kTries; ++t) {
            u[k][t] = max(static_cast<int>(fminf(ceilf(shortest * (1.0f + 0.25f * static_cast<float>(t))), 33554432.0f)), c.min_steps);
            count[kTries * k + t] = 0.0f;
        }
    }
    auto ranges_of = [](int steps, int len) { return static_cast<int>((static_cast<uint32_t>(steps) + len - 1) / static_cast<uint32_t>(len)); };
    for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) {
            rest = own_of(g.rest, false, c * kPlanThreads + tid);
            lead = own_of(g.lead, true, c * kPlanThreads + tid);
        }
#pragma unroll
        for (int t = 0; t < kTries; ++t) {
            count[t] += wave_total(static_cast<float>(ranges_of(rest.steps, u[0][t])) * static_cast<float>(rest.s.tiles));
            count[kTries + t] += wave_total(static_cast<float>(ranges_of(lead.steps, u[1][t])) * static_cast<float>(lead.s.tiles));
        }
    }
    __syncthreads();  // sums have been read
    if (lane == 0)
#pragma unroll
        for (int t = 0; t < 2 * kTries; ++t) sums[t][w] = count[t];
    __syncthreads();
    int best[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        best[k] = u[k][0];
#pragma unroll
        for (int t = kTries - 1; t >= 0; --t)
            if (total_of(kTries * k + t) * static_cast<float>(kvh) <= static_cast<float>(k ? g.lead.slots : g.rest.slots)) best[k] = u[k][t];
    }
    int4 before{0, 0, 0, 0};  // blocks and partial rows (in tokens) of the rest, and of what is shared
    for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) {
            rest = own_of(g.rest, false, c * kPlanThreads + tid);
            lead = own_of(g.lead, true, c * kPlanThreads + tid);
        }
        rest.s.ranges = ranges_of(rest.steps, best[0]);
        lead.s.ranges = ranges_of(lead.steps, best[1]);
        const int4 own{rest.s.ranges * rest.s.tiles * kvh, rest.s.ranges * rest.s.rows, lead.s.ranges * lead.s.tiles * kvh, lead.s.ranges * lead.s.rows};
        const int4 upto{wave_scan(own.x), wave_scan(own.y), wave_scan(own.z), wave_scan(own.w)};
        if (lane == 63) scans[w] = upto;
        __syncthreads();
        int4 ahead = before;
        for (int i = 0; i < kPlanWaves; ++i) {
            const int4 x = scans[i];
            if (i < w) ahead = int4{ahead.x + x.x, ahead.y + x.y, ahead.z + x.z, ahead.w + x.w};
            before = int4{before.x + x.x, before.y + x.y, before.z + x.z, before.w + x.w};
        }
        __syncthreads();
        auto put = [&](const CutArgs& a, Own& x, int b, int n, int block, int part) {
            if (b >= n) return;
            x.s.keys = x.s.ranges > 0 ? static_cast<int>((static_cast<uint32_t>(x.steps) + x.s.ranges - 1) / static_cast<uint32_t>(x.s.ranges)) << a.step_shift : 0;
            x.s.first_part = part;
            a.seqs[b] = x.s;
            a.first_block[b] = block;
        };
        const int b = c * kPlanThreads + tid;
        put(g.rest, rest, b, batch, ahead.x + upto.x - own.x, ahead.y + upto.y - own.y);
        put(g.lead, lead, b, g.count, ahead.z + upto.z - own.z, ahead.w + upto.w - own.w);
    }
    if (tid == 0) {
        g.rest.first_block[batch] = before.x;
        g.lead.first_block[g.count] = before.z;
    }
}

// Both parts in one launch, what is shared first, as it takes the longest.  Where tiles of 128 rows serve it and few rows each the
// others, these have fewer workgroups at once in it than in a launch of their own, so large calls of that kind have two
// (kOneLaunch).
struct LeadArgs {
    const PartSeq* seqs;
    const int32_t* first_block;
    int count, blocks;  // of groups, of workgroups
    int64_t parts;
    int4* cut;
};

__device__ __forceinline__ AttnArgs lead_args(const View& v, const AttnArgs& a, const LeadArgs& l) {
    AttnArgs b = a;
    b.in.mask = nullptr;
    b.in.mask_words = 0;
    b.part_o = a.part_o + a.parts * a.in.heads * v.c.head_dim;
    b.part_ml = a.part_ml + a.parts * a.in.heads;
    b.parts = l.parts;
    b.cut = l.cut;
    b.seqs = l.seqs;
    b.first_block = l.first_block;
    b.n_seqs = l.count;
    return b;
}

// kLeadTile, kRestTile: which kernel's workgroups serve the parts.  The first l.blocks are the shared rows', the others the rest's.
template <class T, class C, int D, bool kLeadTile, bool kRestTile, int NT, int RG>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void attention_shared_kernel(View v, AttnArgs a, LeadArgs l) {
    const bool is_lead = static_cast<int>(blockIdx.x) < l.blocks;
    const AttnArgs b = is_lead ? lead_args(v, a, l) : a;
    const int block = static_cast<int>(blockIdx.x) - (is_lead ? 0 : l.blocks);
    auto& rows_lds = *reinterpret_cast<RowsLds<D, Part>*>(tile_lds);
    if constexpr (kLeadTile && kRestTile) {
        attend_tile<T, C, D, Part>(v, b, block);
    } else if constexpr (!kLeadTile) {
        attend_rows<T, C, D, NT, RG, Part>(v, b, block, rows_lds);
    } else {
        if (is_lead) attend_tile<T, C, D, Part>(v, b, block);
        else attend_rows<T, C, D, NT, RG, Part>(v, b, block, rows_lds);
    }
}

template <class T, class C, int D, class Fn>
auto with_shared_kernel(Kind lead, Kind rest, int row_tiles, Fn f) {
    constexpr size_t rows = sizeof(RowsLds<D, Part>), tile = TileGeom<D>::kLds, both = rows > tile ? rows : tile;
    if (rest == Kind::kTile) return f(attention_shared_kernel<T, C, D, true, true, 1, 1>, tile);
    auto few = [&](auto lead_tile, size_t lds) {
        constexpr bool L = decltype(lead_tile)::value;
        if constexpr (D <= 128) {
            if (row_tiles == 2) return f(attention_shared_kernel<T, C, D, L, false, 2, 1>, lds);
            if (row_tiles > 2) return f(attention_shared_kernel<T, C, D, L, false, 2, 2>, lds);
        }
        return f(attention_shared_kernel<T, C, D, L, false, 1, 1>, lds);
    };
    return lead == Kind::kTile ? few(std::true_type{}, both) : few(std::false_type{}, rows);
}

// Calls f with the kernel of both parts' kinds and its LDS.
template <class Fn>
auto with_shared_kernel(const View& v, const qmm_paged_query& in, Kind lead, Kind rest, int row_tiles, Fn f) {
    auto types = [&](auto tc, auto cc) {
        using T = decltype(tc);
        using C = decltype(cc);
        switch (v.c.head_dim) {
            case 64: return with_shared_kernel<T, C, 64>(lead, rest, row_tiles, f);
            case 96: return with_shared_kernel<T, C, 96>(lead, rest, row_tiles, f);
            case 128: return with_shared_kernel<T, C, 128>(lead, rest, row_tiles, f);
            default: return with_shared_kernel<T, C, 256>(lead, rest, row_tiles, f);
        }
    };
    const bool fp8 = v.c.dtype == QMM_DTYPE_E4M3;
    if (in.dtype == QMM_DTYPE_F16) return fp8 ? types(_Float16{}, Fp8{}) : types(_Float16{}, _Float16{});
    return fp8 ? types(__bf16{}, Fp8{}) : types(__bf16{}, __bf16{});
}

// Products of queries and keys, by the table's width, up to which parts of different kinds go in one launch (16 x 8 beams behind
// 1000 rows of 32 heads, 4e6: 46 us with two launches, 42 with one; 45 sequences behind 585 rows of 16 heads, 6e5: 34 and 26; the
// attention alone of 64 sequences of 64 heads behind 16384, 7e7: 93 and 103).
constexpr int64_t kOneLaunch = int64_t{3} << 23;

struct SharedPlan {
    Plan lead, rest;
    bool one;                                  // launch
    int row_tiles;                             // of both, where both are of rows
    size_t seqs, first, cut, ml, o, bytes;     // where the workspace's parts begin
    int64_t parts;                             // in rows
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

SharedPlan shared_plan(const View& v, const qmm_paged_query& in, const qmm_paged_groups& g) {
    SharedPlan p{};
    View u = v;
    u.c.batch = g.count;
    qmm_paged_query q = in;
    q.max_new = in.tokens;  // of a group
    // each part has the kernel that it would have by itself; a group has at least a sequence's rows
    p.row_tiles = part_kind(u, q) == Kind::kRows ? row_tiles_of(u, q) : row_tiles_of(v, in);
    const Kind lead = part_kind(u, q), rest = part_kind(v, in);
    p.one = lead == rest || static_cast<int64_t>(in.tokens) * in.heads * v.c.table_width <= kOneLaunch / v.c.page_size;
    auto slots = [&](Kind l, Kind r) { return with_shared_kernel(v, in, l, r, p.row_tiles, [](auto kern, size_t lds) { return kernel_slots(kern, lds); }); };
    p.rest = plan<Part>(v, in, p.one ? slots(lead, rest) : slots(rest, rest));
    p.lead = plan<Part>(u, q, p.one ? slots(lead, rest) : slots(lead, lead));
    p.parts = p.rest.parts + p.lead.parts;
    p.seqs = whole((2 * static_cast<size_t>(g.count) + 1) * sizeof(int32_t));
    p.first = p.seqs + (static_cast<size_t>(g.count) + v.c.batch) * sizeof(PartSeq);
    p.cut = p.first + whole((static_cast<size_t>(g.count) + v.c.batch + 2) * sizeof(int32_t));
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
    if (p.lead.blocks + p.rest.blocks > INT32_MAX) return bad("too many sequences, heads and tokens for one call.");
    char* base = static_cast<char*>(workspace);
    auto cut_args = [&](const Plan& part, PartSeq* seqs, int32_t* first) {
        const bool tile = part.kind == Kind::kTile;
        static_assert(kTileRows == 1 << 7 && kTileKeys == 1 << 6 && kRowsStep == 1 << 7);
        return CutArgs{tile ? 7 : -1, tile ? 6 : 7, tile ? CallPlan<kTileRows, kTileKeys, Part>::kMinSteps : 1,
                       part.slots, seqs, first};
    };
    PartSeq* seqs = reinterpret_cast<PartSeq*>(base + p.seqs);
    int32_t* first = reinterpret_cast<int32_t*>(base + p.first);
    Groups g{groups->first, groups->shared, groups->count, reinterpret_cast<int32_t*>(base), reinterpret_cast<int32_t*>(base) + groups->count + 1,
             cut_args(p.lead, seqs, first), cut_args(p.rest, seqs + groups->count, first + groups->count + 1)};
    hipLaunchKernelGGL(cut_kernel, dim3(1), dim3(kPlanThreads), 0, stream, v, *in, g);
    rc = launched(hipGetLastError(), "paged attention plan kernel launch");
    if (rc != QMM_OK) return rc;

    AttnArgs a{};
    a.in = *in;
    a.scale_log2 = score_scale(v, *in);
    a.v_scale = v.c.v_scale;
    a.part_o = reinterpret_cast<float*>(base + p.o);
    a.part_ml = reinterpret_cast<float2*>(base + p.ml);
    a.parts = p.rest.parts / in->heads;
    a.cut = reinterpret_cast<int4*>(base + p.cut);
    a.seqs = g.rest.seqs;
    a.first_block = g.rest.first_block;
    a.n_seqs = v.c.batch;
    LeadArgs l{g.lead.seqs, g.lead.first_block, g.count, static_cast<int>(p.lead.blocks), p.lead.parts / in->heads, a.cut + in->tokens};
    auto launch = [&](Kind lead, Kind rest, int64_t blocks, const LeadArgs& args) {
        with_shared_kernel(v, *in, lead, rest, p.row_tiles, [&](auto kern, size_t lds) {
            hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), lds, stream, v, a, args);
        });
    };
    if (p.one) {
        launch(p.lead.kind, p.rest.kind, p.lead.blocks + p.rest.blocks, l);
    } else {
        launch(p.lead.kind, p.lead.kind, p.lead.blocks, l);
        LeadArgs none = l;
        none.blocks = 0;
        launch(p.rest.kind, p.rest.kind, p.rest.blocks, none);
    }
    rc = launched(hipGetLastError(), "paged attention kernel launch");
    if (rc != QMM_OK) return rc;
    a.lead_cut = l.cut;
    a.lead_part = a.parts;
    a.all_parts = a.parts + l.parts;
    return launch_merge<Part>(v, a, true, p.rest.most_ranges + p.lead.most_ranges, stream);
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
