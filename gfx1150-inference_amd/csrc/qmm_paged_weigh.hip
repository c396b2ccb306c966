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

// The sum over the 16 lanes of a row of lanes, in all of them.
__device__ __forceinline__ float row_sum(float x) {
    auto step = [&](auto ctrl) { x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, false)); };
    step(std::integral_constant<int, 0xB1>{});   // lane ^ 1
    step(std::integral_constant<int, 0x4E>{});   // lane ^ 2
    step(std::integral_constant<int, 0x141>{});  // the mirrored lane of 8
    step(std::integral_constant<int, 0x140>{});  // .. and of 16
    return x;
}

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

// ---- matrix-core kernels ---------------------------------------------------------------------------
// A workgroup takes a share of the call's steps of kStep keys, in the order sequence, kv head, key: every sum is one
// workgroup's, and no sequence's length leaves the others waiting.
template <int kStep>
struct Steps {
    int seq, g, step, left;  // where a share begins; the sequence's steps from there on

    static __device__ __forceinline__ int of(const View& v, const AttnArgs& a, const WeighArgs& wa, int b) {
        if (b >= v.c.batch) return 0;
        return (summed_rows(wa, span_of<Lse>(v, a, b)) + kStep - 1) / kStep;
    }
    // every lane of the wave must be active
    static __device__ __forceinline__ int count(const View& v, const AttnArgs& a, const WeighArgs& wa, int lane) {
        int n = 0;
        for (int b0 = 0; b0 < v.c.batch; b0 += 64) n += __builtin_amdgcn_readlane(wave_scan(of(v, a, wa, b0 + lane)), 63);
        return n * v.c.kv_heads;
    }
    // Finds step `at` of them, which is below the count.
    __device__ __forceinline__ void find(const View& v, const AttnArgs& a, const WeighArgs& wa, int at, int lane) {
        int before = 0;
        for (int b0 = 0; b0 < v.c.batch; b0 += 64) {
            const int own = of(v, a, wa, b0 + lane) * v.c.kv_heads, upto = wave_scan(own);
            const int here = min(v.c.batch - b0, 64);
            const int hit = static_cast<int>(__popcll(__ballot(lane < here && before + upto <= at)));
            if (hit < here) {
                const int steps = __builtin_amdgcn_readlane(own, hit), rest = at - (before + __builtin_amdgcn_readlane(upto - own, hit));
                const int each = steps / v.c.kv_heads;
                seq = b0 + hit;
                g = rest / each;
                step = rest % each;
                left = each - step;
                return;
            }
            before += __builtin_amdgcn_readlane(upto, here - 1);
        }
    }
};

// Up to 16 NT rows (tokens x query heads of one kv head): decoding, small trees.  As in the attention over them a wave takes 32 keys
// at a time, straight into registers, and lane (l, q) = (lane % 16, lane / 16) receives the scores of row l with keys 4q ..
// 4q + 3 of each 16; their weights are added up over the 16 lanes.  Bound by reading K: 308 MB in 71 us, 4.3 TB/s.
constexpr int kRowsKeys = 128;

template <class T, class C, int D, int NT>
__global__ __launch_bounds__(kThreads) void weigh_rows_kernel(View v, AttnArgs a, WeighArgs wa) {
    using F = Frag<T>;
    using v8 = typename F::v8;
    constexpr bool kFp8 = std::is_same_v<C, Fp8>;
    constexpr int kF = D / 32;
    const int kvh = v.c.kv_heads, group = a.in.heads / kvh;
    const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = Steps<kRowsKeys>::count(v, a, wa, lane), share = (steps + gridDim.x - 1) / gridDim.x;
    int at = blockIdx.x * share;
    const int until = min(steps, at + share);
    const uint32_t k_off = static_cast<uint32_t>((l * v.c.k_slot + (kFp8 ? 16 : 8) * q) * sizeof(C));
    const uint32_t k_last = static_cast<uint32_t>((l * v.c.k_slot + 32 * (kF - 1) + 8 * q) * sizeof(C));  // fp8, an odd count of 32 dims
    while (at < until) {
        Steps<kRowsKeys> st;
        st.find(v, a, wa, at, lane);
        const int run = min(st.left, until - at), g = st.g;
        at += run;
        const Span s = span_of<Lse>(v, a, st.seq);
        const int held = summed_rows(wa, s), n_rows = min(s.n, a.in.max_new) * group;
        const float* from = wa.w.old_sums + st.seq * wa.w.old_batch + g * wa.w.old_head;
        float* to = wa.w.new_sums + st.seq * wa.w.new_batch + g * wa.w.new_head;
        // queries and their logarithms: rows past the last repeat it, and do not count
        v8 qf[NT][kF];
        float lse[NT];
        int tok[NT];
        bool counts[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = max(min(16 * nt + l, n_rows - 1), 0);
            tok[nt] = r / group;
            counts[nt] = 16 * nt + l < n_rows;
            lse[nt] = 0.0f;
            if (n_rows > 0) {
                const int head = g * group + r % group;
                const T* qrow = static_cast<const T*>(a.in.q) + static_cast<int64_t>(s.first + tok[nt]) * a.in.q_token + head * a.in.q_head;
#pragma unroll
                for (int f = 0; f < kF; ++f) {
                    const int d = kFp8 && (f | 1) < kF ? 64 * (f >> 1) + 16 * q + 8 * (f & 1) : 32 * f + 8 * q;
                    __builtin_memcpy(&qf[nt][f], __builtin_assume_aligned(qrow + d, 16), 16);
                }
                lse[nt] = a.lse[static_cast<int64_t>(s.first + tok[nt]) * a.in.heads + head];
            }
        }
        const char* kbase = reinterpret_cast<const char*>(static_cast<const C*>(v.c.k) + g * v.c.k_head);
        auto page_at = [&](int k0) { return n_rows > 0 && k0 < s.total ? page_of(v, s.seq, k0) : -1; };
        int kb = st.step * kRowsKeys + 32 * w;
        int id[2] = {page_at(kb), page_at(kb + 16)};
#pragma unroll 1
        for (int i = 0; i < run; ++i, kb += kRowsKeys) {
            u32x4 kr[2][kFp8 ? (kF + 1) / 2 : kF];
            bool ok[2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                const int k0 = kb + 16 * tt, u = __builtin_amdgcn_readfirstlane(id[tt]);
                ok[tt] = u >= 0;
                const char* kp = kbase + (static_cast<int64_t>(max(u, 0)) * v.c.k_page + (k0 & (v.c.page_size - 1)) * v.c.k_slot) * static_cast<int64_t>(sizeof(C));
#pragma unroll
                for (int f = 0; f < (kFp8 ? kF / 2 : kF); ++f) {
                    uint32_t x[4];
                    load_row_bytes<16, 16, true>(x, kp + 64 * f + k_off);
                    kr[tt][f] = u32x4{x[0], x[1], x[2], x[3]};
                }
                if constexpr (kFp8 && kF % 2) {
                    const u32x2 x = *reinterpret_cast<const u32x2*>(kp + k_last);
                    kr[tt][kF / 2] = u32x4{x[0], x[1], 0, 0};
                }
            }
            // lane (l < 8, q) ends up with key 16 (l / 4) + 4q + l % 4
            const int own = kb + 16 * ((l >> 2) & 1) + 4 * q + (l & 3);
            float old = 0.0f;
            if (l < 8 && own < min(s.ctx, held)) old = from[own];
            id[0] = page_at(kb + kRowsKeys);
            id[1] = page_at(kb + kRowsKeys + 16);
            __builtin_amdgcn_sched_barrier(0);
            const bool full = kb + 32 <= s.ctx && ok[0] && ok[1];
            v8 kf[2][kF];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int f = 0; f < kF; ++f) {
                    if constexpr (kFp8) {
                        const uint32_t x = kr[tt][f >> 1][2 * (f & 1)], y = kr[tt][f >> 1][2 * (f & 1) + 1];
                        const u32x4 t = {F::from_fp8(x), F::from_fp8_hi(x), F::from_fp8(y), F::from_fp8_hi(y)};
                        kf[tt][f] = __builtin_bit_cast(v8, t);
                    } else {
                        kf[tt][f] = __builtin_bit_cast(v8, kr[tt][f]);
                    }
                }
            // what every row sees, ahead of the first product: round a branch between a product and its use the compiler has
            // left out the wait for the result (tests/test_matrix_waits.py)
            uint32_t vis[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) vis[nt] = 0xFFFFFFFFu;
            if (!full)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    vis[nt] = visible32(a, s, tok[nt], kb);
                    if (!ok[0]) vis[nt] &= 0xFFFF0000u;
                    if (!ok[1]) vis[nt] &= 0x0000FFFFu;
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) vis[nt] = counts[nt] ? vis[nt] >> (4 * q) : 0;
            float sum[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] = 0.0f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int f = 0; f < kF; ++f) sc = F::mma16(kf[tt][f], qf[nt][f], sc);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p = __builtin_amdgcn_exp2f(__fmaf_rn(sc[e], a.scale_log2, -lse[nt]));
                        sum[4 * tt + e] += (vis[nt] >> (16 * tt + e)) & 1 ? p : 0.0f;
                    }
                }
            float mine = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = row_sum(sum[e]);
                if (l == e) mine = x;
            }
            if (l < 8 && own < held) to[own] = old + mine;
        }
    }
}

// Up to 16 rows whose scores the attention has left: 8 bytes a row and key go to memory and back where the keys would be read again
// (256 bytes of 128 dimensions in 16 bits).  A lane takes a key.  The first `joins` workgroups join the attention's ranges
// meanwhile, so the others find the logarithms from the ranges' sums themselves, 16 lanes a row: a launch less (one decode at 4096 rows: 18.4 us
// with it, 14.4 without).
constexpr int kStoredKeys = kThreads;

template <class T>
__global__ __launch_bounds__(kThreads) void weigh_stored_kernel(View v, AttnArgs a, WeighArgs wa, JoinShape shape, int joins) {
    __shared__ float lse[16];
    if (static_cast<int>(blockIdx.x) < joins) {
        join_ranges<T, true, Lse>(v, a, shape.sg, static_cast<int>(blockIdx.x) / shape.per_token, static_cast<int>(blockIdx.x) % shape.per_token);
        return;
    }
    const int kvh = v.c.kv_heads, group = a.in.heads / kvh, lane = threadIdx.x & 63, blocks = gridDim.x - joins;
    const int steps = Steps<kStoredKeys>::count(v, a, wa, lane), share = (steps + blocks - 1) / blocks;
    const float scale = fabsf(a.scale_log2);  // the attention takes a negative one into its queries
    int at = (blockIdx.x - joins) * share;
    const int until = min(steps, at + share);
    while (at < until) {
        Steps<kStoredKeys> st;
        st.find(v, a, wa, at, lane);
        const int run = min(st.left, until - at), g = st.g;
        at += run;
        const Span s = span_of<Lse>(v, a, st.seq);
        const int held = summed_rows(wa, s), n_rows = min(s.n, a.in.max_new) * group;
        const float* from = wa.w.old_sums + st.seq * wa.w.old_batch + g * wa.w.old_head;
        float* to = wa.w.new_sums + st.seq * wa.w.new_batch + g * wa.w.new_head;
        const float* scores = a.scores + (static_cast<int64_t>(st.seq) * kvh + g) * a.score_rows * a.score_keys;
        __syncthreads();  // the last run's logarithms have been read
        if (const int r = threadIdx.x >> 4; r < n_rows) {
            const int t = s.first + r / group;
            const int64_t row = static_cast<int64_t>(t) * a.in.heads + g * group + r % group;
            const int4 cut = a.cut ? a.cut[t] : int4{1, 0, 0, 0};
            float m = -INFINITY, sum = 0.0f;
            const bool whole = cut.x <= 1, fits = cut.y >= 0 && cut.z >= 1 && cut.y + static_cast<int64_t>(cut.x - 1) * cut.z < a.parts;
            if (!whole && fits) {
                for (int c = lane & 15; c < cut.x; c += 16) {
                    const int64_t part = (cut.y + static_cast<int64_t>(c) * cut.z) * a.in.heads + g * group + r % group;
                    const float pm = a.part_ml[part].x, ps = a.part_sum[part];
                    if (ps == 0.0f) continue;
                    const float mn = fmaxf(m, pm);
                    sum = (m == mn ? sum : sum * __builtin_amdgcn_exp2f(m - mn)) + (pm == mn ? ps : ps * __builtin_amdgcn_exp2f(pm - mn));
                    m = mn;
                }
            }
            float top = m;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 16));
            if (sum != 0.0f && m != top) sum *= __builtin_amdgcn_exp2f(m - top);
            sum = row_sum(sum);
            if ((lane & 15) == 0) lse[r] = whole ? a.lse[row] : log_sum(top, sum);
        }
        __syncthreads();
        for (int k = st.step * kStoredKeys + static_cast<int>(threadIdx.x), i = 0; i < run; ++i, k += kStoredKeys) {
            if (k >= held) continue;
            const float old = k < s.ctx ? from[k] : 0.0f;
            float sum = 0.0f;
            if (k < s.total)
#pragma unroll 8
                for (int r = 0; r < n_rows; ++r) {
                    // of a key that the row does not see nothing, also where the row's logarithm is NaN
                    const float x = __builtin_nontemporal_load(scores + (static_cast<int64_t>(k >> 2) * a.score_rows + r) * 4 + (k & 3));
                    const float p = __builtin_amdgcn_exp2f(__fmaf_rn(x, scale, -lse[r]));
                    sum += x == -INFINITY ? 0.0f : p;
                }
            to[k] = old + sum;
        }
    }
}

// More rows.  A workgroup takes 64 keys, held in registers as an operand of 32x32x16, and its waves the rows in turns of 32: a lane
// has one row (lane % 32) and 16 of every 32 keys, so that a row's logarithm is the lane's and the sums of its keys gather in
// registers; they are added up over the lanes and the waves, in order, at the end.  Two chunks of up to 600 tokens, 32 heads of 128 over
// up to 2100 keys (14 GFLOP): 44 us, bound by the waits of two waves a SIMD (matrix cores busy for 14 % of the cycles, vector ALUs 33 %).
constexpr int kTileKeysW = 64;

template <class T, class C, int D>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void weigh_tile_kernel(View v, AttnArgs a, WeighArgs wa) {
    using F = Frag<T>;
    using v8 = typename F::v8;
    constexpr bool kFp8 = std::is_same_v<C, Fp8>;
    __shared__ float part[4][kTileKeysW];
    const int kvh = v.c.kv_heads, group = a.in.heads / kvh;
    const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = Steps<kTileKeysW>::count(v, a, wa, lane);
    for (int at = blockIdx.x; at < steps; at += gridDim.x) {
        Steps<kTileKeysW> st;
        st.find(v, a, wa, at, lane);
        const Span s = span_of<Lse>(v, a, st.seq);
        const int g = st.g, held = summed_rows(wa, s), n_rows = min(s.n, a.in.max_new) * group, kb = st.step * kTileKeysW;
        // keys: lane's key l32 of each 32, dims 16 db + 8 h ..
        v8 kf[2][D / 16];
        uint32_t have = 0;  // bit t: the page of keys 16 t .. is there
        if (n_rows > 0) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (kb + 16 * t < s.total && page_of(v, s.seq, kb + 16 * t) >= 0) have |= 1u << t;
            const C* kbase = static_cast<const C*>(v.c.k) + g * v.c.k_head;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int k = kb + 32 * hh + l32, id = k < s.total ? page_of(v, s.seq, k) : -1;
                const C* kp = kbase + static_cast<int64_t>(max(id, 0)) * v.c.k_page + (k & (v.c.page_size - 1)) * v.c.k_slot + 8 * h;
#pragma unroll
                for (int db = 0; db < D / 16; ++db) {
                    if constexpr (kFp8) {
                        const u32x2 x = *reinterpret_cast<const u32x2*>(kp + 16 * db);
                        const u32x4 y = {F::from_fp8(x[0]), F::from_fp8_hi(x[0]), F::from_fp8(x[1]), F::from_fp8_hi(x[1])};
                        kf[hh][db] = __builtin_bit_cast(v8, y);
                    } else {
                        __builtin_memcpy(&kf[hh][db], __builtin_assume_aligned(kp + 16 * db, 16), 16);
                    }
                }
            }
        }
        f32x16 sum[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[hh][e] = 0.0f;
        const bool cached = kb + kTileKeysW <= s.ctx && have == 15;
        // a chain's rows ahead of the first key see none of them
        const int first = a.in.mask == nullptr ? max(kb - s.ctx, 0) * group / 32 : 0;
        v8 next[D / 16];  // the next rows are on the way while these are multiplied
        float next_lse = 0.0f;
        int next_i = 0;
        auto request = [&](int r0) {
            const int r = max(min(r0 + l32, n_rows - 1), 0), head = g * group + r % group;
            next_i = r / group;
            const T* qrow = static_cast<const T*>(a.in.q) + static_cast<int64_t>(s.first + next_i) * a.in.q_token + head * a.in.q_head + 8 * h;
#pragma unroll
            for (int db = 0; db < D / 16; ++db) __builtin_memcpy(&next[db], __builtin_assume_aligned(qrow + 16 * db, 16), 16);
            next_lse = a.lse[static_cast<int64_t>(s.first + next_i) * a.in.heads + head];
        };
        const int begin = 32 * (first + ((w - first) & 3));
        if (begin < n_rows) request(begin);
#pragma unroll 1
        for (int r0 = begin; r0 < n_rows; r0 += 128) {
            v8 qf[D / 16];
#pragma unroll
            for (int db = 0; db < D / 16; ++db) qf[db] = next[db];
            const float lse = next_lse;
            const int i = next_i;
            const bool counts = r0 + l32 < n_rows;
            if (D <= 128) {
                if (r0 + 128 < n_rows) request(r0 + 128);
            }
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                f32x16 x;
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = 0.0f;
#pragma unroll
                for (int db = 0; db < D / 16; ++db) x = F::mma32(kf[hh][db], qf[db], x);
                uint32_t vis = 0xFFFFFFFFu;
                if (!cached) {
                    vis = visible32(a, s, i, kb + 32 * hh);
                    if (!((have >> (2 * hh)) & 1)) vis &= 0xFFFF0000u;
                    if (!((have >> (2 * hh + 1)) & 1)) vis &= 0x0000FFFFu;
                }
                vis = counts ? vis >> (4 * h) : 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float p = __builtin_amdgcn_exp2f(__fmaf_rn(x[e], a.scale_log2, -lse));
                    sum[hh][e] += (vis >> (8 * (e >> 2) + (e & 3))) & 1 ? p : 0.0f;
                }
            }
            if (D > 128 && r0 + 128 < n_rows) request(r0 + 128);  // no registers for both
        }
        // register e of half hh is key 32 hh + 8 (e / 4) + 4 h + e % 4
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float x = row_sum(sum[hh][e]);
                x += __shfl_xor(x, 16, 64);
                if (l32 == 0) part[w][32 * hh + 8 * (e >> 2) + 4 * h + (e & 3)] = x;
            }
        __syncthreads();
        const int k = kb + static_cast<int>(threadIdx.x);
        if (threadIdx.x < kTileKeysW && k < held) {
            const int c = threadIdx.x;
            const float x = ((part[0][c] + part[1][c]) + part[2][c]) + part[3][c];
            const float* from = wa.w.old_sums + st.seq * wa.w.old_batch + g * wa.w.old_head;
            wa.w.new_sums[st.seq * wa.w.new_batch + g * wa.w.new_head + k] = k < s.ctx ? from[k] + x : x;
        }
        __syncthreads();
    }
}

struct WeighPlan {
    Plan attend;
    size_t lse, scores, bytes;  // where the logarithms and the scores begin
    int score_rows, score_keys;  // 0: the keys are read again
};

// The scores of few rows are kept where they cost less than the keys' second reading (16 sequences of up to 16384 keys, 8 rows a kv
// head of 128 dimensions: the attention takes 143 us with the stores, 114 without; this pass 22 us, 71 with the keys), a byte
// written for about two read, and do not take too much memory.
constexpr int64_t kMostScores = int64_t{1} << 29;

WeighPlan weigh_plan(const View& v, const qmm_paged_query& in, const qmm_paged_weights& w) {
    WeighPlan p{};
    p.attend = plan<Lse>(v, in);
    p.lse = (p.attend.bytes + 15) / 16 * 16;
    p.bytes = p.scores = p.lse + (static_cast<size_t>(in.tokens) * in.heads * sizeof(float) + 15) / 16 * 16;
    const int64_t rows = static_cast<int64_t>(std::min(in.max_new, in.tokens)) * (in.heads / v.c.kv_heads);
    if (p.attend.kind == Kind::kRows && rows > 0 && rows <= 16 && 12 * rows <= static_cast<int64_t>(v.c.head_dim) * elem_bytes(v.c.dtype)) {
        const int64_t keys = (std::min<int64_t>(w.rows, static_cast<int64_t>(v.c.table_width) * v.c.page_size) + 3) / 4 * 4;
        const int64_t bytes = static_cast<int64_t>(v.c.batch) * v.c.kv_heads * rows * keys * 4;
        if (keys > 0 && keys < INT32_MAX - 64 && bytes <= kMostScores && static_cast<int64_t>(in.tokens) * in.heads < 1 << 28) {
            p.score_rows = static_cast<int>(rows);
            p.score_keys = static_cast<int>(keys);
            p.bytes += bytes;
        }
    }
    return p;
}

int check_weights(const View& v, const qmm_paged_weights* w) {
    if (!w) return bad("weights must be non-null.");
    if (w->rows < 0) return bad("rows must be non-negative.");
    if (w->rows > 0 && v.c.batch > 0 && (!w->old_sums || !w->new_sums)) return bad("old_sums and new_sums must be non-null.");
    if ((reinterpret_cast<uintptr_t>(w->old_sums) | reinterpret_cast<uintptr_t>(w->new_sums)) % 4 != 0) return bad("old_sums and new_sums must be aligned to their elements.");
    if (w->old_sums == w->new_sums && (w->old_batch != w->new_batch || w->old_head != w->new_head)) return bad("sums in place need the same strides.");
    if (v.c.kv_heads > 65535) return bad("too many heads.");
    if (w->rows > 0 && !apart({{v.c.kv_heads, w->new_head}, {v.c.batch, w->new_batch}}, w->rows)) return bad("new_sums must not overlap itself.");
    return QMM_OK;
}

// Calls f with the matrix-core kernel for a call's rows and types.
template <class T, class C, int D, class Fn>
void with_weigh_kernel(int64_t rows, Fn f) {
    if (rows <= 16) return f(weigh_rows_kernel<T, C, D, 1>);
    if (rows <= 32) return f(weigh_rows_kernel<T, C, D, 2>);
    if (D <= 128 && rows <= 64) return f(weigh_rows_kernel<T, C, D, D <= 128 ? 4 : 2>);
    f(weigh_tile_kernel<T, C, D>);
}

template <class Fn>
void with_weigh_kernel(const View& v, const qmm_paged_query& in, Fn f) {
    const int64_t rows = static_cast<int64_t>(std::min(in.max_new, in.tokens)) * (in.heads / v.c.kv_heads);
    auto types = [&](auto tc, auto cc) {
        using T = decltype(tc);
        using C = decltype(cc);
        switch (v.c.head_dim) {
            case 64: return with_weigh_kernel<T, C, 64>(rows, f);
            case 96: return with_weigh_kernel<T, C, 96>(rows, f);
            case 128: return with_weigh_kernel<T, C, 128>(rows, f);
            default: return with_weigh_kernel<T, C, 256>(rows, f);
        }
    };
    const bool fp8 = v.c.dtype == QMM_DTYPE_E4M3;
    if (in.dtype == QMM_DTYPE_F16) return fp8 ? types(_Float16{}, Fp8{}) : types(_Float16{}, _Float16{});
    return fp8 ? types(__bf16{}, Fp8{}) : types(__bf16{}, __bf16{});
}

int weighted_attention(const qmm_paged_kv* kv, const qmm_paged_query* in, const qmm_paged_weights* weights, void* workspace,
                       size_t workspace_bytes, hipStream_t stream) {
    View v;
    int rc = check_query(kv, in, &v);
    if (rc == QMM_OK) rc = check_weights(v, weights);
    if (rc != QMM_OK) return rc;
    if (v.c.batch == 0) return QMM_OK;
    const bool attends = in->tokens > 0 && in->max_new > 0;
    const WeighPlan p = weigh_plan(v, *in, *weights);
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
    if (p.score_rows > 0) {
        a.scores = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.scores);
        a.score_rows = p.score_rows;
        a.score_keys = p.score_keys;
    }
    if (attends) {
        rc = launch_attention<Lse>(v, a, p.attend, stream);
        if (rc == QMM_OK && p.attend.merge && !a.scores) rc = launch_merge<Lse>(v, a, p.attend.kind != Kind::kLanes, p.attend.most_ranges, stream);
        if (rc != QMM_OK) return rc;
    }
    WeighArgs wa{*weights, 1};
    if (a.scores) {
        auto stored = [&](auto kern) {
            const JoinShape shape = join_shape(v, a, p.attend.most_ranges);
            const int64_t joins = p.attend.merge ? static_cast<int64_t>(in->tokens) * shape.per_token : 0;
            const int64_t steps = static_cast<int64_t>(v.c.batch) * v.c.kv_heads * ((weights->rows + kStoredKeys - 1) / kStoredKeys);
            const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(kernel_slots(kern, 0), steps));
            hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(joins + blocks)), dim3(kThreads), 0, stream, v, a, wa, shape, static_cast<int>(joins));
        };
        in->dtype == QMM_DTYPE_F16 ? stored(weigh_stored_kernel<_Float16>) : stored(weigh_stored_kernel<__bf16>);
        return launched(hipGetLastError(), "paged weights kernel launch");
    }
    if (weights->rows == 0) return QMM_OK;
    if (p.attend.kind != Kind::kLanes) {
        with_weigh_kernel(v, *in, [&](auto kern) {
            // workgroups that run at once, or one for each step that there can be
            const int64_t steps = static_cast<int64_t>(v.c.batch) * v.c.kv_heads * ((weights->rows + kTileKeysW - 1) / kTileKeysW);
            const int64_t blocks = std::min<int64_t>(kernel_slots(kern, 0), steps);
            hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, v, a, wa);
        });
        return launched(hipGetLastError(), "paged weights kernel launch");
    }
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
        if (rc == QMM_OK && in->tokens > 0 && v.c.batch > 0) bytes = qmm::paged::weigh_plan(v, *in, *weights).bytes;
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
