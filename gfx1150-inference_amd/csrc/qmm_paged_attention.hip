// Attention of new tokens over a paged key/value cache:
//   out_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r k_j - max_j),
// over the rows j that row r = (token, query head) sees: the sequence's cached rows, and those of its new
// rows that a bit mask (a drafted tree) or the order (a chain) lets it see.
//
// The keys of a sequence are cut into ranges, one workgroup each, where the rows alone leave the chip idle; a
// range's maximum (base 2), sum and unnormalised output are joined by a second kernel in the order of the ranges,
// so a call repeats itself to the bit.  Its bits go by what chooses the kernel and the cut: all sequences' lengths,
// max_new, alignment, the workgroups that the device runs at once, and, on the vector ALUs, the table's width.  How long a range is, every workgroup works out from all
// sequences' lengths, which only the device knows (plan_call): the host sees no more than the width of the table.
#include "qmm_device.h"
#include "qmm_paged.h"

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <type_traits>
#include <utility>

namespace qmm {
namespace paged {
namespace {

constexpr int kThreads = 256;

struct AttnArgs {
    qmm_paged_query in;
    float scale_log2;  // scale * k_scale * log2 e
    float v_scale;
    int kps;           // keys per range of the kernel without a plan
    int slots;         // workgroups that a plan cuts the call into: those that run at once
    float* part_o;     // [partial row][D]
    float2* part_ml;   // [partial row]: maximum, sum
    int64_t parts;     // tokens that the partial rows have room for
    int4* cut;         // [token]: ranges, its first partial row and the rows between ranges, in tokens
};

// The new tokens of one sequence.
struct Span {
    int seq, first, n, ctx, total;  // first token, count, cached rows, rows that the table can hold of both
};

__device__ __forceinline__ Span span_of(const View& v, const AttnArgs& a, int seq) {
    Span s;
    s.seq = seq;
    s.first = max(v.c.cu[seq], 0);
    s.n = max(min(max(v.c.cu[seq + 1], 0), a.in.tokens) - s.first, 0);
    s.ctx = cached_rows(v, seq);
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

// Writes what scan_row left (lanes below D / 8 hold 8 dimensions each): the output where its range is the only one
// (part < 0), else the partial row.
template <class T>
__device__ __forceinline__ void write_state(const View& v, const AttnArgs& a, int t, int head, int64_t part, const RowState& r, int lane) {
    const int d0 = 8 * lane;
    if (part < 0) {
        if (d0 >= v.c.head_dim) return;
        T* out = static_cast<T*>(a.in.out) + static_cast<int64_t>(t) * a.in.out_token + head * a.in.out_head;
        const float inv = r.l == 0.0f ? 0.0f : a.v_scale / r.l;
#pragma unroll
        for (int e = 0; e < 8; ++e) out[d0 + e] = static_cast<T>(r.l == 0.0f ? 0.0f : r.o[e] * inv);
    } else {
        if (lane == 0) a.part_ml[part] = float2{r.m, r.l};
        if (d0 < v.c.head_dim)
#pragma unroll
            for (int e = 0; e < 8; ++e) a.part_o[part * v.c.head_dim + d0 + e] = r.o[e];
    }
}

// Every head size and alignment: one wave per row and range.  Block (x, y, z): token, range, heads.
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
    const int end = begin + min(s.total - begin, a.kps);  // kps may be INT32_MAX
    const RowState r = scan_row<T, C>(v, a, s, t - s.first, head, begin, end, lane, lpk, aligned != 0);
    const int64_t part = s.total <= a.kps ? -1 : (static_cast<int64_t>(split) * a.in.tokens + t) * a.in.heads + head;
    write_state<T>(v, a, t, head, part, r, lane);
}

// ---- matrix-core kernels: shared parts ---------------------------------------------------------
// Both take head_dim 64, 96, 128 and 256, pages of 16 rows and more, and 16-byte aligned operands.  The page
// ids of up to kWindow keys of a range are read into LDS together, so that no load of a row waits for one of the table.
constexpr int kWindow = 8 * 1024, kWindowPages = kWindow / 16 + 1;
// The running maximum that the weights are relative to moves only when a score passes it by 2^kSlack, so that most
// blocks of keys rescale nothing; weights enter the second product as 2^(x - m + kShift), f16's range used from
// 2^(kSlack + kShift) down.  Both cancel against the sum.
constexpr float kSlack = 8.0f, kShift = 5.0f;

template <class T>
struct Frag;
template <>
struct Frag<_Float16> {
    using v8 = f16x8;
    static __device__ __forceinline__ f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    // c + a[i] + a[i + 1]
    static __device__ __forceinline__ float add2(v8 a, int i, float c) {
        return __builtin_amdgcn_fdot2(f16x2{a[i], a[i + 1]}, f16x2{static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)}, c, false);
    }
    static __device__ __forceinline__ uint32_t from_fp8(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    }
    static __device__ __forceinline__ uint32_t from_fp8_hi(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
};
template <>
struct Frag<__bf16> {
    using v8 = bf16x8;
    static __device__ __forceinline__ f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float add2(v8 a, int i, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(bf16x2{a[i], a[i + 1]}, bf16x2{static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)}, c, false);
    }
    static __device__ __forceinline__ uint32_t from_fp8(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    }
    static __device__ __forceinline__ uint32_t from_fp8_hi(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
    }
};

// The keys k0 .. k0 + 31 that new token i of the sequence sees, as bits (pages apart).
__device__ __forceinline__ uint32_t visible32(const AttnArgs& a, const Span& s, int i, int k0) {
    const int c = s.ctx - k0, e = s.total - k0;  // cached keys, keys at all
    auto low = [](int n) { return n >= 32 ? 0xFFFFFFFFu : n > 0 ? (1u << n) - 1u : 0u; };
    uint32_t m = low(c);
    if (c < 32) {
        if (a.in.mask == nullptr) {
            m |= low(c + i + 1);
        } else {
            const int j = max(-c, 0), word = j >> 5;  // new token of the first key that is none of the cached
            const int32_t* row = a.in.mask + (s.first + i) * a.in.mask_stride;
            const uint32_t w0 = word < a.in.mask_words ? row[word] : 0, w1 = word + 1 < a.in.mask_words ? row[word + 1] : 0;
            const uint32_t bits = static_cast<uint32_t>(((static_cast<uint64_t>(w1) << 32) | w0) >> (j & 31));
            m |= bits << max(c, 0);
        }
    }
    return m & low(e);
}

// Sums of lanes 0 .. l of the wave (every lane must be active): rows of 16 by shifts, then the rows' last lanes
// broadcast.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}

__device__ __forceinline__ float wave_total(float x) {
    auto step = [&](auto ctrl, auto rows) {
        x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
    };
    step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});
    step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
    step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
    step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// How a call is cut, from its sequences' lengths; the same in every wave of every workgroup.
//   steps      64 keys of a 128-row tile, or 128 keys of the one tile of few rows, is a step; a chain's row tiles
//              see fewer keys than the last one does, so their mean counts;
//   ranges     a sequence of S steps a row tile is cut into ceil(S / u) ranges of the same length, u the smallest of
//              four lengths from W / slots (W: the steps of the call) to 1.75 times that whose workgroups all find a place
//              (`slots`) at once, W / slots where none does.  So a long sequence is cut and a short one beside it is
//              not, whatever the table's width;
//   blocks     (sequence, range, row tile, kv head), kv head fastest, in the sequences' order;
//   partials   the rows of sequences with more than one range, in the same order.
template <int kTile, int kStep>
struct CallPlan {
    static constexpr int kMinSteps = kTile >= 128 ? 4 : 1, kTries = 4;
    int seq, block;           // block within the sequence
    int rows, tiles, ranges;  // of the sequence: tokens with rows, row tiles
    int keys;                 // per range
    int first_part;           // of the sequence, in tokens

    struct Lane {
        int rows, tiles, steps;  // steps of all keys of a row tile
        float work;              // mean steps of all row tiles
    };
    static __device__ __forceinline__ Lane lane_of(const View& v, const AttnArgs& a, int b) {
        Lane x{0, 0, 0, 0.0f};
        if (b < v.c.batch) {
            const Span s = span_of(v, a, b);
            x.rows = min(s.n, a.in.max_new);
            x.tiles = kTile >= 128 ? (x.rows * (a.in.heads / v.c.kv_heads) + kTile - 1) / kTile : x.rows > 0;
            x.steps = x.rows > 0 ? max((s.total + kStep - 1) / kStep, 1) : 0;
            const int seen = a.in.mask ? s.total : min(s.total, s.ctx + (s.n + 1) / 2);
            x.work = static_cast<float>(max((seen + kStep - 1) / kStep, 1)) * static_cast<float>(x.tiles);
        }
        return x;
    }

    // Finds the sequence of workgroup `at`; false: there is none.  Lengths and counts of workgroups are compared in fp32,
    // whose roundings are the same everywhere.
    __device__ __forceinline__ bool find(const View& v, const AttnArgs& a, int at, int lane) {
        const int kvh = v.c.kv_heads;
        double own_work = 0.0;  // of this lane's sequences, up to a thousand: no rounding, whatever the batch
        Lane x{};
        for (int b0 = 0; b0 < v.c.batch; b0 += 64) {
            x = lane_of(v, a, b0 + lane);
            own_work += static_cast<double>(x.work);
        }
        const float work = wave_total(static_cast<float>(own_work));
        // 1e-5 covers the ten roundings from here on (and one in a lane's work): a length is never below W / slots, or it is 2^25 steps, which no sequence passes
        const float shortest = work * static_cast<float>(kvh) / static_cast<float>(a.slots) * 1.00001f;
        int u[kTries];
        float count[kTries];
#pragma unroll
        for (int c = 0; c < kTries; ++c) {
            u[c] = max(static_cast<int>(fminf(ceilf(shortest * (1.0f + 0.25f * static_cast<float>(c))), 33554432.0f)), kMinSteps);
            count[c] = 0.0f;
        }
        auto ranges_of = [&](int steps, int len) { return static_cast<int>((static_cast<uint32_t>(steps) + len - 1) / static_cast<uint32_t>(len)); };
        for (int b0 = 0; b0 < v.c.batch; b0 += 64) {
            if (v.c.batch > 64) x = lane_of(v, a, b0 + lane);
#pragma unroll
            for (int c = 0; c < kTries; ++c) count[c] += wave_total(static_cast<float>(ranges_of(x.steps, u[c])) * static_cast<float>(x.tiles));
        }
        int best = u[0];
#pragma unroll
        for (int c = kTries - 1; c >= 0; --c)
            if (count[c] * static_cast<float>(kvh) <= static_cast<float>(a.slots)) best = u[c];
        int blocks = 0, parts = 0;
        for (int b0 = 0; b0 < v.c.batch; b0 += 64) {
            if (v.c.batch > 64) x = lane_of(v, a, b0 + lane);
            const int n = ranges_of(x.steps, best);
            const int own_blocks = n * x.tiles * kvh, own_parts = n > 1 ? n * x.rows : 0;
            const int sb = wave_scan(own_blocks), sp = wave_scan(own_parts);
            const int here = min(v.c.batch - b0, 64);
            const int hit = static_cast<int>(__popcll(__ballot(lane < here && blocks + sb <= at)));
            if (hit < here) {
                auto of = [&](int t) { return __builtin_amdgcn_readlane(t, hit); };
                seq = b0 + hit;
                rows = of(x.rows);
                tiles = of(x.tiles);
                ranges = of(n);
                keys = (of(x.steps) + ranges - 1) / ranges * kStep;
                block = at - (blocks + of(sb - own_blocks));
                first_part = parts + of(sp - own_parts);
                // room is short only where cu descends and sequences overlap
                return ranges == 1 || first_part + static_cast<int64_t>(ranges) * rows <= a.parts;
            }
            blocks += __builtin_amdgcn_readlane(sb, here - 1);
            parts += __builtin_amdgcn_readlane(sp, here - 1);
        }
        return false;
    }
    __device__ __forceinline__ int64_t part_of(const AttnArgs& a, int range, int i, int head) const {
        return ranges == 1 ? -1 : (first_part + static_cast<int64_t>(range) * rows + i) * a.in.heads + head;
    }
    // what the join needs to know of token i of the sequence
    __device__ __forceinline__ int4 cut_of(int i) const { return int4{ranges, first_part + i, rows, 0}; }
};

// Page ids of the rows [begin, end) into LDS; true if one of them is missing.
__device__ __forceinline__ bool stage_pages(const View& v, int seq, int begin, int end, int* pages) {
    bool missing = false;
    if (begin < end) {
        const int p0 = begin >> v.page_shift, n = ((end - 1) >> v.page_shift) - p0 + 1;
        for (int p = threadIdx.x; p < n; p += kThreads) {
            const int id = page_of(v, seq, (p0 + p) << v.page_shift);
            pages[p] = id;
            missing |= id < 0;
        }
    }
    return __syncthreads_or(missing);
}

// B bytes of a cache row.  kOnce: no other wave reads them, so they need not stay in the caches.
template <int B, int kAlign, bool kOnce>
__device__ __forceinline__ void load_row_bytes(uint32_t* dst, const char* src) {
    if constexpr (kOnce && B % 16 == 0 && kAlign == 16) {
#pragma unroll
        for (int i = 0; i < B / 16; ++i) {
            const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src) + i);
            __builtin_memcpy(dst + 4 * i, &x, 16);
        }
    } else if constexpr (kOnce && B == 8 && kAlign == 8) {
        const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(src));
        __builtin_memcpy(dst, &x, 8);
    } else {
        __builtin_memcpy(dst, __builtin_assume_aligned(src, kAlign), B);
    }
}

// ---- few rows: keys straight into registers ------------------------------------------------------
// Up to 64 rows (tokens x query heads of one kv head) against one kv head's keys: decoding, small trees.  Bound by
// reading K and V from HBM, each once (1.32 GB of 32 users in 220 us, 6.0 TB/s; 238 us with loads that keep the lines).  A wave
// takes 32 keys at a time, no LDS on the way, and every row tile of 16 uses them:
//   * S^T = K Q^T on 16x16x32: lane (l, q) = (lane % 16, lane / 16) loads key l's dims 8 q.. of every 32 (fp8: 16 bytes of
//     every 64, the queries' dims in the same order) and receives the scores of row l with keys 4q .. 4q + 3 of
//     each 16;
//   * those 8 keys are the k order of the second product's operand, so the weights go straight from the score
//     registers into O^T += V^T P^T; lane (l, q) loads dims D/16 l .. of its 8 keys' values (16 lanes read one
//     row) and v_perm transposes them in registers.
// With one row tile the weights enter as hi + lo in the operands' type, two products: 16 bits and more, where memory
// hides them.  With more tiles the products are a good part of the time and the weights are rounded once, half a
// step of each weight (as large as the output's own rounding, and of either sign): f16 outputs of 13-node trees are
// 2.8e-4 off in the 2-norm, 2.1e-4 with hi + lo, which is their own rounding; the kernel takes 42 us, 49 with hi + lo.
// The 4 waves take every fourth 32-key block of the range; above 32 rows two take half of the rows each (RG = 2), their
// keys from the L1 cache: one wave's 64 rows of head_dim 128 leave no registers for a second wave on the SIMD (an fp8 cache
// of 57000 rows, 52 rows a kv head: 51 us with four row tiles a wave, 42 us).  Joined through LDS in wave order.
constexpr int kRowsStep = 128;

template <class T, class C, int D, int NT, int RG>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void attention_rows_kernel(View v, AttnArgs a) {
    using F = Frag<T>;
    using v8 = typename F::v8;
    constexpr bool kFp8 = std::is_same_v<C, Fp8>;
    constexpr int kF = D / 32, kVB = D / 16 * static_cast<int>(sizeof(C)), kVW = D / 32;  // fragments; bytes of a value slice; its dwords of T
    constexpr int kVAlign = (kVB & -kVB) < 16 ? kVB & -kVB : 16;
    constexpr bool kLo = NT == 1;
    constexpr int kRowF = D + 4, kWaves = kThreads / 64, kKeyWaves = kWaves / RG;
    __shared__ __align__(16) float so[kWaves][16 * kRowF];
    __shared__ float2 sml[kWaves][16];
    __shared__ int pages[kWindowPages];
    const int kvh = v.c.kv_heads, group = a.in.heads / kvh;
    const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    CallPlan<16, kRowsStep> cp;
    if (!cp.find(v, a, static_cast<int>(blockIdx.x), lane)) return;
    const int g = cp.block % kvh, range = cp.block / kvh;
    const Span s = span_of(v, a, cp.seq);
    const int kps = cp.keys;
    const int begin = range * kps, end = min(s.total, begin + kps);
    const int n_rows = cp.rows * group, rg = w / kKeyWaves, kw = w % kKeyWaves, rb = 16 * NT * rg;  // the wave's rows from rb on
    if (g == 0 && range == 0 && a.cut && static_cast<int>(threadIdx.x) < cp.rows) a.cut[s.first + threadIdx.x] = cp.cut_of(threadIdx.x);

    // queries: rows past the last repeat it
    v8 qf[NT][kF];
    int tok[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = min(rb + 16 * nt + l, n_rows - 1);
        tok[nt] = r / group;
        const T* qrow = static_cast<const T*>(a.in.q) + static_cast<int64_t>(s.first + tok[nt]) * a.in.q_token + (g * group + r % group) * a.in.q_head;
#pragma unroll
        for (int f = 0; f < kF; ++f) {
            const int d = kFp8 && (f | 1) < kF ? 64 * (f >> 1) + 16 * q + 8 * (f & 1) : 32 * f + 8 * q;
            __builtin_memcpy(&qf[nt][f], __builtin_assume_aligned(qrow + d, 16), 16);
            if (a.scale_log2 < 0.0f) qf[nt][f] = -qf[nt][f];  // the same scores from -q and the scale's magnitude
        }
    }
    const float scale = fabsf(a.scale_log2);
    f32x4 o[NT][D / 16];
    float m_run[NT], l_run[NT];  // l_run: of this lane's keys
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m_run[nt] = -INFINITY;
        l_run[nt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[nt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // A block's 16 keys share a page: a scalar address for them and an offset of the lane that never changes.
    const char* kbase = reinterpret_cast<const char*>(static_cast<const C*>(v.c.k) + g * v.c.k_head);
    const char* vbase = reinterpret_cast<const char*>(static_cast<const C*>(v.c.v) + g * v.c.v_head);
    const uint32_t k_off = static_cast<uint32_t>((l * v.c.k_slot + (kFp8 ? 16 : 8) * q) * sizeof(C));
    const uint32_t v_off = static_cast<uint32_t>((4 * q * v.c.v_slot + D / 16 * l) * sizeof(C));
    const uint32_t k_last = static_cast<uint32_t>((l * v.c.k_slot + 32 * (kF - 1) + 8 * q) * sizeof(C));  // fp8, an odd count of 32 dims
    for (int from = begin; from < end; from += kWindow) {
        const int until = min(end, from + kWindow), p0 = from >> v.page_shift;
        if (from > begin) __syncthreads();
        stage_pages(v, s.seq, from, until, pages);
        for (int kb = from + 32 * kw; kb < until && rb < n_rows; kb += 32 * kKeyWaves) {
            u32x4 kr[2][kFp8 ? (kF + 1) / 2 : kF];
            uint32_t vr[8][(kVB + 3) / 4];
            bool ok[2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                // rows of the page past the sequence's end are read and masked
                const int k0 = kb + 16 * tt;
                const int id = k0 < end ? __builtin_amdgcn_readfirstlane(pages[(k0 >> v.page_shift) - p0]) : -1;
                ok[tt] = id >= 0;
                const int64_t page = max(id, 0), slot = k0 & (v.c.page_size - 1);
                const char* kp = kbase + (page * v.c.k_page + slot * v.c.k_slot) * static_cast<int64_t>(sizeof(C));
#pragma unroll
                for (int f = 0; f < (kFp8 ? kF / 2 : kF); ++f) {
                    uint32_t x[4];
                    load_row_bytes<16, 16, RG == 1>(x, kp + 64 * f + k_off);
                    kr[tt][f] = u32x4{x[0], x[1], x[2], x[3]};
                }
                if constexpr (kFp8 && kF % 2) {
                    const u32x2 x = *reinterpret_cast<const u32x2*>(kp + k_last);
                    kr[tt][kF / 2] = u32x4{x[0], x[1], 0, 0};
                }
                const char* vp = vbase + (page * v.c.v_page + slot * v.c.v_slot) * static_cast<int64_t>(sizeof(C));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    vr[4 * tt + j][(kVB + 3) / 4 - 1] = 0;
                    load_row_bytes<kVB, kVAlign, RG == 1>(vr[4 * tt + j], vp + j * v.c.v_slot * static_cast<int64_t>(sizeof(C)) + v_off);
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // every load of the block is out before its first product
            const bool full = kb + 32 <= s.ctx && kb + 32 <= end && ok[0] && ok[1];
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
            float x[NT][8];
            bool moves = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int f = 0; f < kF; ++f) sc = F::mma16(kf[tt][f], qf[nt][f], sc);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[nt][4 * tt + i] = sc[i];
                }
                if (!full) {
                    uint32_t vis = visible32(a, s, tok[nt], kb);
                    if (!ok[0]) vis &= 0xFFFF0000u;
                    if (!ok[1]) vis &= 0x0000FFFFu;
                    vis >>= 4 * q;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!((vis >> (16 * (i >> 2) + (i & 3))) & 1)) x[nt][i] = -INFINITY;
                }
                float mx = x[nt][0];
#pragma unroll
                for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[nt][i]);
                moves |= mx * scale > m_run[nt] + kSlack;
            }
            if (__ballot(moves) != 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float mx = x[nt][0];
#pragma unroll
                    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[nt][i]);
                    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                    const float mn = fmaxf(m_run[nt], mx * scale);
                    const float f = m_run[nt] == mn ? 1.0f : __builtin_amdgcn_exp2f(m_run[nt] - mn);
                    l_run[nt] *= f;
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt) o[nt][dt] *= f;
                    m_run[nt] = mn;
                }
            }
            v8 ph[NT], pl[kLo ? NT : 1];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float base = m_run[nt] == -INFINITY ? 0.0f : m_run[nt] - kShift;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__fmaf_rn(x[nt][i], scale, -base));
                    ph[nt][i] = static_cast<T>(p);
                    if constexpr (kLo) {
                        l_run[nt] += p;
                        pl[nt][i] = static_cast<T>(p - static_cast<float>(ph[nt][i]));
                    } else if (i & 1) {
                        l_run[nt] = F::add2(ph[nt], i - 1, l_run[nt]);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // and V's transposition waits for V alone
            uint32_t vd[8][kVW];  // the value slices as pairs of T
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (kFp8) {
#pragma unroll
                    for (int i = 0; i < kVW; ++i) vd[j][i] = i % 2 ? F::from_fp8_hi(vr[j][i / 2]) : F::from_fp8(vr[j][i / 2]);
                } else {
                    __builtin_memcpy(vd[j], vr[j], kVB);
                }
            }
            if (!full) {  // rows that nobody sees may hold anything
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(ok[j >> 2] && kb + 16 * (j >> 2) + 4 * q + (j & 3) < s.total))
#pragma unroll
                        for (int i = 0; i < kVW; ++i) vd[j][i] = 0;
            }
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) {  // operand row l is dim D/16 l + dt of the lane's 8 keys
                u32x4 t;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    t[i] = __builtin_amdgcn_perm(vd[2 * i + 1][dt >> 1], vd[2 * i][dt >> 1], (dt & 1) ? 0x07060302u : 0x05040100u);
                const v8 vf = __builtin_bit_cast(v8, t);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    o[nt][dt] = F::mma16(vf, ph[nt], o[nt][dt]);
                    if constexpr (kLo) o[nt][dt] = F::mma16(vf, pl[nt], o[nt][dt]);
                }
            }
        }
    }

    // Lane (l, q) holds dims D/4 q + D/16 v + dt of row l in o[nt][dt][v].  A row tile of each row group at a time, its
    // key waves' threads in equal shares of a row.
    constexpr int kRowThreads = 4 * kKeyWaves, kPer = D / kRowThreads, kWaveRows = 64 / kRowThreads;
    const int in_group = threadIdx.x % (64 * kKeyWaves), mr = in_group / kRowThreads, d0 = kPer * (in_group % kRowThreads);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (16 * nt >= n_rows) break;
        float lr = l_run[nt];
        lr += __shfl_xor(lr, 16, 64);
        lr += __shfl_xor(lr, 32, 64);
        if (nt > 0) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int dt = 0; dt < D / 16; dt += 2) {
                float* at = &so[w][l * kRowF + D / 4 * q + D / 16 * i + dt];
                at[0] = o[nt][dt][i];
                at[1] = o[nt][dt + 1][i];
            }
        if (q == 0) sml[w][l] = float2{m_run[nt], lr};
        __syncthreads();
        const int r = rb + 16 * nt + mr;
        const bool live = r < n_rows;
        float mm = -INFINITY, ls = 0.0f;
        float acc[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] = 0.0f;
        for (int i = rg * kKeyWaves; i < (rg + 1) * kKeyWaves; ++i) mm = fmaxf(mm, sml[i][mr].x);
        for (int i = rg * kKeyWaves; i < (rg + 1) * kKeyWaves; ++i) {
            const float2 ml = sml[i][mr];
            if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // no key seen
            const float f = ml.x == mm ? 1.0f : __builtin_amdgcn_exp2f(ml.x - mm);
            ls += ml.y * f;
#pragma unroll
            for (int j = 0; j < kPer; ++j) acc[j] += so[i][mr * kRowF + d0 + j] * f;
        }
        const int t = s.first + (live ? r / group : 0), head = g * group + (live ? r % group : 0);
        const int64_t part = cp.part_of(a, range, t - s.first, head);
        // An infinite or NaN value makes the products NaN also in rows that do not see it, or with a weight that
        // rounds to 0: such rows start over on the vector ALUs, unless their scores are NaN.
        bool nan = false;
#pragma unroll
        for (int j = 0; j < kPer; ++j) nan |= acc[j] != acc[j];
        const uint64_t bad = __ballot(nan && live && ls == ls);
        constexpr uint64_t kRowLanes = (uint64_t{1} << kRowThreads) - 1;
        const bool mine = (bad >> (lane / kRowThreads * kRowThreads)) & kRowLanes;
        if (live && !mine) {
            if (part < 0) {
                const float inv = ls == 0.0f ? 0.0f : a.v_scale / ls;
                T h[kPer];
#pragma unroll
                for (int j = 0; j < kPer; ++j) h[j] = static_cast<T>(acc[j] * inv);
                T* out = static_cast<T*>(a.in.out) + static_cast<int64_t>(t) * a.in.out_token + head * a.in.out_head + d0;
                __builtin_memcpy(__builtin_assume_aligned(out, kPer % 8 == 0 ? 16 : 4), h, sizeof(h));
            } else {
                // 2^-kShift off the sum and the output, so that they belong to the maximum
                float* po = a.part_o + part * D + d0;
#pragma unroll
                for (int j = 0; j < kPer; j += 2) *reinterpret_cast<f32x2*>(po + j) = f32x2{acc[j], acc[j + 1]};
                if (d0 == 0) a.part_ml[part] = float2{mm - kShift, ls};
            }
        }
        if (__builtin_expect(bad != 0, 0)) {
#pragma unroll 1
            for (int rr = 0; rr < kWaveRows; ++rr) {
                if (!((bad >> (kRowThreads * rr)) & kRowLanes)) continue;
                const int br = rb + 16 * nt + kWaveRows * kw + rr;
                const RowState st = scan_row<T, C>(v, a, s, br / group, g * group + br % group, begin, end, lane, lanes_per_key(D), true);
                write_state<T>(v, a, s.first + br / group, g * group + br % group, cp.part_of(a, range, br / group, g * group + br % group), st, lane);
            }
        }
    }
}

// ---- many rows: keys through LDS -----------------------------------------------------------------
// A workgroup of 4 waves owns 128 rows (tokens x query heads of one kv head), 32 a wave, and walks the keys in tiles of 64,
// staged through LDS (two buffers, one barrier a tile):
//   * S^T = K Q^T on 32x32x16, the wave's queries in registers: a lane holds one row (lane % 32) and 16 of every 32
//     keys, the partner lane (lane ^ 32) the others;
//   * the weights go from the S registers into O^T += V^T P^T without leaving the lane (the k order of each 16-key
//     block is the order the lane holds its keys in).  Weights are rounded to the operands' type once, half a step, of
//     either sign, and their sum, in fp32, is of the rounded ones.  As hi + lo they would bring the 2-norm of f16 outputs'
//     errors from 2.8e-4 to the outputs' own rounding, 2.1e-4, and 63-node trees from 91 to 122 us (500 tokens: 44 to 57);
//   * the next tile's scores are formed beside this tile's weights, so keys are copied two tiles ahead, values one;
//   * the lanes keep sums of their own; maxima are exchanged only when the running one moves (kSlack).
// Wave w stages keys 16 w .. 16 w + 15 of a tile, which share a page: a scalar address and lane offsets that never change,
// copied straight into LDS (global_load_lds; an fp8 cache goes through registers, converted on the way).  Both K
// and V lie as they are in memory, with the 16-byte pieces of a row exchanged by its number (TileGeom) so that neither the
// key fragments (16 rows, one piece) nor V's transposing reads (ds_read_b64_tr_b16: half a wave takes four pieces of 4
// rows) meet on a bank.
// Bound by what one or two waves a SIMD can have under way, and in short calls by the start (plan, queries, first tile: 10 us)
// and the partial results.  63-node trees of eight users, 64 heads of 128 over up to 8191 keys (66 GFLOP): 91-93 us, matrix
// cores busy for 33 % of the SIMDs' cycles and vector ALUs for 35 %; chunks of up to 500 tokens, 32 heads of 64 (16 GFLOP):
// 44 us, 14 and 34 % with 1.2 waves a SIMD in the mean (the same buffers in every pass, without the join).  The kv heads come fastest in the grid: with 8 of them
// (or 16, ..) the row tiles of one meet on one XCD and its keys in one L2.
constexpr int kTileRows = 128, kTileKeys = 64;

template <int D>
struct TileGeom {
    static constexpr int kTileE = kTileKeys * D;      // elements of one staged tile
    static constexpr int kBuf = 2 * kTileE;           // K and V
    static constexpr size_t kLds = 2 * static_cast<size_t>(kBuf) * 2;
    static constexpr int kChunks = D / 8, kPieces = D / 32;  // 16-byte pieces of a row; of 16 rows, per lane
    // what the piece number is XORed with
    static __device__ __forceinline__ int swap_k(int row) { return D == 64 ? (row >> 1) & 7 : D == 96 ? (row >> 2) & 3 : row & 15; }
    static __device__ __forceinline__ int swap_v(int row) { return D == 64 ? ((row >> 1) & 1) << 2 : D == 96 ? 0 : (row & 3) << 2; }
};

extern __shared__ __align__(16) uint16_t tile_lds[];

typedef short s16x4 __attribute__((ext_vector_type(4)));
using LdsPtr = __attribute__((address_space(3))) uint16_t*;

// 16 bytes per lane from base + off into LDS at m0 + 16 lane
__device__ __forceinline__ void copy_to_lds(const void* base, uint32_t off, uint32_t lds) {
    __asm__ volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}

template <class T, class C, int D>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void attention_tile_kernel(View v, AttnArgs a) {
    using F = Frag<T>;
    using v8 = typename F::v8;
    using G = TileGeom<D>;
    constexpr bool kFp8 = std::is_same_v<C, Fp8>;
    __shared__ int has_page[4][4];  // [tile % 4][16 keys], kept where a page of the range is missing
    const int kvh = v.c.kv_heads, group = a.in.heads / kvh;
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    CallPlan<kTileRows, kTileKeys> cp;
    if (!cp.find(v, a, static_cast<int>(blockIdx.x), lane)) return;
    const int g = cp.block % kvh, rest = cp.block / kvh;
    const int tiles = cp.tiles, tile = rest % tiles, range = rest / tiles;
    const Span s = span_of(v, a, cp.seq);
    const int kps = cp.keys, begin = range * kps;
    const int n_rows = cp.rows * group, r0 = tile * kTileRows, rw = r0 + 32 * w;
    const int last = (min(r0 + kTileRows, n_rows) - 1) / group;
    if (g == 0 && range == 0 && a.cut)
        for (int t = r0 / group + tid; t <= last; t += kThreads) a.cut[s.first + t] = cp.cut_of(t);
    const int n_keys = a.in.mask ? s.total : min(s.total, s.ctx + last + 1);
    const int end = min(n_keys, begin + kps);
    // row rw + l32; rows past the last repeat it
    const bool row_live = rw + l32 < n_rows;
    const int r = min(rw + l32, n_rows - 1), i = r / group, head = g * group + r % group;
    const int64_t part = cp.part_of(a, range, i, head);
    if (begin >= end && range > 0) {  // keys of later rows only
        if (row_live && h == 0) a.part_ml[part] = float2{-INFINITY, 0.0f};
        return;
    }

    // a negative scale: the same scores from -q and its magnitude
    const float scale = fabsf(a.scale_log2);
    v8 qf[D / 16];
    {
        const T* qrow = static_cast<const T*>(a.in.q) + static_cast<int64_t>(s.first + i) * a.in.q_token + head * a.in.q_head + 8 * h;
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
            __builtin_memcpy(&qf[db], __builtin_assume_aligned(qrow + 16 * db, 16), 16);
            if (a.scale_log2 < 0.0f) qf[db] = -qf[db];
        }
    }
    const C* kbase = static_cast<const C*>(v.c.k) + g * v.c.k_head;
    const C* vbase = static_cast<const C*>(v.c.v) + g * v.c.v_head;

    // Piece 64 j + lane of the wave's 16 rows.  At head_dim 256 (128 of an fp8 cache) the offsets (and the fragments' addresses below) are formed
    // anew in every step: kept, they are 40 registers that the accumulators then spill.
    constexpr bool kKeep = D <= (kFp8 ? 96 : 128);
    auto offset_of = [&](int j, int at, int64_t slot, bool keys) {
        const int row = (64 * j + at) / G::kChunks, pos = (64 * j + at) % G::kChunks;
        return static_cast<uint32_t>((row * static_cast<int>(slot) + 8 * (pos ^ (keys ? G::swap_k(row) : G::swap_v(row)))) * static_cast<int>(sizeof(C)));
    };
    auto fresh = [](int x) {  // the same value, not to be kept from step to step
        if constexpr (!kKeep) __asm__("" : "+v"(x));
        return x;
    };
    uint32_t k_off[kKeep ? G::kPieces : 1], v_off[kKeep ? G::kPieces : 1];
    if constexpr (kKeep)
#pragma unroll
        for (int j = 0; j < G::kPieces; ++j) {
            k_off[j] = offset_of(j, lane, v.c.k_slot, true);
            v_off[j] = offset_of(j, lane, v.c.v_slot, false);
        }
    uint16_t* const mine = tile_lds + 16 * w * D;  // of buffer 0's K
    const uint32_t mine_at = __builtin_amdgcn_readfirstlane(reinterpret_cast<uintptr_t>((LdsPtr)mine));
    const int n_tiles = (end - begin + kTileKeys - 1) / kTileKeys;
    auto key_of = [&](int t) { return begin + kTileKeys * t + 16 * w; };  // the wave's first key of tile t
    // Its page's entry of the table; rows of a page past the sequence's end are read and masked.  A vector load: the
    // LDS reads of a step would wait for a scalar one, whose result is due two steps later.
    int zero = 0;
    __asm__("" : "+v"(zero));
    auto entry = [&](int t) {
        const int p = min(key_of(t) >> v.page_shift, v.c.table_width - 1);
        return v.c.table[static_cast<int64_t>(s.seq) * v.c.table_stride + (p + zero)];
    };
    auto usable = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(v.c.num_pages); };
    auto page = [&](int id) {
        const int u = __builtin_amdgcn_readfirstlane(id);
        return static_cast<int64_t>(usable(u) ? u : 0);
    };
    bool missing = false;  // does the range miss a page?
    u32x2 kr[kFp8 ? G::kPieces : 1], vr[kFp8 ? G::kPieces : 1];
    auto load_k = [&](int t, int id) {
        const C* p = kbase + page(id) * v.c.k_page + (key_of(t) & (v.c.page_size - 1)) * v.c.k_slot;
        const int at = fresh(lane);
#pragma unroll
        for (int j = 0; j < G::kPieces; ++j) {
            const uint32_t off = kKeep ? k_off[kKeep ? j : 0] : offset_of(j, at, v.c.k_slot, true);
            if constexpr (kFp8) kr[j] = *reinterpret_cast<const u32x2*>(reinterpret_cast<const char*>(p) + off);
            else copy_to_lds(p, off, mine_at + 2 * ((t & 1) * G::kBuf) + 1024 * j);
        }
    };
    auto load_v = [&](int t, int id) {
        const C* p = vbase + page(id) * v.c.v_page + (key_of(t) & (v.c.page_size - 1)) * v.c.v_slot;
        const int at = fresh(lane);
#pragma unroll
        for (int j = 0; j < G::kPieces; ++j) {
            const uint32_t off = kKeep ? v_off[kKeep ? j : 0] : offset_of(j, at, v.c.v_slot, false);
            if constexpr (kFp8) vr[j] = *reinterpret_cast<const u32x2*>(reinterpret_cast<const char*>(p) + off);
            else copy_to_lds(p, off, mine_at + 2 * ((t & 1) * G::kBuf + G::kTileE) + 1024 * j);
        }
    };
    auto wide = [](u32x2 x) { return u32x4{F::from_fp8(x[0]), F::from_fp8_hi(x[0]), F::from_fp8(x[1]), F::from_fp8_hi(x[1])}; };
    auto land_k = [&](int t) {
        if constexpr (kFp8)
#pragma unroll
            for (int j = 0; j < G::kPieces; ++j) *reinterpret_cast<u32x4*>(mine + (t & 1) * G::kBuf + 8 * lane + 512 * j) = wide(kr[j]);
    };
    // zeros for the values of rows that nobody sees, which may hold anything
    auto land_v = [&](int t, int id) {
        uint16_t* sv = mine + (t & 1) * G::kBuf + G::kTileE + 8 * lane;
        if constexpr (kFp8) {
#pragma unroll
            for (int j = 0; j < G::kPieces; ++j) *reinterpret_cast<u32x4*>(sv + 512 * j) = wide(vr[j]);
        } else {
            __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");  // and the keys'
        }
        if (key_of(t) + 16 > s.total || missing || t == 0) {  // tile 0 lands before `missing` is known
#pragma unroll
            for (int j = 0; j < G::kPieces; ++j)
                if (!usable(id) || key_of(t) + (64 * j + lane) / G::kChunks >= s.total) *reinterpret_cast<u32x4*>(sv + 512 * j) = u32x4{0, 0, 0, 0};
        }
    };

    // fragment addresses within a buffer: key row l32, piece 2 db + h; and, of the lane's 16, key 4 h + lane / 4, dims
    // 16 (l32 / 16) + 4 (lane % 4) of every 32
    const int kx = h ^ G::swap_k(l32);
    const uint16_t* k_row = tile_lds + l32 * D;
    const int vrow = 4 * h + ((lane & 15) >> 2), vx = (2 * (l32 >> 4) + ((lane & 3) >> 1)) ^ G::swap_v(vrow);
    const uint16_t* v_row = tile_lds + G::kTileE + vrow * D + 4 * (lane & 1);

    f32x16 o[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;
    const bool live = rw < n_rows;  // waves without rows only stage

    // register e of half hh is key 32 hh + 8 (e / 4) + 4 h + e % 4 of row l32
    auto scores = [&](int t, f32x16 (&x)[2]) {
        const uint16_t* sk = k_row + (t & 1) * G::kBuf;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[hh][e] = 0.0f;
#pragma unroll
            for (int db = 0; db < D / 16; ++db) {
                v8 kf;
                __builtin_memcpy(&kf, __builtin_assume_aligned(sk + 32 * hh * D + 8 * ((2 * db) ^ kx), 16), 16);
                x[hh] = F::mma32(kf, qf[db], x[hh]);
            }
        }
    };
    // Tile t, whose scores are in x, while the scores of the next are formed in y.  Its keys are two tiles ahead
    // of the copies, its values one.
    auto step = [&](int t, f32x16 (&x)[2], f32x16 (&y)[2], int& id1, int& id2) {
        const int id3 = entry(t + 3);
        if (t + 1 < n_tiles) load_v(t + 1, id1);
        if (t + 2 < n_tiles) {
            load_k(t + 2, id2);
            if (missing && lane == 0) has_page[(t + 2) & 3][w] = usable(id2);
        }
        if (live) {
            const int kb = begin + kTileKeys * t;
            if (kb + kTileKeys > s.ctx || kb + kTileKeys > end || missing) {
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    uint32_t vis = visible32(a, s, i, kb + 32 * hh);
                    if (missing) {
                        if (!has_page[t & 3][2 * hh]) vis &= 0xFFFF0000u;
                        if (!has_page[t & 3][2 * hh + 1]) vis &= 0x0000FFFFu;
                    }
                    vis >>= 4 * h;
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (!((vis >> (8 * (e >> 2) + (e & 3))) & 1)) x[hh][e] = -INFINITY;
                }
            }
            float mx = x[0][0];
#pragma unroll
            for (int e = 1; e < 32; ++e) mx = fmaxf(mx, x[e >> 4][e & 15]);
            mx *= scale;
            if (__ballot(mx > m_run + kSlack) != 0) {
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float mn = fmaxf(m_run, mx);
                const float f = m_run == mn ? 1.0f : __builtin_amdgcn_exp2f(m_run - mn);
                l_run *= f;
#pragma unroll
                for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[dt][e] *= f;
                m_run = mn;
            }
            const float base = m_run == -INFINITY ? 0.0f : m_run - kShift;
            // The next tile's scores (past the last tile: of stale keys, unused), this tile's weights and its second
            // product, in steps of one matrix instruction whose order the compiler keeps: left alone, it lets every
            // product wait for its own LDS read and the weights wait for the products.  Fragments are read kAhead
            // products ahead; a third of the weights is left for the second product's steps.
            constexpr int kM = D / 8, kPerB = D / 32, kAhead = 4;
            const uint16_t* sk = k_row + ((t + 1) & 1) * G::kBuf;
            const uint16_t* sv = v_row + (t & 1) * G::kBuf;
            const int kxs = fresh(kx), vxs = fresh(vx);
            v8 kf[kM], vf[kM], pf[4];
            auto read_k = [&](int n) {
                __builtin_memcpy(&kf[n], __builtin_assume_aligned(sk + 32 * (n & 1) * D + 8 * ((2 * (n >> 1)) ^ kxs), 16), 16);
            };
            auto read_v = [&](int n) {
                const uint16_t* at = sv + 16 * (n / kPerB) * D + 8 * ((4 * (n % kPerB)) ^ vxs);
                const s16x4 f0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
                const s16x4 f1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 8 * D));
                vf[n] = __builtin_bit_cast(v8, __builtin_shufflevector(f0, f1, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            auto weight = [&](int e) {
                const float p = __builtin_amdgcn_exp2f(__fmaf_rn(x[e >> 4][e & 15], scale, -base));
                pf[e >> 3][e & 7] = static_cast<T>(p);
                if (e & 1) l_run = F::add2(pf[e >> 3], (e & 7) - 1, l_run);
            };
            constexpr int kFirst = 20;  // weights beside the first product
#pragma unroll
            for (int n = 0; n < kAhead; ++n) read_k(n);
            __builtin_amdgcn_s_setprio(1);  // before a wave that masks or rescales (500 tokens of head_dim 64: 43.4 us, 45.7 without)
#pragma unroll
            for (int n = 0; n < kM; ++n) {
                if (n + kAhead < kM) read_k(n + kAhead);
                else read_v(n + kAhead - kM);
                if (n < 2)
#pragma unroll
                    for (int e = 0; e < 16; ++e) y[n][e] = 0.0f;
                y[n & 1] = F::mma32(kf[n], qf[n >> 1], y[n & 1]);
#pragma unroll
                for (int e = kFirst * n / kM; e < kFirst * (n + 1) / kM; ++e) weight(e);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int n = 0; n < kM; ++n) {
                if (n + kAhead < kM) read_v(n + kAhead);
                o[n % kPerB] = F::mma32(vf[n], pf[n / kPerB], o[n % kPerB]);
#pragma unroll
                for (int e = kFirst + (32 - kFirst) * 2 * n / kM; e < kFirst + (32 - kFirst) * 2 * (n + 1) / kM && e < 32; ++e) weight(e);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if (t + 2 < n_tiles) land_k(t + 2);
        if (t + 1 < n_tiles) land_v(t + 1, id1);
        __syncthreads();
        id1 = id2;
        id2 = id3;
    };

    if (n_tiles > 0) {
        int id0 = entry(0), id1 = entry(1), id2 = entry(2);
        for (int p = (begin >> v.page_shift) + tid; p <= (end - 1) >> v.page_shift; p += kThreads)
            missing |= page_of(v, s.seq, p << v.page_shift) < 0;
        load_k(0, id0);
        load_v(0, id0);
        if (!kFp8 && n_tiles > 1) load_k(1, id1);
        land_k(0);
        land_v(0, id0);
        missing = __syncthreads_or(missing);
        if (missing && lane == 0) {
            has_page[0][w] = usable(id0);
            has_page[1][w] = usable(id1);
        }
        if (kFp8 && n_tiles > 1) load_k(1, id1);
        f32x16 xa[2], xb[2];
        if (live) scores(0, xa);
        if (kFp8 && n_tiles > 1) land_k(1);
        __syncthreads();
        for (int t = 0; t < n_tiles; t += 2) {
            step(t, xa, xb, id1, id2);
            if (t + 1 < n_tiles) step(t + 1, xb, xa, id1, id2);
        }
    }
    if (!live) return;
    l_run += __shfl_xor(l_run, 32, 64);
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) nan |= o[dt][e] != o[dt][e];
    uint64_t bad = __ballot(nan && row_live && l_run == l_run);  // as in attention_rows_kernel
    bad = (bad | bad >> 32) & 0xFFFFFFFFu;
    // Out through the wave's quarter of LDS (its last tile's barrier is behind every wave), so that a store covers whole rows,
    // not 16 bytes of each: 16-byte pieces, exchanged by the row's number against bank conflicts.
    const float inv = part < 0 ? (l_run == 0.0f ? 0.0f : a.v_scale / l_run) : 1.0f;
    float* mine_f = reinterpret_cast<float*>(tile_lds) + 32 * D * w;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 x = {o[dt][4 * q4] * inv, o[dt][4 * q4 + 1] * inv, o[dt][4 * q4 + 2] * inv, o[dt][4 * q4 + 3] * inv};
            *reinterpret_cast<f32x4*>(mine_f + l32 * D + 4 * ((8 * dt + 2 * q4 + h) ^ (l32 & 7))) = x;
        }
    wave_lds_sync();
    if (part >= 0 && row_live && h == 0 && !((bad >> l32) & 1)) a.part_ml[part] = float2{m_run - kShift, l_run};
    const int n_wave = min(n_rows - rw, 32);
    if (cp.ranges == 1) {
        for (int u = lane; u < n_wave * G::kChunks; u += 64) {
            const int row = u / G::kChunks, c = u % G::kChunks, ri = (rw + row) / group, rh = g * group + (rw + row) % group;
            if ((bad >> row) & 1) continue;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(mine_f + row * D + 4 * ((2 * c) ^ (row & 7)));
            const f32x4 hi = *reinterpret_cast<const f32x4*>(mine_f + row * D + 4 * ((2 * c + 1) ^ (row & 7)));
            v8 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = static_cast<T>(lo[e]);
                x[4 + e] = static_cast<T>(hi[e]);
            }
            *reinterpret_cast<v8*>(static_cast<T*>(a.in.out) + static_cast<int64_t>(s.first + ri) * a.in.out_token + rh * a.in.out_head + 8 * c) = x;
        }
    } else {
        for (int u = lane; u < n_wave * (D / 4); u += 64) {
            const int row = u / (D / 4), c = u % (D / 4), ri = (rw + row) / group, rh = g * group + (rw + row) % group;
            if ((bad >> row) & 1) continue;
            *reinterpret_cast<f32x4*>(a.part_o + cp.part_of(a, range, ri, rh) * D + 4 * c) =
                *reinterpret_cast<const f32x4*>(mine_f + row * D + 4 * (c ^ (row & 7)));
        }
    }
    while (__builtin_expect(bad != 0, 0)) {
        const int br = rw + __builtin_ctzll(bad), bi = br / group, bh = g * group + br % group;
        bad &= bad - 1;
        const RowState st = scan_row<T, C>(v, a, s, bi, bh, begin, end, lane, lanes_per_key(D), true);
        write_state<T>(v, a, s.first + bi, bh, cp.part_of(a, range, bi, bh), st, lane);
    }
}

// Joins the ranges of each row: D / 4 threads hold a row's output and `sg` such groups share its ranges, four of
// them requested at once; the groups are added in order through LDS.  A few rows of many ranges wait for one or two round
// trips to memory that way (42 tokens of 32 heads, 37 ranges: 10.6 us with one group).  Block (x, y): token, heads.
template <class T, bool kPlanned>
__global__ __launch_bounds__(kThreads) void attention_merge_kernel(View v, AttnArgs a, int sg) {
    __shared__ f32x4 so[kThreads];
    __shared__ float2 sml[kThreads];
    const int t = blockIdx.x, D = v.c.head_dim, per = D / 4, rows = kThreads / per / sg, lane = threadIdx.x & 63;
    int4 cut = {0, 0, 0, 0};
    if constexpr (kPlanned) cut = a.cut[t];  // not written for a token of no sequence, or past max_new
    const int seq = sequence_of(v, t, lane);
    if (seq >= v.c.batch || t < v.c.cu[seq]) return;
    if constexpr (kPlanned) {
        if (t - max(v.c.cu[seq], 0) >= a.in.max_new) return;
    } else {
        const Span s = span_of(v, a, seq);
        cut = int4{s.total > 0 ? (s.total - 1) / a.kps + 1 : 0, t, a.in.tokens, 0};
    }
    if (cut.x <= 1) return;  // written by the range itself
    if (kPlanned && (cut.y < 0 || cut.z < 1 || cut.y + static_cast<int64_t>(cut.x - 1) * cut.z >= a.parts)) return;  // nor where cu descends
    const int n = cut.x;
    int64_t row = static_cast<int64_t>(cut.y) * a.in.heads;
    const int64_t step = static_cast<int64_t>(cut.z) * a.in.heads;  // between ranges
    const int slot = threadIdx.x / per, d0 = 4 * (threadIdx.x % per), gi = slot % sg, head = blockIdx.y * rows + slot / sg;
    const bool live = slot < rows * sg && head < a.in.heads;
    row += live ? head : 0;
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 4 * gi; live && c0 < n; c0 += 4 * sg) {
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
    if (sg > 1) {
        so[threadIdx.x] = o;
        sml[threadIdx.x] = float2{m, l};
        __syncthreads();
        if (gi != 0) return;
        for (int i = 1; live && i < sg; ++i) {
            const float2 x = sml[threadIdx.x + i * per];
            if (x.y == 0.0f) continue;
            const f32x4 xo = so[threadIdx.x + i * per];
            const float mn = fmaxf(m, x.x);
            const float f = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn), w = x.x == mn ? 1.0f : __builtin_amdgcn_exp2f(x.x - mn);
            l = l * f + x.y * w;
            if (f > 0.0f) o *= f;
            else o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (!(w <= 0.0f)) o += xo * w;
            m = mn;
        }
    }
    if (!live) return;
    T h[4];
    const float inv = a.v_scale / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = static_cast<T>(l == 0.0f ? 0.0f : o[i] * inv);
    T* out = static_cast<T*>(a.in.out) + static_cast<int64_t>(t) * a.in.out_token + head * a.in.out_head + d0;
    if (kPlanned) __builtin_memcpy(__builtin_assume_aligned(out, 8), h, 8);  // such a call's operands are aligned
    else
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = h[i];
}

// ---- host side -------------------------------------------------------------------------------
// Which kernel serves a call, by the rows (tokens x query heads) that share a kv head, and how its keys are cut.  Up to 64 rows go
// straight into registers: an fp8 cache is then converted where it is used (52 rows, 57000 keys: 48.5 us, 55.0 through LDS),
// short calls start sooner (64 rows, 900 keys: 16.1 / 18.1; 28 rows: 14.0 / 16.7), the others are even (52 rows, f16: 38.1 / 38.7)
// but for many sequences (16 of 64 rows and 2000 keys: 36.5 / 32.7).
enum class Kind { kLanes, kRows, kTile };
struct Plan {
    Kind kind;
    int row_tiles;      // of 16 rows (kRows)
    int kps, splits;    // kLanes
    int slots;          // the others: workgroups to cut the call into ..
    int64_t blocks;     // .. and what that makes at most
    bool merge;
    int64_t most_ranges;  // of a sequence
    int64_t parts;      // partial rows at most
    size_t o_bytes, ml_bytes, bytes;
};

bool matrix_operands(const View& v, const qmm_paged_query& in) {
    const int D = v.c.head_dim;
    if ((D != 64 && D != 96 && D != 128 && D != 256) || v.c.page_size < 16 || v.c.num_pages == 0) return false;
    const uint64_t els = static_cast<uint64_t>(v.c.k_page | v.c.k_head | v.c.k_slot | v.c.v_page | v.c.v_head | v.c.v_slot);
    const uint64_t rows = static_cast<uint64_t>(in.q_token | in.q_head | in.out_token | in.out_head);
    const uint64_t ptr = reinterpret_cast<uintptr_t>(v.c.k) | reinterpret_cast<uintptr_t>(v.c.v) | reinterpret_cast<uintptr_t>(in.q) |
                         reinterpret_cast<uintptr_t>(in.out);
    // 16 slots are within 2^31 bytes of each other
    for (int64_t slot : {v.c.k_slot, v.c.v_slot})
        if (slot < 0 || slot >= 1 << 25) return false;
    return els % (v.c.dtype == QMM_DTYPE_E4M3 ? 16 : 8) == 0 && rows % 8 == 0 && ptr % 16 == 0;
}

// Calls f with the kernel that serves a plan's kind, row tiles and the call's types.
template <class T, class C, int D, class Fn>
auto with_matrix_kernel(Kind kind, int row_tiles, Fn f) {
    if (kind == Kind::kTile) return f(attention_tile_kernel<T, C, D>, TileGeom<D>::kLds);
    if constexpr (D <= 128) {
        if (row_tiles == 2) return f(attention_rows_kernel<T, C, D, 2, 1>, size_t{0});
        if (row_tiles > 2) return f(attention_rows_kernel<T, C, D, 2, 2>, size_t{0});
    }
    return f(attention_rows_kernel<T, C, D, 1, 1>, size_t{0});
}

template <class Fn>
auto with_matrix_kernel(const View& v, const qmm_paged_query& in, Kind kind, int row_tiles, Fn f) {
    auto types = [&](auto tc, auto cc) {
        using T = decltype(tc);
        using C = decltype(cc);
        switch (v.c.head_dim) {
            case 64: return with_matrix_kernel<T, C, 64>(kind, row_tiles, f);
            case 96: return with_matrix_kernel<T, C, 96>(kind, row_tiles, f);
            case 128: return with_matrix_kernel<T, C, 128>(kind, row_tiles, f);
            default: return with_matrix_kernel<T, C, 256>(kind, row_tiles, f);
        }
    };
    const bool fp8 = v.c.dtype == QMM_DTYPE_E4M3;
    if (in.dtype == QMM_DTYPE_F16) return fp8 ? types(_Float16{}, Fp8{}) : types(_Float16{}, _Float16{});
    return fp8 ? types(__bf16{}, Fp8{}) : types(__bf16{}, __bf16{});
}

// Workgroups of a kernel that run at once, asked for once per kernel and device.
template <class K>
int kernel_slots(K kern, size_t lds) {
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, int> known;
    const void* fn = reinterpret_cast<const void*>(kern);
    int per_cu = 0, dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess) {
        (void)hipGetLastError();
        return 256;  // without a device: argument checks only
    }
    std::lock_guard<std::mutex> lock(mu);
    const auto it = known.find({fn, dev});
    if (it != known.end()) return it->second;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        (lds > 65536 && hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)) != hipSuccess) ||
        hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kern, kThreads, lds) != hipSuccess || per_cu < 1 || cus < 1) {
        (void)hipGetLastError();
        return 256;
    }
    return known[{fn, dev}] = per_cu * cus;
}

Plan plan(const View& v, const qmm_paged_query& in) {
    Plan p{};
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(static_cast<int64_t>(v.c.table_width) * v.c.page_size, INT32_MAX - 65536));
    const int64_t rows = static_cast<int64_t>(in.tokens) * in.heads;
    const int64_t per_kv = static_cast<int64_t>(std::min(in.max_new, in.tokens)) * (in.heads / v.c.kv_heads);
    const int kvh = v.c.kv_heads;
    if (!matrix_operands(v, in) || per_kv > (1 << 28)) {
        p.kind = Kind::kLanes;
        int64_t kps = 64;
        while (kps < most && (rows * ((most + kps - 1) / kps) > 16384 || (most + kps - 1) / kps > 1024)) kps *= 2;
        // a length that no longer fits its 32 bits is past `most`: one range takes everything
        p.kps = static_cast<int>(std::min<int64_t>(kps, INT32_MAX));
        p.splits = static_cast<int>((most + kps - 1) / kps);
        p.merge = p.splits > 1;
        p.most_ranges = p.splits;
        p.parts = rows * p.splits;
    } else {
        // more row tiles of head_dim 256 do not fit a wave's registers
        p.kind = per_kv <= (v.c.head_dim <= 128 ? 64 : 16) ? Kind::kRows : Kind::kTile;
        const bool few = p.kind == Kind::kRows;
        p.row_tiles = few ? static_cast<int>((per_kv + 15) / 16) : 0;
        p.slots = with_matrix_kernel(v, in, p.kind, p.row_tiles, [](auto kern, size_t lds) { return kernel_slots(kern, lds); });
        // A plan's ranges are cut by a length of at least `least` keys.  With W steps in all and u >= W / slots steps a
        // range, the ranges of all row tiles are at most 2 W / u and one more per row tile (a chain's last tile sees up to
        // twice the mean), and those of sequences with more than one range at most twice that, 4 slots.
        const int64_t least = few ? kRowsStep : kTileKeys * CallPlan<kTileRows, kTileKeys>::kMinSteps;
        const int64_t most_ranges = p.most_ranges = (most + least - 1) / least;
        const int64_t seqs = std::min(v.c.batch, in.tokens);
        const int64_t items = kvh * (few ? seqs : seqs + (static_cast<int64_t>(in.tokens) * (in.heads / kvh) + kTileRows - 1) / kTileRows);
        p.blocks = std::min(items * most_ranges, 2 * static_cast<int64_t>(p.slots) + items);
        p.merge = most_ranges > 1;
        const int64_t tile_rows = few ? 16 * p.row_tiles : kTileRows;
        p.parts = std::min(rows * most_ranges, 4 * static_cast<int64_t>(p.slots) * tile_rows);
    }
    if (p.merge) {
        p.o_bytes = static_cast<size_t>(p.parts) * v.c.head_dim * sizeof(float);
        p.ml_bytes = (static_cast<size_t>(p.parts) * sizeof(float2) + 15) / 16 * 16;
        p.bytes = p.o_bytes + p.ml_bytes + static_cast<size_t>(in.tokens) * sizeof(int4);
    }
    return p;
}

// What a score in base 2 is of the product with the stored key.
float score_scale(const View& v, const qmm_paged_query& in) {
    const float scale = in.scale != 0.0f ? in.scale : 1.0f / std::sqrt(static_cast<float>(v.c.head_dim));
    return scale * v.c.k_scale * 1.4426950408889634f;
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
    if (!std::isnormal(score_scale(*v, *in))) return bad("scale * k_scale is out of fp32's range.");
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
    a.scale_log2 = score_scale(v, *in);
    a.v_scale = v.c.v_scale;
    a.kps = p.kps;
    a.slots = p.slots;
    a.part_o = static_cast<float*>(workspace);
    a.parts = p.parts / in->heads;
    if (p.merge) {
        a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + p.o_bytes);
        a.cut = reinterpret_cast<int4*>(static_cast<char*>(workspace) + p.o_bytes + p.ml_bytes);
    }
    if (p.kind == Kind::kLanes) {
        const dim3 grid(static_cast<unsigned>(in->tokens), static_cast<unsigned>(p.splits), static_cast<unsigned>((in->heads + 3) / 4));
        const int aligned = operands_aligned(v, *in) ? 1 : 0;
        auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, stream, v, a, aligned); };
        const bool fp8 = v.c.dtype == QMM_DTYPE_E4M3;
        if (in->dtype == QMM_DTYPE_F16) fp8 ? go(attention_lanes_kernel<_Float16, Fp8>) : go(attention_lanes_kernel<_Float16, _Float16>);
        else fp8 ? go(attention_lanes_kernel<__bf16, Fp8>) : go(attention_lanes_kernel<__bf16, __bf16>);
    } else {
        if (p.blocks > INT32_MAX) return bad("too many sequences, heads and tokens for one call.");
        with_matrix_kernel(v, *in, p.kind, p.row_tiles, [&](auto kern, size_t lds) {
            hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(p.blocks)), dim3(kThreads), lds, stream, v, a);
        });
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return launched(e, "paged attention kernel launch");
    if (p.merge) {
        const int groups = kThreads / (v.c.head_dim / 4);
        int sg = 1;
        while (2 * sg <= groups && 4 * sg < p.most_ranges && static_cast<int64_t>(in->tokens) * in->heads * sg < 8192) sg *= 2;
        const int rows = groups / sg;
        const dim3 mgrid(static_cast<unsigned>(in->tokens), static_cast<unsigned>((in->heads + rows - 1) / rows));
        auto merge = [&](auto tc) {
            using T = decltype(tc);
            auto go = [&](auto kern) { hipLaunchKernelGGL(kern, mgrid, dim3(kThreads), 0, stream, v, a, sg); };
            if (p.kind == Kind::kLanes) go(attention_merge_kernel<T, false>);
            else go(attention_merge_kernel<T, true>);
        };
        in->dtype == QMM_DTYPE_F16 ? merge(_Float16{}) : merge(__bf16{});
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
