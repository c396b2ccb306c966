// Writing and moving the rows of a paged key/value cache: the append of new tokens with the position
// rotation on the way, the commit of a drafted tree's accepted path, and the reordering of a beam
// search's sequences.  All three are bound by memory traffic (each row read once and written once) and, for
// a decode step's few rows, by the chain of dependent loads cu -> ctx -> table -> row.
#include "qmm_paged.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace qmm {
namespace paged {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;  // rotary_dim <= 256

// ---- append ------------------------------------------------------------------------------------
// Angles in turns as 64-bit fractions: pair i turns by pos * turn[i] mod 2^64 (of 2^64 a turn).  The
// product wraps exactly, so a position of 10^6 loses 20 of the 64 bits and no more; the remaining fraction
// is rounded to fp32 once.
struct RopeTurns {
    uint64_t turn[kMaxPairs];
};

__device__ __forceinline__ float2 cos_sin(uint64_t turn, int pos) {
    const uint64_t f = turn * static_cast<uint64_t>(static_cast<int64_t>(pos));
    // the signed top 32 bits: [-1/2, 1/2) of a turn
    const float half_turns = static_cast<float>(static_cast<int32_t>(f >> 32)) * 0x1p-31f;
    float s, c;
    sincospif(half_turns, &s, &c);
    return float2{c, s};
}

struct AppendArgs {
    qmm_paged_new in;
    float k_div, v_div;    // E4M3: what the value is divided by ...
    float k_mul, v_mul;    // ... or multiplied by, where the scale is a power of two (exact)
    int k_exact, v_exact;
    int units_rot, units_v, units, per_block;
};

template <class T>
struct Vec8;
template <>
struct Vec8<_Float16> {
    using type = f16x8;
};
template <>
struct Vec8<__bf16> {
    using type = bf16x8;
};

// 8 fp32 values of a K or V row, scaled and rounded to the cache's type
template <class T, bool kFp8>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&x)[8], float div, float mul, int exact) {
    if constexpr (kFp8) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = clamp_e4m3(exact ? x[e] * mul : x[e] / div);
        *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(base) + at) =
            u32x2{pack_e4m3(y[0], y[1], y[2], y[3]), pack_e4m3(y[4], y[5], y[6], y[7])};
    } else {
        typename Vec8<T>::type o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = static_cast<T>(x[e]);
        *reinterpret_cast<typename Vec8<T>::type*>(static_cast<T*>(base) + at) = o;
    }
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const auto v = *reinterpret_cast<const typename Vec8<T>::type*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(v[e]);
}

// Memory-bound: 6818 tokens of 80 heads of 128 (279 MB) in 55.7 us, 5.0 TB/s; a decode step's few tokens are bound by the chain of
// loads (8 tokens: 4.1 us).  One block per (token, range of units).  A unit is 8 dimensions of a query, key or value head, or, for
// rotated (i, i + half) pairs, 8 of the first half with their 8 partners; units of the rotated heads (q
// then k) come first.  The block's first wave turns the token's angles into cos / sin in LDS once for all
// heads, after every thread has requested its first unit.
template <class T, bool kFp8, bool kNeox>
__global__ __launch_bounds__(kThreads) void append_kernel(View v, AppendArgs a, RopeTurns fr) {
    __shared__ float2 cs[kMaxPairs];
    const int t = blockIdx.x, tid = threadIdx.x;
    const int heads = a.in.q ? a.in.heads : 0, kvh = v.c.kv_heads, half = a.in.rotary_dim / 2;
    const int rot_total = (heads + kvh) * a.units_rot;
    int u = blockIdx.y * a.per_block + tid;
    const int u_end = min(a.units, static_cast<int>(blockIdx.y + 1) * a.per_block);

    struct Unit {
        int kind, head, d0;  // kind 0 query, 1 key, 2 value
        bool paired;         // d0 + half goes with it
    };
    auto decode = [&](int i) {
        Unit n;
        int c;
        if (i < rot_total) {
            n.head = i / a.units_rot;
            c = i % a.units_rot;
            n.kind = n.head < heads ? 0 : 1;
            if (n.kind) n.head -= heads;
            n.paired = kNeox && 8 * c < half;
            n.d0 = kNeox && !n.paired ? 8 * c + half : 8 * c;  // past the first half's units: from 2 half on
        } else {
            const int j = i - rot_total;
            n.kind = 2;
            n.head = j / a.units_v;
            n.d0 = 8 * (j % a.units_v);
            n.paired = false;
        }
        return n;
    };
    auto source = [&](const Unit& n) {
        const int64_t tt = t;
        return n.kind == 0   ? static_cast<const T*>(a.in.q) + tt * a.in.q_token + n.head * a.in.q_head
               : n.kind == 1 ? static_cast<const T*>(a.in.k) + tt * a.in.k_token + n.head * a.in.k_head
                             : static_cast<const T*>(a.in.v) + tt * a.in.v_token + n.head * a.in.v_head;
    };
    float x[8], y[8];
    Unit n{};
    if (u < u_end) {
        n = decode(u);
        load8(source(n) + n.d0, x);
        if (n.paired) load8(source(n) + n.d0 + half, y);
    }
    const int seq = sequence_of(v, t, tid & 63);
    if (seq >= v.c.batch || t < v.c.cu[seq]) return;  // a token of no sequence (the same in every wave)
    const int row = row_behind(cached_rows(v, seq), t - max(v.c.cu[seq], 0));
    const int page = page_of(v, seq, row), slot = row & (v.c.page_size - 1);
    if (half > 0) {
        const int pos = a.in.positions ? a.in.positions[t] : row;
        if (tid < half) cs[tid] = cos_sin(fr.turn[tid], pos);
        __syncthreads();
    }
    const int64_t k_at = page * v.c.k_page + slot * v.c.k_slot, v_at = page * v.c.v_page + slot * v.c.v_slot;
    while (u < u_end) {
        const Unit cur = n;
        float p[8], r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = x[e];
            r[e] = y[e];
        }
        u += kThreads;
        if (u < u_end) {  // the next unit's loads are out before this one's stores
            n = decode(u);
            load8(source(n) + n.d0, x);
            if (n.paired) load8(source(n) + n.d0 + half, y);
        }
        if (cur.kind != 2) {
            if constexpr (kNeox) {
                if (cur.paired) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 w = cs[cur.d0 + e];
                        const float f = p[e], g = r[e];
                        p[e] = f * w.x - g * w.y;
                        r[e] = f * w.y + g * w.x;
                    }
                }
            } else if (cur.d0 < 2 * half) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 w = cs[cur.d0 / 2 + e];
                    const float f = p[2 * e], g = p[2 * e + 1];
                    p[2 * e] = f * w.x - g * w.y;
                    p[2 * e + 1] = f * w.y + g * w.x;
                }
            }
        }
        if (cur.kind == 0) {
            const int64_t at = static_cast<int64_t>(t) * a.in.qo_token + cur.head * a.in.qo_head + cur.d0;
            store8<T, false>(a.in.q_out, at, p, 1.0f, 1.0f, 1);
            if (cur.paired) store8<T, false>(a.in.q_out, at + half, r, 1.0f, 1.0f, 1);
        } else if (page >= 0) {
            if (cur.kind == 1) {
                const int64_t at = k_at + cur.head * v.c.k_head + cur.d0;
                store8<T, kFp8>(v.c.k, at, p, a.k_div, a.k_mul, a.k_exact);
                if (cur.paired) store8<T, kFp8>(v.c.k, at + half, r, a.k_div, a.k_mul, a.k_exact);
            } else {
                store8<T, kFp8>(v.c.v, v_at + cur.head * v.c.v_head + cur.d0, p, a.v_div, a.v_mul, a.v_exact);
            }
        }
    }
}

// The same element by element, for operands that are not 16-byte aligned and rotations that 8 dimensions
// do not divide.  A unit is a rotated pair, a plain dimension, or a dimension of a value head.
template <class T, bool kFp8>
__global__ __launch_bounds__(kThreads) void append_scalar_kernel(View v, AppendArgs a, RopeTurns fr) {
    __shared__ float2 cs[kMaxPairs];
    const int t = blockIdx.x, tid = threadIdx.x;
    const int D = v.c.head_dim, heads = a.in.q ? a.in.heads : 0, kvh = v.c.kv_heads, half = a.in.rotary_dim / 2;
    const int seq = sequence_of(v, t, tid & 63);
    if (seq >= v.c.batch || t < v.c.cu[seq]) return;
    const int row = row_behind(cached_rows(v, seq), t - max(v.c.cu[seq], 0));
    const int page = page_of(v, seq, row), slot = row & (v.c.page_size - 1);
    if (half > 0) {
        const int pos = a.in.positions ? a.in.positions[t] : row;
        if (tid < half) cs[tid] = cos_sin(fr.turn[tid], pos);
        __syncthreads();
    }
    const int64_t tt = t;
    auto put = [&](void* base, int64_t at, float x, float div, float mul, int exact) {
        if constexpr (kFp8)
            static_cast<uint8_t*>(base)[at] = static_cast<uint8_t>(pack_e4m3(clamp_e4m3(exact ? x * mul : x / div), 0.0f, 0.0f, 0.0f));
        else
            static_cast<T*>(base)[at] = static_cast<T>(x);
    };
    const int rot_total = (heads + kvh) * a.units_rot;
    const int u_end = min(a.units, static_cast<int>(blockIdx.y + 1) * a.per_block);
    for (int u = blockIdx.y * a.per_block + tid; u < u_end; u += kThreads) {
        if (u >= rot_total) {
            const int h = (u - rot_total) / D, d = (u - rot_total) % D;
            if (page >= 0)
                put(v.c.v, page * v.c.v_page + slot * v.c.v_slot + h * v.c.v_head + d,
                    to_float(static_cast<const T*>(a.in.v)[tt * a.in.v_token + h * a.in.v_head + d]), a.v_div, a.v_mul, a.v_exact);
            continue;
        }
        int h = u / a.units_rot;
        const int c = u % a.units_rot;
        const bool is_q = h < heads;
        if (!is_q) h -= heads;
        const T* src = is_q ? static_cast<const T*>(a.in.q) + tt * a.in.q_token + h * a.in.q_head
                            : static_cast<const T*>(a.in.k) + tt * a.in.k_token + h * a.in.k_head;
        const bool pair = c < half;
        const int d0 = !pair ? c + half : a.in.neox ? c : 2 * c, d1 = a.in.neox ? c + half : 2 * c + 1;
        float f = to_float(src[d0]), g = 0.0f;
        if (pair) {
            g = to_float(src[d1]);
            const float2 w = cs[c];
            const float f2 = f * w.x - g * w.y;
            g = f * w.y + g * w.x;
            f = f2;
        }
        if (is_q) {
            T* dst = static_cast<T*>(a.in.q_out) + tt * a.in.qo_token + h * a.in.qo_head;
            dst[d0] = static_cast<T>(f);
            if (pair) dst[d1] = static_cast<T>(g);
        } else if (page >= 0) {
            const int64_t at = page * v.c.k_page + slot * v.c.k_slot + h * v.c.k_head;
            put(v.c.k, at + d0, f, a.k_div, a.k_mul, a.k_exact);
            if (pair) put(v.c.k, at + d1, g, a.k_div, a.k_mul, a.k_exact);
        }
    }
}

// ---- moving rows ---------------------------------------------------------------------------------
// Rows are copied in units of U bytes, the largest that every address is a multiple of.
template <int B>
struct Unit;
template <>
struct Unit<16> {
    using type = u32x4;
};
template <>
struct Unit<4> {
    using type = uint32_t;
};
template <>
struct Unit<1> {
    using type = uint8_t;
};

struct Strides {  // in units
    int64_t k_layer, k_page, k_head, k_slot, v_layer, v_page, v_head, v_slot;
    int per_row;
};

// Commit of a path: block (x, b) takes 256 of the (layer, K or V, head, piece) columns of sequence b; a
// thread moves its column of every step, eight loads in flight.  The j-th node that is taken, path's j-th entry or a
// later one, is at least j where the path ascends, and its row becomes row j: in that order no step reads what an earlier
// batch of steps has overwritten, and within a batch the loads come first.  The steps that move something are listed in LDS first.  48 sequences, up to 6 rows
// in 32 layers (38 MB read and written): 8.2 us, of which 4 are the launch and the chain of loads before the first row.
constexpr int kSteps = 64, kInFlight = 8;

template <int B>
__global__ __launch_bounds__(kThreads) void commit_kernel(View v, Strides st, const int32_t* __restrict__ path, int64_t path_stride,
                                                          int path_len, int32_t* __restrict__ lens) {
    using U = typename Unit<B>::type;
    __shared__ int4 moves[kSteps];  // source page, slot; target page, slot
    __shared__ int n_moves;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int ctx = cached_rows(v, b), n_new = max(v.c.cu[b + 1], 0) - max(v.c.cu[b], 0);
    const int64_t columns = static_cast<int64_t>(v.c.num_layers) * 2 * v.c.kv_heads * st.per_row;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
    const int piece = static_cast<int>(col % st.per_row);
    int64_t rest = col / st.per_row;
    const int head = static_cast<int>(rest % v.c.kv_heads);
    rest /= v.c.kv_heads;
    const bool is_v = rest & 1;
    const int64_t layer = rest >> 1;
    U* base = static_cast<U*>(is_v ? v.c.v : v.c.k) + layer * (is_v ? st.v_layer : st.k_layer) +
              head * (is_v ? st.v_head : st.k_head) + piece;
    const int64_t sp = is_v ? st.v_page : st.k_page, ss = is_v ? st.v_slot : st.k_slot;
    int taken = 0;
    for (int j0 = 0; j0 < path_len; j0 += kSteps) {
        if (tid < 64) {
            const int j = j0 + lane;
            const int node = j < path_len ? path[b * path_stride + j] : -1;
            const bool live = node >= 0 && node < n_new;
            const uint64_t below = (uint64_t{1} << lane) - 1, lives = __ballot(live);
            const int to = taken + static_cast<int>(__popcll(lives & below));
            int4 m{-1, 0, -1, 0};
            if (live && node != to) {
                const int from_row = row_behind(ctx, node), to_row = row_behind(ctx, to);
                m.x = page_of(v, b, from_row);
                m.y = from_row & (v.c.page_size - 1);
                m.z = page_of(v, b, to_row);
                m.w = to_row & (v.c.page_size - 1);
            }
            const bool moves_row = m.x >= 0 && m.z >= 0;
            const uint64_t mask = __ballot(moves_row);
            if (moves_row) moves[__popcll(mask & below)] = m;
            if (lane == 0) n_moves = __popcll(mask);
            taken += __popcll(lives);
        }
        __syncthreads();
        const int n = n_moves;
        if (col < columns) {
            for (int i0 = 0; i0 < n; i0 += kInFlight) {
                U r[kInFlight];
#pragma unroll
                for (int i = 0; i < kInFlight; ++i) {
                    if (i0 + i < n) {
                        const int4 m = moves[i0 + i];
                        r[i] = base[m.x * sp + m.y * ss];
                    }
                }
#pragma unroll
                for (int i = 0; i < kInFlight; ++i) {
                    if (i0 + i < n) {
                        const int4 m = moves[i0 + i];
                        base[m.z * sp + m.w * ss] = r[i];
                    }
                }
            }
        }
        __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0) lens[b] = ctx + taken;
}

// Reordering: block (x, i) copies a share of what sequence i takes over of its parent's open page, as
// (layer, K or V, head, slot, piece) with the pieces of a slot and the slots of a head adjacent; block x = 0 also
// writes the sequence's row of the table.  At the rate of a copy: 128 sequences, 32 layers (250 MB read and written) in 43 us,
// 5.8 TB/s.
template <int B>
__global__ __launch_bounds__(kThreads) void reorder_kernel(View v, Strides st, const int32_t* __restrict__ parents,
                                                           const int32_t* __restrict__ fresh, int beams, int32_t* __restrict__ table_out,
                                                           int32_t* __restrict__ lens_out) {
    using U = typename Unit<B>::type;
    const int i = blockIdx.y, tid = threadIdx.x;
    const int first = i / beams * beams;
    const int parent = first + min(max(parents[i], 0), beams - 1);
    const int len = max(v.c.ctx[parent], 0), own = fresh[i];
    const int full = len >> v.page_shift, held = len & (v.c.page_size - 1);
    if (blockIdx.x == 0) {
        const int32_t* old = v.c.table + parent * v.c.table_stride;
        int32_t* row = table_out + static_cast<int64_t>(i) * v.c.table_width;
        for (int p = tid; p < v.c.table_width; p += kThreads) row[p] = p < full ? old[p] : p == full ? own : -1;
        if (tid == 0) lens_out[i] = len;
    }
    const int tail = page_of(v, parent, len);
    if (held == 0 || tail < 0 || static_cast<uint32_t>(own) >= static_cast<uint32_t>(v.c.num_pages) || tail == own) return;
    const int per_head = held * st.per_row;
    const int64_t total = static_cast<int64_t>(v.c.num_layers) * 2 * v.c.kv_heads * per_head;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + tid; at < total; at += kInFlight * step) {
        U r[kInFlight];
        U* to[kInFlight];
#pragma unroll
        for (int j = 0; j < kInFlight; ++j) {
            const int64_t u = at + j * step;
            if (u < total) {
                const int in_head = static_cast<int>(u % per_head);
                int64_t rest = u / per_head;
                const int head = static_cast<int>(rest % v.c.kv_heads);
                rest /= v.c.kv_heads;
                const bool is_v = rest & 1;
                const int slot = in_head / st.per_row, piece = in_head % st.per_row;
                U* base = static_cast<U*>(is_v ? v.c.v : v.c.k) + (rest >> 1) * (is_v ? st.v_layer : st.k_layer) +
                          head * (is_v ? st.v_head : st.k_head) + slot * (is_v ? st.v_slot : st.k_slot) + piece;
                const int64_t sp = is_v ? st.v_page : st.k_page;
                r[j] = base[tail * sp];
                to[j] = base + own * sp;
            }
        }
#pragma unroll
        for (int j = 0; j < kInFlight; ++j)
            if (at + j * step < total) *to[j] = r[j];
    }
}

// ---- host side -------------------------------------------------------------------------------
bool power_of_two(float x) {
    int e;
    return std::isfinite(x) && x > 0.0f && std::frexp(x, &e) == 0.5f && std::isfinite(1.0f / x) && 1.0f / x >= 0x1p-126f;
}

// The largest unit of 16, 4 and 1 bytes that divides every address of the cache's rows; strides in it.
int copy_unit(const qmm_paged_kv& c, Strides* st) {
    const int64_t eb = elem_bytes(c.dtype);
    const int64_t s[8] = {c.k_layer, c.k_page, c.k_head, c.k_slot, c.v_layer, c.v_page, c.v_head, c.v_slot};
    uint64_t all = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | static_cast<uint64_t>(c.head_dim * eb);
    for (int64_t x : s) all |= static_cast<uint64_t>(x * eb);
    const int unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    *st = {s[0] * eb / unit, s[1] * eb / unit, s[2] * eb / unit, s[3] * eb / unit, s[4] * eb / unit, s[5] * eb / unit,
           s[6] * eb / unit, s[7] * eb / unit, static_cast<int>(c.head_dim * eb / unit)};
    return unit;
}

// Turns per position of each pair, 2^64 a turn.  A program's layers share one base, so a thread's last table is kept.
const RopeTurns& rope_turns(float base, int rotary_dim) {
    thread_local RopeTurns turns{};
    thread_local float of_base = 0.0f;
    thread_local int of_dim = 0;
    if (of_base != base || of_dim != rotary_dim) {
        for (int i = 0; i < rotary_dim / 2; ++i) {
            const long double t = std::pow(static_cast<long double>(base), -2.0L * i / rotary_dim) / (2.0L * 3.14159265358979323846264338327950288L);
            turns.turn[i] = static_cast<uint64_t>(std::fmod(t, 1.0L) * 0x1p64L);
        }
        of_base = base;
        of_dim = rotary_dim;
    }
    return turns;
}

}  // namespace

int check_view(const qmm_paged_kv* kv, bool need_cu, View* out) {
    if (!kv) return bad("kv must be non-null.");
    const qmm_paged_kv& c = *kv;
    if (c.dtype != QMM_DTYPE_F16 && c.dtype != QMM_DTYPE_BF16 && c.dtype != QMM_DTYPE_E4M3)
        return bad("the cache's dtype must be F16, BF16 or E4M3.");
    if (c.batch < 0 || c.num_pages < 0 || c.table_width < 0 || c.num_layers < 1)
        return bad("batch, num_pages and table_width must be non-negative and num_layers positive.");
    if (c.kv_heads <= 0 || c.head_dim <= 0 || c.head_dim > 256 || c.head_dim % 8 != 0)
        return bad("kv_heads must be positive and head_dim a multiple of 8 up to 256.");
    if (c.page_size <= 0 || (c.page_size & (c.page_size - 1)) != 0 || c.page_size > 65536)
        return bad("page_size must be a power of two up to 65536.");
    if (c.batch > 65535) return bad("batch must be at most 65535.");
    const bool scaled = c.dtype == QMM_DTYPE_E4M3;
    for (float s : {c.k_scale, c.v_scale}) {
        if (!(s > 0.0f) || !std::isfinite(s)) return bad("k_scale and v_scale must be positive and finite.");
        if (!scaled && s != 1.0f) return bad("k_scale and v_scale are for E4M3 caches; they must be 1 for the others.");
    }
    if (c.batch > 0 && ((c.num_pages > 0 && (!c.k || !c.v)) || (c.table_width > 0 && !c.table) || !c.ctx || (need_cu && !c.cu)))
        return bad("k, v, table, ctx and cu must be non-null.");
    const uintptr_t align = scaled ? 1 : 2;
    if (reinterpret_cast<uintptr_t>(c.k) % align != 0 || reinterpret_cast<uintptr_t>(c.v) % align != 0)
        return bad("k and v must be aligned to their elements.");
    out->c = c;
    out->page_shift = 0;
    while ((1 << out->page_shift) < c.page_size) ++out->page_shift;
    return QMM_OK;
}

namespace {

int append(const qmm_paged_kv* kv, const qmm_paged_new* in, hipStream_t stream) {
    View v;
    int rc = check_view(kv, true, &v);
    if (rc != QMM_OK) return rc;
    if (!in) return bad("in must be non-null.");
    AppendArgs a{};
    a.in = *in;
    const int D = v.c.head_dim, rot = in->rotary_dim;
    if (in->dtype != QMM_DTYPE_F16 && in->dtype != QMM_DTYPE_BF16) return bad("the new tokens' dtype must be F16 or BF16.");
    if (v.c.dtype != QMM_DTYPE_E4M3 && v.c.dtype != in->dtype) return bad("the cache must be E4M3 or of the new tokens' dtype.");
    if (in->tokens < 0 || in->heads < 0) return bad("tokens and heads must be non-negative.");
    if (rot < 0 || rot % 2 != 0 || rot > D) return bad("rotary_dim must be even, between 0 and head_dim.");
    if (rot > 0 && !(in->freq_base > 0.0f && std::isfinite(in->freq_base))) return bad("freq_base must be positive and finite.");
    if (in->tokens == 0 || v.c.batch == 0) return QMM_OK;
    if (!in->k || !in->v) return bad("k and v of the new tokens must be non-null.");
    if (in->q && (!in->q_out || in->heads == 0)) return bad("q needs q_out and a positive count of heads.");
    const int heads = in->q ? in->heads : 0;
    const bool fp8 = v.c.dtype == QMM_DTYPE_E4M3;
    a.k_div = v.c.k_scale;
    a.v_div = v.c.v_scale;
    a.k_exact = power_of_two(a.k_div);
    a.v_exact = power_of_two(a.v_div);
    a.k_mul = a.k_exact ? 1.0f / a.k_div : 0.0f;
    a.v_mul = a.v_exact ? 1.0f / a.v_div : 0.0f;
    // 16-byte pieces of the new tokens, 8 elements of the cache
    uint64_t els = static_cast<uint64_t>(in->k_token | in->k_head | in->v_token | in->v_head | v.c.k_page | v.c.k_head | v.c.k_slot |
                                         v.c.v_page | v.c.v_head | v.c.v_slot);
    uint64_t ptr = reinterpret_cast<uintptr_t>(in->k) | reinterpret_cast<uintptr_t>(in->v);
    if (heads) {
        els |= static_cast<uint64_t>(in->q_token | in->q_head | in->qo_token | in->qo_head);
        ptr |= reinterpret_cast<uintptr_t>(in->q) | reinterpret_cast<uintptr_t>(in->q_out);
    }
    const uint64_t cache = reinterpret_cast<uintptr_t>(v.c.k) | reinterpret_cast<uintptr_t>(v.c.v);
    const bool vec = els % 8 == 0 && ptr % 16 == 0 && cache % (fp8 ? 8 : 16) == 0 && rot % (in->neox ? 16 : 8) == 0;
    const int step = vec ? 8 : 1;
    // interleaved pairs lie within 8 dimensions
    a.units_rot = vec && !in->neox ? D / 8 : (D - rot / 2) / step;
    a.units_v = D / step;
    const int64_t units = static_cast<int64_t>(heads + v.c.kv_heads) * a.units_rot + static_cast<int64_t>(v.c.kv_heads) * a.units_v;
    if (units > (1 << 30)) return bad("too many heads.");
    a.units = static_cast<int>(units);
    // A block takes a whole token where that leaves a thousand blocks, as its angles then serve all heads (6818 tokens of 80
    // heads: 55.8 us, 57.4 in two blocks a token, 63.1 in three); few tokens are cut into blocks of one unit a thread.
    const int64_t passes = std::max<int64_t>(1, std::min<int64_t>((units + kThreads - 1) / kThreads, in->tokens * ((units + kThreads - 1) / kThreads) / 1024));
    a.per_block = static_cast<int>(passes * kThreads);
    const dim3 grid(static_cast<unsigned>(in->tokens), static_cast<unsigned>((units + a.per_block - 1) / a.per_block));
    if (grid.y > 65535) return bad("too many heads.");
    static const RopeTurns none{};
    const RopeTurns& fr = rot > 0 ? rope_turns(in->freq_base, rot) : none;
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, stream, v, a, fr); };
    auto pick = [&](auto tc, auto f8) {
        using T = decltype(tc);
        constexpr bool F = decltype(f8)::value;
        if (!vec) go(append_scalar_kernel<T, F>);
        else if (in->neox) go(append_kernel<T, F, true>);
        else go(append_kernel<T, F, false>);
    };
    if (in->dtype == QMM_DTYPE_F16) fp8 ? pick(_Float16{}, std::true_type{}) : pick(_Float16{}, std::false_type{});
    else fp8 ? pick(__bf16{}, std::true_type{}) : pick(__bf16{}, std::false_type{});
    return launched(hipGetLastError(), "paged append kernel launch");
}

int commit_path(const qmm_paged_kv* kv, const int32_t* path, int64_t path_stride, int path_len, int32_t* lens, hipStream_t stream) {
    View v;
    int rc = check_view(kv, true, &v);
    if (rc != QMM_OK) return rc;
    if (path_len < 0) return bad("path_len must be non-negative.");
    if (v.c.batch == 0) return QMM_OK;
    if (!lens || (path_len > 0 && !path)) return bad("path and lens must be non-null.");
    Strides st;
    const int unit = copy_unit(v.c, &st);
    const int64_t columns = static_cast<int64_t>(v.c.num_layers) * 2 * v.c.kv_heads * st.per_row;
    const int64_t blocks = (columns + kThreads - 1) / kThreads;
    if (blocks > INT32_MAX) return bad("too many layers and heads.");
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(v.c.batch));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, stream, v, st, path, path_stride, path_len, lens); };
    unit == 16 ? go(commit_kernel<16>) : unit == 4 ? go(commit_kernel<4>) : go(commit_kernel<1>);
    return launched(hipGetLastError(), "paged commit kernel launch");
}

int reorder(const qmm_paged_kv* kv, const int32_t* parents, const int32_t* fresh, int beams, int32_t* table_out, int32_t* lens_out,
            hipStream_t stream) {
    View v;
    int rc = check_view(kv, false, &v);
    if (rc != QMM_OK) return rc;
    if (beams <= 0 || v.c.batch % beams != 0) return bad("beams must be positive and divide the batch.");
    if (v.c.batch == 0) return QMM_OK;
    if (!parents || !fresh || !lens_out || (v.c.table_width > 0 && !table_out)) return bad("parents, fresh, table_out and lens_out must be non-null.");
    if (table_out == v.c.table || lens_out == v.c.ctx) return bad("table_out and lens_out must not be the inputs.");
    Strides st;
    const int unit = copy_unit(v.c, &st);
    // as many blocks as a whole page needs with kInFlight pieces a thread
    const int64_t most = static_cast<int64_t>(v.c.num_layers) * 2 * v.c.kv_heads * v.c.page_size * st.per_row;
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((most + kInFlight * kThreads - 1) / (kInFlight * kThreads), 65535));
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(v.c.batch));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, stream, v, st, parents, fresh, beams, table_out, lens_out); };
    unit == 16 ? go(reorder_kernel<16>) : unit == 4 ? go(reorder_kernel<4>) : go(reorder_kernel<1>);
    return launched(hipGetLastError(), "beam reorder kernel launch");
}

}  // namespace
}  // namespace paged
}  // namespace qmm

extern "C" {

int qmm_paged_append(const qmm_paged_kv* kv, const qmm_paged_new* in, void* stream) {
    return qmm::paged::entry([&] { return qmm::paged::append(kv, in, static_cast<hipStream_t>(stream)); });
}

int qmm_paged_commit_path(const qmm_paged_kv* kv, const int32_t* path, int64_t path_stride, int path_len, int32_t* lens, void* stream) {
    return qmm::paged::entry([&] { return qmm::paged::commit_path(kv, path, path_stride, path_len, lens, static_cast<hipStream_t>(stream)); });
}

int qmm_beam_reorder(const qmm_paged_kv* kv, const int32_t* parents, const int32_t* fresh, int beams, int32_t* table_out,
                     int32_t* lens_out, void* stream) {
    return qmm::paged::entry([&] { return qmm::paged::reorder(kv, parents, fresh, beams, table_out, lens_out, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
