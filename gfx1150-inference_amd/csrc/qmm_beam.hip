// One step of beam search's selection: the best `beams` of beams x vocab totals
//   total(w, j) = score_w + x_wj - log sum_i exp(x_wi),
// without storing any of them.  Bound by reading the logits once.
//   Pass 1: a block holds one chunk of one beam's logits in registers.  Within a beam the totals are ordered
//           as the logits, so the chunk's best `beams` logits are found there, beside its maximum and its sum
//           of exp(x - max).
//   Pass 2: one block per sentence joins the chunks' sums into each beam's logarithm, in 64 bits, and
//           ranks the chunks' candidates by (total in 64 bits, beam, logit, token): where a score's size leaves totals of
//           different logits equal, a beam keeps the order of its logits, as pass 1 does.  A beam that is out (all of its totals count as
//           -inf: its score or a logit is NaN, its score is -inf or a logit +inf) has its lowest tokens as candidates.
// 128 rows of 128256 f16 logits (33 MB): 14.7 us of pass 1, whose blocks all run at once, so that its parts follow each
// other (7.3 us of reading and maxima, 3 of exponentials, 4 of finding the candidates), and 6.8 us of pass 2, whose sixteen
// blocks wait for loads and a 64-bit exponential and logarithm.
// The order of equal totals and every sum are fixed by the sizes alone, so equal beams give equal totals.
#include "qmm_paged.h"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace qmm {
namespace paged {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxBeams = 64;
constexpr int kWaveList = 128;     // candidates that a wave may list before it narrows them down exactly
constexpr int kMergeThreads = 1024, kMergeList = 1024;

struct Sum {  // sum of exp(x - m) over a wave's logits
    double m, s;
};

struct Candidate {
    float x;
    int32_t token;  // -1: none
};

// A monotone image of the float order; both zeros alike, NaN (of either sign) as -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 becomes +0
    const uint32_t k = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
    return x != x ? 0x007FFFFFu : k;
}

// x joined over the wave, the result in every lane (all of them must be active): neighbours, pairs and halves of 16 lanes
// by DPP, rows of 16 and halves of the wave by swaps.  4 beams of 32000 f32 logits: 0.3 us less in pass 1 and 0.8 in pass 2
// than with shuffles through LDS (and the partial sums read twice); 5.2 + 4.2 us now.
template <class V, class Join>
__device__ __forceinline__ V wave_join(V x, Join join) {
    constexpr int kWords = sizeof(V) / 4;
    struct Words {
        uint32_t w[kWords];
    };
    auto dpp = [&](auto ctrl) {
        Words t = __builtin_bit_cast(Words, x);
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            t.w[i] = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(t.w[i]), decltype(ctrl)::value, 0xF, 0xF, false));
        x = join(x, __builtin_bit_cast(V, t));
    };
    dpp(std::integral_constant<int, 0xB1>{});   // quad_perm [1, 0, 3, 2]
    dpp(std::integral_constant<int, 0x4E>{});   // quad_perm [2, 3, 0, 1]
    dpp(std::integral_constant<int, 0x141>{});  // row_half_mirror
    dpp(std::integral_constant<int, 0x140>{});  // row_mirror
    auto swap = [&](auto f) {  // of a value with itself: what the lower and the upper rows hold, in all of them
        const Words t = __builtin_bit_cast(Words, x);
        Words a, b;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const auto y = f(t.w[i]);
            a.w[i] = y[0];
            b.w[i] = y[1];
        }
        x = join(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b));
    };
    swap([](uint32_t v) { return __builtin_amdgcn_permlane16_swap(v, v, false, false); });
    swap([](uint32_t v) { return __builtin_amdgcn_permlane32_swap(v, v, false, false); });
    return x;
}

__device__ __forceinline__ double wave_add(double x) {
    return wave_join(x, [](double a, double b) { return a + b; });
}

__device__ __forceinline__ float wave_max(float x) {
    return wave_join(x, [](float a, float b) { return fmaxf(a, b); });
}

// The largest t, of sign, exponent and 11 bits of the float, that at least n of the wave's keys reach (n <= 64), one
// bit at a time.
__device__ __forceinline__ uint32_t wave_threshold(uint32_t key, int n) {
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t c = t | (1u << bit);
        if (__popcll(__ballot(key >= c)) >= n) t = c;
    }
    return t;
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// exp(d), d <= 0, as 2^(d log2 e) with log2 e in two parts: the rounding of the constant alone would give the terms' errors
// one sign and move a beam against the others; the product's rounding has either.
__device__ __forceinline__ float exp_of(float d) {
    constexpr float kLog2e = 1.44269502162933349609f, kLog2eLow = 1.92596299112661746887e-8f;
    return __builtin_amdgcn_exp2f(__fmaf_rn(d, kLog2e, d * kLog2eLow));
}

// The float whose order_key is k.
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

template <class T>
struct Piece;  // 16 bytes of logits
template <>
struct Piece<float> {
    using type = f32x4;
};
template <>
struct Piece<_Float16> {
    using type = f16x8;
};
template <>
struct Piece<__bf16> {
    using type = bf16x8;
};

// Chunk blockIdx.x of beam blockIdx.y: E logits a thread, in pieces of 16 bytes.  Which thread takes a token does not
// depend on the row's address (rows of an odd vocabulary start anywhere), so that equal beams have equal sums to the
// last bit and their ties stay ties; the pieces are loaded at whatever alignment they have.
template <class T, int E>
__global__ __launch_bounds__(kThreads) void select_chunk_kernel(const T* __restrict__ logits, int64_t sentence_stride, int64_t beam_stride,
                                                                const float* __restrict__ scores, int beams, int vocab,
                                                                Sum* __restrict__ sums, Candidate* __restrict__ cands) {
    constexpr int kP = 16 / sizeof(T), kN = E / kP;
    __shared__ uint64_t list[kWaves * kWaveList];
    __shared__ int counts[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = blockIdx.y, chunk = blockIdx.x;
    const T* base = logits + (row / beams) * sentence_stride + (row % beams) * beam_stride;
    const int first = chunk * (E * kThreads);  // token of the chunk's first element
    // The logits stay as they came, 16 bytes a piece, and are converted where they are used: 64 of them as floats left
    // three waves a SIMD (19.8 us, where it is 14.8).
    using P = typename Piece<T>::type;
    P raw[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const int at = first + (j * kThreads + tid) * kP;
        if (at + kP <= vocab) {
            __builtin_memcpy(&raw[j], base + at, 16);
        } else {
#pragma unroll
            for (int e = 0; e < kP; ++e) raw[j][e] = at + e < vocab ? base[at + e] : static_cast<T>(-INFINITY);
        }
    }
    auto unkept = [&] {  // what was converted before is not kept beyond this point
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            u32x4 t = __builtin_bit_cast(u32x4, raw[j]);
            __asm__("" : "+v"(t));
            raw[j] = __builtin_bit_cast(P, t);
        }
    };
    auto x = [&](int e) { return static_cast<float>(raw[e / kP][e % kP]); };
    // the wave's maximum and sum
    float piece_best[kN], m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        piece_best[j] = x(j * kP);
#pragma unroll
        for (int e = 1; e < kP; ++e) piece_best[j] = fmaxf(piece_best[j], x(j * kP + e));
        m = fmaxf(m, piece_best[j]);
    }
    const float lane_best = m;
    m = wave_max(m);
    const float ref = m == -INFINITY ? 0.0f : m;  // nothing but -inf: every term is 0
    float s = 0.0f;
    unkept();
#pragma unroll
    for (int e = 0; e < E; ++e) s += exp_of(x(e) - ref);
    unkept();
    const double ws = wave_add(static_cast<double>(s));
    if (lane == 0) sums[(static_cast<int64_t>(row) * gridDim.x + chunk) * kWaves + w] = Sum{static_cast<double>(m), ws};

    // the wave's best `beams`: a lower bound from the lanes' maxima, then every logit that reaches it
    auto token_of = [&](int e) { return first + ((e / kP) * kThreads + tid) * kP + e % kP; };
    auto inside = [&](int token) { return token < vocab; };
    uint64_t* mine = list + w * kWaveList;
    auto put = [&](bool take, uint32_t key, int e, int n) {
        const uint64_t mask = __ballot(take);
        if (mask == 0) return n;
        const int at = n + lanes_below(mask);
        if (take && at < kWaveList) mine[at] = (static_cast<uint64_t>(key) << 32) | static_cast<uint32_t>(~token_of(e));
        return n + static_cast<int>(__popcll(mask));
    };
    int n = 0;
    if (scores[row] > -INFINITY) {  // the beam is out otherwise, and pass 2 needs no candidates of it
        // (a piece at a time: few hold one).  What lies past the vocabulary is -inf, and NaN reaches nothing, so a bound
        // of -inf takes the other way too.
        const float least = key_value(wave_threshold(order_key(lane_best), beams));
        if (least > -INFINITY) {
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                if (__ballot(piece_best[j] >= least) == 0) continue;
#pragma unroll
                for (int e = 0; e < kP; ++e) n = put(x(j * kP + e) >= least, order_key(x(j * kP + e)), j * kP + e, n);
            }
        }
        if (n > kWaveList || !(least > -INFINITY)) {
            // many equal logits: the exact bound, then the lowest tokens of those that equal it
            auto key = [&](int e) { return inside(token_of(e)) ? order_key(x(e)) : 0; };  // 0: below every key
            uint32_t t = 0;
#pragma unroll 1
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t c = t | (1u << bit);
                int count = 0;
                unkept();
#pragma unroll
                for (int e = 0; e < E; ++e) count += static_cast<int>(__popcll(__ballot(key(e) >= c)));
                if (count >= beams) t = c;
            }
            // (t is 0 where the wave holds fewer than `beams`: all of them are above it)
            int above = 0;
            unkept();
#pragma unroll
            for (int e = 0; e < E; ++e) above += static_cast<int>(__popcll(__ballot(key(e) > t)));
            uint32_t last = 0x7FFFFFFFu;  // the lowest bound on the token that keeps beams - above of the equal ones
#pragma unroll 1
            for (int bit = 30; t > 0 && bit >= 0; --bit) {
                const uint32_t c = last & ~(1u << bit);
                int count = 0;
                unkept();
#pragma unroll
                for (int e = 0; e < E; ++e) count += static_cast<int>(__popcll(__ballot(key(e) == t && static_cast<uint32_t>(token_of(e)) <= c)));
                if (above + count >= beams) last = c;
            }
            n = 0;
            unkept();
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t k = key(e);
                n = put(k > t || (t > 0 && k == t && static_cast<uint32_t>(token_of(e)) <= last), k, e, n);
            }
        }
    }
    if (lane == 0) counts[w] = n;
    __syncthreads();

    const int64_t out = static_cast<int64_t>(row) * gridDim.x + chunk;
    // rank the waves' lists against each other
    int start[kWaves], total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        start[i] = total;
        total += counts[i];
    }
    auto nth = [&](int i) {
        int from = 0;
#pragma unroll
        for (int k = 1; k < kWaves; ++k)
            if (i >= start[k]) from = k;
        return list[from * kWaveList + i - start[from]];
    };
    Candidate* dst = cands + out * beams;
    for (int i = tid; i < total; i += kThreads) {
        const uint64_t own = nth(i);
        int rank = 0;
        for (int k = 0; k < kWaves; ++k)
            for (int c = 0; c < counts[k]; ++c) rank += list[k * kWaveList + c] > own;
        if (rank < beams) {
            const int token = static_cast<int>(~static_cast<uint32_t>(own));
            dst[rank] = Candidate{static_cast<float>(base[token]), token};
        }
    }
    for (int i = total + tid; i < beams; i += kThreads) dst[i] = Candidate{0.0f, -1};
}

struct Entry {  // a candidate's beam, and its place there: the logit's order and then the lower token are larger
    double total;
    uint64_t place;
    int beam;
    __device__ __forceinline__ int token() const { return static_cast<int>(~static_cast<uint32_t>(place)); }
};

__device__ __forceinline__ bool better(const Entry& a, const Entry& b) {
    return a.total > b.total || (a.total == b.total && (a.beam < b.beam || (a.beam == b.beam && a.place > b.place)));
}

__global__ __launch_bounds__(kMergeThreads) void select_merge_kernel(const float* __restrict__ scores, const Sum* __restrict__ sums,
                                                                     const Candidate* __restrict__ cands, int beams, int vocab,
                                                                     int chunks, float* __restrict__ out_scores, int32_t* __restrict__ out_parents,
                                                                     int32_t* __restrict__ out_tokens) {
    constexpr int kW = kMergeThreads / 64;
    __shared__ double offset[kMaxBeams];  // score - logarithm; -inf: the beam is out
    __shared__ uint32_t bounds[kW];
    __shared__ double l_total[kMergeList];
    __shared__ uint64_t l_place[kMergeList];
    __shared__ int l_beam[kMergeList];
    __shared__ Entry waves[kW];
    __shared__ int l_n;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t first_row = static_cast<int64_t>(blockIdx.x) * beams;
    const int per_beam = chunks * beams, n = beams * per_beam;
    const Candidate* cs = cands + first_row * per_beam;
    const Candidate own = cs[min(tid, n - 1)];  // requested before the sums' chain
    for (int b = w; b < beams; b += kW) {
        const int parts = chunks * kWaves;
        const Sum* sm = sums + (first_row + b) * parts;
        const float score = scores[first_row + b];
        const Sum p0 = lane < parts ? sm[lane] : Sum{-INFINITY, 0.0};
        float best = static_cast<float>(p0.m);  // an fp32 value
        for (int i = lane + 64; i < parts; i += 64) best = fmaxf(best, static_cast<float>(sm[i].m));
        const double m = static_cast<double>(wave_max(best));
        double s = 0.0;
        auto add = [&](const Sum& p) {
            if (p.m > -INFINITY || p.s != p.s) s += p.s * exp(p.m - m);
        };
        add(p0);
        for (int i = lane + 64; i < parts; i += 64) add(sm[i]);
        s = wave_add(s);
        const double at = static_cast<double>(score) - (m + log(s));
        if (lane == 0) offset[b] = at == at ? at : -INFINITY;
    }
    if (tid == 0) l_n = 0;
    __syncthreads();
    auto entry_of = [&](int i, Entry& x) {  // false: there is none
        const Candidate c = i == tid ? own : cs[i];
        x.beam = i / per_beam;
        const double off = offset[x.beam];
        if (off == -INFINITY) {  // the beam is out: its lowest tokens
            const int at = i - x.beam * per_beam;
            x.total = off;
            x.place = static_cast<uint32_t>(~at);
            return at < min(beams, vocab);
        }
        const double t = static_cast<double>(c.x) + off;
        x.total = t == t ? t : -INFINITY;
        x.place = (static_cast<uint64_t>(order_key(c.x)) << 32) | static_cast<uint32_t>(~c.token);
        return c.token >= 0;
    };
    // a bound that at least `beams` candidates of some wave reach: totals rounded to fp32 keep their order
    uint32_t best = 0;
    for (int i = tid; i < n; i += kMergeThreads) {
        Entry x;
        if (entry_of(i, x)) best = max(best, order_key(static_cast<float>(x.total)));
    }
    const uint32_t t_wave = wave_threshold(best, beams);
    if (lane == 0) bounds[w] = t_wave;
    __syncthreads();
    uint32_t bound = 0;
    for (int i = 0; i < kW; ++i) bound = max(bound, bounds[i]);
    for (int i = tid; i < n; i += kMergeThreads) {
        Entry x;
        if (entry_of(i, x) && order_key(static_cast<float>(x.total)) >= bound) {
            const int at = atomicAdd(&l_n, 1);
            if (at < kMergeList) {
                l_total[at] = x.total;
                l_place[at] = x.place;
                l_beam[at] = x.beam;
            }
        }
    }
    __syncthreads();
    auto write = [&](int rank, const Entry& x) {
        out_scores[first_row + rank] = static_cast<float>(x.total);
        out_parents[first_row + rank] = x.beam;
        out_tokens[first_row + rank] = x.token();
    };
    const int listed = l_n;
    if (listed <= kMergeList) {
        if (tid < listed) {
            const Entry x{l_total[tid], l_place[tid], l_beam[tid]};
            int rank = 0, equal = 0;
            for (int i = 0; i < listed; ++i) {
                const double t = l_total[i];
                rank += t > x.total;
                equal += t == x.total;
            }
            if (equal > 1)  // few: the places of these alone
                for (int i = 0; i < listed; ++i) rank += l_total[i] == x.total && better(Entry{x.total, l_place[i], l_beam[i]}, x);
            if (rank < beams) write(rank, x);
        }
        return;
    }
    // Many equal totals: one after the other, each the best of those after the last one in order.
    Entry last{INFINITY, 0, -1};
    for (int r = 0; r < beams; ++r) {
        Entry top{-INFINITY, 0, INT32_MAX};
        for (int i = tid; i < n; i += kMergeThreads) {
            Entry x;
            if (entry_of(i, x) && better(last, x) && better(x, top)) top = x;
        }
        for (int o = 32; o > 0; o >>= 1) {
            const Entry x{__shfl_xor(top.total, o, 64), __shfl_xor(top.place, o, 64), __shfl_xor(top.beam, o, 64)};
            if (better(x, top)) top = x;
        }
        if (lane == 0) waves[w] = top;
        __syncthreads();
        top = waves[0];
        for (int i = 1; i < kW; ++i)
            if (better(waves[i], top)) top = waves[i];
        last = top;
        if (tid == 0) write(r, top);
        __syncthreads();
    }
}

// ---- host side -------------------------------------------------------------------------------
// Logits a thread: as few as leave 512 chunks, so that small calls use the chip's width and large ones read up to 64 logits a
// thread at once and leave few candidates (128 rows of 128256: 14.8 + 8.6 us at 64, 15.0 + 12.5 at 32, with sums joined through LDS).
int per_thread(int64_t rows, int vocab) {
    int e = 8;
    while (e < 64 && rows * ((vocab + 2 * e * kThreads - 1) / (2 * e * kThreads)) >= 512) e *= 2;
    return e;
}

struct SelectPlan {
    int e, chunks;
    size_t cands, bytes;
};

SelectPlan select_plan(int sentences, int beams, int vocab) {
    SelectPlan p{};
    const int64_t rows = static_cast<int64_t>(sentences) * beams;
    p.e = per_thread(rows, vocab);
    p.chunks = (vocab + p.e * kThreads - 1) / (p.e * kThreads);
    p.cands = static_cast<size_t>(rows) * p.chunks * kWaves * sizeof(Sum);
    p.bytes = p.cands + static_cast<size_t>(rows) * p.chunks * beams * sizeof(Candidate);
    return p;
}

int check_select(int dtype, int sentences, int beams, int vocab) {
    if (dtype != QMM_DTYPE_F32 && dtype != QMM_DTYPE_F16 && dtype != QMM_DTYPE_BF16) return bad("logits must be F32, F16 or BF16.");
    if (sentences < 0 || vocab <= 0) return bad("sentences must be non-negative and vocab positive.");
    if (beams <= 0 || beams > kMaxBeams) return bad("beams must be between 1 and 64.");
    if (vocab > (1 << 30) || static_cast<int64_t>(sentences) * beams > 65535) return bad("vocab must be at most 2^30 and sentences * beams at most 65535.");
    return QMM_OK;
}

int select(const void* logits, int dtype, int64_t sentence_stride, int64_t beam_stride, const float* scores, int sentences, int beams,
           int vocab, float* out_scores, int32_t* out_parents, int32_t* out_tokens, void* workspace, size_t workspace_bytes,
           hipStream_t stream) {
    const int rc = check_select(dtype, sentences, beams, vocab);
    if (rc != QMM_OK) return rc;
    if (sentences == 0) return QMM_OK;
    if (!logits || !scores || !out_scores || !out_parents || !out_tokens) return bad("logits, scores and the outputs must be non-null.");
    if (reinterpret_cast<uintptr_t>(logits) % elem_bytes(dtype) != 0) return bad("logits must be aligned to their elements.");
    const SelectPlan p = select_plan(sentences, beams, vocab);
    std::unique_lock<std::mutex> held;
    if (workspace) {
        if (workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return bad("the workspace must be 16-byte aligned and hold qmm_beam_select_workspace() bytes.");
    } else {
        const hipError_t e = take_workspace(WorkspaceKind::kAttention, stream, p.bytes, held, &workspace);
        if (e != hipSuccess) return launched(e, "beam select workspace");
    }
    Sum* sums = static_cast<Sum*>(workspace);
    Candidate* cands = reinterpret_cast<Candidate*>(static_cast<char*>(workspace) + p.cands);
    const dim3 grid(static_cast<unsigned>(p.chunks), static_cast<unsigned>(sentences * beams));
    auto go = [&](auto tc, auto ec) {
        using T = decltype(tc);
        hipLaunchKernelGGL((select_chunk_kernel<T, decltype(ec)::value>), grid, dim3(kThreads), 0, stream, static_cast<const T*>(logits),
                           sentence_stride, beam_stride, scores, beams, vocab, sums, cands);
    };
    auto pick = [&](auto tc) {
        switch (p.e) {
            case 8: go(tc, std::integral_constant<int, 8>{}); break;
            case 16: go(tc, std::integral_constant<int, 16>{}); break;
            case 32: go(tc, std::integral_constant<int, 32>{}); break;
            default: go(tc, std::integral_constant<int, 64>{}); break;
        }
    };
    if (dtype == QMM_DTYPE_F32) pick(float{});
    else if (dtype == QMM_DTYPE_F16) pick(_Float16{});
    else pick(__bf16{});
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return launched(e, "beam select kernel launch");
    hipLaunchKernelGGL(select_merge_kernel, dim3(static_cast<unsigned>(sentences)), dim3(kMergeThreads), 0, stream, scores, sums, cands,
                       beams, vocab, p.chunks, out_scores, out_parents, out_tokens);
    return launched(hipGetLastError(), "beam select merge kernel launch");
}

}  // namespace
}  // namespace paged
}  // namespace qmm

extern "C" {

size_t qmm_beam_select_workspace(int dtype, int sentences, int beams, int vocab) {
    if (qmm::paged::entry([&] { return qmm::paged::check_select(dtype, sentences, beams, vocab); }) != QMM_OK) return 0;
    return qmm::paged::select_plan(sentences, beams, vocab).bytes;
}

int qmm_beam_select(const void* logits, int dtype, int64_t sentence_stride, int64_t beam_stride, const float* scores, int sentences,
                    int beams, int vocab, float* out_scores, int32_t* out_parents, int32_t* out_tokens, void* workspace,
                    size_t workspace_bytes, void* stream) {
    return qmm::paged::entry([&] {
        return qmm::paged::select(logits, dtype, sentence_stride, beam_stride, scores, sentences, beams, vocab, out_scores, out_parents,
                                  out_tokens, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
