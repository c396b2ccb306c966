// Device-side access to a paged key/value cache, shared by the kernels that write, move and attend over it.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <exception>
#include <string>

#include "qmm_internal.h"

namespace qmm {
namespace paged {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Fp8 {  // a byte of e4m3fn
    uint8_t bits;
};

// A cache as the kernels take it: the caller's description with the page size as a shift.
struct View {
    qmm_paged_kv c;
    int page_shift;
};

// Page id of row `row` of sequence `seq`, -1 where the table or the pool has no such page (a row past 2^31 is negative).
__device__ __forceinline__ int page_of(const View& v, int seq, int row) {
    const int p = row >> v.page_shift;
    if (static_cast<uint32_t>(p) >= static_cast<uint32_t>(v.c.table_width)) return -1;
    const int id = v.c.table[static_cast<int64_t>(seq) * v.c.table_stride + p];
    return static_cast<uint32_t>(id) < static_cast<uint32_t>(v.c.num_pages) ? id : -1;
}

// Cached rows of a sequence, as every call takes them.
__device__ __forceinline__ int cached_rows(const View& v, int seq) { return min(max(v.c.ctx[seq], 0), 1 << 30); }

// Row `i` behind `cached` ones; past 2^31 it is negative, and on no page.
__device__ __forceinline__ int row_behind(int cached, int i) {
    return static_cast<int>(static_cast<uint32_t>(cached) + static_cast<uint32_t>(i));
}

// The sequence of token t: the count of ends cu[1..batch] at or below it (every lane of the wave must be
// active).  One round of loads for up to 64 sequences, where a binary search would wait for each of its steps.
__device__ __forceinline__ int sequence_of(const View& v, int t, int lane) {
    int n = 0;
    for (int i = 0; i < v.c.batch; i += 64) {
        const bool below = i + lane < v.c.batch && v.c.cu[1 + i + lane] <= t;
        n += __popcll(__ballot(below));
    }
    return n;
}

__device__ __forceinline__ float to_float(_Float16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float to_float(__bf16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float to_float(Fp8 x) {
    return __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(x.bits), false)[0];
}

// x saturated at the largest finite e4m3 value; NaN stays NaN
__device__ __forceinline__ float clamp_e4m3(float x) { return x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f); }

// Four floats -> four e4m3 bytes, round to nearest even (arguments within +-448).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return static_cast<uint32_t>(w);
}

// ---- host side -------------------------------------------------------------------------------

inline int elem_bytes(int dtype) { return dtype == QMM_DTYPE_E4M3 ? 1 : dtype == QMM_DTYPE_F32 ? 4 : 2; }

inline int bad(const std::string& msg) { return set_last_error(QMM_ERR_INVALID_ARGUMENT, msg); }

inline int launched(hipError_t e, const char* what) {
    if (e == hipSuccess) return QMM_OK;
    return set_last_error(QMM_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

// Checks a cache description; fills `out`.  need_cu: the call reads cu.
int check_view(const qmm_paged_kv* kv, bool need_cu, View* out);

// Runs the body of a C entry point: no exception leaves it.
template <class Body>
int entry(Body body) noexcept {
    try {
        return body();
    } catch (const std::exception& e) {
        try {
            return set_last_error(QMM_ERR_HIP, std::string("host error: ") + e.what());
        } catch (...) {
            return QMM_ERR_HIP;
        }
    } catch (...) {
        return QMM_ERR_HIP;
    }
}

}  // namespace paged
}  // namespace qmm
