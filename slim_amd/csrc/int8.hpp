// What the products with int8 codes (int8.hip) and their gradient (int8grad.hip) have in common.
#pragma once
#include "common.hpp"
#include "../../include/slim_hip.h"
#include <type_traits>

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef const __attribute__((address_space(1))) void* glb_ptr_t;

int64_t pad128(int64_t k) { return (k + 127) / 128 * 128; }
int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }
bool known(int dtype) { return dtype == SLIM_DTYPE_F32 || dtype == SLIM_DTYPE_BF16 || dtype == SLIM_DTYPE_F16; }
int64_t element_size(int dtype) { return dtype == SLIM_DTYPE_F32 ? 4 : 2; }

// ---- element types --------------------------------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }

// eight consecutive elements from any element-aligned address (global loads need no more than that)
template <typename T>
struct Packed8 {
    typedef T vec __attribute__((ext_vector_type(8)));
    struct __attribute__((packed, aligned(sizeof(T)))) type { vec v; };
};
// (ONCE: data that is not read again and need not stay in the caches)
template <bool ONCE = false, typename T>
__device__ __forceinline__ void load8(const T* p, int64_t valid, float out[8]) {
    if (valid >= 8) {
        typedef typename Packed8<T>::vec unaligned __attribute__((aligned(sizeof(T))));
        const typename Packed8<T>::vec v = ONCE ? __builtin_nontemporal_load((const unaligned*)p) : ((const typename Packed8<T>::type*)p)->v;
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = to_f32((T)v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = j < valid ? to_f32(p[j]) : 0.f;
    }
}

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// CNT (8 or 4) consecutive results of one row, to any element-aligned address
template <int CNT, typename T, typename F>
__device__ __forceinline__ void store_run(T* dst, int64_t left, F value) {
    if (left >= CNT) {
        typedef T vec __attribute__((ext_vector_type(CNT)));
        struct __attribute__((packed, aligned(sizeof(T)))) unaligned { vec v; };
        vec v;
#pragma unroll
        for (int j = 0; j < CNT; ++j) v[j] = value(j);
        ((unaligned*)dst)->v = v;
    } else {
#pragma unroll
        for (int j = 0; j < CNT; ++j)
            if (j < left) dst[j] = value(j);
    }
}
template <int CNT, typename T>
__device__ __forceinline__ void load_run(const T* src, int64_t left, float* out) {
    if constexpr (CNT == 8) {
        load8(src, left, out);
    } else {
#pragma unroll
        for (int c = 0; c < CNT; ++c) out[c] = c < left ? to_f32(src[c]) : 0.f;
    }
}

// Tile and slice of workgroup b of tiles_m * tiles_n * splits.  Workgroups go to the eight XCDs in turn; each XCD gets a run of
// consecutive tiles, and a run walks groups of eight rows of tiles column by column, so that the 32 workgroups of an XCD share 8
// panels of A and 4 of B in its L2 (groups of four, 4 panels of A and 8 of B: the same within 3 % either way on the 256 x 256 tile).
__device__ __forceinline__ void tile_of(int b, int tiles_m, int tiles_n, int splits, int& tm, int& tn, int& slice) {
    const int per = tiles_m * tiles_n, total = per * splits, x = b & 7, share = total >> 3, rest = total & 7;
    const int t = x * share + min(x, rest) + (b >> 3);
    slice = t / per;
    const int u = t - slice * per, group = u / (8 * tiles_n), m0 = group * 8, gm = min(8, tiles_m - m0), r = u - group * 8 * tiles_n;
    tm = m0 + r % gm;
    tn = r / gm;
}

// The runs of consecutive columns that a lane holds of a row of its wave's part, 4 FN values: eight per two fragments, four of an odd last one.
// each(n0, fq, take) calls take(how many, first value, column) for each.
template <int FN>
struct Columns {
    static constexpr int PAIRS = FN / 2 * 32, RUNS = (FN + 1) / 2;
    template <typename F>
    static __device__ __forceinline__ void each(int64_t n0, int fq, F take) {
#pragma unroll
        for (int c = 0; c < FN / 2; ++c) take(std::integral_constant<int, 8>(), c * 8, n0 + c * 32 + fq * 8);
        if constexpr (FN % 2) take(std::integral_constant<int, 4>(), 4 * FN - 4, n0 + PAIRS + fq * 4);
    }
};

}  // namespace

// the longest reduction whose sums of products of codes in [-128, 127] fit 32 bits
#define SLIM_INT8_MAX_REDUCTION 131071
// rows and columns: a workgroup of 256 threads each stays below a grid's 2^32 threads (long rows take 1024: 2^22 - 1 of more than 16384 elements)
#define SLIM_INT8_MAX_DIM ((1 << 24) - 1)
