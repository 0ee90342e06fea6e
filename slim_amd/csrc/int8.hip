// Linears in 8-bit integers: rows quantised to int8 codes with one fp32 scale each (tokens of an activation, output channels
// of a weight), the product of two such matrices on the int8 matrix instructions with the scales in its epilogue, and the
// straight-through gradient with respect to the input.  The reference only emulates quantised inputs and weights with dense
// floating-point products (slim/quantization/quantization.py:219-263, :266-304).
#include "common.hpp"
#include "../../include/slim_hip.h"

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef const __attribute__((address_space(1))) void* glb_ptr_t;

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
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t valid, float out[8]) {
    if (valid >= 8) {
        const typename Packed8<T>::vec v = ((const typename Packed8<T>::type*)p)->v;
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = to_f32((T)v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = j < valid ? to_f32(p[j]) : 0.f;
    }
}

// ---- rows -> codes --------------------------------------------------------------------------------------------------
// a = max |x| over the row, scale = a / L, q = rint(x * (L / a)) with L = 127 for one plane of codes.  PLANES > 1 (gradients):
// the row, each element first multiplied by its column's factor, is kept as integers of more bits, q = sum 256^i * plane_i with
// every plane in [-128, 127], so L = 127 * (256^PLANES - 1) / 255 (32639, 8355711).  Rows with a < 2^-100 become zero (scale 0); rows
// that hold an infinity or a NaN get the scale NaN and zero codes, which makes every product with them NaN.
// Plane rows are stored sixteen rows of plane PLANES-1 (the highest), then the sixteen of the next plane, and so on, per
// sixteen rows of x: a fragment of the matrix product then holds all planes of its rows in one lane's accumulators.
template <int PLANES>
struct Levels {
    static constexpr float value = PLANES == 1 ? 127.f : PLANES == 2 ? 32639.f : 8355711.f;
};

template <int PLANES>
__device__ __forceinline__ void store_codes(const float x[8], float r, int8_t* codes, int64_t ldc, int64_t row, int64_t col) {
    uint32_t out[PLANES][2];
#pragma unroll
    for (int p = 0; p < PLANES; ++p) out[p][0] = out[p][1] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float t = x[j] * r;
        if (PLANES == 3) t = fminf(fmaxf(t, -Levels<3>::value), Levels<3>::value);    // two roundings at 23 bits can pass the last level
        int q = (int)rintf(t);
#pragma unroll
        for (int p = PLANES - 1; p >= 0; --p) {          // the lowest plane first
            const int low = p ? (int)(int8_t)(q & 255) : q;
            out[p][j >> 2] |= (uint32_t)(low & 255) << (8 * (j & 3));
            q = (q - low) >> 8;
        }
    }
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
        const int64_t at = PLANES == 1 ? row : ((row >> 4) * PLANES + p) * 16 + (row & 15);
        *(uint2*)(codes + at * ldc + col) = make_uint2(out[p][0], out[p][1]);
    }
}

// WPR waves work on a row (four rows per workgroup, or one); each thread keeps NV pieces of eight elements in registers, so
// the row is read once.  NV = 0: rows too long for that are read twice.
template <typename T, int PLANES, int NV, int WPR>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t R, int64_t K, int64_t ldx,
                                                            const float* __restrict__ colscale, int8_t* __restrict__ codes,
                                                            int64_t ldc, float* __restrict__ scale) {
    constexpr int TPR = 64 * WPR;                        // threads of a row
    __shared__ uint32_t part[4];
    const int wave = threadIdx.x >> 6;
    const int64_t row = WPR == 4 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (WPR == 1 && row >= R) return;
    const int t = WPR == 4 ? threadIdx.x : threadIdx.x & 63;
    const T* src = x + row * ldx;
    float keep[NV > 0 ? NV : 1][8];
    uint32_t m = 0;
    auto fetch = [&](int64_t c, float v[8]) {
        load8(src + c, K - c, v);
        if (PLANES > 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c + j < K ? v[j] * colscale[c + j] : 0.f;
        }
    };
    auto take = [&](const float v[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t b = f32_bits(v[j]) & 0x7fffffffu;
            m = b > m ? b : m;
        }
    };
    if (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = ((int64_t)i * TPR + t) * 8;
            if (c < K) {
                fetch(c, keep[i]);
                take(keep[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) keep[i][j] = 0.f;
            }
        }
    } else {
        for (int64_t c = (int64_t)t * 8; c < K; c += TPR * 8) {
            float v[8];
            fetch(c, v);
            take(v);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t b = (uint32_t)__shfl_xor((int)m, o, 64);
        m = b > m ? b : m;
    }
    if (WPR == 4) {
        if ((threadIdx.x & 63) == 0) part[wave] = m;
        __syncthreads();
        m = max(max(part[0], part[1]), max(part[2], part[3]));
    }
    const float a = __uint_as_float(m);
    const bool bad = m >= 0x7f800000u, none = bad || a < 0x1p-100f;
    const float r = none ? 0.f : Levels<PLANES>::value / a;
    if (t == 0) scale[row] = bad ? __uint_as_float(0x7fc00000u) : none ? 0.f : a / Levels<PLANES>::value;
    const int64_t end = (K + 127) / 128 * 128;
    auto put = [&](int64_t c, float v[8]) {
        if (none) {                                      // (x * 0 would be a NaN for what is not finite)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        }
        store_codes<PLANES>(v, r, codes, ldc, row, c);
    };
    if (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = ((int64_t)i * TPR + t) * 8;
            if (c < end) put(c, keep[i]);
        }
    } else {
        for (int64_t c = (int64_t)t * 8; c < end; c += TPR * 8) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (c < K) fetch(c, v);
            put(c, v);
        }
    }
}

template <typename T, int PLANES>
int quantize_rows(const T* x, int64_t R, int64_t K, int64_t ldx, const float* colscale, int8_t* codes, int64_t ldc, float* scale,
                  hipStream_t st) {
    const int64_t pieces = (K + 127) / 128 * 16;         // pieces of eight codes in a padded row
#define SLIM_ROWS(NV, WPR)                                                                                                  \
    quantize_rows_kernel<T, PLANES, NV, WPR><<<(unsigned)(WPR == 4 ? R : ceil_div64(R, 4)), 256, 0, st>>>(x, R, K, ldx, colscale, codes, ldc, scale)
    if (pieces <= 64) SLIM_ROWS(1, 1);
    else if (pieces <= 128) SLIM_ROWS(2, 1);
    else if (pieces <= 256) SLIM_ROWS(4, 1);
    else if (pieces <= 512) SLIM_ROWS(2, 4);
    else if (pieces <= 1024) SLIM_ROWS(4, 4);
    else if (pieces <= 2048) SLIM_ROWS(8, 4);
    else SLIM_ROWS(0, 4);
#undef SLIM_ROWS
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

template <int PLANES>
int quantize_rows_any(const void* x, int dtype, int64_t R, int64_t K, int64_t ldx, const float* colscale, int8_t* codes, int64_t ldc,
                      float* scale, hipStream_t st) {
    if (dtype == SLIM_DTYPE_F32) return quantize_rows<float, PLANES>((const float*)x, R, K, ldx, colscale, codes, ldc, scale, st);
    if (dtype == SLIM_DTYPE_BF16) return quantize_rows<bf16_t, PLANES>((const bf16_t*)x, R, K, ldx, colscale, codes, ldc, scale, st);
    return quantize_rows<_Float16, PLANES>((const _Float16*)x, R, K, ldx, colscale, codes, ldc, scale, st);
}

// ---- codes x codes --------------------------------------------------------------------------------------------------
struct Gemm8Args {
    const int8_t* A;                                     // [rows, lda]: rows of codes (planes interleaved when PLANES > 1)
    const int8_t* B;                                     // [N, ldb]
    int64_t lda, ldb;
    int64_t rows, M, N;                                  // rows of A, rows of the result
    int steps;                                           // 128-byte steps of the reduction
    const float* sa;                                     // [M]
    const float* sb;                                     // [N] or null
    const void* bias;                                    // [N] of the output's type, or null
    void* out;
    int64_t ldo;
    int dtype;
    int tiles_m, tiles_n;
};

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
    if (dtype == SLIM_DTYPE_F32) return ((const float*)p)[i];
    if (dtype == SLIM_DTYPE_BF16) return bf16_to_f32(((const bf16_t*)p)[i]);
    return (float)((const _Float16*)p)[i];
}

// n (4 .. 32) consecutive results of one row, from any element-aligned address
template <int CNT, typename T, typename F>
__device__ __forceinline__ void store_row(T* dst, int64_t left, F value) {
    if (left >= CNT) {
#pragma unroll
        for (int c = 0; c < CNT; c += 8) {
            typename Packed8<T>::vec v;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = value(c + j);
            ((typename Packed8<T>::type*)(dst + c))->v = v;
        }
    } else {
#pragma unroll
        for (int j = 0; j < CNT; ++j)
            if (j < left) dst[j] = value(j);
    }
}

// D = A B^T on 16 x 16 x 64 int8 instructions, operands delivered by LDS-DMA (16 bytes per lane) one 128-byte step ahead.
// LDS image of a stage: BM rows of A, then BN rows of B, 128 bytes each; the 16-byte piece c of a row is stored at c ^ key(row),
// applied on the source side.  The result is computed transposed (B's fragment as the first operand): a lane then holds
// consecutive columns of one row, and with the rows of B dealt to the fragments in runs of four (row (r / 4) * 4 FN + 4 j + r % 4
// for lane row r of fragment j) all 4 FN of them are consecutive, so a lane stores its part of a row in 16-byte pieces.
// key(row) = the lane row's low three bits in either operand, which spreads eight lanes over the eight pieces of a row.
template <int PLANES, int FM, int FN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void gemm8_kernel(const Gemm8Args g) {
    constexpr int BM = 16 * FM * WM, BN = 16 * FN * WN, NW = WM * WN;
    constexpr int PIECES = (BM + BN) / 8, PPW = (PIECES + NW - 1) / NW;
    constexpr int STAGE_BYTES = (BM + BN) * 128;
    constexpr int KB = FN == 8 ? 5 : FN == 4 ? 4 : FN == 2 ? 3 : 2;      // the bit of a B row that tells lane rows r and r + 4 apart
    static_assert(FM % PLANES == 0, "a wave holds whole groups of planes");
    static_assert(BM % 8 == 0 && BN % 8 == 0, "pieces are eight rows");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int64_t row0 = (int64_t)(blockIdx.x % g.tiles_m) * BM, col0 = (int64_t)(blockIdx.x / g.tiles_m) * BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wr = wave / WN, wc = wave % WN;
    const int fr = lane & 15, fq = lane >> 4;

    i32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    const int8_t* src[PPW];
    int dst[PPW];
    {
        const int pr = lane >> 3, pc = lane & 7;
#pragma unroll
        for (int s = 0; s < PPW; ++s) {
            const int q = min(s * NW + wave, PIECES - 1);
            const int R = q * 8 + pr;
            if (R < BM) {
                src[s] = g.A + min(row0 + R, g.rows - 1) * g.lda + (pc ^ (R & 7)) * 16;
            } else {
                const int b = R - BM, key = (b & 3) | (((b >> KB) & 1) << 2);
                src[s] = g.B + min(col0 + b, g.N - 1) * g.ldb + (pc ^ key) * 16;
            }
            dst[s] = q * 1024;
        }
    }
    auto issue = [&](int kt, int buf) {
#pragma unroll
        for (int s = 0; s < PPW; ++s)
            __builtin_amdgcn_global_load_lds((glb_ptr_t)(src[s] + (int64_t)kt * 128), (lds_ptr_t)(lds + buf * STAGE_BYTES + dst[s]), 16, 0, 0);
    };
    issue(0, 0);
    const int x0 = (fq ^ (fr & 7)) * 16;
    const int a_off = (wr * 16 * FM + fr) * 128;
    const int b_off = (BM + wc * 16 * FN + (fr >> 2) * 4 * FN + (fr & 3)) * 128;
    for (int kt = 0; kt < g.steps; ++kt) {
        const int buf = kt & 1;
        wait_vmcnt<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (kt + 1 < g.steps) issue(kt + 1, buf ^ 1);
        const char* a_base = lds + buf * STAGE_BYTES + a_off;
        const char* b_base = lds + buf * STAGE_BYTES + b_off;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const int x = x0 ^ (ks * 64);
            i32x4 af[FM], bf[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) bf[j] = *(const i32x4*)(b_base + j * 4 * 128 + x);
#pragma unroll
            for (int i = 0; i < FM; ++i) af[i] = *(const i32x4*)(a_base + i * 16 * 128 + x);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j], af[i], acc[i][j], 0, 0, 0);
        }
    }

    const int64_t n0 = col0 + wc * 16 * FN + fq * 4 * FN, left = g.N - n0;
    if (left <= 0) return;
    float sb[4 * FN], bias[4 * FN];
#pragma unroll
    for (int c = 0; c < 4 * FN; ++c) {
        const int64_t n = min(n0 + c, g.N - 1);
        sb[c] = g.sb ? g.sb[n] : 1.f;
        bias[c] = g.bias ? load_as_f32(g.bias, n, g.dtype) : 0.f;
    }
    const int64_t group0 = (row0 / 16 + wr * FM) / PLANES;
#pragma unroll
    for (int i = 0; i < FM / PLANES; ++i) {
        const int64_t m = (group0 + i) * 16 + fr;
        if (m >= g.M) continue;
        const float sa = g.sa[m];
        auto value = [&](int c) {
            float v = (float)acc[i * PLANES][c >> 2][c & 3];
#pragma unroll
            for (int p = 1; p < PLANES; ++p) v = v * 256.f + (float)acc[i * PLANES + p][c >> 2][c & 3];
            v = (v * sa) * sb[c];
            return g.bias ? v + bias[c] : v;
        };
        if (g.dtype == SLIM_DTYPE_F32) store_row<4 * FN>((float*)g.out + m * g.ldo + n0, left, value);
        else if (g.dtype == SLIM_DTYPE_BF16) store_row<4 * FN>((bf16_t*)g.out + m * g.ldo + n0, left, [&](int c) { return f32_to_bf16(value(c)); });
        else store_row<4 * FN>((_Float16*)g.out + m * g.ldo + n0, left, [&](int c) { return (_Float16)value(c); });
    }
}

template <int PLANES, int FM, int FN, int WM, int WN>
int launch_gemm8(Gemm8Args g, hipStream_t st) {
    constexpr int BM = 16 * FM * WM, BN = 16 * FN * WN, bytes = 2 * (BM + BN) * 128;
    g.tiles_m = (int)ceil_div64(g.rows, BM);
    g.tiles_n = (int)ceil_div64(g.N, BN);
    auto kernel = gemm8_kernel<PLANES, FM, FN, WM, WN>;
    SLIM_REQUIRE((int64_t)g.tiles_m * g.tiles_n * 64 * WM * WN < (int64_t)1 << 32, "gemm8: the result is too large for one launch");
    SLIM_HIP(slim_allow_dynamic_lds((const void*)kernel, bytes));
    kernel<<<(unsigned)((int64_t)g.tiles_m * g.tiles_n), 64 * WM * WN, bytes, st>>>(g);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

template <int PLANES>
int gemm8(const Gemm8Args& g, hipStream_t st) {
    SLIM_PROF("gemm8", st, (double)g.rows * g.steps * 128 + (double)g.N * g.steps * 128 + (double)g.M * g.N * 2,
              2.0 * g.rows * g.N * g.steps * 128);
    return launch_gemm8<PLANES, PLANES == 3 ? 3 : 4, 4, 2, 2>(g, st);
}

// ---- codes [N, K] -> codes [K, N] -----------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void transpose8_kernel(const int8_t* __restrict__ in, int64_t N, int64_t K, int64_t ld, int8_t* __restrict__ out,
                                                         int64_t ldt) {
    __shared__ int8_t tile[64][68];
    const int64_t n0 = (int64_t)blockIdx.y * 64, k0 = (int64_t)blockIdx.x * 64;
    const int c = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < 64; r += 4) tile[r][c] = n0 + r < N && k0 + c < K ? in[(n0 + r) * ld + k0 + c] : 0;
    __syncthreads();
    for (int r = threadIdx.x >> 6; r < 64; r += 4)
        if (k0 + r < K && n0 + c < ldt) out[(k0 + r) * ldt + n0 + c] = tile[c][r];
}

int64_t pad128(int64_t k) { return (k + 127) / 128 * 128; }
int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }
int planes_of(int dtype) { return dtype == SLIM_DTYPE_F32 ? 3 : 2; }
bool known(int dtype) { return dtype == SLIM_DTYPE_F32 || dtype == SLIM_DTYPE_BF16 || dtype == SLIM_DTYPE_F16; }
int64_t element_size(int dtype) { return dtype == SLIM_DTYPE_F32 ? 4 : 2; }

}  // namespace

// the longest reduction whose sums of products of codes in [-128, 127] fit 32 bits
#define SLIM_INT8_MAX_REDUCTION 131071
// rows and columns: a workgroup of 256 threads each stays below a grid's 2^32 threads
#define SLIM_INT8_MAX_DIM ((1 << 24) - 1)

extern "C" int64_t slim_rows8_ld(int64_t K) { return K > 0 ? pad128(K) : 0; }

extern "C" int slim_quantize_rows8(const void* x, int dtype, int64_t R, int64_t K, int64_t ldx, int8_t* codes, int64_t ldc, float* scale,
                                   void* stream) {
    SLIM_REQUIRE(x && codes && scale && R > 0 && K > 0 && ldx >= K, "slim_quantize_rows8: bad arguments");
    SLIM_REQUIRE(known(dtype), "slim_quantize_rows8: unknown element type %d", dtype);
    SLIM_REQUIRE(R <= SLIM_INT8_MAX_DIM, "slim_quantize_rows8: too many rows");
    SLIM_REQUIRE(ldc >= pad128(K) && ldc % 16 == 0 && (uintptr_t)codes % 16 == 0,
                 "slim_quantize_rows8: rows of codes hold slim_rows8_ld(K) bytes and start at multiples of 16");
    SLIM_PROF("quantize_rows8", stream, (double)R * K * (element_size(dtype) + 1) + 4.0 * R);
    return quantize_rows_any<1>(x, dtype, R, K, ldx, nullptr, codes, ldc, scale, (hipStream_t)stream);
}

extern "C" int slim_transpose8(const int8_t* codes, int64_t N, int64_t K, int64_t ld, int8_t* codes_t, int64_t ldt, void* stream) {
    SLIM_REQUIRE(codes && codes_t && codes != codes_t && N > 0 && K > 0 && ld >= K && ldt >= pad128(N), "slim_transpose8: bad arguments");
    SLIM_REQUIRE(ceil_div64(ldt, 64) <= 65535, "slim_transpose8: too many rows");
    dim3 grid((unsigned)ceil_div64(K, 64), (unsigned)ceil_div64(ldt, 64));
    transpose8_kernel<<<grid, 256, 0, (hipStream_t)stream>>>(codes, N, K, ld, codes_t, ldt);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

extern "C" int64_t slim_gemm8_workspace_bytes(int64_t M, int64_t N, int64_t K) { return 0; }

extern "C" int slim_gemm8_nt(const int8_t* a, int64_t lda, const float* sa, const int8_t* b, int64_t ldb, const float* sb, int64_t M, int64_t N,
                             int64_t K, const void* bias, int dtype, void* out, int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
    SLIM_REQUIRE(a && sa && b && sb && out && M > 0 && N > 0 && K > 0 && ldo >= N, "slim_gemm8_nt: bad arguments");
    SLIM_REQUIRE(known(dtype), "slim_gemm8_nt: unknown element type %d", dtype);
    SLIM_REQUIRE(K <= SLIM_INT8_MAX_REDUCTION && M <= SLIM_INT8_MAX_DIM && N <= SLIM_INT8_MAX_DIM, "slim_gemm8_nt: too large");
    SLIM_REQUIRE(lda >= pad128(K) && ldb >= pad128(K) && lda % 16 == 0 && ldb % 16 == 0 && (uintptr_t)a % 16 == 0 && (uintptr_t)b % 16 == 0,
                 "slim_gemm8_nt: rows of codes hold slim_rows8_ld(K) bytes and start at multiples of 16");
    SLIM_REQUIRE(workspace_bytes >= slim_gemm8_workspace_bytes(M, N, K) && (workspace || workspace_bytes == 0) && (uintptr_t)workspace % 16 == 0,
                 "slim_gemm8_nt: workspace too small or misaligned");
    Gemm8Args g{a, b, lda, ldb, M, M, N, (int)(pad128(K) / 128), sa, sb, bias, out, ldo, dtype, 0, 0};
    return gemm8<1>(g, (hipStream_t)stream);
}

extern "C" int64_t slim_linear8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    (void)N;
    return M > 0 && K > 0 ? align256(M * pad128(K)) + align256(M * 4) : 0;
}

extern "C" int slim_linear8_forward(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, const int8_t* codes, const float* scale, int64_t N,
                                    const void* bias, void* y, int64_t ldy, void* workspace, int64_t workspace_bytes, void* stream) {
    SLIM_REQUIRE(x && codes && scale && y && workspace && M > 0 && N > 0 && K > 0 && ldx >= K && ldy >= N, "slim_linear8_forward: bad arguments");
    SLIM_REQUIRE(workspace_bytes >= slim_linear8_workspace_bytes(M, N, K) && (uintptr_t)workspace % 16 == 0,
                 "slim_linear8_forward: workspace too small or misaligned");
    int8_t* xc = (int8_t*)workspace;
    float* sx = (float*)(xc + align256(M * pad128(K)));
    const int rc = slim_quantize_rows8(x, dtype, M, K, ldx, xc, pad128(K), sx, stream);
    if (rc) return rc;
    return slim_gemm8_nt(xc, pad128(K), sx, codes, pad128(K), scale, M, N, K, bias, dtype, y, ldy, nullptr, 0, stream);
}

extern "C" int64_t slim_linear8_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype) {
    (void)K;
    return M > 0 && N > 0 && known(dtype) ? align256((M + 15) / 16 * 16 * planes_of(dtype) * pad128(N)) + align256(M * 4) : 0;
}

extern "C" int slim_linear8_backward(const void* dy, int dtype, int64_t lddy, int64_t M, int64_t N, const int8_t* codes_t, const float* scale, int64_t K,
                                     void* dx, int64_t lddx, void* workspace, int64_t workspace_bytes, void* stream) {
    SLIM_REQUIRE(dy && codes_t && scale && dx && workspace && M > 0 && N > 0 && K > 0 && lddy >= N && lddx >= K, "slim_linear8_backward: bad arguments");
    SLIM_REQUIRE(known(dtype), "slim_linear8_backward: unknown element type %d", dtype);
    SLIM_REQUIRE(N <= SLIM_INT8_MAX_REDUCTION && M <= SLIM_INT8_MAX_DIM && K <= SLIM_INT8_MAX_DIM, "slim_linear8_backward: too large");
    SLIM_REQUIRE(workspace_bytes >= slim_linear8_backward_workspace_bytes(M, N, K, dtype) && (uintptr_t)workspace % 16 == 0,
                 "slim_linear8_backward: workspace too small or misaligned");
    SLIM_REQUIRE((uintptr_t)codes_t % 16 == 0, "slim_linear8_backward: codes must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    const int planes = planes_of(dtype);
    const int64_t rows = (M + 15) / 16 * 16 * planes, ld = pad128(N);
    int8_t* q = (int8_t*)workspace;
    float* sq = (float*)(q + align256(rows * ld));
    const int rc = planes == 3 ? quantize_rows_any<3>(dy, dtype, M, N, lddy, scale, q, ld, sq, st)
                               : quantize_rows_any<2>(dy, dtype, M, N, lddy, scale, q, ld, sq, st);
    if (rc) return rc;
    Gemm8Args g{q, codes_t, ld, ld, rows, M, K, (int)(ld / 128), sq, nullptr, nullptr, dx, lddx, dtype, 0, 0};
    return planes == 3 ? gemm8<3>(g, st) : gemm8<2>(g, st);
}
