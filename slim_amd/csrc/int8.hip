// Linears in 8-bit integers: rows quantised to int8 codes with one fp32 scale each (tokens of an activation, output channels
// of a weight), and the product of two such matrices on the int8 matrix instructions with the scales in its epilogue (the gradient
// with respect to the input: int8grad.hip).  The reference only emulates quantised inputs and weights with dense floating-point
// products (slim/quantization/quantization.py:219-263, :266-304).
#include "int8.hpp"

namespace {

// ---- rows -> codes --------------------------------------------------------------------------------------------------
// a = max |x| over the row, scale = a / 127, q = rint(x * (127 / a)).  Rows with a < 2^-100 become zero (scale 0); rows that hold an
// infinity or a NaN get the scale NaN and zero codes, which makes every product with them NaN.
struct RowScale {
    float scale, inverse;
    bool none;                                           // nothing to keep, or nothing that could be kept
};
__device__ __forceinline__ RowScale row_scale(uint32_t max_bits) {
    const float a = __uint_as_float(max_bits);
    const bool bad = max_bits >= 0x7f800000u, none = bad || a < 0x1p-100f;
    return {bad ? __uint_as_float(0x7fc00000u) : none ? 0.f : a / 127.f, none ? 0.f : 127.f / a, none};
}

__device__ __forceinline__ uint2 encode(const float x[8], float r) {
    uint32_t out[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j >> 2] |= (uint32_t)((int)rintf(x[j] * r) & 255) << (8 * (j & 3));
    return make_uint2(out[0], out[1]);
}

// WPR waves work on a row (one: four rows per workgroup; four or sixteen: one); each thread keeps NV pieces of eight elements in registers, so
// the row is read once, with loads that do not stay in the caches (28672 x 8192 bf16: 111 us, 6.3 TB/s; 127 without).
// NV = 0: rows too long for that are read twice.
template <typename T, int NV, int WPR>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void quantize_rows_kernel(const T* __restrict__ x, int64_t R, int64_t K, int64_t ldx,
                                                            int8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scale) {
    constexpr int TPR = 64 * WPR;                        // threads of a row
    __shared__ uint32_t part[WPR];
    const int wave = threadIdx.x >> 6;
    const int64_t row = WPR > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (WPR == 1 && row >= R) return;
    const int t = WPR > 1 ? threadIdx.x : threadIdx.x & 63;
    const T* src = x + row * ldx;
    float keep[NV > 0 ? NV : 1][8];
    uint32_t m = 0;
    auto fetch = [&](int64_t c, float v[8]) { load8<(NV > 0)>(src + c, K - c, v); };
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
    if (WPR > 1) {
        if ((threadIdx.x & 63) == 0) part[wave] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WPR; ++i) m = max(m, part[i]);
    }
    const RowScale rs = row_scale(m);
    if (t == 0) scale[row] = rs.scale;
    const int64_t end = (K + 127) / 128 * 128;
    auto put = [&](int64_t c, float v[8]) {
        if (rs.none) {                                   // (x * 0 would be a NaN for what is not finite)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        }
        *(uint2*)(codes + row * ldc + c) = encode(v, rs.inverse);
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

template <typename T>
int quantize_rows(const T* x, int64_t R, int64_t K, int64_t ldx, int8_t* codes, int64_t ldc, float* scale, hipStream_t st) {
    const int64_t pieces = (K + 127) / 128 * 16;         // pieces of eight codes in a padded row
#define SLIM_ROWS(NV, WPR)                                                                                                  \
    do {                                                                                                                    \
        SLIM_REQUIRE(R * 64 * WPR < ((int64_t)1 << 32) - 1024, "slim_quantize_rows8: too many rows of this length for one launch"); \
        quantize_rows_kernel<T, NV, WPR><<<(unsigned)(WPR > 1 ? R : ceil_div64(R, 4)), WPR == 16 ? 1024 : 256, 0, st>>>(x, R, K, ldx, codes, ldc, scale); \
    } while (0)
    if (pieces <= 64) SLIM_ROWS(1, 1);
    else if (pieces <= 128) SLIM_ROWS(2, 1);
    else if (pieces <= 256) SLIM_ROWS(4, 1);
    else if (pieces <= 512) SLIM_ROWS(2, 4);
    else if (pieces <= 1024) SLIM_ROWS(4, 4);
    else if (pieces <= 2048 && R >= 4096) SLIM_ROWS(8, 4);             // (8192 x 13824 bf16: 63 us, with sixteen waves a row 71; 301 rows 5.4 and 4.9)
    else if (pieces <= 2048) SLIM_ROWS(2, 16);
    else if (pieces <= 4096) SLIM_ROWS(4, 16);
    else SLIM_ROWS(0, 16);
#undef SLIM_ROWS
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

int quantize_rows_any(const void* x, int dtype, int64_t R, int64_t K, int64_t ldx, int8_t* codes, int64_t ldc, float* scale, hipStream_t st) {
    if (dtype == SLIM_DTYPE_F32) return quantize_rows<float>((const float*)x, R, K, ldx, codes, ldc, scale, st);
    if (dtype == SLIM_DTYPE_BF16) return quantize_rows<bf16_t>((const bf16_t*)x, R, K, ldx, codes, ldc, scale, st);
    return quantize_rows<_Float16>((const _Float16*)x, R, K, ldx, codes, ldc, scale, st);
}

// ---- codes x codes --------------------------------------------------------------------------------------------------
struct Gemm8Args {
    const int8_t* A;                                     // [M, lda]: rows of codes
    const int8_t* B;                                     // [N, ldb]
    int64_t lda, ldb;
    int64_t M, N;
    int steps;                                           // 128-byte steps of the reduction
    const float* sa;                                     // [M]
    const float* sb;                                     // [N]
    const void* bias;                                    // [N] of the output's type, or null
    void* out;
    int64_t ldo;
    int dtype;
    int tiles_m, tiles_n;
    int splits, steps_per_split;                         // slices of the reduction, each into a slab of its own
    int32_t* slab;                                       // [splits][tiles_m * BM][tiles_n * BN], or null: one slice, results written here
    int rest_n;                                          // columns of narrower tiles behind the tiles_n full ones (0: none)
};

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
    if (dtype == SLIM_DTYPE_F32) return ((const float*)p)[i];
    if (dtype == SLIM_DTYPE_BF16) return bf16_to_f32(((const bf16_t*)p)[i]);
    return (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ void store_as(void* p, int64_t i, int dtype, float v) {
    if (dtype == SLIM_DTYPE_F32) ((float*)p)[i] = v;
    else if (dtype == SLIM_DTYPE_BF16) ((bf16_t*)p)[i] = f32_to_bf16(v);
    else ((_Float16*)p)[i] = (_Float16)v;
}

// A wave's sums, scaled, with the bias, rounded and stored: rows 16 (group0 + i) + fr of the result.
template <int FM, int FN>
__device__ __forceinline__ void write_results(const Gemm8Args& g, const i32x4 (&acc)[FM][FN], const float (&sa)[FM], const float (&sb)[4 * FN],
                                              int64_t group0, int64_t n0, int fr, int fq) {
    float bias[4 * FN];
#pragma unroll
    for (int c = 0; c < 4 * FN; ++c) bias[c] = 0.f;
    if (g.bias) {
        auto load = [&](const auto* p) { Columns<FN>::each(n0, fq, [&](auto count, int c, int64_t n) { load_run<count.value>(p + n, g.N - n, bias + c); }); };
        if (g.dtype == SLIM_DTYPE_F32) load((const float*)g.bias);
        else if (g.dtype == SLIM_DTYPE_BF16) load((const bf16_t*)g.bias);
        else load((const _Float16*)g.bias);
#pragma unroll
        for (int c = 0; c < 4 * FN; ++c) asm volatile("" : "+v"(bias[c]));     // (arrived: no wait for them is left to whoever follows)
    }
    auto rows = [&](auto* out, auto convert) {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int64_t m = (group0 + i) * 16 + fr;
            if (m >= g.M) continue;
            auto value = [&](int c) {
                const float v = ((float)acc[i][c >> 2][c & 3] * sa[i]) * sb[c];
                return convert(g.bias ? v + bias[c] : v);
            };
            Columns<FN>::each(n0, fq, [&](auto count, int c, int64_t n) { store_run<count.value>(out + m * g.ldo + n, g.N - n, [&](int k) { return value(c + k); }); });
        }
    };
    if (g.dtype == SLIM_DTYPE_F32) rows((float*)g.out, [](float v) { return v; });
    else if (g.dtype == SLIM_DTYPE_BF16) rows((bf16_t*)g.out, [](float v) { return f32_to_bf16(v); });
    else rows((_Float16*)g.out, [](float v) { return (_Float16)v; });
}

// D = A B^T on 16 x 16 x 64 int8 instructions, operands delivered by LDS-DMA (16 bytes per lane) a 128-byte step ahead, two
// stages.  LDS image of a stage: BM rows of A, then BN rows of B, 128 bytes each; the 16-byte piece c of a row is stored at
// c ^ key(row), applied on the source side.  The result is computed transposed (B's fragment as the first operand): a lane then holds
// consecutive columns of one row, and with the rows of B dealt to the fragments in runs of four (row (r / 4) * 4 FN + 4 j + r % 4
// for lane row r of fragment j) all 4 FN of them are consecutive, so a lane stores its part of a row in 16-byte pieces.
// key(row) = the lane row's low three bits in either operand, which spreads eight lanes over the eight pieces of a row (no bank
// conflicts measured).
// Fragments are double-buffered in registers: while a step's first half (64 bytes) is multiplied its second half is read, and
// while that is multiplied the next step's first half is read and the stage just emptied is requested again -- one read or request
// per two matrix instructions, one barrier per step.  Left to the compiler the reads come in a burst that the matrix instructions
// wait for (4096 x 11008 x 4096 on 256 x 256 tiles: 176 us against 169; 8192^3: 404 against 393 us, 2.8e15 operations/s).
// Whole 128-byte lines per row: with 64-byte steps, which would allow four stages, the requests take twice as long (8 % of the whole).
// What bounds it: without requests the loop takes 87 % of its time, without fragment reads as well 77 %; the matrix instructions alone
// hold the clock at about 2.1 GHz.
template <int FM, int FN, int WM, int WN, int STAGES>
__device__ __forceinline__ void gemm8_tile(const Gemm8Args& g, char* lds, int64_t row0, int64_t col0, int slice) {
    constexpr int BM = 16 * FM * WM, BN = 16 * FN * WN, NW = WM * WN;
    constexpr int PIECES = (BM + BN) / 8, PPW = (PIECES + NW - 1) / NW;     // (a last wave repeats the final piece)
    constexpr int STAGE_BYTES = (BM + BN) * 128;
    constexpr int PAIRS = FN / 2 * 32;                   // columns (rows of B) of a wave's fragments taken in pairs
    constexpr int READS = FM + FN, PRODUCTS = FM * FN;
    constexpr int PACE1 = PRODUCTS / READS > 0 ? PRODUCTS / READS : 1, PACE2 = PRODUCTS / (READS + PPW) > 0 ? PRODUCTS / (READS + PPW) : 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WN, wc = wave % WN;
    const int fr = lane & 15, fq = lane >> 4;

    i32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    // this lane's sources: row lane / 8 of each of the wave's pieces; rows behind the last are read from the last one
    const int8_t* base[PPW];
    uint32_t off[PPW];
    {
        const int pr = lane >> 3, pc = lane & 7;
#pragma unroll
        for (int s = 0; s < PPW; ++s) {
            const int q = min(s * NW + wave, PIECES - 1);
            if (q * 8 < BM) {
                const int R = q * 8 + pr;
                base[s] = g.A + row0 * g.lda;
                off[s] = (uint32_t)(min((int64_t)R, g.M - 1 - row0) * g.lda) + (pc ^ (R & 7)) * 16;
            } else {
                const int R = q * 8 - BM + pr, w = R % (16 * FN), key = w < PAIRS ? (w & 3) | (((w >> 3) & 1) << 2) : w & 7;
                base[s] = g.B + col0 * g.ldb;
                off[s] = (uint32_t)(min((int64_t)R, g.N - 1 - col0) * g.ldb) + (pc ^ key) * 16;
            }
        }
    }
    const int first = slice * g.steps_per_split, steps = min(g.steps_per_split, g.steps - first);
    auto request = [&](int kt, int stage) {              // (behind the last step: the last one again, which nothing reads)
        const int64_t k = (int64_t)(first + min(kt, steps - 1)) * 128;
#pragma unroll
        for (int s = 0; s < PPW; ++s)
            __builtin_amdgcn_global_load_lds((glb_ptr_t)(base[s] + k + off[s]), (lds_ptr_t)(lds + stage * STAGE_BYTES + min(s * NW + wave, PIECES - 1) * 1024), 16, 0, 0);
    };
#pragma unroll
    for (int st = 0; st < STAGES; ++st) request(st, st);
    const int x0 = (fq ^ (fr & 7)) * 16;
    const int a_off = (wr * 16 * FM + fr) * 128 + x0;
    const int b_off = (BM + wc * 16 * FN + (fr >> 2) * 8 + (fr & 3)) * 128 + x0;
    const int odd_off = (BM + wc * 16 * FN + PAIRS + fr) * 128 + x0;     // the last fragment of an odd number
    i32x4 af[2][FM], bf[2][FN];
    auto read = [&](int half, int stage) {
        const char* a = lds + ((stage * STAGE_BYTES + a_off) ^ (half * 64));
        const char* b = lds + ((stage * STAGE_BYTES + b_off) ^ (half * 64));
#pragma unroll
        for (int j = 0; j < FN / 2 * 2; ++j) bf[half][j] = *(const i32x4*)(b + ((j >> 1) * 32 + (j & 1) * 4) * 128);
        if (FN % 2) bf[half][FN - 1] = *(const i32x4*)(lds + ((stage * STAGE_BYTES + odd_off) ^ (half * 64)));
#pragma unroll
        for (int i = 0; i < FM; ++i) af[half][i] = *(const i32x4*)(a + i * 16 * 128);
    };
    auto multiply = [&](int half) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[half][j], af[half][i], acc[i][j], 0, 0, 0);
    };
    wait_vmcnt<(STAGES - 1) * PPW>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, 0);
    int stage = 0;
    for (int kt = 0; kt < steps; ++kt) {
        const int next = stage + 1 == STAGES ? 0 : stage + 1;
        __builtin_amdgcn_sched_barrier(0);
        read(1, stage);
        multiply(0);
#pragma unroll
        for (int s = 0; s < READS; ++s) {
            __builtin_amdgcn_sched_group_barrier(0x008, PACE1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        // this wave's reads of the stage are done and its requests of the next one have landed; behind the barrier so are everyone's
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_vmcnt<(STAGES - 2) * PPW>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        read(0, next);
        request(kt + STAGES, stage);
        multiply(1);
#pragma unroll
        for (int s = 0; s < READS; ++s) {
            __builtin_amdgcn_sched_group_barrier(0x008, PACE2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
#pragma unroll
        for (int s = 0; s < PPW; ++s) {
            __builtin_amdgcn_sched_group_barrier(0x008, PACE2, 0);
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        stage = next;
    }
    wait_vmcnt<0>();                                     // (the requests behind the last step land before the LDS is given up)

    const int64_t n0 = col0 + wc * 16 * FN;              // value 8 c + k of a lane: column n0 + 32 c + 8 fq + k, of an odd fragment n0 + PAIRS + 4 fq + k
    if (g.slab) {
        int32_t* slab = g.slab + ((int64_t)slice * g.tiles_m * BM + row0 + wr * 16 * FM + fr) * ((int64_t)g.tiles_n * BN) + n0;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                *(i32x4*)(slab + (int64_t)i * 16 * g.tiles_n * BN + (j < FN / 2 * 2 ? (j >> 1) * 32 + fq * 8 + (j & 1) * 4 : PAIRS + fq * 4)) = acc[i][j];
        return;
    }
    // everything the epilogue reads is requested at once (loaded row by row it costs a trip to memory per row: 4 us of a 256 x 256 tile)
    const int64_t group0 = row0 / 16 + wr * FM;
    float sa[FM], sb[4 * FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[i] = g.sa[min((group0 + i) * 16 + fr, g.M - 1)];
    Columns<FN>::each(n0, fq, [&](auto count, int c, int64_t n) { load_run<count.value>(g.sb + n, g.N - n, sb + c); });
    write_results<FM, FN>(g, acc, sa, sb, group0, n0, fr, fq);
}

template <int FM, int FN, int WM, int WN, int STAGES, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void gemm8_kernel(const Gemm8Args g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int tm, tn, slice;
    tile_of(blockIdx.x, g.tiles_m, g.tiles_n, g.splits, tm, tn, slice);
    gemm8_tile<FM, FN, WM, WN, STAGES>(g, lds, (int64_t)tm * 16 * FM * WM, (int64_t)tn * 16 * FN * WN, slice);
}

// The same product by workgroups that stay, for more tiles than CUs: each takes every gridDim.x-th tile, and the stream of requests
// runs on from one tile into the next, so that the next tile's first steps travel while the finished one is scaled and stored, and its
// stores drain under the next tile's products (us, a workgroup a tile / so: 4096 x 11008 x 4096 169 / 164, 8192^3 393 / 382, 8192 x 4096 x
// 1024 43 / 38).  REST > 0: behind the columns of full tiles lie g.rest_n columns of tiles of 16 REST WN columns, which fill the last
// round of workgroups better.  The scales of a tile come by LDS-DMA while it is multiplied.  (g.steps >= 2)
template <int FM, int FN, int WM, int WN, int REST>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm8_stream_kernel(const Gemm8Args g) {
    constexpr int BM = 16 * FM * WM, BN = 16 * FN * WN, NW = WM * WN, STAGE_BYTES = (BM + BN) * 128;
    constexpr int ALOADS = BM / 8 / NW, LOADS = (BM + BN) / 8 / NW;      // requests of a wave and step: eight rows each, A's first
    static_assert(BM % 64 == 0 && BM % (8 * NW) == 0 && 16 * WN % (8 * NW) == 0 && BM + BN <= 64 * NW, "requests and scales are dealt out evenly");
    constexpr int LEAST = REST && REST < FN ? REST : FN, STORES = FM * Columns<LEAST>::RUNS, STORES32 = FM * LEAST;     // of a whole tile, at least
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* const scales = (float*)(lds + 2 * STAGE_BYTES);              // [BM] of the rows, [BN] of the columns
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WN, wc = wave % WN, fr = lane & 15, fq = lane >> 4;
    const int full = g.tiles_m * g.tiles_n, total = full + g.tiles_m * g.rest_n, steps = g.steps;
    // what depends on the lane and is needed once a tile is computed anew, not kept over the loop, where 250 of 256 registers are taken
    auto this_lane = []() {
        uint32_t zero = 0;
        asm volatile("" : "+v"(zero));
        return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
    };
    auto place = [&](int b, int64_t& row0, int64_t& col0) {
        int tm, tn, slice;
        if (REST && b >= full) {
            tile_of(b - full, g.tiles_m, g.rest_n, 1, tm, tn, slice);
            col0 = (int64_t)g.tiles_n * BN + (int64_t)tn * 16 * REST * WN;
        } else {
            tile_of(b, g.tiles_m, g.tiles_n, 1, tm, tn, slice);
            col0 = (int64_t)tn * BN;
        }
        row0 = (int64_t)tm * BM;
    };
    // where the requests are: tile, step, this lane's sources in it (as in gemm8_tile; in a narrow tile the rows behind its own are never read)
    int at = blockIdx.x, ks = 0;
    const int8_t *pa, *pb;
    uint32_t off[LOADS];
    auto aim = [&]() {
        int64_t row0, col0;
        place(at, row0, col0);
        pa = g.A + row0 * g.lda, pb = g.B + col0 * g.ldb;
        const bool narrow = REST && at >= full;
        const int l = this_lane(), pr = l >> 3, pc = l & 7;
#pragma unroll
        for (int s = 0; s < LOADS; ++s) {
            const int R = (s * NW + wave) * 8 + pr;
            if (s < ALOADS) {
                off[s] = (uint32_t)(min((int64_t)R, g.M - 1 - row0) * g.lda) + (pc ^ (R & 7)) * 16;
            } else {
                const int r = R - BM, w = narrow ? r % (16 * (REST ? REST : 1)) : r % (16 * FN), pairs = narrow ? Columns<REST>::PAIRS : Columns<FN>::PAIRS;
                const int key = w < pairs ? (w & 3) | (((w >> 3) & 1) << 2) : w & 7;
                off[s] = (uint32_t)(min((int64_t)r, g.N - 1 - col0) * g.ldb) + (pc ^ key) * 16;
            }
        }
    };
    auto advance = [&]() {                               // (behind the last tile: its last step again, which nothing reads)
        if (at + (int)gridDim.x < total) at += gridDim.x, ks = 0, aim();
        else ks = steps - 1;
    };
    auto request = [&](auto loads, int stage) {
        const int64_t k = (int64_t)ks * 128;
#pragma unroll
        for (int s = 0; s < loads.value; ++s)
            __builtin_amdgcn_global_load_lds((glb_ptr_t)((s < ALOADS ? pa : pb) + k + off[s]), (lds_ptr_t)(lds + stage * STAGE_BYTES + (s * NW + wave) * 1024), 16, 0, 0);
        ++ks;
    };
    aim();
    request(std::integral_constant<int, LOADS>(), 0);
    request(std::integral_constant<int, LOADS>(), 1);    // (steps >= 2)
    wait_vmcnt<LOADS>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    int b = blockIdx.x, stage = 0;
    bool stores = false;                                 // the tile before stored all of its rows and columns
    auto tiles = [&](auto width, int end) {              // this workgroup's tiles in front of `end`, all `width` fragments wide
        constexpr int F = width.value, PAIRS = Columns<F>::PAIRS, L = ALOADS + (LOADS - ALOADS) * F / FN;
        constexpr int READS = FM + F, PRODUCTS = FM * F, PACE1 = PRODUCTS / READS, PACE2 = PRODUCTS / (READS + L);
        if (b >= end) return;
        const int x0 = (fq ^ (fr & 7)) * 16;
        const int a_off = (wr * 16 * FM + fr) * 128 + x0;
        const int b_off = (BM + wc * 16 * F + (fr >> 2) * 8 + (fr & 3)) * 128 + x0;
        const int odd_off = (BM + wc * 16 * F + PAIRS + fr) * 128 + x0;
        i32x4 af[2][FM], bf[2][F];
        auto read = [&](int half, int st) {
            const char* pa = lds + ((st * STAGE_BYTES + a_off) ^ (half * 64));
            const char* pb = lds + ((st * STAGE_BYTES + b_off) ^ (half * 64));
#pragma unroll
            for (int j = 0; j < F / 2 * 2; ++j) bf[half][j] = *(const i32x4*)(pb + ((j >> 1) * 32 + (j & 1) * 4) * 128);
            if (F % 2) bf[half][F - 1] = *(const i32x4*)(lds + ((st * STAGE_BYTES + odd_off) ^ (half * 64)));
#pragma unroll
            for (int i = 0; i < FM; ++i) af[half][i] = *(const i32x4*)(pa + i * 16 * 128);
        };
        for (; b < end; b += gridDim.x) {
            int64_t row0, col0;
            place(b, row0, col0);
            read(0, stage);                              // (again: kept over the end of the tile before they would not fit the registers)
            i32x4 acc[FM][F];
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
            auto multiply = [&](int half) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[half][j], af[half][i], acc[i][j], 0, 0, 0);
            };
            for (int kt = 0; kt < steps; ++kt) {
                if (ks >= steps) advance();
                __builtin_amdgcn_sched_barrier(0);
                read(1, stage);
                multiply(0);
#pragma unroll
                for (int s = 0; s < READS; ++s) {
                    __builtin_amdgcn_sched_group_barrier(0x008, PACE1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                // this wave's reads of the stage are done and its requests of the next one have landed (at a tile's first step they
                // are older than the stores of the tile before, which need not be waited for); behind the barrier so are everyone's
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (kt || !stores) wait_vmcnt<0>();
                else if (g.dtype == SLIM_DTYPE_F32) wait_vmcnt<STORES32>();
                else wait_vmcnt<STORES>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (kt == 0) {                           // every wave is past the tile before: this one's scales, for its end
                    const int t = wave * 64 + this_lane();
                    const float* src = wave * 64 < BM ? g.sa + min(row0 + t, g.M - 1) : g.sb + min(col0 + t - BM, g.N - 1);
                    if (wave * 64 < BM + BN) __builtin_amdgcn_global_load_lds((glb_ptr_t)src, (lds_ptr_t)(scales + wave * 64), 4, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                read(0, stage ^ 1);
                request(std::integral_constant<int, L>(), stage);
                multiply(1);
#pragma unroll
                for (int s = 0; s < READS; ++s) {
                    __builtin_amdgcn_sched_group_barrier(0x008, PACE2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
#pragma unroll
                for (int s = 0; s < L; ++s) {
                    __builtin_amdgcn_sched_group_barrier(0x008, PACE2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                stage ^= 1;
            }
            asm volatile("" ::: "memory");               // (no store moves in front of the requests)
            const int l = this_lane(), er = l & 15, eq = l >> 4;
            float sa[FM], sb[4 * F];
#pragma unroll
            for (int i = 0; i < FM; ++i) sa[i] = scales[(wr * FM + i) * 16 + er];
            const int64_t n0 = col0 + wc * 16 * F;
            Columns<F>::each(n0, eq, [&](auto count, int c, int64_t n) {
#pragma unroll
                for (int j = 0; j < count.value; ++j) sb[c + j] = scales[BM + (int)(n - col0) + j];
            });
            write_results<FM, F>(g, acc, sa, sb, row0 / 16 + wr * FM, n0, er, eq);
            asm volatile("" ::: "memory");
            stores = row0 + BM <= g.M && col0 + 16 * F * WN <= g.N;
        }
    };
    tiles(std::integral_constant<int, FN>(), full);
    if constexpr (REST > 0) tiles(std::integral_constant<int, REST>(), total);
    wait_vmcnt<0>();                                     // (the requests behind the last step land before the LDS is given up)
}

// The slices' sums added (whole numbers: any order gives the same), scaled and rounded: a thread per four columns.
__global__ __launch_bounds__(256) void join_slices_kernel(const Gemm8Args g, int64_t slab_rows, int64_t slab_cols) {
    const int64_t quads = (g.N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t m = i / quads, n = (i - m * quads) * 4;
    if (m >= g.M) return;
    i32x4 sum = i32x4{0, 0, 0, 0};
    const int32_t* src = g.slab + m * slab_cols + n;
    for (int z = 0; z < g.splits; ++z, src += slab_rows * slab_cols) sum += *(const i32x4*)src;
    const float sa = g.sa[m];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (n + c >= g.N) break;
        float v = ((float)sum[c] * sa) * g.sb[n + c];
        if (g.bias) v += load_as_f32(g.bias, n + c, g.dtype);
        store_as(g.out, m * g.ldo + n + c, g.dtype, v);
    }
}

// ---- which tile, how many slices ------------------------------------------------------------------------------------
// Every tile's time, as measured over 32 to 4096 rows of weights 1024 x 1024 to 5120 x 13824 (us): a workgroup's start and end, a
// 128-byte step while it has its CU to itself (few workgroups) and while all CUs, and both places of a CU where there are two, are
// taken.  Larger tiles need fewer bytes per product (256 x 256: 2.3e15 operations/s at 4096 x 11008 x 4096, 128 x 128: 1.7e15),
// smaller ones fill the chip sooner (300 x 4096 x 4096: 64 x 128 12 us, 256 x 256 38 us).  Slices of the reduction pay where tiles
// alone leave CUs idle over a long reduction (64 x 5120 x 13824: four slices 19 us, one 31 us), for the pass that adds them.
struct Tile {
    int bm, bn, places;                                  // workgroups that share a CU
    double ends, alone, full;
};
constexpr int TILES = 5;
constexpr Tile tiles[TILES] = {{256, 256, 1, 7.0, 1.02, 1.60}, {128, 256, 1, 5.0, 0.60, 0.97}, {128, 128, 1, 4.3, 0.34, 0.53},
                               {64, 128, 1, 3.6, 0.24, 0.345},     // four stages, a CU for each workgroup ...
                               {64, 128, 2, 3.4, 0.34, 0.65}};     // ... or three and two workgroups a CU
struct Plan {
    int tile = 0, splits = 1, steps_per_split = 0;
    int64_t tiles_m = 0, tiles_n = 0, slab_rows = 0, slab_cols = 0;
    int rest = 0;                                        // fragments (of 64 columns) of the narrower tiles behind the full ones
    int64_t rest_n = 0;
    bool stays() const { return tile == 0 && splits == 1 && steps_per_split >= 2 && tiles_m * (tiles_n + rest_n) > 256; }     // workgroups take several tiles
    int64_t slab_bytes() const { return splits > 1 ? splits * slab_rows * slab_cols * 4 : 0; }
};
Plan plan_gemm8(int64_t M, int64_t N, int64_t steps) {
    Plan best;
    double best_time = 1e30;
    for (int k = 0; k < TILES; ++k) {
        const Tile t = tiles[k];
        const int64_t tiles_m = ceil_div64(M, t.bm), tiles_n = ceil_div64(N, t.bn), count = tiles_m * tiles_n;
        for (int splits = 1; splits <= 8 && (splits == 1 || (steps >= 8 * splits && count * splits <= 256)); splits *= 2) {
            const int64_t each = ceil_div64(steps, splits), groups = count * splits, slots = 256 * t.places;
            const int64_t rest = groups % slots;
            auto round = [&](int64_t n) {                // n workgroups, at most `slots`
                const double busy = t.places == 2 ? (n > 256 ? 1.0 : 0.0) : n / 256.0;
                return t.ends + each * (t.alone + (t.full - t.alone) * busy);
            };
            double time = (groups / slots) * round(slots) + (rest ? round(rest) : 0.0);
            if (splits > 1) time += 3.0 + 2.0 * splits * count * t.bm * t.bn * 4 / 4e6;
            if (time < best_time) {
                best_time = time;
                best.tile = k, best.splits = (int)ceil_div64(steps, each), best.steps_per_split = (int)each;
                best.tiles_m = tiles_m, best.tiles_n = tiles_n, best.slab_rows = tiles_m * t.bm, best.slab_cols = tiles_n * t.bn;
            }
        }
    }
    // The largest tile's last round, when it is not full, on narrower tiles that fill it better (4096 x 11008: 512 full tiles and 240 of
    // 192 columns in place of 176 full ones: reduction 4096 150 us, full tiles 153; 2048 x 11008 88 and 96).
    if (best.tile == 0 && best.splits == 1 && best.steps_per_split >= 2 && best.tiles_m <= 256) {
        const int64_t count = best.tiles_m * best.tiles_n, columns = count / 256 * 256 / best.tiles_m;
        if (count > 256 && count % 256 && columns < best.tiles_n) {
            for (int rest = 3; rest >= 2; --rest) {
                const int64_t n = ceil_div64(N - columns * 256, 64 * rest);
                if (columns * best.tiles_m + n * best.tiles_m <= (count / 256 + 1) * 256) best.rest = rest, best.rest_n = n;
            }
            if (best.rest) best.tiles_n = columns;
        }
    }
    return best;
}

template <int TILE, int FM, int FN, int WM, int WN, int STAGES, int OCC>
int launch_gemm8(const Gemm8Args& g, const Plan& p, hipStream_t st) {
    constexpr int BM = 16 * FM * WM, BN = 16 * FN * WN, bytes = STAGES * (BM + BN) * 128;
    const int64_t blocks = p.tiles_m * p.tiles_n * p.splits;
    static_assert(tiles[TILE].bm == BM && tiles[TILE].bn == BN, "the plan's tile");
    SLIM_REQUIRE(blocks * 64 * WM * WN < (int64_t)1 << 32 && blocks < 0x7fffffff, "gemm8: the result is too large for one launch");
    auto kernel = gemm8_kernel<FM, FN, WM, WN, STAGES, OCC>;
    SLIM_HIP(slim_allow_dynamic_lds((const void*)kernel, bytes));
    kernel<<<(unsigned)blocks, 64 * WM * WN, bytes, st>>>(g);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

template <int REST>
int launch_stream8(const Gemm8Args& g, const Plan& p, hipStream_t st) {
    constexpr int bytes = (256 + 256) * (2 * 128 + 4);
    static_assert(tiles[0].bm == 256 && tiles[0].bn == 256, "the plan's tile");
    SLIM_REQUIRE(p.tiles_m * (p.tiles_n + p.rest_n) < 0x7fffffff - 256, "gemm8: the result is too large for one launch");
    auto kernel = gemm8_stream_kernel<8, 4, 2, 4, REST>;
    SLIM_HIP(slim_allow_dynamic_lds((const void*)kernel, bytes));
    kernel<<<256, 512, bytes, st>>>(g);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

int gemm8(Gemm8Args g, void* slab, hipStream_t st) {
    SLIM_PROF("gemm8", st, (double)(g.M + g.N) * g.steps * 128 + (double)g.M * g.N * element_size(g.dtype), 2.0 * g.M * g.N * g.steps * 128);
    const Plan p = plan_gemm8(g.M, g.N, g.steps);
    g.tiles_m = (int)p.tiles_m, g.tiles_n = (int)p.tiles_n;
    g.splits = p.splits, g.steps_per_split = p.steps_per_split, g.rest_n = (int)p.rest_n;
    g.slab = p.splits > 1 ? (int32_t*)slab : nullptr;
    int rc;
    if (p.stays() && p.rest == 3) rc = launch_stream8<3>(g, p, st);
    else if (p.stays() && p.rest == 2) rc = launch_stream8<2>(g, p, st);
    else if (p.stays()) rc = launch_stream8<0>(g, p, st);
    else if (p.tile == 0) rc = launch_gemm8<0, 8, 4, 2, 4, 2, 2>(g, p, st);
    else if (p.tile == 1) rc = launch_gemm8<1, 4, 4, 2, 4, 3, 2>(g, p, st);
    else if (p.tile == 2) rc = launch_gemm8<2, 4, 2, 2, 4, 4, 2>(g, p, st);
    else if (p.tile == 3) rc = launch_gemm8<3, 2, 2, 2, 4, 4, 2>(g, p, st);
    else rc = launch_gemm8<4, 2, 2, 2, 4, 3, 4>(g, p, st);
    if (rc || p.splits == 1) return rc;
    const int64_t threads = g.M * ((g.N + 3) / 4);
    join_slices_kernel<<<(unsigned)ceil_div64(threads, 256), 256, 0, st>>>(g, p.slab_rows, p.slab_cols);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

// ---- few tokens -----------------------------------------------------------------------------------------------------
// Up to 16 FM tokens: a workgroup owns 16 FN output channels over the whole reduction, each of its waves every NW-th 128-byte unit of
// it, so nothing is joined outside the workgroup.  A wave keeps STAGES units of its own (the weight's rows and the tokens') under way
// by LDS-DMA, eight whole 128-byte lines per request; as no other wave touches them it waits for its own requests only, and the one
// barrier is that in front of the sums' addition.  (Loaded straight into the matrix instructions' layout, 16 rows by 64 bytes a
// request, the weight takes half as long again.)
struct RingArgs {
    const int8_t* A;                                     // codes of the tokens
    int64_t lda;
    const float* sa;
    const int8_t* B;
    int64_t ldb;
    const float* sb;
    const void* bias;
    void* out;
    int64_t ldo;
    int dtype;
    int64_t M, N;
    int units;
};
// The waves' sums, `stride` bytes from one wave's to the next, added: a result per thread and turn, channel n of token m (the
// instruction's rows are channels, its columns tokens).  sa: the scales of the workgroup's tokens.
template <int FM, int FN, int NW>
__device__ __forceinline__ void wave_results(const RingArgs& g, const char* sums, int stride, const float* sa, int64_t m0, int64_t n0) {
    for (int t = threadIdx.x; t < 256 * FM * FN; t += 64 * NW) {
        const int n = t % (16 * FN), m = t / (16 * FN);
        if (m0 + m >= g.M || n0 + n >= g.N) continue;
        const int at = ((m >> 4) * FN + (n >> 4)) * 64 + ((n & 15) >> 2) * 16 + (m & 15);
        int sum = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum += ((const int*)(sums + w * stride))[at * 4 + (n & 3)];
        float v = ((float)sum * sa[m]) * g.sb[n0 + n];
        if (g.bias) v += load_as_f32(g.bias, n0 + n, g.dtype);
        store_as(g.out, (m0 + m) * g.ldo + n0 + n, g.dtype, v);
    }
}
template <int FM, int FN, int NW, int STAGES>
__global__ __launch_bounds__(64 * NW) void ring8_kernel(const RingArgs g) {
    constexpr int REQ = 2 * FM + 2 * FN, UNIT = REQ * 1024;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fq = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16 * FN, m0 = (int64_t)blockIdx.y * 16 * FM;
    char* const ring = lds + wave * STAGES * UNIT;
    uint32_t off[REQ];                                   // a request: eight rows, lane / 8, of which it takes piece (lane % 8) ^ row
    {
        const int pr = lane >> 3, pc = (lane & 7) ^ pr;
#pragma unroll
        for (int s = 0; s < REQ; ++s)
            off[s] = (s < 2 * FM ? (uint32_t)(min((int64_t)s * 8 + pr, g.M - 1 - m0) * g.lda) : (uint32_t)(min((int64_t)(s - 2 * FM) * 8 + pr, g.N - 1 - n0) * g.ldb)) + pc * 16;
    }
    const int8_t *const a0 = g.A + m0 * g.lda, *const b0 = g.B + n0 * g.ldb;
    const int mine = wave < g.units ? (g.units - wave + NW - 1) / NW : 0;
    auto request = [&](int i, int stage) {
        const int64_t k = (int64_t)(wave + i * NW) * 128;
#pragma unroll
        for (int s = 0; s < REQ; ++s)
            __builtin_amdgcn_global_load_lds((glb_ptr_t)((s < 2 * FM ? a0 : b0) + k + off[s]), (lds_ptr_t)(ring + stage * UNIT + s * 1024), 16, 0, 0);
    };
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
        if (i < mine) request(i, i);
    i32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    const int x0 = fr * 128 + (fq ^ (fr & 7)) * 16;
    int stage = 0;
    for (int i = 0; i < mine; ++i) {
        // the oldest unit has landed once only the younger ones are outstanding (at the end there are fewer of them: wait for all)
        if (i + STAGES <= mine) wait_vmcnt<(STAGES - 1) * REQ>();
        else wait_vmcnt<0>();
        const char* unit = ring + stage * UNIT;
        i32x4 a[FM][2], b[FN][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < FM; ++j) a[j][h] = *(const i32x4*)(unit + j * 2048 + (x0 ^ (h * 64)));
#pragma unroll
            for (int j = 0; j < FN; ++j) b[j][h] = *(const i32x4*)(unit + (FM + j) * 2048 + (x0 ^ (h * 64)));
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");               // (read before it is requested again)
        if (i + STAGES < mine) request(i + STAGES, stage);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int f = 0; f < FM; ++f) acc[f][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[j][h], a[f][h], acc[f][j], 0, 0, 0);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    // every wave's sums over its own ring, nothing of which is under way any more
    i32x4* const sums = (i32x4*)ring;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) sums[(i * FN + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    wave_results<FM, FN, NW>(g, lds, STAGES * UNIT, g.sa + m0, m0, n0);
}

template <int FM, int FN, int NW, int STAGES>
int launch_ring8_as(const RingArgs& g, hipStream_t st) {
    constexpr int bytes = NW * STAGES * (FM + FN) * 2048;
    auto kernel = ring8_kernel<FM, FN, NW, STAGES>;
    SLIM_HIP(slim_allow_dynamic_lds((const void*)kernel, bytes));
    kernel<<<dim3((unsigned)ceil_div64(g.N, 16 * FN), (unsigned)ceil_div64(g.M, 16 * FM)), 64 * NW, bytes, st>>>(g);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}
// Up to 32 tokens, measured over both (us with the tokens' quantisation, weights 4096 x 4096, 11008 x 4096 and 5120 x 13824): sixteen
// channels and eight waves 7.0, 13.8 and 21.5 for 16 tokens, 32 channels and four waves 8.0, 11.5 and 18.0; 8.2, 15.8 and 24.3 against
// 8.9, 13.5 and 19.2 for 32.  From 33 to 64 all rows in one workgroup and eight waves where two to a CU would fill the chip (40 x 4096
// x 11008: 12.8 against 15.4; but 64 x 1024 x 1024 3.7 against 3.2).
// Small results of more rows go the same way while every workgroup finds a place at once: four waves share a reduction that a tile
// walks step by step (rows x channels x reduction, us, tile / here: 128 x 512 x 2048 7.5 / 3.6, 512 x 512 x 8192 14.6 / 11.8).  First in
// workgroups of 32 rows by sixteen channels, two a CU, then in four times that, one a CU (128 x 4096 x 2048 7.6 / 6.4); with more of them
// the tiles win (512 workgroups of the second: 1024 x 1024 x 2048 8.1 / 11.5).
int takes_ring(int64_t M, int64_t N) {                   // 0: no; 1, 2: the smaller or the larger workgroups
    if (M <= 32) return 1;
    return ceil_div64(M, 32) * ceil_div64(N, 16) <= 512 ? 1 : ceil_div64(M, 64) * ceil_div64(N, 32) <= 256 ? 2 : 0;
}
int launch_ring8(const RingArgs& g, hipStream_t st) {
    SLIM_PROF("ring8", st, (double)(g.N + g.M) * g.units * 128 + (double)g.M * g.N * element_size(g.dtype), 2.0 * g.M * g.N * g.units * 128);
    const bool narrow = g.N <= 4096;
    if (g.M <= 16) return narrow ? launch_ring8_as<1, 1, 8, 3>(g, st) : launch_ring8_as<1, 2, 4, 3>(g, st);
    if (g.M <= 32) return narrow ? launch_ring8_as<2, 1, 8, 2>(g, st) : launch_ring8_as<2, 2, 4, 2>(g, st);
    if (g.M <= 64 && narrow && g.N > 2048) return launch_ring8_as<4, 1, 8, 2>(g, st);
    return takes_ring(g.M, g.N) == 2 ? launch_ring8_as<4, 2, 4, 3>(g, st) : launch_ring8_as<2, 1, 4, 3>(g, st);
}

// ---- small products in one launch -----------------------------------------------------------------------------------
// Sixteen rows by sixteen channels a workgroup, which quantises its rows itself (as quantize_rows_kernel does, to the same codes), two
// rows a wave, while the weight's rows, all units at once, travel by LDS-DMA.  N / 16 workgroups repeat that: over a short reduction it
// takes no longer than the kernel it replaces, and saves a launch and the workspace (us on the GPU, then per call from Python, two launches /
// one: 64 x 480 x 480 5.6 / 3.9, 12.2 / 7.8).  Four waves and four rows each: 5.1.
constexpr int SMALL_WAVES = 8;
template <typename T, int NP>
__global__ __launch_bounds__(64 * SMALL_WAVES) void small8_kernel(const RingArgs g, const T* __restrict__ x, int64_t ldx, int K) {
    constexpr int NW = SMALL_WAVES, EACH = 16 / NW;      // rows of a wave
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float sa[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fq = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16;
    char* const weight = lds + g.units * 2048;
    {
        const int pr = lane >> 3, pc = (lane & 7) ^ pr;
        const int8_t* const b0 = g.B + n0 * g.ldb;
        for (int u = wave; u < g.units; u += NW)
#pragma unroll
            for (int s = 0; s < 2; ++s)
                __builtin_amdgcn_global_load_lds((glb_ptr_t)(b0 + u * 128 + (uint32_t)(min((int64_t)s * 8 + pr, g.N - 1 - n0) * g.ldb) + pc * 16), (lds_ptr_t)(weight + u * 2048 + s * 1024), 16, 0, 0);
    }
    float v[EACH][NP][8];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int c = (i * 64 + lane) * 8;
        if (c < K) {
#pragma unroll
            for (int r = 0; r < EACH; ++r) load8(x + min(m0 + wave * EACH + r, g.M - 1) * ldx + c, (int64_t)K - c, v[r][i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int r = 0; r < EACH; ++r) v[r][i][j] = 0.f;
        }
    }
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
        const int row = wave * EACH + r;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, f32_bits(v[r][i][j]) & 0x7fffffffu);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        const RowScale rs = row_scale(top);
        if (lane == 0) sa[row] = rs.scale;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = (i * 64 + lane) * 8;
            if (c >= g.units * 128) continue;
            if (rs.none) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[r][i][j] = 0.f;
            }
            *(uint2*)(lds + (c >> 7) * 2048 + row * 128 + ((((c >> 4) & 7) ^ (row & 7)) * 16) + (c & 8)) = encode(v[r][i], rs.inverse);
        }
    }
    wait_vmcnt<0>();                                     // this wave's units of the weight
    __syncthreads();
    i32x4 acc = i32x4{0, 0, 0, 0};
    const int x0 = fr * 128 + (fq ^ (fr & 7)) * 16;
    for (int u = wave; u < g.units; u += NW)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const i32x4 a = *(const i32x4*)(lds + u * 2048 + (x0 ^ (h * 64))), b = *(const i32x4*)(weight + u * 2048 + (x0 ^ (h * 64)));
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, acc, 0, 0, 0);
        }
    __syncthreads();                                     // (no one reads the codes any more)
    ((i32x4*)lds)[wave * 64 + lane] = acc;
    __syncthreads();
    wave_results<1, 1, NW>(g, lds, 1024, sa, m0, n0);
}
// How many workgroups may repeat a reduction of one, two or four pieces of 512 (us on the GPU, two launches / one: 512 x 512 x 512 6.2 / 6.2,
// 3000 x 100 x 500 9.9 / 9.0 - 10.7; 64 x 2048 x 1000 6.1 / 5.8, 256 x 1024 x 1024 7.0 / 8.5; 64 x 480 x 2048 7.2 / 5.9, 128 x 1024 x 2048 7.4 /
// 8.6).
bool takes_small(int64_t M, int64_t N, int64_t K) {
    if (K > 2048) return false;
    const int64_t pieces = K <= 512 ? 1 : K <= 1024 ? 2 : 4;
    return ceil_div64(M, 16) * ceil_div64(N, 16) <= 1024 / pieces;
}
template <typename T>
int launch_small8(const RingArgs& g, const T* x, int64_t ldx, int64_t K, hipStream_t st) {
    SLIM_PROF("small8", st, (double)g.M * K * sizeof(T) + (double)g.N * g.units * 128 + (double)g.M * g.N * sizeof(T), 2.0 * g.M * g.N * K);
    auto kernel = K <= 512 ? small8_kernel<T, 1> : K <= 1024 ? small8_kernel<T, 2> : small8_kernel<T, 4>;
    const int bytes = max(g.units * 2 * 2048, SMALL_WAVES * 1024);      // codes of the rows and of the channels; the waves' sums take their place
    SLIM_HIP(slim_allow_dynamic_lds((const void*)kernel, bytes));
    kernel<<<dim3((unsigned)ceil_div64(g.N, 16), (unsigned)ceil_div64(g.M, 16)), 64 * SMALL_WAVES, bytes, st>>>(g, x, ldx, (int)K);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

// ---- one or two tokens ----------------------------------------------------------------------------------------------
// A product with one or two tokens reads the weight once and computes next to nothing, so it goes through the dot instructions and
// the loads are laid out for memory alone: a wave's load is 1024 consecutive bytes of one row (in the matrix instructions' layout, 16
// rows by 64 bytes, the same bytes take 1.5 times as long: 5120 x 13824, one token: 14.7 us against 21.4).  The workgroup quantises
// the tokens itself (NP pieces of eight channels per thread, as in quantize_rows_kernel) and keeps them in LDS, so one launch does
// it all; the tokens are requested before the weight, as loads return in order, and quantised while it travels.  A wave walks groups of
// R rows with U loads of each under way, across the groups' ends.
struct TokenArgs {
    const void* x;
    int64_t ldx;
    const int8_t* B;
    int64_t ldb;
    const float* sb;
    const void* bias;
    void* out;
    int64_t ldo;
    int dtype, N, K;
};
template <typename T, int M, int NP, int R>
__global__ __launch_bounds__(512) void token8_kernel(const TokenArgs g) {
    constexpr int U = 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int waves = blockDim.x >> 6, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row_bytes = (g.K + 127) / 128 * 128, chunks = (row_bytes + 1023) / 1024, ldl = chunks * 1024;
    uint32_t* const part = (uint32_t*)lds;               // [waves][M]
    char* const codes = lds + 64;
    float keep[M][NP][8];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = (i * (int)blockDim.x + (int)threadIdx.x) * 8;
            load8((const T*)g.x + m * g.ldx + c, (int64_t)g.K - c, keep[m][i]);
        }
    // step s of this wave: chunk s % chunks of its group s / chunks; group v holds the rows (v * all waves + this wave) * R ...
    const int all = gridDim.x * waves, me = blockIdx.x * waves + wave, groups = (g.N + R - 1) / R, mine = me < groups ? (groups - me + all - 1) / all : 0;
    const int steps = mine * chunks;
    i32x4 buf[U][R];
    int load_chunk = 0;
    int64_t load_row = (int64_t)me * R;
    auto load = [&](int i) {
        const int o = min(load_chunk * 1024 + lane * 16, row_bytes - 16);
#pragma unroll
        for (int r = 0; r < R; ++r) buf[i][r] = *(const i32x4*)(g.B + min(load_row + r, (int64_t)g.N - 1) * g.ldb + o);
        if (++load_chunk == chunks) load_chunk = 0, load_row += (int64_t)all * R;
    };
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (i < steps) load(i);
    float scale[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = f32_bits(keep[m][i][j]) & 0x7fffffffu;
                top = b > top ? b : top;
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint32_t b = (uint32_t)__shfl_xor((int)top, o, 64);
            top = b > top ? b : top;
        }
        if (lane == 0) part[wave * M + m] = top;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
        uint32_t top = 0;
        for (int i = 0; i < waves; ++i) top = max(top, part[i * M + m]);
        const RowScale s = row_scale(top);
        scale[m] = s.scale;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = (i * (int)blockDim.x + (int)threadIdx.x) * 8;
            if (c >= ldl) continue;
            if (s.none) {
#pragma unroll
                for (int j = 0; j < 8; ++j) keep[m][i][j] = 0.f;
            }
            *(uint2*)(codes + m * ldl + c) = encode(keep[m][i], s.inverse);
        }
    }
    __syncthreads();
    int acc[R][M];
    auto clear = [&]() {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int m = 0; m < M; ++m) acc[r][m] = 0;
    };
    clear();
    int chunk = 0;
    int64_t row = (int64_t)me * R;
    for (int s = 0; s < steps; s += U) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (s + i >= steps) break;
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const i32x4 x = *(const i32x4*)(codes + m * ldl + chunk * 1024 + lane * 16);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[r][m] = __builtin_amdgcn_sdot4(buf[i][r][j], x[j], acc[r][m], false);
            }
            if (s + i + U < steps) load(i);
            if (++chunk < chunks) continue;
            chunk = 0;
            int sum = 0;
            float sx = scale[0];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int m = 0; m < M; ++m) {
#pragma unroll
                    for (int o = 32; o > 0; o >>= 1) acc[r][m] += __shfl_xor(acc[r][m], o, 64);
                    if (lane == r * M + m) sum = acc[r][m], sx = scale[m];
                }
            const int m = lane % M;
            const int64_t n = row + lane / M;
            if (lane < R * M && n < g.N) {               // lane r * M + m writes row r's result for token m
                float v = ((float)sum * sx) * g.sb[n];
                if (g.bias) v += load_as_f32(g.bias, n, g.dtype);
                store_as(g.out, m * g.ldo + n, g.dtype, v);
            }
            row += (int64_t)all * R;
            clear();
        }
    }
}
template <typename T, int M, int NP>
int launch_token8(const TokenArgs& g, int waves, hipStream_t st) {
    SLIM_PROF("token8", st, (double)g.N * pad128(g.K) + (double)M * (g.N + g.K) * sizeof(T), 2.0 * M * g.N * g.K);
    const int bytes = 64 + M * (int)(ceil_div64(pad128(g.K), 1024) * 1024);
    // (two rows a wave and up to 768 workgroups, four rows and 512: 6.5 and 6.6 us at 4096 x 4096, 12.0 and 10.0 at 11008 x 4096)
    const int64_t pairs = ceil_div64(g.N, waves * 2), fours = ceil_div64(g.N, waves * 4);
    if (g.N < 8192) token8_kernel<T, M, NP, 2><<<(unsigned)(pairs < 768 ? pairs : 768), 64 * waves, bytes, st>>>(g);
    else token8_kernel<T, M, NP, 4><<<(unsigned)(fours < 512 ? fours : 512), 64 * waves, bytes, st>>>(g);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

// tokens kept in registers while they are quantised: NP pieces of eight channels per thread, 256 or 512 threads
constexpr int TOKEN_PIECES[3] = {0, 7, 4};
int token_waves(int64_t M, int64_t K) {                  // 0: not this kernel's
    if (M > 2) return 0;
    const int64_t pieces = ceil_div64(pad128(K), 1024) * 128;
    return pieces <= TOKEN_PIECES[M] * 256 ? 4 : pieces <= TOKEN_PIECES[M] * 512 ? 8 : 0;
}
template <typename T>
int token8(const TokenArgs& g, int64_t M, int waves, hipStream_t st) {
    return M == 1 ? launch_token8<T, 1, TOKEN_PIECES[1]>(g, waves, st) : launch_token8<T, 2, TOKEN_PIECES[2]>(g, waves, st);
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


}  // namespace

extern "C" int64_t slim_rows8_ld(int64_t K) { return K > 0 ? pad128(K) : 0; }

extern "C" int slim_quantize_rows8(const void* x, int dtype, int64_t R, int64_t K, int64_t ldx, int8_t* codes, int64_t ldc, float* scale,
                                   void* stream) {
    SLIM_REQUIRE(x && codes && scale && R > 0 && K > 0 && ldx >= K, "slim_quantize_rows8: bad arguments");
    SLIM_REQUIRE(known(dtype), "slim_quantize_rows8: unknown element type %d", dtype);
    SLIM_REQUIRE(R <= SLIM_INT8_MAX_DIM, "slim_quantize_rows8: too many rows");
    SLIM_REQUIRE(ldc >= pad128(K) && ldc % 16 == 0 && (uintptr_t)codes % 16 == 0,
                 "slim_quantize_rows8: rows of codes hold slim_rows8_ld(K) bytes and start at multiples of 16");
    SLIM_PROF("quantize_rows8", stream, (double)R * K * (element_size(dtype) + 1) + 4.0 * R);
    return quantize_rows_any(x, dtype, R, K, ldx, codes, ldc, scale, (hipStream_t)stream);
}

extern "C" int slim_transpose8(const int8_t* codes, int64_t N, int64_t K, int64_t ld, int8_t* codes_t, int64_t ldt, void* stream) {
    SLIM_REQUIRE(codes && codes_t && codes != codes_t && N > 0 && K > 0 && ld >= K && ldt >= pad128(N), "slim_transpose8: bad arguments");
    SLIM_REQUIRE(ceil_div64(ldt, 64) <= 65535, "slim_transpose8: too many rows");
    dim3 grid((unsigned)ceil_div64(K, 64), (unsigned)ceil_div64(ldt, 64));
    transpose8_kernel<<<grid, 256, 0, (hipStream_t)stream>>>(codes, N, K, ld, codes_t, ldt);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

extern "C" int64_t slim_gemm8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    return M > 0 && N > 0 && K > 0 && !takes_ring(M, N) ? plan_gemm8(M, N, pad128(K) / 128).slab_bytes() : 0;
}

extern "C" int slim_gemm8_nt(const int8_t* a, int64_t lda, const float* sa, const int8_t* b, int64_t ldb, const float* sb, int64_t M, int64_t N,
                             int64_t K, const void* bias, int dtype, void* out, int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
    SLIM_REQUIRE(a && sa && b && sb && out && M > 0 && N > 0 && K > 0 && ldo >= N, "slim_gemm8_nt: bad arguments");
    SLIM_REQUIRE(known(dtype), "slim_gemm8_nt: unknown element type %d", dtype);
    SLIM_REQUIRE(K <= SLIM_INT8_MAX_REDUCTION && M <= SLIM_INT8_MAX_DIM && N <= SLIM_INT8_MAX_DIM, "slim_gemm8_nt: too large");
    SLIM_REQUIRE(lda >= pad128(K) && ldb >= pad128(K) && lda % 16 == 0 && ldb % 16 == 0 && (uintptr_t)a % 16 == 0 && (uintptr_t)b % 16 == 0,
                 "slim_gemm8_nt: rows of codes hold slim_rows8_ld(K) bytes and start at multiples of 16");
    SLIM_REQUIRE(workspace_bytes >= slim_gemm8_workspace_bytes(M, N, K) && (workspace || workspace_bytes == 0) && (uintptr_t)workspace % 16 == 0,
                 "slim_gemm8_nt: workspace too small or misaligned");
    SLIM_REQUIRE(lda < 1 << 23 && ldb < 1 << 23, "slim_gemm8_nt: rows of codes lie too far apart");
    if (takes_ring(M, N)) return launch_ring8(RingArgs{a, lda, sa, b, ldb, sb, bias, out, ldo, dtype, M, N, (int)(pad128(K) / 128)}, (hipStream_t)stream);
    Gemm8Args g{a, b, lda, ldb, M, N, (int)(pad128(K) / 128), sa, sb, bias, out, ldo, dtype, 0, 0, 1, 0, nullptr, 0};
    return gemm8(g, workspace, (hipStream_t)stream);
}

extern "C" int64_t slim_linear8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || token_waves(M, K) || takes_small(M, N, K)) return 0;
    return align256(M * pad128(K)) + align256(M * 4) + slim_gemm8_workspace_bytes(M, N, K);
}

extern "C" int slim_linear8_forward(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, const int8_t* codes, const float* scale, int64_t N,
                                    const void* bias, void* y, int64_t ldy, void* workspace, int64_t workspace_bytes, void* stream) {
    SLIM_REQUIRE(x && codes && scale && y && M > 0 && N > 0 && K > 0 && ldx >= K && ldy >= N, "slim_linear8_forward: bad arguments");
    const int64_t need = slim_linear8_workspace_bytes(M, N, K);
    SLIM_REQUIRE(workspace_bytes >= need && (workspace || !need) && (uintptr_t)workspace % 16 == 0, "slim_linear8_forward: workspace too small or misaligned");
    if (const int waves = token_waves(M, K)) {
        SLIM_REQUIRE(known(dtype), "slim_linear8_forward: unknown element type %d", dtype);
        SLIM_REQUIRE(N <= SLIM_INT8_MAX_DIM && (uintptr_t)codes % 16 == 0, "slim_linear8_forward: weight too large or misaligned");
        const TokenArgs g{x, ldx, codes, pad128(K), scale, bias, y, ldy, dtype, (int)N, (int)K};
        if (dtype == SLIM_DTYPE_F32) return token8<float>(g, M, waves, (hipStream_t)stream);
        if (dtype == SLIM_DTYPE_BF16) return token8<bf16_t>(g, M, waves, (hipStream_t)stream);
        return token8<_Float16>(g, M, waves, (hipStream_t)stream);
    }
    if (takes_small(M, N, K)) {
        SLIM_REQUIRE(known(dtype), "slim_linear8_forward: unknown element type %d", dtype);
        SLIM_REQUIRE(N <= SLIM_INT8_MAX_DIM && (uintptr_t)codes % 16 == 0, "slim_linear8_forward: weight too large or misaligned");
        const RingArgs g{nullptr, 0, nullptr, codes, pad128(K), scale, bias, y, ldy, dtype, M, N, (int)(pad128(K) / 128)};
        if (dtype == SLIM_DTYPE_F32) return launch_small8<float>(g, (const float*)x, ldx, K, (hipStream_t)stream);
        if (dtype == SLIM_DTYPE_BF16) return launch_small8<bf16_t>(g, (const bf16_t*)x, ldx, K, (hipStream_t)stream);
        return launch_small8<_Float16>(g, (const _Float16*)x, ldx, K, (hipStream_t)stream);
    }
    int8_t* xc = (int8_t*)workspace;
    float* sx = (float*)(xc + align256(M * pad128(K)));
    const int rc = slim_quantize_rows8(x, dtype, M, K, ldx, xc, pad128(K), sx, stream);
    if (rc) return rc;
    char* slab = (char*)sx + align256(M * 4);
    return slim_gemm8_nt(xc, pad128(K), sx, codes, pad128(K), scale, M, N, K, bias, dtype, y, ldy, slab, (char*)workspace + workspace_bytes - slab, stream);
}
