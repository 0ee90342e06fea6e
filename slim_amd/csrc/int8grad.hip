// The straight-through gradient of a linear in 8-bit integers with respect to its input: dx[m][k] = sum_n v[m][n] codes[n][k] with
// v = dy * scale (the reference: slim/quantization/quantization.py:322-328).
//
// v is a float of its own for every element, and stays one: it is written as a sum of half-precision numbers, v = 2^-k (p0 + p1 2^-11
// [+ p2 2^-22]), each the rounding of what the ones before leave, and multiplied by the codes, which half precision holds exactly, on
// the half-precision matrix instructions; products of 11 by 8 bits are exact, sums are fp32.  2^k brings the row's largest element to
// 2^14, so two planes keep every element to 2^-23 of itself, but no closer than 2^-50 of the row's largest; a third plane (fp32) keeps
// all 24 bits, or 2^-61.  (Two planes of whole numbers against the row's largest element, on the int8 instructions, took half the time,
// 149 us for 2048 x 4096 x 11008, and lost what is small beside one large element: with one element 1e5 times the others, 80 % of
// dx where its code is 0.  One plane of bf16 would take half the time too, for 2^-9 of every element, as much as the result's own rounding.)
//
// Every element of dx is one chain of sums over n in steps of 32, whichever kernel computes it: a row's gradient does not depend on
// the rows beside it.
#include "int8.hpp"

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
constexpr int STEP = 64;                                 // codes of a step of the reduction; a row of a plane takes 128 bytes of it

constexpr int planes_of(int dtype) { return dtype == SLIM_DTYPE_F32 ? 3 : 2; }

// ---- rows -> planes -------------------------------------------------------------------------------------------------
struct RowPower {
    float power, back;                                   // 2^k and 2^-k; back: NaN where the row is not finite
    bool none;
};
__device__ __forceinline__ RowPower row_power(uint32_t max_bits) {
    const bool bad = max_bits >= 0x7f800000u, none = bad || max_bits == 0;
    const int k = min(14 - ((int)(max_bits >> 23) - 127), 126);          // -113 ... 126
    return {__uint_as_float((uint32_t)(127 + k) << 23), bad ? __uint_as_float(0x7fc00000u) : none ? 0.f : __uint_as_float((uint32_t)(127 - k) << 23), none};
}
template <int PLANES>
__device__ __forceinline__ void split(const float v[8], float power, f16x8 (&out)[PLANES]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float t = v[j] * power;
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
            const _Float16 h = (_Float16)t;
            out[p][j] = h;
            t = (t - (float)h) * 2048.f;                 // (exact: what eleven of 24 bits leave)
        }
    }
}
template <int PLANES>
__device__ __forceinline__ float join(const float* sums, int stride) {
    float v = sums[0] + sums[stride] * 0x1p-11f;
    if (PLANES == 3) v += sums[2 * stride] * 0x1p-22f;
    return v;
}

// dy * scale of a row as planes, zeros up to the padded length.  Rows of a plane are stored sixteen rows of the first plane, then the same
// sixteen of the next, so that a wave's fragments of a product hold all planes of its rows.  WPR waves work on a row (one: four
// rows per workgroup); each thread keeps NV pieces of eight elements, so the row is read once (NV = 0: twice, for rows too long for that).
template <typename T, int PLANES, int NV, int WPR>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void split_rows_kernel(const T* __restrict__ dy, int64_t R, int64_t N, int64_t lddy, const float* __restrict__ scale,
                                                                            _Float16* __restrict__ planes, int64_t ld, float* __restrict__ back) {
    constexpr int TPR = 64 * WPR;
    __shared__ uint32_t part[WPR];
    const int wave = threadIdx.x >> 6;
    const int64_t row = WPR > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (WPR == 1 && row >= R) return;
    const int t = WPR > 1 ? threadIdx.x : threadIdx.x & 63;
    const T* src = dy + row * lddy;
    float keep[NV > 0 ? NV : 1][8];
    uint32_t m = 0;
    auto fetch = [&](int64_t c, float v[8]) {
        float f[8];
        load8<(NV > 0)>(src + c, N - c, v);
        load8(scale + c, N - c, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= f[j];
    };
    auto take = [&](const float v[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, f32_bits(v[j]) & 0x7fffffffu);
    };
    if (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = ((int64_t)i * TPR + t) * 8;
            if (c < N) {
                fetch(c, keep[i]);
                take(keep[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) keep[i][j] = 0.f;
            }
        }
    } else {
        for (int64_t c = (int64_t)t * 8; c < N; c += TPR * 8) {
            float v[8];
            fetch(c, v);
            take(v);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
    if (WPR > 1) {
        if ((threadIdx.x & 63) == 0) part[wave] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WPR; ++i) m = max(m, part[i]);
    }
    const RowPower rp = row_power(m);
    if (t == 0) back[row] = rp.back;
    const int64_t end = (N + 127) / 128 * 128;
    auto put = [&](int64_t c, float v[8]) {
        if (rp.none) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        }
        f16x8 out[PLANES];
        split<PLANES>(v, rp.power, out);
#pragma unroll
        for (int p = 0; p < PLANES; ++p) *(f16x8*)(planes + (((row >> 4) * PLANES + p) * 16 + (row & 15)) * ld + c) = out[p];
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
            if (c < N) fetch(c, v);
            put(c, v);
        }
    }
}

template <typename T, int PLANES>
int split_rows(const T* dy, int64_t R, int64_t N, int64_t lddy, const float* scale, _Float16* planes, int64_t ld, float* back, hipStream_t st) {
    const int64_t pieces = ld / 8;
#define SLIM_ROWS(NV, WPR)                                                                                                                              \
    do {                                                                                                                                                \
        SLIM_REQUIRE(R * 64 * WPR < ((int64_t)1 << 32) - 1024, "slim_linear8_backward: too many rows for one launch");                                  \
        split_rows_kernel<T, PLANES, NV, WPR><<<(unsigned)(WPR > 1 ? R : ceil_div64(R, 4)), WPR == 16 ? 1024 : 256, 0, st>>>(dy, R, N, lddy, scale, planes, ld, back); \
    } while (0)
    if (pieces <= 64) SLIM_ROWS(1, 1);
    else if (pieces <= 128) SLIM_ROWS(2, 1);
    else if (pieces <= 512) SLIM_ROWS(2, 4);
    else if (pieces <= 1024) SLIM_ROWS(4, 4);
    else if (pieces <= 2048) SLIM_ROWS(8, 4);
    else SLIM_ROWS(0, 16);
#undef SLIM_ROWS
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

// ---- codes -> operands ----------------------------------------------------------------------------------------------
// Eight codes of eight bits as half-precision numbers: 1024 + (code + 128), whose low mantissa bits are the byte itself, less 1152.
__device__ __forceinline__ f16x8 halves(int lo, int hi) {
    const f16x2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    f16x8 out;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const uint32_t u = (uint32_t)(w ? hi : lo) ^ 0x80808080u;
        const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
        const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
        out[4 * w] = a[0], out[4 * w + 1] = a[1], out[4 * w + 2] = b[0], out[4 * w + 3] = b[1];
    }
    return out;
}
// half h of a lane's sixteen codes
__device__ __forceinline__ f16x8 halves(const i32x4& raw, int h) { return halves(raw[2 * h], raw[2 * h + 1]); }

// ---- planes x codes -------------------------------------------------------------------------------------------------
struct GradArgs {
    const _Float16* A;                                   // planes of the rows
    int64_t lda, rows;                                   // halves from row to row, rows of planes
    const float* back;                                   // [M]
    const int8_t* B;                                     // codes [K, ldb]
    int64_t ldb, M, K;
    void* out;
    int64_t ldo;
    int dtype, steps;                                    // steps of 64
    int tiles_m, tiles_n;
};

template <int PLANES, int FM, int FN>
__device__ __forceinline__ void write_gradient(const GradArgs& g, const f32x4 (&acc)[FM][FN], const float (&back)[FM / PLANES], int64_t group0, int64_t n0, int fr, int fq) {
    auto rows = [&](auto* out, auto convert) {
#pragma unroll
        for (int i = 0; i < FM / PLANES; ++i) {
            const int64_t m = (group0 + i) * 16 + fr;
            if (m >= g.M) continue;
            auto value = [&](int c) {
                float sums[PLANES];
#pragma unroll
                for (int p = 0; p < PLANES; ++p) sums[p] = acc[i * PLANES + p][c >> 2][c & 3];
                return convert(join<PLANES>(sums, 1) * back[i]);
            };
            Columns<FN>::each(n0, fq, [&](auto count, int c, int64_t n) { store_run<count.value>(out + m * g.ldo + n, g.K - n, [&](int k) { return value(c + k); }); });
        }
    };
    if (g.dtype == SLIM_DTYPE_F32) rows((float*)g.out, [](float v) { return v; });
    else if (g.dtype == SLIM_DTYPE_BF16) rows((bf16_t*)g.out, [](float v) { return f32_to_bf16(v); });
    else rows((_Float16*)g.out, [](float v) { return (_Float16)v; });
}

// D = A B^T on 16 x 16 x 32 half-precision instructions, operands delivered by LDS-DMA (16 bytes per lane) STAGES steps ahead.  LDS image of a
// stage: BM rows of planes, 128 bytes each, then BN rows of codes, 64 bytes each; the 16-byte piece c of a row is stored at c ^ key(row),
// applied on the source side: the row's low three bits for the planes; for the codes, two rows of which share the 128 bytes of all
// banks, the two bits that differ between the rows of either parity that a group of eight lanes reads.
// A lane's sixteen codes of a step are the two halves of one 16-byte piece; the planes' pieces are read in the same order (any
// order of a step's elements will do, so long as it is the same for both operands and for all kernels of the gradient).
// The result is computed transposed (codes first), rows of codes dealt to the fragments in runs of four, as in gemm8_tile: a lane holds
// consecutive columns of one row.
// While a step's first half is multiplied its second half is read and converted, and while that is multiplied the next step's first
// half is read and the stage just emptied is requested again; one barrier per step.  Paced by scheduling barriers, as gemm8_tile is: left to
// the compiler, the reads come late and in bursts (2048 x 4096 x 11008 bf16: 310 us a call against 292).
// What bounds it: the matrix instructions.  2048 x 4096 x 11008 bf16 292 us with the split (1.27e15 operations/s over both planes; a large bf16
// library product reaches 1.41e15), fp32 465 (1.19e15 over three).  Few rows: the chain of sums itself, about 0.1 us a step of 64 (16 x 4096 x
// 4096 bf16 16.5 us; several waves that share a reduction took 9 and gave other sums for other numbers of rows).
template <int PLANES, int FM, int FN, int WM, int WN, int STAGES, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void grad8_kernel(const GradArgs g) {
    constexpr int BM = 16 * FM * WM, BN = 16 * FN * WN, NW = WM * WN;
    constexpr int PIECES = BM / 8 + BN / 16, PPW = (PIECES + NW - 1) / NW;     // (a last wave repeats the final piece)
    constexpr int STAGE_BYTES = BM * 128 + BN * 64, PAIRS = FN / 2 * 32;
    static_assert(FM % PLANES == 0, "a wave holds whole groups of planes");
    constexpr int PRODUCTS = FM * FN, PACE1 = FN, PACE2 = PRODUCTS / (FM + FN + PPW + FM) > 0 ? PRODUCTS / (FM + FN + PPW + FM) : 1, VALU1 = FN * 10 / FM + 1;
    static_assert((STAGES - 1) * PPW < 64, "requests under way are counted in six bits");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int tm, tn, slice;
    tile_of(blockIdx.x, g.tiles_m, g.tiles_n, 1, tm, tn, slice);
    const int64_t row0 = (int64_t)tm * BM, col0 = (int64_t)tn * BN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WN, wc = wave % WN, fr = lane & 15, fq = lane >> 4;

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // this lane's sources: a piece of 1024 bytes is eight rows of planes or sixteen of codes; rows behind the last are read from the last one
    const char* base[PPW];
    uint32_t off[PPW];
#pragma unroll
    for (int s = 0; s < PPW; ++s) {
        const int q = min(s * NW + wave, PIECES - 1);
        if (q * 8 < BM) {
            const int R = q * 8 + (lane >> 3);
            base[s] = (const char*)(g.A + row0 * g.lda);
            off[s] = (uint32_t)(min((int64_t)R, g.rows - 1 - row0) * g.lda * 2) + ((lane & 7) ^ (R & 7)) * 16;
        } else {
            const int R = (q - BM / 8) * 16 + (lane >> 2), w = R % (16 * FN), key = w < PAIRS ? ((w >> 1) & 1) | (((w >> 3) & 1) << 1) : (w >> 1) & 3;
            base[s] = (const char*)(g.B + col0 * g.ldb);
            off[s] = (uint32_t)(min((int64_t)R, g.K - 1 - col0) * g.ldb) + ((lane & 3) ^ key) * 16;
        }
    }
    const int steps = g.steps;
    auto request = [&](int kt, int stage) {              // (behind the last step: the last one again, which nothing reads)
        const int64_t k = (int64_t)min(kt, steps - 1) * 64;
#pragma unroll
        for (int s = 0; s < PPW; ++s) {
            const int q = min(s * NW + wave, PIECES - 1);
            __builtin_amdgcn_global_load_lds((glb_ptr_t)(base[s] + (q * 8 < BM ? 2 * k : k) + off[s]), (lds_ptr_t)(lds + stage * STAGE_BYTES + q * 1024), 16, 0, 0);
        }
    };
#pragma unroll
    for (int st = 0; st < STAGES; ++st) request(st, st);
    const int a_off = (wr * 16 * FM + fr) * 128 + ((2 * fq) ^ (fr & 7)) * 16;
    const int b_piece = (fq ^ ((fr >> 1) & 3)) * 16;
    const int b_off = BM * 128 + (wc * 16 * FN + (fr >> 2) * 8 + (fr & 3)) * 64 + b_piece;
    const int odd_off = BM * 128 + (wc * 16 * FN + PAIRS + fr) * 64 + b_piece;
    f16x8 af[2][FM], bf[2][FN];
    i32x4 raw[FN];
    auto read = [&](int half, int stage) {
        const char* a = lds + ((stage * STAGE_BYTES + a_off) ^ (half * 16));
#pragma unroll
        for (int i = 0; i < FM; ++i) af[half][i] = *(const f16x8*)(a + i * 16 * 128);
    };
    auto read_codes = [&](int stage) {
#pragma unroll
        for (int j = 0; j < FN / 2 * 2; ++j) raw[j] = *(const i32x4*)(lds + stage * STAGE_BYTES + b_off + ((j >> 1) * 32 + (j & 1) * 4) * 64);
        if (FN % 2) raw[FN - 1] = *(const i32x4*)(lds + stage * STAGE_BYTES + odd_off);
    };
    auto convert = [&](int half) {
#pragma unroll
        for (int j = 0; j < FN; ++j) bf[half][j] = halves(raw[j], half);
    };
    auto multiply = [&](int half) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[half][j], af[half][i], acc[i][j], 0, 0, 0);
    };
    wait_vmcnt<(STAGES - 1) * PPW>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read_codes(0);
    read(0, 0);
    convert(0);
    int stage = 0;
    for (int kt = 0; kt < steps; ++kt) {
        const int next = stage + 1 == STAGES ? 0 : stage + 1;
        __builtin_amdgcn_sched_barrier(0);
        read(1, stage);
        convert(1);
        multiply(0);
#pragma unroll
        for (int s = 0; s < FM; ++s) {
            __builtin_amdgcn_sched_group_barrier(0x008, PACE1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, VALU1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        // this wave's reads of the stage are done and its requests of the next one have landed; behind the barrier so are everyone's
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_vmcnt<(STAGES - 2) * PPW>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        read_codes(next);
        read(0, next);
        request(kt + STAGES, stage);
        multiply(1);
        convert(0);
#pragma unroll
        for (int s = 0; s < FN + FM; ++s) {
            __builtin_amdgcn_sched_group_barrier(0x008, PACE2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
#pragma unroll
        for (int s = 0; s < PPW; ++s) {
            __builtin_amdgcn_sched_group_barrier(0x008, PACE2, 0);
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        }
#pragma unroll
        for (int s = 0; s < FM; ++s) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, VALU1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        stage = next;
    }
    wait_vmcnt<0>();                                     // (the requests behind the last step land before the LDS is given up)

    const int64_t group0 = (row0 / 16 + wr * FM) / PLANES;
    float back[FM / PLANES];
#pragma unroll
    for (int i = 0; i < FM / PLANES; ++i) back[i] = g.back[min((group0 + i) * 16 + fr, g.M - 1)];
    write_gradient<PLANES, FM, FN>(g, acc, back, group0, col0 + wc * 16 * FN, fr, fq);
}

template <int PLANES, int FM, int FN, int WM, int WN, int STAGES, int OCC>
int launch_grad8(GradArgs g, hipStream_t st) {
    constexpr int BM = 16 * FM * WM, BN = 16 * FN * WN, bytes = STAGES * (BM * 128 + BN * 64);
    const int64_t tiles_m = ceil_div64(g.rows, BM), tiles_n = ceil_div64(g.K, BN), blocks = tiles_m * tiles_n;
    SLIM_REQUIRE(blocks * 64 * WM * WN < (int64_t)1 << 32 && blocks < 0x7fffffff, "slim_linear8_backward: the result is too large for one launch");
    g.tiles_m = (int)tiles_m, g.tiles_n = (int)tiles_n;
    auto kernel = grad8_kernel<PLANES, FM, FN, WM, WN, STAGES, OCC>;
    SLIM_HIP(slim_allow_dynamic_lds((const void*)kernel, bytes));
    kernel<<<(unsigned)blocks, 64 * WM * WN, bytes, st>>>(g);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}
// The largest tile that gives enough workgroups (us on the largest, middle and smallest one: 768 x 4096 x 4096 fp32, 192 of the largest, 78, 94
// and 137; 1024 x 4096 x 4096 bf16, 128 of them, 91, 87 and 142; 300 x 4096 x 4096 bf16, 160 of the middle one, 83, 41 and 51; 128 x 4096 x 4096
// fp32, 128 of it, 70, 37 and 30, 256 x 4096 x 4096 bf16, also 128, 83, 40 and 41).
template <int PLANES>
int grad8(const GradArgs& g, hipStream_t st) {
    SLIM_PROF("grad8", st, (double)g.rows * g.steps * 128 + (double)g.K * g.steps * 64 + (double)g.M * g.K * element_size(g.dtype), 2.0 * g.rows * g.K * g.steps * 64);
    constexpr int LARGE = PLANES == 3 ? 6 : 8, SMALL = PLANES == 3 ? 3 : 4;
    if (ceil_div64(g.rows, 32 * LARGE) * ceil_div64(g.K, 256) >= 192) return launch_grad8<PLANES, LARGE, 4, 2, 4, 3, 2>(g, st);
    if (ceil_div64(g.rows, 32 * SMALL) * ceil_div64(g.K, 128) > 128) return launch_grad8<PLANES, SMALL, 2, 2, 4, 4, 2>(g, st);
    return launch_grad8<PLANES, PLANES, 1, 1, 4, 8, 1>(g, st);
}

// ---- small gradients in one launch ----------------------------------------------------------------------------------
// Sixteen rows by 128 columns a workgroup, sixteen of them a wave: it splits its rows itself (as split_rows_kernel does, to the same planes), two
// rows a wave, while each wave's codes, the whole reduction at once, travel into its registers.  One launch, no workspace (64 x 480 x 480 bf16
// 4.9 us, 77 x 1000 x 776 fp32 9.3: launch, the rows' trip, the split, the chain of sums).
template <typename T, int PLANES, int NP>
__global__ __launch_bounds__(512) void small_grad8_kernel(const GradArgs g, const T* __restrict__ dy, int64_t lddy, int N, const float* __restrict__ scale) {
    constexpr int UNITS = NP * 8;                        // steps of 64: always as many, with planes of zeros behind the last (a loop without branches)
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float back[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fq = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 128 + wave * 16, m0 = (int64_t)blockIdx.y * 16;
    float v[2][NP][8], f[NP][8];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int c = (i * 64 + lane) * 8;
        if (c < N) {
            load8(scale + c, (int64_t)N - c, f[i]);
#pragma unroll
            for (int r = 0; r < 2; ++r) load8(dy + min(m0 + wave * 2 + r, g.M - 1) * lddy + c, (int64_t)N - c, v[r][i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[i][j] = v[0][i][j] = v[1][i][j] = 0.f;
        }
    }
    i32x4 raw[UNITS];
    const int8_t* const b = g.B + min(n0 + fr, g.K - 1) * g.ldb + fq * 16;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) raw[u] = *(const i32x4*)(b + min(u, g.steps - 1) * 64);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = wave * 2 + r;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[r][i][j] *= f[i][j];
                top = max(top, f32_bits(v[r][i][j]) & 0x7fffffffu);
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        const RowPower rp = row_power(top);
        if (lane == 0) back[row] = rp.back;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = (i * 64 + lane) * 8;
            if (rp.none) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[r][i][j] = 0.f;
            }
            f16x8 out[PLANES];
            split<PLANES>(v[r][i], rp.power, out);
            char* const dst = lds + (c >> 6) * PLANES * 2048 + row * 128 + ((((c >> 3) & 7) ^ (row & 7)) * 16);
#pragma unroll
            for (int p = 0; p < PLANES; ++p) *(f16x8*)(dst + p * 2048) = out[p];
        }
    }
    __syncthreads();
    if (n0 >= g.K) return;
    f32x4 acc[PLANES][1];
#pragma unroll
    for (int p = 0; p < PLANES; ++p) acc[p][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    const char* const a = lds + fr * 128;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f16x8 codes = halves(raw[u], h);
#pragma unroll
            for (int p = 0; p < PLANES; ++p)
                acc[p][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, *(const f16x8*)(a + (u * PLANES + p) * 2048 + (((2 * fq + h) ^ (fr & 7)) * 16)), acc[p][0], 0, 0, 0);
        }
    const float mine[1] = {back[fr]};
    write_gradient<PLANES, PLANES, 1>(g, acc, mine, m0 / 16, n0, fr, fq);
}
// Up to two rounds of workgroups may repeat the split of a reduction up to 1024 (us, two launches on the best tile / one: bf16 64 x 480 x 480
// 6.7 / 4.9, 1024 x 512 x 512 8.9 / 5.3, 2048 x 512 x 512 13.3 / 8.2, 1024 x 1000 x 1024 17.3 / 16.3).
bool takes_small(int64_t M, int64_t N, int64_t K) { return N <= 1024 && ceil_div64(M, 16) * ceil_div64(K, 128) <= 512; }
template <typename T, int PLANES>
int launch_small_grad8(const GradArgs& g, const T* dy, int64_t lddy, int64_t N, const float* scale, hipStream_t st) {
    SLIM_PROF("small_grad8", st, (double)g.M * N * sizeof(T) + (double)g.K * g.steps * 64 + (double)g.M * g.K * sizeof(T), 2.0 * PLANES * g.M * g.K * N);
    auto kernel = N <= 512 ? small_grad8_kernel<T, PLANES, 1> : small_grad8_kernel<T, PLANES, 2>;
    const int bytes = (N <= 512 ? 8 : 16) * PLANES * 2048;
    SLIM_HIP(slim_allow_dynamic_lds((const void*)kernel, bytes));
    kernel<<<dim3((unsigned)ceil_div64(g.K, 128), (unsigned)ceil_div64(g.M, 16)), 512, bytes, st>>>(g, dy, lddy, (int)N, scale);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

// rows of planes of M rows
int64_t plane_rows(int64_t M, int dtype) { return (M + 15) / 16 * 16 * planes_of(dtype); }

}  // namespace

extern "C" int64_t slim_linear8_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype) {
    if (M <= 0 || N <= 0 || K <= 0 || !known(dtype) || takes_small(M, N, K)) return 0;
    return align256(plane_rows(M, dtype) * pad128(N) * 2) + align256(M * 4);
}

extern "C" int slim_linear8_backward(const void* dy, int dtype, int64_t lddy, int64_t M, int64_t N, const int8_t* codes_t, const float* scale, int64_t K,
                                     void* dx, int64_t lddx, void* workspace, int64_t workspace_bytes, void* stream) {
    SLIM_REQUIRE(dy && codes_t && scale && dx && M > 0 && N > 0 && K > 0 && lddy >= N && lddx >= K, "slim_linear8_backward: bad arguments");
    SLIM_REQUIRE(known(dtype), "slim_linear8_backward: unknown element type %d", dtype);
    SLIM_REQUIRE(N <= SLIM_INT8_MAX_REDUCTION && M <= SLIM_INT8_MAX_DIM && K <= SLIM_INT8_MAX_DIM, "slim_linear8_backward: too large");
    const int64_t need = slim_linear8_backward_workspace_bytes(M, N, K, dtype), ld = pad128(N);
    SLIM_REQUIRE(workspace_bytes >= need && (workspace || !need) && (uintptr_t)workspace % 16 == 0,
                 "slim_linear8_backward: workspace too small or misaligned");
    SLIM_REQUIRE((uintptr_t)codes_t % 16 == 0, "slim_linear8_backward: codes must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    GradArgs g{nullptr, ld, plane_rows(M, dtype), nullptr, codes_t, ld, M, K, dx, lddx, dtype, (int)(ld / STEP), 0, 0};
    if (!need) {
        if (dtype == SLIM_DTYPE_F32) return launch_small_grad8<float, 3>(g, (const float*)dy, lddy, N, scale, st);
        if (dtype == SLIM_DTYPE_BF16) return launch_small_grad8<bf16_t, 2>(g, (const bf16_t*)dy, lddy, N, scale, st);
        return launch_small_grad8<_Float16, 2>(g, (const _Float16*)dy, lddy, N, scale, st);
    }
    _Float16* planes = (_Float16*)workspace;
    float* back = (float*)((char*)workspace + align256(g.rows * ld * 2));
    g.A = planes, g.back = back;
    {
        SLIM_PROF("split_rows", st, (double)M * N * element_size(dtype) + 4.0 * N + 2.0 * g.rows * ld);
        const int rc = dtype == SLIM_DTYPE_F32    ? split_rows<float, 3>((const float*)dy, M, N, lddy, scale, planes, ld, back, st)
                       : dtype == SLIM_DTYPE_BF16 ? split_rows<bf16_t, 2>((const bf16_t*)dy, M, N, lddy, scale, planes, ld, back, st)
                                                  : split_rows<_Float16, 2>((const _Float16*)dy, M, N, lddy, scale, planes, ld, back, st);
        if (rc) return rc;
    }
    return dtype == SLIM_DTYPE_F32 ? grad8<3>(g, st) : grad8<2>(g, st);
}
