// AdamW over many tensors in one launch, after the global norm of their gradients (fine-tuning; the reference leaves both to the
// Trainer's optimizer, slim/fine_tune.py:197-219).  Moments in fp32, or in 8 bits with one pair of scales per 512 elements.
#include "common.hpp"
#include "../../include/slim_hip.h"
#include <cmath>

namespace {

constexpr int BLOCK = 512;       // elements that share a pair of scales: eight per lane, one wave
constexpr int CHUNK = 4 * BLOCK; // elements of a workgroup of the update: one block per wave
constexpr int NORM_CHUNK = 8192; // elements of a workgroup's step of the norm

// one launch takes this many tensors: their addresses travel as kernel arguments (4 KB), which a captured graph keeps by
// value and which needs no staging buffer
constexpr int NORM_TENSORS = 160;
constexpr int STEP_TENSORS = 60;

// a grid holds fewer than 2^32 threads; a tensor takes at most half of one.  The norm's grid is NORM_BLOCKS whatever its tensors hold, so
// a launch always takes NORM_TENSORS of them: its workspace, a partial sum per workgroup, is a function of their number alone.
constexpr int64_t MAX_CHUNKS = (1 << 24) - 1, MAX_NUMEL = (int64_t)CHUNK << 23;
static_assert(NORM_TENSORS * (MAX_NUMEL / NORM_CHUNK) < (int64_t)1 << 31, "the norm's chunks are counted in 32 bits");

typedef __attribute__((ext_vector_type(2))) float f32x2;

struct NormArgs {
    const void* g[NORM_TENSORS];
    int64_t n[NORM_TENSORS];
    uint32_t first[NORM_TENSORS + 1];        // first chunk of each tensor; [count]: all chunks
    int count;
};

struct StepArgs {
    void* p[STEP_TENSORS];
    const void* g[STEP_TENSORS];
    void* m[STEP_TENSORS];
    void* v[STEP_TENSORS];
    float* s[STEP_TENSORS];                  // [blocks][2], 8-bit moments only
    float* w[STEP_TENSORS];                  // fp32 master copies, or null
    int64_t n[STEP_TENSORS];
    uint32_t first[STEP_TENSORS + 1];
    int count;
    int index0;                              // ordinal of the launch's first tensor
    const float* norm;                       // gradient norm, or null
    double max_norm;
    float b1, c1, b2, c2;                    // beta, 1 - beta
    float keep, rate, root, eps;             // 1 - lr * decay; lr / (1 - beta1^t); 1 / sqrt(1 - beta2^t)
    uint32_t seed;
};
static_assert(sizeof(NormArgs) <= 4096 && sizeof(StepArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ void from_f32(float f, float& o) { o = f; }
__device__ __forceinline__ void from_f32(float f, bf16_t& o) { o = f32_to_bf16(f); }
__device__ __forceinline__ void from_f32(float f, _Float16& o) { o = (_Float16)f; }

// COUNT consecutive elements from any element-aligned address
template <typename T, int COUNT>
struct Packed {
    typedef T vec __attribute__((ext_vector_type(COUNT)));
};
// Every byte is used once and the arrays are larger than the caches: loads and stores that do not stay there (the sum of
// squares of 512 MB takes 80 us with them and 132 without, which leave dirty lines of earlier kernels to be written back first; the
// update of 14 adapters of a 4096-wide block with its norm 167 against 191).
template <int COUNT, typename T>
__device__ __forceinline__ typename Packed<T, COUNT>::vec stream_load(const T* p) {
    typedef typename Packed<T, COUNT>::vec vec;
    typedef vec unaligned __attribute__((aligned(sizeof(T))));
    return __builtin_nontemporal_load((const unaligned*)p);
}
template <int COUNT, typename T>
__device__ __forceinline__ void stream_store(T* p, typename Packed<T, COUNT>::vec v) {
    typedef typename Packed<T, COUNT>::vec vec;
    typedef vec unaligned __attribute__((aligned(sizeof(T))));
    __builtin_nontemporal_store(v, (unaligned*)p);
}
template <int COUNT, typename T>
__device__ __forceinline__ void load_run(const T* p, int64_t valid, float out[COUNT]) {
    if (valid >= COUNT) {
        const typename Packed<T, COUNT>::vec v = stream_load<COUNT>(p);
#pragma unroll
        for (int j = 0; j < COUNT; ++j) out[j] = to_f32((T)v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < COUNT; ++j) out[j] = j < valid ? to_f32(p[j]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, int64_t valid, float out[4]) { load_run<4>(p, valid, out); }
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t valid, const float in[4]) {
    T o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) from_f32(in[j], o[j]);
    if (valid >= 4) {
        typename Packed<T, 4>::vec v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = o[j];
        stream_store<4>(p, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < valid) p[j] = o[j];
    }
}
__device__ __forceinline__ uint32_t load4_codes(const uint8_t* p, int64_t valid) {
    typedef uint32_t word __attribute__((aligned(1)));
    if (valid >= 4) return __builtin_nontemporal_load((const word*)p);
    uint32_t v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) v |= (j < valid ? (uint32_t)p[j] : 0u) << (8 * j);
    return v;
}
__device__ __forceinline__ void store4_codes(uint8_t* p, int64_t valid, uint32_t c) {
    typedef uint32_t word __attribute__((aligned(1)));
    if (valid >= 4) {
        __builtin_nontemporal_store(c, (word*)p);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < valid) p[j] = (uint8_t)(c >> (8 * j));
}

// the tensor that chunk c belongs to
__device__ __forceinline__ int tensor_of(const uint32_t* first, int count, uint32_t c) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ---- sqrt(sum of squares) -------------------------------------------------------------------------------------------
// Squares and sums in 64 bits: the sum runs over up to 10^10 elements, and the update's clipping factor, which it decides, should
// not depend on how the elements were dealt out.  Partial sums are added in a fixed order.
// A workgroup takes NORM_CHUNK elements at a time, sixteen bytes per load and four loads per thread under way.
template <typename T>
__global__ __launch_bounds__(256) void sumsq_kernel(const NormArgs a, double* __restrict__ part) {
    constexpr int V = 16 / sizeof(T), U = NORM_CHUNK / (256 * V);
    __shared__ double ws[4];
    double sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sum[u] = 0.0;
    for (uint32_t c = blockIdx.x; c < a.first[a.count]; c += gridDim.x) {
        const int t = tensor_of(a.first, a.count, c);
        const int64_t base = (int64_t)(c - a.first[t]) * NORM_CHUNK, n = a.n[t];
        const T* g = (const T*)a.g[t];
        if (n - base >= NORM_CHUNK) {
            typename Packed<T, V>::vec v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = stream_load<V>(g + base + (u * 256 + threadIdx.x) * V);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const double x = (double)to_f32((T)v[u][j]);
                    sum[u] = __builtin_fma(x, x, sum[u]);
                }
        } else {
            for (int64_t i = base + threadIdx.x; i < n; i += 256) {
                const double x = (double)to_f32(g[i]);
                sum[0] = __builtin_fma(x, x, sum[0]);
            }
        }
    }
    double all = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u) all += sum[u];
    all = wave_sum_d(all);
    if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = all;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

__global__ __launch_bounds__(256) void norm_kernel(const double* __restrict__ part, int count, float* __restrict__ norm) {
    __shared__ double ws[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < count; i += 256) sum += part[i];
    sum = wave_sum_d(sum);
    if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) norm[0] = (float)sqrt((ws[0] + ws[1]) + (ws[2] + ws[3]));
}

constexpr int NORM_BLOCKS = 1024;

int64_t chunks_of(int64_t n) { return ceil_div64(n, CHUNK); }
int64_t norm_chunks_of(int64_t n) { return ceil_div64(n, NORM_CHUNK); }

// ---- the update -----------------------------------------------------------------------------------------------------
// a 32-bit mix of position and key, the published integer hash lowbias32 (C. Wellons, 2018: xor-shifts by 16, 15 and 16 around two odd
// factors) over a Weyl sequence; its halves are the random numbers of the two moments.  (The keys' odd factors are those that the
// MurmurHash3 and xxHash mixes use; any odd numbers with as many bits would do.)
__device__ __forceinline__ uint32_t mix(uint32_t i, uint32_t key) {
    uint32_t h = i * 0x9e3779b9u + key;
    h ^= h >> 16;
    h *= 0x7feb352du;
    h ^= h >> 15;
    h *= 0x846ca68bu;
    return h ^ (h >> 16);
}

// Four codes of float formats of eight bits (e4m3, or e5m2 of numbers >= 0), each rounded up with the probability of its value's
// place between its neighbours: the conversion adds the seed's high bits below the last bit it keeps; sixteen of them are random
// (compared with the same sum in integer arithmetic for 16 million values of either format, subnormals among them).
__device__ __forceinline__ uint32_t encode_e4m3(const float t[4], const uint32_t h[4]) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_sr_fp8_f32(t[0], h[0] << 16, c, 0);
    c = __builtin_amdgcn_cvt_sr_fp8_f32(t[1], h[1] << 16, c, 1);
    c = __builtin_amdgcn_cvt_sr_fp8_f32(t[2], h[2] << 16, c, 2);
    return __builtin_amdgcn_cvt_sr_fp8_f32(t[3], h[3] << 16, c, 3);
}
__device__ __forceinline__ uint32_t encode_e5m2(const float t[4], const uint32_t h[4]) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_sr_bf8_f32(t[0], h[0] & 0xffff0000u, c, 0);
    c = __builtin_amdgcn_cvt_sr_bf8_f32(t[1], h[1] & 0xffff0000u, c, 1);
    c = __builtin_amdgcn_cvt_sr_bf8_f32(t[2], h[2] & 0xffff0000u, c, 2);
    return __builtin_amdgcn_cvt_sr_bf8_f32(t[3], h[3] & 0xffff0000u, c, 3);
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t t = (uint32_t)__shfl_xor((int)v, o, 64);
        v = t > v ? t : v;
    }
    return v;
}

struct Scale {
    float scale, inverse;
    bool none;
};
// maximum / top, but 2^-126 at least, so that the scale and its reciprocal are normal numbers: then the codes are fixed point, down to
// 2^-142 in the second moment, and what is positive below that takes its smallest code.  (A second moment lost beside a first one that is
// kept would be a division by eps alone.)
__device__ __forceinline__ Scale scale_for(uint32_t max_bits, float top) {
    const float a = __uint_as_float(max_bits), s = a / top;
    const bool bad = max_bits >= 0x7f800000u, none = bad || max_bits == 0, low = s < 0x1p-126f;
    return {bad ? __uint_as_float(0x7fc00000u) : none ? 0.f : low ? 0x1p-126f : s, none ? 0.f : low ? 0x1p126f : top / a, none};
}

// Per element: g *= clip; m = b1 m + c1 g; v = b2 v + c2 g^2; w = w (1 - lr decay) - rate m / (sqrt(v) root + eps).  A wave takes 512
// consecutive elements, four per lane at a time, everything in registers between one read and one write.  The moments follow
// the formula's fp32 operations exactly (their 8-bit codes are compared bit for bit); the quotient and the root of the update
// itself are the 1-ulp hardware ones.
template <typename T, bool EIGHT, bool MASTER, bool FULL>
__device__ __forceinline__ void adamw_block(const StepArgs& a, int t, int64_t block, int64_t n, float clip) {
    const int lane = threadIdx.x & 63;
    const int64_t base = block * BLOCK;
    T* const p = (T*)a.p[t];
    const T* const g = (const T*)a.g[t];
    float scale_m = 1.f, scale_v = 1.f;
    if (EIGHT) {
        scale_m = a.s[t][2 * block];
        scale_v = a.s[t][2 * block + 1];
    }
    float w[2][4], x[2][4], m[2][4], v[2][4];
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int64_t i = base + u * 256 + lane * 4, valid = FULL ? 4 : n - i;
        load4(g + i, valid, x[u]);
        if (MASTER) load4(a.w[t] + i, valid, w[u]);
        else load4(p + i, valid, w[u]);
        if (EIGHT) {
            const uint32_t cm = load4_codes((const uint8_t*)a.m[t] + i, valid), cv = load4_codes((const uint8_t*)a.v[t] + i, valid);
            const f32x2 m0 = __builtin_amdgcn_cvt_pk_f32_fp8(cm, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8(cm, true);
            const f32x2 v0 = __builtin_amdgcn_cvt_pk_f32_bf8(cv, false), v1 = __builtin_amdgcn_cvt_pk_f32_bf8(cv, true);
            m[u][0] = m0[0] * scale_m, m[u][1] = m0[1] * scale_m, m[u][2] = m1[0] * scale_m, m[u][3] = m1[1] * scale_m;
            v[u][0] = v0[0] * scale_v, v[u][1] = v0[1] * scale_v, v[u][2] = v1[0] * scale_v, v[u][3] = v1[1] * scale_v;
        } else {
            load4((const float*)a.m[t] + i, valid, m[u]);
            load4((const float*)a.v[t] + i, valid, v[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float d = x[u][j] * clip;
            m[u][j] = m[u][j] * a.b1 + d * a.c1;
            v[u][j] = v[u][j] * a.b2 + (d * d) * a.c2;
            const bool low = v[u][j] < 0x1p-96f;         // (the instruction takes the root of a subnormal number for 0)
            const float root = __builtin_amdgcn_sqrtf(low ? v[u][j] * 0x1p64f : v[u][j]) * (low ? 0x1p-32f : 1.f);
            const float denominator = root * a.root + a.eps;
            w[u][j] = w[u][j] * a.keep - (m[u][j] * __builtin_amdgcn_rcpf(denominator)) * a.rate;
            if (EIGHT) {                                 // (elements behind the last were read as zeros and stay zeros)
                top_m = max(top_m, f32_bits(m[u][j]) & 0x7fffffffu);
                top_v = max(top_v, f32_bits(v[u][j]) & 0x7fffffffu);
            }
        }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int64_t i = base + u * 256 + lane * 4, valid = FULL ? 4 : n - i;
        store4(p + i, valid, w[u]);
        if (MASTER) store4(a.w[t] + i, valid, w[u]);
        if (!EIGHT) {
            store4((float*)a.m[t] + i, valid, m[u]);
            store4((float*)a.v[t] + i, valid, v[u]);
        }
    }
    if (EIGHT) {
        const Scale sm = scale_for(wave_max_u32(top_m), 448.f), sv = scale_for(wave_max_u32(top_v), 57344.f);
        if (lane == 0) {
            a.s[t][2 * block] = sm.scale;
            a.s[t][2 * block + 1] = sv.scale;
        }
        const uint32_t key = a.seed * 0x85ebca6bu + (uint32_t)(a.index0 + t) * 0xc2b2ae35u + 0x27d4eb2fu;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t i = base + u * 256 + lane * 4, valid = FULL ? 4 : n - i;
            float tm[4], tv[4];
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[j] = mix((uint32_t)i + j, key);
                tm[j] = sm.none ? 0.f : fminf(fmaxf(m[u][j] * sm.inverse, -448.f), 448.f);
                // a positive second moment never becomes zero: below the smallest number it is that number
                tv[j] = sv.none || v[u][j] == 0.f ? 0.f : fminf(fmaxf(v[u][j] * sv.inverse, 0x1p-16f), 57344.f);
            }
            store4_codes((uint8_t*)a.m[t] + i, valid, encode_e4m3(tm, h));
            store4_codes((uint8_t*)a.v[t] + i, valid, encode_e5m2(tv, h));
        }
    }
}

template <typename T, bool EIGHT, bool MASTER>
__global__ __launch_bounds__(256) void adamw_kernel(const StepArgs a) {
    const uint32_t c = blockIdx.x;
    const int t = tensor_of(a.first, a.count, c);
    const int64_t n = a.n[t], block = (int64_t)(c - a.first[t]) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (block * BLOCK >= n) return;
    float clip = 1.f;
    if (a.norm) {
        const double q = a.max_norm / ((double)a.norm[0] + 1e-6);
        clip = q < 1.0 || q != q ? (float)q : 1.f;
    }
    if (n - block * BLOCK >= BLOCK) adamw_block<T, EIGHT, MASTER, true>(a, t, block, n, clip);
    else adamw_block<T, EIGHT, MASTER, false>(a, t, block, n, clip);
}

template <typename T>
int launch_step(const StepArgs& a, bool eight, bool master, uint32_t chunks, hipStream_t st) {
    constexpr bool SHORT = sizeof(T) == 2;               // only 16-bit parameters have master copies
    if (eight && master) adamw_kernel<T, true, SHORT><<<chunks, 256, 0, st>>>(a);
    else if (eight) adamw_kernel<T, true, false><<<chunks, 256, 0, st>>>(a);
    else if (master) adamw_kernel<T, false, SHORT><<<chunks, 256, 0, st>>>(a);
    else adamw_kernel<T, false, false><<<chunks, 256, 0, st>>>(a);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

bool known(int dtype) { return dtype == SLIM_DTYPE_F32 || dtype == SLIM_DTYPE_BF16 || dtype == SLIM_DTYPE_F16; }
int64_t element_size(int dtype) { return dtype == SLIM_DTYPE_F32 ? 4 : 2; }

}  // namespace

extern "C" int64_t slim_grad_norm_workspace_bytes(int count) {
    return count > 0 ? ceil_div64(count, NORM_TENSORS) * NORM_BLOCKS * 8 : 0;
}

extern "C" int slim_grad_norm(const void* const* grads, const int64_t* numel, int count, int dtype, float* norm, void* workspace,
                              int64_t workspace_bytes, void* stream) {
    SLIM_REQUIRE(grads && numel && count > 0 && norm && workspace, "slim_grad_norm: bad arguments");
    SLIM_REQUIRE(known(dtype), "slim_grad_norm: unknown element type %d", dtype);
    SLIM_REQUIRE(workspace_bytes >= slim_grad_norm_workspace_bytes(count) && (uintptr_t)workspace % 8 == 0, "slim_grad_norm: workspace too small or misaligned");
    double total = 0;
    for (int i = 0; i < count; ++i) {
        SLIM_REQUIRE(grads[i] && numel[i] > 0 && numel[i] <= MAX_NUMEL, "slim_grad_norm: tensor %d is empty or too large", i);
        SLIM_REQUIRE((uintptr_t)grads[i] % element_size(dtype) == 0, "slim_grad_norm: tensor %d is misaligned", i);
        total += (double)numel[i];
    }
    hipStream_t st = (hipStream_t)stream;
    SLIM_PROF("grad_norm", st, total * element_size(dtype), 2 * total);
    int parts = 0;
    for (int i = 0; i < count;) {
        NormArgs a;
        int64_t chunks = 0;
        for (a.count = 0; a.count < NORM_TENSORS && i < count; ++a.count, ++i) {
            a.g[a.count] = grads[i];
            a.n[a.count] = numel[i];
            a.first[a.count] = (uint32_t)chunks;
            chunks += norm_chunks_of(numel[i]);
        }
        a.first[a.count] = (uint32_t)chunks;
        const int blocks = (int)(chunks < NORM_BLOCKS ? chunks : NORM_BLOCKS);
        double* part = (double*)workspace + parts;
        if (dtype == SLIM_DTYPE_F32) sumsq_kernel<float><<<blocks, 256, 0, st>>>(a, part);
        else if (dtype == SLIM_DTYPE_BF16) sumsq_kernel<bf16_t><<<blocks, 256, 0, st>>>(a, part);
        else sumsq_kernel<_Float16><<<blocks, 256, 0, st>>>(a, part);
        SLIM_LAUNCH_CHECK();
        parts += blocks;
    }
    norm_kernel<<<1, 256, 0, st>>>((const double*)workspace, parts, norm);
    SLIM_LAUNCH_CHECK();
    return SLIM_OK;
}

extern "C" int64_t slim_adamw_blocks(int64_t numel) { return numel > 0 ? ceil_div64(numel, BLOCK) : 0; }

extern "C" int slim_adamw_step(void* const* params, const void* const* grads, void* const* exp_avg, void* const* exp_avg_sq, float* const* scales,
                               float* const* masters, const int64_t* numel, int count, int dtype, int first_index, int64_t step, double lr,
                               double beta1, double beta2, double eps, double weight_decay, const float* norm, double max_norm, uint32_t seed,
                               void* stream) {
    SLIM_REQUIRE(params && grads && exp_avg && exp_avg_sq && numel && count > 0, "slim_adamw_step: bad arguments");
    SLIM_REQUIRE(known(dtype), "slim_adamw_step: unknown element type %d", dtype);
    SLIM_REQUIRE(step >= 1 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && lr >= 0 && weight_decay >= 0 && first_index >= 0,
                 "slim_adamw_step: step counts from 1, betas lie in [0, 1), lr, eps and weight_decay are not negative");
    SLIM_REQUIRE(eps == 0 || eps >= 0x1p-126, "slim_adamw_step: eps is 0 or a normal fp32 number");
    SLIM_REQUIRE(!norm || max_norm > 0, "slim_adamw_step: max_norm must be positive");
    SLIM_REQUIRE(!masters || dtype != SLIM_DTYPE_F32, "slim_adamw_step: fp32 parameters need no master copies");
    const int64_t size = element_size(dtype);
    double total = 0;
    for (int i = 0; i < count; ++i) {
        SLIM_REQUIRE(params[i] && grads[i] && exp_avg[i] && exp_avg_sq[i] && (!scales || scales[i]) && (!masters || masters[i]), "slim_adamw_step: tensor %d: null pointer", i);
        SLIM_REQUIRE(numel[i] > 0 && numel[i] <= MAX_NUMEL, "slim_adamw_step: tensor %d is empty or too large", i);
        SLIM_REQUIRE((uintptr_t)params[i] % size == 0 && (uintptr_t)grads[i] % size == 0 && (scales ? (uintptr_t)scales[i] % 4 == 0 : ((uintptr_t)exp_avg[i] | (uintptr_t)exp_avg_sq[i]) % 4 == 0) &&
                     (!masters || (uintptr_t)masters[i] % 4 == 0), "slim_adamw_step: tensor %d is misaligned", i);
        total += (double)numel[i];
    }
    hipStream_t st = (hipStream_t)stream;
    SLIM_PROF("adamw", st, total * (3 * size + (scales ? 4 + 16.0 / BLOCK : 16) + (masters ? 8 - size : 0)), 16 * total);
    StepArgs a;
    a.norm = norm;
    a.max_norm = max_norm;
    a.b1 = (float)beta1, a.c1 = (float)(1 - beta1), a.b2 = (float)beta2, a.c2 = (float)(1 - beta2);
    a.keep = (float)(1 - lr * weight_decay);
    a.rate = (float)(lr / (1 - std::pow(beta1, (double)step)));
    a.root = (float)(1 / std::sqrt(1 - std::pow(beta2, (double)step)));
    a.eps = (float)eps;
    a.seed = seed;
    for (int i = 0; i < count;) {
        int64_t chunks = 0;
        a.index0 = first_index + i;
        for (a.count = 0; a.count < STEP_TENSORS && i < count && chunks + chunks_of(numel[i]) <= MAX_CHUNKS; ++a.count, ++i) {
            a.p[a.count] = params[i];
            a.g[a.count] = grads[i];
            a.m[a.count] = exp_avg[i];
            a.v[a.count] = exp_avg_sq[i];
            a.s[a.count] = scales ? scales[i] : nullptr;
            a.w[a.count] = masters ? masters[i] : nullptr;
            a.n[a.count] = numel[i];
            a.first[a.count] = (uint32_t)chunks;
            chunks += chunks_of(numel[i]);
        }
        a.first[a.count] = (uint32_t)chunks;
        int rc;
        if (dtype == SLIM_DTYPE_F32) rc = launch_step<float>(a, scales, false, (uint32_t)chunks, st);
        else if (dtype == SLIM_DTYPE_BF16) rc = launch_step<bf16_t>(a, scales, masters, (uint32_t)chunks, st);
        else rc = launch_step<_Float16>(a, scales, masters, (uint32_t)chunks, st);
        if (rc) return rc;
    }
    return SLIM_OK;
}
