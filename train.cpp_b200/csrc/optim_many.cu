// optim_many.cu -- the optimizer over many tensors at once: AdamW with 32-bit or 8-bit states, and the
// squared norm of all gradients that clips it.
//
// A low-rank adapter gives two small tensors for every projection, hundreds for a model, so one launch
// per tensor costs more than its work. Here the tensors of a call are a table in the kernel's parameters,
// cut into runs of 1024 elements; one CTA of four warps takes one run. Many short CTAs overlap one another's
// loads, roots and stores best. 202 M elements, clipped 32-bit step / 8-bit step with the states read back, in us, as
// the forms compared when they were tried (the kept one, the first, since took 937 - 951 / 888 - 1004 on several machines):
//   four warps, one block of 256 for each         937 /  886
//   eight warps, one, two or four blocks in turn   935 /  928, 946 / 1103, 977 / 1065
//   eight warps, one block, 24 warps on an SM (80 registers instead of 64)  934 / 1027
//   eight warps, eight blocks in turn, the next one's loads through a ring of asynchronous copies  - / 1110
//
// 32-bit states: every fp32 operation is rounded by itself, in the order of train_ops.cu's adamw_kernel, so the
// step is bit-exact with the one-tensor step. 28 bytes for each element leave room for its two divisions and square
// root.
// 8-bit states: 16 bytes for each element leave about 60 instructions. The new moments and their codes are still
// those of separately rounded operations; only the parameter's own step takes the approximate quotient and square
// root (5 * 2^-23 of the step at most). A code is round(sqrt(x * per)): the approximate square root (2^-23)
// decides it except next to a border, where the rounded one does. Codes become numbers and numbers codes through
// the low bits of 2^23 + c, because the conversion unit is the one that the roots need. 83 instructions for each element were
// left of 126 (conversions, four rounded roots, two rounded quotients): 202 M elements take 585 - 700 us, 4.7 - 5.6 TB/s.
// What bounds it is their latency at 32 warps on an SM, no longer one unit. With a rounded root and rounded quotients in the
// parameter's own step, measured in turn and with the states read back: 1140 us against 967. 64 registers leave 32 - 36
// bytes of a thread in local memory.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "trc_internal.h"
#include "trc_ptx.cuh"

namespace trc {

namespace {

constexpr int kThreads = 256;
constexpr int kStepThreads = 128, kRun = 1024;  // a CTA of the step: 8 elements per thread, 4 blocks of an 8-bit state
constexpr int kBlock   = TRC_CUDA_STATE8_BLOCK;
constexpr int kFewJobs = 32, kMaxJobs = 480;  // tensors of one launch (2 or 31 KB of kernel parameters)
static_assert(kRun == kStepThreads * 8 && kBlock == 256, "a warp takes one block of 256, 8 elements per lane");

// 1 / 127^2 and 1 / 255^2: the units of the two square laws.
constexpr float kUnitM = 1.0f / 16129.0f, kUnitV = 1.0f / 65025.0f;
constexpr float kTinyM = 7.888609052210118e-31f;  // 2^-100: below it 16129 / max|m| could overflow

struct AdamwParams {
    float step_sz, bc2_sqrt, decay, beta1, beta2, eps, max_norm, clip_eps;
};

struct StepJob {
    float*       p;
    const float* g;
    void*        m;
    void*        v;
    float*       m_scale;
    float*       v_scale;
    int64_t      n;
    int32_t      run_begin;  // first run of this tensor
    int32_t      aligned;    // its vectors may be loaded whole
};

// Two sizes of table: a launch copies all of its parameters.
template <int JOBS>
struct StepBatch {
    static constexpr int kJobs = JOBS;
    const float* norm;
    AdamwParams  a;
    int32_t      n_jobs;
    StepJob      job[JOBS];
};
static_assert(sizeof(StepBatch<kMaxJobs>) <= 32764, "kernel parameter limit");

// The tensor that run `run` belongs to (run_begin ascends).
template <class JOB>
__device__ __forceinline__ int job_of(const JOB* job, int n_jobs, int run) {
    int lo = 0, hi = n_jobs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (job[mid].run_begin <= run) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Four consecutive floats at i, those beyond n as zero.
__device__ __forceinline__ void load4(const float* q, int64_t i, int64_t n, bool whole, float (&x)[4]) {
    if (whole && i + 4 <= n) {
        const float4 t = *reinterpret_cast<const float4*>(q + i);
        x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = i + e < n ? q[i + e] : 0.0f;
    }
}

__device__ __forceinline__ void store4(float* q, int64_t i, int64_t n, bool whole, const float (&x)[4]) {
    if (whole && i + 4 <= n) {
        *reinterpret_cast<float4*>(q + i) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) q[i + e] = x[e];
    }
}

// The same for one-byte codes (four in a word, byte e = element e).
__device__ __forceinline__ uint32_t load4c(const uint8_t* q, int64_t i, int64_t n, bool whole) {
    if (whole && i + 4 <= n) return *reinterpret_cast<const uint32_t*>(q + i);
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < n) w |= static_cast<uint32_t>(q[i + e]) << (8 * e);
    return w;
}

__device__ __forceinline__ void store4c(uint8_t* q, int64_t i, int64_t n, bool whole, uint32_t w) {
    if (whole && i + 4 <= n) {
        *reinterpret_cast<uint32_t*>(q + i) = w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) q[i + e] = static_cast<uint8_t>(w >> (8 * e));
    }
}

// The whole number in byte e of w, exactly: 0x4B0000cc is the float 2^23 + c.
__device__ __forceinline__ float byte_value(uint32_t w, int e, float bias) {
    return __fsub_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440u + e)), bias);
}

__device__ __forceinline__ float decode_m(uint32_t w, int e, float scale) {
    const float c = byte_value(w ^ 0x80808080u, e, 8388608.0f + 128.0f);
    return __fmul_rn(__fmul_rn(c, fabsf(c)), scale);  // c * |c| is exact
}

__device__ __forceinline__ float decode_v(uint32_t w, int e, float scale) {
    const float c = byte_value(w, e, 8388608.0f);
    const float u = __fmul_rn(__fmul_rn(c, c), scale);
    return __fmul_rn(u, u);
}

// The largest of the warp's values, NaN if one of them is infinite, NaN or negative: the bits of floats that are not
// negative are in their order, and the bits of the others are larger.
__device__ __forceinline__ float block_max(const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]));
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    return top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(top);
}

__device__ __forceinline__ float sqrt_approx(float x) {  // relative error 2^-23; 0 below 2^-126
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// a, |a| <= 256, rounded to nearest even: the low byte of 1.5 * 2^23 + a (of a two's complement number where a < 0).
// off: how far a is from it, at most 1/2.
__device__ __forceinline__ uint32_t code_of(float a, float& off) {
    const float up = __fadd_rn(a, 12582912.0f);
    off = fmaxf(off, fabsf(__fsub_rn(a, __fsub_rn(up, 12582912.0f))));
    return __float_as_uint(up);
}

__device__ __forceinline__ float with_sign(float a, float of) {
    return __uint_as_float(__float_as_uint(a) | (__float_as_uint(of) & 0x80000000u));
}

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {  // their low bytes
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// One block's new codes from the warp's 8 values per lane (a lane's values 0-3 in w[0], 4-7 in
// w[1]); returns the scale. The borders that the rounded operations decide: a root is at most 127.001 or 255.001; for
// m the approximate and the rounded root of the same product differ by 1.5 * 2^-23 of it, below 2^-15; for v the
// product's own root is approximate too, together 2.75 * 2^-23, below 2^-13.
__device__ __forceinline__ float encode_m(const float (&m)[8], uint32_t (&w)[2]) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fabsf(m[e]);
    float top = block_max(x);
    if (top < kTinyM) top = 0.0f;
    const float per = top > 0.0f ? __fdiv_rn(16129.0f, top) : 0.0f;  // 0 for NaN too
    w[0] = w[1] = 0;
    if (per > 0.0f) {  // the same for the whole warp
        uint32_t c[8];
        float    off = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = code_of(with_sign(sqrt_approx(__fmul_rn(x[e], per)), m[e]), off);
        if (off > 0.5f - 0x1p-15f)
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e] = code_of(with_sign(__fsqrt_rn(__fmul_rn(x[e], per)), m[e]), off);
        w[0] = pack4(c[0], c[1], c[2], c[3]);
        w[1] = pack4(c[4], c[5], c[6], c[7]);
    }
    return __fmul_rn(top, kUnitM);
}

// root: the approximate roots of v, exact ones below 2^-126. The largest root is the root of the largest value:
// rounding keeps the order. A v > 0 takes the code 1 at least, or, where that would read back as 0 (the block's largest root
// is below 2^-59, so the square of its scale rounds to 0), the first code that does not; 255 never does.
__device__ __forceinline__ float encode_v(const float (&v)[8], const float (&root)[8], uint32_t (&w)[2]) {
    const float top = __fsqrt_rn(block_max(v));
    const float per = top > 0.0f ? __fdiv_rn(65025.0f, top) : 0.0f, scale = __fmul_rn(top, kUnitV);
    w[0] = w[1] = 0;
    if (per > 0.0f) {
        uint32_t c[8];
        float    off = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            c[e] = code_of(fmaxf(sqrt_approx(__fmul_rn(root[e], per)), v[e] > 0.0f ? 1.0f : 0.0f), off);
        if (off > 0.5f - 0x1p-13f)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                c[e] = code_of(fmaxf(__fsqrt_rn(__fmul_rn(__fsqrt_rn(v[e]), per)), v[e] > 0.0f ? 1.0f : 0.0f), off);
        if (__fmul_rn(scale, scale) == 0.0f) {  // the same for the whole warp
            uint32_t least = 2;
            while (least < 255 && decode_v(least, 0, scale) == 0.0f) ++least;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v[e] > 0.0f) c[e] = max(c[e], __float_as_uint(12582912.0f) + least);
        }
        w[0] = pack4(c[0], c[1], c[2], c[3]);
        w[1] = pack4(c[4], c[5], c[6], c[7]);
    }
    return scale;
}

__device__ __forceinline__ float root_of(float v) {
    float root = sqrt_approx(v);
    if (__float_as_uint(v) - 1u < 0x007FFFFFu) root = __fsqrt_rn(v);  // 0 < v < 2^-126
    return root;
}

// One element's step: train_ops.cu's adamw_kernel.
__device__ __forceinline__ void adamw_one(float& p, float g, float& m, float& v, const AdamwParams& a, float one_b1,
                                          float one_b2) {
    m = __fadd_rn(m, __fmul_rn(__fsub_rn(g, m), one_b1));
    v = __fadd_rn(__fmul_rn(v, a.beta2), __fmul_rn(__fmul_rn(g, g), one_b2));
    const float denom = __fadd_rn(__fdiv_rn(__fsqrt_rn(v), a.bc2_sqrt), a.eps);
    p = __fsub_rn(__fmul_rn(p, a.decay), __fmul_rn(a.step_sz, __fdiv_rn(m, denom)));
}

// The same with 8-bit states: m and v as above, the parameter's step with approximate operations (inv_bc2 is
// 1 / bc2_sqrt rounded; the quotient is within 2 units, the root and the two products within one: 5 * 2^-23).
__device__ __forceinline__ void adamw_one_8(float& p, float g, float& m, float& v, float& root,
                                            const AdamwParams& a, float one_b1, float one_b2, float inv_bc2) {
    m = __fadd_rn(m, __fmul_rn(__fsub_rn(g, m), one_b1));
    v = __fadd_rn(__fmul_rn(v, a.beta2), __fmul_rn(__fmul_rn(g, g), one_b2));
    root = root_of(v);
    const float denom = fmaf(root, inv_bc2, a.eps);
    p = __fsub_rn(__fmul_rn(p, a.decay), __fmul_rn(a.step_sz, __fdividef(m, denom)));
}

// One block of 256 by one warp, 8 elements per lane. FULL: the block lies inside the tensor and may be loaded whole.
template <int BITS, bool FULL>
__device__ __forceinline__ void step_block(const StepJob& J, int64_t b0, const AdamwParams& a, bool clipped, float clip) {
    const int     lane = threadIdx.x & 31;
    const int64_t i0 = b0 * kBlock + lane * 4, n = FULL ? INT64_MAX : J.n;
    const float   one_b1 = __fsub_rn(1.0f, a.beta1), one_b2 = __fsub_rn(1.0f, a.beta2);
    float p[2][4], g[2][4], m[8], v[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        load4(J.p, i0 + 128 * h, n, FULL, p[h]);
        load4(J.g, i0 + 128 * h, n, FULL, g[h]);
    }
    if constexpr (BITS == 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            load4(static_cast<const float*>(J.m), i0 + 128 * h, n, FULL, reinterpret_cast<float (&)[4]>(m[4 * h]));
            load4(static_cast<const float*>(J.v), i0 + 128 * h, n, FULL, reinterpret_cast<float (&)[4]>(v[4 * h]));
        }
    } else {
        const float sm = J.m_scale[b0], sv = J.v_scale[b0];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t wm = load4c(static_cast<const uint8_t*>(J.m), i0 + 128 * h, n, FULL);
            const uint32_t wv = load4c(static_cast<const uint8_t*>(J.v), i0 + 128 * h, n, FULL);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[4 * h + e] = decode_m(wm, e, sm);
                v[4 * h + e] = decode_v(wv, e, sv);
            }
        }
    }
    [[maybe_unused]] const float inv_bc2 = __fdiv_rn(1.0f, a.bc2_sqrt);
    [[maybe_unused]] float root[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float ge = clipped ? __fmul_rn(g[h][e], clip) : g[h][e];
            if constexpr (BITS == 32) adamw_one(p[h][e], ge, m[4 * h + e], v[4 * h + e], a, one_b1, one_b2);
            else adamw_one_8(p[h][e], ge, m[4 * h + e], v[4 * h + e], root[4 * h + e], a, one_b1, one_b2, inv_bc2);
        }
#pragma unroll
    for (int h = 0; h < 2; ++h) store4(J.p, i0 + 128 * h, n, FULL, p[h]);
    if constexpr (BITS == 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            store4(static_cast<float*>(J.m), i0 + 128 * h, n, FULL, reinterpret_cast<float (&)[4]>(m[4 * h]));
            store4(static_cast<float*>(J.v), i0 + 128 * h, n, FULL, reinterpret_cast<float (&)[4]>(v[4 * h]));
        }
    } else {
        if constexpr (!FULL)  // what lies behind the tensor's end is not part of its last block
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i0 + 128 * (e >> 2) + (e & 3) >= n) m[e] = v[e] = root[e] = 0.0f;
        uint32_t wm[2], wv[2];
        const float sm = encode_m(m, wm), sv = encode_v(v, root, wv);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            store4c(static_cast<uint8_t*>(J.m), i0 + 128 * h, n, FULL, wm[h]);
            store4c(static_cast<uint8_t*>(J.v), i0 + 128 * h, n, FULL, wv[h]);
        }
        if (lane == 0) {
            J.m_scale[b0] = sm;
            J.v_scale[b0] = sv;
        }
    }
}

template <int BITS, int JOBS>
__global__ void __launch_bounds__(kStepThreads, 8) adamw_many_kernel(const __grid_constant__ StepBatch<JOBS> batch) {
    grid_wait();
    grid_dependents();
    // From the last run to the first: the norm's pass read the gradients from the first to the last, so
    // those that are still in L2 come first.
    const int      run = static_cast<int>(gridDim.x - 1 - blockIdx.x);
    const StepJob& J   = batch.job[job_of(batch.job, batch.n_jobs, run)];
    const bool     clipped = batch.norm != nullptr;
    float clip = 1.0f;
    if (clipped) {  // clip_scale_kernel's factor
        clip = __fdiv_rn(batch.a.max_norm, __fadd_rn(__fsqrt_rn(batch.norm[0]), batch.a.clip_eps));
        if (clip > 1.0f) clip = 1.0f;
    }
    const int64_t b0 = static_cast<int64_t>(run - J.run_begin) * (kRun / kBlock) + (threadIdx.x >> 5);
    if (b0 * kBlock >= J.n) return;
    if (J.aligned && (b0 + 1) * kBlock <= J.n) step_block<BITS, true>(J, b0, batch.a, clipped, clip);
    else step_block<BITS, false>(J, b0, batch.a, clipped, clip);
}

// ------------------------------------------------------------------ 8-bit states <-> values
// To values: a warp takes four blocks of 256 (one left 22 % more time at 202 M elements), back: one.
constexpr int kToF32 = 4;

template <int WHICH>
__global__ void __launch_bounds__(kThreads) state8_to_f32_kernel(const uint8_t* codes, const float* scales, float* values,
                                                                 int64_t n, bool whole) {
    const int64_t b = (static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5)) * kToF32;
    const int64_t i0 = b * kBlock + (threadIdx.x & 31) * 4;
    uint32_t w[kToF32][2];
    float    s[kToF32];
#pragma unroll
    for (int k = 0; k < kToF32; ++k) {
        s[k] = (b + k) * kBlock < n ? scales[b + k] : 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) w[k][h] = load4c(codes, i0 + kBlock * k + 128 * h, n, whole);
    }
#pragma unroll
    for (int k = 0; k < kToF32; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = WHICH == 0 ? decode_m(w[k][h], e, s[k]) : decode_v(w[k][h], e, s[k]);
            store4(values, i0 + kBlock * k + 128 * h, n, whole, x);
        }
}

template <int WHICH>
__global__ void __launch_bounds__(kThreads) state8_from_f32_kernel(const float* values, uint8_t* codes, float* scales,
                                                                   int64_t n, bool whole) {
    const int64_t b = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
    const int64_t i0 = b * kBlock + (threadIdx.x & 31) * 4;
    if (b * kBlock >= n) return;
    float x[8];
    load4(values, i0, n, whole, reinterpret_cast<float (&)[4]>(x[0]));
    load4(values, i0 + 128, n, whole, reinterpret_cast<float (&)[4]>(x[4]));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(x[e], 0.0f);  // no -0
    uint32_t w[2];
    float s;
    if constexpr (WHICH == 0) {
        s = encode_m(x, w);
    } else {
        float root[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) root[e] = root_of(x[e]);
        s = encode_v(x, root, w);
    }
    store4c(codes, i0, n, whole, w[0]);
    store4c(codes, i0 + 128, n, whole, w[1]);
    if ((threadIdx.x & 31) == 0) scales[b] = s;
}

// ------------------------------------------------------------------ squared norm of many tensors
// Pass 1: one double for each chunk of a span (each square is exact in double). Pass 2 adds them in a
// fixed order.
constexpr int64_t kChunk    = 16384;
constexpr int     kMaxSpans = 1000;

struct Span {
    const float* a;
    int64_t      n;
    int32_t      run_begin;
    int32_t      aligned;
};

template <int JOBS>
struct SpanBatch {
    static constexpr int kJobs = JOBS;
    double* partials;
    int32_t n_jobs;
    Span    job[JOBS];
};
static_assert(sizeof(SpanBatch<kMaxSpans>) <= 32764, "kernel parameter limit");

struct SumBatch {
    const double* partials;
    int64_t       n;
    float*        out;
};

__device__ __forceinline__ double block_sum(double s) {
    __shared__ double sh[kThreads / 32];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_down_sync(0xFFFFFFFFu, s, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0.0;
    if (threadIdx.x == 0)
        for (int w = 0; w < kThreads / 32; ++w) s = __dadd_rn(s, sh[w]);
    return s;
}

template <int JOBS>
__global__ void __launch_bounds__(kThreads) sum_sqr_many_kernel(const __grid_constant__ SpanBatch<JOBS> batch) {
    grid_wait();
    grid_dependents();
    const int     run = static_cast<int>(blockIdx.x);
    const Span&   J   = batch.job[job_of(batch.job, batch.n_jobs, run)];
    const int64_t lo = static_cast<int64_t>(run - J.run_begin) * kChunk, hi = min(J.n, lo + kChunk);
    // 8 loads on their way at a time, four sums of their own
    double part[4] = {};
    for (int64_t i = lo + threadIdx.x * 4; i < hi; i += kThreads * 32) {
        float x[8][4];
#pragma unroll
        for (int u = 0; u < 8; ++u) load4(J.a, i + kThreads * 4 * u, hi, J.aligned != 0, x[u]);
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double d = static_cast<double>(x[u][e]);
                part[e] = fma(d, d, part[e]);
            }
    }
    double s = __dadd_rn(__dadd_rn(part[0], part[1]), __dadd_rn(part[2], part[3]));
    s = block_sum(s);
    if (threadIdx.x == 0) batch.partials[run] = s;
}

__global__ void __launch_bounds__(kThreads) sum_sqr_many_final_kernel(const __grid_constant__ SumBatch b) {
    grid_wait();
    grid_dependents();
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < b.n; i += kThreads) s = __dadd_rn(s, b.partials[i]);
    s = block_sum(s);
    if (threadIdx.x == 0) b.out[0] = __double2float_rn(s);
}

bool aligned_to(const void* p, uint64_t bytes) { return (reinterpret_cast<uint64_t>(p) & (bytes - 1)) == 0; }

int64_t chunks_of(const trc_cuda_span* spans, int n_spans) {
    int64_t c = 0;
    for (int i = 0; i < n_spans; ++i) c += spans[i].n > 0 ? (spans[i].n + kChunk - 1) / kChunk : 0;
    return c;
}

// Launches a kernel that may be set up while the one before it on the stream drains: it begins with grid_wait().
template <class ARGS>
int launch(void (*kernel)(ARGS), int64_t grid, int threads, const ARGS& args, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    void* list[] = {const_cast<ARGS*>(&args)};
    const cudaError_t e = cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), list);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return cuda_fail(e);
    }
    note_launch();
    return TRC_CUDA_OK;
}

constexpr int64_t kMaxElems = int64_t(1) << 40;  // of one tensor: its runs and chunks fit a grid

template <int JOBS>
int step_many(const trc_cuda_adamw_job* jobs, int n_jobs, int state_bits, const AdamwParams& a, const float* norm, cudaStream_t s) {
    const uint64_t state_bytes = state_bits == 32 ? 4 : 1;
    StepBatch<JOBS> batch;
    batch.norm = norm;
    batch.a = a;
    // Batches from the last tensor to the first, as the runs inside a launch.
    for (int last = n_jobs; last > 0;) {
        int64_t runs = 0;
        int first = last;
        batch.n_jobs = 0;
        while (first > 0 && last - first < JOBS) {
            const int64_t r = (jobs[first - 1].n + kRun - 1) / kRun;
            if (runs + r > INT32_MAX) break;
            runs += r;
            --first;
        }
        runs = 0;
        for (int i = first; i < last; ++i) {
            const trc_cuda_adamw_job& in = jobs[i];
            if (in.n == 0) continue;
            StepJob& J  = batch.job[batch.n_jobs++];
            J.p         = in.param;
            J.g         = in.grad;
            J.m         = in.m;
            J.v         = in.v;
            J.m_scale   = in.m_scale;
            J.v_scale   = in.v_scale;
            J.n         = in.n;
            J.run_begin = static_cast<int32_t>(runs);
            J.aligned   = aligned_to(in.param, 16) && aligned_to(in.grad, 16) && aligned_to(in.m, 4 * state_bytes) &&
                        aligned_to(in.v, 4 * state_bytes);
            runs += (in.n + kRun - 1) / kRun;
        }
        last = first;
        if (runs == 0) continue;
        const int st = state_bits == 32 ? launch(&adamw_many_kernel<32, JOBS>, runs, kStepThreads, batch, s)
                                          : launch(&adamw_many_kernel<8, JOBS>, runs, kStepThreads, batch, s);
        if (st != TRC_CUDA_OK) return st;
    }
    return TRC_CUDA_OK;
}

template <int JOBS>
int sum_many(const trc_cuda_span* spans, int n_spans, float* out, double* partials, cudaStream_t s) {
    int64_t done = 0;
    SpanBatch<JOBS> batch;
    for (int i = 0; i < n_spans;) {
        int64_t runs = 0;
        batch.n_jobs = 0;
        batch.partials = partials + done;
        for (; i < n_spans && batch.n_jobs < JOBS; ++i) {
            const int64_t r = (spans[i].n + kChunk - 1) / kChunk;
            if (r == 0) continue;
            if (runs + r > INT32_MAX) break;
            batch.job[batch.n_jobs++] = Span{spans[i].data, spans[i].n, static_cast<int32_t>(runs),
                                             aligned_to(spans[i].data, 16) ? 1 : 0};
            runs += r;
        }
        if (runs == 0) continue;
        const int st = launch(&sum_sqr_many_kernel<JOBS>, runs, kThreads, batch, s);
        if (st != TRC_CUDA_OK) return st;
        done += runs;
    }
    return launch(&sum_sqr_many_final_kernel, 1, kThreads, SumBatch{partials, done, out}, s);
}

}  // namespace

}  // namespace trc

using namespace trc;

extern "C" {

int trc_cuda_opt_step_adamw_many(const trc_cuda_adamw_job* jobs, int n_jobs, int state_bits, const float* params6,
                                 const float* norm, float max_norm, float clip_eps, void* stream) {
    if (n_jobs < 0 || (n_jobs > 0 && jobs == nullptr) || params6 == nullptr) return TRC_CUDA_EINVAL;
    if (state_bits != 32 && state_bits != 8) return TRC_CUDA_EUNSUPPORTED;
    if (!aligned_to(norm, 4)) return TRC_CUDA_EINVAL;
    const uint64_t state_bytes = state_bits == 32 ? 4 : 1;
    for (int i = 0; i < n_jobs; ++i) {  // every tensor before the first launch
        const trc_cuda_adamw_job& in = jobs[i];
        if (in.n < 0 || in.n > kMaxElems) return TRC_CUDA_EINVAL;
        if (in.n == 0) continue;
        if (in.param == nullptr || in.grad == nullptr || in.m == nullptr || in.v == nullptr) return TRC_CUDA_EINVAL;
        if (!aligned_to(in.param, 4) || !aligned_to(in.grad, 4) || !aligned_to(in.m, state_bytes) ||
            !aligned_to(in.v, state_bytes))
            return TRC_CUDA_EINVAL;
        if (state_bits == 8 && (in.m_scale == nullptr || in.v_scale == nullptr || !aligned_to(in.m_scale, 4) ||
                                !aligned_to(in.v_scale, 4)))
            return TRC_CUDA_EINVAL;
    }
    const AdamwParams a{params6[0], params6[1], params6[2], params6[3], params6[4], params6[5], max_norm, clip_eps};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return n_jobs <= kFewJobs ? step_many<kFewJobs>(jobs, n_jobs, state_bits, a, norm, s)
                              : step_many<kMaxJobs>(jobs, n_jobs, state_bits, a, norm, s);
}

int trc_cuda_state8_to_f32(int which, const void* codes, const float* scales, float* values, int64_t n, void* stream) {
    if (which != 0 && which != 1) return TRC_CUDA_EUNSUPPORTED;
    if (n < 0 || n > kMaxElems) return TRC_CUDA_EINVAL;
    if (n == 0) return TRC_CUDA_OK;
    if (codes == nullptr || scales == nullptr || values == nullptr || !aligned_to(scales, 4) || !aligned_to(values, 4))
        return TRC_CUDA_EINVAL;
    const unsigned grid = static_cast<unsigned>((n + kThreads * 8 * kToF32 - 1) / (kThreads * 8 * kToF32));
    const bool whole = aligned_to(codes, 4) && aligned_to(values, 16);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint8_t* c = static_cast<const uint8_t*>(codes);
    if (which == 0) state8_to_f32_kernel<0><<<grid, kThreads, 0, s>>>(c, scales, values, n, whole);
    else state8_to_f32_kernel<1><<<grid, kThreads, 0, s>>>(c, scales, values, n, whole);
    note_launch();
    return check_launch();
}

int trc_cuda_state8_from_f32(int which, const float* values, void* codes, float* scales, int64_t n, void* stream) {
    if (which != 0 && which != 1) return TRC_CUDA_EUNSUPPORTED;
    if (n < 0 || n > kMaxElems) return TRC_CUDA_EINVAL;
    if (n == 0) return TRC_CUDA_OK;
    if (codes == nullptr || scales == nullptr || values == nullptr || !aligned_to(scales, 4) || !aligned_to(values, 4))
        return TRC_CUDA_EINVAL;
    const unsigned grid = static_cast<unsigned>((n + kThreads * 8 - 1) / (kThreads * 8));
    const bool whole = aligned_to(codes, 4) && aligned_to(values, 16);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint8_t* c = static_cast<uint8_t*>(codes);
    if (which == 0) state8_from_f32_kernel<0><<<grid, kThreads, 0, s>>>(values, c, scales, n, whole);
    else state8_from_f32_kernel<1><<<grid, kThreads, 0, s>>>(values, c, scales, n, whole);
    note_launch();
    return check_launch();
}

size_t trc_cuda_sum_sqr_many_workspace_bytes(const trc_cuda_span* spans, int n_spans) {
    if (n_spans < 0 || (n_spans > 0 && spans == nullptr)) return 0;
    return static_cast<size_t>(std::max<int64_t>(1, chunks_of(spans, n_spans))) * sizeof(double);
}

int trc_cuda_sum_sqr_many(const trc_cuda_span* spans, int n_spans, float* out, void* workspace,
                          size_t workspace_bytes, void* stream) {
    if (n_spans < 0 || (n_spans > 0 && spans == nullptr) || out == nullptr || !aligned_to(out, 4)) return TRC_CUDA_EINVAL;
    for (int i = 0; i < n_spans; ++i) {
        if (spans[i].n < 0 || spans[i].n > kMaxElems) return TRC_CUDA_EINVAL;
        if (spans[i].n > 0 && (spans[i].data == nullptr || !aligned_to(spans[i].data, 4))) return TRC_CUDA_EINVAL;
    }
    if (workspace == nullptr || !aligned_to(workspace, 8) ||
        workspace_bytes < trc_cuda_sum_sqr_many_workspace_bytes(spans, n_spans))
        return TRC_CUDA_EINVAL;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    double* partials = static_cast<double*>(workspace);
    return n_spans <= kFewJobs ? sum_many<kFewJobs>(spans, n_spans, out, partials, s)
                               : sum_many<kMaxSpans>(spans, n_spans, out, partials, s);
}

}  // extern "C"
