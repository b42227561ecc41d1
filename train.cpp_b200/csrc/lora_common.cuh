// lora_common.cuh -- what the kernels of the low-rank adapters share (lora.cu, lora_tc.cu).
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "trc_internal.h"
#include "trc_ptx.cuh"

namespace trc {
namespace lora {

struct Adapter {
    const void* a;
    const void* b;
    float*      da;
    float*      db;
    float       scale;
    int16_t     rank;
    int16_t     vec;  // bit 0: A may be loaded four values at a time, bit 1: B
};

struct Adapters {
    Adapter ad[TRC_CUDA_LORA_MAX_ADAPTERS];
    int32_t n;
};

// The rows of a ggml view: row t = (i1, i2, i3) in ggml order.
struct Rows {
    char*   data;
    int64_t nb0, nb1, nb2, nb3;
    int32_t n1, n2;
    int32_t step;  // rows are this many floats apart throughout; -1: they are not
    template <bool EVEN>
    __device__ __forceinline__ char* row(int64_t t) const {
        if (EVEN || step >= 0) return data + 4 * (t * step);
        const int64_t i1 = t % n1, r = t / n1;
        return data + i1 * nb1 + (r % n2) * nb2 + (r / n2) * nb3;
    }
};

__device__ __forceinline__ int adapter_of(const int32_t* ids, int64_t t, int n) {
    const int id = ids == nullptr ? 0 : ids[t];
    return id >= 0 && id < n ? id : -1;
}

// x = head + tail, the head rounded to TF32's 11 bits and the tail exact; the tensor core reads the
// tail's first 11 bits, so head + tail as it sees them are within 2^-21 of x.
__device__ __forceinline__ void split(float x, uint32_t& head, uint32_t& tail) {
    head = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    tail = __float_as_uint(x - __uint_as_float(head));
}

// N factor values held in the words of one load, as floats.
template <typename W, int N>
__device__ __forceinline__ void widen(const uint32_t (&raw)[N * sizeof(W) / 4], float (&w)[N]) {
    if constexpr (sizeof(W) == 4) {
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = __uint_as_float(raw[j]);
    } else {
        const W* e = reinterpret_cast<const W*>(raw);
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = static_cast<float>(e[j]);
    }
}

// N consecutive factor values as they are, in one load (WHOLE) or one by one, as far as there are any: `have`
// counts those from p on that are inside; the others are zero.
template <typename W, int N, bool WHOLE>
__device__ __forceinline__ void load_raw(const W* p, int have, uint32_t (&raw)[N * sizeof(W) / 4]) {
    constexpr int kWords = N * static_cast<int>(sizeof(W)) / 4;
#pragma unroll
    for (int j = 0; j < kWords; ++j) raw[j] = 0;
    if constexpr (WHOLE) {
        if (have > 0) {
            if constexpr (kWords == 4) {
                const uint4 t = __ldg(reinterpret_cast<const uint4*>(p));
                raw[0] = t.x; raw[1] = t.y; raw[2] = t.z; raw[3] = t.w;
            } else if constexpr (kWords == 2) {
                const uint2 t = __ldg(reinterpret_cast<const uint2*>(p));
                raw[0] = t.x; raw[1] = t.y;
            } else {
                raw[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < have) {
                if constexpr (sizeof(W) == 4) raw[j] = *reinterpret_cast<const uint32_t*>(p + j);
                else raw[j / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + j)) << (16 * (j % 2));
            }
    }
}

// The same as floats.
template <typename W, int N, bool WHOLE>
__device__ __forceinline__ void load_w(const W* p, int have, float (&w)[N]) {
    uint32_t raw[N * sizeof(W) / 4];
    load_raw<W, N, WHOLE>(p, have, raw);
    widen<W, N>(raw, w);
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t cluster_nctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

inline bool aligned_to(const void* p, uint64_t bytes) { return (reinterpret_cast<uint64_t>(p) & (bytes - 1)) == 0; }

inline int64_t item_bytes(int type) { return type == TRC_CUDA_TYPE_F32 ? 4 : 2; }

// d = base + h W^T on the tensor cores' 5th-generation path (lora_tc.cu): rows of floats that TMA can address, ranks up to
// 64. TRC_CUDA_EUNSUPPORTED, with nothing launched, where it does not apply. back: W is A^T, else B.
int up_tc(bool back, int type, const Adapters& tab, const int32_t* ids, const trc_cuda_view* base, const trc_cuda_view* d,
          int64_t rows, const float* h, int ld, cudaStream_t s);

// dA (from x and g) and dB (from dy and h) of every adapter that wants them (lora_tc.cu). vec: rows of floats in whole
// 16-byte pieces on both sides.
int grad_tc(const Adapters& tab, const int32_t* ids, const trc_cuda_view& x, const Rows& x_rows, const trc_cuda_view& dy,
            const Rows& dy_rows, bool vec, int64_t rows, const float* g, const float* h, int ld, int accumulate, cudaStream_t s);

}  // namespace lora
}  // namespace trc
