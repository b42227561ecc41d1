// lora.cu -- low-rank adapters of many requests beside a shared projection, forward and backward.
//
//   h[t]  = scale * A x[t]             (down: K -> rank)
//   y[t]  = base[t] + B h[t]           (up: rank -> N)
//   g[t]  = scale * B^T dy[t]          (down, with B in A's place)
//   dx[t] = base[t] + A^T g[t]         (up, with A in B's place)
//   dA    = sum g[t] x[t]^T,  dB = sum dy[t] h[t]^T   (over the adapter's rows)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "trc_internal.h"
#include "trc_ptx.cuh"

namespace trc {

namespace {

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
    int32_t flat;  // rows are nb1 apart throughout
    __device__ __forceinline__ char* row(int64_t t) const {
        if (flat) return data + t * nb1;
        const int64_t i1 = t % n1, r = t / n1;
        return data + i1 * nb1 + (r % n2) * nb2 + (r / n2) * nb3;
    }
};

__device__ __forceinline__ int adapter_of(const int32_t* ids, int64_t t, int n) {
    const int id = ids == nullptr ? 0 : ids[t];
    return id >= 0 && id < n ? id : -1;
}

// ------------------------------------------------------------------ tensor-core pieces
// All products run as m16n8k8 TF32 with fp32 sums. In a warp, lane = 4 * c + q (c = 0..7, q = 0..3):
//   first operand   a[0..3] = (row c, k q), (c + 8, q), (c, q + 4), (c + 8, q + 4)
//   second operand  b[0..1] = (k q, column c), (q + 4, c)
//   sums            c[0..3] = (row c, columns 2q, 2q + 1), (row c + 8, the same)
// The order of k within a sum is free, so a lane takes four consecutive values 4q .. 4q + 3 of a group of 16
// with one wide load: step s of the group (s = 0, 1) uses 4q + 2s as k = q and 4q + 2s + 1 as k = q + 4, on both
// operands.
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// x = head + tail, the head rounded to TF32's 11 bits and the tail exact; the tensor core reads the
// tail's first 11 bits, so head + tail as it sees them are within 2^-21 of x.
__device__ __forceinline__ void split(float x, uint32_t& head, uint32_t& tail) {
    head = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    tail = __float_as_uint(x - __uint_as_float(head));
}

// d += a * b in three TF32 products (two where b is a half-precision factor, whose values TF32 holds
// exactly): the small ones first.
template <bool HALF>
__device__ __forceinline__ void mma_split(float (&d)[4], const uint32_t (&ah)[4], const uint32_t (&at)[4],
                                          const uint32_t (&bh)[2], const uint32_t (&bt)[2]) {
    mma8(d, at, bh);
    if constexpr (!HALF) mma8(d, ah, bt);
    mma8(d, ah, bh);
}

template <bool HALF>
__device__ __forceinline__ void split_b(float x, uint32_t& head, uint32_t& tail) {
    if constexpr (HALF) {
        head = __float_as_uint(x);
        tail = 0;
    } else {
        split(x, head, tail);
    }
}

// Four consecutive factor values from p[i], as floats; those at lim and beyond are zero. `vec`: p and
// every i are multiples of four values.
template <typename W>
__device__ __forceinline__ void load_w4(const W* p, int64_t i, int have, bool vec, float (&w)[4]) {
    if (vec && have >= 4) {
        if constexpr (sizeof(W) == 4) {
            const float4 t = __ldg(reinterpret_cast<const float4*>(p + i));
            w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
        } else {
            const uint2 t = __ldg(reinterpret_cast<const uint2*>(p + i));
            const W* e = reinterpret_cast<const W*>(&t);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = static_cast<float>(e[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = j < have ? static_cast<float>(p[i + j]) : 0.0f;
    }
}

// Two consecutive factor values.
template <typename W>
__device__ __forceinline__ void load_w2(const W* p, int64_t i, int have, bool vec, float (&w)[2]) {
    if (vec && have >= 2) {
        if constexpr (sizeof(W) == 4) {
            const float2 t = __ldg(reinterpret_cast<const float2*>(p + i));
            w[0] = t.x; w[1] = t.y;
        } else {
            const uint32_t t = __ldg(reinterpret_cast<const uint32_t*>(p + i));
            const W* e = reinterpret_cast<const W*>(&t);
            w[0] = static_cast<float>(e[0]);
            w[1] = static_cast<float>(e[1]);
        }
    } else {
        w[0] = have > 0 ? static_cast<float>(p[i]) : 0.0f;
        w[1] = have > 1 ? static_cast<float>(p[i + 1]) : 0.0f;
    }
}

// Four consecutive activations of a row from column k on; those at k_len and beyond, and a row that is
// null, are zero. VEC: the view's elements are side by side and every row starts at a multiple of 16 bytes.
template <bool VEC>
__device__ __forceinline__ void load_x4(const char* row, int64_t nb0, int k, int k_len, float (&x)[4]) {
    if (VEC && row != nullptr && k + 4 <= k_len) {
        const float4 t = *reinterpret_cast<const float4*>(row + 4ll * k);
        x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            x[j] = row != nullptr && k + j < k_len ? *reinterpret_cast<const float*>(row + (k + j) * nb0) : 0.0f;
    }
}

// The adapters of a tile of up to 32 rows: lane l holds row l's adapter (or -1).
struct TileIds {
    int      id;       // this lane's row
    uint32_t same;     // rows with the same adapter
    uint32_t leaders;  // the first row of every adapter
    __device__ __forceinline__ TileIds(const int32_t* ids, int64_t row0, int tile, int64_t rows, int n) {
        const int     lane = threadIdx.x & 31;
        const int64_t t    = row0 + lane;
        id      = lane < tile && t < rows ? adapter_of(ids, t, n) : -1;
        same    = __match_any_sync(0xFFFFFFFFu, id);
        leaders = __ballot_sync(0xFFFFFFFFu, id >= 0 && __ffs(same) - 1 == lane);
    }
};

__device__ __forceinline__ void grid_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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

constexpr int kWarps = 8, kThreads = 256;

// ------------------------------------------------------------------ down: h = scale * x W^T
// One cluster per tile of 16 * MT rows and slice of the tile's adapters: each CTA takes its share of
// the columns of x in steps of 32 (one line of every row), each warp every 8th of those; the partial sums
// meet in shared memory and then across the cluster, always in the same order. BACK: x is dy and W is
// B^T, whose values for one rank are `rank` apart: a lane loads V ranks of one column at once and tile i of a
// group of V takes rank V * c + i.
template <typename W, bool BACK, int NT, int MT, bool VEC>
__global__ void __launch_bounds__(kThreads) down_kernel(const __grid_constant__ Adapters tab, const int32_t* ids, Rows x,
                                                        int64_t rows, int k_len, float* h, int ld) {
    constexpr bool HALF = sizeof(W) == 2;
    constexpr int  V = NT < 4 ? NT : 4, kRows = 16 * MT, kCols = 8 * NT;
    extern __shared__ float red[];  // [kWarps][kRows][kCols]
    const int     warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane >> 2, q = lane & 3;
    const int     ranks = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / ranks) * kRows;
    const TileIds tile(ids, row0, kRows, rows, tab.n);
    grid_dependents();

    if (blockIdx.y == 0 && rank == 0) {  // rows without an adapter
        for (int r = warp; r < kRows; r += kWarps) {
            if (row0 + r < rows && __shfl_sync(0xFFFFFFFFu, tile.id, r) < 0)
                for (int j = lane; j < ld; j += 32) h[(row0 + r) * ld + j] = 0.0f;
        }
    }
    int turn = 0;
    for (uint32_t left = tile.leaders; left != 0; left &= left - 1) {
        if (turn++ % gridDim.y != blockIdx.y) continue;
        const int      lead = __ffs(left) - 1;
        const int      id = __shfl_sync(0xFFFFFFFFu, tile.id, lead);
        const uint32_t mine = __shfl_sync(0xFFFFFFFFu, tile.same, lead);
        const Adapter& A = tab.ad[id];
        const int      r = A.rank;
        const W*       w = static_cast<const W*>(BACK ? A.b : A.a);
        const bool     vec = (A.vec & (BACK ? 2 : 1)) != 0;
        const char*    xr[2 * MT];  // rows c, c + 8, c + 16, c + 24
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) xr[i] = (mine >> (c + 8 * i)) & 1u ? x.row(row0 + c + 8 * i) : nullptr;
        for (int j0 = 0; j0 < r; j0 += kCols) {
            float acc[MT][NT][4] = {};
            for (int k0 = 32 * (rank * kWarps + warp); k0 < k_len; k0 += 32 * kWarps * ranks) {
                float xv[2][2 * MT][4];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 2 * MT; ++i) load_x4<VEC>(xr[i], x.nb0, k0 + 16 * s + 4 * q, k_len, xv[s][i]);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int kg = k0 + 16 * s + 4 * q;
                    float wv[NT][4];
                    if constexpr (!BACK) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const int j = j0 + 8 * n + c;
                            load_w4(w, static_cast<int64_t>(j) * k_len + kg, j < r ? k_len - kg : 0, vec, wv[n]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int n = 0; n < NT; n += V) {
                                const int j = j0 + 8 * n + V * c;
                                const int have = kg + e < k_len ? r - j : 0;
                                float t[V];
                                if constexpr (V == 4) load_w4(w, static_cast<int64_t>(kg + e) * r + j, have, vec, t);
                                else load_w2(w, static_cast<int64_t>(kg + e) * r + j, have, vec, t);
#pragma unroll
                                for (int i = 0; i < V; ++i) wv[n + i][e] = t[i];
                            }
                    }
                    uint32_t ah[2][MT][4], at[2][MT][4];
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int e = 0; e < 4; ++e)  // a[e]: row c + 8 (e & 1), value 2u + (e >> 1)
                                split(xv[s][2 * m + (e & 1)][2 * u + (e >> 1)], ah[u][m][e], at[u][m][e]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (j0 + 8 * (BACK ? n / V * V : n) >= r) continue;  // the same for the whole warp
                        uint32_t bh[2][2], bt[2][2];
#pragma unroll
                        for (int e = 0; e < 4; ++e) split_b<HALF>(wv[n][e], bh[e >> 1][e & 1], bt[e >> 1][e & 1]);
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            // the tensor core's own sums lose a little at every step: 16 columns at a time
                            float d[4] = {};
                            mma_split<HALF>(d, ah[0][m], at[0][m], bh[0], bt[0]);
                            mma_split<HALF>(d, ah[1][m], at[1][m], bh[1], bt[1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[m][n][e] += d[e];
                        }
                    }
                }
            }
            // partial sums of the 8 warps, then of the cluster
            float* mywarp = red + warp * kRows * kCols;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int col = 2 * q + (e & 1);
                        const int j = BACK ? 8 * (n / V * V) + V * col + n % V : 8 * n + col;
                        mywarp[(16 * m + c + 8 * (e >> 1)) * kCols + j] = acc[m][n][e];
                    }
            __syncthreads();
            for (int i = threadIdx.x; i < kRows * kCols; i += kThreads) {
                float s = red[i];
#pragma unroll
                for (int v = 1; v < kWarps; ++v) s += red[v * kRows * kCols + i];
                red[i] = s;  // only this thread reads or writes column i
            }
            if (ranks > 1) cluster_sync();
            else __syncthreads();
            for (int i = rank * kThreads + threadIdx.x; i < kRows * kCols; i += kThreads * ranks) {
                const int t = i / kCols, j = j0 + i % kCols;
                if (!((mine >> t) & 1u) || j >= ld) continue;
                float s = 0.0f;
                if (ranks > 1) {
                    for (int v = 0; v < ranks; ++v) s += ld_cluster(mapa_shared(red + i, v));
                } else {
                    s = red[i];
                }
                h[(row0 + t) * ld + j] = j < r ? s * A.scale : 0.0f;
            }
            if (ranks > 1) cluster_sync();
            else __syncthreads();
        }
        // whole chunks of ranks that the adapter does not have
        for (int j0 = (r + kCols - 1) / kCols * kCols; j0 < ld; j0 += kCols) {
            for (int i = rank * kThreads + threadIdx.x; i < kRows * kCols; i += kThreads * ranks)
                if (((mine >> (i / kCols)) & 1u) && j0 + i % kCols < ld) h[(row0 + i / kCols) * ld + j0 + i % kCols] = 0.0f;
        }
    }
}

// ------------------------------------------------------------------ up: d = base + h W^T
// A warp takes 16 * MT rows and walks over groups of 16 columns; wr warps of a CTA stand side by side in the
// rows (the factor's values then come from L1 for all but one), the others in the columns. The two 8-column
// tiles of a group take columns 4 (c >> 1) + 2 i + (c & 1), i = 0, 1, so that a lane ends up with four
// consecutive columns of a row: 16-byte loads of base and stores of d. Every row has one adapter at most,
// so the adapters of a tile (and the slices of the grid that share them) write rows of their own.
template <typename W, bool BACK, int JG, int MT, bool VEC>
__global__ void __launch_bounds__(kThreads) up_kernel(const __grid_constant__ Adapters tab, const int32_t* ids, Rows base, Rows d,
                                                      int64_t rows, int n_len, const float* h, int ld, int wr, int iters, int col_blocks) {
    constexpr bool HALF = sizeof(W) == 2;
    constexpr int  kRows = 16 * MT;
    const int     warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane >> 2, q = lane & 3;
    const int     wn = kWarps / wr;
    const int64_t row0 = (static_cast<int64_t>(blockIdx.x / col_blocks) * wr + warp % wr) * kRows;
    const int     group0 = static_cast<int>(blockIdx.x % col_blocks) * wn * iters + warp / wr, groups = (n_len + 15) / 16;
    const TileIds tile(ids, row0, kRows, rows, tab.n);
    grid_wait();  // h is written
    if (row0 >= rows) return;

    float hv[JG][2 * MT][4];  // the first 16 * JG ranks of rows c, c + 8, ...: values 4q .. 4q + 3 of each 16
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        const bool live = row0 + c + 8 * i < rows;
#pragma unroll
        for (int g = 0; g < JG; ++g) {
            float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (live && 16 * g < ld) t = *reinterpret_cast<const float4*>(h + (row0 + c + 8 * i) * ld + 16 * g + 4 * q);
            hv[g][i][0] = t.x; hv[g][i][1] = t.y; hv[g][i][2] = t.z; hv[g][i][3] = t.w;
        }
    }
    for (int it = 0; it < iters; ++it) {
        const int group = group0 + it * wn;
        if (group >= groups) break;
        const int n0 = 16 * group;
        float y[2 * MT][4];  // columns n0 + 4q .. + 3 of rows c + 8 i
        bool  keep[2 * MT];  // rows that this slice writes
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            const int64_t t = row0 + c + 8 * i;
            const int     id = __shfl_sync(0xFFFFFFFFu, tile.id, c + 8 * i);
            const uint32_t same = __shfl_sync(0xFFFFFFFFu, tile.same, c + 8 * i);
            // the turn of the row's adapter among the tile's; rows without one go with the first slice
            const uint32_t turn = id >= 0 ? __popc(tile.leaders & ((same & (~same + 1u)) - 1u)) % gridDim.z : 0u;
            keep[i] = t < rows && turn == blockIdx.z;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[i][e] = 0.0f;
            if (keep[i] && base.data != nullptr) load_x4<VEC>(base.row(t), base.nb0, n0 + 4 * q, n_len, y[i]);
        }
        int turn = 0;
        for (uint32_t left = tile.leaders; left != 0; left &= left - 1) {
            if (turn++ % gridDim.z != blockIdx.z) continue;
            const int      lead = __ffs(left) - 1;
            const int      id = __shfl_sync(0xFFFFFFFFu, tile.id, lead);
            const uint32_t mine = __shfl_sync(0xFFFFFFFFu, tile.same, lead);
            const Adapter& A = tab.ad[id];
            const int      r = A.rank;
            const W*       w = static_cast<const W*>(BACK ? A.a : A.b);
            const bool     vec = (A.vec & (BACK ? 1 : 2)) != 0;
            float acc[MT][2][4] = {};
            for (int j0 = 0; j0 < r; j0 += 16 * JG) {
                float hj[JG][2 * MT][4];
#pragma unroll
                for (int g = 0; g < JG; ++g)
#pragma unroll
                    for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) hj[g][i][e] = hv[g][i][e];
                if (j0 > 0) {  // ranks beyond 16 * JG: from memory for each group of columns
#pragma unroll
                    for (int g = 0; g < JG; ++g)
#pragma unroll
                        for (int i = 0; i < 2 * MT; ++i) {
                            float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (row0 + c + 8 * i < rows && j0 + 16 * g < ld)
                                t = *reinterpret_cast<const float4*>(h + (row0 + c + 8 * i) * ld + j0 + 16 * g + 4 * q);
                            hj[g][i][0] = t.x; hj[g][i][1] = t.y; hj[g][i][2] = t.z; hj[g][i][3] = t.w;
                        }
                }
#pragma unroll
                for (int g = 0; g < JG; ++g) {
                    if (j0 + 16 * g >= r) continue;
                    const int jq = j0 + 16 * g + 4 * q;
                    float wv[2][4];  // tile i, ranks jq .. jq + 3
                    if constexpr (!BACK) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int n = n0 + 4 * (c >> 1) + 2 * i + (c & 1);
                            load_w4(w, static_cast<int64_t>(n) * r + jq, n < n_len ? r - jq : 0, vec, wv[i]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int n = n0 + 4 * (c >> 1);
                            float t[4];
                            load_w4(w, static_cast<int64_t>(jq + e) * n_len + n, jq + e < r ? n_len - n : 0, vec, t);
                            wv[0][e] = c & 1 ? t[1] : t[0];
                            wv[1][e] = c & 1 ? t[3] : t[2];
                        }
                    }
                    uint32_t bh[2][2][2], bt[2][2][2];  // [step][tile]
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) split_b<HALF>(wv[i][e], bh[e >> 1][i][e & 1], bt[e >> 1][i][e & 1]);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        uint32_t ah[2][4], at[2][4];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                split(hj[g][2 * m + (e & 1)][2 * u + (e >> 1)], ah[u][e], at[u][e]);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float t[4] = {};
                            mma_split<HALF>(t, ah[0], at[0], bh[0][i], bt[0][i]);
                            mma_split<HALF>(t, ah[1], at[1], bh[1][i], bt[1][i]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[m][i][e] += t[e];
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i)  // row c + 8 i: sums 2 (i & 1) .. of tile 0, then of tile 1
                if ((mine >> (c + 8 * i)) & 1u) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[i][e] += acc[i >> 1][e >> 1][2 * (i & 1) + (e & 1)];
                }
        }
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            if (!keep[i]) continue;
            char* out = d.row(row0 + c + 8 * i);
            const int n = n0 + 4 * q;
            if (VEC && n + 4 <= n_len) {
                *reinterpret_cast<float4*>(out + 4ll * n) = make_float4(y[i][0], y[i][1], y[i][2], y[i][3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < n_len) *reinterpret_cast<float*>(out + (n + e) * d.nb0) = y[i][e];
            }
        }
    }
}

// ------------------------------------------------------------------ gradients of the factors
// out(j, k) (+)= sum over the adapter's rows t of h[t, j] x[t, k]; dA (h = g, x) is j-major, dB (h, x = dy)
// k-major. The ranks are the 16-row side of the tensor core's tile, so a warp holds all ranks (up to 64)
// of 32 columns and x is read once, straight into registers. Four warps of a CTA stand side by side in the
// columns, two share the rows in turns of 32, and so do the CTAs of a cluster. Lane (c, q) takes the
// columns 4c .. 4c + 3 (column 4c + i in tile i) and the ranks 2 MT c .. (the two halves of the MT tiles in turn).
struct GradSide {
    Rows         x;
    const float* h;
    int32_t      k_len;
    int32_t      strips;  // of 128 columns
    int32_t      vec;
};

template <int MT>
__global__ void __launch_bounds__(kThreads) grad_kernel(const __grid_constant__ Adapters tab, const int32_t* ids,
                                                        const __grid_constant__ GradSide side_a,
                                                        const __grid_constant__ GradSide side_b, int64_t rows, int ld,
                                                        int accumulate) {
    constexpr int kR = 16 * MT;
    __shared__ float sum[kR][128 + 4];
    const int  warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane >> 2, q = lane & 3;
    const int  ranks = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
    int        strip = static_cast<int>(blockIdx.x) / ranks;
    const bool is_b = strip >= side_a.strips;
    const GradSide& S = is_b ? side_b : side_a;
    if (is_b) strip -= side_a.strips;
    const Adapter& A = tab.ad[blockIdx.z];
    float* out = is_b ? A.db : A.da;
    const int j0 = blockIdx.y * kR, r = A.rank;
    grid_wait();
    if (out == nullptr || j0 >= r) return;  // the whole cluster
    const int col = strip * 128 + (warp & 3) * 32 + 4 * c;

    float acc[MT][4][4] = {};
    const int64_t tiles = (rows + 31) / 32;
    for (int64_t i = rank + static_cast<int64_t>(warp >> 2) * ranks; i < tiles; i += 2 * ranks) {
        const int64_t  t0 = i * 32;
        const uint32_t mine = __ballot_sync(0xFFFFFFFFu, t0 + lane < rows && adapter_of(ids, t0 + lane, tab.n) == static_cast<int>(blockIdx.z));
        if (mine == 0) continue;
#pragma unroll
        for (int s = 0; s < 2; ++s) {  // 16 rows: t0 + 16 s + q + 4 e
            if (((mine >> (16 * s)) & 0xFFFFu) == 0) continue;
            float xv[4][4], hv[4][2 * MT];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int  l = 16 * s + q + 4 * e;
                const bool live = (mine >> l) & 1u;
                const char* xr = live ? S.x.row(t0 + l) : nullptr;
                if (S.vec) load_x4<true>(xr, 4, col, S.k_len, xv[e]);
                else load_x4<false>(xr, S.x.nb0, col, S.k_len, xv[e]);
                const float* hr = S.h + (t0 + l) * ld + j0 + 2 * MT * c;
#pragma unroll
                for (int j = 0; j < 2 * MT; j += 2) {
                    float2 t = make_float2(0.0f, 0.0f);
                    if (live && j0 + 2 * MT * c + j < ld) t = *reinterpret_cast<const float2*>(hr + j);
                    hv[e][j] = t.x;
                    hv[e][j + 1] = t.y;
                }
            }
            uint32_t bh[2][4][2], bt[2][4][2];  // [8 rows][tile]
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int n = 0; n < 4; ++n) split(xv[e][n], bh[e >> 1][n][e & 1], bt[e >> 1][n][e & 1]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                uint32_t ah[2][4], at[2][4];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e)  // a[e]: half e & 1, row q + 4 (e >> 1) of the 8
                        split(hv[2 * u + (e >> 1)][2 * m + (e & 1)], ah[u][e], at[u][e]);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    float d[4] = {};
                    mma_split<false>(d, ah[0], at[0], bh[0][n], bt[0][n]);
                    mma_split<false>(d, ah[1], at[1], bh[1][n], bt[1][n]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[m][n][e] += d[e];
                }
            }
        }
    }
    // the two row halves of the CTA, then the cluster
    const int col0 = (warp & 3) * 32;
#pragma unroll
    for (int half = 1; half >= 0; --half) {
        if ((warp >> 2) == half) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float* s = &sum[2 * MT * c + 2 * m + (e >> 1)][col0 + 4 * (2 * q + (e & 1)) + n];
                        *s = half == 1 ? acc[m][n][e] : *s + acc[m][n][e];
                    }
        }
        __syncthreads();
    }
    if (ranks > 1) cluster_sync();
    for (int i = rank * kThreads + threadIdx.x; i < kR * 128; i += kThreads * ranks) {
        // neighbours in memory are neighbours in the lanes
        const int j = is_b ? i % kR : i / 128, k = is_b ? i / kR : i % 128;
        if (j0 + j >= r || strip * 128 + k >= S.k_len) continue;
        float s = 0.0f;
        if (ranks > 1) {
            for (int v = 0; v < ranks; ++v) s += ld_cluster(mapa_shared(&sum[j][k], v));
        } else {
            s = sum[j][k];
        }
        const int64_t kk = strip * 128 + k;
        float* o = out + (is_b ? kk * r + j0 + j : static_cast<int64_t>(j0 + j) * S.k_len + kk);
        *o = accumulate ? *o + s : s;
    }
    if (ranks > 1) cluster_sync();
}

constexpr int64_t kMaxLen = int64_t(1) << 30;  // rows, K and N of a call

bool aligned_to(const void* p, uint64_t bytes) { return (reinterpret_cast<uint64_t>(p) & (bytes - 1)) == 0; }

int64_t item_bytes(int type) { return type == TRC_CUDA_TYPE_F32 ? 4 : 2; }

// TRC_CUDA_OK if the adapters are valid for trc_cuda_lora*; *ld = the row length of h.
int check_adapters(const trc_cuda_lora_adapter* ad, int n, int64_t item, int64_t* ld) {
    if (n < 0 || (n > 0 && ad == nullptr)) return TRC_CUDA_EINVAL;
    if (n > TRC_CUDA_LORA_MAX_ADAPTERS) return TRC_CUDA_EUNSUPPORTED;
    int rank = 1;
    for (int i = 0; i < n; ++i) {
        if (ad[i].rank < 1 || ad[i].a == nullptr || ad[i].b == nullptr) return TRC_CUDA_EINVAL;
        if (ad[i].rank > TRC_CUDA_LORA_MAX_RANK) return TRC_CUDA_EUNSUPPORTED;
        if (!aligned_to(ad[i].a, item) || !aligned_to(ad[i].b, item) || !aligned_to(ad[i].da, 4) || !aligned_to(ad[i].db, 4))
            return TRC_CUDA_EINVAL;
        rank = std::max(rank, ad[i].rank);
    }
    *ld = (rank + 15) / 16 * 16;
    return TRC_CUDA_OK;
}

// A view of rows: extents in range, floats at multiples of 4 bytes.
int check_rows(const trc_cuda_view* v) {
    if (!view_ok(v) || !aligned_to(v->data, 4)) return TRC_CUDA_EINVAL;
    if (v->ne[0] < 1) return TRC_CUDA_EINVAL;
    for (int i = 0; i < 4; ++i) {
        if ((v->nb[i] & 3) != 0) return TRC_CUDA_EINVAL;
        if (v->ne[i] > kMaxLen) return TRC_CUDA_EUNSUPPORTED;
    }
    const int64_t r = v->ne[1] * v->ne[2];  // each factor at most 2^30
    if (r > kMaxLen || r * v->ne[3] > kMaxLen) return TRC_CUDA_EUNSUPPORTED;
    return TRC_CUDA_OK;
}

// A view that is written: no two of its elements may be the same by a stride of zero.
bool writable(const trc_cuda_view& v) {
    for (int i = 0; i < 4; ++i)
        if (v.ne[i] > 1 && v.nb[i] == 0) return false;
    return true;
}

bool same_rows(const trc_cuda_view& a, const trc_cuda_view& b) {
    return a.ne[1] == b.ne[1] && a.ne[2] == b.ne[2] && a.ne[3] == b.ne[3];
}

Rows rows_of(const trc_cuda_view* v) {
    Rows r{};
    if (v == nullptr) return r;
    r.data = static_cast<char*>(v->data);
    r.nb0 = v->nb[0];
    r.nb1 = v->nb[1];
    r.nb2 = v->nb[2];
    r.nb3 = v->nb[3];
    r.n1 = static_cast<int32_t>(v->ne[1]);
    r.n2 = static_cast<int32_t>(v->ne[2]);
    // one stride for all rows, whichever extents are 1
    int64_t step = 0, want = 0, count = 1;
    r.flat = 1;
    for (int i = 1; i < 4; ++i) {
        if (v->ne[i] == 1) continue;
        if (count == 1) step = v->nb[i];
        else if (v->nb[i] != want) r.flat = 0;
        count *= v->ne[i];
        want = step * count;
    }
    if (r.flat) r.nb1 = step;
    return r;
}

// K: the row length of A.
void make_table(Adapters& t, const trc_cuda_lora_adapter* ad, int n, int type, int64_t k) {
    t.n = n;
    const uint64_t four = 4 * item_bytes(type);
    for (int i = 0; i < n; ++i) {
        const int vec = (k % 4 == 0 && aligned_to(ad[i].a, four) ? 1 : 0) | (ad[i].rank % 4 == 0 && aligned_to(ad[i].b, four) ? 2 : 0);
        t.ad[i] = Adapter{ad[i].a, ad[i].b, ad[i].da, ad[i].db, ad[i].scale, static_cast<int16_t>(ad[i].rank),
                          static_cast<int16_t>(vec)};
    }
}

// Rows of floats side by side that start at multiples of 16 bytes.
bool vec_rows(const trc_cuda_view* v) {
    if (v == nullptr) return true;
    if (!aligned_to(v->data, 16) || (v->ne[0] > 1 && v->nb[0] != 4)) return false;
    for (int i = 1; i < 4; ++i)
        if (v->ne[i] > 1 && (v->nb[i] & 15) != 0) return false;
    return true;
}

int launch(const void* kernel, dim3 grid, unsigned cluster, size_t smem, bool after, void** args, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    unsigned n = 0;
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
    if (after) {  // may be set up while the kernel before it drains; it waits for that kernel's results itself
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, args);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return cuda_fail(e);
    }
    note_launch();
    return TRC_CUDA_OK;
}

// A power of two up to `most` that brings `count` units to about `want`.
int power_for(int64_t count, int64_t want, int most) {
    int p = 1;
    while (p < most && count * p < want) p *= 2;
    return p;
}

// CTAs that a launch aims at: two for each SM.
int64_t full_grid() { return 2 * static_cast<int64_t>(std::max(1, sm_count_current())); }

template <typename W, bool BACK, int NT, int MT>
int run_down(const Adapters& tab, const int32_t* ids, const Rows& x, bool vec, int64_t rows, int k, float* h, int ld,
             cudaStream_t s) {
    const int64_t tiles = (rows + 16 * MT - 1) / (16 * MT);
    // the columns of one tile go to 1 - 8 CTAs while each of their warps keeps a step of 32
    const int cluster = std::min(power_for(tiles, full_grid(), 8), power_for(1, (k + 255) / 256, 8));
    const int64_t most = std::min<int64_t>({tab.n, 16 * MT, rows});
    const int64_t slices = std::max<int64_t>(1, std::min(most, full_grid() / (tiles * cluster)));
    const size_t smem = sizeof(float) * kWarps * 16 * MT * 8 * NT;
    const void* kernel = vec ? reinterpret_cast<const void*>(&down_kernel<W, BACK, NT, MT, true>)
                             : reinterpret_cast<const void*>(&down_kernel<W, BACK, NT, MT, false>);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return cuda_fail(e);
    }
    void* args[] = {const_cast<Adapters*>(&tab), &ids, const_cast<Rows*>(&x), &rows, &k, &h, &ld};
    return launch(kernel, dim3(static_cast<unsigned>(tiles * cluster), static_cast<unsigned>(slices)), cluster, smem, false, args, s);
}

template <bool BACK, typename W>
int down_of(const Adapters& tab, const int32_t* ids, const Rows& x, bool vec, int64_t rows, int k, float* h, int ld,
            cudaStream_t s) {
    if (rows <= 16) {
        if (ld == 16) return run_down<W, BACK, 2, 1>(tab, ids, x, vec, rows, k, h, ld, s);
        if (ld == 32) return run_down<W, BACK, 4, 1>(tab, ids, x, vec, rows, k, h, ld, s);
        return run_down<W, BACK, 8, 1>(tab, ids, x, vec, rows, k, h, ld, s);
    }
    if (ld == 16) return run_down<W, BACK, 2, 2>(tab, ids, x, vec, rows, k, h, ld, s);
    if (ld == 32) return run_down<W, BACK, 4, 2>(tab, ids, x, vec, rows, k, h, ld, s);
    return run_down<W, BACK, 8, 2>(tab, ids, x, vec, rows, k, h, ld, s);
}

template <typename W, bool BACK, int JG, int MT>
int run_up(const Adapters& tab, const int32_t* ids, const Rows& base, const Rows& d, bool vec, int64_t rows, int n,
           const float* h, int ld, cudaStream_t s) {
    const int64_t tiles = (rows + 16 * MT - 1) / (16 * MT), groups = (n + 15) / 16;
    int wr = power_for(1, tiles, 4);  // warps side by side in the rows
    const int64_t row_blocks = (tiles + wr - 1) / wr;
    int iters = 8;
    while (iters > 1 && row_blocks * (groups / (iters * (kWarps / wr))) < 2 * full_grid()) iters /= 2;
    const int64_t col_blocks = (groups + iters * (kWarps / wr) - 1) / (iters * (kWarps / wr));
    const int64_t most = std::min<int64_t>({tab.n, 16 * MT, rows});
    const int64_t slices = std::max<int64_t>(1, std::min(most, 2 * full_grid() / (row_blocks * col_blocks)));
    const void* kernel = vec ? reinterpret_cast<const void*>(&up_kernel<W, BACK, JG, MT, true>)
                             : reinterpret_cast<const void*>(&up_kernel<W, BACK, JG, MT, false>);
    if (row_blocks * col_blocks > INT32_MAX) return TRC_CUDA_EUNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(row_blocks * col_blocks), 1, static_cast<unsigned>(slices));
    int cols = static_cast<int>(col_blocks);
    void* args[] = {const_cast<Adapters*>(&tab), &ids, const_cast<Rows*>(&base), const_cast<Rows*>(&d), &rows, &n, &h, &ld, &wr,
                    &iters, &cols};
    return launch(kernel, grid, 1, 0, true, args, s);
}

template <bool BACK, typename W>
int up_of(const Adapters& tab, const int32_t* ids, const Rows& base, const Rows& d, bool vec, int64_t rows, int n,
          const float* h, int ld, cudaStream_t s) {
    if (rows <= 16) {
        if (ld == 16) return run_up<W, BACK, 1, 1>(tab, ids, base, d, vec, rows, n, h, ld, s);
        if (ld == 32) return run_up<W, BACK, 2, 1>(tab, ids, base, d, vec, rows, n, h, ld, s);
        return run_up<W, BACK, 4, 1>(tab, ids, base, d, vec, rows, n, h, ld, s);
    }
    if (ld == 16) return run_up<W, BACK, 1, 2>(tab, ids, base, d, vec, rows, n, h, ld, s);
    if (ld == 32) return run_up<W, BACK, 2, 2>(tab, ids, base, d, vec, rows, n, h, ld, s);
    return run_up<W, BACK, 4, 2>(tab, ids, base, d, vec, rows, n, h, ld, s);
}

template <bool BACK>
int down(int type, const Adapters& tab, const int32_t* ids, const trc_cuda_view* x, int64_t rows, float* h, int ld, cudaStream_t s) {
    const Rows r = rows_of(x);
    const int k = static_cast<int>(x->ne[0]);
    const bool vec = vec_rows(x);
    if (type == TRC_CUDA_TYPE_F32) return down_of<BACK, float>(tab, ids, r, vec, rows, k, h, ld, s);
    if (type == TRC_CUDA_TYPE_F16) return down_of<BACK, __half>(tab, ids, r, vec, rows, k, h, ld, s);
    return down_of<BACK, __nv_bfloat16>(tab, ids, r, vec, rows, k, h, ld, s);
}

template <bool BACK>
int up(int type, const Adapters& tab, const int32_t* ids, const trc_cuda_view* base, const trc_cuda_view* d, int64_t rows,
       const float* h, int ld, cudaStream_t s) {
    const Rows rb = rows_of(base), rd = rows_of(d);
    const int n = static_cast<int>(d->ne[0]);
    const bool vec = vec_rows(base) && vec_rows(d);
    if (type == TRC_CUDA_TYPE_F32) return up_of<BACK, float>(tab, ids, rb, rd, vec, rows, n, h, ld, s);
    if (type == TRC_CUDA_TYPE_F16) return up_of<BACK, __half>(tab, ids, rb, rd, vec, rows, n, h, ld, s);
    return up_of<BACK, __nv_bfloat16>(tab, ids, rb, rd, vec, rows, n, h, ld, s);
}

// Both factors' gradients; the kernel before it on the stream has to be down's.
int grad(const Adapters& tab, const int32_t* ids, const trc_cuda_view* x, const trc_cuda_view* dy, int64_t rows, const float* g,
         const float* h, int ld, int accumulate, cudaStream_t s) {
    bool any_a = false, any_b = false;
    for (int i = 0; i < tab.n; ++i) {
        any_a = any_a || tab.ad[i].da != nullptr;
        any_b = any_b || tab.ad[i].db != nullptr;
    }
    if (!any_a && !any_b) return TRC_CUDA_OK;
    GradSide a{rows_of(x), g, static_cast<int32_t>(x->ne[0]), 0, vec_rows(x)};
    GradSide b{rows_of(dy), h, static_cast<int32_t>(dy->ne[0]), 0, vec_rows(dy)};
    if (any_a) a.strips = (a.k_len + 127) / 128;
    if (any_b) b.strips = (b.k_len + 127) / 128;
    const int mt = std::min(ld / 16, 3) == 3 ? 4 : ld / 16;
    const unsigned chunks = static_cast<unsigned>((ld + 16 * mt - 1) / (16 * mt));
    const int64_t strips = a.strips + b.strips;
    const int cluster = std::min(power_for(strips * tab.n * chunks, full_grid(), 8), power_for(1, (rows + 63) / 64, 8));
    const void* kernel = mt == 1   ? reinterpret_cast<const void*>(&grad_kernel<1>)
                         : mt == 2 ? reinterpret_cast<const void*>(&grad_kernel<2>)
                                   : reinterpret_cast<const void*>(&grad_kernel<4>);
    void* args[] = {const_cast<Adapters*>(&tab), &ids, &a, &b, &rows, &ld, &accumulate};
    return launch(kernel, dim3(static_cast<unsigned>(strips * cluster), chunks, static_cast<unsigned>(tab.n)), cluster, 0,
                  false, args, s);
}

}  // namespace

}  // namespace trc

using namespace trc;

extern "C" {

int64_t trc_cuda_lora_h_ld(const trc_cuda_lora_adapter* adapters, int n_adapters) {
    int64_t ld = 0;
    const int st = check_adapters(adapters, n_adapters, 1, &ld);
    return st == TRC_CUDA_OK ? ld : st;
}

int trc_cuda_lora(int type, const trc_cuda_lora_adapter* adapters, int n_adapters, const int32_t* ids,
                  const trc_cuda_view* x, const trc_cuda_view* base, const trc_cuda_view* d, float* h, void* stream) {
    if (type != TRC_CUDA_TYPE_F32 && type != TRC_CUDA_TYPE_F16 && type != TRC_CUDA_TYPE_BF16) return TRC_CUDA_EUNSUPPORTED;
    int64_t ld = 0;
    int st = check_adapters(adapters, n_adapters, item_bytes(type), &ld);
    if (st != TRC_CUDA_OK) return st;
    if ((st = check_rows(x)) != TRC_CUDA_OK || (st = check_rows(d)) != TRC_CUDA_OK) return st;
    if (base != nullptr && (st = check_rows(base)) != TRC_CUDA_OK) return st;
    if (!same_rows(*x, *d) || !writable(*d)) return TRC_CUDA_EINVAL;
    if (base != nullptr && (base->ne[0] != d->ne[0] || !same_rows(*base, *d))) return TRC_CUDA_EINVAL;
    if (!aligned_to(ids, 4)) return TRC_CUDA_EINVAL;
    const int64_t rows = d->ne[1] * d->ne[2] * d->ne[3];
    if (rows == 0) return TRC_CUDA_OK;
    if (h == nullptr || !aligned_to(h, 16)) return TRC_CUDA_EINVAL;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Adapters tab;
    make_table(tab, adapters, n_adapters, type, x->ne[0]);
    st = down<false>(type, tab, ids, x, rows, h, static_cast<int>(ld), s);
    if (st != TRC_CUDA_OK) return st;
    return up<false>(type, tab, ids, base, d, rows, h, static_cast<int>(ld), s);
}

size_t trc_cuda_lora_back_workspace_bytes(const trc_cuda_lora_adapter* adapters, int n_adapters, int64_t rows) {
    int64_t ld = 0;
    if (rows < 0 || rows > kMaxLen || check_adapters(adapters, n_adapters, 1, &ld) != TRC_CUDA_OK) return 0;
    return static_cast<size_t>(std::max<int64_t>(rows, 1) * ld) * sizeof(float);  // g
}

int trc_cuda_lora_back(int type, const trc_cuda_lora_adapter* adapters, int n_adapters, const int32_t* ids,
                       const trc_cuda_view* x, const trc_cuda_view* dy, const float* h, const trc_cuda_view* base,
                       const trc_cuda_view* dx, void* workspace, size_t workspace_bytes, uint32_t flags,
                       void* stream) {
    if (type != TRC_CUDA_TYPE_F32 && type != TRC_CUDA_TYPE_F16 && type != TRC_CUDA_TYPE_BF16) return TRC_CUDA_EUNSUPPORTED;
    if ((flags & ~TRC_CUDA_MM_ACCUMULATE) != 0) return TRC_CUDA_EUNSUPPORTED;
    int64_t ld = 0;
    int st = check_adapters(adapters, n_adapters, item_bytes(type), &ld);
    if (st != TRC_CUDA_OK) return st;
    if ((st = check_rows(x)) != TRC_CUDA_OK || (st = check_rows(dy)) != TRC_CUDA_OK) return st;
    if (!same_rows(*x, *dy)) return TRC_CUDA_EINVAL;
    if (dx != nullptr) {
        if ((st = check_rows(dx)) != TRC_CUDA_OK) return st;
        if (dx->ne[0] != x->ne[0] || !same_rows(*dx, *x) || !writable(*dx)) return TRC_CUDA_EINVAL;
    }
    if (base != nullptr) {
        if (dx == nullptr) return TRC_CUDA_EINVAL;
        if ((st = check_rows(base)) != TRC_CUDA_OK) return st;
        if (base->ne[0] != dx->ne[0] || !same_rows(*base, *dx)) return TRC_CUDA_EINVAL;
    }
    if (!aligned_to(ids, 4)) return TRC_CUDA_EINVAL;
    const int64_t rows = x->ne[1] * x->ne[2] * x->ne[3];
    if (rows > 0 && (h == nullptr || !aligned_to(h, 16))) return TRC_CUDA_EINVAL;
    if (workspace == nullptr || !aligned_to(workspace, 16) ||
        workspace_bytes < trc_cuda_lora_back_workspace_bytes(adapters, n_adapters, rows))
        return TRC_CUDA_EINVAL;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Adapters tab;
    make_table(tab, adapters, n_adapters, type, x->ne[0]);
    const int accumulate = (flags & TRC_CUDA_MM_ACCUMULATE) != 0 ? 1 : 0, l = static_cast<int>(ld);
    float* g = static_cast<float*>(workspace);
    if (rows > 0) {
        if ((st = down<true>(type, tab, ids, dy, rows, g, l, s)) != TRC_CUDA_OK) return st;
        if (dx != nullptr && (st = up<true>(type, tab, ids, base, dx, rows, g, l, s)) != TRC_CUDA_OK) return st;
    }
    return grad(tab, ids, x, dy, rows, g, h, l, accumulate, s);
}

}  // extern "C"
