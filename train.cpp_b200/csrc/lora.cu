// lora.cu -- low-rank adapters of many requests beside a shared projection, forward and backward.
//
//   h[t]  = scale * A x[t]             (down: K -> rank)
//   y[t]  = base[t] + B h[t]           (up: rank -> N)
//   g[t]  = scale * B^T dy[t]          (down, with B in A's place)
//   dx[t] = base[t] + A^T g[t]         (up, with A in B's place)
//   dA    = sum g[t] x[t]^T,  dB = sum dy[t] h[t]^T   (over the adapter's rows)
//
// F32 accuracy: every product is three TF32 products of heads and tails (two with a half-precision factor), sums leave the
// tensor core for fp32 every 16 - 64 terms. The whole is bound by memory up to rank 16 (4 K + 8 N bytes and 2 r (K + N)
// flops for each row); at rank 64 the narrow product, on mma.sync, is bound by that pipe (278 TFLOP/s of TF32 measured, 93 of
// split products).
// Which kernel runs: decode batches the one-launch form (few); else down, then up. up and the gradients run on tcgen05
// (lora_tc.cu), up from 128 rows on with rows that TMA can address and ranks up to 64, else on the kernel here. down stays on
// mma.sync: the same scheme on tcgen05 (x to TMEM, clusters over the columns) took 25 us against 24 at 4096 rows of rank 16 and
// a third more at ranks 64: its CTA's 1400 clocks for a step of 128 rows by 32 columns go into the operand's way to TMEM.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "lora_common.cuh"

namespace trc {

using namespace lora;

namespace {

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

// What a warp works on streams through a ring in shared memory: a lane asynchronously copies the 4 - 16 bytes
// that it will need itself into its own place (so the ring needs no barrier, only the lane's own wait, as long as its
// layout stays: where another one follows, few_kernel, the warp meets in between), and takes
// them into registers some steps later. In flight are thus `stages - 1` steps of every warp, without a register.
// Loads into registers a step ahead took 15 - 30 % more time than this: the registers for it left 8 warps on
// an SM.
// Copies four consecutive activations of a row from column k on; those at k_len and beyond, and a row
// that is not `live`, become zero. VEC: the view's elements are side by side, every row starts
// at a multiple of 16 bytes and k_len is a multiple of 4.
template <bool VEC>
__device__ __forceinline__ void ring_x4(uint32_t place, const char* row, bool live, int64_t nb0, int k, int k_len) {
    if constexpr (VEC) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place), "l"(row + 4ll * k), "r"(live && k < k_len ? 16 : 0)
                     : "memory");
    } else {
        const int have = live ? min(4, k_len - k) : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(place + 4 * j),
                         "l"(row + (j < have ? (k + j) * nb0 : 0)), "r"(j < have ? 4 : 0)
                         : "memory");
    }
}

__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ring_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// BYTES of a factor or of h, or zeros.
template <int BYTES>
__device__ __forceinline__ void ring_w(uint32_t place, const void* p, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(place), "l"(p), "n"(BYTES), "r"(live ? BYTES : 0) : "memory");
}

template <typename W, int N>
__device__ __forceinline__ void ring_take_w(uint32_t place, float (&w)[N]) {
    constexpr int kWords = N * static_cast<int>(sizeof(W)) / 4;
    uint32_t raw[kWords];
    if constexpr (kWords == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3]) : "r"(place) : "memory");
    else if constexpr (kWords == 2)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(raw[0]), "=r"(raw[1]) : "r"(place) : "memory");
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(raw[0]) : "r"(place) : "memory");
    widen<W, N>(raw, w);
}

__device__ __forceinline__ void ring_take(uint32_t place, float (&x)[4]) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(place) : "memory");
}

template <bool VEC>
__device__ __forceinline__ void store_x4(char* row, int64_t nb0, int k, int k_len, const float (&x)[4]) {
    if constexpr (VEC) {
        if (k < k_len) *reinterpret_cast<float4*>(row + 4ll * k) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < k_len) *reinterpret_cast<float*>(row + (k + j) * nb0) = x[j];
    }
}

template <bool VEC>
__device__ __forceinline__ void load_x4(const char* row, int64_t nb0, int k, int k_len, float (&x)[4]) {
    if constexpr (VEC) {
        const float4 t = k < k_len ? *reinterpret_cast<const float4*>(row + 4ll * k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = k + j < k_len ? *reinterpret_cast<const float*>(row + (k + j) * nb0) : 0.0f;
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

constexpr int kWarps = 8, kThreads = 256;

// Bytes of one stage of a warp's ring: the rows' part and the factor's, and the stages that keep two
// CTAs on an SM where the registers allow it (else one).
template <typename W, int NT>
struct DownRing {
    static constexpr int kX = 8 * 512, kW = 2 * NT * 32 * 4 * static_cast<int>(sizeof(W)), kStage = kX + kW;
    static constexpr int kCtas = NT == 2 ? 2 : 1;
    static constexpr int kStages = NT == 2 ? 2 : kWarps * kStage * 3 <= 224 * 1024 ? 3 : 2;
    static constexpr int kBytes = kWarps * kStages * kStage;
};
template <typename W, bool BACK, int JG>
struct UpRing {
    static constexpr int kX = 4 * 512, kW = JG * (BACK ? 4 : 2) * 32 * 4 * static_cast<int>(sizeof(W)), kStage = kX + kW;
    static constexpr int kCtas = JG <= 2 ? 2 : 1;
    static constexpr int kRoom = kCtas == 2 ? 112 * 1024 : 224 * 1024;
    static constexpr int kStages = kWarps * kStage * 4 <= kRoom ? 4 : kWarps * kStage * 3 <= kRoom ? 3 : 2;
    static constexpr int kBytes = kWarps * kStages * kStage;
};

using True  = std::true_type;
using False = std::false_type;

// ------------------------------------------------------------------ down: h = scale * x W^T
// One cluster per tile of 32 rows and slice of the tile's adapters: each CTA takes its share of the columns
// of x in steps of 32 (one line of every row), each warp every 8th of those; the partial sums meet in
// shared memory and then across the cluster, always in the same order. BACK: x is dy and W is B^T, whose
// values for one rank are `rank` apart: a lane loads V ranks of one column at once and tile i of a group of V takes
// rank V * c + i.
// Measured (rank 16, 4096 rows of 4096: 67 MB): 24 us, 2.8 TB/s; 2048 rows of 14336 (117 MB): 36 us, 3.3 TB/s; at
// ranks 64 and 32 37 us for 2048 rows of 4096, 71 us for 11008, 45 % of the pipe's cycles. Latency of 16 (rank 16) or 8
// warps on an SM bounds it.
template <typename W, bool BACK, int NT, bool VEC>
__global__ void __launch_bounds__(kThreads, DownRing<W, NT>::kCtas) down_kernel(const __grid_constant__ Adapters tab,
                                                                                   const int32_t* ids, Rows x, int64_t rows, int k_len, float* h, int ld) {
    constexpr bool HALF = sizeof(W) == 2;
    constexpr int  V = NT < 4 ? NT : 4, kRows = 32, kCols = 8 * NT;
    extern __shared__ __align__(16) float red[];  // the warps' rings, and [kWarps][kRows][kCols] partial sums
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane >> 2, q = lane & 3;
    using Ring = DownRing<W, NT>;
    constexpr int  kStages = Ring::kStages, kPiece = (BACK ? V : 4) * static_cast<int>(sizeof(W));  // of one load of W
    const uint32_t ring = smem_u32(red) + warp * (kStages * Ring::kStage);
    const int      ranks = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
    const int64_t  row0 = static_cast<int64_t>(blockIdx.x / ranks) * kRows;
    grid_wait();
    grid_dependents();
    const TileIds  tile(ids, row0, kRows, rows, tab.n);

    if (blockIdx.y == 0 && rank == 0) {  // rows without an adapter
        for (int r = warp; r < kRows; r += kWarps) {
            const int id = __shfl_sync(0xFFFFFFFFu, tile.id, r);
            if (row0 + r < rows && id < 0)
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
        const char*    xr[4];  // rows c, c + 8, c + 16, c + 24
#pragma unroll
        for (int i = 0; i < 4; ++i) xr[i] = VEC || ((mine >> (c + 8 * i)) & 1u) ? x.row<VEC>(row0 + c + 8 * i) : x.data;
        for (int j0 = 0; j0 < r; j0 += kCols) {
            float acc[2][NT][4] = {};
            auto sweep = [&](auto whole) {
                constexpr bool WV = decltype(whole)::value;
                const int step = 32 * kWarps * ranks, k_first = 32 * (rank * kWarps + warp);
                auto fetch = [&](int k, int stage) {
                    const uint32_t place = ring + stage * Ring::kStage;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int kg = k + 16 * s + 4 * q;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            ring_x4<VEC>(place + (4 * s + i) * 512 + lane * 16, xr[i], (mine >> (c + 8 * i)) & 1u, x.nb0, kg, k_len);
                        if constexpr (WV) {
                            const uint32_t wplace = place + Ring::kX + s * NT * 32 * 4 * sizeof(W) + lane * kPiece;
                            if constexpr (!BACK) {
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    const int j = j0 + 8 * n + c;
                                    ring_w<kPiece>(wplace + n * 32 * kPiece, w + static_cast<int64_t>(j) * k_len + kg, j < r && kg < k_len);
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; ++e)
#pragma unroll
                                    for (int n = 0; n < NT; n += V) {
                                        const int j = j0 + 8 * n + V * c;
                                        ring_w<kPiece>(wplace + (e * (NT / V) + n / V) * 32 * kPiece,
                                                       w + static_cast<int64_t>(kg + e) * r + j, j < r && kg < k_len);
                                    }
                            }
                        }
                    }
                    ring_commit();
                };
#pragma unroll
                for (int p = 0; p < kStages - 1; ++p) fetch(k_first + p * step, p);
                int stage = 0;
                for (int k0 = k_first; k0 < k_len; k0 += step) {
                    fetch(k0 + (kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1);
                    // the tensor core's own sums lose a little at every product: 32 columns at a time
                    float d[2][NT][4] = {};
                    ring_wait<kStages - 1>();
                    const uint32_t place = ring + stage * Ring::kStage;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int kg = k0 + 16 * s + 4 * q;
                        float wv[NT][4];
                        const uint32_t wplace = place + Ring::kX + s * NT * 32 * 4 * sizeof(W) + lane * kPiece;
                        if constexpr (!BACK) {
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const int j = j0 + 8 * n + c;
                                if constexpr (WV) ring_take_w<W, 4>(wplace + n * 32 * kPiece, wv[n]);
                                else load_w<W, 4, false>(w + static_cast<int64_t>(j) * k_len + kg, j < r ? k_len - kg : 0, wv[n]);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
#pragma unroll
                                for (int n = 0; n < NT; n += V) {
                                    const int j = j0 + 8 * n + V * c;
                                    float t[V];
                                    if constexpr (WV) ring_take_w<W, V>(wplace + (e * (NT / V) + n / V) * 32 * kPiece, t);
                                    else load_w<W, V, false>(w + static_cast<int64_t>(kg + e) * r + j, kg + e < k_len ? r - j : 0, t);
#pragma unroll
                                    for (int i = 0; i < V; ++i) wv[n + i][e] = t[i];
                                }
                        }
                        uint32_t ah[2][2][4], at[2][2][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float xv[4];
                            ring_take(place + (4 * s + i) * 512 + lane * 16, xv);
#pragma unroll
                            for (int e = 0; e < 4; ++e)  // a[e]: row c + 8 (e & 1), value 2u + (e >> 1)
                                split(xv[e], ah[e >> 1][i >> 1][(i & 1) + 2 * (e & 1)], at[e >> 1][i >> 1][(i & 1) + 2 * (e & 1)]);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (NT > 2 && j0 + 8 * (BACK ? n / V * V : n) >= r) continue;  // the same for the whole warp
                            uint32_t bh[2][2], bt[2][2];
#pragma unroll
                            for (int e = 0; e < 4; ++e) split_b<HALF>(wv[n][e], bh[e >> 1][e & 1], bt[e >> 1][e & 1]);
#pragma unroll
                            for (int u = 0; u < 2; ++u)
#pragma unroll
                                for (int m = 0; m < 2; ++m) mma_split<HALF>(d[m][n], ah[u][m], at[u][m], bh[u], bt[u]);
                        }
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[m][n][e] += d[m][n][e];
                    stage = stage + 1 == kStages ? 0 : stage + 1;
                }
                ring_wait<0>();
            };
            if (VEC && (A.vec & (BACK ? 2 : 1)) != 0) sweep(True());
            else sweep(False());
            __syncthreads();  // the partial sums take the rings' place
            // partial sums of the 8 warps, then of the cluster
            float* mywarp = red + warp * kRows * kCols;
#pragma unroll
            for (int m = 0; m < 2; ++m)
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
                red[i] = s;  // only this thread reads or writes place i
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
// A warp takes 32 rows, holds their h, and walks over groups of 16 columns; wr warps of a CTA stand side by
// side in the rows (the factor's values then come from L1 for all but one), the others in the columns. The two
// 8-column tiles of a group take columns 4 (c >> 1) + 2 i + (c & 1), i = 0, 1, so that a lane ends up with four
// consecutive columns of a row: 16-byte loads of base and stores of d. Every row has one adapter at most, so the
// adapters of a tile (and the slices of the grid that share them) go one after the other, each with its own
// rows.
template <typename W, bool BACK, int JG, bool VEC>
__global__ void __launch_bounds__(kThreads, UpRing<W, BACK, JG>::kCtas) up_kernel(const __grid_constant__ Adapters tab, const int32_t* ids,
                                                                      Rows base, Rows d, int64_t rows, int n_len, const float* h,
                                                                      int ld, int wr, int iters, int col_blocks) {
    constexpr bool HALF = sizeof(W) == 2;
    constexpr bool HELD = JG == 1;  // h is held as heads and tails
    constexpr int  kRows = 32;
    extern __shared__ __align__(16) char up_smem[];  // the warps' rings
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane >> 2, q = lane & 3;
    using Ring = UpRing<W, BACK, JG>;
    constexpr int  kStages = Ring::kStages, kPiece = 4 * static_cast<int>(sizeof(W)), kPieces = BACK ? 4 : 2;  // of 16 ranks
    const uint32_t ring = smem_u32(up_smem) + warp * (kStages * Ring::kStage);
    const int      wn = kWarps / wr;
    const int64_t  row0 = (static_cast<int64_t>(blockIdx.x / col_blocks) * wr + warp % wr) * kRows;
    const int      first = 16 * (static_cast<int>(blockIdx.x % col_blocks) * wn * iters + warp / wr), stride = 16 * wn;
    const int      last = min(n_len, first + stride * iters);
    const TileIds  tile(ids, row0, kRows, rows, tab.n);
    grid_wait();  // h is written
    grid_dependents();
    if (row0 >= rows || first >= n_len) return;

    float hv[JG][4][4];  // the first 16 * JG ranks of rows c, c + 8, ...: values 4q .. 4q + 3 of each 16
    auto load_h = [&](int j0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int g = 0; g < JG; ++g) {
                float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (row0 + c + 8 * i < rows && j0 + 16 * g < ld)
                    t = *reinterpret_cast<const float4*>(h + (row0 + c + 8 * i) * ld + j0 + 16 * g + 4 * q);
                hv[g][i][0] = t.x; hv[g][i][1] = t.y; hv[g][i][2] = t.z; hv[g][i][3] = t.w;
            }
    };
    load_h(0);
    uint32_t hh[2][2][4], ht[2][2][4];  // [rows 16 m][step]
    auto split_h = [&](int g) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) split(hv[g][2 * m + (e & 1)][2 * u + (e >> 1)], hh[m][u][e], ht[m][u][e]);
    };
    if constexpr (HELD) split_h(0);

    // rows without an adapter: the first slice copies their base
    const uint32_t none = __ballot_sync(0xFFFFFFFFu, tile.id < 0 && row0 + lane < rows);
    if (none != 0 && blockIdx.z == 0 && base.data != d.data) {
        for (int n0 = first; n0 < last; n0 += stride)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if ((none >> (c + 8 * i)) & 1u) {
                    const int64_t t = row0 + c + 8 * i;
                    float y[4] = {};
                    if (base.data != nullptr) load_x4<VEC>(base.row<VEC>(t), base.nb0, n0 + 4 * q, n_len, y);
                    store_x4<VEC>(d.row<VEC>(t), d.nb0, n0 + 4 * q, n_len, y);
                }
    }
    int turn = 0;
    for (uint32_t left = tile.leaders; left != 0; left &= left - 1) {
        if (turn++ % gridDim.z != blockIdx.z) continue;
        const int      lead = __ffs(left) - 1;
        const int      id = __shfl_sync(0xFFFFFFFFu, tile.id, lead);
        const uint32_t mine = __shfl_sync(0xFFFFFFFFu, tile.same, lead) >> c;  // bit 8 i: row c + 8 i
        const Adapter& A = tab.ad[id];
        const int      r = A.rank;
        const W*       w = static_cast<const W*>(BACK ? A.a : A.b);
        const bool     add = base.data != nullptr;
        const char*    in[4];
        char*          out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool live = (mine >> (8 * i)) & 1u;
            in[i]  = (VEC || live) && add ? base.row<VEC>(row0 + c + 8 * i) : base.data;
            out[i] = VEC || live ? d.row<VEC>(row0 + c + 8 * i) : d.data;
        }
        // RING: the factor's values come through the ring (they are whole, and all ranks are held); else straight from
        // memory, in whole loads (WV) or one by one.
        auto walk = [&](auto through, auto whole) {
            constexpr bool RING = decltype(through)::value, WV = decltype(whole)::value;
            // group g's piece i: FWD tile i's column n0 + 4 (c >> 1) + (c & 1) + 2 i, ranks 4q ..; BACK rank 4q + i, columns
            // n0 + 4 (c >> 1) ..
            auto piece = [&](int n0, int j0, int g, int i, int& have) -> const W* {
                const int jq = j0 + 16 * g + 4 * q;
                if constexpr (!BACK) {
                    const int n = n0 + 4 * (c >> 1) + (c & 1) + 2 * i;
                    have = n < n_len ? r - jq : 0;
                    return w + (static_cast<int64_t>(n) * r + jq);
                } else {
                    const int n = n0 + 4 * (c >> 1);
                    have = jq + i < r ? n_len - n : 0;
                    return w + (static_cast<int64_t>(jq + i) * n_len + n);
                }
            };
            auto fetch = [&](int n0, int stage) {
                const uint32_t place = ring + stage * Ring::kStage;
                if (add)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        ring_x4<VEC>(place + i * 512 + lane * 16, in[i], ((mine >> (8 * i)) & 1u) && n0 < last, base.nb0,
                                     n0 + 4 * q, n_len);
                if constexpr (RING)
#pragma unroll
                    for (int g = 0; g < JG; ++g)
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
                            int have;
                            const W* p = piece(n0, 0, g, i, have);
                            ring_w<kPiece>(place + Ring::kX + (g * kPieces + i) * 32 * kPiece + lane * kPiece, p, have > 0 && n0 < last);
                        }
                ring_commit();
            };
#pragma unroll
            for (int p = 0; p < kStages - 1; ++p) fetch(first + p * stride, p);
            int stage = 0;
            for (int n0 = first; n0 < last; n0 += stride) {
                fetch(n0 + (kStages - 1) * stride, stage == 0 ? kStages - 1 : stage - 1);
                const uint32_t place = ring + stage * Ring::kStage;
                ring_wait<kStages - 1>();
                float acc[2][2][4] = {};
                for (int j0 = 0; j0 < (RING ? 1 : r); j0 += 16 * JG) {
                    if (!RING && r > 16 * JG) load_h(j0);  // ranks beyond the ones held: anew for each group of columns
                    float wv[JG][2][4];
#pragma unroll
                    for (int g = 0; g < JG; ++g)
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
                            float p[4];
                            if constexpr (RING) {
                                ring_take_w<W, 4>(place + Ring::kX + (g * kPieces + i) * 32 * kPiece + lane * kPiece, p);
                            } else {
                                int have;
                                const W* from = piece(n0, j0, g, i, have);
                                load_w<W, 4, WV>(from, have, p);
                            }
                            if constexpr (!BACK) {
#pragma unroll
                                for (int e = 0; e < 4; ++e) wv[g][i][e] = p[e];
                            } else {
                                wv[g][0][i] = c & 1 ? p[1] : p[0];
                                wv[g][1][i] = c & 1 ? p[3] : p[2];
                            }
                        }
                    float t[2][2][4] = {};
#pragma unroll
                    for (int g = 0; g < JG; ++g) {
                        if (JG > 1 && j0 + 16 * g >= r) continue;
                        uint32_t bh[2][2][2], bt[2][2][2];  // [tile][step]
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) split_b<HALF>(wv[g][i][e], bh[i][e >> 1][e & 1], bt[i][e >> 1][e & 1]);
                        if constexpr (!HELD) split_h(g);
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int m = 0; m < 2; ++m)
#pragma unroll
                                for (int i = 0; i < 2; ++i) mma_split<HALF>(t[m][i], hh[m][u], ht[m][u], bh[i][u], bt[i][u]);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[e >> 3][(e >> 2) & 1][e & 3] += t[e >> 3][(e >> 2) & 1][e & 3];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // row c + 8 i: sums 2 (i & 1) .. of tile 0, then of tile 1
                    float y[4] = {};
                    if (add) ring_take(place + i * 512 + lane * 16, y);
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] += acc[i >> 1][e >> 1][2 * (i & 1) + (e & 1)];
                    if ((mine >> (8 * i)) & 1u) store_x4<VEC>(out[i], d.nb0, n0 + 4 * q, n_len, y);
                }
                stage = stage + 1 == kStages ? 0 : stage + 1;
            }
            ring_wait<0>();
        };
        const bool whole = VEC && (A.vec & (BACK ? 1 : 2)) != 0;
        if (whole && (JG < 4 || r <= 16 * JG)) walk(True(), True());
        else if (JG == 4 && whole) walk(False(), True());
        else walk(False(), False());
        if (JG == 4 && r > 16 * JG) load_h(0);
    }
}

// ------------------------------------------------------------------ few rows: both products in one launch
// A decode batch: up to 256 rows, each a request of its own, so the time is what it takes to bring the
// adapters' factors in once. One cluster of 8 CTAs takes one adapter (and, where there are few of them, one of gridDim.x / 8
// parts of the columns): it looks its rows up in ids, gathers them 16 at a time, and computes their h with the columns
// of x shared among its 64 warps; every CTA then adds the 8 CTAs' partial sums up for itself and goes on with its share of
// the output's columns, whose factor values are already on their way. The last slice of the grid takes the rows without an
// adapter. Against the two launches of down and up: 64 rows of 16 adapters (ranks 8 - 64, 4096 -> 11008, bf16)
// 23 us against 73, one row of one adapter (rank 16, 4096 -> 4096, f16) 6.7 us against 9.7. What is left is a chain of latencies:
// ids, the first columns of x and A (3 - 5 us), the sums across the cluster (3 us), the walk over the columns of B.
constexpr int kFewRows = 256, kFewCtas = 8;

// Two CTAs fit an SM (registers and shared memory). With more than 16 ranks two groups of warps take half of them each in the
// first product.
template <typename W, int NT>
struct FewRing {
    static constexpr int kGroups = NT == 2 ? 1 : 2, kTiles = NT / kGroups;  // of ranks: 8-rank tiles of a warp
    static constexpr int kKWarps = kWarps / kGroups;                        // warps that share the columns of x
    static constexpr int kDownX = 4 * 512, kDownW = 2 * kTiles * 32 * 4 * static_cast<int>(sizeof(W));
    static constexpr int kUpX = 2 * 512, kUpW = NT * 32 * 4 * static_cast<int>(sizeof(W));
    static constexpr int kStage = kDownX + kDownW, kStages = 2;
    static constexpr int kFit = 2 * kStage / (kUpX + kUpW), kUpStages = kFit >= 4 ? 4 : kFit;
    static constexpr int kWarp = kStages * kStage;
    static constexpr int kPart = 16 * 8 * NT;  // floats of one set of partial sums
    static constexpr int kBytes = kWarps * kWarp + kKWarps * kPart * 4;
    static_assert(kUpStages >= 2 && kBytes <= 112 * 1024, "two CTAs on an SM");
};

template <typename W, int NT, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) few_kernel(const __grid_constant__ Adapters tab, const int32_t* ids, Rows x, Rows base,
                                                       Rows d, int rows, int k_len, int n_len, float* h, int ld, int share) {
    constexpr bool HALF = sizeof(W) == 2;
    using Ring = FewRing<W, NT>;
    constexpr int JG = NT / 2, kCols = 8 * NT, kPiece = 4 * static_cast<int>(sizeof(W));
    extern __shared__ __align__(16) char few_smem[];
    __shared__ int16_t list[kFewRows];
    __shared__ int     counts[kWarps];
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane >> 2, q = lane & 3;
    const uint32_t ring = smem_u32(few_smem) + warp * Ring::kWarp;
    float* part = reinterpret_cast<float*>(few_smem + kWarps * Ring::kWarp);
    float* hs = part + Ring::kPart;  // the second set's place, once the first holds their sum
    constexpr int TN = Ring::kTiles;
    const int kwarp = warp % Ring::kKWarps, tile0 = warp / Ring::kKWarps * TN;  // this warp's ranks: 8 tile0 ..
    const int rank = static_cast<int>(cluster_ctarank());
    const int a = static_cast<int>(blockIdx.y);
    const bool none = a == tab.n;
    grid_wait();
    grid_dependents();
    // clusters of this adapter: `share` for each 16 of its ranks
    const int clusters = min(static_cast<int>(gridDim.x) / kFewCtas, none ? 1 : share * ((tab.ad[a].rank + 15) / 16));
    if (static_cast<int>(blockIdx.x) >= clusters * kFewCtas) return;

    // this adapter's rows, in their order
    int total = 0;
    {
        const int      t = static_cast<int>(threadIdx.x);
        const int      id = t < rows ? adapter_of(ids, t, tab.n) : -2;
        const bool     hit = id == (none ? -1 : a);
        const uint32_t hits = __ballot_sync(0xFFFFFFFFu, hit);
        if (lane == 0) counts[warp] = __popc(hits);
        __syncthreads();
        int before = 0;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
            if (v < warp) before += counts[v];
            total += counts[v];
        }
        if (hit) list[before + __popc(hits & ((1u << lane) - 1u))] = static_cast<int16_t>(t);
        __syncthreads();
    }
    if (total == 0) return;  // the whole cluster

    const int first = 16 * (static_cast<int>(blockIdx.x) * kWarps + warp), stride = 16 * kWarps * kFewCtas * clusters;
    if (none) {
        for (int i = 0; i < total; ++i) {
            const int64_t t = list[i];
            if (h != nullptr && blockIdx.x == 0)
                for (int j = threadIdx.x; j < ld; j += kThreads) h[t * ld + j] = 0.0f;
            if (base.data == d.data) continue;
            for (int n = blockIdx.x * kThreads + threadIdx.x; n < n_len; n += kThreads * kFewCtas)
                *reinterpret_cast<float*>(d.row<false>(t) + n * d.nb0) =
                    base.data != nullptr ? *reinterpret_cast<const float*>(base.row<false>(t) + n * base.nb0) : 0.0f;
        }
        return;
    }
    const Adapter& A = tab.ad[a];
    const int      r = A.rank;
    const W*       wa = static_cast<const W*>(A.a);
    const W*       wb = static_cast<const W*>(A.b);
    const bool     whole_a = VEC && (A.vec & 1) != 0, whole_b = VEC && (A.vec & 2) != 0;
    const bool     add = base.data != nullptr;
    for (int at = 0; at < total; at += 16) {
        int  t[2];
        bool live[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            live[i] = at + c + 8 * i < total;
            t[i] = live[i] ? list[at + c + 8 * i] : 0;
        }
        // h: this warp's steps of 32 columns
        float acc[TN][4] = {};
        const char* xr[2] = {x.row<VEC>(t[0]), x.row<VEC>(t[1])};
        const int   step = 32 * Ring::kKWarps * kFewCtas;
        const W*    wa_lane = wa + (static_cast<int64_t>(8 * tile0 + c) * k_len + 4 * q);
        auto fetch = [&](int k, int stage) {
            const uint32_t place = ring + stage * Ring::kStage;
            const W* p = wa_lane + k;
            if (whole_a)
#pragma unroll
                for (int n = 0; n < TN; ++n) {
                    const bool some = 8 * (tile0 + n) + c < r;
#pragma unroll
                    for (int s = 0; s < 2; ++s)
                        ring_w<kPiece>(place + Ring::kDownX + ((s * TN + n) * 32 + lane) * kPiece, p + 16 * s,
                                       some && k + 16 * s + 4 * q < k_len);
                    p += 8ll * k_len;
                }
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    ring_x4<VEC>(place + (2 * s + i) * 512 + lane * 16, xr[i], live[i], x.nb0, k + 16 * s + 4 * q, k_len);
            ring_commit();
        };
        if (8 * tile0 < r) {
            int k0 = 32 * (rank * Ring::kKWarps + kwarp), stage = 0;
            fetch(k0, 0);
            for (; k0 < k_len; k0 += step, stage ^= 1) {
                fetch(k0 + step, stage ^ 1);
                ring_wait<1>();
                const uint32_t place = ring + stage * Ring::kStage;
                float dsum[TN][4] = {};
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    uint32_t ah[2][4], at_[2][4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float xv[4];
                        ring_take(place + (2 * s + i) * 512 + lane * 16, xv);
#pragma unroll
                        for (int e = 0; e < 4; ++e) split(xv[e], ah[e >> 1][i + 2 * (e & 1)], at_[e >> 1][i + 2 * (e & 1)]);
                    }
#pragma unroll
                    for (int n = 0; n < TN; ++n) {
                        if (NT > 2 && 8 * (tile0 + n) >= r) continue;
                        const int kg = k0 + 16 * s + 4 * q, j = 8 * (tile0 + n) + c;
                        float wv[4];
                        if (whole_a) ring_take_w<W, 4>(place + Ring::kDownX + ((s * TN + n) * 32 + lane) * kPiece, wv);
                        else load_w<W, 4, false>(wa + static_cast<int64_t>(j) * k_len + kg, j < r ? k_len - kg : 0, wv);
                        uint32_t bh[2][2], bt[2][2];
#pragma unroll
                        for (int e = 0; e < 4; ++e) split_b<HALF>(wv[e], bh[e >> 1][e & 1], bt[e >> 1][e & 1]);
                        mma_split<HALF>(dsum[n], ah[0], at_[0], bh[0], bt[0]);
                        mma_split<HALF>(dsum[n], ah[1], at_[1], bh[1], bt[1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < TN; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[n][e] += dsum[n][e];
            }
            ring_wait<0>();
            __syncwarp();  // a lane's places of the next layout were other lanes' in this one (half-precision factors)
        }
        // the first groups of columns set out
        const char* in[2] = {add ? base.row<VEC>(t[0]) : nullptr, add ? base.row<VEC>(t[1]) : nullptr};
        char*       out[2] = {d.row<VEC>(t[0]), d.row<VEC>(t[1])};
        const int n_lane = 4 * (c >> 1) + (c & 1);
        const W*  wb_lane = wb + (static_cast<int64_t>(n_lane) * r + 4 * q);
        auto fetch_up = [&](int n0, int st) {
            const uint32_t place = ring + st * (Ring::kUpX + Ring::kUpW);
            if (whole_b)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const W* p = wb_lane + static_cast<int64_t>(n0 + 2 * i) * r;
                    const bool some = n0 + n_lane + 2 * i < n_len;
#pragma unroll
                    for (int g = 0; g < JG; ++g) {
                        if (JG > 1 && 16 * g >= r) break;
                        ring_w<kPiece>(place + Ring::kUpX + ((g * 2 + i) * 32 + lane) * kPiece, p + 16 * g, some && 16 * g + 4 * q < r);
                    }
                }
            if (add)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    ring_x4<VEC>(place + i * 512 + lane * 16, in[i], live[i] && n0 < n_len, base.nb0, n0 + 4 * q, n_len);
            ring_commit();
        };
#pragma unroll
        for (int p = 0; p < Ring::kUpStages - 1; ++p) fetch_up(first + p * stride, p);
        // partial sums: of the CTA's warps, then of the cluster's CTAs
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                part[kwarp * Ring::kPart + (c + 8 * (e >> 1)) * kCols + 8 * (tile0 + n) + 2 * q + (e & 1)] = acc[n][e];
        __syncthreads();
        const int n_sums = min(16, total - at) * kCols;  // of the rows that are there
        for (int i = threadIdx.x; i < n_sums; i += kThreads) {
            float s = part[i];
#pragma unroll
            for (int v = 1; v < Ring::kKWarps; ++v) s += part[v * Ring::kPart + i];
            part[i] = s;
        }
        cluster_sync();
        for (int i = threadIdx.x; i < n_sums; i += kThreads) {
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < kFewCtas; ++v) s += ld_cluster(mapa_shared(part + i, v));
            s = i % kCols < r ? s * A.scale : 0.0f;
            hs[i] = s;
            if (h != nullptr && blockIdx.x == 0 && i % kCols < ld)
                h[static_cast<int64_t>(list[at + i / kCols]) * ld + i % kCols] = s;
        }
        cluster_sync();  // every CTA has read the partial sums, and this one's h is complete
        uint32_t hh[JG][2][4], ht[JG][2][4];
#pragma unroll
        for (int g = 0; g < JG; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // (rows that are not there hold anything: their sums are not written)
                const float4 v = *reinterpret_cast<const float4*>(hs + (c + 8 * i) * kCols + 16 * g + 4 * q);
                split(v.x, hh[g][0][i], ht[g][0][i]);
                split(v.y, hh[g][0][i + 2], ht[g][0][i + 2]);
                split(v.z, hh[g][1][i], ht[g][1][i]);
                split(v.w, hh[g][1][i + 2], ht[g][1][i + 2]);
            }
        for (int n0 = first, st = 0; n0 < n_len; n0 += stride, st = st + 1 == Ring::kUpStages ? 0 : st + 1) {
            fetch_up(n0 + (Ring::kUpStages - 1) * stride, st == 0 ? Ring::kUpStages - 1 : st - 1);
            ring_wait<Ring::kUpStages - 1>();
            const uint32_t place = ring + st * (Ring::kUpX + Ring::kUpW);
            float y[2][4] = {};
#pragma unroll
            for (int g = 0; g < JG; ++g) {
                if (JG > 1 && 16 * g >= r) continue;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int n = n0 + 4 * (c >> 1) + (c & 1) + 2 * i, jq = 16 * g + 4 * q;
                    float wv[4];
                    if (whole_b) ring_take_w<W, 4>(place + Ring::kUpX + ((g * 2 + i) * 32 + lane) * kPiece, wv);
                    else load_w<W, 4, false>(wb + (static_cast<int64_t>(n) * r + jq), n < n_len ? r - jq : 0, wv);
                    uint32_t bh[2][2], bt[2][2];
#pragma unroll
                    for (int e = 0; e < 4; ++e) split_b<HALF>(wv[e], bh[e >> 1][e & 1], bt[e >> 1][e & 1]);
                    mma_split<HALF>(y[i], hh[g][0], ht[g][0], bh[0], bt[0]);
                    mma_split<HALF>(y[i], hh[g][1], ht[g][1], bh[1], bt[1]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // row c + 8 i
                float v[4] = {};
                if (add) ring_take(place + i * 512 + lane * 16, v);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += y[e >> 1][2 * i + (e & 1)];
                if (live[i]) store_x4<VEC>(out[i], d.nb0, n0 + 4 * q, n_len, v);
            }
        }
        ring_wait<0>();
        __syncthreads();  // hs and the rings before the next rows
    }
}

constexpr int64_t kMaxLen = int64_t(1) << 30;  // rows, K and N of a call

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
    bool    even = true;
    for (int i = 1; i < 4; ++i) {
        if (v->ne[i] == 1) continue;
        if (count == 1) step = v->nb[i];
        else if (v->nb[i] != want) even = false;
        count *= v->ne[i];
        want = step * count;
    }
    r.step = even && step / 4 <= INT32_MAX ? static_cast<int32_t>(step / 4) : -1;
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

// Evenly spaced rows of a multiple of four floats, side by side, that start at multiples of 16 bytes.
bool vec_rows(const trc_cuda_view* v) {
    if (v == nullptr) return true;
    if (rows_of(v).step < 0) return false;
    if (!aligned_to(v->data, 16) || v->ne[0] % 4 != 0 || v->nb[0] != 4) return false;
    for (int i = 1; i < 4; ++i)
        if (v->ne[i] > 1 && (v->nb[i] & 15) != 0) return false;
    return true;
}

int launch(const void* kernel, dim3 grid, unsigned cluster, size_t smem, void** args, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, args);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return cuda_fail(e);
    }
    note_launch();
    return TRC_CUDA_OK;
}

// The largest power of two up to `most` with which `count` units stay within `room`.
int power_for(int64_t count, int64_t room, int most) {
    int p = 1;
    while (p < most && 2 * p * count <= room) p *= 2;
    return p;
}

// CTAs that a launch aims at: two for each SM.
int64_t full_grid() { return 2 * static_cast<int64_t>(std::max(1, sm_count_current())); }

// Allows a kernel more than 48 KB of shared memory.
int allow_smem(const void* kernel, size_t smem) {
    if (smem <= 48 * 1024) return TRC_CUDA_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    return e == cudaSuccess ? TRC_CUDA_OK : cuda_fail(e);
}

// Into how many slices the adapters of a tile go, with `most` of them there and `room` for slices in a full grid:
// at least 4, so that the tiles at the borders between requests, which have two adapters or three, do not take two or three
// times as long as the rest (2048 rows, ranks 64, 32, 64: 66 -> 37 us for h, 127 -> 70 us for g); a slice without work ends at once.
int64_t slices_for(int64_t most, int64_t room) { return std::max<int64_t>(1, std::min(most, std::max<int64_t>(room, 4))); }

template <typename W, bool BACK, int NT>
int run_down(const Adapters& tab, const int32_t* ids, const Rows& x, bool vec, int64_t rows, int k, float* h, int ld,
             cudaStream_t s) {
    const int64_t tiles = (rows + 31) / 32;
    // one wave of CTAs: the columns of a tile go to 1 - 8 of them while each of their warps keeps a step of 32
    const int64_t room = full_grid() * DownRing<W, NT>::kCtas / 2;
    const int cluster = std::min(power_for(tiles, room, 8), power_for(1, (k + 255) / 256, 8));
    const int64_t most = std::min<int64_t>({tab.n, 32, rows});
    const int64_t slices = slices_for(most, room / (tiles * cluster));
    const size_t smem = std::max<size_t>(sizeof(float) * kWarps * 32 * 8 * NT, DownRing<W, NT>::kBytes);
    const void* kernel = vec ? reinterpret_cast<const void*>(&down_kernel<W, BACK, NT, true>)
                             : reinterpret_cast<const void*>(&down_kernel<W, BACK, NT, false>);
    const int st = allow_smem(kernel, smem);
    if (st != TRC_CUDA_OK) return st;
    void* args[] = {const_cast<Adapters*>(&tab), &ids, const_cast<Rows*>(&x), &rows, &k, &h, &ld};
    return launch(kernel, dim3(static_cast<unsigned>(tiles * cluster), static_cast<unsigned>(slices)), cluster, smem, args, s);
}

template <bool BACK, typename W>
int down_of(const Adapters& tab, const int32_t* ids, const Rows& x, bool vec, int64_t rows, int k, float* h, int ld,
            cudaStream_t s) {
    if (ld == 16) return run_down<W, BACK, 2>(tab, ids, x, vec, rows, k, h, ld, s);
    if (ld == 32) return run_down<W, BACK, 4>(tab, ids, x, vec, rows, k, h, ld, s);
    return run_down<W, BACK, 8>(tab, ids, x, vec, rows, k, h, ld, s);
}

template <typename W, bool BACK, int JG>
int run_up(const Adapters& tab, const int32_t* ids, const Rows& base, const Rows& d, bool vec, int64_t rows, int n,
           const float* h, int ld, cudaStream_t s) {
    const int64_t tiles = (rows + 31) / 32, groups = (n + 15) / 16;
    int wr = power_for(1, tiles, 4);  // warps side by side in the rows
    const int64_t row_blocks = (tiles + wr - 1) / wr;
    const int64_t slots = full_grid() * UpRing<W, BACK, JG>::kCtas / 2;
    int iters = 16;
    while (iters > 1 && 2 * row_blocks * (groups / (iters * (kWarps / wr))) < 3 * slots) iters /= 2;
    const int64_t col_blocks = (groups + iters * (kWarps / wr) - 1) / (iters * (kWarps / wr));
    const int64_t most = std::min<int64_t>({tab.n, 32, rows});
    const int64_t slices = std::max<int64_t>(1, std::min(most, slots / (row_blocks * col_blocks)));
    const void* kernel = vec ? reinterpret_cast<const void*>(&up_kernel<W, BACK, JG, true>)
                             : reinterpret_cast<const void*>(&up_kernel<W, BACK, JG, false>);
    if (row_blocks * col_blocks > INT32_MAX) return TRC_CUDA_EUNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(row_blocks * col_blocks), 1, static_cast<unsigned>(slices));
    const size_t smem = UpRing<W, BACK, JG>::kBytes;
    const int st = allow_smem(kernel, smem);
    if (st != TRC_CUDA_OK) return st;
    int cols = static_cast<int>(col_blocks);
    void* args[] = {const_cast<Adapters*>(&tab), &ids, const_cast<Rows*>(&base), const_cast<Rows*>(&d), &rows, &n, &h, &ld, &wr,
                    &iters, &cols};
    return launch(kernel, grid, 1, smem, args, s);
}

template <bool BACK, typename W>
int up_of(const Adapters& tab, const int32_t* ids, const Rows& base, const Rows& d, bool vec, int64_t rows, int n,
          const float* h, int ld, cudaStream_t s) {
    if (ld == 16) return run_up<W, BACK, 1>(tab, ids, base, d, vec, rows, n, h, ld, s);
    if (ld == 32) return run_up<W, BACK, 2>(tab, ids, base, d, vec, rows, n, h, ld, s);
    return run_up<W, BACK, 4>(tab, ids, base, d, vec, rows, n, h, ld, s);
}

// Both products for a batch of few rows (h may be null: then it is not wanted).
template <typename W, int NT>
int run_few(const Adapters& tab, const int32_t* ids, const Rows& x, const Rows& base, const Rows& d, bool vec, int rows, int k,
            int n, float* h, int ld, cudaStream_t s) {
    const void* kernel = vec ? reinterpret_cast<const void*>(&few_kernel<W, NT, true>) : reinterpret_cast<const void*>(&few_kernel<W, NT, false>);
    const size_t smem = FewRing<W, NT>::kBytes;
    const int st = allow_smem(kernel, smem);
    if (st != TRC_CUDA_OK) return st;
    // Every 16 ranks of an adapter get `share` clusters, so that adapters of all ranks take about the same time; together
    // they fill the SMs if every adapter occurs, as long as each warp has a group of 16 columns.
    int64_t units = 0;
    for (int i = 0; i < tab.n; ++i) units += (tab.ad[i].rank + 15) / 16;
    units = std::max<int64_t>(1, std::min<int64_t>(units, static_cast<int64_t>(rows) * (ld / 16)));
    const int64_t most = std::max<int64_t>(1, (n + 16 * kFewCtas * kWarps - 1) / (16 * kFewCtas * kWarps));
    int share = static_cast<int>(std::max<int64_t>(1, full_grid() / (units * kFewCtas)));
    const int64_t parts = std::min<int64_t>(most, static_cast<int64_t>(share) * (ld / 16));
    void* args[] = {const_cast<Adapters*>(&tab), &ids, const_cast<Rows*>(&x), const_cast<Rows*>(&base), const_cast<Rows*>(&d), &rows, &k, &n, &h, &ld,
                    &share};
    return launch(kernel, dim3(static_cast<unsigned>(parts * kFewCtas), static_cast<unsigned>(tab.n + 1)), kFewCtas, smem, args, s);
}

template <typename W>
int few_of(const Adapters& tab, const int32_t* ids, const Rows& x, const Rows& base, const Rows& d, bool vec, int rows, int k,
           int n, float* h, int ld, cudaStream_t s) {
    if (ld == 16) return run_few<W, 2>(tab, ids, x, base, d, vec, rows, k, n, h, ld, s);
    if (ld == 32) return run_few<W, 4>(tab, ids, x, base, d, vec, rows, k, n, h, ld, s);
    return run_few<W, 8>(tab, ids, x, base, d, vec, rows, k, n, h, ld, s);
}

// Whether the one-launch form takes a batch: its clusters go through an adapter's rows 16 at a time, one after the other, so
// it is for batches of up to that many rows for each adapter, and for ranks whose partial sums fit its shared memory. How
// the rows are spread over the adapters stands on the device, so the rule cannot see it. Measured against down and up,
// 4096 -> 11008, bf16 factors, 16 adapters, in us (one launch / two):
//                          64 rows                             256 rows
//                  even      half on one   all on one    even      half on one   all on one
//   rank 16        12 / 37   21 / 30       27 / 10       14 / 71   62 / 69       103 / 16
//   ranks 8 - 64   22 / 98   45 / 74       55 / 19       25 / 177  130 / 142     212 / 25
// Only a batch that (nearly) all names one of many adapters loses, up to nine times.
bool is_few(int64_t rows, int n_adapters, int64_t ld) {
    return ld <= 64 && (rows <= 16 || (rows <= kFewRows && rows <= 16 * static_cast<int64_t>(n_adapters)));
}

int few(int type, const Adapters& tab, const int32_t* ids, const trc_cuda_view* x, const trc_cuda_view* base,
        const trc_cuda_view* d, int64_t rows, float* h, int ld, cudaStream_t s) {
    const Rows rx = rows_of(x), rb = rows_of(base), rd = rows_of(d);
    const int k = static_cast<int>(x->ne[0]), n = static_cast<int>(d->ne[0]), t = static_cast<int>(rows);
    const bool vec = vec_rows(x) && vec_rows(base) && vec_rows(d);
    if (type == TRC_CUDA_TYPE_F32) return few_of<float>(tab, ids, rx, rb, rd, vec, t, k, n, h, ld, s);
    if (type == TRC_CUDA_TYPE_F16) return few_of<__half>(tab, ids, rx, rb, rd, vec, t, k, n, h, ld, s);
    return few_of<__nv_bfloat16>(tab, ids, rx, rb, rd, vec, t, k, n, h, ld, s);
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
    if (vec) {
        const int st = up_tc(BACK, type, tab, ids, base, d, rows, h, ld, s);
        if (st != TRC_CUDA_EUNSUPPORTED) return st;
    }
    if (type == TRC_CUDA_TYPE_F32) return up_of<BACK, float>(tab, ids, rb, rd, vec, rows, n, h, ld, s);
    if (type == TRC_CUDA_TYPE_F16) return up_of<BACK, __half>(tab, ids, rb, rd, vec, rows, n, h, ld, s);
    return up_of<BACK, __nv_bfloat16>(tab, ids, rb, rd, vec, rows, n, h, ld, s);
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

int trc_cuda_lora_needs_h(const trc_cuda_lora_adapter* adapters, int n_adapters, int64_t rows) {
    int64_t ld = 0;
    const int st = check_adapters(adapters, n_adapters, 1, &ld);
    if (st != TRC_CUDA_OK) return st;
    return rows <= 0 || is_few(rows, n_adapters, ld) ? 0 : 1;
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
    const bool in_one = is_few(rows, n_adapters, ld);
    if ((h == nullptr && !in_one) || !aligned_to(h, 16)) return TRC_CUDA_EINVAL;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Adapters tab;
    make_table(tab, adapters, n_adapters, type, x->ne[0]);
    if (in_one) return few(type, tab, ids, x, base, d, rows, h, static_cast<int>(ld), s);
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
    return grad_tc(tab, ids, *x, rows_of(x), *dy, rows_of(dy), vec_rows(x) && vec_rows(dy), rows, g, h, l, accumulate, s);
}

}  // extern "C"
