// lora_tc.cu -- the wide product of the low-rank adapters, d = base + h W^T, on tcgen05.
//
// It moves base and d once (8 bytes for each output) and computes 2 * rank flops for it in three TF32
// products: at rank 64 that is 3 * 128 flops for 8 bytes, more than the mma.sync pipe gives beside the copy (93
// TFLOP/s of split products), and a quarter of what tcgen05 does.
//
// A CTA takes 128 rows (the MMA's M) and walks over blocks of 32 columns (its N). The rows' h is the first
// operand and stays in TMEM for the whole walk, as heads and tails; the factor's block is the second, built in shared
// memory by four warps (heads and tails, K-major, 64-byte swizzle); the sums land in TMEM, double-buffered; four
// warps, one row per lane, add them to base's block, which TMA has brought, in place, and TMA takes it to d. A tile whose rows
// have several adapters goes through all of them for each block, each row keeping the sums of its own: base and d
// still move once.
// Measured against the warp-level kernel (mma.sync): 2048 rows, ranks 64 and 32, N = 11008: 45 us against 95 (4 TB/s); at rank 16,
// 4096 rows, N = 14336, both about 93 us (5 TB/s), bound by the adding warps (1.1 us for a block and CTA, two CTAs on an SM).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "lora_common.cuh"

namespace trc {
namespace lora {

namespace {

constexpr int kTile = 128, kBlock = 32;           // rows and columns of a step
constexpr int kSlotBytes = kTile * kBlock * 4;     // 16 KB
constexpr int kTcThreads = 288;                    // 4 warps add and store, 4 build the factor's blocks, 1 issues

template <typename W, int LD>
struct TcSmem {
    static constexpr int kPart = kBlock * LD * 4;                  // heads or tails of a block of the factor
    static constexpr int kW = kPart * (sizeof(W) == 2 ? 1 : 2);    // half factors have no tails
    // blocks of base and d: as many as leave room for two CTAs on an SM
    static constexpr int kSlots = 2 * kW <= 8 * 1024 ? 6 : 2 * kW <= 16 * 1024 ? 5 : 4;
    static constexpr int kBytes = kSlots * kSlotBytes + 2 * kW + 1024;
    static_assert(kBytes <= 112 * 1024, "two CTAs on an SM");
    static constexpr uint32_t kCols = 2 * LD + 2 * kBlock <= 128 ? 128 : 256;  // TMEM: heads, tails, two blocks of sums
};

// The MMA with its first operand in TMEM.
__device__ __forceinline__ void umma_tf32_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void* map, uint64_t* bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_store_2d(const void* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(c0), "r"(c1), "r"(src)
                 : "memory");
}

template <int kSlots>
struct Bars {
    uint64_t w_full[2];          // the factor's block is built (128 arrivals)
    uint64_t d_full[2];          // the sums are complete, the factor's block is read (the MMA's commit)
    uint64_t d_free[2];          // the sums are in registers (128 arrivals)
    uint64_t slot_full[kSlots];  // base's block is there
    uint64_t slot_free[kSlots];  // d's block has left
};

template <typename W, bool BACK, int LD>
__global__ void __launch_bounds__(kTcThreads, 2) up_tc_kernel(const __grid_constant__ Adapters tab, const int32_t* ids,
                                                           const __grid_constant__ CUtensorMap base_map,
                                                           const __grid_constant__ CUtensorMap d_map, int add, int64_t rows,
                                                           int n_len, const float* h, int ld, int blocks_per, int splits) {
    constexpr bool HALF = sizeof(W) == 2;
    using S = TcSmem<W, LD>;
    constexpr int kSlots = S::kSlots;
    extern __shared__ uint8_t tc_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* wbuf = smem + kSlots * kSlotBytes;
    __shared__ __align__(8) Bars<kSlots> bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int      tile_id[kTile], list[kTile], counts[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / splits) * kTile;
    const int block0 = static_cast<int>(blockIdx.x % splits) * blocks_per;
    const int blocks = min(blocks_per, (n_len + kBlock - 1) / kBlock - block0);

    if (threadIdx.x == 256) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.w_full[i], 128);
            mbar_init(&bars.d_full[i], 1);
            mbar_init(&bars.d_free[i], 128);
        }
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&bars.slot_full[i], 1);
            mbar_init(&bars.slot_free[i], 1);
        }
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(&tmem_slot, S::kCols);
        tmem_relinquish();
    }
    if (threadIdx.x < kTile) {
        const int64_t t = row0 + threadIdx.x;
        tile_id[threadIdx.x] = t < rows ? adapter_of(ids, t, tab.n) : -1;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // the tile's adapters, in the order of their first rows
    if (warp < 4) {
        const int t = threadIdx.x, id = tile_id[t];
        bool first = id >= 0 && (t == 0 || tile_id[t - 1] != id);
        for (int u = 0; first && u < t; ++u) first = tile_id[u] != id;
        const uint32_t firsts = __ballot_sync(0xFFFFFFFFu, first);
        if (lane == 0) counts[warp] = __popc(firsts);
        named_barrier_sync(1, 128);
        int at = __popc(firsts & ((1u << lane) - 1u));
        for (int v = 0; v < warp; ++v) at += counts[v];
        if (first) list[at] = id;
    }
    __syncthreads();
    const int n_ad = counts[0] + counts[1] + counts[2] + counts[3];
    const int per = max(n_ad, 1);  // steps of a block; a tile without adapters only passes base through
    const int steps = blocks * per;
    bool ok = true;

    if (warp < 4) {
        // ---------------- one row per lane: sums + base -> d
        const int  my_id = tile_id[threadIdx.x];
        const bool leader = threadIdx.x == 0;
        grid_wait();  // nothing comes before; the bounded waits below start their clocks after it
        for (int b = 0; b < blocks && ok; ++b) {
            const int slot = b % kSlots;
            // base first: its way from shared memory overlaps the wait for the sums. 16-byte unit u of row r lies at unit
            // u ^ (r & 7) (128-byte swizzle).
            ok = ok && mbar_wait(&bars.slot_full[slot], (b / kSlots) & 1, TRC_DEVERR_WAIT_FULL);
            uint8_t* row = smem + slot * kSlotBytes + threadIdx.x * 128;
            float    o[32];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float4 t = add ? *reinterpret_cast<const float4*>(row + ((u ^ (threadIdx.x & 7)) << 4)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                o[4 * u] = t.x; o[4 * u + 1] = t.y; o[4 * u + 2] = t.z; o[4 * u + 3] = t.w;
            }
            for (int i = 0; i < n_ad; ++i) {
                const int s = b * per + i, buf = s & 1;
                ok = ok && mbar_wait(&bars.d_full[buf], (s >> 1) & 1, TRC_DEVERR_WAIT_ACCUM);
                tc_fence_after();
                uint32_t v[32];
                __syncwarp();
                tmem_ld_32x32b_x32(tmem + (static_cast<uint32_t>(warp * 32) << 16) + 2 * LD + buf * kBlock, v);
                tmem_ld_wait();
                tc_fence_before();
                mbar_arrive(&bars.d_free[buf]);
                if (my_id == list[i])
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] += __uint_as_float(v[e]);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
                *reinterpret_cast<float4*>(row + ((u ^ (threadIdx.x & 7)) << 4)) = make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
            fence_proxy_async_smem();
            ok = named_barrier_and(1, 128, ok);
            if (leader && ok) {
                tma_store_2d(&d_map, smem_u32(smem + slot * kSlotBytes), (block0 + b) * kBlock, static_cast<int>(row0));
                bulk_commit_group();
                bulk_wait_group_read<1>();  // the block before has left its slot
                if (b > 0) mbar_arrive(&bars.slot_free[(b - 1) % kSlots]);
            }
        }
        if (leader) bulk_wait_group_all();
    } else if (warp < 8) {
        // ---------------- the rows' h to TMEM, then the factor's blocks to shared memory
        const int tid = threadIdx.x - 128;
        grid_wait();  // h is written
        if (n_ad > 0) {
            const int64_t t = row0 + tid;
            const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll
            for (int g = 0; g < LD / 16; ++g) {
                uint32_t head[16], tail[16];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (t < rows && 16 * g < ld) v = *reinterpret_cast<const float4*>(h + t * ld + 16 * g + 4 * u);
                    split(v.x, head[4 * u], tail[4 * u]);
                    split(v.y, head[4 * u + 1], tail[4 * u + 1]);
                    split(v.z, head[4 * u + 2], tail[4 * u + 2]);
                    split(v.w, head[4 * u + 3], tail[4 * u + 3]);
                }
                __syncwarp();
                tmem_st_32x32b_x16(lane_base + 16 * g, head);
                tmem_st_32x32b_x16(lane_base + LD + 16 * g, tail);
            }
            tmem_st_wait();
            tc_fence_before();
        }
        // Pieces of four values of a block: FWD column i / (LD / 4), ranks 4 (i % (LD / 4)) ..; BACK rank j, columns kq ..
        // (8 ranks and 4 groups of columns to a warp, so that the transposing stores meet in two lanes a bank).
        // Loads run kAhead steps ahead, so that a step does not wait for L2.
        constexpr int kPieces = kBlock * LD / 4 / 128, kAhead = LD == 16 ? 4 : 2;
        uint32_t raw[kAhead][kPieces][sizeof(W)];
        auto place = [&](int p, int& n, int& j) {
            const int i = tid + 128 * p;
            if constexpr (!BACK) {
                n = i / (LD / 4);
                j = 4 * (i % (LD / 4));
            } else {
                j = (i & 7) + 8 * (i / 64);
                n = 4 * ((i >> 3) & 7);
            }
        };
        auto load = [&](int s, uint32_t (&to)[kPieces][sizeof(W)]) {
            const Adapter& A = tab.ad[list[s % per]];
            const int      r = A.rank, n0 = (block0 + s / per) * kBlock;
            const W*       w = static_cast<const W*>(BACK ? A.a : A.b);
            const bool     whole = (A.vec & (BACK ? 1 : 2)) != 0;
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
                int n, j;
                place(p, n, j);
                const W* from = BACK ? w + (static_cast<int64_t>(j) * n_len + n0 + n) : w + (static_cast<int64_t>(n0 + n) * r + j);
                const int have = BACK ? (j < r ? n_len - (n0 + n) : 0) : (n0 + n < n_len ? r - j : 0);
                if (whole) load_raw<W, 4, true>(from, have, to[p]);
                else load_raw<W, 4, false>(from, have, to[p]);
            }
        };
        const int my_steps = n_ad > 0 ? steps : 0;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (u < my_steps) load(u, raw[u]);
        for (int s0 = 0; s0 < my_steps && ok; s0 += kAhead) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int s = s0 + u, buf = u & 1;  // kAhead is even
                if (s >= my_steps || !ok) continue;
                if (s >= 2) ok = mbar_wait(&bars.d_full[buf], ((s >> 1) - 1) & 1, TRC_DEVERR_WAIT_EMPTY);
                uint8_t* heads = wbuf + buf * S::kW;
                uint8_t* tails = heads + S::kPart;
#pragma unroll
                for (int p = 0; p < kPieces; ++p) {
                    int n, j;
                    place(p, n, j);
                    float    v[4];
                    uint32_t hd[4], tl[4];
                    widen<W, 4>(raw[u][p], v);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (HALF) hd[e] = __float_as_uint(v[e]);
                        else split(v[e], hd[e], tl[e]);
                    }
                    if constexpr (!BACK) {
                        const int off = (j >> 4) * (kBlock * 64) + n * 64 + ((((j >> 2) & 3) ^ ((n >> 1) & 3)) << 4);
                        *reinterpret_cast<uint4*>(heads + off) = make_uint4(hd[0], hd[1], hd[2], hd[3]);
                        if constexpr (!HALF) *reinterpret_cast<uint4*>(tails + off) = make_uint4(tl[0], tl[1], tl[2], tl[3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int m = n + e;
                            const int off = (j >> 4) * (kBlock * 64) + m * 64 + ((((j >> 2) & 3) ^ ((m >> 1) & 3)) << 4) + 4 * (j & 3);
                            *reinterpret_cast<uint32_t*>(heads + off) = hd[e];
                            if constexpr (!HALF) *reinterpret_cast<uint32_t*>(tails + off) = tl[e];
                        }
                    }
                }
                fence_proxy_async_smem();
                mbar_arrive(&bars.w_full[buf]);
                if (s + kAhead < my_steps) load(s + kAhead, raw[u]);
            }
        }
    } else if (lane == 0) {
        // ---------------- base's blocks and the MMAs
        const uint32_t idesc = make_idesc_tf32(kTile, kBlock, 0, 0);
        const uint32_t wbase = smem_u32(wbuf);
        int asked = 0, issued = 0;
        auto ask = [&](int b) {  // base's block b into its slot
            const int slot = b % kSlots;
            if (b >= kSlots && !mbar_wait(&bars.slot_free[slot], (b / kSlots - 1) & 1, TRC_DEVERR_WAIT_EMPTY)) return false;
            if (add) {
                mbar_arrive_expect_tx(&bars.slot_full[slot], kSlotBytes);
                tma_load_2d(smem_u32(smem + slot * kSlotBytes), &base_map, &bars.slot_full[slot], (block0 + b) * kBlock,
                            static_cast<int>(row0));
            } else {
                mbar_arrive(&bars.slot_full[slot]);
            }
            ++asked;
            return true;
        };
        for (int b = 0; b < min(blocks, kSlots - 1); ++b) ok = ok && ask(b);
        grid_wait();
        for (int s = 0; s < steps && ok; ++s) {
            // After a block's last MMAs, so that they run while d's block before it is still being added up: the slot of the
            // block two before is free once that one has left.
            const int b = s / per;
            auto ask_next = [&] {
                if (s % per == per - 1 && b > 0 && b + kSlots - 2 < blocks) ok = ask(b + kSlots - 2);
            };
            if (n_ad == 0) {
                ask_next();
                continue;
            }
            const int buf = s & 1;
            ok = ok && mbar_wait(&bars.w_full[buf], (s >> 1) & 1, TRC_DEVERR_WAIT_XFORM);
            if (s >= 2) ok = ok && mbar_wait(&bars.d_free[buf], ((s >> 1) - 1) & 1, TRC_DEVERR_WAIT_ACCFREE);
            if (!ok) break;
            tc_fence_after();
            const uint32_t heads = wbase + buf * S::kW, tails = heads + S::kPart, dst = tmem + 2 * LD + buf * kBlock;
            const int groups = min(LD / 16, (tab.ad[list[s % per]].rank + 15) / 16);
            for (int g = 0; g < groups; ++g)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint64_t bh = make_smem_desc(heads + g * (kBlock * 64) + k * 32, 16, 512, 4);
                    const uint32_t a = tmem + 16 * g + 8 * k;
                    umma_tf32_ts(dst, a + LD, bh, idesc, g + k > 0);
                    if constexpr (!HALF) umma_tf32_ts(dst, a, make_smem_desc(tails + g * (kBlock * 64) + k * 32, 16, 512, 4), idesc, 1);
                    umma_tf32_ts(dst, a, bh, idesc, 1);
                }
            umma_commit(&bars.d_full[buf]);
            issued = s + 1;
            ask_next();
        }
        // nothing may still write to shared memory or TMEM when the CTA ends
        for (int b = max(0, asked - kSlots); b < asked; ++b) mbar_wait_drain(&bars.slot_full[b % kSlots], (b / kSlots) & 1);
        for (int s = max(0, issued - 2); s < issued; ++s) mbar_wait_drain(&bars.d_full[s & 1], (s >> 1) & 1);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tmem, S::kCols);
}

// ------------------------------------------------------------------ gradients of the factors
// out(j, k) (+)= sum over the adapter's rows t of h[t, j] x[t, k]; dA (h = g, x) is j-major, dB (h, x = dy)
// k-major. The MMA's M are 128 columns of x, its N the ranks (up to 64 at a time), its K the rows. A thread of four
// warps owns a column: it takes 32 rows of it, splits them and puts them into its lane of TMEM, the first operand. Four
// other warps build the ranks' rows in shared memory (heads and tails, MN-major as they come) and add the sums of every 64
// rows up in fp32, because the tensor core's own sums lose a little at every product (7e-8 of the result for 8 rows in a chain).
// x comes through TMA, three to four steps ahead (rows that TMA cannot address: through asynchronous copies of each warp's
// own columns), h through copies of each lane's own pieces. With loads one step ahead, in registers, a step took a DRAM
// round trip, 1.9 us; with the four warps of x copying for themselves 0.9 us, most of it their copies' instructions.
// The CTAs of a cluster share the steps of 32 rows in turns and join their sums in order.
// Measured: 2048 rows, K = 4096, N = 14336, rank 16: 41 us (150 MB, 3.7 TB/s), mma.sync kernel 55; N = 11008, ranks 64 and 32:
// 73 us against 131. The four warps of x bound it: 1700 clocks for a step, most of them a lane's 32 loads, splits and stores to TMEM.
constexpr int kGradThreads = 320;  // 4 warps for x, 4 for the ranks, 1 issues, 1 loads
constexpr int kGradMasks = 768;
constexpr int kGradRows = 32, kGradPromote = 2;  // rows of a step, steps between two additions in fp32

struct GradSide {
    Rows         x;
    const float* h;
    int32_t      k_len;
    int32_t      strips;  // of 128 columns
};

struct GradBars {
    uint64_t a_full[2], b_full[2];  // a step's operands are there (128 arrivals each)
    uint64_t ab_free[2];            // and read (commit)
    uint64_t d_full[2];             // the sums of some steps are complete (commit)
    uint64_t d_free[2];             // and in registers (128 arrivals)
    uint64_t x_full[4], x_free[4];  // x's stages: landed, taken (128 arrivals)
};

template <int LD>
struct GradSmem {
    // The ranks' heads and, as further columns of the same operand, their tails: up to 32 ranks one MMA multiplies both
    // with x's heads, which leaves two for 8 rows instead of three (an MMA takes 46 clocks to issue whatever its N up to 64).
    // 64 ranks would need all of TMEM for it.
    static constexpr bool kJoint = LD <= 32;
    // MN-major: 2 KB for 16 rows of 32 columns (heads, then tails), 128-byte swizzle in 32-byte units
    static constexpr int  kChunk = 2 * LD / 32 * 2048, kBuf = 2 * kChunk;  // 16 rows each
    static constexpr int  kSums = kJoint ? 2 * LD : LD;             // columns of sums
    static constexpr int kStages = LD == 64 ? 3 : 4;
    static constexpr int kX = kGradRows * kTile * 4, kH = kGradRows * LD * 4;  // a stage of the rings
    static constexpr int kXAt = 2 * kBuf, kHAt = kXAt + kStages * kX, kAll = kHAt + kStages * kH;
    static constexpr int kSum = LD * (kTile + 4) * 4;
    static constexpr int kBytes = (kAll > kSum ? kAll : kSum) + 1024;
    static_assert(kBytes <= 112 * 1024, "two CTAs on an SM");
    static constexpr uint32_t kD = 4 * kGradRows, kCols = 4 * kGradRows + 2 * kSums <= 128 ? 128 : 256;
};

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t place, const void* from, bool live) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place), "l"(from), "r"(live ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(place), "l"(from), "n"(BYTES), "r"(live ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// VEC: both sides' rows are evenly spaced, whole in 16-byte pieces and start at multiples of 16 bytes.
template <int LD, bool VEC>
__global__ void __launch_bounds__(kGradThreads, 2) grad_tc_kernel(const __grid_constant__ Adapters tab, const int32_t* ids,
                                                                const __grid_constant__ CUtensorMap map_a,
                                                                const __grid_constant__ CUtensorMap map_b,
                                                                const __grid_constant__ GradSide side_a,
                                                                const __grid_constant__ GradSide side_b, int64_t rows, int ld,
                                                                int accumulate) {
    using S = GradSmem<LD>;
    extern __shared__ uint8_t tc_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) GradBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int      is_last[2];  // of a step's operands: no step follows
    __shared__ uint32_t stage_rows[4], masks[kGradMasks];
    __shared__ int      stage_last[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ranks = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
    int        strip = static_cast<int>(blockIdx.x) / ranks;
    const bool is_b = strip >= side_a.strips;
    const GradSide& G = is_b ? side_b : side_a;
    if (is_b) strip -= side_a.strips;
    const int      ad = static_cast<int>(blockIdx.z);
    const Adapter& A = tab.ad[ad];
    float*         out = is_b ? A.db : A.da;
    const int      j0 = blockIdx.y * LD, r = A.rank;
    if (out == nullptr || j0 >= r) {  // the whole cluster
        grid_wait();
        return;
    }

    if (threadIdx.x == 256) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.a_full[i], 128);
            mbar_init(&bars.b_full[i], 128);
            mbar_init(&bars.ab_free[i], 1);
            mbar_init(&bars.d_full[i], 1);
            mbar_init(&bars.d_free[i], 128);
        }
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(&bars.x_full[i], 1);
            mbar_init(&bars.x_free[i], 128);
        }
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(&tmem_slot, S::kCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    grid_wait();
    grid_dependents();

    // This CTA's steps are those of its turn that have a row of the adapter. Which rows: looked up for all of them at once,
    // at the start (step by step every one waited for its ids, and an adapter's first step for all those before it: 25 us
    // with three adapters and 2048 rows); beyond kGradMasks steps, as they come.
    const int64_t all = (rows + kGradRows - 1) / kGradRows, my = all > rank ? (all - rank + ranks - 1) / ranks : 0;
    auto rows_of_step = [&](int64_t i) {  // of the i-th step of this CTA's turn
        const int64_t t = (rank + i * ranks) * kGradRows + lane;
        return __ballot_sync(0xFFFFFFFFu, t < rows && adapter_of(ids, t, tab.n) == ad);
    };
    const int known = static_cast<int>(min(my, static_cast<int64_t>(kGradMasks)));
#pragma unroll 4
    for (int i = warp; i < known; i += kGradThreads / 32) {
        const uint32_t m = rows_of_step(i);
        if (lane == 0) masks[i] = m;
    }
    __syncthreads();
    int64_t at = -1;
    auto next = [&](uint32_t& mine) {  // the next step's number, its rows in `mine`; mine = 0: there is none
        mine = 0;
        while (mine == 0 && at + 1 < my) {
            ++at;
            mine = at < known ? masks[at] : rows_of_step(at);
        }
        return rank + at * ranks;
    };
    bool ok = true;
    // A warp's lanes go the same way after a wait, also when it has run out for only some of them: what they do next, votes
    // and moves to and from TMEM, takes the whole warp.
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) { return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, code)) != 0; };
    float (*sum)[kTile + 4] = reinterpret_cast<float (*)[kTile + 4]>(smem);  // in the place of all that
    constexpr int kStages = S::kStages;
    uint32_t ahead[kStages] = {};  // the rows of the steps in a warp's ring, the oldest step first
    auto turn = [&](auto&& fetch, int stage) {  // one more step into the ring
        uint32_t mine;
        const int64_t step = next(mine);
#pragma unroll
        for (int p = 0; p + 1 < kStages; ++p) ahead[p] = ahead[p + 1];
        ahead[kStages - 1] = mine;
        if (mine != 0) fetch(step, mine, stage);
        copy_commit();
    };

    if (warp < 4) {
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        // 32 rows of this lane's column, `pitch` floats apart, into TMEM; rows that are not the adapter's as zeros
        auto put = [&](int s, const float* x, auto pitch, uint32_t mine, bool last) {
            constexpr int kPitch = decltype(pitch)::value;
            const int buf = s & 1;
            if (s >= 2) ok = ok && wait(&bars.ab_free[buf], ((s >> 1) - 1) & 1, TRC_DEVERR_WAIT_EMPTY);
            tc_fence_after();
            const uint32_t heads = lane_base + buf * 2 * kGradRows;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float    v[16];
                uint32_t hd[16], tl[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = x[kPitch * (16 * g + e)];
                if (mine != 0xFFFFFFFFu)
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] = (mine >> (16 * g + e)) & 1u ? v[e] : 0.0f;
#pragma unroll
                for (int e = 0; e < 16; ++e) split(v[e], hd[e], tl[e]);
                __syncwarp();
                tmem_st_32x32b_x16(heads + 16 * g, hd);
                tmem_st_32x32b_x16(heads + kGradRows + 16 * g, tl);
            }
            tmem_st_wait();
            tc_fence_before();
            if (threadIdx.x == 0) is_last[buf] = last;
            mbar_arrive(&bars.a_full[buf]);
        };
        if constexpr (VEC) {
            bool last = false;
            for (int s = 0, stage = 0; !last && ok; ++s) {
                ok = wait(&bars.x_full[stage], (s / kStages) & 1, TRC_DEVERR_WAIT_FULL);
                const uint32_t mine = stage_rows[stage];
                last = stage_last[stage] != 0;
                if (!ok || mine == 0) break;  // no step at all
                put(s, reinterpret_cast<const float*>(smem + S::kXAt + stage * S::kX) + threadIdx.x,
                    std::integral_constant<int, kTile>(), mine, last);
                mbar_arrive(&bars.x_free[stage]);
                stage = stage + 1 == kStages ? 0 : stage + 1;
            }
        } else {
            const int col0 = strip * kTile + warp * 32;  // this warp's columns: [32 rows][32] floats in each stage
            const uint8_t* mine_at = smem + S::kXAt + warp * 4096;
            auto fetch = [&](int64_t step, uint32_t mine, int stage) {
                const uint32_t place = smem_u32(mine_at + stage * S::kX);
                const bool inside = col0 + lane < G.k_len;
                for (int e = 0; e < kGradRows; ++e) {
                    const bool live = inside && ((mine >> e) & 1u);
                    copy_async<4>(place + e * 128 + lane * 4,
                                  live ? G.x.row<false>(step * kGradRows + e) + (col0 + lane) * G.x.nb0 : G.x.data, live);
                }
            };
#pragma unroll
            for (int p = 0; p < kStages - 1; ++p) turn(fetch, p);
            for (int s = 0, stage = 0; ok; ++s, stage = stage + 1 == kStages ? 0 : stage + 1) {
                turn(fetch, stage == 0 ? kStages - 1 : stage - 1);
                if (ahead[0] == 0) break;
                copy_wait<kStages - 1>();
                put(s, reinterpret_cast<const float*>(mine_at + stage * S::kX) + lane, std::integral_constant<int, 32>(), 0xFFFFFFFFu,
                    ahead[1] == 0);
            }
            copy_wait<0>();
        }
        named_barrier_sync(1, 256);
    } else if (warp < 8) {
        const int tid = threadIdx.x - 128;
        float acc[LD];  // this lane's column, all ranks
#pragma unroll
        for (int j = 0; j < LD; ++j) acc[j] = 0.0f;
        constexpr int kPieces = kGradRows * LD / 4 / 128;  // four ranks of a row each
        auto place = [&](int p, int& t, int& j) {
            const int i = tid + 128 * p;  // a row's pieces side by side
            t = i / (LD / 4);
            j = 4 * (i % (LD / 4));
        };
        const uint8_t* mine_at = smem + S::kHAt + tid * 16;  // this lane's own pieces
        auto fetch = [&](int64_t step, uint32_t mine, int stage) {
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
                int t, j;
                place(p, t, j);
                copy_async<16>(smem_u32(mine_at + stage * S::kH + p * 2048), G.h + (step * kGradRows + t) * ld + j0 + j,
                               ((mine >> t) & 1u) && j0 + j < ld);
            }
        };
        auto add = [&](int q) {  // the sums of steps kGradPromote * q ..
            const int buf = q & 1;
            ok = ok && wait(&bars.d_full[buf], (q >> 1) & 1, TRC_DEVERR_WAIT_ACCUM);
            tc_fence_after();
            __syncwarp();
#pragma unroll
            for (int g = 0; g < S::kSums / 16; ++g) {
                uint32_t d[16];
                tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + S::kD + buf * S::kSums + 16 * g, d);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[(16 * g + e) % LD] += __uint_as_float(d[e]);
            }
            tc_fence_before();
            mbar_arrive(&bars.d_free[buf]);
        };
#pragma unroll
        for (int p = 0; p < kStages - 1; ++p) turn(fetch, p);
        int s = 0;
        for (int stage = 0; ok; ++s, stage = stage + 1 == kStages ? 0 : stage + 1) {
            turn(fetch, stage == 0 ? kStages - 1 : stage - 1);
            if (ahead[0] == 0) break;
            const int buf = s & 1;
            if (s >= 2) ok = wait(&bars.ab_free[buf], ((s >> 1) - 1) & 1, TRC_DEVERR_WAIT_EMPTY);
            copy_wait<kStages - 1>();
            uint8_t* heads = smem + buf * S::kBuf;
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
                int t, j;
                place(p, t, j);
                const float4 v = *reinterpret_cast<const float4*>(mine_at + stage * S::kH + p * 2048);
                uint32_t hd[4], tl[4];
                split(v.x, hd[0], tl[0]);
                split(v.y, hd[1], tl[1]);
                split(v.z, hd[2], tl[2]);
                split(v.w, hd[3], tl[3]);
                // columns m .. m + 3 of row t: chunk m / 32, 32-byte unit (m % 32) / 8 exchanged by the row
                auto at_column = [&](int m) {
                    return (t >> 4) * S::kChunk + (m >> 5) * 2048 + (t & 15) * 128 + ((((m & 31) >> 3) ^ (t & 3)) << 5) + ((m & 4) << 2);
                };
                *reinterpret_cast<uint4*>(heads + at_column(j)) = make_uint4(hd[0], hd[1], hd[2], hd[3]);
                *reinterpret_cast<uint4*>(heads + at_column(LD + j)) = make_uint4(tl[0], tl[1], tl[2], tl[3]);
            }
            fence_proxy_async_smem();
            mbar_arrive(&bars.b_full[buf]);
            // while this group of steps runs, the one before
            if (s % kGradPromote == kGradPromote - 1 && s >= kGradPromote) add(s / kGradPromote - 1);
        }
        copy_wait<0>();
        // the groups that are left: the loop has added group q when it built the last step of group q + 1
        const int groups = (s + kGradPromote - 1) / kGradPromote, added = s >= 2 * kGradPromote ? s / kGradPromote - 1 : 0;
        for (int q = added; q < groups && ok; ++q) add(q);
        // every MMA of this CTA is complete, and so are all copies once the other warps are through
        named_barrier_sync(1, 256);
#pragma unroll
        for (int j = 0; j < LD; ++j) sum[j][tid] = acc[j];
    } else if (warp == 8) {
        const uint32_t idesc = make_idesc_tf32(kTile, LD, 0, 1), joint = make_idesc_tf32(kTile, 2 * LD, 0, 1);
        const uint32_t base = smem_u32(smem);
        uint32_t mine;
        next(mine);  // is there a step at all?
        int s = 0;
        if (lane == 0 && mine != 0)
            for (bool last = false; !last && ok; ++s) {
                const int buf = s & 1, q = s / kGradPromote, part = s % kGradPromote;
                ok = mbar_wait(&bars.a_full[buf], (s >> 1) & 1, TRC_DEVERR_WAIT_XFORM) &&
                     mbar_wait(&bars.b_full[buf], (s >> 1) & 1, TRC_DEVERR_WAIT_XFORM);
                if (part == 0 && q >= 2) ok = ok && mbar_wait(&bars.d_free[q & 1], ((q >> 1) - 1) & 1, TRC_DEVERR_WAIT_ACCFREE);
                if (!ok) break;
                last = is_last[buf] != 0;
                tc_fence_after();
                const uint32_t dst = tmem + S::kD + (q & 1) * S::kSums, a0 = tmem + buf * 2 * kGradRows, b0 = base + buf * S::kBuf;
#pragma unroll
                for (int k = 0; k < kGradRows / 8; ++k) {
                    const uint64_t bh = make_smem_desc(b0 + (k >> 1) * S::kChunk + (k & 1) * 1024, 2048, 512, 1);
                    if constexpr (S::kJoint) {
                        umma_tf32_ts(dst, a0 + 8 * k, bh, joint, part + k > 0);
                        umma_tf32_ts(dst, a0 + kGradRows + 8 * k, bh, idesc, 1);
                    } else {
                        const uint64_t bt = make_smem_desc(b0 + LD / 32 * 2048 + (k >> 1) * S::kChunk + (k & 1) * 1024, 2048, 512, 1);
                        umma_tf32_ts(dst, a0 + kGradRows + 8 * k, bh, idesc, part + k > 0);
                        umma_tf32_ts(dst, a0 + 8 * k, bt, idesc, 1);
                        umma_tf32_ts(dst, a0 + 8 * k, bh, idesc, 1);
                    }
                }
                umma_commit(&bars.ab_free[buf]);
                if (part == kGradPromote - 1 || last) umma_commit(&bars.d_full[q & 1]);
            }
        // nothing may still read shared memory or TMEM when they are used anew
        if (lane == 0)
            for (int p = max(0, s - 2); p < s; ++p) mbar_wait_drain(&bars.ab_free[p & 1], (p >> 1) & 1);
    } else if constexpr (VEC) {
        // x's tiles: 32 rows of 128 columns, whoever's they are; `stage_rows` says which of them count
        uint32_t mine, following;
        int64_t  step = next(mine);
        int s = 0;
        for (bool go = true; go && ok; ++s) {
            const int     stage = s % kStages;
            const int64_t after = next(following);
            if (lane == 0) {
                if (s >= kStages) ok = mbar_wait(&bars.x_free[stage], (s / kStages - 1) & 1, TRC_DEVERR_WAIT_EMPTY);
                if (ok) {
                    stage_rows[stage] = mine;
                    stage_last[stage] = following == 0;
                    if (mine != 0) {
                        mbar_arrive_expect_tx(&bars.x_full[stage], S::kX);
                        tma_load_2d(smem_u32(smem + S::kXAt + stage * S::kX), is_b ? &map_b : &map_a, &bars.x_full[stage],
                                    strip * kTile, static_cast<int>(step * kGradRows));
                    } else {
                        mbar_arrive(&bars.x_full[stage]);
                    }
                }
            }
            ok = __shfl_sync(0xFFFFFFFFu, ok ? 1 : 0, 0) != 0;
            if (!ok) break;  // nothing was asked for in this turn
            go = following != 0;
            mine = following;
            step = after;
        }
        if (lane == 0)
            for (int p = max(0, s - kStages); p < s; ++p) mbar_wait_drain(&bars.x_full[p % kStages], (p / kStages) & 1);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tmem, S::kCols);

    // this CTA's sums, then the cluster's
    if (ranks > 1) cluster_sync();
    for (int i = rank * kGradThreads + threadIdx.x; i < LD * kTile; i += kGradThreads * ranks) {
        // neighbours in memory are neighbours in the lanes
        const int j = is_b ? i % LD : i / kTile, k = is_b ? i / LD : i % kTile;
        if (j0 + j >= r || strip * kTile + k >= G.k_len) continue;
        float total = 0.0f;
        if (ranks > 1) {
            for (int v = 0; v < ranks; ++v) total += ld_cluster(mapa_shared(&sum[j][k], v));
        } else {
            total = sum[j][k];
        }
        const int64_t kk = strip * kTile + k;
        float* o = out + (is_b ? kk * r + j0 + j : static_cast<int64_t>(j0 + j) * G.k_len + kk);
        *o = accumulate ? *o + total : total;
    }
    if (ranks > 1) cluster_sync();
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// Evenly spaced rows of floats (the caller has checked them), in boxes of box_rows by box_cols.
bool encode_rows(const trc_cuda_view& v, int64_t rows, CUtensorMap& map, int box_rows, int box_cols, CUtensorMapSwizzle swizzle) {
    auto enc = encoder();
    if (enc == nullptr) return false;
    // one stride for all rows, that of the first extent over 1
    int64_t step = 4 * v.ne[0];
    for (int i = 3; i >= 1; --i)
        if (v.ne[i] > 1) step = v.nb[i];
    if (step <= 0 || step % 16 != 0) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(v.ne[0]), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(step)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)}, one[2] = {1, 1};
    return enc(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, v.data, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int LD>
int run_grad(const Adapters& tab, const int32_t* ids, const CUtensorMap& map_a, const CUtensorMap& map_b, const GradSide& a,
             const GradSide& b, bool vec, int64_t rows, int ld, int accumulate, cudaStream_t s) {
    auto kernel = vec ? &grad_tc_kernel<LD, true> : &grad_tc_kernel<LD, false>;
    const int smem = GradSmem<LD>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e);
    const int64_t chunks = (ld + LD - 1) / LD, units = (a.strips + b.strips) * chunks * tab.n;
    // The rows of a strip go to 1 - 8 CTAs, at least four steps for each, as the least time asks: waves of two CTAs for each
    // SM, each as long as a CTA's steps (its share of an adapter's rows) and some 20 more for its start and end.
    const int64_t room = 2 * static_cast<int64_t>(std::max(1, sm_count_current())), steps = (rows + kGradRows - 1) / kGradRows;
    const int64_t share = steps / std::max(1, tab.n) + 1;
    auto time = [&](unsigned c) { return (units * c + room - 1) / room * (share / c + 20); };
    unsigned cluster = 1;
    for (unsigned c = 2; c <= 8 && 4 * static_cast<int64_t>(c) <= steps; c *= 2)
        if (time(c) < time(cluster)) cluster = c;
    if ((a.strips + b.strips) * static_cast<int64_t>(cluster) > INT32_MAX) return TRC_CUDA_EUNSUPPORTED;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((a.strips + b.strips) * cluster), static_cast<unsigned>(chunks), static_cast<unsigned>(tab.n));
    cfg.blockDim = dim3(kGradThreads);
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
    e = cudaLaunchKernelEx(&cfg, kernel, tab, ids, map_a, map_b, a, b, rows, ld, accumulate);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return cuda_fail(e);
    }
    note_launch();
    return TRC_CUDA_OK;
}

template <typename W, bool BACK, int LD>
int run(const Adapters& tab, const int32_t* ids, const CUtensorMap& base_map, const CUtensorMap& d_map, int add, int64_t rows, int n,
        const float* h, int ld, cudaStream_t s) {
    auto kernel = &up_tc_kernel<W, BACK, LD>;
    const int smem = TcSmem<W, LD>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e);
    // two waves of two CTAs for each SM (tiles at the borders between requests take longer than others), at least 2
    // blocks to a CTA
    const int64_t tiles = (rows + kTile - 1) / kTile;
    const int blocks = (n + kBlock - 1) / kBlock;
    const int64_t want = std::max<int64_t>(1, 4 * static_cast<int64_t>(std::max(1, sm_count_current())) / tiles);
    const int per = static_cast<int>(std::max<int64_t>(std::min(blocks, 2), (blocks + want - 1) / want));
    const int splits = (blocks + per - 1) / per;
    if (tiles * splits > INT32_MAX) return TRC_CUDA_EUNSUPPORTED;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * splits));
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    // It waits for down's h itself. It does not let its own successor start early: that one's CTAs would wait with most of
    // an SM's shared memory, which made the step of 2048 rows of ranks 64 and 32 6 % slower.
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, tab, ids, base_map, d_map, add, rows, n, h, ld, per, splits);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return cuda_fail(e);
    }
    note_launch();
    return TRC_CUDA_OK;
}

template <typename W, bool BACK>
int run_ld(const Adapters& tab, const int32_t* ids, const CUtensorMap& base_map, const CUtensorMap& d_map, int add, int64_t rows,
           int n, const float* h, int ld, cudaStream_t s) {
    if (ld == 16) return run<W, BACK, 16>(tab, ids, base_map, d_map, add, rows, n, h, ld, s);
    if (ld == 32) return run<W, BACK, 32>(tab, ids, base_map, d_map, add, rows, n, h, ld, s);
    return run<W, BACK, 64>(tab, ids, base_map, d_map, add, rows, n, h, ld, s);
}

template <typename W>
int run_dir(bool back, const Adapters& tab, const int32_t* ids, const CUtensorMap& base_map, const CUtensorMap& d_map, int add,
            int64_t rows, int n, const float* h, int ld, cudaStream_t s) {
    return back ? run_ld<W, true>(tab, ids, base_map, d_map, add, rows, n, h, ld, s)
                : run_ld<W, false>(tab, ids, base_map, d_map, add, rows, n, h, ld, s);
}

}  // namespace

int up_tc(bool back, int type, const Adapters& tab, const int32_t* ids, const trc_cuda_view* base, const trc_cuda_view* d,
          int64_t rows, const float* h, int ld, cudaStream_t s) {
    // a tile of 128 rows has to be worth its own: below, the warp-level kernel's tiles of 32 rows fill more SMs
    if (ld > 64 || rows < 128) return TRC_CUDA_EUNSUPPORTED;
    CUtensorMap d_map, base_map;
    if (!encode_rows(*d, rows, d_map, kTile, kBlock, CU_TENSOR_MAP_SWIZZLE_128B)) return TRC_CUDA_EUNSUPPORTED;
    base_map = d_map;
    if (base != nullptr && !encode_rows(*base, rows, base_map, kTile, kBlock, CU_TENSOR_MAP_SWIZZLE_128B)) return TRC_CUDA_EUNSUPPORTED;
    const int add = base != nullptr, n = static_cast<int>(d->ne[0]);
    if (type == TRC_CUDA_TYPE_F32) return run_dir<float>(back, tab, ids, base_map, d_map, add, rows, n, h, ld, s);
    if (type == TRC_CUDA_TYPE_F16) return run_dir<__half>(back, tab, ids, base_map, d_map, add, rows, n, h, ld, s);
    return run_dir<__nv_bfloat16>(back, tab, ids, base_map, d_map, add, rows, n, h, ld, s);
}

int grad_tc(const Adapters& tab, const int32_t* ids, const trc_cuda_view& x, const Rows& x_rows, const trc_cuda_view& dy,
            const Rows& dy_rows, bool vec, int64_t rows, const float* g, const float* h, int ld, int accumulate, cudaStream_t s) {
    bool any_a = false, any_b = false;
    for (int i = 0; i < tab.n; ++i) {
        any_a = any_a || tab.ad[i].da != nullptr;
        any_b = any_b || tab.ad[i].db != nullptr;
    }
    if (!any_a && !any_b) return TRC_CUDA_OK;
    const GradSide a{x_rows, g, static_cast<int32_t>(x.ne[0]), any_a ? static_cast<int32_t>((x.ne[0] + kTile - 1) / kTile) : 0};
    const GradSide b{dy_rows, h, static_cast<int32_t>(dy.ne[0]), any_b ? static_cast<int32_t>((dy.ne[0] + kTile - 1) / kTile) : 0};
    CUtensorMap map_a{}, map_b{};
    if (vec && rows > 0)
        vec = encode_rows(x, rows, map_a, kGradRows, kTile, CU_TENSOR_MAP_SWIZZLE_NONE) &&
              encode_rows(dy, rows, map_b, kGradRows, kTile, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (ld == 16) return run_grad<16>(tab, ids, map_a, map_b, a, b, vec, rows, ld, accumulate, s);
    if (ld == 32) return run_grad<32>(tab, ids, map_a, map_b, a, b, vec, rows, ld, accumulate, s);
    return run_grad<64>(tab, ids, map_a, map_b, a, b, vec, rows, ld, accumulate, s);
}

}  // namespace lora
}  // namespace trc
