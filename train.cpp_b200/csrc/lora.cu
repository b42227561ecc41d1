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

namespace trc {

namespace {

struct Adapter {
    const void* a;
    const void* b;
    float*      da;
    float*      db;
    float       scale;
    int32_t     rank;
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

template <typename W>
__device__ __forceinline__ float to_float(W w) {
    if constexpr (sizeof(W) == 4) return w;
    else return static_cast<float>(w);
}

__device__ __forceinline__ int adapter_of(const int32_t* ids, int64_t t, int n) {
    const int id = ids == nullptr ? 0 : ids[t];
    return id >= 0 && id < n ? id : -1;
}

// One warp per row and rank: h[t, j] = scale * sum_k W(j, k) x[t, k].
template <typename W, bool BACK>
__global__ void __launch_bounds__(256) down_kernel(const __grid_constant__ Adapters tab, const int32_t* ids, Rows x,
                                                   int64_t rows, int k_len, float* h, int ld) {
    const int64_t task = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (task >= rows * ld) return;
    const int64_t t = task / ld;
    const int j = static_cast<int>(task % ld);
    const int id = adapter_of(ids, t, tab.n);
    float s = 0.0f;
    if (id >= 0 && j < tab.ad[id].rank) {
        const int r = tab.ad[id].rank;
        const W* w = static_cast<const W*>(BACK ? tab.ad[id].b : tab.ad[id].a);
        const char* xr = x.row(t);
        for (int k = lane; k < k_len; k += 32) {
            const float wk = to_float(BACK ? w[static_cast<int64_t>(k) * r + j] : w[static_cast<int64_t>(j) * k_len + k]);
            s = fmaf(wk, *reinterpret_cast<const float*>(xr + k * x.nb0), s);
        }
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        s *= tab.ad[id].scale;
    }
    if (lane == 0) h[t * ld + j] = s;
}

// One thread per output: out[t, n] = base[t, n] + sum_j W(n, j) h[t, j].
template <typename W, bool BACK>
__global__ void __launch_bounds__(256) up_kernel(const __grid_constant__ Adapters tab, const int32_t* ids, Rows base, Rows d,
                                                 int64_t rows, int n_len, const float* h, int ld) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * n_len; i += gridDim.x * 256ll) {
        const int64_t t = i / n_len;
        const int n = static_cast<int>(i % n_len);
        const int id = adapter_of(ids, t, tab.n);
        float s = 0.0f;
        if (id >= 0) {
            const int r = tab.ad[id].rank;
            const W* w = static_cast<const W*>(BACK ? tab.ad[id].a : tab.ad[id].b);
            for (int j = 0; j < r; ++j)
                s = fmaf(to_float(BACK ? w[static_cast<int64_t>(j) * n_len + n] : w[static_cast<int64_t>(n) * r + j]),
                         h[t * ld + j], s);
        }
        if (base.data != nullptr) s += *reinterpret_cast<const float*>(base.row(t) + n * base.nb0);
        *reinterpret_cast<float*>(d.row(t) + n * d.nb0) = s;
    }
}

// One thread per gradient element: out(j, k) (+)= sum over the adapter's rows of h[t, j] x[t, k];
// dA is j-major, dB k-major.
template <bool DB>
__global__ void __launch_bounds__(256) grad_kernel(const __grid_constant__ Adapters tab, const int32_t* ids, Rows x,
                                                   int64_t rows, int k_len, const float* h, int ld, bool accumulate) {
    const int id = blockIdx.y;
    const Adapter& A = tab.ad[id];
    float* out = DB ? A.db : A.da;
    if (out == nullptr) return;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < static_cast<int64_t>(A.rank) * k_len; i += gridDim.x * 256ll) {
        const int j = static_cast<int>(i / k_len), k = static_cast<int>(i % k_len);
        float s = 0.0f;
        for (int64_t t = 0; t < rows; ++t)
            if (adapter_of(ids, t, tab.n) == id)
                s = fmaf(h[t * ld + j], *reinterpret_cast<const float*>(x.row(t) + k * x.nb0), s);
        float* o = out + (DB ? static_cast<int64_t>(k) * A.rank + j : i);
        *o = accumulate ? *o + s : s;
    }
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

Adapters table_of(const trc_cuda_lora_adapter* ad, int n) {
    Adapters t;
    t.n = n;
    for (int i = 0; i < n; ++i) t.ad[i] = Adapter{ad[i].a, ad[i].b, ad[i].da, ad[i].db, ad[i].scale, ad[i].rank};
    return t;
}

template <bool BACK>
int run_down(int type, const Adapters& tab, const int32_t* ids, const Rows& x, int64_t rows, int k, float* h, int ld,
             cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>((rows * ld + 7) / 8);
    if (type == TRC_CUDA_TYPE_F32) down_kernel<float, BACK><<<grid, 256, 0, s>>>(tab, ids, x, rows, k, h, ld);
    else if (type == TRC_CUDA_TYPE_F16) down_kernel<__half, BACK><<<grid, 256, 0, s>>>(tab, ids, x, rows, k, h, ld);
    else down_kernel<__nv_bfloat16, BACK><<<grid, 256, 0, s>>>(tab, ids, x, rows, k, h, ld);
    note_launch();
    return check_launch();
}

template <bool BACK>
int run_up(int type, const Adapters& tab, const int32_t* ids, const Rows& base, const Rows& d, int64_t rows, int n,
           const float* h, int ld, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((rows * n + 255) / 256, 148 * 16));
    if (type == TRC_CUDA_TYPE_F32) up_kernel<float, BACK><<<grid, 256, 0, s>>>(tab, ids, base, d, rows, n, h, ld);
    else if (type == TRC_CUDA_TYPE_F16) up_kernel<__half, BACK><<<grid, 256, 0, s>>>(tab, ids, base, d, rows, n, h, ld);
    else up_kernel<__nv_bfloat16, BACK><<<grid, 256, 0, s>>>(tab, ids, base, d, rows, n, h, ld);
    note_launch();
    return check_launch();
}

template <bool DB>
int run_grad(const Adapters& tab, const int32_t* ids, const Rows& x, int64_t rows, int k, const float* h, int ld,
             bool accumulate, cudaStream_t s) {
    if (tab.n == 0) return TRC_CUDA_OK;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((int64_t(k) * ld + 255) / 256, 148 * 16)), tab.n);
    grad_kernel<DB><<<grid, 256, 0, s>>>(tab, ids, x, rows, k, h, ld, accumulate);
    note_launch();
    return check_launch();
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
    const Adapters tab = table_of(adapters, n_adapters);
    st = run_down<false>(type, tab, ids, rows_of(x), rows, static_cast<int>(x->ne[0]), h, static_cast<int>(ld), s);
    if (st != TRC_CUDA_OK) return st;
    return run_up<false>(type, tab, ids, rows_of(base), rows_of(d), rows, static_cast<int>(d->ne[0]), h,
                         static_cast<int>(ld), s);
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
    const Adapters tab = table_of(adapters, n_adapters);
    const bool accumulate = (flags & TRC_CUDA_MM_ACCUMULATE) != 0;
    const int k = static_cast<int>(x->ne[0]), n = static_cast<int>(dy->ne[0]), l = static_cast<int>(ld);
    float* g = static_cast<float*>(workspace);
    if (rows > 0) {
        if ((st = run_down<true>(type, tab, ids, rows_of(dy), rows, n, g, l, s)) != TRC_CUDA_OK) return st;
        if (dx != nullptr &&
            (st = run_up<true>(type, tab, ids, rows_of(base), rows_of(dx), rows, k, g, l, s)) != TRC_CUDA_OK)
            return st;
    }
    if ((st = run_grad<false>(tab, ids, rows_of(x), rows, k, g, l, accumulate, s)) != TRC_CUDA_OK) return st;
    return run_grad<true>(tab, ids, rows_of(dy), rows, n, h, l, accumulate, s);
}

}  // extern "C"
