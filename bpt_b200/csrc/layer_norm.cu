// y = LayerNorm(x + r) over the last dimension, one pass over memory.
//
// The block of modules/attention.py ends each of its two halves with `norm(h + sublayer(h))`
// (attention.py:79-81, 141, 168-171).  As two torch operators that is a read of two tensors and a
// write for the sum, then a read and a write for the normalisation; here a warp owns a row, keeps
// the sum in registers (fp32), reduces mean and variance with shuffles and writes the result
// once: 3 passes of N x dim instead of 5.  HBM-bound: (2 reads + 1 write) x N x dim x bytes.
//
// With a = x + r, mean and rstd of a row of a, n = (a - mean) rstd and q = gy gamma the derivative is
//     d a     = rstd (q - mean(q) - n mean(q n))         (the gradient of x and of r)
//     d gamma = sum over rows of gy n,   d beta = sum over rows of gy
// so one pass that reads x, r and gy and writes d a has everything; the sums over rows stay in the registers of
// the threads that own a column, then go through one partial row per block (no atomics: the order is fixed).
#include <initializer_list>
#include <type_traits>

#include "common.cuh"

namespace bpt {
namespace {

constexpr int kLnWarps = 8;

// load8 / store8: 8 elements = one 16-byte piece (bf16, fp16) or two (fp32), widened to fp32.
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&f)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4 *>(p);
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __bfloat1622float2(h[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}
__device__ __forceinline__ void load8(const __half *p, float (&f)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4 *>(p);
    const __half2 *h = reinterpret_cast<const __half2 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(h[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}
__device__ __forceinline__ void load8(const float *p, float (&f)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&f)[8]) {
    uint4 raw;
    __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = raw;
}
__device__ __forceinline__ void store8(__half *p, const float (&f)[8]) {
    uint4 raw;
    __half2 *h = reinterpret_cast<__half2 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = raw;
}
__device__ __forceinline__ void store8(float *p, const float (&f)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}

// kVecs pieces of 8 elements per lane: dim <= 256 * kVecs.  A warp per row.
template <typename T, int kVecs>
__global__ void __launch_bounds__(kLnWarps * 32)
add_layer_norm_kernel(const T *__restrict__ x, const T *__restrict__ r, const T *__restrict__ gamma,
                      const T *__restrict__ beta, float eps, T *__restrict__ y, float *__restrict__ mean_out,
                      float *__restrict__ rstd_out, int64_t n_rows, int dim) {
    const int lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x * static_cast<int64_t>(kLnWarps) + (threadIdx.x >> 5);
    if (row >= n_rows) return;
    const T *xr = x + row * dim;
    const T *rr = r ? r + row * dim : nullptr;
    float v[kVecs][8];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        const int c = (u * 32 + lane) * 8;
        if (c < dim) {
            load8(xr + c, v[u]);
            if (rr) {
                float t[8];
                load8(rr + c, t);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[u][i] += t[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += v[u][i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float mean = sum / static_cast<float>(dim);
    float sq = 0.f;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        const int c = (u * 32 + lane) * 8;
        if (c < dim) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = v[u][i] - mean;
                sq = fmaf(d, d, sq);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const float rstd = rsqrtf(sq / static_cast<float>(dim) + eps);  // biased variance, as torch.nn.LayerNorm
    if (mean_out && lane == 0) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
    T *yr = y + row * dim;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        const int c = (u * 32 + lane) * 8;
        if (c < dim) {
            float g[8], b[8], out[8];
            if (gamma) load8(gamma + c, g);
            if (beta) load8(beta + c, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n = (v[u][i] - mean) * rstd;
                out[i] = fmaf(n, gamma ? g[i] : 1.f, beta ? b[i] : 0.f);
            }
            store8(yr + c, out);
        }
    }
}

template <typename T>
int launch_add_layer_norm(const void *x, const void *r, const void *gamma, const void *beta, float eps, void *y,
                          float *mean, float *rstd, int64_t n_rows, int dim, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>((n_rows + kLnWarps - 1) / kLnWarps);
    const int vecs = (dim + 255) / 256;
#define BPT_LN_LAUNCH(V)                                                                                      \
    add_layer_norm_kernel<T, V><<<grid, kLnWarps * 32, 0, stream>>>(                                          \
        static_cast<const T *>(x), static_cast<const T *>(r), static_cast<const T *>(gamma),                  \
        static_cast<const T *>(beta), eps, static_cast<T *>(y), mean, rstd, n_rows, dim)
    if (vecs <= 1) BPT_LN_LAUNCH(1);
    else if (vecs <= 2) BPT_LN_LAUNCH(2);
    else if (vecs <= 4) BPT_LN_LAUNCH(4);
    else if (vecs <= 8) BPT_LN_LAUNCH(8);
    else BPT_LN_LAUNCH(16);
#undef BPT_LN_LAUNCH
    BPT_LAUNCH_CHECK();
    return BPT_OK;
}

// ---- any width: a row belongs to `tpr` threads of a block (a power of two from 32 to 512), each with kVecs pieces
// of kVec neighbouring elements, at most kPerThread elements in all, so the column sums of the backward fit in
// registers.  kVec is the widest of 8, 4, 1 that the width and the pointers allow.
constexpr int kPerThread = 16;
constexpr int kMaxDim = 512 * kPerThread;
constexpr int kMaxGrid = 148 * 4;  // blocks of the backward = partial rows of d gamma and d beta

template <typename T, int kVec> __device__ __forceinline__ void load_vec(const T *p, float (&f)[kVec]) {
    if constexpr (kVec == 8) {
        load8(p, f);
    } else if constexpr (kVec == 4 && sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4 *>(p);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    } else if constexpr (kVec == 4) {
        const uint2 raw = *reinterpret_cast<const uint2 *>(p);
        const T *h = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = to_acc<T>(h[i]);
    } else {
        f[0] = to_acc<T>(*p);
    }
}
template <typename T, int kVec> __device__ __forceinline__ void store_vec(T *p, const float (&f)[kVec]) {
    if constexpr (kVec == 8) {
        store8(p, f);
    } else if constexpr (kVec == 4 && sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    } else if constexpr (kVec == 4) {
        uint2 raw;
        T *h = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = from_acc<T>(f[i]);
        *reinterpret_cast<uint2 *>(p) = raw;
    } else {
        *p = from_acc<T>(f[0]);
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum over the `tpr` threads of a row.  `slot` is this call's own piece of shared memory (16 floats), not written
// again before every thread has passed another barrier.
__device__ __forceinline__ float row_sum(float v, int tpr, float *slot) {
    v = warp_sum(v);
    if (tpr == 32) return v;
    const int warp = threadIdx.x >> 5, per_row = tpr >> 5;
    if ((threadIdx.x & 31) == 0) slot[warp] = v;
    __syncthreads();
    const int first = warp / per_row * per_row;
    v = 0.f;
    for (int i = 0; i < per_row; ++i) v += slot[first + i];
    return v;
}

template <typename T, int kVec, int kVecs>
__global__ void __launch_bounds__(512)
layer_norm_any_kernel(const T *__restrict__ x, const T *__restrict__ r, const T *__restrict__ gamma,
                      const T *__restrict__ beta, float eps, T *__restrict__ y, float *__restrict__ mean_out,
                      float *__restrict__ rstd_out, int64_t n_rows, int dim, int tpr) {
    __shared__ float slots[2][16];
    const int t = threadIdx.x & (tpr - 1);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / tpr) + threadIdx.x / tpr;
    const bool live = row < n_rows;  // every thread of the block takes part in the barriers
    const int64_t base = live ? row * dim : 0;
    float v[kVecs][kVec];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        const int c = (u * tpr + t) * kVec;
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[u][i] = 0.f;
        if (live && c < dim) {
            load_vec<T, kVec>(x + base + c, v[u]);
            if (r) {
                float w[kVec];
                load_vec<T, kVec>(r + base + c, w);
#pragma unroll
                for (int i = 0; i < kVec; ++i) v[u][i] += w[i];
            }
#pragma unroll
            for (int i = 0; i < kVec; ++i) sum += v[u][i];
        }
    }
    const float mean = row_sum(sum, tpr, slots[0]) / static_cast<float>(dim);
    float sq = 0.f;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        if ((u * tpr + t) * kVec < dim) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const float d = v[u][i] - mean;
                sq = fmaf(d, d, sq);
            }
        }
    }
    const float rstd = rsqrtf(row_sum(sq, tpr, slots[1]) / static_cast<float>(dim) + eps);
    if (!live) return;
    if (mean_out && t == 0) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        const int c = (u * tpr + t) * kVec;
        if (c < dim) {
            float g[kVec], b[kVec], out[kVec];
            if (gamma) load_vec<T, kVec>(gamma + c, g);
            if (beta) load_vec<T, kVec>(beta + c, b);
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                out[i] = fmaf((v[u][i] - mean) * rstd, gamma ? g[i] : 1.f, beta ? b[i] : 0.f);
            store_vec<T, kVec>(y + base + c, out);
        }
    }
}

template <typename T, int kVec, int kVecs>
__global__ void __launch_bounds__(512)
layer_norm_backward_kernel(const T *__restrict__ gy, const T *__restrict__ x, const T *__restrict__ r,
                           const T *__restrict__ gamma, const float *__restrict__ mean_in,
                           const float *__restrict__ rstd_in, T *__restrict__ da, float *__restrict__ partial,
                           int64_t n_rows, int dim, int tpr) {
    __shared__ float slots[2][2][16];
    extern __shared__ float sums[];  // [rows of the block][dim]
    const int t = threadIdx.x & (tpr - 1), rows_here = blockDim.x / tpr, mine = threadIdx.x / tpr;
    const float inv_dim = 1.f / static_cast<float>(dim);
    float g[kVecs][kVec], acc_g[kVecs][kVec], acc_b[kVecs][kVec];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            g[u][i] = 1.f;
            acc_g[u][i] = acc_b[u][i] = 0.f;
        }
        const int c = (u * tpr + t) * kVec;
        if (gamma && c < dim) load_vec<T, kVec>(gamma + c, g[u]);
    }
    int parity = 0;
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_here; row0 < n_rows;
         row0 += static_cast<int64_t>(gridDim.x) * rows_here) {
        const int64_t row = row0 + mine;
        const bool live = row < n_rows;
        const int64_t base = live ? row * dim : 0;
        const float mean = live ? mean_in[row] : 0.f, rstd = live ? rstd_in[row] : 0.f;
        float n[kVecs][kVec], q[kVecs][kVec];
        float sq = 0.f, sqn = 0.f;
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            const int c = (u * tpr + t) * kVec;
            if (live && c < dim) {
                load_vec<T, kVec>(x + base + c, n[u]);
                load_vec<T, kVec>(gy + base + c, q[u]);
                if (r) {
                    float w[kVec];
                    load_vec<T, kVec>(r + base + c, w);
#pragma unroll
                    for (int i = 0; i < kVec; ++i) n[u][i] += w[i];
                }
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    n[u][i] = (n[u][i] - mean) * rstd;
                    acc_g[u][i] = fmaf(q[u][i], n[u][i], acc_g[u][i]);
                    acc_b[u][i] += q[u][i];
                    q[u][i] *= g[u][i];
                    sq += q[u][i];
                    sqn = fmaf(q[u][i], n[u][i], sqn);
                }
            }
        }
        if (da) {
            // both sums, then one barrier for the pair when a row spans warps
            sq = warp_sum(sq);
            sqn = warp_sum(sqn);
            if (tpr > 32) {
                const int warp = threadIdx.x >> 5, per_row = tpr >> 5, first = warp / per_row * per_row;
                if ((threadIdx.x & 31) == 0) {
                    slots[parity][0][warp] = sq;
                    slots[parity][1][warp] = sqn;
                }
                __syncthreads();  // the other parity's slots were last read before this barrier
                sq = sqn = 0.f;
                for (int i = 0; i < per_row; ++i) {
                    sq += slots[parity][0][first + i];
                    sqn += slots[parity][1][first + i];
                }
                parity ^= 1;
            }
            const float mq = sq * inv_dim, mqn = sqn * inv_dim;
#pragma unroll
            for (int u = 0; u < kVecs; ++u) {
                const int c = (u * tpr + t) * kVec;
                if (live && c < dim) {
                    float out[kVec];
#pragma unroll
                    for (int i = 0; i < kVec; ++i) out[i] = rstd * (q[u][i] - mq - n[u][i] * mqn);
                    store_vec<T, kVec>(da + base + c, out);
                }
            }
        }
    }
    if (!partial) return;
    // the block's rows of sums -> one partial row: [block][d gamma, d beta][dim]
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const int c = (u * tpr + t) * kVec + i;
                if (c < dim) sums[mine * dim + c] = which ? acc_b[u][i] : acc_g[u][i];
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < dim; c += blockDim.x) {
            float s = 0.f;
            for (int k = 0; k < rows_here; ++k) s += sums[k * dim + c];
            partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * dim + c] = s;
        }
    }
}

// d gamma and d beta from the partial rows, in block order within a thread and thread order within a column.
constexpr int kReduceRows = 16;
template <typename T>
__global__ void __launch_bounds__(32 * kReduceRows)
layer_norm_reduce_kernel(const float *__restrict__ partial, int n_partial, int dim, T *__restrict__ dgamma,
                         T *__restrict__ dbeta) {
    __shared__ float part[kReduceRows][32];
    const int c = blockIdx.x * 32 + threadIdx.x;
    float s = 0.f;
    if (c < 2 * dim)
        for (int k = threadIdx.y; k < n_partial; k += kReduceRows) s += partial[static_cast<int64_t>(k) * 2 * dim + c];
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < 2 * dim) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < kReduceRows; ++k) s += part[k][threadIdx.x];
        T *out = c < dim ? dgamma : dbeta;
        if (out) out[c < dim ? c : c - dim] = from_acc<T>(s);
    }
}

struct LnLayout {
    int tpr, block, vec;
};
// Threads per row so that a thread has at most kPerThread elements.  Rows wider than a block's 256 threads hold
// take a block of 512.
LnLayout ln_layout(int dim, int vec) {
    LnLayout l;
    l.vec = vec;
    l.tpr = 32;
    while (l.tpr * kPerThread < dim) l.tpr *= 2;
    l.block = l.tpr > 256 ? l.tpr : 256;
    return l;
}
int ln_vec(int dim, size_t elem, std::initializer_list<const void *> ptrs) {
    uintptr_t all = 0;
    for (const void *p : ptrs) all |= reinterpret_cast<uintptr_t>(p);
    if (dim % 8 == 0 && all % 16 == 0) return 8;
    if (dim % 4 == 0 && all % (4 * elem) == 0) return 4;
    return 1;
}
// Calls f(kVec, kVecs) as compile-time constants for the pieces a thread of this layout has.
template <typename F> int ln_dispatch(const LnLayout &l, int dim, F f) {
    const int n = (dim + l.tpr * l.vec - 1) / (l.tpr * l.vec);
    if (l.vec == 8) return n <= 1 ? f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>())
                                  : f(std::integral_constant<int, 8>(), std::integral_constant<int, 2>());
    if (l.vec == 4) return n <= 2 ? f(std::integral_constant<int, 4>(), std::integral_constant<int, 2>())
                         : n <= 3 ? f(std::integral_constant<int, 4>(), std::integral_constant<int, 3>())
                                  : f(std::integral_constant<int, 4>(), std::integral_constant<int, 4>());
    return n <= 4 ? f(std::integral_constant<int, 1>(), std::integral_constant<int, 4>())
                  : f(std::integral_constant<int, 1>(), std::integral_constant<int, 16>());
}

template <typename T>
int launch_layer_norm_any(const void *x, const void *r, const void *gamma, const void *beta, float eps, void *y,
                          float *mean, float *rstd, int64_t n_rows, int dim, cudaStream_t stream) {
    const LnLayout l = ln_layout(dim, ln_vec(dim, sizeof(T), {x, r, gamma, beta, y}));
    const int64_t rows_here = l.block / l.tpr;
    const unsigned grid = static_cast<unsigned>((n_rows + rows_here - 1) / rows_here);
    return ln_dispatch(l, dim, [&](auto vec, auto vecs) -> int {
        layer_norm_any_kernel<T, vec.value, vecs.value><<<grid, l.block, 0, stream>>>(
            static_cast<const T *>(x), static_cast<const T *>(r), static_cast<const T *>(gamma),
            static_cast<const T *>(beta), eps, static_cast<T *>(y), mean, rstd, n_rows, dim, l.tpr);
        BPT_LAUNCH_CHECK();
        return BPT_OK;
    });
}

int64_t ln_backward_grid(int64_t n_rows, int dim) {
    const LnLayout l = ln_layout(dim, 1);
    const int64_t blocks = (n_rows + l.block / l.tpr - 1) / (l.block / l.tpr);
    return blocks < kMaxGrid ? blocks : kMaxGrid;
}

template <typename T>
int launch_layer_norm_backward(const void *gy, const void *x, const void *r, const void *gamma, const float *mean,
                               const float *rstd, void *da, void *dgamma, void *dbeta, float *partial,
                               int64_t n_rows, int dim, cudaStream_t stream) {
    const LnLayout l = ln_layout(dim, ln_vec(dim, sizeof(T), {gy, x, r, gamma, da}));
    const unsigned grid = static_cast<unsigned>(ln_backward_grid(n_rows, dim));
    const size_t smem = sizeof(float) * static_cast<size_t>(l.block / l.tpr) * dim;  // at most 512 * 16 floats
    if (n_rows > 0) {
        const int rc = ln_dispatch(l, dim, [&](auto vec, auto vecs) -> int {
            layer_norm_backward_kernel<T, vec.value, vecs.value><<<grid, l.block, smem, stream>>>(
                static_cast<const T *>(gy), static_cast<const T *>(x), static_cast<const T *>(r),
                static_cast<const T *>(gamma), mean, rstd, static_cast<T *>(da), partial, n_rows, dim, l.tpr);
            BPT_LAUNCH_CHECK();
            return BPT_OK;
        });
        if (rc != BPT_OK) return rc;
    }
    if (partial) {
        layer_norm_reduce_kernel<T><<<(2 * dim + 31) / 32, dim3(32, kReduceRows), 0, stream>>>(
            partial, static_cast<int>(grid), dim, static_cast<T *>(dgamma), static_cast<T *>(dbeta));
        BPT_LAUNCH_CHECK();
    }
    return BPT_OK;
}

}  // namespace
}  // namespace bpt

using namespace bpt;

extern "C" int bpt_add_layer_norm(const void *x, const void *r, const void *gamma, const void *beta, double eps,
                                  void *y, int64_t n_rows, int dim, int dtype, bpt_stream_t stream_) {
    BPT_CHECK_ARG(n_rows >= 0 && dim >= 8 && dim % 8 == 0 && dim <= 4096,
                  "add_layer_norm: dim must be a multiple of 8 in [8, 4096] (got %d)", dim);
    BPT_CHECK_ARG(n_rows < (int64_t(1) << 31) * kLnWarps, "add_layer_norm: too many rows");
    if (n_rows == 0) return BPT_OK;
    BPT_CHECK_ARG(x && y, "add_layer_norm: null tensor");
    BPT_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(r) | reinterpret_cast<uintptr_t>(gamma) |
                    reinterpret_cast<uintptr_t>(beta) | reinterpret_cast<uintptr_t>(y)) & 15) == 0,
                  "add_layer_norm: tensors must be 16-byte aligned");
    return bpt_layer_norm_forward(x, r, gamma, beta, eps, y, nullptr, nullptr, n_rows, dim, dtype, stream_);
}

extern "C" int bpt_layer_norm_forward(const void *x, const void *r, const void *gamma, const void *beta, double eps,
                                      void *y, float *mean, float *rstd, int64_t n_rows, int dim, int dtype,
                                      bpt_stream_t stream_) {
    BPT_CHECK_ARG(n_rows >= 0 && dim >= 1 && dim <= kMaxDim, "layer_norm: dim must be in [1, %d] (got %d)", kMaxDim, dim);
    BPT_CHECK_ARG((mean == nullptr) == (rstd == nullptr), "layer_norm: mean and rstd go together");
    if (n_rows == 0) return BPT_OK;
    BPT_CHECK_ARG(x && y, "layer_norm: null tensor");
    cudaStream_t stream = as_stream(stream_);
    const float e = static_cast<float>(eps);
    // multiples of 8 up to 4096 keep the kernel of a warp per row
    const bool warp_rows = dim <= 4096 && ln_vec(dim, 2, {x, r, gamma, beta, y}) == 8;
    BPT_CHECK_ARG(n_rows < (int64_t(1) << 31) * (warp_rows ? kLnWarps : 1), "layer_norm: too many rows");
#define BPT_LN_FORWARD(T)                                                                                       \
    return warp_rows ? launch_add_layer_norm<T>(x, r, gamma, beta, e, y, mean, rstd, n_rows, dim, stream)        \
                     : launch_layer_norm_any<T>(x, r, gamma, beta, e, y, mean, rstd, n_rows, dim, stream)
    switch (dtype) {
        case BPT_F32: BPT_LN_FORWARD(float);
        case BPT_BF16: BPT_LN_FORWARD(__nv_bfloat16);
        case BPT_F16: BPT_LN_FORWARD(__half);
        default: return fail(BPT_ERR_UNSUPPORTED, "layer_norm: dtype %d is not supported", dtype);
    }
#undef BPT_LN_FORWARD
}

extern "C" size_t bpt_layer_norm_backward_workspace_bytes(int64_t n_rows, int dim) {
    if (n_rows < 0 || dim < 1 || dim > kMaxDim) return 0;
    return align_up(sizeof(float) * 2 * static_cast<size_t>(ln_backward_grid(n_rows, dim)) * dim, 256);
}

extern "C" int bpt_layer_norm_backward(const void *gy, const void *x, const void *r, const void *gamma,
                                       const float *mean, const float *rstd, void *da, void *dgamma, void *dbeta,
                                       int64_t n_rows, int dim, int dtype, void *workspace, size_t workspace_bytes,
                                       bpt_stream_t stream_) {
    BPT_CHECK_ARG(n_rows >= 0 && dim >= 1 && dim <= kMaxDim, "layer_norm backward: dim must be in [1, %d] (got %d)",
                  kMaxDim, dim);
    BPT_CHECK_ARG(n_rows == 0 || (gy && x && mean && rstd), "layer_norm backward: null tensor");
    if (!da && !dgamma && !dbeta) return BPT_OK;
    float *partial = nullptr;
    if (dgamma || dbeta) {
        const size_t need = bpt_layer_norm_backward_workspace_bytes(n_rows, dim);
        if (need > 0) {
            if (!workspace || workspace_bytes < need)
                return fail(BPT_ERR_WORKSPACE, "layer_norm backward: workspace of %zu bytes is too small (%zu needed)",
                            workspace_bytes, need);
            BPT_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "layer_norm backward: workspace must be 4-byte aligned");
        }
        partial = static_cast<float *>(workspace);
    }
    cudaStream_t stream = as_stream(stream_);
    if (n_rows == 0) {  // the sums over no rows
        const size_t elem = dtype == BPT_F32 ? 4 : 2;
        BPT_CHECK_ARG(dtype == BPT_F32 || dtype == BPT_BF16 || dtype == BPT_F16, "layer_norm backward: dtype %d is not supported", dtype);
        if (dgamma) BPT_CUDA(cudaMemsetAsync(dgamma, 0, elem * dim, stream));
        if (dbeta) BPT_CUDA(cudaMemsetAsync(dbeta, 0, elem * dim, stream));
        return BPT_OK;
    }
    switch (dtype) {
#define BPT_LN_BACKWARD(T) \
    return launch_layer_norm_backward<T>(gy, x, r, gamma, mean, rstd, da, dgamma, dbeta, partial, n_rows, dim, stream)
        case BPT_F32: BPT_LN_BACKWARD(float);
        case BPT_BF16: BPT_LN_BACKWARD(__nv_bfloat16);
        case BPT_F16: BPT_LN_BACKWARD(__half);
#undef BPT_LN_BACKWARD
        default: return fail(BPT_ERR_UNSUPPORTED, "layer_norm backward: dtype %d is not supported", dtype);
    }
}
