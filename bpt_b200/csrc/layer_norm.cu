// y = LayerNorm(x + r) over the last dimension, one pass over memory.
//
// The block of modules/attention.py ends each of its two halves with `norm(h + sublayer(h))`
// (attention.py:79-81, 141, 168-171).  As two torch operators that is a read of two tensors and a
// write for the sum, then a read and a write for the normalisation; here a row belongs to one warp (wide ones to
// several), which keeps the sum in registers (fp32), reduces mean and variance with
// shuffles and writes the result once: 3 passes of N x dim instead of 5.
//
// With a = x + r, mean and rstd of a row of a, n = (a - mean) rstd and q = gy gamma the derivative is
//     d a     = rstd (q - mean(q) - n mean(q n))         (the gradient of x and of r)
//     d gamma = sum over rows of gy n,   d beta = sum over rows of gy
// so one pass that reads x, r and gy and writes d a has everything; the sums over rows stay in the registers of
// the threads that own a column, then go through one partial row per block (no atomics: the order is fixed).
//
// HBM-bound: (2 reads + 1 write) x N x dim x bytes forward, (3 reads + 1 write) backward.  131064 x 512 in bf16:
// forward 64 to 66 us, backward 91 us, 6.2 and 5.9 TB/s or 95 and 90% of what a copy reaches; the sums of the partial rows
// 8 us by themselves, half of it behind the backward's end.  What is left: the reads and writes of a memory that turns
// round between them, and of the warps an SM could hold 65% (forward) and 24% (backward, whose column sums take the
// registers; the rows ahead make up for that).
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "tma.cuh"

namespace bpt {
namespace {

// A row belongs to `tpr` threads of a block (a power of two from 32 to 512), each with kVecs pieces of kVec
// neighbouring elements, at most kPerThread elements in all, so that a row (and the backward's column sums) stays in
// registers.  kVec is the widest of 8, 4, 2, 1 that the width and the pointers allow.  (33985 x 474 in bf16, forward +
// backward: 83 us with pairs, 160 with single elements.)
constexpr int kPerThread = 16;
constexpr int kMaxDim = 512 * kPerThread;
constexpr int kMaxGrid = 148 * 2;  // blocks of the backward = partial rows of d gamma and d beta

// kVec elements as they lie in memory, in whole words (16-bit elements held one by one would take a register each).
template <typename T, int kVec> struct Raw {
    static constexpr int kWords = kVec * sizeof(T) >= 4 ? kVec * sizeof(T) / 4 : 1;
    uint32_t w[kWords];
};
template <typename T, int kVec> __device__ __forceinline__ Raw<T, kVec> load_raw(const T *p) {
    Raw<T, kVec> r;
    if constexpr (kVec * sizeof(T) >= 16) {
#pragma unroll
        for (int i = 0; i < Raw<T, kVec>::kWords; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
            r.w[i] = v.x;
            r.w[i + 1] = v.y;
            r.w[i + 2] = v.z;
            r.w[i + 3] = v.w;
        }
    } else if constexpr (kVec * sizeof(T) == 8) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        r.w[0] = v.x;
        r.w[1] = v.y;
    } else if constexpr (kVec * sizeof(T) == 4) {
        r.w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else {
        r.w[0] = *reinterpret_cast<const uint16_t *>(p);
    }
    return r;
}
template <typename T, int kVec> __device__ __forceinline__ void widen(const Raw<T, kVec> &r, float (&f)[kVec]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) f[i] = __uint_as_float(r.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const uint32_t w = r.w[i / 2];
            if constexpr (std::is_same<T, __half>::value) {
                const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w));
                f[i] = v.x;
                if (kVec > 1) f[i + 1 < kVec ? i + 1 : 0] = kVec > 1 ? v.y : v.x;
            } else {
                f[i] = __uint_as_float(w << 16);
                if (kVec > 1) f[i + 1 < kVec ? i + 1 : 0] = __uint_as_float(w & 0xFFFF0000u);
            }
        }
    }
}
template <typename T, int kVec> __device__ __forceinline__ void store_vec(T *p, const float (&f)[kVec]) {
    if constexpr (kVec == 1) {
        *p = from_acc<T>(f[0]);
    } else {
        constexpr int kWords = Raw<T, kVec>::kWords;
        uint32_t w[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = __float_as_uint(f[i]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        if constexpr (kWords == 1) {
            *reinterpret_cast<uint32_t *>(p) = w[0];
        } else if constexpr (kWords == 2) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 4)
                *reinterpret_cast<uint4 *>(reinterpret_cast<uint32_t *>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        }
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

// Elementwise arithmetic of a piece, two elements an instruction where there are two (the same roundings).
template <int n> __device__ __forceinline__ void add(float (&a)[n], const float (&b)[n]) {
    if constexpr (n == 1) {
        a[0] += b[0];
    } else {
#pragma unroll
        for (int i = 0; i < n; i += 2) {
            const float2 s = tc5::add2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
            a[i] = s.x;
            a[i + 1] = s.y;
        }
    }
}
template <int n> __device__ __forceinline__ void add(float (&a)[n], float b) {
    float all[n];
#pragma unroll
    for (int i = 0; i < n; ++i) all[i] = b;
    add(a, all);
}
template <int n> __device__ __forceinline__ void multiply(float (&a)[n], const float (&b)[n]) {
    if constexpr (n == 1) {
        a[0] *= b[0];
    } else {
#pragma unroll
        for (int i = 0; i < n; i += 2) {
            const float2 s = tc5::mul2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
            a[i] = s.x;
            a[i + 1] = s.y;
        }
    }
}
template <int n> __device__ __forceinline__ void multiply(float (&a)[n], float b) {
    float all[n];
#pragma unroll
    for (int i = 0; i < n; ++i) all[i] = b;
    multiply(a, all);
}
// c += a b
template <int n> __device__ __forceinline__ void multiply_add(float (&c)[n], const float (&a)[n], const float (&b)[n]) {
    if constexpr (n == 1) {
        c[0] = fmaf(a[0], b[0], c[0]);
    } else {
#pragma unroll
        for (int i = 0; i < n; i += 2) {
            const float2 s = tc5::fma2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), make_float2(c[i], c[i + 1]));
            c[i] = s.x;
            c[i + 1] = s.y;
        }
    }
}
// A piece a - mean -> y, with gamma and beta from column c on (or null: ones, zeros).  v is used up.
template <typename T, int kVec>
__device__ __forceinline__ void finish_piece(float (&v)[kVec], float rstd, const T *gamma, const T *beta, int c, T *y) {
    multiply(v, rstd);
    float g[kVec], b[kVec];
    if (gamma) {
        widen(load_raw<T, kVec>(gamma + c), g);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) g[i] = 1.f;
    }
    if (beta) {
        widen(load_raw<T, kVec>(beta + c), b);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) b[i] = 0.f;
    }
    multiply_add(b, v, g);
    store_vec<T, kVec>(y, b);
}
// The sums of a block's rows -> one partial row: [block][d gamma, d beta][dim].
template <int kVec, int kVecs>
__device__ __forceinline__ void store_partial(const float (&acc_g)[kVecs][kVec], const float (&acc_b)[kVecs][kVec], float *sums, float *partial,
                                              int t, int tpr, int rows_here, int mine, int dim) {
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

// The forward of rows of whole pieces of 8 that a warp holds by itself: a warp a row, a block for every few rows, nothing
// kept from row to row.  No barrier, and the SM's other warps cover a row's loads.  Against the kernel below, whose rows to
// come travel by cp.async and whose wider rows belong to several warps (x, r -> y, us):
//     131064 x 8     fp16 27 / 36                         131064 x 1024  fp32 238 / 300, bf16 138 / 165
//     131064 x 512   fp32 117 / 132, bf16 64 / 66         131064 x 1536  fp32 403 / 465, bf16 244 / 285
//     131064 x 520   fp32 124 / 223, bf16 79 / 144        131064 x 2048  fp32 631 / 575, bf16 358 / 320
// A few wide rows are better off with several warps each, more of them not before the memory is what bounds both:
//     555 x 1536     fp32 7.7 / 5.2, bf16 4.6 / 4.1       4096 x 2048    fp32 20 / 23, bf16 10.4 / 11.5
//     4096 x 1536    fp32 14 / 18, bf16 8.4 / 10.4        10000 x 2048   fp32 59 / 52, bf16 33 / 29
bool ln_row_a_warp(int64_t n_rows, int dim) {
    return dim <= 1024 || (n_rows > 2048 && (dim <= 1536 || (dim <= 2048 && n_rows <= 8192)));
}
template <typename T, int kVecs, bool kHasR, int kBlock>
__global__ void __launch_bounds__(kBlock)
layer_norm_row_kernel(const T *x, const T *r, const T *gamma, const T *beta, float eps, T *y, float *mean_out, float *rstd_out,
                      int64_t n_rows, int dim) {
    tc5::let_next_start();
    tc5::wait_for_previous();
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / 32) + (threadIdx.x >> 5), at = row * dim;
    if (row >= n_rows) return;
    float v[kVecs][8];
    float sum = 0.f, sq = 0.f;  // piece by piece: chains of 8 additions and of kVecs
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        const int c = (u * 32 + lane) * 8;
        if (c < dim) {
            widen(load_raw<T, 8>(x + at + c), v[u]);
            if constexpr (kHasR) {
                float w[8];
                widen(load_raw<T, 8>(r + at + c), w);
                add(v[u], w);
            }
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) part += v[u][i];
            sum += part;
        }
    }
    const float mean = warp_sum(sum) / static_cast<float>(dim);
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        if ((u * 32 + lane) * 8 < dim) {
            add(v[u], -mean);
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) part = fmaf(v[u][i], v[u][i], part);
            sq += part;
        }
    }
    const float rstd = rsqrtf(warp_sum(sq) / static_cast<float>(dim) + eps);
    if (mean_out && lane == 0) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        const int c = (u * 32 + lane) * 8;
        if (c < dim) finish_piece<T, 8>(v[u], rstd, gamma, beta, c, y + at + c);
    }
}

// Blocks are persistent (the backward's column sums then stay in registers).  Where pieces are 16 bytes or more, a
// thread's pieces of the kAhead rows to come travel to shared memory by cp.async, into places that only this thread
// reads: no barrier, no registers, and two or three rows a warp under way instead of one.
template <typename T, int kVec, int kVecs, int kArrays, int kBlock, int kAhead> struct Rows {
    static constexpr int kBytes = kVec * sizeof(T);
    static constexpr int kSmem = kAhead * kArrays * kVecs * kBlock * kBytes;
    const T *arrays[kArrays];
    unsigned char *smem;
    int64_t n_rows;
    int dim, first, step, ahead;  // this thread's first column, columns from piece to piece

    __device__ bool in(int u) const { return u * step + first < dim; }
    __device__ unsigned char *place(int slot, int array, int u) const {
        return smem + ((slot * kArrays + array) * kVecs + u) * (kBlock * kBytes) + threadIdx.x * kBytes;
    }
    __device__ void send(int64_t row, int slot) const {
        if (row < n_rows) {
#pragma unroll
            for (int u = 0; u < kVecs; ++u) {
                if (in(u)) {
#pragma unroll
                    for (int k = 0; k < kArrays; ++k)
#pragma unroll
                        for (int b = 0; b < kBytes; b += 16)
                            tc5::cp_async16(tc5::smem_u32(place(slot, k, u) + b),
                                            reinterpret_cast<const char *>(arrays[k] + row * dim + first + u * step) + b);
                }
            }
        }
        tc5::cp_async_commit();
    }
    __device__ void start(int64_t row, int64_t stride) {
        ahead = 0;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) send(row + k * stride, k);
    }
    __device__ void get(int64_t row, Raw<T, kVec> (&v)[kArrays][kVecs]) const {
        if constexpr (kAhead > 0) asm volatile("cp.async.wait_group %0;\n" ::"n"(kAhead > 0 ? kAhead - 1 : 0) : "memory");
        if (row >= n_rows) return;
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            if (in(u)) {
#pragma unroll
                for (int k = 0; k < kArrays; ++k) {
                    if constexpr (kAhead > 0) v[k][u] = load_raw<T, kVec>(reinterpret_cast<const T *>(place(ahead, k, u)));
                    else v[k][u] = load_raw<T, kVec>(arrays[k] + row * dim + first + u * step);
                }
            }
        }
    }
    // The places of the row that get() brought are free once its values have been used: the row kAhead further on.
    __device__ void next(int64_t row, int64_t stride) {
        if constexpr (kAhead > 0) {
            send(row + kAhead * stride, ahead);
            if (++ahead == kAhead) ahead = 0;
        }
    }
};

template <typename T, int kVec, int kVecs, bool kHasR, int kBlock, int kAhead>
__global__ void __launch_bounds__(kBlock)
layer_norm_kernel(const T *x, const T *r, const T *gamma, const T *beta, float eps,
                  T *y, float *mean_out, float *rstd_out, int64_t n_rows, int dim, int tpr) {
    tc5::let_next_start();
    tc5::wait_for_previous();
    __shared__ float slots[2][16];
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kArrays = kHasR ? 2 : 1;
    const int t = threadIdx.x & (tpr - 1), rows_here = kBlock / tpr, step = tpr * kVec;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * rows_here;
    Rows<T, kVec, kVecs, kArrays, kBlock, kAhead> rows;
    rows.arrays[0] = x;
    if constexpr (kHasR) rows.arrays[1] = r;
    rows.smem = smem;
    rows.n_rows = n_rows;
    rows.dim = dim;
    rows.first = t * kVec;
    rows.step = step;
    int64_t row = static_cast<int64_t>(blockIdx.x) * rows_here + threadIdx.x / tpr;
    rows.start(row, stride);
    // every thread of the block takes part in the barriers: the loop ends for all when the block's first row is past the end
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_here; row0 < n_rows; row0 += stride, row += stride) {
        const bool live = row < n_rows;
        Raw<T, kVec> a[kArrays][kVecs];
        rows.get(row, a);
        float v[kVecs][kVec];
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            if (live && rows.in(u)) {
                widen(a[0][u], v[u]);
                if constexpr (kHasR) {
                    float w[kVec];
                    widen(a[kArrays - 1][u], w);
                    add(v[u], w);
                }
#pragma unroll
                for (int i = 0; i < kVec; ++i) sum += v[u][i];
            }
        }
        rows.next(row, stride);
        const float mean = row_sum(sum, tpr, slots[0]) / static_cast<float>(dim);
        float sq = 0.f;
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            if (live && rows.in(u)) {
                add(v[u], -mean);
#pragma unroll
                for (int i = 0; i < kVec; ++i) sq = fmaf(v[u][i], v[u][i], sq);
            }
        }
        const float rstd = rsqrtf(row_sum(sq, tpr, slots[1]) / static_cast<float>(dim) + eps);  // biased variance, as torch.nn.LayerNorm
        if (!live) continue;
        if (mean_out && t == 0) {
            mean_out[row] = mean;
            rstd_out[row] = rstd;
        }
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            if (rows.in(u)) finish_piece<T, kVec>(v[u], rstd, gamma, beta, t * kVec + u * step, y + row * dim + t * kVec + u * step);
        }
    }
    if constexpr (kAhead > 0) tc5::cp_async_wait_all();
}

template <typename T, int kVec, int kVecs, bool kHasR, int kBlock, int kAhead>
__global__ void __launch_bounds__(kBlock, kBlock == 256 ? 2 : 1)
layer_norm_backward_kernel(const T *gy, const T *x, const T *r, const T *gamma,
                           const float *mean_in, const float *rstd_in, T *da,
                           float *partial, int64_t n_rows, int dim, int tpr) {
    tc5::let_next_start();
    tc5::wait_for_previous();
    __shared__ float slots[2][2][16];
    extern __shared__ __align__(16) unsigned char smem[];  // rows ahead; at the end the sums, [rows of the block][dim]
    const int t = threadIdx.x & (tpr - 1), rows_here = kBlock / tpr, mine = threadIdx.x / tpr, step = tpr * kVec;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * rows_here;
    const float inv_dim = 1.f / static_cast<float>(dim);
    constexpr int kArrays = kHasR ? 3 : 2;
    Rows<T, kVec, kVecs, kArrays, kBlock, kAhead> rows;
    rows.arrays[0] = x;
    rows.arrays[1] = gy;
    if constexpr (kHasR) rows.arrays[2] = r;
    rows.smem = smem;
    rows.n_rows = n_rows;
    rows.dim = dim;
    rows.first = t * kVec;
    rows.step = step;
    float acc_g[kVecs][kVec], acc_b[kVecs][kVec];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) acc_g[u][i] = acc_b[u][i] = 0.f;
    }
    int64_t row = static_cast<int64_t>(blockIdx.x) * rows_here + mine;
    float next_mean = 0.f, next_rstd = 0.f;  // a row ahead
    if (row < n_rows) {
        next_mean = mean_in[row];
        next_rstd = rstd_in[row];
    }
    rows.start(row, stride);
    int parity = 0;
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_here; row0 < n_rows; row0 += stride, row += stride) {
        const bool live = row < n_rows;
        Raw<T, kVec> v[kArrays][kVecs];
        rows.get(row, v);
        const float mean = next_mean, rstd = next_rstd;
        if (row + stride < n_rows) {
            next_mean = mean_in[row + stride];
            next_rstd = rstd_in[row + stride];
        }
        float n[kVecs][kVec], q[kVecs][kVec], sq[kVec], sqn[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) sq[i] = sqn[i] = 0.f;
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            if (live && rows.in(u)) {
                widen(v[0][u], n[u]);
                float w[kVec];
                if constexpr (kHasR) {
                    widen(v[kArrays - 1][u], w);
                    add(n[u], w);
                }
                add(n[u], -mean);
                multiply(n[u], rstd);
                widen(v[1][u], q[u]);
                multiply_add(acc_g[u], q[u], n[u]);
                add(acc_b[u], q[u]);
                if (gamma) {
                    widen(load_raw<T, kVec>(gamma + t * kVec + u * step), w);  // from L1: registers for it spilled
                    multiply(q[u], w);
                }
                add(sq, q[u]);
                multiply_add(sqn, q[u], n[u]);
            }
        }
        rows.next(row, stride);
        if (da) {
            // both sums, then one barrier for the pair when a row spans warps
            float s = 0.f, sn = 0.f;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                s += sq[i];
                sn += sqn[i];
            }
            s = warp_sum(s);
            sn = warp_sum(sn);
            if (tpr > 32) {
                const int warp = threadIdx.x >> 5, per_row = tpr >> 5, first = warp / per_row * per_row;
                if ((threadIdx.x & 31) == 0) {
                    slots[parity][0][warp] = s;
                    slots[parity][1][warp] = sn;
                }
                __syncthreads();  // the other parity's slots were last read before this barrier
                s = sn = 0.f;
                for (int i = 0; i < per_row; ++i) {
                    s += slots[parity][0][first + i];
                    sn += slots[parity][1][first + i];
                }
                parity ^= 1;
            }
            const float mq = -s * inv_dim, mqn = -sn * inv_dim;
#pragma unroll
            for (int u = 0; u < kVecs; ++u) {
                if (live && rows.in(u)) {
                    float w[kVec];
#pragma unroll
                    for (int i = 0; i < kVec; ++i) w[i] = mqn;
                    add(q[u], mq);
                    multiply_add(q[u], n[u], w);
                    multiply(q[u], rstd);
                    store_vec<T, kVec>(da + row * dim + t * kVec + u * step, q[u]);
                }
            }
        }
    }
    if constexpr (kAhead > 0) tc5::cp_async_wait_all();
    float *sums = reinterpret_cast<float *>(smem);
    if (partial) store_partial(acc_g, acc_b, sums, partial, t, tpr, rows_here, mine, dim);
}

// d gamma and d beta from the partial rows, in block order within a thread and thread order within a column.
constexpr int kReduceRows = 16;
template <typename T>
__global__ void __launch_bounds__(32 * kReduceRows)
layer_norm_reduce_kernel(const float *partial, int n_partial, int dim, T *dgamma, T *dbeta) {
    tc5::wait_for_previous();
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
    if (dim % 2 == 0 && all % (2 * elem) == 0) return 2;
    return 1;
}
// Calls f(kVec, kVecs) as compile-time constants for the pieces a thread of this layout has.  kLeast8: the fewest pieces of 8
// that there are calls for: 2, where one would be a row that a warp holds by itself, or 3, where 4 is the widest piece.
template <int kLeast8, typename F> int ln_dispatch(const LnLayout &l, int dim, F f) {
    const int n = (dim + l.tpr * l.vec - 1) / (l.tpr * l.vec);
    if constexpr (kLeast8 <= 1) {
        if (l.vec == 8 && n <= 1) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    }
    if constexpr (kLeast8 <= 2) {
        if (l.vec == 8) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 2>());
    }
    if (l.vec == 4) return n <= 2 ? f(std::integral_constant<int, 4>(), std::integral_constant<int, 2>())
                         : n <= 3 ? f(std::integral_constant<int, 4>(), std::integral_constant<int, 3>())
                                  : f(std::integral_constant<int, 4>(), std::integral_constant<int, 4>());
    if (l.vec == 2) return n <= 4 ? f(std::integral_constant<int, 2>(), std::integral_constant<int, 4>())
                                  : f(std::integral_constant<int, 2>(), std::integral_constant<int, 8>());
    return n <= 4 ? f(std::integral_constant<int, 1>(), std::integral_constant<int, 4>())
                  : f(std::integral_constant<int, 1>(), std::integral_constant<int, 16>());
}

// Blocks of a kernel that run at once.
template <typename K> int ln_resident(K kernel, int block, size_t smem) {
    int per_sm = 1;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, block, smem) != cudaSuccess || per_sm < 1) per_sm = 1;
    return per_sm * 148;
}

// Blocks of the backward: as many as run at once.
int64_t ln_backward_grid(int64_t n_rows, int dim) {
    const LnLayout l = ln_layout(dim, 1);
    const int64_t blocks = (n_rows + l.block / l.tpr - 1) / (l.block / l.tpr);
    return std::min<int64_t>(blocks, l.block == 256 ? kMaxGrid : kMaxGrid / 2);
}

template <typename T>
int launch_layer_norm(const void *x, const void *r, const void *gamma, const void *beta, float eps, void *y, float *mean, float *rstd,
                      int64_t n_rows, int dim, cudaStream_t stream) {
    const LnLayout l = ln_layout(dim, ln_vec(dim, sizeof(T), {x, r, gamma, beta, y}));
    if (l.vec == 8 && ln_row_a_warp(n_rows, dim)) {
        auto go = [&](auto vecs, auto has_r) -> int {
            constexpr int kBlock = vecs.value == 1 ? 256 : 128;  // 131064 x 512 bf16 63 against 65, x 8 35 against 27
            const auto blocks = static_cast<unsigned>((n_rows + kBlock / 32 - 1) / (kBlock / 32));
            BPT_CUDA(tc5::launch_after(layer_norm_row_kernel<T, vecs.value, has_r.value, kBlock>, blocks, kBlock, 0, stream,
                                       static_cast<const T *>(x), static_cast<const T *>(r), static_cast<const T *>(gamma),
                                       static_cast<const T *>(beta), eps, static_cast<T *>(y), mean, rstd, n_rows, dim));
            return BPT_OK;
        };
        auto with_vecs = [&](auto has_r) -> int {
            switch ((dim + 255) / 256) {
                case 1: return go(std::integral_constant<int, 1>(), has_r);
                case 2: return go(std::integral_constant<int, 2>(), has_r);
                case 3: return go(std::integral_constant<int, 3>(), has_r);
                case 4: return go(std::integral_constant<int, 4>(), has_r);
                case 5: return go(std::integral_constant<int, 5>(), has_r);
                case 6: return go(std::integral_constant<int, 6>(), has_r);
                default: return go(std::integral_constant<int, 8>(), has_r);
            }
        };
        return r ? with_vecs(std::true_type()) : with_vecs(std::false_type());
    }
    const int64_t rows_here = l.block / l.tpr, blocks = (n_rows + rows_here - 1) / rows_here;
    return ln_dispatch<2>(l, dim, [&](auto vec, auto vecs) -> int {
        auto go = [&](auto has_r, auto block) -> int {
            constexpr int kPiece = vec.value * sizeof(T), kAhead = kPiece >= 16 ? 2 : 0;
            using R = Rows<T, vec.value, vecs.value, has_r.value ? 2 : 1, block.value, kAhead>;
            auto kernel = layer_norm_kernel<T, vec.value, vecs.value, has_r.value, block.value, kAhead>;
            static tc5::OncePerDevice allowed;
            BPT_CUDA(tc5::allow_smem(allowed, kernel, R::kSmem));
            static const int resident = ln_resident(kernel, block.value, R::kSmem);  // one wave of persistent blocks
            BPT_CUDA(tc5::launch_after(kernel, static_cast<unsigned>(std::min<int64_t>(blocks, resident)), block.value, R::kSmem, stream,
                                       static_cast<const T *>(x), static_cast<const T *>(r), static_cast<const T *>(gamma),
                                       static_cast<const T *>(beta), eps, static_cast<T *>(y), mean, rstd, n_rows, dim, l.tpr));
            return BPT_OK;
        };
        auto with_block = [&](auto has_r) -> int {
            return l.block == 256 ? go(has_r, std::integral_constant<int, 256>()) : go(has_r, std::integral_constant<int, 512>());
        };
        return r ? with_block(std::true_type()) : with_block(std::false_type());
    });
}

template <typename T>
int launch_layer_norm_backward(const void *gy, const void *x, const void *r, const void *gamma, const float *mean,
                               const float *rstd, void *da, void *dgamma, void *dbeta, float *partial,
                               int64_t n_rows, int dim, cudaStream_t stream) {
    const LnLayout l = ln_layout(dim, std::min<int>(ln_vec(dim, sizeof(T), {gy, x, r, gamma, da}), 16 / sizeof(T)));
    const unsigned grid = static_cast<unsigned>(ln_backward_grid(n_rows, dim));
    const int rc = ln_dispatch<sizeof(T) == 4 ? 3 : 1>(l, dim, [&](auto vec, auto vecs) -> int {
        auto go = [&](auto has_r) -> int {
            // three rows ahead where two blocks a SM have the room, else two; pieces that are not 16 bytes come directly
            constexpr int kRow = 256 * 16 * vecs.value * (has_r.value ? 3 : 2);
            constexpr int kAhead = vec.value * sizeof(T) != 16 ? 0 : 3 * kRow <= (100 << 10) ? 3 : 2;
            auto kernel = l.block == 256 ? layer_norm_backward_kernel<T, vec.value, vecs.value, has_r.value, 256, kAhead>
                                         : layer_norm_backward_kernel<T, vec.value, vecs.value, has_r.value, 512, kAhead>;
            const size_t sums = sizeof(float) * static_cast<size_t>(l.block / l.tpr) * dim;  // at most 512 * 16 floats
            const size_t smem = std::max<size_t>(kAhead * kRow * (l.block / 256), partial ? sums : 0);
            static tc5::OncePerDevice allowed[2];
            BPT_CUDA(tc5::allow_smem(allowed[l.block == 512], kernel, std::max<size_t>(kAhead * kRow * (l.block / 256), 32 << 10)));
            BPT_CUDA(tc5::launch_after(kernel, grid, l.block, smem, stream, static_cast<const T *>(gy), static_cast<const T *>(x),
                                       static_cast<const T *>(r), static_cast<const T *>(gamma), mean, rstd, static_cast<T *>(da), partial, n_rows,
                                       dim, l.tpr));
            return BPT_OK;
        };
        return r ? go(std::true_type()) : go(std::false_type());
    });
    if (rc != BPT_OK) return rc;
    if (partial) {
        BPT_CUDA(tc5::launch_after(layer_norm_reduce_kernel<T>, (2 * dim + 31) / 32, dim3(32, kReduceRows), 0, stream, partial,
                                   static_cast<int>(grid), dim, static_cast<T *>(dgamma), static_cast<T *>(dbeta)));
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
#define BPT_LN_FORWARD(T) return launch_layer_norm<T>(x, r, gamma, beta, e, y, mean, rstd, n_rows, dim, stream)
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
