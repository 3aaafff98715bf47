// Softmax cross entropy fused with the projection that makes the logits, forward and backward, without the logits
// ever being in memory as a whole.
//
// For token i with features x_i (D numbers) and target t, a weight W (V x D), a bias b and a label smoothing e,
//     z_iv   = <x_i, W_v> + b_v,          lse_i = log sum_v exp(z_iv)
//     loss_i = lse_i - (1 - e) z_it - (e / V) sum_v z_iv
//     d z_iv = g_i (exp(z_iv - lse_i) - e / V - (1 - e) [v = t])       (g_i: gradient that reaches loss_i)
//     d x = dZ W,   d W = dZ^T X,   d b = column sums of dZ
// Tokens whose target is `ignore_index` have loss 0 and g = 0.
//
// All four products run in one kernel shape on the 5th-generation tensor cores: a persistent block per SM walks
// 128 x 256 tiles; one warp brings operand tiles in by TMA (128-byte swizzle, four stages), one issues tcgen05.mma
// into one of two accumulators in tensor memory, eight warps read the other accumulator and finish the tile.
//   stats  Z tiles of consecutive vocabulary blocks of one block of tokens: a running maximum and sum per row stay in
//          registers, a row's pieces (one per block that worked on it) are merged by the loss kernel;
//   grad   Z tiles once more (cheaper than keeping them: at D = 512 a logit costs 0.7 ps of tensor time, its fp32
//          copy 1.2 ps of HBM time), turned into dZ, which is kept for one piece of the vocabulary x tokens at a time;
//   dx, dw dZ W and dZ^T X of the piece.  dZ is read K-major by the one and MN-major by the other.
// dZ is rounded to the operands' 16-bit type, without g where all g_i are one number (the scale goes onto the fp32
// results): a half-step error of each probability, the size of the rounding of the gradients themselves.
// fp32 operands are split into three bf16 planes (8 + 8 + 8 significant bits, by truncation, exact) and each product
// is run as the six products of planes whose weight is above 2^-24, smallest first.
#include <algorithm>
#include <type_traits>

#include "fused_common.cuh"
#include "tma.cuh"

namespace bpt {
namespace {

using namespace tc5;

constexpr int kBM = 128, kBN = 256, kBK = 64, kStages = 4;
constexpr int kABytes = kBM * kBK * 2, kBBytes = kBN * kBK * 2, kStageBytes = kABytes + kBBytes;
constexpr int kChunkBytes = 64 * 128;  // an MN-major tile: 64 rows along K of 64 elements
constexpr int kFinishWarps = 8, kThreads = (kFinishWarps + 2) * 32;
constexpr int kGrid = 148;             // blocks at most: one per SM
constexpr int kSmemBytes = kStages * kStageBytes + 2 * kBN * 4 + 256 + 1024;

enum Kind { kStats, kGrad, kDx, kDw };
enum { kReduceNone = 0, kReduceMean = 1, kReduceSum = 2 };

struct Params {
    int m_tiles, n_tiles, k_tiles, n_ext;  // tiles; columns in all (the last tile may be narrower)
    int n_pairs;                           // plane products: 1, or 6 for fp32
    int a0, b0;                            // added to the row coordinate of A and of B
    int *status;                           // set to 1 when a wait ran out
    // stats, grad
    int64_t n_rows, ignore_index;          // tokens in all
    int vocab;
    const void *bias;
    const int64_t *target;
    float *partial, *z_target;             // stats: [piece][max, sum, sum of z][row], z of the target
    unsigned *ticket;                      // stats: zeroed here for the loss kernel
    int smoothed;
    const float *lse, *grad;               // grad
    float smoothing;
    int reduction;
    uint16_t *dz;
    int64_t dz_ld, dz_plane;
    // dx, dw
    float *acc;                            // fp32 sums of earlier pieces (leading dimension acc_ld), or null
    int64_t acc_ld, row_offset, row_end;   // rows of the output: row_offset + tile row, below row_end
    int add, last;                         // acc holds earlier pieces; write `out`
    void *out;
    const float *count;
    const unsigned *grad_top;              // none: bits of max |g|
    const unsigned char *clean;            // dw: per 64 tokens, 1 = read the copy with ignored rows zeroed
};

__constant__ const int kPairA[6] = {2, 0, 1, 1, 0, 0}, kPairB[6] = {0, 2, 1, 0, 1, 0};

template <typename T> constexpr bool kIsHalf = std::is_same<T, __half>::value;
// fp16 dZ is kept times 2^14: |dz| <= 2, and probabilities down to 2^-28 stay normal numbers
template <typename T> constexpr float kDzScale = kIsHalf<T> ? 16384.f : 1.f;

template <typename T> __device__ constexpr uint32_t ce_instr(int n, bool a_mn, bool b_mn) {
    const uint32_t fmt = kIsHalf<T> ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(a_mn) << 15) | (static_cast<uint32_t>(b_mn) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kBM >> 4) << 24);
}

// Power of two at or below the largest |g| (its bits), so that g / scale is exact and below 2.
__device__ __forceinline__ float top_scale(unsigned bits) {
    const unsigned e = bits >> 23;
    if (e >= 255u) return __int_as_float(0x7fffffff);  // a gradient that is not finite: everything is NaN
    return e == 0u ? (bits ? 1.17549435e-38f : 1.f) : __uint_as_float(e << 23);
}

// The first tile of block c when t tiles are dealt in order to g blocks; the block that has tile i.
__host__ __device__ __forceinline__ int first_tile(int64_t t, int g, int c) { return static_cast<int>(t * c / g); }
__host__ __device__ __forceinline__ int block_of_tile(int64_t t, int g, int64_t i) {
    return static_cast<int>(((i + 1) * g + t - 1) / t) - 1;
}

__device__ __forceinline__ void st_global_v8(void *p, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (kIsHalf<T>) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
// The next bf16 plane of a, b (truncated, so what is left is exact); a and b become what is left.
__device__ __forceinline__ uint32_t take_plane(float &a, float &b) {
    const uint32_t ha = __float_as_uint(a) & 0xFFFF0000u, hb = __float_as_uint(b) & 0xFFFF0000u;
    const uint32_t word = (ha >> 16) | hb;
    a = isfinite(a) ? a - __uint_as_float(ha) : 0.f;
    b = isfinite(b) ? b - __uint_as_float(hb) : 0.f;
    return word;
}

// 32 neighbouring results of one row to the output: 32-byte stores where the row's address allows, else 4 elements, else one.
template <typename T> __device__ __forceinline__ void store_row(T *row, int64_t row_bytes, int col, int n, const float (&v)[32]) {
    T *p = row + col;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(row_bytes);
    if (n >= 32 && at % 32 == 0) {
#pragma unroll
        for (int u = 0; u < 32 * static_cast<int>(sizeof(T)) / 32; ++u) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[u * 8 + i]);
                else w[i] = pack2<T>(v[u * 16 + 2 * i], v[u * 16 + 2 * i + 1]);
            }
            st_global_v8(reinterpret_cast<char *>(p) + 32 * u, w);
        }
    } else if (at % (4 * sizeof(T)) == 0) {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (4 * u + 4 <= n) {
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4 *>(p + 4 * u) = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
                } else {
                    uint2 w;
                    w.x = pack2<T>(v[4 * u], v[4 * u + 1]);
                    w.y = pack2<T>(v[4 * u + 2], v[4 * u + 3]);
                    *reinterpret_cast<uint2 *>(p + 4 * u) = w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * u + i < n) p[4 * u + i] = from_acc<T>(v[4 * u + i]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < n) p[i] = from_acc<T>(v[i]);
    }
}

// A block's tiles: stats has consecutive ones (a row's running sums go from tile to tile), the others every gridDim-th.
template <int kKind> struct Tiles {
    int64_t total;
    int at, end, step;
    __device__ explicit Tiles(const Params &p) {
        total = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
        const int g = gridDim.x, c = blockIdx.x;
        at = kKind == kStats ? first_tile(total, g, c) : c;
        end = kKind == kStats ? first_tile(total, g, c + 1) : static_cast<int>(total);
        step = kKind == kStats ? 1 : g;
    }
};

// Barrier of the finishing warps that also says whether any of their threads gave up.
__device__ __forceinline__ bool finish_barrier_or(bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.b32 %0, 1, 0, q;\n\t}\n"
                 : "=r"(r)
                 : "r"(static_cast<uint32_t>(v))
                 : "memory");
    return r;
}
static_assert(kFinishWarps * 32 == 256, "finish_barrier_or names its thread count");

template <typename T, int kKind>
__global__ void __launch_bounds__(kThreads, 1)
linear_ce_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_b2, const Params p) {
    constexpr bool kAMn = kKind == kDw, kBMn = kKind == kDx || kKind == kDw;
    constexpr bool kPrecise = std::is_same<T, float>::value;
    extern __shared__ unsigned char smem_raw[];
    __shared__ int stop_flag;
    volatile int *stop = &stop_flag;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char *sm = smem_raw + (base - raw);
    float *s_bias = reinterpret_cast<float *>(sm + kStages * kStageBytes);  // [2][256]
    const uint32_t bars = base + kStages * kStageBytes + 2 * kBN * 4;
    const uint32_t bar_full = bars, bar_empty = bars + 8 * kStages, bar_tfull = bars + 16 * kStages,
                   bar_tempty = bar_tfull + 16, bar_drain = bar_tempty + 16, tmem_slot = bar_drain + 8;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        stop_flag = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_tfull + 8 * b, 1);
            mbar_init(bar_tempty + 8 * b, kFinishWarps);
        }
        mbar_init(bar_drain, 1);
        fence_mbar_init();
        prefetch_map(&map_a);
        prefetch_map(&map_b);
        if (kKind == kStats && blockIdx.x == 0) {
            *p.ticket = 0u;
            *p.status = 0;
        }
    }
    if (warp == kFinishWarps + 1) tmem_alloc(tmem_slot, 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + (tmem_slot - base));
    Tiles<kKind> tiles(p);
    const int steps = p.n_pairs * p.k_tiles;

    if (warp == kFinishWarps) {
        if (lane == 0) {  // ---- loads
            int s = 0;
            uint32_t phase = 0, issued = 0;
            bool ok = true;
            for (int t = tiles.at; ok && t < tiles.end; t += tiles.step) {
                const int m = t / p.n_tiles, n = t % p.n_tiles;
                const int cols = min(kBN, p.n_ext - n * kBN), chunks = (cols + 63) / 64;
                for (int step = 0; step < steps; ++step) {
                    const int pair = p.n_pairs == 1 ? 5 : step / p.k_tiles, k = step % p.k_tiles;
                    const int pa = kPairA[pair], pb = kPairB[pair];
                    ok = mbar_wait_or_stop(bar_empty + 8 * s, phase ^ 1u, stop);
                    if (!ok) break;
                    const uint32_t a = base + s * kStageBytes, b = a + kABytes, full = bar_full + 8 * s;
                    mbar_expect(full, kABytes + (kBMn ? chunks * kChunkBytes : kBBytes));
                    if constexpr (kAMn) {
                        tma_load(a, &map_a, m * kBM, p.a0 + k * kBK, pa, full);
                        tma_load(a + kChunkBytes, &map_a, m * kBM + 64, p.a0 + k * kBK, pa, full);
                    } else {
                        tma_load(a, &map_a, k * kBK, p.a0 + m * kBM, pa, full);
                    }
                    if constexpr (kBMn) {
                        const bool copy = kKind == kDw && p.clean && p.clean[p.b0 / kBK + k];
                        for (int c = 0; c < chunks; ++c)
                            tma_load(b + c * kChunkBytes, copy ? &map_b2 : &map_b, n * kBN + 64 * c, p.b0 + k * kBK, pb, full);
                    } else {
                        tma_load(b, &map_b, k * kBK, p.b0 + n * kBN, pb, full);
                    }
                    ++issued;
                    if (++s == kStages) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok) {  // the last loads of every stage land before the block ends
                for (int i = 0; i < kStages; ++i) {
                    if (issued <= static_cast<uint32_t>(i)) break;
                    const uint32_t last = (issued - 1 - i) / kStages;
                    const uint32_t bar = bar_full + 8 * ((issued - 1 - i) % kStages);
                    const long long start = clock64();
                    while (!mbar_try(bar, last & 1u) && clock64() - start < kWaitCycles) {}
                }
            }
        }
    } else if (warp == kFinishWarps + 1) {
        if (lane == 0) {  // ---- products
            int s = 0, buf = 0;
            uint32_t phase = 0, tphase = 0;
            bool ok = true;
            for (int t = tiles.at; ok && t < tiles.end; t += tiles.step) {
                const int n = t % p.n_tiles;
                const int cols = (min(kBN, p.n_ext - n * kBN) + 31) / 32 * 32;
                const uint32_t instr = ce_instr<T>(cols, kAMn, kBMn), d = tmem + buf * kBN;
                ok = mbar_wait_or_stop(bar_tempty + 8 * buf, tphase ^ 1u, stop);
                if (!ok) break;
                fence_after_sync();
                for (int step = 0; step < steps; ++step) {
                    ok = mbar_wait_or_stop(bar_full + 8 * s, phase, stop);
                    if (!ok) break;
                    fence_after_sync();
                    const uint32_t a = base + s * kStageBytes, b = a + kABytes;
#pragma unroll
                    for (int ks = 0; ks < kBK / 16; ++ks)
                        mma_ss(d, kAMn ? desc_mnmajor(a, ks) : desc_kmajor(a, ks), kBMn ? desc_mnmajor(b, ks) : desc_kmajor(b, ks),
                               instr, step > 0 || ks > 0);
                    mma_commit(bar_empty + 8 * s);
                    if (++s == kStages) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                mma_commit(bar_tfull + 8 * buf);
                if (++buf == 2) {
                    buf = 0;
                    tphase ^= 1u;
                }
            }
            if (!ok) {  // products under way end before the tensor memory is freed
                mma_commit(bar_drain);
                const long long start = clock64();
                while (!mbar_try(bar_drain, 0u) && clock64() - start < kWaitCycles) {}
            }
        }
    } else {  // ---- finishing: warp % 4 names the tile's 32 rows, warp / 4 its half of the columns
        const int quarter = warp & 3, half = warp >> 2, trow = quarter * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        int buf = 0, parity = 0, row_m = -1;
        uint32_t tphase = 0;
        float run_max = -INFINITY, run_sum = 0.f, run_z = 0.f;
        int tgt = -1;
        float row_lse = 0.f, row_g = 0.f;
        float scale = 1.f;
        if constexpr (kKind == kDx || kKind == kDw) {
            if (p.last) {
                if (p.reduction == kReduceNone) scale = top_scale(*p.grad_top);
                else scale = *p.grad;
                if (p.reduction == kReduceMean) scale = *p.count > 0.f ? scale / *p.count : 0.f;
                scale *= 1.f / kDzScale<T>;
            }
        }
        for (int t = tiles.at; t < tiles.end; t += tiles.step) {
            const int m = t / p.n_tiles, n = t % p.n_tiles;
            const int cols = min(kBN, p.n_ext - n * kBN);
            bool ok;
            const float *bias = s_bias + parity * kBN;
            if constexpr (kKind == kStats || kKind == kGrad) {
                const int col = n * kBN + tid;  // 256 finishing threads, 256 columns
                float b = -INFINITY;
                if (col < p.n_ext) {
                    const int64_t v = p.b0 + col;
                    if constexpr (kPrecise) b = p.bias ? static_cast<const float *>(p.bias)[v] : 0.f;
                    else b = p.bias ? to_acc<T>(static_cast<const T *>(p.bias)[v]) : 0.f;
                }
                s_bias[parity * kBN + tid] = b;
                parity ^= 1;
                if (m != row_m) {
                    row_m = m;
                    const int64_t row = p.a0 + static_cast<int64_t>(m) * kBM + trow;
                    const bool live = row < p.n_rows;
                    const int64_t target = live ? p.target[row] : p.ignore_index;
                    const bool counted = live && target != p.ignore_index;
                    tgt = counted && target >= 0 && target < p.vocab ? static_cast<int>(target) : -1;
                    if constexpr (kKind == kStats) {
                        run_max = -INFINITY;
                        run_sum = run_z = 0.f;
                    } else {
                        row_lse = live ? p.lse[row] : 0.f;
                        row_g = 0.f;
                        if (counted) {
                            row_g = 1.f;
                            if (p.reduction == kReduceNone) row_g = p.grad[row] * (1.f / top_scale(*p.grad_top));
                            if (tgt < 0) row_g = __int_as_float(0x7fffffff);  // no such class: the gradients say so
                            row_g *= kDzScale<T>;
                        }
                    }
                }
                ok = mbar_wait_or_stop(bar_tfull + 8 * buf, tphase, stop);
                ok = !finish_barrier_or(!ok);  // s_bias is whole, and all these warps go on or none does
            } else {
                ok = mbar_wait_or_stop(bar_tfull + 8 * buf, tphase, stop);
                ok = __all_sync(0xffffffffu, ok);
            }
            if (!ok) break;
            fence_after_sync();
            const uint32_t acc = tmem + lanes + buf * kBN;
            for (int c0 = half * (kBN / 2); c0 < (half + 1) * (kBN / 2) && c0 < cols; c0 += 32) {
                uint32_t r[32];
                __syncwarp();
                tmem_ld32(acc + c0, r);
                tmem_ld_wait();
                if constexpr (kKind == kStats || kKind == kGrad) {
                    float z[32];
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 b = *reinterpret_cast<const float4 *>(bias + c0 + i);
                        z[i] = __uint_as_float(r[i]) + b.x;
                        z[i + 1] = __uint_as_float(r[i + 1]) + b.y;
                        z[i + 2] = __uint_as_float(r[i + 2]) + b.z;
                        z[i + 3] = __uint_as_float(r[i + 3]) + b.w;
                    }
                    const int local = tgt - (p.b0 + n * kBN + c0);  // the target's place in these 32, if it is there
                    const bool here = tgt >= 0 && local >= 0 && local < 32;
                    if constexpr (kKind == kStats) {
                        float top = z[0];
#pragma unroll
                        for (int i = 1; i < 32; ++i) top = fmaxf(top, z[i]);
                        if (top > run_max) {
                            run_sum *= ex2((run_max - top) * kLog2e);
                            run_max = top;
                        }
                        const float m0 = run_max == -INFINITY ? 0.f : run_max, m2 = m0 * kLog2e;
                        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            sum[i & 3] += kPrecise ? ex2((z[i] - m0) * kLog2e) : ex2(fmaf(z[i], kLog2e, -m2));
                        run_sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                        if (p.smoothed) {
                            float total = 0.f;
#pragma unroll
                            for (int i = 0; i < 32; ++i) total += c0 + i < cols ? z[i] : 0.f;
                            run_z += total;
                        }
                        if (here) {
                            float zt = 0.f;
#pragma unroll
                            for (int i = 0; i < 32; ++i) zt = i == local ? z[i] : zt;
                            p.z_target[p.a0 + static_cast<int64_t>(m) * kBM + trow] = zt;
                        }
                    } else {
                        const float l2 = row_lse * kLog2e, uniform = p.smoothing / static_cast<float>(p.vocab) * row_g;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float prob = kPrecise ? ex2((z[i] - row_lse) * kLog2e) : ex2(fmaf(z[i], kLog2e, -l2));
                            z[i] = row_g == 0.f ? 0.f : fmaf(prob, row_g, -uniform);
                        }
                        if (here) {
                            const float sub = (1.f - p.smoothing) * row_g;
#pragma unroll
                            for (int i = 0; i < 32; ++i) z[i] -= i == local ? sub : 0.f;
                        }
                        // the buffer's rows and columns are padded to whole tiles
                        uint16_t *at = p.dz + (static_cast<int64_t>(m) * kBM + trow) * p.dz_ld + n * kBN + c0;
#pragma unroll
                        for (int plane = 0; plane < (kPrecise ? 3 : 1); ++plane) {
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                uint32_t w[8];
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    if constexpr (kPrecise) w[i] = take_plane(z[16 * u + 2 * i], z[16 * u + 2 * i + 1]);
                                    else w[i] = pack2<T>(z[16 * u + 2 * i], z[16 * u + 2 * i + 1]);
                                }
                                st_global_v8(at + plane * p.dz_plane + 16 * u, w);
                            }
                        }
                    }
                } else {
                    const int64_t row = p.row_offset + static_cast<int64_t>(m) * kBM + trow;
                    if (row < p.row_end) {
                        float v[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
                        const int col = n * kBN + c0, left = p.n_ext - col;
                        float *sums = p.acc ? p.acc + row * p.acc_ld + col : nullptr;
                        if (p.add) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] += i < left ? sums[i] : 0.f;
                        }
                        if (p.last) {
                            const bool ignored = kKind == kDx && p.target[row] == p.ignore_index;
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = ignored ? 0.f : v[i] * scale;
                            store_row(static_cast<T *>(p.out) + row * p.n_ext, p.n_ext * static_cast<int64_t>(sizeof(T)), col, left, v);
                        } else {
                            store_row(p.acc + row * p.acc_ld, p.acc_ld * 4, col, left, v);
                        }
                    }
                }
            }
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_tempty + 8 * buf);
            if (++buf == 2) {
                buf = 0;
                tphase ^= 1u;
            }
            if constexpr (kKind == kStats) {
                if (n == p.n_tiles - 1 || t + 1 == tiles.end) {  // the last tile of these rows in this block
                    const int64_t rows_padded = static_cast<int64_t>(p.m_tiles) * kBM;
                    const int piece = blockIdx.x - block_of_tile(tiles.total, gridDim.x, static_cast<int64_t>(m) * p.n_tiles);
                    float *at = p.partial + (static_cast<int64_t>(piece) * 2 + half) * 3 * rows_padded + static_cast<int64_t>(m) * kBM + trow;
                    at[0] = run_max;
                    at[rows_padded] = run_sum;
                    at[2 * rows_padded] = run_z;
                }
            }
        }
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    if (warp == kFinishWarps + 1) {
        fence_after_sync();
        tmem_free(tmem, 512);
    }
    if (tid == 0 && *stop) *p.status = 1;
}

// ---- the loss from the pieces: kLanes threads a row, one row or many pieces a thread.
constexpr int kLossThreads = 256;
struct LossParams {
    const float *partial, *z_target;
    const int64_t *target;
    int64_t n_rows, ignore_index;
    int m_tiles, n_tiles, grid, vocab, reduction;
    float smoothing;
    float *loss, *lse, *count;
    double *block_sums;  // [blocks][sum, count]
    unsigned *ticket;
    const int *status;
};

template <int kLanes> __global__ void __launch_bounds__(kLossThreads) linear_ce_loss_kernel(const LossParams p) {
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * kLossThreads + threadIdx.x) / kLanes;
    const int lane = threadIdx.x % kLanes;
    float loss = 0.f;
    bool counted = false;
    if (row < p.n_rows) {
        const int64_t total = static_cast<int64_t>(p.m_tiles) * p.n_tiles, m = row / kBM, rows_padded = static_cast<int64_t>(p.m_tiles) * kBM;
        const int pieces = 2 * (block_of_tile(total, p.grid, (m + 1) * p.n_tiles - 1) - block_of_tile(total, p.grid, m * p.n_tiles) + 1);
        float top = -INFINITY, sum = 0.f, z = 0.f;
        for (int i = lane; i < pieces; i += kLanes) top = fmaxf(top, p.partial[static_cast<int64_t>(i) * 3 * rows_padded + row]);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        for (int i = lane; i < pieces; i += kLanes) {
            const float *at = p.partial + static_cast<int64_t>(i) * 3 * rows_padded + row;
            const float s = at[rows_padded];
            if (!(s == 0.f)) sum += s * exp2f((at[0] - top) * kLog2e);  // a piece without any finite logit has sum 0
            z += at[2 * rows_padded];
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            z += __shfl_xor_sync(0xffffffffu, z, o);
        }
        if (lane == 0) {
            const float lse = top + logf(sum);
            const int64_t target = p.target[row];
            counted = target != p.ignore_index;
            if (counted) {
                const bool known = target >= 0 && target < p.vocab;
                const float zt = known ? p.z_target[row] : __int_as_float(0x7fffffff);
                loss = lse - zt;
                if (p.smoothing != 0.f) loss += p.smoothing * (zt - z / static_cast<float>(p.vocab));
            }
            if (*p.status) loss = __int_as_float(0x7fffffff);
            if (p.lse) p.lse[row] = lse;
            if (p.reduction == kReduceNone) p.loss[row] = loss;
        }
    }
    if (p.reduction == kReduceNone) return;
    // sums in 64 bits: of the block, then (the block that ends last) of the blocks in their order
    __shared__ double sums[2][kLossThreads / 32];
    __shared__ bool last;
    auto block_sum = [&](double a, double b) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) {
            sums[0][threadIdx.x >> 5] = a;
            sums[1][threadIdx.x >> 5] = b;
        }
        __syncthreads();
        a = b = 0.0;
        for (int i = 0; i < kLossThreads / 32; ++i) {
            a += sums[0][i];
            b += sums[1][i];
        }
        return make_double2(a, b);
    };
    const double2 here = block_sum(loss, counted ? 1.0 : 0.0);
    if (threadIdx.x == 0) {
        p.block_sums[2 * blockIdx.x] = here.x;
        p.block_sums[2 * blockIdx.x + 1] = here.y;
        __threadfence();
        last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double a = 0.0, b = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += kLossThreads) {
        a += __ldcg(p.block_sums + 2 * i);
        b += __ldcg(p.block_sums + 2 * i + 1);
    }
    const double2 all = block_sum(a, b);
    if (threadIdx.x == 0) {
        *p.loss = static_cast<float>(p.reduction == kReduceMean ? all.x / all.y : all.x);
        if (p.count) *p.count = static_cast<float>(all.y);
    }
}

// ---- operands that TMA cannot read where they lie (fp32, rows or bases off 16 bytes): copied into rows of a multiple
// of 8 elements, fp32 as three bf16 planes.  Rows whose target is ignored (target given) are zeroed: their features
// may hold anything, and 0 * NaN would reach every gradient of W.
template <typename T>
__global__ void linear_ce_pack_kernel(const T *__restrict__ src, int64_t ld, int64_t rows, int dim, uint16_t *__restrict__ dst,
                                      int64_t dst_ld, int64_t plane, const int64_t *__restrict__ target, int64_t ignore_index) {
    const int64_t pieces = dst_ld / 8, total = rows * pieces;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t row = i / pieces;
        const int c = static_cast<int>(i % pieces) * 8;
        const bool skip = target && target[row] == ignore_index;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = !skip && c + j < dim ? to_acc<T>(src[row * ld + c + j]) : 0.f;
        constexpr int kPlanes = std::is_same<T, float>::value ? 3 : 1;
#pragma unroll
        for (int q = 0; q < kPlanes; ++q) {
            uint4 w;
            if constexpr (kPlanes == 3) {
                w.x = take_plane(v[0], v[1]);
                w.y = take_plane(v[2], v[3]);
                w.z = take_plane(v[4], v[5]);
                w.w = take_plane(v[6], v[7]);
            } else {
                w.x = pack2<T>(v[0], v[1]);
                w.y = pack2<T>(v[2], v[3]);
                w.z = pack2<T>(v[4], v[5]);
                w.w = pack2<T>(v[6], v[7]);
            }
            *reinterpret_cast<uint4 *>(dst + q * plane + row * dst_ld + c) = w;
        }
    }
}

// Per 64 tokens: whether any is ignored; their rows are then copied with the ignored ones zeroed, and the dW product
// reads the copy.  Where nothing is ignored nothing is copied.
__global__ void __launch_bounds__(256) linear_ce_clean_kernel(const uint16_t *__restrict__ x, int64_t ld, int64_t rows, int dim,
                                                              const int64_t *__restrict__ target, int64_t ignore_index,
                                                              uint16_t *__restrict__ copy, int64_t copy_ld,
                                                              unsigned char *__restrict__ clean) {
    __shared__ unsigned char skip[64];
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * 64;
    bool ignored = false;
    if (threadIdx.x < 64) {
        ignored = row0 + threadIdx.x < rows && target[row0 + threadIdx.x] == ignore_index;
        skip[threadIdx.x] = ignored;
    }
    const bool any = __syncthreads_or(ignored);
    if (threadIdx.x == 0) clean[blockIdx.x] = any;
    if (!any) return;
    const int pieces = (dim + 7) / 8;
    for (int i = threadIdx.x; i < 64 * pieces; i += 256) {
        const int r = i / pieces, c = i % pieces * 8;
        if (row0 + r >= rows) break;
        const uint16_t *from = x + (row0 + r) * ld + c;
        uint16_t *to = copy + (row0 + r) * copy_ld + c;
        if (c + 8 <= dim) {
            *reinterpret_cast<uint4 *>(to) = skip[r] ? make_uint4(0u, 0u, 0u, 0u) : *reinterpret_cast<const uint4 *>(from);
        } else {
            for (int j = 0; j < dim - c; ++j) to[j] = skip[r] ? uint16_t(0) : from[j];
        }
    }
}

// max |g| over the tokens that count, as bits (ordered like the numbers; a NaN is above all).
__global__ void linear_ce_top_kernel(const float *__restrict__ grad, const int64_t *__restrict__ target, int64_t rows,
                                     int64_t ignore_index, unsigned *__restrict__ top) {
    unsigned best = 0u;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < rows; i += static_cast<int64_t>(gridDim.x) * blockDim.x)
        if (target[i] != ignore_index) best = max(best, __float_as_uint(grad[i]) & 0x7FFFFFFFu);
    best = __reduce_max_sync(0xffffffffu, best);
    if ((threadIdx.x & 31) == 0) atomicMax(top, best);
}

// Column sums of a dZ piece over each 128 rows: thread per pair of columns.
template <typename T>
__global__ void __launch_bounds__(128) linear_ce_colsum_kernel(const uint16_t *__restrict__ dz, int64_t ld, int64_t plane, int rows,
                                                               int cols, float *__restrict__ out, int64_t out_ld) {
    const int c = (blockIdx.x * 128 + threadIdx.x) * 2;
    if (c >= cols) return;
    float a = 0.f, b = 0.f;
    for (int r = blockIdx.y * 128; r < min(rows, static_cast<int>(blockIdx.y) * 128 + 128); ++r) {
        constexpr int kPlanes = std::is_same<T, float>::value ? 3 : 1;
        float va = 0.f, vb = 0.f;
#pragma unroll
        for (int q = kPlanes - 1; q >= 0; --q) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(dz + q * plane + r * ld + c);
            if constexpr (kIsHalf<T>) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
                va += f.x;
                vb += f.y;
            } else {
                va += __uint_as_float(w << 16);
                vb += __uint_as_float(w & 0xFFFF0000u);
            }
        }
        a += va;
        b += vb;
    }
    out[blockIdx.y * out_ld + c] = a;
    if (c + 1 < cols) out[blockIdx.y * out_ld + c + 1] = b;
}

// d b of a piece: sums over its blocks of rows, added to those of earlier rows; the last one is scaled and stored.
template <typename T>
__global__ void __launch_bounds__(256) linear_ce_bias_kernel(const float *__restrict__ sums, int64_t ld, int blocks, int cols, float *acc,
                                                             int add, int last, T *__restrict__ out, Params p) {
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    __shared__ float s_part[8][32];
    float s = 0.f;
    if (c < cols)
        for (int r = part; r < blocks; r += 8) s += sums[r * ld + c];
    s_part[part][threadIdx.x & 31] = s;
    __syncthreads();
    if (part > 0 || c >= cols) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += s_part[i][threadIdx.x];
    if (add) s += acc[c];
    if (!last) {
        acc[c] = s;
        return;
    }
    float scale = p.reduction == kReduceNone ? top_scale(*p.grad_top) : *p.grad;
    if (p.reduction == kReduceMean) scale = *p.count > 0.f ? scale / *p.count : 0.f;
    out[c] = from_acc<T>(s * (scale / kDzScale<T>));
}

// A wait that ran out leaves results that mean nothing: say so in them.
template <typename T> __global__ void linear_ce_poison_kernel(const int *status, T *dx, T *dw, T *db) {
    if (*status) {
        const T nan = from_acc<T>(__int_as_float(0x7fffffff));
        if (dx) *dx = nan;
        if (dw) *dw = nan;
        if (db) *db = nan;
    }
}

// ---- host side
struct Operand {  // a matrix as TMA reads it
    const void *at;
    int64_t ld, plane;
};

bool tma_ready(const void *p, int64_t ld, int dtype) {
    return dtype != BPT_F32 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0;
}
int64_t ce_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Shape {
    int64_t n;
    int vocab, dim, dtype, planes;
    int64_t packed_ld;
    bool pack_x, pack_w;
    Shape(const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t n_, int vocab_, int dim_, int dtype_)
        : n(n_), vocab(vocab_), dim(dim_), dtype(dtype_), planes(dtype_ == BPT_F32 ? 3 : 1), packed_ld(ce_div(dim_, 8) * 8),
          pack_x(!tma_ready(x, ldx, dtype_)), pack_w(!tma_ready(w, ldw, dtype_)) {}
    int64_t m_tiles() const { return ce_div(n, kBM); }
    int v_tiles() const { return static_cast<int>(ce_div(vocab, kBN)); }
    int64_t packed(int64_t rows) const { return align_up(rows * packed_ld, 64) * planes; }
    int stats_grid() const { return static_cast<int>(std::min<int64_t>(kGrid, m_tiles() * v_tiles())); }
    int64_t pieces() const {  // blocks that share one block of rows, at most
        return std::min<int64_t>(stats_grid(), static_cast<int64_t>(v_tiles()) * stats_grid() / (m_tiles() * v_tiles()) + 2);
    }
};

struct ForwardSpace {
    float *partial, *z_target;
    double *block_sums;
    unsigned *ticket;
    int *status;
    uint16_t *x, *w;
    ForwardSpace(Workspace &ws, const Shape &s) {
        status = ws.take<int>(1);
        ticket = ws.take<unsigned>(1);
        block_sums = ws.take<double>(2 * ce_div(s.n * 32, kLossThreads));
        z_target = ws.take<float>(s.n);
        partial = ws.take<float>(s.pieces() * 2 * 3 * s.m_tiles() * kBM);
        x = s.pack_x ? ws.take<uint16_t>(s.packed(s.n)) : nullptr;
        w = s.pack_w ? ws.take<uint16_t>(s.packed(s.vocab)) : nullptr;
    }
};

// Bytes of dZ kept at a time.  It is written by one product and read by two, so it should stay in the 126 MB L2.
constexpr int64_t kDzBytes = 64 << 20;

struct BackwardSpace {
    int64_t rows, cols;  // tokens x vocabulary of a piece
    int64_t dz_ld, dz_plane, acc_ld;
    int *status;
    unsigned *grad_top;
    uint16_t *dz, *x, *w, *x_clean;
    unsigned char *clean;
    float *dx_acc, *dw_acc, *col_sums, *db_acc;
    BackwardSpace(Workspace &ws, const Shape &s, bool want_dx, bool want_dw, bool want_db) {
        // Pieces of rows x cols cells.  Cutting the vocabulary has dX pass through memory once a cut, cutting the
        // tokens dW: take the cheaper of the two, whole tiles, at least 1024 each way.
        const int64_t cells = kDzBytes / (2 * s.planes), n_pad = ce_div(s.n, kBM) * kBM, v_pad = ce_div(s.vocab, kBN) * kBN;
        rows = n_pad;
        cols = v_pad;
        if (n_pad * v_pad > cells) {
            int64_t best = -1;
            for (int64_t r = std::min<int64_t>(n_pad, 1024);; r = std::min(r * 2, n_pad)) {
                int64_t c = std::max<int64_t>(cells / r / kBN * kBN, 1024);
                c = std::min(c, v_pad);
                const int64_t row_cuts = ce_div(n_pad, r), col_cuts = ce_div(v_pad, c);
                const int64_t cost = (col_cuts - 1) * s.n + (row_cuts - 1) * s.vocab;
                if (r * c <= cells + cells / 8 && (best < 0 || cost < best)) {
                    best = cost;
                    rows = r;
                    cols = c;
                }
                if (r == n_pad) break;
            }
            if (best < 0) {
                rows = std::min<int64_t>(n_pad, 1024);
                cols = std::min<int64_t>(v_pad, std::max<int64_t>(1024, cells / rows / kBN * kBN));
            }
            // pieces of one size instead of a small last one
            rows = ce_div(ce_div(n_pad, kBM), ce_div(n_pad, rows)) * kBM;
            cols = ce_div(ce_div(v_pad, kBN), ce_div(v_pad, cols)) * kBN;
        }
        dz_ld = cols;
        dz_plane = rows * cols;
        acc_ld = ce_div(s.dim, 8) * 8;
        const bool own_acc = s.dtype == BPT_F32 && s.dim == acc_ld;  // fp32 sums can live in the output itself
        status = ws.take<int>(1);
        grad_top = ws.take<unsigned>(1);
        dz = ws.take<uint16_t>(dz_plane * s.planes);
        x = s.pack_x ? ws.take<uint16_t>(s.packed(s.n)) : nullptr;
        w = s.pack_w ? ws.take<uint16_t>(s.packed(s.vocab)) : nullptr;
        x_clean = !s.pack_x && want_dw ? ws.take<uint16_t>(s.n * ce_div(s.dim, 8) * 8) : nullptr;
        clean = !s.pack_x && want_dw ? ws.take<unsigned char>(ce_div(s.n, 64)) : nullptr;
        dx_acc = want_dx && !own_acc && cols < s.vocab ? ws.take<float>(s.n * acc_ld) : nullptr;
        dw_acc = want_dw && !own_acc && rows < s.n ? ws.take<float>(s.vocab * acc_ld) : nullptr;
        col_sums = want_db ? ws.take<float>(rows / kBM * cols) : nullptr;
        db_acc = want_db && rows < s.n ? ws.take<float>(s.vocab) : nullptr;
    }
};

template <typename T, int kKind>
int launch_ce(const CUtensorMap &a, const CUtensorMap &b, const CUtensorMap &b2, const Params &p, cudaStream_t stream) {
    const int64_t total = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
    BPT_CUDA(cudaFuncSetAttribute(linear_ce_kernel<T, kKind>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    linear_ce_kernel<T, kKind><<<static_cast<unsigned>(std::min<int64_t>(kGrid, total)), kThreads, kSmemBytes, stream>>>(a, b, b2, p);
    BPT_LAUNCH_CHECK();
    return BPT_OK;
}

template <typename T>
int pack_operand(const void *src, int64_t ld, int64_t rows, const Shape &s, uint16_t *dst, const int64_t *target, int64_t ignore_index,
                 cudaStream_t stream, Operand *out) {
    out->at = dst;
    out->ld = s.packed_ld;
    out->plane = align_up(rows * s.packed_ld, 64);
    const int64_t blocks = std::min<int64_t>(ce_div(rows * (s.packed_ld / 8), 256), 148 * 16);
    linear_ce_pack_kernel<T><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<const T *>(src), ld, rows, s.dim, dst,
                                                                               s.packed_ld, out->plane, target, ignore_index);
    BPT_LAUNCH_CHECK();
    return BPT_OK;
}

#define BPT_TRY(call)                  \
    do {                               \
        const int rc__ = (call);       \
        if (rc__ != BPT_OK) return rc__; \
    } while (0)

struct Call {
    const void *x, *w, *bias;
    int64_t ldx, ldw;
    const int64_t *target;
    int64_t ignore_index;
    float smoothing;
    int reduction;
};

template <typename T> int ce_forward(const Shape &s, const Call &c, ForwardSpace &f, float *loss, float *lse, float *count, cudaStream_t stream) {
    constexpr bool kHalf = kIsHalf<T>;
    Operand x{c.x, c.ldx, 0}, w{c.w, c.ldw, 0};
    if (s.pack_x) BPT_TRY(pack_operand<T>(c.x, c.ldx, s.n, s, f.x, nullptr, 0, stream, &x));
    if (s.pack_w) BPT_TRY(pack_operand<T>(c.w, c.ldw, s.vocab, s, f.w, nullptr, 0, stream, &w));
    CUtensorMap ma, mb;
    BPT_TRY(make_map(&ma, kHalf, x.at, s.n, s.dim, x.ld, s.planes, x.plane, kBM));
    BPT_TRY(make_map(&mb, kHalf, w.at, s.vocab, s.dim, w.ld, s.planes, w.plane, kBN));
    Params p{};
    p.m_tiles = static_cast<int>(s.m_tiles());
    p.n_tiles = s.v_tiles();
    p.k_tiles = static_cast<int>(ce_div(s.dim, kBK));
    p.n_ext = s.vocab;
    p.n_pairs = s.planes == 3 ? 6 : 1;
    p.status = f.status;
    p.n_rows = s.n;
    p.ignore_index = c.ignore_index;
    p.vocab = s.vocab;
    p.bias = c.bias;
    p.target = c.target;
    p.partial = f.partial;
    p.z_target = f.z_target;
    p.ticket = f.ticket;
    p.smoothed = c.smoothing != 0.f;
    BPT_TRY((launch_ce<T, kStats>(ma, mb, mb, p, stream)));
    LossParams l{};
    l.partial = f.partial;
    l.z_target = f.z_target;
    l.target = c.target;
    l.n_rows = s.n;
    l.ignore_index = c.ignore_index;
    l.m_tiles = p.m_tiles;
    l.n_tiles = p.n_tiles;
    l.grid = s.stats_grid();
    l.vocab = s.vocab;
    l.reduction = c.reduction;
    l.smoothing = c.smoothing;
    l.loss = loss;
    l.lse = lse;
    l.count = count;
    l.block_sums = f.block_sums;
    l.ticket = f.ticket;
    l.status = f.status;
    // a row of many pieces (few rows, so many blocks shared each) is merged by a warp
    if (s.pieces() > 8) linear_ce_loss_kernel<32><<<static_cast<unsigned>(ce_div(s.n * 32, kLossThreads)), kLossThreads, 0, stream>>>(l);
    else linear_ce_loss_kernel<1><<<static_cast<unsigned>(ce_div(s.n, kLossThreads)), kLossThreads, 0, stream>>>(l);
    BPT_LAUNCH_CHECK();
    return BPT_OK;
}

template <typename T>
int ce_backward(const Shape &s, const Call &c, BackwardSpace &f, const float *lse, const float *count, const float *grad, void *dx,
                void *dw, void *db, cudaStream_t stream) {
    constexpr bool kHalf = kIsHalf<T>;
    constexpr bool kFloat = std::is_same<T, float>::value;
    Operand x{c.x, c.ldx, 0}, w{c.w, c.ldw, 0};
    BPT_CUDA(cudaMemsetAsync(f.status, 0, sizeof(int), stream));
    if (s.pack_x) BPT_TRY(pack_operand<T>(c.x, c.ldx, s.n, s, f.x, c.target, c.ignore_index, stream, &x));
    if (s.pack_w) BPT_TRY(pack_operand<T>(c.w, c.ldw, s.vocab, s, f.w, nullptr, 0, stream, &w));
    const int64_t clean_ld = ce_div(s.dim, 8) * 8;
    if (f.clean) {
        linear_ce_clean_kernel<<<static_cast<unsigned>(ce_div(s.n, 64)), 256, 0, stream>>>(
            static_cast<const uint16_t *>(c.x), c.ldx, s.n, s.dim, c.target, c.ignore_index, f.x_clean, clean_ld, f.clean);
        BPT_LAUNCH_CHECK();
    }
    if (c.reduction == kReduceNone) {
        BPT_CUDA(cudaMemsetAsync(f.grad_top, 0, sizeof(unsigned), stream));
        linear_ce_top_kernel<<<static_cast<unsigned>(std::min<int64_t>(ce_div(s.n, 256), 148)), 256, 0, stream>>>(grad, c.target, s.n,
                                                                                                               c.ignore_index, f.grad_top);
        BPT_LAUNCH_CHECK();
    }
    CUtensorMap x_rows, w_rows, w_cols, x_cols, x_clean;
    BPT_TRY(make_map(&x_rows, kHalf, x.at, s.n, s.dim, x.ld, s.planes, x.plane, kBM));
    BPT_TRY(make_map(&w_rows, kHalf, w.at, s.vocab, s.dim, w.ld, s.planes, w.plane, kBN));
    BPT_TRY(make_map(&w_cols, kHalf, w.at, s.vocab, s.dim, w.ld, s.planes, w.plane, 64));
    BPT_TRY(make_map(&x_cols, kHalf, x.at, s.n, s.dim, x.ld, s.planes, x.plane, 64));
    x_clean = x_cols;
    if (f.clean) BPT_TRY(make_map(&x_clean, kHalf, f.x_clean, s.n, s.dim, clean_ld, 1, 0, 64));
    Params p{};
    p.n_pairs = s.planes == 3 ? 6 : 1;
    p.status = f.status;
    p.n_rows = s.n;
    p.ignore_index = c.ignore_index;
    p.vocab = s.vocab;
    p.bias = c.bias;
    p.target = c.target;
    p.lse = lse;
    p.grad = grad;
    p.grad_top = f.grad_top;
    p.count = count;
    p.smoothing = c.smoothing;
    p.reduction = c.reduction;
    p.dz = f.dz;
    p.dz_ld = f.dz_ld;
    p.dz_plane = f.dz_plane;
    const bool own_acc = kFloat && s.dim == f.acc_ld;
    for (int64_t n0 = 0; n0 < s.n; n0 += f.rows) {
        const int64_t rows = std::min(f.rows, s.n - n0);
        const bool last_rows = n0 + f.rows >= s.n;
        for (int64_t v0 = 0; v0 < s.vocab; v0 += f.cols) {
            const int64_t cols = std::min<int64_t>(f.cols, s.vocab - v0);
            const bool last_cols = v0 + f.cols >= s.vocab;
            CUtensorMap dz_rows, dz_cols;
            BPT_TRY(make_map(&dz_rows, kHalf, f.dz, rows, cols, f.dz_ld, s.planes, f.dz_plane, kBM));
            BPT_TRY(make_map(&dz_cols, kHalf, f.dz, rows, cols, f.dz_ld, s.planes, f.dz_plane, 64));
            Params g = p;
            g.m_tiles = static_cast<int>(ce_div(rows, kBM));
            g.n_tiles = static_cast<int>(ce_div(cols, kBN));
            g.k_tiles = static_cast<int>(ce_div(s.dim, kBK));
            g.n_ext = static_cast<int>(cols);
            g.a0 = static_cast<int>(n0);
            g.b0 = static_cast<int>(v0);
            BPT_TRY((launch_ce<T, kGrad>(x_rows, w_rows, w_rows, g, stream)));
            if (dx) {
                Params q = p;
                q.m_tiles = g.m_tiles;
                q.n_tiles = static_cast<int>(ce_div(s.dim, kBN));
                q.k_tiles = static_cast<int>(ce_div(cols, kBK));
                q.n_ext = s.dim;
                q.b0 = static_cast<int>(v0);
                q.acc = own_acc ? static_cast<float *>(dx) : f.dx_acc;
                q.acc_ld = f.acc_ld;
                q.row_offset = n0;
                q.row_end = n0 + rows;
                q.add = v0 > 0;
                q.last = last_cols;
                q.out = dx;
                BPT_TRY((launch_ce<T, kDx>(dz_rows, w_cols, w_cols, q, stream)));
            }
            if (dw) {
                Params q = p;
                q.m_tiles = static_cast<int>(ce_div(cols, kBM));
                q.n_tiles = static_cast<int>(ce_div(s.dim, kBN));
                q.k_tiles = static_cast<int>(ce_div(rows, kBK));
                q.n_ext = s.dim;
                q.b0 = static_cast<int>(n0);
                q.acc = own_acc ? static_cast<float *>(dw) : f.dw_acc;
                q.acc_ld = f.acc_ld;
                q.row_offset = v0;
                q.row_end = v0 + cols;
                q.add = n0 > 0;
                q.last = last_rows;
                q.out = dw;
                q.clean = f.clean;
                BPT_TRY((launch_ce<T, kDw>(dz_cols, x_cols, x_clean, q, stream)));
            }
            if (db) {
                const int blocks = static_cast<int>(ce_div(rows, kBM));
                linear_ce_colsum_kernel<T><<<dim3(static_cast<unsigned>(ce_div(cols, 256)), blocks), 128, 0, stream>>>(
                    f.dz, f.dz_ld, f.dz_plane, static_cast<int>(rows), static_cast<int>(cols), f.col_sums, f.cols);
                BPT_LAUNCH_CHECK();
                linear_ce_bias_kernel<T><<<static_cast<unsigned>(ce_div(cols, 32)), 256, 0, stream>>>(
                    f.col_sums, f.cols, blocks, static_cast<int>(cols), f.db_acc ? f.db_acc + v0 : nullptr, n0 > 0, last_rows,
                    static_cast<T *>(db) + v0, p);
                BPT_LAUNCH_CHECK();
            }
        }
    }
    linear_ce_poison_kernel<T><<<1, 1, 0, stream>>>(f.status, static_cast<T *>(dx), static_cast<T *>(dw), static_cast<T *>(db));
    BPT_LAUNCH_CHECK();
    return BPT_OK;
}

int check_call(const char *name, const void *x, int64_t ldx, const void *w, int64_t ldw, const int64_t *target, double smoothing,
               int reduction, int64_t n, int vocab, int dim, int dtype) {
    BPT_CHECK_ARG(n >= 0 && n < (int64_t(1) << 31) - kBM, "%s: bad token count", name);
    BPT_CHECK_ARG(vocab >= 1 && vocab <= (1 << 30) && dim >= 1 && dim <= (1 << 20), "%s: bad vocabulary or dim (%d, %d)", name, vocab, dim);
    BPT_CHECK_ARG(ldx >= dim && ldw >= dim, "%s: a row stride is smaller than dim", name);
    BPT_CHECK_ARG(smoothing >= 0.0 && smoothing <= 1.0, "%s: label smoothing must be in [0, 1]", name);
    BPT_CHECK_ARG(reduction >= kReduceNone && reduction <= kReduceSum, "%s: unknown reduction %d", name, reduction);
    BPT_CHECK_ARG(ce_div(n, kBM) * ce_div(vocab, kBN) < (int64_t(1) << 30), "%s: too many cells", name);
    if (dtype != BPT_F32 && dtype != BPT_BF16 && dtype != BPT_F16) return fail(BPT_ERR_UNSUPPORTED, "%s: dtype %d is not supported", name, dtype);
    BPT_CHECK_ARG(n == 0 || (x && w && target), "%s: null tensor", name);
    return BPT_OK;
}
bool sizes_ok(int64_t n, int vocab, int dim, int dtype) {
    return n >= 1 && n < (int64_t(1) << 31) - kBM && vocab >= 1 && vocab <= (1 << 30) && dim >= 1 && dim <= (1 << 20) &&
           (dtype == BPT_F32 || dtype == BPT_BF16 || dtype == BPT_F16);
}

// Workspace that only counts: take() moves `used` on as if there were room.
size_t counted(Workspace &ws) { return ws.used + 256; }
}  // namespace
}  // namespace bpt

using namespace bpt;

extern "C" size_t bpt_linear_ce_forward_workspace_bytes(const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t n, int vocab,
                                                        int dim, int dtype) {
    if (!sizes_ok(n, vocab, dim, dtype)) return 0;
    Workspace ws(reinterpret_cast<void *>(256), ~size_t(0) / 2);
    ForwardSpace f(ws, Shape(x, ldx, w, ldw, n, vocab, dim, dtype));
    return counted(ws);
}

extern "C" int bpt_linear_ce_forward(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const int64_t *target,
                                     int64_t ignore_index, double smoothing, int reduction, float *loss, float *lse, float *count,
                                     int64_t n, int vocab, int dim, int dtype, void *workspace, size_t workspace_bytes,
                                     bpt_stream_t stream_) {
    BPT_TRY(check_call("linear_ce_forward", x, ldx, w, ldw, target, smoothing, reduction, n, vocab, dim, dtype));
    cudaStream_t stream = as_stream(stream_);
    if (n == 0) {  // the sum over no tokens is 0, their mean 0 / 0
        if (reduction == kReduceNone) return BPT_OK;
        BPT_CHECK_ARG(loss, "linear_ce_forward: null tensor");
        BPT_CUDA(cudaMemsetAsync(loss, reduction == kReduceMean ? 0xFF : 0, sizeof(float), stream));
        if (count) BPT_CUDA(cudaMemsetAsync(count, 0, sizeof(float), stream));
        return BPT_OK;
    }
    BPT_CHECK_ARG(loss, "linear_ce_forward: null tensor");
    const Shape s(x, ldx, w, ldw, n, vocab, dim, dtype);
    const uintptr_t at = reinterpret_cast<uintptr_t>(workspace), up = align_up(at, 256) - at;
    Workspace ws(workspace ? static_cast<char *>(workspace) + up : nullptr, workspace_bytes > up ? workspace_bytes - up : 0);
    ForwardSpace f(ws, s);
    if (!workspace || !ws.ok()) return fail(BPT_ERR_WORKSPACE, "linear_ce_forward: workspace of %zu bytes is too small", workspace_bytes);
    const Call c{x, w, bias, ldx, ldw, target, ignore_index, static_cast<float>(smoothing), reduction};
    switch (dtype) {
        case BPT_F32: return ce_forward<float>(s, c, f, loss, lse, count, stream);
        case BPT_BF16: return ce_forward<__nv_bfloat16>(s, c, f, loss, lse, count, stream);
        default: return ce_forward<__half>(s, c, f, loss, lse, count, stream);
    }
}

extern "C" size_t bpt_linear_ce_backward_workspace_bytes(const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t n, int vocab,
                                                         int dim, int dtype, int want_dx, int want_dw, int want_db) {
    if (!sizes_ok(n, vocab, dim, dtype)) return 0;
    Workspace ws(reinterpret_cast<void *>(256), ~size_t(0) / 2);
    BackwardSpace f(ws, Shape(x, ldx, w, ldw, n, vocab, dim, dtype), want_dx, want_dw, want_db);
    return counted(ws);
}

extern "C" int bpt_linear_ce_backward(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const int64_t *target,
                                      int64_t ignore_index, double smoothing, int reduction, const float *lse, const float *count,
                                      const float *grad, void *dx, void *dw, void *db, int64_t n, int vocab, int dim, int dtype,
                                      void *workspace, size_t workspace_bytes, bpt_stream_t stream_) {
    BPT_TRY(check_call("linear_ce_backward", x, ldx, w, ldw, target, smoothing, reduction, n, vocab, dim, dtype));
    cudaStream_t stream = as_stream(stream_);
    if (!dx && !dw && !db) return BPT_OK;
    const size_t elem = dtype == BPT_F32 ? 4 : 2;
    if (n == 0) {
        if (dw) BPT_CUDA(cudaMemsetAsync(dw, 0, elem * vocab * dim, stream));
        if (db) BPT_CUDA(cudaMemsetAsync(db, 0, elem * vocab, stream));
        return BPT_OK;
    }
    BPT_CHECK_ARG(lse && grad, "linear_ce_backward: null tensor");
    BPT_CHECK_ARG(reduction != kReduceMean || count, "linear_ce_backward: the mean needs the forward's count");
    const Shape s(x, ldx, w, ldw, n, vocab, dim, dtype);
    const uintptr_t at = reinterpret_cast<uintptr_t>(workspace), up = align_up(at, 256) - at;
    Workspace ws(workspace ? static_cast<char *>(workspace) + up : nullptr, workspace_bytes > up ? workspace_bytes - up : 0);
    BackwardSpace f(ws, s, dx, dw, db);
    if (!workspace || !ws.ok()) return fail(BPT_ERR_WORKSPACE, "linear_ce_backward: workspace of %zu bytes is too small", workspace_bytes);
    const Call c{x, w, bias, ldx, ldw, target, ignore_index, static_cast<float>(smoothing), reduction};
    switch (dtype) {
        case BPT_F32: return ce_backward<float>(s, c, f, lse, count, grad, dx, dw, db, stream);
        case BPT_BF16: return ce_backward<__nv_bfloat16>(s, c, f, lse, count, grad, dx, dw, db, stream);
        default: return ce_backward<__half>(s, c, f, lse, count, grad, dx, dw, db, stream);
    }
}
