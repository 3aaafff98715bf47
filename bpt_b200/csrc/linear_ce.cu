// Softmax cross entropy fused with the projection that makes the logits, forward and backward, without the logits
// ever being in memory as a whole.
//
// For token i with features x_i (D numbers) and target t, a weight W (V x D), a bias b and a label smoothing e,
//     z_iv   = <x_i, W_v> + b_v,          lse_i = log sum_v exp(z_iv)
//     loss_i = lse_i - (1 - e) z_it - (e / V) sum_v z_iv
//     d z_iv = g_i (exp(z_iv - lse_i) - e / V - (1 - e) [v = t])       (g_i: gradient that reaches loss_i)
//     d x = dZ W,   d W = dZ^T X,   d b = column sums of dZ
// Tokens whose target is `ignore_index` have loss 0 and g = 0.  The others are counted and listed first; where some are
// ignored, the features of the others are brought together and only they are worked on (whatever the ignored ones hold).
//
// All four products run in one kernel shape on the 5th-generation tensor cores: a persistent pair of blocks (a cluster
// of two on one pair of SMs) walks 256 x 256 tiles, 128 rows of the result in each block.  In each block one warp brings
// operand tiles in by TMA (128-byte swizzle, six stages of 32 KB; B's rows are shared, half in each block), one thread
// of the pair issues tcgen05.mma.cta_group::2 into one of two accumulators in tensor memory, and eight warps read the
// other accumulator and finish the tile.  (Sixteen warps spilled grad's sums and made stats no faster.)
//   stats     Z tiles of consecutive vocabulary blocks of one block of tokens: a running maximum and sum per row stay in
//             registers, a row's pieces (one per pair that worked on it) are merged by the loss kernel;
//   grad      Z tiles once more (cheaper than keeping them: at D = 512 a logit costs 0.7 ps of tensor time, its fp32
//             copy 1.2 ps of HBM time), turned into dZ, which is kept for one piece of tokens x vocabulary at a time.
//             A pair walks the token blocks of one vocabulary block, so d b stays in registers, summed over the rows
//             of a thread, before the rounding of dZ;
//   products  dZ W and dZ^T X of the piece in one launch.  dZ is read K-major by the one and MN-major by the other.
// What bounds them, at 8192 x 10000 x 512 in bf16, each by itself: stats 66 us (1270 TFLOP/s) and grad 95 us (880; it also
// writes 164 MB) by the finishing of a tile, whose exponentials, sums and stores two warps a scheduler do; products 114 us
// (1470, 90% of what a library product of 8192 x 8192 x 8192 reaches) by the 11.7 TB/s at which operands come from the L2.
// Long walks hide the finishing: stats of 65536 x 8000 x 512 take 332 us (1620 TFLOP/s) alone, 400 in a long run, where the
// power limit slows everything (library products: 1640 and 1400 TFLOP/s).
// dZ is rounded to the operands' 16-bit type, without g where all g_i are one number (the scale goes onto the fp32
// results): a half-step error of each probability, the size of the rounding of the gradients themselves.
// fp32 operands are split into 16-bit planes, and each product of matrices is run as the products of planes whose weight
// is above 2^-24.  Scaled by a power of two to the top of fp16's range, an operand is two fp16 planes, the second kept
// times 2^11: 22 significant bits by rounding, down to 2^-28 of the largest number, and good to 2^-50 of that number
// below; three products (that of second planes adds 2^-22 of a term at most, or 2^-50 as below).  That is taken where no
// row's and no column's largest is below 2^-24 of the matrix's largest: the logits' sums run along a row, the gradients'
// along a column, and the logits need the columns, too, where the other operand's are as much smaller.  With the product
// that is left out a number counts as off by at most 2^-21 of itself or 2^-25 of its row's and of its column's largest.  Nor
// may the tokens' own gradients (reduction none) lie further apart, since the rows of dZ have one scale: an entry of dZ
// counts as off by at most 2^-21 of itself or 2^-49 of the largest |g| (half a step of a second plane, 2^-25 / 2^11 / 2^14,
// and a second plane of up to 2^-25 / 2^14 times the other operand's of up to 2^-11).  Otherwise three bf16 planes (24
// bits by truncation, exact, any range above 2^-110), six products.  A first pass over X and W finds which, on the
// device.  The tensor core rounds its running sum towards zero, a bias that grows with K, so the fp32 kernels take the
// accumulators out every 512 of K and add these runs up in registers; the products of the first planes have an accumulator
// of their own, so that the small ones do not lose their low bits to it.  4099 x 8003 x 300, 12% ignored, forward +
// backward: 300 us, 1.0e-6 from the values in 64 bits (an fp32 library product: 2.1e-6); stats 50, grad 71, products 125,
// copies 30 us.  (Runs of 1024 of K were no faster.)
#include <algorithm>
#include <type_traits>

#include "fused_common.cuh"
#include "tma.cuh"

namespace bpt {
namespace {

using namespace tc5;

constexpr int kBM = 256, kBN = 256, kBK = 64, kStages = 6;  // a pair's tile; each block has 128 of the rows
constexpr int kRows = kBM / 2, kCols = kBN / 2;               // what a block loads of A and of B
constexpr int kABytes = kRows * kBK * 2, kBBytes = kCols * kBK * 2, kStageBytes = kABytes + kBBytes;
constexpr int kChunkBytes = 64 * 128;  // an MN-major tile: 64 rows along K of 64 elements
// Eight warps finish tiles, one loads, one issues products (two more make its warpgroup whole).  The finishing warps take
// registers that the others leave: 256 * 208 + 128 * 88 = 384 * 168, what the block is launched with.
constexpr int kFinishWarps = 8, kThreads = (kFinishWarps + 4) * 32;
constexpr int kFinishRegs = 208, kOtherRegs = 88;
static_assert(kFinishWarps * 32 * kFinishRegs + 128 * kOtherRegs <= kThreads * 168, "the block's registers");
constexpr int kPairs = 74;             // pairs of blocks at most: one block per SM
constexpr int kRunTiles = 8;           // fp32: K blocks added up by the tensor core before the sum is taken out

enum Kind { kStats, kGrad, kProducts };
// Shared memory: the bias of two tiles, barriers; from the next 1024-byte boundary on operand stages, and 4 KB of each
// finishing warp for results on their way out (grad: 32 rows x 64 columns of dZ).
constexpr int kOutBytes = 32 * 128;
constexpr int kHeadBytes = 3 << 10;
constexpr int kSmemBytes = kHeadBytes + kStages * kStageBytes + kFinishWarps * kOutBytes;
static_assert(kSmemBytes <= 227 * 1024, "a block's shared memory");
// stats and grad, 16-bit, rows of at most kKeepTiles K blocks: the operand that stays the same from tile to tile along a
// pair's walk is kept, one K block in each 16 KB, and the rest of the shared memory has stages of the other operand alone:
// half the loads.  Where a pair has at least kKeepRun tiles.  65536 x 8000 x 512 forward (109 tiles a pair) kept 392 us,
// else 411; 8192 x 50000 x 512 forward + backward (85, 17 a piece) 1572 against 1634; 65536 x 256 x 512 (3.5) 133
// against 130, whose walks end before the fewer stages have paid.
constexpr int kKeepTiles = 8, kKeepRun = 8;
constexpr int flow_stages(int kind, int k_tiles) { return (kStages * kStageBytes + (kind == kStats ? kFinishWarps * kOutBytes : 0)) / kABytes - k_tiles; }
constexpr int kMostStages = flow_stages(kStats, 1);
static_assert(kABytes == kBBytes && flow_stages(kGrad, kKeepTiles) >= 4 && kMostStages >= kStages, "stages of one operand");
enum { kReduceNone = 0, kReduceMean = 1, kReduceSum = 2 };

// One of the two products of a piece.  A unit of work is a tile and a part of its K.
struct Product {
    int m_tiles, n_tiles, k_tiles, n_ext, width;  // width: columns of a tile, the same for all but the last
    int parts;                             // K parts of a tile (their sums go to `partial` if parts > 1)
    int64_t row_offset, row_end;           // d w: rows of the output are row_offset + tile row, below row_end
    float *acc;                            // fp32 sums of earlier pieces (leading dimension acc_ld), or null
    float *partial;                        // [part][row of the piece][acc_ld], partial_plane from part to part
    int64_t acc_ld, partial_plane;
    int add, last;                         // acc holds earlier pieces; write `out`
    void *out;
    __host__ __device__ int64_t tiles() const { return static_cast<int64_t>(m_tiles) * n_tiles; }
    __host__ __device__ int64_t units() const { return tiles() * parts; }
};

struct Params {
    int n_tiles, k_tiles, n_ext;           // stats, grad: tiles; columns in all (the last tile may be narrower)
    int m_ext, piece, pieces;              // tokens of the piece, if all count (the first is a0); which of how many it is
    int a_planes;                          // 16-bit products: of dZ, as A, 1 or 2
    const unsigned *split;                 // fp32: see Split
    int dz_planes;                         // grad: planes of dZ that are written
    int a0, b0;                            // added to the row coordinate of A and of B
    int *status;                           // set to 1 when a wait ran out
    int64_t n_rows, ignore_index;          // tokens in all
    const int *n_counted;                  // tokens that count, and which they are; rows of X, Z, dZ count these alone
    const int32_t *index;
    int gathered;                          // where some are ignored, X is read from a copy of the others' rows
    int vocab;
    const void *bias;
    const int64_t *target;
    float *partial, *z_target;             // stats: [piece][max, sum, part of mean z][row], z of the target
    unsigned *ticket;                      // zeroed by stats and grad for what follows them: its last block speaks for all
    int starts;                            // the call's first kernel: status is cleared
    void *spoilt;                          // db, where a wait that ran out is made known when its kernel has written it
    float mean_of;                         // stats: 1 / vocab where the mean of a row's logits is wanted, else 0
    const float *lse, *grad;               // grad
    float smoothing;
    int reduction;
    float *col_sums;                       // grad: column sums of dZ, 8 rows a piece (a warp's rows each), or null
    int64_t col_ld;
    int grad_pairs, grad_n_tiles, grad_n_ext;  // products: the grad launch that left them
    float *db_acc;                         // products: sums of earlier pieces
    int db_add, db_last;
    void *db;                              // of this piece, or null
    const float *count;
    const unsigned *grad_top;              // none: bits of the largest finite |g|
    // products: 0 = d x, 1 = d w.  The one with the longer units goes first, dealt in turn; pairs below `busy` have one
    // more of them.  The shorter units follow in runs of `after_busy` and `after` per pair.
    Product product[2];
    int first, busy, after_busy, after;
};

constexpr float kLowScale = 2048.f;  // of the second of two fp16 planes

template <typename T> constexpr bool kIsHalf = std::is_same<T, __half>::value;
template <typename T> constexpr bool kIsFloat = std::is_same<T, float>::value;
// fp16 dZ is kept times 2^14: |dz| <= 2, and probabilities down to 2^-28 stay normal numbers
template <typename T> constexpr float kDzScale = kIsHalf<T> ? 16384.f : 1.f;

__device__ constexpr uint32_t ce_instr(bool fp16, int n, bool a_mn, bool b_mn) {
    const uint32_t fmt = fp16 ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(a_mn) << 15) | (static_cast<uint32_t>(b_mn) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kBM >> 4) << 24);  // M = 256 over the pair
}

// Power of two at or below the largest |g| (its bits), so that g / scale is exact and below 2.
__device__ __forceinline__ float top_scale(unsigned bits) {
    const unsigned e = bits >> 23;
    return e == 0u ? (bits ? 1.17549435e-38f : 1.f) : __uint_as_float(e << 23);
}

// How fp32 operands are split, from what the pass over X and W found: bits of the largest finite |x|, complement of the
// bits of the smallest of its rows' and columns' largest (see linear_ce_spread_kernel), the same of w.
struct Split {
    bool half = false;                                 // two fp16 planes
    float x = 1.f, w = 1.f, x_back = 1.f, w_back = 1.f;  // scales before the split, and their inverses
};
// those four; bits of the largest finite |g|, complement of the bits of the smallest (zeros aside), both zero where all
// tokens have one gradient
constexpr int kFound = 6, kFoundGrad = 4;
constexpr unsigned kSpread = 24;
__device__ __forceinline__ Split read_split(const unsigned *found) {
    Split s;
    unsigned f[kFound];  // all under way at once: kernels start with this
#pragma unroll
    for (int k = 0; k < kFound; ++k) f[k] = found[k];
    const unsigned x_top = f[0] >> 23, x_low = ~f[1] >> 23, w_top = f[2] >> 23, w_low = ~f[3] >> 23;
    auto fits = [](unsigned top, unsigned low) { return top == 0u || (top >= 15u && top <= 254u && top - low <= kSpread); };
    // a matrix of zeros (or of nothing but denormal numbers, which the planes do not hold) has top 0
    if (f[0] != 0u && x_top == 0u) return s;
    if (f[2] != 0u && w_top == 0u) return s;
    if (!fits(x_top, x_low) || !fits(w_top, w_low)) return s;
    // dZ's planes have one scale, too: a token's row is good to 2^-49 of the largest |g|
    const unsigned g_top = f[kFoundGrad] >> 23, g_low = ~f[kFoundGrad + 1] >> 23;
    if (f[kFoundGrad] != 0u && (g_low == 0u || g_top - g_low > kSpread)) return s;
    s.half = true;
    if (x_top) {
        s.x = __uint_as_float((268u - x_top) << 23);  // the largest comes to [2^14, 2^15)
        s.x_back = __uint_as_float((x_top - 14u) << 23);
    }
    if (w_top) {
        s.w = __uint_as_float((268u - w_top) << 23);
        s.w_back = __uint_as_float((w_top - 14u) << 23);
    }
    return s;
}

// What is larger than this in size is not in fp32's range when multiplied by log2(e).
constexpr float kMostForExp = 2.3e38f;

// The first tile of pair c when t tiles are dealt in order to g pairs; the pair that has tile i.
__host__ __device__ __forceinline__ int64_t first_tile(int64_t t, int g, int c) { return t * c / g; }
__host__ __device__ __forceinline__ int pair_of_tile(int64_t t, int g, int64_t i) {
    return static_cast<int>(((i + 1) * g + t - 1) / t) - 1;
}

// Of the pairs launched, those that have tiles.
__device__ __forceinline__ int pairs_used(int pairs, int64_t tiles) { return static_cast<int>(min(static_cast<int64_t>(pairs), tiles)); }

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
template <typename T> __device__ __forceinline__ float unpack_low(uint32_t w) {
    if constexpr (kIsHalf<T>) return __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xFFFFu)));
    else return __uint_as_float(w << 16);
}
template <typename T> __device__ __forceinline__ float unpack_high(uint32_t w) {
    if constexpr (kIsHalf<T>) return __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)));
    else return __uint_as_float(w & 0xFFFF0000u);
}
// The next bf16 plane of a, b (truncated, so what is left is exact); a and b become what is left.
__device__ __forceinline__ uint32_t take_plane(float &a, float &b) {
    const uint32_t ha = __float_as_uint(a) & 0xFFFF0000u, hb = __float_as_uint(b) & 0xFFFF0000u;
    const uint32_t word = (ha >> 16) | hb;
    a = isfinite(a) ? a - __uint_as_float(ha) : 0.f;
    b = isfinite(b) ? b - __uint_as_float(hb) : 0.f;
    return word;
}

// The next fp16 plane of a, b (rounded); a and b become what is left, times kLowScale.
__device__ __forceinline__ uint32_t take_half(float &a, float &b) {
    const uint32_t word = pack2<__half>(a, b);
    const float ha = unpack_low<__half>(word), hb = unpack_high<__half>(word);
    a = isfinite(ha) ? (a - ha) * kLowScale : 0.f;
    b = isfinite(hb) ? (b - hb) * kLowScale : 0.f;
    return word;
}

// The same of gradients of logits, which are finite (or NaN, and then all planes may be).
__device__ __forceinline__ uint32_t take_half_finite(float &a, float &b) {
    const uint32_t word = pack2<__half>(a, b);
    const float2 left = fma2(make_float2(unpack_low<__half>(word), unpack_high<__half>(word)), make_float2(-1.f, -1.f), make_float2(a, b));
    const float2 next = mul2(left, make_float2(kLowScale, kLowScale));
    a = next.x;
    b = next.y;
    return word;
}

// 32 neighbouring results of one row to the output: 32-byte stores where the row's address allows, else 4 elements, else one
// (sums of a caller's own fp32 gradient that starts anywhere).
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

// The same for the warp's 32 rows where rows do not start on a multiple of 4 elements: across the lanes by way of shared
// memory (tile, 4 KB of this warp), so that the lanes write neighbouring elements.  The products of 6 x 5194 in fp16: with
// rows of 134 elements 26 us, by single elements of 32 rows at a time 108; with rows of 136, 8 bytes a lane, 17 us, across
// the lanes 26.
template <typename T> __device__ __forceinline__ void store_across(T *row, bool there, int n, const float (&v)[32], uint32_t tile, int lane) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; ++i)
        asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(tile + lane * 128 + ((i ^ lane) << 2)), "f"(v[i]) : "memory");
    __syncwarp();
    const unsigned rows = __ballot_sync(0xffffffffu, there);
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
        float one;
        asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(one) : "r"(tile + r * 128 + ((lane ^ r) << 2)) : "memory");
        T *const to = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), r));
        if ((rows >> r & 1u) && lane < n) to[lane] = from_acc<T>(one);
    }
}

// How the two products of a piece are dealt to the pairs of blocks.
struct Deal {
    int pairs, first, busy, after_busy, after;
    int steps;  // of the pair with the most work
};
// Unit lengths l0, l1 (in K blocks, with what a unit costs besides) and numbers u0, u1: the longer units in turn, then
// runs of the shorter ones so that the pair with the most work has as little as possible.
__host__ __device__ inline Deal deal(int pairs, int l0, int u0, int l1, int u1) {
    Deal d;
    d.pairs = pairs;
    d.first = u0 > 0 && (l0 >= l1 || u1 == 0) ? 0 : 1;
    const int long_l = d.first == 0 ? l0 : l1, long_u = d.first == 0 ? u0 : u1, short_l = d.first == 0 ? l1 : l0, short_u = d.first == 0 ? u1 : u0;
    const int each = long_u / pairs;
    d.busy = long_u % pairs;
    auto room = [&](int t, int units) { return t < units * long_l ? 0 : (t - units * long_l) / short_l; };
    int low = d.busy ? (each + 1) * long_l : each * long_l, high = low + (short_u / pairs + 1) * short_l + long_l;
    while (short_u > 0 && low < high) {
        const int t = (low + high) / 2;
        if (d.busy * room(t, each + 1) + (pairs - d.busy) * room(t, each) >= short_u) high = t;
        else low = t + 1;
    }
    d.steps = low;
    d.after_busy = short_u > 0 ? room(low, each + 1) : 0;
    d.after = short_u > 0 ? room(low, each) : 0;
    return d;
}
// A unit's fixed cost, and that of its sums through memory where a tile has several parts, in stages (0.3 us): measured.
// 65536 x 256 x 512, forward + backward: fixed costs of 2 / 4 / 8 stages 139 / 133 / 130 us, 10 / 20 / 40 for the sums
// 132 / 133 / 137; the larger sizes moved by less than 2%.
constexpr int64_t kUnitSteps = 8, kPartSteps = 20;
__host__ __device__ inline int unit_steps(int k_tiles, int parts, int stages) {
    return (k_tiles + parts - 1) / parts * stages + kUnitSteps + (parts > 1 ? kPartSteps : 0);
}
// The work of a pair, in the order in which all its warps take it: a tile, the K blocks of it, and for the products
// which product and part.
template <int kKind> struct Work {
    const Params &p;
    int64_t at, end;              // stats, grad: consecutive tiles
    int pair, pairs, stage;       // products
    int m_tiles;                  // stats, grad: with the tokens that count
    int x_units, w_units, x_k, w_k, first, busy, after_busy, after;
    int cur_tiles, cur_n, cur_width, cur_k, cur_part;  // of the product that is being worked on
    int m, n, k0, k1, which, part;
    // rows: tokens of the piece that count
    __device__ Work(const Params &p_, int rows) : p(p_) {
        pair = blockIdx.x >> 1;
        pairs = gridDim.x >> 1;
        which = part = 0;
        m_tiles = (rows + kBM - 1) / kBM;
        if constexpr (kKind != kProducts) {
            const int64_t total = tiles();
            pairs = pairs_used(pairs, total);
            at = pair < pairs ? first_tile(total, pairs, pair) : 0;
            end = pair < pairs ? first_tile(total, pairs, pair + 1) : 0;
            k0 = 0;
            k1 = p.k_tiles;
        } else {
            const Product &x = p.product[0], &w = p.product[1];
            x_units = x.m_tiles ? m_tiles * x.n_tiles * x.parts : 0;
            w_units = static_cast<int>(w.units());
            x_k = x.k_tiles;
            w_k = (rows + kBK - 1) / kBK;
            first = p.first;
            busy = p.busy;
            after_busy = p.after_busy;
            after = p.after;
        }
    }
    // products: where fewer tokens count, they are dealt again (by one thread for its block)
    __device__ Deal deal_again(int stages) const {
        return deal(pairs, unit_steps(x_k, p.product[0].parts, stages), x_units, unit_steps(w_k, p.product[1].parts, stages), w_units);
    }
    __device__ void start() {
        if constexpr (kKind == kProducts) {
            stage = 0;
            at = pair;
            take(first);
            end = first == 0 ? x_units : w_units;
        }
    }
    __device__ void take(int product) {
        which = product;
        const Product &q = p.product[product];
        cur_n = q.n_tiles;
        cur_width = q.width;
        cur_k = product == 0 ? x_k : w_k;
        cur_tiles = (product == 0 ? x_units : w_units) / q.parts;
        cur_part = (cur_k + q.parts - 1) / q.parts;
    }
    __device__ bool next() {
        if constexpr (kKind != kProducts) {
            if (at >= end) return false;
            // stats: the vocabulary blocks of a token block in a row; grad: the token blocks of a vocabulary block
            m = static_cast<int>(kKind == kStats ? at / p.n_tiles : at % m_tiles);
            n = static_cast<int>(kKind == kStats ? at % p.n_tiles : at / m_tiles);
            ++at;
            return true;
        } else {
            if (stage == 0 && at >= end) {
                stage = 1;
                const int64_t before = pair < busy ? static_cast<int64_t>(pair) * after_busy
                                                   : static_cast<int64_t>(busy) * after_busy + static_cast<int64_t>(pair - busy) * after;
                at = before;
                end = before + (pair < busy ? after_busy : after);
                take(1 - first);
                const int units = first == 0 ? w_units : x_units;
                if (end > units) end = units;
            }
            if (at >= end) return false;
            part = static_cast<int>(at) / cur_tiles;
            const int tile = static_cast<int>(at) - part * cur_tiles;
            m = tile / cur_n;
            n = tile - m * cur_n;
            k0 = part * cur_part;
            k1 = min(k0 + cur_part, cur_k);
            at += stage == 0 ? pairs : 1;
            return true;
        }
    }
    __device__ int64_t tiles() const { return static_cast<int64_t>(m_tiles) * p.n_tiles; }  // stats, grad
    __device__ int n_ext() const { return kKind == kProducts ? p.product[which].n_ext : p.n_ext; }
    __device__ int n0() const { return n * (kKind == kProducts ? cur_width : kBN); }  // the tile's first column
    __device__ int cols() const { return min(kKind == kProducts ? cur_width : kBN, n_ext() - n0()); }
    // columns of the product instruction: whole 32s, half of them from each block's B
    __device__ int width() const { return (cols() + 31) / 32 * 32; }
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
static_assert(kFinishWarps * 32 == 256 && kBN == 256, "finish_barrier_or names its thread count, a thread brings one bias");

// Sums over the warp's lanes of 32 columns: lane l gets the sum of v[l].  v is used up.
__device__ __forceinline__ float column_sum(float (&v)[32], int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const float keep = upper ? v[i + o] : v[i], give = upper ? v[i] : v[i + o];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    return v[0];
}

// What the gradients are multiplied by (0: of x, 1: of w, 2: of b): the one gradient of the loss, or the power of two that
// the tokens' own ones were divided by; and what dZ and the other operand were scaled by.
constexpr float kHalfDz = 16384.f;  // fp32 dZ in fp16 planes, as fp16 dZ
struct Scale {  // two factors, the smaller first: their product, or a result times the larger alone, may leave fp32's range
    float first, then;
};
template <typename T> __device__ __forceinline__ float scaled(float v, Scale s) {
    v *= s.first;
    if constexpr (kIsFloat<T>) v *= s.then;
    return v;
}
template <typename T> __device__ __forceinline__ Scale result_scale(const Params &p, const Split &split, int which) {
    float scale = p.reduction == kReduceNone ? top_scale(*p.grad_top) : *p.grad;
    if (p.reduction == kReduceMean) scale = *p.count > 0.f ? scale / *p.count : 0.f;
    if constexpr (kIsFloat<T>) {
        if (!split.half) return Scale{scale, 1.f};
        scale *= 1.f / kHalfDz;
        const float back = which == 0 ? split.w_back : which == 1 ? split.x_back : 1.f;
        return fabsf(scale) < back ? Scale{scale, back} : Scale{back, scale};
    }
    return Scale{scale * (1.f / kDzScale<T>), 1.f};
}

// A piece's part of the tokens that count, evenly cut where some are ignored.
struct PieceRows {
    int first, rows;
};
__device__ __forceinline__ PieceRows piece_rows(const Params &p) {
    const int counted = *p.n_counted;
    PieceRows r{p.a0, p.m_ext};
    if (counted < p.n_rows) {
        const int each = ((counted + p.pieces - 1) / p.pieces + kBM - 1) / kBM * kBM;
        r.first = min(p.piece * each, counted);
        r.rows = min(each, counted - r.first);
    }
    return r;
}

// d b of a piece, by two warps of each products block that have nothing else to do, 32 columns at a time: the column sums
// that the pairs of the grad launch (fp32: the token blocks) left, added to those of earlier rows; the last are scaled
// and stored.
template <typename T> __device__ __forceinline__ void finish_bias(const Params &p, const Split &split, int rows_here, int warp, int warps, int lane) {
    const Scale scale = result_scale<T>(p, split, 2);
    const int64_t m_tiles = (rows_here + kBM - 1) / kBM, total = m_tiles * p.grad_n_tiles;
    const int pairs = pairs_used(p.grad_pairs, total);
    for (int c0 = warp * 32; c0 < p.grad_n_ext; c0 += warps * 32) {
        const int c = c0 + lane, n = c0 / kBN;
        int pieces = static_cast<int>(m_tiles);
        if (!kIsFloat<T> && m_tiles) pieces = pair_of_tile(total, pairs, (n + 1) * m_tiles - 1) - pair_of_tile(total, pairs, n * m_tiles) + 1;
        if (c >= p.grad_n_ext) continue;
        const float *from = p.col_sums + c;
        float s[8];  // the eight rows of every piece
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = 0.f;
#pragma unroll 2
        for (int r = 0; r < pieces; ++r) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += from[(static_cast<int64_t>(r) * 8 + i) * p.col_ld];
        }
        float all = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
        if (p.db_add) all += p.db_acc[c];
        if (!p.db_last) p.db_acc[c] = all;
        else static_cast<T *>(p.db)[c] = from_acc<T>(scaled<T>(all, scale));
    }
}

// map_a, map_b: stats, grad: X and W rows; products: dZ rows and W columns.  map_c: dZ, as it is stored (grad), its columns
// (products).  map_d, map_e: stats, grad: the copy of X, rows; products: X columns, those of its copy.
template <typename T, int kKind, bool kKeep>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
linear_ce_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_c,
                 const __grid_constant__ CUtensorMap map_d, const __grid_constant__ CUtensorMap map_e, const __grid_constant__ Params p) {
    constexpr bool kPrecise = std::is_same<T, float>::value;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    float *s_bias = reinterpret_cast<float *>(smem_raw);  // [2][256]
    // full (block 0's is used) and empty per stage and per K block that is kept, sums ready and sums read (block 0's) per
    // accumulator
    const uint32_t bars = smem_u32(smem_raw) + 2 * kBN * 4;
    constexpr int kLoadBars = 8 * 2 * (kMostStages + kKeepTiles);
    const uint32_t bar_full = bars, bar_empty = bar_full + 8 * kMostStages, keep_full = bar_empty + 8 * kMostStages,
                   keep_empty = keep_full + 8 * kKeepTiles, bar_ready = bars + kLoadBars, bar_read = bar_ready + 16, bar_drain = bar_read + 16,
                   tmem_slot = bar_drain + 8;
    constexpr int kWordsAt = 2 * kBN * 4 + kLoadBars + 40;
    volatile uint32_t *tmem_word = reinterpret_cast<volatile uint32_t *>(smem_raw + kWordsAt);
    volatile int *stop = reinterpret_cast<volatile int *>(smem_raw + kWordsAt + 4);
    const uint32_t base = (bars + kLoadBars + 48 + 1023u) & ~1023u;  // the same offset in both blocks
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank();

    static_assert(kLoadBars / 8 + 5 <= kThreads, "a thread sets up a barrier");
    if (tid < kLoadBars / 8 + 5) {  // ready and read, two each, and drain come last
        const int last = tid - kLoadBars / 8;
        mbar_init(bars + 8 * tid, last == 2 || last == 3 ? 2 * kFinishWarps : 1);
        fence_mbar_init();
        if (tid == 0) *stop = 0;
    }
    if (warp == kFinishWarps + 1) tmem_alloc_pair(tmem_slot, 512);
    fence_before_sync();
    __syncthreads();
    cluster_sync();  // both blocks' barriers are set up
    fence_after_sync();
    let_next_start();
    wait_for_previous();
    if (kKind != kProducts && blockIdx.x == 0 && tid == 0) {
        *p.ticket = 0u;
        if (p.starts) *p.status = 0;
    }
    const uint32_t tmem = *tmem_word;
    const bool some_ignored = *p.n_counted < p.n_rows, copied = some_ignored && p.gathered;
    const int32_t *const index = some_ignored ? p.index : nullptr;
    const PieceRows part_of = piece_rows(p);
    const int rows_here = part_of.rows, a0 = part_of.first;
    Work<kKind> work(p, rows_here);
    Split split;
    if constexpr (kPrecise) split = read_split(p.split);
    // Stages of a K block.  fp32: one for each plane of A and of B, which all products of planes share.  16-bit: one, or one
    // for each plane of dZ with its own copy of B (first the second planes' product, whose terms are the smaller ones).
    const int planes = kPrecise ? (split.half ? 2 : 3) : kKind == kProducts ? p.a_planes : 1;
    if constexpr (kKind == kProducts) {
        if (some_ignored) {
            int *const s_deal = reinterpret_cast<int *>(smem_raw);  // the bias' place, which products have no use for
            if (tid == 0) {
                const Deal d = work.deal_again(planes);
                s_deal[0] = d.first;
                s_deal[1] = d.busy;
                s_deal[2] = d.after_busy;
                s_deal[3] = d.after;
            }
            __syncthreads();
            work.first = s_deal[0];
            work.busy = s_deal[1];
            work.after_busy = s_deal[2];
            work.after = s_deal[3];
        }
    }
    work.start();
    if (warp >= kFinishWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
        const bool keep_b = kKind == kGrad || p.n_tiles == 1;  // W's rows, else X's
        const int stages = kKeep ? flow_stages(kKind, p.k_tiles) : kStages;
        const uint32_t flow = base + p.k_tiles * kABytes;      // kKeep: the stages
        if (warp == kFinishWarps) {
            if (elect_one()) {  // ---- loads of this block's rows of A and half of B
                int s = 0;
                uint32_t phase = 0, issued = 0, keep_issued = 0;
                bool ok = true;
                for (int kept = -1; kKeep && ok && work.next();) {
                    const int m0 = a0 + work.m * kBM + static_cast<int>(rank) * kRows, n0 = p.b0 + work.n0() + static_cast<int>(rank) * (work.width() / 2);
                    const bool fresh = kept != (keep_b ? work.n : work.m);
                    kept = keep_b ? work.n : work.m;
                    auto load = [&](uint32_t to, bool of_b, int k, uint32_t full) {
                        if (rank == 0) mbar_expect(full, 2 * kABytes);
                        tma_load_pair(to, of_b ? &map_b : copied ? &map_d : &map_a, k * kBK, of_b ? n0 : m0, 0, map_to(full, 0));
                    };
                    for (int k = 0; k < p.k_tiles; ++k) {
                        if (fresh) {
                            ok = mbar_wait_or_stop(keep_empty + 8 * k, (keep_issued / p.k_tiles & 1u) ^ 1u, stop);
                            if (!ok) break;
                            load(base + k * kABytes, keep_b, k, keep_full + 8 * k);
                            ++keep_issued;
                        }
                        ok = mbar_wait_or_stop(bar_empty + 8 * s, phase ^ 1u, stop);
                        if (!ok) break;
                        load(flow + s * kABytes, !keep_b, k, bar_full + 8 * s);
                        ++issued;
                        if (++s == stages) {
                            s = 0;
                            phase ^= 1u;
                        }
                    }
                }
                while (!kKeep && ok && work.next()) {
                    const int m0 = work.m * kBM + static_cast<int>(rank) * kRows, half = work.width() / 2;
                    const int n0 = work.n0() + static_cast<int>(rank) * half, chunks = (half + 63) / 64;
                    const int run = kPrecise ? kRunTiles : work.k1;
                    for (int kr = work.k0; ok && kr < work.k1; kr += run) {
                        const int k_end = min(kr + run, work.k1);
                        int k = kr, plane = kPrecise ? 0 : planes - 1;
                        while (true) {
                            ok = mbar_wait_or_stop(bar_empty + 8 * s, phase ^ 1u, stop);
                            if (!ok) break;
                            const uint32_t a = base + s * kStageBytes, b = a + kABytes, full = map_to(bar_full + 8 * s, 0);
                            const int b_bytes = kKind == kProducts ? chunks * kChunkBytes : kBBytes, b_plane = kPrecise ? plane : 0;
                            if (rank == 0) mbar_expect(bar_full + 8 * s, 2 * (kABytes + b_bytes));
                            if constexpr (kKind == kProducts) {
                                const int b_row = (work.which == 0 ? p.b0 : a0) + k * kBK;
                                if (work.which == 0) {
                                    tma_load_pair(a, &map_a, k * kBK, m0, plane, full);
                                    for (int c = 0; c < chunks; ++c) tma_load_pair(b + c * kChunkBytes, &map_b, n0 + 64 * c, b_row, b_plane, full);
                                } else {
                                    tma_load_pair(a, &map_c, m0, k * kBK, plane, full);
                                    tma_load_pair(a + kChunkBytes, &map_c, m0 + 64, k * kBK, plane, full);
                                    for (int c = 0; c < chunks; ++c)
                                        tma_load_pair(b + c * kChunkBytes, copied ? &map_e : &map_d, n0 + 64 * c, b_row, b_plane, full);
                                }
                            } else {
                                tma_load_pair(a, copied ? &map_d : &map_a, k * kBK, a0 + m0, plane, full);
                                tma_load_pair(b, &map_b, k * kBK, p.b0 + n0, b_plane, full);
                            }
                            ++issued;
                            if (++s == kStages) {
                                s = 0;
                                phase ^= 1u;
                            }
                            if constexpr (kPrecise) {
                                if (++plane == planes) {
                                    plane = 0;
                                    if (++k == k_end) break;
                                }
                            } else if (++k == k_end) {
                                k = kr;
                                if (plane-- == 0) break;
                            }
                        }
                    }
                }
            if (!ok) {  // the last loads of every stage land before the block ends (block 0's barriers know)
                    auto landed = [&](uint32_t bars, uint32_t n, uint32_t count) {
                        for (uint32_t i = 0; i < n && i < count; ++i) {
                            const uint32_t load = count - 1 - i;
                            const long long start = clock64();
                            while (clock64() - start < kWaitCycles / 8 && !(rank == 0 && mbar_try(bars + 8 * (load % n), (load / n) & 1u))) {}
                        }
                    };
                    landed(bar_full, stages, issued);
                    if constexpr (kKeep) landed(keep_full, p.k_tiles, keep_issued);
                }
            }
        } else if (warp == kFinishWarps + 1) {
            if (rank == 0 && elect_one()) {  // ---- products
                int s = 0, buf = 0;
                uint32_t phase = 0, read_phase = 0;
                bool ok = true;
                uint32_t keep_phase = 1;
                for (int kept = -1; kKeep && ok && work.next();) {
                    const bool fresh = kept != (keep_b ? work.n : work.m);
                    if (fresh) {
                        keep_phase ^= 1u;
                        if (kept >= 0)
                            for (int k = 0; k < p.k_tiles; ++k) mma_commit_pair(keep_empty + 8 * k);  // once the products so far are done
                        kept = keep_b ? work.n : work.m;
                    }
                    ok = mbar_wait_or_stop(bar_read + 8 * buf, read_phase ^ 1u, stop);
                    if (!ok) break;
                    const uint32_t instr = ce_instr(kIsHalf<T>, work.width(), false, false);
                    const uint64_t kept_desc = desc_kmajor(base, 0), flow_desc = desc_kmajor(flow, 0);
                    for (int k = 0; k < p.k_tiles; ++k) {
                        ok = (!fresh || mbar_wait_or_stop(keep_full + 8 * k, keep_phase, stop)) && mbar_wait_or_stop(bar_full + 8 * s, phase, stop);
                        if (!ok) break;
                        fence_after_sync();
                        const uint64_t of_kept = kept_desc + k * (kABytes / 16), of_flow = flow_desc + s * (kABytes / 16);
#pragma unroll
                        for (int ks = 0; ks < kBK / 16; ++ks)
                            mma_pair(tmem + buf * kBN, (keep_b ? of_flow : of_kept) + 2 * ks, (keep_b ? of_kept : of_flow) + 2 * ks, instr, k + ks > 0);
                        mma_commit_pair(bar_empty + 8 * s);
                        if (++s == stages) {
                            s = 0;
                            phase ^= 1u;
                        }
                    }
                    if (!ok) break;
                    mma_commit_pair(bar_ready + 8 * buf);
                    if (++buf == 2) {
                        buf = 0;
                        read_phase ^= 1u;
                    }
                }
                while (!kKeep && ok && work.next()) {
                    const bool a_mn = kKind == kProducts && work.which == 1, b_mn = kKind == kProducts;
                    const uint32_t instr = ce_instr(kPrecise ? split.half : kIsHalf<T>, work.width(), a_mn, b_mn);
                    // descriptors (addresses in them count 16 bytes) of the first stage, made once a tile: one thread issues all
                    const uint64_t a_desc = a_mn ? desc_mnmajor(base, 0) : desc_kmajor(base, 0);
                    const uint64_t b_desc = b_mn ? desc_mnmajor(base + kABytes, 0) : desc_kmajor(base + kABytes, 0);
                    const uint32_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;
                    constexpr uint32_t kStageStep = kStageBytes / 16;
                    const int run = kPrecise ? kRunTiles : work.k1;
                    for (int kr = work.k0; ok && kr < work.k1; kr += run) {
                        const int k_tiles = min(kr + run, work.k1) - kr;
                        auto multiply = [&](uint32_t d, int a, int b, uint32_t accumulate) {  // of A in stage a, B in stage b
#pragma unroll
                            for (int ks = 0; ks < kBK / 16; ++ks)
                                mma_pair(d, a_desc + a * kStageStep + ks * a_step, b_desc + b * kStageStep + ks * b_step, instr, ks > 0 ? 1u : accumulate);
                        };
                        ok = mbar_wait_or_stop(bar_read + 8 * buf, read_phase ^ 1u, stop);
                        if (!ok) break;
                        fence_after_sync();
                        if constexpr (kPrecise) {
                            for (int k = 0; ok && k < k_tiles; ++k) {  // a K block's stages are neighbours: planes divides kStages
                                for (int q = 0; q < planes; ++q) {     // with plane q come the products of it and those before
                                    ok = mbar_wait_or_stop(bar_full + 8 * (s + q), phase, stop);
                                    if (!ok) break;
                                    fence_after_sync();
                                    for (int i = 0; i <= q; ++i) {
                                        for (int j = i < q ? q : 0; j <= q && i + j < planes; ++j) {
                                            const bool low = i + j > 0;
                                            multiply(tmem + (low ? 0 : kBN), s + i, s + j,
                                                     k > 0 || (low && !(q == 1 && i == 0)) ? 1u : 0u);
                                        }
                                    }
                                }
                                if (!ok) break;
                                for (int q = 0; q < planes; ++q) mma_commit_pair(bar_empty + 8 * (s + q));
                                s += planes;
                                if (s == kStages) {
                                    s = 0;
                                    phase ^= 1u;
                                }
                            }
                            if (!ok) break;
                            mma_commit_pair(bar_ready);
                            read_phase ^= 1u;
                        } else {
                            for (int step = 0; step < planes * k_tiles; ++step) {
                                ok = mbar_wait_or_stop(bar_full + 8 * s, phase, stop);
                                if (!ok) break;
                                fence_after_sync();
                                multiply(tmem + buf * kBN, s, s, step > 0);
                                mma_commit_pair(bar_empty + 8 * s);
                                if (++s == kStages) {
                                    s = 0;
                                    phase ^= 1u;
                                }
                            }
                            if (!ok) break;
                            mma_commit_pair(bar_ready + 8 * buf);
                            if (++buf == 2) {
                                buf = 0;
                                read_phase ^= 1u;
                            }
                        }
                    }
                }
                if (!ok) {  // products under way end before the tensor memory is freed
                    mma_commit_pair(bar_drain);
                    const long long start = clock64();
                    while (!mbar_try(bar_drain, 0u) && clock64() - start < kWaitCycles) {}
                }
            }
        } else if (kKind == kProducts && p.db) {
            finish_bias<T>(p, split, rows_here, static_cast<int>(blockIdx.x) * 2 + warp - (kFinishWarps + 2), static_cast<int>(gridDim.x) * 2, lane);
        }
    } else {  // ---- finishing: warp % 4 names the 32 of this block's rows, warp / 4 the half of the columns
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kFinishRegs));
        const int quarter = warp & 3, half = warp >> 2, trow = static_cast<int>(rank) * kRows + quarter * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t bar_read_0 = map_to(bar_read, 0);
        int buf = 0, parity = 0, row_m = -1, col_n = -1;
        uint32_t ready_phase = 0;
        float run_max = -INFINITY, run_sum = 0.f, run_z = 0.f;
        int tgt = -1;
        float row_lse = 0.f, row_l2 = 0.f, row_unit = 0.f, row_g = 0.f, uniform = 0.f;
        bool row_plain = true, row_skips = false;  // of the warp's rows: every g is 1 (or 0) and nothing smoothed; some g is 0 (none there)
        Scale x_scale{}, w_scale{};
        if constexpr (kKind == kProducts) {
            x_scale = result_scale<T>(p, split, 0);
            w_scale = result_scale<T>(p, split, 1);
        }
        // grad, 16-bit: column sums over the pair's token blocks of one vocabulary block
        constexpr bool kKeepSums = kKind == kGrad && !kPrecise;
        const uint32_t out_tile = base + kStages * kStageBytes + warp * kOutBytes;
        float col_sum[kKeepSums ? 4 : 1][32];
        if constexpr (kKeepSums) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 32; ++i) col_sum[j][i] = 0.f;
        }
        auto store_col_sums = [&](float (&v)[32], int j, int n, int piece) {
            const float total = column_sum(v, lane);
            p.col_sums[(static_cast<int64_t>(piece) * 8 + rank * 4 + quarter) * p.col_ld + n * kBN + half * (kBN / 2) + j * 32 + lane] = total;
        };
        auto release = [&] {  // this warp has read the accumulator
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_at(bar_read_0 + 8 * buf);
            if constexpr (kPrecise) {  // one sum is under way at a time, in both accumulators
                ready_phase ^= 1u;
            } else if (++buf == 2) {
                buf = 0;
                ready_phase ^= 1u;
            }
        };
        while (work.next()) {
            const int m = work.m, n = work.n, cols = work.cols();
            const float *bias = s_bias + parity * kBN;
            if constexpr (kKind != kProducts) {
                const int col = n * kBN + tid;  // 256 finishing threads, 256 columns
                float b = -INFINITY;
                if (col < p.n_ext) {
                    const int64_t v = p.b0 + col;
                    b = p.bias ? to_acc<T>(static_cast<const T *>(p.bias)[v]) : 0.f;
                }
                s_bias[parity * kBN + tid] = b;
                parity ^= 1;
                if (m != row_m) {
                    row_m = m;
                    const bool live = m * kBM + trow < rows_here;
                    const int64_t at = a0 + static_cast<int64_t>(m) * kBM + trow, row = live && index ? index[at] : at;
                    const int64_t target = live ? p.target[row] : -1;
                    tgt = target >= 0 && target < p.vocab ? static_cast<int>(target) : -1;
                    if constexpr (kKind == kStats) {
                        run_max = -INFINITY;
                        run_sum = run_z = 0.f;
                    } else {
                        row_lse = live ? p.lse[row] : 0.f;
                        row_g = 0.f;
                        if (live) {
                            row_g = 1.f;
                            if (p.reduction == kReduceNone) row_g = p.grad[row] * (1.f / top_scale(*p.grad_top));
                            if (tgt < 0) row_g = __int_as_float(0x7fffffff);  // no such class: the gradients say so
                            row_g *= kPrecise ? (split.half ? kHalfDz : 1.f) : kDzScale<T>;
                        }
                        uniform = p.smoothing / static_cast<float>(p.vocab) * row_g;
                        row_skips = __any_sync(0xffffffffu, row_g == 0.f);
                        row_plain = p.smoothing == 0.f && __all_sync(0xffffffffu, row_g == kDzScale<T> || row_g == 0.f);
                        // beyond kMostForExp two numbers are equal or 2^104 apart: the factor changes no exponential
                        row_unit = fabsf(row_lse) > kMostForExp ? 1.f : kLog2e;
                        row_l2 = row_lse * row_unit - (row_plain && kIsHalf<T> ? 14.f : 0.f);
                    }
                }
                if constexpr (kKeepSums) {
                    if (n != col_n && col_n >= 0 && p.col_sums) {
                        const int piece = work.pair - pair_of_tile(work.tiles(), work.pairs, static_cast<int64_t>(col_n) * work.m_tiles);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            store_col_sums(col_sum[j], j, col_n, piece);
#pragma unroll
                            for (int i = 0; i < 32; ++i) col_sum[j][i] = 0.f;
                        }
                    }
                    col_n = n;
                }
            }
            // finishes 32 neighbouring columns from c0 on; v: the products, left as what went out (grad)
            auto finish = [&](float (&v)[32], int c0) {
                if constexpr (kKind != kProducts) {
                    const int local = tgt - (p.b0 + n * kBN + c0);  // the target's place in these 32, if it is there
                    const bool here = tgt >= 0 && local >= 0 && local < 32;
                    // logits.  Not times log2(e), which would take a bias near the type's lowest number to -inf.
                    if constexpr (kPrecise) {
                        // the smaller scale first: the larger one alone may take the sum past the type's range
                        const float low = fminf(split.x_back, split.w_back), high = fmaxf(split.x_back, split.w_back);
                        const float2 first_back = make_float2(low, low), then_back = make_float2(high, high);
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 b = *reinterpret_cast<const float4 *>(bias + c0 + i);
                            const float2 lo = fma2(mul2(make_float2(v[i], v[i + 1]), first_back), then_back, make_float2(b.x, b.y));
                            const float2 hi = fma2(mul2(make_float2(v[i + 2], v[i + 3]), first_back), then_back, make_float2(b.z, b.w));
                            v[i] = lo.x;
                            v[i + 1] = lo.y;
                            v[i + 2] = hi.x;
                            v[i + 3] = hi.y;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 b = *reinterpret_cast<const float4 *>(bias + c0 + i);
                            const float2 lo = add2(make_float2(v[i], v[i + 1]), make_float2(b.x, b.y));
                            const float2 hi = add2(make_float2(v[i + 2], v[i + 3]), make_float2(b.z, b.w));
                            v[i] = lo.x;
                            v[i + 1] = lo.y;
                            v[i + 2] = hi.x;
                            v[i + 3] = hi.y;
                        }
                    }
                    const float2 log2e = make_float2(kLog2e, kLog2e);
                    if constexpr (kKind == kStats) {
                        if (p.mean_of != 0.f) {  // parts of the mean: several of the lowest numbers have no sum
                            if (cols == kBN) {
                                float2 mean = make_float2(0.f, 0.f);
#pragma unroll
                                for (int i = 0; i < 32; i += 2) mean = fma2(make_float2(v[i], v[i + 1]), make_float2(p.mean_of, p.mean_of), mean);
                                run_z += mean.x + mean.y;
                            } else {
#pragma unroll
                                for (int i = 0; i < 32; ++i) run_z += c0 + i < cols ? v[i] * p.mean_of : 0.f;
                            }
                        }
                        if (here) {
                            float zt = 0.f;
#pragma unroll
                            for (int i = 0; i < 32; ++i) zt = i == local ? v[i] : zt;
                            p.z_target[a0 + static_cast<int64_t>(m) * kBM + trow] = zt;
                        }
                        // Sums of exp(v - run_max), where run_max is a number near the largest so far: it moves only when
                        // a sum gets large (or is not a number), which saves looking for the maximum of every 32.
                        float2 sum = make_float2(0.f, 0.f);
                        if constexpr (!kPrecise) {
                            const float2 from = make_float2(-run_max * kLog2e, -run_max * kLog2e);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 d = fma2(make_float2(v[i], v[i + 1]), log2e, from);
                                sum = add2(sum, make_float2(ex2(d.x), ex2(d.y)));
                            }
                        }
                        float more = sum.x + sum.y;
                        if (kPrecise || !(more < 1e18f) || !(fabsf(run_max) <= kMostForExp)) {
                            float tops[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                            for (int i = 4; i < 32; ++i) tops[i & 3] = fmaxf(tops[i & 3], v[i]);
                            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                            if (top > run_max) {
                                run_sum *= ex2((run_max - top) * kLog2e);
                                run_max = top;
                            }
                            const float m0 = run_max == -INFINITY ? 0.f : run_max;
                            const float2 from = make_float2(-m0, -m0);
                            sum = make_float2(0.f, 0.f);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 d = mul2(add2(make_float2(v[i], v[i + 1]), from), log2e);
                                sum = add2(sum, make_float2(ex2(d.x), ex2(d.y)));
                            }
                            more = sum.x + sum.y;
                        }
                        run_sum += more;
                    } else {
                        // p g - e / V g, with p = exp(z - lse); where every g of the warp is 1 and nothing is smoothed,
                        // the type's scale rides in the exponent
                        if constexpr (kPrecise) {
                            const float2 from = make_float2(-row_lse, -row_lse), g2 = make_float2(row_g, row_g), u2 = make_float2(-uniform, -uniform);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 d = mul2(add2(make_float2(v[i], v[i + 1]), from), log2e);
                                const float2 dz = fma2(make_float2(ex2(d.x), ex2(d.y)), g2, u2);
                                v[i] = dz.x;
                                v[i + 1] = dz.y;
                            }
                        } else {
                            const float2 from = make_float2(-row_l2, -row_l2), unit = make_float2(row_unit, row_unit);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 d = fma2(make_float2(v[i], v[i + 1]), unit, from);
                                v[i] = ex2(d.x);
                                v[i + 1] = ex2(d.y);
                            }
                            if (!row_plain) {
                                const float2 g2 = make_float2(row_g, row_g), u2 = make_float2(-uniform, -uniform);
#pragma unroll
                                for (int i = 0; i < 32; i += 2) {
                                    const float2 d = fma2(make_float2(v[i], v[i + 1]), g2, u2);
                                    v[i] = d.x;
                                    v[i + 1] = d.y;
                                }
                            }
                        }
                        if (row_skips) {  // some of the warp's rows are not there or have no gradient: zeros, whatever the logits are
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = row_g == 0.f ? 0.f : v[i];
                        }
                        if (here) {
                            const float sub = (1.f - p.smoothing) * row_g;
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] -= i == local ? sub : 0.f;
                        }
                        // Out through shared memory: with one plane 64 columns of the warp's 32 rows at a time (whole
                        // 128-byte lines, sent after the second 32), else 32 columns of each plane.
                        const int y = m * kBM + trow - lane;
                        auto send = [&](int x, int plane, uint32_t tile) {
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0) {  // rows that are not there go out as zeros: the next product reads whole K blocks
                                tma_store(&map_c, x, y, plane, tile);
                                store_commit();
                            }
                        };
                        auto next_tile = [&] {  // what it held has left
                            if (lane == 0) store_wait_read<0>();
                            __syncwarp();
                            return out_tile;
                        };
                        const uint32_t narrow = lane * 64, turn = lane >> 1 & 3;  // a row of a 64-byte-swizzled tile
                        if constexpr (kPrecise) {
                            float left[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) left[i] = v[i];
                            auto store_plane = [&](int plane, auto next_word) {
                                const uint32_t tile = next_tile();
#pragma unroll
                                for (int u = 0; u < 4; ++u) {
                                    uint32_t w[4];
#pragma unroll
                                    for (int i = 0; i < 4; ++i) w[i] = next_word(left[8 * u + 2 * i], left[8 * u + 2 * i + 1]);
                                    st_shared_v4(tile + narrow + ((u ^ turn) << 4), w[0], w[1], w[2], w[3]);
                                }
                                send(n * kBN + c0, plane, tile);
                            };
                            if (split.half) {
                                store_plane(0, [](float &a, float &b) { return take_half_finite(a, b); });
                                store_plane(1, [](float &a, float &b) { return pack2<__half>(a, b); });
                            } else {
                                for (int plane = 0; plane < 3; ++plane) store_plane(plane, [](float &a, float &b) { return take_plane(a, b); });
                            }
                        } else if (p.dz_planes == 1) {
                            const int at = (c0 >> 5) & 1;  // which half of the tile's 64 columns
                            const uint32_t tile = at == 0 ? next_tile() : out_tile;
#pragma unroll
                            for (int u = 0; u < 4; ++u)
                                st_shared_v4(tile + swz(lane, at * 4 + u), pack2<T>(v[8 * u], v[8 * u + 1]), pack2<T>(v[8 * u + 2], v[8 * u + 3]),
                                             pack2<T>(v[8 * u + 4], v[8 * u + 5]), pack2<T>(v[8 * u + 6], v[8 * u + 7]));
                            if (at == 1 || c0 + 32 >= cols) send(n * kBN + (c0 & ~63), 0, tile);
                        } else {
#pragma unroll
                            for (int plane = 0; plane < 2; ++plane) {
                                const uint32_t tile = next_tile();
#pragma unroll
                                for (int u = 0; u < 4; ++u) {
                                    uint32_t w[4];
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        const float a = v[8 * u + 2 * i], b = v[8 * u + 2 * i + 1];
                                        w[i] = pack2<T>(a, b);
                                        if (plane == 1) w[i] = pack2<T>(a - unpack_low<T>(w[i]), b - unpack_high<T>(w[i]));
                                    }
                                    st_shared_v4(tile + narrow + ((u ^ turn) << 4), w[0], w[1], w[2], w[3]);
                                }
                                send(n * kBN + c0, plane, tile);
                            }
                        }
                    }
                } else {
                    const Product &q = p.product[work.which];
                    const int64_t in_piece = static_cast<int64_t>(m) * kBM + trow;
                    const int col = work.n0() + c0, left = q.n_ext - col;
                    const bool there = work.which == 0 ? in_piece < rows_here : q.row_offset + in_piece < q.row_end;
                    if (q.parts > 1) {
                        if (there) store_row(q.partial + work.part * q.partial_plane + in_piece * q.acc_ld, q.acc_ld * 4, col, left, v);
                    } else {
                        const int64_t at = (work.which == 0 ? a0 : q.row_offset) + in_piece, row = work.which == 0 && there && index ? index[at] : at;
                        if (q.add && there) {
                            const float *sums = q.acc + row * q.acc_ld + col;
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] += i < left ? sums[i] : 0.f;
                        }
                        if (!q.last) {
                            if (there) store_row(q.acc + row * q.acc_ld, q.acc_ld * 4, col, left, v);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = scaled<T>(v[i], work.which == 0 ? x_scale : w_scale);
                            T *const out = static_cast<T *>(q.out);
                            if ((reinterpret_cast<uintptr_t>(out) | q.n_ext * sizeof(T)) % (4 * sizeof(T)) == 0) {
                                if (there) store_row(out + row * q.n_ext, q.n_ext * static_cast<int64_t>(sizeof(T)), col, left, v);
                            } else {
                                store_across(out + row * q.n_ext + col, there, left, v, out_tile, lane);
                            }
                        }
                    }
                }
            };
            // of the products' narrower tiles each half has half of the 32s, too
            const int middle = kKind == kProducts ? (cols + 63) / 64 * 32 : kBN / 2, first = half * middle;
            const int until = kKind == kProducts && half == 0 ? min(cols, middle) : cols;
            bool ok;
            if constexpr (kPrecise) {  // add the runs up in registers, then finish
                const float low_weight = split.half ? 1.f / kLowScale : 1.f;
                float sum[4][32];
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[j][i] = 0.f;
                ok = true;
                for (int kr = work.k0; ok && kr < work.k1; kr += kRunTiles) {
                    ok = __all_sync(0xffffffffu, mbar_wait_or_stop(bar_ready, ready_phase, stop));
                    if (!ok) break;
                    fence_after_sync();
                    const float2 weight = make_float2(low_weight, low_weight);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (first + 32 * j < until) {
                            uint32_t low[32], high[32];
                            tmem_ld32(tmem + lanes + first + 32 * j, low);
                            tmem_ld32(tmem + lanes + kBN + first + 32 * j, high);
                            tmem_ld_wait_for(low);
                            tmem_ld_wait_for(high);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                float2 v = make_float2(sum[j][i], sum[j][i + 1]);
                                v = fma2(make_float2(__uint_as_float(low[i]), __uint_as_float(low[i + 1])), weight, v);
                                v = add2(v, make_float2(__uint_as_float(high[i]), __uint_as_float(high[i + 1])));
                                sum[j][i] = v.x;
                                sum[j][i + 1] = v.y;
                            }
                        }
                    }
                    release();
                }
                if constexpr (kKind != kProducts) ok = !finish_barrier_or(!ok);  // s_bias is whole, and all these warps go on or none does
                if (!ok) break;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (first + 32 * j < until) {
                        finish(sum[j], first + 32 * j);
                        __syncwarp();
                        if constexpr (kKind == kGrad) {
                            if (p.col_sums) store_col_sums(sum[j], j, n, m);
                        }
                    }
                }
            } else {
                const bool empty = kKind == kProducts && work.k1 <= work.k0;  // no token counts: there are no products
                ok = empty || mbar_wait_or_stop(bar_ready + 8 * buf, ready_phase, stop);
                if constexpr (kKind != kProducts) ok = !finish_barrier_or(!ok);
                else ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after_sync();
                // (loading the next 32 columns ahead was slower: 1.4 times for grad, whose sums then spill, 1.03 for stats)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (first + 32 * j < until) {
                        uint32_t r[32];
                        float v[32];
                        if (!empty) {
                            tmem_ld32(tmem + lanes + buf * kBN + first + 32 * j, r);
                            tmem_ld_wait_for(r);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) r[i] = 0u;
                        }
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
                        finish(v, first + 32 * j);
                        if constexpr (kKeepSums) {
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 sum = add2(make_float2(col_sum[j][i], col_sum[j][i + 1]), make_float2(v[i], v[i + 1]));
                                col_sum[j][i] = sum.x;
                                col_sum[j][i + 1] = sum.y;
                            }
                        }
                        __syncwarp();
                    }
                }
                if (!empty) release();
            }
            if constexpr (kKind == kStats) {
                if (n == p.n_tiles - 1 || work.at == work.end) {  // the last tile of these rows in this pair
                    const int64_t rows_padded = static_cast<int64_t>(work.m_tiles) * kBM;
                    const int piece = work.pair - pair_of_tile(work.tiles(), work.pairs, static_cast<int64_t>(m) * p.n_tiles);
                    float *at = p.partial + (static_cast<int64_t>(piece) * 2 + half) * 3 * rows_padded + static_cast<int64_t>(m) * kBM + trow;
                    at[0] = run_max;
                    at[rows_padded] = run_sum;
                    at[2 * rows_padded] = run_z;
                }
            }
        }
        if constexpr (kKeepSums) {
            if (col_n >= 0 && p.col_sums) {
                const int piece = work.pair - pair_of_tile(work.tiles(), work.pairs, static_cast<int64_t>(col_n) * work.m_tiles);
#pragma unroll
                for (int j = 0; j < 4; ++j) store_col_sums(col_sum[j], j, col_n, piece);
            }
        }
        if constexpr (kKind == kGrad) {
            if (lane == 0) store_wait();
        }
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    cluster_sync();  // nothing of the pair is under way any more
    if (warp == kFinishWarps + 1) {
        fence_after_sync();
        tmem_free_pair(tmem, 512);
    }
    if (tid == 0) {
        if (*stop) *p.status = 1;
        if constexpr (kKind == kProducts) {  // a wait that ran out leaves results that mean nothing: the last block says so in
                                             // their first elements (in those of earlier pieces, too: status outlasts them)
            __threadfence();
            if (atomicAdd(p.ticket, 1u) == gridDim.x - 1) {
                __threadfence();
                if (*static_cast<volatile int *>(p.status)) {
                    const T nan = from_acc<T>(__int_as_float(0x7fffffff));
                    const Product &x = p.product[0], &w = p.product[1];
                    if (x.tiles() && x.last) *static_cast<T *>(x.out) = nan;
                    if (w.tiles() && w.last) *static_cast<T *>(w.out) = nan;
                    if (p.spoilt) *static_cast<T *>(p.spoilt) = nan;
                }
            }
        }
    }
}

// 16 bytes that nothing reads again.
__device__ __forceinline__ uint4 ld_stream(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// ---- forward of a handful of tokens: there is nothing to compute, the weight has to pass by once.  A warp takes eight rows
// of W at a time, 16 bytes a lane and piece, against all the tokens (fp32 in shared memory).  Adding up over the lanes
// halves the rows a lane has at each of the first three steps, so a lane ends with one row's logit (four lanes with the
// same one) and keeps its own running maximum and sum; a block leaves one piece.  One token against 50000 x 512 in bf16: 8.7 us
// for 51 MB, 5.9 TB/s with its beginning and end.
template <typename T, int kTokens>
__global__ void __launch_bounds__(256, 2) linear_ce_few_kernel(const T *x, int64_t ldx, const T *w, int64_t ldw, const T *bias,
                                                            const int64_t *target, int n, int vocab, int dim, float *partial,
                                                            float *z_target, unsigned *ticket, int *status) {
    let_next_start();
    wait_for_previous();
    constexpr int kVec = 16 / sizeof(T), kFew = 8;
    extern __shared__ float xs[];  // [kTokens][dim]
    __shared__ float s_max[8][kTokens], s_sum[8][kTokens], s_z[8][kTokens];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *ticket = 0u;
        *status = 0;
    }
    for (int i = threadIdx.x; i < kTokens * dim; i += 256) xs[i] = i / dim < n ? to_acc<T>(x[i / dim * ldx + i % dim]) : 0.f;
    __syncthreads();
    float top[kTokens], sum[kTokens], total[kTokens];
    const float mean_of = 1.f / static_cast<float>(vocab);
    int tgt[kTokens];
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
        top[k] = -INFINITY;
        sum[k] = total[k] = 0.f;
        const int64_t t = k < n ? target[k] : -1;
        tgt[k] = t >= 0 && t < vocab ? static_cast<int>(t) : -1;
    }
    for (int64_t v0 = (static_cast<int64_t>(blockIdx.x) * 8 + warp) * kFew; v0 < vocab; v0 += static_cast<int64_t>(gridDim.x) * 8 * kFew) {
        float acc[kFew][kTokens];
#pragma unroll
        for (int r = 0; r < kFew; ++r)
#pragma unroll
            for (int k = 0; k < kTokens; ++k) acc[r][k] = 0.f;
#pragma unroll(kTokens <= 2 ? 2 : 1)
        for (int c = lane * kVec; c < dim; c += 32 * kVec) {
            uint4 raw[kFew];
#pragma unroll
            for (int r = 0; r < kFew; ++r) {  // rows past the end read the last one; they are left out below
                const int64_t v = v0 + r < vocab ? v0 + r : vocab - 1;
                raw[r] = ld_stream(w + v * ldw + c);
            }
            float wf[kFew][kVec];
#pragma unroll
            for (int r = 0; r < kFew; ++r) {
                const uint32_t words[4] = {raw[r].x, raw[r].y, raw[r].z, raw[r].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (kVec == 4) {
                        wf[r][i] = __uint_as_float(words[i]);
                    } else {
                        wf[r][2 * i] = unpack_low<T>(words[i]);
                        wf[r][2 * i + 1] = unpack_high<T>(words[i]);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kTokens; ++k) {
#pragma unroll
                for (int i = 0; i < kVec; i += 4) {
                    const float4 xv = *reinterpret_cast<const float4 *>(xs + k * dim + c + i);
#pragma unroll
                    for (int r = 0; r < kFew; ++r) {
                        acc[r][k] = fmaf(wf[r][i], xv.x, acc[r][k]);
                        acc[r][k] = fmaf(wf[r][i + 1], xv.y, acc[r][k]);
                        acc[r][k] = fmaf(wf[r][i + 2], xv.z, acc[r][k]);
                        acc[r][k] = fmaf(wf[r][i + 3], xv.w, acc[r][k]);
                    }
                }
            }
        }
        const int64_t v = v0 + (lane >> 4) * 4 + (lane >> 3 & 1) * 2 + (lane >> 2 & 1);  // the row this lane ends with
        const float b = bias && v < vocab ? to_acc<T>(bias[v]) : 0.f;
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
#pragma unroll
            for (int o = 16, half = kFew / 2; o >= 4; o >>= 1, half >>= 1) {
#pragma unroll
                for (int r = 0; r < half; ++r) {
                    const bool upper = lane & o;
                    const float keep = upper ? acc[r + half][k] : acc[r][k], give = upper ? acc[r][k] : acc[r + half][k];
                    acc[r][k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
            }
            float z = acc[0][k];
            z += __shfl_xor_sync(0xffffffffu, z, 2);
            z += __shfl_xor_sync(0xffffffffu, z, 1);
            if (v >= vocab) continue;
            z += b;
            if (z > top[k]) {
                sum[k] *= ex2((top[k] - z) * kLog2e);
                top[k] = z;
            }
            sum[k] += ex2((z - (top[k] == -INFINITY ? 0.f : top[k])) * kLog2e);
            total[k] = fmaf(z, mean_of, total[k]);
            if (tgt[k] == v && (lane & 3) == 0) z_target[k] = z;
        }
    }
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {  // one of the four lanes of a row counts
        if (lane & 3) {
            sum[k] = total[k] = 0.f;
            top[k] = -INFINITY;
        }
        float m = top[k];
#pragma unroll
        for (int o = 16; o >= 4; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        m = __shfl_sync(0xffffffffu, m, 0);
        if (!(sum[k] == 0.f)) sum[k] *= ex2((top[k] - m) * kLog2e);
        top[k] = m;
#pragma unroll
        for (int o = 16; o >= 4; o >>= 1) {
            sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
            total[k] += __shfl_xor_sync(0xffffffffu, total[k], o);
        }
    }
    if (lane == 0) {
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
            s_max[warp][k] = top[k];
            s_sum[warp][k] = sum[k];
            s_z[warp][k] = total[k];
        }
    }
    __syncthreads();
    if (threadIdx.x < n) {
        const int k = threadIdx.x;
        float m = -INFINITY, s = 0.f, z = 0.f;
        for (int i = 0; i < 8; ++i) m = fmaxf(m, s_max[i][k]);
        for (int i = 0; i < 8; ++i) {
            if (!(s_sum[i][k] == 0.f)) s += s_sum[i][k] * ex2((s_max[i][k] - m) * kLog2e);
            z += s_z[i][k];
        }
        float *at = partial + static_cast<int64_t>(blockIdx.x) * 3 * n + k;
        at[0] = m;
        at[n] = s;
        at[2 * n] = z;
    }
}

// ---- the loss from the pieces: kLanes threads a row, one row or many pieces a thread.
constexpr int kLossThreads = 256;
struct LossParams {
    const float *partial, *z_target;
    const int64_t *target;
    int64_t n_rows, ignore_index;
    const int *n_counted;  // null: rows are all the tokens, ignored ones among them
    const int32_t *index;
    int n_tiles, pairs, vocab, reduction;
    int pieces;            // of every row, or 0: what the tiles' dealing gives
    int64_t rows_padded;   // between a piece's numbers, or 0: whole tiles of the rows
    float smoothing;
    float *loss, *lse, *count;
    double *block_sums;  // [blocks][sum, count]
    unsigned *ticket;
    const int *status;
};

template <int kLanes> __global__ void __launch_bounds__(kLossThreads) linear_ce_loss_kernel(const LossParams p) {
    let_next_start();
    wait_for_previous();
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * kLossThreads + threadIdx.x) / kLanes;
    const int lane = threadIdx.x % kLanes;
    float loss = 0.f;
    bool counted = false;
    const int64_t n_rows = p.n_counted ? *p.n_counted : p.n_rows;
    if (row < n_rows) {
        const int64_t m_tiles = (n_rows + kBM - 1) / kBM, total = m_tiles * p.n_tiles, m = row / kBM;
        const int64_t rows_padded = p.rows_padded ? p.rows_padded : m_tiles * kBM;
        const int pairs = pairs_used(p.pairs, total);
        const int pieces = p.pieces ? p.pieces
                                    : 2 * (pair_of_tile(total, pairs, (m + 1) * p.n_tiles - 1) - pair_of_tile(total, pairs, m * p.n_tiles) + 1);
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
            const int64_t token = n_rows < p.n_rows ? p.index[row] : row, target = p.target[token];
            counted = target != p.ignore_index;
            if (counted) {
                const bool known = target >= 0 && target < p.vocab;
                const float zt = known ? p.z_target[row] : __int_as_float(0x7fffffff);
                loss = lse - zt;
                if (p.smoothing != 0.f) loss = (1.f - p.smoothing) * loss + p.smoothing * (lse - z);
            }
            if (*p.status) loss = __int_as_float(0x7fffffff);
            if (p.lse) p.lse[token] = lse;
            if (p.reduction == kReduceNone) p.loss[token] = loss;
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
    const volatile double *const sums_of = p.block_sums;  // other blocks'
    for (unsigned i = threadIdx.x; i < gridDim.x; i += kLossThreads) {
        a += sums_of[2 * i];
        b += sums_of[2 * i + 1];
    }
    const double2 all = block_sum(a, b);
    if (threadIdx.x == 0) {
        *p.loss = static_cast<float>(p.reduction == kReduceMean ? all.x / all.y : all.x);
        if (p.count) *p.count = static_cast<float>(all.y);
    }
}

// ---- operands that TMA cannot read where they lie (fp32, rows or bases off 16 bytes): copied into rows of a multiple
// of 8 elements, fp32 as planes.

// What decides how fp32 operands are split: the largest number of each matrix, and the smallest of the largest numbers of
// its rows and of its columns (those of zeros aside).  Rows and columns are looked at in stretches, rows of 128 kUnits
// columns and columns of one block's rows (kSpreadRows or more), so that a block needs nothing from another: a warp brings
// four rows in, a lane keeps the largest of its 4 kUnits columns.  Stretches are no larger than what they are part of, so this
// errs towards three planes.  Loads past the end take the last columns or row again.  kPiece: elements of a load, as many as
// dim and the rows' places allow.  By itself, without the columns' part and with it: 50000 x 512 16 and 19 us, 34558 x 626
// 14 and 19, 12102 x 300 7.3 and 7.3; with stretches of 512 columns for every width 20300 x 101 took 15 us, now 7.
constexpr int kSpreadRows = 32, kSpreadBlocks = 148 * 8;
template <int kPiece, int kUnits>
__global__ void __launch_bounds__(256) linear_ce_spread_kernel(const float *x, int64_t ldx, int64_t x_rows, const float *w,
                                                               int64_t ldw, int64_t w_rows, int dim, int64_t block_rows,
                                                               int64_t x_blocks, const int64_t *target, int64_t ignore_index,
                                                               unsigned *found) {
    constexpr int kCols = 128 * kUnits, kRowsAtOnce = 4, kPieces = kCols / 32 / kPiece;
    __shared__ unsigned s_found[2], s_col[8][kCols];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < 2) s_found[threadIdx.x] = 0u;
    let_next_start();
    wait_for_previous();
    const bool of_x = blockIdx.x < x_blocks;
    const int64_t first = (of_x ? blockIdx.x : blockIdx.x - x_blocks) * block_rows, end = min(first + block_rows, of_x ? x_rows : w_rows);
    const float *const from = of_x ? x : w;
    const int64_t ld = of_x ? ldx : ldw;
    int at[kPieces];
    unsigned col[kPieces][kPiece], top = 0u, low = 0u;  // low: complement of the smallest
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
        at[k] = min(static_cast<int>(blockIdx.y) * kCols + (32 * k + lane) * kPiece, dim - kPiece);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) col[k][i] = 0u;
    }
    for (int64_t row0 = first + warp * kRowsAtOnce; row0 < end; row0 += 8 * kRowsAtOnce) {
        float v[kRowsAtOnce][kPieces][kPiece];
        bool live[kRowsAtOnce];
#pragma unroll
        for (int r = 0; r < kRowsAtOnce; ++r) {
            const int64_t row = min(row0 + r, end - 1);
            live[r] = !of_x || target[row] != ignore_index;
            const float *const p = from + row * ld;
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                if constexpr (kPiece == 4) {
                    const float4 piece = *reinterpret_cast<const float4 *>(p + at[k]);
                    v[r][k][0] = piece.x;
                    v[r][k][1] = piece.y;
                    v[r][k][2] = piece.z;
                    v[r][k][3] = piece.w;
                } else if constexpr (kPiece == 2) {
                    const float2 piece = *reinterpret_cast<const float2 *>(p + at[k]);
                    v[r][k][0] = piece.x;
                    v[r][k][1] = piece.y;
                } else {
                    v[r][k][0] = p[at[k]];
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kRowsAtOnce; ++r) {
            unsigned largest = 0u;
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
#pragma unroll
                for (int i = 0; i < kPiece; ++i) {
                    const unsigned bits = __float_as_uint(v[r][k][i]) & 0x7FFFFFFFu, finite = live[r] && bits < 0x7F800000u ? bits : 0u;
                    col[k][i] = max(col[k][i], finite);
                    largest = max(largest, finite);
                }
            }
            largest = __reduce_max_sync(0xffffffffu, largest);
            top = max(top, largest);
            if (largest) low = max(low, ~largest);
        }
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) s_col[warp][(32 * k + lane) * kPiece + i] = col[k][i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < kCols; c += 256) {
        unsigned largest = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) largest = max(largest, s_col[k][c]);
        if (largest) low = max(low, ~largest);
    }
    low = __reduce_max_sync(0xffffffffu, low);
    if (lane == 0) {
        atomicMax(&s_found[0], top);
        atomicMax(&s_found[1], low);
    }
    __syncthreads();
    if (threadIdx.x < 2) atomicMax(&found[(of_x ? 0 : 2) + threadIdx.x], s_found[threadIdx.x]);
}

template <typename T> struct Unpacked {
    const T *at;
    int64_t ld, rows;
    uint16_t *to;  // null: this operand is read where it lies
    int64_t plane;
};
template <typename T>
__global__ void __launch_bounds__(256) linear_ce_pack_kernel(const Unpacked<T> x, const Unpacked<T> w, int dim, int64_t to_ld,
                                                             const int32_t *index, const int *n_counted,
                                                             const unsigned *found) {
    let_next_start();
    wait_for_previous();
    // of X the rows that count, and rows of zeros up to a whole K block
    const int64_t counted = *n_counted, pieces = to_ld / 8;
    const int64_t of_x = x.to ? min((counted + kBK - 1) / kBK * kBK, x.rows) * pieces : 0, total = of_x + (w.to ? w.rows * pieces : 0);
    Split split;
    if constexpr (kIsFloat<T>) split = read_split(found);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const bool is_w = i >= of_x;
        const Unpacked<T> &o = is_w ? w : x;
        const int64_t in = is_w ? i - of_x : i, row = in / pieces;
        const int c = static_cast<int>(in - row * pieces) * 8;
        const bool there = is_w || row < counted;
        // the index is there where some tokens are ignored
        const T *from = o.at + (!is_w && counted < x.rows && there ? index[row] : row) * o.ld + c;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = there && c + j < dim ? to_acc<T>(from[j]) : 0.f;
        uint16_t *to = o.to + row * to_ld + c;
        if constexpr (kIsFloat<T>) {
            if (split.half) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= is_w ? split.w : split.x;
            }
            for (int q = 0; q < (split.half ? 2 : 3); ++q) {
                uint4 word;
                word.x = split.half ? take_half(v[0], v[1]) : take_plane(v[0], v[1]);
                word.y = split.half ? take_half(v[2], v[3]) : take_plane(v[2], v[3]);
                word.z = split.half ? take_half(v[4], v[5]) : take_plane(v[4], v[5]);
                word.w = split.half ? take_half(v[6], v[7]) : take_plane(v[6], v[7]);
                *reinterpret_cast<uint4 *>(to + q * o.plane) = word;
            }
        } else {
            *reinterpret_cast<uint4 *>(to) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        }
    }
}

// ---- the tokens that count: how many a block has, then, where some are ignored, which they are, in their order.  A block
// has 256 tokens, or as many times 256 as keep the blocks' number (each block reads all their counts) below kTokenBlocks.
// Up to kTokensAlone tokens each block counts them all itself, which spares a launch: 777 x 10001 x 512 forward + backward,
// bound by host time, 86 us against 90; with 4099 x 8003 x 300 in fp32 it is slower, 316 against 313.
constexpr int kTokenBlock = 256, kTokenBlocks = 4096, kTokensAlone = 2048;
__host__ __device__ __forceinline__ int64_t block_tokens(int64_t n) {
    return (n + int64_t(kTokenBlocks) * kTokenBlock - 1) / (int64_t(kTokenBlocks) * kTokenBlock) * kTokenBlock;
}
__global__ void __launch_bounds__(kTokenBlock) linear_ce_count_kernel(const int64_t *target, int64_t n, int64_t ignore_index,
                                                                      int32_t *counts) {
    let_next_start();
    wait_for_previous();
    const int64_t start = blockIdx.x * block_tokens(n), end = min(start + block_tokens(n), n);
    int here = 0;
    for (int64_t i = start + threadIdx.x; i < start + block_tokens(n); i += kTokenBlock)
        here += __syncthreads_count(i < end && target[i] != ignore_index);
    if (threadIdx.x == 0) counts[blockIdx.x] = here;
}

__device__ __forceinline__ int block_sum(int v, int *s_warp) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < kTokenBlock / 32; ++i) v += s_warp[i];
    return v;
}

// A column of four blocks (which share the copying of rows, a warp a row: latency) writes the index of its tokens, brings
// the features of those that count to their places in the copy (if given; the last column adds rows of zeros up to a whole
// K block), and puts zeros where the ignored ones' loss (reduction none) and rows of d x (backward) go.  Where every token
// counts it does nothing.  28701 tokens of 512 in bf16, 12% ignored: 20 us in all, against the 120 us by which the products
// of the ignored ones would be longer.
__global__ void __launch_bounds__(kTokenBlock) linear_ce_gather_kernel(const uint16_t *x, int64_t ld, int64_t n, int dim,
                                                                       const int64_t *target, int64_t ignore_index,
                                                                       const int32_t *counts, int32_t *index,
                                                                       int *n_counted, uint16_t *copy,
                                                                       int64_t copy_ld, unsigned char *dx, int64_t dx_row_bytes,
                                                                       float *loss, unsigned *found) {
    __shared__ int s_warp[kTokenBlock / 32], s_place[kTokenBlock];
    let_next_start();
    wait_for_previous();
    const int64_t first = blockIdx.x * block_tokens(n), end = min(first + block_tokens(n), n);
    int all = 0, before = 0;
    if (n > kTokensAlone) {
        for (unsigned i = threadIdx.x; i < gridDim.x; i += kTokenBlock) {
            const int v = counts[i];
            all += v;
            if (i < blockIdx.x) before += v;
        }
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < static_cast<int>(n); i += kTokenBlock) {
            const int v = target[i] != ignore_index;
            all += v;
            if (i < first) before += v;
        }
    }
    all = block_sum(all, s_warp);
    const bool last = blockIdx.x == gridDim.x - 1;
    if (last && blockIdx.y == 0 && threadIdx.x == 0) *n_counted = all;
    if (last && blockIdx.y == 0 && threadIdx.x < kFound) found[threadIdx.x] = 0u;  // for the next kernels
    if (all == n) return;
    before = block_sum(before, s_warp);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool dx_wide = ((reinterpret_cast<uintptr_t>(dx) | dx_row_bytes) & 15) == 0;
    for (int64_t start = first; start < end; start += kTokenBlock) {
        const int64_t token = start + threadIdx.x;
        const bool counts_here = token < end && target[token] != ignore_index;
        const unsigned ballot = __ballot_sync(0xffffffffu, counts_here);
        __syncthreads();
        if (lane == 0) s_warp[warp] = __popc(ballot);
        __syncthreads();
        int place = before + __popc(ballot & ((1u << lane) - 1u));
        for (int i = 0; i < kTokenBlock / 32; ++i) {
            if (i < warp) place += s_warp[i];
            before += s_warp[i];
        }
        s_place[threadIdx.x] = counts_here ? place : -1;
        if (blockIdx.y == 0) {
            if (counts_here) index[place] = static_cast<int32_t>(token);
            else if (loss && token < end) loss[token] = 0.f;
        }
        __syncthreads();
        for (int t = blockIdx.y * (kTokenBlock / 32) + warp; t < kTokenBlock && start + t < end; t += gridDim.y * (kTokenBlock / 32)) {  // a warp a row
            const int to_row = s_place[t];
            if (to_row >= 0 && copy) {
                const uint16_t *from = x + (start + t) * ld;
                uint16_t *to = copy + to_row * copy_ld;
                for (int c = lane * 8; c < dim; c += 256) {
                    if (c + 8 <= dim) {
                        *reinterpret_cast<uint4 *>(to + c) = *reinterpret_cast<const uint4 *>(from + c);
                    } else {
                        for (int j = c; j < dim; ++j) to[j] = from[j];
                    }
                }
            } else if (to_row < 0 && dx) {
                unsigned char *to = dx + (start + t) * dx_row_bytes;
                if (dx_wide) {
                    for (int64_t c = lane * 16; c < dx_row_bytes; c += 512) *reinterpret_cast<uint4 *>(to + c) = make_uint4(0u, 0u, 0u, 0u);
                } else {
                    for (int64_t c = lane * 2; c < dx_row_bytes; c += 64) *reinterpret_cast<uint16_t *>(to + c) = uint16_t(0);
                }
            }
        }
    }
    if (last && blockIdx.y == 0 && copy) {
        const int64_t zeros_end = min((static_cast<int64_t>(all) + kBK - 1) / kBK * kBK, n);
        for (int64_t row = all + warp; row < zeros_end; row += kTokenBlock / 32)
            for (int c = lane; c < dim; c += 32) copy[row * copy_ld + c] = 0;
    }
}

// Over the tokens that count and whose g is finite: max |g| as bits (ordered like the numbers), and the complement of the
// smallest that is not zero.  A g that is not finite takes no part: it spoils its own row of dZ, not the others' scale.
__global__ void linear_ce_top_kernel(const float *grad, const int64_t *target, int64_t rows,
                                     int64_t ignore_index, unsigned *found) {
    let_next_start();
    wait_for_previous();
    unsigned best = 0u, low = 0u;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < rows; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        if (target[i] == ignore_index) continue;
        const unsigned bits = __float_as_uint(grad[i]) & 0x7FFFFFFFu;
        if (bits == 0u || bits >= 0x7F800000u) continue;
        best = max(best, bits);
        low = max(low, ~bits);
    }
    best = __reduce_max_sync(0xffffffffu, best);
    low = __reduce_max_sync(0xffffffffu, low);
    if ((threadIdx.x & 31) == 0) {
        atomicMax(found, best);
        atomicMax(found + 1, low);
    }
}

// Sums of a product's K parts (and of earlier pieces), in their order: a thread has 4 neighbouring columns.
template <typename T>
__global__ void __launch_bounds__(256) linear_ce_parts_kernel(const __grid_constant__ Params p, int which) {
    let_next_start();
    wait_for_previous();
    const Product &q = p.product[which];
    const int64_t pieces = q.acc_ld / 4, rows = which == 0 ? piece_rows(p).rows : q.row_end - q.row_offset, total = rows * pieces;
    const int32_t *const index = which == 0 && *p.n_counted < p.n_rows ? p.index : nullptr;
    Scale scale = result_scale<T>(p, kIsFloat<T> ? read_split(p.split) : Split(), which);
    if (*p.status) scale.first = __int_as_float(0x7fffffff);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t in_piece = i / pieces, at = (which == 0 ? piece_rows(p).first : q.row_offset) + in_piece, row = index ? index[at] : at;
        const int col = static_cast<int>(i % pieces) * 4, left = min(4, q.n_ext - col);
        const float *from = q.partial + in_piece * q.acc_ld + col;
        float4 s = *reinterpret_cast<const float4 *>(from);
        for (int k = 1; k < q.parts; ++k) {
            const float4 t = *reinterpret_cast<const float4 *>(from + k * q.partial_plane);
            s.x += t.x;
            s.y += t.y;
            s.z += t.z;
            s.w += t.w;
        }
        float v[4] = {s.x, s.y, s.z, s.w};
        float *sums = q.acc + row * q.acc_ld + col;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j >= left) break;
            if (q.add) v[j] += sums[j];
            if (!q.last) {
                sums[j] = v[j];
            } else {
                static_cast<T *>(q.out)[row * q.n_ext + col + j] = from_acc<T>(scaled<T>(v[j], scale));
            }
        }
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

int pairs_for(int64_t tiles) { return static_cast<int>(std::min<int64_t>(kPairs, tiles)); }
// Pairs that get a share of `run` consecutive tiles of `total`, at most.
int64_t shared_pieces(int64_t run, int64_t total) {
    const int64_t pairs = pairs_for(total);
    return std::min<int64_t>(pairs, run * pairs / total + 2);
}

// Up to so many tokens the 16-bit kernels keep dZ in two planes, 16 significant bits of it: the rounding of a handful of
// probabilities does not average out (a single token's gradients were off by up to 4e-3), and the products of a single
// block of tokens wait for memory, not for the second product.
constexpr int64_t kFewTokens = 256;

// Up to so many tokens the forward reads W on the CUDA cores (rows of whole 16-byte pieces, the tokens' features in
// shared memory).  W of 50000 x 512, a call: bf16, 1 / 2 / 3 / 4 tokens 15 / 18 / 23 / 25 us against 26 / 27 / 25 / 25 on the
// tiles; fp32, whose tiles need W split into planes first, 1 / 4 / 8 tokens 22 / 30 / 43 us against 109 / 108 / 109.
constexpr int64_t few_tokens(int dtype) { return dtype == BPT_F32 ? 8 : 2; }
constexpr int kFewBlocks = 148 * 2;

// Elements from row to row of a copied operand: whole 128-byte lines, which a row of a TMA box is one of, unless that would
// be much longer.
int64_t packed_row(int dim) { return dim > 128 ? ce_div(dim, kBK) * kBK : ce_div(dim, 8) * 8; }

struct Shape {
    int64_t n;
    int vocab, dim, dtype, planes, dz_planes;
    int64_t packed_ld;
    bool pack_x, pack_w, few;
    Shape(const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t n_, int vocab_, int dim_, int dtype_)
        : n(n_), vocab(vocab_), dim(dim_), dtype(dtype_), planes(dtype_ == BPT_F32 ? 3 : 1),
          dz_planes(dtype_ == BPT_F32 ? 3 : n_ <= kFewTokens ? 2 : 1), packed_ld(packed_row(dim_)),
          pack_x(!tma_ready(x, ldx, dtype_)), pack_w(!tma_ready(w, ldw, dtype_)) {
        const int vec = dtype_ == BPT_F32 ? 4 : 8;
        const int tokens = n_ <= 1 ? 1 : n_ <= 2 ? 2 : n_ <= 4 ? 4 : 8;  // whose features fit in 40 KB
        few = n_ <= few_tokens(dtype_) && int64_t(tokens) * dim_ <= 10000 && dim_ % vec == 0 && ldw % vec == 0 &&
              reinterpret_cast<uintptr_t>(w) % 16 == 0;
    }
    // stages of a K block: `planes` for the logits, for the gradients
    int product_stages() const { return planes == 3 ? 3 : dz_planes; }
    int64_t m_tiles() const { return ce_div(n, kBM); }
    int v_tiles() const { return static_cast<int>(ce_div(vocab, kBN)); }
    int64_t packed(int64_t rows) const { return align_up(rows * packed_ld, 64) * planes; }
    // pairs that share one block of rows in the forward, at most
    int64_t pieces() const { return shared_pieces(v_tiles(), m_tiles() * v_tiles()); }
};

struct ForwardSpace {
    float *partial, *z_target;
    double *block_sums;
    unsigned *ticket, *found;
    int *status;
    uint16_t *x, *w, *gathered;
    int *n_counted;
    int32_t *index, *counts;
    ForwardSpace(Workspace &ws, const Shape &s) {
        status = ws.take<int>(1);
        ticket = ws.take<unsigned>(1);
        found = ws.take<unsigned>(kFound);
        block_sums = ws.take<double>(2 * ce_div(s.n * 32, kLossThreads));
        z_target = ws.take<float>(s.n);
        // pieces x rows, with whatever part of the tokens counts: at most (pairs + two a block of rows) blocks of rows
        partial = ws.take<float>(s.few ? static_cast<int64_t>(kFewBlocks) * 3 * s.n : (kPairs + 2 * s.m_tiles()) * 2 * 3 * kBM);
        n_counted = ws.take<int>(1);
        index = s.few ? nullptr : ws.take<int32_t>(s.n);
        counts = s.few ? nullptr : ws.take<int32_t>(kTokenBlocks);
        gathered = s.few || s.pack_x ? nullptr : ws.take<uint16_t>(s.n * s.packed_ld);
        x = s.pack_x && !s.few ? ws.take<uint16_t>(s.packed(s.n)) : nullptr;
        w = s.pack_w && !s.few ? ws.take<uint16_t>(s.packed(s.vocab)) : nullptr;
    }
};

// Bytes of dZ kept at a time.  More than the L2 holds: the products read it at 3 TB/s, which HBM has to spare, and larger
// pieces leave fewer pairs of blocks idle at their ends.  28701 x 8000 x 512 / 8192 x 50000 x 512, forward + backward:
// 128 MB 905 / 1731 us, 256 MB 838 / 1568, 512 MB 833 / 1545.
constexpr int64_t kDzBytes = 256 << 20;

// What a launch costs in stages, and the elements of a sum that is read and written once more in the time of one.
constexpr int64_t kLaunchSteps = 15, kStepElements = 200000;
// Splits the longer tiles along K where that shortens the work of the pair with the most of it: few tiles, long K.
Deal split_and_deal(Product &x, Product &w, int stages) {
    Product &longer = w.tiles() == 0 || (x.tiles() > 0 && x.k_tiles >= w.k_tiles) ? x : w;
    Product &other = &longer == &x ? w : x;
    auto dealt = [&](int parts) {
        const int l = unit_steps(longer.k_tiles, parts, stages), u = static_cast<int>(longer.tiles() * parts);
        const int lo = unit_steps(other.k_tiles, 1, stages), uo = static_cast<int>(other.tiles());
        const int pairs = std::max(1, std::min(kPairs, u + uo));
        return &longer == &x ? deal(pairs, l, u, lo, uo) : deal(pairs, lo, uo, l, u);
    };
    Deal best{};
    int best_parts = 0;
    for (int parts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 36, 72}) {
        if (parts > 1 && (longer.k_tiles < 4 * parts || longer.tiles() * parts > 2 * kPairs)) break;
        const Deal d = dealt(parts);
        if (best_parts == 0 || d.steps < best.steps) {
            best = d;
            best_parts = parts;
        }
    }
    x.parts = w.parts = 1;
    longer.parts = static_cast<int>(ce_div(longer.k_tiles, std::max<int64_t>(1, ce_div(longer.k_tiles, best_parts))));
    return longer.parts == best_parts ? best : dealt(longer.parts);  // rounding may have left fewer parts
}

struct BackwardSpace {
    int64_t rows, cols;  // tokens x vocabulary of a piece
    int64_t dz_ld, dz_plane, acc_ld;
    int *status;
    unsigned *ticket, *grad_top, *found;
    uint16_t *dz, *x, *w, *gathered;
    int *n_counted;
    int32_t *index, *counts;
    float *dx_acc, *dw_acc, *col_sums, *db_acc, *partial;
    BackwardSpace(Workspace &ws, const Shape &s, bool want_dx, bool want_dw, bool want_db) {
        choose_pieces(s, want_dx, want_dw);
        dz_ld = cols;
        dz_plane = rows * cols;
        acc_ld = ce_div(s.dim, 8) * 8;
        const bool own_acc = s.dtype == BPT_F32 && s.dim == acc_ld;  // fp32 sums can live in the output itself
        status = ws.take<int>(1);
        ticket = ws.take<unsigned>(1);
        found = ws.take<unsigned>(kFound);
        grad_top = found + kFoundGrad;
        dz = ws.take<uint16_t>(dz_plane * s.dz_planes);
        x = s.pack_x ? ws.take<uint16_t>(s.packed(s.n)) : nullptr;
        w = s.pack_w ? ws.take<uint16_t>(s.packed(s.vocab)) : nullptr;
        gathered = s.pack_x ? nullptr : ws.take<uint16_t>(s.n * s.packed_ld);
        n_counted = ws.take<int>(1);
        index = ws.take<int32_t>(s.n);
        counts = ws.take<int32_t>(kTokenBlocks);
        dx_acc = want_dx && !own_acc && cols < s.vocab ? ws.take<float>(s.n * acc_ld) : nullptr;
        dw_acc = want_dw && !own_acc && rows < s.n ? ws.take<float>(s.vocab * acc_ld) : nullptr;
        db_acc = want_db && rows < s.n ? ws.take<float>(s.vocab) : nullptr;
        // the rows of column sums and the parts that any of the pieces may need (the last ones are smaller)
        int64_t sum_rows = 0, parts = 0;
        const int64_t last_r = s.n - (ce_div(s.n, rows) - 1) * rows, last_c = s.vocab - (ce_div(s.vocab, cols) - 1) * cols;
        for (int64_t r : {rows, last_r}) {
            for (int64_t c : {cols, last_c}) {
                if ((r == rows && rows > s.n) || (c == cols && cols > s.vocab)) continue;  // there is the last one only
                const int64_t m = ce_div(r, kBM), n = ce_div(c, kBN);
                sum_rows = std::max(sum_rows, 8 * (s.planes == 3 ? m : shared_pieces(m, m * n)));
                Product px, pw;
                products(s, want_dx, want_dw, r, c, &px, &pw);
                split_and_deal(px, pw, s.product_stages());
                if (px.parts > 1) parts = std::max(parts, px.parts * rows * acc_ld);
                if (pw.parts > 1) parts = std::max(parts, pw.parts * cols * acc_ld);
            }
        }
        col_sums = want_db ? ws.take<float>(sum_rows * cols) : nullptr;
        partial = parts ? ws.take<float>(parts) : nullptr;
    }
    // Pieces of rows x cols cells, whole tiles, that fit kDzBytes: as few K blocks' time as possible on the pair of
    // blocks with the most work, over all pieces, with a launch's cost for each piece and with what passes through
    // memory more than once (dX once more a cut of the vocabulary, dW a cut of the tokens).
    void choose_pieces(const Shape &s, bool want_dx, bool want_dw) {
        const int64_t cells = kDzBytes / (2 * s.dz_planes), m = ce_div(s.n, kBM), n = ce_div(s.vocab, kBN);
        rows = m * kBM;
        cols = n * kBN;
        if (rows * cols <= cells) return;
        const int64_t least = ce_div(rows * cols, cells);  // pieces at least
        int64_t best = -1;
        auto consider = [&](int64_t row_cuts, int64_t col_cuts) {
            const int64_t pm = ce_div(m, row_cuts), pn = ce_div(n, col_cuts);
            if (pm * kBM * pn * kBN > cells) return;
            row_cuts = ce_div(m, pm);
            col_cuts = ce_div(n, pn);
            Product x, w;
            products(s, want_dx, want_dw, pm * kBM, pn * kBN, &x, &w);
            const int64_t steps = split_and_deal(x, w, s.product_stages()).steps +
                                  ce_div(pm * pn, kPairs) * (ce_div(s.dim, kBK) * s.planes + 1) + 2 * kLaunchSteps;
            const int64_t again = ((col_cuts - 1) * s.n + (row_cuts - 1) * s.vocab) * s.dim / kStepElements;
            const int64_t cost = row_cuts * col_cuts * steps + again;
            if (best < 0 || cost < best) {
                best = cost;
                rows = pm * kBM;
                cols = pn * kBN;
            }
        };
        for (int64_t cuts = least; cuts < least + least / 2 + 6; ++cuts) {
            if (cuts <= m) consider(cuts, 1);
            if (cuts <= n) consider(1, cuts);
        }
        // both ways, where one way leaves a piece too narrow to keep the products busy
        for (int64_t r = 2; r * r <= 4 * least && r <= m; r *= 2) {
            const int64_t c = ce_div(least, r) + 1;
            if (c > 1 && c <= n) consider(r, c);
        }
        for (int64_t r = m; best < 0; r = ce_div(r, 2)) {  // nothing fitted: smaller and smaller
            consider(ce_div(m, r), n);
            if (r == 1) break;
        }
    }
    // Tiles of the products of a piece of r x c cells.
    static void products(const Shape &s, bool want_dx, bool want_dw, int64_t r, int64_t c, Product *x, Product *w) {
        *x = Product{};
        *w = Product{};
        x->n_ext = w->n_ext = s.dim;
        // tiles of about the same width, so that the pairs' shares are alike: 4099 x 8003 x 300 in fp32 361 us with tiles of
        // 160 and 140 columns, 366 with 256 and 44
        x->width = w->width = static_cast<int>(ce_div(ce_div(s.dim, ce_div(s.dim, kBN)), 32) * 32);
        x->n_tiles = w->n_tiles = static_cast<int>(ce_div(s.dim, x->width));
        x->m_tiles = want_dx ? static_cast<int>(ce_div(r, kBM)) : 0;
        w->m_tiles = want_dw ? static_cast<int>(ce_div(c, kBM)) : 0;
        x->k_tiles = static_cast<int>(ce_div(c, kBK));
        w->k_tiles = static_cast<int>(ce_div(r, kBK));
        x->parts = w->parts = 1;
    }
};

struct Maps {
    CUtensorMap a, b, c, d, e;
};

template <typename T, int kKind> int launch_ce(const Maps &m, const Params &p, int pairs, cudaStream_t stream) {
    auto launch = [&](auto keep) -> int {
        static OncePerDevice allowed;
        auto kernel = linear_ce_kernel<T, kKind, keep.value>;
        BPT_CUDA(allow_smem(allowed, kernel, kSmemBytes));
        BPT_CUDA(launch_after(kernel, 2 * pairs, kThreads, kSmemBytes, stream, m.a, m.b, m.c, m.d, m.e, p));
        return BPT_OK;
    };
    if constexpr (!kIsFloat<T> && kKind != kProducts) {
        if (p.k_tiles <= kKeepTiles && ce_div(p.m_ext, kBM) * p.n_tiles >= kKeepRun * pairs) return launch(std::true_type());
    }
    return launch(std::false_type());
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

struct Tokens {  // the index and its length, on the device
    int32_t *index, *counts;
    int *n_counted;
    uint16_t *gathered;
};

int launch_spread(const Shape &s, const Call &c, unsigned *found, cudaStream_t stream) {
    const int64_t units = ce_div(s.dim, 128), stretches = ce_div(units, 4);
    const int64_t block_rows = std::max<int64_t>(kSpreadRows, ce_div((s.n + s.vocab) * stretches, kSpreadBlocks)), x_blocks = ce_div(s.n, block_rows);
    const dim3 grid(static_cast<unsigned>(x_blocks + ce_div(s.vocab, block_rows)), static_cast<unsigned>(stretches));
    auto launch = [&](auto piece, auto units_each) -> int {
        BPT_CUDA(launch_after(linear_ce_spread_kernel<piece.value, units_each.value>, grid, 256, 0, stream, static_cast<const float *>(c.x), c.ldx,
                              s.n, static_cast<const float *>(c.w), c.ldw, int64_t(s.vocab), s.dim, block_rows, x_blocks, c.target,
                              c.ignore_index, found));
        return BPT_OK;
    };
    auto with_piece = [&](auto piece) -> int {
        switch (ce_div(units, stretches)) {
            case 1: return launch(piece, std::integral_constant<int, 1>());
            case 2: return launch(piece, std::integral_constant<int, 2>());
            case 3: return launch(piece, std::integral_constant<int, 3>());
            default: return launch(piece, std::integral_constant<int, 4>());
        }
    };
    const uint64_t places = static_cast<uint64_t>(s.dim | c.ldx | c.ldw) * sizeof(float) | reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.w);
    return places % 16 == 0  ? with_piece(std::integral_constant<int, 4>())
           : places % 8 == 0 ? with_piece(std::integral_constant<int, 2>())
                             : with_piece(std::integral_constant<int, 1>());
}

// The index of the tokens that count; X and W as the tiles read them: where they lie (X, where tokens are ignored: from
// the copy), or packed.  loss: where ignored tokens' zeros go, or null; dx: the same for their rows of d x; grad: the
// backward's gradients, or null.
template <typename T>
int prepare_operands(const Shape &s, const Call &c, const Tokens &t, uint16_t *x_to, uint16_t *w_to, unsigned *found, float *loss, void *dx,
                     const float *grad, cudaStream_t stream, Operand *x, Operand *w) {
    *x = Operand{c.x, c.ldx, 0};
    *w = Operand{c.w, c.ldw, 0};
    const unsigned blocks = static_cast<unsigned>(ce_div(s.n, block_tokens(s.n)));
    if (s.n > kTokensAlone)
        BPT_CUDA(launch_after(linear_ce_count_kernel, blocks, kTokenBlock, 0, stream, c.target, s.n, c.ignore_index, t.counts));
    BPT_CUDA(launch_after(linear_ce_gather_kernel, dim3(blocks, 4), kTokenBlock, 0, stream, static_cast<const uint16_t *>(c.x), c.ldx, s.n, s.dim,
                          c.target, c.ignore_index, t.counts, t.index, t.n_counted, t.gathered, s.packed_ld, static_cast<unsigned char *>(dx),
                          static_cast<int64_t>(s.dim) * static_cast<int64_t>(sizeof(T)), loss, found));
    if (grad && c.reduction == kReduceNone) {
        BPT_CUDA(launch_after(linear_ce_top_kernel, static_cast<unsigned>(std::min<int64_t>(ce_div(s.n, 256), 148)), 256, 0, stream, grad,
                              c.target, s.n, c.ignore_index, found + kFoundGrad));
    }
    if constexpr (kIsFloat<T>) {
        BPT_TRY(launch_spread(s, c, found, stream));
    }
    if (!s.pack_x && !s.pack_w) return BPT_OK;
    const Unpacked<T> from_x{static_cast<const T *>(c.x), c.ldx, s.n, x_to, static_cast<int64_t>(align_up(s.n * s.packed_ld, 64))};
    const Unpacked<T> from_w{static_cast<const T *>(c.w), c.ldw, s.vocab, w_to, static_cast<int64_t>(align_up(s.vocab * s.packed_ld, 64))};
    if (s.pack_x) *x = Operand{x_to, s.packed_ld, from_x.plane};
    if (s.pack_w) *w = Operand{w_to, s.packed_ld, from_w.plane};
    const int64_t rows = (s.pack_x ? s.n : 0) + (s.pack_w ? s.vocab : 0);
    BPT_CUDA(launch_after(linear_ce_pack_kernel<T>, static_cast<unsigned>(std::min<int64_t>(ce_div(rows * (s.packed_ld / 8), 256), 148 * 16)), 256, 0,
                          stream, from_x, from_w, s.dim, s.packed_ld, static_cast<const int32_t *>(t.index), static_cast<const int *>(t.n_counted),
                          static_cast<const unsigned *>(found)));
    return BPT_OK;
}

template <typename T> int launch_few(const Shape &s, const Call &c, ForwardSpace &f, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(kFewBlocks, ce_div(s.vocab, 64)));
    auto go = [&](auto tokens) -> int {
        BPT_CUDA(launch_after(linear_ce_few_kernel<T, tokens.value>, grid, 256, tokens.value * s.dim * sizeof(float), stream,
                              static_cast<const T *>(c.x), c.ldx, static_cast<const T *>(c.w), c.ldw, static_cast<const T *>(c.bias), c.target,
                              static_cast<int>(s.n), s.vocab, s.dim, f.partial, f.z_target, f.ticket, f.status));
        return BPT_OK;
    };
    if (s.n <= 1) return go(std::integral_constant<int, 1>());
    if constexpr (kIsFloat<T>) {
        if (s.n > 4) return go(std::integral_constant<int, 8>());
        if (s.n > 2) return go(std::integral_constant<int, 4>());
    }
    return go(std::integral_constant<int, 2>());
}

template <typename T> int ce_forward(const Shape &s, const Call &c, ForwardSpace &f, float *loss, float *lse, float *count, cudaStream_t stream) {
    constexpr bool kHalf = kIsHalf<T>;
    LossParams l{};
    const int pairs = pairs_for(s.m_tiles() * s.v_tiles());
    if (s.few) {
        BPT_TRY(launch_few<T>(s, c, f, stream));
        l.pieces = static_cast<int>(std::min<int64_t>(kFewBlocks, ce_div(s.vocab, 64)));
        l.rows_padded = s.n;
    } else {
        Operand x, w;
        BPT_TRY(prepare_operands<T>(s, c, Tokens{f.index, f.counts, f.n_counted, f.gathered}, f.x, f.w, f.found,
                                    c.reduction == kReduceNone ? loss : nullptr, nullptr, nullptr, stream, &x, &w));
        Maps maps;
        BPT_TRY(make_map(&maps.a, kHalf, x.at, s.n, s.dim, x.ld, s.planes, x.plane, kRows));
        BPT_TRY(make_map(&maps.b, kHalf, w.at, s.vocab, s.dim, w.ld, s.planes, w.plane, kCols));
        maps.c = maps.d = maps.e = maps.a;
        if (f.gathered) BPT_TRY(make_map(&maps.d, kHalf, f.gathered, s.n, s.dim, s.packed_ld, 1, 0, kRows));
        Params p{};
        p.n_tiles = s.v_tiles();
        p.k_tiles = static_cast<int>(ce_div(s.dim, kBK));
        p.n_ext = s.vocab;
        p.dz_planes = s.dz_planes;
        p.status = f.status;
        p.split = f.found;
        p.m_ext = static_cast<int>(s.n);
        p.pieces = 1;
        p.n_counted = f.n_counted;
        p.index = f.index;
        p.gathered = f.gathered != nullptr;
        p.n_rows = s.n;
        p.ignore_index = c.ignore_index;
        p.vocab = s.vocab;
        p.bias = c.bias;
        p.target = c.target;
        p.partial = f.partial;
        p.z_target = f.z_target;
        p.ticket = f.ticket;
        p.starts = 1;
        p.mean_of = c.smoothing != 0.f ? 1.f / static_cast<float>(s.vocab) : 0.f;
        BPT_TRY((launch_ce<T, kStats>(maps, p, pairs, stream)));
        l.n_counted = f.n_counted;
        l.index = f.index;
    }
    l.partial = f.partial;
    l.z_target = f.z_target;
    l.target = c.target;
    l.n_rows = s.n;
    l.ignore_index = c.ignore_index;
    l.n_tiles = s.v_tiles();
    l.pairs = pairs;
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
    const bool many = l.pieces > 8 || s.pieces() > 8;
    BPT_CUDA(launch_after(many ? linear_ce_loss_kernel<32> : linear_ce_loss_kernel<1>,
                          static_cast<unsigned>(ce_div(many ? s.n * 32 : s.n, kLossThreads)), kLossThreads, 0, stream, l));
    return BPT_OK;
}

template <typename T>
int ce_backward(const Shape &s, const Call &c, BackwardSpace &f, const float *lse, const float *count, const float *grad, void *dx,
                void *dw, void *db, cudaStream_t stream) {
    constexpr bool kHalf = kIsHalf<T>;
    constexpr bool kFloat = std::is_same<T, float>::value;
    Operand x, w;
    BPT_TRY(prepare_operands<T>(s, c, Tokens{f.index, f.counts, f.n_counted, f.gathered}, f.x, f.w, f.found, nullptr, dx, grad, stream, &x, &w));
    Maps grad_maps, maps;
    BPT_TRY(make_map(&grad_maps.a, kHalf, x.at, s.n, s.dim, x.ld, s.planes, x.plane, kRows));
    BPT_TRY(make_map(&grad_maps.b, kHalf, w.at, s.vocab, s.dim, w.ld, s.planes, w.plane, kCols));
    grad_maps.d = grad_maps.e = grad_maps.a;
    if (f.gathered) BPT_TRY(make_map(&grad_maps.d, kHalf, f.gathered, s.n, s.dim, s.packed_ld, 1, 0, kRows));
    BPT_TRY(make_map(&maps.b, kHalf, w.at, s.vocab, s.dim, w.ld, s.planes, w.plane, 64));
    BPT_TRY(make_map(&maps.d, kHalf, x.at, s.n, s.dim, x.ld, s.planes, x.plane, 64));
    maps.e = maps.d;
    if (f.gathered) BPT_TRY(make_map(&maps.e, kHalf, f.gathered, s.n, s.dim, s.packed_ld, 1, 0, 64));
    Params p{};
    p.dz_planes = s.dz_planes;
    p.status = f.status;
    p.split = f.found;
    p.ticket = f.ticket;
    p.spoilt = db;
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
    p.col_sums = f.col_sums;
    p.col_ld = f.cols;
    p.n_counted = f.n_counted;
    p.index = f.index;
    p.gathered = f.gathered != nullptr;
    p.pieces = static_cast<int>(ce_div(s.n, f.rows));
    const bool own_acc = kFloat && s.dim == f.acc_ld;
    for (int64_t n0 = 0; n0 < s.n; n0 += f.rows) {
        const int64_t rows = std::min(f.rows, s.n - n0);
        const bool last_rows = n0 + f.rows >= s.n;
        for (int64_t v0 = 0; v0 < s.vocab; v0 += f.cols) {
            const int64_t cols = std::min<int64_t>(f.cols, s.vocab - v0);
            const bool last_cols = v0 + f.cols >= s.vocab;
            p.piece = static_cast<int>(n0 / f.rows);
            Params g = p;
            g.n_tiles = static_cast<int>(ce_div(cols, kBN));
            g.k_tiles = static_cast<int>(ce_div(s.dim, kBK));
            g.n_ext = static_cast<int>(cols);
            g.m_ext = static_cast<int>(rows);
            g.a0 = static_cast<int>(n0);
            g.starts = n0 == 0 && v0 == 0;
            g.b0 = static_cast<int>(v0);
            BPT_TRY(make_map(&grad_maps.c, kHalf, f.dz, f.rows, cols, f.dz_ld, s.dz_planes, f.dz_plane, 32, s.dz_planes == 1 ? 64 : 32));
            const int pairs = pairs_for(ce_div(rows, kBM) * g.n_tiles);
            BPT_TRY((launch_ce<T, kGrad>(grad_maps, g, pairs, stream)));
            BPT_TRY(make_map(&maps.a, kHalf, f.dz, f.rows, cols, f.dz_ld, s.dz_planes, f.dz_plane, kRows));
            BPT_TRY(make_map(&maps.c, kHalf, f.dz, f.rows, cols, f.dz_ld, s.dz_planes, f.dz_plane, 64));
            Params q = p;
            q.a0 = static_cast<int>(n0);
            q.m_ext = static_cast<int>(rows);
            BackwardSpace::products(s, dx, dw, rows, cols, &q.product[0], &q.product[1]);
            Product &px = q.product[0], &pw = q.product[1];
            const Deal d = split_and_deal(px, pw, s.product_stages());
            q.a_planes = s.dz_planes;
            q.first = d.first;
            q.busy = d.busy;
            q.after_busy = d.after_busy;
            q.after = d.after;
            q.b0 = static_cast<int>(v0);
            px.partial_plane = f.rows * f.acc_ld;
            pw.partial_plane = f.cols * f.acc_ld;
            px.acc = own_acc ? static_cast<float *>(dx) : f.dx_acc;
            px.add = v0 > 0;
            px.last = last_cols;
            px.out = dx;
            pw.row_offset = v0;
            pw.row_end = v0 + cols;
            pw.acc = own_acc ? static_cast<float *>(dw) : f.dw_acc;
            pw.add = n0 > 0;
            pw.last = last_rows;
            pw.out = dw;
            px.acc_ld = pw.acc_ld = f.acc_ld;
            q.grad_pairs = pairs;
            q.grad_n_tiles = g.n_tiles;
            q.grad_n_ext = g.n_ext;
            q.db = db ? static_cast<T *>(db) + v0 : nullptr;
            q.db_acc = f.db_acc ? f.db_acc + v0 : nullptr;
            q.db_add = n0 > 0;
            q.db_last = last_rows;
            px.partial = pw.partial = f.partial;  // at most one of them has parts
            // d b is shared by the blocks of all pairs, also where there are fewer units than pairs
            BPT_TRY((launch_ce<T, kProducts>(maps, q, db ? kPairs : d.pairs, stream)));
            for (int which = 0; which < 2; ++which) {
                const Product &r = q.product[which];
                if (r.parts <= 1) continue;
                const int64_t blocks = std::min<int64_t>(ce_div((which == 0 ? f.rows : cols) * (r.acc_ld / 4), 256), 148 * 8);
                BPT_CUDA(launch_after(linear_ce_parts_kernel<T>, static_cast<unsigned>(blocks), 256, 0, stream, q, which));
            }
        }
    }
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
