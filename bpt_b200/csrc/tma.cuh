// TMA tensor maps and loads, mbarrier transactions and bounded waits with a block-wide give-up flag.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "tc5.cuh"

namespace bpt {
namespace tc5 {

// cuTensorMapEncodeTiled through the runtime's entry-point query, so the library needs no -lcuda.
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn encode_tiled() {
    static const EncodeTiledFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// A map over `planes` row-major matrices of 16-bit elements (rows x cols, `ld` elements from row to row, `plane`
// elements from matrix to matrix): a load brings 64 columns x box_rows rows into a 128-byte-swizzled tile; what lies
// outside the matrix reads as zero.  base and ld * 2 must be multiples of 16 bytes.
inline int make_map(CUtensorMap *map, bool fp16, const void *base, int64_t rows, int64_t cols, int64_t ld, int64_t planes,
                    int64_t plane, int box_rows) {
    const EncodeTiledFn encode = encode_tiled();
    if (!encode) return fail(BPT_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * 2, static_cast<cuuint64_t>(planes > 1 ? plane : ld * rows) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1}, step[3] = {1, 1, 1};
    const CUresult rc = encode(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                               const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(BPT_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", static_cast<int>(rc));
    return BPT_OK;
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}\n"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done;
}
// Waits for the phase with the given parity.  False = some wait of the block ran out (about 2 s), this one or, as the
// flag in shared memory says, another one.
constexpr long long kWaitCycles = 4000000000ll;
__device__ __forceinline__ bool mbar_wait_or_stop(uint32_t bar, uint32_t parity, volatile int *stop) {
    if (mbar_try(bar, parity)) return true;
    const long long start = clock64();
    for (;;) {
        if (mbar_try(bar, parity)) return true;
        if (*stop) return false;
        if (clock64() - start > kWaitCycles) {
            *stop = 1;
            return false;
        }
    }
}

}  // namespace tc5
}  // namespace bpt
