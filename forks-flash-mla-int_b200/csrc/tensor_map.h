// Host helpers shared by the kernels with TMA operands: 3-D tensor maps of 16-bit rows, per-device facts.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <atomic>
#include <cstdint>

namespace smla {

int device_status_address(int **addr_out);

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, fetched through the runtime so that libcuda need not be linked.
inline EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// A tensor {d0, d1, d2} of 16-bit elements, d0 contiguous, s1 / s2 bytes between neighbours along the others; boxes
// {64, rows, 1} land as [rows][128 B] slabs with the 128-byte swizzle, zeros where they reach outside.
inline bool make_slab_map(CUtensorMap *map, bool fp16, const void *base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t s1,
                          uint64_t s2, uint32_t rows) {
    const EncodeTiled enc = encode_tiled();
    if (enc == nullptr) return false;
    const cuuint64_t dims[3] = {d0, d1, d2};
    const cuuint64_t strides[2] = {s1, s2};
    const cuuint32_t box[3] = {64, rows, 1}, one[3] = {1, 1, 1};
    return enc(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims,
               strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The status word's address and the permission for `bytes` of shared memory, settled once per device and kernel.
struct KernelSetup {
    std::atomic<int *> status[64] = {};
    // `regs`: registers per thread that the kernel must have been compiled to (it redistributes them; 0 = any)
    int get(const void *kernel, int bytes, int **status_out, int regs = 0) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return static_cast<int>(e);
        const bool tracked = dev >= 0 && dev < 64;
        int *s = tracked ? status[dev].load(std::memory_order_acquire) : nullptr;
        if (s == nullptr) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (e != cudaSuccess) return static_cast<int>(e);
            cudaFuncAttributes attr;
            e = cudaFuncGetAttributes(&attr, kernel);
            if (e != cudaSuccess) return static_cast<int>(e);
            if (attr.numRegs < regs) return static_cast<int>(cudaErrorInvalidKernelImage);
            const int rc = device_status_address(&s);
            if (rc != 0) return rc;
            if (tracked) status[dev].store(s, std::memory_order_release);
        }
        *status_out = s;
        return 0;
    }
};

}  // namespace smla
