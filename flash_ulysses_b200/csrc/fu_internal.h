// Internal helpers shared by the C-ABI translation units.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace fu {
// Records a printf-style message for fu_last_error() and returns `code`.
int set_error(int code, const char* fmt, ...);

// The driver's cuTensorMapEncodeTiled (signature as in cuda.h), fetched once at
// run time so the library needs no link-time dependency on libcuda; NULL if the
// driver does not provide it.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn();

// Makes `device` current for a scope.
struct DeviceGuard {
    int prev = -1;
    bool changed = false, failed = false;
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&prev) != cudaSuccess) {
            failed = true;
        } else if (prev != device) {
            changed = cudaSetDevice(device) == cudaSuccess;
            failed = !changed;
        }
        if (failed) cudaGetLastError();
    }
    ~DeviceGuard() {
        if (changed) cudaSetDevice(prev);
    }
    bool ok() const { return !failed; }
};

// The configuration of one launch, by default with programmatic stream
// serialization (the kernel waits with griddepcontrol.wait before it touches
// global memory).
struct Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr = {};
    Launch(dim3 grid, dim3 block, size_t smem, void* stream, bool pdl) {
        cfg.gridDim = grid;
        cfg.blockDim = block;
        cfg.dynamicSmemBytes = smem;
        cfg.stream = static_cast<cudaStream_t>(stream);
        if (pdl) {
            attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr.val.programmaticStreamSerializationAllowed = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
        }
    }
    Launch(const Launch&) = delete;
    Launch& operator=(const Launch&) = delete;
};
}  // namespace fu
