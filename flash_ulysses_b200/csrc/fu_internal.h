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

// The range within which no factor of an attention score leaves FP32's (a softcap of
// 10^-30 would make an infinity of scale / softcap, and NaN of a score of 0).
inline int check_scores(float scale, float softcap) {
    const float size = scale < 0.f ? -scale : scale;
    if (!(size <= 1e30f)) return set_error(1, "scale must be within -1e30 and 1e30");
    if (softcap != 0.f && !(softcap >= 1e-3f && softcap <= 1e6f && size <= 1e9f * softcap))
        return set_error(1, "softcap must be 0, or within 1e-3 and 1e6 and no less than "
                            "1e-9 times the scale");
    return 0;
}

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
