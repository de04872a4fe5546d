// Attention over the exchanged Q/K/V rows (sm_100a): packed documents, causal,
// prefix or full masks, scores capped by a tanh and/or lowered with distance.
//
// One warp per (row, query head): lane l holds dims 4l..4l+3 of q, of the
// running output and of each key's k and v; scores by a warp sum, with the
// running maximum m and sum l of an online softmax in FP32.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "flash_ulysses_b200.h"
#include "fu_internal.h"
#include "fu_ptx.cuh"

namespace fu {
namespace attention {

constexpr int D = FU_HEAD_DIM;
constexpr int WARPS = 4;

// Status "where" codes of this kernel.
enum : int { W_CU_SEQLENS = 64 };

struct Params {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    __nv_bfloat16* out;
    int64_t q_stride, k_stride, v_stride, out_stride;
    const int32_t* cu_seqlens;
    const int32_t* prefix_lens;
    const float* alibi_slopes;
    int32_t* status;
    int32_t tokens, docs, group, causal;
    float scale, softcap;
};

// Rows [lo, hi) that row i sees; empty for a row behind the last document.
// Safe for any content of cu_seqlens.
__device__ __forceinline__ int2 seen_rows(const Params& p, int i) {
    int d = 0, lo = 0, hi = p.tokens;
    if (p.cu_seqlens != nullptr) {
        // The last document that starts at or before row i (empty ones skipped).
        int a = 0, b = p.docs;
        while (b - a > 1) {
            const int mid = (a + b) >> 1;
            if (__ldg(p.cu_seqlens + mid) <= i) a = mid; else b = mid;
        }
        d = a;
        lo = max(__ldg(p.cu_seqlens + d), 0);
        hi = min(__ldg(p.cu_seqlens + d + 1), p.tokens);
    }
    if (i < lo || i >= hi) return make_int2(0, 0);
    if (p.causal) {
        int seen = i + 1;
        if (p.prefix_lens != nullptr)
            seen = max(seen, lo + min(max(__ldg(p.prefix_lens + d), 0), hi - lo));
        hi = seen;
    }
    return make_int2(lo, hi);
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

__global__ void __launch_bounds__(32 * WARPS) attention_kernel(const Params p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    if (blockIdx.x == 0 && blockIdx.y == 0 && p.cu_seqlens != nullptr) {
        for (int d = threadIdx.x; d <= p.docs; d += blockDim.x) {
            const int c = p.cu_seqlens[d];
            const int before = d > 0 ? p.cu_seqlens[d - 1] : 0;
            if (c < before || c > p.tokens || (d == 0 && c != 0))
                report_status(p.status, FU_DEV_LENGTHS, W_CU_SEQLENS);
        }
    }
    const int i = blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int h = blockIdx.y;
    if (i >= p.tokens) return;
    const int2 seen = seen_rows(p, i);
    if (seen.x >= seen.y) return;
    const int hk = h / p.group;
    const float4 q = load4(p.q + i * p.q_stride + h * D + 4 * lane);
    const float slope = p.alibi_slopes != nullptr ? p.alibi_slopes[h] : 0.f;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = seen.x; j < seen.y; ++j) {
        const float4 k = load4(p.k + j * p.k_stride + hk * D + 4 * lane);
        const float4 v = load4(p.v + j * p.v_stride + hk * D + 4 * lane);
        float x = p.scale * warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w);
        if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
        x -= slope * fabsf(static_cast<float>(i - j));
        const float m2 = fmaxf(m, x);
        const float old = m == m2 ? 1.f : __expf(m - m2);
        const float w = __expf(x - m2);
        m = m2;
        l = l * old + w;
        o.x = o.x * old + w * v.x;
        o.y = o.y * old + w * v.y;
        o.z = o.z * old + w * v.z;
        o.w = o.w * old + w * v.w;
    }
    __nv_bfloat162 r[2] = {__floats2bfloat162_rn(o.x / l, o.y / l),
                           __floats2bfloat162_rn(o.z / l, o.w / l)};
    *reinterpret_cast<uint2*>(p.out + i * p.out_stride + h * D + 4 * lane) =
        *reinterpret_cast<const uint2*>(r);
}

}  // namespace attention
}  // namespace fu

using namespace fu;

extern "C" int fu_attention_forward(const fu_attention_args* a, uint32_t flags, void* stream) {
    if (a == nullptr) return set_error(FU_ERR_INVALID, "null arguments");
    if (a->kv_heads < 1 || a->q_heads < 1 || a->q_heads % a->kv_heads || a->q_heads > 65535)
        return set_error(FU_ERR_INVALID, "q_heads %d must be a positive multiple of kv_heads %d",
                         a->q_heads, a->kv_heads);
    if (a->tokens < 1 || a->tokens > (1 << 30))
        return set_error(FU_ERR_INVALID, "tokens %lld not in [1, 2^30]",
                         static_cast<long long>(a->tokens));
    if (a->docs < 1 || a->docs > (1 << 30) || (a->cu_seqlens == nullptr && a->docs != 1))
        return set_error(FU_ERR_INVALID, "docs %d does not go with cu_seqlens", a->docs);
    if (a->prefix_lens != nullptr && !a->causal)
        return set_error(FU_ERR_INVALID, "prefix_lens need a causal mask");
    if (!(a->softcap >= 0.f) || !std::isfinite(a->softcap) || !std::isfinite(a->scale))
        return set_error(FU_ERR_INVALID, "scale must be finite, softcap finite and 0 or more");
    if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->out == nullptr)
        return set_error(FU_ERR_INVALID, "null tensor argument");
    const struct { const void* ptr; int64_t stride; int heads; const char* name; } rows[4] = {
        {a->q, a->q_stride, a->q_heads, "q"},
        {a->k, a->k_stride, a->kv_heads, "k"},
        {a->v, a->v_stride, a->kv_heads, "v"},
        {a->out, a->out_stride, a->q_heads, "out"}};
    for (const auto& r : rows)
        if ((reinterpret_cast<uintptr_t>(r.ptr) & 15) || r.stride % 8 ||
            r.stride < static_cast<int64_t>(r.heads) * FU_HEAD_DIM || r.stride > (1ll << 31))
            return set_error(FU_ERR_INVALID, "%s must be 16-byte aligned with a row stride that "
                             "is a multiple of 8 and no less than its width", r.name);
    if (a->status_host != nullptr && *reinterpret_cast<volatile int32_t*>(a->status_host) != 0)
        return set_error(FU_ERR_DEVICE, "an earlier launch reported device status 0x%x",
                         static_cast<unsigned>(*a->status_host));

    attention::Params p = {};
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.k = static_cast<const __nv_bfloat16*>(a->k);
    p.v = static_cast<const __nv_bfloat16*>(a->v);
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.q_stride = a->q_stride;
    p.k_stride = a->k_stride;
    p.v_stride = a->v_stride;
    p.out_stride = a->out_stride;
    p.cu_seqlens = a->cu_seqlens;
    p.prefix_lens = a->prefix_lens;
    p.alibi_slopes = a->alibi_slopes;
    p.status = a->status;
    p.tokens = static_cast<int32_t>(a->tokens);
    p.docs = a->docs;
    p.group = a->q_heads / a->kv_heads;
    p.causal = a->causal;
    p.scale = a->scale;
    p.softcap = a->softcap;

    DeviceGuard guard(a->device);
    if (!guard.ok()) return set_error(FU_ERR_INVALID, "device %d is not available", a->device);
    Launch launch(dim3((p.tokens + attention::WARPS - 1) / attention::WARPS, a->q_heads),
                  dim3(32 * attention::WARPS), 0, stream, (flags & FU_FWD_NO_PDL) == 0);
    cudaError_t e = cudaLaunchKernelEx(&launch.cfg, attention::attention_kernel, p);
    if (e != cudaSuccess) return set_error(FU_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    return FU_OK;
}
