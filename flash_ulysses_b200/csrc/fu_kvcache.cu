// The 8-bit K/V cache (sm_100a): the append that quantises full blocks of 64
// tokens, and the attention of single tokens that reads them.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "flash_ulysses_b200.h"
#include "fu_internal.h"
#include "fu_ptx.cuh"

namespace fu {
namespace kvcache {

constexpr int D = FU_HEAD_DIM;
constexpr int BLOCK = FU_KV_BLOCK;

// Status "where" codes of these kernels.
enum : int { W_APPEND = 80, W_ATTENTION = 81 };

// ------------------------------------------------------------ append
struct AppendParams {
    uint8_t* blocks[2];                // K [.., 64, 128], V [.., 128, 64]
    float* scales[2];
    __nv_bfloat16* tail[2];
    const int32_t* block_table;
    const __nv_bfloat16* rows[2];
    int64_t stride[2];
    const int32_t* slots;
    const int32_t* seq_lens;
    const int32_t* cu_seqlens;
    int32_t* status;
    int32_t kv_heads, num_blocks, max_seqs, max_blocks, seqs, tokens;
};

constexpr int APPEND_THREADS = 256;    // 128 for K, 128 for V
constexpr int PITCH = 17;              // words of one dim's 64 transposed bytes, padded

// Work units of a ragged call: sequence i has the units from
// c_i / 64 + 2 i on, c_i its first row.  n rows at any offset touch at most
// (n + 62) / 64 + 1 blocks, and unit_base(i + 1) - unit_base(i) is no less than
// that, so the grid depends on the number of rows and sequences alone.
__host__ __device__ inline int64_t unit_base(int64_t first_row, int64_t i) {
    return first_row / BLOCK + 2 * i;
}

__device__ __forceinline__ int clamp_row(int c, int tokens) { return min(max(c, 0), tokens); }

// Largest finite magnitude bits of two BF16 values, or-ing into `odd` whether
// one is not finite.
__device__ __forceinline__ uint32_t finite_max(uint32_t pair, uint32_t best, bool& odd) {
    const uint32_t a = pair & 0x7fffu, b = (pair >> 16) & 0x7fffu;
    odd = odd || a >= 0x7f80u || b >= 0x7f80u;
    if (a < 0x7f80u) best = max(best, a);
    if (b < 0x7f80u) best = max(best, b);
    return best;
}

// Four tokens' values of one dim -> four e4m3 bytes.
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// One CTA per (work unit, K/V head): one block of 64 tokens, K in threads
// 0..127 and V in 128..255.  A thread holds two groups of 4 tokens x 8 dims:
// coalesced 16-byte loads, the block's largest value by a reduction over the
// 128 threads, and both output orders (tokens x dims for K, dims x tokens for
// V) are words of four bytes.  Bound by memory: each new row is read once and
// leaves as half its bytes.
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(const AppendParams p) {
    __shared__ uint32_t s_max[2][4];
    __shared__ uint32_t s_v[D * PITCH];
    grid_dependency_wait();
    grid_launch_dependents();

    const int h = blockIdx.y;
    const int which = threadIdx.x >> 7;                // 0: K, 1: V
    const int t = threadIdx.x & 127;
    int i = blockIdx.x, j = 0, row0 = i, n = 1;
    if (p.cu_seqlens != nullptr) {
        int a = 0, b = p.seqs;
        while (b - a > 1) {
            const int mid = (a + b) >> 1;
            if (unit_base(clamp_row(__ldg(p.cu_seqlens + mid), p.tokens), mid) <= blockIdx.x)
                a = mid;
            else
                b = mid;
        }
        i = a;
        const int c0 = __ldg(p.cu_seqlens + i), c1 = __ldg(p.cu_seqlens + i + 1);
        if (c0 < 0 || c1 < c0 || c1 > p.tokens || (i == 0 && c0 != 0)) {
            if (threadIdx.x == 0) report_status(p.status, FU_DEV_LENGTHS, W_APPEND);
            return;
        }
        j = blockIdx.x - static_cast<int>(unit_base(c0, i));
        row0 = c0;
        n = c1 - c0;
    }
    const int slot = __ldg(p.slots + i);
    const int len = __ldg(p.seq_lens + i);
    if (slot < 0 || n == 0 || j < 0) return;
    if (slot >= p.max_seqs || len < n || len > p.max_blocks * BLOCK) {
        if (threadIdx.x == 0)
            report_status(p.status, slot >= p.max_seqs ? FU_DEV_CACHE_RANGE : FU_DEV_LENGTHS,
                          W_APPEND);
        return;
    }
    // Two rows of one call that name the same slot would write over each other:
    // the first one counts.
    bool again = false;
    for (int o = threadIdx.x; o < i; o += APPEND_THREADS) again |= __ldg(p.slots + o) == slot;
    if (__syncthreads_or(again)) {
        if (threadIdx.x == 0) report_status(p.status, FU_DEV_SLOT_TWICE, W_APPEND);
        return;
    }

    const int start = len - n;
    const int full = len / BLOCK;                      // blocks that are complete afterwards
    const int b = start / BLOCK + j;
    const __nv_bfloat16* rows = p.rows[which] + static_cast<int64_t>(row0) * p.stride[which] + h * D;
    const int64_t stride = p.stride[which];
    __nv_bfloat16* tail = p.tail[which] + (static_cast<int64_t>(slot) * p.kv_heads + h) * BLOCK * D;
    const int tg = t >> 4, c = t & 15;                 // token group (and tg + 8), 8-dim chunk

    if (b < full) {
        const int id = __ldg(p.block_table + static_cast<int64_t>(slot) * p.max_blocks + b);
        // Tokens of this block held before the call are in the tail.
        uint4 x[2][4];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = (tg + 8 * g) * 4 + r;
                const int pos = b * BLOCK + at - start;
                const __nv_bfloat16* src = pos < 0 ? tail + at * D : rows + pos * stride;
                x[g][r] = *reinterpret_cast<const uint4*>(src + 8 * c);
            }
        uint32_t best = 0;
        bool odd = false;
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                best = finite_max(x[g][r].x, best, odd);
                best = finite_max(x[g][r].y, best, odd);
                best = finite_max(x[g][r].z, best, odd);
                best = finite_max(x[g][r].w, best, odd);
            }
        best = __reduce_max_sync(0xffffffffu, best);
        if ((t & 31) == 0) s_max[which][t >> 5] = best;
        __syncthreads();
        best = max(max(s_max[which][0], s_max[which][1]), max(s_max[which][2], s_max[which][3]));
        // best = (1 + m / 128) 2^(e - 127) in BF16's bits; 448 = 1.75 * 2^8.
        const int e = best >> 7;
        const int power = max(e - 127 - 8 + ((best & 127u) > 96u ? 1 : 0), -126);
        const float scale = __int_as_float((127 + power) << 23);
        const float inv = __int_as_float((127 - power) << 23);
        uint32_t word[2][8];                           // [dim]: the group's four tokens
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                float f[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t w = (&x[g][r].x)[d >> 1];
                    f[r] = __uint_as_float(d & 1 ? w & 0xffff0000u : w << 16) * inv;
                }
                word[g][d] = to_e4m3x4(f[0], f[1], f[2], f[3]);
                if (odd) {                             // infinities and NaN become NaN
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!isfinite(f[r])) word[g][d] |= 0x7fu << (8 * r);
                }
            }
        const bool there = static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks);
        if (!there && threadIdx.x == 0) report_status(p.status, FU_DEV_CACHE_RANGE, W_APPEND);
        const int64_t at = static_cast<int64_t>(id) * p.kv_heads + h;
        if (there && t == 0) p.scales[which][at] = scale;
        uint8_t* dst = p.blocks[which] + at * BLOCK * D;
        if (which == 0) {
            if (there) {
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {      // byte r of each dim's word
                        const uint32_t sel = r | ((r + 4) << 4);
                        const uint32_t lo = __byte_perm(__byte_perm(word[g][0], word[g][1], sel),
                                                        __byte_perm(word[g][2], word[g][3], sel),
                                                        0x5410);
                        const uint32_t hi = __byte_perm(__byte_perm(word[g][4], word[g][5], sel),
                                                        __byte_perm(word[g][6], word[g][7], sel),
                                                        0x5410);
                        *reinterpret_cast<uint2*>(dst + ((tg + 8 * g) * 4 + r) * D + 8 * c) =
                            make_uint2(lo, hi);
                    }
            }
        } else {
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int d = 0; d < 8; ++d) s_v[(8 * c + d) * PITCH + tg + 8 * g] = word[g][d];
        }
        __syncthreads();
        if (which == 1 && there) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {              // 16 bytes of one dim's 64 tokens
                const int dim = k * 32 + (t >> 2), part = (t & 3) * 4;
                const uint32_t* w = s_v + dim * PITCH + part;
                *reinterpret_cast<uint4*>(dst + dim * BLOCK + part * 4) =
                    make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    // The first unit, which alone reads the tail, also writes the rows of the
    // block that stays unfinished (after the barriers above when it read it).
    if (j == 0) {
        const int first = max(full * BLOCK - start, 0);     // first row that goes to the tail
        for (int o = first * 16 + t; o < n * 16; o += 128) {
            const int r = o >> 4, at = (start + r) % BLOCK;
            *reinterpret_cast<uint4*>(tail + at * D + 8 * (o & 15)) =
                *reinterpret_cast<const uint4*>(rows + r * stride + 8 * (o & 15));
        }
    }
}

// ------------------------------------------------------------ attention
struct AttentionParams {
    const uint8_t* blocks[2];
    const float* scales[2];
    const __nv_bfloat16* tail[2];
    const int32_t* block_table;
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    int64_t q_stride, out_stride;
    const int32_t* slots;
    const int32_t* seq_lens;
    const float* alibi_slopes;
    int32_t* status;
    int32_t kv_heads, num_blocks, max_seqs, max_blocks, seqs, group;
    float scale, softcap;
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

__device__ __forceinline__ float e4m3(uint8_t x) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(x, __NV_E4M3)));
}

// One warp per (sequence, query head); lane l holds dims 4l..4l+3.
__global__ void __launch_bounds__(32) attention_kernel(const AttentionParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int i = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
    const int h = head / p.group;
    const int slot = p.slots[i], len = p.seq_lens[i];
    if (slot < 0) return;
    if (slot >= p.max_seqs || len < 0 || len > p.max_blocks * BLOCK) {
        if (lane == 0)
            report_status(p.status, slot >= p.max_seqs ? FU_DEV_CACHE_RANGE : FU_DEV_LENGTHS,
                          W_ATTENTION);
        return;
    }
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int d = 0; d < 4; ++d)
        q[d] = __bfloat162float(p.q[i * p.q_stride + head * D + 4 * lane + d]);
    const float slope = p.alibi_slopes != nullptr ? p.alibi_slopes[head] : 0.f;
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < len; ++j) {
        const int b = j / BLOCK, r = j % BLOCK;
        float k[4], v[4];
        if (b < len / BLOCK) {
            const int id = p.block_table[static_cast<int64_t>(slot) * p.max_blocks + b];
            if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.num_blocks)) {
                if (lane == 0) report_status(p.status, FU_DEV_CACHE_RANGE, W_ATTENTION);
                continue;
            }
            const int64_t at = static_cast<int64_t>(id) * p.kv_heads + h;
            for (int d = 0; d < 4; ++d) {
                k[d] = e4m3(p.blocks[0][at * BLOCK * D + r * D + 4 * lane + d]) * p.scales[0][at];
                v[d] = e4m3(p.blocks[1][at * BLOCK * D + (4 * lane + d) * BLOCK + r]) *
                       p.scales[1][at];
            }
        } else {
            const int64_t at =
                ((static_cast<int64_t>(slot) * p.kv_heads + h) * BLOCK + r) * D + 4 * lane;
            for (int d = 0; d < 4; ++d) {
                k[d] = __bfloat162float(p.tail[0][at + d]);
                v[d] = __bfloat162float(p.tail[1][at + d]);
            }
        }
        float x = p.scale * warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]);
        if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
        x -= slope * static_cast<float>(len - 1 - j);
        const float m2 = fmaxf(m, x);
        const float old = m == m2 ? 1.f : __expf(m - m2);
        const float w = __expf(x - m2);
        m = m2;
        l = l * old + w;
        for (int d = 0; d < 4; ++d) o[d] = o[d] * old + w * v[d];
    }
    for (int d = 0; d < 4; ++d)
        p.out[i * p.out_stride + head * D + 4 * lane + d] =
            __float2bfloat16_rn(l == 0.f ? 0.f : o[d] / l);
}

// ------------------------------------------------------------ host side
static int check_cache(const fu_kvcache* c) {
    if (c == nullptr) return set_error(FU_ERR_INVALID, "null cache");
    if (c->kv_heads < 1 || c->kv_heads > 65535 || c->num_blocks < 1 || c->max_seqs < 1 ||
        c->max_blocks < 1 || c->max_blocks > (INT32_MAX - BLOCK) / BLOCK)
        return set_error(FU_ERR_INVALID, "bad cache sizes");
    const void* ptrs[7] = {c->k_blocks, c->v_blocks, c->k_scales, c->v_scales,
                           c->k_tail, c->v_tail, c->block_table};
    for (const void* ptr : ptrs) {
        if (ptr == nullptr) return set_error(FU_ERR_INVALID, "null cache tensor");
        if (reinterpret_cast<uintptr_t>(ptr) & 15)
            return set_error(FU_ERR_INVALID, "cache tensors must be 16-byte aligned");
    }
    return FU_OK;
}

static int check_rows(const void* ptr, int64_t stride, int heads, const char* name) {
    if (ptr == nullptr) return set_error(FU_ERR_INVALID, "null tensor argument %s", name);
    if ((reinterpret_cast<uintptr_t>(ptr) & 15) || stride % 8 ||
        stride < static_cast<int64_t>(heads) * D || stride > (1ll << 31))
        return set_error(FU_ERR_INVALID, "%s must be 16-byte aligned with a row stride that is a "
                         "multiple of 8 and no less than its width", name);
    return FU_OK;
}

static int check_batch(const int32_t* slots, const int32_t* seq_lens, int32_t seqs,
                       const int32_t* status_host) {
    if (slots == nullptr || seq_lens == nullptr)
        return set_error(FU_ERR_INVALID, "null slots or seq_lens");
    if (seqs < 1 || seqs > (1 << 24))
        return set_error(FU_ERR_INVALID, "seqs %d not in [1, 2^24]", seqs);
    if (status_host != nullptr && *reinterpret_cast<const volatile int32_t*>(status_host) != 0)
        return set_error(FU_ERR_DEVICE, "an earlier launch reported device status 0x%x",
                         static_cast<unsigned>(*status_host));
    return FU_OK;
}

}  // namespace kvcache
}  // namespace fu

using namespace fu;

extern "C" int fu_kvcache_append(const fu_kvcache* c, const void* k, const void* v,
                                 int64_t k_stride, int64_t v_stride, int64_t tokens,
                                 const int32_t* slots, const int32_t* seq_lens,
                                 const int32_t* cu_seqlens, int32_t seqs, int32_t* status,
                                 int32_t* status_host, uint32_t flags, void* stream) {
    int rc = kvcache::check_cache(c);
    if (rc == FU_OK) rc = kvcache::check_rows(k, k_stride, c->kv_heads, "k");
    if (rc == FU_OK) rc = kvcache::check_rows(v, v_stride, c->kv_heads, "v");
    if (rc == FU_OK) rc = kvcache::check_batch(slots, seq_lens, seqs, status_host);
    if (rc != FU_OK) return rc;
    if (tokens < 1 || tokens > (1 << 30) || (cu_seqlens == nullptr && tokens != seqs))
        return set_error(FU_ERR_INVALID, "%lld rows do not go with %d sequences",
                         static_cast<long long>(tokens), seqs);
    kvcache::AppendParams p = {};
    p.blocks[0] = static_cast<uint8_t*>(c->k_blocks);
    p.blocks[1] = static_cast<uint8_t*>(c->v_blocks);
    p.scales[0] = c->k_scales;
    p.scales[1] = c->v_scales;
    p.tail[0] = static_cast<__nv_bfloat16*>(c->k_tail);
    p.tail[1] = static_cast<__nv_bfloat16*>(c->v_tail);
    p.block_table = c->block_table;
    p.rows[0] = static_cast<const __nv_bfloat16*>(k);
    p.rows[1] = static_cast<const __nv_bfloat16*>(v);
    p.stride[0] = k_stride;
    p.stride[1] = v_stride;
    p.slots = slots;
    p.seq_lens = seq_lens;
    p.cu_seqlens = cu_seqlens;
    p.status = status;
    p.kv_heads = c->kv_heads;
    p.num_blocks = c->num_blocks;
    p.max_seqs = c->max_seqs;
    p.max_blocks = c->max_blocks;
    p.seqs = seqs;
    p.tokens = static_cast<int32_t>(tokens);
    const int64_t units = cu_seqlens == nullptr ? seqs : kvcache::unit_base(tokens, seqs);
    DeviceGuard guard(c->device);
    if (!guard.ok()) return set_error(FU_ERR_INVALID, "device %d is not available", c->device);
    Launch launch(dim3(static_cast<unsigned>(units), c->kv_heads), dim3(kvcache::APPEND_THREADS), 0,
                  stream, (flags & FU_FWD_NO_PDL) == 0);
    cudaError_t e = cudaLaunchKernelEx(&launch.cfg, kvcache::append_kernel, p);
    if (e != cudaSuccess) return set_error(FU_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    return FU_OK;
}

extern "C" int64_t fu_kvcache_attention_workspace(int32_t, int32_t q_heads, int32_t kv_heads,
                                                  int32_t seqs) {
    if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || seqs < 1) return 0;
    return 16;
}

extern "C" int fu_kvcache_attention(const fu_kvcache* c, const void* q, int64_t q_stride,
                                    void* out, int64_t out_stride, int32_t q_heads,
                                    const int32_t* slots, const int32_t* seq_lens, int32_t seqs,
                                    float scale, float softcap, const float* alibi_slopes,
                                    void* workspace, int64_t workspace_bytes, int32_t* status,
                                    int32_t* status_host, uint32_t flags, void* stream) {
    int rc = kvcache::check_cache(c);
    if (rc != FU_OK) return rc;
    if (q_heads < 1 || q_heads % c->kv_heads || q_heads > 65535)
        return set_error(FU_ERR_INVALID, "q_heads %d must be a positive multiple of kv_heads %d",
                         q_heads, c->kv_heads);
    rc = kvcache::check_rows(q, q_stride, q_heads, "q");
    if (rc == FU_OK) rc = kvcache::check_rows(out, out_stride, q_heads, "out");
    if (rc == FU_OK) rc = kvcache::check_batch(slots, seq_lens, seqs, status_host);
    if (rc != FU_OK) return rc;
    if (!(softcap >= 0.f) || !std::isfinite(softcap) || !std::isfinite(scale))
        return set_error(FU_ERR_INVALID, "scale must be finite, softcap finite and 0 or more");
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
        workspace_bytes < fu_kvcache_attention_workspace(c->device, q_heads, c->kv_heads, seqs))
        return set_error(FU_ERR_INVALID, "workspace too small or not 16-byte aligned");
    kvcache::AttentionParams p = {};
    p.blocks[0] = static_cast<const uint8_t*>(c->k_blocks);
    p.blocks[1] = static_cast<const uint8_t*>(c->v_blocks);
    p.scales[0] = c->k_scales;
    p.scales[1] = c->v_scales;
    p.tail[0] = static_cast<const __nv_bfloat16*>(c->k_tail);
    p.tail[1] = static_cast<const __nv_bfloat16*>(c->v_tail);
    p.block_table = c->block_table;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.out = static_cast<__nv_bfloat16*>(out);
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.slots = slots;
    p.seq_lens = seq_lens;
    p.alibi_slopes = alibi_slopes;
    p.status = status;
    p.kv_heads = c->kv_heads;
    p.num_blocks = c->num_blocks;
    p.max_seqs = c->max_seqs;
    p.max_blocks = c->max_blocks;
    p.seqs = seqs;
    p.group = q_heads / c->kv_heads;
    p.scale = scale;
    p.softcap = softcap;
    DeviceGuard guard(c->device);
    if (!guard.ok()) return set_error(FU_ERR_INVALID, "device %d is not available", c->device);
    Launch launch(dim3(seqs, q_heads), dim3(32), 0, stream, (flags & FU_FWD_NO_PDL) == 0);
    cudaError_t e = cudaLaunchKernelEx(&launch.cfg, kvcache::attention_kernel, p);
    if (e != cudaSuccess) return set_error(FU_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    return FU_OK;
}
