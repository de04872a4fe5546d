// The 8-bit K/V cache (sm_100a): the append that quantises full blocks of 64
// tokens, and the attention of single tokens that reads them.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
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

constexpr int APPEND_THREADS = 128;
constexpr int PITCH = 17;              // words of one dim's 64 transposed bytes, padded

// Work units of a ragged call: sequence i has the units from
// c_i / 64 + 2 i on, c_i its first row.  n rows at any offset touch at most
// (n + 62) / 64 + 1 blocks, and unit_base(i + 1) - unit_base(i) is no less than
// that, so the grid depends on the number of rows and sequences alone.
__host__ __device__ inline int64_t unit_base(int64_t first_row, int64_t i) {
    return first_row / BLOCK + 2 * i;
}

__device__ __forceinline__ int clamp_row(int c, int tokens) { return min(max(c, 0), tokens); }

// The larger magnitude bits of two BF16 values, if finite, or `best`.
__device__ __forceinline__ uint32_t finite_max(uint32_t pair, uint32_t best) {
    const uint32_t a = pair & 0x7fffu, b = (pair >> 16) & 0x7fffu;
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

// One CTA per (work unit, K/V head, K or V): one block of 64 tokens.  A thread
// holds two groups of 4 tokens x 8 dims: coalesced 16-byte loads, the block's
// largest value by a reduction over the CTA, and both output orders (tokens x dims
// for K, dims x tokens for V) are words of four bytes.  Each new row is read once
// and leaves as half its bytes.  What bounds it is latency: a CTA is one chain of
// loads (the sequence, its length, the rows), and there are two rounds of CTAs with
// nothing in flight between them: 8192 rows of 8 heads take 15.0 us, 3.4 TB/s, where
// memory alone would take 7.9 us.  One trip to memory is all that the search and the
// check for slots named twice add to the chain.  (Nine CTAs per SM: with the 63
// registers that it would take unbounded eight fit, 13.40 us for 13.25 us on inputs that
// are in part in L2.)
__global__ void __launch_bounds__(APPEND_THREADS, 9) append_kernel(const AppendParams p) {
    constexpr uint32_t KEEP_TAIL = 1u << 31;
    __shared__ uint32_t s_max[4];                      // of a warp, and KEEP_TAIL
    __shared__ uint32_t s_v[D * PITCH];
    grid_dependency_wait();
    grid_launch_dependents();

    const int h = blockIdx.y;
    const int which = blockIdx.z;                      // 0: K, 1: V
    const int t = threadIdx.x, lane = threadIdx.x & 31;
    int i = blockIdx.x, j = 0, row0 = i, n = 1;
    if (p.cu_seqlens != nullptr) {
        // All of cu_seqlens is looked at once, by the last unit, which never has rows of its
        // own: where an entry decreases, the search may pass by the sequence that shows it.
        if (blockIdx.x == gridDim.x - 1 && h == 0 && which == 0)
            for (int d = t; d < p.seqs; d += APPEND_THREADS) {
                const int c0 = __ldg(p.cu_seqlens + d), c1 = __ldg(p.cu_seqlens + d + 1);
                if (c1 < c0 || c1 > p.tokens || (d == 0 && c0 != 0))
                    report_status(p.status, FU_DEV_LENGTHS, W_APPEND);
            }
        // The last sequence whose units begin at this one or before: a 32-ary search,
        // one trip to memory up to 32 sequences.
        int lo = 0, count = p.seqs;
        while (count > 1) {
            const int step = (count + 31) / 32, at = lo + lane * step;
            const bool before =
                lane * step < count &&
                unit_base(clamp_row(__ldg(p.cu_seqlens + at), p.tokens), at) <= blockIdx.x;
            const uint32_t others = ~__ballot_sync(0xffffffffu, before);
            const int last = others == 0 ? 31 : max(__ffs(others) - 2, 0);
            lo += last * step;
            count = min(step, count - last * step);
        }
        i = lo;
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
    const int start = len - n;
    const int full = len / BLOCK;                      // blocks that are complete afterwards
    const int b = start / BLOCK + j;
    if (b >= full && j > 0) return;                    // a unit to spare
    // Two rows of one call that name the same slot would write over each other:
    // the first one counts.  (Looked at by the barrier that comes before any write.)
    bool again = false;
    for (int o = threadIdx.x; o < i; o += APPEND_THREADS) again |= __ldg(p.slots + o) == slot;

    const int64_t stride = p.stride[which];
    const __nv_bfloat16* rows = p.rows[which] + row0 * stride + h * D;
    __nv_bfloat16* tail = p.tail[which] + (static_cast<int64_t>(slot) * p.kv_heads + h) * BLOCK * D;
    const int tg = t >> 4, c = t & 15;                 // token group (and tg + 8), 8-dim chunk

    bool keep_tail = false;
    if (b >= full) {
        if (__syncthreads_or(again)) {
            if (threadIdx.x == 0) report_status(p.status, FU_DEV_SLOT_TWICE, W_APPEND);
            return;
        }
    } else {
        const int32_t* table = p.block_table + static_cast<int64_t>(slot) * p.max_blocks;
        const int id = __ldg(table + b);
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
        // The largest magnitude, by BF16's bits (two at a time); only a thread that met
        // an infinity or NaN looks again for the finite ones.
        const uint32_t* words = &x[0][0].x;
        uint32_t both = 0;
#pragma unroll
        for (int k = 0; k < 32; k += 2)
            both = __vimax3_s16x2(both, words[k] & 0x7fff7fffu, words[k + 1] & 0x7fff7fffu);
        uint32_t best = max(both & 0xffffu, both >> 16);
        const bool odd = best >= 0x7f80u;
        if (odd) {
            best = 0;
#pragma unroll
            for (int k = 0; k < 32; ++k) best = finite_max(words[k], best);
        }
        best = __reduce_max_sync(0xffffffffu, best);
        // A tail that holds tokens of a block that is done now is their only source when a
        // call that met a block outside the cache is made again: then it stays.
        if (j == 0 && start % BLOCK != 0) {
            bool outside = false;
            for (int o = b + t; o < full; o += APPEND_THREADS)
                outside |= static_cast<uint32_t>(__ldg(table + o)) >=
                           static_cast<uint32_t>(p.num_blocks);
            if (__any_sync(0xffffffffu, outside)) best |= KEEP_TAIL;
        }
        if (lane == 0) s_max[t >> 5] = best;
        if (__syncthreads_or(again)) {
            if (threadIdx.x == 0) report_status(p.status, FU_DEV_SLOT_TWICE, W_APPEND);
            return;
        }
        keep_tail = ((s_max[0] | s_max[1] | s_max[2] | s_max[3]) & KEEP_TAIL) != 0;
        best = max(max(s_max[0] & ~KEEP_TAIL, s_max[1] & ~KEEP_TAIL),
                   max(s_max[2] & ~KEEP_TAIL, s_max[3] & ~KEEP_TAIL));
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
    if (j == 0 && !keep_tail) {
        const int first = max(full * BLOCK - start, 0);     // first row that goes to the tail
        for (int o = t; o < (n - first) * 16; o += 128) {   // (fewer than 64 rows)
            const int r = first + (o >> 4), at = (start + r) % BLOCK;
            *reinterpret_cast<uint4*>(tail + at * D + 8 * (o & 15)) =
                *reinterpret_cast<const uint4*>(rows + r * stride + 8 * (o & 15));
        }
    }
}

// ------------------------------------------------------------ attention
// Decode: per (sequence, K/V head) the group's query heads are the rows of a
// small matrix product over the sequence's blocks of 64 tokens.  One pass over
// the cache bounds it (256 bytes per token and head), so the work is split
// along the tokens over all SMs and joined afterwards:
//
//   attention_split_kernel   every warp takes a share of whole blocks, with an
//                            online softmax of its own, and writes the output
//                            of a (sequence, head) that it had all of, or a
//                            partial
//   attention_join_kernel    joins the partials of split (sequence, head)s,
//                            in their order, so results do not depend on timing
//
// Warps work alone: a CTA that joined its four warps at the end of each
// (sequence, head) lost 5 to 8 us there to the chain of loads and barriers
// (64 sequences of up to 8192 tokens, 8 K/V heads: 134 us).
//
// A block is two contiguous 8 KiB tiles (K, V transposed), which each warp has
// copied into a ring of its own in shared memory (cp.async.bulk), across the
// borders of sequences.  From there mma.sync (m16n8k16, f16, FP32 accumulation)
// reads them as they lie, 16 bytes per lane and load, with nothing shuffled:
//   * The order of a product's summation index is free as long as both operands
//     agree, so lane (g, t) = (lane / 4, lane % 4) takes 16 consecutive dims of
//     a K row, and the matching dims of q.
//   * Scores come out as rows = query heads, columns = tokens; with K row
//     16 (n / 2) + 2 j + n % 2 as column n of score tile j, lane (g, t) ends up
//     with row g's scores of tokens 16 t .. 16 t + 15, and these are what the
//     second product needs from it next to 16 bytes of a row of V transposed.
//   * e4m3 becomes f16 exactly.  (mma.sync with e4m3 operands, q and the weights
//     as sums of two e4m3, took more instructions per block, 1370 against 1080.)
//   * q is scaled by a power of two per row and the weights by 2^15, so that f16 keeps
//     11 bits of what is down to 2^-28 (2^-29) of the largest; their sums carry the
//     same factor.  (Weights in [0, 1] lost bits from 2^-14 on: the many small ones
//     behind one large score.)  Block scales are applied in FP32.
// tcgen05 would pad 4 to 16 rows to 128; here the tensor work is far below the
// time of the loads, and the instructions per block are what has to stay low.
//
// The unfinished block is BF16 and takes the same route with BF16 products, its
// weights as a sum of two BF16 so that they keep 16 bits.
constexpr int WARPS = 4;
constexpr int SPLIT_THREADS = 32 * WARPS;
constexpr int MAX_BATCH = 1024;        // sequences per launch (prefix sums in shared memory)
constexpr int TILE_BYTES = BLOCK * D;  // one stage of a warp's ring: K or V of a block
constexpr float LOG2E = 1.4426950408889634f;

struct AttentionParams {
    const uint8_t* k_blocks;
    const uint8_t* v_blocks;
    const float* k_scales;
    const float* v_scales;
    const __nv_bfloat16* k_tail;
    const __nv_bfloat16* v_tail;
    const int32_t* block_table;
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    int64_t q_stride, out_stride;
    const int32_t* slots;
    const int32_t* seq_lens;
    const float* alibi_slopes;
    int32_t* status;
    struct Plan* plan;
    float* partial;                    // [worker][2][rows of a pair][PART]
    int32_t kv_heads, num_blocks, max_seqs, max_blocks, seqs, group, row_tiles;
    int32_t workers;                   // warps of the split kernel
    int32_t min_share;                 // of the line of costs (Plan)
    float scale, softcap;
};
constexpr int PART = D + 4;            // one row of a partial: 128 sums, m, l, padding

// How the call's blocks are dealt to the warps.  All (sequence, K/V head, row
// tile)s -- pairs -- lie one after another on a line of costs: a block costs 2,
// the unfinished one 4 (it is BF16), and a pair 1 (its q, its output).  Measured
// on 256 sequences of up to 1500 tokens, where blocks dealt by number left the
// warps between 21 and 36 us.  A block belongs to the warp in whose share of the
// line it starts.
//   aligned (few pairs): every pair is cut into shares of its own, one a warp;
//     those of sequence i begin with warp unit[i].
//   otherwise the line as a whole is cut into equal shares.
// No share is shorter than the widest gap between two starts (3), so every warp
// between a pair's first and last has some of it.
struct alignas(16) Plan {
    int32_t share, aligned;
    int32_t first[MAX_BATCH + 1];      // where sequence i begins on the line
    int32_t unit[MAX_BATCH + 1];
};
constexpr int MIN_SHARE = 3;
__host__ __device__ constexpr int pair_cost(int len) {
    return len <= 0 ? 0 : 1 + 2 * (len / BLOCK) + (len % BLOCK ? 4 : 0);
}
// Where block b of a pair starts, from the pair's start.
__host__ __device__ constexpr int block_start(int b) { return b == 0 ? 0 : 1 + 2 * b; }
// Blocks that start before x (the unfinished one not left out where there is none).
__host__ __device__ constexpr int blocks_before(int x) { return x <= 0 ? 0 : x <= 3 ? 1 : x / 2; }
static_assert(sizeof(Plan) % 16 == 0, "the partials behind it are written 16 bytes at a time");

// Shared memory of a split CTA.  Three stages a warp put 192 KiB per SM in
// flight.
constexpr int STAGES = 3;
struct SplitSmem {
    uint8_t ring[WARPS][STAGES][TILE_BYTES];
    uint64_t full[WARPS][STAGES];
    float scale[WARPS][STAGES];        // of the stage's block
    int32_t first[MAX_BATCH + 1], unit[MAX_BATCH + 1];      // as in Plan
    int32_t slot[MAX_BATCH], len[MAX_BATCH];
    int32_t scan[WARPS];
};
static_assert(2 * (sizeof(SplitSmem) + 1024) <= 228 * 1024, "two CTAs per SM");

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Words {
    uint32_t a[4];
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], const Words& w, uint32_t b0, uint32_t b1) {
    const uint32_t* a = w.a;
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
                 "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four e4m3 bytes -> two pairs of f16.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// `bytes` (a multiple of 16) of global memory -> shared memory, counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes "
                 "[%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Four bytes, counted on `bar` as one arrival when they are there.
__device__ __forceinline__ void async_load_4(uint32_t dst, const void* src, uint32_t bar) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n\t"
                 "cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%2];"
                 ::"r"(dst), "l"(src), "r"(bar) : "memory");
}

// A warp's running softmax and output for its rows: row g (and g + 8 if kWide).
// o[h][dn][c] is row g + 8 h, dim 32 t + 16 c + dn of lane (g, t).
template <bool kWide>
struct Rows {
    static constexpr int H = kWide ? 2 : 1;
    float m[H], l[H], o[H][16][2];
    __device__ void clear() {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.f;
#pragma unroll
            for (int d = 0; d < 16; ++d) o[h][d][0] = o[h][d][1] = 0.f;
        }
    }
};

// A score's path from the product to log2 units, and what it needs of a row.  kMode: 1
// capped by a tanh, 2 lowered with distance, 4 (with 1) by a cap above FINE.
//
// With x = 2 log2(e) z, cap tanh(z) = cap (1 - 2 / (1 + 2^x)) is off by less than 2^-21
// cap: up to a cap of FINE a small part of what rounding the weights to f16 costs.  Larger
// caps matter for scores far below them, which take an odd polynomial of degree 7 in z, off
// by 2e-7 with the slope at 0 exact: relative to the score it is off by less than 2^-19
// (1.0e-6 and the roundings) whatever the cap.  (Both forms in one kernel: 34.8 us instead
// of 33.5 us for 256 sequences of up to 1500 tokens with the first.)
constexpr float FINE = 256.f;
template <int kMode>
struct Score {
    float factor, cap_out, slope;      // per row; with a cap `factor` is that of x
    __device__ float operator()(float raw, float block_scale, int distance) const {
        float x = raw * (factor * block_scale);
        if (kMode & 1) {
            const float far = fmaf(-2.f * cap_out, __fdividef(1.f, 1.f + ex2(x)), cap_out);
            if (kMode & 4) {
                constexpr float Z = 0.5f / LOG2E;              // z = Z x
                const float u = x * x;
                float near = fmaf(u, -0.04422929883003235f * Z * Z * Z * Z * Z * Z * Z,
                                  0.13185861706733704f * Z * Z * Z * Z * Z);
                near = fmaf(near, u, -0.33326461911201477f * Z * Z * Z);
                near = fmaf(near, u, Z) * (x * cap_out);
                x = fabsf(x) <= LOG2E ? near : far;            // |z| = 1/2
            } else {
                x = far;
            }
        }
        if (kMode & 2) x = fmaf(-slope, static_cast<float>(distance), x);
        return x;
    }
};

// One block's scores s[h][j][c] (token 16 t + 2 j + c of the block, already in
// log2 units, -inf where not seen) -> weights in place, times 2^15, and the factor of
// what was summed before.
template <bool kWide>
__device__ __forceinline__ void softmax_step(Rows<kWide>& r, float (&s)[Rows<kWide>::H][8][2],
                                             float (&old)[Rows<kWide>::H]) {
#pragma unroll
    for (int h = 0; h < Rows<kWide>::H; ++h) {
        float top = r.m[h];
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fmaxf(s[h][j][0], s[h][j][1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float base = top == -INFINITY ? 0.f : top;
        old[h] = ex2(r.m[h] - base);
        r.m[h] = top;
        float sum = 0.f;
        const float from = base - 15.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                s[h][j][c] = ex2(s[h][j][c] - from);
                sum += s[h][j][c];
            }
        r.l[h] = fmaf(r.l[h], old[h], sum);            // this lane's tokens only
    }
}

// The last i in [0, n) with x[i] <= v (x does not decrease, x[0] <= v).
__device__ __forceinline__ int last_at_or_before(const int32_t* x, int n, int v) {
    int i = 0;
    while (n - i > 1) {
        const int mid = (i + n) >> 1;
        if (x[mid] <= v) i = mid; else n = mid;
    }
    return i;
}

// A way through a warp's share [at, end), pair by pair.  The feed of the ring
// and the arithmetic each have one.
struct Walk {
    int at, end;                       // the part of the line not entered yet
    int i, pair, b0, b1, nb;           // the current pair, its blocks here [b0, b1) of nb
    int head, row0;                    // the pair's K/V head and first query head of its group
    int slot, len, b;                  // b: the current block
    int id;                            // lane k: cache block of the k-th of 32 blocks

    __device__ bool enter(const SplitSmem& sm, int row_tiles) {
        while (at < end) {
            while (sm.first[i + 1] <= at) ++i;
            slot = sm.slot[i];
            len = sm.len[i];
            nb = (len + BLOCK - 1) / BLOCK;
            const int cost = pair_cost(len);
            pair = (at - sm.first[i]) / cost;
            const int base = sm.first[i] + pair * cost;
            b = b0 = blocks_before(at - base);
            b1 = min(nb, blocks_before(end - base));
            at = base + cost;
            if (b0 >= b1) continue;
            head = row_tiles == 1 ? pair : pair / row_tiles;
            row0 = (pair - head * row_tiles) * 16;
            return true;
        }
        return false;
    }
    __device__ bool is_full() const { return b < len / BLOCK; }
    // Cache block of block b (a full one), -1 if it is outside the cache.  The
    // warp looks up 32 at a time.
    __device__ int lookup(const AttentionParams& p, int lane) {
        const int k = (b - b0) & 31;
        if (k == 0) {
            id = b + lane < min(b1, len / BLOCK)
                     ? __ldg(p.block_table + static_cast<int64_t>(slot) * p.max_blocks + b + lane)
                     : 0;
            if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.num_blocks)) id = -1;
        }
        return __shfl_sync(0xffffffffu, id, k);
    }
};

template <bool kWide, int kMode>
__global__ void __launch_bounds__(SPLIT_THREADS, 2)
attention_split_kernel(const AttentionParams p) {
    constexpr int H = Rows<kWide>::H, ROWS = 8 * H;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    SplitSmem& sm = *reinterpret_cast<SplitSmem*>(smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(smem_u32(&sm.full[warp][s]), 2);
        fence_mbar_init();
    }
    grid_dependency_wait();
    grid_launch_dependents();

    // Prefix sums of the sequences' blocks; a row that is padding or does not
    // fit has none.
    const int pairs = p.kv_heads * p.row_tiles;
    // Sum of x over the threads before this one; adds all of them to `total`.
    const auto scan = [&](int x, int& total) {
        int sum = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        if (lane == 31) sm.scan[warp] = sum;
        __syncthreads();
        int before = total;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += sm.scan[w];
            total += sm.scan[w];
        }
        __syncthreads();
        return before + sum - x;
    };
    constexpr int EACH = 4;            // sequences a thread looks at together
    int total = 0;
    for (int i0 = 0; i0 < p.seqs; i0 += EACH * SPLIT_THREADS) {
        int slot[EACH], len[EACH], sum = 0;
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int i = i0 + EACH * threadIdx.x + k;
            slot[k] = i < p.seqs ? __ldg(p.slots + i) : -1;
            len[k] = i < p.seqs ? __ldg(p.seq_lens + i) : 0;
        }
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int i = i0 + EACH * threadIdx.x + k;
            if (slot[k] < 0) {
                len[k] = 0;
            } else if (slot[k] >= p.max_seqs || len[k] < 0 || len[k] > p.max_blocks * BLOCK) {
                if (blockIdx.x == 0)
                    report_status(p.status,
                                  slot[k] >= p.max_seqs ? FU_DEV_CACHE_RANGE : FU_DEV_LENGTHS,
                                  W_ATTENTION);
                len[k] = 0;
            } else if (len[k] == 0 && i % gridDim.x == blockIdx.x) {
                // A sequence without tokens: its output is 0, and nobody else writes it.
                for (int c = 0; c < p.kv_heads * p.group * D; c += 8)
                    *reinterpret_cast<uint4*>(p.out + i * p.out_stride + c) =
                        make_uint4(0, 0, 0, 0);
            }
            sum += pair_cost(len[k]);
        }
        int before = scan(sum, total);
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int i = i0 + EACH * threadIdx.x + k;
            if (i < p.seqs) {
                sm.slot[i] = slot[k];
                sm.len[i] = len[k];
                sm.first[i] = before * pairs;
            }
            before += pair_cost(len[k]);
        }
    }
    const int line = total * pairs;
    if (threadIdx.x == 0) sm.first[p.seqs] = line;
    // Few pairs: each is cut into shares of its own that give at most one to
    // every warp; else the line is.
    const int all_pairs = p.seqs * pairs;
    const bool aligned = all_pairs <= p.workers / 4;
    const int over = aligned ? p.workers - all_pairs : p.workers;
    const int share = max(line / over + (line % over != 0), p.min_share);
    __syncthreads();
    if (aligned) {
        int units = 0;
        for (int i0 = 0; i0 < p.seqs; i0 += SPLIT_THREADS) {
            const int i = i0 + threadIdx.x;
            const int nb = i < p.seqs ? (sm.len[i] + BLOCK - 1) / BLOCK : 0;
            const int before = scan(nb ? (block_start(nb - 1) / share + 1) * pairs : 0, units);
            if (i < p.seqs) sm.unit[i] = before;
        }
        if (threadIdx.x == 0) sm.unit[p.seqs] = units;
        __syncthreads();
    }
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i <= p.seqs; i += SPLIT_THREADS) {
            p.plan->first[i] = sm.first[i];
            if (aligned) p.plan->unit[i] = sm.unit[i];
        }
        if (threadIdx.x == 0) {
            p.plan->share = share;
            p.plan->aligned = aligned;
        }
    }

    // This warp's share.  Neighbours on the line are on different SMs.
    const int worker = warp * gridDim.x + blockIdx.x;
    Walk walk = {};
    if (aligned) {
        if (worker >= sm.unit[p.seqs]) return;
        const int i = walk.i = last_at_or_before(sm.unit, p.seqs, worker);
        const int cost = pair_cost(sm.len[i]);
        const int per = block_start((sm.len[i] + BLOCK - 1) / BLOCK - 1) / share + 1;
        const int pair = (worker - sm.unit[i]) / per;
        const int part = worker - sm.unit[i] - pair * per;
        walk.at = sm.first[i] + pair * cost + part * share;
        walk.end = min(walk.at + share, sm.first[i] + (pair + 1) * cost);
    } else {
        const int64_t at = static_cast<int64_t>(worker) * share;
        if (at >= line) return;
        walk.at = static_cast<int>(at);
        walk.end = static_cast<int>(min(at + share, static_cast<int64_t>(line)));
        walk.i = last_at_or_before(sm.first, p.seqs, walk.at);
    }

    // The feed: each call requests one stage, in the order in which the warp
    // will read them: K and V of a block; of the unfinished block the 32-row
    // halves of K, then of V.
    Walk feed = walk;
    bool feeding = false;
    int sub = 0, fed = 0;              // part of the current block; the stage to fill next
    const auto request = [&]() {
        while (true) {
            if (!feeding && !feed.enter(sm, p.row_tiles)) return;
            feeding = true;
            if (feed.b >= feed.b1) {
                feeding = false;
                continue;
            }
            const uint8_t* src;
            const float* scale = nullptr;
            int bytes = TILE_BYTES, parts = 2;
            if (feed.is_full()) {
                const int id = feed.lookup(p, lane);
                if (id < 0) {
                    ++feed.b;
                    continue;
                }
                const int64_t block = static_cast<int64_t>(id) * p.kv_heads + feed.head;
                src = (sub ? p.v_blocks : p.k_blocks) + block * TILE_BYTES;
                scale = (sub ? p.v_scales : p.k_scales) + block;
            } else {
                const int left = feed.len % BLOCK;
                const int halves = left > 32 ? 2 : 1;
                parts = 2 * halves;
                const int part = sub % halves;
                src = reinterpret_cast<const uint8_t*>(sub < halves ? p.k_tail : p.v_tail) +
                      (static_cast<int64_t>(feed.slot) * p.kv_heads + feed.head) * 2 * TILE_BYTES +
                      part * TILE_BYTES;
                bytes = min(left - 32 * part, 32) * D * 2;
            }
            if (lane == 0) {
                const uint32_t bar = smem_u32(&sm.full[warp][fed]);
                mbar_arrive_expect_tx(bar, bytes);
                bulk_load(smem_u32(sm.ring[warp][fed]), src, bytes, bar);
                if (scale != nullptr)
                    async_load_4(smem_u32(&sm.scale[warp][fed]), scale, bar);
                else
                    mbar_arrive(bar);
            }
            fed = fed + 1 == STAGES ? 0 : fed + 1;
            if (++sub == parts) {
                sub = 0;
                ++feed.b;
            }
            return;
        }
    };
    int stage = 0;                     // the next stage to read
    uint32_t phase = 0;
    bool alive = true;                 // no wait has given up
    const auto await = [&](int ahead) {
        const int s = stage + ahead;
        const int slot = s >= STAGES ? s - STAGES : s;
        const uint32_t parity = s >= STAGES ? phase ^ 1 : phase;
        const uint32_t bar = smem_u32(&sm.full[warp][slot]);
        if (alive && !mbar_try_wait(bar, parity)) {
            const uint64_t t0 = globaltimer_ns();
            while (alive && !mbar_try_wait(bar, parity))
                if (globaltimer_ns() - t0 > FU_DEFAULT_TIMEOUT_NS) {
                    report_status(p.status, FU_DEV_PIPELINE_TIMEOUT, W_ATTENTION);
                    alive = false;
                }
        }
        return static_cast<const uint8_t*>(sm.ring[warp][slot]);
    };

    // One round per half block: first K (scores and weights), then V (output).
    // A single loop, so that there is one copy of everything: unrolled code that
    // does not fit the instruction caches was what held short sequences up.
    int todo = STAGES;                 // stages to request: those just read
    int half = 0;
    bool open = false;
    int rows = 0;
    const __nv_bfloat16* q = nullptr;
    uint32_t qf[H][16];                // f16, times 2^-e
    Score<kMode> score[H];
    Rows<kWide> r;
    float s[H][8][2], old[H];
    const float raw = kMode & 1 ? 2.f * LOG2E * p.scale / p.softcap : p.scale * LOG2E;
    // Lane's dims of row g + 8 h: word pair y of chunk c covers dims 64 c + 16 t + 4 y .. + 3.
    const auto load_q = [&](int h, int c) {
        return g + 8 * h < rows ? *reinterpret_cast<const uint4*>(
                                      q + (g + 8 * h) * D + 64 * (c >> 1) + 16 * t + 8 * (c & 1))
                                : make_uint4(0, 0, 0, 0);
    };
    while (true) {
        uint4 raw_q[H][4];
        const bool fresh = !open;
        if (fresh) {
            if (!walk.enter(sm, p.row_tiles)) break;
            open = true;
            q = p.q + walk.i * p.q_stride + (walk.head * p.group + walk.row0) * D;
            rows = min(p.group - walk.row0, ROWS);
#pragma unroll
            for (int h = 0; h < H; ++h) {
#pragma unroll
                for (int c = 0; c < 4; ++c) raw_q[h][c] = load_q(h, c);
                score[h].slope =
                    (kMode & 2) && g + 8 * h < rows
                        ? __ldg(p.alibi_slopes + walk.head * p.group + walk.row0 + g + 8 * h) *
                              LOG2E
                        : 0.f;
            }
        }
        __syncwarp();
#pragma unroll 1
        for (; todo > 0; --todo) request();
        if (fresh) {
            r.clear();
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const uint32_t* w = &raw_q[h][0].x;
                float top = 0.f;
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    top = fmaxf(top, fmaxf(fabsf(bf16_lo(w[k])), fabsf(bf16_hi(w[k]))));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // q = (q 2^-e) 2^e with the row's largest value in [2^14, 2^15).
                const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 141, -96), 96);
                const float down = __int_as_float((127 - e) << 23);
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    qf[h][k] = pack_f16x2(bf16_lo(w[k]) * down, bf16_hi(w[k]) * down);
                score[h].factor = raw * __int_as_float((127 + e) << 23);
                score[h].cap_out = p.softcap * LOG2E;
            }
        }

        if (walk.is_full()) {
            if (half == 0 && walk.lookup(p, lane) < 0) {
                report_status(p.status, FU_DEV_CACHE_RANGE, W_ATTENTION);
                half = 1;                              // not seen: neither K nor V is here
            } else if (half == 0) {
                const uint8_t* tile = await(0) + (16 * (g >> 1) + (g & 1)) * D + 16 * t;
                const float ks = sm.scale[warp][stage];
                // Four score tiles at a time: their chains of products overlap.
#pragma unroll
                for (int j0 = 0; j0 < 8; j0 += 4) {
                    float acc[4][4] = {};
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        uint4 x[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            x[j] = *reinterpret_cast<const uint4*>(tile + 2 * (j0 + j) * D +
                                                                   64 * y);
#pragma unroll
                        for (int k = 4 * y; k < 4 * y + 4; ++k)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t b0, b1;
                                e4m3x4_to_f16x4((&x[j].x)[k & 3], b0, b1);
                                mma_f16(acc[j], qf[0][2 * k], kWide ? qf[H - 1][2 * k] : 0u,
                                        qf[0][2 * k + 1], kWide ? qf[H - 1][2 * k + 1] : 0u, b0,
                                        b1);
                            }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int h = 0; h < H; ++h)
#pragma unroll
                            for (int c = 0; c < 2; ++c)
                                s[h][j0 + j][c] = score[h](
                                    acc[j][2 * h + c], ks,
                                    walk.len - 1 - (walk.b * BLOCK + 16 * t + 2 * (j0 + j) + c));
                }
                todo = 1;
                softmax_step<kWide>(r, s, old);
            } else {
                uint32_t pf[H][8];                     // weights of tokens 16 t + 2 k, + 1
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int k = 0; k < 8; ++k) pf[h][k] = pack_f16x2(s[h][k][0], s[h][k][1]);
                const uint8_t* tile = await(0) + 16 * g * BLOCK + 16 * t;
                const float vs = sm.scale[warp][stage];
#pragma unroll
                for (int d0 = 0; d0 < 16; d0 += 4) {
                    uint4 x[4];
                    float acc[4][4] = {};
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        x[d] = *reinterpret_cast<const uint4*>(tile + (d0 + d) * BLOCK);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            uint32_t b0, b1;
                            e4m3x4_to_f16x4((&x[d].x)[k], b0, b1);
                            mma_f16(acc[d], pf[0][2 * k], kWide ? pf[H - 1][2 * k] : 0u,
                                    pf[0][2 * k + 1], kWide ? pf[H - 1][2 * k + 1] : 0u, b0, b1);
                        }
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int h = 0; h < H; ++h)
#pragma unroll
                            for (int c = 0; c < 2; ++c)
                                r.o[h][d0 + d][c] =
                                    fmaf(acc[d][2 * h + c], vs, r.o[h][d0 + d][c] * old[h]);
                }
                todo = 1;
            }
        } else {
            // The unfinished block; rows behind its last token are not read.
            const int left = walk.len % BLOCK;
            const bool both = left > 32;
            const uint8_t* tile = await(0);
            const uint8_t* tile2 = both ? await(1) : tile;
            if (half == 0) {
                tile = g < 4 ? tile : tile2 - TILE_BYTES;             // rows from 32 on
                uint4 qb[H][4];
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c) qb[h][c] = load_q(h, c);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int row = 16 * (g >> 1) + 2 * j + (g & 1);
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint4 x = row < left
                                            ? *reinterpret_cast<const uint4*>(
                                                  tile + (row * D + 64 * (c >> 1) + 16 * t +
                                                          8 * (c & 1)) * 2)
                                            : make_uint4(0, 0, 0, 0);
                        const uint4 q0 = qb[0][c], q1 = qb[H - 1][c];
                        mma_bf16(acc, Words{{q0.x, kWide ? q1.x : 0u, q0.y, kWide ? q1.y : 0u}},
                                 x.x, x.y);
                        mma_bf16(acc, Words{{q0.z, kWide ? q1.z : 0u, q0.w, kWide ? q1.w : 0u}},
                                 x.z, x.w);
                    }
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        Score<kMode> plain = score[h];
                        plain.factor = raw;
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int token = 16 * t + 2 * j + c;
                            const float x = plain(acc[2 * h + c], 1.f, left - 1 - token);
                            s[h][j][c] = token < left ? x : -INFINITY;
                        }
                    }
                }
                softmax_step<kWide>(r, s, old);
            } else {
                tile = t < 2 ? tile : tile2 - TILE_BYTES;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint4 x[4][2];                     // four tokens, dims 16 g .. 16 g + 15
#pragma unroll
                    for (int y = 0; y < 4; ++y)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int row = 16 * t + 4 * k + y;
                            x[y][c] = row < left ? *reinterpret_cast<const uint4*>(
                                                       tile + (row * D + 16 * g + 8 * c) * 2)
                                                 : make_uint4(0, 0, 0, 0);
                        }
                    uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int h = 0; h < H; ++h) {
                            const float w0 = s[h][2 * k + y][0], w1 = s[h][2 * k + y][1];
                            const uint32_t top = pack_bf16x2(w0, w1);
                            hi[2 * y + h] = top;
                            lo[2 * y + h] = pack_bf16x2(w0 - bf16_lo(top), w1 - bf16_hi(top));
                        }
#pragma unroll
                    for (int d = 0; d < 16; ++d) {
                        const uint32_t sel = d & 1 ? 0x7632 : 0x5410;
                        const uint32_t w0 = (&x[0][d >> 3].x)[(d & 7) >> 1];
                        const uint32_t w1 = (&x[1][d >> 3].x)[(d & 7) >> 1];
                        const uint32_t w2 = (&x[2][d >> 3].x)[(d & 7) >> 1];
                        const uint32_t w3 = (&x[3][d >> 3].x)[(d & 7) >> 1];
                        const uint32_t f0 = __byte_perm(w0, w1, sel), f1 = __byte_perm(w2, w3, sel);
                        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int h = 0; h < H; ++h) {
                            acc[2 * h] = k ? r.o[h][d][0] : r.o[h][d][0] * old[h];
                            acc[2 * h + 1] = k ? r.o[h][d][1] : r.o[h][d][1] * old[h];
                        }
                        mma_bf16(acc, Words{{hi[0], hi[1], hi[2], hi[3]}}, f0, f1);
                        mma_bf16(acc, Words{{lo[0], lo[1], lo[2], lo[3]}}, f0, f1);
#pragma unroll
                        for (int h = 0; h < H; ++h) {
                            r.o[h][d][0] = acc[2 * h];
                            r.o[h][d][1] = acc[2 * h + 1];
                        }
                    }
                }
            }
            todo = both ? 2 : 1;
        }
        stage += todo;
        if (stage >= STAGES) {
            stage -= STAGES;
            phase ^= 1;
        }
        half ^= 1;
        if (half == 1) continue;
        if (++walk.b < walk.b1) continue;
        open = false;

        const bool whole = walk.b1 - walk.b0 == walk.nb;
        // A warp shares at most two pairs with others: one that begins before its
        // share (slot 0) and one that ends behind it (slot 1).
        float* part =
            p.partial + (static_cast<int64_t>(worker) * 2 + (walk.b0 == 0)) * ROWS * PART;
        const int64_t out0 =
            walk.i * p.out_stride + (walk.head * p.group + walk.row0) * D;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int row = g + 8 * h;
            float l = r.l[h];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (row >= rows) continue;
            if (whole) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                __nv_bfloat16* out = p.out + out0 + row * D + 32 * t;
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int d = 0; d < 16; d += 8) {
                        uint4 x;
                        uint32_t* w = &x.x;
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            w[y] = pack_bf16x2(r.o[h][d + 2 * y][c] * inv,
                                               r.o[h][d + 2 * y + 1][c] * inv);
                        *reinterpret_cast<uint4*>(out + 16 * c + d) = x;
                    }
            } else {
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int d = 0; d < 16; d += 4)
                        *reinterpret_cast<float4*>(part + row * PART + 32 * t + 16 * c + d) =
                            make_float4(r.o[h][d][c], r.o[h][d + 1][c], r.o[h][d + 2][c],
                                        r.o[h][d + 3][c]);
                if (t == 0) {
                    part[row * PART + D] = r.m[h];
                    part[row * PART + D + 1] = l;
                }
            }
        }
    }
    // Nothing is in flight here unless a wait gave up: then the copies must
    // land before shared memory is released.
    if (!alive) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000) {
        }
    }
}

// Joins the partials of pairs that were split.  Four dims a lane, eight partials in
// flight, with a running maximum.  A pair of few partials gets a warp for each row;
// of many, the CTA's warps share them, row by row, and are joined in order.  Few
// pairs have a CTA of 512 threads for each row, many pairs one of 256 for all rows
// (one of 128 for each row: 1.3 us more for 512 pairs).
struct Joined {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;

    __device__ void add(float4 x, float pm, float pl) {
        const float top = fmaxf(m, pm), base = top == -INFINITY ? 0.f : top;
        const float f = ex2(m - base), g = ex2(pm - base);
        o = make_float4(fmaf(x.x, g, o.x * f), fmaf(x.y, g, o.y * f), fmaf(x.z, g, o.z * f),
                        fmaf(x.w, g, o.w * f));
        l = fmaf(pl, g, l * f);
        m = top;
    }
};

template <int kThreads>
__global__ void __launch_bounds__(kThreads)
attention_join_kernel(const AttentionParams p, int part_rows) {
    constexpr int JOIN_WARPS = kThreads / 32, DEEP = 8, FEW = 2 * DEEP;
    __shared__ float s_m[JOIN_WARPS], s_l[JOIN_WARPS];
    __shared__ float4 s_o[JOIN_WARPS][32];
    grid_dependency_wait();
    grid_launch_dependents();
    const int i = blockIdx.x, pair = blockIdx.y, pairs = gridDim.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = p.plan->first[i], after = p.plan->first[i + 1], share = p.plan->share;
    const int aligned = p.plan->aligned, unit = p.plan->unit[i], len = __ldg(p.seq_lens + i);
    if (first == after) return;
    // The warps of the split that hold a part: the first one's is its slot 1, the
    // others' their slot 0.
    const int last = block_start((len + BLOCK - 1) / BLOCK - 1);
    int c0, c1;
    if (aligned) {
        const int per = last / share + 1;
        c0 = unit + pair * per;
        c1 = c0 + per;
    } else {
        const int base = first + (after - first) / pairs * pair;
        c0 = base / share;
        c1 = (base + last) / share + 1;
    }
    if (c1 - c0 == 1) return;
    const int head = pair / p.row_tiles, row0 = pair % p.row_tiles * 16;
    const int rows = min(p.group - row0, part_rows);

    const auto gather = [&](int row, int from, int step) {
        Joined r;
#pragma unroll 1
        for (int c = from; c < c1; c += DEEP * step) {
            float4 x[DEEP];
            float pm[DEEP], pl[DEEP];
#pragma unroll
            for (int k = 0; k < DEEP; ++k) {
                const int at = c + k * step;
                pm[k] = -INFINITY;
                pl[k] = 0.f;
                x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (at < c1) {
                    const float* src = p.partial + ((static_cast<int64_t>(at) * 2 + (at == c0)) *
                                                        part_rows + row) * PART;
                    x[k] = *reinterpret_cast<const float4*>(src + 4 * lane);
                    pm[k] = src[D];
                    pl[k] = src[D + 1];
                }
            }
            float top = r.m;
#pragma unroll
            for (int k = 0; k < DEEP; ++k) top = fmaxf(top, pm[k]);
            const float base = top == -INFINITY ? 0.f : top;
            float f = ex2(r.m - base);
            r.m = top;
            r.l *= f;
            r.o = make_float4(r.o.x * f, r.o.y * f, r.o.z * f, r.o.w * f);
#pragma unroll
            for (int k = 0; k < DEEP; ++k) {
                f = ex2(pm[k] - base);
                r.l = fmaf(pl[k], f, r.l);
                r.o = make_float4(fmaf(x[k].x, f, r.o.x), fmaf(x[k].y, f, r.o.y),
                                  fmaf(x[k].z, f, r.o.z), fmaf(x[k].w, f, r.o.w));
            }
        }
        return r;
    };
    const auto store = [&](int row, const Joined& r) {
        const float inv = r.l == 0.f ? 0.f : 1.f / r.l;
        *reinterpret_cast<uint2*>(p.out + i * p.out_stride + (head * p.group + row0 + row) * D +
                                  4 * lane) =
            make_uint2(pack_bf16x2(r.o.x * inv, r.o.y * inv),
                       pack_bf16x2(r.o.z * inv, r.o.w * inv));
    };
    if (gridDim.z == 1 && c1 - c0 <= FEW) {
        for (int row = warp; row < rows; row += JOIN_WARPS) store(row, gather(row, c0, 1));
        return;
    }
    for (int row = blockIdx.z; row < rows; row += gridDim.z) {
        Joined r = gather(row, c0 + warp, JOIN_WARPS);
        s_o[warp][lane] = r.o;
        if (lane == 0) {
            s_m[warp] = r.m;
            s_l[warp] = r.l;
        }
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int w = 1; w < JOIN_WARPS; ++w) r.add(s_o[w][lane], s_m[w], s_l[w]);
            store(row, r);
        }
        __syncthreads();
    }
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
    Launch launch(dim3(static_cast<unsigned>(units), c->kv_heads, 2),
                  dim3(kvcache::APPEND_THREADS), 0, stream, (flags & FU_FWD_NO_PDL) == 0);
    cudaError_t e = cudaLaunchKernelEx(&launch.cfg, kvcache::append_kernel, p);
    if (e != cudaSuccess) return set_error(FU_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    return FU_OK;
}

typedef void (*SplitKernel)(kvcache::AttentionParams);
constexpr int MODES = 6;
template <bool kWide>
static SplitKernel split_kernel(int n) {
    static const SplitKernel kernels[MODES] = {
        kvcache::attention_split_kernel<kWide, 0>, kvcache::attention_split_kernel<kWide, 2>,
        kvcache::attention_split_kernel<kWide, 1>, kvcache::attention_split_kernel<kWide, 3>,
        kvcache::attention_split_kernel<kWide, 5>, kvcache::attention_split_kernel<kWide, 7>};
    return kernels[n];
}

// CTAs of the split kernel on a device: two per SM (its shared memory allows no
// more).  Asked once; 0 if there is no such device.
constexpr int MAX_DEVICES = 64;
static int split_ctas(int device) {
    static std::atomic<int> known[MAX_DEVICES];
    if (device < 0 || device >= MAX_DEVICES) return 0;
    int ctas = known[device].load(std::memory_order_relaxed);
    if (ctas == 0) {
        int sms = 0;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        ctas = 2 * sms;
        known[device].store(ctas, std::memory_order_relaxed);
    }
    return ctas;
}

// Raises the split kernels' shared-memory limit once per device (the current one).
static cudaError_t prepare_split(int device) {
    static std::atomic<bool> done[MAX_DEVICES];
    if (done[device].load(std::memory_order_acquire)) return cudaSuccess;
    for (int k = 0; k < 2 * MODES; ++k) {
        cudaError_t e = cudaFuncSetAttribute(k < MODES ? split_kernel<false>(k)
                                                       : split_kernel<true>(k - MODES),
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             sizeof(kvcache::SplitSmem));
        if (e != cudaSuccess) return e;
    }
    done[device].store(true, std::memory_order_release);
    return cudaSuccess;
}

extern "C" int64_t fu_kvcache_attention_workspace(int32_t device, int32_t q_heads,
                                                  int32_t kv_heads, int32_t seqs) {
    if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || seqs < 1) return 0;
    const int rows = q_heads / kv_heads > 8 ? 16 : 8;
    return static_cast<int64_t>(sizeof(kvcache::Plan)) +
           static_cast<int64_t>(split_ctas(device)) * kvcache::WARPS * 2 * rows *
               kvcache::PART * 4;
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
    rc = check_scores(scale, softcap);
    if (rc != FU_OK) return rc;
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
        workspace_bytes < fu_kvcache_attention_workspace(c->device, q_heads, c->kv_heads, seqs))
        return set_error(FU_ERR_INVALID, "workspace too small or not 16-byte aligned");
    kvcache::AttentionParams p = {};
    p.k_blocks = static_cast<const uint8_t*>(c->k_blocks);
    p.v_blocks = static_cast<const uint8_t*>(c->v_blocks);
    p.k_scales = c->k_scales;
    p.v_scales = c->v_scales;
    p.k_tail = static_cast<const __nv_bfloat16*>(c->k_tail);
    p.v_tail = static_cast<const __nv_bfloat16*>(c->v_tail);
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
    p.group = q_heads / c->kv_heads;
    p.row_tiles = (p.group + 15) / 16;
    p.plan = static_cast<kvcache::Plan*>(workspace);
    p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + sizeof(kvcache::Plan));
    const int ctas = split_ctas(c->device);
    if (ctas == 0) return set_error(FU_ERR_INVALID, "device %d is not available", c->device);
    p.workers = ctas * kvcache::WARPS;
    // The longest part of the line that one sequence can take.
    const int64_t per_seq = (2ll * c->max_blocks + 3) * c->kv_heads * p.row_tiles;
    if (per_seq > INT32_MAX)
        return set_error(FU_ERR_INVALID, "max_blocks * kv_heads is too large for one call");
    const int64_t batch = std::min<int64_t>(kvcache::MAX_BATCH, INT32_MAX / per_seq);
    p.scale = scale;
    p.softcap = softcap;
    DeviceGuard guard(c->device);
    if (!guard.ok()) return set_error(FU_ERR_INVALID, "device %d is not available", c->device);
    // Few sequences of a few blocks: a warp takes all of a pair, and there is nothing
    // to join.  (One sequence of 100 tokens, 2 K/V heads: 9.4 us, 10.0 split and joined.)
    constexpr int SHORT_BLOCKS = 4;
    const int64_t largest = std::min<int64_t>(batch, seqs) * c->kv_heads * p.row_tiles;
    const bool unsplit = c->max_blocks <= SHORT_BLOCKS && largest <= p.workers / 4;
    p.min_share = unsplit ? 2 * c->max_blocks + 3 : kvcache::MIN_SHARE;
    const bool wide = p.group > 8, pdl = (flags & FU_FWD_NO_PDL) == 0;
    const int capped = softcap == 0.f ? 0 : softcap <= kvcache::FINE ? 1 : 2;
    const int mode = 2 * capped + (alibi_slopes != nullptr);
    const SplitKernel kernel = wide ? split_kernel<true>(mode) : split_kernel<false>(mode);
    const int smem = sizeof(kvcache::SplitSmem);
    cudaError_t e = prepare_split(c->device);
    if (e != cudaSuccess)
        return set_error(FU_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    for (int64_t done = 0; done < seqs; done += batch) {
        p.seqs = static_cast<int32_t>(std::min(seqs - done, batch));
        p.q = static_cast<const __nv_bfloat16*>(q) + done * q_stride;
        p.out = static_cast<__nv_bfloat16*>(out) + done * out_stride;
        p.slots = slots + done;
        p.seq_lens = seq_lens + done;
        Launch split(dim3(ctas), dim3(kvcache::SPLIT_THREADS), smem, stream, pdl);
        e = cudaLaunchKernelEx(&split.cfg, kernel, p);
        if (e == cudaSuccess && !unsplit) {
            const int rows = std::min(p.group, wide ? 16 : 8);
            const bool few = p.seqs * c->kv_heads * p.row_tiles <= p.workers / 4;
            Launch join(dim3(p.seqs, c->kv_heads * p.row_tiles, few ? rows : 1),
                        dim3(few ? 512 : 256), 0, stream, pdl);
            e = cudaLaunchKernelEx(&join.cfg, few ? kvcache::attention_join_kernel<512>
                                                  : kvcache::attention_join_kernel<256>,
                                   static_cast<const kvcache::AttentionParams>(p), wide ? 16 : 8);
        }
        if (e != cudaSuccess)
            return set_error(FU_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    }
    return FU_OK;
}
