// Attention over the exchanged Q/K/V rows (sm_100a): packed documents, causal,
// prefix or full masks, scores capped by a tanh and/or lowered with distance.
//
// A CTA takes items -- one query head's 256 rows, as two tiles of 128, or 128 rows
// where there are few -- and for each walks the keys that any of the rows sees in
// tiles of 128 with an online softmax:
//     S = Q K^T          tcgen05, Q and K from shared memory, S in TMEM
//     m' = max(m, S), P = 2^(c S - c m'), l = l 2^(c m - c m') + sum P
//     O = O 2^(c m - c m') + P V     tcgen05, P from TMEM, V from shared memory
// c = scale * log2(e); out = O / l.  A thread of the softmax owns one row, so
// the maximum and the sum need no exchange between threads.
//
// 384 threads: warps 0-3 and 4-7 the softmax of tile 0 and tile 1, warp 8 the
// TMA loads, warp 9 the MMA issue (and TMEM), warps 10-11 clean V tiles at the
// edge of a mask (below).  While one tile's scores go through its softmax the
// tensor cores work on the other tile.
//
// The grid has a CTA per item, but one that runs (one per SM) takes over the items of
// CTAs that have not started, one after another.  Warp 8 works out the next one and
// hands it to the others through a ring in shared memory, so that an item's loads
// and first scores run under the end of the one before (a CTA per item spent 3.3 us
// before its first scores and 1.5 us after its last product).  Items go longest
// first; with documents their order is found by counting (Params::ranked).
//
// TMEM (512 columns): S0, S1, O0, O1, 128 columns each; P, two BF16 per
// column, overwrites the first 64 columns of its tile's S.  The tile's next S
// is issued behind the product that reads P, so when S arrives that product
// is complete too and the softmax warps may rescale O in place.  They do so
// only when a row's maximum has grown by more than 2^8 (the reference m may
// lag behind the maximum: P and l stay far inside FP32's and BF16's range),
// which happens in the first tiles of a row and hardly ever after.
//
// Masks: row i sees keys [lo_i, hi_i), both nondecreasing in i, so a tile of
// rows needs the keys [lo_first, hi_last) and only key tiles that cross a
// row's lo or hi apply a mask.  In those a key may be hidden from some rows
// while its V row holds infinities or NaN, and 0 * NaN would reach rows that
// do not see it: warps 10-11 replace what is not finite by 0 in shared memory
// before the product, and if they found any, the epilogue adds it back for the
// rows that see it.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "flash_ulysses_b200.h"
#include "fu_internal.h"
#include "fu_ptx.cuh"

namespace fu {
namespace attention {

constexpr int D = FU_HEAD_DIM;
constexpr int TILE = 128;                       // rows of a query tile, keys of a key tile
constexpr int ROWS = 2 * TILE;                  // query rows of an item, or (few items) TILE
constexpr int NUM_THREADS = 384;
constexpr int TILE_BYTES = TILE * D * 2;        // 32 KiB: two 64-column boxes
constexpr int BOX_BYTES = TILE_BYTES / 2;
constexpr int STAGES = 5;                       // K and V tiles in turn
constexpr int SLOTS = 4;                        // items handed out and not finished
constexpr int SMS = 148;
constexpr int MAX_RANKED = 256;                 // row blocks that are put in order of their length
constexpr int OFF_Q = 0;
constexpr int OFF_KV = OFF_Q + 2 * TILE_BYTES;
constexpr int OFF_ITEM = OFF_KV + STAGES * TILE_BYTES;      // Item[SLOTS]
constexpr int OFF_RANK = OFF_ITEM + SLOTS * 64;             // uint8_t[MAX_RANKED]
constexpr int OFF_BAR = OFF_RANK + MAX_RANKED;
constexpr int OFF_MISC = OFF_BAR + 8 * 40;
constexpr int SMEM_BYTES = OFF_MISC + 64;
constexpr int SMEM_ALLOC = SMEM_BYTES + 1024;   // room to align the base to 1 KiB
static_assert(SMEM_ALLOC <= 232448, "exceeds the 227 KiB per-CTA shared memory limit");
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t TM_S = 0, TM_O = 256;        // + 128 * tile
// Registers: 3 warpgroups launch with 168 each; the softmax takes 208, the
// others keep 88 (208 + 208 + 88 = 3 * 168); neither spills.
constexpr int SOFTMAX_REGS = 208, OTHER_REGS = 88;
constexpr float LOG2E = 1.4426950408889634f;
// Every so manieth pair of a row's weights is computed on the FMA pipes
// (ex2_poly), the others by the special-function unit, whose 16 results per
// clock and SM take as long as the tile's matrix products.  (Every fourth or
// none took the same time or longer; with a cap the FMA pipes are busy with it.)
constexpr int POLY_EVERY = 8;

// Status "where" codes of this kernel.
enum : int {
    W_CU_SEQLENS = 64, W_Q = 65, W_KV_FULL = 66, W_KV_EMPTY = 67, W_S = 68, W_P = 69, W_O = 70,
    W_CLEAN = 71, W_DRAIN = 72, W_ITEM = 73, W_SLOT = 74, W_Q_EMPTY = 75,
};

struct Params {
    CUtensorMap tm_q, tm_k, tm_v;      // [tokens, heads * 128], box {64, 128}, 128-byte swizzle
    const __nv_bfloat16* v;
    __nv_bfloat16* out;
    int64_t v_stride, out_stride;
    const int32_t* cu_seqlens;
    const int32_t* prefix_lens;
    const float* alibi_slopes;
    int32_t* status;
    unsigned long long timeout_ns;
    int32_t tokens, docs, q_heads, group, causal;
    int32_t key_step;                  // from a key tile to the next: 128, or -128 (below)
    int32_t row_blocks;                // row_blocks * q_heads items, a CTA of the grid each
    int32_t block_rows;                // rows of an item: 256 or 128
    int32_t ends_per_item;             // of cu_seqlens, to check
    int32_t ranked;                    // row blocks go by length, else from the last to the first
    int32_t wide_store;                // out rows are 32-byte aligned
    uint32_t negate;                   // scale < 0: the MMA negates Q, `scale` is positive
    float scale, softcap;
};

struct Bars {
    uint32_t q, q_empty, kv_full, kv_empty, clean, s, p, o, item_full, item_empty, done, next;
    __device__ explicit Bars(uint32_t base)
        : q(base), q_empty(q + 16), kv_full(q_empty + 16), kv_empty(kv_full + 8 * STAGES),
          clean(kv_empty + 8 * STAGES), s(clean + 8 * STAGES), p(s + 16), o(p + 32),
          item_full(o + 16), item_empty(item_full + 8 * SLOTS), done(item_empty + 8 * SLOTS),
          next(done + 8) {}
};
static_assert(16 + 16 + 24 * STAGES + 16 + 32 + 16 + 16 * SLOTS + 16 <= 8 * 40, "barrier area");

// Rows [lo, hi) that row i sees; (0, 0) for a row behind the last document.
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

// What every role needs to know of an item.  Key tile j is rows kv0 + 128 j on, with a
// bias kv0 - 128 j (Params::key_step); query tile t takes part in the key tiles
// [first[t], last[t]).
struct Item {
    int row0, head, kv0, tiles;        // tiles < 0: there are no more items
    int first[2], last[2];
    int clear0, clear1;                // key tiles that every row of a document sees all of
    int found;                         // run_clean() took something out
    // Whether some row does not see some key of tile j.
    __device__ bool edge(int j) const { return j < clear0 || j >= clear1; }
};
static_assert(sizeof(Item) <= 64, "item slot");

// Rows of documents, as a bound for the row numbers.
__device__ __forceinline__ int document_rows(const Params& p) {
    if (p.cu_seqlens == nullptr) return p.tokens;
    return min(max(__ldg(p.cu_seqlens + p.docs), 0), p.tokens);
}

// One tile's key tiles from the ranges of its first and last row.
__device__ __forceinline__ void tile_range(int2 head, int2 tail, int kv0, int& first, int& last) {
    first = max(head.x - kv0, 0) / TILE;
    last = max((tail.y - kv0 + TILE - 1) / TILE, first);
}

// The row block's item, by a whole warp; `valid` (> 0) of its rows belong to
// documents.
__device__ __forceinline__ Item make_item(const Params& p, int row0, int head, int valid) {
    const int lane = threadIdx.x & 31;
    int2 seen = make_int2(0, 0);
    if (lane < 4) {
        const int t = lane >> 1, end = min(valid, (t + 1) * TILE) - 1;
        if (valid > t * TILE) seen = seen_rows(p, row0 + (lane & 1 ? end : t * TILE));
    }
    int2 at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        at[k] = make_int2(__shfl_sync(0xffffffffu, seen.x, k), __shfl_sync(0xffffffffu, seen.y, k));
    Item w;
    w.row0 = row0;
    w.head = head;
    w.kv0 = at[0].x;
    w.clear0 = (max((valid > TILE ? at[3].x : at[1].x) - w.kv0, 0) + TILE - 1) / TILE;
    w.clear1 = max(at[0].y - w.kv0, 0) / TILE;
    w.first[1] = w.last[1] = 0;
    tile_range(at[0], at[1], w.kv0, w.first[0], w.last[0]);
    if (valid > TILE) tile_range(at[2], at[3], w.kv0, w.first[1], w.last[1]);
    w.tiles = max(w.last[0], w.last[1]);
    w.found = 0;
    if (p.key_step < 0) {
        // The other way round: tile j becomes tiles - 1 - j.
        w.kv0 += (w.tiles - 1) * TILE;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int first = w.first[t];
            w.first[t] = w.last[t] > first ? w.tiles - w.last[t] : 0;
            w.last[t] = w.last[t] > first ? w.tiles - first : 0;
        }
        const int clear0 = w.clear0;
        w.clear0 = w.tiles - w.clear1;
        w.clear1 = w.tiles - clear0;
    }
    return w;
}

__device__ __forceinline__ bool drain_wait(uint32_t bar, uint32_t parity, uint64_t timeout_ns,
                                           int32_t* status) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (globaltimer_ns() - t0 > timeout_ns) {
            report_status(status, FU_DEV_PIPELINE_TIMEOUT, W_DRAIN);
            return false;
        }
    }
    return true;
}

// The MMAs' issue has to stay ahead of the tensor cores, 64 clocks an instruction,
// in a warp that shares its scheduler with two of the softmax.  So a descriptor is
// not put together for each (only its low word differs, the address in units of 16
// bytes, by constants), and the whole warp runs the issuing code with the same
// values, so that they sit in uniform registers; `one` is set in the lane that
// issues.  (In one lane's branch each operand of each instruction had to be moved
// there: 75 to 110 clocks an instruction.)
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);    // stride 1024, version 1, swizzle 128
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t leading_bytes) {
    return ((saddr >> 4) & 0x3fffu) | ((leading_bytes >> 4) << 16);
}

__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(r));
    return r;
}

// D[tmem] (+)= A[smem] * B[smem], BF16 inputs, FP32 accumulate.
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                       uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)),
          "n"(DESC_HI), "r"(one)
        : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem], BF16 inputs, FP32 accumulate.
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d_tmem, uint32_t a_tmem,
                                       uint32_t b_lo, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)),
          "n"(DESC_HI), "r"(one)
        : "memory");
}

// Arrive on `bar` once every tcgen05 op issued so far by lane `one` is done.
__device__ __forceinline__ void commit(uint32_t one, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(bar), "r"(one) : "memory");
}

// Each thread's 32 (16) registers -> consecutive columns of its TMEM lane.
__device__ __forceinline__ void tmem_st_32cols(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
          "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
          "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
          "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
          "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st_16cols(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
          "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
          "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two FP32 values in one 64-bit register: sm_100 adds and multiplies them with
// one instruction, each rounded as by the scalar one.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float x, float y) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ f32x2 pair(float x) { return pair(x, x); }
__device__ __forceinline__ float2 both(f32x2 x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2_down(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rm.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 2^x of two values without the special-function unit: x = n + f with n = floor(x),
// 2^f by a cubic (minimax on [0, 1), relative error 7.5e-5: a fiftieth of the
// BF16 rounding that follows), 2^n from its exponent bits.  0 below -126, NaN
// stays NaN; x < 128.
__device__ __forceinline__ f32x2 ex2_poly(f32x2 x) {
    constexpr float MAGIC = 12582912.f;               // 1.5 * 2^23: the integer part in the low bits
    const float2 in = both(x);
    const f32x2 xc = pair(max_nan(in.x, -127.f), max_nan(in.y, -127.f));
    const f32x2 t = add2_down(xc, pair(MAGIC));
    const f32x2 f = add2(xc, mul2(add2(t, pair(-MAGIC)), pair(-1.f)));
    f32x2 r = fma2(f, pair(0.07802452147006989f), pair(0.22606715559959412f));
    r = fma2(r, f, pair(0.6958335638046265f));
    r = fma2(r, f, pair(0.9999251961708069f));
    const float2 n = both(t);
    return mul2(r, pair(__int_as_float((__float_as_int(n.x) << 23) + 0x3f800000),
                        __int_as_float((__float_as_int(n.y) << 23) + 0x3f800000)));
}

// One sector with one instruction: 32-byte aligned.
__device__ __forceinline__ void store_32_bytes(void* p, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
                   "r"(r[6]), "r"(r[7])
                 : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16x2_rn(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// ------------------------------------------------------------ items and loads
// Takes over a CTA of this grid that has not started yet; 16 bytes of answer,
// counted on `bar`.
__device__ __forceinline__ void claim_cta(uint32_t answer, uint32_t bar) {
    asm volatile(
        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128"
        " [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}

// The x index of the CTA taken over, -1 if there was none left.
__device__ __forceinline__ int claimed_cta(uint32_t answer) {
    uint32_t x, got;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t.reg .b64 lo, hi;\n\t"
        "ld.shared.v2.b64 {lo, hi}, [%2];\n\tmov.b128 r, {lo, hi};\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %1, 1, 0, p;\n\tmov.u32 %0, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, _, _, _}, r;\n\t}"
        : "=r"(x), "=r"(got) : "r"(answer) : "memory");
    return got ? static_cast<int>(x) : -1;
}

// Reports document ends that do not start at 0, decrease or leave the call: item k's share
// of them, by a whole warp.
__device__ void check_cu_seqlens(const Params& p, int k) {
    const int64_t first = static_cast<int64_t>(k) * p.ends_per_item;
    const int64_t after = min(first + p.ends_per_item, static_cast<int64_t>(p.docs) + 1);
    for (int64_t d = first + (threadIdx.x & 31); d < after; d += 32) {
        const int x = __ldg(p.cu_seqlens + d);
        const int before = d > 0 ? __ldg(p.cu_seqlens + d - 1) : 0;
        if (x < before || x > p.tokens || (d == 0 && x != 0))
            report_status(p.status, FU_DEV_LENGTHS, W_CU_SEQLENS);
    }
    __syncwarp();
}

// Ring order per item: K_0, V_0, K_1, V_1, ...  The whole warp works out the
// items, its first lane loads.
__device__ void run_loads(const Params& p, uint8_t* smem, const Bars& b, volatile int* abort_flag) {
    const uint32_t q = smem_u32(smem + OFF_Q), ring = smem_u32(smem + OFF_KV);
    const uint8_t* rank = smem + OFF_RANK;
    const int lane = threadIdx.x & 31;
    const int rows = document_rows(p);
    const auto wait = [&](uint32_t bar, uint32_t parity, int where) -> bool {
        return __all_sync(0xffffffffu, fu_wait_parity(bar, parity, abort_flag, p.timeout_ns,
                                                      p.status, where));
    };
    int n = 0, stage = 0;              // items handed out, ring stage
    uint32_t use = 0;                  // the stage's phase
    int loads = 0;                     // ring loads issued, up to STAGES
    int q_loads[2] = {0, 0};
    bool ok = true;
    int k = blockIdx.x;                // the item; < 0: there are no more
    uint32_t asked = 0;                // phase of `next`
    // The next item is that of a CTA that has not started, which then never does; asked
    // for when this one's last loads are out.
    const uint32_t answer = smem_u32(smem + OFF_MISC + 16);
    const auto claim = [&]() {
        // With the items, which are all done by someone (any CTA, the first too, may have
        // been taken over).  This one's loads are out, so nothing waits for it.
        if (p.cu_seqlens != nullptr) check_cu_seqlens(p, k);
        if (lane == 0) {
            mbar_arrive_expect_tx(b.next, 16);
            claim_cta(answer, b.next);
        }
        if (!(ok = wait(b.next, asked, W_ITEM))) return -1;
        asked ^= 1;
        const int next = claimed_cta(answer);
        fence_proxy_async_smem();
        __syncwarp();
        return next;
    };
    while (ok) {
        Item w;
        w.tiles = -1;
        if (k >= 0) {
            const int block = k / p.q_heads;
            const int head = k - block * p.q_heads;
            const int row0 = (p.ranked ? rank[block] : p.row_blocks - 1 - block) * p.block_rows;
            const int valid = min(rows - row0, p.block_rows);
            if (valid > 0) w = make_item(p, row0, head, valid);
            if (w.tiles <= 0) {        // (0: cu_seqlens that make no sense)
                k = claim();
                continue;
            }
        }
        const int slot = n % SLOTS;
        const uint32_t phase = (n / SLOTS) & 1;
        if (!(ok = wait(b.item_empty + 8 * slot, phase ^ 1, W_SLOT))) break;
        if (lane == 0) {
            *reinterpret_cast<Item*>(smem + OFF_ITEM + 64 * slot) = w;
            mbar_arrive(b.item_full + 8 * slot);
        }
        __syncwarp();
        if (k < 0) break;
        const int q_col = w.head * D, kv_col = w.head / p.group * D;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (!ok || !(ok = wait(b.q_empty + 8 * t, (n & 1) ^ 1, W_Q_EMPTY))) break;
            ++q_loads[t];
            if (lane == 0) {
                mbar_arrive_expect_tx(b.q + 8 * t, TILE_BYTES);
                for (int c = 0; c < 2; ++c)
                    tma_load_2d(q + t * TILE_BYTES + c * BOX_BYTES, &p.tm_q, b.q + 8 * t,
                                q_col + 64 * c, w.row0 + t * TILE);
            }
            if (t == 1) ++n;
            // The first keys go between the two tiles' rows.
            for (int i = t; ok && i < (t == 0 ? 1 : 2 * w.tiles); ++i) {
                if (!(ok = wait(b.kv_empty + 8 * stage, use ^ 1, W_KV_EMPTY))) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(b.kv_full + 8 * stage, TILE_BYTES);
                    for (int c = 0; c < 2; ++c)
                        tma_load_2d(ring + stage * TILE_BYTES + c * BOX_BYTES,
                                    i & 1 ? &p.tm_v : &p.tm_k, b.kv_full + 8 * stage,
                                    kv_col + 64 * c, w.kv0 + (i >> 1) * p.key_step);
                }
                loads = min(loads + 1, STAGES);
                if (++stage == STAGES) {
                    stage = 0;
                    use ^= 1;
                }
            }
        }
        if (ok) k = claim();
    }
    // What was issued must land before shared memory is released, whatever the
    // other roles did.
    for (int k = 0; k < loads; ++k) {
        if (--stage < 0) {
            stage = STAGES - 1;
            use ^= 1;
        }
        drain_wait(b.kv_full + 8 * stage, use, p.timeout_ns, p.status);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
        if (q_loads[t] > 0) drain_wait(b.q + 8 * t, (q_loads[t] - 1) & 1, p.timeout_ns, p.status);
}

// ------------------------------------------------------------ MMA
__device__ void run_mma(const Params& p, uint8_t* smem, uint32_t tmem, const Bars& b,
                        volatile int* abort_flag) {
    // S = Q K^T: both K-major.  O += P V: P from TMEM, V [keys, dims] MN-major.
    const uint32_t idesc_s = make_idesc_bf16_f32(TILE, TILE, false, false) | (p.negate << 13);
    constexpr uint32_t idesc_o = make_idesc_bf16_f32(TILE, D, false, true);
    const uint32_t q_lo = desc_lo(smem_u32(smem + OFF_Q), 16), ring = smem_u32(smem + OFF_KV);
    const uint32_t one = elect_one();
    const auto wait = [&](uint32_t bar, uint32_t parity, int where) -> bool {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        return __all_sync(0xffffffffu, fu_wait_parity(bar, parity, abort_flag, p.timeout_ns,
                                                      p.status, where));
    };
    const auto same = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
    tmem = same(tmem);
    uint32_t p_phase0 = 0, p_phase1 = 0;
    // Ring stages and phases of the next V and the next K, and the next V's count.
    int sk = 0, sv = 1, sc = 0;
    uint32_t k_phase = 0, v_phase = 0, c_phase = 0;
    // An item's fields; `tiles` < 0 when there are no more.
    struct Range { int first0, first1, last0, last1, tiles, clear0, clear1; };
    int n = 0;                         // items taken
    bool ok = true;
    const auto take = [&]() {
        Range r = {0, 0, 0, 0, -1, 0, 0};
        const int slot = n % SLOTS;
        if (!(ok = wait(b.item_full + 8 * slot, (n / SLOTS) & 1, W_ITEM))) return r;
        const Item& w = *reinterpret_cast<const Item*>(smem + OFF_ITEM + 64 * slot);
        r.first0 = same(w.first[0]);
        r.first1 = same(w.first[1]);
        r.last0 = same(w.last[0]);
        r.last1 = same(w.last[1]);
        r.tiles = same(w.tiles);
        r.clear0 = same(w.clear0);
        r.clear1 = same(w.clear1);
        __syncwarp();
        if (one) mbar_arrive(b.item_empty + 8 * slot);
        ++n;
        return r;
    };
    // A step takes, for one query tile and then the other, the product P V of key
    // tile j and the scores of the key tile after it: j + 1, or the first of the next
    // item, whose work on the first query tile so begins while the second still has
    // the last key tiles of this one to do.
    Range w = {0, 0, 0, 0, 0, 0, 0}, next = take();
    int j = -1;
#pragma unroll 1
    while (ok) {
        const bool turn = j + 1 == w.tiles;            // scores for the next item
        if (turn && j >= 0) next = take();
        if (!ok || (turn && j < 0 && next.tiles < 0)) break;
        const int jn = turn ? 0 : j + 1;
        const bool more = turn ? next.tiles > 0 : true;
        const uint32_t v_lo = desc_lo(ring + sv * TILE_BYTES, BOX_BYTES);   // 64-column boxes
        const uint32_t k_lo = desc_lo(ring + sk * TILE_BYTES, 16);
        const uint32_t v_empty = b.kv_empty + 8 * sv, k_empty = b.kv_empty + 8 * sk;
        if (j >= 0) {
            const bool edge = j < w.clear0 || j >= w.clear1;
            ok = wait(edge ? b.clean + 8 * sc : b.kv_full + 8 * sv, edge ? c_phase : v_phase,
                      edge ? W_CLEAN : W_KV_FULL);
            if (!ok) break;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int first = t ? w.first1 : w.first0, last = t ? w.last1 : w.last0;
            const int firstn = turn ? (t ? next.first1 : next.first0) : first;
            const int lastn = turn ? (t ? next.last1 : next.last0) : last;
            uint32_t& p_phase = t ? p_phase1 : p_phase0;
            if (j >= first && j < last) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (ok) ok = wait(b.p + 16 * t + 8 * half, p_phase, W_P);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 4 * half; k < 4 * half + 4; ++k)
                        mma_ts(one, tmem + TM_O + t * TILE, tmem + TM_S + t * TILE + 8 * k,
                               v_lo + (k * 16 * 128 >> 4), idesc_o, k > 0 || j > first);
                }
                if (!ok) break;
                p_phase ^= 1;
                if (j + 1 == last) commit(one, b.o + 8 * t);
            }
            if (t == 1 && j >= 0) commit(one, v_empty);
            if (!more) continue;
            if (turn && !(ok = wait(b.q + 8 * t, (n - 1) & 1, W_Q))) break;
            if (t == 0 && !(ok = wait(b.kv_full + 8 * sk, k_phase, W_KV_FULL))) break;
            if (jn >= firstn && jn < lastn) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t at = ((k / 4) * BOX_BYTES + (k % 4) * 32) >> 4;
                    mma_ss(one, tmem + TM_S + t * TILE, q_lo + t * (TILE_BYTES >> 4) + at,
                           k_lo + at, idesc_s, k > 0);
                }
                commit(one, b.s + 8 * t);
            }
            // The tile's rows are no longer needed (a tile without rows: at once).
            if (lastn > firstn ? jn + 1 == lastn : turn) commit(one, b.q_empty + 8 * t);
            if (t == 1) commit(one, k_empty);
        }
        if (!ok || !more) break;
        if (j >= 0) {
            sv = sv + 2 < STAGES ? sv + 2 : (v_phase ^= 1, sv + 2 - STAGES);
            sc = sc + 1 < STAGES ? sc + 1 : (c_phase ^= 1, 0);
        }
        sk = sk + 2 < STAGES ? sk + 2 : (k_phase ^= 1, sk + 2 - STAGES);
        if (turn) w = next;
        j = jn;
    }
    // Every MMA this warp issued must finish before TMEM is released.
    commit(one, b.done);
    drain_wait(b.done, 0, p.timeout_ns, p.status);
}

// ------------------------------------------------------------ V at a mask's edge
// These warps take every load off the ring in its order, K tiles too, and give each
// stage back as the products do: by its parity alone a phase of kv_full cannot be told
// from the one two before or behind, so a warp that waits for a stage must have seen its
// last load, and the stage must not be filled again before it has seen this one.  Every V
// tile is counted on a ring of barriers of its own; only those at an edge are looked at.
__device__ void run_clean(const Params& p, uint8_t* smem, const Bars& b,
                          volatile int* abort_flag) {
    const int me = threadIdx.x & 63;
    int stage = 0, count = 0;          // ring stage of the next load, place of the next V tile
    uint32_t use = 0;
    const auto full = [&]() {
        return __all_sync(0xffffffffu, fu_wait_parity(b.kv_full + 8 * stage, use, abort_flag,
                                                      p.timeout_ns, p.status, W_KV_FULL));
    };
    const auto give_back = [&]() {
        __syncwarp();
        if ((me & 31) == 0) mbar_arrive(b.kv_empty + 8 * stage);
        if (++stage == STAGES) {
            stage = 0;
            use ^= 1;
        }
    };
    for (int n = 0;; ++n) {
        const int slot = n % SLOTS;
        const bool ok = fu_wait_parity(b.item_full + 8 * slot, (n / SLOTS) & 1, abort_flag,
                                       p.timeout_ns, p.status, W_ITEM);
        if (!__all_sync(0xffffffffu, ok)) return;
        Item& w = *reinterpret_cast<Item*>(smem + OFF_ITEM + 64 * slot);
        const int tiles = w.tiles;
        for (int j = 0; j < tiles; ++j) {
            if (!full()) return;                       // K
            give_back();
            if (!full()) return;                       // V
            if (w.edge(j)) {
                uint4* v = reinterpret_cast<uint4*>(smem + OFF_KV + stage * TILE_BYTES);
                // A BF16 is not finite if its exponent bits are all set; one more then
                // carries into the sign's place.
                uint32_t bad = 0;
#pragma unroll 8
                for (int o = me; o < TILE_BYTES / 16; o += 64) {
                    const uint4 x = v[o];
                    bad |= ((x.x & 0x7f807f80u) + 0x00800080u) | ((x.y & 0x7f807f80u) + 0x00800080u) |
                           ((x.z & 0x7f807f80u) + 0x00800080u) | ((x.w & 0x7f807f80u) + 0x00800080u);
                }
                if (bad & 0x80008000u) {
#pragma unroll 1
                    for (int o = me; o < TILE_BYTES / 16; o += 64) {
                        uint4 x = v[o];
                        uint32_t* word = &x.x;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            word[k] &= ~__vcmpeq2(word[k] & 0x7f807f80u, 0x7f807f80u);
                        v[o] = x;
                    }
                    *const_cast<volatile int*>(&w.found) = 1;
                    fence_proxy_async_smem();
                }
            }
            __syncwarp();
            if ((me & 31) == 0) mbar_arrive(b.clean + 8 * count);
            if (++count == STAGES) count = 0;
            give_back();
        }
        __syncwarp();
        if ((me & 31) == 0) mbar_arrive(b.item_empty + 8 * slot);
        if (tiles < 0) return;
    }
}

// ------------------------------------------------------------ softmax
// kMode: 1 scores capped by a tanh, 2 lowered with distance (3 both).
template <int kMode>
__device__ void run_softmax(const Params& p, uint8_t* smem, uint32_t tmem, const Bars& b, int t,
                            volatile int* abort_flag) {
    const int lane = threadIdx.x & 31;
    const int warp = (threadIdx.x >> 5) & 3;              // of this tile
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t tm_s = tmem + TM_S + t * TILE + lanes, tm_o = tmem + TM_O + t * TILE + lanes;
    // Scores in units of log2: x = c * s here, m in the units of s (so c m is
    // its logarithm), or with a cap or a bias x = s, c = 1.
    const float c = kMode ? 1.f : fmaxf(p.scale * LOG2E, 1e-30f);
    const float lin = p.scale * LOG2E;
    const float to_cap = kMode & 1 ? p.scale / p.softcap : 0.f;
    const float z2 = to_cap * to_cap;
    // tanh(z) = z + .. to z^7 for |z| <= 1/2, off by 2e-7, as a polynomial in s, where
    // its coefficients stay within FP32's range.
    const float cap_low[4] = {lin, -0.33326461911201477f * lin * z2,
                              0.13185861706733704f * lin * z2 * z2,
                              -0.04422929883003235f * lin * z2 * z2 * z2};
    const bool cap_small = to_cap >= 1e-5f && to_cap <= 1e4f;
    const auto wait = [&](uint32_t bar, uint32_t parity, int where) -> bool {
        return __all_sync(0xffffffffu, fu_wait_parity(bar, parity, abort_flag, p.timeout_ns,
                                                      p.status, where));
    };
    uint32_t phase = 0, o_phase = 0;
    for (int n = 0;; ++n) {
        const int slot = n % SLOTS;
        if (!wait(b.item_full + 8 * slot, (n / SLOTS) & 1, W_ITEM)) return;
        const Item& w = *reinterpret_cast<const Item*>(smem + OFF_ITEM + 64 * slot);
        if (w.tiles < 0) return;
        const int first = w.first[t], last = w.last[t], kv0 = w.kv0;
        const int row = w.row0 + t * TILE + warp * 32 + lane;
        const float slope = kMode & 2 ? __ldg(p.alibi_slopes + w.head) * LOG2E : 0.f;
        const int2 seen = row < p.tokens ? seen_rows(p, row) : make_int2(0, 0);
        const bool valid = seen.x < seen.y;
        // A row without a document is computed like one that sees everything, and not
        // stored.
        const int lo = valid ? seen.x : 0, hi = valid ? seen.y : INT_MAX / 2;
        // What some and what all of the warp's rows of documents see.
        constexpr uint32_t ALL = 0xffffffffu;
        const int lo_some = __reduce_min_sync(ALL, valid ? seen.x : INT_MAX);
        const int lo_all = __reduce_max_sync(ALL, valid ? seen.x : INT_MIN);
        const int hi_some = __reduce_max_sync(ALL, valid ? seen.y : INT_MIN);
        const int hi_all = __reduce_min_sync(ALL, valid ? seen.y : INT_MAX);
        // A bias may be taken from its ends (below) as long as 32 keys change it little.
        const bool flat = fabsf(slope) <= 1.f;

        float m = -INFINITY, l = 0.f;
        for (int j = first; j < last; ++j) {
            if (!wait(b.s + 8 * t, phase, W_S)) return;
            phase ^= 1;
            tc_fence_after();
            const int k0 = kv0 + j * p.key_step;
            if (hi_some <= k0 || lo_some >= k0 + TILE) {
                // Other rows' document or prefix, nothing for this warp's.  (Computed and
                // masked, 8191 tokens in 3 documents took 116 us instead of 110 us: the
                // longest item ends one document and begins the next.)
                const uint32_t none[16] = {};
#pragma unroll
                for (int k = 0; k < 4; ++k) tmem_st_16cols(tm_s + 16 * k, none);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane < 2) mbar_arrive(b.p + 16 * t + 8 * lane);
                continue;
            }
            uint32_t r[TILE];
            float* s = reinterpret_cast<float*>(r);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                tmem_ld_32cols(tm_s + 32 * k, *reinterpret_cast<uint32_t(*)[32]>(r + 32 * k));
            tmem_ld_wait();
            if (kMode & 1) {
                // cap tanh(z), z = scale s / cap.  Where all of the warp's |z| are at most
                // 1/2 (scores well below the cap, the ordinary case) by an odd polynomial
                // of degree 7, at most 1 by one of degree 11, off by 7.3e-7 with the slope at 0
                // exact; else as cap (1 - 2 / (1 + 2^(2 log2(e) z))), off by less than 2^-21.
                // Times the cap these are absolute errors, which for a cap above FINE matter for
                // scores far below it: there the last form takes the polynomial for |z| <= 1,
                // and a score is off by less than 2^-19 of itself (1.2e-6 and the roundings).
                // What a cap costs is its instructions between a row's scores and its weights:
                // 8192 tokens of 8 heads take 1040 a warp and key tile, 695 without, and 161 us
                // for 115, while no pipe is busy for more than 46 % of the time; the last form
                // also takes three special-function results per score with the weight's.
                constexpr float FINE = 1024.f;
                const f32x2 to_cap2 = pair(to_cap), lin2 = pair(lin);
                const auto degree_11 = [&](f32x2 x) {
                    const f32x2 z = mul2(x, to_cap2), u = mul2(z, z);
                    f32x2 h = fma2(u, pair(-0.0030804092530161142f), pair(0.016842123121023178f));
                    h = fma2(h, u, pair(-0.051767539232969284f));
                    h = fma2(h, u, pair(0.1329089254140854f));
                    h = fma2(h, u, pair(-0.3333089351654053f));
                    h = fma2(h, u, pair(1.f));
                    return both(mul2(mul2(x, lin2), h));
                };
                float far = 0.f;
#pragma unroll
                for (int k = 0; k < TILE; k += 2) far = max3(far, fabsf(s[k]), fabsf(s[k + 1]));
                if (__all_sync(0xffffffffu, cap_small && far * to_cap <= 0.5f)) {
#pragma unroll
                    for (int k = 0; k < TILE; k += 2) {
                        const f32x2 x = pair(s[k], s[k + 1]), u = mul2(x, x);
                        f32x2 h = fma2(u, pair(cap_low[3]), pair(cap_low[2]));
                        h = fma2(h, u, pair(cap_low[1]));
                        h = fma2(h, u, pair(cap_low[0]));
                        const float2 y = both(mul2(x, h));
                        s[k] = y.x;
                        s[k + 1] = y.y;
                    }
                } else if (__all_sync(0xffffffffu, far * to_cap <= 1.f)) {
#pragma unroll
                    for (int k = 0; k < TILE; k += 2) {
                        const float2 y = degree_11(pair(s[k], s[k + 1]));
                        s[k] = y.x;
                        s[k + 1] = y.y;
                    }
                } else {
                    const float in = 2.f * LOG2E * to_cap, out = p.softcap * LOG2E;
                    const auto full = [&](float x) {
                        return fmaf(-2.f * out, __fdividef(1.f, 1.f + ex2(x * in)), out);
                    };
                    if (p.softcap <= FINE) {
#pragma unroll
                        for (int k = 0; k < TILE; ++k) s[k] = full(s[k]);
                    } else {
#pragma unroll
                        for (int k = 0; k < TILE; k += 2) {
                            const float2 y = degree_11(pair(s[k], s[k + 1]));
                            s[k] = fabsf(s[k] * to_cap) <= 1.f ? y.x : full(s[k]);
                            s[k + 1] = fabsf(s[k + 1] * to_cap) <= 1.f ? y.y : full(s[k + 1]);
                        }
                    }
                }
            }
            // With a bias: x = times * s + start[k / 32] + step * (k % 32).
            float times = 1.f, step = 0.f, start[4] = {0.f, 0.f, 0.f, 0.f};
            if (kMode & 2) {
                // Without keys behind the row, or with only such, |i - j| is linear in j
                // (keys that a causal mask hides may come out as they like).  There the
                // bias joins the scores in the exponent, and the maximum is taken from its
                // larger end for each 32 keys: at most 2^31 above the true one, which FP32
                // has room for.
                const bool below = (p.causal && p.prefix_lens == nullptr) ||
                                   k0 + TILE - 1 <= row - lane;
                const bool above = k0 >= row - lane + 31;
                if ((below || above) && flat) {
                    times = kMode & 1 ? 1.f : fmaxf(lin, 1e-30f);
                    step = below ? slope : -slope;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        start[k] = static_cast<float>(k0 + 32 * k - row) * step;
                } else {
                    const float at = static_cast<float>(row - k0);
#pragma unroll
                    for (int k = 0; k < TILE; ++k)
                        s[k] = fmaf(-slope, fabsf(at - static_cast<float>(k)),
                                    kMode & 1 ? s[k] : s[k] * lin);
                }
            }
            if (hi_all < k0 + TILE || lo_all > k0) {
                // A bit for each key that the row sees: tested in place, two instructions a
                // score.  (Two comparisons with the ends: 4096 packed tokens 68 us, 58 us
                // with the bits.)
                const auto before = [](int n) {
                    return static_cast<uint32_t>((1ull << min(max(n, 0), 32)) - 1);
                };
#pragma unroll
                for (int k = 0; k < TILE; k += 32) {
                    const uint32_t sees = before(hi - k0 - k) & ~before(lo - k0 - k);
#pragma unroll
                    for (int q = 0; q < 32; ++q) s[k + q] = sees >> q & 1 ? s[k + q] : -INFINITY;
                }
            }
            float best[4];
#pragma unroll
            for (int k = 0; k < TILE; k += 2) {
                // Four running maxima: of 32 neighbours with a bias.
                float& x = best[kMode & 2 ? k >> 5 : (k >> 1) & 3];
                const bool begin = kMode & 2 ? k % 32 == 0 : k < 8;
                x = begin ? fmaxf(s[k], s[k + 1]) : max3(x, s[k], s[k + 1]);
            }
            if (kMode & 2) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    best[k] = fmaf(best[k], times, fmaxf(start[k], fmaf(31.f, step, start[k])));
            }
            const float top = fmaxf(max3(best[0], best[1], best[2]), fmaxf(best[3], m));
            if (j == first) {
                m = top;
            } else if (__any_sync(0xffffffffu, (top - m) * c > 8.f)) {
                const float f = top == -INFINITY ? 1.f : ex2((m - top) * c);
                l *= f;
                m = top;
#pragma unroll 1
                for (int k = 0; k < 4; ++k) {
                    uint32_t o[32];
                    tmem_ld_32cols(tm_o + 32 * k, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int q = 0; q < 32; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
                    tmem_st_32cols(tm_o + 32 * k, o);
                }
            }
            const float zero = m == -INFINITY ? 0.f : -m * c;
            const f32x2 times2 = pair(kMode & 2 ? times : c), step2 = pair(2.f * step);
            f32x2 sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t packed[16];
                f32x2 base = kMode & 2 ? pair(start[k] + zero, start[k] + zero + step) : pair(zero);
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const f32x2 x = pair(s[32 * k + 2 * q], s[32 * k + 2 * q + 1]);
                    f32x2 y = kMode == 1 ? add2(x, base) : fma2(x, times2, base);
                    if (kMode & 2) base = add2(base, step2);
                    if (!(kMode & 1) && q % POLY_EVERY == POLY_EVERY - 1) {
                        y = ex2_poly(y);
                    } else {
                        const float2 z = both(y);
                        y = pair(ex2(z.x), ex2(z.y));
                    }
                    sum[q & 3] = add2(sum[q & 3], y);
                    const float2 z = both(y);
                    packed[q] = pack_bf16x2_rn(z.x, z.y);
                }
                tmem_st_16cols(tm_s + 16 * k, packed);
                if (k & 1) {
                    // Half of P is there: the product may begin.
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(b.p + 16 * t + 8 * (k >> 1));
                }
            }
            const float2 total = both(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
            l += total.x + total.y;
        }
        if (first < last) {
            // out = O / l, a row of 256 bytes a thread.
            if (!wait(b.o + 8 * t, o_phase, W_O)) return;
            o_phase ^= 1;
            tc_fence_after();
            const float inv = 1.f / l;
            const bool poison = *const_cast<const volatile int*>(&w.found) != 0;
            __nv_bfloat16* dst = p.out + static_cast<int64_t>(row) * p.out_stride + w.head * D;
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
                uint32_t o[32];
                tmem_ld_32cols(tm_o + 32 * k, o);
                tmem_ld_wait();
#pragma unroll
                for (int q = 0; q < 32; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * inv);
                if (poison && valid) {
                    // What run_clean() took out, for the rows that see it.
                    for (int j = first; j < last; ++j) {
                        if (!w.edge(j)) continue;
                        const int k0 = kv0 + j * p.key_step;
                        const int a = max(lo, k0), e = min(hi, k0 + TILE);
                        for (int key = a; key < e; ++key) {
                            const __nv_bfloat16* v =
                                p.v + key * p.v_stride + w.head / p.group * D + 32 * k;
#pragma unroll
                            for (int q = 0; q < 32; ++q) {
                                const float x = __bfloat162float(v[q]);
                                if (!isfinite(x)) o[q] = __float_as_uint(__uint_as_float(o[q]) + x);
                            }
                        }
                    }
                }
                uint32_t packed[16];
#pragma unroll
                for (int q = 0; q < 16; ++q)
                    packed[q] =
                        pack_bf16x2_rn(__uint_as_float(o[2 * q]), __uint_as_float(o[2 * q + 1]));
                if (!valid) continue;
                if (p.wide_store) {
                    store_32_bytes(dst + 32 * k, packed);
                    store_32_bytes(dst + 32 * k + 16, packed + 8);
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<uint4*>(dst + 32 * k + 8 * q) = make_uint4(
                            packed[4 * q], packed[4 * q + 1], packed[4 * q + 2], packed[4 * q + 3]);
                }
            }
            // The next product into O comes behind weights of these warps.
            tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(b.item_empty + 8 * slot);
    }
}

// ------------------------------------------------------------ kernel
template <int kMode>
__global__ void __launch_bounds__(NUM_THREADS, 1)
attention_kernel(const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5;
    const Bars b(smem_u32(smem + OFF_BAR));
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + OFF_MISC);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + OFF_MISC + 4);

    // Prologue: shared memory, TMEM and parameters only (it may overlap the
    // previous kernel of the stream under a programmatic dependent launch).
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(b.kv_full + 8 * s, 1);
            mbar_init(b.kv_empty + 8 * s, 3);          // the products, two cleaning warps
            mbar_init(b.clean + 8 * s, 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(b.q + 8 * t, 1);
            mbar_init(b.q_empty + 8 * t, 1);
            mbar_init(b.s + 8 * t, 1);
            mbar_init(b.p + 16 * t, 4);
            mbar_init(b.p + 16 * t + 8, 4);
            mbar_init(b.o + 8 * t, 1);
        }
        for (int k = 0; k < SLOTS; ++k) {
            mbar_init(b.item_full + 8 * k, 1);
            mbar_init(b.item_empty + 8 * k, 11);       // warps: 8 softmax, MMA, 2 cleaning
        }
        mbar_init(b.done, 1);
        mbar_init(b.next, 1);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&p.tm_q);
        tma_prefetch_desc(&p.tm_k);
        tma_prefetch_desc(&p.tm_v);
    }
    if (warp == 9) {
        tmem_alloc(smem_u32(tmem_holder), TMEM_COLS);
        tmem_relinquish();
    }
    // Global memory from here on: the previous kernel of the stream is done.
    grid_dependency_wait();
    grid_launch_dependents();

    if (p.ranked) {
        // Row blocks by the key tiles that their two query tiles walk, longest
        // first: each counts those that go before it.
        int* cost = reinterpret_cast<int*>(smem + OFF_KV);
        const int me = threadIdx.x, rows = document_rows(p);
        int mine = 0;
        if (me < p.row_blocks) {
            const int row0 = me * p.block_rows, valid = min(rows - row0, p.block_rows);
            int kv0 = 0;
            for (int t = 0; t < 2 && valid > t * TILE; ++t) {
                const int2 head = seen_rows(p, row0 + t * TILE);
                const int2 tail = seen_rows(p, row0 + min(valid, (t + 1) * TILE) - 1);
                if (t == 0) kv0 = head.x;
                int first, last;
                tile_range(head, tail, kv0, first, last);
                mine += last - first;
            }
            cost[me] = mine;
        }
        __syncthreads();
        if (me < p.row_blocks) {
            int before = 0;
            for (int k = 0; k < p.row_blocks; ++k) {
                const int other = cost[k];
                before += other > mine || (other == mine && k > me);
            }
            smem[OFF_RANK + before] = static_cast<uint8_t>(me);
        }
        fence_proxy_async_smem();                      // the ring's loads go over `cost`
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
        run_softmax<kMode>(p, smem, tmem, b, warp >> 2, abort_flag);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        if (warp == 8)
            run_loads(p, smem, b, abort_flag);
        else if (warp == 9)
            run_mma(p, smem, tmem, b, abort_flag);
        else
            run_clean(p, smem, b, abort_flag);
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_dealloc(tmem, TMEM_COLS);
}

// ------------------------------------------------------------ host side
// BF16 [rows, cols] with a row stride, box {64, 128}, 128-byte swizzle.
static int encode_rows(CUtensorMap* map, const void* base, int64_t rows, int64_t cols,
                       int64_t stride, const char* what) {
    auto fn = encode_tiled_fn();
    if (fn == nullptr) return set_error(FU_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
    const cuuint32_t box[2] = {64, TILE};
    const cuuint32_t elem[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
                    strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(FU_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with %d", what,
                         static_cast<int>(r));
    return FU_OK;
}

typedef void (*Kernel)(const Params);

// Raises the kernels' shared-memory limit once per device (the current one).
static cudaError_t prepare(int device) {
    constexpr int MAX_DEVICES = 64;
    static std::atomic<bool> done[MAX_DEVICES];
    if (device < MAX_DEVICES && done[device].load(std::memory_order_acquire)) return cudaSuccess;
    for (Kernel k : {attention_kernel<0>, attention_kernel<1>, attention_kernel<2>,
                     attention_kernel<3>}) {
        cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             SMEM_ALLOC);
        if (e != cudaSuccess) return e;
    }
    if (device < MAX_DEVICES) done[device].store(true, std::memory_order_release);
    return cudaSuccess;
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
    int rc = check_scores(a->scale, a->softcap);
    if (rc != FU_OK) return rc;
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

    // Two tiles of 128 rows keep a CTA's tensor cores busy in turn.  Where the call has at
    // most two tiles per SM an item is one tile: more CTAs, and shorter ones.  (700 tokens of
    // 8 heads 14.1 us, 15.9 us with two; 2048 of 4 heads 30.3 and 32.2 us; 6800 of 4 heads, 216
    // tiles, 88.8 and 92.5 us.)
    const int64_t tiles = (a->tokens + attention::TILE - 1) / attention::TILE;
    const int block_rows = tiles * a->q_heads <= 2 * attention::SMS ? attention::TILE : attention::ROWS;
    const int64_t row_blocks = (a->tokens + block_rows - 1) / block_rows;
    const int64_t blocks = row_blocks * a->q_heads;
    if (blocks > INT32_MAX)
        return set_error(FU_ERR_INVALID, "tokens * q_heads is too large for one call");

    attention::Params p = {};
    rc = attention::encode_rows(&p.tm_q, a->q, a->tokens, a->q_heads * attention::D, a->q_stride,
                                "q");
    if (rc == FU_OK)
        rc = attention::encode_rows(&p.tm_k, a->k, a->tokens, a->kv_heads * attention::D,
                                    a->k_stride, "k");
    if (rc == FU_OK)
        rc = attention::encode_rows(&p.tm_v, a->v, a->tokens, a->kv_heads * attention::D,
                                    a->v_stride, "v");
    if (rc != FU_OK) return rc;
    p.v = static_cast<const __nv_bfloat16*>(a->v);
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.v_stride = a->v_stride;
    p.out_stride = a->out_stride;
    p.cu_seqlens = a->cu_seqlens;
    p.prefix_lens = a->prefix_lens;
    p.alibi_slopes = a->alibi_slopes;
    p.status = a->status;
    p.timeout_ns = a->timeout_ns ? a->timeout_ns : FU_DEFAULT_TIMEOUT_NS;
    p.tokens = static_cast<int32_t>(a->tokens);
    p.docs = a->docs;
    p.q_heads = a->q_heads;
    p.group = a->q_heads / a->kv_heads;
    p.causal = a->causal;
    p.row_blocks = static_cast<int32_t>(row_blocks);
    p.block_rows = block_rows;
    p.ends_per_item = static_cast<int32_t>(p.docs / blocks + 1);
    p.ranked = a->cu_seqlens != nullptr && p.row_blocks > 1 && p.row_blocks <= attention::MAX_RANKED;
    p.wide_store = (reinterpret_cast<uintptr_t>(a->out) | a->out_stride * 2) % 32 == 0;
    p.negate = a->scale < 0.f ? 1u : 0u;
    p.scale = std::fabs(a->scale);
    p.softcap = a->softcap;
    // A bias falls with distance.  From the keys before a row towards it the maximum would
    // grow in every tile, and O be rescaled; from the last key on it is found at once.
    // (8192 causal tokens of 8 heads: 154 us the one way and 134 us the other, before the
    // bias moved into the exponent; 123 us with that.)
    p.key_step = a->alibi_slopes != nullptr ? -attention::TILE : attention::TILE;

    DeviceGuard guard(a->device);
    if (!guard.ok()) return set_error(FU_ERR_INVALID, "device %d is not available", a->device);
    cudaError_t e = attention::prepare(a->device);
    if (e == cudaSuccess) {
        const attention::Kernel kernels[4] = {
            attention::attention_kernel<0>, attention::attention_kernel<1>,
            attention::attention_kernel<2>, attention::attention_kernel<3>};
        const int mode = (a->softcap > 0.f ? 1 : 0) | (a->alibi_slopes != nullptr ? 2 : 0);
        Launch launch(dim3(static_cast<unsigned>(blocks)), dim3(attention::NUM_THREADS),
                      attention::SMEM_ALLOC, stream, (flags & FU_FWD_NO_PDL) == 0);
        e = cudaLaunchKernelEx(&launch.cfg, kernels[mode], p);
    }
    if (e != cudaSuccess) return set_error(FU_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    return FU_OK;
}
