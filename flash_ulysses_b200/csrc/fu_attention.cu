// Attention over the exchanged Q/K/V rows (sm_100a): packed documents, causal,
// prefix or full masks, scores capped by a tanh and/or lowered with distance.
//
// A CTA computes one query head's 256 rows as two tiles of 128, and walks the
// keys that any of its rows sees in tiles of 128 with an online softmax:
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
constexpr int ROWS = 2 * TILE;                  // query rows per CTA
constexpr int NUM_THREADS = 384;
constexpr int TILE_BYTES = TILE * D * 2;        // 32 KiB: two 64-column boxes
constexpr int BOX_BYTES = TILE_BYTES / 2;
constexpr int STAGES = 5;                       // K and V tiles in turn
constexpr int OFF_Q = 0;
constexpr int OFF_KV = OFF_Q + 2 * TILE_BYTES;
constexpr int OFF_SEEN = OFF_KV + STAGES * TILE_BYTES;      // int2[2][2]
constexpr int OFF_BAR = OFF_SEEN + 64;
constexpr int OFF_MISC = OFF_BAR + 8 * 32;
constexpr int SMEM_BYTES = OFF_MISC + 64;
constexpr int SMEM_ALLOC = SMEM_BYTES + 1024;   // room to align the base to 1 KiB
static_assert(SMEM_ALLOC <= 232448, "exceeds the 227 KiB per-CTA shared memory limit");
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t TM_S = 0, TM_O = 256;        // + 128 * tile
// Registers: 3 warpgroups launch with 168 each; the softmax takes 216, the
// others keep 72 (216 + 216 + 72 = 3 * 168).
constexpr int SOFTMAX_REGS = 216, OTHER_REGS = 72;
constexpr float LOG2E = 1.4426950408889634f;
// Every so manieth pair of a row's weights is computed on the FMA pipes
// (ex2_poly), the others by the special-function unit, whose 16 results per
// clock and SM take as long as the tile's matrix products.  (Every fourth or
// none took the same time or longer; with a cap the FMA pipes are busy with it.)
constexpr int POLY_EVERY = 8;

// Status "where" codes of this kernel.
enum : int {
    W_CU_SEQLENS = 64, W_Q = 65, W_KV_FULL = 66, W_KV_EMPTY = 67, W_S = 68, W_P = 69, W_O = 70,
    W_CLEAN = 71, W_DRAIN = 72,
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
    uint32_t negate;                   // scale < 0: the MMA negates Q, `scale` is positive
    float scale, softcap;
};

struct Bars {
    uint32_t q, kv_full, kv_empty, s, p, o, done, clean;
    __device__ explicit Bars(uint32_t base)
        : q(base), kv_full(base + 8), kv_empty(kv_full + 8 * STAGES), s(kv_empty + 8 * STAGES),
          p(s + 16), o(p + 32), done(o + 16), clean(done + 8) {}
};

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

// What every role needs to know of the CTA's work.  Key tile j is rows
// kv0 + 128 j on; query tile t takes part in the key tiles [first[t], last[t]).
struct Work {
    int row0, head, kv0, tiles, first[2], last[2];
    int clear0, clear1;                // key tiles that every valid row sees all of
    // Whether some row does not see some key of tile j.
    __device__ bool edge(int j) const { return j < clear0 || j >= clear1; }
};

// `seen[t]` holds the ranges of tile t's first and last row that belongs to a
// document; `valid` rows of the CTA do.
__device__ __forceinline__ Work make_work(const int2 (*seen)[2], int row0, int head, int valid) {
    Work w;
    w.row0 = row0;
    w.head = head;
    w.kv0 = seen[0][0].x;
    w.clear0 = (max(seen[valid > TILE][1].x - w.kv0, 0) + TILE - 1) / TILE;
    w.clear1 = max(seen[0][0].y - w.kv0, 0) / TILE;
    w.tiles = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        w.first[t] = w.last[t] = 0;
        if (valid > t * TILE) {
            w.first[t] = max(seen[t][0].x - w.kv0, 0) / TILE;
            w.last[t] = max((seen[t][1].y - w.kv0 + TILE - 1) / TILE, w.first[t]);
        }
        w.tiles = max(w.tiles, w.last[t]);
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

__device__ __forceinline__ uint32_t pack_bf16x2_rn(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// ------------------------------------------------------------ loads
// Ring order: K_0, V_0, K_1, V_1, ...
__device__ void run_loads(const Params& p, const Work& w, uint8_t* smem, const Bars& b,
                          volatile int* abort_flag) {
    const uint32_t q = smem_u32(smem + OFF_Q), ring = smem_u32(smem + OFF_KV);
    const int q_col = w.head * D, kv_col = w.head / p.group * D;
    mbar_arrive_expect_tx(b.q, 2 * TILE_BYTES);
    for (int t = 0; t < 2; ++t)
        for (int c = 0; c < 2; ++c)
            tma_load_2d(q + t * TILE_BYTES + c * BOX_BYTES, &p.tm_q, b.q, q_col + 64 * c,
                        w.row0 + t * TILE);
    int i = 0;
    for (; i < 2 * w.tiles; ++i) {
        const int s = i % STAGES, use = i / STAGES;
        if (!fu_wait_parity(b.kv_empty + 8 * s, (use & 1) ^ 1, abort_flag, p.timeout_ns, p.status,
                            W_KV_EMPTY))
            break;
        mbar_arrive_expect_tx(b.kv_full + 8 * s, TILE_BYTES);
        for (int c = 0; c < 2; ++c)
            tma_load_2d(ring + s * TILE_BYTES + c * BOX_BYTES, i & 1 ? &p.tm_v : &p.tm_k,
                        b.kv_full + 8 * s, kv_col + 64 * c, w.kv0 + (i >> 1) * TILE);
    }
    // What was issued must land before shared memory is released, whatever the
    // other roles did.
    drain_wait(b.q, 0, p.timeout_ns, p.status);
    for (int k = i > STAGES ? i - STAGES : 0; k < i; ++k)
        drain_wait(b.kv_full + 8 * (k % STAGES), (k / STAGES) & 1, p.timeout_ns, p.status);
}

// ------------------------------------------------------------ MMA
__device__ void run_mma(const Params& p, const Work& w, uint8_t* smem, uint32_t tmem, const Bars& b,
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
    const int first0 = same(w.first[0]), first1 = same(w.first[1]);
    const int last0 = same(w.last[0]), last1 = same(w.last[1]);
    const int tiles = same(w.tiles), clear0 = same(w.clear0), clear1 = same(w.clear1);
    tmem = same(tmem);
    uint32_t p_phase0 = 0, p_phase1 = 0;
    // Ring stages and phases of V_j and K_(j+1), and the count of V_j.
    int sv = STAGES - 1, sk = 0, sc = STAGES - 1;
    uint32_t v_phase = 1, k_phase = 0, c_phase = 1;
    const auto v_arrived = [&](int j) {
        if (j < 0 || j >= tiles) return true;
        const bool edge = j < clear0 || j >= clear1;
        return wait(edge ? b.clean + 8 * sc : b.kv_full + 8 * sv, edge ? c_phase : v_phase,
                    edge ? W_CLEAN : W_KV_FULL);
    };
    bool ok = wait(b.q, 0, W_Q);
    // Step j: the products P V of key tile j, each followed by the same query
    // tile's scores of key tile j + 1.
#pragma unroll 1
    for (int j = -1; ok && j < tiles; ++j) {
        const uint32_t v_lo = desc_lo(ring + sv * TILE_BYTES, BOX_BYTES);   // 64-column boxes
        const uint32_t k_lo = desc_lo(ring + sk * TILE_BYTES, 16);
        const uint32_t v_empty = b.kv_empty + 8 * sv, k_empty = b.kv_empty + 8 * sk;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int first = t ? first1 : first0, last = t ? last1 : last0;
            uint32_t& p_phase = t ? p_phase1 : p_phase0;
            if (t == 1) {
                // The next step's V is looked for while the first query tile's
                // products run; K, which comes later, just before it is needed.
                sv = sv + 2 < STAGES ? sv + 2 : (v_phase ^= 1, sv + 2 - STAGES);
                sc = sc + 1 < STAGES ? sc + 1 : (c_phase ^= 1, 0);
                if (!(ok = v_arrived(j + 1))) break;
            }
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
            if (t == 0 && j + 1 < tiles && !(ok = wait(b.kv_full + 8 * sk, k_phase, W_KV_FULL)))
                break;
            if (j + 1 >= first && j + 1 < last) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t at = ((k / 4) * BOX_BYTES + (k % 4) * 32) >> 4;
                    mma_ss(one, tmem + TM_S + t * TILE, q_lo + t * (TILE_BYTES >> 4) + at,
                           k_lo + at, idesc_s, k > 0);
                }
                commit(one, b.s + 8 * t);
            }
            if (t == 1 && j + 1 < tiles) commit(one, k_empty);
        }
        sk = sk + 2 < STAGES ? sk + 2 : (k_phase ^= 1, sk + 2 - STAGES);
    }
    // Every MMA this warp issued must finish before TMEM is released.
    commit(one, b.done);
    drain_wait(b.done, 0, p.timeout_ns, p.status);
}

// ------------------------------------------------------------ V at a mask's edge
// Every V tile is counted (on a ring of barriers of its own), so that neither
// side gets more than the ring ahead; only those at an edge are looked at.
__device__ void run_clean(const Params& p, const Work& w, uint8_t* smem, const Bars& b,
                          volatile int* abort_flag, volatile int* found) {
    const int me = threadIdx.x & 63;
    for (int j = 0; j < w.tiles; ++j) {
        const int i = 2 * j + 1, s = i % STAGES;
        if (!fu_wait_parity(b.kv_full + 8 * s, (i / STAGES) & 1, abort_flag, p.timeout_ns, p.status,
                            W_KV_FULL))
            return;
        uint4* v = reinterpret_cast<uint4*>(smem + OFF_KV + s * TILE_BYTES);
        bool wrote = false;
#pragma unroll 8
        for (int o = me; o < (w.edge(j) ? TILE_BYTES / 16 : 0); o += 64) {
            uint4 x = v[o];
            uint32_t* word = &x.x;
            bool odd = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // A BF16 is not finite if its exponent bits are all set.
                const uint32_t bad = __vcmpeq2(word[k] & 0x7f807f80u, 0x7f807f80u);
                word[k] &= ~bad;
                odd = odd || bad != 0;
            }
            if (odd) {
                v[o] = x;
                wrote = true;
            }
        }
        if (wrote) {
            *found = 1;
            fence_proxy_async_smem();
        }
        __syncwarp();
        if ((me & 31) == 0) mbar_arrive(b.clean + 8 * (j % STAGES));
    }
}

// ------------------------------------------------------------ softmax
// kMode: 1 scores capped by a tanh, 2 lowered with distance (3 both).
template <int kMode>
__device__ void run_softmax(const Params& p, const Work& w, uint8_t* smem, uint32_t tmem,
                            const Bars& b, int t, int2 seen, bool valid,
                            volatile int* abort_flag, volatile int* found) {
    const int first = t ? w.first[1] : w.first[0], last = t ? w.last[1] : w.last[0];
    const int lane = threadIdx.x & 31;
    const int warp = (threadIdx.x >> 5) & 3;              // of this tile
    const int row = w.row0 + t * TILE + warp * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t tm_s = tmem + TM_S + t * TILE + lanes, tm_o = tmem + TM_O + t * TILE + lanes;
    // Scores in units of log2: x = c * s here, m in the units of s (so c m is
    // its logarithm), or with a cap or a bias x = s, c = 1.
    const float c = kMode ? 1.f : fmaxf(p.scale * LOG2E, 1e-30f);
    const float slope =
        kMode & 2 ? __ldg(p.alibi_slopes + w.head) * LOG2E : 0.f;
    const float lin = p.scale * LOG2E;
    const float to_cap = kMode & 1 ? p.scale / p.softcap : 0.f;
    // A row without a document is computed like one that sees everything, and
    // not stored.
    const int lo = valid ? seen.x : INT_MIN / 2, hi = valid ? seen.y : INT_MAX / 2;

    float m = -INFINITY, l = 0.f;
    uint32_t phase = 0;
    bool ok = true;
    for (int j = first; j < last; ++j) {
        ok = fu_wait_parity(b.s + 8 * t, phase, abort_flag, p.timeout_ns, p.status, W_S);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        phase ^= 1;
        tc_fence_after();
        uint32_t r[TILE];
        float* s = reinterpret_cast<float*>(r);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            tmem_ld_32cols(tm_s + 32 * k, *reinterpret_cast<uint32_t(*)[32]>(r + 32 * k));
        tmem_ld_wait();
        const int k0 = w.kv0 + j * TILE;
        if (kMode & 1) {
            // cap tanh(z), z = scale s / cap.  Where all of the warp's |z| are at
            // most 1 (scores below the cap, the ordinary case) by an odd polynomial
            // of degree 11, off by 7e-7; else as cap (1 - 2 / (1 + 2^(2 log2(e) z))),
            // off by 2^-22: absolute errors in both, which is what a score needs.
            // The second takes three special-function results per score with the
            // weight's, 4.5 us per tile against 1.1 us without a cap.
            float far = 0.f;
#pragma unroll
            for (int k = 0; k < TILE; k += 2) far = max3(far, fabsf(s[k]), fabsf(s[k + 1]));
            if (__any_sync(0xffffffffu, !(far * to_cap <= 1.f))) {
                const float in = 2.f * LOG2E * to_cap, out = p.softcap * LOG2E;
#pragma unroll
                for (int k = 0; k < TILE; ++k)
                    s[k] = fmaf(-2.f * out, __fdividef(1.f, 1.f + ex2(s[k] * in)), out);
            } else {
#pragma unroll
                for (int k = 0; k < TILE; k += 2) {
                    const f32x2 x = pair(s[k], s[k + 1]);
                    const f32x2 z = mul2(x, pair(to_cap)), u = mul2(z, z);
                    f32x2 h = fma2(u, pair(-0.0030804092530161142f), pair(0.016842123121023178f));
                    h = fma2(h, u, pair(-0.051767539232969284f));
                    h = fma2(h, u, pair(0.1329089254140854f));
                    h = fma2(h, u, pair(-0.3333089351654053f));
                    h = fma2(h, u, pair(1.f));
                    const float2 y = both(mul2(mul2(x, pair(lin)), h));
                    s[k] = y.x;
                    s[k + 1] = y.y;
                }
            }
        }
        if (kMode & 2) {
            const f32x2 scale2 = pair(kMode & 1 ? 1.f : lin);
            // Without keys behind the row (or with only such) |i - j| is linear in
            // j; keys that a causal mask hides may come out as they like.
            const bool below = (p.causal && p.prefix_lens == nullptr) || k0 + TILE - 1 <= row - lane;
            const bool above = k0 >= row - lane + 31;
            if (below || above) {
                const float step = below ? slope : -slope;
#pragma unroll
                for (int k = 0; k < TILE; k += 32) {
                    const float start = static_cast<float>(k0 + k - row) * step;
                    f32x2 bias = pair(start, start + step);
#pragma unroll
                    for (int q = k; q < k + 32; q += 2) {
                        const float2 y = both(fma2(pair(s[q], s[q + 1]), scale2, bias));
                        s[q] = y.x;
                        s[q + 1] = y.y;
                        bias = add2(bias, pair(2.f * step));
                    }
                }
            } else {
                const float at = static_cast<float>(row - k0);
#pragma unroll
                for (int k = 0; k < TILE; ++k)
                    s[k] = fmaf(-slope, fabsf(at - static_cast<float>(k)),
                                kMode & 1 ? s[k] : s[k] * lin);
            }
        }
        const int from = lo - k0, to = hi - k0;
        if (__any_sync(0xffffffffu, from > 0 || to < TILE)) {
#pragma unroll
            for (int k = 0; k < TILE; ++k)
                s[k] = k >= from && k < to ? s[k] : -INFINITY;
        }
        float best[4] = {m, s[0], s[1], s[2]};
#pragma unroll
        for (int k = 3; k + 1 < TILE; k += 2)
            best[(k >> 1) & 3] = max3(best[(k >> 1) & 3], s[k], s[k + 1]);
        const float top = fmaxf(max3(best[0], best[1], best[2]), fmaxf(best[3], s[TILE - 1]));
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
        const f32x2 base = pair(m == -INFINITY ? 0.f : -m * c), c2 = pair(c);
        f32x2 sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t packed[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const f32x2 x = pair(s[32 * k + 2 * q], s[32 * k + 2 * q + 1]);
                f32x2 y = kMode ? add2(x, base) : fma2(x, c2, base);
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
    if (first == last || !ok) return;

    // out = O / l, through this tile's Q rows in shared memory (no longer
    // needed): a thread writes its row, then the warp's 32 rows leave as whole
    // 256-byte rows.
    ok = fu_wait_parity(b.o + 8 * t, 0, abort_flag, p.timeout_ns, p.status, W_O);
    if (!__all_sync(0xffffffffu, ok)) return;
    tc_fence_after();
    const float inv = 1.f / l;
    const bool poison = *found != 0;
    uint8_t* stage = smem + OFF_Q + t * TILE_BYTES + warp * 32 * 256;
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
                const int a = max(lo, w.kv0 + j * TILE), e = min(hi, w.kv0 + (j + 1) * TILE);
                for (int key = a; key < e; ++key) {
                    const __nv_bfloat16* v = p.v + key * p.v_stride + w.head / p.group * D + 32 * k;
#pragma unroll
                    for (int q = 0; q < 32; ++q) {
                        const float x = __bfloat162float(v[q]);
                        if (!isfinite(x)) o[q] = __float_as_uint(__uint_as_float(o[q]) + x);
                    }
                }
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int chunk = 4 * k + q;
            const uint32_t* x = o + 8 * q;
            *reinterpret_cast<uint4*>(stage + lane * 256 + ((chunk ^ (lane & 7)) << 4)) = make_uint4(
                pack_bf16x2_rn(__uint_as_float(x[0]), __uint_as_float(x[1])),
                pack_bf16x2_rn(__uint_as_float(x[2]), __uint_as_float(x[3])),
                pack_bf16x2_rn(__uint_as_float(x[4]), __uint_as_float(x[5])),
                pack_bf16x2_rn(__uint_as_float(x[6]), __uint_as_float(x[7])));
        }
    }
    const uint32_t stored = __ballot_sync(0xffffffffu, valid);
    __syncwarp();
    __nv_bfloat16* dst = p.out + static_cast<int64_t>(row - lane) * p.out_stride + w.head * D;
#pragma unroll 4
    for (int r = lane >> 4; r < 32; r += 2) {
        const int chunk = lane & 15;
        if (stored >> r & 1)
            *reinterpret_cast<uint4*>(dst + r * p.out_stride + 8 * chunk) =
                *reinterpret_cast<const uint4*>(stage + r * 256 + ((chunk ^ (r & 7)) << 4));
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
    int2 (*seen)[2] = reinterpret_cast<int2 (*)[2]>(smem + OFF_SEEN);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + OFF_MISC);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + OFF_MISC + 4);
    volatile int* found = reinterpret_cast<volatile int*>(smem + OFF_MISC + 8);

    // Prologue: shared memory, TMEM and parameters only (it may overlap the
    // previous kernel of the stream under a programmatic dependent launch).
    if (threadIdx.x == 0) {
        mbar_init(b.q, 1);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(b.kv_full + 8 * s, 1);
            mbar_init(b.kv_empty + 8 * s, 1);
            mbar_init(b.clean + 8 * s, 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(b.s + 8 * t, 1);
            mbar_init(b.p + 16 * t, 4);
            mbar_init(b.p + 16 * t + 8, 4);
            mbar_init(b.o + 8 * t, 1);
        }
        mbar_init(b.done, 1);
        *abort_flag = 0;
        *found = 0;
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

    // The longest rows first: with a causal mask the last CTAs to start then
    // have the least to do.
    const int head = blockIdx.x % p.q_heads;
    const int row0 = (gridDim.x / p.q_heads - 1 - blockIdx.x / p.q_heads) * ROWS;
    if (blockIdx.x == 0 && p.cu_seqlens != nullptr) {
        for (int d = threadIdx.x; d <= p.docs; d += NUM_THREADS) {
            const int x = __ldg(p.cu_seqlens + d);
            const int before = d > 0 ? __ldg(p.cu_seqlens + d - 1) : 0;
            if (x < before || x > p.tokens || (d == 0 && x != 0))
                report_status(p.status, FU_DEV_LENGTHS, W_CU_SEQLENS);
        }
    }
    int rows = p.tokens;                               // rows of documents
    if (p.cu_seqlens != nullptr) rows = min(max(__ldg(p.cu_seqlens + p.docs), 0), p.tokens);
    const int valid = min(rows - row0, ROWS);
    int2 mine = make_int2(0, 0);
    if (warp < 8) {
        const int i = threadIdx.x, t = i / TILE;
        if (row0 + i < p.tokens) mine = seen_rows(p, row0 + i);
        if (i == t * TILE) seen[t][0] = mine;
        if (i == min(valid, (t + 1) * TILE) - 1) seen[t][1] = mine;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    if (valid > 0) {
        const Work w = make_work(seen, row0, head, valid);
        if (warp < 8) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
            run_softmax<kMode>(p, w, smem, tmem, b, warp >> 2, mine, mine.x < mine.y, abort_flag,
                               found);
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
            if (warp == 8) {
                if ((threadIdx.x & 31) == 0) run_loads(p, w, smem, b, abort_flag);
            } else if (warp == 9) {
                run_mma(p, w, smem, tmem, b, abort_flag);
            } else {
                run_clean(p, w, smem, b, abort_flag, found);
            }
            __syncwarp();
        }
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

// Raises the kernels' shared-memory limit once per device.
static cudaError_t prepare(int device) {
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = 1ull << (device & 63);
    if (device < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    for (Kernel k : {attention_kernel<0>, attention_kernel<1>, attention_kernel<2>,
                     attention_kernel<3>}) {
        cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             SMEM_ALLOC);
        if (e != cudaSuccess) return e;
    }
    if (device < 64) done.fetch_or(bit, std::memory_order_release);
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

    const int64_t blocks = (a->tokens + attention::ROWS - 1) / attention::ROWS * a->q_heads;
    if (blocks > INT32_MAX)
        return set_error(FU_ERR_INVALID, "tokens * q_heads is too large for one call");

    attention::Params p = {};
    int rc = attention::encode_rows(&p.tm_q, a->q, a->tokens, a->q_heads * attention::D,
                                    a->q_stride, "q");
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
    p.negate = a->scale < 0.f ? 1u : 0u;
    p.scale = std::fabs(a->scale);
    p.softcap = a->softcap;

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
