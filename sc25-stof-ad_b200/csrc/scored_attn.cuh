// Attention whose scores are changed by a formula (tanh cap, distance bias) and masked by rules (causal, window, prefix, documents,
// padding), for sm_100a: TMA-fed tcgen05 products with the accumulators in tensor memory, online softmax in registers.
//
// Per thread block one stretch of 128 query rows, or two (HALVES) that share every K/V tile of 128 keys.  Each half has its own S
// (128 x 128 fp32 in tensor memory), P (16-bit numbers, also in tensor memory) and O (128 x D fp32), its own softmax warps - one row a
// thread - and its own list of tiles: those that the rules leave anything of.  While one half's warps work on their scores the tensor
// core serves the other half.
//   warps 0..3 (and 4..7)   softmax of the half
//   next warp               TMA producer: Q, then K and V tiles through rings of slots (scored_slots)
//   last warp               tcgen05 issuer
// Where tensor memory has room (OWN_P: D = 64) P lies beside S, and S = Q K^T of the next tile is issued as soon as S has been read into
// registers; else P lies over S and the next product waits for O += P V.  P is handed over in two parts.
// A tile is classified per warp (32 rows): nothing to mask, or masked by 128 bits a row.
// What a call does not use is not in its kernel's loop (WHAT): the loop a warp spends its time in has to fit the instruction caches.
//
// What bounds it: long sequences the hand-overs between tensor core and softmax warps.  A tile of 2 x 128 rows costs the tensor core 2048
// cycles (D = 128: 16.8 MFLOP at 8192 a cycle; heads of 64 half of that) and the exponentials 2048 too (16 a cycle on an SM), side by side;
// with the loads from tensor memory, the maxima and the packing a warp comes to about 3300 between two tiles of its own: 8192 x 8192, 32
// heads on 8 of 128: 860 us = 1278 TFLOP/s, causal 462 (bf16 447), causal with cap 529 to 540; heads of 64, which the exponentials bound:
// 729 us = 754 TFLOP/s, causal 379, with slopes 525, dense with a table 840 (all of them 1 to 3 % more in long runs; the cap with a prefix
// in a run of seconds 608, at the power cap).  Short ones a block's beginning and end (the chain
// launch - Q, K - S - softmax - O - store, 4 to 6 us, half of it hidden by the other block on the SM).  Measured and slower: a persistent grid
// (1.8 us less per block, more per tile: 4 x 12 x 1120 with documents 35 us against 29, 2 x 32 x 2048 queries with a window 145 against
// 138); part of the exponentials as polynomials (plain 3 % faster, with a cap slower, and a NaN is lost); eight chains of maxima;
// the second half of a row on its way while the first is looked at (dense 893).
#pragma once

#include "cache_common.cuh"
#include "stof_host.h"
#include "stof_ptx.cuh"

namespace stof {

constexpr int SA_T = 128;                    // rows of a half, keys of a tile
constexpr int SA_PAD = 160;                  // the distance table in shared memory goes on for so long on both sides: a tile that meets the table needs no clamp
constexpr float SA_RESCALE = 8.0f;           // log2 units by which a row's maximum may outgrow the reference of its P (P <= 2^8)
constexpr long long SA_DRAIN_CYCLES = 1 << 17;
constexpr float SA_LOG2E = 1.4426950408889634f;
enum { SA_PLAIN = 0, SA_CAP = 1, SA_ANY = 2, SA_DOCS = 4 };   // what is done to scores: nothing, the cap alone, whatever the call asks for; and documents

struct ScoredParams {
    const float *slopes, *distance_bias;
    const int *documents, *prefix_lens, *key_lens;
    long long documents_stride;
    int* status;
    float scale, softcap;
    int causal, window, radius;
    int batch, heads, group, q_len, k_len, q_tiles;
    int slot_s[4], slot_h[4], slot_b[4];     // of q, k, v, out: which coordinate of the tensor map is the row, the head, the batch
    int table_bytes, range_bytes;
};

// barriers, two of each (a half's, or a slot's): Q is there; S is there; parts 0 and 1 of P are there; S has been read; O is complete up
// to the last P; slots
enum { SB_Q = 0, SB_S = 2, SB_P0 = 4, SB_P1 = 6, SB_READ = 8, SB_O = 10, SB_FIX = 12, SB_K_FULL = 13, SB_K_EMPTY = 15, SB_V_FULL = 17, SB_V_EMPTY = 19, SB_COUNT = 21 };

static __device__ __forceinline__ void load_tile(unsigned char* dst, const CUtensorMap* map, uint64_t* bar, int col, int row, int head, int batch, int slot_s, int slot_h) {
    // the three outer coordinates are in the order of their strides
    const int c1 = slot_s == 1 ? row : slot_h == 1 ? head : batch;
    const int c2 = slot_s == 2 ? row : slot_h == 2 ? head : batch;
    const int c3 = slot_s == 3 ? row : slot_h == 3 ? head : batch;
    tma_load_4d(dst, map, bar, col, c1, c2, c3);
}

static __device__ __forceinline__ void store_rows(const CUtensorMap* map, const unsigned char* src, int col, int row, int head, int batch, int slot_s, int slot_h) {
    const int c1 = slot_s == 1 ? row : slot_h == 1 ? head : batch;
    const int c2 = slot_s == 2 ? row : slot_h == 2 ? head : batch;
    const int c3 = slot_s == 3 ? row : slot_h == 3 ? head : batch;
    tma_store_4d(map, src, col, c1, c2, c3);
}

static __device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
static __device__ __forceinline__ float min3f(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// from_u * tanh(s * to_u) near zero: an odd polynomial of s, the factors in its coefficients.  Relative errors of the fits (weighted least
// squares moved towards the minimax one): 2.9e-6 of three terms up to |u| = 0.35, 7e-6 of five up to 1; a score of 40 is then off by
// 3e-4 at most, less than P's rounding to fp16 makes of it.
struct NearTanh {
    float near[3], far[5];                   // of s, s^3, s^5, ..
    float near_end, far_end;                 // up to which |s| they are used: -1, not even for 0, where a coefficient leaves fp32's range
    __device__ __forceinline__ NearTanh() : near{}, far{}, near_end(-1.f), far_end(-1.f) {}
    __device__ __forceinline__ NearTanh(float to_u, float from_u) {
        const float w = to_u * to_u, a = to_u * from_u;
        // Where a coefficient is below fp32's normal numbers the polynomial ends where the term is below 1e-7 of the sum, and where the
        // smallest number that stands for the last one (below) makes 1e-7 of it
        const float u_end = a * w * w > 1e-36f ? 0.35f : a * w > 1e-36f ? 0.03f : 5e-4f;
        near_end = to_u > 1e-37f && a * w * w < 1e37f ? u_end / to_u : -1.f;
        if (u_end < 0.35f) near_end = fminf(near_end, sqrtf(sqrtf(fminf(a, 1.f) * 7e37f)));
        far_end = a * w * w * w * w > 1e-34f && a * w * w * w * w < 1e37f ? 1.f / to_u : -1.f;
        near[0] = a * 0.9999971389770508f;
        near[1] = a * w * -0.33290955424308777f;
        near[2] = a * w * w * 0.1239503026008606f;
        far[0] = a * 0.999993085861206f;
        far[1] = a * w * -0.3329806625843048f;
        far[2] = a * w * w * 0.13036811351776123f;
        far[3] = a * w * w * w * -0.044817544519901276f;
        far[4] = a * w * w * w * w * 0.009036419913172722f;
        // (never 0: minus infinity, a masked score, stays what it is)
        near[2] = fmaxf(near[2], 1e-45f);
        far[4] = fmaxf(far[4], 1e-45f);
    }
};
template <int N>
static __device__ __forceinline__ float2 odd_polynomial(float2 s, const float (&c)[N]) {
    const float2 w = mul2(s, s);
    float2 q = pk2(c[N - 1], c[N - 1]);
#pragma unroll
    for (int i = N - 2; i >= 0; --i) q = fma2(q, w, pk2(c[i], c[i]));
    return mul2(q, s);
}
template <int N>
static __device__ __forceinline__ float2 odd_polynomial_plus(float2 s, const float (&c)[N], float2 added) {
    const float2 w = mul2(s, s);
    float2 q = pk2(c[N - 1], c[N - 1]);
#pragma unroll
    for (int i = N - 2; i >= 0; --i) q = fma2(q, w, pk2(c[i], c[i]));
    return fma2(q, s, added);
}

// The bounded wait without a call of a function (which does not go with moved registers)
static __device__ __forceinline__ void wait_inline(uint32_t bar, uint32_t parity, const WaitCtx& ctx, int barrier_id) {
    if (__builtin_expect(mbar_test_wait_addr(bar, parity), 1)) return;
    const long long t0 = clock64();
#pragma unroll 1
    while (!mbar_try_wait_addr(bar, parity)) {
        if (*ctx.abort_smem) return;
        if (clock64() - t0 > WAIT_BUDGET_CYCLES) {
            *ctx.abort_smem = 1;
            if (ctx.status_gmem) atomicCAS(ctx.status_gmem, 0, (barrier_id << 8) | STATUS_WAIT_TIMEOUT);
            return;
        }
    }
}

// tanh of a whole row's scores in tensor memory that are not near enough to zero for a polynomial: s = from_u * tanh(s * scale * to_u), in place (one after
// the other: together they may be no normal number)
static __device__ __forceinline__ void cap_in_tmem(uint32_t t_s, float scale, float to_u, float from_u) {
#pragma unroll 1
    for (int c = 0; c < SA_T; c += 16) {
        uint32_t s[16];
        tmem_ld16(t_s + c, s);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __float_as_uint(tanh_any(__uint_as_float(s[i]) * scale * to_u) * from_u);
        tmem_st16(t_s + c, s);
    }
    tc_wait_st();
}

// Bits of the 128 keys of a tile that a row sees: those in [from, to] or in front of `front`, and in front of `end` (all relative to the tile).
static __device__ __forceinline__ uint4 visible_keys(int from, int to, int front, int end) {
    // bits lo .. hi of word w
    auto bits = [](int lo, int hi, int w) -> uint32_t {
        lo -= 32 * w;
        hi -= 32 * w;
        if (hi < 0 || lo > 31 || hi < lo) return 0u;
        const uint32_t upto = hi >= 31 ? 0xFFFFFFFFu : (2u << hi) - 1u;
        return lo <= 0 ? upto : upto & (0xFFFFFFFFu << lo);
    };
    uint32_t r[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) r[w] = (bits(from, to, w) | bits(0, front - 1, w)) & bits(0, end - 1, w);
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// COUNT K = 16 products in one instruction sequence: the issuing thread is one lane, and every instruction that it spends between two
// products delays all of them.  `a` and `b` advance by 32 bytes (2 in descriptor units) a product, by a panel after four.
template <int COUNT>
static __device__ __forceinline__ void mma_chain_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    static_assert(COUNT == 4 || COUNT == 8, "64 or 128 of K");
#define SA_MMA(off, p) "add.s64 a, %1, " #off ";\n\tadd.s64 b, %2, " #off ";\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, " #p ";\n\t"
    if constexpr (COUNT == 4)
        asm volatile("{\n\t.reg .pred p0, p1;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p0, 0, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\t"
                     SA_MMA(0, p0) SA_MMA(2, p1) SA_MMA(4, p1) SA_MMA(6, p1) "}" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
    else
        asm volatile("{\n\t.reg .pred p0, p1;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p0, 0, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\t"
                     SA_MMA(0, p0) SA_MMA(2, p1) SA_MMA(4, p1) SA_MMA(6, p1) SA_MMA(1024, p1) SA_MMA(1026, p1) SA_MMA(1028, p1) SA_MMA(1030, p1)
                     "}" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
#undef SA_MMA
}
// Four K = 16 products with A in tensor memory (8 columns each) and B key-row-major (16 rows of 128 bytes each); the first one
// overwrites the accumulator where `accumulate` is 0
static __device__ __forceinline__ void mma_chain_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p0, p1;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\t"
        "setp.ne.b32 p0, %4, 0;\n\t"
        "setp.eq.b32 p1, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p0;\n\t"
        "add.u32 a, %1, 8;\n\tadd.s64 b, %2, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, p1;\n\t"
        "add.u32 a, %1, 16;\n\tadd.s64 b, %2, 256;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, p1;\n\t"
        "add.u32 a, %1, 24;\n\tadd.s64 b, %2, 384;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, p1;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <int D>
static __device__ __forceinline__ void rescale_o(uint32_t t_o, float alpha) {
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
        uint32_t o[16];
        tmem_ld16(t_o + c, o);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
        tmem_st16(t_o + c, o);
    }
    tc_wait_st();
}

// Registers are moved to the softmax warps from the others (setmaxnreg, which is a whole warpgroup's: two of the others' four warps are
// idle).  Two halves: 384 x 168 at the launch, 256 x R + 128 x r afterwards.  One half, two blocks on an SM: 256 x 128, then 128 x R + 128 x r.
constexpr int SA_R2 = 224, SA_R1 = 208;      // (216 and 232, 200 and 216: up to 3 % slower)
constexpr int scored_threads(int halves) { return halves == 2 ? 384 : 256; }
constexpr int scored_per_sm(int halves) { return halves == 1 ? 2 : 1; }
constexpr int scored_slots(int dim, int halves) { return dim == 128 && halves == 1 ? 1 : 2; }       // as many as shared memory holds
constexpr int scored_regs_softmax(int halves) { return halves == 2 ? SA_R2 : SA_R1; }
constexpr int scored_regs_other(int halves) { return halves == 2 ? (384 * 168 - 256 * SA_R2) / 128 : (256 * 128 - 128 * SA_R1) / 128; }
static_assert(256 * SA_R2 + 128 * scored_regs_other(2) <= 384 * 168 && 128 * SA_R1 + 128 * scored_regs_other(1) <= 256 * 128 && SA_R1 % 8 == 0 && SA_R2 % 8 == 0 &&
                  scored_regs_other(1) % 8 == 0 && scored_regs_other(2) % 8 == 0, "more registers than the block was launched with would be waited for forever");

// What a stretch of rows sees: tiles [lo, hi) and [0, prefix), where documents agree
struct Reach {
    int lo, hi, prefix, doc_min, doc_max;
};

template <int D, int HALVES, bool BF16, int WHAT>
__global__ void __launch_bounds__(scored_threads(HALVES), scored_per_sm(HALVES)) scored_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o,
                                                                        const ScoredParams p) {
    constexpr int MODE = WHAT & 3;
    constexpr bool DOCS = (WHAT & SA_DOCS) != 0;
    constexpr int PANELS = D / 64;                           // 64-column panels of a tile, 128 rows of 128 swizzled bytes each
    constexpr int PANEL_BYTES = SA_T * 128, TILE_BYTES = PANELS * PANEL_BYTES;
    constexpr int W_LOAD = HALVES * 4, W_MMA = W_LOAD + 1;
    constexpr bool OWN_P = scored_per_sm(HALVES) * HALVES * (SA_T + SA_T / 2 + D) <= 512;
    constexpr unsigned SLOTS = scored_slots(D, HALVES);     // of K, and of V
    constexpr int COL_O = HALVES * SA_T, COL_P = OWN_P ? COL_O + HALVES * D : 0, P_STEP = OWN_P ? SA_T / 2 : SA_T;
    constexpr int TMEM_COLS = (OWN_P ? COL_P + HALVES * SA_T / 2 : COL_O + HALVES * D) > 256 ? 512 : 256;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* q_smem = smem;
    unsigned char* ring = q_smem + HALVES * TILE_BYTES;
    float* table = reinterpret_cast<float*>(ring + 2 * SLOTS * TILE_BYTES);
    int2* range = reinterpret_cast<int2*>(reinterpret_cast<unsigned char*>(table) + p.table_bytes);
    __shared__ __align__(8) uint64_t bars[SB_COUNT];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ int2 row_docs[HALVES * 4];                    // smallest and largest document of each softmax warp's rows

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &abort_word;
    const WaitCtx wctx{abort_flag, p.status};
    const bool loader = warp == W_LOAD && lane == 0;
    if (loader) {
        tma_prefetch_desc(&map_q);
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
        tma_prefetch_desc(&map_o);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars[SB_Q + i], 1);
            mbar_init(&bars[SB_S + i], 1);
            mbar_init(&bars[SB_P0 + i], 4);
            mbar_init(&bars[SB_P1 + i], 4);
            mbar_init(&bars[SB_READ + i], 4);
            mbar_init(&bars[SB_O + i], 1);
        }
        mbar_init(&bars[SB_FIX], 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars[SB_K_FULL + i], 1);
            mbar_init(&bars[SB_K_EMPTY + i], 1);
            mbar_init(&bars[SB_V_FULL + i], 1);
            mbar_init(&bars[SB_V_EMPTY + i], 1);
        }
        fence_mbar_init();
    }
    if (warp == W_MMA) {
        tmem_alloc(&tmem_slot, TMEM_COLS);
        tmem_relinquish();
    }
    grid_dependency_wait();
    grid_launch_dependents();

    // the heaviest stretches first: with a causal mask those at the end of the sequence
    const int heads_all = p.batch * p.heads;
    const int row_tile = p.q_tiles - 1 - static_cast<int>(blockIdx.x / heads_all), bh = static_cast<int>(blockIdx.x % heads_all);
    const int b = bh / p.heads, head = bh % p.heads, kv = head / p.group;
    const int q0 = row_tile * (SA_T * HALVES), shift = p.k_len - p.q_len;
    const int* docs = DOCS ? p.documents + b * p.documents_stride : nullptr;
    // what a block waits for before its first tile are loads of a word or a few, so all are asked for before any is used
    const int key_len = p.key_lens != nullptr ? __ldca(p.key_lens + b) : p.k_len, prefix_len = p.prefix_lens != nullptr ? __ldca(p.prefix_lens + b) : 0;
    const bool muted = loader && failure_reported(p.status);
    const int my_row = q0 + static_cast<int>(threadIdx.x);
    int my_doc = 0;
    if (DOCS && warp < HALVES * 4) my_doc = __ldca(docs + min(my_row, p.q_len - 1) + shift);
    // (the loading warp has Q and K to see to)
    const int helper = static_cast<int>(threadIdx.x) - (warp > W_LOAD ? 32 : 0), helpers = scored_threads(HALVES) - 32;
    if (p.distance_bias != nullptr && warp != W_LOAD) {
        const float* src = p.distance_bias + static_cast<size_t>(head) * (2 * p.radius + 1);
        const int count = 2 * p.radius + 1 + 2 * SA_PAD;
        for (int i0 = helper; i0 < count; i0 += 4 * helpers) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __ldca(src + min(max(i0 + j * helpers - SA_PAD, 0), 2 * p.radius));
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i0 + j * helpers < count) table[i0 + j * helpers] = v[j] == -INFINITY ? v[j] : finite_or_nan(v[j] * SA_LOG2E);
        }
    }
    // the documents of the tiles that the rules may want, whatever the lengths are
    constexpr int DOC_WARPS = scored_threads(HALVES) / 32 - 1;
    const int r_last = min(q0 + SA_T * HALVES, p.q_len) - 1 + shift;
    const int doc_from = p.window > 0 && p.prefix_lens == nullptr ? max(q0 + shift - p.window + 1, 0) / SA_T : 0;
    const int doc_to = (max(min(p.prefix_lens != nullptr ? p.k_len : p.causal ? r_last + 1 : p.window > 0 ? r_last + p.window : p.k_len, p.k_len), 0) + SA_T - 1) / SA_T;
    int doc_ids[2][4];
    auto ask_docs = [&](int t) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) doc_ids[n][i] = __ldca(docs + min((t + n * DOC_WARPS) * SA_T + 32 * i + lane, p.k_len - 1));
    };
    if (DOCS && warp != W_LOAD) ask_docs(doc_from + helper / 32);
    const int k_end = min(max(key_len, 0), p.k_len), prefix = min(max(prefix_len, 0), k_end);

    auto reach_of = [&](int h) {
        Reach r = {0, 0, 0, 0, 0};
        const int r0 = q0 + h * SA_T, r1 = min(r0 + SA_T, p.q_len) - 1;
        if (r0 > r1) return r;
        int end = p.causal ? r1 + shift + 1 : p.window > 0 ? r1 + shift + p.window : p.k_len;
        end = min(max(end, prefix), k_end);
        const int begin = p.window > 0 ? max(r0 + shift - p.window + 1, 0) : 0;
        r.lo = begin / SA_T;
        r.hi = end > 0 ? (end + SA_T - 1) / SA_T : 0;
        r.prefix = (prefix + SA_T - 1) / SA_T;
        return r;
    };
    Reach reach[HALVES];
    int t_begin = 0x7FFFFFFF, t_end = 0;
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        reach[h] = reach_of(h);
        if (reach[h].hi > 0) t_begin = min(t_begin, reach[h].prefix > 0 ? 0 : reach[h].lo);
        t_end = max(t_end, reach[h].hi);
    }
    auto wanted_by = [&](const Reach& r, int t) {
        if (t >= r.hi || (t < r.lo && t >= r.prefix)) return false;
        if (!DOCS) return true;
        const int2 d = range[t];
        return d.x <= r.doc_max && d.y >= r.doc_min;
    };
    auto wanted = [&](int h, int t) { return wanted_by(reach[h], t); };     // (h known to the compiler: `reach` stays in registers)
    auto next = [&](int t) {                                 // first tile from t on that a half wants
        for (; t < t_end; ++t) {
            bool any = wanted(0, t);
            if constexpr (HALVES == 2) any = any || wanted(1, t);
            if (any) break;
        }
        return t;
    };
    // the n-th tile goes into slot n % SLOTS of its side, K a tile ahead of V
    auto load = [&](int kind, int t, unsigned n) {
        const int s = static_cast<int>(n % SLOTS);
        uint64_t *full = &bars[(kind == 0 ? SB_K_FULL : SB_V_FULL) + s], *empty = &bars[(kind == 0 ? SB_K_EMPTY : SB_V_EMPTY) + s];
        wait_inline(smem_u32(empty), ((n / SLOTS) & 1) ^ 1, wctx, (kind == 0 ? SB_K_EMPTY : SB_V_EMPTY) + s);
        mbar_arrive_expect_tx(full, TILE_BYTES);
        for (int c = 0; c < PANELS; ++c)
            load_tile(ring + (SLOTS * kind + s) * TILE_BYTES + c * PANEL_BYTES, kind == 0 ? &map_k : &map_v, full, c * 64, t * SA_T, kv, b, p.slot_s[1 + kind],
                      p.slot_h[1 + kind]);
    };
    // Q, and the first K where the rules alone say which that is, are on their way while the rest is set up
    if (loader) *abort_flag = muted ? 1 : 0;
    if (loader && !muted) {
        for (int h = 0; h < HALVES; ++h) {
            if (q0 + h * SA_T >= p.q_len) break;
            mbar_arrive_expect_tx(&bars[SB_Q + h], TILE_BYTES);
            for (int c = 0; c < PANELS; ++c)
                load_tile(q_smem + h * TILE_BYTES + c * PANEL_BYTES, &map_q, &bars[SB_Q + h], c * 64, q0 + h * SA_T, head, b, p.slot_s[0], p.slot_h[0]);
            if (h == 0 && !DOCS && next(t_begin) < t_end) load(0, next(t_begin), 0);
        }
    }
    if (DOCS) {
        if (warp != W_LOAD)
            for (int t = doc_from + helper / 32; t < doc_to; t += 2 * DOC_WARPS) {
                if (t >= doc_from + 2 * DOC_WARPS) ask_docs(t);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    int lo = 0x7FFFFFFF, hi = -0x7FFFFFFF - 1;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if ((t + n * DOC_WARPS) * SA_T + 32 * i + lane < k_end) {
                            lo = min(lo, doc_ids[n][i]);
                            hi = max(hi, doc_ids[n][i]);
                        }
                    lo = __reduce_min_sync(0xffffffffu, lo);
                    hi = __reduce_max_sync(0xffffffffu, hi);
                    if (lane == 0 && t + n * DOC_WARPS < doc_to) range[t + n * DOC_WARPS] = make_int2(lo, hi);
                }
            }
        if (warp < HALVES * 4) {
            const bool there = my_row < p.q_len;
            const int lo = __reduce_min_sync(0xffffffffu, there ? my_doc : 0x7FFFFFFF), hi = __reduce_max_sync(0xffffffffu, there ? my_doc : -0x7FFFFFFF - 1);
            if (lane == 0) row_docs[warp] = make_int2(lo, hi);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    if (DOCS) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            reach[h].doc_min = min(min(row_docs[4 * h].x, row_docs[4 * h + 1].x), min(row_docs[4 * h + 2].x, row_docs[4 * h + 3].x));
            reach[h].doc_max = max(max(row_docs[4 * h].y, row_docs[4 * h + 1].y), max(row_docs[4 * h + 2].y, row_docs[4 * h + 3].y));
        }
    }
    // the tile in which the keys end before the tensor does: what V holds there behind the last key is set to zero (P is zero there,
    // but zero times a NaN is none)
    const int fix_tile = k_end < p.k_len && k_end % SA_T != 0 ? k_end / SA_T : -1;

    if (warp < HALVES * 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(scored_regs_softmax(HALVES)));
        if (*abort_flag == 0) {
            // ---------------------------------------------------------------- softmax: one row a thread
            const int h = HALVES == 2 ? warp >> 2 : 0, tid = threadIdx.x & 127;
            Reach mine = reach_of(h);
            if (DOCS) {
                for (int i = 0; i < 4; ++i) {
                    const int2 d = row_docs[4 * h + i];
                    mine.doc_min = i == 0 ? d.x : min(mine.doc_min, d.x);
                    mine.doc_max = i == 0 ? d.y : max(mine.doc_max, d.y);
                }
            }
            const int row = q0 + h * SA_T + tid, pos = row + shift;
            const int warp_row = q0 + static_cast<int>(threadIdx.x & ~31u);
            const int pos0 = warp_row + shift, pos1 = min(warp_row + 31, p.q_len - 1) + shift;       // of the warp's first and last row
            const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
            const uint32_t t_s = t_lane + h * SA_T, t_o = t_lane + COL_O + h * D, t_p = t_lane + COL_P + h * P_STEP;
            constexpr bool changed = MODE != SA_PLAIN;
            const bool capped = MODE == SA_CAP || (MODE == SA_ANY && p.softcap > 0.f);
            const float to_u = capped ? fminf(p.scale / p.softcap, 1e38f) : 0.f, from_u = p.softcap * SA_LOG2E;
            const uint32_t s_bar = smem_u32(&bars[SB_S + h]);
            NearTanh tanh_near;
            if (capped) tanh_near = NearTanh(to_u, from_u);
            const float raw_scale = p.scale * SA_LOG2E;      // of a score that nothing changes, to log2 units
            const float sc = changed ? 1.f : raw_scale;      // what is left to multiply by when the exponential is taken
            const float slope = p.slopes != nullptr ? __ldca(p.slopes + head) * SA_LOG2E : 0.f;
            const int2 warp_docs = DOCS ? row_docs[warp] : make_int2(0, 0);
            const int see_lo = p.window > 0 ? pos - p.window + 1 : -0x40000000, see_hi = p.causal ? pos : p.window > 0 ? pos + p.window - 1 : 0x40000000;
            // the tiles of which all is visible to all of the warp's rows (documents aside): [0, full_prefix) and [full_from, full_to)
            const int full_prefix = prefix / SA_T, full_from = p.window > 0 ? max(pos1 - p.window + SA_T, 0) / SA_T : 0;
            const int full_to = max(min(p.causal ? pos0 + 1 : p.window > 0 ? pos0 + p.window : p.k_len, k_end), 0) / SA_T;
            float m_ref = -INFINITY, l_sum = 0.f;
            int done = 0;
            for (int t = mine.prefix > 0 ? 0 : mine.lo; t < mine.hi; ++t) {
                if (t < mine.lo && t >= mine.prefix) {                       // from the prefix to the window
                    t = mine.lo;
                    if (t >= mine.hi) break;
                }
                if (DOCS) {
                    const int2 d = range[t];
                    if (d.x > mine.doc_max || d.y < mine.doc_min) continue;
                }
                const int k0 = t * SA_T;
                const bool full = t < full_prefix || (t >= full_from && t < full_to);
                // Which keys are of the row's document: a ballot for each document among the warp's rows (one to three of them, where
                // sequences are packed), before the scores are there
                bool one_doc = true;
                uint32_t doc_keys[4] = {0u, 0u, 0u, 0u};
                if (DOCS) {
                    const int2 d = range[t];
                    one_doc = d.x == d.y && warp_docs.x == warp_docs.y && d.x == warp_docs.x;
                    if (!one_doc) {
                        int key_doc[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) key_doc[i] = __ldca(docs + min(k0 + 32 * i + lane, p.k_len - 1));
                        for (unsigned rest = 0xffffffffu; rest != 0u;) {
                            const int doc = __shfl_sync(0xffffffffu, my_doc, __ffs(rest) - 1);
                            const bool is = my_doc == doc;
                            rest &= ~__ballot_sync(0xffffffffu, is);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t keys = __ballot_sync(0xffffffffu, key_doc[i] == doc);
                                doc_keys[i] = is ? keys : doc_keys[i];
                            }
                        }
                    }
                }
                wait_inline(s_bar, static_cast<uint32_t>(done & 1), wctx, SB_S + h);
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld32(t_s + 32 * i, s[i]);
                tc_wait_ld();
#define S_AT(c) s[(c) >> 5][(c) & 31]
                // The cap alone: a row's largest score is its largest raw one, capped, so that the polynomial can go into the loop of
                // exponentials, whose unit is busy all along while the others idle (in_loop 1, 2: which; 0: the scores are final)
                int in_loop = 0;
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                auto largest = [&] {
#pragma unroll
                    for (int c = 0; c < SA_T; c += 8)
#pragma unroll
                        for (int i = 0; i < 4; ++i) mx[i] = max3f(mx[i], __uint_as_float(S_AT(c + 2 * i)), __uint_as_float(S_AT(c + 2 * i + 1)));
                    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                };
                auto cap_exactly = [&] {
                    cap_in_tmem(t_s, p.scale, 1.f / p.softcap, from_u);
#pragma unroll
                    for (int i = 0; i < 4; ++i) tmem_ld32(t_s + 32 * i, s[i]);
                    tc_wait_ld();
                };
                float top = -INFINITY;
                if constexpr (MODE == SA_CAP) {
                    float mn[4] = {INFINITY, INFINITY, INFINITY, INFINITY};
                    top = largest();
#pragma unroll
                    for (int c = 0; c < SA_T; c += 8)
#pragma unroll
                        for (int i = 0; i < 4; ++i) mn[i] = min3f(mn[i], __uint_as_float(S_AT(c + 2 * i)), __uint_as_float(S_AT(c + 2 * i + 1)));
                    const float reached = fmaxf(top, -fminf(fminf(mn[0], mn[1]), fminf(mn[2], mn[3])));
                    if (__builtin_expect(__all_sync(0xffffffffu, reached <= tanh_near.near_end), 1)) in_loop = 1;
                    else if (__all_sync(0xffffffffu, reached <= tanh_near.far_end)) in_loop = 2;
                    else cap_exactly();
                }
                if constexpr (MODE == SA_ANY) {
                    if (capped) {
                        float reached = 0.f;
#pragma unroll
                        for (int c = 0; c < SA_T; c += 2) reached = max3f(reached, fabsf(__uint_as_float(S_AT(c))), fabsf(__uint_as_float(S_AT(c + 1))));
                        if (__builtin_expect(__all_sync(0xffffffffu, reached <= tanh_near.near_end), 1)) {
#pragma unroll
                            for (int c = 0; c < SA_T; c += 2) {
                                const float2 y = odd_polynomial(pk2(__uint_as_float(S_AT(c)), __uint_as_float(S_AT(c + 1))), tanh_near.near);
                                S_AT(c) = __float_as_uint(y.x);
                                S_AT(c + 1) = __float_as_uint(y.y);
                            }
                        } else if (__all_sync(0xffffffffu, reached <= tanh_near.far_end)) {
#pragma unroll
                            for (int c = 0; c < SA_T; c += 2) {
                                const float2 y = odd_polynomial(pk2(__uint_as_float(S_AT(c)), __uint_as_float(S_AT(c + 1))), tanh_near.far);
                                S_AT(c) = __float_as_uint(y.x);
                                S_AT(c + 1) = __float_as_uint(y.y);
                            }
                        } else {
                            cap_exactly();
                        }
                    }
                }
                if constexpr (OWN_P) {                       // S may be overwritten from here on
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars[SB_READ + h]);
                }
                if constexpr (MODE == SA_ANY) {
                    float sc_now = capped ? 1.f : raw_scale;
                    // distances of the warp's rows in this tile: k0 - pos1 .. k0 + 127 - pos0
                    const int near = k0 - pos1, far = k0 + SA_T - 1 - pos0;
                    if (p.slopes != nullptr) {
                        if (far <= 0 || near >= 0) {         // all behind or all ahead: -slope * |distance| is linear
                            const float g = far <= 0 ? slope : -slope, at = g * static_cast<float>(k0 - pos);
                            const float2 now2 = pk2(sc_now, sc_now);
                            const float2 step[4] = {pk2(0.f, g), pk2(2.f * g, 3.f * g), pk2(4.f * g, 5.f * g), pk2(6.f * g, 7.f * g)};
#pragma unroll
                            for (int c = 0; c < SA_T; c += 8) {
                                const float from = fmaf(g, static_cast<float>(c), at);
                                const float2 from2 = pk2(from, from);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float2 y = fma2(pk2(__uint_as_float(S_AT(c + 2 * i)), __uint_as_float(S_AT(c + 2 * i + 1))), now2, add2(from2, step[i]));
                                    S_AT(c + 2 * i) = __float_as_uint(y.x);
                                    S_AT(c + 2 * i + 1) = __float_as_uint(y.y);
                                }
                            }
                        } else {
                            const float away = static_cast<float>(k0 - pos);
#pragma unroll
                            for (int c = 0; c < SA_T; ++c)
                                S_AT(c) = __float_as_uint(fmaf(__uint_as_float(S_AT(c)), sc_now, -slope * fabsf(away + static_cast<float>(c))));
                        }
                        sc_now = 1.f;
                    }
                    if (p.distance_bias != nullptr) {
                        if (far <= -p.radius || near >= p.radius) {          // all of it beyond the table
                            const float x = table[near >= p.radius ? 2 * p.radius + SA_PAD : SA_PAD];
                            const float2 x2 = pk2(x, x), now2 = pk2(sc_now, sc_now);
#pragma unroll
                            for (int c = 0; c < SA_T; c += 2) {
                                const float2 y = fma2(pk2(__uint_as_float(S_AT(c)), __uint_as_float(S_AT(c + 1))), now2, x2);
                                S_AT(c) = __float_as_uint(y.x);
                                S_AT(c + 1) = __float_as_uint(y.y);
                            }
                        } else {
                            // (rows behind the last one are kept inside the table)
                            const float* at = table + min(max(k0 - pos + p.radius + SA_PAD, 0), 2 * p.radius + 2 * SA_PAD - SA_T + 1);
#pragma unroll
                            for (int c = 0; c < SA_T; c += 2) {
                                const float2 y = fma2(pk2(__uint_as_float(S_AT(c)), __uint_as_float(S_AT(c + 1))), pk2(sc_now, sc_now), pk2(at[c], at[c + 1]));
                                S_AT(c) = __float_as_uint(y.x);
                                S_AT(c + 1) = __float_as_uint(y.y);
                            }
                        }
                    }
                }
                if (__builtin_expect(!full || !one_doc, DOCS)) {
                    const uint4 on = full ? make_uint4(~0u, ~0u, ~0u, ~0u) : visible_keys(see_lo - k0, see_hi - k0, prefix - k0, k_end - k0);
                    uint32_t word[4] = {on.x, on.y, on.z, on.w};
                    if (DOCS && !one_doc) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) word[i] &= doc_keys[i];
                    }
#pragma unroll
                    for (int c = 0; c < SA_T; ++c)
                        if ((word[c >> 5] & (1u << (c & 31))) == 0) S_AT(c) = 0xFF800000u;
                }
                if (in_loop == 0 || !full) {
                    mx[0] = mx[1] = mx[2] = mx[3] = -INFINITY;
                    top = largest();
                }
                if (in_loop == 1 && top > -INFINITY) top = odd_polynomial(pk2(top, top), tanh_near.near).x;
                if (in_loop == 2 && top > -INFINITY) top = odd_polynomial(pk2(top, top), tanh_near.far).x;
                top *= sc;
                const bool need = top > m_ref + SA_RESCALE || (m_ref == -INFINITY && top > -INFINITY);
                if (__builtin_expect(__any_sync(0xffffffffu, need), 0)) {
                    float alpha = 1.f;
                    if (need) {
                        alpha = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - top);
                        m_ref = top;
                        l_sum *= alpha;
                    }
                    if (done > 0) {
                        // Where P lies over S, S was issued behind the products before it and is there: so are they.  Else they have to
                        // be waited for (SB_O counts them).
                        if constexpr (OWN_P) {
                            wait_inline(smem_u32(&bars[SB_O + h]), static_cast<uint32_t>((done - 1) & 1), wctx, SB_O + h);
                            tc_fence_after();
                        }
                        rescale_o<D>(t_o, alpha);
                    }
                }
                const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
                const float2 sc2 = pk2(sc, sc), negm2 = pk2(neg_m, neg_m);
                float2 sum_a = pk2(0.f, 0.f), sum_b = pk2(0.f, 0.f);
                auto exponentials = [&](auto&& less_reference) {
#pragma unroll
                    for (int part = 0; part < 2; ++part) {       // P goes to the issuer in two parts of 64 keys
#pragma unroll
                        for (int i = part * 32; i < part * 32 + 32; ++i) {
                            const float2 x = less_reference(pk2(__uint_as_float(S_AT(2 * i)), __uint_as_float(S_AT(2 * i + 1))));
                            const float e0 = fast_exp2(x.x), e1 = fast_exp2(x.y);
                            if (i & 1) sum_b = add2(sum_b, pk2(e0, e1));
                            else sum_a = add2(sum_a, pk2(e0, e1));
                            S_AT(i) = pack_pair<BF16>(e0, e1);   // the scores of pair i were used above
                        }
                        if constexpr (OWN_P) {
                            // the products that read the P before this one have to be through: they are where O is complete
                            if (part == 0 && done > 0) {
                                wait_inline(smem_u32(&bars[SB_O + h]), static_cast<uint32_t>((done - 1) & 1), wctx, SB_O + h);
                                tc_fence_after();
                            }
                        }
                        tmem_st32(t_p + 32 * part, s[part]);
                        tc_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bars[(part == 0 ? SB_P0 : SB_P1) + h]);
                    }
                };
                if (in_loop == 1) exponentials([&](float2 v) { return odd_polynomial_plus(v, tanh_near.near, negm2); });
                else if (in_loop == 2) exponentials([&](float2 v) { return odd_polynomial_plus(v, tanh_near.far, negm2); });
                else exponentials([&](float2 v) { return fma2(v, sc2, negm2); });
                const float2 sum = add2(sum_a, sum_b);
                l_sum += sum.x + sum.y;
#undef S_AT
                ++done;
            }
            // ---------------------------------------------------------------- O / l
            // The rows leave through shared memory, 32 of a warp at a time, over the half's Q: every product that read it is complete.  (Stored
            // from registers, each lane its row, they took 1200 cycles a warp for heads of 64 and up to 6000 for heads of 128.)
            if (done > 0) {
                wait_inline(smem_u32(&bars[SB_O + h]), static_cast<uint32_t>((done - 1) & 1), wctx, SB_O + h);
                tc_fence_after();
            } else if (q0 + h * SA_T < p.q_len) {
                wait_inline(smem_u32(&bars[SB_Q + h]), 0, wctx, SB_Q + h);       // nobody used it: it may still be on its way
            }
            // a row that saw nothing has no maximum; where all it saw is NaN its sum says so
            const bool any = done > 0 && (m_ref > -INFINITY || l_sum != l_sum);
            const float inv = any ? 1.f / l_sum : 0.f;
            if (warp_row < p.q_len) {
#pragma unroll
                for (int c = 0; c < PANELS; ++c) {
                    unsigned char* slab = q_smem + h * TILE_BYTES + c * PANEL_BYTES + (warp & 3) * 4096;
                    uint32_t o[2][32];
                    if (done > 0) {
                        tmem_ld32(t_o + 64 * c, o[0]);
                        tmem_ld32(t_o + 64 * c + 32, o[1]);
                        tc_wait_ld();
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        auto two = [&](int j) {
                            const int k = 8 * i + j;
                            return any ? pack_pair<BF16>(__uint_as_float(o[k >> 5][k & 31]) * inv, __uint_as_float(o[k >> 5][(k & 31) + 1]) * inv) : 0u;
                        };
                        *reinterpret_cast<uint4*>(slab + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(two(0), two(2), two(4), two(6));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        store_rows(&map_o, slab, 64 * c, warp_row, head, b, p.slot_s[3], p.slot_h[3]);
                        tma_store_commit();
                    }
                }
                if (lane == 0) tma_store_wait_all();
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(scored_regs_other(HALVES)));
        if (*abort_flag == 0 && warp == W_LOAD) {
            // ---------------------------------------------------------------- TMA producer
            int fix_slot = -1;
            uint32_t fix_phase = 0;
            if (lane == 0) {
                int t = next(t_begin);
                if (DOCS && t < t_end) load(0, t, 0);
                for (unsigned n = 0; t < t_end; ++n) {
                    const int tn = next(t + 1);
                    // (the one slot of K is free later than the one of V)
                    if (SLOTS == 1) load(1, t, n);
                    if (tn < t_end) load(0, tn, n + 1);
                    if (SLOTS > 1) load(1, t, n);
                    if (t == fix_tile) {
                        fix_slot = static_cast<int>(n % SLOTS);
                        fix_phase = (n / SLOTS) & 1;
                    }
                    t = tn;
                }
            }
            fix_slot = __shfl_sync(0xffffffffu, fix_slot, 0);
            fix_phase = __shfl_sync(0xffffffffu, fix_phase, 0);
            if (fix_slot >= 0) {                             // it is the last tile of all: nothing more goes into its slot
                mbar_wait(&bars[SB_V_FULL + fix_slot], fix_phase, wctx, SB_V_FULL + fix_slot);
                for (int i = (k_end % SA_T) * 8 + lane; i < SA_T * 8; i += 32)
#pragma unroll
                    for (int c = 0; c < PANELS; ++c)
                        *reinterpret_cast<uint4*>(ring + (SLOTS + fix_slot) * TILE_BYTES + c * PANEL_BYTES + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[SB_FIX]);
            }
        } else if (*abort_flag == 0 && warp == W_MMA) {
            // ---------------------------------------------------------------- tcgen05 issuer
            if (elect_one()) {
                constexpr uint32_t type = BF16 ? (1u << 7) | (1u << 10) : 0u;
                constexpr uint32_t idesc_qk = make_idesc_f16(SA_T, SA_T, false) | type, idesc_pv = make_idesc_f16(SA_T, D, true) | type;
                const uint64_t q_desc = make_smem_desc_sw128(smem_u32(q_smem), 16, 1024);
                const uint64_t k_desc = make_smem_desc_sw128(smem_u32(ring), 16, 1024);
                const uint64_t v_desc = make_smem_desc_sw128(smem_u32(ring + SLOTS * TILE_BYTES), PANEL_BYTES, 1024);
                const uint32_t bar0 = smem_u32(bars);
                auto wait = [&](int bar, uint32_t parity) { wait_inline(bar0 + 8 * bar, parity, wctx, bar); };
                int done[HALVES];                            // tiles whose PV has been issued
#pragma unroll
                for (int h = 0; h < HALVES; ++h) done[h] = 0;
                auto qk = [&](int h, unsigned n) {           // S = Q K^T of the n-th tile
                    if (done[h] == 0) wait(SB_Q + h, 0);
                    tc_fence_after();
                    mma_chain_ss<D / 16>(tmem + h * SA_T, q_desc + static_cast<uint64_t>(h * (TILE_BYTES >> 4)), k_desc + static_cast<uint64_t>((n % SLOTS) * (TILE_BYTES >> 4)), idesc_qk);
                    tc_commit_addr(bar0 + 8 * (SB_S + h));
                };
                auto pv = [&](int h, unsigned n) {           // O (+)= P V
                    const uint64_t v = v_desc + static_cast<uint64_t>((n % SLOTS) * (TILE_BYTES >> 4));
                    const uint32_t parity = static_cast<uint32_t>(done[h] & 1), o = tmem + COL_O + h * D, q = tmem + COL_P + h * P_STEP;
                    wait(SB_P0 + h, parity);
                    tc_fence_after();
                    mma_chain_ts(o, q, v, idesc_pv, done[h] > 0 ? 1u : 0u);
                    wait(SB_P1 + h, parity);
                    tc_fence_after();
                    mma_chain_ts(o, q + 32, v + 512, idesc_pv, 1u);
                    tc_commit_addr(bar0 + 8 * (SB_O + h));
                    ++done[h];
                };
                int t = next(t_begin);
                if (t < t_end) {
                    wait(SB_K_FULL, 0);
#pragma unroll
                    for (int h = 0; h < HALVES; ++h)
                        if (wanted(h, t)) qk(h, 0);
                    tc_commit_addr(bar0 + 8 * SB_K_EMPTY);
                }
                for (unsigned n = 0; t < t_end; ++n) {
                    const int tn = next(t + 1);
                    const int ks = static_cast<int>((n + 1) % SLOTS), vs = static_cast<int>(n % SLOTS);
                    auto k_there = [&] { wait(SB_K_FULL + ks, ((n + 1) / SLOTS) & 1); };
                    if constexpr (OWN_P) {
                        if (tn < t_end) k_there();
#pragma unroll
                        for (int h = 0; h < HALVES; ++h) {
                            if (tn < t_end && wanted(h, tn)) {
                                if (wanted(h, t)) wait(SB_READ + h, static_cast<uint32_t>(done[h] & 1));     // S is in registers
                                qk(h, n + 1);
                            }
                        }
                        if (tn < t_end) tc_commit_addr(bar0 + 8 * (SB_K_EMPTY + ks));
                    }
                    wait(SB_V_FULL + vs, (n / SLOTS) & 1);
                    if (t == fix_tile) wait(SB_FIX, 0);
#pragma unroll
                    for (int h = 0; h < HALVES; ++h) {
                        if (wanted(h, t)) pv(h, n);
                        if constexpr (!OWN_P)
                            if (tn < t_end && wanted(h, tn)) {
                                k_there();
                                qk(h, n + 1);
                            }
                    }
                    tc_commit_addr(bar0 + 8 * (SB_V_EMPTY + vs));
                    if constexpr (!OWN_P)
                        if (tn < t_end) tc_commit_addr(bar0 + 8 * (SB_K_EMPTY + ks));
                    t = tn;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        if (*abort_flag != 0)                                // a wait ran out: copies and products in flight end before their memory is given back
            for (const long long t0 = clock64(); clock64() - t0 < SA_DRAIN_CYCLES;) {}
        tmem_dealloc(tmem, TMEM_COLS);
    }
}


using ScoredMaps = CUtensorMap[4];             // q, k, v, out
// Launches the kernel for one head size (scored_attn_64.cu, scored_attn_128.cu: a translation unit each, they take long to compile)
template <int D>
int launch_scored(const ScoredMaps& maps, const ScoredParams& p, int halves, bool bf16, int what, long long blocks, size_t smem, cudaStream_t stream);

template <int D, int HALVES, bool BF16, int WHAT>
int launch_one(const ScoredMaps& maps, const ScoredParams& p, long long blocks, size_t smem, cudaStream_t stream) {
    if (int rc = allow_shared_memory<scored_attn_kernel<D, HALVES, BF16, WHAT>>()) return rc;
    LaunchConfig lc(dim3(static_cast<unsigned>(blocks)), static_cast<unsigned>(scored_threads(HALVES)), smem, stream);
    STOF_CUDA(cudaLaunchKernelEx(&lc.cfg, scored_attn_kernel<D, HALVES, BF16, WHAT>, maps[0], maps[1], maps[2], maps[3], p));
    return STOF_OK;
}
template <int D, int HALVES, bool BF16>
int launch_what(const ScoredMaps& maps, const ScoredParams& p, int what, long long blocks, size_t smem, cudaStream_t stream) {
    switch (what) {
        case SA_PLAIN: return launch_one<D, HALVES, BF16, SA_PLAIN>(maps, p, blocks, smem, stream);
        case SA_CAP: return launch_one<D, HALVES, BF16, SA_CAP>(maps, p, blocks, smem, stream);
        case SA_ANY: return launch_one<D, HALVES, BF16, SA_ANY>(maps, p, blocks, smem, stream);
        case SA_PLAIN | SA_DOCS: return launch_one<D, HALVES, BF16, SA_PLAIN | SA_DOCS>(maps, p, blocks, smem, stream);
        default: return launch_one<D, HALVES, BF16, SA_ANY | SA_DOCS>(maps, p, blocks, smem, stream);
    }
}
template <int D>
int launch_scored_impl(const ScoredMaps& maps, const ScoredParams& p, int halves, bool bf16, int what, long long blocks, size_t smem, cudaStream_t stream) {
    if constexpr (D == 128)                                  // (heads of 64: one half, see the caller)
        if (halves == 2) return bf16 ? launch_what<D, 2, true>(maps, p, what, blocks, smem, stream) : launch_what<D, 2, false>(maps, p, what, blocks, smem, stream);
    return bf16 ? launch_what<D, 1, true>(maps, p, what, blocks, smem, stream) : launch_what<D, 1, false>(maps, p, what, blocks, smem, stream);
}

}  // namespace stof
