// Attention whose scores are changed by a formula (tanh cap, distance bias) and masked by rules (causal, window, prefix, documents,
// padding), for sm_100a: TMA-fed tcgen05 products with the accumulators in tensor memory, online softmax in registers.
//
// Per thread block one stretch of 128 query rows, or two (HALVES) that share every K/V tile of 128 keys.  Each half has its own S
// (128 x 128 fp32 in tensor memory; P overwrites it as 16-bit numbers) and O (128 x D fp32), its own softmax warps - one row a
// thread - and its own list of tiles: those that the rules leave anything of.  While one half's warps work on their scores the
// tensor core serves the other half.
//   warps 0..3 (and 4..7)   softmax of the half
//   next warp               TMA producer: Q, then K and V tiles through one ring of four slots
//   last warp               tcgen05 issuer: O += P V of tile t, then S = Q K^T of the next one, half by half
// A tile is classified per warp (32 rows): nothing to mask, or masked element by element.
#include <atomic>

#include "cache_common.cuh"
#include "stof_host.h"
#include "stof_ptx.cuh"

namespace stof {
namespace {

constexpr int SA_T = 128;                    // rows of a half, keys of a tile
constexpr int SA_STAGES = 4;
constexpr int SA_PAD = 256;                  // the distance table in shared memory goes on for so long on both sides: a tile that meets the table needs no clamp
constexpr float SA_RESCALE = 8.0f;           // log2 units by which a row's maximum may outgrow the reference of its P (P <= 2^8)
constexpr float SA_LOG2E = 1.4426950408889634f;
#ifndef SA_POLY_PAIRS
#define SA_POLY_PAIRS 2                      // of every 8 pairs of exponentials, so many on the FMA pipe
#endif

struct ScoredParams {
    void* out;
    long long out_stride[3];
    const float *slopes, *distance_bias;
    const int *documents, *prefix_lens, *key_lens;
    long long documents_stride;
    int* status;
    float scale, softcap;
    int causal, window, radius;
    int batch, heads, group, q_len, k_len, q_tiles;
    int slot_s[3], slot_h[3], slot_b[3];     // of q, k, v: which coordinate of the tensor map is the row, the head, the batch
    int table_bytes, range_bytes;
};

enum { SB_Q = 0, SB_S = 2, SB_P = 4, SB_O = 6, SB_FIX = 8, SB_FULL = 9, SB_EMPTY = SB_FULL + SA_STAGES, SB_COUNT = SB_EMPTY + SA_STAGES };

__device__ __forceinline__ void load_tile(unsigned char* dst, const CUtensorMap* map, uint64_t* bar, int col, int row, int head, int batch, int slot_s, int slot_h) {
    // the three outer coordinates are in the order of their strides
    const int c1 = slot_s == 1 ? row : slot_h == 1 ? head : batch;
    const int c2 = slot_s == 2 ? row : slot_h == 2 ? head : batch;
    const int c3 = slot_s == 3 ? row : slot_h == 3 ? head : batch;
    tma_load_4d(dst, map, bar, col, c1, c2, c3);
}

__device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// tanh of a pair, |u| <= 1: odd polynomial, relative error below 7e-6 (a weighted least-squares fit moved towards the minimax one).
// A score of 40 is then off by 3e-4, less than P's rounding to fp16 makes of it.
__device__ __forceinline__ float2 tanh_near(float2 u) {
    const float2 w = mul2(u, u);
    float2 p = fma2(w, pk2(0.009036419913172722f, 0.009036419913172722f), pk2(-0.044817544519901276f, -0.044817544519901276f));
    p = fma2(p, w, pk2(0.13036811351776123f, 0.13036811351776123f));
    p = fma2(p, w, pk2(-0.3329806625843048f, -0.3329806625843048f));
    p = fma2(p, w, pk2(0.999993085861206f, 0.999993085861206f));
    return mul2(p, u);
}
// tanh(u) = 1 - 2 / (1 + e^(2u)) for any u
__device__ __forceinline__ float tanh_any(float u) { return 1.f - 2.f * fast_reciprocal(1.f + fast_exp2(u * (2.f * SA_LOG2E))); }

template <int D>
__device__ __noinline__ void rescale_o(uint32_t t_o, float alpha) {
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

// What a stretch of rows sees: tiles [lo, hi) and [0, prefix), where documents agree
struct Reach {
    int lo, hi, prefix, doc_min, doc_max;
};

template <int D, int HALVES, bool BF16>
__global__ void __launch_bounds__(HALVES * 128 + 64, HALVES == 1 && D == 64 ? 2 : 1) scored_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                        const __grid_constant__ CUtensorMap map_v, const ScoredParams p) {
    constexpr int PANELS = D / 64;                           // 64-column panels of a tile, 128 rows of 128 swizzled bytes each
    constexpr int PANEL_BYTES = SA_T * 128, TILE_BYTES = PANELS * PANEL_BYTES;
    constexpr int W_LOAD = HALVES * 4, W_MMA = W_LOAD + 1;
    constexpr int TMEM_COLS = HALVES == 2 ? 512 : 256;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* q_smem = smem;
    unsigned char* ring = q_smem + HALVES * TILE_BYTES;
    float* table = reinterpret_cast<float*>(ring + SA_STAGES * TILE_BYTES);
    int2* range = reinterpret_cast<int2*>(reinterpret_cast<unsigned char*>(table) + p.table_bytes);
    __shared__ __align__(8) uint64_t bars[SB_COUNT];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ int2 row_docs[HALVES * 4];                    // smallest and largest document of each softmax warp's rows
    __shared__ __align__(16) int key_docs[HALVES][2][SA_T];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &abort_word;
    const WaitCtx wctx{abort_flag, p.status};
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars[SB_Q + i], 1);
            mbar_init(&bars[SB_S + i], 1);
            mbar_init(&bars[SB_P + i], 4);
            mbar_init(&bars[SB_O + i], 1);
        }
        mbar_init(&bars[SB_FIX], 1);
        for (int i = 0; i < SA_STAGES; ++i) {
            mbar_init(&bars[SB_FULL + i], 1);
            mbar_init(&bars[SB_EMPTY + i], 1);
        }
        fence_mbar_init();
    }
    if (warp == W_MMA) {
        tmem_alloc(&tmem_slot, TMEM_COLS);
        tmem_relinquish();
    }
    grid_dependency_wait();
    grid_launch_dependents();
    if (threadIdx.x == 0) *abort_flag = failure_reported(p.status) ? 1 : 0;

    // the heaviest stretches first: with a causal mask those at the end of the sequence
    const int heads_all = p.batch * p.heads;
    const int row_tile = p.q_tiles - 1 - static_cast<int>(blockIdx.x / heads_all), bh = static_cast<int>(blockIdx.x % heads_all);
    const int b = bh / p.heads, head = bh % p.heads, kv = head / p.group;
    const int q0 = row_tile * (SA_T * HALVES), shift = p.k_len - p.q_len;
    const int k_end = p.key_lens != nullptr ? min(max(p.key_lens[b], 0), p.k_len) : p.k_len;
    const int prefix = p.prefix_lens != nullptr ? min(max(p.prefix_lens[b], 0), k_end) : 0;
    const int* docs = p.documents != nullptr ? p.documents + b * p.documents_stride : nullptr;

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
    // tables into shared memory
    if (p.distance_bias != nullptr) {
        const float* src = p.distance_bias + static_cast<size_t>(head) * (2 * p.radius + 1);
        for (int i = threadIdx.x; i < 2 * p.radius + 1 + 2 * SA_PAD; i += blockDim.x) table[i] = __ldca(src + min(max(i - SA_PAD, 0), 2 * p.radius)) * SA_LOG2E;
    }
    int my_doc = 0;
    if (docs != nullptr) {
        for (int t = t_begin + warp; t < t_end; t += HALVES * 4 + 2) {
            int lo = 0x7FFFFFFF, hi = -0x7FFFFFFF - 1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = t * SA_T + 32 * i + lane;
                if (j < k_end) {
                    const int d = __ldca(docs + j);
                    lo = min(lo, d);
                    hi = max(hi, d);
                }
            }
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi);
            if (lane == 0) range[t] = make_int2(lo, hi);
        }
        if (warp < HALVES * 4) {
            const int row = q0 + static_cast<int>(threadIdx.x);
            if (row < p.q_len) my_doc = __ldca(docs + row + shift);
            const int lo = __reduce_min_sync(0xffffffffu, row < p.q_len ? my_doc : 0x7FFFFFFF), hi = __reduce_max_sync(0xffffffffu, row < p.q_len ? my_doc : -0x7FFFFFFF - 1);
            if (lane == 0) row_docs[warp] = make_int2(lo, hi);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    if (docs != nullptr) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            reach[h].doc_min = min(min(row_docs[4 * h].x, row_docs[4 * h + 1].x), min(row_docs[4 * h + 2].x, row_docs[4 * h + 3].x));
            reach[h].doc_max = max(max(row_docs[4 * h].y, row_docs[4 * h + 1].y), max(row_docs[4 * h + 2].y, row_docs[4 * h + 3].y));
        }
    }
    auto wanted = [&](int h, int t) {
        const Reach& r = reach[h];
        if (t >= r.hi || (t < r.lo && t >= r.prefix)) return false;
        if (docs == nullptr) return true;
        const int2 d = range[t];
        return d.x <= r.doc_max && d.y >= r.doc_min;
    };
    auto next = [&](int t) {                                 // first tile from t on that a half wants
        for (; t < t_end; ++t) {
            bool any = wanted(0, t);
            if constexpr (HALVES == 2) any = any || wanted(1, t);
            if (any) break;
        }
        return t;
    };
    // the tile in which the keys end before the tensor does: what V holds there behind the last key is set to zero (P is zero there,
    // but zero times a NaN is none)
    const int fix_tile = k_end < p.k_len && k_end % SA_T != 0 ? k_end / SA_T : -1;

    if (*abort_flag == 0) {
        if (warp == W_LOAD) {
            // ---------------------------------------------------------------- TMA producer
            unsigned u = 0;
            int fix_slot = -1;
            uint32_t fix_phase = 0;
            if (lane == 0) {
                tma_prefetch_desc(&map_q);
                tma_prefetch_desc(&map_k);
                tma_prefetch_desc(&map_v);
                int t = next(t_begin);
                if (t < t_end) {
                    for (int h = 0; h < HALVES; ++h) {
                        if (q0 + h * SA_T >= p.q_len) break;
                        mbar_arrive_expect_tx(&bars[SB_Q + h], TILE_BYTES);
                        for (int c = 0; c < PANELS; ++c)
                            load_tile(q_smem + h * TILE_BYTES + c * PANEL_BYTES, &map_q, &bars[SB_Q + h], c * 64, q0 + h * SA_T, head, b, p.slot_s[0], p.slot_h[0]);
                    }
                }
                for (; t < t_end; t = next(t + 1)) {
                    for (int kind = 0; kind < 2; ++kind, ++u) {
                        const int s = static_cast<int>(u % SA_STAGES);
                        mbar_wait(&bars[SB_EMPTY + s], ((u / SA_STAGES) & 1) ^ 1, wctx, SB_EMPTY + s);
                        mbar_arrive_expect_tx(&bars[SB_FULL + s], TILE_BYTES);
                        for (int c = 0; c < PANELS; ++c)
                            load_tile(ring + s * TILE_BYTES + c * PANEL_BYTES, kind == 0 ? &map_k : &map_v, &bars[SB_FULL + s], c * 64, t * SA_T, kv, b,
                                      p.slot_s[1 + kind], p.slot_h[1 + kind]);
                        if (kind == 1 && t == fix_tile) {
                            fix_slot = s;
                            fix_phase = (u / SA_STAGES) & 1;
                        }
                    }
                }
            }
            fix_slot = __shfl_sync(0xffffffffu, fix_slot, 0);
            fix_phase = __shfl_sync(0xffffffffu, fix_phase, 0);
            if (fix_slot >= 0) {                             // it is the last tile of all: nothing more goes into its slot
                mbar_wait(&bars[SB_FULL + fix_slot], fix_phase, wctx, SB_FULL + fix_slot);
                for (int i = (k_end % SA_T) * 8 + lane; i < SA_T * 8; i += 32)
#pragma unroll
                    for (int c = 0; c < PANELS; ++c)
                        *reinterpret_cast<uint4*>(ring + fix_slot * TILE_BYTES + c * PANEL_BYTES + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[SB_FIX]);
            }
        } else if (warp == W_MMA) {
            // ---------------------------------------------------------------- tcgen05 issuer
            if (lane == 0) {
                constexpr uint32_t type = BF16 ? (1u << 7) | (1u << 10) : 0u;
                constexpr uint32_t idesc_qk = make_idesc_f16(SA_T, SA_T, false) | type, idesc_pv = make_idesc_f16(SA_T, D, true) | type;
                const uint64_t q_desc = make_smem_desc_sw128(smem_u32(q_smem), 16, 1024);
                const uint64_t k_desc = make_smem_desc_sw128(smem_u32(ring), 16, 1024);
                const uint64_t v_desc = make_smem_desc_sw128(smem_u32(ring), PANEL_BYTES, 1024);
                auto qk = [&](int h, int slot) {             // S = Q K^T
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = static_cast<uint32_t>((kk / 4) * PANEL_BYTES + (kk % 4) * 32) >> 4;
                        mma_f16_ss(tmem + h * SA_T, q_desc + static_cast<uint64_t>(h * (TILE_BYTES >> 4) + off), k_desc + static_cast<uint64_t>(slot * (TILE_BYTES >> 4) + off),
                                   idesc_qk, kk > 0 ? 1u : 0u);
                    }
                    tc_commit(&bars[SB_S + h]);
                };
                auto pv = [&](int h, int slot, uint32_t accumulate) {        // O (+)= P V
#pragma unroll
                    for (int kk = 0; kk < SA_T / 16; ++kk)
                        mma_f16_ts(tmem + HALVES * SA_T + h * D, tmem + h * SA_T + kk * 8, v_desc + static_cast<uint64_t>((slot * TILE_BYTES + kk * 2048) >> 4), idesc_pv,
                                   kk > 0 ? 1u : accumulate);
                };
                unsigned u = 0;                              // ring slots taken: K, V, K, V, ...
                int done[HALVES];
#pragma unroll
                for (int h = 0; h < HALVES; ++h) done[h] = 0;
                int t = next(t_begin);
                if (t < t_end) {
                    mbar_wait(&bars[SB_FULL], 0, wctx, SB_FULL);
#pragma unroll
                    for (int h = 0; h < HALVES; ++h)
                        if (wanted(h, t)) {
                            mbar_wait(&bars[SB_Q + h], 0, wctx, SB_Q + h);
                            tc_fence_after();
                            qk(h, 0);
                        }
                    tc_commit(&bars[SB_EMPTY]);
                    ++u;
                }
                while (t < t_end) {
                    const int tn = next(t + 1);
                    const int vs = static_cast<int>(u % SA_STAGES), ks = static_cast<int>((u + 1) % SA_STAGES);
                    mbar_wait(&bars[SB_FULL + vs], (u / SA_STAGES) & 1, wctx, SB_FULL + vs);
                    if (t == fix_tile) mbar_wait(&bars[SB_FIX], 0, wctx, SB_FIX);
                    if (tn < t_end) mbar_wait(&bars[SB_FULL + ks], ((u + 1) / SA_STAGES) & 1, wctx, SB_FULL + ks);
#pragma unroll
                    for (int h = 0; h < HALVES; ++h) {
                        if (wanted(h, t)) {
                            mbar_wait(&bars[SB_P + h], static_cast<uint32_t>(done[h] & 1), wctx, SB_P + h);
                            tc_fence_after();
                            pv(h, vs, done[h] > 0 ? 1u : 0u);
                            ++done[h];
                        }
                        if (tn < t_end && wanted(h, tn)) {
                            if (done[h] == 0) mbar_wait(&bars[SB_Q + h], 0, wctx, SB_Q + h);
                            tc_fence_after();
                            qk(h, ks);
                        }
                    }
                    tc_commit(&bars[SB_EMPTY + vs]);
                    if (tn < t_end) tc_commit(&bars[SB_EMPTY + ks]);
                    u += 2;
                    t = tn;
                }
#pragma unroll
                for (int h = 0; h < HALVES; ++h) tc_commit(&bars[SB_O + h]);
            }
        } else {
            // ---------------------------------------------------------------- softmax: one row a thread
            const int h = HALVES == 2 ? warp >> 2 : 0, tid = threadIdx.x & 127;
            const Reach mine = h == 0 ? reach[0] : reach[HALVES - 1];
            const int row = q0 + h * SA_T + tid, pos = row + shift;
            const int warp_row = q0 + static_cast<int>(threadIdx.x & ~31u);
            const int pos0 = warp_row + shift, pos1 = min(warp_row + 31, p.q_len - 1) + shift;       // of the warp's first and last row
            const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
            const uint32_t t_s = t_lane + h * SA_T, t_o = t_lane + HALVES * SA_T + h * D;
            const bool changed = p.softcap > 0.f || p.slopes != nullptr || p.distance_bias != nullptr;
            const float raw_scale = p.scale * SA_LOG2E;      // of a score that nothing changes, to log2 units
            const float sc = changed ? 1.f : raw_scale;      // what is left to multiply by when the exponential is taken
            const float slope = p.slopes != nullptr ? __ldca(p.slopes + head) * SA_LOG2E : 0.f;
            const int2 warp_docs = docs != nullptr ? row_docs[warp] : make_int2(0, 0);
            const int see_lo = p.window > 0 ? pos - p.window + 1 : -0x40000000, see_hi = p.causal ? pos : p.window > 0 ? pos + p.window - 1 : 0x40000000;
            float m_ref = -INFINITY, l_sum = 0.f;
            int done = 0;
            for (int t = t_begin; t < t_end; ++t) {
                if (!wanted(h, t)) continue;
                const int k0 = t * SA_T;
                // all of the tile visible to all of the warp's rows?
                const bool full = k0 + SA_T <= k_end &&
                            (k0 + SA_T <= prefix || ((p.window == 0 || k0 >= pos1 - p.window + 1) &&
                                                     (p.causal ? k0 + SA_T - 1 <= pos0 : p.window == 0 || k0 + SA_T - 1 <= pos0 + p.window - 1)));
                bool same_doc = true, mixed = false;         // mixed: the half's rows or the tile's keys are of more than one document
                if (docs != nullptr) {
                    const int2 d = range[t];
                    same_doc = d.x == d.y && warp_docs.x == warp_docs.y && d.x == warp_docs.x;
                    mixed = d.x != d.y || mine.doc_min != mine.doc_max;
                    if (mixed) {                             // the keys' documents, 128 threads together: all warps of the half or none
                        int* stage = key_docs[h][done & 1];
                        stage[tid] = k0 + tid < k_end ? __ldca(docs + k0 + tid) : 0;
                        if (HALVES == 1 || h == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
                        else asm volatile("bar.sync 2, 128;" ::: "memory");
                    }
                }
                mbar_wait(&bars[SB_S + h], static_cast<uint32_t>(done & 1), wctx, SB_S + h);
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld32(t_s + 32 * i, s[i]);
                tc_wait_ld();
#define S_AT(c) s[(c) >> 5][(c) & 31]
                if (p.softcap > 0.f) {
                    const float to_u = p.scale / p.softcap, from_u = p.softcap * SA_LOG2E;
                    float top = 0.f;
#pragma unroll
                    for (int c = 0; c < SA_T; c += 2) top = max3f(top, fabsf(__uint_as_float(S_AT(c))), fabsf(__uint_as_float(S_AT(c + 1))));
                    const float2 to2 = pk2(to_u, to_u), from2 = pk2(from_u, from_u);
                    if (__all_sync(0xffffffffu, top * to_u <= 1.f)) {
#pragma unroll
                        for (int c = 0; c < SA_T; c += 2) {
                            const float2 y = mul2(tanh_near(mul2(pk2(__uint_as_float(S_AT(c)), __uint_as_float(S_AT(c + 1))), to2)), from2);
                            S_AT(c) = __float_as_uint(y.x);
                            S_AT(c + 1) = __float_as_uint(y.y);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < SA_T; ++c) S_AT(c) = __float_as_uint(tanh_any(__uint_as_float(S_AT(c)) * to_u) * from_u);
                    }
                } else if (changed) {
#pragma unroll
                    for (int c = 0; c < SA_T; c += 2) {
                        const float2 y = mul2(pk2(__uint_as_float(S_AT(c)), __uint_as_float(S_AT(c + 1))), pk2(raw_scale, raw_scale));
                        S_AT(c) = __float_as_uint(y.x);
                        S_AT(c + 1) = __float_as_uint(y.y);
                    }
                }
                if (p.slopes != nullptr) {
                    const float away = static_cast<float>(k0 - pos);
#pragma unroll
                    for (int c = 0; c < SA_T; ++c) S_AT(c) = __float_as_uint(fmaf(-slope, fabsf(away + static_cast<float>(c)), __uint_as_float(S_AT(c))));
                }
                if (p.distance_bias != nullptr) {
                    // distances of the warp's rows in this tile: k0 - pos1 .. k0 + 127 - pos0
                    if (k0 + SA_T - 1 - pos0 <= -p.radius || k0 - pos1 >= p.radius) {
                        const float x = table[k0 - pos1 >= p.radius ? 2 * p.radius + SA_PAD : SA_PAD];
                        const float2 x2 = pk2(x, x);
#pragma unroll
                        for (int c = 0; c < SA_T; c += 2) {
                            const float2 y = add2(pk2(__uint_as_float(S_AT(c)), __uint_as_float(S_AT(c + 1))), x2);
                            S_AT(c) = __float_as_uint(y.x);
                            S_AT(c + 1) = __float_as_uint(y.y);
                        }
                    } else {
                        // rows behind the last one read what lies next to the table's end in shared memory: kept inside it
                        const float* at = table + min(max(k0 - pos + p.radius + SA_PAD, 0), 2 * p.radius + 2 * SA_PAD - SA_T + 1);
#pragma unroll
                        for (int c = 0; c < SA_T; ++c) S_AT(c) = __float_as_uint(__uint_as_float(S_AT(c)) + at[c]);
                    }
                }
                if (!full) {
                    const int from = see_lo - k0, to = see_hi - k0, front = prefix - k0, end = k_end - k0;
#pragma unroll
                    for (int c = 0; c < SA_T; ++c)
                        if (!(((c >= from && c <= to) || c < front) && c < end)) S_AT(c) = 0xFF800000u;
                }
                if (mixed && !same_doc) {
                    const int* stage = key_docs[h][done & 1];
#pragma unroll
                    for (int c = 0; c < SA_T; c += 4) {
                        const int4 k = *reinterpret_cast<const int4*>(stage + c);
                        if (k.x != my_doc) S_AT(c) = 0xFF800000u;
                        if (k.y != my_doc) S_AT(c + 1) = 0xFF800000u;
                        if (k.z != my_doc) S_AT(c + 2) = 0xFF800000u;
                        if (k.w != my_doc) S_AT(c + 3) = 0xFF800000u;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < SA_T; c += 8)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx[i] = max3f(mx[i], __uint_as_float(S_AT(c + 2 * i)), __uint_as_float(S_AT(c + 2 * i + 1)));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
                const bool need = top > m_ref + SA_RESCALE || (m_ref == -INFINITY && top > -INFINITY);
                if (__any_sync(0xffffffffu, need)) {
                    float alpha = 1.f;
                    if (need) {
                        // a whole number, for the polynomial exponential
                        const float now = fminf(fmaxf(ceilf(top), -2097152.0f), 2097152.0f);
                        alpha = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - now);
                        m_ref = now;
                        l_sum *= alpha;
                    }
                    // S is there, so the products that the issuer put before it have landed in O, too
                    if (done > 0) rescale_o<D>(t_o, alpha);
                }
                const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
                const float2 sc2 = pk2(sc, sc), negm2 = pk2(neg_m, neg_m), mm2 = pk2(12582912.0f + neg_m, 12582912.0f + neg_m);
                const float lo = (-120.0f - neg_m) / sc;
                float2 sum_a = pk2(0.f, 0.f), sum_b = pk2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < SA_T / 2; ++i) {
                    const float s0 = __uint_as_float(S_AT(2 * i)), s1 = __uint_as_float(S_AT(2 * i + 1));
                    float e0, e1;
                    if (((i * SA_POLY_PAIRS) & 7) < SA_POLY_PAIRS) {
                        exp2_poly_pair(s0, s1, lo, sc2, mm2, e0, e1);
                    } else {
                        const float2 x = fma2(pk2(s0, s1), sc2, negm2);
                        e0 = fast_exp2(x.x);
                        e1 = fast_exp2(x.y);
                    }
                    if (i & 1) sum_b = add2(sum_b, pk2(e0, e1));
                    else sum_a = add2(sum_a, pk2(e0, e1));
                    S_AT(i) = pack_pair<BF16>(e0, e1);       // the scores of pair i were used above
                }
                const float2 sum = add2(sum_a, sum_b);
                l_sum += sum.x + sum.y;
                tmem_st32(t_s, s[0]);
                tmem_st32(t_s + 32, s[1]);
#undef S_AT
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[SB_P + h]);
                ++done;
            }
            // ---------------------------------------------------------------- O / l
            if (done > 0) {
                mbar_wait(&bars[SB_O + h], 0, wctx, SB_O + h);
                tc_fence_after();
            }
            // a row that saw nothing has no maximum; where all it saw is NaN its sum says so
            const bool any = done > 0 && (m_ref > -INFINITY || l_sum != l_sum);
            const float inv = any ? 1.f / l_sum : 0.f;
            uint16_t* dst = static_cast<uint16_t*>(p.out) + b * p.out_stride[0] + head * p.out_stride[1] + static_cast<long long>(row) * p.out_stride[2];
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                if (done > 0) {
                    tmem_ld32(t_o + c, o);
                    tc_wait_ld();
                }
                if (row < p.q_len) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        auto two = [&](int j) { return any ? pack_pair<BF16>(__uint_as_float(o[i + j]) * inv, __uint_as_float(o[i + j + 1]) * inv) : 0u; };
                        *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(two(0), two(2), two(4), two(6));
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

// A 4-D map of (batch, heads, rows, dim) with boxes of 128 rows x 64 columns; the outer dimensions in the order of their strides
int make_map(CUtensorMap* map, const void* base, int batch, int heads, int rows, int dim, const long long st[3], int* slot_s, int* slot_h, int* slot_b) {
    struct Dim { uint64_t size; long long stride; int logical; } d[3] = {
        {static_cast<uint64_t>(rows), st[2], 0}, {static_cast<uint64_t>(heads), st[1], 1}, {static_cast<uint64_t>(batch), st[0], 2}};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (d[j].stride < d[i].stride) { Dim t = d[i]; d[i] = d[j]; d[j] = t; }
    uint64_t dims[4] = {static_cast<uint64_t>(dim), 0, 0, 0}, strides[3];
    uint32_t box[4] = {64, 1, 1, 1};
    for (int i = 0; i < 3; ++i) {
        dims[i + 1] = d[i].size;
        strides[i] = static_cast<uint64_t>(d[i].stride) * 2;
        if (d[i].logical == 0) { box[i + 1] = SA_T; *slot_s = i + 1; }
        if (d[i].logical == 1) *slot_h = i + 1;
        if (d[i].logical == 2) *slot_b = i + 1;
    }
    return make_tensor_map_f16(map, base, 4, dims, strides, box);        // (bf16 moves as fp16 does: 16 bits)
}

}  // namespace
}  // namespace stof

using namespace stof;

extern "C" int stof_scored_attn(const void* q, const void* k, const void* v, void* out, int dtype, int batch, int heads, int kv_heads, int q_len, int k_len,
                                int head_dim, const long long q_strides[3], const long long k_strides[3], const long long v_strides[3],
                                const long long out_strides[3], const stof_score_rules* rules, int* status_dev, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    STOF_REQUIRE(batch >= 0 && heads > 0 && kv_heads > 0 && q_len >= 0 && k_len >= 0, "scored_attn: bad shape");
    STOF_REQUIRE(heads % kv_heads == 0, "scored_attn: %d heads are not a multiple of %d K/V heads", heads, kv_heads);
    STOF_REQUIRE(head_dim == 64 || head_dim == 128, "scored_attn: head_dim %d not in {64, 128}", head_dim);
    STOF_REQUIRE(dtype == STOF_DTYPE_F16 || dtype == STOF_DTYPE_BF16, "scored_attn: fp16 or bf16 expected");
    STOF_REQUIRE(static_cast<long long>(q_len) + k_len < (1ll << 29), "scored_attn: %d queries and %d keys are beyond 2^29", q_len, k_len);
    STOF_REQUIRE(rules != nullptr, "scored_attn: null rules");
    STOF_REQUIRE(rules->softmax_scale > 0.f && rules->softmax_scale < INFINITY, "scored_attn: softmax_scale must be positive and finite");
    STOF_REQUIRE(rules->softcap >= 0.f && rules->softcap < INFINITY, "scored_attn: softcap must not be negative");
    STOF_REQUIRE(rules->window >= 0, "scored_attn: window must not be negative");
    STOF_REQUIRE(rules->distance_bias == nullptr || (rules->bias_radius >= 0 && rules->bias_radius <= STOF_SCORED_MAX_RADIUS), "scored_attn: bias radius %d beyond %d",
                 rules->bias_radius, STOF_SCORED_MAX_RADIUS);
    STOF_REQUIRE(rules->prefix_lens == nullptr || rules->causal, "scored_attn: a prefix makes keys visible that a causal mask hides: it needs causal");
    if (rules->documents != nullptr) {
        STOF_REQUIRE(q_len <= k_len, "scored_attn: documents name keys: %d queries need as many keys, got %d", q_len, k_len);
        STOF_REQUIRE(rules->documents_stride >= k_len || batch <= 1, "scored_attn: row stride of documents below the number of keys");
        if (k_len > STOF_SCORED_MAX_DOC_KEYS) {
            set_error("scored_attn: documents over %d keys, beyond the maximum of %d", k_len, STOF_SCORED_MAX_DOC_KEYS);
            return STOF_E_LIMIT;
        }
    }
    if (batch == 0 || q_len == 0) return STOF_OK;
    STOF_REQUIRE(k_len > 0, "scored_attn: no keys");
    STOF_REQUIRE(q && k && v && out && q_strides && k_strides && v_strides && out_strides, "scored_attn: null pointer");
    STOF_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), "scored_attn: pointers must be 16-byte aligned");
    for (const long long* st : {q_strides, k_strides, v_strides, out_strides})
        for (int i = 0; i < 3; ++i) STOF_REQUIRE(st[i] > 0 && st[i] % 8 == 0, "scored_attn: strides must be positive multiples of 8 elements");
    ScoredParams p;
    p.out = out;
    for (int i = 0; i < 3; ++i) p.out_stride[i] = out_strides[i];
    p.slopes = rules->slopes; p.distance_bias = rules->distance_bias; p.documents = rules->documents; p.prefix_lens = rules->prefix_lens;
    p.key_lens = rules->key_lens; p.documents_stride = rules->documents_stride; p.status = status_dev;
    p.scale = rules->softmax_scale; p.softcap = rules->softcap; p.causal = rules->causal != 0; p.radius = rules->bias_radius;
    p.window = rules->window > q_len + k_len ? q_len + k_len : rules->window;
    p.batch = batch; p.heads = heads; p.group = heads / kv_heads; p.q_len = q_len; p.k_len = k_len;
    p.table_bytes = rules->distance_bias != nullptr ? (2 * p.radius + 1 + 2 * SA_PAD) * 4 + 4 : 0;       // (an even number of words: pairs follow)
    p.range_bytes = rules->documents != nullptr ? (k_len + SA_T - 1) / SA_T * 8 : 0;
    CUtensorMap mq, mk, mv;
    if (int rc = make_map(&mq, q, batch, heads, q_len, head_dim, q_strides, &p.slot_s[0], &p.slot_h[0], &p.slot_b[0])) return rc;
    if (int rc = make_map(&mk, k, batch, kv_heads, k_len, head_dim, k_strides, &p.slot_s[1], &p.slot_h[1], &p.slot_b[1])) return rc;
    if (int rc = make_map(&mv, v, batch, kv_heads, k_len, head_dim, v_strides, &p.slot_s[2], &p.slot_h[2], &p.slot_b[2])) return rc;
    // two halves to a block where that leaves a block for every multiprocessor
    const long long pairs = static_cast<long long>(batch) * heads;
    const int halves = pairs * ((q_len + 2 * SA_T - 1) / (2 * SA_T)) >= sm_count() ? 2 : 1;
    p.q_tiles = (q_len + halves * SA_T - 1) / (halves * SA_T);
    STOF_REQUIRE(pairs * p.q_tiles < (1ll << 31), "scored_attn: batch * heads * query tiles beyond 2^31");
    const size_t smem = 1024 + static_cast<size_t>(halves + SA_STAGES) * SA_T * head_dim * 2 + p.table_bytes + p.range_bytes;
    auto launch = [&](auto kernel) -> int {
        STOF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
        LaunchConfig lc(dim3(static_cast<unsigned>(pairs * p.q_tiles)), halves * 128 + 64, smem, stream);
        STOF_CUDA(cudaLaunchKernelEx(&lc.cfg, kernel, mq, mk, mv, p));
        return STOF_OK;
    };
    const bool bf16 = dtype == STOF_DTYPE_BF16;
    if (head_dim == 64) {
        if (halves == 2) return bf16 ? launch(scored_attn_kernel<64, 2, true>) : launch(scored_attn_kernel<64, 2, false>);
        return bf16 ? launch(scored_attn_kernel<64, 1, true>) : launch(scored_attn_kernel<64, 1, false>);
    }
    if (halves == 2) return bf16 ? launch(scored_attn_kernel<128, 2, true>) : launch(scored_attn_kernel<128, 2, false>);
    return bf16 ? launch(scored_attn_kernel<128, 1, true>) : launch(scored_attn_kernel<128, 1, false>);
}
