// Attention of a few query tokens per request over a paged 8-bit key/value cache (HBM-bound: every entry is read once).
//
// The query rows that share a K/V head (heads / kv_heads heads of each token) are the columns of both products, in tiles of 8:
//   S^T (16 keys x 8 rows) = K (16 keys x D) Q^T       O^T (D x 8 rows) += V^T (D x 16 keys) P^T
// on mma.sync m16n8k16.  A tcgen05 product has at least 64 rows of which a decoding step fills one to eight, and takes its operands
// from shared memory as 8 or 16 bits; here the entries go from global memory to registers, become fp16 there (exactly) and are
// multiplied, with no shared memory in between.  The scales stay out of the products: K's goes into the score, V's into P,
// relative to a reference that the accumulator carries (so that P keeps fp16's precision whatever the scales are).
//
// Which lane holds which entry is free as long as both operands agree, so that every load is 16 bytes of a row: with g = lane / 4,
// c = lane % 4, a lane reads chunk c (and c + 4) of the rows of keys g and g + 8 for S, and chunk g of the rows of keys 2c, 2c + 1,
// 2c + 8, 2c + 9 for O.  P leaves the first product with keys along g and is wanted with rows along g: one 8 x 8 transpose.
//
// Work is counted in units of 64 keys (16 for each of a block's four warps) over all requests and K/V heads; every block takes an
// equal stretch of that line, whatever the lengths.  A (request, head) that one block covers is written at once, the others in parts
// that cache_attn_join_kernel adds in the order of the blocks.
#include "cache_common.cuh"
#include "stof_host.h"
#include "stof_ptx.cuh"

namespace stof {
namespace {

constexpr int CT_WARPS = 4, CT_THREADS = CT_WARPS * 32;
constexpr int CT_UNIT = 16 * CT_WARPS;       // keys of a unit
constexpr float LOG2E = 1.4426950408889634f;

struct CacheAttnParams {
    const void* q;
    void* out;
    long long q_stride[3], out_stride[3];    // request, token, head
    const void *k_pages, *v_pages;
    const float *k_scales, *v_scales;
    const int* block_table;
    long long table_stride;
    const int* lengths;
    const float *slopes, *distance_bias;
    float* workspace;
    int* status;
    float scale, softcap;
    int window, radius;
    int requests, tokens, heads, kv_heads, group;            // group = heads / kv_heads
    int rows, row_groups;                                    // query rows of a K/V head, and how many blocks of them
    int table_width, page_count, page_shift;
    int bf16;
};

// keys [first, first + 64 * units) cover what the request's tokens see
struct Span { int length, first, units; };
__device__ __forceinline__ Span span_of(const CacheAttnParams& p, int b) {
    const long long most = static_cast<long long>(p.table_width) << p.page_shift;
    const int length = static_cast<int>(min(static_cast<long long>(max(p.lengths[b], 0)), most));
    int first = 0;
    if (p.window > 0) first = max(length - p.tokens - p.window + 1, 0) & ~(CT_UNIT - 1);
    return {length, first, (length - first + CT_UNIT - 1) / CT_UNIT};
}

__device__ __forceinline__ long long block_sum(long long v, long long* shared) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    long long s = 0;
#pragma unroll
    for (int i = 0; i < CT_WARPS; ++i) s += shared[i];
    return s;
}

// blocks that get a stretch of the line: each at least a unit
__device__ __forceinline__ int blocks_at_work(long long total, int blocks) { return static_cast<int>(min(total, static_cast<long long>(blocks))); }
// where block i's stretch of the line begins
__device__ __forceinline__ long long stretch(long long total, int i, int blocks) { return total * i / blocks; }

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// what a lane loads of 16 keys
template <int D>
struct Tile {
    uint4 k[2][D / 64];                      // keys g, g + 8
    uint4 v[4];                              // keys 2c, 2c + 1, 2c + 8, 2c + 9 (D = 64: the first half)
    float k_scale, v_scale;
    int key;                                 // first key; -1: no page, nothing loaded
};

template <int NT, int D, bool E4M3>
__global__ void __launch_bounds__(CT_THREADS, NT == 1 ? 4 : 3) cache_attn_kernel(const CacheAttnParams p) {
    constexpr int CH = D / 64, KS = D / 16, MT = D / 16, ROWS = NT * 8;
    constexpr int V_BYTES = D / 8;           // of a row, per lane
    __shared__ long long sums[CT_WARPS];
    __shared__ long long found_base;
    __shared__ int found_request;
    __shared__ float merge_m[CT_WARPS][ROWS], merge_l[CT_WARPS][ROWS];
    __shared__ __align__(16) float merge_o[ROWS][D + 4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    grid_dependency_wait();
    grid_launch_dependents();
    if (__syncthreads_or(failure_reported(p.status))) return;
    const int pairs = p.kv_heads * p.row_groups;             // of a request
    long long total = 0;
    for (int b = threadIdx.x; b < p.requests; b += CT_THREADS) total += span_of(p, b).units;
    total = block_sum(total, sums) * pairs;
    const int blocks = blocks_at_work(total, gridDim.x);
    if (static_cast<int>(blockIdx.x) >= blocks) return;
    long long at = stretch(total, blockIdx.x, blocks);
    const long long end = stretch(total, blockIdx.x + 1, blocks);
    // the request in which the stretch begins
    long long base = 0;
    for (int b0 = 0; b0 < p.requests; b0 += CT_THREADS) {
        const int b = b0 + static_cast<int>(threadIdx.x);
        long long mine = b < p.requests ? static_cast<long long>(span_of(p, b).units) * pairs : 0, upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        long long all = 0;
        for (int i = 0; i < CT_WARPS; ++i) {
            if (i < warp) upto += sums[i];
            all += sums[i];
        }
        if (at >= base + upto - mine && at < base + upto) {
            found_request = b;
            found_base = base + upto - mine;
        }
        base += all;
        if (at < base) break;
    }
    __syncthreads();
    int b = found_request;
    base = found_base;

    while (at < end) {
        const Span span = span_of(p, b);
        const long long behind = base + static_cast<long long>(span.units) * pairs;
        if (at >= behind) {                                  // (requests of length 0 are passed over here)
            base = behind;
            ++b;
            continue;
        }
        const int pair = static_cast<int>((at - base) / span.units), u0 = static_cast<int>((at - base) % span.units);
        const int u1 = static_cast<int>(min(static_cast<long long>(span.units), u0 + (end - at)));
        const int kv = pair / p.row_groups, row0 = (pair % p.row_groups) * ROWS;

        // ---- the query rows: fp16, each row times a power of two (bf16 has more range than fp16; fp16 rows are taken as they are)
        uint32_t qf[NT][KS][2];
        float row_scale[NT][2], slope[NT][2];
        const float* table[NT][2];
        int pos[NT][2];                                      // of the lane's rows 2c and 2c + 1; nothing is visible from -1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = row0 + nt * 8 + g;
            float shrink = 1.f;
            if (r < p.rows) {
                const uint16_t* src = static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] + (r / p.group) * p.q_stride[1] +
                                      (kv * p.group + r % p.group) * p.q_stride[2];
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const uint4 x = __ldca(reinterpret_cast<const uint4*>(src + (c + 4 * i) * 16)), y = __ldca(reinterpret_cast<const uint4*>(src + (c + 4 * i) * 16 + 8));
                    qf[nt][4 * i][0] = x.x; qf[nt][4 * i][1] = x.y; qf[nt][4 * i + 1][0] = x.z; qf[nt][4 * i + 1][1] = x.w;
                    qf[nt][4 * i + 2][0] = y.x; qf[nt][4 * i + 2][1] = y.y; qf[nt][4 * i + 3][0] = y.z; qf[nt][4 * i + 3][1] = y.w;
                }
                if (p.bf16) {
#pragma unroll
                    for (int s = 0; s < KS; ++s)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float2 f = unpack_pair<true>(qf[nt][s][h]);
                            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                        }
                }
                shrink = top;
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) qf[nt][s][0] = qf[nt][s][1] = 0u;
            }
            if (p.bf16) {
                shrink = fmaxf(shrink, __shfl_xor_sync(0xffffffffu, shrink, 1));
                shrink = fmaxf(shrink, __shfl_xor_sync(0xffffffffu, shrink, 2));
                // 2^(14 - exponent of the largest), inside fp32's range: the largest becomes 2^14 .. 2^15
                const int e = static_cast<int>((__float_as_uint(shrink) >> 23) & 255u) - 127;
                shrink = (r < p.rows && shrink > 0.f) ? __uint_as_float(static_cast<uint32_t>(127 + min(max(14 - e, -126), 126)) << 23) : 1.f;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 f = unpack_pair<true>(qf[nt][s][h]);
                        qf[nt][s][h] = pack_half2(f.x * shrink, f.y * shrink);
                    }
            } else {
                shrink = 1.f;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float f = __shfl_sync(0xffffffffu, shrink, (2 * c + e) * 4);
                const int rr = row0 + nt * 8 + 2 * c + e, head = kv * p.group + rr % p.group;
                const bool on = rr < p.rows;
                row_scale[nt][e] = p.scale / f;
                pos[nt][e] = on ? span.length - p.tokens + rr / p.group : -1;
                slope[nt][e] = on && p.slopes != nullptr ? p.slopes[head] : 0.f;
                table[nt][e] = on && p.distance_bias != nullptr ? p.distance_bias + static_cast<size_t>(head) * (2 * p.radius + 1) + p.radius : p.distance_bias;
            }
        }

        float o[NT][MT][4], m[NT][2], l[NT][2], v_ref = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][mt][e] = 0.f;
        }

        const int* pages = p.block_table + b * p.table_stride;
        auto page_of = [&](int u) {                          // of this warp's keys in unit u; -1 behind the last key
            const int key = span.first + u * CT_UNIT + warp * 16;
            return u < u1 && key < span.length ? pages[key >> p.page_shift] : -1;
        };
        auto load = [&](Tile<D>& t, int u, int page) {
            const int key = span.first + u * CT_UNIT + warp * 16;
            t.key = -1;
            if (u >= u1 || key >= span.length) return;
            if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.page_count)) {
                if (lane == 0 && p.status != nullptr) atomicCAS(p.status, 0, STATUS_BAD_INDEX);
                return;
            }
            t.key = key;
            const size_t slot = static_cast<size_t>(page) * p.kv_heads + kv;
            t.k_scale = __ldca(p.k_scales + slot);
            t.v_scale = __ldca(p.v_scales + slot);
            const size_t row = (slot << p.page_shift) + (key & ((1 << p.page_shift) - 1));
            const char *kp = static_cast<const char*>(p.k_pages) + row * D, *vp = static_cast<const char*>(p.v_pages) + row * D;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < CH; ++i) t.k[h][i] = __ldcs(reinterpret_cast<const uint4*>(kp + (g + 8 * h) * D + (c + 4 * i) * 16));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const char* src = vp + (2 * c + (j & 1) + 8 * (j >> 1)) * D + g * V_BYTES;
                if constexpr (D == 128) {
                    t.v[j] = __ldcs(reinterpret_cast<const uint4*>(src));
                } else {
                    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(src));
                    t.v[j].x = w.x;
                    t.v[j].y = w.y;
                }
            }
        };
        auto word = [](const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; };
        auto compute = [&](Tile<D>& t) {
            if (t.key < 0) return;
            const int left = span.length - t.key;            // keys of the tile that exist; what lies behind them may be anything
            if (left < 16) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (2 * c + (j & 1) + 8 * (j >> 1) >= left) t.v[j] = make_uint4(0u, 0u, 0u, 0u);
            }
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t x = word(t.k[0][i], w), y = word(t.k[1][i], w);
                    const uint32_t a0 = entries_to_half2<E4M3>(x), a2 = entries_to_half2<E4M3>(x >> 16);
                    const uint32_t a1 = entries_to_half2<E4M3>(y), a3 = entries_to_half2<E4M3>(y >> 16);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(s[nt], a0, a1, a2, a3, qf[nt][4 * i + w][0], qf[nt][4 * i + w][1]);
                }
            // scores in units of log2; element e: key g + 8 * (e / 2), row 2c + e % 2
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = s[nt][e] * (t.k_scale * row_scale[nt][e & 1]);
                    if (p.softcap > 0.f) {
                        // tanh(y) = 1 - 2 / (1 + e^(2y))
                        const float ex = fast_exp2(x * (2.f * LOG2E / p.softcap));
                        x = p.softcap - 2.f * p.softcap * __frcp_rn(1.f + ex);
                    }
                    const int away = t.key + g + 8 * (e >> 1) - pos[nt][e & 1];      // at most 0 where visible
                    x += slope[nt][e & 1] * static_cast<float>(away);
                    const bool on = pos[nt][e & 1] >= 0 && away <= 0 && (p.window == 0 || away > -p.window);
                    if (p.distance_bias != nullptr && on) x += __ldca(table[nt][e & 1] + max(away, -p.radius));
                    s[nt][e] = on ? x * LOG2E : -INFINITY;
                }
            // V's scale against the reference that o is held in
            if (t.v_scale > v_ref * 256.f || v_ref == 0.f) {
                const float f = t.v_scale > 0.f ? v_ref / t.v_scale : 1.f;
                v_ref = t.v_scale > 0.f ? t.v_scale : v_ref;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[nt][mt][e] *= f;
            }
            const float v_rel = v_ref > 0.f ? t.v_scale / v_ref : t.v_scale;
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float top0 = fmaxf(s[nt][0], s[nt][2]), top1 = fmaxf(s[nt][1], s[nt][3]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, d));
                    top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, d));
                }
                if (__any_sync(0xffffffffu, top0 > m[nt][0] || top1 > m[nt][1])) {
                    const float n0 = fmaxf(m[nt][0], top0), n1 = fmaxf(m[nt][1], top1);
                    const float a0 = n0 == m[nt][0] ? 1.f : fast_exp2(m[nt][0] - n0), a1 = n1 == m[nt][1] ? 1.f : fast_exp2(m[nt][1] - n1);
                    m[nt][0] = n0;
                    m[nt][1] = n1;
                    l[nt][0] *= a0;
                    l[nt][1] *= a1;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        o[nt][mt][0] *= a0;
                        o[nt][mt][1] *= a1;
                        o[nt][mt][2] *= a0;
                        o[nt][mt][3] *= a1;
                    }
                }
                const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
                const float p0 = fast_exp2(s[nt][0] - m0), p1 = fast_exp2(s[nt][1] - m1), p2 = fast_exp2(s[nt][2] - m0), p3 = fast_exp2(s[nt][3] - m1);
                l[nt][0] += p0 + p2;
                l[nt][1] += p1 + p3;
                // to fp16 for the product, as the other attention kernels do; the sum is of the values before rounding
                pf[nt][0] = transpose8x8(pack_half2(p0 * v_rel, p1 * v_rel));
                pf[nt][1] = transpose8x8(pack_half2(p2 * v_rel, p3 * v_rel));
            }
#pragma unroll
            for (int w = 0; w < V_BYTES / 4; ++w) {
                const uint32_t x0 = word(t.v[0], w), x1 = word(t.v[1], w), y0 = word(t.v[2], w), y1 = word(t.v[3], w);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t x = __byte_perm(x0, x1, h == 0 ? 0x5140 : 0x7362), y = __byte_perm(y0, y1, h == 0 ? 0x5140 : 0x7362);
                    const uint32_t a0 = entries_to_half2<E4M3>(x), a1 = entries_to_half2<E4M3>(x >> 16);
                    const uint32_t a2 = entries_to_half2<E4M3>(y), a3 = entries_to_half2<E4M3>(y >> 16);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][2 * w + h], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
                }
            }
        };
        // two tiles in flight: one is loaded while the other is used; a page's number is asked for a unit earlier still
        Tile<D> t0, t1;
        int page0 = page_of(u0), page1 = page_of(u0 + 1);
        load(t0, u0, page0);
        for (int u = u0; u < u1; u += 2) {
            page0 = page_of(u + 2);
            load(t1, u + 1, page1);
            compute(t0);
            page1 = page_of(u + 3);
            load(t0, u + 2, page0);
            compute(t1);
        }

        // ---- the four warps' results are added in smem, in their order
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
                if (g == 0) {
                    merge_m[warp][nt * 8 + 2 * c + e] = m[nt][e];
                    merge_l[warp][nt * 8 + 2 * c + e] = l[nt][e];
                }
            }
        __syncthreads();
        float weight[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = nt * 8 + 2 * c + e;
                float top = merge_m[0][r];
#pragma unroll
                for (int w = 1; w < CT_WARPS; ++w) top = fmaxf(top, merge_m[w][r]);
                // a row without a maximum saw nothing (sum 0) or only NaN (sum NaN, which has to come out)
                weight[nt][e] = m[nt][e] == -INFINITY ? l[nt][e] : fast_exp2(m[nt][e] - top) * v_ref;
            }
        for (int w = 0; w < CT_WARPS; ++w) {
            if (warp == w) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float* dst = &merge_o[nt * 8 + 2 * c + e][g * 2 * MT];
#pragma unroll
                        for (int i = 0; i < 2 * MT; i += 4) {
                            // d = g * 2 MT + i: m-tile i / 2, first row or second
                            float4 x = make_float4(o[nt][i / 2][e], o[nt][i / 2][2 + e], o[nt][i / 2 + 1][e], o[nt][i / 2 + 1][2 + e]);
                            const float f = weight[nt][e];
                            x = f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
                            if (w > 0) {
                                const float4 y = *reinterpret_cast<const float4*>(dst + i);
                                x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
                            }
                            *reinterpret_cast<float4*>(dst + i) = x;
                        }
                    }
            }
            __syncthreads();
        }
        const bool whole = u0 == 0 && u1 == span.units;
        float* part = p.workspace + (static_cast<size_t>(blockIdx.x) * 2 + (u0 == 0 ? 1 : 0)) * (ROWS * (D + 2));
        for (int i = threadIdx.x; i < ROWS * (D / 8); i += CT_THREADS) {
            const int r = i / (D / 8), d = i % (D / 8) * 8;
            if (row0 + r >= p.rows) continue;
            float top = merge_m[0][r];
            for (int w = 1; w < CT_WARPS; ++w) top = fmaxf(top, merge_m[w][r]);
            float sum = 0.f;
            for (int w = 0; w < CT_WARPS; ++w)
                sum += merge_m[w][r] > -INFINITY ? merge_l[w][r] * fast_exp2(merge_m[w][r] - top) : merge_l[w][r];
            const float4 x = *reinterpret_cast<const float4*>(&merge_o[r][d]), y = *reinterpret_cast<const float4*>(&merge_o[r][d + 4]);
            if (whole) {
                const float inv = sum != 0.f ? 1.f / sum : 0.f;
                uint4 u;
                if (p.bf16) u = make_uint4(pack_pair<true>(x.x * inv, x.y * inv), pack_pair<true>(x.z * inv, x.w * inv), pack_pair<true>(y.x * inv, y.y * inv), pack_pair<true>(y.z * inv, y.w * inv));
                else u = make_uint4(pack_pair<false>(x.x * inv, x.y * inv), pack_pair<false>(x.z * inv, x.w * inv), pack_pair<false>(y.x * inv, y.y * inv), pack_pair<false>(y.z * inv, y.w * inv));
                uint16_t* dst = static_cast<uint16_t*>(p.out) + b * p.out_stride[0] + ((row0 + r) / p.group) * p.out_stride[1] + (kv * p.group + (row0 + r) % p.group) * p.out_stride[2];
                *reinterpret_cast<uint4*>(dst + d) = u;
            } else {
                float* dst = part + 2 * ROWS + r * D + d;
                *reinterpret_cast<float4*>(dst) = x;
                *reinterpret_cast<float4*>(dst + 4) = y;
                if (d == 0) {
                    part[r] = top;
                    part[ROWS + r] = sum;
                }
            }
        }
        __syncthreads();                                     // smem is free again
        at += u1 - u0;
    }
}

// Adds the parts of the (request, K/V head, row group)s that more than one block worked on, and writes the zeros of empty requests.
template <int NT, int D>
__global__ void __launch_bounds__(CT_THREADS) cache_attn_join_kernel(const CacheAttnParams p, int launched) {
    constexpr int ROWS = NT * 8, EACH = D / 32;
    __shared__ long long sums[CT_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dependency_wait();
    grid_launch_dependents();
    if (__syncthreads_or(failure_reported(p.status))) return;
    const int pairs = p.kv_heads * p.row_groups;
    const int b = blockIdx.x / pairs, pair = blockIdx.x % pairs, kv = pair / p.row_groups, row0 = (pair % p.row_groups) * ROWS;
    long long total = 0, base = 0;
    for (int i = threadIdx.x; i < p.requests; i += CT_THREADS) {
        const int units = span_of(p, i).units;
        total += units;
        if (i < b) base += units;
    }
    total = block_sum(total, sums) * pairs;
    base = block_sum(base, sums) * pairs;
    const int blocks = blocks_at_work(total, launched);
    const int units = span_of(p, b).units;
    const long long from = base + static_cast<long long>(pair) * units, to = from + units;
    // blocks whose stretch meets [from, to)
    int i0 = 0, i1 = 0;
    if (units > 0) {
        i0 = static_cast<int>(from * blocks / total);
        while (i0 > 0 && stretch(total, i0, blocks) > from) --i0;
        while (stretch(total, i0 + 1, blocks) <= from) ++i0;
        i1 = i0 + 1;
        while (i1 < blocks && stretch(total, i1, blocks) < to) ++i1;
        if (i1 == i0 + 1) return;                            // one block had all of it
    }
    for (int r = warp; r < ROWS && row0 + r < p.rows; r += CT_WARPS) {
        auto part = [&](int i) { return p.workspace + (static_cast<size_t>(i) * 2 + (stretch(total, i, blocks) <= from ? 1 : 0)) * (ROWS * (D + 2)); };
        float top = -INFINITY, sum = 0.f, o[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) o[e] = 0.f;
        for (int i = i0 + lane; i < i1; i += 32) top = fmaxf(top, __ldca(part(i) + r));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        for (int i = i0; i < i1; ++i) {
            const float* x = part(i);
            const float m = __ldca(x + r), f = m > -INFINITY ? fast_exp2(m - top) : 1.f;
            sum += __ldca(x + ROWS + r) * f;
#pragma unroll
            for (int e = 0; e < EACH; ++e) o[e] += f * __ldca(x + 2 * ROWS + r * D + lane * EACH + e);
        }
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + b * p.out_stride[0] + ((row0 + r) / p.group) * p.out_stride[1] + (kv * p.group + (row0 + r) % p.group) * p.out_stride[2] + lane * EACH;
#pragma unroll
        for (int e = 0; e < EACH; e += 2) {
            const float x = o[e] * inv, y = o[e + 1] * inv;
            *reinterpret_cast<uint32_t*>(dst + e) = p.bf16 ? pack_pair<true>(x, y) : pack_pair<false>(x, y);
        }
    }
}

struct Shape {
    int rows, nt, row_groups;
    long long blocks;
};
// row tiles of 8: one up to 8 rows, else two at a time; blocks: what the GPU holds at once, no more than there can be units
Shape shape_of(int requests, int tokens, int heads, int kv_heads, int page_size, int table_width) {
    Shape s;
    s.rows = tokens * (heads / kv_heads);
    s.nt = s.rows <= 8 ? 1 : 2;
    s.row_groups = (s.rows + 8 * s.nt - 1) / (8 * s.nt);
    const long long units = static_cast<long long>(requests) * kv_heads * s.row_groups * ((static_cast<long long>(table_width) * page_size + CT_UNIT - 1) / CT_UNIT);
    s.blocks = static_cast<long long>(sm_count()) * (s.nt == 1 ? 4 : 3);
    if (s.blocks > units) s.blocks = units > 0 ? units : 1;
    return s;
}

}  // namespace
}  // namespace stof

using namespace stof;

extern "C" size_t stof_cache_attn_workspace_bytes(int requests, int tokens, int heads, int kv_heads, int head_dim, int page_size, int table_width) {
    if (requests <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || page_size <= 0 || table_width < 0) return 0;
    const Shape s = shape_of(requests, tokens, heads, kv_heads, page_size, table_width);
    return static_cast<size_t>(s.blocks) * 2 * (8 * s.nt) * (static_cast<size_t>(head_dim) + 2) * sizeof(float);
}

extern "C" int stof_cache_attn(const void* q, void* out, int dtype, const long long q_strides[3], const long long out_strides[3], const void* k_pages,
                               const void* v_pages, const float* k_scales, const float* v_scales, int cache_dtype, int pages, int page_size, int kv_heads,
                               int head_dim, const int* block_table, long long table_stride, int table_width, const int* lengths, int requests, int tokens,
                               int heads, const stof_score_rules* rules, void* workspace, size_t workspace_bytes, int* status_dev, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    STOF_REQUIRE(requests >= 0 && tokens >= 0 && heads > 0 && kv_heads > 0 && pages >= 0 && table_width >= 0, "cache_attn: bad shape");
    STOF_REQUIRE(heads % kv_heads == 0, "cache_attn: %d heads are not a multiple of %d K/V heads", heads, kv_heads);
    STOF_REQUIRE(head_dim == 64 || head_dim == 128, "cache_attn: head_dim %d not in {64, 128}", head_dim);
    STOF_REQUIRE(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128, "cache_attn: page size %d not in {16, 32, 64, 128}", page_size);
    STOF_REQUIRE(cache_dtype == STOF_DTYPE_INT8 || cache_dtype == STOF_DTYPE_E4M3, "cache_attn: cache entries must be int8 or e4m3");
    STOF_REQUIRE(dtype == STOF_DTYPE_F16 || dtype == STOF_DTYPE_BF16, "cache_attn: queries must be fp16 or bf16");
    STOF_REQUIRE(static_cast<long long>(table_width) * page_size < (1ll << 31) - 256, "cache_attn: a row of the block table spans more than 2^31 tokens");
    STOF_REQUIRE(rules != nullptr, "cache_attn: null rules");
    STOF_REQUIRE(rules->softmax_scale > 0.f && rules->softmax_scale < INFINITY, "cache_attn: softmax_scale must be positive and finite");
    STOF_REQUIRE(rules->softcap >= 0.f && rules->softcap < INFINITY, "cache_attn: softcap must not be negative");
    STOF_REQUIRE(rules->window >= 0, "cache_attn: window must not be negative");
    STOF_REQUIRE(rules->distance_bias == nullptr || (rules->bias_radius >= 0 && rules->bias_radius <= STOF_SCORED_MAX_RADIUS), "cache_attn: bias radius %d beyond %d",
                 rules->bias_radius, STOF_SCORED_MAX_RADIUS);
    if (requests == 0 || tokens == 0) return STOF_OK;
    STOF_REQUIRE(q && out && k_scales && v_scales && lengths && q_strides && out_strides, "cache_attn: null pointer");
    STOF_REQUIRE((k_pages && v_pages) || pages == 0, "cache_attn: null pages");
    STOF_REQUIRE(table_width == 0 || (block_table && table_stride >= table_width), "cache_attn: null block table, or a row stride below its width");
    STOF_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_pages) && aligned16(v_pages) && aligned16(workspace), "cache_attn: pointers must be 16-byte aligned");
    for (int i = 0; i < 3; ++i)
        STOF_REQUIRE(q_strides[i] % 8 == 0 && out_strides[i] % 8 == 0, "cache_attn: strides must be multiples of 8 elements");
    const Shape s = shape_of(requests, tokens, heads, kv_heads, page_size, table_width);
    const size_t need = stof_cache_attn_workspace_bytes(requests, tokens, heads, kv_heads, head_dim, page_size, table_width);
    if (workspace == nullptr || workspace_bytes < need) {
        set_error("cache_attn: workspace of %zu bytes, need %zu", workspace == nullptr ? static_cast<size_t>(0) : workspace_bytes, need);
        return STOF_E_WORKSPACE;
    }
    const long long joins = static_cast<long long>(requests) * kv_heads * s.row_groups;
    STOF_REQUIRE(joins < (1ll << 31), "cache_attn: requests * K/V heads * row groups beyond 2^31");
    CacheAttnParams p;
    p.q = q; p.out = out;
    for (int i = 0; i < 3; ++i) {
        p.q_stride[i] = q_strides[i];
        p.out_stride[i] = out_strides[i];
    }
    p.k_pages = k_pages; p.v_pages = v_pages; p.k_scales = k_scales; p.v_scales = v_scales;
    p.block_table = block_table; p.table_stride = table_stride; p.lengths = lengths;
    p.slopes = rules->slopes; p.distance_bias = rules->distance_bias; p.radius = rules->bias_radius;
    p.workspace = static_cast<float*>(workspace); p.status = status_dev;
    p.scale = rules->softmax_scale; p.softcap = rules->softcap; p.window = rules->window;
    p.requests = requests; p.tokens = tokens; p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads;
    p.rows = s.rows; p.row_groups = s.row_groups;
    p.table_width = table_width; p.page_count = pages; p.bf16 = dtype == STOF_DTYPE_BF16;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    auto launch = [&](auto kernel, auto join) -> int {
        LaunchConfig lc(dim3(static_cast<unsigned>(s.blocks)), CT_THREADS, 0, stream);
        STOF_CUDA(cudaLaunchKernelEx(&lc.cfg, kernel, p));
        LaunchConfig lj(dim3(static_cast<unsigned>(joins)), CT_THREADS, 0, stream);
        STOF_CUDA(cudaLaunchKernelEx(&lj.cfg, join, p, static_cast<int>(s.blocks)));
        return STOF_OK;
    };
    const bool e4m3 = cache_dtype == STOF_DTYPE_E4M3;
    if (head_dim == 64) {
        if (s.nt == 1) return e4m3 ? launch(cache_attn_kernel<1, 64, true>, cache_attn_join_kernel<1, 64>) : launch(cache_attn_kernel<1, 64, false>, cache_attn_join_kernel<1, 64>);
        return e4m3 ? launch(cache_attn_kernel<2, 64, true>, cache_attn_join_kernel<2, 64>) : launch(cache_attn_kernel<2, 64, false>, cache_attn_join_kernel<2, 64>);
    }
    if (s.nt == 1) return e4m3 ? launch(cache_attn_kernel<1, 128, true>, cache_attn_join_kernel<1, 128>) : launch(cache_attn_kernel<1, 128, false>, cache_attn_join_kernel<1, 128>);
    return e4m3 ? launch(cache_attn_kernel<2, 128, true>, cache_attn_join_kernel<2, 128>) : launch(cache_attn_kernel<2, 128, false>, cache_attn_join_kernel<2, 128>);
}
