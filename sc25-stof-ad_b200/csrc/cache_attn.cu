// Attention of a few query tokens per request over a paged 8-bit key/value cache (HBM-bound: every entry is read once).
//
// The query rows that share a K/V head (heads / kv_heads heads of each token) are the columns of both products, in tiles of 8:
//   S^T (16 keys x 8 rows) = K (16 keys x D) Q^T       O^T (D x 8 rows) += V^T (D x 16 keys) P^T
// on mma.sync m16n8k16.  A tcgen05 product has at least 64 rows of which a decoding step fills one to eight, and takes its operands
// from shared memory as 8 or 16 bits; here the entries become fp16 (exactly) on their way from shared memory to registers and are
// multiplied.  The scales stay out of the products: K's goes into the score, V's into P, relative to a reference of the row's own
// that follows the largest p * |scale| it has met: what carries weight keeps fp16's precision, whatever the scales are and in whatever order
// (a p below 2^-126 of its row's largest is 0 in fp32, as it would be in any softmax).
//
// Which lane holds which entry is free as long as both operands agree, so that every read is 16 bytes of a row: with g = lane / 4,
// c = lane % 4, a lane reads chunk c (and c + 4) of the rows of keys g and g + 8 for S, and chunk g of the rows of keys 2c, 2c + 1,
// 2c + 8, 2c + 9 for O.  P leaves the first product with keys along g and is wanted with rows along g: one 8 x 8 transpose.
//
// Work is counted in units of 128 keys (32 for each of a block's four warps).  The units of a (request, K/V head, row group) are cut into
// pieces of about the same length everywhere, a piece a block, whatever the lengths of the requests (which only the device knows).
// What one block covers is written at once, the rest in parts that cache_attn_join_kernel adds in the order of the blocks.
//
// Measured (int8 or e4m3 alike, pages of 16 to 128 alike): 96 requests of up to 16000 tokens, 32 heads on 8 of 128 (1.82 GB), 301 us = 6.0 TB/s,
// bound by memory (with a cap, in a run of seconds, 321 to 338 us = 5.2 to 5.5 TB/s, by the box); 48 of up to 8000, 32 heads on 8 of 64
// (0.22 GB), 64 us = 3.4 TB/s, bound by the instructions of a key, of which a row of 64 has almost as many as one of 128 for half the bytes
// (issue slots 61 % taken), 89 us with a distance table; one request of 4000 tokens 10.2 us, where the chain launch - lengths - pages' numbers -
// entries - parts - joining launch is all there is.  References of V for each row cost 0 to 6 % of that (one for all rows: 300, 63, 84, 9.9 us).
#include "cache_common.cuh"
#include "stof_host.h"
#include "stof_ptx.cuh"

#include <type_traits>

namespace stof {
namespace {

constexpr int CT_WARPS = 4, CT_THREADS = CT_WARPS * 32;
constexpr int CT_TILES = 2;                  // tiles of 16 keys that a warp takes at a time: independent chains of products, and half the work around them
constexpr int CT_STEP = 16 * CT_TILES, CT_UNIT = CT_STEP * CT_WARPS;     // keys of a warp's step, of a block's: the unit
constexpr int CT_STAGES = 2;                 // of a warp's ring: one step on its way while one is used (three: the same times, and less on an SM)
constexpr unsigned CT_LONG = 16, CT_WAVES = 4;                           // see piece_units
// Blocks on an SM: as many as registers (and for D = 128 shared memory) hold without spills.  D = 64, 16 requests of 12 heads: 22.0 us with
// four, 25.7 with three, 22.0 to 22.8 with five and six that spill a little (before slopes had a path without tests: 19.9 now).
constexpr int ct_blocks(int nt, int dim) { return nt == 2 ? 2 : dim == 64 ? 4 : 3; }
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
    int2* parts;                             // workspace: (first block, blocks) of every request's (K/V head, row group) ...
    float* workspace;                        // ... and the partial result of every block
    int* status;
    float scale, softcap;
    int window, radius;
    int requests, tokens, heads, kv_heads, group;            // group = heads / kv_heads
    int rows, row_groups;                                    // query rows of a K/V head, and how many blocks of them
    int table_width, page_count, page_shift;
    int resident;                                            // blocks that the GPU holds at once
    int bf16;
};

// keys [first, first + 128 * units) cover what the request's tokens see
struct Span { int length, first, units; };
__device__ __forceinline__ Span span_of(const CacheAttnParams& p, int b) {
    const int length = min(max(p.lengths[b], 0), p.table_width << p.page_shift);     // (at most 2^30)
    int first = 0;
    if (p.window > 0) first = max(length - p.tokens - p.window + 1, 0) & ~(CT_UNIT - 1);
    return {length, first, (length - first + CT_UNIT - 1) / CT_UNIT};
}

// How long the pieces are that the (request, K/V head, row group)s are cut into, in units, for `total` units in `pairs` of them: such that
// there are about as many pieces as blocks that the GPU holds at once (a piece too many would wait for a whole round: every pair rounds
// up, by half a piece on average), or more of CT_LONG units where there is work for more, up to CT_WAVES times as many, so that blocks that
// get on faster take over from the others towards the end (96 requests of up to 16000 tokens, when this was chosen: 297 us; once as many 355, twice 312, eight
// times 302; pieces of 8 or 32 units at least make no difference).
__device__ __forceinline__ unsigned piece_units(unsigned total, unsigned pairs, unsigned resident) {
    const unsigned at_once = pairs < resident ? resident - pairs / 2 : resident;
    const unsigned target = max(at_once, min(total / CT_LONG, resident * CT_WAVES));
    return max((total + target - 1) / target, 1u);
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// A warp's ring in shared memory, CT_TILES tiles of 16 keys a stage, filled by 16-byte asynchronous copies that only the warp itself waits for.  The
// chunks of a row are permuted, in D = 64 the rows of V too, so that the eight (or sixteen) lanes that a shared-memory access serves at
// once meet all banks.
template <int D>
struct Ring {
    static constexpr int STAGES = CT_STAGES;
    static constexpr int SIDE = 16 * D, TILE = 2 * SIDE + 16, STAGE = CT_TILES * TILE;       // of a tile: K, V, {k scale, v scale, valid, -}
    static constexpr int BYTES = STAGES * STAGE;
    static constexpr int CHUNKS = D / 16, LOADS = CHUNKS / 2;                // of a row; copies of a lane per side
    static __device__ __forceinline__ int k_at(int row, int chunk) {
        return D == 128 ? row * D + ((chunk ^ ((row & 1) << 2)) << 4) : row * D + (chunk << 4);
    }
    static __device__ __forceinline__ int v_at(int row, int chunk) {
        if (D == 128) return row * D + ((chunk ^ (row & 6)) << 4);
        const int place = (row >> 1) | ((row & 1) << 3);
        return place * D + ((chunk ^ (place & 2)) << 4);
    }
};
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

template <int NT, int D, bool E4M3>
__global__ void __launch_bounds__(CT_THREADS, ct_blocks(NT, D)) cache_attn_kernel(const CacheAttnParams p) {
    constexpr int CH = D / 64, KS = D / 16, MT = D / 16, ROWS = NT * 8;
    constexpr int V_BYTES = D / 8;           // of a row, per lane
    using R = Ring<D>;
    extern __shared__ __align__(128) unsigned char ca_smem[];
    __shared__ float merge_m[CT_WARPS][ROWS], merge_l[CT_WARPS][ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    float (*merge_o)[D + 4] = reinterpret_cast<float (*)[D + 4]>(ca_smem);   // the rings are free when it is used
    static_assert(CT_WARPS * ROWS * (D + 4) * 4 <= CT_WARPS * R::BYTES, "merge_o lies over the rings");
    unsigned char* ring = ca_smem + warp * R::BYTES;
    const uint32_t ring_addr = smem_u32(ring);
    grid_dependency_wait();
    grid_launch_dependents();
    const bool muted = failure_reported(p.status);           // asked for now, looked at when there is something to write
    // which piece is this block's?  Every warp finds out for itself, a lane a request (no barrier, the lengths are in the cache)
    const unsigned pairs = static_cast<unsigned>(p.kv_heads * p.row_groups);     // of a request
    Span span = {0, 0, 0};                                   // of the lane's request: the first 32 stay in registers
    unsigned total = 0, some = 0;
    for (int i = p.requests - 1 - (p.requests - 1 - lane & 31); i >= 0; i -= 32) {       // the last of lane, lane + 32, .. to the first
        span = span_of(p, i);
        total += static_cast<unsigned>(span.units);
        some += span.units > 0 ? 1u : 0u;
    }
    total = __reduce_add_sync(0xffffffffu, total) * pairs;
    some = __reduce_add_sync(0xffffffffu, some) * pairs;
    const unsigned length_each = piece_units(total, some, static_cast<unsigned>(p.resident));
    int b = -1;
    unsigned base = 0;
    for (int b0 = 0; b0 < p.requests; b0 += 32) {
        if (b0 > 0) span = b0 + lane < p.requests ? span_of(p, b0 + lane) : Span{0, 0, 0};
        const unsigned mine = (static_cast<unsigned>(span.units) + length_each - 1) / length_each * pairs;
        unsigned upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned here = __ballot_sync(0xffffffffu, blockIdx.x >= base + upto - mine && blockIdx.x < base + upto);
        if (here != 0) {
            const int at = __ffs(here) - 1;
            b = b0 + at;
            base += __shfl_sync(0xffffffffu, upto - mine, at);
            span = {__shfl_sync(0xffffffffu, span.length, at), __shfl_sync(0xffffffffu, span.first, at), __shfl_sync(0xffffffffu, span.units, at)};
            break;
        }
        base += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (b < 0) return;
    const unsigned pieces = (static_cast<unsigned>(span.units) + length_each - 1) / length_each;
    const unsigned pair = (blockIdx.x - base) / pieces, piece = (blockIdx.x - base) - pair * pieces;
    const unsigned each = static_cast<unsigned>(span.units) / pieces, extra = static_cast<unsigned>(span.units) - each * pieces;
    const int u0 = static_cast<int>(piece * each + min(piece, extra)), u1 = u0 + static_cast<int>(each + (piece < extra ? 1u : 0u));
    const int kv = static_cast<int>(pair) / p.row_groups, row0 = (static_cast<int>(pair) % p.row_groups) * ROWS;
    if (piece == 0 && threadIdx.x == 0) p.parts[b * pairs + pair] = make_int2(static_cast<int>(blockIdx.x), static_cast<int>(pieces));   // for the kernel that joins them
    {
        const int* pages = p.block_table + b * p.table_stride;
        const int last_key = min(span.length, span.first + u1 * CT_UNIT);
        // tiles that end in front of what the first token sees (a unit may begin with some) are not there: their pages may be anybody's
        const int seen_from = p.window > 0 ? span.length - p.tokens - p.window + 1 : 0;
        struct Pages { int of[CT_TILES]; };
        auto pages_of = [&](int key) {                       // of the tiles from this key on; -1 behind the last
            Pages r;
#pragma unroll
            for (int i = 0; i < CT_TILES; ++i) r.of[i] = key + 16 * i < last_key ? pages[(key + 16 * i) >> p.page_shift] : -1;
            return r;
        };
        // asks for the tiles from this key on; what cannot be had is marked
        auto ask = [&](int key, int stage, const Pages& page) {
#pragma unroll
            for (int i = 0; i < CT_TILES; ++i) {
                const int offset = stage * R::STAGE + i * R::TILE;
                const bool there = key + 16 * i < last_key && key + 16 * i + 15 >= seen_from, good = there && static_cast<unsigned>(page.of[i]) < static_cast<unsigned>(p.page_count);
                if (lane == 0) {
                    *reinterpret_cast<int*>(ring + offset + 2 * R::SIDE + 8) = good;
                    if (there && !good && p.status != nullptr) atomicCAS(p.status, 0, STATUS_BAD_INDEX);
                }
                if (good) {
                    const uint32_t dst = ring_addr + offset;
                    const size_t slot = static_cast<size_t>(page.of[i]) * p.kv_heads + kv;
                    const size_t at = ((slot << p.page_shift) + ((key + 16 * i) & ((1 << p.page_shift) - 1))) * D + lane * 16;
                    const char *kp = static_cast<const char*>(p.k_pages) + at, *vp = static_cast<const char*>(p.v_pages) + at;
#pragma unroll
                    for (int j = 0; j < R::LOADS; ++j) copy16(dst + R::k_at((j * 32 + lane) / R::CHUNKS, lane % R::CHUNKS), kp + j * 512);
#pragma unroll
                    for (int j = 0; j < R::LOADS; ++j) copy16(dst + R::SIDE + R::v_at((j * 32 + lane) / R::CHUNKS, lane % R::CHUNKS), vp + j * 512);
                    if (lane < 2) copy4(dst + 2 * R::SIDE + lane * 4, (lane == 0 ? p.k_scales : p.v_scales) + slot);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // STAGES - 1 steps on their way while one is used; pages' numbers are asked for a step before their tiles
        int key = span.first + u0 * CT_UNIT + warp * CT_STEP, far = key;
        Pages page = pages_of(far);
#pragma unroll
        for (int i = 0; i < R::STAGES - 1; ++i) {
            const Pages after = pages_of(far + CT_UNIT);
            ask(far, i, page);
            page = after;
            far += CT_UNIT;
        }
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
                row_scale[nt][e] = p.scale / f * LOG2E;
                pos[nt][e] = on ? span.length - p.tokens + rr / p.group : -1;
                slope[nt][e] = on && p.slopes != nullptr ? p.slopes[head] * LOG2E : 0.f;
                table[nt][e] = on && p.distance_bias != nullptr ? p.distance_bias + static_cast<size_t>(head) * (2 * p.radius + 1) + p.radius : p.distance_bias;
            }
        }

        // m: reference of the row's P, 0 as long as it has seen nothing; most: what a score may be above it, minus infinity until then
        // (NO_VALUE: it has seen keys, but no values other than 0).  o holds sum(P * scale * v) * c, with c a power of two, 0 until there are
        // values: the largest |P * scale * c| that has gone into it was 2^-5 at least, and is 2^15 at most.
        constexpr float NO_VALUE = -1e30f, FAR = 320.f;      // (2^254 is the largest ratio of two scales)
        float o[NT][MT][4], m[NT][2], most[NT][2], l[NT][2], c_row[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = 0.f;
            most[nt][0] = most[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = c_row[nt][0] = c_row[nt][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][mt][e] = 0.f;
        }

        auto word = [](const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; };
        // keys [see_from, see_to] are visible to every row of the block (none where a table has to be read for each)
        const int first_pos = span.length - p.tokens + row0 / p.group, last_pos = span.length - p.tokens + min(row0 + ROWS - 1, p.rows - 1) / p.group;
        const int see_from = p.window > 0 ? last_pos - p.window + 1 : 0, see_to = p.distance_bias == nullptr ? first_pos : -1;
        auto compute = [&](int key, const unsigned char* tiles) {
            float k_scale[CT_TILES], v_scale[CT_TILES];
            int left[CT_TILES];                              // keys of the tile that exist; what lies behind them may be anything
            bool any = false;
#pragma unroll
            for (int i = 0; i < CT_TILES; ++i) {
                const float4 head = *reinterpret_cast<const float4*>(tiles + i * R::TILE + 2 * R::SIDE);
                const bool good = __float_as_int(head.z) != 0;
                any = any || good;
                k_scale[i] = good ? head.x : 0.f;
                v_scale[i] = good && !(fabsf(head.y) < 1.17549435e-38f) ? head.y : 0.f;      // (1 / scale has to be finite)
                left[i] = good ? span.length - key - 16 * i : 0;
            }
            if (!any) return;
            float s[CT_TILES][NT][4];
            auto scores = [&] {                              // of the step's keys
#pragma unroll
                for (int t = 0; t < CT_TILES; ++t)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[t][nt][e] = 0.f;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    uint4 x[CT_TILES], y[CT_TILES];
#pragma unroll
                    for (int t = 0; t < CT_TILES; ++t) {
                        x[t] = *reinterpret_cast<const uint4*>(tiles + t * R::TILE + R::k_at(g, c + 4 * i));
                        y[t] = *reinterpret_cast<const uint4*>(tiles + t * R::TILE + R::k_at(g + 8, c + 4 * i));
                    }
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int t = 0; t < CT_TILES; ++t) {
                            uint32_t a0, a1, a2, a3;
                            entries_to_half<E4M3>(word(x[t], w), a0, a2);
                            entries_to_half<E4M3>(word(y[t], w), a1, a3);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma16816(s[t][nt], a0, a1, a2, a3, qf[nt][4 * i + w][0], qf[nt][4 * i + w][1]);
                        }
                }
                // in units of log2, less the row's reference; element e: key g + 8 * (e / 2), row 2c + e % 2
                if (p.softcap > 0.f) {
                    const float to = 1.f / (p.softcap * LOG2E), from = p.softcap * LOG2E;
                    float top = 0.f;                             // of |score / softcap|
#pragma unroll
                    for (int t = 0; t < CT_TILES; ++t)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                s[t][nt][e] *= k_scale[t] * row_scale[nt][e & 1] * to;
                                top = fmaxf(top, fabsf(s[t][nt][e]));
                            }
                    if (__all_sync(0xffffffffu, top <= 0.35f)) {
#pragma unroll
                        for (int t = 0; t < CT_TILES; ++t)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[t][nt][e] = from * tanh_near_zero(s[t][nt][e]);
                    } else {
#pragma unroll
                        for (int t = 0; t < CT_TILES; ++t)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[t][nt][e] = from * tanh_any(s[t][nt][e]);
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < CT_TILES; ++t)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[t][nt][e] *= k_scale[t] * row_scale[nt][e & 1];
                }
                if (key >= see_from && key + CT_STEP - 1 <= see_to && left[0] > 0 && left[CT_TILES - 1] > 0) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float away = static_cast<float>(key + g - pos[nt][e]), less = fmaf(slope[nt][e], away, -m[nt][e]);
#pragma unroll
                            for (int t = 0; t < CT_TILES; ++t) {
                                s[t][nt][e] += fmaf(slope[nt][e], static_cast<float>(16 * t), less);
                                s[t][nt][2 + e] += fmaf(slope[nt][e], static_cast<float>(16 * t + 8), less);
                            }
                        }
                } else {
#pragma unroll
                    for (int t = 0; t < CT_TILES; ++t)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float x = s[t][nt][e];
                                const int away = key + 16 * t + g + 8 * (e >> 1) - pos[nt][e & 1];   // at most 0 where visible
                                x += slope[nt][e & 1] * static_cast<float>(away);
                                const bool on = left[t] > 0 && pos[nt][e & 1] >= 0 && away <= 0 && (p.window == 0 || away > -p.window);
                                if (p.distance_bias != nullptr && on) {
                                    const float bias = __ldca(table[nt][e & 1] + max(away, -p.radius));
                                    const float y = finite_or_nan(fmaf(bias, LOG2E, x));
                                    x = bias == -INFINITY ? bias : y;
                                }
                                s[t][nt][e] = on ? x - m[nt][e & 1] : -INFINITY;
                            }
                }
            };
            scores();
            // Rows' references move where a score is more than 2^8 above one (P is at most that, then), where the first values come, and where V's
            // scale leaves P * scale * c more than 2^15
            float v_size = 0.f, c_most = 0.f;
#pragma unroll
            for (int t = 0; t < CT_TILES; ++t) v_size = fabsf(v_scale[t]) <= v_size ? v_size : fabsf(v_scale[t]);    // (a NaN stays)
            bool move = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
                    for (int t = 1; t < CT_TILES; ++t) top = fmaxf(top, fmaxf(s[t][nt][e], s[t][nt][2 + e]));
                    move = move || top > most[nt][e];
                    c_most = fmaxf(c_most, c_row[nt][e]);
                }
            bool uneven = false;                             // V's scale * c of some row is large, or none at all
            if (__any_sync(0xffffffffu, move || !(v_size * c_most <= 128.f))) {
                float tops[NT][2];
                auto largest = [&] {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            tops[nt][e] = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
                            for (int t = 1; t < CT_TILES; ++t) tops[nt][e] = fmaxf(tops[nt][e], fmaxf(s[t][nt][e], s[t][nt][2 + e]));
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) tops[nt][e] = fmaxf(tops[nt][e], __shfl_xor_sync(0xffffffffu, tops[nt][e], d));
                        }
                };
                largest();
                // A score so far above the reference has lost digits to it, and nothing that came before has weight beside it (no ratio of
                // scales makes up for it): the row begins anew, from scores less nothing
                bool anew = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) anew = anew || (tops[nt][0] > FAR && most[nt][0] > -INFINITY) || (tops[nt][1] > FAR && most[nt][1] > -INFINITY);
                if (__builtin_expect(__any_sync(0xffffffffu, anew), 0)) {
                    asm volatile("" ::: "memory");           // (the step's keys are read again, not kept)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (tops[nt][e] > FAR && most[nt][e] > -INFINITY) {
                                m[nt][e] = c_row[nt][e] = 0.f;
                                most[nt][e] = -INFINITY;
                                l[nt][e] *= 0.f;             // (a NaN stays)
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    o[nt][mt][e] *= 0.f;
                                    o[nt][mt][2 + e] *= 0.f;
                                }
                            }
                    scores();
                    largest();
                }
                // the largest P * |scale| of a row: where the tiles' scales are alike, the largest P's will do
                float v_log[CT_TILES];
                bool alike = true;
#pragma unroll
                for (int t = 0; t < CT_TILES; ++t) {
                    alike = alike && fabsf(v_scale[t]) * 16.f >= v_size;
                    v_log[t] = __log2f(fabsf(v_scale[t]));
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float top = tops[nt][e];
                        const bool seen = top > -INFINITY, first = most[nt][e] == -INFINITY;
                        float up = 0.f;
                        if (seen && (first || top > 0.f)) {  // by a whole number of powers of two, behind the first
                            const float to = m[nt][e] + (first ? top : ceilf(top));
                            up = to - m[nt][e];
                            m[nt][e] = to;
                            l[nt][e] *= first ? 0.f : fast_exp2(-up);
#pragma unroll
                            for (int t = 0; t < CT_TILES; ++t) {
                                s[t][nt][e] -= up;
                                s[t][nt][2 + e] -= up;
                            }
                        }
                        float weight = top - up + v_log[0];  // log2 of the row's largest P * |scale|
                        if (!alike) {
                            weight = -INFINITY;
#pragma unroll
                            for (int t = 0; t < CT_TILES; ++t) weight = fmaxf(weight, fmaxf(s[t][nt][e], s[t][nt][2 + e]) + v_log[t]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) weight = fmaxf(weight, __shfl_xor_sync(0xffffffffu, weight, d));
                        }
                        if (seen) {
                            const float c_old = c_row[nt][e], log_c = static_cast<float>(static_cast<int>(__float_as_uint(c_old) >> 23) - 127);
                            // as P shrinks by 2^up c may grow by it, and o stays as it is, unless the new P * |scale| asks for less
                            float log_to = log_c + rintf(up);
                            if (c_old == 0.f || weight + log_to > 0.f) log_to = floorf(-weight);
                            log_to = fminf(fmaxf(log_to, -126.f), 126.f);
                            most[nt][e] = 8.f;
                            if (c_old == 0.f && weight == -INFINITY) {
                                most[nt][e] = NO_VALUE;
                            } else {
                                c_row[nt][e] = __uint_as_float(static_cast<uint32_t>(127 + static_cast<int>(log_to)) << 23);
                                const float f = c_old == 0.f ? 0.f : fast_exp2(log_to - log_c - up);
                                if (f != 1.f) {
#pragma unroll
                                    for (int mt = 0; mt < MT; ++mt) {
                                        o[nt][mt][e] *= f;
                                        o[nt][mt][2 + e] *= f;
                                    }
                                }
                            }
                        }
                        uneven = uneven || !(v_size * c_row[nt][e] <= 128.f);
                    }
                uneven = __any_sync(0xffffffffu, uneven);
            }
            uint32_t pf[CT_TILES][NT][2];
            // `masked`: p * scale where p is not 0 (zero times infinity or NaN for a row that sees nothing of the tile)
            auto weights = [&](auto masked) {
#pragma unroll
                for (int t = 0; t < CT_TILES; ++t)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float x[4], w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            x[e] = fast_exp2(s[t][nt][e]);
                            w[e] = x[e] * (v_scale[t] * c_row[nt][e & 1]);
                            if constexpr (decltype(masked)::value) {
                                const float c = c_row[nt][e & 1];            // (large, its product with a large scale may leave fp32; small, p's may)
                                w[e] = x[e] == 0.f ? 0.f : c >= 1.f ? x[e] * v_scale[t] * c : w[e];
                            }
                        }
                        l[nt][0] += x[0] + x[2];
                        l[nt][1] += x[1] + x[3];
                        // to fp16 for the product, as the other attention kernels do; the sum is of the values before rounding
                        pf[t][nt][0] = transpose8x8(pack_half2(w[0], w[1]));
                        pf[t][nt][1] = transpose8x8(pack_half2(w[2], w[3]));
                    }
            };
            if (__builtin_expect(uneven, 0)) weights(std::true_type());
            else weights(std::false_type());
#pragma unroll
            for (int t = 0; t < CT_TILES; ++t) {
                uint4 v[4];                                  // keys 2c, 2c + 1, 2c + 8, 2c + 9 (D = 64: the first half)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = 2 * c + (j & 1) + 8 * (j >> 1);
                    const unsigned char* src = tiles + t * R::TILE + R::SIDE + R::v_at(row, D == 128 ? g : g >> 1);
                    if constexpr (D == 128) {
                        v[j] = *reinterpret_cast<const uint4*>(src);
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(src + (g & 1) * 8);
                        v[j] = make_uint4(w.x, w.y, 0u, 0u);
                    }
                }
                const int hidden = seen_from - key - 16 * t;             // keys of the tile in front of every token's window
                if (left[t] < 16 || hidden > 0) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int row = 2 * c + (j & 1) + 8 * (j >> 1);
                        if (row >= left[t] || row < hidden) v[j] = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
#pragma unroll
                for (int w = 0; w < V_BYTES / 4; ++w) {
                    const uint32_t x0 = word(v[0], w), x1 = word(v[1], w), y0 = word(v[2], w), y1 = word(v[3], w);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t a0, a1, a2, a3;
                        entries_to_half<E4M3>(__byte_perm(x0, x1, h == 0 ? 0x5140 : 0x7362), a0, a1);
                        entries_to_half<E4M3>(__byte_perm(y0, y1, h == 0 ? 0x5140 : 0x7362), a2, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][2 * w + h], a0, a1, a2, a3, pf[t][nt][0], pf[t][nt][1]);
                    }
                }
            }
        };
        for (int u = u0, stage = 0; u < u1; ++u) {
            asm volatile("cp.async.wait_group %0;" ::"n"(R::STAGES - 2) : "memory");
            __syncwarp();                                    // the tiles are there for all lanes, and all have used those before
            const Pages after = pages_of(far + CT_UNIT);
            ask(far, stage == 0 ? R::STAGES - 1 : stage - 1, page);
            page = after;
            far += CT_UNIT;
            compute(key, ring + stage * R::STAGE);
            key += CT_UNIT;
            stage = stage + 1 == R::STAGES ? 0 : stage + 1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (__syncthreads_or(muted)) return;                 // merge_o lies over the rings

        // ---- the four warps' results are added in smem, in their order
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (most[nt][e] == -INFINITY) m[nt][e] = -INFINITY;
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
                weight[nt][e] = m[nt][e] == -INFINITY ? l[nt][e] : fast_exp2(m[nt][e] - top) * (c_row[nt][e] > 0.f ? 1.f / c_row[nt][e] : 1.f);
            }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float* dst = &merge_o[warp * ROWS + nt * 8 + 2 * c + e][g * 2 * MT];
                const float f = weight[nt][e];
#pragma unroll
                for (int i = 0; i < 2 * MT; i += 4)          // d = g * 2 MT + i: m-tile i / 2, first row or second
                    *reinterpret_cast<float4*>(dst + i) = f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                                                   : make_float4(o[nt][i / 2][e] * f, o[nt][i / 2][2 + e] * f, o[nt][i / 2 + 1][e] * f, o[nt][i / 2 + 1][2 + e] * f);
            }
        __syncthreads();
        const bool whole = pieces == 1;
        float* part = p.workspace + static_cast<size_t>(blockIdx.x) * (ROWS * (D + 2));
        for (int i = threadIdx.x; i < ROWS * (D / 8); i += CT_THREADS) {
            const int r = i / (D / 8), d = i % (D / 8) * 8;
            if (row0 + r >= p.rows) continue;
            float top = merge_m[0][r];
            for (int w = 1; w < CT_WARPS; ++w) top = fmaxf(top, merge_m[w][r]);
            float sum = 0.f;
            for (int w = 0; w < CT_WARPS; ++w)
                sum += merge_m[w][r] > -INFINITY ? merge_l[w][r] * fast_exp2(merge_m[w][r] - top) : merge_l[w][r];
            float4 x = *reinterpret_cast<const float4*>(&merge_o[r][d]), y = *reinterpret_cast<const float4*>(&merge_o[r][d + 4]);
#pragma unroll
            for (int w = 1; w < CT_WARPS; ++w) {
                const float4 xw = *reinterpret_cast<const float4*>(&merge_o[w * ROWS + r][d]), yw = *reinterpret_cast<const float4*>(&merge_o[w * ROWS + r][d + 4]);
                x = make_float4(x.x + xw.x, x.y + xw.y, x.z + xw.z, x.w + xw.w);
                y = make_float4(y.x + yw.x, y.y + yw.y, y.z + yw.z, y.w + yw.w);
            }
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
    }
}

// Adds the parts of what more than one block worked on, a row a block, in the order of the blocks within each warp; and writes the zeros of
// empty requests.
template <int NT, int D>
__global__ void __launch_bounds__(CT_THREADS) cache_attn_join_kernel(const CacheAttnParams p) {
    constexpr int ROWS = NT * 8, EACH = D / 32, AHEAD = 8;
    __shared__ float add_o[CT_WARPS][D], add_l[CT_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dependency_wait();
    grid_launch_dependents();
    const int pairs = p.kv_heads * p.row_groups;
    const int b = blockIdx.x / pairs, pair = blockIdx.x % pairs, kv = pair / p.row_groups, row = (pair % p.row_groups) * ROWS + blockIdx.y;
    if (row >= p.rows) return;
    // what the launch costs is its loads one after the other: status, parts and length together, then the first parts and all maxima
    const int2 parts = __ldca(p.parts + blockIdx.x);
    const bool muted = failure_reported(p.status);
    const bool empty = span_of(p, b).units == 0;             // (its entry was not written)
    if (__syncthreads_or(muted) || (!empty && parts.y == 1)) return;         // (one block had all of it)
    const int count = empty ? 0 : parts.y, r = blockIdx.y;
    auto part = [&](int i) { return p.workspace + static_cast<size_t>(parts.x + i) * (ROWS * (D + 2)); };
    float m[AHEAD], l[AHEAD], x[AHEAD][EACH];
    auto load = [&](int i0) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {                    // no branches: all loads are on their way together
            const float* at = part(min(i0 + j * CT_WARPS, count - 1));
            m[j] = __ldca(at + r);
            l[j] = __ldca(at + ROWS + r);
            at += 2 * ROWS + r * D + lane * EACH;
            if constexpr (EACH == 4) {
                const float4 v = __ldca(reinterpret_cast<const float4*>(at));
                x[j][0] = v.x; x[j][1] = v.y; x[j][2] = v.z; x[j][3] = v.w;
            } else {
                const float2 v = __ldca(reinterpret_cast<const float2*>(at));
                x[j][0] = v.x; x[j][1] = v.y;
            }
        }
    };
    float top = -INFINITY, sum = 0.f, o[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) o[e] = 0.f;
    float own = -INFINITY;
    if (lane < count) own = __ldca(part(lane) + r);
    if (warp < count) load(warp);
    top = own;
    for (int i = lane + 32; i < count; i += 32) top = fmaxf(top, __ldca(part(i) + r));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    for (int i0 = warp; i0 < count; i0 += CT_WARPS * AHEAD) {
        if (i0 != warp) load(i0);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            // (a part that saw nothing is 0, or NaN)
            const float f = i0 + j * CT_WARPS >= count ? 0.f : m[j] > -INFINITY ? fast_exp2(m[j] - top) : 1.f;
            if (f == 0.f) continue;                          // (nothing of a part that is there twice, nor zero times an infinity)
            sum += l[j] * f;
#pragma unroll
            for (int e = 0; e < EACH; ++e) o[e] += x[j][e] * f;
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) add_o[warp][lane * EACH + e] = o[e];
    if (lane == 0) add_l[warp] = sum;
    __syncthreads();
    if (threadIdx.x < D / 2) {
        const int d = threadIdx.x * 2;
        float l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < CT_WARPS; ++w) {
            l += add_l[w];
            x += add_o[w][d];
            y += add_o[w][d + 1];
        }
        const float inv = l != 0.f ? 1.f / l : 0.f;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + b * p.out_stride[0] + (row / p.group) * p.out_stride[1] + (kv * p.group + row % p.group) * p.out_stride[2] + d;
        *reinterpret_cast<uint32_t*>(dst) = p.bf16 ? pack_pair<true>(x * inv, y * inv) : pack_pair<false>(x * inv, y * inv);
    }
}

struct Shape {
    int rows, nt, row_groups;
    int resident;
    long long blocks, joins, units;          // joins: (request, K/V head, row group)s; units: at most
};
// row tiles of 8: one up to 8 rows, else two at a time; blocks: as many as there may be pieces (piece_units)
Shape shape_of(int requests, int tokens, int heads, int kv_heads, int head_dim, int page_size, int table_width) {
    Shape s;
    s.rows = tokens * (heads / kv_heads);
    s.nt = s.rows <= 8 ? 1 : 2;
    s.row_groups = (s.rows + 8 * s.nt - 1) / (8 * s.nt);
    s.joins = static_cast<long long>(requests) * kv_heads * s.row_groups;
    s.units = s.joins * ((static_cast<long long>(table_width) * page_size + CT_UNIT - 1) / CT_UNIT);
    s.resident = sm_count() * ct_blocks(s.nt, head_dim);
    long long pieces = s.units / CT_LONG;
    if (pieces > static_cast<long long>(s.resident) * CT_WAVES) pieces = static_cast<long long>(s.resident) * CT_WAVES;
    if (pieces < s.resident) pieces = s.resident;
    s.blocks = pieces + s.joins;
    if (s.blocks > s.units) s.blocks = s.units > 0 ? s.units : 1;
    return s;
}

template <int NT, int D, bool E4M3>
int launch(const CacheAttnParams& p, const Shape& s, cudaStream_t stream) {
    if (int rc = allow_shared_memory<cache_attn_kernel<NT, D, E4M3>>()) return rc;
    LaunchConfig lc(dim3(static_cast<unsigned>(s.blocks)), CT_THREADS, CT_WARPS * Ring<D>::BYTES, stream);
    STOF_CUDA(cudaLaunchKernelEx(&lc.cfg, cache_attn_kernel<NT, D, E4M3>, p));
    LaunchConfig lj(dim3(static_cast<unsigned>(s.joins), static_cast<unsigned>(s.rows < 8 * NT ? s.rows : 8 * NT)), CT_THREADS, 0, stream);
    STOF_CUDA(cudaLaunchKernelEx(&lj.cfg, cache_attn_join_kernel<NT, D>, p));
    return STOF_OK;
}

}  // namespace
}  // namespace stof

using namespace stof;

extern "C" size_t stof_cache_attn_workspace_bytes(int requests, int tokens, int heads, int kv_heads, int head_dim, int page_size, int table_width) {
    if (requests <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || page_size <= 0 || table_width < 0 ||
        static_cast<long long>(tokens) * (heads / kv_heads) > (1ll << 30))
        return 0;
    const Shape s = shape_of(requests, tokens, heads, kv_heads, head_dim, page_size, table_width);
    return (static_cast<size_t>(s.joins) * sizeof(int2) + 15) / 16 * 16 + static_cast<size_t>(s.blocks) * (8 * s.nt) * (static_cast<size_t>(head_dim) + 2) * sizeof(float);
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
    STOF_REQUIRE(static_cast<long long>(table_width) * page_size <= (1ll << 30), "cache_attn: a row of the block table spans more than 2^30 tokens");
    STOF_REQUIRE(static_cast<long long>(tokens) * (heads / kv_heads) <= (1ll << 30), "cache_attn: more than 2^30 query rows of a K/V head");
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
    const Shape s = shape_of(requests, tokens, heads, kv_heads, head_dim, page_size, table_width);
    const size_t need = stof_cache_attn_workspace_bytes(requests, tokens, heads, kv_heads, head_dim, page_size, table_width);
    if (workspace == nullptr || workspace_bytes < need) {
        set_error("cache_attn: workspace of %zu bytes, need %zu", workspace == nullptr ? static_cast<size_t>(0) : workspace_bytes, need);
        return STOF_E_WORKSPACE;
    }
    STOF_REQUIRE(s.joins < (1ll << 31) && s.units < (1ll << 31), "cache_attn: requests * K/V heads * row groups * units of %d keys beyond 2^31", CT_UNIT);
    CacheAttnParams p;
    p.q = q; p.out = out;
    for (int i = 0; i < 3; ++i) {
        p.q_stride[i] = q_strides[i];
        p.out_stride[i] = out_strides[i];
    }
    p.k_pages = k_pages; p.v_pages = v_pages; p.k_scales = k_scales; p.v_scales = v_scales;
    p.block_table = block_table; p.table_stride = table_stride; p.lengths = lengths;
    p.slopes = rules->slopes; p.distance_bias = rules->distance_bias; p.radius = rules->bias_radius;
    p.parts = static_cast<int2*>(workspace);
    p.workspace = reinterpret_cast<float*>(static_cast<char*>(workspace) + (static_cast<size_t>(s.joins) * sizeof(int2) + 15) / 16 * 16); p.status = status_dev;
    p.scale = rules->softmax_scale; p.softcap = usable_cap(rules->softcap);
    // (a window as long as a request may be hides nothing; below that, positions less it stay inside 32 bits)
    p.window = rules->window >= static_cast<long long>(table_width) * page_size ? 0 : rules->window;
    p.requests = requests; p.tokens = tokens; p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads;
    p.rows = s.rows; p.row_groups = s.row_groups; p.resident = s.resident;
    p.table_width = table_width; p.page_count = pages; p.bf16 = dtype == STOF_DTYPE_BF16;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    const bool e4m3 = cache_dtype == STOF_DTYPE_E4M3;
    if (head_dim == 64) {
        if (s.nt == 1) return e4m3 ? launch<1, 64, true>(p, s, stream) : launch<1, 64, false>(p, s, stream);
        return e4m3 ? launch<2, 64, true>(p, s, stream) : launch<2, 64, false>(p, s, stream);
    }
    if (s.nt == 1) return e4m3 ? launch<1, 128, true>(p, s, stream) : launch<1, 128, false>(p, s, stream);
    return e4m3 ? launch<2, 128, true>(p, s, stream) : launch<2, 128, false>(p, s, stream);
}
