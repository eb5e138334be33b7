// New keys and values into the slots of a paged 8-bit cache, one scale per page and head (HBM-bound for prompts, latency-bound for
// the tokens of a step).
//
// What bounds it: the chain slots -> rows -> maximum -> entries, of which the SM has to hold many at once: 18000 tokens of 8 heads of 128
// (111 MB) take 24 to 25 us, 4.4 to 4.6 TB/s, with eight blocks of 64 registers on an SM; 29 with six of 80, 30 with ten of 48 that spill, 31 with twice
// the warps for a run, 97 with keys and values in blocks of their own and runs held whole (168 registers).
//
// A run is a stretch of tokens whose slots follow one another inside a page; its scale needs the largest magnitude of all its
// rows, so a run belongs to one warp (up to four tokens) or one thread block: the rows are read once, held in registers as they
// came, reduced, and written as entries.  Runs are found from the slots alone: a thread block looks at a few neighbouring tokens for
// one head and serves the runs that begin there; every warp finds them for itself, from ballots, without a barrier.
#include "cache_common.cuh"
#include "stof_host.h"
#include "stof_ptx.cuh"

namespace stof {
namespace {

constexpr int CA_WARPS = 4;
constexpr int CA_SHORT = 4;                  // tokens up to which a warp serves a run alone
constexpr int CA_MAX_CHUNK = 32;

struct AppendParams {
    void* pages[2];
    float* scales[2];
    const void* x[2];
    long long token_stride[2], head_stride[2];
    const int* slots;
    int* status;
    int page_count, heads, page_shift, tokens, chunk;
};

template <bool BF16, bool E4M3, int D>
struct Rows {
    static constexpr int LANES = D / 8;                      // lanes that share a row, 16 bytes each
    static constexpr int EACH = 32 / LANES;                  // rows of one warp-wide load

    // An e4m3 entry can be NaN itself, an int8 one cannot: there a NaN goes into the page's scale, so that it comes out of what reads the page
    static __device__ __forceinline__ float larger(float a, float b) {
        if constexpr (E4M3) return fmaxf(a, b);
        float c;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
        return c;
    }
    static __device__ __forceinline__ float magnitude(const uint4& u) {
        auto pair = [](uint32_t w) {
            const float2 f = unpack_pair<BF16>(w);
            return larger(fabsf(f.x), fabsf(f.y));
        };
        return larger(larger(pair(u.x), pair(u.y)), larger(pair(u.z), pair(u.w)));
    }
    static __device__ __forceinline__ uint2 entries(const uint4& u, float inv) {
        return make_uint2(quantise4<E4M3>(unpack_pair<BF16>(u.x), unpack_pair<BF16>(u.y), inv), quantise4<E4M3>(unpack_pair<BF16>(u.z), unpack_pair<BF16>(u.w), inv));
    }
};

// One run: tokens [token, token + n) into rows [row, row + n) of a page, keys and values.  `part` of `parts` warps work on it (1: this warp
// alone).  NV loads a side hold a warp's share of a pass; a run of more than one pass is read twice, the second time from cache.
template <bool BF16, bool E4M3, int D, int NV>
__device__ __forceinline__ void write_run(const AppendParams& p, int head, int token, int n, int page, int row, int part, int parts, float (*shared)[2]) {
    using R = Rows<BF16, E4M3, D>;
    const int lane = threadIdx.x & 31, sub = lane / R::LANES, col = lane % R::LANES;
    const long long at = static_cast<long long>(page) * p.heads + head;
    const int pass = NV * parts * R::EACH;                   // rows of a pass
    uint4 v[2][NV];
    auto load = [&](int from) {
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const uint16_t* x = static_cast<const uint16_t*>(p.x[side]) + head * p.head_stride[side] + col * 8;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int r = from + (i * parts + part) * R::EACH + sub;
                v[side][i] = make_uint4(0u, 0u, 0u, 0u);
                if (r < n) v[side][i] = __ldca(reinterpret_cast<const uint4*>(x + (token + r) * p.token_stride[side]));
            }
        }
    };
    float old[2] = {0.f, 0.f}, top[2] = {0.f, 0.f};
    int from = 0;
    while (true) {
        load(from);
        if (from == 0 && row > 0) {
            old[0] = p.scales[0][at];
            old[1] = p.scales[1][at];
        }
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int i = 0; i < NV; ++i) top[side] = R::larger(top[side], R::magnitude(v[side][i]));
        if (from + pass >= n) break;
        from += pass;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        top[0] = R::larger(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
        top[1] = R::larger(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
    }
    if (parts > 1) {
        if (lane < 2) shared[part][lane] = lane == 0 ? top[0] : top[1];
        __syncthreads();                                     // (and everyone has read the old scales)
#pragma unroll
        for (int w = 0; w < CA_WARPS; ++w) {
            top[0] = R::larger(top[0], shared[w][0]);
            top[1] = R::larger(top[1], shared[w][1]);
        }
    }
    float inv[2], ratio[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        float now = top[side] * (1.0f / entry_max<E4M3>());
        if (now < 1.17549435e-38f) now = 0.f;
        now = R::larger(now, old[side]);
        inv[side] = now > 0.f ? 1.0f / now : 0.f;
        ratio[side] = row > 0 && now > old[side] ? old[side] / now : 1.f;    // 1: what is in front of the run stays
        if (part == 0 && lane == 0) p.scales[side][at] = now;
    }
    const bool again[2] = {ratio[0] != 1.f, ratio[1] != 1.f};
    while (true) {                                           // from the last pass, which is still there, to the first
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            uint8_t* entries = static_cast<uint8_t*>(p.pages[side]) + ((at << p.page_shift) + row) * D + col * 8;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int r = from + (i * parts + part) * R::EACH + sub;
                if (r < n) *reinterpret_cast<uint2*>(entries + static_cast<size_t>(r) * D) = R::entries(v[side][i], inv[side]);
            }
        }
        if (from == 0) break;
        from -= pass;
        load(from);
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        if (!again[side]) continue;                          // the entries in front of the run, rounded again to the new scale
        uint4* front = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.pages[side]) + (at << p.page_shift) * D);
        for (int i = part * 32 + lane; i < row * D / 16; i += parts * 32) {
            const uint4 u = front[i];
            auto round_again = [&](uint32_t w) {
                uint32_t lo, hi;
                entries_to_half<E4M3>(w, lo, hi);
                const float2 a = unpack_pair<false>(lo), b = unpack_pair<false>(hi);
                return quantise4<E4M3>(a, b, ratio[side]);
            };
            front[i] = make_uint4(round_again(u.x), round_again(u.y), round_again(u.z), round_again(u.w));
        }
    }
}

template <bool BF16, bool E4M3, int D>
__global__ void __launch_bounds__(CA_WARPS * 32, 8) cache_append_kernel(const AppendParams p) {
    __shared__ float shared[CA_WARPS][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = blockIdx.y, page = 1 << p.page_shift;
    grid_dependency_wait();
    grid_launch_dependents();
    // every warp looks at the chunk's tokens and at as many behind them as a run can take: where a run begins (or nothing is written)
    constexpr int SEEN = 1 + 128 / 32;
    const int t0 = blockIdx.x * p.chunk;
    int slot[SEEN];
#pragma unroll
    for (int i = 0; i < SEEN; ++i) slot[i] = t0 + 32 * i + lane < p.tokens ? p.slots[t0 + 32 * i + lane] : -1;
    const int in_front = t0 > 0 ? p.slots[t0 - 1] : -2;
    if (__syncthreads_or(failure_reported(p.status))) return;
    const long long slot_end = static_cast<long long>(p.page_count) << p.page_shift;
    unsigned begins[SEEN], good = 0;
#pragma unroll
    for (int i = 0; i < SEEN; ++i) {
        int before = __shfl_up_sync(0xffffffffu, slot[i], 1);
        const int carried = i > 0 ? __shfl_sync(0xffffffffu, slot[i > 0 ? i - 1 : 0], 31) : in_front;
        if (lane == 0) before = carried;
        begins[i] = __ballot_sync(0xffffffffu, slot[i] < 0 || slot[i] != before + 1 || (slot[i] & (page - 1)) == 0);
        if (i == 0) {
            good = __ballot_sync(0xffffffffu, lane < p.chunk && slot[0] >= 0 && slot[0] < slot_end);
            if (lane < p.chunk && slot[0] >= slot_end && p.status != nullptr) atomicCAS(p.status, 0, STATUS_BAD_INDEX);
        }
    }
    int found = 0;
    for (unsigned leads = begins[0] & good; leads != 0; leads &= leads - 1) {
        const int at = __ffs(leads) - 1;
        // to the next beginning
        int n = -at;
        const unsigned later = at == 31 ? 0u : begins[0] & ~((2u << at) - 1u);
        if (later != 0) {
            n += __ffs(later) - 1;
        } else {
            n += 32;
#pragma unroll
            for (int i = 1; i < SEEN; ++i) {
                if (begins[i] != 0) {
                    n += __ffs(begins[i]) - 1;
                    break;
                }
                n += 32;
            }
        }
        const int s = __shfl_sync(0xffffffffu, slot[0], at);
        if (n <= CA_SHORT) {                                 // a warp each, in turn
            if (found++ % CA_WARPS == warp)
                write_run<BF16, E4M3, D, CA_SHORT / Rows<BF16, E4M3, D>::EACH>(p, head, t0 + at, n, s >> p.page_shift, s & (page - 1), 0, 1, shared);
        } else {
            __syncthreads();                                 // `shared` is free
            write_run<BF16, E4M3, D, 32 / (CA_WARPS * Rows<BF16, E4M3, D>::EACH)>(p, head, t0 + at, n, s >> p.page_shift, s & (page - 1), warp, CA_WARPS, shared);
        }
    }
}

}  // namespace
}  // namespace stof

using namespace stof;

extern "C" int stof_cache_append(void* k_pages, void* v_pages, float* k_scales, float* v_scales, int cache_dtype, int pages, int page_size,
                                 int kv_heads, int head_dim, const void* k, const void* v, int dtype, const long long k_strides[2],
                                 const long long v_strides[2], const int* slots, int tokens, int* status_dev, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    STOF_REQUIRE(tokens >= 0 && pages >= 0 && kv_heads > 0 && kv_heads <= 65535, "cache_append: bad shape");
    STOF_REQUIRE(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128, "cache_append: page size %d not in {16, 32, 64, 128}", page_size);
    STOF_REQUIRE(head_dim == 64 || head_dim == 128, "cache_append: head_dim %d not in {64, 128}", head_dim);
    STOF_REQUIRE(static_cast<long long>(pages) * page_size < (1ll << 31), "cache_append: %d pages of %d tokens do not fit 32-bit slots", pages, page_size);
    STOF_REQUIRE(cache_dtype == STOF_DTYPE_INT8 || cache_dtype == STOF_DTYPE_E4M3, "cache_append: cache entries must be int8 or e4m3");
    STOF_REQUIRE(dtype == STOF_DTYPE_F16 || dtype == STOF_DTYPE_BF16, "cache_append: keys and values must be fp16 or bf16");
    if (tokens == 0) return STOF_OK;
    STOF_REQUIRE(k_pages && v_pages && k_scales && v_scales && k && v && k_strides && v_strides && slots, "cache_append: null pointer");
    STOF_REQUIRE(aligned16(k_pages) && aligned16(v_pages) && aligned16(k) && aligned16(v), "cache_append: pointers must be 16-byte aligned");
    for (int i = 0; i < 2; ++i)
        STOF_REQUIRE(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0, "cache_append: strides must be multiples of 8 elements");
    STOF_REQUIRE(k_pages != v_pages && k_scales != v_scales, "cache_append: keys and values need pages and scales of their own");
    AppendParams p;
    p.pages[0] = k_pages; p.pages[1] = v_pages; p.scales[0] = k_scales; p.scales[1] = v_scales; p.x[0] = k; p.x[1] = v;
    p.token_stride[0] = k_strides[0]; p.head_stride[0] = k_strides[1]; p.token_stride[1] = v_strides[0]; p.head_stride[1] = v_strides[1];
    p.slots = slots; p.status = status_dev; p.page_count = pages; p.heads = kv_heads; p.tokens = tokens;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    // few tokens: a warp for every run; many: runs are as long as pages, and a block that finds none costs its launch
    p.chunk = tokens <= 1024 ? CA_WARPS : CA_MAX_CHUNK;
    const dim3 grid(static_cast<unsigned>((tokens + p.chunk - 1) / p.chunk), static_cast<unsigned>(kv_heads));
    auto launch = [&](auto kernel) -> int {
        LaunchConfig lc(grid, CA_WARPS * 32, 0, stream);
        STOF_CUDA(cudaLaunchKernelEx(&lc.cfg, kernel, p));
        return STOF_OK;
    };
    const bool bf16 = dtype == STOF_DTYPE_BF16, e4m3 = cache_dtype == STOF_DTYPE_E4M3;
    if (head_dim == 64) {
        if (bf16) return e4m3 ? launch(cache_append_kernel<true, true, 64>) : launch(cache_append_kernel<true, false, 64>);
        return e4m3 ? launch(cache_append_kernel<false, true, 64>) : launch(cache_append_kernel<false, false, 64>);
    }
    if (bf16) return e4m3 ? launch(cache_append_kernel<true, true, 128>) : launch(cache_append_kernel<true, false, 128>);
    return e4m3 ? launch(cache_append_kernel<false, true, 128>) : launch(cache_append_kernel<false, false, 128>);
}
