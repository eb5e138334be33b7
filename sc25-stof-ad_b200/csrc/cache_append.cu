// New keys and values into the slots of a paged 8-bit cache, one scale per page and head (HBM-bound for prompts, latency-bound for
// the tokens of a step).
//
// A run is a stretch of tokens whose slots follow one another inside a page; its scale needs the largest magnitude of all its
// rows, so a run belongs to one warp (up to four tokens) or one thread block: the rows are read once, held in registers as they
// came, reduced, and written as entries.  Runs are found from the slots alone: a thread block looks at a few neighbouring tokens of
// one head and serves the runs that begin there.
#include "cache_common.cuh"
#include "stof_host.h"
#include "stof_ptx.cuh"

namespace stof {
namespace {

constexpr int CA_WARPS = 4;
constexpr int CA_SHORT = 4;                  // tokens up to which a warp serves a run alone
constexpr int CA_MAX_CHUNK = 16;

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

    static __device__ __forceinline__ float magnitude(const uint4& u) {
        auto pair = [](uint32_t w) {
            const float2 f = unpack_pair<BF16>(w);
            return fmaxf(fabsf(f.x), fabsf(f.y));
        };
        return fmaxf(fmaxf(pair(u.x), pair(u.y)), fmaxf(pair(u.z), pair(u.w)));
    }
    static __device__ __forceinline__ uint2 entries(const uint4& u, float inv) {
        auto four = [&](uint32_t a, uint32_t b) {
            const float2 f = unpack_pair<BF16>(a), g = unpack_pair<BF16>(b);
            return quantise2<E4M3>(f.x, f.y, inv) | (quantise2<E4M3>(g.x, g.y, inv) << 16);
        };
        return make_uint2(four(u.x, u.y), four(u.z, u.w));
    }
};

// One run: tokens [token, token + n) into rows [row, row + n) of a page.  `part` of `parts` warps work on it (1: this warp alone),
// NV loads hold a warp's share.
template <bool BF16, bool E4M3, int D, int NV>
__device__ __forceinline__ void write_run(const AppendParams& p, int side, int head, int token, int n, int page, int row, int part, int parts, float* shared) {
    using R = Rows<BF16, E4M3, D>;
    const int lane = threadIdx.x & 31, sub = lane / R::LANES, col = lane % R::LANES;
    const uint16_t* x = static_cast<const uint16_t*>(p.x[side]) + head * p.head_stride[side] + col * 8;
    const long long at = static_cast<long long>(page) * p.heads + head;
    uint8_t* entries = static_cast<uint8_t*>(p.pages[side]) + ((at << p.page_shift) + row) * D;
    float* scale = p.scales[side] + at;
    uint4 v[NV];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int r = (i * parts + part) * R::EACH + sub;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < n) v[i] = __ldca(reinterpret_cast<const uint4*>(x + (token + r) * p.token_stride[side]));
    }
    const float old = row > 0 ? *scale : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) top = fmaxf(top, R::magnitude(v[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (parts > 1) {
        if (lane == 0) shared[part] = top;
        __syncthreads();                                     // (and everyone has read the old scale)
        top = fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
    }
    float now = top * (1.0f / entry_max<E4M3>());
    if (now < 1.17549435e-38f) now = 0.f;
    now = fmaxf(now, old);
    const float inv = now > 0.f ? 1.0f / now : 0.f;
    if (part == 0 && lane == 0) *scale = now;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int r = (i * parts + part) * R::EACH + sub;
        if (r < n) *reinterpret_cast<uint2*>(entries + static_cast<size_t>(r) * D + col * 8) = R::entries(v[i], inv);
    }
    if (row > 0 && now > old) {                              // the entries in front of the run, rounded again to the new scale
        const float ratio = old / now;
        uint4* front = reinterpret_cast<uint4*>(entries - static_cast<size_t>(row) * D);
        for (int i = part * 32 + lane; i < row * D / 16; i += parts * 32) {
            const uint4 u = front[i];
            auto again = [&](uint32_t w) {
                uint32_t lo, hi;
                entries_to_half<E4M3>(w, lo, hi);
                const float2 a = unpack_pair<false>(lo), b = unpack_pair<false>(hi);
                return quantise2<E4M3>(a.x, a.y, ratio) | (quantise2<E4M3>(b.x, b.y, ratio) << 16);
            };
            front[i] = make_uint4(again(u.x), again(u.y), again(u.z), again(u.w));
        }
    }
}

template <bool BF16, bool E4M3, int D>
__global__ void __launch_bounds__(CA_WARPS * 32) cache_append_kernel(const AppendParams p) {
    __shared__ int run_token[CA_MAX_CHUNK], run_length[CA_MAX_CHUNK], runs;
    __shared__ float shared[CA_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = blockIdx.y, side = blockIdx.z, page = 1 << p.page_shift;
    grid_dependency_wait();
    grid_launch_dependents();
    if (__syncthreads_or(failure_reported(p.status))) return;
    const long long slot_end = static_cast<long long>(p.page_count) << p.page_shift;
    if (warp == 0) {
        const int t = blockIdx.x * p.chunk + lane;
        bool first = false;
        if (lane < p.chunk && t < p.tokens) {
            const int s = p.slots[t];
            first = s >= 0 && (t == 0 || s != p.slots[t - 1] + 1 || (s & (page - 1)) == 0);
            if (first && s >= slot_end) {
                if (p.status != nullptr) atomicCAS(p.status, 0, STATUS_BAD_INDEX);
                first = false;
            }
        }
        const unsigned found = __ballot_sync(0xffffffffu, first);
        if (first) run_token[__popc(found & ((1u << lane) - 1u))] = t;
        if (lane == 0) runs = __popc(found);
    }
    __syncthreads();
    const int count = runs;
    for (int i = warp; i < count; i += CA_WARPS) {           // lengths, and the short runs at once
        const int t = run_token[i], s = p.slots[t], most = min(page - (s & (page - 1)), p.tokens - t);
        int n = 1;
        for (int at = 1; at < most; at += 32) {
            const bool on = at + lane < most && p.slots[t + at + lane] == s + at + lane;
            const unsigned run = __ballot_sync(0xffffffffu, on);
            const int more = run == 0xffffffffu ? 32 : __ffs(~run) - 1;
            n += more;
            if (more < 32) break;
        }
        if (lane == 0) run_length[i] = n;
        if (n <= CA_SHORT)
            write_run<BF16, E4M3, D, CA_SHORT / Rows<BF16, E4M3, D>::EACH>(p, side, head, t, n, s >> p.page_shift, s & (page - 1), 0, 1, shared);
    }
    __syncthreads();
    for (int i = 0; i < count; ++i) {
        const int n = run_length[i];
        if (n <= CA_SHORT) continue;
        const int t = run_token[i], s = p.slots[t];
        constexpr int SHARE = CA_WARPS * Rows<BF16, E4M3, D>::EACH;      // rows of one load of the whole block
        if (n <= 32)
            write_run<BF16, E4M3, D, 32 / SHARE>(p, side, head, t, n, s >> p.page_shift, s & (page - 1), warp, CA_WARPS, shared);
        else
            write_run<BF16, E4M3, D, 128 / SHARE>(p, side, head, t, n, s >> p.page_shift, s & (page - 1), warp, CA_WARPS, shared);
        __syncthreads();                                     // `shared` is free again
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
    AppendParams p;
    p.pages[0] = k_pages; p.pages[1] = v_pages; p.scales[0] = k_scales; p.scales[1] = v_scales; p.x[0] = k; p.x[1] = v;
    p.token_stride[0] = k_strides[0]; p.head_stride[0] = k_strides[1]; p.token_stride[1] = v_strides[0]; p.head_stride[1] = v_strides[1];
    p.slots = slots; p.status = status_dev; p.page_count = pages; p.heads = kv_heads; p.tokens = tokens;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    // few tokens: a warp for every run; many: runs are as long as pages, and a block that finds none costs its launch
    p.chunk = tokens <= 1024 ? CA_WARPS : CA_MAX_CHUNK;
    const dim3 grid(static_cast<unsigned>((tokens + p.chunk - 1) / p.chunk), static_cast<unsigned>(kv_heads), 2);
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
