// Block tables and slot maps of a paged cache from request lengths (integers, latency-bound: a few KB in, the slots out).
//
// A request's pages taken and given back, and its new tokens, are differences of rounded-up lengths; where they go are exclusive
// sums over the requests in front of it.  One cluster of thread blocks does the call in one launch: every block scans all
// requests for itself (a few KB from L2, cheaper than passing sums between blocks), then the warps of the cluster take requests in
// turn.  Pages given back have to be on the stack before they are taken again: a cluster barrier stands between the two, which is
// why the call stays inside one cluster.
#include "stof_host.h"
#include "stof_ptx.cuh"

namespace stof {
namespace {

constexpr int PT_THREADS = 1024, PT_WARPS = PT_THREADS / 32;
constexpr int PT_MAX_CLUSTER = 8;

struct PageTablesParams {
    const int *lengths, *held;
    int* block_table;
    long long table_stride;
    int* free_pages;
    const int* free_count;
    int *slots, *starts, *free_count_out, *missing_out;
    int* status;
    int requests, table_width, free_capacity, page_shift, slot_count;
};

struct Sums {
    unsigned take, give;                     // pages
    unsigned long long fresh;                // tokens
    __device__ __forceinline__ Sums operator+(const Sums& o) const { return {take + o.take, give + o.give, fresh + o.fresh}; }
};
__device__ __forceinline__ Sums shfl_up(const Sums& s, int d) {
    return {__shfl_up_sync(0xffffffffu, s.take, d), __shfl_up_sync(0xffffffffu, s.give, d), __shfl_up_sync(0xffffffffu, s.fresh, d)};
}

struct Request {                             // what the warps that serve it need
    int held, have, need;                    // tokens and pages before, pages after
    unsigned take_at, give_at;
    unsigned long long start;
    unsigned fresh;
};

__global__ void __launch_bounds__(PT_THREADS) page_tables_kernel(const PageTablesParams p) {
    __shared__ Request req[PT_THREADS];
    __shared__ Sums warp_sum[PT_WARPS];
    __shared__ unsigned long long totals[2];                 // pages taken, pages that rows are too short for (64 bits: lengths are not trusted)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dependency_wait();
    grid_launch_dependents();
    const bool muted = __syncthreads_or(failure_reported(p.status));        // one answer for the block: it has barriers ahead
    const int blocks = gridDim.x, rank = blockIdx.x;         // the grid is one cluster
    const int page = 1 << p.page_shift, chunks = (p.requests + PT_THREADS - 1) / PT_THREADS;
    if (threadIdx.x < 2) totals[threadIdx.x] = 0;
    __syncthreads();

    // requests [chunk * PT_THREADS, ..) into `req`, `before` = sums in front of them; returns the sums behind them
    auto scan = [&](int chunk, const Sums& before, bool count) -> Sums {
        const int r = chunk * PT_THREADS + static_cast<int>(threadIdx.x);
        Request q = {0, 0, 0, 0u, 0u, 0ull, 0u};
        Sums own = {0u, 0u, 0ull};
        if (r < p.requests) {
            const int len = max(p.lengths[r], 0);
            q.held = static_cast<int>(min(static_cast<long long>(max(p.held[r], 0)), static_cast<long long>(p.table_width) << p.page_shift));
            q.have = static_cast<int>((static_cast<long long>(q.held) + page - 1) >> p.page_shift);
            q.need = static_cast<int>((static_cast<long long>(len) + page - 1) >> p.page_shift);
            q.fresh = static_cast<unsigned>(max(len - q.held, 0));
            own = {static_cast<unsigned>(max(q.need - q.have, 0)), static_cast<unsigned>(max(q.have - q.need, 0)), q.fresh};
            if (count) {
                if (own.take > 0) atomicAdd(&totals[0], static_cast<unsigned long long>(own.take));
                if (q.need > p.table_width) atomicAdd(&totals[1], static_cast<unsigned long long>(q.need - p.table_width));
            }
        }
        Sums s = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const Sums o = shfl_up(s, d);
            if (lane >= d) s = s + o;
        }
        __syncthreads();                                     // the chunk before has been used
        if (lane == 31) warp_sum[warp] = s;
        __syncthreads();
        if (warp == 0) {
            Sums w = warp_sum[lane];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const Sums o = shfl_up(w, d);
                if (lane >= d) w = w + o;
            }
            warp_sum[lane] = w;
        }
        __syncthreads();
        Sums at = before;
        if (warp > 0) at = at + warp_sum[warp - 1];
        q.take_at = at.take + s.take - own.take;
        q.give_at = at.give + s.give - own.give;
        q.start = at.fresh + s.fresh - own.fresh;
        req[threadIdx.x] = q;
        const Sums after = before + warp_sum[PT_WARPS - 1];
        __syncthreads();
        return after;
    };
    const Sums none = {0u, 0u, 0ull};
    Sums all = none;
    for (int c = 0; c < chunks; ++c) all = scan(c, all, true);

    const int on_stack = min(max(*p.free_count, 0), p.free_capacity);
    const long long top = static_cast<long long>(on_stack) + all.give;
    long long missing = top > p.free_capacity ? p.free_capacity - top : 0;                   // negative: given back more than fits
    if (missing == 0) missing = max(static_cast<long long>(totals[0]) - top, 0ll) + static_cast<long long>(totals[1]);
    const bool good = missing == 0 && !muted;

    // every warp of the cluster walks its requests of a chunk that is in `req`
    auto each = [&](auto&& f) {
        Sums at = none;
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1) at = scan(c, at, false);                                         // (a single chunk is still there)
            const int n = min(p.requests - c * PT_THREADS, PT_THREADS);
            for (int i = rank * PT_WARPS + warp; i < n; i += blocks * PT_WARPS) f(c * PT_THREADS + i, req[i]);
        }
    };
    if (good && all.give > 0)
        each([&](int r, const Request& q) {
            const int* row = p.block_table + r * p.table_stride;
            for (int b = q.need + lane; b < q.have; b += 32) p.free_pages[on_stack + q.give_at + (b - q.need)] = row[b];
        });
    if (blocks > 1) cluster_sync_all();                      // given before taken; and everyone has read *free_count
    else __syncthreads();
    if (!muted)
        each([&](int r, const Request& q) {
            int* row = p.block_table + r * p.table_stride;
            if (lane == 0) p.starts[r] = static_cast<int>(min(q.start, 0x7FFFFFFFull));
            // the page of block b >= have: popped from the stack
            auto taken = [&](int b) { return p.free_pages[top - 1 - q.take_at - (b - q.have)]; };
            if (good)
                for (int b = q.have + lane; b < q.need; b += 32) row[b] = taken(b);
            const unsigned long long room = q.start < static_cast<unsigned>(p.slot_count) ? p.slot_count - q.start : 0ull;
            const unsigned n = static_cast<unsigned>(min(static_cast<unsigned long long>(q.fresh), room));
            for (unsigned i = lane; i < n; i += 32) {
                int slot = -1;
                if (good) {
                    const int at = q.held + static_cast<int>(i), b = at >> p.page_shift;
                    slot = ((b < q.have ? row[b] : taken(b)) << p.page_shift) + (at & (page - 1));
                }
                p.slots[q.start + i] = slot;
            }
        });
    if (!muted) {
        for (unsigned long long t = all.fresh + rank * PT_THREADS + threadIdx.x; t < static_cast<unsigned>(p.slot_count); t += blocks * PT_THREADS)
            p.slots[t] = -1;
        if (rank == 0 && threadIdx.x == 0) {
            p.starts[p.requests] = static_cast<int>(min(all.fresh, 0x7FFFFFFFull));
            *p.free_count_out = good ? static_cast<int>(top - all.take) : on_stack;
            *p.missing_out = static_cast<int>(max(min(missing, 0x7FFFFFFFll), -0x7FFFFFFFll));
        }
    }
}

}  // namespace
}  // namespace stof

using namespace stof;

extern "C" int stof_page_tables(const int* lengths, const int* held, int requests, int* block_table, long long table_stride, int table_width,
                                int* free_pages, int free_capacity, const int* free_count, int page_size, int* slots, int slot_count, int* starts,
                                int* free_count_out, int* missing_out, int* status_dev, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    STOF_REQUIRE(requests >= 0 && table_width >= 0 && free_capacity >= 0 && slot_count >= 0, "page_tables: negative size");
    STOF_REQUIRE(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128, "page_tables: page size %d not in {16, 32, 64, 128}", page_size);
    STOF_REQUIRE(requests == 0 || (lengths && held), "page_tables: null lengths or held");
    STOF_REQUIRE(requests == 0 || table_width == 0 || (block_table && table_stride >= table_width), "page_tables: null block table, or a row stride below its width");
    STOF_REQUIRE((free_pages || free_capacity == 0) && free_count && free_count_out && missing_out && starts, "page_tables: null pointer");
    STOF_REQUIRE(slots || slot_count == 0, "page_tables: null slots");
    PageTablesParams p;
    p.lengths = lengths; p.held = held; p.block_table = block_table; p.table_stride = table_stride; p.free_pages = free_pages;
    p.free_count = free_count; p.slots = slots; p.starts = starts; p.free_count_out = free_count_out; p.missing_out = missing_out; p.status = status_dev;
    p.requests = requests; p.table_width = table_width; p.free_capacity = free_capacity; p.slot_count = slot_count;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    const int cluster = requests > PT_WARPS || slot_count > 4096 ? PT_MAX_CLUSTER : 1;
    LaunchConfig lc(dim3(static_cast<unsigned>(cluster)), PT_THREADS, 0, stream, static_cast<unsigned>(cluster));
    STOF_CUDA(cudaLaunchKernelEx(&lc.cfg, page_tables_kernel, p));
    return STOF_OK;
}
