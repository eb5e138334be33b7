// Block tables and slot maps of a paged cache from request lengths (integers, latency-bound: a few KB in, the slots out).
//
// A request's pages taken and given back, and its new tokens, are differences of rounded-up lengths; where they go are exclusive
// sums over the requests in front of it.  One cluster of thread blocks does the call in one launch: every block scans all
// requests for itself (a few KB from L2, cheaper than passing sums between blocks), then the warps of the cluster take requests in
// turn.  Pages given back have to be on the stack before they are taken again: a cluster barrier stands between the two, which is
// why this stays inside one cluster.  What is done for a request is mostly a page and a token: its thread does that itself; what takes
// longer (a prompt, a request that leaves) is done by warps.  The slots of many tokens are written by a second kernel over the whole
// GPU, which looks its requests up in the running counts.
//
// Measured: 256 requests that take a token each or leave 6.2 to 6.4 us (with 256 threads 9.7: a request that leaves is a warp's work, and waits
// for one), 1000 that come, go and take prompts of hundreds of tokens 11.4 to 11.8 us; the launches and the
// chain lengths - sums - stack - table are all of it (a block scans 1000 requests in about 2 us; with sums by atomics of 64 bits in shared
// memory, or loads behind stores that they cannot pass, the second took 32 us).
#include "stof_host.h"
#include "stof_ptx.cuh"

namespace stof {
namespace {

constexpr int PT_THREADS = 1024, PT_WARPS = PT_THREADS / 32;
constexpr int PT_MAX_CLUSTER = 8;
constexpr int PT_FEW = 4;                    // pages or tokens up to which a request's thread sees to them itself
constexpr int PT_MANY = 4096;                // tokens from which on their slots are a kernel of their own

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

// put(i, get(i)) for i = first, first + step, .. < n, eight on their way at a time: the compiler may not move a load over a store that it
// cannot tell apart from it
template <class Get, class Put>
__device__ __forceinline__ void move_all(int first, int step, int n, Get&& get, Put&& put) {
    for (int i0 = first; i0 < n; i0 += 8 * step) {
        int v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i0 + j * step < n) v[j] = get(i0 + j * step);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i0 + j * step < n) put(i0 + j * step, v[j]);
    }
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
    __shared__ unsigned long long beyond;                    // pages that rows are too short for (64 bits: lengths are not trusted)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dependency_wait();
    grid_launch_dependents();
    // asked for now, with the lengths of the first requests, and looked at behind the sums: every load that waits for another is 0.4 us
    const bool failed = failure_reported(p.status);
    const int free_count = __ldca(p.free_count);
    const int blocks = gridDim.x, rank = blockIdx.x;         // the grid is one cluster
    const int page = 1 << p.page_shift, chunks = (p.requests + PT_THREADS - 1) / PT_THREADS;
    if (threadIdx.x == 0) beyond = 0;
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
            if (count && q.need > p.table_width) atomicAdd(&beyond, static_cast<unsigned long long>(q.need - p.table_width));
            q.need = min(q.need, p.table_width);             // (sums of what rows hold fit 32 bits: the table has fewer entries)
            own = {static_cast<unsigned>(max(q.need - q.have, 0)), static_cast<unsigned>(max(q.have - q.need, 0)), q.fresh};
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

    const bool muted = __syncthreads_or(failed);             // one answer for the block: it has barriers ahead
    const int on_stack = min(max(free_count, 0), p.free_capacity);
    const long long top = static_cast<long long>(on_stack) + all.give;
    long long missing = top > p.free_capacity ? p.free_capacity - top : 0;                   // negative: given back more than fits
    if (missing == 0) missing = max(static_cast<long long>(all.take + beyond) - top, 0ll) + static_cast<long long>(beyond);
    const bool good = missing == 0 && !muted;

    // f(request, q, first, step) for the requests of every chunk: by the request's thread (0, 1) where `small`, else by a warp (lane, 32)
    auto each = [&](auto&& small, auto&& f) {
        Sums at = none;
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1) at = scan(c, at, false);                                         // (a single chunk is still there)
            const int n = min(p.requests - c * PT_THREADS, PT_THREADS);
            const int mine = threadIdx.x;
            if (mine < n && mine % blocks == rank && small(req[mine])) f(c * PT_THREADS + mine, req[mine], 0, 1);
            for (int i = rank * PT_WARPS + warp; i < n; i += blocks * PT_WARPS)
                if (!small(req[i])) f(c * PT_THREADS + i, req[i], lane, 32);
        }
    };
    if (good && all.give > 0)
        each([](const Request& q) { return q.have - q.need <= PT_FEW; },
             [&](int r, const Request& q, int first, int step) {
                 const int* row = p.block_table + r * p.table_stride;
                 int* to = p.free_pages + on_stack + q.give_at;
                 move_all(first, step, q.have - q.need, [&](int i) { return row[q.need + i]; }, [&](int i, int v) { to[i] = v; });
             });
    if (blocks > 1) cluster_sync_all();                      // given before taken; and everyone has read *free_count
    else __syncthreads();
    if (muted) return;
    const bool slots_here = p.slots != nullptr;
    each([&](const Request& q) { return q.need - q.have <= PT_FEW && (!slots_here || q.fresh <= PT_FEW); },
         [&](int r, const Request& q, int first, int step) {
             int* row = p.block_table + r * p.table_stride;
             if (first == 0) p.starts[r] = static_cast<int>(min(q.start, 0x7FFFFFFFull));
             // the page of block b >= have: popped from the stack
             const int* from = p.free_pages + (top - 1 - q.take_at);
             auto taken = [&](int b) { return *(from - (b - q.have)); };
             if (good) move_all(first, step, q.need - q.have, [&](int i) { return *(from - i); }, [&](int i, int v) { row[q.have + i] = v; });
             if (!slots_here) return;
             const unsigned long long room = q.start < static_cast<unsigned>(p.slot_count) ? p.slot_count - q.start : 0ull;
             const unsigned n = static_cast<unsigned>(min(static_cast<unsigned long long>(q.fresh), room));
             for (unsigned i = first; i < n; i += step) {
                 int slot = -1;
                 if (good) {
                     const int at = q.held + static_cast<int>(i), b = at >> p.page_shift;
                     slot = ((b < q.have ? row[b] : taken(b)) << p.page_shift) + (at & (page - 1));
                 }
                 p.slots[q.start + i] = slot;
             }
         });
    if (slots_here)
        for (unsigned long long t = all.fresh + rank * PT_THREADS + threadIdx.x; t < static_cast<unsigned>(p.slot_count); t += blocks * PT_THREADS)
            p.slots[t] = -1;
    if (rank == 0 && threadIdx.x == 0) {
        p.starts[p.requests] = static_cast<int>(min(all.fresh, 0x7FFFFFFFull));
        *p.free_count_out = good ? static_cast<int>(top - all.take) : on_stack;
        *p.missing_out = static_cast<int>(max(min(missing, 0x7FFFFFFFll), -0x7FFFFFFFll));
    }
}

// The slots of many tokens, four to a thread, from the tables that page_tables_kernel left.
__global__ void __launch_bounds__(256) page_slots_kernel(const PageTablesParams p, int* slots) {
    grid_dependency_wait();
    grid_launch_dependents();
    if (failure_reported(p.status)) return;
    const int t0 = static_cast<int>(blockIdx.x * 256 + threadIdx.x) * 4, page = 1 << p.page_shift;
    if (t0 >= p.slot_count) return;
    const bool good = *p.missing_out == 0;
    int r = 0;                                               // the last request that begins at t0 or in front of it
    for (int n = p.requests; n > 1;) {
        const int half = n >> 1;
        if (p.starts[r + half] <= t0) r += half;
        n -= half;
    }
    int out[4], from = 0, behind = 0, held = 0;
    const int* row = nullptr;
    auto request = [&] {
        from = p.starts[r];
        behind = p.starts[r + 1];
        held = static_cast<int>(min(static_cast<long long>(max(p.held[r], 0)), static_cast<long long>(p.table_width) << p.page_shift));
        row = p.block_table + r * p.table_stride;
    };
    if (p.requests > 0) request();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = t0 + i;
        while (t >= behind && r + 1 < p.requests) {          // (requests without new tokens are passed over)
            ++r;
            request();
        }
        out[i] = -1;
        if (good && t < behind) {
            const int at = held + (t - from);
            out[i] = (row[at >> p.page_shift] << p.page_shift) + (at & (page - 1));
        }
    }
    if (t0 + 4 <= p.slot_count) {
        *reinterpret_cast<int4*>(slots + t0) = make_int4(out[0], out[1], out[2], out[3]);
    } else {
        for (int i = 0; t0 + i < p.slot_count; ++i) slots[t0 + i] = out[i];
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
    STOF_REQUIRE(static_cast<long long>(requests) * table_width < (1ll << 31), "page_tables: a block table of 2^31 entries or more");
    STOF_REQUIRE((free_pages || free_capacity == 0) && free_count && free_count_out && missing_out && starts, "page_tables: null pointer");
    STOF_REQUIRE(slots || slot_count == 0, "page_tables: null slots");
    PageTablesParams p;
    p.lengths = lengths; p.held = held; p.block_table = block_table; p.table_stride = table_stride; p.free_pages = free_pages;
    p.free_count = free_count; p.slots = slots; p.starts = starts; p.free_count_out = free_count_out; p.missing_out = missing_out; p.status = status_dev;
    p.requests = requests; p.table_width = table_width; p.free_capacity = free_capacity; p.slot_count = slot_count;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    // slots of many tokens: a kernel of their own, which stores 16 bytes at a time
    const bool apart = slot_count >= PT_MANY && aligned16(slots);
    if (apart) p.slots = nullptr;
    // A step (a token or two for each request) is done by the requests' own threads: one block, which also starts faster than a cluster.
    // Else warps see to prompts and to requests that leave, and there are more of them in a cluster.
    const int cluster = requests <= PT_THREADS && slot_count <= 2 * requests ? 1 : requests > 4 * PT_WARPS || (!apart && slot_count >= PT_MANY) ? PT_MAX_CLUSTER : 1;
    LaunchConfig lc(dim3(static_cast<unsigned>(cluster)), PT_THREADS, 0, stream, static_cast<unsigned>(cluster));
    STOF_CUDA(cudaLaunchKernelEx(&lc.cfg, page_tables_kernel, p));
    if (apart) {
        LaunchConfig ls(dim3(static_cast<unsigned>((static_cast<long long>(slot_count) + 1023) / 1024)), 256, 0, stream);
        STOF_CUDA(cudaLaunchKernelEx(&ls.cfg, page_slots_kernel, p, slots));
    }
    return STOF_OK;
}
