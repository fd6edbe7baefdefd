// Page tables, slots and positions of a step, from the streams' lengths.
//
// Of a stream with p tokens in the cache and f to come, pages of P tokens, a
// window W and sinks in the first S pages, the table's entries are
//   kept    below ceil(p / P), and with a window only below S or from
//           floor((p - W + 1) / P) on;
//   needed  below ceil((p + f) / P).
// What is held of a table row follows from two numbers a stream, so no table is
// searched: what goes back and what is taken are ranges of entries, and prefix
// sums over the streams give each of them its place in the stack of free pages.
//
// Bound by latency: one workgroup does the table (lengths, three scans, the few
// entries that change), and the tokens too where they are few; more of them are
// a second launch over all CUs, bound by 8 bytes written a token.

#include "attention.hpp"

#include <algorithm>

namespace mlvc_hip {
namespace {

struct PlanArgs {
    int streams, pages, page, tokens, window, sink_pages, table_stride, slots_here;
    std::int32_t* table;
    int2* held;
    std::int32_t* free_pages;
    std::int32_t* free_count;
    const std::int32_t* past;
    const std::int32_t* fresh;
    const unsigned long long* seen;
    std::int32_t* lengths;
    std::int32_t* starts;
    std::int32_t* slots;
    std::int32_t* positions;
    std::int32_t* lacking;
};

__device__ __forceinline__ int pages_of(const PlanArgs& a, std::int64_t tokens)
{
    return static_cast<int>((static_cast<unsigned>(tokens) + static_cast<unsigned>(a.page) - 1u) / static_cast<unsigned>(a.page));
}

// A stream's tokens, and the entries of its row that change.
struct Row {
    int past = 0, fresh = 0, kept = 0, back = 0, front = 0, need = 0;
    bool fits = true;
    // Entries that go back: `count` from `first` on, of sinks, behind the context, before the window.
    int first[3] = {}, count[3] = {};
    __device__ Row() = default;
    __device__ Row(const PlanArgs& a, int past_, int fresh_, int2 held)
    {
        past = fresh_ < 0 ? 0 : max(past_, 0);
        fresh = max(fresh_, 0);
        kept = pages_of(a, past);
        const int end = min(max(held.y, 0), a.table_stride), begin = max(held.x, 0);
        const int window = a.window ? max(a.sink_pages, static_cast<int>(static_cast<unsigned>(max(past - a.window + 1, 0)) / static_cast<unsigned>(a.page))) : 0;
        const int outside = max(begin, a.sink_pages);
        auto range = [&](int i, int from, int to) { first[i] = from, count[i] = max(to - from, 0); };
        range(0, kept, min(a.sink_pages, end));
        range(1, max(kept, outside), end);
        range(2, outside, min(min(window, kept), end));
        back = min(end, kept);
        front = a.window ? max(window, min(begin, kept)) : 0;
        const std::int64_t all = static_cast<std::int64_t>(past) + fresh;
        fits = all <= static_cast<std::int64_t>(a.table_stride) * a.page;
        need = fits ? max(pages_of(a, all) - back, 0) : 0;
    }
    __device__ int returned() const { return count[0] + count[1] + count[2]; }
};

__device__ __forceinline__ int chain_or_depth(const PlanArgs& a, int token, int i, int drafts)
{
    if (!a.seen) return i;
    unsigned long long others = a.seen[token];
    if (drafts < 64) others &= (1ull << drafts) - 1;
    if (i < 64) others &= ~(1ull << i);
    return __popcll(others);
}

// Sum over this thread and those before it in the workgroup; `total` in all.
__device__ std::int64_t scan(std::int64_t x, std::int64_t* waves, std::int64_t& total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const std::int64_t up = __shfl_up(x, o);
        if (lane >= o) x += up;
    }
    __syncthreads();  // before the last scan's sums
    if (lane == 63) waves[wave] = x;
    __syncthreads();
    std::int64_t before = 0;
    total = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) {
        if (w < wave) before += waves[w];
        total += waves[w];
    }
    return before + x;
}

__device__ __forceinline__ int capped(std::int64_t x) { return static_cast<int>(min(x, static_cast<std::int64_t>(INT_MAX))); }

constexpr int kMostThreads = 1024;

// One workgroup, a stream a thread; more streams than threads by turns.
__global__ __launch_bounds__(kMostThreads) void plan_kernel(PlanArgs a)
{
    __shared__ std::int64_t waves[kMostThreads / 64];
    const int tid = threadIdx.x, threads = blockDim.x;
    auto row_of = [&](int n) { return n < a.streams ? Row(a, a.past[n], a.fresh[n], a.held[n]) : Row(); };
    const std::int64_t count = min(max(*a.free_count, 0), a.pages);

    // Pages that go back: the first entry on top.
    std::int64_t returned = 0;
    for (int b = 0; b < a.streams; b += threads) {
        std::int64_t total;
        scan(row_of(b + tid).returned(), waves, total);
        returned += total;
    }
    const std::int64_t top = min(count + returned, static_cast<std::int64_t>(a.pages));
    std::int64_t carry = 0;
    if (returned > 0)
        for (int b = 0; b < a.streams; b += threads) {
            const Row r = row_of(b + tid);
            std::int64_t total, at = scan(r.returned(), waves, total) - r.returned() + carry;
            carry += total;
            std::int32_t* const row = a.table + static_cast<std::int64_t>(b + tid) * a.table_stride;
            for (int k = 0; k < 3; ++k)
                for (int e = 0; e < r.count[k]; ++e, ++at) {
                    const std::int64_t to = count + returned - 1 - at;
                    if (to < a.pages) a.free_pages[to] = row[r.first[k] + e];
                    row[r.first[k] + e] = -1;
                }
        }
    __syncthreads();

    // Pages that are taken, and the lengths. `held` changes last: a turn reads its own streams' only.
    std::int64_t needed = 0, tokens = 0, taken = 0;
    int lacking = 0;
    for (int b = 0; b < a.streams; b += threads) {
        const int n = b + tid;
        const Row r = row_of(n);
        std::int64_t total, all_fresh, none;
        const std::int64_t upto = scan(r.need, waves, total) + needed, until = scan(r.fresh, waves, all_fresh) + tokens;
        const bool served = r.fits && (r.need == 0 || upto <= top);
        const int got = served ? r.need : 0;
        if (n < a.streams) {
            std::int32_t* const row = a.table + static_cast<std::int64_t>(n) * a.table_stride;
            for (int e = 0; e < got; ++e) {
                const int page = a.free_pages[top - 1 - (upto - r.need + e)];
                row[r.back + e] = page >= 0 && page < a.pages ? page : -1;
            }
            a.lengths[n] = r.past + (served ? r.fresh : 0);
            a.starts[n + 1] = capped(until);
            a.held[n] = make_int2(r.front, r.back + got);
        }
        scan(got, waves, none);
        taken += none;
        scan(n < a.streams && !served, waves, none);
        lacking += static_cast<int>(none);
        needed += total, tokens += all_fresh;
    }
    if (tid == 0) {
        a.starts[0] = 0;
        *a.free_count = static_cast<std::int32_t>(top - taken);
        *a.lacking = lacking;
    }
}

__global__ __launch_bounds__(256) void slots_kernel(PlanArgs a)
{
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.tokens) return;
    int slot = -1, position = 0;
    if (t < a.starts[a.streams]) {
        int lo = 0, hi = a.streams;  // the stream that starts at or before the token, and ends behind it
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (a.starts[mid] <= t) lo = mid;
            else hi = mid;
        }
        const int past = max(a.past[lo], 0), i = t - a.starts[lo];
        if (a.lengths[lo] > past) {
            const unsigned place = static_cast<unsigned>(past) + i, entry = place / static_cast<unsigned>(a.page);
            const int page = a.table[static_cast<std::int64_t>(lo) * a.table_stride + entry];
            if (page >= 0) slot = page * a.page + static_cast<int>(place - entry * a.page);
        }
        position = past + chain_or_depth(a, t, i, a.starts[lo + 1] - a.starts[lo]);
    }
    a.slots[t] = slot;
    if (a.positions) a.positions[t] = position;
}

void kv_plan(const mlvc_hip_kv_plan_desc* d, hipStream_t s)
{
    const char* op = "kv_plan";
    require(d != nullptr, op, "no descriptor");
    require(d->streams >= 0 && d->tokens >= 0 && d->table_stride >= 0, op, "negative size");
    require(d->window >= 0 && d->sinks >= 0, op, "window and sinks must not be negative");
    require(d->page_size >= 16 && d->page_size % 16 == 0, op, "page_size must be a multiple of 16");
    require(d->pages >= 0 && static_cast<std::int64_t>(d->pages) * d->page_size <= INT_MAX, op, "pages * page_size must be below 2^31");
    require(static_cast<std::int64_t>(d->streams) * d->table_stride <= INT_MAX, op, "streams * table_stride must be below 2^31");
    require(d->held && d->free_count && d->past && d->fresh && d->lengths && d->starts && d->lacking && (d->slots || d->tokens == 0) &&
                (d->table || d->streams == 0 || d->table_stride == 0) && (d->free_pages || d->pages == 0), op, "null tensor");
    require(d->lengths != d->past && d->lengths != d->fresh, op, "lengths must not be past or fresh");
    for (const void* p : {static_cast<const void*>(d->table), static_cast<const void*>(d->free_pages), static_cast<const void*>(d->free_count),
                          static_cast<const void*>(d->past), static_cast<const void*>(d->fresh), static_cast<const void*>(d->lengths),
                          static_cast<const void*>(d->starts), static_cast<const void*>(d->slots), static_cast<const void*>(d->positions),
                          static_cast<const void*>(d->lacking)})
        require(aligned_to<4>(p), op, "a tensor is not aligned to its values");
    require(aligned_to<8>(d->held) && aligned_to<8>(d->seen), op, "held and seen must be 8-byte aligned");
    PlanArgs a{};
    a.streams = d->streams, a.pages = d->pages, a.page = d->page_size, a.tokens = d->tokens, a.window = d->window;
    a.sink_pages = d->window ? static_cast<int>((static_cast<std::int64_t>(d->sinks) + d->page_size - 1) / d->page_size) : 0;
    a.table = d->table, a.table_stride = d->table_stride, a.held = reinterpret_cast<int2*>(d->held);
    a.free_pages = d->free_pages, a.free_count = d->free_count, a.past = d->past, a.fresh = d->fresh;
    a.seen = reinterpret_cast<const unsigned long long*>(d->seen);
    a.lengths = d->lengths, a.starts = d->starts, a.slots = d->slots, a.positions = d->positions, a.lacking = d->lacking;
    const int threads = std::min(kMostThreads, std::max(64, (d->streams + 63) / 64 * 64));
    plan_kernel<<<1, threads, 0, s>>>(a);
    check(hipGetLastError(), "kv_plan launch");
    if (d->tokens == 0) return;
    slots_kernel<<<(d->tokens + 255u) / 256u, 256, 0, s>>>(a);
    check(hipGetLastError(), "kv_plan slots launch");
}

}  // namespace
}  // namespace mlvc_hip

using namespace mlvc_hip;

extern "C" int mlvc_hip_kv_plan(const mlvc_hip_kv_plan_desc* desc, mlvc_hip_stream s)
{
    return guard([&] { kv_plan(desc, to_stream(s)); });
}
