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
// Bound by latency: one workgroup does the table (lengths, scans, the few entries
// that change, dealt to all threads), and the tokens too where they are few; more
// of them are a second launch over all CUs. 64 streams of one token: 4.3 us in the
// kernel, of them 3 for an empty launch; 64 ragged prompts of up to 2040 tokens
// behind a window, 61 thousand slots and 4 thousand pages handed out, 10.7 + 3.4
// (37 + 5 with a stream's pages by one thread).

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
    std::int32_t* placed;
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
        fits = all <= min(static_cast<std::int64_t>(a.table_stride) * a.page, static_cast<std::int64_t>(INT_MAX));  // lengths have 32 bits
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

constexpr int kMostThreads = 1024;
constexpr int kTokensHere = 4096;  // tokens that the one workgroup takes too
constexpr int kAtOnce = 4;         // pages of a thread that are on their way at once

// Three sums over this thread and those before it in the workgroup, of 32, 32 and
// 64 bits, and their totals.
struct Sums {
    int a, b;
    std::int64_t c;
};
__device__ __forceinline__ Sums scan(int a, int b, int c, Sums (&waves)[kMostThreads / 64], Sums& total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums s{wave_scan(a), wave_scan(b), (static_cast<std::int64_t>(wave_scan(c >> 16)) << 16) + wave_scan(c & 0xffff)};
    if (lane == 63) waves[wave] = s;
    __syncthreads();
    total = {};
    for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) {
        const Sums x = waves[w];
        if (w == wave) s.a += total.a, s.b += total.b, s.c += total.c;
        total.a += x.a, total.b += x.b, total.c += x.c;
    }
    return s;
}

__device__ __forceinline__ int capped(std::int64_t x) { return static_cast<int>(min(x, static_cast<std::int64_t>(INT_MAX))); }

// The first of n ascending sums that is above x.
__device__ __forceinline__ int above(const int* sums, int n, int x)
{
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (sums[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Calls take(several) for a thread's entries of n that are dealt to all threads,
// a few at once; several(f) calls f(u, e) for each of them. What the first of its
// calls reads is on its way for all before the next one uses it.
template <class F>
__device__ __forceinline__ void each_entry(int n, int threads, F&& take)
{
    if (n <= threads) {
        const int e = threadIdx.x;
        if (e < n) take([&](auto&& f) { f(0, e); });
        return;
    }
    for (int e0 = threadIdx.x; e0 < n; e0 += kAtOnce * threads)
        take([&](auto&& f) {
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (e0 + u * threads < n) f(u, e0 + u * threads);
        });
}

// Slot and position of the i-th new token, the t-th of all, of a stream with a row of the table.
__device__ __forceinline__ void place_token(const PlanArgs& a, int t, const std::int32_t* row, int past, int i, int drafts, bool served)
{
    const unsigned place = static_cast<unsigned>(past) + i, entry = place / static_cast<unsigned>(a.page);
    const int page = served ? row[entry] : -1;
    a.slots[t] = page < 0 ? -1 : page * a.page + static_cast<int>(place - entry * a.page);
    if (a.positions) a.positions[t] = past + chain_or_depth(a, t, i, drafts);
}

// One workgroup, a stream a thread; more streams than threads by turns. Entries
// that change, and tokens, are dealt to all threads by the sums before them.
__global__ __launch_bounds__(kMostThreads) void plan_kernel(PlanArgs a)
{
    __shared__ Sums waves[kMostThreads / 64];
    __shared__ int upto[kMostThreads], first[3][kMostThreads], count[2][kMostThreads];
    __shared__ int taken_here, lacking_here;
    const int tid = threadIdx.x, threads = blockDim.x;
    auto row_of = [&](int n) { return n < a.streams ? Row(a, a.past[n], a.fresh[n], a.held[n]) : Row(); };
    auto table = [&](int n) { return a.table + static_cast<std::int64_t>(n) * a.table_stride; };
    const bool one_turn = a.streams <= threads;
    Row r = row_of(tid);
    const int held = min(max(*a.free_count, 0), a.pages);
    if (tid == 0) lacking_here = 0;

    // Pages that go back: the first entry on top.
    Sums total, sums = scan(r.returned(), r.need, r.fresh, waves, total);
    std::int64_t returned = total.a;
    if (!one_turn)
        for (int b = threads; b < a.streams; b += threads) {
            Sums more;
            __syncthreads();
            scan(row_of(b + tid).returned(), 0, 0, waves, more);
            returned += more.a;
        }
    const int top = static_cast<int>(min(held + returned, static_cast<std::int64_t>(a.pages)));
    if (returned > 0) {
        std::int64_t before = 0;
        for (int b = 0; b < a.streams; b += threads) {
            Row back = r;
            Sums all = total, here = sums;
            if (!one_turn) {
                back = row_of(b + tid);
                __syncthreads();
                here = scan(back.returned(), 0, 0, waves, all);
            }
            upto[tid] = here.a;
            for (int k = 0; k < 3; ++k) first[k][tid] = back.first[k];
            for (int k = 0; k < 2; ++k) count[k][tid] = back.count[k];
            __syncthreads();
            const int here_streams = min(threads, a.streams - b);
            each_entry(all.a, threads, [&](auto&& several) {
                std::int32_t* entry[kAtOnce];
                std::int32_t page[kAtOnce];
                several([&](int u, int e) {
                    const int i = above(upto, here_streams, e);
                    int k = 0, at = e - (i ? upto[i - 1] : 0);
                    if (at >= count[0][i]) at -= count[0][i], k = 1;
                    if (k == 1 && at >= count[1][i]) at -= count[1][i], k = 2;
                    entry[u] = table(b + i) + first[k][i] + at;
                    page[u] = *entry[u];
                });
                several([&](int u, int e) {
                    const std::int64_t to = held + returned - 1 - (before + e);
                    if (to < a.pages) a.free_pages[to] = page[u];
                    *entry[u] = -1;
                });
            });
            before += all.a;
        }
    }

    // Pages that are taken, the lengths, and where few the tokens. `held` changes
    // last: a turn reads its own streams' only.
    std::int64_t needed = 0, tokens = 0;
    int taken = 0;
    for (int b = 0; b < a.streams; b += threads) {
        const int n = b + tid;
        __syncthreads();  // what the last turn left in LDS is read; what went back is there
        if (!one_turn) {
            r = row_of(n);
            sums = scan(0, r.need, r.fresh, waves, total);
        }
        const std::int64_t until = needed + sums.b;
        const bool served = r.fits && (r.need == 0 || until <= top);
        const int got = served ? r.need : 0;
        upto[tid] = sums.b, first[0][tid] = r.back;
        if (tid == 0) taken_here = 0;
        __syncthreads();
        if (got) atomicMax(&taken_here, sums.b);
        const unsigned long long short_of = __ballot(!served);
        if ((tid & 63) == 0 && short_of) atomicAdd(&lacking_here, __popcll(short_of));
        if (n < a.streams) {
            a.lengths[n] = r.past + (served ? r.fresh : 0);
            if (a.placed) a.placed[n] = served ? r.fresh : 0;
            a.starts[n + 1] = capped(tokens + sums.c);
            a.held[n] = make_int2(r.front, r.back + got);
        }
        __syncthreads();
        // The streams that are served are those up to the last sum within the pool.
        const int now = taken_here, here_streams = min(threads, a.streams - b);
        each_entry(now, threads, [&](auto&& several) {
            std::int32_t page[kAtOnce];
            several([&](int u, int e) { page[u] = a.free_pages[top - 1 - needed - e]; });
            several([&](int u, int e) {
                const int i = above(upto, here_streams, e);
                table(b + i)[first[0][i] + e - (i ? upto[i - 1] : 0)] = page[u] >= 0 && page[u] < a.pages ? page[u] : -1;
            });
        });
        taken += now;
        needed += total.b, tokens += total.c;
        if (a.slots_here) {  // one turn
            __syncthreads();
            first[0][tid] = r.past, first[1][tid] = served, first[2][tid] = r.fresh;
            upto[tid] = capped(sums.c);
            __syncthreads();
            for (int t = tid; t < a.tokens; t += threads) {
                if (t >= total.c) {
                    a.slots[t] = -1;
                    if (a.positions) a.positions[t] = 0;
                    continue;
                }
                const int i = above(upto, here_streams, t);
                place_token(a, t, table(i), first[0][i], t - (i ? upto[i - 1] : 0), first[2][i], first[1][i]);
            }
        }
    }
    if (tid == 0) {
        a.starts[0] = 0;
        *a.free_count = top - taken;
        *a.lacking = lacking_here;
    }
}

__global__ __launch_bounds__(256) void slots_kernel(PlanArgs a)
{
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.tokens) return;
    if (t >= a.starts[a.streams]) {
        a.slots[t] = -1;
        if (a.positions) a.positions[t] = 0;
        return;
    }
    const int n = above(a.starts + 1, a.streams, t), start = a.starts[n], past = max(a.past[n], 0);
    place_token(a, t, a.table + static_cast<std::int64_t>(n) * a.table_stride, past, t - start, a.starts[n + 1] - start, a.lengths[n] > past);
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
    require(!d->placed || (d->placed != d->past && d->placed != d->fresh && d->placed != d->lengths), op, "placed must not be past, fresh or lengths");
    for (const void* p : {static_cast<const void*>(d->table), static_cast<const void*>(d->free_pages), static_cast<const void*>(d->free_count),
                          static_cast<const void*>(d->past), static_cast<const void*>(d->fresh), static_cast<const void*>(d->lengths),
                          static_cast<const void*>(d->starts), static_cast<const void*>(d->slots), static_cast<const void*>(d->positions),
                          static_cast<const void*>(d->lacking), static_cast<const void*>(d->placed)})
        require(aligned_to<4>(p), op, "a tensor is not aligned to its values");
    require(aligned_to<8>(d->held) && aligned_to<8>(d->seen), op, "held and seen must be 8-byte aligned");
    PlanArgs a{};
    a.streams = d->streams, a.pages = d->pages, a.page = d->page_size, a.tokens = d->tokens, a.window = d->window;
    a.sink_pages = d->window ? static_cast<int>((static_cast<std::int64_t>(d->sinks) + d->page_size - 1) / d->page_size) : 0;
    a.table = d->table, a.table_stride = d->table_stride, a.held = reinterpret_cast<int2*>(d->held);
    a.free_pages = d->free_pages, a.free_count = d->free_count, a.past = d->past, a.fresh = d->fresh;
    a.seen = reinterpret_cast<const unsigned long long*>(d->seen);
    a.lengths = d->lengths, a.starts = d->starts, a.slots = d->slots, a.positions = d->positions, a.lacking = d->lacking, a.placed = d->placed;
    // A stream a thread, and enough of them for the pages and the tokens.
    const std::int64_t work = std::max<std::int64_t>(d->streams, d->tokens / 4);
    const int threads = static_cast<int>(std::min<std::int64_t>(kMostThreads, std::max<std::int64_t>(64, (work + 63) / 64 * 64)));
    a.slots_here = d->streams > 0 && d->streams <= threads && d->tokens <= kTokensHere;
    plan_kernel<<<1, threads, 0, s>>>(a);
    check(hipGetLastError(), "kv_plan launch");
    if (d->tokens == 0 || a.slots_here) return;
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
