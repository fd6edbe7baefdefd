// The paged cache of keys and values: rows quantised as they are written, and
// read back.
//
//   a = max |x|,  stored = round(x A / a),  scale = a / A,  value = stored scale
//
// x A is exact in FP32 (11 + 7 bits), and x A / a, a quotient of integers of
// at most 18 and 11 bits up to a power of two, is either a tie between two
// stored values or at least 2^-19 of itself away from one. An FP32 quotient
// therefore rounds to the stored value that exact arithmetic gives if it is
// exact at the ties: t = x A (1 / a) corrected once by its remainder,
// t + (x A - t a) (1 / a), is (the remainder is exact), with three operations
// a value instead of a full division's ten.
//
// Bound by memory: a row is read and written once. 4 streams of 1020 new
// tokens, 8 heads of 128, k and v to E4M3: 25 MB in 8.5 us; 2039 tokens of each
// read back, 50 MB, 10.9 us. 64 rows take 2.8 and 2.6 us, a launch's time. A row
// for each group of lanes: several, the next one asked for early, took as long.

#include "attention.hpp"

namespace mlvc_hip {

void check_cache(const mlvc_hip_kv_cache* c, const char* op)
{
    require(c != nullptr, op, "no cache");
    require(c->kind == MLVC_KV_F16 || c->kind == MLVC_KV_E4M3 || c->kind == MLVC_KV_INT8, op, "unknown cache kind");
    require(c->heads >= 1 && c->heads <= 65535, op, "cache heads must be 1..65535");
    require(c->head_dim >= 8 && c->head_dim <= kMaxHeadDim && c->head_dim % 8 == 0, op,
            "cache head_dim must be a multiple of 8 up to 512");
    require(c->page_size >= 16 && c->page_size % 16 == 0, op, "page_size must be a multiple of 16");
    require(c->pages >= 0 && static_cast<std::int64_t>(c->pages) * c->page_size <= INT_MAX, op,
            "pages * page_size must be below 2^31");
    if (c->pages == 0) return;
    require(c->k && c->v && aligned16(c->k) && aligned16(c->v), op, "cache tensors must be 16-byte aligned");
    if (c->kind != MLVC_KV_F16)
        require(c->k_scale && c->v_scale && aligned16(c->k_scale) && aligned16(c->v_scale), op,
                "cache scales must be 16-byte aligned");
}

namespace {

constexpr int kBlock = 256;
constexpr float kLevelE4m3 = 448.0f, kLevelInt8 = 127.0f;

struct RowsArgs {
    std::uint8_t* cache[2];  // k, v
    float* scale[2];
    std::uint16_t* x[2];
    std::int64_t stride[2];
    const std::int32_t* slots;
    unsigned rows;           // tokens * heads
    int heads, dim, page, slot_count;
};

// Row of the cache (of all its heads' rows) of a slot's head, or -1.
__device__ __forceinline__ std::int64_t cache_row(const RowsArgs& a, std::int32_t slot, int head)
{
    if (slot < 0 || slot >= a.slot_count) return -1;
    const int page = static_cast<int>(static_cast<unsigned>(slot) / static_cast<unsigned>(a.page));
    return (static_cast<std::int64_t>(page) * a.heads + head) * a.page + (slot - page * a.page);
}

struct Quantiser {
    float level, top, inv, scale;
    // bits: the row's largest magnitude as FP16 bits, above 0x7bff if it
    // holds an infinity or NaN.
    __device__ Quantiser(int kind, std::uint32_t bits)
    {
        level = kind == MLVC_KV_INT8 ? kLevelInt8 : kLevelE4m3;
        const bool finite = bits < 0x7c00u;
        top = finite ? h2f(static_cast<std::uint16_t>(bits)) : 1.0f;
        inv = bits && finite ? 1.0f / top : 0.0f;
        scale = finite ? top / level : __builtin_nanf("");
    }
    __device__ float operator()(float x) const
    {
        const float v = x * level, t = v * inv;
        return fmaf(fmaf(-t, top, v), inv, t);
    }
};

// Four stored values as bytes.
__device__ __forceinline__ std::uint32_t bytes_of(int kind, float a, float b, float c, float d)
{
    if (kind == MLVC_KV_INT8) {
        // 1.5 * 2^23 + t leaves round(t), ties to even, in the low byte.
        constexpr float kMagic = 12582912.0f;
        const std::uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(b + kMagic), __float_as_uint(a + kMagic), 0x0c0c0400u),
                            cd = __builtin_amdgcn_perm(__float_as_uint(d + kMagic), __float_as_uint(c + kMagic), 0x04000c0cu);
        return ab | cd;
    }
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<std::uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}

__device__ __forceinline__ void values_of(int kind, std::uint32_t v, float* f)
{
    if (kind == MLVC_KV_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = static_cast<float>(static_cast<std::int8_t>(v >> (8 * i)));
        return;
    }
    typedef float floatx2 __attribute__((ext_vector_type(2)));
    const floatx2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(v), false),
                  hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(v), true);
    f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
}

__device__ __forceinline__ std::uint32_t magnitude2(std::uint32_t a, std::uint32_t b)
{
    typedef std::uint16_t u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(std::uint32_t,
                              __builtin_elementwise_max(__builtin_bit_cast(u16x2, a & 0x7fff7fffu), __builtin_bit_cast(u16x2, b & 0x7fff7fffu)));
}

// LANES lanes hold a row, 8 values each (heads of at most 8 * LANES). blockIdx.y: k or v.
// What is read does not wait for what is known later: lanes past the row read
// its first values, and the arguments of k and v are both there.
template <int KIND, int LANES>
__global__ __launch_bounds__(kBlock) void kv_write_kernel(RowsArgs a)
{
    const bool is_v = blockIdx.y != 0;
    const int lane = threadIdx.x % LANES;
    const bool mine = lane * 8 < a.dim;
    const int d0 = mine ? lane * 8 : 0;
    const unsigned row = blockIdx.x * (kBlock / LANES) + threadIdx.x / LANES;
    if (row >= a.rows) return;
    const unsigned token = row / static_cast<unsigned>(a.heads);
    const int head = static_cast<int>(row - token * a.heads);
    const std::int32_t slot = a.slots[token];
    u32x4 v = *reinterpret_cast<const u32x4*>((is_v ? a.x[1] : a.x[0]) + token * (is_v ? a.stride[1] : a.stride[0]) + head * a.dim + d0);
    const std::int64_t to = cache_row(a, slot, head);
    if (to < 0) return;
    std::uint8_t* const cache = is_v ? a.cache[1] : a.cache[0];
    if constexpr (KIND == MLVC_KV_F16) {
        if (mine) *reinterpret_cast<u32x4*>(cache + 2 * (to * a.dim + d0)) = v;
    } else {
        // Magnitudes as integers, so that an infinity or NaN is the largest.
        const std::uint32_t m2 = magnitude2(magnitude2(v[0], v[1]), magnitude2(v[2], v[3]));
        const Quantiser q(KIND, group_max<LANES>(max(m2 & 0xffffu, m2 >> 16)));
        std::uint32_t b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            b[i] = bytes_of(KIND, q(lo_f16(v[2 * i])), q(hi_f16(v[2 * i])), q(lo_f16(v[2 * i + 1])), q(hi_f16(v[2 * i + 1])));
        if (mine) *reinterpret_cast<uint2*>(cache + to * a.dim + d0) = make_uint2(b[0], b[1]);
        if (lane == 0) (is_v ? a.scale[1] : a.scale[0])[to] = q.scale;
    }
}

template <int KIND, int LANES>
__global__ __launch_bounds__(kBlock) void kv_read_kernel(RowsArgs a)
{
    const bool is_v = blockIdx.y != 0;
    const int lane = threadIdx.x % LANES, d0 = lane * 8;
    const unsigned row = blockIdx.x * (kBlock / LANES) + threadIdx.x / LANES;
    if (row >= a.rows || d0 >= a.dim) return;
    const unsigned token = row / static_cast<unsigned>(a.heads);
    const int head = static_cast<int>(row - token * a.heads);
    const std::int64_t from = cache_row(a, a.slots[token], head);
    const std::uint8_t* const cache = is_v ? a.cache[1] : a.cache[0];
    u32x4 v = {0, 0, 0, 0};
    if (from >= 0) {
        if constexpr (KIND == MLVC_KV_F16) {
            v = *reinterpret_cast<const u32x4*>(cache + 2 * (from * a.dim + d0));
        } else {
            const uint2 b = *reinterpret_cast<const uint2*>(cache + from * a.dim + d0);
            const float scale = (is_v ? a.scale[1] : a.scale[0])[from];
            float f[8];
            values_of(KIND, b.x, f);
            values_of(KIND, b.y, f + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = pack_rounded(f[2 * i] * scale, f[2 * i + 1] * scale);
        }
    }
    *reinterpret_cast<u32x4*>((is_v ? a.x[1] : a.x[0]) + token * (is_v ? a.stride[1] : a.stride[0]) + head * a.dim + d0) = v;
}

// Rows off 16 bytes, or heads of over 256 or under 40 values: one wave a row, value by value.
template <int KIND, bool WRITE>
__global__ __launch_bounds__(kBlock) void kv_any_kernel(RowsArgs a)
{
    const int of = blockIdx.y, lane = threadIdx.x & 63;
    const unsigned row = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    const unsigned token = row / static_cast<unsigned>(a.heads);
    const int head = static_cast<int>(row - token * a.heads);
    std::uint16_t* x = a.x[of] + token * a.stride[of] + static_cast<std::int64_t>(head) * a.dim;
    const std::int64_t at = cache_row(a, a.slots[token], head);
    if (WRITE && at < 0) return;
    std::uint8_t* kept = a.cache[of] + (at < 0 ? 0 : at * a.dim * (KIND == MLVC_KV_F16 ? 2 : 1));
    if constexpr (KIND == MLVC_KV_F16) {
        std::uint16_t* h = reinterpret_cast<std::uint16_t*>(kept);
        for (int d = lane; d < a.dim; d += 64) {
            if (WRITE) h[d] = x[d];
            else x[d] = at < 0 ? 0 : h[d];
        }
    } else if constexpr (WRITE) {
        std::uint32_t m = 0;
        for (int d = lane; d < a.dim; d += 64) m = max(m, x[d] & 0x7fffu);
        const Quantiser q(KIND, group_max<64>(m));
        for (int d = lane; d < a.dim; d += 64) kept[d] = static_cast<std::uint8_t>(bytes_of(KIND, q(h2f(x[d])), 0.0f, 0.0f, 0.0f));
        if (lane == 0) a.scale[of][at] = q.scale;
    } else {
        const float scale = at < 0 ? 0.0f : a.scale[of][at];
        for (int d = lane; d < a.dim; d += 64) x[d] = at < 0 ? 0 : f2h(opaque(from_byte(KIND, kept[d]) * scale));
    }
}

template <int KIND, bool WRITE, int LANES>
void launch_rows(const RowsArgs& a, hipStream_t s)
{
    const dim3 grid(static_cast<unsigned>((a.rows + kBlock / LANES - 1) / (kBlock / LANES)), 2);
    if constexpr (WRITE) kv_write_kernel<KIND, LANES><<<grid, kBlock, 0, s>>>(a);
    else kv_read_kernel<KIND, LANES><<<grid, kBlock, 0, s>>>(a);
}

template <int KIND, bool WRITE>
void launch(const RowsArgs& a, bool vectors, hipStream_t s)
{
    if (!vectors) kv_any_kernel<KIND, WRITE><<<dim3(static_cast<unsigned>((a.rows + 3) / 4), 2), kBlock, 0, s>>>(a);
    else if (a.dim <= 64) launch_rows<KIND, WRITE, 8>(a, s);
    else if (a.dim <= 128) launch_rows<KIND, WRITE, 16>(a, s);
    else launch_rows<KIND, WRITE, 32>(a, s);
}

template <bool WRITE>
void run(const mlvc_hip_kv_cache* c, const mlvc_hip_kv_rows* r, hipStream_t s)
{
    const char* op = WRITE ? "kv_write" : "kv_read";
    check_cache(c, op);
    require(r != nullptr, op, "no rows");
    require(r->tokens >= 0, op, "negative token count");
    const std::int64_t row = static_cast<std::int64_t>(c->heads) * c->head_dim;
    require(r->k_stride >= row && r->v_stride >= row, op, "a stride is shorter than a row of heads");
    if (r->tokens == 0) return;
    require(r->k && r->v && r->slots, op, "null tensor");
    require(aligned2(r->k) && aligned2(r->v), op, "a tensor is not aligned to its FP16 values");
    RowsArgs a{};
    a.cache[0] = static_cast<std::uint8_t*>(c->k), a.cache[1] = static_cast<std::uint8_t*>(c->v);
    a.scale[0] = c->k_scale, a.scale[1] = c->v_scale;
    a.x[0] = static_cast<std::uint16_t*>(r->k), a.x[1] = static_cast<std::uint16_t*>(r->v);
    a.stride[0] = r->k_stride, a.stride[1] = r->v_stride;
    a.slots = r->slots;
    const std::int64_t rows = static_cast<std::int64_t>(r->tokens) * c->heads;
    require(launchable(rows / 4 + 1, kBlock), op, "too many rows in one call");
    a.rows = static_cast<unsigned>(rows);
    a.heads = c->heads, a.dim = c->head_dim, a.page = c->page_size, a.slot_count = c->pages * c->page_size;
    const bool vectors = c->head_dim > 32 && c->head_dim <= 256 && vector_rows(r->k, r->k_stride) && vector_rows(r->v, r->v_stride);
    if (c->kind == MLVC_KV_F16) launch<MLVC_KV_F16, WRITE>(a, vectors, s);
    else if (c->kind == MLVC_KV_E4M3) launch<MLVC_KV_E4M3, WRITE>(a, vectors, s);
    else launch<MLVC_KV_INT8, WRITE>(a, vectors, s);
    check(hipGetLastError(), WRITE ? "kv_write launch" : "kv_read launch");
}

struct KeepArgs {
    std::uint8_t* cache[2];  // k, v
    float* scale[2];
    const std::int32_t* table;
    const std::int32_t* starts;
    const std::int32_t* lengths;
    const std::int32_t* kept;
    const std::int32_t* placed;
    std::int32_t* lengths_out;
    int streams, heads, row_bytes, page, pages, table_stride, kept_stride, quantised;
};

constexpr int kMostKept = 64;

// A workgroup for the kept rows of one head of a stream. The places they go to
// may be those of others that move too, so a group of columns is read for all
// rows before any of it is written; columns do not meet. Bound by latency, of the
// lengths, the table and the rows one after the other: 64 streams that keep 31 of
// 64 drafts, 8 heads of 128, FP16, 16 MB read and written in 4.7 us; 8 that keep 4
// of 8 in 3.6.
template <typename T>
__global__ __launch_bounds__(kBlock) void kv_keep_kernel(KeepArgs a)
{
    __shared__ std::int64_t from[kMostKept], to[kMostKept];
    __shared__ int kept_count;
    const int head = blockIdx.x % a.heads, stream = blockIdx.x / a.heads, tid = threadIdx.x;
    if (tid < 64) {
        int drafts = max(a.starts[stream + 1] - a.starts[stream], 0);
        if (a.placed) drafts = min(drafts, max(a.placed[stream], 0));
        const int past = max(a.lengths[stream], 0) - drafts;
        const int draft = tid < a.kept_stride ? a.kept[static_cast<std::int64_t>(stream) * a.kept_stride + tid] : -1;
        const unsigned long long ends = ~__ballot(draft >= 0 && draft < drafts);
        const int count = ends ? __builtin_ctzll(ends) : 64;
        auto row = [&](int i) -> std::int64_t {
            const std::int64_t place = static_cast<std::int64_t>(past) + i;
            if (place < 0 || place >= static_cast<std::int64_t>(a.table_stride) * a.page) return -1;
            const int entry = static_cast<int>(static_cast<unsigned>(place) / static_cast<unsigned>(a.page));
            const int page = a.table[static_cast<std::int64_t>(stream) * a.table_stride + entry];
            return page < 0 || page >= a.pages ? -1 : (static_cast<std::int64_t>(page) * a.heads + head) * a.page + (place - static_cast<std::int64_t>(entry) * a.page);
        };
        const bool moves = tid < count && draft != tid;
        const std::int64_t f = moves ? row(draft) : -1, t = moves ? row(tid) : -1;
        from[tid] = t < 0 ? -1 : f;
        to[tid] = t;
        if (tid == 0) {
            kept_count = count;
            if (head == 0) a.lengths_out[stream] = max(past + count, 0);
        }
    }
    __syncthreads();
    const int count = kept_count;
    if (count == 0) return;
    const int pieces = a.row_bytes / static_cast<int>(sizeof(T)), columns = kBlock / count;  // of a turn
    const int row = tid / columns, column = tid - row * columns;
    const bool mine = row < count && from[min(row, kMostKept - 1)] >= 0;
    for (int c = 0; c < pieces; c += columns) {
        const bool here = mine && c + column < pieces;
        T k{}, v{};
        if (here) {
            const std::int64_t at = from[row] * a.row_bytes + static_cast<std::int64_t>(c + column) * sizeof(T);
            k = *reinterpret_cast<const T*>(a.cache[0] + at), v = *reinterpret_cast<const T*>(a.cache[1] + at);
        }
        __syncthreads();
        if (here) {
            const std::int64_t at = to[row] * a.row_bytes + static_cast<std::int64_t>(c + column) * sizeof(T);
            *reinterpret_cast<T*>(a.cache[0] + at) = k, *reinterpret_cast<T*>(a.cache[1] + at) = v;
        }
    }
    if (a.quantised && tid < kMostKept) {  // one wave: reads before writes
        const bool here = tid < count && from[tid] >= 0;
        const float k = here ? a.scale[0][from[tid]] : 0.0f, v = here ? a.scale[1][from[tid]] : 0.0f;
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (here) a.scale[0][to[tid]] = k, a.scale[1][to[tid]] = v;
    }
}

void kv_keep(const mlvc_hip_kv_keep_desc* d, hipStream_t s)
{
    const char* op = "kv_keep";
    require(d != nullptr, op, "no descriptor");
    check_cache(d->cache, op);
    require(d->streams >= 0 && d->table_stride >= 0, op, "negative size");
    require(d->kept_stride >= 0 && d->kept_stride <= kMostKept, op, "kept_stride must be 0..64");
    if (d->streams == 0) return;
    require(d->starts && d->lengths && d->lengths_out && (d->kept || d->kept_stride == 0) && (d->table || d->table_stride == 0), op, "null tensor");
    require(d->lengths_out != d->lengths && d->lengths_out != d->starts && d->lengths_out != d->placed, op,
            "lengths_out must not be lengths, starts or placed");
    for (const std::int32_t* p : {d->table, d->starts, d->lengths, d->kept, d->placed, static_cast<const std::int32_t*>(d->lengths_out)})
        require(aligned_to<4>(p), op, "a tensor is not aligned to its values");
    const mlvc_hip_kv_cache* c = d->cache;
    const std::int64_t grid = static_cast<std::int64_t>(d->streams) * c->heads;
    require(launchable(grid, kBlock), op, "too many streams and heads in one call");
    KeepArgs a{};
    a.cache[0] = static_cast<std::uint8_t*>(c->k), a.cache[1] = static_cast<std::uint8_t*>(c->v);
    a.scale[0] = c->k_scale, a.scale[1] = c->v_scale;
    a.table = d->table, a.starts = d->starts, a.lengths = d->lengths, a.kept = d->kept, a.placed = d->placed, a.lengths_out = d->lengths_out;
    a.streams = d->streams, a.heads = c->heads, a.page = c->page_size, a.pages = c->pages, a.table_stride = d->table_stride;
    a.kept_stride = d->kept_stride, a.quantised = c->kind != MLVC_KV_F16;
    a.row_bytes = c->head_dim * (a.quantised ? 1 : 2);
    if (a.row_bytes % 16 == 0) kv_keep_kernel<u32x4><<<static_cast<unsigned>(grid), kBlock, 0, s>>>(a);
    else kv_keep_kernel<uint2><<<static_cast<unsigned>(grid), kBlock, 0, s>>>(a);
    check(hipGetLastError(), "kv_keep launch");
}

size_t values_of_cache(const mlvc_hip_kv_cache* c)
{
    return static_cast<size_t>(c->pages) * c->heads * c->page_size;
}

}  // namespace
}  // namespace mlvc_hip

using namespace mlvc_hip;

extern "C" {

size_t mlvc_hip_kv_cache_bytes(const mlvc_hip_kv_cache* c)
{
    if (!c || c->pages <= 0 || c->heads <= 0 || c->page_size <= 0 || c->head_dim <= 0) return 0;
    return values_of_cache(c) * c->head_dim * (c->kind == MLVC_KV_F16 ? 2 : 1);
}

size_t mlvc_hip_kv_cache_scale_bytes(const mlvc_hip_kv_cache* c)
{
    if (!c || c->kind == MLVC_KV_F16 || c->pages <= 0 || c->heads <= 0 || c->page_size <= 0) return 0;
    return values_of_cache(c) * sizeof(float);
}

int mlvc_hip_kv_write(const mlvc_hip_kv_cache* cache, const mlvc_hip_kv_rows* rows, mlvc_hip_stream s)
{
    return guard([&] { run<true>(cache, rows, to_stream(s)); });
}

int mlvc_hip_kv_read(const mlvc_hip_kv_cache* cache, const mlvc_hip_kv_rows* rows, mlvc_hip_stream s)
{
    return guard([&] { run<false>(cache, rows, to_stream(s)); });
}

int mlvc_hip_kv_keep(const mlvc_hip_kv_keep_desc* desc, mlvc_hip_stream s)
{
    return guard([&] { kv_keep(desc, to_stream(s)); });
}

}  // extern "C"
