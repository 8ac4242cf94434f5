// Rows of a table by id, scaled, and the table's gradient.
//
//   y[i] = scale table[ids[i]]                     0 for an id outside [0, vocab)
//   dtable[v] = scale sum over ids[i] = v of dy[i]  fp32 sums, rounded once; 0 for rows without ids
//
// The forward reads each id's row and is bound by HBM (by L2 where the table fits it).  The gradient
// sorts the ids (sort.hip) and sums runs of equal ones, so that no two workgroups add to one row and the
// result does not depend on timing:
//   runs   each group of lanes walks kRun sorted places; a row whose places all lie in one run is
//          written at once, one that crosses into the next leaves a partial sum (`tail` in the run
//          where it begins, `head` in every later run it reaches)
//   join   for every run whose last row goes on, adds the later runs' heads to its tail
#include "elements.h"
#include "sort.h"
#include "tiles.h"

namespace odie {
namespace {

constexpr int kEmbedBlock = 256;

struct LookupArgs {
    const void* table;
    const void* ids;
    void* out;
    int64_t n, vocab, stride;
    float scale;
    Divisor by_chunks;
    uint32_t block_rows;
    int id_bytes, width, chunks;
};

template <class T> __global__ __launch_bounds__(kEmbedBlock) void lookup_kernel(LookupArgs a) {
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.block_rows;
    const int64_t left = a.n - row0;
    const uint32_t items = (left < a.block_rows ? static_cast<uint32_t>(left) : a.block_rows) * a.chunks;
    for (uint32_t t = threadIdx.x; t < items; t += kEmbedBlock) {
        const uint32_t r = divide(t, a.by_chunks);
        const int column = static_cast<int>(t - r * a.chunks) * kPerVec<T>, count = a.width - column;
        const int64_t i = row0 + r;
        const int64_t id = a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
        vec16 v{};
        if (id >= 0 && id < a.vocab) {
            float f[kPerVec<T>];
            widen<T>(load_some(static_cast<const T*>(a.table) + id * a.stride + column, count), f);
#pragma unroll
            for (int e = 0; e < kPerVec<T>; ++e) f[e] *= a.scale;
            v = narrow<T>(f);
        }
        store_some(static_cast<T*>(a.out) + i * a.width + column, v, count);
    }
}

struct RunArgs {
    const void* up;           // [n][width], stride
    const int32_t* order;     // sorted place -> input position
    const int32_t* sorted;    // sorted place -> row; `vocab` for an id outside the table
    void* out;                // [vocab][width]
    float* head;              // [runs][columns]: fp32 sums, columns padded to whole chunks
    float* tail;
    int64_t n, vocab, stride, runs;
    float scale;
    int run;                  // sorted places a run
    int width, chunks, lanes; // lanes a run and block of columns
    int blocks;               // blocks of `lanes` chunks across the columns
};

template <class T> __device__ inline void add_to(float* sum, const vec16& v) {
    float f[kPerVec<T>];
    widen<T>(v, f);
#pragma unroll
    for (int e = 0; e < kPerVec<T>; ++e) sum[e] += f[e];
}

template <class T> __device__ inline void write_row(const RunArgs& a, int64_t row, int chunk, const float* sum) {
    float f[kPerVec<T>];
#pragma unroll
    for (int e = 0; e < kPerVec<T>; ++e) f[e] = sum[e] * a.scale;
    const int column = chunk * kPerVec<T>;
    store_some(static_cast<T*>(a.out) + row * a.width + column, narrow<T>(f), a.width - column);
}

template <class T> __device__ inline void keep(float* to, const RunArgs& a, int64_t run, int chunk, const float* sum) {
    float* p = to + (run * a.chunks + chunk) * kPerVec<T>;
#pragma unroll
    for (int e = 0; e < kPerVec<T>; e += 4)
        *reinterpret_cast<float4*>(p + e) = make_float4(sum[e], sum[e + 1], sum[e + 2], sum[e + 3]);
}

template <class T> __global__ __launch_bounds__(kEmbedBlock) void runs_kernel(RunArgs a) {
    const int64_t group = (static_cast<int64_t>(blockIdx.x) * kEmbedBlock + threadIdx.x) / a.lanes;
    const int64_t run = group / a.blocks;
    const int chunk = static_cast<int>(group % a.blocks) * a.lanes + static_cast<int>(threadIdx.x) % a.lanes;
    if (run >= a.runs || chunk >= a.chunks) return;
    const int64_t begin = run * a.run, end = begin + a.run < a.n ? begin + a.run : a.n;
    const T* up = static_cast<const T*>(a.up) + chunk * kPerVec<T>;
    const int count = a.width - chunk * kPerVec<T>;
    const int32_t before = begin > 0 ? a.sorted[begin - 1] : -1;
    const int32_t after = end < a.n ? a.sorted[end] : -1;
    constexpr int kAhead = 8;
    float sum[kPerVec<T>] = {};
    int32_t row = a.sorted[begin];
    bool first = true;   // the row began at or before this run's first place
    for (int64_t p = begin; p < end; p += kAhead) {
        int32_t rows[kAhead];
        vec16 v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t q = p + u < end ? p + u : end - 1;
            rows[u] = a.sorted[q];
            v[u] = load_some(up + a.order[q] * a.stride, count);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (p + u >= end) break;
            if (rows[u] != row) {
                if (row < a.vocab) {
                    if (first && row == before) keep<T>(a.head, a, run, chunk, sum);
                    else write_row<T>(a, row, chunk, sum);
                }
                row = rows[u];
                first = false;
#pragma unroll
                for (int e = 0; e < kPerVec<T>; ++e) sum[e] = 0.0f;
            }
            add_to<T>(sum, v[u]);
        }
    }
    if (row >= a.vocab) return;
    if (first && row == before) keep<T>(a.head, a, run, chunk, sum);
    else if (row == after) keep<T>(a.tail, a, run, chunk, sum);
    else write_row<T>(a, row, chunk, sum);
}

// One wave looks at 64 runs, then joins those that go on one after the other: its lanes take 64 / lanes
// of the heads at once, which are added pairwise at the end.
template <class T> __global__ __launch_bounds__(kEmbedBlock) void join_kernel(RunArgs a) {
    const int lane = static_cast<int>(threadIdx.x % 64);
    const int64_t wave = static_cast<int64_t>(blockIdx.x) * (kEmbedBlock / 64) + threadIdx.x / 64;
    const int64_t own = wave / a.blocks * 64 + lane;
    const int block = static_cast<int>(wave % a.blocks);
    bool goes_on = false;
    if (own < a.runs - 1) {
        const int64_t begin = own * a.run, end = begin + a.run;   // not the last run: whole
        const int32_t row = a.sorted[end - 1];
        goes_on = row < a.vocab && a.sorted[end] == row && (begin == 0 || a.sorted[begin - 1] != row);
    }
    for (uint64_t todo = __ballot(goes_on); todo; todo &= todo - 1) {
        const int64_t run = wave / a.blocks * 64 + __ffsll(static_cast<unsigned long long>(todo)) - 1;
        const int64_t from = (run + 1) * a.run;
        const int32_t row = a.sorted[from];
        int64_t low = from, high = a.n;   // the first place past the row
        while (low < high) {
            const int64_t mid = (low + high) / 2;
            if (a.sorted[mid] <= row) low = mid + 1; else high = mid;
        }
        const int64_t last = (low - 1) / a.run;   // heads of runs run + 1 .. last
        const int chunk = block * a.lanes + lane % a.lanes;
        float sum[kPerVec<T>] = {};
        if (chunk < a.chunks) {
            const int part = lane / a.lanes, parts = 64 / a.lanes;
            const int64_t pitch = static_cast<int64_t>(a.chunks) * kPerVec<T>;
            const float* head = a.head + static_cast<int64_t>(chunk) * kPerVec<T>;
            for (int64_t r = run + 1 + part; r <= last; r += parts)
#pragma unroll
                for (int e = 0; e < kPerVec<T>; ++e) sum[e] += head[r * pitch + e];
            if (part == 0)
#pragma unroll
                for (int e = 0; e < kPerVec<T>; ++e) sum[e] += a.tail[run * pitch + static_cast<int64_t>(chunk) * kPerVec<T> + e];
        }
        for (int m = a.lanes; m < 64; m *= 2)
#pragma unroll
            for (int e = 0; e < kPerVec<T>; ++e) sum[e] += __shfl_xor(sum[e], m);
        if (chunk < a.chunks && lane < a.lanes) write_row<T>(a, row, chunk, sum);
    }
}

__global__ __launch_bounds__(kEmbedBlock) void clear_kernel(char* data, int64_t bytes) {
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kEmbedBlock * 16;
    for (int64_t at = (static_cast<int64_t>(blockIdx.x) * kEmbedBlock + threadIdx.x) * 16; at < bytes; at += stride) {
        if (at + 16 <= bytes) {
            store16(data + at, vec16{});
        } else {
            for (int64_t i = at; i < bytes; ++i) data[i] = 0;
        }
    }
}

int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

int chunks_of(int64_t width, int dtype) {
    const int64_t per = 16 / dtype_bytes(dtype);
    return static_cast<int>((width + per - 1) / per);
}

// Lanes for a run: the most (up to 32) that keep three of four busy over whole blocks of columns.
int run_lanes(int chunks) {
    int best = 4;
    for (int lanes = 8; lanes <= 32; lanes *= 2)
        if (4 * chunks >= 3 * ((chunks + lanes - 1) / lanes * lanes)) best = lanes;
    return best;
}

// Sorted places a run: eight waves a CU, between 8 and 64 places.
int run_length(int64_t n, int chunks) {
    const int64_t wanted = n * chunks / (int64_t{8} * 64 * kCus);
    int run = 8;
    while (run < 64 && run < wanted) run *= 2;
    return run;
}

struct EmbedPlan {
    int64_t order, sorted, heads, sort;   // bytes
    int run, chunks;
    int64_t runs;
};

EmbedPlan embed_plan(int64_t n, int64_t vocab, int64_t width, int dtype) {
    EmbedPlan p{};
    p.chunks = chunks_of(width, dtype);
    p.run = run_length(n, p.chunks);
    p.runs = (n + p.run - 1) / p.run;
    p.order = padded(4 * n);
    p.sorted = padded(4 * n);
    p.heads = padded(p.runs * p.chunks * (16 / dtype_bytes(dtype)) * 4);
    p.sort = padded(sort_workspace(n, vocab));
    return p;
}

int check_embed(const std::string& what, int64_t n, int64_t vocab, int64_t width, int id_bytes, int dtype) {
    if (!known_dtype(dtype)) return fail(what + ": dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (check_sort(what.c_str(), SortKeys{nullptr, id_bytes, n, vocab})) return -1;
    if (width < 1 || width > 1 << 20) return fail(what + ": width must be within 1..2^20");
    return 0;
}

}  // namespace
}  // namespace odie

using namespace odie;

ODIE_API int odie_embed_forward(const void* table, int64_t table_stride, int64_t vocab, const void* ids, int id_bytes,
                                int64_t n, float scale, int64_t width, int dtype, void* out, uint64_t stream) {
    const std::string what = "odie_embed_forward";
    if (check_embed(what, n, vocab, width, id_bytes, dtype)) return -1;
    if (n == 0) return 0;
    if (!table || !ids || !out) return fail(what + ": null pointer");
    if (table_stride < width) return fail(what + ": rows overlap (a stride below the row's width)");
    LookupArgs a{};
    a.table = table;
    a.ids = ids;
    a.out = out;
    a.n = n;
    a.vocab = vocab;
    a.stride = table_stride;
    a.scale = scale;
    a.id_bytes = id_bytes;
    a.width = static_cast<int>(width);
    a.chunks = chunks_of(width, dtype);
    a.by_chunks = make_divisor(static_cast<uint32_t>(a.chunks));
    a.block_rows = a.chunks >= 1024 ? 1u : static_cast<uint32_t>(1024 / a.chunks);
    const uint32_t blocks = static_cast<uint32_t>((n + a.block_rows - 1) / a.block_rows);
    with_dtype(dtype, [&](auto t) { lookup_kernel<decltype(t)><<<blocks, kEmbedBlock, 0, as_stream(stream)>>>(a); });
    return check_launch("embed");
}

ODIE_API int64_t odie_embed_workspace(int64_t n, int64_t vocab, int64_t width, int dtype) {
    if (check_embed("odie_embed_workspace", n, vocab, width, 4, dtype)) return -1;
    const EmbedPlan p = embed_plan(n, vocab, width, dtype);
    return p.order + p.sorted + 2 * p.heads + p.sort;
}

ODIE_API int odie_embed_backward(const void* upstream, int64_t upstream_stride, const void* ids, int id_bytes,
                                 int64_t n, int64_t vocab, float scale, int64_t width, int dtype, void* dtable,
                                 void* workspace, int64_t workspace_bytes, uint64_t stream) {
    const std::string what = "odie_embed_backward";
    if (check_embed(what, n, vocab, width, id_bytes, dtype)) return -1;
    if (!dtable || (n > 0 && (!upstream || !ids))) return fail(what + ": null pointer");
    if (n > 0 && upstream_stride < width) return fail(what + ": rows overlap (a stride below the row's width)");
    const EmbedPlan p = embed_plan(n, vocab, width, dtype);
    const int64_t need = p.order + p.sorted + 2 * p.heads + p.sort;
    if (n > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0))
        return fail(what + ": needs a 256-byte aligned workspace of " + std::to_string(need) + " bytes");
    hipStream_t s = as_stream(stream);
    const int64_t bytes = vocab * width * dtype_bytes(dtype);
    const int64_t fill = (bytes + kEmbedBlock * 16 - 1) / (kEmbedBlock * 16);
    clear_kernel<<<static_cast<uint32_t>(fill > 16 * kCus ? 16 * kCus : fill), kEmbedBlock, 0, s>>>(static_cast<char*>(dtable), bytes);
    if (check_launch("embed gradient")) return -1;
    if (n == 0) return 0;
    char* scratch = static_cast<char*>(workspace);
    RunArgs a{};
    int32_t* order = reinterpret_cast<int32_t*>(scratch);
    int32_t* sorted = reinterpret_cast<int32_t*>(scratch + p.order);
    a.head = reinterpret_cast<float*>(scratch + p.order + p.sorted);
    a.tail = reinterpret_cast<float*>(scratch + p.order + p.sorted + p.heads);
    if (launch_sort(SortKeys{ids, id_bytes, n, vocab}, SortOut{order, sorted, nullptr, nullptr},
                    scratch + p.order + p.sorted + 2 * p.heads, s))
        return -1;
    a.up = upstream;
    a.order = order;
    a.sorted = sorted;
    a.out = dtable;
    a.n = n;
    a.vocab = vocab;
    a.stride = upstream_stride;
    a.runs = p.runs;
    a.run = p.run;
    a.scale = scale;
    a.width = static_cast<int>(width);
    a.chunks = p.chunks;
    a.lanes = run_lanes(p.chunks);
    a.blocks = (p.chunks + a.lanes - 1) / a.lanes;
    const int64_t threads = p.runs * a.blocks * a.lanes, waves = (p.runs + 63) / 64 * a.blocks;
    if (threads / kEmbedBlock >= int64_t{1} << 31) return fail(what + ": too many runs for one launch");
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        runs_kernel<T><<<static_cast<uint32_t>((threads + kEmbedBlock - 1) / kEmbedBlock), kEmbedBlock, 0, s>>>(a);
        if (p.runs > 1)
            join_kernel<T><<<static_cast<uint32_t>((waves + kEmbedBlock / 64 - 1) / (kEmbedBlock / 64)), kEmbedBlock, 0, s>>>(a);
    });
    return check_launch("embed gradient");
}
