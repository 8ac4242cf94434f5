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
// 4M ids of 16384 rows, 32 bf16 columns: lookup 88 us (3.4 TB/s), gradient 223: the sort 91 (scattered stores of 8
// bytes), runs 95 (rows of 64 bytes in the ids' order, 2.8 TB/s), join 35 (one row a run or less: its latency).
// 300007 ids on few of 65032 rows, 97 fp32 columns: 28, and sort 33, runs 38, join 21 (the longest row's chain).
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

template <class T, bool kStream> __global__ __launch_bounds__(kEmbedBlock) void lookup_kernel(LookupArgs a) {
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.block_rows;
    const int64_t left = a.n - row0;
    const uint32_t items = (left < a.block_rows ? static_cast<uint32_t>(left) : a.block_rows) * a.chunks;
    constexpr int kAhead = 4;   // chunks a thread has in flight
    for (uint32_t t = threadIdx.x; t < items; t += kAhead * kEmbedBlock) {
        vec16 v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t item = t + u * kEmbedBlock < items ? t + u * kEmbedBlock : t;
            const uint32_t r = divide(item, a.by_chunks);
            const int64_t i = row0 + r;
            const int64_t id = a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
            v[u] = vec16{};
            if (id >= 0 && id < a.vocab)
                v[u] = load_chunk(static_cast<const T*>(a.table) + id * a.stride, static_cast<int>(item - r * a.chunks), a.width);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t item = t + u * kEmbedBlock;
            if (item >= items) break;
            const uint32_t r = divide(item, a.by_chunks);
            float f[kPerVec<T>];
            widen<T>(v[u], f);
#pragma unroll
            for (int e = 0; e < kPerVec<T>; ++e) f[e] *= a.scale;
            store_chunk<kStream>(static_cast<T*>(a.out) + (row0 + r) * a.width, static_cast<int>(item - r * a.chunks), a.width,
                                 narrow<T>(f));
        }
    }
}

struct RunArgs {
    const void* up;           // [n][width], stride
    const int2* sorted;       // sorted place -> (input position, row; `vocab` for an id outside the table)
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
    store_chunk(static_cast<T*>(a.out) + row * a.width, chunk, a.width, narrow<T>(f));
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
    const T* up = static_cast<const T*>(a.up);
    const int32_t before = begin > 0 ? a.sorted[begin - 1].y : -1;
    const int32_t after = end < a.n ? a.sorted[end].y : -1;
    constexpr int kAhead = 8;
    float sum[kPerVec<T>] = {};
    int32_t row = a.sorted[begin].y;
    bool first = true;   // the row began at or before this run's first place
    for (int64_t p = begin; p < end; p += kAhead) {
        int32_t rows[kAhead];
        vec16 v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t q = p + u < end ? p + u : end - 1;
            const int2 at = a.sorted[q];
            rows[u] = at.y;
            v[u] = load_chunk(up + static_cast<int64_t>(at.x) * a.stride, chunk, a.width);
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

constexpr int kNear = 16;    // runs a group of lanes follows by itself,
constexpr int kAtOnce = 4;   // so many heads in flight

// Each group of lanes takes one run, and where its last row goes on adds the heads of up to kNear runs after
// it.  Rows that reach further are left to the whole workgroup, one after the other: its groups take every
// so many heads each and their sums are added in order.
template <class T> __global__ __launch_bounds__(kEmbedBlock) void join_kernel(RunArgs a) {
    __shared__ float part[kEmbedBlock * kPerVec<T>];
    __shared__ int far[kEmbedBlock / 4];
    __shared__ int count;
    const int groups = kEmbedBlock / a.lanes, group = static_cast<int>(threadIdx.x) / a.lanes;
    const int lane = static_cast<int>(threadIdx.x) % a.lanes;
    const int64_t run0 = blockIdx.x / a.blocks * static_cast<int64_t>(groups);
    const int chunk = static_cast<int>(blockIdx.x % a.blocks) * a.lanes + lane;
    const int64_t pitch = static_cast<int64_t>(a.chunks) * kPerVec<T>;
    const float* head = a.head + static_cast<int64_t>(chunk) * kPerVec<T>;
    const float* tail = a.tail + static_cast<int64_t>(chunk) * kPerVec<T>;
    const bool own = chunk < a.chunks;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const int64_t run = run0 + group;
    if (run < a.runs - 1) {
        const int64_t begin = run * a.run, end = begin + a.run;   // not the last run: whole
        const int32_t row = a.sorted[end].y;
        if (row < a.vocab && a.sorted[end - 1].y == row && (begin == 0 || a.sorted[begin - 1].y != row)) {
            const int64_t past = end + static_cast<int64_t>(kNear) * a.run;
            if (past < a.n && a.sorted[past].y == row) {
                if (lane == 0) far[atomicAdd(&count, 1)] = group;
            } else if (own) {
                float sum[kPerVec<T>];
#pragma unroll
                for (int e = 0; e < kPerVec<T>; ++e) sum[e] = tail[run * pitch + e];
                for (int64_t r = run + 1; r < a.runs; r += kAtOnce) {
                    float h[kAtOnce][kPerVec<T>];
                    bool goes_on[kAtOnce];
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u) {   // heads of runs that the row does not reach are not added
                        const int64_t q = r + u < a.runs ? r + u : a.runs - 1;
                        goes_on[u] = r + u < a.runs && a.sorted[q * a.run].y == row;
#pragma unroll
                        for (int e = 0; e < kPerVec<T>; ++e) h[u][e] = head[q * pitch + e];
                    }
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                        for (int e = 0; e < kPerVec<T>; ++e) sum[e] += goes_on[u] ? h[u][e] : 0.0f;
                    if (!goes_on[kAtOnce - 1]) break;
                }
                write_row<T>(a, row, chunk, sum);
            }
        }
    }
    __syncthreads();
    const int rows = count;
    for (int k = 0; k < rows; ++k) {   // their order does not matter: each is another row
        const int64_t from = run0 + far[k] + 1;
        const int32_t row = a.sorted[from * a.run].y;
        int64_t low = from * a.run, high = a.n;   // the first place past the row
        while (low < high) {
            const int64_t mid = (low + high) / 2;
            if (a.sorted[mid].y <= row) low = mid + 1; else high = mid;
        }
        const int64_t last = (low - 1) / a.run;
        float sum[kPerVec<T>] = {};
        if (own)
#pragma unroll 2
            for (int64_t r = from + group; r <= last; r += groups)
#pragma unroll
                for (int e = 0; e < kPerVec<T>; ++e) sum[e] += head[r * pitch + e];
#pragma unroll
        for (int e = 0; e < kPerVec<T>; ++e) part[e * kEmbedBlock + threadIdx.x] = sum[e];
        __syncthreads();
        if (group == 0 && own) {
#pragma unroll
            for (int e = 0; e < kPerVec<T>; ++e) {
                float s = tail[(from - 1) * pitch + e];
                for (int g = 0; g < groups; ++g) s += part[e * kEmbedBlock + g * a.lanes + lane];
                sum[e] = s;
            }
            write_row<T>(a, row, chunk, sum);
        }
        __syncthreads();
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
    int64_t sorted, heads, sort;   // bytes
    int run, chunks;
    int64_t runs;
};

EmbedPlan embed_plan(int64_t n, int64_t vocab, int64_t width, int dtype) {
    EmbedPlan p{};
    p.chunks = chunks_of(width, dtype);
    p.run = run_length(n, p.chunks);
    p.runs = (n + p.run - 1) / p.run;
    p.sorted = padded(8 * n);
    p.heads = padded(p.runs * p.chunks * (16 / dtype_bytes(dtype)) * 4);
    p.sort = padded(sort_workspace(n, vocab));
    return p;
}

int check_embed(const std::string& what, int64_t n, int64_t vocab, int64_t width, int id_bytes, int dtype) {
    if (!known_dtype(dtype)) return fail(what + ": dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (vocab < 1 || vocab >= (int64_t{1} << 31) - 1) return fail(what + ": vocab must be within 1..2^31 - 2");
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
    const int64_t blocks = (n + a.block_rows - 1) / a.block_rows;
    if (blocks > most_blocks(kEmbedBlock)) return fail(what + ": too many rows for one launch");
    with_dtype(dtype, [&](auto t) {
        with_flag(n * width * dtype_bytes(dtype) >= kStreamBytes, [&](auto far) {
            lookup_kernel<decltype(t), far><<<static_cast<uint32_t>(blocks), kEmbedBlock, 0, as_stream(stream)>>>(a);
        });
    });
    return check_launch("embed");
}

ODIE_API int64_t odie_embed_workspace(int64_t n, int64_t vocab, int64_t width, int dtype) {
    if (check_embed("odie_embed_workspace", n, vocab, width, 4, dtype)) return -1;
    const EmbedPlan p = embed_plan(n, vocab, width, dtype);
    return p.sorted + 2 * p.heads + p.sort;
}

ODIE_API int odie_embed_backward(const void* upstream, int64_t upstream_stride, const void* ids, int id_bytes,
                                 int64_t n, int64_t vocab, float scale, int64_t width, int dtype, void* dtable,
                                 void* workspace, int64_t workspace_bytes, uint64_t stream) {
    const std::string what = "odie_embed_backward";
    if (check_embed(what, n, vocab, width, id_bytes, dtype)) return -1;
    if (!dtable || (n > 0 && (!upstream || !ids))) return fail(what + ": null pointer");
    if (n > 0 && upstream_stride < width) return fail(what + ": rows overlap (a stride below the row's width)");
    const EmbedPlan p = embed_plan(n, vocab, width, dtype);
    const int64_t need = p.sorted + 2 * p.heads + p.sort;
    if (n > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0))
        return fail(what + ": needs a 256-byte aligned workspace of " + std::to_string(need) + " bytes");
    const int lanes = run_lanes(p.chunks), across = (p.chunks + lanes - 1) / lanes;
    const int64_t walks = (p.runs * across * lanes + kEmbedBlock - 1) / kEmbedBlock;
    const int64_t joins = (p.runs + kEmbedBlock / lanes - 1) / (kEmbedBlock / lanes) * across;
    if (walks > most_blocks(kEmbedBlock) || joins > most_blocks(kEmbedBlock))
        return fail(what + ": too many runs for one launch");
    hipStream_t s = as_stream(stream);
    const int64_t bytes = vocab * width * dtype_bytes(dtype);
    const int64_t fill = (bytes + kEmbedBlock * 16 - 1) / (kEmbedBlock * 16);
    clear_kernel<<<static_cast<uint32_t>(fill > 16 * kCus ? 16 * kCus : fill), kEmbedBlock, 0, s>>>(static_cast<char*>(dtable), bytes);
    if (check_launch("embed gradient")) return -1;
    if (n == 0) return 0;
    char* scratch = static_cast<char*>(workspace);
    RunArgs a{};
    int2* sorted = reinterpret_cast<int2*>(scratch);
    a.head = reinterpret_cast<float*>(scratch + p.sorted);
    a.tail = reinterpret_cast<float*>(scratch + p.sorted + p.heads);
    if (launch_sort(SortKeys{ids, id_bytes, n, vocab}, SortOut{nullptr, sorted, nullptr, nullptr, nullptr},
                    scratch + p.sorted + 2 * p.heads, s))
        return -1;
    a.up = upstream;
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
    a.lanes = lanes;
    a.blocks = across;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        runs_kernel<T><<<static_cast<uint32_t>(walks), kEmbedBlock, 0, s>>>(a);
        if (p.runs > 1)
            join_kernel<T><<<static_cast<uint32_t>(joins), kEmbedBlock, 0, s>>>(a);
    });
    return check_launch("embed gradient");
}
