// Rows sent to their experts' slots and brought back with weights, and their gradients.
//
// Row i has `choices` entries f = i choices + j; entry f lies at slots[f] of the sorted rows (odie_sort
// over the entries' experts), or nowhere (-1: its choice is no expert).
//   dispatch   out[slots[f]] = x[i]                            0 from offsets[experts] on
//   combine    y[i] = sum_j weights[f] rows[slots[f]]
//   gradients  drows[slots[f]] = weights[f] dy[i]              0 from offsets[experts] on
//              dweights[f] = <dy[i], rows[slots[f]]>
// The gradient of dispatch is combine without weights.  Each of them reads and writes every row once and
// is bound by HBM, so the walk is over input rows: x and dy are read once however many choices there are,
// and the scattered side moves whole rows.  Sums are fp32 in the order of the choices, rounded once.
#include "elements.h"
#include "tiles.h"

namespace odie {
namespace {

constexpr int kMoveBlock = 256;

struct MoveArgs {
    const void* x;            // dispatch: [n]; combine: [n choices]; both [.][width], stride ldx
    const void* rows;         // the gradient of combine: the sorted rows, stride ldr
    const int32_t* slots;     // [n choices]
    const float* weights;     // [n choices], or null: 1
    const int32_t* offsets;   // [experts + 1]
    void* out;
    float* dweights;
    int64_t n, ldx, ldr;
    Divisor by_chunks;
    uint32_t block_rows;      // input rows a workgroup takes
    int choices, experts, width, chunks;
    int lanes;                // gradient of combine: lanes a row
};

// Zeros in the slots that no expert owns, shared out over the workgroups.
template <class T> __device__ inline void clear_rest(const MoveArgs& a) {
    const int64_t entries = a.n * a.choices;
    const int64_t held = group_start(a.offsets, a.experts, entries), rest = entries - held;
    if (rest == 0) return;
    const int64_t each = (rest + gridDim.x - 1) / gridDim.x;
    const int64_t begin = held + each * blockIdx.x, end = begin + each < entries ? begin + each : entries;
    for (int64_t s = begin; s < end; ++s) {
        T* to = static_cast<T*>(a.out) + s * a.width;
        for (int c = threadIdx.x; c < a.chunks; c += kMoveBlock)
            store_some(to + c * kPerVec<T>, vec16{}, a.width - c * kPerVec<T>);
    }
}

template <class T> __global__ __launch_bounds__(kMoveBlock) void dispatch_kernel(MoveArgs a) {
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.block_rows;
    const int64_t left = a.n - row0;
    const uint32_t items = (left < a.block_rows ? static_cast<uint32_t>(left) : a.block_rows) * a.chunks;
    const int64_t entries = a.n * a.choices;
    for (uint32_t t = threadIdx.x; t < items; t += kMoveBlock) {
        const uint32_t r = divide(t, a.by_chunks);
        const int column = static_cast<int>(t - r * a.chunks) * kPerVec<T>, count = a.width - column;
        const int64_t i = row0 + r;
        const vec16 v = load_some(static_cast<const T*>(a.x) + i * a.ldx + column, count);
        for (int j = 0; j < a.choices; ++j) {
            const int64_t slot = a.slots[i * a.choices + j];
            if (slot >= 0 && slot < entries) store_some(static_cast<T*>(a.out) + slot * a.width + column, v, count);
        }
    }
    clear_rest<T>(a);
}

template <class T> __global__ __launch_bounds__(kMoveBlock) void combine_kernel(MoveArgs a) {
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.block_rows;
    const int64_t left = a.n - row0;
    const uint32_t items = (left < a.block_rows ? static_cast<uint32_t>(left) : a.block_rows) * a.chunks;
    const int64_t entries = a.n * a.choices;
    for (uint32_t t = threadIdx.x; t < items; t += kMoveBlock) {
        const uint32_t r = divide(t, a.by_chunks);
        const int column = static_cast<int>(t - r * a.chunks) * kPerVec<T>, count = a.width - column;
        const int64_t i = row0 + r;
        float sum[kPerVec<T>] = {};
        for (int j = 0; j < a.choices; ++j) {
            const int64_t slot = a.slots[i * a.choices + j];
            if (slot < 0 || slot >= entries) continue;
            float v[kPerVec<T>];
            widen<T>(load_some(static_cast<const T*>(a.x) + slot * a.ldx + column, count), v);
            const float w = a.weights ? a.weights[i * a.choices + j] : 1.0f;
#pragma unroll
            for (int e = 0; e < kPerVec<T>; ++e) sum[e] += w * v[e];
        }
        store_some(static_cast<T*>(a.out) + i * a.width + column, narrow<T>(sum), count);
    }
}

// A group of `lanes` lanes takes an input row; lanes divides 64.
template <class T> __global__ __launch_bounds__(kMoveBlock) void combine_backward_kernel(MoveArgs a) {
    const int lane = static_cast<int>(threadIdx.x) % a.lanes;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * (kMoveBlock / a.lanes) + static_cast<int>(threadIdx.x) / a.lanes;
    const int64_t entries = a.n * a.choices;
    if (i < a.n) {
        const T* up = static_cast<const T*>(a.x) + i * a.ldx;
        for (int j = 0; j < a.choices; ++j) {
            const int64_t f = i * a.choices + j, slot = a.slots[f];
            const bool held = slot >= 0 && slot < entries;
            const float w = a.weights ? a.weights[f] : 1.0f;
            float dot = 0.0f;
            if (held)
                for (int c = lane; c < a.chunks; c += a.lanes) {
                    const int column = c * kPerVec<T>, count = a.width - column;
                    float d[kPerVec<T>], v[kPerVec<T>];
                    widen<T>(load_some(up + column, count), d);
                    if (a.dweights) {
                        widen<T>(load_some(static_cast<const T*>(a.rows) + slot * a.ldr + column, count), v);
#pragma unroll
                        for (int e = 0; e < kPerVec<T>; ++e) dot += d[e] * v[e];
                    }
                    if (a.out) {
#pragma unroll
                        for (int e = 0; e < kPerVec<T>; ++e) d[e] *= w;
                        store_some(static_cast<T*>(a.out) + slot * a.width + column, narrow<T>(d), count);
                    }
                }
            if (a.dweights) {
                for (int m = a.lanes / 2; m > 0; m /= 2) dot += __shfl_xor(dot, m);
                if (lane == 0) a.dweights[f] = dot;
            }
        }
    }
    if (a.out) clear_rest<T>(a);
}

// Lanes for a row of `chunks` 16-byte pieces: the most (up to 64) that keep four of five busy.
int row_lanes(int chunks) {
    int best = 4;
    for (int lanes = 8; lanes <= 64; lanes *= 2)
        if (5 * chunks >= 4 * ((chunks + lanes - 1) / lanes * lanes)) best = lanes;
    return best;
}

int check_move(const std::string& what, int64_t n, int choices, int experts, int64_t width, int dtype) {
    if (!known_dtype(dtype)) return fail(what + ": dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (n < 0 || choices < 1 || n > ((int64_t{1} << 31) - 1) / choices)
        return fail(what + ": n * choices must be within 0..2^31 - 1, choices at least 1");
    if (width < 1 || width > 1 << 20) return fail(what + ": width must be within 1..2^20");
    if (experts < 1) return fail(what + ": experts must be at least 1");
    return 0;
}

MoveArgs move_args(int64_t n, int choices, int experts, int64_t width, int dtype) {
    MoveArgs a{};
    a.n = n;
    a.choices = choices;
    a.experts = experts;
    a.width = static_cast<int>(width);
    const int per = static_cast<int>(16 / dtype_bytes(dtype));
    a.chunks = (a.width + per - 1) / per;
    a.by_chunks = make_divisor(static_cast<uint32_t>(a.chunks));
    // about 1024 pieces of 16 bytes a workgroup
    a.block_rows = a.chunks >= 1024 ? 1u : static_cast<uint32_t>(1024 / a.chunks);
    a.lanes = row_lanes(a.chunks);
    return a;
}

uint32_t move_blocks(const MoveArgs& a) { return static_cast<uint32_t>((a.n + a.block_rows - 1) / a.block_rows); }

}  // namespace
}  // namespace odie

using namespace odie;

ODIE_API int odie_rows_dispatch(const void* x, int64_t x_stride, const int32_t* slots, const int32_t* offsets,
                                int64_t n, int choices, int experts, int64_t width, int dtype, void* out,
                                uint64_t stream) {
    const std::string what = "odie_rows_dispatch";
    if (check_move(what, n, choices, experts, width, dtype)) return -1;
    if (n == 0) return 0;
    if (!x || !slots || !offsets || !out) return fail(what + ": null pointer");
    if (x_stride < width) return fail(what + ": rows overlap (a stride below the row's width)");
    MoveArgs a = move_args(n, choices, experts, width, dtype);
    a.x = x;
    a.ldx = x_stride;
    a.slots = slots;
    a.offsets = offsets;
    a.out = out;
    with_dtype(dtype, [&](auto t) { dispatch_kernel<decltype(t)><<<move_blocks(a), kMoveBlock, 0, as_stream(stream)>>>(a); });
    return check_launch("rows dispatch");
}

ODIE_API int odie_rows_combine(const void* rows, int64_t rows_stride, const int32_t* slots, const float* weights,
                               int64_t n, int choices, int64_t width, int dtype, void* out, uint64_t stream) {
    const std::string what = "odie_rows_combine";
    if (check_move(what, n, choices, 1, width, dtype)) return -1;
    if (n == 0) return 0;
    if (!rows || !slots || !out) return fail(what + ": null pointer");
    if (rows_stride < width) return fail(what + ": rows overlap (a stride below the row's width)");
    MoveArgs a = move_args(n, choices, 1, width, dtype);
    a.x = rows;
    a.ldx = rows_stride;
    a.slots = slots;
    a.weights = weights;
    a.out = out;
    with_dtype(dtype, [&](auto t) { combine_kernel<decltype(t)><<<move_blocks(a), kMoveBlock, 0, as_stream(stream)>>>(a); });
    return check_launch("rows combine");
}

ODIE_API int odie_rows_combine_backward(const void* upstream, int64_t upstream_stride, const void* rows,
                                        int64_t rows_stride, const int32_t* slots, const float* weights,
                                        const int32_t* offsets, int64_t n, int choices, int experts, int64_t width,
                                        int dtype, void* drows, float* dweights, uint64_t stream) {
    const std::string what = "odie_rows_combine_backward";
    if (check_move(what, n, choices, experts, width, dtype)) return -1;
    if (n == 0 || (!drows && !dweights)) return 0;
    if (!upstream || !slots || (drows && !offsets) || (dweights && !rows)) return fail(what + ": null pointer");
    if (upstream_stride < width || (dweights && rows_stride < width))
        return fail(what + ": rows overlap (a stride below the row's width)");
    MoveArgs a = move_args(n, choices, experts, width, dtype);
    a.x = upstream;
    a.ldx = upstream_stride;
    a.rows = rows;
    a.ldr = rows_stride;
    a.slots = slots;
    a.weights = weights;
    a.offsets = offsets;
    a.out = drows;
    a.dweights = dweights;
    const int height = kMoveBlock / a.lanes;
    with_dtype(dtype, [&](auto t) {
        combine_backward_kernel<decltype(t)>
            <<<static_cast<uint32_t>((n + height - 1) / height), kMoveBlock, 0, as_stream(stream)>>>(a);
    });
    return check_launch("rows combine gradient");
}
