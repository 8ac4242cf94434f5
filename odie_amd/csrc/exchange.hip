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
// 65536 rows x 2 choices of 256 fp16: dispatch and combine 17 us each (5.8 TB/s, the caches helping), gradients 29.
// 300007 x 4 of 131 bf16, which share lines: 104, 99 and 198 us (3.6 to 4.0 TB/s).  (By slot instead of by row:
// dispatch 114 -> 116 and the gradients 302 -> 339 at the time.)
#include <type_traits>

#include "elements.h"
#include "tiles.h"

namespace odie {
namespace {

constexpr int kMoveBlock = 256;

struct MoveArgs {
    const void* x;            // dispatch: x; combine: the sorted rows; gradient of combine: dy; stride ldx
    const void* rows;         // gradient of combine: the sorted rows, stride ldr
    const int32_t* slots;     // [n choices]
    const float* weights;     // [n choices], or null: 1
    const int32_t* offsets;   // [experts + 1]
    void* out;
    float* dweights;
    int64_t n, ldx, ldr;
    Divisor by_chunks;
    uint32_t block_rows;      // input rows a workgroup takes
    int choices, experts, width, chunks;
    int lanes;                // dispatch and the gradient of combine: lanes a row,
    uint32_t first;           // and the first workgroup of this launch
    bool by_xcd;
};

// Zeros in the slots that no expert owns, shared out over the workgroups of the first launch.
template <class T> __device__ inline void clear_rest(const MoveArgs& a) {
    if (a.first > 0) return;
    const int64_t entries = a.n * a.choices;
    const int64_t held = group_start(a.offsets, a.experts, entries), rest = entries - held;
    if (rest == 0) return;
    const int64_t each = (rest + gridDim.x - 1) / gridDim.x;
    const int64_t begin = held + each * blockIdx.x, end = begin + each < entries ? begin + each : entries;
    for (int64_t s = begin; s < end; ++s) {
        T* to = static_cast<T*>(a.out) + s * a.width;
        for (int c = threadIdx.x; c < a.chunks; c += kMoveBlock) store_chunk(to, c, a.width, vec16{});
    }
}

// The slot of entry first + j of row i; -1 where there is none.
template <int kChoices> __device__ inline int64_t slot_of(const MoveArgs& a, int64_t i, int choices, int j) {
    if (!kChoices && j >= choices) return -1;
    const int64_t slot = a.slots[i * choices + j];
    return slot < a.n * choices ? slot : -1;
}

// The input row of this thread's group of `lanes` lanes (lanes divides 64), n or more for none.  Where rows do
// not fill their 64-byte blocks, workgroups that follow each other in rows run on one XCD: the rows that they
// send to an expert lie side by side, and the lines that two of them share meet in that XCD's L2 (300007 x 4
// rows of 272 bytes sent: 124 -> 92 us).  Whole blocks go faster spread over the XCDs (256 bytes: 81 -> 74 us).
__device__ inline int64_t lane_row(const MoveArgs& a) {
    const uint32_t block = a.first + (a.by_xcd ? xcd_major(blockIdx.x, gridDim.x) : blockIdx.x);
    return static_cast<int64_t>(block) * (kMoveBlock / a.lanes) + static_cast<int>(threadIdx.x) / a.lanes;
}

// kChoices entries of a row are handled together (0: any number of choices, in twos).
template <class T, int kChoices, bool kStream> __global__ __launch_bounds__(kMoveBlock) void dispatch_kernel(MoveArgs a) {
    constexpr int kStep = kChoices ? kChoices : 2;
    const int choices = kChoices ? kChoices : a.choices;
    const int lane = static_cast<int>(threadIdx.x) % a.lanes;
    const int64_t i = lane_row(a);
    if (i < a.n)
        for (int first = 0; first < choices; first += kStep) {
            int64_t slot[kStep];
#pragma unroll
            for (int j = 0; j < kStep; ++j) slot[j] = slot_of<kChoices>(a, i, choices, first + j);
            for (int c = lane; c < a.chunks; c += a.lanes) {
                const vec16 v = load_chunk(static_cast<const T*>(a.x) + i * a.ldx, c, a.width);
#pragma unroll
                for (int j = 0; j < kStep; ++j)
                    if (slot[j] >= 0) store_chunk<kStream>(static_cast<T*>(a.out) + slot[j] * a.width, c, a.width, v);
            }
        }
    clear_rest<T>(a);
}

template <class T, int kChoices, bool kStream> __global__ __launch_bounds__(kMoveBlock) void combine_kernel(MoveArgs a) {
    constexpr int kStep = kChoices ? kChoices : 2;
    const int choices = kChoices ? kChoices : a.choices;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.block_rows;
    const int64_t left = a.n - row0;
    const uint32_t items = (left < a.block_rows ? static_cast<uint32_t>(left) : a.block_rows) * a.chunks;
    for (uint32_t t = threadIdx.x; t < items; t += kMoveBlock) {
        const uint32_t r = divide(t, a.by_chunks);
        const int chunk = static_cast<int>(t - r * a.chunks);
        const int64_t i = row0 + r;
        float sum[kPerVec<T>] = {};
        for (int first = 0; first < choices; first += kStep) {
            vec16 v[kStep];
            float w[kStep];
#pragma unroll
            for (int j = 0; j < kStep; ++j) {
                const int64_t slot = slot_of<kChoices>(a, i, choices, first + j);
                w[j] = slot >= 0 ? (a.weights ? a.weights[i * choices + first + j] : 1.0f) : 0.0f;
                v[j] = slot >= 0 ? load_chunk(static_cast<const T*>(a.x) + slot * a.ldx, chunk, a.width) : vec16{};
            }
#pragma unroll
            for (int j = 0; j < kStep; ++j) {
                float f[kPerVec<T>];
                widen<T>(v[j], f);
#pragma unroll
                for (int e = 0; e < kPerVec<T>; ++e) sum[e] += w[j] * f[e];
            }
        }
        store_chunk<kStream>(static_cast<T*>(a.out) + i * a.width, chunk, a.width, narrow<T>(sum));
    }
}

template <class T, int kChoices, bool kStream> __global__ __launch_bounds__(kMoveBlock) void combine_backward_kernel(MoveArgs a) {
    constexpr int kStep = kChoices ? kChoices : 2;
    const int choices = kChoices ? kChoices : a.choices;
    const int lane = static_cast<int>(threadIdx.x) % a.lanes;
    const int64_t i = lane_row(a);
    if (i < a.n) {
        const T* up = static_cast<const T*>(a.x) + i * a.ldx;
        for (int first = 0; first < choices; first += kStep) {
            int64_t slot[kStep];
            float w[kStep], dot[kStep] = {};
#pragma unroll
            for (int j = 0; j < kStep; ++j) {
                slot[j] = slot_of<kChoices>(a, i, choices, first + j);
                w[j] = slot[j] >= 0 && a.weights ? a.weights[i * choices + first + j] : 1.0f;
            }
            for (int c = lane; c < a.chunks; c += a.lanes) {
                const vec16 u = load_chunk(up, c, a.width);
                vec16 v[kStep];
#pragma unroll
                for (int j = 0; j < kStep; ++j)
                    v[j] = a.dweights && slot[j] >= 0
                               ? load_chunk(static_cast<const T*>(a.rows) + slot[j] * a.ldr, c, a.width) : vec16{};
                const int again = chunk_overlap<T>(c, a.width);   // elements that the chunk before holds too
                float d[kPerVec<T>];
                widen<T>(u, d);
#pragma unroll
                for (int j = 0; j < kStep; ++j) {
                    float f[kPerVec<T>], g[kPerVec<T>];
                    widen<T>(v[j], f);
#pragma unroll
                    for (int e = 0; e < kPerVec<T>; ++e) {
                        if (e >= again) dot[j] += d[e] * f[e];
                        g[e] = d[e] * w[j];
                    }
                    if (a.out && slot[j] >= 0)
                        store_chunk<kStream>(static_cast<T*>(a.out) + slot[j] * a.width, c, a.width, narrow<T>(g));
                }
            }
            if (a.dweights) {
#pragma unroll
                for (int j = 0; j < kStep; ++j) {
                    for (int m = a.lanes / 2; m > 0; m /= 2) dot[j] += __shfl_xor(dot[j], m);
                    if (lane == 0 && (kChoices || first + j < choices))
                        a.dweights[i * choices + first + j] = slot[j] >= 0 ? dot[j] : 0.0f;   // not NaN times 0
                }
            }
        }
    }
    if (a.out) clear_rest<T>(a);
}

// f with the number of choices as a constant where it is 1, 2 or 4, else 0, and whether to stream.
template <class F> void with_choices(int choices, bool stream, F&& f) {
    with_flag(stream, [&](auto far) {
        if (choices == 1) f(std::integral_constant<int, 1>{}, far);
        else if (choices == 2) f(std::integral_constant<int, 2>{}, far);
        else if (choices == 4) f(std::integral_constant<int, 4>{}, far);
        else f(std::integral_constant<int, 0>{}, far);
    });
}

// Whether rows scattered over the sorted ones are streamed: those that share lines have to meet in the L2 (131 bf16
// columns: 102 us through it, 144 past it; 256 columns 145 and 117).
bool stream_scattered(const MoveArgs& a, int dtype) {
    return !a.by_xcd && a.n * a.choices * a.width * dtype_bytes(dtype) >= kStreamBytes;
}

// Lanes for a row of `chunks` 16-byte pieces: a whole row at once where 64 lanes can.
int row_lanes(int chunks) {
    int lanes = 1;
    while (lanes < 64 && lanes < chunks) lanes *= 2;
    return lanes;
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
    a.by_xcd = width * dtype_bytes(dtype) % 64 != 0;
    return a;
}

int64_t row_blocks(const MoveArgs& a) {
    const int64_t height = kMoveBlock / a.lanes, blocks = (a.n + height - 1) / height;
    return (blocks + kXcds - 1) / kXcds * kXcds;
}

int64_t move_blocks(const MoveArgs& a) { return (a.n + a.block_rows - 1) / a.block_rows; }

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
    with_dtype(dtype, [&](auto t) {
        with_choices(choices, stream_scattered(a, dtype), [&](auto k, auto far) {
            in_launches(row_blocks(a), kMoveBlock, [&](uint32_t first, uint32_t count) {
                a.first = first;
                dispatch_kernel<decltype(t), k, far><<<count, kMoveBlock, 0, as_stream(stream)>>>(a);
            });
        });
    });
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
    const int64_t blocks = move_blocks(a);
    if (blocks > most_blocks(kMoveBlock)) return fail(what + ": too many rows for one launch");
    a.x = rows;
    a.ldx = rows_stride;
    a.slots = slots;
    a.weights = weights;
    a.out = out;
    with_dtype(dtype, [&](auto t) {
        with_choices(choices, n * width * dtype_bytes(dtype) >= kStreamBytes, [&](auto k, auto far) {
            combine_kernel<decltype(t), k, far><<<static_cast<uint32_t>(blocks), kMoveBlock, 0, as_stream(stream)>>>(a);
        });
    });
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
    with_dtype(dtype, [&](auto t) {
        with_choices(choices, drows && stream_scattered(a, dtype), [&](auto k, auto far) {
            in_launches(row_blocks(a), kMoveBlock, [&](uint32_t first, uint32_t count) {
                a.first = first;
                combine_backward_kernel<decltype(t), k, far><<<count, kMoveBlock, 0, as_stream(stream)>>>(a);
            });
        });
    });
    return check_launch("rows combine gradient");
}
