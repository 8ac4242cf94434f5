// The kernels of linear.hip, instantiated by linear_f16.hip, linear_bf16.hip and linear_f32.hip.
#pragma once
#include "linear.h"

namespace odie {
namespace {

// Tiles: 128 x 128 with 64 x 64 a wave; 128 x 64 with 32 x 64 a wave for narrow outputs; 64 x 64 with 32 x 32 a
// wave where there are too few tiles otherwise.
template <class T, bool kAByRow, bool kBByRow> using Wide = Tile<T, kAByRow, kBByRow, 128, 128, 64, 64>;
template <class T, bool kAByRow, bool kBByRow> using Narrow = Tile<T, kAByRow, kBByRow, 128, 64, 32, 64>;
template <class T, bool kAByRow, bool kBByRow> using Small = Tile<T, kAByRow, kBByRow, 64, 64, 32, 32>;

template <class T, bool kForward, int kBM, int kBN, int kWM, int kWN>
__global__ __launch_bounds__(64 * (kBM / kWM) * (kBN / kWN)) void rows_kernel(RowsArgs a, uint32_t blocks) {
    using Work = Tile<T, true, kForward, kBM, kBN, kWM, kWN>;
    __shared__ __attribute__((aligned(16))) char lds[Work::kLds];
    const uint32_t id = xcd_major(blockIdx.x, gridDim.x);
    if (id >= blocks) return;
    const uint32_t across = (a.columns + kBN - 1) / kBN;
    const Piece p = find_piece(a.offsets, a.experts, a.experts + 1, a.rows, kBM, id / across);
    if (p.begin >= p.end) return;
    const int column0 = static_cast<int>(id % across) * kBN;
    const T* residual = static_cast<const T*>(a.residual);
    T* out = static_cast<T*>(a.out);
    if (p.group >= a.experts) {   // rows of no expert
        for (int i = threadIdx.x; i < kBM * (kBN / 8); i += Work::kThreads) {
            const int64_t row = p.begin + i / (kBN / 8);
            const int column = column0 + i % (kBN / 8) * 8;
            if (row >= p.end || column >= a.columns) continue;
            float value[8] = {};
            if (residual) load8(residual + row * a.ldr + column, a.columns - column, value);
            store8(out + row * a.ldo + column, a.columns - column, value);
        }
        return;
    }
    const int64_t matrix = static_cast<int64_t>(a.columns) * a.depth;
    const T* b = static_cast<const T*>(a.b) + p.group * matrix;
    typename Work::A opa;
    typename Work::B opb;
    opa.begin(static_cast<const T*>(a.a), a.lda, p.begin, p.end);
    opb.begin(b, kForward ? a.depth : a.columns, column0, a.columns);
    Work work;
    work.sum(opa, opb, a.depth, lds);
    const T* bias = a.bias ? static_cast<const T*>(a.bias) + static_cast<int64_t>(p.group) * a.columns : nullptr;
    T* pre = static_cast<T*>(a.pre);
    work.rows(lds, [&](int r, int c, float value[8]) {
        const int64_t row = p.begin + r;
        const int column = column0 + c, count = a.columns - column;
        if (row >= p.end || count <= 0) return;
        float more[8];
        if (bias) {
            load8(bias + column, count, more);
#pragma unroll
            for (int i = 0; i < 8; ++i) value[i] += more[i];
        }
        if (pre) store8(pre + row * a.columns + column, count, value);
        if (a.activation != kNone) {
#pragma unroll
            for (int i = 0; i < 8; ++i) value[i] = activate(a.activation, value[i]);
        }
        if (residual) {
            load8(residual + row * a.ldr + column, count, more);
#pragma unroll
            for (int i = 0; i < 8; ++i) value[i] += more[i];
        }
        store8(out + row * a.ldo + column, count, value);
    });
}

template <class T, int kBM, int kBN, int kWM, int kWN>
__global__ __launch_bounds__(64 * (kBM / kWM) * (kBN / kWN)) void weight_kernel(WeightArgs a, uint32_t blocks) {
    using Work = Tile<T, false, false, kBM, kBN, kWM, kWN>;
    __shared__ __attribute__((aligned(16))) char lds[Work::kLds];
    const uint32_t id = xcd_major(blockIdx.x, gridDim.x);
    if (id >= blocks) return;
    const uint32_t across = (a.inputs + kBN - 1) / kBN, tiles = (a.outputs + kBM - 1) / kBM * across;
    const uint32_t piece = id / tiles, tile = id % tiles;
    const Piece p = find_piece(a.offsets, a.experts, a.experts, a.rows, a.piece, piece);
    if (p.first > 0 && p.begin >= p.end) return;
    const int row0 = static_cast<int>(tile / across) * kBM, column0 = static_cast<int>(tile % across) * kBN;
    Work work;
    const int64_t depth = p.end > p.begin ? p.end - p.begin : 0;
    typename Work::A opa;
    typename Work::B opb;
    opa.begin(static_cast<const T*>(a.dz) + p.begin * a.ldz, a.ldz, row0, a.outputs);
    opb.begin(static_cast<const T*>(a.x) + p.begin * a.ldx, a.ldx, column0, a.inputs);
    work.sum(opa, opb, depth, lds);   // no rows: zeros
    const int64_t matrix = static_cast<int64_t>(a.outputs) * a.inputs;
    const bool whole = p.group_end - p.group_begin <= a.piece;
    T* dw = static_cast<T*>(a.dw) + p.group * matrix;
    float* partial = whole ? nullptr : a.partial + piece * matrix;
    work.rows(lds, [&](int r, int c, float value[8]) {
        const int row = row0 + r, column = column0 + c, count = a.inputs - column;
        if (row >= a.outputs || count <= 0) return;
        const int64_t at = static_cast<int64_t>(row) * a.inputs + column;
        if (whole)
            store8(dw + at, count, value);
        else
            store8(partial + at, count, value);
    });
}

constexpr int kSlopeBlock = 256;

// A workgroup takes one piece of rows and `lanes` groups of 8 columns; 256 / lanes rows at a time.
template <class T> __global__ __launch_bounds__(kSlopeBlock) void slope_kernel(SlopeArgs a, int lanes, uint32_t across) {
    __shared__ float total[kSlopeBlock * 8];
    const Piece p = find_piece(a.offsets, a.experts, a.experts, a.rows, a.piece, blockIdx.x / across);
    if (p.begin >= p.end) return;
    const int lane = static_cast<int>(threadIdx.x) % lanes, height = kSlopeBlock / lanes;
    const int column = (static_cast<int>(blockIdx.x % across) * lanes + lane) * 8, count = a.columns - column;
    float sum[8] = {};
    if (count > 0) {
        const T* dy = static_cast<const T*>(a.dy);
        const T* pre = static_cast<const T*>(a.pre);
        T* dz = static_cast<T*>(a.dz);
        for (int64_t row = p.begin + static_cast<int>(threadIdx.x) / lanes; row < p.end; row += height) {
            float d[8];
            load8(dy + row * a.ldy + column, count, d);
            if (dz) {
                float z[8];
                load8(pre + row * a.columns + column, count, z);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] *= slope(a.activation, z[i]);
                store8(dz + row * a.columns + column, count, d);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += d[i];
        }
    }
    if (!a.sums) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) total[i * kSlopeBlock + threadIdx.x] = sum[i];
    __syncthreads();
    if (static_cast<int>(threadIdx.x) >= lanes || count <= 0) return;
    float* to = a.sums + blockIdx.x / across * static_cast<int64_t>(a.columns) + column;
    for (int i = 0; i < 8 && i < count; ++i) {
        float s = 0.0f;
        for (int r = 0; r < height; ++r) s += total[i * kSlopeBlock + r * lanes + lane];
        to[i] = s;
    }
}

template <class T> __global__ __launch_bounds__(256) void fold_kernel(FoldArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.size) return;
    const int e = static_cast<int>(blockIdx.y);
    const int64_t begin = a.offsets ? group_start(a.offsets, e, a.rows) : 0;
    const int64_t end = a.offsets ? group_start(a.offsets, e + 1, a.rows) : a.rows;
    const int64_t first = a.offsets ? whole_pieces(a.offsets, e, a.rows, a.piece) + e : 0;
    const int64_t pieces = end > begin ? (end - begin + a.piece - 1) / a.piece : 0;
    if (pieces <= 1 && !a.single) return;
    const float* from = a.partial + first * a.size + i;
    float sum = 0.0f;
    for (int64_t p = 0; p < pieces; ++p) sum += from[p * a.size];
    static_cast<T*>(a.out)[e * a.size + i] = static_cast<T>(sum);
}

uint32_t whole_xcds(int64_t blocks) { return static_cast<uint32_t>((blocks + kXcds - 1) / kXcds * kXcds); }

template <class T, bool kForward, int kBM, int kBN, int kWM, int kWN> int launch_rows_as(RowsArgs a, hipStream_t stream) {
    const int64_t across = (a.columns + kBN - 1) / kBN;
    a.tiles = piece_ids(a.rows, kBM, a.offsets != nullptr, a.experts, true);
    const int64_t blocks = a.tiles * across;
    if (blocks >= int64_t{1} << 31) return fail("linear: too many tiles for one launch");
    rows_kernel<T, kForward, kBM, kBN, kWM, kWN>
        <<<whole_xcds(blocks), 64 * (kBM / kWM) * (kBN / kWN), 0, stream>>>(a, static_cast<uint32_t>(blocks));
    return check_launch("linear");
}

template <class T, bool kForward> int launch_rows_of(const RowsArgs& a, hipStream_t stream) {
    const int64_t wide = (a.rows + 127) / 128 * ((a.columns + 127) / 128);
    if (a.columns <= 64 && a.rows >= 128 * kCus) return launch_rows_as<T, kForward, 128, 64, 32, 64>(a, stream);
    if (a.columns > 64 && wide >= kCus) return launch_rows_as<T, kForward, 128, 128, 64, 64>(a, stream);
    return launch_rows_as<T, kForward, 64, 64, 32, 32>(a, stream);
}

template <class T, int kBM, int kBN, int kWM, int kWN> int launch_weight_as(const WeightArgs& a, hipStream_t stream) {
    const int64_t tiles = static_cast<int64_t>((a.outputs + kBM - 1) / kBM) * ((a.inputs + kBN - 1) / kBN);
    const int64_t blocks = a.pieces * tiles;
    if (blocks >= int64_t{1} << 31) return fail("linear: too many tiles for one launch");
    weight_kernel<T, kBM, kBN, kWM, kWN>
        <<<whole_xcds(blocks), 64 * (kBM / kWM) * (kBN / kWN), 0, stream>>>(a, static_cast<uint32_t>(blocks));
    return check_launch("linear weight gradient");
}

}  // namespace

template <class T> int launch_rows(const RowsArgs& a, bool forward, hipStream_t stream) {
    return forward ? launch_rows_of<T, true>(a, stream) : launch_rows_of<T, false>(a, stream);
}

template <class T> int launch_weight(const WeightArgs& a, hipStream_t stream) {
    if (a.outputs <= 64 || a.inputs <= 64) return launch_weight_as<T, 64, 64, 32, 32>(a, stream);
    return launch_weight_as<T, 128, 128, 64, 64>(a, stream);
}

template <class T> int launch_slope(const SlopeArgs& a, hipStream_t stream) {
    const int groups = (a.columns + 7) / 8;
    int lanes = 1;
    while (lanes < 32 && lanes < groups) lanes *= 2;
    const int64_t across = (groups + lanes - 1) / lanes, blocks = a.pieces * across;
    if (blocks >= int64_t{1} << 31) return fail("linear: too many workgroups for one launch");
    if (blocks == 0) return 0;
    slope_kernel<T><<<static_cast<uint32_t>(blocks), kSlopeBlock, 0, stream>>>(a, lanes, static_cast<uint32_t>(across));
    return check_launch("linear activation gradient");
}

template <class T> int launch_fold(const FoldArgs& a, hipStream_t stream) {
    if ((a.size + 255) / 256 >= int64_t{1} << 31) return fail("linear: too many sums for one launch");
    const dim3 grid(static_cast<uint32_t>((a.size + 255) / 256), static_cast<uint32_t>(a.experts));
    fold_kernel<T><<<grid, 256, 0, stream>>>(a);
    return check_launch("linear fold");
}

}  // namespace odie

#define ODIE_LINEAR_FOR(T)                                                                       \
    namespace odie {                                                                             \
    template int launch_rows<T>(const RowsArgs&, bool, hipStream_t);                             \
    template int launch_weight<T>(const WeightArgs&, hipStream_t);                               \
    template int launch_slope<T>(const SlopeArgs&, hipStream_t);                                 \
    template int launch_fold<T>(const FoldArgs&, hipStream_t);                                   \
    }
