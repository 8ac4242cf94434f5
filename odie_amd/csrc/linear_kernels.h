// The kernels of linear.hip, instantiated by linear_f16.hip, linear_bf16.hip and linear_f32.hip.
#pragma once
#include "linear_epilogue.h"

namespace odie {
namespace {

// One tile of act(a b^T + bias) + residual (forward) or of a b (the input's gradient).  65536 rows, 1024 -> 4096,
// bf16: 550 GFLOP; the bare product 540 to 615 us (900 to 1020 TFLOP/s), bound by the feeding of the matrix
// instructions.  With bias, gelu, the sums kept and a residual 800 to 980 us (the least over and over, the most in a
// training step): 1.1 GB more, which come in bursts as the workgroups, one a CU, reach their ends together (120 us
// at least), and the gelu's arithmetic (about 80).
template <class T, bool kForward, Way kWay, int kBM, int kBN, int kWM, int kWN, int kStages>
__global__ __launch_bounds__(64 * (kBM / kWM) * (kBN / kWN)) void rows_kernel(RowsArgs a, uint32_t first, uint32_t blocks) {
    using Work = Tile<T, true, kForward, kWay, kBM, kBN, kWM, kWN, kStages>;
    __shared__ __attribute__((aligned(16))) char lds[Work::kLds];
    const uint32_t id = first + xcd_major(blockIdx.x, gridDim.x);
    if (id >= blocks) return;
    const TileAt t = tile_at(id, static_cast<uint32_t>(a.tiles), (a.columns + kBN - 1) / kBN);
    const Piece p = find_piece(a.offsets, a.experts, a.experts + 1, a.rows, kBM, t.row);
    if (p.begin >= p.end) return;
    const int column0 = static_cast<int>(t.column) * kBN;
    if (p.group >= a.experts) return rows_of_none<T, kBM, kBN, Work::kThreads>(a, p, column0);
    const int64_t matrix = static_cast<int64_t>(a.columns) * a.depth;
    const T* b = static_cast<const T*>(a.b) + p.group * matrix;
    typename Work::A opa;
    typename Work::B opb;
    opa.begin(static_cast<const T*>(a.a), a.lda, p.begin, p.end, a.depth);
    opb.begin(b, kForward ? a.depth : a.columns, column0, a.columns, a.depth);
    Work work;
    work.sum(opa, opb, a.depth, lds);
    finish_tile<T, kBM == 256>(work, a, p, column0, lds);   // 256: taken for outputs near the L2s' size and larger alone (17 MB at least)
}

// Few rows a group: the weights are read once for every 16 kRowTiles rows, straight into registers in the layout of the
// products, and everything else is small beside them.  A wave takes 16 columns of the output, 16 kRowTiles rows and one of
// kSplit shares of the depth, of which it has several hundred bytes of every weight row under way; the
// shares' sums are added in order through LDS.  Bound by the latency of one chain of loads: one bf16 row through
// 2048 x 2048 (8.4 MB) 4.9 us; 16 rows over 64 fp16 experts of 512 -> 1024 (17 MB of
// weights touched) 9.5 us.
template <class T, int kRowTiles, int kSplit> __global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(RowsArgs a) {
    constexpr int kColumns = 16 * kFewWaves / kSplit;   // of a workgroup
    __shared__ accum4 part[kFewWaves][kRowTiles][64];
    constexpr int kStep = 4 * kPerVec<T>;          // k values a wave takes at a time
    constexpr int kAhead = kRowTiles == 1 ? 8 : 4; // steps in flight
    const uint32_t across = (a.columns + kColumns - 1) / kColumns;
    const Piece p = find_piece(a.offsets, a.experts, a.experts + 1, a.rows, 16 * kRowTiles, blockIdx.x / across);
    if (p.begin >= p.end) return;
    const int column0 = static_cast<int>(blockIdx.x % across) * kColumns;
    const int lane = static_cast<int>(threadIdx.x % 64);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
    const bool owned = p.group < a.experts;        // else rows of no expert
    if (owned && column0 + wave / kSplit * 16 < a.columns) {
        const int own = lane % 16, quarter = lane / 16 * kPerVec<T>;
        int column = column0 + wave / kSplit * 16 + own;
        column = column < a.columns ? column : a.columns - 1;   // those past the last are not stored
        const T* w = static_cast<const T*>(a.b) + (static_cast<int64_t>(p.group) * a.columns + column) * a.depth;
        const T* x[kRowTiles];
#pragma unroll
        for (int t = 0; t < kRowTiles; ++t) {
            const int64_t row = p.begin + 16 * t + own;
            x[t] = static_cast<const T*>(a.a) + (row < p.end ? row : p.end - 1) * a.lda;
        }
        accum4 acc[kRowTiles] = {};
        const int share = ((a.depth + kStep - 1) / kStep + kSplit - 1) / kSplit * kStep;
        const int first = wave % kSplit * share, last = first + share < a.depth ? first + share : a.depth;
        for (int k0 = first; k0 < last; k0 += kAhead * kStep) {
            vec16 fw[kAhead], fx[kAhead][kRowTiles];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int k = k0 + u * kStep + quarter, count = last - k;
                if (k0 + u * kStep + kStep <= last) {
                    fw[u] = load16(w + k);
#pragma unroll
                    for (int t = 0; t < kRowTiles; ++t) fx[u][t] = load16(x[t] + k);
                } else {
                    fw[u] = count > 0 ? load_end(w + k, count, k) : vec16{};
#pragma unroll
                    for (int t = 0; t < kRowTiles; ++t) fx[u][t] = count > 0 ? load_end(x[t] + k, count, k) : vec16{};
                }
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
                for (int t = 0; t < kRowTiles; ++t) acc[t] = multiply16(T{}, fw[u], fx[u][t], acc[t]);
        }
#pragma unroll
        for (int t = 0; t < kRowTiles; ++t) part[wave][t][lane] = acc[t];
    }
    __syncthreads();
    finish_few<T, kRowTiles, kSplit>(part, a, p, column0, owned);
}

// One tile of one piece of rows: dw[e] = dz^T x where the piece is all of the expert's rows, else a partial sum
// that fold_kernel adds up in order.  Both operands are stored one row per k and are transposed as they leave LDS.
// 65536 rows, 4096 x 1024, bf16: 520 us (1060 TFLOP/s), bound like rows_kernel.
template <class T, Way kWay, int kBM, int kBN, int kWM, int kWN>
__global__ __launch_bounds__(64 * (kBM / kWM) * (kBN / kWN)) void weight_kernel(WeightArgs a, uint32_t blocks) {
    using Work = Tile<T, false, false, kWay, kBM, kBN, kWM, kWN, kBM == 64 ? 4 : 2>;
    __shared__ __attribute__((aligned(16))) char lds[Work::kLds];
    const uint32_t across = (a.inputs + kBN - 1) / kBN, down = (a.outputs + kBM - 1) / kBM, tiles = down * across;
    // A piece's tiles share its rows in one XCD's L2.  Several experts' pieces differ in length, and an XCD could be
    // left with the long ones: where there are tiles enough each piece is spread over the XCDs instead, eighths of
    // its tiles together (bf16, 131072 x 1024 x 1024 over 64 experts: 604 -> 561 us, 262144 x 512 x 2048 over 8: 1180 ->
    // 921; but 131072 x 256 x 512 over 64, 8 tiles a piece: 104 -> 148).
    const bool spread = a.offsets && tiles >= 64 && tiles % kXcds == 0;
    const uint32_t id = spread ? blockIdx.x : xcd_major(blockIdx.x, gridDim.x);
    if (id >= blocks) return;
    const uint32_t piece = id / tiles;
    uint32_t tile = id % tiles;
    if (spread) tile = tile % kXcds * (tiles / kXcds) + tile / kXcds;
    const TileAt t = tile_at(tile, down, across);
    const Piece p = find_piece(a.offsets, a.experts, a.experts, a.rows, a.piece, piece);
    if (p.first > 0 && p.begin >= p.end) return;
    const int row0 = static_cast<int>(t.row) * kBM, column0 = static_cast<int>(t.column) * kBN;
    Work work;
    const int64_t depth = p.end > p.begin ? p.end - p.begin : 0;
    typename Work::A opa;
    typename Work::B opb;
    opa.begin(static_cast<const T*>(a.dz) + p.begin * a.ldz, a.ldz, row0, a.outputs, depth);
    opb.begin(static_cast<const T*>(a.x) + p.begin * a.ldx, a.ldx, column0, a.inputs, depth);
    work.sum(opa, opb, depth, lds);   // no rows: zeros
    const int64_t matrix = static_cast<int64_t>(a.outputs) * a.inputs;
    const bool whole = p.group_end - p.group_begin <= a.piece;
    T* dw = static_cast<T*>(a.dw) + p.group * matrix;
    float* partial = whole ? nullptr : a.partial + partial_slot(p.group_begin, a.piece, p.first) * matrix;
    const int column = column0 + Work::own_column(), count = a.inputs - column;
    work.rows(
        lds, [](int) { return 0; },
        [&](int r, float value[Work::kGroup][8], int) {
#pragma unroll
            for (int u = 0; u < Work::kGroup; ++u) {
                const int row = row0 + r + u * Work::kHeight;
                if (row >= a.outputs || count <= 0) continue;
                const int64_t at = static_cast<int64_t>(row) * a.inputs + column;
                if (whole) store8(dw + at, count, value[u]);
                else store8(partial + at, count, value[u]);
            }
        });
}

constexpr int kSlopeBlock = 256;

// dz = dy act'(pre), rounded to the tensors' type as every operand of a 16-bit product is, and its column sums,
// which take dz before that rounding (its slope is that of the kept sums).  The rounding is most of what the gradients
// are off by beside their own: 65536 x 1024 -> 4096 bf16, gelu, dx and dw relative to 64 bits 0.0024; the result's own
// rounding alone 0.0017, with the kept sums' 0.00175, with dz's 0.00235.  A workgroup takes one piece of rows and `lanes` groups of 8 columns;
// 256 / lanes rows at a time.  Bound by HBM: 65536 x 4096 bf16 gelu 322 us, 1.6 GB at 5.0 TB/s.
template <class T, bool kStream> __global__ __launch_bounds__(kSlopeBlock) void slope_kernel(SlopeArgs a, int lanes, uint32_t across) {
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
        const int64_t start = p.begin + static_cast<int>(threadIdx.x) / lanes;
        constexpr int kAhead = 4;   // rows whose loads are in flight together
        with_activation(dz ? a.activation : kNone, [&](auto activation) {
            for (int64_t row = start; row < p.end; row += kAhead * height) {
                float d[kAhead][8], z[kAhead][8];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int64_t r = row + u * height < p.end ? row + u * height : row;
                    load8(dy + r * a.ldy + column, count, d[u]);
                    if (activation != kNone) load8(pre + r * a.columns + column, count, z[u]);
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int64_t r = row + u * height;
                    if (r >= p.end) break;
                    if (activation != kNone) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) d[u][i] *= slope<activation, sizeof(T) == 4>(z[u][i]);
                        store8<kStream>(dz + r * a.columns + column, count, d[u]);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[i] += d[u][i];
                }
            }
        });
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

// A workgroup takes 256 / kGroups elements; its groups take every kGroups-th piece, added up at the end in order.
template <class T, int kGroups> __global__ __launch_bounds__(256) void fold_kernel(FoldArgs a) {
    constexpr int kLanes = 256 / kGroups;
    __shared__ float total[kGroups > 1 ? 256 : 1];
    const int lane = static_cast<int>(threadIdx.x) % kLanes, group = static_cast<int>(threadIdx.x) / kLanes;
    const int e = static_cast<int>(blockIdx.y);
    const int64_t begin = a.offsets ? group_start(a.offsets, e, a.rows) : 0;
    const int64_t end = a.offsets ? group_start(a.offsets, e + 1, a.rows) : a.rows;
    const int64_t first = a.single ? (a.offsets ? whole_pieces(a.offsets, e, a.rows, a.piece) + e : 0)
                                   : partial_slot(begin, a.piece, 0);
    const int64_t pieces = end > begin ? (end - begin + a.piece - 1) / a.piece : 0;
    if (pieces <= 1 && !a.single) return;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kLanes; base < a.size; base += static_cast<int64_t>(gridDim.x) * kLanes) {
        const int64_t i = base + lane;
        float sum = 0.0f;
        if (i < a.size) {
            const float* from = a.partial + first * a.size + i;
#pragma unroll 4
            for (int64_t p = group; p < pieces; p += kGroups) sum += from[p * a.size];
        }
        if constexpr (kGroups > 1) {
            total[threadIdx.x] = sum;
            __syncthreads();
            if (group == 0)
                for (int g = 1; g < kGroups; ++g) sum += total[g * kLanes + lane];
            __syncthreads();
        }
        if (group == 0 && i < a.size) static_cast<T*>(a.out)[e * a.size + i] = static_cast<T>(sum);
    }
}

template <class T, bool kForward, Way kWay, int kBM, int kBN, int kWM, int kWN, int kStages = 2>
int launch_rows_as(RowsArgs a, hipStream_t stream) {
    const int64_t across = (a.columns + kBN - 1) / kBN;
    a.tiles = piece_ids(a.rows, kBM, a.offsets != nullptr, a.experts, true);
    const int64_t blocks = a.tiles * across;
    if (blocks >= int64_t{1} << 31) return fail("linear: too many tiles for one launch");
    constexpr int kThreads = 64 * (kBM / kWM) * (kBN / kWN);
    in_launches(blocks, kThreads, [&](uint32_t first, uint32_t count) {
        rows_kernel<T, kForward, kWay, kBM, kBN, kWM, kWN, kStages>
            <<<whole_xcds(count), kThreads, 0, stream>>>(a, first, static_cast<uint32_t>(blocks));
    });
    return check_launch("linear");
}

template <class T, int kRowTiles, int kSplit> int launch_few_rows_as(const RowsArgs& a, hipStream_t stream) {
    const int64_t across = (a.columns + 16 * kFewWaves / kSplit - 1) / (16 * kFewWaves / kSplit);
    const int64_t blocks = piece_ids(a.rows, 16 * kRowTiles, a.offsets != nullptr, a.experts, true) * across;
    if (blocks > most_blocks(64 * kFewWaves)) return fail("linear: too many tiles for one launch");
    few_rows_kernel<T, kRowTiles, kSplit><<<static_cast<uint32_t>(blocks), 64 * kFewWaves, 0, stream>>>(a);
    return check_launch("linear");
}

// The depth is split over all eight waves where a share is still long or there are too few workgroups otherwise.  us
// with eight shares and with two: one bf16 row, 2048 -> 2048 4.6 and 11.1, 512 -> 4096 3.6 and 4.7, 512 -> 16384 6.4
// and 5.0; 16 fp16 rows over 64 experts of 512 -> 1024 12.5 and 8.3.  Long shares with workgroups enough lose a little:
// 2048 -> 16384 15.2 and 12.5, 4096 -> 16384 22.1 and 21.8.
template <class T, int kRowTiles> int launch_few_rows(const RowsArgs& a, hipStream_t stream) {
    const int64_t steps = a.depth / (4 * kPerVec<T>);
    const int64_t busy = a.rows < a.experts ? a.rows : a.experts;
    if (steps >= 64 || busy * a.columns < 64 * kCus) return launch_few_rows_as<T, kRowTiles, 8>(a, stream);
    return launch_few_rows_as<T, kRowTiles, 2>(a, stream);
}

// Tiles by the work there is (us of one bf16 product, 65536 x 1024 x 4096; and with its epilogue, 131072 x 256 x 512
// over 64 experts):
//   256 x 256, 64 x 128 a wave   620, 112  where they go round and a group's rows fill them (the path through
//                                          registers has no room)
//   128 x 128, 64 x 64 a wave    777, 130  two a CU, where they go round
//   128 x 64, 32 x 64 a wave     narrow outputs: no columns wasted (64 -> 64 fp16: 262144 rows 14.8 us, as 64 x 64
//                                25.3; 32768 rows 4.9 and 5.1; 16384 rows 4.5 and 4.2)
//   64 x 64, 32 x 32 a wave      what is left; straight to LDS with three slabs under way (seven are no
//                                faster: 512 x 2048 x 2048 14.4 us with three, 15.5 with seven)
// Tiles that leave CUs idle in their last round are passed over where the products bound them: the largest, and fp32's
// (4096 x 1023 x 1025: 288 tiles of 128 x 128 155 us, 1105 of 64 x 64 119 us; in bf16 31 and 37).
template <class T, bool kForward, Way kWay> int launch_rows_of(const RowsArgs& a, hipStream_t stream) {
    const int64_t each = a.rows / a.experts;   // rows of a group, on average
    const int64_t large = (a.rows + 255) / 256 * ((a.columns + 255) / 256);
    const int64_t wide = (a.rows + 127) / 128 * ((a.columns + 127) / 128);
    if constexpr (kWay == kDirect)
        if (a.columns > 128 && even(large) && each >= 1024)
            return launch_rows_as<T, kForward, kWay, 256, 256, 64, 128>(a, stream);
    if constexpr (kWay != kGathered) {
        if (a.columns <= 64 && a.rows >= 128 * kCus) return launch_rows_as<T, kForward, kWay, 128, 64, 32, 64>(a, stream);
        if (a.columns > 64 && (sizeof(T) == 4 ? even(wide) : wide >= kCus) && each >= 128)
            return launch_rows_as<T, kForward, kWay, 128, 128, 64, 64>(a, stream);
    }
    return launch_rows_as<T, kForward, kWay, 64, 64, 32, 32, kWay == kDirect ? 4 : 2>(a, stream);
}

template <class T, bool kForward> int launch_rows_by(Way way, const RowsArgs& a, hipStream_t stream) {
    if (way == kDirect) return launch_rows_of<T, kForward, kDirect>(a, stream);
    if (way == kStaged) return launch_rows_of<T, kForward, kStaged>(a, stream);
    return launch_rows_of<T, kForward, kGathered>(a, stream);
}

template <class T, Way kWay, int kBM, int kBN, int kWM, int kWN> int launch_weight_as(const WeightArgs& a, hipStream_t stream) {
    const int64_t tiles = static_cast<int64_t>((a.outputs + kBM - 1) / kBM) * ((a.inputs + kBN - 1) / kBN);
    const int64_t blocks = a.pieces * tiles;
    if (blocks > most_blocks(64 * (kBM / kWM) * (kBN / kWN))) return fail("linear: too many tiles for one launch");
    weight_kernel<T, kWay, kBM, kBN, kWM, kWN>
        <<<whole_xcds(blocks), 64 * (kBM / kWM) * (kBN / kWN), 0, stream>>>(a, static_cast<uint32_t>(blocks));
    return check_launch("linear weight gradient");
}

}  // namespace

template <class T> int launch_rows(const RowsArgs& a, bool forward, hipStream_t stream) {
    if (forward) {
        // Groups of varying sizes: room for twice the average.  us of 16, 32, 64 rows a piece, and of tiles: 2048 -> 2048
        // bf16, 16, 32, 64 rows 6.1, 7.8, 11.7 and 14.5 to 14.7 (128 rows 11.9 and 14.8); fp32, 64 rows 26 and 50.  Over 64
        // fp16 experts of 512 -> 1024, 16 and 64 rows in all 8.9, 13.1 and 13.1, 17.5; groups of several rows read
        // their weights for each piece, and tiles would be faster: 512 rows 21.9 and 18.9, 2048 rows 39.5 and 23.9.
        const int64_t each = (a.rows + a.experts - 1) / a.experts * (a.experts > 1 ? 2 : 1);
        if (each <= 16) return launch_few_rows<T, 1>(a, stream);
        if (each <= 32) return launch_few_rows<T, 2>(a, stream);
        if (each <= 64) return launch_few_rows<T, 4>(a, stream);
        return launch_rows_by<T, true>(slower(way_of<T>(a.a, a.lda, a.depth), way_of<T>(a.b, a.depth, a.depth)), a, stream);
    }
    return launch_rows_by<T, false>(slower(way_of<T>(a.a, a.lda, a.depth), way_of<T>(a.b, a.columns, a.columns)), a, stream);
}

template <class T, Way kWay> int launch_weight_of(const WeightArgs& a, hipStream_t stream) {
    if constexpr (kWay == kDirect)
        if (a.edge == 256) return launch_weight_as<T, kWay, 256, 256, 64, 128>(a, stream);
    if constexpr (kWay != kGathered)
        if (a.edge >= 128) return launch_weight_as<T, kWay, 128, 128, 64, 64>(a, stream);
    return launch_weight_as<T, kWay, 64, 64, 32, 32>(a, stream);
}

template <class T> int launch_weight(const WeightArgs& a, hipStream_t stream) {
    const Way way = slower(way_of<T>(a.dz, a.ldz, a.outputs), way_of<T>(a.x, a.ldx, a.inputs));
    if (way == kDirect) return launch_weight_of<T, kDirect>(a, stream);
    if (way == kStaged) return launch_weight_of<T, kStaged>(a, stream);
    return launch_weight_of<T, kGathered>(a, stream);
}

template <class T> int launch_slope(const SlopeArgs& a, hipStream_t stream) {
    const int groups = (a.columns + 7) / 8, lanes = slope_lanes(a.columns);
    const int64_t across = (groups + lanes - 1) / lanes, blocks = a.pieces * across;
    if (blocks > most_blocks(kSlopeBlock)) return fail("linear: too many workgroups for one launch");
    if (blocks == 0) return 0;
    with_flag(a.rows * a.columns * static_cast<int64_t>(sizeof(T)) >= kStreamBytes, [&](auto far) {
        slope_kernel<T, far><<<static_cast<uint32_t>(blocks), kSlopeBlock, 0, stream>>>(a, lanes, static_cast<uint32_t>(across));
    });
    return check_launch("linear activation gradient");
}

template <class T> int launch_fold(const FoldArgs& a, hipStream_t stream) {
    // many pieces of few elements (a bias): several groups share them (us, shared and not: a bias over 2^20 x 64 fp16
    // 36 and 158 with its slope pass, over 131072 x 512 and 64 experts 27 and 26; a weight gradient of 64 x 64 over
    // 65536 rows 10 and 25, of 1024 x 1024 over 4096, four pieces, 41 and 25)
    const bool tall = a.rows / a.piece >= 8 * static_cast<int64_t>(a.experts);
    const int64_t lanes = tall ? 16 : 256;
    // most experts' groups are whole and have nothing to add: few workgroups each
    const int64_t most = a.experts > 1 ? 16 * kCus / a.experts + 8 : 16 * kCus;
    const int64_t blocks = (a.size + lanes - 1) / lanes < most ? (a.size + lanes - 1) / lanes : most;
    const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(a.experts));
    if (tall) fold_kernel<T, 16><<<grid, 256, 0, stream>>>(a);
    else fold_kernel<T, 1><<<grid, 256, 0, stream>>>(a);
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
