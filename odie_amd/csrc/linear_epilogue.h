// What the products' kernels share beside the tile engine (linear_kernels.h, mx_kernels.h): the order of their tiles,
// rows of no expert, and the epilogue act(sums + bias) + residual of tiles and of few rows.
#pragma once
#include "linear.h"

namespace odie {
namespace {

constexpr uint32_t kBand = 4;

struct TileAt {
    uint32_t row, column;
};

// Tiles in bands of kBand rows, down each band's columns first: tiles that run at the same time on an XCD
// form a block of about kBand by 8, and read the fewest rows of both operands through its L2.
__device__ inline TileAt tile_at(uint32_t id, uint32_t down, uint32_t across) {
    const uint32_t band = id / (kBand * across), inside = id - band * kBand * across;
    const uint32_t high = down - band * kBand < kBand ? down - band * kBand : kBand;
    return TileAt{band * kBand + inside % high, inside / high};
}

// A tile of rows of no expert: the residual, or 0.
template <class T, int kBM, int kBN, int kThreads> __device__ inline void rows_of_none(const RowsArgs& a, const Piece& p, int column0) {
    const T* residual = static_cast<const T*>(a.residual);
    T* out = static_cast<T*>(a.out);
    for (int i = threadIdx.x; i < kBM * (kBN / 8); i += kThreads) {
        const int64_t row = p.begin + i / (kBN / 8);
        const int column = column0 + i % (kBN / 8) * 8;
        if (row >= p.end || column >= a.columns) continue;
        float value[8] = {};
        if (residual) load8(residual + row * a.ldr + column, a.columns - column, value);
        store8(out + row * a.ldo + column, a.columns - column, value);
    }
}

// The epilogue of a tile's sums.
template <class T, bool kStream, class Work>
__device__ inline void finish_tile(Work& work, const RowsArgs& a, const Piece& p, int column0, char* lds) {
    const T* bias = a.bias ? static_cast<const T*>(a.bias) + static_cast<int64_t>(p.group) * a.columns : nullptr;
    const T* residual = static_cast<const T*>(a.residual);
    T* out = static_cast<T*>(a.out);
    T* pre = static_cast<T*>(a.pre);
    constexpr int kGroup = Work::kGroup, kHeight = Work::kHeight;
    struct Fetched {
        Eight<T> row[kGroup];
    };
    const int column = column0 + Work::own_column(), count = a.columns - column;   // the lane's through every row
    float shift[8] = {};
    if (bias && count > 0) load8(bias + column, count, shift);
    work.rows(
        lds,
        [&](int r) {
            Fetched f{};
            if (residual && count > 0)
#pragma unroll
                for (int u = 0; u < kGroup; ++u) {
                    const int64_t row = p.begin + r + u * kHeight;
                    if (row < p.end) f.row[u].load(residual + row * a.ldr + column, count);
                }
            return f;
        },
        [&](int r, float value[kGroup][8], const Fetched& f) {
#pragma unroll
            for (int u = 0; u < kGroup; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) value[u][i] += shift[i];
            if (pre && count > 0)      // in T: linear.hip and mx_linear.hip say what that costs the gradients
#pragma unroll
                for (int u = 0; u < kGroup; ++u) {
                    const int64_t row = p.begin + r + u * kHeight;
                    if (row < p.end) store8<kStream>(pre + row * a.columns + column, count, value[u]);
                }
            with_activation(a.activation, [&](auto activation) {
#pragma unroll
                for (int u = 0; u < kGroup; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) value[u][i] = activate<activation, sizeof(T) == 4>(value[u][i]);
            });
#pragma unroll
            for (int u = 0; u < kGroup; ++u) {
                const int64_t row = p.begin + r + u * kHeight;
                if (row >= p.end || count <= 0) continue;
                if (residual) {
                    float more[8];
                    f.row[u].get(more);
#pragma unroll
                    for (int i = 0; i < 8; ++i) value[u][i] += more[i];
                }
                store8<kStream>(out + row * a.ldo + column, count, value[u]);
            }
        });
}

constexpr int kFewWaves = 8;

// The epilogue of few rows: the shares' sums of 16 x 16 tiles, added in order.
template <class T, int kRowTiles, int kSplit>
__device__ inline void finish_few(const accum4 (&part)[kFewWaves][kRowTiles][64], const RowsArgs& a, const Piece& p, int column0, bool owned) {
    constexpr int kColumns = 16 * kFewWaves / kSplit;
    const T* bias = a.bias && owned ? static_cast<const T*>(a.bias) + static_cast<int64_t>(p.group) * a.columns : nullptr;
    const T* residual = static_cast<const T*>(a.residual);
    T* out = static_cast<T*>(a.out);
    T* pre = static_cast<T*>(a.pre);
    for (int i = threadIdx.x; i < 16 * kRowTiles * kColumns; i += 64 * kFewWaves) {
        const int r = i / kColumns, c = i % 16, tile = i % kColumns / 16, column = column0 + i % kColumns;
        const int64_t row = p.begin + r;
        if (row >= p.end || column >= a.columns) continue;
        float value = 0.0f;
        if (owned) {
            // accumulator element v of lane l: row l % 16, column 4 (l / 16) + v
#pragma unroll
            for (int s = 0; s < kSplit; ++s) value += part[tile * kSplit + s][r / 16][c / 4 * 16 + r % 16][c % 4];
            if (bias) value += static_cast<float>(bias[column]);
            if (pre) pre[row * a.columns + column] = static_cast<T>(value);
            with_activation(a.activation, [&](auto activation) { value = activate<activation, sizeof(T) == 4>(value); });
        }
        if (residual) value += static_cast<float>(residual[row * a.ldr + column]);
        out[row * a.ldo + column] = static_cast<T>(value);
    }
}

uint32_t whole_xcds(int64_t blocks) { return static_cast<uint32_t>((blocks + kXcds - 1) / kXcds * kXcds); }

// The way to LDS of rows of `width` elements: directly where each row starts on 16 bytes and is a multiple of them.
template <class T> Way way_of(const void* data, int64_t stride, int64_t width) {
    const int64_t pitch = stride * static_cast<int64_t>(sizeof(T));
    if (width < kPerVec<T>) return kGathered;
    return reinterpret_cast<uintptr_t>(data) % 16 == 0 && pitch % 16 == 0 && width % kPerVec<T> == 0 &&
                   pitch < (int64_t{1} << 22)   // 256 rows of a tile within 2^30 bytes
               ? kDirect : kStaged;
}

inline Way slower(Way a, Way b) { return a > b ? a : b; }

// Whether `tiles` keep three quarters of the CUs busy to the end.
inline bool even(int64_t tiles) { return tiles >= kCus && 4 * tiles >= 3 * ((tiles + kCus - 1) / kCus * kCus); }

}  // namespace
}  // namespace odie
