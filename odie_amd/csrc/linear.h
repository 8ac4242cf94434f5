// Matrix products with a fused epilogue on MFMA: the tile engine of linear.hip, compiled per element
// type (linear_f16.hip, linear_bf16.hip, linear_f32.hip).
//
// Every product is C[m][n] = sum_k A(m, k) B(n, k).  An operand lies in memory either with k
// consecutive (rows of k) or with its own index consecutive (one row per k):
//   forward   y[m][n]  = sum_k  x[m][k]  w[n][k]     both with k consecutive
//   input     dx[m][k] = sum_n  dz[m][n] w[n][k]     dz with n consecutive, w one row per n
//   weight    dw[n][k] = sum_m  dz[m][n] x[m][k]     both one row per m
//
// A workgroup owns a kBM x kBN tile of C and walks k in slabs of 128 bytes (64 16-bit or 32 fp32
// values).  Per slab both operands pass through LDS in their memory orientation: global loads of the
// next slab are in flight while the current one is multiplied, two LDS buffers, one barrier a slab.
// A 16-bit operand stored one row per k is turned by ds_read_b64_tr_b16 as it is read.  Products are
// v_mfma_f32_32x32x16 (16-bit) or v_mfma_f32_32x32x2 (fp32), accumulated in fp32.
//
// The epilogue passes each wave's accumulators through its own part of the LDS, so that bias,
// activation, residual and the stores run on rows of 8 consecutive columns a lane.
#pragma once
#include "elements.h"

namespace odie {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float accum16 __attribute__((ext_vector_type(16)));
typedef int16_t i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4* lds_i16x4;

constexpr int kSlabBytes = 128;
template <class T> constexpr int kSlab = kSlabBytes / static_cast<int>(sizeof(T));   // k values a slab

// acc[n][m] += sum over the 16 bytes of k that each lane holds (lane l: row l % 32, k half l / 32).
__device__ inline accum16 multiply(_Float16, const vec16& b, const vec16& a, accum16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
}
__device__ inline accum16 multiply(__bf16, const vec16& b, const vec16& a, accum16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
}
__device__ inline accum16 multiply(float, const vec16& b, const vec16& a, accum16 c) {
    float fb[4], fa[4];
    __builtin_memcpy(fb, &b, 16);
    __builtin_memcpy(fa, &a, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[i], fa[i], c, 0, 0, 0);
    return c;
}

// One operand of a tile: kRows of its own index times one slab of k, kThreads threads.
// LDS image, k consecutive: kRows rows of 128 bytes; the 16-byte chunk c of row r lies at slot
// c ^ (r / 2 % 8), so that 16 consecutive rows of one chunk fall on all 64 banks.
// LDS image, one row per k: rows of kRows elements; chunk c of row k lies at slot c ^ turn(k), so
// that the rows one transposing read touches at once (k .. k + 3, 32 columns) fall on all 64 banks.
template <class T, bool kByRow, int kRows, int kThreads> struct Operand {
    static constexpr int kBytes = kRows * kSlabBytes;
    static constexpr int kChunks = kRows * 8 / kThreads;       // 16-byte chunks a thread moves per slab
    static constexpr int kVec = kPerVec<T>;
    static constexpr int kPerRow = kRows / kVec;                // chunks a row (one row per k)
    static_assert(kChunks * kThreads == kRows * 8 && (kByRow || kThreads % kPerRow == 0), "whole chunks a thread");

    vec16 held[kChunks];
    const T* at[kByRow ? kChunks : 1];
    int64_t row_step;    // one row per k: elements between this thread's consecutive chunks
    int64_t slab_step;   // elements from slab to slab
    int lead;            // k of this thread's first chunk, relative to the slab
    int columns;         // one row per k: columns of this thread's chunk inside the tensor

    // One row per k: XOR on the chunk index of row k.
    static __device__ int turn(int k) {
        if constexpr (sizeof(T) == 4) return (k >> 2 & 1) << 3;
        return kPerRow >= 16 ? (k & 3) << 2 : (k >> 1 & 1) << 2;
    }

    // k consecutive: rows first .. first + kRows - 1 of base (those past last read row `last`, their
    // products are not stored).  One row per k: columns first .. of base, `limit` of them in all.
    __device__ void begin(const T* base, int64_t stride, int64_t first, int64_t limit) {
        const int thread = static_cast<int>(threadIdx.x);
        if constexpr (kByRow) {
            lead = thread % 8 * kVec;
            slab_step = kSlab<T>;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int64_t row = first + thread / 8 + i * (kThreads / 8);
                at[i] = base + (row < limit ? row : limit - 1) * stride + lead;
            }
        } else {
            lead = thread / kPerRow;
            const int64_t column = first + thread % kPerRow * kVec;
            const int64_t left = limit - column;
            columns = left >= kVec ? kVec : (left > 0 ? static_cast<int>(left) : 0);
            at[0] = base + lead * stride + column;
            row_step = kThreads / kPerRow * stride;
            slab_step = kSlab<T> * stride;
        }
    }

    // Starts the loads of the next slab, of which `left` values of k exist (the rest read as 0).
    __device__ void load(int64_t left) {
        if constexpr (kByRow) {
            if (left >= kSlab<T>) {
#pragma unroll
                for (int i = 0; i < kChunks; ++i) held[i] = load16(at[i]);
            } else {
                const int count = static_cast<int>(left) - lead;
#pragma unroll
                for (int i = 0; i < kChunks; ++i) held[i] = count > 0 ? load_some(at[i], count) : vec16{};
            }
#pragma unroll
            for (int i = 0; i < kChunks; ++i) at[i] += slab_step;
        } else {
            constexpr int kStride = kThreads / kPerRow;
            if (left >= kSlab<T> && columns == kVec) {
#pragma unroll
                for (int i = 0; i < kChunks; ++i) held[i] = load16(at[0] + i * row_step);
            } else {
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    const bool inside = lead + i * kStride < left && columns > 0;
                    held[i] = inside ? load_some(at[0] + i * row_step, columns) : vec16{};
                }
            }
            at[0] += slab_step;
        }
    }

    __device__ void store(char* lds) const {
        const int thread = static_cast<int>(threadIdx.x);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            int to;
            if constexpr (kByRow) {
                const int row = thread / 8 + i * (kThreads / 8);
                to = row * kSlabBytes + ((thread % 8 ^ (row >> 1 & 7)) << 4);
            } else {
                const int k = lead + i * (kThreads / kPerRow);
                to = k * (kPerRow * 16) + ((thread % kPerRow ^ turn(k)) << 4);
            }
            *reinterpret_cast<vec16*>(lds + to) = held[i];
        }
    }

    // The 16 bytes of k that lane l holds of row base + l % 32: k chunk 2 * step + l / 32.
    static __device__ vec16 fragment(const char* lds, int base, int step, int lane) {
        if constexpr (kByRow) {
            const int row = base + lane % 32;
            return *reinterpret_cast<const vec16*>(lds + row * kSlabBytes + (((2 * step + lane / 32) ^ (row >> 1 & 7)) << 4));
        } else if constexpr (sizeof(T) == 4) {
            const int column = base + lane % 32, k = 8 * step + 4 * (lane / 32);
            vec16 v;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = *reinterpret_cast<const uint32_t*>(lds + (k + i) * (kPerRow * 16) + ((column >> 2 ^ turn(k + i)) << 4) + (column & 3) * 4);
            return v;
        } else {
            // Each group of 16 lanes fetches 4 rows of k times 16 columns and gets back 4 values of k of
            // its own column: lane j fetches columns 4 (j % 4) .. + 3 of row j / 4.
            const int j = lane % 16, group = lane / 16;
            const int column = base + group % 2 * 16 + j % 4 * 4;
            i16x4 part[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = 16 * step + 8 * (group / 2) + 4 * h + j / 4;
                const char* p = lds + k * (kPerRow * 16) + ((column >> 3 ^ turn(k)) << 4) + (column & 4) * 2;
                part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(p));
            }
            vec16 v;
            __builtin_memcpy(&v, part, 16);
            return v;
        }
    }
};

// One workgroup's tile: kWaves waves in kBM / kWM x kBN / kWN.
template <class T, bool kAByRow, bool kBByRow, int kBM, int kBN, int kWM, int kWN> struct Tile {
    static constexpr int kThreads = 64 * (kBM / kWM) * (kBN / kWN);
    using A = Operand<T, kAByRow, kBM, kThreads>;
    using B = Operand<T, kBByRow, kBN, kThreads>;
    static constexpr int kMs = kWM / 32, kNs = kWN / 32;
    static constexpr int kBuffer = A::kBytes + B::kBytes;
    static constexpr int kPitch = kWN + 4;                  // floats a row of the epilogue's region
    static constexpr int kRegion = 32 * kPitch * 4;
    static constexpr int kLds = 2 * kBuffer > kThreads / 64 * kRegion ? 2 * kBuffer : kThreads / 64 * kRegion;

    accum16 acc[kMs][kNs];

    // Sums `depth` values of k.  a and b have begun.
    __device__ void sum(A& a, B& b, int64_t depth, char* lds) {
        const int lane = static_cast<int>(threadIdx.x % 64);
        const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
        const int wm = wave % (kBM / kWM) * kWM, wn = wave / (kBM / kWM) * kWN;
#pragma unroll
        for (int i = 0; i < kMs; ++i)
#pragma unroll
            for (int j = 0; j < kNs; ++j) acc[i][j] = accum16{};
        a.load(depth);
        b.load(depth);
        a.store(lds);
        b.store(lds + A::kBytes);
        __syncthreads();
        int buffer = 0;
        for (int64_t k = 0; k < depth; k += kSlab<T>) {
            const char* now = lds + buffer * kBuffer;
            const bool more = k + kSlab<T> < depth;
            if (more) {
                a.load(depth - k - kSlab<T>);
                b.load(depth - k - kSlab<T>);
            }
#pragma unroll
            for (int step = 0; step < kSlabBytes / 32; ++step) {
                vec16 fa[kMs], fb[kNs];
#pragma unroll
                for (int i = 0; i < kMs; ++i) fa[i] = A::fragment(now, wm + 32 * i, step, lane);
#pragma unroll
                for (int j = 0; j < kNs; ++j) fb[j] = B::fragment(now + A::kBytes, wn + 32 * j, step, lane);
#pragma unroll
                for (int i = 0; i < kMs; ++i)
#pragma unroll
                    for (int j = 0; j < kNs; ++j) acc[i][j] = multiply(T{}, fb[j], fa[i], acc[i][j]);
            }
            buffer ^= 1;
            if (more) {
                a.store(lds + buffer * kBuffer);
                b.store(lds + buffer * kBuffer + A::kBytes);
            }
            __syncthreads();
        }
    }

    // Hands out the tile's values in rows: f(row, column, value[8]) with row and column relative to the tile.
    template <class F> __device__ void rows(char* lds, F&& f) {
        const int lane = static_cast<int>(threadIdx.x % 64);
        const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
        const int wm = wave % (kBM / kWM) * kWM, wn = wave / (kBM / kWM) * kWN;
        float* region = reinterpret_cast<float*>(lds + wave * kRegion);
        constexpr int kLanes = kWN / 8, kPass = 64 / kLanes;
#pragma unroll
        for (int i = 0; i < kMs; ++i) {
            // accumulator element v of lane l: row l % 32, column 8 (v / 4) + 4 (l / 32) + v % 4
            float* to = region + lane % 32 * kPitch + lane / 32 * 4;
#pragma unroll
            for (int j = 0; j < kNs; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4*>(to + 32 * j + 8 * q) =
                        make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
            wave_fence();
#pragma unroll
            for (int pass = 0; pass < 32 / kPass; ++pass) {
                const int row = pass * kPass + lane / kLanes, column = lane % kLanes * 8;
                const float* from = region + row * kPitch + column;
                const float4 lo = *reinterpret_cast<const float4*>(from), hi = *reinterpret_cast<const float4*>(from + 4);
                float value[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                f(wm + 32 * i + row, wn + column, value);
            }
            wave_fence();
        }
    }
};

enum Activation { kNone = 0, kRelu, kSigmoid, kSoftplus, kGelu, kSilu, kActivations };

// exp of the negated absolute value never overflows; a NaN stays one.
__device__ inline float activate(int activation, float z) {
    switch (activation) {
        case kRelu: return z < 0.0f ? 0.0f : z;
        case kSigmoid: return 1.0f / (1.0f + expf(-z));
        case kSoftplus: return (z > 0.0f ? z : 0.0f) + log1pf(expf(-fabsf(z)));
        case kGelu: return 0.5f * z * erfcf(-0.70710678f * z);
        case kSilu: return z / (1.0f + expf(-z));
        default: return z;
    }
}

// Derivative at z.
__device__ inline float slope(int activation, float z) {
    switch (activation) {
        case kRelu: return z > 0.0f ? 1.0f : 0.0f;
        case kSigmoid: return 1.0f / ((1.0f + expf(-z)) * (1.0f + expf(z)));
        case kSoftplus: return 1.0f / (1.0f + expf(-z));
        case kGelu: return 0.5f * erfcf(-0.70710678f * z) + z * 0.39894228f * expf(-0.5f * z * z);
        case kSilu: {
            const float s = 1.0f / (1.0f + expf(-z));
            return s * (1.0f + z / (1.0f + expf(z)));
        }
        default: return 1.0f;
    }
}

struct RowsArgs {             // y = act(a b^T + bias) + residual over groups of rows
    const void* a;            // [rows][depth], stride lda
    const void* b;            // per expert [columns][depth] (forward) or [depth][columns] (input gradient)
    const void* bias;         // per expert [columns], or null
    const void* residual;     // [rows][columns], stride ldr, or null
    void* out;                // [rows][columns], stride ldo
    void* pre;                // the sums before the activation, [rows][columns], or null
    const int32_t* offsets;   // or null: one expert
    int64_t rows, lda, ldr, ldo;
    int64_t tiles;            // row tiles (piece ids)
    int experts, depth, columns, activation;
};

struct WeightArgs {           // dw[e] = dz^T x over each expert's rows
    const void* dz;           // [rows][outputs], stride ldz
    const void* x;            // [rows][inputs], stride ldx
    void* dw;                 // [experts][outputs][inputs]
    float* partial;           // [piece ids][outputs][inputs] sums of groups cut into several pieces
    const int32_t* offsets;
    int64_t rows, ldz, ldx;
    int64_t piece;            // rows a workgroup sums
    int64_t pieces;           // piece ids
    int experts, outputs, inputs;
};

struct SlopeArgs {            // dz = dy act'(pre), and the column sums of dz
    const void* dy;           // [rows][columns], stride ldy
    const void* pre;          // [rows][columns]
    void* dz;                 // [rows][columns], or null: dy is dz
    float* sums;              // [piece ids][columns], or null
    const int32_t* offsets;
    int64_t rows, ldy;
    int64_t piece, pieces;
    int experts, columns, activation;
};

struct FoldArgs {             // out[e][i] = sum over e's pieces of partial[piece][i]
    const float* partial;
    void* out;
    const int32_t* offsets;
    int64_t rows, piece, size;
    int experts;
    bool single;              // also the groups of one piece (and zeros for those of none)
};

// Launches, per element type.
template <class T> int launch_rows(const RowsArgs& a, bool forward, hipStream_t stream);
template <class T> int launch_weight(const WeightArgs& a, hipStream_t stream);
template <class T> int launch_slope(const SlopeArgs& a, hipStream_t stream);
template <class T> int launch_fold(const FoldArgs& a, hipStream_t stream);

}  // namespace odie
