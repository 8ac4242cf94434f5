// The gradient of a layer's rows through a 4-bit weight, dx = (dy act'(z)) w, with the column sums of dy act'(z), in
// one pass over dy and z where the inputs fit a tile: what a layer that stays as it is needs, and no more.  The weight
// lies in T here.
#pragma once
#include "linear_epilogue.h"

namespace odie {

struct MxInputArgs {
    // a: dy; b: the weight [experts][outputs], stride `pitch`; out: dx; depth: outputs; columns: inputs
    RowsArgs rows;
    const void* pre;      // z [rows][outputs]
    float* sums;          // [piece ids][outputs], or null
    int64_t pitch;
};

// The tile of such a gradient: rows, and the most inputs.
struct MxInputTile {
    int rows, inputs;
};
inline MxInputTile mx_input_tile(int inputs) {
    return MxInputTile{128, inputs <= 64 ? 64 : (inputs <= 128 ? 128 : 256)};
}

template <class T> int launch_mx_input(const MxInputArgs& a, hipStream_t stream);

namespace {

// dy and z on their way to LDS as dz = dy act'(z).  Loads as Staged's; a thread's chunks are of the same columns of a
// slab.  dz is rounded to T because the matrix instruction takes T, and so it is wherever a 16-bit layer's gradient is
// formed: that is most of what dx is off by beside its own rounding (mx_linear.hip).
template <class T, int kRows, int kThreads> struct SlopeRows : Image<T, true, kRows, kThreads> {
    using I = Image<T, true, kRows, kThreads>;
    struct Held {
        vec16 dy[I::kChunks], z[I::kChunks];
    };
    const T* dy[I::kChunks];
    const T* tile;                    // z of the tile's first row, uniform over the workgroup
    uint32_t z[I::kChunks];           // its rows' places from there
    int depth, next, lead, rows;      // rows: of this thread's, how many exist

    __device__ void begin(const T* dys, int64_t stride, const T* zs, int64_t first, int64_t limit, int outputs) {
        depth = outputs;
        next = 0;
        lead = I::chunk() * I::kVec;
        rows = 0;
        tile = zs + first * outputs;
#pragma unroll
        for (int i = 0; i < I::kChunks; ++i) {
            const int64_t at = first + I::row() + i * I::kStep, r = at < limit ? at : limit - 1;
            rows += at < limit;
            dy[i] = dys + r * stride;
            z[i] = static_cast<uint32_t>(r - first) * static_cast<uint32_t>(outputs);
        }
    }
    __device__ void load(Held& held) {
        const int k = next + lead < depth - I::kVec ? next + lead : depth - I::kVec;
#pragma unroll
        for (int i = 0; i < I::kChunks; ++i)
            held.dy[i] = load16(dy[i] + k), held.z[i] = load16(tile + (z[i] + static_cast<uint32_t>(k)));
        next += kSlab<T>;
    }
    // `left` columns of this slab exist; the rest become 0.  sum: this thread's rows' sums, before the rounding.
    template <int kActivation> __device__ void store(const Held& held, char* lds, int left,
                                                     float (&sum)[I::kVec]) const {
        const int count = left < kSlab<T> ? left - lead : kSlab<T>;
        const int moved = count < I::kVec ? (I::kVec - count) * static_cast<int>(sizeof(T)) : 0;
#pragma unroll
        for (int i = 0; i < I::kVec; ++i) sum[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < I::kChunks; ++i) {
            float d[I::kVec], at[I::kVec];
            widen<T>(held.dy[i], d);
            widen<T>(held.z[i], at);
#pragma unroll
            for (int e = 0; e < I::kVec; ++e) d[e] *= slope<kActivation, sizeof(T) == 4>(at[e]);
            vec16 v = narrow<T>(d);
            if (moved) {      // a slab's end: what was loaded from further back moves down
                v = count > 0 ? shift_down(v, moved) : vec16{};
#pragma unroll
                for (int e = 0; e < I::kVec; ++e) {
                    float other = 0.0f;
#pragma unroll
                    for (int f = 0; f < I::kVec; ++f) other = f == e + I::kVec - count ? d[f] : other;
                    at[e] = count > 0 && e < count ? other : 0.0f;
                }
            } else {
#pragma unroll
                for (int e = 0; e < I::kVec; ++e) at[e] = d[e];
            }
            if (i < rows)
#pragma unroll
                for (int e = 0; e < I::kVec; ++e) sum[e] += at[e];
            *reinterpret_cast<vec16*>(lds + (threadIdx.x + i * kThreads) * 16) = v;
        }
    }
    // Adds the sums of a wave's threads that hold the same columns: rows 8 apart in lanes, whose chunks turn with them.
    static __device__ void join(float (&sum)[I::kVec]) {
#pragma unroll
        for (int e = 0; e < I::kVec; ++e) {
            float s = sum[e];
            // the next row: lane ^ 8
            s += __builtin_bit_cast(float, dpp_move<0x128>(__builtin_bit_cast(uint32_t, s)));
            // two on: lane ^ 17
            s += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, s), 0x441F));
            s += __shfl_xor(s, 34);                                                               // four on
            sum[e] = s;
        }
    }
};

// Waits for this wave's LDS reads, then for the other waves; loads under way stay so.
__device__ inline void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A tile.  A slab's slope takes a workgroup three times as long as its products do, and all of its waves are at the one
// or the other: one buffer an operand, so that a CU has two workgroups, one at each.  131072 rows over 64 experts, 256
// <- 512 fp16, silu: 107 to 120 us, 335 MB at 2.8 to 3.1 TB/s (71 us at a large copy's rate).  With relu, whose slope is
// a comparison, 105, with gelu 142, without the sums 112: silu's arithmetic is 15 us of it.  Most is that a workgroup's
// loads, slopes, products and epilogue follow one another, and two workgroups a CU cover them only in part (256 x 256
// tiles with two buffers, one workgroup a CU: 142).
template <class T, int kBM, int kBN, int kWM, int kWN> struct InputTile : Sums<kBM, kBN, kWM, kWN> {
    using Base = Sums<kBM, kBN, kWM, kWN>;
    using Base::acc;
    using Base::kMs;
    using Base::kNs;
    using Base::kThreads;
    using A = SlopeRows<T, kBM, kThreads>;
    using B = Direct<T, false, kBN, kThreads>;
    static constexpr int kWaves = kThreads / 64, kColumns = kSlab<T>;
    static constexpr int kBytes = A::kBytes + B::kBytes + kWaves * kColumns * 4;
    static constexpr int kLds = kBytes > kWaves * Base::kRegion ? kBytes : kWaves * Base::kRegion;

    __device__ void add_slab(const char* rows, const char* weight) {
        const int lane = static_cast<int>(threadIdx.x % 64);
#pragma unroll
        for (int step = 0; step < kSlabBytes / 32; ++step) {
            vec16 fa[kMs], fb[kNs];
#pragma unroll
            for (int i = 0; i < kMs; ++i) fa[i] = A::fragment(rows, Base::wave_row() + 32 * i, step, lane);
#pragma unroll
            for (int j = 0; j < kNs; ++j) fb[j] = B::fragment(weight, Base::wave_column() + 32 * j, step, lane);
#pragma unroll
            for (int i = 0; i < kMs; ++i)
#pragma unroll
                for (int j = 0; j < kNs; ++j) acc[i][j] = multiply(T{}, fb[j], fa[i], acc[i][j]);
        }
    }

    // Sums `depth` columns of dz; their own sums go to `sums` (of this piece), unless it is null.
    template <int kActivation> __device__ void sum(A& a, B& b, int depth, float* sums, char* lds) {
        Base::clear();
        char* const weight = lds + A::kBytes;
        float* const parts = reinterpret_cast<float*>(weight + B::kBytes);
        typename A::Held held;
        a.load(held);
        b.load(depth, weight);
        for (int done = 0; done < depth; done += kColumns) {
            const int left = depth - done;
            float part[A::kVec];
            a.template store<kActivation>(held, lds, left, part);
            if (sums) {
                A::join(part);
                if (threadIdx.x % 64 < 8)
#pragma unroll
                    for (int e = 0; e < A::kVec; ++e) parts[Base::wave() * kColumns + a.lead + e] = part[e];
            }
            arrived<0>();
            if (left > kColumns) a.load(held);
            if (sums && threadIdx.x < kColumns && static_cast<int>(threadIdx.x) < left) {
                float total = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) total += parts[w * kColumns + threadIdx.x];
                sums[done + threadIdx.x] = total;
            }
            add_slab(lds, weight);
            reads_done();
            if (left > kColumns) b.load(left - kColumns, weight);
        }
    }
};

template <class T, int kBM, int kBN, int kWM, int kWN>
__global__ __launch_bounds__(64 * (kBM / kWM) * (kBN / kWN), 2) void mx_input_kernel(
    MxInputArgs m, uint32_t first, uint32_t blocks) {
    using Work = InputTile<T, kBM, kBN, kWM, kWN>;
    __shared__ __attribute__((aligned(16))) char lds[Work::kLds];
    const RowsArgs& a = m.rows;
    const uint32_t id = first + xcd_major(blockIdx.x, gridDim.x);
    if (id >= blocks) return;
    const Piece p = find_piece(a.offsets, a.experts, a.experts + 1, a.rows, kBM, id);
    if (p.begin >= p.end) return;
    if (p.group >= a.experts) return rows_of_none<T, kBM, kBN, Work::kThreads>(a, p, 0);
    typename Work::A opa;
    typename Work::B opb;
    opa.begin(static_cast<const T*>(a.a), a.lda, static_cast<const T*>(m.pre), p.begin, p.end, a.depth);
    opb.begin(static_cast<const T*>(a.b) + static_cast<int64_t>(p.group) * a.depth * m.pitch, m.pitch, 0, a.columns,
              a.depth);
    Work work;
    with_activation(a.activation, [&](auto activation) {
        work.template sum<activation>(opa, opb, a.depth,
                                     m.sums ? m.sums + static_cast<int64_t>(id) * a.depth : nullptr, lds);
    });
    RowsArgs plain = a;      // dx as it is
    plain.activation = kNone;
    finish_tile<T, kBN == 256>(work, plain, p, 0, lds);
}

template <class T, int kBM, int kBN, int kWM, int kWN> int launch_mx_input_as(MxInputArgs m, hipStream_t stream) {
    const int64_t blocks = piece_ids(m.rows.rows, kBM, m.rows.offsets != nullptr, m.rows.experts, true);
    constexpr int kThreads = 64 * (kBM / kWM) * (kBN / kWN);
    if (blocks >= int64_t{1} << 31) return fail("linear: too many tiles for one launch");
    in_launches(blocks, kThreads, [&](uint32_t first, uint32_t count) {
        mx_input_kernel<T, kBM, kBN, kWM, kWN>
            <<<whole_xcds(count), kThreads, 0, stream>>>(m, first, static_cast<uint32_t>(blocks));
    });
    return check_launch("linear of 4-bit weights, gradient");
}

}  // namespace

template <class T> int launch_mx_input(const MxInputArgs& m, hipStream_t stream) {
    const MxInputTile tile = mx_input_tile(m.rows.columns);
    if (tile.inputs == 64) return launch_mx_input_as<T, 128, 64, 32, 64>(m, stream);
    if (tile.inputs == 128) return launch_mx_input_as<T, 128, 128, 64, 64>(m, stream);
    return launch_mx_input_as<T, 128, 256, 64, 128>(m, stream);
}

}  // namespace odie
