// Products with a microscaled 4-bit weight, instantiated by mx_f16.hip, mx_bf16.hip and mx_f32.hip; the tiles' sums,
// their epilogue and the way of rows to LDS are linear.h's.
//
//   y[m][n] = act(sum_k x[m][k] w[n][k] + bias[n]) + residual[m][n],  w[n][k] = code(n, k) 2^(s(n, k / 32) - 127)
//
// Rows of 4 bits too: v_mfma_scale_f32_32x32x64_f8f6f4 takes both operands' codes and their scales as they are stored;
// products are exact.  Rows of T: the weight stays in 4 bits up to the registers, where it becomes T for
// v_mfma_f32_32x32x16 (fp32: 32x32x2), each value once for all 32-row tiles of a wave.
//
// Which k a lane holds at a step is free as long as both operands agree.  Here a lane of half h = lane / 32 takes whole
// blocks: its 16 bytes of codes belong to one scale, and the scales of its next four blocks are the bytes
// of one word.
#pragma once
#include "linear_epilogue.h"
#include "mx.h"

namespace odie {

struct MxRowsArgs {
    RowsArgs rows;               // a: rows of T, or their codes; b: the weight's codes
    const uint8_t* a_scales;     // null: rows of T
    const uint8_t* b_scales;
    int64_t code_pitch, scale_pitch;   // bytes a row of codes and of scales
};

template <class T> int launch_mx(const MxRowsArgs& a, hipStream_t stream);

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kMxSlab = 256;          // values of k in a 128-byte row of codes: 8 blocks
constexpr int kMxSlabScales = 8;

__device__ inline i32x8 mx_operand(const vec16& v) {
    return i32x8{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]),
                 0, 0, 0, 0};
}

// acc[n][m] += the 64 values of k of two blocks, one a lane half; kByte of the scale words is theirs.  4: 4-bit
// operands.
template <int kByte>
__device__ inline accum16 multiply_mx(const vec16& b, const vec16& a, uint32_t sb, uint32_t sa, accum16 c) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(b), mx_operand(a), c, 4, 4, kByte,
                                                           static_cast<int>(sb), kByte, static_cast<int>(sa));
}
// The same for 16 x 16 tiles and 128 values, a block a lane quarter.
__device__ inline accum4 multiply16_mx(const vec16& b, const vec16& a, uint32_t sb, uint32_t sa, accum4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(b), mx_operand(a), c, 4, 4, 0,
                                                            static_cast<int>(sb), 0, static_cast<int>(sa));
}

// Queues 4 bytes a lane from buffer + offset to LDS address `to` + 4 * lane, as queue16 does 16.
__device__ inline void queue4(uint32_t to, uint32_t offset, const vec16& buffer) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(offset),
                 "s"(buffer)
                 : "memory", "m0");
}

// An operand's scales on their way to LDS, two words a row and slab: kRows rows of 8 bytes.
template <int kRows, int kThreads> struct Scales {
    static constexpr int kBytes = kRows * kMxSlabScales;
    static constexpr int kLoads = kBytes / 256, kWaves = kThreads / 64;    // loads of 64 words, over the waves
    static constexpr int kOwn = (kLoads + kWaves - 1) / kWaves;
    uint32_t offset[kOwn];
    const uint8_t* base;     // uniform over the workgroup
    int left;                // words from this lane's on to its row's end

    static __device__ int wave() { return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64)); }

    __device__ void begin(const uint8_t* data, int64_t pitch, int64_t first, int64_t limit) {
        const int lane = static_cast<int>(threadIdx.x % 64);
        const int last = limit - first < kRows ? static_cast<int>(limit - first) - 1 : kRows - 1;
        base = data + first * pitch;
        left = static_cast<int>(pitch / 4) - lane % 2;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int r = ((wave() + i * kWaves) * 64 + lane) / 2;
            offset[i] = static_cast<uint32_t>(r < last ? r : last) * static_cast<uint32_t>(pitch) + lane % 2 * 4;
        }
    }
    __device__ void skip(int slabs) {
        base += slabs * kMxSlabScales;
        left -= 2 * slabs;
    }
    __device__ void load(char* lds) {
        const uint64_t address = reinterpret_cast<uint64_t>(base);
        vec16 buffer{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(address))),
                     static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(address >> 32))),
                     kBufferLimit, kBufferWord3};
        asm volatile("s_nop 4" : "+s"(buffer));   // wait states between its writing and the loads
        const uint32_t to =
            __builtin_amdgcn_readfirstlane(static_cast<int>(reinterpret_cast<uintptr_t>((lds_void)(lds))));
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (kLoads % kWaves == 0 || wave() + i * kWaves < kLoads)
                queue4(to + (wave() + i * kWaves) * 256, left > 0 ? offset[i] : kNowhere, buffer);
        base += kMxSlabScales;
        left -= 2;
    }
    static __device__ uint32_t byte(const char* lds, int row, int block) {
        return *reinterpret_cast<const uint8_t*>(lds + row * kMxSlabScales + block);
    }
};

// Chunk c (16 bytes) of row r of an image of 128-byte rows.
template <class I> __device__ inline vec16 chunk_at(const char* lds, int r, int c) {
    return *reinterpret_cast<const vec16*>(lds + r * kSlabBytes + ((c ^ I::turn(r)) << 4));
}

// The buffer descriptor of what lies from a uniform address on.
__device__ inline vec16 buffer_of(const uint8_t* base) {
    const uint64_t address = reinterpret_cast<uint64_t>(base);
    vec16 buffer{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(address))),
                 static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(address >> 32))),
                 kBufferLimit, kBufferWord3};
    asm volatile("s_nop 4" : "+s"(buffer));   // wait states between its writing and the loads
    return buffer;
}
__device__ inline uint32_t lds_address(const char* lds, int more) {
    return __builtin_amdgcn_readfirstlane(static_cast<int>(reinterpret_cast<uintptr_t>((lds_void)(lds))) + more);
}

// Both operands' scales on their way to LDS, 16 bytes a row: those of two slabs, a group.  Four lanes take a row, so
// that a load touches 16 lines (two lanes a row and slab: 32; all loads of a 256 x 256 tile alone then took a third
// longer).
template <int kBM, int kBN, int kThreads> struct ScaleRows {
    static constexpr int kRowBytes = 16, kBytes = (kBM + kBN) * kRowBytes, kWaves = kThreads / 64;
    static constexpr int kLoads = kBytes / 256 / kWaves;       // a wave's loads of 16 rows
    static_assert(kLoads * kWaves * 256 == kBytes && kBM % 16 == 0, "whole loads a wave");
    uint32_t offset[kLoads];
    const uint8_t *a, *b;    // uniform over the workgroup
    int left;                // words from this lane's on to its row's end

    static __device__ int part(int i) {
        return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64)) + i * kWaves;
    }

    // Rows past the last read the last.
    __device__ void begin(const uint8_t* rows, const uint8_t* columns, int64_t pitch, int64_t rows_left,
                          int64_t columns_left) {
        a = rows, b = columns;
        const int lane = static_cast<int>(threadIdx.x % 64);
        left = static_cast<int>(pitch / 4) - lane % 4;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = part(i) * 16 + lane / 4, r = at < kBM ? at : at - kBM;
            const int64_t limit = (at < kBM ? rows_left : columns_left) - 1;
            offset[i] = static_cast<uint32_t>(r < limit ? r : limit) * static_cast<uint32_t>(pitch) + lane % 4 * 4;
        }
    }
    __device__ void skip(int groups) {
        a += groups * kRowBytes, b += groups * kRowBytes;
        left -= groups * 4;
    }
    // Queues the next group's into lds.
    __device__ void load(char* lds) {
        const vec16 buffer_a = buffer_of(a), buffer_b = buffer_of(b);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t to = lds_address(lds, part(i) * 256), from = left > 0 ? offset[i] : kNowhere;
            if (part(i) * 16 < kBM) queue4(to, from, buffer_a);
            else queue4(to, from, buffer_b);
        }
        a += kRowBytes, b += kRowBytes;
        left -= 4;
    }
    // The scales of the four blocks that a lane half takes of slab `slab % 2` of the group, a byte each.
    static __device__ uint32_t word(const char* lds, int r, int slab, int half) {
        return *reinterpret_cast<const uint32_t*>(lds + r * kRowBytes + slab % 2 * kMxSlabScales + half * 4);
    }
};

// A tile of a product of codes with codes.  A slab is eight blocks of k, 128 bytes of codes: a lane of half h takes
// blocks 4 h .. 4 h + 3, one at each of four steps.
//
// 16384 x 4096 x 4096, bf16 out: 162 to 185 us, 3.0 to 3.4 PFLOP/s, with bias and gelu 197 to 230; 4096 more of k take
// 124 to 158 us (the clock falls by a tenth and more under this load).  Parts of it timed alone: the products from
// registers 85 us, with their LDS reads 98 to 120, the loads 95.  Loads of the next slab take most of a slab's
// products' time, and neither covers the other wholly.  Slower, with the epilogue's arithmetic: 128 x 128 tiles 234 to
// 280 us (twice the loads); 256 x 128, two workgroups a CU, slabs of half the depth in three buffers 246 to 285 (half
// lines), or one buffer each 229 to 256; fragments read a step ahead, eight waves 259 to 275, four waves of 128 x 128
// 239 to 254.
template <int kBM, int kBN, int kWM, int kWN, bool kShared> struct MxTile : Sums<kBM, kBN, kWM, kWN> {
    using Base = Sums<kBM, kBN, kWM, kWN>;
    using Base::acc;
    using Base::kMs;
    using Base::kNs;
    using Base::kThreads;
    using A = Direct<uint8_t, true, kBM, kThreads>;
    using B = Direct<uint8_t, true, kBN, kThreads>;
    using S = ScaleRows<kBM, kBN, kThreads>;
    static constexpr int kBuffer = A::kBytes + B::kBytes;
    static constexpr int kBytes = 2 * (kBuffer + S::kBytes);
    static constexpr int kLds = kBytes > kThreads / 64 * Base::kRegion ? kBytes : kThreads / 64 * Base::kRegion;

    template <int kStep> __device__ void add_step(const char* here, const uint32_t (&sa)[kMs],
                                                  const uint32_t (&sb)[kNs]) {
        const int lane = static_cast<int>(threadIdx.x % 64), chunk = 4 * (lane / 32) + kStep;
        vec16 fa[kMs], fb[kNs];
#pragma unroll
        for (int i = 0; i < kMs; ++i) fa[i] = chunk_at<A>(here, Base::wave_row() + 32 * i + lane % 32, chunk);
#pragma unroll
        for (int j = 0; j < kNs; ++j)
            fb[j] = chunk_at<B>(here + A::kBytes, Base::wave_column() + 32 * j + lane % 32, chunk);
#pragma unroll
        for (int i = 0; i < kMs; ++i)
#pragma unroll
            for (int j = 0; j < kNs; ++j) acc[i][j] = multiply_mx<kStep>(fb[j], fa[i], sb[j], sa[i], acc[i][j]);
    }

    __device__ void add_slab(const char* here, const char* scales, int slab) {
        const int lane = static_cast<int>(threadIdx.x % 64);
        uint32_t sa[kMs], sb[kNs];
#pragma unroll
        for (int i = 0; i < kMs; ++i) sa[i] = S::word(scales, Base::wave_row() + 32 * i + lane % 32, slab, lane / 32);
#pragma unroll
        for (int j = 0; j < kNs; ++j)
            sb[j] = S::word(scales, kBM + Base::wave_column() + 32 * j + lane % 32, slab, lane / 32);
        add_step<0>(here, sa, sb);
        add_step<1>(here, sa, sb);
        add_step<2>(here, sa, sb);
        add_step<3>(here, sa, sb);
    }

    // Sums `bytes` bytes of codes a row, in `slabs` slabs: those past the bytes add nothing, but wait as the others do.
    // The operands have begun.
    __device__ void sum(A& a, B& b, S& s, int bytes, int slabs, char* lds) {
        Base::clear();
        char* const scales = lds + 2 * kBuffer;
        auto load = [&](int slab) {
            const int left = bytes - slab * kSlabBytes;
            if (left <= 0) return;
            char* const to = lds + slab % 2 * kBuffer;
            a.load(left, to);
            b.load(left, to + A::kBytes);
            if (slab % 2 == 0) s.load(scales + slab / 2 % 2 * S::kBytes);
        };
        load(0);
        for (int i = 0; i < slabs; ++i) {
            arrived<0>();   // this slab; and no wave reads the other buffer any more
            load(i + 1);
            if (!kShared || i * kSlabBytes < bytes) add_slab(lds + i % 2 * kBuffer, scales + i / 2 % 2 * S::kBytes, i);
        }
        __syncthreads();
    }
};

// The depth of a product over kSplit groups of a tile's threads (threadIdx.y), whole slabs of codes each: a tile of few
// rows is a long chain of slabs that wait for their loads, and one of four waves leaves a CU idle at each (shares_of).
struct Share {
    int64_t first, count;    // slabs of codes: the group's first, and each group's number of them
};
template <int kSplit> __device__ inline Share share_of(int64_t slabs) {
    const int64_t count = (slabs + kSplit - 1) / kSplit;
    return Share{count * __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.y)), count};
}

// Adds the groups' sums up in the first one's, in their order.  `lds` holds them behind its epilogue's.
template <int kSplit, class Work> __device__ inline void join_groups(Work& work, char* lds) {
    constexpr int kValues = Work::kMs * Work::kNs * 16, kWaves = Work::kThreads / 64;
    float* const own = reinterpret_cast<float*>(lds + kWaves * Work::kRegion);
    float* const held = own + Work::wave() * kValues * 64 + threadIdx.x % 64;
    auto& acc = work.acc;
    if (threadIdx.y > 0)
#pragma unroll
        for (int v = 0; v < kValues; ++v)
            held[((threadIdx.y - 1) * kWaves * kValues + v) * 64] = acc[v / 16 / Work::kNs][v / 16 % Work::kNs][v % 16];
    __syncthreads();
    if (threadIdx.y > 0) return;
    for (int g = 0; g < kSplit - 1; ++g)
#pragma unroll
        for (int v = 0; v < kValues; ++v)
            acc[v / 16 / Work::kNs][v / 16 % Work::kNs][v % 16] += held[(g * kWaves * kValues + v) * 64];
}
template <int kSplit, class Work> constexpr int shared_bytes() {
    constexpr int kJoin = Work::kThreads / 64 * (Work::kRegion + (kSplit - 1) * Work::kMs * Work::kNs * 16 * 256);
    return kSplit == 1 ? Work::kLds : (kSplit * Work::kBytes > kJoin ? kSplit * Work::kBytes : kJoin);
}

template <class T, int kBM, int kBN, int kWM, int kWN, int kSplit>
__global__ __launch_bounds__(kSplit * 64 * (kBM / kWM) * (kBN / kWN)) void mx_rows4_kernel(
    MxRowsArgs m, uint32_t first, uint32_t blocks) {
    using Work = MxTile<kBM, kBN, kWM, kWN, (kSplit > 1)>;
    __shared__ __attribute__((aligned(16))) char lds[shared_bytes<kSplit, Work>()];
    const RowsArgs& a = m.rows;
    const uint32_t id = first + xcd_major(blockIdx.x, gridDim.x);
    if (id >= blocks) return;
    const TileAt t = tile_at(id, static_cast<uint32_t>(a.tiles), (a.columns + kBN - 1) / kBN);
    const Piece p = find_piece(a.offsets, a.experts, a.experts + 1, a.rows, kBM, t.row);
    if (p.begin >= p.end) return;
    const int column0 = static_cast<int>(t.column) * kBN;
    if (p.group >= a.experts) {
        if (threadIdx.y == 0) rows_of_none<T, kBM, kBN, Work::kThreads>(a, p, column0);
        return;
    }
    const int64_t matrix = static_cast<int64_t>(p.group) * a.columns;
    const int64_t slabs = (m.code_pitch + kSlabBytes - 1) / kSlabBytes;
    Share share{0, slabs};
    if constexpr (kSplit > 1) {
        share = share_of<kSplit>((slabs + 1) / 2);      // in pairs, which share their scales' loads
        share.first *= 2, share.count *= 2;
    }
    const int64_t skip = share.first * kSlabBytes;
    char* const own = lds + (kSplit > 1 ? share.first / share.count * Work::kBytes : 0);
    typename Work::A opa;
    typename Work::B opb;
    typename Work::S scales;
    opa.begin(static_cast<const uint8_t*>(a.a) + skip, m.code_pitch, p.begin, p.end, m.code_pitch);
    opb.begin(static_cast<const uint8_t*>(a.b) + matrix * m.code_pitch + skip, m.code_pitch, column0, a.columns,
              m.code_pitch);
    scales.begin(m.a_scales + p.begin * m.scale_pitch, m.b_scales + (matrix + column0) * m.scale_pitch, m.scale_pitch,
                 p.end - p.begin, a.columns - column0);
    scales.skip(static_cast<int>(share.first / 2));
    Work work;
    const int64_t bytes = m.code_pitch - skip;
    work.sum(opa, opb, scales, static_cast<int>(kSplit > 1 && bytes > share.count * kSlabBytes
                                                ? share.count * kSlabBytes : bytes),
             static_cast<int>(share.count), own);
    if constexpr (kSplit > 1) {
        join_groups<kSplit>(work, lds);
        if (threadIdx.y > 0) return;
    }
    finish_tile<T, kBM == 256>(work, a, p, column0, lds);
}

// A tile of a product of rows of T with codes.  A slab of the weight's codes lasts for kRatio slabs of the rows. 16384
// x 4096 x 4096 bf16 450 to 500 us, 1100 to 1220 TFLOP/s, with bias and gelu 490 to 530; 131072 rows over 64 experts,
// 256 -> 512 fp16 with silu and the sums kept 100 to 110 us, 340 MB at 3.1 to 3.4 TB/s.
template <class T, Way kWay, int kBM, int kBN, int kWM, int kWN, bool kShared>
struct MixedTile : Sums<kBM, kBN, kWM, kWN> {
    using Base = Sums<kBM, kBN, kWM, kWN>;
    using Base::acc;
    using Base::kMs;
    using Base::kNs;
    using Base::kThreads;
    using A = std::conditional_t<kWay == kDirect, Direct<T, true, kBM, kThreads>,
                                 std::conditional_t<kWay == kStaged, Staged<T, true, kBM, kThreads>,
                                                    Gathered<T, true, kBM, kThreads>>>;
    using B = Direct<uint8_t, true, kBN, kThreads>;
    using SB = Scales<kBN, kThreads>;
    static constexpr int kRatio = kMxSlab / kSlab<T>;
    static constexpr int kCodes = B::kBytes + SB::kBytes;
    static constexpr int kBytes = 2 * (A::kBytes + kCodes);
    static constexpr int kLds = kBytes > kThreads / 64 * Base::kRegion ? kBytes : kThreads / 64 * Base::kRegion;

    // Slab `part` of the kRatio of these codes.  A lane of half h takes values 32 (2 part + h) .. + 31 of the codes'
    // slab, a block (fp32: half a block, 32 part + 16 h .. + 15), eight (four) at a step.
    __device__ void add_slab(const char* rows, const char* codes, int part) {
        const int lane = static_cast<int>(threadIdx.x % 64), half = lane / 32;
        constexpr bool kWide = sizeof(T) == 4;
        vec16 held[kNs];
        float scale[kNs];
#pragma unroll
        for (int j = 0; j < kNs; ++j) {
            const int r = Base::wave_column() + 32 * j + lane % 32, block = kWide ? part : 2 * part + half;
            held[j] = chunk_at<B>(codes, r, block);
            scale[j] = mx_scale(SB::byte(codes + B::kBytes, r, block));
        }
#pragma unroll
        for (int step = 0; step < 4; ++step) {
            vec16 fa[kMs], fb[kNs];
#pragma unroll
            for (int i = 0; i < kMs; ++i)
                fa[i] = chunk_at<A>(rows, Base::wave_row() + 32 * i + lane % 32, 4 * half + step);
#pragma unroll
            for (int j = 0; j < kNs; ++j) {
                const uint32_t word = kWide ? (half ? held[j][2 + step / 2] : held[j][step / 2]) : held[j][step];
                fb[j] = mx_values<T>(word, scale[j], step % 2 == 1);
            }
#pragma unroll
            for (int i = 0; i < kMs; ++i)
#pragma unroll
                for (int j = 0; j < kNs; ++j) acc[i][j] = multiply(T{}, fb[j], fa[i], acc[i][j]);
        }
    }

    // Sums `depth` values of k; `bytes` bytes of codes a row.  kShared: in `slabs` slabs of the rows, of which those
    // past the depth add nothing, but wait as the others do.  The operands have begun.
    __device__ void sum(A& a, B& b, SB& sb, int64_t depth, int64_t bytes, int slabs, char* lds) {
        Base::clear();
        char* const codes = lds + 2 * A::kBytes;
        int64_t codes_left = bytes;
        int next = 0;                // buffer of the codes' next slab
        auto load_codes = [&] {
            if (codes_left <= 0) return;
            b.load(codes_left, codes + next * kCodes);
            sb.load(codes + next * kCodes + B::kBytes);
            codes_left -= kSlabBytes;
            next ^= 1;
        };
        load_codes();
        int now = 0, part = 0, at = 0;
        if constexpr (kWay == kDirect) {
            a.load(depth, lds);
            for (int64_t left = depth; kShared ? slabs-- > 0 : left > 0; left -= kSlab<T>) {
                arrived<0>();   // this slab; and no wave reads the other buffers any more
                if (left > kSlab<T>) a.load(left - kSlab<T>, lds + (now ^ 1) * A::kBytes);
                if (part == 0) load_codes();
                if (!kShared || left > 0) add_slab(lds + now * A::kBytes, codes + at * kCodes, part);
                now ^= 1;
                if (++part == kRatio) part = 0, at ^= 1;
            }
        } else {
            typename A::Held held;
            a.load(held);
            for (int64_t left = depth; left > 0; left -= kSlab<T>) {
                a.store(held, lds + now * A::kBytes, left);
                arrived<0>();   // the slab is there; and no wave reads the buffer of the slab before
                if (left > kSlab<T>) a.load(held);
                if (part == 0) load_codes();
                add_slab(lds + now * A::kBytes, codes + at * kCodes, part);
                now ^= 1;
                if (++part == kRatio) part = 0, at ^= 1;
            }
        }
        __syncthreads();
    }
};

template <class T, Way kWay, int kBM, int kBN, int kWM, int kWN, int kSplit>
__global__ __launch_bounds__(kSplit * 64 * (kBM / kWM) * (kBN / kWN)) void mx_mixed_kernel(
    MxRowsArgs m, uint32_t first, uint32_t blocks) {
    static_assert(kSplit == 1 || kWay == kDirect, "shares are of rows that go straight to LDS");
    using Work = MixedTile<T, kWay, kBM, kBN, kWM, kWN, (kSplit > 1)>;
    __shared__ __attribute__((aligned(16))) char lds[shared_bytes<kSplit, Work>()];
    const RowsArgs& a = m.rows;
    const uint32_t id = first + xcd_major(blockIdx.x, gridDim.x);
    if (id >= blocks) return;
    const TileAt t = tile_at(id, static_cast<uint32_t>(a.tiles), (a.columns + kBN - 1) / kBN);
    const Piece p = find_piece(a.offsets, a.experts, a.experts + 1, a.rows, kBM, t.row);
    if (p.begin >= p.end) return;
    const int column0 = static_cast<int>(t.column) * kBN;
    if (p.group >= a.experts) {
        if (threadIdx.y == 0) rows_of_none<T, kBM, kBN, Work::kThreads>(a, p, column0);
        return;
    }
    const int64_t matrix = static_cast<int64_t>(p.group) * a.columns;
    Share share{0, 0};
    if constexpr (kSplit > 1) share = share_of<kSplit>((m.code_pitch + kSlabBytes - 1) / kSlabBytes);
    const int64_t skip = share.first * kMxSlab, most = share.count * kMxSlab;     // values of k
    char* const own = lds + (kSplit > 1 ? share.first / share.count * Work::kBytes : 0);
    typename Work::A opa;
    typename Work::B opb;
    typename Work::SB sb;
    opa.begin(static_cast<const T*>(a.a) + skip, a.lda, p.begin, p.end, a.depth);
    opb.begin(static_cast<const uint8_t*>(a.b) + matrix * m.code_pitch + skip / 2, m.code_pitch, column0, a.columns,
              m.code_pitch);
    sb.begin(m.b_scales + matrix * m.scale_pitch, m.scale_pitch, column0, a.columns);
    int64_t depth = a.depth - skip, bytes = m.code_pitch - skip / 2;
    if constexpr (kSplit > 1) {
        sb.skip(static_cast<int>(share.first));
        depth = depth < most ? depth : most;
        bytes = bytes < most / 2 ? bytes : most / 2;
    }
    Work work;
    work.sum(opa, opb, sb, depth, bytes, static_cast<int>(share.count) * Work::kRatio, own);
    if constexpr (kSplit > 1) {
        join_groups<kSplit>(work, lds);
        if (threadIdx.y > 0) return;
    }
    finish_tile<T, kBM == 256>(work, a, p, column0, lds);
}

// Few rows a group, as few_rows_kernel: the weight's codes go straight into registers, once for every 16 kRowTiles
// rows. A step takes four blocks of k, one a lane quarter, and a wave one of kSplit shares of the blocks.  Bound by the
// latency of a chain of loads: one bf16 row through 2048 -> 2048 (2.2 MB) 4.3 us, 16 rows over 64 experts of 512 ->
// 1024 7.2 us.  Twice the steps in flight: 4.7 and 7.4.
template <class T, bool kRows4, int kRowTiles, int kSplit>
__global__ __launch_bounds__(64 * kFewWaves) void mx_few_rows_kernel(MxRowsArgs m) {
    constexpr int kColumns = 16 * kFewWaves / kSplit;   // of a workgroup
    constexpr int kAhead = kRows4 ? 4 : 2;              // steps in flight
    constexpr int kParts = kRows4 ? 1 : kMxBlock / kPerVec<T>;   // 16-byte parts of a block of a row
    __shared__ accum4 part[kFewWaves][kRowTiles][64];
    const RowsArgs& a = m.rows;
    const uint32_t across = (a.columns + kColumns - 1) / kColumns;
    const Piece p = find_piece(a.offsets, a.experts, a.experts + 1, a.rows, 16 * kRowTiles, blockIdx.x / across);
    if (p.begin >= p.end) return;
    const int column0 = static_cast<int>(blockIdx.x % across) * kColumns;
    const int lane = static_cast<int>(threadIdx.x % 64);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
    const bool owned = p.group < a.experts;        // else rows of no expert
    if (owned && column0 + wave / kSplit * 16 < a.columns) {
        const int own = lane % 16, quarter = lane / 16;
        int column = column0 + wave / kSplit * 16 + own;
        column = column < a.columns ? column : a.columns - 1;   // those past the last are not stored
        const int64_t at = static_cast<int64_t>(p.group) * a.columns + column;
        const uint8_t* w = static_cast<const uint8_t*>(a.b) + at * m.code_pitch;
        const uint8_t* ws = m.b_scales + at * m.scale_pitch;
        const T* x[kRowTiles];
        const uint8_t* xc[kRowTiles];
        const uint8_t* xs[kRowTiles];
#pragma unroll
        for (int t = 0; t < kRowTiles; ++t) {
            int64_t row = p.begin + 16 * t + own;
            row = row < p.end ? row : p.end - 1;
            x[t] = static_cast<const T*>(a.a) + row * a.lda;
            xc[t] = static_cast<const uint8_t*>(a.a) + row * m.code_pitch;
            xs[t] = m.a_scales + row * m.scale_pitch;
        }
        accum4 acc[kRowTiles] = {};
        const int total = static_cast<int>(m.code_pitch / kMxBytes), steps = (total + 3) / 4;
        const int share = (steps + kSplit - 1) / kSplit * 4;
        const int first = wave % kSplit * share, last = first + share < total ? first + share : total;
        for (int b0 = first; b0 < last; b0 += 4 * kAhead) {
            vec16 fw[kAhead], fx[kAhead][kRowTiles][kParts];
            uint32_t sw[kAhead], sx[kAhead][kRowTiles];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int block = b0 + 4 * u + quarter;
                const bool inside = block < last;
                fw[u] = inside ? *reinterpret_cast<const vec16*>(w + block * kMxBytes) : vec16{};
                sw[u] = inside ? ws[block] : 0u;
#pragma unroll
                for (int t = 0; t < kRowTiles; ++t) {
                    if constexpr (kRows4) {
                        fx[u][t][0] = inside ? *reinterpret_cast<const vec16*>(xc[t] + block * kMxBytes) : vec16{};
                        sx[u][t] = inside ? xs[t][block] : 0u;
                    } else {
#pragma unroll
                        for (int i = 0; i < kParts; ++i) {
                            const int k = block * kMxBlock + i * kPerVec<T>, count = inside ? a.depth - k : 0;
                            fx[u][t][i] = count > 0 ? load_end(x[t] + k, count, k) : vec16{};
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if constexpr (kRows4) {
#pragma unroll
                    for (int t = 0; t < kRowTiles; ++t)
                        acc[t] = multiply16_mx(fw[u], fx[u][t][0], sw[u], sx[u][t], acc[t]);
                } else {
                    const float scale = mx_scale(sw[u]);
#pragma unroll
                    for (int i = 0; i < kParts; ++i) {
                        const vec16 values =
                            mx_values<T>(fw[u][i * kPerVec<T> / 8], scale, sizeof(T) == 4 && i % 2 == 1);
#pragma unroll
                        for (int t = 0; t < kRowTiles; ++t) acc[t] = multiply16(T{}, values, fx[u][t][i], acc[t]);
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < kRowTiles; ++t) part[wave][t][lane] = acc[t];
    }
    __syncthreads();
    finish_few<T, kRowTiles, kSplit>(part, a, p, column0, owned);
}

template <int kBM, int kBN, int kWM, int kWN, int kSplit, class Launch> int in_tiles(MxRowsArgs m, Launch&& launch) {
    const int64_t across = (m.rows.columns + kBN - 1) / kBN;
    m.rows.tiles = piece_ids(m.rows.rows, kBM, m.rows.offsets != nullptr, m.rows.experts, true);
    const int64_t blocks = m.rows.tiles * across;
    if (blocks >= int64_t{1} << 31) return fail("linear: too many tiles for one launch");
    constexpr int kThreads = 64 * (kBM / kWM) * (kBN / kWN);
    in_launches(blocks, kSplit * kThreads, [&](uint32_t first, uint32_t count) {
        launch(m, whole_xcds(count), dim3(kThreads, kSplit), first, static_cast<uint32_t>(blocks));
    });
    return check_launch("linear of 4-bit weights");
}

template <class T, int kBM, int kBN, int kWM, int kWN, int kSplit = 1>
int launch_rows4(const MxRowsArgs& m, hipStream_t stream) {
    return in_tiles<kBM, kBN, kWM, kWN, kSplit>(m, [&](const MxRowsArgs& a, uint32_t grid, dim3 threads,
                                                       uint32_t first, uint32_t blocks) {
        mx_rows4_kernel<T, kBM, kBN, kWM, kWN, kSplit><<<grid, threads, 0, stream>>>(a, first, blocks);
    });
}

template <class T, Way kWay, int kBM, int kBN, int kWM, int kWN, int kSplit = 1>
int launch_mixed(const MxRowsArgs& m, hipStream_t stream) {
    return in_tiles<kBM, kBN, kWM, kWN, kSplit>(m, [&](const MxRowsArgs& a, uint32_t grid, dim3 threads,
                                                       uint32_t first, uint32_t blocks) {
        mx_mixed_kernel<T, kWay, kBM, kBN, kWM, kWN, kSplit><<<grid, threads, 0, stream>>>(a, first, blocks);
    });
}

template <class T, bool kRows4, int kRowTiles, int kSplit>
int launch_mx_few_as(const MxRowsArgs& m, hipStream_t stream) {
    const RowsArgs& a = m.rows;
    const int64_t across = (a.columns + 16 * kFewWaves / kSplit - 1) / (16 * kFewWaves / kSplit);
    const int64_t blocks = piece_ids(a.rows, 16 * kRowTiles, a.offsets != nullptr, a.experts, true) * across;
    if (blocks > most_blocks(64 * kFewWaves)) return fail("linear: too many tiles for one launch");
    mx_few_rows_kernel<T, kRows4, kRowTiles, kSplit><<<static_cast<uint32_t>(blocks), 64 * kFewWaves, 0, stream>>>(m);
    return check_launch("linear of 4-bit weights");
}

// The depth over all eight waves where a share is still long or there are too few workgroups otherwise, else over two.
// us with eight and with two: 2048 -> 2048 bf16, one row 4.3 and 8.3, 16 rows 5.5 and 13.6; 512 -> 4096 3.4 and 4.0;
// 512 -> 16384 5.3 and 4.2; 16 rows over 64 experts of 512 -> 1024 10.8 and 7.2; 4096 -> 16384 16.0 and 17.7.
template <class T, bool kRows4, int kRowTiles> int launch_mx_few(const MxRowsArgs& m, hipStream_t stream) {
    const int64_t steps = m.code_pitch / (4 * kMxBytes);
    const int64_t busy = m.rows.rows < m.rows.experts ? m.rows.rows : m.rows.experts;
    if (steps >= 16 || busy * m.rows.columns < 64 * kCus) return launch_mx_few_as<T, kRows4, kRowTiles, 8>(m, stream);
    return launch_mx_few_as<T, kRows4, kRowTiles, 2>(m, stream);
}

// Shares that the depth of a tile of 64 x 64 is cut into, where there are few tiles.  us of bf16 rows as one, two and
// four: 100 x 4096 x 4096 27.7, 20.0 and 17.0, 300 35.3, 29.0 and 33.8, 512 36.9, 32.9 and 34.9; 256 x 2048 x 2048
// 15.8, 12.2 and 11.1, 1000 20.3, 18.6 and 21.6; 100 x 1024 x 1024 9.5, 8.1 and 7.9; 100 x 512 x 512 6.5, 6.2 and 7.0;
// 1000 rows over 64 experts of 512 -> 1024 14.0, 17.5 and 31.1.  Rows of 4 bits, whose slabs take less time: 100 x 4096
// x 4096 11.4, 9.5 and 9.3, 300 15.1, 14.1 and 19.3; 100 x 2048 x 2048 7.6, 6.9 and 7.4, 1000 10.0, 10.2 and 14.5; 100
// x 1024 x 1024 5.7, 5.8 and 6.6.
inline int shares_of(const MxRowsArgs& m) {
    const RowsArgs& a = m.rows;
    const int64_t tiles = piece_ids(a.rows, 64, a.offsets != nullptr, a.experts, true) * ((a.columns + 63) / 64);
    const int64_t slabs = (m.code_pitch + kSlabBytes - 1) / kSlabBytes;
    if (m.a_scales) return slabs >= (tiles <= kCus ? 8 : 16) && tiles <= 2 * kCus ? 2 : 1;
    if (tiles > 2 * kCus || slabs < 2) return 1;
    return tiles <= kCus && slabs >= 4 ? 4 : 2;
}

// Tiles as linear's, by the work there is.  us of bf16 products as 256 x 256, 128 x 128 and 64 x 64: rows of bf16,
// 65536 x 1024 x 4096 522, 624 and 849, 16384 x 1024 x 1024 37, 45 and 57, 4096 x 2048 x 2048 (128 tiles of the
// largest) -, 42 and 58, 131072 rows over 64 experts of 256 -> 512 88, 90 and 110; 4-bit rows 247, 308 and 382, 17, 22
// and 28, -, 19 and 22, 61, 63 and 72.
template <class T, Way kWay> int launch_mixed_of(const MxRowsArgs& m, hipStream_t stream) {
    const RowsArgs& a = m.rows;
    const int64_t each = a.rows / a.experts;
    const int64_t large = (a.rows + 255) / 256 * ((a.columns + 255) / 256);
    const int64_t wide = (a.rows + 127) / 128 * ((a.columns + 127) / 128);
    if constexpr (kWay == kDirect)
        if (a.columns > 128 && even(large) && each >= 1024) return launch_mixed<T, kWay, 256, 256, 64, 128>(m, stream);
    if constexpr (kWay != kGathered)
        if (a.columns > 64 && wide >= kCus && each >= 128) return launch_mixed<T, kWay, 128, 128, 64, 64>(m, stream);
    if constexpr (kWay == kDirect)
        switch (shares_of(m)) {
            case 4: return launch_mixed<T, kWay, 64, 64, 32, 32, 4>(m, stream);
            case 2: return launch_mixed<T, kWay, 64, 64, 32, 32, 2>(m, stream);
        }
    return launch_mixed<T, kWay, 64, 64, 32, 32>(m, stream);
}

template <class T, bool kRows4> int launch_mx_by_rows(const MxRowsArgs& m, hipStream_t stream) {
    const RowsArgs& a = m.rows;
    // Few rows: up to 64 for one matrix (4-bit rows 32), up to 256 (128) in all over several.  Each 16 columns read all
    // the rows, so that rows times columns tell how long that takes.  us of few rows and of tiles, bf16: 4096 -> 4096,
    // 16 rows 8.2 and 16.0, 32 rows 11.8 and 16.1, 48 rows 17.5 and 16.4, 64 rows 20.1 and 16.4; 1024 -> 4096, 64 rows
    // 8.1 and 8.1; 2048 -> 2048, 48 rows 10.3 and 10.6, 64 rows 11.6 and 10.8; 2048 -> 16384, one row 9.0 and 11.1, 8
    // rows 11.9 and 11.2, 16 rows 13.8 and 11.4, 64 rows 44.8 and 12.1; 4-bit rows, 4096 -> 4096, 32 rows 8.1 and 9.2,
    // 4096 -> 16384, 16 rows 17.9 and 11.1.  Over 64 experts of 512 -> 1024, 64 rows 8.0 and 12.8, 256 rows 13.0 and
    // 13.4, 512 rows 15.8 and 13.6; 4-bit rows, 64 rows 7.2 and 8.2, 256 rows 8.7 and 8.5, 512 rows 11.5 and 8.6.
    if (a.experts > 1) {
        if (a.rows <= (kRows4 ? 128 : 256)) return launch_mx_few<T, kRows4, 1>(m, stream);
    } else if (a.rows * a.columns < 1 << 18 && (a.rows <= 48 || a.depth < 2048)) {
        if (a.rows <= 16) return launch_mx_few<T, kRows4, 1>(m, stream);
        if (a.rows <= 32) return launch_mx_few<T, kRows4, 2>(m, stream);
        if constexpr (!kRows4)
            if (a.rows <= 64) return launch_mx_few<T, kRows4, 4>(m, stream);
    }
    if constexpr (kRows4) {
        const int64_t large = (a.rows + 255) / 256 * ((a.columns + 255) / 256);
        const int64_t wide = (a.rows + 127) / 128 * ((a.columns + 127) / 128);
        if (a.columns > 128 && even(large) && a.rows / a.experts >= 1024)
            return launch_rows4<T, 256, 256, 64, 128>(m, stream);
        if (a.columns > 64 && wide >= kCus && a.rows / a.experts >= 128)
            return launch_rows4<T, 128, 128, 64, 64>(m, stream);
        if (shares_of(m) == 2) return launch_rows4<T, 64, 64, 32, 32, 2>(m, stream);
        return launch_rows4<T, 64, 64, 32, 32>(m, stream);
    } else {
        switch (way_of<T>(a.a, a.lda, a.depth)) {
            case kDirect: return launch_mixed_of<T, kDirect>(m, stream);
            case kStaged: return launch_mixed_of<T, kStaged>(m, stream);
            default: return launch_mixed_of<T, kGathered>(m, stream);
        }
    }
}

}  // namespace

template <class T> int launch_mx(const MxRowsArgs& m, hipStream_t stream) {
    return m.a_scales ? launch_mx_by_rows<T, true>(m, stream) : launch_mx_by_rows<T, false>(m, stream);
}

}  // namespace odie

#define ODIE_MX_FOR(T)                                                        \
    namespace odie {                                                          \
    template int launch_mx<T>(const MxRowsArgs&, hipStream_t);                \
    }
