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
// values).  Per slab both operands pass through LDS in their memory orientation, with one barrier a slab and later
// slabs under way while one is multiplied: straight to LDS one in a second buffer, in 64 x 64 tiles three in four
// buffers; through registers two in registers (64 x 64 tiles three, element by element one) and two buffers.
// A 16-bit operand stored one row per k is turned by ds_read_b64_tr_b16 as it is read.  Products are
// v_mfma_f32_32x32x16 (16-bit) or v_mfma_f32_32x32x2 (fp32), accumulated in fp32.
//
// The epilogue passes each wave's accumulators through its own part of the LDS, so that bias,
// activation, residual and the stores run on rows of 8 consecutive columns a lane.
#pragma once
#include <type_traits>

#include "elements.h"

namespace odie {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float accum16 __attribute__((ext_vector_type(16)));
typedef int16_t i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4* lds_i16x4;
typedef __attribute__((address_space(3))) void* lds_void;

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

// The same for 16 x 16 tiles: lane l holds row l % 16, k quarter l / 16.
typedef float accum4 __attribute__((ext_vector_type(4)));
__device__ inline accum4 multiply16(_Float16, const vec16& b, const vec16& a, accum4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
}
__device__ inline accum4 multiply16(__bf16, const vec16& b, const vec16& a, accum4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
}
__device__ inline accum4 multiply16(float, const vec16& b, const vec16& a, accum4 c) {
    float fb[4], fa[4];
    __builtin_memcpy(fb, &b, 16);
    __builtin_memcpy(fa, &a, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[i], fa[i], c, 0, 0, 0);
    return c;
}

// One operand of a tile: kRows of its own index times one slab of k, kThreads threads.
// LDS image, k consecutive: kRows rows of 128 bytes; the 16-byte chunk c of row r lies at slot
// c ^ (r / 2 % 8), so that 16 consecutive rows of one chunk fall on all 64 banks.
// LDS image, one row per k: rows of kRows elements; chunk c of row k lies at slot c ^ turn(k), so
// that the rows one transposing read touches at once (k .. k + 3, 32 columns) fall on all 64 banks.
// Thread t fills the slots t, t + kThreads, ... of the image, in the order of their addresses.
template <class T, bool kByRow, int kRows, int kThreads> struct Image {
    static constexpr int kBytes = kRows * kSlabBytes;
    static constexpr int kChunks = kRows * 8 / kThreads;       // 16-byte chunks a thread moves per slab
    static constexpr int kVec = kPerVec<T>;
    static constexpr int kPerRow = kByRow ? 8 : kRows / kVec;   // chunks a row of the image
    static constexpr int kStep = kThreads / kPerRow;            // rows between a thread's chunks
    static_assert(kChunks * kThreads == kRows * 8 && kThreads % kPerRow == 0, "whole chunks a thread");

    // XOR on the chunk number in row r of the image.
    static __device__ int turn(int r) {
        if constexpr (kByRow) return r >> 1 & 7;
        if constexpr (sizeof(T) == 4) return (r >> 2 & 1) << 3;
        return kPerRow >= 16 ? (r & 3) << 2 : (r >> 1 & 1) << 2;
    }
    static_assert(kStep % 16 == 0 || (!kByRow && kStep % 8 == 0), "a thread's chunks turn alike");

    static __device__ int row() { return static_cast<int>(threadIdx.x) / kPerRow; }    // of the first chunk
    static __device__ int chunk() { return static_cast<int>(threadIdx.x) % kPerRow ^ turn(row()); }

    // The 16 bytes of k that lane l holds of own index base + l % 32: k chunk 2 * step + l / 32.
    static __device__ vec16 fragment(const char* lds, int base, int step, int lane) {
        if constexpr (kByRow) {
            const int r = base + lane % 32;
            return *reinterpret_cast<const vec16*>(lds + r * kSlabBytes + ((2 * step + lane / 32 ^ turn(r)) << 4));
        } else if constexpr (sizeof(T) == 4) {
            const int column = base + lane % 32, k = 8 * step + 4 * (lane / 32);
            vec16 v;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = *reinterpret_cast<const uint32_t*>(lds + (k + i) * (kPerRow * 16) +
                                                          ((column >> 2 ^ turn(k + i)) << 4) + (column & 3) * 4);
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

constexpr uint32_t kNowhere = 0x80000000u;          // past every buffer: such a lane's bytes arrive as 0
constexpr uint32_t kBufferLimit = 0x7fffffff;
constexpr uint32_t kBufferWord3 = 0x00027000;

// Queues 16 bytes a lane from buffer + offset to LDS address `to` + 16 * lane (`to` and buffer uniform over the
// wave).  Written out, with no register result, because of the builtin's transposing LDS reads the compiler waits for
// every such load in flight, the next slab's too.  So it knows of none of them: arrived() has to come before the
// bytes are read.
__device__ inline void queue16(uint32_t to, uint32_t offset, const vec16& buffer) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(buffer)
                 : "memory", "m0");
}

// Waits until this wave's queued loads but the last kPending have arrived and its LDS reads are done, then for the
// other waves of the workgroup.
template <int kPending> __device__ inline void arrived() {
    static_assert(kPending < 64, "the wait's count has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kPending) : "memory");
}

// Global to LDS without registers, 16 bytes a lane, for rows that start on 16 bytes and hold whole
// chunks.  Offsets of a tile's chunks from its first row stay below 2^31 (checked on the host).
template <class T, bool kByRow, int kRows, int kThreads> struct Direct : Image<T, kByRow, kRows, kThreads> {
    using I = Image<T, kByRow, kRows, kThreads>;
    uint32_t offset[I::kChunks];
    const char* base;    // uniform over the workgroup
    int64_t slab;        // bytes from slab to slab
    int lead;            // k of the first chunk, relative to the slab

    // Own indices first .. of `limit` in all; k consecutive: rows past the last read the last (their products are
    // not stored), else columns past the last read 0.
    __device__ void begin(const T* data, int64_t stride, int64_t first, int64_t limit, int64_t) {
        const uint32_t pitch = static_cast<uint32_t>(stride * sizeof(T));
        if constexpr (kByRow) {
            base = reinterpret_cast<const char*>(data + first * stride);
            slab = kSlabBytes;
            lead = I::chunk() * I::kVec;
            const int last = limit - first < kRows ? static_cast<int>(limit - first) - 1 : kRows - 1;
#pragma unroll
            for (int i = 0; i < I::kChunks; ++i) {
                const int r = I::row() + i * I::kStep;
                offset[i] = static_cast<uint32_t>(r < last ? r : last) * pitch + I::chunk() * 16;
            }
        } else {
            base = reinterpret_cast<const char*>(data + first);
            slab = kSlab<T> * stride * static_cast<int64_t>(sizeof(T));
            lead = I::row();
            const bool inside = first + I::chunk() * I::kVec < limit;
#pragma unroll
            for (int i = 0; i < I::kChunks; ++i)
                offset[i] = inside ? static_cast<uint32_t>(lead + i * I::kStep) * pitch + I::chunk() * 16 : kNowhere;
        }
    }

    // Queues the next slab into lds; `left` values of k exist, the rest arrive as 0.
    __device__ void load(int64_t left, char* lds) {
        const uint64_t address = reinterpret_cast<uint64_t>(base);
        vec16 buffer{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(address))),
                           static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(address >> 32))),
                           kBufferLimit, kBufferWord3};
        asm volatile("s_nop 4" : "+s"(buffer));   // wait states between its writing and the loads
        const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void)(lds))) +
                            __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64) * 1024;
        if (left >= kSlab<T>) {
#pragma unroll
            for (int i = 0; i < I::kChunks; ++i) queue16(to + i * kThreads * 16, offset[i], buffer);
        } else {
#pragma unroll
            for (int i = 0; i < I::kChunks; ++i) {
                const bool inside = (kByRow ? lead : lead + i * I::kStep) < left;
                queue16(to + i * kThreads * 16, inside ? offset[i] : kNowhere, buffer);
            }
        }
        base += slab;
    }
};

// Through registers, for rows of any alignment.  Every load is issued without a condition, from an address moved
// back into the tensor where it would leave it (a branch around loads makes the compiler wait for those in
// flight); what was moved is put right on the way to LDS.  Needs 16 bytes of k (k consecutive) or of columns (one row
// per k) at least, and one k.
template <class T, bool kByRow, int kRows, int kThreads> struct Staged : Image<T, kByRow, kRows, kThreads> {
    using I = Image<T, kByRow, kRows, kThreads>;
    struct Held {
        vec16 chunk[I::kChunks];
    };
    const T* at[kByRow ? I::kChunks : 1];   // k consecutive: the rows' begins; else this thread's column in row 0
    int64_t stride, next;                   // next: k of the slab to load
    int64_t depth;
    int lead;            // k of the first chunk, relative to the slab
    int back;            // one row per k: columns that the chunk was moved back by

    __device__ void begin(const T* data, int64_t pitch, int64_t first, int64_t limit, int64_t ks) {
        stride = pitch;
        depth = ks;
        next = 0;
        back = 0;
        if constexpr (kByRow) {
            lead = I::chunk() * I::kVec;
#pragma unroll
            for (int i = 0; i < I::kChunks; ++i) {
                const int64_t r = first + I::row() + i * I::kStep;
                at[i] = data + (r < limit ? r : limit - 1) * stride;
            }
        } else {
            lead = I::row();
            const int64_t column = first + I::chunk() * I::kVec, last = limit - I::kVec;
            at[0] = data + (column < last ? column : last);
            if (column > last) back = column - last < I::kVec ? static_cast<int>(column - last) : 0;
        }
    }

    __device__ void load(Held& held) {
        if constexpr (kByRow) {
            const int64_t k = next + lead < depth - I::kVec ? next + lead : depth - I::kVec;
#pragma unroll
            for (int i = 0; i < I::kChunks; ++i) held.chunk[i] = load16(at[i] + k);
        } else {
#pragma unroll
            for (int i = 0; i < I::kChunks; ++i) {
                const int64_t k = next + lead + i * I::kStep;
                held.chunk[i] = load16(at[0] + (k < depth ? k : depth - 1) * stride);
            }
        }
        next += kSlab<T>;
    }

    // `left` values of k of this slab exist; the rest become 0.
    __device__ void store(const Held& held, char* lds, int64_t left) const {
        const int count = left < kSlab<T> ? static_cast<int>(left) - lead : kSlab<T>;   // of k, from the first chunk on
#pragma unroll
        for (int i = 0; i < I::kChunks; ++i) {
            vec16 v = held.chunk[i];
            if constexpr (kByRow) {
                if (count < I::kVec) v = count > 0 ? shift_down(v, (I::kVec - count) * static_cast<int>(sizeof(T))) : vec16{};
            } else {
                if (i * I::kStep >= count) v = vec16{};
                if (back > 0) v = shift_down(v, back * static_cast<int>(sizeof(T)));
            }
            *reinterpret_cast<vec16*>(lds + (threadIdx.x + i * kThreads) * 16) = v;
        }
    }
};

// The same element by element, for tensors without 16 bytes a row.
template <class T, bool kByRow, int kRows, int kThreads> struct Gathered : Image<T, kByRow, kRows, kThreads> {
    using I = Image<T, kByRow, kRows, kThreads>;
    struct Held {
        vec16 chunk[I::kChunks];
    };
    const T* data;
    int64_t stride, next, first, limit, depth;

    __device__ void begin(const T* base, int64_t pitch, int64_t begin, int64_t end, int64_t ks) {
        data = base;
        stride = pitch;
        next = 0;
        first = begin;
        limit = end;
        depth = ks;
    }

    __device__ void load(Held& held) {
#pragma unroll
        for (int i = 0; i < I::kChunks; ++i) {
            const int r = I::row() + i * I::kStep, c = I::chunk() * I::kVec;
            const int64_t own = first + (kByRow ? r : c), k = next + (kByRow ? c : r);
            const int64_t left = kByRow ? depth - k : limit - own;
            const bool inside = own < limit && k < depth;
            held.chunk[i] = inside ? gather16(data + (kByRow ? own * stride + k : k * stride + own),
                                              left < I::kVec ? static_cast<int>(left) : I::kVec) : vec16{};
        }
        next += kSlab<T>;
    }

    __device__ void store(const Held& held, char* lds, int64_t) const {
#pragma unroll
        for (int i = 0; i < I::kChunks; ++i)
            *reinterpret_cast<vec16*>(lds + (threadIdx.x + i * kThreads) * 16) = held.chunk[i];
    }
};

// How operands reach LDS.
enum Way { kDirect, kStaged, kGathered };

// One workgroup's tile: waves of kWM x kWN, kBM / kWM x kBN / kWN of them.
template <class T, bool kAByRow, bool kBByRow, Way kWay, int kBM, int kBN, int kWM, int kWN, int kWantedStages = 2>
struct Tile {
    static constexpr int kThreads = 64 * (kBM / kWM) * (kBN / kWN);
    template <bool kByRow, int kRows>
    using Loader = std::conditional_t<kWay == kDirect, Direct<T, kByRow, kRows, kThreads>,
                                      std::conditional_t<kWay == kStaged, Staged<T, kByRow, kRows, kThreads>,
                                                         Gathered<T, kByRow, kRows, kThreads>>>;
    using A = Loader<kAByRow, kBM>;
    using B = Loader<kBByRow, kBN>;
    static constexpr int kMs = kWM / 32, kNs = kWN / 32;
    static constexpr int kBuffer = A::kBytes + B::kBytes;
    static constexpr int kPitch = kWN + 4;                  // floats a row of the epilogue's region
    static constexpr int kRegion = 32 * kPitch * 4;
    static constexpr int kStages = kWay == kDirect ? kWantedStages : 2;   // slabs in LDS: one read, the others under way
    static constexpr int kLds = kStages * kBuffer > kThreads / 64 * kRegion ? kStages * kBuffer : kThreads / 64 * kRegion;

    accum16 acc[kMs][kNs];

    static __device__ int wave() { return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64)); }
    static __device__ int wave_row() { return wave() % (kBM / kWM) * kWM; }
    static __device__ int wave_column() { return wave() / (kBM / kWM) * kWN; }

    __device__ void clear() {
#pragma unroll
        for (int i = 0; i < kMs; ++i)
#pragma unroll
            for (int j = 0; j < kNs; ++j) acc[i][j] = accum16{};
    }

    // (Reading a step's fragments while the step before is multiplied gains nothing: two waves a SIMD do that already.)
    __device__ void add_slab(const char* here) {
        const int lane = static_cast<int>(threadIdx.x % 64);
        const int wm = wave_row(), wn = wave_column();
#pragma unroll
        for (int step = 0; step < kSlabBytes / 32; ++step) {
            vec16 fa[kMs], fb[kNs];
#pragma unroll
            for (int i = 0; i < kMs; ++i) fa[i] = A::fragment(here, wm + 32 * i, step, lane);
#pragma unroll
            for (int j = 0; j < kNs; ++j) fb[j] = B::fragment(here + A::kBytes, wn + 32 * j, step, lane);
#pragma unroll
            for (int i = 0; i < kMs; ++i)
#pragma unroll
                for (int j = 0; j < kNs; ++j) acc[i][j] = multiply(T{}, fb[j], fa[i], acc[i][j]);
        }
    }

    // Sums `depth` values of k, the same for the whole workgroup.  a and b have begun.
    __device__ void sum(A& a, B& b, int64_t depth, char* lds) {
        clear();
        if (depth <= 0) return;
        if constexpr (kStages > 2) {
            // Each wave waits for its own loads of the slab (the kAhead - 1 later slabs stay under way) and for its
            // reads of the one before; past the barrier all of it is there, and the buffer read last is
            // free.  Slabs past the end are queued as well, as zeros, so that the count of loads is constant.
            constexpr int kAhead = kStages - 1, kPending = (kAhead - 1) * (A::kChunks + B::kChunks);
            int64_t left = depth;   // of the next slab to queue
#pragma unroll
            for (int s = 0; s < kAhead; ++s, left -= kSlab<T>) {
                a.load(left, lds + s * kBuffer);
                b.load(left, lds + s * kBuffer + A::kBytes);
            }
            int now = 0;
            for (int64_t done = 0; done < depth; done += kSlab<T>, left -= kSlab<T>) {
                arrived<kPending>();
                const int then = now == 0 ? kStages - 1 : now - 1;
                a.load(left, lds + then * kBuffer);
                b.load(left, lds + then * kBuffer + A::kBytes);
                add_slab(lds + now * kBuffer);
                now = now + 1 == kStages ? 0 : now + 1;
            }
            arrived<0>();   // the zeros too, before the LDS is used otherwise
        } else if constexpr (kWay == kDirect) {
            a.load(depth, lds);
            b.load(depth, lds + A::kBytes);
            int now = 0;
            for (int64_t left = depth; left > 0; left -= kSlab<T>) {
                arrived<0>();   // this slab; and no wave reads the other buffer any more
                char* const next = lds + (now ^ 1) * kBuffer;
                if (left > kSlab<T>) {
                    a.load(left - kSlab<T>, next);
                    b.load(left - kSlab<T>, next + A::kBytes);
                }
                add_slab(lds + now * kBuffer);
                now ^= 1;
            }
        } else {
            // kAhead slabs under way in registers, two in LDS
            constexpr int kAhead = kWay == kGathered ? 1 : (kBM * kBN <= 64 * 64 ? 3 : 2);
            typename A::Held ha[kAhead];
            typename B::Held hb[kAhead];
#pragma unroll
            for (int s = 0; s < kAhead; ++s) {
                a.load(ha[s]);
                b.load(hb[s]);
            }
            int now = 0;
            for (int64_t left = depth; left > 0;) {
#pragma unroll
                for (int s = 0; s < kAhead; ++s) {
                    if (left <= 0) break;
                    char* const here = lds + now * kBuffer;
                    a.store(ha[s], here, left);
                    b.store(hb[s], here + A::kBytes, left);
                    __syncthreads();   // the slab is there; and no wave reads the buffer of the slab before last
                    a.load(ha[s]);
                    b.load(hb[s]);
                    add_slab(here);
                    left -= kSlab<T>;
                    now ^= 1;
                }
            }
        }
        __syncthreads();
    }

    static constexpr int kLanes = kWN / 8;                   // lanes a row of the epilogue, 8 columns each
    static constexpr int kHeight = 64 / kLanes;              // rows a pass
    static constexpr int kPasses = 32 / kHeight;
    static constexpr int kGroup = kPasses < 4 ? kPasses : 4; // passes handed out together

    static __device__ int own_column() { return wave_column() + static_cast<int>(threadIdx.x % kLanes) * 8; }

    // Hands out the tile's values: a lane's are the 8 columns from own_column() on of kGroup rows at a time, row,
    // row + kHeight, ... (relative to the tile).
    //   fetch(row) -> what use needs from memory for these rows, asked for a group ahead of
    //   use(row, value[kGroup][8], fetched)
    template <class Fetch, class Use> __device__ void rows(char* lds, Fetch&& fetch, Use&& use) {
        const int lane = static_cast<int>(threadIdx.x % 64);
        float* region = reinterpret_cast<float*>(lds + wave() * kRegion);
        const float* from = region + lane / kLanes * kPitch + lane % kLanes * 8;
        // accumulator element v of lane l: row l % 32, column 8 (v / 4) + 4 (l / 32) + v % 4
        float* to = region + lane % 32 * kPitch + lane / 32 * 4;
#pragma unroll
        for (int i = 0; i < kMs; ++i) {
            const int row = wave_row() + 32 * i + lane / kLanes;
            auto fetched = fetch(row);
#pragma unroll
            for (int j = 0; j < kNs; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4*>(to + 32 * j + 8 * q) =
                        make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
            wave_fence();
#pragma unroll 1
            for (int pass = 0; pass < kPasses; pass += kGroup) {
                auto ahead = fetched;
                if (pass + kGroup < kPasses) ahead = fetch(row + (pass + kGroup) * kHeight);
                float value[kGroup][8];
#pragma unroll
                for (int u = 0; u < kGroup; ++u) {
                    const float* p = from + (pass + u) * kHeight * kPitch;
                    const float4 lo = *reinterpret_cast<const float4*>(p), hi = *reinterpret_cast<const float4*>(p + 4);
                    value[u][0] = lo.x, value[u][1] = lo.y, value[u][2] = lo.z, value[u][3] = lo.w;
                    value[u][4] = hi.x, value[u][5] = hi.y, value[u][6] = hi.z, value[u][7] = hi.w;
                }
                use(row + pass * kHeight, value, fetched);
                fetched = ahead;
            }
            wave_fence();
        }
    }
};

enum Activation { kNone = 0, kRelu, kSigmoid, kSoftplus, kGelu, kSilu, kActivations };

// Activations and their slopes in fp32.  A NaN stays one (but for relu's slope: 0).
// kExact, for fp32 tensors: the library's exp, log1p and erfc.  Otherwise, for values that are rounded to
// 16 bits: the hardware's exp2, log2 and reciprocal (1 ulp each) and, for erfc(x), exp(-x^2) t P(t) with
// t = 1 / (1 + 0.368 x) and P fitted for it over 0 <= x <= 10, by weighted least squares towards the smallest largest
// relative error: 1.8e-6, and 1.8e-7 near 0.  The normal distribution is off by 2.5e-7, and relatively by less than
// 1e-5 down to z = -13, where exp ends; gelu's left tail is as small as that.  It shares its exp(-z^2 / 2)
// with the slope: on 65536 x 4096 the gelu's slope would otherwise be bound by its arithmetic, not by HBM.
template <bool kExact> __device__ inline float exp_of(float x) {
    if constexpr (kExact) return expf(x);
    return __builtin_amdgcn_exp2f(x * 1.44269504f);
}
template <bool kExact> __device__ inline float inverse(float x) {
    if constexpr (kExact) return 1.0f / x;
    return __builtin_amdgcn_rcpf(x);
}

// The normal distribution at z, and exp(-z^2 / 2).
template <bool kExact> __device__ inline float normal_below(float z, float& bell) {
    bell = exp_of<kExact>(-0.5f * z * z);
    if constexpr (kExact) return 0.5f * erfcf(-0.70710678f * z);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.26021528f, fabsf(z), 1.0f));   // 0.368 / sqrt 2
    float p = fmaf(t, -0.147252902f, 0.461173415f);
    p = fmaf(t, p, -0.217935473f);
    p = fmaf(t, p, 0.336780846f);
    p = fmaf(t, p, 0.145215213f);
    p = fmaf(t, p, 0.214837208f);
    p = fmaf(t, p, 0.207181513f);
    const float above = 0.5f * t * p * bell;   // beyond |z|
    return z < 0.0f ? above : 1.0f - above;
}

template <int kActivation, bool kExact> __device__ inline float activate(float z) {
    if constexpr (kActivation == kRelu) return z < 0.0f ? 0.0f : z;
    if constexpr (kActivation == kSigmoid) return inverse<kExact>(1.0f + exp_of<kExact>(-z));
    if constexpr (kActivation == kSoftplus) {
        const float e = exp_of<kExact>(-fabsf(z)), top = z > 0.0f ? z : 0.0f;
        if constexpr (kExact) return top + log1pf(e);
        const float log = e < 0.015625f ? e * fmaf(e, fmaf(e, 0.33333333f, -0.5f), 1.0f)
                                        : 0.69314718f * __builtin_amdgcn_logf(1.0f + e);
        return top + log;
    }
    if constexpr (kActivation == kGelu) {
        float bell;
        return z * normal_below<kExact>(z, bell);
    }
    if constexpr (kActivation == kSilu) return z * inverse<kExact>(1.0f + exp_of<kExact>(-z));
    return z;
}

// The limits at infinity: a sum past fp16's range is kept as an infinite one.  gelu's and silu's slopes multiply z by a
// factor that is 0 in fp32 well before |z| = 128, and take z no further than that (a NaN stays in the other factor).
template <int kActivation, bool kExact> __device__ inline float slope(float z) {
    if constexpr (kActivation == kRelu) return z > 0.0f ? 1.0f : 0.0f;
    const float near = __builtin_amdgcn_fmed3f(z, -128.0f, 128.0f);
    if constexpr (kActivation == kGelu) {
        float bell;
        const float below = normal_below<kExact>(z, bell);
        return fmaf(near * 0.39894228f, bell, below);
    }
    if constexpr (kActivation == kSigmoid || kActivation == kSoftplus || kActivation == kSilu) {
        // sigmoid(|z|) and sigmoid(-|z|), neither by a difference
        const float e = exp_of<kExact>(-fabsf(z)), more = inverse<kExact>(1.0f + e), less = e * more;
        if constexpr (kActivation == kSigmoid) return more * less;
        const float s = z < 0.0f ? less : more;
        if constexpr (kActivation == kSoftplus) return s;
        return s * fmaf(near, z < 0.0f ? more : less, 1.0f);
    }
    return 1.0f;
}

// f<kActivation>() for the activation of this launch: one branch, the same for every lane.
template <class F> __device__ inline void with_activation(int activation, F&& f) {
    switch (activation) {
        case kRelu: return f(std::integral_constant<int, kRelu>{});
        case kSigmoid: return f(std::integral_constant<int, kSigmoid>{});
        case kSoftplus: return f(std::integral_constant<int, kSoftplus>{});
        case kGelu: return f(std::integral_constant<int, kGelu>{});
        case kSilu: return f(std::integral_constant<int, kSilu>{});
        default: return f(std::integral_constant<int, kNone>{});
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
    float* partial;           // [partial slots][outputs][inputs] sums of groups cut into several pieces
    const int32_t* offsets;
    int64_t rows, ldz, ldx;
    int64_t piece;            // rows a workgroup sums
    int64_t pieces;           // piece ids
    int edge;                 // of the tiles: 256, 128 or 64
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

// Lanes across the columns, 8 each, of the slope pass' workgroups.
inline int slope_lanes(int columns) {
    int lanes = 1;
    while (lanes < 32 && 8 * lanes < columns) lanes *= 2;
    return lanes;
}

struct FoldArgs {             // out[e][i] = sum over e's pieces of partial[place of the piece][i]
    const float* partial;
    void* out;
    const int32_t* offsets;
    int64_t rows, piece, size;
    int experts;
    bool single;              // partial sums of every piece by its id, whole groups' too (zeros for groups of none);
                              // else by partial_slot, and whole groups are left alone
};

// Launches, per element type.
template <class T> int launch_rows(const RowsArgs& a, bool forward, hipStream_t stream);
template <class T> int launch_weight(const WeightArgs& a, hipStream_t stream);
template <class T> int launch_slope(const SlopeArgs& a, hipStream_t stream);
template <class T> int launch_fold(const FoldArgs& a, hipStream_t stream);

}  // namespace odie
