// The three element types of the row operators (fp32, fp16, bf16) and their 16-byte vectors.
//
// Values are widened to fp32 for every sum and rounded once, to nearest even, where they are
// stored.  Rows may start at any element: 16-byte accesses go through memcpy, which compiles to the
// wide global instructions whether or not the address is 16-byte aligned (unaligned access mode).
#pragma once
#include <cstdint>
#include <type_traits>

#include "common.h"
#include "../../include/odie_amd.h"

namespace odie {

typedef uint32_t vec16 __attribute__((ext_vector_type(4)));   // 16 bytes of any element type

constexpr int64_t kStreamBytes = int64_t{32} << 20;   // the L2s' 4 MB on each of 8 XCDs

template <class T> constexpr int kPerVec = 16 / static_cast<int>(sizeof(T));

template <class T> __device__ inline vec16 load16(const T* p) {
    vec16 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// kStream: past the caches' retention, for outputs too large for the L2s to hold until they are read
// (kStreamBytes): 4M looked-up rows of 64 bytes 92 -> 44 us over and over, and with their gradient in between 88,
// the two together 356 -> 337.  A constant, because the compiler makes one store of the two sides of a branch.
typedef uint32_t vec16_any __attribute__((ext_vector_type(4), aligned(2)));
template <bool kStream = false, class T> __device__ inline void store16(T* p, const vec16& v) {
    if constexpr (kStream) __builtin_nontemporal_store(v, reinterpret_cast<vec16_any*>(p));
    else __builtin_memcpy(p, &v, 16);
}

// The first `count` elements at p (0 <= count), zeros after them, element by element.
template <class T> __device__ inline vec16 gather16(const T* p, int count) {
    vec16 v{};
    if constexpr (sizeof(T) == 4) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < count ? q[i] : 0u;
    } else {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t low = 2 * i < count ? q[2 * i] : 0u, high = 2 * i + 1 < count ? q[2 * i + 1] : 0u;
            v[i] = low | high << 16;
        }
    }
    return v;
}

template <class T> __device__ inline void scatter16(T* p, const vec16& v, int count) {
    if constexpr (sizeof(T) == 4) {
        uint32_t* q = reinterpret_cast<uint32_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) q[i] = v[i];
    } else {
        uint16_t* q = reinterpret_cast<uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (2 * i < count) q[2 * i] = static_cast<uint16_t>(v[i]);
            if (2 * i + 1 < count) q[2 * i + 1] = static_cast<uint16_t>(v[i] >> 16);
        }
    }
}

template <class T> __device__ inline vec16 load_some(const T* p, int count) {
    return count >= kPerVec<T> ? load16(p) : gather16(p, count);
}

template <bool kStream = false, class T> __device__ inline void store_some(T* p, const vec16& v, int count) {
    if (count >= kPerVec<T>) store16<kStream>(p, v);
    else scatter16(p, v, count);
}

// A row of `width` elements as ceil(width / kPerVec) chunks of 16 bytes.  The last chunk ends with the row:
// where the width is no multiple it begins inside the chunk before it, and writes the same values there
// again.  Only a row shorter than a chunk goes element by element.
template <class T> __device__ inline int chunk_column(int chunk, int width) {
    const int column = chunk * kPerVec<T>, last = width - kPerVec<T>;
    return column < last || last < 0 ? column : last;
}

// Elements of the chunk that the chunk before it holds as well.
template <class T> __device__ inline int chunk_overlap(int chunk, int width) {
    return chunk * kPerVec<T> - chunk_column<T>(chunk, width);
}

template <class T> __device__ inline vec16 load_chunk(const T* row, int chunk, int width) {
    const T* p = row + chunk_column<T>(chunk, width);
    return width >= kPerVec<T> ? load16(p) : gather16(p, width);
}

template <bool kStream = false, class T> __device__ inline void store_chunk(T* row, int chunk, int width, const vec16& v) {
    T* p = row + chunk_column<T>(chunk, width);
    if (width >= kPerVec<T>) store16<kStream>(p, v);
    else scatter16(p, v, width);
}

// v moved down by `bytes` (0..15), zeros above.
__device__ inline vec16 shift_down(const vec16& v, int bytes) {
    uint64_t low = static_cast<uint64_t>(v.y) << 32 | v.x, high = static_cast<uint64_t>(v.w) << 32 | v.z;
    if (bytes >= 8) {
        low = high;
        high = 0;
        bytes -= 8;
    }
    if (bytes > 0) {
        low = low >> 8 * bytes | high << (64 - 8 * bytes);
        high >>= 8 * bytes;
    }
    return vec16{static_cast<uint32_t>(low), static_cast<uint32_t>(low >> 32), static_cast<uint32_t>(high),
                 static_cast<uint32_t>(high >> 32)};
}

// The first `count` elements at p (at least one) and zeros after them, where the `back` elements before p can be
// read too: the last 16 bytes that end with them, moved down.
template <class T> __device__ inline vec16 load_end(const T* p, int count, int64_t back) {
    if (count >= kPerVec<T>) return load16(p);
    const int missing = kPerVec<T> - count;
    if (back < missing) return gather16(p, count);
    return shift_down(load16(p - missing), missing * static_cast<int>(sizeof(T)));
}

template <class T> __device__ inline void widen(const vec16& v, float out[kPerVec<T>]) {
    T e[kPerVec<T>];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int i = 0; i < kPerVec<T>; ++i) out[i] = static_cast<float>(e[i]);
}

// Rounds fp32 values.  They are materialised first: folded into the conversion, a product or sum is rounded
// once instead of twice, and the compiler does so for some places of a vector and not for others, so that
// an element's value would depend on where in a chunk it lies.
template <class T> __device__ inline vec16 narrow(const float in[kPerVec<T>]) {
    T e[kPerVec<T>];
#pragma unroll
    for (int i = 0; i < kPerVec<T>; ++i) {
        float value = in[i];
        asm("" : "+v"(value));
        e[i] = static_cast<T>(value);
    }
    vec16 v;
    __builtin_memcpy(&v, e, 16);
    return v;
}

// Eight consecutive elements, of which `count` exist (those past them read as 0 and are not written).
template <class T> struct Eight {
    static constexpr int kWords = 8 / kPerVec<T>;
    vec16 word[kWords];

    __device__ void load(const T* p, int count) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) word[w] = load_some(p + w * kPerVec<T>, count - w * kPerVec<T>);
    }
    __device__ void get(float out[8]) const {
#pragma unroll
        for (int w = 0; w < kWords; ++w) widen<T>(word[w], out + w * kPerVec<T>);
    }
};

template <class T> __device__ inline void load8(const T* p, int count, float out[8]) {
    Eight<T> e;
    e.load(p, count);
    e.get(out);
}

template <bool kStream = false, class T> __device__ inline void store8(T* p, int count, const float in[8]) {
#pragma unroll
    for (int w = 0; w < 8 / kPerVec<T>; ++w)
        store_some<kStream>(p + w * kPerVec<T>, narrow<T>(in + w * kPerVec<T>), count - w * kPerVec<T>);
}

// A wave orders its own LDS accesses: lanes read what other lanes of the wave wrote.
__device__ inline void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Workgroups of `threads` threads that one launch takes, in whole rounds of the XCDs.  Past 2^32 threads the runtime
// launches fewer workgroups than it was asked for, without an error.
inline int64_t most_blocks(int threads) { return ((int64_t{1} << 32) - 1) / threads / kXcds * kXcds; }

// Calls f(first, count) for as many launches as `blocks` workgroups need: one, up to billions of rows.
template <class F> void in_launches(int64_t blocks, int threads, F&& f) {
    const int64_t most = most_blocks(threads);
    for (int64_t first = 0; first < blocks; first += most)
        f(static_cast<uint32_t>(first), static_cast<uint32_t>(blocks - first < most ? blocks - first : most));
}

inline bool known_dtype(int dtype) { return dtype == ODIE_F32 || dtype == ODIE_F16 || dtype == ODIE_BF16; }
inline int64_t dtype_bytes(int dtype) { return dtype == ODIE_F32 ? 4 : 2; }

// Calls f with a constant of the flag's value.
template <class F> void with_flag(bool flag, F&& f) {
    if (flag) f(std::true_type{});
    else f(std::false_type{});
}

// Calls f with a value of the element type `dtype` names (checked by the caller).
template <class F> auto with_dtype(int dtype, F&& f) {
    if (dtype == ODIE_F16) return f(_Float16{});
    if (dtype == ODIE_BF16) return f(__bf16{});
    return f(float{});
}

// Rows grouped by expert: expert e owns rows [offsets[e], offsets[e + 1]), the rows from
// offsets[experts] on belong to none (they form group `experts`); a null offsets is one expert
// that owns every row.  Groups are cut into pieces of `piece` rows.  Piece ids: group e's begin at
//   s(e) = floor(offsets[e] / piece) + e,
// which leaves each group room for its pieces, because s(e + 1) - s(e) >= ceil(rows of e / piece) and
// >= 1; so a piece id finds its group by comparing s alone, with no table of counts, and ids left
// over find no rows.  There are piece_ids() of them.
struct Piece {
    int group;
    int first;       // piece number inside the group
    int64_t begin;   // rows [begin, end) of the tensor; begin >= end: nothing to do
    int64_t end;
    int64_t group_begin;
    int64_t group_end;
};

inline int64_t piece_ids(int64_t rows, int64_t piece, bool grouped, int experts, bool tail) {
    return grouped ? rows / piece + experts + (tail ? 1 : 0) : (rows + piece - 1) / piece;
}

__device__ inline int64_t group_start(const int32_t* offsets, int group, int64_t rows) {
    const int64_t at = offsets[group];
    return at < 0 ? 0 : (at > rows ? rows : at);   // whatever offsets hold, no row outside the tensor
}

// floor(offsets[group] / piece) (offsets and, with them, rows are below 2^31).
__device__ inline int64_t whole_pieces(const int32_t* offsets, int group, int64_t rows, int64_t piece) {
    return static_cast<uint32_t>(group_start(offsets, group, rows)) / static_cast<uint32_t>(piece);
}

// Partial sums of groups that are longer than a piece, and of those alone: piece `first` of a group that begins at row
// `begin` has slot floor(2 begin / piece) + first.  A group of more than a piece has at most twice its length in
// pieces, rounded down, so that the next group's slots begin past its own, and partial_slots(rows) are enough
// however many groups there are.
inline int64_t partial_slots(int64_t rows, int64_t piece, bool grouped) {
    return grouped ? 2 * rows / piece : (rows + piece - 1) / piece;
}

__device__ inline int64_t partial_slot(int64_t begin, int64_t piece, int first) {
    return static_cast<uint32_t>(2 * begin) / static_cast<uint32_t>(piece) + static_cast<int64_t>(first);
}

// The piece `id` of groups 0..groups-1 (groups = experts + 1 with the rows of no expert, else
// experts).  All 64 lanes of the wave call it with the same id.
__device__ inline Piece find_piece(const int32_t* offsets, int experts, int groups, int64_t rows, int64_t piece,
                                   int64_t id) {
    Piece p{};
    if (!offsets) {
        p.first = static_cast<int>(id);
        p.group_end = rows;
    } else {
        const int lane = static_cast<int>(threadIdx.x % 64);
        // the last group g with s(g) <= id: 64 probes a round, first spaced, then closer
        int low = 0, span = groups;
        while (span > 1) {
            const int step = (span + 63) / 64;
            const int g = low + lane * step;
            const bool below = lane * step < span && whole_pieces(offsets, g, rows, piece) + g <= id;
            const int count = __popcll(__ballot(below));    // s increases: the lanes below come first
            const int found = count > 1 ? count : 1;
            low += (found - 1) * step;                      // s(low) <= id always: lane 0 is one of them
            span = span - (found - 1) * step < step ? span - (found - 1) * step : step;
        }
        p.group = __builtin_amdgcn_readfirstlane(low);
        p.group_begin = group_start(offsets, p.group, rows);
        p.group_end = p.group < experts ? group_start(offsets, p.group + 1, rows) : rows;
        p.first = static_cast<int>(id - (whole_pieces(offsets, p.group, rows, piece) + p.group));
    }
    p.begin = p.group_begin + p.first * piece;
    p.end = p.begin + piece < p.group_end ? p.begin + piece : p.group_end;
    return p;
}

}  // namespace odie
