// A learned router over experts: the choice of each row's experts with their softmax weights, and the loss that
// keeps their load even, with their gradients.
//
//   choose   e_1 .. e_k: the row's largest logits, the lowest index first among equal ones; w_j = exp(l_ej - m) / s, s
//            over the chosen (normalised) or over all experts
//            dl_e = [e = e_j] w_j g_j - q_e sum_i w_i g_i, q the softmax over the chosen or over all
//   balance  c_e entries of expert e, M in all; R rows that have an entry; t_i = sum_e c_e p_ie over row i's softmax
//            loss = E / (M R) sum_i t_i,  dl_ie = g E / (M R) p_ie (c_e - t_i)
//
// The loss is E sum_e (c_e / M) (mean over rows of p_ie) with its sums exchanged: each row needs its own
// logits and the counts alone, and no sums down the columns exist.  Counts are whole numbers, and everything else
// is added in a fixed order: the same call gives the same bits.  c_e - t_i may be far smaller than either: in an even
// load both are near M / E, and in a row that is sure of one expert both are near that one's count.  So a row takes a
// whole number near its t_i off the counts, which is exact, and t_i is that number and the mean of what is left; nothing
// is rounded relative to a count.
#include "softmax.h"

namespace odie {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxExperts = 1 << 15;
constexpr int kMaxChoices = 64;
constexpr int64_t kMaxEntries = (int64_t{1} << 31) - 1;

template <class N> __device__ inline N most_of(N a, N b) { return a > b ? a : b; }
template <class N> __device__ inline N least_of(N a, N b) { return a < b ? a : b; }

// Logits with their indices as whole numbers: the larger the logit and, among equal ones, the lower the index, the
// larger the key.  A logit's bits become a signed number in the order of the values by negating the magnitude of
// negative ones (which makes -0 and 0 alike); a NaN is the largest.  A 16-bit logit and its index fit 32 bits.  No fp32
// key is INT64_MAX, below which choose_long_kernel's search for the first choice begins.
template <class T> struct Keys {
    using Key = int32_t;
    static constexpr Key kNone = INT32_MIN;
    static constexpr uint32_t kInfinity = std::is_same_v<T, __bf16> ? 0x7f80u : 0x7c00u;
    typedef int16_t two __attribute__((ext_vector_type(2)));

    // The keys of a 16-byte chunk whose first index is `index` (a multiple of 8).  kChecked: with NaN in it.
    template <bool kChecked> static __device__ void of(const vec16& chunk, int index, Key key[8]) {
        const uint32_t rest = static_cast<uint32_t>(0xffff - index);      // its low three bits are ones
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t word = chunk[w];       // a bit cast of the element itself would take the vector's first
            const two bits = __builtin_bit_cast(two, word), sign = bits >> static_cast<int16_t>(15);
            const two size = bits & static_cast<int16_t>(0x7fff), order = (size ^ sign) - sign;
            uint32_t pair = __builtin_bit_cast(uint32_t, order);
            if constexpr (kChecked) {
                const uint32_t sizes = __builtin_bit_cast(uint32_t, size);
                if ((sizes & 0xffffu) > kInfinity) pair |= 0x7fffu, pair &= 0xffff7fffu;
                if (sizes >> 16 > kInfinity) pair |= 0x7fff0000u, pair &= 0x7fffffffu;
            }
            key[2 * w] = static_cast<Key>(pair << 16 | (rest ^ (2 * w)));
            key[2 * w + 1] = static_cast<Key>((pair & 0xffff0000u) | (rest ^ (2 * w + 1)));
        }
    }
    static __device__ bool has_nan(const vec16& chunk) {
        typedef uint16_t twos __attribute__((ext_vector_type(2)));
        twos most{};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t sizes = chunk[w] & 0x7fff7fffu;
            most = __builtin_elementwise_max(most, __builtin_bit_cast(twos, sizes));
        }
        return most[0] > kInfinity || most[1] > kInfinity;
    }
    static __device__ int index(Key key) { return 0xffff - static_cast<int>(key & 0xffff); }
    static __device__ float value(Key key) {
        const int order = key >> 16;
        return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(order < 0 ? 0x8000 | -order : order)));
    }
    // the middle one
    static __device__ Key second(Key most, Key less, Key key) {
        return most_of(least_of(most, less), least_of(most_of(most, less), key));
    }
    template <int kLanes> static __device__ Key best(Key key) {
        return static_cast<Key>(across<kLanes>(static_cast<uint32_t>(key), [](uint32_t a, uint32_t b) {
            return static_cast<uint32_t>(most_of(static_cast<int32_t>(a), static_cast<int32_t>(b)));
        }));
    }
};
template <> struct Keys<float> {
    using Key = int64_t;
    static constexpr Key kNone = INT64_MIN;

    static __device__ Key of(float value, int index) {
        const int32_t bits = __builtin_bit_cast(int32_t, value), sign = bits >> 31, size = bits & 0x7fffffff;
        const int32_t order = size > 0x7f800000 ? 0x7fc00000 : (size ^ sign) - sign;
        return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(order)) << 32 |
                                    static_cast<uint32_t>(~index));
    }
    template <bool kChecked> static __device__ void of(const vec16& chunk, int index, Key key[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) key[i] = of(as_float(chunk[i]), index + i);
    }
    static __device__ bool has_nan(const vec16&) { return false; }      // of() tells
    static __device__ int index(Key key) { return static_cast<int>(~static_cast<uint32_t>(key)); }
    static __device__ float value(Key key) {
        const int32_t order = static_cast<int32_t>(key >> 32);
        return __builtin_bit_cast(float, order < 0 ? INT32_MIN | -order : order);
    }
    static __device__ Key second(Key most, Key less, Key key) { return most_of(less, least_of(most, key)); }
    template <int kLanes> static __device__ Key best(Key key) {
        // the largest order first, then the largest rest among the lanes that hold it
        const int32_t order = static_cast<int32_t>(key >> 32);
        const auto larger_order = [](uint32_t a, uint32_t b) {
            return static_cast<uint32_t>(most_of(static_cast<int32_t>(a), static_cast<int32_t>(b)));
        };
        const int32_t top = static_cast<int32_t>(across<kLanes>(static_cast<uint32_t>(order), larger_order));
        const uint32_t rest = across<kLanes>(order == top ? static_cast<uint32_t>(key) : 0u,
                                             [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(top)) << 32 | rest);
    }
};

// A row's 16-byte chunks, kVecs a lane, loaded ahead of their use: without conditions, which would make the compiler
// wait for loads in flight, from addresses moved back into the row where they would leave it; settle() puts that right.
// The first half of several chunks is always whole (with_row).  Rows shorter than a chunk are gathered.
template <class T, int kLanes, int kVecs> struct RowHold {
    static constexpr int kV = kPerVec<T>;
    vec16 chunk[kVecs];

    __device__ void load(const T* row, int lane, int width) {
        if (width < kV) {
            chunk[0] = gather16(row, lane == 0 ? width : 0);
            return;
        }
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const int column = (v * kLanes + lane) * kV;
            chunk[v] = load16(row + (v < kVecs / 2 || column < width - kV ? column : width - kV));
        }
    }
    // Moves what lies across the row's end to its place, zeros past it; before get().
    __device__ void settle(int lane, int width) {
#pragma unroll
        for (int v = kVecs / 2; v < kVecs; ++v) {
            const int count = width - (v * kLanes + lane) * kV;
            if (count < kV && width >= kV)
                chunk[v] = count > 0 ? shift_down(chunk[v], (kV - count) * static_cast<int>(sizeof(T))) : vec16{};
        }
    }
    __device__ void get(int v, int lane, int width, float value[kV]) const {
        const int count = width - (v * kLanes + lane) * kV;
        widen<T>(chunk[v], value);
        if (v >= kVecs / 2 && count < kV)
#pragma unroll
            for (int i = 0; i < kV; ++i) value[i] = i < count ? value[i] : kNegInfinity;
    }
};

struct ChooseArgs {
    const void* logits;       // [n][experts], stride
    int64_t stride, n;
    int32_t* expert;          // [n][choices]
    float* weights;           // [n][choices]
    float* stats;             // [n][2]: m and 1 / s over all experts (0 in a row of none), or null
    int experts, choices;
    int normalize;
};

// The largest key, and the sum, over the kLanes threads of a row, for each of them.  More than a wave: by LDS, where
// every other call (`turn`) takes the same place, so that one barrier a call is enough.
template <class K, int kLanes, int kWaves>
__device__ inline typename K::Key best_of(typename K::Key key, typename K::Key (&part)[2][kWaves], int& turn) {
    if constexpr (kLanes <= 64) return K::template best<kLanes>(key);
    key = K::template best<64>(key);
    turn ^= 1;
    if (threadIdx.x % 64 == 0) part[turn][threadIdx.x / 64] = key;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) key = most_of(key, part[turn][w]);
    return key;
}
template <int kLanes, int kWaves> __device__ inline float sum_of(float x, float (&part)[2][kWaves], int& turn) {
    if constexpr (kLanes <= 64) return sum_across<kLanes>(x);
    x = sum_across<64>(x);
    turn ^= 1;
    if (threadIdx.x % 64 == 0) part[turn][threadIdx.x / 64] = x;
    __syncthreads();
    x = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) x += part[turn][w];
    return x;
}

// Rows of up to kLanes kVecs chunks in registers, the next one under way.  Each lane keeps its two largest keys; a
// choice takes the largest of all lanes, whose lane goes on to its second, and looks through its keys again once both
// are gone: at four choices of 1024 about once in 500 rows.  65536 x 1024 fp16, four choices with weights among all: 47
// to 50 us, 134 MB at 2.7 to 2.9 TB/s, bound by the arithmetic (about 450 instructions a row, of which each choice's
// reduction over a whole wave serves one row; with a search of all keys for each choice 61 us); one row 2 us.  8192
// rows of 4096, 8000, 16000 and 32000 bf16: 24, 39, 92 and 172 us (a row read for
// each choice -, 124, 235 and 454).
template <class T, int kLanes, int kVecs>
__global__ __launch_bounds__(kLanes > kBlock ? kLanes : kBlock) void choose_kernel(ChooseArgs a) {
    using K = Keys<T>;
    using Key = typename K::Key;
    constexpr int kV = kPerVec<T>, kValues = kVecs * kV;
    constexpr int kThreads = kLanes > kBlock ? kLanes : kBlock, kRows = kThreads / kLanes, kWaves = kThreads / 64;
    __shared__ Key part[2][kWaves];
    __shared__ float sums[2][kWaves];
    int turn = 0, sums_turn = 0;
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    const T* logits = static_cast<const T*>(a.logits);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int64_t at = static_cast<int64_t>(blockIdx.x) * kRows + static_cast<int>(threadIdx.x) / kLanes;
    constexpr bool kAhead = kLanes < 1024;      // whose registers do not hold two rows
    RowHold<T, kLanes, kVecs> next;
    if constexpr (kAhead) next.load(logits + (at < a.n ? at : a.n - 1) * a.stride, lane, a.experts);
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.n; base += step, at += step) {
        if constexpr (!kAhead) next.load(logits + at * a.stride, lane, a.experts);
        RowHold<T, kLanes, kVecs> row = next;
        if constexpr (kAhead) next.load(logits + (at + step < a.n ? at + step : a.n - 1) * a.stride, lane, a.experts);
        row.settle(lane, a.experts);
        Key key[kValues];
        bool nan = false;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            K::template of<false>(row.chunk[v], (v * kLanes + lane) * kV, key + v * kV);
            nan |= K::has_nan(row.chunk[v]);
        }
        if (__any(nan)) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) K::template of<true>(row.chunk[v], (v * kLanes + lane) * kV, key + v * kV);
        }
#pragma unroll
        for (int v = kVecs / 2; v < kVecs; ++v) {
            const int count = a.experts - (v * kLanes + lane) * kV;
            if (count < kV)
#pragma unroll
                for (int i = 0; i < kV; ++i) key[v * kV + i] = i < count ? key[v * kV + i] : K::kNone;
        }
        Key most = K::kNone, less = K::kNone;
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            less = K::second(most, less, key[i]);
            most = most_of(most, key[i]);
        }
        Key mine = K::kNone, first = K::kNone;      // lane j: the j-th choice
        bool left = most != K::kNone;
        for (int j = 0; j < a.choices; ++j) {
            const Key best = best_of<K, kLanes>(most, part, turn);
            if (j == 0) first = best;
            if (lane == j) mine = best;
            if (most == best) most = less, less = K::kNone;
            if (__any(left && most == K::kNone)) {
                Key below = K::kNone;
#pragma unroll
                for (int i = 0; i < kValues; ++i) below = most_of(below, key[i] < best ? key[i] : K::kNone);
                if (most == K::kNone) {
                    most = below;
                    left = below != K::kNone;
                }
            }
        }
        const float m = first == K::kNone ? kNegInfinity : K::value(first), base_value = base_of(m);
        const float chosen = mine == K::kNone ? kNegInfinity : K::value(mine);
        const bool held = !(chosen == kNegInfinity);
        const float own = held ? expf(chosen - base_value) : 0.0f;
        float s = own;
        if (!a.normalize) {
            s = 0.0f;
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                float value[kV];
                row.get(v, lane, a.experts, value);
#pragma unroll
                for (int i = 0; i < kV; ++i) s += exponential<sizeof(T) == 4>(value[i] - base_value);
            }
        }
        s = sum_of<kLanes>(s, sums, sums_turn);
        const float inverse = m == kNegInfinity ? 0.0f : 1.0f / s;
        if (at >= a.n) continue;
        if (lane < a.choices) {
            a.expert[at * a.choices + lane] = held ? K::index(mine) : -1;
            a.weights[at * a.choices + lane] = held ? own * inverse : 0.0f;
        }
        if (a.stats && lane == 0) *reinterpret_cast<float2*>(a.stats + at * 2) = make_float2(m, inverse);
    }
}

// The largest key of the workgroup, for every thread; `part` holds a key a wave.
__device__ inline int64_t block_best(int64_t key, int64_t* part) {
    key = Keys<float>::best<64>(key);
    __syncthreads();
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = key;
    __syncthreads();
    for (int w = 0; w < kBlock / 64; ++w) key = most_of(key, part[w]);
    return key;
}

// A workgroup a row of fp32, whose keys take 64 bits: it reads the row once for each choice, the one below the last.  For
// rows that do not fit its registers, and long rows of few choices (by_turns).
__global__ __launch_bounds__(kBlock) void choose_long_kernel(ChooseArgs a) {
    using T = float;
    using K = Keys<T>;
    constexpr int kV = kPerVec<T>;
    __shared__ int64_t part[kBlock / 64];
    __shared__ float sums[kBlock / 64];
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
        const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
        int64_t mine = K::kNone, first = K::kNone, last = INT64_MAX;
        for (int j = 0; j < a.choices; ++j) {
            int64_t local = K::kNone;
            for (int column = static_cast<int>(threadIdx.x) * kV; column < a.experts; column += kBlock * kV) {
                float value[kV];
                load_logits(logits, column, a.experts, value);
#pragma unroll
                for (int i = 0; i < kV; ++i) {
                    const int64_t key = column + i < a.experts ? K::of(value[i], column + i) : K::kNone;
                    if (key < last) local = most_of(local, key);
                }
            }
            last = block_best(local, part);
            if (j == 0) first = last;
            if (static_cast<int>(threadIdx.x) == j) mine = last;
        }
        const float m = K::value(first), base = base_of(m), chosen = mine == K::kNone ? kNegInfinity : K::value(mine);
        const bool held = !(chosen == kNegInfinity);
        const float own = held ? expf(chosen - base) : 0.0f;
        float s = own;
        if (!a.normalize) {
            s = 0.0f;
            for (int column = static_cast<int>(threadIdx.x) * kV; column < a.experts; column += kBlock * kV) {
                float value[kV];
                load_logits(logits, column, a.experts, value);
#pragma unroll
                for (int i = 0; i < kV; ++i) s += exponential<true>(value[i] - base);
            }
        }
        s = sum_across<64>(s);
        __syncthreads();
        if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = s;
        __syncthreads();
        s = 0.0f;
        for (int w = 0; w < kBlock / 64; ++w) s += sums[w];
        const float inverse = m == kNegInfinity ? 0.0f : 1.0f / s;
        if (static_cast<int>(threadIdx.x) < a.choices) {
            a.expert[row * a.choices + threadIdx.x] = held ? K::index(mine) : -1;
            a.weights[row * a.choices + threadIdx.x] = held ? own * inverse : 0.0f;
        }
        if (a.stats && threadIdx.x == 0) {
            a.stats[row * 2] = m;
            a.stats[row * 2 + 1] = inverse;
        }
    }
}

struct ChooseBackwardArgs {
    const float* upstream;    // [n][choices]
    const int32_t* expert;
    const float* weights;
    const void* logits;       // null where the weights are normalised
    const float* stats;
    void* dlogits;            // [n][experts]
    int64_t stride, n;
    int experts, choices;
};

// kLanes lanes a row write its gradient chunk by chunk; each lane holds one of the row's entries, and writes it once more
// afterwards (kPatched) or hands it to the lane whose chunk it falls in.  Handing out costs about 26 instructions an
// entry and round of chunks; writing again moves lines a second time.  us handed out and patched, rows of 2^26 values in
// all, choices among themselves and with weights of all:
//   fp16 x 64    two 28, 48 and 41, 54    four 35, 54 and 40, 56    five 37, 56 and 42, 57    eight 47, 66 and 48, 61
//        x 512   two 23, 48 and 26, 47    four 30, 52 and 29, 48    five 35, 55 and 30, 49    eight 45, 62 and 32, 49
//        x 1024  two 23, 41 and 27, 43    four 27, 44 and 29, 44    five 30, 47 and 30, 45    eight 42, 57 and 34, 46
//        x 1032  two 39, 49 and 38, 47    four 36, 56 and 40, 49    five 42, 62 and 42, 49    eight 60, 77 and 45, 51
//        x 2048  two 24, 42 and 25, 43    four 26, 43 and 28, 43    five 30, 45 and 29, 44    eight 41, 55 and 31, 45
//   fp32 x 512   two 46, 93 and 52, 107   four 45, 98 and 59, 106   five 43, 100 and 62, 105  eight 52, 114 and 69, 104
//        x 520   two 64, 99 and 65, 114   four 68, 111 and 71, 117  five 67, 116 and 73, 119  eight 72, 135 and 80, 126
//        x 1024  two 48, 84 and 52, 95    four 47, 90 and 56, 93    five 47, 92 and 58, 93    eight 50, 100 and 63, 94
// and 64 of 1024 in fp16 309 and 61.  More than four choices are patched, which fp32 would do without up to eight among
// themselves, and rows of more than two rounds, whose entries would be handed out as often: there the two are level but
// for a few sizes, 13 % for one and up to 25 % (fp16 x 1280, two among themselves: 21 and 27) for the other.  65536 x 1024
// fp16, four of all: 268 MB at 6 TB/s (the logits partly from the last-level cache).
template <class T, int kLanes, bool kAll, bool kStream, bool kPatched>
__global__ __launch_bounds__(kBlock) void choose_backward_kernel(ChooseBackwardArgs a, uint32_t first) {
    constexpr int kV = kPerVec<T>;
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    const int64_t at =
        (static_cast<int64_t>(first) + blockIdx.x) * (kBlock / kLanes) + static_cast<int>(threadIdx.x) / kLanes;
    const int64_t row = at < a.n ? at : a.n - 1;
    int own = -1;
    float weighted = 0.0f, weight = 0.0f;      // w_j g_j, w_j
    if (lane < a.choices) {
        own = a.expert[row * a.choices + lane];
        if (own >= 0 && own < a.experts) {
            weight = a.weights[row * a.choices + lane];
            weighted = weight * a.upstream[row * a.choices + lane];
        } else {
            own = -1;
        }
    }
    const float total = sum_across<kLanes>(weighted);
    const float result = fmaf(-weight, total, weighted);       // w_j is the entry's share in both kinds of weights
    float m = 0.0f, share = 0.0f;
    if constexpr (kAll) {
        m = base_of(a.stats[row * 2]);
        share = -total * a.stats[row * 2 + 1];
    }
    const bool empty = kAll && a.stats[row * 2 + 1] == 0.0f;   // a row of none; else 1 / s > 0 or NaN
    const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
    T* out = static_cast<T*>(a.dlogits) + row * a.experts;
    const int chunks = (a.experts + kV - 1) / kV;
    for (int c = 0; c < chunks; c += kLanes) {
        const int column = (c + lane) * kV;
        float value[kV] = {};
        if (kAll && !empty) {
            load_logits(logits, column, a.experts, value);
#pragma unroll
            for (int i = 0; i < kV; ++i) value[i] = share * exponential<sizeof(T) == 4>(value[i] - m);
        }
        if constexpr (!kPatched)
            for (int j = 0; j < a.choices; ++j) {
                const int e = __shfl(own, j, kLanes);
                const float whole = __shfl(result, j, kLanes);
                const int place = e < 0 ? -1 : e - column;
#pragma unroll
                for (int i = 0; i < kV; ++i) value[i] = place == i ? whole : value[i];
            }
        if (at < a.n && column < a.experts) store_some<kStream>(out + column, narrow<T>(value), a.experts - column);
    }
    if constexpr (kPatched) {
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");      // after the other lanes' stores
        float value = result;
        asm("" : "+v"(value));      // rounded to fp32, then to T, as its neighbours are
        if (at < a.n && own >= 0) out[own] = static_cast<T>(value);
    }
}

// --- balance -------------------------------------------------------------------------------------------

constexpr int kCountBlock = 1024;
constexpr int kSharedCounts = 1 << 14;   // experts whose counts a workgroup keeps in LDS
constexpr int64_t kFewEntries = 1 << 14; // counted by one workgroup, which needs nothing cleared before
constexpr uint32_t kFewBlocks = 256;     // of which the last one makes the loss

struct BalanceArgs {
    const void* logits;
    const int32_t* expert;    // [n][choices]
    int32_t* counts;          // [experts]
    uint32_t* entries;        // M
    uint32_t* done;           // workgroups that have left their sums, or null: a launch of its own makes the loss
    uint32_t blocks;          // workgroups of the rows
    float* stats;             // [n][4]: m, 1 / s (0: the row takes no part), t less `whole`, the whole number's bits
    double* partial;          // [blocks]: sum of t
    uint32_t* parts;          // [blocks]: rows that take part
    float* norm;              // E / (M R)
    float* loss;
    int64_t stride, n;
    int choices, experts;
};

__global__ __launch_bounds__(kBlock) void balance_clear_kernel(BalanceArgs a) {
    for (int e = blockIdx.x * kBlock + threadIdx.x; e < a.experts; e += gridDim.x * kBlock) a.counts[e] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *a.entries = 0;
        if (a.done) *a.done = 0;
    }
}

// Each workgroup counts its entries in LDS and adds what it found (whole numbers, in any order).  kAlone: one workgroup
// of all entries, which needs no launch that clears (16384 entries 4.1 us; 131072 by several 5.0, and 1.5 to clear).
// Entries that lie 16-byte aligned are read four at a time. 1.2 million entries of 1000 experts: 6 us (with 512
// workgroups, whose counts are half a million additions, 27).
template <bool kAlone> __global__ __launch_bounds__(kCountBlock) void balance_count_kernel(BalanceArgs a) {
    extern __shared__ int32_t held[];
    __shared__ uint32_t all;
    const bool shared = a.experts <= kSharedCounts;
    const int64_t entries = a.n * a.choices, step = static_cast<int64_t>(gridDim.x) * kCountBlock;
    const int64_t self = static_cast<int64_t>(blockIdx.x) * kCountBlock + threadIdx.x;
    int32_t* to = shared ? held : a.counts;
    if (threadIdx.x == 0) all = 0;
    if (shared) {
        for (int e = threadIdx.x; e < a.experts; e += kCountBlock) to[e] = 0;
        if (kAlone && a.done && threadIdx.x == 0) *a.done = 0;
    }
    __syncthreads();
    uint32_t found = 0;
    auto add = [&](int e) {
        if (e >= 0 && e < a.experts) atomicAdd(to + e, 1), ++found;
    };
    const int64_t fours = reinterpret_cast<uintptr_t>(a.expert) % 16 == 0 ? entries / 4 : 0;
    const int4* four = reinterpret_cast<const int4*>(a.expert);
#pragma unroll 2
    for (int64_t i = self; i < fours; i += step) {
        const int4 e = four[i];
        add(e.x), add(e.y), add(e.z), add(e.w);
    }
    for (int64_t i = 4 * fours + self; i < entries; i += step) add(a.expert[i]);
    found = sum_across<64>(found);
    if (threadIdx.x % 64 == 0) atomicAdd(&all, found);
    __syncthreads();
    if (threadIdx.x == 0) {
        if (kAlone) *a.entries = all;
        else atomicAdd(a.entries, all);
    }
    if (!shared) return;
    for (int e = threadIdx.x; e < a.experts; e += kCountBlock) {
        if (kAlone) a.counts[e] = held[e];
        else if (held[e]) atomicAdd(a.counts + e, held[e]);
    }
}

// The whole number next to M / E.
__device__ inline int32_t even_count(const BalanceArgs& a) {
    const uint32_t experts = static_cast<uint32_t>(a.experts);
    return static_cast<int32_t>((*a.entries + experts / 2) / experts);
}

// The counts of a lane's columns; past the last, the last.
template <class T, int kLanes, int kVecs>
__device__ inline void hold_counts(const int32_t* counts, int lane, int experts, int32_t (&to)[kVecs][kPerVec<T>]) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
        for (int i = 0; i < kPerVec<T>; ++i) {
            const int e = (v * kLanes + lane) * kPerVec<T> + i;
            to[v][i] = counts[e < experts ? e : experts - 1];
        }
}

// Whether a row has an entry among those of its lanes (of a wave's, where there are more): asked for ahead, one entry a
// lane, and told later.
template <int kLanes> struct Part {
    int32_t id;

    __device__ void load(const BalanceArgs& a, int64_t row, int lane) {
        id = a.expert[row * a.choices + (lane < a.choices ? lane : a.choices - 1)];
    }
    __device__ bool get(const BalanceArgs& a, int64_t row, int lane) const {
        uint32_t any = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.experts);
        for (int j = lane + kLanes; j < a.choices; j += kLanes)
            any |= static_cast<uint32_t>(a.expert[row * a.choices + j]) < static_cast<uint32_t>(a.experts);
        return across<(kLanes < 64 ? kLanes : 64)>(any, [](uint32_t x, uint32_t y) { return x | y; }) != 0;
    }
};

__device__ inline void keep_row(const BalanceArgs& a, int64_t row, float m, float inverse, float t, uint32_t whole) {
    if (a.stats)
        *reinterpret_cast<float4*>(a.stats + row * 4) =
            make_float4(m, inverse, t, as_float(whole));
}

// The sums of the workgroup's threads, in thread 0.
struct BalanceSums {
    double total;
    uint32_t rows;
};
__device__ inline BalanceSums sum_block(BalanceSums x) {
    __shared__ BalanceSums part[kBlock / 64];
    x = BalanceSums{sum_across<64>(x.total), sum_across<64>(x.rows)};
    __syncthreads();
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < kBlock / 64; ++w)
            x.total += part[w].total, x.rows += part[w].rows;
    return x;
}

// The loss from the workgroups' sums, in their order.
__device__ inline void make_loss(const BalanceArgs& a) {
    BalanceSums x{};
#pragma unroll 8
    for (uint32_t b = threadIdx.x; b < a.blocks; b += kBlock) {
        x.total += __hip_atomic_load(a.partial + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        x.rows += __hip_atomic_load(a.parts + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    x = sum_block(x);
    if (threadIdx.x != 0) return;
    const uint32_t entries = *a.entries;
    const double norm = entries > 0 ? a.experts / (static_cast<double>(entries) * static_cast<double>(x.rows)) : 0.0;
    *a.norm = static_cast<float>(norm);
    *a.loss = static_cast<float>(entries > 0 ? x.total * norm : 0.0);
}

// Leaves the workgroup's sums.  Of few workgroups the last one to come goes on to the loss, which saves a launch (3 us
// of host time); each of them takes its turn at one address, about 10 ns (65536 x 64: 1536 workgroups 25 us, with a
// launch of its own 8.4 and 3.4; 4096 x 64: 256 workgroups 7.0, and 3.8 and 1.8).
__device__ inline void finish_balance(const BalanceArgs& a, double total, uint32_t rows) {
    __shared__ bool last;
    const BalanceSums x = sum_block(BalanceSums{total, rows});
    if (threadIdx.x == 0) {
        __hip_atomic_store(a.partial + blockIdx.x, x.total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(a.parts + blockIdx.x, x.rows, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = false;
        if (a.done) {
            // Stores and loads of agent scope go past the XCD's own L2, so that their order is all it takes: a release
            // would write that L2 back, in every workgroup.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            last = __hip_atomic_fetch_add(a.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.blocks - 1;
        }
    }
    __syncthreads();
    if (last) make_loss(a);
}

__global__ __launch_bounds__(kBlock) void balance_loss_kernel(BalanceArgs a) { make_loss(a); }

// Two numbers of each wave of a workgroup, to all of its threads by LDS; `turn` as for best_of.
template <class F>
__device__ inline void over_waves(float2 own, float2 (&part)[2][kBlock / 64], int& turn, F&& f) {
    turn ^= 1;
    if (threadIdx.x % 64 == 0) part[turn][threadIdx.x / 64] = own;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBlock / 64; ++w) f(part[turn][w]);
}

// Rows of up to kLanes kVecs chunks: kLanes lanes a row, a row in registers and the next one under way, the counts of
// the lane's columns, less M / E, in registers for all of its rows.  A first sum gives a row's t and with it the whole
// number that comes off for a second one, which costs 4 to 11 % (300007 x 1000 bf16: 136 to 154 us).  300007 x 1000 bf16:
// 150 to 164 us, 600 MB at 3.7 to 4 TB/s (with the counts read for each row and one sum 524 us; with loads under
// conditions, which the compiler waits for, 214); 8192 x 8000 43 us (a wave a row and one sum 122).
template <class T, int kLanes, int kVecs> __global__ __launch_bounds__(kBlock) void balance_rows_kernel(BalanceArgs a) {
    constexpr bool kExact = sizeof(T) == 4;
    constexpr int kV = kPerVec<T>, kRows = kBlock / kLanes;
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    const int32_t even = even_count(a);
    int32_t held_counts[kVecs][kV];
    hold_counts<T, kLanes, kVecs>(a.counts, lane, a.experts, held_counts);
    float counts[kVecs][kV];
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
        for (int i = 0; i < kV; ++i) counts[v][i] = static_cast<float>(held_counts[v][i] - even);
    const T* logits = static_cast<const T*>(a.logits);
    double total = 0.0;
    uint32_t rows = 0;
    constexpr int kTogether = kLanes < 64 ? kLanes : 64;
    __shared__ float2 held[2][kBlock / 64];
    int turn = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int64_t at = static_cast<int64_t>(blockIdx.x) * kRows + static_cast<int>(threadIdx.x) / kLanes;
    RowHold<T, kLanes, kVecs> next;
    Part<kLanes> part_next;
    if (a.n > 0) {      // without rows there is none to load ahead
        next.load(logits + (at < a.n ? at : a.n - 1) * a.stride, lane, a.experts);
        part_next.load(a, at < a.n ? at : a.n - 1, lane);
    }
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.n; base += step, at += step) {
        RowHold<T, kLanes, kVecs> row = next;
        const Part<kLanes> part = part_next;
        const int64_t now = at < a.n ? at : a.n - 1, then = at + step < a.n ? at + step : a.n - 1;
        next.load(logits + then * a.stride, lane, a.experts);
        part_next.load(a, then, lane);
        bool any = part.get(a, now, lane);
        row.settle(lane, a.experts);
        float value[kVecs][kV], top = kNegInfinity;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            row.get(v, lane, a.experts, value[v]);
#pragma unroll
            for (int i = 0; i < kV; ++i) top = larger(top, value[v][i]);
        }
        top = max_across<kTogether>(top);
        if constexpr (kLanes > 64)
            over_waves(make_float2(top, any ? 1.0f : 0.0f), held, turn, [&](const float2& x) {
                top = larger(top, x.x);
                any |= x.y != 0.0f;
            });
        const float from = base_of(top);
        float s = 0.0f, t = 0.0f;
#pragma unroll
        for (int v = 0; v < kVecs; ++v)
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                const float e = exponential<kExact>(value[v][i] - from);
                value[v][i] = e;
                s += e;
                t = fmaf(e, counts[v][i], t);
            }
        s = sum_across<kTogether>(s);
        t = sum_across<kTogether>(t);
        if constexpr (kLanes > 64) {
            const float2 own = make_float2(s, t);
            s = t = 0.0f;
            over_waves(own, held, turn, [&](const float2& x) { s += x.x, t += x.y; });
        }
        const float inverse = any && !(top == kNegInfinity) ? 1.0f / s : 0.0f;
        const float near = inverse == 0.0f || !(inverse < INFINITY) ? 0.0f : rintf(t * inverse);    // NaN: 0
        t = 0.0f;
#pragma unroll
        for (int v = 0; v < kVecs; ++v)
#pragma unroll
            for (int i = 0; i < kV; ++i) t = fmaf(value[v][i], counts[v][i] - near, t);
        t = sum_across<kTogether>(t);
        if constexpr (kLanes > 64) {
            const float2 own = make_float2(t, 0.0f);
            t = 0.0f;
            over_waves(own, held, turn, [&](const float2& x) { t += x.x; });
        }
        t = inverse == 0.0f ? 0.0f : t * inverse;
        if (at < a.n && lane == 0) {
            total += inverse == 0.0f ? 0.0 : static_cast<double>(even) + near + t;
            rows += any;
            keep_row(a, at, top, inverse, t,
                     static_cast<uint32_t>(even) + static_cast<uint32_t>(static_cast<int32_t>(near)));
        }
    }
    finish_balance(a, total, rows);
}

// The counts of a chunk's columns; 0 past the last.
template <int kV>
__device__ inline void load_counts(const int32_t* counts, int column, int experts, int32_t (&to)[kV]) {
    if (column + kV <= experts) {
#pragma unroll
        for (int w = 0; w < kV / 4; ++w) {
            const vec16 four = load16(counts + column + 4 * w);
#pragma unroll
            for (int i = 0; i < 4; ++i) to[4 * w + i] = static_cast<int32_t>(four[i]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kV; ++i) to[i] = column + i < experts ? counts[column + i] : 0;
}

// Longer rows: a wave a row, with a running maximum.  They are not held for a second sum: one takes M / E off, another
// nothing, and the row keeps the one that is off by less, the second where t is below half of M / E.  8192 x 32000 bf16:
// 145 us forward and 228 backward.
template <class T> __global__ __launch_bounds__(kBlock) void balance_long_kernel(BalanceArgs a) {
    constexpr bool kExact = sizeof(T) == 4;
    constexpr int kV = kPerVec<T>;
    const int lane = static_cast<int>(threadIdx.x) % 64;
    const int32_t even = even_count(a);
    double total = 0.0;
    uint32_t rows = 0;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / 64) + static_cast<int>(threadIdx.x) / 64; row < a.n;
         row += static_cast<int64_t>(gridDim.x) * (kBlock / 64)) {
        Part<64> part;
        part.load(a, row, lane);
        const bool any = part.get(a, row, lane);
        const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
        float m = kNegInfinity, s = 0.0f, t = 0.0f, all = 0.0f;
        for (int column = lane * kV; column < a.experts; column += 64 * kV) {
            float value[kV];
            int32_t counts[kV];
            load_logits(logits, column, a.experts, value);
            load_counts(a.counts, column, a.experts, counts);
            float top = m;
#pragma unroll
            for (int i = 0; i < kV; ++i) top = larger(top, value[i]);
            const float base = base_of(top), old = exponential<kExact>(m - base);
            s *= old;
            t *= old;
            all *= old;
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                const float e = exponential<kExact>(value[i] - base);
                s += e;
                t = fmaf(e, static_cast<float>(counts[i] - even), t);
                all = fmaf(e, static_cast<float>(counts[i]), all);
            }
            m = top;
        }
        const float top = max_across<64>(m), old = exponential<kExact>(m - base_of(top));
        s = sum_across<64>(s * old);
        t = sum_across<64>(t * old);
        all = sum_across<64>(all * old);
        const float inverse = any && !(top == kNegInfinity) ? 1.0f / s : 0.0f;
        const bool few = all * inverse < 0.5f * static_cast<float>(even);
        t = inverse == 0.0f ? 0.0f : (few ? all : t) * inverse;
        if (lane == 0) {
            const int32_t whole = few ? 0 : even;
            total += inverse == 0.0f ? 0.0 : static_cast<double>(whole) + t;
            rows += any;
            keep_row(a, row, top, inverse, t, static_cast<uint32_t>(whole));
        }
    }
    finish_balance(a, total, rows);
}

struct BalanceBackwardArgs {
    const float* upstream;    // one value
    const void* logits;
    const int32_t* counts;
    const float* stats;
    const float* norm;
    void* dlogits;            // [n][experts]
    int64_t stride, n;
    int experts;
};

// c_e - t of a row: its whole number comes off first, exactly.
__device__ inline float count_less_mean(int32_t count, const float4& stats) {
    return static_cast<float>(static_cast<int32_t>(static_cast<uint32_t>(count) - as_bits(stats.w))) - stats.z;
}

// The same way.  300007 x 1000 bf16: 255 us, 1.2 GB at 4.7 TB/s: HBM.
template <class T, int kLanes, int kVecs, bool kStream>
__global__ __launch_bounds__(kBlock) void balance_backward_kernel(BalanceBackwardArgs a) {
    constexpr int kV = kPerVec<T>, kRows = kBlock / kLanes;
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    int32_t counts[kVecs][kV];
    hold_counts<T, kLanes, kVecs>(a.counts, lane, a.experts, counts);
    const float scale = *a.upstream * *a.norm;
    const T* logits = static_cast<const T*>(a.logits);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int64_t at = static_cast<int64_t>(blockIdx.x) * kRows + static_cast<int>(threadIdx.x) / kLanes;
    if (at >= a.n) return;
    RowHold<T, kLanes, kVecs> next;
    next.load(logits + at * a.stride, lane, a.experts);
    float4 stats_next = *reinterpret_cast<const float4*>(a.stats + at * 4);
    for (; at < a.n; at += step) {
        RowHold<T, kLanes, kVecs> row = next;
        const float4 stats = stats_next;
        const int64_t then = at + step < a.n ? at + step : a.n - 1;
        next.load(logits + then * a.stride, lane, a.experts);
        stats_next = *reinterpret_cast<const float4*>(a.stats + then * 4);
        row.settle(lane, a.experts);
        const float each = scale * stats.y;
        T* out = static_cast<T*>(a.dlogits) + at * a.experts;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const int column = (v * kLanes + lane) * kV;
            float value[kV];
            row.get(v, lane, a.experts, value);
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                const float d =
                    each * exponential<sizeof(T) == 4>(value[i] - stats.x) * count_less_mean(counts[v][i], stats);
                value[i] = stats.y == 0.0f ? 0.0f : d;
            }
            if (column < a.experts) store_some<kStream>(out + column, narrow<T>(value), a.experts - column);
        }
    }
}

template <class T, bool kStream>
__global__ __launch_bounds__(kBlock) void balance_long_backward_kernel(BalanceBackwardArgs a) {
    constexpr int kV = kPerVec<T>;
    const int lane = static_cast<int>(threadIdx.x) % 64;
    const float scale = *a.upstream * *a.norm;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / 64) + static_cast<int>(threadIdx.x) / 64; row < a.n;
         row += static_cast<int64_t>(gridDim.x) * (kBlock / 64)) {
        const float4 stats = *reinterpret_cast<const float4*>(a.stats + row * 4);
        const float each = scale * stats.y;
        const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
        T* out = static_cast<T*>(a.dlogits) + row * a.experts;
        for (int column = lane * kV; column < a.experts; column += 64 * kV) {
            float value[kV];
            int32_t counts[kV];
            load_logits(logits, column, a.experts, value);
            load_counts(a.counts, column, a.experts, counts);
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                const float d =
                    each * exponential<sizeof(T) == 4>(value[i] - stats.x) * count_less_mean(counts[i], stats);
                value[i] = stats.y == 0.0f ? 0.0f : d;
            }
            store_some<kStream>(out + column, narrow<T>(value), a.experts - column);
        }
    }
}

template <int kNumber> using Number = std::integral_constant<int, kNumber>;

// Calls f with the lanes a row of `width` values takes: 8 to 64, and at least `least`.
template <class T, class F> void with_lanes(int width, int least, F&& f) {
    const int chunks = (width + kPerVec<T> - 1) / kPerVec<T>, wanted = chunks > least ? chunks : least;
    if (wanted <= 8) f(std::integral_constant<int, 8>{});
    else if (wanted <= 16) f(std::integral_constant<int, 16>{});
    else if (wanted <= 32) f(std::integral_constant<int, 32>{});
    else f(std::integral_constant<int, 64>{});
}

int check_rows_of(const std::string& what, int64_t stride, int64_t n, int choices, int experts, int dtype) {
    if (!known_dtype(dtype)) return fail(what + ": dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (experts < 1 || experts > kMaxExperts) return fail(what + ": experts must be within 1..32768");
    if (choices < 1) return fail(what + ": choices must be at least 1");
    if (n < 0 || n > kMaxEntries / choices) return fail(what + ": rows times choices must be within 0..2^31 - 1");
    if (n > 0 && stride < experts) return fail(what + ": rows overlap (a stride below the row's width)");
    return 0;
}

// Lanes and 16-byte chunks a lane that hold a row; 0 chunks: longer rows.
template <class T, class F> void with_row(int width, int least, F&& f) {
    const int chunks = (width + kPerVec<T> - 1) / kPerVec<T>;
    if (chunks <= 64) with_lanes<T>(width, least, [&](auto lanes) { f(lanes, std::integral_constant<int, 1>{}); });
    else if (chunks <= 128) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (chunks <= 256) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    else if (chunks <= 512) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
    else if (chunks <= 1024) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else if (chunks <= 2048) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
    else f(std::integral_constant<int, 64>{}, std::integral_constant<int, 0>{});
}

// Workgroups of the passes over rows, `lanes` lanes a row: as many as the CUs hold together by their registers, so that
// all of them run to the end: two each with 8 chunks a lane, four with 4, six with fewer (65536 x 1024 fp16, choice:
// 52.5 us with four, 50 with six, 49 with eight; 300007 x 1000 bf16, balance: 170, 160, 158).  Passes that also write a
// row lose by more than four (its gradient: 243, 251, 262).
uint32_t row_blocks(int64_t n, int lanes, int vecs, bool writes = false) {
    const int rows = lanes > kBlock ? 1 : kBlock / lanes;
    const int64_t blocks = (n + rows - 1) / rows;
    const int64_t most = (vecs == 8 ? 2 : (vecs == 4 || writes ? 4 : 6)) * kCus;
    return static_cast<uint32_t>(blocks < 1 ? 1 : (blocks < most ? blocks : most));
}

// The most workgroups that any width takes: a row each, six a CU.
int64_t most_row_blocks(int64_t n) { return row_blocks(n, kBlock, 1); }

// Whether a choice reads its fp32 rows once for each of the choices, instead of once in all.  us in registers and by
// turns: 8192 x 4000, one choice 37 and 25, two 43 and 41, four 52 and 73; 8192 x 8000, four 165 and 143; 8192 x 16000,
// one 173 and 100, four 304 and 294, eight 476 and 580; 1000 x 8000, four 24 and 26; one row of 8000 6.5 and 16.
bool by_turns(int64_t n, int chunks, int choices) {
    return chunks > 4096 || (n >= 4 * kCus && chunks > 512 && choices <= (chunks > 1024 ? 4 : 1));
}
static_assert(kMaxExperts <= 4096 * kPerVec<_Float16>, "16-bit rows stay in registers");

}  // namespace
}  // namespace odie

using namespace odie;

ODIE_API int odie_choose_forward(const void* logits, int64_t stride, int64_t n, int experts, int choices, int normalize,
                                 int dtype, int32_t* expert, float* weights, float* stats, uint64_t stream) {
    const std::string what = "odie_choose_forward";
    if (check_rows_of(what, stride, n, choices, experts, dtype)) return -1;
    if (choices > kMaxChoices || choices > experts)
        return fail(what + ": choices must be within 1..64 and the experts");
    if (n == 0) return 0;
    if (!logits || !expert || !weights) return fail(what + ": null pointer");
    if (reinterpret_cast<uintptr_t>(stats) % 8) return fail(what + ": stats must be 8-byte aligned");
    ChooseArgs a{logits, stride, n, expert, weights, stats, experts, choices, normalize};
    const hipStream_t s = as_stream(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const int chunks = (experts + kPerVec<T> - 1) / kPerVec<T>;
        if constexpr (sizeof(T) == 4)
            if (by_turns(n, chunks, choices)) {
                choose_long_kernel<<<static_cast<uint32_t>(n < 16 * kCus ? n : 16 * kCus), kBlock, 0, s>>>(a);
                return check_launch("choose");
            }
        const auto launch = [&](auto lanes, auto vecs) {
            constexpr int kThreads = lanes > kBlock ? lanes : kBlock;
            choose_kernel<T, lanes, vecs><<<row_blocks(n, lanes, vecs), kThreads, 0, s>>>(a);
        };
        if (chunks <= 64) with_lanes<T>(experts, choices, [&](auto lanes) { launch(lanes, Number<1>{}); });
        else if (chunks <= 128) launch(Number<64>{}, Number<2>{});
        else if (chunks <= 256) launch(Number<64>{}, Number<4>{});
        else if (chunks <= 512) launch(Number<256>{}, Number<2>{});
        else if (chunks <= 1024) launch(Number<256>{}, Number<4>{});
        else if (chunks <= 2048) launch(Number<512>{}, Number<4>{});
        else launch(Number<1024>{}, Number<4>{});
        return check_launch("choose");
    });
}

ODIE_API int odie_choose_backward(const float* upstream, const int32_t* expert, const float* weights,
                                  const void* logits, int64_t stride, const float* stats, int64_t n, int experts,
                                  int choices, int dtype, void* dlogits, uint64_t stream) {
    const std::string what = "odie_choose_backward";
    if (check_rows_of(what, logits ? stride : experts, n, choices, experts, dtype)) return -1;
    if (choices > kMaxChoices || choices > experts)
        return fail(what + ": choices must be within 1..64 and the experts");
    if (n == 0) return 0;
    if (!upstream || !expert || !weights || !dlogits || (logits && !stats)) return fail(what + ": null pointer");
    ChooseBackwardArgs a{upstream, expert, weights, logits, stats, dlogits, stride, n, experts, choices};
    const hipStream_t s = as_stream(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        with_lanes<T>(experts, choices, [&](auto lanes) {
            with_flag(logits != nullptr, [&](auto all) {
                with_flag(n * experts * dtype_bytes(dtype) >= kStreamBytes, [&](auto far) {
                    with_flag(choices > 4 || experts > 2 * lanes * kPerVec<T>, [&](auto patched) {
                        in_launches((n + kBlock / lanes - 1) / (kBlock / lanes), kBlock,
                                    [&](uint32_t first, uint32_t count) {
                            choose_backward_kernel<T, lanes, all, far, patched><<<count, kBlock, 0, s>>>(a, first);
                        });
                    });
                });
            });
        });
        return check_launch("choose gradient");
    });
}

ODIE_API int64_t odie_balance_workspace(int64_t n, int choices, int experts) {
    if (check_rows_of("odie_balance_workspace", experts, n, choices, experts, ODIE_F32)) return -1;
    return 12 * most_row_blocks(n) + 8;      // sums of t, rows, entries, workgroups that are done
}

ODIE_API int odie_balance_forward(const void* logits, int64_t stride, const int32_t* expert, int64_t n, int choices,
                                  int experts, int dtype, float* loss, int32_t* counts, float* stats, float* norm,
                                  void* workspace, int64_t workspace_bytes, uint64_t stream) {
    const std::string what = "odie_balance_forward";
    if (check_rows_of(what, stride, n, choices, experts, dtype)) return -1;
    if (!loss || !counts || !norm || (n > 0 && (!logits || !expert))) return fail(what + ": null pointer");
    if (reinterpret_cast<uintptr_t>(stats) % 16) return fail(what + ": stats must be 16-byte aligned");
    const int64_t need = odie_balance_workspace(n, choices, experts);
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8 != 0)
        return fail(what + ": needs an 8-byte aligned workspace of " + std::to_string(need) + " bytes");
    const int64_t most = most_row_blocks(n);
    BalanceArgs a{};
    a.logits = logits;
    a.expert = expert;
    a.counts = counts;
    a.stats = stats;
    a.partial = static_cast<double*>(workspace);
    a.parts = reinterpret_cast<uint32_t*>(a.partial + most);
    with_dtype(dtype, [&](auto t) {
        with_row<decltype(t)>(experts, 1, [&](auto lanes, auto vecs) { a.blocks = row_blocks(n, lanes, vecs); });
    });
    a.entries = a.parts + most;
    a.done = a.blocks <= kFewBlocks ? a.entries + 1 : nullptr;
    a.norm = norm;
    a.loss = loss;
    a.stride = stride;
    a.n = n;
    a.choices = choices;
    a.experts = experts;
    const hipStream_t s = as_stream(stream);
    const int64_t entries = n * choices;
    const int shared = experts <= kSharedCounts ? experts * 4 : 0;
    if (entries <= kFewEntries && experts <= kSharedCounts) {
        balance_count_kernel<true><<<1, kCountBlock, shared, s>>>(a);
    } else {
        // Sixteen entries a thread at least, and two for each count that a workgroup adds at its end.
        const int64_t each = 16 * kCountBlock > 2 * experts ? 16 * kCountBlock : 2 * experts;
        const int64_t blocks = (entries + each - 1) / each;
        balance_clear_kernel<<<(experts + kBlock - 1) / kBlock, kBlock, 0, s>>>(a);
        if (entries > 0)      // none: the counts are cleared, and a launch of no workgroups is an error
            balance_count_kernel<false>
                <<<static_cast<uint32_t>(blocks < kCus ? blocks : kCus), kCountBlock, shared, s>>>(a);
    }
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        with_row<T>(experts, 1, [&](auto lanes, auto vecs) {
            if constexpr (vecs > 0) balance_rows_kernel<T, lanes, vecs><<<a.blocks, kBlock, 0, s>>>(a);
            else balance_long_kernel<T><<<a.blocks, kBlock, 0, s>>>(a);
        });
    });
    if (!a.done) balance_loss_kernel<<<1, kBlock, 0, s>>>(a);
    return check_launch("balance");
}

ODIE_API int odie_balance_backward(const float* upstream, const void* logits, int64_t stride, const int32_t* counts,
                                   const float* stats, const float* norm, int64_t n, int experts, int dtype,
                                   void* dlogits, uint64_t stream) {
    const std::string what = "odie_balance_backward";
    if (check_rows_of(what, stride, n, 1, experts, dtype)) return -1;
    if (n == 0) return 0;
    if (!upstream || !logits || !counts || !stats || !norm || !dlogits) return fail(what + ": null pointer");
    if (reinterpret_cast<uintptr_t>(stats) % 16) return fail(what + ": stats must be 16-byte aligned");
    BalanceBackwardArgs a{upstream, logits, counts, stats, norm, dlogits, stride, n, experts};
    const hipStream_t s = as_stream(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        with_flag(n * experts * dtype_bytes(dtype) >= kStreamBytes, [&](auto far) {
            with_row<T>(experts, 1, [&](auto lanes, auto vecs) {
                if constexpr (vecs > 0)
                    balance_backward_kernel<T, lanes, vecs, far>
                        <<<row_blocks(n, lanes, vecs, true), kBlock, 0, s>>>(a);
                else balance_long_backward_kernel<T, far><<<row_blocks(n, 64, 1, true), kBlock, 0, s>>>(a);
            });
        });
        return check_launch("balance gradient");
    });
}
