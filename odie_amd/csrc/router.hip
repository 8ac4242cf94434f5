// A learned router over experts: the choice of each row's experts with their softmax weights, and the loss that
// keeps their load even, with their gradients.
//
//   choose   e_1 .. e_k: the row's largest logits, the lowest index first among equal ones; w_j = exp(l_ej - m) / s, s over
//            the chosen (normalised) or over all experts
//            dl_e = [e = e_j] w_j g_j - q_e sum_i w_i g_i, q the softmax over the chosen or over all
//   balance  c_e entries of expert e, M in all; R rows that have an entry; t_i = sum_e c_e p_ie over row i's softmax
//            loss = E / (M R) sum_i t_i,  dl_ie = g E / (M R) p_ie (c_e - t_i)
//
// The loss is E sum_e (c_e / M) (mean over rows of p_ie) with its sums exchanged: each row needs its own
// logits and the counts alone, and no sums down the columns exist.  Counts are whole numbers, and everything else
// is added in a fixed order: the same call gives the same bits.
#include "softmax.h"

namespace odie {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxExperts = 1 << 15;
constexpr int kMaxChoices = 64;
constexpr int64_t kMaxEntries = (int64_t{1} << 31) - 1;

// Whole numbers in the order of the values, above 0 but for -inf: -0 and 0 alike, every NaN above +inf.
__device__ inline uint32_t order_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t bits = as_bits(x + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ inline float value_of(uint32_t order) {
    if (order == 0xffffffffu) return as_float(0x7fc00000u);
    return as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
template <class T> __device__ inline uint32_t order16(float x) {   // x a value of T
    if (x != x) return 0xffffu;
    const uint32_t bits = __builtin_bit_cast(uint16_t, static_cast<T>(x + 0.0f));
    return bits & 0x8000u ? bits ^ 0xffffu : bits | 0x8000u;
}
template <class T> __device__ inline float value16(uint32_t order) {
    if (order == 0xffffu) return as_float(0x7fc00000u);
    return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(order & 0x8000u ? order & 0x7fffu : order ^ 0xffffu)));
}

// A logit above -inf with its index as one whole number above 0: the larger the logit and, among equal ones, the lower
// the index, the larger the key.  A 16-bit logit and its index fit 32 bits.
template <class T> struct Keys {
    using Key = uint32_t;
    static __device__ Key of(float value, int index) { return order16<T>(value) << 16 | static_cast<uint32_t>(0xffff - index); }
    static __device__ int index(Key key) { return 0xffff - static_cast<int>(key & 0xffffu); }
    static __device__ float value(Key key) { return value16<T>(key >> 16); }
    template <int kLanes> static __device__ Key best(Key key) {
        return across<kLanes>(key, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    }
};
template <> struct Keys<float> {
    using Key = uint64_t;
    static __device__ Key of(float value, int index) { return static_cast<uint64_t>(order_of(value)) << 32 | static_cast<uint32_t>(~index); }
    static __device__ int index(Key key) { return static_cast<int>(~static_cast<uint32_t>(key)); }
    static __device__ float value(Key key) { return value_of(static_cast<uint32_t>(key >> 32)); }
    template <int kLanes> static __device__ Key best(Key key) {
        // the largest order first, then the largest rest among the lanes that hold it
        const auto most = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
        const uint32_t order = static_cast<uint32_t>(key >> 32), top = across<kLanes>(order, most);
        const uint32_t rest = across<kLanes>(order == top ? static_cast<uint32_t>(key) : 0u, most);
        return static_cast<uint64_t>(top) << 32 | rest;
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

// Rows of up to 64 kVecs 16-byte chunks in registers, kLanes lanes and kVecs chunks a lane.
template <class T, int kLanes, int kVecs>
__global__ __launch_bounds__(kBlock) void choose_kernel(ChooseArgs a, uint32_t first_block) {
    using K = Keys<T>;
    using Key = typename K::Key;
    constexpr int kV = kPerVec<T>, kValues = kVecs * kV;
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    const int64_t at = (static_cast<int64_t>(first_block) + blockIdx.x) * (kBlock / kLanes) + static_cast<int>(threadIdx.x) / kLanes;
    const int64_t row = at < a.n ? at : a.n - 1;
    const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
    float value[kVecs][kV];
    Key key[kValues], local = 0;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) load_logits(logits, (v * kLanes + lane) * kV, a.experts, value[v]);
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            const int index = (v * kLanes + lane) * kV + i;
            key[v * kV + i] = value[v][i] == kNegInfinity ? 0 : K::of(value[v][i], index);
            local = key[v * kV + i] > local ? key[v * kV + i] : local;
        }
    Key mine = 0, first = 0;      // lane j: the j-th choice
    for (int j = 0; j < a.choices; ++j) {
        const Key best = K::template best<kLanes>(local);
        if (j == 0) first = best;
        if (lane == j) mine = best;
        local = 0;
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            key[i] = key[i] == best ? 0 : key[i];
            local = key[i] > local ? key[i] : local;
        }
    }
    const float m = first ? K::value(first) : kNegInfinity, base = base_of(m);
    const float own = mine ? expf(K::value(mine) - base) : 0.0f;
    float s;
    if (a.normalize) {
        s = sum_across<kLanes>(own);
    } else {
        s = 0.0f;
#pragma unroll
        for (int v = 0; v < kVecs; ++v)
#pragma unroll
            for (int i = 0; i < kV; ++i) s += exponential<sizeof(T) == 4>(value[v][i] - base);
        s = sum_across<kLanes>(s);
    }
    const float inverse = first ? 1.0f / s : 0.0f;
    if (at >= a.n) return;
    if (lane < a.choices) {
        a.expert[row * a.choices + lane] = mine ? K::index(mine) : -1;
        a.weights[row * a.choices + lane] = mine ? own * inverse : 0.0f;
    }
    if (a.stats && lane == 0) {
        a.stats[row * 2] = m;
        a.stats[row * 2 + 1] = inverse;
    }
}

// The largest key of the workgroup, for every thread; `part` holds a key a wave.
__device__ inline uint64_t block_best(uint64_t key, uint64_t* part) {
    key = Keys<float>::best<64>(key);
    __syncthreads();
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = key;
    __syncthreads();
    for (int w = 0; w < kBlock / 64; ++w) key = part[w] > key ? part[w] : key;
    return key;
}

// Longer rows: a workgroup a row, which it reads once for each choice, the one below the last.
template <class T> __global__ __launch_bounds__(kBlock) void choose_long_kernel(ChooseArgs a) {
    using K = Keys<float>;
    constexpr int kV = kPerVec<T>;
    __shared__ uint64_t part[kBlock / 64];
    __shared__ float sums[kBlock / 64];
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
        const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
        uint64_t mine = 0, first = 0, last = ~uint64_t{0};
        for (int j = 0; j < a.choices; ++j) {
            uint64_t local = 0;
            for (int column = static_cast<int>(threadIdx.x) * kV; column < a.experts; column += kBlock * kV) {
                float value[kV];
                load_logits(logits, column, a.experts, value);
#pragma unroll
                for (int i = 0; i < kV; ++i) {
                    const uint64_t key = value[i] == kNegInfinity ? 0 : K::of(value[i], column + i);
                    if (key < last && key > local) local = key;
                }
            }
            last = block_best(local, part);
            if (j == 0) first = last;
            if (static_cast<int>(threadIdx.x) == j) mine = last;
        }
        const float m = first ? K::value(first) : kNegInfinity, base = base_of(m);
        const float own = mine ? expf(K::value(mine) - base) : 0.0f;
        float s = own;
        if (!a.normalize) {
            s = 0.0f;
            for (int column = static_cast<int>(threadIdx.x) * kV; column < a.experts; column += kBlock * kV) {
                float value[kV];
                load_logits(logits, column, a.experts, value);
#pragma unroll
                for (int i = 0; i < kV; ++i) s += exponential<sizeof(T) == 4>(value[i] - base);
            }
        }
        s = sum_across<64>(s);
        __syncthreads();
        if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = s;
        __syncthreads();
        s = 0.0f;
        for (int w = 0; w < kBlock / 64; ++w) s += sums[w];
        const float inverse = first ? 1.0f / s : 0.0f;
        if (static_cast<int>(threadIdx.x) < a.choices) {
            a.expert[row * a.choices + threadIdx.x] = mine ? K::index(mine) : -1;
            a.weights[row * a.choices + threadIdx.x] = mine ? own * inverse : 0.0f;
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

// kLanes lanes a row write its gradient chunk by chunk; each lane holds one of the row's entries.
template <class T, int kLanes, bool kAll, bool kStream>
__global__ __launch_bounds__(kBlock) void choose_backward_kernel(ChooseBackwardArgs a, uint32_t first) {
    constexpr int kV = kPerVec<T>;
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    const int64_t at = (static_cast<int64_t>(first) + blockIdx.x) * (kBlock / kLanes) + static_cast<int>(threadIdx.x) / kLanes;
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
    float m = 0.0f, share = 0.0f;
    if constexpr (kAll) {
        m = base_of(a.stats[row * 2]);
        share = -total * a.stats[row * 2 + 1];
    } else {
        weighted = fmaf(-weight, total, weighted);
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
        for (int j = 0; j < a.choices; ++j) {
            const int e = __shfl(own, j, kLanes);
            const float add = __shfl(weighted, j, kLanes);
            const int place = e < 0 ? -1 : e - column;
#pragma unroll
            for (int i = 0; i < kV; ++i) value[i] += place == i ? add : 0.0f;
        }
        if (at < a.n && column < a.experts) store_some<kStream>(out + column, narrow<T>(value), a.experts - column);
    }
}

// --- balance -------------------------------------------------------------------------------------------

constexpr int kCountBlocks = 2 * kCus;
constexpr int kSharedCounts = 8192;      // experts whose counts a workgroup keeps in LDS

struct BalanceArgs {
    const void* logits;
    const int32_t* expert;    // [n][choices]
    int32_t* counts;          // [experts]
    int32_t* rows;            // R
    float* stats;             // [n][3]: m, 1 / s (0: the row takes no part), t
    double* partial;          // [blocks]
    float* norm;              // E / (M R)
    float* loss;
    int64_t stride, n, blocks;
    int choices, experts;
};

__global__ __launch_bounds__(kBlock) void balance_clear_kernel(BalanceArgs a) {
    for (int e = blockIdx.x * kBlock + threadIdx.x; e < a.experts; e += gridDim.x * kBlock) a.counts[e] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.rows = 0;
}

__global__ __launch_bounds__(kBlock) void balance_count_kernel(BalanceArgs a) {
    extern __shared__ int32_t held[];
    const bool shared = a.experts <= kSharedCounts;
    int32_t* to = shared ? held : a.counts;
    if (shared) {
        for (int e = threadIdx.x; e < a.experts; e += kBlock) held[e] = 0;
        __syncthreads();
    }
    int32_t rows = 0;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; row < a.n; row += static_cast<int64_t>(gridDim.x) * kBlock) {
        bool any = false;
        for (int j = 0; j < a.choices; ++j) {
            const int e = a.expert[row * a.choices + j];
            if (e < 0 || e >= a.experts) continue;
            any = true;
            atomicAdd(to + e, 1);
        }
        rows += any;
    }
    for (int step = 32; step > 0; step /= 2) rows += __shfl_down(rows, step);
    if (threadIdx.x % 64 == 0 && rows) atomicAdd(a.rows, rows);
    if (!shared) return;
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kBlock)
        if (held[e]) atomicAdd(a.counts + e, held[e]);
}

template <class T, int kLanes> __global__ __launch_bounds__(kBlock) void balance_rows_kernel(BalanceArgs a) {
    constexpr bool kExact = sizeof(T) == 4;
    constexpr int kV = kPerVec<T>;
    __shared__ double sums[kBlock / 64];
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    double total = 0.0;
    for (int64_t base_row = static_cast<int64_t>(blockIdx.x) * (kBlock / kLanes); base_row < a.n;
         base_row += static_cast<int64_t>(gridDim.x) * (kBlock / kLanes)) {
        const int64_t at = base_row + static_cast<int>(threadIdx.x) / kLanes, row = at < a.n ? at : a.n - 1;
        uint32_t any = 0;
        for (int j = lane; j < a.choices; j += kLanes) {
            const int e = a.expert[row * a.choices + j];
            any |= e >= 0 && e < a.experts;
        }
        any = across<kLanes>(any, [](uint32_t x, uint32_t y) { return x | y; });
        const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
        Running<kExact> run;
        float t = 0.0f;
        for (int column = lane * kV; column < a.experts; column += kLanes * kV) {
            float value[kV];
            load_logits(logits, column, a.experts, value);
            float top = value[0];
#pragma unroll
            for (int i = 1; i < kV; ++i) top = larger(top, value[i]);
            top = larger(run.m, top);
            const float base = base_of(top);
            float s = 0.0f, more = 0.0f;
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                const float e = exponential<kExact>(value[i] - base);
                s += e;
                if (column + i < a.experts) more = fmaf(e, static_cast<float>(a.counts[column + i]), more);
            }
            const float old = exponential<kExact>(run.m - base);
            run.s = fmaf(run.s, old, s);
            t = fmaf(t, old, more);
            run.m = top;
        }
        const float top = max_across<kLanes>(run.m), old = exponential<kExact>(run.m - base_of(top));
        const float s = sum_across<kLanes>(run.s * old);
        t = sum_across<kLanes>(t * old);
        const bool part = any && !(top == kNegInfinity);
        const float inverse = part ? 1.0f / s : 0.0f;
        t = part ? t * inverse : 0.0f;
        if (at < a.n && lane == 0) {
            total += static_cast<double>(t);
            if (a.stats) {
                a.stats[row * 3] = top;
                a.stats[row * 3 + 1] = inverse;
                a.stats[row * 3 + 2] = t;
            }
        }
    }
    for (int step = 32; step > 0; step /= 2) total += __shfl_down(total, step);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kBlock / 64; ++w) total += sums[w];
        a.partial[blockIdx.x] = total;
    }
}

__global__ __launch_bounds__(kBlock) void balance_finish_kernel(BalanceArgs a) {
    __shared__ double sums[kBlock / 64];
    __shared__ int64_t entries[kBlock / 64];
    double total = 0.0;
    int64_t count = 0;
    for (int64_t b = threadIdx.x; b < a.blocks; b += kBlock) total += a.partial[b];
    for (int e = threadIdx.x; e < a.experts; e += kBlock) count += a.counts[e];
    for (int step = 32; step > 0; step /= 2) {
        total += __shfl_down(total, step);
        count += __shfl_down(count, step);
    }
    if (threadIdx.x % 64 == 0) {
        sums[threadIdx.x / 64] = total;
        entries[threadIdx.x / 64] = count;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < kBlock / 64; ++w) {
        total += sums[w];
        count += entries[w];
    }
    const double norm = count > 0 ? a.experts / (static_cast<double>(count) * *a.rows) : 0.0;
    *a.norm = static_cast<float>(norm);
    *a.loss = static_cast<float>(count > 0 ? total * norm : 0.0);
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

template <class T, int kLanes, bool kStream>
__global__ __launch_bounds__(kBlock) void balance_backward_kernel(BalanceBackwardArgs a, uint32_t first) {
    constexpr int kV = kPerVec<T>;
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    const int64_t row = (static_cast<int64_t>(first) + blockIdx.x) * (kBlock / kLanes) + static_cast<int>(threadIdx.x) / kLanes;
    if (row >= a.n) return;
    const float m = a.stats[row * 3], inverse = a.stats[row * 3 + 1], t = a.stats[row * 3 + 2];
    const float scale = *a.upstream * *a.norm * inverse;
    const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
    T* out = static_cast<T*>(a.dlogits) + row * a.experts;
    for (int column = lane * kV; column < a.experts; column += kLanes * kV) {
        float value[kV] = {};
        if (inverse != 0.0f) {
            load_logits(logits, column, a.experts, value);
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                const float count = column + i < a.experts ? static_cast<float>(a.counts[column + i]) : 0.0f;
                value[i] = scale * exponential<sizeof(T) == 4>(value[i] - m) * (count - t);
            }
        }
        store_some<kStream>(out + column, narrow<T>(value), a.experts - column);
    }
}

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

template <class T, int kLanes, int kVecs> void launch_choose(const ChooseArgs& a, hipStream_t stream) {
    in_launches((a.n + kBlock / kLanes - 1) / (kBlock / kLanes), kBlock, [&](uint32_t first, uint32_t count) {
        choose_kernel<T, kLanes, kVecs><<<count, kBlock, 0, stream>>>(a, first);
    });
}

}  // namespace
}  // namespace odie

using namespace odie;

ODIE_API int odie_choose_forward(const void* logits, int64_t stride, int64_t n, int experts, int choices, int normalize,
                                 int dtype, int32_t* expert, float* weights, float* stats, uint64_t stream) {
    const std::string what = "odie_choose_forward";
    if (check_rows_of(what, stride, n, choices, experts, dtype)) return -1;
    if (choices > kMaxChoices || choices > experts) return fail(what + ": choices must be within 1..64 and the experts");
    if (n == 0) return 0;
    if (!logits || !expert || !weights) return fail(what + ": null pointer");
    ChooseArgs a{logits, stride, n, expert, weights, stats, experts, choices, normalize};
    const hipStream_t s = as_stream(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const int chunks = (experts + kPerVec<T> - 1) / kPerVec<T>;
        if (chunks > 64 * (sizeof(T) == 4 ? 16 : 8)) {
            choose_long_kernel<T><<<static_cast<uint32_t>(n < 16 * kCus ? n : 16 * kCus), kBlock, 0, s>>>(a);
            return check_launch("choose");
        }
        if (chunks <= 64) with_lanes<T>(experts, choices, [&](auto lanes) { launch_choose<T, lanes, 1>(a, s); });
        else if (chunks <= 128) launch_choose<T, 64, 2>(a, s);
        else if (chunks <= 256) launch_choose<T, 64, 4>(a, s);
        else if (chunks <= 512) launch_choose<T, 64, 8>(a, s);
        else if constexpr (sizeof(T) == 4) launch_choose<T, 64, 16>(a, s);
        return check_launch("choose");
    });
}

ODIE_API int odie_choose_backward(const float* upstream, const int32_t* expert, const float* weights, const void* logits,
                                  int64_t stride, const float* stats, int64_t n, int experts, int choices, int dtype,
                                  void* dlogits, uint64_t stream) {
    const std::string what = "odie_choose_backward";
    if (check_rows_of(what, logits ? stride : experts, n, choices, experts, dtype)) return -1;
    if (choices > kMaxChoices || choices > experts) return fail(what + ": choices must be within 1..64 and the experts");
    if (n == 0) return 0;
    if (!upstream || !expert || !weights || !dlogits || (logits && !stats)) return fail(what + ": null pointer");
    ChooseBackwardArgs a{upstream, expert, weights, logits, stats, dlogits, stride, n, experts, choices};
    const hipStream_t s = as_stream(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        with_lanes<T>(experts, choices, [&](auto lanes) {
            with_flag(logits != nullptr, [&](auto all) {
                with_flag(n * experts * dtype_bytes(dtype) >= kStreamBytes, [&](auto far) {
                    in_launches((n + kBlock / lanes - 1) / (kBlock / lanes), kBlock, [&](uint32_t first, uint32_t count) {
                        choose_backward_kernel<T, lanes, all, far><<<count, kBlock, 0, s>>>(a, first);
                    });
                });
            });
        });
        return check_launch("choose gradient");
    });
}

namespace odie {
namespace {

int64_t balance_blocks(int64_t n) {
    const int64_t most = 8 * kCus, blocks = (n + 3) / 4;
    return blocks < 1 ? 1 : (blocks < most ? blocks : most);
}

}  // namespace
}  // namespace odie

ODIE_API int64_t odie_balance_workspace(int64_t n, int choices, int experts) {
    if (check_rows_of("odie_balance_workspace", experts, n, choices, experts, ODIE_F32)) return -1;
    return 8 * (balance_blocks(n) + 1);
}

ODIE_API int odie_balance_forward(const void* logits, int64_t stride, const int32_t* expert, int64_t n, int choices,
                                  int experts, int dtype, float* loss, int32_t* counts, float* stats, float* norm,
                                  void* workspace, int64_t workspace_bytes, uint64_t stream) {
    const std::string what = "odie_balance_forward";
    if (check_rows_of(what, stride, n, choices, experts, dtype)) return -1;
    if (!loss || !counts || !norm || (n > 0 && (!logits || !expert))) return fail(what + ": null pointer");
    const int64_t need = odie_balance_workspace(n, choices, experts);
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8 != 0)
        return fail(what + ": needs an 8-byte aligned workspace of " + std::to_string(need) + " bytes");
    BalanceArgs a{logits, expert, counts, nullptr, stats, nullptr, norm, loss, stride, n, balance_blocks(n), choices, experts};
    a.partial = static_cast<double*>(workspace);
    a.rows = reinterpret_cast<int32_t*>(a.partial + a.blocks);
    const hipStream_t s = as_stream(stream);
    balance_clear_kernel<<<(experts + kBlock - 1) / kBlock, kBlock, 0, s>>>(a);
    if (n > 0) {
        const int64_t wanted = (n + kBlock - 1) / kBlock;
        balance_count_kernel<<<static_cast<uint32_t>(wanted < kCountBlocks ? wanted : kCountBlocks), kBlock,
                               experts <= kSharedCounts ? experts * 4 : 0, s>>>(a);
    }
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        with_lanes<T>(experts, 1, [&](auto lanes) {
            balance_rows_kernel<T, lanes><<<static_cast<uint32_t>(a.blocks), kBlock, 0, s>>>(a);
        });
    });
    balance_finish_kernel<<<1, kBlock, 0, s>>>(a);
    return check_launch("balance");
}

ODIE_API int odie_balance_backward(const float* upstream, const void* logits, int64_t stride, const int32_t* counts,
                                   const float* stats, const float* norm, int64_t n, int experts, int dtype, void* dlogits,
                                   uint64_t stream) {
    const std::string what = "odie_balance_backward";
    if (check_rows_of(what, stride, n, 1, experts, dtype)) return -1;
    if (n == 0) return 0;
    if (!upstream || !logits || !counts || !stats || !norm || !dlogits) return fail(what + ": null pointer");
    BalanceBackwardArgs a{upstream, logits, counts, stats, norm, dlogits, stride, n, experts};
    const hipStream_t s = as_stream(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        with_lanes<T>(experts, 1, [&](auto lanes) {
            with_flag(n * experts * dtype_bytes(dtype) >= kStreamBytes, [&](auto far) {
                in_launches((n + kBlock / lanes - 1) / (kBlock / lanes), kBlock, [&](uint32_t first, uint32_t count) {
                    balance_backward_kernel<T, lanes, far><<<count, kBlock, 0, s>>>(a, first);
                });
            });
        });
        return check_launch("balance gradient");
    });
}
