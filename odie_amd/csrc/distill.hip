// Distillation from a teacher's top logits: the divergence of a row's softmax from the teacher's, which holds its K
// largest logits alone, and the logits' gradient.
//
//   q_j = softmax over the row's valid entries of teacher_j / T
//   loss = sum_j q_j (log q_j - log p[id_j]),  p = softmax(logits / T)
//   dlogits = g / T (p - Q),  Q[e] = sum of q_j over the entries of class e
//
// The forward reads the logits once, with the running maximum and sum of their softmax, and keeps two numbers a row
// for each softmax; the backward reads the logits and writes their gradient, K entries of each row once more.
// Both are bound by HBM where there are many classes.
#include "softmax.h"

namespace odie {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxClasses = 1 << 24;
constexpr int kMaxTop = 1024;
constexpr int kShort = 512;        // classes of a row that some lanes of a wave take
constexpr int kMedium = 4096;      // and where there are many rows
constexpr int kMostPiece = 1 << 16; // classes of a longer row's piece in the backward

struct DistillArgs {
    const void* logits;       // [n][classes], stride
    const void* ids;          // [n][top], int32 or int64
    const void* teacher;      // [n][top]
    const float* upstream;    // [n] (backward)
    float* loss;              // [n] (forward)
    // [n][4]: m and 1 / s of logits / T (1 / s 0: all masked), and of teacher / T (0: no entries)
    float* stats;
    void* dlogits;            // [n][classes] (backward)
    float2* partial;          // [n][pieces]: m and s of a piece of a row (forward)
    int64_t stride, n;
    int classes, top, id_bytes, teacher_dtype;
    int pieces, piece;        // a row's pieces, their classes
    float inverse;            // 1 / T
};

__device__ inline int64_t id_of(const DistillArgs& a, int64_t at) {
    return a.id_bytes == 4 ? static_cast<const int32_t*>(a.ids)[at] : static_cast<const int64_t*>(a.ids)[at];
}
__device__ inline float teacher_of(const DistillArgs& a, int64_t at) {
    if (a.teacher_dtype == ODIE_F32) return static_cast<const float*>(a.teacher)[at];
    if (a.teacher_dtype == ODIE_F16) return static_cast<float>(static_cast<const _Float16*>(a.teacher)[at]);
    return static_cast<float>(static_cast<const __bf16*>(a.teacher)[at]);
}

// The scaled teacher logit of the row's entry j, -inf where its class is none.
__device__ inline float entry_of(const DistillArgs& a, int64_t row, int j, int64_t& id) {
    id = id_of(a, row * a.top + j);
    return id >= 0 && id < a.classes ? teacher_of(a, row * a.top + j) * a.inverse : kNegInfinity;
}

// Calls f(column, values) for the chunks of columns [begin, end) that lane `lane` of kLanes takes, kAhead whole ones at
// a time, whose loads are in flight together.
template <class T, int kLanes, int kAhead, class F>
__device__ inline void for_chunks(const T* row, int begin, int end, int width, int lane, F&& f) {
    constexpr int kV = kPerVec<T>, kStep = kLanes * kV;
    int column = begin + lane * kV;
    for (; column + (kAhead - 1) * kStep + kV <= end; column += kAhead * kStep) {
        vec16 chunk[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) chunk[u] = load16(row + column + u * kStep);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            float value[kV];
            widen<T>(chunk[u], value);
            f(column + u * kStep, value);
        }
    }
    for (; column < end; column += kStep) {
        float value[kV];
        load_logits(row, column, width, value);
        f(column, value);
    }
}

// Adds the logits / T of columns [begin, end) to run.
template <class T, int kLanes, class R>
__device__ inline void add_columns(const DistillArgs& a, const T* row, int begin, int end, int lane, R& run) {
    constexpr int kV = kPerVec<T>;
    for_chunks<T, kLanes, kLanes == kBlock ? 4 : 1>(row, begin, end, a.classes, lane, [&](int, float (&value)[kV]) {
#pragma unroll
        for (int i = 0; i < kV; ++i) value[i] *= a.inverse;
        run.add(value);
    });
}

// A row's loss from its softmax (m, s): kLanes lanes of one wave share the entries.
template <class T, int kLanes>
__device__ inline void finish_row(const DistillArgs& a, int64_t row, int lane, bool store, float m, float s) {
    float top = kNegInfinity;
    for (int j = lane; j < a.top; j += kLanes) {
        int64_t id;
        top = larger(top, entry_of(a, row, j, id));
    }
    top = max_across<kLanes>(top);
    const float base = base_of(top);
    float total = 0.0f;
    for (int j = lane; j < a.top; j += kLanes) {
        int64_t id;
        total += expf(entry_of(a, row, j, id) - base);
    }
    total = sum_across<kLanes>(total);
    const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
    // a row whose logits are all masked has no p above 0
    const float log_total = logf(total), log_s = s == 0.0f ? 0.0f : logf(s), own_base = base_of(m);
    float loss = 0.0f;
    for (int j = lane; j < a.top; j += kLanes) {
        int64_t id;
        const float entry = entry_of(a, row, j, id) - base, q = expf(entry) / total;
        if (id < 0 || id >= a.classes || q == 0.0f) continue;       // a share that is 0 in fp32 adds nothing
        const float own = static_cast<float>(logits[id]) * a.inverse - own_base - log_s;
        loss = fmaf(q, entry - log_total - own, loss);
    }
    loss = sum_across<kLanes>(loss);
    const bool none = top == kNegInfinity;
    if (!store || lane != 0) return;
    a.loss[row] = none ? 0.0f : loss;
    if (a.stats) {
        float* to = a.stats + row * 4;
        to[0] = own_base;
        to[1] = s == 0.0f ? 0.0f : 1.0f / s;
        to[2] = base;
        to[3] = none ? 0.0f : 1.0f / total;
    }
}

// Shorter rows, kLanes lanes each.
template <class T, int kLanes>
__global__ __launch_bounds__(kBlock) void distill_short_kernel(DistillArgs a, uint32_t first) {
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    const int64_t at =
        (static_cast<int64_t>(first) + blockIdx.x) * (kBlock / kLanes) + static_cast<int>(threadIdx.x) / kLanes;
    const int64_t row = at < a.n ? at : a.n - 1;
    Running<sizeof(T) == 4> run;
    add_columns<T, kLanes>(a, static_cast<const T*>(a.logits) + row * a.stride, 0, a.classes, lane, run);
    run.template join_lanes<kLanes>();
    finish_row<T, kLanes>(a, row, lane, at < a.n, run.m, run.s);
}

// Longer rows: a workgroup a piece.  Where a row is one piece, its loss too.  8192 x 65032 bf16: 208 us, 1.07 GB at 5.1
// TB/s: HBM (a chunk at a time 221).
template <class T> __global__ __launch_bounds__(kBlock) void distill_piece_kernel(DistillArgs a, uint32_t first) {
    __shared__ float2 part[kBlock / 64];
    const int64_t id = static_cast<int64_t>(first) + blockIdx.x, row = id / a.pieces;
    const int piece = static_cast<int>(id % a.pieces), begin = piece * a.piece;
    const int end = begin + a.piece < a.classes ? begin + a.piece : a.classes;
    Running<sizeof(T) == 4> run;
    add_columns<T, kBlock>(a, static_cast<const T*>(a.logits) + row * a.stride, begin, end,
                           static_cast<int>(threadIdx.x), run);
    run.template join_lanes<64>();
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = make_float2(run.m, run.s);
    __syncthreads();
    if (threadIdx.x >= 64) return;
    run = {};
    for (int w = 0; w < kBlock / 64; ++w) run.join(part[w].x, part[w].y);
    if (a.pieces == 1) finish_row<T, 64>(a, row, static_cast<int>(threadIdx.x), true, run.m, run.s);
    else if (threadIdx.x == 0) a.partial[id] = make_float2(run.m, run.s);
}

// Joins a row's pieces, a wave a row.
template <class T> __global__ __launch_bounds__(64) void distill_join_kernel(DistillArgs a) {
    const int64_t row = blockIdx.x;
    Running<sizeof(T) == 4> run;
    for (int p = threadIdx.x; p < a.pieces; p += 64) {
        const float2 part = a.partial[row * a.pieces + p];
        run.join(part.x, part.y);
    }
    run.template join_lanes<64>();
    finish_row<T, 64>(a, row, static_cast<int>(threadIdx.x), true, run.m, run.s);
}

// The gradient at the row's entry j, p - Q, from the piece [begin, end) of the row.  The first entry of a class that
// several name (`twice`, a bit for each class of the piece) adds up the others'.
template <class T>
__device__ inline void patch_entry(const DistillArgs& a, int64_t row, int j, int begin, int end, const uint32_t* twice,
                                   const T* logits, T* out, float scale, const float (&stats)[4]) {
    int64_t id, other;
    const float entry = entry_of(a, row, j, id);
    if (id < begin || id >= end) return;
    float share = expf(entry - stats[2]) * stats[3];
    const int place = static_cast<int>(id) - begin;
    if (twice[place / 32] >> place % 32 & 1)
        for (int i = 0; i < a.top; ++i) {
            if (i == j || id_of(a, row * a.top + i) != id) continue;
            if (i < j) return;
            share += expf(entry_of(a, row, i, other) - stats[2]) * stats[3];
        }
    const float p = expf(static_cast<float>(logits[id]) * a.inverse - stats[0]) * stats[1];
    float value = scale * (p - share);
    asm("" : "+v"(value));      // rounded to fp32, then to T, as its neighbours are
    out[id] = static_cast<T>(value);
}

// A piece of a row's gradient: kLanes threads (some of a wave's, or the workgroup).  A workgroup's stores begin on
// lines of 128 bytes, whatever the row does (8192 x 65032 bf16: 514 -> 465 us; rows that begin on lines themselves 455;
// 452, 2.13 GB at 4.7 TB/s, in all): the row's elements before the first line go one by one, and its pieces are cut at
// lines.  Two bits for each class of the piece tell whether no, one or several entries name it: those of a class that
// one names, as a teacher's largest logits do, need not look for others (8192 x 1024 with 128 entries a row: 129 us
// where each looks at all, 18 so).
template <class T, int kLanes, bool kStream>
__global__ __launch_bounds__(kBlock) void distill_backward_kernel(DistillArgs a, uint32_t first) {
    constexpr int kV = kPerVec<T>;
    constexpr int kWords = kLanes == kBlock ? (kMostPiece + 64) / 32 : (kLanes == 64 ? kMedium / 32 : kLanes / 4);
    __shared__ uint32_t bits[kBlock / kLanes][2][kWords];
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    uint32_t *const once = bits[static_cast<int>(threadIdx.x) / kLanes][0],
                   *const twice = bits[static_cast<int>(threadIdx.x) / kLanes][1];
    const int64_t at =
        (static_cast<int64_t>(first) + blockIdx.x) * (kBlock / kLanes) + static_cast<int>(threadIdx.x) / kLanes;
    const int64_t row = at / a.pieces;
    const bool inside = row < a.n;
    const int piece = static_cast<int>(at % a.pieces);
    const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
    T* out = static_cast<T*>(a.dlogits) + row * a.classes;
    constexpr int kLine = 128 / static_cast<int>(sizeof(T));
    // elements of the line before
    const int past = kLanes == kBlock ? static_cast<int>(reinterpret_cast<uintptr_t>(out) / sizeof(T) % kLine) : 0;
    const int begin = piece == 0 ? 0 : piece * a.piece - past;
    const int end = piece == a.pieces - 1 ? a.classes : (piece + 1) * a.piece - past;
    const int head = piece == 0 && past > 0 ? (kLine - past < end ? kLine - past : end) : 0;
    for (int w = lane; w < (end - begin + 31) / 32; w += kLanes) once[w] = twice[w] = 0;
    if constexpr (kLanes == kBlock) __syncthreads();
    else wave_fence();
    if (inside)
        for (int j = lane; j < a.top; j += kLanes) {
            const int64_t id = id_of(a, row * a.top + j);
            if (id < begin || id >= end) continue;
            const int place = static_cast<int>(id) - begin;
            const uint32_t bit = 1u << place % 32;
            if (atomicOr(once + place / 32, bit) & bit) atomicOr(twice + place / 32, bit);
        }
    float stats[4] = {}, scale = 0.0f;
    if (inside) {
#pragma unroll
        for (int i = 0; i < 4; ++i) stats[i] = a.stats[row * 4 + i];
        scale = a.upstream[row] * a.inverse;
        const float each = scale * stats[1];
        const auto gradient = [&](float logit) {
            const float p = each * exponential<sizeof(T) == 4>(fmaf(logit, a.inverse, -stats[0]));
            return stats[3] == 0.0f ? 0.0f : p;
        };
        for (int column = lane; column < head; column += kLanes) {
            float value = gradient(static_cast<float>(logits[column]));
            asm("" : "+v"(value));      // rounded to fp32, then to T, as its neighbours are
            out[column] = static_cast<T>(value);
        }
        for_chunks<T, kLanes, kLanes == kBlock ? 4 : 1>(logits, begin + head, end, a.classes, lane,
                                                        [&](int column, float (&value)[kV]) {
#pragma unroll
            for (int i = 0; i < kV; ++i) value[i] = gradient(value[i]);
            store_some<kStream>(out + column, narrow<T>(value), a.classes - column);
        });
    }
    // the entries' classes once more, after every lane's stores
    if constexpr (kLanes == kBlock) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
    if (!inside || stats[3] == 0.0f) return;
    for (int j = lane; j < a.top; j += kLanes) patch_entry(a, row, j, begin, end, twice, logits, out, scale, stats);
}

int check_distill(const std::string& what, int64_t n, int classes, int top, int dtype) {
    if (!known_dtype(dtype)) return fail(what + ": dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (n < 0 || n > (int64_t{1} << 31) - 1) return fail(what + ": rows must be within 0..2^31 - 1");
    if (classes < 1 || classes > kMaxClasses) return fail(what + ": classes must be within 1..2^24");
    if (top < 1 || top > kMaxTop) return fail(what + ": a row's entries must be within 1..1024");
    return 0;
}

// Whether a row takes some lanes or a wave, else a workgroup or several.  us forward and backward as a wave and as a
// workgroup, bf16: 8192 x 1024 (forward) 7.8 and 12.2, 8192 x 2048 25 and 33, 8192 x 8192 73 and 68, 1024 x 4000 14.3
// and 12.0.
bool by_lanes(int64_t n, int classes) { return classes <= kShort || (classes <= kMedium && n >= 4096); }

// Pieces that a long row is cut into, each of whole rounds of its workgroup: about four workgroups a CU at least, and
// at most `most` classes a piece.
void cut(DistillArgs& a, int values, int64_t most) {
    const int64_t wanted = a.n < 4 * kCus ? (4 * kCus + a.n - 1) / a.n : 1;
    const int64_t round = static_cast<int64_t>(kBlock) * values;
    const int64_t rounds = (a.classes + round - 1) / round, least = (a.classes + most - 1) / most;
    int64_t pieces = wanted < rounds ? wanted : rounds;
    pieces = pieces < least ? least : pieces;
    a.piece = static_cast<int>((rounds + pieces - 1) / pieces * round);
    a.pieces = (a.classes + a.piece - 1) / a.piece;
}

template <class T, class F> void with_lanes(int classes, F&& f) {
    const int chunks = (classes + kPerVec<T> - 1) / kPerVec<T>;
    if (chunks <= 8) f(std::integral_constant<int, 8>{});
    else if (chunks <= 16) f(std::integral_constant<int, 16>{});
    else if (chunks <= 32) f(std::integral_constant<int, 32>{});
    else f(std::integral_constant<int, 64>{});
}

}  // namespace
}  // namespace odie

using namespace odie;

ODIE_API int64_t odie_distill_workspace(int64_t n, int classes, int dtype) {
    if (check_distill("odie_distill_workspace", n, classes, 1, dtype)) return -1;
    if (n == 0 || by_lanes(n, classes)) return 0;
    DistillArgs a{};
    a.n = n;
    a.classes = classes;
    cut(a, dtype == ODIE_F32 ? 4 : 8, kMaxClasses);
    return a.pieces > 1 ? n * a.pieces * static_cast<int64_t>(sizeof(float2)) : 0;
}

ODIE_API int odie_distill_forward(const void* logits, int64_t stride, const void* ids, int id_bytes,
                                  const void* teacher, int teacher_dtype, int64_t n, int classes, int top,
                                  float temperature, int dtype, float* loss, float* stats, void* workspace,
                                  int64_t workspace_bytes, uint64_t stream) {
    const std::string what = "odie_distill_forward";
    if (check_distill(what, n, classes, top, dtype)) return -1;
    if (!known_dtype(teacher_dtype)) return fail(what + ": teacher_dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (id_bytes != 4 && id_bytes != 8) return fail(what + ": id_bytes must be 4 or 8");
    if (!(temperature > 0.0f) || !(1.0f / temperature > 0.0f) || std::isinf(1.0f / temperature))
        return fail(what + ": temperature must be above 0 and finite");
    if (n == 0) return 0;
    if (!logits || !ids || !teacher || !loss) return fail(what + ": null pointer");
    if (stride < classes) return fail(what + ": rows overlap (a stride below the row's width)");
    const int64_t need = odie_distill_workspace(n, classes, dtype);
    if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8 != 0))
        return fail(what + ": needs an 8-byte aligned workspace of " + std::to_string(need) + " bytes");
    DistillArgs a{logits, ids, teacher, nullptr, loss, stats, nullptr, static_cast<float2*>(workspace), stride, n,
                  classes, top, id_bytes, teacher_dtype, 1, classes, 1.0f / temperature};
    const hipStream_t s = as_stream(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (by_lanes(n, classes)) {
            with_lanes<T>(classes, [&](auto lanes) {
                in_launches((n + kBlock / lanes - 1) / (kBlock / lanes), kBlock,
                                [&](uint32_t first, uint32_t count) {
                    distill_short_kernel<T, lanes><<<count, kBlock, 0, s>>>(a, first);
                });
            });
            return check_launch("distill");
        }
        cut(a, kPerVec<T>, kMaxClasses);
        in_launches(n * a.pieces, kBlock, [&](uint32_t first, uint32_t count) {
            distill_piece_kernel<T><<<count, kBlock, 0, s>>>(a, first);
        });
        if (a.pieces > 1) distill_join_kernel<T><<<static_cast<uint32_t>(n), 64, 0, s>>>(a);
        return check_launch("distill");
    });
}

ODIE_API int odie_distill_backward(const float* upstream, const void* logits, int64_t stride, const void* ids,
                                   int id_bytes, const void* teacher, int teacher_dtype, const float* stats, int64_t n,
                                   int classes, int top, float temperature, int dtype, void* dlogits, uint64_t stream) {
    const std::string what = "odie_distill_backward";
    if (check_distill(what, n, classes, top, dtype)) return -1;
    if (!known_dtype(teacher_dtype)) return fail(what + ": teacher_dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (id_bytes != 4 && id_bytes != 8) return fail(what + ": id_bytes must be 4 or 8");
    if (!(temperature > 0.0f) || !(1.0f / temperature > 0.0f) || std::isinf(1.0f / temperature))
        return fail(what + ": temperature must be above 0 and finite");
    if (n == 0) return 0;
    if (!upstream || !logits || !ids || !teacher || !stats || !dlogits) return fail(what + ": null pointer");
    if (stride < classes) return fail(what + ": rows overlap (a stride below the row's width)");
    DistillArgs a{logits, ids, teacher, upstream, nullptr, const_cast<float*>(stats), dlogits, nullptr, stride, n,
                  classes, top, id_bytes, teacher_dtype, 1, classes, 1.0f / temperature};
    const hipStream_t s = as_stream(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        with_flag(n * classes * dtype_bytes(dtype) >= kStreamBytes, [&](auto far) {
            if (by_lanes(n, classes)) {
                with_lanes<T>(classes, [&](auto lanes) {
                    in_launches((n + kBlock / lanes - 1) / (kBlock / lanes), kBlock,
                                [&](uint32_t first, uint32_t count) {
                        distill_backward_kernel<T, lanes, far><<<count, kBlock, 0, s>>>(a, first);
                    });
                });
            } else {
                cut(a, kPerVec<T>, kMostPiece);
                in_launches(n * a.pieces, kBlock, [&](uint32_t first, uint32_t count) {
                    distill_backward_kernel<T, kBlock, far><<<count, kBlock, 0, s>>>(a, first);
                });
            }
        });
        return check_launch("distill gradient");
    });
}
