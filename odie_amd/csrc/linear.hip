// Linear layers with bias, activation and residual fused into the product, dense or with one weight
// matrix per expert over rows sorted by expert, and their gradients.
//
//   z = x w[e]^T + bias[e],  y = act(z) + residual            rows offsets[e] .. offsets[e + 1] - 1
//   dz = dy act'(z),  dx = dz w[e],  dw[e] = dz^T x,  dbias[e] = sum dz,  dresidual = dy
//
// The forward is one launch.  The backward forms dz and its column sums in one pass over dy and z, then
// dx and dw as products of dz; dw sums over rows, so the rows are cut into pieces whose fp32 sums are
// joined in a fixed order: the result does not depend on timing.  Workspaces are the caller's.
//
// z is kept in the tensors' own type for the backward, in half the bytes of fp32 where that is 16 bits.  Its rounding
// moves act'(z) by at most |z act''(z)| half units of 1, which is at most a third of one.  That is an absolute bound: of
// act'(z) itself it is up to |z| half units where the slope decays exponentially (sigmoid and softplus in bf16: 3 % at
// z = -12.8, 6 % at -20), and without bound where gelu's and silu's slopes cross 0.
#include "linear.h"

namespace odie {
namespace {

constexpr int64_t kMaxRows = (int64_t{1} << 31) - 1;
constexpr int kMaxWidth = 1 << 20;
constexpr int kMaxExperts = 1 << 15;

// Rows a piece of the slope pass takes (and a partial bias sums): about eight workgroups a CU, each of
// them of at most 256 columns, and two rows a lane at least (4099 x 517 bf16, 256 columns a workgroup: 13.8 us with
// 16 rows, 19.5 with 64; 16384 x 64, 64 columns: 10.1 us with 64 rows, 16.1 with 16).
int64_t slope_piece(int64_t rows, int outputs) {
    const int64_t across = (outputs + 255) / 256, least = 512 / slope_lanes(outputs), most = int64_t{1} << 30;
    const int64_t piece = (rows * across / (8 * kCus) + least - 1) / least * least;
    return piece < least ? least : (piece < most ? piece : most);
}

// Tiles of the weight gradient and the rows a workgroup sums.  Three CUs of four at least are to have a workgroup (four
// of the smallest tiles, two of the middle ones), from several pieces of the rows where there are too few tiles;
// but partial sums, written and read again, are to stay below twice what the operands hold, with several experts
// too (131072 bf16 rows over 1024 experts of 1024 x 1024: pieces of 1024 rows and 1.1 GB of sums).  The
// largest tiles that manage it are taken (a 1024 x 1024 gradient over 4096 bf16 rows: 61 us as 16 tiles of
// 256 x 256 and 16 pieces, 29 us as 64 of 128 x 128 and 4 pieces).
struct WeightPlan {
    int edge;
    int64_t piece;
};

WeightPlan weight_plan(int64_t rows, int experts, int outputs, int inputs, int dtype) {
    const int least = outputs < inputs ? outputs : inputs;
    const int64_t matrix = static_cast<int64_t>(outputs) * inputs;
    const int64_t most = rows * (static_cast<int64_t>(outputs) + inputs) * dtype_bytes(dtype) / (4 * matrix);
    auto tiles_of = [&](int64_t edge) { return ((outputs + edge - 1) / edge) * ((inputs + edge - 1) / edge); };
    auto whole = [](int64_t piece) { return piece < 256 ? 256 : (piece + 255) / 256 * 256; };
    if (experts > 1) {
        // Groups of up to twice the average stay whole where there are workgroups enough.
        const int edge = least > 64 ? 128 : 64;   // 256 gains nothing where groups differ in length
        const int64_t wanted = 4 * kCus / tiles_of(edge), pieces = wanted < most ? wanted : most;
        const int64_t twice = 2 * (rows / experts), least_piece = most > 0 ? (rows + most - 1) / most : rows;
        if (pieces <= 2 * experts) return WeightPlan{edge, whole(twice > least_piece ? twice : least_piece)};
        return WeightPlan{edge, whole((rows + pieces - experts / 2 - 1) / (pieces - experts / 2))};
    }
    for (int edge = 256;; edge /= 2) {
        if (edge > 64 && least <= edge / 2) continue;
        const int64_t tiles = tiles_of(edge);
        int64_t pieces = 256 / edge * kCus / tiles;
        if (pieces > most) pieces = most;
        if (pieces < 1) pieces = 1;
        if (edge > 64 && 4 * tiles * pieces < 3 * kCus) continue;
        return WeightPlan{edge, whole((rows + pieces - 1) / pieces)};
    }
}

struct Plan {
    int64_t dz_bytes, sums_bytes, partial_bytes;   // each a multiple of 256
    int64_t slope_piece, slope_pieces, weight_piece, weight_pieces;
    int weight_edge;
};

int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

Plan make_plan(int64_t rows, int experts, bool grouped, int outputs, int inputs, int dtype, int activation,
               bool want_dweight, bool want_dbias) {
    Plan p{};
    p.slope_piece = slope_piece(rows, outputs);
    p.slope_pieces = piece_ids(rows, p.slope_piece, grouped && want_dbias, experts, false);
    const WeightPlan weight = weight_plan(rows, experts, outputs, inputs, dtype);
    p.weight_piece = weight.piece;
    p.weight_edge = weight.edge;
    p.weight_pieces = piece_ids(rows, p.weight_piece, grouped, experts, false);
    if (p.weight_pieces < 1) p.weight_pieces = 1;
    p.dz_bytes = activation == kNone ? 0 : padded(rows * outputs * dtype_bytes(dtype));
    p.sums_bytes = want_dbias ? padded(p.slope_pieces * outputs * 4) : 0;
    p.partial_bytes = want_dweight && rows > p.weight_piece
                          ? padded(partial_slots(rows, p.weight_piece, grouped) * outputs * static_cast<int64_t>(inputs) * 4) : 0;
    return p;
}

int check_sizes(const std::string& what, int64_t rows, int experts, bool grouped, int inputs, int outputs, int dtype,
                int activation) {
    if (!known_dtype(dtype)) return fail(what + ": dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (activation < 0 || activation >= kActivations) return fail(what + ": activation must be within 0..5");
    if (rows < 0 || rows > kMaxRows) return fail(what + ": rows must be within 0..2^31 - 1");
    if (inputs < 1 || outputs < 1 || inputs > kMaxWidth || outputs > kMaxWidth)
        return fail(what + ": inputs and outputs must be within 1..2^20");
    if (experts < 1 || experts > kMaxExperts) return fail(what + ": experts must be within 1..32768");
    if (!grouped && experts != 1) return fail(what + ": several experts need offsets");
    return 0;
}

}  // namespace
}  // namespace odie

using namespace odie;

ODIE_API int odie_linear_forward(const void* x, int64_t x_stride, int64_t rows, const void* weight, const void* bias,
                                 const void* residual, int64_t residual_stride, const int32_t* offsets, int experts,
                                 int inputs, int outputs, int dtype, int activation, void* out, int64_t out_stride,
                                 void* pre, uint64_t stream) {
    const char* what = "odie_linear_forward";
    if (check_sizes(what, rows, experts, offsets != nullptr, inputs, outputs, dtype, activation)) return -1;
    if (rows == 0) return 0;
    if (!x || !weight || !out) return fail(std::string(what) + ": null pointer");
    if (x_stride < inputs || out_stride < outputs || (residual && residual_stride < outputs))
        return fail(std::string(what) + ": rows overlap (a stride below the row's width)");
    RowsArgs a{};
    a.a = x;
    a.lda = x_stride;
    a.b = weight;
    a.bias = bias;
    a.residual = residual;
    a.ldr = residual_stride;
    a.out = out;
    a.ldo = out_stride;
    a.pre = pre;
    a.offsets = offsets;
    a.rows = rows;
    a.experts = experts;
    a.depth = inputs;
    a.columns = outputs;
    a.activation = activation;
    return with_dtype(dtype, [&](auto t) { return launch_rows<decltype(t)>(a, true, as_stream(stream)); });
}

ODIE_API int64_t odie_linear_workspace(int64_t rows, int experts, int grouped, int inputs, int outputs, int dtype,
                                       int activation, int want_dweight, int want_dbias) {
    if (check_sizes("odie_linear_workspace", rows, experts, grouped != 0, inputs, outputs, dtype, activation)) return -1;
    const Plan p = make_plan(rows, experts, grouped != 0, outputs, inputs, dtype, activation, want_dweight != 0,
                             want_dbias != 0);
    return p.dz_bytes + p.sums_bytes + p.partial_bytes;
}

ODIE_API int odie_linear_backward(const void* upstream, int64_t upstream_stride, const void* x, int64_t x_stride,
                                  const void* pre, int64_t rows, const void* weight, const int32_t* offsets,
                                  int experts, int inputs, int outputs, int dtype, int activation, void* dx,
                                  void* dweight, void* dbias, void* workspace, int64_t workspace_bytes,
                                  uint64_t stream) {
    const std::string what = "odie_linear_backward";
    if (check_sizes(what, rows, experts, offsets != nullptr, inputs, outputs, dtype, activation)) return -1;
    if (rows > 0 && (!upstream || (dweight && !x) || (dx && !weight) || (activation != kNone && !pre)))
        return fail(what + ": null pointer");
    if (rows > 0 && (upstream_stride < outputs || (dweight && x_stride < inputs)))
        return fail(what + ": rows overlap (a stride below the row's width)");
    const Plan p = make_plan(rows, experts, offsets != nullptr, outputs, inputs, dtype, activation, dweight != nullptr,
                             dbias != nullptr);
    const int64_t need = p.dz_bytes + p.sums_bytes + p.partial_bytes;
    if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0))
        return fail(what + ": needs a 256-byte aligned workspace of " + std::to_string(need) + " bytes");
    hipStream_t s = as_stream(stream);
    char* scratch = static_cast<char*>(workspace);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const void* dz = upstream;
        int64_t dz_stride = upstream_stride;
        float* sums = p.sums_bytes ? reinterpret_cast<float*>(scratch + p.dz_bytes) : nullptr;
        if ((activation != kNone || dbias) && rows > 0) {
            SlopeArgs a{};
            a.dy = upstream;
            a.ldy = upstream_stride;
            a.pre = pre;
            a.dz = activation != kNone ? scratch : nullptr;
            a.sums = sums;
            a.offsets = dbias ? offsets : nullptr;   // the sums alone go by expert
            a.rows = rows;
            a.piece = p.slope_piece;
            a.pieces = p.slope_pieces;
            a.experts = experts;
            a.columns = outputs;
            a.activation = activation;
            if (launch_slope<T>(a, s)) return -1;
            if (activation != kNone) {
                dz = scratch;
                dz_stride = outputs;
            }
        }
        if (dbias) {
            FoldArgs a{};
            a.partial = sums;
            a.out = dbias;
            a.offsets = offsets;
            a.rows = rows;
            a.piece = p.slope_piece;
            a.size = outputs;
            a.experts = experts;
            a.single = true;
            if (launch_fold<T>(a, s)) return -1;
        }
        if (dx && rows > 0) {
            RowsArgs a{};
            a.a = dz;
            a.lda = dz_stride;
            a.b = weight;
            a.out = dx;
            a.ldo = inputs;
            a.offsets = offsets;
            a.rows = rows;
            a.experts = experts;
            a.depth = outputs;
            a.columns = inputs;
            if (launch_rows<T>(a, false, s)) return -1;
        }
        if (dweight) {
            WeightArgs a{};
            a.dz = dz;
            a.ldz = dz_stride;
            a.x = x;
            a.ldx = x_stride;
            a.dw = dweight;
            a.partial = reinterpret_cast<float*>(scratch + p.dz_bytes + p.sums_bytes);
            a.offsets = offsets;
            a.rows = rows;
            a.piece = p.weight_piece;
            a.pieces = p.weight_pieces;
            a.edge = p.weight_edge;
            a.experts = experts;
            a.outputs = outputs;
            a.inputs = inputs;
            if (launch_weight<T>(a, s)) return -1;
            if (p.partial_bytes) {
                FoldArgs f{};
                f.partial = a.partial;
                f.out = dweight;
                f.offsets = offsets;
                f.rows = rows;
                f.piece = p.weight_piece;
                f.size = static_cast<int64_t>(outputs) * inputs;
                f.experts = experts;
                f.single = false;
                if (launch_fold<T>(f, s)) return -1;
            }
        }
        return 0;
    });
}
