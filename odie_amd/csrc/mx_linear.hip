// Linear layers whose weight is microscaled 4-bit codes, dense or with one matrix per expert over rows sorted by
// expert: act(x w[e]^T + bias[e]) + residual, for rows of 16 or 32 bits or rows of 4 bits.
//
// All sums are fp32.  Two values that the backward takes are rounded to the rows' type T where that is 16 bits, as in
// linear.hip: z, kept in half the bytes of fp32 (131072 x 512 fp16: 134 MB written and read again instead of 268), and
// dz = dy act'(z), an operand of the matrix instruction.  131072 rows, 256 -> 512 fp16, silu, dx relative to 64 bits: 2.1e-4
// by its own rounding, 2.2e-4 with z's, 3.0e-4 with dz's too; 3.3e-4 apart from a dx that is rounded once.  bf16: 0.0017,
// 0.0018, 0.0024 and 0.0026.  linear.hip has the bound of z's rounding; the bias' gradient adds dz up before dz is
// rounded, and fp32 rows round neither.
#include "mx_input.h"
#include "mx_kernels.h"

namespace odie {

// in mx_<type>.hip and mx_input_<type>.hip
extern template int launch_mx<float>(const MxRowsArgs&, hipStream_t);
extern template int launch_mx<_Float16>(const MxRowsArgs&, hipStream_t);
extern template int launch_mx<__bf16>(const MxRowsArgs&, hipStream_t);
extern template int launch_mx_input<_Float16>(const MxInputArgs&, hipStream_t);
extern template int launch_mx_input<__bf16>(const MxInputArgs&, hipStream_t);

namespace {

int check_sizes(const std::string& what, int64_t rows, int experts, bool grouped, int inputs, int outputs, int dtype,
                int activation) {
    constexpr int kMost = 1 << 20;
    if (!known_dtype(dtype)) return fail(what + ": dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (activation < 0 || activation >= kActivations) return fail(what + ": activation must be within 0..5");
    if (rows < 0 || rows > (int64_t{1} << 31) - 1) return fail(what + ": rows must be within 0..2^31 - 1");
    if (inputs < 1 || outputs < 1 || inputs > kMost || outputs > kMost)
        return fail(what + ": inputs and outputs must be within 1..2^20");
    if (experts < 1 || experts > 1 << 15) return fail(what + ": experts must be within 1..32768");
    if (!grouped && experts != 1) return fail(what + ": several experts need offsets");
    if (static_cast<int64_t>(experts) * outputs > (int64_t{1} << 31) - 1)
        return fail(what + ": experts times outputs must be below 2^31");
    return 0;
}

int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

struct GradientPlan {
    bool fused;
    int64_t pitch;                       // of the weight in dtype
    int64_t weight_bytes, sums_bytes, rest_bytes;   // the weight, its fused sums, or what odie_linear_backward takes
};

// Fused where dz is formed once for all of dx: the inputs fit a tile, in 16 bits, and the rows make two tiles a CU;
// fewer leave each CU one long chain of slabs.  us apart and fused, with the weight and the bias: 131072 rows over 64
// fp16 experts, silu, 64 -> 64 36 and 24, 128 -> 256 79 and 60, 256 -> 512 173 and 130; 65536 rows, 256 -> 512, gelu,
// 77 and 66; 300007 rows, 192 -> 40, 77 and 70; but 16384 rows over 64, 256 -> 1024, 63 and 74, 2048 over 4 20 and 37.
GradientPlan gradient_plan(int64_t rows, int experts, bool grouped, int inputs, int outputs, int dtype, int activation,
                           bool want_dx, bool want_dbias) {
    GradientPlan p{};
    p.fused = want_dx && activation != kNone && dtype != ODIE_F32 && inputs <= 256 && outputs >= 8 &&
        rows >= 2 * kCus * mx_input_tile(inputs).rows && rows / experts >= 128;
    p.pitch = p.fused ? (inputs + 7) / 8 * 8 : inputs;
    p.weight_bytes = want_dx ? padded(static_cast<int64_t>(experts) * outputs * p.pitch * dtype_bytes(dtype)) : 0;
    if (p.fused) {
        if (want_dbias)
            p.sums_bytes =
                padded(piece_ids(rows, mx_input_tile(inputs).rows, grouped, experts, false) * outputs * 4);
    } else {
        p.rest_bytes = odie_linear_workspace(rows, experts, grouped, inputs, outputs, dtype, activation, 0,
                                             want_dbias);
    }
    return p;
}

}  // namespace
}  // namespace odie

using namespace odie;

ODIE_API int odie_mx_linear_forward(const void* x, const uint8_t* x_scales, int64_t x_stride, int64_t rows,
                                    const uint8_t* codes, const uint8_t* scales, const void* bias, const void* residual,
                                    int64_t residual_stride, const int32_t* offsets, int experts, int inputs,
                                    int outputs, int dtype, int activation, void* out, int64_t out_stride, void* pre,
                                    uint64_t stream) {
    const std::string what = "odie_mx_linear_forward";
    if (check_sizes(what, rows, experts, offsets != nullptr, inputs, outputs, dtype, activation)) return -1;
    if (rows == 0) return 0;
    if (!x || !codes || !scales || !out) return fail(what + ": null pointer");
    if ((!x_scales && x_stride < inputs) || out_stride < outputs || (residual && residual_stride < outputs))
        return fail(what + ": rows overlap (a stride below the row's width)");
    if (reinterpret_cast<uintptr_t>(codes) % 16 || reinterpret_cast<uintptr_t>(scales) % 4 ||
        (x_scales && (reinterpret_cast<uintptr_t>(x) % 16 || reinterpret_cast<uintptr_t>(x_scales) % 4)))
        return fail(what + ": codes must be 16-byte and scales 4-byte aligned");
    MxRowsArgs m{};
    m.rows.a = x;
    m.rows.lda = x_stride;
    m.rows.b = codes;
    m.rows.bias = bias;
    m.rows.residual = residual;
    m.rows.ldr = residual_stride;
    m.rows.out = out;
    m.rows.ldo = out_stride;
    m.rows.pre = pre;
    m.rows.offsets = offsets;
    m.rows.rows = rows;
    m.rows.experts = experts;
    m.rows.depth = inputs;
    m.rows.columns = outputs;
    m.rows.activation = activation;
    m.a_scales = x_scales;
    m.b_scales = scales;
    m.code_pitch = mx_code_pitch(inputs);
    m.scale_pitch = mx_scale_pitch(inputs);
    return with_dtype(dtype, [&](auto t) { return launch_mx<decltype(t)>(m, as_stream(stream)); });
}

ODIE_API int64_t odie_mx_linear_workspace(int64_t rows, int experts, int grouped, int inputs, int outputs, int dtype,
                                          int activation, int want_dx, int want_dbias) {
    if (check_sizes("odie_mx_linear_workspace", rows, experts, grouped != 0, inputs, outputs, dtype, activation))
        return -1;
    const GradientPlan p = gradient_plan(rows, experts, grouped != 0, inputs, outputs, dtype, activation, want_dx != 0,
                                         want_dbias != 0);
    return p.weight_bytes + p.sums_bytes + p.rest_bytes;
}

ODIE_API int odie_mx_linear_backward(const void* upstream, int64_t upstream_stride, const void* pre, int64_t rows,
                                     const uint8_t* codes, const uint8_t* scales, const int32_t* offsets, int experts,
                                     int inputs, int outputs, int dtype, int activation, void* dx, void* dbias,
                                     void* workspace, int64_t workspace_bytes, uint64_t stream) {
    const std::string what = "odie_mx_linear_backward";
    if (check_sizes(what, rows, experts, offsets != nullptr, inputs, outputs, dtype, activation)) return -1;
    if (rows > 0 && (!upstream || (dx && (!codes || !scales)) || (activation != kNone && !pre)))
        return fail(what + ": null pointer");
    if (rows > 0 && upstream_stride < outputs) return fail(what + ": rows overlap (a stride below the row's width)");
    if (dx && (reinterpret_cast<uintptr_t>(codes) % 16 || reinterpret_cast<uintptr_t>(scales) % 4))
        return fail(what + ": codes must be 16-byte and scales 4-byte aligned");
    const GradientPlan p = gradient_plan(rows, experts, offsets != nullptr, inputs, outputs, dtype, activation,
                                         dx != nullptr, dbias != nullptr);
    const int64_t need = p.weight_bytes + p.sums_bytes + p.rest_bytes;
    if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0))
        return fail(what + ": needs a 256-byte aligned workspace of " + std::to_string(need) + " bytes");
    char* const weight = static_cast<char*>(workspace);
    if (dx && rows > 0 && odie_mx_dequantize(codes, scales, static_cast<int64_t>(experts) * outputs, inputs, dtype,
                                             weight, p.pitch, stream))
        return -1;
    if (!p.fused)
        return odie_linear_backward(upstream, upstream_stride, nullptr, 0, pre, rows, dx ? weight : nullptr, offsets,
                                    experts, inputs, outputs, dtype, activation, dx, nullptr, dbias,
                                    weight + p.weight_bytes, p.rest_bytes, stream);
    const hipStream_t s = as_stream(stream);
    MxInputArgs m{};
    m.rows.a = upstream;
    m.rows.lda = upstream_stride;
    m.rows.b = weight;
    m.rows.out = dx;
    m.rows.ldo = inputs;
    m.rows.offsets = offsets;
    m.rows.rows = rows;
    m.rows.experts = experts;
    m.rows.depth = outputs;
    m.rows.columns = inputs;
    m.rows.activation = activation;
    m.pre = pre;
    m.sums = dbias ? reinterpret_cast<float*>(weight + p.weight_bytes) : nullptr;
    m.pitch = p.pitch;
    FoldArgs f{};
    f.partial = m.sums;
    f.out = dbias;
    f.offsets = offsets;
    f.rows = rows;
    f.piece = mx_input_tile(inputs).rows;
    f.size = outputs;
    f.experts = experts;
    f.single = true;
    if (dtype == ODIE_F16) {
        if (launch_mx_input<_Float16>(m, s)) return -1;
        return dbias ? launch_fold<_Float16>(f, s) : 0;
    }
    if (launch_mx_input<__bf16>(m, s)) return -1;
    return dbias ? launch_fold<__bf16>(f, s) : 0;
}
