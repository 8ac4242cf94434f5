// Linear layers whose weight is microscaled 4-bit codes, dense or with one matrix per expert over rows sorted by
// expert: act(x w[e]^T + bias[e]) + residual, for rows of 16 or 32 bits or rows of 4 bits.
#include "mx_kernels.h"

using namespace odie;

ODIE_API int odie_mx_linear_forward(const void* x, const uint8_t* x_scales, int64_t x_stride, int64_t rows,
                                    const uint8_t* codes, const uint8_t* scales, const void* bias, const void* residual,
                                    int64_t residual_stride, const int32_t* offsets, int experts, int inputs, int outputs,
                                    int dtype, int activation, void* out, int64_t out_stride, void* pre, uint64_t stream) {
    const std::string what = "odie_mx_linear_forward";
    constexpr int kMost = 1 << 20;
    if (!known_dtype(dtype)) return fail(what + ": dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (activation < 0 || activation >= kActivations) return fail(what + ": activation must be within 0..5");
    if (rows < 0 || rows > (int64_t{1} << 31) - 1) return fail(what + ": rows must be within 0..2^31 - 1");
    if (inputs < 1 || outputs < 1 || inputs > kMost || outputs > kMost)
        return fail(what + ": inputs and outputs must be within 1..2^20");
    if (experts < 1 || experts > 1 << 15) return fail(what + ": experts must be within 1..32768");
    if (!offsets && experts != 1) return fail(what + ": several experts need offsets");
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
