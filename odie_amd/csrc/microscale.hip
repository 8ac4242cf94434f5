// Rows to microscaled 4-bit codes and back.
//
//   s = floor(log2 max |x|) - 2 + 127, within 0..254
//   code = nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} to x 2^(127 - s)
//
// The largest magnitude lands in [4, 8): above 6 it is clamped.  Dividing by a power of two is exact (a subnormal scale
// too), so each value is rounded once.  Four lanes take a block, eight values each; their largest magnitude goes round
// by two lane moves.  Both directions are bound by HBM: 65536 x 4096 fp16 (537 MB, and 151 MB of codes and scales) 123
// us there, 121 back, 5.6 TB/s, codes in the last-level cache.
#include "mx.h"

namespace odie {
namespace {

constexpr int kBlock = 256;
constexpr int kLanesOfBlock = 4;   // lanes that share a block of 32 values
constexpr int kMaxWidth = 1 << 20;

struct MxArgs {
    const void* x;
    void* out;
    const uint8_t* codes_in;
    const uint8_t* scales_in;
    uint8_t* codes;
    uint8_t* scales;
    int64_t stride, rows;
    int width, blocks, lanes, parts;   // lanes: threads across a row; parts: workgroups across it (1 where lanes < 256)
};

template <int kByte> __device__ inline uint32_t to_pair(uint32_t old, float a, float b, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, scale, kByte);
}

// The place of this thread: row and chunk of eight values.
struct Place {
    int64_t row;
    int chunk;
};
__device__ inline Place place_of(const MxArgs& a, uint32_t first) {
    const uint32_t block = first + blockIdx.x;
    if (a.parts > 1)
        return Place{block / a.parts, static_cast<int>(block % a.parts) * kBlock + static_cast<int>(threadIdx.x)};
    return Place{static_cast<int64_t>(block) * (kBlock / a.lanes) + static_cast<int>(threadIdx.x) / a.lanes,
                 static_cast<int>(threadIdx.x) % a.lanes};
}

template <class T> __global__ __launch_bounds__(kBlock) void quantize_kernel(MxArgs a, uint32_t first) {
    const Place p = place_of(a, first);
    const int block = p.chunk / kLanesOfBlock, padded = (a.blocks + 3) / 4 * 4;
    const bool inside = p.row < a.rows && block < a.blocks;
    float value[8] = {};
    if (inside) load8(static_cast<const T*>(a.x) + p.row * a.stride + p.chunk * 8, a.width - p.chunk * 8, value);
    uint32_t most = 0;                 // magnitudes in the order of their bits: infinities and NaN above every number
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t size = __builtin_bit_cast(uint32_t, value[i]) & 0x7fffffffu;
        most = size > most ? size : most;
    }
    uint32_t other = dpp_move<0xB1>(most);     // quad_perm [1, 0, 3, 2]
    most = other > most ? other : most;
    other = dpp_move<0x4E>(most);              // quad_perm [2, 3, 0, 1]
    most = other > most ? other : most;
    const uint32_t exponent = most >> 23;      // 0 for subnormal magnitudes: their scale is the least
    const uint32_t s = exponent == 255 ? 255u : (exponent > 2 ? exponent - 2 : 0u);
    const float scale = mx_scale(s);
    uint32_t codes = 0;
    if (s != 255) {
        codes = to_pair<0>(codes, value[0], value[1], scale);
        codes = to_pair<1>(codes, value[2], value[3], scale);
        codes = to_pair<2>(codes, value[4], value[5], scale);
        codes = to_pair<3>(codes, value[6], value[7], scale);
    }
    if (inside) *reinterpret_cast<uint32_t*>(a.codes + (p.row * a.blocks * kLanesOfBlock + p.chunk) * 4) = codes;
    if (p.row < a.rows && block < padded && p.chunk % kLanesOfBlock == 0)
        a.scales[p.row * padded + block] = block < a.blocks ? static_cast<uint8_t>(s) : 0;
}

// A lane writes 16 bytes, so that a wave's store is of whole lines (65536 x 4096 fp32, 1.07 GB: 493 us with 32 bytes a
// lane in two stores past the caches, 237 so).
template <class T, bool kStream> __global__ __launch_bounds__(kBlock) void dequantize_kernel(MxArgs a, uint32_t first) {
    constexpr int kV = kPerVec<T>, kChunks = kMxBlock / kV;     // of a block
    using Codes = std::conditional_t<kV == 8, uint32_t, uint16_t>;
    const Place p = place_of(a, first);
    const int block = p.chunk / kChunks, padded = (a.blocks + 3) / 4 * 4, count = a.width - p.chunk * kV;
    if (p.row >= a.rows || count <= 0) return;
    const uint32_t codes = reinterpret_cast<const Codes*>(a.codes_in)[p.row * a.blocks * kChunks + p.chunk];
    const float scale = mx_scale(a.scales_in[p.row * padded + block]);
    T* out = static_cast<T*>(a.out) + p.row * a.stride + p.chunk * kV;
    store_some<kStream>(out, mx_values<T>(codes, scale, false), count);
}

// Threads across a row: a power of two of its chunks, `each` a block, or whole workgroups of them.
void spread(MxArgs& a, int each) {
    const int chunks = (a.blocks + 3) / 4 * 4 * each;
    a.lanes = 16;
    while (a.lanes < kBlock && a.lanes < chunks) a.lanes *= 2;
    a.parts = (chunks + kBlock - 1) / kBlock;
}

int64_t blocks_of(const MxArgs& a) {
    return a.parts > 1 ? a.rows * a.parts : (a.rows + kBlock / a.lanes - 1) / (kBlock / a.lanes);
}

int check_mx(const std::string& what, int64_t rows, int64_t width, int64_t stride, int dtype) {
    if (!known_dtype(dtype)) return fail(what + ": dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    if (rows < 0 || rows > (int64_t{1} << 31) - 1) return fail(what + ": rows must be within 0..2^31 - 1");
    if (width < 1 || width > kMaxWidth) return fail(what + ": width must be within 1..2^20");
    if (rows > 0 && stride < width) return fail(what + ": rows overlap (a stride below the row's width)");
    return 0;
}

int check_codes(const std::string& what, const uint8_t* codes, const uint8_t* scales) {
    if (!codes || !scales) return fail(what + ": null pointer");
    if (reinterpret_cast<uintptr_t>(codes) % 16 || reinterpret_cast<uintptr_t>(scales) % 4)
        return fail(what + ": codes must be 16-byte and scales 4-byte aligned");
    return 0;
}

}  // namespace
}  // namespace odie

using namespace odie;

ODIE_API int odie_mx_quantize(const void* x, int64_t x_stride, int64_t rows, int64_t width, int dtype, uint8_t* codes,
                              uint8_t* scales, uint64_t stream) {
    const std::string what = "odie_mx_quantize";
    if (check_mx(what, rows, width, x_stride, dtype)) return -1;
    if (rows == 0) return 0;
    if (!x) return fail(what + ": null pointer");
    if (check_codes(what, codes, scales)) return -1;
    MxArgs a{};
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    a.stride = x_stride;
    a.rows = rows;
    a.width = static_cast<int>(width);
    a.blocks = static_cast<int>(mx_blocks(width));
    spread(a, kLanesOfBlock);
    return with_dtype(dtype, [&](auto t) -> int {
        in_launches(blocks_of(a), kBlock, [&](uint32_t first, uint32_t count) {
            quantize_kernel<decltype(t)><<<count, kBlock, 0, as_stream(stream)>>>(a, first);
        });
        return check_launch("quantize");
    });
}

ODIE_API int odie_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t width, int dtype,
                                void* out, int64_t out_stride, uint64_t stream) {
    const std::string what = "odie_mx_dequantize";
    if (check_mx(what, rows, width, out_stride, dtype)) return -1;
    if (rows == 0) return 0;
    if (!out) return fail(what + ": null pointer");
    if (check_codes(what, codes, scales)) return -1;
    MxArgs a{};
    a.out = out;
    a.codes_in = codes;
    a.scales_in = scales;
    a.stride = out_stride;
    a.rows = rows;
    a.width = static_cast<int>(width);
    a.blocks = static_cast<int>(mx_blocks(width));
    spread(a, dtype == ODIE_F32 ? 8 : 4);       // of 16 bytes
    return with_dtype(dtype, [&](auto t) -> int {
        with_flag(rows * width * dtype_bytes(dtype) >= kStreamBytes, [&](auto far) {
            in_launches(blocks_of(a), kBlock, [&](uint32_t first, uint32_t count) {
                dequantize_kernel<decltype(t), far><<<count, kBlock, 0, as_stream(stream)>>>(a, first);
            });
        });
        return check_launch("dequantize");
    });
}
