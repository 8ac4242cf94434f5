// Stable counting sort of bucket numbers: rows by expert, samples by table row.
//
// Keys are split into digits of at most 11 bits (one pass up to 2047 buckets), least significant first.
// A pass cuts the keys into one part per workgroup:
//   count    each workgroup counts its part's digits in LDS -> table[digit][part]
//   scan     one workgroup per digit turns its row of the table into running sums and leaves its total
//   scatter  each workgroup finds every digit's first place (a scan of the totals), counts again per
//            wave, and walks its keys 64 at a time: lanes that share a digit take consecutive
//            places (one ballot per bit of the digit), a running count in LDS carries on.
// 4M keys in two passes 91 us: scatter 32 each, whose stores of 8 bytes go where the digits say; count 8, scan 5.
// 131072 keys in one pass 12 us, most of it the three launches' latency.  (Scattering through LDS so that stores are runs:
// 64 -> 53 us with few digits, 20 -> 37 with 1025.)
// No global atomics: the same keys give the same places every time.  Up to 4096 keys one workgroup does
// all of it in LDS, in one launch.
#include "sort.h"
#include "elements.h"

namespace odie {
namespace {

constexpr int kDigitBits = 11;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortBlock = 512, kSortWaves = kSortBlock / 64;
constexpr int kMaxParts = 2048;

constexpr int kSmall = 4096;
constexpr int kSmallBlock = 1024, kSmallWaves = kSmallBlock / 64;
constexpr int kSmallBits = 8;

__device__ inline uint32_t read_key(const void* keys, int bytes, int64_t i, uint32_t buckets) {
    if (bytes == 8) {
        const int64_t k = static_cast<const int64_t*>(keys)[i];
        return static_cast<uint64_t>(k) < buckets ? static_cast<uint32_t>(k) : buckets;
    }
    const uint32_t k = static_cast<const uint32_t*>(keys)[i];
    return k < buckets ? k : buckets;
}

// The lanes of `active` whose digit is this lane's.
__device__ inline uint64_t same_digit(uint32_t digit, int bits, uint64_t active) {
    uint64_t same = active;
    for (int b = 0; b < bits; ++b) {
        const bool set = digit >> b & 1;
        const uint64_t with = __ballot(set);
        same &= set ? with : ~with;
    }
    return same;
}

__device__ inline int lanes_below(uint64_t mask, int lane) { return __popcll(mask & ((uint64_t{1} << lane) - 1)); }

// Exclusive sum over the wave.
__device__ inline uint32_t wave_exclusive(uint32_t x, int lane, uint32_t& total) {
    uint32_t sum = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    total = __shfl(sum, 63);
    return sum - x;
}

// In-place exclusive scan of `count` LDS words by a workgroup of kThreads.
template <int kThreads> __device__ inline void block_scan(uint32_t* data, int count, uint32_t* wave_sums) {
    const int lane = static_cast<int>(threadIdx.x % 64), wave = static_cast<int>(threadIdx.x / 64);
    const int each = (count + kThreads - 1) / kThreads, begin = static_cast<int>(threadIdx.x) * each;
    uint32_t sum = 0;
    for (int i = 0; i < each && begin + i < count; ++i) sum += data[begin + i];
    uint32_t total;
    uint32_t before = wave_exclusive(sum, lane, total);
    if (lane == 0) wave_sums[wave] = total;
    __syncthreads();
    for (int w = 0; w < wave; ++w) before += wave_sums[w];
    for (int i = 0; i < each && begin + i < count; ++i) {
        const uint32_t x = data[begin + i];
        data[begin + i] = before;
        before += x;
    }
    __syncthreads();
}

struct SmallArgs {
    SortKeys in;
    SortOut out;
    int bits;
};

__global__ __launch_bounds__(kSmallBlock) void small_sort_kernel(SmallArgs a) {
    __shared__ uint32_t key[2][kSmall];
    __shared__ uint16_t from[2][kSmall];
    __shared__ uint32_t count[(1 << kSmallBits) * kSmallWaves];   // [digit][wave]
    __shared__ uint32_t wave_sums[kSmallWaves];
    const int n = static_cast<int>(a.in.n), lane = static_cast<int>(threadIdx.x % 64);
    const int wave = static_cast<int>(threadIdx.x / 64);
    const uint32_t buckets = static_cast<uint32_t>(a.in.buckets);
    for (int i = threadIdx.x; i < n; i += kSmallBlock) {
        key[0][i] = read_key(a.in.keys, a.in.bytes, i, buckets);
        from[0][i] = static_cast<uint16_t>(i);
    }
    const int rounds = (n + kSmallBlock - 1) / kSmallBlock;
    const int first = wave * rounds * 64;
    int now = 0;
    for (int shift = 0; shift < a.bits; shift += kSmallBits) {
        const int bits = a.bits - shift < kSmallBits ? a.bits - shift : kSmallBits;
        const uint32_t mask = (1u << bits) - 1;
        for (int i = threadIdx.x; i < (kSmallWaves << bits); i += kSmallBlock) count[i] = 0;
        __syncthreads();
        for (int r = 0; r < rounds; ++r) {
            const int i = first + r * 64 + lane;
            if (i < n) atomicAdd(&count[(key[now][i] >> shift & mask) * kSmallWaves + wave], 1u);
        }
        __syncthreads();
        block_scan<kSmallBlock>(count, kSmallWaves << bits, wave_sums);
        for (int r = 0; r < rounds; ++r) {
            const int i = first + r * 64 + lane;
            const bool valid = i < n;
            const uint32_t k = valid ? key[now][i] : 0u;
            const uint32_t digit = k >> shift & mask;
            const uint64_t same = same_digit(digit, bits, __ballot(valid));
            const uint32_t at = valid ? count[digit * kSmallWaves + wave] : 0u;
            const int rank = lanes_below(same, lane);
            wave_fence();
            if (valid && rank == 0) count[digit * kSmallWaves + wave] = at + __popcll(same);
            wave_fence();
            if (valid) {
                key[now ^ 1][at + rank] = k;
                from[now ^ 1][at + rank] = from[now][i];
            }
        }
        now ^= 1;
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += kSmallBlock) {
        const int f = from[now][i];
        if (a.out.order) a.out.order[i] = f;
        if (a.out.pairs) a.out.pairs[i] = make_int2(f, static_cast<int>(key[now][i]));
        if (a.out.sorted) a.out.sorted[i] = static_cast<int32_t>(key[now][i]);
        if (a.out.slots) a.out.slots[f] = key[now][i] < buckets ? i : -1;
    }
    if (!a.out.offsets) return;
    for (int64_t v = threadIdx.x; v <= a.in.buckets; v += kSmallBlock) {
        int low = 0, high = n;   // the first place whose key is at least v
        while (low < high) {
            const int mid = (low + high) / 2;
            if (key[now][mid] < v) low = mid + 1; else high = mid;
        }
        a.out.offsets[v] = low;
    }
}

struct PassArgs {
    const void* raw;          // the caller's keys (first pass)
    int raw_bytes;
    const uint2* pairs;       // later passes: (input position, key) so far
    uint2* pairs_out;         // earlier passes
    uint32_t* table;          // [digits][parts]
    uint32_t* totals;         // [digits]
    SortOut out;              // last pass
    int64_t n;
    int64_t part;             // keys a workgroup (a multiple of kSortBlock)
    uint32_t parts;
    uint32_t buckets;
    int shift, bits, digits;
    bool last, only;          // only: the sole pass, digits are buckets
};

constexpr int kHeld = 8;   // keys a lane loads together: 4M in two passes 118 -> 91 us against one at a time

// (input position, key) of places i, i + 64, ... below end, which is past i's wave; places from end on repeat the last.
__device__ inline void load_pairs(const PassArgs& a, int64_t i, int64_t end, uint2 pair[kHeld]) {
    auto at = [&](int u) { return i + u * 64 < end ? i + u * 64 : end - 1; };
    if (!a.raw) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) pair[u] = a.pairs[at(u)];
    } else if (a.raw_bytes == 8) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) pair[u] = make_uint2(static_cast<uint32_t>(at(u)), read_key(a.raw, 8, at(u), a.buckets));
    } else {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) pair[u] = make_uint2(static_cast<uint32_t>(at(u)), read_key(a.raw, 4, at(u), a.buckets));
    }
}

// Counts the digits of the wave's places begin..end - 1 in LDS.
__device__ inline void count_digits(const PassArgs& a, int64_t begin, int64_t end, int lane, uint32_t* count) {
    const uint32_t mask = (1u << a.bits) - 1;
    for (int64_t base = begin; base < end; base += 64 * kHeld) {
        uint2 pair[kHeld];
        load_pairs(a, base + lane, end, pair);
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (base + u * 64 + lane < end) atomicAdd(&count[pair[u].y >> a.shift & mask], 1u);
    }
}

__global__ __launch_bounds__(kSortBlock) void count_kernel(PassArgs a) {
    __shared__ uint32_t count[kDigits];
    for (int d = threadIdx.x; d < a.digits; d += kSortBlock) count[d] = 0;
    __syncthreads();
    const int64_t share = a.part / kSortWaves, begin = blockIdx.x * a.part + threadIdx.x / 64 * share;
    const int64_t end = begin + share < a.n ? begin + share : a.n;
    count_digits(a, begin, end, static_cast<int>(threadIdx.x % 64), count);
    __syncthreads();
    for (int d = threadIdx.x; d < a.digits; d += kSortBlock) a.table[static_cast<int64_t>(d) * a.parts + blockIdx.x] = count[d];
}

__global__ __launch_bounds__(256) void scan_kernel(PassArgs a) {
    __shared__ uint32_t row[kMaxParts];
    __shared__ uint32_t wave_sums[4];
    uint32_t* table = a.table + static_cast<int64_t>(blockIdx.x) * a.parts;
    const int parts = static_cast<int>(a.parts);
    for (int p = threadIdx.x; p < parts; p += 256) row[p] = table[p];
    __syncthreads();
    const uint32_t last = row[parts - 1];
    __syncthreads();
    block_scan<256>(row, parts, wave_sums);
    for (int p = threadIdx.x; p < parts; p += 256) table[p] = row[p];
    if (threadIdx.x == 0) a.totals[blockIdx.x] = row[parts - 1] + last;
}

__global__ __launch_bounds__(kSortBlock) void scatter_kernel(PassArgs a) {
    extern __shared__ uint32_t lds[];              // as much as the digits need: more workgroups a CU
    __shared__ uint32_t wave_sums[kSortWaves];
    uint32_t* const start = lds;                   // first place of each digit
    uint32_t* const next = lds + a.digits;         // [wave][digit]: the next key's
    const int lane = static_cast<int>(threadIdx.x % 64), wave = static_cast<int>(threadIdx.x / 64);
    uint32_t* const own_next = next + wave * a.digits;
    for (int d = threadIdx.x; d < a.digits; d += kSortBlock) {
        start[d] = a.totals[d];
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) next[w * a.digits + d] = 0;
    }
    __syncthreads();
    block_scan<kSortBlock>(start, a.digits, wave_sums);
    const uint32_t mask = (1u << a.bits) - 1;
    const int64_t share = a.part / kSortWaves;
    const int64_t begin = blockIdx.x * a.part + wave * share, end = begin + share < a.n ? begin + share : a.n;
    count_digits(a, begin, end, lane, own_next);
    __syncthreads();
    for (int d = threadIdx.x; d < a.digits; d += kSortBlock) {
        uint32_t place = start[d] + a.table[static_cast<int64_t>(d) * a.parts + blockIdx.x];
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const uint32_t own = next[w * a.digits + d];
            next[w * a.digits + d] = place;
            place += own;
        }
    }
    if (a.only && a.out.offsets && blockIdx.x == 0)
        for (int d = threadIdx.x; d < a.digits; d += kSortBlock) a.out.offsets[d] = static_cast<int32_t>(start[d]);
    __syncthreads();
    for (int64_t base = begin; base < end; base += 64 * kHeld) {
        uint2 pair[kHeld];
        load_pairs(a, base + lane, end, pair);
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            if (base + u * 64 >= end) break;
            const bool valid = base + u * 64 + lane < end;
            const uint32_t k = pair[u].y, f = pair[u].x;
            const uint32_t digit = k >> a.shift & mask;
            const uint64_t same = same_digit(digit, a.bits, __ballot(valid));
            const uint32_t place = valid ? own_next[digit] : 0u;
            const int rank = lanes_below(same, lane);
            wave_fence();
            if (valid && rank == 0) own_next[digit] = place + __popcll(same);
            wave_fence();
            if (!valid) continue;
            const uint32_t to = place + rank;
            if (!a.last) {
                a.pairs_out[to] = pair[u];
                continue;
            }
            if (a.out.order) a.out.order[to] = static_cast<int32_t>(f);
            if (a.out.pairs) a.out.pairs[to] = make_int2(static_cast<int>(f), static_cast<int>(k));
            if (a.out.sorted) a.out.sorted[to] = static_cast<int32_t>(k);
            if (a.out.slots) a.out.slots[f] = k < a.buckets ? static_cast<int32_t>(to) : -1;
        }
    }
}

// offsets of more buckets than one pass tells apart: the first place whose bucket is at least v.
__global__ __launch_bounds__(256) void offsets_kernel(const uint32_t* sorted, int64_t n, int64_t buckets, int32_t* offsets) {
    const int64_t v = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (v > buckets) return;
    int64_t low = 0, high = n;
    while (low < high) {
        const int64_t mid = (low + high) / 2;
        if (sorted[mid] < v) low = mid + 1; else high = mid;
    }
    offsets[v] = static_cast<int32_t>(low);
}

int key_bits(int64_t buckets) {   // of the numbers 0..buckets
    int bits = 1;
    while (buckets >> bits) ++bits;
    return bits;
}

// Keys a workgroup: enough for two workgroups a CU where there are, at least one round of every wave.
int64_t sort_part(int64_t n) {
    int64_t part = kSortBlock;
    while ((part < 4096 && part * 2 * kCus < n) || part * kMaxParts < n) part *= 2;
    return part;
}

int64_t padded(int64_t words) { return (words + 63) / 64 * 64; }

}  // namespace

int check_sort(const char* what, const SortKeys& k) {
    if (k.bytes != 4 && k.bytes != 8) return fail(std::string(what) + ": keys must be 4 or 8 bytes wide");
    if (k.n < 0 || k.n >= int64_t{1} << 31) return fail(std::string(what) + ": the count must be within 0..2^31 - 1");
    if (k.buckets < 1 || k.buckets >= (int64_t{1} << 31) - 1)
        return fail(std::string(what) + ": the number of buckets must be within 1..2^31 - 2");
    return 0;
}

// 32-bit words: the table and totals of a pass, two arrays of (position, key) for several passes
// (one of them keeps the sorted keys for the offsets).
int64_t sort_workspace(int64_t n, int64_t buckets) {
    if (n <= kSmall) return 0;
    const int bits = key_bits(buckets), passes = (bits + kDigitBits - 1) / kDigitBits;
    const int64_t parts = (n + sort_part(n) - 1) / sort_part(n);
    const int64_t digits = passes == 1 ? buckets + 1 : int64_t{1} << ((bits + passes - 1) / passes);
    return 4 * (padded(digits * parts) + padded(digits) + (passes > 1 ? 4 * padded(n) : 0));
}

int launch_sort(const SortKeys& k, const SortOut& out, void* workspace, hipStream_t stream) {
    if (k.n <= kSmall) {
        small_sort_kernel<<<1, kSmallBlock, 0, stream>>>(SmallArgs{k, out, key_bits(k.buckets)});
        return check_launch("sort");
    }
    const int bits = key_bits(k.buckets), passes = (bits + kDigitBits - 1) / kDigitBits;
    const int width = (bits + passes - 1) / passes;
    PassArgs a{};
    a.n = k.n;
    a.part = sort_part(k.n);
    a.parts = static_cast<uint32_t>((k.n + a.part - 1) / a.part);
    a.buckets = static_cast<uint32_t>(k.buckets);
    a.out = out;
    a.only = passes == 1;
    const int64_t digits = passes == 1 ? k.buckets + 1 : int64_t{1} << width;
    uint32_t* words = static_cast<uint32_t*>(workspace);
    a.table = words;
    a.totals = a.table + padded(digits * a.parts);
    uint2* pairs[2] = {reinterpret_cast<uint2*>(a.totals + padded(digits)),
                       reinterpret_cast<uint2*>(a.totals + padded(digits)) + padded(k.n)};
    for (int pass = 0; pass < passes; ++pass) {
        a.raw = pass == 0 ? k.keys : nullptr;
        a.raw_bytes = k.bytes;
        a.pairs = pairs[(pass + 1) % 2];
        a.last = pass == passes - 1;
        a.pairs_out = pairs[pass % 2];
        a.shift = pass * width;
        a.bits = bits - a.shift < width ? bits - a.shift : width;
        a.digits = static_cast<int>(passes == 1 ? digits : int64_t{1} << a.bits);
        if (a.last && passes > 1 && out.offsets && !out.sorted)   // the offsets read the sorted buckets
            a.out.sorted = reinterpret_cast<int32_t*>(a.pairs_out);
        count_kernel<<<a.parts, kSortBlock, 0, stream>>>(a);
        scan_kernel<<<a.digits, 256, 0, stream>>>(a);
        scatter_kernel<<<a.parts, kSortBlock, (1 + kSortWaves) * a.digits * sizeof(uint32_t), stream>>>(a);
        if (check_launch("sort")) return -1;
    }
    if (passes > 1 && out.offsets) {
        offsets_kernel<<<static_cast<uint32_t>(k.buckets / 256 + 1), 256, 0, stream>>>(
            reinterpret_cast<const uint32_t*>(a.out.sorted), k.n, k.buckets, out.offsets);
        return check_launch("sort offsets");
    }
    return 0;
}

}  // namespace odie

using namespace odie;

ODIE_API int64_t odie_sort_workspace(int64_t n, int64_t buckets) {
    if (check_sort("odie_sort_workspace", SortKeys{nullptr, 4, n, buckets})) return -1;
    return sort_workspace(n, buckets);
}

ODIE_API int odie_sort(const void* keys, int key_bytes, int64_t n, int64_t buckets, int32_t* order, int32_t* sorted,
                       int32_t* slots, int32_t* offsets, void* workspace, int64_t workspace_bytes, uint64_t stream) {
    const SortKeys k{keys, key_bytes, n, buckets};
    if (check_sort("odie_sort", k)) return -1;
    if (n > 0 && (!keys || !order)) return fail("odie_sort: null pointer");
    if (n == 0 && !offsets) return 0;
    const int64_t need = sort_workspace(n, buckets);
    if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
        return fail("odie_sort: needs a 16-byte aligned workspace of " + std::to_string(need) + " bytes");
    return launch_sort(k, SortOut{order, nullptr, sorted, slots, offsets}, workspace, as_stream(stream));
}
