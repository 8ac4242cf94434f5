// Stable sort of bucket numbers (sort.hip), for the callers inside the library.
#pragma once
#include "common.h"

namespace odie {

struct SortKeys {
    const void* keys;   // int32 or int64 [n]; a key outside [0, buckets) sorts as `buckets`
    int bytes;          // 4 or 8
    int64_t n;
    int64_t buckets;
};

struct SortOut {
    int32_t* order;     // [n] input position of each sorted place, or null
    int2* pairs;        // [n] (input position, bucket) of each sorted place, or null
    int32_t* sorted;    // [n] bucket of each sorted place, or null
    int32_t* slots;     // [n] sorted place of each input position, -1 where its key is no bucket, or null
    int32_t* offsets;   // [buckets + 1] first place of each bucket, then that of the keys without one, or null
};

int check_sort(const char* what, const SortKeys& k);
int64_t sort_workspace(int64_t n, int64_t buckets);
int launch_sort(const SortKeys& k, const SortOut& out, void* workspace, hipStream_t stream);

}  // namespace odie
