// Sequences of different lengths packed one behind the other: rows starts[i] .. starts[i + 1] - 1 of the packed tensors are sequence i.
#pragma once

#include "common.cuh"

namespace puter {

namespace pk {

struct Seqs {
    const int32_t* starts;
    int batch, total, maxLen;
    int* errorFlag;
};

// rows [s0, s1) of sequence b; false (and the flag) where the starts make none
__device__ __forceinline__ bool seq_rows(const Seqs& s, int b, int& s0, int& s1) {
    s0 = s.starts[b];
    s1 = s.starts[b + 1];
    if (s0 < 0 || s1 < s0 || s1 > s.total || s1 - s0 > s.maxLen) {
        atomicExch(s.errorFlag, 1);
        s1 = s0;
        return false;
    }
    return s1 > s0;
}

// the sequence that holds `row`: the last one that starts at or before it
__device__ __forceinline__ int seq_of(const Seqs& s, int row) {
    int a = 0, z = s.batch;
    while (z - a > 1) {
        const int m = (a + z) >> 1;
        if (s.starts[m] <= row) a = m;
        else z = m;
    }
    return a;
}

}  // namespace pk

}  // namespace puter
