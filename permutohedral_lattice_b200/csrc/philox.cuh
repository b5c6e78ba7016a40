// Random words from a counter (Philox4x32-10: Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): four
// words for a counter of 128 bits under a key of 64.  A value's word depends on its place and the caller's key and offset alone, so a
// mask is made again wherever it is needed, in any order, and never stored.
#pragma once
#include "common.cuh"

namespace pl {

struct Dropout {
    u32 threshold;            // a value whose word is below it is dropped; 0: none is
    float scale;              // of those that stay, 1 / (1 - p)
    u64 key, offset;          // where seed is NULL
    const long long* seed;    // device: key, offset
};

// The ten keys of a call's rounds: the same for all values, so made once for all that a thread does.
struct Philox {
    u32 k0[10], k1[10], o0, o1;
    __device__ __forceinline__ explicit Philox(const Dropout& d) {
        const u64 key = d.seed ? (u64)__ldg(d.seed) : d.key, offset = d.seed ? (u64)__ldg(d.seed + 1) : d.offset;
#pragma unroll
        for (int r = 0; r < 10; r++) {
            k0[r] = (u32)key + r * 0x9E3779B9u;
            k1[r] = (u32)(key >> 32) + r * 0xBB67AE85u;
        }
        o0 = (u32)offset, o1 = (u32)(offset >> 32);
    }
    __device__ __forceinline__ uint4 words(u64 quad) const {   // of values 4 quad to 4 quad + 3
        u32 a = (u32)quad, b = (u32)(quad >> 32), c = o0, d = o1;
#pragma unroll
        for (int r = 0; r < 10; r++) {
            const u64 p = (u64)a * 0xD2511F53u, q = (u64)c * 0xCD9E8D57u;
            a = (u32)(q >> 32) ^ b ^ k0[r];
            b = (u32)q;
            c = (u32)(p >> 32) ^ d ^ k1[r];
            d = (u32)p;
        }
        return make_uint4(a, b, c, d);
    }
};

}  // namespace pl
