// What a CTA of the gated block leaves where one of its waits has run out (plain C++, no CUDA: the CPU tests compile this file on its own).
#pragma once
#ifdef __CUDACC__
#define PL_GIVE_UP __host__ __device__ __forceinline__
#else
#define PL_GIVE_UP inline
#endif

namespace pl {

struct GatedTiles {          // of a CTA: `first`, and every `step`-th one after it, of `tile` rows each
    long long rows, first, step;
    int tile;
};
template <typename T>
struct GatedRows {           // an output with a row for each of x; to: NULL where there is none
    T* to;
    int width;
};

// `value` to all rows of the CTA's tiles, in each of the outputs that it writes: a part of them may be there already, others never will be.
template <typename T, int OUTPUTS>
PL_GIVE_UP void give_up(const GatedRows<T> (&outputs)[OUTPUTS], const GatedTiles& t, T value, int thread, int threads) {
    for (const GatedRows<T>& o : outputs) {
        if (!o.to) continue;
        for (long long row0 = t.first * t.tile; row0 < t.rows; row0 += t.step * t.tile) {
            const long long left = t.rows - row0, count = (left < t.tile ? left : t.tile) * o.width;
            for (long long i = thread; i < count; i += threads) o.to[row0 * o.width + i] = value;
        }
    }
}

}  // namespace pl
