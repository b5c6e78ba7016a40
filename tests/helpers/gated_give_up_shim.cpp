// What the CTAs of a gated block leave where their waits have run out (csrc/gated_give_up.h): all threads of a CTA, one after another.
#include "gated_give_up.h"

extern "C" void give_up_as(float* out, int out_width, float* other, int other_width, long long rows, int tile, long long cta, long long ctas, int threads) {
    const pl::GatedRows<float> outputs[2] = {{out, out_width}, {other, other_width}};
    for (int t = 0; t < threads; t++) pl::give_up(outputs, pl::GatedTiles{rows, cta, ctas, tile}, __builtin_nanf(""), t, threads);
}
