// slices.h -- how many CTAs of a cluster share the reduction of one tile (host only; gemm_f8.cu,
// rank_ckpt8.cu).
#pragma once

namespace act {

// Slices for `tiles` tiles of nk blocks each, up to `most`: the least rounds of clusters times the blocks
// of a slice and `join`, what starting a cluster and adding its slices takes, counted in blocks.
// one: the cost of not slicing, in blocks too, which is always possible.
// at_once(n): clusters of n CTAs that run at once; 0: the GPU (or the part of it that this process has)
// runs none of that size, so that n is no choice.
template <typename AtOnce>
int best_slices(long tiles, int nk, int most, int join, long one, AtOnce&& at_once) {
    int slices = 1;
    for (int n = 2; n <= most && n <= nk; ++n) {
        const long room = at_once(n);
        if (room < 1) continue;
        const long cost = (tiles + room - 1) / room * ((nk + n - 1) / n + join);
        if (cost < one) {
            one = cost;
            slices = n;
        }
    }
    return slices;
}

}  // namespace act
