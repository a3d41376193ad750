// Host planning of the streamed products of w4_stream.cuh: how a block splits a row tile's columns.  No CUDA in here.
#pragma once
#include <algorithm>
#include <cmath>

namespace vela {
namespace w4 {

constexpr int WARPS = 16;                 // of a block; one block on each SM
constexpr int ROOM = 96;                  // columns times rounds whose sums a block's shared memory holds

// ks warps share out the units (128 columns) of a row tile, uw to each at a time (a chunk; several where there are more), and the
// block takes slots = WARPS / ks row tiles in a round.
struct Split { int ks, slots, chunks; };
// The split with the least time for runs of about nrow row tiles: a chunk costs its rounds and about two more to bring the
// activations.
inline Split plan(int nu, int uw, int nrow) {
    Split best{1, WARPS, nu};
    long long cost = 0;
    for (int ks = 1; ks <= WARPS && (ks == 1 || (ks - 1) * uw < nu); ++ks) {
        const Split s{ks, WARPS / ks, (nu + ks * uw - 1) / (ks * uw)};
        const long long c = (long long)((nrow + s.slots - 1) / s.slots + 2) * s.chunks;
        if (ks == 1 || c < cost) { best = s; cost = c; }
    }
    return best;
}
// Row tiles of one expert that a block has, on average over as many experts as the tokens reach: E experts of row_tiles, topk of
// them for each token, blocks of the grid.
inline int run_length(int row_tiles, int E, int topk, int tokens, int blocks) {
    const double experts = E * (1 - std::pow(1 - double(topk) / E, tokens));
    return std::min(row_tiles, std::max(1, int(experts * row_tiles / blocks)));
}
// Units of a row tile that a warp takes in the up phase: two share their sums' way to shared memory, but with four scales for each
// the registers spill (32 tokens, 32 experts of 4096 x 1536: groups of 64 take 118 us with two and 122 with one, groups of 32 181
// and 149).
constexpr int up_units(int fold) { return fold >= 64 ? 2 : 1; }

}  // namespace w4
}  // namespace vela
