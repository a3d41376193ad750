// Prints the library's planning of a streamed product: "ks slots chunks room" for the arguments row tiles, units, the group size (0 for down products), experts, topk,
// tokens, blocks.
#include "w4_plan.h"
#include <cstdio>
#include <cstdlib>

int main(int argc, char** argv) {
    if (argc != 8) return 2;
    int v[7];
    for (int i = 0; i < 7; ++i) v[i] = std::atoi(argv[i + 1]);
    const int uw = v[2] > 0 ? vela::w4::up_units(v[2]) : 1;
    const vela::w4::Split s = vela::w4::plan(v[1], uw, vela::w4::run_length(v[0], v[3], v[4], v[5], v[6]));
    std::printf("%d %d %d %d\n", s.ks, s.slots, s.chunks, vela::w4::ROOM);
    return 0;
}
