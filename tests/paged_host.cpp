// The division of a paged batch into tiles (tritify_amd/csrc/kt_paged.h) built for the host with g++, a wave's ballots
// worked out lane by lane, for tests/test_paged_tiles.py.
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <vector>

using std::min;

static struct {
    unsigned x;
} threadIdx;

// Each lane runs the function from the start; at the first ballot whose mask is not known yet it hands its bit over.
struct Vote {
    bool bit;
};
static std::vector<uint64_t> masks;
static size_t ballots;
static uint64_t __ballot(bool p) {
    if (ballots == masks.size()) throw Vote{p};
    return masks[ballots++];
}
static int __popcll(uint64_t x) { return __builtin_popcountll(x); }

#include "kt_paged.h"

extern "C" int paged_tile_seq(const int32_t* row_start, int seqs, int tokens, int t, int mul, int step, int per, int* first) {
    kt::Paged a = {};
    a.row_start = row_start, a.seqs = seqs, a.tokens = tokens;
    masks.clear();
    for (;;) {
        uint64_t mask = 0;
        int b = 0;
        bool done = false;
        for (unsigned lane = 0; lane < 64; lane++) {
            threadIdx.x = lane, ballots = 0;
            try {
                b = kt::pg_tile_seq(a, t, mul, step, per, first);
                done = true;
            } catch (const Vote& v) {
                mask |= (uint64_t)v.bit << lane;
            }
        }
        if (done) return b;
        masks.push_back(mask);
    }
}
