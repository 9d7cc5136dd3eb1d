// How the tiles of a linear layer are shared out between thread blocks (linear_kernel.cuh).
//
// The product is a list of output tiles, each `kb` k-blocks deep (a k-block here is one ring stage of the kernel).
// `workers` blocks (or pairs of blocks) run at the same time, one per SM (pair of SMs).  Tiles are dealt out whole, worker c
// taking tiles c, c + workers, ...; of what does not fill a last round -- or of everything, where there are fewer tiles
// than workers, as for a few tokens -- every tile can instead be cut into `parts` runs of k-blocks, one run per worker.  The
// pieces of a tile are parked as fp32 in the workspace, one numbered slot per worker, and added in worker order by whichever of
// them comes last.  Everything is computed from the sizes by every role of every block for itself (group sizes are known on the
// device only), and the sums do not depend on which worker came last.
//
// Equal parts, although (tiles * parts) workers may be fewer than there are: with runs of equal length over all workers, run
// borders lie anywhere in a tile, tiles have more pieces and workers two of them (28 tiles of 56 k-blocks on 74 pairs: 37 us,
// 31 with two parts each on 56 of them; 28 since stores have become wider).
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define SPMM_B200_HD __host__ __device__ __forceinline__
#else
#define SPMM_B200_HD inline
#endif

namespace spmm_b200 {

struct LinearPartition {
    int kb;       // k-blocks per tile
    int workers;  // blocks (pairs) of the launch
    int whole;    // tiles 0 .. whole - 1 are dealt out whole
    int rest;     // tiles whole .. whole + rest - 1 are cut
    int parts;    // into so many runs each
};

struct LinearSegment {
    int tile;         // < 0: no such segment
    int kb0, kb1;     // its k-blocks
    int first, last;  // workers that hold the pieces of the tile (the same one: the tile is whole)
};

constexpr int kMinRun = 2;  // k-blocks a run has at least

struct LinearCutting {
    int overhead;  // what parking and adding the pieces of a tile costs, in k-blocks; < 0: no workspace, nothing is cut
    int pieces;    // of one tile at most: bounds what the last worker has to add up
};

SPMM_B200_HD int linear_min(int a, int b)
{
    return a < b ? a : b;
}

SPMM_B200_HD LinearPartition make_linear_partition(int tiles, int kb, int workers, LinearCutting cut)
{
    LinearPartition p;
    p.kb      = kb;
    p.workers = workers;
    p.rest    = tiles % workers;
    p.whole   = tiles - p.rest;
    p.parts   = 1;
    if (p.rest > 0 && cut.overhead >= 0) {
        // p parts take kb / p for the runs and about 1.4 p for adding the pieces, which the last worker does alone: the sum is
        // smallest near p * p = kb / 1.4 (1 token, 1024 x 9216, 36 k-blocks: 11.2 us in five parts, 13.9 in sixteen)
        int parts = linear_min(workers / p.rest, linear_min(cut.pieces, kb / kMinRun));
        while (parts > 1 && 7 * parts * parts > 5 * kb)
            parts--;
        if (parts > 1 && (kb - 1) / parts + 1 + cut.overhead < kb)
            p.parts = parts;
    }
    if (p.parts == 1) {
        p.whole = tiles;
        p.rest  = 0;
    }
    return p;
}

// Segment i (0, 1, ...) of a worker.
SPMM_B200_HD LinearSegment linear_segment(const LinearPartition& p, int worker, int i)
{
    LinearSegment s;
    s.tile = -1;
    s.kb0 = 0, s.kb1 = p.kb;
    s.first = s.last = worker;
    const int rounds = worker < p.whole ? (p.whole - worker - 1) / p.workers + 1 : 0;
    if (i < rounds) {
        s.tile = worker + i * p.workers;
        return s;
    }
    if (i > rounds || worker >= p.rest * p.parts)
        return s;
    const int t = worker / p.parts, part = worker % p.parts;
    s.tile  = p.whole + t;
    s.kb0   = static_cast<int>(static_cast<int64_t>(p.kb) * part / p.parts);
    s.kb1   = static_cast<int>(static_cast<int64_t>(p.kb) * (part + 1) / p.parts);
    s.first = t * p.parts;
    s.last  = s.first + p.parts - 1;
    return s;
}

}  // namespace spmm_b200
