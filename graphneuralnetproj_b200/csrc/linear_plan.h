// How the tiles of a linear layer are shared out between thread blocks (linear_kernel.cuh).
//
// The product is a list of output tiles, each `kb` k-blocks deep (a k-block here is
// one ring stage of the kernel).  `workers` blocks (or
// pairs of blocks) run at the same time, one per SM (pair of SMs).  Tiles are dealt out whole, worker c taking tiles
// c, c + workers, ...; what does not fill a last round -- or everything, where there are fewer tiles than workers, as
// for a few tokens -- can instead be cut into equal runs of k-blocks, one run per worker.  A run then covers the end of
// one tile and perhaps the beginning of the next; the pieces of a tile are parked as fp32 in numbered slots of the
// workspace and added in worker order by whichever of its workers comes last.  Everything is computed from the sizes
// by every role of every block for itself (group sizes are known on the device only), and the sums do not depend on
// which worker came last.
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
    int rest;     // tiles whole .. whole + rest - 1 are cut into runs of k-blocks
    int cutters;  // workers 0 .. cutters - 1 get a run each
};

struct LinearSegment {
    int tile;         // < 0: no such segment
    int kb0, kb1;     // its k-blocks
    int slot;         // where a piece is parked; < 0: the tile is whole
    int first, last;  // workers that hold the pieces of the tile
};

constexpr int kMaxPieces = 16;  // pieces of one tile: bounds what the last worker has to add up
constexpr int kMinRun    = 2;   // k-blocks a run has at least

// overhead: what parking and adding a piece costs, in k-blocks; < 0: no workspace, nothing is cut
SPMM_B200_HD LinearPartition make_linear_partition(int tiles, int kb, int workers, int overhead)
{
    LinearPartition p;
    p.kb      = kb;
    p.workers = workers;
    p.rest    = tiles % workers;
    p.whole   = tiles - p.rest;
    p.cutters = 0;
    if (p.rest > 0 && overhead >= 0) {
        const int64_t units   = static_cast<int64_t>(p.rest) * kb;
        int64_t       cutters = units / kMinRun;
        if (cutters > static_cast<int64_t>(p.rest) * kMaxPieces)
            cutters = static_cast<int64_t>(p.rest) * kMaxPieces;
        if (cutters > workers)
            cutters = workers;
        if (cutters > p.rest && (units + cutters - 1) / cutters + overhead < kb)
            p.cutters = static_cast<int>(cutters);
    }
    if (p.cutters == 0) {
        p.whole = tiles;
        p.rest  = 0;
    }
    return p;
}

// The worker whose run holds k-block `unit` of the `units` that are cut.
SPMM_B200_HD int linear_cutter_of(const LinearPartition& p, int64_t unit)
{
    const int64_t units = static_cast<int64_t>(p.rest) * p.kb;
    return static_cast<int>(((unit + 1) * p.cutters - 1) / units);
}

// Segment i (0, 1, ...) of a worker.
SPMM_B200_HD LinearSegment linear_segment(const LinearPartition& p, int worker, int i)
{
    LinearSegment s;
    s.tile = -1;
    s.kb0 = 0, s.kb1 = p.kb;
    s.slot = -1, s.first = s.last = worker;
    const int rounds = worker < p.whole ? (p.whole - worker - 1) / p.workers + 1 : 0;
    if (i < rounds) {
        s.tile = worker + i * p.workers;
        return s;
    }
    const int part = i - rounds;  // a run covers two tiles at most: there are no fewer cutters than tiles to cut
    if (worker >= p.cutters || part > 1)
        return s;
    const int64_t units = static_cast<int64_t>(p.rest) * p.kb;
    const int64_t u0 = worker * units / p.cutters, u1 = (worker + 1) * units / p.cutters;
    const int     t = static_cast<int>(u0 / p.kb) + part;
    const int64_t begin = static_cast<int64_t>(t) * p.kb, end = begin + p.kb;
    if (u1 <= begin)
        return s;
    s.tile  = p.whole + t;
    s.kb0   = part == 0 ? static_cast<int>(u0 - begin) : 0;
    s.kb1   = static_cast<int>((u1 < end ? u1 : end) - begin);
    s.first = linear_cutter_of(p, begin);
    s.last  = linear_cutter_of(p, end - 1);
    if (s.first != s.last)
        s.slot = 2 * worker + part;
    return s;
}

// The slot in which worker `w` parks its piece of the tile that segment `s` belongs to.
SPMM_B200_HD int linear_slot_of(const LinearPartition& p, const LinearSegment& s, int w)
{
    const int64_t units = static_cast<int64_t>(p.rest) * p.kb;
    return 2 * w + (w * units / p.cutters < static_cast<int64_t>(s.tile - p.whole) * p.kb ? 1 : 0);
}

}  // namespace spmm_b200
