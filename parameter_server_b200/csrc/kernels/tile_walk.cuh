// How the CTA pairs of a persistent GEMM share its tiles.
//
// Whole waves of tiles are dealt out one by one. What is left over (fewer tiles than pairs, or all of them if there are
// few) is cut along the contraction: the k-steps of these tiles, laid end to end, are dealt in equal runs of `len`, so that
// every pair ends at about the same time. A tile that is shared this way meets in global memory: every pair stores its fp32
// partial tile, and whoever finds that the others are there adds all of them in run order (whichever pair it is, the sum is
// the same) and runs the epilogue. Nobody waits for anybody. The runs come first, so that the traffic of the partial tiles
// hides behind the whole tiles.
#pragma once
#include <cuda_runtime.h>

namespace psb {

namespace {

constexpr int kMaxPairs = 74;     // 148 SMs
constexpr int kMaxRuns = 8;       // of one shared tile: bounds the partial tiles that its last pair has to add

struct TileGrid {
    int m_tiles, n_tiles, k_steps;
    int pairs;      // launched
    int shared;     // tiles [0, shared) are cut into runs
    int len;        // k-steps of a run
    int group;      // m-tiles that are walked together: with 8 the tiles in flight form a block of about 8 x 9, whose rows of A
                    // and columns of B come from HBM once; with 1 the walk goes along n, for a B that stays in L2 as a whole
};

struct Tile {
    int m, n;             // tile coordinates
    int k0, nk;           // k-steps
    int index;            // shared tile: its number
    int runs, run;        // shared tile: how many runs it has (1: it is whole) and which one this is
    int first;            // pair that has run 0
    int slot;             // which of this pair's two places for partial tiles
};

struct TileWalk {
    int pair, pos, end, whole;
    __device__ __forceinline__ TileWalk(const TileGrid& g, int pair_index) : pair(pair_index) {
        const int total = g.shared * g.k_steps;
        pos = min(pair * g.len, total);
        end = min(pos + g.len, total);
        whole = g.shared + pair;
    }
    __device__ __forceinline__ bool next(const TileGrid& g, Tile& t) {
        int index;
        if (pos < end) {
            index = pos / g.k_steps;
            const int start = index * g.k_steps, lim = min(end, start + g.k_steps);
            t.k0 = pos - start;
            t.nk = lim - pos;
            t.first = start / g.len;
            t.runs = (start + g.k_steps - 1) / g.len - t.first + 1;
            t.run = pair - t.first;
            t.slot = pos == pair * g.len ? 0 : 1;
            t.index = index;
            pos = lim;
        } else {
            if (whole >= g.m_tiles * g.n_tiles) return false;
            index = whole;
            whole += g.pairs;
            t.k0 = 0;
            t.nk = g.k_steps;
            t.runs = 1;
            t.run = t.first = t.slot = t.index = 0;
        }
        const int per_group = g.group * g.n_tiles;
        const int group = index / per_group, in = index - group * per_group;
        const int height = min(g.group, g.m_tiles - group * g.group);
        t.n = in / height;
        t.m = group * g.group + in - t.n * height;
        return true;
    }
    // the slot of run `r` of the tile (its pair's first place, or the second if the pair began in an earlier tile)
    static __device__ __forceinline__ int slot_of(const TileGrid& g, const Tile& t, int r) {
        return (t.first + r) * g.len >= t.index * g.k_steps ? 0 : 1;
    }
};

// Cutting pays when it shortens the last wave by more than the partial tiles cost (a tile's way through memory and its joining
// take about as long as `min_gain` k-steps), and by a quarter of the whole at least: pairs that run through different parts of
// the contraction share nothing in L2, and a GPU at its power limit makes up for idle SMs with its clock (192 tiles of 256
// k-steps on 74 pairs, back to back: 347 us in three whole waves, 369 with the third one cut).
inline TileGrid plan_tiles(int m_tiles, int n_tiles, int k_steps, int max_pairs, int min_gain, int group) {
    TileGrid g;
    g.group = group;
    g.m_tiles = m_tiles;
    g.n_tiles = n_tiles;
    g.k_steps = k_steps;
    const int tiles = m_tiles * n_tiles;
    g.pairs = tiles < max_pairs ? tiles : max_pairs;
    g.shared = 0;
    g.len = 1;
    const int rest = tiles % max_pairs;
    if (rest == 0) return g;
    int len = (int)(((long long)rest * k_steps + max_pairs - 1) / max_pairs);
    const int least = (k_steps + kMaxRuns - 1) / kMaxRuns;
    if (len < least) len = least;
    if (len < 4) len = 4;
    const int waves = tiles / max_pairs + 1;
    if (k_steps - len < min_gain || 4 * (k_steps - len) < waves * k_steps) return g;
    g.shared = rest;
    g.len = len;
    const int workers = (int)(((long long)rest * k_steps + len - 1) / len);
    g.pairs = tiles > max_pairs ? max_pairs : (workers < max_pairs ? workers : max_pairs);
    return g;
}

}  // namespace

}  // namespace psb
