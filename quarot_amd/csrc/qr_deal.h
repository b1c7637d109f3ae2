// How the steps of one shared prefix's tiles of 256 rows are dealt out over a launch's workgroups: the host's cut and the workgroups' own arithmetic, apart from
// everything else so that both can be gone through for all sizes on the CPU.
#pragma once
#include <stdint.h>

constexpr int64_t kMostStates = 32;                        // of a row, of one launch

// The steps of `tiles` tiles lie one behind the other and are cut into equal shares, one to a workgroup; a tile has a state for every share that has steps of it.  Of
// S = q tiles + r shares a tile has q where r is 0, one where S divides the tiles, else q + 2 at most: its bounds, in shares, lie at i S / tiles and (i + 1) S / tiles, and
// between the whole numbers around them are q + 2 shares at most.  That goes for any number of steps: the launch is cut for a hinted one.
struct DealtCut {
    int64_t shares, states;
};
// steps: of a tile, 0: not known.  Five steps to a share at least, a share to a CU at most.
__host__ __device__ __forceinline__ DealtCut dealt_cut(int64_t tiles, int64_t steps, int64_t cus) {
    int64_t shares = steps > 0 && tiles * steps < 5 * cus ? tiles * steps / 5 : cus;
    if (shares < 1) shares = 1;
    if (shares < tiles && 8 * shares > 7 * tiles) shares = tiles;              // (a little more than one tile each)
    int64_t states = shares % tiles == 0 ? shares / tiles : tiles % shares == 0 ? 1 : shares / tiles + 2;
    if (states > kMostStates) {
        // whole shares to a tile, as many as there are states for (31 and a part would need 33)
        states = shares >= kMostStates * tiles ? kMostStates : kMostStates - 1;
        shares = states * tiles;
    }
    return DealtCut{shares, states};
}

// The shares that tiles of `tile_steps` steps are cut into by workgroups for `cut` of them: none is empty, so that a tile's states are 0, 1, ... without a gap whatever length the
// launch was cut for.  (One to a step where there are fewer steps than workgroups; a tile has that many states then, fewer than the cut's.)
__host__ __device__ __forceinline__ int dealt_shares(int64_t tiles, int tile_steps, int cut) {
    const int64_t all = tiles * tile_steps;
    return all < cut ? (int)all : cut;
}

// The piece of share number `share` that begins `done` steps behind its first one: steps first .. end - 1 of a tile, whose state `state` they are; false: the share ends
// there.  A workgroup whose number is not below `shares` has none.
struct DealtPiece {
    int tile, first, end, state;
};
__host__ __device__ __forceinline__ bool dealt_piece(int64_t tiles, int tile_steps, int shares, int share, int done, DealtPiece& p) {
    const int64_t all = tiles * tile_steps, at = all * share / shares + done, end = all * (share + 1) / shares;
    if (share >= shares || at >= end) return false;
    const int64_t tile = at / tile_steps;
    p.tile = (int)tile;
    p.first = (int)(at - tile * tile_steps);
    p.end = end - at < tile_steps - p.first ? p.first + (int)(end - at) : tile_steps;
    p.state = share - (int)(((tile * tile_steps + 1) * shares - 1) / all);     // (the share that has the tile's first step is state 0)
    return true;
}
