"""How the steps of a shared prefix's tiles of 256 rows are dealt out (csrc/qr_deal.h), without a GPU: the plan's arithmetic and the workgroups', compiled for the host and gone
through share by share.  The cut is made for a hinted length; the prefix may have any."""
import ctypes
import pathlib
import shutil
import subprocess

import pytest

from quarot_amd import _lib

CSRC = pathlib.Path(__file__).resolve().parent.parent / "quarot_amd" / "csrc"
WALK = r"""
#include "qr_deal.h"
#include <vector>
// What goes wrong with a cut of `tiles` tiles for `hinted` steps (0: no hint) where a tile has `steps`; 0: nothing.  states: of the cut
extern "C" int walk(int64_t tiles, int64_t hinted, int steps, int64_t cus, int* states) {
    const DealtCut cut = dealt_cut(tiles, hinted, cus);
    *states = (int)cut.states;
    if (cut.states < 1 || cut.states > kMostStates || cut.shares < 1) return 1;
    std::vector<int64_t> next(tiles, 0);                   // steps that have been done, from the tile's first on
    std::vector<uint64_t> written(tiles, 0);
    const int shares = dealt_shares(tiles, steps, (int)cut.shares);
    for (int share = 0; share < cut.shares; ++share) {
        DealtPiece p;
        for (int done = 0; dealt_piece(tiles, steps, shares, share, done, p); done += p.end - p.first) {
            if (p.tile < 0 || p.tile >= tiles || p.first < 0 || p.end <= p.first || p.end > steps) return 2;
            if (p.first != next[p.tile]) return 3;
            next[p.tile] = p.end;
            if (p.state < 0 || p.state >= cut.states) return 4;                // (a state beyond the row's is the next row's first, or behind the workspace)
            if (written[p.tile] >> p.state & 1) return 5;
            written[p.tile] |= (uint64_t)1 << p.state;
        }
    }
    for (int64_t t = 0; t < tiles; ++t) {
        if (next[t] != steps) return 6;
        if (written[t] & (written[t] + 1)) return 7;       // (those behind the last one are marked empty, a state between them would be what the workspace held)
    }
    return 0;
}
// the first fault over all tiles and hinted steps up to those given and prefixes as long as hinted, and shorter and longer: {fault, tiles, hinted, steps}
extern "C" int walk_all(int most_tiles, int most_steps, int64_t cus, int* at) {
    int states;
    for (int tiles = 1; tiles <= most_tiles; ++tiles)
        for (int hinted = 0; hinted <= most_steps; ++hinted) {
            const int real[] = {hinted, hinted - 1, hinted + 1, 2 * hinted + 3, hinted / 2, hinted / 5, hinted / 17, 1, 2, 3, 100, 157};
            for (const int steps : real)
                if (steps >= 1) {
                    const int fault = walk(tiles, hinted, steps, cus, &states);
                    if (fault) return at[0] = tiles, at[1] = hinted, at[2] = steps, fault;
                }
        }
    return 0;
}
"""


@pytest.fixture(scope="module")
def shares(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("needs g++")
    at = tmp_path_factory.mktemp("shares")
    (at / "walk.cpp").write_text(WALK)
    subprocess.run(["g++", "-O2", "-shared", "-fPIC", "-std=c++17", "-D__host__=", "-D__device__=", "-D__forceinline__=inline", f"-I{CSRC}", "walk.cpp", "-o", "walk.so"],
                   cwd=at, check=True)
    lib = ctypes.CDLL(str(at / "walk.so"))
    lib.walk.argtypes = (ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int64, ctypes.POINTER(ctypes.c_int))
    lib.walk_all.argtypes = (ctypes.c_int, ctypes.c_int, ctypes.c_int64, ctypes.POINTER(ctypes.c_int))
    return lib


@pytest.mark.parametrize("tiles,hinted", [(8, 157), (8, 159), (7, 157), (7, 158), (5, 158), (4, 159), (3, 159)])
def test_a_tile_has_no_more_states_than_its_rows(shares, tiles, hinted):
    """31 shares and a fraction to a tile touch 33 of its states' places: one more than a row has."""
    states = ctypes.c_int()
    for steps in (hinted, 100, 1000, 2 * hinted):
        assert shares.walk(tiles, hinted, steps, 256, ctypes.byref(states)) == 0 and states.value <= 32, steps


@pytest.mark.parametrize("tiles,hinted,steps", [(8, 256, 16), (16, 125, 10), (1, 20, 2), (8, 0, 3), (64, 0, 2), (3, 1 << 20, 5)])
def test_a_prefix_shorter_than_its_hint_leaves_no_state_out(shares, tiles, hinted, steps):
    """More workgroups than steps: those without any may not have states between a tile's others."""
    states = ctypes.c_int()
    assert shares.walk(tiles, hinted, steps, 256, ctypes.byref(states)) == 0


@pytest.mark.parametrize("cus,most_tiles,most_steps", [(256, 66, 260), (256, 300, 24), (304, 24, 260), (64, 70, 170), (1, 20, 200)])
def test_all_steps_are_done_once_and_into_states_of_their_rows(shares, cus, most_tiles, most_steps):
    at = (ctypes.c_int * 3)()
    assert shares.walk_all(most_tiles, most_steps, cus, at) == 0, list(at)


def test_the_workspace_holds_the_states_of_the_cut(shares):
    """32 sequences of one token, 64 heads on 8, fp16 pages, a prefix of 10000: a state for each of a tile's shares (their own launch has none)."""
    states = ctypes.c_int()
    for length in (9985, 10000, 10048, 10113, 10176):
        assert shares.walk(8, -(-length // 64), -(-length // 64), 256, ctypes.byref(states)) == 0
        assert _lib.lib().qr_batch_shared_workspace_bytes(1, 32, 64, 8, 32, 1, 100, 0, 0, 1, length) == 32 * 64 * 528 * states.value, length
