"""CPU test of the order in which the few-row FP4 kernel's quantizing warps take the K blocks of a CTA (csrc/fp4_deal.h)."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROWS = range(1, 17)
BLOCKS = [1, 2, 3, 4, 5, 7, 8, 9, 12, 15, 16, 17, 24, 31, 32, 33, 48, 64, 65, 130]

PROGRAM = """
#include "%s"
#include <cstdio>
using namespace lyraq::fp4;
int main()
{
    std::printf("%%d %%d\\n", kDealWarps, kDealStages);
    for (int rows = 1; rows <= 16; ++rows) {
        const FewRowsDeal d = few_rows_deal(rows);
        for (int w = 0; w < kDealWarps; ++w) {
            std::printf("%%d %%d %%d", rows, w, d.warps_per_kb);
            for (int v = 0; v < 140; ++v)
                for (int t = 0; t < d.per_visit; ++t) std::printf(" %%d", few_rows_block(d, w, v, t));
            std::printf("\\n");
        }
    }
}
"""


@pytest.fixture(scope="module")
def dealt(tmp_path_factory):
    """(warps, stages, {rows: (warps per K block, K blocks of each warp in its order)})."""
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    at = tmp_path_factory.mktemp("deal")
    (at / "deal.cpp").write_text(PROGRAM % os.path.join(ROOT, "lyradiff_b200", "csrc", "fp4_deal.h"))
    subprocess.run(["g++", "-std=c++17", str(at / "deal.cpp"), "-o", str(at / "deal")], check=True)
    lines = [[int(v) for v in li.split()] for li in subprocess.run([str(at / "deal")], check=True, capture_output=True, text=True).stdout.splitlines()]
    warps, stages = lines[0]
    rows = {}
    for r, w, per, *blocks in lines[1:]:
        rows.setdefault(r, (per, []))[1].append(blocks)
        assert len(rows[r][1]) == w + 1
    return warps, stages, rows


@pytest.mark.parametrize("rows", ROWS)
def test_every_block_is_filled_once_by_each_of_its_warps(dealt, rows):
    warps, _, deal = dealt
    per, order = deal[rows]
    assert warps % per == 0 and 4 * per >= rows and len(order) == warps     # a warp has the place of four rows
    for blocks in BLOCKS:
        filled = [[i for i in o if i < blocks] for o in order]
        for i in range(blocks):
            who = [w for w in range(warps) for j in filled[w] if j == i]
            assert sorted(w % per for w in who) == list(range(per))
        # a warp stops at its first block beyond the end
        assert all(o[:len(f)] == f for o, f in zip(order, filled))


@pytest.mark.parametrize("rows", ROWS)
def test_no_wait_can_pass_early(dealt, rows):
    """Filling block i needs i / stages completions of its stage's barrier, and the wait for them is by parity: it tells that number from one
    less.  So the warp must know of one less already, from its own last wait for that stage (of a new barrier it knows that there are none).  More than
    needed there cannot be: the completion after them takes this block, which this warp fills."""
    _, stages, deal = dealt
    for order in deal[rows][1]:
        seen = {}
        for i in (j for j in order if j < max(BLOCKS)):
            need = i // stages
            assert need - seen.get(i % stages, 0) <= 1, "block %d needs %d completions, %d are known" % (i, need, seen.get(i % stages, 0))
            seen[i % stages] = need


@pytest.mark.parametrize("rows", ROWS)
def test_warps_and_ring_get_through(dealt, rows):
    """The ring simulated: a block is multiplied in turn once its warps have filled it, a stage is free once its block has been multiplied, a warp
    waits for its next block's stage.  Every order of events ends, whichever warp is held back."""
    warps, stages, deal = dealt
    per, order = deal[rows]
    for blocks in BLOCKS:
        for slow in range(-1, warps):
            at, fills, done = [0] * warps, [0] * blocks, 0
            left = [[i for i in o if i < blocks] for o in order]
            while done < blocks:
                moved = False
                for w in [w for w in range(warps) if w != slow] + ([slow] if slow >= 0 else []):
                    while at[w] < len(left[w]) and (w != slow or not moved) and left[w][at[w]] // stages <= (done + stages - 1 - left[w][at[w]] % stages) // stages:
                        i = left[w][at[w]]
                        fills[i] += 1
                        assert fills[i] <= per and done > i - stages
                        at[w] += 1
                        moved = True
                while done < blocks and fills[done] == per:
                    done += 1
                    moved = True
                assert moved, "stuck at block %d" % done
