"""How a call of attention over whole prompts is cut into parts, from what the host knows of it (csrc/prompt_way.hpp, compiled
here into a host program; no GPU needed)."""

import subprocess

import pytest

from holmes_amd import build as hb

MAIN = r"""
#include "prompt_way.hpp"
#include <cstdio>
#include <cstdlib>
// tokens seqs heads group dim most causal units: the way, and the parts that a tile of so many units comes in
int main(int, char** a) {
  const long long tokens = atoll(a[1]), seqs = atoll(a[2]);
  const int heads = atoi(a[3]), group = atoi(a[4]), dim = atoi(a[5]), most = atoi(a[6]), units = atoi(a[8]);
  const hck::WholeWay w(tokens, seqs, heads, group, most, atoi(a[7]));
  printf("%lld %d %d %zu\n", (long long)w.items, w.part, w.parts, w.bytes(heads, dim));
  if (w.parts == 1) return 0;
  for (int p = 0; p < hck::parts_of(units, w.part, w.parts); ++p) printf("%d %d\n", p * w.part, hck::part_end(units, w.part, w.parts, p));
}
"""


@pytest.fixture(scope="module")
def way(tmp_path_factory):
    at = tmp_path_factory.mktemp("way")
    (at / "main.hip").write_text(MAIN)
    done = subprocess.run([hb.HIPCC, *hb.FLAGS, f"-I{hb.CSRC}", str(at / "main.hip"), "-o", str(at / "way")],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-3000:]

    def run(*a):
        got = subprocess.run([str(at / "way"), *(str(int(x)) for x in a)], capture_output=True, text=True, check=True).stdout.split()
        got = [int(x) for x in got]
        return got[:4], list(zip(got[4::2], got[5::2]))

    return run


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("tokens,seqs,heads,group,dim,most", [
    (4000, 1, 2, 3, 128, 2000), (5000, 1, 1, 1, 64, 2000), (3000, 1, 1, 2, 64, 1500), (3000, 1, 1, 2, 64, 3000),
    (9000, 4, 1, 1, 128, 1100), (40000, 100, 1, 1, 64, 1300), (1 << 20, 1, 1, 1, 64, 1100),
])
def test_parts_cover_every_unit_once(way, tokens, seqs, heads, group, dim, most, causal):
    """Of tiles whose rows see up to `most` tokens, and without `causal` up to all, though `most` is less."""
    seen = most if causal else tokens
    for units in sorted({1, 2, 8, 9, 16, 17, -(-most // 64), -(-most // 64) + 1, -(-seen // 64) - 1, -(-seen // 64)}):
        if units > -(-seen // 64):
            continue
        (items, part, parts, size), cuts = way(tokens, seqs, heads, group, dim, most, causal, units)
        if parts == 1:
            assert size == 0      # a workgroup takes a whole tile, whatever its units
            continue
        assert 1 <= len(cuts) <= parts
        assert cuts[0][0] == 0 and cuts[-1][1] == units
        assert all(a < b for a, b in cuts) and all(a[1] == b[0] for a, b in zip(cuts, cuts[1:]))
        # the last slot that the last tile's parts have, [item][part][head]
        slot = 4 * 64 * (1 + dim // 8) * 16
        assert (((items - 1) * parts + len(cuts) - 1) * heads + heads) * slot <= size
        assert (len(cuts) > 1) == (units > part)      # one part writes the rows itself, and is not joined
