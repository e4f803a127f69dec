"""How a call of the cleartext attention is run, from what the host knows of it (csrc/kv4_attend.hpp, compiled here into
a host program; no GPU needed)."""

import subprocess

import pytest

from holmes_amd import build as hb

MAIN = r"""
#include "kv4_attend.hpp"
#include <cstdio>
#include <cstdlib>
// seqs heads group dim most cols pages
int main(int, char** a) {
  const int n = atoi(a[1]), heads = atoi(a[2]), group = atoi(a[3]), dim = atoi(a[4]), most = atoi(a[5]), cols = atoi(a[6]);
  const hck::Way w(n, heads, group, dim, false, most, cols);
  printf("%d\n", (int)w.once(n, cols, atoll(a[7]), heads, dim));
}
"""


@pytest.fixture(scope="module")
def way(tmp_path_factory):
    at = tmp_path_factory.mktemp("way")
    (at / "main.hip").write_text(MAIN)
    done = subprocess.run([hb.HIPCC, *hb.FLAGS, f"-I{hb.CSRC}", str(at / "main.hip"), "-o", str(at / "way")],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-3000:]

    def run(**k):
        return subprocess.run([str(at / "way"), *map(str, k.values())], capture_output=True, text=True, check=True).stdout.split()

    return run


def once(way, seqs, cols, pages, heads=8, dim=128, most=1, group=4):
    return way(seqs=seqs, heads=heads, group=group, dim=dim, most=most, cols=cols, pages=pages)[0] == "1"


def test_loads_past_the_caches(way):
    page = 8 * 128 * 136
    full = (32 << 20) // page     # pages that the L2s hold
    assert once(way, 48, 192, 9000) and once(way, 32, 64, 460)
    assert not once(way, 32, 2000, 200)        # tables with room for any cache over a pool of 28 MB
    assert not once(way, 1, full, 1 << 40) and once(way, 1, full + 1, 1 << 40)
    assert not once(way, 1, 1 << 20, full) and once(way, 1, 1 << 20, full + 1)
    assert once(way, 1, 1 << 20, 2 * full + 2, dim=64) and not once(way, 1, 1 << 20, 2 * full, dim=64)
    assert not once(way, 48, 192, 9000, most=300)   # several tiles of rows read a page
