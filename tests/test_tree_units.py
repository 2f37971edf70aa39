"""The arithmetic that divides attention over drafted trees among workgroups (``csrc/attn_units.hpp``), compiled for the host: what rows see at least and at most,
numbers of units beyond 32 bits, and the bound that chooses between 32 and 64."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "avelang_amd", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include <initializer_list>
#include "attn_units.hpp"
using namespace ave;

// new tokens, keys, group, key heads, window, item units
template <int ROWS, typename U>
int units(char** v) {
  TreeArgs p{};
  Sequence s{0, atoi(v[0]), atoi(v[1])};
  set_group(p, atoi(v[2]));
  p.a.tokens = s.n, p.a.batch = 1, p.page_shift = 4, p.a.table_pages = (s.len + 15) / 16;
  p.c.kv_heads = atoi(v[3]);
  p.a.window = atoi(v[4]), p.a.causal = 1, p.item_units = atoi(v[5]);
  // one by one, and as a product
  const int64_t rows = (int64_t)s.n * p.group;
  const U product = sequence_units<ROWS, 64, U>(p, s);
  U listed = 0;
  int tile0 = 0;
  for (int64_t row0 = 0; row0 < rows; row0 += ROWS) listed += (unsigned)block_units<ROWS, 64>(p, s, (int)row0, tile0);
  if (listed != product) return printf("%llu units one by one, %llu\n", (unsigned long long)listed, (unsigned long long)product), 1;
  printf("%llu %d %llu\n", (unsigned long long)((unsigned)p.c.kv_heads * product), tile0, (unsigned long long)units_bound(p, ROWS, 64));
  return 0;
}
template <int ROWS>
int both(char** v) { return units<ROWS, Units>(v) + units<ROWS, unsigned>(v); }

// Rows whose window counts from 0 to all of the new tokens, against what `bounds` says of them
int seen(int most) {
  TreeArgs p{};
  set_group(p, 1);
  for (int n = 1; n <= most; ++n)
    for (int len = 0; len <= 2 * most; ++len)
      for (int w : {0, 1, 2, 3, 5, 8, most, 2 * most, 3 * most, INT32_MAX - 1, INT32_MAX}) {
        p.a.window = w;
        const Sequence s{0, n, len};
        const Bounds b = bounds(p, s, 0, n - 1);
        const int base = len - n > 0 ? len - n : 0;
        int least = INT32_MAX, most_of_all = 0;
        for (int many = 0; many <= n; ++many) {   // bits that are set in a row
          const int64_t from = (int64_t)len - n + many - w;
          const int lo = w == 0 || from < 0 ? 0 : (int)from;
          least = lo < least ? lo : least, most_of_all = lo > most_of_all ? lo : most_of_all;
        }
        if (b.lo_min != least || b.lo_max < most_of_all || b.hi_min != base || b.hi_max != len)
          return printf("%d of %d, window %d: [%d, %d) and [%d, %d)\n", n, len, w, b.lo_min, b.hi_max, b.lo_max, b.hi_min), 1;
      }
  return 0;
}
int main(int n, char** v) {
  if (n == 2) return seen(atoi(v[1]));
  switch (atoi(v[1])) {
    case 16: return both<16>(v + 2);
    case 32: return both<32>(v + 2);
    case 64: return both<64>(v + 2);
    default: return both<128>(v + 2);
  }
}
"""

# rows of a block, new tokens, keys, group, key heads, window, item units
CASES = [
    (128, 600000, 600000, 16, 8, 0, 3),               # beyond 32 bits
    (64, 600000, 600000, 16, 8, 0, 3),
    (128, 260000, 1 << 20, 16, 8, 0, 3),
    (128, 260000, 1 << 20, 16, 8, 700000, 3),         # a window shorter than the new tokens and the keys before them
    (128, 260000, 1 << 20, 16, 8, (1 << 31) - 1, 3),
    (64, 64, (1 << 31) - 256, 16, 32, 0, 3),          # 64 nodes on as many keys as a table covers
    (64, 64, (1 << 31) - 256, 16, 32, (1 << 31) - 1, 3),
    (64, 64, (1 << 31) - 256, 16, 32, 1 << 30, 3),
    (64, 16, 4096, 4, 8, 0, 3),
    (64, 64, 3000, 8, 8, 1000, 3),
    (64, 64, 3000, 8, 8, 1, 3),
    (128, 500, 300, 3, 5, 0, 3),                      # more new tokens than keys
    (128, 500, 300, 3, 5, 100, 3),
    (32, 5, 700, 4, 8, 0, 0),
    (16, 4, (1 << 31) - 256, 4, 128, 0, 0),
    (16, 1, 0, 16, 8, 0, 0),
]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    where = tmp_path_factory.mktemp("tree_units")
    (where / "units.cc").write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-ftrapv", f"-I{CSRC}", str(where / "units.cc"), "-o", str(where / "units")], check=True)
    return str(where / "units")


def _expected(rows_of_block, new, keys, group, heads, window, item):
    before = max(0, keys - new)
    lo = max(0, before - window) if window else 0
    tiles = -(-keys // 64) - lo // 64 if keys > lo else 1
    return -(-new * group // rows_of_block) * heads * (tiles + item), lo // 64


@pytest.mark.parametrize("case", CASES, ids=str)
def test_units(program, case):
    done = subprocess.run([program, *map(str, case)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr
    wide, narrow = (list(map(int, line.split())) for line in done.stdout.splitlines())
    units, tile0, bound = wide
    assert (units, tile0) == _expected(*case)
    # the bound by which the host chooses: never below, so that 32 bits hold what they are given
    assert units <= bound
    assert bound >= 1 << 32 or narrow == wide


def test_some_of_these_pass_32_bits():
    assert sum(_expected(*c)[0] >= 1 << 32 for c in CASES) >= 5


def test_what_rows_see(program):
    done = subprocess.run([program, "24"], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr
