"""The arithmetic that divides attention among workgroups (``csrc/attn_units.hpp``), compiled for the host: numbers of units beyond 32 bits, equal
and complete parts, the bound that chooses between 32 and 64, what rows see, and the division by the group size."""
import ctypes
import os
import subprocess

import pytest
import torch

from avelang_amd import _lib, attention as mod

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "avelang_amd", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include <initializer_list>
#include "attn_units.hpp"
using namespace ave;

// new tokens, keys, group, key heads, window, causal, item units, smallest part (log2), workgroups
template <int ROWS, typename U>
int units(char** v) {
  AttnArgs p{};
  Sequence s{0, atoi(v[0]), atoi(v[1])};
  set_group(p, atoi(v[2]));
  p.a.tokens = s.n, p.a.batch = 1, p.page_shift = 4, p.a.table_pages = (s.len + 15) / 16;
  p.c.kv_heads = atoi(v[3]);
  p.a.window = atoi(v[4]), p.a.causal = atoi(v[5]), p.item_units = atoi(v[6]), p.min_units_log2 = atoi(v[7]);
  const unsigned workgroups = (unsigned)atoi(v[8]);
  Part<U> r{};
  r.units = (unsigned)p.c.kv_heads * sequence_units<ROWS, 64, U>(p, s);
  U at = 0, most = 0, least = ~(U)0;
  for (unsigned g = 0; g < workgroups; ++g) {
    cut(p, r, g, workgroups);
    if (r.u0 != at || r.u1 < r.u0) return printf("part %u starts at %llu behind %llu\n", g, (unsigned long long)r.u0, (unsigned long long)at), 1;
    at = r.u1;
    if (g < r.parts) {
      if (r.u1 - r.u0 > most) most = r.u1 - r.u0;
      if (r.u1 - r.u0 < least) least = r.u1 - r.u0;
    }
  }
  printf("%llu %llu %llu %llu %u %llu\n", (unsigned long long)r.units, (unsigned long long)at, (unsigned long long)most, (unsigned long long)least, r.parts,
         (unsigned long long)units_bound(p, ROWS, 64));
  return 0;
}
template <int ROWS>
int both(char** v) { return units<ROWS, Units>(v) + units<ROWS, unsigned>(v); }
int groups(int from, int to) {
  for (int d = from; d < to; ++d) {
    AttnArgs p{};
    set_group(p, d);
    const int64_t top = 2147483647;
    for (int64_t k = 0; k < 64; ++k)
      for (int64_t n : {k, k * d - 1, k * d, k * d + 1, top - k, top / d * d - 1, top / d * d, top / d * d - k * d - 1, (top >> (k % 31)) * 1})
        if (n >= 0 && n <= top && p.token_of((int)n) != n / d) return printf("%lld / %d\n", (long long)n, d), 1;
  }
  return 0;
}
int main(int n, char** v) {
  if (n == 3) return groups(atoi(v[1]), atoi(v[2]));
  switch (atoi(v[1])) {
    case 16: return both<16>(v + 2);
    case 32: return both<32>(v + 2);
    case 64: return both<64>(v + 2);
    default: return both<128>(v + 2);
  }
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    where = tmp_path_factory.mktemp("units")
    (where / "units.cc").write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-ftrapv", f"-I{CSRC}", str(where / "units.cc"), "-o", str(where / "units")], check=True)
    return str(where / "units")


def _expected(rows_of_block, new, keys, group, heads, window, causal, item):
    total = 0
    for row0 in range(0, new * group, rows_of_block):
        first, last = row0 // group, (min(row0 + rows_of_block, new * group) - 1) // group
        hi = max(0, keys - new + last + 1) if causal else keys
        at = keys - new + first
        lo = at - window + 1 if window and at >= window else 0
        total += ((hi + 63) // 64 - lo // 64 if hi > lo else 1) + item
    return total * heads


CASES = [
    (128, 600000, 600000, 16, 8, 0, 0, 3, 2, 768),        # 5.6e9: beyond 32 bits
    (128, 520000, 1 << 20, 16, 8, 0, 1, 3, 2, 768),
    (128, 786448, 786448, 8, 8, 0, 0, 2, 2, 1024),
    (128, 100, 2000, 16, 8, 0, 1, 3, 2, 768),
    (128, 5000, 300, 3, 5, 0, 1, 3, 2, 768),              # more new tokens than keys
    (128, 5000, 90000, 3, 5, 1000, 1, 3, 2, 1000),
    (16, 1, 1 << 20, 1, 4096, 0, 1, 0, 2, 512),
    (16, 1, (1 << 31) - 4096, 8, 1024, 0, 1, 0, 2, 512),  # one token on as many keys as a table covers: 3.4e10
    (16, 1, (1 << 31) - 256, 8, 1, 0, 1, 0, 2, 512),      # ... with pages of 256 and less
    (128, 3000, (1 << 31) - 256, 2, 1, 0, 1, 3, 2, 768),
    (32, 1, 0, 32, 8, 0, 1, 0, 2, 512),
    (64, 2, 131072, 32, 1, 0, 1, 0, 2, 256),
    (16, 4, 1500, 8, 8, 128, 1, 0, 3, 512),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_units_and_parts(program, case):
    done = subprocess.run([program, *map(str, case)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr
    wide, narrow = (list(map(int, line.split())) for line in done.stdout.splitlines())
    units, covered, most, least, parts, bound = wide
    rows, new, keys, group, heads, window, causal, item, smallest, workgroups = case
    assert units == _expected(rows, new, keys, group, heads, window, causal, item)
    assert covered == units and most - least <= 1
    assert parts == max(1, min(workgroups, -(-units // (1 << smallest))))
    # the bound by which the host chooses: never below, so that 32 bits hold what they are given
    assert units <= bound
    assert bound >= 1 << 32 or narrow == wide


def test_some_of_these_pass_32_bits():
    assert sum(_expected(c[0], *c[1:8]) > 1 << 32 for c in CASES) >= 4


def test_division_by_the_group(program):
    done = subprocess.run([program, "1", "1025"], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.parametrize("page,pages,tokens,heads,text", [
    (16, (1 << 27) - 1, 1, 8, "2^31 - 256"), (128, (1 << 24) - 1, 1, 8, "2^31 - 256"), (256, (1 << 23) - 1, 1, 8, None), (4096, (1 << 19) - 1, 1, 8, None),
    (16, 1, (1 << 28) - 1, 8, "2^14 to spare"), (16, 1, (1 << 28) - 2049, 8, None), (16, 1, (1 << 28) - 2048, 8, "2^14 to spare")])
def test_sizes_next_to_2_to_the_31(page, pages, tokens, heads, text):
    """What is looked for behind the last key or row has to have a number, too: at 2^31 - 16 keys the next tile's was negative, and the page table was
    read in front of its start."""
    p = 1 << 20   # any aligned address: nothing is launched
    c = _lib.KVCache(k=p, k_scale=p, v=p, v_scale=p, k_page_stride=page * 64, k_scale_page_stride=page * 4, v_page_stride=page * 64, v_scale_page_stride=page * 4,
                     pages=3, kv_heads=1, page_size=page, head_dim=128)
    a = _lib.Attention(q=p, out=p, page_table=p, seq_lens=p, cu_q=p, tokens=tokens, batch=1, heads=heads, table_pages=pages, max_q=1, causal=1, scale=1)
    lib = _lib.load()
    if text is None:   # (a call would launch)
        lib.ave_fp4_attention_mxfp4_workspace_bytes(ctypes.byref(a), ctypes.byref(c))
        assert _lib.last_error() == ""
    else:
        assert lib.ave_fp4_attention_mxfp4(ctypes.byref(a), ctypes.byref(c), None, 0, None) == -1
        assert text in _lib.last_error(), _lib.last_error()


def test_sizes_beyond_31_bits_are_refused():
    """The C ABI's numbers of tokens, heads and pages have 32 bits: a larger size must not reach it cut to them."""
    many = lambda *shape, dtype=torch.bfloat16: torch.empty(1, dtype=dtype, device="meta").expand(*shape)   # noqa: E731
    with pytest.raises(ValueError, match="sizes below 2.31"):
        mod._heads(many((1 << 32) + 1, 1, 64), "k", None, 64, None, torch.device("meta"))
    with pytest.raises(ValueError, match="sizes below 2.31"):
        mod._vector(many(1 << 31, dtype=torch.int32), "slots", torch.int32, 1 << 31, torch.device("meta"))
    with pytest.raises(ValueError, match="sizes below 2.31"):
        mod._cache([many(1 << 33, 1, 16, n, dtype=torch.uint8) for n in (64, 4, 64, 4)])
    with pytest.raises(ValueError, match="sizes below 2.31"):
        mod._how(*[many(1 << 31, 32, dtype=torch.float32)] * 2, None, None, None, 1e-6, False, 1, 64, torch.device("meta"))
