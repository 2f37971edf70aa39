"""Loads to LDS in inline assembly: the compiler does not look inside, so the wait states that a scalar base needs behind a vector instruction that
wrote it (five) have to be there already.  A kernel in which such an instruction stands right in front is compiled, and its assembly read."""
import os
import re
import shutil
import struct
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "avelang_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"

KERNEL = r"""
#include "attn_common.hpp"
using namespace ave;
__global__ void probe(const uint8_t* p, const int* i, int* out) {
  __shared__ __align__(16) unsigned char lds[4][1024];
  const unsigned at = lds_address(lds);
  to_lds16(uniform_pointer(p + (int64_t)i[threadIdx.x] * 1024), threadIdx.x * 16, at);
  to_lds16<true>(uniform_pointer(p + (int64_t)i[threadIdx.x + 64] * 1024), threadIdx.x * 16, at + 1024);
  to_lds4(uniform_pointer(p + (int64_t)i[threadIdx.x + 128] * 1024), threadIdx.x * 4, at + 2048);
  wait_loads<0>();
  __syncthreads();
  out[threadIdx.x] = lds[0][threadIdx.x] + lds[1][threadIdx.x] + lds[2][threadIdx.x];
}
"""


def _scalars(operand):
    """Numbers of the scalar registers that an operand names."""
    m = re.fullmatch(r"s(\d+)|s\[(\d+):(\d+)\]", operand)
    return set() if not m else {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))


def _wait_states(lines, at, wanted):
    """Wait states between the load at `at` and the last vector instruction in front of it that writes one of `wanted` (None: there is none)."""
    states = 0
    for line in reversed(lines[:at]):
        op, *rest = line.replace(",", " ").split()
        if op.startswith("v_") and rest and _scalars(rest[0]) & wanted:
            return states
        states += int(rest[0], 0) + 1 if op == "s_nop" else 1
    return None


def test_wait_states_in_front_of_loads_with_a_scalar_base(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    (tmp_path / "probe.hip").write_text(KERNEL)
    subprocess.run([HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-w", "--cuda-device-only",
                    f"-I{CSRC}", "-S", str(tmp_path / "probe.hip"), "-o", str(tmp_path / "probe.s")], check=True)
    body = re.search(r"^\S*probe\S*:.*?s_endpgm", (tmp_path / "probe.s").read_text(), re.M | re.S)[0]
    lines = [line.split(";")[0].strip() for line in body.splitlines()]
    lines = [line for line in lines if re.match(r"[a-z]+_", line)]
    seen = 0
    for at, line in enumerate(lines):
        if line.startswith("global_load_lds"):
            base = _scalars(line.replace(",", " ").split()[2])
            states = _wait_states(lines, at, base)
            assert base and states is not None, line           # (the probe is made so that there is one)
            assert states >= 5, (line, states)
            seen += 1
    assert seen == 3


def _code_objects(library):
    """The gfx950 code objects of a library built by hipcc: bundles of (offset, size, target) entries, one for each source."""
    data = open(library, "rb").read()
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = data.find(magic)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(magic))
        entry = at + len(magic) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            target = data[entry + 24:entry + 24 + length]
            entry += 24 + length
            if b"gfx950" in target:
                yield data[at + offset:at + offset + size]
        at = data.find(magic, at + 1)


def test_wait_states_in_the_built_library(tmp_path):
    """Every load and store of the library's kernels that names a scalar base: no vector instruction within five wait states in front of it writes that
    base.  (In order of address: a branch in between only adds to them.)"""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    loads, bad = 0, []
    for n, code in enumerate(_code_objects(os.path.join(os.path.dirname(CSRC), "libave_fp4.so"))):
        (tmp_path / "code").write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(tmp_path / "code")], check=True, capture_output=True, text=True).stdout
        kernel, last = "", []
        for line in text.splitlines():
            if line.endswith(">:"):
                kernel, last = line, []
                continue
            line = line.split("//")[0].strip()
            if line.startswith(("global_", "buffer_", "scratch_")):
                wanted = set().union(*map(_scalars, line.replace(",", " ").split()[1:]))
                if wanted:
                    loads += 1
                    states = _wait_states(last, len(last), wanted)
                    if states is not None and states < 5:
                        bad.append((kernel, line, states))
            if line:
                last = last[-7:] + [line]
    assert loads > 10000
    assert not bad, (len(bad), bad[:3])
