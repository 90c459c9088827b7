"""The loads to LDS that are written in assembly (csrc/lds_load.h), by the
instructions they become: the compiler does not look into the statement, so that it
has to hold the waits it needs and name the registers it writes."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "velo-mind_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

# The address comes straight from v_readfirstlane, and m0 is in use on both sides.
KERNEL = """
#include <hip/hip_runtime.h>
#include "lds_load.h"
typedef __attribute__((address_space(3))) void* Lds;
typedef const __attribute__((address_space(1))) void* Global;
__global__ void kernel(const char** p, const char* q, char* out) {
    __shared__ __align__(16) char tile[8192];
    const uint64_t a = reinterpret_cast<uint64_t>(p[threadIdx.x / 64]);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
    __builtin_amdgcn_global_load_lds((Global)(q + threadIdx.x * 4), (Lds)tile, 4, 0, 0);
    vmhip::lds_load16(reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo), threadIdx.x * 16, tile + 1024);
    __builtin_amdgcn_global_load_lds((Global)(q + threadIdx.x * 4 + 4096), (Lds)tile, 4, 0, 0);
    vmhip::wait_loads();
    __syncthreads();
    out[threadIdx.x] = tile[threadIdx.x * 4];
}
"""


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    """The kernel's instructions, in order."""
    d = tmp_path_factory.mktemp("lds_load")
    src, out = d / "kernel.hip", d / "kernel.s"
    src.write_text(KERNEL)
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-I", CSRC, "--cuda-device-only", "-S", str(src), "-o", str(out)], check=True,
                   stderr=subprocess.DEVNULL)
    lines = out.read_text().split("s_endpgm")[0].splitlines()
    lines = [line.split(";")[0].strip() for line in lines]
    return [line for line in lines if re.match(r"[sv]_|global_|ds_", line)]


def test_the_address_is_there(listing):
    """A scalar instruction wrote it last (it waits for its operands), or a vector
    instruction did so five wait states ahead."""
    at = next(i for i, line in enumerate(listing) if line.startswith("global_load_lds_dwordx4"))
    lo, hi = map(int, re.search(r"s\[(\d+):(\d+)\]", listing[at]).groups())
    todo, states = set(range(lo, hi + 1)), 0
    for line in reversed(listing[:at]):
        one, two = re.match(r"([sv])_\w+ s(\d+),", line), re.match(r"([sv])_\w+ s\[(\d+):(\d+)\],", line)
        written = {int(one[2])} if one else set(range(int(two[2]), int(two[3]) + 1)) if two else set()
        if written & todo and (one or two)[1] == "v":
            assert states >= 5, line
        todo -= written
        if not todo:
            return
        nop = re.match(r"s_nop (\d+)", line)
        states += int(nop.group(1)) + 1 if nop else 1
    pytest.fail("nothing wrote the address")


def test_a_wait_state_between_m0_and_the_load(listing):
    at = next(i for i, line in enumerate(listing) if line.startswith("global_load_lds_dwordx4"))
    wrote = max(i for i in range(at) if re.match(r"s_\w+ m0,", listing[i]))
    assert wrote < at - 1
    assert not any(line.startswith("global_load_lds") for line in listing[wrote:at]), "m0 is an earlier load's"


def test_m0_is_written_again_behind_the_load(listing):
    at = next(i for i, line in enumerate(listing) if line.startswith("global_load_lds_dwordx4"))
    behind = next(i for i in range(at + 1, len(listing)) if listing[i].startswith("global_load_lds_dword "))
    assert any(re.match(r"s_\w+ m0,", line) for line in listing[at + 1:behind])
