"""The ring of key tiles of the shared-prefix attention, on the CPU.

tests/c/prefix_ring_check.cpp runs the waits and arrivals of the kernel's roles in
many orders, with the number of arrivals that csrc/prefix_plan.h gives the kernel. A
preparing warp that is held back while the others run must not lose the ring's count:
with the MMAs' arrival alone it did, and the kernel would have waited for good."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "qwen3-embedding-webgpu-prepacked_b200", "csrc")


@pytest.fixture(scope="module")
def ring_check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("ring") / "prefix_ring_check")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", CSRC,
                    os.path.join(HERE, "c", "prefix_ring_check.cpp"), "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("slots,warps,converts", [(4, 2, 0), (3, 4, 1)])
def test_roles_end_in_any_order(ring_check, slots, warps, converts):
    for seed in range(400):
        out = subprocess.run([ring_check, str(slots), str(warps), str(converts), str(seed)],
                             capture_output=True, text=True)
        assert out.returncode == 0, (seed, out.stdout)
