"""The single-row form of the 4-bit linear layer reads no codes outside the weights: its index arithmetic
(csrc/yvmoe_linear_stream.h), compiled for the host and walked as the kernel walks it."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("stream") / "check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I" + os.path.join(ROOT, "pisceslx_amd", "csrc"), "-o", exe,
                    os.path.join(ROOT, "tests", "int4_stream_check.cpp")], check=True)

    def run(cases):
        r = subprocess.run([exe], input="\n".join("%d %d %d" % c for c in cases), capture_output=True, text=True,
                           timeout=120)
        assert r.returncode == 0, r.stdout[-4000:]
        assert r.stdout.endswith(f"{3 * len(cases)} cases, 0 failed\n")
    return run


@pytest.mark.parametrize("grid", [256, 512])
@pytest.mark.parametrize("groups", list(range(1, 18)) + [32, 33])
def test_no_read_past_the_weights(walk, groups, grid):
    """Fewer groups than wavefronts and more, one item per work-group, two and several, whole and part sets."""
    blocks = [1, 2, 3, 5, 255, 256, 257, 300, 511, 512, 513, 771, 1023, 1024, 1025, 1250, 1500, 1535, 1536, 1537,
              2047, 2048, 2049, 3000, 5000]
    walk([(b, groups, grid) for b in blocks])


@pytest.mark.parametrize("O,K", [(20000, 128), (24000, 512), (4112, 896), (20000, 7)])
def test_layers_of_few_groups(walk, O, K):
    walk([(-(-O // 16), -(-K // 128), grid) for grid in (256, 512)])
