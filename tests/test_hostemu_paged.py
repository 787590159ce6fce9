"""The paged-cache operators' kernels on the CPU under AddressSanitizer (tests/native/hostemu): append
with rotation, then attention, every buffer of exactly its size, stale slots NaN; no access outside a
buffer and the outputs of a double-precision evaluation."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CXX = "/opt/rocm/llvm/bin/clang++"
EXE = os.path.join(os.path.dirname(HERE), "_build", "hostemu", "paged_check")

pytestmark = pytest.mark.skipif(not os.path.exists(CXX) or shutil.which("make") is None,
                                reason="needs the ROCm clang++ for the host build")


@pytest.fixture(scope="module")
def check():
    r = subprocess.run(["make", "-s", "-j8", "-C", os.path.join(HERE, "native", "hostemu")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    return EXE


# hd bf16 nh nkv page window prefix f32 poison tail, then new:keys of each sequence
@pytest.mark.parametrize("args", [
    "32 0 4 4 16 0 0 0 0 2 1:1 1:40 1:300 3:70 0:9 0:0",     # single tokens and a draft
    "64 1 8 2 32 0 0 1 0 0 1:3000",                          # split over the keys and joined
    "128 1 2 1 16 0 0 0 0 1 90:1400",                        # a chunk split over the keys
    "32 0 4 2 16 0 0 0 1 2 300:1500 1:40 0:0 40:900 200:200 129:700",   # unequal row tiles cut into equal runs
    "64 1 8 1 32 0 0 0 0 0 33:3000 70:90",
    "128 0 4 1 16 0 0 0 0 1 1:100 90:200 0:7 1:33",          # a mix
    "128 1 6 2 16 50 0 0 1 0 40:97 70:70",                   # a window; NaN in each chunk's last key
    "32 0 2 2 64 0 60 0 2 3 100:130 1:500",                  # a prefix; entries that name no page
    "64 0 32 1 16 100 0 0 1 0 3:900 17:600",                 # wide groups
    "128 1 17 1 16 0 0 1 0 0 1:130 2:80 20:40",              # groups that are no power of two
    "64 1 10 2 128 0 0 0 0 2 130:400 1:1 1:257 9:9",         # tiles that end inside a page
    "64 0 4 4 16 7 0 0 1 1 33:80 100:300",                   # a window smaller than a tile
    "64 0 4 2 16 1 0 0 0 0 129:300 40:40",                   # waves whose rows see none of the first tiles
    "32 0 3 3 32 0 200 0 2 0 60:150 1:300",                  # a prefix past the sequence's end
], ids=lambda s: s.replace(" ", "_"))
def test_paged_operators_in_bounds(check, args):
    r = subprocess.run([check] + args.split(), capture_output=True, text=True,
                       env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"), timeout=900)
    assert r.returncode == 0, (r.stdout + r.stderr)[-4000:]
