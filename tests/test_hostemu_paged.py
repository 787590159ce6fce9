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
    _run(check, args)


def _run(check, args):
    r = subprocess.run([check] + args.split(), capture_output=True, text=True,
                       env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"), timeout=900)
    assert r.returncode == 0, (r.stdout + r.stderr)[-4000:]
    return int(r.stdout.rsplit(" ", 1)[1])      # bytes of workspace


@pytest.mark.parametrize("args", [
    "64 1 8 2 32 0 0 1 0 0 1:5000",                          # one token: many splits joined
    "32 0 4 4 64 0 0 0 2 1 1:30000",
    "128 0 64 64 16 0 0 0 2 0 1:1200",                       # four splits
    "128 1 2 1 16 0 0 0 0 1 90:3000",                        # a chunk: equal runs of keys joined
    "128 0 2 1 16 0 0 0 1 2 140:2000 1:40 0:0 40:600",      # unequal row tiles beside a token
    "64 1 4 1 32 0 0 0 0 0 33:3500 40:90 1:2100",
    "32 1 1 1 16 0 0 0 2 0 130:4000 1:9 70:700",             # entries that name no page
    "64 0 8 2 64 700 0 1 1 1 100:4000 40:2900 1:3000",       # a window
], ids=lambda s: s.replace(" ", "_"))
def test_cut_work_in_bounds(check, args):
    """Calls whose keys are divided among workgroups: partial results through the workspace."""
    assert _run(check, args) > 0 or " 700 " in args


@pytest.mark.parametrize("args", [
    "128 0 2 1 16 0 0 0 3 2 140:2000 1:40 0:0 40:600",
    "64 0 8 2 16 0 0 0 3 0 1:400 3:70 1:2 2:9", "32 1 2 2 32 9 40 1 3 5 70:100 60:80 1:500",
], ids=lambda s: s.replace(" ", "_"))
def test_malformed_batches_stay_in_bounds(check, args):
    """seq_start that descends, overlaps and leaves the rows, kv_len of any value: nothing outside the
    buffers is touched (what the rows get is not defined)."""
    _run(check, args)


@pytest.mark.parametrize("poison", [0, 3])
def test_chunks_among_many_sequences_in_bounds(check, poison):
    """More row tiles of chunks, taken whole from the list, than are put in order; as they should be (0) and with
    a malformed batch (3)."""
    lens = "1500:1500 1500:1500 " + "1:9 " * 120 + "1500:1500 " + "1:40 " * 132
    _run(check, f"32 0 8 1 16 16 0 0 {poison} 1 {lens}")
