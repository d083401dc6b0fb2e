"""The layer and optimizer operators' GPU tests, a quick subset, on the CPU emulation of the kernel sources (emu/, tests/emu_util.py): part of the `-m "not gpu"` suite.

A subprocess, because the mapping of "cuda" to the CPU is process-wide and must not leak into the tests that check that CPU tensors are refused."""
import os
import re
import subprocess
import sys

from emu_util import EMU_DIR, ROOT, build_emu

QUICK = [
    "tests/test_gpu_group_norm.py", "tests/test_gpu_group_norm_mean.py::test_a_constant_segment_gives_exactly_the_bias", "tests/test_gpu_grouped_linear.py",
    "tests/test_gpu_adamw.py", "tests/test_gpu_adamw_autograd.py", "tests/test_gpu_adamw_layouts.py", "tests/test_gpu_adamw_random_bits.py", "tests/test_gpu_layers_autograd.py",
    "tests/test_gpu_typed_layer.py", "tests/test_gpu_operator_bounds.py",
]


def _run(args, **env):
    workers = str(max(1, min(4, os.cpu_count() or 1)))
    full = dict(os.environ, DGCNN_EMU="1", **env)
    full.pop("DGCNN_HIP_LIB", None)
    return subprocess.run([sys.executable, "-m", "pytest", "-m", "gpu", "-q", "-n", workers, "-p", "no:cacheprovider", *args], cwd=ROOT, env=full, stdout=subprocess.PIPE,
                          stderr=subprocess.STDOUT, text=True, timeout=1500)


def test_the_operators_gpu_tests_on_the_emulation():
    build_emu()
    # (left out for their time: many workgroups or long sums for a scheduler that runs one lane after the other)
    res = _run(QUICK + ["-k", "not long and not many and not large and not walk and not stall and not 130 and not chunks and not 9000 and not 6000 and not 3000"])
    m = re.search(r"(\d+) passed", res.stdout)
    assert res.returncode == 0 and m and int(m.group(1)) >= 250, res.stdout[-3000:]


def test_no_wave_meets_another_in_lds(tmp_path):
    """the race detector's build: no word of LDS is touched by two waves between two barriers, one of them writing"""
    res = subprocess.run(["make", "-C", EMU_DIR, "race", "-j8"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    lib = os.path.join(EMU_DIR, "libdgcnn_emu_race.so")
    assert res.returncode == 0 and os.path.exists(lib), res.stdout[-3000:]
    log = tmp_path / "races"
    log.touch()
    r = _run(["tests/test_gpu_group_norm_mean.py", "tests/test_gpu_operator_bounds.py", "-k", "(constant and whole) or (grouped and good and 1300) or (group_norm and dense and 1500)"],
             DG_EMU_RACE="1", DG_EMU_RACE_LOG=str(log), DGCNN_EMU_LIB=lib)
    assert r.returncode == 0 and re.search(r"\d+ passed", r.stdout), r.stdout[-3000:]
    assert log.read_text() == ""
