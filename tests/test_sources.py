"""Rules of the sources that a compiler does not check."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_build_switch_takes_a_barrier_out():
    """a barrier or a wait that some build leaves out would make that build race: whether one is needed is looked at on the CPU (emu/, the race detector), in a
    copy.  The one `#ifndef` allowed is the emulation's own, which has another barrier in its other branch; an `#ifdef` adds what is inside it."""
    for path in glob.glob(os.path.join(ROOT, "dgcnn_amd", "csrc", "*.h*")):
        open_ifs = []
        for n, line in enumerate(open(path), 1):
            s = line.strip()
            if re.match(r"#\s*if", s):
                open_ifs.append(s)
            elif re.match(r"#\s*endif", s):
                open_ifs.pop()
            elif re.search(r"barrier\w*(<[^>]*>)?\(|s_waitcnt|__syncthreads\(", s.split("//")[0]):
                out = [c for c in open_ifs if re.match(r"#\s*ifndef", c) and not re.search(r"DG_EMU|\w+_H\b", c)]
                assert not out, f"{path}:{n}: {s} is left out by {out}"


def test_no_script_runs_a_build_without_barriers():
    for pattern in ("tools/*", "dgcnn_amd/csrc/Makefile", "emu/Makefile"):
        for path in glob.glob(os.path.join(ROOT, pattern)):
            if os.path.isfile(path):
                text = open(path, errors="replace").read().lower()
                assert "nobar" not in text and not re.search(r"-d\w*no_\w*(barrier|wait)", text), path


def test_no_assembly_writes_m0_behind_the_compilers_back():
    """m0 is reserved: a clobber of it is not honoured, so its value goes in as an operand ("{m0}") or not at all"""
    for path in glob.glob(os.path.join(ROOT, "dgcnn_amd", "csrc", "*.h*")):
        for n, line in enumerate(open(path), 1):
            assert not re.search(r"\bs_\w+ m0\b", line), f"{path}:{n}"
