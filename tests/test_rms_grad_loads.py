"""Static check of the norm gradient's gfx950 assembly: where a thread's values leave room for them, the next
row's x, dy and dsum are loaded while this row is summed, so each run of 16 bytes has two loads (one before
the loop, one in it); and no form spills registers."""
import re
import subprocess

import pytest

from my_own_cnn_amd import build as B

WIDE = {"f": 4, "DF16b": 8}  # values of 16 bytes


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    dst = tmp_path_factory.mktemp("asm") / "k.s"
    subprocess.run([B.hipcc(), *B.common_flags(), "--cuda-device-only", "-S", str(B.CSRC / "rms_grad.hip"), "-o", str(dst)],
                   check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    return dst.read_text()


def test_the_next_row_is_loaded_ahead(asm):
    bodies = re.findall(r"^(_Z\S*15rms_grad_kernelI(f|DF16b)(?:f|DF16b)Li(\d+)ELi(\d+)E\S*):(.*?)^\.Lfunc_end", asm, re.S | re.M)
    assert len(bodies) >= 36
    ahead = 0
    for name, kind, threads, runs, body in bodies:
        threads, runs = int(threads), int(runs)
        if runs * WIDE[kind] * (2 if threads == 1024 else 1) <= 16:
            ahead += 1
            assert len(re.findall(r"^\s+global_load_dwordx4 ", body, re.M)) >= 6 * runs, name
    assert ahead >= 28


def test_no_register_is_spilled(asm):
    spills = re.findall(r"\.name:\s+(_Z\S+)[\s\S]*?\.vgpr_spill_count:\s+(\d+)", asm)
    assert len(spills) > 40 and not [s for s in spills if s[1] != "0"]
