"""Rules of the attention kernels' sources that no run would show."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_what_a_call_writes_is_read_by_ordinary_loads():
    # Kernels of a call may begin under the one before: what that one writes (workspace) is not read-only while they run, which __ldg() asks for.
    written = re.compile(r"(__ldg|ld\.global\.nc)\(?[^();]*\bp\.(delta|d_o_most|part_o|part_lse)\b")
    files = glob.glob(os.path.join(ROOT, "sddmm_gpu_b200", "csrc", "attention*.cu*"))
    assert len(files) > 5
    for f in files:
        with open(f) as text:
            for number, line in enumerate(text, 1):
                assert not written.search(line), f"{f}:{number}"
