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


def test_blocks_end_with_no_copy_of_theirs_in_flight():
    # The general kernels ask for a block's own rows before they know of a tile, and a block may have none: the wait stands behind the loop.
    with open(os.path.join(ROOT, "sddmm_gpu_b200", "csrc", "attention_general.cu")) as text:
        source = text.read()
    loops = [m.end() for m in re.finditer(r"for \(int t = mine\.first; t < mine\.end; \+\+t\) \{", source)]
    assert len(loops) == 3
    for at in loops:
        depth = 1
        while depth:
            depth += {"{": 1, "}": -1}.get(source[at], 0)
            at += 1
        assert source[at:].lstrip().startswith("arrived<0>();")
