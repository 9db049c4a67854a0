"""Rules that a kernel's source has to keep because no run can show that they hold: what the compiler may move, and what
orders a read of shared memory before the asynchronous copy that overwrites it."""

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bridge_b200", "csrc")


def _sources():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        with open(path) as f:
            yield os.path.basename(path), f.read()


def test_warp_collectives_in_assembly_are_volatile():
    """A statement that every lane of a warp has to reach may not be moved into a branch that only some lanes take."""
    seen = 0
    for name, text in _sources():
        for m in re.finditer(r"\basm(\s+volatile)?\s*\(((?:[^;\"]|\"(?:[^\"\\]|\\.)*\")*)\)\s*;", text):
            if re.search(r"\.sync\b", m.group(2)):
                seen += 1
                assert m.group(1), f"{name}: {' '.join(m.group(2).split())[:60]}"
    assert seen > 10


def test_slots_are_read_before_they_are_refilled():
    """Nothing but a barrier orders a lane's read of shared memory before the asynchronous copy into the same slot that
    it issues afterwards: reading a batch ends with one."""
    text = dict(_sources())["vocab_rows.cu"]
    body = re.search(r"void take\(Unit<T>\* u\) \{(.*?)\n  \}", text, re.S).group(1)
    assert body.rindex("__syncwarp()") > body.rindex("read<3>(")
    # and every read of a slot goes through it
    assert len(re.findall(r"\bread<\d>\(ring", text)) == len(re.findall(r"\bread<\d>\(ring", body)) == 4


def test_store_buffers_take_turns_across_tiles():
    """A wait for all but the last store frees the other buffer only if every store takes the buffer that the one before
    it did not, through all tiles of a warp."""
    text = dict(_sources())["adapter_linear.cu"]
    body = re.search(r"\n    adapter_joint_kernel\(.*?\n}\n", text, re.S).group(0)
    assert len(re.findall(r"tma_store_2d\(", body)) == len(re.findall(r"tma_store_wait_read<1>", body)) == 1
    assert re.search(r"buf = store \+ \(quarter \* 2 \+ turn\) \* kStoreBytes;\s+turn \^= 1;", body)
    assert len(re.findall(r"\bturn\b", re.sub(r"//[^\n]*", "", body))) == 3
    assert body.index("turn = 0") < body.rindex("for (int q = pair;") < body.index("+ turn)")


def test_aligned_cluster_barriers_take_whole_warps():
    """An aligned barrier is for a converged warp; after a loop of which each lane has its own number of rounds nothing but
    a warp barrier says that it is."""
    seen = 0
    for name, text in _sources():
        for m in re.finditer(r"barrier\.cluster\.arrive[\w.]*\.aligned", text):
            seen += 1
            before = re.sub(r"//[^\n]*", "", text[:m.start()])
            assert re.search(r"__syncwarp\(\);\s*asm volatile\(\s*\"$", before), name
    assert seen
