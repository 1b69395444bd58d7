"""Every wait in a kernel has a limit, which the launch gives it: a wait without one hangs the GPU for everybody where what it waits for
does not come.  Shown by reading the sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ac4k_kernel_b200", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.cu*")))


def _code(path):
    return re.sub(r"//[^\n]*", "", open(path).read())


def _arguments(text, at):
    """the arguments of the call whose opening parenthesis is text[at]"""
    depth, args, start = 0, [], at + 1
    for i in range(at, len(text)):
        depth += text[i] in "([{"
        depth -= text[i] in ")]}"
        if depth == 0 or (depth == 1 and text[i] == ","):
            args.append(text[start:i].strip())
            start = i + 1
        if depth == 0:
            return args


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_waits_carry_the_limit_of_the_launch(path):
    text = _code(path)
    for call in re.finditer(r"(?<!bool )\bmbar_wait\(", text):
        args = _arguments(text, call.end() - 1)
        assert len(args) == 3 and args[2].endswith("wait_ns"), args


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_no_grid_barrier_without_a_limit(path):
    assert not re.search(r"cooperative_groups|this_grid\(|grid_group", _code(path))


@pytest.mark.parametrize("name", ["linear_nvfp4_skinny.cu", "linear_nvfp4_grouped.cu"])
def test_no_copy_to_a_peer_outlives_an_expired_wait(name):
    """The slices of a tile send one another their sums by bulk copies, which complete at the owner.  One that gave up on its own sum sends none, and an
    owner whose wait ran out gives those of the others one more limit before it leaves: a copy never writes to, or reads from, the memory of a CTA
    that has left.  What was not received is not stored."""
    text = _code(os.path.join(CSRC, name))
    sends = [m.start() for m in re.finditer(r"bulk_copy_to_cluster\(", text)]
    assert len(sends) == 1
    condition = text[text.rindex("if (", 0, sends[0]):sends[0]]
    assert condition.startswith("if (tfull_ok && ")
    behind = text[sends[0]:]
    wait = re.search(r"const bool got = mbar_wait\((part_bar[^,]*), 0, p\.wait_ns\);\s*if \(!got\) \{[^}]*mbar_wait\(\1, 0, p\.wait_ns\);\s*\}\s*if \([^)]*&& got\)", behind)
    assert wait and behind.index("cluster_sync_relaxed()") > wait.end()
