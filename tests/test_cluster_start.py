"""Every kernel that touches the shared memory of another CTA of its cluster waits on a cluster barrier first: the CTAs of a
cluster are scheduled together but do not begin together, and a peer's shared memory may be accessed only once the peer
runs.  A missing barrier shows in no result, so this reads the sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ac4k_kernel_b200", "csrc")
# helpers that write to, or signal in, the shared memory of a CTA of the cluster
REMOTE = r"\b(st_shared_cluster_\w+|bulk_copy_to_cluster|mbar_arrive_cluster\w*|tma_load_\w*pair\w*|tc_commit_pair\w*)\("
BARRIER = r"\b(cluster_sync(_relaxed)?|cluster_wait)\("


def _kernels():
    """(file, name, body) of the kernels, comments taken out; a body reaches to the next kernel or host function"""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for part in re.split(r"(?=__global__)", text)[1:]:
            name = re.search(r"(\w+_kernel)\(", part).group(1)
            yield os.path.basename(path), name, re.split(r"\n}\n", part, maxsplit=1)[0]


@pytest.mark.parametrize("file,name,body", [k for k in _kernels() if re.search(REMOTE, k[2])], ids=lambda v: v if len(v) < 60 else "")
def test_barrier_before_a_peers_shared_memory(file, name, body):
    first = re.search(REMOTE, body).start()
    barrier = re.search(BARRIER, body)
    assert barrier and barrier.start() < first, f"{file}: {name} reaches a peer's shared memory before any cluster barrier"


def test_kernels_with_peers_are_found():
    assert {n for _, n, b in _kernels() if re.search(REMOTE, b)} >= {
        "nvfp4_quantize_flat_kernel", "linear_nvfp4_skinny_kernel", "linear_nvfp4_2cta_kernel"}


# plain loads and stores, in either direction
ACCESS = r"\b(st|ld)_shared_cluster_\w+\("


def _stands_between(body):
    """whether a cluster barrier stands in front of the first access to a peer's shared memory, and one behind the last"""
    at = [m.start() for m in re.finditer(ACCESS, body)]
    barriers = [m.start() for m in re.finditer(BARRIER, body)]
    return bool(barriers) and barriers[0] < at[0] and barriers[-1] > at[-1]


@pytest.mark.parametrize("file,name,body", [k for k in _kernels() if re.search(ACCESS, k[2])], ids=lambda v: v if len(v) < 60 else "")
def test_barriers_around_loads_and_stores(file, name, body):
    """A CTA that has left has no shared memory: the last access is behind a barrier that all pass as well"""
    assert _stands_between(body), f"{file}: {name}"


def test_no_access_goes_by_without_a_name():
    """What these tests look for are the helpers' names, so no kernel writes the instructions out"""
    for file, name, body in _kernels():
        assert not re.search(r"\bshared::cluster\b|\bmapa\.", body), f"{file}: {name}"
    assert {n for _, n, b in _kernels() if re.search(ACCESS, b)} >= {"lora_kernel", "nvfp4_quantize_flat_kernel"}


def test_a_barrier_that_is_missing_is_seen():
    body = {n: b for _, n, b in _kernels()}["lora_kernel"]
    assert _stands_between(body)
    calls = list(re.finditer(r"ptx::cluster_sync\(\)", body))
    assert len(calls) == 2
    for call in calls:
        assert not _stands_between(body[:call.start()] + "__syncthreads()" + body[call.end():])
