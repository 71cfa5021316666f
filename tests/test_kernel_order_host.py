"""Orders that no run shows to be broken, by reading the kernels: a CTA's shared
memory is reached by the others of its cluster only behind a cluster barrier, which
is what tells that the CTA runs; a bounded wait does not time the kernel before."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "aoh_b200" / "csrc"
REMOTE = re.compile(r"mapa_shared\(")  # every address in another CTA's shared memory is made by it
BARRIER = re.compile(r"\bcluster_(sync_all|wait)\(\)")


def _kernels():
    """(file, kernel, body without comments) of every kernel."""
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__global__ void\s+(?:__launch_bounds__\([^)]*\)\s*)?(\w+)\s*\(", text):
            start = at = text.index("{", m.end())
            depth = 0
            while True:
                depth += {"{": 1, "}": -1}.get(text[at], 0)
                at += 1
                if depth == 0:
                    break
            yield path.name, m[1], text[start:at]


BARRIER_OR_ARRIVE = re.compile(r"\bcluster_(sync_all|wait|arrive)\(\)")
REACHING = [k for k in _kernels() if REMOTE.search(k[2])]


def test_the_reading_finds_the_cluster_kernels():
    assert {k[1] for k in REACHING} >= {"decode_bf16_kernel", "few_scores_kernel", "logits_kernel", "select_kernel"}


@pytest.mark.parametrize("file,kernel,body", REACHING, ids=[k[1] for k in REACHING])
def test_a_cluster_barrier_stands_before_the_first_remote_access(file, kernel, body):
    barrier = BARRIER.search(body)
    assert barrier and barrier.start() < REMOTE.search(body).start(), (file, kernel)


@pytest.mark.parametrize("file,kernel,body", REACHING, ids=[k[1] for k in REACHING])
def test_warps_converge_before_a_cluster_barrier(file, kernel, body):
    """The barriers are the .aligned ones: a branch on the thread just before one is closed by a warp or CTA
    barrier."""
    for m in BARRIER_OR_ARRIVE.finditer(body):
        before = body[:m.start()].rstrip()
        # the barrier's own condition, alike in every thread
        before = re.sub(r"if (constexpr )?\([^()]*\)\s*\{?$", "", before).rstrip()
        while before.endswith("}"):  # the blocks that end here, from the outermost to the innermost
            depth, at = 0, len(before)
            while True:
                at -= 1
                depth += {"}": 1, "{": -1}.get(before[at], 0)
                if depth == 0:
                    break
            head = before[:at].rstrip().rsplit("\n", 1)[-1]
            assert not re.search(r"\btid\b|threadIdx\.x|\blane\b|\bwarp\b", head), (file, kernel, head.strip())
            before = before[at + 1:-1].rstrip()


def test_the_streamed_passs_loads_wait_for_the_pass_before():
    """Stages from the third tile on come free only behind the pass before: the loading warp waits for that grid
    itself before it enters a bounded wait for one."""
    body = next(k[2] for k in _kernels() if k[1] == "tensor_pass_kernel")
    loads = body[body.index("if (warp == 0) {\n    \n"):body.index("} else if (warp == 1)")]
    free = loads.index("mbar_wait(&bar_empty")
    assert re.search(r"kPass == kStream && i == kStages \+ 2\) griddep_wait\(\)", loads[:free])
    # what is issued ahead: products 0 and 1
    assert "kPass == kStream && i == 2 && w == 0) griddep_wait()" in body


def test_clusters_that_are_not_portable_are_asked_for():
    """A size that the kernel may be launched with, or half of it: where one attribute is set, so is the question."""
    users = [p for p in sorted(CSRC.glob("*.cu")) if re.search(r"(kMaxCluster|kMaxOne) = 16", p.read_text())]
    assert {p.name for p in users} >= {"key_weights_sm100.cu", "logits.cu"}
    for path in users:
        text = path.read_text()
        assert "NonPortable" not in text and text.count("larger_cluster(") >= 1, path.name
    text = (CSRC / "launch.cuh").read_text()
    asked = text[text.index("int larger_cluster("):]
    assert asked.index("NonPortableClusterSizeAllowed") < asked.index("cudaOccupancyMaxActiveClusters")
