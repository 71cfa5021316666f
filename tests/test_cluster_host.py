"""Thread-block clusters, by reading the kernels: a CTA's shared memory is reached
by the others only behind a cluster barrier, which is what tells that the CTA runs."""
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


REACHING = [k for k in _kernels() if REMOTE.search(k[2])]


def test_the_reading_finds_the_cluster_kernels():
    assert {k[1] for k in REACHING} >= {"decode_bf16_kernel", "few_scores_kernel", "logits_kernel", "select_kernel"}


@pytest.mark.parametrize("file,kernel,body", REACHING, ids=[k[1] for k in REACHING])
def test_a_cluster_barrier_stands_before_the_first_remote_access(file, kernel, body):
    barrier = BARRIER.search(body)
    assert barrier and barrier.start() < REMOTE.search(body).start(), (file, kernel)
