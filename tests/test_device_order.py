"""What the kernels' sources have to keep to so that accesses on the device are ordered: rules that no
run can show broken with certainty, read from the text (comments taken out)."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "loopfuse_b200", "csrc")


def source(path):
    with open(path) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


SOURCES = {os.path.basename(p): source(p) for p in sorted(glob.glob(os.path.join(CSRC, "*.cu*")))}


def function_start(text, at):
    """Where the function that holds offset ``at`` begins (functions are told by their qualifiers)."""
    return max(m.start() for m in re.finditer(r"^(?:template[^\n]*\n)?(?:static )?__(?:global|device)__", text[:at], re.M))


REMOTE = [(name, m.start()) for name, text in SOURCES.items() for m in re.finditer(r"\bmap_shared_rank\(", text)]


def test_there_are_accesses_to_other_ctas_shared_memory():
    assert {name for name, _ in REMOTE} == {"decode_q4.cu", "logprobs.cu", "lora.cu"}


@pytest.mark.parametrize("name,at", REMOTE)
def test_other_ctas_shared_memory_is_reached_behind_a_cluster_barrier(name, at):
    """A CTA may touch another one's shared memory once that one is known to run, and until it ends: a
    barrier of the cluster before the first access and one after the last."""
    text = SOURCES[name]
    barrier = r"\bcluster\.sync\(\)|\bcluster_wait\(\)"
    assert re.search(barrier, text[function_start(text, at):at]), "no barrier before"
    assert re.search(barrier, text[at:].split("\n}\n")[0]), "no barrier after"
