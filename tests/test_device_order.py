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


EARLY = sorted({(name, k) for name, text in SOURCES.items()
                for m in re.finditer(r"launch_early(?:_clusters)?\(\"([^;]*);", text)
                for k in re.findall(r"\b(\w+_kernel)\b", m.group(1))})


def test_kernels_that_begin_early_are_found():
    assert len(EARLY) >= 10 and ("logprobs.cu", "logprobs_kernel") in EARLY and ("pool_q4.cu", "append_kernel") in EARLY


@pytest.mark.parametrize("name,kernel", EARLY)
def test_a_kernel_that_begins_early_reads_through_coherent_loads(name, kernel):
    """What the stream's last kernel writes changes during the lifetime of a kernel that begins early.  So
    neither non-coherent loads (their memory has to be read-only for as long as the kernel runs) nor
    __restrict__ (it lets the compiler take such loads, or move a load up over the wait)."""
    files = [name] + [f for f in SOURCES if f.endswith(".cuh") and f in SOURCES[name] and kernel in SOURCES[f]]
    found = 0
    for f in files:
        text = SOURCES[f]
        for m in re.finditer(r"\b%s\(([^;{}]*)\)\s*\{" % kernel, text):
            found += 1
            assert "__restrict__" not in m.group(1)
            body = text[m.end():].split("\n}\n")[0]
            assert not re.search(r"\b__ldg\(|\bldg_stream\(|\.nc\b", body)
    assert found >= 1
