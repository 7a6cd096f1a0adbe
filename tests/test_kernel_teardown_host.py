"""Every kernel that starts asynchronous loads ends an aborted CTA by waiting for them (its waits run out
only where something is broken, which no test makes happen in a product kernel; this reads the sources)."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "3d-dit-distillation_b200" / "csrc"
LOAD = re.compile(r"\b(tma_load_\w+|load_box<CG>|(?:tc::)?bulk_load|bulk_copy|tma_gather4)\(")
FILES = {p.name: re.sub(r"//.*", "", p.read_text()) for p in sorted(CSRC.glob("*.cu"))}
LOADING = [n for n, s in FILES.items() if LOAD.search(s)]


def test_the_kernels_with_loads_are_found():
    assert {"attention.cu", "gemm.cu", "dense_conv.cu", "dwconv_plan.cu", "rowops.cu", "unpatchify.cu", "mxlinear.cu",
            "kvcache.cu"} <= set(LOADING)


@pytest.mark.parametrize("name", LOADING)
def test_an_aborted_cta_waits_for_its_loads(name):
    text = FILES[name]
    # the shared helpers, or a wait of its own that no abort flag ends early
    assert re.search(r"\bdrain_(pair_)?loads\(", text) or "no_abort" in text or \
        re.search(r"for \(int64_t j = \(issued > 2 \? issued - 2 : 0\); j < issued; \+\+j\)\s*mbar_wait\(", text)


@pytest.mark.parametrize("name", ["attention.cu", "gemm.cu", "mxlinear.cu", "dense_conv.cu"])
def test_tensor_memory_is_freed_after_the_last_product(name):
    """After an abort a commit on a barrier of its own, and a wait for it, stand before the deallocation."""
    text = FILES[name]
    assert text.index("drained") < text.index("tcgen05.dealloc")
    assert re.search(r"tc_commit_(pair_)?elect\((smem_u32\(&sm\.drained\)|b_drained)", text)


@pytest.mark.parametrize("name", ["gemm.cu", "mxlinear.cu"])
def test_a_cta_of_a_pair_leaves_after_every_commit_on_its_stages(name):
    """The tensor core delivers a commit to both CTAs by itself; each waits for the last one of every stage."""
    assert re.search(r"for \(int j = max\(0, it - (NST|STAGES)\); ok && j < it; \+\+j\)\s*"
                     r"ok = mbar_wait\(smem_u32\(&sm\.empty\[", FILES[name])


def test_cluster_barriers_are_for_whole_warps():
    """The aligned form of the cluster barrier stands in one place, behind a warp barrier."""
    header = re.sub(r"//.*", "", (CSRC / "tc.cuh").read_text())
    assert re.search(r"void cluster_sync\(\) \{\s*__syncwarp\(\);\s*asm volatile\(\s*\"barrier\.cluster\.arrive", header)
    assert len(re.findall(r"barrier\.cluster", header)) == 2 and not any("barrier.cluster" in t for t in FILES.values())
