"""What the 8-bit product's kernels do when a bounded wait runs out cannot be run on a shared GPU without copies in flight being abandoned on
purpose, so the rules the code has to keep are checked on its source, as for the bf16 kernels."""
import re
from pathlib import Path

import pytest

KERNELS = Path(__file__).resolve().parent.parent / "csrc" / "kernels"


def _source(name):
    """The file without comments."""
    return re.sub(r"//[^\n]*", "", (KERNELS / name).read_text())


@pytest.mark.parametrize("name", ["gemm_fp8.cu", "gemm_fp8_small.cu", "gemm_fp8.cuh"])
def test_a_role_waits_as_a_whole_warp(name):
    """Lanes can get different answers from a wait that runs out: one that decides what a role does is mbar_wait_warp, or two of them."""
    text = _source(name)
    decides = re.findall(r"(?:if \(!?|=\s*|\|\| |&& |return )(mbar_wait\w*)\(", text)
    assert decides and set(decides) <= {"mbar_wait_warp", "mbar_wait_both"}
    # a single look is agreed on by the warp before it decides anything
    assert not re.findall(r"if \(!?mbar_(?:try_wait|test)\(", text)


@pytest.mark.parametrize("name", ["gemm_fp8.cu", "gemm_fp8_small.cu"])
def test_a_producer_stays_until_its_loads_have_landed(name):
    """The last thing the producer does on every path is to wait (bounded) for its last loads; the warp that brings scales and the warps that
    store results wait for their own copies."""
    text = _source(name)
    start = text.index("if (warp == 0) {\n      uint32_t" if name == "gemm_fp8.cu" else "if (warp == 0) {\n    uint32_t")
    producer = text[start:]
    producer = producer[:re.search(r"\} else if \(warp (?:< 3|== 1)\)", producer).start()]
    assert re.search(r"loads_land\(&ctl->full\[0\], NS, [^;]*\);\s*(if \(!ok\) loads_land\([^;]*;\s*\})?\s*$", producer), producer[-300:]
    assert text.count("copies_wait();") == 1 and (name == "gemm_fp8_small.cu" or "if (lane == 0) bulk_wait_all();" in text)


def test_a_loop_of_a_role_ends_with_its_first_wait_that_ran_out():
    """`ok` is looked at after every wait, and by every loop around one."""
    for name in ("gemm_fp8.cu", "gemm_fp8_small.cu"):
        for wait in re.finditer(r"\bok = [^;]*mbar_wait_\w+\([^;]*;\s*([^\n]*)", _source(name)):
            assert wait[1].startswith("if (!ok) break;"), wait[0]
    for loop in re.findall(r"for \(int t = pair; [^)]*\)", _source("gemm_fp8.cu")):
        assert "&& ok" in loop


@pytest.mark.parametrize("name,kernels", [("gemm_fp8.cu", 1), ("gemm_fp8_small.cu", 1), ("gemm_fp8_rows.cu", 1), ("fp8_quantize.cu", 3)])
def test_a_kernel_that_starts_early_waits_before_it_reads(name, kernels):
    """Every kernel launched before the one ahead has ended waits for it, in all threads, before it lets the next one start, and reads nothing
    through pointers that promise that nobody writes there."""
    text = _source(name)
    bodies = re.split(r"__global__ ", text)[1:]
    assert len(bodies) == kernels
    for body in bodies:
        wait, start = body.index("wait_for_previous();\n"), body.index("let_next_start();")
        assert wait < start and body.count("let_next_start();") == 1
        assert not re.search(r"\breturn;", body[:wait])
    assert "__ldg" not in text and not re.search(r"const \w+\*\s*__restrict__", text)
    assert "early_start()" in text or "launch_early(" in text
    if "tmem_alloc" in text:
        assert text.index("tmem_alloc") < text.index("let_next_start();")
