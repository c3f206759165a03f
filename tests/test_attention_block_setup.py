"""Who pays for the 22 instances of the attention kernel with modified scores: only their callers, one instance at a time. Read from the
source; the first call of another operator took 10 ms on a B200 while it set all of them up, and takes 6 without."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "infinity_b200" / "csrc"


def _body(name: str, head: str) -> str:
    code = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    at = code.index(head)
    return code[at:code.index("\n}", at)]


def test_the_common_set_up_leaves_the_scored_attention_out():
    assert "attention_scored" not in _body("runtime.cu", "int kernels_init_device() {")


def test_a_launch_sets_up_its_own_kernel_only():
    code = re.sub(r"//[^\n]*", "", (CSRC / "attention_scored.cu").read_text())
    assert "kernels_init_device" not in code and code.count("cudaFuncSetAttribute(") == 1
    launch = _body("attention_scored.cu", "static int as_launch(")
    assert launch.index("as_init_kernel<D, PAGED, MODE>(") < launch.index("launch_pdl(")
