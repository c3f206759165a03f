"""Every launch through launch_pdl takes the status that it returns: a failed launch leaves nothing for cudaGetLastError, so a status that
is dropped would be a failure that nobody reports. Read from the source, since no call makes such a launch fail."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "infinity_b200" / "csrc"


def test_every_launch_status_is_taken():
    seen = 0
    for path in sorted(CSRC.glob("*.cu")):
        code = re.sub(r"//[^\n]*", "", path.read_text())
        for at in re.finditer(r"\blaunch_pdl\(", code):
            before = code[max(0, at.start() - 40):at.start()].rstrip()
            assert before.endswith(("=", "return", "?", ":")), (path.name, before)
            seen += 1
    assert seen >= 8


def test_statuses_of_the_attention_launch_are_taken():
    code = (CSRC / "attention_tc2.cu").read_text()
    calls = re.findall(r"(.{3})\bt2_launch<", code)
    assert len(calls) == 4 and all(c.rstrip()[-1] in "?:" for c in calls), calls
