"""The bounded waits of the attention kernel, read from its source: a wait that runs out in some lanes of a warp only cannot be brought
about on a GPU without hanging it, and what keeps it harmless is that a warp takes one answer from every wait."""
import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parent.parent / "infinity_b200" / "csrc" / "attention_scored.cu"


def _code() -> str:
    return re.sub(r"//[^\n]*", "", SOURCE.read_text())


def test_every_wait_is_a_vote_of_its_warp():
    waits = re.findall(r"[^;{}]*\bmbar_(?:try_)?wait\w*\([^;]*;", _code())
    assert waits and all(re.search(r"__all_sync\(0xffffffffu, mbar_(try_)?wait\(bar, parity\)\)", x) for x in waits), waits


def test_every_look_is_a_vote_of_its_warp():
    """The loading warps look at barriers without waiting: what they do next hangs on the vote alone."""
    code = _code().replace("bool as_test(uint64_t* bar, uint32_t parity)", "")
    looks = re.findall(r"[^;{}]*\bas_test\([^;]*;", code)
    assert looks and all(re.match(r"\s*(bool ready =|if \(is_k && w\[t\]\.first\) ready = ready &&)", x) for x in looks), looks
    assert "if (!__all_sync(0xffffffffu, ready)) continue;" in code


def test_what_ran_out_is_set_by_votes_only():
    """The softmax warps' `failed` follows from as_wait alone, so it is the same in all lanes wherever they branch on it."""
    code = _code()
    sets = re.findall(r"[^;{}]*\bfailed = [^;]*;", code)
    assert sets and all(re.match(r"\s*(bool failed = false|if \(!(as_wait|pv_wait)\(.*\)\) failed = true)", x, re.S) for x in sets), sets
    assert re.search(r"auto pv_wait = \[&\]\(uint32_t s\) \{ return as_wait\(", code)
