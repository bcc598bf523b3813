"""Waits of the tree kernels whose violation would stop a GPU: shown on the sources, never by running a kernel that breaks them."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "mllm_b200" / "csrc"


def test_warps_that_may_give_up_meet_at_bounded_waits():
    """A softmax warp of tree attention leaves its loop when a wait runs out.  Warps that met at a named barrier would then wait for it without
    an end; mbarrier waits give up with it."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", (CSRC / "attention_tree.cu").read_text(), flags=re.S)
    assert "mbar_wait(" in text
    assert not re.search(r"\b(bar|barrier(\.cta)?)\.(sync|red|arrive)\b", text)
