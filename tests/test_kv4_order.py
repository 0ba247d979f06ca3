"""CPU test of an ordering in the prompt kernel's source: an mbarrier arrival
publishes what its own lane stored before it, and what other lanes stored only
where the warp has synchronised in between."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "zero_b200" / "csrc"


def test_the_loading_warps_flags_are_ordered_before_their_arrival():
    """Eight lanes store a key tile's flags (s_bad); lane 0 arrives on rfull."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "kv4_prompt.cu").read_text())
    store = re.search(r"s_bad\[kc & 7\]\[lane\] = \w+;", text)
    arrive = re.compile(r"mbar_arrive_expect_tx\(smem_addr\(&bars\.rfull").search(text, store.end())
    assert "__syncwarp();" in text[store.end():arrive.start()]
