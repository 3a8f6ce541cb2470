"""The 8-bit cache and forks at the ends of their ranges, as far as no device is needed; what only the sources can show."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rosellm_b200", "csrc")


def test_the_next_block_is_asked_for_when_all_lanes_have_read_the_answer():
    """Both answers lie in one place of shared memory, written by the device's asynchronous part: between a reading by all lanes and one lane's next
    question the warp has to meet."""
    source = open(os.path.join(CSRC, "kv8_attention.cuh")).read()
    loops = re.findall(r"for \(uint32_t n = 0;; \+\+n\) \{\n(.*?)read_answer\(", source, re.S)
    asking = [body for body in loops if "ask_for_block(" in body]
    assert len(asking) == 1 == len(re.findall(r"\bask_for_block\(base", source)) == len(re.findall(r"\bread_answer\(base", source))
    assert "__syncwarp();" in asking[0].split("ask_for_block(")[0]
