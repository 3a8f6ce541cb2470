"""The 8-bit cache and forks at the ends of their ranges, as far as no device is needed; what only the sources can show."""
import os
import re

import torch

from rosellm_b200.ops import kernels as K

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rosellm_b200", "csrc")


def test_the_next_block_is_asked_for_when_all_lanes_have_read_the_answer():
    """Both answers lie in one place of shared memory, written by the device's asynchronous part: between a reading by all lanes and one lane's next
    question the warp has to meet."""
    source = open(os.path.join(CSRC, "kv8_attention.cuh")).read()
    loops = re.findall(r"for \(uint32_t n = 0;; \+\+n\) \{\n(.*?)read_answer\(", source, re.S)
    asking = [body for body in loops if "ask_for_block(" in body]
    assert len(asking) == 1 == len(re.findall(r"\bask_for_block\(base", source)) == len(re.findall(r"\bread_answer\(base", source))
    assert "__syncwarp();" in asking[0].split("ask_for_block(")[0]


def test_a_pool_without_pages_is_refused():
    """The tcgen05 kernel reads the pool's first page in the place of one that is not there (its keys are hidden): there has to be one."""
    at = torch.zeros(64).data_ptr()

    def attend(rows, sms, n_pages):
        return K._lib().rl_kv8_attention(1, at, 128, at, at, at, 1, 1, at, at, at, at, 128, at, 1, 1, 1, 2, 1, 64, 16, n_pages, 0, 1.0,
                                         rows, 1, sms, 148, at, at, at, at, None)

    assert [attend(128, 148, 0), attend(8, 0, 0), attend(64, 148, -1)] == [-11] * 3


def test_plans_that_are_kept_are_few(monkeypatch):
    """A process whose contexts grow by a token a step, in batches of ever other sizes, keeps a bounded number of plans, the same for contexts that are
    treated alike."""
    monkeypatch.setattr(K, "device_facts_given", (148, 233472))
    monkeypatch.setattr(K, "_KV8_PLANS", {})
    size = dict(dtype=torch.bfloat16, n_heads=12, n_kv=12, head_dim=64, page_size=16)
    plans = {K.kv8_attention_plan(span=span, n_tiles=4, max_q=64, n_decode=3, **size) for span in range(512, 20000)}
    assert len(K._KV8_PLANS) <= 4 and len(plans) <= 2
    for n in range(1, 6000):
        K.kv8_attention_plan(span=3000, n_tiles=n, max_q=64, n_decode=n, **size)
        assert len(K._KV8_PLANS) <= 4096
    assert K.kv8_attention_plan(span=511, n_tiles=4, max_q=64, **size) != K.kv8_attention_plan(span=512, n_tiles=4, max_q=64, **size)
