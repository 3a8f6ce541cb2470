"""The 8-bit cache and forks at the ends of their ranges, as far as no device is needed; what only the sources can show."""
import os
import re
from types import SimpleNamespace

import pytest
import torch

from rosellm_b200.engine.llm import InferenceEngine
from rosellm_b200.ops import kernels as K
from rosellm_b200.sampling.params import SamplingParams
from test_scheduler_cpu import make

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rosellm_b200", "csrc")


def test_the_next_block_is_asked_for_when_all_lanes_have_read_the_answer():
    """Both answers lie in one place of shared memory, written by the device's asynchronous part: between a reading by all lanes and one lane's next
    question the warp has to meet."""
    source = open(os.path.join(CSRC, "kv8_attention.cuh")).read()
    loops = re.findall(r"for \(uint32_t n = 0;; \+\+n\) \{\n(.*?)read_answer\(", source, re.S)
    asking = [body for body in loops if "ask_for_block(" in body]
    assert len(asking) == 1 == len(re.findall(r"\bask_for_block\(base", source)) == len(re.findall(r"\bread_answer\(base", source))
    assert "__syncwarp();" in asking[0].split("ask_for_block(")[0]


def test_kernels_behind_are_let_in_when_a_block_has_its_tensor_memory():
    """A kernel that takes tensor memory and then waits for the kernels ahead may stand beside a block of those that has not taken its own yet, if that
    block has let it in before: both would wait for good."""
    source = open(os.path.join(CSRC, "kv8_attention_tc.cuh")).read()
    kernel = source[source.index("void kv8_attention_tc_kernel("):source.index("int launch_attention_tc(")]
    assert "pdl_begin(" not in kernel and kernel.count("launch_dependents") == 1 == kernel.count("tcgen05.alloc") == kernel.count("griddepcontrol.wait")
    own = re.search(r"if \(warp == 16\) \{(.*?)\n  \}", kernel, re.S).group(1)
    assert own.index("tcgen05.alloc") < own.index("launch_dependents") and kernel.index("launch_dependents") < kernel.index("griddepcontrol.wait")


@pytest.mark.parametrize("name", sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")) and "tcgen05.alloc" in open(os.path.join(CSRC, f)).read()))
def test_tensor_memory_comes_first_in_every_kernel_that_takes_some(name):
    """The same of the products and the attention that stand beside it on an SM."""
    source = open(os.path.join(CSRC, name)).read()
    assert source.count("launch_dependents;") == 1
    assert source.rindex("tcgen05.alloc") < source.index("launch_dependents;")


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


# ---- requests that fork, through the engine's own bookkeeping --------------------------------------

class Engine(InferenceEngine):
    """The engine's bookkeeping in overlapped mode around a model that is not there: token n of any request is 10 + n."""

    def __init__(self, **kw):
        self.scheduler, self.cache = make(**kw)
        self.runner = SimpleNamespace(fork=self.cache.fork, check_status=lambda: None)
        self.overlap_schedule, self.tokenizer = True, None
        self._inflight, self._requests, self._finished_ids = None, {}, []
        self.num_steps = self.num_preemptions = self._since_status_check = 0

    def _launch(self, plan):
        for item in plan.items:
            self.cache.commit(item.request.slot, item.count)
        sampling = [i.request for i in plan.items if i.samples]
        tokens = [10 + len(r.output_ids) for r in sampling]
        return sampling, SimpleNamespace(tokens=lambda: tokens)

    def add(self, n=3, request_id=None):
        return self.add_request(prompt_token_ids=list(range(1, 6)), request_id=request_id, sampling_params=SamplingParams(max_new_tokens=n, stop_on_eos=False))


@pytest.mark.parametrize("end", ["discard_request", "pop_response"])
def test_tokens_read_for_a_fork_are_not_reported_for_a_request_that_is_gone(end):
    """A fork reads the tokens of the step in flight, which the next call of ``step`` reports: not those of requests that the caller has meanwhile
    taken away, nor those as a later request's of the same name."""
    e = Engine()
    a, b = e.add(9, "a"), e.add(3 if end == "pop_response" else 9, "b")
    assert [e.step() for _ in range(3)] == [{}, {"a": 10, "b": 10}, {"a": 11, "b": 11}]
    f = e.fork_request(a)  # the third token of each has been sampled: b's last, where it has three
    assert e.get_generated_ids(f) == e.get_generated_ids(a) == [10, 11, 12]
    getattr(e, end)(b)
    again = e.add(2, "b")
    assert e.step() == {"a": 12}
    reported = {a: [], f: [], again: []}
    while e.has_unfinished():
        for rid, token in e.step().items():
            reported[rid].append(token)
    assert reported == {a: list(range(13, 19)), f: list(range(13, 19)), "b": [10, 11]}


def test_nothing_is_left_to_do_when_what_was_read_early_is_gone():
    e = Engine()
    a = e.add(3)
    for _ in range(3):
        e.step()
    with pytest.raises(ValueError, match="finished"):
        e.fork_request(a)  # its last token was the one in flight
    assert e.has_unfinished()  # to be reported
    e.discard_request(a)
    assert not e.has_unfinished()


def test_a_fork_without_a_name_takes_no_others():
    """Names that the engine gives itself are numbers that no request it knows of has, however the caller has numbered its own."""
    e = Engine(seqs=6)
    own = e.add(8, 1)
    e.step(), e.step()
    f = e.fork_request(own)
    names = [own, f, e.fork_request(f), e.add(8, 4), e.add(8), e.add(8)]
    assert len(set(names)) == 6 == len(e._requests)
    while e.has_unfinished():
        e.step()
    assert sorted(e.pop_finished_ids()) == sorted(names) and all(e.pop_response(n).token_ids == list(range(10, 18)) for n in names)


def test_names_of_requests_that_bring_none_are_counted():
    e = Engine()
    assert [e.add(), e.add(), e.add(3, "x"), e.add()] == [0, 1, "x", 3]
