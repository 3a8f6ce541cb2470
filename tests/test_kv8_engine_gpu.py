"""An engine whose cache is held in 8 bits: its products, the write, the attention over it and the copies of pages together."""
import numpy as np
import pytest
import torch

import plain_gpt2 as P
import plain_kv8 as P8
from tiny import TINY, write_tiny

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B = 16


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return write_tiny("B_sharp", str(tmp_path_factory.mktemp("models")))


def engine(folder, dtype="float32", **kw):
    from rosellm_b200.engine.llm import InferenceEngine

    return InferenceEngine(folder, dtype=dtype, kv_cache_dtype="fp8", **({"page_size": 16, "max_batch_size": 6, "kv_cache_max_tokens": 2048} | kw))


def runner(folder, dtype="float32", **kw):
    return engine(folder, dtype, **kw).runner


def entry(slot, ids, want):
    from rosellm_b200.engine import StepEntry

    return StepEntry(slot, ids, want)


def cached(r, layer, slot, n):
    """(keys and values [n, 2, heads, dim], scales [n, 2, heads]) of a request, in 64 bits."""
    g = r.cache.groups[r.cache.group_of_layer[layer]]
    at = torch.arange(n)
    pages = torch.tensor(g.table[slot])[at // r.cache.page_size].long()
    rows = at % r.cache.page_size
    scales = r.cache.kv_scales(layer).cpu().double()[pages, :, :, rows // B]
    return P8.values_of(r.cache.kv_pool(layer))[pages, :, :, rows] * scales[..., None], scales


def plain_step(cfg, t, r, slot, ids, first):
    """Logits of ``ids[first:]`` from the formulas in 64 bits, with the keys and values that the cache holds; what it holds of the new ones is
    checked to be what rounding to the code allows.

    A key or value x of the layer is off by e from the 32-bit products before it; the code with scale s is at most half a step off: |x| 2^-4, or s 2^-10
    below the smallest normal value; where a later token of the block made the scale grow, a code below the new smallest normal value was rounded again, each time by
    half of the step 2^-9 s of that time, and the scales at least doubled: altogether less than s 2^-9."""
    D, H, eps = cfg["n_embd"], cfg["n_head"], cfg.get("layer_norm_epsilon", 1e-5)
    dh, n = D // H, len(ids)
    x = t["wte.weight"][torch.tensor(ids[first:])] + t["wpe.weight"][first:n]
    act = P.activation_of(cfg.get("activation_function", "gelu_new"))
    for i in range(cfg["n_layer"]):
        p = f"h.{i}."
        qkv = P.layer_norm(x, t[p + "ln_1.weight"], t[p + "ln_1.bias"], eps) @ t[p + "attn.c_attn.weight"] + t[p + "attn.c_attn.bias"]
        q, k, v = (a.view(-1, H, dh) for a in qkv.split(D, dim=-1))
        kv, scales = cached(r, i, slot, n)
        exact = torch.stack([k, v], dim=1)
        off = (kv[first:] - exact).abs()
        allowed = exact.abs() * 2.0 ** -4 + scales[first:, ..., None] * 2.0 ** -9 + 1e-4 * exact.abs().amax()
        assert (off <= allowed).all(), (i, float((off / allowed).max()))
        assert off.max() > 0  # it is a rounded cache
        s = torch.einsum("qhd,khd->hqk", q, kv[:, 0]) * dh ** -0.5
        s = s.masked_fill(torch.arange(n)[None] > torch.arange(first, n)[:, None], float("-inf"))
        o = torch.einsum("hqk,khd->qhd", torch.softmax(s, dim=-1), kv[:, 1]).reshape(-1, D)
        x = x + o @ t[p + "attn.c_proj.weight"] + t[p + "attn.c_proj.bias"]
        h = P.layer_norm(x, t[p + "ln_2.weight"], t[p + "ln_2.bias"], eps)
        x = x + P.mlp(h, t[p + "mlp.c_fc.weight"], t[p + "mlp.c_fc.bias"], t[p + "mlp.c_proj.weight"], t[p + "mlp.c_proj.bias"], act)
    return P.layer_norm(x, t["ln_f.weight"], t["ln_f.bias"], eps) @ t["wte.weight"].t()


def check(logits, want):
    """32 bits throughout: the tolerance of the engine's own cache type, 1e-4 of the logits' size."""
    got = logits.cpu().double()
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4 * max(1.0, float(want.abs().max())))


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("page", [16, 48])
def test_steps(folder, graphs, page):
    """Prompts in portions, decoded tokens, both in one step, and a batch filled up with padding (three requests in the graph of four)."""
    cfg, t = P.load_folder(folder)
    r = runner(folder, page_size=page, cuda_graphs=graphs)
    rng = np.random.default_rng(0)
    ids = [rng.integers(0, 1000, n).tolist() for n in (90, 140, 33)]
    slots = [r.cache.new_request() for _ in ids]
    at = [0, 0, 0]
    for step in ([70, 100, 0], [1, 30, 31], [1, 1, 1], [1, 1, 1], [5, 1, 0], [1, 1, 0], [1, 1, 0]):
        entries = [entry(slots[i], ids[i][at[i]:at[i] + n], list(range(n))) for i, n in enumerate(step) if n]
        logits = r.step(entries).clone()
        r.check_status()
        row = 0
        for i, n in enumerate(step):
            if n:
                check(logits[row:row + n], plain_step(cfg, t, r, slots[i], ids[i][:at[i] + n], at[i]))
                at[i] += n
                row += n
    for s in slots:
        r.cache.release(s)
    r.cache.check()


@pytest.mark.parametrize("tokens", [1, 16, 45])
def test_a_fork_goes_its_own_way(folder, tokens):
    """Both requests go on, with other tokens, in one step: each as if it had been alone with what was cached when it was forked."""
    cfg, t = P.load_folder(folder)
    r = runner(folder)
    rng = np.random.default_rng(tokens)
    ids = rng.integers(0, 1000, tokens).tolist()
    a = r.cache.new_request()
    r.step([entry(a, ids, [])])
    before = [cached(r, layer, a, tokens)[0] for layer in range(cfg["n_layer"])]
    b = r.fork(a)
    one, two = list(ids), list(ids)
    for n in (1, 20, 1):
        more = [rng.integers(0, 1000, n).tolist() for _ in range(2)]
        logits = r.step([entry(a, more[0], list(range(n))), entry(b, more[1], list(range(n)))]).clone()
        check(logits[:n], plain_step(cfg, t, r, a, one + more[0], len(one)))
        check(logits[n:], plain_step(cfg, t, r, b, two + more[1], len(two)))
        one, two = one + more[0], two + more[1]
    r.check_status()
    whole = tokens // 16 * 16
    for layer, was in enumerate(before):
        assert torch.equal(cached(r, layer, b, tokens)[0][:whole], was[:whole]) and torch.equal(cached(r, layer, a, tokens)[0][:whole], was[:whole])
    r.cache.check()
    r.cache.release(a)
    c = r.fork(b)
    r.cache.release(b)
    assert c is not None
    r.cache.release(c)
    r.cache.check()


@pytest.mark.parametrize("overlap", [False, True])
def test_requests_that_fork(folder, overlap):
    """Through the engine: greedy forks give the first one's tokens, sampled ones go their own ways, also while others come and go."""
    e = engine(folder, overlap_schedule=overlap, max_batch_size=4)
    rng = np.random.default_rng(1)
    prompt = rng.integers(0, 1000, 37).tolist()
    a = e.add_request(prompt_token_ids=prompt, max_new_tokens=24, stop_on_eos=False)
    other = e.add_request(prompt_token_ids=prompt[:9], max_new_tokens=40, stop_on_eos=False)
    with pytest.raises(ValueError, match="waiting"):
        e.fork_request(a)
    reported = {}

    def run(n):
        while n and e.has_unfinished():
            for rid, tok in e.step().items():
                reported.setdefault(rid, []).append(tok)
            n -= 1

    run(8)
    have = len(e.get_generated_ids(a))
    b = e.fork_request(a)
    have_b = len(e.get_generated_ids(b))
    assert have <= have_b < 24
    c = e.fork_request(a, new_request_id="c", seed=5, sampling_params=e._requests[a].params.__class__(
        max_new_tokens=24, do_sample=True, temperature=5.0, stop_on_eos=False))
    with pytest.raises(ValueError, match="exists"):
        e.fork_request(a, new_request_id="c")
    with pytest.raises(ValueError, match="running"):
        e.fork_request(a)  # four run already
    run(1000)
    assert sorted(map(str, e.pop_finished_ids())) == sorted(map(str, [a, other, b, c]))
    out = {rid: e.pop_response(rid).token_ids for rid in (a, other, b, c)}
    assert [len(out[i]) for i in (a, other, b, c)] == [24, 40, 24, 24]
    assert reported[a] == out[a] and reported[other] == out[other]
    assert out[b][:have_b] == out[a][:have_b] == out[c][:have_b] and reported[b] == out[b][have_b:] and reported["c"] == out[c][have_b:]
    assert out[b] == out[a] and out[c] != out[a]
    e.runner.cache.check()
    assert e.runner.cache.num_free_slots == 4


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_same_tokens_again(folder, dtype):
    """Two engines of the same options, with graphs and launches issued again, generate the same tokens twice; and the second run of one as well."""
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (5, 60, 17, 120)]
    runs = []
    for _ in range(2):
        e = engine(folder, dtype)
        for _ in range(2):
            runs.append(e.generate_batch(prompts, max_new_tokens=30, stop_on_eos=False))
    assert all(run == runs[0] for run in runs) and all(len(o) == 30 for o in runs[0])


def test_models_that_8_bits_do_not_fit(tmp_path):
    from rosellm_b200.config.base import ConfigError
    from rosellm_b200.engine.llm import InferenceEngine

    with pytest.raises(ValueError, match="head size 16"):
        InferenceEngine(write_tiny("A", str(tmp_path)), kv_cache_dtype="fp8")
    import tiny_lebedra

    name = next(iter(tiny_lebedra.TINY))
    with pytest.raises((ConfigError, ValueError)):
        InferenceEngine(tiny_lebedra.write_tiny(name, str(tmp_path)), kv_cache_dtype="fp8")
    with pytest.raises(ConfigError, match="multiple of 16"):
        engine(write_tiny("B", str(tmp_path)), page_size=8)


@pytest.mark.parametrize("family,name", [("", "B_sharp"), ("lebedra", "X"), ("porovik", "A"), ("porovik", "B"), ("fikevik", "A"), ("fikevik", "B"), ("soporax", "A"),
                                         ("soporax", "B"), ("vebotar", "A"), ("vebotar", "B"), ("kugadra", "A"), ("kugadra", "B")])
def test_forks_of_other_caches(family, name, tmp_path):
    """Latent rows, biased rows, windows, chunks, states and several copies of a stack, in the engine's own type: a fork and the first request, going on
    with the same tokens and with others, each give what a request gives that was never forked.  Both sides lie within 1e-4 of the logits' size
    of the formulas (the replay tests' tolerance of 32 bits), so within twice that of one another."""
    import importlib
    import inspect

    from rosellm_b200.engine.llm import InferenceEngine

    mod = importlib.import_module(f"tiny_{family}" if family else "tiny")
    more = dict(decisive=True) if "decisive" in inspect.signature(mod.write_tiny).parameters else {}
    r = InferenceEngine(mod.write_tiny(name, str(tmp_path), **more), dtype="float32", page_size=mod.TINY[name]["page_size"], max_batch_size=6,
                        kv_cache_max_tokens=1024, cuda_graphs=False).runner
    vocab = r.config.vocab_size if hasattr(r.config, "vocab_size") else 100
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, vocab, 37).tolist()
    steps = [([t], [t]) for t in rng.integers(0, vocab, 2).tolist()] + [(rng.integers(0, vocab, 5).tolist(), rng.integers(0, vocab, 5).tolist()), ([3], [4]), ([6], [6])]
    a = r.cache.new_request()
    r.step([entry(a, prompt[:20], [])])
    r.step([entry(a, prompt[20:], [])])
    b = r.fork(a)
    r.cache.check()
    got = [r.step([entry(a, x, list(range(len(x)))), entry(b, y, list(range(len(y))))]).clone() for x, y in steps]
    r.cache.check()
    r.cache.release(a)
    r.cache.release(b)
    r.cache.check()
    alone = [r.cache.new_request() for _ in range(2)]
    for s in alone:
        r.step([entry(s, prompt[:20], [])])
        r.step([entry(s, prompt[20:], [])])
    for g, (x, y) in zip(got, steps):
        want = r.step([entry(alone[0], x, list(range(len(x)))), entry(alone[1], y, list(range(len(y))))])
        torch.testing.assert_close(g, want, rtol=0, atol=2e-4 * max(1.0, float(want.abs().max())))
    r.check_status()


def test_the_command_line(folder):
    """The ids that the command line prints with ``--kv-cache-dtype fp8`` are those that the engine gives with the same options."""
    from test_cli_gpu import printed_ids, run_cli

    prompt = [5, 17, 3, 250, 9, 44, 101]
    out = run_cli("--model", folder, "--dtype", "fp32", "--kv-cache-dtype", "fp8", "--prompt-ids", ",".join(map(str, prompt)), "--max-new-tokens", "8",
                  "--no-stop-on-eos")
    e = engine(folder)
    assert printed_ids(out, False) == e.generate_batch([prompt], max_new_tokens=8, stop_on_eos=False)[0]
