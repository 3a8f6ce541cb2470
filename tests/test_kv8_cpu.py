"""The 8-bit cache and requests that go on as two, as far as the host has to do with them; what the C entry points refuse."""
import random

import numpy as np
import pytest
import torch

from rosellm_b200.cache import CacheManager, IdAllocator
from rosellm_b200.cache.sizing import kv_bytes_per_token
from rosellm_b200.config.base import ConfigError
from rosellm_b200.config.engine import EngineConfig
from rosellm_b200.ops import kernels as K
from rosellm_b200.parts import KVCacheSpec, StateSpec
from rosellm_b200.sampling.params import SamplingParams
from test_scheduler_cpu import fake_token, make, run_all, run_step


# ---- options, sizes ----------------------------------------------------------------------------

def test_option():
    assert EngineConfig().kv_cache_dtype == "auto"
    assert EngineConfig(kv_cache_dtype="fp8_e4m3", page_size=32).kv_cache_dtype == "fp8"
    for kw in (dict(kv_cache_dtype="int4"), dict(kv_cache_dtype="fp8", page_size=8), dict(kv_cache_dtype="fp8", page_size=24)):
        with pytest.raises(ConfigError):
            EngineConfig(**kw)


def test_bytes_of_a_token():
    """A byte an entry and a quarter of a byte a row: 12 heads of 64, keys and values, 1536 + 6; rounded up over the layers together."""
    assert kv_bytes_per_token([KVCacheSpec(12, 64, None)], "bfloat16") == 2 * 2 * 12 * 64
    assert kv_bytes_per_token([KVCacheSpec(12, 64, None)], "bfloat16", True) == 1542
    assert kv_bytes_per_token({0: KVCacheSpec(1, 32, None)}, "float32", True) == 65
    assert kv_bytes_per_token([KVCacheSpec(1, 32, None)] * 2, "float32", True) == 129


@pytest.mark.parametrize("kw", [dict(page_size=8), dict(dim=48), dict(dim=288), dict(planes=1)])
def test_what_8_bits_do_not_take(kw):
    spec = KVCacheSpec(2, kw.get("dim", 64), None, planes=kw.get("planes", 2))
    with pytest.raises(ValueError, match="8 bits"):
        CacheManager({0: spec}, {}, page_size=kw.get("page_size", 16), num_pages=4, max_slots=2, max_seq_len=64, device="cpu", eight_bits=True)


def test_pools_of_8_bits():
    m = CacheManager({0: KVCacheSpec(2, 64, None), 1: KVCacheSpec(3, 32, 20)}, {}, page_size=32, num_pages=5, max_slots=2, max_seq_len=64,
                     dtype=torch.bfloat16, device="cpu", eight_bits=True)
    assert m.kv_pool(0).dtype == torch.float8_e4m3fn and m.kv_pool(0).shape == (5, 2, 2, 32, 64)
    assert m.kv_scales(0).dtype == torch.float32 and m.kv_scales(1).shape == (5, 2, 3, 2)
    plain = CacheManager({0: KVCacheSpec(2, 64, None)}, {}, page_size=8, num_pages=5, max_slots=2, max_seq_len=64, device="cpu")
    assert plain.kv_scales(0) is None and not plain.eight_bits


# ---- pages with several holders ------------------------------------------------------------------

def test_shared_ids():
    a = IdAllocator(3)
    one, two = a.alloc(2)
    a.share([one, one])
    assert (a.holders(one), a.holders(two), a.num_held) == (3, 1, 2)
    a.free([one])
    a.free([one])
    assert a.is_held(one) and a.num_free == 1
    a.free([one, two])
    assert not a.is_held(one) and a.num_free == 3
    a.check()
    for ids in ([one], [5], [-1]):
        with pytest.raises(ValueError):
            a.share(ids)


def manager(eight_bits, window=None, pages=12, state=False):
    kv = {0: KVCacheSpec(2, 32, None), 1: KVCacheSpec(1, 64, window)}
    return CacheManager(kv, {0: StateSpec((3,), torch.float32)} if state else {}, page_size=16, num_pages=pages, max_slots=4, max_seq_len=128,
                        device="cpu", eight_bits=eight_bits)


def fill(m):
    g = torch.Generator().manual_seed(0)
    for group in m.groups:
        for t in group.pools.values():
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        for t in group.scales.values():
            t.copy_(torch.rand(t.shape, generator=g))


def bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


@pytest.mark.parametrize("eight_bits", [False, True])
@pytest.mark.parametrize("tokens", [0, 1, 15, 16, 17, 48, 61])
def test_fork(eight_bits, tokens):
    m = manager(eight_bits)
    fill(m)
    s = m.new_request()
    if tokens:
        assert m.reserve(s, tokens)
        m.commit(s, tokens)
    assert m.reserve(s, 40)  # for a step that is yet to be issued
    held = [g.allocator.num_held for g in m.groups]
    f = m.fork(s)
    assert f not in (None, s) and m.num_tokens[f] == tokens
    whole, rest = divmod(tokens, 16)
    for g, before in zip(m.groups, held):
        a, b = g.table[s], g.table[f]
        assert (a[:whole] == b[:whole]).all() and (b[whole + (rest > 0):] == -1).all()
        assert g.allocator.num_held == before + (rest > 0)
        assert [g.allocator.holders(int(p)) for p in a[:whole]] == [2] * whole
        if rest:
            assert a[whole] != b[whole]
            for t in (*g.pools.values(), *g.scales.values()):
                assert torch.equal(bits(t[int(a[whole])]), bits(t[int(b[whole])]))
    # both go on, and neither's pages are the other's
    assert m.reserve(f, 30)
    m.commit(f, 30)
    m.commit(s, 40)
    for g in m.groups:
        assert not set(g.table[s, whole:].tolist()) & set(g.table[f, whole:].tolist()) - {-1}
    first, second = (s, f) if tokens % 2 else (f, s)
    m.release(first)
    m.check()
    assert all(g.allocator.holders(int(p)) == 1 for g in m.groups for p in g.table[second, :whole])
    m.release(second)
    m.check()
    assert m.num_free_pages == 12 and m.num_free_slots == 4


def test_fork_of_a_window_and_of_state():
    m = manager(True, window=20, state=True)
    s = m.new_request()
    m.sync_to_device() if m.device.type == "cuda" else m._slots_to_reset.clear()
    m.state(0)[s] = torch.tensor([1.0, 2.0, 3.0])
    assert m.reserve(s, 70)
    m.commit(s, 70)
    f = m.fork(s)
    assert m.state(0)[f].tolist() == [1.0, 2.0, 3.0]
    m.check()
    for slot in (f, s):  # each gives back what its window has left behind, by itself
        assert m.reserve(slot, 20)
        m.commit(slot, 20)
    m.check()
    m.release(s)
    m.release(f)
    assert m.num_free_pages == 12
    a = m.new_request()
    b = m.fork(a)  # nothing has run: zeros for both
    assert sorted(m._slots_to_reset) == sorted([a, b])


def test_fork_takes_nothing_when_it_cannot():
    m = manager(True, pages=3)
    s = m.new_request()
    assert m.reserve(s, 40)
    m.commit(s, 40)
    assert m.fork(s) is None  # no page for the third, partly filled one
    assert m.num_free_slots == 3 and m.num_free_pages == 0
    m.check()
    assert m.reserve(s, 8)
    m.commit(s, 8)
    forks = [m.fork(s) for _ in range(4)]  # whole pages alone: they cost slots only
    assert None not in forks[:3] and forks[3] is None
    m.check()
    m.release(forks[0])
    with pytest.raises(ValueError, match="not live"):
        m.fork(forks[0])


# ---- requests ------------------------------------------------------------------------------------

@pytest.mark.parametrize("seed", range(8))
def test_random_workloads_with_forks(seed):
    """Forks at random moments in a cache that is often full: each request, forked or not, gets the tokens that it gets alone, all ends, and
    everything is given back."""
    rnd = random.Random(seed)
    page, max_len, seqs = rnd.choice([1, 4, 8]), 48, rnd.randint(2, 6)
    pages = -(-max_len // page) + rnd.randint(0, max_len // page)
    s, cache = make(pages=pages, page=page, seqs=seqs, budget=rnd.randint(4, 40), chunk=rnd.randint(2, 20), max_len=max_len)
    alive, step, forked = [], 0, 0
    while step < 60 or s.has_unfinished():
        if step < 60 and rnd.random() < 0.3:
            n = rnd.randint(1, max_len - 2)
            alive.append(s.add_request([rnd.randint(1, 90) for _ in range(n)], SamplingParams(max_new_tokens=rnd.randint(1, max_len - n), stop_on_eos=False)))
        if step < 60 and s.running and rnd.random() < 0.4:
            req = rnd.choice(s.running)
            full = len(s.running) >= seqs

            def fork_slot(slot):
                got = cache.fork(slot)
                if got is None:
                    raise RuntimeError("full")
                return got

            try:
                new = s.fork(req, fork_slot)
            except (ValueError, RuntimeError):
                assert full or cache.num_free_pages == 0 or cache.num_free_slots == 0
            else:
                forked += 1
                assert new.seed != req.seed and new.all_ids == req.all_ids
                alive.append(new)
            cache.check()
        if s.has_unfinished():
            run_step(s, cache)
        step += 1
        assert step < 3000
    assert forked
    for r in alive:
        c, cc = make(pages=max_len, page=page, seqs=1, budget=max_len, chunk=max_len, max_len=max_len)
        alone = c.add_request(r.prompt_ids, SamplingParams(max_new_tokens=r.params.max_new_tokens, stop_on_eos=False))
        run_all(c, cc)
        assert r.output_ids == alone.output_ids
    assert cache.num_free_pages == pages and cache.num_free_slots == seqs


def test_fork_of_a_request_that_does_not_run():
    s, cache = make()
    r = s.add_request([1, 2, 3], SamplingParams(max_new_tokens=2, seed=5))
    with pytest.raises(ValueError, match="waiting"):
        s.fork(r, cache.fork)
    run_step(s, cache)
    done = s.fork(r, cache.fork, params=SamplingParams(max_new_tokens=1))  # it has its one token already
    assert done.status == "finished" and done.finish_reason == "length" and done.output_ids == r.output_ids
    again = s.fork(r, cache.fork, params=SamplingParams(max_new_tokens=4, seed=9))
    assert again.seed == 9 and s.fork(r, cache.fork, seed=3).seed == 3
    run_all(s, cache)
    assert len(again.output_ids) == 4 and fake_token(again) is not None
    with pytest.raises(ValueError, match="finished"):
        s.fork(r, cache.fork)


# ---- plans, and what is refused before anything is launched ----------------------------------------

def test_plans(monkeypatch):
    monkeypatch.setattr(K, "device_facts_given", (148, 233472))
    monkeypatch.setattr(K, "_KV8_PLANS", {})
    size = dict(dtype=torch.bfloat16, n_heads=32, n_kv=8, head_dim=128, page_size=16)
    assert K.kv8_attention_scratch(span=700, n_decode=1, **size) == 0  # each unit has a block
    few = K.kv8_attention_scratch(span=4000, n_tiles=2, max_q=64, **size)
    assert few == K.kv8_attention_scratch(span=4000, n_tiles=2, max_q=1000, **size) > 148 * 2 * 128 * 130  # a tile has 64 queries at most
    assert K.kv8_attention_plan(span=4000, n_tiles=2, max_q=64, **size) != K.kv8_attention_plan(span=400, n_tiles=2, max_q=64, **size)
    assert K.kv8_attention_plan(span=4000, n_tiles=2, max_q=64, window=100, **size) == K.kv8_attention_plan(span=164, n_tiles=2, max_q=64, **size)
    assert K.kv8_attention_scratch(span=1 << 30, n_tiles=5000, max_q=64, **size) == 0  # more blocks of rows than the plan holds


def test_entries_refuse():
    some = torch.zeros(64, dtype=torch.float32)
    at = some.data_ptr()

    def write(dtype=1, stride=64, k=at, dim=64, page=16, heads=1):
        return K._lib().rl_kv8_write(dtype, k, stride, at, stride, at, at, at, 1, 1, at, at, at, at, 1, 1, heads, dim, page, 1, 1, at, None)

    assert [write(dim=80), write(dim=288), write(dim=0), write(page=8), write(page=0), write(stride=12), write(k=at + 8), write(heads=0)] == \
        [-2, -2, -2, -3, -3, -4, -4, -5]

    def attend(dtype=1, dim=64, heads=2, kv=1, page=16, rows=8, row_blocks=1, sms=0, blocks=0, scratch=at, status=at, items=1):
        return K._lib().rl_kv8_attention(dtype, at, 128, at, at, at, 1, 1, at, at, at, at, 128, at, items, 0, 1, heads, kv, dim, page, 1, 0, 1.0,
                                         rows, row_blocks, sms, blocks, scratch, scratch, scratch, status, None)

    assert attend(items=0) == 0
    assert [attend(dim=48), attend(heads=3, kv=2), attend(page=24), attend(rows=12), attend(row_blocks=0), attend(rows=128), attend(rows=128, dtype=0, sms=4),
            attend(rows=128, dim=96, sms=4), attend(rows=128, page=8192, sms=4), attend(kv=0), attend(sms=4, blocks=0), attend(sms=4, blocks=4, scratch=None),
            attend(status=None)] == [-2, -3, -4, -5, -5, -5, -5, -5, -5, -3, -7, -7, -8]


def test_wrappers_refuse_what_is_not_on_a_device():
    pool, scales = torch.zeros(4, 2, 1, 16, 32, dtype=torch.float8_e4m3fn), torch.zeros(4, 2, 1, 1)
    ints = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: K.kv8_write(scales, scales, pool, scales, ints, ints, ints, ints, ints, 4),
                 lambda: K.kv8_attention(scales, pool, scales, ints, ints, ints, ints, scales, n_heads=1, scale=1.0, span=4),
                 lambda: K.PagePools([pool])):
        with pytest.raises(K.KernelError, match="CUDA"):
            call()
    with pytest.raises(K.KernelError, match="the pool must be"):
        K.kv8_write(scales, scales, pool[0], scales, ints, ints, ints, ints, ints, 4)
    assert np.all([K.kv8_fits(16, 32), K.kv8_fits(4096, 256), not K.kv8_fits(0, 64), not K.kv8_fits(16, 0), not K.kv8_fits(16, 272)])
