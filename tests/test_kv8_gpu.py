"""The operators of the 8-bit cache against their definition in 64 bits: writing, attention, copies of pages."""
import math

import pytest
import torch

import plain_kv8 as P

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def K():
    from rosellm_b200.ops import kernels

    kernels._lib()
    return kernels


def cache_of(batch, heads, dim, gen, spread=1.0):
    """(pool, scales) on the host, every block filled with normal values of its own size."""
    shape = (batch.n_pages, 2, heads, batch.page // 16, 16, dim)
    x = torch.randn(shape, generator=gen, dtype=torch.float64) * torch.exp(spread * torch.randn(shape[:4], generator=gen, dtype=torch.float64))[..., None, None]
    s = torch.tensor([P.scale_for(float(t)) for t in x.abs().amax(dim=(4, 5)).flatten()], dtype=torch.float64).reshape(shape[:4])
    codes = P.nearest(x / s[..., None, None]).flatten(3, 4)
    return codes.float().to(torch.float8_e4m3fn), s.float()


def packed(batch, heads, dim, dtype, gen):
    """Keys and values as the last columns of rows that hold queries too."""
    w = heads * dim
    rows = (torch.randn(batch.tokens, 3 * w, generator=gen) * torch.exp(torch.randn(batch.tokens, 1, generator=gen))).to(dtype)
    return rows[:, w:2 * w], rows[:, 2 * w:]


def do_write(K, batch, k, v, pool, scales):
    a = batch.arrays(DEV)
    K.kv8_write(k, v, pool, scales, a["block_table"], a["positions"], a["req_of_token"], a["q_start"], a["slots"], batch.table.shape[1] * batch.page)


def check_write(K, batch, heads, dim, dtype, k, v, pool, scales):
    want, s = P.values_of(pool), scales.double()
    P.write(batch, k.double().unflatten(1, (heads, dim)), v.double().unflatten(1, (heads, dim)), want, s)
    rows = torch.cat([torch.zeros_like(k), k, v], dim=1).to(DEV)
    w = heads * dim
    dp, ds = pool.to(DEV), scales.to(DEV)
    do_write(K, batch, rows[:, w:2 * w], rows[:, 2 * w:], dp, ds)
    K.check_status(DEV)
    torch.testing.assert_close(P.values_of(dp), want, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(ds.cpu().double(), s, rtol=0, atol=0)
    return dp, ds


EACH = [(1, 1), (16, 16), (17, 1), (17, 17), (31, 15), (40, 3), (48, 1), (65, 64), (100, 37), (33, 2), (15, 15), (130, 1)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,dim,page", [(1, 32, 16), (3, 64, 16), (2, 96, 48), (5, 128, 32), (1, 160, 128), (2, 192, 16), (1, 224, 64), (2, 256, 32)])
def test_write(K, dtype, heads, dim, page):
    gen = torch.Generator().manual_seed(dim + page)
    batch = P.Batch(EACH, page, seed=dim)
    pool, scales = cache_of(batch, heads, dim, gen)
    check_write(K, batch, heads, dim, dtype, *packed(batch, heads, dim, dtype, gen), pool, scales)


@pytest.mark.parametrize("each", [[(700, 700)], [(700, 650), (90, 5)], [(9 + i, 1) for i in range(70)], [(40, 40), (300, 270), (20, 20), (16, 16)]])
def test_write_of_portions_and_decoded_tokens(K, each):
    gen = torch.Generator().manual_seed(5)
    batch = P.Batch(each, 16)
    pool, scales = cache_of(batch, 2, 64, gen)
    check_write(K, batch, 2, 64, BF16, *packed(batch, 2, 64, BF16, gen), pool, scales)


def test_write_of_values_at_the_borders(K):
    batch = P.Batch([(40, 40), (20, 4), (20, 4), (20, 4), (20, 4)], 32)
    gen = torch.Generator().manual_seed(6)
    pool, scales = cache_of(batch, 1, 64, gen)
    k, v = torch.zeros(batch.tokens, 64), torch.zeros(batch.tokens, 64)
    k[0, 0], k[1, :4] = 448.0, torch.tensor([447.9, -0.01, 2.0 ** -9, 2.0 ** -10])  # needs exactly 1; the last is halfway to nothing
    k[16, 0], k[17, 1] = 448.0 * (1 + 2.0 ** -23), 3e38                              # needs a little more; the largest
    k[32:40] = 1e-40                                                                 # below the smallest scale
    v[:40] = torch.randn(40, 64, generator=gen)
    v[3, 5], v[4, 6], v[5, 7] = math.inf, -math.inf, math.nan
    v[16:32] = math.nan                                                              # nothing finite in the block
    k[40:44] = 1e6                                                                   # the scale grows by far: earlier codes vanish
    k[44:48] = 1e-6                                                                  # it stays
    k[48:52] = 30.0
    v[48:52, 3] = math.nan
    for i in range(3):                                                               # earlier codes that are NaN stay so
        page, row = batch.row_of(i + 1, 16)
        pool.view(torch.uint8)[page, 0, 0, row:row + 1, 9] = 0x7F
    check_write(K, batch, 1, 64, F32, k, v, pool, scales)


def test_write_twice_is_write_once(K):
    batch = P.Batch([(40, 9), (33, 1)], 16)
    gen = torch.Generator().manual_seed(8)
    pool, scales = cache_of(batch, 2, 64, gen)
    k, v = packed(batch, 2, 64, BF16, gen)
    dp, ds = check_write(K, batch, 2, 64, BF16, k * 50, v * 50, pool, scales)
    check_write(K, batch, 2, 64, BF16, k * 50, v * 50, dp.cpu(), ds.cpu())


@pytest.mark.parametrize("fault", ["page", "past the pool", "position", "slot", "table"])
def test_write_refuses_tokens_without_a_place(K, fault):
    batch = P.Batch([(40, 12), (20, 20)], 16)
    gen = torch.Generator().manual_seed(9)
    pool, scales = cache_of(batch, 2, 64, gen)
    k, v = packed(batch, 2, 64, BF16, gen)
    want, s = P.values_of(pool), scales.double()
    only = P.Batch([(40, 12), (20, 20)], 16)
    only.each = [(40, 12), (0, 0)]  # the second request's tokens go nowhere (its second block where the fault is a page of that)
    P.write(only, k.double().unflatten(1, (2, 64)), v.double().unflatten(1, (2, 64)), want, s)
    a = batch.arrays(DEV)
    if fault == "page":
        a["block_table"][batch.slots[1]] = -1
    elif fault == "past the pool":
        a["block_table"][batch.slots[1]] = batch.n_pages
    elif fault == "position":
        a["positions"][12:] += 1000
    elif fault == "slot":
        a["slots"][1] = 99
    else:
        a["positions"][12:] += 48  # beyond the table's columns, below max_pos
    dp, ds = pool.to(DEV), scales.to(DEV)
    K.kv8_write(k.to(DEV).contiguous(), v.to(DEV).contiguous(), dp, ds, a["block_table"], a["positions"], a["req_of_token"], a["q_start"], a["slots"],
                1000 if fault == "table" else 48)
    with pytest.raises(K.KernelError, match="position" if fault == "position" else "page"):
        K.check_status(DEV)
    torch.testing.assert_close(P.values_of(dp), want, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(ds.cpu().double(), s, rtol=0, atol=0)


# ---- attention ---------------------------------------------------------------------------------

def do_attention(K, batch, q, pool, scales, heads, *, window=None, span=None, out=None, scratch=None):
    a = batch.arrays(DEV)
    dim = pool.shape[4]
    out = torch.full((batch.tokens, heads * dim), 7.0, dtype=q.dtype, device=DEV) if out is None else out
    K.kv8_attention(q, pool, scales, a["block_table"], a["q_start"], a["kv_len"], a["slots"], out, n_heads=heads, scale=dim ** -0.5, window=window,
                    span=span or max(k for k, _ in batch.each), tiles=a["tiles"], n_tiles=len(batch.tiles), max_q=max(n for _, n in batch.each),
                    decode_reqs=a["decode_reqs"], n_decode=len(batch.single), scratch=scratch)
    return out


def compare(got, want, rough, fine, dtype):
    """Half a step of the output's own rounding, and the bound of what goes before it."""
    want, bound = want.flatten(1), (fine if dtype == F32 else rough).flatten(1)
    limit = bound + (bound + want.abs()) * torch.finfo(dtype).eps / 2 + 1e-30
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    over = ((got - want).abs() / limit).nan_to_num(0.0)
    assert over.max() <= 1.0, (float(over.max()), divmod(int(over.argmax()), want.shape[1]))


def check_attention(K, each, heads, n_kv, dim, page, dtype, *, window=None, span=None, seed=1, spread=1.0, touch=None):
    gen = torch.Generator().manual_seed(seed)
    batch = P.Batch(each, page, seed=seed)
    pool, scales = cache_of(batch, n_kv, dim, gen, spread)
    # whatever lies behind the last token is NaN, and so are the pages that nobody holds
    held = {batch.row_of(r, j) for r, (n, _) in enumerate(each) for j in range(n)}
    for p in range(batch.n_pages):
        for row in range(page):
            if (p, row) not in held:
                pool.view(torch.uint8)[p, :, :, row] = 0x7F
    q = (torch.randn(batch.tokens, heads * dim, generator=gen) * 1.5).to(dtype)
    if touch is not None:
        touch(batch, q, pool, scales)
    want = P.attention(batch, q.double().unflatten(1, (heads, dim)), P.values_of(pool), scales.double(), heads, dim ** -0.5, window)
    wide = torch.zeros(batch.tokens, heads * dim + 16, dtype=dtype, device=DEV)  # rows with a stride
    wide[:, :heads * dim] = q.to(DEV)
    got = do_attention(K, batch, wide[:, :heads * dim], pool.to(DEV), scales.to(DEV), heads, window=window, span=span)
    K.check_status(DEV)
    compare(got, *want, dtype)
    return got


DECODES = [(n, 1) for n in (1, 2, 15, 16, 17, 63, 64, 65, 127, 255, 300, 700)]
PORTIONS = [(2, 2), (5, 5), (17, 3), (64, 64), (65, 65), (200, 2), (130, 70), (333, 5), (128, 128), (91, 1)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,n_kv,dim,page", [(2, 2, 32, 16), (3, 3, 64, 16), (4, 1, 64, 48), (4, 2, 96, 16), (6, 2, 128, 64), (20, 1, 64, 16),
                                                 (2, 1, 160, 32), (2, 2, 192, 16), (3, 1, 224, 128), (2, 1, 256, 64), (17, 1, 128, 32)])
def test_decoded_tokens(K, dtype, heads, n_kv, dim, page):
    check_attention(K, DECODES, heads, n_kv, dim, page, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,n_kv,dim,page", [(1, 1, 32, 16), (3, 3, 64, 16), (4, 1, 64, 64), (5, 1, 96, 48), (4, 2, 128, 32), (1, 1, 256, 16),
                                                 (2, 1, 192, 128)])
def test_portions(K, dtype, heads, n_kv, dim, page):
    check_attention(K, PORTIONS, heads, n_kv, dim, page, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 63, 100, 400])
@pytest.mark.parametrize("each", [DECODES, PORTIONS], ids=["decoded", "portions"])
def test_windows(K, dtype, window, each):
    check_attention(K, each, 4, 2, 64, 16, dtype, window=window)


@pytest.mark.parametrize("span", [1, 300, 100000])
@pytest.mark.parametrize("each", [[(1500, 1), (3, 1), (900, 1)], [(1500, 5), (40, 2)], [(1300, 130)]], ids=["decoded", "few", "portion"])
def test_a_span_that_is_not_the_longest_context(K, span, each):
    check_attention(K, each, 2, 2, 64, 16, BF16, span=span)
    check_attention(K, each, 4, 1, 128, 32, F32, span=span)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales_that_differ_by_far(K, dtype):
    """Blocks whose values differ by factors of up to e^6 or so: those of small scale count as well."""
    check_attention(K, [(400, 1), (300, 9), (64, 64)], 2, 1, 64, 16, dtype, spread=2.0)


@pytest.mark.parametrize("each", [[(200, 1)], [(200, 150)], [(100, 3)]])
def test_nan_of_a_token_reaches_who_sees_it_alone(K, each):
    n, nq = each[0]
    at = n - nq // 2 - 1  # a token of the step, or the last

    def value(batch, q, pool, scales):
        page, row = batch.row_of(0, at)
        pool.view(torch.uint8)[page, 1, 0, row, 5] = 0x7F

    got = check_attention(K, each, 2, 2, 64, 16, BF16, touch=value)
    assert torch.isnan(got[nq - 1, 5]) and not torch.isnan(got[:, 64:]).any()

    def key(batch, q, pool, scales):
        page, row = batch.row_of(0, at)
        pool.view(torch.uint8)[page, 0, 1, row, 5] = 0x7F

    gen = torch.Generator().manual_seed(1)
    batch = P.Batch(each, 16, seed=1)
    pool, scales = cache_of(batch, 2, 64, gen)
    q = torch.randn(batch.tokens, 128, generator=gen).to(BF16).to(DEV)
    key(batch, q, pool, scales)
    got = do_attention(K, batch, q, pool.to(DEV), scales.to(DEV), 2)
    sees = torch.tensor([j >= at for j in range(n - nq, n)], device=DEV)
    assert torch.isnan(got[:, 64:]).all(dim=1).equal(sees) and not torch.isnan(got[:, :64]).any()


def test_rows_of_no_item_stay(K):
    batch = P.Batch([(40, 1), (50, 6), (30, 1)], 16)
    gen = torch.Generator().manual_seed(3)
    pool, scales = cache_of(batch, 2, 64, gen)
    q = torch.randn(batch.tokens, 128, generator=gen).to(BF16).to(DEV)
    out = torch.full((batch.tokens + 3, 128), 7.0, dtype=BF16, device=DEV)
    batch.single, batch.tiles = [2], []
    do_attention(K, batch, q, pool.to(DEV), scales.to(DEV), 2, out=out)
    assert (out[:7] == 7).all() and (out[8:] == 7).all() and not (out[7] == 7).any()


@pytest.mark.parametrize("each", [[(30, 1), (40, 1), (20, 1), (1, 1)], [(600, 64), (90, 1), (700, 100), (20, 1)]])
def test_padding(K, each):
    """Requests in negative slots, as a batch of a fixed size is filled up with: nothing is written for them, their rows of the output are zeros,
    the others are as they would be, and the status word stays clear."""
    batch = P.Batch(each, 16)
    gen = torch.Generator().manual_seed(6)
    pool, scales = (t.to(DEV) for t in cache_of(batch, 2, 64, gen))
    k, v = (x.to(DEV) for x in packed(batch, 2, 64, BF16, gen))
    q = torch.randn(batch.tokens, 256, generator=gen).to(BF16).to(DEV)
    slots = list(batch.slots)
    batch.slots = [slots[0], -1, -5, slots[3]]
    before = pool.view(torch.uint8).clone(), scales.clone()
    do_write(K, batch, k, v, pool, scales)
    out = do_attention(K, batch, q, pool, scales, 4)
    K.check_status(DEV)
    rows = [slice(batch.q_start[r], batch.q_start[r + 1]) for r in range(4)]
    assert (out[rows[1]] == 0).all() and (out[rows[2]] == 0).all()
    for r in (1, 2):
        pages = [p for p in batch.table[slots[r]].tolist() if p >= 0]
        assert pool.view(torch.uint8)[pages].equal(before[0][pages]) and scales[pages].equal(before[1][pages])
    batch.slots = slots
    alone_pool, alone_scales = before[0].clone().view(torch.float8_e4m3fn), before[1].clone()
    do_write(K, batch, k, v, alone_pool, alone_scales)
    want, rough, fine = P.attention(batch, q.cpu().double().unflatten(1, (4, 64)), P.values_of(alone_pool), alone_scales.cpu().double(), 4, 64 ** -0.5)
    for r in (0, 3):
        pages = [p for p in batch.table[slots[r]].tolist() if p >= 0]
        assert pool.view(torch.uint8)[pages].equal(alone_pool.view(torch.uint8)[pages]) and scales[pages].equal(alone_scales[pages])
        compare(out[rows[r]], want[rows[r]], rough[rows[r]], fine[rows[r]], BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_key_in_sight(K, dtype):
    """A request without keys, and one whose pages are missing: zeros, and the status word for the second."""
    batch = P.Batch([(30, 1), (40, 1), (33, 33)], 16)
    gen = torch.Generator().manual_seed(4)
    pool, scales = cache_of(batch, 1, 64, gen)
    q = torch.randn(batch.tokens, 64, generator=gen).to(dtype).to(DEV)
    a = batch.arrays(DEV)
    a["kv_len"][0] = 0
    out = torch.full((batch.tokens, 64), 7.0, dtype=dtype, device=DEV)

    def go():
        K.kv8_attention(q, pool.to(DEV), scales.to(DEV), a["block_table"], a["q_start"], a["kv_len"], a["slots"], out, n_heads=1, scale=0.125, span=40,
                        tiles=a["tiles"], n_tiles=len(batch.tiles), max_q=33, decode_reqs=a["decode_reqs"], n_decode=2)

    go()
    K.check_status(DEV)
    assert (out[0] == 0).all() and not (out[1:] == 0).all(dim=1).any()
    before = out.clone()
    a["block_table"][batch.slots[1], :] = -1
    a["block_table"][batch.slots[2], 1] = batch.n_pages  # the second page of three
    go()
    with pytest.raises(K.KernelError, match="page"):
        K.check_status(DEV)
    assert (out[1] == 0).all() and out[2:18].equal(before[2:18])
    batch.table[batch.slots[2], 1] = -1
    batch.each[0] = (0, 1)
    want = P.attention(batch, q.cpu().double().unflatten(1, (1, 64)), P.values_of(pool), scales.double(), 1, 0.125)
    compare(out[18:], *(t[18:] for t in want), dtype)


def test_captured_and_longer(K):
    """A graph captured at one length serves longer ones, and its own scratch, on a stream of its own."""
    page, heads = 16, 4
    batch = P.Batch([(5000, 1), (700, 1), (3900, 6)], page)
    gen = torch.Generator().manual_seed(5)
    pool, scales = cache_of(batch, heads, 64, gen)
    pool, scales = pool.to(DEV), scales.to(DEV)
    q = torch.randn(batch.tokens, heads * 64, generator=gen).to(BF16).to(DEV)
    a = batch.arrays(DEV)
    full = a["kv_len"].clone()
    out = torch.zeros(batch.tokens, heads * 64, dtype=BF16, device=DEV)

    def go(into):
        K.kv8_attention(q, pool, scales, a["block_table"], a["q_start"], a["kv_len"], a["slots"], into, n_heads=heads, scale=0.125, span=2100,
                        tiles=a["tiles"], n_tiles=1, max_q=6, decode_reqs=a["decode_reqs"], n_decode=2)

    assert K.kv8_attention_scratch(dtype=BF16, n_heads=heads, n_kv=heads, head_dim=64, page_size=page, span=2100, n_tiles=1, max_q=6, n_decode=2) > 0
    a["kv_len"].copy_(torch.tensor([2100, 30, 600], dtype=torch.int32))
    go(out)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        go(out)
    for lens in (full, torch.tensor([2100, 30, 600], dtype=torch.int32, device=DEV), torch.tensor([1, 1, 6], dtype=torch.int32, device=DEV)):
        a["kv_len"].copy_(lens)
        graph.replay()
        torch.cuda.synchronize()
        b = P.Batch([(int(n), k) for n, (_, k) in zip(lens, batch.each)], page)
        b.table, b.slots = batch.table, batch.slots
        want = P.attention(b, q.cpu().double().unflatten(1, (heads, 64)), P.values_of(pool), scales.cpu().double(), heads, 0.125)
        compare(out, *want, BF16)
    K.check_status(DEV)


def test_the_same_bits_every_time(K):
    batch = P.Batch([(3000, 1), (2500, 4), (700, 1)], 32)
    gen = torch.Generator().manual_seed(6)
    pool, scales = cache_of(batch, 2, 128, gen)
    pool, scales = pool.to(DEV), scales.to(DEV)
    q = torch.randn(batch.tokens, 8 * 128, generator=gen).to(BF16).to(DEV)
    first = do_attention(K, batch, q, pool, scales, 8)
    for _ in range(5):
        assert do_attention(K, batch, q, pool, scales, 8).equal(first)


def test_steps_of_a_conversation(K):
    """A prompt in portions, then decoded tokens, each step written and attended over, beside the same in 64 bits."""
    heads, n_kv, dim, page = 4, 2, 64, 32
    gen = torch.Generator().manual_seed(7)
    steps = [[(37, 37), (5, 5)], [(90, 53), (6, 1)], [(91, 1), (7, 1)], [(95, 4), (40, 33)]] + [[(96 + i, 1), (41 + i, 1)] for i in range(12)]
    last = P.Batch(steps[-1], page)
    pool = torch.zeros(last.n_pages, 2, n_kv, page, dim, dtype=torch.float8_e4m3fn, device=DEV)
    scales = torch.zeros(last.n_pages, 2, n_kv, page // 16, device=DEV)
    want, s = P.values_of(pool), scales.cpu().double()
    for each in steps:
        batch = P.Batch(each, page)
        batch.table, batch.slots, batch.n_pages = last.table, last.slots, last.n_pages
        rows = (torch.randn(batch.tokens, (heads + 2 * n_kv) * dim, generator=gen) * 2).to(BF16)
        q, k, v = rows.split([heads * dim, n_kv * dim, n_kv * dim], dim=1)
        P.write(batch, k.double().unflatten(1, (n_kv, dim)), v.double().unflatten(1, (n_kv, dim)), want, s)
        dev = rows.to(DEV)
        dq, dk, dv = dev.split([heads * dim, n_kv * dim, n_kv * dim], dim=1)
        do_write(K, batch, dk, dv, pool, scales)
        got = do_attention(K, batch, dq, pool, scales, heads)
        torch.testing.assert_close(P.values_of(pool), want, rtol=0, atol=0)
        compare(got, *P.attention(batch, q.double().unflatten(1, (heads, dim)), want, s, heads, dim ** -0.5), BF16)
    K.check_status(DEV)


# ---- copies of pages ---------------------------------------------------------------------------

@pytest.mark.parametrize("pages,pairs", [(2, [(1, 0)]), (40, [(3, 9), (3, 10), (0, 39), (20, 21)]), (600, [(i, 599 - i) for i in range(300)])])
def test_copies(K, pages, pairs):
    gen = torch.Generator().manual_seed(pages)
    shapes = [((pages, 2, 3, 16, 64), torch.uint8), ((pages, 2, 3, 1), F32), ((pages, 2, 3, 32, 32), BF16), ((pages, 5), F32), ((pages, 7, 8), F32)] * 25
    host = [torch.randint(0, 100, s, generator=gen).to(t) for s, t in shapes]
    dev = [t.to(DEV) for t in host]
    handle = K.PagePools(dev)
    K.copy_pages(handle, torch.tensor(pairs, dtype=torch.int32, device=DEV))
    K.check_status(DEV)
    src, dst = torch.tensor(pairs).unbind(1)
    for h, d in zip(host, dev):
        h[dst] = h[src]
        assert torch.equal(d.cpu(), h)


def test_copies_of_pages_that_are_not_there(K):
    pool = torch.arange(64, dtype=F32, device=DEV).reshape(4, 16)
    before = pool.clone()
    K.copy_pages(K.PagePools([pool]), torch.tensor([[0, 4], [-1, 1], [5, 2], [1, 3]], dtype=torch.int32, device=DEV))
    with pytest.raises(K.KernelError, match="page"):
        K.check_status(DEV)
    before[3] = before[1]
    assert pool.equal(before)


# ---- refusals ----------------------------------------------------------------------------------

def test_refusals(K):
    batch = P.Batch([(20, 1), (20, 3)], 16)
    a = batch.arrays(DEV)
    gen = torch.Generator().manual_seed(1)
    pool, scales = (t.to(DEV) for t in cache_of(batch, 2, 64, gen))
    q = torch.zeros(batch.tokens, 256, dtype=BF16, device=DEV)
    k = torch.zeros(batch.tokens, 128, dtype=BF16, device=DEV)

    def write(**change):
        x = dict(k=k, v=k, pool=pool, scales=scales, block_table=a["block_table"], positions=a["positions"], req_of_token=a["req_of_token"],
                 q_start=a["q_start"], slots=a["slots"], max_pos=32)
        K.kv8_write(**(x | change))

    def attend(**change):
        x = dict(q=q, pool=pool, scales=scales, block_table=a["block_table"], q_start=a["q_start"], kv_len=a["kv_len"], slots=a["slots"],
                 out=torch.empty_like(q), n_heads=4, scale=0.1, span=20, tiles=a["tiles"], n_tiles=1, max_q=3, decode_reqs=a["decode_reqs"], n_decode=1)
        K.kv8_attention(**(x | change))

    write()
    attend()
    for change, why in [(dict(pool=pool.view(torch.uint8)), "float8"), (dict(pool=pool[:, :, :, :8]), "contiguous"), (dict(scales=scales[:1]), "scales"),
                        (dict(k=k.cpu()), "CUDA"), (dict(k=k.half(), v=k.half()), "element type"), (dict(v=k.float()), "bfloat16"), (dict(k=k[:, :64]), "rows"),
                        (dict(k=torch.zeros(batch.tokens, 130, dtype=BF16, device=DEV)[:, 2:]), "16 bytes"),
                        (dict(k=torch.zeros(batch.tokens, 129, dtype=BF16, device=DEV)[:, :128]), "16 bytes"), (dict(k=k[:1]), "rows"),
                        (dict(positions=a["positions"].long()), "int32"), (dict(req_of_token=a["req_of_token"][:1]), "as long")]:
        with pytest.raises(K.KernelError, match=why):
            write(**change)
    with pytest.raises(K.KernelError, match="multiple of 16"):
        write(pool=torch.zeros(4, 2, 2, 24, 64, dtype=torch.float8_e4m3fn, device=DEV))
    with pytest.raises(K.KernelError, match="one of 32"):
        write(pool=torch.zeros(4, 2, 2, 16, 80, dtype=torch.float8_e4m3fn, device=DEV))
    for change, why in [(dict(n_heads=3), "multiple of 2"), (dict(n_heads=8), "rows of heads"), (dict(out=torch.empty_like(q)[:2]), "fewer rows"),
                        (dict(q=q.float()), "bfloat16|float32"), (dict(tiles=None), "without tiles"), (dict(n_decode=2), "shorter"), (dict(n_tiles=2), "shorter"),
                        (dict(window=0), "window"), (dict(kv_len=a["kv_len"].long()), "int32"),
                        (dict(span=100000, scratch=torch.empty(8, device=DEV)), "scratch")]:
        with pytest.raises(K.KernelError, match=why):
            attend(**change)
    with pytest.raises(K.KernelError, match="recorded"):
        with K.recording():
            attend(span=100000)
    K.copy_pages(K.PagePools([pool, scales]), torch.zeros(0, 2, dtype=torch.int32, device=DEV))
    for pools, why in [([], "no pool"), ([pool, scales[:1]], "numbers of pages"), ([pool.cpu()], "CUDA"), ([torch.zeros(3, 5, dtype=BF16, device=DEV)], "4 bytes")]:
        with pytest.raises(K.KernelError, match=why):
            K.PagePools(pools)
    with pytest.raises(K.KernelError, match=r"\[n, 2\]"):
        K.copy_pages(K.PagePools([pool]), torch.zeros(3, dtype=torch.int32, device=DEV))
    K.check_status(DEV)


# ---- calls beside one another, pages of other sizes ------------------------------------------------

@pytest.mark.parametrize("page", [1024, 4096, 8192])
def test_large_pages(K, page):
    """Few large pages, of more tokens than the tcgen05 kernel's division takes as well; decoded tokens beside portions of 64 rows and more."""
    check_attention(K, [(700, 64), (1030, 1), (600, 20), (5, 1)], 4, 1, 64, page, BF16)


def test_two_streams(K):
    """Two calls that may run at the same time, each with scratch of its own and none, on streams that are not the default one."""
    gen = torch.Generator().manual_seed(9)
    jobs = []
    for each in ([(3000, 1)] * 3, [(2500, 40), (900, 64)]):
        batch = P.Batch(each, 16, seed=len(each))
        pool, scales = cache_of(batch, 2, 128, gen)
        q = torch.randn(batch.tokens, 1024, generator=gen).to(BF16)
        want = P.attention(batch, q.double().unflatten(1, (8, 128)), P.values_of(pool), scales.double(), 8, 128 ** -0.5)
        jobs.append((batch, pool.to(DEV), scales.to(DEV), q.to(DEV), want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for turn in range(4):
        for batch, pool, scales, q, want, stream in jobs:
            with torch.cuda.stream(stream):
                outs.append((do_attention(K, batch, q, pool, scales, 8), want))
    torch.cuda.synchronize()
    for out, (o, rough, fine) in outs:
        compare(out, o, rough, fine, BF16)
    K.check_status(DEV)
