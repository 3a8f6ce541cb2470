"""The operators of the 8-bit cache at the ends of their ranges, against their definition in 64 bits."""
import pytest
import torch

import plain_kv8 as P
import test_kv8_gpu as T

pytestmark = pytest.mark.gpu
DEV = T.DEV
F32, BF16 = T.F32, T.BF16
K = T.K  # the fixture


def test_batches_without_a_request_or_a_page_are_refused(K):
    pool = torch.zeros(3, 2, 1, 16, 64, dtype=torch.float8_e4m3fn, device=DEV)
    scales = torch.zeros(3, 2, 1, 1, device=DEV)
    q = torch.zeros(64, 64, dtype=BF16, device=DEV)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731

    def attend(**change):
        x = dict(q=q, pool=pool, scales=scales, block_table=ints(0, 1, 2).reshape(1, 3), q_start=ints(0, 64), kv_len=ints(48), slots=ints(0),
                 out=torch.empty_like(q), n_heads=1, scale=0.125, span=600, tiles=ints(0, 0).reshape(1, 2), n_tiles=1, decode_reqs=ints(0), n_decode=0)
        K.kv8_attention(**(x | change))

    for change, why in [(dict(pool=pool[:0], scales=scales[:0]), "no page"), (dict(q_start=ints(), kv_len=ints(), slots=ints()), "q_start"),
                        (dict(q_start=ints(0)), "without requests"), (dict(q_start=ints(0), n_tiles=0, n_decode=1), "without requests")]:
        with pytest.raises(K.KernelError, match=why):
            attend(**change)
    attend(q_start=ints(0), n_tiles=0)  # nothing to do is no fault
    K.check_status(DEV)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_largest_finite_values_are_values(K, dtype):
    """Entries from 3.4e38 to the largest finite one of the type are stored and count for the scale, also beside infinities; rows that are continued too."""
    most = torch.finfo(dtype).max
    batch = P.Batch([(40, 40), (25, 5), (20, 4)], 16)
    gen = torch.Generator().manual_seed(11)
    pool, scales = T.cache_of(batch, 1, 64, gen)
    k, v = (torch.randn(batch.tokens, 64, generator=gen).to(dtype) for _ in range(2))
    k[0, 0], k[3, 9], k[20, 63] = most, -most, most
    k[16:32, 5] = torch.tensor(3.401e38, dtype=torch.float64).to(dtype) if dtype == F32 else most
    v[33, 1], v[34, 2], v[35, 3] = most, float("inf"), float("nan")  # the largest beside what is none
    k[41, 7], v[46, 8] = -most, most  # in blocks that hold earlier tokens
    dp, _ = T.check_write(K, batch, 1, 64, dtype, k, v, pool, scales)
    assert int(torch.isnan(dp.float()).sum()) == 2


def on_tcgen05(K, each, heads, n_kv, dim, page, window=None):
    """Whether the portions of such a batch run on the tcgen05 kernel."""
    plan = K.kv8_attention_plan(dtype=BF16, n_heads=heads, n_kv=n_kv, head_dim=dim, page_size=page, span=max(n for n, _ in each), window=window,
                                n_tiles=sum(-(-k // 64) for _, k in each if k > 1), max_q=max(k for _, k in each))[0]
    return plan is not None and plan[0] == 128


@pytest.mark.parametrize("dtype,each", [(F32, [(200, 1), (150, 40)]), (BF16, [(200, 1), (150, 20)]), (BF16, [(600, 70), (40, 1)])])
def test_queries_of_the_largest_size(K, dtype, each):
    """Queries up to the largest finite value over keys of the smallest scale: their scores are ordinary numbers."""
    def touch(batch, q, pool, scales):
        top = q.float().abs().unflatten(1, (2, 64)).amax(dim=2, keepdim=True)
        q.copy_((q.float().unflatten(1, (2, 64)) / top * torch.finfo(dtype).max).flatten(1).to(dtype))
        assert torch.isfinite(q).all() and (q.abs() > 2.0 ** 127).any(dim=1).all()
        scales[:, 0] = 2.0 ** -126

    T.check_attention(K, each, 2, 2, 64, 16, dtype, touch=touch)
    assert on_tcgen05(K, each, 2, 2, 64, 16) == (each[0][1] == 70)


@pytest.mark.parametrize("scale", [-0.125, -1.0, 0.0])
@pytest.mark.parametrize("dtype,each,dim", [(F32, [(200, 1), (150, 40)], 64), (BF16, [(2300, 1), (150, 20)], 96), (BF16, [(600, 70), (40, 1)], 64), (BF16, [(600, 130)], 128)])
def test_scales_that_are_not_positive(K, dtype, each, dim, scale):
    """The smallest product is the largest score then; with none, all keys in sight weigh the same."""
    gen = torch.Generator().manual_seed(13)
    batch = P.Batch(each, 16, seed=13)
    pool, scales = T.cache_of(batch, 2, dim, gen)
    q = (torch.randn(batch.tokens, 2 * dim, generator=gen) * 1.5).to(dtype)
    want = list(P.attention(batch, q.double().unflatten(1, (2, dim)), P.values_of(pool), scales.double(), 2, scale))
    if scale < 0:  # the bounds for a scale of that size
        want[1:] = P.attention(batch, -q.double().unflatten(1, (2, dim)), P.values_of(pool), scales.double(), 2, -scale)[1:]
    a = batch.arrays(DEV)
    out = torch.full((batch.tokens, 2 * dim), 7.0, dtype=dtype, device=DEV)
    K.kv8_attention(q.to(DEV), pool.to(DEV), scales.to(DEV), a["block_table"], a["q_start"], a["kv_len"], a["slots"], out, n_heads=2, scale=scale,
                    span=max(n for n, _ in each), tiles=a["tiles"], n_tiles=len(batch.tiles), max_q=max(n for _, n in each), decode_reqs=a["decode_reqs"],
                    n_decode=len(batch.single))
    K.check_status(DEV)
    T.compare(out, *want, dtype)


# ---- values of very different sizes ----------------------------------------------------------------

def blocks_of(batch, r):
    """(block of 16 keys, page, block of the page) of a request."""
    for b in range(-(-batch.each[r][0] // 16)):
        page, row = batch.row_of(r, b * 16)
        yield b, page, row // 16


def apart(shift, down, every=3):
    """Keys of every third block score ``shift`` (nats) lower than the others, and values of the other blocks are 2^-down of theirs."""
    def touch(batch, q, pool, scales):
        dim, n_kv = pool.shape[4], pool.shape[2]
        heads = q.shape[1] // dim
        q.view(batch.tokens, heads, dim)[:, :, 0] = 8.0
        low = torch.tensor(-shift * dim ** 0.5 / 8.0 / 0.25).to(torch.float8_e4m3fn).view(torch.uint8)
        codes = pool.view(torch.uint8)
        for r in range(len(batch.each)):
            for b, page, sub in blocks_of(batch, r):
                rows = slice(16 * sub, 16 * sub + 16)
                if b % every == 0:
                    codes[page, 0, :, rows] = 0
                    codes[page, 0, :, rows, 0] = low
                    scales[page, 0, :, sub] = 0.25
                else:
                    codes[page, 0, :, rows, 0] = 0
                    scales[page, 1, :, sub] *= 2.0 ** -down

    return touch


# a unit a block, shares that are joined, few queries, many, in 32 bits; tcgen05 with heads of 64 and 128 and in shares
SHAPES = [([(700, 1), (90, 1)], 2, 2, 64, 16, BF16), ([(3000, 1), (40, 1)], 4, 1, 64, 32, BF16), ([(300, 5), (33, 1)], 4, 1, 128, 16, BF16),
          ([(300, 100)], 1, 1, 96, 16, BF16), ([(700, 1), (200, 60)], 2, 2, 64, 16, F32), ([(2500, 4)], 2, 1, 256, 64, F32),
          ([(700, 130), (20, 1)], 2, 2, 64, 16, BF16), ([(900, 70)], 4, 2, 128, 64, BF16)]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("shift,down", [(40, 12), (40, 20), (40, 24), (40, 32), (60, 60), (26, 50), (26, 90), (0, 40)])
def test_values_of_very_different_sizes(K, shape, shift, down):
    """What a row weighs most may lie in blocks whose values are the smallest in its sight, or the product of a tiny probability and a huge value: every
    entry is within the bound of its own sum of probabilities times values."""
    each, heads, n_kv, dim, page, dtype = SHAPES[shape]
    assert on_tcgen05(K, each, heads, n_kv, dim, page) == (shape >= 6)
    T.check_attention(K, each, heads, n_kv, dim, page, dtype, spread=0.0, touch=apart(shift, down))


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_values_of_nothing_beside_others(K, shape):
    """Blocks whose values are all zero (their scale is the smallest) beside ordinary ones."""
    def touch(batch, q, pool, scales):
        for r in range(len(batch.each)):
            for b, page, sub in blocks_of(batch, r):
                if b % 2 == 0:
                    rows = slice(16 * sub, 16 * sub + 16)
                    codes = pool.view(torch.uint8)
                    codes[page, 1, :, rows] = torch.where(codes[page, 1, :, rows] == 0x7F, codes[page, 1, :, rows], 0)  # (NaN behind the last token stays)
                    scales[page, 1, :, sub] = 2.0 ** -126

    each, heads, n_kv, dim, page, dtype = SHAPES[shape]
    T.check_attention(K, each, heads, n_kv, dim, page, dtype, touch=touch)


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_values_of_the_largest_size(K, shape):
    """Means of values near the largest finite one are finite."""
    def touch(batch, q, pool, scales):
        scales[:, 1] = 2.0 ** 119  # codes of up to 448

    each, heads, n_kv, dim, page, dtype = SHAPES[shape]
    got = T.check_attention(K, each, heads, n_kv, dim, page, dtype, touch=touch)
    assert torch.isfinite(got).all() and got.abs().max() > 1e37


@pytest.mark.parametrize("up", [20, 31, 60, 125])
@pytest.mark.parametrize("each,heads,n_kv,dim,dtype", [([(160, 100)], 2, 2, 64, BF16), ([(160, 100)], 3, 1, 32, BF16), ([(96, 40)], 2, 1, 64, F32), ([(640, 200)], 2, 1, 64, BF16),
                                                       ([(1024, 150)], 2, 2, 128, BF16)])
def test_a_value_that_a_row_does_not_see_changes_nothing_for_it(K, each, heads, n_kv, dim, dtype, up):
    """The values of one block, that some rows see and others do not, become 2^up times as large: the rows ahead of it keep every bit, the others are right."""
    n, nq = each[0]
    block = (n - nq // 3) // 16
    outs = []
    for by in (0, up):
        def touch(batch, q, pool, scales):
            page, row = batch.row_of(0, 16 * block)
            scales[page, 1, :, row // 16] = 2.0 ** (by - 6)

        outs.append(T.check_attention(K, each, heads, n_kv, dim, 16, dtype, touch=touch))
    ahead = 16 * block - (n - nq)
    assert 0 < ahead < nq and outs[0][:ahead].equal(outs[1][:ahead]) and not outs[0][ahead:].equal(outs[1][ahead:])


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_a_query_that_is_not_finite_is_its_own_row_s_matter(K, shape):
    """A NaN in one token's one head: that row is NaN, all the others are what they were, bit by bit."""
    each, heads, n_kv, dim, page, dtype = SHAPES[shape]
    batch = P.Batch(each, page, seed=9)
    gen = torch.Generator().manual_seed(9)
    pool, scales = (t.to(DEV) for t in T.cache_of(batch, n_kv, dim, gen))
    q = torch.randn(batch.tokens, heads, dim, generator=gen).to(dtype).to(DEV)
    want = T.do_attention(K, batch, q.flatten(1), pool, scales, heads).view_as(q)
    for token, head in ((0, heads - 1), (batch.tokens // 2, 0)):
        spoilt = q.clone()
        spoilt[token, head, dim // 3] = float("nan")
        got = T.do_attention(K, batch, spoilt.flatten(1), pool, scales, heads).view_as(q)
        assert torch.isnan(got[token, head]).all()
        got[token, head] = want[token, head]
        assert got.equal(want)
    K.check_status(DEV)


# ---- the tcgen05 kernel: portions of 64 rows and more over contexts of 512 and more ----------------

WIDE = [(700, 64), (1300, 130), (520, 520), (90, 70), (640, 1), (515, 2), (64, 64), (777, 191)]


def check_wide(K, each, heads, n_kv, dim, page, **kw):
    assert on_tcgen05(K, each, heads, n_kv, dim, page, kw.get("window"))
    return T.check_attention(K, each, heads, n_kv, dim, page, BF16, **kw)


@pytest.mark.parametrize("heads,n_kv,dim,page", [(1, 1, 64, 16), (3, 1, 64, 48), (5, 1, 128, 80), (4, 2, 128, 32), (2, 2, 64, 112), (12, 1, 64, 64), (1, 1, 128, 4096)])
def test_wide_portions(K, heads, n_kv, dim, page):
    """Groups of heads that straddle a block of rows, pages whose number of blocks is no power of two, portions that end anywhere."""
    check_wide(K, WIDE, heads, n_kv, dim, page)


@pytest.mark.parametrize("heads,n_kv,dim,page", [(2, 1, 64, 16), (2, 2, 128, 48)])
@pytest.mark.parametrize("window", [448, 449, 511, 512, 700, 1100, 5000])
def test_wide_portions_with_windows(K, heads, n_kv, dim, page, window):
    check_wide(K, WIDE, heads, n_kv, dim, page, window=window)


@pytest.mark.parametrize("spread", [0.0, 2.0, 4.0])
def test_wide_portions_of_spread_values(K, spread):
    check_wide(K, WIDE, 3, 1, 64, 16, spread=spread)


@pytest.mark.parametrize("dim,n,nq,at", [(64, 700, 150, 640), (64, 700, 150, 100), (128, 600, 80, 599), (64, 1024, 512, 512), (128, 900, 130, 895)])
@pytest.mark.parametrize("window", [None, 500])
def test_wide_portions_and_nan(K, dim, n, nq, at, window):
    """A value that is NaN reaches its dim of the rows that see the token, whatever the token weighs; a key that is NaN all of those rows of its head."""
    heads = 2
    sees = torch.tensor([at <= p and (window is None or at > p - window) for p in range(n - nq, n)])

    def value(batch, q, pool, scales):
        page, row = batch.row_of(0, at)
        pool.view(torch.uint8)[page, 1, 0, row, [5, dim - 1]] = 0x7F

    got = check_wide(K, [(n, nq)], heads, 2, dim, 16, window=window, touch=value).cpu()
    assert torch.isnan(got[:, 5]).equal(sees) and torch.isnan(got[:, dim - 1]).equal(sees) and int(torch.isnan(got).sum()) == 2 * int(sees.sum())
    gen = torch.Generator().manual_seed(2)
    batch = P.Batch([(n, nq)], 16, seed=2)
    pool, scales = T.cache_of(batch, 2, dim, gen)
    page, row = batch.row_of(0, at)
    pool.view(torch.uint8)[page, 0, 1, row, 7] = 0x7F
    q = torch.randn(batch.tokens, heads * dim, generator=gen).to(BF16).to(DEV)
    got = T.do_attention(K, batch, q, pool.to(DEV), scales.to(DEV), heads, window=window).cpu()
    assert torch.isnan(got[:, dim:]).all(dim=1).equal(sees) and torch.isnan(got[:, dim:]).any(dim=1).equal(sees) and not torch.isnan(got[:, :dim]).any()


@pytest.mark.parametrize("dim,page", [(64, 16), (64, 48), (128, 64)])
def test_wide_portions_without_some_pages(K, dim, page):
    """Pages that are not there, first, in the middle of a tile and last, and a request without any: their keys are nobody's, and the status word says so."""
    each = [(700, 130), (600, 64), (560, 70), (0, 66)]
    batch = P.Batch([(max(n, 66), q) for n, q in each], page, seed=4)
    batch.each = each
    gen = torch.Generator().manual_seed(4)
    pool, scales = T.cache_of(batch, 1, dim, gen)
    q = torch.randn(batch.tokens, 2 * dim, generator=gen).to(BF16)
    assert on_tcgen05(K, each, 2, 1, dim, page)
    T.compare(T.do_attention(K, batch, q.to(DEV), pool.to(DEV), scales.to(DEV), 2), *P.attention(batch, q.double().unflatten(1, (2, dim)), P.values_of(pool),
                                                                                             scales.double(), 2, dim ** -0.5), BF16)
    K.check_status(DEV)
    table = batch.table.clone()
    table[batch.slots[0], 0], table[batch.slots[0], 300 // page], table[batch.slots[0], 699 // page] = -1, batch.n_pages, -7
    table[batch.slots[2], :] = -1
    batch.table = table
    out = T.do_attention(K, batch, q.to(DEV), pool.to(DEV), scales.to(DEV), 2)
    with pytest.raises(K.KernelError, match="page"):
        K.check_status(DEV)
    batch.table = torch.where(table >= batch.n_pages, -1, table)
    want = P.attention(batch, q.double().unflatten(1, (2, dim)), P.values_of(pool), scales.double(), 2, dim ** -0.5)
    T.compare(out, *want, BF16)
    assert (out[batch.q_start[2]:] == 0).all()


def test_wide_portions_give_the_same_bits_every_time(K):
    batch = P.Batch([(1500, 200), (900, 70), (600, 64), (33, 1)], 32)
    gen = torch.Generator().manual_seed(6)
    pool, scales = (t.to(DEV) for t in T.cache_of(batch, 2, 128, gen))
    q = torch.randn(batch.tokens, 8 * 128, generator=gen).to(BF16).to(DEV)
    assert on_tcgen05(K, batch.each, 8, 2, 128, 32)
    first = T.do_attention(K, batch, q, pool, scales, 8)
    for _ in range(5):
        assert T.do_attention(K, batch, q, pool, scales, 8).equal(first)


@pytest.mark.parametrize("dim", [64, 128])
def test_wide_portions_captured(K, dim):
    """A graph of the tcgen05 kernel and its join, captured at one length, serves longer and shorter contexts."""
    batch = P.Batch([(2600, 100), (1800, 64)], 16)
    gen = torch.Generator().manual_seed(5)
    pool, scales = (t.to(DEV) for t in T.cache_of(batch, 2, dim, gen))
    q = torch.randn(batch.tokens, 4 * dim, generator=gen).to(BF16).to(DEV)
    a = batch.arrays(DEV)
    out = torch.zeros(batch.tokens, 4 * dim, dtype=BF16, device=DEV)
    sizes = dict(n_heads=4, span=600, n_tiles=3, max_q=100)
    floats = K.kv8_attention_scratch(dtype=BF16, n_kv=2, head_dim=dim, page_size=16, **sizes)
    assert floats > 0 and on_tcgen05(K, [(600, 100)], 4, 2, dim, 16)
    scratch = torch.full((floats,), float("nan"), device=DEV)

    def go():
        K.kv8_attention(q, pool, scales, a["block_table"], a["q_start"], a["kv_len"], a["slots"], out, scale=dim ** -0.5, tiles=a["tiles"], scratch=scratch, **sizes)

    go()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        go()
    for lens in ([2600, 1800], [600, 500], [100, 64], [2601 - 16, 700]):
        a["kv_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        b = P.Batch(list(zip(lens, (100, 64))), 16)
        b.table, b.slots = batch.table, batch.slots
        T.compare(out, *P.attention(b, q.cpu().double().unflatten(1, (4, dim)), P.values_of(pool), scales.cpu().double(), 4, dim ** -0.5), BF16)
    K.check_status(DEV)


@pytest.mark.parametrize("heads,n_kv,dim", [(1, 1, 64), (2, 2, 128), (2, 1, 64)])
@pytest.mark.parametrize("tiles", [[(0, 0)], [(0, 64)], [(0, 64), (0, 0)], [(0, 128), (1, 0)], [(0, 64), (0, 128), (1, 64)], [(1, 0), (0, 0), (0, 128), (0, 64)], [(0, 0), (1, 64)]])
def test_wide_portions_of_some_tiles(K, heads, n_kv, dim, tiles):
    """A list that names some of a request's tiles, in any order: the rows of those are written, the others stay (two neighbours may share a block of rows)."""
    each = [(700, 200), (600, 128)]
    batch = P.Batch(each, 16, seed=8)
    gen = torch.Generator().manual_seed(8)
    pool, scales = T.cache_of(batch, n_kv, dim, gen)
    q = torch.randn(batch.tokens, heads * dim, generator=gen).to(BF16)
    assert on_tcgen05(K, each, heads, n_kv, dim, 16)
    want = P.attention(batch, q.double().unflatten(1, (heads, dim)), P.values_of(pool), scales.double(), heads, dim ** -0.5)
    batch.tiles = tiles
    out = T.do_attention(K, batch, q.to(DEV), pool.to(DEV), scales.to(DEV), heads)
    K.check_status(DEV)
    named = torch.zeros(batch.tokens, dtype=torch.bool)
    for r, t in tiles:
        named[batch.q_start[r] + t:batch.q_start[r] + min(t + 64, each[r][1])] = True
    assert (out[~named.to(DEV)] == 7).all()
    T.compare(out[named.to(DEV)], *(x[named] for x in want), BF16)


# ---- through the engine, at contexts where all of these kernels run ---------------------------------

def formulas(cfg, t, r, slot, ids, first, rounding=lambda x: x):
    """Logits of ``ids[first:]`` in 64 bits with the keys and values that the cache holds; ``rounding``: of what a 16-bit engine stores between products."""
    import test_kv8_engine_gpu as E

    G, D, H, eps = E.P, cfg["n_embd"], cfg["n_head"], cfg.get("layer_norm_epsilon", 1e-5)
    n, act = len(ids), E.P.activation_of(cfg.get("activation_function", "gelu_new"))
    x = t["wte.weight"][torch.tensor(ids[first:])] + t["wpe.weight"][first:n]
    for i in range(cfg["n_layer"]):
        p = f"h.{i}."
        h = rounding(G.layer_norm(x, t[p + "ln_1.weight"], t[p + "ln_1.bias"], eps))
        q = rounding(h @ t[p + "attn.c_attn.weight"] + t[p + "attn.c_attn.bias"])[:, :D].view(-1, H, D // H)
        kv, _ = E.cached(r, i, slot, n)
        s = torch.einsum("qhd,khd->hqk", q, kv[:, 0]) * (D // H) ** -0.5
        s = s.masked_fill(torch.arange(n)[None] > torch.arange(first, n)[:, None], float("-inf"))
        o = rounding(torch.einsum("hqk,khd->qhd", torch.softmax(s, dim=-1), kv[:, 1]).reshape(-1, D))
        x = rounding(x + o @ t[p + "attn.c_proj.weight"] + t[p + "attn.c_proj.bias"])
        h = rounding(G.layer_norm(x, t[p + "ln_2.weight"], t[p + "ln_2.bias"], eps))
        x = rounding(x + rounding(act(h @ t[p + "mlp.c_fc.weight"] + t[p + "mlp.c_fc.bias"])) @ t[p + "mlp.c_proj.weight"] + t[p + "mlp.c_proj.bias"])
    return rounding(G.layer_norm(x, t["ln_f.weight"], t["ln_f.bias"], eps)) @ t["wte.weight"].t()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("graphs", [False, True])
def test_long_contexts_through_the_engine(K, tmp_path, dtype, graphs):
    """Prompts in portions on tcgen05, decoded tokens beside them and alone over contexts whose keys are shared out and joined, steps issued again from
    launch lists with their scratch, graphs, and a fork.  Tolerances are those of the engine's other tests: 1e-4 of the logits' size in 32 bits, and in
    16 bits three times what rounding the formulas' activations to bfloat16 does to these very logits."""
    import test_kv8_engine_gpu as E
    from rosellm_b200.config import GPT2Config
    from rosellm_b200.weights import write_model_folder

    folder = str(tmp_path / "long")
    write_model_folder(GPT2Config(n_layer=2, n_embd=128, n_head=2, n_inner=256, vocab_size=500, n_positions=4608, layer_norm_epsilon=1e-5,
                                  activation_function="gelu_new"), 7, folder, std=0.1, norm_affine="random")
    cfg, t = E.P.load_folder(folder)
    half = dtype == "bfloat16"
    if half:
        t = {k: (v.to(BF16).double() if v.dim() > 1 else v) for k, v in t.items()}
    r = E.runner(folder, dtype, cuda_graphs=graphs, kv_cache_max_tokens=16384, max_batch_size=4, max_num_batched_tokens=2048)
    rng = torch.Generator().manual_seed(3)
    ids = [torch.randint(0, 500, (n,), generator=rng).tolist() for n in (2400, 2400, 700)]
    assert K.kv8_on_tcgen05(K.BF16, 64, 64, 16, 1024)
    assert K.kv8_attention_scratch(dtype=BF16 if half else F32, n_heads=2, n_kv=2, head_dim=64, page_size=16, span=2300, n_decode=1) > 0

    def step(slots, at, counts, who=(0, 1, 2)):
        """One step, each of whose last rows is compared with the formulas."""
        entries = [E.entry(slots[i], ids[i][at[i]:at[i] + n], list(range(max(0, n - 80), n))) for i, n in zip(who, counts) if n]
        logits = r.step(entries).clone()
        row = 0
        for i, n in zip(who, counts):
            if n:
                keep = min(n, 80)
                at[i] += n
                x = formulas(cfg, t, r, slots[i], ids[i][:at[i]], at[i] - keep)
                limit = 1e-4 * max(1.0, float(x.abs().max()))
                if half:
                    limit = 3 * float((formulas(cfg, t, r, slots[i], ids[i][:at[i]], at[i] - keep, E.P.to_bfloat16_and_back) - x).abs().max())
                off = float((logits[row:row + keep].cpu().double() - x).abs().max())
                assert off <= limit, (i, n, at[i], off, limit)
                row += keep
        return logits

    slots, at = [r.cache.new_request() for _ in ids], [0, 0, 0]
    step(slots, at, (1024, 0, 0))
    first = step(slots, at, (1024, 0, 0))
    step(slots, at, (252, 0, 0))
    step(slots, at, (1, 0, 600))
    step(slots, at, (1, 0, 1))
    ids[1][:2048] = ids[0][:2048]
    before = r.launch_list_replays
    step(slots, at, (0, 1024, 0))
    again = step(slots, at, (0, 1024, 0))
    # the same launches over other pages (a list that was noted before a buffer of the workspace grew is noted again)
    assert r.launch_list_replays > before and again.equal(first)
    step(slots, at, (1, 200, 1))
    for _ in range(3):
        step(slots, at, (1, 1, 1))
    f = r.fork(slots[0])
    slots.append(f)
    ids.append(ids[0][:at[0]] + ids[2][:20])
    at.append(at[0])
    step(slots, at, (1, 2, 1), who=(0, 1, 3))
    step(slots, at, (1, 1, 1, 1), who=(0, 1, 2, 3))
    r.check_status()
    for s in slots:
        r.cache.release(s)
    r.cache.check()
