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
