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
