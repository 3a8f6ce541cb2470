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
