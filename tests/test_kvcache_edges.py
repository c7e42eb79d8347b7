"""More of the KV-cache operators at their edges: batches padded on the left, and what the other tests
of test_kvcache.py, whose helpers and tolerances these use, do not reach."""

import numpy as np
import pytest
import torch

import flash_lab
from flash_lab import ops
from test_kvcache import Cache, check_extend, check_rows

BOTH = pytest.mark.parametrize("int8", [False, True], ids=["16bit", "int8"])
DIMS = pytest.mark.parametrize("d", [64, 128])


# ------------------------------------------------------------------------------------------------
# More rows than keys
# ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@BOTH
@DIMS
@pytest.mark.parametrize("lens", [(20, 20, 20, 64), (64, 1, 32), (33, 0, 20, 31, 200), (20, 32, 65)],
                         ids=lambda x: "-".join(map(str, x)))
def test_extend_left_padded_batches(lens, d, int8):
    # 64 rows per sequence, two tiles of 32 tokens: the first tile of up to 32 keys sees none. About
    # 768 items, five and more per CTA, short ones in runs before and after full ones.
    lens = [lens[b % len(lens)] for b in range(96)]
    check_extend(Cache(lens, 8, d, torch.bfloat16, int8, page=16), [64] * 96, 32, torch.bfloat16)


@pytest.mark.gpu
@BOTH
@DIMS
def test_extend_left_padded_batches_of_long_rows(d, int8):
    # One query head per KV head, tiles of 128 tokens: n - L from less than a tile to two tiles and more.
    rng = np.random.RandomState(7)
    lens = [int(x) for x in rng.choice([3, 100, 128, 129, 140, 255, 256, 300, 700], 60)]
    new = [int(x) for x in rng.choice([256, 250, 129, 300], 60)]
    check_extend(Cache(lens, 16, d, torch.float16, int8), new, 16, torch.float16)


@pytest.mark.gpu
@BOTH
@DIMS
def test_extend_left_padded_uniform_rows(d, int8):
    # The same as [B, n, H, D], where n is known on the host.
    lens = [(20, 20, 20, 64)[b % 4] for b in range(96)]
    cache = Cache(lens, 8, d, torch.float16, int8)
    q = torch.randn(96, 64, 32, d, device="cuda").half()
    for _ in range(3):
        out, lse = flash_lab.extend(q, cache.k, cache.v, cache.seq_lens, return_lse=True,
                                    **cache.kwargs())
        torch.cuda.synchronize()
        assert ops.device_status(0) == 0
        for b in range(96):
            k, v = cache.keys(b)
            check_rows(out[b], lse[b], q[b], k, v, True, d ** -0.5, int8)
