"""More of the operators that check drafted tokens, on the GPU: what the sizes of test_gpu_drafts.py do not
reach, against the same 64-bit definitions and with the same tolerances."""
import numpy as np
import pytest
import torch

import leaf_b200 as lq
from test_gpu_drafts import _plan
from test_gpu_kv8 import _i32, _status_ok

pytestmark = pytest.mark.gpu
LEAST = 2.0 ** -149  # of the 32-bit numbers above zero


# ----------------------------------------------------------------- compact
def _two_pages(codes, scales, kept, path, context=14):
    cache = lq.Kv8Cache(*(torch.from_numpy(codes.copy()).cuda() for _ in range(2)), *(torch.from_numpy(scales.copy()).cuda() for _ in range(2)))
    lq.kv8_compact(lq.Kv8Layers([cache]), _plan([context], [[-1] * 9], table=[[0, 1]], page=16), _i32([path]), _i32([kept]))
    torch.cuda.synchronize()
    return cache


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_compact_codes_stay_within_eight_bits(cuda_device, dim):
    # Scales of a few times the least 32-bit number: what the rows need, 180 / 127 and 300 / 127 of it, is rounded to one
    # and two of it, and codes of up to 180 and 150 times that would be needed: they stop at the ends, with their signs.
    rng = np.random.default_rng(dim)
    for old, new, scale in ((0, 3, 1), (1, 3, 1), (2, 5, 2)):
        codes = rng.integers(-60, 61, (2, 1, 16, dim)).astype(np.int8)
        codes[1, 0, 2, :2] = (60, -60)  # the row that moves: token 4 behind a context of 14
        cache = _two_pages(codes, np.array([[old * LEAST], [new * LEAST]], np.float32), 2, [0, 4])
        expect = np.clip(np.rint(codes[1, 0, 2].astype(np.float64) * (new / scale)), -128, 127)
        for got, got_scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            assert float(got_scale[0, 0]) == scale * LEAST
            assert np.array_equal(got[0, 0, 15].cpu().numpy(), expect)
            if old == scale:
                assert np.array_equal(got[0, 0, :15].cpu().numpy(), codes[0, 0, :15])
    # What needs less than half of the least number is zero.
    codes = rng.integers(-1, 2, (2, 1, 16, dim)).astype(np.int8)
    cache = _two_pages(codes, np.array([[0.0], [LEAST]], np.float32), 2, [0, 4])
    assert float(cache.k_scale[0, 0]) == 0.0 and torch.all(cache.k[0, 0, 15] == 0) and torch.all(cache.v[0, 0, 15] == 0)
    assert _status_ok()
