"""Forms of the norm / rotation / append operators: block-scaled appends of the
sizes between which the launch changes.  Tolerances as in test_gpu_rope_cache."""

import numpy as np
import pytest

import rope_cache_reference as ref
from test_gpu_rope_cache import EPS, _block_device, _block_state, _rows, _table, _want, _weight

pytestmark = pytest.mark.gpu


def _inputs(rng, dtype, T, H, Hkv, D, R, layout, weights, std=1.0):
    import torch

    table, table_h = _table(rng, 400, R)
    pos = rng.integers(0, 400, T).astype(np.int32)
    rows = [_rows(rng, dtype, T, n, D, layout, std) for n in (H, Hkv, Hkv)]
    w = [_weight(rng, weights, dtype, D) for _ in range(2)]
    return rows, w, table, table_h, pos, torch.from_numpy(pos).cuda()


@pytest.mark.parametrize("T,H,Hkv,D", [(2300, 3, 1, 64), (2400, 8, 2, 128), (3300, 32, 8, 128), (3700, 16, 1, 64),
                                       (4500, 2, 2, 256)])
def test_block_scaled_between_the_waves(cflib, T, H, Hkv, D):
    """Windows just below and past a CTA per SM, with few and many query rows: the
    queries are those of the pass without a cache, and V's bytes the definition's."""
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(T)
    ((q, _), (k, kh), (v, vh)), ((qw, _), (kw, kwh)), table, table_h, pos, dpos = _inputs(
        rng, "bf16", T, H, Hkv, D, D, "fused", "own")
    pool = T // 16 + 4
    slots = (np.arange(T) + 7).astype(np.int32)
    slots[rng.integers(0, T, 20)] = -1
    codes, scales = _block_state(rng, pool, Hkv, D)
    dev = _block_device(codes, scales)
    qo, ko, q2 = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
    ops.rope_and_cache_fp8_block(qo, q, k, v, *dev, torch.from_numpy(slots).cuda(), dpos, table, qw, kw, EPS)
    ops.qk_norm_rope(q2, ko, q, k, dpos, table, qw, kw, EPS)
    assert torch.equal(qo, q2)
    ref.append_block(vh, codes[1], scales[1], slots)
    assert np.array_equal(dev[3].cpu().numpy(), scales[1])
    assert np.array_equal(ref.from_e4m3(dev[1].view(torch.uint8).cpu().numpy()), ref.from_e4m3(codes[1]))
    y, bound = _want(kh, kwh, table_h, pos, False)
    ref.append_block(y, codes[0], scales[0], slots)
    assert np.array_equal(dev[2].cpu().numpy(), scales[0])
    live = slots >= 0
    b, o = slots[live] // 16, slots[live] % 16
    s = scales[0][b][..., None]
    got = ref.from_e4m3(dev[0].view(torch.uint8).cpu().numpy()[b, :, o]) * s
    assert (np.abs(got - y[live]) <= 2.0 ** -4 * np.maximum(np.abs(y[live]), 2.0 ** -6 * s) + bound[live]).all()
    assert ops.device_errors(0) == 0
