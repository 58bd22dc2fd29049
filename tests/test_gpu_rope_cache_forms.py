"""Combinations of the norm / rotation / append operators' forms: adjacent
pairs and norm weights into every kind of cache, and block-scaled appends of
the sizes between which the launch changes.  Tolerances as in
test_gpu_rope_cache."""

import numpy as np
import pytest

import rope_cache_reference as ref
from test_gpu_rope_cache import EPS, U, _block_device, _block_state, _close, _rows, _table, _want, _weight

pytestmark = pytest.mark.gpu


def _inputs(rng, dtype, T, H, Hkv, D, R, layout, weights, std=1.0):
    import torch

    table, table_h = _table(rng, 400, R)
    pos = rng.integers(0, 400, T).astype(np.int32)
    rows = [_rows(rng, dtype, T, n, D, layout, std) for n in (H, Hkv, Hkv)]
    w = [_weight(rng, weights, dtype, D) for _ in range(2)]
    return rows, w, table, table_h, pos, torch.from_numpy(pos).cuda()


@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("weights", [None, "own", "f32"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,H,Hkv,D,R,layout", [(37, 6, 2, 128, 128, "fused"), (5, 3, 1, 80, 40, "odd"),
                                                (50, 4, 4, 256, 128, "fused")])
def test_into_caches_of_the_rows_type(cflib, dtype, T, H, Hkv, D, R, layout, weights, il):
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(T + D)
    ((q, qh), (k, kh), (v, vh)), ((qw, qwh), (kw, kwh)), table, table_h, pos, dpos = _inputs(
        rng, dtype, T, H, Hkv, D, R, layout, weights)
    bs, pool = 16, 6
    slots = rng.permutation(pool * bs)[:T].astype(np.int32)
    kc, vc = (torch.zeros(pool, Hkv, bs, D, dtype=q.dtype, device="cuda") for _ in range(2))
    qo = torch.full((T, H, D), 9.0, dtype=q.dtype, device="cuda")
    ops.rope_and_cache(qo, q, k, v, kc, vc, torch.from_numpy(slots).cuda(), dpos, table, qw, kw, EPS, il)
    _close(qo.double().cpu().numpy(), *_want(qh, qwh, table_h, pos, il), dtype, "q")
    b, o = (torch.from_numpy(x).cuda() for x in (slots // bs, slots % bs))
    _close(kc[b, :, o].double().cpu().numpy(), *_want(kh, kwh, table_h, pos, il), dtype, "k")
    assert torch.equal(vc[b, :, o], v)
    assert ops.device_errors(0) == 0


@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("weights", [None, "own", "f32"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,H,Hkv,D,R,layout", [(37, 6, 2, 128, 128, "fused"), (5, 3, 1, 80, 40, "odd"),
                                                (50, 4, 4, 256, 128, "fused")])
def test_into_caches_of_one_scale(cflib, dtype, T, H, Hkv, D, R, layout, weights, il):
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(T + D + 1)
    ((q, qh), (k, kh), (v, vh)), ((qw, qwh), (kw, kwh)), table, table_h, pos, dpos = _inputs(
        rng, dtype, T, H, Hkv, D, R, layout, weights, std=4.0)
    ksc, vsc, pool = 0.013, 0.029, 6
    slots = rng.permutation(pool * 16)[:T].astype(np.int32)
    kc, vc = (torch.zeros(pool, Hkv, 16, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
              for _ in range(2))
    qo = torch.full((T, H, D), 9.0, dtype=q.dtype, device="cuda")
    ops.rope_and_cache_fp8(qo, q, k, v, kc, vc, torch.from_numpy(slots).cuda(), dpos, table, ksc, vsc, qw, kw, EPS, il)
    _close(qo.double().cpu().numpy(), *_want(qh, qwh, table_h, pos, il), dtype, "q")
    b, o = slots // 16, slots % 16
    got = vc.view(torch.uint8).cpu().numpy()[b, :, o]
    # V is divided in f32, then rounded
    assert np.array_equal(got, ref.to_e4m3((vh.astype(np.float32) / np.float32(vsc)).astype(np.float64)))
    y, bound = _want(kh, kwh, table_h, pos, il)
    y, bound = y / np.float64(np.float32(ksc)), bound / ksc
    got = ref.from_e4m3(kc.view(torch.uint8).cpu().numpy()[b, :, o])
    y = np.clip(y, -448, 448)
    assert (np.abs(got - y) <= 2.0 ** -4 * np.maximum(np.abs(y), 2.0 ** -6) + bound + 2 * U * np.abs(y)).all()
    assert ops.device_errors(0) == 0


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
