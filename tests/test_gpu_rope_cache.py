"""Query / key norms with the position rotation (cf_qk_norm_rope), and the
appends that carry them (cf_rope_and_cache, _fp8, _fp8_block,
cf_reshape_and_cache_fp8_block), against their definitions in float64.

Tolerance of a normed and rotated element, with u = 2^-24 and a pair (a, b)
scaled to its norm: the sum of squares is off by at most (16 + 5 + 1) u
relatively (chains of up to 16 additions, a tree of 5, the division), half of
that through the square root, rsqrtf by 4 u, the two products that fold weight
and angle by 2 u, the rotation's products and sum by 3 u: below 24 u (|a| +
|b|).  The result's own rounding is half a step of its type more.  e4m3 bytes:
half a step 2^-4 |x| (2^-10 below the normals) more.
"""

import numpy as np
import pytest

import rope_cache_reference as ref
from helpers import half_ulp, torch_dtype

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}
EPS = 1e-6


def _rows(rng, dtype, T, heads, D, layout, std=1.0):
    """A CUDA tensor [T, heads, D] in one of the layouts a caller may have, and its values."""
    import torch

    x = torch.from_numpy((rng.standard_normal((T, heads, D)) * std).astype(np.float32)).to(torch_dtype(dtype))
    if layout == "dense":
        t = x.cuda()
    elif layout == "fused":  # a slice of a wider row
        w = torch.zeros((T, heads + 3, D), dtype=x.dtype, device="cuda")
        w[:, 2:2 + heads] = x.cuda()
        t = w[:, 2:2 + heads]
    elif layout == "odd":  # starts and strides of one element
        w = torch.zeros((T * (heads * D + 1) + 1,), dtype=x.dtype, device="cuda")
        t = w[1:].as_strided((T, heads, D), (heads * D + 1, D, 1), 1)
        t.copy_(x.cuda())
    else:  # heads outermost
        w = torch.zeros((heads, T, D), dtype=x.dtype, device="cuda")
        t = w.transpose(0, 1)
        t.copy_(x.cuda())
    return t, x.double().numpy()


def _weight(rng, kind, dtype, D):
    import torch

    if kind is None:
        return None, None
    w = torch.from_numpy((1 + 0.3 * rng.standard_normal(D)).astype(np.float32))
    w = w if kind == "f32" else w.to(torch_dtype(dtype))
    return w.cuda(), w.double().numpy()


def _want(x, w, table, pos, il):
    """Values, and the bound of the f32 arithmetic before the last rounding."""
    y = ref.norm_rope(x, w, table, pos, il, EPS)
    r = table.shape[1]
    z = np.abs(ref.norm_rope(x, w, table[:1] * 0 + np.r_[np.ones(r // 2), np.zeros(r // 2)], pos * 0, il, EPS))
    s = z.copy()
    i = np.arange(r // 2)
    ia, ib = (2 * i, 2 * i + 1) if il else (i, i + r // 2)
    s[..., ia] = s[..., ib] = z[..., ia] + z[..., ib]
    return y, 24 * U * s


def _close(got, y, bound, dtype, what=""):
    lim = bound + half_ulp(np.abs(y) + bound, dtype) + TINY[dtype]
    err = np.abs(got - y)
    assert (err <= lim).all(), f"{what}: {(err / lim).max():.3f} of the bound"


def _table(rng, n, r):
    from cacheflow_b200 import ops

    t = ops.rope_table(n, r)
    i = np.arange(r // 2)
    a = np.arange(n)[:, None] * 10000.0 ** (-2.0 * i / r)
    want = np.concatenate([np.cos(a), np.sin(a)], 1)
    # an f32 rounding, and float64's own of an angle up to n
    assert np.abs(t.cpu().numpy() - want).max() <= U + n * 2.0 ** -52
    return t, t.cpu().numpy()


SHAPES = [  # T, H, Hkv, D, rotary
    (1, 32, 8, 128, 128),
    (3, 5, 1, 64, 64),
    (33, 7, 7, 128, 64),
    (17, 4, 2, 256, 256),
    (5, 3, 3, 80, 40),
    (9, 6, 2, 96, 96),
    (2, 1, 1, 192, 192),
    (40, 9, 3, 80, 20),
    (4, 2, 1, 2, 2),
    (6, 3, 2, 250, 134),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["dense", "fused", "odd", "heads"])
@pytest.mark.parametrize("T,H,Hkv,D,R", SHAPES)
def test_qk_norm_rope(cflib, dtype, layout, T, H, Hkv, D, R):
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(T + H + D + R)
    table, table_h = _table(rng, 700, R)
    pos = rng.integers(0, 700, T).astype(np.int32)
    for il, qk, kk in ((False, "own", "own"), (True, None, None), (True, "f32", None), (False, None, "f32")):
        q, qh = _rows(rng, dtype, T, H, D, layout)
        k, kh = _rows(rng, dtype, T, Hkv, D, layout)
        qw, qwh = _weight(rng, qk, dtype, D)
        kw, kwh = _weight(rng, kk, dtype, D)
        qo = torch.full((T, H, D), 9.0, dtype=q.dtype, device="cuda")
        ko = torch.full((T, Hkv, D), 9.0, dtype=q.dtype, device="cuda")
        ops.qk_norm_rope(qo, ko, q, k, torch.from_numpy(pos).cuda(), table, qw, kw, EPS, il)
        for got, x, w, what in ((qo, qh, qwh, "q"), (ko, kh, kwh, "k")):
            _close(got.double().cpu().numpy(), *_want(x, w, table_h, pos, il), dtype, f"{what} {il} {qk} {kk}")
        # in place
        before = q.clone(), k.clone()
        ops.qk_norm_rope(q, k, q, k, torch.from_numpy(pos).cuda(), table, qw, kw, EPS, il)
        assert torch.equal(q, qo) and torch.equal(k, ko)
        assert not torch.equal(before[0], q) or D == 2
    assert ops.device_errors(0) == 0


def test_zero_rows_and_values_that_are_not_finite(cflib):
    """A row of zeros stays zero under the norm; NaN and infinity stay in their row."""
    import torch

    from cacheflow_b200 import ops

    q = torch.randn(4, 3, 128, device="cuda").bfloat16()
    q[0, 1] = 0
    q[1, 0, 5] = float("nan")
    q[2, 2, 7] = float("inf")
    k = torch.randn(4, 1, 128, device="cuda").bfloat16()
    w = torch.ones(128, device="cuda")
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    ops.qk_norm_rope(qo, ko, q, k, pos, ops.rope_table(8, 128), w, w)
    assert (qo[0, 1] == 0).all()
    assert torch.isnan(qo[1, 0]).all() and torch.isfinite(qo[1, 1:]).all()
    assert torch.isfinite(qo[2, :2]).all() and torch.isfinite(ko).all()
    # without norm only the pair of the column
    ops.qk_norm_rope(qo, ko, q, k, pos, ops.rope_table(8, 128))
    assert torch.isnan(qo[1, 0]).sum() == 2 and torch.isfinite(qo[0]).all()
    # columns that do not rotate pass as they are, whatever is in them
    q[3, :, 64:] = float("inf")
    ops.qk_norm_rope(qo, ko, q, k, pos, ops.rope_table(8, 64))
    assert torch.equal(qo[3, :, 64:], q[3, :, 64:]) and torch.isfinite(qo[3, :, :64]).all()


@pytest.mark.parametrize("op", ["qk", "same", "fp8", "block"])
def test_padding_and_positions_out_of_range(cflib, op):
    import torch

    from cacheflow_b200 import _lib, ops

    T, H, Hkv, D = 6, 4, 2, 64
    g = torch.Generator().manual_seed(3)
    q = torch.randn(T, H, D, generator=g).half().cuda()
    k, v = (torch.randn(T, Hkv, D, generator=g).half().cuda() for _ in range(2))
    pos = torch.tensor([3, -1, 0, 10, 9, 2], dtype=torch.int32, device="cuda")  # 10: one past the table
    slots = torch.tensor([5, 6, -1, 7, 100000, 16], dtype=torch.int32, device="cuda")  # 100000: past the pool
    table = ops.rope_table(10, D)
    qo = torch.full_like(q, 7.0)
    ops.device_errors(0)
    dt = torch.half if op in ("qk", "same") else torch.float8_e4m3fn
    kc, vc = (torch.full((4, Hkv, 16, D), 3.0, device="cuda").to(dt) for _ in range(2))
    ks, vs = torch.ones(4, Hkv, device="cuda"), torch.ones(4, Hkv, device="cuda")
    args = (qo, q, k, v, kc, vc)
    if op == "qk":
        ko = torch.full_like(k, 7.0)
        ops.qk_norm_rope(qo, ko, q, k, pos, table)
        assert (ko[[1, 3]] == 7).all() and (ko[[0, 2, 4, 5]] != 7).any(-1).all()
        want = _lib.CF_DEVERR_POSITION
    else:
        if op == "same":
            ops.rope_and_cache(*args, slots, pos, table)
        elif op == "fp8":
            ops.rope_and_cache_fp8(*args, slots, pos, table, 0.05, 0.05)
        else:
            ops.rope_and_cache_fp8_block(*args, ks, vs, slots, pos, table)
        want = _lib.CF_DEVERR_POSITION | _lib.CF_DEVERR_SLOT
        touched = torch.zeros(4, 16, dtype=torch.bool, device="cuda")
        touched.view(-1)[[5, 16]] = True  # the slots of tokens 0 and 5
        for c in (kc, vc):
            c = c.float()
            same = (c == 3).all(-1).all(1)
            assert not same[touched].any()
            if op != "block":  # there a grown scale stores a block's other rows anew
                assert same[~touched].all()
            assert (c[2:] == 3).all()
    assert ops.device_errors(0) == want
    # a token that is not in range writes no query either; one that only has no slot does
    assert (qo[[1, 3]] == 7).all() and (qo[[0, 2, 4, 5]] != 7).any(-1).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["fused", "odd"])
@pytest.mark.parametrize("T,H,Hkv,D,R", [(1, 4, 1, 128, 128), (50, 5, 3, 64, 32), (21, 2, 2, 256, 256), (7, 3, 1, 80, 80)])
def test_rope_and_cache(cflib, dtype, layout, T, H, Hkv, D, R):
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(T + D)
    bs, pool = 8, 20  # any block size
    table, table_h = _table(rng, 300, R)
    pos = rng.integers(0, 300, T).astype(np.int32)
    slots = rng.permutation(pool * bs)[:T].astype(np.int32)
    if T > 4:
        slots[3] = -1
    q, qh = _rows(rng, dtype, T, H, D, layout)
    k, kh = _rows(rng, dtype, T, Hkv, D, layout)
    v, vh = _rows(rng, dtype, T, Hkv, D, layout)
    qw, qwh = _weight(rng, "own", dtype, D)
    kw, kwh = _weight(rng, "own", dtype, D)
    kc = torch.randn(pool, Hkv, bs, D, device="cuda").to(q.dtype)
    vc = torch.randn(pool, Hkv, bs, D, device="cuda").to(q.dtype)
    k0, v0 = kc.clone(), vc.clone()
    qo = torch.empty((T, H, D), dtype=q.dtype, device="cuda")
    ops.rope_and_cache(qo, q, k, v, kc, vc, torch.from_numpy(slots).cuda(), torch.from_numpy(pos).cuda(), table, qw,
                       kw, EPS)
    _close(qo.double().cpu().numpy(), *_want(qh, qwh, table_h, pos, False), dtype, "q")
    live = slots >= 0
    b, o = torch.from_numpy(slots[live] // bs).cuda(), torch.from_numpy(slots[live] % bs).cuda()
    y, bound = _want(kh, kwh, table_h, pos, False)
    _close(kc[b, :, o].double().cpu().numpy(), y[live], bound[live], dtype, "k")
    assert torch.equal(vc[b, :, o], v[torch.from_numpy(live).cuda()])  # bit for bit
    kc[b, :, o], vc[b, :, o] = k0[b, :, o], v0[b, :, o]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)  # every other slot as it was
    # the same query rows as the pass without a cache
    ko = torch.empty_like(k)
    q2 = torch.empty_like(qo)
    ops.qk_norm_rope(q2, ko, q, k, torch.from_numpy(pos).cuda(), table, qw, kw, EPS)
    assert torch.equal(q2, qo)
    assert ops.device_errors(0) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_rope_and_cache_fp8(cflib, dtype, D):
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(D)
    T, H, Hkv, pool = 40, 3, 2, 6
    ksc, vsc = 0.037, 0.011
    table, table_h = _table(rng, 100, D)
    pos = rng.integers(0, 100, T).astype(np.int32)
    slots = rng.permutation(pool * 16)[:T].astype(np.int32)
    q, qh = _rows(rng, dtype, T, H, D, "fused")
    k, kh = _rows(rng, dtype, T, Hkv, D, "fused", std=8.0)
    v, vh = _rows(rng, dtype, T, Hkv, D, "fused", std=4.0)  # some past 448 * scale
    kc, vc = (torch.zeros(pool, Hkv, 16, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
              for _ in range(2))
    qo = torch.empty((T, H, D), dtype=q.dtype, device="cuda")
    ops.rope_and_cache_fp8(qo, q, k, v, kc, vc, torch.from_numpy(slots).cuda(), torch.from_numpy(pos).cuda(), table,
                           ksc, vsc)
    b, o = slots // 16, slots % 16
    got_v = vc.view(torch.uint8).cpu().numpy()[b, :, o]
    # V is divided in f32, then rounded: as reshape_and_cache_fp8 stores it
    assert np.array_equal(got_v, ref.to_e4m3((vh.astype(np.float32) / np.float32(vsc)).astype(np.float64)))
    y, bound = _want(kh, None, table_h, pos, False)
    y, bound = y / np.float64(np.float32(ksc)), bound / ksc
    got = ref.from_e4m3(kc.view(torch.uint8).cpu().numpy()[b, :, o])
    y = np.clip(y, -448, 448)
    step = np.maximum(np.abs(y), 2.0 ** -6)
    assert (np.abs(got - y) <= 2.0 ** -4 * step + bound + 2 * U * np.abs(y)).all()


def _block_state(rng, pool, Hkv, D, lo=-9, hi=-4):
    codes = ref.to_e4m3(rng.standard_normal((2, pool, Hkv, 16, D)) * 96)
    scales = np.exp2(rng.integers(lo, hi, (2, pool, Hkv))).astype(np.float32)
    return codes, scales


def _block_device(codes, scales):
    import torch

    return ([torch.from_numpy(c.copy()).cuda().view(torch.float8_e4m3fn) for c in codes]
            + [torch.from_numpy(s.copy()).cuda() for s in scales])


def _same_block(dev, codes, scales, what=""):
    import torch

    for i, name in enumerate(("K", "V")):
        s = dev[2 + i].cpu().numpy()
        assert np.array_equal(s, scales[i], equal_nan=True), f"{what} {name} scales: {(s != scales[i]).sum()} differ"
        c = dev[i].view(torch.uint8).cpu().numpy()
        # -0 and 0 are one value
        a, b = ref.from_e4m3(c), ref.from_e4m3(codes[i])
        assert np.array_equal(a, b, equal_nan=True), f"{what} {name}: {(a != b).sum()} of {a.size} differ"


def _orders(rng, name, pool):
    if name == "decode":  # one token of each block, every offset, offset 0 among them
        return np.array([b * 16 + (b * 7) % 16 for b in rng.permutation(pool)], np.int32)
    if name == "prompt":  # runs that begin and end inside blocks, padding behind
        s = []
        for first, n, blocks in ((0, 40, [3, 1, 7]), (5, 11, [0]), (9, 7, [2]), (0, 16, [5]), (15, 2, [6, 4])):
            for i in range(n):
                p = first + i
                s.append(blocks[p // 16] * 16 + p % 16)
        return np.array(s + [-1] * 5, np.int32)
    if name == "scattered":  # rows of a block far apart in the call, in any order, padding between
        s = rng.permutation(pool * 16)[: pool * 9].astype(np.int32)
        s[::13] = -1
        return s
    # duplicates: the later token of a slot is stored
    return rng.integers(0, pool * 16, 300).astype(np.int32)


@pytest.mark.parametrize("order", ["decode", "prompt", "scattered", "twice"])
@pytest.mark.parametrize("dtype,Hkv,D", [("bf16", 2, 128), ("f16", 3, 64), ("f32", 1, 256), ("bf16", 1, 80),
                                         ("f32", 2, 16), ("f16", 1, 48)])
def test_reshape_and_cache_fp8_block(cflib, order, dtype, Hkv, D):
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(len(order) + D)
    pool = 8 if order == "prompt" else 40
    slots = _orders(rng, order, pool)
    codes, scales = _block_state(rng, pool, Hkv, D)
    dev = _block_device(codes, scales)
    for step in range(3):  # growing values: scales rise, rows are stored anew
        x = rng.standard_normal((2, len(slots), Hkv, D)) * np.exp(rng.standard_normal((2, len(slots), 1, 1))) * 4.0 ** step
        t = [torch.from_numpy(v.astype(np.float32)).to(torch_dtype(dtype)).cuda() for v in x]
        ops.reshape_and_cache_fp8_block(t[0], t[1], *dev, torch.from_numpy(slots).cuda())
        for i in range(2):
            ref.append_block(t[i].double().cpu().numpy(), codes[i], scales[i], slots)
        _same_block(dev, codes, scales, f"step {step}")
    assert ops.device_errors(0) == 0


def test_block_append_one_row_at_a_time(cflib):
    """A block filled token by token holds the values within e4m3's steps of
    what it would hold filled at once, at a scale that is the same."""
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(6)
    D, n = 128, 40
    x = (rng.standard_normal((n, 1, D)) * np.exp(1.5 * rng.standard_normal((n, 1, 1)))).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    codes, scales = _block_state(rng, 4, 1, D)
    once, each = _block_device(codes, scales), _block_device(codes, scales)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    ops.reshape_and_cache_fp8_block(t, t, *once, slots)
    for i in range(n):
        ops.reshape_and_cache_fp8_block(t[i:i + 1], t[i:i + 1], *each, slots[i:i + 1])
    assert torch.equal(once[2], each[2]) and torch.equal(once[3], each[3])
    for dev in (once, each):
        s = dev[2].cpu().numpy()[:3, 0]
        got = ref.from_e4m3(dev[0].view(torch.uint8).cpu().numpy()[:3, 0]) * s[:, None, None]
        got = got.reshape(48, D)[:n]
        step = np.repeat(s, 16)[:n, None]
        # each storing anew may round once more below the smallest normal: 2^-10 of the scale, at most 16 times
        assert (np.abs(got - x[:, 0]) <= 2.0 ** -4 * np.abs(x[:, 0]) + 16 * 2.0 ** -10 * step).all()


def test_block_append_of_odd_values(cflib):
    """Zeros, values that are not finite, tiny and huge ones, and scales that
    are no powers of two or were never set."""
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(9)
    Hkv, D, pool = 1, 32, 8
    codes, scales = _block_state(rng, pool, Hkv, D)
    scales[:, 1] = 0.0       # an empty block
    scales[:, 2] = 0.0371    # no power of two
    scales[:, 3] = np.nan    # never set: written from its offset 0 on
    scales[:, 4] = -1.0
    slots = np.array([16 * 0, 16 * 0 + 1, 16 * 1 + 4, 16 * 2 + 3, 16 * 3, 16 * 4 + 2, 16 * 5, 16 * 6, 16 * 7 + 9],
                     np.int32)
    x = rng.standard_normal((len(slots), Hkv, D)).astype(np.float32)
    x[0] = 0
    x[1] = 0            # block 0: fresh, all zero: scale 0
    x[2] = 0            # block 1: nothing but zeros in an empty block
    x[3] = 448 * 0.0371 * 0.9  # block 2: fits its scale
    x[5, 0, :4] = [np.nan, np.inf, -np.inf, 1.0]
    x[6] = 1e-42        # block 5: f32 subnormals, fresh
    x[7] = 3e38         # block 6: the largest, fresh
    x[8] = 1e30         # block 7: grows from an ordinary scale
    dev = _block_device(codes, scales)
    t = torch.from_numpy(x).cuda()
    ops.reshape_and_cache_fp8_block(t, t, *dev, torch.from_numpy(slots).cuda())
    for i in range(2):
        ref.append_block(x.astype(np.float64), codes[i], scales[i], slots)
    _same_block(dev, codes, scales)


def test_block_append_past_one_piece(cflib):
    """Calls of more than 16384 tokens are appended as consecutive pieces."""
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(10)
    Hkv, D, T = 1, 16, 2 * 16384 + 777
    pool = T // 16 + 2
    slots = (np.arange(T) + 5).astype(np.int32)
    slots[40000 - 16384 * 2: 40030 - 16384 * 2] = -1
    codes, scales = _block_state(rng, pool, Hkv, D)
    dev = _block_device(codes, scales)
    x = (rng.standard_normal((T, Hkv, D)) * np.exp(rng.standard_normal((T, 1, 1)))).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    ops.reshape_and_cache_fp8_block(t, t, *dev, torch.from_numpy(slots).cuda())
    for i in range(2):
        for p in range(0, T, 16384):
            ref.append_block(x[p:p + 16384].astype(np.float64), codes[i], scales[i], slots[p:p + 16384])
    _same_block(dev, codes, scales)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,Hkv,D,R,il", [(4, 2, 128, 128, False), (3, 1, 64, 32, True), (2, 1, 256, 256, False),
                                          (5, 1, 80, 40, False)])
def test_rope_and_cache_fp8_block(cflib, dtype, H, Hkv, D, R, il):
    """Scales, and bytes within e4m3's half step of the definition (a value
    next to a border may go to either side of it)."""
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(D + R)
    pool = 8
    slots = _orders(rng, "prompt", pool)
    T = len(slots)
    table, table_h = _table(rng, 500, R)
    pos = rng.integers(0, 500, T).astype(np.int32)
    pos[7] = -1  # a padding token: neither its query nor its rows
    codes, scales = _block_state(rng, pool, Hkv, D)
    dev = _block_device(codes, scales)
    q, qh = _rows(rng, dtype, T, H, D, "fused")
    k, kh = _rows(rng, dtype, T, Hkv, D, "fused", std=3.0)
    v, vh = _rows(rng, dtype, T, Hkv, D, "fused", std=3.0)
    qw, qwh = _weight(rng, "f32", dtype, D)
    kw, kwh = _weight(rng, "f32", dtype, D)
    qo = torch.full((T, H, D), 7.0, dtype=q.dtype, device="cuda")
    ops.rope_and_cache_fp8_block(qo, q, k, v, *dev, torch.from_numpy(slots).cuda(), torch.from_numpy(pos).cuda(),
                                 table, qw, kw, EPS, il)
    live = pos >= 0
    assert (qo[7] == 7).all()
    y, bound = _want(qh, qwh, table_h, np.maximum(pos, 0), il)
    _close(qo.double().cpu().numpy()[live], y[live], bound[live], dtype, "q")
    y, bound = _want(kh, kwh, table_h, np.maximum(pos, 0), il)
    ref.append_block(y, codes[0], scales[0], slots, live)
    ref.append_block(vh, codes[1], scales[1], slots, live)
    assert np.array_equal(dev[2].cpu().numpy(), scales[0])
    got = ref.from_e4m3(dev[0].view(torch.uint8).cpu().numpy())
    want = ref.from_e4m3(codes[0])
    differ = got != want
    assert differ.mean() < 1e-3
    assert (np.abs(got - want) <= 2.0 ** -3 * np.abs(want) + 2.0 ** -9)[differ].all()
    # V has no arithmetic: equal
    _same_block([dev[1], dev[1], dev[3], dev[3]], [codes[1]] * 2, [scales[1]] * 2)
    # the rows that the definition says are appended, within their steps
    for t in np.flatnonzero(live & (slots >= 0)):
        b, o = slots[t] // 16, slots[t] % 16
        s = scales[0][b][:, None]
        e = np.abs(got[b, :, o] * s - y[t])
        assert (e <= 2.0 ** -4 * np.maximum(np.abs(y[t]), 2.0 ** -6 * s) + bound[t]).all()


def test_padding_tokens_do_not_hide_a_slot(cflib):
    """Padding rows that all name a slot of a real token, before and after it,
    near and far in the call: the real token is stored."""
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(15)
    T, H, Hkv, D, pool = 100, 2, 2, 64, 6
    table, table_h = _table(rng, 50, D)
    pos = np.full(T, -1, np.int32)
    slots = np.full(T, 35, np.int32)  # every padding row names slot 35
    for t, s, p in ((40, 35, 7), (41, 36, 8), (10, 0, 3), (95, 1, 4)):
        pos[t], slots[t] = p, s
    slots[60:70] = 0
    codes, scales = _block_state(rng, pool, Hkv, D)
    dev = _block_device(codes, scales)
    q, k, v = (torch.from_numpy(rng.standard_normal((T, n, D)).astype(np.float32)).cuda() for n in (H, Hkv, Hkv))
    ops.rope_and_cache_fp8_block(q, q, k, v, *dev, torch.from_numpy(slots).cuda(), torch.from_numpy(pos).cuda(), table)
    live = pos >= 0
    ref.append_block(v.double().cpu().numpy(), codes[1], scales[1], slots, live)
    _same_block([dev[1], dev[1], dev[3], dev[3]], [codes[1]] * 2, [scales[1]] * 2)
    y = ref.norm_rope(k.double().cpu().numpy(), None, table_h, np.maximum(pos, 0), False, EPS)
    ref.append_block(y, codes[0], scales[0], slots, live)
    assert np.array_equal(dev[2].cpu().numpy(), scales[0])
    assert ops.device_errors(0) == 0


def test_scales_move_with_their_blocks(cflib):
    """copy_blocks, compact_kv_cache, memset_blocks and swap_blocks take the
    scale arrays as caches of one element a head."""
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(12)
    pool, Hkv, D = 10, 3, 64
    codes, scales = _block_state(rng, pool, Hkv, D)
    kc, vc, ks, vs = _block_device(codes, scales)
    pairs = torch.tensor([[1, 4], [2, 7]], dtype=torch.int64, device="cuda")
    ops.copy_blocks(kc, vc, pairs)
    ops.copy_blocks(ks.view(pool, Hkv, 1, 1), vs.view(pool, Hkv, 1, 1), pairs)
    src, dst = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([9], [0]))
    ops.compact_kv_cache(kc, vc, src, dst)
    ops.compact_kv_cache(ks.view(pool, Hkv, 1, 1), vs.view(pool, Hkv, 1, 1), src, dst)
    ops.memset_blocks(ks.view(pool, Hkv, 1, 1), torch.tensor([5], dtype=torch.int32, device="cuda"))
    want = scales.copy()
    for s, d in ((1, 4), (2, 7), (9, 0)):
        want[:, d] = want[:, s]
        codes[:, d] = codes[:, s]
    want[0, 5] = 0
    _same_block([kc, vc, ks, vs], codes, want)
    host = torch.zeros(pool, Hkv).pin_memory()
    ops.swap_blocks(ks.view(pool, Hkv, 1, 1), host.view(pool, Hkv, 1, 1), pairs)
    torch.cuda.synchronize()
    assert np.array_equal(host.numpy()[[4, 7]], want[0][[1, 2]])


def test_on_a_stream_and_captured(cflib):
    """The appends and the attention after them, on a side stream and in a
    graph that is replayed with other tokens."""
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(14)
    S, H, Hkv, D, pool = 3, 8, 2, 128, 12
    table, table_h = _table(rng, 200, D)
    tables = torch.from_numpy(rng.permutation(pool).astype(np.int32).reshape(S, 4)).cuda()
    dev = _block_device(np.zeros((2, pool, Hkv, 16, D), np.uint8), np.zeros((2, pool, Hkv), np.float32))
    q = torch.zeros(S, H, D, dtype=torch.bfloat16, device="cuda")
    k, v = torch.zeros(S, Hkv, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(S, Hkv, D, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(S, dtype=torch.int32, device="cuda")
    lens, slots, out = pos + 1, pos.clone(), torch.zeros_like(q)

    def step():
        ops.rope_and_cache_fp8_block(q, q, k, v, *dev, slots, pos, table)
        ops.paged_attention_fp8_block_v1(out, q, *dev, tables, lens, None, 64)

    side = torch.cuda.Stream()
    slots.fill_(-1)
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    th = tables.cpu().numpy()
    keys, vals = [], []
    for i in range(40):
        x = [rng.standard_normal(s).astype(np.float32) for s in ((S, H, D), (S, Hkv, D), (S, Hkv, D))]
        for t, a in zip((q, k, v), x):
            t.copy_(torch.from_numpy(a))
        qh = q.double().cpu().numpy()
        keys.append(ref.norm_rope(k.double().cpu().numpy(), None, table_h, np.full(S, i), False, EPS))
        vals.append(v.double().cpu().numpy())
        pos.fill_(i)
        lens.fill_(i + 1)
        slots.copy_(torch.from_numpy((th[:, i // 16] * 16 + i % 16).astype(np.int32)))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            g.replay()
        side.synchronize()
    qr = ref.norm_rope(qh, None, table_h, np.full(S, 39), False, EPS)
    kk, vv = np.stack(keys, 1), np.stack(vals, 1)  # [S, 40, Hkv, D]
    lg = np.einsum("shgd,sthd->shgt", qr.reshape(S, Hkv, H // Hkv, D), kk) / np.sqrt(D)
    p = np.exp(lg - lg.max(-1, keepdims=True))
    want = (np.einsum("shgt,sthd->shgd", p, vv) / p.sum(-1, keepdims=True)).reshape(S, H, D)
    got = out.double().cpu().numpy()
    # stored in e4m3: each value off by up to 2^-4, 2.6e-2 of it on the mean square
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < 0.06
    assert ops.device_errors(0) == 0


def test_numbers_past_f32_are_refused(cflib):
    import torch

    from cacheflow_b200 import ops

    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    w = torch.ones(128, device="cuda")
    for eps in (1e300, float("inf"), 0.0):
        with pytest.raises(ops.CacheFlowError):
            ops.qk_norm_rope(q, q.clone(), q, q.clone(), pos, ops.rope_table(8, 128), w, w, eps=eps)
    c8 = torch.zeros(2, 4, 16, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    sc = torch.zeros(2, 4, device="cuda")
    with pytest.raises(ops.CacheFlowError):
        ops.paged_attention_fp8_block_v1(q.clone(), q, c8, c8, sc, sc, pos[:, None], pos, scale=1e300)


@pytest.mark.parametrize("blocks", [1, 2, 3])
@pytest.mark.parametrize("op", ["append", "rope"])
def test_block_append_of_rows_far_from_their_window(cflib, blocks, op):
    """A window that leads one, two or three blocks, block 0 among them, whose
    other rows, some of them twice, lie anywhere in the call, beside padding
    with every negative slot and tokens whose positions are out of the table."""
    import torch

    from cacheflow_b200 import ops

    rng = np.random.default_rng(60 + blocks)
    T, Hkv, D, pool = 600, 2, 128, 40
    ids = [0, 7, 39][:blocks]
    slots = -rng.integers(1, 40, T).astype(np.int32)
    rest = rng.permutation([b for b in range(pool) if b not in ids])
    slots[16:32] = [ids[i % blocks] * 16 + i // blocks % 3 for i in range(16)]
    for i in rng.choice(np.arange(48, T), 60, replace=False):
        slots[i] = ids[rng.integers(blocks)] * 16 + rng.integers(16)
    for n, i in enumerate(rng.choice(np.flatnonzero(slots < 0), 200, replace=False)):
        slots[i] = rest[n % 30] * 16 + rng.integers(16)
    pos = rng.integers(0, 50, T).astype(np.int32)
    if op == "rope":
        pos[rng.random(T) < 0.1] = -1
    x = rng.standard_normal((2, T, Hkv, D)).astype(np.float32)
    codes, sc = np.zeros((2, pool, Hkv, 16, D), np.uint8), np.zeros((2, pool, Hkv), np.float32)
    dev = _block_device(codes, sc)
    k, v = (torch.from_numpy(a).bfloat16().cuda() for a in x)
    s, p = torch.from_numpy(slots).cuda(), torch.from_numpy(pos).cuda()
    want = slots.copy()
    if op == "append":
        ops.reshape_and_cache_fp8_block(k, v, *dev, s)
    else:
        table = torch.cat([torch.ones(50, D // 2), torch.zeros(50, D // 2)], 1).cuda()  # angles of zero
        q = torch.zeros(T, 1, D, dtype=torch.bfloat16, device="cuda")
        ops.rope_and_cache_fp8_block(q, q, k, v, *dev, s, p, table)
        want[pos < 0] = -1
    for i, t in enumerate((k, v)):
        ref.append_block(t.double().cpu().numpy(), codes[i], sc[i], want)
    assert np.array_equal(dev[0].view(torch.uint8).cpu().numpy(), codes[0])
    assert np.array_equal(dev[1].view(torch.uint8).cpu().numpy(), codes[1])
    assert np.array_equal(dev[2].cpu().numpy(), sc[0]) and np.array_equal(dev[3].cpu().numpy(), sc[1])
    assert ops.device_errors(0) == 0
