"""Decode attention over e4m3 caches with a scale for each block and KV head
(cf_paged_attention_fp8_block_v1) against its definition in float64.

Tolerance: the queries are e4m3 terms that hold a bf16 exactly and an f16 to
2^-12, the weights two terms (bf16 outputs) or three (f16): |p' - p| <= 2^-8 p
or 2^-11 p at most (an f16 rounding included), so a weighted mean of values v
is off by at most that times the mean of |v|.  Logits are off by at most 2^-18
of the sum of |q k| per 32 products, below 1e-3 for every case here, which
moves a weight by as much.  The output's own rounding is half a step more.
"""

import math

import numpy as np
import pytest

import rope_cache_reference as ref
from cacheflow_b200.workloads import host_values
from helpers import as_f64, half_ulp, random_tables, to_dev, torch_dtype

pytestmark = pytest.mark.gpu

REL = {"bf16": 2.0 ** -8 + 1e-3, "f16": 2.0 ** -11 + 1e-3}


def _codes(rng, shape, spread=96.0):
    return ref.to_e4m3(rng.standard_normal(shape) * spread)


def _fp8(codes):
    import torch

    return torch.from_numpy(np.ascontiguousarray(codes)).cuda().view(torch.float8_e4m3fn)


def _f64(a, dtype):
    return as_f64(to_dev(a, dtype))


def _case(dtype, H, Hkv, D, ctx, seed=0, lo=-10, hi=-5, q_std=1.0, spare=3):
    rng = np.random.default_rng(seed)
    pool = sum((c + 15) // 16 for c in ctx) + spare
    tables = random_tables(rng, ctx, pool)
    q = host_values((len(ctx), H, D), dtype, q_std, rng)
    kc, vc = _codes(rng, (pool, Hkv, 16, D)), _codes(rng, (pool, Hkv, 16, D))
    ks = np.exp2(rng.integers(lo, hi, (pool, Hkv))).astype(np.float32)
    vs = np.exp2(rng.integers(lo, hi, (pool, Hkv))).astype(np.float32)
    return q, kc, vc, ks, vs, tables, np.array(ctx, np.int32)


def _mean_abs_v(q, kc, vc, ks, vs, tables, lens, scale):
    """sum p |v|: what a relative error of the weights can move."""
    return ref.attention(q, kc, vc & 0x7F, ks, vs, tables, lens, scale)


def _run(dtype, case, workspace="own", max_context_len=None, scale=None, out=None):
    import torch

    from cacheflow_b200 import ops

    q, kc, vc, ks, vs, tables, lens = case
    dq = to_dev(q, dtype)
    args = (dq, _fp8(kc), _fp8(vc), to_dev(ks), to_dev(vs), to_dev(tables), to_dev(lens))
    m = int(lens.max()) if max_context_len is None else max_context_len
    out = torch.full_like(dq, 7.0) if out is None else out
    ws = None
    if workspace == "own":
        n = ops.paged_attention_fp8_block_workspace_size(dq, args[1], args[5], m)
        ws = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device="cuda")
    ops.paged_attention_fp8_block_v1(out, *args, scale, m, workspace=ws)
    torch.cuda.synchronize()
    return out


def _check(dtype, case, got, scale=None):
    q, *rest = case
    q = _f64(q, dtype)
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    want = ref.attention(q, *rest, scale)
    lim = REL[dtype] * _mean_abs_v(q, *rest, scale) + half_ulp(want, dtype) + 2.0 ** -24
    got = as_f64(got)
    if dtype == "f16":  # a mean of 65520 or more rounds to infinity in f16
        past = np.abs(want) + lim >= 65520
        assert (np.sign(got[past]) == np.sign(want[past])).all()
        surely = np.abs(want) - lim >= 65520
        assert np.isinf(got[surely]).all()
        got = np.where(past, want, got)
    err = np.abs(got - want)
    assert (err <= lim).all(), f"worst {np.nanmax(err - lim):.3e} over, max err {np.nanmax(err):.3e}"
    # and on the whole no further off than a weight's and the output's roundings
    if np.linalg.norm(want) > 0:
        rel = np.linalg.norm(err) / np.linalg.norm(want)
        assert rel < {"bf16": 3e-3, "f16": 5e-4}[dtype], rel


EDGES = [0, 1, 15, 16, 17, 127, 128, 129, 255, 300, 0, 1000]


@pytest.mark.parametrize("workspace", ["own", None])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("H,Hkv,D", [
    (1, 1, 128), (2, 2, 256), (4, 2, 128), (3, 1, 128), (8, 2, 256), (5, 1, 128), (16, 2, 128), (7, 1, 256),
    (9, 1, 128), (32, 2, 128), (16, 1, 256), (20, 1, 128), (33, 1, 256),
])
def test_matches_definition(cflib, dtype, H, Hkv, D, workspace):
    from cacheflow_b200 import ops

    case = _case(dtype, H, Hkv, D, EDGES, seed=H + D)
    got = _run(dtype, case, workspace)
    _check(dtype, case, got)
    assert ops.device_errors(0) == 0


@pytest.mark.parametrize("dtype,H,Hkv,D,ctx", [
    ("bf16", 32, 8, 128, [9001]),
    ("bf16", 8, 1, 128, [20000, 3, 129]),
    ("f16", 8, 8, 128, [5000, 1, 4097, 0, 640]),
    ("f16", 16, 2, 256, [3001, 1300]),
    ("bf16", 16, 1, 128, [6000, 128]),
    ("bf16", 64, 8, 128, [600, 20, 4000, 1111] * 3),
])
def test_long_contexts_are_shared_and_joined(cflib, dtype, H, Hkv, D, ctx):
    case = _case(dtype, H, Hkv, D, ctx, seed=3)
    shared = _run(dtype, case, "own")
    _check(dtype, case, shared)
    _check(dtype, case, _run(dtype, case, None))


def test_many_short_rows(cflib):
    # more items than CTAs, most of one tile
    rng = np.random.default_rng(8)
    ctx = rng.integers(0, 200, 700).tolist()
    case = _case("bf16", 8, 2, 128, ctx, seed=9)
    got = _run("bf16", case, "own")
    _check("bf16", case, got)
    _check("bf16", case, _run("bf16", case, None))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_scales_far_apart(cflib, dtype):
    """Values in blocks whose scales differ by powers of 2^40, whatever block the
    weights favour; scales that are no powers of two; blocks of scale 0."""
    case = _case(dtype, 8, 2, 128, [400, 90, 33], seed=4)
    q, kc, vc, ks, vs, tables, lens = case
    rng = np.random.default_rng(1)
    vs[:] = np.exp2(rng.integers(-20, 20, vs.shape)).astype(np.float32)
    vs[::3] *= np.float32(1.37)
    ks[::4] *= np.float32(0.71)
    ks[1::5] = 0.0
    vs[2::5] = 0.0
    _check(dtype, case, _run(dtype, case))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_scales_at_the_ends_of_their_range(cflib, dtype):
    """Rows that begin with blocks of the least scales (a block of f32's
    smallest values has 2^-126) and go on with ordinary ones; 2^60 beside 1."""
    case = _case(dtype, 8, 2, 128, [700, 300, 140], seed=14)
    q, kc, vc, ks, vs, tables, lens = case
    vs[tables[0, :16]] = 2.0 ** -126
    vs[tables[0, 20]] = 2.0 ** -75
    vs[tables[1, :19]] = 2.0 ** -60
    vs[tables[2, 3]] = 2.0 ** 60
    if dtype == "f16":
        vs[tables[2, 3]] = 2.0 ** 4  # (2^60 is infinity in f16)
    _check(dtype, case, _run(dtype, case))


def test_bytes_outside_the_context_do_not_matter(cflib):
    """NaN bytes and scales past each row's last token and in unused blocks."""
    case = _case("bf16", 8, 2, 128, [1, 15, 130, 257], seed=5, spare=4)
    q, kc, vc, ks, vs, tables, lens = case
    clean = _run("bf16", case)
    used = np.zeros(kc.shape[0], bool)
    for s, n in enumerate(lens):
        ids = tables[s, : (n + 15) // 16]
        used[ids] = True
        if n % 16:
            kc[ids[-1], :, n % 16:] = 0x7F
            vc[ids[-1], :, n % 16:] = 0xFF
    kc[~used] = 0x7F
    vc[~used] = 0x7F
    ks[~used] = np.nan
    vs[~used] = np.nan
    got = _run("bf16", case)
    assert np.array_equal(as_f64(got), as_f64(clean))


def test_nan_where_a_token_or_query_is_nan(cflib):
    case = _case("f16", 4, 2, 128, [70, 40], seed=6)
    q, kc, vc, ks, vs, tables, lens = case
    q[0, 1, 5] = np.nan        # head 1 of row 0
    vc[tables[1, 0], 1, 3, 9] = 0x7F  # row 1, KV head 1, dimension 9
    got = as_f64(_run("f16", case))
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[0, [0, 2, 3]]).all()
    assert np.isnan(got[1, 2:, 9]).all()
    assert np.isfinite(got[1, :2]).all() and np.isfinite(np.delete(got[1, 2:], 9, axis=-1)).all()


@pytest.mark.parametrize("dtype,value", [("f16", 65504.0), ("bf16", 1e30), ("f16", 0.0), ("bf16", 1e-30)])
def test_queries_of_any_size(cflib, dtype, value):
    import torch

    case = _case(dtype, 4, 1, 128, [50], seed=7)
    q = case[0]
    x = np.full(q.shape, value, np.float32)
    x[..., ::2] *= -1
    t = torch.from_numpy(x).to(torch_dtype(dtype))
    q[...] = t.view(torch.int16).numpy().view(q.dtype) if dtype == "bf16" else t.numpy()
    # keep the logits of an ordinary size
    scale = 0.05 / value if value else 0.05
    got = _run(dtype, case, scale=scale)
    _check(dtype, case, got, scale=scale)


def test_rejected_blocks_and_lengths(cflib):
    """A block id outside the pool is left out and recorded; a length past the
    table is cut and recorded; a negative one is an empty row."""
    from cacheflow_b200 import _lib, ops

    case = _case("bf16", 8, 2, 128, [200, 300, 64], seed=10)
    q, kc, vc, ks, vs, tables, lens = case
    t2 = tables.copy()
    t2[0, 3], t2[1, 0] = kc.shape[0], -5
    ops.device_errors(0)
    got = as_f64(_run("bf16", (q, kc, vc, ks, vs, t2, lens)))
    assert ops.device_errors(0) & _lib.CF_DEVERR_BLOCK_ID
    assert np.isfinite(got).all()
    # rows without a bad block are as ever; the others are the mean over their good tokens
    qf = _f64(q, "bf16")
    want = ref.attention(qf, kc, vc, ks, vs, tables, lens, 1 / math.sqrt(128))
    assert np.abs(got[2] - want[2]).max() < 0.05
    keep = np.r_[0:48, 64:200]
    k = (ref.from_e4m3(kc[tables[0, :13]]) * ks[tables[0, :13]][..., None, None]).transpose(1, 0, 2, 3)
    v = (ref.from_e4m3(vc[tables[0, :13]]) * vs[tables[0, :13]][..., None, None]).transpose(1, 0, 2, 3)
    k, v = k.reshape(2, -1, 128)[:, keep], v.reshape(2, -1, 128)[:, keep]
    lg = np.einsum("hgd,htd->hgt", qf[0].reshape(2, 4, 128), k) / math.sqrt(128)
    p = np.exp(lg - lg.max(-1, keepdims=True))
    w0 = (np.einsum("hgt,htd->hgd", p, v) / p.sum(-1, keepdims=True)).reshape(8, 128)
    assert np.abs(got[0] - w0).max() <= 0.02 * np.abs(w0).max() + 1e-3

    bad = lens.copy()
    bad[0], bad[2] = tables.shape[1] * 16 + 1, -1
    got = as_f64(_run("bf16", (q, kc, vc, ks, vs, np.maximum(tables, 0), bad), max_context_len=tables.shape[1] * 16))
    assert ops.device_errors(0) & _lib.CF_DEVERR_CONTEXT_LEN
    assert np.isfinite(got[0]).all() and (got[2] == 0).all()
    assert np.abs(got[1] - want[1]).max() < 0.05


def test_max_context_len_is_a_bound_only(cflib):
    """Results do not hang on max_context_len where it bounds the contexts."""
    case = _case("bf16", 8, 2, 128, [700, 3], seed=11)
    q, kc, vc, ks, vs, tables, lens = case
    wide = np.zeros((2, 4096), np.int32)
    wide[:, : tables.shape[1]] = tables
    _check("bf16", case, _run("bf16", (q, kc, vc, ks, vs, wide, lens), max_context_len=65536))


def test_captured_and_replayed_with_other_lengths(cflib):
    """A captured call, replayed after its lengths, queries and caches changed;
    two graphs with a workspace each on two streams."""
    import torch

    from cacheflow_b200 import ops

    cases = [_case("bf16", 16, 2, 128, [900, 40, 2000], seed=20 + i) for i in range(3)]
    pool = max(c[1].shape[0] for c in cases)
    graphs = []
    for i in range(2):
        q, kc, vc, ks, vs, tables, lens = cases[i]
        t = [to_dev(q, "bf16"), _fp8(kc), _fp8(vc), to_dev(ks), to_dev(vs), to_dev(tables), to_dev(lens)]
        out = torch.zeros_like(t[0])
        ws = torch.empty((ops.paged_attention_fp8_block_workspace_size(t[0], t[1], t[5], 2000),), dtype=torch.uint8,
                         device="cuda")
        ops.paged_attention_fp8_block_v1(out, *t, None, 2000, workspace=ws)  # first run outside the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_attention_fp8_block_v1(out, *t, None, 2000, workspace=ws)
        graphs.append((g, t, out, ws))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (g, *_), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        _check("bf16", cases[i], graphs[i][2])
    g, t, out, _ = graphs[0]
    q, kc, vc, ks, vs, tables, lens = cases[2]
    assert kc.shape[0] == t[1].shape[0] == pool
    lens = np.array([0, 31, 1999], np.int32)
    for dst, src in zip(t, (to_dev(q, "bf16"), _fp8(kc), _fp8(vc), to_dev(ks), to_dev(vs), to_dev(tables),
                            to_dev(lens))):
        dst.copy_(src)
    g.replay()
    torch.cuda.synchronize()
    _check("bf16", (q, kc, vc, ks, vs, tables, lens), out)


def test_same_answer_twice(cflib):
    """Bit-identical on the same inputs: nothing depends on the order of CTAs."""
    case = _case("bf16", 32, 4, 128, [3000, 17, 800, 5000], seed=12)
    a, b = _run("bf16", case), _run("bf16", case)
    assert np.array_equal(as_f64(a), as_f64(b))


@pytest.mark.parametrize("D", [128, 256])
def test_wait_runs_out_and_the_next_call_is_correct(cflib, D):
    """As the other decode kernels': no copy is issued for the first stage, so
    its wait ends with CF_DEVERR_TIMEOUT and nothing is written."""
    import time

    import torch

    from cacheflow_b200 import _lib, ops

    case = _case("bf16", 8, 2, D, [5], seed=13)
    ops.device_errors(0)
    sentinel = torch.full((1, 8, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = sentinel.clone()
    _run("bf16", case)  # loads the kernel
    assert cflib.cf_testing_set_pipeline_faults(1_000_000, 1) == _lib.CF_OK
    try:
        t0 = time.perf_counter()
        _run("bf16", case, out=out)
        elapsed = time.perf_counter() - t0
    finally:
        assert cflib.cf_testing_set_pipeline_faults(0, 0) == _lib.CF_OK
    assert ops.device_errors(0) & _lib.CF_DEVERR_TIMEOUT
    assert elapsed < 1.0 and torch.equal(out, sentinel)
    _check("bf16", case, _run("bf16", case))
    assert ops.device_errors(0) == 0
