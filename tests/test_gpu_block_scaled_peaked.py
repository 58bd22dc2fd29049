"""Decode attention over block-scaled e4m3 caches where one token takes most of
a row's weight: what is left for the others must not be lost.

Tolerance: a weight p of a tile of 128 tokens is two e4m3 terms (bf16) or three
(f16) of p / P, P the largest p vs / vs_p of the tile: off by at most 2^-8 p (2^-11
p) while a term is normal, and by half the last term's subnormal step below,
2^-22 P (2^-26 P).  So the mean of the values is off by at most
sum |v| (REL p + FLOOR P) / sum p; the scales of V are equal here.  REL has 1e-3
for the logits' error beside the weights' rounding.  The output's own rounding is
half a step more.
"""

import math

import numpy as np
import pytest

import rope_cache_reference as ref
from helpers import as_f64, half_ulp, to_dev, torch_dtype

pytestmark = pytest.mark.gpu

REL = {"bf16": 2.0 ** -8 + 1e-3, "f16": 2.0 ** -11 + 1e-3}
FLOOR = {"bf16": 2.0 ** -22, "f16": 2.0 ** -26}
TILE = 128


def _case(dtype, H, D, n, rest, at, spread, seed=0):
    """One row of n tokens and one KV head.  Token `at` has the whole weight but
    `rest`, and a value row of zeros; the others' values have one sign a column,
    so what is lost of their weight is lost of the output."""
    import torch

    rng = np.random.default_rng(seed)
    nblk = (n + 15) // 16
    pool = nblk + 2
    table = rng.permutation(pool)[:nblk].astype(np.int32)
    u = rng.choice([-1.0, 1.0], D)
    q = as_f64(torch.from_numpy(rng.standard_normal((1, H, D)) * 0.1 + u).to(torch_dtype(dtype)))
    codes = ref.to_e4m3(rng.standard_normal(1 << 16) * 96)
    kc, vc = (codes[rng.integers(0, codes.size, (pool, 1, 16, D))] for _ in range(2))
    vc = (vc & 0x7F) | rng.choice([0, 0x80], D).astype(np.uint8)
    ks = np.full((pool, 1), spread / 96, np.float32)
    vs = np.full((pool, 1), 2.0 ** -7, np.float32)
    b, o = table[at // 16], at % 16
    kc[b] = 0
    kc[b, 0, o] = ref.to_e4m3(96 * u)
    vc[b, 0, o] = 0
    # its block's scale puts it where, of the least favoured head, all but `rest` is its own
    scale = 1 / math.sqrt(D)
    keys = (ref.from_e4m3(kc[table]) * ks[table][..., None, None].astype(np.float64)).reshape(-1, D)[:n]
    lg = np.einsum("hd,td->ht", q[0], keys) * scale
    lg[:, at] = -np.inf
    top = lg.max(-1)
    tail = np.log(np.exp(lg - top[:, None]).sum(-1)) + top
    need = (tail + math.log((1 - rest) / rest)).max()
    ks[b] = need / ((q[0] @ (ref.from_e4m3(kc[b, 0, o]))).min() * scale)
    return q, kc, vc, ks, vs, table[None], np.array([n], np.int32)


def _run(dtype, case, workspace):
    import torch

    from cacheflow_b200 import ops

    q, kc, vc, ks, vs, tables, lens = case
    t = [torch.from_numpy(np.ascontiguousarray(c)).cuda().view(torch.float8_e4m3fn) for c in (kc, vc)]
    dq = torch.from_numpy(q).to(torch_dtype(dtype)).cuda()
    rest = [to_dev(x) for x in (ks, vs, tables, lens)]
    out, ws = torch.full_like(dq, 7.0), None
    if workspace:
        n = ops.paged_attention_fp8_block_workspace_size(dq, t[0], rest[2], int(lens.max()))
        ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    ops.paged_attention_fp8_block_v1(out, dq, *t, *rest, None, int(lens.max()), workspace=ws)
    torch.cuda.synchronize()
    return as_f64(out)


def _check(dtype, case, got):
    q, kc, vc, ks, vs, tables, lens = case
    n, D = int(lens[0]), q.shape[-1]
    keys = (ref.from_e4m3(kc[tables[0]]) * ks[tables[0]][..., None, None].astype(np.float64)).reshape(-1, D)[:n]
    vals = (ref.from_e4m3(vc[tables[0]]) * vs[tables[0]][..., None, None].astype(np.float64)).reshape(-1, D)[:n]
    lg = np.einsum("hd,td->ht", q[0], keys) / math.sqrt(D)
    p = np.exp(lg - lg.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    want = p @ vals
    pad = np.zeros((p.shape[0], -n % TILE))
    tops = np.concatenate([p, pad], 1).reshape(p.shape[0], -1, TILE).max(-1).repeat(TILE, 1)[:, :n]
    lim = (REL[dtype] * p + FLOOR[dtype] * tops) @ np.abs(vals)
    lim += half_ulp(np.abs(want) + lim, dtype) + 2.0 ** -24
    err = np.abs(got[0] - want)
    assert (err <= lim).all(), f"{(err / lim).max():.2f} of the bound; off by {np.linalg.norm(err) / np.linalg.norm(want):.4f}"


def _both(dtype, case):
    """With the context shared among CTAs, and whole."""
    for workspace in (True, False):
        _check(dtype, case, _run(dtype, case, workspace))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("H,D,n,rest", [
    (1, 128, 131072, 0.01), (8, 128, 131072, 0.01), (8, 128, 131072, 0.1), (4, 128, 32768, 0.01),
    (12, 128, 32768, 0.01), (8, 256, 32768, 0.01), (1, 256, 131072, 0.02),
])
def test_what_one_token_leaves(cflib, dtype, H, D, n, rest):
    _both(dtype, _case(dtype, H, D, n, rest, at=5, spread=0.8, seed=H + D))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("at", [0, 127, 128, 20000, 39998])
def test_wherever_the_token_is(cflib, dtype, at):
    """First, last, in the middle: the maximum is there from the start, moves at the end, or moves once."""
    _both(dtype, _case(dtype, 8, 128, 39999, 0.002, at, spread=0.3, seed=at))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [2, 16, 127, 129, 1000])
def test_short_rows(cflib, dtype, n):
    """In the token's own tile the rest stands on FLOOR of its weight."""
    case = _case(dtype, 8, 128, n, 2.0 ** -14, n // 2, spread=0.5)
    _both(dtype, case)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_tiles_far_apart(cflib, dtype):
    """Tiles whose best tokens are up to 60 binades apart, in rising, falling and mixed order."""
    rng = np.random.default_rng(3)
    for order in ("up", "down", "mixed"):
        n = 20 * TILE - 7
        case = _case(dtype, 4, 128, n, 0.5, 3, spread=0.2, seed=4)
        q, kc, vc, ks, vs, tables, lens = case
        step = {"up": np.arange(20), "down": np.arange(20)[::-1], "mixed": rng.permutation(20)}[order]
        kc[...] = ref.to_e4m3(96 * np.sign(q[0, 0]))   # every key along the queries: its scale is its logit
        for i in range(tables.shape[1]):
            ks[tables[0, i]] = 0.002 * step[i // 8] * (1 + 0.01 * (i % 8))
        _both(dtype, case)
