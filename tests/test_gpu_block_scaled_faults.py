"""Decode attention over block-scaled caches when a pipeline wait runs out:
the call ends, says so, writes no row that it could not finish, and the next
call is correct.  The waits are made to run out by leaving a CTA's first copies
out (cf_testing_set_pipeline_faults), with a limit of 1 ms
(20 ms where the other CTAs go on)."""

import contextlib
import math
import time

import numpy as np
import pytest

import rope_cache_reference as ref
from cacheflow_b200.workloads import host_values
from helpers import as_f64, random_tables, to_dev

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def _faults(lib, cta=-1):
    from cacheflow_b200 import _lib

    assert lib.cf_testing_set_pipeline_fault_cta(cta) == _lib.CF_OK
    # where the other CTAs go on, their own waits must not run out
    assert lib.cf_testing_set_pipeline_faults(1_000_000 if cta < 0 else 20_000_000, 1) == _lib.CF_OK
    try:
        yield
    finally:
        assert lib.cf_testing_set_pipeline_faults(0, 0) == _lib.CF_OK
        assert lib.cf_testing_set_pipeline_fault_cta(-1) == _lib.CF_OK


def _case(dtype, H, Hkv, D, ctx, seed=0):
    rng = np.random.default_rng(seed)
    pool = sum((c + 15) // 16 for c in ctx) + 3
    tables = random_tables(rng, ctx, pool)
    q = host_values((len(ctx), H, D), dtype, 1.0, rng)
    codes = ref.to_e4m3(rng.standard_normal((2, pool, Hkv, 16, D)) * 96)
    sc = np.exp2(rng.integers(-10, -5, (2, pool, Hkv))).astype(np.float32)
    lens = np.array(ctx, np.int32)
    want = ref.attention(as_f64(to_dev(q, dtype)), *codes, *sc, tables, lens, 1 / math.sqrt(D))
    return [q, *codes, *sc, tables, lens], want


class _Call:
    """The operands of a call, its output and a workspace that holds `stale` bytes."""

    def __init__(self, dtype, case, workspace=True, stale=0x3F):
        import torch

        from cacheflow_b200 import ops

        q, kc, vc, ks, vs, tables, lens = case
        e4m3 = [torch.from_numpy(c).cuda().view(torch.float8_e4m3fn) for c in (kc, vc)]
        self.args = [to_dev(q, dtype), *e4m3, to_dev(ks), to_dev(vs), to_dev(tables), to_dev(lens)]
        self.longest = int(lens.max())
        n = ops.paged_attention_fp8_block_workspace_size(self.args[0], e4m3[0], self.args[5], self.longest)
        self.ws = torch.full((n,), stale, dtype=torch.uint8, device="cuda") if workspace and n else None

    def run(self):
        import torch

        from cacheflow_b200 import ops

        out = torch.full_like(self.args[0], 7.0)
        ops.paged_attention_fp8_block_v1(out, *self.args, None, self.longest, workspace=self.ws)
        torch.cuda.synchronize()
        return as_f64(out)


def _correct(got, want):
    return np.linalg.norm(got - want) <= 4e-3 * np.linalg.norm(want)


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("dtype,H,Hkv,D", [("bf16", 1, 1, 128), ("bf16", 8, 2, 128), ("f16", 8, 1, 128),
                                           ("bf16", 16, 1, 128), ("f16", 8, 1, 256)])
def test_every_cta_gives_up(cflib, dtype, H, Hkv, D, workspace):
    """Long rows in many CTAs, several items a CTA: each leaves after its first wait, nothing is written."""
    from cacheflow_b200 import _lib, ops

    case, want = _case(dtype, H, Hkv, D, [3000, 5, 700] + [129] * 300, seed=H + D)
    call = _Call(dtype, case, workspace)
    assert _correct(call.run(), want)
    ops.device_errors(0)
    for _ in range(5):
        with _faults(cflib):
            t0 = time.perf_counter()
            got = call.run()
            elapsed = time.perf_counter() - t0
        assert ops.device_errors(0) & _lib.CF_DEVERR_TIMEOUT
        assert (got == 7).all() and elapsed < 1.0
    assert _correct(call.run(), want)
    assert ops.device_errors(0) == 0


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("H", [1, 3, 8, 12])
def test_one_cta_gives_up(cflib, H, D):
    """One row's piece is not finished: that row (or the head chunk of it) is
    left unwritten whatever the workspace holds, the others are as ever.  With
    no more tiles than CTAs, CTA i has tile i of the rows laid end to end."""
    from cacheflow_b200 import _lib, ops

    chunks = (H + 7) // 8
    tiles = [4, 1, 20, 3]  # few pieces, one, many
    case, want = _case("bf16", H, 1, D, [128 * t - 5 for t in tiles], seed=H)
    stale = _Call("bf16", case)
    stale.run()  # leaves pieces of these sizes behind
    ops.device_errors(0)
    first = np.cumsum([0] + [t * chunks for t in tiles])
    for cta in (0, 1, 3, 4 * chunks, 5 * chunks, 5 * chunks + 7, 25 * chunks - 1, 28 * chunks - 1):
        for values in ("old", 0xFF, 0x3F):
            call = stale
            if values != "old":
                call = _Call("bf16", case, stale=values)
            with _faults(cflib, cta):
                got = call.run()
            assert ops.device_errors(0) & _lib.CF_DEVERR_TIMEOUT
            row = int(np.searchsorted(first, cta, side="right")) - 1
            chunk = (cta - first[row]) // tiles[row]
            lost = slice(8 * chunk, min(H, 8 * chunk + 8))
            assert (got[row, lost] == 7).all(), (cta, values)
            keep = np.ones(want.shape[:2], bool)
            keep[row, lost] = False
            assert _correct(got[keep], want[keep]), (cta, values)
    assert _correct(stale.run(), want)
    assert ops.device_errors(0) == 0


def test_hook_checks_its_argument(cflib):
    from cacheflow_b200 import _lib

    assert cflib.cf_testing_set_pipeline_fault_cta(-2) == _lib.CF_ERR_INVALID_ARGUMENT
    assert cflib.cf_testing_set_pipeline_fault_cta(-1) == _lib.CF_OK
