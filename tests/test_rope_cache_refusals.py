"""Refusals of the norm / rotation, block-scaled append and block-scaled
attention entry points, and the append's definition in the tests against
itself.  No compute call: there may be no GPU."""

import ctypes

import numpy as np
import pytest

import rope_cache_reference as ref


def _rope(_lib, **over):
    p = _lib.RopeParams()
    p.query = p.key = p.value = p.query_out = p.key_out = p.positions = p.cos_sin = 0x1000
    for s in ("query", "key", "value", "query_out", "key_out"):
        getattr(p, s + "_stride")[:] = (512, 128)
    p.num_tokens, p.num_heads, p.num_kv_heads, p.head_dim, p.rotary_dim, p.max_positions = 4, 4, 2, 128, 128, 64
    p.eps, p.interleaved, p.dtype, p.weight_dtype = 1e-6, 0, _lib.CF_BF16, _lib.CF_BF16
    for k, v in over.items():
        if k.endswith("_stride"):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return p


BAD, UNS = 1, 2  # CF_ERR_INVALID_ARGUMENT, CF_ERR_UNSUPPORTED


@pytest.mark.parametrize("over,status", [
    ({"query": None}, BAD), ({"key": None}, BAD), ({"key_out": None}, BAD), ({"query_out": None}, BAD),
    ({"positions": None}, BAD), ({"cos_sin": None}, BAD), ({"query": 0x1001}, BAD), ({"cos_sin": 0x1002}, BAD),
    ({"num_tokens": -1}, BAD), ({"num_heads": 0}, BAD), ({"num_kv_heads": 0}, BAD), ({"head_dim": 0}, BAD),
    ({"rotary_dim": 0}, BAD), ({"rotary_dim": 63}, BAD), ({"rotary_dim": 130}, BAD), ({"max_positions": 0}, BAD),
    ({"interleaved": 2}, BAD), ({"dtype": 3}, BAD), ({"dtype": 9}, BAD), ({"weight_dtype": 1}, BAD),
    ({"head_dim": 512, "rotary_dim": 128}, UNS), ({"head_dim": 65, "rotary_dim": 64}, UNS),
    ({"num_heads": 65535}, UNS),
    ({"query_weight": 0x1000, "eps": 0.0}, BAD), ({"key_weight": 0x1000, "eps": float("nan")}, BAD),
    ({"query_weight": 0x1001}, BAD),
    ({"query_out_stride": (0, 128)}, BAD), ({"query_out_stride": (512, 0)}, BAD), ({"key_out_stride": (64, 128)}, BAD),
])
def test_rope_refusals(cflib, over, status):
    from cacheflow_b200 import _lib

    assert cflib.cf_qk_norm_rope(ctypes.byref(_rope(_lib, **over)), None) == status
    assert cflib.cf_qk_norm_rope(None, None) == BAD


@pytest.mark.parametrize("stride,tokens,ok", [
    ((128, 128), 4, False),    # a token's second head is the next token's first
    ((256, 128), 4, False), ((511, 128), 4, False), ((512, 128), 4, True), ((-512, 128), 4, True),
    ((512, -128), 4, True), ((128, 512), 4, True), ((128, 500), 4, False),  # heads outermost
    ((0, 128), 1, True), ((128, 0), 1, False), ((2 ** 63 - 1, 128), 4, True), ((-2 ** 63, 128), 4, True),
])
def test_output_rows_that_meet_are_refused(cflib, stride, tokens, ok):
    """Four heads of 128 columns.  What passes gets as far as the missing GPU."""
    import torch

    from cacheflow_b200 import _lib

    if ok and torch.cuda.is_available():
        pytest.skip("would launch")
    st = cflib.cf_qk_norm_rope(ctypes.byref(_rope(_lib, query_out_stride=stride, num_tokens=tokens)), None)
    assert (st != BAD) if ok else (st == BAD)


def test_empty_calls_do_nothing(cflib):
    from cacheflow_b200 import _lib

    p = _rope(_lib, num_tokens=0, query=None, key=None)
    assert cflib.cf_qk_norm_rope(ctypes.byref(p), None) == 0
    assert cflib.cf_rope_and_cache(ctypes.byref(p), None, None, None, 16, 4, None) == 0
    assert cflib.cf_rope_and_cache_fp8(ctypes.byref(p), None, None, None, 16, 4, 1.0, 1.0, None) == 0
    assert cflib.cf_rope_and_cache_fp8_block(ctypes.byref(p), None, None, None, None, None, 16, 4, None) == 0
    assert cflib.cf_reshape_and_cache_fp8_block(None, None, None, None, None, None, None, 0, 2, 128, 256, 256, 16,
                                                4, _lib.CF_BF16, None) == 0


def test_append_refusals(cflib):
    from cacheflow_b200 import _lib

    p, A = _rope(_lib), 0x1000
    q = ctypes.byref(p)
    assert cflib.cf_rope_and_cache(q, None, A, A, 16, 4, None) == BAD
    assert cflib.cf_rope_and_cache(q, A, A, None, 16, 4, None) == BAD
    assert cflib.cf_rope_and_cache(q, A, A, A, 0, 4, None) == BAD
    assert cflib.cf_rope_and_cache(q, A, A, A, 16, 0, None) == BAD  # the pool's size is needed
    assert cflib.cf_rope_and_cache(q, A + 1, A, A, 16, 4, None) == BAD
    assert cflib.cf_rope_and_cache(ctypes.byref(_rope(_lib, value=None)), A, A, A, 16, 4, None) == BAD
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert cflib.cf_rope_and_cache_fp8(q, A, A, A, 16, 4, scale, 1.0, None) == BAD
    assert cflib.cf_rope_and_cache_fp8(q, A + 8, A, A, 16, 4, 1.0, 1.0, None) == BAD
    assert cflib.cf_rope_and_cache_fp8(ctypes.byref(_rope(_lib, head_dim=72, rotary_dim=72)), A, A, A, 16, 4, 1.0, 1.0,
                                       None) == UNS
    blk = cflib.cf_rope_and_cache_fp8_block
    assert blk(q, A, A, None, A, A, 16, 4, None) == BAD
    assert blk(q, A, A, A, A, A, 8, 4, None) == UNS   # blocks of 16 tokens
    assert blk(q, A, A, A, A, A, 16, 0, None) == BAD
    assert blk(q, A, A, A, A, A, 16, 1 << 40, None) == UNS
    assert blk(ctypes.byref(_rope(_lib, head_dim=72, rotary_dim=72)), A, A, A, A, A, 16, 4, None) == UNS
    rc = cflib.cf_reshape_and_cache_fp8_block
    assert rc(A, None, A, A, A, A, A, 4, 2, 128, 256, 256, 16, 4, _lib.CF_BF16, None) == BAD
    assert rc(A, A, A, A, A, A, A, 4, 2, 128, 256, 256, 16, 4, _lib.CF_FP8_E4M3, None) == BAD
    assert rc(A + 1, A, A, A, A, A, A, 4, 2, 128, 256, 256, 16, 4, _lib.CF_BF16, None) == BAD
    assert rc(A, A, A, A, A, A, A, 4, 2, 272, 544, 544, 16, 4, _lib.CF_BF16, None) == UNS
    assert rc(A, A, A, A, A, A, A, -1, 2, 128, 256, 256, 16, 4, _lib.CF_BF16, None) == BAD


def test_block_scaled_attention_refusals(cflib):
    from cacheflow_b200 import _lib

    def params(**over):
        p = _lib.AttentionParams()
        p.query = p.key_cache = p.value_cache = p.output = p.block_tables = p.context_lens = 0x1000
        p.scale, p.num_seqs, p.num_heads, p.num_kv_heads, p.head_dim, p.block_size = 0.1, 2, 8, 2, 128, 16
        p.max_context_len, p.max_blocks_per_seq, p.num_blocks, p.dtype = 4096, 256, 600, _lib.CF_BF16
        for k, v in over.items():
            setattr(p, k, v)
        return ctypes.byref(p)

    f, A = cflib.cf_paged_attention_fp8_block_v1, 0x1000
    assert f(None, A, A, None, 0, None) == BAD
    assert f(params(), None, A, None, 0, None) == BAD
    assert f(params(), A, None, None, 0, None) == BAD
    assert f(params(num_blocks=0), A, A, None, 0, None) == BAD
    assert f(params(dtype=_lib.CF_F32), A, A, None, 0, None) == UNS
    assert f(params(head_dim=64), A, A, None, 0, None) == UNS
    assert f(params(block_size=32), A, A, None, 0, None) == UNS
    assert f(params(num_heads=7), A, A, None, 0, None) == BAD
    assert f(params(query=None), A, A, None, 0, None) == BAD
    assert f(params(key_cache=0x1008), A, A, None, 0, None) == BAD
    assert f(params(max_context_len=4097), A, A, None, 0, None) == BAD
    assert f(params(num_blocks=1 << 40), A, A, None, 0, None) == UNS
    assert f(params(), A, A, 0x1001, 1 << 20, None) == BAD  # workspace alignment
    assert f(params(num_seqs=0), A, A, None, 0, None) == 0
    size = cflib.cf_paged_attention_fp8_block_workspace_size
    assert size(params(query=None, output=None)) > 0
    assert size(params(max_context_len=128)) == 0 == size(params(num_seqs=0)) == size(params(head_dim=64))
    # one size does for every shorter context and any number of rows
    assert size(params(max_context_len=129)) == size(params()) == size(params(num_seqs=500))


def test_ops_refuse_before_the_library(cflib):
    import torch

    from cacheflow_b200 import ops

    x = torch.zeros(2, 4, 128)
    with pytest.raises(ops.CacheFlowError):
        ops.qk_norm_rope(x, x, x, x, torch.zeros(2, dtype=torch.int32), torch.zeros(8, 128))  # not on a GPU
    with pytest.raises(ops.CacheFlowError):
        ops.rope_table(16, 7)


def test_reference_e4m3():
    v = ref.e4m3_values()
    ok = ~np.isnan(v)
    assert np.array_equal(ref.from_e4m3(ref.to_e4m3(v[ok])), v[ok])
    pos = np.sort(v[ok & (v >= 0)])
    mid = (pos[1:] + pos[:-1]) / 2
    got = ref.to_e4m3(mid)
    assert (got % 2 == 0).all()  # ties to even
    assert ref.to_e4m3(np.array([1e9, -1e9, np.nan])).tolist() == [0x7E, 0xFE, 0x7F]
    assert ref.power_of_two(448.0) == 1.0 and ref.power_of_two(448.1) == 2.0 and ref.power_of_two(0.0) == 0.0
