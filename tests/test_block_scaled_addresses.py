"""Addresses of the norm / rotation / append and block-scaled entry points that
a 4-byte load or store cannot use are refused on the host (on the device they
would fault).  No compute call."""

import ctypes

import pytest

from test_rope_cache_refusals import BAD, _rope

A = 0x1000


@pytest.mark.parametrize("odd", [A + 1, A + 2])
def test_slots_and_scales(cflib, odd):
    from cacheflow_b200 import _lib

    q = ctypes.byref(_rope(_lib))
    assert cflib.cf_rope_and_cache(q, A, A, odd, 16, 4, None) == BAD
    assert cflib.cf_rope_and_cache_fp8(q, A, A, odd, 16, 4, 1.0, 1.0, None) == BAD
    for i in range(3):
        ptr = [A, A, A]
        ptr[i] = odd
        assert cflib.cf_rope_and_cache_fp8_block(q, A, A, *ptr, 16, 4, None) == BAD
        assert cflib.cf_reshape_and_cache_fp8_block(A, A, A, A, *ptr, 4, 2, 128, 256, 256, 16, 4, _lib.CF_BF16,
                                                    None) == BAD


@pytest.mark.parametrize("odd", [A + 1, A + 2])
def test_attention(cflib, odd):
    from cacheflow_b200 import _lib

    def params(**over):
        p = _lib.AttentionParams()
        p.query = p.key_cache = p.value_cache = p.output = p.block_tables = p.context_lens = A
        p.scale, p.num_seqs, p.num_heads, p.num_kv_heads, p.head_dim, p.block_size = 0.1, 2, 8, 2, 128, 16
        p.max_context_len, p.max_blocks_per_seq, p.num_blocks, p.dtype = 4096, 256, 600, _lib.CF_BF16
        for k, v in over.items():
            setattr(p, k, v)
        return ctypes.byref(p)

    f = cflib.cf_paged_attention_fp8_block_v1
    assert f(params(), odd, A, None, 0, None) == BAD
    assert f(params(), A, odd, None, 0, None) == BAD
    assert f(params(block_tables=odd), A, A, None, 0, None) == BAD
    assert f(params(context_lens=odd), A, A, None, 0, None) == BAD
