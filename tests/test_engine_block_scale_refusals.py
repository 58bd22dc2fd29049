"""What DecodeEngine refuses of block-scaled caches, before any buffer is made
(on the CPU: a refused engine touches no device)."""

import pytest
import torch


def _caches(blocks=4, heads=2, block=16, dim=128):
    return [torch.zeros(blocks, heads, block, dim, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]


def _engine(caches, scales, query_dtype=torch.bfloat16, **kw):
    from cacheflow_b200.engine import DecodeEngine

    return DecodeEngine(*caches, 4, 2, 4, kv_scales=scales, query_dtype=query_dtype, **kw)


def _scales(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("dim", [64, 80, 112])
def test_heads_that_the_attention_does_not_take(cflib, dim):
    """The append takes them: without the refusal a step would append and then fail."""
    with pytest.raises(ValueError, match="head_dim"):
        _engine(_caches(dim=dim), _scales(4, 2))


def test_blocks_and_query_types(cflib):
    with pytest.raises(ValueError, match="16 tokens"):
        _engine(_caches(block=8), _scales(4, 2))
    for dt in (torch.float32, None):
        with pytest.raises(ValueError, match="query_dtype"):
            _engine(_caches(), _scales(4, 2), query_dtype=dt)


@pytest.mark.parametrize("scales", [
    _scales(4, 3), _scales(5, 2), _scales(4, 2, 1), _scales(8), _scales(4, 2, dtype=torch.float64),
    (torch.zeros(4, 2), 0.5), (0.5, torch.zeros(4, 2)), (torch.zeros(4, 2), torch.tensor(0.5)),
    (torch.zeros(2, 4).t(), torch.zeros(4, 2)), (torch.zeros(4, 2),), (torch.zeros(4, 2),) * 3,
])
def test_scales_that_do_not_fit_the_caches(cflib, scales):
    with pytest.raises(ValueError, match="block scales"):
        _engine(_caches(), scales)


def test_one_number_is_a_caches_scale(cflib):
    """Also as [[x]], as float() takes it; with a pool of one block and head it is that block's."""
    from cacheflow_b200.engine import _block_scales

    pool, one = _caches()[0], _caches(1, 1)[0]
    for x in (0.5, torch.tensor(0.5), torch.tensor([0.5]), torch.tensor([[0.5]])):
        assert not _block_scales(x, pool)
    assert _block_scales(torch.zeros(4, 2), pool) and _block_scales(torch.zeros(1, 1), one)
    assert not _block_scales(torch.zeros(1), one)
