"""DecodeEngine with a rotation and with block-scaled caches: steps from pinned
host buffers give what the same operators give in turn, and the definition's
answer; one new token a row for many steps, through block borders."""

import math

import numpy as np
import pytest

import rope_cache_reference as ref
from helpers import random_tables, torch_dtype

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("cache", ["same", "fp8", "block"])
def test_steps(cflib, dtype, cache):
    import torch

    from cacheflow_b200 import ops
    from cacheflow_b200.engine import DecodeEngine, Rotation

    rng = np.random.default_rng(21)
    S, H, Hkv, D, steps = 3, 8, 2, 128, 20
    dt = torch_dtype(dtype)
    tables = random_tables(rng, [steps + 200] * S, S * 16)
    pool = S * 16
    cdt = dt if cache == "same" else torch.float8_e4m3fn
    kc, vc = (torch.zeros((pool, Hkv, 16, D), dtype=torch.uint8, device="cuda") for _ in range(2))
    if cache == "same":
        kc, vc = (torch.zeros((pool, Hkv, 16, D), dtype=dt, device="cuda") for _ in range(2))
    else:
        kc, vc = kc.view(cdt), vc.view(cdt)
    scales = {"same": None, "fp8": (0.02, 0.02),
              "block": (torch.zeros(pool, Hkv, device="cuda"), torch.zeros(pool, Hkv, device="cuda"))}[cache]
    w = torch.from_numpy((1 + 0.2 * rng.standard_normal((2, D))).astype(np.float32)).cuda()
    rot = Rotation(ops.rope_table(512, D), w[0], w[1])
    eng = DecodeEngine(kc, vc, H, S, tables.shape[1], kv_scales=scales, query_dtype=dt, rotation=rot)
    first = np.array([0, 30, 190])  # rows at different positions, earlier tokens all zero
    # the same steps by the operators in turn
    kc2, vc2 = kc.clone(), vc.clone()
    sc2 = tuple(s.clone() for s in scales) if cache == "block" else scales
    keys, vals, outs = [], [], []
    pins = []
    for i in range(steps):
        pos = (first + i).astype(np.int32)
        q, k, v = (torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(dt)
                   for s in ((S, H, D), (S, Hkv, D), (S, Hkv, D)))
        slots = (tables[np.arange(S), pos // 16] * 16 + pos % 16).astype(np.int32)
        pin = [t.pin_memory() for t in (q, k, v)] + [torch.from_numpy(a).pin_memory() for a in (slots, tables, pos + 1)]
        o = torch.empty((S, H, D), dtype=dt).pin_memory()
        p = torch.from_numpy(pos).pin_memory()
        eng.step(*pin, o, int(pos.max()) + 1, positions_host=p)
        pins.append((pin, p))
        outs.append(o)
        qd, out = q.cuda(), torch.empty((S, H, D), dtype=dt, device="cuda")
        common = (torch.from_numpy(slots).cuda(), p.cuda(), rot.cos_sin)
        lens, bt = torch.from_numpy(pos + 1).cuda(), torch.from_numpy(tables).cuda()
        if cache == "same":
            ops.rope_and_cache(qd, qd, k.cuda(), v.cuda(), kc2, vc2, *common, w[0], w[1])
            ops.paged_attention_v1(out, qd, kc2, vc2, bt, lens, None, int(pos.max()) + 1)
        elif cache == "fp8":
            ops.rope_and_cache_fp8(qd, qd, k.cuda(), v.cuda(), kc2, vc2, *common, *sc2, w[0], w[1])
            ops.paged_attention_fp8_v1(out, qd, kc2, vc2, bt, lens, *sc2, None, int(pos.max()) + 1)
        else:
            ops.rope_and_cache_fp8_block(qd, qd, k.cuda(), v.cuda(), kc2, vc2, *sc2, *common, w[0], w[1])
            ops.paged_attention_fp8_block_v1(out, qd, kc2, vc2, *sc2, bt, lens, None, int(pos.max()) + 1,
                                             workspace=eng.workspace.clone() if eng.workspace is not None else None)
        eng.synchronize()
        tol = {"bf16": 2.0 ** -8, "f16": 2.0 ** -10}[dtype]
        # the same kernels on the same bytes; only where v1 splits a context differs
        assert (o.float() - out.float().cpu()).abs().max() <= tol * out.float().abs().max().cpu()
        keys.append(ref.norm_rope(k.double().numpy(), w[1].double().cpu().numpy(), rot.cos_sin.cpu().numpy(), pos,
                                  False, rot.eps))
        vals.append(v.double().numpy())
    assert torch.equal(kc.view(torch.uint8), kc2.view(torch.uint8))
    assert torch.equal(vc.view(torch.uint8), vc2.view(torch.uint8))
    assert ops.device_errors(0) == 0
    # the last step's row 0: nothing before its first token
    qr = ref.norm_rope(q.double().numpy(), w[0].double().cpu().numpy(), rot.cos_sin.cpu().numpy(), pos, False, rot.eps)
    kk, vv = np.stack(keys, 1)[0], np.stack(vals, 1)[0]  # [steps, Hkv, D]
    lg = np.einsum("hgd,thd->hgt", qr[0].reshape(Hkv, H // Hkv, D), kk) / math.sqrt(D)
    pr = np.exp(lg - lg.max(-1, keepdims=True))
    want = (np.einsum("hgt,thd->hgd", pr, vv) / pr.sum(-1, keepdims=True)).reshape(H, D)
    got = outs[-1][0].double().numpy()
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < (0.01 if cache == "same" else 0.06)


def test_block_scaled_steps_without_a_rotation(cflib):
    import torch

    from cacheflow_b200 import ops
    from cacheflow_b200.engine import DecodeEngine

    rng = np.random.default_rng(5)
    S, H, Hkv, D = 4, 8, 4, 128
    ctx = np.array([1, 17, 600, 300], np.int32)
    pool = 80
    tables = random_tables(rng, ctx, pool)
    codes = ref.to_e4m3(rng.standard_normal((2, pool, Hkv, 16, D)) * 96)
    sc = np.exp2(rng.integers(-9, -4, (2, pool, Hkv))).astype(np.float32)
    kc, vc = (torch.from_numpy(c).cuda().view(torch.float8_e4m3fn) for c in codes.copy())
    ks, vs = (torch.from_numpy(s.copy()).cuda() for s in sc)
    eng = DecodeEngine(kc, vc, H, S, tables.shape[1], kv_scales=(ks, vs), query_dtype=torch.bfloat16)
    q, k, v = (torch.from_numpy(rng.standard_normal(s).astype(np.float32)).bfloat16()
               for s in ((S, H, D), (S, Hkv, D), (S, Hkv, D)))
    pos = ctx - 1
    slots = (tables[np.arange(S), pos // 16] * 16 + pos % 16).astype(np.int32)
    pin = [t.pin_memory() for t in (q, k, v)] + [torch.from_numpy(a).pin_memory() for a in (slots, tables, ctx)]
    out = torch.empty((S, H, D), dtype=torch.bfloat16).pin_memory()
    eng.step(*pin, out, 600)
    eng.synchronize()
    ref.append_block(k.double().numpy(), codes[0], sc[0], slots)
    ref.append_block(v.double().numpy(), codes[1], sc[1], slots)
    assert np.array_equal(ks.cpu().numpy(), sc[0]) and np.array_equal(vs.cpu().numpy(), sc[1])
    want = ref.attention(q.double().numpy(), codes[0], codes[1], sc[0], sc[1], tables, ctx, 1 / math.sqrt(D))
    got = out.double().numpy()
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < 3e-3
    assert ops.device_errors(0) == 0


def test_refusals(cflib):
    import torch

    from cacheflow_b200 import ops
    from cacheflow_b200.engine import DecodeEngine, Rotation

    c8 = torch.zeros(4, 2, 16, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    c16 = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16, device="cuda")
    sc = torch.zeros(4, 2, device="cuda")
    rot = Rotation(ops.rope_table(64, 128))
    with pytest.raises(ValueError):
        DecodeEngine(c8, c8.clone(), 4, 2, 4, kv_scales=(sc, sc), query_dtype=torch.bfloat16, fused_append=True)
    with pytest.raises(ValueError):
        DecodeEngine(c8, c8.clone(), 4, 2, 4, kv_scales=(sc, sc), query_dtype=torch.bfloat16, kernel="reference")
    with pytest.raises(ValueError):
        DecodeEngine(c16, c16.clone(), 4, 2, 4, kv_scales=(sc, sc))
    with pytest.raises(ValueError):
        DecodeEngine(c16, c16.clone(), 4, 2, 4, rotation=rot, fused_append=True)
    eng = DecodeEngine(c16, c16.clone(), 4, 2, 4, rotation=rot)
    q, k = torch.zeros(2, 4, 128, dtype=torch.bfloat16), torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        eng.step(q, k, k, i, torch.zeros(2, 4, dtype=torch.int32), i, q.clone(), 1)  # no positions
    with pytest.raises(ValueError):
        eng.attend(2, 1)
    e8 = DecodeEngine(c8, c8.clone(), 4, 2, 4, kv_scales=(sc, sc), query_dtype=torch.bfloat16)
    with pytest.raises(ops.CacheFlowError):  # prefill chunks take 16-bit caches
        e8.step(q, k, k, i, torch.zeros(2, 4, dtype=torch.int32), i, q.clone(), 1, chunks_host=(1, i, i[:1], i[None]))


def test_refused_chunks_leave_the_cache_alone(cflib):
    """Chunks over an 8-bit cache are refused before anything is rotated or appended; a step that has none is not."""
    import torch

    from cacheflow_b200 import ops
    from cacheflow_b200.engine import DecodeEngine, Rotation

    rng = np.random.default_rng(8)
    c8 = torch.zeros(2, 4, 2, 16, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    sc = torch.zeros(2, 4, 2, device="cuda")
    eng = DecodeEngine(c8[0], c8[1], 4, 2, 4, kv_scales=(sc[0], sc[1]), query_dtype=torch.bfloat16,
                       rotation=Rotation(ops.rope_table(64, 128)), max_chunks=1)
    q, k, v = (torch.from_numpy(rng.standard_normal(s).astype(np.float32)).bfloat16().pin_memory()
               for s in ((2, 4, 128), (2, 2, 128), (2, 2, 128)))
    slots, pos, ctx, start = (torch.tensor(x, dtype=torch.int32).pin_memory() for x in ([0, 16], [0, 0], [1, 1], [0, 0]))
    tables = torch.tensor([[0, 0, 0, 0], [1, 0, 0, 0]], dtype=torch.int32).pin_memory()
    new = (k.cuda(), v.cuda(), slots.cuda())
    eng.q.copy_(q)
    with pytest.raises(ops.CacheFlowError):
        eng.attend(2, 1, chunks=(1, 1, 1), new=new, positions=pos.cuda())
    torch.cuda.synchronize()
    assert torch.equal(eng.q.cpu(), q) and not c8.view(torch.uint8).any() and not sc.any()
    out = torch.zeros(2, 4, 128, dtype=torch.bfloat16).pin_memory()
    # no chunk: both rows decode; at position 0 a row's output is its own V
    eng.step(q, k, v, slots, tables, ctx, out, 1, chunks_host=(2, start[:1], ctx[:0], tables[:0]),
             positions_host=pos)
    eng.synchronize()
    want = v.double().repeat_interleave(2, 1)
    assert (out.double() - want).abs().max() <= 2.0 ** -4 * (1 + 2.0 ** -7) * want.abs().max()
    assert sc.all(2)[:, :2].all() and ops.device_errors(0) == 0


def test_rotation_with_prefill_chunks(cflib):
    """A decode row and a chunk of a prompt in one step: as rope_and_cache and the two attentions in turn."""
    import torch

    from cacheflow_b200 import ops
    from cacheflow_b200.engine import DecodeEngine, Rotation

    rng = np.random.default_rng(4)
    H, Hkv, D, n = 8, 2, 128, 21
    S = n + 1
    kc, vc = (torch.zeros(8, Hkv, 16, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k2, v2 = kc.clone(), vc.clone()
    rot = Rotation(ops.rope_table(64, D))
    eng = DecodeEngine(kc, vc, H, S, 2, rotation=rot, max_chunks=1)
    q, k, v = (torch.from_numpy(rng.standard_normal(s).astype(np.float32)).bfloat16().pin_memory()
               for s in ((S, H, D), (S, Hkv, D), (S, Hkv, D)))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).pin_memory()  # noqa: E731
    tables = i32([[5, 0]] + [[2, 7]] * n)
    pos = i32([0] + list(range(n)))
    slots = i32([80] + [(2, 7)[p // 16] * 16 + p % 16 for p in range(n)])
    out = torch.empty(S, H, D, dtype=torch.bfloat16).pin_memory()
    chunk = (1, i32([0, n]), i32([n]), tables[1:2])
    eng.step(q, k, v, slots, tables, pos + 1, out, n, chunks_host=chunk, positions_host=pos)
    eng.synchronize()
    qd, want = q.cuda(), torch.empty(S, H, D, dtype=torch.bfloat16, device="cuda")
    ops.rope_and_cache(qd, qd, k.cuda(), v.cuda(), k2, v2, slots.cuda(), pos.cuda(), rot.cos_sin)
    ops.paged_attention_v1(want[:1], qd[:1], k2, v2, tables[:1].cuda(), i32([1]).cuda(), None, 1)
    ops.paged_prefill_attention(want[1:], qd[1:], k2, v2, tables[1:2].cuda(), i32([n]).cuda(), i32([0, n]).cuda(),
                                None, n)
    assert torch.equal(kc, k2) and torch.equal(vc, v2)
    # the decode row attends to itself alone and the chunk's launch is the same one
    assert torch.equal(out, want.cpu())
    assert ops.device_errors(0) == 0


def test_scales_given_as_scalar_tensors(cflib):
    """A scale for a whole cache may still be a tensor of one number."""
    import torch

    from cacheflow_b200.engine import DecodeEngine

    outs = []
    for scales in ((0.5, 0.25), (torch.tensor(0.5), torch.tensor([0.25]))):
        c8 = torch.zeros(2, 4, 2, 16, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        eng = DecodeEngine(c8[0], c8[1], 4, 2, 4, kv_scales=scales, query_dtype=torch.bfloat16)
        g = torch.Generator().manual_seed(3)
        q, k, v = (torch.randn(s, generator=g).bfloat16().pin_memory() for s in ((1, 4, 128), (1, 2, 128), (1, 2, 128)))
        one = torch.ones(1, dtype=torch.int32).pin_memory()
        out = torch.empty(1, 4, 128, dtype=torch.bfloat16).pin_memory()
        eng.step(q, k, v, one * 0, one[:, None] * 0, one, out, 1)
        eng.synchronize()
        outs.append(out)
    assert torch.equal(*outs) and outs[0].any()
