"""The operators' cases: what is called, on which sizes, their plain forms and their definitions in 64 bits.

Operators, in the order in which a serving step uses them:

  qk_norm_rope      per-head RMS norms of queries and keys with the position rotation, one pass
  rope_and_cache    the same pass, with K (rotated) and V written to their slots of the paged cache:
                    caches of the inputs' type ("same"), e4m3 with one scale for each cache ("fp8") and
                    e4m3 with a scale for each block of 16 tokens and KV head ("block"); without
                    positions ("append") the block-scaled write alone
  attention         decode attention over e4m3 caches with a scale for each block and KV head

Sizes are those of the benchmark's batches (8, 32 or 64 query heads, head_dim 64 / 128 / 256, contexts
from one token to 128K) and odd ones around them.
"""

import math

import torch

own = False

BLOCK = 16
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _rope(name, tokens, heads, kv_heads, dim, dtype, rotary, op="qk", norm=True, interleaved=False, max_pos=32768,
          mode="prefill", chunk=512, pads=0):
    c = {"op": op, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
         "rotary": rotary, "norm": norm, "interleaved": interleaved, "max_pos": max_pos, "mode": mode,
         "chunk": chunk, "pads": pads}
    return c if name is None else {"name": name, **c}


def _attn(name, seqs, lo, hi, heads, kv_heads, dim, dtype):
    c = {"op": "attention", "seqs": seqs, "lo": lo, "hi": hi, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "dtype": dtype}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one sequence's newest token: latency counts
        _rope("qk one token", 1, 32, 8, 128, "bf16", 128, mode="decode"),
        # a large prefill step's projection before the attention, Q, K, V slices of one fused buffer
        _rope("qk prefill 8192", 8192, 64, 8, 128, "bf16", 128),
        # f32, a rotation of half the head in adjacent pairs, no norm, an odd number of tokens
        _rope("qk f32 partial 4095", 4095, 32, 32, 64, "f32", 32, norm=False, interleaved=True),
        # a decode step of 64 ragged sequences (f16 caches, one KV head per query head, no norm)
        _rope("append f16 decode 64", 64, 32, 32, 128, "f16", 128, op="same", norm=False, mode="decode", max_pos=4096),
        # a mixed step: 32 chunks of 512 prompt tokens, bf16 caches
        _rope("append bf16 chunks 16384", 16384, 32, 8, 128, "bf16", 128, op="same"),
        # ragged prompts into an 8-bit cache with one scale, with padding rows, wide heads
        _rope("append fp8 ragged 2047", 2047, 16, 4, 256, "bf16", 256, op="fp8", chunk=173, pads=9),
        # a decode step of 1024 sequences into a block-scaled cache
        _rope("append block decode 1024", 1024, 64, 8, 128, "bf16", 128, op="block", mode="decode"),
        # prompts whose chunks start and end inside blocks, block-scaled
        _rope("append block ragged 16384", 16384, 32, 8, 128, "bf16", 128, op="block", chunk=501, pads=17),
        # one sequence, a context of an odd length: latency counts
        _attn("attend one sequence", 1, 1001, 1001, 32, 8, 128, "bf16"),
        # 64 ragged sequences, one KV head per query head
        _attn("attend f16 ragged 64", 64, 128, 4096, 32, 32, 128, "f16"),
        # few sequences, long contexts
        _attn("attend long 16", 16, 16384, 131072, 32, 8, 128, "bf16"),
        # many sequences, 8 query heads per KV head
        _attn("attend batch 256", 256, 512, 8192, 64, 8, 128, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kv = rng.choice([1, 2, 4, 8, 8, 32])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 12, 16]) if kv < 32 else 1
    op = rng.choice(["qk", "same", "fp8", "block", "append", "attention", "attention", "attention"])
    if op == "attention":
        lo = _log_int(rng, 1, 16384)
        hi = _log_int(rng, lo, min(131072, 64 * lo + 1024))
        dim = rng.choice([128, 128, 256])
        # no more KV bytes than the largest listed case
        most = 256 * 8192 * 8 * 128 // (hi * kv * dim)
        seqs = _log_int(rng, 1, max(1, min(512, most)))
        return _attn(None, seqs, lo, hi, kv * group, kv, dim, rng.choice(["bf16", "f16"]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
    rotary = rng.choice([dim, dim, dim // 2])
    mode = rng.choice(["decode", "prefill"])
    most = 16384 * (64 + 16) * 128 * 2 // ((kv * group + 2 * kv) * dim * BYTES[dtype])
    tokens = _log_int(rng, 1, max(1, min(16384 if mode == "prefill" else 2048, most)))
    chunk = _log_int(rng, 1, 2048)
    return _rope(None, tokens, kv * group, kv, dim, dtype, rotary, op=op, norm=rng.random() < 0.6,
                 interleaved=rng.random() < 0.3, max_pos=rng.choice([2048, 32768, 131072]), mode=mode, chunk=chunk,
                 pads=rng.choice([0, 0, 3]) if tokens > 8 else 0)


def work(case):
    c = case
    if c["op"] == "attention":
        lens = _lengths(c)
        tok, blocks = sum(lens), sum(-(-n // BLOCK) for n in lens)
        e = BYTES[c["dtype"]]
        b = (tok * 2 * c["kv_heads"] * c["dim"] + blocks * (c["kv_heads"] * 8 + 4)
             + c["seqs"] * (2 * c["heads"] * c["dim"] * e + 4))
        return {"bytes": b, "flops": 4 * tok * c["heads"] * c["dim"]}
    t, e, d = c["tokens"], BYTES[c["dtype"]], c["dim"]
    live = t - c["pads"]
    q = 0 if c["op"] == "append" else 2 * c["heads"] * d * e
    table = 0 if c["op"] == "append" else c["rotary"] * 4 + 4
    if c["op"] == "qk":
        b = t * (q + 2 * c["kv_heads"] * d * e + table)
    else:
        store = e if c["op"] == "same" else 1
        b = t * (q + table + 4) + live * c["kv_heads"] * 2 * d * (e + store)
        if c["op"] in ("block", "append"):
            b += _touched(c)[0] * c["kv_heads"] * 2 * 8
    heads = (0 if c["op"] == "append" else c["heads"]) + c["kv_heads"]
    return {"bytes": b, "flops": t * heads * d * 7}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _lengths(c):
    """Context lengths, spread evenly over the logarithm of [lo, hi], the longest first."""
    n = c["seqs"]
    return [int(round(c["hi"] * (c["lo"] / c["hi"]) ** (i / max(1, n - 1)))) for i in range(n)]


def _touched(c):
    """(number of touched blocks, (block, offset) of each token): tokens of a chunk sit at consecutive
    positions of their own blocks, the first chunk at a block's start, the next ones 5, 10, ... tokens in;
    a decode step's tokens each in a block of its own, at any offset."""
    t = c["tokens"] - c["pads"]
    if c["mode"] == "decode":
        return t, [(i, (7 * i + 3) % BLOCK) for i in range(t)]
    at, base, i, n = [], 0, 0, 0
    while i < t:
        first = 5 * n % BLOCK
        m = min(c["chunk"], t - i)
        at += [(base + (first + j) // BLOCK, (first + j) % BLOCK) for j in range(m)]
        base += (first + m - 1) // BLOCK + 1
        i, n = i + m, n + 1
    return base, at


def _table(max_pos, rotary):
    i = torch.arange(rotary // 2, dtype=torch.float64, device=DEV)
    a = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-2 * i / rotary)
    return torch.cat([a.cos(), a.sin()], 1).float()


def _pool(g, shape, dtype=None):
    """An 8-bit pool's bytes in earnest: what a block's scale leaves of its rows, the largest near 448."""
    out = torch.empty(shape, dtype=torch.float8_e4m3fn, device=DEV)
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = (torch.randn(n, generator=g, device=DEV) * 96).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return out


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "attention":
        lens = _lengths(c)
        nblk = [-(-n // BLOCK) for n in lens]
        used, most = sum(nblk), max(nblk)
        pool = used + used // 8 + 1
        ids = torch.randperm(pool, generator=g, device=DEV)[:used].to(torch.int32)
        start = torch.tensor([sum(nblk[:i]) for i in range(len(nblk))], device=DEV)
        col = torch.arange(most, device=DEV)[None]
        n = torch.tensor(nblk, device=DEV)[:, None]
        s["block_tables"] = torch.where(col < n, ids[(start[:, None] + col).clamp_(max=used - 1)], 0).to(torch.int32)
        s["context_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["max_context_len"] = max(lens)
        shape = (pool, c["kv_heads"], BLOCK, c["dim"])
        s["key_cache"], s["value_cache"] = _pool(g, shape), _pool(g, shape)
        for name in ("k_scales", "v_scales"):
            s[name] = torch.exp2(torch.randint(-10, -5, shape[:2], generator=g, device=DEV).float())
        s["query"] = torch.randn((c["seqs"], c["heads"], c["dim"]), generator=g, device=DEV).to(dt)
        s["out"] = torch.empty_like(s["query"])
        s["scale"] = c["dim"] ** -0.5
        return s
    t, d, h, kv = c["tokens"], c["dim"], c["heads"], c["kv_heads"]
    # one fused projection's output: Q, K and V are strided slices of it
    qkv = torch.randn((t, (h + 2 * kv) * d), generator=g, device=DEV)
    qkv *= torch.exp(0.7 * torch.randn((t, 1), generator=g, device=DEV))
    qkv = qkv.to(dt)
    s["query"] = qkv[:, : h * d].view(t, h, d)
    s["key"] = qkv[:, h * d: (h + kv) * d].view(t, kv, d)
    s["value"] = qkv[:, (h + kv) * d:].view(t, kv, d)
    if c["op"] != "append":
        s["positions"] = torch.randint(0, c["max_pos"], (t,), generator=g, device=DEV, dtype=torch.int32)
        s["cos_sin"] = _table(c["max_pos"], c["rotary"])
        s["q_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt) if c["norm"] else None
        s["k_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt) if c["norm"] else None
        s["q_out"] = torch.empty((t, h, d), dtype=dt, device=DEV)
    if c["op"] == "qk":
        s["k_out"] = torch.empty((t, kv, d), dtype=dt, device=DEV)
        return s
    touched, at = _touched(c)
    pool = touched + touched // 8 + 1
    ids = torch.randperm(pool, generator=g, device=DEV)[:touched]
    at = torch.tensor(at, device=DEV)
    slots = (ids[at[:, 0]] * BLOCK + at[:, 1]).to(torch.int32)
    # padding rows at the end append nothing
    s["slot_mapping"] = torch.cat([slots, torch.full((c["pads"],), -1, dtype=torch.int32, device=DEV)])
    s["touched"], s["run_of"], s["offset"] = ids, at[:, 0].contiguous(), at[:, 1].contiguous()
    shape = (pool, kv, BLOCK, d)
    if c["op"] == "same":
        s["key_cache"] = torch.randn(shape, generator=g, device=DEV).to(dt)
        s["value_cache"] = torch.randn(shape, generator=g, device=DEV).to(dt)
        return s
    s["key_cache"], s["value_cache"] = _pool(g, shape), _pool(g, shape)
    if c["op"] == "fp8":
        s["k_scale"], s["v_scale"] = 0.0371, 0.0613
    else:
        for name in ("k_scales", "v_scales"):
            s[name] = torch.exp2(torch.randint(-9, -4, shape[:2], generator=g, device=DEV).float())
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _norm_rope(x, weight, cos_sin, positions, interleaved, eps=1e-6):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    r = cos_sin.shape[1]
    row = cos_sin[positions.long()][:, None]
    cos, sin = row[..., : r // 2], row[..., r // 2:]
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., r:]], -1)


def _power_of_two(amax):
    """The smallest power of two s with amax <= 448 s; 0 for 0."""
    m, e = torch.frexp(amax.double() / E4M3_MAX)
    s = torch.ldexp(torch.ones_like(m), e - (m == 0.5).to(e.dtype)).float()
    return torch.where(amax > 0, s, torch.zeros_like(s))


def _to_e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _append_block(x, cache, scales, s):
    n = s["run_of"].shape[0]
    x = x[:n].float()
    runs, off, ids = s["run_of"], s["offset"], s["touched"]
    kv = x.shape[1]
    zero = torch.zeros((ids.shape[0], kv), device=x.device)
    need = _power_of_two(zero.index_reduce(0, runs, x.abs().amax(-1), "amax"))
    fresh = torch.zeros(ids.shape[0], device=x.device).index_reduce(0, runs, (off == 0).float(), "amax") > 0
    old = scales[ids]
    new = torch.where(fresh[:, None], need, torch.maximum(old, need))
    ratio = torch.where(fresh[:, None] | (new == 0), torch.ones_like(new), old / new)
    blocks = cache[ids].float() * ratio[:, :, None, None]
    step = torch.where(new > 0, new, torch.ones_like(new))[runs]
    blocks[runs, :, off] = (x / step[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    cache[ids] = blocks.to(torch.float8_e4m3fn)
    scales[ids] = new


def _append(x, cache, s, scale):
    n = s["run_of"].shape[0]
    b, o = s["touched"][s["run_of"]], s["offset"]
    cache[b, :, o] = x[:n].to(cache.dtype) if scale is None else _to_e4m3(x[:n].float() / scale)


def _plain_attention(s):
    q, bt = s["query"], s["block_tables"].long()
    c = s["case"]
    n, h, d = q.shape
    kv = c["kv_heads"]

    def rows(cache, scales):
        x = cache[bt].float() * scales[bt][..., None, None]  # [S, blocks, Hkv, 16, D]
        return x.permute(0, 2, 1, 3, 4).reshape(n, kv, -1, d)

    logits = torch.matmul(q.float().view(n, kv, h // kv, d) * s["scale"],
                          rows(s["key_cache"], s["k_scales"]).transpose(-1, -2))
    masked = torch.arange(logits.shape[-1], device=q.device)[None] >= s["context_lens"][:, None]
    logits.masked_fill_(masked[:, None, None], -math.inf)
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    o = torch.matmul(p, rows(s["value_cache"], s["v_scales"])) / p.sum(-1, keepdim=True)
    return o.reshape(n, h, d).to(q.dtype)


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        from cacheflow_b200 import ops

        if op == "attention":
            if "workspace" not in s:  # kept by the caller, as for paged_attention_v1
                size = ops.paged_attention_fp8_block_workspace_size(s["query"], s["key_cache"], s["block_tables"],
                                                                    s["max_context_len"])
                s["workspace"] = torch.empty((size,), dtype=torch.uint8, device=DEV)
            return ops.paged_attention_fp8_block_v1(
                s["out"], s["query"], s["key_cache"], s["value_cache"], s["k_scales"], s["v_scales"],
                s["block_tables"], s["context_lens"], s["scale"], s["max_context_len"], workspace=s["workspace"])
        if op == "append":
            ops.reshape_and_cache_fp8_block(s["key"], s["value"], s["key_cache"], s["value_cache"], s["k_scales"],
                                            s["v_scales"], s["slot_mapping"])
            return [s["key_cache"], s["value_cache"], s["k_scales"], s["v_scales"]]
        norms = {"q_weight": s["q_weight"], "k_weight": s["k_weight"], "eps": 1e-6, "interleaved": c["interleaved"]}
        if op == "qk":
            ops.qk_norm_rope(s["q_out"], s["k_out"], s["query"], s["key"], s["positions"], s["cos_sin"], **norms)
            return [s["q_out"], s["k_out"]]
        caches = (s["q_out"], s["query"], s["key"], s["value"], s["key_cache"], s["value_cache"])
        if op == "same":
            ops.rope_and_cache(*caches, s["slot_mapping"], s["positions"], s["cos_sin"], **norms)
        elif op == "fp8":
            ops.rope_and_cache_fp8(*caches, s["slot_mapping"], s["positions"], s["cos_sin"], s["k_scale"],
                                   s["v_scale"], **norms)
        else:
            ops.rope_and_cache_fp8_block(*caches, s["k_scales"], s["v_scales"], s["slot_mapping"], s["positions"],
                                         s["cos_sin"], **norms)
            return [s["q_out"], s["key_cache"], s["value_cache"], s["k_scales"], s["v_scales"]]
        return [s["q_out"], s["key_cache"], s["value_cache"]]
    if op == "attention":
        return _plain_attention(s)
    if op == "append":
        _append_block(s["key"], s["key_cache"], s["k_scales"], s)
        _append_block(s["value"], s["value_cache"], s["v_scales"], s)
        return [s["key_cache"], s["value_cache"], s["k_scales"], s["v_scales"]]
    dt = s["query"].dtype
    q = _norm_rope(s["query"], s["q_weight"], s["cos_sin"], s["positions"], c["interleaved"]).to(dt)
    k = _norm_rope(s["key"], s["k_weight"], s["cos_sin"], s["positions"], c["interleaved"])
    if op == "qk":
        return [q, k.to(dt)]
    if op == "block":
        _append_block(k, s["key_cache"], s["k_scales"], s)
        _append_block(s["value"], s["value_cache"], s["v_scales"], s)
        return [q, s["key_cache"], s["value_cache"], s["k_scales"], s["v_scales"]]
    _append(k, s["key_cache"], s, s.get("k_scale"))
    _append(s["value"], s["value_cache"], s, s.get("v_scale"))
    return [q, s["key_cache"], s["value_cache"]]


# ---------------------------------------------------------------------------
# Definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rotated(x, weight, s, interleaved):
    """Norm and rotation as complex products, the pair (a, b) being a + ib."""
    z = x.double()
    if weight is not None:
        z = weight.double() * z / ((z ** 2).sum(-1, keepdim=True) / z.shape[-1] + 1e-6).sqrt()
    r = s["cos_sin"].shape[1]
    f = s["cos_sin"].double()[s["positions"].long()]
    turn = torch.complex(f[:, : r // 2], f[:, r // 2:])[:, None, :]
    even = torch.arange(r // 2, device=z.device)
    first, second = (2 * even, 2 * even + 1) if interleaved else (even, even + r // 2)
    y = torch.complex(z[..., first], z[..., second]) * turn
    z[..., first], z[..., second] = y.real, y.imag
    return z


def _binade(x):
    """The largest power of two not over x > 0: a guess by logarithms, put right by comparisons."""
    b = torch.exp2(torch.floor(torch.log2(x))).float().double()
    b = torch.where(b > x, b / 2, b)
    return torch.where(2 * b <= x, 2 * b, b)


def _exact_e4m3(x):
    """To the nearest multiple of the step at |x| (ties to even), 2^-9 at least, no further than 448."""
    step = _binade(x.abs().clamp(min=2.0 ** -6)) / 8
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append_block(x, cache, scales, s):
    cache, scales = cache.double(), scales.double().clone()
    n = s["run_of"].shape[0]
    order = torch.argsort(s["run_of"], stable=True)
    runs, off = s["run_of"][order], s["offset"][order]
    # every run as a full block of 16 rows, the absent ones 0 and not `there`
    rows = torch.zeros((s["touched"].shape[0], BLOCK) + tuple(x.shape[1:]), dtype=torch.float64, device=x.device)
    there = torch.zeros(rows.shape[:2], dtype=torch.bool, device=x.device)
    rows[runs, off] = x[:n].double()[order]
    there[runs, off] = True
    rows = rows.transpose(1, 2)  # [runs, Hkv, 16, D]
    top = rows.abs().amax((-1, -2))
    # 448 = 1.75 * 2^8: a power of two b with b <= top < 2b has scale b / 2^8 up to 1.75 b, 2b / 2^8 beyond
    b = _binade(top.clamp(min=1e-300))
    need = torch.where(top > 0, torch.where(top <= 1.75 * b, b, 2 * b) / 256, 0.0)
    was = scales[s["touched"]]
    begun = there[:, :1]
    now = torch.where(begun, need, torch.maximum(was, need))
    kept = cache[s["touched"]]
    moved = torch.where((begun | (now == 0))[..., None, None], kept,
                        _exact_e4m3(kept * (was / now.clamp(min=1e-300))[..., None, None]))
    put = _exact_e4m3(rows / torch.where(now > 0, now, 1.0)[..., None, None])
    cache[s["touched"]] = torch.where(there[:, None, :, None], put, moved)
    scales[s["touched"]] = now
    return cache, scales


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "attention":
        outs = []
        g = c["heads"] // c["kv_heads"]
        for i, n in enumerate(_lengths(c)):
            b = s["block_tables"][i, : -(-n // BLOCK)].long()
            k = (s["key_cache"][b].double() * s["k_scales"][b].double()[..., None, None])
            v = (s["value_cache"][b].double() * s["v_scales"][b].double()[..., None, None])
            k, v = (x.transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :n] for x in (k, v))
            q = s["query"][i].double().view(c["kv_heads"], g, c["dim"])
            p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) * s["scale"], -1)
            outs.append(torch.einsum("hgt,htd->hgd", p, v).reshape(c["heads"], c["dim"]))
        return torch.stack(outs)
    if c["op"] == "append":
        kc, ks = _exact_append_block(s["key"], s["key_cache"], s["k_scales"], s)
        vc, vs = _exact_append_block(s["value"], s["value_cache"], s["v_scales"], s)
        return [kc, vc, ks, vs]
    q = _exact_rotated(s["query"], s["q_weight"], s, c["interleaved"])
    k = _exact_rotated(s["key"], s["k_weight"], s, c["interleaved"])
    if c["op"] == "qk":
        return [q, k]
    if c["op"] == "block":
        kc, ks = _exact_append_block(k, s["key_cache"], s["k_scales"], s)
        vc, vs = _exact_append_block(s["value"], s["value_cache"], s["v_scales"], s)
        return [q, kc, vc, ks, vs]
    n = s["run_of"].shape[0]
    b, o = s["touched"][s["run_of"]], s["offset"]
    outs = [q]
    for x, cache, name in ((k, "key_cache", "k_scale"), (s["value"].double(), "value_cache", "v_scale")):
        full = s[cache].double()
        full[b, :, o] = x[:n] if c["op"] == "same" else _exact_e4m3(x[:n] / s[name])
        outs.append(full)
    return outs
