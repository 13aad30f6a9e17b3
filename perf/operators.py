"""Measured cases of the attention-side operators: rotary positions, the append to the paged KV cache and the attention
that reads that cache.

Three operators, each through its public entry point in ``unified_cache_management_b200.ops``:

  rotary      y = mscale * R(position * inv_freq) x on the first ``rot`` elements of every head, the rest copied;
              half and interleaved layouts, and the transposed rotation (its gradient).
  append      a step's new keys (rotated on the way) and values go to their slots of the paged caches.  A cache of
              e4m3 codes has one scale per (block, kv head): the smallest power of two that keeps the block's largest
              value within 448.  A block whose row 0 is written starts anew; any other keeps its scale, or takes the
              larger one that the new tokens need, and the codes of its other rows are then re-rounded.  The step's
              queries are rotated in the same call.
  attention   softmax(scale * q k^T) v over the blocks that a table lists, shared by all heads or chosen per kv head,
              one query token per request (decode), a few (speculative verification) or a chunk (prefill), with the
              log-sum-exp of every row.

``run`` computes the plain form (elementary torch operations in 32 bits) unless ``own`` is set.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
WORKSPACE = 32 << 20   # bytes of zeros handed to the attention; more than any call asks for


# --------------------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------------------
def _rotary(name, tokens, heads, dim, rot, interleaved, transpose, dtype, far, scaling, packed):
    return dict(name=name, op="rotary", tokens=tokens, heads=heads, dim=dim, rot=rot, interleaved=interleaved,
                transpose=transpose, dtype=dtype, far=far, scaling=scaling, packed=packed)


def _append(name, requests, tokens, context, pad, q_heads, kv_heads, dim, rot, block, cache, dtype, scaling):
    return dict(name=name, op="append", requests=requests, tokens=tokens, context=context, pad=pad, q_heads=q_heads,
                kv_heads=kv_heads, dim=dim, rot=rot, block=block, cache=cache, dtype=dtype, scaling=scaling)


def _attention(name, requests, queries, context, ragged, selected, q_heads, kv_heads, dim, block, cache, dtype):
    return dict(name=name, op="attention", requests=requests, queries=queries, context=context, ragged=ragged,
                selected=selected, q_heads=q_heads, kv_heads=kv_heads, dim=dim, block=block, cache=cache, dtype=dtype)


def listed():
    return [
        # one decode step's queries of 16 requests at 131072 tokens: a launch and little else
        _rotary("rotary_decode", 16, 32, 128, 128, False, False, "bf16", 131072, "llama3", False),
        # a 32768-token prefill of a YaRN-scaled model, far into a four-million-token context
        _rotary("rotary_prefill", 32768, 32, 128, 128, False, False, "bf16", 4194304, "yarn", False),
        # gradient of a partial interleaved rotation; the heads are a view of a packed qkv row, an odd token count
        _rotary("rotary_partial_grad", 5001, 16, 128, 64, True, True, "fp16", 8192, "none", True),
        # a decode step of the 16-request benchmark: 16 new tokens into half-full blocks of 128, 32 query heads rotated
        _append("append_decode16_e4m3", 16, 16, 131072, 0, 32, 8, 128, 128, 128, "e4m3", "bf16", "llama3"),
        # chunked prefill of four requests that start inside a block, padded at the end
        _append("append_prefill_e4m3", 4, 32768, 5000, 64, 32, 8, 128, 128, 128, "e4m3", "bf16", "llama3"),
        # the same into a 16-bit cache with the engine's default block of 16 tokens
        _append("append_prefill_16bit", 7, 9000, 333, 5, 16, 2, 64, 32, 16, "same", "fp16", "none"),
        # one short chat request, blocks of 16
        _attention("attn_decode_short", 1, 1, 333, False, False, 32, 8, 128, 16, "e4m3", "bf16"),
        # after the retrieval: 64 blocks of 128 chosen per kv head for each of 16 requests
        _attention("attn_decode16_selected", 16, 1, 8192, False, True, 32, 8, 128, 128, "e4m3", "bf16"),
        # the rollback layers of the same step attend to everything: 16 x 131072 tokens
        _attention("attn_decode16_full", 16, 1, 131072, False, False, 32, 8, 128, 128, "e4m3", "bf16"),
        # ragged 16-bit cache, one query head per kv head, heads of 64, blocks of 16
        _attention("attn_decode_ragged_16bit", 33, 1, 30000, True, False, 8, 8, 64, 16, "same", "fp16"),
        # speculative verification: four tokens per request, eight query heads per kv head
        _attention("attn_verify4", 8, 4, 65000, True, False, 64, 8, 128, 64, "e4m3", "bf16"),
        # chunked prefill of two requests, 4096 new tokens each behind a longer context
        _attention("attn_prefill", 2, 4096, 16384, True, False, 32, 8, 128, 128, "e4m3", "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        heads = rng.choice([1, 2, 7, 8, 16, 32, 64])
        rot = rng.choice([dim, dim // 2, 32])
        tokens = _log(rng, 1, 32768 * 32 * 128 // (heads * dim))
        c = _rotary("", tokens, heads, dim, rot, rng.random() < 0.5, rng.random() < 0.3, dtype,
                    rng.choice([tokens, 131072, 4194304]), rng.choice(["none", "linear", "llama3", "yarn"]),
                    rng.random() < 0.3)
    elif op == "append":
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        requests = _log(rng, 1, 64)
        if rng.random() < 0.4:
            tokens = requests
        else:
            tokens = max(requests, _log(rng, 1, 32768))
        c = _append("", requests, tokens, _log(rng, 1, 8000), rng.choice([0, 3, 17]), kv_heads * rng.choice([1, 4, 5, 8]),
                    kv_heads, dim, rng.choice([dim, dim // 2]), rng.choice([16, 24, 32, 64, 128]),
                    rng.choice(["e4m3", "e4m3", "same"]), dtype, rng.choice(["none", "llama3", "yarn"]))
        while c["tokens"] * (c["q_heads"] + 2 * c["kv_heads"]) * dim > 32768 * 48 * 128:
            c["tokens"] //= 2
        c["tokens"] = max(c["tokens"], requests)
    else:
        dim = rng.choice([64, 128, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        g = rng.choice([1, 2, 4, 5, 8, 16])
        kind = rng.choice(["decode", "decode", "verify", "prefill"])
        queries = 1 if kind == "decode" else rng.choice([2, 3, 4, 7]) if kind == "verify" else _log(rng, 17, 4096)
        requests = _log(rng, 1, 64) if kind != "prefill" else rng.choice([1, 2, 3])
        context = max(queries, _log(rng, 16, 131072 if kind != "prefill" else 16384))
        block = rng.choice([16, 24, 32, 64, 128])
        while requests * context * kv_heads * dim > 16 * 131072 * 8 * 128 or \
                requests * kv_heads * g * queries * context > 2 * 32 * 4096 * 16384:
            if requests > 1:
                requests //= 2
            else:
                context //= 2
                queries = min(queries, context)
        c = _attention("", requests, queries, context, rng.random() < 0.6, kind == "decode" and rng.random() < 0.4,
                       kv_heads * g, kv_heads, dim, block, rng.choice(["e4m3", "e4m3", "same"]), dtype)
    del c["name"]
    return c


def _lengths(c):
    """(tokens in the cache, query tokens) of each request; ragged ones run from a handful to the whole context."""
    r, q, n = c["requests"], c["queries"], c["context"]
    if not c["ragged"]:
        return [n] * r, [q] * r
    lens = [max(1, int(round(n ** ((i + 1) / r)))) if r > 3 else n * (i + 1) // r for i in range(r)]
    if r > 8:
        lens[0] = 0                                      # a request that has nothing to attend to
    qs = [q if q <= 8 else max(1, q - 37 * i) for i in range(r)]
    return [max(n_, q_) if n_ else 0 for n_, q_ in zip(lens, qs)], qs


def _new_tokens(c):
    """(tokens before the call, new tokens) of each request of an append."""
    r, t = c["requests"], c["tokens"]
    new = [t // r + (1 if i < t % r else 0) for i in range(r)]
    return [max(0, c["context"] - 29 * i) for i in range(r)], new


# --------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------
def _inv_freq(rot, scaling, device):
    """Radians per position of each pair, in 64 bits, and the factor on the rotated values."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    base = 500000.0 if scaling == "llama3" else 10000.0
    f = base ** (-2.0 * i / rot)
    m = 1.0
    if scaling == "linear":
        f = f / 4.0
    elif scaling == "llama3":                            # wave lengths beyond the original context are stretched
        wave = 2 * math.pi / f
        smooth = ((8192.0 / wave - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        f = f * (smooth + (1.0 - smooth) / 8.0)
    elif scaling == "yarn":                              # a ramp over the pairs between the two rotation counts
        def pair(turns):
            return rot * math.log(4096.0 / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        f = f * (1.0 - ramp) + f / 40.0 * ramp
        m = 0.1 * math.log(40.0) + 1.0
    return f.to(device), m


def _gen(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def _codes(shape, g, device):
    """e4m3 codes of normal values, as a block's scale leaves them: the largest near 448."""
    out = torch.empty(shape, dtype=E4M3, device=device)
    for part in out.view(torch.uint8).split(max(1, (1 << 28) // max(1, math.prod(shape[1:])))):
        x = torch.randn(part.shape, dtype=torch.float32 if part.numel() < 1 << 20 else torch.bfloat16, device=device,
                        generator=g)
        part.copy_(x.mul_(80.0).clamp_(-448.0, 448.0).to(E4M3).view(torch.uint8))
    return out


def _scales(shape, g, device):
    return torch.pow(2.0, torch.randint(-8, -5, shape, device=device, generator=g).float())


def prepare(case, seed):
    dev = torch.device("cuda")
    c, g = case, _gen(seed, dev)
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "rotary":
        extra = 2 * max(1, c["heads"] // 4) if c["packed"] else 0
        s["x"] = torch.randn((c["tokens"], c["heads"] + extra, c["dim"]), device=dev, generator=g, dtype=dt)[:, :c["heads"]]
        s["inv_freq"], s["mscale"] = _inv_freq(c["rot"], c["scaling"], dev)
        s["positions"] = torch.arange(c["tokens"], device=dev) + \
            torch.randint(0, max(1, c["far"] - c["tokens"]) + 1, (1,), device=dev, generator=g)
    elif c["op"] == "append":
        before, new = _new_tokens(c)
        bs, d = c["block"], c["dim"]
        t, pad = sum(new), c["pad"]
        blocks = [-(-(b + n) // bs) - b // bs for b, n in zip(before, new)]   # blocks that the call touches
        nb = sum(blocks) + 9
        perm = torch.randperm(nb, device=dev, generator=g)
        slots, pos, at = [], [], 0
        for b, n, m in zip(before, new, blocks):
            p = torch.arange(b, b + n, device=dev)
            slots.append(perm[at + p // bs - b // bs] * bs + p % bs)
            pos.append(p)
            at += m
        none = torch.full((pad,), -1, dtype=torch.int64, device=dev)
        s["slots"] = torch.cat(slots + [none])
        s["positions"] = torch.cat(pos + [torch.zeros_like(none)])
        s["touched"] = perm[:at]
        qkv = torch.randn((t + pad, c["q_heads"] + 2 * c["kv_heads"], d), device=dev, generator=g, dtype=dt)
        s["q"], s["k"], s["v"] = qkv.split([c["q_heads"], c["kv_heads"], c["kv_heads"]], 1)
        s["inv_freq"], s["mscale"] = _inv_freq(c["rot"], c["scaling"], dev)
        shape = (nb, bs, c["kv_heads"], d)
        if c["cache"] == "e4m3":
            s["k_cache"], s["v_cache"] = _codes(shape, g, dev), _codes(shape, g, dev)
            s["k_scale"], s["v_scale"] = _scales((nb, c["kv_heads"]), g, dev), _scales((nb, c["kv_heads"]), g, dev)
        else:
            s["k_cache"] = torch.randn(shape, device=dev, generator=g, dtype=dt)
            s["v_cache"] = torch.randn(shape, device=dev, generator=g, dtype=dt)
            s["k_scale"] = s["v_scale"] = None
        s["q_out"] = torch.empty((t + pad, c["q_heads"], d), dtype=dt, device=dev)
    else:
        lens, qs = _lengths(c)
        r, bs, d, hkv = c["requests"], c["block"], c["dim"], c["kv_heads"]
        per = [-(-n // bs) for n in lens]
        mb = max(1, max(per))
        if c["selected"]:                                # every kv head has its own blocks, out of a larger pool
            nb = 4 * sum(per) + 7
            order = torch.argsort(torch.rand((hkv, nb), device=dev, generator=g), dim=1).to(torch.int32)
            table = torch.zeros((r, hkv, mb), dtype=torch.int32, device=dev)
        else:
            nb = sum(per) + 7
            order = torch.randperm(nb, device=dev, generator=g).to(torch.int32)[None]
            table = torch.zeros((r, 1, mb), dtype=torch.int32, device=dev)
        at = 0
        for i, m in enumerate(per):
            table[i, :, :m] = order[:, at:at + m]
            at += m
        s["table"] = table if c["selected"] else table[:, 0].contiguous()
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["query_start"] = torch.tensor([sum(qs[:i]) for i in range(r + 1)], dtype=torch.int32, device=dev)
        s["max_query_len"] = max(qs)
        s["q"] = torch.randn((sum(qs), c["q_heads"], d), device=dev, generator=g).mul_(2.5).to(dt)
        shape = (nb, bs, hkv, d)
        if c["cache"] == "e4m3":
            s["k_cache"], s["v_cache"] = _codes(shape, g, dev), _codes(shape, g, dev)
            s["k_scale"], s["v_scale"] = _scales((nb, hkv), g, dev), _scales((nb, hkv), g, dev)
        else:
            s["k_cache"] = torch.randn(shape, device=dev, generator=g, dtype=dt)
            s["v_cache"] = torch.randn(shape, device=dev, generator=g, dtype=dt)
            s["k_scale"] = s["v_scale"] = None
        s["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device=dev)
    return s


# --------------------------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------------------------
def _plain_rotate(x, positions, inv_freq, mscale, interleaved, transpose):
    """float32 [T, H, D]; the angles in 64 bits, since far positions lose them in 32."""
    r = 2 * inv_freq.numel()
    a = positions.double()[:, None, None] * inv_freq
    cos, sin = (a.cos() * mscale).float(), (a.sin() * mscale).float()
    if transpose:
        sin = -sin
    x = x.float()
    y = x.clone()
    one, two = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., one] = x[..., one] * cos - x[..., two] * sin
    y[..., two] = x[..., two] * cos + x[..., one] * sin
    return y


def _plain_scale(largest):
    """Smallest power of two that brings `largest` within 448; 0 for an empty or all-zero block."""
    m, e = torch.frexp(largest)                          # largest = m * 2^e, m in [0.5, 1)
    e = e - 9 + (m > 0.875).int()
    return torch.where(largest > 0, torch.ldexp(torch.ones_like(m), e.clamp(min=-126)), torch.zeros_like(m))


def _plain_store(x, slots, cache, scale, touched):
    """x float32 [T, H, D] to its slots of a paged cache, in place."""
    nb, bs, h, d = cache.shape
    if scale is None:
        cache.view(nb * bs, h, d).index_copy_(0, slots, x.to(cache.dtype))
        return
    block = slots // bs
    largest = torch.zeros((nb, h), device=x.device)
    largest.scatter_reduce_(0, block[:, None].expand(-1, h), x.abs().amax(-1), "amax")
    anew = torch.zeros(nb, device=x.device).scatter_reduce_(0, block, (slots % bs == 0).float(), "amax")[touched, None] > 0
    old = torch.where(anew, torch.zeros_like(largest[touched]), scale[touched])
    new = torch.maximum(old, _plain_scale(largest[touched]))
    codes = cache.view(torch.uint8)
    had = codes[touched]
    again = (had.view(E4M3).float() * (old / new)[:, None, :, None]).to(E4M3).view(torch.uint8)
    codes[touched] = torch.where(((new > old) & ~anew)[:, None, :, None], again, had)
    scale[touched] = new
    y = (x / scale[block][..., None]).to(E4M3).view(torch.uint8)
    codes.view(nb * bs, h, d).index_copy_(0, slots, y)


def _plain_attention(s, c):
    r, hkv, d = c["requests"], c["kv_heads"], c["dim"]
    g = c["q_heads"] // hkv
    table = s["table"].long()
    if table.dim() == 2:
        table = table[:, None].expand(-1, hkv, -1)
    heads = torch.arange(hkv, device=table.device)[None, :, None, None]
    rows = torch.arange(c["block"], device=table.device)

    def fetch(cache, scale):
        """float32 [r, hkv, tokens, d] of the listed blocks."""
        raw = cache.view(torch.uint8) if scale is not None else cache
        x = raw[table[..., None], rows, heads]
        if scale is None:
            x = x.float()
        else:
            x = x.view(E4M3).float().mul_(scale[table, heads[..., 0]][..., None, None])
        return x.reshape(r, hkv, -1, d)

    start, lens = s["query_start"].long(), s["seq_lens"].long()
    qn = start[1:] - start[:-1]
    mq, t = s["max_query_len"], s["q"].shape[0]
    i = torch.arange(mq, device=table.device)
    at = (start[:-1, None] + i).clamp(max=t - 1)
    q = s["q"].float()[at].view(r, mq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(r, hkv, g * mq, d)
    x = torch.matmul(q, fetch(s["k_cache"], s["k_scale"]).transpose(2, 3)).mul_(d ** -0.5)
    sees = (lens - qn)[:, None] + i + 1                  # query i sees the tokens before this one
    hidden = torch.arange(x.shape[-1], device=x.device) >= sees[:, :, None]
    x.view(r, hkv * g, mq, -1).masked_fill_(hidden[:, None], -math.inf)
    big = x.amax(-1, keepdim=True)
    x.sub_(torch.where(big > -math.inf, big, torch.zeros_like(big))).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x, fetch(s["v_cache"], s["v_scale"]))
    y = y / torch.where(total > 0, total, torch.ones_like(total))
    lse = (big + total.log()).view(r, hkv, g, mq).permute(0, 3, 1, 2).reshape(r, mq, hkv * g)
    y = y.view(r, hkv, g, mq, d).permute(0, 3, 1, 2, 4).reshape(r, mq, hkv * g, d)
    token = torch.arange(t, device=x.device)
    req = torch.bucketize(token, start[1:], right=True)
    return {"out": y[req, token - start[req]].to(s["q"].dtype), "lse": lse[req, token - start[req]]}


def run(state):
    c = state["case"]
    if own:
        return _run_own(state, c)
    if c["op"] == "rotary":
        return _plain_rotate(state["x"], state["positions"], state["inv_freq"], state["mscale"], c["interleaved"],
                             c["transpose"]).to(state["x"].dtype)
    if c["op"] == "append":
        q = _plain_rotate(state["q"], state["positions"], state["inv_freq"], state["mscale"], False, False)
        k = _plain_rotate(state["k"], state["positions"], state["inv_freq"], state["mscale"], False, False)
        n = sum(_new_tokens(c)[1])                       # the rest is padding
        slots, touched = state["slots"][:n], state["touched"]
        _plain_store(k[:n], slots, state["k_cache"], state["k_scale"], touched)
        _plain_store(state["v"][:n].float(), slots, state["v_cache"], state["v_scale"], touched)
        return _append_outputs(state, q.to(state["q"].dtype))
    return _plain_attention(state, c)


def _append_outputs(state, q):
    out = {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    if state["k_scale"] is not None:
        out["k_scale"], out["v_scale"] = state["k_scale"], state["v_scale"]
    return out


# --------------------------------------------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------------------------------------------
def _run_own(state, c):
    from unified_cache_management_b200 import ops
    if c["op"] == "rotary":
        return ops.rotary(state["x"], state["positions"], state["inv_freq"], interleaved=c["interleaved"],
                          mscale=state["mscale"], transpose=c["transpose"])
    if c["op"] == "append":
        ops.kv_append(state["k"], state["v"], state["slots"], state["k_cache"], state["v_cache"],
                      k_scale=state["k_scale"], v_scale=state["v_scale"], positions=state["positions"],
                      inv_freq=state["inv_freq"], mscale=state["mscale"], q=state["q"], q_out=state["q_out"])
        return _append_outputs(state, state["q_out"])
    out, lse = ops.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["table"], state["seq_lens"],
                                   k_scale=state["k_scale"], v_scale=state["v_scale"],
                                   query_start=state["query_start"], max_query_len=state["max_query_len"],
                                   workspace=state["workspace"], want_lse=True)
    return {"out": out, "lse": lse}


# --------------------------------------------------------------------------------------------------------------
# work and exact results
# --------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "rotary":
        n = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 4 * n + 8 * c["tokens"] + 4 * c["rot"], "flops": 3 * c["tokens"] * c["heads"] * c["rot"]}
    if c["op"] == "append":
        n = c["tokens"] * c["dim"]
        e = 1 if c["cache"] == "e4m3" else 2
        return {"bytes": 4 * n * c["q_heads"] + (2 + e) * 2 * n * c["kv_heads"] + 16 * c["tokens"],
                "flops": 3 * c["tokens"] * (c["q_heads"] + c["kv_heads"]) * c["rot"]}
    lens, qs = _lengths(c)
    e = 1 if c["cache"] == "e4m3" else 2
    blocks = sum(-(-n // c["block"]) for n in lens)
    scales = 8 * blocks * c["kv_heads"] if e == 1 else 0
    table = 4 * blocks * (c["kv_heads"] if c["selected"] else 1)
    rows = sum(qs) * c["q_heads"]
    pairs = sum(sum(max(0, n - q + 1 + i) for i in range(q)) for n, q in zip(lens, qs)) * c["q_heads"]
    return {"bytes": 2 * e * sum(lens) * c["kv_heads"] * c["dim"] + scales + table + rows * (4 * c["dim"] + 4),
            "flops": 4 * c["dim"] * pairs}


def exact(case, seed):
    """The definitions in 64 bits."""
    c, s = case, prepare(case, seed)

    def turned(x):
        z = x.double()
        r = c["rot"]
        even = c["op"] == "rotary" and c["interleaved"]
        pairs = z[..., :r].unflatten(-1, (r // 2, 2)) if even else z[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        sign = -1.0 if c["op"] == "rotary" and c["transpose"] else 1.0
        by = torch.polar(torch.full_like(s["inv_freq"], s["mscale"]), torch.zeros_like(s["inv_freq"])) * \
            torch.exp(1j * sign * s["positions"].double()[:, None] * s["inv_freq"])[:, None]
        w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        z = z.clone()
        z[..., :r] = w.flatten(-2) if even else w.transpose(-1, -2).flatten(-2)
        return z

    if c["op"] == "rotary":
        return turned(s["x"])
    if c["op"] == "append":
        out = {"q": turned(s["q"])}
        slots = s["slots"][s["slots"] >= 0]
        blocks = slots // c["block"]
        for what, x in (("k", turned(s["k"])), ("v", s["v"].double())):
            x = x[s["slots"] >= 0]
            cache, scale = s[what + "_cache"].double(), s[what + "_scale"]
            if scale is not None:
                scale = scale.double()
                for b in s["touched"].tolist():
                    mine = blocks == b
                    big = x[mine].abs().amax((0, 2))
                    need = torch.exp2(torch.ceil(torch.log2(big / 448.0)))
                    if bool((slots[mine] % c["block"] == 0).any()):
                        scale[b] = need
                    else:
                        new = torch.maximum(scale[b], need)
                        cache[b] *= (scale[b] / new)[None, :, None]
                        scale[b] = new
                x = x / scale[blocks][..., None]
                out[what + "_scale"] = scale
            cache[blocks, slots % c["block"]] = x
            out[what + "_cache"] = cache
        return out
    lens, qs = _lengths(c)
    g = c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, m) in enumerate(zip(lens, qs)):
        for h in range(c["kv_heads"] if n else 0):
            blocks = (s["table"][i, h] if c["selected"] else s["table"][i])[:-(-n // c["block"])].long()
            k, v = s["k_cache"][blocks, :, h].double(), s["v_cache"][blocks, :, h].double()
            if s["k_scale"] is not None:
                k = k * s["k_scale"][blocks, h].double()[:, None, None]
                v = v * s["v_scale"][blocks, h].double()[:, None, None]
            k, v = k.flatten(0, 1)[:n], v.flatten(0, 1)[:n]
            for j in range(h * g, h * g + g):
                x = (s["q"][first:first + m, j].double() @ k.T) / math.sqrt(c["dim"])
                x += torch.triu(torch.full((m, n), -math.inf, dtype=torch.float64, device="cuda"), n - m + 1)
                lse[first:first + m, j] = torch.logsumexp(x, 1)
                out[first:first + m, j] = torch.softmax(x, 1) @ v
        first += m
    return {"out": out, "lse": lse}
