"""Plain 64-bit forms of the operators that fill the paged KV cache and attend over it (torch, any device)."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def rotate(x, positions, inv_freq, interleaved=False, mscale=1.0, transpose=False):
    """float64 [T, H, D]."""
    y = x.double().clone()
    r = 2 * inv_freq.numel()
    a = positions.double()[:, None, None] * inv_freq.double()
    c, s = a.cos() * mscale, a.sin() * mscale * (-1.0 if transpose else 1.0)
    one, two = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    p, q = x.double()[..., one], x.double()[..., two]
    y[..., one], y[..., two] = p * c - q * s, q * c + p * s
    return y


def rotate_slack(x, inv_freq, interleaved=False, mscale=1.0):
    """What float32 arithmetic may add to a rotated element: cosine, sine, their product with mscale, two products and a sum
    are off by at most 2^-22 each of |a| + |b|, and the angle (2^-23) moves the pair by as much."""
    r = 2 * inv_freq.numel()
    one, two = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    s = torch.zeros_like(x, dtype=torch.float64)
    s[..., one] = s[..., two] = (x.double()[..., one].abs() + x.double()[..., two].abs()) * mscale * 6 * 2.0 ** -22
    return s


def half_step(dtype, value):
    """Largest rounding error of a value stored as dtype (its smallest step where the value is subnormal)."""
    f = torch.finfo(dtype)
    return torch.maximum(value.abs() * (f.eps / 2), torch.full_like(value, f.smallest_normal * f.eps / 2))


def scale_for(largest):
    """Smallest 2^e >= 2^-126 with 448 * 2^e >= largest; 0 for 0."""
    return 0.0 if largest == 0 else max(2.0 ** -126, 2.0 ** math.ceil(math.log2(largest / 448.0)))


def append(x, slots, cache, scale):
    """What the cache's values (float64 [NB, BS, H, D]) and scales have to be after x [T, H, D] went to its slots, and how
    far a stored value may be off."""
    nb, bs, h, _ = cache.shape
    slots = slots.tolist()
    token = {s: t for t, s in enumerate(slots) if 0 <= s < nb * bs}     # the later token wins
    value = cache.double()
    if scale is None:
        room = torch.zeros_like(value)
        for s, t in token.items():
            value[s // bs, s % bs] = x[t]
            room[s // bs, s % bs] = half_step(cache.dtype, x[t])
        return value, None, room
    scale = scale.double().clone()
    value = value * scale[:, None, :, None]
    value[(scale == 0)[:, None, :, None].expand_as(value)] = 0.0
    room = torch.zeros_like(value)
    for b in sorted({s // bs for s in token}):
        rows = {s % bs: t for s, t in token.items() if s // bs == b}
        anew = 0 in rows
        others = [r for r in range(bs) if r not in rows]
        for i in range(h):
            new = torch.stack([x[t, i] for t in rows.values()])
            fin = new[torch.isfinite(new)].abs()
            need = scale_for(float(fin.max()) if fin.numel() else 0.0)
            old = float(scale[b, i])
            now = need if anew else max(old, need)
            if not anew and now > old:
                room[b, others, i] = now * 2.0 ** -10           # half the smallest step of a code
            if anew:
                value[b, others, i] = math.nan                  # without meaning
            scale[b, i] = now
            for r, t in rows.items():
                v = x[t, i].clone()
                v[~torch.isfinite(v)] = math.nan
                value[b, r, i] = v
                room[b, r, i] = torch.maximum(v.nan_to_num(0.0).abs() * 2.0 ** -4, torch.full_like(v, now * 2.0 ** -10))
    return value, scale, room


def attention(q, k_cache, v_cache, table, seq_lens, *, k_scale=None, v_scale=None, query_start=None, scale=None,
              causal=True):
    """(out, lse, out room, lse room), float64 [T, Hq, D] and [T, Hq]; nan where no request has a token.

    Room: scores are sums of D products in float32 (each product and each sum off by 2^-24, twice that where a tensor core
    cuts instead of rounding) times three factors; the exponential adds 2^-22 of its value; so a weight is off by e =
    2 * scale * sum|q k| * D * 2^-23 + 2^-20 of itself at most, sums over tokens by 2^-18.  The weight is rounded once for its
    product with v: by finfo.eps / 2 of itself, 2^-8 (bf16: eps 2^-7) or 2^-11 (fp16: eps 2^-10; e4m3 codes use it too).  With numerator and denominator each off by e, the
    result is off by (2 e + rounding + 2^-17) * sum(p |v|) / sum(p), and by half a step of its own type."""
    t, hq, d = q.shape
    nb, bs, hkv, _ = k_cache.shape
    g = hq // hkv
    b = seq_lens.numel()
    start = list(range(b + 1)) if query_start is None else query_start.tolist()
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((t, hq, d), math.nan, dtype=torch.float64, device=q.device)
    lse = torch.full((t, hq), math.nan, dtype=torch.float64, device=q.device)
    room, lse_room = torch.zeros_like(out), torch.zeros_like(lse)
    weight_step = torch.finfo(torch.bfloat16 if k_cache.dtype == torch.bfloat16 else torch.float16).eps / 2
    for i in range(b):
        n = min(max(int(seq_lens[i]), 0), table.shape[-1] * bs)
        nq = start[i + 1] - start[i]
        rows = slice(start[i], start[i + 1])
        for h in range(hkv):
            ids = (table[i] if table.dim() == 2 else table[i, h])[:-(-n // bs)].long()
            ok = (ids >= 0) & (ids < nb)
            safe = torch.where(ok, ids, torch.zeros_like(ids))
            k, v = k_cache[safe][:, :, h].double(), v_cache[safe][:, :, h].double()
            if k_scale is not None:
                k, v = k * k_scale[safe, h].double()[:, None, None], v * v_scale[safe, h].double()[:, None, None]
            live = ok[:, None].expand(-1, bs).reshape(-1)[:n]
            k, v = k.reshape(-1, d)[:n], v.reshape(-1, d)[:n]
            sees = torch.arange(n, device=q.device)[None] < ((n - nq + 1 + torch.arange(nq, device=q.device))[:, None] if causal else n)
            sees = sees.expand(nq, n) & live
            for j in range(h * g, h * g + g):
                qj = q[rows, j].double()
                s = (qj[:, None, :] * k[None]).sum(-1) * scale if n * nq * d < 1 << 22 else qj @ k.T * scale
                s = torch.where(sees, s, torch.full_like(s, -math.inf))
                m = s.amax(1, keepdim=True) if n else torch.full((nq, 1), -math.inf, dtype=torch.float64, device=q.device)
                p = torch.where(sees, (s - torch.where(m > -math.inf, m, torch.zeros_like(m))).exp(), torch.zeros_like(s))
                total = p.sum(1, keepdim=True)
                w = torch.where(total > 0, p / total, torch.zeros_like(p))
                vv = torch.where(sees[:, :, None], v[None], torch.zeros_like(v)[None]) if not torch.isfinite(v).all() else None
                o = (w[:, :, None] * vv).sum(1) if vv is not None else w @ v
                av = (w[:, :, None] * vv.abs()).sum(1) if vv is not None else w @ v.abs()
                fine = k.nan_to_num(0.0, 0.0, 0.0).abs()
                big = torch.where(sees, qj.abs() @ fine.T, torch.zeros_like(s)).amax(1, keepdim=True) * abs(scale) if n else torch.zeros_like(m)
                e = 2 * big * d * 2.0 ** -23 + 2.0 ** -20
                out[rows, j], lse[rows, j] = o, (m + total.log())[:, 0]
                room[rows, j] = (2 * e + weight_step + 2.0 ** -17) * av + half_step(q.dtype, o)
                lse_room[rows, j] = (e + 2.0 ** -18 + (m + total.log()).abs().nan_to_num(0, 0, 0) * 2.0 ** -22)[:, 0]
    return out, lse, room, lse_room
