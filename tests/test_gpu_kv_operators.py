"""GPU: rotary positions, append to the paged KV cache, attention over it, against 64-bit forms of their definitions."""
import math

import pytest
import torch

from tests import kv_reference as R

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
BF, FP = torch.bfloat16, torch.float16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(shape, g, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _close(got, want, room, what=""):
    got = got.double()
    bad = ~((got - want).abs() <= room) & ~(got.isnan() & want.isnan()) & ~(got == want)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: " \
                          f"{got[bad][0].item()} for {want[bad][0].item()} +- {room[bad][0].item()}"


# ---------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("t,h,d,rot,dtype,interleaved,transpose", [
    (1, 1, 128, 128, BF, False, False), (7, 3, 128, 64, BF, True, False), (16, 32, 128, 128, FP, False, True),
    (33, 5, 80, 80, BF, False, False), (5, 2, 96, 32, FP, True, True), (300, 8, 64, 64, BF, True, False),
    (2, 64, 256, 256, BF, False, False), (9, 3, 66, 18, FP, False, False), (9, 3, 65, 6, BF, True, True),
    (4000, 2, 128, 128, BF, False, False), (1100, 40, 128, 96, FP, False, False), (3, 2, 2, 2, BF, True, False)])
def test_rotary(cuda_device, t, h, d, rot, dtype, interleaved, transpose):
    from unified_cache_management_b200 import ops
    g = _gen(t + d)
    x = _randn((t, h, d), g, dtype)
    f, m = ops.rotary_frequencies(rot, 10000.0, device="cuda")
    m = 1.25
    for far, kind in ((0, torch.int64), (1 << 22, torch.int32), (1 << 40, torch.int64)):
        pos = (torch.arange(t, device="cuda") * 3 + far).to(kind)
        y = ops.rotary(x, pos, f, interleaved=interleaved, mscale=m, transpose=transpose)
        want = R.rotate(x, pos, f, interleaved, m, transpose)
        # (64-bit angles themselves are off by far * 2^-53; both sides)
        slack = R.rotate_slack(x, f, interleaved, m)
        _close(y, want, R.half_step(dtype, want) + slack * (1 + far * 2.0 ** -31), f"far {far}")
        assert torch.equal(y[..., rot:], x[..., rot:])


def test_rotary_strides_in_place_and_inverse(cuda_device):
    from unified_cache_management_b200 import ops
    g = _gen(1)
    f, _ = ops.rotary_frequencies(64, device="cuda")
    for off in (0, 8, 3):                       # 16-byte aligned rows, and rows that are not
        packed = _randn((37, 11 * 128 + 8), g, BF)
        x = packed.as_strided((37, 5, 128), (packed.stride(0), 128, 1), off)
        pos = torch.randint(0, 100000, (37,), device="cuda", generator=g)
        keep = packed.clone()
        plain = ops.rotary(x.contiguous(), pos, f)
        y = ops.rotary(x, pos, f)
        want = R.rotate(x, pos, f)
        _close(y, want, R.half_step(BF, want) + R.rotate_slack(x, f), f"offset {off}")
        assert torch.equal(packed, keep) and (off == 3 or torch.equal(y, plain))
        assert ops.rotary(x, pos, f, out=x) is x and torch.equal(x, y)
        untouched = torch.ones_like(packed, dtype=torch.bool)
        untouched.as_strided((37, 5, 128), x.stride(), off)[:] = False
        assert torch.equal(packed[untouched], keep[untouched])
    x = _randn((50, 4, 128), g, BF)
    pos = torch.arange(50, device="cuda")
    back = ops.rotary(ops.rotary(x, pos, f), pos, f, transpose=True)
    # two roundings of each of a pair's elements
    pair = R.rotate_slack(x, f) / (6 * 2.0 ** -22)
    _close(back, x.double(), pair * 2.0 ** -8 * 2 + R.half_step(BF, x.double()))


def test_rotary_gradient_against_differences(cuda_device):
    """<transposed(dy), dx> is the change of <y, dy>: the map is linear, so a finite step gives the derivative exactly, but
    for the roundings of both results (half a step of each element)."""
    from unified_cache_management_b200 import ops
    g = _gen(2)
    for inter in (False, True):
        f, _ = ops.rotary_frequencies(48, device="cuda")
        x, dx, dy = (_randn((13, 3, 64), g, FP) for _ in range(3))
        pos = torch.randint(0, 5000, (13,), device="cuda", generator=g)
        kw = dict(interleaved=inter, mscale=1.5)
        grad = ops.rotary(dy, pos, f, transpose=True, **kw)
        _close(grad, R.rotate(dy, pos, f, inter, 1.5, True), R.half_step(FP, R.rotate(dy, pos, f, inter, 1.5, True)) + R.rotate_slack(dy, f, inter, 1.5))
        one, two = (x.double() + dx.double() * 0.5).half(), (x.double() - dx.double() * 0.5).half()
        step = one.double() - two.double()
        change = ((ops.rotary(one, pos, f, **kw).double() - ops.rotary(two, pos, f, **kw).double()) * dy.double()).sum()
        room = sum((R.half_step(FP, R.rotate(z, pos, f, inter, 1.5)) + R.rotate_slack(z, f, inter, 1.5)).mul(dy.double().abs()).sum() for z in (one, two))
        room = room + ((R.half_step(FP, grad.double()) + R.rotate_slack(dy, f, inter, 1.5)) * step.abs()).sum() * 2
        assert abs(float(change - (grad.double() * step).sum())) <= float(room)


def test_rotary_empty(cuda_device):
    from unified_cache_management_b200 import ops
    f, _ = ops.rotary_frequencies(64, device="cuda")
    y = ops.rotary(torch.empty((0, 4, 64), dtype=BF, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), f)
    assert y.shape == (0, 4, 64)


# ---------------------------------------------------------------------------------------------- append
def _caches(nb, bs, h, d, kind, g, layout="NTHD"):
    """K and V caches of given layout with some content; e4m3 ones with scales."""
    shape = (2, nb, bs, h, d) if layout == "NTHD" else (2, nb, h, bs, d)
    x = _randn(shape, g, torch.float32, 80.0 if kind == E4M3 else 1.0).clamp(-448, 448).to(kind)
    if layout != "NTHD":
        x = x.transpose(2, 3)
    scales = (None, None)
    if kind == E4M3:
        scales = tuple(torch.pow(2.0, torch.randint(-9, -5, (nb, h), device="cuda", generator=g).float()) for _ in range(2))
    return x[0], x[1], scales[0], scales[1]


def _check_append(cache, scale, want, name):
    value, wscale, room = want
    if wscale is None:
        _close(cache, value, room, name)
        return
    assert torch.equal(scale.double(), wscale), name
    got = cache.double() * scale.double()[:, None, :, None]
    got[(scale == 0)[:, None, :, None].expand_as(got) & ~cache.double().isnan()] = 0.0
    known = ~value.isnan()
    _close(got[known], value[known], room[known], name)


def _do_append(seed, slots, nb, bs, h, d, kind, dtype, rot=0, inter=False, hq=0, layout="NTHD", index=torch.int64, magnitude=1.0,
               packed=True, change=None):
    from unified_cache_management_b200 import ops
    g = _gen(seed)
    t = len(slots)
    kc, vc, ks, vs = _caches(nb, bs, h, d, E4M3 if kind == "e4m3" else dtype, g, layout)
    if packed:
        qkv = _randn((t, max(hq, 1) + 2 * h, d), g, dtype, magnitude)
        q, k, v = qkv.split([max(hq, 1), h, h], 1)
    else:
        q, k, v = (_randn((t, n, d), g, dtype, magnitude) for n in (max(hq, 1), h, h))
    if change is not None:
        change(k, v, ks, vs)
    slot = torch.tensor(slots, dtype=index, device="cuda")
    kw, pos, f, m = {}, None, None, 1.0
    if rot:
        f, _ = ops.rotary_frequencies(rot, device="cuda")
        pos, m = torch.randint(0, 200000, (t,), device="cuda", generator=g), 1.1
        kw = dict(positions=pos, inv_freq=f, mscale=m, interleaved=inter, k_out=torch.zeros_like(k))
        if hq:
            kw["q"] = q
    k64 = R.rotate(k, pos, f, inter, m) if rot else k.double()
    before = (kc.clone(), vc.clone(), None if ks is None else ks.clone(), None if vs is None else vs.clone())
    want_k, want_v = R.append(k64, slot, before[0], before[2]), R.append(v.double(), slot, before[1], before[3])
    out = ops.kv_append(k, v, slot, kc, vc, k_scale=ks, v_scale=vs, **kw)
    torch.cuda.synchronize()
    if rot:
        slack = R.rotate_slack(k, f, inter, m)
        live = [i for i, s in enumerate(slots) if 0 <= s < nb * bs]
        for i in live:
            s = slots[i]
            want_k[2][s // bs, s % bs] += slack[i]
        _close(kw["k_out"], k64, R.half_step(dtype, k64) + slack, "k_out")
        if hq:
            q64 = R.rotate(q, pos, f, inter, m)
            _close(out, q64, R.half_step(dtype, q64) + R.rotate_slack(q, f, inter, m), "q_out")
    _check_append(kc, ks, want_k, "keys")
    _check_append(vc, vs, want_v, "values")
    # blocks without a new row are as they were, bit for bit
    still = torch.ones(nb, dtype=torch.bool)
    still[[s // bs for s in slots if 0 <= s < nb * bs]] = False
    for new, old in ((kc, before[0]), (vc, before[1])):
        assert torch.equal(new[still].contiguous().view(torch.uint8), old[still].contiguous().view(torch.uint8))
    return kc, vc, ks, vs


@pytest.mark.parametrize("kind", ["e4m3", "same"])
@pytest.mark.parametrize("h,d,bs,rot,dtype,inter", [(8, 128, 128, 128, BF, False), (2, 64, 16, 32, FP, True), (1, 128, 24, 0, BF, False),
                                                    (3, 80, 7, 80, FP, False), (2, 256, 128, 256, BF, False), (5, 16, 1, 16, BF, True),
                                                    (1, 512, 64, 512, BF, False)])
def test_append_decode_and_chunks(cuda_device, kind, h, d, bs, rot, dtype, inter):
    hq = 4 * h if rot else 0
    n = 12
    # one token per request, somewhere in its block (row 0 among them), a padded one and one out of range
    slots = [b * bs + (b * 5) % bs for b in range(n)]
    _do_append(1, slots + [-1, n * bs + 3], n, bs, h, d, kind, dtype, rot, inter, hq)
    # chunks that begin inside a block, run over several, and end inside one; blocks in no order
    perm = [5, 2, 9, 0, 7, 3, 11, 1, 10, 4, 8, 6]
    first = bs // 2
    slots = [perm[p // bs] * bs + p % bs for p in range(first, first + 3 * bs + bs // 3 + 1)]
    slots += [perm[6 + p // bs] * bs + p % bs for p in range(0, bs + 1)]
    _do_append(2, slots + [-1] * 3, n, bs, h, d, kind, dtype, rot, inter, hq, layout="NHTD", index=torch.int32, packed=False)


@pytest.mark.parametrize("kind", ["e4m3", "same"])
def test_append_order_and_duplicates(cuda_device, kind):
    """Tokens of a block scattered over the list, and slots listed twice: the later token is stored, whatever runs first."""
    bs, nb, h, d = 16, 40, 2, 64
    gen = torch.Generator().manual_seed(4)
    slots = torch.randint(0, nb * bs, (700,), generator=gen).tolist()
    slots[100:140] = [7 * bs + 3] * 40
    a = _do_append(5, slots, nb, bs, h, d, kind, BF, 64, False, 4)
    b = _do_append(5, slots, nb, bs, h, d, kind, BF, 64, False, 4)
    for x, y in zip(a, b):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # more tokens of one block than the walk's list holds
    _do_append(6, [3 * bs + i % 13 for i in range(2500)], nb, bs, h, d, kind, BF)
    # a large call in chunks of 128
    perm = torch.randperm(1200, generator=gen)
    slots = (perm[:, None] * bs + torch.arange(bs)).reshape(-1).tolist()
    _do_append(7, slots[5:16000], 1200, bs, 8, 32, kind, BF, 32, False, 8)


def test_append_scale_rules(cuda_device):
    from unified_cache_management_b200 import ops
    bs, h, d = 32, 2, 64
    dev = "cuda"

    def fresh():
        kc = torch.zeros((3, bs, h, d), dtype=E4M3, device=dev)
        return kc, kc.clone(), torch.zeros((3, h), device=dev), torch.zeros((3, h), device=dev)

    def put(state, x, slots):
        x = x.to(BF)
        ops.kv_append(x, x, torch.tensor(slots, device=dev), state[0], state[1], k_scale=state[2], v_scale=state[3])

    s = fresh()
    one = torch.ones((1, h, d), device=dev)
    put(s, one * 448.0, [0])                                  # exactly the largest code
    assert s[2][0].tolist() == [1.0, 1.0] and (s[0][0, 0].float() == 448).all()
    put(s, one * 450.0, [1])                                  # one bf16 step above: the scale doubles, the row moves
    assert s[2][0].tolist() == [2.0, 2.0]
    assert (s[0][0, 0].float() == 224).all() and (s[0][0, 1].float() == 224).all()
    put(s, one * 1e-3, [2])                                   # small values do not shrink it
    assert s[2][0].tolist() == [2.0, 2.0]
    put(s, one * 1e-3, [0])                                   # row 0 starts the block anew
    need = R.scale_for(float(torch.tensor(1e-3).to(BF)))
    assert s[2][0].tolist() == [need, need] and (s[0][0, 1].float() == 224).all()
    # a block that held nothing but zeros has scale 0; its codes, whatever they are, stand for 0 and become 0
    s = fresh()
    s[0][1] = torch.full((bs, h, d), 3.0, device=dev).to(E4M3)
    put(s, one * 7.0, [bs + 4])
    assert (s[0][1, 5].float() == 0).all() and (s[0][1, 4].float() == 7.0 / R.scale_for(7.0)).all()
    put(s, one * 0.0, [2 * bs])
    assert s[2][2].tolist() == [0.0, 0.0] and (s[0][2, 0].float() == 0).all()
    # values that are not finite: NaN codes, no say in the scale
    x = one.clone()
    x[..., 0], x[..., 1], x[..., 2] = math.inf, math.nan, -math.inf
    put(s, x, [2 * bs])
    assert s[2][2].tolist() == [R.scale_for(1.0)] * 2
    assert s[0][2, 0, :, :3].float().isnan().all() and (s[0][2, 0, :, 3:].float() == 1.0 / R.scale_for(1.0)).all()
    # largest and smallest bf16 values
    big = float(torch.finfo(BF).max)
    put(s, one * big, [2 * bs])
    assert s[2][2].tolist() == [R.scale_for(big)] * 2 and s[0][2, 0].float().isfinite().all()
    tiny = 2.0 ** -126
    put(s, one * tiny, [2 * bs])
    assert s[2][2].tolist() == [2.0 ** -126] * 2 and (s[0][2, 0].float() == 1).all()


def test_append_growth_of_old_blocks(cuda_device):
    """Scales of every size before, values up to 2^6 times larger or smaller, per head: codes move by exponents."""
    def change(k, v, ks, vs):
        k *= torch.pow(2.0, torch.randint(-6, 7, k.shape[1:2], device="cuda")).to(k.dtype)[None, :, None]
        ks[0] = 0.0
        vs[1] = 3.1                                            # a scale that is no power of two
    for seed in range(3):
        _do_append(20 + seed, [b * 32 + 5 + b for b in range(20)], 21, 32, 4, 64, "e4m3", BF, change=change)


# ---------------------------------------------------------------------------------------------- attention
def _case(seed, lens, qs, hq, hkv, d, bs, kind, dtype, per_head=False, layout="NTHD", spare=3, q_scale=1.5):
    g = _gen(seed)
    b = len(lens)
    per = [-(-n // bs) for n in lens]
    nb, mb = sum(per) + spare, max(1, max(per) + 2)
    kc, vc, ks, vs = _caches(nb, bs, hkv, d, E4M3 if kind == "e4m3" else dtype, g, layout)
    lists = hkv if per_head else 1
    table = torch.full((b, lists, mb), -7, dtype=torch.int32, device="cuda")   # entries that nothing may read as blocks
    for h in range(lists):
        perm = torch.randperm(nb, device="cuda", generator=g).int()
        at = 0
        for i, n in enumerate(per):
            table[i, h, :n] = perm[at:at + n]
            at += n
    table = table if per_head else table[:, 0].contiguous()
    start = torch.tensor([sum(qs[:i]) for i in range(b + 1)], dtype=torch.int32, device="cuda")
    q = _randn((sum(qs), hq, d), g, dtype, q_scale)
    return dict(q=q, k_cache=kc, v_cache=vc, table=table, seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                k_scale=ks, v_scale=vs, query_start=start), max(qs + [0])


def _attend(c, mq, **kw):
    from unified_cache_management_b200 import ops
    return ops.paged_attention(c["q"], c["k_cache"], c["v_cache"], c["table"], c["seq_lens"], k_scale=c["k_scale"],
                               v_scale=c["v_scale"], query_start=c["query_start"], max_query_len=mq, want_lse=True, **kw)


def _check(c, mq, causal=True, scale=None, **kw):
    out, lse = _attend(c, mq, causal=causal, scale=scale, **kw)
    torch.cuda.synchronize()
    want, wlse, room, lroom = R.attention(c["q"], c["k_cache"], c["v_cache"], c["table"], c["seq_lens"], k_scale=c["k_scale"],
                                          v_scale=c["v_scale"], query_start=c["query_start"], causal=causal, scale=scale)
    inside = ~wlse.isnan()
    _close(out[inside], want[inside], room[inside], "out")
    _close(lse[inside], wlse[inside], lroom[inside], "lse")
    return out, lse


LENS = [0, 1, 15, 16, 17, 127, 128, 129, 1000, 2049]


@pytest.mark.parametrize("kind", ["e4m3", "same"])
@pytest.mark.parametrize("hq,hkv,d,bs,dtype", [(32, 8, 128, 128, BF), (8, 8, 64, 16, FP), (5, 1, 128, 24, FP), (16, 2, 64, 64, BF),
                                               (16, 1, 128, 32, BF), (40, 2, 128, 7, BF), (4, 4, 128, 1, FP)])
def test_attention_decode(cuda_device, kind, hq, hkv, d, bs, dtype):
    c, mq = _case(d + hq, LENS, [1] * len(LENS), hq, hkv, d, bs, kind, dtype, layout="NHTD" if hq == 40 else "NTHD")
    a = _check(c, mq)
    b = _attend(c, mq)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c["query_start"], plain = None, a
    from unified_cache_management_b200 import ops
    out = ops.paged_attention(c["q"], c["k_cache"], c["v_cache"], c["table"], c["seq_lens"], k_scale=c["k_scale"], v_scale=c["v_scale"])
    assert torch.equal(out, plain[0])


@pytest.mark.parametrize("kind,d", [("e4m3", 128), ("same", 64)])
@pytest.mark.parametrize("qs", [[2, 4, 1, 3, 7], [1, 17, 0, 64, 33], [5, 200, 129, 3, 300]])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_several_queries(cuda_device, kind, d, qs, causal):
    lens = [300, 2, 77, 64, 1025]                             # more queries than tokens among them: rows that see nothing
    for hq, hkv in ((8, 2), (3, 3), (16, 1)):
        c, mq = _case(sum(qs) + hq, lens, qs, hq, hkv, d, 32, kind, BF if d == 128 else FP)
        _check(c, mq, causal=causal, scale=0.07)


@pytest.mark.parametrize("kind", ["e4m3", "same"])
def test_attention_long_and_per_head(cuda_device, kind):
    c, mq = _case(3, [70001], [1], 8, 2, 128, 16, kind, BF)   # one request over the whole GPU
    _check(c, mq)
    c, mq = _case(4, [513, 2048, 40, 700], [1] * 4, 16, 4, 128, 64, kind, FP, per_head=True)
    _check(c, mq)
    c, mq = _case(5, [5000, 900], [3, 600], 8, 4, 128, 128, kind, BF, per_head=True)
    _check(c, mq)
    c, mq = _case(6, [17 + 3 * i for i in range(700)], [1] * 700, 4, 1, 64, 16, kind, BF)   # more requests than CTAs
    _check(c, mq)


@pytest.mark.parametrize("kind,dtype", [("e4m3", BF), ("same", BF), ("same", FP)])
@pytest.mark.parametrize("nq", [1, 5, 150])
def test_attention_masked_places(cuda_device, kind, dtype, nq):
    """NaN and infinities behind a request's length and above the diagonal stay there; visible ones show."""
    lens = [max(70, nq + 3), max(33, nq), nq]
    c, mq = _case(nq, lens, [nq] * 3, 8, 2, 128, 32, kind, dtype)
    bs = 32
    for name in ("k_cache", "v_cache"):
        cache = c[name]
        seen = torch.zeros(cache.shape[:2], dtype=torch.bool, device="cuda")
        for i, n in enumerate(lens):
            for p in range(n):
                seen[c["table"][i, p // bs], p % bs] = True
        x = cache.float()
        x[~seen] = math.nan
        # the last token's value: above the diagonal for all queries but the last
        if name == "v_cache":
            for i, n in enumerate(lens):
                x[c["table"][i, (n - 1) // bs], (n - 1) % bs, :, 5] = math.nan if kind == "e4m3" else (math.inf if i else -math.inf)
        cache.copy_(x.to(cache.dtype))
    out, lse = _attend(c, mq)
    want, wlse, room, lroom = R.attention(c["q"], c["k_cache"], c["v_cache"], c["table"], c["seq_lens"], k_scale=c["k_scale"],
                                          v_scale=c["v_scale"], query_start=c["query_start"])
    last = c["query_start"][1:].long() - 1
    assert not out[last, :, 5].isfinite().any()
    want[last, :, 5] = out[last, :, 5].double()
    _close(out, want, room.nan_to_num(0, 0, 0), "out")
    _close(lse, wlse, lroom, "lse")


def test_attention_extreme_scales(cuda_device):
    """Value scales that differ by 2^20 from block to block, scales of 0, large and tiny ones."""
    for lo, hi in ((-20, 0), (-90, -60), (60, 90)):
        c, mq = _case(50, [400, 90], [1, 3], 8, 2, 64, 16, "e4m3", BF)
        for i, v in enumerate(torch.linspace(lo, hi, c["v_scale"].shape[0]).round().tolist()):
            c["v_scale"][i] = 2.0 ** v
        c["v_scale"][3] = 0.0
        c["k_scale"][5] = 0.0
        c["k_scale"][6] = 0.37
        out, lse = _attend(c, mq)
        want, wlse, room, lroom = R.attention(c["q"], c["k_cache"], c["v_cache"], c["table"], c["seq_lens"], k_scale=c["k_scale"],
                                              v_scale=c["v_scale"], query_start=c["query_start"])
        # weights are counted from the largest value scale: below 2^-28 of the largest product the step is 2^-39 of it
        top = 448.0 * float(c["v_scale"].max()) * 400 * 2.0 ** -38
        _close(out, want, room + top, "out")
        _close(lse, wlse, lroom, "lse")
    # queries of every size
    for size in (1e-30, 1e-3, 1e4):
        c, mq = _case(51, [300], [1], 4, 1, 128, 64, "e4m3", BF, q_scale=size)
        c["k_scale"] *= min(1.0, 1.0 / size)
        _check(c, mq)


def test_attention_bad_blocks_rows_outside_and_strides(cuda_device):
    from unified_cache_management_b200 import ops
    for kind in ("e4m3", "same"):
        c, mq = _case(9, [100, 64, 50], [2, 1, 20], 8, 2, 128, 16, kind, BF)
        c["table"][0, 2] = 10 ** 6
        c["table"][1, 0] = -1
        ws = ops.new_attention_workspace(128, "cuda")
        _check(c, mq, workspace=ws)
        assert ops.workspace_status(ws) == 1
    # a padded batch: rows of q and out behind the last request and in front of the first are left alone
    c, _ = _case(10, [40, 90], [3, 2], 8, 2, 128, 16, "e4m3", FP)
    want, wlse = _attend(c, 3)
    big_q = torch.full((12, 10, 128), math.nan, dtype=FP, device="cuda")
    big_o, big_l = torch.full_like(big_q, 7.0), torch.full((12, 8), 9.0, device="cuda")
    big_q[4:9, 1:9] = c["q"]
    out, lse = ops.paged_attention(big_q[:, 1:9], c["k_cache"], c["v_cache"], c["table"], c["seq_lens"], k_scale=c["k_scale"],
                                   v_scale=c["v_scale"], query_start=c["query_start"] + 4, max_query_len=3, out=big_o[:, 1:9], lse=big_l)
    assert torch.equal(out[4:9], want) and torch.equal(lse[4:9], wlse)
    big_o[4:9, 1:9] = 7.0
    big_l[4:9] = 9.0
    assert (big_o == 7.0).all() and (big_l == 9.0).all()
    # lengths beyond the table are cut to it
    c, _ = _case(11, [64, 32], [1, 1], 4, 2, 64, 16, "same", BF)
    c["table"] = c["table"][:, :2].contiguous()
    _check(c, 1)
    # nothing to do
    z = torch.zeros
    e = ops.paged_attention(z((0, 4, 64), dtype=BF, device="cuda"), c["k_cache"], c["v_cache"], z((0, 3), dtype=torch.int32, device="cuda"),
                            z((0,), dtype=torch.int32, device="cuda"))
    assert e.shape == (0, 4, 64)


def test_attention_streams_and_graphs(cuda_device):
    """Two captured graphs with a workspace each, replayed side by side and after the lengths changed."""
    from unified_cache_management_b200 import ops
    c, mq = _case(12, [900, 3000, 50], [1] * 3, 8, 2, 128, 16, "e4m3", BF)
    full = c["seq_lens"].clone()
    outs, graphs, streams, wss = [], [], [], []
    for i in range(2):
        st = torch.cuda.Stream()
        ws, out = ops.new_attention_workspace(128, "cuda"), torch.empty_like(c["q"])
        lse = torch.empty((3, 8), device="cuda")
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            _attend(c, mq, workspace=ws, out=out, lse=lse)
        outs.append((out, lse)), graphs.append(gr), streams.append(st), wss.append(ws)
    for cut in (0, 333, 2, 0):
        c["seq_lens"].copy_((full - cut).clamp(min=0))
        torch.cuda.synchronize()
        for _ in range(3):
            for st, gr in zip(streams, graphs):
                with torch.cuda.stream(st):
                    gr.replay()
        torch.cuda.synchronize()
        want, wlse = _attend(c, mq)
        for out, lse in outs:
            assert torch.equal(out, want) and torch.equal(lse, wlse)
    for ws in wss:
        assert int(ws[:2304].count_nonzero()) == 0              # header and counters are back at zero


@pytest.mark.parametrize("kind,dtype", [("e4m3", BF), ("e4m3", FP), ("same", BF), ("same", FP)])
@pytest.mark.parametrize("hq,hkv,d,bs,layout", [(10, 5, 64, 16, "NTHD"), (9, 9, 128, 48, "NHTD"), (12, 12, 64, 7, "NTHD"), (6, 1, 128, 128, "NHTD"),
                                                (300, 1, 64, 32, "NTHD")])
def test_attention_many_rows(cuda_device, kind, dtype, hq, hkv, d, bs, layout):
    """Every pair of types; odd head counts, blocks that end inside a tile of 128 tokens, a block listed twice, lengths around
    a tile's end, and a batch in which one request has many queries and the others one."""
    qs = [1, 65, 1, 9, 0, 30] if hq < 300 else [1, 1, 2, 1, 0, 1]
    c, mq = _case(hq + d, [257, 129, 128, 9, 40, 127], qs, hq, hkv, d, bs, kind, dtype, layout=layout)
    c["table"][0, 1] = c["table"][0, 0]
    for causal in (True, False):
        a = _check(c, mq, causal=causal)
        b = _attend(c, mq, causal=causal)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("kind", ["e4m3", "same"])
@pytest.mark.parametrize("hq,hkv,d,bs", [(35, 5, 128, 16), (18, 9, 64, 32), (60, 12, 128, 48), (17, 17, 64, 5), (48, 3, 128, 16)])
def test_attention_decode_head_counts(cuda_device, kind, hq, hkv, d, bs):
    """Head counts that do not divide a block of eight warps, groups that are no multiple of four, a block listed twice."""
    c, mq = _case(hq, [1, 700, 31, 96, 5000], [1] * 5, hq, hkv, d, bs, kind, BF)
    c["table"][1, 2] = c["table"][1, 0]
    _check(c, mq)


def test_attention_extreme_scales_many_rows(cuda_device):
    """Scales that differ by more than fp16 holds within a tile, scales of 0 and no power of two, tiles of equal ones.  A weight
    is counted from 2^(6 - E), 2^E at most twice the largest value scale, in fp16, whose smallest step is 2^-24: each of the
    n tokens adds at most 448 * 2 * scale * 2^-25 * 2^-6, over a sum of weights of 1 or more (the reference is a score)."""
    for lo, hi in ((-20, 0), (-90, -60), (60, 90), (-9, 0), (0, 0)):
        c, mq = _case(52, [400, 90], [33, 20], 8, 2, 64, 16, "e4m3", BF)
        for i, v in enumerate(torch.linspace(lo, hi, c["v_scale"].shape[0]).round().tolist()):
            c["v_scale"][i] = 2.0 ** v
        if lo != hi:
            c["v_scale"][3] = 0.0
            c["k_scale"][5] = 0.0
        if lo == -20:
            c["k_scale"][6] = 0.37
        out, lse = _attend(c, mq)
        want, wlse, room, lroom = R.attention(c["q"], c["k_cache"], c["v_cache"], c["table"], c["seq_lens"], k_scale=c["k_scale"],
                                              v_scale=c["v_scale"], query_start=c["query_start"])
        _close(out, want, room + 448.0 * float(c["v_scale"].max()) * 400 * 2.0 ** -30, "out")
        _close(lse, wlse, lroom, "lse")


@pytest.mark.parametrize("kind", ["e4m3", "same"])
@pytest.mark.parametrize("bs", [16, 24])
def test_far_blocks(cuda_device, kind, bs):
    """The last blocks of a cache of more than 2^32 bytes give what they give in a small one, bit for bit."""
    from unified_cache_management_b200 import ops
    h, d, dt = 2, 128, E4M3 if kind == "e4m3" else BF
    qs = [1, 3, 30]
    c, mq = _case(60, [300, 77, 129], qs, 8, h, d, bs, kind, BF)
    nb = c["k_cache"].shape[0]
    many = (1 << 32) // (bs * h * d * dt.itemsize) + 2 * nb
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    far = many - nb
    big = dict(c)
    for name in ("k_cache", "v_cache"):
        big[name] = torch.empty((many, bs, h, d), dtype=dt, device="cuda")
        big[name][far:] = c[name]
    for name in ("k_scale", "v_scale"):
        if c[name] is not None:
            big[name] = torch.ones((many, h), device="cuda")
            big[name][far:] = c[name]
    big["table"] = torch.where(c["table"] >= 0, c["table"] + far, c["table"])
    one = [0, 1, 4]                                            # the requests' first queries, as a decode step
    for x, y in zip(_attend(big, mq), _attend(c, mq)):
        assert torch.equal(x, y)
    for z in (big, c):
        z["q"], z["query_start"] = z["q"][one].contiguous(), None
    for x, y in zip(_attend(big, 1), _attend(c, 1)):
        assert torch.equal(x, y)
    g = _gen(61)
    slots = torch.randint(0, nb * bs, (50,), device="cuda", generator=g)
    k, v = _randn((50, h, d), g, BF, 3.0), _randn((50, h, d), g, BF, 0.1)
    for z, first in ((big, far * bs), (c, 0)):
        ops.kv_append(k, v, slots + first, z["k_cache"], z["v_cache"], k_scale=z["k_scale"], v_scale=z["v_scale"])
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        if c[name] is not None:
            assert torch.equal(big[name][far:].view(torch.uint8), c[name].view(torch.uint8)), name


def test_append_slots_beyond_31_bits(cuda_device):
    """Slot numbers above 2^31, in a cache whose rows overlap (block b's row r is row b + r of the memory)."""
    from unified_cache_management_b200 import ops
    nb, bs, d = (1 << 21) + 8, 1024, 16
    mem = [torch.zeros((nb + bs, d), dtype=BF, device="cuda") for _ in range(2)]
    kc, vc = (m.as_strided((nb, bs, 1, d), (d, d, d, 1)) for m in mem)
    at = [(nb - 1, 5), (nb - 4, 0), (7, 3), (1 << 20, 1000), (nb - 3, 1)]
    slots = torch.tensor([b * bs + r for b, r in at] + [nb * bs], device="cuda")
    x = torch.arange(1.0, 7.0, device="cuda")[:, None, None].expand(6, 1, d).to(BF).contiguous()
    ops.kv_append(x, -x, slots, kc, vc)
    for i, (b, r) in enumerate(at[:3]):
        assert (mem[0][b + r] == i + 1).all() and (mem[1][b + r] == -i - 1).all()
    assert int(mem[0].count_nonzero()) == 5 * d


@pytest.mark.parametrize("kind", ["e4m3", "same"])
def test_step_captured_and_replayed(cuda_device, kind):
    """Rotation, append and attention captured into one graph on a stream of its own; replayed with other positions, slots and
    lengths, it leaves what the eager calls leave."""
    from unified_cache_management_b200 import ops
    g = _gen(70)
    b, hq, h, d, bs, nb = 3, 8, 2, 128, 16, 40
    kc, vc, ks, vs = _caches(nb, bs, h, d, E4M3 if kind == "e4m3" else BF, g)
    f, _ = ops.rotary_frequencies(64, device="cuda")
    table = torch.arange(36, device="cuda").reshape(3, 12).int()
    qkv = _randn((b, hq + 2 * h, d), g, BF)
    pos, slot = torch.zeros(b, dtype=torch.int64, device="cuda"), torch.zeros(b, dtype=torch.int64, device="cuda")
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    ws, out, lse, extra = ops.new_attention_workspace(d, "cuda"), torch.zeros((b, hq, d), dtype=BF, device="cuda"), torch.zeros((b, hq), device="cuda"), torch.zeros_like(qkv)

    def step(kc, vc, ks, vs, ws, out, lse, extra):
        q, k, v = qkv.split([hq, h, h], 1)
        ops.rotary(qkv, pos, f, interleaved=True, out=extra)
        q = ops.kv_append(k, v, slot, kc, vc, k_scale=ks, v_scale=vs, positions=pos, inv_freq=f, q=q)
        ops.paged_attention(q, kc, vc, table, lens, k_scale=ks, v_scale=vs, workspace=ws, out=out, lse=lse)

    mine = [kc, vc, ks, vs, ws, out, lse, extra]
    other = [None if x is None else x.clone() for x in mine]
    slot.fill_(-1)                                             # (nothing is stored while the graph is captured)
    torch.cuda.synchronize()
    st, gr = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        step(*mine)
    for n in ((1, 30, 16), (2, 31, 17), (3, 0, 18), (140, 192, 19)):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        pos.copy_((lens - 1).long())
        slot.copy_(torch.where(lens > 0, table[torch.arange(b), (pos // bs).clamp(min=0)].long() * bs + pos % bs, -1))
        qkv.copy_(_randn(qkv.shape, g, BF))
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            gr.replay()
        torch.cuda.synchronize()
        step(*other)
        torch.cuda.synchronize()
        for x, y in zip(mine[:4] + mine[5:], other[:4] + other[5:]):
            assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_in_place_and_empty_tables(cuda_device):
    """Results over their own inputs; requests without a single block."""
    from unified_cache_management_b200 import ops
    g = _gen(80)
    f, _ = ops.rotary_frequencies(64, device="cuda")
    pos = torch.arange(300, device="cuda")
    for shape, inter in (((300, 40, 128), False), ((300, 2, 72), True)):
        x = _randn(shape, g, BF)
        want = ops.rotary(x, pos, f, interleaved=inter)
        y = x.clone()
        ops.rotary(y, pos, f, interleaved=inter, out=y)
        assert torch.equal(y, want)
    for qs in ([1, 1], [40, 3]):
        c, mq = _case(81, [5000, 60], qs, 8, 2, 128, 32, "e4m3", BF)
        want, _ = _attend(c, mq)
        q = c["q"].clone()
        c["q"] = q
        _attend(c, mq, out=q)
        assert torch.equal(q, want)
        c["table"] = torch.empty((2, 0), dtype=torch.int32, device="cuda")
        out, lse = _attend(c, mq)
        assert (out == 0).all() and (lse == -math.inf).all()


# ---------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("kind", ["e4m3", "same"])
def test_decode_step_from_append_to_attention(cuda_device, kind):
    """Prefill and two decode steps: rotate and append, hash the rotated keys, retrieve blocks per kv head, attend over the
    chosen blocks - against the 64-bit attention over the same blocks."""
    from unified_cache_management_b200 import ops
    g = _gen(77)
    dev, dt = cuda_device, BF
    b, hkv, grp, d, bs, nb, mb, k = 3, 2, 4, 128, 16, 100, 30, 6
    hq = hkv * grp
    kc = torch.zeros((nb, bs, hkv, d), dtype=E4M3 if kind == "e4m3" else dt, device=dev)
    vc = torch.zeros_like(kc)
    ks = vs = None
    if kind == "e4m3":
        ks, vs = torch.zeros((nb, hkv), device=dev), torch.zeros((nb, hkv), device=dev)
    codes = torch.zeros((nb, bs, hkv, 4), dtype=torch.int32, device=dev)
    proj = _randn((d, 128), g, dt)
    f, m = ops.rotary_frequencies(d, 500000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                                "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}, dev)
    table = torch.randperm(nb, device=dev, generator=g)[:b * mb].reshape(b, mb).int()
    lens = torch.tensor([200, 333, 97], device=dev)
    ws = ops.new_attention_workspace(d, dev)

    def slots_of(req, pos):
        return table[req, pos // bs].long() * bs + pos % bs

    req = torch.repeat_interleave(torch.arange(b, device=dev), lens)
    pos = torch.cat([torch.arange(int(n), device=dev) for n in lens])
    kn, vn = _randn((len(pos), hkv, d), g, dt), _randn((len(pos), hkv, d), g, dt)
    rotated = torch.empty_like(kn)
    slot = slots_of(req, pos)
    ops.kv_append(kn, vn, slot, kc, vc, k_scale=ks, v_scale=vs, positions=pos, inv_freq=f, mscale=m, k_out=rotated)
    ops.hash_encode_and_cache(rotated, slot, codes, proj)
    for _ in range(2):
        lens = lens + 1
        pos = lens - 1
        slot = slots_of(torch.arange(b, device=dev), pos)
        q, kn, vn = _randn((b, hq, d), g, dt, 1.5), _randn((b, hkv, d), g, dt), _randn((b, hkv, d), g, dt)
        rotated = torch.empty_like(kn)
        q = ops.kv_append(kn, vn, slot, kc, vc, k_scale=ks, v_scale=vs, positions=pos, inv_freq=f, mscale=m, q=q, k_out=rotated)
        q_codes = ops.hash_encode_decode_step(q, rotated, slot, codes, proj)
        r = ops.hamming_topk(codes, q_codes, table, lens.int(), k, reduce="sum", must_select=(0, -1))
        out, lse = ops.paged_attention(q, kc, vc, r.physical, r.new_seq_lens, k_scale=ks, v_scale=vs, workspace=ws, want_lse=True)
        torch.cuda.synchronize()
        want, wlse, room, lroom = R.attention(q, kc, vc, r.physical, r.new_seq_lens, k_scale=ks, v_scale=vs)
        _close(out, want, room, "out")
        _close(lse, wlse, lroom, "lse")
        assert ops.workspace_status(ws) == 0
