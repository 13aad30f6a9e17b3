"""GPU: corners of attention over the paged KV cache for many rows: value scales far apart, of 0 and at their floor, rows of
very small queries, whole items of 256 rows, and long runs of rows that see nothing."""
import math

import pytest
import torch

from tests import kv_reference as R
from tests.test_gpu_kv_operators import BF, FP, _attend, _case, _check, _close, _gen

pytestmark = pytest.mark.gpu


def _compare(c, mq, room_of, causal=True):
    """Against the 64-bit form; room_of: what the fp16 weights may add, per output row, beyond the usual room."""
    out, lse = _attend(c, mq, causal=causal)
    torch.cuda.synchronize()
    want, wlse, room, lroom = R.attention(c["q"], c["k_cache"], c["v_cache"], c["table"], c["seq_lens"], k_scale=c["k_scale"],
                                          v_scale=c["v_scale"], query_start=c["query_start"], causal=causal)
    _close(out, want, room + room_of, "out")
    _close(lse, wlse, lroom, "lse")


def _tile_blocks(c, i, tile, bs):
    """Blocks of request i's token tile (128 tokens)."""
    return c["table"][i, tile * 128 // bs:(tile + 1) * 128 // bs].long()


# A weight is counted from 2^(6 - E) in fp16, 2^E at most twice the largest value scale; half of fp16's smallest step is 2^-25: a
# token adds at most 448 * 2 * scale * 2^-25 * 2^-6 = 448 * scale * 2^-30, over a sum of weights of 1 or more.
def _fp16_room(scale, tokens):
    return 448.0 * scale * tokens * 2.0 ** -30


@pytest.mark.parametrize("exponent", [-13, -20, -30])
@pytest.mark.parametrize("nq", [33, 300])
def test_tiles_of_scale_zero(cuda_device, exponent, nq):
    """Whole tiles of 128 tokens whose value scales are all 0 (as the append leaves blocks of zeros), or whose blocks are all
    missing, at the start, in the middle and at the end of a request: the others' weights keep their bits.  Many tiles per
    CTA: at least as many items as SMs."""
    n, bs = 1024, 16
    b, h = (20, 8) if nq < 128 else (40, 16)
    c, mq = _case(90 - exponent, [n] * b, [nq] * b, h, h, 64, bs, "e4m3", BF)
    c["v_scale"][:] = 2.0 ** exponent
    for i, tiles in enumerate([(0,), (1,), (0, 1), (3,), (4,), (7,), (6, 7), (0, 4, 5), (2, 3, 6), ()] * (b // 10)):
        for t in tiles:
            c["v_scale"][_tile_blocks(c, i, t, bs)] = 0.0
        if i % 20 >= 15 and tiles:
            c["table"][i, tiles[0] * 8:tiles[0] * 8 + 8] = -1
    _compare(c, mq, _fp16_room(2.0 ** exponent, n))


@pytest.mark.parametrize("nq", [33, 300])
@pytest.mark.parametrize("exponents", [(0, -126), (60, -126, 0), (60, -90), (7, -126), (100, -20)])
def test_value_scales_far_apart(cuda_device, nq, exponents):
    """Tiles whose value scales differ by more than float32's exponents allow for in a product: a value scale has no say in
    the weights' sum."""
    n, bs = 1024, 16
    b, h = (20, 8) if nq < 128 else (40, 16)
    c, mq = _case(91, [n] * b, [nq] * b, h, h, 64, bs, "e4m3", FP if nq < 128 else BF)
    for i in range(b):
        for t in range(n // 128):
            c["v_scale"][_tile_blocks(c, i, t, bs)] = 2.0 ** exponents[(t + i) // (1 + i % 3) % len(exponents)]
    if max(exponents) > 7:
        c["q"] = c["q"].to(BF)                    # (fp16 results would overflow)
    _compare(c, mq, _fp16_room(2.0 ** max(exponents), n))


@pytest.mark.parametrize("nq", [33, 300])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_rows_of_tiny_queries(cuda_device, nq, dtype):
    """Rows whose score factor (a power of two of the row's size times the key scale) underflows, beside rows where it does
    not: every warp takes one way through a tile."""
    n, bs = 700, 16
    b, h = (20, 8) if nq < 128 else (40, 16)
    c, mq = _case(93, [n - 5 * i for i in range(b)], [nq] * b, h, h, 64, bs, "e4m3", dtype)
    tiny = 2.0 ** -125 if dtype == BF else 2.0 ** -24          # (the smallest fp16 value)
    c["q"][::7] = torch.where(c["q"][::7] > 0, tiny, -tiny).to(dtype)
    for i in range(b):
        for t in range(5):
            if (t + i) % 3 == 0:
                c["k_scale"][_tile_blocks(c, i, t, bs)] = 2.0 ** (-26 if dtype == BF else -126)
    _compare(c, mq, _fp16_room(float(c["v_scale"].max()), n))


@pytest.mark.parametrize("exponent", [-100, -110, -119, -126])
@pytest.mark.parametrize("b,h,g,nq", [(3, 2, 4, 1), (5, 2, 4, 4), (3, 2, 4, 30), (20, 8, 1, 33), (40, 16, 1, 300)])
def test_smallest_value_scales(cuda_device, exponent, b, h, g, nq):
    """Values down to the append's smallest scale, 2^-126.  Weights are counted from 2^14 (up to 16 rows) or 2^6 over the
    largest scale, as far as float32 holds that: from 2^126 over 1 at most.  So half of fp16's smallest step is 2^-25 of
    448 * 2^-126 for a token at least, or what it is for larger scales."""
    n = 1024
    c, mq = _case(92 + exponent, [n] * b, [nq] * b, h * g, h, 64, 16, "e4m3", BF)
    c["v_scale"][:] = 2.0 ** exponent
    room = max(_fp16_room(2.0 ** exponent, n), 448.0 * 2.0 ** -126 * n * 2.0 ** -25)
    _compare(c, mq, room)
    # one token with a weight 2^13 times the others' and nothing but zeros as its value: the result is the others'
    c["q"][:] = 1.125
    c["k_cache"].view(torch.uint8).zero_()
    c["k_scale"][:] = 1.0
    c["v_cache"].copy_(torch.full_like(c["v_cache"], 448.0, dtype=BF).to(c["v_cache"].dtype))
    first = c["table"][:, 0].long()
    c["k_cache"][first, 0] = torch.ones_like(c["k_cache"][first, 0], dtype=BF).to(c["k_cache"].dtype)
    c["v_cache"].view(torch.uint8)[first, 0] = 0
    _compare(c, mq, room)


def _whole_items(c, hq, hkv, lens, qs):
    """The rule by which a call takes whole items of 256 rows: at least four per CTA, none above a third of a CTA's share."""
    ctas = min(152, torch.cuda.get_device_properties(0).multi_processor_count)
    g = hq // hkv
    tiles = [-(-nq * g // 256) for nq in qs]
    units = [max(1, -(-n // 128)) + 4 for n in lens]
    total = sum(t * u for t, u in zip(tiles, units)) * hkv
    largest = max(u for u, nq in zip(units, qs) if nq > 0)
    return sum(tiles) * hkv >= 4 * ctas and 3 * largest * ctas <= total


@pytest.mark.parametrize("kind,dtype,d", [("e4m3", BF, 128), ("e4m3", FP, 64), ("e4m3", BF, 64), ("e4m3", FP, 128),
                                          ("same", BF, 128), ("same", BF, 64), ("same", FP, 128), ("same", FP, 64)])
@pytest.mark.parametrize("g,per_head,bs", [(1, True, 16), (4, False, 24), (8, True, 128)])
def test_whole_items(cuda_device, kind, dtype, d, g, per_head, bs):
    """Items of 256 rows, taken whole: both chains on rows of their own, tails of 128 rows or fewer, rows that see nothing,
    several query heads per kv head, lists per kv head."""
    h, b = 8, 56
    qs = [(260 + 37 * (i % 9)) // g - (i % 5 == 4) * (130 // g) for i in range(b)]
    lens = [qs[i] + (i * 53) % 400 if i % 7 else qs[i] - 30 // g for i in range(b)]
    c, mq = _case(d + g, lens, qs, h * g, h, d, bs, kind, dtype, per_head=per_head)
    assert _whole_items(c, h * g, h, lens, qs)
    for causal in (True, False):
        a = _check(c, mq, causal=causal)
        b2 = _attend(c, mq, causal=causal)
        assert torch.equal(a[0], b2[0]) and torch.equal(a[1], b2[1])


@pytest.mark.parametrize("kind,dtype", [("e4m3", BF), ("e4m3", FP), ("same", BF), ("same", FP)])
def test_whole_items_masked_places(cuda_device, kind, dtype):
    """NaN and infinities behind a length and above the diagonal, block ids out of range, in whole items."""
    from unified_cache_management_b200 import ops
    h, b, bs, d = 8, 64, 32, 64
    qs = [290 - (i % 4) * 10 for i in range(b)]
    lens = [q + (i * 31) % 150 for i, q in enumerate(qs)]
    c, mq = _case(7, lens, qs, h, h, d, bs, kind, dtype)
    assert _whole_items(c, h, h, lens, qs)
    # positions of each cache row: the request and token that it holds
    token = torch.full(c["k_cache"].shape[:2], 1 << 30, device="cuda")
    first = torch.full_like(token, 0)
    for i, n in enumerate(lens):
        p = torch.arange(n, device="cuda")
        blk = c["table"][i, p // bs].long()
        token[blk, p % bs] = p
        first[blk, p % bs] = n - qs[i]                         # tokens that all of the request's queries see
    hidden = token == 1 << 30
    for name in ("k_cache", "v_cache"):
        x = c[name].float()
        x[hidden] = math.nan
        c[name].copy_(x.to(c[name].dtype))
    odd = (token >= first + 5) & (token % 61 == 7) & ~hidden   # above the diagonal of the first queries at least
    x = c["v_cache"].float()
    x[odd, :, 3] = math.nan
    if kind == "same":
        x[odd, :, 5] = math.inf
    c["v_cache"].copy_(x.to(c["v_cache"].dtype))
    c["table"][3, 1], c["table"][11, 2] = -5, 1 << 20
    ws = ops.new_attention_workspace(d, "cuda")
    out, lse = _attend(c, mq, workspace=ws)
    assert ops.workspace_status(ws) == 1
    want, wlse, room, lroom = R.attention(c["q"], c["k_cache"], c["v_cache"], c["table"], c["seq_lens"], k_scale=c["k_scale"],
                                          v_scale=c["v_scale"], query_start=c["query_start"])
    clean = [j for j in range(d) if j not in (3, 5)]
    _close(out[..., clean], want[..., clean], room[..., clean], "out")
    _close(lse, wlse, lroom, "lse")
    # the odd columns: not finite exactly where the row sees such a token
    for j in (3, 5) if kind == "same" else (3,):
        assert torch.equal(out[..., j].isfinite(), want[..., j].isfinite())
        fine = want[..., j].isfinite()
        assert fine.any() and not fine.all()
        _close(out[..., j][fine], want[..., j][fine], room[..., j][fine], "out")


@pytest.mark.parametrize("d,dtype", [(64, FP), (128, BF)])
def test_whole_items_scales(cuda_device, d, dtype):
    """Scales in whole items: equal within a tile, powers of two that fold into the codes, too far apart for that, no powers
    of two, zeros."""
    h, b, bs = 8, 40, 16
    qs, lens = [280] * b, [400 + (i * 37) % 300 for i in range(b)]
    c, mq = _case(8, lens, qs, h, h, d, bs, "e4m3", dtype)
    g = _gen(9)
    nb = c["v_scale"].shape[0]
    for name, base in (("k_scale", -7), ("v_scale", -6)):
        wide = torch.randint(base - 18, base + 1, (nb, h), device="cuda", generator=g).float()
        near = torch.randint(base - 6, base + 1, (nb, h), device="cuda", generator=g).float()
        s = torch.pow(2.0, near)
        for i in range(b):
            mine = c["table"][i, :-(-lens[i] // bs)].long()
            if i % 5 == 1:
                s[mine] = 2.0 ** base
            elif i % 5 == 2:
                s[mine] = torch.pow(2.0, wide[mine])
            elif i % 5 == 3:
                s[mine] *= 1.0 + torch.rand((len(mine), h), device="cuda", generator=g)
            elif i % 5 == 4:
                s[mine[::3]] = 0.0
        c[name].copy_(s)
    assert _whole_items(c, h, h, lens, qs)
    _compare(c, mq, _fp16_room(float(c["v_scale"].max()), max(lens)))


@pytest.mark.parametrize("kind,dtype,d", [("e4m3", BF, 128), ("same", FP, 64)])
@pytest.mark.parametrize("hq,hkv,lens,qs", [
    (36, 9, [828, 900, 330, 15, 627, 900, 15], [200] * 7),
    (72, 9, [5, 310, 0, 357, 5, 423, 3], [300] * 6 + [148]),
    (21, 3, [194, 3, 5, 137, 1, 1, 3, 230, 0, 2, 4, 276, 2, 5, 163, 5], [187, 200, 66, 200, 84, 149, 200, 200, 51, 200, 11, 166, 200, 200, 38, 200]),
    (8, 2, [700, 3] + [0] * 250 + [129, 0, 0, 0, 0, 0, 0, 1], [33] * 260),          # a batch padded with empty requests
    (64, 8, [40 + i % 3 for i in range(40)], [200] * 40)])                          # whole items of 256 rows
def test_many_items_that_see_nothing(cuda_device, kind, dtype, d, hq, hkv, lens, qs):
    """Long runs of row tiles without a single visible token, behind tiles with some: no role waits for another for ever."""
    from unified_cache_management_b200 import ops
    c, mq = _case(len(lens), lens, qs, hq, hkv, d, 16, kind, dtype)
    ws = ops.new_attention_workspace(d, "cuda")
    out, lse = _check(c, mq, workspace=ws)
    assert ops.workspace_status(ws) == 0
    rows = torch.cat([torch.arange(n, device="cuda") < n - l for l, n in zip(lens, qs)])     # those that see nothing
    assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()


@pytest.mark.parametrize("kind", ["e4m3", "same"])
def test_many_requests_and_long_ones(cuda_device, kind):
    """More requests than threads look at, empty ones among them; one request whose few row tiles are cut over the whole GPU."""
    from unified_cache_management_b200 import ops
    ws = ops.new_attention_workspace(64, "cuda")
    lens = [(i * 37) % 60 if i % 5 else 0 for i in range(1500)]
    c, mq = _case(94, lens, [1 + i % 2 for i in range(1500)], 20, 1, 64, 16, kind, BF)
    _check(c, mq, workspace=ws)
    c, mq = _case(95, [90001], [33], 4, 2, 64, 64, kind, BF)
    _check(c, mq, workspace=ws)
    assert ops.workspace_status(ws) == 0


def test_many_rows_captured(cuda_device):
    """Two graphs with a workspace each, replayed side by side, with other lengths and other splits of the query tokens than
    they were captured with."""
    from unified_cache_management_b200 import ops
    c, mq = _case(96, [900, 3000, 50, 400], [40, 1, 30, 29], 8, 2, 128, 16, "e4m3", BF)
    outs, graphs, streams = [], [], []
    for _ in range(2):
        st, ws = torch.cuda.Stream(), ops.new_attention_workspace(128, "cuda")
        out, lse = torch.empty_like(c["q"]), torch.empty((100, 8), device="cuda")
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            _attend(c, mq, workspace=ws, out=out, lse=lse)
        outs.append((out, lse, ws)), graphs.append(gr), streams.append(st)
    for lens, starts in (((900, 3000, 50, 400), (0, 40, 41, 71, 100)), ((1, 2999, 0, 399), (0, 40, 41, 71, 100)),
                         ((0, 0, 50, 0), (0, 25, 50, 75, 100)), ((333, 70, 7, 129), (0, 97, 98, 99, 100))):
        c["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        c["query_start"].copy_(torch.tensor(starts, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for st, gr in zip(streams, graphs):
                with torch.cuda.stream(st):
                    gr.replay()
        torch.cuda.synchronize()
        want, wlse = _check(c, 97)
        for out, lse, ws in outs:
            assert torch.equal(out, want) and torch.equal(lse, wlse) and ops.workspace_status(ws) == 0
