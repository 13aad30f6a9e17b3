"""GPU: corners of attention over the paged KV cache for many rows: value scales far apart, of 0 and at their floor, rows of
very small queries, and whole items of 256 rows."""
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
