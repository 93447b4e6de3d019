"""Decode and prompt attention over rows in which one key scores far above all others (a first token that every later one
looks at), through the C ABI against 64 bits.  The other keys' softmax weights are then small, e^-10 to e^-24 of the largest,
and make up the whole output where the first key's value is zero.

Bound: the one of attention_ref.py, which takes a weight's rounding as relative to the weight, and beside it the smallest
step of the 16-bit type that the weights enter the products in.  An f16 cache has the weights times 2^L (L = 15 in decode, in a
prompt 13 with f32 and 11 with f16 queries) as f16 pieces; the last piece is a multiple of 2^-24 and so off by at most 2^-25, which is
2^-(25 + L) of the largest weight.  So each key adds at most 2^-(25 + L) |v| to the weighted sum's error, whose denominator is
the sum of all weights over the largest.  The pieces of a bf16 cache have f32's range: nothing is added."""
import pytest
import torch

from attention_ref import DT, Batch, raw
from moe680m_b200 import host

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
LIFT = {("decode", "f32"): 15, ("decode", "f16"): 15, ("prompt", "f32"): 13, ("prompt", "f16"): 11}


@pytest.fixture
def ctx():
    c = host.Context(0, 512 << 20)
    yield c
    c.close()


def sink_batch(ctx, seed, new, lens, heads, hkv, dim, page, act, cache, gap, at, values):
    """Scores of standard deviation about 0.5, and key at[i] of sequence i `gap` above them with a value of zero.  Column 0 of the
    queries and of that key alone makes the gap, by powers of two and `gap` itself: exact in every type."""
    b = Batch(ctx, seed, new, lens, heads, hkv, dim, page, act, cache, q_scale=0.5)
    b.scale = 2.0 ** -3
    b.rows.view(b.tokens, -1, dim)[:, :, 0] = 2.0
    b.k[0, :, :, :, 0].nan_to_num_(0.0).mul_(0.0)
    g = torch.Generator().manual_seed(seed + 1)
    held = torch.isfinite(b.v)
    fresh = 1 + torch.rand(b.v.shape, generator=g) if values == "one sign" else torch.randn(b.v.shape, generator=g)
    b.v = torch.where(held, fresh.to(DT[cache]), b.v)
    for i, n in enumerate(lens):
        if n:
            p, row = b.table[i, at[i] // page], at[i] % page
            b.k[0, p, :, row, 0] = 4.0 * gap
            b.v[0, p, :, row] = 0.0
    for off, t in ((b.q_off, b.rows), (b.k_off, b.k), (b.v_off, b.v)):
        ctx.upload(off, raw(t))
    return b


def check(b, kind, rows=None):
    one_piece = kind == "prompt" and b.act != "f32"
    want, bound = b.expected(0, one_piece, rows)
    want, bound = (x.view(b.tokens, b.heads, b.dim) for x in (want, bound))
    if b.cache == "f16":
        for i, n in enumerate(b.new):
            k, v = (x.double() for x in b.cached(i))
            for t in range(int(b.cu[i]), int(b.cu[i]) + n):
                keys = b.lens[i] - (int(b.cu[i]) + n - t) + 1
                if keys <= 0 or (rows is not None and t not in rows):
                    continue
                q = b.rows[t, :b.heads * b.dim].double().view(b.hkv, -1, b.dim)
                s = torch.einsum("hgd,hkd->hgk", q, k[:, :keys]) * b.scale
                total = (s - s.amax(-1, keepdim=True)).exp().sum(-1)
                step = 2.0 ** -(25 + LIFT[kind, b.act]) / total[..., None] * v[:, :keys].abs().sum(1)[:, None]
                bound[t] += step.reshape(b.heads, b.dim)
    got = b.out()[:, :b.heads * b.dim].double().view_as(want)
    seen = torch.isfinite(want)
    assert seen.any() and torch.isfinite(got[seen]).all()
    off, bound = (got - want).abs()[seen], bound[seen]
    assert (off <= bound).all(), (int((off > bound).sum()), off.numel(), float((off / bound).nan_to_num(0).max()))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("gap", [10, 14, 17, 18, 20, 24])
@pytest.mark.parametrize("heads", [4, 12])
def test_decode_one_key_above_the_rest(ctx, act, cache, gap, heads):
    """Up to 8 and more than 8 heads to a kv head; the key at the front, at the end and between."""
    lens = [9000, 3000, 0, 513, 33]
    b = sink_batch(ctx, 51, [1] * 5, lens, heads, 1, 128, 32, act, cache, gap, [0, 2999, 0, 200, 0], "one sign")
    b.decode()
    check(b, "decode")


@pytest.mark.parametrize("gap", [10, 14, 17, 18])
def test_decode_one_key_above_a_long_tail(ctx, gap):
    b = sink_batch(ctx, 52, [1], [262144], 2, 1, 64, 64, "f32", "f16", gap, [0], "both signs")
    b.decode()
    check(b, "decode")


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("gap", [10, 14, 17, 18, 20, 24])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_one_key_above_the_rest(ctx, act, cache, gap, dim):
    """The key at the front, in the middle and among the prompt's own; some rows do not see it yet."""
    new, lens = [20, 40, 0, 37], [8192, 4100, 50, 127]
    b = sink_batch(ctx, 53, new, lens, 4, 1, dim, 32, act, cache, gap, [0, 2900, 0, 100], "one sign")
    b.prompt()
    check(b, "prompt")


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_maximum_that_grows_by_small_steps(ctx, act, cache, dim):
    """Scores that climb by 1/4 of a unit every 64 keys to 20 and fall back: each step moves the maximum a little, and at the
    end most weights are far below the largest."""
    n = 8192
    b = sink_batch(ctx, 54, [16], [n], 4, 1, dim, 64, act, cache, 0, [0], "one sign")
    for i in range(0, n, 64):
        b.k[0, b.table[0, i // 64], :, :, 0] = min(i // 64, 80) * 0.25 * 4 if i < n // 2 else -40.0
    ctx.upload(b.k_off, raw(b.k))
    b.prompt()
    check(b, "prompt")
