"""Scores so large that a step of f32 between them is several units: the largest of a row is far above the others, its
weight is 1 and the output its value, however the score, its product with log2(e) and their difference round."""
import pytest
import torch

from attention_ref import DT, Batch, half_step, raw
from moe680m_b200 import host

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    c = host.Context(0, 256 << 20)
    yield c
    c.close()


@pytest.mark.parametrize("kind", ["prompt", "decode"])
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [2, 12])
@pytest.mark.parametrize("size", [2.0 ** n for n in (16, 20, 22, 23, 24, 25, 26, 27, 28, 29)])
def test_one_large_score(ctx, kind, act, cache, dim, heads, size):
    """Column 0 alone makes the scores: up to `size` and down to half of it, 60 rows of different ones, the key of the largest
    anywhere (also behind others that were the largest so far, so that the running maximum grows by any amount)."""
    n, keys, new = 60, 150, 2 if kind == "prompt" else 1
    b = Batch(ctx, 81, [new] * n, [keys] * n, heads, 1, dim, 16, act, cache, dirty=False)
    g = torch.Generator().manual_seed(82)
    b.scale = 1.0
    b.rows.zero_()
    b.rows.view(b.tokens, -1, dim)[:, :, 0] = (size ** 0.5 * (0.7 + 0.3 * torch.rand(b.tokens, 1, generator=g))).to(DT[act])
    b.k.zero_()
    top = torch.randint(0, keys - 1, (n,), generator=g)  # every new token sees it
    for i in range(n):
        col = 0.5 + 0.4 * torch.rand(keys, generator=g)
        col[top[i]] = 1.0
        at = torch.arange(keys)
        b.k[0, b.table[i, at // 16].long(), 0, at % 16, 0] = (size ** 0.5 * col).to(DT[cache])
    for off, t in ((b.q_off, b.rows), (b.k_off, b.k)):
        ctx.upload(off, raw(t))
    getattr(b, kind)()
    got = b.out()[:, :heads * dim].double().view(b.tokens, heads, dim)
    want = torch.stack([b.v[0, b.table[i, top[i] // 16], 0, top[i] % 16].double() for i in range(n) for _ in range(new)])[:, None]
    # one weight, w / w: two roundings of f32, the weight's pieces (one: u(cache); two: its square) and the output's rounding
    u = half_step(DT[cache])
    rel = 4 * 2.0 ** -24 + half_step(DT[act]) + (u if kind == "prompt" and act != "f32" else u * u)
    assert torch.isfinite(got).all(), (~torch.isfinite(got)).any(2).nonzero()[:5].tolist()
    assert ((got - want).abs() <= rel * want.abs() * 1.01 + 2.0 ** -25).all(), float(((got - want).abs() / want.abs()).max())
