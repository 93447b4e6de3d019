"""A key that is not a number makes every row that sees it NaN, whichever key of a step it is, and no other row."""
import pytest
import torch

from attention_ref import Batch, raw
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
@pytest.mark.parametrize("first", [0, 64, 300])
def test_nan_key_at_each_place(ctx, kind, act, cache, dim, first):
    """Sequence i has its one NaN key at first + i: 33 places in a row, in front of the causal edge and on it."""
    n, new = 33, 3 if kind == "prompt" else 1
    lens = [first + 40 + i % 5 for i in range(n)]
    b = Batch(ctx, 71, [new] * n, lens, 2, 1, dim, 16, act, cache)
    for i in range(n):
        p = first + i
        b.k[0, b.table[i, p // 16], 0, p % 16, (7 * i) % dim] = float("nan")
    ctx.upload(b.k_off, raw(b.k))
    getattr(b, kind)()
    got = b.out()
    sees = torch.tensor([first + i < lens[i] - (new - 1 - j) for i in range(n) for j in range(new)])
    assert sees.any()
    assert torch.isnan(got[sees]).all(), (~torch.isnan(got[sees]).all(1)).nonzero().flatten().tolist()
    assert torch.isfinite(got[~sees]).all()
