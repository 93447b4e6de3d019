"""Prompt attention over wrong packed offsets: reported by sync, wherever in the list they stand."""
import numpy as np
import pytest

from attention_ref import Batch
from moe680m_b200 import host

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    c = host.Context(0, 256 << 20)
    yield c
    c.close()


@pytest.mark.parametrize("act,cache,dim", [("f32", "f16", 128), ("f16", "f16", 64), ("bf16", "bf16", 128)])
@pytest.mark.parametrize("n_seqs", [3, 32, 33, 400, 1500])
@pytest.mark.parametrize("what", ["descend", "past the rows", "negative"])
def test_wrong_offsets_at_the_end(ctx, act, cache, dim, n_seqs, what):
    """The first sequences, one token each, are right, and every block of the launch finds its rows among them; the last
    sequence's offsets are wrong."""
    held = min(n_seqs - 1, 60)
    new = [1] * held + [0] * (n_seqs - held)
    b = Batch(ctx, 61, new, [5 + i % 40 for i in range(n_seqs)], 1, 1, dim, 16, act, cache)
    cu = b.cu.numpy().copy()
    cu[-1] = {"descend": held - 1, "past the rows": held + 1, "negative": -7}[what]
    ctx.upload(b.cu_off, cu)
    b.prompt()
    with pytest.raises(host.MoeError) as e:
        ctx.sync()
    assert e.value.code == -5
    b.check(b.out(), one_piece=act != "f32")  # the right sequences' rows
    ctx.upload(b.cu_off, b.cu.numpy())
    b.prompt()
    b.check(b.out(), one_piece=act != "f32")
