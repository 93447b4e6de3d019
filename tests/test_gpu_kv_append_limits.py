"""Append over batches at the ends of their ranges."""
import numpy as np
import pytest

from moe680m_b200 import host

pytestmark = pytest.mark.gpu


def test_append_tokens_past_2_to_27():
    """A packed batch whose sequence's rows lie behind 2^27 rows of none, so that the numbers of the tokens'
    threads pass 32 bits.  16-bit rows of 64 columns, 17.2 GB; keys and values are the same rows."""
    tokens, first, dim = (1 << 27) + 48, 1 << 27, 64
    ctx = host.Context(0, tokens * dim * 2 + (16 << 20))
    try:
        rows_off = ctx.alloc(tokens * dim * 2)
        pool = (1, 4, 1, 16, dim)
        k_off, v_off = (ctx.put(np.zeros(pool, np.int16)) for _ in range(2))
        kv = ctx.kv_create(host.MOE_T_F16, 1, 1, dim, 16, 4, k_off, v_off)
        rows = np.arange(1, 48 * dim + 1, dtype=np.int16).reshape(48, dim)
        ctx.upload(rows_off + first * dim * 2, rows)
        ctx.upload(rows_off, -rows)  # not the sequence's
        table, lens, cu = ctx.put(np.array([2, 0, 3], np.int32)), ctx.put(np.array([48], np.int32)), ctx.put(np.array([first, first + 48], np.int32))
        ctx.kv_append(kv, 0, host.MOE_T_F16, rows_off, rows_off, dim, 1, cu, tokens, table, 3, lens)
        ctx.sync()
        for off in (k_off, v_off):
            got = ctx.download(off, pool, np.int16)[0, :, 0]
            assert np.array_equal(got[[2, 0, 3]].reshape(48, dim), rows) and not got[1].any()
    finally:
        ctx.close()
