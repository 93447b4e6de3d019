"""Append over batches at the ends of their ranges, and over wrong offsets."""
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


@pytest.mark.parametrize("cu,lens,written", [
    ([0, 10, 5, 20], [10, 16, 15], {0: range(5), 2: range(10, 20)}),  # tokens 5 to 9 lie in sequences 0 and 2
    ([0, 10, 4], [10, 6], {0: range(4)}),                             # as many in front of the end as behind the start
    ([0, 30, 30], [30, 0], {}),                                       # past the rows
    ([-5, 10, 20], [15, 10], {1: range(10, 20)}),
    ([0, 20, 20, 3], [20, 0, 9], {0: range(3)}),
    ([0, 10, 20] + [20] * 700 + [19], [10, 10] + [0] * 701, {0: range(10), 1: range(10, 19)}),
])
def test_append_reports_wrong_offsets(cu, lens, written):
    """Each is an error from sync; a sequence whose offsets are wrong takes no row, and tokens that lie in one sequence
    alone go where they belong.  Unused table entries name page 0, which none of the batch's sequences owns."""
    ctx = host.Context(0, 64 << 20)
    try:
        n, tokens, page, dim = len(lens), 20, 16, 64
        pages = [-(-x // page) for x in lens]
        table, n_pages = np.zeros((n, 3), np.int32), 1 + sum(pages)
        for i, p in enumerate(pages):
            table[i, :p] = range(1 + sum(pages[:i]), 1 + sum(pages[:i]) + p)
        pool = (1, n_pages, 1, page, dim)
        k_off, v_off = (ctx.put(np.zeros(pool, np.int16)) for _ in range(2))
        kv = ctx.kv_create(host.MOE_T_F16, 1, 1, dim, page, n_pages, k_off, v_off)
        rows = np.arange(1, tokens * dim + 1, dtype=np.int16).reshape(tokens, dim)
        rows_off, cu_off, table_off, lens_off = (ctx.put(x) for x in (rows, np.array(cu, np.int32), table, np.array(lens, np.int32)))
        ctx.kv_append(kv, 0, host.MOE_T_F16, rows_off, rows_off, dim, n, cu_off, tokens, table_off, 3, lens_off)
        with pytest.raises(host.MoeError) as e:
            ctx.sync()
        assert e.value.code == -5
        ctx.sync()  # reported once
        want = np.zeros(pool, np.int16)
        for s, ts in written.items():
            for t in ts:
                pos = lens[s] - (cu[s + 1] - t)
                want[0, table[s, pos // page], 0, pos % page] = rows[t]
        for off in (k_off, v_off):
            assert np.array_equal(ctx.download(off, pool, np.int16), want)
    finally:
        ctx.close()
