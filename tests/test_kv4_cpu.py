"""The paged 4-bit key/value cache without a GPU: refusals, sizes and the oracle's layout."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import oracle as O


@pytest.fixture()
def call(ks):
    """Valid arguments of every entry point; call(name, **changes) gives the return code."""
    buf = np.zeros(4096, np.uint8)
    base = (ks.addr(buf) + 255) // 256 * 256
    cache = dict(pool=base, weights=base, n_pages=4, page_size=32, kv_heads=2, head_dim=64, group_size=32)
    common = dict(page_table=base, page_table_stride=4, seq_lens=base, token_offsets=base, n_seqs=2, n_tokens=3)
    rows = dict(k=base, k_token=128, k_head=64, v=base, v_token=128, v_head=64, dtype=ks.DTYPE_F32, status=None,
                stream=None)
    calls = {
        "append": dict(common, **rows),
        "read": dict(common, **rows),
        "attention": dict(common, max_new=2, max_len=64, q=base, q_token=256, q_head=64, q_heads=4, scale=0.125,
                          out=base, out_token=256, out_head=64, dtype=ks.DTYPE_F32, lse=base, accumulate=0,
                          workspace=base, workspace_bytes=1 << 40, status=None, stream=None),
        "evict": dict(page_table=base, page_table_stride=4, seq_lens=base, n_seqs=2, max_len=64, to_table=base,
                      to_table_stride=1, to_lens=base, budget=32, recent=8, kept=None, workspace=base,
                      workspace_bytes=1 << 40, status=None, stream=None),
    }

    def run(name, **changes):
        c = dict(cache, **{k: changes.pop(k) for k in list(changes) if k in cache})
        args = dict(calls[name], **changes)
        assert set(args) == set(calls[name])
        s = ks.Kv4Cache(c["pool"], c["n_pages"], c["page_size"], c["kv_heads"], c["head_dim"], c["group_size"],
                        c["weights"])
        return getattr(ks.lib(), f"ks_b200_kv4_{name}_async")(ctypes.byref(s), *args.values())

    run.base, run.buf = base, buf
    return run


ALL = ["append", "read", "attention", "evict"]


@pytest.mark.parametrize("name", ALL)
def test_cache_refusals(ks, call, name):
    for bad in (dict(pool=None), dict(pool=call.base + 8), dict(weights=call.base + 2), dict(n_pages=0),
                dict(page_size=0), dict(kv_heads=0), dict(head_dim=0), dict(group_size=0), dict(page_table=None),
                dict(seq_lens=None), dict(n_seqs=0), dict(page_table_stride=0), dict(seq_lens=call.base + 1)):
        assert call(name, **bad) == ks.KS_ERR_INVALID_ARG, bad
        assert ks.last_error()
    for bad in (dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(head_dim=96), dict(head_dim=256),
                dict(group_size=16), dict(group_size=128), dict(kv_heads=70000), dict(n_pages=1 << 31)):
        assert call(name, **bad) == ks.KS_ERR_UNSUPPORTED, bad
    n = dict(n_seqs=65536) if name == "evict" else dict(n_seqs=65536, n_tokens=65536)
    assert call(name, **n) == ks.KS_ERR_UNSUPPORTED


@pytest.mark.parametrize("name", ["append", "read"])
def test_row_refusals(ks, call, name):
    for bad in (dict(k=None), dict(v=None), dict(dtype=3), dict(dtype=-1), dict(k=call.base + 2),
                dict(v=call.base + 1, dtype=1), dict(token_offsets=None), dict(token_offsets=call.base + 2),
                dict(k_token=1 << 31)):
        assert call(name, **bad) == ks.KS_ERR_INVALID_ARG, bad
    if name == "read":  # written: rows may not lie over each other
        for bad in (dict(k_token=0), dict(v_head=32)):
            assert call(name, **bad) == ks.KS_ERR_INVALID_ARG, bad
    assert call(name, n_tokens=0, k=None, v=None) == ks.KS_OK  # nothing to do


def test_attention_refusals(ks, call):
    for bad in (dict(q=None), dict(out=None), dict(dtype=7), dict(q_heads=0), dict(q_heads=3), dict(max_new=0),
                dict(max_len=0), dict(max_new=65), dict(max_len=129), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(out_token=0), dict(out_head=63), dict(q=call.base + 2),
                dict(lse=call.base + 2), dict(accumulate=1, lse=None), dict(accumulate=1, weights=None),
                dict(token_offsets=None)):
        assert call("attention", **bad) == ks.KS_ERR_INVALID_ARG, bad
    big = dict(max_len=1 << 20, page_table_stride=1 << 15)
    for bad in (dict(workspace=None), dict(workspace_bytes=16), dict(workspace=call.base + 8)):
        assert call("attention", **big, **bad) == ks.KS_ERR_WORKSPACE, bad
    assert call("attention", n_tokens=0, q=None, out=None, lse=None) == ks.KS_OK


def test_evict_refusals(ks, call):
    for bad in (dict(weights=None), dict(to_table=None), dict(to_lens=None), dict(budget=0), dict(recent=33),
                dict(max_len=0), dict(max_len=129), dict(budget=33), dict(to_lens=call.base + 2),
                dict(kept=call.base + 1)):
        assert call("evict", **bad) == ks.KS_ERR_INVALID_ARG, bad
    for bad in (dict(workspace=None), dict(workspace_bytes=8), dict(workspace=call.base + 4)):
        assert call("evict", **bad) == ks.KS_ERR_WORKSPACE, bad


def test_sizes(ks):
    # 16 tokens: codes of keys and values, and their scales
    assert ks.kv4_page_bytes(16, 1, 128, 32) == 2 * 16 * (64 + 8)
    assert ks.kv4_page_bytes(64, 8, 64, 64) == 4 * 8 * 2 * 16 * (32 + 2)
    for bad in ((8, 1, 128, 32), (16, 0, 128, 32), (16, 1, 96, 32), (16, 1, 64, 128), (24, 1, 64, 32)):
        assert ks.kv4_page_bytes(*bad) == 0
    c = ks.Kv4Cache(16, 4, 64, 8, 128, 32)
    small = ks.kv4_attention_workspace(c, 32, 1, 1, 1, 256)
    need = ks.kv4_attention_workspace(c, 32, 2, 2, 1, 100000)
    assert 8192 < small < need and need % 4 == 0
    assert ks.kv4_attention_workspace(c, 33, 2, 2, 1, 100000) == 0
    assert ks.kv4_evict_workspace(c, 3, 1000, 100) >= 3 * 8 * 1100 * 4


def test_python_shape_checks(ks):
    torch = pytest.importorskip("torch")
    c = ks.Kv4Cache(16, 4, 16, 2, 64, 32)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    k = torch.zeros(1, 2, 64)
    with pytest.raises(ValueError):
        ks.kv4_append_async(c, table, lens, k, k.half())
    with pytest.raises(ValueError):
        ks.kv4_append_async(c, table, lens, torch.zeros(1, 3, 64), torch.zeros(1, 3, 64))
    with pytest.raises(ValueError):
        ks.kv4_read_async(c, table, lens, k.transpose(1, 2).contiguous().transpose(1, 2), k)
    with pytest.raises(ValueError):
        ks.kv4_attention_async(c, table, lens, k, torch.zeros(1, 4, 64), 1.0, torch.zeros(16, dtype=torch.uint8))
    with pytest.raises(ks.KernelSmithError):
        ks.kv4_attention_async(c, table, lens, k, k, float("nan"), torch.zeros(16, dtype=torch.uint8))


@pytest.mark.parametrize("d", [64, 128])
def test_oracle_layout(d):
    """Every byte of a row is one pair; a lane's bytes are next to each other."""
    for values in (False, True):
        at = O.kv4_byte(d, values)
        assert (at[::2] == at[1::2]).all() and sorted(at[::2]) == list(range(d // 2))
    keys = O.kv4_byte(d, False).reshape(d // 32, 4, 8)  # word, lane t, element
    assert (keys[:, :, 0] == np.arange(4)[None] * (d // 8) + 4 * np.arange(d // 32)[:, None]).all()
    values = O.kv4_byte(d, True).reshape(d // 16, 8, 2)
    assert (values[:, :, 0] == np.arange(8)[None] * (d // 16) + np.arange(d // 16)[:, None]).all()


def test_oracle_quantize():
    x = np.zeros((1, 64))
    x[0, 0], x[0, 1], x[0, 40] = 7.0, 2.5, -1e30
    q, s = O.kv4_quantize(x, 32)
    assert s.tolist() == [[1.0, 65504.0]] and q[0, 0] == 7 and q[0, 1] == 2 and q[0, 40] == -8
    q, s = O.kv4_quantize(np.full((1, 32), 1e-30), 32)
    assert s[0, 0] == np.float16(2.0**-24) and (q == 0).all()


def test_evict_workspace_lies_behind_the_attentions_counters(ks):
    """One workspace may serve both in turn: the first 8192 bytes are not the eviction's."""
    c = ks.Kv4Cache(1 << 12, 10, 64, 8, 128, 32)
    assert ks.kv4_evict_workspace(c, 3, 1000, 100) >= 8192 + 3 * 8 * 1100 * 4


def test_python_index_checks(ks):
    """Tables, lengths and offsets that the library would read wrongly or past their ends."""
    torch = pytest.importorskip("torch")
    c = ks.Kv4Cache(16, 4, 16, 2, 64, 32, weights=4)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    k, ws = torch.zeros(2, 2, 64), torch.zeros(16, dtype=torch.uint8)
    off = torch.arange(3, dtype=torch.int32)
    kept = torch.zeros(2, 2, 8, dtype=torch.int64)
    for bad in ((table.long(), lens, off), (table, lens.long(), off), (table, lens, off.long()), (table, lens, off[:2]),
                (table[:1], lens, off), (table.t().contiguous().t(), lens, off),
                (table, torch.zeros(4).int()[::2], off), (table.float(), lens, off)):
        for call in (ks.kv4_append_async, ks.kv4_read_async):
            with pytest.raises(ValueError):
                call(c, bad[0], bad[1], k, k, token_offsets=bad[2])
        with pytest.raises(ValueError):
            ks.kv4_attention_async(c, bad[0], bad[1], k, k.clone(), 1.0, ws, token_offsets=bad[2])
    with pytest.raises(ValueError):
        ks.kv4_attention_async(c, table, lens, k, k.clone(), 1.0, ws, lse=torch.zeros(2, 2, dtype=torch.float64))
    for bad in ((table.long(), lens, None), (table, lens.long(), None), (table, lens[:1], None), (table, lens, kept)):
        with pytest.raises(ValueError):
            ks.kv4_evict_async(c, table, lens, bad[0], bad[1], 64, 8, 4, ws, kept=bad[2])


def test_python_cache_checks(ks):
    """A pool or weights smaller than the pages they are said to be."""
    torch = pytest.importorskip("torch")
    need = 4 * ks.kv4_page_bytes(16, 2, 64, 32)
    pool, w = torch.zeros(need, dtype=torch.uint8), torch.zeros(4, 2, 16)
    ks.Kv4Cache(pool, 4, 16, 2, 64, 32, weights=w)
    for bad in ((pool[1:], w), (torch.zeros(2 * need, dtype=torch.uint8)[::2], w), (pool, w[:3]), (pool, w.half())):
        with pytest.raises(ValueError):
            ks.Kv4Cache(bad[0], 4, 16, 2, 64, 32, weights=bad[1])


def test_evict_sizes_beyond_64_bits(ks):
    most = 2**31 - 1
    c = ks.Kv4Cache(16, 1, 16, 65535, 64, 32, weights=4)
    assert ks.kv4_evict_workspace(c, 65535, most, most) == 0
    assert ks.kv4_evict_workspace(c, 1, most, most) > 65535 * 2 * most * 4
    rc = ks.lib().ks_b200_kv4_evict_async(c._address, 16, most, 16, 65535, most, 16, most, 16, most, 0, None, 16,
                                          2**64 - 1, None, None)
    assert rc == ks.KS_ERR_UNSUPPORTED


def test_python_tables_that_are_columns_of_wider_ones(ks):
    """What a row of a table holds are its columns, not the distance to the next row."""
    torch = pytest.importorskip("torch")
    c = ks.Kv4Cache(1 << 12, 40, 16, 2, 64, 32, weights=1 << 12)
    big, lens = torch.zeros(2, 10, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    x, ws = torch.zeros(2, 2, 64), torch.zeros(1 << 16, dtype=torch.uint8)

    def refused(call, *args, **kwargs):
        with pytest.raises(ks.KernelSmithError) as e:
            call(*args, **kwargs)
        assert e.value.rc == ks.KS_ERR_INVALID_ARG, e.value

    for table in (big[:, :2], big[:, 8:], big[:, 4:6]):
        refused(ks.kv4_attention_async, c, table, lens, x, x.clone(), 1.0, ws, max_len=33)
        refused(ks.kv4_evict_async, c, table, lens, big, lens, 33, 40, 8, ws)
        refused(ks.kv4_evict_async, c, big, lens, table, lens, 100, 40, 8, ws)  # 40 tokens are three pages
        refused(ks.kv4_evict_async, c, big, lens, table, lens, 33, 40, 8, ws)
    # rows that lie over each other, and a table without columns
    over = torch.zeros(20, dtype=torch.int32).as_strided((2, 10), (4, 1))
    for call in (ks.kv4_append_async, ks.kv4_read_async):
        with pytest.raises(ValueError):
            call(c, over, lens, x, x.clone())
        refused(call, c, big[:, :0], lens, x, x.clone())
    with pytest.raises(ValueError):
        ks.kv4_attention_async(c, over, lens, x, x.clone(), 1.0, ws)


@pytest.mark.parametrize("name", ["append", "read"])
def test_bounded_refusals(ks, call, name):
    """max_len of the bounded forms; all else as in the forms without."""
    s = ks.Kv4Cache(call.base, 4, 32, 2, 64, 32)
    f = getattr(ks.lib(), f"ks_b200_kv4_{name}_bounded_async")

    def run(max_len, n_tokens=3, k=call.base):
        return f(s._address, call.base, 4, call.base, call.base, 2, n_tokens, max_len, k, 128, 64, call.base, 128, 64,
                 ks.DTYPE_F32, None, None)

    for bad in (0, 129, 2**64 - 1):
        assert run(bad) == ks.KS_ERR_INVALID_ARG and ks.last_error()
    assert run(128, k=None) == ks.KS_ERR_INVALID_ARG
    assert run(128, n_tokens=0) == ks.KS_OK


def test_python_offsets_need_max_new(ks):
    """Without it, rows behind the first of a sequence were left unwritten and, without status, nothing said so."""
    torch = pytest.importorskip("torch")
    c = ks.Kv4Cache(16, 4, 16, 2, 64, 32)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q, ws, offsets = torch.zeros(5, 2, 64), torch.zeros(16, dtype=torch.uint8), torch.tensor([0, 2, 5]).int()
    with pytest.raises(ValueError, match="max_new"):
        ks.kv4_attention_async(c, table, lens, q, q.clone(), 1.0, ws, token_offsets=offsets)
    # with it, and without offsets, the library looks at what follows (too small a workspace)
    for rows, kwargs in ((5, dict(token_offsets=offsets, max_new=3)), (2, {})):
        with pytest.raises(ks.KernelSmithError) as e:
            ks.kv4_attention_async(c, table, lens, q[:rows], q[:rows].clone(), 1.0, ws, **kwargs)
        assert e.value.rc == ks.KS_ERR_WORKSPACE


def test_workspaces_of_tables_beyond_31_bits(ks, call):
    """A table may hold more tokens than a sequence may have: the sizes suffice for what the calls go by."""
    c = ks.Kv4Cache(call.base, 4, 32, 2, 64, 32, weights=call.base)
    stride = 1 << 27  # 2^32 tokens
    for max_len in (2**31 - 16384, 2**31 - 1, 2**31, 2**32):
        need = ks.kv4_attention_workspace(c, 4, 2, 3, 2, max_len)
        assert need == ks.kv4_attention_workspace(c, 4, 2, 3, 2, 2**31 - 16385) > 0
        rc = call("attention", page_table_stride=stride, max_len=max_len, workspace_bytes=need - 1)
        assert rc == ks.KS_ERR_WORKSPACE
        need = ks.kv4_evict_workspace(c, 2, 2**31 - 16385, 32)
        assert ks.kv4_evict_workspace(c, 2, max_len, 32) >= need > 0
        assert call("evict", page_table_stride=stride, max_len=max_len, workspace_bytes=need - 1) == ks.KS_ERR_WORKSPACE


def test_python_workspaces_are_contiguous(ks):
    """One byte expanded to many is no workspace."""
    torch = pytest.importorskip("torch")
    c = ks.Kv4Cache(1 << 12, 40, 16, 2, 64, 32, weights=1 << 12)
    table, lens, x = torch.zeros(2, 10, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 64)
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 20, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="contiguous"):
            ks.kv4_attention_async(c, table, lens, x, x.clone(), 1.0, ws)
        with pytest.raises(ValueError, match="contiguous"):
            ks.kv4_evict_async(c, table, lens, table + 1, lens, 100, 40, 8, ws)


@pytest.mark.parametrize("name", ["attention", "evict"])
def test_the_largest_max_len_is_refused(ks, call, name):
    for bad in (129, 2**31, 2**63, 2**64 - 1):
        assert call(name, max_len=bad) == ks.KS_ERR_INVALID_ARG, bad
