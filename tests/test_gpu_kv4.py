"""The paged 4-bit key/value cache on the GPU against its definition in 64 bits (oracle.kv4_*): append and read bit
for bit, attention within bounds that follow from its roundings, eviction exactly."""

from __future__ import annotations

import numpy as np
import pytest

import oracle as O

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]


def _type(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Seqs:
    """A cache on the GPU with random contents, its sequences, and the same keys and values in f64."""

    def __init__(self, ks, cuda, lens, news, heads, d, group, page, seed=0, weights=False, spare=2, garbage=True,
                 table_slack=1):
        import torch

        rng = np.random.default_rng(seed)
        self.ks, self.cuda, self.rng = ks, cuda, rng
        self.lens, self.news, self.heads, self.d, self.group, self.page = list(lens), list(news), heads, d, group, page
        each = [-(-x // page) for x in lens]
        self.n_pages = sum(each) + spare
        channel = 1 + 3 * (rng.random((heads, 1, d)) < 0.06)
        k = rng.standard_normal((self.n_pages, heads, page, d)) * channel
        v = rng.standard_normal((self.n_pages, heads, page, d)) * np.exp(rng.standard_normal((self.n_pages, heads,
                                                                                              page, 1)))
        self.k = O.kv4_value(*O.kv4_quantize(k, group))
        self.v = O.kv4_value(*O.kv4_quantize(v, group))
        self.scale_max = O.kv4_quantize(k, group)[1].astype(np.float64).max()
        pool = O.kv4_pool(k, v, group)
        ids = rng.permutation(self.n_pages)
        self.pages, at = [], 0
        self.table_np = np.full((len(lens), max(each + [1]) + table_slack), -1, np.int32)
        for s, n in enumerate(each):
            self.pages.append(ids[at:at + n])
            self.table_np[s, :n] = ids[at:at + n]
            at += n
        if garbage:  # slots that no token stands in hold anything, NaN scales among it
            used = np.zeros((self.n_pages, page), bool)
            for s, n in enumerate(lens):
                for i, p in enumerate(self.pages[s]):
                    used[p, : min(page, n - i * page)] = True
            half, codes, per = pool.shape[-1] // 2, 8 * d, 2 * (d // group)
            p, slot = np.nonzero(~used)
            for h in (0, half):
                for b in range(per):
                    pool[p, :, slot // 16, h + codes + (slot % 16) * per + b] = 0xFF
        self.pool = torch.from_numpy(pool).to(cuda)
        self.table = torch.from_numpy(self.table_np).to(cuda)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
        self.first = np.concatenate([[0], np.cumsum(news)]).astype(int)
        self.tokens = int(self.first[-1])
        self.offsets = torch.tensor(self.first, dtype=torch.int32, device=cuda)
        self.w = None
        if weights:
            self.w = torch.from_numpy(rng.random((self.n_pages, heads, page)).astype(np.float32)).to(cuda)
        self.cache = ks.Kv4Cache(self.pool, self.n_pages, page, heads, d, group, weights=self.w)
        self.status = torch.zeros(2, dtype=torch.int32, device=cuda)

    def cached(self, s, which):
        """Keys or values of sequence s, [len, heads, d]."""
        x = (self.k if which == "k" else self.v)[self.pages[s]]
        return x.transpose(0, 2, 1, 3).reshape(-1, self.heads, self.d)[: self.lens[s]]

    def weights_of(self, s, w):
        return w[self.pages[s]].transpose(1, 0, 2).reshape(self.heads, -1)[:, : self.lens[s]]

    def ok(self):
        import torch

        torch.cuda.synchronize()
        assert self.status.cpu().tolist() == [0, 0]


def _query(c, heads, dtype, seed=1, size=1.5):
    import torch

    q = torch.from_numpy(np.random.default_rng(seed).standard_normal((c.tokens, heads, c.d)) * size)
    return q.to(_type(dtype)).to(c.cuda)


def _attend(c, q, scale, out=None, lse=True, max_new=None, max_len=None, accumulate=False, offsets=True, stream=None):
    import torch

    out = torch.full_like(q, float("nan")) if out is None else out
    lse = torch.full(q.shape[:2], float("nan"), device=c.cuda) if lse is True else lse
    max_new = max(c.news + [1]) if max_new is None else max_new
    max_len = max(c.lens + [max_new]) if max_len is None else max_len
    need = c.ks.kv4_attention_workspace(c.cache, q.shape[1], len(c.lens), c.tokens, max_new, max_len)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=c.cuda)  # NaN: nothing may be taken from it
    ws[:8192] = 0
    c.ks.kv4_attention_async(c.cache, c.table, c.seq_lens, q, out, scale, ws,
                             token_offsets=c.offsets if offsets else None, max_new=max_new, max_len=max_len,
                             lse=lse, accumulate=accumulate, status=c.status, stream=stream)
    assert not ws[:8192].any()  # ready for the next call
    return out, lse


def _check(c, q, scale, out, lse, dtype, weights=None, before=None):
    """Bounds.  A score is a sum of products code * q, exact in f32, over up to 2 x 8 tensor-core steps of at most
    2^-23 of the largest partial sum (15 + 8 times sum |q| and the scale: codes are taken from 0 to 15, from -8
    sum(q)), and of some six more roundings: |dx| <= 22 * 23 * 2^-23 * scale * s_max * sum |q| <= E.  A probability is
    then within 2 E + 2^-18 (exponentials, sums, the two parts) relatively, 2^-11 more in one f16 part (bf16 results),
    and the result is rounded once."""
    import torch

    half = torch.finfo(_type(dtype)).eps / 2
    out, lse, qn = out.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().cpu().numpy()
    err = norm = top = 0.0
    for s in range(len(c.lens)):
        a, n = c.first[s], c.news[s]
        want, z, w, size, _ = O.kv4_attention(qn[a:a + n], c.cached(s, "k"), c.cached(s, "v"), scale, n)
        e = 512 * 2.0**-23 * abs(scale) * c.scale_max * np.abs(qn[a:a + n]).sum(-1)  # [n, heads]
        rel = 2 * e + 2.0**-18 + (2.0**-11 if dtype == "bf16" else 0)
        tol = half * np.abs(want) + rel[..., None] * size + 2.0**-24
        bad = ~(np.abs(out[a:a + n] - want) <= tol)
        assert not bad.any(), (s, np.argwhere(bad)[:5], out[a:a + n][bad][:5], want[bad][:5])
        empty = np.isinf(z)
        assert (np.isneginf(lse[a:a + n]) == empty).all() and (out[a:a + n][empty] == 0).all()
        with np.errstate(invalid="ignore"):
            assert (empty | (np.abs(lse[a:a + n] - z) <= e + 2.0**-20 + 2.0**-22 * np.abs(z))).all()
        top = max([top] + np.abs(z[~empty]).tolist())
        err, norm = err + ((out[a:a + n] - want) ** 2).sum(), norm + (want**2).sum()
        if weights is not None:
            got = c.weights_of(s, weights.double().cpu().numpy())
            old = c.weights_of(s, before)
            # f32 sums of the rows' weights, each within 2 E + 2^-18
            worst = 2 * e.max() + 2.0**-18 if n else 0.0
            assert (np.abs(got - old - w) <= worst * w + 2.0**-23 * (old + w) * (1 + n)).all(), s
    # The products' roundings are independent, far below their worst case.  What does not average out: the score x (in
    # units of log2, rounded to f32 four times: scale * log2(e), the row's factor, the product with it, the difference
    # to the maximum) is off by up to 4 * 2^-24 |x|, so the probabilities by 2^-22 |x| relatively and, divided by their
    # sum, by twice that; |x| is about |lse| where it matters (at x = 66, 3e-5).
    most = half + 2.0**-17 + 2.0**-21 * top + (2.0**-12 if dtype == "bf16" else 0)
    assert err**0.5 <= most * norm**0.5 + 1e-30


# ------------------------------------------------------------------ append, read
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("page,heads", [(16, 3), (64, 8), (256, 33)])
def test_append_and_read(ks, cuda, dtype, d, group, page, heads):
    import torch

    lens, news = [1, page + 5, 40, 0, 2 * page], [1, 7, 40, 0, 1]
    c = Seqs(ks, cuda, lens, news, heads, d, group, page, seed=d + group + page, weights=True, garbage=False)
    rng = np.random.default_rng(9)
    x = torch.from_numpy(rng.standard_normal((2, c.tokens + 2, heads, d)) * np.exp(2 * rng.standard_normal(
        (2, c.tokens + 2, heads, 1)))).to(_type(dtype)).to(cuda)
    x[0, 0, 0, :group] = 0
    before, wbefore = c.pool.clone(), c.w.clone()
    ks.kv4_append_async(c.cache, c.table, c.seq_lens, x[0], x[1], token_offsets=c.offsets, status=c.status)
    k, v = torch.full_like(x[0], 7), torch.full_like(x[0], 7)
    ks.kv4_read_async(c.cache, c.table, c.seq_lens, k, v, token_offsets=c.offsets, status=c.status)
    c.ok()
    # rows behind the last sequence are left
    assert (k[c.tokens:] == 7).all() and (v[c.tokens:] == 7).all()
    want = before.cpu().numpy()
    wwant = wbefore.cpu().numpy()
    for values, got in ((0, k), (1, v)):
        codes, scale = O.kv4_quantize(x[values].double().cpu().numpy(), group)
        value = torch.from_numpy(O.kv4_value(codes, scale)).to(_type(dtype))
        assert torch.equal(got[: c.tokens].cpu(), value[: c.tokens])
        at, half = O.kv4_byte(d, bool(values)), want.shape[-1] // 2 * values
        for s in range(len(lens)):
            for j in range(news[s]):
                pos, i = lens[s] - news[s] + j, c.first[s] + j
                p, slot = c.pages[s][pos // page], pos % page
                q = (codes[i] & 15).astype(np.uint8)
                row = want[p, :, slot // 16]
                row[:, half + slot % 16 * (d // 2) + at[::2]] = q[:, ::2] | (q[:, 1::2] << 4)
                per = 2 * (d // group)
                o = half + 8 * d + slot % 16 * per
                row[:, o:o + per] = np.ascontiguousarray(scale[i]).view(np.uint8)
                wwant[p, :, slot] = 0
    assert (c.pool.cpu().numpy() == want).all()
    assert (c.w.cpu().numpy() == wwant).all()


def test_append_ties_and_strides(ks, cuda):
    """Quotients on and next to a tie, decided by the exact quotient; strided and unaligned rows."""
    import torch

    heads, d, group = 2, 64, 32
    c = Seqs(ks, cuda, [20], [20], heads, d, group, 32, garbage=False)
    rng = np.random.default_rng(3)
    x = np.zeros((20, heads, d), np.float32)
    scale = np.float16(np.exp(rng.standard_normal((20, heads, 2)))).astype(np.float32)
    tie = (rng.integers(-8, 7, (20, heads, 2, group)) + 0.5).astype(np.float32) * scale[..., None]
    tie = np.nextafter(tie, np.where(rng.random(tie.shape) < 0.5, np.inf, -np.inf).astype(np.float32)) \
        * (rng.random(tie.shape) < 0.7) + tie * (rng.random(tie.shape) < 0.2)
    tie[..., 0] = 7 * scale  # the group's scale, exactly
    tie = np.clip(tie, -8 * scale[..., None], 7 * scale[..., None])
    x[:] = tie.reshape(20, heads, d)
    big = torch.zeros(20 * (heads * d + 3) + 1, device=cuda)
    k = big[1:].as_strided((20, heads, d), (heads * d + 3, d, 1))  # 4-byte aligned rows
    k.copy_(torch.from_numpy(x))
    v = torch.from_numpy(x).to(cuda).transpose(0, 1).contiguous().transpose(0, 1)
    ks.kv4_append_async(c.cache, c.table, c.seq_lens, k, v, token_offsets=c.offsets, status=c.status)
    ko = torch.zeros(20, heads, d + 1, device=cuda)[..., 1:]
    vo = torch.zeros(heads, 20, d, device=cuda).transpose(0, 1)
    ks.kv4_read_async(c.cache, c.table, c.seq_lens, ko, vo, token_offsets=c.offsets, status=c.status)
    c.ok()
    want = torch.from_numpy(O.kv4_value(*O.kv4_quantize(x, group)).astype(np.float32))
    assert torch.equal(ko.cpu(), want) and torch.equal(vo.cpu(), want)


def test_append_not_finite(ks, cuda):
    import torch

    c = Seqs(ks, cuda, [3], [3], 1, 64, 32, 16, garbage=False)
    x = torch.ones(3, 1, 64, device=cuda)
    x[0, 0, 3], x[0, 0, 40], x[1, 0, 5], x[2, 0, 0] = float("nan"), float("inf"), -float("inf"), 1e-30
    x[2, 0, 32:] = 3e38
    y = torch.zeros_like(x)
    ks.kv4_append_async(c.cache, c.table, c.seq_lens, x, torch.ones_like(x), token_offsets=c.offsets, status=c.status)
    ks.kv4_read_async(c.cache, c.table, c.seq_lens, y, torch.zeros_like(x), token_offsets=c.offsets, status=None)
    torch.cuda.synchronize()
    assert c.status.cpu().tolist() == [1, 0]
    want = O.kv4_value(*O.kv4_quantize(x.double().cpu().numpy(), 32))
    assert np.isfinite(want).all() and (y.double().cpu().numpy() == want).all()
    assert y[0, 0, 3] == 0 and y[0, 0, 40] == 7 * 65504 and y[1, 0, 5] == -8 * 65504 and y[2, 0, 33] == 7 * 65504
    with pytest.raises(ks.KernelSmithError):
        ks.check(ks.lib().ks_b200_status_check(ks.addr(c.status), None))


# --------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("heads,q_heads", [(2, 2), (1, 4), (2, 10), (1, 8), (1, 12)])
def test_decode(ks, cuda, dtype, d, group, heads, q_heads):
    """One new token: lengths around tiles, blocks, pages and chunks."""
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 100, 255, 257, 700]
    c = Seqs(ks, cuda, lens, [1] * len(lens), heads, d, group, 32, seed=d + group + q_heads)
    q = _query(c, q_heads, dtype)
    out, lse = _attend(c, q, d**-0.5)
    c.ok()
    _check(c, q, d**-0.5, out, lse, dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages(ks, cuda, page):
    lens = [1, page - 1, page, page + 1, 3 * page + 7, 300]
    for d, group in ((128, 32), (64, 64)):
        c = Seqs(ks, cuda, lens, [1] * len(lens), 2, d, group, page, seed=page)
        q = _query(c, 8, "f32")
        out, lse = _attend(c, q, 0.1, offsets=False)
        c.ok()
        _check(c, q, 0.1, out, lse, "f32")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 32), (128, 32), (128, 128)])
@pytest.mark.parametrize("q_heads,heads,lens,news", [
    (4, 1, [5, 40, 70, 0, 9], [2, 3, 1, 0, 9]),  # a prompt, drafts, one token, an idle place
    (7, 1, [130, 33], [5, 33]),
    (6, 2, [300, 64], [31, 64]),
    (2, 2, [700], [17]),
])
def test_several_new_tokens(ks, cuda, dtype, d, group, q_heads, heads, lens, news):
    c = Seqs(ks, cuda, lens, news, heads, d, group, 16, seed=len(lens) + d)
    q = _query(c, q_heads, dtype)
    out, lse = _attend(c, q, d**-0.5)
    c.ok()
    _check(c, q, d**-0.5, out, lse, dtype)


def test_long_and_split(ks, cuda):
    """Many chunks to a row, one head."""
    for d, group, dtype in ((128, 64, "f32"), (64, 32, "bf16")):
        c = Seqs(ks, cuda, [20000, 3, 9001], [1, 1, 2], 1, d, group, 64, seed=5)
        q = _query(c, 5, dtype)
        out, lse = _attend(c, q, d**-0.5)
        c.ok()
        _check(c, q, d**-0.5, out, lse, dtype)


@pytest.mark.parametrize("n,heads,q_heads,dtype", [(33, 32, 32, "bf16"), (40, 1, 3, "f32"), (100, 2, 8, "f16"),
                                                   (129, 1, 2, "f32"), (300, 3, 3, "bf16")])
def test_many_sequences(ks, cuda, n, heads, q_heads, dtype):
    """More sequences than a warp has lanes and a CTA threads, of unequal lengths, some without tokens."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(0, 90, n)]
    lens[n // 2] = 1500
    news = [min(int(x), 1) if s % 7 else min(int(x), 3) for s, x in enumerate(lens)]
    news[1], lens[1] = 1, 0
    c = Seqs(ks, cuda, lens, news, heads, 64, 64, 32, seed=n, weights=True)
    before = c.w.double().cpu().numpy()
    q = _query(c, q_heads, dtype)
    out, lse = _attend(c, q, 0.125, accumulate=True)
    c.ok()
    _check(c, q, 0.125, out, lse, dtype, weights=c.w, before=before)


def test_weights_beside_sequences_without_tokens(ks, cuda):
    """Every other sequence has a new token but no cached one: the others' tokens all get their weights."""
    for n in (20, 40, 150):
        lens = [0 if s % 2 else 40 + s for s in range(n)]
        c = Seqs(ks, cuda, lens, [1] * n, 8, 64, 64, 32, seed=n, weights=True)
        before = c.w.double().cpu().numpy()
        q = _query(c, 16, "bf16")
        out, lse = _attend(c, q, 0.125, accumulate=True)
        c.ok()
        _check(c, q, 0.125, out, lse, "bf16", weights=c.w, before=before)


def test_one_workspace_for_calls_of_all_sizes(ks, cuda):
    """Calls of any sizes follow one another in one workspace, zeroed once."""
    import torch

    cases = []
    for i, (lens, heads, q_heads, d, new) in enumerate([([5000], 1, 4, 128, 1), ([40, 900, 3], 2, 4, 64, 3),
                                                        ([17] * 20, 4, 4, 128, 1), ([2500], 1, 1, 64, 1)]):
        c = Seqs(ks, cuda, lens, [min(new, n) for n in lens], heads, d, 32, 64, seed=i)
        cases.append((c, _query(c, q_heads, "f32"), max(lens), new))
    need = max(ks.kv4_attention_workspace(c.cache, q.shape[1], len(c.lens), c.tokens, new, most)
               for c, q, most, new in cases)
    ws = torch.zeros(need, dtype=torch.uint8, device=cuda)
    outs = []
    for _ in range(2):
        for c, q, most, new in cases:
            out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device=cuda)
            ks.kv4_attention_async(c.cache, c.table, c.seq_lens, q, out, 0.1, ws, token_offsets=c.offsets, max_new=new,
                                   max_len=most, lse=lse, status=c.status)
            outs.append((c, q, out, lse))
    for c, q, out, lse in outs:
        c.ok()
        _check(c, q, 0.1, out, lse, "f32")


def test_empty_rows_and_rows_behind(ks, cuda):
    """Sequences without tokens, new tokens before position 0, rows before and behind the sequences, strided rows."""
    import torch

    lens, news = [0, 3, 50, 0], [2, 5, 1, 0]
    c = Seqs(ks, cuda, lens, news, 2, 64, 32, 16)
    c.first = c.first + 1
    c.offsets = c.offsets + 1
    big = torch.randn(c.tokens + 3, 6, 64 + 3, device=cuda)
    q = big[:, :4, :64]
    out = torch.full((4, c.tokens + 3, 64), 7.0, device=cuda).transpose(0, 1)
    lse = torch.full((c.tokens + 3, 4), 7.0, device=cuda)
    c.tokens += 3
    _attend(c, q, 0.125, out=out, lse=lse, max_len=64)
    c.ok()
    assert (out[0] == 7).all() and (out[-2:] == 7).all() and (lse[0] == 7).all() and (lse[-2:] == 7).all()
    assert (out[1:3] == 0).all() and torch.isneginf(lse[1:3]).all()  # no token
    assert (out[3:5] == 0).all() and torch.isneginf(lse[3:5]).all()  # before position 0
    _check(c, q, 0.125, out, lse, "f32")


def test_extreme_scores(ks, cuda):
    """Scores far apart, all equal, negative and zero scale; values of very unlike size; huge and tiny queries."""
    import torch

    for scale, size in ((1.0, 30.0), (0.0, 1.0), (-0.125, 1.0), (1e-20, 1e18), (1e20, 1e-20)):
        c = Seqs(ks, cuda, [400, 7], [1, 2], 1, 128, 32, 64, seed=11)
        q = _query(c, 4, "f32", size=size)
        out, lse = _attend(c, q, scale)
        c.ok()
        _check(c, q, scale, out, lse, "f32")
    # one token with all the weight and values 2^-18 of the others'
    c = Seqs(ks, cuda, [320], [1], 1, 64, 32, 64, seed=12)
    k = torch.zeros(320, 1, 64, device=cuda)
    v = torch.randn(320, 1, 64, device=cuda) * 2.0**14
    k[7], v[7] = 4.0, v[7] * 2.0**-18
    offsets = torch.tensor([0, 320], dtype=torch.int32, device=cuda)
    ks.kv4_append_async(c.cache, c.table, c.seq_lens, k, v, token_offsets=offsets, status=c.status)
    c.k[c.pages[0]] = _paged(c, O.kv4_value(*O.kv4_quantize(k.double().cpu().numpy(), 32)))
    c.v[c.pages[0]] = _paged(c, O.kv4_value(*O.kv4_quantize(v.double().cpu().numpy(), 32)))
    q = torch.full((1, 2, 64), 1.0, device=cuda)
    out, lse = _attend(c, q, 1.0)
    c.ok()
    _check(c, q, 1.0, out, lse, "f32")


def _paged(c, x):
    full = np.zeros((len(c.pages[0]) * c.page, c.heads, c.d))
    full[: len(x)] = x
    return full.reshape(-1, c.page, c.heads, c.d).transpose(0, 2, 1, 3)


def test_queries_not_finite_stay_in_their_rows(ks, cuda):
    import torch

    c = Seqs(ks, cuda, [300], [1], 1, 128, 64, 32)
    q = _query(c, 8, "f32")
    good, _ = _attend(c, q, 0.1)
    bad = q.clone()
    bad[0, 2, 5], bad[0, 6, 0] = float("nan"), float("inf")
    out, lse = _attend(c, bad, 0.1)
    c.ok()
    rows = [0, 1, 3, 4, 5, 7]
    assert torch.equal(out[0, rows], good[0, rows])
    assert torch.isnan(out[0, 2]).all() and torch.isnan(out[0, 6]).all() and torch.isnan(lse[0, [2, 6]]).all()


@pytest.mark.parametrize("q_heads,heads,lens,news", [
    (4, 1, [5, 40, 300, 0], [1, 1, 1, 0]),
    (3, 3, [17, 600], [1, 1]),
    (8, 2, [90, 33, 512], [7, 33, 1]),
])
@pytest.mark.parametrize("dtype,d,group", [("f32", 128, 32), ("bf16", 64, 64), ("f16", 128, 128)])
def test_accumulated_weights(ks, cuda, q_heads, heads, lens, news, dtype, d, group):
    import torch

    c = Seqs(ks, cuda, lens, news, heads, d, group, 16, weights=True)
    before = c.w.double().cpu().numpy()
    q = _query(c, q_heads, dtype)
    out, lse = _attend(c, q, d**-0.5, accumulate=True)
    c.ok()
    _check(c, q, d**-0.5, out, lse, dtype, weights=c.w, before=before)
    used = np.zeros(before.shape, bool)
    for s, n in enumerate(lens):
        for i, p in enumerate(c.pages[s]):
            used[p, :, : min(16, n - i * 16)] = True
    assert (c.w.double().cpu().numpy()[~used] == before[~used]).all()
    # in a fixed order: the same again, bit for bit
    first, again = c.w.clone(), torch.from_numpy(before.astype(np.float32)).to(cuda)
    c.w.copy_(again)
    out2, lse2 = _attend(c, q, d**-0.5, accumulate=True)
    assert torch.equal(c.w, first) and torch.equal(out, out2) and torch.equal(lse, lse2)


def test_far_pages(ks, cuda):
    """A pool of more than 4 GiB, tokens at its end."""
    import torch

    heads, d, group, page = 8, 128, 32, 256
    c = Seqs(ks, cuda, [300, 20], [1, 1], heads, d, group, page, weights=True)
    per = ks.kv4_page_bytes(page, heads, d, group)
    n = (9 << 29) // per + c.n_pages
    pool = torch.empty(n, per, dtype=torch.uint8, device=cuda)
    pool[n - c.n_pages:] = c.pool.reshape(c.n_pages, per)
    w = torch.zeros(n, heads, page, device=cuda)
    c.table += (c.table >= 0).int() * (n - c.n_pages)
    c.cache = ks.Kv4Cache(pool, n, page, heads, d, group, weights=w)
    q = _query(c, 16, "f32")
    out, lse = _attend(c, q, 0.1, accumulate=True)
    c.ok()
    _check(c, q, 0.1, out, lse, "f32", weights=w[n - c.n_pages:], before=np.zeros((c.n_pages, heads, page)))
    k = torch.zeros(2, heads, d, device=cuda)
    ks.kv4_append_async(c.cache, c.table, c.seq_lens, k + 3, k - 5, status=c.status)
    ko, vo = torch.zeros_like(k), torch.zeros_like(k)
    ks.kv4_read_async(c.cache, c.table, c.seq_lens, ko, vo, status=c.status)
    c.ok()
    assert torch.allclose(ko, k + 3, rtol=2**-10) and torch.allclose(vo, k - 5, rtol=2**-10)


def test_streams_and_graphs(ks, cuda):
    """A captured step follows lengths, table and queries; two graphs with a workspace each on two streams."""
    import torch

    c = Seqs(ks, cuda, [900, 350], [1, 1], 2, 128, 32, 64, garbage=False)
    qs = [_query(c, 8, "f32", seed=i) for i in range(2)]
    graphs, outs, ws = [], [], []
    need = ks.kv4_attention_workspace(c.cache, 8, 2, 2, 1, 960)
    assert need > 0
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        out, lse = torch.zeros_like(qs[i]), torch.zeros(2, 8, device=cuda)
        ws.append(torch.zeros(need, dtype=torch.uint8, device=cuda))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            ks.kv4_attention_async(c.cache, c.table, c.seq_lens, qs[i], out, 0.1, ws[i], max_len=960, lse=lse,
                                   status=c.status, stream=streams[i])
        graphs.append(g)
        outs.append((out, lse))
    pages = np.concatenate(c.pages)  # without accumulated weights, sequences may share pages
    for lens in ([900, 350], [1, 960], [257, 0]):
        c.lens, c.pages = lens, [pages[: -(-n // 64)] for n in lens]
        c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        for s in range(2):
            c.table[s] = -1
            c.table[s, : len(c.pages[s])] = torch.from_numpy(c.pages[s].astype(np.int32)).to(cuda)
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        c.ok()
        for i in range(2):
            _check(c, qs[i], 0.1, *outs[i], "f32")
    del graphs


def test_bad_descriptors_are_reported(ks, cuda):
    """Pages outside the pool, lengths beyond the table, offsets beyond the rows: status word 0, nothing outside
    the buffers is touched, the other sequences are served."""
    import torch

    def fresh():
        return Seqs(ks, cuda, [100, 40], [1, 1], 2, 64, 32, 16, weights=True)

    def good(c, q, out, lse, s=1):
        torch.cuda.synchronize()
        assert c.status.cpu().tolist() == [1, 0]
        want, _, _, _, _ = O.kv4_attention(q.double().cpu().numpy()[s:s + 1], c.cached(s, "k"), c.cached(s, "v"),
                                           0.1, 1)
        assert np.abs(out.double().cpu().numpy()[s] - want[0]).max() < 1e-3

    for page in (-1, 1 << 20, -(1 << 31)):
        c = fresh()
        q = _query(c, 4, "f32")
        c.table[0, 2] = page
        out, lse = _attend(c, q, 0.1, accumulate=True)
        good(c, q, out, lse)
    for length in (-1, 1 << 30, 200):
        c = fresh()
        q = _query(c, 4, "f32")
        c.seq_lens[0] = length
        out, lse = _attend(c, q, 0.1, max_len=112)
        good(c, q, out, lse)
        assert (out[0] == 0).all()
        x = torch.randn(2, 2, 64, device=cuda)
        before = c.pool.clone()
        ks.kv4_append_async(c.cache, c.table, c.seq_lens, x, x, status=c.status)
        changed = (c.pool != before).flatten(1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= set(c.pages[1].tolist())
    c = fresh()
    q = _query(c, 4, "f32")
    c.offsets = torch.tensor([0, 1, 7], dtype=torch.int32, device=cuda)
    out = torch.full_like(q, 7)
    _attend(c, q, 0.1, out=out)
    torch.cuda.synchronize()
    assert c.status.cpu().tolist() == [1, 0] and (out[1] == 7).all()


# ---------------------------------------------------------------------- eviction
def _evict(c, budget, recent, kept=True, to_lens=None, status=None):
    import torch

    keep = [min(n, budget) for n in c.lens]
    each = [-(-n // c.page) for n in keep]
    used = c.n_pages
    n = used + sum(each) + 1
    pool = torch.full((n, *c.pool.shape[1:]), 0xEE, dtype=torch.uint8, device=c.cuda)
    pool[:used] = c.pool
    w = torch.full((n, c.heads, c.page), 7.0, device=c.cuda)
    w[:used] = c.w
    table = np.full((len(c.lens), max(each + [1]) + 1), -1, np.int32)
    at = used
    for s, k in enumerate(each):
        table[s, :k] = np.arange(at, at + k)
        at += k
    cache = c.ks.Kv4Cache(pool, n, c.page, c.heads, c.d, c.group, weights=w)
    max_len = max(c.lens)
    kept = torch.full((len(c.lens), c.heads, budget), -1, dtype=torch.int32, device=c.cuda) if kept else None
    to_lens = torch.full((len(c.lens),), -5, dtype=torch.int32, device=c.cuda) if to_lens is None else to_lens
    ws = torch.full((c.ks.kv4_evict_workspace(cache, len(c.lens), max_len, budget),), 255, dtype=torch.uint8,
                    device=c.cuda)
    to_table = torch.from_numpy(table).to(c.cuda)
    c.ks.kv4_evict_async(cache, c.table, c.seq_lens, to_table, to_lens, max_len, budget, recent, ws, kept=kept,
                         status=c.status)
    return cache, pool, w, table, to_table, to_lens, kept, keep


def _kept_of(w, n, budget, recent):
    """Positions kept of one head's weights w [n]."""
    if n <= budget:
        return np.arange(n)
    old = n - recent
    key = np.where(np.isnan(w[:old]), -np.inf, w[:old].astype(np.float64))
    key = np.where(np.isnan(w[:old]), np.finfo(np.float64).min, np.where(np.isneginf(w[:old]), -1e300, key))
    order = np.argsort(-key, kind="stable")[: budget - recent]
    return np.concatenate([np.sort(order), np.arange(old, n)])


@pytest.mark.parametrize("d,group,page", [(128, 32, 16), (64, 64, 64), (128, 128, 256), (64, 32, 32)])
@pytest.mark.parametrize("lens,budget,recent", [
    ([100, 1, 40, 0, 41], 40, 8),
    ([300, 5000], 33, 33),    # only the newest
    ([700, 64], 63, 0),       # only the heaviest
    ([9000], 4099, 17),
    ([3], 1, 1),
])
def test_evict(ks, cuda, d, group, page, lens, budget, recent):
    import torch

    c = Seqs(ks, cuda, lens, [0] * len(lens), 2, d, group, page, weights=True, seed=budget)
    ties = torch.from_numpy(np.random.default_rng(1).integers(0, 6, tuple(c.w.shape)).astype(np.float32)).to(cuda)
    c.w.copy_(torch.where(torch.rand_like(c.w) < 0.5, ties / 5, c.w))
    c.w[torch.rand_like(c.w) < 0.02] = float("nan")
    c.w[torch.rand_like(c.w) < 0.02] = -0.0
    c.w[torch.rand_like(c.w) < 0.01] = float("inf")
    c.w[torch.rand_like(c.w) < 0.01] = -float("inf")
    before = c.pool.clone()
    cache, pool, w, table, to_table, to_lens, kept, keep = _evict(c, budget, recent)
    c.ok()
    assert to_lens.tolist() == keep and torch.equal(pool[: c.n_pages], before)
    old, new = c.w.cpu().numpy(), w.cpu().numpy()
    src, dst = c.pool.cpu().numpy(), pool.cpu().numpy()
    per, half = 2 * (d // group), src.shape[-1] // 2

    def row(p, h, page_id, slot):
        b = p[page_id, h, slot // 16]
        i = slot % 16
        return np.concatenate([x for o in (0, half) for x in (b[o + i * (d // 2):o + (i + 1) * (d // 2)],
                                                              b[o + 8 * d + i * per:o + 8 * d + (i + 1) * per])])

    for s, n in enumerate(lens):
        for h in range(c.heads):
            at = c.weights_of(s, old)[h]
            want = _kept_of(at, n, budget, recent)
            assert kept[s, h, : keep[s]].tolist() == want.tolist(), (s, h)
            assert (kept[s, h, keep[s]:] == -1).all()
            for i in list(range(min(keep[s], 20))) + list(range(max(keep[s] - 20, 0), keep[s])):
                a, b = c.pages[s][want[i] // page], table[s, i // page]
                assert (row(src, h, a, want[i] % page) == row(dst, h, b, i % page)).all()
            got = np.concatenate([new[p, h] for p in table[s] if p >= 0] + [np.zeros(0, np.float32)])
            np.testing.assert_array_equal(got[: keep[s]], at[want])
            assert (got[keep[s]:] == 7).all()


def test_evict_long(ks, cuda):
    """More tokens than keys fit shared memory."""
    import torch

    n, budget, recent = 60001, 20011, 13
    c = Seqs(ks, cuda, [n, 300], [0, 0], 1, 64, 64, 256, weights=True)
    c.w.copy_(torch.floor(c.w * 4096) / 4096)  # with ties
    _, _, w, _, _, to_lens, kept, keep = _evict(c, budget, recent)
    c.ok()
    assert to_lens.tolist() == keep == [budget, 300]
    at = c.weights_of(0, c.w.cpu().numpy())[0]
    assert (kept[0, 0].cpu().numpy() == _kept_of(at, n, budget, recent)).all()
    assert kept[1, 0, :300].tolist() == list(range(300))


def test_evict_in_place_lengths_and_no_list(ks, cuda):
    c = Seqs(ks, cuda, [90, 20, 64], [0] * 3, 3, 64, 32, 16, weights=True)
    _, _, _, _, _, to_lens, _, keep = _evict(c, 50, 10, kept=False, to_lens=c.seq_lens)
    c.ok()
    assert c.seq_lens.tolist() == keep


# ------------------------------------------------------------------ all together
@pytest.mark.parametrize("dtype,d,group,q_heads", [("f32", 128, 32, 8), ("bf16", 64, 64, 6)])
def test_generation(ks, cuda, dtype, d, group, q_heads):
    """A prompt, decode steps that accumulate weights, an eviction, more steps: as the definition has them."""
    import torch

    heads, page, prompts = 2, 16, [70, 30]
    rng = np.random.default_rng(4)
    T = _type(dtype)
    n_pages = 40
    pool = torch.full((n_pages, ks.kv4_page_bytes(page, heads, d, group)), 0xFF, dtype=torch.uint8, device=cuda)
    w = torch.full((n_pages, heads, page), float("nan"), device=cuda)
    cache = ks.Kv4Cache(pool, n_pages, page, heads, d, group, weights=w)
    ids = rng.permutation(n_pages).astype(np.int32)
    table = torch.from_numpy(ids[:20].reshape(2, 10).copy()).to(cuda)
    lens = torch.zeros(2, dtype=torch.int32, device=cuda)
    status = torch.zeros(2, dtype=torch.int32, device=cuda)
    ref = [dict(k=[np.zeros((0, d))] * heads, v=[np.zeros((0, d))] * heads, w=[np.zeros(0)] * heads) for _ in range(2)]
    half = torch.finfo(T).eps / 2

    def step(news):
        tokens = sum(news)
        x = [torch.from_numpy(rng.standard_normal((tokens, n, d))).to(T).to(cuda) for n in (q_heads, heads, heads)]
        offsets = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=cuda)
        lens.add_(torch.tensor(news, dtype=torch.int32, device=cuda))
        ks.kv4_append_async(cache, table, lens, x[1], x[2], token_offsets=offsets, status=status)
        out, lse = torch.zeros_like(x[0]), torch.zeros(tokens, q_heads, device=cuda)
        ws = torch.zeros(max(16, ks.kv4_attention_workspace(cache, q_heads, 2, tokens, max(news), 160)),
                         dtype=torch.uint8, device=cuda)
        ks.kv4_attention_async(cache, table, lens, x[0], out, d**-0.5, ws, token_offsets=offsets, max_new=max(news),
                               max_len=160, lse=lse, accumulate=True, status=status)
        torch.cuda.synchronize()
        assert status.tolist() == [0, 0]
        q, k, v = (t.double().cpu().numpy() for t in x)
        at = 0
        for s, n in enumerate(news):
            r = ref[s]
            for h in range(heads):
                for name, y in (("k", k), ("v", v)):
                    r[name][h] = np.concatenate([r[name][h], O.kv4_value(*O.kv4_quantize(y[at:at + n, h], group))])
                r["w"][h] = np.concatenate([r["w"][h], np.zeros(n)])
            g = q_heads // heads
            for h in range(heads):
                want, z, add, size, _ = O.kv4_attention(q[at:at + n, h * g:(h + 1) * g], r["k"][h][:, None],
                                                        r["v"][h][:, None], d**-0.5, n)
                r["w"][h] = r["w"][h] + add[0]
                got = out[at:at + n, h * g:(h + 1) * g].double().cpu().numpy()
                assert (np.abs(got - want) <= half * np.abs(want) + 2.0**-10 * size).all()
            at += n

    step(prompts)
    for _ in range(3):
        step([1, 1])
    step([2, 4])
    # the heads keep different tokens
    to = torch.from_numpy(ids[20:40].reshape(2, 10).copy()).to(cuda)
    budget, recent = 40, 6
    kept = torch.full((2, heads, budget), -1, dtype=torch.int32, device=cuda)
    ws = torch.zeros(ks.kv4_evict_workspace(cache, 2, 160, budget), dtype=torch.uint8, device=cuda)
    old = lens.tolist()
    ks.kv4_evict_async(cache, table, lens, to, lens, 160, budget, recent, ws, kept=kept, status=status)
    torch.cuda.synchronize()
    assert lens.tolist() == [min(n, budget) for n in old]
    for s in range(2):
        for h in range(heads):
            at = kept[s, h, : lens[s]].tolist()
            r = ref[s]
            assert at == sorted(set(at)) and at[-recent:] == list(range(old[s] - recent, old[s]))
            # f32 sums and the roundings of the scores may swap weights that are nearly the same
            low = np.sort(r["w"][h][: old[s] - recent])[::-1]
            if old[s] > budget:
                assert r["w"][h][at[:-recent]].min() >= low[budget - recent - 1] * (1 - 2.0**-10)
            r["k"][h], r["v"][h], r["w"][h] = r["k"][h][at], r["v"][h][at], r["w"][h][at]
    table.copy_(to)
    for _ in range(3):
        step([1, 1])
    step([3, 1])


def test_with_the_w4a8_products(ks, cuda, oracle):
    """A decode step around the cache, as the library's other calls make it: queries, keys and values are columns of one
    W4A8 GEMM's output, read and appended in place, and the attention's result is quantised for the next GEMM."""
    import torch

    m, hidden, heads, kv_heads, d, group, page = 6, 512, 8, 2, 64, 32, 16
    cols = (heads + 2 * kv_heads) * d
    rng = np.random.default_rng(8)
    x = rng.integers(-127, 128, (m, hidden), dtype=np.int8)
    sx = rng.uniform(0.002, 0.004, m).astype(np.float32)
    w = [rng.integers(0, 256, (n, k // 2), dtype=np.uint8) for n, k in ((cols, hidden), (hidden, heads * d))]
    sw = [rng.uniform(2e-3, 4e-3, (n, k // 32)).astype(np.float16) for n, k in ((cols, hidden), (hidden, heads * d))]
    dev = lambda a: torch.from_numpy(a.view(np.uint16) if a.dtype == np.float16 else a).to(cuda)  # noqa: E731
    lens = [9, 40, 1, 17, 33, 64]
    c = Seqs(ks, cuda, lens, [1] * m, kv_heads, d, group, page)
    qkv = torch.zeros(m, cols, device=cuda)
    ks.gemm_w4a8_async(dev(x), dev(sx), dev(w[0]), dev(sw[0]), qkv, m, cols, hidden, 32, status=c.status)
    rows = qkv.view(m, heads + 2 * kv_heads, d)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    ks.kv4_append_async(c.cache, c.table, c.seq_lens, k, v, status=c.status)
    out, lse = _attend(c, q, d**-0.5, out=torch.zeros(m, heads, d, device=cuda), offsets=False)
    a, sa = torch.zeros(m, heads * d, dtype=torch.int8, device=cuda), torch.zeros(m, device=cuda)
    ks.quantize_per_token_async(out, heads * d, m, heads * d, a, heads * d, sa)
    y = torch.zeros(m, hidden, device=cuda)
    ks.gemm_w4a8_async(a, sa, dev(w[1]), dev(sw[1]), y, m, hidden, heads * d, 32, status=c.status)
    c.ok()
    # the definition, from the GEMM's own output on
    for s, n in enumerate(lens):
        p, slot = c.pages[s][(n - 1) // page], (n - 1) % page
        c.k[p, :, slot] = O.kv4_value(*O.kv4_quantize(k[s].double().cpu().numpy(), group))
        c.v[p, :, slot] = O.kv4_value(*O.kv4_quantize(v[s].double().cpu().numpy(), group))
        c.scale_max = max(c.scale_max, O.kv4_quantize(k[s].double().cpu().numpy(), group)[1].astype(np.float64).max())
    _check(c, q, d**-0.5, out, lse, "f32")
    for s in range(m):
        rc, want = oracle.matvec_w4a8_f16(x[s], w[0], hidden // 2, sw[0].view(np.uint16), hidden // 32, cols, hidden, 32,
                                          float(sx[s]))
        assert rc == 0 and O.w4a8_tolerance_ok(qkv[s].cpu().numpy(), want)[0]
        rc, qs, scale = oracle.quantize_per_token(out[s].reshape(-1).cpu().numpy())
        assert (a[s].cpu().numpy() == qs).all() and float(sa[s]) == np.float32(scale)
        rc, want = oracle.matvec_w4a8_f16(qs, w[1], heads * d // 2, sw[1].view(np.uint16), heads * d // 32, hidden,
                                          heads * d, 32, float(scale))
        assert rc == 0 and O.w4a8_tolerance_ok(y[s].cpu().numpy(), want)[0]


def test_one_workspace_for_attention_and_eviction_in_turn(ks, cuda):
    """The eviction leaves the words alone that the attention wants to be 0, whatever they hold."""
    import torch

    c = Seqs(ks, cuda, [3000, 700], [1, 1], 2, 128, 32, 64, weights=True, seed=4)
    q = _query(c, 8, "f32")
    to_pool_pages = 2 * 32
    n = c.n_pages + to_pool_pages
    pool, w = torch.zeros((n, *c.pool.shape[1:]), dtype=torch.uint8, device=cuda), torch.zeros((n, 2, 64), device=cuda)
    pool[: c.n_pages], w[: c.n_pages] = c.pool, c.w
    cache = ks.Kv4Cache(pool, n, 64, 2, 128, 32, weights=w)
    to_table = torch.arange(c.n_pages, n, dtype=torch.int32, device=cuda).reshape(2, 32)
    to_lens = torch.zeros(2, dtype=torch.int32, device=cuda)
    need = max(ks.kv4_attention_workspace(cache, 8, 2, 2, 1, 3000), ks.kv4_evict_workspace(cache, 2, 3000, 2000))
    ws = torch.zeros(need, dtype=torch.uint8, device=cuda)
    outs = []
    for _ in range(2):
        out, lse = torch.zeros_like(q), torch.zeros(2, 8, device=cuda)
        ks.kv4_attention_async(cache, c.table, c.seq_lens, q, out, 0.1, ws, max_len=3000, lse=lse, status=c.status)
        outs.append((out, lse))
        ks.kv4_evict_async(cache, c.table, c.seq_lens, to_table, to_lens, 3000, 2000, 100, ws, status=c.status)
        assert not ws[:8192].any()
    ws[:8192] = 3
    ks.kv4_evict_async(cache, c.table, c.seq_lens, to_table, to_lens, 3000, 2000, 100, ws, status=c.status)
    c.ok()
    assert (ws[:8192] == 3).all() and to_lens.tolist() == [2000, 700]
    for out, lse in outs:
        _check(c, q, 0.1, out, lse, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_overlapping_launches_give_the_same(ks, cuda, dtype):
    """Steps that feed one another directly (append of what the attention gave, attention on its own result, eviction,
    read), on the default stream, where no launch overlaps another, on a stream of their own and as a graph there: the
    same bits."""
    import torch

    heads, q_heads, d, page, steps, n_seqs = 2, 8, 128, 64, 6, 3
    start = [700, 1, 130]
    pages = 16
    results = []
    side = torch.cuda.Stream()
    for mode in ("default", "side", "graph"):
        rng = torch.Generator(device=cuda).manual_seed(3)
        pool = torch.zeros(2 * n_seqs * pages, ks.kv4_page_bytes(page, heads, d, 32), dtype=torch.uint8, device=cuda)
        w = torch.zeros(2 * n_seqs * pages, heads, page, device=cuda)
        cache = ks.Kv4Cache(pool, len(pool), page, heads, d, 32, weights=w)
        table = torch.arange(n_seqs * pages, dtype=torch.int32, device=cuda).reshape(n_seqs, pages)
        to_table = table + n_seqs * pages
        status = torch.zeros(2, dtype=torch.int32, device=cuda)
        first = np.concatenate([[0], np.cumsum(start)])
        kv = torch.randn(2, first[-1], heads, d, generator=rng, device=cuda).to(_type(dtype))
        offsets = torch.tensor(first, dtype=torch.int32, device=cuda)
        lens = [torch.tensor([n + i for n in start], dtype=torch.int32, device=cuda) for i in range(steps + 1)]
        x = torch.randn(n_seqs, q_heads, d, generator=rng, device=cuda).to(_type(dtype))
        outs = [x] + [torch.zeros_like(x) for _ in range(steps)]
        lse = torch.zeros(n_seqs, q_heads, device=cuda)
        ws = torch.zeros(max(ks.kv4_attention_workspace(cache, q_heads, n_seqs, n_seqs, 1, 1024),
                             ks.kv4_evict_workspace(cache, n_seqs, 1024, 100)), dtype=torch.uint8, device=cuda)
        to_lens = torch.zeros(n_seqs, dtype=torch.int32, device=cuda)
        back = torch.zeros(2, n_seqs * 100, heads, d, device=cuda, dtype=_type(dtype))
        kept = [min(n + steps, 100) for n in start]
        back_offsets = torch.tensor(np.concatenate([[0], np.cumsum(kept)]), dtype=torch.int32, device=cuda)

        def chain(stream):
            pool.zero_()
            w.zero_()
            ks.kv4_append_async(cache, table, lens[0], kv[0], kv[1], token_offsets=offsets, status=status,
                                stream=stream)
            for i in range(steps):
                ks.kv4_append_async(cache, table, lens[i + 1], outs[i][:, ::4], outs[i][:, 1::4], status=status,
                                    stream=stream)
                ks.kv4_attention_async(cache, table, lens[i + 1], outs[i], outs[i + 1], 0.3, ws, max_len=1024, lse=lse,
                                       accumulate=True, status=status, stream=stream)
            ks.kv4_evict_async(cache, table, lens[steps], to_table, to_lens, 1024, 100, 10, ws, status=status,
                               stream=stream)
            ks.kv4_read_async(cache, to_table, to_lens, back[0], back[1], token_offsets=back_offsets, status=status,
                              stream=stream)

        torch.cuda.synchronize()
        if mode == "default":
            chain(None)
        else:
            with torch.cuda.stream(side):
                chain(side)
            side.synchronize()
            if mode == "graph":
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=side):
                    chain(torch.cuda.current_stream())
                for t in outs[1:] + [back, lse]:
                    t.zero_()
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        assert status.tolist() == [0, 0] and to_lens.tolist() == kept
        results.append([t.clone() for t in outs[1:] + [back, lse, w, pool]])
    assert results[0][-4].float().abs().sum() > 0 and results[0][-2].sum() > 0
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("tokens,heads", [(80000, 1), (60001, 2), (9473, 3)])
def test_append_and_read_more_tokens_than_the_gpu_holds_at_once(ks, cuda, tokens, heads):
    """CTAs of many tokens, in one wave or several, the last one short."""
    import torch

    d, group, page = 64, 32, 256
    pages = -(-tokens // page)
    pool = torch.zeros(pages, ks.kv4_page_bytes(page, heads, d, group), dtype=torch.uint8, device=cuda)
    cache = ks.Kv4Cache(pool, pages, page, heads, d, group)
    table = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=cuda)[None]
    lens = torch.tensor([tokens], dtype=torch.int32, device=cuda)
    offsets = torch.tensor([0, tokens], dtype=torch.int32, device=cuda)
    kv = torch.randn(2, tokens, heads, d, generator=torch.Generator(device=cuda).manual_seed(5), device=cuda)
    back = torch.full_like(kv, float("nan"))
    status = torch.zeros(2, dtype=torch.int32, device=cuda)
    ks.kv4_append_async(cache, table, lens, kv[0], kv[1], token_offsets=offsets, status=status)
    ks.kv4_read_async(cache, table, lens, back[0], back[1], token_offsets=offsets, status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0]
    q, s = O.kv4_quantize(kv.double().cpu().numpy().reshape(-1, d), group)
    want = q.reshape(-1, d // group, group) * s.reshape(-1, d // group, 1).astype(np.float64)
    assert (back.double().cpu().numpy().reshape(want.shape) == want).all()


def test_captured_over_two_streams(ks, cuda):
    """Calls after a join of streams, and after copies and fills, in a graph: launches that may overlap what is before
    them in one stream still come after all of it."""
    import torch

    c = Seqs(ks, cuda, [900, 333], [1, 1], 2, 128, 32, 64, weights=True, seed=8)
    q = _query(c, 8, "f32")
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    k, v = torch.randn(2, 2, 2, 128, device=cuda)
    want_cache, want_w = c.pool.clone(), c.w.clone()
    ws = [torch.zeros(ks.kv4_attention_workspace(c.cache, 8, 2, 2, 1, 1024), dtype=torch.uint8, device=cuda)
          for _ in range(2)]
    out = [torch.zeros_like(q) for _ in range(2)]
    lse = [torch.zeros(2, 8, device=cuda) for _ in range(2)]
    back = torch.zeros(2, 2, 2, 128, device=cuda)
    qa, ka = torch.zeros_like(q), torch.zeros_like(k)

    def both(first, second):
        qa.copy_(q)
        ka.copy_(k)
        ks.kv4_append_async(c.cache, c.table, c.seq_lens, ka, v, status=c.status, stream=first)
        second.wait_stream(first)
        with torch.cuda.stream(second):
            ks.kv4_attention_async(c.cache, c.table, c.seq_lens, qa, out[1], 0.2, ws[1], max_len=1024, lse=lse[1],
                                   status=c.status, stream=second)
        ks.kv4_read_async(c.cache, c.table, c.seq_lens, back[0], back[1], status=c.status, stream=first)
        first.wait_stream(second)
        ks.kv4_attention_async(c.cache, c.table, c.seq_lens, out[1], out[0], 0.2, ws[0], max_len=1024, lse=lse[0],
                               accumulate=True, status=c.status, stream=first)
        qa.zero_()

    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        both(a, b)
    torch.cuda.synchronize()
    wants = [t.clone() for t in (*out, *lse, back, c.pool, c.w)]
    assert wants[0].abs().sum() > 0 and not torch.equal(wants[6], want_w)
    g = torch.cuda.CUDAGraph()
    c.pool.copy_(want_cache)
    with torch.cuda.graph(g, stream=a):
        c.w.copy_(want_w)
        both(torch.cuda.current_stream(), b)
    for t in (*out, *lse, back):
        t.zero_()
    for _ in range(4):
        g.replay()
    c.ok()
    for got, want in zip((*out, *lse, back, c.pool, c.w), wants):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,d,q_heads,n", [("f16", 64, 1, 524288), ("f16", 128, 12, 262144), ("bf16", 64, 4, 262144)])
def test_long_items_whole_in_a_cta(ks, cuda, dtype, d, q_heads, n):
    """As many sequences as there are CTAs (more than there are with 16 rows), on the same pages, each of them long, with
    values of one sign and a late rise of the scores: sums over many tiles of one CTA.

    Bound.  Truncating steps of the accumulators, each up to 2^-23 of the sum, go on for 128 products:
    2^-16.  The f32 sums over a warp's (at most 128) such stretches and 4 warps: 2^-17.  Exponentials and the two parts of
    the weights (2^-18), their sum and the division (2^-20): 2^-15 in all, 2^-11 more in one f16 part (bf16).  The scores
    (at most about 2^5, over 2^4 products of 2^-23 or less) move all the weights of a row by 2^-16 at most.  Values are
    positive, so all of this is relative to the result, which is then rounded once."""
    import torch

    T, page, seqs = _type(dtype), 256, 444
    pages = n // page
    pool = torch.zeros(pages, ks.kv4_page_bytes(page, 1, d, 64), dtype=torch.uint8, device=cuda)
    cache = ks.Kv4Cache(pool, pages, page, 1, d, 64)
    table = torch.arange(pages, dtype=torch.int32, device=cuda).repeat(seqs, 1)
    lens = torch.full((seqs,), n, dtype=torch.int32, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randn(1, q_heads, d, generator=gen, device=cuda)
    k = torch.randn(n, 1, d, generator=gen, device=cuda) * 0.1
    k[n // 2:] += 6.0 / 0.125 * q.mean(1) / (q.mean(1) ** 2).sum()  # the mean query's scores by 6
    v = torch.rand(n, 1, d, generator=gen, device=cuda) + 1.0
    q = q.to(T)
    offsets = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    status = torch.zeros(2, dtype=torch.int32, device=cuda)
    ks.kv4_append_async(cache, table[:1], lens[:1], k, v, token_offsets=offsets, status=status)
    ks.kv4_read_async(cache, table[:1], lens[:1], k, v, token_offsets=offsets, status=status)
    out = torch.zeros(seqs, q_heads, d, dtype=T, device=cuda)
    lse = torch.zeros(seqs, q_heads, device=cuda)
    ws = torch.zeros(ks.kv4_attention_workspace(cache, q_heads, seqs, seqs, 1, n), dtype=torch.uint8, device=cuda)
    ks.kv4_attention_async(cache, table, lens, q.expand(seqs, q_heads, d), out, 0.125, ws, max_len=n, lse=lse,
                           status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0]
    x = q[0].double() @ k[:, 0].double().T * 0.125
    want, z = torch.softmax(x, -1) @ v[:, 0].double(), torch.logsumexp(x, -1)
    assert x.abs().max() < 40
    rel = torch.finfo(T).eps / 2 + 2.0**-15 + 2.0**-16 + (2.0**-11 if dtype == "bf16" else 0)
    worst = max(float(((o.double() - want) / want).abs().max()) for o in out)
    assert worst <= rel, worst
    assert ((lse.double() - z).abs() <= 2.0**-16 + 2.0**-22 * z.abs()).all()


@pytest.mark.parametrize("part", ["first", "last", "middle"])
def test_tables_that_are_columns_of_wider_ones(ks, cuda, part):
    """The same as with tables of their own; a sequence longer than the columns hold is reported, and the pages that the
    columns beside them name are neither read nor written."""
    import torch

    c = Seqs(ks, cuda, [100, 40], [1, 1], 2, 64, 32, 16, weights=True, spare=30)
    columns, to_columns, budget = c.table.shape[1], 2, 32
    at = {"first": 0, "last": 12, "middle": 5}[part]
    others = np.setdiff1d(np.arange(c.n_pages), np.concatenate(c.pages))
    to_pages = others[:4].reshape(2, 2)
    beside = torch.from_numpy(others[4:24].astype(np.int32)).to(cuda)

    def wide(table):  # columns of a wider one, which for the last rows ends the storage
        n = table.shape[1]
        big = beside.repeat(2)[: 2 * 20].reshape(2, 20).clone()[:, : at + n if part == "last" else 20].contiguous()
        big[:, at:at + n] = table
        return big[:, at:at + n]

    own = c.table.clone()
    to_own = torch.from_numpy(to_pages.astype(np.int32)).to(cuda)
    q = _query(c, 4, "f32")
    x = torch.randn(2, 2, 2, 64, device=cuda)
    start, wstart = c.pool.clone(), c.w.clone()
    results = []
    for table, to_table in ((own, to_own), (wide(own), wide(to_own))):
        c.pool.copy_(start)
        c.w.copy_(wstart)
        c.table = table
        ks.kv4_append_async(c.cache, table, c.seq_lens, x[0], x[1], status=c.status)
        back = torch.zeros_like(x)
        ks.kv4_read_async(c.cache, table, c.seq_lens, back[0], back[1], status=c.status)
        out, lse = _attend(c, q, 0.1, accumulate=True, max_len=16 * columns)
        to_lens = torch.zeros(2, dtype=torch.int32, device=cuda)
        ws = torch.zeros(ks.kv4_evict_workspace(c.cache, 2, 100, budget), dtype=torch.uint8, device=cuda)
        ks.kv4_evict_async(c.cache, table, c.seq_lens, to_table, to_lens, 100, budget, 8, ws, status=c.status)
        c.ok()
        results.append((back, out, lse, to_lens, c.pool.clone(), c.w.clone()))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    # the last row's sequence one page longer than its columns
    before, wbefore = c.pool.clone(), c.w.clone()
    long = torch.tensor([100, 16 * columns + 5], dtype=torch.int32, device=cuda)
    ks.kv4_append_async(c.cache, c.table, long, x[0], x[1], status=c.status)
    torch.cuda.synchronize()
    assert c.status.tolist() == [1, 0]
    changed = (c.pool != before).flatten(1).any(1) | (c.w != wbefore).flatten(1).any(1)
    assert set(changed.nonzero().flatten().tolist()) <= set(c.pages[0].tolist())
    c.status.zero_()
    back = torch.full_like(x, 7)
    ks.kv4_read_async(c.cache, c.table, long, back[0], back[1], status=c.status)
    torch.cuda.synchronize()
    assert c.status.tolist() == [1, 0] and (back[:, 1] == 7).all() and not (back[:, 0] == 7).any()
    # one sequence, whose table of one row has no distance to a next one
    column = torch.from_numpy(c.pages[0].astype(np.int32)).to(cuda)[:, None]
    c.status.zero_()
    back = torch.zeros(2, 1, 2, 64, device=cuda)
    ks.kv4_read_async(c.cache, column.t(), c.seq_lens[:1], back[0], back[1], status=c.status)
    c.ok()
    assert torch.equal(back[:, 0], results[0][0][:, 0])


@pytest.mark.parametrize("name", ["append", "read"])
@pytest.mark.parametrize("n", [3, 600])
def test_bad_descriptors_of_sequences_without_rows(ks, cuda, name, n):
    """Offsets beyond the rows and offsets that fall are reported though no row of the call is theirs, a bad length though
    the sequence has no new token."""
    import torch

    d, heads, page = 64, 2, 16
    pool = torch.zeros(2 * n, ks.kv4_page_bytes(page, heads, d, 32), dtype=torch.uint8, device=cuda)
    cache = ks.Kv4Cache(pool, 2 * n, page, heads, d, 32)
    table = torch.arange(2 * n, dtype=torch.int32, device=cuda).reshape(n, 2)
    call = ks.kv4_append_async if name == "append" else ks.kv4_read_async

    def status_of(news, tokens, change=None, at=0, value=0):
        offsets = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=cuda)
        lens = torch.full((n,), 20, dtype=torch.int32, device=cuda)
        if change == "offset":
            offsets[at] = value
        if change == "length":
            lens[at] = value
        x = torch.ones(2, tokens, heads, d, device=cuda)
        status = torch.zeros(2, dtype=torch.int32, device=cuda)
        call(cache, table, lens, x[0], x[1], token_offsets=offsets, status=status)
        torch.cuda.synchronize()
        return status.tolist()

    idle = [4] + [0] * (n - 1)
    assert status_of(idle, 4) == [0, 0] and status_of([4] * n, 4 * n) == [0, 0]
    assert status_of(idle[:-1] + [5], 4) == [1, 0]  # the last sequence's rows are all beyond the tensors'
    for at in (1, n - 1):
        for length in (-1, 33, 1 << 30):
            assert status_of(idle, 4, "length", at, length) == [1, 0]
    for value in (2, -5, 5):  # fall at the sequence before or behind, or go beyond the rows
        assert status_of(idle, 4, "offset", n - 1, value) == [1, 0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group,heads,q_heads,lens,news", [
    (128, 32, 2, 8, [3000, 700, 33, 1], [1, 1, 1, 1]),
    (64, 64, 3, 3, [1500, 90, 400], [1, 1, 1]),
    (128, 128, 1, 6, [800, 64], [9, 5]),
    (64, 32, 2, 2, [900, 5], [30, 5]),
])
def test_lse_and_weights_by_their_norms(ks, cuda, dtype, d, group, heads, q_heads, lens, news):
    """lse and the added weights of all rows together, where roundings do not add up to their worst case.

    A score's error, per row: its roundings to f32 (as for the outputs' norm) 2^-22 |z|, sums, exponentials and the
    logarithm 2^-20.  f16 and bf16 queries: the products run in accumulators that truncate, half of 2^-23 of the partial
    sum in the mean over d / 16 steps, and that partial sum is about 8 |sum q| of a group (from which it starts) and
    8 sqrt(sum q^2) (codes + 8, of random signs) times the key scale.  f32 queries: what is left of two parts, 2^-23 of
    the row's largest element over d elements of random sign, times the keys' root mean square.  A weight's relative
    error is that of the score and of lse, an exponential (2^-21) and the sums (2^-23)."""
    c = Seqs(ks, cuda, lens, news, heads, d, group, 16, seed=d + group, weights=True)
    before = c.w.double().cpu().numpy()
    q, scale = _query(c, q_heads, dtype), d**-0.5
    out, lse = _attend(c, q, scale, accumulate=True)
    c.ok()
    qn, lse = q.double().cpu().numpy(), lse.double().cpu().numpy()
    after = c.w.double().cpu().numpy()
    sums = np.abs(qn.reshape(*qn.shape[:2], -1, group).sum(-1)).max(-1)
    if dtype == "f32":
        product = 2.0**-23 * np.abs(qn).max(-1) * d**0.5 * (c.k**2).mean() ** 0.5
    else:
        product = 2.0**-24 * d / 16 * 8 * c.scale_max * (sums + np.sqrt((qn**2).sum(-1)))
    err = most = werr = wmost = 0.0
    for s in range(len(lens)):
        a, n = c.first[s], news[s]
        _, z, w, _, _ = O.kv4_attention(qn[a:a + n], c.cached(s, "k"), c.cached(s, "v"), scale, n)
        seen = np.isfinite(z)
        bound = np.where(seen, 2.0**-20 + 2.0**-22 * np.abs(np.where(seen, z, 0)), 0) \
            + scale * product[a:a + n]
        err, most = err + ((lse[a:a + n] - z)[seen] ** 2).sum(), most + (bound[seen] ** 2).sum()
        old, got = c.weights_of(s, before), c.weights_of(s, after)
        rel = 2 * bound.max() + 2.0**-21
        werr = werr + ((got - old - w) ** 2).sum()
        wmost = wmost + ((rel * w + 2.0**-23 * (old + w)) ** 2).sum()
    assert err**0.5 <= most**0.5, (err**0.5, most**0.5)
    assert werr**0.5 <= wmost**0.5, (werr**0.5, wmost**0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group,q_heads", [(128, 32, 4), (64, 64, 1), (128, 64, 12), (128, 128, 2), (64, 32, 9)])
@pytest.mark.parametrize("order", ["last", "first", "groups", "shared"])
def test_values_of_unlike_sizes(ks, cuda, dtype, d, group, q_heads, order):
    """A result far below the values that have next to no weight in it keeps its bits.

    last, first: one token has all the weight, its values are 2^-k of the others', which come before or after it.
    groups: the first groups' values are 2^k of the others', in every token.  shared: the large values have weights of
    about 2^-k, so that both are in the result.  Errors by group and head, against the group's norm: scores of up to 64
    are rounded to f32 (2^-21 of |lse|), exponentials, sums and the two parts are within 2^-17, one part of bf16 2^-12,
    and the result is rounded once."""
    import torch

    T, n, page = _type(dtype), 300, 32
    half = torch.finfo(T).eps / 2
    for k in (12, 18, 24, 30, 38):
        c = Seqs(ks, cuda, [n], [1], 1, d, group, page, seed=k, garbage=True)
        gen = torch.Generator(device=cuda).manual_seed(k)
        # the largest scale is 2^12, the least 2^(12 - k) about
        big, small = 2.0**12 * 7, 2.0**12 * 7 * 2.0**-min(k, 34)
        keys = torch.zeros(n, 1, d, device=cuda)
        values = torch.randn(n, 1, d, generator=gen, device=cuda).clamp(-1, 1) * 0.83  # scales of many bits
        one = {"first": 7, "last": 290}.get(order, 150)
        gap = min(k, 34) * 0.693 if order == "shared" else 64.0
        if order == "groups":
            values *= torch.where(torch.arange(d, device=cuda) < max(group, d // 2), big, small)
            if group == d:
                continue
        else:
            keys[one] = gap / d
            values *= big
            values[one] *= small / big
        offsets = torch.tensor([0, n], dtype=torch.int32, device=cuda)
        ks.kv4_append_async(c.cache, c.table, c.seq_lens, keys, values, token_offsets=offsets, status=c.status)
        ks.kv4_read_async(c.cache, c.table, c.seq_lens, keys, values, token_offsets=offsets, status=c.status)
        q = torch.ones(1, q_heads, d, device=cuda).to(T)
        out, lse = _attend(c, q, 1.0)
        c.ok()
        want, z, _, _, _ = O.kv4_attention(q.double().cpu().numpy(), keys.double().cpu().numpy(),
                                           values.double().cpu().numpy(), 1.0, 1)
        got = out.double().cpu().numpy()
        tiny = float(torch.finfo(T).smallest_normal) * half  # of results below the type's normal numbers
        most = half + 2.0**-17 + 2.0**-21 * np.abs(z).max() + (2.0**-12 if dtype == "bf16" else 0)
        err = np.sqrt(((got - want).reshape(q_heads, -1, group) ** 2).sum(-1))
        norm = np.sqrt((want.reshape(q_heads, -1, group) ** 2).sum(-1))
        assert (err <= most * norm + 2 * tiny * group**0.5).all(), (k, (err / norm).max(), most)


@pytest.mark.parametrize("dtype,d,q_heads", [("f16", 128, 2), ("bf16", 64, 9), ("f32", 128, 1)])
def test_values_of_unlike_sizes_in_long_items(ks, cuda, dtype, d, q_heads):
    """The same where each CTA goes over a long item: its first three quarters have the large values and together a weight
    of 2^-24, the rest values 2^-30 of theirs and, but for the last token, lower scores still."""
    import torch

    T, n, page, seqs, group = _type(dtype), 40000, 64, 444, 64
    pages = -(-n // page)
    pool = torch.zeros(pages, ks.kv4_page_bytes(page, 1, d, group), dtype=torch.uint8, device=cuda)
    cache = ks.Kv4Cache(pool, pages, page, 1, d, group)
    table = torch.arange(pages, dtype=torch.int32, device=cuda).repeat(seqs, 1)
    lens = torch.full((seqs,), n, dtype=torch.int32, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(2)
    score = torch.rand(n, 1, 1, generator=gen, device=cuda) * 8  # e^8 = 2^11.5
    score[3 * n // 4:] -= 8
    score[-1] = 33  # 2^47.6 against the sum of 30000 of up to 2^11.5
    k = (score / d).expand(n, 1, d).contiguous()
    v = torch.randn(n, 1, d, generator=gen, device=cuda) * 2.0**12
    v[3 * n // 4:] *= 2.0**-30
    offsets = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    status = torch.zeros(2, dtype=torch.int32, device=cuda)
    ks.kv4_append_async(cache, table[:1], lens[:1], k, v, token_offsets=offsets, status=status)
    ks.kv4_read_async(cache, table[:1], lens[:1], k, v, token_offsets=offsets, status=status)
    q = torch.ones(seqs, q_heads, d, dtype=T, device=cuda)
    out, lse = torch.zeros_like(q), torch.zeros(seqs, q_heads, device=cuda)
    ws = torch.zeros(ks.kv4_attention_workspace(cache, q_heads, seqs, seqs, 1, n), dtype=torch.uint8, device=cuda)
    ks.kv4_attention_async(cache, table, lens, q, out, 1.0, ws, max_len=n, lse=lse, status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0]
    x = q[0].double() @ k[:, 0].double().T
    p = torch.softmax(x, -1)
    want, z = p @ v[:, 0].double(), torch.logsumexp(x, -1)
    # both parts are in the result, within 2^6 of one another
    parts = [(p[:, a] @ v[a, 0].double()).norm() for a in (slice(0, 3 * n // 4), slice(3 * n // 4, n))]
    assert 2.0**-6 < parts[0] / parts[1] < 2.0**6
    most = torch.finfo(T).eps / 2 + 2.0**-17 + 2.0**-16 + 2.0**-21 * z.max() + (2.0**-12 if dtype == "bf16" else 0)
    tiny = torch.finfo(T).smallest_normal * torch.finfo(T).eps  # of results below the type's normal numbers
    err = (out.double() - want).unflatten(-1, (-1, group)).norm(dim=-1)
    norm = want.unflatten(-1, (-1, group)).norm(dim=-1)
    assert (err <= most * norm + tiny * group**0.5).all(), ((err / norm).max(), most)


def test_append_from_most_rows(ks, cuda):
    """As many rows as a call takes (one in memory, its stride 0), three of them a sequence's."""
    import torch

    d, page, rows = 64, 16, 2**31 - 1
    pool = torch.zeros(2, ks.kv4_page_bytes(page, 1, d, 64), dtype=torch.uint8, device=cuda)
    cache = ks.Kv4Cache(pool, 2, page, 1, d, 64)
    table = torch.arange(2, dtype=torch.int32, device=cuda)[None]
    lens = torch.tensor([20], dtype=torch.int32, device=cuda)
    status = torch.zeros(2, dtype=torch.int32, device=cuda)
    x = torch.randn(1, 1, d, device=cuda).expand(rows, 1, d)
    offsets = torch.tensor([rows - 3, rows], dtype=torch.int32, device=cuda)
    ks.kv4_append_async(cache, table, lens, x, x, token_offsets=offsets, status=status)
    back = torch.zeros(2, 3, 1, d, device=cuda)
    ks.kv4_read_async(cache, table, lens, back[0], back[1], token_offsets=offsets - (rows - 3), status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0]
    want = O.kv4_value(*O.kv4_quantize(x[0].double().cpu().numpy(), 64))
    assert (back.double().cpu().numpy() == want).all()


@pytest.mark.parametrize("heads", [65, 130])
def test_more_heads_than_a_turn_of_a_cta(ks, cuda, heads):
    """Append and read, attention with weights and eviction with more heads than a CTA has rows under way."""
    import torch

    d, group, page = 64, 64, 16
    c = Seqs(ks, cuda, [40, 7, 19], [5, 7, 1], heads, d, group, page, weights=True, garbage=False)
    x = torch.randn(2, c.tokens, heads, d, device=cuda)
    ks.kv4_append_async(c.cache, c.table, c.seq_lens, x[0], x[1], token_offsets=c.offsets, status=c.status)
    back = torch.zeros_like(x)
    ks.kv4_read_async(c.cache, c.table, c.seq_lens, back[0], back[1], token_offsets=c.offsets, status=c.status)
    c.ok()
    want = O.kv4_value(*O.kv4_quantize(x.double().cpu().numpy(), group))
    assert (back.double().cpu().numpy() == want).all()
    for s in range(3):
        for j in range(c.news[s]):
            pos = c.lens[s] - c.news[s] + j
            c.k[c.pages[s][pos // page], :, pos % page] = want[0, c.first[s] + j]
            c.v[c.pages[s][pos // page], :, pos % page] = want[1, c.first[s] + j]
    c.scale_max = max(c.scale_max, np.abs(want[0]).max() / 7)
    before = c.w.double().cpu().numpy()
    q = _query(c, heads, "f32")
    out, lse = _attend(c, q, 0.125, accumulate=True)
    c.ok()
    _check(c, q, 0.125, out, lse, "f32", weights=c.w, before=before)
    _, _, _, _, _, to_lens, kept, keep = _evict(c, 12, 3)
    c.ok()
    w = c.w.cpu().numpy()
    assert to_lens.tolist() == keep
    for s in range(3):
        for h in range(heads):
            assert kept[s, h, : keep[s]].tolist() == _kept_of(c.weights_of(s, w)[h], c.lens[s], 12, 3).tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group,q_heads,heads,lens,news", [
    (64, 32, 128, 1, [50, 300], [1, 1]),  # one key/value head for all
    (128, 64, 142, 2, [77, 9], [1, 2]),
    (64, 64, 2, 1, [300, 40], [300, 1]),  # a prompt from its first token, beside a decode row
    (128, 128, 1, 1, [500], [213]),
])
def test_many_rows_to_a_head(ks, cuda, dtype, d, group, q_heads, heads, lens, news):
    c = Seqs(ks, cuda, lens, news, heads, d, group, 32, seed=q_heads, weights=True)
    before = c.w.double().cpu().numpy()
    big = _query(c, q_heads + 1, dtype).reshape(c.tokens, -1)  # rows that start at any element
    q = big[:, 1:1 + q_heads * d].unflatten(1, (q_heads, d))
    out, lse = _attend(c, q, d**-0.5, accumulate=True)
    c.ok()
    _check(c, q, d**-0.5, out, lse, dtype, weights=c.w, before=before)


def test_thousands_of_sequences(ks, cuda):
    lens = [int(x) for x in np.random.default_rng(0).integers(0, 4, 5000)]
    c = Seqs(ks, cuda, lens, [min(x, 1) for x in lens], 1, 64, 64, 16, weights=True, spare=3)
    before = c.w.double().cpu().numpy()
    q = _query(c, 2, "f32")
    out, lse = _attend(c, q, 0.125, accumulate=True)
    c.ok()
    _check(c, q, 0.125, out, lse, "f32", weights=c.w, before=before)


def test_a_captured_step_follows_its_offsets(ks, cuda):
    """Drafted tokens in a graph: how many each sequence has, and where its rows are, changes between replays."""
    import torch

    heads, q_heads, d, group, page, rows = 2, 6, 64, 32, 16, 12
    c = Seqs(ks, cuda, [96, 80, 48], [4, 4, 4], heads, d, group, page, garbage=False)  # pages for what comes
    x = torch.randn(2, rows, heads, d, device=cuda)
    q = torch.randn(rows, q_heads, d, device=cuda)
    out, lse = torch.zeros_like(q), torch.zeros(rows, q_heads, device=cuda)
    ws = torch.zeros(ks.kv4_attention_workspace(c.cache, q_heads, 3, rows, 8, 96), dtype=torch.uint8, device=cuda)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        ks.kv4_append_async(c.cache, c.table, c.seq_lens, x[0], x[1], token_offsets=c.offsets, status=c.status,
                            stream=stream)
        ks.kv4_attention_async(c.cache, c.table, c.seq_lens, q, out, 0.125, ws, token_offsets=c.offsets, max_new=8,
                               max_len=96, lse=lse, status=c.status, stream=stream)
    values = O.kv4_value(*O.kv4_quantize(x.double().cpu().numpy(), group))
    for news, first, lens in (([4, 4, 4], 0, [90, 64, 33]), ([1, 8, 0], 2, [91, 70, 33]), ([0, 1, 1], 10, [91, 71, 34])):
        c.lens, c.news, c.first = lens, news, first + np.concatenate([[0], np.cumsum(news)]).astype(int)
        c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        c.offsets.copy_(torch.tensor(c.first, dtype=torch.int32))
        out.fill_(7)
        g.replay()
        c.ok()
        for s in range(3):
            for j in range(news[s]):
                pos = lens[s] - news[s] + j
                c.k[c.pages[s][pos // page], :, pos % page] = values[0, c.first[s] + j]
                c.v[c.pages[s][pos // page], :, pos % page] = values[1, c.first[s] + j]
        c.scale_max = max(c.scale_max, np.abs(values[0]).max() / 7)
        _check(c, q, 0.125, out, lse, "f32")
        assert (out[:first] == 7).all() and (out[c.first[-1]:] == 7).all()
    del g
