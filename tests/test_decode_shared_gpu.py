"""Attention over a paged cache with a shared history (``esgpt::attn_decode_shared``) against a plain implementation in
64 bits, alone and together with the operators that fill the cache.

Tolerances, from u = 2^-24: a score is a chain of hd products and additions, off by (hd + 8) u of its terms'
sizes, and a probability by twice that (its own and the normaliser's) + 16 u; the sum over n keys adds (n / 16 + 64) u
(16 or 32 keys enter each accumulation). All of it relative to sum_j p_j |v_j|. With bf16 data P is rounded for the
matrix product, half a step (2^-8) of each term, and so is the result.
"""
import math

import pytest
import torch

U = 2.0**-24
gpu = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def ops():
    from eventstreamgpt_amd import ops as O

    return O.load()


def err():
    from eventstreamgpt_amd import kernels as K

    return K.err_word(torch.device(DEV, torch.cuda.current_device()))


@pytest.fixture(autouse=True)
def _clear(request):
    on = request.node.get_closest_marker("gpu") is not None
    if on:
        err().zero_()
    yield
    if on:
        err().zero_()


class Case:
    """Pools, tables and lengths on the CPU (``dev`` moves them), queries [G n, Lq, H hd]."""

    def __init__(self, G, n, Lq, H, hd, ps, P, s, window=0, dt=F32, seed=0, ragged=True, share=False, masked=False):
        g = torch.Generator().manual_seed(seed)
        S = G * n
        self.G, self.n, self.S, self.Lq, self.H, self.hd, self.ps, self.window, self.dt = G, n, S, Lq, H, hd, ps, window, dt
        pp, sp = -(-P // ps), -(-s // ps)
        pages = (pp + sp if share else G * pp + S * sp) + 2
        at = torch.randperm(pages, generator=g).int()
        if share:  # every group reads the same pages, and so does every sequence
            self.prefix_table = at[:pp].repeat(G, 1)
            self.table = at[pp: pp + sp].repeat(S, 1)
        else:
            self.prefix_table, self.table = at[: G * pp].view(G, pp), at[G * pp: G * pp + S * sp].view(S, sp)
        self.prefix_lens = torch.randint(P // 2 if ragged else P, P + 1, (G,), generator=g).int()
        self.past = torch.randint(0 if ragged else s - Lq, s - Lq + 1, (S,), generator=g).int()
        self.row_mask = torch.rand(S, Lq, generator=g) < 0.6 if masked else None
        std = 1.3 * hd**-0.25
        self.q = (std * torch.randn(S, Lq, H * hd, generator=g)).to(dt)
        self.kp = (std * torch.randn(pages, H, ps, hd, generator=g)).to(dt)
        self.vp = torch.randn(pages, H, ps, hd, generator=g).to(dt)
        self.P, self.s = P, s

    def own_row(self, s, i):
        return int(self.past[s]) + (i if self.row_mask is None else int(self.row_mask[s, :i].sum()))

    def run(self, **kw):
        d = dict(q=self.q, k_pages=self.kp, v_pages=self.vp, prefix_table=self.prefix_table if self.P else None,
                 prefix_lens=self.prefix_lens if self.P else None, page_table=self.table, past=self.past,
                 row_mask=self.row_mask, prefix_cap=self.P, cap=self.s, window=self.window)
        d.update(kw)
        d = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
        d.setdefault("err", err())
        return ops().attn_decode_shared(**d)

    def rows(self, pool, table, lo, hi):
        """Rows lo .. hi - 1 named by one table row, [hi - lo, H, hd], in 64 bits; bad pages leave no rows: their
        places are returned too."""
        j = torch.arange(lo, hi)
        page = table.long()[j // self.ps] if hi > lo else j
        ok = (page >= 0) & (page < pool.shape[0])
        return pool[page.clamp(0, max(pool.shape[0] - 1, 0)), :, j % self.ps].double(), ok

    def oracle(self):
        """(o, sum_j p_j |v_j|, largest sum_d |q_d k_d| of a row, keys of a row), [S, Lq, H, hd] or broadcastable."""
        o = torch.zeros(self.S, self.Lq, self.H, self.hd, dtype=torch.float64)
        mag, size = torch.zeros_like(o), torch.zeros(self.S, self.Lq, self.H, 1, dtype=torch.float64)
        for s in range(self.S):
            gr = s // self.n
            P = min(max(int(self.prefix_lens[gr]), 0), self.P) if self.P else 0
            for i in range(self.Lq):
                if self.row_mask is not None and not bool(self.row_mask[s, i]) or int(self.past[s]) < 0:
                    continue
                at = self.own_row(s, i)
                lo_p = max(0, P + at - self.window + 1) if self.window else 0
                lo_s = max(0, at - self.window + 1) if self.window else 0
                hi_s = min(at + 1, self.s)
                parts = []
                if min(lo_p, P) < P:
                    parts.append((self.prefix_table[gr], lo_p, P))
                if lo_s < hi_s:
                    parts.append((self.table[s], lo_s, hi_s))
                ks, vs = [], []
                for tab, lo, hi in parts:
                    k, ok = self.rows(self.kp, tab, lo, hi)
                    v, _ = self.rows(self.vp, tab, lo, hi)
                    ks.append(k[ok])
                    vs.append(v[ok])
                if not ks or sum(k.shape[0] for k in ks) == 0:
                    continue
                k, v = torch.cat(ks), torch.cat(vs)
                q = self.q[s, i].double().view(1, self.H, self.hd)
                p = torch.softmax((q * k).sum(-1), 0)[..., None]
                o[s, i], mag[s, i] = (p * v).sum(0), (p * v.abs()).sum(0)
                size[s, i, :, 0] = (q * k).abs().sum(-1).amax(0)
        return o, mag, size

    def check(self, got, want=None):
        o, mag, size = want or self.oracle()
        got = got.cpu().double().view(self.S, self.Lq, self.H, self.hd)
        n = self.P + self.s
        rel = 2 * (self.hd + 8) * U * size + (16 + n / 16 + 64) * U
        lim = (rel + (2.0**-8 if self.dt == BF16 else 0)) * mag + (2.0**-8 if self.dt == BF16 else U) * o.abs()
        bad = ~((got - o).abs() <= lim)
        assert not bad.any(), (bad.sum().item(), (got - o).abs().max().item(), ((got - o).abs() / lim.clamp_min(1e-30)).max().item())


CASES = [
    # G, n, Lq, H, hd, ps, P, s, window
    (1, 1, 1, 1, 8, 16, 1, 1, 0),        # the smallest call: one history row, one own row
    (1, 4, 1, 4, 16, 16, 40, 6, 0), (2, 3, 1, 2, 24, 16, 0, 19, 0),  # no history at all
    (3, 5, 1, 4, 64, 64, 77, 33, 0), (2, 16, 1, 2, 32, 32, 130, 64, 0),
    (2, 17, 1, 2, 64, 64, 300, 20, 0),   # a row tile of one row
    (1, 40, 1, 2, 96, 32, 201, 9, 0), (2, 3, 1, 3, 128, 16, 99, 40, 0), (1, 33, 1, 1, 128, 128, 640, 5, 0),
    (2, 4, 3, 2, 64, 32, 70, 21, 0), (1, 9, 16, 2, 40, 16, 50, 31, 0), (2, 2, 2, 2, 16, 16, 17, 2, 0),
    (2, 4, 1, 2, 64, 64, 300, 40, 32),   # the window reaches from the own rows into the history
    (2, 20, 1, 2, 64, 64, 150, 90, 64), (2, 4, 4, 2, 32, 16, 40, 30, 5), (1, 3, 2, 1, 64, 16, 33, 18, 1),
    (2, 3, 1, 2, 64, 64, 90, 20, 100000),
    (1, 6, 1, 2, 64, 64, 9001, 700, 0),  # many parts of a row
    (1, 2, 1, 1, 64, 16, 500, 3000, 0), (1, 40, 2, 1, 64, 64, 5000, 40, 700),
    # enough (group, head)s for one workgroup each to do history and own rows in one launch
    (16, 9, 1, 8, 64, 32, 100, 40, 0), (32, 3, 2, 4, 128, 16, 70, 20, 0), (16, 3, 1, 8, 96, 16, 90, 12, 20),
    (33, 2, 1, 8, 40, 16, 20, 5, 0), (32, 20, 1, 4, 24, 16, 33, 9, 0), (32, 2, 5, 8, 16, 16, 600, 70, 0),
    (64, 8, 1, 4, 16, 16, 30, 200, 0), (64, 8, 1, 4, 64, 16, 60, 200, 150),  # own rows are most of it, even among the waves
    (64, 1, 1, 4, 64, 64, 20, 400, 0), (1, 100, 1, 1, 64, 64, 90, 12, 0), (70, 1, 1, 4, 64, 16, 0, 90, 0),
]


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", CASES, ids=str)
def test_against_the_oracle(c, dt):
    x = Case(*c, dt=dt)
    x.check(x.run())
    assert int(err()[0]) == 0


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [(64, 1, 1, 16, 16, 64, 4500, 1300, 0), (64, 1, 1, 16, 16, 64, 9000, 1100, 0),
                               (64, 20, 1, 16, 16, 32, 8300, 2, 0), (300, 1, 1, 16, 16, 64, 3, 2300, 0)], ids=str)
def test_more_keys_in_a_part_than_a_round_of_page_ids(c, dt):
    """Enough workgroups that a history (or own) part is longer than 64 page ids reach; all sequences name the same
    pages. The first sequences and the last one are checked."""
    x = Case(*c, dt=dt, share=True)
    got = x.run()
    keep = sorted({0, 1, x.S // 2, x.S - 1})
    G, n = x.G, x.n
    sub = Case(*c, dt=dt, share=True)
    for s in keep:
        sub.S, sub.G, sub.n = 1, 1, 1
        sub.prefix_table, sub.prefix_lens = x.prefix_table[s // n: s // n + 1], x.prefix_lens[s // n: s // n + 1]
        sub.table, sub.past, sub.q = x.table[s: s + 1], x.past[s: s + 1], x.q[s: s + 1]
        sub.check(got[s: s + 1])


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [(2, 5, 4, 2, 64, 16, 50, 20, 0), (2, 9, 3, 2, 32, 16, 60, 30, 7), (3, 4, 1, 2, 64, 16, 20, 9, 0)],
                         ids=str)
def test_padded_rows(c, dt):
    """Rows that row_mask drops are zeros; a sequence with none left gives zeros; the others see the same keys as ever."""
    x = Case(*c, dt=dt, masked=True)
    x.row_mask[0] = False
    got = x.run()
    x.check(got)
    assert (got[~x.row_mask.to(DEV)] == 0).all()


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf, "lowest"])
def test_what_lies_beyond_a_length_never_counts(dt, junk):
    """Unused rows of used pages and unused pages hold NaN, infinities or the type's lowest value."""
    junk = torch.finfo(dt).min if junk == "lowest" else junk
    for c in [(2, 5, 1, 2, 64, 64, 70, 21, 0), (2, 3, 3, 2, 24, 16, 30, 12, 9), (1, 18, 1, 2, 96, 32, 45, 33, 0)]:
        x = Case(*c, dt=dt)
        want = x.oracle()
        clean = x.run()
        used = torch.zeros(x.kp.shape[0], x.ps, dtype=torch.bool)
        for gr in range(x.G):
            for j in range(int(x.prefix_lens[gr])):
                used[x.prefix_table[gr, j // x.ps], j % x.ps] = True
        for s in range(x.S):
            for j in range(x.own_row(s, x.Lq - 1) + 1):
                used[x.table[s, j // x.ps], j % x.ps] = True
        m = ~used[:, None, :, None]
        x.kp.masked_fill_(m, junk)
        x.vp.masked_fill_(m, junk)
        got = x.run()
        assert torch.equal(got, clean)
        x.check(got, want)


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("junk", [math.nan, math.inf])
def test_not_finite_values_reach_only_the_rows_that_see_them(dt, junk):
    """A value that is not finite at a key which some rows of a tile see and others do not (a window's edge in the
    history, a later new event, another trajectory's own row)."""
    x = Case(1, 6, 3, 2, 64, 16, 60, 14, window=20, dt=dt, ragged=True, seed=3)
    clean = x.run().view(x.S, x.Lq, x.H, x.hd)
    want = x.oracle()
    P = int(x.prefix_lens[0])
    kill = torch.zeros(x.S, x.Lq, x.H, x.hd, dtype=torch.bool)
    # one history row near the windows' edges, dimension 5 of head 1; one row of sequence 2, dimension 40 of head 0
    j = P - 12
    x.vp[x.prefix_table[0, j // 16], 1, j % 16, 5] = junk
    t = x.own_row(2, 1)
    x.vp[x.table[2, t // 16], 0, t % 16, 40] = junk
    for s in range(x.S):
        for i in range(x.Lq):
            if P + x.own_row(s, i) - j < x.window:
                kill[s, i, 1, 5] = True
    kill[2, 1:, 0, 40] = True
    assert kill[:, :, 1, 5].any() and not kill[:, :, 1, 5].all()
    got = x.run().view(x.S, x.Lq, x.H, x.hd)
    assert not torch.isfinite(got.cpu()[kill]).any()
    ok = ~kill
    o, mag, size = want
    x.check(torch.where(kill.to(DEV), clean, got), want)
    assert torch.isfinite(got.cpu()[ok]).all()
    # a key that is not finite makes the rows that see it NaN and no other
    x.kp[x.table[4, x.own_row(4, 2) // 16], 0, x.own_row(4, 2) % 16, 3] = math.nan
    got = x.run().view(x.S, x.Lq, x.H, x.hd)
    assert got[4, 2, 0].isnan().all() and torch.isfinite(got[4, :2, 0].cpu()).all()


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_large_scores(dt):
    """Scores of several hundred, one key far above the rest, all keys equal: the running maximum carries them."""
    for c in [(1, 4, 1, 2, 64, 16, 200, 20, 0), (1, 20, 1, 2, 64, 64, 900, 20, 0)]:
        x = Case(*c, dt=dt)
        x.q *= 40
        x.check(x.run())
        x = Case(*c, dt=dt)
        x.kp[x.prefix_table[0, 3], :, 7] *= 30
        x.check(x.run())
        x.kp.fill_(0.25)
        x.check(x.run())


@gpu
def test_bad_pages_and_lengths_are_flagged_and_not_read():
    from eventstreamgpt_amd import kernels as K

    for spoil in ("page", "own_page", "prefix_len", "prefix_len_negative", "past", "past_negative"):
        x = Case(2, 3, 2, 2, 32, 16, 64, 32, ragged=False)
        x.check(x.run())
        K.check_errors()
        if spoil == "page":
            x.prefix_table[0, 1], x.prefix_table[1, 2] = x.kp.shape[0], -5
        elif spoil == "own_page":
            x.table[1, 0], x.table[4, 1] = 2**31 - 1, -(2**31)
        elif spoil == "prefix_len":
            x.prefix_lens[1] = 2**31 - 1
        elif spoil == "prefix_len_negative":
            x.prefix_lens[0] = -7
        elif spoil == "past":
            x.past[2] = 2**31 - 1
        else:
            x.past[3] = -1
        got = x.run()
        if spoil == "past":  # all of the table's rows are visible, no more
            x.past[2] = x.s - 1
        x.check(got)
        with pytest.raises(IndexError, match="paged cache"):
            K.check_errors()
        K.check_errors()
    x = Case(2, 3, 1, 2, 32, 16, 64, 32)
    got = x.run(k_pages=x.kp[:0], v_pages=x.vp[:0])
    assert (got == 0).all()
    with pytest.raises(IndexError):
        K.check_errors()


@gpu
def test_bounds_wider_than_the_lengths():
    """Caps far above the lengths (a cache with room to grow) change the split, not the result beyond rounding."""
    for dt in (F32, BF16):
        x = Case(2, 3, 1, 2, 64, 16, 400, 300, dt=dt)
        x.prefix_lens, x.past = torch.tensor([3, 0]).int(), torch.tensor([0, 1, 2, 0, 17, 299]).int()
        want = x.oracle()
        x.check(x.run(), want)
        x.P, x.s = 400, 300
        x.check(x.run(prefix_cap=x.prefix_table.shape[1] * 16, cap=x.table.shape[1] * 16), want)


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [(2, 33, 1, 8, 64, 16, 300, 20, 0), (2, 25, 2, 8, 20, 64, 700, 20, 0), (1, 70, 1, 16, 32, 16, 90, 9, 0),
                               (2, 17, 3, 8, 96, 16, 200, 12, 0)], ids=str)
def test_tiles_of_32_rows_over_long_bounds(c, dt):
    """Bounds that a long history would need (the work is split by them) over short ones, which makes the tiles 32 rows
    high; padded rows; NaN in the used pages' unused rows."""
    x = Case(*(c if c[4] % 8 == 0 or dt == F32 else (*c[:4], 24, *c[5:])), dt=dt, masked=c[2] > 1)
    want = x.oracle()
    for table, lens in ((x.prefix_table, x.prefix_lens), (x.table, torch.tensor([x.own_row(s, x.Lq) for s in range(x.S)]))):
        for pages, n in zip(table.long(), lens.tolist()):
            for i, page in enumerate(pages.tolist()):
                x.kp[page, :, min(max(n - i * x.ps, 0), x.ps):] = math.nan
                x.vp[page, :, min(max(n - i * x.ps, 0), x.ps):] = math.nan
    x.prefix_table = torch.cat([x.prefix_table, torch.full((x.G, 16384 // x.ps), -1).int()], 1)
    cap = x.prefix_table.shape[1] * x.ps
    got = x.run(prefix_cap=cap)
    x.P = cap
    x.check(got, want)
    assert int(err()[0]) == 0


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_long_windows_and_an_infinity_at_their_edges(dt):
    """32 rows a tile whose windows of 8,500 begin at different history rows; then an infinity where some begin."""
    x = Case(2, 20, 1, 16, 40, 64, 9000, 30, 8500, dt=dt, seed=5)
    x.prefix_lens = torch.tensor([9000, 8777]).int()
    want = x.oracle()
    got = x.run()
    x.check(got, want)
    j = 9000 - 8500 + 12  # seen by the first group's rows with at most 11 own rows before them
    x.vp[x.prefix_table[0, j // 64], 3, j % 64, 7] = math.inf
    sees = torch.zeros(x.S, 1, x.H, x.hd, dtype=torch.bool)
    sees[:20, 0, 3, 7] = 9000 + x.past[:20] - j < 8500
    assert sees.any() and not sees[:20, 0, 3, 7].all()
    dirty = x.run().view(sees.shape)
    assert not torch.isfinite(dirty.cpu()[sees]).any()
    x.check(torch.where(sees.to(DEV), got.view(sees.shape), dirty), want)


@gpu
def test_layouts_streams_and_repeats():
    x = Case(2, 9, 2, 4, 64, 64, 700, 50, dt=BF16)
    want = x.run()
    D = x.H * x.hd
    wide = torch.zeros(x.S, x.Lq, 3 * D, dtype=BF16, device=DEV)
    wide[..., :D] = x.q.to(DEV)
    odd = torch.zeros(x.q.numel() + 1, dtype=BF16, device=DEV)
    odd[1:] = x.q.reshape(-1).to(DEV)
    for q in (wide[..., :D], odd[1:].view(x.q.shape)):
        assert torch.equal(x.run(q=q), want)
    st = torch.cuda.Stream()
    q, e = x.q.to(DEV), err()
    st.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        got = x.run(q=q, err=e)
    here = x.run()  # at the same time on this stream: workspaces are the calls' own
    st.synchronize()
    assert torch.equal(got, want) and torch.equal(here, want)


@gpu
def test_captured_generation_steps():
    """One graph with an append and the attention; each replay takes the next event (past grows on the device), with
    eager work on the same cache layout in between."""
    x = Case(2, 4, 1, 2, 64, 16, 100, 48, dt=BF16, ragged=False)
    D = x.H * x.hd
    d = {k: getattr(x, k).to(DEV) for k in ("prefix_table", "prefix_lens", "table", "kp", "vp")}
    past = torch.zeros(x.S, dtype=torch.int32, device=DEV)
    qkv = torch.zeros(x.S, 1, 3 * D, dtype=BF16, device=DEV)
    pos = torch.zeros(x.S, 1, device=DEV)
    f = torch.exp(-torch.arange(32, device=DEV) / 8).float()
    w = torch.full((64,), 64**-0.25, device=DEV)

    def step(kp, vp):
        q = ops().kv_append_paged(qkv, kp, vp, d["table"], past, None, w, w, pos, f, 1e-6, err())
        return ops().attn_decode_shared(q, kp, vp, d["prefix_table"], d["prefix_lens"], d["table"], past, None, 100, 48, 0,
                                        err())

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(d["kp"].clone(), d["vp"].clone())
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(d["kp"], d["vp"])
    kp, vp = d["kp"].clone(), d["vp"].clone()
    g = torch.Generator().manual_seed(1)
    for i in range(20):
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF16))
        pos.add_(37.5)
        graph.replay()
        eager = step(kp, vp)
        past.add_(1)
        torch.cuda.synchronize()
        assert torch.equal(held, eager) and torch.equal(kp, d["kp"]) and torch.equal(vp, d["vp"]), i
    assert int(err()[0]) == 0


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 24])
def test_prompt_then_generation(dt, window):
    """As a model layer runs them: the left-padded histories are normalised, rotated and attended with esgpt::attention
    and stored once; four trajectories of each continue event by event. Every new event's output equals causal
    attention over the whole sequence (history and own events) in 64 bits, and esgpt::attention's last row on it."""
    from eventstreamgpt_amd import kernels as K

    B, L, n, T, H, hd, ps = 3, 37, 4, 9, 4, 64, 16
    D, S = H * hd, B * n
    g = torch.Generator().manual_seed(2)
    pads = torch.tensor([0, 11, 30])
    mask = (torch.arange(L)[None] >= pads[:, None]).to(DEV)
    w = [(hd**-0.25 * (1 + 0.2 * torch.randn(hd, generator=g))).to(DEV) for _ in range(2)]
    f = torch.exp(torch.arange(0, hd, 2) * (-math.log(10000.0) / hd)).float().to(DEV)
    hist = torch.randn(B, L, 3 * D, generator=g).to(dt).to(DEV)
    t_hist = torch.exp(3 + torch.randn(B, L, generator=g)).cumsum(1).to(DEV)
    new = torch.randn(S, T, 3 * D, generator=g).to(dt).to(DEV)
    t_new = (t_hist[:, -1:].repeat_interleave(n, 0).cpu() + torch.exp(3 + torch.randn(S, T, generator=g)).cumsum(1)).to(DEV)

    cache = K.PagedKV(64, ps, H, hd, dt, DEV)
    prefix_table = torch.stack([cache.pages(-(-L // ps)) for _ in range(B)])
    table = torch.stack([cache.pages(-(-T // ps)) for _ in range(S)])
    zero = torch.zeros(B, dtype=torch.int32, device=DEV)
    ops().kv_append_paged(hist, cache.k, cache.v, prefix_table, zero, mask, *w, t_hist, f, 1e-6, err())
    prefix_lens = mask.sum(1).int()
    past = torch.zeros(S, dtype=torch.int32, device=DEV)
    whole = torch.cat([hist.repeat_interleave(n, 0), new], 1)
    times = torch.cat([t_hist.repeat_interleave(n, 0), t_new], 1)
    keys = torch.cat([mask.repeat_interleave(n, 0), torch.ones(S, T, dtype=torch.bool, device=DEV)], 1)
    y = K.qk_norm_rope(whole, *w, times, f, H)
    for i in range(T):
        q = cache.append(new[:, i: i + 1], table, past, None, *w, t_new[:, i: i + 1], f)
        o = cache.attend(q, table, past, T, prefix_table, prefix_lens, L, window=window)
        past += 1
        end = L + i + 1
        yq, yk, yv = y[:, :end].double().view(S, end, 3, H, hd).unbind(2)
        assert torch.equal(q[:, 0], y[:, end - 1, :D])
        sc = (yq[:, -1:] * yk).sum(-1)
        far = torch.arange(end, device=DEV)
        # index distance counts stored events: left padding is not stored, so it is the plain distance
        see = keys[:, :end] & ((end - 1 - far < window) if window else torch.ones_like(far, dtype=torch.bool))
        p = torch.softmax(sc.masked_fill(~see[..., None], -math.inf), 1)[..., None]
        want, mag = (p * yv).sum(1).reshape(S, D), (p * yv.abs()).sum(1).reshape(S, D)
        size = (yq[:, -1:] * yk).abs().sum(-1).amax().item()
        lim = (2 * (hd + 8) * U * size + 96 * U + (2.0**-8 if dt == BF16 else 0)) * mag + (2.0**-8 if dt == BF16 else U) * want.abs()
        assert ((o[:, 0].double() - want).abs() <= lim).all(), i
        ref, _, _ = ops().attention(y[:, :end].contiguous(), keys[:, :end].contiguous(), None, H, window, False, 0.0, None)
        assert ((ref[:, -1].double() - want).abs() <= 4 * lim + 1e-5).all(), i
    K.check_errors()


@gpu
def test_without_a_history_it_is_the_dense_cache_attention():
    """Paged rows of unequal lengths against esgpt::attn_decode over a dense copy, f32: two f32 results, each within
    its bound of the same number."""
    x = Case(5, 1, 1, 4, 32, 16, 0, 60)
    got = x.run()
    D = x.H * x.hd
    for s in range(x.S):
        Lk = int(x.past[s]) + 1
        k, v = (torch.stack([p[x.table[s, j // 16], :, j % 16] for j in range(Lk)]).reshape(1, Lk, D) for p in (x.kp, x.vp))
        qkv = torch.cat([x.q[s: s + 1], k[:, -1:], v[:, -1:]], -1).to(DEV)
        ref = ops().attn_decode(qkv, k.contiguous().to(DEV), v.contiguous().to(DEV), None, None, x.H, Lk, 0)
        assert (got[s] - ref[0]).abs().max() <= 2e-5
    x.check(got)


@gpu
def test_pools_beyond_32_bit_offsets():
    """Pages of 2 MiB whose elements lie past 2^31 (5 GiB pools): stored and read at their place."""
    H, hd, ps, pages = 8, 128, 1024, 2300
    kp, vp = (torch.empty(pages, H, ps, hd, dtype=BF16, device=DEV) for _ in range(2))
    for at in (kp, vp):
        at[0].zero_()
        at[-3:].zero_()
    x = Case(1, 2, 1, H, hd, 16, 20, 40, dt=BF16)
    table = torch.tensor([[pages - 1], [pages - 2]], dtype=torch.int32, device=DEV)
    pre = torch.tensor([[pages - 3]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(0)
    for tab, S, L in ((pre, 1, 20), (table, 2, 33)):
        rows = torch.randn(S, L, 3 * H * hd, generator=g).to(BF16).to(DEV)
        ops().kv_append_paged(rows, kp, vp, tab, torch.zeros(S, dtype=torch.int32, device=DEV), None, None, None, None, None,
                              1e-6, err())
        for s in range(S):
            assert torch.equal(kp[tab[s, 0], :, :L].transpose(0, 1).reshape(L, -1), rows[s, :, H * hd: 2 * H * hd])
    q = (0.1 * torch.randn(2, 1, H * hd, generator=g)).to(BF16)
    args = (torch.tensor([20]).int().to(DEV), table, torch.tensor([32, 7]).int().to(DEV), None, 20, 33, 0, err())
    big = ops().attn_decode_shared(q.to(DEV), kp, vp, pre, *args)
    sk, sv = kp[-3:].clone(), vp[-3:].clone()
    small = ops().attn_decode_shared(q.to(DEV), sk, sv, pre - (pages - 3), args[0], table - (pages - 3), *args[2:])
    assert torch.equal(big, small) and torch.isfinite(big).all() and (big != 0).any()
    assert (kp[0] == 0).all() and int(err()[0]) == 0


@gpu
def test_empty_calls():
    x = Case(2, 3, 1, 2, 32, 16, 64, 32)
    e = dict(q=x.q[:0], page_table=x.table[:0], past=x.past[:0], prefix_table=None, prefix_lens=None, prefix_cap=0)
    assert x.run(**e).shape == (0, 1, 64)
    assert x.run(q=x.q[:, :0]).shape == (6, 0, 64)


@gpu
def test_refusals():
    x = Case(2, 3, 1, 2, 32, 16, 64, 32)
    for kw, text in [
        (dict(q=x.q[..., :32]), "q must be"), (dict(q=x.q[0]), "q must be"), (dict(q=x.q.bfloat16()), "pages must be"),
        (dict(q=x.q.expand(6, 17, 64)), "at most 16"), (dict(prefix_table=None), "together"),
        (dict(prefix_lens=None), "together"), (dict(prefix_table=None, prefix_lens=None), "together"),
        (dict(prefix_table=x.prefix_table[:1].repeat(4, 1), prefix_lens=x.prefix_lens[:1].repeat(4)), "divide"),
        (dict(prefix_lens=x.prefix_lens[:1]), "prefix_lens"), (dict(prefix_table=x.prefix_table.long()), "prefix_table"),
        (dict(page_table=x.table[:3]), "page_table"), (dict(past=x.past.long()), "past"),
        (dict(row_mask=torch.ones(6, 2).bool()), "row_mask"), (dict(prefix_cap=65), "prefix_cap"),
        (dict(prefix_cap=-1), "prefix_cap"), (dict(cap=33), "cap"), (dict(cap=0), "cap"), (dict(window=-1), "window"),
        (dict(k_pages=x.kp[:, :, ::2]), "k_pages and v_pages"), (dict(err=torch.zeros(2, dtype=torch.int64)), "error block"),
    ]:
        if "err" in kw:
            with pytest.raises(RuntimeError, match=text):
                ops().attn_decode_shared(x.q.to(DEV), x.kp.to(DEV), x.vp.to(DEV), None, None, x.table.to(DEV), x.past.to(DEV),
                                         None, 0, 32, 0, kw["err"])
            continue
        with pytest.raises(RuntimeError, match=text):
            x.run(**kw)


# ------------------------------------------------------------------------------------------- without a device
def test_c_abi_refuses_before_it_launches():
    import os

    from eventstreamgpt_amd import _lib as L

    if not os.path.exists(L.LIB_PATH):
        pytest.skip("library not built")
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: only where no device could read them")
    lib = L.load(require_device=False)
    P = 4096

    def call(q=P, kp=P, vp=P, n_pages=9, ps=64, pt=P, pw=256, pl=P, G=2, tab=P, tw=2, past=P, o=P, S=6, Lq=1, H=4, hd=64,
             pcap=16384, cap=128, window=0, dt=1, ws=P, nb=1 << 30):
        return lib.esgpt_attn_decode_shared(q, kp, vp, n_pages, ps, pt, pw, pl, G, tab, tw, past, None, o, S, Lq, H, hd, pcap,
                                            cap, window, dt, ws, nb, None, None)

    for bad in (dict(q=None), dict(q=P + 8), dict(kp=None), dict(vp=P + 4), dict(n_pages=-1), dict(ps=8), dict(ps=96),
                dict(ps=131072), dict(pt=None), dict(pl=None), dict(G=0), dict(G=4), dict(G=7), dict(tab=None), dict(past=None),
                dict(o=None), dict(o=P + 2), dict(S=-1), dict(Lq=0), dict(Lq=17), dict(H=0), dict(hd=12), dict(hd=136), dict(hd=0),
                dict(pcap=-1), dict(pcap=16385), dict(cap=0), dict(cap=129), dict(window=-1), dict(dt=2), dict(ws=None),
                dict(ws=P + 4), dict(nb=64), dict(S=1 << 27), dict(S=1 << 22, H=16, hd=8), dict(tw=1 << 40),
                dict(pw=1 << 31)):
        assert call(**bad) == 1, bad
    assert call(S=0) == 0
    need = lib.esgpt_attn_decode_shared_workspace
    assert need(2, 6, 1, 4, 64, 16384, 128, 0, 1) > 0
    assert need(6, 6, 1, 4, 64, 0, 16, 0, 1) == 0         # one part: written directly
    assert need(2, 6, 17, 4, 64, 16384, 128, 0, 1) == 0   # not a valid call


def test_fake_tensors():
    o = ops()
    m = dict(device="meta", dtype=torch.int32)
    kp = torch.empty(4, 2, 16, 32, device="meta")
    q = torch.empty(3, 1, 64, device="meta")
    out = o.attn_decode_shared(q, kp, kp, None, None, torch.empty(3, 1, **m), torch.empty(3, **m), None, 0, 16, 0,
                               torch.empty(2, device="meta", dtype=torch.int64))
    assert out.shape == q.shape
    with pytest.raises(NotImplementedError, match="no_grad"):
        o.attn_decode_shared(q.requires_grad_(), kp, kp, None, None, torch.empty(3, 1, **m), torch.empty(3, **m), None, 0,
                             16, 0, torch.empty(2, device="meta", dtype=torch.int64))


def test_paged_cache_hands_out_each_page_once():
    from eventstreamgpt_amd import _lib as L
    from eventstreamgpt_amd import kernels as K
    from eventstreamgpt_amd.kernels import PagedKV

    c = PagedKV(6, 16, 2, 32, torch.float32, "cpu")
    assert c.k.shape == (6, 2, 16, 32) and c.v.shape == c.k.shape and c.k.dtype == torch.float32
    a, b = c.pages(2), c.pages(3)
    assert a.dtype == torch.int32 and sorted(a.tolist() + b.tolist()) == sorted(set(a.tolist() + b.tolist()))
    with pytest.raises(RuntimeError, match="1 of 6"):
        c.pages(2)
    c.release(a.view(1, 2))  # a page table's shape
    assert sorted(c.pages(3).tolist() + b.tolist()) == list(range(6))
    with pytest.raises(ValueError, match="not handed out"):
        c.release(torch.tensor([0, 0]))
    with pytest.raises(L.HipExtensionMissing):
        c.append(torch.zeros(1, 1, 192), a[None, :1], a[:1])
    with pytest.raises(NotImplementedError, match="no_grad"):
        c.attend(torch.zeros(1, 1, 64, requires_grad=True), a[None, :1], a[:1], 16)
    with pytest.raises(L.HipExtensionMissing):
        K.qk_norm_rope(torch.zeros(1, 1, 192), None, None, None, None, 2)
    for ps in (8, 24, 1 << 17):
        with pytest.raises(ValueError, match="page size"):
            PagedKV(2, ps, 2, 32, torch.float32, "cpu")


# ------------------------------------------------------------------------------------- accuracy of bf16 probabilities
def tight(x, got, want, extra=2.0**-15 + 2.0**-20):
    """As Case.check, but nothing is granted for P in bf16: P enters the product as its upper half and, rounded (2^-8), what
    that leaves (below 2^-7 of P) and 2^-20 of P. The output's half step is of the computed value."""
    o, mag, size = want
    got = got.cpu().double().view(x.S, x.Lq, x.H, x.hd)
    rel = 2 * (x.hd + 8) * U * size + (16 + (x.P + x.s) / 16 + 64) * U
    off = (rel + extra) * mag
    lim = off + 2.0**-8 * (o.abs() + off)
    bad = ~((got - o).abs() <= lim)
    assert not bad.any(), (bad.sum().item(), ((got - o).abs() / lim.clamp_min(1e-30)).max().item())


@gpu
@pytest.mark.parametrize("c", [
    (16, 9, 1, 8, 64, 32, 100, 40, 0), (32, 3, 2, 4, 128, 16, 70, 20, 0), (16, 3, 1, 8, 96, 16, 90, 12, 20),
    (33, 2, 1, 8, 40, 16, 20, 5, 0), (1, 4, 1, 4, 16, 16, 40, 6, 0),                # whole
    (1, 6, 1, 2, 64, 64, 9001, 700, 0), (2, 3, 1, 2, 24, 16, 0, 19, 0), (1, 40, 2, 1, 64, 64, 5000, 40, 700),
    (64, 20, 1, 16, 16, 64, 1100, 8, 0),                                            # split, tiles of 16 and 32 rows
], ids=str)
def test_bf16_probabilities_keep_sixteen_bits(c):
    """Values that cancel: a probability rounded to bf16 would be off by more than the small result's own rounding."""
    x = Case(*c, dt=BF16, share=c[0] == 64)
    if c[0] == 64:  # the oracle's time: a few sequences
        got = x.run()
        y = Case(*c, dt=BF16, share=True)
        for s in (0, 700, 1279):
            y.S = y.G = y.n = 1
            y.prefix_table, y.prefix_lens = x.prefix_table[s // 20: s // 20 + 1], x.prefix_lens[s // 20: s // 20 + 1]
            y.table, y.past, y.q = x.table[s: s + 1], x.past[s: s + 1], x.q[s: s + 1]
            tight(y, got[s: s + 1], y.oracle())
        return
    tight(x, x.run(), x.oracle())


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [(2, 5, 1, 2, 64, 64, 300, 21, 0), (16, 5, 1, 8, 64, 64, 300, 21, 0), (1, 20, 1, 2, 96, 32, 700, 9, 0)],
                         ids=str)
def test_a_visible_infinity_stays_one(c, dt):
    """Where a row sees an infinite value with a probability above zero its result is that infinity, and the rest of
    the row is as accurate as without it."""
    x = Case(*c, dt=dt, ragged=False)
    want = x.oracle()
    for j, d, v in ((3, 5, math.inf), (130, 6, -math.inf)):
        for gr in range(x.G):
            x.vp[x.prefix_table[gr, j // x.ps], 1, j % x.ps, d] = v
    got = x.run().view(x.S, x.Lq, x.H, x.hd)
    assert (got[:, :, 1, 5] == math.inf).all() and (got[:, :, 1, 6] == -math.inf).all()
    mask = torch.ones(got.shape, dtype=torch.bool)
    mask[:, :, 1, 5:7] = False
    o, mag, size = want
    got = torch.where(mask, got.cpu().double(), torch.zeros(()).double())
    tight(x, got, (o * mask, mag * mask, size), *(() if dt == BF16 else (0.0,)))


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [(1, 4, 1, 1, 64, 16, 120, 6, 0), (16, 4, 1, 8, 64, 32, 90, 7, 0), (1, 40, 1, 2, 96, 64, 900, 9, 0),
                               (2, 3, 2, 2, 32, 16, 0, 100, 0), (1, 6, 1, 2, 64, 64, 9001, 70, 0)], ids=str)
def test_scores_of_any_size(c, dt):
    """Scores up to 2^110 whose smallest distance is far above 1: the row is its largest key's value, bit for bit
    (one probability of 1, the others 0; in bf16 the parts of 1 are 1 and 2^-20, far below half a step)."""
    x = Case(*c, dt=dt, ragged=False)
    g = torch.Generator().manual_seed(1)
    for scale in (2.0**29, -(2.0**29), 2.0**33, 2.0**47, 2.0**101):
        for top in (191, 254):
            # key j is a_j in each dimension (integers, exact in bf16), the query `scale` in the first one and 0 elsewhere
            a = torch.randint(1, top - 1, x.kp.shape[:3], generator=g)
            x.kp = a[..., None].to(dt).expand(x.kp.shape).clone()
            x.q = torch.zeros_like(x.q).view(x.S, x.Lq, x.H, x.hd)
            x.q[..., 0] = scale
            x.q = x.q.view(x.S, x.Lq, -1)
            # one own row of every sequence outdoes all others
            for s in range(x.S):
                r = int(x.past[s]) // 2
                x.kp[x.table[s, r // x.ps], :, r % x.ps] = top if scale > 0 else 0
            got = x.run().view(x.S, x.Lq, x.H, x.hd).cpu()
            for s in range(x.S):
                r = int(x.past[s]) // 2
                want = x.vp[x.table[s, r // x.ps], :, r % x.ps].expand(x.Lq, -1, -1)
                assert torch.equal(got[s], want), (scale, top, s)


@gpu
def test_a_history_beyond_a_bound_of_zero_is_flagged():
    """prefix_cap = 0 (PagedKV.attend's default) with a history: nothing of it is seen, and that is said; histories of no
    rows are within the bound."""
    from eventstreamgpt_amd import kernels as K

    x = Case(2, 3, 1, 2, 32, 16, 64, 32)
    got = x.run(prefix_cap=0)
    with pytest.raises(IndexError, match="paged cache"):
        K.check_errors()
    empty = x.run(prefix_cap=0, prefix_lens=torch.zeros(2).int())
    assert torch.equal(got, empty)
    x.P = 0
    x.check(got)
    assert torch.equal(got, x.run())
    K.check_errors()


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [(2, 3, 2, 2, 32, 16, 64, 32, 20), (2, 3, 1, 2, 64, 16, 64, 37, 50), (16, 3, 1, 8, 96, 16, 90, 12, 20),
                               (1, 6, 3, 2, 64, 64, 9001, 700, 300), (3, 2, 1, 2, 16, 16, 0, 70, 33), (32, 3, 2, 4, 128, 16, 70, 20, 100),
                               (2, 3, 1, 2, 24, 16, 64, 37, 200)], ids=str)
def test_windows_of_a_past_beyond_its_bound(c, dt):
    """A length beyond its bound is flagged, and what lies there counts as not visible: a window still counts from the row
    itself and not from the bound. Pasts that leave some of the bounded rows in the window, and none."""
    from eventstreamgpt_amd import kernels as K

    x = Case(*c, dt=dt)
    clean = x.run()
    K.check_errors()
    far = [x.s, x.s + x.window // 2, x.s + x.window, x.s + x.window + x.P, 2**30, 2**31 - 1]
    for i, past in enumerate(far):
        x.past[i % x.S] = past
        want = x.oracle()
        got = x.run()
        x.check(got, want)
        with pytest.raises(IndexError, match="paged cache"):
            K.check_errors()
        if past >= x.s + x.window + x.P:
            assert (got[i % x.S] == 0).all()
        keep = torch.ones(x.S, dtype=torch.bool)  # the other groups; a group's walk begins where its rows' windows do
        keep[: (min(i, x.S - 1) // x.n + 1) * x.n] = False
        assert torch.equal(got[keep.to(DEV)], clean[keep.to(DEV)])


# ------------------------------------------------------------------- forms that the rule takes and no test above reaches
WHOLE = [  # G, n, Lq, H, hd, ps, P, s, window: one launch without a workspace, in both types
    (8, 32, 1, 16, 32, 64, 11560, 1685, 0),   # more blocks a wave, in the history and in an own segment, than page ids come at once
    (8, 32, 1, 16, 32, 64, 16000, 1685, 15000), (8, 32, 1, 16, 24, 16, 300, 1700, 0), (8, 32, 1, 16, 32, 64, 900, 1690, 1300),
    (32, 32, 2, 4, 128, 64, 256, 64, 0), (16, 64, 1, 8, 128, 64, 1000, 20, 0), (32, 64, 1, 4, 100, 64, 256, 20, 100),
]


def test_the_whole_form_is_what_those_cases_take():
    """No workspace with a history: the whole form. In f32 at 128 dimensions, and with more than 32 (f32), 16 (bf16) blocks
    a wave and segment, which is what one load of page ids reaches."""
    import os

    from eventstreamgpt_amd import _lib as L

    if not os.path.exists(L.LIB_PATH):
        pytest.skip("library not built")
    need = L.load(require_device=False).esgpt_attn_decode_shared_workspace
    for G, n, Lq, H, hd, ps, P, s, window in WHOLE:
        for dt in (L.F32, L.BF16):
            hd = -(-hd // 8) * 8 if dt == L.BF16 else hd
            assert need(G, G * n, Lq, H, hd, P, s, window, dt) == 0, (G, n, hd, P, s, dt)
    # keys of a block: 32 in f32, 64 in bf16; eight waves share a history, one takes an own segment; 64 page ids a load, one a
    # 16-key tile
    for kb, per in ((32, 32), (64, 16)):
        assert -(-11560 // (8 * kb)) > per and -(-1685 // kb) > per


def whole_case(c, dt, **kw):
    return Case(*(c if c[4] % 8 == 0 or dt == F32 else (*c[:4], -(-c[4] // 8) * 8, *c[5:])), dt=dt, share=True, **kw)


def check_some(x, got, c, dt, masked, want_of=lambda y: y.oracle(), seqs=None):
    """The oracle's answer for a few sequences of a case whose tables all name the same pages."""
    for s in seqs or sorted({0, 1, x.n, x.S // 2 + 3, x.S - 1}):
        y = whole_case(c, dt, masked=masked)
        y.kp, y.vp = x.kp, x.vp
        y.S = y.G = y.n = 1
        y.prefix_table, y.prefix_lens = x.prefix_table[s // x.n: s // x.n + 1], x.prefix_lens[s // x.n: s // x.n + 1]
        y.table, y.past, y.q = x.table[s: s + 1], x.past[s: s + 1], x.q[s: s + 1]
        y.row_mask = None if x.row_mask is None else x.row_mask[s: s + 1]
        y.check(got[s: s + 1], want_of(y))


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", WHOLE, ids=str)
def test_whole_form_over_long_segments_and_wide_heads(c, dt):
    masked = c[2] > 1
    x = whole_case(c, dt, masked=masked)
    got = x.run()
    check_some(x, got, c, dt, masked)
    if masked:
        assert (got[~x.row_mask.to(DEV)] == 0).all()
    assert int(err()[0]) == 0


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [WHOLE[4], WHOLE[6]], ids=str)
def test_whole_form_keeps_what_is_not_finite_to_the_rows_that_see_it(c, dt):
    """128 and 100 dimensions, padded rows: NaN beyond every length, an infinity at an own row that only some sequences are
    long enough to see."""
    masked = c[2] > 1
    x = whole_case(c, dt, masked=masked)
    P, t = int(x.prefix_lens.max()), x.s // 2
    clean = x.run()
    for pool in (x.kp, x.vp):
        # every table names the same pages: what no sequence reaches
        for tab, last in ((x.prefix_table[0], P), (x.table[0], int(x.past.max()) + x.Lq)):
            for i, page in enumerate(tab.tolist()):
                pool[page, :, min(max(last - i * x.ps, 0), x.ps):] = math.nan
    assert torch.equal(x.run(), clean)
    x.vp[x.table[0, t // x.ps], 1, t % x.ps, 9] = math.inf
    got = x.run().view(x.S, x.Lq, x.H, -1)
    at = torch.tensor([[x.own_row(s, i) for i in range(x.Lq)] for s in range(x.S)])
    active = torch.ones(x.S, x.Lq, dtype=torch.bool) if x.row_mask is None else x.row_mask
    sees = active & (at >= t) & ((at - t < x.window) if x.window else torch.ones_like(active))
    assert sees.any() and not sees.all()
    assert (got[..., 1, 9].cpu()[sees] == math.inf).all() and torch.isfinite(got[..., 1, 9].cpu()[~sees]).all()
    got[..., 1, 9] = torch.where(sees.to(DEV), clean.view(got.shape)[..., 1, 9], got[..., 1, 9])

    def want(y):
        vp = y.vp
        y.vp = vp.clone()
        y.vp[x.table[0, t // x.ps], 1, t % x.ps, 9] = clean_value
        out = y.oracle()
        y.vp = vp
        return out

    clean_value = float(whole_case(c, dt, masked=masked).vp[x.table[0, t // x.ps], 1, t % x.ps, 9])
    check_some(x, got.view(x.S, x.Lq, -1), c, dt, masked, want, [0, int((~sees).any(1).nonzero()[0]), x.S - 1])


@gpu
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_a_normalised_prompt_is_stored_as_it_is(dt):
    """A prompt that was normalised and rotated for its own attention is stored without weights and positions: the pools
    get the bits that an append with them leaves, and the queries are the prompt's own."""
    from eventstreamgpt_amd import kernels as K

    B, L, H, hd, ps = 3, 45, 4, 64, 16
    D = H * hd
    g = torch.Generator().manual_seed(7)
    rows = torch.randn(B, L, 3 * D, generator=g).to(dt).to(DEV)
    times = torch.exp(3 + torch.randn(B, L, generator=g)).cumsum(1).to(DEV)
    mask = (torch.arange(L)[None] >= torch.tensor([0, 17, 44])[:, None]).to(DEV)
    w = [(hd**-0.25 * (1 + 0.2 * torch.randn(hd, generator=g))).to(DEV) for _ in range(2)]
    f = torch.exp(torch.arange(0, hd, 2) * (-math.log(10000.0) / hd)).float().to(DEV)
    a, b = (K.PagedKV(9, ps, H, hd, dt, DEV) for _ in range(2))
    table, zero = a.pages(9).view(3, 3), torch.zeros(B, dtype=torch.int32, device=DEV)
    for pool in (a.k, a.v, b.k, b.v):
        pool.zero_()
    y = K.qk_norm_rope(rows, *w, times, f, H)
    q = a.append(rows, table, zero, mask, *w, times, f)
    q2 = b.append(y, table, zero, mask)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(q, q2)
    assert torch.equal(q, torch.where(mask[..., None], y[..., :D], torch.zeros_like(q)))
    assert K.attention(y, mask, None, H, 0, False).shape == (B, L, D)
    K.check_errors()


@gpu
@pytest.mark.parametrize("c", [(2, 5, 1, 3, 4, 16, 70, 21, 0), (2, 3, 2, 2, 12, 16, 130, 20, 30), (16, 9, 1, 8, 20, 32, 100, 40, 0),
                               (1, 6, 1, 2, 68, 64, 3000, 300, 0), (32, 3, 2, 4, 124, 16, 70, 20, 0)], ids=str)
def test_f32_heads_that_are_multiples_of_four(c):
    x = Case(*c, dt=F32)
    x.check(x.run())
    assert int(err()[0]) == 0
