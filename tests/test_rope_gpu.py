"""Query / key norm with the position rotation (``esgpt::qk_norm_rope``, its backward) and the paged cache's append
(``esgpt::kv_append_paged``) against a plain implementation in 64 bits.

Tolerances, from u = 2^-24 (an f32 rounding). A head's mean square is a chain of at most 2V + log2(lanes) + 2 <= 24
roundings, halved by the root, and the root's own 2: 14 u on r. x r w adds 2, and each of the two products of the
rotation 2 plus the angle's 4 (a turn rounded to f32 is off by 2^-26 turns = 1.6 u radians, sincospi by 2 ulp):
below 32 u of the rotated pair's length. The backward adds the two sums over the head and three products: below 96 u
of the largest term. bf16 outputs add half a step, 2^-8 of the value.
"""
import math

import pytest
import torch

U = 2.0**-24
HALF = {torch.float32: U, torch.bfloat16: 2.0**-8}
EPS = 1e-6
gpu = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------------------------------------- 64-bit oracle
def rotate(z, pos, inv_freq):
    """z [B, T, h, hd] by pos [B, T]: (z_i, z_{i + R/2}) turned by pos * inv_freq_i."""
    R2 = inv_freq.numel()
    a = (pos.double()[..., None] * inv_freq.double())[:, :, None]
    lo, hi = z[..., :R2], z[..., R2: 2 * R2]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), z[..., 2 * R2:]], -1)


def oracle(qkv, q_w, k_w, pos, inv_freq, H, eps=EPS):
    """[B, T, 3D] in 64 bits; differentiable in qkv, q_w, k_w."""
    B, T, D3 = qkv.shape
    q, k, v = qkv.double().view(B, T, 3, H, D3 // 3 // H).unbind(2)
    out = []
    for x, w in ((q, q_w), (k, k_w)):
        if w is not None:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
        out.append(x if pos is None else rotate(x, pos, inv_freq))
    return torch.stack([*out, v], 2).reshape(B, T, D3)


def freqs(R, dev="cpu"):
    return torch.exp(torch.arange(0, R, 2, device=dev) * (-math.log(10000.0) / max(R, 1))).float()


def inputs(B, T, H, hd, R, dt, pos="time", norm=True, seed=0, dev=DEV):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, T, 3 * H * hd, generator=g).to(dt)
    w = [1 + 0.3 * torch.randn(hd, generator=g) for _ in range(2)] if norm else [None, None]
    times = torch.exp(3 + torch.randn(B, T, generator=g)).cumsum(1)
    p = None if R == 0 else times if pos == "time" else torch.arange(T).repeat(B, 1) + 1000 * torch.arange(B)[:, None]
    f = None if R == 0 else freqs(R)
    return [None if t is None else t.to(dev) for t in (qkv, *w, p, f)]


def ops():
    from eventstreamgpt_amd import ops as O

    return O.load()


def close(got, want, dt, scale, k=32):
    """|got - want| <= half a step of dt + k u of the largest term ``scale``."""
    err = (got.double() - want).abs()
    lim = HALF[dt] * want.abs() + k * U * scale
    bad = err > lim
    assert not bad.any(), (err.max().item(), (err / lim).max().item())


SHAPES = [
    # B, T, H, hd, R: one token; the smallest head; odd head sizes and rotations (chunks of 8, 4, 2 and 1 elements);
    # more lanes than a workgroup for one token; a run that ends inside a workgroup
    (1, 1, 4, 64, 64), (4, 16, 4, 16, 16), (2, 33, 1, 8, 8), (3, 7, 5, 24, 8), (2, 9, 3, 24, 12), (2, 5, 2, 40, 6),
    (1, 3, 2, 128, 2), (2, 70, 8, 64, 32), (1, 17, 12, 96, 96), (1, 5, 9, 128, 2), (1, 4, 40, 128, 128),
    (33, 129, 4, 64, 64), (2, 31, 4, 64, 0),
    # three and eight passes of a workgroup over one token's lanes, whose dw sums share memory with the next pass's weights
    (3, 41, 80, 128, 64), (1, 700, 128, 128, 128),
]


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
def test_forward_and_backward(shape, dt, norm):
    B, T, H, hd, R = shape
    if not norm and R == 0:
        pytest.skip("neither a norm nor a rotation: a copy")
    qkv, q_w, k_w, pos, f = inputs(B, T, H, hd, R, dt, "index" if T == 70 else "time", norm)
    got = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    x = qkv.double().requires_grad_()
    w = [None if t is None else t.double().requires_grad_() for t in (q_w, k_w)]
    want = oracle(x, *w, pos, f, H)
    assert got.shape == qkv.shape and got.dtype == dt
    close(got, want.detach(), dt, want.abs().max().item() * math.sqrt(2))
    assert torch.equal(got[..., 2 * H * hd:], qkv[..., 2 * H * hd:])  # v bit for bit

    dout = torch.randn(qkv.shape, generator=torch.Generator().manual_seed(1)).to(dt).to(DEV)
    leaves = [x] + ([*w] if norm else [])
    grads = torch.autograd.grad(want, leaves, dout.double())
    dqkv, dw = ops().qk_norm_rope_bwd(dout, qkv, q_w, k_w, pos, f, H, EPS)
    # dx = r (g - x r^2 mean(g x)): each term at most r |g| sqrt(hd) in size
    r = 1.0
    if norm:
        xs = qkv[..., : 2 * H * hd].double().view(B, T, 2 * H, hd)
        r = torch.rsqrt(xs.pow(2).mean(-1) + EPS).max().item() * max(t.abs().max().item() for t in (q_w, k_w))
    close(dqkv, grads[0], dt, 2 * r * dout.double().abs().max().item() * math.sqrt(2), 96)
    assert torch.equal(dqkv[..., 2 * H * hd:], dout[..., 2 * H * hd:])
    if norm:
        # a sum of B T H terms u * x r: each off by 24 u, and a chain of at most B T H + 64 additions
        u = torch.ones_like(qkv[..., : 2 * H * hd].double())
        xh = qkv[..., : 2 * H * hd].double().view(B, T, 2, H, hd)
        xh = (xh * torch.rsqrt(xh.pow(2).mean(-1, keepdim=True) + EPS)).abs()
        mag = (xh * math.sqrt(2) * dout.double().abs().max()).sum((0, 1, 3))
        for i in range(2):
            lim = (24 + 64 + min(B * T * H, 512)) * U * mag[i]
            assert ((dw[i].double() - grads[1 + i]).abs() <= lim).all()
    else:
        assert dw.shape == (0, hd)


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_autograd_is_the_backward_operator(dt):
    B, T, H, hd, R = 3, 21, 4, 32, 16
    qkv, q_w, k_w, pos, f = inputs(B, T, H, hd, R, dt)
    for t in (qkv, q_w, k_w):
        t.requires_grad_()
    out = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    dout = torch.randn_like(out)
    out.backward(dout)
    with torch.no_grad():
        dqkv, dw = ops().qk_norm_rope_bwd(dout, qkv, q_w, k_w, pos, f, H, EPS)
    assert torch.equal(qkv.grad, dqkv) and torch.equal(q_w.grad, dw[0]) and torch.equal(k_w.grad, dw[1])
    # a gradient that broadcasts (stride 0) and one leaf only
    q2 = qkv.detach().clone().requires_grad_()
    ops().qk_norm_rope(q2, q_w.detach(), k_w.detach(), pos, f, H, EPS).sum().backward()
    with torch.no_grad():
        want, _ = ops().qk_norm_rope_bwd(torch.ones_like(qkv), qkv, q_w, k_w, pos, f, H, EPS)
    assert torch.equal(q2.grad, want)


@gpu
def test_gradient_against_differences():
    """The operator's gradient along random directions against central differences of the 64-bit forward: those are
    off by the third derivative times h^2 / 6 (about 1e-10) and 1e-16 / h, the operator by 96 u of its largest term."""
    B, T, H, hd, R = 2, 5, 3, 24, 12
    qkv, q_w, k_w, pos, f = inputs(B, T, H, hd, R, torch.float32, seed=4)
    dout = torch.randn_like(qkv)
    dqkv, dw = ops().qk_norm_rope_bwd(dout, qkv, q_w, k_w, pos, f, H, EPS)
    g = torch.Generator().manual_seed(9)
    h = 1e-5
    for _ in range(4):
        v = [torch.randn(t.shape, generator=g, dtype=torch.float64).to(DEV) for t in (qkv, q_w, k_w)]
        at = [(oracle(qkv.double() + s * v[0], q_w.double() + s * v[1], k_w.double() + s * v[2], pos, f, H)
               * dout.double()).sum() for s in (h, -h)]
        want = (at[0] - at[1]) / (2 * h)
        terms = [dqkv.double() * v[0], dw[0].double() * v[1], dw[1].double() * v[2]]
        got = sum(t.sum() for t in terms)
        lim = 96 * U * 8 * sum(t.abs().sum() for t in terms) + 1e-6
        assert (got - want).abs() <= lim, (got.item(), want.item(), lim.item())


@gpu
def test_far_positions_keep_their_angle():
    """Index positions up to 2^28 and times of a million minutes: an angle formed in f32 would be off by radians."""
    B, T, H, hd, R = 1, 64, 2, 32, 32
    qkv, _, _, _, f = inputs(B, T, H, hd, R, torch.float32, norm=False)
    for pos in (torch.arange(T, device=DEV)[None] * 4194301 + 17, 1e6 + 0.25 * torch.arange(T, device=DEV)[None].float()):
        got = ops().qk_norm_rope(qkv, None, None, pos, f, H, EPS)
        want = oracle(qkv, None, None, pos, f, H)
        close(got, want, torch.float32, want.abs().max().item() * math.sqrt(2))


@gpu
def test_special_rows():
    """A row of zeros has a zero norm (gradient 1 / sqrt(eps) of dout, no NaN); an infinity or NaN stays in its head."""
    B, T, H, hd, R = 1, 4, 2, 64, 64
    qkv, q_w, k_w, pos, f = inputs(B, T, H, hd, R, torch.bfloat16)
    clean = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    qkv[0, 0] = 0
    qkv[0, 1, 3] = math.inf
    qkv[0, 2, hd + 3] = math.nan
    out = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    assert (out[0, 0] == 0).all()
    assert torch.equal(out[0, 1, hd:], clean[0, 1, hd:]) and not torch.isfinite(out[0, 1, :hd]).all()
    assert torch.equal(out[0, 2, :hd], clean[0, 2, :hd]) and out[0, 2, hd: 2 * hd].isnan().all()
    assert torch.equal(out[0, 2, 2 * hd:], clean[0, 2, 2 * hd:]) and torch.equal(out[0, 3], clean[0, 3])
    dqkv, dw = ops().qk_norm_rope_bwd(torch.ones_like(qkv[:, :1]), qkv[:, :1], q_w, k_w, pos[:, :1], f, H, EPS)
    assert torch.isfinite(dqkv).all() and (dw == 0).all()


@gpu
def test_layouts_streams_and_repeats():
    """A strided view, a view at an odd offset and another stream give the contiguous call's bits; a repeat too."""
    B, T, H, hd, R = 5, 19, 4, 16, 16
    qkv, q_w, k_w, pos, f = inputs(B, T, H, hd, R, torch.bfloat16)
    want = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    dout = torch.randn_like(qkv)
    wd, ww = ops().qk_norm_rope_bwd(dout, qkv, q_w, k_w, pos, f, H, EPS)
    big = torch.zeros(B, T, 3 * H * hd + 24, dtype=qkv.dtype, device=DEV)
    big[..., 8:-16] = qkv
    odd = torch.zeros(qkv.numel() + 1, dtype=qkv.dtype, device=DEV)
    odd[1:] = qkv.reshape(-1)
    tp = pos.t().contiguous().t()
    for x in (big[..., 8:-16], odd[1:].view(qkv.shape)):
        assert torch.equal(ops().qk_norm_rope(x, q_w, k_w, tp, f, H, EPS), want)
        d, w = ops().qk_norm_rope_bwd(dout.transpose(0, 1).contiguous().transpose(0, 1), x, q_w, k_w, tp, f, H, EPS)
        assert torch.equal(d, wd) and torch.equal(w, ww)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    st.synchronize()
    assert torch.equal(other, want)


@gpu
def test_captured_and_replayed():
    """One graph with the forward and the backward, replayed on changed inputs with eager calls in between."""
    B, T, H, hd, R = 4, 40, 4, 64, 64
    qkv, q_w, k_w, pos, f = inputs(B, T, H, hd, R, torch.bfloat16)
    dout = torch.randn_like(qkv)

    def step():
        return (ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS),
                *ops().qk_norm_rope_bwd(dout, qkv, q_w, k_w, pos, f, H, EPS))

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        qkv.copy_(torch.randn_like(qkv))
        pos.add_(100.0 * i)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


@gpu
def test_captured_backward_through_autograd():
    """A graph with a layer's forward and backward through autograd. Captured while an eager graph of the same leaves lives
    on the default stream it is refused, before anything is launched; without one every replay gives the eager bits."""
    B, T, H, hd, R = 4, 40, 4, 64, 64
    qkv, q_w, k_w, pos, f = inputs(B, T, H, hd, R, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (qkv, q_w, k_w)]
    dout = torch.randn(qkv.shape, device=DEV, dtype=qkv.dtype)

    def step():
        out = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    eager = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    eager.backward(dout)  # the graph that was there is none the worse
    del eager
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            qkv.copy_(torch.randn_like(qkv))
            q_w.add_(0.1)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


@gpu
def test_empty_batches():
    qkv, q_w, k_w, pos, f = inputs(2, 3, 2, 16, 16, torch.float32)
    for B, T in ((0, 3), (2, 0)):
        e = qkv[:B, :T]
        assert ops().qk_norm_rope(e, q_w, k_w, pos[:B, :T], f, 2, EPS).shape == e.shape
        d, w = ops().qk_norm_rope_bwd(e, e, q_w, k_w, pos[:B, :T], f, 2, EPS)
        assert d.shape == e.shape and w.shape == (2, 16) and (w == 0).all()


@gpu
def test_refusals():
    qkv, q_w, k_w, pos, f = inputs(2, 3, 2, 16, 16, torch.float32)
    o = ops()
    bad = [
        ((qkv, q_w, None, pos, f, 2, EPS), "together"),
        ((qkv, q_w, k_w, pos, None, 2, EPS), "together"),
        ((qkv, q_w[:8], k_w, pos, f, 2, EPS), "norm weights"),
        ((qkv, q_w.double(), k_w, pos, f, 2, EPS), "norm weights"),
        ((qkv, q_w.cpu(), k_w, pos, f, 2, EPS), "norm weights"),
        ((qkv, q_w, k_w, pos.double(), f, 2, EPS), "pos must be"),
        ((qkv, q_w, k_w, pos[:1], f, 2, EPS), "pos must be"),
        ((qkv, q_w, k_w, pos, torch.ones(9, device=DEV), 2, EPS), "inv_freq"),
        ((qkv, q_w, k_w, pos, f, 5, EPS), "H = 5"),
        ((qkv, q_w, k_w, pos, f, 0, EPS), "H = 0"),
        ((qkv[0], q_w, k_w, pos, f, 2, EPS), "qkv must be"),
        ((qkv.half(), q_w, k_w, pos, f, 2, EPS), "dtype"),
        ((qkv, q_w, k_w, pos, f, 2, -1.0), "invalid argument"),
    ]
    for args, text in bad:
        with pytest.raises(RuntimeError, match=text):
            o.qk_norm_rope(*args)
    with pytest.raises(RuntimeError, match="invalid argument"):  # head size 136
        o.qk_norm_rope(torch.zeros(1, 1, 408, device=DEV), None, None, pos[:1, :1], f, 1, EPS)
    with pytest.raises(RuntimeError, match="invalid argument"):  # head size 12 in bf16
        o.qk_norm_rope(torch.zeros(1, 1, 36, device=DEV, dtype=torch.bfloat16), None, None, pos[:1, :1], f[:4], 1, EPS)
    with pytest.raises(RuntimeError, match="dout"):
        o.qk_norm_rope_bwd(qkv[:1], qkv, q_w, k_w, pos, f, 2, EPS)
    with pytest.raises(NotImplementedError, match="no gradient"):
        o.qk_norm_rope(qkv.requires_grad_(), q_w, k_w, pos.requires_grad_(), f, 2, EPS)


# ---------------------------------------------------------------------------------------------- the paged append
def cache(n_pages, H, ps, hd, dt, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n_pages, H, ps, hd, generator=g).to(dt).to(DEV) for _ in range(2)]


def err():
    from eventstreamgpt_amd import kernels as K

    return K.err_word(torch.device(DEV, torch.cuda.current_device()))


@pytest.fixture(autouse=True)
def _clear(request):
    if request.node.get_closest_marker("gpu"):
        err().zero_()
    yield
    if request.node.get_closest_marker("gpu"):
        err().zero_()


def append_oracle(y, kp, vp, table, past, mask, H):
    """The stored rows one by one: (q, k_pages, v_pages); y = the normalised, rotated packed rows."""
    S, Lq, D3 = y.shape
    hd, ps = D3 // 3 // H, kp.shape[2]
    kp, vp = kp.clone(), vp.clone()
    q, k, v = y.view(S, Lq, 3, H, hd).unbind(2)
    q = q.clone()
    for s in range(S):
        at = int(past[s])
        for i in range(Lq):
            if mask is not None and not bool(mask[s, i]):
                q[s, i] = 0
                continue
            page = int(table[s, at // ps]) if 0 <= at < table.shape[1] * ps else -1
            if 0 <= page < kp.shape[0]:
                kp[page, :, at % ps], vp[page, :, at % ps] = k[s, i], v[s, i]
            at += 1
    return q.reshape(S, Lq, -1), kp, vp


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("S,Lq,H,hd,R,ps,masked", [
    (1, 1, 1, 8, 8, 16, False), (5, 1, 4, 64, 64, 64, False), (3, 40, 4, 16, 16, 16, True), (4, 77, 2, 24, 12, 32, True),
    (2, 300, 4, 64, 64, 128, True), (3, 5, 9, 128, 2, 16, True), (6, 3, 2, 32, 0, 16, False),
    (3, 21, 80, 128, 64, 16, True),
], ids=str)
def test_append(S, Lq, H, hd, R, ps, masked, dt):
    """Ragged pasts, left, right and scattered padding, pages in any order; every other row of the pools as it was."""
    qkv, q_w, k_w, pos, f = inputs(S, Lq, H, hd, R, dt, norm=R != 0)
    g = torch.Generator().manual_seed(5)
    past = torch.randint(0, 3 * ps, (S,), generator=g).int()
    W = -(-(3 * ps + Lq) // ps)
    table = torch.randperm(S * W + 4, generator=g)[: S * W].view(S, W).int()
    mask = None
    if masked:
        mask = torch.rand(S, Lq, generator=g) < 0.6
        mask[0] = False                                    # nothing to store
        mask[-1] = torch.arange(Lq) >= Lq // 3             # left padding
    kp, vp = cache(S * W + 4, H, ps, hd, dt)
    y = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS) if R else qkv
    wq, wk, wv = append_oracle(y, kp, vp, table, past, mask, H)
    q = ops().kv_append_paged(qkv, kp, vp, table.to(DEV), past.to(DEV), None if mask is None else mask.to(DEV), q_w, k_w,
                              pos, f, EPS, err())
    assert torch.equal(q, wq) and torch.equal(kp, wk) and torch.equal(vp, wv)  # the forward's own bits
    assert int(err()[0]) == 0


@gpu
def test_append_flags_what_has_no_place():
    """A page outside the pool, a row beyond the table and a negative past: flagged, nothing stored out of place, the
    other sequences and the queries as ever."""
    from eventstreamgpt_amd import kernels as K

    S, Lq, H, hd, ps = 6, 3, 2, 16, 16
    qkv, q_w, k_w, pos, f = inputs(S, Lq, H, hd, 16, torch.float32)
    past = torch.tensor([0, 31, -1, 5, 2**31 - 1, 0], dtype=torch.int32)
    table = torch.arange(12).view(S, 2).int()
    table[3, 0], table[5, 0] = 12, -1
    kp, vp = cache(12, H, ps, hd, torch.float32)
    y = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    rows = append_oracle(y, kp, vp, table, torch.where(past < 0, torch.tensor(2**30), past), None, H)
    q = ops().kv_append_paged(qkv, kp, vp, table.to(DEV), past.to(DEV), None, q_w, k_w, pos, f, EPS, err())
    assert all(torch.equal(a, b) for a, b in zip((q, kp, vp), rows))
    with pytest.raises(IndexError, match="paged cache"):
        K.check_errors()
    K.check_errors()
    # no pages at all, and no table
    q0 = ops().kv_append_paged(qkv, kp[:0], vp[:0], table.to(DEV)[:, :0].contiguous(), past.to(DEV), None, q_w, k_w, pos, f,
                               EPS, err())
    assert torch.equal(q0, q)
    with pytest.raises(IndexError):
        K.check_errors()


@gpu
def test_append_refusals():
    S, Lq, H, hd, ps = 2, 3, 2, 16, 16
    qkv, q_w, k_w, pos, f = inputs(S, Lq, H, hd, 16, torch.float32)
    kp, vp = cache(4, H, ps, hd, torch.float32)
    table, past = torch.arange(4, device=DEV).view(2, 2).int(), torch.zeros(2, device=DEV).int()
    ok = dict(qkv=qkv, k_pages=kp, v_pages=vp, page_table=table, past=past, row_mask=None, q_w=q_w, k_w=k_w, pos=pos,
              inv_freq=f, eps=EPS, err=err())
    odd = torch.zeros(kp.numel() + 1, device=DEV)[1:].view(kp.shape)
    for change, text in [
        ({"v_pages": vp[:2]}, "k_pages and v_pages"), ({"k_pages": kp.bfloat16()}, "pages must be"),
        ({"k_pages": kp.transpose(2, 3).contiguous().transpose(2, 3)}, "pages must be"), ({"k_pages": odd}, "pages must be"),
        ({"k_pages": kp[:, :, :8].contiguous(), "v_pages": vp[:, :, :8].contiguous()}, "page size"),
        ({"k_pages": torch.zeros(1, H, 48, hd, device=DEV), "v_pages": torch.zeros(1, H, 48, hd, device=DEV)}, "page size"),
        ({"k_pages": kp[..., :8].contiguous(), "v_pages": vp[..., :8].contiguous()}, "heads of 8"),
        ({"page_table": table.long()}, "page_table"), ({"page_table": table[:1]}, "page_table"),
        ({"page_table": table.flatten()}, "page_table"), ({"past": past.cpu()}, "past"), ({"past": past[:1]}, "past"),
        ({"row_mask": torch.ones(2, 2, device=DEV).bool()}, "row_mask"), ({"row_mask": torch.ones(2, 3, device=DEV)}, "row_mask"),
        ({"err": torch.zeros(2, dtype=torch.int64)}, "error block"), ({"k_w": None}, "together"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            ops().kv_append_paged(**{**ok, **change})
    want = [t.clone() for t in (ops().kv_append_paged(**ok), kp, vp)]
    wide = torch.full((2, 5), -1, device=DEV).int()  # a slice of a wider table
    wide[:, 1:3] = table
    got = ops().kv_append_paged(**{**ok, "page_table": wide[:, 1:3], "past": wide[:, 0] + 1})
    assert all(torch.equal(a, b) for a, b in zip((got, kp, vp), want)) and int(err()[0]) == 0


# ------------------------------------------------------------------------------------------- without a device
def _lib():
    import os

    from eventstreamgpt_amd import _lib as L

    if not os.path.exists(L.LIB_PATH):
        pytest.skip("library not built")
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: only where no device could read them")
    return L.load(require_device=False)


def test_c_abi_refuses_before_it_launches():
    """Every refusal is an error code from the host checks (no device is touched)."""
    lib = _lib()
    P = 4096  # an aligned address that is never read

    def fwd(x=P, qw=P, kw=P, pos=P, pd=0, f=P, R=64, N=4, H=4, hd=64, eps=1e-6, out=P, dt=1):
        return lib.esgpt_qk_norm_rope_fwd(x, qw, kw, pos, pd, f, R, N, H, hd, eps, out, dt, None)

    for bad in (dict(x=None), dict(x=P + 2), dict(out=None), dict(out=P + 8), dict(kw=None), dict(pos=None), dict(f=None),
                dict(pd=2), dict(R=63), dict(R=66), dict(R=-2), dict(N=-1), dict(H=0), dict(hd=12), dict(hd=136), dict(hd=0),
                dict(H=257), dict(eps=-1.0), dict(eps=float("nan")), dict(dt=2)):
        assert fwd(**bad) == 1, bad
    assert fwd(N=0) == 0 and fwd(N=0, x=None, out=None) == 0

    def bwd(do=P, x=P, dx=P, dw=P, ws=P, nb=1 << 20, N=4):
        return lib.esgpt_qk_norm_rope_bwd(do, x, P, P, P, 0, P, 64, N, 4, 64, 1e-6, dx, dw, ws, nb, 1, None)

    for bad in (dict(do=None), dict(x=None), dict(dx=None), dict(dw=None), dict(dw=P + 4), dict(ws=None), dict(nb=16)):
        assert bwd(**bad) == 1, bad
    assert lib.esgpt_qk_norm_rope_bwd_workspace(0, 4, 64, 64, 1) == 0
    assert lib.esgpt_qk_norm_rope_bwd_workspace(8192, 4, 64, 64, 1) >= 2 * 64 * 4

    def app(past=P, tab=P, W=2, kp=P, n_pages=4, ps=64, q=P, S=2, Lq=1, mask=None):
        return lib.esgpt_kv_append_paged(P, P, P, P, 0, P, 64, 1e-6, mask, past, tab, W, kp, P, n_pages, ps, q, S, Lq, 4,
                                         64, 1, None, None)

    for bad in (dict(past=None), dict(tab=None), dict(W=-1), dict(kp=None), dict(kp=P + 4), dict(n_pages=-1), dict(ps=8),
                dict(ps=48), dict(ps=131072), dict(q=None), dict(S=-1), dict(Lq=-1), dict(S=1, Lq=(1 << 24) + 1),
                dict(S=1 << 20, Lq=1 << 11), dict(W=1 << 31)):
        assert app(**bad) == 1, bad
    assert app(S=0) == 0 and app(Lq=0) == 0


def test_cpu_tensors_raise():
    o = ops()
    qkv, q_w, k_w, pos, f = inputs(2, 3, 2, 16, 16, torch.float32, dev="cpu")
    with pytest.raises(NotImplementedError):
        o.qk_norm_rope(qkv, q_w, k_w, pos, f, 2, EPS)


def test_fake_tensors_and_autograd_formula():
    """Shapes and types without a device, through the registered autograd formula."""
    o = ops()
    qkv, q_w, k_w, pos, f = inputs(2, 3, 2, 16, 16, torch.bfloat16, dev="meta")
    for t in (qkv, q_w, k_w):
        t.requires_grad_()
    out = o.qk_norm_rope(qkv, q_w, k_w, pos, f, 2, EPS)
    assert out.shape == qkv.shape and out.dtype == qkv.dtype
    out.sum().backward()
    assert qkv.grad.dtype == torch.bfloat16 and q_w.grad.shape == (16,) and k_w.grad.dtype == torch.float32
    kp = torch.empty(4, 2, 16, 16, device="meta", dtype=torch.bfloat16)
    q = o.kv_append_paged(qkv.detach(), kp, kp.clone(), torch.empty(2, 2, device="meta", dtype=torch.int32),
                          torch.empty(2, device="meta", dtype=torch.int32), None, None, None, None, None, EPS,
                          torch.empty(2, device="meta", dtype=torch.int64))
    assert q.shape == (2, 3, 32) and q.dtype == torch.bfloat16
    args = (kp, kp.clone(), torch.empty(2, 2, device="meta", dtype=torch.int32),
            torch.empty(2, device="meta", dtype=torch.int32), None, q_w, k_w, pos, f, EPS,
            torch.empty(2, device="meta", dtype=torch.int64))
    with pytest.raises(NotImplementedError, match="no_grad"):  # the weights ask for a gradient
        o.kv_append_paged(qkv.detach(), *args)
    with torch.no_grad():
        assert o.kv_append_paged(qkv, *args).shape == q.shape


def test_error_flag_raises_index_error():
    from eventstreamgpt_amd import _lib as L
    from eventstreamgpt_amd.kernels import raise_for_error

    with pytest.raises(IndexError, match="paged cache"):
        raise_for_error(L.FLAG_BAD_PAGE, 0)


def test_second_derivatives_are_refused():
    """A recorded backward gives its gradients; a derivative of those raises, and so does one through the backward
    operator itself. An unrecorded call of it is not in any graph."""
    o = ops()
    qkv, q_w, k_w, pos, f = inputs(2, 3, 2, 16, 16, torch.float32, dev="meta")
    leaves = [t.requires_grad_() for t in (qkv, q_w, k_w)]
    for leaf in leaves:
        out = o.qk_norm_rope(qkv, q_w, k_w, pos, f, 2, EPS)
        grads = torch.autograd.grad(out.square().sum(), leaves, create_graph=True)
        assert [g.shape for g in grads] == [t.shape for t in leaves]
        with pytest.raises(NotImplementedError, match="second derivative"):
            torch.autograd.grad(sum(g.sum() for g in grads), leaf)
    dout = torch.empty_like(qkv).requires_grad_()
    for kw in (dict(dout=dout), dict(dout=dout.detach())):
        dqkv, dw = o.qk_norm_rope_bwd(kw["dout"], qkv, q_w, k_w, pos, f, 2, EPS)
        with pytest.raises(NotImplementedError, match="second derivative"):
            (dqkv.sum() + dw.sum()).backward()
    with torch.no_grad():
        dqkv, dw = o.qk_norm_rope_bwd(dout, qkv, q_w, k_w, pos, f, 2, EPS)
    assert not dqkv.requires_grad and not dw.requires_grad and dw.shape == (2, 16)
    dqkv, dw = o.qk_norm_rope_bwd(*(t.detach() for t in (dout, qkv)), None, None, pos, f, 2, EPS)
    assert not dqkv.requires_grad and dw.shape == (0, 16)


@pytest.mark.parametrize("which", ["qkv", "k_pages", "v_pages", "q_w", "inv_freq", "q", "ak_pages", "av_pages"])
def test_forward_mode_tangents_are_refused(which):
    """A tangent on any input of the paged operators, which have no derivative, raises instead of being dropped, without
    gradients enabled too; a tangent that forward mode itself ignores does not."""
    import torch.autograd.forward_ad as fw

    o = ops()
    m, i = dict(device="meta"), dict(device="meta", dtype=torch.int32)
    t = dict(qkv=torch.empty(2, 3, 96, **m), k_pages=torch.empty(4, 2, 16, 16, **m), v_pages=torch.empty(4, 2, 16, 16, **m),
             q_w=torch.empty(16, **m), inv_freq=torch.empty(8, **m), q=torch.empty(2, 3, 32, **m))
    t.update(ak_pages=t["k_pages"], av_pages=t["v_pages"])
    table, past, e = torch.empty(2, 2, **i), torch.empty(2, **i), torch.empty(2, device="meta", dtype=torch.int64)

    def call(t):
        if which in ("q", "ak_pages", "av_pages"):
            return o.attn_decode_shared(t["q"], t["ak_pages"], t["av_pages"], None, None, table, past, None, 0, 16, 0, e)
        return o.kv_append_paged(t["qkv"], t["k_pages"], t["v_pages"], table, past, None, t["q_w"], torch.empty(16, **m),
                                 torch.empty(2, 3, **m), t["inv_freq"], EPS, e)

    assert call(t).shape == (2, 3, 32)
    with fw.dual_level():
        dual = {**t, which: fw.make_dual(t[which], torch.empty_like(t[which]))}
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="no gradient"):
                call(dual)
        with fw._set_fwd_grad_enabled(False):
            assert call(dual).shape == (2, 3, 32)
        with pytest.raises(RuntimeError, match="jvp"):
            o.qk_norm_rope_bwd(t["qkv"], t["qkv"], fw.make_dual(t["q_w"], torch.empty_like(t["q_w"])), t["q_w"], None, None, 2,
                               EPS)


def test_an_append_counts_as_a_write_to_the_pools():
    """Both pools' versions grow with each append, in inference mode too, so that a graph which saved a pool refuses to run
    backward after it; inference tensors, which have no version, are taken as ever."""
    o = ops()
    i = dict(device="meta", dtype=torch.int32)
    kp, vp = (torch.empty(4, 2, 16, 16, device="meta") for _ in range(2))

    def append(kp, vp):
        return o.kv_append_paged(torch.empty(2, 3, 96, device="meta"), kp, vp, torch.empty(2, 2, **i), torch.empty(2, **i),
                                 None, None, None, None, None, EPS, torch.empty(2, device="meta", dtype=torch.int64))

    w = torch.empty(4, 2, 16, 16, device="meta", requires_grad=True)
    for n, mode in enumerate((torch.enable_grad, torch.no_grad, torch.inference_mode)):
        loss = [(w * pool).sum() for pool in (kp, vp)]
        with mode():
            assert append(kp, vp).shape == (2, 3, 32)
        assert kp._version == vp._version == n + 1
        for at in loss:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                at.backward()
    with torch.inference_mode():
        ki, vi = kp.clone(), vp.clone()
        append(ki, vi)
    append(ki, vi)


def test_frequencies_that_are_parameters():
    """pos and inv_freq that require a gradient are refused where one is recorded, and only there."""
    o = ops()
    qkv, q_w, k_w, pos, f = inputs(2, 3, 2, 16, 16, torch.float32, dev="meta")
    for kw in (dict(inv_freq=torch.nn.Parameter(f), pos=pos), dict(inv_freq=f, pos=pos.clone().requires_grad_())):
        with pytest.raises(NotImplementedError, match="no gradient for pos and inv_freq"):
            o.qk_norm_rope(qkv, q_w, k_w, H=2, eps=EPS, **kw)
        for mode in (torch.no_grad, torch.inference_mode):
            with mode():
                assert not o.qk_norm_rope(qkv, q_w, k_w, H=2, eps=EPS, **kw).requires_grad


@gpu
def test_unsupported_head_sizes_are_named():
    """The refusal says which head size is not supported and what the rule is, at every entry point."""
    i = dict(device=DEV, dtype=torch.int32)
    for dt, H, hd, step in ((torch.float32, 2, 136, 4), (torch.bfloat16, 2, 12, 8), (torch.float32, 1, 6, 4),
                            (torch.bfloat16, 129, 128, 8)):
        qkv, rule = torch.zeros(1, 1, 3 * H * hd, device=DEV, dtype=dt), f"{H} heads of {hd}: a head size is a multiple of {step} "
        kp, vp = (torch.zeros(1, H, 16, hd, device=DEV, dtype=dt) for _ in range(2))
        table, past = torch.zeros(1, 1, **i), torch.zeros(1, **i)
        calls = [lambda: ops().qk_norm_rope(qkv, None, None, None, None, H, EPS),
                 lambda: ops().qk_norm_rope_bwd(qkv, qkv, None, None, None, None, H, EPS),
                 lambda: ops().kv_append_paged(qkv, kp, vp, table, past, None, None, None, None, None, EPS, err())]
        for call in calls:
            with pytest.raises(RuntimeError, match=rule):
                call()
        if H < 129:
            with pytest.raises(RuntimeError, match=f"heads of {hd}: a head size is a multiple of {step} "):
                ops().attn_decode_shared(torch.zeros(1, 1, H * hd, device=DEV, dtype=dt), kp, vp, None, None, table, past, None, 0,
                                         16, 0, err())


@gpu
def test_overlapping_pools_are_refused():
    """One tensor for both pools, or two views that share rows: keys and values would overwrite each other in no order.
    Neighbouring halves of one tensor are two pools."""
    S, Lq, H, hd, ps = 2, 3, 2, 16, 16
    qkv, q_w, k_w, pos, f = inputs(S, Lq, H, hd, 16, torch.float32)
    both = torch.zeros(8, H, ps, hd, device=DEV)
    table, past = torch.arange(4, device=DEV).view(2, 2).int(), torch.zeros(2, device=DEV).int()
    for kp, vp in ((both[:4], both[:4]), (both[:4], both[3:7]), (both[3:7], both[:4])):
        with pytest.raises(RuntimeError, match="overlap"):
            ops().kv_append_paged(qkv, kp, vp, table, past, None, q_w, k_w, pos, f, EPS, err())
    assert (both == 0).all()
    kp, vp = cache(4, H, ps, hd, torch.float32)
    both[4:], both[:4] = kp, vp
    want = ops().kv_append_paged(qkv, kp, vp, table, past, None, q_w, k_w, pos, f, EPS, err())
    got = ops().kv_append_paged(qkv, both[4:], both[:4], table, past, None, q_w, k_w, pos, f, EPS, err())
    assert torch.equal(got, want) and torch.equal(both[4:], kp) and torch.equal(both[:4], vp)


def test_c_abi_refuses_overlapping_pools():
    lib = _lib()
    P = 1 << 20  # never read
    size = 4 * 4 * 64 * 64 * 2
    for vp in (P, P + size - 16, P - size + 16):
        assert lib.esgpt_kv_append_paged(P, P, P, P, 0, P, 64, 1e-6, None, P, P, 2, P, vp, 4, 64, P, 2, 1, 4, 64, 1, None, None) == 1


@gpu
@pytest.mark.parametrize("shape", [(3, 5, 1, 4, 4), (2, 33, 7, 12, 8), (1, 9, 3, 20, 2), (2, 6, 2, 124, 100), (5, 3, 1, 100, 0)],
                         ids=str)
def test_f32_heads_that_are_multiples_of_four(shape):
    """Through a normalising append and back: the operator on rows, its backward, the append and the pools' rows."""
    B, T, H, hd, R = shape
    qkv, q_w, k_w, pos, f = inputs(B, T, H, hd, R, torch.float32)
    y = ops().qk_norm_rope(qkv, q_w, k_w, pos, f, H, EPS)
    x, w = qkv.double().requires_grad_(), [t.double().requires_grad_() for t in (q_w, k_w)]
    want = oracle(x, *w, pos, f, H)
    close(y, want.detach(), torch.float32, want.abs().max().item() * math.sqrt(2))
    dout = torch.randn(qkv.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    grads = torch.autograd.grad(want, [x, *w], dout.double())
    dqkv, dw = ops().qk_norm_rope_bwd(dout, qkv, q_w, k_w, pos, f, H, EPS)
    xs = qkv[..., : 2 * H * hd].double().view(B, T, 2 * H, hd)
    r = torch.rsqrt(xs.pow(2).mean(-1) + EPS).max().item() * max(t.abs().max().item() for t in (q_w, k_w))
    close(dqkv, grads[0], torch.float32, 2 * r * dout.double().abs().max().item() * math.sqrt(2), 96)
    xh = (xs.view(B, T, 2, H, hd) * torch.rsqrt(xs.view(B, T, 2, H, hd).pow(2).mean(-1, keepdim=True) + EPS)).abs()
    mag = (xh * math.sqrt(2) * dout.double().abs().max()).sum((0, 1, 3))
    for i in range(2):
        assert ((dw[i].double() - grads[1 + i]).abs() <= (24 + 64 + B * T * H) * U * mag[i]).all()
    kp, vp = cache(B * 4, H, 16, hd, torch.float32)
    table, past = torch.randperm(B * 4, generator=torch.Generator().manual_seed(2)).view(B, 4).int(), torch.arange(B).int() * 5
    wq, wk, wv = append_oracle(y, kp, vp, table, past, None, H)
    q = ops().kv_append_paged(qkv, kp, vp, table.to(DEV), past.to(DEV), None, q_w, k_w, pos, f, EPS, err())
    assert torch.equal(q, wq) and torch.equal(kp, wk) and torch.equal(vp, wv) and int(err()[0]) == 0


@gpu
def test_one_weight_for_queries_and_keys():
    """A weight that both share gets the sum of both gradients; in two calls of one graph, of all four."""
    B, T, H, hd, R = 2, 9, 3, 32, 32
    qkv, q_w, _, pos, f = inputs(B, T, H, hd, R, torch.float32)
    dout = torch.randn_like(qkv)
    _, dw = ops().qk_norm_rope_bwd(dout, qkv, q_w, q_w, pos, f, H, EPS)
    q_w.requires_grad_()
    (ops().qk_norm_rope(qkv, q_w, q_w, pos, f, H, EPS) * dout).sum().backward()
    assert torch.equal(q_w.grad, dw[0] + dw[1])
    once, q_w.grad = q_w.grad.clone(), None
    a = ops().qk_norm_rope(qkv, q_w, q_w, pos, f, H, EPS)
    b = ops().qk_norm_rope(qkv, q_w, q_w, pos, f, H, EPS)
    ((a + b) * dout).sum().backward()
    assert (q_w.grad - 2 * once).abs().max() <= 4 * U * 2 * (dw[0].abs() + dw[1].abs()).max()
