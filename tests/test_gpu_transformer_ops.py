"""GPU tests of the transformer-block operators (``ops.qk_norm_rope``, ``ops.mha``, ``ops.attention_rope``) against their definitions in 64 bits.

Every bound is derived, element by element, from the roundings the kernels make: ``u`` = half a step of the 16-bit type
(``torch.finfo(t).eps / 2``), e = 2^-24 for a 32-bit operation; the derivation stands where the bound is formed."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


@pytest.fixture(scope="module")
def R():
    import revisiting_at_amd as R
    assert torch.cuda.is_available()
    R._lib.load()
    return R


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def inside(got, ref, bound, what=""):
    got, ref, bound = got.detach().double().cpu(), ref.detach().double().cpu(), bound.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got - ref).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float((off / bound.clamp(min=1e-300))[bad].max()), float(off[bad].max()))


# ------------------------------------------------------------------------------------------------------------------ qk_norm_rope
def rope_angles(positions, inv_freq, sections):
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)])
    return positions.double().cpu()[..., axis] * inv_freq.double().cpu()          # [(B,) N, d / 2]


def split_pairs(x, il):
    return (x[..., 0::2], x[..., 1::2]) if il else x.chunk(2, -1)


def join_pairs(a, b, il):
    return torch.stack((a, b), -1).flatten(-2) if il else torch.cat((a, b), -1)


def rope_ref(x, w, angle, norm, il, eps, dy=None):
    """(y, bound of y in 32 bits) and, with dy, (dx, its bound, dw, its bound) of one of q, k in 64 bits."""
    x = x.double().cpu()
    d = x.shape[-1]
    w = torch.ones(d, dtype=torch.float64) if w is None else w.detach().double().cpu()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) if norm else torch.ones(x.shape[:-1] + (1,), dtype=torch.float64)
    xh = x * r
    z = xh * w
    c, s = (torch.ones(1).double(), torch.zeros(1).double()) if angle is None else (angle.cos().unsqueeze(-2), angle.sin().unsqueeze(-2))
    za, zb = split_pairs(z, il)
    y = join_pairs(za * c - zb * s, zb * c + za * s, il)
    # r: the mean of d squares (16 in a lane, then at most 4 exchanges), all positive: 21 roundings, halved by the root; + eps, root, quotient,
    # the factor 1/d: 5;  x r w: 2;  the angle in turns rounded to 24 bits: 2 pi / 4 e, cos and sin: 2 e each;  the turn: 3.  Sum under 32.
    both = za.abs() + zb.abs()
    yb = join_pairs(both, both, il) * 32 * E
    if dy is None:
        return y, yb
    dy = dy.double().cpu()
    ga, gb = split_pairs(dy, il)
    dz = join_pairs(ga * c + gb * s, gb * c - ga * s, il)
    mag = join_pairs(ga.abs() + gb.abs(), ga.abs() + gb.abs(), il)                # >= |dz|; dz is 8 e off relative to it
    t = dz * xh
    dw, dwb = t.sum((0, 1, 2)), (mag * xh.abs()).sum((0, 1, 2))
    if norm:
        dot = (t * w).mean(-1, keepdim=True)
        tall = (mag * xh.abs() * w.abs()).mean(-1, keepdim=True)
        dx = r * (dz * w - xh * dot)
        # dz w: 9; xh: 20; the mean of d products of 30 e each, 21 deep: 52; the last two: 2 + r's 16
        dxb = r * (mag * w.abs() * 32 + xh.abs() * tall * 96) * E
    else:
        dx, dxb = dz, mag * 10 * E
    # a sum over all rows: 30 e each, as deep as there are rows at most (tested sizes: 2^12 rows' worth at most)
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    return y, yb, dx, dxb, dw, dwb * (30 + min(rows, 4096) + 100) * E


ROPE = [  # B, N, Hq, Hk, d, axes, norm, interleaved, per-batch positions, far
    (2, 5, 3, 3, 64, 2, True, False, False, 0),
    (1, 1, 1, 1, 64, 1, True, False, False, 0),
    (2, 1, 4, 1, 128, 1, True, False, True, 1_000_000),
    (1, 197, 6, 6, 64, 2, True, False, False, 0),
    (3, 50, 12, 4, 128, 3, True, True, True, 1000),
    (2, 33, 2, 2, 32, 2, True, True, False, 7),
    (1, 7, 5, 2, 96, 3, True, False, True, 0),
    (1, 7, 3, 3, 80, 4, True, True, False, 0),
    (2, 9, 2, 1, 16, 1, True, False, False, 100),
    (1, 9, 2, 1, 256, 2, True, False, False, 100),
    (2, 40, 4, 2, 64, 2, False, False, False, 0),
    (2, 40, 4, 2, 64, 2, False, True, True, 0),
    (1, 6, 2, 2, 64, 0, True, False, False, 0),
    (1, 1300, 3, 1, 64, 2, True, False, False, 0),
    (8, 700, 1, 1, 48, 1, True, False, True, 0),
]


def rope_inputs(R, case, dtype, wdtype, seed):
    B, N, Hq, Hk, d, axes, norm, il, per, far = case
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, N, Hq + 2 * Hk, d, generator=g).to(dtype).cuda()
    q, k = qkv[:, :, :Hq].detach().requires_grad_(), qkv[:, :, Hq:Hq + Hk].detach().requires_grad_()
    wq = wk = pos = inv = sec = None
    if norm:
        wq, wk = ((1 + 0.3 * torch.randn(d, generator=g)).to(wdtype).cuda().requires_grad_() for _ in range(2))
    if axes:
        sec = [d // 2 // axes + (a < d // 2 % axes) for a in range(axes)]
        inv = torch.cat([100.0 ** (-torch.arange(n).float() / n) for n in sec]).cuda()
        pos = torch.randint(0, 60, (B, N, axes) if per else (N, axes), generator=g) + far
        pos = pos.to([torch.int64, torch.int32, torch.float32][seed % 3]).cuda()
    dq, dk = (torch.randn(B, N, h, d, generator=g).to(dtype).cuda() for h in (Hq, Hk))
    return q, k, wq, wk, pos, inv, sec, dq, dk


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(str(int(v)) for v in c))
def test_qk_norm_rope_against_its_definition(R, case, dtype):
    norm, il = case[6], case[7]
    wdtype = dtype if case[1] % 2 else torch.float32
    q, k, wq, wk, pos, inv, sec, dq, dk = rope_inputs(R, case, dtype, wdtype, case[1] + case[4])
    yq, yk = R.ops.qk_norm_rope(q, k, wq, wk, pos, inv, sec, norm=norm, interleaved=il)
    leaves = (q, k) + ((wq, wk) if norm else ())
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    angle = None if pos is None else rope_angles(pos, inv, sec)
    u = 0.0 if dtype == torch.float32 else half_step(dtype)
    uw = 0.0 if wdtype == torch.float32 else half_step(wdtype)
    for i, (x, w, dy, y) in enumerate(((q, wq, dq, yq), (k, wk, dk, yk))):
        ry, by, rx, bx, rw, bw = rope_ref(x, w, angle, norm, il, 1e-6, dy)
        assert y.dtype == dtype and y.is_contiguous()
        inside(y, ry, by * (1 + u) + u * ry.abs(), "y")
        inside(grads[i], rx, bx * (1 + u) + u * rx.abs(), "dx")
        if norm:
            assert grads[2 + i].dtype == wdtype
            inside(grads[2 + i], rw, bw * (1 + uw) + uw * rw.abs(), "dw")


def test_qk_norm_rope_gradient_against_differences(R):
    """d/dh of <y(x + h u), dy> by central differences of the definition in 64 bits: the derivative along a direction through q, k and both weights."""
    case = (2, 11, 3, 2, 64, 2, True, False, False, 0)
    q, k, wq, wk, pos, inv, sec, dq, dk = rope_inputs(R, case, torch.float32, torch.float32, 4)
    grads = torch.autograd.grad(R.ops.qk_norm_rope(q, k, wq, wk, pos, inv, sec), (q, k, wq, wk), (dq, dk))
    angle = rope_angles(pos, inv, sec)
    g = torch.Generator().manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g).double() for t in (q, k, wq, wk)]

    def value(h):
        xq, xk, vq, vk = (t.detach().double().cpu() + h * u for t, u in zip((q, k, wq, wk), dirs))
        return sum(float((rope_ref(x, w, angle, True, False, 1e-6)[0] * dy.double().cpu()).sum()) for x, w, dy in ((xq, vq, dq), (xk, vk, dk)))
    h = 1e-5
    want = (value(h) - value(-h)) / (2 * h)
    got = sum(float((t.double().cpu() * u).sum()) for t, u in zip(grads, dirs))
    # the differences are h^2 of the third derivative off (1e-10 of a value of the sum's size), the gradients 100 e of their sizes
    size = sum(float((t.double().cpu() * u).abs().sum()) for t, u in zip(grads, dirs))
    assert abs(got - want) <= 100 * E * size + 1e-7 * size


def test_qk_norm_rope_strides_and_shared_inputs(R):
    """Views that cannot be read in place, broadcast inputs and expanded gradients give what contiguous copies give."""
    g = torch.Generator().manual_seed(0)
    pos, inv = torch.arange(10).view(10, 1).cuda(), (100.0 ** (-torch.arange(32).float() / 32)).cuda()
    wide = torch.randn(2, 10, 3, 130, generator=g).cuda()
    for q in (wide[..., 1:65], wide[..., ::2][..., :64], wide.permute(0, 1, 2, 3)[..., :64], wide[:1, :, :, :64].expand(2, 10, 3, 64),
              torch.randn(2, 3, 10, 64, generator=g).cuda().transpose(1, 2)):
        a = R.ops.qk_norm_rope(q, q, positions=pos, inv_freq=inv)
        b = R.ops.qk_norm_rope(q.contiguous(), q.contiguous(), positions=pos, inv_freq=inv)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = torch.randn(1, 10, 3, 64, generator=g).cuda().requires_grad_()
    yq, yk = R.ops.qk_norm_rope(x.expand(2, 10, 3, 64), x.expand(2, 10, 3, 64), positions=pos, inv_freq=inv)
    (gx,) = torch.autograd.grad(yq.sum() + yk.sum(), x)
    one = x.detach().requires_grad_()
    y1, _ = R.ops.qk_norm_rope(one, one.detach(), positions=pos, inv_freq=inv)
    (g1,) = torch.autograd.grad(y1.sum(), one)
    torch.testing.assert_close(gx, 4 * g1, rtol=4 * E, atol=0)                    # a sum of four equal numbers: two roundings
    # only one output used; and no tokens at all
    (g2,) = torch.autograd.grad(R.ops.qk_norm_rope(one, one.detach(), positions=pos, inv_freq=inv)[0].sum(), one)
    assert torch.equal(g1, g2)
    w = torch.ones(64, device="cuda", requires_grad=True)
    none = torch.empty(0, 10, 3, 64, device="cuda", requires_grad=True)
    y = R.ops.qk_norm_rope(none, none, w, w, pos, inv)[0]
    gn, gw = torch.autograd.grad(y.sum(), (none, w))
    assert y.shape == none.shape and gn.shape == none.shape and not bool(gw.any())


# ------------------------------------------------------------------------------------------------------------------ mha
def mha_ref(q, k, v, scale, causal, q_lens, kv_lens, dout, u, rounded=True, scaled=False):
    """The definition in 64 bits, a sample and head at a time, and how far the kernel's roundings may lead from it:
    out: P is rounded to 16 bits (u) and the result once more; exp's argument and the sums in 32 bits (t).
    dv: the same with P^T and dout.   D is formed from the rounded out.   dS is rounded once, the products' results once.
    scaled: dS is rounded to fp16 after a power of two has brought 2 max|dout| max|v| to 2^13 or more: 2^-11 of it, or half of fp16's smallest step."""
    B, Nq, H, d = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    q, k, v, dout = (x.detach().double().cpu() for x in (q, k, v, dout))
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    bo, bq, bk, bv = (torch.zeros_like(x) for x in (q, q, k, v))
    for b in range(B):
        ql = Nq if q_lens is None else min(max(int(q_lens[b]), 0), Nq)
        kl = Nk if kv_lens is None else min(max(int(kv_lens[b]), 0), Nk)
        i, j = torch.arange(Nq).view(-1, 1), torch.arange(Nk).view(1, -1)
        ok = (i < ql) & (j < kl)
        if causal:
            ok &= j <= i + kl - ql
        for h in range(H):
            hk = h // (H // Hkv)
            Q, K, V, G = q[b, :, h].clone(), k[b, :, hk].clone(), v[b, :, hk].clone(), dout[b, :, h].clone()
            Q[ql:], G[ql:], K[kl:], V[kl:] = 0, 0, 0, 0
            S = (Q @ K.T) * scale
            Sm = S.masked_fill(~ok, -torch.inf)
            top = Sm.amax(1, keepdim=True) if Nk else torch.full((Nq, 1), -torch.inf).double()
            P = torch.exp(Sm - torch.where(top == -torch.inf, 0.0, top))
            Z = P.sum(1, keepdim=True)
            P = P / torch.where(Z == 0, 1.0, Z)
            G = torch.where(ok.any(1, keepdim=True), G, 0.0)
            # 32-bit part, relative to P: a score is d + 2 operations of e of sum |q k| off, twice (against the maximum's or lse's own error),
            # the sums over keys Nk deep, exp and log themselves 2^-20
            t = 2 * (d + 4) * E * scale * float((Q.abs() @ K.abs().T).max() if Nk else 0) + (Nk + Nq) * E + 2.0 ** -20
            O = P @ V
            eo = (u + t) * (P @ V.abs())
            out[b, :, h], bo[b, :, h] = O, eo + u * (O.abs() + eo)
            DP, Dv = G @ V.T, (G * O).sum(1, keepdim=True)
            DS = P * (DP - Dv)
            size = G.abs() @ V.abs().T
            eD = (G.abs() * (eo + u * (O.abs() + eo))).sum(1, keepdim=True) + d * E * (G.abs() * O.abs()).sum(1, keepdim=True)
            us = 2.0 ** -11 if scaled else u
            eS = (us + 2 * t) * DS.abs() + (1 + us) * P * (d * E * size + eD)
            if scaled:
                eS = eS + 2.0 ** -25 * 2.0 ** -13 * 2 * G.norm(dim=1).max() * V.norm(dim=1).max()
            # the 16-bit type's smallest steps (fp16: 2^-25 half a step below 2^-14)
            tiny = 2.0 ** -25 if u == 2.0 ** -11 else 0.0
            eP = torch.where(ok, (u + 2 * t) * P + tiny, 0.0)
            eS = torch.where(ok, eS + tiny, 0.0)
            for acc, err, x, ex in ((dq[b, :, h], bq[b, :, h], DS @ K, eS @ K.abs()), (dk[b, :, hk], bk[b, :, hk], DS.T @ Q, eS.T @ Q.abs())):
                acc += x * scale
                err += (ex + (Nq + Nk) * E * x.abs()) * scale
            dv[b, :, hk] += P.T @ G
            bv[b, :, hk] += eP.T @ G.abs()
    for g, e in ((dq, bq), (dk, bk), (dv, bv)) if rounded else ((dv, bv),):        # not rounded: dq and dk as they are in 32 bits
        e += u * (g.abs() + e) + (2.0 ** -25 if u == 2.0 ** -11 else 0.0)
    bo += 2.0 ** -24 if u == 2.0 ** -11 else 0.0                                   # P's smallest step times v, and out's own
    return (out, dq, dk, dv), (bo, bq, bk, bv)


def heads(B, N, H, d, layout, dtype, g, scale=1.0):
    x = (torch.randn(B, N, H, d, generator=g) * scale).to(dtype).cuda()
    if layout == "heads":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "packed":
        return torch.cat((x, x, x), 2)[:, :, H:2 * H]
    return x


MHA = [  # B, Nq, Nk, H, Hkv, d, causal, lens (q, kv) or None, layout
    (1, 1, 1, 1, 1, 64, False, None, "tokens"),
    (2, 197, 197, 3, 3, 64, False, None, "packed"),
    (1, 63, 65, 2, 2, 64, False, None, "heads"),
    (1, 128, 64, 2, 1, 64, True, None, "tokens"),              # causal with more queries than keys: the first 64 see nothing
    (1, 129, 257, 4, 2, 64, True, None, "tokens"),
    (2, 300, 300, 2, 2, 128, True, None, "packed"),
    (1, 64, 128, 6, 2, 128, False, None, "heads"),
    (3, 130, 130, 2, 2, 64, False, ([0, 130, 77], [0, 130, 77]), "tokens"),
    (3, 130, 130, 2, 2, 64, True, ([0, 130, 77], [0, 130, 77]), "heads"),
    (4, 70, 200, 4, 1, 64, True, ([70, 1, 69, 200], [3, 200, 0, -5]), "tokens"),   # lengths are clamped; some queries see nothing
    (2, 90, 140, 3, 3, 128, False, (None, [1, 140]), "tokens"),
    (2, 1, 2000, 8, 2, 64, False, None, "heads"),              # split over the keys
    (1, 3, 1500, 4, 4, 128, True, None, "tokens"),
    (2, 17, 900, 2, 1, 64, False, ([17, 3], [900, 5]), "tokens"),                   # splits that hold no key
    (1, 577, 577, 2, 2, 64, False, None, "packed"),
    (1, 5, 0, 2, 2, 64, False, None, "tokens"),                # no key at all
    (1, 700, 150, 4, 1, 64, True, None, "tokens"),             # few key tiles: dk and dv split over the rows
    (2, 1100, 70, 2, 1, 128, False, ([1100, 9], [70, 33]), "heads"),
    (1, 20, 140, 70, 1, 64, True, None, "packed"),             # more heads on a key head than rows in a tile
    (2, 600, 600, 2, 1, 128, True, ([600, 5], [600, 300]), "tokens"),
]


def mha_case(case, dtype, seed=0, spread=1.0):
    B, Nq, Nk, H, Hkv, d, causal, lens, layout = case
    g = torch.Generator().manual_seed(seed + Nq + Nk)
    q = heads(B, Nq, H, d, layout, dtype, g, spread).detach().requires_grad_()
    k, v = (heads(B, Nk, Hkv, d, layout, dtype, g).detach().requires_grad_() for _ in range(2))
    ql, kl = (None, None) if lens is None else (None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in lens)
    return q, k, v, torch.randn(B, Nq, H, d, generator=g).to(dtype).cuda(), ql, kl, causal


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", MHA, ids=lambda c: "-".join(map(str, c[:6])) + ("-causal" if c[6] else "") + ("-lens" if c[7] else ""))
def test_mha_against_its_definition(R, case, dtype):
    q, k, v, dout, ql, kl, causal = mha_case(case, dtype)
    out = R.ops.mha(q, k, v, causal=causal, q_lens=ql, kv_lens=kl)
    assert out.dtype == dtype and out.shape == q.shape and out.is_contiguous()
    got = (out,) + torch.autograd.grad(out, (q, k, v), dout)
    ref, bound = mha_ref(q, k, v, case[5] ** -0.5, causal, ql, kl, dout, half_step(dtype))
    for name, a, b, c in zip(("out", "dq", "dk", "dv"), got, ref, bound):
        inside(a, b, c, name)
    with torch.no_grad():
        assert torch.equal(R.ops.mha(q, k, v, causal=causal, q_lens=ql, kv_lens=kl), out)


@pytest.mark.parametrize("spread", [8.0, 0.0])
def test_mha_with_peaked_and_flat_scores(R, spread):
    """Scores of +-100 (one key takes all) and equal scores."""
    case = (1, 150, 290, 2, 2, 64, False, None, "tokens")
    q, k, v, dout, ql, kl, causal = mha_case(case, torch.bfloat16, 3, spread)
    out = R.ops.mha(q, k, v)
    got = (out,) + torch.autograd.grad(out, (q, k, v), dout)
    ref, bound = mha_ref(q, k, v, 0.125, False, None, None, dout, half_step(torch.bfloat16))
    for name, a, b, c in zip(("out", "dq", "dk", "dv"), got, ref, bound):
        inside(a, b, c, name)


def test_mha_gradient_against_differences(R):
    """<gradient, direction> against central differences of the definition in 64 bits."""
    case = (2, 40, 70, 4, 2, 64, True, None, "tokens")
    q, k, v, dout, _, _, causal = mha_case(case, torch.bfloat16, 5)
    grads = torch.autograd.grad(R.ops.mha(q, k, v, causal=True), (q, k, v), dout)
    u = half_step(torch.bfloat16)
    _, bound = mha_ref(q, k, v, 0.125, True, None, None, dout, u)
    g = torch.Generator().manual_seed(2)
    dirs = [torch.randn(t.shape, generator=g).double() for t in (q, k, v)]

    def value(h):
        x = [t.detach().double().cpu() + h * e for t, e in zip((q, k, v), dirs)]
        return float((mha_ref(*x, 0.125, True, None, None, dout, u)[0][0] * dout.double().cpu()).sum())
    h = 1e-4
    want = (value(h) - value(-h)) / (2 * h)
    got = sum(float((t.double().cpu() * e).sum()) for t, e in zip(grads, dirs))
    off = sum(float((b * e.abs()).sum()) for b, e in zip(bound[1:], dirs))
    assert abs(got - want) <= off + 1e-5 * abs(want) + 1e-4          # the differences' own error: h^2 times a third derivative


def test_mha_padding_is_never_used(R):
    """NaN and infinities behind the lengths change no bit, forward and backward, and padded rows come out as zeros."""
    case = (3, 130, 130, 4, 2, 64, False, ([0, 130, 77], [0, 130, 77]), "tokens")
    for causal in (False, True):
        q, k, v, dout, ql, kl, _ = mha_case(case, torch.bfloat16)
        clean = R.ops.mha(q, k, v, causal=causal, q_lens=ql, kv_lens=kl)
        want = (clean,) + torch.autograd.grad(clean, (q, k, v), dout)
        bad = [t.detach().clone() for t in (q, k, v, dout)]
        for t, val in zip(bad, (float("nan"), float("inf"), float("nan"), float("-inf"))):
            t[0], t[2, 77:] = val, val
        x = [t.requires_grad_() for t in bad[:3]]
        out = R.ops.mha(*x, causal=causal, q_lens=ql, kv_lens=kl)
        for name, a, b in zip(("out", "dq", "dk", "dv"), (out,) + torch.autograd.grad(out, x, bad[3]), want):
            assert torch.equal(a, b), name
            assert not bool(a[0].any()) and not bool(a[2, 77:].any())


def test_mha_same_bits_every_time_on_any_stream_and_in_a_graph(R):
    for case in (MHA[1], MHA[5], MHA[11]):
        q, k, v, dout, ql, kl, causal = mha_case(case, torch.bfloat16)

        def both():
            out = R.ops.mha(q, k, v, causal=causal)
            return (out.detach(),) + torch.autograd.grad(out, (q, k, v), dout)
        want = both()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = both()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both()
        for _ in range(3):
            for t in got:
                t.fill_(7)
            both()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_mha_broadcast_inputs_and_expanded_gradient(R):
    g = torch.Generator().manual_seed(0)
    q = torch.randn(3, 40, 4, 64, generator=g).to(torch.bfloat16).cuda()
    k = torch.randn(1, 50, 2, 64, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    out = R.ops.mha(q, k.expand(3, 50, 2, 64), k.expand(3, 50, 2, 64))
    (gk,) = torch.autograd.grad(out.sum(), k)                                      # dout: a zero-stride tensor of ones
    kk = k.detach().repeat(3, 1, 1, 1).requires_grad_()
    out2 = R.ops.mha(q, kk, kk)
    (g2,) = torch.autograd.grad(out2, kk, torch.ones_like(out2))
    assert torch.equal(out, out2)
    torch.testing.assert_close(gk.float(), g2.float().sum(0, keepdim=True), rtol=2.0 ** -6, atol=2.0 ** -6)   # sums of three in bf16


def test_refusals_name_what_is_wrong(R):
    bf = dict(device="cuda", dtype=torch.bfloat16)
    q, k = torch.zeros(2, 5, 4, 64, **bf), torch.zeros(2, 7, 2, 64, **bf)
    mha, rope, layer = R.ops.mha, R.ops.qk_norm_rope, R.ops.attention_rope
    for err, f in (
            (TypeError, lambda: mha(q.float(), k.float(), k.float())), (ValueError, lambda: mha(q, k, k[:, :6])),
            (ValueError, lambda: mha(q[:, :, :3], k, k)), (ValueError, lambda: mha(q[..., :32], k[..., :32], k[..., :32])),
            (ValueError, lambda: mha(q, k, k, scale=0.0)), (ValueError, lambda: mha(q, k, k, scale=float("nan"))),
            (TypeError, lambda: mha(q, k.half(), k.half())), (ValueError, lambda: mha(q[0], k, k)),
            (ValueError, lambda: mha(q, k, k, kv_lens=torch.tensor([1, 2], device="cuda"))),
            (ValueError, lambda: mha(q, k, k, kv_lens=torch.tensor([1], dtype=torch.int32, device="cuda"))),
            (ValueError, lambda: mha(q, k, k, q_lens=torch.tensor([1, 2], dtype=torch.int32))),
            (R._lib.ApgdHipError, lambda: mha(q.cpu(), k.cpu(), k.cpu())), (TypeError, lambda: mha(q, k, None)),
            (ValueError, lambda: rope(q, k)), (ValueError, lambda: rope(q[..., :40], q[..., :40])),
            (ValueError, lambda: rope(q, q, inv_freq=torch.ones(32, device="cuda"))),
            (ValueError, lambda: rope(q, q, positions=torch.zeros(5, 1, device="cuda"))),
            (ValueError, lambda: rope(q, q, positions=torch.zeros(4, 1, device="cuda"), inv_freq=torch.ones(32, device="cuda"))),
            (TypeError, lambda: rope(q, q, positions=torch.zeros(5, 1, device="cuda").half(), inv_freq=torch.ones(32, device="cuda"))),
            (ValueError, lambda: rope(q, q, positions=torch.zeros(5, 2, device="cuda"), inv_freq=torch.ones(32, device="cuda"), sections=[16, 15])),
            (ValueError, lambda: rope(q, q, positions=torch.zeros(5, 5, device="cuda"), inv_freq=torch.ones(32, device="cuda"), sections=[8, 8, 8, 8, 0])),
            (ValueError, lambda: rope(q, q, torch.ones(64, device="cuda"), norm=False)), (ValueError, lambda: rope(q, q, torch.ones(32, device="cuda"))),
            (TypeError, lambda: rope(q, q, torch.ones(64, device="cuda").half())), (ValueError, lambda: rope(q, q, eps=-1.0)),
            (ValueError, lambda: layer(torch.zeros(2, 5, 3 * 4 * 32, **bf), 4)), (ValueError, lambda: layer(torch.zeros(2, 5, 100, **bf), 4)),
            (TypeError, lambda: layer(torch.zeros(2, 5, 768, device="cuda"), 4)), (R._lib.ApgdHipError, lambda: layer(torch.zeros(2, 5, 768), 4))):
        with pytest.raises(err):
            f()
    x = q.clone().requires_grad_()                                                  # once differentiable: a second derivative is refused
    (gx,) = torch.autograd.grad(mha(x, k, k).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.float().sum(), x)


# ------------------------------------------------------------------------------------------------------------------ attention_rope
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("norm,rotate", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("B,side,H,d", [(2, 14, 3, 64), (1, 24, 2, 64), (2, 6, 2, 128), (1, 0, 1, 64)])
def test_attention_rope_is_its_two_operators(R, B, side, H, d, norm, rotate, dtype):
    """Bit for bit ``qk_norm_rope`` then ``mha`` on slices of the projection, where q' and k' are of the projection's type: forward, and dv where no row
    is split over workgroups; all gradients where nothing is turned.  (Elsewhere dq' and dk' are not rounded in between.)"""
    if norm and dtype == torch.bfloat16:
        pytest.skip("q' and k' in fp16: against the definition below")
    N = side * side + 1
    g = torch.Generator().manual_seed(N)
    qkv = torch.randn(B, N, 3 * H * d, generator=g).to(dtype).cuda().requires_grad_()
    wq, wk = ((1 + 0.1 * torch.randn(d, generator=g)).cuda().requires_grad_() for _ in range(2)) if norm else (None, None)
    n = torch.arange(side * side)
    pos = torch.cat([torch.zeros(1, 2, dtype=torch.int64), torch.stack([n // max(side, 1), n % max(side, 1)], -1) + 1]).cuda() if rotate else None
    sec = [d // 4, d // 4] if rotate else None
    inv = torch.cat([100.0 ** (-torch.arange(s).float() / s) for s in sec]).cuda() if rotate else None
    dout = torch.randn(B, N, H * d, generator=g).to(dtype).cuda()
    out = R.ops.attention_rope(qkv, H, None, wq, wk, pos, inv, sec, norm=norm)
    leaves = (qkv,) + ((wq, wk) if norm else ())
    got = (out,) + torch.autograd.grad(out, leaves, dout)
    x = qkv.detach().requires_grad_()
    q, k, v = x.view(B, N, 3, H, d).unbind(2)
    if norm or rotate:
        q, k = R.ops.qk_norm_rope(q, k, wq, wk, pos, inv, sec, norm=norm)
    o2 = R.ops.mha(q, k, v).reshape(B, N, H * d)
    want = (o2,) + torch.autograd.grad(o2, (x,) + ((wq, wk) if norm else ()), dout)
    assert torch.equal(got[0], want[0])
    if R._lib.load().cnx_mha_bwd_ws_floats(B, N, N, H, H, d, 0) == 0:
        assert torch.equal(got[1][..., 2 * H * d:], want[1][..., 2 * H * d:])
    if not norm and not rotate:
        assert torch.equal(got[1], want[1])
    with torch.no_grad():
        assert torch.equal(R.ops.attention_rope(qkv, H, None, wq, wk, pos, inv, sec, norm=norm), out)


ATTN = [  # B, N, H, d, norm, rotate, interleaved, per-batch positions, weights' type (None: none), dout
    (2, 17, 2, 64, True, True, False, False, torch.float32, "whole"),
    (1, 1, 1, 64, True, True, False, False, torch.float32, "whole"),
    (2, 130, 2, 64, True, True, True, True, torch.float32, "whole"),
    (1, 200, 2, 128, True, True, False, True, None, "part"),
    (2, 129, 1, 128, True, True, True, False, torch.float32, "whole"),
    (1, 64, 3, 64, True, False, False, False, "x", "expanded"),
    (1, 65, 2, 64, False, True, False, True, None, "whole"),
    (43, 257, 2, 64, True, True, False, False, torch.float32, "whole"),          # more than one tile of rows and keys
    (3, 577, 2, 64, True, True, False, True, torch.float32, "whole"),           # few tiles: keys and rows split, joined with the way back
    (1, 600, 2, 128, True, True, True, True, torch.float32, "part"),
    (2, 520, 1, 64, False, True, False, False, None, "whole"),
    (1, 1030, 1, 64, True, False, False, False, "x", "expanded"),
    (29, 260, 3, 128, False, True, True, False, None, "part"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(str(v).split(".")[-1] for v in c))
def test_attention_rope_against_its_definition(R, case, dtype):
    """The result of q' and k' as they are rounded - to fp16 where they are normalised, whatever the projection's type - and the backward pass in one:
    dq' and dk' of the same, through the rotation and the norm, rounded once at the end."""
    B, N, H, d, norm, rotate, il, per_batch, wt, part = case
    g = torch.Generator().manual_seed(N + d)
    u = half_step(dtype)
    qkv = torch.randn(B, N, 3 * H * d, generator=g).to(dtype).cuda().requires_grad_()
    wt = dtype if wt == "x" else wt
    wq, wk = (None, None) if wt is None else ((1 + 0.1 * torch.randn(d + 1, generator=g)).to(wt).cuda()[1:].requires_grad_() for _ in range(2))
    pos = torch.randint(-5, 40, (B, N, 2) if per_batch else (N, 2), generator=g).cuda() if rotate else None
    sec = [d // 2 - d // 8, d // 8] if rotate else None
    inv = torch.cat([100.0 ** (-torch.arange(s).float() / s) for s in sec]).cuda() if rotate else None
    dout = torch.randn(B, N, 2 * H * d, generator=g).to(dtype).cuda()
    dout = dout[..., H * d:] if part == "part" else dout[:, :1, :H * d].expand(B, N, H * d) if part == "expanded" else dout[..., :H * d].contiguous()
    out = R.ops.attention_rope(qkv, H, None, wq, wk, pos, inv, sec, norm=norm, interleaved=il)
    leaves = (qkv,) + (() if wt is None else (wq, wk))
    got = torch.autograd.grad(out, leaves, dout)
    q, k, v = qkv.detach().view(B, N, 3, H, d).unbind(2)
    with torch.no_grad():                                                           # the same arithmetic in 32 bits on the same numbers
        yq, yk = R.ops.qk_norm_rope(q.float(), k.float(), *(None if w is None else w.float() for w in (wq, wk)), pos, inv, sec, norm=norm, interleaved=il)
    yq, yk = (y.to(torch.float16 if norm else dtype) for y in (yq, yk))
    scaled = norm and dtype == torch.bfloat16
    (o, dq, dk, dv), (bo, bq, bk, bv) = mha_ref(yq, yk, v, d ** -0.5, False, None, None, dout.reshape(B, N, H, d), u, rounded=False, scaled=scaled)
    angle = rope_angles(pos, inv, sec) if rotate else None
    mine = got[0].view(B, N, 3, H, d).unbind(2)
    inside(out.view(B, N, H, d), o, bo, "out")
    inside(mine[2], dv, bv, "dv")
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for i, (name, x, w, dy, b) in enumerate((("dq", q, wq, dq, bq), ("dk", k, wk, dk, bk))):
        _, _, dx, dxb, dw, dwb = rope_ref(x, w, angle, norm, il, 1e-6, dy)
        # b is carried through the rotation (each member takes part of both) and the norm's linear map, each term by its size
        ea, eb = split_pairs(b, il)
        c, s = (1.0, 0.0) if angle is None else (angle.cos().abs().unsqueeze(-2), angle.sin().abs().unsqueeze(-2))
        eb = join_pairs(ea * c + eb * s, eb * c + ea * s, il)
        if norm:
            x64 = x.double().cpu()
            r = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + 1e-6)
            xh, wa = (x64 * r).abs(), torch.ones(d).double() if w is None else w.detach().double().cpu().abs()
            dwb = dwb + (eb * xh).sum((0, 1, 2))
            eb = r * (eb * wa + xh * (eb * xh * wa).mean(-1, keepdim=True))
        e = eb + 1.01 * dxb                                                         # (32-bit part: of dy's size with its own error)
        inside(mine[i], dx, e + u * (dx.abs() + e) + tiny, name)
        if w is not None:
            last = u if w.dtype == dtype else 0.0
            inside(got[1 + i], dw, 1.01 * dwb + last * (dw.abs() + 1.01 * dwb) + (2.0 ** -25 if w.dtype == torch.float16 else 0.0), "d" + name[1] + " weight")
    with torch.no_grad():
        assert torch.equal(R.ops.attention_rope(qkv, H, None, wq, wk, pos, inv, sec, norm=norm, interleaved=il), out)
    x2 = qkv.detach().requires_grad_()                                              # without weight gradients: the same bits
    (again,) = torch.autograd.grad(R.ops.attention_rope(x2, H, None, None if wq is None else wq.detach(), None if wk is None else wk.detach(), pos, inv, sec,
                                                        norm=norm, interleaved=il), (x2,), dout)
    assert torch.equal(again, got[0])


@pytest.mark.parametrize("B,N,H", [(0, 5, 2), (2, 0, 2)])
def test_empty_calls(R, B, N, H):
    """No sample or no token: empty results and gradients, zeros for the weights'."""
    w = torch.ones(64, device="cuda", requires_grad=True)
    q, k = (torch.zeros(B, N, H, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    pos, inv = torch.zeros(N, 1, device="cuda", dtype=torch.int32), torch.ones(32, device="cuda")
    y = R.ops.qk_norm_rope(q, k, w, w, pos, inv)
    gq, gw = torch.autograd.grad(y, (q, w), [torch.zeros_like(t) for t in y])
    assert y[0].shape == gq.shape == q.shape and not bool(gw.any())
    out = R.ops.mha(q, k, k)
    assert out.shape == q.shape and torch.autograd.grad(out, q, torch.zeros_like(out))[0].shape == q.shape
    qkv = torch.zeros(B, N, 3 * H * 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = R.ops.attention_rope(qkv, H, None, w, w, pos, inv)
    gq, gw = torch.autograd.grad(out, (qkv, w), torch.zeros_like(out))
    assert out.shape == (B, N, H * 64) and gq.shape == qkv.shape and not bool(gw.any())


def test_attention_rope_backward_in_a_graph(R):
    """Forward and backward captured, replayed with eager work in between."""
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(2, 150, 3 * 128, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    pos, inv = torch.arange(150, device="cuda").view(-1, 1), 100.0 ** (-torch.arange(32, device="cuda") / 32)
    dout = torch.randn(2, 150, 128, generator=g).to(torch.bfloat16).cuda()

    def both():
        out = R.ops.attention_rope(qkv, 2, None, w, w, pos, inv)
        return (out.detach(),) + torch.autograd.grad(out, (qkv, w), dout)
    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(both(), want))


def test_attention_rope_with_gradients_and_values_of_any_size(R):
    """dS travels in fp16 behind a power of two: gradients and values far from 1 give the same bits, scaled; rows of very different sizes stay within
    what the scale allows; an infinite gradient does not come out finite."""
    B, N, H, d = 2, 150, 2, 64
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(B, N, 3 * H * d, generator=g).to(torch.bfloat16).cuda()
    dout = torch.randn(B, N, H * d, generator=g).to(torch.bfloat16).cuda()

    def run(qkv, dout):
        x = qkv.clone().requires_grad_()
        out = R.ops.attention_rope(x, H)
        return out.detach(), torch.autograd.grad(out, x, dout)[0]
    out, grad = run(qkv, dout)
    for up in (2.0 ** 40, 2.0 ** -40):
        assert torch.equal(run(qkv, dout * up)[1], grad * up)
        big = qkv.clone()
        big[..., 2 * H * d:] *= up
        o, gr = run(big, dout)
        assert torch.equal(o, out * up) and torch.equal(gr[..., :2 * H * d], grad[..., :2 * H * d] * up) and torch.equal(gr[..., 2 * H * d:], grad[..., 2 * H * d:])
    # a row with 2^-20 of the others' gradient: its dq has a scale of its own
    small = dout.clone()
    small[:, 7] *= 2.0 ** -20
    dq = run(qkv, small)[1][:, 7, :H * d]
    assert torch.equal(dq, grad[:, 7, :H * d] * 2.0 ** -20)
    bad = dout.clone()
    bad[0, 3, 5] = float("inf")
    assert not bool(torch.isfinite(run(qkv, bad)[1][0, 3, :d]).any())


def test_uses_of_autograd(R):
    """Some of the outputs or inputs only, a graph used twice, checkpointing, inputs changed under a graph, a second derivative."""
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(2, 40, 2, 64, generator=g).to(torch.bfloat16).cuda().requires_grad_() for _ in range(3))
    qkv = torch.randn(2, 40, 384, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    w = (1 + 0.1 * torch.randn(64, generator=g)).cuda().requires_grad_()
    pos, inv = torch.arange(40, device="cuda").view(-1, 1), 100.0 ** (-torch.arange(32, device="cuda") / 32)
    do = torch.randn(2, 40, 2, 64, generator=g).to(torch.bfloat16).cuda()
    calls = {"mha": (lambda: R.ops.mha(q, k, v), (q, k, v), do), "rope": (lambda: R.ops.qk_norm_rope(q, k, w, w, pos, inv)[0], (q, w), do),
             "layer": (lambda: R.ops.attention_rope(qkv, 2, None, w, w, pos, inv), (qkv, w), do.flatten(2))}
    for name, (f, leaves, cot) in calls.items():
        want = torch.autograd.grad(f(), leaves, cot)
        out = f()
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, cot, retain_graph=True), want)), name
        for leaf, x in zip(leaves, want):                                           # one at a time
            assert torch.equal(torch.autograd.grad(out, leaf, cot, retain_graph=True)[0], x), name
        torch.autograd.grad(out, leaves, cot)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(out, leaves, cot)
        out = torch.utils.checkpoint.checkpoint(f, use_reentrant=False)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, cot), want)), name
        (gx,) = torch.autograd.grad(f().float().square().sum(), leaves[0], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(gx.float().sum(), leaves[0])
        out = f()
        with torch.no_grad():
            leaves[0].mul_(1)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(out, leaves, cot)
        assert f().requires_grad and not f().detach().requires_grad
        with torch.no_grad():
            assert not f().requires_grad
    yq, yk = R.ops.qk_norm_rope(q, k, w, w, pos, inv)                               # one output only: the other's gradient is zeros
    a = torch.autograd.grad(yq, (q, k), do, retain_graph=True)
    b = torch.autograd.grad((yq, yk), (q, k), (do, torch.zeros_like(do)))
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and not bool(a[1].any())
    x = qkv.detach().requires_grad_()
    with R.ops.input_grad_only():                                                   # the attack's backward: the input's gradient, no weights'
        gx, gw = torch.autograd.grad(R.ops.attention_rope(x, 2, None, w, w, pos, inv), (x, w), do.flatten(2), allow_unused=True)
    assert gw is None and torch.equal(gx, torch.autograd.grad(R.ops.attention_rope(qkv, 2, None, w, w, pos, inv), qkv, do.flatten(2))[0])


@pytest.mark.parametrize("d", [64, 128])
def test_attention_rope_with_gradients_whose_squares_no_fp32_holds(R, d):
    """The power of two that dS is formed behind: gradients and values whose sums of squares would vanish or overflow in 32 bits give the same bits,
    scaled; so do the weights' gradients."""
    B, N, H = 2, 150, 2
    g = torch.Generator().manual_seed(19)
    qkv = torch.randn(B, N, 3 * H * d, generator=g).to(torch.bfloat16).cuda()
    dout = torch.randn(B, N, H * d, generator=g).to(torch.bfloat16).cuda()
    w = (1 + 0.1 * torch.randn(d, generator=g)).cuda()

    def run(qkv, dout):
        x, wq, wk = qkv.clone().requires_grad_(), w.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.autograd.grad(R.ops.attention_rope(x, H, None, wq, wk), (x, wq, wk), dout)
    want = run(qkv, dout)
    C = H * d
    for k in (-75, -77, -79, -80, -82, -86, -90, 64, 80):
        up = 2.0 ** k
        for a, b in zip(run(qkv, dout * up), want):
            assert torch.equal(a, b * up), k
        big = qkv.clone()
        big[..., 2 * C:] *= up                                                      # dq, dk and the weights' follow v, dv does not
        gx, gq, gk = run(big, dout)
        assert torch.equal(gx[..., :2 * C], want[0][..., :2 * C] * up) and torch.equal(gx[..., 2 * C:], want[0][..., 2 * C:]), k
        assert torch.equal(gq, want[1] * up) and torch.equal(gk, want[2] * up), k
        gx, gq, gk = run(big, dout * (1 / up))                                      # and both: their product is what it was
        assert torch.equal(gx[..., :2 * C], want[0][..., :2 * C]) and torch.equal(gx[..., 2 * C:], want[0][..., 2 * C:] * (1 / up)), k
        assert torch.equal(gq, want[1]) and torch.equal(gk, want[2]), k
    # one sample's gradient tiny or zero, or one row's: the others keep their bits (dq), nothing becomes infinite
    for up in (2.0 ** -80, 0.0):
        one = dout.clone()
        one[1] *= up
        gx = run(qkv, one)[0]
        assert torch.equal(gx[0], want[0][0]) and torch.equal(gx[1], want[0][1] * up)
        one = dout.clone()
        one[:, 7] *= up
        gx, gq, gk = run(qkv, one)
        assert all(bool(torch.isfinite(t).all()) for t in (gx, gq, gk))
        rest = [i for i in range(N) if i != 7]
        assert torch.equal(gx[:, 7, :C], want[0][:, 7, :C] * up) and torch.equal(gx[:, rest, :C], want[0][:, rest, :C])
    for a, b in zip(run(qkv, dout * 2.0 ** -110), want):                            # down to bf16's smallest normal number
        assert bool(((a.double() - b.double() * 2.0 ** -110).abs() <= 2.0 ** -8 * b.double().abs() * 2.0 ** -110 + 2.0 ** -126).all())


def test_positions_changed_under_a_graph_raise(R):
    """Positions and frequencies are inputs like the others: changed in place between forward and backward, the backward raises."""
    q, k = (torch.randn(2, 40, 2, 64, device="cuda").to(torch.bfloat16).requires_grad_() for _ in range(2))
    qkv = torch.randn(2, 40, 384, device="cuda").to(torch.bfloat16).requires_grad_()
    pos, inv = torch.arange(40, device="cuda").view(-1, 1), 100.0 ** (-torch.arange(32, device="cuda") / 32)
    calls = ((lambda: R.ops.qk_norm_rope(q, k, None, None, pos, inv)[0], q), (lambda: R.ops.attention_rope(qkv, 2, None, None, None, pos, inv), qkv))
    for f, leaf in calls:
        for change in (lambda: pos.add_(1), lambda: inv.mul_(0.5)):
            out = f()
            change()
            with pytest.raises(RuntimeError, match="inplace"):
                torch.autograd.grad(out, leaf, torch.ones_like(out))
        out = f()                                                                   # unchanged ones, twice, from the same graph
        a, b = (torch.autograd.grad(out, leaf, torch.ones_like(out), retain_graph=True)[0] for _ in range(2))
        assert torch.equal(a, b)
        with torch.no_grad():
            out = f()
            pos.add_(1)                                                             # no graph: nobody minds
    with torch.inference_mode():
        frozen = torch.arange(40, device="cuda").view(-1, 1)
    out = R.ops.qk_norm_rope(q, k, None, None, frozen, inv)[0]                      # a tensor that has no version
    torch.autograd.grad(out, q, torch.ones_like(out))


def test_forward_mode_derivatives_are_refused(R):
    """A dual tensor raises, where it would come back without a tangent (a derivative of zero)."""
    import torch.autograd.forward_ad as fwd
    q = torch.randn(2, 40, 2, 64, device="cuda").to(torch.bfloat16)
    qkv = torch.randn(2, 40, 384, device="cuda").to(torch.bfloat16)
    w, pos, inv = torch.ones(64, device="cuda"), torch.arange(40.0, device="cuda").view(-1, 1), torch.ones(32, device="cuda")
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))                       # noqa: E731
        for f in (lambda: R.ops.mha(dual(q), q, q), lambda: R.ops.mha(q, q, dual(q)), lambda: R.ops.qk_norm_rope(q, dual(q)),
                  lambda: R.ops.qk_norm_rope(q, q, dual(w)), lambda: R.ops.attention_rope(dual(qkv), 2), lambda: R.ops.attention_rope(qkv, 2, None, w, dual(w)),
                  lambda: R.ops.qk_norm_rope(q, q, None, None, dual(pos), inv), lambda: R.ops.attention_rope(qkv, 2, None, None, None, pos, dual(inv))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                f()
        assert bool(torch.isfinite(R.ops.mha(q, q, q)).all())


@pytest.mark.parametrize("d", [64, 128])
def test_padded_queries_give_zeros_beside_keys_that_are_not_finite(R, d):
    """A query that sees no key has zeros and no gradient also where its tile holds queries that see infinities and NaN."""
    g = torch.Generator().manual_seed(4)
    for N, H, Hkv in ((130, 2, 2), (70, 4, 1), (1000, 2, 1)):                       # (1000 keys under 2 heads: split)
        q, k, v, dout = (torch.randn(2, N, h, d, generator=g).to(torch.bfloat16).cuda() for h in (H, Hkv, Hkv, H))
        k[:, 3], v[:, 5], v[:, 6] = float("inf"), float("inf"), float("nan")
        ql, kl = torch.tensor([20, 0], dtype=torch.int32, device="cuda"), torch.tensor([N, N], dtype=torch.int32, device="cuda")
        x = [t.clone().requires_grad_() for t in (q, k, v)]
        for causal in (False, True):
            out = R.ops.mha(*x, causal=causal, q_lens=ql, kv_lens=kl)
            dq, dk, dv = torch.autograd.grad(out, x, dout)
            for t in (out, dq):
                assert not bool(torch.isfinite(t[0, :20]).all())
                assert not bool(t[0, 20:].any()) and not bool(t[1].any())
            assert not bool(dk[1].any()) and not bool(dv[1].any())


def test_long_caches_are_read_in_place(R):
    """A [B, H, N, d] cache whose heads lie 2^25 and more elements apart, offsets beyond 32 bits: one query over a view of it, and no copy."""
    H, N, d, n = 9, 2 ** 18 + 77, 128, 2 ** 18 - 5
    k, v = (torch.empty(1, H, N, d, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator("cuda").manual_seed(s)) for s in (1, 2))
    q = torch.randn(1, 1, H, d, device="cuda").to(torch.bfloat16)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = R.ops.mha(q, k.transpose(1, 2), v.transpose(1, 2), kv_lens=lens)
        assert torch.cuda.max_memory_allocated() - before < k.numel()               # (a copy of one of them: twice that)
    s = torch.stack([k[0, h, :n].float() @ q[0, 0, h].float() for h in range(H)]).double() * d ** -0.5
    p = torch.softmax(s, 1)
    ref = torch.stack([p[h].float() @ v[0, h, :n].float() for h in range(H)])
    # P is rounded to 16 bits (u) and the result once; sums of |v| weighted by P are below the largest |v|, 6 here: 2 u 6, and 2^-20 n^(1/2) of 32-bit sums
    assert float((out[0, 0].float() - ref).abs().max()) <= 2 * 2.0 ** -8 * 6
    assert float((out[0, 0].float() - ref).norm() / ref.norm()) < 2.0 ** -7


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("Nq,Nk,causal,lens", [(300, 1, False, None), (300, 2, False, None), (40, 3, True, None), (70, 64, False, None), (200, 200, True, None),
                                               (130, 600, False, [5, 64, 600])])
def test_mha_gradients_of_queries_with_few_keys(R, Nq, Nk, causal, lens, dtype):
    """Of two or three keys' dP little is left when D is taken away: for queries that see 64 keys or fewer, all in the first tile, D does not come from
    the rounded output."""
    B, H, Hkv, d = 3, 4, 2, 64
    g = torch.Generator().manual_seed(Nq + Nk)
    q, k, v, dout = (torch.randn(B, n, h, d, generator=g).to(dtype).cuda() for n, h in ((Nq, H), (Nk, Hkv), (Nk, Hkv), (Nq, H)))
    x = [t.requires_grad_() for t in (q, k, v)]
    kl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    dq = torch.autograd.grad(R.ops.mha(*x, causal=causal, kv_lens=kl), x, dout)[0].double().cpu()
    u, scale = half_step(dtype), d ** -0.5
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for b in range(B):
        n = Nk if lens is None else lens[b]
        ok = torch.arange(Nk).view(1, -1) < n
        if causal:
            ok = ok & (torch.arange(Nk).view(1, -1) <= torch.arange(Nq).view(-1, 1) + n - Nq)
        ok = ok.expand(Nq, Nk)
        few = (ok.sum(1) <= 64) & (ok.sum(1) > 0)
        for h in range(H):
            Q, G, K, V = (t.detach()[b, :, i].double().cpu() for t, i in ((q, h), (dout, h), (k, h // 2), (v, h // 2)))
            P = torch.softmax(((Q @ K.T) * scale).masked_fill(~ok, -1e300), 1) * ok
            DP = G @ V.T
            DS = P * (DP - (P * DP).sum(1, keepdim=True))
            # dS is rounded once (u); its 32-bit part: the score's d + 2 operations of sum |q k|, exp and log (2^-20) twice over, dP and D d deep
            t = 2 * (d + 4) * E * scale * float((Q.abs() @ K.abs().T).max()) + 2.0 ** -20
            size = G.abs() @ V.abs().T
            eS = u * DS.abs() + 2 * t * P * (DP.abs() + (P * DP.abs()).sum(1, keepdim=True)) + 2 * (d + 64) * E * P * (size + (P * size).sum(1, keepdim=True)) + tiny * ok
            want, bound = (DS @ K) * scale, (eS @ K.abs()) * scale
            inside(dq[b, few, h], want[few], (bound * (1 + u) + u * want.abs() + tiny)[few], (b, h))
