"""What is measured of the transformer-block operators: attention over any number of tokens with its backward pass (``ops.mha``), the
per-head norms of queries and keys with the rotation by positions of one to three axes (``ops.qk_norm_rope``), the two chained on a packed
projection (``ops.attention_rope``), and the AdamW step over many tensors with states in 32 or 8 bits (``optim.FusedAdamW``).

``own`` false: the same operators in elementary torch operations, 32 bits (64 for angles), rounded once at the end."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256             # elements that share a scale in an 8-bit state
SMALL = 4096            # tensors with fewer elements keep 32-bit states
LR, BETAS, EPS, DECAY, STEP = 1e-3, (0.9, 0.95), 1e-8, 0.05, 100
MOST = 2 * 16 * 4096 * 4096 * 128       # B * H * Nq * Nk * d of the largest listed attention


# ------------------------------------------------------------------------------------------------------------------ the cases
def _mha(name, B, Nq, Nk, H, Hkv, d, dtype="bf16", causal=False, lens=False, layout="packed", train=True):
    return {"op": "mha", "name": name, "B": B, "Nq": Nq, "Nk": Nk, "H": H, "Hkv": Hkv, "d": d, "dtype": dtype, "causal": causal,
            "lens": lens, "layout": layout, "train": train}


def _rope(name, B, N, H, Hkv, d, axes, dtype="bf16", norm=True, interleaved=False, far=0, per_batch=False, train=True):
    return {"op": "rope", "name": name, "B": B, "N": N, "H": H, "Hkv": Hkv, "d": d, "axes": axes, "dtype": dtype, "norm": norm,
            "interleaved": interleaved, "far": far, "per_batch": per_batch, "train": train}


def _block(name, B, side, H, norm=True, train=True):
    return {"op": "attention_rope", "name": name, "B": B, "N": side * side + 1, "side": side, "H": H, "d": 64, "norm": norm, "train": train}


def _adamw(name, width, layers, bits, dtype="fp32", classes=1000, tokens=197):
    return {"op": "adamw", "name": name, "width": width, "layers": layers, "bits": bits, "dtype": dtype, "classes": classes,
            "tokens": tokens}


def listed():
    return [
        # one image's worth of small attention: 224 x 224 tokens of the small ViT, where launches and the host's work count
        _mha("mha_train_small", 4, 197, 197, 6, 6, 64),
        # the small ViT at 512 x 512: 32 x 32 patches and the class token, a training batch
        _mha("mha_train_512px", 64, 1025, 1025, 6, 6, 64),
        # images of different resolutions padded to one length: an empty and a full sample among them
        _mha("mha_train_padded", 16, 777, 777, 12, 12, 64, lens=True, layout="tokens"),
        # the largest: causal, shared key / value heads, 128-wide, half precision
        _mha("mha_train_causal_gqa", 2, 4096, 4096, 16, 4, 128, dtype="fp16", causal=True, layout="tokens"),
        # one query of each sequence against a long one: a class token's attention, a decoder's next token
        _mha("mha_single_query", 8, 1, 16384, 16, 4, 128, layout="heads", train=False),
        # two-axis positions of 32 x 32 patches, forward and backward, 12 heads
        _rope("rope_train_image", 32, 1025, 12, 12, 64, 2),
        # time, height, width of a short clip, shared key heads, fp32, forward only
        _rope("rope_video_fp32", 2, 1571, 16, 4, 128, 3, dtype="fp32", interleaved=True, train=False),
        # the next token of each sequence, far down
        _rope("rope_single_far", 16, 1, 16, 4, 128, 1, dtype="fp16", far=1000000, per_batch=True, train=False),
        # a whole attention layer of the base ViT at 384 x 384 from its packed projection, forward and backward
        _block("layer_train_384px", 32, 24, 12),
        # the same at 224 x 224 for one image, forward: an evaluation's smallest call
        _block("layer_eval_224px", 1, 14, 6, train=False),
        # the small ViT's parameters, 32-bit states
        _adamw("adamw32_vit_s", 384, 12, 32),
        # a model of 150 M parameters, 8-bit states
        _adamw("adamw8_large", 1024, 12, 8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mha", "mha", "mha", "rope", "rope", "attention_rope", "adamw", "adamw"])
    if op == "mha":
        d, Hkv = rng.choice([64, 64, 128]), rng.choice([1, 2, 3, 4, 6])
        H = Hkv * rng.choice([1, 1, 2, 4])
        train = rng.random() < 0.75
        Nq = _log(rng, 1, 4096) if train else _log(rng, 1, 64)
        Nk = Nq if rng.random() < 0.7 and train else _log(rng, 1, 16384)
        B = _log(rng, 1, 64)
        while B > 1 and B * H * Nq * Nk * d > MOST:
            B = B // 2
        while B * H * Nq * Nk * d > MOST:
            Nk = Nk // 2
        layout = rng.choice(["packed", "tokens", "heads"])
        return _mha("", B, Nq, Nk, H, Hkv, d, rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.4, rng.random() < 0.4,
                    "tokens" if layout == "packed" and Nq != Nk else layout, train)
    if op == "rope":
        d, Hkv = rng.choice([32, 64, 64, 96, 128]), rng.choice([1, 2, 3, 4, 6, 12])
        H = Hkv * rng.choice([1, 1, 2, 4])
        N = _log(rng, 1, 4096)
        B = _log(rng, 1, 64)
        while B > 1 and B * N * (H + Hkv) * d > 32 * 1025 * 24 * 64:
            B = B // 2
        while B * N * (H + Hkv) * d > 32 * 1025 * 24 * 64:
            N = N // 2
        return _rope("", B, N, H, Hkv, d, rng.choice([1, 2, 2, 3]), rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.8,
                     rng.random() < 0.3, rng.choice([0, 0, 1000, 1000000]), rng.random() < 0.3, rng.random() < 0.6)
    if op == "attention_rope":
        side, H = rng.randint(3, 40), rng.choice([1, 3, 6, 8, 12])
        B = _log(rng, 1, 64)
        while B > 1 and B * H * (side * side + 1) ** 2 * 64 > 32 * 12 * 577 * 577 * 64:
            B = B // 2
        while B * H * (side * side + 1) ** 2 * 64 > 32 * 12 * 577 * 577 * 64:
            side -= 1
        return _block("", B, side, H, rng.random() < 0.8, rng.random() < 0.7)
    width, layers = 8 * _log(rng, 8, 128), rng.randint(1, 12)
    return _adamw("", width, layers, rng.choice([8, 32]), rng.choice(["fp32", "fp32", "bf16"]), rng.randint(10, 1000), rng.randint(17, 1025))


# ------------------------------------------------------------------------------------------------------------------ the inputs
def _lens(case):
    """Lengths of a padded batch, evenly from an empty sample to a full one (all full if there is one sample)."""
    B = case["B"]
    kv = [case["Nk"] if B == 1 else case["Nk"] * b // (B - 1) for b in range(B)]
    return (kv if case["Nq"] == case["Nk"] else None), kv


def _axes_of(d, axes):
    """Pairs of each axis: d / 2 in nearly equal parts."""
    return [d // 2 // axes + (1 if a < d // 2 % axes else 0) for a in range(axes)]


def _inv_freq(sections, base=100.0 ** 2):
    return torch.cat([base ** (-torch.arange(s, dtype=torch.float64) / s) for s in sections]).float().cuda()


def _grid_positions(N, axes, far, B, per_batch, gen):
    """Token n at its place in a grid of `axes` axes, offset by up to `far` (another offset for each sample if per_batch)."""
    n = torch.arange(N, device="cuda")
    side = max(1, math.ceil(N ** (1 / axes)))
    pos = torch.stack([(n // side ** (axes - 1 - a)) % (side if a else N + 1) for a in range(axes)], -1)
    if per_batch:
        return pos + torch.randint(0, far + 1, (B, 1, axes), device="cuda", generator=gen)
    return pos + far


def _adamw_sizes(case):
    """[(shape, decayed)] of a transformer of this width."""
    w, out = case["width"], []
    for _ in range(case["layers"]):
        out += [((3 * w, w), True), ((3 * w,), False), ((w, w), True), ((w,), False), ((4 * w, w), True), ((4 * w,), False),
                ((w, 4 * w), True), ((w,), False)] + [((w,), False)] * 4
    return out + [((1, 1, w), True), ((1, case["tokens"], w), True), ((case["classes"], w), True), ((case["classes"],), False),
                  ((7, 13), True), ((5,), False)]


def _adamw_parts(case):
    """{bits of the state: [shapes without decay, shapes with decay]}."""
    parts = {32: [[], []], 8: [[], []]}
    for shape, decayed in _adamw_sizes(case):
        parts[8 if case["bits"] == 8 and math.prod(shape) >= SMALL else 32][decayed].append(shape)
    return parts


def _padded(shape):
    return -(-math.prod(shape) // BLOCK) * BLOCK


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "mha":
        B, Nq, Nk, H, Hkv, d = (case[k] for k in ("B", "Nq", "Nk", "H", "Hkv", "d"))
        dt = DTYPES[case["dtype"]]
        if case["layout"] == "packed":          # views of one projection's output
            qkv = randn(B, Nq, H + 2 * Hkv, d, dtype=dt)
            q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hkv], qkv[:, :, H + Hkv:]
        elif case["layout"] == "tokens":        # [B, N, H, d], each its own
            q, k, v = (randn(B, n, h, d, dtype=dt) for n, h in ((Nq, H), (Nk, Hkv), (Nk, Hkv)))
        else:                                   # [B, H, N, d] as a cache lies, seen as [B, N, H, d]
            q, k, v = (randn(B, h, n, d, dtype=dt).transpose(1, 2) for n, h in ((Nq, H), (Nk, Hkv), (Nk, Hkv)))
        s["q"], s["k"], s["v"] = (t.detach().requires_grad_(case["train"]) for t in (q, k, v))
        s["q_lens"] = s["kv_lens"] = None
        if case["lens"]:
            ql, kl = (None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in _lens(case))
            s["q_lens"], s["kv_lens"] = ql, kl
        if case["train"]:
            s["dout"] = randn(B, Nq, H, d, dtype=dt)
    elif case["op"] == "rope":
        B, N, H, Hkv, d = (case[k] for k in ("B", "N", "H", "Hkv", "d"))
        dt = DTYPES[case["dtype"]]
        qkv = randn(B, N, H + 2 * Hkv, d, dtype=dt)         # q and k lie in a packed projection
        s["q"], s["k"] = (t.detach().requires_grad_(case["train"]) for t in (qkv[:, :, :H], qkv[:, :, H:H + Hkv]))
        s["sections"] = _axes_of(d, case["axes"])
        s["inv_freq"] = _inv_freq(s["sections"])
        s["positions"] = _grid_positions(N, case["axes"], case["far"], B, case["per_batch"], gen)
        s["wq"] = s["wk"] = None
        if case["norm"]:
            s["wq"], s["wk"] = (((1 + 0.1 * randn(d))).requires_grad_(case["train"]) for _ in range(2))
        if case["train"]:
            s["dq"], s["dk"] = randn(B, N, H, d, dtype=dt), randn(B, N, Hkv, d, dtype=dt)
    elif case["op"] == "attention_rope":
        B, N, H, d = (case[k] for k in ("B", "N", "H", "d"))
        s["qkv"] = randn(B, N, 3 * H * d, dtype=torch.bfloat16).requires_grad_(case["train"])
        s["sections"] = _axes_of(d, 2)
        s["inv_freq"] = _inv_freq(s["sections"])
        side = case["side"]                                 # the class token at the origin, the patches from (1, 1) on
        n = torch.arange(side * side, device="cuda")
        s["positions"] = torch.cat([torch.zeros(1, 2, dtype=n.dtype, device="cuda"), torch.stack([n // side, n % side], -1) + 1])
        s["wq"] = s["wk"] = None
        if case["norm"]:
            # a model cast to bfloat16: its weights' gradients come out of a chain of such activations
            s["wq"], s["wk"] = (((1 + 0.1 * randn(d)).to(torch.bfloat16)).requires_grad_(case["train"]) for _ in range(2))
        if case["train"]:
            s["dout"] = randn(B, N, H * d, dtype=torch.bfloat16)
    else:
        dt = DTYPES[case["dtype"]]
        s["parts"] = {}
        for bits, (plain, decayed) in _adamw_parts(case).items():
            shapes = plain + decayed
            if not shapes:
                continue
            n = sum(_padded(x) for x in shapes)
            real = torch.zeros(n, dtype=torch.bool, device="cuda")
            tensor_scale, at, spots = torch.zeros(n, device="cuda"), 0, []
            scales = torch.rand(len(shapes), device="cuda", generator=gen) * 4 - 6
            for i, x in enumerate(shapes):
                size = math.prod(x)
                real[at:at + size] = True
                tensor_scale[at:at + size] = scales[i]
                spots.append((at, x))
                at += _padded(x)
            size = torch.pow(10.0, tensor_scale) * real     # gradients of 1e-6 to 1e-2, another size for each tensor
            part = {"p": (randn(n, scale=0.02) * real).to(dt), "g": (randn(n) * size).to(dt), "spots": spots,
                    "split": sum(_padded(x) for x in plain), "plain": len(plain)}
            m, r = randn(n) * size * 0.3, (0.5 + torch.rand(n, device="cuda", generator=gen)) * size
            if bits == 32:
                part["m"], part["v"] = m, r * r
            else:
                part["mc"], part["ms"] = _encode(m, 3, True)
                part["vc"], part["vs"] = _encode(r, 4, False)
            s["parts"][bits] = part
        s["t"] = STEP
        if own:
            _optimizer(s)
    return s


def _optimizer(s):
    """The optimizer that a training program keeps, over parameters that lie where prepare() put them."""
    from revisiting_at_amd import optim
    groups, states = [[], []], [[], []]
    for bits, part in s["parts"].items():
        for i, (at, shape) in enumerate(part["spots"]):
            n = math.prod(shape)
            p = torch.nn.Parameter(part["p"][at:at + n].view(shape))
            p.grad = part["g"][at:at + n].view(shape)
            which = int(i >= part["plain"])
            groups[which].append(p)
            step = torch.tensor(float(STEP))
            if bits == 32:
                states[which].append({"step": step, "exp_avg": part["m"][at:at + n].view(shape), "exp_avg_sq": part["v"][at:at + n].view(shape)})
            else:
                a, b, e = at // BLOCK, (at + _padded(shape)) // BLOCK, at + _padded(shape)
                states[which].append({"step": step, "exp_avg_codes": part["mc"][at:e], "exp_avg_scales": part["ms"][a:b],
                                      "exp_avg_sq_codes": part["vc"][at:e], "exp_avg_sq_scales": part["vs"][a:b]})
    opt = optim.FusedAdamW([{"params": groups[0], "weight_decay": 0.0}, {"params": groups[1], "weight_decay": DECAY}], lr=LR, betas=BETAS,
                           eps=EPS, state_bits=s["case"]["bits"])
    sd = opt.state_dict()
    sd["state"] = dict(enumerate(states[0] + states[1]))
    opt.load_state_dict(sd)
    s["optimizer"] = opt


# ------------------------------------------------------------------------------------------------------------------ the plain forms
def _allowed(case, q_lens, kv_lens):
    """[B, 1, 1, Nq, Nk] truth values: which keys a query sees (None: all)."""
    B, Nq, Nk = case["B"], case["Nq"], case["Nk"]
    if not case["causal"] and not case["lens"]:
        return None
    i = torch.arange(Nq, device="cuda").view(1, Nq, 1)
    j = torch.arange(Nk, device="cuda").view(1, 1, Nk)
    ql = torch.full((B,), Nq, device="cuda") if q_lens is None else q_lens
    kl = torch.full((B,), Nk, device="cuda") if kv_lens is None else kv_lens
    ql, kl = ql.view(B, 1, 1), kl.view(B, 1, 1)
    ok = (i < ql) & (j < kl)
    if case["causal"]:
        ok = ok & (j <= i + (kl - ql))          # the last query sees the last key
    return ok.view(B, 1, 1, Nq, Nk)


def _plain_attention(q, k, v, scale, allowed, dout=None):
    """q [B, N, H, d], k, v [B, N, Hkv, d] in 32 bits -> out, and the gradients where dout is given."""
    B, Nq, H, d = q.shape
    Hkv = k.shape[2]
    G = H // Hkv
    rows = lambda t: t.reshape(B, Nq, Hkv, G, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Nq, d)     # noqa: E731
    back = lambda t: t.reshape(B, Hkv, G, Nq, d).permute(0, 3, 1, 2, 4).reshape(B, Nq, H, d)           # noqa: E731
    qr, kh, vh = rows(q), k.transpose(1, 2), v.transpose(1, 2)
    p = torch.matmul(qr, kh.transpose(-2, -1)).mul_(scale).view(B, Hkv, G, Nq, -1)
    if allowed is not None:
        p = p.masked_fill_(~allowed, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total)).view(B, Hkv, G * Nq, -1)
    out = torch.matmul(p, vh)
    if dout is None:
        return back(out)
    do = rows(dout)
    dv = torch.matmul(p.transpose(-2, -1), do)
    ds = torch.matmul(do, vh.transpose(-2, -1)).sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, kh), torch.matmul(ds.transpose(-2, -1), qr)
    return back(out), back(dq), dk.transpose(1, 2), dv.transpose(1, 2)


def _turn(x, cos, sin, interleaved):
    """Rotates the pairs of the last axis: (i, i + d/2), or (2i, 2i + 1)."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _cos_sin(positions, inv_freq, sections):
    """[(B,) N, 1, d / 2] cosines and sines; the angles in 64 bits."""
    axis = torch.repeat_interleave(torch.arange(len(sections), device="cuda"), torch.tensor(sections, device="cuda"), output_size=sum(sections))
    angle = (positions.double()[..., axis] * inv_freq.double()).unsqueeze(-2)
    return angle.cos().float(), angle.sin().float()


def _plain_norm_turn(x, w, cos, sin, interleaved, eps=1e-6):
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
    return _turn(x, cos, sin, interleaved)


def _plain_norm_turn_back(dy, x, w, cos, sin, interleaved, eps=1e-6):
    """(dx, dw)."""
    dz = _turn(dy, cos, -sin, interleaved)
    if w is None:
        return dz, None
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    xh = x * r
    dw = (dz * xh).sum((0, 1, 2))
    dz = dz * w
    return r * (dz - xh * (dz * xh).mean(-1, keepdim=True)), dw


def _decode(codes, scales, bits, signed):
    """Values of 8-bit codes: a zero, or the top of a 32-bit number's exponent and `bits` of its mantissa, 1.0 the largest; times the scale."""
    top, shift = (127, 20) if signed else (255, 19)
    c = codes.to(torch.int32)
    mag = (c & 127) if signed else c
    one = 0x3F800000 >> shift
    x = ((mag + (one - top)) << shift).view(torch.float32) * (mag > 0)
    if signed:
        x = torch.where(c > 127, -x, x)
    return (x.view(-1, BLOCK) * scales.view(-1, 1)).view(-1)


def _encode(x, bits, signed):
    """(codes, scales) of a flat tensor in blocks of 256: nearest, ties to even; a number other than zero keeps at least the smallest
    code where it has no sign (it is divided by)."""
    top, shift = (127, 20) if signed else (255, 19)
    x = x.view(-1, BLOCK)
    scales = x.abs().amax(1)
    scales = torch.where(scales < 2.0 ** -126, 0.0, scales)
    inv = torch.where(scales > 0, 1.0 / scales, 0.0)
    b = (x.abs() * inv.view(-1, 1)).view(torch.int32)
    b = (b + ((1 << (shift - 1)) - 1) + ((b >> shift) & 1)) >> shift
    c = (b - ((0x3F800000 >> shift) - top)).clamp(0, top)
    if signed:
        c = c | ((x < 0).to(torch.int32) << 7)
    else:
        c = torch.where((x > 0) & (scales > 0).view(-1, 1), c.clamp(min=1), c)
    return c.to(torch.uint8).view(-1), scales


def _plain_adamw(s):
    t = s["t"] = s["t"] + 1
    b1, b2 = BETAS
    out = []
    for bits, part in s["parts"].items():
        m = part["m"] if bits == 32 else _decode(part["mc"], part["ms"], 3, True)
        r = None if bits == 32 else _decode(part["vc"], part["vs"], 4, False)
        v = part["v"] if bits == 32 else r * r
        g = part["g"].float()
        m.mul_(b1).add_(g * (1 - b1))
        v.mul_(b2).add_((g * g) * (1 - b2))
        r = v.sqrt()
        move = m / (r * (1 / math.sqrt(1 - b2 ** t)) + EPS) * (LR / (1 - b1 ** t))
        p = part["p"].float()
        k = part["split"]
        p[k:] *= 1 - LR * DECAY                 # (in place where p is the parameters themselves)
        part["p"].copy_(p - move)
        if bits == 32:
            out += [part["p"], m, v]
        else:
            part["mc"], part["ms"] = _encode(m, 3, True)
            part["vc"], part["vs"] = _encode(r, 4, False)
            r = _decode(part["vc"], part["vs"], 4, False)
            # an 8-bit moment has 4 or 5 significant bits: bfloat16 holds what it stands for
            out += [part["p"], _decode(part["mc"], part["ms"], 3, True).to(torch.bfloat16), (r * r).to(torch.bfloat16)]
    return out


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    return {"mha": _run_mha, "rope": _run_rope, "attention_rope": _run_block, "adamw": _run_adamw}[case["op"]](s, case)


def _run_mha(s, case):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        from revisiting_at_amd import ops
        out = ops.mha(q, k, v, causal=case["causal"], q_lens=s["q_lens"], kv_lens=s["kv_lens"])
        if not case["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), s["dout"])
    with torch.no_grad():
        r = _plain_attention(q.float(), k.float(), v.float(), case["d"] ** -0.5, _allowed(case, s["q_lens"], s["kv_lens"]),
                             s["dout"].float() if case["train"] else None)
        return tuple(t.to(q.dtype) for t in r) if case["train"] else r.to(q.dtype)


def _run_rope(s, case):
    q, k, wq, wk = s["q"], s["k"], s["wq"], s["wk"]
    if own:
        from revisiting_at_amd import ops
        yq, yk = ops.qk_norm_rope(q, k, wq, wk, s["positions"], s["inv_freq"], s["sections"], norm=case["norm"], interleaved=case["interleaved"])
        if not case["train"]:
            return yq, yk
        return (yq.detach(), yk.detach()) + torch.autograd.grad((yq, yk), (q, k) + ((wq, wk) if case["norm"] else ()), (s["dq"], s["dk"]))
    with torch.no_grad():
        cos, sin = _cos_sin(s["positions"], s["inv_freq"], s["sections"])
        x = (q.float(), k.float())
        y = [_plain_norm_turn(t, w, cos, sin, case["interleaved"]).to(q.dtype) for t, w in zip(x, (wq, wk))]
        if not case["train"]:
            return tuple(y)
        g = [_plain_norm_turn_back(dy.float(), t, w, cos, sin, case["interleaved"]) for dy, t, w in zip((s["dq"], s["dk"]), x, (wq, wk))]
        return tuple(y) + tuple(d[0].to(q.dtype) for d in g) + (tuple(d[1] for d in g) if case["norm"] else ())


def _run_block(s, case):
    qkv, wq, wk, H, d = s["qkv"], s["wq"], s["wk"], case["H"], case["d"]
    if own:
        from revisiting_at_amd import ops
        out = ops.attention_rope(qkv, H, d ** -0.5, wq, wk, s["positions"], s["inv_freq"], s["sections"], norm=case["norm"])
        if not case["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, (qkv,) + ((wq, wk) if case["norm"] else ()), s["dout"])
    with torch.no_grad():
        B, N, _ = qkv.shape
        q, k, v = qkv.float().view(B, N, 3, H, d).unbind(2)
        cos, sin = _cos_sin(s["positions"], s["inv_freq"], s["sections"])
        yq, yk = (_plain_norm_turn(t, w, cos, sin, False) for t, w in ((q, wq), (k, wk)))
        if not case["train"]:
            return _plain_attention(yq, yk, v, d ** -0.5, None).reshape(B, N, H * d).to(qkv.dtype)
        out, dyq, dyk, dv = _plain_attention(yq, yk, v, d ** -0.5, None, s["dout"].float().view(B, N, H, d))
        (dq, dwq), (dk, dwk) = (_plain_norm_turn_back(dy, t, w, cos, sin, False) for dy, t, w in ((dyq, q, wq), (dyk, k, wk)))
        grad = torch.stack((dq, dk, dv), 2).view(B, N, 3 * H * d).to(qkv.dtype)
        return (out.reshape(B, N, H * d).to(qkv.dtype), grad) + ((dwq.to(wq.dtype), dwk.to(wk.dtype)) if case["norm"] else ())


def _run_adamw(s, case):
    if own:
        opt = s["optimizer"]
        opt.step()
        return [t for bits, (m, v) in opt.moments().items() for t in (s["parts"][bits]["p"], m, v)]
    return _plain_adamw(s)


# ------------------------------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """Query-key pairs that are not masked, over the batch."""
    B, Nq, Nk = case["B"], case["Nq"], case["Nk"]
    ql, kl = _lens(case) if case["lens"] else (None, None)
    n = 0
    for b in range(B):
        nq, nk = (Nq if ql is None else ql[b]), (Nk if kl is None else kl[b])
        off = nk - nq
        n += sum(max(0, min(nk, i + off + 1)) for i in range(nq)) if case["causal"] else nq * nk
    return n


def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] == "mha":
        B, Nq, Nk, H, Hkv, d = (case[k] for k in ("B", "Nq", "Nk", "H", "Hkv", "d"))
        q, kv = B * Nq * H * d * size, B * Nk * Hkv * d * size
        n = _pairs(case) * H * d
        if case["train"]:                       # q, k, v, dout in, out and three gradients out; seven products' worth of the minimum
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * n}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * n}
    if case["op"] == "rope":
        n = case["B"] * case["N"] * (case["H"] + case["Hkv"]) * case["d"]
        return {"bytes": n * size * (5 if case["train"] else 2), "flops": n * (24 if case["train"] else 8)}
    if case["op"] == "attention_rope":
        B, N, H, d = (case[k] for k in ("B", "N", "H", "d"))
        c = B * N * H * d
        return {"bytes": 2 * c * (8 if case["train"] else 4), "flops": B * H * N * N * d * (14 if case["train"] else 4)}
    total = 0
    for bits, both in _adamw_parts(case).items():
        n = sum(math.prod(x) for part in both for x in part)
        # parameters in and out, gradients in, two moments in and out (8 bits: their values out once more, 16 bits each)
        total += n * (3 * size + (16 if bits == 32 else 4 * (1 + 4 / BLOCK) + 4))
    return {"bytes": total, "flops": 15 * total / 16}


# ------------------------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_attention(q, k, v, scale, ok):
    """softmax over the allowed keys, one sample [N, H, d] at a time; gradients by autograd."""
    G = q.shape[1] // k.shape[1]
    sc = torch.einsum("ihd,jhd->hij", q * scale, k.repeat_interleave(G, 1))
    if ok is not None:
        sc = sc.masked_fill(~ok, -1e300)
    e = torch.exp(sc - sc.detach().max(-1, keepdim=True).values)
    if ok is not None:
        e = e * ok
    z = e.sum(-1, keepdim=True)
    return torch.einsum("hij,jhd->ihd", e / (z + (z == 0)), v.repeat_interleave(G, 1))


def _exact_rope(x, w, positions, inv_freq, sections, interleaved):
    """As complex numbers: the pair (a, b) is a + ib, turned by exp(i angle)."""
    if w is not None:
        x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + 1e-6) * w
    d = x.shape[-1]
    first, angles = 0, []
    for a, n in enumerate(sections):
        angles.append(positions[..., a:a + 1].double() * inv_freq[first:first + n].double())
        first += n
    angle = torch.cat(angles, -1).unsqueeze(-2)
    pairs = x.unflatten(-1, (d // 2, 2)) if interleaved else x.unflatten(-1, (2, d // 2)).transpose(-1, -2)
    z = torch.complex(pairs[..., 0], pairs[..., 1]) * torch.polar(torch.ones_like(angle), angle)
    z = torch.stack((z.real, z.imag), -1)
    return z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda t: None if t is None else t.detach().double().requires_grad_(t.requires_grad)        # noqa: E731
    if case["op"] == "mha":
        got, allowed = [], _allowed(case, s["q_lens"], s["kv_lens"])
        for b in range(case["B"]):
            x = [wide(s[n][b]) for n in "qkv"]
            x = [t.detach().requires_grad_(case["train"]) for t in x]
            ok = None if allowed is None else allowed[b if allowed.shape[0] > 1 else 0, 0]
            out = _exact_attention(*x, case["d"] ** -0.5, ok)
            got.append([out.detach()] + (list(torch.autograd.grad(out, x, s["dout"][b].double())) if case["train"] else []))
            del out
        got = [torch.stack(t) for t in zip(*got)]
        return tuple(got) if case["train"] else got[0]
    if case["op"] == "rope":
        q, k, wq, wk = (wide(s[n]) for n in ("q", "k", "wq", "wk"))
        y = [_exact_rope(x, w, s["positions"], s["inv_freq"], s["sections"], case["interleaved"]) for x, w in ((q, wq), (k, wk))]
        if not case["train"]:
            return tuple(y)
        leaves = (q, k) + ((wq, wk) if case["norm"] else ())
        return tuple(t.detach() for t in y) + torch.autograd.grad(y, leaves, (s["dq"].double(), s["dk"].double()))
    if case["op"] == "attention_rope":
        B, N, H, d = (case[k] for k in ("B", "N", "H", "d"))
        wq, wk = wide(s["wq"]), wide(s["wk"])
        outs, grads, dw = [], [], 0
        for b in range(B):
            x = s["qkv"][b].detach().double().requires_grad_(case["train"])
            q, k, v = x.view(N, 3, H, d).unbind(1)
            q, k = (_exact_rope(t, w, s["positions"], s["inv_freq"], s["sections"], False) for t, w in ((q, wq), (k, wk)))
            out = _exact_attention(q, k, v, d ** -0.5, None).reshape(N, H * d)
            outs.append(out.detach())
            if case["train"]:
                g = torch.autograd.grad(out, (x,) + ((wq, wk) if case["norm"] else ()), s["dout"][b].double())
                grads.append(g[0])
                dw = [a + b_ for a, b_ in zip(dw, g[1:])] if b else list(g[1:])
            del out
        if not case["train"]:
            return torch.stack(outs)
        return (torch.stack(outs), torch.stack(grads)) + tuple(dw)
    b1, b2 = BETAS
    t, got = STEP + 1, []
    for bits, part in s["parts"].items():
        p, g = part["p"].double(), part["g"].double()
        if bits == 32:
            m, v = part["m"].double(), part["v"].double()
        else:
            m = _exact_value(part["mc"], 8, 127) * part["ms"].double().repeat_interleave(BLOCK)
            v = (_exact_value(part["vc"], 16, 255) * part["vs"].double().repeat_interleave(BLOCK)) ** 2
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        decay = torch.ones_like(p)
        decay[part["split"]:] = 1 - LR * DECAY
        got.append(p * decay - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS))
        if bits == 32:
            got += [m, v]
        else:
            got += [_exact_round(m, 8, 127, False), _exact_round(v.sqrt(), 16, 255, True) ** 2]
    return got


def _exact_value(codes, steps, top):
    """Code c > 0 is (1 + f / steps) * 2^e with c = top + f + steps * e; for the signed one the eighth bit is the sign."""
    c = codes.long()
    sign = torch.where(c > 127, -1.0, 1.0).double() if top == 127 else 1.0
    c = c & 127 if top == 127 else c
    e, f = torch.div(c - top, steps, rounding_mode="floor"), torch.remainder(c - top, steps)
    return sign * torch.where(c > 0, torch.ldexp(1 + f.double() / steps, e), 0.0)


def _exact_round(x, steps, top, keep):
    """x to the nearest value of an 8-bit state, block by block."""
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1, keepdim=True)
    y = x.abs() / torch.where(scale > 0, scale, 1.0)
    e = torch.floor(torch.log2(torch.where(y > 0, y, 1.0)))
    f = torch.round((y / 2.0 ** e - 1) * steps)
    c = torch.where(y > 0, top + f + steps * e, 0.0).clamp(0, top)
    if keep:
        c = torch.where(y > 0, c.clamp(min=1), c)
    c = c.long()
    value = _exact_value(c, steps, 255 if top == 255 else 127)
    return (torch.sign(x) * value.view_as(x) * scale).view(-1)
