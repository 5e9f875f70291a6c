"""``optim.FusedAdamW`` on a machine without a GPU: the 8-bit moments outside the kernel, written out code by code, and their memory order."""
import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def O():
    import revisiting_at_amd as R
    return R.optim


# value of every code: 3 (4) mantissa bits counting down from 1.0
VALUES = {"exp_avg": np.array([0.0] + [(1 + (c - 127) % 8 / 8) * 2.0 ** ((c - 127) // 8) for c in range(1, 128)]),
          "exp_avg_sq": np.array([0.0] + [(1 + (c - 255) % 16 / 16) * 2.0 ** ((c - 255) // 16) for c in range(1, 256)])}


@pytest.mark.parametrize("kind", ["exp_avg", "exp_avg_sq"])
def test_codes_outside_the_kernel(O, kind):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(256 * 60, generator=g) * 10.0 ** (torch.rand(256 * 60, generator=g) * 8 - 6)
    x = x if kind == "exp_avg" else x.abs()
    x[256:512], x[600], x[1024:1280] = 0, 0, 1e-40                                  # a block of zeros; one too small to be divided by
    codes, scales = O._encode(x, kind)
    top = x.abs().view(-1, 256).amax(1)
    assert torch.equal(scales, torch.where(top < 2.0 ** -126, 0.0, top))
    low = codes.numpy().astype(np.int64) & (127 if kind == "exp_avg" else 255)
    val, mant = VALUES[kind], 8 if kind == "exp_avg" else 16
    back = O._decode(codes, scales, kind)
    size = scales.repeat_interleave(256)
    assert np.array_equal(back.numpy(), (val[low].astype(np.float32) * size.numpy()) * np.where(codes.numpy() > low, -1, 1).astype(np.float32))
    # nearest: a code's step is that of the binade of x / scale, so half of it times the scale (the quotient itself is 2^-23 off); below the smallest
    # code zero from half a step beneath it on
    x64, s64 = x.abs().double().numpy(), size.double().numpy()
    off = np.abs(back.abs().double().numpy() - x64)
    small = (x64 < val[1] * s64) | (s64 == 0)
    step = 2.0 ** np.floor(np.log2(x64[~small] / s64[~small])) / mant * s64[~small]
    assert (off[~small] <= step / 2 + 2.0 ** -22 * x64[~small]).all()
    assert (off[small] <= np.where(s64[small] == 0, 2.0 ** -126, val[1] * s64[small])).all()      # (no scale: all of a value below 2^-126)
    if kind == "exp_avg_sq":
        assert ((back > 0) == ((x > 0) & (size > 0))).all()
    else:
        assert torch.equal(codes > 127, x < 0)
    again = O._encode(back, kind)                                                   # what a code stands for is its own nearest code
    assert torch.equal(again[1], scales) and torch.equal(O._decode(*again, kind), back)


def test_a_block_that_is_not_finite_stays_so(O):
    for bad in (float("nan"), float("inf")):
        x = torch.ones(512)
        x[3] = bad
        for kind in ("exp_avg", "exp_avg_sq"):
            back = O._decode(*O._encode(x, kind), kind)
            assert not bool(torch.isfinite(back[:256]).any()) and bool((back[256:] == 1).all())


def test_memory_orders(O):
    x = torch.zeros(4, 5, 6, 7)
    assert O._order(x) == O._order(torch.zeros(3)) == O._order(torch.zeros(())) == ()
    assert O._order(x.to(memory_format=torch.channels_last)) == (0, 2, 3, 1)
    assert O._order(torch.zeros(4, 1, 6, 7).to(memory_format=torch.channels_last)) == () and O._order(torch.zeros(5, 4).t()) == (1, 0)


def test_moments_are_brought_into_another_order(O):
    g = torch.Generator().manual_seed(1)
    shape = (8, 12, 5, 9)                                                           # 4320 elements: a last block of 224
    n, pad = 4320, 4352
    m, r = torch.randn(n, generator=g), torch.rand(n, generator=g) + 0.5
    for formats in ((torch.contiguous_format, torch.channels_last), (torch.channels_last, torch.contiguous_format)):
        old, new = (torch.empty(shape).to(memory_format=f) for f in formats)
        state = {"step": torch.tensor(3.0), "exp_avg_order": torch.tensor(O._order(old))}
        for kind, x in (("exp_avg", m), ("exp_avg_sq", r)):
            state[kind + "_codes"], state[kind + "_scales"] = O._encode(torch.nn.functional.pad(x, (0, pad - n)), kind)
        assert O._reorder(state, old) is state
        out = O._reorder(state, new)
        assert float(out["step"]) == 3
        for kind, bits in (("exp_avg", 4), ("exp_avg_sq", 5)):
            a, b = (O._decode(s[kind + "_codes"], s[kind + "_scales"], kind) for s in (state, out))
            a, b = a[:n].as_strided(shape, old.stride()), b[:n].as_strided(shape, new.stride())
            # one more rounding, half a step of a code: 2^-bits of the value at most; of m below its smallest code up to 1.1875 2^-16 of the scale
            assert bool(((a - b).abs() <= a.abs() * 2.0 ** -bits * 1.001 + (4.0 * 2.0 ** -15 if kind == "exp_avg" else 0)).all())
        assert not bool(O._decode(out["exp_avg_codes"], out["exp_avg_scales"], "exp_avg")[n:].any())
