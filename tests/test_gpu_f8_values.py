"""The fp8 operators on values where a form may go wrong alone: codes that are NaN, columns far below their neighbours, values
on the border between two codes, gates at the ends of fp32. Each case in every form of the experts: the direct one and the row
tiles of 32, 64, 128 and 192."""
import numpy as np
import pytest

from oracle import f8 as of

pytestmark = pytest.mark.gpu
# tokens of one of four experts each: the direct form, then 20, 40, 150 and 250 mean rows an expert
TOKENS = (3, 80, 160, 600, 1000)


def _codes_dev(dev, q):
    import torch
    return torch.from_numpy(np.ascontiguousarray(q)).to(dev).view(torch.float8_e4m3fn)


def _layer(dev, E, H, I, seed):
    """Random experts: what the oracle takes and what the call takes."""
    import torch
    r = np.random.default_rng(seed)
    hb, ib = of.blocks(H), of.blocks(I)
    gq = of.codes_of(np.clip(r.standard_normal((E, 2 * I, hb * 128)) * 100, -448, 448))
    dq = of.codes_of(np.clip(r.standard_normal((E, H, ib * 128)) * 100, -448, 448))
    gq[..., H:], dq[..., I:] = 0, 0
    gs, ds = (r.uniform(1e-4, 3e-4, s).astype(np.float32) for s in ((E, 2 * ib, hb), (E, hb, ib)))
    return gq, gs, dq, ds, [torch.from_numpy(s).to(dev) for s in (gs, ds)]


def _routing(dev, T, E, k, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    w, ids = torch.topk(torch.softmax(torch.randn(T, E, generator=g), -1), k, -1)
    return w.to(dev), ids.to(dev)


def _np(t):
    import torch
    return t.detach().to(torch.float64).cpu().numpy()


@pytest.mark.parametrize("T", TOKENS)
def test_nan_codes_spoil_what_they_are_part_of(dev, T):
    """A NaN code of a down weight makes its column NaN for the tokens that its expert serves, one of a gate or up weight the
    whole of those tokens; every other output is what it is without them."""
    import torch
    from infinitemodel_amd import ops
    E, H, I, k = 4, 300, 256, 1
    gq, gs, dq, ds, (gst, dst) = _layer(dev, E, H, I, seed=T)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(dev)
    w, ids = _routing(dev, T, E, k, seed=T)
    want, tol = of.experts(of.dequantize(*of.quantize(_np(x))), ids.cpu().numpy(), w.cpu().numpy(), (gq, gs), (dq, ds), H, I)
    mine = _np(ids)[:, 0].astype(int)
    e = int(mine[0])
    for place in ("down", "gate", "up"):
        g, d = gq.copy(), dq.copy()
        bad = np.zeros((T, H), dtype=bool)
        if place == "down":
            d[e, 1, 5], d[e, 130, 255], d[e, 299, 0] = 0x7f, 0xff, 0x7f
            bad[:, [1, 130, 299]] = (mine == e)[:, None]
        else:
            g[e, 7 if place == "gate" else I + 200, 3] = 0x7f
            bad[mine == e] = True
        out = _np(ops.moe_experts_f8(x, ids, w, (_codes_dev(dev, g), gst, H), (_codes_dev(dev, d), dst, I)))
        np.testing.assert_array_equal(np.isnan(out), bad)
        assert (np.abs(out - want) <= tol)[~bad].all(), place


@pytest.mark.parametrize("T", TOKENS)
def test_columns_far_below_their_neighbours(dev, T):
    """A column 2^-36 of the one beside it comes out as exact as that one: h holds 448 and 2^-9, and each output is one product of
    a code of down with one of them."""
    import torch
    from infinitemodel_amd import ops
    E, H, I = 4, 128, 128
    one, gate = of.codes_of(np.array([1.0, 64.0]))
    gq, dq = np.zeros((E, 2 * I, 128), np.uint8), np.zeros((E, H, 128), np.uint8)
    gq[:, :I, 1] = gate                                       # g = 64 at every column: silu(64) is 64 in fp32
    gq[:, I, 1], gq[:, I + 1, 1] = of.codes_of(np.array([448.0, 2.0 ** -9]))
    dq[:, 0, 0] = of.codes_of(np.array(448.0))
    dq[:, 1:, 1] = np.arange(1, H)                            # every magnitude from 2^-9 on
    s = torch.ones(E, 2, 1, device=dev), torch.ones(E, 1, 1, device=dev)
    x = torch.zeros(T, H)
    x[:, 0], x[:, 1] = 448.0, 1.0                             # scale 1
    ids = (torch.arange(T) % E)[:, None].to(dev)
    dq[:, 127, 1] = one
    out = ops.moe_experts_f8(x.to(dev), ids, torch.ones(T, 1, device=dev), (_codes_dev(dev, gq), s[0], H), (_codes_dev(dev, dq), s[1], I))
    want = 64 * of.values_of(dq[0, :, 1]) * 2.0 ** -9
    want[0] = 64 * 448.0 * 448.0
    np.testing.assert_array_equal(_np(out), np.tile(want, (T, 1)))


@pytest.mark.parametrize("T", TOKENS)
def test_h_on_the_border_of_two_codes(dev, T):
    """h's codes are e4m3 of the exact quotient, in every form: values halfway between two codes, at scales whose rounded
    reciprocal would put some of them on the other side."""
    import torch
    from infinitemodel_amd import ops
    E, H, I = 4, 128, 128
    mids = of.MIDS[(of.MIDS >= 17) & (of.MIDS == np.round(of.MIDS))]
    gq, dq, want = np.zeros((E, 2 * I, 128), np.uint8), np.zeros((E, H, 128), np.uint8), np.zeros((E, H))
    gq[:, :I, 1] = of.codes_of(np.array(64.0))               # g = 64: silu(g) u is 64 u in fp32
    dq[:, np.arange(I), np.arange(I)] = of.codes_of(np.array(1.0))
    for e, j in enumerate((7, 15, 61, 126)):                  # the block's scale is 64 j
        u = np.zeros(I, dtype=np.int64)
        u[0], u[1:1 + len(mids)] = 448 * j, mids * j
        digits = [u >> 12 & 15, u >> 8 & 15, u >> 4 & 15, u & 15]          # times 4096, 256, 16, 1
        for col, d in enumerate(digits):
            gq[e, I:, 2 + col] = of.codes_of(d * (16.0 if col == 0 else 1.0))
        h = 64.0 * u
        s = np.float32(64 * j)
        codes = of.codes_of(h / np.float64(s))
        assert (codes != of.codes_of((h.astype(np.float32) * (np.float32(1) / s)).astype(np.float64))).any()
        want[e] = of.values_of(codes) * 64 * j
    s = torch.ones(E, 2, 1, device=dev), torch.ones(E, 1, 1, device=dev)
    x = torch.zeros(T, H)
    x[:, 0] = 448.0                                           # scale 1
    x[:, 1:6] = torch.tensor([1.0, 256.0, 256.0, 16.0, 1.0])
    ids = torch.arange(T) % E
    out = ops.moe_experts_f8(x.to(dev), ids[:, None].to(dev), torch.ones(T, 1, device=dev), (_codes_dev(dev, gq), s[0], H),
                             (_codes_dev(dev, dq), s[1], I))
    w = want[ids.numpy()]
    assert (np.abs(_np(out) - w) <= 2.0 ** -8 * w).all()       # bf16's rounding; the next code is 2^-4 away


@pytest.mark.parametrize("T", TOKENS)
def test_gates_at_the_ends_of_fp32(dev, T):
    """silu of gates up to 3e38 of either sign, beside an ordinary one in the same block of h: g itself or 0, and never NaN."""
    import torch
    from infinitemodel_amd import ops
    E, H, I = 4, 256, 128
    sizes = [2.0 ** 119, 2.0 ** 60, 1.0, 0.125]               # of each expert's gate, in the first 128 columns
    codes = np.array([448.0, 256.0, 1.0, 2.0 ** -9])
    gq, dq = np.zeros((E, 2 * I, 256), np.uint8), np.zeros((E, H, 128), np.uint8)
    gq[:, :4, 1] = of.codes_of(codes)
    gq[:, 4, 129] = of.codes_of(np.array(64.0))
    gq[:, I:I + 4, 129] = of.codes_of(np.array(2.0 ** -9))
    gq[:, I + 4, 129] = of.codes_of(np.array(1.0))
    dq[:, np.arange(5), np.arange(5)] = of.codes_of(np.array(1.0))
    gs = np.ones((E, 2, 2), np.float32)
    gs[:, 0, 0] = sizes
    x = torch.zeros(T, H)
    x[:, [0, 128]] = 448.0                                    # scale 1
    sign = torch.where(torch.arange(T) % 8 < 4, 1.0, -1.0) if T > 4 else torch.tensor([1.0, -1.0, 1.0])
    x[:, 1], x[:, 129] = sign, 1.0
    ids = torch.arange(T) % E if T > 4 else torch.zeros(T, dtype=torch.int64)
    out = _np(ops.moe_experts_f8(x.to(dev), ids[:, None].to(dev), torch.ones(T, 1, device=dev),
                                 (_codes_dev(dev, gq), torch.from_numpy(gs).to(dev), H), (_codes_dev(dev, dq), torch.ones(E, 2, 1, device=dev), I)))
    g = sign.double().numpy()[:, None] * np.array(sizes)[ids.numpy()][:, None] * codes
    h = np.zeros((T, I))
    h[:, :4] = np.where(g < -700, 0.0, g / (1 + np.exp(-np.maximum(g, -700)))) * 2.0 ** -9
    h[:, 4] = 64.0
    q, s = of.quantize(h)
    near = np.abs(h / s.astype(np.float64))[:, :5, None] / of.MIDS - 1
    assert np.abs(near).min() > 1e-4                          # no value where fp32's errors would choose the code
    want = of.dequantize(q, s)[:, :5]
    assert (np.abs(out[:, :5] - want) <= 2.0 ** -8 * np.abs(want)).all()
    assert not out[:, 5:].any()
