"""Every form of the fp8 linear and of the experts at least once, each case held to the form it is meant for by the dispatcher's own
plan: all tiles, with and without K ranges, more tiles than workgroups that run at once; the few-row kernel's ways to its rows;
the experts' row tiles with more of them than workgroups, over odd and even numbers of steps."""
import numpy as np
import pytest

from oracle import f8 as of

pytestmark = pytest.mark.gpu

# M, N, K, x handed over quantized; the plan (weight rows, activation rows, K ranges; few rows: 0, waves, way of the rows)
LINEAR = [(2947, 9596, 645, False, (256, 256, 1)), (393, 9787, 8771, False, (256, 256, 3)), (3728, 6147, 129, False, (128, 128, 1)),
          (264, 6737, 6523, False, (128, 128, 3)), (69, 11162, 7623, True, (128, 128, 5)), (425, 7039, 263, False, (128, 64, 1)),
          (4715, 198, 5581, False, (128, 64, 3)), (5677, 130, 389, True, (64, 64, 1)), (36, 5571, 4294, False, (64, 64, 5)),
          (17, 68, 135, False, (64, 32, 1)), (17, 66, 4623, False, (64, 32, 8)),
          (3, 100, 700, False, (0, 4, 1)), (3, 100, 2000, False, (0, 8, 1)), (2, 100, 7000, False, (0, 16, 1)),
          (16, 100, 1400, False, (0, 4, 0)), (9, 4096, 2100, False, (0, 8, 0)), (3, 100, 14336, False, (0, 16, 0)),
          (1, 333, 1024, True, (0, 4, 0)), (9, 8200, 2100, False, (0, 16, 2)), (9, 8200, 2100, True, (0, 16, 2)),
          (16, 9001, 128, True, (0, 16, 2))]
# more tiles than this many workgroups
LOOPS = {(256, 256): 256, (128, 128): 512}


def _plan(kind, *a, **kw):
    import torch
    from infinitemodel_amd import _lib
    return _lib.launch_plan(getattr(_lib, kind), *a, cus=torch.cuda.get_device_properties(0).multi_processor_count, **kw)


def _bytes(dev, shape, seed):
    """Random codes but NaN: every magnitude alike, so sums are led by the large ones."""
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.uint8)
    return torch.where(q & 127 == 127, q - 1, q)


def _values(q, s, rows):
    """What e4m3 codes [M, K_pad] and their scales stand for, in 64 bits."""
    s = s.double().repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(128, 1)
    return q.double() * s


def _bound(xv, wv):
    """of.linear on the device, in 64 bits."""
    y = xv @ wv.t().contiguous()
    gx, gw = (v.abs().unflatten(1, (-1, 8)).amax(2) ** 2 for v in (xv, wv))
    cut = 6 * 2.0 ** -13 * (8 / 3 * (gx @ gw.t().contiguous())).sqrt()
    e = of.sum_slack(xv.shape[1]) * (xv.abs() @ wv.abs().t().contiguous()) + cut
    return y, 2.0 ** -8 * y.abs() + (1 + 2.0 ** -8) * e


@pytest.mark.parametrize("M,N,K,given,plan", LINEAR)
def test_linear_plans(dev, M, N, K, given, plan):
    import torch
    from infinitemodel_amd import _lib, ops
    kp = of.blocks(K) * 128
    assert _plan("IMQ_PLAN_LINEAR_F8", M, kp, 0, N, sdt=_lib.IMQ_DT_F8 if given else _lib.IMQ_DT_BF16)[:3] == plan
    if plan[2] == 1 and plan[:2] in LOOPS:
        assert -(-N // plan[0]) * -(-M // plan[1]) > LOOPS[plan[:2]]
    g = torch.Generator(device=dev).manual_seed(M + N)
    x = torch.randn(M, K, generator=g, device=dev) * torch.exp(0.7 * torch.randn(M, 1, generator=g, device=dev))
    q = torch.randn(N, kp, generator=g, device=dev).mul_(100).clamp_(-448, 448)
    q[:, K:] = 0
    q, s = q.to(torch.float8_e4m3fn), 1e-4 + 2e-4 * torch.rand(of.blocks(N), kp // 128, generator=g, device=dev)
    x = x.to(torch.bfloat16)
    xq, xs = ops.quant_f8(x)
    out = torch.full((M + 2, N + 5), 7.0, dtype=torch.bfloat16, device=dev)
    call = (lambda **kw: ops.linear_f8(xq, q, s, x_scale=xs, **kw)) if given else (lambda **kw: ops.linear_f8(x, q, s, **kw))
    y = call()
    want, tol = _bound(_values(xq, xs, 1), _values(q, s, 128))
    over = (y.double() - want).abs() - tol
    assert bool((over <= 0).all()), (float(over.max()), divmod(int(over.argmax()), N))
    assert torch.equal(y, call(out=out[1:M + 1, 2:N + 2]))   # rows at other addresses, the same bits
    out[1:M + 1, 2:N + 2] = 7.0
    assert bool((out == 7.0).all())


# T, k, E, H, I; the plan (routed rows a tile; direct form: 0, waves of gate_up, of down); whether gate_up and down have more tiles
# than workgroups at once
EXPERTS = [(3001, 3, 8, 1300, 700, (192, 0, 0), True, True), (9000, 3, 4, 200, 1500, (192, 0, 0), True, False),
           (1400, 2, 16, 2400, 1300, (128, 0, 0), True, True), (700, 3, 16, 390, 300, (128, 0, 0), False, False),
           (500, 2, 20, 640, 260, (64, 0, 0), False, False), (300, 2, 48, 260, 500, (32, 0, 0), False, False),
           (2, 3, 8, 1600, 900, (0, 8, 8), False, False), (1, 9, 16, 300, 2100, (0, 4, 16), False, False),
           (2, 1, 8, 200, 300, (0, 4, 4), False, False)]


@pytest.mark.parametrize("T,k,E,H,I,plan,loop_gu,loop_dn", EXPERTS)
def test_experts_plans(dev, T, k, E, H, I, plan, loop_gu, loop_dn):
    import torch
    from infinitemodel_amd import _lib, ops
    assert _plan("IMQ_PLAN_MOE_F8", T, H, k, I, sqn=E)[:3] == plan
    bm = plan[0]
    hb, ib = of.blocks(H), of.blocks(I)
    g = torch.Generator().manual_seed(T)
    rank = torch.randn(T, E, generator=g) + 0.5 * torch.randn(E, generator=g)
    w, ids = torch.topk(torch.softmax(rank, -1), k, -1)
    if bm > 0:
        tiles = int((-(-torch.bincount(ids.reshape(-1), minlength=E) // bm)).sum())
        assert (tiles * ib > 256) == loop_gu                  # a workgroup a CU
        assert {192: tiles * -(-H // 256) > 256, 128: tiles * -(-H // 128) > 512}.get(bm, False) == loop_dn
    gq, dq = _bytes(dev, (E, 2 * I, hb * 128), T), _bytes(dev, (E, H, ib * 128), T + 1)
    gq[..., H:], dq[..., I:] = 0, 0
    gs, ds = (1e-4 + 2e-4 * torch.rand(*sh, generator=g) for sh in ((E, 2 * ib, hb), (E, hb, ib)))
    x = (torch.randn(T, H, generator=g) * torch.exp(0.5 * torch.randn(T, 1, generator=g))).to(torch.bfloat16)
    f8 = torch.float8_e4m3fn
    out = ops.moe_experts_f8(x.to(dev), ids.to(dev), w.to(dev), (gq.view(f8), gs.to(dev), H), (dq.view(f8), ds.to(dev), I))
    assert bool(torch.isfinite(out).all())
    # tokens enough to meet every tile of rows, the first and last of all among them
    pick = torch.unique(torch.cat([torch.randperm(T, generator=g)[:250], torch.tensor([0, T - 1])]))
    want, tol = of.experts(of.dequantize(*of.quantize(x[pick].double().numpy())), ids[pick].numpy(), w[pick].numpy(),
                           (gq.cpu().numpy(), gs.numpy()), (dq.cpu().numpy(), ds.numpy()), H, I)
    got = out[pick.to(dev)].double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    assert torch.equal(out, ops.moe_experts_f8(x.to(dev), ids.to(dev), w.to(dev), (gq.view(f8), gs.to(dev), H), (dq.view(f8), ds.to(dev), I)))
