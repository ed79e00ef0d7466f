"""The fp8 operators' calls on the GPU: what refused ones leave behind, outputs over inputs, captured ones."""
import pytest

pytestmark = pytest.mark.gpu


def test_refused_sizes_take_no_workspace(dev, monkeypatch):
    """Experts of more bytes than 32-bit offsets reach, by the native host path and by the Python one: refused, and no workspace is
    taken for them."""
    import torch
    from infinitemodel_amd import _lib, ops
    T, k, H, I = 131072, 8, 7168, 2048
    f8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)     # noqa: E731
    gu = (f8(1, 2 * I, H), torch.ones(1, 2 * I // 128, H // 128, device=dev), H)
    dn = (f8(1, H, I), torch.ones(1, H // 128, I // 128, device=dev), I)
    x = torch.zeros(T, H, dtype=torch.bfloat16, device=dev)
    ids, w = torch.zeros(T, k, dtype=torch.int64, device=dev), torch.ones(T, k, device=dev)
    monkeypatch.setattr(ops, "_scratch", lambda *a: pytest.fail("took a workspace"))
    with torch.cuda.stream(torch.cuda.Stream()):
        for check in (True, False):
            with pytest.raises(_lib.ImqError) as e:
                ops.moe_experts_f8(x, ids, w, gu, dn, check_ids=check)
            assert e.value.status == _lib.IMQ_ERR_UNSUPPORTED
    torch.cuda.synchronize()


@pytest.mark.parametrize("M", [1, 5, 16, 40])
def test_out_over_x(dev, M):
    """A result that goes where its input is (or a row further) is that of a call with an output of its own."""
    import torch
    from infinitemodel_amd import ops
    K = 2048
    W = torch.randn(K, K, generator=torch.Generator().manual_seed(M)) * 0.02
    q, s, _ = ops.pack_f8(W.to(dev))
    x = torch.randn(M + 1, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(dev)
    want = ops.linear_f8(x[:M], q, s)
    for row in (0, 1):
        buf = x.clone()
        y = ops.linear_f8(buf[:M], q, s, out=buf[row:row + M])
        assert y.data_ptr() == buf[row].data_ptr() and torch.equal(y, want)
        assert torch.equal(buf[M if row == 0 else 0], x[M if row == 0 else 0])
