"""The bound that the fp8 linear is held to tells a kernel's mistakes from its roundings, at short sums and at the longest."""
import numpy as np
import pytest

from oracle import f8 as of


def _bf16(v):
    u = v.astype(np.float32).view(np.uint32).astype(np.uint64)
    return (((u + 0x7fff + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)


@pytest.mark.parametrize("K", [256, 2048, 14336, 128 * 129])
def test_linear_bound_tells_mistakes(K):
    r = np.random.default_rng(K)
    M, N, nb = 8, 128, of.blocks(K)
    x = r.standard_normal((M, K)).astype(np.float32)
    xq, xs = of.quantize(x)
    codes = of.codes_of(np.clip(r.standard_normal((N, K)) * 100, -448, 448))
    ws = r.uniform(1e-4, 3e-4, (1, nb)).astype(np.float32)
    xv, wv = of.dequantize(xq, xs), of.dequantize(codes, ws, 128)
    y, tol = of.linear(xv, wv)
    blocks = [(codes_x, codes_w) for codes_x, codes_w in zip(np.split(of.values_of(xq), nb, 1), np.split(of.values_of(codes), nb, 1))]

    def outside(z):
        return (np.abs(z - y) > tol).mean()

    def summed(keep):
        """As the kernel sums: blocks in fp32, each times its factor, `keep` of the running sum."""
        acc = np.zeros((M, N), np.float32)
        for b, (cx, cw) in enumerate(blocks):
            part = np.zeros((M, N), np.float32)
            for k in range(128):
                part += (cx[:, k:k + 1] * cw[:, k]).astype(np.float32)
            acc = keep(acc + part * (xs[:, b:b + 1] * ws[0, b]))
        return _bf16(acc)

    assert outside(summed(lambda a: a)) == 0                  # a right kernel
    assert outside(summed(_bf16)) > 0.005                     # the running sum in bf16
    short = xv.copy()
    short[:, -128:] = 0
    assert outside(_bf16(short @ wv.T)) > 0.8                 # the last block left out
    assert outside(_bf16(x.astype(np.float64) @ wv.T)) > 0.5  # x not quantized
    assert outside(_bf16(1.01 * y)) > 0.3                     # every scale off by 1%
    off = ws.copy()
    off[0, nb // 2] *= 1.2
    assert outside(_bf16(xv @ of.dequantize(codes, off, 128).T)) > 0.3      # one block's scale off by 20%
    turned = xs[:, ::-1]
    assert outside(_bf16(of.dequantize(xq, turned) @ wv.T)) > 0.5           # scales of other blocks
