"""What the fp8 operators do around a launch, without a device: refusals before any memory is taken, the stream that is asked
about capture, outputs that lie over inputs, sizes at the ends of the C entry points."""
import contextlib
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from infinitemodel_amd import _lib

F8 = torch.float8_e4m3fn
BF, F32 = _lib.IMQ_DT_BF16, _lib.IMQ_DT_FP32
UNSUP, SCRATCH = _lib.IMQ_ERR_UNSUPPORTED, _lib.IMQ_ERR_SCRATCH
P = ctypes.c_void_p(4096)          # never dereferenced: every call here is refused on the host
TOP = 2 ** 31 - 1


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


@pytest.fixture
def host_ops(monkeypatch):
    """ops on host tensors, the entries as they are (what gets past their checks fails for want of a device); a workspace
    fails the test."""
    from infinitemodel_amd import ops
    monkeypatch.setattr(ops, "_check_dev", lambda *a: torch.device("cpu"))
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "_scratch", lambda *a: pytest.fail("took a workspace"))
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    return ops


def _experts(L, T, k, E, H, I, gsq=None, dsq=None, ws=P, wsb=1 << 62):
    up = lambda n: -(-n // 128) * 128                                        # noqa: E731
    gsq, dsq = up(H) if gsq is None else gsq, up(I) if dsq is None else dsq
    return L.imq_moe_experts_f8(P, H, BF, T, H, k, P, _lib.IMQ_DT_I64, P, F32, E, P, 0, gsq, P, 0, 0, I, P, 0, dsq, P, 0, 0, P, H, ws,
                                wsb, None)


SIZES = [(131072, 8, 64, 7168, 2048), (262144, 8, 64, 8192, 2048), (1 << 24, 1, 4, 129, 128), (1 << 23, 2, 4, 128, 129), (4, 1, 4, 1 << 24, 256),
         (4, 1, 4, 256, 1 << 24), (TOP, 1, 4, 1, 1), (1, TOP, 4, 1, 1), (1, 1, 4, TOP, 1), (1, 1, 4, 1, TOP), (TOP, TOP, 4, TOP, TOP),
         (1 << 60, 1 << 60, 4, 1 << 60, 1 << 60), (3, 2, 4097, 128, 128), (1 << 24, 1, 4, 128, 128), (1 << 23, 1, 4, 128, 128)]


@pytest.mark.parametrize("T,k,E,H,I", SIZES)
def test_experts_sizes_that_are_refused_need_no_workspace(L, T, k, E, H, I):
    """imq_moe_f8_workspace_bytes says -1 exactly where the entry refuses the sizes; it never overflows."""
    need = L.imq_moe_f8_workspace_bytes(T, k, E, H, I)
    rc = _experts(L, T, k, E, H, I, ws=None, wsb=0)
    assert (need == -1) == (rc == UNSUP) and rc in (UNSUP, SCRATCH)
    assert need == -1 or T * k * 4 * H < need < 2 ** 50


def test_experts_strides_that_are_refused(L):
    assert _experts(L, 3, 2, 4, 256, 128, ws=None, wsb=0) == SCRATCH
    assert _experts(L, 3, 2, 4, 256, 128, gsq=1 << 26, ws=None, wsb=0) == UNSUP
    assert _experts(L, 3, 2, 4, 256, 128, dsq=1 << 26, ws=None, wsb=0) == UNSUP


def _refused(f):
    with pytest.raises(_lib.ImqError) as e:
        f()
    assert e.value.status == UNSUP


def test_refused_experts_take_no_memory(host_ops):
    """Sizes past 32-bit offsets, and strides past them, are refused before a workspace is taken."""
    stack = lambda E, N, K: torch.empty(E, N, -(-K // 128) * 128, dtype=F8)    # noqa: E731
    T, k, H, I = 131072, 8, 7168, 2048
    gu = (stack(1, 2 * I, H), torch.empty(1, 2 * I // 128, H // 128), H)
    dn = (stack(1, H, I), torch.empty(1, H // 128, I // 128), I)
    x = torch.empty(T, H, dtype=torch.bfloat16)
    ids, w = torch.zeros(T, k, dtype=torch.int64), torch.ones(T, k)
    for check in (True, False):
        _refused(lambda: host_ops.moe_experts_f8(x, ids, w, gu, dn, check_ids=check))
    far = torch.empty(128 << 24, dtype=torch.uint8).view(F8).as_strided((1, 128, 256), (0, 1 << 24, 1))   # never written
    gu = (far, torch.empty(1, 2, 2), 256)
    dn = (stack(1, 256, 64), torch.empty(1, 2, 1), 64)
    _refused(lambda: host_ops.moe_experts_f8(x[:3, :256], ids[:3], w[:3], gu, dn, check_ids=False))


def test_refused_linears_take_no_memory(host_ops):
    far = torch.empty(2 << 24, dtype=torch.uint8).view(F8).as_strided((2, 512), (1 << 24, 1))
    for M in (16, 40, 200):
        _refused(lambda: host_ops.linear_f8(torch.empty(M, 64 << 7)[:, :512], far, torch.ones(1, 4)))


# ---- capture -------------------------------------------------------------------------------------
class _OnDevice:
    """As much of a tensor of device ``index`` as the questions about capture ask for."""
    is_cuda = True

    def __init__(self, index):
        self.index, self.device = index, torch.device("cuda", index)

    def get_device(self):
        return self.index

    def numel(self):
        return 4


@pytest.mark.parametrize("captured", [0, 1])
@pytest.mark.parametrize("index", [0, 1])
def test_capture_is_asked_of_the_tensor_s_device(monkeypatch, captured, index):
    """With device 0 current, and the stream of one of two devices under capture: what counts is the stream of the device that the
    call runs on, for the workspace and for the ids' check alike."""
    from infinitemodel_amd import ops
    now = [0]

    @contextlib.contextmanager
    def device(d):
        old, now[0] = now[0], torch.device("cuda", d).index if isinstance(d, int) else torch.device(d).index
        yield
        now[0] = old
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == captured)
    monkeypatch.setattr(torch, "aminmax", lambda t: (0, 9))
    x = _OnDevice(index)
    assert ops._capturing(x) == (index == captured) and now[0] == 0
    if index == captured:
        ops._check_expert_ids(x, 4)                # a read would end the capture
    else:
        with pytest.raises(ValueError):
            ops._check_expert_ids(x, 4)
    assert not ops._capturing(torch.zeros(1))


# ---- out over an input ---------------------------------------------------------------------------
def test_out_over_an_input_is_not_what_the_launch_writes(host_ops, monkeypatch):
    """Where out shares memory with x, the weights or a scale, the launch gets a tensor of its own and out a copy of it; elsewhere,
    also right beside an input, out itself."""
    seen = []

    def launch(name, dev, need, captured, *a):
        seen.append(a[-2])                         # y: filled as a kernel would
        ctypes.memset(a[-2], 0x40, 2 * 256)
    monkeypatch.setattr(host_ops, "_f8_launch", launch)
    buf = torch.zeros(3, 256, dtype=torch.bfloat16)
    raw = torch.zeros(1 << 16, dtype=torch.uint8)
    q, s = raw.view(F8).view(256, 256), torch.ones(2, 512)[:, ::256]
    xq, xs = torch.zeros(1, 256).to(F8), torch.ones(1, 512)[:, ::256]

    def over(t, at):                               # a [1, 256] bf16 view of t's memory from byte `at`
        return torch.empty(0, dtype=torch.bfloat16).set_(t.untyped_storage(), at // 2, (1, 256))
    x = buf[:1]
    for call, out, own in ((lambda o: host_ops.linear_f8(x, q, s, out=o), buf[1:2], False),
                           (lambda o: host_ops.linear_f8(x, q, s, out=o), buf[:1], True),
                           (lambda o: host_ops.linear_f8(x, q, s, out=o), over(raw, 1000), True),
                           (lambda o: host_ops.linear_f8(x, q, s, out=o), over(s, 600), True),
                           (lambda o: host_ops.linear_f8(xq, q, s, x_scale=xs, out=o), over(xs, 600), True)):
        y = call(out)
        assert (seen[-1] != out.data_ptr()) == own and y.data_ptr() == out.data_ptr()
        assert bool((out.view(torch.uint8) == 0x40).all())


# ---- the ends of the C entries -------------------------------------------------------------------
def test_one_row_of_down_without_a_stride():
    """H = 1 takes any stride of down's one row, 0 as well; in a process of its own, as a division by it would end that."""
    code = ("import ctypes, torch\nfrom infinitemodel_amd import _lib\nP = ctypes.c_void_p(4096)\n"
            "f = lambda ds: _lib.lib().imq_moe_experts_f8(P, 1, 0, 3, 1, 2, P, 4, P, 2, 4, P, 0, 128, P, 0, 0, 128, P, 0, ds, P, 0, 0, "
            "P, 1, None, 0, None)\nprint(f(0), f(128), f(-16))")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(__file__)))
    assert r.returncode == 0 and r.stdout.split() == [str(SCRATCH), str(SCRATCH), str(_lib.IMQ_ERR_INVALID)], r


def test_linear_strides_whose_multiples_overflow(L):
    """Row strides are held against the limit by division: 257 times this one is 256 in 64 bits."""
    wraps = 0xff00ff00ff0100
    assert wraps * 257 % 2 ** 64 == 256

    def f(sx=512, dt=BF, sq=512, xs=None):
        return L.imq_linear_f8(P, sx, dt, 40, 512, xs, 4, 1, P, sq, P, 4, 1, 300, 512, P, 300, None, 0, None)
    assert f() == SCRATCH
    assert f(sq=wraps) == UNSUP and f(sq=1 << 23) == UNSUP and f(sq=1 << 22) == SCRATCH
    assert f(dt=_lib.IMQ_DT_F8, xs=P, sx=wraps) == UNSUP and f(dt=_lib.IMQ_DT_F8, xs=P, sx=1 << 23) == UNSUP
