"""The C ABI of the packed and served forms on the GPU: outputs, checkpoints and
workspaces stay inside their buffers whatever the device's offsets say, and the
steps honour `fresh`."""

import ctypes

import pytest
import torch

from mlx_vision_mamba_amd import _lib
from tests import seq_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODE = {torch.float32: 0, torch.bfloat16: 1}


class Fenced:
    """Buffers between two runs of a pattern, of which no byte may change."""
    EDGE, MARK = 4096, 0xA5

    def __init__(self, device):
        self.device, self.bufs = device, {}

    def __call__(self, name, count, dtype=torch.float32):
        n = count * torch.empty(0, dtype=dtype).element_size()
        buf = torch.full((2 * self.EDGE + (n + 255) // 256 * 256,), self.MARK, dtype=torch.uint8, device=self.device)
        self.bufs[name] = buf, n
        return buf.data_ptr() + self.EDGE

    def value(self, name, *shape, dtype=torch.float32):
        buf, n = self.bufs[name]
        return buf[self.EDGE:self.EDGE + n].view(dtype).view(*shape)

    def check(self):
        for name, (buf, n) in self.bufs.items():
            assert bool((buf[:self.EDGE] == self.MARK).all()), f"before {name}"
            assert bool((buf[self.EDGE + n:] == self.MARK).all()), f"past {name}"


@pytest.mark.parametrize("at", [-1, 100])
def test_fence_notices_a_write(cuda, at):
    buf = Fenced(cuda)
    buf("x", 25)
    buf.check()
    buf.bufs["x"][0][Fenced.EDGE + at] = 0
    with pytest.raises(AssertionError, match="before x" if at < 0 else "past x"):
        buf.check()


def _stream():
    return torch.cuda.current_stream().cuda_stream


# device offsets that no host check would let through (six for five sequences of
# 64 tokens: they decrease, lie outside, or both), and good ones
OFFSETS = {"good": [0, 9, 9, 30, 40, 64], "mixed": [9, 70, -5, 30, 12, 1 << 30], "far": [2 ** 31 - 1] * 6,
           "negative": [-2 ** 31] * 6, "falling": [64, 50, 33, 32, 17, 0], "zigzag": [0, 64, 0, 64, 0, 64]}


@pytest.mark.parametrize("offsets", list(OFFSETS))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,D,chunk", [(16, 70, 0), (16, 70, 16), (5, 130, 16)])
def test_scan_stays_in_its_buffers(cuda, N, D, chunk, dtype, offsets):
    T, S, t = 64, 5, TYPES[dtype]
    g = torch.Generator().manual_seed(1)
    r = lambda *s, d=torch.float32: torch.randn(*s, generator=g).to(cuda, d)  # noqa: E731
    u, delta, z, dy = (r(T, D, d=t) for _ in range(4))
    B, C = r(T, N, d=t), r(T, N, d=t)
    A, Dv, bias, h0, dh1 = r(D, N), r(D), r(D), r(S, D, N), r(S, D, N)
    off = torch.tensor(OFFSETS[offsets], dtype=torch.int32, device=cuda)
    d = _lib.SeqScanDesc()
    d.seq.tokens, d.seq.nseq, d.seq.dim, d.seq.state_rows, d.seq.offsets = T, S, D, S, off.data_ptr()
    d.dstate, d.bc_stride = N, N
    d.u_stride = d.delta_stride = d.y_stride = d.z_stride = D
    d.dtype = d.delta_dtype = CODE[t]
    d.delta_softplus, d.a_is_log, d.chunk_len = 1, 1, chunk
    lib, p, buf = _lib.lib(), ctypes.byref(d), Fenced(cuda)
    ins = [x.data_ptr() for x in (u, delta, bias, A, B, C, Dv, z)]
    ckpt = buf("ckpt", _lib.check(lib.mvm_seq_scan_ckpt_elems(p)))
    n = _lib.check(lib.mvm_seq_scan_workspace_bytes(p, 0))
    _lib.check(lib.mvm_seq_scan_fwd(p, *ins, h0.data_ptr(), buf("h1", S * D * N), buf("y", T * D, t), ckpt,
                                    buf("workspace", n, torch.uint8), n, _stream()))
    buf.check()
    n = _lib.check(lib.mvm_seq_scan_workspace_bytes(p, 1))
    wide = [buf(k, T * D, t) for k in ("du", "ddelta")] + [buf("ddelta_bias", D), buf("dA", D * N)] \
        + [buf(k, T * N, t) for k in ("dB", "dC")] + [buf("dD", D), buf("dz", T * D, t), buf("dh0", S * D * N)]
    _lib.check(lib.mvm_seq_scan_bwd(p, *ins, ckpt, dy.data_ptr(), dh1.data_ptr(), *wide,
                                    buf("workspace of the backward", n, torch.uint8), n, _stream()))
    buf.check()
    if offsets == "good":
        want = ref.scan(OFFSETS[offsets], u, delta, A, B, C, Dv, z, bias, True, True, h0, dy, dh1)
        for name, shape, dt in [("y", (T, D), t), ("h1", (S, D, N), None), ("du", (T, D), t), ("ddelta", (T, D), t),
                                ("ddelta_bias", (D,), None), ("dA", (D, N), None), ("dB", (T, N), t),
                                ("dC", (T, N), t), ("dD", (D,), None), ("dz", (T, D), t), ("dh0", (S, D, N), None)]:
            ref.check(name, buf.value(name, *shape, dtype=dt or torch.float32),
                      want[{"h1": "final", "dh0": "dinitial"}.get(name, name)])


@pytest.mark.parametrize("offsets", list(OFFSETS))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("W,D", [(4, 72), (4, 71), (2, 130), (8, 72), (1, 72)])
def test_conv_stays_in_its_buffers(cuda, W, D, dtype, offsets):
    T, S, t = 64, 5, TYPES[dtype]
    g = torch.Generator().manual_seed(2)
    r = lambda *s, d=torch.float32: torch.randn(*s, generator=g).to(cuda, d)  # noqa: E731
    x, dy, w, b = r(T, D, d=t), r(T, D, d=t), r(D, W), r(D)
    c0, dc1 = r(S, W - 1, D, d=t), r(S, W - 1, D, d=t)
    off = torch.tensor(OFFSETS[offsets], dtype=torch.int32, device=cuda)
    d = _lib.SeqConvDesc()
    d.seq.tokens, d.seq.nseq, d.seq.dim, d.seq.state_rows, d.seq.offsets = T, S, D, S, off.data_ptr()
    d.kwidth, d.x_stride, d.y_stride, d.dtype = W, D, D, CODE[t]
    lib, p, buf = _lib.lib(), ctypes.byref(d), Fenced(cuda)
    rows = S * (W - 1) * D
    _lib.check(lib.mvm_seq_conv_fwd(p, x.data_ptr(), w.data_ptr(), b.data_ptr(), c0.data_ptr(), buf("c1", rows, t),
                                    buf("y", T * D, t), _stream()))
    buf.check()
    n = _lib.check(lib.mvm_seq_conv_workspace_bytes(p))
    _lib.check(lib.mvm_seq_conv_bwd(p, x.data_ptr(), w.data_ptr(), b.data_ptr(), c0.data_ptr(), dy.data_ptr(),
                                    dc1.data_ptr(), buf("dx", T * D, t), buf("dw", D * W), buf("db", D),
                                    buf("dc0", rows, t), buf("workspace", n, torch.uint8), n, _stream()))
    buf.check()
    if offsets == "good":
        want = ref.conv(OFFSETS[offsets], x, w, b, c0, dy, dc1)
        for name, to, shape, dt in [("y", "y", (T, D), t), ("c1", "final", (S, W - 1, D), t), ("dx", "dx", (T, D), t),
                                    ("dw", "dweight", (D, W), torch.float32), ("db", "dbias", (D,), torch.float32),
                                    ("dc0", "dinitial", (S, W - 1, D), t)]:
            ref.check(name, buf.value(name, *shape, dtype=dt), want[to])


def _step_seq(d, S, D, slots, fresh, rows):
    d.seq.tokens, d.seq.nseq, d.seq.seqlen, d.seq.dim, d.seq.state_rows = S, S, 1, D, rows
    d.seq.slots, d.seq.fresh = slots.data_ptr(), fresh.data_ptr()


# 13 states: the path of single values; 259 x 512 and 1027 x 64: several sequences a wave
@pytest.mark.parametrize("S,D,N", [(5, 70, 16), (5, 70, 13), (7, 64, 4), (9, 64, 8), (259, 512, 16)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_scan_step_honours_fresh(cuda, S, D, N, dtype):
    """A fresh sequence starts from zero whatever its row holds, here NaN."""
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a = dict(u=r(S, D).to(t), delta=r(S, D).to(t), A=-torch.rand(D, N, generator=g), B=r(S, N).to(t),
             C=r(S, N).to(t), D=r(D))
    z, bias, rows = r(S, D).to(t), r(D), S + 2
    slots, fresh = torch.randperm(rows, generator=g)[:S], torch.rand(S, generator=g) < 0.5
    fresh[:2] = torch.tensor([True, False])
    slots[S - 1] = -1  # no row: its y is zero
    states = r(rows, D, N)
    init = torch.where(fresh[:, None, None], 0.0, states[slots.clamp(min=0)])
    states[slots[:S - 1][fresh[:S - 1]]] = float("nan")
    want = ref.scan(list(range(S + 1)), **a, z=z, delta_bias=bias, delta_softplus=True, initial=init)
    live = {k: v.to(cuda) for k, v in a.items()}
    zc, bc, st, sl, fr = z.to(cuda), bias.to(cuda), states.to(cuda), slots.int().to(cuda), fresh.to(cuda)
    d = _lib.SeqScanDesc()
    _step_seq(d, S, D, sl, fr, rows)
    d.dstate, d.bc_stride = N, N
    d.u_stride = d.delta_stride = d.y_stride = d.z_stride = D
    d.dtype = d.delta_dtype = CODE[t]
    d.delta_softplus = 1
    y = torch.full((S, D), 7.0, dtype=t, device=cuda)
    p = {k: v.data_ptr() for k, v in live.items()}
    _lib.check(_lib.lib().mvm_seq_scan_step(ctypes.byref(d), p["u"], p["delta"], bc.data_ptr(), p["A"], p["B"], p["C"],
                                            p["D"], zc.data_ptr(), st.data_ptr(), y.data_ptr(), _stream()))
    n = S - 1
    ref.check("y", y[:n], want["y"][slice(0, n)])
    assert not y[n].any()
    ref.check("states", st[sl[:n].long()], want["final"][slice(0, n)])
    rest = [i for i in range(rows) if i not in slots[:n].tolist()]
    assert torch.equal(st[rest].cpu(), states[rest])


@pytest.mark.parametrize("S,D,W", [(5, 72, 4), (5, 71, 4), (3, 64, 8), (1027, 64, 4)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_conv_step_honours_fresh(cuda, S, D, W, dtype):
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, w, b, rows = r(S, D).to(t), r(D, W), r(D), S + 2
    slots, fresh = torch.randperm(rows, generator=g)[:S], torch.rand(S, generator=g) < 0.5
    fresh[:2] = torch.tensor([True, False])
    slots[S - 1] = rows
    states = r(rows, W - 1, D).to(t)
    init = torch.where(fresh[:, None, None], 0.0, states[slots.clamp(max=rows - 1)].float()).to(t)
    states[slots[:S - 1][fresh[:S - 1]]] = float("nan")
    want = ref.conv(list(range(S + 1)), x, w, b, initial=init)
    xc, wc, bc, st, sl, fr = x.to(cuda), w.to(cuda), b.to(cuda), states.to(cuda), slots.int().to(cuda), fresh.to(cuda)
    d = _lib.SeqConvDesc()
    _step_seq(d, S, D, sl, fr, rows)
    d.kwidth, d.x_stride, d.y_stride, d.dtype = W, D, D, CODE[t]
    y = torch.full((S, D), 7.0, dtype=t, device=cuda)
    _lib.check(_lib.lib().mvm_seq_conv_step(ctypes.byref(d), xc.data_ptr(), wc.data_ptr(), bc.data_ptr(), st.data_ptr(),
                                            y.data_ptr(), _stream()))
    n = S - 1
    ref.check("y", y[:n], want["y"][slice(0, n)])
    assert not y[n].any()
    ref.check("states", st[sl[:n].long()], want["final"][slice(0, n)])
    rest = [i for i in range(rows) if i not in slots[:n].tolist()]
    assert torch.equal(st[rest].cpu(), states[rest])
