"""Rotary positions on the GPU against the definition in float64.

Tolerance: the angle is exact to 1e-9, its sine and cosine and the products are f32 operations (at most 2^-22 of the
pair's size together), so f32 results are within 2^-21 of the pair's size; bf16 adds half a step, 2^-8 of the value."""
import numpy as np
import pytest

import kv8_model as M
from gpu_util import BF16, F32, Bufs, QwRef, from_io, io_np, to_io
from qwasar_b200 import synth

pytestmark = pytest.mark.gpu


def run(be, rows, heads, hd, rot, inter, io, x_pad=0, y_pad=0, pos=None, amp=1.0, in_place=False, x_off=0, freq=None):
    rng = np.random.default_rng(rows * 131 + heads * 17 + hd + rot)
    w = heads * hd
    x = rng.standard_normal((rows, w + x_pad)).astype(np.float32)
    x = synth.bf16_round(x)
    pos = np.arange(rows, dtype=np.int32) if pos is None else np.asarray(pos, np.int32)
    freq = (1e6 ** (-2.0 * np.arange(rot // 2) / rot)).astype(np.float32) if freq is None else freq
    el = 2 if io == BF16 else 4
    with Bufs(be) as B:
        flat = np.concatenate([np.zeros(x_off, np.float32), x.ravel()])
        xb = B.device(to_io(flat, io))
        yb = xb if in_place else B.device(np.full(rows * (w + y_pad), 0x55, io_np(io)))
        c = be.cmd_begin()
        ok = be.op_rope(c, QwRef(yb, x_off * el if in_place else 0), QwRef(xb, x_off * el), QwRef(B.device(pos), 0), QwRef(B.device(freq), 0), rows, heads, hd, rot,
                        int(inter), w + (x_pad if in_place else y_pad), w + x_pad, amp, io)
        assert ok, be.cmd_error(c)
        be.cmd_wait(c); be.cmd_free(c)
        n = rows * (w + (x_pad if in_place else y_pad))
        got = np.empty(n, io_np(io))
        be.buf_download(yb, x_off * el if in_place else 0, got)
    got = got.reshape(rows, -1)
    if in_place:
        assert np.array_equal(got[:, w:], to_io(x[:, w:], io))
    else:
        assert np.all(got[:, w:] == np.full((), 0x55, io_np(io)))       # nothing between the rows was touched
    xx = x[:, :w].reshape(rows, heads, hd)
    want = M.rope(xx, pos, freq, rot, inter, amp)
    got = from_io(np.ascontiguousarray(got[:, :w]), io).reshape(rows, heads, hd).astype(np.float64)
    i0 = np.arange(0, rot, 2) if inter else np.arange(rot // 2)
    i1 = i0 + 1 if inter else i0 + rot // 2
    size = np.abs(want)
    size[..., i0] = size[..., i1] = np.hypot(want[..., i0], want[..., i1])
    tol = 2.0 ** -21 * size + (2.0 ** -8 * np.abs(want) if io == BF16 else 0)
    assert np.all(np.abs(got - want) <= tol)
    assert np.array_equal(got[..., rot:], xx[..., rot:])


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("rows,heads,hd,rot", [(1, 1, 2, 2), (1, 16, 256, 64), (3, 5, 64, 64), (7, 3, 96, 36), (33, 24, 256, 256), (2, 9, 80, 10), (1, 40, 4096, 4096), (5, 1, 192, 6)])
def test_rope(be, io, inter, rows, heads, hd, rot):
    run(be, rows, heads, hd, rot, inter, io)


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("kw", [dict(x_pad=40, y_pad=8), dict(x_pad=3, y_pad=5), dict(in_place=True), dict(in_place=True, x_pad=16), dict(x_off=64, amp=1.25), dict(in_place=True, x_pad=1)],
                         ids=["padded", "odd-strides", "in-place", "in-place-padded", "offset-amp", "in-place-odd"])
def test_rope_layouts(be, io, inter, kw):
    run(be, 9, 4, 128, 64, inter, io, **kw)


@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
def test_rope_far_and_negative_positions(be, inter):
    pos = [0, 1, -1, 262143, 1000003, 2 ** 31 - 1, -2 ** 31, 123456789]
    run(be, 8, 2, 64, 64, inter, F32, pos=pos)
    run(be, 8, 2, 64, 64, inter, F32, pos=pos, freq=np.linspace(0.1, 3.0, 32).astype(np.float32))


def test_rope_refusals(be):
    with Bufs(be) as B:
        x = QwRef(B.device(np.zeros(4096, np.float32)), 0)
        y = QwRef(B.device(np.zeros(4096, np.float32)), 0)
        pos, fr = QwRef(B.device(np.zeros(8, np.int32)), 0), QwRef(B.device(np.zeros(64, np.float32)), 0)
        call = lambda c, y=y, x=x, p=pos, f=fr, rows=2, h=2, hd=64, rot=64, lay=0, ys=128, xs=128, io=F32: be.op_rope(c, y, x, p, f, rows, h, hd, rot, lay, ys, xs, 1.0, io)  # noqa: E731
        z = QwRef(None, 0)
        bad = [dict(rows=-1), dict(h=0), dict(hd=0), dict(hd=5000), dict(rot=0), dict(rot=63), dict(rot=66), dict(lay=2), dict(lay=-1), dict(ys=127), dict(xs=100), dict(xs=2 ** 40),
               dict(io=5), dict(x=z), dict(y=z), dict(p=z), dict(f=z), dict(rows=9), dict(rows=40), dict(y=QwRef(x.buf, 512)), dict(y=x, ys=160), dict(x=QwRef(x.buf, 4)),
               dict(f=QwRef(fr.buf, 252)), dict(rot=2, f=QwRef(fr.buf, 2))]
        launches = be.launch_count()
        for kw in bad:
            c = be.cmd_begin()
            assert not call(c, **kw), kw
            be.cmd_wait(c, check=False); be.cmd_free(c)
        assert be.launch_count() == launches
        c = be.cmd_begin()
        assert call(c, rows=0) and call(c, y=x)
        be.cmd_wait(c); be.cmd_free(c)
