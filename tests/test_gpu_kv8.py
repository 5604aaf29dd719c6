"""The 8-bit cache on the GPU against its definition in float64 (kv8_model): append, read, attention.

Tolerances.  Append and read are exact: the exponents are whole numbers, scaling by them is exact, and the one
rounding (to e4m3, ties to even) is defined.  Attention over the same codes:
  f32   q and the softmax weights enter as two fp16 parts, 22 bits: 2^-22 of each product, with 2^-24 per f32
        addition; the exponential's argument is up to ~30, so a weight is off by about 30 * 2^-23 = 4e-6 at most and
        the norm of a row's error stays below 1e-5 of the row's norm.
  bf16  the output's rounding (half a step, 2^-8 of the value at most) plus the weights' rounding to fp16 (2^-11
        each, of either sign): 2^-8 + 2^-10 of the row's largest value.
  bf16, many rows: the bounds of the bf16 cache's prefill in test_gpu_attn.py, 1e-2 of the row's largest value and
        5e-3 in the norm: enough for weights rounded to bf16 (2^-8 each)."""
import numpy as np
import pytest

import kv8_model as M
from conftest import max_rel_err, rel_l2
from gpu_util import BF16, F32, Bufs, NULL_REF, QwRef, from_io, io_np, to_io
from qwasar_b200 import synth

pytestmark = pytest.mark.gpu
HD = 256


def draw_kv(rng, rows, heads, spread=0.0):
    """Rows of keys or values whose size varies by channel and, with `spread`, from one block of 64 to the next."""
    x = rng.standard_normal((rows, heads, HD)) * np.exp(0.5 * rng.standard_normal((1, heads, HD)))
    if spread:
        x = x * np.exp2(np.rint(rng.uniform(-spread, spread, (rows // 64 + 1, heads)))).repeat(64, 0)[:rows, :, None]
    return synth.bf16_round(x.astype(np.float32))


class Pair:
    """K and V caches of one layer on the device and their models: a plain buffer each, or arenas."""

    def __init__(self, be, B, heads, ctx, paged, pool=None, layers=1, layer=0, seed=0):
        self.be, self.heads, self.ctx, self.paged = be, heads, ctx, paged
        self.k, self.v = M.Cache(heads, ctx), M.Cache(heads, ctx)
        self.bytes = be.kv8_layer_bytes(heads, ctx)
        if paged:
            mk = lambda: be.kv8_arena_alloc_in(pool, layers, heads, ctx) if pool else be.kv8_arena_alloc(layers, heads, ctx, shuffle_seed=seed)  # noqa: E731
            self.bufs = [mk(), mk()]
            B.all += self.bufs
        else:
            self.bufs = [be.buf_alloc_device(self.bytes * layers) for _ in range(2)]
            B.all += self.bufs
        self.kr, self.vr = (QwRef(b, layer * self.bytes) for b in self.bufs)

    def append(self, c, B, k, v, base, io, pad=0):
        rows = k.shape[0]
        stride = self.heads * HD + pad
        refs = []
        for x in (k, v):
            wide = np.full((rows, stride), 7.0, np.float32)
            wide[:, :self.heads * HD] = x.reshape(rows, -1)
            refs.append(QwRef(B.device(to_io(wide, io)), 0))
        ok = self.be.op_kv8_write(c, self.kr, self.vr, *refs, rows, self.heads, HD, self.ctx, base, stride, io)
        self.k.append(k, base)
        self.v.append(v, base)
        return ok

    def read(self, c, B, which, lo, n, io=F32):
        b = B.device(np.full((self.heads, n, HD), 9, io_np(io)))
        assert self.be.op_kv8_read(c, QwRef(b, 0), self.vr if which else self.kr, lo, n, self.heads, HD, self.ctx, io)
        return b

    def check(self, be, B, hi, lo=0, io=F32):
        c = be.cmd_begin()
        bufs = [self.read(c, B, w, lo, hi - lo, io) for w in (0, 1)]
        be.cmd_wait(c); be.cmd_free(c)
        for b, m in zip(bufs, (self.k, self.v)):
            got = np.empty((self.heads, hi - lo, HD), io_np(io))
            be.buf_download(b, 0, got)
            assert np.array_equal(from_io(got, io).astype(np.float64), m.values(lo, hi))


# ---- append and read ----------------------------------------------------------------------
@pytest.mark.parametrize("paged", [False, True], ids=["plain", "arena"])
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads,base,rows,pad", [(1, 0, 1, 0), (4, 63, 1, 0), (2, 64, 1, 8), (3, 5, 200, 40), (2, 0, 64, 0), (4, 100, 29, 0),
                                                 (1, 127, 130, 16), (2, 0, 300, 0)])
def test_append(be, paged, io, heads, base, rows, pad):
    rng = np.random.default_rng(heads * 1000 + base + rows)
    with Bufs(be) as B:
        p = Pair(be, B, heads, base + rows + 41, paged, seed=7)
        c = be.cmd_begin()
        if base:
            assert p.append(c, B, draw_kv(rng, base, heads), draw_kv(rng, base, heads), 0, F32)
        assert p.append(c, B, draw_kv(rng, rows, heads), draw_kv(rng, rows, heads) * 4, base, io, pad)
        be.cmd_wait(c); be.cmd_free(c)
        p.check(be, B, base + rows)
        p.check(be, B, base + rows, lo=base // 2, io=BF16)
        if not paged:                                       # the bytes themselves: nothing else was written
            for b, m in zip(p.bufs, (p.k, p.v)):
                got = np.empty(p.bytes, np.uint8)
                be.buf_download(b, 0, got)
                want = m.layer_bytes()
                nb = -(-(base + rows) // 64)                # blocks never written keep the buffer's zeros
                e = want[m.codes.size:m.codes.size + m.exps.size].reshape(heads, -1)
                e[:, nb:] = 0
                assert np.array_equal(got, want)


def test_one_token_at_a_time_with_growing_rows(be):
    """Every append but the first meets a block that holds rows; some rows force it to a larger exponent."""
    rng = np.random.default_rng(11)
    with Bufs(be) as B:
        p = Pair(be, B, 2, 200, True, seed=3)
        c = be.cmd_begin()
        for t in range(140):
            f = 2.0 ** int(rng.integers(-6, 7)) if t % 3 == 0 else 1.0
            assert p.append(c, B, draw_kv(rng, 1, 2) * np.float32(f), draw_kv(rng, 1, 2) / np.float32(f), t, F32 if t & 1 else BF16)
        be.cmd_wait(c); be.cmd_free(c)
        p.check(be, B, 140)


def test_sizes_at_the_ends_of_the_range(be):
    rng = np.random.default_rng(12)
    rows = []
    for f in (0.0, 1e-30, 1e-18, 1e-3, 1.0, 3e38):
        x = np.clip(rng.standard_normal((64, 1, HD)), -1, 1) * f
        rows.append(synth.bf16_round(x.astype(np.float32)))
    x = np.concatenate(rows)
    x[70, 0, 3] = -0.0
    with Bufs(be) as B:
        p = Pair(be, B, 1, 400, False)
        c = be.cmd_begin()
        assert p.append(c, B, x, x[::-1].copy(), 0, F32)
        be.cmd_wait(c); be.cmd_free(c)
        assert p.k.exps[0, 0] == M.E_MIN and p.k.exps[0, 5] == M.E_MAX
        p.check(be, B, 384)


def test_nonfinite_rows_are_reported(be):
    rng = np.random.default_rng(13)
    for bad, io in ((np.nan, F32), (np.inf, F32), (-np.inf, BF16), (np.nan, BF16)):
        k, v = draw_kv(rng, 5, 2), draw_kv(rng, 5, 2)
        v[3, 1, 17] = bad
        with Bufs(be) as B:
            p = Pair(be, B, 2, 64, False)
            c = be.cmd_begin()
            wide = [to_io(x.reshape(5, -1), F32) for x in (k, v)] if io == F32 else [
                np.where(np.isnan(x), 0x7FC0, np.where(np.isinf(x), np.where(x < 0, 0xFF80, 0x7F80), synth.f32_to_bf16_bits(np.nan_to_num(x, posinf=0, neginf=0)))).astype(np.uint16).reshape(5, -1)
                for x in (k, v)]
            refs = [QwRef(B.device(w), 0) for w in wide]
            assert be.op_kv8_write(c, p.kr, p.vr, *refs, 5, 2, HD, 64, 0, 512, io)
            assert "NaN or infinite" in be.cmd_wait(c, check=False)
            be.cmd_free(c)
            p.k.append(k, 0); p.v.append(v, 0)
            p.check(be, B, 5)


def test_rewind_overwrites(be):
    rng = np.random.default_rng(14)
    with Bufs(be) as B:
        p = Pair(be, B, 2, 256, True)
        c = be.cmd_begin()
        assert p.append(c, B, draw_kv(rng, 150, 2), draw_kv(rng, 150, 2), 0, F32)
        assert p.append(c, B, draw_kv(rng, 10, 2) * 64, draw_kv(rng, 10, 2), 100, F32)     # the block keeps the larger exponent
        assert p.append(c, B, draw_kv(rng, 3, 2) / 64, draw_kv(rng, 3, 2), 101, BF16)
        assert p.append(c, B, draw_kv(rng, 70, 2) / 64, draw_kv(rng, 70, 2), 64, F32)      # begins its block: exponent forgotten
        be.cmd_wait(c); be.cmd_free(c)
        p.check(be, B, 134)


def test_batch_append_over_64_sequences(be):
    rng = np.random.default_rng(15)
    n, rows, heads, ctx = 70, 3, 2, 200
    with Bufs(be) as B:
        pool = be.kv_pool_alloc(64 << 20, 5)
        ps = [Pair(be, B, heads, ctx, i % 3 > 0, pool=pool) for i in range(n)]
        c = be.cmd_begin()
        bases = [int(rng.integers(0, 190)) if i % 2 else 64 * (i % 3) for i in range(n)]
        for p, b in zip(ps, bases):
            if b:
                assert p.append(c, B, draw_kv(rng, b, heads), draw_kv(rng, b, heads), 0, F32)
        ks, vs = [draw_kv(rng, rows, heads) for _ in range(n)], [draw_kv(rng, rows, heads) for _ in range(n)]
        kr, vr = ([QwRef(B.device(to_io(x.reshape(rows, -1), BF16)), 0) for x in xs] for xs in (ks, vs))
        assert be.op_kv8_write_batch(c, [p.kr for p in ps], [p.vr for p in ps], kr, vr, bases, rows, heads, HD, ctx, heads * HD, BF16)
        be.cmd_wait(c); be.cmd_free(c)
        for p, b, k, v in zip(ps, bases, ks, vs):
            p.k.append(k, b); p.v.append(v, b)
            p.check(be, B, b + rows)
        for b in B.all:
            be.buf_free(b)
        B.all = [pool]


def test_unmapped_pages_read_as_zeros(be):
    rng = np.random.default_rng(16)
    with Bufs(be) as B:
        p = Pair(be, B, 2, 600, True, layers=3, layer=1)
        c = be.cmd_begin()
        assert p.append(c, B, draw_kv(rng, 10, 2), draw_kv(rng, 10, 2), 256, F32)
        be.cmd_wait(c); be.cmd_free(c)
        p.check(be, B, 600)
        assert be.kv_arena_pages_in_use(p.bufs[0]) == 2
        be.kv_arena_trim(p.bufs[0], 256)
        assert be.kv_arena_pages_in_use(p.bufs[0]) == 0


# ---- attention ---------------------------------------------------------------------------------
def run_attn(be, rng, rows, base, qh, heads, io, gate, paged, spread=0.0, scale=1 / 16.0, poison=True, q=None, kv=None, seed=0):
    n = base + rows
    ctx = n + 45
    with Bufs(be) as B:
        p = Pair(be, B, heads, ctx, paged, seed=seed)
        c = be.cmd_begin()
        k, v = kv if kv else (draw_kv(rng, n, heads, spread), draw_kv(rng, n, heads, spread))
        assert p.append(c, B, k, v, 0, F32)
        be.cmd_wait(c); be.cmd_free(c)
        if poison and not paged:                            # positions past the last key: NaN codes, wild exponents
            for b, m in zip(p.bufs, (p.k, p.v)):
                raw = m.layer_bytes()
                codes = raw[:m.codes.size].reshape(heads, ctx, HD)
                codes[:, n:] = rng.choice(np.array([0x7F, 0xFF, 0x7E, 0x80], np.uint8), codes[:, n:].shape)
                raw[m.codes.size:m.codes.size + m.exps.size].reshape(heads, -1)[:, -(-n // 64):] = 255
                be.buf_upload(b, 0, raw)
        if q is None:
            q = synth.bf16_round((rng.standard_normal((rows, qh, HD)) * 1.5).astype(np.float32))
        if io == F32:
            q = (q * np.float32(1.0001)).astype(np.float32)  # not a bf16 number
        gt = synth.bf16_round(rng.standard_normal((rows, qh, 512)).astype(np.float32)) if gate else None
        qb, gb = B.device(to_io(q, io)), B.device(to_io(gt, io)) if gate else None
        el = 2 if io == BF16 else 4
        ob = B.device(np.full((rows + 1, qh, HD), 0x4141, io_np(io)))
        c = be.cmd_begin()
        gr = QwRef(gb, 256 * el) if gate else NULL_REF       # the gate half of [q | gate] rows
        for _ in range(2):                                   # the second call finds the first one's scratch
            assert be.op_attn_kv8(c, QwRef(ob, 0), gr, QwRef(qb, 0), p.kr, p.vr, rows, qh, heads, HD, ctx, base, scale, 512, io)
        be.cmd_wait(c); be.cmd_free(c)
        got = np.empty((rows + 1, qh, HD), io_np(io))
        be.buf_download(ob, 0, got)
        assert np.all(got[rows] == np.full((), 0x4141, io_np(io)))        # the row behind the last
        want = M.attention(q, p.k.values(0, n), p.v.values(0, n), base, scale, gt[..., 256:] if gate else None)
        return from_io(got[:rows], io).astype(np.float64), want


def check_attn(got, want, io, many=False):
    assert np.isfinite(got).all()
    if io == F32:
        assert rel_l2(got, want) < 1e-5 and max_rel_err(got, want) < 1e-4
    elif many:
        assert max_rel_err(got, want) <= 1e-2 and rel_l2(got, want) < 5e-3
    else:
        assert max_rel_err(got, want) <= 2.0 ** -8 + 2.0 ** -10


CASES = [  # rows, base, q_heads, kv_heads
    (1, 0, 1, 1), (1, 0, 8, 2), (1, 1, 16, 4), (1, 31, 16, 4), (1, 32, 24, 4), (1, 63, 6, 1), (1, 64, 12, 2), (1, 127, 16, 2), (1, 1000, 24, 4),
    (1, 5000, 16, 4), (2, 0, 24, 4), (4, 61, 24, 4), (4, 3000, 24, 4), (5, 130, 21, 3), (3, 700, 16, 1), (16, 40, 4, 1), (8, 2000, 8, 8),
    (2, 333, 32, 1), (64, 0, 1, 1), (11, 97, 7, 7)]


@pytest.mark.parametrize("rows,base,qh,heads", CASES)
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_attn_few_rows(be, io, rows, base, qh, heads):
    rng = np.random.default_rng(rows * 7919 + base * 31 + qh)
    got, want = run_attn(be, rng, rows, base, qh, heads, io, gate=(base + qh) % 2 == 0, paged=base % 3 == 1, seed=9)
    check_attn(got, want, io, many=io == BF16 and rows * qh // heads > 64)


@pytest.mark.parametrize("rows,base,qh,heads", [(40, 0, 8, 2), (128, 0, 4, 1), (129, 77, 12, 2), (300, 1000, 6, 1), (65, 63, 16, 4)])
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("paged", [False, True], ids=["plain", "arena"])
def test_attn_many_rows(be, io, paged, rows, base, qh, heads):
    rng = np.random.default_rng(rows + base)
    got, want = run_attn(be, rng, rows, base, qh, heads, io, gate=rows % 2 == 0, paged=paged, seed=4)
    check_attn(got, want, io, many=True)


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 4, 130])
def test_attn_blocks_of_very_different_size(be, io, rows):
    """Exponents that change from block to block by up to 2^16, a block of zeros among the values."""
    rng = np.random.default_rng(21 + rows)
    base = 900
    k, v = draw_kv(rng, base + rows, 2), draw_kv(rng, base + rows, 2, spread=8)
    v[128:192] = 0
    got, want = run_attn(be, rng, rows, base, 8, 2, io, True, rows == 4, kv=(k, v))
    check_attn(got, want, io, many=rows > 16)


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_attn_one_key_outweighs_all_and_has_no_value(be, io):
    """The first key takes nearly the whole softmax and its value is zero: what is left of the output is the many
    small weights (2^-20 of the largest), which must not be flushed."""
    rng = np.random.default_rng(23)
    base = 6000
    q = np.zeros((1, 2, HD), np.float32); q[..., 0] = 14.0
    k = np.zeros((base + 1, 1, HD), np.float32); k[0, 0, 0] = 16.0
    v = draw_kv(rng, base + 1, 1) + 3
    v = synth.bf16_round(v)
    v[:64] = 0
    got, want = run_attn(be, rng, 1, base, 2, 1, io, False, False, q=q, kv=(k, v))
    check_attn(got, want, io)


@pytest.mark.parametrize("rows", [1, 5, 200])
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_attn_nan_query_stays_in_its_row(be, io, rows):
    rng = np.random.default_rng(25)
    qh = 6
    q = synth.bf16_round(rng.standard_normal((rows, qh, HD)).astype(np.float32))
    n = 100 + rows
    ctx = n + 3
    with Bufs(be) as B:
        p = Pair(be, B, 2, ctx, False)
        c = be.cmd_begin()
        assert p.append(c, B, draw_kv(rng, n, 2), draw_kv(rng, n, 2), 0, F32)
        bits = to_io(q, io)
        bits = bits.view(np.uint32).copy() if io == F32 else bits.copy()
        bits[rows // 2, 3, 7] = 0x7FC00000 if io == F32 else 0x7FC0
        qb = B.device(bits)
        ob = B.device(np.zeros((rows, qh, HD), io_np(io)))
        assert be.op_attn_kv8(c, QwRef(ob, 0), NULL_REF, QwRef(qb, 0), p.kr, p.vr, rows, qh, 2, HD, ctx, 100, 1 / 16.0, 256, io)
        be.cmd_wait(c); be.cmd_free(c)
        got = np.empty((rows, qh, HD), io_np(io))
        be.buf_download(ob, 0, got)
        got = from_io(got, io)
        want = M.attention(q, p.k.values(0, n), p.v.values(0, n), 100, 1 / 16.0)
    assert np.isnan(got[rows // 2, 3]).all()
    rest = np.ones((rows, qh), bool); rest[rows // 2, 3] = False
    check_attn(got[rest], want[rest], io, many=rows > 16)


@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0])
def test_attn_other_scales(be, scale):
    rng = np.random.default_rng(26)
    got, want = run_attn(be, rng, 2, 200, 4, 2, F32, False, False, scale=scale)
    assert rel_l2(got, want) < (1e-4 if scale == 1.0 else 1e-5)      # scale 1: arguments up to ~500, 16 times the 30 above


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 3])
def test_attn_batch(be, io, rows):
    """70 sequences of different depth, in a shared pool, arenas of their own and plain buffers: several launches."""
    rng = np.random.default_rng(27)
    n, qh, heads, ctx = 70, 8, 2, 700
    bases = [int(b) for b in rng.integers(0, 690, n)]
    with Bufs(be) as B:
        pool = be.kv_pool_alloc(64 << 20, 5)
        ps = [Pair(be, B, heads, ctx, i % 5 > 0, pool=None if i % 7 == 3 else pool) for i in range(n)]
        c = be.cmd_begin()
        qs, outs, gates, want = [], [], [], []
        for i, (p, b) in enumerate(zip(ps, bases)):
            assert p.append(c, B, draw_kv(rng, b + rows, heads), draw_kv(rng, b + rows, heads), 0, F32)
            q = synth.bf16_round(rng.standard_normal((rows, qh, HD)).astype(np.float32))
            g = synth.bf16_round(rng.standard_normal((rows, qh, HD)).astype(np.float32)) if i % 2 else None
            qs.append(QwRef(B.device(to_io(q, io)), 0))
            gates.append(QwRef(B.device(to_io(g, io)), 0) if i % 2 else NULL_REF)
            outs.append(QwRef(B.device(np.zeros((rows, qh, HD), io_np(io))), 0))
            want.append(M.attention(q, p.k.values(0, b + rows), p.v.values(0, b + rows), b, 1 / 16.0, g))
        assert be.op_attn_kv8_batch(c, outs, gates, qs, [p.kr for p in ps], [p.vr for p in ps], bases, rows, qh, heads, HD, ctx, 1 / 16.0, HD, io)
        be.cmd_wait(c); be.cmd_free(c)
        for o, w in zip(outs, want):
            got = np.empty((rows, qh, HD), io_np(io))
            be.buf_download(o.buf, 0, got)
            check_attn(from_io(got, io).astype(np.float64), w, io)
        for b in B.all:
            be.buf_free(b)
        B.all = [pool]


@pytest.mark.parametrize("rows,base,qh,heads", [(300, 700, 9, 3), (400, 300, 15, 3), (600, 40, 32, 1), (1200, 0, 24, 4), (170, 2300, 21, 3)])
def test_attn_many_rows_of_odd_groupings(be, rows, base, qh, heads):
    """Groupings that do not divide a tile of 128 query rows, one and several shares of the keys."""
    rng = np.random.default_rng(rows + qh)
    got, want = run_attn(be, rng, rows, base, qh, heads, BF16, gate=heads == 3, paged=rows % 200 > 0, spread=3.0, seed=6)
    check_attn(got, want, BF16, many=True)


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.25, 1e-14])
@pytest.mark.parametrize("rows,base", [(400, 300), (1000, 0)])
def test_attn_many_rows_other_scales(be, rows, base, scale):
    rng = np.random.default_rng(33)
    got, want = run_attn(be, rng, rows, base, 8, 2, BF16, True, False, scale=scale)
    check_attn(got, want, BF16, many=True)


@pytest.mark.parametrize("rows", [1, 6, 300])
@pytest.mark.parametrize("kinds", [(True, False), (False, True)], ids=["arena-plain", "plain-arena"])
def test_attn_keys_and_values_in_caches_of_different_kinds(be, kinds, rows):
    rng = np.random.default_rng(34)
    heads, qh, base = 3, 6, 500
    n, ctx = base + rows, base + rows + 77
    with Bufs(be) as B:
        ps = [Pair(be, B, heads, ctx, paged, seed=8) for paged in kinds]
        k, v = draw_kv(rng, n, heads), draw_kv(rng, n, heads)
        c = be.cmd_begin()
        kr, vr = (QwRef(B.device(x.reshape(n, -1)), 0) for x in (k, v))
        assert be.op_kv8_write(c, ps[0].kr, ps[1].vr, kr, vr, n, heads, HD, ctx, 0, heads * HD, F32)
        ps[0].k.append(k, 0); ps[1].v.append(v, 0)
        q = synth.bf16_round(rng.standard_normal((rows, qh, HD)).astype(np.float32))
        qb, ob = B.device(to_io(q, BF16)), B.device(np.zeros((rows, qh, HD), np.uint16))
        assert be.op_attn_kv8(c, QwRef(ob, 0), NULL_REF, QwRef(qb, 0), ps[0].kr, ps[1].vr, rows, qh, heads, HD, ctx, base, 1 / 16.0, HD, BF16)
        be.cmd_wait(c); be.cmd_free(c)
        got = np.empty((rows, qh, HD), np.uint16)
        be.buf_download(ob, 0, got)
        check_attn(from_io(got, BF16).astype(np.float64), M.attention(q, ps[0].k.values(0, n), ps[1].v.values(0, n), base, 1 / 16.0), BF16, many=rows > 16)


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,base", [(1, 40), (6, 900), (300, 700), (1000, 0)])
def test_attn_nan_and_infinite_gates_stay_in_their_elements(be, io, rows, base):
    rng = np.random.default_rng(35)
    heads, qh = 2, 8
    n = base + rows
    with Bufs(be) as B:
        p = Pair(be, B, heads, n, False)
        c = be.cmd_begin()
        assert p.append(c, B, draw_kv(rng, n, heads), draw_kv(rng, n, heads), 0, F32)
        q = synth.bf16_round(rng.standard_normal((rows, qh, HD)).astype(np.float32))
        g = synth.bf16_round(rng.standard_normal((rows, qh, HD)).astype(np.float32))
        g[rows // 2, 3, 8] = np.inf
        g[rows // 2, 3, 10] = -np.inf
        g[0, 5, 200] = 300.0
        want = M.attention(q, p.k.values(0, n), p.v.values(0, n), base, 1 / 16.0, np.clip(g, -700, 700))
        bits = to_io(g, io)
        bits = bits.view(np.uint32).copy() if io == F32 else bits.copy()
        bits[rows // 2, 3, 6] = bits[rows // 2, 3, 13] = 0x7FC00000 if io == F32 else 0x7FC0
        ob = B.device(np.zeros((rows, qh, HD), io_np(io)))
        assert be.op_attn_kv8(c, QwRef(ob, 0), QwRef(B.device(bits), 0), QwRef(B.device(to_io(q, io)), 0), p.kr, p.vr, rows, qh, heads, HD, n, base, 1 / 16.0, HD, io)
        be.cmd_wait(c); be.cmd_free(c)
        got = np.empty((rows, qh, HD), io_np(io))
        be.buf_download(ob, 0, got)
        got = from_io(got, io).astype(np.float64)
    odd = np.zeros(got.shape, bool)
    odd[rows // 2, 3, [6, 13]] = True
    assert np.array_equal(np.isnan(got), odd)
    got[odd] = want[odd]
    check_attn(got, want, io, many=rows > 16)


@pytest.mark.parametrize("gate_stride", [HD, 260, 512])
def test_attn_batch_of_many_rows(be, gate_stride):
    """A tile kernel's launch per sequence, one after the other over the same scratch; 260: gate rows that the copy engine
    does not take."""
    rng = np.random.default_rng(36)
    rows, qh, heads, bases = 150, 8, 2, [2500, 0, 1201]
    ctx = 2800
    with Bufs(be) as B:
        ps = [Pair(be, B, heads, ctx, i != 1, seed=i) for i in range(3)]
        c = be.cmd_begin()
        qs, outs, gates, want = [], [], [], []
        for p, b in zip(ps, bases):
            assert p.append(c, B, draw_kv(rng, b + rows, heads), draw_kv(rng, b + rows, heads), 0, BF16)
            q = synth.bf16_round(rng.standard_normal((rows, qh, HD)).astype(np.float32))
            g = synth.bf16_round(rng.standard_normal((rows, qh, gate_stride)).astype(np.float32))
            qs.append(QwRef(B.device(to_io(q, BF16)), 0))
            gates.append(QwRef(B.device(to_io(g, BF16)), 0))
            outs.append(QwRef(B.device(np.zeros((rows, qh, HD), np.uint16)), 0))
            want.append(M.attention(q, p.k.values(0, b + rows), p.v.values(0, b + rows), b, 1 / 16.0, g[..., :HD]))
        assert be.op_attn_kv8_batch(c, outs, gates, qs, [p.kr for p in ps], [p.vr for p in ps], bases, rows, qh, heads, HD, ctx, 1 / 16.0, gate_stride, BF16)
        be.cmd_wait(c); be.cmd_free(c)
        for o, w in zip(outs, want):
            got = np.empty((rows, qh, HD), np.uint16)
            be.buf_download(o.buf, 0, got)
            check_attn(from_io(got, BF16).astype(np.float64), w, BF16, many=True)


def test_call_refused_for_its_last_sequence_encodes_nothing(be):
    rng = np.random.default_rng(37)
    rows, qh, heads, ctx = 150, 8, 2, 400
    with Bufs(be) as B:
        ps = [Pair(be, B, heads, ctx, False) for _ in range(66)]
        x = QwRef(B.device(rng.standard_normal((rows, heads * HD)).astype(np.float32)), 0)
        q = QwRef(B.device(np.zeros((rows, qh, HD), np.uint16)), 0)
        outs = [QwRef(B.device(np.zeros((rows, qh, HD), np.uint16)), 0) for _ in range(2)] + [QwRef(B.device(np.zeros(64, np.uint16)), 0)]
        launches = be.launch_count()
        c = be.cmd_begin()
        assert not be.op_kv8_write_batch(c, [p.kr for p in ps], [p.vr for p in ps], [x] * 66, [x] * 65 + [NULL_REF], [0] * 66, 1, heads, HD, ctx, heads * HD, F32)
        be.cmd_wait(c, check=False); be.cmd_free(c)
        c = be.cmd_begin()
        assert not be.op_attn_kv8_batch(c, outs, None, [q] * 3, [p.kr for p in ps[:3]], [p.vr for p in ps[:3]], [200] * 3, rows, qh, heads, HD, ctx, 0.1, HD, BF16)
        be.cmd_wait(c, check=False); be.cmd_free(c)
        assert be.launch_count() == launches


def test_captured_prompt_replays_beside_an_eager_one(be):
    """Many rows, keys in shares: the graph's partial sums and those of a call on another stream lie apart."""
    import torch
    rng = np.random.default_rng(38)
    rows, qh, heads, base = 170, 8, 2, 2000
    n = base + rows
    with Bufs(be) as B:
        p = Pair(be, B, heads, n, True)
        c0 = be.cmd_begin()
        assert p.append(c0, B, draw_kv(rng, n, heads), draw_kv(rng, n, heads), 0, F32)
        be.cmd_wait(c0); be.cmd_free(c0)
        k, v = p.k.values(0, n), p.v.values(0, n)
        qs = [synth.bf16_round(rng.standard_normal((rows, qh, HD)).astype(np.float32)) for _ in range(3)]
        want = [M.attention(q, k, v, base, 1 / 16.0) for q in qs]
        t = [torch.from_numpy(q).to("cuda", torch.bfloat16) for q in qs]
        live = t[0].clone()
        outs = [torch.zeros(rows, qh, HD, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        ref = lambda x: QwRef(be.buf_wrap_device(x.data_ptr(), x.numel() * 2), 0)  # noqa: E731
        r_live, r_two, r_out = ref(live), ref(t[2]), [ref(o) for o in outs]
        B.all += [r_live.buf, r_two.buf] + [r.buf for r in r_out]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        cs = [be.cmd_begin(s.cuda_stream) for s in streams]
        call = lambda c, q, o: be.op_attn_kv8(c, o, NULL_REF, q, p.kr, p.vr, rows, qh, heads, HD, n, base, 1 / 16.0, HD, BF16)  # noqa: E731
        assert call(cs[0], r_live, r_out[0])
        be.cmd_wait(cs[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            assert call(cs[0], r_live, r_out[0])
        live.copy_(t[1])
        torch.cuda.synchronize()
        for _ in range(10):
            with torch.cuda.stream(streams[0]):
                g.replay()
            assert call(cs[1], r_two, r_out[1])
        torch.cuda.synchronize()
        be.cmd_wait(cs[1])
        for o, w in zip(outs, want[1:]):
            check_attn(o.float().cpu().numpy().astype(np.float64), w, BF16, many=True)
        g.reset()
        for c in cs:
            be.cmd_free(c)


def test_offsets_past_32_bits(be):
    """Codes that lie more than 4 GB into the buffer; the untouched positions are zeros and take their share."""
    rng = np.random.default_rng(28)
    heads, ctx, base, rows = 8, 2_200_000, 2_199_000, 2
    k, v = draw_kv(rng, rows, heads), draw_kv(rng, rows, heads) * 64
    q = synth.bf16_round((rng.standard_normal((rows, heads, HD)) * 3).astype(np.float32))
    with Bufs(be) as B:
        kb, vb = (be.buf_alloc_device(be.kv8_layer_bytes(heads, ctx)) for _ in range(2))
        B.all += [kb, vb]
        refs = [QwRef(B.device(x.reshape(rows, -1)), 0) for x in (k, v)]
        ob = B.device(np.zeros((rows, heads, HD), np.float32))
        rb = [B.device(np.zeros((heads, 72, HD), np.float32)) for _ in range(2)]
        qb = B.device(q)
        c = be.cmd_begin()
        assert be.op_kv8_write(c, QwRef(kb, 0), QwRef(vb, 0), *refs, rows, heads, HD, ctx, base, heads * HD, F32)
        for b, r in zip((kb, vb), rb):
            assert be.op_kv8_read(c, QwRef(r, 0), QwRef(b, 0), base - 70, 72, heads, HD, ctx, F32)
        assert be.op_attn_kv8(c, QwRef(ob, 0), NULL_REF, QwRef(qb, 0), QwRef(kb, 0), QwRef(vb, 0), rows, heads, heads, HD, ctx, base, 1.0, HD, F32)
        be.cmd_wait(c); be.cmd_free(c)
        mk, mv = M.Cache(heads, 130), M.Cache(heads, 130)
        off = base % 64
        mk.append(k, off); mv.append(v, off)
        got = np.empty((heads, 72, HD), np.float32)
        for r, m in zip(rb, (mk, mv)):
            be.buf_download(r, 0, got)
            assert not got[:, :70].any() and np.array_equal(got[:, 70:].astype(np.float64), m.values(off, off + rows))
        kk, vv = mk.values(off, off + rows), mv.values(off, off + rows)
        want = np.empty((rows, heads, HD))
        for r in range(rows):
            for h in range(heads):
                s = kk[h, :r + 1] @ q[r, h].astype(np.float64)
                m = max(s.max(), 0.0)
                w = np.exp(s - m)
                want[r, h] = w @ vv[h, :r + 1] / (w.sum() + base * np.exp(-m))
        got = np.empty((rows, heads, HD), np.float32)
        be.buf_download(ob, 0, got)
        # arguments of the exponential up to ~300 here, and 2.2 million equal weights added in f32
        assert rel_l2(got, want) < 2e-4


def test_repeated_calls_agree_bit_for_bit(be):
    rng = np.random.default_rng(29)
    n, heads = 3000, 4
    with Bufs(be) as B:
        p = Pair(be, B, heads, n, True)
        c = be.cmd_begin()
        assert p.append(c, B, draw_kv(rng, n, heads), draw_kv(rng, n, heads), 0, F32)
        q = B.device(rng.standard_normal((1, 16, HD)).astype(np.float32))
        outs = [B.device(np.zeros((1, 16, HD), np.float32)) for _ in range(6)]
        for o in outs:
            assert be.op_attn_kv8(c, QwRef(o, 0), NULL_REF, QwRef(q, 0), p.kr, p.vr, 1, 16, heads, HD, n, n - 1, 1 / 16.0, HD, F32)
        be.cmd_wait(c); be.cmd_free(c)
        got = np.empty((6, 1, 16, HD), np.float32)
        for i, o in enumerate(outs):
            be.buf_download(o, 0, got[i])
    assert got.any() and all(np.array_equal(got[0], g) for g in got[1:])


# ---- the operators together ----------------------------------------------------------------
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_prompt_then_decode_steps(be, io):
    """What a layer does with an 8-bit cache: rotary positions on q and k (slices of the joint projection), append,
    gated attention; a prompt of 90, then a verify step of 4 of which 2 stay, then single tokens."""
    rng = np.random.default_rng(30)
    qh, heads, ctx, rot = 8, 2, 300, 64
    inv, amp = be.rope_scaled_tables(rot, 1e6, 3, 4.0, 32768)
    width = qh * 512 + 2 * heads * HD
    el = 2 if io == BF16 else 4
    with Bufs(be) as B:
        p = Pair(be, B, heads, ctx, True, seed=5)
        fb = B.device(inv)
        c = be.cmd_begin()
        base = 0
        for rows, keep in ((90, 90), (4, 2), (1, 1), (1, 1)):
            x = synth.bf16_round(rng.standard_normal((rows, width)).astype(np.float32))
            pos = (np.arange(rows) + base + 100000).astype(np.int32)
            xb, pb = B.device(to_io(x, io)), B.device(pos)
            qb, kb = B.device(np.zeros((rows, qh, HD), io_np(io))), B.device(np.zeros((rows, heads, HD), io_np(io)))
            ob = B.device(np.zeros((rows, qh, HD), io_np(io)))
            # [q | k | v | gate] columns
            cq, ck, cv, cg = 0, qh * HD, (qh + heads) * HD, (qh + 2 * heads) * HD
            assert be.op_rope(c, QwRef(qb, 0), QwRef(xb, cq * el), QwRef(pb, 0), QwRef(fb, 0), rows, qh, HD, rot, 0, qh * HD, width, amp, io)
            assert be.op_rope(c, QwRef(kb, 0), QwRef(xb, ck * el), QwRef(pb, 0), QwRef(fb, 0), rows, heads, HD, rot, 0, heads * HD, width, amp, io)
            # keys from their own buffer, values in place in the projection: the same row stride is asked for, so values are copied
            vb = B.device(to_io(x[:, cv:cv + heads * HD], io))
            assert be.op_kv8_write(c, p.kr, p.vr, QwRef(kb, 0), QwRef(vb, 0), rows, heads, HD, ctx, base, heads * HD, io)
            gb = B.device(to_io(x[:, cg:].reshape(rows, qh, HD), io))
            assert be.op_attn_kv8(c, QwRef(ob, 0), QwRef(gb, 0), QwRef(qb, 0), p.kr, p.vr, rows, qh, heads, HD, ctx, base, 1 / 16.0, HD, io)
            be.cmd_wait(c)
            kq = [np.empty((rows, n, HD), io_np(io)) for n in (qh, heads)]
            be.buf_download(qb, 0, kq[0]); be.buf_download(kb, 0, kq[1])
            rq, rk = (from_io(a, io) for a in kq)
            wq, wk = (M.rope(x[:, a:a + n * HD].reshape(rows, n, HD), pos, inv, rot, False, amp) for a, n in ((cq, qh), (ck, heads)))
            tol = 2.0 ** -8 if io == BF16 else 2e-6
            assert max_rel_err(rq, wq) <= tol and max_rel_err(rk, wk) <= tol
            p.k.append(rk, base); p.v.append(x[:, cv:cv + heads * HD].reshape(rows, heads, HD), base)
            got = np.empty((rows, qh, HD), io_np(io))
            be.buf_download(ob, 0, got)
            n = base + rows
            want = M.attention(rq, p.k.values(0, n), p.v.values(0, n), base, 1 / 16.0, x[:, cg:].reshape(rows, qh, HD))
            check_attn(from_io(got, io).astype(np.float64), want, io, many=rows > 16)
            base += keep
        be.cmd_free(c)


# ---- streams, graphs, refusals -----------------------------------------------------------------
def test_captured_step_replays(be):
    """Append and attention captured on a caller's stream and replayed on new inputs; a second graph on a command
    buffer of its own runs beside it."""
    import torch
    rng = np.random.default_rng(31)
    heads, qh, ctx, base = 2, 8, 1000, 777
    with Bufs(be) as B:
        sets = []
        for _ in range(2):
            p = Pair(be, B, heads, ctx, True)
            s = torch.cuda.Stream()
            c = be.cmd_begin(s.cuda_stream)
            assert p.append(c, B, draw_kv(rng, base, heads), draw_kv(rng, base, heads), 0, F32)
            t = {n: torch.zeros(1, w, HD, device="cuda") for n, w in (("k", heads), ("v", heads), ("q", qh), ("o", qh))}
            r = {n: QwRef(be.buf_wrap_device(x.data_ptr(), x.numel() * 4), 0) for n, x in t.items()}
            B.all += [x.buf for x in r.values()]

            def step():
                assert be.op_kv8_write(c, p.kr, p.vr, r["k"], r["v"], 1, heads, HD, ctx, base, heads * HD, F32)
                assert be.op_attn_kv8(c, r["o"], NULL_REF, r["q"], p.kr, p.vr, 1, qh, heads, HD, ctx, base, 1 / 16.0, HD, F32)
            step()
            be.cmd_wait(c)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step()
            assert be.cmd_error(c) is None
            sets.append((p, c, s, t, g))
        torch.cuda.synchronize()
        want = []
        for p, c, s, t, g in sets:
            x = {n: torch.from_numpy(draw_kv(rng, 1, qh if n in "qo" else heads)) for n in "kvq"}
            for n in x:
                t[n].copy_(x[n])
            k, v = M.Cache(heads, ctx), M.Cache(heads, ctx)
            k.codes[:], k.exps[:], v.codes[:], v.exps[:] = p.k.codes, p.k.exps, p.v.codes, p.v.exps
            k.append(x["k"].numpy(), base); v.append(x["v"].numpy(), base)
            want.append(M.attention(x["q"].numpy(), k.values(0, base + 1), v.values(0, base + 1), base, 1 / 16.0))
        torch.cuda.synchronize()
        for _ in range(20):
            for p, c, s, t, g in sets:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for (p, c, s, t, g), w in zip(sets, want):
            check_attn(t["o"].cpu().numpy().astype(np.float64), w, F32)
        for p, c, s, t, g in sets:
            g.reset()
            be.cmd_free(c)


def test_capture_without_pages_or_scratch_is_refused(be):
    import torch
    with Bufs(be) as B:
        p = Pair(be, B, 2, 1000, True)
        s = torch.cuda.Stream()
        x = torch.zeros(1, 2, HD, device="cuda")
        r = QwRef(be.buf_wrap_device(x.data_ptr(), 2048), 0)
        B.all.append(r.buf)
        torch.cuda.synchronize()
        for op in (lambda c: be.op_kv8_write(c, p.kr, p.vr, r, r, 1, 2, HD, 1000, 0, 512, F32),):
            c = be.cmd_begin(s.cuda_stream)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                x.add_(1)
                ok = op(c)
            assert not ok and "captured" in be.cmd_error(c)
            g.reset()
            be.cmd_free(c)


def test_refusals(be):
    z = NULL_REF
    with Bufs(be) as B:
        p = Pair(be, B, 2, 128, True)
        plain = Pair(be, B, 2, 128, False)
        bf = QwRef(B.arena(1, 2, 128), 0)
        x = QwRef(B.device(np.zeros(16 * 512, np.float32)), 0)
        y = QwRef(B.device(np.zeros(16 * 512, np.float32)), 0)
        small = QwRef(B.device(np.zeros(256, np.float32)), 0)
        pool = be.kv_pool_alloc(1 << 20)
        B.all.append(pool)
        w = lambda c, k=p.kr, v=p.vr, a=x, b=y, rows=1, h=2, hd=HD, ctx=128, base=0, st=512, io=F32: be.op_kv8_write(c, k, v, a, b, rows, h, hd, ctx, base, st, io)  # noqa: E731
        rd = lambda c, d=x, k=p.kr, lo=0, n=4, h=2, hd=HD, ctx=128, io=F32: be.op_kv8_read(c, d, k, lo, n, h, hd, ctx, io)  # noqa: E731
        at = lambda c, o=x, g=z, q=y, k=p.kr, v=p.vr, rows=1, qh=4, h=2, hd=HD, ctx=128, base=0, gs=HD, io=F32: be.op_attn_kv8(c, o, g, q, k, v, rows, qh, h, hd, ctx, base, 0.1, gs, io)  # noqa: E731
        off = lambda r, n: QwRef(r.buf, n)  # noqa: E731
        bad = [
            lambda c: w(c, rows=-1), lambda c: w(c, h=3), lambda c: w(c, hd=128), lambda c: w(c, ctx=64), lambda c: w(c, base=-1), lambda c: w(c, base=128),
            lambda c: w(c, base=2 ** 31 - 1), lambda c: w(c, st=511), lambda c: w(c, st=514), lambda c: w(c, io=2), lambda c: w(c, io=BF16, st=516),
            lambda c: w(c, k=z), lambda c: w(c, a=z), lambda c: w(c, a=small), lambda c: w(c, k=bf, v=bf), lambda c: w(c, v=p.kr), lambda c: w(c, k=off(p.kr, 256)),
            lambda c: w(c, k=QwRef(pool, 0)), lambda c: w(c, k=x), lambda c: w(c, a=off(x, 4)), lambda c: w(c, k=off(plain.kr, 16), v=plain.vr), lambda c: w(c, rows=200, base=0),
            lambda c: rd(c, n=-1), lambda c: rd(c, lo=126), lambda c: rd(c, lo=-1), lambda c: rd(c, d=small), lambda c: rd(c, k=bf), lambda c: rd(c, d=p.kr), lambda c: rd(c, io=7),
            lambda c: at(c, rows=-1), lambda c: at(c, qh=3), lambda c: at(c, qh=0), lambda c: at(c, qh=66), lambda c: at(c, hd=64), lambda c: at(c, base=128), lambda c: at(c, base=-1),
            lambda c: at(c, g=x, gs=255), lambda c: at(c, q=z), lambda c: at(c, o=small), lambda c: at(c, k=bf), lambda c: at(c, v=z), lambda c: at(c, io=3), lambda c: at(c, q=off(y, 8)),
            lambda c: be.op_attn_kv8_batch(c, [x, x], None, [y, y], [p.kr] * 2, [p.vr] * 2, [0, 0], 1, 4, 2, HD, 128, 0.1, HD, F32),
            lambda c: be.op_kv8_write_batch(c, [p.kr] * 2, [p.vr, plain.vr], [x, x], [y, y], [0, 64], 1, 2, HD, 128, 512, F32),
            lambda c: be.op_kv8_write_batch(c, [p.kr, p.vr], [plain.kr, plain.vr][:1] + [p.kr], [x, x], [y, y], [0, 64], 1, 2, HD, 128, 512, F32),
        ]
        launches = be.launch_count()
        for i, f in enumerate(bad):
            c = be.cmd_begin()
            assert not f(c), f"call {i} was taken"
            be.cmd_wait(c, check=False)
            be.cmd_free(c)
        assert be.launch_count() == launches and be.kv_arena_pages_in_use(p.bufs[0]) == 0
        c = be.cmd_begin()                                    # nothing to do is not an error
        assert w(c, rows=0) and rd(c, n=0) and at(c, rows=0)
        assert be.op_attn_kv8_batch(c, [], None, [], [], [], [], 1, 4, 2, HD, 128, 0.1, HD, F32)
        be.cmd_wait(c); be.cmd_free(c)
        # the bf16 ops refuse an 8-bit arena
        for f in (lambda c: be.op_kv_write(c, p.kr, p.vr, x, y, 1, 2, HD, 128, 0), lambda c: be.op_attn_decode(c, x, y, p.kr, p.vr, 1, 4, 2, HD, 128, 0, 0.1)):
            c = be.cmd_begin()
            f(c)
            assert "8-bit" in be.cmd_wait(c, check=False)
            be.cmd_free(c)
        with pytest.raises(RuntimeError):
            be.kv_read(p.bufs[0], 0, 0, 0, 1, 2, 128)
        with pytest.raises(MemoryError):
            be.kv8_arena_alloc(1, 2, 128, 128)
        with pytest.raises(MemoryError):
            be.kv8_arena_alloc_in(x.buf, 1, 2, 128)


def test_attention_over_pages_never_mapped_is_reported(be):
    """Positions whose pages were never mapped: an error string, no fault."""
    with Bufs(be) as B:
        p = Pair(be, B, 1, 512, True)
        x = QwRef(B.device(np.zeros(1024, np.float32)), 0)
        y = QwRef(B.device(np.zeros(1024, np.float32)), 0)
        c = be.cmd_begin()
        assert p.append(c, B, np.ones((4, 1, HD), np.float32), np.ones((4, 1, HD), np.float32), 300, F32)
        assert be.op_attn_kv8(c, x, NULL_REF, y, p.kr, p.vr, 1, 2, 1, HD, 512, 303, 0.1, HD, F32)
        assert "never mapped" in be.cmd_wait(c, check=False)
        be.cmd_free(c)
