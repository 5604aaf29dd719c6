"""The 8-bit cache's boundary without a GPU: header, binding, sizes, frequency tables, and the model the GPU
tests compare with against torch's own e4m3 conversion."""
import ctypes as C
import math
import os
import re
import subprocess

import numpy as np
import pytest

import kv8_model as M
from qwasar_b200 import backend

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declared():
    text = re.sub(r"/\*.*?\*/", "", open(backend.KV8_HEADER).read(), flags=re.S)
    return set(re.findall(r"\b(qw_[a-z0-9_]+)\s*\(", text))


def test_header_binding_and_library_agree():
    lib = C.CDLL(backend.LIB_PATH)
    assert declared() == set(backend.KV8_SIGNATURES)
    for n in declared():
        assert hasattr(lib, n), n


def test_header_compiles_as_c99_and_links(tmp_path):
    src = tmp_path / "kv8.c"
    uses = ", ".join(f"(any_fn){n}" for n in sorted(declared()))
    src.write_text('#include "qwasar_kv8.h"\ntypedef void (*any_fn)(void);\nint main(void) {\n    any_fn f[] = {' + uses +
                   "};\n    return f[0] && qw_kv8_layer_bytes(2, 100, 256) == 51456 ? 0 : 1;\n}\n")
    lib = os.path.join(ROOT, "qwasar_b200")
    cmd = ["gcc", "-std=c99", "-pedantic", "-Wall", "-Wextra", "-Werror", "-I" + os.path.join(ROOT, "include"), str(src), "-o",
           str(tmp_path / "kv8"), "-L" + lib, "-lqwasar_cuda", "-Wl,-rpath," + lib]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert subprocess.run([str(tmp_path / "kv8")]).returncode == 0


@pytest.mark.parametrize("h,ctx", [(1, 1), (2, 64), (4, 65), (8, 262144), (3, 1000)])
def test_layer_bytes(h, ctx):
    lib = backend.load_library()
    assert lib.qw_kv8_layer_bytes(h, ctx, 256) == -(-(h * ctx * 256 + h * -(-ctx // 64)) // 256) * 256


def test_layer_bytes_refusals():
    lib = backend.load_library()
    for a in [(0, 64, 256), (1, 0, 256), (1, 64, 128), (-1, 64, 256)]:
        assert lib.qw_kv8_layer_bytes(*a) == 0


def test_ops_without_a_command_buffer_decline():
    lib = backend.load_library()
    r = backend.NULL_REF
    assert not lib.qw_op_rope(None, r, r, r, r, 1, 1, 64, 64, 0, 64, 64, 1.0, 0)
    assert not lib.qw_op_kv8_write(None, r, r, r, r, 1, 1, 256, 64, 0, 256, 0)
    assert not lib.qw_op_kv8_write_batch(None, 0, None, None, None, None, None, 1, 1, 256, 64, 256, 0)
    assert not lib.qw_op_kv8_read(None, r, r, 0, 1, 1, 256, 64, 0)
    assert not lib.qw_op_attn_kv8(None, r, r, r, r, r, 1, 1, 1, 256, 64, 0, 1.0, 256, 0)
    assert not lib.qw_op_attn_kv8_batch(None, 0, None, None, None, None, None, None, 1, 1, 1, 256, 64, 1.0, 256, 0)


def tables(kind, rotary=64, theta=1e6, factor=4.0, ctx=32768, fast=32.0, slow=1.0):
    lib = backend.load_library()
    inv, amp = np.zeros(rotary // 2, np.float32), C.c_float(-1)
    ok = lib.qw_rope_scaled_tables(inv.ctypes.data, C.addressof(amp), rotary, theta, kind, factor, ctx, fast, slow)
    return ok, inv, amp.value


def test_plain_linear_and_ntk_tables():
    j = np.arange(32)
    f = 1e6 ** (-2.0 * j / 64)
    eps = 2.0 ** -24                                       # one rounding of an exact product
    ok, inv, amp = tables(backend.ROPE_PLAIN)
    assert ok and amp == 1.0 and np.all(np.abs(inv - f) <= 1.01 * eps * f)
    ok, inv, amp = tables(backend.ROPE_LINEAR)
    assert ok and amp == 1.0 and np.all(np.abs(inv - f / 4) <= 1.01 * eps * f / 4)
    ok, inv, amp = tables(backend.ROPE_NTK)
    g = (1e6 * 4.0 ** (64 / 62)) ** (-2.0 * j / 64)
    assert ok and amp == 1.0 and np.all(np.abs(inv - g) <= 1.01 * eps * g)
    assert abs(inv[31] * 4 / f[31] - 1) < 1e-6 and inv[0] == 1.0      # slowest pair stretched by the factor, fastest kept


def test_band_tables():
    ok, inv, amp = tables(backend.ROPE_BANDS)
    f = 1e6 ** (-2.0 * np.arange(32) / 64)
    turns = 32768 * f / (2 * math.pi)
    assert ok and abs(amp - (0.1 * math.log(4.0) + 1)) < 1e-7
    r = inv / f
    assert np.all(np.abs(r[turns > 40] - 1) < 1e-6) and np.all(np.abs(r[turns < 0.6] - 0.25) < 1e-6)
    assert np.all(np.diff(r) <= 1e-7) and np.any((r > 0.3) & (r < 0.95))
    d = np.diff(r)[(r[1:] < 0.999) & (r[:-1] > 0.251)]      # the ramp is linear in the pair index
    assert np.ptp(d[1:-1]) < 1e-6


@pytest.mark.parametrize("kw", [dict(rotary=63 + 1, theta=0.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(factor=0.0), dict(factor=-2.0),
                                dict(kind=4), dict(kind=-1), dict(kind=2, rotary=2), dict(kind=3, ctx=0), dict(kind=3, fast=1.0, slow=1.0),
                                dict(kind=3, slow=0.0), dict(kind=3, factor=0.5), dict(kind=3, theta=1.0)])
def test_table_refusals(kw):
    assert not tables(kw.pop("kind", 0), **kw)[0]


def test_table_refuses_odd_width_and_null():
    lib = backend.load_library()
    inv = np.zeros(32, np.float32)
    assert not lib.qw_rope_scaled_tables(inv.ctypes.data, None, 63, 1e6, 0, 1.0, 0, 32.0, 1.0)
    assert not lib.qw_rope_scaled_tables(None, None, 64, 1e6, 0, 1.0, 0, 32.0, 1.0)
    assert lib.qw_rope_scaled_tables(inv.ctypes.data, None, 64, 1e6, 0, 1.0, 0, 32.0, 1.0)


def test_model_codes_match_torch():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(5)
    x = np.concatenate([rng.standard_normal(4000) * 2.0 ** rng.integers(-12, 9, 4000), M.VALUES[np.isfinite(M.VALUES)], [0.0, -0.0, 448.0, 2.0 ** -10, 1.5 * 2.0 ** -9]])
    mid = np.sort(M.VALUES[np.isfinite(M.VALUES)])
    x = np.concatenate([x, (mid[1:] + mid[:-1]) / 2]).astype(np.float32)      # every tie
    x = x[np.abs(x) <= 448]
    t = torch.from_numpy(x)
    assert np.array_equal(M.to_code(x), t.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(np.isnan(v), np.isnan(M.VALUES)) and np.array_equal(v[~np.isnan(v)], M.VALUES[~np.isnan(v)])


def test_model_exponent_is_the_smallest_that_fits():
    rng = np.random.default_rng(6)
    for a in list(np.exp(rng.uniform(-30, 30, 200))) + [448.0, 448.0001, 224.0, 1e-30, 3.4e38]:
        e = M.needed(a)
        assert e == M.E_MAX or a <= 448 * 2.0 ** e
        assert e == M.E_MIN or a > 448 * 2.0 ** (e - 1)
