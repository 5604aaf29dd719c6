"""The operators around the 8-bit K/V cache, as they are measured: rotary positions, the append to the
cache, the dequantising read, and attention over it (one token, a few tokens, a batch, a prompt).

`run` is one call (or the write and the read that belong together) in the plain form, elementary torch
operations in 32 bits, or, with `own`, through the C ABI of this framework as its binding exposes it.

The cache format both sides share: one layer is a byte buffer [kv_heads, max_ctx, 256] of e4m3 codes and
behind it one exponent byte (value 2^(byte - 127)) per head and 64-token block, [kv_heads, ceil(max_ctx / 64)],
padded to a multiple of 256 bytes."""
import ctypes
import math

import torch

own = False

HD = 256                 # head width of the attention path
BLOCK = 64               # tokens that share an exponent
E_MIN, E_MAX = -60, 119
DEV = "cuda"


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoded token's query heads, a quarter of each head rotated: the smallest call there is
        dict(name="rope_token", op="rope", rows=1, heads=16, head_dim=256, rotary=64, interleaved=False, bf16=False, pad=0,
             pos0=4096, theta=1e7, factor=1.0),
        # a prompt's query heads, whole head rotated in adjacent pairs, read out of the joint projection's
        # rows, far positions with stretched frequencies
        dict(name="rope_prompt_far", op="rope", rows=4096, heads=24, head_dim=256, rotary=256, interleaved=True, bf16=True, pad=2048,
             pos0=131072, theta=1e7, factor=4.0),
        # one decoded token's append into a block that is partly filled
        dict(name="write_token", op="write", rows=1, kv_heads=4, base=4133, bf16=False, pad=0),
        # a prompt's append
        dict(name="write_prompt", op="write", rows=4096, kv_heads=4, base=0, bf16=True, pad=0),
        # a saved prefix taken back out of the cache, odd length and start
        dict(name="read_odd", op="read", kv_heads=2, n=1001, pos0=37, bf16=False),
        # a long prefix taken out as bf16
        dict(name="read_prefix", op="read", kv_heads=4, n=32768, pos0=0, bf16=True),
        # decode, 4 K keys, f32 activations: the latency case
        dict(name="decode_4k", op="attn", seqs=1, rows=1, q_heads=16, kv_heads=4, base=4096, bf16=False, gate=True, paged=False),
        # decode of eight sequences in a shared page pool, 32 K keys each
        dict(name="decode_32k_batch8", op="attn", seqs=8, rows=1, q_heads=24, kv_heads=4, base=32768, bf16=True, gate=True, paged=True),
        # speculative verify of four draft tokens
        dict(name="verify_32k", op="attn", seqs=1, rows=4, q_heads=24, kv_heads=4, base=32768, bf16=True, gate=False, paged=False),
        # decode at the longest context
        dict(name="decode_262k", op="attn", seqs=1, rows=1, q_heads=16, kv_heads=2, base=262143, bf16=True, gate=True, paged=False),
        # a whole prompt
        dict(name="prefill_4k", op="attn", seqs=1, rows=4096, q_heads=16, kv_heads=4, base=0, bf16=True, gate=True, paged=False),
        # a chunk of a prompt behind a long cached prefix, ragged on both ends
        dict(name="prefill_chunk_16k", op="attn", seqs=1, rows=499, q_heads=24, kv_heads=4, base=16001, bf16=True, gate=True, paged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attn", "attn", "attn"])
    if op == "rope":
        hd = rng.choice([64, 96, 128, 192, 256])
        rotary = 2 * rng.randint(1, hd // 2) if rng.random() < 0.3 else rng.choice([hd // 4, hd // 2, hd])
        return dict(op=op, rows=_log(rng, 1, 4096), heads=rng.randint(1, 24), head_dim=hd, rotary=rotary, interleaved=rng.random() < 0.5,
                    bf16=rng.random() < 0.5, pad=rng.choice([0, 0, 8, 24, 1000]), pos0=_log(rng, 1, 1 << 20) - 1, theta=rng.choice([1e4, 1e6, 1e7]),
                    factor=rng.choice([1.0, 1.0, 2.0, 8.0]))
    kv_heads = rng.choice([1, 2, 4, 4, 8])
    if op == "write":
        return dict(op=op, rows=_log(rng, 1, 16384 // kv_heads), kv_heads=kv_heads, base=rng.choice([0, _log(rng, 1, 8192)]),
                    bf16=rng.random() < 0.5, pad=rng.choice([0, 0, 256, 40]))
    if op == "read":
        return dict(op=op, kv_heads=kv_heads, n=_log(rng, 1, 131072 // kv_heads), pos0=rng.choice([0, _log(rng, 1, 4096)]), bf16=rng.random() < 0.5)
    group = rng.choice([1, 3, 4, 6, 7, 8, 12])
    kv_heads = rng.choice([1, 2, 4, 8]) if group * 8 <= 64 else rng.choice([1, 2, 4])
    kind = rng.choice(["decode", "verify", "prompt"])
    rows = 1 if kind == "decode" else rng.randint(2, 16) if kind == "verify" else _log(rng, 17, 2048)
    seqs = rng.choice([1, 1, 2, 5]) if kind != "prompt" else 1
    most = (1 << 18) // (kv_heads * seqs) if kind != "prompt" else 8192
    if kind == "prompt":                                   # no more products than the largest listed prompt
        most = max(64, min(most, int(1.2e11 / (4 * HD * kv_heads * group * rows)) - rows))
    elif kind == "verify":
        most //= 4
    return dict(op=op, seqs=seqs, rows=rows, q_heads=kv_heads * group, kv_heads=kv_heads, base=rng.choice([0, _log(rng, 1, most), _log(rng, 1, most)]),
                bf16=True if kind == "prompt" else rng.random() < 0.6, gate=rng.random() < 0.6, paged=rng.random() < 0.4)


# ---------------------------------------------------------------------------------------------
# the format, in elementary torch operations
# ---------------------------------------------------------------------------------------------
def _pow2(e):
    """2^e for whole e in [-126, 127], exactly."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _needed(amax):
    """The smallest e with amax <= 448 * 2^e = 1.75 * 2^(e + 8)."""
    u = amax.view(torch.int32)
    return ((u >> 23) - 127 - 8 + ((u & 0x7FFFFF) > 0x600000)).clamp(E_MIN, E_MAX)


def _codes(x, e):
    return (x * _pow2(-e)).to(torch.float8_e4m3fn)


def _layer_bytes(kv_heads, ctx):
    return (kv_heads * ctx * HD + kv_heads * ((ctx + BLOCK - 1) // BLOCK) + 255) // 256 * 256


def _views(buf, kv_heads, ctx):
    """Codes [S, H, ctx, 256] and exponent bytes [S, H, blocks] of the layers in buf [S, layer bytes]."""
    n, b = kv_heads * ctx * HD, (ctx + BLOCK - 1) // BLOCK
    return buf[:, :n].view(-1, kv_heads, ctx, HD), buf[:, n:n + kv_heads * b].view(-1, kv_heads, b)


def _fill(buf, x, ctx):
    """Quantises x [S, H, n, 256] into the layers of buf."""
    s, h, n, _ = x.shape
    codes, exps = _views(buf, h, ctx)
    nb = (n + BLOCK - 1) // BLOCK
    pad = torch.zeros(s, h, nb * BLOCK, HD, device=x.device)
    pad[:, :, :n] = x
    e = _needed(pad.view(s, h, nb, BLOCK * HD).abs().amax(-1))
    q = _codes(pad.view(s, h, nb, BLOCK * HD), e[..., None]).view(torch.uint8).view(s, h, nb * BLOCK, HD)
    codes[:, :, :n] = q[:, :, :n]
    exps[:, :, :nb] = (e + 127).to(torch.uint8)


def _values(buf, kv_heads, ctx, lo, hi):
    """The values of positions [lo, hi), f32 [S, H, hi - lo, 256]."""
    codes, exps = _views(buf, kv_heads, ctx)
    at = torch.arange(lo, hi, device=buf.device) // BLOCK
    return codes[:, :, lo:hi].view(torch.float8_e4m3fn).float() * _pow2(exps[:, :, at].int() - 127)[..., None]


# ---------------------------------------------------------------------------------------------
# the framework's side of a state
# ---------------------------------------------------------------------------------------------
_backend = None


class _Own:
    """What a user's program keeps: the backend, a command buffer on torch's stream, and buffer handles."""

    def __init__(self):
        global _backend
        import qwasar_b200
        from qwasar_b200 import backend
        if _backend is None:
            _backend = qwasar_b200.Backend()
        self.be, self.mod, self.lib = _backend, backend, _backend.lib
        self.bufs = []
        self.cmd = self.be.cmd_begin(torch.cuda.current_stream().cuda_stream)

    def ref(self, t):
        b = self.be.buf_wrap_device(t.data_ptr(), t.numel() * t.element_size())
        self.bufs.append(b)
        return self.mod.QwRef(b, 0)

    def buf(self, b):
        self.bufs.append(b)
        return b

    def check(self, ok=True):
        e = self.be.cmd_error(self.cmd)
        if e or not ok:
            raise RuntimeError(e or "declined")

    def __del__(self):
        try:
            self.be.cmd_wait(self.cmd, check=False)
            self.be.cmd_free(self.cmd)
            for b in reversed(self.bufs):
                self.be.buf_free(b)
        except Exception:
            pass


def _refs(o, rows):
    return (o.mod.QwRef * len(rows))(*[o.ref(r) for r in rows])


# ---------------------------------------------------------------------------------------------
# states
# ---------------------------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _keys(g, s, h, n):
    """Keys as they come from a normed, rotated projection: a few channels are much larger than the rest."""
    return _normal(g, s, h, n, HD) * torch.exp(0.6 * _normal(g, 1, h, 1, HD))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 17)
    return {"rope": _prepare_rope, "write": _prepare_write, "read": _prepare_read, "attn": _prepare_attn}[case["op"]](case, g)


def _act(case):
    return torch.bfloat16 if case["bf16"] else torch.float32


def _prepare_rope(case, g):
    rows, heads, hd, r = case["rows"], case["heads"], case["head_dim"], case["rotary"]
    st = dict(case=case, stride=heads * hd + case["pad"])
    st["x"] = _normal(g, rows, st["stride"]).to(_act(case))
    st["pos"] = (case["pos0"] + torch.randint(0, 64, (1,), generator=g, device=DEV) + torch.arange(rows, device=DEV)).to(torch.int32)
    j = torch.arange(r // 2, device=DEV, dtype=torch.float64)
    freq = case["theta"] ** (-2.0 * j / r)
    # long contexts: slow frequencies are stretched by the factor, fast ones kept, and the result is a little louder
    slow = ((2 * j / r - 0.25) / 0.5).clamp(0, 1)
    st["freq"] = (freq * (1 - slow) + freq / case["factor"] * slow).float()
    st["amp"] = float(torch.tensor(0.1 * math.log(case["factor"]) + 1.0, dtype=torch.float32))
    if own:
        o = st["own"] = _Own()
        st["y"] = torch.empty(rows, heads, hd, dtype=st["x"].dtype, device=DEV)
        st["refs"] = [o.ref(st[k]) for k in ("y", "x", "pos", "freq")]
    return st


def _prepare_write(case, g):
    rows, h, base = case["rows"], case["kv_heads"], case["base"]
    ctx = base + rows + 37
    st = dict(case=case, ctx=ctx, stride=h * HD + case["pad"])
    st["k"] = (_normal(g, rows, st["stride"]) * 1.5).to(_act(case))
    st["v"] = (_normal(g, rows, st["stride"]) * 0.5).to(_act(case))
    st["kc"], st["vc"] = (torch.zeros(1, _layer_bytes(h, ctx), dtype=torch.uint8, device=DEV) for _ in range(2))
    if base:
        _fill(st["kc"], _keys(g, 1, h, base), ctx)
        _fill(st["vc"], _normal(g, 1, h, base, HD) * 0.5, ctx)
    if own:
        o = st["own"] = _Own()
        n = base + rows - base // BLOCK * BLOCK
        st["ko"], st["vo"] = (torch.empty(h, n, HD, dtype=_act(case), device=DEV) for _ in range(2))
        st["refs"] = {k: o.ref(st[k]) for k in ("k", "v", "kc", "vc", "ko", "vo")}
    return st


def _prepare_read(case, g):
    h, n, pos0 = case["kv_heads"], case["n"], case["pos0"]
    ctx = pos0 + n + 5
    st = dict(case=case, ctx=ctx, kc=torch.zeros(1, _layer_bytes(h, ctx), dtype=torch.uint8, device=DEV))
    _fill(st["kc"], _keys(g, 1, h, pos0 + n), ctx)
    if own:
        o = st["own"] = _Own()
        st["out"] = torch.empty(h, n, HD, dtype=_act(case), device=DEV)
        st["refs"] = [o.ref(st["out"]), o.ref(st["kc"])]
    return st


def _prepare_attn(case, g):
    s, rows, qh, h, base = case["seqs"], case["rows"], case["q_heads"], case["kv_heads"], case["base"]
    n = base + rows
    ctx = n + 37
    st = dict(case=case, ctx=ctx, scale=1.0 / 16.0)
    st["q"] = (_normal(g, s, rows, qh, HD) * 1.2).to(_act(case))
    st["gate"] = _normal(g, s, rows, qh, HD).to(_act(case)) if case["gate"] else None
    st["kc"], st["vc"] = (torch.zeros(s, _layer_bytes(h, ctx), dtype=torch.uint8, device=DEV) for _ in range(2))
    _fill(st["kc"], _keys(g, s, h, n), ctx)
    _fill(st["vc"], _normal(g, s, h, n, HD) * 0.5, ctx)
    if own:
        o = st["own"] = _Own()
        st["out"] = torch.empty_like(st["q"])
        st["or"], st["qr"] = _refs(o, st["out"]), _refs(o, st["q"])
        st["gr"] = _refs(o, st["gate"]) if case["gate"] else None
        if case["paged"]:
            # one pool, two arenas per sequence, filled through the append: the values are e4m3 times a power of two
            # already, so the arena holds the same values
            blocks = 2 * s * h * ((ctx + 127) // 128)
            pool = o.buf(o.be.kv_pool_alloc(blocks * 32768))
            for name in ("kr", "vr"):
                st[name] = (o.mod.QwRef * s)(*[o.mod.QwRef(o.buf(o.be.kv8_arena_alloc_in(pool, 1, h, ctx)), 0) for _ in range(s)])
            for i in range(s):
                kv = [_values(st[b][i:i + 1], h, ctx, 0, n)[0].transpose(0, 1).contiguous() for b in ("kc", "vc")]
                ok = o.lib.qw_op_kv8_write(o.cmd, st["kr"][i], st["vr"][i], o.ref(kv[0]), o.ref(kv[1]), n, h, HD, ctx, 0, h * HD, o.mod.F32)
                o.check(ok)
                torch.cuda.current_stream().synchronize()
        else:
            st["kr"], st["vr"] = _refs(o, st["kc"]), _refs(o, st["vc"])
        st["base"] = (ctypes.c_int32 * s)(*[base] * s)
    return st


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if own:
        return {"rope": _own_rope, "write": _own_write, "read": _own_read, "attn": _own_attn}[op](st)
    return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "attn": _plain_attn}[op](st)


def _own_rope(st):
    c, o = st["case"], st["own"]
    y, x, pos, freq = st["refs"]
    if not o.lib.qw_op_rope(o.cmd, y, x, pos, freq, c["rows"], c["heads"], c["head_dim"], c["rotary"], int(c["interleaved"]),
                            c["heads"] * c["head_dim"], st["stride"], st["amp"], o.mod.BF16 if c["bf16"] else o.mod.F32):
        o.check(False)
    return st["y"]


def _plain_rope(st):
    c = st["case"]
    heads, hd, r = c["heads"], c["head_dim"], c["rotary"]
    x = st["x"][:, :heads * hd].reshape(-1, heads, hd).float()
    ang = st["pos"].double()[:, None] * st["freq"].double()
    cos, sin = ((f(ang) * st["amp"]).float()[:, None] for f in (torch.cos, torch.sin))
    rot = x[..., :r]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if c["interleaved"] else (rot[..., :r // 2], rot[..., r // 2:])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([ya, yb], -1).flatten(-2) if c["interleaved"] else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., r:]], -1).to(st["x"].dtype)


def _own_write(st):
    c, o, r = st["case"], st["own"], st["refs"]
    h, io = c["kv_heads"], o.mod.BF16 if c["bf16"] else o.mod.F32
    lo = c["base"] // BLOCK * BLOCK
    n = c["base"] + c["rows"] - lo
    ok = o.lib.qw_op_kv8_write(o.cmd, r["kc"], r["vc"], r["k"], r["v"], c["rows"], h, HD, st["ctx"], c["base"], st["stride"], io)
    ok = ok and o.lib.qw_op_kv8_read(o.cmd, r["ko"], r["kc"], lo, n, h, HD, st["ctx"], io)
    ok = ok and o.lib.qw_op_kv8_read(o.cmd, r["vo"], r["vc"], lo, n, h, HD, st["ctx"], io)
    if not ok:
        o.check(False)
    return [st["ko"], st["vo"]]


def _plain_append(st, cache, x):
    c = st["case"]
    h, base, rows, ctx = c["kv_heads"], c["base"], c["rows"], st["ctx"]
    b0, b1 = base // BLOCK, (base + rows + BLOCK - 1) // BLOCK
    lo, n = b0 * BLOCK, (b1 - b0) * BLOCK
    codes, exps = _views(cache, h, ctx)
    new = torch.zeros(h, n, HD, device=x.device)
    new[:, base - lo:base - lo + rows] = x[:, :h * HD].reshape(rows, h, HD).transpose(0, 1).float()
    e = _needed(new.view(h, b1 - b0, BLOCK * HD).abs().amax(-1))
    if base > lo:                                          # the first block holds rows already: its exponent only grows
        was = exps[0, :, b0].int() - 127
        e[:, 0] = torch.maximum(e[:, 0], was)
        old = codes[0, :, lo:base].view(torch.float8_e4m3fn).float() * _pow2(was)[:, None, None]
        new[:, :base - lo] = old
    scale = e.repeat_interleave(BLOCK, 1)[..., None]
    q = _codes(new, scale)
    end = base + rows
    codes[0, :, lo:end] = q.view(torch.uint8)[:, :end - lo]
    exps[0, :, b0:b1] = (e + 127).to(torch.uint8)
    return (q.float() * _pow2(scale))[:, :end - lo].to(x.dtype)


def _plain_write(st):
    return [_plain_append(st, st["kc"], st["k"]), _plain_append(st, st["vc"], st["v"])]


def _own_read(st):
    c, o = st["case"], st["own"]
    if not o.lib.qw_op_kv8_read(o.cmd, st["refs"][0], st["refs"][1], c["pos0"], c["n"], c["kv_heads"], HD, st["ctx"],
                                o.mod.BF16 if c["bf16"] else o.mod.F32):
        o.check(False)
    return st["out"]


def _plain_read(st):
    c = st["case"]
    return _values(st["kc"], c["kv_heads"], st["ctx"], c["pos0"], c["pos0"] + c["n"])[0].to(_act(c))


def _own_attn(st):
    c, o = st["case"], st["own"]
    s, io = c["seqs"], o.mod.BF16 if c["bf16"] else o.mod.F32
    if s == 1:
        ok = o.lib.qw_op_attn_kv8(o.cmd, st["or"][0], st["gr"][0] if st["gr"] else o.mod.NULL_REF, st["qr"][0], st["kr"][0], st["vr"][0],
                                  c["rows"], c["q_heads"], c["kv_heads"], HD, st["ctx"], c["base"], st["scale"], HD, io)
    else:
        ok = o.lib.qw_op_attn_kv8_batch(o.cmd, s, st["or"], st["gr"], st["qr"], st["kr"], st["vr"], st["base"], c["rows"], c["q_heads"],
                                        c["kv_heads"], HD, st["ctx"], st["scale"], HD, io)
    if not ok:
        o.check(False)
    return st["out"]


def _plain_attn(st):
    c = st["case"]
    s, rows, qh, h, base = c["seqs"], c["rows"], c["q_heads"], c["kv_heads"], c["base"]
    n, grp = base + rows, qh // h
    k, v = _values(st["kc"], h, st["ctx"], 0, n), _values(st["vc"], h, st["ctx"], 0, n)
    q = st["q"].float().view(s, rows, h, grp, HD).permute(0, 2, 1, 3, 4).reshape(s, h, rows * grp, HD)
    t = (q @ k.transpose(-1, -2)) * st["scale"]
    row = torch.arange(rows * grp, device=t.device) // grp
    t.masked_fill_(torch.arange(n, device=t.device) > (base + row)[:, None], float("-inf"))
    t -= t.amax(-1, keepdim=True)
    t.exp_()
    out = (t @ v) / t.sum(-1, keepdim=True)
    out = out.view(s, h, rows, grp, HD).permute(0, 2, 1, 3, 4).reshape(s, rows, qh, HD)
    if st["gate"] is not None:
        out = out / (1 + torch.exp(-st["gate"].float()))
    return out.to(st["q"].dtype)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    el = 2 if case["bf16"] else 4
    if case["op"] == "rope":
        n = case["rows"] * case["heads"] * case["head_dim"]
        return {"bytes": 2 * n * el + case["rows"] * 4 + case["rotary"] * 2, "flops": 3.0 * case["rows"] * case["heads"] * case["rotary"]}
    if case["op"] == "write":
        h, lo = case["kv_heads"], case["base"] // BLOCK * BLOCK
        n = case["base"] + case["rows"] - lo
        new, old = 2 * case["rows"] * h * HD, 2 * (case["base"] - lo) * h * HD
        return {"bytes": new * (el + 1) + old + 2 * n * h * HD * el, "flops": 2.0 * new}
    if case["op"] == "read":
        n = case["kv_heads"] * case["n"] * HD
        return {"bytes": n * (1 + el), "flops": float(n)}
    s, rows, qh, h, base = case["seqs"], case["rows"], case["q_heads"], case["kv_heads"], case["base"]
    keys = rows * base + rows * (rows + 1) // 2
    io = (3 if case["gate"] else 2) * s * rows * qh * HD * el
    return {"bytes": 2 * s * h * (base + rows) * HD + io, "flops": 4.0 * HD * s * qh * keys}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _decode64(codes):
    """e4m3 codes by their fields: sign, 4 exponent bits (bias 7), 3 mantissa bits."""
    c = codes.to(torch.int64)
    man, ex = (c & 7).double(), (c >> 3) & 15
    mag = torch.where(ex == 0, man * 2.0 ** -9, torch.ldexp(1.0 + man / 8, ex - 7))
    return torch.where(c >= 128, -mag, mag)


def _round64(x):
    """x rounded to the nearest e4m3 value, ties to even, largest 448."""
    a = x.abs()
    ex = torch.frexp(a)[1].to(torch.int64) - 1
    step = torch.ldexp(torch.ones_like(a), ex.clamp(min=-6) - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=448.0)


def _needed64(amax):
    m, k = torch.frexp(amax)
    return torch.where(amax > 0, k.to(torch.int64) - 9 + (m > 0.875), E_MIN).clamp(E_MIN, E_MAX)


def _at64(buf, kv_heads, ctx, lo, hi):
    n = kv_heads * ctx * HD
    nb = (ctx + BLOCK - 1) // BLOCK
    out = _decode64(buf[:n].view(kv_heads, ctx, HD)[:, lo:hi])
    e = buf[n:n + kv_heads * nb].view(kv_heads, nb).to(torch.int64) - 127
    return torch.ldexp(out, e[:, [t // BLOCK for t in range(lo, hi)]][..., None])


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        heads, hd, r = case["heads"], case["head_dim"], case["rotary"]
        y = st["x"][:, :heads * hd].double().reshape(-1, heads, hd).clone()
        x = y.clone()
        half = r // 2
        for j in range(half):
            a = st["pos"].double() * float(st["freq"][j])
            co, si = (torch.cos(a) * st["amp"])[:, None], (torch.sin(a) * st["amp"])[:, None]
            p, q = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
            y[..., p] = x[..., p] * co - x[..., q] * si
            y[..., q] = x[..., q] * co + x[..., p] * si
        return y
    if case["op"] == "write":
        h, base, rows, out = case["kv_heads"], case["base"], case["rows"], []
        lo = base // BLOCK * BLOCK
        for cache, x in ((st["kc"][0], st["k"]), (st["vc"][0], st["v"])):
            x = x[:, :h * HD].double().reshape(rows, h, HD).transpose(0, 1)
            got = torch.zeros(h, base + rows - lo, HD, dtype=torch.float64, device=x.device)
            for b in range(base // BLOCK, (base + rows + BLOCK - 1) // BLOCK):
                f, t = max(b * BLOCK, base), min((b + 1) * BLOCK, base + rows)
                e = _needed64(x[:, f - base:t - base].abs().amax((1, 2)))
                if f > b * BLOCK:
                    n, nb = h * st["ctx"] * HD, (st["ctx"] + BLOCK - 1) // BLOCK
                    was = cache[n:n + h * nb].view(h, nb)[:, b].to(torch.int64) - 127
                    e = torch.maximum(e, was)
                    old = _at64(cache, h, st["ctx"], b * BLOCK, f)
                    got[:, :f - lo] = torch.ldexp(_round64(torch.ldexp(old, -e[:, None, None])), e[:, None, None])
                got[:, f - lo:t - lo] = torch.ldexp(_round64(torch.ldexp(x[:, f - base:t - base], -e[:, None, None])), e[:, None, None])
            out.append(got)
        return out
    if case["op"] == "read":
        return _at64(st["kc"][0], case["kv_heads"], st["ctx"], case["pos0"], case["pos0"] + case["n"])
    s, rows, qh, h, base = case["seqs"], case["rows"], case["q_heads"], case["kv_heads"], case["base"]
    if s * rows * qh * (base + rows) > 4e8:
        return None
    grp = qh // h
    out = torch.empty(s, rows, qh, HD, dtype=torch.float64, device=DEV)
    seen = torch.arange(base + rows, device=DEV)[None] <= base + torch.arange(rows, device=DEV)[:, None]
    for i in range(s):
        k, v = (_at64(st[b][i], h, st["ctx"], 0, base + rows) for b in ("kc", "vc"))
        for j in range(qh):
            t = st["q"][i, :, j].double() @ k[j // grp].T * st["scale"]
            out[i, :, j] = torch.softmax(torch.where(seen, t, -math.inf), -1) @ v[j // grp]
    if st["gate"] is not None:
        out *= torch.sigmoid(st["gate"].double())
    return out
