"""GPU: normalised and rotated heads, forward and backward, against the float64 oracle.

Bounds, u = 2^-24 (half a step of float32).  Forward: the mean of D <= 256 squares is a sum of at most 16 terms a lane and a tree over the
lanes (below 24 u relative, halved by the root), rsqrtf 2 steps, three products, then two products and a sum of the rotation, whose
cosine and sine are off by at most 2^-23 plus the float32 angle's pi u: together below 40 u of (|n0| + |n1|) gain, n0, n1 the pair before
the rotation.  A bf16 result adds half a step, 2^-8 of it.  Backward: the same for r and the rotation of dy, and one more such mean,
below 80 u of (r |w| G + |x| r^3 mean(|w| G |x|)), G = |dy0| + |dy1| of the pair.  A weight gradient is a sum over rows, at most
a few of which one warp adds; below 100 u of the sum of G |x| r.
"""
import ctypes as C

import numpy as np
import pytest

from oracle import tree_oracle as orc
from oracle.attention_oracle import from_bf16_bits, round_bf16, to_bf16_bits

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
MODES = {"none": 0, "interleaved": 1, "half": 2}


@pytest.fixture(scope="module")
def dev():
    from grilly_next import cabi
    d = cabi.Device(0)
    yield d
    d.close()


class Buf:
    """A device array of float32 or bf16 with guard rows on both ends that must stay as they were."""
    GUARD = 64

    def __init__(self, dev, shape, dtype, data=None, shift=0):
        self.dev, self.shape, self.dtype, self.n = dev, tuple(shape), dtype, int(np.prod(shape))
        self.kind = np.float32 if dtype == "f32" else np.uint16
        self.host = np.full(self.n + 2 * self.GUARD + shift, 0x4242, self.kind)
        self.off = self.GUARD + shift
        if data is not None:
            d = np.asarray(data, np.float32).reshape(-1)
            self.host[self.off:self.off + self.n] = d if dtype == "f32" else to_bf16_bits(d)
        self.p = dev.upload(self.host)
        self.ptr = self.p.value + self.off * self.host.itemsize

    def get(self):
        now = self.dev.download(self.p, self.host.shape, self.kind)
        a, b = self.off, self.off + self.n
        assert np.array_equal(now[:a], self.host[:a]) and np.array_equal(now[b:], self.host[b:]), "written outside the tensor"
        x = now[a:b].reshape(self.shape)
        return x.copy() if self.dtype == "f32" else from_bf16_bits(x)

    def free(self):
        self.dev.free(self.p)


def make(B, S, Hq, Hk, D, *, rotary=None, mode="half", dtype="f32", out=None, layout="plain", weight=True, scaled=False, gain=0.0, start=0,
         positions=False, scaling=0.0, shift=0, seed=0, scale=1.0):
    return dict(B=B, S=S, Hq=Hq, Hk=Hk, D=D, rotary=D if rotary is None else rotary, mode=mode, dtype=dtype, out=out or dtype, layout=layout,
                weight=weight, scaled=scaled, gain=gain, start=start, positions=positions, scaling=scaling, shift=shift, seed=seed, scale=scale)


CASES = {
    "one_row": make(1, 1, 1, 1, 64),
    "prompt_bf16": make(2, 37, 8, 2, 128, dtype="bf16", layout="head_major"),
    "interleaved_bf16": make(2, 37, 8, 2, 128, dtype="bf16", mode="interleaved"),
    "packed": make(3, 19, 4, 4, 64, layout="packed", mode="interleaved"),
    "packed_bf16": make(3, 19, 6, 2, 128, layout="packed", dtype="bf16"),
    "part_half": make(2, 21, 4, 2, 128, rotary=64),
    "part_interleaved_bf16": make(2, 21, 4, 2, 128, rotary=32, mode="interleaved", dtype="bf16"),
    "part_odd": make(2, 9, 3, 1, 64, rotary=20),
    "no_rotation": make(2, 9, 3, 1, 128, mode="none"),
    "no_weight": make(2, 9, 3, 1, 128, weight=False),
    "queries_only": make(2, 9, 5, 0, 128),
    "scaled_far": make(1, 11, 4, 2, 128, scaled=True, gain=1.2079, start=(1 << 22) + 7),
    "scaling": make(1, 11, 4, 2, 64, scaling=4.0, start=1000),
    "positions": make(3, 13, 4, 2, 64, positions=True, dtype="bf16"),
    "dim_32": make(2, 33, 4, 4, 32), "dim_80": make(2, 15, 3, 1, 80), "dim_96": make(2, 15, 3, 1, 96, rotary=48, dtype="bf16"),
    "dim_256": make(2, 15, 2, 1, 256, mode="interleaved", dtype="bf16"), "dim_256_f32": make(2, 15, 2, 1, 256), "dim_2": make(1, 5, 1, 1, 2), "dim_6": make(2, 5, 2, 1, 6),
    "off_alignment": make(2, 7, 3, 2, 64, shift=1), "off_alignment_bf16": make(2, 7, 3, 2, 128, dtype="bf16", shift=3),
    "bf16_to_f32": make(2, 7, 3, 2, 128, dtype="bf16", out="f32"), "f32_to_bf16": make(2, 7, 3, 2, 128, out="bf16"),
    "small_values": make(1, 7, 3, 2, 128, scale=1e-6), "large_values": make(1, 7, 3, 2, 128, scale=1e6, dtype="bf16"),
    "many_tokens": make(2, 700, 4, 2, 64, dtype="bf16"), "many_tokens_f32": make(1, 1001, 4, 1, 128, layout="packed"),
}


class Call:
    def __init__(self, dev, c):
        from grilly_next import cabi
        self.cabi, self.dev, self.c = cabi, dev, c
        r = np.random.default_rng(c["seed"])
        B, S, Hq, Hk, D = (c[k] for k in ("B", "S", "Hq", "Hk", "D"))
        rnd = round_bf16 if c["dtype"] == "bf16" else (lambda x: x)
        self.q, self.k = (rnd((c["scale"] * r.standard_normal((B, S, h, D))).astype(np.float32)) for h in (Hq, Hk))
        self.wq, self.wk = ((1 + 0.2 * r.standard_normal(D)).astype(np.float32) for _ in range(2))
        self.pos = r.integers(0, 5000, (B, S)).astype(np.int32) if c["positions"] else np.broadcast_to(np.arange(S), (B, S))
        self.freq32 = orc.frequencies(c["rotary"]).astype(np.float32) * np.linspace(1, 0.2, c["rotary"] // 2).astype(np.float32) if c["scaled"] else None
        self.freq = orc.frequencies(c["rotary"], 10000.0, c["scaling"] or 1.0, self.freq32)
        self.keep, self.bufs = [], []
        p = self.p = cabi.QKNormParams()
        if c["layout"] == "packed":
            rows = self.buf((B, S, Hq + 2 * Hk, D), c["dtype"], np.concatenate([self.q, self.k, self.k], 2), c["shift"])
            size = rows.host.itemsize
            p.q, p.k = rows.ptr, rows.ptr + Hq * D * size
            p.q_strides[:] = p.k_strides[:] = [S * (Hq + 2 * Hk) * D, (Hq + 2 * Hk) * D, D]
        else:
            p.q = self.buf(self.q.shape, c["dtype"], self.q, c["shift"]).ptr
            if Hk:
                p.k = self.buf(self.k.shape, c["dtype"], self.k, c["shift"]).ptr
        if c["weight"]:
            p.q_weight, p.k_weight = self.up(self.wq), self.up(self.wk)
        code = {"f32": cabi.F32, "bf16": cabi.BF16}
        p.in_dtype, p.out_dtype = code[c["dtype"]], code[c["out"]]
        p.batch, p.seq_len, p.num_q_heads, p.num_kv_heads, p.head_dim = B, S, Hq, Hk, D
        p.eps, p.rope.mode, p.rope.rotary_dim, p.rope.theta = 1e-5, MODES[c["mode"]], c["rotary"], 10000.0
        p.rope.gain, p.rope.scaling, p.pos_base = c["gain"], c["scaling"], c["start"]
        if self.freq32 is not None:
            p.rope.inv_freq = self.up(self.freq32)
        if c["positions"]:
            p.positions = self.up(self.pos)
        if c["layout"] == "head_major":
            p.q_out_strides[:], p.k_out_strides[:] = [Hq * S * D, D, S * D], [Hk * S * D, D, S * D]

    def up(self, a):
        h = self.dev.upload(a)
        self.keep.append(h)
        return h

    def buf(self, shape, dtype, data=None, shift=0):
        b = Buf(self.dev, shape, dtype, data, shift)
        self.bufs.append(b)
        return b

    def result(self, h, dtype, data=None):
        """A (B,S,h,D) tensor, in memory (B,h,S,D) for head_major, and how to read it in index order."""
        c = self.c
        major = c["layout"] == "head_major"
        shape = (c["B"], h, c["S"], c["D"]) if major else (c["B"], c["S"], h, c["D"])
        turn = (lambda x: x.transpose(0, 2, 1, 3)) if major else (lambda x: x)
        return self.buf(shape, dtype, None if data is None else turn(data), c["shift"]), turn

    def oracle(self, x, w):
        c = self.c
        mode = c["mode"]
        return orc.norm_rope(x, w if c["weight"] else None, self.pos + c["start"], self.freq, mode, float(np.float32(1e-5)), float(np.float32(c["gain"])) or 1.0)

    def pair_size(self, x):
        """|x0| + |x1| of every element's pair, times the gain, where the rotation turns it; |x| elsewhere."""
        c, n = self.c, len(self.freq) if self.c["mode"] != "none" else 0
        a = np.abs(np.asarray(x, np.float64))
        out = a.copy()
        if n:
            lo, hi = (slice(0, n), slice(n, 2 * n)) if c["mode"] == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
            out[..., lo] = out[..., hi] = (a[..., lo] + a[..., hi]) * (c["gain"] or 1.0)
        return out

    def done(self):
        for b in self.bufs:
            b.free()
        for h in self.keep:
            self.dev.free(h)


def within(got, want, tol, what):
    over = np.abs(got - want) - tol
    assert np.all(over <= 0), f"{what}: off by {np.abs(got - want).max():.3g}, over the bound by {over.max():.3g}"


@pytest.mark.parametrize("name", list(CASES))
def test_forward(dev, name):
    c = CASES[name]
    call = Call(dev, c)
    p = call.p
    yq, turn = call.result(c["Hq"], c["out"])
    p.q_out = yq.ptr
    if c["Hk"]:
        yk, _ = call.result(c["Hk"], c["out"])
        p.k_out = yk.ptr
    call.cabi.check(dev.L.grl_qk_norm_rope(dev.h, C.byref(p)))
    dev.sync()
    for x, w, y in ((call.q, call.wq, yq), (call.k, call.wk, yk if c["Hk"] else None)):
        if y is None:
            continue
        want = call.oracle(x, w)
        tol = 40 * U * call.pair_size(orc.norm(x, w if c["weight"] else None, 1e-5))
        if c["out"] == "bf16":
            tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
        within(turn(y.get()), want, tol, name)
    call.done()


@pytest.mark.parametrize("name", list(CASES))
def test_backward(dev, name):
    c = CASES[name]
    call = Call(dev, c)
    cabi, B, S, Hq, Hk, D = call.cabi, c["B"], c["S"], c["Hq"], c["Hk"], c["D"]
    r = np.random.default_rng(100 + c["seed"])
    rnd = round_bf16 if c["out"] == "bf16" else (lambda x: x)
    dyq, dyk = (rnd(r.standard_normal((B, S, h, D)).astype(np.float32)) for h in (Hq, Hk))
    p = cabi.QKNormGradParams()
    p.fwd = call.p
    p.q_out_grad = call.result(Hq, c["out"], dyq)[0].ptr
    dxq = call.buf((B, S, Hq, D), c["dtype"], None, c["shift"])
    dwq, dwk = call.buf((D,), "f32"), call.buf((D,), "f32")
    p.q_grad, p.q_weight_grad = dxq.ptr, dwq.ptr
    sides = [(call.q, call.wq, dyq, dxq, dwq)]
    if Hk:
        p.k_out_grad = call.result(Hk, c["out"], dyk)[0].ptr
        dxk = call.buf((B, S, Hk, D), c["dtype"], None, c["shift"])
        p.k_grad, p.k_weight_grad = dxk.ptr, dwk.ptr
        sides.append((call.k, call.wk, dyk, dxk, dwk))
    size = C.c_size_t()
    cabi.check(dev.L.grl_qk_norm_rope_backward_workspace_bytes(dev.h, C.byref(p), C.byref(size)))
    assert size.value > 0
    ws = dev.malloc(size.value)
    p.workspace, p.workspace_bytes = ws, size.value
    cabi.check(dev.L.grl_qk_norm_rope_backward(dev.h, C.byref(p)))
    dev.sync()
    first = [(dx.get(), dw.get()) for _, _, _, dx, dw in sides]
    for (x, w, dy, _, _), (dx, dw) in zip(sides, first):
        w64 = w if c["weight"] else np.ones(D)
        want_dx, want_dw = orc.norm_rope_grad(x, w64, dy, call.pos + c["start"], call.freq, c["mode"], 1e-5, float(np.float32(c["gain"])) or 1.0)
        x64 = np.asarray(x, np.float64)
        rr = 1 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + 1e-5)
        G = call.pair_size(dy)
        tol = 80 * U * (rr * np.abs(w64) * G + np.abs(x64) * rr ** 3 * (np.abs(w64) * G * np.abs(x64)).mean(-1, keepdims=True))
        if c["dtype"] == "bf16":
            tol = tol + 2.0 ** -8 * (np.abs(want_dx) + tol)
        within(dx, want_dx, tol, name + " dx")
        within(dw, want_dw, 100 * U * (G * np.abs(x64) * rr).reshape(-1, D).sum(0), name + " dw")
    # the same inputs give the same bits, and a call without weight gradients the same gradients of the inputs without a workspace
    cabi.check(dev.L.grl_qk_norm_rope_backward(dev.h, C.byref(p)))
    dev.sync()
    for (_, _, _, dx, dw), (a, b) in zip(sides, first):
        assert np.array_equal(dx.get(), a) and np.array_equal(dw.get(), b)
    p.q_weight_grad = p.k_weight_grad = p.workspace = None
    p.workspace_bytes = 0
    cabi.check(dev.L.grl_qk_norm_rope_backward(dev.h, C.byref(p)))
    dev.sync()
    for (_, _, _, dx, _), (a, _) in zip(sides, first):
        assert np.array_equal(dx.get(), a)
    dev.free(ws)
    call.done()


def test_backward_refuses_a_small_workspace(dev):
    call = Call(dev, CASES["prompt_bf16"])
    p = call.cabi.QKNormGradParams()
    p.fwd = call.p
    p.q_out_grad = p.k_out_grad = p.q_grad = p.k_grad = p.q_weight_grad = call.p.q
    assert dev.L.grl_qk_norm_rope_backward(dev.h, C.byref(p)) == call.cabi.ERR_INVALID
    assert b"workspace too small" in dev.L.grl_last_error()
    call.done()


def test_in_place_and_zero_rows(dev):
    """q_out may be q; a row of zeros stays zeros."""
    c = make(2, 50, 4, 2, 128, dtype="bf16")
    call = Call(dev, c)
    call.q[0, 3] = 0
    q = call.buf(call.q.shape, "bf16", call.q)
    k = call.buf(call.k.shape, "bf16", call.k)
    call.p.q = call.p.q_out = q.ptr
    call.p.k = call.p.k_out = k.ptr
    call.cabi.check(dev.L.grl_qk_norm_rope(dev.h, C.byref(call.p)))
    dev.sync()
    want = call.oracle(call.q, call.wq)
    within(q.get(), want, 2.0 ** -8 * np.abs(want) + 41 * U * call.pair_size(orc.norm(call.q, call.wq, 1e-5)), "in place")
    assert np.all(q.get()[0, 3] == 0)
    call.done()


def test_broadcast_inputs(dev):
    """An input whose sequences share memory (stride 0) is read as it is; its gradients need places of their own."""
    c = make(3, 17, 4, 2, 64)
    call = Call(dev, c)
    p = call.p
    p.q_strides[:], p.k_strides[:] = [0, 4 * 64, 64], [0, 2 * 64, 64]
    yq, yk = call.buf(call.q.shape, "f32"), call.buf(call.k.shape, "f32")
    p.q_out, p.k_out = yq.ptr, yk.ptr
    call.cabi.check(dev.L.grl_qk_norm_rope(dev.h, C.byref(p)))
    dev.sync()
    for x, w, y in ((call.q, call.wq, yq), (call.k, call.wk, yk)):
        x = np.broadcast_to(x[:1], x.shape)
        within(y.get(), call.oracle(x, w), 40 * U * call.pair_size(orc.norm(x, w, 1e-5)), "broadcast")
    call.done()


def test_captured_and_replayed_on_new_inputs(dev):
    """A graph of forward and backward gives, on other inputs in the same buffers, what direct calls give."""
    c = make(2, 64, 4, 2, 128, dtype="bf16")
    call = Call(dev, c)
    cabi, p = call.cabi, call.p
    yq, yk = call.buf(call.q.shape, "bf16"), call.buf(call.k.shape, "bf16")
    p.q_out, p.k_out = yq.ptr, yk.ptr
    gp = cabi.QKNormGradParams()
    gp.fwd = p
    gp.q_out_grad, gp.k_out_grad = yq.ptr, yk.ptr
    outs = [call.buf(call.q.shape, "bf16"), call.buf(call.k.shape, "bf16"), call.buf((128,), "f32"), call.buf((128,), "f32")]
    gp.q_grad, gp.k_grad, gp.q_weight_grad, gp.k_weight_grad = (o.ptr for o in outs)
    size = C.c_size_t()
    cabi.check(dev.L.grl_qk_norm_rope_backward_workspace_bytes(dev.h, C.byref(gp), C.byref(size)))
    ws = dev.malloc(size.value)
    gp.workspace, gp.workspace_bytes = ws, size.value

    def both():
        cabi.check(dev.L.grl_qk_norm_rope(dev.h, C.byref(p)))
        cabi.check(dev.L.grl_qk_norm_rope_backward(dev.h, C.byref(gp)))

    both()
    dev.sync()
    g = C.c_void_p()
    cabi.check(dev.L.grl_graph_begin(dev.h))
    both()
    cabi.check(dev.L.grl_graph_end(dev.h, C.byref(g)))
    new = to_bf16_bits(np.random.default_rng(9).standard_normal(call.q.size).astype(np.float32))
    cabi.check(dev.L.grl_memcpy_h2d(dev.h, p.q, new.ctypes.data_as(C.c_void_p), new.nbytes))
    dev.sync()
    both()
    dev.sync()
    want = [o.get() for o in outs + [yq, yk]]
    for o in outs + [yq, yk]:
        cabi.check(dev.L.grl_memset(dev.h, o.ptr, 0, o.n * o.host.itemsize))
    cabi.check(dev.L.grl_graph_launch(dev.h, g))
    dev.sync()
    for o, w in zip(outs + [yq, yk], want):
        assert np.array_equal(o.get(), w)
    cabi.check(dev.L.grl_graph_destroy(g))
    dev.free(ws)
    call.done()
