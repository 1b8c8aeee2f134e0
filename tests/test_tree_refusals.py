"""CPU: what the entry points of normalised heads and drafted steps refuse (nothing is launched: the checks come before the device), and
the float64 oracle's gradients against differences."""
import ctypes as C

import numpy as np
import pytest

from grilly_next import cabi
from oracle import tree_oracle as orc

P = 1 << 20        # an aligned pointer that nothing follows


def said(rc):
    return rc, cabi.lib().grl_last_error().decode()


def norm_params(**kw):
    p = cabi.QKNormParams()
    p.q = p.k = p.q_out = p.k_out = P
    p.in_dtype = p.out_dtype = cabi.BF16
    p.batch, p.seq_len, p.num_q_heads, p.num_kv_heads, p.head_dim = 2, 5, 4, 2, 64
    p.rope.mode, p.rope.theta = cabi.ROPE_HALF, 10000.0
    for k, v in kw.items():
        if k.startswith("rope_"):
            setattr(p.rope, k[5:], v)
        elif k.endswith("strides"):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return p


def layout(**kw):
    kv = cabi.KVLayout()
    kv.k_pages = kv.v_pages = kv.block_table = kv.seq_lens = P
    kv.cache_dtype = cabi.BF16
    kv.batch, kv.num_kv_heads, kv.head_dim, kv.page_tokens, kv.max_pages = 2, 2, 64, 16, 4
    for k, v in kw.items():
        setattr(kv, k, v)
    return kv


def params(cls, kv, **kw):
    p = cls()
    p.kv = layout(**kv)
    for k, v in kw.items():
        if k.startswith("rope_"):
            setattr(p.rope, k[5:], v)
        else:
            setattr(p, k, v)
    return p


def append(kv=None, **kw):
    return params(cabi.AppendNormParams, kv or {}, **{**dict(k_new=P, v_new=P, q_in=P, q_out=P, num_q_heads=4, n_new=3, rope_mode=cabi.ROPE_HALF,
                                                        rope_theta=10000.0), **kw})


def tree(kv=None, **kw):
    return params(cabi.TreeParams, kv or {}, **{**dict(q=P, out=P, io_dtype=cabi.BF16, num_q_heads=4, n_tree=3), **kw})


def commit(kv=None, **kw):
    return params(cabi.CommitParams, kv or {}, **{**dict(path=P, n_path=P, max_path=2, n_tree=3), **kw})


NORM = [
    (dict(q=None), "q is NULL"), (dict(q_out=None), "q_out or k_out is NULL"), (dict(k_out=None), "q_out or k_out is NULL"),
    (dict(in_dtype=2), "in_dtype"), (dict(out_dtype=7), "out_dtype"), (dict(batch=0), "bad shape"), (dict(seq_len=-1), "bad shape"),
    (dict(num_kv_heads=0), "bad shape"), (dict(head_dim=63), "even"), (dict(head_dim=258), "256"), (dict(eps=-1.0), "eps"),
    (dict(rope_mode=3), "rope mode"), (dict(rope_rotary_dim=66), "rotary_dim"), (dict(rope_rotary_dim=31), "rotary_dim"),
    (dict(rope_theta=0.0), "theta"), (dict(rope_scaling=-1.0), "scaling"), (dict(q_strides=[-1, 64, 64]), "negative"),
    (dict(q_out_strides=[0, 256, 64]), "overlap"), (dict(q_out_strides=[1280, 256, 63]), "overlap"), (dict(k_out_strides=[640, 64, 64]), "overlap"),
]


@pytest.mark.parametrize("change,words", NORM, ids=[str(c[0]) for c in NORM])
def test_qk_norm_refuses(change, words):
    rc, msg = said(cabi.lib().grl_qk_norm_rope(None, C.byref(norm_params(**change))))
    assert rc == cabi.ERR_INVALID and words in msg


def test_valid_calls_come_as_far_as_the_device():
    L = cabi.lib()
    head_major = [4 * 5 * 64, 64, 5 * 64]
    packed = [5 * 8 * 64, 8 * 64, 64]
    for p in (norm_params(), norm_params(k=None, k_out=None, num_kv_heads=0), norm_params(q_out_strides=head_major, q_strides=packed),
              norm_params(q_strides=[0, 256, 64]), norm_params(rope_rotary_dim=32), norm_params(rope_mode=0, rope_theta=0.0),
              norm_params(head_dim=2), norm_params(batch=1, q_out_strides=[0, 256, 64])):
        rc, msg = said(L.grl_qk_norm_rope(None, C.byref(p)))
        assert rc == cabi.ERR_INVALID and msg == "dev is NULL", msg
    for fn, p in ((L.grl_kv_append_norm, append()), (L.grl_kv_append_norm, append(q_in=None, q_out=None, num_q_heads=0)),
                  (L.grl_kv_append_norm, append(n_new=2000)), (L.grl_kv_append_norm, append(n_new=128, parents=P)),
                  (L.grl_tree_attention, tree()), (L.grl_tree_attention, tree(n_tree=128)), (L.grl_kv_commit, commit())):
        rc, msg = said(fn(None, C.byref(p)))
        assert rc == cabi.ERR_INVALID and msg == "dev is NULL", msg


def test_null_parameter_blocks():
    L = cabi.lib()
    for fn in (L.grl_qk_norm_rope, L.grl_qk_norm_rope_backward, L.grl_kv_append_norm, L.grl_tree_attention, L.grl_kv_commit):
        rc, msg = said(fn(None, None))
        assert rc == cabi.ERR_INVALID and "NULL" in msg


GRAD = [(dict(q_out_grad=None), "q_out_grad"), (dict(q_grad=None), "q_out_grad or q_grad"), (dict(k_grad=None), "k_grad"),
        (dict(q_grad_strides=[0, 256, 64]), "overlap"), (dict(k_grad_strides=[640, 128, 0]), "overlap")]


@pytest.mark.parametrize("change,words", GRAD, ids=[str(c[0]) for c in GRAD])
def test_qk_norm_backward_refuses(change, words):
    p = cabi.QKNormGradParams()
    p.fwd = norm_params(q_out=None, k_out=None)
    p.q_out_grad = p.k_out_grad = p.q_grad = p.k_grad = P
    rc, msg = said(cabi.lib().grl_qk_norm_rope_backward(None, C.byref(p)))
    assert rc == cabi.ERR_INVALID and msg == "dev is NULL"
    for k, v in change.items():
        if k.endswith("strides"):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    rc, msg = said(cabi.lib().grl_qk_norm_rope_backward(None, C.byref(p)))
    assert rc == cabi.ERR_INVALID and words in msg


def test_weight_gradient_without_keys_is_refused():
    p = cabi.QKNormGradParams()
    p.fwd = norm_params(k=None, k_out=None)
    p.q_out_grad = p.q_grad = p.k_weight_grad = P
    rc, msg = said(cabi.lib().grl_qk_norm_rope_backward(None, C.byref(p)))
    assert rc == cabi.ERR_INVALID and "k_weight_grad" in msg


LAYOUT = [(dict(k_pages=None), "NULL cache"), (dict(seq_lens=None), "NULL cache"), (dict(batch=0), "cache shape"), (dict(page_tokens=0), "cache shape"),
          (dict(num_pages=-1), "cache shape"), (dict(head_dim=65), "head_dim"), (dict(cache_dtype=5), "cache dtype"),
          (dict(max_pages=1 << 28), "2^31")]


@pytest.mark.parametrize("make,fn", [(append, "grl_kv_append_norm"), (tree, "grl_tree_attention"), (commit, "grl_kv_commit")])
def test_cache_layouts_are_refused(make, fn):
    call = getattr(cabi.lib(), fn)
    for change, words in LAYOUT:
        rc, msg = said(call(None, C.byref(make(kv=change))))
        assert rc == cabi.ERR_INVALID and words in msg, (change, msg)
    rc, msg = said(call(None, C.byref(make(kv=dict(cache_dtype=cabi.FP8_INT4)))))
    assert rc == cabi.ERR_UNSUPPORTED and "quantised" in msg


@pytest.mark.parametrize("p,words", [
    (append(k_new=None), "k_new"), (append(q_out=None), "q_out"), (append(num_q_heads=0), "num_q_heads"), (append(n_new=0), "n_new"),
    (append(in_dtype=3), "in_dtype"), (append(q_out_dtype=3), "q_out_dtype"), (append(eps=-1.0), "eps"), (append(q_token_stride=-4), "negative"),
    (append(parents=P, n_new=129), "128"), (append(rope_rotary_dim=66), "rotary_dim"),
    (tree(q=None), "q or out"), (tree(io_dtype=2), "io_dtype"), (tree(num_q_heads=3), "multiple"), (tree(num_q_heads=0), "multiple"),
    (tree(n_tree=0), "n_tree"), (tree(n_tree=129), "n_tree"), (tree(n_splits=-1), "n_splits"), (tree(scale=-1.0), "scale"),
    (tree(kernel=9), "kernel"), (tree(q=P + 2), "aligned"), (tree(num_q_heads=1 << 20), "too many"),
    (commit(path=None), "path"), (commit(max_path=0), "max_path"), (commit(n_tree=0), "n_tree")], ids=lambda v: v if isinstance(v, str) else "")
def test_steps_refuse(p, words):
    fn = {cabi.AppendNormParams: "grl_kv_append_norm", cabi.TreeParams: "grl_tree_attention", cabi.CommitParams: "grl_kv_commit"}[type(p)]
    rc, msg = said(getattr(cabi.lib(), fn)(None, C.byref(p)))
    assert rc == cabi.ERR_INVALID and words in msg


def test_tree_attention_refuses_other_head_dims():
    rc, msg = said(cabi.lib().grl_tree_attention(None, C.byref(tree(kv=dict(head_dim=96)))))
    assert rc == cabi.ERR_UNSUPPORTED and "96" in msg


def test_commit_refuses_bad_metadata():
    m = cabi.KVMeta()
    m.cum_score = m.tombstone = P
    m.capacity = 63
    rc, msg = said(cabi.lib().grl_kv_commit(None, C.byref(commit(meta=C.pointer(m)))))
    assert rc == cabi.ERR_INVALID and "capacity" in msg
    m.capacity, m.tombstone = 64, None
    rc, msg = said(cabi.lib().grl_kv_commit(None, C.byref(commit(meta=C.pointer(m)))))
    assert rc == cabi.ERR_INVALID and "metadata" in msg


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"grl_rope_spec": (cabi.RopeSpec, ["inv_freq"]), "grl_qk_norm_params": (cabi.QKNormParams, ["q_strides", "rope", "pos_base"]),
             "grl_qk_norm_grad_params": (cabi.QKNormGradParams, ["q_grad_strides", "workspace_bytes"]),
             "grl_append_norm_params": (cabi.AppendNormParams, ["k_token_stride", "rope", "n_nodes"]),
             "grl_tree_params": (cabi.TreeParams, ["parents", "workspace_bytes"]), "grl_commit_params": (cabi.CommitParams, ["max_path", "meta"])}
    want, lines = [], []
    for c, (t, fields) in names.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(C.sizeof(t))
        for f in fields:
            lines.append(f'printf("%zu\\n", offsetof({c}, {f}));')
            want.append(getattr(t, f).offset)
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "grilly_cuda.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    cc = "/usr/bin/gcc" if os.path.exists("/usr/bin/gcc") else "gcc"
    subprocess.check_call([cc, "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "sz")])
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "sz")]).split()] == want


@pytest.mark.parametrize("mode,rotary", [("half", 8), ("interleaved", 8), ("half", 4), ("interleaved", 4), ("none", 0)])
def test_oracle_gradients_match_differences(mode, rotary):
    r = np.random.default_rng(3)
    x, dy, w = r.standard_normal((2, 3, 2, 8)), r.standard_normal((2, 3, 2, 8)), 1 + 0.2 * r.standard_normal(8)
    pos, freq = np.array([[0, 5, 9], [100, 101, 7]]), orc.frequencies(rotary) if rotary else np.zeros(0)
    f = lambda x, w: (orc.norm_rope(x, w, pos, freq, mode, 1e-3, 1.25) * dy).sum()  # noqa: E731
    dx, dw = orc.norm_rope_grad(x, w, dy, pos, freq, mode, 1e-3, 1.25)
    h = 1e-5        # central differences of a function with third derivatives of order 1: h^2 + 2^-53 / h, relative, is below 1e-9
    for got, name, a in ((dx, "x", x), (dw, "w", w)):
        num = np.zeros_like(a)
        for i in np.ndindex(a.shape):
            up, dn = a.copy(), a.copy()
            up[i] += h
            dn[i] -= h
            num[i] = ((f(up, w) - f(dn, w)) if name == "x" else (f(x, up) - f(x, dn))) / (2 * h)
        np.testing.assert_allclose(got, num, atol=1e-7, rtol=1e-7)


def test_oracle_trees():
    parents = [-1, 0, 0, 1, -1, 3]
    s = orc.ancestors(parents, 6)
    assert [list(np.flatnonzero(row)) for row in s] == [[0], [0, 1], [0, 2], [0, 1, 3], [4], [0, 1, 3, 5]]
    assert list(orc.depths(parents, 6)) == [0, 1, 1, 2, 0, 3]
    assert np.array_equal(orc.ancestors(None, 4), np.tril(np.ones((4, 4), bool)))


def test_python_operators_are_there():
    import grilly_core
    import grilly_next
    from grilly_next.backend import _bridge
    for n in ("qk_norm_rope", "qk_norm_rope_backward", "draft_step", "tree_attention", "kv_cache_keep"):
        assert hasattr(grilly_core, n) and hasattr(_bridge, n) and hasattr(grilly_next.Compute, n)


def test_heads_refuse_what_the_c_structures_would_read_as_a_default(tmp_path):
    """A caller of the operators who names 0 as eps, scaling or gain would get 1e-6 or 1 without a word."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "heads.cpp").write_text(r"""
#include <cmath>
#include <cstdio>
#include "grilly/ops/rope.h"
using namespace grilly::ops;
template <typename F> static void say(F f) { try { f(); std::puts("ok"); } catch (const std::runtime_error& e) { std::puts(e.what()); } }
int main() {
    for (float v : {1e-30f, 1.0f, 0.0f, -1.0f, NAN}) {
        say([&] { HeadNorm n; n.eps = v; n.epsilon(); });
        say([&] { HeadRope r; r.scaling = v; r.spec(); });
        say([&] { HeadRope r; r.gain = v; r.spec(); });
    }
}
""")
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    subprocess.check_call([cxx, "-std=c++17", "-I", os.path.join(root, "include"), "-I", os.path.join(root, "grilly-next_b200", "cpp", "include"),
                           str(tmp_path / "heads.cpp"), "-o", str(tmp_path / "heads")])
    said = subprocess.check_output([str(tmp_path / "heads")], text=True).split("\n")[:15]
    assert said == ["ok"] * 6 + ["eps must be positive"] + ["rope scaling and gain must be positive"] * 2 + (
        ["eps must be positive"] + ["rope scaling and gain must be positive"] * 2) * 2
