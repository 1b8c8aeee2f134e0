"""GPU: the Python operators of normalised heads and drafted steps, used together as a serving loop and a training step use them, against the
float64 oracle; host arrays against DeviceTensors; refusals.

Bounds, u = 2^-24.  A normalised and rotated head: the mean square is a float32 sum of D squares (relative error D u, half of that in its root), then
some eight roundings: (D/2 + 8) u of the head's length, which is at most sqrt(D) max|w|.  Two such heads in a product of D terms: a score is off by
at most (2 D + 16) u D max|w_q| max|w_k| scale.  A probability is off by twice that plus 2^-21 of the exponential, an output by that of
sum p|v| plus one u for every key.  Gradients: the row's terms r g and x r^3 mean(g x) are at most r |g|_2 each and carry the error of r three
times and of a sum of D products: (3 D + 32) u of twice r |g|_2; a weight's gradient adds N terms, (N + D + 16) u of their absolute sum.
"""
import numpy as np
import pytest

from oracle import tree_oracle as orc

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def core():
    import grilly_core
    return grilly_core


@pytest.fixture(scope="module")
def gpu():
    from grilly_next import Compute
    return Compute()


def draw(r, *shape):
    return r.standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("mode,rotary,D,group,batch", [("half", 0, 64, 2, 1), ("interleaved", 16, 32, 3, 3), ("half", 64, 128, 4, 2)])
def test_a_serving_loop(gpu, mode, rotary, D, group, batch):
    """Prompt, then three drafted trees of which a path is kept: outputs, lengths and the cache's rows."""
    r = np.random.default_rng(D + batch)
    hkv, hq, T, prompt, rot = 2, 2 * group, 9, 21, rotary or D
    wq, wk = (1 + 0.3 * draw(r, D)), (1 + 0.3 * draw(r, D))
    freq = orc.frequencies(rot)
    kw = dict(rope_theta=10000.0, rope_mode=mode, rotary_dim=rotary)
    kv = gpu.create_kv_cache(num_heads=hkv, head_dim=D, compression_ratio=1, max_cache_tokens=128, use_h2o=False, batch_size=batch, page_tokens=8,
                             dtype="fp32")
    q0, k0, v0 = draw(r, batch, prompt, hq, D), draw(r, batch, prompt, hkv, D), draw(r, batch, prompt, hkv, D)
    _, k_rot = gpu.qk_norm_rope(q0, k0, wq, wk, **kw)
    row_bound = (D / 2 + 8) * U * np.sqrt(D) * np.abs(wk).max()
    pos = np.broadcast_to(np.arange(prompt), (batch, prompt))
    assert np.abs(k_rot - orc.norm_rope(k0, wk, pos, freq, mode)).max() <= row_bound
    gpu.kv_cache_append(kv, k_rot, v0)
    keys = [list(orc.norm_rope(k0[b], wk, np.arange(prompt), freq, mode)) for b in range(batch)]
    values = [list(v0[b]) for b in range(batch)]
    for step in range(3):
        counts = [int(r.integers(0 if b else 1, T + 1)) for b in range(batch)]
        parents = np.array([[-1] + [int(r.integers(-1, t)) for t in range(1, T)] for _ in range(batch)], np.int32)
        q, k, v = draw(r, batch, T, hq, D), draw(r, batch, T, hkv, D), draw(r, batch, T, hkv, D)
        out = gpu.draft_step(kv, q, k, v, parents, counts, q_weight=wq, k_weight=wk, **kw)
        paths = []
        for b, n in enumerate(counts):
            assert not out[b, n:].any()
            at = len(keys[b]) + orc.depths(parents[b], n)
            kb, qb = orc.norm_rope(k[b, :n], wk, at, freq, mode), orc.norm_rope(q[b, :n], wq, at, freq, mode)
            if n:
                K, V = np.array(keys[b] + list(kb)), np.array(values[b] + list(v[b, :n]), np.float64)
                want, size = orc.tree_attention(qb, K, V, n, parents[b], D ** -0.5)
                score = (2 * D + 16) * U * D * np.abs(wq).max() * np.abs(wk).max() * D ** -0.5
                assert (np.abs(out[b, :n] - want) <= (2 * score + 2.0 ** -21 + len(K) * U) * size + 2 * U * np.abs(want)).all()
            leaf = int(r.integers(0, n)) if n else -1
            path = np.flatnonzero(orc.ancestors(parents[b], n)[leaf]).tolist() if n else []
            paths.append(path)
            keys[b] += [kb[t] for t in path]
            values[b] += [v[b, t] for t in path]
        gpu.kv_cache_keep(kv, paths)
        assert kv.seq_lens == [len(x) for x in keys]
        for b in range(batch):
            got = gpu.kv_cache_decode(kv, b)
            assert np.abs(got["keys"] - np.array(keys[b])).max() <= row_bound and np.array_equal(got["values"], np.array(values[b], np.float32))
    gpu.destroy_kv_cache(kv)


def test_device_tensors_and_host_arrays_give_the_same(core):
    """bf16 over the tensor cores and float32: the same bits either way, and the attention alone repeats the step's."""
    r = np.random.default_rng(5)
    ctx = core.Device()
    B, T, hq, hkv, D = 2, 12, 8, 2, 128
    parents = np.array([[-1] + [int(r.integers(-1, t)) for t in range(1, T)] for _ in range(B)], np.int32)
    k0 = draw(r, B, 150, hkv, D)
    q, k, v, w = draw(r, B, T, hq, D), draw(r, B, T, hkv, D), draw(r, B, T, hkv, D), 1 + 0.1 * draw(r, D)
    for dtype in ("bf16", "fp32"):
        caches = [core.create_kv_cache(ctx, num_heads=hkv, head_dim=D, compression_ratio=1, max_cache_tokens=256, use_h2o=False, batch_size=B,
                                       dtype=dtype) for _ in range(2)]
        for kv in caches:
            core.kv_cache_append(ctx, kv, k0, k0)
        tq, tk, tv = (core.DeviceTensor.from_numpy(ctx, x, dtype=dtype) for x in (q, k, v))
        tw = core.DeviceTensor.from_numpy(ctx, w)
        host = core.draft_step(ctx, caches[0], q, k, v, parents, [T, T - 5], q_weight=w, k_weight=w, dtype=dtype)
        dev = core.draft_step(ctx, caches[1], tq, tk, tv, parents, [T, T - 5], q_weight=tw, k_weight=tw)
        assert dev.dtype == dtype and np.array_equal(dev.to_numpy(), host)
        pos = np.array([[150 + d for d in orc.depths(parents[b], T)] for b in range(B)], np.int32)
        rotated = core.qk_norm_rope(ctx, tq, q_weight=tw, positions=pos)
        again = core.tree_attention(ctx, rotated, caches[1], parents).to_numpy()
        assert np.array_equal(again[0], host[0]) and np.array_equal(again[1, :T - 5], host[1, :T - 5]) and not again[1, T - 5:].any()
        for kv in caches:
            core.kv_cache_keep(ctx, kv, [[0], []])
            assert kv.seq_lens == [151, 150]
            core.destroy_kv_cache(ctx, kv)


@pytest.mark.parametrize("mode,D,rotary", [("half", 64, 0), ("interleaved", 96, 32)])
def test_a_training_step(gpu, mode, D, rotary):
    """Forward and gradients through the operators: against the formula's, and along one direction against differences of the oracle."""
    r = np.random.default_rng(D)
    B, S, hq, hkv, rot = 2, 37, 6, 2, rotary or D
    freq, pos = orc.frequencies(rot), np.broadcast_to(np.arange(S) + 3, (B, S))
    q, k, dq, dk = draw(r, B, S, hq, D), draw(r, B, S, hkv, D), draw(r, B, S, hq, D), draw(r, B, S, hkv, D)
    wq, wk = 1 + 0.2 * draw(r, D), 1 + 0.2 * draw(r, D)
    g = gpu.qk_norm_rope_backward(dq, dk, q, k, wq, wk, rope_mode=mode, rotary_dim=rotary, pos_base=3)
    for x, w, dy, gx, gw in ((q, wq, dq, "grad_q", "grad_q_weight"), (k, wk, dk, "grad_k", "grad_k_weight")):
        want, want_w = orc.norm_rope_grad(x, w, dy, pos, freq, mode)
        x64 = x.astype(np.float64)
        root = 1 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + 1e-6)
        size = root * np.abs(w).max() * np.sqrt((dy.astype(np.float64) ** 2).sum(-1, keepdims=True))
        assert (np.abs(g[gx] - want) <= (3 * D + 32) * U * 2 * size).all()
        terms = np.abs(orc.rotate(dy, pos, freq, mode, back=True) * x64 * root).reshape(-1, D).sum(0)
        assert (np.abs(g[gw] - want_w) <= (x.size // D + D + 16) * U * 4 * terms).all()
        step = draw(r, *x.shape).astype(np.float64)
        h = 1e-5
        diff = ((orc.norm_rope(x64 + h * step, w, pos, freq, mode) - orc.norm_rope(x64 - h * step, w, pos, freq, mode)) * dy).sum() / (2 * h)
        # the gradient's own bound along the step, and the difference's: its third derivative times h^2, and cancellation
        slack = ((3 * D + 32) * U * 2 * size * np.abs(step)).sum() + 1e-6 * (np.abs(want * step)).sum()
        assert abs((g[gx].astype(np.float64) * step).sum() - diff) <= slack


def test_refusals(gpu):
    z = lambda *s: np.zeros(s, np.float32)
    kv = gpu.create_kv_cache(num_heads=2, head_dim=32, compression_ratio=1, max_cache_tokens=64, use_h2o=False, batch_size=2, page_tokens=16)
    q, k = z(2, 4, 4, 32), z(2, 4, 2, 32)
    with pytest.raises(RuntimeError, match="does not end with the nodes"):
        gpu.kv_cache_keep(kv, [[0], [0]])
    with pytest.raises(RuntimeError, match="does not end with the nodes"):
        gpu.tree_attention(q, kv)
    for parents, counts, text in (([[0, 0, 0, 0]] * 2, None, "earlier node"), ([[-1, 0, 2, 0]] * 2, None, "earlier node"),
                                  ([[-2, 0, 0, 0]] * 2, None, "earlier node"), ([[-1, 0, 0]] * 2, None, "parents must be"), (None, [5, 1], "out of range"),
                                  (None, [-1, 1], "out of range"), (None, [1], "n_nodes must be")):
        with pytest.raises(RuntimeError, match=text):
            gpu.draft_step(kv, q, k, k, parents, counts)
    for bad in (dict(q=z(2, 4, 3, 32)), dict(q=z(2, 4, 4, 64)), dict(k=z(2, 3, 2, 32)), dict(v=z(2, 4, 1, 32)), dict(q=z(1, 4, 4, 32)), dict(q=z(4, 4, 32))):
        with pytest.raises(RuntimeError):
            gpu.draft_step(kv, bad.get("q", q), bad.get("k", k), bad.get("v", k))
    with pytest.raises(RuntimeError, match="q_weight must be"):
        gpu.draft_step(kv, q, k, k, q_weight=z(16))
    with pytest.raises(RuntimeError, match="1 to 128 nodes"):
        gpu.draft_step(kv, z(2, 129, 4, 32), z(2, 129, 2, 32), z(2, 129, 2, 32))
    with pytest.raises(RuntimeError, match="max_cache_tokens"):
        gpu.draft_step(kv, z(2, 65, 4, 32), z(2, 65, 2, 32), z(2, 65, 2, 32))
    assert kv.seq_lens == [0, 0]
    gpu.draft_step(kv, q, k, k, None, [4, 2])
    for paths in ([[0]], [[1, 1], []], [[2, 1], []], [[0], [2]], [[-1], []]):
        with pytest.raises(RuntimeError):
            gpu.kv_cache_keep(kv, paths)
    assert kv.seq_lens == [4, 2]
    gpu.kv_cache_keep(kv, [[0, 3], [1]])
    assert kv.seq_lens == [2, 1]
    with pytest.raises(RuntimeError, match="does not end with the nodes"):
        gpu.kv_cache_keep(kv, [[0], [0]])
    gpu.draft_step(kv, q, k, k)
    gpu.kv_cache_append(kv, k, k)
    with pytest.raises(RuntimeError, match="does not end with the nodes"):       # the nodes are no longer the last rows
        gpu.kv_cache_keep(kv, [[0], [0]])
    for extra in (dict(use_asymmetric_quant=True, compression_ratio=1, batch_size=2), dict(compression_ratio=4)):
        other = gpu.create_kv_cache(num_heads=2, head_dim=32, max_cache_tokens=64, use_h2o=False, **extra)
        n = extra.get("batch_size", 1)
        with pytest.raises(RuntimeError, match="not built for the"):
            gpu.draft_step(other, q[:n], k[:n], k[:n])
        gpu.destroy_kv_cache(other)
    gpu.destroy_kv_cache(kv)
    with pytest.raises(RuntimeError, match="destroyed"):
        gpu.draft_step(kv, q, k, k)
    with pytest.raises(RuntimeError):
        gpu.qk_norm_rope(z(2, 4, 32))
    with pytest.raises(RuntimeError, match="positions must be"):
        gpu.qk_norm_rope(q, positions=np.zeros((2, 5), np.int32))
    with pytest.raises(RuntimeError, match="go together"):
        gpu.qk_norm_rope_backward(q, None, q, k)


@pytest.mark.parametrize("mode,rotary", [("interleaved", 0), ("interleaved", 40), ("half", 0), ("half", 40)])
@pytest.mark.parametrize("D", [40, 72, 80, 136])
def test_rows_that_leave_threads_idle(gpu, D, mode, rotary):
    """Head sizes between powers of two, behind a call that has left NaN in every multiprocessor's shared memory."""
    r = np.random.default_rng(D)
    big, nan = np.ones((4, 256, 8, 256), np.float32), np.full(256, np.nan, np.float32)
    x, dy, w = draw(r, 4, 99, 5, D), draw(r, 4, 99, 5, D), 1 + 0.2 * draw(r, D)
    rotary = rotary if rotary <= D else 0
    gpu.qk_norm_rope_backward(big, None, big, None, nan)
    g = gpu.qk_norm_rope_backward(dy, None, x, None, w, rope_mode=mode, rotary_dim=rotary)
    pos = np.broadcast_to(np.arange(99), (4, 99))
    want, _ = orc.norm_rope_grad(x, w, dy, pos, orc.frequencies(rotary or D), mode)
    x64 = x.astype(np.float64)
    size = np.abs(w).max() * np.sqrt((dy.astype(np.float64) ** 2).sum(-1, keepdims=True) / ((x64 * x64).mean(-1, keepdims=True) + 1e-6))
    assert (np.abs(g["grad_q"] - want) <= (3 * D + 32) * U * 2 * size).all()


@pytest.mark.parametrize("T,group,dtype", [(4, 4, "bf16"), (5, 4, "bf16"), (16, 4, "bf16"), (31, 4, "bf16"), (61, 4, "bf16"), (128, 8, "bf16"),
                                           (11, 3, "fp32")])
def test_many_calls_give_the_same_bits(core, T, group, dtype):
    """Ragged sequences, calls back to back without a wait between them."""
    r = np.random.default_rng(T)
    ctx = core.Device()
    B, hkv, D = 6, 8, 128
    kv = core.create_kv_cache(ctx, num_heads=hkv, head_dim=D, compression_ratio=1, max_cache_tokens=2048, use_h2o=False, batch_size=B, dtype=dtype)
    core.kv_cache_append(ctx, kv, draw(r, B, 1501, hkv, D), draw(r, B, 1501, hkv, D))
    q, k, v = (core.DeviceTensor.from_numpy(ctx, draw(r, B, T, h, D), dtype=dtype) for h in (hkv * group, hkv, hkv))
    parents = np.array([[-1] + [int(r.integers(-1, t)) for t in range(1, T)] for _ in range(B)], np.int32)
    core.draft_step(ctx, kv, q, k, v, parents, [T, 1, 0, T // 2, T, T - 1])
    outs = [core.tree_attention(ctx, q, kv, parents) for _ in range(120)]
    first = outs[0].to_numpy()
    assert np.isfinite(first).all() and first[0].any() and not first[2].any()
    assert all(np.array_equal(o.to_numpy(), first) for o in outs[1:])
    core.destroy_kv_cache(ctx, kv)


def test_heads_without_a_rotation(gpu):
    """rope_theta = 0: normalised only, wherever the tokens stand."""
    r = np.random.default_rng(3)
    x, w = draw(r, 2, 7, 3, 64), 1 + 0.1 * draw(r, 64)
    want = orc.norm(x, w, 1e-6)
    got = gpu.qk_norm_rope(x, q_weight=w, rope_theta=0.0, pos_base=1000)
    assert (np.abs(got - want) <= (64 / 2 + 8) * U * np.abs(want) + 2.0 ** -126).all()


def test_a_refused_step_gives_out_no_pages(gpu):
    """One sequence has room and the other has not: the call is refused, and the next one finds the pages as they were."""
    r = np.random.default_rng(11)
    kv = gpu.create_kv_cache(num_heads=1, head_dim=32, compression_ratio=1, max_cache_tokens=32, use_h2o=False, batch_size=2, page_tokens=8, dtype="fp32")
    rows = [[], []]
    for counts, fits in (([8, 28], True), ([8, 8], False), ([8, 2], True), ([8, 0], True)):
        n = max(counts)
        q, k, v = draw(r, 2, n, 2, 32), draw(r, 2, n, 1, 32), draw(r, 2, n, 1, 32)
        if not fits:
            with pytest.raises(RuntimeError, match="max_cache_tokens"):
                gpu.draft_step(kv, q, k, v, None, counts)
            continue
        gpu.draft_step(kv, q, k, v, None, counts)
        for b in range(2):
            rows[b] += list(v[b, :counts[b]])
    for b in range(2):
        assert np.array_equal(gpu.kv_cache_decode(kv, b)["values"], np.array(rows[b]))
    gpu.destroy_kv_cache(kv)


def test_a_step_that_the_attention_refuses_is_not_appended(gpu):
    """What only the attention refuses comes before the append: the lengths stay, and the step that follows is that of a cache which saw no refusal."""
    r = np.random.default_rng(12)
    make = lambda: gpu.create_kv_cache(num_heads=2, head_dim=32, compression_ratio=1, max_cache_tokens=64, use_h2o=False, batch_size=2,  # noqa: E731
                                       page_tokens=16, dtype="fp32")
    q, k, v = draw(r, 2, 3, 4, 32), draw(r, 2, 3, 2, 32), draw(r, 2, 3, 2, 32)
    kv, fresh = make(), make()
    for cache in (kv, fresh):
        gpu.draft_step(cache, q, k, v, None, [3, 2])
    for bad in (dict(scale=-1.0), dict(scale=float("nan"))):
        with pytest.raises(RuntimeError, match="scale"):
            gpu.draft_step(kv, q, k, v, **bad)
        assert kv.seq_lens == [3, 2]
    gpu.kv_cache_keep(kv, [[0], [0, 1]])                         # the nodes are still those of the step before
    gpu.kv_cache_keep(fresh, [[0], [0, 1]])
    assert np.array_equal(gpu.draft_step(kv, q, k, v), gpu.draft_step(fresh, q, k, v))
    assert kv.seq_lens == fresh.seq_lens == [4, 5]
    for cache in (kv, fresh):
        gpu.destroy_kv_cache(cache)


@pytest.mark.parametrize("bad", [dict(eps=0.0), dict(eps=-1e-6), dict(rope_scaling=0.0), dict(rope_gain=0.0), dict(rope_gain=-1.0)], ids=str)
def test_numbers_that_would_be_read_as_a_default_are_refused(gpu, bad):
    x = np.ones((2, 3, 2, 32), np.float32)
    kv = gpu.create_kv_cache(num_heads=2, head_dim=32, compression_ratio=1, max_cache_tokens=64, use_h2o=False, batch_size=2, page_tokens=16)
    for call in (lambda: gpu.qk_norm_rope(x, x, **bad), lambda: gpu.qk_norm_rope_backward(x, x, x, x, **bad), lambda: gpu.draft_step(kv, x, x, x, **bad)):
        with pytest.raises(RuntimeError, match="must be positive"):
            call()
    assert kv.seq_lens == [0, 0]
    gpu.destroy_kv_cache(kv)
