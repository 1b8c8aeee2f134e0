"""GPU: drafted steps over the paged cache -- append of normalised and rotated heads, attention of trees, keeping the accepted path --
against the float64 oracle.

Bounds of the attention, u = 2^-24.  Scores: a float32 sum of D products, off by at most D u sum|q_d k_d| scale (bf16 products are exact in it),
and the factor scale; a probability then is off by twice the largest such error of its row plus 2^-21 of the exponential, an output
by that of sum p|v|, plus one u for every key that is added up.  Tensor cores: probabilities are rounded to bf16, half a step = 2^-8 of
each.  A bf16 output adds half a step, 2^-8 of itself.  What test_gpu_qk_norm.py says of rows holds for the append's.
"""
import ctypes as C

import numpy as np
import pytest

from oracle import tree_oracle as orc
from oracle.attention_oracle import from_bf16_bits, round_bf16, to_bf16_bits

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    from grilly_next import cabi
    d = cabi.Device(0)
    yield d
    d.close()


def draw_parents(r, T, kind):
    if kind == "chain":
        return None
    if kind == "star":                       # all of them follow the cached tokens
        return [-1] * T
    if kind == "line":                       # a chain, given as a tree
        return [t - 1 for t in range(T)]
    return [-1] + [int(r.integers(max(-1, t - 9), t)) for t in range(1, T)]


class Cache:
    """A paged cache filled from the host: rows[b] (len, Hkv, D) for keys and values; everything else is NaN."""

    def __init__(self, dev, lens, Hkv, D, page, dtype, room=0, seed=0, spare=3):
        from grilly_next import cabi
        self.cabi, self.dev, self.B, self.Hkv, self.D, self.P, self.dtype = cabi, dev, len(lens), Hkv, D, page, dtype
        r = np.random.default_rng(1000 + seed)
        rnd = round_bf16 if dtype == "bf16" else (lambda x: x)
        self.rows = [[rnd(r.standard_normal((n, Hkv, D)).astype(np.float32)) for n in lens] for _ in range(2)]
        self.max_pages = max(1, -(-(max(lens) + room) // page))
        self.num_pages = self.B * self.max_pages + spare
        self.table = r.permutation(self.num_pages)[:self.B * self.max_pages].reshape(self.B, self.max_pages).astype(np.int32)
        self.pools = [np.full((self.num_pages, Hkv, page, D), np.nan, np.float32) for _ in range(2)]
        for i in range(2):
            for b, n in enumerate(lens):
                for t in range(n):
                    self.pools[i][self.table[b, t // page], :, t % page] = self.rows[i][b][t]
        self.ptr = [self.upload(p) for p in self.pools]
        self.lens = np.array(lens, np.int32)
        self.table_ptr, self.lens_ptr = dev.upload(self.table), dev.upload(self.lens)

    def upload(self, p):
        return self.dev.upload(p if self.dtype == "f32" else to_bf16_bits(p.reshape(-1)))

    def put(self, which, b, t, value):
        """Overwrites row t of sequence b in the device pools."""
        p = self.pools[which]
        p[self.table[b, t // self.P], :, t % self.P] = value
        self.dev.free(self.ptr[which])
        self.ptr[which] = self.upload(p)

    def read(self):
        """Both pools as they are now."""
        kind = np.float32 if self.dtype == "f32" else np.uint16
        got = [self.dev.download(p, self.pools[0].shape, kind) for p in self.ptr]
        return got if self.dtype == "f32" else [from_bf16_bits(g) for g in got]

    def row_of(self, pools, b, t):
        return [p[self.table[b, t // self.P], :, t % self.P] for p in pools]

    def set_lens(self, lens):
        self.lens = np.asarray(lens, np.int32)
        self.cabi.check(self.dev.L.grl_memcpy_h2d(self.dev.h, self.lens_ptr, self.lens.ctypes.data_as(C.c_void_p), self.lens.nbytes))
        self.dev.sync()

    def layout(self):
        kv = self.cabi.KVLayout()
        kv.k_pages, kv.v_pages = self.ptr
        kv.cache_dtype = self.cabi.F32 if self.dtype == "f32" else self.cabi.BF16
        kv.block_table, kv.seq_lens = self.table_ptr, self.lens_ptr
        kv.batch, kv.num_kv_heads, kv.head_dim, kv.page_tokens = self.B, self.Hkv, self.D, self.P
        kv.max_pages, kv.num_pages = self.max_pages, self.num_pages
        return kv

    def free(self):
        for p in self.ptr + [self.table_ptr, self.lens_ptr]:
            self.dev.free(p)


def attend(dev, cache, q, parents, counts, *, io="f32", splits=0, kernel=0, scale=0.0, max_seq_len=None):
    """q (B,T,Hq,D) float32 values of the io type; returns out."""
    cabi = cache.cabi
    B, T, Hq, D = q.shape
    p = cabi.TreeParams()
    p.kv = cache.layout()
    up = (lambda x: dev.upload(x)) if io == "f32" else (lambda x: dev.upload(to_bf16_bits(x.reshape(-1))))
    size = 4 if io == "f32" else 2
    keep = [up(q), dev.upload(np.full(q.size * size + 64, 0x55, np.uint8))]
    p.q, p.out, p.io_dtype = keep[0], keep[1], cabi.F32 if io == "f32" else cabi.BF16
    p.num_q_heads, p.n_tree, p.scale, p.n_splits, p.kernel = Hq, T, scale, splits, kernel
    p.max_seq_len = int(cache.lens.max()) if max_seq_len is None else max_seq_len
    if parents is not None:
        keep.append(dev.upload(np.array(parents, np.int32)))
        p.parents = keep[-1]
    if counts is not None:
        keep.append(dev.upload(np.array(counts, np.int32)))
        p.n_nodes = keep[-1]
    need = C.c_size_t()
    cabi.check(dev.L.grl_tree_workspace_bytes(dev.h, C.byref(p), C.byref(need)))
    if need.value:
        keep.append(dev.upload(np.full(need.value + 64, 0xFF, np.uint8)))       # NaN everywhere; 64 bytes behind it
        p.workspace, p.workspace_bytes = keep[-1], need.value
    cabi.check(dev.L.grl_tree_attention(dev.h, C.byref(p)))
    try:
        dev.sync()
        raw = dev.download(keep[1], (q.size * size + 64,), np.uint8)
        assert np.all(raw[q.size * size:] == 0x55), "written behind the output"
        if need.value:
            assert np.all(dev.download(keep[-1], (need.value + 64,), np.uint8)[need.value:] == 0xFF), "written behind the workspace"
        out = raw[:q.size * size].view(np.float32 if io == "f32" else np.uint16).reshape(q.shape)
        return out.copy() if io == "f32" else from_bf16_bits(out)
    finally:
        for k in keep:
            dev.free(k)


def check_attention(got, cache, q, parents, counts, io, exact_arithmetic, scale=0.0):
    B, T, Hq, D = q.shape
    scale = scale or 1 / np.sqrt(D)
    for b in range(B):
        n = T if counts is None else counts[b]
        assert np.all(got[b, n:] == 0), "rows past a sequence's nodes are zero"
        if n == 0:
            continue
        k, v = cache.rows[0][b], cache.rows[1][b]
        par = None if parents is None else parents[b]
        want, size = orc.tree_attention(q[b, :n], k, v, n, par, scale)
        products = np.abs(q[b, :n].reshape(n, Hq, D)).max() * np.abs(k).sum(-1).max() * scale
        rel = 2 * D * U * products + 2.0 ** -21 + len(k) * U + (0 if exact_arithmetic else 2.0 ** -8)
        tol = rel * size
        if io == "bf16":
            tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
        over = np.abs(got[b, :n] - want) - tol
        assert np.all(over <= 0), f"sequence {b}: off by {np.abs(got[b, :n] - want).max():.3g}, over the bound by {over.max():.3g}"


def tree_case(T, Hq, Hkv, D, page, lens, counts=None, kind="tree", cache="bf16", io=None, **kw):
    """lens: cached tokens and nodes together."""
    return dict(T=T, Hq=Hq, Hkv=Hkv, D=D, page=page, lens=lens, counts=counts, kind=kind, cache=cache, io=io or cache, kw=kw)


TREES = {
    "one_token": tree_case(1, 8, 2, 128, 64, [1]),
    "one_node": tree_case(1, 8, 2, 128, 64, [77, 300]),
    "chain": tree_case(5, 8, 2, 128, 64, [300, 70], kind="chain"),
    "chain_pages_16": tree_case(4, 32, 8, 128, 16, [1005], kind="chain"),
    "tree": tree_case(13, 8, 2, 128, 64, [400, 129]),
    "no_prefix": tree_case(40, 8, 2, 128, 32, [40, 40]),
    "no_prefix_star": tree_case(128, 4, 1, 128, 64, [128], kind="star"),
    "star": tree_case(100, 4, 1, 128, 64, [163], kind="star"),
    "line": tree_case(128, 2, 2, 128, 64, [128 + 64], kind="line"),
    "ragged": tree_case(16, 8, 2, 128, 64, [200, 5, 64, 80], [16, 5, 0, 11]),
    "nobody": tree_case(4, 8, 2, 128, 64, [100, 0], [0, 0]),
    "prefix_only_rows": tree_case(16, 8, 2, 128, 64, [130, 65], [1, 1]),
    "wide_128": tree_case(128, 8, 2, 128, 64, [500, 129], [128, 100]),
    "wide_64": tree_case(61, 16, 2, 64, 32, [333, 61]),
    "group_1": tree_case(33, 2, 2, 128, 64, [222]),
    "group_3": tree_case(11, 6, 2, 64, 16, [222, 100]),
    "group_16": tree_case(9, 32, 2, 128, 64, [222]),
    "group_5": tree_case(7, 5, 1, 128, 32, [515]),
    "page_edge": tree_case(64, 8, 2, 128, 64, [64, 128, 192, 65], [64, 64, 63, 2]),
    "scale": tree_case(6, 8, 2, 128, 64, [300], kw_scale=0.02),
    "large_scores": tree_case(6, 8, 2, 128, 64, [300], kw_scale=3.0),
    "splits_3": tree_case(16, 8, 2, 128, 64, [1000, 100, 16], kw_splits=3),
    "splits_7_wide": tree_case(64, 16, 2, 128, 64, [900, 64, 65], kw_splits=7),
    "splits_beyond": tree_case(8, 8, 2, 64, 64, [100], kw_splits=9),
    "long": tree_case(20, 8, 2, 128, 64, [9000]),
    "long_few_rows": tree_case(2, 8, 2, 128, 64, [9000, 8000], kind="chain"),
    "batch": tree_case(16, 8, 4, 128, 64, [300 + 17 * i for i in range(40)]),
    "batch_few_rows": tree_case(3, 8, 4, 64, 64, [300 + 17 * i for i in range(40)]),
    "many_sequences": tree_case(3, 4, 2, 64, 64, [1 + 5 * i % 300 for i in range(3, 140)], [(i % 4) if 1 + 5 * i % 300 >= (i % 4) else 0 for i in range(3, 140)]),
    "shares_whole_and_cut": tree_case(9, 8, 4, 128, 64, [64 * (1 + 7 * i % 13) + i for i in range(9, 60)]),
    "shares_of_wide": tree_case(70, 8, 2, 128, 32, [70 + 64 * (5 * i % 11) for i in range(30)], [70 - i for i in range(30)]),
    "shares_of_three_groups": tree_case(128, 16, 2, 64, 64, [900, 128, 300]),
    "shares_of_one_tile": tree_case(30, 8, 2, 128, 64, [30 + 100 * (5 * i % 11) for i in range(30)]),
    "few_rows_one_split": tree_case(4, 8, 2, 128, 64, [700, 65, 4], kw_splits=1),
    "few_rows_joined": tree_case(4, 8, 2, 128, 16, [3000, 65, 4], [4, 2, 0], kw_splits=17),
    "few_rows_clusters": tree_case(8, 8, 2, 128, 32, [1500, 65, 8], [8, 2, 0], kw_splits=5),
    "few_rows_64": tree_case(5, 6, 2, 64, 16, [2500, 200]), "few_rows_64_wide": tree_case(10, 6, 2, 64, 64, [2500, 200], [10, 0]),
    "few_rows_32": tree_case(32, 2, 2, 128, 64, [600, 40], [32, 30]), "few_rows_17": tree_case(17, 1, 1, 128, 64, [333]),
    "few_rows_star": tree_case(16, 2, 1, 128, 64, [16, 80], kind="star"),
    "hint_too_short": tree_case(8, 8, 2, 128, 64, [700, 64], kw_max_seq_len=100),
    "f32": tree_case(11, 6, 2, 64, 24, [300, 97, 11], cache="f32"),
    "f32_dim_32": tree_case(11, 6, 2, 32, 7, [100, 50], cache="f32"),
    "f32_dim_256": tree_case(9, 4, 2, 256, 16, [100, 50], cache="f32"),
    "f32_dim_128": tree_case(128, 4, 2, 128, 64, [300, 128], cache="f32", kw_splits=4),
    "f32_one": tree_case(1, 2, 1, 64, 1, [1], cache="f32"),
    "f32_chain_splits": tree_case(3, 4, 1, 128, 48, [5000], kind="chain", cache="f32"),
    "f32_over_bf16": tree_case(11, 8, 2, 128, 64, [300, 64], io="f32"),
    "bf16_over_f32": tree_case(11, 8, 2, 128, 64, [300, 64], cache="f32", io="bf16"),
    "bf16_dim_32": tree_case(11, 8, 2, 32, 64, [300, 64]),
    "bf16_dim_256": tree_case(11, 8, 2, 256, 64, [300, 64]),
    "bf16_page_24": tree_case(11, 8, 2, 128, 24, [300, 64]),
}


def run_tree(dev, c, kernel=0, seed=0):
    r = np.random.default_rng(seed)
    cache = Cache(dev, c["lens"], c["Hkv"], c["D"], c["page"], c["cache"], seed=seed)
    q = r.standard_normal((len(c["lens"]), c["T"], c["Hq"], c["D"])).astype(np.float32)
    q = round_bf16(q) if c["io"] == "bf16" else q
    parents = None if c["kind"] == "chain" else [draw_parents(r, c["T"], c["kind"]) for _ in c["lens"]]
    kw = {k[3:]: v for k, v in c["kw"].items()}
    got = attend(dev, cache, q, parents, c["counts"], io=c["io"], kernel=kernel, **kw)
    return got, cache, q, parents


@pytest.mark.parametrize("name", list(TREES))
def test_tree_attention(dev, name):
    c = TREES[name]
    got, cache, q, parents = run_tree(dev, c)
    check_attention(got, cache, q, parents, c["counts"], c["io"], not (c["cache"] == c["io"] == "bf16"), c["kw"].get("kw_scale", 0.0))
    cache.free()


@pytest.mark.parametrize("name", ["one_token", "tree", "ragged", "wide_128", "wide_64", "splits_3", "star", "hint_too_short"])
def test_float32_arithmetic_on_request(dev, name):
    from grilly_next import cabi
    c = TREES[name]
    got, cache, q, parents = run_tree(dev, c, kernel=cabi.KERNEL_SIMT_F32)
    check_attention(got, cache, q, parents, c["counts"], c["io"], True, c["kw"].get("kw_scale", 0.0))
    cache.free()


@pytest.mark.parametrize("T,kind,cache_type", [(4, "tree", "bf16"), (6, "tree", "bf16"), (30, "tree", "bf16"), (15, "tree", "bf16"), (70, "tree", "bf16"), (2, "star", "bf16"), (6, "tree", "f32")])
def test_what_a_row_does_not_see_may_be_anything(dev, T, kind, cache_type):
    """Keys and values of other branches hold NaN and infinities: rows that do not see them are as if they were not there; the rest of the
    pools, past every sequence's end, is NaN in all of these tests."""
    r = np.random.default_rng(5)
    bad = T // 2
    for which, value in ((0, np.nan), (0, np.inf), (1, np.nan), (1, -np.inf)):
        cache = Cache(dev, [100 + T, T], 2, 128, 64, cache_type, seed=3)
        parents = [draw_parents(r, T, kind) for _ in range(2)]
        q = round_bf16(r.standard_normal((2, T, 8, 128)).astype(np.float32))
        clean = attend(dev, cache, q, parents, None, io=cache_type)
        for b, n in enumerate(cache.lens):
            cache.put(which, b, n - T + bad, value)
        got = attend(dev, cache, q, parents, None, io=cache_type)
        for b in range(2):
            sees = orc.ancestors(parents[b], T)[:, bad]
            assert np.array_equal(got[b, ~sees], clean[b, ~sees])
            if which == 1:
                assert np.all(np.isnan(got[b, sees]) if np.isnan(value) else got[b, sees] == value)
        cache.free()


@pytest.mark.parametrize("T", [2, 8, 12, 30, 64])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(T):
    """A budget of one cycle for the waits of long streams (a wait that the hardware suspends may still succeed, so the call is made until one runs
    out): the kernel returns, the failure is reported, and the call after it gives what the call before gave."""
    from grilly_next import cabi
    dev = cabi.Device(0)
    cache = Cache(dev, [20000, 9000 + T], 2, 128, 64, "bf16", seed=6)
    r = np.random.default_rng(6)
    q = round_bf16(r.standard_normal((2, T, 8, 128)).astype(np.float32))
    parents = [draw_parents(r, T, "tree") for _ in range(2)]
    want = attend(dev, cache, q, parents, None, io="bf16")
    cabi.check(dev.L.grl_device_set_wait_limits(dev.h, 1, 0))
    for _ in range(100):
        try:
            assert np.array_equal(attend(dev, cache, q, parents, None, io="bf16"), want)
        except cabi.GrlError as e:
            assert e.code == cabi.ERR_TIMEOUT and "tree attention" in str(e)
            break
    else:
        raise AssertionError("no wait ran out")
    cabi.check(dev.L.grl_device_set_wait_limits(dev.h, 0, 0))
    for _ in range(3):
        assert np.array_equal(attend(dev, cache, q, parents, None, io="bf16"), want)
    cache.free()
    dev.close()


# T, group, cache and io type, splits: every form of the kernels, whole, joined in a cluster and joined behind
FORMS = [(1, 4, "bf16", 1), (4, 4, "bf16", 3), (4, 4, "bf16", 17), (12, 4, "bf16", 1), (12, 4, "bf16", 4), (24, 4, "bf16", 1), (24, 4, "bf16", 5),
         (40, 4, "bf16", 1), (40, 4, "bf16", 3), (100, 4, "bf16", 2), (6, 4, "f32", 1), (6, 4, "f32", 4)]


@pytest.mark.parametrize("T,group,io,splits", FORMS)
def test_what_is_no_number_comes_out_as_none(T, group, io, splits):
    """A row whose scores hold a NaN is NaN, and so is one whose scores are all -inf, in every form; a single score of -inf has no weight; the other
    rows are as without it."""
    from grilly_next import cabi
    dev = cabi.Device(0)
    r = np.random.default_rng(21)
    Hkv, D, lens = 2, 128, [700 + T, T, 130 + T]
    counts = [T, T, T // 2]
    cache = Cache(dev, lens[:2] + [130 + T // 2], Hkv, D, 64, io, seed=21)
    parents = [draw_parents(r, T, "tree") for _ in lens]
    q = round_bf16(r.standard_normal((3, T, Hkv * group, D)).astype(np.float32))
    q[..., 0] = 1 + np.abs(q[..., 0])
    q = round_bf16(q)
    call = lambda x: attend(dev, cache, x, parents, counts, io=io, splits=splits)  # noqa: E731
    clean = call(q)
    check_attention(clean, cache, q, parents, counts, io, io == "f32")
    # a query
    bad = q.copy()
    bad[0, T - 1, 1, 5] = bad[1, 0, group, 77] = bad[2, 0, 0, 0] = np.nan
    bad[2, T // 2:] = np.nan                                     # rows of padding
    got = call(bad)
    hit = np.isnan(bad).any(-1)
    hit[2, T // 2:] = False
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])
    # a key among the cached tokens, of one head; a key of a node
    for b, at, value in ((0, 3, np.nan), (0, 699, np.nan), (2, 129, np.nan), (1, T // 3, np.nan)):
        keep = cache.pools[0].copy()
        cache.pools[0][cache.table[b, at // 64], 1, at % 64, 9] = value
        cache.put(0, b, at, cache.pools[0][cache.table[b, at // 64], :, at % 64].copy())
        got = call(q)
        hit = np.zeros(got.shape[:3], bool)
        first = cache.lens[b] - counts[b]
        sees = np.ones(counts[b], bool) if at < first else orc.ancestors(parents[b], counts[b])[:, at - first]
        hit[b, :counts[b], group:] = sees[:, None]
        assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])
        cache.pools[0] = keep
    # every key of a head -inf, then all but one
    keep = cache.pools[0].copy()
    cache.pools[0][:, 1, :, 0] = -np.inf
    cache.put(0, 0, 0, cache.pools[0][cache.table[0, 0], :, 0].copy())
    got = call(q)
    hit = np.zeros(got.shape[:3], bool)
    for b in range(3):
        hit[b, :counts[b], group:] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])
    cache.put(0, 0, 5, keep[cache.table[0, 0], :, 5])
    got = call(q)
    for h in range(group, 2 * group):
        v = cache.rows[1][0][5, 1]
        assert (np.abs(got[0, :, h] - v) <= 2.0 ** -7 * np.abs(v)).all()       # a weight of one, rounded twice at the most
    cache.free()
    dev.close()


@pytest.mark.parametrize("T,group,io,splits", FORMS)
def test_infinities_among_the_cached_values(dev, T, group, io, splits):
    """Every node sees the cached tokens: an infinite value of one is the result of its column, both infinities are NaN, in every form; the other columns,
    heads and sequences are as without them."""
    r = np.random.default_rng(22)
    Hkv, D, P = 2, 128, 64
    counts = [T, T, max(T // 2, 1)]
    first = [700, 0, 130]
    cache = Cache(dev, [f + n for f, n in zip(first, counts)], Hkv, D, P, io, seed=22)
    parents = [draw_parents(r, T, "tree") for _ in counts]
    q = round_bf16(r.standard_normal((3, T, Hkv * group, D)).astype(np.float32))
    call = lambda: attend(dev, cache, q, parents, counts, io=io, splits=splits)  # noqa: E731
    clean = call()
    want = clean.copy()
    for b, at, column, value in ((0, 3, 9, np.inf), (0, 697, 10, -np.inf), (0, 300, 127, np.inf), (2, 129, 64, -np.inf), (2, 100, 65, np.inf)):
        cache.pools[1][cache.table[b, at // P], 1, at % P, column] = value
        want[b, :counts[b], group:, column] = value
    for at, value in ((40, np.inf), (41, -np.inf), (500, np.inf)):
        cache.pools[1][cache.table[0, at // P], 1, at % P, 77] = value
    want[0, :, group:, 77] = np.nan
    cache.pools[1][cache.table[0, 650 // P], 0, 650 % P, 0] = np.nan
    want[0, :, :group, 0] = np.nan
    # and a node's: added to an infinity of the other sign it is NaN, for the rows that see it
    node = T // 2
    sees = orc.ancestors(parents[0], T)[:, node]
    cache.pools[1][cache.table[0, (700 + node) // P], 1, (700 + node) % P, 9] = -np.inf
    want[0, sees, group:, 9] = np.nan
    cache.put(1, 0, 0, cache.pools[1][cache.table[0, 0], :, 0].copy())
    assert np.array_equal(call(), want, equal_nan=True)
    cache.free()


def single_stages_that_run_out(T, splits, B=24):
    """Shares of one stage: all copies are on their way before any wait begins, and whoever asked for them waits no more.  With waits of one cycle
    it is a reader that gives up, and the kernel may leave only when the copies have landed: the calls in between take the same shared memory,
    and give what they gave before.  Many CTAs and a cold L2, so that copies take longer than the hardware suspends a wait."""
    from grilly_next import cabi
    dev = cabi.Device(0)
    cache = Cache(dev, [64 * (splits - 1) + T + b % (65 - T) for b in range(B)], 8, 128, 64, "bf16", seed=12)
    other = dev.malloc(1 << 28)
    q = round_bf16(np.random.default_rng(12).standard_normal((B, T, 32, 128)).astype(np.float32))
    call = lambda: attend(dev, cache, q, None, None, io="bf16", splits=splits)  # noqa: E731
    want = call()
    check_attention(want, cache, q, None, None, "bf16", False)
    ran_out = 0
    for _ in range(100):
        cabi.check(dev.L.grl_memset(dev.h, other, 0, 1 << 28))
        cabi.check(dev.L.grl_device_set_wait_limits(dev.h, 1, 0))
        try:
            assert np.array_equal(call(), want)
        except cabi.GrlError as e:
            assert e.code == cabi.ERR_TIMEOUT and "tree attention" in str(e)
            ran_out += 1
        cabi.check(dev.L.grl_device_set_wait_limits(dev.h, 0, 0))
        assert np.array_equal(call(), want)
        if ran_out == 8:
            break
    assert ran_out
    dev.free(other)
    cache.free()
    dev.close()


@pytest.mark.parametrize("T,splits,B", [(1, 9, 24), (4, 6, 24), (4, 20, 24), (4, 6, 2), (4, 12, 1)])
def test_a_reader_that_gives_up_leaves_no_copies_behind_few_rows(T, splits, B):
    """Joined behind, and in clusters where there are few sequences."""
    single_stages_that_run_out(T, splits, B)


@pytest.mark.parametrize("T,splits", [(8, 9), (16, 6), (20, 8), (61, 7)])
def test_a_reader_that_gives_up_leaves_no_copies_behind_tiles(T, splits):
    """Shares of a chain, the folded and the split tile and two tiles: products in flight end as well before the tensor memory is given back."""
    single_stages_that_run_out(T, splits, 6)


def test_refusals_of_the_tensor_core_kernel(dev):
    from grilly_next import cabi
    for c in (TREES["f32"], TREES["bf16_page_24"], TREES["bf16_dim_32"], TREES["f32_over_bf16"]):
        with pytest.raises(cabi.GrlError) as e:
            run_tree(dev, c, kernel=cabi.KERNEL_TCGEN05)
        assert e.value.code == cabi.ERR_UNSUPPORTED


@pytest.mark.parametrize("fault", ["parent_forward", "parent_self", "parent_below", "count_high", "count_negative", "length", "length_long"])
@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_bad_numbers_raise_the_status_word_and_give_zeros(dev, fault, io):
    """The numbers are checked by the kernel before it uses them: nothing is read out of range."""
    from grilly_next import cabi
    T = 8
    cache = Cache(dev, [100, 90], 2, 128, 64, io, seed=1)
    r = np.random.default_rng(0)
    parents = [draw_parents(r, T, "tree") for _ in range(2)]
    counts = [T, T]
    if fault == "parent_forward": parents[1][3] = 5
    if fault == "parent_self": parents[1][3] = 3
    if fault == "parent_below": parents[1][3] = -2
    if fault == "count_high": counts[1] = T + 1
    if fault == "count_negative": counts[1] = -1
    if fault == "length": cache.set_lens([100, T - 1])
    if fault == "length_long": cache.set_lens([100, cache.max_pages * 64 + 1])
    q = round_bf16(r.standard_normal((2, T, 8, 128)).astype(np.float32))
    with pytest.raises(cabi.GrlError) as e:
        attend(dev, cache, q, parents, counts, io=io)
    assert e.value.code == cabi.ERR_KERNEL and "sequence 1" in str(e.value)
    # and the next call is served
    cache.set_lens([100, 90])
    parents = [draw_parents(r, T, "tree") for _ in range(2)]
    got = attend(dev, cache, q, parents, None, io=io)
    check_attention(got, cache, q, parents, None, io, io == "f32")
    cache.free()


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_page_outside_the_pool_raises_the_status_word(dev, io):
    from grilly_next import cabi
    cache = Cache(dev, [200, 90], 2, 128, 64, io, seed=1)
    q = round_bf16(np.random.default_rng(0).standard_normal((2, 4, 8, 128)).astype(np.float32))
    for page in (cache.num_pages, -1):
        bad = cache.table.copy()
        bad[0, 1] = page
        cabi.check(dev.L.grl_memcpy_h2d(dev.h, cache.table_ptr, bad.ctypes.data_as(C.c_void_p), bad.nbytes))
        with pytest.raises(cabi.GrlError) as e:
            attend(dev, cache, q, None, None, io=io)
        assert e.value.code == cabi.ERR_KERNEL and "page" in str(e.value)
    cache.free()


@pytest.mark.parametrize("fault", ["parent_forward", "parent_below", "count_high", "count_negative", "length", "length_long", "page_high", "page_negative"])
@pytest.mark.parametrize("T,splits", [(4, 1), (4, 4), (4, 17), (8, 1), (24, 3), (40, 1), (100, 2)])
def test_bad_numbers_in_every_tensor_core_form(dev, T, splits, fault):
    """Few rows, the folded and the split tile, two tiles; whole, in a cluster and joined.  The kernels check every number before they use it; the rows of
    a sequence whose numbers do not fit are 0 (with a page outside the pool they mean nothing), those of the other sequence are right."""
    from grilly_next import cabi
    lens = [T + 200, T + 130]
    cache = Cache(dev, lens, 2, 128, 64, "bf16", seed=1)
    r = np.random.default_rng(0)
    parents, counts = [draw_parents(r, T, "tree") for _ in range(2)], [T, T]
    q = round_bf16(r.standard_normal((2, T, 8, 128)).astype(np.float32))
    given, table = [list(x) for x in parents], cache.table.copy()
    if fault == "parent_forward": given[1][2] = 3
    if fault == "parent_below": given[1][2] = -2
    if fault == "count_high": counts[1] = T + 1
    if fault == "count_negative": counts[1] = -1
    if fault == "length": cache.set_lens([lens[0], T - 1])
    if fault == "length_long": cache.set_lens([lens[0], cache.max_pages * 64 + 1])
    if fault == "page_high": table[1, 1] = cache.num_pages
    if fault == "page_negative": table[1, 0] = -1
    cabi.check(dev.L.grl_memcpy_h2d(dev.h, cache.table_ptr, table.ctypes.data_as(C.c_void_p), table.nbytes))
    p = cabi.TreeParams()
    p.kv = cache.layout()
    p.io_dtype, p.num_q_heads, p.n_tree, p.n_splits, p.max_seq_len = cabi.BF16, 8, T, splits, max(lens)
    need = C.c_size_t()
    keep = [dev.upload(to_bf16_bits(q.reshape(-1))), dev.upload(np.full(q.size, 0x5555, np.uint16)), dev.upload(np.array(given, np.int32)),
            dev.upload(np.array(counts, np.int32))]
    p.q, p.out, p.parents, p.n_nodes = keep
    cabi.check(dev.L.grl_tree_workspace_bytes(dev.h, C.byref(p), C.byref(need)))
    if need.value:
        keep.append(dev.upload(np.full(need.value, 0xFF, np.uint8)))
        p.workspace, p.workspace_bytes = keep[-1], need.value
    cabi.check(dev.L.grl_tree_attention(dev.h, C.byref(p)))
    with pytest.raises(cabi.GrlError) as e:
        dev.sync()
    assert e.value.code == cabi.ERR_KERNEL and "sequence 1" in str(e.value)
    got = from_bf16_bits(dev.download(keep[1], q.shape, np.uint16))
    if "page" not in fault:
        assert np.all(got[1] == 0)
    cache.rows = [x[:1] for x in cache.rows]
    check_attention(got[:1], cache, q[:1], parents[:1], None, "bf16", False)
    for k in keep:
        dev.free(k)
    cache.free()


@pytest.mark.parametrize("T,splits,lens,counts", [(4, 5, [1500, 65, 4], [4, 2, 0]), (4, 16, [4000, 65, 4], [4, 1, 0]), (1, 8, [1030, 1, 0], [1, 1, 0]),
                                                  (3, 3, [300, 3, 200], [3, 3, 2])])
def test_few_rows_joined_in_a_cluster(dev, T, splits, lens, counts):
    """Sequences without nodes, and shorter than their splits, among them."""
    c = tree_case(T, 8, 2, 128, 32, lens, counts, kw_splits=splits)
    got, cache, q, parents = run_tree(dev, c)
    check_attention(got, cache, q, parents, counts, "bf16", False)
    cache.free()


def test_pages_past_32_bits(dev):
    """A pool of more than 2^31 elements: the sequence's pages lie at its end."""
    from grilly_next import cabi
    P, Hkv, D, T = 64, 8, 128, 6
    pages = (1 << 31) // (P * Hkv * D) + 8
    small = Cache(dev, [200], Hkv, D, P, "bf16", seed=2, spare=0)
    big = [dev.malloc(pages * P * Hkv * D * 2) for _ in range(2)]
    page_bytes = P * Hkv * D * 2
    first = pages - small.num_pages
    for dst, src in zip(big, small.ptr):
        cabi.check(dev.L.grl_memcpy_d2d(dev.h, dst.value + first * page_bytes, src, small.num_pages * page_bytes))
    q = round_bf16(np.random.default_rng(0).standard_normal((1, T, 32, D)).astype(np.float32))
    keep = small.ptr, small.num_pages
    table = (small.table + first).astype(np.int32)
    cabi.check(dev.L.grl_memcpy_h2d(dev.h, small.table_ptr, table.ctypes.data_as(C.c_void_p), table.nbytes))
    dev.sync()
    small.ptr, small.num_pages = big, pages
    got = attend(dev, small, q, None, None, io="bf16")
    check_attention(got, small, q, None, None, "bf16", False)
    got = attend(dev, small, q, None, None, io="bf16", kernel=cabi.KERNEL_SIMT_F32)
    check_attention(got, small, q, None, None, "bf16", True)
    small.ptr, small.num_pages = keep
    for b in big:
        dev.free(b)
    small.free()


# ------------------------------------------------------------------------------------------------------ append and commit
def append_step(dev, cache, k, v, q, counts, parents, *, io="bf16", q_io=None, rotary=None, mode="half", wq=None, wk=None, update=False, pos_base=0,
                offsets=None, packed=False, gain=0.0):
    cabi = cache.cabi
    B, T, Hq, D = (k.shape[0], k.shape[1], 0, k.shape[3]) if q is None else q.shape
    p = cabi.AppendNormParams()
    p.kv = cache.layout()
    up = (lambda x: dev.upload(x)) if io == "f32" else (lambda x: dev.upload(to_bf16_bits(np.ascontiguousarray(x).reshape(-1))))
    keep, size = [], 4 if io == "f32" else 2
    if packed:
        rows = up(np.concatenate([q, k, v], 2))
        keep.append(rows)
        H, Hkv = q.shape[2], k.shape[2]
        p.q_in, p.k_new, p.v_new = rows, rows.value + H * D * size, rows.value + (H + Hkv) * D * size
        p.q_token_stride = p.k_token_stride = p.v_token_stride = (H + 2 * Hkv) * D
    else:
        keep += [up(k), up(v)]
        p.k_new, p.v_new = keep[:2]
        if q is not None:
            keep.append(up(q))
            p.q_in = keep[-1]
    q_io = q_io or io
    qs = 4 if q_io == "f32" else 2
    qn = B * T * Hq * D
    if q is not None:
        qo = dev.upload(np.full(qn * qs + 64, 0x55, np.uint8))
        keep.append(qo)
        p.q_out, p.num_q_heads = qo, Hq
    p.in_dtype = cabi.F32 if io == "f32" else cabi.BF16
    p.q_out_dtype = cabi.F32 if q_io == "f32" else cabi.BF16
    p.n_new, p.eps, p.update_lens, p.pos_base = T, 1e-5, int(update), pos_base
    p.rope.mode, p.rope.theta, p.rope.rotary_dim, p.rope.gain = {"none": 0, "interleaved": 1, "half": 2}[mode], 10000.0, rotary or D, gain
    for name, a in (("q_weight", wq), ("k_weight", wk), ("n_nodes", None if counts is None else np.array(counts, np.int32)),
                    ("parents", None if parents is None else np.array(parents, np.int32)),
                    ("pos_offsets", None if offsets is None else np.array(offsets, np.int32))):
        if a is not None:
            keep.append(dev.upload(a))
            setattr(p, name, keep[-1])
    cabi.check(dev.L.grl_kv_append_norm(dev.h, C.byref(p)))
    try:
        dev.sync()
        if q is None:
            return None
        raw = dev.download(qo, (qn * qs + 64,), np.uint8)
        assert np.all(raw[qn * qs:] == 0x55)
        out = raw[:qn * qs].view(np.float32 if q_io == "f32" else np.uint16).reshape(q.shape)
        return out.copy() if q_io == "f32" else from_bf16_bits(out)
    finally:
        for h in keep:
            dev.free(h)


def app(T, Hq, Hkv, D, page, before, counts=None, kind="tree", cache="bf16", io=None, **kw):
    return dict(T=T, Hq=Hq, Hkv=Hkv, D=D, page=page, before=before, counts=counts, kind=kind, cache=cache, io=io or cache, kw=kw)


APPENDS = {
    "one": app(1, 4, 2, 128, 64, [0, 63, 64]), "tree": app(13, 8, 2, 128, 64, [100, 51, 0]), "interleaved": app(13, 8, 2, 128, 64, [100, 51, 0], mode="interleaved"),
    "ragged": app(16, 8, 2, 128, 16, [100, 51, 0, 9], [16, 0, 7, 1]), "chain": app(16, 8, 2, 128, 16, [100, 51], kind="chain"),
    "prompt": app(300, 8, 2, 128, 64, [0, 51], kind="chain"), "prompt_f32": app(133, 6, 2, 64, 24, [0, 51], kind="chain", cache="f32"),
    "line_128": app(128, 4, 2, 64, 32, [100], kind="line"), "part": app(13, 8, 2, 128, 64, [100, 51], rotary=64),
    "part_odd": app(5, 3, 1, 64, 64, [100], rotary=20), "packed": app(9, 8, 2, 128, 64, [100, 51], packed=True),
    "packed_f32": app(9, 6, 2, 64, 16, [100, 51], packed=True, cache="f32", mode="interleaved"), "no_queries": app(9, 0, 2, 128, 64, [100, 51]),
    "f32_into_bf16": app(9, 8, 2, 128, 64, [100, 51], io="f32"), "f32_q_bf16": app(9, 8, 2, 128, 64, [100, 51], io="f32", q_io="bf16"),
    "bf16_q_f32": app(9, 8, 2, 128, 64, [100, 51], q_io="f32"), "bf16_into_f32": app(9, 8, 2, 128, 64, [100, 51], cache="f32", io="bf16"),
    "offsets": app(9, 8, 2, 128, 64, [100, 51], offsets=[1000, 0], pos_base=5), "no_weights": app(9, 8, 2, 128, 64, [100, 51], weights=False),
    "dim_80": app(9, 3, 1, 80, 8, [100, 51]), "dim_256": app(9, 3, 1, 256, 8, [100, 51]), "dim_32": app(9, 8, 4, 32, 8, [100, 51]),
    "gain": app(9, 8, 2, 128, 64, [100], gain=1.125), "update": app(13, 8, 2, 128, 64, [100, 51, 0], [13, 0, 5], update=True),
    "update_prompt": app(300, 8, 2, 128, 64, [0, 51], [300, 17], kind="chain", update=True), "batch": app(7, 4, 2, 64, 16, [10 * i for i in range(50)]),
}


@pytest.mark.parametrize("name", list(APPENDS))
def test_append_norm(dev, name):
    c = APPENDS[name]
    r = np.random.default_rng(11)
    kw = dict(c["kw"])
    weights = kw.pop("weights", True)
    B, T, D, Hq, Hkv = len(c["before"]), c["T"], c["D"], c["Hq"], c["Hkv"]
    counts = c["counts"] or [T] * B
    cache = Cache(dev, c["before"], Hkv, D, c["page"], c["cache"], room=T)
    old = cache.read()
    rnd = round_bf16 if c["io"] == "bf16" else (lambda x: x)
    k, v, q = (rnd(r.standard_normal((B, T, h, D)).astype(np.float32)) for h in (Hkv, Hkv, Hq))
    wq, wk = ((1 + 0.2 * r.standard_normal(D)).astype(np.float32) if weights else None for _ in range(2))
    parents = None if c["kind"] == "chain" else [draw_parents(r, T, c["kind"]) for _ in range(B)]
    got_q = append_step(dev, cache, k, v, q if Hq else None, c["counts"], parents, io=c["io"], wq=wq, wk=wk, **kw)
    new = cache.read()
    rotary, mode, gain = kw.get("rotary") or D, kw.get("mode", "half"), kw.get("gain") or 1.0
    freq, offsets = orc.frequencies(rotary), kw.get("offsets") or [0] * B

    def bound(x, w, want, t):
        n = np.abs(orc.norm(x, w, 1e-5))
        tol = 40 * U * 2 * n.max() * gain            # |n0| + |n1| is at most twice the largest element of the row
        return tol + (2.0 ** -8 * (np.abs(want) + tol) if t == "bf16" else 0)

    touched = np.zeros(old[0].shape[:1] + old[0].shape[2:3], bool)
    for b in range(B):
        n = counts[b]
        depth = (np.arange(n) if parents is None else orc.depths(parents[b], n)) if n else np.zeros(0)
        pos = kw.get("pos_base", 0) + offsets[b] + c["before"][b] + depth
        want_k = orc.norm_rope(k[b, :n], wk, pos, freq, mode, 1e-5, gain)
        for t in range(n):
            at = c["before"][b] + t
            touched[cache.table[b, at // cache.P], at % cache.P] = True
            kr, vr = cache.row_of(new, b, at)
            assert np.all(np.abs(kr - want_k[t]) <= bound(k[b, t], wk, want_k[t], c["cache"])), (b, t)
            want_v = round_bf16(v[b, t]) if c["cache"] == "bf16" else v[b, t]
            assert np.array_equal(vr, want_v)
        if Hq:
            want_q = orc.norm_rope(q[b, :n], wq, pos, freq, mode, 1e-5, gain)
            if n:
                assert np.all(np.abs(got_q[b, :n] - want_q) <= bound(q[b, :n], wq, want_q, kw.get("q_io") or c["io"]))
            assert np.all(got_q[b, n:] == 0)
    for o, m in zip(old, new):               # all other rows of the pools are as they were
        assert np.array_equal(o.transpose(0, 2, 1, 3)[~touched], m.transpose(0, 2, 1, 3)[~touched], equal_nan=True)
    lens = dev.download(cache.lens_ptr, (B,), np.int32)
    assert list(lens) == [x + (n if kw.get("update") else 0) for x, n in zip(c["before"], counts)]
    cache.free()


@pytest.mark.parametrize("fault", ["parent", "count", "room", "page"])
@pytest.mark.parametrize("update", [False, True])
def test_append_leaves_a_sequence_whose_numbers_do_not_fit(dev, fault, update):
    from grilly_next import cabi
    T, r = 5, np.random.default_rng(0)
    cache = Cache(dev, [20, 30], 2, 64, 16, "f32", room=T)
    old = cache.read()
    k, v, q = (r.standard_normal((2, T, h, 64)).astype(np.float32) for h in (2, 2, 4))
    parents, counts = [[-1, 0, 1, 0, 2]] * 2, [T, T]
    if fault == "parent": parents = [parents[0], [-1, 0, 2, 0, 2]]
    if fault == "count": counts = [T, T + 1]
    if fault == "room": cache.set_lens([20, cache.max_pages * 16 - T + 1])
    if fault == "page":
        bad = cache.table.copy()
        bad[1, 30 // 16] = cache.num_pages
        cabi.check(dev.L.grl_memcpy_h2d(dev.h, cache.table_ptr, bad.ctypes.data_as(C.c_void_p), bad.nbytes))
    before = list(cache.lens)
    with pytest.raises(cabi.GrlError) as e:
        append_step(dev, cache, k, v, q, counts, parents, io="f32", update=update)
    assert e.value.code == cabi.ERR_KERNEL and "sequence 1" in str(e.value)
    new = cache.read()
    for o, m in zip(old, new):
        for b, t in ((1, t) for t in range(cache.max_pages * 16)):
            page, slot = cache.table[b, t // 16], t % 16
            assert np.array_equal(o[page, :, slot], m[page, :, slot], equal_nan=True)
    assert not np.array_equal(*(cache.row_of(x, 0, 20)[0] for x in (old, new)))          # the other sequence was served
    assert list(dev.download(cache.lens_ptr, (2,), np.int32)) == [before[0] + (T if update else 0), before[1]]
    cache.free()


def commit(dev, cache, paths, counts, T, *, separate=False, meta=None):
    cabi = cache.cabi
    p = cabi.CommitParams()
    p.kv = cache.layout()
    most = max(1, max(len(x) for x in paths))
    keep = [dev.upload(np.array([x + [0] * (most - len(x)) for x in paths], np.int32)), dev.upload(np.array([len(x) for x in paths], np.int32))]
    p.path, p.n_path, p.max_path, p.n_tree = keep[0], keep[1], most, T
    if counts is not None:
        keep.append(dev.upload(np.array(counts, np.int32)))
        p.n_nodes = keep[-1]
    if separate:
        lens = dev.upload(np.full(cache.B, -7, np.int32))
        keep.append(lens)
        p.lens_out = lens
    if meta is not None:
        p.meta = C.pointer(meta)
    cabi.check(dev.L.grl_kv_commit(dev.h, C.byref(p)))
    try:
        dev.sync()
        return list(dev.download(lens if separate else cache.lens_ptr, (cache.B,), np.int32))
    finally:
        for h in keep:
            dev.free(h)


@pytest.mark.parametrize("D,page,cache_type", [(128, 64, "bf16"), (64, 16, "f32"), (80, 7, "bf16"), (6, 4, "bf16"), (256, 16, "f32")])
@pytest.mark.parametrize("separate", [False, True])
def test_commit(dev, D, page, cache_type, separate):
    T, before = 40, [100, 0, 55, 7, 30]
    counts = [40, 40, 17, 0, 1]
    paths = [[0, 3, 9, 39], list(range(40)), [16], [], []]
    cache = Cache(dev, [x + n for x, n in zip(before, counts)], 3, D, page, cache_type)
    old = cache.read()
    lens = commit(dev, cache, paths, counts, T, separate=separate)
    new = cache.read()
    assert lens == [x + len(path) for x, path in zip(before, paths)]
    if separate:
        assert list(dev.download(cache.lens_ptr, (5,), np.int32)) == [x + n for x, n in zip(before, counts)]
    for b, path in enumerate(paths):
        for t in range(before[b]):
            assert all(np.array_equal(*x) for x in zip(cache.row_of(old, b, t), cache.row_of(new, b, t)))
        for i, t in enumerate(path):
            assert all(np.array_equal(*x) for x in zip(cache.row_of(old, b, before[b] + t), cache.row_of(new, b, before[b] + i)))
    cache.free()


def test_commit_moves_the_metadata(dev):
    from grilly_next import cabi
    cache = Cache(dev, [60, 30], 2, 64, 16, "bf16", room=20)
    cap = cache.max_pages * 16
    r = np.random.default_rng(0)
    cum, rel = (r.random((2, cap)).astype(np.float32) for _ in range(2))
    tomb = (r.random((2, cap)) < 0.5).astype(np.uint8)
    m = cabi.KVMeta()
    ptrs = [dev.upload(x) for x in (cum, tomb, rel)]
    m.cum_score, m.tombstone, m.relevance, m.capacity = ptrs[0], ptrs[1], ptrs[2], cap
    assert commit(dev, cache, [[1, 4, 5], [0]], [10, 10], 10, meta=m) == [53, 21]
    for x, p in zip((cum, tomb, rel), ptrs):
        want = x.copy()
        want[0, 50:60], want[1, 20:30] = 0, 0
        want[0, 50:53], want[1, 20] = x[0, [51, 54, 55]], x[1, 20]
        assert np.array_equal(dev.download(p, x.shape, x.dtype), want)
        dev.free(p)
    cache.free()


@pytest.mark.parametrize("path", [[0, 0], [2, 1], [3, 10], [-1], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 9]])
def test_commit_refuses_paths_that_are_none(dev, path):
    from grilly_next import cabi
    cache = Cache(dev, [60, 30], 2, 64, 16, "bf16")
    old = cache.read()
    with pytest.raises(cabi.GrlError) as e:
        commit(dev, cache, [[1], path], [10, 10], 10)
    assert e.value.code == cabi.ERR_KERNEL and "sequence 1" in str(e.value) and "path" in str(e.value)
    new = cache.read()
    assert list(dev.download(cache.lens_ptr, (2,), np.int32)) == [51, 30]
    for t in range(30):
        assert all(np.array_equal(*x) for x in zip(cache.row_of(old, 1, t), cache.row_of(new, 1, t)))
    cache.free()


# ---------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("cache_type,page", [("bf16", 64), ("f32", 24)])
def test_steps_in_a_row(dev, cache_type, page):
    """Append, attend, commit, three times over: the cache in the end is that of the accepted tokens one after another, and every step's
    attention is that of the rows as the cache holds them."""
    r = np.random.default_rng(4)
    B, T, Hq, Hkv, D = 3, 11, 8, 2, 128
    cache = Cache(dev, [70, 0, 33], Hkv, D, page, cache_type, room=3 * T)
    lens, rnd = [70, 0, 33], round_bf16 if cache_type == "bf16" else (lambda x: x)
    wq, wk = ((1 + 0.2 * r.standard_normal(D)).astype(np.float32) for _ in range(2))
    for step in range(3):
        counts = [T, 5, [T, 0, 1][step]]
        parents = [draw_parents(r, T, "tree") for _ in range(B)]
        k, v, q = (rnd(r.standard_normal((B, T, h, D)).astype(np.float32)) for h in (Hkv, Hkv, Hq))
        got_q = append_step(dev, cache, k, v, q, counts, parents, io=cache_type, wq=wq, wk=wk, update=True)
        cache.lens = np.array([a + n for a, n in zip(lens, counts)], np.int32)
        pools = cache.read()
        for b in range(B):
            rows = [cache.row_of(pools, b, t) for t in range(lens[b] + counts[b])]
            for i in range(2):
                cache.rows[i][b] = np.array([x[i] for x in rows]).reshape(-1, Hkv, D)
            want = orc.norm_rope(k[b, :counts[b]], wk, lens[b] + orc.depths(parents[b], counts[b]), orc.frequencies(D), "half", 1e-5)
            tol = 80 * U * 8 + (2.0 ** -8 * np.abs(want) if cache_type == "bf16" else 0)
            assert np.all(np.abs(cache.rows[0][b][lens[b]:] - want) <= tol)
        out = attend(dev, cache, got_q, parents, counts, io=cache_type)
        check_attention(out, cache, got_q, parents, counts, cache_type, cache_type == "f32")
        paths = []
        for b in range(B):
            t, path = (int(r.integers(counts[b])) if counts[b] else -1), []
            while t >= 0:
                path.append(t)
                t = parents[b][t]
            paths.append(path[::-1])
        kept = commit(dev, cache, paths, counts, T)
        pools = cache.read()
        for b in range(B):
            order = list(range(lens[b])) + [lens[b] + t for t in paths[b]]
            assert kept[b] == len(order)
            for t, old in enumerate(order):
                assert all(np.array_equal(x, cache.rows[i][b][old]) for i, x in enumerate(cache.row_of(pools, b, t)))
        lens = kept
    cache.free()


def test_captured_step_replays_on_new_lengths(dev):
    """A graph of one step's three calls, replayed: every replay goes by the lengths, trees and rows that the buffers then hold."""
    from grilly_next import cabi
    r = np.random.default_rng(8)
    B, T, Hq, Hkv, D = 2, 6, 8, 2, 128
    cache = Cache(dev, [100, 40], Hkv, D, 64, "bf16", room=64)
    keep = {}

    def up(name, a):
        if name in keep:
            a = np.ascontiguousarray(a)
            cabi.check(dev.L.grl_memcpy_h2d(dev.h, keep[name], a.ctypes.data_as(C.c_void_p), a.nbytes))
        else:
            keep[name] = dev.upload(a)
        return keep[name]

    def inputs(seed):
        s = np.random.default_rng(seed)
        x = {n: round_bf16(s.standard_normal((B, T, h, D)).astype(np.float32)) for n, h in (("k", Hkv), ("v", Hkv), ("q", Hq))}
        parents = [draw_parents(s, T, "tree") for _ in range(B)]
        for n, a in x.items():
            up(n, to_bf16_bits(a.reshape(-1)))
        up("parents", np.array(parents, np.int32))
        up("path", np.array([[0, 0]] * B, np.int32))
        up("n_path", np.array([1] * B, np.int32))
        dev.sync()
        return x, parents

    inputs(0)
    q_out, out = dev.malloc(B * T * Hq * D * 2), dev.malloc(B * T * Hq * D * 2)
    a, t, m = cabi.AppendNormParams(), cabi.TreeParams(), cabi.CommitParams()
    a.kv = t.kv = m.kv = cache.layout()
    a.k_new, a.v_new, a.q_in, a.q_out, a.in_dtype, a.q_out_dtype = keep["k"], keep["v"], keep["q"], q_out, cabi.BF16, cabi.BF16
    a.n_new, a.num_q_heads, a.parents, a.update_lens, a.rope.mode, a.rope.theta = T, Hq, keep["parents"], 1, cabi.ROPE_HALF, 10000.0
    t.q, t.out, t.io_dtype, t.num_q_heads, t.n_tree, t.parents = q_out, out, cabi.BF16, Hq, T, keep["parents"]
    need = C.c_size_t()
    cabi.check(dev.L.grl_tree_workspace_bytes(dev.h, C.byref(t), C.byref(need)))
    if need.value:
        t.workspace, t.workspace_bytes = dev.malloc(need.value), need.value
    m.path, m.n_path, m.max_path, m.n_tree = keep["path"], keep["n_path"], 2, T

    def step():
        cabi.check(dev.L.grl_kv_append_norm(dev.h, C.byref(a)))
        cabi.check(dev.L.grl_tree_attention(dev.h, C.byref(t)))
        cabi.check(dev.L.grl_kv_commit(dev.h, C.byref(m)))

    step()
    dev.sync()
    cache.set_lens([100, 40])
    g = C.c_void_p()
    cabi.check(dev.L.grl_graph_begin(dev.h))
    step()
    cabi.check(dev.L.grl_graph_end(dev.h, C.byref(g)))
    for replay in range(3):
        x, parents = inputs(20 + replay)
        cabi.check(dev.L.grl_graph_launch(dev.h, g))
        dev.sync()
        lens = [100 + replay, 40 + replay]              # ahead of this step; one node is kept each time
        assert list(dev.download(cache.lens_ptr, (B,), np.int32)) == [n + 1 for n in lens]
        pools = cache.read()
        for b in range(B):
            for i in range(2):
                cache.rows[i][b] = np.array([cache.row_of(pools, b, u)[i] for u in range(lens[b] + T)])
        got_q = from_bf16_bits(dev.download(q_out, (B, T, Hq, D), np.uint16))
        got = from_bf16_bits(dev.download(out, (B, T, Hq, D), np.uint16))
        check_attention(got, cache, got_q, parents, None, "bf16", False)
        cache.lens = np.array([n + 1 for n in lens], np.int32)
    cabi.check(dev.L.grl_graph_destroy(g))
    cache.free()
    for h in list(keep.values()) + [q_out, out]:
        dev.free(h)


def test_two_handles_at_once(dev):
    """Two handles (two streams) with a workspace each run the same call side by side, many times: the results are those of one alone."""
    from grilly_next import cabi
    other = cabi.Device(0)
    c = TREES["splits_3"]
    want, cache, q, parents = run_tree(dev, c)
    calls = []
    for d in (dev, other):
        p = cabi.TreeParams()
        p.kv = cache.layout()
        bufs = [d.upload(to_bf16_bits(q.reshape(-1))), d.malloc(q.size * 2), d.upload(np.array(parents, np.int32))]
        p.q, p.out, p.parents = bufs
        p.io_dtype, p.num_q_heads, p.n_tree, p.max_seq_len, p.n_splits = cabi.BF16, c["Hq"], c["T"], int(cache.lens.max()), 3
        need = C.c_size_t()
        cabi.check(d.L.grl_tree_workspace_bytes(d.h, C.byref(p), C.byref(need)))
        p.workspace, p.workspace_bytes = d.malloc(need.value), need.value
        calls.append((d, p, bufs[1]))
    for _ in range(50):
        for d, p, _ in calls:
            cabi.check(d.L.grl_tree_attention(d.h, C.byref(p)))
    for d, p, out in calls:
        d.sync()
        assert np.array_equal(from_bf16_bits(d.download(out, q.shape, np.uint16)), want)
    cache.free()
    other.close()
