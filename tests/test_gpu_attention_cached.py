"""Attention over the 8-bit cache through the C ABI, against float64 of the held
values, with the bound of cached.attention: lengths from one to long ones, every rule,
rows that see nothing, values of every size, what lies in places that are not seen, and the
operators in the order a program runs them."""
import numpy as np
import pytest

import cached
from conftest import record_margin
from test_gpu_patch_block import normals

pytestmark = pytest.mark.gpu

vh = pytest.importorskip("vestra_hip")


class Case:
    """A filled cache and queries of it; `held` the values, all as [S, heads, ..]."""

    def __init__(self, rt, rng, fmt, S, H, KV, cap, n, starts=None, counts=None, layout=0, ks=1.5,
                 vs=1.0, qs=1.5):
        self.rt, self.fmt, self.n, self.layout = rt, fmt, n, layout
        self.q = np.ascontiguousarray(normals(rng, S, H, n, 64) * np.float32(qs), np.float32)
        self.k = np.ascontiguousarray(normals(rng, S, KV, cap, 64) * np.asarray(ks, np.float32))
        self.v = np.ascontiguousarray(normals(rng, S, KV, cap, 64) * np.asarray(vs, np.float32))
        self.starts = None if starts is None else np.asarray(starts, np.int32)
        self.counts = None if counts is None else np.asarray(counts, np.int32)
        self.S, self.H, self.KV, self.cap = S, H, KV, cap

    def fill(self):
        """The cache through the library's own write."""
        rt = self.rt
        self.cache = rt.kv_cache(self.fmt, self.S, self.KV, self.cap)
        rt.kv_cache_write_f32(self.cache, rt.upload_f32(self.k), rt.upload_f32(self.v), self.cap,
                              layout=vh.VK_QK_VIEWS_OUTER)
        (kc, kd), (vc, self.v_scale) = (cached.quantise(x, self.fmt) for x in (self.k, self.v))
        self.kh, self.vheld = cached.values(kc, kd, self.fmt), cached.values(vc, self.v_scale, self.fmt)
        return self

    def lay(self, x):
        return cached.heads_outer(x) if self.layout == vh.VK_QK_HEADS_OUTER else x

    def run(self, rules=None, max_length=0, fill=7.0):
        rt = self.rt
        r = dict(rules or {})
        self.dev = {k: rt.upload_i32(r[k]) for k in ("prefix", "q_docs", "k_docs") if r.get(k) is not None}
        if r.get("slopes") is not None:
            self.dev["slopes"] = rt.upload_f32(r["slopes"])
        args = vh.AttentionRules(**{**r, **self.dev}) if r else None
        self.qd = rt.upload_f32(self.lay(self.q))
        self.out = rt.upload_f32(np.full(self.q.size, fill))
        self.st, self.ct = (None if x is None else rt.upload_i32(x) for x in (self.starts, self.counts))
        self.call = lambda: rt.attention_cached_f32(self.cache, self.qd, self.H, self.n, self.st,
                                                    self.ct, max_length, args, self.out, self.layout)
        self.call()
        return self.got()

    def got(self):
        o = self.out.numpy()
        return cached.heads_outer(o.reshape(self.H, self.S, self.n, 64)) \
            if self.layout == vh.VK_QK_HEADS_OUTER else o.reshape(self.S, self.H, self.n, 64)

    def check(self, rules=None, max_length=0, label="", pick=None):
        got = self.run(rules, max_length)
        want, tol = cached.attention(self.q, self.kh, self.vheld, self.v_scale, self.n, self.starts,
                                     self.counts, rules or {}, max_length, pick)
        for s in range(self.S):
            _, count = cached.spans(self.n, self.cap, self.starts, self.counts, s)
            assert np.all(got[s, :, count:] == 7.0), "a row past the count was written"
        written = ~np.isnan(want)
        off = np.abs(got.astype(np.float64) - want)
        record_margin("attention cached", got[written], want[written], tol=tol[written], label=label)
        assert np.all((off <= tol)[written]), \
            f"{label}: {np.sum(~(off <= tol)[written])} off, worst {np.nanmax((off / tol)[written])}"
        return got


SIZES = [  # S, H, KV, cap, n, starts, counts
    (1, 1, 1, 1, 1, None, None), (1, 12, 12, 38, 1, [37], None), (2, 4, 2, 64, 1, [63, 0], None),
    (1, 3, 1, 65, 3, [62], None), (3, 2, 1, 70, 5, [0, 30, 65], [5, 0, 3]),
    (1, 2, 2, 129, 33, [96], None), (2, 3, 3, 200, 64, [100, 7], [64, 63]),
    (1, 2, 1, 300, 257, [20], None), (1, 16, 4, 1000, 2, [998], None),
    (1, 12, 12, 866, 1, [865], None), (2, 16, 2, 700, 9, [600, 64], [9, 8]),
    (1, 1, 1, 5000, 1, [4999], None), (1, 2, 1, 3000, 100, [2900], None),
    (2, 12, 12, 600, 301, [250, 299], [301, 280]),
]


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("S,H,KV,cap,n,starts,counts", SIZES)
def test_sizes(rt, rng, fmt, S, H, KV, cap, n, starts, counts):
    c = Case(rt, rng, fmt, S, H, KV, cap, n, starts, counts, layout=fmt).fill()
    c.check(label=f"{S} {H} {KV} {cap} {n}")


def rules_of(kind, rng, S, H, cap, n, starts):
    pos = np.asarray(starts)[:, None] + np.arange(n)
    r = {}
    if "causal" in kind or "prefix" in kind:
        r["causal"] = True
    if "prefix" in kind:
        r["prefix"] = rng.integers(0, cap, S).astype(np.int32)
    if "cap" in kind.split("+"):
        r["cap"] = 5.0
    if "bias" in kind:
        r["slopes"] = (2.0 ** (-8.0 * np.arange(1, H + 1) / H)).astype(np.float32)
    if "scale" in kind:
        r["scale"] = 0.3
    if "docs" in kind:
        unit = 37
        r["q_docs"], r["k_docs"] = (pos // unit).astype(np.int32), \
            np.tile(np.arange(cap) // unit, (S, 1)).astype(np.int32)
    if "mixed" in kind:  # no order among the documents, and some that nothing matches
        r["q_docs"] = rng.integers(0, 4, (S, n)).astype(np.int32)
        r["k_docs"] = rng.integers(1, 5, (S, cap)).astype(np.int32)
    if "ordered" in kind:
        r["docs_ordered"] = True
    return r


KINDS = ["causal", "prefix", "cap", "bias", "scale", "docs", "docs+ordered", "mixed", "mixed+ordered",
         "cap+bias+causal", "docs+causal", "docs+ordered+cap+bias+prefix", "mixed+bias"]
SHAPES = [(2, 4, 2, 200, 1, [199, 70]), (2, 2, 1, 220, 7, [100, 213]), (1, 3, 3, 333, 150, [183]),
          (2, 2, 2, 420, 300, [0, 120]), (1, 2, 1, 2100, 40, [2060])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("S,H,KV,cap,n,starts", SHAPES)
def test_rules(rt, rng, kind, S, H, KV, cap, n, starts):
    c = Case(rt, rng, len(kind) % 2, S, H, KV, cap, n, starts, layout=n % 2).fill()
    c.check(rules_of(kind, rng, S, H, cap, n, starts), label=kind)


def test_rows_that_see_nothing(rt, rng):
    S, H, cap, n = 2, 2, 100, 70
    c = Case(rt, rng, 0, S, H, 1, cap, n, [0, 30]).fill()
    r = {"q_docs": np.full((S, n), 5, np.int32), "k_docs": np.full((S, cap), 6, np.int32)}
    r["q_docs"][0, 3] = r["q_docs"][1, 69] = 6
    got = c.check(r)
    assert np.all(got[0, :, :3] == 0) and np.any(got[0, :, 3] != 0)
    # no key at all: everything before slot 0
    c = Case(rt, rng, 1, 1, 2, 2, 50, 4, [-4]).fill()
    assert np.all(c.check() == 0)
    c = Case(rt, rng, 1, 1, 2, 2, 50, 4, [-2]).fill()
    c.check()
    c = Case(rt, rng, 1, 1, 2, 2, 50, 4, [-2]).fill()
    c.check({"causal": True})


SIZE_SHAPES = [(1, 2, 1, 300, 1, [299]), (1, 2, 2, 330, 70, [260])]


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("qs,ks,vs", [(1, 1, 1e-5), (1, 1, 1e20), (1e-4, 1e4, 1), (1e4, 1e-4, 1),
                                      (1e-20, 1, 1e-26), (1e15, 1e-15, 1), (30, 10, 1),
                                      (1e-30, 1e30, 1e30), (1, 1e-6, 1e-3)])
@pytest.mark.parametrize("S,H,KV,cap,n,starts", SIZE_SHAPES)
def test_value_ranges(rt, rng, fmt, qs, ks, vs, S, H, KV, cap, n, starts):
    c = Case(rt, rng, fmt, S, H, KV, cap, n, starts, ks=ks, vs=vs, qs=qs).fill()
    c.check(label=f"{qs} {ks} {vs}")


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("S,H,KV,cap,n,starts", SIZE_SHAPES)
@pytest.mark.parametrize("least,most", [(-25, 25), (-3, 3)])
def test_rows_of_different_sizes(rt, rng, fmt, S, H, KV, cap, n, starts, least, most):
    """Every key its own size, some of them zeros, every query too."""
    size = 10.0 ** rng.uniform(least, most, (S, KV, cap, 1))
    size[:, :, 5:9] = 0
    size[:, :, 64:128] = 0  # a block of zeros
    c = Case(rt, rng, fmt, S, H, KV, cap, n, starts, ks=1, vs=size).fill()
    c.check(label="values")
    c = Case(rt, rng, fmt, S, H, KV, cap, n, starts, ks=np.minimum(size, 1e2), vs=1).fill()
    c.q *= (10.0 ** rng.uniform(-6, 0, (S, H, n, 1))).astype(np.float32)
    c.check(label="keys and queries")


@pytest.mark.parametrize("S,H,KV,cap,n,starts", SIZE_SHAPES)
def test_what_is_not_seen_has_no_effect(rt, rng, S, H, KV, cap, n, starts):
    """Infinities, NaN and huge values in keys of other documents, of later positions and
    past the length change nothing; seen, they give NaN."""
    c = Case(rt, rng, 0, S, H, KV, cap, n, [starts[0] - 40]).fill()
    docs = {"q_docs": np.zeros((S, n), np.int32), "k_docs": np.zeros((S, cap), np.int32)}
    docs["k_docs"][:, 3::17] = 1
    want = c.check(docs)
    bad = c.k.copy(), c.v.copy()
    for x in bad:
        x[:, :, 3::51, 5] = np.nan
        x[:, :, 20::51] = 3e38
        x[:, :, 37::51, 0] = -np.inf
        x[:, :, starts[0] - 40 + n:] = np.nan
    c.k, c.v = bad
    c.fill()
    got = c.run(docs)
    assert np.array_equal(got, want)
    got = c.run({**docs, "k_docs": np.zeros((S, cap), np.int32)})
    assert np.isnan(got).all()
    # a NaN in V's row or K's row alone, late in the sequence, with a causal mask
    for which in "kv":
        c = Case(rt, rng, 1, S, H, KV, cap, n, starts)
        getattr(c, which)[:, :, starts[0] + n // 2] = np.inf
        c.fill()
        got = c.run({"causal": True})
        assert np.isfinite(got[:, :, :n // 2]).all() and np.isnan(got[:, :, n // 2:]).all()


def test_queries_that_are_not_numbers(rt, rng):
    for cap, n in ((300, 1), (300, 40)):
        c = Case(rt, rng, 0, 1, 2, 1, cap, n, [cap - n]).fill()
        clean = c.run()
        c.q[0, 0, 0, 3] = np.nan
        c.q[0, 1, n - 1, 9] = np.inf
        got = c.run()
        assert np.isnan(got[0, 0, 0]).all() and np.isnan(got[0, 1, n - 1]).all()
        rest = np.ones(got.shape[:3], bool)
        rest[0, 0, 0] = rest[0, 1, n - 1] = False
        assert np.array_equal(got[rest], clean[rest])


@pytest.mark.parametrize("n", [1, 5, 40, 200])
def test_a_row_depends_on_itself_alone(rt, rng, n):
    """The bits of a query's output do not change with the other queries."""
    cap = 700
    c = Case(rt, rng, 0, 1, 2, 2, cap, n, [cap - n]).fill()
    a = c.run()
    keep = n // 2
    c.q[:, :, np.arange(n) != keep] *= np.float32(1e6)
    c.q[:, :, :keep:2] = 0
    assert np.array_equal(a[:, :, keep], c.run()[:, :, keep])


def test_max_length(rt, rng):
    c = Case(rt, rng, 0, 2, 2, 2, 900, 3, [400, 100]).fill()
    a = c.check(max_length=403)
    b = c.check()
    assert np.allclose(a, b, rtol=1e-5, atol=1e-6)
    c.check(max_length=200)


def test_replays_follow_the_lengths(rt, rng):
    """Two captured calls that share the runtime's work buffer, replayed with eager work
    between, at other starts and queries."""
    import vestra_hip
    rt2 = vestra_hip.Runtime(0)
    a = Case(rt2, rng, 0, 1, 2, 1, 4000, 2, [3998]).fill()
    b = Case(rt2, rng, 1, 2, 2, 2, 1500, 60, [1440, 900]).fill()
    a.check()
    b.check({"causal": True})
    rt2.synchronize()
    ga, gb = cached.captured(rt2, a.call), cached.captured(rt2, b.call)
    for step in range(4):
        for c, g, lo in ((a, ga, 3000), (b, gb, 300)):
            c.starts = rng.integers(0, lo, c.S).astype(np.int32)
            cached.set_i32(rt2, c.st, c.starts)
            c.q = normals(rng, *c.q.shape)
            c.qd.write(c.lay(c.q))
            g.launch()
        both = [c.got() for c in (a, b)]
        for c, rules, got in ((a, {}, both[0]), (b, {"causal": True}, both[1])):
            want, tol = cached.attention(c.q, c.kh, c.vheld, c.v_scale, c.n, c.starts, c.counts, rules)
            assert np.all(np.abs(got - want) <= tol)
            assert np.array_equal(c.run(rules), got)  # eager: the same bits
            c.call()
        # run() made new tensors: capture again
        rt2.synchronize()
        ga, gb = cached.captured(rt2, a.call), cached.captured(rt2, b.call)


def test_a_video_step_by_step(rt, rng):
    """Frames one after another: QKV projection, rotary axes with Q/K-norm, the cache's write
    and the attention, the output projection; the cache then holds what a whole clip's
    write holds, and the last frame's rows are those of the formula."""
    D, H, frames, gh, gw = 128, 2, 4, 3, 5
    n = 2 + gh * gw
    qkv = rt.prepare_linear_f32(D, 3 * D, normals(rng, D, 3 * D, scale=0.1), normals(rng, 3 * D, scale=0.1))
    proj = rt.prepare_linear_f32(D, D, normals(rng, D, D, scale=0.1), normals(rng, D, scale=0.1))
    g = [rt.upload_f32(normals(rng, 64, scale=0.1, shift=s)) for s in (1, 0, 1, 0)]
    axes = vh.RopeAxes((8, 12, 12))
    cap = frames * n
    step, clip = rt.kv_cache(0, 1, H, cap), rt.kv_cache(0, 1, H, cap)
    x = normals(rng, cap, D)
    grid = [(0, 0)] * 2 + [(y + 1, z + 1) for y in range(gh) for z in range(gw)]
    pos = np.array([(t, y, z) for t in range(frames) for y, z in grid], np.int32)

    def rows(cache, x, pos, start):
        m = len(x)
        q, k, v, qr, kr, o = (rt.alloc_f32(m * D) for _ in range(6))
        qkv.run_qkv_hnd(rt.upload_f32(x), m, H, q, k, v)
        rt.qk_norm_rope_axes_f32(q, k, *g, rt.upload_i32(pos), H, H, m, axes, 1e-5, qr, kr)
        st = rt.upload_i32(np.array([start], np.int32))
        rt.kv_cache_write_f32(cache, kr, v, m, st)
        docs = rt.upload_i32((np.arange(cap) // n).astype(np.int32))
        rules = vh.AttentionRules(q_docs=docs.view(start, m), k_docs=docs, docs_ordered=True)
        rt.attention_cached_f32(cache, qr, H, m, st, None, start + m, rules, o)
        out = rt.upload_f32(np.zeros((m, D)))
        proj.run_hnd_residual(o, m, H, out)
        return out.numpy().reshape(m, D), o.numpy().reshape(H, m, 64), qr.numpy().reshape(1, H, m, 64)

    outs = [rows(step, x[f * n:(f + 1) * n], pos[f * n:(f + 1) * n], f * n) for f in range(frames)]
    whole = rows(clip, x, pos, 0)
    back = [rt.alloc_f32(H * cap * 64) for _ in range(4)]
    rt.kv_cache_read_f32(step, cap, None, None, *back[:2])
    rt.kv_cache_read_f32(clip, cap, None, None, *back[2:])
    held = [t.numpy().reshape(1, H, cap, 64).astype(np.float64) for t in back]
    # the projections of one frame and of the clip differ by their tiles' rounding: a code
    # (int8: 1/127 of the row's largest) at most
    for a, b in ((held[0], held[2]), (held[1], held[3])):
        assert np.all(np.abs(a - b) <= 1.02 / 127 * np.abs(a).max(-1, keepdims=True))
    f = frames - 1
    want, tol = cached.attention(outs[f][2], held[0], held[1],
                                 np.abs(held[1]).max(-1).astype(np.float32) / 127, n,
                                 [f * n], None, {})
    assert np.all(np.abs(outs[f][1] - want[0]) <= tol[0])
    for f in range(frames):
        assert np.allclose(outs[f][0], whole[0][f * n:(f + 1) * n], rtol=0.02, atol=0.02)


def test_refusals(rt):
    S, H, cap, n = 2, 4, 8, 3
    c = rt.kv_cache(0, S, 2, cap)
    q, o = rt.upload_f32(np.ones(S * H * n * 64)), rt.alloc_f32(S * H * n * 64)
    z = rt.upload_i32(np.zeros(S, np.int32))
    slopes, docs = rt.upload_f32(np.ones(H)), rt.upload_i32(np.zeros(S * cap, np.int32))
    R = vh.AttentionRules

    def call(cache=c, q=q, heads=H, n=n, st=z, ct=None, rules=None, out=o, layout=0):
        rt.attention_cached_f32(cache, q, heads, n, st, ct, 0, rules, out, layout)

    rt.kv_cache_write_f32(c, rt.upload_f32(np.ones(S * 2 * cap * 64)),
                          rt.upload_f32(np.ones(S * 2 * cap * 64)), cap)
    call(rules=R(slopes=slopes, causal=True, prefix=z, q_docs=docs.view(0, S * n), k_docs=docs))
    assert np.allclose(o.numpy(), 1, rtol=1e-6)
    bad = [dict(heads=3), dict(heads=0), dict(n=4), dict(layout=7), dict(st=slopes), dict(out=q),
           dict(ct=docs), dict(rules=R(cap=-1.0)), dict(rules=R(cap=float("nan"))),
           dict(rules=R(scale=float("inf"))), dict(rules=R(slopes=z)), dict(rules=R(prefix=z)),
           dict(rules=R(causal=True, prefix=docs)), dict(rules=R(q_docs=docs.view(0, S * n))),
           dict(rules=R(k_docs=docs)), dict(rules=R(docs_ordered=True)),
           dict(rules=R(q_docs=docs, k_docs=docs)),
           dict(rules=R(slopes=o.view(0, H))), dict(out=rt.alloc_f32(len(o) + 4).view(1, len(o))),
           dict(q=rt.upload_f16(np.zeros(len(q))))]
    for args in bad:
        with pytest.raises(vh.VestraError) as e:
            call(**args)
        assert e.value.code == vh.VK_ERR_INVALID, args
    call(n=0, q=rt.alloc_f32(0), out=rt.alloc_f32(0))
    rt.synchronize()


def test_capture_refuses_to_grow_the_work_buffer(rng):
    """A call that needs more of the work buffer than there is cannot be captured; after an
    eager call of its kind it can."""
    import vestra_hip
    own = vestra_hip.Runtime(0)
    c = Case(own, rng, 0, 1, 2, 1, 9000, 1, [8999]).fill()
    own.synchronize()
    q, out = own.upload_f32(c.q), own.alloc_f32(c.q.size)
    st = own.upload_i32(c.starts)
    args = (c.cache, q, c.H, c.n, st, None, 0, None, out)

    def refused():
        with pytest.raises(vh.VestraError):
            own.attention_cached_f32(*args)

    cached.captured(own, refused)
    own.attention_cached_f32(*args)
    want = out.numpy()
    graph = cached.captured(own, lambda: own.attention_cached_f32(*args))
    out.write(np.zeros(c.q.size))
    graph.launch()
    assert np.array_equal(out.numpy(), want)
