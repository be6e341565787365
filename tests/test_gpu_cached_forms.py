"""The forms of the attention over the 8-bit cache where they begin and end: one query, few,
tiles of 128, each with its keys in one workgroup and split; lists of blocks of more than one run,
tiles across documents' borders, scores on both sides of the cap's series, caches past 4 GiB, graphs
and runtimes side by side."""
import numpy as np
import pytest

import cached
from test_gpu_attention_cached import Case
from test_gpu_patch_block import normals

pytestmark = pytest.mark.gpu

vh = pytest.importorskip("vestra_hip")

# (pairs, queries of each, keys): (form, split)
FORM_OF = {(2, 1, 700): (0, False), (2, 1, 3000): (0, True), (4, 9, 600): (1, False),
           (2, 20, 3000): (1, True), (300, 40, 300): (2, False), (3, 260, 1500): (2, True)}


def docs_of(S, n, cap, starts, borders):
    """Documents that begin at the slots `borders`, of keys and of the queries among them."""
    d = np.searchsorted(np.asarray(borders), np.arange(cap), side="right").astype(np.int32)
    q = np.stack([d[s:s + n] for s in starts])
    return {"q_docs": q, "k_docs": np.tile(d, (S, 1))}


@pytest.mark.parametrize("pairs,queries,keys", FORM_OF)
@pytest.mark.parametrize("fmt", [0, 1])
def test_every_form(rt, rng, fmt, pairs, queries, keys):
    """Two query heads to a cache head where the queries are even, and twice the same bits."""
    group = 2 if queries % 2 == 0 else 1
    n = queries // group
    c = Case(rt, rng, fmt, 1, pairs * group, pairs, keys, n, [keys - n], layout=1).fill()
    pick = [0, n // 2, n - 1]
    got = c.check(pick=pick)
    c.call()
    assert np.array_equal(got, c.got())
    c.check({"causal": True, "prefix": np.array([keys // 3], np.int32)}, pick=pick)
    c.check({**docs_of(1, n, keys, [keys - n], [keys // 2, keys - 1]), "cap": 4.0,
             "slopes": np.linspace(0.001, 0.1, pairs * group, dtype=np.float32)}, pick=pick)


@pytest.mark.parametrize("H,KV,n", [(1, 1, 1), (2, 1, 1), (2, 1, 10), (2, 1, 100)])
@pytest.mark.parametrize("kind", ["none", "causal", "docs", "ordered", "prefix"])
def test_more_blocks_than_a_list_holds(rt, rng, H, KV, n, kind):
    """140,000 keys: 2,188 blocks, the last 140 in a run of their own."""
    cap = 140000
    c = Case(rt, rng, 0, 1, H, KV, cap, n, [cap - n], layout=1).fill()
    r = {}
    if kind == "causal":
        r = {"causal": True}
    if kind == "prefix":
        c.starts = np.array([cap - 5000], np.int32)
        r = {"causal": True, "prefix": np.array([132000], np.int32)}
    if kind in ("docs", "ordered"):
        borders = [50, 130900, 131100, cap - 60]
        r = docs_of(1, n, cap, [cap - n], borders)
        # the first and the last query of documents far apart
        r["q_docs"][0, 0], r["q_docs"][0, n // 2] = 2, 0
        r["docs_ordered"] = kind == "ordered"
    c.check(r, pick=[0, n // 2, n - 1])


BORDERS = [[100], [128], [64, 256], [1], [127], [10, 20, 30], [300, 428], [299, 300, 301], []]


@pytest.mark.parametrize("H,KV", [(2, 2), (2, 1), (3, 1)])
@pytest.mark.parametrize("borders", BORDERS)
def test_borders_of_documents_inside_tiles(rt, rng, H, KV, borders):
    """Queries of documents that begin anywhere in a tile (with 2 and 3 heads to a cache head
    128 and 85 queries fill no whole tile), of all keys and of those before them."""
    n = cap = 430
    c = Case(rt, rng, H % 2, 2, H, KV, cap, n, [0, 0], [n, 301], layout=0).fill()
    r = docs_of(2, n, cap, [0, 0], borders)
    pick = sorted({i for b in borders for i in (b - 1, b) if i < n} | {0, 63, 64, 300, n - 1})
    c.check(r, pick=pick)
    c.check({**r, "causal": True, "slopes": np.full(H, 0.02, np.float32)}, pick=pick)
    c.check({**r, "docs_ordered": True}, pick=pick)
    # a document that comes back
    r["q_docs"][:, n - 3:] = r["q_docs"][0, 0]
    r["q_docs"][:, 120:124] = r["q_docs"][0, 0]
    c.check(r, pick=pick + [119, 121, 124, n - 2])


@pytest.mark.parametrize("n", [1, 12, 200])
@pytest.mark.parametrize("cap", [1e-3, 2.0, 30.0, 1e6])
@pytest.mark.parametrize("bias", [False, True])
def test_scores_on_both_sides_of_the_caps_series(rt, rng, n, cap, bias):
    """Blocks of keys whose scores are all far below the cap, all above it, and mixed (one
    large key in a block), zeros among them."""
    keys = 400
    size = np.full((1, 1, keys, 1), 1.0)
    size[:, :, 64:128] = 1e-3
    size[:, :, 70] = 60.0
    size[:, :, 128:192] = 40.0
    size[:, :, 200] = 0.0
    c = Case(rt, rng, n % 2, 1, 2, 1, keys, n, [keys - n], ks=size).fill()
    r = {"cap": cap}
    if bias:
        r["slopes"] = np.array([0.5, 0.01], np.float32)
    c.check(r, label=f"cap {cap}")
    c.check({**r, "causal": True}, label=f"cap {cap} causal")


def test_a_cache_past_4_gib(rt, rng):
    """Codes, scales and f32 rows behind 2^32 bytes: the last head's rows, written, read
    back and attended to; the slots that nothing wrote are of another document."""
    H, cap, n = 70, 1000000, 5
    c = rt.kv_cache(0, 1, H, cap)
    assert len(c.k) > 2 ** 32
    k, v, q = (normals(rng, 1, H, n, 64) for _ in range(3))
    st = rt.upload_i32(np.array([cap - n], np.int32))
    rt.kv_cache_write_f32(c, rt.upload_f32(k), rt.upload_f32(v), n, st)
    (kc, kd), (vc, vd) = cached.quantise(k, 0), cached.quantise(v, 0)
    kh, vheld = cached.values(kc, kd, 0), cached.values(vc, vd, 0)
    docs = np.zeros(cap, np.int32)
    docs[cap - n:] = 1
    out = rt.alloc_f32(q.size)
    rules = vh.AttentionRules(q_docs=rt.upload_i32(np.ones(n, np.int32)), k_docs=rt.upload_i32(docs))
    rt.attention_cached_f32(c, rt.upload_f32(q), H, n, st, None, 0, rules, out)
    want, tol = cached.attention(q, kh, vheld, vd, n, None, None, {})
    assert np.all(np.abs(out.numpy().reshape(want.shape) - want) <= tol)
    # one row, and a tile of each head (its other rows see the same keys)
    one, docs = rt.alloc_f32(H * 64), rt.upload_i32(docs)
    rules = vh.AttentionRules(q_docs=rt.upload_i32(np.ones(1, np.int32)), k_docs=docs)
    last = rt.upload_i32(np.array([cap - 1], np.int32))
    rt.attention_cached_f32(c, rt.upload_f32(q[:, :, -1:]), H, 1, last, None, 0, rules, one)
    assert np.all(np.abs(one.numpy().reshape(1, H, 1, 64) - want[:, :, -1:]) <= tol[:, :, -1:])
    m = 40
    many = rt.alloc_f32(H * m * 64)
    qm = np.repeat(q[:, :, -1:], m, axis=2)
    rules = vh.AttentionRules(q_docs=rt.upload_i32(np.ones(m, np.int32)), k_docs=docs)
    rt.attention_cached_f32(c, rt.upload_f32(qm), H, m, rt.upload_i32(np.array([cap - m], np.int32)),
                            None, 0, rules, many)
    got = many.numpy().reshape(1, H, m, 64)
    assert np.all(np.abs(got - want[:, :, -1:]) <= tol[:, :, -1:])
    # 250,000 rows a head as f32: 4.48 GB
    rows = 250000
    assert H * rows * 256 > 2 ** 32
    back = rt.alloc_f32(H * rows * 64)
    rt.kv_cache_read_f32(c, rows, rt.upload_i32(np.array([cap - rows], np.int32)), None, back, None)
    for h in (0, 67, H - 1):
        tail = back.view((h * rows + rows - n) * 64, n * 64).numpy().reshape(n, 64)
        assert np.array_equal(tail, kh[0, h].astype(np.float32))


def test_no_slots_and_no_rows(rt, rng):
    for n in (1, 7, 150):
        c = Case(rt, rng, 0, 2, 2, 1, 0, n)
        c.cache = rt.kv_cache(0, 2, 1, 0)
        c.kh, c.vheld = np.zeros((2, 1, 0, 64)), np.zeros((2, 1, 0, 64))
        c.v_scale = np.zeros((2, 1, 0), np.float32)
        assert np.all(c.check() == 0)
        c = Case(rt, rng, 1, 2, 2, 1, 90, n, [5, 9], [0, -3]).fill()
        assert np.all(c.run({"causal": True}) == 7.0)


def test_padded_batches(rt, rng):
    """Sequences of every length beside one another, in each form; the rows behind the last one
    hold numbers that would show."""
    for H, KV, n, cap in ((2, 2, 1, 200), (4, 2, 12, 200), (4, 2, 150, 400)):
        S = 5
        counts = np.array([n, 0, max(n // 2, 1), 1, n], np.int32)
        starts = np.array([cap - n, 3, 0, cap - 1, 64], np.int32)
        c = Case(rt, rng, 0, S, H, KV, cap, n, starts, counts, layout=n % 2).fill()
        for s in range(S):
            c.q[s, :, counts[s]:] = np.nan
        c.check({"causal": True, "slopes": np.full(H, 0.1, np.float32)})
        c.check({**docs_of(S, n, 2 * cap, starts, [40, 130]),
                 "k_docs": docs_of(S, n, cap, [0] * S, [40, 130])["k_docs"]})


def test_two_runtimes_side_by_side(rng):
    """Calls of two runtimes (each its stream and work buffer), queued together."""
    a, b = vh.Runtime(0), vh.Runtime(0)
    cases = [Case(r, rng, 0, 1, 2, 1, 5000, n, [5000 - n]).fill() for n in (1, 8, 200) for r in (a, b)]
    want = [c.run() for c in cases]
    for _ in range(3):
        for c in cases:
            c.call()
    for c, w in zip(cases, want):
        assert np.array_equal(c.got(), w)


def test_graphs_outlive_a_larger_work_buffer(rng):
    """Captured calls of each form, an eager call that needs a larger buffer, replays."""
    rt = vh.Runtime(0)
    cases = [Case(rt, rng, 1, 1, 2, 1, 6000, n, [6000 - n]).fill() for n in (1, 9, 130)]
    want = [c.run({"causal": True}) for c in cases]
    rt.synchronize()
    graphs = [cached.captured(rt, c.call) for c in cases]
    big = Case(rt, rng, 0, 8, 8, 8, 2000, 450).fill()
    first = big.run()
    for _ in range(3):
        for c in cases:
            c.out.write(np.zeros(c.q.size, np.float32))
        for g in graphs:
            g.launch()
        big.call()
        for c, w in zip(cases, want):
            assert np.array_equal(c.got(), w)
        assert np.array_equal(big.got(), first)


def test_keys_and_values_of_one_tensor(rt, rng):
    """The same tensor as K and V, and one tensor as starts and counts."""
    x = normals(rng, 2, 3, 40, 64)
    c = rt.kv_cache(1, 2, 3, 90)
    t, sc = rt.upload_f32(x), rt.upload_i32(np.array([30, 40], np.int32))
    rt.kv_cache_write_f32(c, t, t, 40, sc, sc, vh.VK_QK_VIEWS_OUTER)
    k, v = rt.alloc_f32(x.size), rt.alloc_f32(x.size)
    rt.kv_cache_read_f32(c, 40, sc, sc, k, v, vh.VK_QK_VIEWS_OUTER)
    held = cached.values(*cached.quantise(x, 1), 1).astype(np.float32)
    for got in (k.numpy().reshape(x.shape), v.numpy().reshape(x.shape)):
        assert np.array_equal(got[0, :, :30], held[0, :, :30]) and np.array_equal(got[1], held[1])


def garbage(rng, c, slots):
    """Fills `slots` of every sequence and head of a cache with bytes and scales of every kind."""
    def put(t, width, dtype, values):
        a = np.empty(len(t), dtype)
        if dtype == np.uint8:
            assert vh.lib.vk_download_u8(c.rt.handle, t.handle, a.ctypes.data, a.size) == 0
        else:
            a = t.numpy()
        a = a.reshape(c.S, c.KV, c.cap, width)
        a[:, :, slots] = rng.choice(values, a[:, :, slots].shape)
        t.write(np.ascontiguousarray(a.reshape(-1)))
    for t in (c.cache.k, c.cache.v):
        put(t, 64, np.uint8, np.array([0x7f, 0xff, 0x80, 0, 0x7e, 0xfe, 1, 77], np.uint8))
    for t in (c.cache.k_scale, c.cache.v_scale):
        put(t, 1, np.float32, np.array([np.nan, np.inf, -np.inf, 3.4e38, -3.4e38, 1e-44, -0.0, 5.0],
                                       np.float32))


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("n,cap", [(1, 300), (1, 3000), (11, 300), (11, 3000), (150, 500)])
@pytest.mark.parametrize("rule", [{}, {"cap": 20.0}])
def test_slots_that_nothing_wrote(rt, rng, fmt, n, cap, rule):
    """Slots of another document, of later positions and past the length may hold anything:
    the same bits."""
    end = cap - 40
    c = Case(rt, rng, fmt, 2, 2, 1, cap, n, [end - n] * 2).fill()
    r = {**rule, "causal": True, "q_docs": np.zeros((2, n), np.int32),
         "k_docs": np.zeros((2, cap), np.int32)}
    hidden = np.concatenate([np.arange(0, 70), np.arange(100, end - n, 7)])
    r["k_docs"][:, hidden] = 1
    want = c.check(r, pick=[0, n // 2, n - 1])
    later = np.arange(end - n // 2, cap)  # behind the length, and behind the first queries
    garbage(rng, c, np.concatenate([hidden, np.arange(end, cap)]))
    assert np.array_equal(c.run(r), want)
    garbage(rng, c, later)
    keep = n - n // 2
    assert np.array_equal(c.run(r)[:, :, :keep], want[:, :, :keep])


@pytest.mark.parametrize("n", [1, 11, 150])
def test_codes_that_are_no_number(rt, rng, n):
    """e4m3's codes 0x7f and 0xff, put there by hand: zeros in V, NaN to who sees them in K."""
    c = Case(rt, rng, 1, 1, 2, 2, 300, n, [300 - n]).fill()
    clean = c.run()
    codes = cached.quantise(c.v, 1)[0]
    codes[0, 0, 100, ::3], codes[0, 1, 5, 7] = 0x7f, 0xff
    c.cache.v.write(codes.reshape(-1))
    c.vheld = np.nan_to_num(cached.values(codes, c.v_scale, 1), nan=0.0)
    got = c.check()
    assert not np.array_equal(got, clean)
    codes = cached.quantise(c.k, 1)[0]
    codes[0, 1, 200, 9] = 0x7f
    c.cache.k.write(codes.reshape(-1))
    assert np.array_equal(c.run()[:, 0], got[:, 0]) and np.isnan(c.got()[:, 1]).all()


def test_scales_out_of_range_are_refused(rt):
    c = rt.kv_cache(0, 1, 1, 4)
    q, o = rt.upload_f32(np.ones(64)), rt.alloc_f32(64)
    for args in (dict(scale=1e-13), dict(scale=-1e13), dict(cap=1e-14), dict(cap=1e12),
                 dict(scale=1e6, cap=1e-7), dict(scale=1e-44)):
        with pytest.raises(vh.UnsupportedShape):
            rt.attention_cached_f32(c, q, 1, 1, None, None, 0, vh.AttentionRules(**args), o)


@pytest.mark.parametrize("n", [1, 11, 150])
@pytest.mark.parametrize("rule", [{"scale": -0.25}, {"scale": 2.0 ** -39}, {"scale": -0.5, "cap": 3.0},
                                  {"scale": 0.125, "cap": 1e11}, {"scale": 0.125, "cap": 2e-13}])
def test_scales_at_the_ends_of_the_range(rt, rng, n, rule):
    c = Case(rt, rng, n % 2, 1, 2, 1, 260, n, [260 - n]).fill()
    c.check(rule)


def test_more_workgroups_than_a_launch_holds_are_refused(rt):
    """16,777,215 sequences of one query: 2^33 threads."""
    S = 0xffffff
    c = rt.kv_cache(0, S, 1, 1)
    q, o = rt.alloc_f32(S * 64), rt.alloc_f32(S * 64)
    with pytest.raises(vh.UnsupportedShape):
        rt.attention_cached_f32(c, q, 1, 1, None, None, 0, None, o)
    rt.synchronize()


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("S,H,keys", [(1, 1, 1), (1, 64, 130), (1, 65, 130), (16, 4, 1536),
                                      (13, 5, 65), (2, 3, 1537)])
def test_single_rows_of_few_and_many_heads(rt, rng, fmt, S, H, keys):
    """Rows whose columns are shared out over workgroups (64 at most on 256 CUs) and rows of
    one, up to the longest unsplit cache and a key past it."""
    starts = [max(keys - 1 - 7 * s, 0) for s in range(S)]
    c = Case(rt, rng, fmt, S, H, H, keys, 1, starts, layout=fmt).fill()
    c.check()
    c.check({"causal": True, "cap": 10.0, "slopes": np.linspace(0.0, 0.2, H, dtype=np.float32)})


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("qs,ks", [(1e-36, 1e36), (1e-34, 1e37), (1e36, 1e-26), (1e30, 1e-28),
                                   (1e-36, 1.0)])
@pytest.mark.parametrize("n", [1, 9, 70])
def test_queries_at_the_ends_of_f32(rt, rng, fmt, qs, ks, n):
    """Products that stay in range, of factors that do not: the largest and the smallest
    queries with keys the other way round."""
    c = Case(rt, rng, fmt, 1, 2, 1, 330, n, [330 - n], qs=qs, ks=ks).fill()
    c.check(label=f"{qs} {ks}")


def test_misaligned_tensors_are_refused(rt):
    import ctypes
    c = rt.kv_cache(0, 2, 1, 4)
    q, o = rt.upload_f32(np.ones(128)), rt.alloc_f32(128)
    raw = rt.upload_i32(np.zeros(8, np.int32))
    h = ctypes.c_void_p()
    if vh.lib.vk_tensor_wrap(rt.handle, vh.VK_I32, raw.device_ptr + 2, 2, ctypes.byref(h)) != 0:
        return
    odd = vh.Tensor(rt, h)
    for call in (lambda: rt.kv_cache_write_f32(c, q, q, 1, odd),
                 lambda: rt.kv_cache_read_f32(c, 1, None, odd, o, None),
                 lambda: rt.attention_cached_f32(c, q, 1, 1, odd, None, 0, None, o),
                 lambda: rt.attention_cached_f32(c, q, 1, 1, None, None, 0,
                                                 vh.AttentionRules(causal=True, prefix=odd), o)):
        with pytest.raises(vh.VestraError) as e:
            call()
        assert e.value.code == vh.VK_ERR_INVALID


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("n,cap,seen", [(1, 300, 100), (1, 4000, 2500), (9, 300, 100), (9, 4000, 2500),
                                        (150, 500, 100), (150, 4000, 2500)])
@pytest.mark.parametrize("slope", [2.0 ** 7, 2.0 ** 14, 2.0 ** 20])
@pytest.mark.parametrize("vs", [1e-5, 1.0, 1e8])
def test_scores_far_from_zero(rt, rng, fmt, n, cap, seen, slope, vs):
    """Keys all far from the queries under a steep bias: scores of -2^17 to -2^32, where f32's
    step is up to 512; the nearest key outweighs the next by 2^100 at least."""
    c = Case(rt, rng, fmt, 1, 3, 3, cap, n, [cap - n], vs=vs).fill()
    c.check({"slopes": np.array([slope, slope, 0.0], np.float32)}, max_length=seen,
            pick=[0, n // 2, n - 1])


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("n", [1, 20, 70])
def test_single_heads_at_the_ends_of_f32(rt, rng, fmt, n):
    """As the test of both ends above, a head to a cache head."""
    for qs, ks in ((1e36, 1e-26), (1e-36, 1e36), (3e37, 1e-28)):
        c = Case(rt, rng, fmt, 1, 2, 2, 200, n, [200 - n], qs=qs, ks=ks).fill()
        c.check(label=f"{qs} {ks}")
