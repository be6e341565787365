"""Plain 64-bit forms of the cache's and the cached attention's operators, for their tests."""
import numpy as np

U = 2.0 ** -24
TOP = {0: 127.0, 1: 448.0}  # VK_CACHE_Q8, VK_CACHE_F8
LEAST = 2.0 ** -100


def e4m3_values():
    """The values of the 256 codes (NaN for 0x7f and 0xff)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    x = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    x = np.where((c & 127) == 127, np.nan, x)
    return np.where(c & 128, -x, x)


def quantise(x, fmt):
    """(codes u8, scales f32) of f32 rows [..., 64], from the definition: the scale
    rounded to f32, the quotient to f32 and then to the nearest code."""
    x = np.asarray(x, np.float32)
    odd = ~np.isfinite(x).all(-1)
    top = np.abs(np.where(np.isfinite(x), x, 0)).max(-1)
    d = (top / np.float32(TOP[fmt])).astype(np.float32)
    most = float(np.finfo(np.float32).max) / TOP[fmt]  # no held value is infinite
    most = np.nextafter(np.float32(most), np.float32(0)) if float(np.float32(most)) > most else np.float32(most)
    d = np.minimum(d, most)
    none = odd | (d < LEAST)
    safe = np.where(none, np.float32(1), d)
    with np.errstate(over="ignore", invalid="ignore"):
        y = np.where(none[..., None], np.float32(0), x / safe[..., None]).astype(np.float32)
    if fmt == 0:
        codes = np.rint(y).astype(np.int64) & 255
    else:
        table = e4m3_values()[:127]
        a = np.abs(y).astype(np.float64)
        hi = np.clip(np.searchsorted(table, a), 1, 126)
        lo = hi - 1
        dl, dh = a - table[lo], table[hi] - a
        code = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
        codes = code + 128 * (np.signbit(y) & True)
    d = np.where(odd, np.float32(np.nan), np.where(none, np.float32(0), d)).astype(np.float32)
    return codes.astype(np.uint8), d


def values(codes, scales, fmt):
    """The held values in 64 bits."""
    c = codes.astype(np.uint8)
    x = c.view(np.int8).astype(np.float64) if fmt == 0 else e4m3_values()[c]
    return x * scales.astype(np.float64)[..., None]


def spans(n, cap, starts, counts, s):
    start = 0 if starts is None else int(starts[s])
    count = n if counts is None else max(min(int(counts[s]), n), 0)
    return start, count


def visible(s, i, start, end, rules):
    """Which of the keys 0..end-1 query i of sequence s sees."""
    j = np.arange(end)
    p = start + i
    seen = np.ones(end, bool)
    if rules.get("causal"):
        seen &= j <= p
        if rules.get("prefix") is not None:
            seen |= j < int(rules["prefix"][s])
    if rules.get("q_docs") is not None:
        qd, kd = int(rules["q_docs"][s, i]), rules["k_docs"][s, :end]
        seen &= (kd <= qd) if rules.get("docs_ordered") else (kd == qd)
    return seen


def attention(q, kv, vv, v_scale, n, starts, counts, rules, limit=0, pick=None):
    """out [S, H, n, 64] and the bound of its error, from q [S, H, n, 64], the held
    values [S, KV, cap, 64] and V's scales; rows past the counts are NaN (not written).

    An f32 kernel's weight of key j is off by e_j of itself: the score's products and
    sums (16 u of the sum of their sizes: 2 u a factor held as two f16 parts and eight
    roundings of a 64-term sum with room), the scale, the cap (tanh to 8 u of the cap), the
    bias and the running reference (a rounding each, at their size), 2^x and the
    weight's own two parts (64 u with the constant terms).  The output then moves by sum_j
    p_j e_j |v_j - o|, and the value sum rounds (2 sqrt(n) + blocks + 8) u of sum p |v|.

    Two floors beside these.  A query's values are scaled so that its largest is at least 1,
    and their second part is a multiple of 2^-24: off by 2^-25 = u / 2 of the row's largest
    |q| at most, whatever the value's own size, which moves a score by that times sum
    |k_d|.  A weight (2^x times V's scale) is at least 2^9 for the largest and its second part
    a multiple of 2^-24: off by 2^-34 of the largest at most, whatever its own size (and
    left out below), which moves the output by that times sum_j |code_j|."""
    S, H, _, _ = q.shape
    KV, cap = kv.shape[1], kv.shape[2]
    out = np.full(q.shape, np.nan)
    tol = np.zeros(q.shape)
    scale = rules.get("scale") or 0.125
    c = rules.get("cap") or 0.0
    for s in range(S):
        start, count = spans(n, cap, starts, counts, s)
        end = max(min(start + count, limit or cap, cap), 0)
        for h in range(H):
            k, v = kv[s, h * KV // H, :end], vv[s, h * KV // H, :end]
            lsv = np.abs(np.log2(np.maximum(v_scale[s, h * KV // H, :end].astype(np.float64), LEAST)))
            rows = range(count) if pick is None else [i for i in pick if i < count]
            for i in rows:
                seen = visible(s, i, start, end, rules)
                if not seen.any():
                    out[s, h, i] = 0
                    continue
                ks, vs = k[seen], v[seen]
                x = q[s, h, i].astype(np.float64)
                u = ks @ x * scale
                terms = np.abs(ks) @ np.abs(x) * abs(scale)
                e = 16 * terms + 8 * np.abs(u) + 64 + 2 * lsv[seen]
                e = e + 0.5 * np.abs(x).max() * np.abs(ks).sum(1) * abs(scale)
                if c:
                    u = c * np.tanh(u / c)
                    e = e + 8 * c
                if rules.get("slopes") is not None:
                    b = float(rules["slopes"][h]) * np.abs(start + i - np.arange(end)[seen])
                    u = u - b
                    e = e + 4 * np.abs(b)
                top = u.max()
                e = (e + 2 * abs(top)) * U
                p = np.exp(u - top)
                p /= p.sum()
                o = p @ vs
                out[s, h, i] = o
                size = p @ np.abs(vs)
                tol[s, h, i] = (p * e) @ np.abs(vs - o) + 2 * U * np.abs(o) + (
                    2 * np.sqrt(len(p)) + len(p) / 64 + 8) * U * size + 1e-38
                sv = np.maximum(v_scale[s, h * KV // H, :end][seen].astype(np.float64), LEAST)
                tol[s, h, i] += 2.0 ** -34 * (p * sv).max() * (np.abs(vs) / sv[:, None]).sum(0)
    return out, tol


def set_i32(rt, t, a):
    """New values for an i32 tensor of the library (through an f32 view of its bits)."""
    import ctypes

    import vestra_hip as vh
    h = ctypes.c_void_p()
    assert vh.lib.vk_tensor_wrap(rt.handle, vh.VK_F32, t.device_ptr, len(t), ctypes.byref(h)) == 0
    vh.Tensor(rt, h).write(np.asarray(a, np.int32).view(np.float32))


def captured(rt, run):
    """The graph of what `run` enqueues.  Tensors of earlier tests that the collector
    frees meanwhile would end the capture."""
    import gc
    gc.collect()
    gc.disable()
    try:
        rt.begin_capture()
        try:
            run()
        finally:
            graph = rt.end_capture()
    finally:
        gc.enable()
    return graph


def heads_outer(x):
    """[S, H, n, 64] -> [H, S, n, 64] and back."""
    return np.ascontiguousarray(x.swapaxes(0, 1))
