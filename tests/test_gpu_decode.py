"""The decode operators against float64 statements (oracle/decode_ref.py): norm and rotation of queries and keys, the
8-bit key/value cache, attention over it, products with 4-bit weights, and a run of them together.  The bounds come with
the references; codes have to be equal."""
import numpy as np
import pytest

import decode_ref as ref
from conftest import seeded

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16"]


def code_of(wgf, kind):
    return {"f32": wgf.F32, "f16": wgf.F16, "bf16": wgf.BF16}[kind]


def give(wgf, dev, x, kind):
    return dev.tensor(ref.store(x, kind), dtype=code_of(wgf, kind))


def take(t, kind):
    return ref.load(t.as_slice(), kind)


def draw(g, shape, kind, std=1.0, mean=0.0):
    return ref.round_to(g.standard_normal(shape) * std + mean, kind)


def tables(positions, d, kind):
    a = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)[None, :]
    return ref.round_to(np.cos(a), kind), ref.round_to(np.sin(a), kind)


def close(got, want, bound):
    assert got.shape == want.shape
    bad = ~(np.abs(got.astype(np.float64) - want) <= bound)
    assert not bad.any(), (int(bad.sum()), float(np.max(np.where(bad, np.abs(got - want) / bound, 0))))


# ---- norm and rotation -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,seq,heads,kv_heads,dim,start", [
    (1, 1, 1, 1, 2, 0), (2, 3, 4, 2, 64, 5), (1, 700, 6, 1, 128, 0), (3, 1, 32, 8, 128, 90), (2, 37, 5, 3, 80, 2), (1, 9, 2, 2, 6, 1),
    (1, 5, 3, 1, 96, 0), (1, 5, 3, 1, 256, 0), (1, 4, 2, 1, 512, 3), (2, 65, 7, 5, 34, 0)])
def test_qk_norm_rope(kind, batch, seq, heads, kv_heads, dim, start, wgf, dev):
    g = seeded(20, dim + seq)
    q, k = draw(g, (batch, seq, heads, dim), kind), draw(g, (batch, seq, kv_heads, dim), kind, 3.0)
    wq, wk = draw(g, (dim,), kind, 0.2, 1.0), draw(g, (dim,), kind, 0.2, 1.0)
    cos, sin = tables(start + seq + 2, dim, kind)
    t = [give(wgf, dev, x, kind) for x in (q, k, wq, wk, cos, sin)]
    before = dev.launch_count
    a, b = t[0].transpose(1, 2).qk_norm_rope(t[1].transpose(1, 2), *t[2:], eps=1e-5, start=start)
    wgf.Tensor.materialize_all([a, b])
    assert dev.launch_count - before == 1
    for got, x, w in ((a, q, wq), (b, k, wk)):
        want, off = ref.norm_rope(x.transpose(0, 2, 1, 3), w, cos, sin, 1e-5, start + np.arange(seq))
        close(take(got, kind), want, off * 1.01 + ref.rounding(want, kind) * 1.01)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_qk_norm_rope_of_views(kind, wgf, dev):
    """Offsets and strides that no vector fits, a last axis that is not the dense one, rank 3, and both results
    used as operands."""
    g = seeded(20, 1000)
    d, s = 64, 7
    q, k = draw(g, (4, s, d + 1), kind), draw(g, (d, s, 2), kind)
    w = draw(g, (2 * d + 1,), kind, 0.2, 1.0)
    cos, sin = tables(20, d, kind)
    tq, tk, tw, tc, ts = (give(wgf, dev, x, kind) for x in (q, k, w, cos, sin))
    a, b = tq.slice([(0, 4), (0, s), (1, d + 1)]).qk_norm_rope(tk.transpose(0, 2), tw.slice([(1, d + 1)]), tw.slice([(d, 2 * d)]), tc, ts,
                                                              eps=0.5, start=3)
    wa, oa = ref.norm_rope(q[:, :, 1:], w[1: d + 1], cos, sin, 0.5, 3 + np.arange(s))
    wb, ob = ref.norm_rope(k.transpose(2, 1, 0), w[d: 2 * d], cos, sin, 0.5, 3 + np.arange(s))
    close(take(a, kind), wa, oa + ref.rounding(wa, kind) * 1.01)
    close(take(b, kind), wb, ob + ref.rounding(wb, kind) * 1.01)
    np.testing.assert_array_equal(take(b * 2.0, kind), take(b, kind) * 2)


def test_qk_norm_rope_keeps_a_bad_head_to_itself(wgf, dev):
    g = seeded(20, 1001)
    x = draw(g, (3, 4, 64), "f32")
    x[1, 2, 5], x[0, 1, 0], x[2, 3] = np.nan, np.inf, 0.0
    cos, sin = tables(4, 64, "f32")
    w = np.ones(64, np.float32)
    a, b = dev.tensor(x).qk_norm_rope(dev.tensor(x), dev.tensor(w), dev.tensor(w), dev.tensor(cos), dev.tensor(sin), eps=1e-5)
    a = a.as_slice()
    np.testing.assert_array_equal(a, b.as_slice())
    bad = np.zeros((3, 4), bool)
    bad[1, 2] = bad[0, 1] = True
    assert np.isfinite(a[~bad]).all() and np.isnan(a[1, 2]).all() and np.isnan(a[0, 1]).any()
    np.testing.assert_array_equal(a[2, 3], 0)


# ---- the cache ----------------------------------------------------------------------------------------------------------
def kept(x, lengths):
    """What read() has to give for x [batch, heads, tokens, dim] cut at each length, as float32 before the last rounding."""
    y = np.zeros(x.shape[:2] + (max(lengths), x.shape[3]), np.float32)
    for b, n in enumerate(lengths):
        for h in range(x.shape[1]):
            y[b, h, :n] = ref.stands_for(x[b, h, :n])
    return y


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,heads,dim", [([1], 1, 64), ([64], 2, 128), ([65, 0, 3], 2, 64), ([200, 63, 128], 3, 128), ([130], 1, 8),
                                               ([77, 90], 2, 80), ([70], 1, 256), ([129, 5], 2, 96), ([66], 2, 200)])
def test_cache_codes(kind, lengths, heads, dim, wgf, dev):
    g = seeded(21, dim + lengths[0])
    t = max(lengths)
    k, v = draw(g, (len(lengths), heads, t, dim), kind, 2.0), draw(g, (len(lengths), heads, t, dim), kind)
    k[..., dim // 2] *= 8
    k = ref.round_to(k, kind)
    v[0, 0, 0] = 0
    c = dev.kv_cache(len(lengths), heads, dim, t + 3, code_of(wgf, kind))
    c.append(give(wgf, dev, k, kind), give(wgf, dev, v, kind), counts=lengths)
    assert c.lengths == lengths
    for got, x in zip(c.read(), (k, v)):
        np.testing.assert_array_equal(take(got, kind), ref.round_to(kept(x, lengths), kind))


@pytest.mark.parametrize("kind", KINDS)
def test_cache_codes_of_ties_and_of_far_sizes(kind, wgf, dev):
    """Values half way between two codes, blocks of zeros, of the type's smallest and of its largest numbers."""
    top = {"f32": 2.0 ** 127, "f16": 60000.0, "bf16": 2.0 ** 127}[kind]
    low = {"f32": 2.0 ** -120, "f16": 2.0 ** -24, "bf16": 2.0 ** -120}[kind]
    x = np.zeros((1, 1, 5 * 64, 64), np.float32)
    x[0, 0, :64] = np.linspace(-127, 127, 64 * 64).reshape(64, 64)
    x[0, 0, 0, 0], x[0, 0, 1, :40] = 127, np.arange(40) + 0.5
    x[0, 0, 64:128] = np.linspace(-1, 1, 64 * 64).reshape(64, 64) * top
    x[0, 0, 128:192, :3] = low
    x[0, 0, 192:256] = np.linspace(-1, 1, 64 * 64).reshape(64, 64) * 2.0 ** -8
    x = ref.round_to(x, kind)
    c = dev.kv_cache(1, 1, 64, 5 * 64, code_of(wgf, kind))
    c.append(give(wgf, dev, x, kind), give(wgf, dev, -x, kind))
    for got, want in zip(c.read(), (x, -x)):
        np.testing.assert_array_equal(take(got, kind), ref.round_to(kept(want, [5 * 64]), kind))


def contents(c, q, kind):
    return [a.as_slice() for a in c.read()] + [c.attention(q).as_slice()]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("steps", [[1] * 9 + [60] + [1] * 70, [10, 150, 64, 40], [64, 64, 136], [1, 263], [63, 1, 1, 199], [130, 134]])
def test_cache_does_not_depend_on_how_tokens_came(kind, steps, wgf, dev):
    g = seeded(21, 7)
    n = sum(steps)
    k, v = draw(g, (2, 2, n, 64), kind), draw(g, (2, 2, n, 64), kind)
    k[:, :, ::7] *= 5
    k = ref.round_to(k, kind)
    tk, tv, q = give(wgf, dev, k, kind), give(wgf, dev, v, kind), give(wgf, dev, draw(g, (2, 4, 1, 64), kind), kind)
    whole, parts = (dev.kv_cache(2, 2, 64, n, code_of(wgf, kind)) for _ in range(2))
    whole.append(tk, tv)
    at = 0
    for s in steps:
        w = [(0, 2), (0, 2), (at, at + s), (0, 64)]
        parts.append(tk.slice(w), tv.slice(w))
        at += s
    for a, b in zip(contents(whole, q, kind), contents(parts, q, kind)):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("first,second,back,more", [(100, 60, 101, 30), (10, 150, 64, 90), (10, 200, 192, 5), (10, 120, 65, 1), (70, 190, 193, 64),
                                                    (64, 64, 64, 70), (64, 63, 64, 3), (5, 3, 0, 130), (130, 100, 128, 10), (60, 10, 30, 1)])
def test_truncate_then_append(first, second, back, more, wgf, dev):
    """Tokens taken back and others appended: as if the first had never come."""
    g = seeded(21, first + back)
    n = first + second + more
    k, v = draw(g, (2, 3, n, 64), "f16", 2.0), draw(g, (2, 3, n, 64), "f16")
    k[:, :, first + 2:] *= 6
    k = ref.round_to(k, "f16")
    q = give(wgf, dev, draw(g, (2, 3, 1, 64), "f16"), "f16")
    t = lambda x, a, b: give(wgf, dev, x[:, :, a:b], "f16")
    c, plain = (dev.kv_cache(2, 3, 64, n, wgf.F16) for _ in range(2))
    c.append(t(k, 0, first), t(v, 0, first))
    c.append(t(k, first, first + second), t(v, first, first + second))
    c.truncate([back, c.lengths[1]])
    kk, vv = np.concatenate([k[:, :, :back], k[:, :, -more:]], 2), np.concatenate([v[:, :, :back], v[:, :, -more:]], 2)
    # right behind the truncation ...
    if back:
        plain.append(t(k, 0, back), t(v, 0, back))
        for a, b in zip(c.read(), plain.read()):
            np.testing.assert_array_equal(a.as_slice()[0, :, :back], b.as_slice()[0])
    # ... and behind the next append
    other = dev.kv_cache(2, 3, 64, n, wgf.F16)
    other.append(give(wgf, dev, kk, "f16"), give(wgf, dev, vv, "f16"))
    c.append(t(k, n - more, n), t(v, n - more, n), counts=[more, 0])
    for a, b in zip(contents(c, q, "f16"), contents(other, q, "f16")):
        b = b[0]
        np.testing.assert_array_equal(a[0][:, : b.shape[1]], b)


def test_cache_takes_views_and_padding_is_not_read(wgf, dev):
    g = seeded(21, 9)
    k = draw(g, (2, 90, 3, 65), "f16")
    v = draw(g, (64, 2, 3, 90), "f16")
    k[0, 70:], v[:, 0, :, 70:] = np.nan, np.inf
    tk = dev.tensor(ref.store(k, "f16")).transpose(1, 2).slice([(0, 2), (0, 3), (0, 90), (1, 65)])       # odd offset, odd row stride
    tv = dev.tensor(ref.store(v, "f16")).transpose(0, 1).transpose(1, 2).transpose(2, 3)                  # [2, 3, 90, 64], last axis strided
    c = dev.kv_cache(2, 3, 64, 128, wgf.F16)
    c.append(tk, tv, counts=[70, 90])
    kk, vv = k.transpose(0, 2, 1, 3)[..., 1:], v.transpose(1, 2, 3, 0)
    for got, x in zip(c.read(), (kk, vv)):
        np.testing.assert_array_equal(take(got, "f16"), ref.round_to(kept(x, [70, 90]), "f16"))
    q = draw(g, (2, 3, 2, 64), "f16")
    out = take(c.attention(dev.tensor(ref.store(q, "f16"))), "f16")
    assert np.isfinite(out).all()


# ---- attention over the cache ---------------------------------------------------------------------------------------------
def check_attention(wgf, dev, kind, lengths, heads, kv_heads, dim, t, counts=None, scale=None, room=5, grow=1.0, g=None, q=None):
    g = g or seeded(22, dim + t + heads)
    b, n = len(lengths), max(max(lengths), 1)
    k, v = draw(g, (b, kv_heads, n, dim), kind), draw(g, (b, kv_heads, n, dim), kind)
    if grow != 1.0:
        k = ref.round_to(k * (1 + grow * np.arange(n)[None, None, :, None] / n), kind)
    q = draw(g, (b, heads, t, dim), kind) if q is None else q
    c = dev.kv_cache(b, kv_heads, dim, n + room, code_of(wgf, kind))
    c.append(give(wgf, dev, k, kind), give(wgf, dev, v, kind), counts=lengths)
    before = dev.launch_count
    out = c.attention(give(wgf, dev, q, kind), scale=scale, counts=counts)
    assert dev.launch_count - before == 1
    out = take(out, kind)
    s = scale if scale is not None else dim ** -0.5
    for i, m in enumerate(lengths):
        kk = np.stack([ref.stands_for(k[i, h, :m]) for h in range(kv_heads)])
        vv = np.stack([ref.stands_for(v[i, h, :m]) for h in range(kv_heads)])
        want, bound = ref.attention(q[i], kk, vv, s, None if counts is None else counts[i])
        close(out[i], want, bound + ref.rounding(want, kind))
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,t", [
    ([1], 1, 1, 64, 1), ([64], 8, 1, 128, 1), ([65, 0, 3], 4, 2, 64, 1), ([700, 63, 128], 12, 3, 128, 1), ([2000], 32, 8, 128, 1),
    ([77, 90], 14, 2, 80, 1), ([270], 9, 1, 256, 1), ([129, 5], 4, 4, 192, 1), ([333], 40, 2, 96, 1), ([50], 2, 1, 8, 1),
    ([300, 2], 8, 2, 64, 5), ([100, 700], 3, 3, 128, 17), ([260], 4, 1, 64, 130)])
def test_cache_attention(kind, lengths, heads, kv_heads, dim, t, wgf, dev):
    check_attention(wgf, dev, kind, lengths, heads, kv_heads, dim, t)


def test_cache_attention_split_over_many_ctas(wgf, dev):
    check_attention(wgf, dev, "f16", [20011], 4, 1, 128, 1)
    check_attention(wgf, dev, "f32", [9000, 64, 5000], 2, 2, 64, 3)


def test_cache_attention_with_counts_and_scale(wgf, dev):
    out = check_attention(wgf, dev, "f16", [100, 30, 2, 0], 4, 2, 64, 4, counts=[4, 0, 3, 2], scale=0.3)
    assert not out[1].any() and not out[3].any() and not out[0, :, 4:].any() and not out[2, :, 0].any()


def test_cache_attention_of_rising_scores(wgf, dev):
    """Keys whose norms grow along the sequence: the running maximum moves with most blocks, across warps and parts."""
    check_attention(wgf, dev, "f32", [3000], 4, 1, 64, 1, grow=20.0)
    check_attention(wgf, dev, "bf16", [3000], 4, 1, 128, 1, grow=20.0)


@pytest.mark.parametrize("kind,size", [("f32", 1e30), ("f32", 1e-30), ("bf16", 1e30), ("f16", 6e4), ("f16", 1e-7)])
def test_cache_attention_of_far_query_sizes(kind, size, wgf, dev):
    """The scale brings the scores back to ordinary sizes; the queries keep their digits on the way."""
    g = seeded(22, 99)
    q = ref.round_to(np.clip(g.standard_normal((1, 4, 1, 64)) / 5, -1, 1) * size, kind)
    check_attention(wgf, dev, kind, [200], 4, 2, 64, 1, scale=0.5 / size, g=g, q=q)


def test_cache_attention_keeps_bad_values_where_they_are(wgf, dev):
    """NaN and infinity in a token reach the queries that see its block and no others; a NaN query its own row alone."""
    g = seeded(22, 98)
    k, v = draw(g, (1, 2, 200, 64), "f16"), draw(g, (1, 2, 200, 64), "f16")
    k[0, 0, 130, 5], v[0, 1, 199, 0] = np.nan, np.inf
    q = draw(g, (1, 4, 80, 64), "f16")
    q[0, 3, 0, 0] = np.nan
    c = dev.kv_cache(1, 2, 64, 256, wgf.F16)
    c.append(*(dev.tensor(ref.store(x, "f16")) for x in (k, v)))
    out = take(c.attention(dev.tensor(ref.store(q, "f16"))), "f16")[0]
    # queries stand at 120 .. 199; kv head 0's block 2 (128 .. 191) has a NaN, kv head 1's block 3 (192 .. 199) an infinity
    pos = np.arange(120, 200)
    assert np.isfinite(out[:2][:, pos < 128]).all() and np.isnan(out[:2][:, pos >= 128]).all()
    assert np.isfinite(out[2][pos < 192]).all() and np.isnan(out[2][pos >= 192]).all()
    assert np.isnan(out[3][0]).all() and np.isfinite(out[3][1:72]).all()


def test_cache_attention_gives_the_same_bits_again(wgf, dev):
    g = seeded(22, 97)
    k, v, q = (draw(g, s, "bf16") for s in ((3, 2, 5000, 128), (3, 2, 5000, 128), (3, 8, 1, 128)))
    c = dev.kv_cache(3, 2, 128, 5000, wgf.BF16)
    c.append(give(wgf, dev, k, "bf16"), give(wgf, dev, v, "bf16"), counts=[5000, 70, 1234])
    t = give(wgf, dev, q, "bf16")
    first = c.attention(t).as_slice()
    for _ in range(20):
        np.testing.assert_array_equal(c.attention(t).as_slice(), first)


def test_cache_beyond_four_gigabytes(wgf, dev):
    """The last sequence's codes lie past 2^32 bytes."""
    g = seeded(22, 96)
    k, v, q = draw(g, (3, 8, 100, 128), "f16"), draw(g, (3, 8, 100, 128), "f16"), draw(g, (3, 8, 1, 128), "f16")
    c = dev.kv_cache(3, 8, 128, 1_100_000, wgf.F16)
    c.append(dev.tensor(ref.store(k, "f16")), dev.tensor(ref.store(v, "f16")), counts=[100, 0, 77])
    out = take(c.attention(dev.tensor(ref.store(q, "f16"))), "f16")
    for b, n in ((0, 100), (2, 77)):
        kk, vv = (np.stack([ref.stands_for(x[b, h, :n]) for h in range(8)]) for x in (k, v))
        want, bound = ref.attention(q[b], kk, vv, 128 ** -0.5)
        close(out[b], want, bound + ref.rounding(want, "f16"))
    assert not out[1].any()


def test_cache_of_many_sequences(wgf, dev):
    """More sequences than a launch takes counts by value, and taken back, appended to and attended to by counts."""
    g = seeded(22, 95)
    b, t = 301, 70
    lens = [int(n) for n in g.integers(0, t + 1, b)]
    k, v = draw(g, (b, 1, t, 8), "f16", 2.0), draw(g, (b, 1, t, 8), "f16", 2.0)
    c = dev.kv_cache(b, 1, 8, t + 9, wgf.F16)
    tk, tv = give(wgf, dev, k, "f16"), give(wgf, dev, v, "f16")
    c.append(tk, tv, counts=lens)
    back = [max(n - int(d), 0) for n, d in zip(lens, g.integers(0, 3, b))]
    c.truncate(back)
    more = [int(n) for n in g.integers(0, 5, b)]
    nk, nv = draw(g, (b, 1, 4, 8), "f16", 2.0), draw(g, (b, 1, 4, 8), "f16", 2.0)
    c.append(give(wgf, dev, nk, "f16"), give(wgf, dev, nv, "f16"), counts=more)
    assert c.lengths == [n + m for n, m in zip(back, more)]
    both = [[np.concatenate([x[i, 0, :n], y[i, 0, :m]]) for i, (n, m) in enumerate(zip(back, more))] for x, y in ((k, nk), (v, nv))]
    for got, want in zip(c.read(), both):
        got = take(got, "f16")
        for i, x in enumerate(want):
            np.testing.assert_array_equal(got[i, 0, : len(x)], ref.round_to(ref.stands_for(x), "f16"))
            assert not got[i, 0, len(x):].any()
    q = draw(g, (b, 2, 4, 8), "f16")
    out = take(c.attention(give(wgf, dev, q, "f16"), counts=more), "f16")
    for i in range(b):
        want, bound = ref.attention(q[i], *(ref.stands_for(x[i])[None] for x in both), 8 ** -0.5, more[i])
        close(out[i], want, bound + ref.rounding(want, "f16"))


def test_cache_attention_of_very_many_jobs(wgf, dev):
    """More sequences times heads than there are tickets to join parts with."""
    g = seeded(22, 94)
    b, heads = 8300, 8
    lens = [int(n) for n in g.integers(0, 4, b)]
    lens[17], lens[b - 1] = 64, 61
    k, v, q = draw(g, (b, heads, 64, 8), "f16"), draw(g, (b, heads, 64, 8), "f16"), draw(g, (b, heads, 1, 8), "f16")
    c = dev.kv_cache(b, heads, 8, 64, wgf.F16)
    c.append(give(wgf, dev, k, "f16"), give(wgf, dev, v, "f16"), counts=lens)
    out = take(c.attention(give(wgf, dev, q, "f16")), "f16")
    for i in [17, b - 1, *(int(n) for n in g.integers(0, b, 100))]:
        kk, vv = (np.stack([ref.stands_for(x[i, h, : lens[i]]) for h in range(heads)]) for x in (k, v))
        want, bound = ref.attention(q[i], kk, vv, 8 ** -0.5)
        close(out[i], want, bound + ref.rounding(want, "f16"))


# ---- 4-bit weights --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (16, 64, 64), (33, 70, 32), (50, 300, 128), (17, 200, 64), (40, 129, 128)])
def test_q4_codes(kind, n, k, group, wgf, dev):
    g = seeded(23, n + k)
    w = draw(g, (n, k), kind, 0.02)
    w[0] = 0
    if n > 16:
        w[3] *= 0
        w[5, 0] = np.inf
    t = give(wgf, dev, w, kind).quantize_q4(group)
    c, s = ref.q4_quantize(np.where(np.isfinite(w), w, 0), group, kind)
    want = ref.q4_values(c, s, group).astype(np.float32)
    got = t.dequantize(wgf.F32).as_slice()
    if n > 16:
        assert np.isnan(got[5, :group]).all()
        got[5, :group] = want[5, :group]
    np.testing.assert_array_equal(got, want)
    other = "bf16" if kind == "f16" else "f16"
    got, want = ref.load(t.dequantize(code_of(wgf, other)).as_slice(), other), ref.round_to(want, other)
    if n > 16:
        got[5, :group] = want[5, :group]
    np.testing.assert_array_equal(got, want)
    # strided and transposed weights give the same codes
    if n == 33:
        np.testing.assert_array_equal(give(wgf, dev, w.T, kind).transpose(0, 1).quantize_q4(group).dequantize().as_slice(), t.dequantize().as_slice())


def test_q4_codes_of_far_sizes(wgf, dev):
    g = seeded(23, 5)
    for kind, sizes in (("f32", (1e38, 1e-36, 1e-40)), ("f16", (6e4, 3e-5, 2e-7)), ("bf16", (1e38, 1e-36))):
        for size in sizes:
            w = ref.round_to(g.uniform(-1, 1, (16, 64)) * size, kind)
            c, s = ref.q4_quantize(w, 32, kind)
            got = give(wgf, dev, w, kind).quantize_q4(32).dequantize().as_slice()
            np.testing.assert_array_equal(got, ref.q4_values(c, s, 32).astype(np.float32))


@pytest.mark.parametrize("scale_kind", KINDS)
@pytest.mark.parametrize("n,k,group", [(20, 77, 32), (5, 64, 64), (33, 301, 128)])
def test_q4_weights_from_codes(scale_kind, n, k, group, wgf, dev):
    g = seeded(23, 6)
    c = g.integers(0, 16, (n, k + (k & 1)))
    s = draw(g, (n, -(-k // group)), scale_kind, 0.01)
    t = dev.q4_weight((c[:, ::2] | c[:, 1::2] << 4).astype(np.uint8), ref.store(s, scale_kind), k, group, code_of(wgf, scale_kind))
    assert t.info == (n, k, group, code_of(wgf, scale_kind))
    values = ref.q4_values(c[:, :k] - 8, s, group)
    np.testing.assert_array_equal(t.dequantize().as_slice(), values.astype(np.float32))
    x = draw(g, (3, k), "f32")
    close(dev.tensor(x).mat_mul_q4(t).as_slice(), *ref.q4_product(x, values, "f32"))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 10, 11, 16, 17, 32, 33, 100])
@pytest.mark.parametrize("n,k,group", [(64, 256, 64), (33, 70, 32), (300, 1200, 128)])
def test_q4_product(kind, rows, n, k, group, wgf, dev):
    g = seeded(23, rows + k)
    w, x = draw(g, (n, k), kind, 0.02), draw(g, (rows, k), kind)
    c, s = ref.q4_quantize(w, group, kind)
    t = give(wgf, dev, w, kind).quantize_q4(group)
    out = take(give(wgf, dev, x, kind).mat_mul_q4(t), kind)
    # with many rows the weights are rounded to the type on the way, with few they are not: the wider bound holds for both
    close(out, *ref.q4_product(x, ref.q4_values(c, s, group), kind, through=None if rows <= 8 else kind))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n,k,group,way", [(700, 72, 64, 32, {}), (3001, 130, 70, 32, {}), (200, 40, 300, 128, {}), (65, 300, 1100, 64, {}),
                                                (600, 1500, 2100, 64, {"f32": "q4_tc", "f16": "q4_tc", "bf16": "q4_tc"}),
                                                (2300, 3400, 260, 64, {"f32": "q4_tc"})])
def test_q4_product_of_many_rows(kind, rows, n, k, group, way, wgf, dev):
    """Rows in blocks, on the tensor cores, and weights that are written out for the matrix product, in padded rows where k is odd for it."""
    g = seeded(23, rows)
    w, x = draw(g, (n, k), kind, 0.02), draw(g, (rows, k), kind)
    c, s = ref.q4_quantize(w, group, kind)
    t = give(wgf, dev, w, kind).quantize_q4(group)
    dev.set_timing(True)
    out = give(wgf, dev, x, kind).mat_mul_q4(t)
    # rounded on the way, but in blocks
    close(take(out, kind), *ref.q4_product(x, ref.q4_values(c, s, group), kind, through=kind))
    if kind in way:
        assert way[kind] in out.timing_labels()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("scale_kind", KINDS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", [(300, 1100, 1100), (257, 1030, 1091), (320, 2200, 1985), (1000, 260, 1024), (72, 9000, 2112)])
def test_q4_product_on_tensor_cores(kind, scale_kind, group, rows, n, k, wgf, dev):
    """Last tiles, steps and groups that are not full; scales of the rows' own type and of others."""
    g = seeded(29, rows + n + k + group)
    w, x = draw(g, (n, k), scale_kind, 0.02), draw(g, (rows, k), kind)
    c, s = ref.q4_quantize(w, group, scale_kind)
    t = give(wgf, dev, w, scale_kind).quantize_q4(group)
    dev.set_timing(True)
    out = give(wgf, dev, x, kind).mat_mul_q4(t)
    close(take(out, kind), *ref.q4_product(x, ref.q4_values(c, s, group), kind, through=kind))
    assert "q4_tc" in out.timing_labels()


@pytest.mark.parametrize("scale_kind", KINDS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", [(300, 1100, 1100), (257, 1030, 1091), (161, 2200, 1985), (97, 4000, 2113)])
def test_q4_product_of_f32_on_tensor_cores(scale_kind, group, rows, n, k, wgf, dev):
    """Rows of f32 keep their digits: codes and parts are exact, and only sums round."""
    g = seeded(30, rows + n + k + group)
    w, x = draw(g, (n, k), scale_kind, 0.02), draw(g, (rows, k + 1), "f32")
    x[5] *= 1e30
    x[6] *= 1e-25
    c, s = ref.q4_quantize(w, group, scale_kind)
    t = give(wgf, dev, w, scale_kind).quantize_q4(group)
    dev.set_timing(True)
    out = give(wgf, dev, x, "f32").slice([(0, rows), (1, k + 1)]).mat_mul_q4(t)
    got = out.as_slice()
    assert "q4_tc" in out.timing_labels()
    close(got, *ref.q4_product(x[:, 1:], ref.q4_values(c, s, group), "f32"))


def test_q4_product_on_tensor_cores_of_bad_values_and_views(wgf, dev):
    g = seeded(29, 1)
    rows, n, k = 300, 1100, 1091
    w, x = draw(g, (n, k), "f16", 0.02), draw(g, (rows, k + 5), "f16")
    w[7, 1090] = np.inf                     # the last group of one row has no scale
    t = give(wgf, dev, w, "f16").quantize_q4(64)
    x[3, 5], x[4, 6] = np.nan, np.inf
    dev.set_timing(True)
    whole = give(wgf, dev, x, "f16")
    out = whole.slice([(0, rows), (5, k + 5)]).mat_mul_q4(t)
    got = np.asarray(take(out, "f16"))
    assert "q4_tc" in out.timing_labels()
    assert np.isnan(got[:, 7]).all() and np.isnan(got[3]).all()
    keep_rows, keep = [r for r in range(rows) if r not in (3, 4)], [c for c in range(n) if c != 7]
    assert not np.isfinite(got[4][keep]).any()
    w[7] = 0
    c, s = ref.q4_quantize(w, 64, "f16")
    want, bound = ref.q4_product(x[keep_rows][:, 5:], ref.q4_values(c, s, 64), "f16", through="f16")
    close(got[keep_rows][:, keep], want[:, keep], bound[:, keep])
    # behind the last column stands what is not the product's: rows of a wider tensor
    x[3, 5] = x[4, 6] = 0
    x[:, :5] = np.nan
    back = give(wgf, dev, np.concatenate([x[:, 5:], x[:, :5]], 1), "f16").slice([(0, rows), (0, k)]).mat_mul_q4(t)
    assert np.isfinite(np.asarray(take(back, "f16"))[:, keep]).all()


@pytest.mark.parametrize("kind,rows,n,k", [("f16", 500, 11000, 3000), ("bf16", 33, 2000, 8200)])
def test_q4_product_on_tensor_cores_in_shares(kind, rows, n, k, wgf, dev):
    """Whole tiles, and behind them tiles whose columns are dealt out; the same bits each time, whoever is last."""
    g = seeded(29, 3)
    w, x = draw(g, (n, k), kind, 0.02), draw(g, (rows, k), kind)
    c, s = ref.q4_quantize(w, 64, kind)
    t, a = give(wgf, dev, w, kind).quantize_q4(64), give(wgf, dev, x, kind)
    dev.set_timing(True)
    out = a.mat_mul_q4(t)
    got = take(out, kind)
    assert "q4_tc" in out.timing_labels()
    close(got, *ref.q4_product(x, ref.q4_values(c, s, 64), kind, through=kind))
    for _ in range(10):
        np.testing.assert_array_equal(take(a.mat_mul_q4(t), kind), got)


@pytest.mark.parametrize("kind", KINDS)
def test_q4_product_of_very_long_rows(kind, wgf, dev):
    """A row of x is more than the shared memory of eight SMs."""
    g = seeded(29, 4)
    rows, n, k = 3, 20, 700_040
    w, x = draw(g, (n, k), kind, 0.02), draw(g, (rows, k), kind)
    c, s = ref.q4_quantize(w, 128, kind)
    out = give(wgf, dev, x, kind).mat_mul_q4(give(wgf, dev, w, kind).quantize_q4(128))
    close(take(out, kind), *ref.q4_product(x, ref.q4_values(c, s, 128), kind, through=kind))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_q4_product_on_tensor_cores_replayed(kind, wgf, dev):
    g = seeded(29, 2)
    rows, n, k = 300, 1100, 1100
    w, x = draw(g, (n, k), "bf16", 0.02), draw(g, (rows, k), kind)
    t, a = give(wgf, dev, w, kind).quantize_q4(64), give(wgf, dev, x, kind)
    want = take(a.mat_mul_q4(t), kind)
    with dev.record() as s:
        out = a.mat_mul_q4(t).materialize()
    for _ in range(3):
        s.launch()
    np.testing.assert_array_equal(take(out, kind), want)
    other = draw(g, (rows, k), kind)
    a.write(ref.store(other, kind))
    s.launch()
    want = take(give(wgf, dev, other, kind).mat_mul_q4(t), kind)
    np.testing.assert_array_equal(take(out, kind), want)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_q4_product_of_views_and_ranks(kind, wgf, dev):
    g = seeded(23, 77)
    w = draw(g, (40, 128), kind, 0.02)
    c, s = ref.q4_quantize(w, 64, kind)
    values, t = ref.q4_values(c, s, 64), give(wgf, dev, w, kind).quantize_q4(64)
    x = draw(g, (2, 3, 5, 129), kind)
    want, bound = ref.q4_product(x[..., 1:], values, kind)
    close(take(give(wgf, dev, x, kind).slice([(0, 2), (0, 3), (0, 5), (1, 129)]).mat_mul_q4(t), kind), want, bound)
    want, bound = ref.q4_product(x[0, 0, :, 1:], values, kind)
    close(take(give(wgf, dev, x[0, 0, :, 1:].T, kind).transpose(0, 1).mat_mul_q4(t), kind), want, bound)
    close(take(give(wgf, dev, x[0, 0, 2, 1:], kind).mat_mul_q4(t), kind), want[2], bound[2])
    row = give(wgf, dev, x[0, 0, 2:3, 1:], kind).broadcast_axis(0, 4)
    close(take(row.mat_mul_q4(t), kind), np.repeat(want[None, 2:3], 4, 0), np.repeat(bound[None, 2:3], 4, 0))


def test_q4_product_keeps_bad_values_where_they_are(wgf, dev):
    g = seeded(23, 78)
    w, x = draw(g, (40, 128), "f32", 0.02), draw(g, (4, 128), "f32")
    t = dev.tensor(w).quantize_q4(64)
    good = dev.tensor(x).mat_mul_q4(t).as_slice()
    x[1, 3], x[2, 100] = np.nan, np.inf
    out = dev.tensor(x).mat_mul_q4(t).as_slice()
    np.testing.assert_array_equal(out[[0, 3]], good[[0, 3]])
    assert np.isnan(out[1]).all() and not np.isfinite(out[2]).any()
    x[2] = np.float32(3e38) * np.sign(x[2])          # finite, near the end of the range
    x[1] = 0
    w = np.zeros((40, 128), np.float32)
    w[:, 0] = 2.0 ** -20
    out = dev.tensor(x).mat_mul_q4(dev.tensor(w).quantize_q4(64)).as_slice()
    assert np.isfinite(out).all() and not out[1].any()


def test_q4_product_at_full_size(wgf, dev):
    """The gate projection of the decoder block's configuration, every output checked through float64 on the host."""
    g = seeded(23, 79)
    n, k = 11008, 4096
    w, x = draw(g, (n, k), "f16", 0.02), draw(g, (5, k), "f16")
    c, s = ref.q4_quantize(w, 128, "f16")
    t = give(wgf, dev, w, "f16").quantize_q4(128)
    want, bound = ref.q4_product(x, ref.q4_values(c, s, 128), "f16")
    for rows in (1, 5):
        close(take(give(wgf, dev, x[:rows], "f16").mat_mul_q4(t), "f16"), want[:rows], bound[:rows])


# ---- together -------------------------------------------------------------------------------------------------------------
class Layer:
    """One attention layer as it decodes: 4-bit projections, norm and rotation into the cache, attention, 4-bit projection."""

    def __init__(self, wgf, dev, g, kind, batch, hidden, heads, kv_heads, dim, room, group=64):
        self.wgf, self.dev, self.kind, self.group = wgf, dev, kind, group
        self.batch, self.heads, self.kv_heads, self.dim = batch, heads, kv_heads, dim
        self.w = {n: draw(g, s, kind, 0.05) for n, s in (("q", (heads * dim, hidden)), ("k", (kv_heads * dim, hidden)),
                                                        ("v", (kv_heads * dim, hidden)), ("o", (hidden, heads * dim)))}
        self.q4 = {n: give(wgf, dev, w, kind).quantize_q4(group) for n, w in self.w.items()}
        self.norms = [draw(g, (dim,), kind, 0.1, 1.0) for _ in range(2)]
        self.angles = tables(room, dim, kind)
        self.small = [give(wgf, dev, x, kind) for x in (*self.norms, *self.angles)]
        self.cache = dev.kv_cache(batch, kv_heads, dim, room, code_of(wgf, kind))

    def split(self, t, heads):
        return t.reshape((self.batch, t.shape[0] // self.batch, heads, self.dim)).transpose(1, 2)

    def step(self, x, fused=True, counts=None, at=0):
        """x [batch * t, hidden]"""
        q, k, v = (self.split(x.mat_mul_q4(self.q4[n]), h) for n, h in (("q", self.heads), ("k", self.kv_heads), ("v", self.kv_heads)))
        if fused:
            q = self.cache.append_qk(q, k, v, *self.small, eps=1e-5, counts=counts)
        else:
            q, k = q.qk_norm_rope(k, *self.small, eps=1e-5, start=at)
            self.cache.append(k, v)
        o = self.cache.attention(q, counts=counts)
        return o.transpose(1, 2).reshape((x.shape[0], self.heads * self.dim)).mat_mul_q4(self.q4["o"])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 2), (80, 3, 1), (128, 8, 1)])
def test_fused_append_is_the_operators_one_by_one(kind, dim, heads, kv_heads, wgf, dev):
    """Norm, rotation and append in one launch have the bits of the separate calls, for prompts and single tokens."""
    g = seeded(24, dim)
    layers = [Layer(wgf, dev, seeded(24, 1), kind, 2, 128, heads, kv_heads, dim, 300) for _ in range(2)]
    at = 0
    for t in (1, 70, 1, 129, 1, 20):
        x = give(wgf, dev, draw(g, (2 * t, 128), kind), kind)
        a, b = layers[0].step(x, fused=True).as_slice(), layers[1].step(x, fused=False, at=at).as_slice()
        np.testing.assert_array_equal(a, b)
        at += t
    for a, b in zip(layers[0].cache.read(), layers[1].cache.read()):
        np.testing.assert_array_equal(a.as_slice(), b.as_slice())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [8, 24, 72, 200, 248])
def test_fused_append_of_uneven_heads(kind, dim, wgf, dev):
    """Heads whose halves take no whole vector of the type, and operands that stand at odd places."""
    g = seeded(24, dim + 1)
    q, k, v = (draw(g, (2, h, 67, dim + 1), kind) for h in (3, 1, 1))
    w, (cos, sin) = draw(g, (dim,), kind, 0.2, 1.0), tables(100, dim, kind)
    tw, tc, ts = (give(wgf, dev, x, kind) for x in (w, cos, sin))
    tq, tk, tv = (give(wgf, dev, x, kind).slice([(0, 2), (0, x.shape[1]), (0, 67), (1, dim + 1)]) for x in (q, k, v))
    one, two = (dev.kv_cache(2, 1, dim, 100, code_of(wgf, kind)) for _ in range(2))
    for c in (one, two):
        c.append(tv.slice([(0, 2), (0, 1), (0, 5), (0, dim)]), tv.slice([(0, 2), (0, 1), (0, 5), (0, dim)]))
    a = one.append_qk(tq, tk, tv, tw, tw, tc, ts, eps=1e-5)
    b, kk = tq.qk_norm_rope(tk, tw, tw, tc, ts, eps=1e-5, start=5)
    two.append(kk, tv)
    np.testing.assert_array_equal(a.as_slice(), b.as_slice())
    for x, y in zip(one.read(), two.read()):
        np.testing.assert_array_equal(x.as_slice(), y.as_slice())
    want, off = ref.norm_rope(q[..., 1:].reshape(6, 67, dim), w, cos, sin, 1e-5, 5 + np.arange(67))
    close(take(a, kind).reshape(6, 67, dim), want, off * 1.01 + ref.rounding(want, kind) * 1.01)


def test_fused_append_of_a_padded_batch(wgf, dev):
    """Sequences of different lengths stand at their own positions; padding rows are not read and come back as zeros."""
    g = seeded(24, 500)
    kind, d = "f32", 64
    lens, counts = [70, 3, 0], [5, 9, 0]
    layer = Layer(wgf, dev, g, kind, 3, 64, 4, 2, d, 200)
    wq, wk, (cos, sin) = *layer.norms, layer.angles
    old = draw(g, (3, 2, 70, d), kind)
    layer.cache.append(dev.tensor(old), dev.tensor(old), counts=lens)
    q, k, v = draw(g, (3, 4, 9, d), kind), draw(g, (3, 2, 9, d), kind), draw(g, (3, 2, 9, d), kind)
    for b, n in enumerate(counts):
        q[b, :, n:], k[b, :, n:], v[b, :, n:] = np.nan, np.inf, np.nan
    out = layer.cache.append_qk(*(dev.tensor(x) for x in (q, k, v)), *layer.small, eps=1e-5, counts=counts)
    got = out.as_slice()
    assert layer.cache.lengths == [75, 12, 0]
    rk, rv = (t.as_slice() for t in layer.cache.read())
    for b, n in enumerate(counts):
        pos = lens[b] + np.arange(n)
        want, off = ref.norm_rope(q[b, :, :n], wq, cos, sin, 1e-5, pos)
        close(got[b, :, :n], want, off * 1.01 + ref.rounding(want, kind) * 1.01)
        assert not got[b, :, n:].any()
        kk, off = ref.norm_rope(k[b, :, :n], wk, cos, sin, 1e-5, pos)
        for h in range(2):
            m = lens[b] + n
            full = np.concatenate([old[b, h, : lens[b]], kk[h]])
            top = np.array([np.abs(full[i: i + 64]).max() for i in range(0, m, 64)]).repeat(64)[:m, None]
            # half a code's step, and what the norm and rotation may be off
            assert (np.abs(rk[b, h, :m] - full) <= top / 127 * 0.5001 + 2 * top * (d / 2 + 8) * ref.U).all()
            np.testing.assert_array_equal(rv[b, h, :m], ref.stands_for(np.concatenate([old[b, h, : lens[b]], v[b, h, :n]])))
    att = layer.cache.attention(out, counts=counts).as_slice()
    assert np.isfinite(att).all() and not att[2].any()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_layer_decodes_recorded_as_it_does_eagerly(kind, wgf, dev):
    """A prompt, then tokens one by one: by calls, and by one recorded step launched again and again; the same bits, and
    drafts that are taken back leave no trace."""
    g = seeded(24, 600)
    xs = [draw(g, (2 * 50, 128), kind)] + [draw(g, (2, 128), kind) for _ in range(100)]
    eager, replay = (Layer(wgf, dev, seeded(24, 3), kind, 2, 128, 8, 2, 64, 160) for _ in range(2))
    for layer in (eager, replay):
        layer.step(give(wgf, dev, xs[0], kind)).materialize()
    want = [eager.step(give(wgf, dev, x, kind)).as_slice() for x in xs[1:]]
    x = give(wgf, dev, xs[1], kind)
    with dev.record() as s:
        out = replay.step(x).materialize()
    np.testing.assert_array_equal(out.as_slice(), want[0])
    for i, v in enumerate(xs[2:]):
        if i % 9 == 3:                       # a draft that is not accepted
            x.write(ref.store(xs[1], kind))
            s.launch()
            replay.cache.truncate([n - 1 for n in replay.cache.lengths])
        x.write(ref.store(v, kind))
        s.launch()
        np.testing.assert_array_equal(out.as_slice(), want[i + 1])
    assert replay.cache.lengths == eager.cache.lengths == [150, 150]


def test_two_recordings_and_calls_take_turns(wgf, dev):
    """Two schedules over two caches, and calls between them: tickets and scratch of one leave the other's results alone."""
    g = seeded(24, 700)
    k, v, q = draw(g, (1, 1, 3000, 128), "f16"), draw(g, (1, 1, 3000, 128), "f16"), draw(g, (1, 8, 1, 128), "f16")
    tk, tv, tq = (dev.tensor(ref.store(x, "f16")) for x in (k, v, q))
    caches, outs, schedules = [], [], []
    for n in (3000, 1700):
        c = dev.kv_cache(1, 1, 128, 3000, wgf.F16)
        c.append(tk, tv, counts=[n])
        want = c.attention(tq).as_slice()
        with dev.record() as s:
            out = c.attention(tq)
        caches.append(c), outs.append((out, want)), schedules.append(s)
    for _ in range(5):
        for i in (0, 1, 1, 0):
            schedules[i].launch()
            # the split of a recording is its own, so its last bits may be others than a call's; its own are the same each time
            got = outs[i][0].as_slice()
            kk, vv = (ref.stands_for(x[0, 0, : caches[i].lengths[0]])[None] for x in (k, v))
            wanted, bound = ref.attention(q[0], kk, vv, 128 ** -0.5)
            close(ref.load(got, "f16")[0], wanted, bound + ref.rounding(wanted, "f16"))
            np.testing.assert_array_equal(caches[i].attention(tq).as_slice(), outs[i][1])


def test_a_schedule_keeps_its_cache(wgf, dev):
    """The handle goes away before the schedule does."""
    g = seeded(24, 800)
    k, q = draw(g, (1, 2, 100, 64), "f16"), draw(g, (1, 2, 1, 64), "f16")
    tk, tq = dev.tensor(ref.store(k, "f16")), dev.tensor(ref.store(q, "f16"))
    c = dev.kv_cache(1, 2, 64, 200, wgf.F16)
    c.append(tk, tk)
    with dev.record() as s:
        out = c.attention(tq)
    want = out.as_slice()
    del c
    fill = [dev.kv_cache(1, 2, 64, 200, wgf.F16) for _ in range(4)]
    for f in fill:
        f.append(tk * 3.0, tk * 2.0)
    s.launch()
    np.testing.assert_array_equal(out.as_slice(), want)


def test_kernel_times_of_calls_that_run_at_once(wgf, dev):
    c = dev.kv_cache(1, 1, 64, 64, wgf.F16)
    k = dev.tensor(np.ones((1, 1, 3, 64), np.float16))
    dev.set_timing(True)
    c.append(k, k)
    out = c.attention(k)
    assert out.timing_labels() == ["cache_attention"] and len(out.all_timing_information()) == 1


# ---- many rows through 4-bit weights: what is rounded -----------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("scale_kind", KINDS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", [(300, 1100, 1100), (257, 1030, 1091), (72, 9000, 2112), (500, 2200, 1985), (1000, 260, 1024), (130, 3000, 64),
                                      (33, 4100, 40)])
def test_q4_product_of_many_rows_rounds_sums_alone(kind, scale_kind, group, rows, n, k, wgf, dev):
    """The weights' values are not rounded to the type of x on the way: the bound is that of f32 sums of exact products."""
    g = seeded(31, rows + n + k + group)
    w, x = draw(g, (n, k), scale_kind, 0.02), draw(g, (rows, k), kind)
    c, s = ref.q4_quantize(w, group, scale_kind)
    out = take(give(wgf, dev, x, kind).mat_mul_q4(give(wgf, dev, w, scale_kind).quantize_q4(group)), kind)
    close(out, *ref.q4_product(x, ref.q4_values(c, s, group), kind))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(2304, 2304, 2051), (2304, 2304, 2048), (4500, 1280, 1030)])
def test_q4_product_of_very_many_rows_rounds_sums_alone(kind, rows, n, k, wgf, dev):
    g = seeded(31, rows + k)
    w, x = draw(g, (n, k), kind, 0.02), draw(g, (rows, k), kind)
    c, s = ref.q4_quantize(w, 128, kind)
    dev.set_timing(True)
    out = give(wgf, dev, x, kind).mat_mul_q4(give(wgf, dev, w, kind).quantize_q4(128))
    close(take(out, kind), *ref.q4_product(x, ref.q4_values(c, s, 128), kind))
    assert "q4_tc" in out.timing_labels() and "q4_dequantize" not in out.timing_labels()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [9, 17, 33, 100])
@pytest.mark.parametrize("n,k,group", [(64, 256, 64), (33, 70, 32), (300, 1200, 128)])
def test_q4_product_in_blocks_rounds_sums_alone(kind, rows, n, k, group, wgf, dev):
    g = seeded(31, rows + k)
    w, x = draw(g, (n, k), kind, 0.02), draw(g, (rows, k), kind)
    c, s = ref.q4_quantize(w, group, kind)
    dev.set_timing(True)
    out = give(wgf, dev, x, kind).mat_mul_q4(give(wgf, dev, w, kind).quantize_q4(group))
    close(take(out, kind), *ref.q4_product(x, ref.q4_values(c, s, group), kind))
    assert "q4_rows" in out.timing_labels()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_q4_product_of_very_long_rows_rounds_sums_alone(kind, wgf, dev):
    g = seeded(31, 4)
    rows, n, k = 3, 20, 700_040
    w, x = draw(g, (n, k), kind, 0.02), draw(g, (rows, k), kind)
    c, s = ref.q4_quantize(w, 128, kind)
    out = give(wgf, dev, x, kind).mat_mul_q4(give(wgf, dev, w, kind).quantize_q4(128))
    close(take(out, kind), *ref.q4_product(x, ref.q4_values(c, s, 128), kind))


@pytest.mark.parametrize("kind,rows", [("bf16", 300), ("f32", 161), ("f16", 300)])
def test_q4_product_on_tensor_cores_at_the_ends_of_the_range(kind, rows, wgf, dev):
    """Rows near the type's largest number, whose sums of a group are finite where the result is."""
    g = seeded(31, 5)
    n, k = 1100, 1100
    top = {"f32": 3e38, "bf16": 3e38, "f16": 6e4}[kind]
    x = ref.round_to(g.uniform(-1, 1, (rows, k)) * top, kind)
    c = g.integers(0, 16, (n, k))
    s = np.full((n, -(-k // 64)), 2.0 ** -20, np.float32)
    t = dev.q4_weight((c[:, ::2] | c[:, 1::2] << 4).astype(np.uint8), s, k, 64, wgf.F32)
    dev.set_timing(True)
    out = give(wgf, dev, x, kind).mat_mul_q4(t)
    close(take(out, kind), *ref.q4_product(x, ref.q4_values(c - 8, s, 64), kind))
    assert "q4_tc" in out.timing_labels()


# ---- few rows through 4-bit weights: the codes less 8 enter exactly -----------------------------------------------------------
def from_codes(wgf, dev, c, s, group):
    """Weights of codes -8 .. 7 [n, k], k even, and f32 scales."""
    return dev.q4_weight(((c + 8)[:, ::2] | (c + 8)[:, 1::2] << 4).astype(np.uint8), s, c.shape[1], group, wgf.F32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n,k,group", [(1, 40, 256, 64), (3, 40, 256, 32), (9, 40, 256, 128), (300, 1100, 1100, 64)])
def test_q4_product_of_an_infinity_is_one(kind, rows, n, k, group, wgf, dev):
    """An infinite x gives an infinity of the sign that its code has, and NaN only where the code is 8, which stands for zero."""
    g = seeded(32, rows + k)
    c = g.integers(-8, 8, (n, k))
    x = draw(g, (rows, k), kind)
    x[rows - 1, 70], x[0, 3] = np.inf, -np.inf
    s = np.full((n, -(-k // group)), 0.01, np.float32)
    out = take(give(wgf, dev, x, kind).mat_mul_q4(from_codes(wgf, dev, c, s, group)), kind)
    with np.errstate(invalid="ignore"):
        infinite = np.where(np.isinf(x), x, 0.0)[:, None, :] * c[None].astype(np.float32)        # 0 * inf is NaN, as it has to be
        infinite = np.where(np.isinf(x)[:, None, :], infinite, 0.0).sum(-1)
    np.testing.assert_array_equal(np.isnan(out), np.isnan(infinite))
    np.testing.assert_array_equal(out[np.isinf(infinite)], infinite[np.isinf(infinite)])
    assert np.isfinite(out[infinite == 0]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n,k,group", [(1, 40, 256, 64), (2, 33, 512, 32), (7, 100, 256, 128), (12, 40, 256, 64), (300, 1100, 1100, 128)])
def test_q4_product_of_columns_without_weight(kind, rows, n, k, group, wgf, dev):
    """Large x in columns whose weights are zero cost the others no digits; a weight that is all zero gives zero itself."""
    g = seeded(32, rows + n)
    c = g.integers(-8, 8, (n, k))
    x = draw(g, (rows, k), kind)
    for col in range(0, k, 9):
        c[:, col] = 0
        x[:, col] = 6e4 if col % 2 else -5e4
    x = ref.round_to(x, kind)
    c[5] = 0
    s = np.full((n, -(-k // group)), 0.01, np.float32)
    out = take(give(wgf, dev, x, kind).mat_mul_q4(from_codes(wgf, dev, c, s, group)), kind)
    close(out, *ref.q4_product(x, ref.q4_values(c, s, group), kind))
    assert not out[:, 5].any()


# ---- attention: small probabilities beside a dominant one ---------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gap", [5.0, 11.0, 14.0, 17.5])
@pytest.mark.parametrize("lengths,spread", [([900], 0.0), ([8001, 2000], 0.0), ([8001], 1.0), ([60000], 0.0)])
def test_cache_attention_behind_a_dominant_key(kind, gap, lengths, spread, wgf, dev):
    """The first key takes nearly all of the weight and its value is zero: the result is what the others' small weights bring."""
    g = seeded(33, int(gap) + lengths[0])
    b, n, d = len(lengths), max(lengths), 64
    k = np.zeros((b, 1, n, d), np.float32)
    k[..., 0] = g.standard_normal((b, 1, n)) * spread
    k[:, :, 0, 0] = gap
    v = g.standard_normal((b, 1, n, d)) + 1.0
    v[:, :, 0] = 0
    q = np.zeros((b, 2, 1, d), np.float32)
    q[..., 0] = [[[1.0], [0.75]]]
    k, v = ref.round_to(k, kind), ref.round_to(v, kind)
    c = dev.kv_cache(b, 1, d, n, code_of(wgf, kind))
    c.append(give(wgf, dev, k, kind), give(wgf, dev, v, kind), counts=lengths)
    out = take(c.attention(give(wgf, dev, q, kind), scale=1.0), kind)
    for i, m in enumerate(lengths):
        want, bound = ref.attention(q[i], ref.stands_for(k[i, 0, :m])[None], ref.stands_for(v[i, 0, :m])[None], 1.0)
        close(out[i], want, bound + ref.rounding(want, kind))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [0, 7])
def test_fused_append_of_padding_alone_gives_zeros(kind, rows, wgf, dev):
    c = dev.kv_cache(2, 1, 64, 20, code_of(wgf, kind))
    bad = give(wgf, dev, np.full((2, 1, 3, 64), np.nan, np.float32), kind)
    q = give(wgf, dev, np.full((2, 4, 3, 64), np.nan, np.float32), kind)
    w, t = give(wgf, dev, np.ones(64, np.float32), kind), give(wgf, dev, np.ones((rows, 32), np.float32), kind)
    for _ in range(2):
        assert not take(c.append_qk(q, bad, bad, w, w, t, t, counts=[0, 0]), kind).any()
    assert c.lengths == [0, 0] and c.read()[0].shape == (2, 1, 0, 64)


def test_a_recording_that_is_broken_off_keeps_host_and_device_together(wgf, dev):
    g = seeded(34, 1)
    k, v, q = draw(g, (1, 2, 9, 64), "f16", 2.0), draw(g, (1, 2, 9, 64), "f16"), draw(g, (1, 2, 1, 64), "f16")
    t = lambda x, a, b: dev.tensor(ref.store(x[:, :, a:b], "f16"))
    c, plain = (dev.kv_cache(1, 2, 64, 12, wgf.F16) for _ in range(2))
    parts = [(t(k, a, b), t(v, a, b)) for a, b in ((0, 3), (3, 4), (4, 9))]
    tq = dev.tensor(ref.store(q, "f16"))
    c.append(*parts[0])
    with pytest.raises(wgf.WgfError):
        with dev.record():
            c.append(*parts[1])
            c.attention(tq, counts=[1])          # fixed numbers: refused
    assert c.lengths == [4]
    c.append(*parts[2])
    plain.append(t(k, 0, 9), t(v, 0, 9))
    assert c.lengths == plain.lengths == [9]
    for a, b in zip(contents(c, tq, "f16"), contents(plain, tq, "f16")):
        np.testing.assert_array_equal(a, b)


def test_a_schedule_may_go_while_another_is_recorded(wgf, dev):
    """The name of the last schedule is bound anew inside the next one's block, so that the old one is destroyed while the new one is recorded."""
    g = seeded(34, 2)
    k, q = draw(g, (1, 1, 200, 64), "f16"), draw(g, (1, 2, 1, 64), "f16")
    c = dev.kv_cache(1, 1, 64, 200, wgf.F16)
    tk, tq = dev.tensor(ref.store(k, "f16")), dev.tensor(ref.store(q, "f16"))
    c.append(tk, tk)
    want = c.attention(tq).as_slice()
    for _ in range(3):
        with dev.record() as s:
            out = c.attention(tq) * 2.0
            out.materialize()
        for _ in range(2):
            s.launch()
        np.testing.assert_array_equal(ref.load(out.as_slice(), "f16"), ref.load(want, "f16") * 2)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sign", [1, -1])
def test_cache_of_the_largest_numbers_is_finite(kind, sign, wgf, dev):
    """A token of the type's largest (or lowest) number does not come back as an infinity."""
    top = {"f32": float(np.finfo(np.float32).max), "f16": 65504.0, "bf16": float.fromhex("0x1.fep+127")}[kind]
    g = seeded(35, 1)
    x = draw(g, (1, 1, 70, 64), kind)
    x[0, 0, 3], x[0, 0, 66, 5] = sign * top, top
    c = dev.kv_cache(1, 1, 64, 70, code_of(wgf, kind))
    c.append(give(wgf, dev, x, kind), give(wgf, dev, -x, kind))
    for got, want in zip(c.read(), (x, -x)):
        got = take(got, kind)
        assert np.isfinite(got).all()
        np.testing.assert_array_equal(got, ref.round_to(kept(want, [70]), kind))
    # the only key that a query sees: its value
    one = dev.kv_cache(1, 1, 64, 70, code_of(wgf, kind))
    one.append(give(wgf, dev, x[:, :, 3:4] * 0, kind), give(wgf, dev, x[:, :, 3:4], kind))
    out = take(one.attention(give(wgf, dev, x[:, :, :1], kind)), kind)
    np.testing.assert_array_equal(out[0, 0, 0], ref.round_to(ref.stands_for(x[0, 0, 3:4]), kind)[0])


@pytest.mark.parametrize("kind,exponent", [("f32", -107), ("bf16", -120), ("f16", -18), ("f32", 90), ("bf16", 90)])
@pytest.mark.parametrize("rows,n,k", [(3, 40, 256), (300, 1100, 1100)])
def test_q4_product_of_far_sizes_of_x(kind, exponent, rows, n, k, wgf, dev):
    """Small and large rows keep the bound that ordinary ones have, with scales that bring the result back."""
    g = seeded(32, rows - exponent)
    c = g.integers(-8, 8, (n, k))
    s = np.full((n, -(-k // 64)), 2.0 ** (20 if exponent < 0 else -40), np.float32)
    x = ref.round_to(g.standard_normal((rows, k)) * 2.0 ** exponent, kind)
    out = take(give(wgf, dev, x, kind).mat_mul_q4(from_codes(wgf, dev, c, s, 64)), kind)
    want, bound = ref.q4_product(x, ref.q4_values(c, s, 64), kind)
    # denormal numbers: f16 has steps of 2^-24 there, which are exact; of an f32 value half a step of its third part, 2^-134, may be missing
    lost = 2.0 ** -134 * np.abs(ref.q4_values(c, s, 64)).sum(1)[None] if kind == "f32" else 0.0
    close(out, want, bound + lost)
