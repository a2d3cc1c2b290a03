"""The decode operators' host side on the compile-only device: what they refuse, what a refusal leaves, and how a cache's
lengths move with appends, truncations and recorded schedules.  Nothing is executed."""
import numpy as np
import pytest

KINDS = ["F32", "F16", "BF16"]


def blank(wgf, dev, shape, kind="F16"):
    np_type = {"F32": np.float32, "F16": np.float16, "BF16": np.uint16}[kind]
    return dev.tensor(np.zeros(shape, np_type), dtype=getattr(wgf, kind))


def refused(wgf, status, call, *args, **kw):
    with pytest.raises(wgf.WgfError) as e:
        call(*args, **kw)
    assert e.value.status == status, e.value


# ---- cache ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad,status", [
    (dict(batch=0), "SHAPE"), (dict(kv_heads=0), "SHAPE"), (dict(capacity=0), "SHAPE"), (dict(batch=-1), "SHAPE"),
    (dict(head_dim=4), "UNSUPPORTED"), (dict(head_dim=100), "UNSUPPORTED"), (dict(head_dim=264), "UNSUPPORTED"),
    (dict(head_dim=0), "UNSUPPORTED"), (dict(capacity=1 << 40), "UNSUPPORTED"), (dict(batch=1 << 40), "UNSUPPORTED"),
    (dict(dtype=7), "DTYPE")])
def test_cache_shapes_that_are_refused(wgf, drydev, bad, status):
    args = dict(batch=2, kv_heads=2, head_dim=64, capacity=100, dtype=wgf.F16)
    refused(wgf, status, drydev.kv_cache, **{**args, **bad})


def test_cache_lengths_follow_appends_and_counts(wgf, drydev):
    c = drydev.kv_cache(3, 2, 64, 100, wgf.F16)
    k = blank(wgf, drydev, (3, 2, 10, 64))
    assert c.lengths == [0, 0, 0]
    c.append(k, k)
    c.append(k, k, counts=[0, 10, 3])
    assert c.lengths == [10, 20, 13]
    e = blank(wgf, drydev, (3, 2, 0, 64))
    c.append(e, e)
    assert c.lengths == [10, 20, 13]
    c.truncate([0, 20, 13])
    assert c.lengths == [0, 20, 13]


def test_append_that_does_not_fit_changes_nothing(wgf, drydev):
    c = drydev.kv_cache(2, 1, 64, 15, wgf.F16)
    k = blank(wgf, drydev, (2, 1, 10, 64))
    c.append(k, k, counts=[10, 5])
    before = drydev.launch_count
    refused(wgf, "INVALID_ARGUMENT", c.append, k, k)
    refused(wgf, "INVALID_ARGUMENT", c.append, k, k, counts=[6, 0])
    refused(wgf, "INVALID_ARGUMENT", c.append, k, k, counts=[5, 11])
    refused(wgf, "INVALID_ARGUMENT", c.append, k, k, counts=[5, -1])
    assert c.lengths == [10, 5] and drydev.launch_count == before
    c.append(k, k, counts=[5, 10])            # room for fewer than were given, as long as the counts say so
    assert c.lengths == [15, 15]
    with pytest.raises(ValueError):
        c.append(k, k, counts=[1])


def test_append_refuses_other_shapes_types_and_devices(wgf, drydev):
    c = drydev.kv_cache(2, 2, 64, 100, wgf.F16)
    good = blank(wgf, drydev, (2, 2, 3, 64))
    for shape, status in [((2, 2, 64), "RANK"), ((1, 2, 3, 64), "SHAPE"), ((2, 1, 3, 64), "SHAPE"), ((2, 2, 4, 64), "SHAPE"),
                          ((2, 2, 3, 32), "SHAPE")]:
        refused(wgf, status, c.append, good, blank(wgf, drydev, shape))
    refused(wgf, "SHAPE", c.append, blank(wgf, drydev, (2, 1, 3, 64)), blank(wgf, drydev, (2, 1, 3, 64)))
    refused(wgf, "DTYPE", c.append, good, blank(wgf, drydev, (2, 2, 3, 64), "BF16"))
    other = wgf.Device(-1)
    refused(wgf, "INVALID_ARGUMENT", c.append, blank(wgf, other, (2, 2, 3, 64)), good)
    assert c.lengths == [0, 0]


def test_append_qk_refuses_what_does_not_belong_together(wgf, drydev):
    c = drydev.kv_cache(2, 2, 64, 100, wgf.F16)
    q, k = blank(wgf, drydev, (2, 6, 3, 64)), blank(wgf, drydev, (2, 2, 3, 64))
    w, t = blank(wgf, drydev, (64,)), blank(wgf, drydev, (50, 32))
    ok = dict(q=q, k=k, v=k, q_weight=w, k_weight=w, cos=t, sin=t)
    for change, status in [(dict(q=blank(wgf, drydev, (2, 6, 2, 64))), "SHAPE"), (dict(q=blank(wgf, drydev, (1, 6, 3, 64))), "SHAPE"),
                           (dict(q=blank(wgf, drydev, (2, 6, 3, 64), "F32")), "DTYPE"), (dict(q_weight=blank(wgf, drydev, (32,))), "SHAPE"),
                           (dict(k_weight=blank(wgf, drydev, (64,), "F32")), "DTYPE"), (dict(cos=blank(wgf, drydev, (50, 64))), "SHAPE"),
                           (dict(sin=blank(wgf, drydev, (49, 32))), "SHAPE"), (dict(cos=blank(wgf, drydev, (2, 32)), sin=blank(wgf, drydev, (2, 32))), "SHAPE"),
                           (dict(sin=blank(wgf, drydev, (50, 32), "BF16")), "DTYPE")]:
        refused(wgf, status, c.append_qk, **{**ok, **change})
    assert c.lengths == [0, 0]
    for _ in range(16):
        assert c.append_qk(**ok).shape == (2, 6, 3, 64)
    refused(wgf, "SHAPE", c.append_qk, **ok)   # the tables end at position 50
    assert c.lengths == [48, 48]


def test_attention_refusals_and_shapes(wgf, drydev):
    c = drydev.kv_cache(2, 2, 64, 100, wgf.F16)
    assert c.attention(blank(wgf, drydev, (2, 8, 1, 64))).shape == (2, 8, 1, 64)
    assert c.attention(blank(wgf, drydev, (2, 8, 0, 64))).shape == (2, 8, 0, 64)
    for shape, status in [((2, 8, 64), "RANK"), ((1, 8, 1, 64), "SHAPE"), ((2, 3, 1, 64), "SHAPE"), ((2, 8, 1, 32), "SHAPE")]:
        refused(wgf, status, c.attention, blank(wgf, drydev, shape))
    refused(wgf, "DTYPE", c.attention, blank(wgf, drydev, (2, 8, 1, 64), "F32"))
    refused(wgf, "INVALID_ARGUMENT", c.attention, blank(wgf, drydev, (2, 8, 1, 64)), counts=[2, 0])


def test_truncate_keeps_to_what_the_cache_still_has(wgf, drydev):
    c = drydev.kv_cache(2, 1, 64, 1000, wgf.F16)
    k = blank(wgf, drydev, (2, 1, 500, 64))
    c.append(k, k, counts=[500, 300])
    refused(wgf, "INVALID_ARGUMENT", c.truncate, [501, 300])
    refused(wgf, "INVALID_ARGUMENT", c.truncate, [-1, 300])
    # 500 is in block 7: blocks 6 and 7 are held, so 384 and on; 300 is in block 4, so 192 and on
    refused(wgf, "UNSUPPORTED", c.truncate, [383, 300])
    refused(wgf, "UNSUPPORTED", c.truncate, [500, 191])
    assert c.lengths == [500, 300]
    c.truncate([385, 193])
    c.truncate([385, 128])                    # a multiple of 64 needs no tokens
    refused(wgf, "UNSUPPORTED", c.truncate, [383, 128])
    refused(wgf, "UNSUPPORTED", c.truncate, [385, 127])
    one = blank(wgf, drydev, (2, 1, 1, 64))
    c.append(one, one)
    c.truncate([385, 128])
    refused(wgf, "UNSUPPORTED", c.truncate, [385, 100])
    c.truncate([0, 0])
    assert c.lengths == [0, 0]


def test_recorded_appends_move_the_lengths_and_stop_at_the_capacity(wgf, drydev):
    c = drydev.kv_cache(2, 1, 64, 20, wgf.F16)
    k, q = blank(wgf, drydev, (2, 1, 3, 64)), blank(wgf, drydev, (2, 4, 3, 64))
    c.append(k, k, counts=[1, 2])
    with drydev.record() as s:
        c.append(k, k)
        c.attention(q)
        c.append(k, k)
        assert c.lengths == [1, 2]            # nothing has run yet
    assert c.lengths == [7, 8]                # the end of a recording launches it once
    s.launch()
    assert c.lengths == [13, 14]
    s.launch()
    assert c.lengths == [19, 20]
    before = drydev.launch_count
    refused(wgf, "INVALID_ARGUMENT", s.launch)
    assert c.lengths == [19, 20] and drydev.launch_count == before
    c.truncate([0, 0])
    s.launch()
    assert c.lengths == [6, 6]


def test_what_a_recording_refuses(wgf, drydev):
    c = drydev.kv_cache(1, 1, 64, 8, wgf.F16)
    k, q = blank(wgf, drydev, (1, 1, 5, 64)), blank(wgf, drydev, (1, 1, 1, 64))
    w = blank(wgf, drydev, (64, 64))
    with drydev.record():
        refused(wgf, "UNSUPPORTED", c.truncate, [0])
        refused(wgf, "UNSUPPORTED", c.read)
        refused(wgf, "UNSUPPORTED", c.append, k, k, counts=[1])
        refused(wgf, "UNSUPPORTED", c.attention, q, counts=[1])
        refused(wgf, "UNSUPPORTED", drydev.kv_cache, 1, 1, 64, 8)
        refused(wgf, "UNSUPPORTED", w.quantize_q4, 64)
        c.append(k, k)
        refused(wgf, "INVALID_ARGUMENT", c.append, k, k)   # 5 and 5 of this recording are more than 8
    assert c.lengths == [5]


def test_a_recording_that_fails_leaves_the_lengths(wgf, drydev):
    c = drydev.kv_cache(1, 1, 64, 8, wgf.F16)
    k = blank(wgf, drydev, (1, 1, 1, 64))
    with drydev.record() as s:
        c.append(k, k)
    s.destroy()
    assert c.lengths == [1]
    del s
    c.append(k, k)
    assert c.lengths == [2]


# ---- norm and rotation -----------------------------------------------------------------------------------------------
def test_qk_norm_rope_refusals(wgf, drydev):
    q, k = blank(wgf, drydev, (2, 6, 3, 64)), blank(wgf, drydev, (2, 2, 3, 64))
    w, t = blank(wgf, drydev, (64,)), blank(wgf, drydev, (10, 32))
    a, b = q.qk_norm_rope(k, w, w, t, t, start=7)
    assert a.shape == (2, 6, 3, 64) and b.shape == (2, 2, 3, 64)
    before = drydev.launch_count
    wgf.Tensor.materialize_all([a, b])
    assert drydev.launch_count - before == 1
    refused(wgf, "SHAPE", q.qk_norm_rope, k, w, w, t, t, start=8)
    refused(wgf, "SHAPE", q.qk_norm_rope, k, w, w, t, t, start=-1)
    refused(wgf, "SHAPE", q.qk_norm_rope, k, w, w, t, t, start=2 ** 62)
    refused(wgf, "RANK", q.qk_norm_rope, blank(wgf, drydev, (2, 3, 64)), w, w, t, t)
    refused(wgf, "SHAPE", q.qk_norm_rope, blank(wgf, drydev, (1, 2, 3, 64)), w, w, t, t)
    refused(wgf, "SHAPE", q.qk_norm_rope, blank(wgf, drydev, (2, 2, 4, 64)), w, w, t, t)
    refused(wgf, "SHAPE", q.qk_norm_rope, k, blank(wgf, drydev, (32,)), w, t, t)
    refused(wgf, "SHAPE", q.qk_norm_rope, k, w, w, t, blank(wgf, drydev, (11, 32)))
    refused(wgf, "DTYPE", q.qk_norm_rope, k, w, blank(wgf, drydev, (64,), "F32"), t, t)
    x = blank(wgf, drydev, (1, 2, 7))
    refused(wgf, "UNSUPPORTED", x.qk_norm_rope, x, w, w, t, t)
    x = blank(wgf, drydev, (1, 2, 514))
    refused(wgf, "UNSUPPORTED", x.qk_norm_rope, x, w, w, t, t)


# ---- 4-bit weights -----------------------------------------------------------------------------------------------------
def test_q4_refusals_and_shapes(wgf, drydev):
    w = blank(wgf, drydev, (33, 70)).quantize_q4(32)
    assert w.info == (33, 70, 32, wgf.F16)
    assert w.dequantize(wgf.BF16).shape == (33, 70)
    for shape in [(70,), (1, 70), (2, 3, 70), (40, 70), (0, 70)]:
        assert blank(wgf, drydev, shape).mat_mul_q4(w).materialize().shape == shape[:-1] + (33,)
    refused(wgf, "SHAPE", blank(wgf, drydev, (2, 71)).mat_mul_q4, w)
    refused(wgf, "RANK", blank(wgf, drydev, (70,)).sum(0).mat_mul_q4, w)
    refused(wgf, "INVALID_ARGUMENT", blank(wgf, wgf.Device(-1), (1, 70)).mat_mul_q4, w)
    for group in (0, 16, 48, 256):
        refused(wgf, "INVALID_ARGUMENT", blank(wgf, drydev, (4, 64)).quantize_q4, group)
    refused(wgf, "RANK", blank(wgf, drydev, (64,)).quantize_q4, 32)
    refused(wgf, "SHAPE", blank(wgf, drydev, (0, 64)).quantize_q4, 32)
    c, s = np.zeros((4, 35), np.uint8), np.zeros((4, 3), np.float32)
    assert drydev.q4_weight(c, s, 69, 32).info == (4, 69, 32, wgf.F32)
    refused(wgf, "INVALID_ARGUMENT", drydev.q4_weight, c, s, 69, 48 - 24)
    with pytest.raises(ValueError):
        drydev.q4_weight(c, s, 71, 32)


def test_null_handles_are_errors(wgf, drydev):
    import ctypes as C
    out, lib = C.c_void_p(), wgf.lib()
    for call in [lambda: lib.wgf_kv_cache_create(None, C.c_uint32(0), C.c_int64(1), C.c_int64(1), C.c_int64(64), C.c_int64(1), C.byref(out)),
                 lambda: lib.wgf_kv_cache_append(None, None, None, None), lambda: lib.wgf_kv_cache_truncate(None, None),
                 lambda: lib.wgf_kv_cache_attention(None, None, C.c_float(1), None, C.byref(out)), lambda: lib.wgf_kv_cache_read(None, None, None),
                 lambda: lib.wgf_kv_cache_release(None), lambda: lib.wgf_q4_weight_release(None), lambda: lib.wgf_tensor_matmul_q4(None, None, C.byref(out)),
                 lambda: lib.wgf_q4_weight_quantize(None, C.c_uint32(32), C.byref(out)), lambda: lib.wgf_q4_weight_dequantize(None, C.c_uint32(0), C.byref(out)),
                 lambda: lib.wgf_tensor_qk_norm_rope(None, None, None, None, None, None, C.c_float(0), C.c_int64(0), C.byref(out), C.byref(out))]:
        assert call() == 8


# ---- the reference itself -------------------------------------------------------------------------------------------------
def test_the_rounding_to_codes_never_takes_the_wrong_side():
    """What the kernels do to a value, step by step in float32, against the quotient in 64 bits: the product with 127 in two
    parts, the remainder of the nearest integer by a fused multiply-add (emulated in 64 bits and rounded), the two borders."""
    g = np.random.Generator(np.random.PCG64(11))
    f = np.float32
    for bits in (8, 11, 24):
        top = g.uniform(1, 2, 4000)
        n = g.integers(-127, 128, 4000) + np.where(g.random(4000) < 0.5, 0.5, 0.0)
        x = n * top / 127 * (1 + g.integers(-2, 3, 4000) * 2.0 ** -bits)
        cut = lambda v: f(np.ldexp(np.rint(np.ldexp(v, bits - 1)), 1 - bits))
        top = cut(top)
        e = np.floor(np.log2(np.maximum(np.abs(x), 1e-30)))
        x = f(np.ldexp(np.rint(np.ldexp(x, (bits - 1 - e).astype(int))), (e - bits + 1).astype(int)))
        x = np.clip(x, -top, top)
        want = np.rint(127.0 * x.astype(np.float64) / top.astype(np.float64))
        p = f(f(127) * x)
        pl = f(127.0 * x.astype(np.float64) - p.astype(np.float64))
        r = np.rint(f(p * f(f(1) / top)))
        rem = f(p.astype(np.float64) - r.astype(np.float64) * top.astype(np.float64))
        h = f(0.5) * top
        over, under = f(f(rem - h) + pl), f(f(rem + h) + pl)
        odd = r.astype(np.int64) % 2 != 0
        up, down = (over > 0) | ((over == 0) & odd), (under < 0) | ((under == 0) & odd)
        got = r + np.where(up, 1, 0) - np.where(down & ~up, 1, 0)
        np.testing.assert_array_equal(got, want)


# ---- the C++ mirror ---------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def cpp_binary(tmp_path_factory, wgf):
    import os
    import subprocess
    wgf.lib()
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.dirname(wgf.LIB_PATH)
    exe = str(tmp_path_factory.mktemp("cpp") / "decode_test")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(root, "include"), os.path.join(root, "tests", "cpp", "decode_test.cpp"),
                    "-o", exe, "-L", lib, "-lwgf", f"-Wl,-rpath,{lib}"], check=True)
    return exe


def run_cpp(*command):
    import subprocess
    r = subprocess.run(command, capture_output=True, text=True)
    assert r.returncode == 0 and "decode ok" in r.stdout, r.stdout + r.stderr


def test_cpp_mirror_without_gpu(cpp_binary):
    run_cpp(cpp_binary, "--compile-only-device")


@pytest.mark.gpu
def test_cpp_mirror_on_gpu(cpp_binary):
    run_cpp(cpp_binary)


@pytest.mark.parametrize("rows", [0, 5])
def test_fused_append_of_padding_alone_reads_no_tables(wgf, drydev, rows):
    """No sequence has or takes a token: the tables may be empty, so no kernel may look at them."""
    c = drydev.kv_cache(2, 2, 64, 100, wgf.F16)
    q, k = blank(wgf, drydev, (2, 6, 3, 64)), blank(wgf, drydev, (2, 2, 3, 64))
    w, t = blank(wgf, drydev, (64,)), blank(wgf, drydev, (rows, 32))
    before = drydev.launch_count
    out = c.append_qk(q, k, k, w, w, t, t, counts=[0, 0])
    assert out.shape == (2, 6, 3, 64) and c.lengths == [0, 0] and drydev.launch_count == before
    if rows == 0:
        refused(wgf, "SHAPE", c.append_qk, q, k, k, w, w, t, t, counts=[0, 1])
        refused(wgf, "SHAPE", c.append_qk, q, k, k, w, w, t, t)
    assert c.lengths == [0, 0]


def test_a_recording_that_is_broken_off_counts_what_it_recorded(wgf, drydev):
    """A call inside fails and the block is left: what was recorded before it has run once, and the refused call has left nothing."""
    c = drydev.kv_cache(1, 1, 64, 8, wgf.F16)
    k = blank(wgf, drydev, (1, 1, 1, 64))
    for refusal in (dict(counts=[1]), None):
        before = c.lengths[0]
        with pytest.raises(wgf.WgfError):
            with drydev.record():
                c.append(k, k)
                if refusal:
                    c.append(k, k, **refusal)
                c.truncate([0])
        assert c.lengths == [before + 1]
    with pytest.raises(wgf.WgfError):
        with drydev.record():
            c.append(blank(wgf, drydev, (1, 1, 7, 64)), k)
    assert c.lengths == [2]
    with drydev.record() as s:
        c.append(k, k)
    s.launch()
    assert c.lengths == [4]
