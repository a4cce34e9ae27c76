"""GPU tests of the 4-bit KV cache and of the attention over it, against the 64-bit numpy form in oracle/kv4.py.

What the cache holds is compared byte for byte (the quantiser decides its borders exactly).  Attention is held to the
element-wise bound of an f32 evaluation (oracle.kv4.attention derives it) and to 2^-19 of the output in the 2-norm:
independent errors of some 2^-22 per term (the operands' 22 bits) leave that an order of magnitude above what is expected."""
import ctypes as C

import numpy as np
import pytest

from oracle import kv4

pytestmark = pytest.mark.gpu

GEOMETRY = [(8, 2, 64), (32, 8, 128), (5, 1, 96), (6, 3, 32), (16, 1, 128), (3, 3, 64), (14, 2, 96), (24, 3, 128)]


def rng(*seed):
    return np.random.Generator(np.random.PCG64([0x4B5634, *seed]))


def rows(r, n, n_kv, hd, keys):
    x = r.standard_normal((n, n_kv, hd), dtype=np.float32)
    if keys:
        off = r.standard_normal((n_kv, hd), dtype=np.float32)
        x += np.where(np.abs(off) > 1.6, 4 * off, 0)
    return x


def upload(gpu, a):
    return gpu.GpuBuf.upload(np.ascontiguousarray(a))


def put(gpu, buf, a):
    a = np.ascontiguousarray(a)
    gpu.lib().cuda_h2d(buf.ptr, a.ctypes.data, a.nbytes)


def filled(gpu, r, n, n_kv, hd, max_seq, byte=0xFF):
    """A cache of garbage bytes (0xFF: NaN parameters) whose first n positions are written by address on the host."""
    k, v = rows(r, n, n_kv, hd, True), rows(r, n, n_kv, hd, False)
    raw = kv4.store(np.full(kv4.nbytes(max_seq, n_kv, hd), byte, np.uint8), k, v, 0, max_seq)
    return upload(gpu, raw), raw, kv4.values(k), kv4.values(v)


def held(got, want, bound):
    err = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all()
    worst = float((err / bound).max())
    assert worst <= 1.0, worst
    assert np.linalg.norm(err) <= 2.0 ** -19 * np.linalg.norm(want), np.linalg.norm(err) / np.linalg.norm(want)


# ---- rows in and out -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,n_kv,hd,pos0,extra", [(1, 2, 64, 0, 0), (1, 1, 32, 37, 3), (31, 3, 96, 1, 0), (32, 8, 128, 32, 0), (33, 2, 128, 31, 40),
                                                  (77, 5, 32, 60, 1), (200, 4, 96, 3, 7), (65, 1, 64, 0, 30)])
def test_rows_match_byte_for_byte(gpu, n, n_kv, hd, pos0, extra):
    L, r = gpu.lib(), rng(n, n_kv, hd)
    max_seq = pos0 + n + extra
    k, v = rows(r, n, n_kv, hd, True), rows(r, n, n_kv, hd, False)
    raw = r.integers(0, 256, kv4.nbytes(max_seq, n_kv, hd), dtype=np.uint8)
    assert L.cuda_kv4_bytes(max_seq, n_kv, hd) == raw.size
    cache, dk, dv = upload(gpu, raw), upload(gpu, k), upload(gpu, v)
    L.cuda_kv4_append_rows(cache.ptr, dk.ptr, dv.ptr, n, n_kv, hd, max_seq, pos0)
    gpu.check_error()
    want = kv4.store(raw.copy(), k, v, pos0, max_seq)      # what other positions own stays as it was
    assert np.array_equal(cache.download(np.uint8), want)
    ok, ov = gpu.GpuBuf.alloc_f32(k.size + 16), gpu.GpuBuf.alloc_f32(v.size + 16)
    for b in (ok, ov):
        put(gpu, b, np.full(k.size + 16, 7.5, np.float32))
    L.cuda_kv4_read_rows(ok.ptr, ov.ptr, cache.ptr, n, n_kv, hd, max_seq, pos0)
    gpu.check_error()
    for b, x in ((ok, k), (ov, v)):
        got = b.download()
        assert np.array_equal(got[:k.size], kv4.values(x).reshape(-1))
        assert (got[k.size:] == 7.5).all()
    err = np.abs(kv4.values(k).astype(np.float64) - k).reshape(n, n_kv, -1, 32)
    assert (err <= kv4.quantise(k)[2][..., None] / 2 * (1 + 2.0 ** -10)).all()


def test_rows_at_the_borders(gpu):
    """Groups where a rounding could go either way: exact ties between two codes, extremes one f32 ulp beside an f16
    number, constants, zeros, subnormal steps, magnitudes beyond f16, and groups with NaN or an infinity."""
    L, r = gpu.lib(), rng(5)
    hd, groups = 32, []
    for m, d in ((-3.0, 0.25), (0.0, 2.0 ** -24), (-2047.0, 1.0), (5.0, 0.3125), (-0.125, 0.0078125)):
        base = np.float32(m) + np.arange(16, dtype=np.float32) * np.float32(d)
        half = base[:15] + np.float32(d / 2)
        groups.append(np.concatenate((base, half, [base[15]])))
        groups.append(np.concatenate((base, np.nextafter(half, np.float32(9e9)), [base[15]])))
        groups.append(np.concatenate((base, np.nextafter(half, np.float32(-9e9)), [base[15]])))
    for lo in (-1.0, 0.0, 1.0, 2.0 ** -14, 1000.0):
        for a in (np.float32(lo), np.nextafter(np.float32(lo), np.float32(9e9)), np.nextafter(np.float32(lo), np.float32(-9e9))):
            for s in (15.0, 15 * 1.0009765625, 15 * 2.0 ** -20, 15 * 2.0 ** -24):
                for b in (np.float32(a + np.float32(s)), np.nextafter(np.float32(a + np.float32(s)), np.float32(9e9))):
                    groups.append(np.concatenate((np.linspace(a, b, 31, dtype=np.float32).clip(a, b), [b])))
    groups += [np.zeros(32), np.full(32, -0.0), np.full(32, 3.14159), np.full(32, 1e-30), np.linspace(-1e-9, 1e-9, 32), np.linspace(-7e4, 7e4, 32),
               np.linspace(-2e6, 3e6, 32), np.full(32, 1e5), np.full(32, -1e5), np.linspace(-65504, 65504, 32)]
    for bad in (np.nan, np.inf, -np.inf):
        for i in (0, 13, 31):
            g = r.standard_normal(32)
            g[i] = bad
            groups.append(g)
    groups += list(r.standard_normal((400, 32)) * np.exp(r.uniform(-12, 9, (400, 1))))
    x = np.array(groups, np.float32).reshape(-1, 1, hd)
    n = x.shape[0]
    raw = np.zeros(kv4.nbytes(n, 1, hd), np.uint8)
    cache, dk, dv = upload(gpu, raw), upload(gpu, x), upload(gpu, x[::-1])
    L.cuda_kv4_append_rows(cache.ptr, dk.ptr, dv.ptr, n, 1, hd, n, 0)
    gpu.check_error()
    want = kv4.store(raw, x, x[::-1], 0, n)
    assert np.array_equal(cache.download(np.uint8), want)
    ok, ov = gpu.GpuBuf.alloc_f32(x.size), gpu.GpuBuf.alloc_f32(x.size)
    L.cuda_kv4_read_rows(ok.ptr, ov.ptr, cache.ptr, n, 1, hd, n, 0)
    assert np.array_equal(ok.download(), kv4.values(x).reshape(-1), equal_nan=True)
    assert np.array_equal(ov.download(), kv4.values(x[::-1]).reshape(-1), equal_nan=True)


@pytest.mark.parametrize("n,nh,n_kv,hd,pos0,neox,theta", [(1, 4, 2, 64, 0, 0, 1e4), (5, 8, 8, 128, 30, 1, 5e5), (40, 3, 1, 96, 7, 0, 1e4),
                                                          (9, 6, 2, 32, 0, 1, 1e4), (6, 4, 4, 128, 11, 0, 0.0)])
def test_rope_rows_equal_rotation_then_append(gpu, n, nh, n_kv, hd, pos0, neox, theta):
    L, r = gpu.lib(), rng(n, nh, hd)
    max_seq, kv_dim = pos0 + n + 2, n_kv * hd
    q, k, v = (r.standard_normal((n, h, hd), dtype=np.float32) for h in (nh, n_kv, n_kv))
    dq, dk, dv, q2, k2 = (upload(gpu, a) for a in (q, k, v, q, k))
    zero = np.zeros(kv4.nbytes(max_seq, n_kv, hd), np.uint8)
    c1, c2 = upload(gpu, zero), upload(gpu, zero)
    L.cuda_rope_kv4_rows(dq.ptr, dk.ptr, dv.ptr, c1.ptr, n, nh, n_kv, hd, max_seq, pos0, theta, 4.0, 8192, neox)
    if theta > 0:
        f = gpu.GpuBuf.alloc_f32(2 * max_seq * kv_dim)
        L.cuda_rope_kv_rows(q2.ptr, k2.ptr, dv.ptr, f.ptr, f.ptr + 4 * max_seq * kv_dim, n, nh, n_kv, hd, pos0, theta, 4.0, 8192, neox)
    L.cuda_kv4_append_rows(c2.ptr, k2.ptr, dv.ptr, n, n_kv, hd, max_seq, pos0)
    gpu.check_error()
    assert np.array_equal(dq.download(), q2.download()) and np.array_equal(dk.download(), k2.download())
    assert np.array_equal(dv.download(), v.reshape(-1))
    assert np.array_equal(c1.download(np.uint8), c2.download(np.uint8))


@pytest.mark.parametrize("neox", [0, 1])
@pytest.mark.parametrize("nh,n_kv,hd", GEOMETRY)
@pytest.mark.parametrize("n", [1, 3, 700])
def test_rope_rows_of_every_geometry(gpu, nh, n_kv, hd, n, neox):
    test_rope_rows_equal_rotation_then_append(gpu, n, nh, n_kv, hd, 5, neox, 1e4)
    test_rope_rows_equal_rotation_then_append(gpu, n, nh, n_kv, hd, 5, neox, 0.0)


# ---- one token -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("nh,n_kv,hd", GEOMETRY)
@pytest.mark.parametrize("ctx", [1, 2, 31, 32, 33, 64, 95, 300, 1025])
def test_step(gpu, nh, n_kv, hd, ctx):
    run_step(gpu, nh, n_kv, hd, ctx, max_seq=ctx + (ctx % 3) * 17, window=0, sinks=ctx % 2 == 0, append=ctx % 4 == 1)


@pytest.mark.parametrize("ctx,window", [(40, 1), (40, 8), (100, 32), (100, 33), (333, 64), (333, 333), (333, 1000), (1500, 700), (65, 66)])
@pytest.mark.parametrize("append", [False, True])
def test_step_window(gpu, ctx, window, append):
    run_step(gpu, 8, 2, 64, ctx, max_seq=ctx + 5, window=window, sinks=append, append=append)
    run_step(gpu, 32, 8, 128, ctx, max_seq=ctx, window=window, sinks=not append, append=append)


@pytest.mark.parametrize("nh,n_kv,hd,ctx", [(32, 8, 128, 9001), (4, 1, 64, 20011), (16, 2, 96, 6005)])
def test_step_long(gpu, nh, n_kv, hd, ctx):
    run_step(gpu, nh, n_kv, hd, ctx, max_seq=ctx + 64, window=0, sinks=False, append=False)
    run_step(gpu, nh, n_kv, hd, ctx, max_seq=ctx + 64, window=0, sinks=False, append=True, sharp=8.0)


@pytest.mark.parametrize("nh,n_kv,hd,max_seq", [(64, 8, 64, 9000), (40, 8, 32, 8200), (28, 4, 96, 33000), (48, 8, 128, 8192)])
@pytest.mark.parametrize("ctx", [1, 70, 1500, 8111])
def test_step_wide_groups_in_a_long_cache(gpu, nh, n_kv, hd, max_seq, ctx):
    run_step(gpu, nh, n_kv, hd, ctx, max_seq=max_seq, window=0, sinks=ctx == 70, append=ctx != 1500)


def run_step(gpu, nh, n_kv, hd, ctx, max_seq, window, sinks, append, sharp=1.0):
    L, r = gpu.lib(), rng(nh, n_kv, hd, ctx, window)
    pos, scale = ctx - 1, np.float32(1 / np.sqrt(hd))
    old = ctx - 1 if append else ctx
    cache, raw, k, v = filled(gpu, r, old, n_kv, hd, max_seq)
    q = r.standard_normal((1, nh, hd), dtype=np.float32) * np.float32(sharp)
    sink = r.standard_normal(nh).astype(np.float32) * 2 if sinks else None
    dq, out = upload(gpu, q), gpu.GpuBuf.alloc_f32(nh * hd)
    ds = upload(gpu, sink) if sinks else None
    want_raw = raw
    if append:
        kn, vn = rows(r, 1, n_kv, hd, True), rows(r, 1, n_kv, hd, False)
        k, v = np.concatenate((k, kv4.values(kn))), np.concatenate((v, kv4.values(vn)))
        want_raw = kv4.store(raw.copy(), kn, vn, pos, max_seq)
        dk, dv = upload(gpu, kn), upload(gpu, vn)
    L.cuda_attn_step_kv4(out.ptr, dq.ptr, dk.ptr if append else None, dv.ptr if append else None, cache.ptr, nh, n_kv, hd, max_seq, None, pos,
                         window, scale, ds.ptr if sinks else None, 0.0, 1.0, 0, 0, -1)
    got = out.download().reshape(1, nh, hd)
    gpu.check_error()
    held(got, *kv4.attention(q, k, v, pos, window, float(scale), sink))
    assert np.array_equal(cache.download(np.uint8), want_raw)      # only the appended position's bytes changed
    assert np.array_equal(dq.download(), q.reshape(-1))


@pytest.mark.parametrize("neox,yarn", [(0, 1.0), (1, 1.0), (0, 4.0), (1, 8.0)])
@pytest.mark.parametrize("nh,n_kv,hd", [(8, 2, 64), (32, 8, 128), (6, 3, 96), (4, 4, 32)])
def test_step_rotates_as_the_rows_do(gpu, nh, n_kv, hd, neox, yarn):
    """One step with rotation and append = cuda_rope_kv4_rows, then a step without either; q, k_new, v_new untouched."""
    L, r = gpu.lib(), rng(nh, hd, neox)
    ctx, max_seq = 41, 64
    a, _, _, _ = filled(gpu, r, ctx - 1, n_kv, hd, max_seq)
    b = upload(gpu, a.download(np.uint8))
    q, k, v = (r.standard_normal((1, h, hd), dtype=np.float32) for h in (nh, n_kv, n_kv))
    dq, dk, dv, q2, k2 = (upload(gpu, x) for x in (q, k, v, q, k))
    o1, o2 = gpu.GpuBuf.alloc_f32(nh * hd), gpu.GpuBuf.alloc_f32(nh * hd)
    tail = (0.11, None)
    L.cuda_attn_step_kv4(o1.ptr, dq.ptr, dk.ptr, dv.ptr, a.ptr, nh, n_kv, hd, max_seq, None, ctx - 1, 0, *tail, 1e4, yarn, 32, neox, -1)
    L.cuda_rope_kv4_rows(q2.ptr, k2.ptr, dv.ptr, b.ptr, 1, nh, n_kv, hd, max_seq, ctx - 1, 1e4, yarn, 32, neox)
    L.cuda_attn_step_kv4(o2.ptr, q2.ptr, None, None, b.ptr, nh, n_kv, hd, max_seq, None, ctx - 1, 0, *tail, 0.0, 1.0, 0, 0, -1)
    gpu.check_error()
    assert np.array_equal(a.download(np.uint8), b.download(np.uint8))
    got, want = o1.download(), o2.download()
    # the rotation may round differently by an ulp where the compiler contracts it: 2^-22 of a score's terms
    assert np.abs(got - want).max() <= 2.0 ** -18 * np.abs(want).max()
    assert np.array_equal(dq.download(), q.reshape(-1)) and np.array_equal(dk.download(), k.reshape(-1))


def test_step_position_from_the_device(gpu):
    """Position words: a recorded graph serves every position; with the rotation table and without it; clamped at the ends."""
    L, r = gpu.lib(), rng(77)
    nh, n_kv, hd, max_seq = 16, 4, 128, 100
    cache, raw, k, v = filled(gpu, r, 100, n_kv, hd, max_seq)
    kv = [rows(r, 1, n_kv, hd, s) for s in (True, False)]
    q = r.standard_normal((1, nh, hd), dtype=np.float32)
    dq, dk, dv = upload(gpu, q), upload(gpu, kv[0]), upload(gpu, kv[1])
    out, step = gpu.GpuBuf.alloc_f32(nh * hd), gpu.GpuBuf.alloc_f32(4)

    def call(words):
        L.cuda_attn_step_kv4(out.ptr, dq.ptr, dk.ptr, dv.ptr, cache.ptr, nh, n_kv, hd, max_seq, step.ptr if words else None, 0 if words else pos, 16,
                             0.09, None, 1e4, 1.0, 0, 0, -1)
    L.cuda_step_rope_table(step.ptr, hd, 1e4, 1.0, 0)
    L.cuda_step_set(step.ptr, 0, 0)
    call(True)
    assert L.quartz_graph_begin()
    call(True)
    graph = L.quartz_graph_end()
    assert graph
    for pos in (0, 1, 31, 32, 59, 60, 99):
        put(gpu, cache, raw)
        call(False)
        want, bytes_ = out.download(), cache.download(np.uint8)
        for replay in (False, True):
            put(gpu, cache, raw)
            L.cuda_step_set(step.ptr, 5, pos)
            L.quartz_graph_launch(graph) if replay else call(True)
            assert np.array_equal(out.download(), want), pos
            assert np.array_equal(cache.download(np.uint8), bytes_)
    for words, at in ((-3, 0), (100, 99), (2 ** 31 - 1, 99)):      # never outside the cache
        L.cuda_step_set(step.ptr, 5, words)
        call(True)
        got = out.download()
        L.cuda_step_set(step.ptr, 5, at)
        call(True)
        assert np.array_equal(out.download(), got)
    L.quartz_graph_destroy(graph)
    gpu.check_error()


def test_step_activation_form(gpu):
    """out_slot: the slot holds what cuda_quantize_x makes of the result (seen through a GEMV that reads the slot)."""
    from saient_quartz_b200 import synth
    L, r = gpu.lib(), rng(3)
    for nh, n_kv, hd, ctx in ((16, 4, 128, 70), (8, 1, 64, 5), (32, 8, 96, 333), (2, 2, 32, 1)):
        cache, _, _, _ = filled(gpu, r, ctx, n_kv, hd, ctx)
        K, N = nh * hd, 64
        dq, out = upload(gpu, r.standard_normal((1, nh, hd), dtype=np.float32)), gpu.GpuBuf.alloc_f32(K)
        w = upload(gpu, synth.make_weights(8, K, N, tensor_id=3))
        y = [gpu.GpuBuf.alloc_f32(N) for _ in range(2)]
        L.cuda_attn_step_kv4(out.ptr, dq.ptr, None, None, cache.ptr, nh, n_kv, hd, ctx, None, ctx - 1, 0, 0.1, None, 0.0, 1.0, 0, 0, 2)
        L.cuda_quantize_x(out.ptr, K, 1)
        if not L.cuda_gemv_q_supported(8, w.ptr, K):
            gpu.check_error()
            continue
        for slot, b in ((2, y[0]), (1, y[1])):
            L.cuda_gemv_q(8, 1, (C.c_void_p * 1)(w.ptr), (C.c_int * 1)(slot), (C.c_void_p * 1)(b.ptr), K, N, 0)
        gpu.check_error()
        assert np.array_equal(y[0].download(), y[1].download())


def test_step_propagates_nan(gpu):
    """A visible group with a NaN makes that kv head's outputs NaN, no others; behind the window it does nothing."""
    L, r = gpu.lib(), rng(9)
    nh, n_kv, hd, ctx = 8, 4, 64, 50
    k, v = rows(r, ctx, n_kv, hd, True), rows(r, ctx, n_kv, hd, False)
    k[10, 2, 5] = np.inf
    raw = kv4.store(np.zeros(kv4.nbytes(ctx, n_kv, hd), np.uint8), k, v, 0, ctx)
    cache, q = upload(gpu, raw), r.standard_normal((1, nh, hd), dtype=np.float32)
    dq, out = upload(gpu, q), gpu.GpuBuf.alloc_f32(nh * hd)
    for window, hit in ((0, True), (40, True), (39, False)):
        L.cuda_attn_step_kv4(out.ptr, dq.ptr, None, None, cache.ptr, nh, n_kv, hd, ctx, None, ctx - 1, window, 0.1, None, 0.0, 1.0, 0, 0, -1)
        got = out.download().reshape(nh, hd)
        assert np.isnan(got[4:6]).all() == hit and np.isfinite(np.delete(got, (4, 5) if hit else (), 0)).all()
    gpu.check_error()


def test_step_scales_of_values_far_apart(gpu):
    """Values whose steps differ by 2^20 between positions and between groups; scores that leave one position only."""
    L, r = gpu.lib(), rng(10)
    nh, n_kv, hd, ctx = 4, 1, 128, 200
    k, v = rows(r, ctx, n_kv, hd, False), rows(r, ctx, n_kv, hd, False)
    v *= np.exp2(r.integers(-10, 11, (ctx, 1, 4))).repeat(32, -1).astype(np.float32)
    cache = upload(gpu, kv4.store(np.zeros(kv4.nbytes(ctx, n_kv, hd), np.uint8), k, v, 0, ctx))
    out = gpu.GpuBuf.alloc_f32(nh * hd)
    for sharp in (0.0, 1e-20, 1.0, 30.0, 3000.0):
        q = r.standard_normal((1, nh, hd), dtype=np.float32) * np.float32(sharp)
        dq = upload(gpu, q)
        L.cuda_attn_step_kv4(out.ptr, dq.ptr, None, None, cache.ptr, nh, n_kv, hd, ctx, None, ctx - 1, 0, 0.088, None, 0.0, 1.0, 0, 0, -1)
        want, bound = kv4.attention(q, kv4.values(k), kv4.values(v), ctx - 1, 0, float(np.float32(0.088)), None)
        got = out.download().reshape(1, nh, hd)
        assert (np.abs(got - want) <= bound + 2.0 ** -20 * np.abs(want).max()).all(), sharp
    gpu.check_error()


# ---- a prompt --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("nh,n_kv,hd", GEOMETRY)
@pytest.mark.parametrize("n,pos0,window", [(1, 0, 0), (2, 31, 0), (33, 0, 0), (40, 57, 0), (70, 5, 16), (65, 100, 33)])
def test_prompt(gpu, nh, n_kv, hd, n, pos0, window):
    run_prompt(gpu, nh, n_kv, hd, n, pos0, window, sinks=(n + hd) % 2 == 0)


@pytest.mark.parametrize("nh,n_kv,hd,n,pos0,window", [(8, 2, 128, 200, 900, 0), (8, 1, 64, 300, 0, 0), (4, 2, 96, 150, 700, 300)])
def test_prompt_long(gpu, nh, n_kv, hd, n, pos0, window):
    run_prompt(gpu, nh, n_kv, hd, n, pos0, window, sinks=False)
    run_prompt(gpu, nh, n_kv, hd, n, pos0, window, sinks=True, sharp=6.0)


def run_prompt(gpu, nh, n_kv, hd, n, pos0, window, sinks, sharp=1.0):
    L, r = gpu.lib(), rng(nh, n_kv, hd, n, pos0)
    max_seq, scale = pos0 + n + 9, np.float32(1 / np.sqrt(hd))
    cache, raw, k, v = filled(gpu, r, pos0 + n, n_kv, hd, max_seq)
    q = r.standard_normal((n, nh, hd), dtype=np.float32) * np.float32(sharp)
    sink = r.standard_normal(nh).astype(np.float32) if sinks else None
    ds = upload(gpu, sink) if sinks else None
    dq, out = upload(gpu, q), upload(gpu, np.full(q.size + 64, 3.25, np.float32))
    L.cuda_attn_prompt_kv4(out.ptr, dq.ptr, cache.ptr, n, nh, n_kv, hd, max_seq, pos0, window, scale, ds.ptr if sinks else None)
    got = out.download()
    gpu.check_error()
    assert (got[q.size:] == 3.25).all()
    held(got[:q.size].reshape(q.shape), *kv4.attention(q, k, v, pos0, window, float(scale), sink))
    assert np.array_equal(cache.download(np.uint8), raw)


# Long enough that the call takes the tensor-core kernel (fewer tokens go through the step kernel).
@pytest.mark.parametrize("nh,n_kv,hd,n", [(8, 2, 64, 700), (32, 8, 128, 515), (5, 1, 96, 1100), (6, 3, 32, 801), (16, 1, 128, 1000), (3, 3, 64, 703),
                                          (14, 2, 96, 700), (24, 3, 128, 690)])
@pytest.mark.parametrize("pos0,window", [(0, 0), (93, 0), (0, 33), (450, 100), (31, 129)])
def test_prompt_tiles(gpu, nh, n_kv, hd, n, pos0, window):
    run_prompt(gpu, nh, n_kv, hd, n, pos0, window, sinks=pos0 % 2 == 1, sharp=4.0 if window == 100 else 1.0)


def test_prompt_queries_of_any_size(gpu):
    """Scores that single one position out, scores that all but vanish, and queries near both ends of f32."""
    L, r = gpu.lib(), rng(31)
    nh, n_kv, hd, n = 16, 8, 64, 515
    k, v = rows(r, n, n_kv, hd, True), rows(r, n, n_kv, hd, False)
    cache = upload(gpu, kv4.store(np.full(kv4.nbytes(n, n_kv, hd), 0xFF, np.uint8), k, v, 0, n))
    q = r.standard_normal((n, nh, hd), dtype=np.float32)
    q *= np.exp2(r.integers(-10, 11, (n, nh, 1))).astype(np.float32)
    dq, out = upload(gpu, q), gpu.GpuBuf.alloc_f32(q.size)
    L.cuda_attn_prompt_kv4(out.ptr, dq.ptr, cache.ptr, n, nh, n_kv, hd, n, 0, 0, 0.125, None)
    got = out.download().reshape(q.shape)
    gpu.check_error()
    want, bound = kv4.attention(q, kv4.values(k), kv4.values(v), 0, 0, 0.125, None)
    # A value is summed as p d (code - 8) and p (m + 8 d), which cancel where one position decides and its value is near zero
    # (the bound above counts |value|).  With A the larger end of the group's range, 15 d <= 2 A, the two are at most 16 / 15 A
    # and A; either carries 22 bits of p and one f32 rounding, 2^-22 + 2^-24: in all (31 / 15) 1.25 2^-22 A < 2^-20 A a position,
    # and the weights sum to one.  A exceeds the group's largest value by the rounding of d only (2^-10).
    seen = np.maximum.accumulate(np.abs(kv4.values(v)).max(-1), 0).repeat(nh // n_kv, 1)[..., None]
    assert (np.abs(got - want) <= bound + 2.0 ** -20 * seen).all()
    # one key towers over the others: with |q| = 2^120 its row is the answer, with 2^-120 the mean is
    k = np.zeros_like(k)
    k[0] = 1.0
    put(gpu, cache, kv4.store(np.full(kv4.nbytes(n, n_kv, hd), 0xFF, np.uint8), k, v, 0, n))
    vv = kv4.values(v)
    for e, answer in ((120, np.broadcast_to(vv[:1], vv.shape)), (-120, np.cumsum(vv, 0) / np.arange(1, n + 1)[:, None, None])):
        put(gpu, dq, np.full(q.shape, 2.0 ** e, np.float32))
        for tokens in (n, 1):       # the step kernel too
            L.cuda_attn_prompt_kv4(out.ptr, dq.ptr, cache.ptr, tokens, nh, n_kv, hd, n, n - tokens, 0, 0.125, None)
            got = out.download(count=tokens * nh * hd).reshape(tokens, nh, hd)
            want = answer[n - tokens:].repeat(nh // n_kv, 1)
            # a mean of n values of about 1: n roundings of 2^-24 each at most, and 2^-22 of each term
            assert np.abs(got - want).max() <= (n * 2.0 ** -24 + 2.0 ** -21) * np.abs(vv).max(), (e, tokens)
    gpu.check_error()


def test_prompt_scales_of_values_far_apart(gpu):
    """Steps that differ by 2^20 between positions and groups, some of them past 8188 in keys or in values; minima past f16's range."""
    L, r = gpu.lib(), rng(32)
    for nh, n_kv, hd, n in ((16, 8, 128, 515), (12, 6, 96, 515)):
        k, v = rows(r, n, n_kv, hd, False), rows(r, n, n_kv, hd, False)
        g = hd // 32
        v *= np.exp2(r.integers(-10, 11, (n, n_kv, g))).repeat(32, -1).astype(np.float32)
        v[100:103] *= 65000.0                    # spans of up to 2^17 and more: the largest step f16 holds
        v[300, :, :32] = np.linspace(-65504, 65504, 32)
        k[200, :, :32] = np.linspace(-65504, 65504, 32)
        k[201, :, 3] = 9e4
        q = r.standard_normal((n, nh, hd), dtype=np.float32) * np.float32(2.0 ** -14)
        cache = upload(gpu, kv4.store(np.full(kv4.nbytes(n, n_kv, hd), 0xFF, np.uint8), k, v, 0, n))
        dq, out = upload(gpu, q), gpu.GpuBuf.alloc_f32(q.size)
        L.cuda_attn_prompt_kv4(out.ptr, dq.ptr, cache.ptr, n, nh, n_kv, hd, n, 0, 0, 0.088, None)
        got = out.download().reshape(q.shape)
        gpu.check_error()
        want, bound = kv4.attention(q, kv4.values(k), kv4.values(v), 0, 0, float(np.float32(0.088)), None)
        # weights carry 22 bits; a tile's values are scaled by its largest (2^-20 of what the row has seen)
        seen = np.maximum.accumulate(np.abs(kv4.values(v)).max(-1), 0).repeat(nh // n_kv, 1)[..., None]
        assert (np.abs(got - want) <= bound + 2.0 ** -20 * seen).all()


def test_prompt_propagates_nan(gpu):
    """A NaN among a group's keys reaches every output of the rows that see it, one among its values that group's alone; rows
    before it, rows whose window has passed it and other heads are untouched."""
    L, r = gpu.lib(), rng(33)
    for nh, n_kv, hd, n in ((16, 8, 128, 515), (12, 6, 96, 515)):
        G = nh // n_kv
        k, v = rows(r, n, n_kv, hd, True), rows(r, n, n_kv, hd, False)
        q = r.standard_normal((n, nh, hd), dtype=np.float32)
        dq, out = upload(gpu, q), gpu.GpuBuf.alloc_f32(q.size)
        bad_k, bad_v = k.copy(), v.copy()
        bad_k[300, 2, 5] = np.nan
        bad_v[131, 4, 40] = np.inf               # group 1 of kv head 4
        bad_v[400, 4, 70] = np.nan               # and group 2, later
        for window in (0, 60):
            raw = kv4.store(np.full(kv4.nbytes(n + 40, n_kv, hd), 0xFF, np.uint8), bad_k, bad_v, 0, n + 40)
            cache = upload(gpu, raw)
            L.cuda_attn_prompt_kv4(out.ptr, dq.ptr, cache.ptr, n, nh, n_kv, hd, n + 40, 0, window, 0.088, None)
            got = out.download().reshape(q.shape)
            gpu.check_error()
            want, bound = kv4.attention(q, kv4.values(k), kv4.values(v), 0, window, float(np.float32(0.088)), None)
            t = np.arange(n)
            hit = np.zeros(q.shape, bool)
            sees = lambda p: (t >= p) & (t < p + window if window else True)
            hit[sees(300), 2 * G:3 * G] = True
            hit[sees(131), 4 * G:5 * G, 32:64] = True
            hit[sees(400), 4 * G:5 * G, 64:96] = True
            assert (np.isnan(got) == hit).all()
            # (the clean values differ where a NaN is hit only: rows elsewhere do not see positions 300, 131 or 400 of those heads' groups)
            assert (np.abs(got - want) <= bound)[~hit].all()


# ---- together, and where the machinery can go wrong --------------------------------------------------------------
def test_prompt_then_steps(gpu):
    """A prompt appended and attended to, then tokens one at a time, each through one recorded graph: the run of a
    generation loop, against the oracle on everything that was appended."""
    L, r = gpu.lib(), rng(21)
    nh, n_kv, hd, n, more = 8, 2, 128, 45, 25
    max_seq = n + more
    q, k, v = (r.standard_normal((n + more, h, hd), dtype=np.float32) for h in (nh, n_kv, n_kv))
    cache = upload(gpu, np.full(kv4.nbytes(max_seq, n_kv, hd), 0xFF, np.uint8))
    dq, dk, dv = upload(gpu, q[:n]), upload(gpu, k[:n]), upload(gpu, v[:n])
    out = gpu.GpuBuf.alloc_f32(n * nh * hd)
    L.cuda_rope_kv4_rows(dq.ptr, dk.ptr, dv.ptr, cache.ptr, n, nh, n_kv, hd, max_seq, 0, 0.0, 1.0, 0, 0)
    L.cuda_attn_prompt_kv4(out.ptr, dq.ptr, cache.ptr, n, nh, n_kv, hd, max_seq, 0, 0, 0.09, None)
    scale = float(np.float32(0.09))
    held(out.download().reshape(n, nh, hd), *kv4.attention(q[:n], kv4.values(k), kv4.values(v), 0, 0, scale, None))
    sq, sk, sv, step = (gpu.GpuBuf.alloc_f32(x) for x in (nh * hd, n_kv * hd, n_kv * hd, 4))
    one = gpu.GpuBuf.alloc_f32(nh * hd)
    token = upload(gpu, np.array([3], np.int32))
    L.cuda_step_set(step.ptr, 0, n - 1)
    assert L.quartz_graph_begin()
    L.cuda_attn_step_kv4(one.ptr, sq.ptr, sk.ptr, sv.ptr, cache.ptr, nh, n_kv, hd, max_seq, step.ptr, 0, 0, 0.09, None, 0.0, 1.0, 0, 0, -1)
    graph = L.quartz_graph_end()
    for t in range(n, n + more):
        for b, x in ((sq, q), (sk, k), (sv, v)):
            put(gpu, b, x[t])
        L.cuda_step_advance(step.ptr, token.ptr)
        L.quartz_graph_launch(graph)
        held(one.download().reshape(1, nh, hd), *kv4.attention(q[t:t + 1], kv4.values(k), kv4.values(v), t, 0, scale, None))
    assert list(step.download(np.int32, 2)) == [3, n + more - 1]
    L.quartz_graph_destroy(graph)
    gpu.check_error()


def test_appends_right_before_the_attention_in_one_graph(gpu):
    """Rows appended by the call just ahead of the attention, recorded together (programmatic dependents): the attention
    sees them.  Two such graphs on two streams, replayed at the same time, do not disturb one another."""
    import torch
    L, r = gpu.lib(), rng(22)
    nh, n_kv, hd, n = 32, 8, 128, 700
    sets = []
    for i in range(2):
        q, k, v = (r.standard_normal((n if h != nh else 1, h, hd), dtype=np.float32) for h in (nh, n_kv, n_kv))
        b = [upload(gpu, x) for x in (q, k, v, np.full(kv4.nbytes(n, n_kv, hd), 0xFF, np.uint8))] + [gpu.GpuBuf.alloc_f32(nh * hd)]
        assert L.quartz_graph_begin()
        L.cuda_kv4_append_rows(b[3].ptr, b[1].ptr, b[2].ptr, n, n_kv, hd, n, 0)
        L.cuda_attn_step_kv4(b[4].ptr, b[0].ptr, None, None, b[3].ptr, nh, n_kv, hd, n, None, n - 1, 0, 0.09, None, 0.0, 1.0, 0, 0, -1)
        sets.append((L.quartz_graph_end(), q, k, v, b))
    for _ in range(20):
        for g, _, _, v, b in sets:
            L.quartz_graph_launch(g)
    for g, q, k, v, b in sets:
        held(b[4].download().reshape(1, nh, hd), *kv4.attention(q, kv4.values(k), kv4.values(v), n - 1, 0, float(np.float32(0.09)), None))
    # the same calls on two user streams
    streams = [torch.cuda.Stream() for _ in sets]
    for b in (s[4] for s in sets):
        put(gpu, b[4], np.zeros(nh * hd, np.float32))
    for _ in range(20):
        for st, (_, _, _, _, b) in zip(streams, sets):
            L.quartz_set_stream(st.cuda_stream)
            L.cuda_attn_step_kv4(b[4].ptr, b[0].ptr, None, None, b[3].ptr, nh, n_kv, hd, n, None, n - 1, 0, 0.09, None, 0.0, 1.0, 0, 0, -1)
    torch.cuda.synchronize()
    L.quartz_set_stream(None)
    for g, q, k, v, b in sets:
        held(b[4].download().reshape(1, nh, hd), *kv4.attention(q, kv4.values(k), kv4.values(v), n - 1, 0, float(np.float32(0.09)), None))
        L.quartz_graph_destroy(g)
    gpu.check_error()


def test_cache_past_32_bits(gpu):
    """A cache of more than 4 GiB: the last head's rows lie behind 2^32 bytes."""
    L, r = gpu.lib(), rng(23)
    nh, n_kv, hd, max_seq, n = 8, 8, 128, 3_500_001, 70
    size = L.cuda_kv4_bytes(max_seq, n_kv, hd)
    assert size > 2 ** 32
    ptr = L.cuda_alloc(size)
    assert ptr
    try:
        pos0 = max_seq - n
        k, v = rows(r, n, n_kv, hd, True), rows(r, n, n_kv, hd, False)
        q = r.standard_normal((2, nh, hd), dtype=np.float32)
        dq, dk, dv = upload(gpu, q), upload(gpu, k), upload(gpu, v)
        L.cuda_kv4_append_rows(ptr, dk.ptr, dv.ptr, n, n_kv, hd, max_seq, pos0)
        ok, ov, out = gpu.GpuBuf.alloc_f32(k.size), gpu.GpuBuf.alloc_f32(v.size), gpu.GpuBuf.alloc_f32(q.size)
        L.cuda_kv4_read_rows(ok.ptr, ov.ptr, ptr, n, n_kv, hd, max_seq, pos0)
        assert np.array_equal(ok.download(), kv4.values(k).reshape(-1)) and np.array_equal(ov.download(), kv4.values(v).reshape(-1))
        L.cuda_attn_step_kv4(out.ptr, dq.ptr, None, None, ptr, nh, n_kv, hd, max_seq, None, max_seq - 1, 50, 0.09, None, 0.0, 1.0, 0, 0, -1)
        held(out.download(count=nh * hd).reshape(1, nh, hd), *kv4.attention(q[:1], kv4.values(k), kv4.values(v), n - 1, 50, float(np.float32(0.09)), None))
        L.cuda_attn_prompt_kv4(out.ptr, dq.ptr, ptr, 2, nh, n_kv, hd, max_seq, max_seq - 2, 50, 0.09, None)
        held(out.download().reshape(2, nh, hd), *kv4.attention(q, kv4.values(k), kv4.values(v), n - 2, 50, float(np.float32(0.09)), None))
        gpu.check_error()
    finally:
        L.cuda_drop(ptr)


# ---- several clusters and their merge, recorded ------------------------------------------------------------------
def merge_setup(gpu, r, nh, n_kv, hd, max_seq, filled_to):
    cache, raw, k, v = filled(gpu, r, filled_to, n_kv, hd, max_seq)
    q, kn, vn = r.standard_normal((1, nh, hd), dtype=np.float32), rows(r, 1, n_kv, hd, True), rows(r, 1, n_kv, hd, False)
    return cache, raw, k, v, q, kn, vn


@pytest.mark.parametrize("nh,n_kv,hd,max_seq", [(32, 8, 128, 9000), (8, 2, 64, 20000), (64, 8, 128, 9000), (12, 2, 96, 12000)])
def test_recorded_step_of_a_long_cache(gpu, nh, n_kv, hd, max_seq):
    """As a model with a long context issues it: rotation with the table, append, position words, activation slot, recorded, at positions
    that one, some and all clusters of a unit work on, several replays each."""
    from saient_quartz_b200 import synth
    L, r = gpu.lib(), rng(50, nh, hd)
    cache, raw, k, v, q, kn, vn = merge_setup(gpu, r, nh, n_kv, hd, max_seq, max_seq)
    dq, dk, dv = upload(gpu, q), upload(gpu, kn), upload(gpu, vn)
    K, N, scale = nh * hd, 64, 0.09
    out, out2, step = gpu.GpuBuf.alloc_f32(K), gpu.GpuBuf.alloc_f32(K), gpu.GpuBuf.alloc_f32(4)
    w = upload(gpu, synth.make_weights(8, K, N, tensor_id=3))
    y = [gpu.GpuBuf.alloc_f32(N) for _ in range(2)]

    def call():
        L.cuda_attn_step_kv4(out.ptr, dq.ptr, dk.ptr, dv.ptr, cache.ptr, nh, n_kv, hd, max_seq, step.ptr, 0, 0, scale, None, 5e5, 1.0, 0, 0, 2)
    L.cuda_step_rope_table(step.ptr, hd, 5e5, 1.0, 0)
    L.cuda_step_set(step.ptr, 0, 0)
    call()
    assert L.quartz_graph_begin()
    call()
    graph = L.quartz_graph_end()
    assert graph
    for pos in (7, 2000, 3199, max_seq // 2, max_seq - 1):
        L.cuda_step_set(step.ptr, 5, pos)
        got = []
        for _ in range(4):
            put(gpu, cache, raw)
            L.quartz_graph_launch(graph)
            got.append(out.download())
        assert all(np.array_equal(g, got[0]) for g in got)
        after = cache.download(np.uint8)
        # the same by parts: rotation and append by the rows' call, attention without either
        put(gpu, cache, raw)
        q2, k2 = upload(gpu, q), upload(gpu, kn)
        L.cuda_rope_kv4_rows(q2.ptr, k2.ptr, dv.ptr, cache.ptr, 1, nh, n_kv, hd, max_seq, pos, 5e5, 1.0, 0, 0)
        assert np.array_equal(cache.download(np.uint8), after)
        L.cuda_attn_step_kv4(out2.ptr, q2.ptr, None, None, cache.ptr, nh, n_kv, hd, max_seq, None, pos, 0, scale, None, 0.0, 1.0, 0, 0, -1)
        kk, vv = k[:pos + 1].copy(), v[:pos + 1].copy()
        kk[pos], vv[pos] = kv4.values(k2.download().reshape(1, n_kv, hd))[0], kv4.values(vn)[0]
        want, bound = kv4.attention(q2.download().reshape(1, nh, hd), kk, vv, pos, 0, float(np.float32(scale)), None)
        held(out2.download().reshape(1, nh, hd), want, bound)
        # the rotation may round differently by an ulp where the compiler contracts it: 2^-22 of a score's terms
        assert np.abs(got[0] - out2.download()).max() <= 2.0 ** -18 * np.abs(want).max()
        if L.cuda_gemv_q_supported(8, w.ptr, K):      # the slot holds what cuda_quantize_x makes of the result
            put(gpu, cache, raw)
            L.quartz_graph_launch(graph)
            L.cuda_quantize_x(out.ptr, K, 1)
            for slot, b in ((2, y[0]), (1, y[1])):
                L.cuda_gemv_q(8, 1, (C.c_void_p * 1)(w.ptr), (C.c_int * 1)(slot), (C.c_void_p * 1)(b.ptr), K, N, 0)
            assert np.array_equal(y[0].download(), y[1].download())
    L.quartz_graph_destroy(graph)
    gpu.check_error()


def test_graphs_of_long_caches_side_by_side(gpu):
    """Two captured steps that merge, replayed at the same time on two streams, and two eager ones: each has a workspace of its own."""
    import torch
    L, sets = gpu.lib(), []
    nh, n_kv, hd, max_seq = 16, 4, 128, 9000
    for i in range(2):
        r = rng(51, i)
        cache, _, k, v, q, _, _ = merge_setup(gpu, r, nh, n_kv, hd, max_seq, max_seq)
        out = gpu.GpuBuf.alloc_f32(nh * hd)
        want = kv4.attention(q, k, v, max_seq - 1, 0, float(np.float32(0.09)), None)
        sets.append((cache, upload(gpu, q), out, want, torch.cuda.Stream(), torch.cuda.CUDAGraph()))

    def call(s):
        L.cuda_attn_step_kv4(s[2].ptr, s[1].ptr, None, None, s[0].ptr, nh, n_kv, hd, max_seq, None, max_seq - 1, 0, 0.09, None, 0.0, 1.0, 0, 0, -1)

    def check():
        torch.cuda.synchronize()
        got = [s[2].download() for s in sets]
        for g, s in zip(got, sets):
            held(g.reshape(1, nh, hd), *s[3])
            put(gpu, s[2], np.zeros(nh * hd, np.float32))
        return got
    try:
        for s in sets:
            call(s)
        first = check()
        for s in sets:
            with torch.cuda.graph(s[5], stream=s[4]):
                L.quartz_set_stream(torch.cuda.current_stream().cuda_stream)
                call(s)
            L.quartz_set_stream(None)
        for _ in range(3):
            for _ in range(50):
                for s in sets:
                    with torch.cuda.stream(s[4]):
                        s[5].replay()
            assert all(np.array_equal(a, b) for a, b in zip(check(), first))
            for _ in range(50):
                for s in sets:
                    L.quartz_set_stream(s[4].cuda_stream)
                    call(s)
            L.quartz_set_stream(None)
            assert all(np.array_equal(a, b) for a, b in zip(check(), first))
    finally:
        torch.cuda.synchronize()
        L.quartz_set_stream(None)
    gpu.check_error()


def test_workspaces_of_graphs_that_are_gone_are_used_again(gpu):
    import torch
    L, r = gpu.lib(), rng(52)
    nh, n_kv, hd, max_seq = 16, 4, 128, 9000
    cache, _, k, v, q, _, _ = merge_setup(gpu, r, nh, n_kv, hd, max_seq, max_seq)
    dq, out = upload(gpu, q), gpu.GpuBuf.alloc_f32(nh * hd)
    want = kv4.attention(q, k, v, max_seq - 1, 0, float(np.float32(0.09)), None)
    free = []
    for i in range(200):
        assert L.quartz_graph_begin()
        L.cuda_attn_step_kv4(out.ptr, dq.ptr, None, None, cache.ptr, nh, n_kv, hd, max_seq, None, max_seq - 1, 0, 0.09, None, 0.0, 1.0, 0, 0, -1)
        graph = L.quartz_graph_end()
        put(gpu, out, np.zeros(nh * hd, np.float32))
        for _ in range(3):
            L.quartz_graph_launch(graph)
        held(out.download().reshape(1, nh, hd), *want)
        L.quartz_graph_destroy(graph)
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
    # 195 workspaces of their own, 4 * (128 * 32 + 128 * 32 * 34) bytes each, would take 107 MiB; the driver's own pools take chunks
    # of some MiB at times (8 were seen)
    assert free[4] - free[-1] <= 32 << 20
    gpu.check_error()


# ---- groups and positions of very different sizes ----------------------------------------------------------------
def test_step_groups_far_apart_are_each_as_accurate(gpu):
    """Groups whose values lie up to 2^20 below another's: each is held to its own size."""
    L = gpu.lib()
    for nh, n_kv, exps in ((4, 1, (0, -9, -16, -20)), (8, 1, (-20, 0, -12, 3)), (6, 3, (-18, 0)), (16, 2, (0, -15, -20))):
        r, hd, ctx = rng(40, nh), 32 * len(exps), 200
        k, v = rows(r, ctx, n_kv, hd, False), rows(r, ctx, n_kv, hd, False)
        v *= np.exp2(np.array(exps, np.float32)).repeat(32)
        cache = upload(gpu, kv4.store(np.zeros(kv4.nbytes(ctx, n_kv, hd), np.uint8), k, v, 0, ctx))
        out, scale = gpu.GpuBuf.alloc_f32(nh * hd), float(np.float32(hd ** -0.5))
        for sharp in (1e-20, 1.0, 8.0):
            q = r.standard_normal((1, nh, hd), dtype=np.float32) * np.float32(sharp)
            dq = upload(gpu, q)
            L.cuda_attn_step_kv4(out.ptr, dq.ptr, None, None, cache.ptr, nh, n_kv, hd, ctx, None, ctx - 1, 0, scale, None, 0.0, 1.0, 0, 0, -1)
            kk, vv = kv4.values(k), kv4.values(v)
            want, bound = kv4.attention(q, kk, vv, ctx - 1, 0, scale, None)
            # A value is p d (code - 8) + p (m + 8 d); with A the larger end of a group's range 15 d <= 2 A, so the two are at most
            # 16 / 15 A and A.  Each carries 22 bits and one f32 rounding: (31 / 15) 1.25 2^-22 A < 2^-20 A a position, taken with
            # the weights.  p d itself: |code - 8| 2^-35 of the group's largest step D at most, 2^-32 D a position, the largest weight
            # of all being 1.
            A = np.abs(vv.reshape(ctx, n_kv, -1, 32)).max(-1).repeat(32, -1)
            D = kv4.quantise(v)[2].max(0).repeat(32, -1).repeat(nh // n_kv, 0)
            own = 2.0 ** -20 * kv4.attention(q, kk, A, ctx - 1, 0, scale, None)[0] + ctx * 2.0 ** -32 * D
            err = np.abs(out.download().reshape(1, nh, hd) - want)
            assert (err <= bound + own).all(), (nh, sharp, (err / (bound + own)).max())
            # and in the norm, group by group, as the other tests hold all of them together
            by = lambda x: np.linalg.norm(x.reshape(nh, -1, 32), axis=(0, 2))
            assert (by(err) <= 2.0 ** -19 * by(want)).all(), (nh, sharp, by(err) / by(want))
    gpu.check_error()


def test_step_position_far_above_the_others(gpu):
    """One position's values are 2^16 times the others' and its weight is next to nothing: the others keep their bits.  A position's error
    in p d is two roundings to 2^-24 of a scale on which the largest step D is at least 2^11, uniform: 2^-24 0.41 / 2^11 D with codes of 4.6 on
    average, 2^-34 D; that of n positions over the sum l of their weights sqrt(n) 2^-34 D / l.  Twice that, beside 2^-20 of the output."""
    L, r = gpu.lib(), rng(41)
    nh, n_kv, hd, ctx, scale = 4, 1, 128, 200, float(np.float32(0.0883))
    for at in (0, 17, 199):
        k, v = np.abs(rows(r, ctx, n_kv, hd, False)), rows(r, ctx, n_kv, hd, False)
        k[at] = -3
        v[at] *= 2.0 ** 16
        q = np.full((1, nh, hd), 0.5, np.float32)
        cache = upload(gpu, kv4.store(np.zeros(kv4.nbytes(ctx, n_kv, hd), np.uint8), k, v, 0, ctx))
        dq, out = upload(gpu, q), gpu.GpuBuf.alloc_f32(nh * hd)
        L.cuda_attn_step_kv4(out.ptr, dq.ptr, None, None, cache.ptr, nh, n_kv, hd, ctx, None, ctx - 1, 0, scale, None, 0.0, 1.0, 0, 0, -1)
        kk, vv = kv4.values(k), kv4.values(v)
        want, _ = kv4.attention(q, kk, vv, ctx - 1, 0, scale, None)
        s = kk[:, 0].astype(np.float64) @ q[0, 0] * scale
        l = np.exp(s - s.max()).sum()
        D = kv4.quantise(v)[2].max(0).repeat(32, -1).repeat(nh, 0)
        err = out.download().reshape(1, nh, hd) - want
        allowed = 2 * np.linalg.norm(np.sqrt(ctx) * 2.0 ** -34 * D / l) + 2.0 ** -20 * np.linalg.norm(want)
        assert np.linalg.norm(err) <= allowed, (at, np.linalg.norm(err) / allowed, np.linalg.norm(err) / np.linalg.norm(want))
    gpu.check_error()


def test_rows_of_subnormal_numbers(gpu):
    """Ranges of a few f32 subnormals: the step is the smallest one, not none."""
    L, r = gpu.lib(), rng(42)
    tiny = np.float32(2.0 ** -149)
    x = np.zeros((70, 1, 32), np.float32)
    for i in range(10):
        x[i, 0, 3 * i] = (i + 1) * tiny
        x[10 + i, 0, i] = -(i + 1) * tiny
        x[20 + i, 0] = r.integers(0, 2 ** i + 1, 32).astype(np.float32) * tiny
    x[30] = np.float32(2.0 ** -24)
    x[30, 0, 5] = np.nextafter(np.float32(2.0 ** -24), np.float32(1))
    for i in range(31, 70):
        x[i, 0] = (r.standard_normal(32) * 2.0 ** -r.integers(100, 149)).astype(np.float32)
    raw = np.full(kv4.nbytes(70, 1, 32), 7, np.uint8)
    cache, dk, dv = upload(gpu, raw), upload(gpu, x), upload(gpu, x[::-1])
    L.cuda_kv4_append_rows(cache.ptr, dk.ptr, dv.ptr, 70, 1, 32, 70, 0)
    gpu.check_error()
    assert np.array_equal(cache.download(np.uint8), kv4.store(raw, x, x[::-1], 0, 70))
    ok, ov = gpu.GpuBuf.alloc_f32(x.size), gpu.GpuBuf.alloc_f32(x.size)
    L.cuda_kv4_read_rows(ok.ptr, ov.ptr, cache.ptr, 70, 1, 32, 70, 0)
    for got, want in ((ok, x), (ov, x[::-1])):
        assert np.array_equal(got.download(), kv4.values(want).reshape(-1))
        step = kv4.quantise(want)[2].repeat(32, -1).reshape(-1)
        assert (np.abs(got.download().astype(np.float64) - want.reshape(-1)) <= step / 2).all()


def test_many_streams_that_come_and_go(gpu):
    """Forty streams with calls that merge in flight at once, then two hundred that are destroyed with their call still running (their
    handles come back): every result is right, and what the library keeps does not grow with them."""
    import torch
    from cuda.bindings import runtime as rt
    L, r = gpu.lib(), rng(53)
    nh, n_kv, hd, max_seq, n = 16, 4, 128, 9000, 40

    def new():
        err, s = rt.cudaStreamCreateWithFlags(rt.cudaStreamNonBlocking)
        assert err == rt.cudaError_t.cudaSuccess
        return int(s)
    cache, _, k, v, _, _, _ = merge_setup(gpu, r, nh, n_kv, hd, max_seq, max_seq)
    q = r.standard_normal((n, nh, hd), dtype=np.float32)
    dq, out, want = [upload(gpu, x) for x in q], [gpu.GpuBuf.alloc_f32(nh * hd) for _ in q], []

    def call(i):
        L.cuda_attn_step_kv4(out[i].ptr, dq[i].ptr, None, None, cache.ptr, nh, n_kv, hd, max_seq, None, max_seq - 1, 0, 0.09, None, 0.0, 1.0, 0, 0, -1)

    def check():
        torch.cuda.synchronize()
        for i in range(n):
            assert np.array_equal(out[i].download(), want[i]), i
            put(gpu, out[i], np.zeros(nh * hd, np.float32))
    for i in range(n):
        call(i)
        want.append(out[i].download())
    held(want[3].reshape(1, nh, hd), *kv4.attention(q[3:4], k, v, max_seq - 1, 0, float(np.float32(0.09)), None))
    streams = [new() for _ in range(n)]
    try:
        for _ in range(5):
            for _ in range(10):
                for i, s in enumerate(streams):
                    L.quartz_set_stream(s)
                    call(i)
            L.quartz_set_stream(None)
            check()
        free = torch.cuda.mem_get_info()[0]
        for turn in range(5):
            for i in range(n):
                s = new()
                L.quartz_set_stream(s)
                for _ in range(3):
                    call(i)
                rt.cudaStreamDestroy(s)
            L.quartz_set_stream(None)
            check()
        # 200 workspaces would be 109 MiB
        assert free - torch.cuda.mem_get_info()[0] <= 32 << 20
    finally:
        torch.cuda.synchronize()
        L.quartz_set_stream(None)
        for s in streams:
            rt.cudaStreamDestroy(s)
    gpu.check_error()


def test_prompt_groups_far_apart_are_each_as_accurate(gpu):
    """Tiles with steps above 8188 in one group, of the values or of the keys: the small groups beside it are held to their own size."""
    L = gpu.lib()
    for nh, n_kv, hd, n in ((16, 8, 128, 515), (12, 6, 96, 515), (8, 4, 64, 700)):
        r, g, scale = rng(43, hd), hd // 32, float(np.float32(hd ** -0.5))
        k, v = rows(r, n, n_kv, hd, False), rows(r, n, n_kv, hd, False)
        v[..., 32:] *= np.float32(2.0 ** -8)
        v[100:400:37, :, :32] = np.linspace(-65504, 65504, 32)     # a step of 8734
        k[90:420:55, :, :32] = np.linspace(65504, -65504, 32)
        k[..., 32:] *= np.float32(2.0 ** -2)
        q = r.standard_normal((n, nh, hd), dtype=np.float32) * 4
        q[..., :32] = 0                          # (the towering keys weigh nothing: the others decide)
        cache = upload(gpu, kv4.store(np.full(kv4.nbytes(n, n_kv, hd), 0xFF, np.uint8), k, v, 0, n))
        dq, out = upload(gpu, q), gpu.GpuBuf.alloc_f32(q.size)
        L.cuda_attn_prompt_kv4(out.ptr, dq.ptr, cache.ptr, n, nh, n_kv, hd, n, 0, 0, scale, None)
        got = out.download().reshape(q.shape)
        gpu.check_error()
        kk, vv = kv4.values(k), kv4.values(v)
        want, bound = kv4.attention(q, kk, vv, 0, 0, scale, None)
        # bound: its score error is that of the largest key, here one that q does not touch; so that of the dims q has
        e_s = (np.abs(q[..., 32:]).sum(-1) * np.abs(kk[..., 32:]).max() * scale * (hd + 16) * 2.0 ** -23)[..., None]
        # A: the larger end of a group's range, weighed: 2^-20 of it for the two terms of a value, which may cancel; the weights' errors
        # 4 e_s and n 2^-22 of |value| <= A.  (An eighth of a step or minimum is exact down to 2^-11: the small groups' are above that.)
        A = np.abs(vv.reshape(n, n_kv, g, 32)).max(-1).repeat(32, -1)
        own = kv4.attention(q, kk, A, 0, 0, scale, None)[0]
        allowed = own * (2.0 ** -20 + 4 * e_s + (np.arange(n)[:, None, None] + 33) * 2.0 ** -22)
        err = np.abs(got - want)[..., 32:]
        assert (err <= allowed[..., 32:]).all(), (hd, (err / allowed[..., 32:]).max())
        # and in the norm, as the other tests hold all groups together
        assert np.linalg.norm(err) <= 2.0 ** -19 * np.linalg.norm(want[..., 32:]), np.linalg.norm(err) / np.linalg.norm(want[..., 32:])
        assert (np.abs(got - want) <= bound + 2.0 ** -20 * np.maximum.accumulate(np.abs(vv).max(-1), 0).repeat(nh // n_kv, 1)[..., None]).all()
    gpu.check_error()


@pytest.mark.parametrize("mass", [0.5, 0.99])
@pytest.mark.parametrize("nh,n_kv,hd", [(32, 8, 128), (8, 2, 64), (12, 6, 96)])
def test_many_small_weights_beside_a_large_one(gpu, nh, n_kv, hd, mass):
    """The first position takes most of the mass and has no values, as in trained models; the outputs are the sum of the others' small
    weights, 2^-17 of the largest at the end.

    In the norm: 2^-19 of the output for independent errors of some 2^-22 a term, as elsewhere.  The output is a mean of n values of
    both signs here, 1 / sqrt(n) = 0.03 of the sums of p m and of 8 p d that it is made of (about -2 and 2.1 times the sum s of p): what
    errs in these with one sign weighs 33 times as much.  The tensor core rounds towards zero, 12 steps of half an ulp on a sum that grows from nothing: 3 2^-23
    of either, with opposite signs, 3 2^-23 of their difference of 0.1 s together = 3.6e-8 s, 1.2e-6 of the output.  With 2^-19 = 1.9e-6
    that is 3.1e-6 < 2^-18."""
    L, r = gpu.lib(), rng(44, nh)
    n, scale = 1100, float(np.float32(hd ** -0.5))
    k, v = rows(r, n, n_kv, hd, False), rows(r, n, n_kv, hd, False)
    k[..., 0] = 0
    k[0, :, :] = 0
    k[0, :, 0] = np.log(mass / (1 - mass) * n) / (8 * scale)
    v[0] = 0
    q = r.standard_normal((n, nh, hd), dtype=np.float32) * np.float32(0.2)
    q[..., 0] = 8
    cache = upload(gpu, kv4.store(np.full(kv4.nbytes(n, n_kv, hd), 0xFF, np.uint8), k, v, 0, n))
    dq, out = upload(gpu, q), gpu.GpuBuf.alloc_f32(q.size)
    L.cuda_attn_prompt_kv4(out.ptr, dq.ptr, cache.ptr, n, nh, n_kv, hd, n, 0, 0, scale, None)
    got = out.download().reshape(q.shape)
    want, bound = kv4.attention(q, kv4.values(k), kv4.values(v), 0, 0, scale, None)

    def near(a, b, bound):
        assert (np.abs(a - b) <= bound).all()
        assert np.linalg.norm(a - b) <= 2.0 ** -18 * np.linalg.norm(b), np.linalg.norm(a - b) / np.linalg.norm(b)
    near(got, want, bound)
    for t in (n - 1, n // 2):
        near(got[t], want[t], bound[t])
        one = upload(gpu, q[t])
        L.cuda_attn_step_kv4(out.ptr, one.ptr, None, None, cache.ptr, nh, n_kv, hd, n, None, t, 0, scale, None, 0.0, 1.0, 0, 0, -1)
        near(out.download(count=nh * hd).reshape(nh, hd), want[t], bound[t])
    gpu.check_error()
