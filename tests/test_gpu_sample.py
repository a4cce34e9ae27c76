"""GPU tests of the device-side sampler against the 64-bit numpy form in oracle/sampling.py.  Tokens are equal.  A
probability is one rounding to f32 of quotients of weights that are right to 2^-29, and off by the unit of 2^-44 to which
weights are rounded down, the largest weight being 1: 2^-23 relative and 2^-44."""
import numpy as np
import pytest

from oracle import sampling

pytestmark = pytest.mark.gpu

SETTINGS = [dict(), dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.05), dict(top_p=0.9), dict(top_k=1), dict(top_k=5, temperature=2.5),
            dict(min_p=0.1), dict(temperature=0.05), dict(temperature=0.0), dict(top_k=1000, top_p=0.5), dict(top_p=1e-6), dict(top_p=0.0),
            dict(min_p=1.0), dict(min_p=7.0), dict(temperature=1e-30), dict(temperature=1e30, top_p=0.3), dict(top_k=3, top_p=0.999, min_p=1e-4)]


def rng(*seed):
    return np.random.Generator(np.random.PCG64([0x5A3B, *seed]))


def put(gpu, buf, a):
    a = np.ascontiguousarray(a)
    gpu.lib().cuda_h2d(buf.ptr, a.ctypes.data, a.nbytes)


def call(gpu, z, u, ld=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, probs=True):
    L = gpu.lib()
    n, vocab = z.shape
    ld = ld or vocab
    wide = np.full((n, ld), 1e30, np.float32)      # what lies between the rows is not read
    wide[:, :vocab] = z
    dz, du = gpu.GpuBuf.upload(wide), gpu.GpuBuf.upload(np.asarray(u, np.float32))
    dt, dp = gpu.GpuBuf.upload(np.full(n + 4, -77, np.int32)), gpu.GpuBuf.upload(np.full(n + 4, -7, np.float32))
    L.cuda_sample(dz.ptr, n, vocab, ld, temperature, top_k, top_p, min_p, du.ptr, dt.ptr, dp.ptr if probs else None)
    tok, p = dt.download(np.int32), dp.download()
    gpu.check_error()
    assert (tok[n:] == -77).all() and (p[n if probs else 0:] == -7).all()
    return tok[:n], p[:n]


def check(gpu, z, u, ld=None, **kw):
    tok, p = call(gpu, z, u, ld, **kw)
    want = [sampling.sample(row, x, **kw) for row, x in zip(z, np.asarray(u, np.float32))]
    assert list(tok) == [w[0] for w in want], kw
    wp = np.array([w[1] for w in want])
    assert (np.abs(p - wp) <= 2.0 ** -23 * wp + 2.0 ** -44).all(), kw
    return tok


@pytest.mark.parametrize("kw", SETTINGS)
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1025, 5003])
def test_settings(gpu, vocab, kw):
    r = rng(vocab, len(kw))
    z = (r.standard_normal((9, vocab)) * 2.5).astype(np.float32)
    u = r.random(9)
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    check(gpu, z, u, ld=vocab + (vocab % 7), **kw)


@pytest.mark.parametrize("rows,vocab", [(1, 128256), (2, 32000), (3, 151937), (17, 50257), (40, 128256), (150, 8191), (1, 524288), (2, 400001)])
def test_vocabularies(gpu, rows, vocab):
    r = rng(rows, vocab)
    z = (r.standard_normal((rows, vocab)) * 3).astype(np.float32)
    for kw in SETTINGS[:4]:
        check(gpu, z, r.random(rows), **kw)


@pytest.mark.parametrize("kw", SETTINGS)
def test_ties(gpu, kw):
    """Logits on a coarse grid (a 16-bit head), all equal, two values, and the two zeros, which are one value."""
    r = rng(4)
    z = [np.round(r.standard_normal(3001) * 8) / 4, np.zeros(3001), np.where(r.random(3001) < 0.01, 2.0, 1.0), np.where(r.random(3001) < 0.5, 0.0, -0.0),
         np.full(3001, -1e30), np.where(np.arange(3001) == 2999, 1.0, 1 - 2.0 ** -24)]
    z = np.array(z, np.float32)
    for _ in range(3):
        check(gpu, z, r.random(len(z)), **kw)


def test_masked_and_odd_logits(gpu):
    """-inf, NaN, the lowest f32 and +inf; rows with nothing left; subnormal and huge logits."""
    r = rng(5)
    base = (r.standard_normal(2500) * 3).astype(np.float32)
    z = np.tile(base, (12, 1))
    z[0] = -np.inf
    z[1] = np.nan
    z[2, :] = -np.inf
    z[2, 1234] = -5.0
    z[3, ::2] = -np.inf
    z[4, 7::3] = np.nan
    z[5, ::2] = np.finfo(np.float32).min
    z[6] = np.finfo(np.float32).min
    z[7, [5, 900, 901]] = np.inf
    z[8] *= np.float32(1e-42)
    z[9] *= np.float32(1e37)
    z[10, :] = np.nan
    z[10, 2499] = np.inf
    z[11, :] = -np.inf
    z[11, ::1000] = np.finfo(np.float32).min
    for kw in SETTINGS:
        for _ in range(2):
            check(gpu, z, r.random(12), **kw)


@pytest.mark.parametrize("vocab", [700, 9001, 128256, 400001])
def test_a_prefix_that_reaches_top_p_exactly(gpu, vocab):
    """Some equal logits and the rest so far below that it weighs nothing (each token less than a unit of 2^-44, as the call defines its
    weights): half of the equal ones reach one half, no token more."""
    r = rng(12)
    for far in (-1000.0, -60.0, -41.0, -28.0):
        for n, parts in ((2, (0.5,)), (4, (0.25, 0.5, 0.75)), (8, (0.125, 0.625)), (64, (0.5, 0.25))):
            z = np.full((4, vocab), far, np.float32)
            for row in z:
                row[r.choice(vocab, n, replace=False)] = 3.0
            for p in parts:
                for kw in (dict(), dict(top_k=650), dict(top_k=n), dict(min_p=1e-3)):
                    tok, probs = call(gpu, z, [0.0, 0.3, 0.7, 1 - 2.0 ** -24], top_p=p, **kw)
                    want = [sorted(np.flatnonzero(row == 3.0)[:int(n * p)]) for row in z]
                    at = [0, int(0.3 * n * p), int(0.7 * n * p), int(n * p) - 1]
                    assert list(tok) == [w[i] for w, i in zip(want, at)], (far, n, p, kw)
                    assert (np.abs(probs - 1 / (n * p)) <= 2.0 ** -23).all()


@pytest.mark.parametrize("t", [1.4e-45, 1e-44, 1e-40, 1e-38, 1.3e-37, 1e-36, 1e30, 1e37, 3.4e38])
def test_temperatures_at_the_ends(gpu, t):
    """Logits of the temperature's own size, near both ends of f32: their quotients are ordinary numbers."""
    r = rng(11)
    for vocab in (40, 3000, 30001):
        z = (r.standard_normal((5, vocab)) * 2.5 * np.float64(np.float32(t))).clip(-1.5e38, 1.5e38).astype(np.float32)
        z[2] += z[2].max()
        for kw in (dict(), dict(top_k=7), dict(top_p=0.8), dict(min_p=0.05), dict(top_k=700, top_p=0.9, min_p=0.01)):
            check(gpu, z, r.random(5), temperature=t, **kw)


def test_random_numbers_at_the_ends(gpu):
    r = rng(6)
    z = (r.standard_normal((6, 900)) * 2).astype(np.float32)
    for kw in SETTINGS[:6]:
        tok, _ = call(gpu, z, [0.0, -3.0, np.nan, 1.0, 2.0, 1 - 2.0 ** -24], **kw)
        want = [sampling.sample(row, u, **kw)[0] for row, u in zip(z, (0, 0, 0, 1, 1, np.float32(1 - 2.0 ** -24)))]
        assert list(tok) == want


def test_same_answer_however_the_rows_are_batched(gpu):
    r = rng(7)
    z = (r.standard_normal((64, 20011)) * 2.5).astype(np.float32)
    u = r.random(64)
    kw = dict(temperature=0.9, top_k=200, top_p=0.9)
    tok, p = call(gpu, z, u, **kw)
    for lo, hi in ((0, 1), (3, 4), (10, 18), (20, 57)):
        t2, p2 = call(gpu, z[lo:hi], u[lo:hi], **kw)
        assert np.array_equal(t2, tok[lo:hi]) and np.array_equal(p2, p[lo:hi])
    assert np.array_equal(call(gpu, z, u, probs=False, **kw)[0], tok)


def test_many_clusters_at_once(gpu):
    """Rows of two and four CTAs in far more clusters than the device holds at once: the CTAs of a cluster start at different times,
    and write to one another's shared memory only once all of them run.  Every row against the oracle, several times over."""
    r = rng(10)
    for rows, vocab in ((700, 20003), (300, 60007)):
        z = (r.standard_normal((rows, vocab), dtype=np.float32) * 3)
        u = r.random(rows)
        for kw in (dict(temperature=0.0), dict(top_k=3, temperature=0.7), dict(top_p=0.8)):
            tok = check(gpu, z, u, **kw)
            for _ in range(3):
                assert np.array_equal(call(gpu, z, u, **kw)[0], tok)


def test_frequencies(gpu):
    """10,000 draws from eight tokens: a token's count is binomial; six standard deviations (2e-9 a token)."""
    p = np.array([0.3, 0.2, 0.15, 0.1, 0.1, 0.08, 0.05, 0.02])
    n = 10000
    tok, _ = call(gpu, np.tile(np.log(p).astype(np.float32), (n, 1)), rng(8).random(n))
    count = np.bincount(tok, minlength=8)
    assert (np.abs(count - n * p) <= 6 * np.sqrt(n * p * (1 - p))).all()


def test_recorded_with_the_step_words(gpu):
    """cuda_sample then cuda_step_advance in one recording, replayed: token and position follow, a row without a
    token leaves the token word alone, and the rotation table is the one that cuda_step_set writes."""
    L, r = gpu.lib(), rng(9)
    vocab = 4097
    z = (r.standard_normal((1, vocab)) * 2).astype(np.float32)
    dz, du = gpu.GpuBuf.upload(z), gpu.GpuBuf.upload(np.array([0.5], np.float32))
    step, tok = gpu.GpuBuf.alloc_f32(4), gpu.GpuBuf.upload(np.array([-9], np.int32))
    L.cuda_step_rope_table(step.ptr, 64, 1e4, 1.0, 0)
    L.cuda_step_set(step.ptr, 11, 40)
    assert L.quartz_graph_begin()
    L.cuda_sample(dz.ptr, 1, vocab, vocab, 0.8, 30, 0.9, 0.0, du.ptr, tok.ptr, None)
    L.cuda_step_advance(step.ptr, tok.ptr)
    graph = L.quartz_graph_end()
    assert graph
    for i in range(5):
        u = np.float32(r.random())
        put(gpu, du, np.array([u], np.float32))
        L.quartz_graph_launch(graph)
        want = sampling.sample(z[0], u, temperature=0.8, top_k=30, top_p=0.9)[0]
        assert list(step.download(np.int32, 2)) == [want, 41 + i] and tok.download(np.int32)[0] == want
    last = want
    put(gpu, dz, np.full(vocab, -np.inf, np.float32))
    L.quartz_graph_launch(graph)
    assert list(step.download(np.int32, 2)) == [last, 46] and tok.download(np.int32)[0] == -1
    L.quartz_graph_destroy(graph)
    gpu.check_error()
