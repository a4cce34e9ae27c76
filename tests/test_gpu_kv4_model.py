"""GPU tests of a whole model on the 4-bit KV cache and of the generation loop on the device, through the C++ host.

Bar for logits: 5e-3 of the largest against the CPU forward whose cache holds the quantised values, as for f32 caches.
Single codes may differ where the CPU's projection lies on the border between two (each moves one value by a step of its
group); the cache rows are held to that: no value more than one step away, at most one in 200 away at all."""
import numpy as np
import pytest

from oracle import kv4, sampling

pytestmark = pytest.mark.gpu


def _rel(a, b):
    return float(np.abs(a.astype(np.float64) - b).max() / max(np.abs(b).max(), 1e-30))


def _model(kv_bits=4, types=None, extra=None, **over):
    from saient_quartz_b200.host_model import HostModel, Q4K_M_TYPES
    cfg = dict(vocab_size=320, embed_dim=2048, n_heads=16, n_kv_heads=4, n_layers=3, ffn_dim=4096, head_dim=128, rope_theta=500000.0, max_seq=120)
    cfg.update(over)
    m = HostModel(keep_host=True, types=types or Q4K_M_TYPES, kv_bits=kv_bits, **cfg)
    for role, layer, a in extra or []:
        m.set(role, layer, 0, a)
    m.fill_synthetic()
    return m


def _ref(m, n_pos):
    from oracle.forward_ref import RefModel
    hd = m.cfg["head_dim"]

    class Cached(RefModel):
        def cached(self, x):
            return kv4.values(x.reshape(-1, hd)).reshape(-1)
    r = Cached(m.cfg, m.host)
    for l in range(m.cfg["n_layers"]):
        if n_pos:
            r.set_kv(l, *m.read_kv(l, 0, n_pos))
    return r


def _rows_match(m, ref, pos):
    hd = m.cfg["head_dim"]
    for l in range(m.cfg["n_layers"]):
        for got, want in zip(m.read_kv(l, pos, 1), ref.kv[l]):
            g, w = got.reshape(-1, 32), want[pos].reshape(-1, 32)
            step = (w.max(1, keepdims=True) - w.min(1, keepdims=True)) / 10 + 1e-6     # (a step is at least a 15th of the range)
            assert (np.abs(g - w) <= step).all() and np.mean(np.abs(g - w) > 0.02 * step) <= 0.005, (l, hd)


@pytest.mark.parametrize("kw", [dict(), dict(rope_neox=1), dict(swa_window=16), dict(embed_dim=512, n_heads=8, n_kv_heads=2, head_dim=64, ffn_dim=1024,
                                types=dict(Q=12, K=12, V=12, O=12, GATE=12, UP=12, DOWN=8, LM_HEAD=8, EMBED=14))])
def test_sequences_against_the_cpu_forward(gpu, oracle_mod, kw):
    m = _model(**kw)
    kv = m.fill_kv(40, keep=True)
    for l, (k, v) in enumerate(kv):      # written through the quantiser
        hd = m.cfg["head_dim"]
        for got, want in zip(m.read_kv(l, 0, 40), (k, v)):
            assert np.array_equal(got, kv4.values(want.reshape(40, -1, hd)).reshape(40, -1))
    ref = _ref(m, 40)
    for pos, tok in ((40, 17), (41, 300), (42, 0)):
        want = ref.forward(tok, pos)
        plain = m.step(tok, pos, fused=False)
        assert _rel(plain, want) < 5e-3
        _rows_match(m, ref, pos)
        for seq in (1, 2):
            got = m.step(tok, pos, fused=seq)
            assert _rel(got, want) < 5e-3 and _rel(got, plain) < 2e-3, seq
    assert m.H.qh_kv_bits(m.m) == 4
    gpu.check_error()


def test_biases_and_qk_norm_take_the_reference_sequence(gpu, oracle_mod):
    """Models that the fused sequence does not serve: rotation by its own launch, then attention without one."""
    r = np.random.Generator(np.random.PCG64(3))
    extra = [("Q_BIAS", 0, r.standard_normal(2048).astype(np.float32)), ("K_BIAS", 0, r.standard_normal(512).astype(np.float32)),
             ("Q_NORM", 1, np.ones(128, np.float32) * 1.1), ("K_NORM", 1, np.ones(128, np.float32) * 0.9),
             ("SINKS", 2, r.standard_normal(16).astype(np.float32))]
    m = _model(extra=extra)
    m.fill_kv(20)
    ref = _ref(m, 20)
    for pos, tok in ((20, 5), (21, 6)):
        want = ref.forward(tok, pos)
        assert _rel(m.step(tok, pos, fused=True), want) < 5e-3
    gpu.check_error()


def test_prefill_equals_steps(gpu, oracle_mod):
    m = _model()
    toks = list(np.random.Generator(np.random.PCG64(8)).integers(0, 320, 45))
    got = m.prefill(toks)
    rows = [m.read_kv(l, 0, 45) for l in range(3)]
    ref = _ref(m, 0)
    for i, t in enumerate(toks):
        want = ref.forward(int(t), i)
    assert _rel(got, want) < 2e-2      # bf16 projections of the batched pass, as with f32 caches
    s = _model()
    for i, t in enumerate(toks):
        step = s.step(int(t), i, fused=True)
    assert _rel(step, want) < 5e-3
    assert [r[0].shape for r in rows] == [(45, 512)] * 3
    # a second turn on top of the first
    more = m.prefill([3, 4, 5, 6, 7], pos0=45)
    for i, t in enumerate([3, 4, 5, 6, 7]):
        want = ref.forward(t, 45 + i)
    assert _rel(more, want) < 2e-2
    gpu.check_error()


@pytest.mark.parametrize("kv_bits", [4, 32])
@pytest.mark.parametrize("kw", [dict(temperature=0.0), dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.02), dict(temperature=1.3, top_p=0.7)])
def test_generate_equals_steps_and_the_oracle_sampler(gpu, oracle_mod, kv_bits, kw):
    """Tokens chosen in the loop on the device = stepping from the host and sampling its logits in 64 bits."""
    m = _model(kv_bits=kv_bits)
    m.fill_kv(30)
    n, u = 24, np.random.Generator(np.random.PCG64(5)).random(24).astype(np.float32)
    got = m.generate(7, 30, n, u=u, **kw)
    assert m.graphs_recorded() == 1
    tok, want = 7, []
    for i in range(n):
        z = m.step(tok, 30 + i, fused=True)
        tok = sampling.sample(z, u[i], **kw)[0]
        want.append(tok)
    assert list(got) == want
    assert list(m.generate(7, 30, n, u=u, **kw)) == want      # again, on the recorded graph
    gpu.check_error()


def test_a_replay_is_ordered_with_the_stream_that_is_set(gpu):
    """On a non-blocking stream held up by a long kernel: what is issued before a replay runs before it, what follows after it."""
    import torch
    L, n = gpu.lib(), 1 << 16
    a, b, c = (gpu.GpuBuf.upload(np.full(n, x, np.float32)) for x in (5.0, 3.0, 0.0))
    L.quartz_set_stream(None)
    assert L.quartz_graph_begin()
    L.cuda_vec_add(a.ptr, b.ptr, n)          # a += 3
    graph = L.quartz_graph_end()
    st = torch.cuda.Stream()
    L.quartz_set_stream(st.cuda_stream)
    try:
        with torch.cuda.stream(st):
            torch.cuda._sleep(100_000_000)
            L.cuda_vec_zero(a.ptr, n)
            L.quartz_graph_launch(graph)     # a = 3
            L.quartz_graph_launch(graph)     # a = 6
            L.cuda_vec_add(c.ptr, a.ptr, n)  # c = 6
            L.quartz_graph_launch(graph)     # a = 9
        st.synchronize()                     # waits for the last replay as well
    finally:
        L.quartz_set_stream(None)
    assert (a.download() == 9).all() and (c.download() == 6).all()
    L.quartz_graph_destroy(graph)
    gpu.check_error()


def test_a_replay_inside_a_capture_is_refused(gpu):
    """In the library's own recording and in one of the caller's stream: nothing is launched, and what is captured stays whole."""
    import torch
    L, n = gpu.lib(), 1 << 10
    a, b = (gpu.GpuBuf.upload(np.full(n, x, np.float32)) for x in (5.0, 3.0))

    def refused():
        assert L.quartz_last_error() == 2 and b"captured" in L.quartz_error_string()
        L.quartz_clear_error()
    assert L.quartz_graph_begin()
    L.cuda_vec_add(a.ptr, b.ptr, n)
    graph = L.quartz_graph_end()
    assert L.quartz_graph_begin()
    L.quartz_graph_launch(graph)
    L.cuda_vec_add(a.ptr, b.ptr, n)
    other = L.quartz_graph_end()
    assert other
    refused()
    L.quartz_graph_launch(other)
    assert (a.download() == 8).all()
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(g, stream=st):
            L.quartz_set_stream(torch.cuda.current_stream().cuda_stream)
            L.cuda_vec_add(a.ptr, b.ptr, n)
            L.quartz_graph_launch(graph)
            L.cuda_vec_add(a.ptr, b.ptr, n)
    finally:
        L.quartz_set_stream(None)
    refused()
    g.replay()
    torch.cuda.synchronize()
    assert (a.download() == 14).all()
    L.quartz_graph_launch(graph)
    assert (a.download() == 17).all()
    for x in (graph, other):
        L.quartz_graph_destroy(x)
    gpu.check_error()


@pytest.mark.parametrize("kv_bits", [4, 32])
def test_generate_on_a_stream_of_the_callers(gpu, oracle_mod, kv_bits):
    import torch
    L, n = gpu.lib(), 24
    m = _model(kv_bits=kv_bits)
    m.fill_kv(30)
    u = np.random.Generator(np.random.PCG64(6)).random(n).astype(np.float32)
    kw = dict(temperature=1.1, top_k=50, top_p=0.9, u=u)
    want = list(m.generate(7, 30, n, **kw))
    step = m.step(9, 40, fused=True)
    try:
        for st in (torch.cuda.Stream(), torch.cuda.Stream()):
            L.quartz_set_stream(st.cuda_stream)
            for _ in range(3):
                assert list(m.generate(7, 30, n, **kw)) == want
            assert np.array_equal(m.step(9, 40, fused=True), step)
        fresh = _model(kv_bits=kv_bits)      # recorded while the stream is set
        fresh.fill_kv(30)
        assert list(fresh.generate(7, 30, n, **kw)) == want
    finally:
        torch.cuda.synchronize()
        L.quartz_set_stream(None)
    gpu.check_error()


def test_generate_without_the_fused_sequence(gpu, oracle_mod):
    r = np.random.Generator(np.random.PCG64(4))
    m = _model(extra=[("Q_BIAS", 0, r.standard_normal(2048).astype(np.float32))])
    m.fill_kv(10)
    u = r.random(6).astype(np.float32)
    got = m.generate(7, 10, 6, temperature=0.9, top_k=20, u=u)
    tok, want = 7, []
    for i in range(6):
        tok = sampling.sample(m.step(tok, 10 + i, fused=True), u[i], temperature=0.9, top_k=20)[0]
        want.append(tok)
    assert list(got) == want
    gpu.check_error()


def test_bits_from_the_environment(gpu, oracle_mod, monkeypatch):
    monkeypatch.setenv("QUARTZ_KV_BITS", "4")
    assert [m.H.qh_kv_bits(m.m) for m in (_model(kv_bits=32, n_layers=1), _model(kv_bits=4, n_layers=1))] == [4, 4]
    monkeypatch.delenv("QUARTZ_KV_BITS")
    m = _model(kv_bits=32, n_layers=1)
    assert m.H.qh_kv_bits(m.m) == 32


def test_generate_to_the_last_position_and_refusals(gpu, oracle_mod):
    m = _model(max_seq=40)
    m.fill_kv(30)
    assert len(m.generate(1, 30, 10)) == 10
    for bad in (dict(token=-1), dict(token=320), dict(pos=-1), dict(pos=31), dict(n=0), dict(temperature=0.5)):
        a = dict(token=1, pos=30, n=10, temperature=0.0)
        a.update(bad)
        with pytest.raises((RuntimeError, ValueError)):
            m.generate(**a)
    from saient_quartz_b200.host_model import HostModel
    with pytest.raises(ValueError):
        HostModel(kv_bits=8, vocab_size=320, embed_dim=2048, n_heads=16, n_kv_heads=4, n_layers=1, ffn_dim=4096, head_dim=128, rope_theta=1e4, max_seq=8)
    with pytest.raises(ValueError):
        HostModel(kv_bits=4, vocab_size=320, embed_dim=2048, n_heads=32, n_kv_heads=1, n_layers=1, ffn_dim=4096, head_dim=64, rope_theta=1e4, max_seq=8)
    assert m.H.qh_set_kv_bits(m.m, 32) == -1      # too late
    gpu.lib().quartz_clear_error()


@pytest.mark.parametrize("bad", [dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_p=float("nan")),
                                 dict(min_p=float("nan"))])
def test_generate_refuses_what_the_sampler_does_not_take(gpu, oracle_mod, bad):
    m = _model(n_layers=1, max_seq=40)
    m.fill_kv(10)
    before = gpu.lib().quartz_launch_count()
    a = dict(temperature=0.5, u=np.full(5, 0.5, np.float32))
    a.update(bad)
    with pytest.raises(RuntimeError):
        m.generate(1, 10, 5, **a)
    assert gpu.lib().quartz_launch_count() == before and gpu.lib().quartz_last_error() == 0
    assert len(m.generate(1, 10, 5)) == 5
    gpu.check_error()


def test_a_long_context_in_every_sequence(gpu, oracle_mod):
    """A cache in which several clusters of a kv head work and merge: recorded steps, generation, short and long positions."""
    m = _model(max_seq=9000, n_layers=2)
    m.fill_kv(8900)
    ref = _ref(m, 8900)
    for pos, tok in ((8900, 17), (8901, 300)):
        want = ref.forward(tok, pos)
        plain = m.step(tok, pos, fused=False)
        assert _rel(plain, want) < 5e-3
        _rows_match(m, ref, pos)
        for seq in (1, 2):
            got = m.step(tok, pos, fused=seq)
            assert _rel(got, want) < 5e-3 and _rel(got, plain) < 2e-3, seq
    u = np.random.Generator(np.random.PCG64(9)).random(12).astype(np.float32)
    for at in (40, 4000, 8902):
        got = m.generate(7, at, 12, temperature=0.9, top_k=30, u=u)
        tok, want = 7, []
        for i in range(12):
            tok = sampling.sample(m.step(tok, at + i, fused=True), u[i], temperature=0.9, top_k=30)[0]
            want.append(tok)
        assert list(got) == want
    gpu.check_error()


def test_no_positions(gpu, oracle_mod):
    m = _model(n_layers=1, max_seq=40)
    k, v = m.read_kv(0, 3, 0)
    assert k.size == v.size == 0
    gpu.check_error()
