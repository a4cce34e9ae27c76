"""CPU tests: the 4-bit cache's and the sampler's calls refuse what they do not serve before they touch the device."""
import pytest

P = 1 << 20   # a 16-byte aligned address that no refused call dereferences


@pytest.fixture()
def L(pkg):
    lib = pkg.lib()
    lib.quartz_clear_error()
    yield lib
    lib.quartz_clear_error()


def refused(L, code=2):
    got = L.quartz_last_error()
    assert got == code, (got, L.quartz_error_string())
    assert L.quartz_error_string()
    launches = L.quartz_launch_count()
    L.quartz_clear_error()
    return launches


def test_bytes(L):
    assert L.cuda_kv4_bytes(1, 1, 32) == 40 * 32
    assert L.cuda_kv4_bytes(33, 8, 128) == 8 * 2 * 40 * 128
    assert L.cuda_kv4_bytes(2 ** 31 - 1, 64, 128) == 64 * 2 ** 26 * 40 * 128
    for bad in ((0, 8, 128), (-1, 8, 128), (32, 0, 128), (32, 8, 0), (32, 8, 48), (32, 8, 160), (32, 8, 256)):
        assert L.cuda_kv4_bytes(*bad) == 0


def test_supported(L):
    assert L.cuda_attn_kv4_supported(32, 8, 128) == 1 and L.cuda_attn_kv4_supported(16, 1, 32) == 1
    for bad in ((32, 5, 128), (17, 1, 64), (0, 1, 64), (8, 0, 64), (8, 8, 80), (-8, -8, 64)):
        assert L.cuda_attn_kv4_supported(*bad) == 0


def rows(L, name, n_tok=3, n_kv=2, hd=64, max_seq=40, pos0=0, cache=P, k=P, v=P):
    if name == "read":
        L.cuda_kv4_read_rows(k, v, cache, n_tok, n_kv, hd, max_seq, pos0)
    elif name == "append":
        L.cuda_kv4_append_rows(cache, k, v, n_tok, n_kv, hd, max_seq, pos0)
    else:
        L.cuda_rope_kv4_rows(P, k, v, cache, n_tok, 4, n_kv, hd, max_seq, pos0, 1e4, 1.0, 0, 0)


@pytest.mark.parametrize("name", ["append", "read", "rope"])
@pytest.mark.parametrize("bad", [dict(n_tok=-1), dict(n_kv=0), dict(hd=48), dict(hd=256), dict(max_seq=0), dict(pos0=-1), dict(pos0=38),
                                 dict(pos0=2 ** 31 - 1), dict(cache=None), dict(cache=P + 4), dict(k=None), dict(v=None)])
def test_rows_refuse(L, name, bad):
    before = L.quartz_launch_count()
    rows(L, name, **bad)
    assert refused(L) == before


def step(L, out=P, q=P, k=P, v=P, cache=P, nh=8, n_kv=2, hd=64, max_seq=40, step=None, pos=3, slot=-1):
    L.cuda_attn_step_kv4(out, q, k, v, cache, nh, n_kv, hd, max_seq, step, pos, 0, 0.1, None, 1e4, 1.0, 0, 0, slot)


@pytest.mark.parametrize("bad", [dict(out=None), dict(q=None), dict(k=None), dict(v=None), dict(cache=None), dict(cache=P + 8), dict(nh=7),
                                 dict(nh=34), dict(hd=80), dict(max_seq=0), dict(pos=-1), dict(pos=40), dict(slot=4), dict(out=P + 4),
                                 dict(q=P + 8), dict(k=P + 4), dict(v=P + 4)])
def test_step_refuses(L, bad):
    before = L.quartz_launch_count()
    step(L, **bad)
    assert refused(L) == before


@pytest.mark.parametrize("bad", [dict(out=None), dict(q=None), dict(cache=None), dict(nh=7), dict(hd=16), dict(n_tok=-1), dict(n_tok=41),
                                 dict(pos0=-1), dict(pos0=39), dict(out=P + 4), dict(q=P + 4)])
def test_prompt_refuses(L, bad):
    a = dict(out=P, q=P, cache=P, n_tok=5, nh=8, n_kv=2, hd=64, max_seq=40, pos0=0)
    a.update(bad)
    before = L.quartz_launch_count()
    L.cuda_attn_prompt_kv4(a["out"], a["q"], a["cache"], a["n_tok"], a["nh"], a["n_kv"], a["hd"], a["max_seq"], a["pos0"], 0, 0.1, None)
    assert refused(L) == before


@pytest.mark.parametrize("bad,code", [(dict(rows=-1), 2), (dict(vocab=0), 2), (dict(vocab=(1 << 19) + 1, ld=1 << 20), 5), (dict(ld=99), 2),
                                      (dict(t=-0.5), 2), (dict(t=float("nan")), 2), (dict(t=float("inf")), 2), (dict(top_p=float("nan")), 2),
                                      (dict(min_p=float("nan")), 2), (dict(z=None), 2), (dict(tok=None), 2), (dict(u=None), 2)])
def test_sample_refuses(L, bad, code):
    a = dict(z=P, rows=2, vocab=100, ld=100, t=0.8, top_p=0.9, min_p=0.0, u=P, tok=P)
    a.update(bad)
    before = L.quartz_launch_count()
    L.cuda_sample(a["z"], a["rows"], a["vocab"], a["ld"], a["t"], 5, a["top_p"], a["min_p"], a["u"], a["tok"], None)
    assert refused(L, code) == before


def test_advance_refuses(L):
    for args in ((None, P), (P, None)):
        before = L.quartz_launch_count()
        L.cuda_step_advance(*args)
        assert refused(L) == before


def test_nothing_to_do_is_not_an_error(L):
    before = L.quartz_launch_count()
    rows(L, "append", n_tok=0)
    rows(L, "read", n_tok=0)
    rows(L, "rope", n_tok=0)
    L.cuda_attn_prompt_kv4(P, P, P, 0, 8, 2, 64, 40, 0, 0, 0.1, None)
    L.cuda_sample(P, 0, 100, 100, 0.8, 5, 0.9, 0.0, P, P, None)
    assert L.quartz_last_error() == 0 and L.quartz_launch_count() == before


@pytest.mark.parametrize("bad", [0, 1, 2])
def test_rope_rows_refuse_unaligned_rows(L, bad):
    before = L.quartz_launch_count()
    a = [P + 4 * (i == bad) for i in range(3)]
    L.cuda_rope_kv4_rows(*a, P, 3, 4, 2, 64, 40, 0, 1e4, 1.0, 0, 0)
    assert refused(L) == before


@pytest.mark.parametrize("name", ["append", "read"])
def test_rows_refuse_more_than_memory_holds(L, name):
    before = L.quartz_launch_count()
    rows(L, name, n_tok=2 ** 26, n_kv=32, hd=32, max_seq=2 ** 26)
    assert refused(L, 5) == before


def test_sampler_settings(L):
    assert all(L.cuda_sample_supported(*a) == 1 for a in ((1, 0.0, 1.0, 0.0), (1 << 19, 0.8, 0.9, 0.05), (100, 3e38, -1.0, 7.0)))
    nan, inf = float("nan"), float("inf")
    for bad in ((0, 0.8, 0.9, 0.0), (-5, 0.8, 0.9, 0.0), ((1 << 19) + 1, 0.8, 0.9, 0.0), (100, -0.5, 0.9, 0.0), (100, nan, 0.9, 0.0), (100, inf, 0.9, 0.0),
                (100, -inf, 0.9, 0.0), (100, 0.8, nan, 0.0), (100, 0.8, 0.9, nan), (100, 0.0, nan, 0.0)):
        assert L.cuda_sample_supported(*bad) == 0, bad
    assert L.quartz_last_error() == 0
