"""CPU tests of the host's generation loop (qh_generate): the C++ host is compiled against a stand-in for the CUDA library
whose "device" memory is the host's, and which counts what the loop does with it."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST = os.path.join(ROOT, "saient-quartz_b200", "host")

FAKE = r"""
#include <math.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
// what the tests set and read
int fake_error, fake_fail_alloc, fake_fail_sample, fake_vocab, fake_replays, fake_samples, fake_bad_rows, fake_bad_writes;
static int *step_words;
static int valid(const void *p) { return (uintptr_t)p > 65536; }
void *cuda_alloc(size_t n)
{
    if (fake_fail_alloc && --fake_fail_alloc == 0) return 0;
    void *p = malloc(n + 16);
    memset(p, 0x7F, n);            // fresh memory holds tokens of no vocabulary
    return p;
}
void cuda_drop(void *p) { free(p); }
static void copy(void *d, const void *s, size_t n)
{
    if (valid(d) && valid(s)) memcpy(d, s, n);
    else fake_bad_writes++;
}
void cuda_h2d(void *d, const void *s, size_t n) { copy(d, s, n); }
void cuda_d2h(void *d, const void *s, size_t n) { copy(d, s, n); }
int quartz_last_error(void) { return fake_error; }
int quartz_graph_begin(void) { return 1; }
void *quartz_graph_end(void) { return &step_words; }
void quartz_graph_launch(void *g)
{
    fake_replays++;
    if (step_words[0] < 0 || step_words[0] >= fake_vocab) fake_bad_rows++;
}
void cuda_step_set(int *s, int token, int pos) { step_words = s; s[0] = token; s[1] = pos; }
void cuda_step_advance(int *s, const int *token)
{
    if (!valid(token)) { fake_bad_writes++; return; }
    if (*token >= 0) s[0] = *token;
    s[1]++;
}
int cuda_sample_supported(int vocab, float t, float top_p, float min_p)
{
    return vocab > 0 && vocab <= 524288 && t >= 0 && isfinite(t) && top_p == top_p && min_p == min_p;
}
void cuda_sample(const float *z, int rows, int vocab, size_t ld, float t, int top_k, float top_p, float min_p, const float *u, int *tok, float *p)
{
    fake_samples++;
    if (!cuda_sample_supported(vocab, t, top_p, min_p)) { fake_error = 2; return; }
    if (fake_fail_sample) { fake_error = 3; return; }
    if (!valid(tok)) { fake_bad_writes++; return; }
    *tok = (step_words[0] * 7 + step_words[1]) % vocab;
}
int cuda_attn_step_supported(int a, int b, int c) { return 1; }
int cuda_attn_kv4_supported(int a, int b, int c) { return 1; }
int cuda_gemv_q_supported(uint32_t t, const uint8_t *w, int k) { return 1; }
size_t cuda_kv4_bytes(int a, int b, int c) { return 64; }
"""
OWN = ("cuda_alloc cuda_drop cuda_h2d cuda_d2h quartz_last_error quartz_graph_begin quartz_graph_end quartz_graph_launch cuda_step_set "
       "cuda_step_advance cuda_sample_supported cuda_sample cuda_attn_step_supported cuda_attn_kv4_supported cuda_gemv_q_supported cuda_kv4_bytes").split()


class Config(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("vocab_size embed_dim n_heads n_kv_heads n_layers ffn_dim head_dim n_experts n_experts_used moe_renorm "
                                       "clamped_swiglu swa_window rope_neox yarn_orig_ctx max_seq").split()] + [("rope_theta", C.c_float), ("yarn_scale", C.c_float)]


@pytest.fixture(scope="module")
def H(pkg, tmp_path_factory):
    d = tmp_path_factory.mktemp("host")
    rest = "".join(f"long {n}(void) {{ return 0; }}\n" for n in pkg.declared_symbols() if n not in OWN)
    (d / "fake.c").write_text(FAKE + rest)
    subprocess.check_call(["gcc", "-O1", "-w", "-fPIC", "-c", str(d / "fake.c"), "-o", str(d / "fake.o")])
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-o", str(d / "host.so")] +
                          [os.path.join(HOST, f) for f in ("forward_state.cpp", "gguf_loader.cpp", "model_loader.cpp")] + [str(d / "fake.o")])
    L = C.CDLL(str(d / "host.so"))
    L.qh_create.restype = C.c_void_p
    L.qh_create.argtypes = [C.POINTER(Config)]
    L.qh_finalize.argtypes = L.qh_destroy.argtypes = [C.c_void_p]
    L.qh_generate.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_float, C.c_int, C.c_float, C.c_float, C.c_void_p, C.c_void_p]
    return L


class Model:
    def __init__(self, L, vocab=300):
        self.L = L
        for n in ("error", "fail_alloc", "fail_sample", "replays", "samples", "bad_rows", "bad_writes"):
            self.set(n, 0)
        self.set("vocab", vocab)
        c = Config(vocab_size=vocab, embed_dim=256, n_heads=4, n_kv_heads=2, n_layers=1, ffn_dim=256, head_dim=64, max_seq=4000, rope_theta=1e4, yarn_scale=1.0)
        self.m, self.vocab = L.qh_create(C.byref(c)), vocab
        assert L.qh_finalize(self.m) == 0

    def set(self, name, x):
        C.c_int.in_dll(self.L, "fake_" + name).value = x

    def get(self, name):
        return C.c_int.in_dll(self.L, "fake_" + name).value

    def generate(self, n, token=5, pos=10, temperature=0.8, top_k=0, top_p=1.0, min_p=0.0, u=True):
        out, r = np.full(n, -77, np.int32), np.full(n, 0.5, np.float32)
        rc = self.L.qh_generate(self.m, token, pos, n, temperature, top_k, top_p, min_p, r.ctypes.data if u else None, out.ctypes.data)
        return rc, list(out)

    def expected(self, n, token=5, pos=10):
        out = []
        for i in range(n):
            token = (token * 7 + pos + i) % self.vocab
            out.append(token)
        return out


@pytest.fixture()
def model(H):
    m = Model(H)
    yield m
    H.qh_destroy(m.m)


def test_the_loop(model):
    assert model.generate(50) == (0, model.expected(50))
    assert model.get("samples") == 50 and model.get("replays") == 50 and model.get("bad_rows") == 0
    assert model.generate(8, temperature=0.0, u=False) == (0, model.expected(8))


BAD = [dict(temperature=-0.5), dict(temperature=float("nan")), dict(temperature=float("nan"), u=False), dict(temperature=float("inf")),
       dict(temperature=float("-inf")), dict(top_p=float("nan")), dict(min_p=float("nan")), dict(temperature=0.0, min_p=float("nan"))]


@pytest.mark.parametrize("bad", BAD)
def test_settings_that_the_sampler_does_not_take_are_refused(model, bad):
    """Refused before the first launch, not step by step with tokens that nobody wrote."""
    rc, _ = model.generate(20, **bad)
    assert rc == -1 and model.get("error") == 0
    assert [model.get(n) for n in ("samples", "replays", "bad_rows")] == [0, 0, 0]
    assert model.generate(6) == (0, model.expected(6))


def test_a_vocabulary_that_the_sampler_does_not_take_is_refused(H):
    m = Model(H, vocab=600000)
    assert m.generate(20)[0] == -1 and m.get("error") == 0
    assert [m.get(n) for n in ("samples", "replays", "bad_rows")] == [0, 0, 0]
    H.qh_destroy(m.m)


@pytest.mark.parametrize("which", [1, 2])
def test_buffers_that_could_not_grow(model, which):
    """The first or the second of the two does not fit: refused, and a later, shorter call has buffers of its own again."""
    assert model.generate(4)[0] == 0
    model.set("fail_alloc", which)
    assert model.generate(100)[0] == -2
    for n in (1, 3, 4, 100):
        assert model.generate(n) == (0, model.expected(n))
    assert model.get("bad_writes") == 0 and model.get("bad_rows") == 0


def test_a_sampler_that_did_not_run(model):
    """Its launch failed: the steps go on with the last token, never with what the buffer held, and the call fails."""
    assert model.generate(4)[0] == 0
    model.set("fail_sample", 1)
    for n in (4, 40):
        rc, tokens = model.generate(n)
        assert rc != 0 and model.get("bad_rows") == 0
        assert set(tokens) <= {-1, -77}
    model.set("fail_sample", 0)
    model.set("error", 0)
    assert model.generate(40) == (0, model.expected(40))
