"""What the 4-bit KV cache, the attention over it and the device-side sampler are measured on.

The cases are real work of a decode loop: rows of keys and values written into the cache and read back, one token's
attention over a cache of a given length, a prompt's causal attention, and picking the next token of one or many
sequences.  `run` computes them in plain torch, or (own = True) through the library's C entry points.

The cache (one buffer for K and V) is [kv head][block of 32 positions]; a block holds K codes, K parameters, V codes
and V parameters.  With NG = head_dim / 32 groups of 32 dims per row:
  K codes     one row of head_dim / 2 bytes per position; 32-bit word t * NG + g (t < 4) holds dims 32 g + 8 t + i in nibbles i < 8
  V codes     one row of head_dim / 2 bytes per position; 16-bit word r * NG + g (r < 8) holds dims 32 g + 4 r + i in nibbles i < 4
  parameters  one row of 2 * NG halves per position: the NG minima m, then the NG steps d
A value is m + d * code, rounded once to f32.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 32      # positions per cache block, and dims per quantisation group


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def _rows(name, n_tok, heads, head_dim, pos0=0):
    return dict(name=name, op="rows", n_tok=n_tok, kv_heads=heads, head_dim=head_dim, pos0=pos0)


def _step(name, pos, heads, kv_heads, head_dim, window=0, sinks=False, append=False):
    return dict(name=name, op="step", pos=pos, heads=heads, kv_heads=kv_heads, head_dim=head_dim, window=window, sinks=sinks,
                append=append)


def _prompt(name, n_tok, pos0, heads, kv_heads, head_dim, window=0, sinks=False):
    return dict(name=name, op="prompt", n_tok=n_tok, pos0=pos0, heads=heads, kv_heads=kv_heads, head_dim=head_dim, window=window,
                sinks=sinks)


def _sample(name, rows, vocab, temperature, top_k, top_p, min_p, coarse=False):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                coarse=coarse)


def listed():
    return [
        # a 512-token prompt's keys and values of one Llama-3-8B-shaped layer go into the cache and are read back
        _rows("rows 512 x 8 x 128", 512, 8, 128),
        # one token of a small model: latency
        _rows("rows 1 x 2 x 64", 1, 2, 64, pos0=37),
        # a long document, odd start, three groups per head
        _rows("rows 8189 x 4 x 96", 8189, 4, 96, pos0=1027),
        # the first words of a chat on a small model: latency
        _step("step ctx 18", 17, 8, 2, 64),
        # the decode step that the repository's benchmark times, its new key and value appended
        _step("step ctx 1024 append", 1023, 32, 8, 128, append=True),
        # a long chat, odd length, with per-head sinks
        _step("step ctx 16381 sinks", 16380, 32, 8, 128, sinks=True),
        # the longest context
        _step("step ctx 131072", 131071, 32, 8, 128),
        # a 512-token prompt from an empty cache
        _prompt("prompt 512", 512, 0, 32, 8, 128),
        # the next turn of a conversation: ragged prompt on top of a cache, sliding window
        _prompt("prompt 333 at 1700 window", 333, 1700, 24, 3, 64, window=1024),
        # a long prompt
        _prompt("prompt 2048", 2048, 0, 32, 8, 128),
        # the next token of one sequence, usual settings
        _sample("sample 1 x 128256", 1, 128256, 0.7, 40, 0.95, 0.05),
        # a large batch whose head works in 16 bits (ties between logits), nucleus only
        _sample("sample 256 x 128256", 256, 128256, 1.0, 0, 0.9, 0.0, coarse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "step", "step", "prompt", "sample", "sample"])
    head_dim = rng.choice([32, 64, 96, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    if op == "rows":
        c = _rows("", _log(rng, 1, 8000), kv_heads, head_dim, rng.randrange(0, 3000))
    elif op == "step":
        pos = _log(rng, 1, 131072) - 1
        c = _step("", pos, heads, kv_heads, head_dim, rng.choice([0, 0, _log(rng, 1, 8192)]), rng.random() < 0.3, rng.random() < 0.3)
    elif op == "prompt":
        c = _prompt("", _log(rng, 1, 900), rng.choice([0, rng.randrange(0, 2500)]), min(heads, 24) // kv_heads * kv_heads, kv_heads, head_dim,
                    rng.choice([0, 0, _log(rng, 1, 2048)]), rng.random() < 0.3)
    else:
        c = _sample("", _log(rng, 1, 200), _log(rng, 500, 128256), round(rng.uniform(0.3, 1.5), 2), rng.choice([0, 1, 20, 50, 1000]),
                    rng.choice([1.0, 0.5, 0.9, 0.99]), rng.choice([0.0, 0.02, 0.1]), rng.random() < 0.3)
    del c["name"]
    return c


def work(case):
    if case["op"] == "rows":      # f32 rows read, codes and parameters written; then the reverse
        n = 2 * case["n_tok"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": n * 2 * (4 + 0.625), "flops": n * 6}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 12 * case["rows"], "flops": 4 * n}
    h, kv, hd, w = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    if case["op"] == "step":
        seen = min(case["pos"] + 1, w) if w > 0 else case["pos"] + 1
        more = 2 * kv * hd * (4 + 0.625 + 4) if case["append"] else 0
        return {"bytes": seen * kv * hd * 1.25 + 8 * h * hd + more, "flops": 4 * h * hd * seen}
    n, p0 = case["n_tok"], case["pos0"]
    lo = max(0, p0 + 1 - w) if w > 0 else 0
    seen = sum(min(p + 1, w) if w > 0 else p + 1 for p in range(p0, p0 + n))
    return {"bytes": (p0 + n - lo) * kv * hd * 1.25 + 8 * n * h * hd, "flops": 4 * h * hd * seen}


# ---------------------------------------------------------------------------------------------------------------
# the cache's layout in torch
# ---------------------------------------------------------------------------------------------------------------
def _block_bytes(head_dim):
    return BLOCK * head_dim * 5 // 4


def _nibbles(b):      # [..., n] bytes -> [..., 2 n] codes
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _bytes(c):        # [..., 2 n] codes -> [..., n] bytes
    c = c.unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4)


def _pack(k, v):
    """Cache bytes [heads, blocks, block bytes] of (codes [H, S, hd] uint8, m, d [H, S, NG]) for K and V; S % 32 == 0."""
    def part(codes, m, d, per):
        H, S, hd = codes.shape
        c = codes.view(H, S // BLOCK, BLOCK, hd // 32, 32 // per, per).transpose(3, 4).reshape(H, S // BLOCK, BLOCK * hd)
        p = torch.cat((m, d), -1).half().contiguous().view(torch.uint8)
        return _bytes(c), p.reshape(H, S // BLOCK, -1)
    return torch.cat(part(*k, 8) + part(*v, 4), -1).contiguous()


def _unpack(cache, head_dim):
    """K and V of cache bytes [H, nb, block bytes] as f32 [H, 32 nb, hd]."""
    H, nb, _ = cache.shape
    ng, code, par = head_dim // 32, BLOCK * head_dim // 2, BLOCK * head_dim // 8

    def part(at, per):
        c = _nibbles(cache[..., at:at + code]).view(H, nb * BLOCK, 32 // per, ng, per).transpose(2, 3)
        p = cache[..., at + code:at + code + par].contiguous().view(torch.float16).view(H, nb * BLOCK, 2, ng, 1, 1).double()
        return (p[:, :, 0] + p[:, :, 1] * c).float().reshape(H, nb * BLOCK, head_dim)
    return part(0, 8), part(code + par, 4)


def _f16_grid(x):
    """The spacing of f16 numbers around the 64-bit x."""
    return torch.exp2((torch.frexp(x).exponent.double() - 11).clamp(min=-24))


def _quantise(x):
    """The values that rows x [..., head_dim] f32 stand for once they are in the cache (f32)."""
    g = x.double().unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, True), g.amax(-1, True)
    q = _f16_grid(lo)
    m = torch.floor(lo / q) * q
    d = (hi - m) / 15
    q = _f16_grid(d)
    d = torch.ceil(d / q) * q
    code = torch.round((g - m) / torch.where(d > 0, d, torch.ones_like(d))).clamp(0, 15)
    return (m + d * code).float().flatten(-2)


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _kv_rows(gen, n, kv_heads, head_dim, keys):
    """Keys have a few channels with a large offset, as keys of trained models do; values are plain."""
    x = torch.randn(n, kv_heads, head_dim, generator=gen, device="cuda")
    if keys:
        off = torch.randn(kv_heads, head_dim, generator=gen, device="cuda")
        x += torch.where(off.abs() > 1.8, 3 * off, torch.zeros_like(off))
    return x


def _filled(gen, S, kv_heads, head_dim):
    """A cache of S positions (a multiple of 32) filled a stretch at a time."""
    out = []
    for keys in (True, False):
        codes, ms, ds = [], [], []
        off = torch.randn(kv_heads, head_dim, generator=gen, device="cuda")
        off = torch.where(off.abs() > 1.8, 3 * off, torch.zeros_like(off)) if keys else torch.zeros_like(off)
        for s in range(0, S, 16384):
            n = min(16384, S - s)
            g = (torch.randn(kv_heads, n, head_dim, generator=gen, device="cuda") + off[:, None]).unflatten(-1, (-1, 32))
            m = g.amin(-1).half()
            d = ((g.amax(-1) - m.float()) / 15).half()
            c = torch.round((g - m.float()[..., None]) / d.float()[..., None]).clamp(0, 15).to(torch.uint8)
            codes.append(c.flatten(-2)), ms.append(m), ds.append(d)
        out.append((torch.cat(codes, 1), torch.cat(ms, 1), torch.cat(ds, 1)))
    return _pack(*out)


def _max_seq(last):
    return -(-(last + 1) // BLOCK) * BLOCK


def prepare(case, seed):
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    st = dict(case)
    if case["op"] == "rows":
        n, H, hd = case["n_tok"], case["kv_heads"], case["head_dim"]
        st["k"], st["v"] = _kv_rows(gen, n, H, hd, True), _kv_rows(gen, n, H, hd, False)
        st["max_seq"] = _max_seq(case["pos0"] + n - 1)
        st["cache"] = torch.zeros(H, st["max_seq"] // BLOCK, _block_bytes(hd), dtype=torch.uint8, device="cuda")
        st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
    elif case["op"] == "sample":
        z = torch.randn(case["rows"], case["vocab"], generator=gen, device="cuda") * 2.5
        st["logits"] = z.bfloat16().float() if case["coarse"] else z
        for name in ("temperature", "top_p", "min_p"):      # as the 32-bit arguments that the call takes
            st[name] = float(np.float32(case[name]))
        st["u"] = torch.rand(case["rows"], generator=gen, device="cuda")
        st["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        st["probs"] = torch.empty(case["rows"], device="cuda")
    else:
        h, H, hd = case["heads"], case["kv_heads"], case["head_dim"]
        last = case["pos"] if case["op"] == "step" else case["pos0"] + case["n_tok"] - 1
        st["max_seq"] = _max_seq(last)
        st["cache"] = _filled(gen, st["max_seq"], H, hd)
        n = case.get("n_tok", 1)
        st["q"] = torch.randn(n, h, hd, generator=gen, device="cuda")
        st["out"] = torch.empty_like(st["q"])
        st["sink"] = torch.randn(h, generator=gen, device="cuda") if case["sinks"] else None
        if case.get("append"):
            st["k"], st["v"] = _kv_rows(gen, 1, H, hd, True), _kv_rows(gen, 1, H, hd, False)
            st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
    return st


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def _plain_attention(st, k, v, first, p0, k0):
    """q [n, heads, hd] at positions p0.. over k, v [H, S, hd] at positions k0..; keys from first[t] up to the token's own."""
    q, H = st["q"], k.shape[0]
    n, h, hd = q.shape
    G = h // H
    qg = q.view(n, H, G, hd).permute(1, 2, 0, 3).reshape(H, G * n, hd)
    s = (torch.bmm(qg, k.transpose(1, 2)) * (1 / math.sqrt(hd))).view(H, G, n, -1)
    at = k0 + torch.arange(k.shape[1], device=k.device)
    tok = p0 + torch.arange(n, device=k.device)
    s = s.masked_fill((at > tok[:, None]) | (at < first[:, None]), -math.inf)
    top = s.amax(-1, True)
    if st["sink"] is not None:
        top = torch.maximum(top, st["sink"].view(H, G, 1, 1))
    e = torch.exp(s - top)
    total = e.sum(-1, True)
    if st["sink"] is not None:
        total = total + torch.exp(st["sink"].view(H, G, 1, 1) - top)
    o = torch.bmm((e / total).view(H, G * n, -1), v)
    return o.view(H, G, n, hd).permute(2, 0, 1, 3).reshape(n, h, hd)


def _plain_sample(st):
    z = st["logits"]
    n = z.shape[1]
    s, at = torch.sort(z, dim=1, descending=True, stable=True)
    w = torch.exp((s.double() - s[:, :1].double()) / st["temperature"])
    keep = torch.ones_like(w, dtype=torch.bool)
    if 0 < st["top_k"] < n:
        keep[:, st["top_k"]:] = False
    if st["top_p"] < 1:
        inside = w * keep
        before = torch.cumsum(inside, 1) - inside
        keep &= before < st["top_p"] * inside.sum(1, True)
    keep &= w >= st["min_p"]
    by_index = torch.zeros_like(w).scatter_(1, at, w * keep)
    run_sum = torch.cumsum(by_index, 1)
    total = run_sum[:, -1:]
    token = (run_sum <= st["u"].double()[:, None] * total).sum(1, True).clamp(max=n - 1)
    return {"tokens": token[:, 0].int(), "probs": (by_index.gather(1, token) / total)[:, 0].float()}


def _plain(st):
    if st["op"] == "sample":
        return _plain_sample(st)
    if st["op"] == "rows":
        return {"k": _quantise(st["k"]), "v": _quantise(st["v"])}
    n = st.get("n_tok", 1)
    p0 = st["pos"] if st["op"] == "step" else st["pos0"]
    tok = p0 + torch.arange(n, device="cuda")
    first = (tok + 1 - st["window"]).clamp(min=0) if st["window"] > 0 else torch.zeros_like(tok)
    b0 = max(0, p0 + 1 - st["window"]) // BLOCK if st["window"] > 0 else 0
    k, v = _unpack(st["cache"][:, b0:(p0 + n - 1) // BLOCK + 1], st["head_dim"])
    if not st.get("append"):
        return {"out": _plain_attention(st, k, v, first, p0, b0 * BLOCK)}
    kq, vq = _quantise(st["k"]), _quantise(st["v"])
    k[:, p0 - b0 * BLOCK], v[:, p0 - b0 * BLOCK] = kq[0], vq[0]
    return {"out": _plain_attention(st, k, v, first, p0, b0 * BLOCK), "k": kq, "v": vq}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _library():
    import __graft_entry__
    lib = __graft_entry__.load_package().lib()
    lib.quartz_set_stream(torch.cuda.current_stream().cuda_stream)
    return lib


def _own(st):
    L = _library()
    if st["op"] == "sample":
        L.cuda_sample(_ptr(st["logits"]), st["rows"], st["vocab"], st["vocab"], st["temperature"], st["top_k"], st["top_p"], st["min_p"],
                      _ptr(st["u"]), _ptr(st["tokens"]), _ptr(st["probs"]))
        return {"tokens": st["tokens"], "probs": st["probs"]}
    H, hd, cache, last = st["kv_heads"], st["head_dim"], _ptr(st["cache"]), st["max_seq"]
    if st["op"] == "rows":
        L.cuda_kv4_append_rows(cache, _ptr(st["k"]), _ptr(st["v"]), st["n_tok"], H, hd, last, st["pos0"])
        L.cuda_kv4_read_rows(_ptr(st["k_out"]), _ptr(st["v_out"]), cache, st["n_tok"], H, hd, last, st["pos0"])
        return {"k": st["k_out"], "v": st["v_out"]}
    scale = 1 / math.sqrt(hd)
    if st["op"] == "prompt":
        L.cuda_attn_prompt_kv4(_ptr(st["out"]), _ptr(st["q"]), cache, st["n_tok"], st["heads"], H, hd, last, st["pos0"], st["window"], scale,
                               _ptr(st["sink"]))
        return {"out": st["out"]}
    # rotated queries and keys (theta 0: no rotation in the call), as a model with its own rotation passes them
    L.cuda_attn_step_kv4(_ptr(st["out"]), _ptr(st["q"]), _ptr(st.get("k")), _ptr(st.get("v")), cache, st["heads"], H, hd, last, None,
                         st["pos"], st["window"], scale, _ptr(st["sink"]), 0.0, 1.0, 0, 0, -1)
    if not st["append"]:
        return {"out": st["out"]}
    L.cuda_kv4_read_rows(_ptr(st["k_out"]), _ptr(st["v_out"]), cache, 1, H, hd, last, st["pos"])
    return {"out": st["out"], "k": st["k_out"], "v": st["v_out"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_rows(x):
    """numpy: a group's minimum and step on the f16 grid (down, up), the nearest code (ties to even)."""
    g = x.double().cpu().numpy().reshape(x.shape[0], -1, 32)

    def grid(a):
        return np.ldexp(1.0, np.maximum(np.frexp(a)[1] - 11, -24))
    lo = g.min(-1)
    m = np.floor(lo / grid(lo)) * grid(lo)
    step = (g.max(-1) - m) / 15
    step = np.ceil(step / grid(step)) * grid(step)
    code = np.clip(np.rint((g - m[..., None]) / np.where(step > 0, step, 1)[..., None]), 0, 15)
    return torch.from_numpy((m[..., None] + code * step[..., None]).reshape(x.shape))


def _exact_side(cache, head, positions, head_dim, values):
    """K or V of one head at `positions`, by the address of every code; f64 [len, hd]."""
    ng, code, par = head_dim // 32, BLOCK * head_dim // 2, BLOCK * head_dim // 8
    raw = cache[head].reshape(-1)
    start = (positions // BLOCK) * _block_bytes(head_dim) + (code + par if values else 0)
    row = positions % BLOCK
    j = torch.arange(head_dim, device=cache.device)
    g, within = j // 32, j % 32
    nib = ((within // 4) * ng + g) * 4 + within % 4 if values else ((within // 8) * ng + g) * 8 + within % 8
    byte = raw[(start + row * (head_dim // 2))[:, None] + nib // 2]
    c = torch.where(nib % 2 == 1, byte // 16, byte % 16).double()
    half = raw.view(torch.float16)
    base = (start + code + row * (4 * ng))[:, None] // 2
    return half[base + g].double() + half[base + ng + g].double() * c


def _exact_attention(case, st):
    h, H, hd, w = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    n = case.get("n_tok", 1)
    p0 = case["pos"] if case["op"] == "step" else case["pos0"]
    lo = max(0, p0 + 1 - w) if w > 0 else 0
    at = torch.arange(lo, p0 + n, device="cuda")
    tok = p0 + torch.arange(n, device="cuda")[:, None]
    hidden = at > tok
    if w > 0:
        hidden = hidden | (at <= tok - w)
    new = (_exact_rows(st["k"]), _exact_rows(st["v"])) if case.get("append") else None
    out = torch.empty(n, h, hd, dtype=torch.float64, device="cuda")
    for head in range(H):
        k, v = _exact_side(st["cache"], head, at, hd, False), _exact_side(st["cache"], head, at, hd, True)
        if new:
            k[-1], v[-1] = new[0][0, head].float().double(), new[1][0, head].float().double()
        for i in range(head * (h // H), (head + 1) * (h // H)):
            s = st["q"][:, i].double() @ k.T / math.sqrt(hd)
            s[hidden] = -math.inf
            top = s.max(1, keepdim=True).values
            if st["sink"] is not None:
                top = top.clamp(min=float(st["sink"][i]))
            e = torch.exp(s - top)
            total = e.sum(1, keepdim=True) + (torch.exp(st["sink"][i].double() - top) if st["sink"] is not None else 0)
            out[:, i] = (e @ v) / total
    return {"out": out, "k": new[0], "v": new[1]} if new else {"out": out}


def _exact_sample(st):
    tokens, probs = [], []
    for z, u in zip(st["logits"].double().cpu().numpy(), st["u"].double().cpu().numpy()):
        order = np.argsort(-z, kind="stable")
        if 0 < st["top_k"] < z.size:
            order = order[:st["top_k"]]
        w = np.exp((z[order] - z[order[0]]) / st["temperature"])
        if st["top_p"] < 1:
            before = np.concatenate(([0.0], np.cumsum(w)[:-1]))
            n = int(np.count_nonzero(before < st["top_p"] * w.sum()))
            order, w = order[:n], w[:n]
        order, w = order[w >= st["min_p"]], w[w >= st["min_p"]]
        by = np.argsort(order)
        order, w = order[by], w[by]
        total = np.cumsum(w)
        i = min(int(np.searchsorted(total, u * total[-1], side="right")), w.size - 1)
        tokens.append(int(order[i]))
        probs.append(w[i] / total[-1])
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "probs": torch.tensor(probs, dtype=torch.float64)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    if case["op"] == "rows":
        return {"k": _exact_rows(st["k"]), "v": _exact_rows(st["v"])}
    return _exact_attention(case, st)
