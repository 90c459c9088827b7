"""Performance cases of the operators of a verification step: what a decoder
with drafted tokens runs between its norms when it keeps activations and
cache in 8 bits.

  qmm_a8     activations quantised to INT8 with a scale for each token, times
             INT8 weights with a scale for each column
             (vm_hip_a8_stage + vm_hip_qmm_a8).
  kv         rotation of q and k, INT8 quantisation of keys and values into
             the cache with a scale for each token and head, and the cache
             read back as numbers (vm_hip_kv_q8_append + vm_hip_kv_q8_read).
  attention  attention over that cache for single tokens, prompts and trees
             of drafted tokens (vm_hip_attention_q8).
  logits     repetition, frequency and presence penalties, biases and grammar
             masks, with the greedy token (vm_hip_logits_rules).

Where `own` is false, run() computes the same with elementary torch
operations, in 32 bits or more, rounded once at the end.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_CODE = {"f32": 0, "f16": 4, "bf16": 5}  # VM_HIP_DTYPE_*
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _hip():
    """This repository's Python binding; used only where `own` is true."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "velo-mind_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import velomind_hip

    velomind_hip.load()
    return velomind_hip


# ---- the cases --------------------------------------------------------------

def _attn(name, dtype, batch, rows, past, heads, kv_heads, d, tree):
    return dict(name=name, kind="attention", dtype=dtype, batch=batch, rows=rows, past=past, heads=heads,
                kv_heads=kv_heads, d=d, tree=tree)


def listed():
    return [
        # TinyLlama's gate (or up) projection of 16 drafted tokens: weights
        # and launches.
        dict(name="qmm_a8_m16_2048x5632", kind="qmm_a8", dtype="f32", m=16, k=2048, n=5632),
        # The same projection of a 512-token prompt.
        dict(name="qmm_a8_m512_2048x5632", kind="qmm_a8", dtype="f32", m=512, k=2048, n=5632),
        # A 70B-class model's projection of a 2048-token prompt in bfloat16:
        # the matrix cores.
        dict(name="qmm_a8_bf16_m2048_8192x28672", kind="qmm_a8", dtype="bf16", m=2048, k=8192, n=28672),
        # One decoded TinyLlama token into a cache of 512.
        dict(name="kv_1_of_512", kind="kv", dtype="f32", batch=1, rows=1, past=511, heads=32, kv_heads=4, d=64,
             tree=False),
        # Eight sequences with 16 drafted tokens each, wider heads.
        dict(name="kv_b8_16_of_4000", kind="kv", dtype="bf16", batch=8, rows=16, past=3984, heads=64, kv_heads=8,
             d=128, tree=True),
        # One TinyLlama layer's attention of one decoded token: latency.
        _attn("attn_decode_2000", "f32", 1, 1, 1999, 32, 4, 64, False),
        # The same layer verifying a tree of 16 drafted tokens.
        _attn("attn_tree16_2000", "f32", 1, 16, 2000, 32, 4, 64, True),
        # Batched decode of 32 sequences of ragged lengths up to 8 K: bandwidth.
        _attn("attn_decode_b32_8000", "bf16", 32, 1, 8000, 64, 8, 128, False),
        # A 1000-token prompt behind 3001 cached tokens: the matrix cores.
        _attn("attn_prompt1000_3001", "f16", 1, 1000, 3001, 32, 4, 64, False),
        # A tree of 24 drafted tokens over one long context.
        _attn("attn_tree24_131000", "bf16", 1, 24, 131000, 64, 8, 128, True),
        # The next token of one sequence over TinyLlama's vocabulary.
        dict(name="logits_1x32000", kind="logits", dtype="f32", seqs=1, rows=1, vocab=32000, history=700, bias=16),
        # Four sequences' trees of 16 nodes over a large vocabulary.
        dict(name="logits_64x128256", kind="logits", dtype="f32", seqs=4, rows=16, vocab=128256, history=6000,
             bias=300),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, multiple):
    """Log-uniform size; one in four is any integer, the rest multiples."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.25 else max(multiple, v // multiple * multiple)


def draw(rng):
    kind = rng.choice(["qmm_a8", "qmm_a8", "kv", "attention", "attention", "attention", "logits"])
    dtype = rng.choice(["f32", "f32", "f16", "bf16"])
    if kind == "qmm_a8":
        return dict(kind=kind, dtype=dtype, m=_log(rng, 1, 2000), k=_size(rng, 200, 8192, 32),
                    n=_size(rng, 200, 28000, 16))
    if kind == "logits":
        return dict(kind=kind, dtype=dtype, seqs=_log(rng, 1, 8), rows=_log(rng, 1, 16),
                    vocab=_size(rng, 2000, 120000, 16), history=_log(rng, 1, 6000), bias=_log(rng, 1, 300))
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    d = rng.choice([64, 128])
    if kind == "kv":
        return dict(kind=kind, dtype=dtype, batch=_log(rng, 1, 8), rows=_log(rng, 1, 200), past=_log(rng, 1, 3800),
                    heads=heads, kv_heads=kv_heads, d=d, tree=rng.random() < 0.5)
    shape = rng.choice(["decode", "tree", "prompt"])
    if shape == "decode":
        batch = _log(rng, 1, 32)
        return dict(kind=kind, dtype=dtype, batch=batch, rows=1, past=_log(rng, 1, min(120000, 250000 // batch)),
                    heads=heads, kv_heads=kv_heads, d=d, tree=False)
    if shape == "tree":
        batch = _log(rng, 1, 8)
        return dict(kind=kind, dtype=dtype, batch=batch, rows=_log(rng, 2, 100), past=_log(rng, 1, 24000 // batch),
                    heads=heads, kv_heads=kv_heads, d=d, tree=True)
    return dict(kind=kind, dtype=dtype, batch=rng.choice([1, 1, 2]), rows=_log(rng, 17, 900),
                past=rng.choice([0, _log(rng, 1, 2000)]), heads=heads, kv_heads=kv_heads, d=d, tree=False)


# ---- inputs -----------------------------------------------------------------

def _gen(seed, salt=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1009 + salt)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)


def _quantise(x, dim):
    """Symmetric 8-bit codes of fp32 x along `dim` and their scales: scale =
    max|x| / 127, code = x times the scale's reciprocal, rounded half away
    from zero.  (Tensor by tensor: torch divides by a Python number as a
    product with its reciprocal, which moves values that lie at a border.)"""
    amax = x.abs().amax(dim, keepdim=True)
    one = torch.ones_like(amax)
    s = torch.where(amax > 0, amax / (one * 127), one)
    y = x * (one / s)
    codes = (torch.trunc(y.abs().double() + 0.5) * y.sign()).clamp_(-127, 127).to(torch.int8)
    return codes, s.squeeze(dim)


def _tree_words(seqs, rows, seed):
    """(depths int32 [seqs, rows], ancestor words int64 [seqs, rows,
    ceil(rows / 64)], a node its own ancestor): node 0 is the root (the last
    accepted token), every other node hangs below an earlier one."""
    r = np.random.default_rng(seed + 77)
    depths = np.zeros((seqs, rows), np.int32)
    sees = np.zeros((seqs, rows, rows), bool)
    for t in range(rows):
        sees[:, t, t] = True
        if t:
            p = np.maximum(0, t - r.geometric(0.4, seqs))  # near the end: long branches
            depths[:, t] = depths[np.arange(seqs), p] + 1
            sees[:, t] |= sees[np.arange(seqs), p]
    words = -(-rows // 64)
    bits = np.zeros((seqs, rows, words * 64), np.uint8)
    bits[:, :, :rows] = sees
    packed = np.packbits(bits, axis=-1, bitorder="little").view(np.int64)
    return torch.from_numpy(depths).to(DEV), torch.from_numpy(packed.copy()).to(DEV)


def _positions(case, seed):
    """Tokens cached in front of the call, for each sequence (ragged)."""
    r = np.random.default_rng(seed + 5)
    past, b = case["past"], case["batch"]
    pos = np.full(b, past) if b == 1 else r.integers(past // 2, past + 1, b)
    pos[0] = past
    return torch.from_numpy(pos.astype(np.int32)).to(DEV)


def _tables(length, d):
    inv = 10000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    angle = torch.arange(length, device=DEV, dtype=torch.float64)[:, None] * inv[None, :]
    return torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)


def _cache(case, seed):
    """Keys and values of every position, quantised as the cache holds them."""
    b, hk, d, s = case["batch"], case["kv_heads"], case["d"], case["past"] + case["rows"]
    g = _gen(seed, 3)
    # keys with a few large channels, values without
    channel = torch.where(torch.arange(d, device=DEV) % 17 == 3, 4.0, 1.0)
    kc, ks = _quantise(_randn(g, b, hk, s, d) * channel, -1)
    vc, vs = _quantise(_randn(g, b, hk, s, d), -1)
    return dict(k_codes=kc, k_scales=ks.contiguous(), v_codes=vc, v_scales=vs.contiguous())


def prepare(case, seed):
    kind = case["kind"]
    s = dict(case=case)
    dt = _TORCH[case["dtype"]]
    if kind == "qmm_a8":
        m, k, n = case["m"], case["k"], case["n"]
        g = _gen(seed)
        s["a"] = _randn(g, m, k).to(dt)
        s["codes"], s["scales"] = _quantise(_randn(g, k, n) * 0.02, 0)
        if own:  # the weights' layout, the staging buffer and the workspace that a program keeps
            H = _hip()
            s["H"], s["out"] = H, torch.empty(m, n, device=DEV, dtype=dt)
            s["staged"] = torch.empty(H.a8_stage_bytes(m, k), device=DEV, dtype=torch.uint8)
            s["packed"] = torch.empty(H.a8_weights_bytes(k, n), device=DEV, dtype=torch.uint8)
            s["ws"] = torch.zeros(max(1, H.qmm_a8_workspace_bytes(m, k, n)), device=DEV, dtype=torch.uint8)
            H.a8_pack(s["codes"].data_ptr(), k, n, s["packed"].data_ptr())
            del s["codes"]
        return s
    if kind in ("kv", "attention"):
        b, rows, heads, hk, d = (case[x] for x in ("batch", "rows", "heads", "kv_heads", "d"))
        total = case["past"] + rows
        s.update(_cache(case, seed))
        s["pos"] = _positions(case, seed)
        s["depths"] = s["tree"] = None
        if case["tree"]:
            s["depths"], s["tree"] = _tree_words(b, rows, seed)
        if kind == "kv":
            s["qkv"] = _randn(_gen(seed), b, rows, (heads + 2 * hk) * d).to(dt)
            s["cos"], s["sin"] = _tables(total, d)
        else:
            # q carries 1/sqrt(d), as the model loaders fold it into q_proj
            s["q"] = (_randn(_gen(seed), b, heads, rows, d) / math.sqrt(d)).to(dt)
        if own:
            H = _hip()
            s["H"] = H
            s["cache"] = H.KvQ8(s["k_codes"].data_ptr(), s["k_scales"].data_ptr(), s["v_codes"].data_ptr(),
                                s["v_scales"].data_ptr(), b, hk, total, d)
            if kind == "kv":
                s["q_out"] = torch.empty(b, heads, rows, d, device=DEV, dtype=dt)
                s["k_out"] = torch.empty(b, hk, total, d, device=DEV)
                s["v_out"] = torch.empty(b, hk, total, d, device=DEV)
            else:
                s["out"] = torch.empty(b, rows, heads * d, device=DEV, dtype=dt)
                nbytes = H.attention_q8_workspace_bytes(b, rows, heads, hk, d, total)
                s["ws"] = torch.zeros(max(1, nbytes), device=DEV, dtype=torch.uint8)
        return s
    seqs, rows, vocab, hist, nb = (case[x] for x in ("seqs", "rows", "vocab", "history", "bias"))
    g = _gen(seed)
    s["logits"] = (_randn(g, seqs, rows, vocab) * 3).to(dt)
    # a history draws on a few hundred tokens, some of them often
    words = _randint(g, 0, vocab, seqs, max(1, hist // 4))
    s["history"] = words.gather(1, _randint(g, 0, max(1, hist // 4), seqs, hist).long()).contiguous()
    s["lengths"] = _randint(g, (hist + 1) // 2, hist + 1, seqs)
    u = torch.rand(3, seqs, generator=g, device=DEV)
    s["repetition"], s["frequency"], s["presence"] = (1.05 + 0.3 * u[0]).contiguous(), (0.4 * u[1]).contiguous(), (
        0.5 * u[2]).contiguous()
    s["bias_tokens"] = _randint(g, 0, vocab, seqs, nb)
    s["bias_values"] = _randn(g, seqs, nb) * 4
    s["bias_lengths"] = _randint(g, nb // 2, nb + 1, seqs)
    # a grammar that leaves about one token in sixteen
    n_words = -(-vocab // 32)
    a, b2, c, e = (_randint(g, -2**31, 2**31 - 1, seqs, rows, n_words) for _ in range(4))
    s["allowed"] = (a & b2 & c & e).contiguous()
    s["drafted"] = _randint(g, 0, vocab, seqs, rows)
    s["tree"] = _tree_words(seqs, rows, seed)[1]
    if own:
        H = _hip()
        s["H"] = H
        s["out"] = torch.empty_like(s["logits"])
        s["tokens"] = torch.empty(seqs, rows, device=DEV, dtype=torch.int32)
        s["ws"] = torch.zeros(max(1, H.logits_rules_workspace_bytes(seqs, rows, vocab)), device=DEV,
                              dtype=torch.uint8)
        s["rules"] = H.LogitsRules(
            history=s["history"].data_ptr(), history_lengths=s["lengths"].data_ptr(), history_stride=hist,
            repetition=s["repetition"].data_ptr(), frequency=s["frequency"].data_ptr(),
            presence=s["presence"].data_ptr(), bias_tokens=s["bias_tokens"].data_ptr(),
            bias_values=s["bias_values"].data_ptr(), bias_lengths=s["bias_lengths"].data_ptr(), bias_stride=nb,
            allowed=s["allowed"].data_ptr(), drafted=s["drafted"].data_ptr(), tree=s["tree"].data_ptr())
    return s


# ---- one pass: this framework's calls ---------------------------------------

def _run_own(s):
    H, case = s["H"], s["case"]
    kind, code = case["kind"], _CODE[case["dtype"]]
    if kind == "qmm_a8":
        m, k, n = case["m"], case["k"], case["n"]
        H.a8_stage(s["a"].data_ptr(), code, m, k, s["staged"].data_ptr())
        H.qmm_a8(s["staged"].data_ptr(), s["packed"].data_ptr(), s["scales"].data_ptr(), s["out"].data_ptr(), code,
                 m, k, n, s["ws"].data_ptr(), s["ws"].numel())
        return s["out"]
    if kind == "kv":
        H.kv_q8_append(s["cache"], s["qkv"].data_ptr(), code, case["rows"], case["heads"], s["cos"].data_ptr(),
                       s["sin"].data_ptr(), s["pos"].data_ptr(), None,
                       s["depths"].data_ptr() if s["depths"] is not None else None, s["q_out"].data_ptr())
        H.kv_q8_read(s["cache"], 0, s["cache"].max_seq, s["k_out"].data_ptr(), s["v_out"].data_ptr(), H.DTYPE_F32)
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    if kind == "attention":
        H.attention_q8(s["cache"], s["q"].data_ptr(), s["out"].data_ptr(), code, case["rows"], case["heads"],
                       s["pos"].data_ptr(), None, s["tree"].data_ptr() if s["tree"] is not None else None, 1.0,
                       s["ws"].data_ptr(), s["ws"].numel())
        return s["out"]
    H.logits_rules(s["rules"], s["logits"].data_ptr(), s["out"].data_ptr(), code, s["tokens"].data_ptr(),
                   case["seqs"], case["rows"], case["vocab"], None, s["ws"].data_ptr(), s["ws"].numel())
    return {"logits": s["out"], "tokens": s["tokens"]}


# ---- one pass: the plain forms ----------------------------------------------

def _bits(words, count):
    """The first `count` bits of each row of integer words, lowest first."""
    width = words.element_size() * 8
    shifts = torch.arange(width, device=DEV, dtype=words.dtype)
    return ((words[..., None] >> shifts) & 1).flatten(-2)[..., :count].bool()


def _plain_qmm_a8(s):
    a, dt = s["a"].float(), s["a"].dtype
    codes, sa = _quantise(a, 1)
    acc = torch.matmul(codes.double(), s["codes"].double())  # whole numbers past 24 bits
    return (acc.float() * (sa[:, None] * s["scales"][None, :])).to(dt)


def _plain_kv(s):
    case = s["case"]
    b, rows, heads, hk, d = (case[x] for x in ("batch", "rows", "heads", "kv_heads", "d"))
    x = s["qkv"].float().view(b, rows, heads + 2 * hk, d).transpose(1, 2)
    at = s["pos"].long()[:, None] + torch.arange(rows, device=DEV)
    angle = at if s["depths"] is None else s["pos"].long()[:, None] + s["depths"].long()
    c, n = s["cos"][angle][:, None], s["sin"][angle][:, None]
    lo, hi = x[:, :heads + hk, :, :d // 2], x[:, :heads + hk, :, d // 2:]
    y = torch.cat([lo * c - hi * n, hi * c + lo * n], -1)
    kc, ks = _quantise(y[:, heads:], -1)
    vc, vs = _quantise(x[:, heads + hk:], -1)
    seq = torch.arange(b, device=DEV)[:, None].expand(b, rows)
    # [b, rows, hk, ...] rows of the cache
    s["k_codes"][seq, :, at], s["k_scales"][seq, :, at] = kc.transpose(1, 2), ks.transpose(1, 2)
    s["v_codes"][seq, :, at], s["v_scales"][seq, :, at] = vc.transpose(1, 2), vs.transpose(1, 2)
    return {"q": y[:, :heads].to(s["qkv"].dtype), "k": s["k_codes"].float() * s["k_scales"][..., None],
            "v": s["v_codes"].float() * s["v_scales"][..., None]}


def _visible(s, total):
    """[batch, rows, keys]: which cache row each token sees."""
    rows = s["case"]["rows"]
    key = torch.arange(total, device=DEV)
    pos = s["pos"].long()
    node = key[None, :] - pos[:, None]  # the drafted token that a key is
    if s["tree"] is None:
        return node[:, None, :] <= torch.arange(rows, device=DEV)[None, :, None]
    sees = _bits(s["tree"], rows)
    inside = (node >= 0) & (node < rows)
    drafted = sees.gather(2, node.clamp(0, rows - 1)[:, None, :].expand(-1, rows, -1)) & inside[:, None, :]
    return drafted | (node < 0)[:, None, :]


def _plain_attention(s):
    case = s["case"]
    b, rows, heads, hk, d = (case[x] for x in ("batch", "rows", "heads", "kv_heads", "d"))
    g, total = heads // hk, case["past"] + rows
    k = s["k_codes"].float() * s["k_scales"][..., None]
    v = s["v_codes"].float() * s["v_scales"][..., None]
    q = s["q"].float().view(b, hk, g * rows, d)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(b, hk, g, rows, total)
    x = x.masked_fill(~_visible(s, total)[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p.view(b, hk, g * rows, total), v).view(b, hk, g, rows, d) / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(b, rows, heads * d).to(s["q"].dtype)


def _plain_logits(s):
    case = s["case"]
    seqs, rows, vocab, hist, nb = (case[x] for x in ("seqs", "rows", "vocab", "history", "bias"))
    x = s["logits"].float()
    told = (torch.arange(hist, device=DEV)[None, :] < s["lengths"][:, None]).float()
    seen = torch.zeros(seqs, vocab, device=DEV).scatter_add_(1, s["history"].long(), told)
    path = _bits(s["tree"], rows).float()  # [seqs, rows, rows]
    n = seen[:, None, :].expand(seqs, rows, vocab).contiguous()
    n.scatter_add_(2, s["drafted"].long()[:, None, :].expand(seqs, rows, rows), path)
    rep, freq, pres = (s[k][:, None, None] for k in ("repetition", "frequency", "presence"))
    hit = n > 0
    x = torch.where(hit, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(hit, x - n * freq - pres, x)
    # of entries for the same token the last one counts
    entry = torch.arange(nb, device=DEV)[None, :].expand(seqs, nb)
    entry = torch.where(entry < s["bias_lengths"][:, None], entry, -1)
    last = torch.full((seqs, vocab), -1, device=DEV).scatter_reduce_(1, s["bias_tokens"].long(), entry, "amax")
    bias = torch.where(last >= 0, s["bias_values"].gather(1, last.clamp(min=0)), 0.0)
    x = x + bias[:, None, :]
    x = x.masked_fill(~_bits(s["allowed"], vocab), -math.inf)
    best = x.amax(-1, keepdim=True)
    at = torch.where(x == best, torch.arange(vocab, device=DEV), vocab).amin(-1)
    tokens = torch.where(best[..., 0] > -math.inf, at, -1)
    return {"logits": x.to(s["logits"].dtype), "tokens": tokens.to(torch.int32)}


def run(state):
    if own:
        return _run_own(state)
    return {"qmm_a8": _plain_qmm_a8, "kv": _plain_kv, "attention": _plain_attention,
            "logits": _plain_logits}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    kind, e = case["kind"], _BYTES[case["dtype"]]
    if kind == "qmm_a8":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": k * n + 4 * n + e * m * (k + n), "flops": 2 * m * k * n}
    if kind == "logits":
        seqs, rows, vocab = case["seqs"], case["rows"], case["vocab"]
        return {"bytes": seqs * rows * (2 * e * vocab + vocab / 8 + 4) + seqs * (4 * case["history"] + 8 * case["bias"]),
                "flops": 6 * seqs * rows * vocab}
    b, rows, heads, hk, d = (case[x] for x in ("batch", "rows", "heads", "kv_heads", "d"))
    past = case["past"] if b == 1 else 0.75 * case["past"]  # ragged between a half and the whole
    if kind == "kv":
        written = b * rows * hk * 2 * (d + 4)
        back = b * hk * (case["past"] + rows) * 2 * (d + 4 + 4 * d)
        return {"bytes": b * rows * (e * (2 * heads + 2 * hk) * d + 4 * d) + written + back,
                "flops": b * rows * (heads + hk) * d * 3 + b * hk * (case["past"] + rows) * 2 * d}
    pairs = b * heads * rows * (past + (rows + 1) / 2)
    return {"bytes": b * hk * (past + rows) * 2 * (d + 4) + 2 * e * b * rows * heads * d, "flops": 4 * pairs * d}


# ---- the same in 64 bits ----------------------------------------------------

def _codes_of(x):
    """The cache's (and the activations') codes and scales of fp32 rows
    [..., n], as defined: fp32 steps, on the host."""
    x = x.cpu().numpy()
    amax = np.abs(x).max(-1, keepdims=True)
    scale = np.where(amax > 0, amax / np.float32(127), np.float32(1)).astype(np.float32)
    y = x * (np.float32(1) / scale)
    codes = np.copysign(np.floor(np.abs(y).astype(np.float64) + 0.5), y)
    return np.clip(codes, -127, 127), scale[..., 0].astype(np.float64)


def _exact_kv(case, seed):
    s = prepare(case, seed)
    b, rows, heads, hk, d = (case[x] for x in ("batch", "rows", "heads", "kv_heads", "d"))
    qkv, half = s["qkv"].float().cpu().numpy(), d // 2
    cos, sin, pos = s["cos"].cpu().numpy(), s["sin"].cpu().numpy(), s["pos"].cpu().numpy()
    out = {"q": np.empty((b, heads, rows, d)), "k": None, "v": None}
    cache = {}
    for kv in ("k", "v"):
        cache[kv] = s[kv + "_codes"].double().cpu().numpy() * s[kv + "_scales"].double().cpu().numpy()[..., None]
    for i in range(b):
        for t in range(rows):
            p = int(pos[i]) + t
            turn = p if s["depths"] is None else int(pos[i]) + int(s["depths"][i, t])
            x = qkv[i, t].reshape(heads + 2 * hk, d)
            re, im = x[:heads, :half].astype(np.float64), x[:heads, half:].astype(np.float64)
            c, n = cos[turn].astype(np.float64), sin[turn].astype(np.float64)
            out["q"][i, :, t] = np.concatenate([re * c - im * n, im * c + re * n], 1)
            # the key that is quantised is the one rotated in 32 bits
            re, im, c, n = x[heads:heads + hk, :half], x[heads:heads + hk, half:], cos[turn], sin[turn]
            key = np.concatenate([re * c - im * n, im * c + re * n], 1)
            for kv, rowsx in (("k", key), ("v", x[heads + hk:])):
                codes, scale = _codes_of(torch.from_numpy(np.ascontiguousarray(rowsx)))
                cache[kv][i, :, p] = codes * scale[:, None]
    return {"q": out["q"], **cache}


def _exact_attention(case, seed):
    b, rows, heads, hk, d = (case[x] for x in ("batch", "rows", "heads", "kv_heads", "d"))
    s = prepare(case, seed)
    g = heads // hk
    pos = s["pos"].tolist()
    words = None if s["tree"] is None else s["tree"].cpu().numpy().view(np.uint64)
    out = torch.empty(b, rows, heads, d, device=DEV, dtype=torch.float64)
    for i in range(b):
        n = pos[i] + rows
        sees = np.tri(rows, dtype=bool)
        if words is not None:
            sees = np.array([[int(words[i, t, j // 64]) >> (j % 64) & 1 for j in range(rows)] for t in range(rows)], bool)
        see = torch.ones(rows, n, device=DEV, dtype=torch.bool)
        see[:, pos[i]:] = torch.from_numpy(sees).to(DEV)
        for h in range(hk):
            k = s["k_codes"][i, h, :n].double() * s["k_scales"][i, h, :n].double()[:, None]
            v = s["v_codes"][i, h, :n].double() * s["v_scales"][i, h, :n].double()[:, None]
            for u in range(g):
                x = s["q"][i, h * g + u].double() @ k.T.contiguous()
                out[i, :, h * g + u] = torch.softmax(x.masked_fill(~see, -math.inf), -1) @ v
    return out.reshape(b, rows, heads * d)


def _exact_logits(case, seed):
    seqs, rows, vocab = case["seqs"], case["rows"], case["vocab"]
    s = prepare(case, seed)
    h = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "logits"}
    out = s["logits"].double().cpu().numpy()
    words = h["tree"].view(np.uint64)
    for i in range(seqs):
        seen = np.bincount(h["history"][i, :h["lengths"][i]], minlength=vocab).astype(np.float64)
        bias = np.zeros(vocab)
        for e in range(int(h["bias_lengths"][i])):
            bias[h["bias_tokens"][i, e]] = h["bias_values"][i, e]
        rep, freq, pres = (float(h[k][i]) for k in ("repetition", "frequency", "presence"))
        for t in range(rows):
            n = seen.copy()
            for j in range(rows):
                if int(words[i, t, j // 64]) >> (j % 64) & 1:
                    n[h["drafted"][i, j]] += 1
            x = out[i, t]
            hit = n > 0
            x[hit] = np.where(x[hit] > 0, x[hit] / rep, x[hit] * rep) - n[hit] * freq - pres
            x += bias
            on = np.unpackbits(h["allowed"][i, t].view(np.uint8), bitorder="little")[:vocab].astype(bool)
            x[~on] = -np.inf
    # the token is decided by values rounded to 32 bits
    return {"logits": out, "tokens": None}


def exact(case, seed):
    kind = case["kind"]
    if kind == "qmm_a8":
        s = prepare(case, seed)
        codes, sa = _codes_of(s["a"].float())
        sa = torch.from_numpy(sa).to(DEV)
        # whole numbers below 2^53
        acc = torch.from_numpy(codes.astype(np.float64)).to(DEV) @ s["codes"].double()
        return acc * sa[:, None] * s["scales"].double()[None, :]
    if kind == "kv":
        return _exact_kv(case, seed)
    if kind == "attention":
        return _exact_attention(case, seed)
    return _exact_logits(case, seed)
