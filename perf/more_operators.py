"""Performance cases of the operators of a step over a batch of requests that
share one pool of cache pages: what a server runs between its matrix products
when requests of different lengths come and go.

  plan    block tables, packed row offsets, positions and slots of a step from
          the requests' lengths and the pool's free pages (vm_hip_kv_paged_plan).
  rope    tables of the rotation's cosines and sines, frequencies scaled for
          contexts longer than the trained one (vm_hip_rope_tables).
  append  a norm of every query and key head, the rotation of part of the head
          in halves or pairs, and keys and values written to their pages
          (vm_hip_kv_paged_append), or left in rows (vm_hip_qk_norm_rope).
  packed  causal attention over whole prompts of different lengths, one behind
          the other, with grouped heads (vm_hip_attention_packed).
  paged   attention of single tokens and chunks of new tokens over the pages
          (vm_hip_attention_paged).

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
_SCALINGS = {"plain": 0, "linear": 1, "bands": 2, "ramp": 3}  # VM_HIP_ROPE_*


def _hip():
    """This repository's Python binding; used only where `own` is true."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "velo-mind_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import velomind_hip

    velomind_hip.load()
    return velomind_hip


# ---- the cases --------------------------------------------------------------

def _plan(name, batch, past, new, page, spare):
    return dict(name=name, kind="plan", batch=batch, past=past, new=new, page=page, spare=spare)


def _rope(name, rows, dim, theta, scaling, factor, original):
    return dict(name=name, kind="rope", rows=rows, dim=dim, theta=theta, scaling=scaling, factor=factor,
                original=original)


def _append(name, dtype, batch, rows, past, heads, kv_heads, d, page, rotary, pairs, norm, cache):
    return dict(name=name, kind="append", dtype=dtype, batch=batch, rows=rows, past=past, heads=heads,
                kv_heads=kv_heads, d=d, page=page, rotary=rotary, pairs=pairs, norm=norm, cache=cache)


def _packed(name, dtype, batch, rows, heads, kv_heads, d):
    return dict(name=name, kind="packed", dtype=dtype, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, d=d)


def _paged(name, dtype, batch, past, chunk, heads, kv_heads, d, page):
    return dict(name=name, kind="paged", dtype=dtype, batch=batch, past=past, chunk=chunk, heads=heads,
                kv_heads=kv_heads, d=d, page=page)


def listed():
    return [
        # A decoding step of 32 requests: one token each, latency.
        _plan("plan_b32_1_of_2000", 32, 2000, 1, 16, 1.0),
        # Prompts' chunks of 256 requests, more pages wanted than are free.
        _plan("plan_b256_500_of_8000", 256, 8000, 500, 16, 0.9),
        # TinyLlama's tables, as a session of 2000 tokens starts with.
        _rope("rope_2000x64", 2000, 64, 10000.0, "plain", 1.0, 2048),
        # A 128K context of 128-wide heads, the slow frequencies stretched.
        _rope("rope_131072x128_ramp", 131072, 128, 500000.0, "ramp", 16.0, 8192),
        # One decoded TinyLlama token.
        _append("append_1_tinyllama", "f32", 1, 1, 511, 32, 4, 64, 16, 64, False, False, True),
        # Prompts of a 70B-class layer with head norms, half of the head rotated in pairs.
        _append("append_4000_norm_pairs", "bf16", 8, 4000, 1000, 64, 8, 128, 64, 64, True, True, True),
        # Seven short prompts of SmolLM2-360M (15 heads on 5): latency and ragged tiles.
        _packed("packed_7_of_700", "f16", 7, 700, 15, 5, 64),
        # Two TinyLlama prompts in the framework's own fp32.
        _packed("packed_2_of_2000_f32", "f32", 2, 2000, 32, 4, 64),
        # Long prompts of a 70B-class layer: the matrix cores.
        _packed("packed_3_of_12000", "bf16", 3, 12000, 64, 8, 128),
        # One TinyLlama layer's attention of one decoded token: latency.
        _paged("paged_decode_2000", "f32", 1, 1999, 1, 32, 4, 64, 16),
        # Decoding 32 requests of ragged lengths up to 8 K: bandwidth.
        _paged("paged_decode_b32_8000", "bf16", 32, 7999, 1, 64, 8, 128, 16),
        # A chunk of a long prompt next to seven decoding requests.
        _paged("paged_chunk500_30000", "f16", 8, 30000, 500, 32, 8, 128, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "append", "append", "packed", "packed", "paged", "paged", "paged"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if kind == "plan":
        batch, new = _log(rng, 1, 1000), rng.choice([1, _log(rng, 1, 500)])
        return dict(kind=kind, batch=batch, past=_log(rng, 1, 8000), new=min(new, max(1, 100000 // batch)), page=page,
                    spare=rng.choice([1.0, 1.0, 0.5]))
    if kind == "rope":
        return dict(kind=kind, rows=_log(rng, 1, 120000), dim=2 * rng.randint(8, 64),
                    theta=rng.choice([10000.0, 100000.0, 500000.0]), scaling=rng.choice(list(_SCALINGS)),
                    factor=float(rng.choice([2, 4, 8, 32])), original=rng.choice([2048, 4096, 8192]))
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    d = rng.choice([64, 128])
    if kind == "append":
        batch = _log(rng, 1, 32)
        return dict(kind=kind, dtype=dtype, batch=batch, rows=max(batch, _log(rng, 1, 4000)), past=_log(rng, 1, 2000),
                    heads=heads, kv_heads=kv_heads, d=d, page=page, rotary=rng.choice([d, d, d // 2, d // 4 + 2]),
                    pairs=rng.random() < 0.5, norm=rng.random() < 0.5, cache=rng.random() < 0.7)
    if kind == "packed":
        batch = _log(rng, 1, 40)
        return dict(kind=kind, dtype=dtype, batch=batch, rows=max(batch, _log(rng, 1, 6500 if dtype != "f32" else 2500)),
                    heads=heads, kv_heads=kv_heads, d=d)
    batch = _log(rng, 1, 40)
    chunk = rng.choice([1, 1, _log(rng, 2, 30), _log(rng, 30, 600)])
    most = 100000 if chunk <= 30 else 30000 if dtype != "f32" else 4000
    return dict(kind=kind, dtype=dtype, batch=batch, past=_log(rng, 1, min(most, 250000 // batch)), chunk=chunk,
                heads=heads, kv_heads=kv_heads, d=d, page=page)


# ---- inputs -----------------------------------------------------------------

def _gen(seed, salt=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1009 + salt)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def _split(total, parts):
    """`total` rows shared out to `parts` sequences of different lengths, one row each at least."""
    r = np.random.default_rng(total + 11)
    share = r.uniform(0.2, 1.0, parts)
    n = 1 + np.floor((total - parts) * share / share.sum()).astype(np.int64)
    n[int(r.integers(parts))] += total - n.sum()
    return n


def _pages(lengths, page, seed, spare=0):
    """Tables of sequences of these lengths over a pool whose pages have been
    handed out in no order, the pages that are left, and how many there are."""
    r = np.random.default_rng(seed + 23)
    need = -(-np.asarray(lengths) // page)
    count = int(need.sum()) + spare
    order = r.permutation(count)
    tables = np.full((len(need), max(1, int(need.max()))), -1, np.int64)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    return tables, order[at:], count


def _frequencies(case):
    """[dim / 2] in 64 bits."""
    dim, theta, factor, original = case["dim"], case["theta"], case["factor"], case["original"]
    f = theta ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)
    if case["scaling"] == "linear":
        return f / factor
    if case["scaling"] == "bands":
        # 1 turn in the trained length and fewer: stretched; 4 and more: not
        turns = original * f / (2 * np.pi)
        keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0, 1)
        return f * keep + f / factor * (1 - keep)
    if case["scaling"] == "ramp":
        # the same by pair index, between the pairs of 32 turns and of 1
        at = [dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        r = np.clip((np.arange(dim // 2) - low) / max(high - low, 0.001), 0, 1)
        return f / factor * r + f * (1 - r)
    return f


def _attention_factor(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "ramp" else 1.0


def _prepare_plan(case, seed):
    r = np.random.default_rng(seed)
    b, page = case["batch"], case["page"]
    lengths = r.integers((case["past"] + 1) // 2, case["past"] + 1, b)
    counts = r.integers((case["new"] + 1) // 2, case["new"] + 1, b)
    lengths[r.integers(b)] = 0                       # a request's first step
    idle = r.random(b) < 0.05                        # and requests that wait
    counts[idle & (np.arange(b) > 0)] = 0
    wanted = int((-(-(lengths + counts) // page) - -(-lengths // page)).sum())
    tables, free, pages = _pages(lengths, page, seed, spare=max(1, int(wanted * case["spare"])))
    width = -(-(case["past"] + case["new"]) // page)
    wide = np.full((b, width), -1, np.int64)
    wide[:, :tables.shape[1]] = tables
    # as many rows as every request's largest chunk would fill
    s = dict(lengths=_ints(lengths), counts=_ints(counts), tables=_ints(wide), free=_ints(free),
             free_count=_ints([len(free)]), rows=b * case["new"], width=width)
    if own:
        H = _hip()
        s["H"] = H
        s["out"] = {k: torch.empty(n, device=DEV, dtype=torch.int32) for k, n in
                    (("row_start", b + 1), ("lengths", b), ("free_count", 1), ("positions", s["rows"]),
                     ("slots", s["rows"]))}
        s["ws"] = torch.zeros(H.kv_paged_plan_workspace_bytes(b, s["rows"]), device=DEV, dtype=torch.uint8)
        o = s["out"]
        s["plan"] = H.PagePlan(batch=b, rows=s["rows"], max_pages=width, pages=pages, page_size=page,
                               lengths=s["lengths"].data_ptr(), counts=s["counts"].data_ptr(),
                               free_pages=s["free"].data_ptr(), free_count=s["free_count"].data_ptr(),
                               tables=s["tables"].data_ptr(), row_start=o["row_start"].data_ptr(),
                               lengths_out=o["lengths"].data_ptr(), free_count_out=o["free_count"].data_ptr(),
                               positions=o["positions"].data_ptr(), slots=o["slots"].data_ptr())
    return s


def _prepare_rope(case, seed):
    # another seed: the tables of another base
    theta = case["theta"] * (1.0 + (seed % 97) / 97.0)
    s = dict(theta=theta)
    if own:
        H = _hip()
        s["H"] = H
        s["cos"], s["sin"] = (torch.empty(case["rows"], case["dim"] // 2, device=DEV) for _ in "cs")
        s["scaling"] = H.RopeScaling(kind=_SCALINGS[case["scaling"]], factor=case["factor"],
                                     low=1.0, high=4.0 if case["scaling"] == "bands" else 32.0,
                                     original=case["original"], attention=_attention_factor(case))
    return s


def _prepare_append(case, seed):
    b, heads, hk, d, page = (case[x] for x in ("batch", "heads", "kv_heads", "d", "page"))
    r = np.random.default_rng(seed)
    n = _split(case["rows"], b)
    past = r.integers(case["past"] // 2, case["past"] + 1, b)
    pool = int((-(-(case["past"] + n) // page)).sum())   # what the longest contexts would take
    held = int((-(-(past + n) // page)).sum())
    tables, _, pages = _pages(past + n, page, seed, spare=pool - held)
    positions = np.concatenate([p + np.arange(c) for p, c in zip(past, n)])
    seq = np.repeat(np.arange(b), n)
    slots = tables[seq, positions // page] * page + positions % page
    g = _gen(seed)
    s = dict(qkv=_randn(g, case["rows"], (heads + 2 * hk) * d).to(_TORCH[case["dtype"]]),
             positions=_ints(positions), slots=_ints(slots))
    f = torch.from_numpy(10000.0 ** (-np.arange(0, case["rotary"], 2) / case["rotary"])).to(DEV)
    angle = torch.arange(int((past + n).max()), device=DEV, dtype=torch.float64)[:, None] * f
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if case["norm"]:
        s["q_norm"], s["k_norm"] = 1 + 0.1 * _randn(g, d), 1 + 0.1 * _randn(g, d)
    if case["cache"]:
        shape = (pages, hk, page, d)
        s["k"], s["v"] = (_randn(g, *shape).to(_TORCH[case["dtype"]]) for _ in "kv")
    if own:
        H = _hip()
        s["H"] = H
        s["q_out"] = torch.empty(case["rows"], heads * d, device=DEV, dtype=s["qkv"].dtype)
        if case["cache"]:
            s["cache"] = H.KvPaged(s["k"].data_ptr(), s["v"].data_ptr(), _CODE[case["dtype"]], pages, page, hk, d)
        else:
            s["k_out"] = torch.empty(case["rows"], hk * d, device=DEV, dtype=s["qkv"].dtype)
        s["rope"] = H.Rope(s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], case["rotary"],
                           1 if case["pairs"] else 0)
        s["head_norm"] = H.QkNorm(s["q_norm"].data_ptr(), s["k_norm"].data_ptr(), 1e-6) if case["norm"] else None
    return s


def _prepare_packed(case, seed):
    b, rows, heads, hk, d = (case[x] for x in ("batch", "rows", "heads", "kv_heads", "d"))
    n = _split(rows, b)
    dt = _TORCH[case["dtype"]]
    # one projection's rows: q | k | v
    qkv = _randn(_gen(seed), rows, (heads + 2 * hk) * d).to(dt)
    start = np.concatenate([[0], np.cumsum(n)])
    s = dict(qkv=qkv, start=start.tolist(), row_start=_ints(start))
    if own:
        H = _hip()
        s["H"], s["out"] = H, torch.empty(rows, heads * d, device=DEV, dtype=dt)
        nbytes = H.attention_packed_workspace_bytes(b, rows, heads, hk, d)
        s["ws"] = torch.zeros(max(1, nbytes), device=DEV, dtype=torch.uint8)
    return s


def _paged_lengths(case, seed):
    """(new tokens, tokens behind them) of each sequence: the first one has
    the whole chunk behind the longest context, the others one token."""
    r = np.random.default_rng(seed)
    b, past = case["batch"], case["past"]
    n = np.ones(b, np.int64)
    n[0] = case["chunk"]
    before = r.integers(past // 2, past + 1, b)
    before[0] = past
    return n, before


def _prepare_paged(case, seed):
    b, heads, hk, d, page = (case[x] for x in ("batch", "heads", "kv_heads", "d", "page"))
    dt = _TORCH[case["dtype"]]
    n, before = _paged_lengths(case, seed)
    tables, _, pages = _pages(before + n, page, seed)
    rows = int(n.sum())
    g = _gen(seed)
    start = np.concatenate([[0], np.cumsum(n)])
    s = dict(q=_randn(g, rows, heads * d).to(dt), tables=_ints(tables), row_start=_ints(start),
             lengths=_ints(before + n), n=n.tolist(), total=(before + n).tolist())
    # keys with a few large channels, values without
    channel = torch.where(torch.arange(d, device=DEV) % 17 == 3, 3.0, 1.0)
    s["k"] = torch.empty(pages, hk, page, d, device=DEV, dtype=dt)
    s["v"] = torch.empty_like(s["k"])
    s["k"].normal_(generator=g).mul_(channel.to(dt))
    s["v"].normal_(generator=g)
    if own:
        H = _hip()
        s["H"], s["out"] = H, torch.empty(rows, heads * d, device=DEV, dtype=dt)
        s["cache"] = H.KvPaged(s["k"].data_ptr(), s["v"].data_ptr(), _CODE[case["dtype"]], pages, page, hk, d)
        nbytes = H.attention_paged_workspace_bytes(b, rows, case["chunk"], heads, hk, d, tables.shape[1] * page)
        s["ws"] = torch.zeros(max(1, nbytes), device=DEV, dtype=torch.uint8)
    return s


def prepare(case, seed):
    s = {"plan": _prepare_plan, "rope": _prepare_rope, "append": _prepare_append, "packed": _prepare_packed,
         "paged": _prepare_paged}[case["kind"]](case, seed)
    s["case"] = case
    return s


# ---- one pass: this framework's calls ---------------------------------------

def _run_own(s):
    H, case = s["H"], s["case"]
    kind = case["kind"]
    if kind == "plan":
        H.kv_paged_plan(s["plan"], s["ws"].data_ptr(), s["ws"].numel())
        return {"tables": s["tables"], **s["out"]}
    if kind == "rope":
        H.rope_tables(s["cos"].data_ptr(), s["sin"].data_ptr(), 0, case["rows"], case["dim"], s["theta"], s["scaling"])
        return {"cos": s["cos"], "sin": s["sin"]}
    code, heads, hk, d = (_CODE[case["dtype"]], case["heads"], case["kv_heads"], case["d"])
    if kind == "append":
        if case["cache"]:
            H.kv_paged_append(s["cache"], s["qkv"].data_ptr(), case["rows"], heads, s["head_norm"], s["rope"],
                              s["positions"].data_ptr(), s["slots"].data_ptr(), s["q_out"].data_ptr())
            return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
        H.qk_norm_rope(s["qkv"].data_ptr(), code, case["rows"], heads, hk, d, s["head_norm"], s["rope"],
                       s["positions"].data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr())
        return {"q": s["q_out"], "k": s["k_out"]}
    if kind == "packed":
        width, at, size = (heads + 2 * hk) * d, s["qkv"].data_ptr(), s["qkv"].element_size()
        H.attention_packed(at, at + heads * d * size, at + (heads + hk) * d * size, s["out"].data_ptr(), code, width,
                           width, width, case["batch"], case["rows"], heads, hk, d, s["row_start"].data_ptr(), 0.0,
                           s["ws"].data_ptr(), s["ws"].numel())
        return s["out"]
    H.attention_paged(s["cache"], s["tables"].data_ptr(), s["tables"].shape[1], s["q"].data_ptr(), s["out"].data_ptr(),
                      case["batch"], s["q"].shape[0], case["chunk"], heads, s["row_start"].data_ptr(),
                      s["lengths"].data_ptr(), 0.0, s["ws"].data_ptr(), s["ws"].numel())
    return s["out"]


# ---- one pass: the plain forms ----------------------------------------------

def _plain_plan(s):
    page, rows = s["case"]["page"], s["rows"]
    lengths, counts, free = s["lengths"].long(), s["counts"].long(), s["free"]
    total = lengths + counts
    held = (lengths + page - 1) // page
    want = (total + page - 1) // page - held
    asked = torch.cumsum(want, 0)
    # requests that find too few free pages wait, and so do those behind them that want any
    admitted = (asked <= s["free_count"]) | (want == 0)
    counts, want = torch.where(admitted, counts, 0), torch.where(admitted, want, 0)
    start = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)])
    top = s["free_count"].long() - (torch.cumsum(want, 0) - want)
    column = torch.arange(s["width"], device=DEV)
    which = column - held[:, None]
    new = (which >= 0) & (which < want[:, None])
    picked = free[(top[:, None] - 1 - which).clamp(0, free.numel() - 1)]
    tables = torch.where(new, picked, s["tables"])
    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(start, row, right=True) - 1
    real = row < start[-1]
    seq = torch.where(real, seq, 0)
    position = lengths[seq] + row - start[seq]
    slot = tables[seq, (position // page).clamp(max=s["width"] - 1)].long() * page + position % page
    i32 = torch.int32
    return {"tables": tables, "row_start": start.to(i32), "lengths": (lengths + counts).to(i32),
            "free_count": (s["free_count"] - want.sum()).to(i32), "positions": torch.where(real, position, -1).to(i32),
            "slots": torch.where(real, slot, -1).to(i32)}


def _plain_rope(s):
    case = s["case"]
    f = torch.from_numpy(_frequencies({**case, "theta": s["theta"]})).to(DEV)
    angle = torch.arange(case["rows"], device=DEV, dtype=torch.float64)[:, None] * f
    m = _attention_factor(case)
    return {"cos": (torch.cos(angle) * m).float(), "sin": (torch.sin(angle) * m).float()}


def _plain_append(s):
    case = s["case"]
    rows, heads, hk, d, rotary = (case[x] for x in ("rows", "heads", "kv_heads", "d", "rotary"))
    dt = s["qkv"].dtype
    x = s["qkv"].float().view(rows, heads + 2 * hk, d)
    qk = x[:, :heads + hk]
    if case["norm"]:
        w = torch.cat([s["q_norm"].expand(heads, d), s["k_norm"].expand(hk, d)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    at = s["positions"].long()
    c, n = s["cos"][at][:, None], s["sin"][at][:, None]
    turned, kept = qk[..., :rotary], qk[..., rotary:]
    if case["pairs"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    y = torch.cat([turned, kept], -1).to(dt)
    q = y[:, :heads].reshape(rows, heads * d)
    if not case["cache"]:
        return {"q": q, "k": y[:, heads:].reshape(rows, hk * d)}
    page, slot = case["page"], s["slots"].long()
    s["k"][slot // page, :, slot % page] = y[:, heads:]
    s["v"][slot // page, :, slot % page] = x[:, heads + hk:].to(dt)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_heads(q, k, v, first, scale):
    """Attention of q [n, hk, g, d] over k, v [keys, hk, d] in 32 bits: row i sees
    keys up to first + i."""
    n, hk, g, d = q.shape
    keys = k.shape[0]
    out = torch.empty(n, hk, g, d, device=DEV)
    hidden = torch.arange(keys, device=DEV)[None, :] > first + torch.arange(n, device=DEV)[:, None]
    step = max(1, int(2 ** 28 // max(1, n * keys)))   # heads whose scores are held at once
    for h in range(hk):
        kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
        for u in range(0, g, step):
            w = min(step, g - u)
            x = torch.matmul(q[:, h, u:u + w].transpose(0, 1).reshape(w * n, d), kt).view(w, n, keys) * scale
            x.masked_fill_(hidden, -math.inf)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.matmul(p.view(w * n, keys), vh) / p.sum(-1).view(w * n, 1)
            out[:, h, u:u + w] = o.view(w, n, d).transpose(0, 1)
    return out


def _plain_packed(s):
    case = s["case"]
    rows, heads, hk, d = (case[x] for x in ("rows", "heads", "kv_heads", "d"))
    x = s["qkv"].float().view(rows, heads + 2 * hk, d)
    parts = []
    for a, b in zip(s["start"][:-1], s["start"][1:]):
        q = x[a:b, :heads].reshape(b - a, hk, heads // hk, d)
        parts.append(_plain_heads(q, x[a:b, heads:heads + hk], x[a:b, heads + hk:], 0, d ** -0.5))
    return torch.cat(parts).reshape(rows, heads * d).to(s["qkv"].dtype)


def _plain_paged(s):
    case = s["case"]
    heads, hk, d, page = (case[x] for x in ("heads", "kv_heads", "d", "page"))
    parts, at = [], 0
    for i, (n, total) in enumerate(zip(s["n"], s["total"])):
        pages = s["tables"][i, :-(-total // page)].long()
        k, v = (s[x][pages].float().transpose(1, 2).reshape(-1, hk, d)[:total] for x in "kv")
        q = s["q"][at:at + n].float().view(n, hk, heads // hk, d)
        parts.append(_plain_heads(q, k, v, total - n, d ** -0.5))
        at += n
    return torch.cat(parts).reshape(at, heads * d).to(s["q"].dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "rope": _plain_rope, "append": _plain_append, "packed": _plain_packed,
            "paged": _plain_paged}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "plan":
        # lengths (in and out), counts and offsets of each request; a position
        # and a slot of each row; the pages handed out, read and written (means
        # of what is drawn)
        rows = case["batch"] * case["new"]
        return {"bytes": 16 * case["batch"] + 8 * rows + 8 * 0.71 * rows / case["page"], "flops": 4 * rows}
    if kind == "rope":
        return {"bytes": 4 * case["rows"] * case["dim"], "flops": 2 * case["rows"] * case["dim"]}
    e = _BYTES[case["dtype"]]
    heads, hk, d = case["heads"], case["kv_heads"], case["d"]
    if kind == "append":
        rows = case["rows"]
        moved = (heads + 2 * hk) * 2 if case["cache"] else (heads + hk) * 2
        return {"bytes": rows * (e * moved * d + 4 * case["rotary"] + 8),
                "flops": rows * (heads + hk) * (3 * case["rotary"] + (4 * d if case["norm"] else 0))}
    if kind == "packed":
        n = _split(case["rows"], case["batch"]).astype(float)
        return {"bytes": e * case["rows"] * (2 * heads + 2 * hk) * d, "flops": 2 * heads * d * float((n * (n + 1)).sum())}
    b, past, chunk = case["batch"], case["past"], case["chunk"]
    keys = past + chunk + (b - 1) * (0.75 * past + 1)
    pairs = chunk * past + chunk * (chunk + 1) / 2 + (b - 1) * (0.75 * past + 1)
    return {"bytes": e * d * (2 * hk * keys + 2 * heads * (chunk + b - 1)), "flops": 4 * heads * d * pairs}


# ---- the same in 64 bits ----------------------------------------------------

def _exact_plan(case, seed):
    s = prepare(case, seed)
    page, rows = case["page"], s["rows"]
    lengths, counts, free = (s[k].tolist() for k in ("lengths", "counts", "free"))
    tables = s["tables"].cpu().numpy().copy()
    left, short = len(free), False
    start, after, positions, slots = [0], [], [], []
    for b, (n, c) in enumerate(zip(lengths, counts)):
        held, want = -(-n // page), -(-(n + c) // page) - -(-n // page)
        if want > 0 and (short or want > left):
            short, c, want = True, 0, 0
        for j in range(want):
            left -= 1
            tables[b, held + j] = free[left]
        for p in range(n, n + c):
            positions.append(p)
            slots.append(int(tables[b, p // page]) * page + p % page)
        start.append(start[-1] + c)
        after.append(n + c)
    pad = [-1] * (rows - len(positions))
    out = dict(tables=tables, row_start=start, lengths=after, free_count=[left], positions=positions + pad,
               slots=slots + pad)
    return {k: _ints(v) for k, v in out.items()}


def _exact_rope(case, seed):
    theta = prepare(case, seed)["theta"]
    angle = np.multiply.outer(np.arange(case["rows"], dtype=np.float64), _frequencies({**case, "theta": theta}))
    turn = np.exp(1j * angle) * _attention_factor(case)
    return {"cos": np.ascontiguousarray(turn.real), "sin": np.ascontiguousarray(turn.imag)}


def _exact_append(case, seed):
    s = prepare(case, seed)
    rows, heads, hk, d, rotary = (case[x] for x in ("rows", "heads", "kv_heads", "d", "rotary"))
    at = s["positions"].long()
    turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())
    half = rotary // 2
    first = torch.arange(half, device=DEV) * (2 if case["pairs"] else 1)
    second = first + (1 if case["pairs"] else half)
    out = []
    for h in range(heads + 2 * hk):
        x = s["qkv"][:, h * d:(h + 1) * d].double()
        if h < heads + hk:
            if case["norm"]:
                w = s["q_norm"] if h < heads else s["k_norm"]
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6) * w.double()
            z = torch.complex(x[:, first], x[:, second]) * turn
            x = x.clone()
            x[:, first], x[:, second] = z.real, z.imag
        out.append(x)
    q = torch.cat(out[:heads], 1)
    if not case["cache"]:
        return {"q": q, "k": torch.cat(out[heads:heads + hk], 1)}
    got = {}
    for name, parts in (("k", out[heads:heads + hk]), ("v", out[heads + hk:])):
        pages, _, page, _ = s[name].shape
        flat = s[name].double().transpose(0, 1).reshape(hk, pages * page, d).clone()
        for h, x in enumerate(parts):
            flat[h, s["slots"].long()] = x
        got[name] = flat.view(hk, pages, page, d).transpose(0, 1)
    return {"q": q, **got}


def _exact_rows(q, k, v, first):
    """Attention of one head's rows q [n, d] over k, v [keys, d], in 64 bits, a
    few hundred rows at a time over the keys that any of them sees."""
    out = torch.empty(q.shape, device=DEV, dtype=torch.float64)
    for a in range(0, q.shape[0], 512):
        b = min(a + 512, q.shape[0])
        seen = first + b
        x = torch.matmul(q[a:b].double(), k[:seen].double().t().contiguous()) / math.sqrt(q.shape[1])
        last = first + torch.arange(a, b, device=DEV)
        x = torch.where(torch.arange(seen, device=DEV) <= last[:, None], x, -math.inf)
        out[a:b] = torch.matmul(torch.softmax(x, -1), v[:seen].double())
    return out


def _exact_packed(case, seed):
    s = prepare(case, seed)
    heads, hk, d = case["heads"], case["kv_heads"], case["d"]
    out = torch.empty(case["rows"], heads * d, device=DEV, dtype=torch.float64)
    for a, b in zip(s["start"][:-1], s["start"][1:]):
        x = s["qkv"][a:b]
        for h in range(heads):
            kh = heads + h // (heads // hk)
            out[a:b, h * d:(h + 1) * d] = _exact_rows(x[:, h * d:(h + 1) * d], x[:, kh * d:(kh + 1) * d],
                                                      x[:, (kh + hk) * d:(kh + hk + 1) * d], 0)
    return out


def _exact_paged(case, seed):
    s = prepare(case, seed)
    heads, hk, d, page = (case[x] for x in ("heads", "kv_heads", "d", "page"))
    out = torch.empty(s["q"].shape, device=DEV, dtype=torch.float64)
    at = 0
    for i, (n, total) in enumerate(zip(s["n"], s["total"])):
        token = torch.arange(total, device=DEV)
        page_of = s["tables"][i].long()[token // page]
        for h in range(hk):
            k, v = s["k"][page_of, h, token % page], s["v"][page_of, h, token % page]
            for u in range(h * (heads // hk), (h + 1) * (heads // hk)):
                out[at:at + n, u * d:(u + 1) * d] = _exact_rows(s["q"][at:at + n, u * d:(u + 1) * d], k, v, total - n)
        at += n
    return out


def exact(case, seed):
    return {"plan": _exact_plan, "rope": _exact_rope, "append": _exact_append, "packed": _exact_packed,
            "paged": _exact_paged}[case["kind"]](case, seed)
