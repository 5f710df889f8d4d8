"""Serving from a paged key-value cache, as cases that can be timed.

The operators, each in a plain form (elementary torch operations in 32 bits,
64 where scores next to one another are ordered) and, where ``own`` is true,
through the framework's entry points:

* ``decode``  -- ``paged_attention_decode``: one new token of every sequence
                 over its pages, whole or through a window with sinks;
* ``append``  -- ``paged_kv_append``: rotary positions on q and k, k and v
                 written into the sequences' pages;
* ``copy``    -- ``copy_kv_pages``: pages of every layer copied at once, as a
                 fork of sequences or a compaction of the pool asks for it;
* ``window``  -- ``window_attention``: a prompt's attention through a sliding
                 window, the first tokens staying visible;
* ``chunk``   -- ``paged_attention_prefill``: new tokens of every sequence over
                 a prefix that is in pages already;
* ``beam``    -- ``beam_select``: the best continuations of every beam search.

Inputs are made from the seed; lengths come from the case, so that its work
does not depend on the seed.
"""

from __future__ import annotations

import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
# (query heads, KV heads, head size) of the models the framework names, and their RoPE bases
HEADS = {"gpt2": (12, 12, 64), "smollm2-135m": (9, 3, 64), "smollm2-360m": (15, 5, 64), "llama3.2-3b": (24, 8, 128)}
THETA = {"gpt2": 1e4, "smollm2-135m": 1e4, "smollm2-360m": 1e4, "llama3.2-3b": 5e5}


def listed():
    return [
        # One sequence's token with a short prompt behind it, in the reference's own type: latency counts.
        {"name": "decode-one-fp32", "kind": "decode", "model": "smollm2-135m", "dtype": "float32", "batch": 1,
         "page": 16, "max_ctx": 2048, "lo": 100, "hi": 100, "lens": 1, "window": 0, "sinks": 0},
        # An ordinary serving batch behind a sliding window of no round length.
        {"name": "decode-window-fp16", "kind": "decode", "model": "smollm2-360m", "dtype": "float16", "batch": 32,
         "page": 16, "max_ctx": 8192, "lo": 512, "hi": 8191, "lens": 3, "window": 1000, "sinks": 4},
        # The largest decode: 64 long sequences, 2.6 GB of pages read for a token of each.
        {"name": "decode-long-bf16", "kind": "decode", "model": "llama3.2-3b", "dtype": "bfloat16", "batch": 64,
         "page": 64, "max_ctx": 16384, "lo": 4096, "hi": 16383, "lens": 4, "window": 0, "sinks": 0},
        # The cache write of one decode step of a batch: launch and latency.
        {"name": "append-step-bf16", "kind": "append", "model": "llama3.2-3b", "dtype": "bfloat16", "batch": 64,
         "page": 16, "max_ctx": 4096, "lo": 1, "hi": 4095, "lens": 5, "new": 1, "rotary": 128, "pairs": "half"},
        # Prompts of unequal length, padded to the longest; interleaved pairs over half of each head.
        {"name": "append-prompts-fp16", "kind": "append", "model": "smollm2-360m", "dtype": "float16", "batch": 8,
         "page": 32, "max_ctx": 4096, "lo": 0, "hi": 777, "lens": 6, "new": 1999, "rotary": 32,
         "pairs": "interleaved"},
        # Beams part: the last, half-filled page of three beams, in every layer.
        {"name": "copy-fork-fp32", "kind": "copy", "model": "smollm2-135m", "dtype": "float32", "layers": 30,
         "page": 16, "pages": 64, "moved": 3},
        # A pool is compacted: half of its pages move.
        {"name": "copy-compact-bf16", "kind": "copy", "model": "llama3.2-3b", "dtype": "bfloat16", "layers": 16,
         "page": 64, "pages": 256, "moved": 120},
        # A prompt in the reference's own type.
        {"name": "window-1023-fp32", "kind": "window", "model": "smollm2-360m", "dtype": "float32", "batch": 1,
         "seq": 1023, "window": 256, "sinks": 4},
        # A long prompt, most of it outside of any row's window.
        {"name": "window-8192-bf16", "kind": "window", "model": "llama3.2-3b", "dtype": "bfloat16", "batch": 1,
         "seq": 8192, "window": 1024, "sinks": 4},
        # Questions on documents that are in the cache already.
        {"name": "chunk-500-fp16", "kind": "chunk", "model": "smollm2-360m", "dtype": "float16", "batch": 4,
         "page": 32, "max_ctx": 4608, "lo": 1000, "hi": 4000, "lens": 7, "new": 500, "window": 0, "sinks": 0},
        # A beam search's step at GPT-2's vocabulary.
        {"name": "beam-4-fp32", "kind": "beam", "dtype": "float32", "batch": 1, "beams": 4, "vocab": 50257,
         "select": 8},
        # A batch of beam searches at Llama-3.2's.
        {"name": "beam-16x8-bf16", "kind": "beam", "dtype": "bfloat16", "batch": 16, "beams": 8, "vocab": 128256,
         "select": 16},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "append", "copy", "window", "chunk", "beam"])
    model = rng.choice(sorted(HEADS))
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    case = {"kind": kind, "model": model, "dtype": dtype}
    window = rng.choice([0, _log(rng, 16, 4096)])
    sinks = rng.choice([0, 1, 4, 37]) if window else 0
    if kind == "decode":
        ctx = -(-_log(rng, 128, 12000) // page) * page
        lo = rng.randint(1, max(1, ctx // 2))
        batch = _log(rng, 1, max(1, min(96, 300000 // ctx)))
        return {**case, "batch": batch, "page": page, "max_ctx": ctx, "lo": lo, "hi": rng.randint(lo, ctx),
                "lens": rng.randint(0, 1 << 20), "window": window, "sinks": sinks}
    if kind == "append":
        new = rng.choice([1, _log(rng, 2, 3000)])
        batch = _log(rng, 1, 64 if new == 1 else max(1, min(16, 12000 // new)))
        ctx = -(-(new + _log(rng, 16, 3000)) // page) * page
        D = HEADS[model][2]
        return {**case, "batch": batch, "page": page, "max_ctx": ctx, "lo": 0, "hi": ctx - new,
                "lens": rng.randint(0, 1 << 20), "new": new, "rotary": rng.choice([D, D, D // 2, D // 4]),
                "pairs": rng.choice(["half", "interleaved"])}
    if kind == "copy":
        H, Hkv, D = HEADS[model]
        layers = rng.randint(1, 32)
        most = max(4, (1 << 30) // (2 * layers * Hkv * page * D * SIZE[dtype]))
        pages = _log(rng, 4, min(2000, most))
        return {**case, "layers": layers, "page": page, "pages": pages, "moved": _log(rng, 1, pages // 2)}
    if kind == "window":
        seq = _log(rng, 1, 2000 if dtype == "float32" else 7000)
        batch = _log(rng, 1, max(1, min(8, 6000 // seq)))
        return {**case, "batch": batch, "seq": seq, "window": window or _log(rng, 16, 2048), "sinks": sinks}
    if kind == "chunk":
        new = _log(rng, 2, 600 if dtype == "float32" else 2000)
        ctx = -(-(new + _log(rng, 16, 4000)) // page) * page
        return {**case, "batch": _log(rng, 1, max(1, min(8, 3000 // new))), "page": page, "max_ctx": ctx, "lo": 0,
                "hi": ctx - new, "lens": rng.randint(0, 1 << 20), "new": new, "window": window, "sinks": sinks}
    beams = _log(rng, 1, 12)
    vocab = _log(rng, 500, 128256)
    return {"kind": kind, "dtype": dtype, "batch": _log(rng, 1, max(1, min(64, 8000000 // (beams * vocab)))),
            "beams": beams, "vocab": vocab, "select": beams * rng.choice([1, 2, 2, 3])}


# ---- what a program has in hand ------------------------------------------------

class _Make:
    """Seeded inputs on the GPU."""

    def __init__(self, seed, dtype):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))
        self.dtype = dtype

    def normal(self, *shape, scale=1.0):
        if math.prod(shape) > 1 << 28:  # large pools: made in their own type, with no 32-bit copy
            return torch.empty(shape, dtype=TORCH[self.dtype], device="cuda").normal_(0.0, scale, generator=self.g)
        return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=self.g).to(TORCH[self.dtype])


def _lens(case):
    """Tokens that are in the cache of each sequence before the call (decode: the new one among them)."""
    return np.random.default_rng(case["lens"]).integers(case["lo"], case["hi"], size=case["batch"],
                                                        endpoint=True).astype(np.int32)


def _new_lens(case):
    """New tokens of each sequence: the first has all, the others part of them."""
    n = np.random.default_rng(case["lens"] + 1).integers(1, case["new"], size=case["batch"], endpoint=True)
    n[0] = case["new"]
    return n.astype(np.int32)


def _tables(case):
    """cos / sin (max_ctx, rotary / 2) in 32 bits, angles in 64."""
    r = case["rotary"]
    freq = THETA[case["model"]] ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    angle = torch.arange(case["max_ctx"], dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _page_table(case, held, seed):
    """(table (batch, max_ctx / page) int32 with -1 behind each sequence's pages, pages in the pool): every
    sequence's pages lie anywhere in the pool, a few are free."""
    need = -(-held.astype(np.int64) // case["page"])
    total = int(need.sum()) + 3
    table = np.full((case["batch"], case["max_ctx"] // case["page"]), -1, np.int32)
    table[np.arange(table.shape[1]) < need[:, None]] = np.random.default_rng(seed).permutation(total)[:int(need.sum())]
    return torch.from_numpy(table).cuda(), total


def _cuda(x):
    return torch.from_numpy(x).cuda()


def prepare(case, seed):
    kind, mk = case["kind"], _Make(seed, case["dtype"])
    s = {"case": case}
    if kind == "beam":
        # logits of a language model: a few high ones over a broad floor; beams apart by a few units of log probability
        rows = case["batch"] * case["beams"]
        s["logits"] = mk.normal(rows, case["vocab"], scale=2.5)
        s["scores"] = -torch.empty(case["batch"], case["beams"], device="cuda").uniform_(4.0, 9.0, generator=mk.g)
        return s
    H, Hkv, D = HEADS[case["model"]]
    if kind == "copy":
        s["pool"] = mk.normal(2 * case["layers"], case["pages"], Hkv, case["page"], D)
        order = np.random.default_rng(seed).permutation(case["pages"])
        s["src"], s["dst"] = order[:case["moved"]], order[case["moved"]:2 * case["moved"]]
        return s
    if kind == "window":
        B, S = case["batch"], case["seq"]
        s.update(q=mk.normal(B, H, S, D), k=mk.normal(B, Hkv, S, D), v=mk.normal(B, Hkv, S, D))
        return s
    lens, B = _lens(case), case["batch"]
    held = lens if kind == "decode" else lens + _new_lens(case)
    s["table"], pages = _page_table(case, held, seed)
    s["lens"] = _cuda(lens)
    s["kp"], s["vp"] = (mk.normal(pages, Hkv, case["page"], D) for _ in "kv")
    if kind == "decode":
        s["q"] = mk.normal(B, H, D)
        return s
    n = case["new"]
    s["new_lens"] = _cuda(_new_lens(case))
    s["q"] = mk.normal(B, n, H, D)
    if kind == "append":
        s.update(k=mk.normal(B, n, Hkv, D), v=mk.normal(B, n, Hkv, D))
        s["cos"], s["sin"] = _tables(case)
    return s


# ---- the framework's calls -------------------------------------------------------

def _handles(s):
    """The framework's handles on the state's tensors and the buffers a program keeps, made on the first pass."""
    if "own" in s:
        return s["own"]
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-llm_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from triton_llm import gpu, kernels

    kinds = {torch.float32: np.dtype(np.float32), torch.float16: np.dtype(np.float16), torch.bfloat16: gpu.bfloat16,
             torch.int32: np.dtype(np.int32)}

    def dev(t):
        return gpu.DeviceTensor(ctypes.c_void_p(t.data_ptr()), t.shape, kinds[t.dtype], t.numel() * t.element_size(),
                                defer_free=False)

    case = s["case"]
    d = {n: dev(t) for n, t in s.items() if isinstance(t, torch.Tensor)}
    d["kernels"] = kernels
    if case["kind"] == "copy":
        d["caches"] = [dev(t) for t in s["pool"]]
        d["pairs"] = ([int(p) for p in s["src"]], [int(p) for p in s["dst"]])
    elif case["kind"] == "beam":
        shape = (case["batch"], case["select"])
        s["out"] = [torch.empty(shape, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
        d["out"] = tuple(dev(t) for t in s["out"])
    else:
        s["out"] = torch.zeros_like(s["q"])
        d["out"] = dev(s["out"])
    if case["kind"] == "decode":
        H, Hkv, D = HEADS[case["model"]]
        d["ws"] = kernels.paged_decode_workspace(case["batch"], H, Hkv, case["max_ctx"], D)
    torch.cuda.synchronize()
    s["own"] = d
    return d


def _run_own(s):
    case, d = s["case"], _handles(s)
    k = d["kernels"]
    kind = case["kind"]
    if kind == "beam":
        k.beam_select(d["logits"], d["scores"], case["select"], out=d["out"])
        return {"scores": s["out"][0], "parents": s["out"][1], "tokens": s["out"][2]}
    if kind == "copy":
        k.copy_kv_pages(d["caches"], *d["pairs"])
        return s["pool"]
    if kind == "append":
        k.paged_kv_append(d["q"], d["k"], d["v"], d["kp"], d["vp"], d["table"], d["lens"], d["cos"], d["sin"],
                          new_lens=d["new_lens"], q_out=d["out"], interleaved=case["pairs"] == "interleaved")
        return {"q": s["out"], "k_pages": s["kp"], "v_pages": s["vp"]}
    if kind == "window":
        k.window_attention(d["q"], d["k"], d["v"], case["window"], case["sinks"], out=d["out"])
        return s["out"]
    H, Hkv, D = HEADS[case["model"]]
    if kind == "decode":
        k.paged_attention_decode(d["q"], d["kp"], d["vp"], d["table"], d["lens"], H, Hkv, window=case["window"],
                                 sinks=case["sinks"], out=d["out"], workspace=d["ws"])
    else:
        k.paged_attention_prefill(d["q"], d["kp"], d["vp"], d["table"], d["lens"], H, Hkv, new_lens=d["new_lens"],
                                  window=case["window"], sinks=case["sinks"], out=d["out"])
    return s["out"]


# ---- the plain forms --------------------------------------------------------------

def _gather(pages, table):
    """(batch, KV heads, positions, head size) in 32 bits from the pages a table names."""
    x = pages[table.clamp(min=0).long()]  # (batch, pages, KV heads, page, head size)
    B, P, Hkv, ps, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, P * ps, D).float()


def _attend(q, k, v, keep):
    """q (batch, KV heads, rows, D) over k / v (batch, KV heads, keys, D); keep broadcasts over (.., rows, keys).
    A row that sees no key gives zeros."""
    s = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    s = torch.where(keep, s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m.isinf(), 0.0, m))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def _visible(pos, keys, window, sinks):
    """Whether a query at pos sees each key: none after it, and with a window its last `window` keys and the first
    `sinks`."""
    seen = keys <= pos
    return seen & ((keys > pos - window) | (keys < sinks)) if window else seen


def _rotate(x, c, s, pairs, rotary):
    """x (.., D) with c / s (.., rotary / 2): the first `rotary` features turned, the rest as they are."""
    r, rest = x[..., :rotary].float(), x[..., rotary:].float()
    if pairs == "half":
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
        r = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([r, rest], -1).to(x.dtype)


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    kind = case["kind"]
    if kind == "beam":
        B, J, V = case["batch"], case["beams"], case["vocab"]
        x = s["logits"].double()
        m = x.amax(-1, keepdim=True)
        lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
        scores = (s["scores"].double().view(B * J, 1) + (x - lse)).view(B, J * V)
        best, at = torch.sort(scores, dim=-1, descending=True, stable=True)
        best, at = best[:, :case["select"]], at[:, :case["select"]]
        return {"scores": best.float(), "parents": (at // V).int(), "tokens": (at % V).int()}
    if kind == "copy":
        src, dst = _cuda(s["src"]), _cuda(s["dst"])
        s["pool"][:, dst] = s["pool"][:, src]
        return s["pool"]
    H, Hkv, D = HEADS[case["model"]]
    G = H // Hkv
    if kind == "window":
        B, S = case["batch"], case["seq"]
        at = torch.arange(S, device="cuda")
        keep = _visible(at[:, None], at, case["window"], case["sinks"])
        out = _attend(s["q"].float().view(B, Hkv, G * S, D), s["k"].float(), s["v"].float(), keep.repeat(G, 1))
        return out.view(B, H, S, D).to(s["q"].dtype)
    table, lens = s["table"], s["lens"]
    B, ps = case["batch"], case["page"]
    if kind == "decode":
        k, v = _gather(s["kp"], table), _gather(s["vp"], table)
        keys = torch.arange(k.shape[2], device="cuda")
        keep = _visible(lens[:, None] - 1, keys, case["window"], case["sinks"])
        out = _attend(s["q"].float().view(B, Hkv, G, D), k, v, keep[:, None, None, :])
        return out.view(B, H, D).to(s["q"].dtype)
    n = case["new"]
    step = torch.arange(n, device="cuda")
    pos = lens[:, None] + step  # (batch, new)
    real = step < s["new_lens"][:, None]
    if kind == "append":
        c, sn = (t[pos.clamp(max=case["max_ctx"] - 1)][:, :, None] for t in (s["cos"], s["sin"]))
        q = torch.where(real[..., None, None], _rotate(s["q"], c, sn, case["pairs"], case["rotary"]), 0)
        k = _rotate(s["k"], c, sn, case["pairs"], case["rotary"])
        page = torch.gather(table, 1, (pos // ps).clamp(max=table.shape[1] - 1).long())[real].long()
        row = (pos % ps)[real]
        s["kp"][page, :, row] = k[real]
        s["vp"][page, :, row] = s["v"][real]
        return {"q": q, "k_pages": s["kp"], "v_pages": s["vp"]}
    k, v = _gather(s["kp"], table), _gather(s["vp"], table)
    keys = torch.arange(k.shape[2], device="cuda")
    keep = _visible(pos[..., None], keys, case["window"], case["sinks"])  # (batch, new, keys)
    q = s["q"].float().permute(0, 2, 1, 3).reshape(B, Hkv, G * n, D)
    out = _attend(q, k, v, keep[:, None].repeat(1, 1, G, 1)).view(B, H, n, D).permute(0, 2, 1, 3)
    return torch.where(real[..., None, None], out, 0.0).to(s["q"].dtype)


# ---- what a pass cannot do without -------------------------------------------------

def _seen(pos, window, sinks):
    """Keys that queries at positions pos see, in all."""
    pos = np.asarray(pos, np.int64)
    n = pos + 1
    return int((n if not window else np.minimum(n, window) + np.minimum(sinks, np.maximum(n - window, 0))).sum())


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind == "beam":
        rows = case["batch"] * case["beams"]
        return {"bytes": float(rows * case["vocab"] * e + 4 * rows + 12 * case["batch"] * case["select"]),
                "flops": 3.0 * rows * case["vocab"]}
    H, Hkv, D = HEADS[case["model"]]
    if kind == "copy":
        return {"bytes": 4.0 * case["layers"] * case["moved"] * Hkv * case["page"] * D * e, "flops": 0.0}
    B, w, k = case["batch"], case.get("window", 0), case.get("sinks", 0)
    if kind == "window":
        S = case["seq"]
        return {"bytes": float(B * S * D * e * (2 * H + 2 * Hkv)),
                "flops": 4.0 * D * H * B * _seen(np.arange(S), w, k)}
    lens = _lens(case).astype(np.int64)
    if kind == "decode":
        n = _seen(lens - 1, w, k)
        return {"bytes": float((2 * Hkv * n + 2 * B * H) * D * e), "flops": 4.0 * D * H * n}
    new = _new_lens(case).astype(np.int64)
    if kind == "append":
        n = int(new.sum())
        at = np.unique(np.concatenate([np.arange(a, a + m) for a, m in zip(lens, new)])).size
        return {"bytes": float(n * 2 * (H + 2 * Hkv) * D * e + at * case["rotary"] * 4),
                "flops": 3.0 * n * (H + Hkv) * case["rotary"]}
    pairs = sum(_seen(np.arange(a, a + m), w, k) for a, m in zip(lens, new))
    span = sum(int(m + min(a, w - 1 + k) if w else a + m) for a, m in zip(lens, new))  # keys any query sees
    return {"bytes": float((2 * Hkv * span + 2 * H * int(new.sum())) * D * e), "flops": 4.0 * D * H * pairs}


# ---- the definitions in 64 bits ------------------------------------------------------

def _softmax64(q, k, v, first, window, sinks):
    """Rows of q (n, D) at positions first, first + 1, ... over k / v (keys, D)."""
    out = torch.zeros_like(q)
    for r in range(0, q.shape[0], 2048):
        rows = q[r:r + 2048]
        pos = first + r + torch.arange(rows.shape[0], device=q.device)[:, None]
        j = torch.arange(k.shape[0], device=q.device)[None]
        hidden = j > pos
        if window:
            hidden |= (j <= pos - window) & (j >= sinks)
        s = (rows @ k.T) * k.shape[1] ** -0.5
        out[r:r + 2048] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "copy":
        pool = s["pool"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pool[:, b] = pool[:, a]
        return pool
    if kind == "beam":
        B, J = case["batch"], case["beams"]
        logp = torch.log_softmax(s["logits"].double(), -1).view(B, J, -1) + s["scores"].double()[..., None]
        return {"scores": torch.topk(logp.reshape(B, -1), case["select"]).values, "parents": None, "tokens": None}
    H, Hkv, D = HEADS[case["model"]]
    G = H // Hkv
    w, sinks = case.get("window", 0), case.get("sinks", 0)
    if kind == "window":
        q, k, v = (s[n].double() for n in "qkv")
        return torch.stack([torch.stack([_softmax64(q[b, h], k[b, h // G], v[b, h // G], 0, w, sinks)
                                         for h in range(H)]) for b in range(case["batch"])])
    table, lens, ps = s["table"].cpu().numpy(), _lens(case), case["page"]

    def rows(pages, b, n):
        ids = torch.from_numpy(table[b, :-(-n // ps)].astype(np.int64)).cuda()
        return torch.cat(list(pages[ids].double()), 1)[:, :n]  # (KV heads, n, D)

    if kind == "decode":
        out = torch.empty(case["batch"], H, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(int(x) for x in lens):
            k, v = rows(s["kp"], b, n), rows(s["vp"], b, n)
            for h in range(H):
                out[b, h] = _softmax64(s["q"][b, h:h + 1].double(), k[h // G], v[h // G], n - 1, w, sinks)[0]
        return out
    new = _new_lens(case)
    if kind == "chunk":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, (n, m) in enumerate(zip(lens.tolist(), new.tolist())):
            k, v = rows(s["kp"], b, n + m), rows(s["vp"], b, n + m)
            for h in range(H):
                out[b, :m, h] = _softmax64(s["q"][b, :m, h].double(), k[h // G], v[h // G], n, w, sinks)
        return out
    r = case["rotary"]
    out = {"q": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), "k_pages": s["kp"].double(),
           "v_pages": s["vp"].double()}

    def turned(x, n):
        """x (tokens, heads, D) of positions n, n + 1, ...: each pair as a complex number times e^(i angle)."""
        x = x.double()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[n:n + x.shape[0], None]
        first = torch.arange(r // 2, device="cuda") * (1 if case["pairs"] == "half" else 2)
        second = first + (r // 2 if case["pairs"] == "half" else 1)
        z = torch.complex(x[..., first], x[..., second]) * turn
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    for b, (n, m) in enumerate(zip(lens.tolist(), new.tolist())):
        out["q"][b, :m] = turned(s["q"][b, :m], n)
        at = np.arange(n, n + m)
        page, row = (torch.from_numpy(x.astype(np.int64)).cuda() for x in (table[b, at // ps], at % ps))
        out["k_pages"][page, :, row] = turned(s["k"][b, :m], n)
        out["v_pages"][page, :, row] = s["v"][b, :m].double()
    return out
