"""Serving from a paged cache whose tables the GPU keeps, and whose sequences share long prefixes, as cases that can be timed.

The operators, each in a plain form (elementary torch operations in 32 bits,
whole numbers in 64) and, where ``own`` is true, through the framework's entry points:

* ``pages``  -- ``release_kv_pages`` and ``assign_kv_pages``: ended sequences give their pages back, and the step's new
                tokens get theirs: table entries, a slot and a position for every row of the packed batch;
* ``slots``  -- ``paged_kv_append_slots``: rotary positions on packed rows of q and k, k and v written to the rows' slots;
* ``packed`` -- ``paged_attention_packed``: attention of packed rows, one token or many of each sequence, over its pages;
* ``shared`` -- ``plan_shared_attention`` and ``paged_attention_shared``: a token of every sequence, where groups of sequences
                begin with the same pages: one plan a step, then each layer's attention.

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
        # One token more for each of a few sequences, one of them done: launch and latency.
        {"name": "pages-step-8", "kind": "pages", "batch": 8, "page": 16, "max_ctx": 2048, "lo": 1, "hi": 1000,
         "new": 1, "ended": 1, "spare": 5, "lens": 1},
        # A busy server's step: a token of each of 500 sequences, a dozen long ones done.
        {"name": "pages-step-512", "kind": "pages", "batch": 512, "page": 16, "max_ctx": 16384, "lo": 100, "hi": 16000,
         "new": 1, "ended": 12, "spare": 100, "lens": 2},
        # Prompts come in while others end, and the pool is too small for all of them.
        {"name": "pages-prompts-128", "kind": "pages", "batch": 128, "page": 32, "max_ctx": 8192, "lo": 0, "hi": 4000,
         "new": 1500, "ended": 40, "spare": -77, "lens": 3},
        # The cache write of a step of one token a sequence: launch and latency.
        {"name": "slots-step-bf16", "kind": "slots", "model": "llama3.2-3b", "dtype": "bfloat16", "batch": 64,
         "page": 16, "max_ctx": 4096, "lo": 1, "hi": 4000, "lens": 4, "ones": 64, "new": 1, "rotary": 128,
         "pairs": "half"},
        # Tokens of running sequences beside the prompts of new ones; interleaved pairs over half of each head.
        {"name": "slots-mixed-fp16", "kind": "slots", "model": "smollm2-360m", "dtype": "float16", "batch": 60,
         "page": 32, "max_ctx": 4096, "lo": 0, "hi": 2000, "lens": 5, "ones": 48, "new": 999, "rotary": 32,
         "pairs": "interleaved"},
        # Prompts alone, in the reference's own type.
        {"name": "slots-prompts-fp32", "kind": "slots", "model": "smollm2-135m", "dtype": "float32", "batch": 16,
         "page": 16, "max_ctx": 2048, "lo": 0, "hi": 3, "lens": 6, "ones": 0, "new": 2000, "rotary": 64,
         "pairs": "half"},
        # Running sequences beside two pieces of prompts.
        {"name": "packed-mixed-bf16", "kind": "packed", "model": "llama3.2-3b", "dtype": "bfloat16", "batch": 32,
         "page": 16, "max_ctx": 4096, "lo": 100, "hi": 3500, "lens": 7, "ones": 30, "new": 500, "window": 0, "sinks": 0},
        # Prompts of unequal lengths, packed one behind the other.
        {"name": "packed-prompts-fp16", "kind": "packed", "model": "smollm2-360m", "dtype": "float16", "batch": 12,
         "page": 32, "max_ctx": 2048, "lo": 0, "hi": 0, "lens": 8, "ones": 0, "new": 1400, "window": 0, "sinks": 0},
        # Four answers to one short prompt, in the reference's own type: latency.
        {"name": "shared-4-fp32", "kind": "shared", "model": "smollm2-135m", "dtype": "float32", "batch": 4,
         "groups": 1, "page": 16, "prefix": 496, "lo": 1, "hi": 40, "lens": 9, "layers": 1},
        # Two beam searches of eight beams.
        {"name": "shared-beams-fp16", "kind": "shared", "model": "smollm2-360m", "dtype": "float16", "batch": 16,
         "groups": 2, "page": 16, "prefix": 2000, "lo": 30, "hi": 60, "lens": 10, "layers": 4},
        # A batch of users behind one long document.
        {"name": "shared-document-bf16", "kind": "shared", "model": "llama3.2-3b", "dtype": "bfloat16", "batch": 64,
         "groups": 1, "page": 64, "prefix": 8192, "lo": 1, "hi": 500, "lens": 11, "layers": 2},
        # A busy server with eight system prompts.
        {"name": "shared-groups-bf16", "kind": "shared", "model": "llama3.2-3b", "dtype": "bfloat16", "batch": 256,
         "groups": 8, "page": 64, "prefix": 4096, "lo": 1, "hi": 1000, "lens": 12, "layers": 2},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["pages", "slots", "packed", "shared", "shared"])
    page = rng.choice([16, 16, 32, 64, 128])
    lens = rng.randint(0, 1 << 20)
    if kind == "pages":
        batch = _log(rng, 1, 700)
        new = rng.choice([1, 1, _log(rng, 2, max(2, min(3000, 90000 // batch)))])
        ctx = -(-(new + _log(rng, 64, 12000)) // page) * page
        return {"kind": kind, "batch": batch, "page": page, "max_ctx": ctx, "lo": 0, "hi": rng.randint(1, ctx - new),
                "new": new, "ended": rng.randint(0, batch // 2), "spare": rng.choice([0, 3, 200, -1, -9]), "lens": lens}
    model = rng.choice(sorted(HEADS))
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    D = HEADS[model][2]
    case = {"kind": kind, "model": model, "dtype": dtype}
    if kind in ("slots", "packed"):
        most = 12000 if kind == "slots" else 600 if dtype == "float32" else 1200
        new = rng.choice([1, _log(rng, 2, min(most, 1500))])
        batch = _log(rng, 1, 96)
        ones = batch if new == 1 else max(0, batch - rng.randint(1, max(1, most // new)))
        ctx = -(-(new + _log(rng, 16, 2500)) // page) * page
        case.update(batch=batch, page=page, max_ctx=ctx, lo=0, hi=ctx - new, lens=lens, ones=ones, new=new)
        if kind == "slots":
            return {**case, "rotary": rng.choice([D, D, D // 2, D // 4]), "pairs": rng.choice(["half", "interleaved"])}
        window = rng.choice([0, 0, _log(rng, 16, 2000)])
        return {**case, "window": window, "sinks": rng.choice([0, 4, 37]) if window else 0}
    batch = _log(rng, 2, 200)
    prefix = max(1, _log(rng, 100, min(9000, 600000 // batch)) // page) * page
    hi = _log(rng, 1, max(1, min(1500, 150000 // batch)))
    groups = rng.randint(1, max(1, min(8, batch // 3, 24000 // prefix)))
    return {**case, "batch": batch, "groups": groups, "page": page, "prefix": prefix, "lo": rng.randint(1, hi), "hi": hi,
            "lens": lens, "layers": rng.choice([1, 2, 3])}


# ---- lengths: from the case alone ----------------------------------------------------

def _lens(case):
    """Tokens that are in the cache of each sequence before the call."""
    return np.random.default_rng(case["lens"]).integers(case["lo"], case["hi"], size=case["batch"],
                                                        endpoint=True).astype(np.int64)


def _new_lens(case):
    """New tokens of each sequence: one of the first `ones`, of the others part of `new`, one of them all."""
    rng = np.random.default_rng(case["lens"] + 1)
    n = rng.integers(1, case["new"], size=case["batch"], endpoint=True)
    n[:case["ones"]] = 1
    if case["ones"] < case["batch"]:
        n[case["ones"]] = case["new"]
    return rng.permutation(n)


def _turn(case):
    """(lens, new, ended, keep) of a step: `ended` sequences rest, their first `keep` pages being others' too."""
    rng = np.random.default_rng(case["lens"] + 1)
    lens, B = _lens(case), case["batch"]
    ended = np.zeros(B, np.int64)
    ended[rng.permutation(B)[:case["ended"]]] = 1
    new = np.where(ended == 1, 0, rng.integers(1, case["new"], size=B, endpoint=True))
    keep = np.where(ended == 1, -(-lens // case["page"]) // 4, 0)
    return lens, new, ended, keep


def _pages(n, page):
    return -(-n // page)


def _groups(case):
    """(members, starts, prefix of each group, tokens of each sequence with the new one): groups of about equal size, members
    in any order, the first group's prefix the whole one."""
    rng = np.random.default_rng(case["lens"] + 1)
    B, G, page = case["batch"], case["groups"], case["page"]
    starts = np.array([i * B // G for i in range(G + 1)])
    members = rng.permutation(B)
    most = case["prefix"] // page
    prefix = rng.integers(-(-most // 2), most, size=G, endpoint=True) * page
    prefix[0] = most * page
    lens = _lens(case)
    lens[members] += np.repeat(prefix, np.diff(starts))
    return members, starts, prefix, lens


# ---- what a program has in hand ------------------------------------------------

class _Make:
    """Seeded inputs on the GPU."""

    def __init__(self, seed, dtype):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))
        self.dtype = dtype

    def normal(self, *shape):
        if math.prod(shape) > 1 << 28:  # large pools: made in their own type, with no 32-bit copy
            return torch.empty(shape, dtype=TORCH[self.dtype], device="cuda").normal_(generator=self.g)
        return torch.empty(shape, device="cuda").normal_(generator=self.g).to(TORCH[self.dtype])


def _int32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _angles(case):
    """cos / sin (max_ctx, rotary / 2) in 32 bits, angles in 64."""
    r = case["rotary"]
    freq = THETA[case["model"]] ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    angle = torch.arange(case["max_ctx"], dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _shuffled(case, held, rng, spare=3):
    """(table (batch, max_ctx / page), pages in the pool): every sequence's pages lie anywhere in the pool."""
    need = _pages(held, case["page"])
    total = int(need.sum()) + spare
    table = np.full((case["batch"], case["max_ctx"] // case["page"]), -1)
    table[np.arange(table.shape[1]) < need[:, None]] = rng.permutation(total)[:int(need.sum())]
    return table, total


def prepare(case, seed):
    kind, rng = case["kind"], np.random.default_rng(seed)
    s = {"case": case}
    if kind == "pages":
        lens, new, ended, keep = _turn(case)
        ps, held = case["page"], _pages(lens, case["page"])
        need = _pages(lens + new, ps) - held
        given = int(((held - keep) * ended).sum())
        free = max(0, int(need.sum()) - given + case["spare"])
        table, total = _shuffled(case, lens, rng, free)
        order = rng.permutation(total)
        rest = order[~np.isin(order, table)]
        stack = np.full(total, -1)  # what the free list holds behind its last entry is nobody's
        stack[:rest.size] = rest
        s.update(table=_int32(table), lens=_int32(lens), new=_int32(new), ended=_int32(ended), keep=_int32(keep),
                 free=_int32(stack), counts=_int32([free, 0]))
        s["tokens"] = -(-int(new.sum()) // 64) * 64
        return s
    mk = _Make(seed, case["dtype"])
    H, Hkv, D = HEADS[case["model"]]
    if kind == "shared":
        members, starts, prefix, lens = _groups(case)
        ps = case["page"]
        n = _pages(lens, ps)
        first = np.empty(case["batch"], np.int64)  # pages of the prefix
        first[members] = np.repeat(prefix // ps, np.diff(starts))
        total = int((n - first).sum() + (prefix // ps).sum()) + 3
        order = iter(np.split(rng.permutation(total), np.cumsum(np.concatenate([prefix // ps, n - first]))))
        shared = [next(order) for _ in prefix]
        table = np.full((case["batch"], int(n.max()) + 1), -1)
        for g, pages in enumerate(shared):
            table[members[starts[g]:starts[g + 1]], :pages.size] = pages
        for b in range(case["batch"]):
            table[b, first[b]:n[b]] = next(order)
        s.update(table=_int32(table), lens=_int32(lens), members=_int32(members), starts=_int32(starts),
                 prefix=_int32(prefix))
        s["kp"], s["vp"] = ([mk.normal(total, Hkv, ps, D) for _ in range(case["layers"])] for _ in "kv")
        s["q"] = [mk.normal(case["batch"], H, D) for _ in range(case["layers"])]
        return s
    lens, new = _lens(case), _new_lens(case)
    starts = np.concatenate([[0], np.cumsum(new)])
    rows = int(starts[-1])
    table, pages = _shuffled(case, lens + new, rng)
    s.update(table=_int32(table), lens=_int32(lens), starts=_int32(starts))
    s["kp"], s["vp"] = (mk.normal(pages, Hkv, case["page"], D) for _ in "kv")
    s["q"] = mk.normal(rows, H, D)
    if kind == "slots":
        seq = np.repeat(np.arange(case["batch"]), new)
        pos = lens[seq] + np.arange(rows) - starts[seq]
        s.update(k=mk.normal(rows, Hkv, D), v=mk.normal(rows, Hkv, D), positions=_int32(pos),
                 slots=_int32(table[seq, pos // case["page"]] * case["page"] + pos % case["page"]))
        s["cos"], s["sin"] = _angles(case)
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
        if isinstance(t, (list, tuple)):
            return [dev(x) for x in t]
        return gpu.DeviceTensor(ctypes.c_void_p(t.data_ptr()), t.shape, kinds[t.dtype], t.numel() * t.element_size(),
                                defer_free=False)

    case, made = s["case"], {}
    if case["kind"] == "pages":
        B, T = case["batch"], s["tokens"]
        made.update({n: torch.empty(size, dtype=torch.int32, device="cuda") for n, size in (
            ("lens_left", B), ("freed", 2), ("slots", T), ("positions", T), ("starts", B + 1), ("ends", B), ("left", 2))})
    else:
        made["out"] = [torch.zeros_like(q) for q in s["q"]] if case["kind"] == "shared" else torch.zeros_like(s["q"])
    d = {n: dev(t) for n, t in (s | made).items() if isinstance(t, (torch.Tensor, list))}
    d["kernels"], d["plan"] = kernels, None
    s["made"] = made
    torch.cuda.synchronize()
    s["own"] = d
    return d


def _run_own(s):
    case, d = s["case"], _handles(s)
    k, made = d["kernels"], s["made"]
    kind = case["kind"]
    if kind == "pages":
        k.release_kv_pages(d["table"], d["lens"], d["ended"], d["free"], d["counts"], case["page"], keep=d["keep"],
                           lens_out=d["lens_left"], counts_out=d["freed"])
        k.assign_kv_pages(d["lens_left"], d["new"], d["table"], d["free"], d["freed"], case["page"], s["tokens"],
                          out=(d["slots"], d["positions"], d["starts"], d["ends"]), counts_out=d["left"])
        return {"table": s["table"], "free": s["free"], **{n: made[n] for n in (
            "lens_left", "freed", "slots", "positions", "starts", "ends", "left")}}
    if kind == "slots":
        k.paged_kv_append_slots(d["q"], d["k"], d["v"], d["kp"], d["vp"], d["slots"], d["positions"], d["cos"], d["sin"],
                                q_out=d["out"], interleaved=case["pairs"] == "interleaved")
        return {"q": made["out"], "k_pages": s["kp"], "v_pages": s["vp"]}
    H, Hkv, D = HEADS[case["model"]]
    if kind == "packed":
        k.paged_attention_packed(d["q"], d["kp"], d["vp"], d["table"], d["lens"], d["starts"], H, Hkv, case["new"],
                                 window=case["window"], sinks=case["sinks"], out=d["out"])
        return made["out"]
    d["plan"] = k.plan_shared_attention(d["table"], d["lens"], d["members"], d["starts"], d["prefix"], H, Hkv, D, case["page"],
                                        d["q"][0].dtype, plan=d["plan"])
    for q, kp, vp, out in zip(d["q"], d["kp"], d["vp"], d["out"]):
        k.paged_attention_shared(q, kp, vp, d["table"], d["plan"], H, Hkv, out=out)
    return made["out"]


# ---- the plain forms --------------------------------------------------------------

def _plain_pages(s):
    """The ended sequences' pages behind the free list, by sequence and column; then pages from its end for the new tokens,
    sequence by sequence as long as there are enough."""
    case, ps = s["case"], s["case"]["page"]
    table, free = s["table"].long(), s["free"].long()
    lens, new, ended, keep, count = (s[n].long() for n in ("lens", "new", "ended", "keep", "counts"))
    n, width, T = free.numel(), table.shape[1], s["tokens"]
    col = torch.arange(width, device="cuda")
    held = (lens + ps - 1) // ps
    back = (ended[:, None] != 0) & (col >= keep[:, None]) & (col < held[:, None]) & (table >= 0) & (table < n)
    at = torch.cumsum(back.flatten().long(), 0).view_as(back) - 1 + count[0]
    fits = back & (at < n)
    free = torch.cat([free, free[:1]]).scatter(0, torch.where(fits, at, n).flatten(), table.flatten())[:n]
    freed = torch.stack([count[0] + fits.sum(), back.sum() - fits.sum()])
    lens = torch.where(ended != 0, 0, lens)

    new = new.clamp(min=0)
    ends = torch.cumsum(new, 0)
    starts = torch.cat([ends.new_zeros(1), ends])
    held = (lens + ps - 1) // ps
    fine = (lens >= 0) & (lens + new <= width * ps) & (ends <= T)
    need = torch.where(fine, (lens + new + ps - 1) // ps - held, 0)
    upto = torch.cumsum(need, 0)
    granted = fine & ((need == 0) | (upto <= freed[0]))
    left = torch.stack([freed[0] - torch.where(granted, need, 0).sum(), (~granted & (new > 0)).sum()])
    t = torch.arange(T, device="cuda")
    b = (t[:, None] >= ends).sum(1)
    there = b < case["batch"]
    b = b.clamp(max=case["batch"] - 1)
    pos = lens[b] + t - starts[b]
    there &= granted[b]
    c = (pos // ps).clamp(max=width - 1)
    i = upto[b] - need[b] + c - held[b]  # which of the pages from the free list's end on
    fresh = there & (c >= held[b])
    page = torch.where(fresh, free[(freed[0] - 1 - i).clamp(0, n - 1)], table[b, c])
    table = torch.cat([table.flatten(), table.flatten()[:1]])
    table = table.scatter(0, torch.where(fresh & (pos % ps == 0), b * width + c, table.numel() - 1), page)[:-1]
    out = {"table": table.view_as(s["table"]), "free": free, "lens_left": lens, "freed": freed,
           "slots": torch.where(there, page * ps + pos % ps, -1), "positions": torch.where(there, pos, -1),
           "starts": starts.clamp(max=T), "ends": torch.where(granted, lens + new, lens), "left": left}
    return {k: v.int() for k, v in out.items()}


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
    if kind == "pages":
        return _plain_pages(s)
    H, Hkv, D = HEADS[case["model"]]
    G, B, ps, table, lens = H // Hkv, case["batch"], case["page"], s["table"], s["lens"]
    if kind == "slots":
        pos = s["positions"].long()
        c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
        page, row = s["slots"].long() // ps, s["slots"].long() % ps
        s["kp"][page, :, row] = _rotate(s["k"], c, sn, case["pairs"], case["rotary"])
        s["vp"][page, :, row] = s["v"]
        return {"q": _rotate(s["q"], c, sn, case["pairs"], case["rotary"]), "k_pages": s["kp"], "v_pages": s["vp"]}
    if kind == "shared":
        keep = torch.arange(table.shape[1] * ps, device="cuda") < lens[:, None]
        return [_attend(q.float().view(B, Hkv, G, D), _gather(kp, table), _gather(vp, table),
                        keep[:, None, None, :]).view(B, H, D).to(q.dtype) for q, kp, vp in zip(s["q"], s["kp"], s["vp"])]
    # packed rows: padded to the longest sequence's, and back
    starts, n = s["starts"].long(), case["new"]
    rows = s["q"].shape[0]
    at = starts[:-1, None] + torch.arange(n, device="cuda")  # (batch, new)
    q = s["q"][at.clamp(max=rows - 1)].float().permute(0, 2, 1, 3).reshape(B, Hkv, G * n, D)
    k, v = _gather(s["kp"], table), _gather(s["vp"], table)
    keys = torch.arange(k.shape[2], device="cuda")
    pos = (lens[:, None] + torch.arange(n, device="cuda"))[..., None]
    keep = keys <= pos
    if case["window"]:
        keep &= (keys > pos - case["window"]) | (keys < case["sinks"])
    out = _attend(q, k, v, keep[:, None].repeat(1, 1, G, 1)).view(B, H, n, D).transpose(1, 2).to(s["q"].dtype)
    t = torch.arange(rows, device="cuda")
    b = (t[:, None] >= starts[1:]).sum(1)
    return out[b, t - starts[b]]


# ---- what a pass cannot do without -------------------------------------------------

def _seen(pos, window, sinks):
    """Keys that queries at positions pos see, in all."""
    n = np.asarray(pos, np.int64) + 1
    return int((n if not window else np.minimum(n, window) + np.minimum(sinks, np.maximum(n - window, 0))).sum())


def work(case):
    kind = case["kind"]
    if kind == "pages":
        lens, new, ended, keep = _turn(case)
        held = _pages(lens, case["page"])
        back = int(((held - keep) * ended).sum())
        fresh = int(((_pages(lens + new, case["page"]) - held) * (1 - ended)).sum())
        tokens = -(-int(new.sum()) // 64) * 64
        return {"bytes": 8.0 * back + 8.0 * fresh + 8.0 * tokens + 28.0 * case["batch"], "flops": 4.0 * tokens}
    H, Hkv, D = HEADS[case["model"]]
    e, B = SIZE[case["dtype"]], case["batch"]
    if kind == "shared":
        members, starts, prefix, lens = _groups(case)
        first = np.empty(B, np.int64)
        first[members] = np.repeat(prefix, np.diff(starts))
        keys = int((lens - first).sum() + prefix.sum())  # a group's prefix is read once
        return {"bytes": float((2 * Hkv * keys + 2 * B * H) * D * e * case["layers"]),
                "flops": 4.0 * D * H * int(lens.sum()) * case["layers"]}
    lens, new = _lens(case), _new_lens(case)
    n = int(new.sum())
    if kind == "slots":
        at = np.unique(np.concatenate([np.arange(a, a + m) for a, m in zip(lens, new)])).size
        return {"bytes": float(n * 2 * (H + 2 * Hkv) * D * e + 8 * n + at * case["rotary"] * 4),
                "flops": 3.0 * n * (H + Hkv) * case["rotary"]}
    w, k = case["window"], case["sinks"]
    pairs = sum(_seen(np.arange(a, a + m), w, k) for a, m in zip(lens, new))
    span = sum(int(m + min(a, w - 1 + k) if w else a + m) for a, m in zip(lens, new))  # keys any query sees
    return {"bytes": float((2 * Hkv * span + 2 * H * n) * D * e), "flops": 4.0 * D * H * pairs}


# ---- the definitions in 64 bits ------------------------------------------------------

def exact(case, seed):
    kind = case["kind"]
    if kind == "pages":
        return None  # whole numbers throughout
    s = prepare(case, seed)
    H, Hkv, D = HEADS[case["model"]]
    G, ps, table = H // Hkv, case["page"], s["table"].cpu().numpy()

    def rows(pages, b, n):
        ids = torch.from_numpy(table[b, :-(-n // ps)].astype(np.int64)).cuda()
        return torch.cat(list(pages[ids].double()), 1)[:, :n]  # (KV heads, n, D)

    if kind == "shared":
        out = []
        for q, kp, vp in zip(s["q"], s["kp"], s["vp"]):
            o = torch.empty(q.shape, dtype=torch.float64, device="cuda")
            for b, n in enumerate(s["lens"].tolist()):
                x = (q[b].double().view(Hkv, G, 1, D) * rows(kp, b, n)[:, None]).sum(-1) * D ** -0.5
                o[b] = (torch.softmax(x, -1)[..., None] * rows(vp, b, n)[:, None]).sum(2).view(H, D)
            out.append(o)
        return out
    lens, new = _lens(case), _new_lens(case)
    ends = np.cumsum(new)
    if kind == "packed":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, (n, m, e) in enumerate(zip(lens.tolist(), new.tolist(), ends.tolist())):
            k, v = rows(s["kp"], b, n + m), rows(s["vp"], b, n + m)
            j = torch.arange(n + m, device="cuda")
            away = torch.arange(n, n + m, device="cuda")[:, None] - j
            hidden = away < 0
            if case["window"]:
                hidden |= (away >= case["window"]) & (j >= case["sinks"])
            for h in range(H):
                x = (s["q"][e - m:e, h].double() @ k[h // G].T) * D ** -0.5
                out[e - m:e, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h // G]
        return out
    r = case["rotary"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    first = torch.arange(r // 2, device="cuda") * (1 if case["pairs"] == "half" else 2)
    second = first + (r // 2 if case["pairs"] == "half" else 1)

    def turned(x, n):
        """x (tokens, heads, D) of positions n, n + 1, ...: each pair as a complex number times e^(i angle)."""
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * turn[n:n + x.shape[0], None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = {"q": torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), "k_pages": s["kp"].double(),
           "v_pages": s["vp"].double()}
    for b, (n, m, e) in enumerate(zip(lens.tolist(), new.tolist(), ends.tolist())):
        out["q"][e - m:e] = turned(s["q"][e - m:e], n)
        at = np.arange(n, n + m)
        page, row = (torch.from_numpy(x.astype(np.int64)).cuda() for x in (table[b, at // ps], at % ps))
        out["k_pages"][page, :, row] = turned(s["k"][e - m:e], n)
        out["v_pages"][page, :, row] = s["v"][e - m:e].double()
    return out
