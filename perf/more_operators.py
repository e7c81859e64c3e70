"""The calls around a paged cache that is kept for long, measured: attention with a
window and first tokens that stay visible, choosing the next tokens of beams,
forking the beams' sequences page by page, compacting and copying pages.

Together they are a step of a beam search over the text decoder whose cache does not
grow without end: qa_attention_paged_window reads the pages, qa_beam_select gives each
new beam its parent and token, qa_pages_fork gives it the parent's pages (shared where
they are full, copied where it goes on writing), takes back those that no window
reaches, and finds new ones.  qa_pages_compact moves a pool's used pages to its
front; qa_pages_copy moves pages to another pool and back.

Kinds of case:
  window   causal attention of packed rows over the pages, the last `window` keys and the first `sinks`
  select   the best continuations over beams and vocabulary
  fork     tables, references and copied pages of the next step's sequences
  compact  used pages to the front of the pool, tables renamed
  copy     pairs of pages from one pool to another
"""
from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import torch

own = False

TYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # One step of one stream five minutes in, its window the last 80 s or so: latency.
        {"name": "window_decode_1", "kind": "window", "dtype": "f16", "cache": "f16", "page": 16, "nq": 16, "nkv": 8, "hd": 128,
         "seqs": 1, "rows": 1, "long": 1, "past": 4352, "window": 1024, "sinks": 4, "freed": True},
        # One step of 48 streams of up to 32768 tokens, four q heads to a kv head; the pages behind the windows were given back.
        {"name": "window_decode_48_e4m3", "kind": "window", "dtype": "bf16", "cache": "e4m3", "page": 32, "nq": 32, "nkv": 8, "hd": 128,
         "seqs": 48, "rows": 1, "long": 1, "past": 32768, "window": 4096, "sinks": 64, "freed": True},
        # The next part of a long prompt, all of its past still in the cache.
        {"name": "window_chunk_1201", "kind": "window", "dtype": "f16", "cache": "f16", "page": 64, "nq": 16, "nkv": 8, "hd": 128,
         "seqs": 1, "rows": 1201, "long": 1201, "past": 4334, "window": 2048, "sinks": 16, "freed": False},
        # Twenty streams at one token each and one with 501 new rows; heads of 64, three to a kv head.
        {"name": "window_mixed_21", "kind": "window", "dtype": "bf16", "cache": "e4m3", "page": 16, "nq": 12, "nkv": 4, "hd": 64,
         "seqs": 21, "rows": 1, "long": 501, "past": 3100, "window": 700, "sinks": 5, "freed": True},
        # One clip, four beams: latency.
        {"name": "select_1x4", "kind": "select", "dtype": "bf16", "groups": 1, "beams": 4, "width": 8, "vocab": 151936, "done": False},
        # 24 clips of eight beams, some of which have ended.
        {"name": "select_24x8", "kind": "select", "dtype": "f16", "groups": 24, "beams": 8, "width": 8, "vocab": 151936, "done": True},
        # The step of one clip's four beams behind a 15 s clip's prompt, every layer's cache.
        {"name": "fork_1x4", "kind": "fork", "cache": "f16", "page": 16, "nkv": 8, "hd": 128, "layers": 28,
         "groups": 1, "beams": 4, "past": 323, "extra": 40, "window": 0, "sinks": 0},
        # The step of 24 clips of eight beams, e4m3 pages and their scales, with a window.
        {"name": "fork_24x8_e4m3", "kind": "fork", "cache": "e4m3", "page": 32, "nkv": 8, "hd": 128, "layers": 28,
         "groups": 24, "beams": 8, "past": 771, "extra": 60, "window": 500, "sinks": 4},
        # A small pool in which a few pages lie behind others' gaps.
        {"name": "compact_90", "kind": "compact", "cache": "e4m3", "page": 16, "nkv": 8, "hd": 128, "layers": 28, "pages": 90, "used": 0.8, "seqs": 3},
        # A pool of which half has been given back.
        {"name": "compact_4096", "kind": "compact", "cache": "f16", "page": 32, "nkv": 8, "hd": 128, "layers": 4, "pages": 4096, "used": 0.5, "seqs": 40},
        # A 15 s clip's sequence back from a pool it was set aside in.
        {"name": "copy_21", "kind": "copy", "cache": "f16", "page": 16, "nkv": 8, "hd": 128, "layers": 28, "pages": 64, "pairs": 21},
        # A pool's pages into a larger one's.
        {"name": "copy_1900", "kind": "copy", "cache": "e4m3", "page": 64, "nkv": 8, "hd": 128, "layers": 4, "pages": 2048, "pairs": 1900},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("window", "window", "window", "select", "select", "fork", "fork", "compact", "copy"))
    c = {"kind": kind}
    if kind == "select":
        beams = rng.choice((1, 2, 3, 4, 5, 8, 12, 16))
        vocab = rng.choice((5000, 151936, _log(rng, 30, 151936)))
        return {**c, "dtype": rng.choice(("f16", "bf16", "f32")), "groups": _log(rng, 1, min(64, max(1, 96 // beams))), "beams": beams,
                "width": min(rng.choice((beams, beams, 2 * beams)), 32), "vocab": vocab, "done": rng.random() < 0.5}
    if kind == "window":
        t = rng.choice(("f16", "bf16"))
        nkv = rng.choice((1, 2, 4, 8))
        c.update(dtype=t, cache=rng.choice((t, "e4m3")), page=rng.choice((16, 32, 64)), nq=nkv * rng.choice((1, 2, 2, 3, 4)), nkv=nkv,
                 hd=rng.choice((64, 128, 128)), sinks=rng.choice((0, 1, 4, _log(rng, 1, 300))), window=_log(rng, 16, 4096), freed=rng.random() < 0.7)
        seqs = _log(rng, 1, 48)
        shape = rng.choice(("step", "step", "part", "mixed"))
        if shape == "step":
            return {**c, "seqs": seqs, "rows": 1, "long": 1, "past": _log(rng, 1, 32768)}
        c["nkv"], c["nq"] = min(nkv, 4), min(nkv, 4) * (c["nq"] // nkv)
        rows = _log(rng, 2, 1200)
        if shape == "part":  # parts of prompts, of about the same length
            return {**c, "seqs": max(1, min(seqs, 1200 // rows)), "rows": rows, "long": rows, "past": _log(rng, 1, 6000)}
        return {**c, "seqs": min(seqs, 24), "rows": 1, "long": min(rows, 700), "past": _log(rng, 1, 6000)}
    c.update(cache=rng.choice(("f16", "e4m3")), page=rng.choice((16, 32, 64)), nkv=rng.choice((1, 2, 4, 8)), hd=rng.choice((64, 128)),
             layers=rng.choice((1, 3, 4, 28)))
    each = c["page"] * c["nkv"] * c["hd"] * 4 * c["layers"]  # bytes of a page over all layers, at most
    if kind == "fork":
        c.update(groups=_log(rng, 1, 24), beams=rng.choice((1, 2, 4, 5, 8)), extra=_log(rng, 1, 100), window=rng.choice((0, 0, _log(rng, 20, 900))),
                 sinks=rng.choice((0, 4, 40)))
        seqs = c["groups"] * c["beams"]
        left = (5 << 29) // each - seqs * (c["extra"] // c["page"] + 3)
        return {**c, "past": _log(rng, 1, max(2, min(4352, left * c["page"] // c["groups"])))}
    pages = _log(rng, 2, max(2, min(6000, (1 << 31) // each)))
    if kind == "compact":
        return {**c, "pages": pages, "used": rng.choice((0.2, 0.5, 0.8, 0.97)), "seqs": _log(rng, 1, min(pages, 40))}
    return {**c, "pages": pages, "pairs": _log(rng, 1, max(1, pages * 9 // 10))}


# ---- inputs ---------------------------------------------------------------

def _spread(case):
    """Rows and keys of each sequence of a window case: the last has `long` rows, the others up to `rows`; pasts are spread up to `past`."""
    r = random.Random(case["past"] * 64 + case["seqs"])
    n = [case["rows"] if case["rows"] == 1 else r.randint((case["rows"] + 1) // 2, case["rows"]) for _ in range(case["seqs"] - 1)] + [case["long"]]
    past = [case["past"]] + [r.randint(case["past"] // 2, case["past"]) for _ in range(case["seqs"] - 1)]
    return n, [p + k for p, k in zip(past, n)]


def _reach(case, rows, keys):
    """The first key of a sequence's first row's window."""
    return max(0, keys - rows - case["window"] + 1)


def _cache(case, total, g, spread=False):
    """K and V pages of `total` pages of every layer, and their scales."""
    page, nkv, hd, layers = case["page"], case["nkv"], case["hd"], case.get("layers", 1)
    s = {}
    for name, shape, std in (("k", (layers, total, nkv, page, hd), 1.0), ("v", (layers, total, nkv, hd, page), 0.6)):
        if case["cache"] != "e4m3":
            s[name] = torch.empty(shape, dtype=TYPE[case["cache"]], device="cuda").normal_(0, std, generator=g)
            continue
        s[name] = torch.empty(shape, dtype=E4M3, device="cuda")
        s[name + "_scale"] = torch.empty(shape[:3], device="cuda")
        for i in range(layers):
            x = torch.randn(shape[1:], generator=g, device="cuda").mul_(std)
            power = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448)))
            s[name][i], s[name + "_scale"][i] = (x / power[..., None, None]).to(E4M3), power
            del x
    return s


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def _window_state(case, seed, g):
    n, length = _spread(case)
    page, nq, nkv, hd, tokens = case["page"], case["nq"], case["nkv"], case["hd"], sum(n)
    t = TYPE[case["dtype"]]
    used = []  # the pages of each sequence: those that the window and the sinks reach, or all
    for rows, keys in zip(n, length):
        first = _reach(case, rows, keys) // page
        used.append([i for i in range(-(-keys // page)) if not case["freed"] or i >= first or i * page < case["sinks"]])
    total = sum(map(len, used)) + 3
    order = np.random.default_rng(seed).permutation(total)  # pages of a cache in use lie anywhere
    table = np.full((case["seqs"], -(-max(length) // page)), -1, np.int32)
    at = 0
    for q, cols in enumerate(used):
        table[q, cols] = order[at:at + len(cols)]
        at += len(cols)
    start = np.concatenate([[0], np.cumsum(n)])
    seq = np.repeat(np.arange(case["seqs"]), n)
    s = {"row_start": _ints(start), "kv_len": _ints(length), "table": _ints(table), "max_rows": max(n), "max_len": max(length),
         "seq": torch.from_numpy(seq).cuda(), "row": torch.from_numpy(np.arange(tokens) - start[seq]).cuda(),
         "at": torch.from_numpy(np.arange(tokens) - start[seq] + np.array(length)[seq] - np.array(n)[seq]).cuda()}
    # the batch's plan: the keys that any row of a sequence sees, first the sinks in front of its window
    reach = np.array([_reach(case, r, k) for r, k in zip(n, length)])
    most = max(k - w for k, w in zip(length, reach))
    near = reach[:, None] + np.arange(most)[None]
    far = np.repeat(np.arange(case["sinks"])[None], case["seqs"], 0)
    keys = np.concatenate([np.where(far < reach[:, None], far, -1), np.where(near < np.array(length)[:, None], near, -1)], 1)
    s["keys"] = torch.from_numpy(keys).cuda()
    s.update({k: v[0] for k, v in _cache(case, total, g).items()})
    s["q"] = torch.randn(tokens, nq * hd, generator=g, device="cuda").to(t)
    s["out"] = torch.zeros(tokens, nq * hd, dtype=t, device="cuda")
    return s


def _select_state(case, g):
    rows, n = case["groups"] * case["beams"], case["groups"] * case["width"]
    x = torch.randn(rows, case["vocab"], generator=g, device="cuda").mul_(2.0)
    liked = torch.randint(0, case["vocab"], (case["groups"], 12), generator=g, device="cuda").repeat_interleave(case["beams"], 0)
    x.scatter_add_(1, liked, torch.rand(rows, 12, generator=g, device="cuda").mul_(12.0))  # tokens that a clip's beams agree on
    ld = (case["vocab"] + 7) // 8 * 8
    logits = torch.zeros(rows, ld, dtype=TYPE[case["dtype"]], device="cuda")
    logits[:, : case["vocab"]] = x.to(logits.dtype)
    score = torch.rand(rows, generator=g, device="cuda").mul_(-9.0)
    done = (torch.rand(rows, generator=g, device="cuda") < (0.2 if case["done"] else 0.0)).to(torch.int32)
    s = {"logits": logits, "score": score, "done": done, "end": case["vocab"] // 3, "parent": torch.zeros(n, dtype=torch.int32, device="cuda")}
    s.update(token=torch.zeros_like(s["parent"]), done_out=torch.zeros_like(s["parent"]), score_out=torch.zeros(n, device="cuda"))
    return s


def _beams(case):
    """Lengths, shared and own pages of each group of a fork case, and the parents that its next step takes."""
    r = random.Random(case["past"] * 64 + case["groups"] * 8 + case["beams"])
    plan = []
    for _ in range(case["groups"]):
        prompt, extra = r.randint((case["past"] + 1) // 2, case["past"]), r.randint(0, case["extra"])
        keys = prompt + extra
        shared, every = prompt // case["page"], -(-keys // case["page"])
        first = max(0, keys - 1 - case["window"] + 1) // case["page"] if case["window"] else 0
        cols = [i for i in range(every) if i >= first or i * case["page"] < case["sinks"]]
        plan.append((keys, [i for i in cols if i < shared], [i for i in cols if i >= shared], [r.randrange(case["beams"]) for _ in range(case["beams"])]))
    return plan


def _fork_state(case, seed, g):
    plan, beams = _beams(case), case["beams"]
    seqs, width = case["groups"] * beams, max(-(-(p[0] + 1) // case["page"]) for p in plan) + 1
    total = sum(len(p[1]) + beams * (len(p[2]) + 1) for p in plan) + 5
    order = iter(np.random.default_rng(seed).permutation(total).tolist())
    table, refs = np.full((seqs, width), -1, np.int32), np.zeros(total, np.int32)
    for i, (_, shared, mine, _) in enumerate(plan):
        both = [next(order) for _ in shared]
        for b in range(beams):
            table[i * beams + b, shared] = both
            table[i * beams + b, mine] = [next(order) for _ in mine]
    np.add.at(refs, table[table >= 0], 1)
    s = {"tables": [_ints(table), _ints(np.full_like(table, -1))], "turn": 0, "refs": _ints(refs),
         "src_len": _ints([p[0] for p in plan for _ in range(beams)]), "len": _ints(np.zeros(seqs)), "grow": _ints(np.ones(seqs)),
         "parent": _ints([i * beams + q for i, p in enumerate(plan) for q in p[3]]), "missing": _ints([0])}
    s.update(_cache(case, total, g))
    return s


def _compact_state(case, seed, g):
    total, r = case["pages"], np.random.default_rng(seed)
    n = max(case["seqs"], min(total, round(total * case["used"])))
    where = r.permutation(total)[:n]
    cut = np.sort(np.random.default_rng(total).choice(np.arange(1, n), case["seqs"] - 1, replace=False)) if case["seqs"] > 1 else []
    parts = np.split(where, cut)
    table = np.full((case["seqs"], max(map(len, parts)) + 1), -1, np.int32)
    for q, p in enumerate(parts):
        table[q, :len(p)] = p
    if case["seqs"] > 1:
        table[1, 0] = table[0, 0]  # a page that two sequences share; the second's own first page is nobody's
    refs = np.zeros(total, np.int32)
    np.add.at(refs, table[table >= 0], 1)
    s = {"refs": _ints(refs), "table": _ints(table), "refs_out": _ints(refs), "table_out": _ints(table), "map": _ints(refs), "used": _ints([0])}
    s.update(_cache(case, total, g))
    return s


def _copy_state(case, seed, g):
    r = np.random.default_rng(seed)
    s = {"pairs": _ints(np.stack([r.permutation(case["pages"])[: case["pairs"]], r.permutation(case["pages"] + 7)[: case["pairs"]]], 1))}
    s.update(_cache(case, case["pages"], g))
    for n in _planes(case):
        x = s[n]
        s["to_" + n] = torch.zeros((x.shape[0], case["pages"] + 7) + x.shape[2:], dtype=x.dtype, device="cuda")
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    s = (_window_state(case, seed, g) if kind == "window" else _select_state(case, g) if kind == "select" else _fork_state(case, seed, g) if kind == "fork"
         else _compact_state(case, seed, g) if kind == "compact" else _copy_state(case, seed, g))
    torch.cuda.synchronize()
    return {"case": case, **s}


def _planes(case):
    return ("k", "v", "k_scale", "v_scale") if case["cache"] == "e4m3" else ("k", "v")


# ---- the framework's calls ------------------------------------------------

_ctx = None


def _list(pkg, s, prefix=""):
    """Every layer's pages: a pool's planes."""
    each = [(x.data_ptr(), x.element_size() * x[0].numel()) for n in _planes(s["case"]) for x in s[prefix + n]]
    return (pkg.PagePlane * len(each))(*each)


def _workspace(s, d, size):
    s["workspace"] = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = s["workspace"].data_ptr(), size
    return d


def _calls(s):
    """The descriptors that a program keeps for its step: one, or two that take turns."""
    global _ctx
    from __graft_entry__ import load_package
    pkg = load_package()
    if _ctx is None:
        _ctx = pkg.Context(0)
    c = s["case"]
    dt = {"f16": pkg.F16, "bf16": pkg.BF16, "e4m3": pkg.E4M3, "f32": pkg.F32}

    def p(name):
        return s[name].data_ptr() if name in s else None

    if c["kind"] == "window":
        kv = pkg.PagedKV(dtype=dt[c["cache"]], page=c["page"], nkvh=c["nkv"], hd=c["hd"], num_pages=s["k"].shape[0], k=p("k"), v=p("v"),
                         k_scale=p("k_scale"), v_scale=p("v_scale"), table=p("table"), ldtable=s["table"].shape[1], seqs=c["seqs"],
                         row_start=p("row_start"), kv_len=p("kv_len"), max_rows=s["max_rows"], max_len=s["max_len"])
        d = pkg.PagedWindowDesc(dtype=dt[c["dtype"]], flags=0, tokens=s["q"].shape[0], nqh=c["nq"], q=p("q"), ldq=s["q"].shape[1],
                                kv=ctypes.pointer(kv), out=p("out"), ldo=s["out"].shape[1], window=c["window"], sinks=c["sinks"])
        return _ctx.attention_paged_window, [_workspace(s, d, pkg.attention_paged_window_workspace(d))]
    if c["kind"] == "select":
        d = pkg.BeamDesc(dtype=dt[c["dtype"]], flags=0, groups=c["groups"], beams=c["beams"], width=c["width"], vocab=c["vocab"], logits=p("logits"),
                         ldl=s["logits"].shape[1], score=p("score"), done=p("done"), end=s["end"], parent=p("parent"), token=p("token"),
                         score_out=p("score_out"), done_out=p("done_out"))
        return _ctx.beam_select, [_workspace(s, d, pkg.beam_select_workspace(d))]
    planes = _list(pkg, s)
    if c["kind"] == "fork":
        seqs, width = s["tables"][0].shape
        both = [pkg.PagesForkDesc(flags=0, page=c["page"], num_pages=s["refs"].numel(), planes=planes, nplanes=len(planes), refs=p("refs"), src_seqs=seqs,
                                  seqs=seqs, ldtable=width, src_table=s["tables"][i].data_ptr(), src_len=p("src_len"), parent=p("parent"),
                                  table=s["tables"][1 - i].data_ptr(), len=p("len"), grow=p("grow"), window=c["window"], sinks=c["sinks"],
                                  missing=p("missing")) for i in range(2)]
        size = pkg.pages_fork_workspace(both[0])
        return _ctx.pages_fork, [_workspace(s, both[0], size), _workspace(s, both[1], size)]
    if c["kind"] == "compact":
        d = pkg.PagesCompactDesc(flags=0, num_pages=c["pages"], planes=planes, nplanes=len(planes), refs=p("refs"), refs_out=p("refs_out"), seqs=c["seqs"],
                                 ldtable=s["table"].shape[1], table=p("table"), table_out=p("table_out"), map=p("map"), used=p("used"))
        return _ctx.pages_compact, [_workspace(s, d, pkg.pages_compact_workspace(d))]
    to = _list(pkg, s, "to_")
    return _ctx.pages_copy, [pkg.PagesCopyDesc(flags=0, nplanes=len(planes), src=planes, src_pages=c["pages"], dst=to, dst_pages=c["pages"] + 7,
                                               pairs=p("pairs"), npairs=c["pairs"])]


def run(state):
    kind = state["case"]["kind"]
    turn = state.get("turn", 0)
    if kind == "fork":
        state["turn"] = 1 - turn
    if own:
        if "call" not in state:
            state["call"] = _calls(state)
        call, descs = state["call"]
        call(descs[turn])
        return _answer(state, turn)
    return {"window": _window, "select": _select, "fork": _fork, "compact": _compact, "copy": _copy}[kind](state, turn)


def _answer(s, turn):
    kind = s["case"]["kind"]
    if kind == "window":
        return {"out": s["out"]}
    if kind == "select":
        return {"parent": s["parent"], "token": s["token"], "score": s["score_out"], "done": s["done_out"]}
    if kind == "copy":
        return {n: s["to_" + n] for n in _planes(s["case"])}
    out = {n: s[n] for n in _planes(s["case"])}
    if kind == "fork":
        return {"table": s["tables"][1 - turn], "len": s["len"], "refs": s["refs"], "missing": s["missing"], **out}
    return {"table": s["table_out"], "refs": s["refs_out"], "map": s["map"], "used": s["used"], **out}


# ---- the plain forms ------------------------------------------------------

def _bytes(x):
    return x.view(torch.uint8) if x.dtype == E4M3 else x


def _window(s, _):
    c = s["case"]
    nq, nkv, hd, n, page = c["nq"], c["nkv"], c["hd"], c["seqs"], c["page"]
    at = s["keys"].clamp(min=0)
    ids = s["table"].long().gather(1, at // page)
    on = (s["keys"] >= 0) & (ids >= 0)
    ids = ids.clamp(min=0)
    k, v = _bytes(s["k"])[ids, :, at % page], _bytes(s["v"])[ids, :, :, at % page]  # [n, keys, nkv, hd]
    if c["cache"] == "e4m3":
        k, v = (x.view(E4M3).float() * s[m][ids][..., None] for x, m in ((k, "k_scale"), (v, "v_scale")))
    k, v = k.float().transpose(1, 2).contiguous(), v.float().transpose(1, 2).contiguous()
    q = torch.zeros(n, s["max_rows"], nkv, nq // nkv, hd, device="cuda")
    q[s["seq"], s["row"]] = s["q"].view(-1, nkv, nq // nkv, hd).float()
    pos = torch.full((n, s["max_rows"]), -1, dtype=torch.int64, device="cuda")
    pos[s["seq"], s["row"]] = s["at"]
    see = on[:, None] & (s["keys"][:, None] <= pos[..., None]) & ((s["keys"][:, None] > pos[..., None] - c["window"]) | (s["keys"][:, None] < c["sinks"]))
    q = q.permute(0, 2, 1, 3, 4).reshape(n, nkv, -1, hd)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(hd ** -0.5).view(n, nkv, s["max_rows"], nq // nkv, -1)
    score.masked_fill_(~see[:, None, :, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-30)).view(n, nkv, -1, k.shape[2])
    o = torch.matmul(p, v).view(n, nkv, s["max_rows"], nq // nkv, hd).permute(0, 2, 1, 3, 4)
    return {"out": o[s["seq"], s["row"]].reshape(-1, nq * hd).to(TYPE[c["dtype"]])}


def _select(s, _):
    c = s["case"]
    beams, vocab, width, end = c["beams"], c["vocab"], c["width"], s["end"]
    x = s["logits"][:, :vocab].double()  # candidates are ranked across beams: 64 bits
    top = x.amax(1, keepdim=True)
    logp = x - top - (x - top).exp_().sum(1, keepdim=True).log_()
    done = s["done"][:, None] != 0
    only = (torch.arange(vocab, device="cuda") == end).double().log_()  # an ended beam goes on with its end, at no cost
    total = (s["score"].double()[:, None] + torch.where(done, only, logp)).view(c["groups"], -1)
    least = total.topk(width, 1).values[:, -1:]
    above, level = total > least, total == least
    chosen = above | (level & (level.cumsum(1) <= width - above.sum(1, keepdim=True)))
    index = torch.arange(total.shape[1], 0, -1, device="cuda")
    at = total.shape[1] - (chosen * index).topk(width, 1).values  # rising indices
    value, order = total.gather(1, at).sort(dim=1, descending=True, stable=True)
    at, dead = at.gather(1, order), value == -math.inf
    parent = at // vocab + torch.arange(c["groups"], device="cuda")[:, None] * beams
    token = torch.where(dead, -1, at % vocab)
    over = ((s["done"][parent] != 0) | (token == end)) & ~dead
    out = {"parent": torch.where(dead, -1, parent), "token": token, "done": over}
    return {"score": value.float().view(-1), **{n: y.to(torch.int32).view(-1) for n, y in out.items()}}


def _fork(s, turn):
    c = s["case"]
    page, refs, src, dst = c["page"], s["refs"], s["tables"][turn], s["tables"][1 - turn]
    seqs, width = src.shape
    col, i = torch.arange(width, device="cuda"), torch.arange(seqs, device="cuda")
    parent = s["parent"].long()
    have = s["src_len"].long()[parent]
    now = torch.clamp(have + s["grow"], max=width * page)
    keep = col < ((have + page - 1) // page)[:, None]
    if c["window"]:
        keep &= (col * page < c["sinks"]) | ((col + 1) * page > (have - c["window"] + 1)[:, None])
    new = torch.where(keep, src[parent], -1)
    for t, by in ((src, -1), (new, 1)):
        refs.index_add_(0, t.clamp(min=0).view(-1), ((t >= 0) * by).to(torch.int32).view(-1))
    # the page that a sequence goes on writing: its own, or a copy
    last = new.gather(1, (have // page).clamp(max=width - 1)[:, None])[:, 0].long()
    part = (have % page != 0) & (now > have) & (last >= 0)
    writers = torch.zeros_like(refs).index_add_(0, last.clamp(min=0), part.to(torch.int32))
    first = torch.full_like(refs, seqs).scatter_reduce_(0, last.clamp(min=0), torch.where(part, i, seqs).to(torch.int32), "amin")
    copy = part & ~((refs[last] == writers[last]) & (first[last] == i))
    fresh = (col >= ((have + page - 1) // page)[:, None]) & (col < ((now + page - 1) // page)[:, None])
    fresh |= copy[:, None] & (col == (have // page)[:, None])
    free = (refs <= 0).nonzero()[:, 0]
    new[fresh] = free[: int(fresh.sum())].to(torch.int32)  # in order of sequences, then of positions
    refs.index_add_(0, last.clamp(min=0), -copy.to(torch.int32))
    refs[new[fresh].long()] = 1
    for n in _planes(c):
        x = _bytes(s[n])
        x[:, new.gather(1, (have // page).clamp(max=width - 1)[:, None])[copy, 0].long()] = x[:, last[copy]]
    dst.copy_(new)
    s["len"].copy_(now)
    return _answer(s, turn)


def _compact(s, turn):
    refs, table = s["refs"], s["table"]
    used = refs > 0
    n = used.sum()
    at = torch.arange(refs.numel(), device="cuda")
    gaps, late = (~used & (at < n)).nonzero()[:, 0], (used & (at >= n)).nonzero()[:, 0]
    to = torch.where(used, at, -1)
    to[late] = gaps
    s["refs_out"].copy_(torch.where(used & (at < n), refs, 0))
    s["refs_out"][gaps] = refs[late]
    s["table_out"].copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    s["map"].copy_(to)
    s["used"].copy_(n)
    for m in _planes(s["case"]):
        x = _bytes(s[m])
        x[:, gaps] = x[:, late]
    return _answer(s, turn)


def _copy(s, turn):
    src, dst = s["pairs"].long().T
    for n in _planes(s["case"]):
        _bytes(s["to_" + n])[:, dst] = _bytes(s[n])[:, src]
    return _answer(s, turn)


# ---- what a pass cannot do without ----------------------------------------

def _page_bytes(case):
    """A page over all layers."""
    e4m3 = case["cache"] == "e4m3"
    return 2 * case["layers"] * case["nkv"] * (case["page"] * case["hd"] * (1 if e4m3 else 2) + (4 if e4m3 else 0))


def work(case):
    kind = case["kind"]
    if kind == "window":
        hd, nq, nkv = case["hd"], case["nq"], case["nkv"]
        n, length = _spread(case)
        each = 1 if case["cache"] == "e4m3" else 2
        reach = [_reach(case, r, k) for r, k in zip(n, length)]
        keys = sum(k - w + min(case["sinks"], w) for k, w in zip(length, reach))
        pairs = sum(min(case["window"], p + 1) + min(case["sinks"], max(0, p + 1 - case["window"])) for r, k in zip(n, length) for p in range(k - r, k))
        return {"bytes": 4 * sum(n) * nq * hd + 2 * nkv * hd * each * keys, "flops": 4 * pairs * nq * hd}
    if kind == "select":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * case["vocab"] * (4 if case["dtype"] == "f32" else 2) + 8 * rows + 16 * case["groups"] * case["width"],
                "flops": 4 * rows * case["vocab"]}
    if kind == "copy":
        return {"bytes": 2 * case["pairs"] * _page_bytes(case) + 8 * case["pairs"], "flops": 0}
    if kind == "compact":
        n = max(case["seqs"], min(case["pages"], round(case["pages"] * case["used"]))) - (case["seqs"] > 1)
        moved = round(n * (1 - n / case["pages"]))  # of n used pages anywhere, those behind the first n
        return {"bytes": 2 * moved * _page_bytes(case) + 12 * case["pages"] + 8 * n, "flops": 0}
    plan, beams = _beams(case), case["beams"]
    copies = sum(beams - len(set(p[3])) for p in plan if p[0] % case["page"])
    entries = sum(beams * (len(p[1]) + len(p[2])) for p in plan)
    total = sum(len(p[1]) + beams * (len(p[2]) + 1) for p in plan) + 5
    return {"bytes": 2 * copies * _page_bytes(case) + 8 * entries + 8 * total + 16 * len(plan) * beams, "flops": 0}


# ---- the same from the definitions, in 64 bits ------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"window": _exact_window, "select": _exact_select, "fork": _exact_fork, "compact": _exact_compact, "copy": _exact_copy}[case["kind"]](case, s)


def _exact_window(case, s):
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    n, length = _spread(case)
    table, first, out = s["table"].tolist(), 0, []
    for i, (rows, keys) in enumerate(zip(n, length)):
        cols = [j for j, p in enumerate(table[i][: -(-keys // page)]) if p >= 0]
        used = [table[i][j] for j in cols]
        k, v = (s[m].view(torch.uint8)[used].view(s[m].dtype).double() for m in ("k", "v"))
        if case["cache"] == "e4m3":
            k, v = k * s["k_scale"][used].double()[..., None, None], v * s["v_scale"][used].double()[..., None, None]
        k, v = k.transpose(0, 1).reshape(nkv, -1, hd), v.permute(1, 0, 3, 2).reshape(nkv, -1, hd)
        at = (torch.tensor(cols, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).view(1, -1)
        p = torch.arange(keys - rows, keys, device="cuda")[:, None]
        hidden = ~((at <= p) & ((p - at < case["window"]) | (at < case["sinks"])))
        q = s["q"][first:first + rows].double().view(rows, nq, hd)
        heads = [torch.softmax((q[:, h] @ k[h * nkv // nq].T / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1) @ v[h * nkv // nq] for h in range(nq)]
        out.append(torch.stack(heads, 1).view(rows, nq * hd))
        first += rows
    return {"out": torch.cat(out)}


def _exact_select(case, s):
    beams, vocab, width = case["beams"], case["vocab"], case["width"]
    score, done = s["score"].tolist(), s["done"].tolist()
    out = {"parent": [], "token": [], "score": [], "done": []}
    for g in range(case["groups"]):
        found = []
        for b in range(g * beams, (g + 1) * beams):
            if done[b]:
                found.append((-score[b], b, s["end"]))
                continue
            logp = torch.log_softmax(s["logits"][b, :vocab].double(), 0)
            order = torch.argsort(logp, descending=True, stable=True)[:width]
            found += [(-(score[b] + x), b, t) for x, t in zip(logp[order].tolist(), order.tolist())]
        best = (sorted(found) + [(math.inf, -1, -1)] * width)[:width]
        for x, b, t in best:
            for name, y in zip(("score", "parent", "token", "done"), (-x, b, t, int(b >= 0 and (done[b] != 0 or t == s["end"])))):
                out[name].append(y)
    return {n: torch.tensor(y, dtype=torch.float64 if n == "score" else torch.int32) for n, y in out.items()}


def _moved(case, s, pairs, into=""):
    """The planes with page `d` of `into` taking page `a`."""
    out = {n: s[into + n].clone() for n in _planes(case)}
    for n, x in out.items():
        for a, d in pairs:
            _bytes(x)[:, d] = _bytes(s[n])[:, a]
    return out


def _exact_fork(case, s):
    page, refs, src = case["page"], s["refs"].tolist(), s["tables"][0].tolist()
    have, parent = s["src_len"].tolist(), s["parent"].tolist()
    seqs, width = len(src), len(src[0])
    table, length, writes = [], [], {}
    for i, q in enumerate(parent):
        at = [src[q][j] if j * page < have[q] and (not case["window"] or j * page < case["sinks"] or (j + 1) * page - 1 > have[q] - case["window"]) else -1
              for j in range(width)]
        table.append(at)
        length.append(min(have[q] + 1, width * page))
        if have[q] % page and length[i] > have[q] and at[have[q] // page] >= 0:
            writes.setdefault(at[have[q] // page], []).append(i)
    for t, by in ((src, -1), (table, 1)):
        for at in t:
            for p in at:
                if p >= 0:
                    refs[p] += by
    free, pairs = (p for p in range(len(refs)) if refs[p] <= 0), []
    free = list(free)
    whole = {p: refs[p] == len(w) for p, w in writes.items()}
    for i, q in enumerate(parent):
        j = have[q] // page
        p = table[i][j] if have[q] % page and length[i] > have[q] else -1
        if p >= 0 and not (whole[p] and writes[p][0] == i):
            d = free.pop(0)
            pairs.append((p, d))
            table[i][j], refs[d] = d, 1
            refs[p] -= 1
        for j in range(-(-have[q] // page), -(-length[i] // page)):
            table[i][j] = free.pop(0)
            refs[table[i][j]] = 1
    ints = {"table": table, "len": length, "refs": refs, "missing": [0]}
    return {**{n: torch.tensor(y, dtype=torch.int32) for n, y in ints.items()}, **_moved(case, s, pairs)}


def _exact_compact(case, s):
    refs, table = s["refs"].tolist(), s["table"].tolist()
    used = [p for p, r in enumerate(refs) if r > 0]
    n, name = len(used), {p: p for p in used}
    gaps = [p for p in range(n) if refs[p] <= 0]
    pairs = list(zip([p for p in used if p >= n], gaps))
    name.update(pairs)
    after = [0] * len(refs)
    for p, d in name.items():
        after[d] = refs[p]
    ints = {"table": [[name.get(p, -1) for p in at] for at in table], "refs": after, "map": [name.get(p, -1) for p in range(len(refs))], "used": [n]}
    return {**{m: torch.tensor(y, dtype=torch.int32) for m, y in ints.items()}, **_moved(case, s, pairs)}


def _exact_copy(case, s):
    return _moved(case, s, s["pairs"].tolist(), "to_")
