"""The paged decoder operators, measured: rotary rows with several position axes,
appending keys and values to a paged cache, attention over that cache.

Together they let the text decoder run several sequences of different length
at once, whole prompts, parts of prompts and single tokens mixed.  A batch is
packed: row_start[s]..row_start[s + 1] are sequence s's new rows, kv_len[s] its
keys with them, table[s] its pages.  A K page is [page][hd], a V page
[hd][page]; an e4m3 cache has a scale (a power of two) for each page and kv head.

Kinds of case:
  mrope      positions [axes][tokens] to cos / sin rows
  append     q / k head norm, rotation, K and V into the pages
  attention  causal attention of the packed rows over the pages
"""
from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import torch

own = False

TYPE = {"f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
EPS, THETA = 1e-6, 1e6


def listed():
    return [
        # The rotary rows of one step of 32 sequences: a token each, every axis alike.
        {"name": "mrope_step_32", "kind": "mrope", "dtype": "f16", "tokens": 32, "hd": 128, "axes": 1, "inter": False},
        # Two minutes of video between text: time, height and width, interleaved frequencies.
        {"name": "mrope_video", "kind": "mrope", "dtype": "bf16", "tokens": 30720, "hd": 128, "axes": 3, "inter": True},
        # One step of 32 sequences behind prompts of up to five minutes of audio, 16-bit pages.
        {"name": "append_step_32", "kind": "append", "dtype": "f16", "cache": "f16", "page": 16, "nq": 16, "nkv": 8, "hd": 128,
         "seqs": 32, "rows": 1, "long": 1, "past": 4352},
        # The same for 24 sequences into an e4m3 cache: each page may have to take a larger scale.
        {"name": "append_step_e4m3", "kind": "append", "dtype": "bf16", "cache": "e4m3", "page": 64, "nq": 16, "nkv": 8, "hd": 128,
         "seqs": 24, "rows": 1, "long": 1, "past": 2176},
        # The prompt of a 300 s clip into an empty e4m3 cache.
        {"name": "append_prompt_4334", "kind": "append", "dtype": "f16", "cache": "e4m3", "page": 32, "nq": 16, "nkv": 8, "hd": 128,
         "seqs": 1, "rows": 4334, "long": 4334, "past": 0},
        # One step of one sequence behind a 15 s clip's prompt: latency.
        {"name": "decode_1_323", "kind": "attention", "dtype": "f16", "cache": "f16", "page": 16, "nq": 16, "nkv": 8, "hd": 128,
         "seqs": 1, "rows": 1, "long": 1, "past": 322},
        # One step of one sequence with a long past.
        {"name": "decode_1_32771", "kind": "attention", "dtype": "bf16", "cache": "e4m3", "page": 64, "nq": 16, "nkv": 8, "hd": 128,
         "seqs": 1, "rows": 1, "long": 1, "past": 32770},
        # One step of 32 sequences of up to 300 s of audio, 16-bit pages.
        {"name": "decode_32", "kind": "attention", "dtype": "f16", "cache": "f16", "page": 16, "nq": 16, "nkv": 8, "hd": 128,
         "seqs": 32, "rows": 1, "long": 1, "past": 4352},
        # One step of 64 sequences with longer pasts, four q heads to a kv head, e4m3.
        {"name": "decode_64_e4m3", "kind": "attention", "dtype": "bf16", "cache": "e4m3", "page": 32, "nq": 32, "nkv": 8, "hd": 128,
         "seqs": 64, "rows": 1, "long": 1, "past": 8192},
        # The later part of a prompt that is prefilled in two parts.
        {"name": "chunk_771", "kind": "attention", "dtype": "f16", "cache": "f16", "page": 64, "nq": 16, "nkv": 8, "hd": 128,
         "seqs": 1, "rows": 771, "long": 771, "past": 1536},
        # Twenty sequences at one token each and one with 501 rows of its prompt; heads of 64, three to a kv head.
        {"name": "mixed_21", "kind": "attention", "dtype": "bf16", "cache": "e4m3", "page": 16, "nq": 12, "nkv": 4, "hd": 64,
         "seqs": 21, "rows": 1, "long": 501, "past": 1500},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("mrope", "append", "append", "attention", "attention", "attention", "attention"))
    c = {"kind": kind, "dtype": rng.choice(("f16", "bf16"))}
    if kind == "mrope":
        axes = rng.choice((1, 2, 3))
        return {**c, "tokens": _log(rng, 1, 30720), "hd": rng.choice((64, 128)), "axes": axes, "inter": axes > 1 and rng.random() < 0.6}
    nkv = rng.choice((1, 2, 4, 8))
    c.update(cache=rng.choice((c["dtype"], "e4m3")), page=rng.choice((16, 32, 64)), nq=nkv * rng.choice((1, 2, 2, 3, 4)), nkv=nkv,
             hd=rng.choice((64, 128, 128)))
    seqs = _log(rng, 1, 64)
    shape = rng.choice(("step", "step", "part", "mixed"))
    past = _log(rng, 1, min(32768, 64 * 8192 // seqs // 2))
    if shape == "step":
        return {**c, "seqs": seqs, "rows": 1, "long": 1, "past": past}
    c["nkv"], c["nq"] = min(c["nkv"], 4), min(c["nkv"], 4) * (c["nq"] // c["nkv"])
    rows = _log(rng, 2, 1200)
    if shape == "part":  # prompts, or parts of them, of about the same length
        return {**c, "seqs": max(1, min(seqs, 1200 // rows)), "rows": rows, "long": rows, "past": min(rng.choice((0, past)), 1500)}
    return {**c, "seqs": min(seqs, 24), "rows": 1, "long": min(rows, 700), "past": min(past, 2000)}


# ---- inputs ---------------------------------------------------------------

def _batch(case):
    """Rows and keys of each sequence: the last has `long` rows, the others up to `rows`; pasts are spread up to `past`."""
    r = random.Random(case["past"] * 64 + case["seqs"])
    n = [case["rows"] if case["rows"] == 1 else r.randint((case["rows"] + 1) // 2, case["rows"]) for _ in range(case["seqs"] - 1)] + [case["long"]]
    past = [case["past"]] + [r.randint(case["past"] // 8, case["past"]) for _ in range(case["seqs"] - 1)]
    return n, [p + k for p, k in zip(past, n)]


def _sections(case):
    """Frequencies of each axis: most for time, as the rest is split evenly."""
    half, axes = case["hd"] // 2, case["axes"]
    other = half * 5 // 16 if axes > 1 else 0
    return [half - other * (axes - 1)] + [other] * (axes - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPE[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean)

    hd = case["hd"]
    if case["kind"] == "mrope":
        n, axes = case["tokens"], case["axes"]
        i = torch.arange(n, device="cuda")
        grid = [i] if axes == 1 else [i // 576, i // 24 % 24, i % 24][3 - axes:]  # frames of 24 x 24 patches: time, height, width
        pos = torch.stack(grid) + torch.randint(0, 32768, (1, 1), generator=g, device="cuda")  # behind the text before them
        return {"case": case, "pos": pos.to(torch.int32), "sec": _sections(case),
                "cos": torch.empty(n, hd, device="cuda"), "sin": torch.empty(n, hd, device="cuda")}
    n, length = _batch(case)
    page, nq, nkv, tokens = case["page"], case["nq"], case["nkv"], sum(n)
    start = np.concatenate([[0], np.cumsum(n)])
    pages = [-(-k // page) for k in length]
    total, width = sum(pages) + 3, max(pages)
    order = np.random.default_rng(seed).permutation(total)  # pages of a cache in use lie anywhere
    table = np.full((case["seqs"], width), -1, np.int32)
    for s, k in enumerate(pages):
        table[s, :k] = order[sum(pages[:s]):sum(pages[:s]) + k]
    s = {"case": case, "row_start": torch.from_numpy(start.astype(np.int32)).cuda(), "kv_len": torch.tensor(length, dtype=torch.int32, device="cuda"),
         "table": torch.from_numpy(table).cuda(), "max_rows": max(n), "max_len": max(length)}
    # the plan of the batch, made with the table: each row's sequence, position, page and slot
    seq = np.repeat(np.arange(case["seqs"]), n)
    at = np.arange(tokens) - start[seq] + np.array(length)[seq] - np.array(n)[seq]
    row_page = table[seq, at // page]
    s.update({k: torch.from_numpy(np.ascontiguousarray(v, np.int64)).cuda() for k, v in (
        ("seq", seq), ("at", at), ("row", np.arange(tokens) - start[seq]), ("page", row_page), ("slot", at % page), ("touched", np.unique(row_page)))})
    s["fresh"] = torch.from_numpy(np.isin(np.unique(row_page), row_page[at % page == 0])).cuda()[:, None]
    if case["cache"] == "e4m3":
        for name, shape, dim in (("k", (total, nkv, page, hd), 1.0), ("v", (total, nkv, hd, page), 0.6)):
            x = normal(*shape, std=dim)
            scale = _power(x.abs().amax((2, 3)))
            s[name], s[name + "_scale"] = (x / scale[..., None, None]).clamp_(-448, 448).to(E4M3), scale
            del x
    else:
        s["k"], s["v"] = normal(total, nkv, page, hd).to(t), normal(total, nkv, hd, page, std=0.6).to(t)
    if case["kind"] == "append":
        ang = torch.from_numpy(at[:, None] / THETA ** (np.arange(hd // 2) * 2 / hd))
        s.update(qkv=normal(tokens, (nq + 2 * nkv) * hd).to(t), qn=normal(hd, std=0.1, mean=1.0), kn=normal(hd, std=0.1, mean=1.0),
                 q=torch.zeros(tokens, nq * hd, dtype=t, device="cuda"))
        s["cos"], s["sin"] = (torch.cat([f(ang)] * 2, 1).float().to(t).float().cuda() for f in (torch.cos, torch.sin))
    else:
        s.update(q=normal(tokens, nq * hd).to(t), out=torch.zeros(tokens, nq * hd, dtype=t, device="cuda"))
    torch.cuda.synchronize()
    return s


# ---- the framework's calls ------------------------------------------------

_ctx = None


def _calls(s):
    """The descriptor that a program keeps for each call of its step."""
    global _ctx
    from __graft_entry__ import load_package
    pkg = load_package()
    if _ctx is None:
        _ctx = pkg.Context(0)
    c = s["case"]
    dt = {"f16": pkg.F16, "bf16": pkg.BF16, "e4m3": pkg.E4M3}

    def p(name):
        return s[name].data_ptr() if name in s else None

    if c["kind"] == "mrope":
        sec = s["sec"] + [0, 0]
        return _ctx.mrope_rows, pkg.MropeDesc(
            dtype=dt[c["dtype"]], flags=pkg.MROPE_INTERLEAVED if c["inter"] else 0, tokens=c["tokens"], hd=c["hd"], axes=c["axes"],
            sec0=sec[0], sec1=sec[1], sec2=sec[2], theta=THETA, pos=p("pos"), ldpos=c["tokens"], cos=p("cos"), sin=p("sin"))
    kv = pkg.PagedKV(dtype=dt[c["cache"]], page=c["page"], nkvh=c["nkv"], hd=c["hd"], num_pages=s["k"].shape[0], k=p("k"), v=p("v"),
                     k_scale=p("k_scale"), v_scale=p("v_scale"), table=p("table"), ldtable=s["table"].shape[1], seqs=c["seqs"],
                     row_start=p("row_start"), kv_len=p("kv_len"), max_rows=s["max_rows"], max_len=s["max_len"])
    if c["kind"] == "append":
        return _ctx.kv_append, pkg.KvAppendDesc(
            dtype=dt[c["dtype"]], flags=0, tokens=s["qkv"].shape[0], nqh=c["nq"], eps=EPS, qkv=p("qkv"), ldqkv=s["qkv"].shape[1], qn_w=p("qn"),
            kn_w=p("kn"), cos=p("cos"), sin=p("sin"), q_out=p("q"), ldq=s["q"].shape[1], kv=ctypes.pointer(kv))
    d = pkg.PagedAttentionDesc(dtype=dt[c["dtype"]], flags=0, tokens=s["q"].shape[0], nqh=c["nq"], q=p("q"), ldq=s["q"].shape[1], kv=ctypes.pointer(kv),
                               out=p("out"), ldo=s["out"].shape[1], workspace=None, workspace_bytes=0)
    size = pkg.attention_paged_workspace(d)
    s["workspace"] = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = p("workspace"), size
    return _ctx.attention_paged, d


def run(state):
    kind = state["case"]["kind"]
    if own:
        if "call" not in state:
            state["call"] = _calls(state)
        call, desc = state["call"]
        call(desc)
        return {n: state[n] for n in (("cos", "sin") if kind == "mrope" else ("out",) if kind == "attention" else ("q", "k", "v", "k_scale", "v_scale"))
                if n in state}
    return _mrope(state) if kind == "mrope" else _append(state) if kind == "append" else _attention(state)


# ---- the plain forms ------------------------------------------------------

def _axis(case, sec):
    """The axis of each frequency."""
    j = torch.arange(case["hd"] // 2)
    if case["inter"]:
        a = j % case["axes"]
        return torch.where(j < case["axes"] * torch.tensor(sec)[a], a, 0)
    return torch.bucketize(j, torch.tensor(sec).cumsum(0), right=True)


def _mrope(s):
    c = s["case"]
    t = TYPE[c["dtype"]]
    inv = THETA ** (torch.arange(c["hd"] // 2, dtype=torch.float64, device="cuda") * (-2 / c["hd"]))
    ang = s["pos"][_axis(c, s["sec"]).cuda()].T.double() * inv
    cos, sin = torch.cos(ang).float().to(t).float(), torch.sin(ang).float().to(t).float()
    return {"cos": torch.cat([cos, cos], 1), "sin": torch.cat([sin, sin], 1)}


def _power(amax):
    """The least power of two p with amax <= 448 p."""
    m, e = torch.frexp(amax.float())  # amax = m 2^e, m in [0.5, 1)
    return torch.ldexp(torch.ones_like(m), torch.where(m > 0.875, e - 8, e - 9).clamp(-110, 120))


def _append(s):
    c = s["case"]
    t, nq, nkv, hd = TYPE[c["dtype"]], c["nq"], c["nkv"], c["hd"]
    x = s["qkv"].view(-1, nq + 2 * nkv, hd).float()

    def turn(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        return x * s["cos"][:, None] + torch.cat([-x[..., hd // 2:], x[..., : hd // 2]], -1) * s["sin"][:, None]

    q, k, v = turn(x[:, :nq], s["qn"]).to(t), turn(x[:, nq:nq + nkv], s["kn"]), x[:, nq + nkv:]
    out = {"q": q.view(-1, nq * hd), "k": s["k"], "v": s["v"]}
    if c["cache"] == "e4m3":
        out.update(k_scale=_scaled(s, "k", k), v_scale=_scaled(s, "v", v))
        k, v = ((x / s[n][s["page"]][..., None]).clamp(-448, 448).to(E4M3) for n, x in (("k_scale", k), ("v_scale", v)))
        _bytes(s["k"])[s["page"], :, s["slot"]] = _bytes(k)
        _bytes(s["v"])[s["page"], :, :, s["slot"]] = _bytes(v)
    else:
        s["k"][s["page"], :, s["slot"]] = k.to(t)
        s["v"][s["page"], :, :, s["slot"]] = v.to(t)
    return out


def _bytes(x):
    return x.view(torch.uint8)


def _scaled(s, name, x):
    """The scales with the new rows x; what touched pages held is rounded to them."""
    scale, at = s[name + "_scale"], s["touched"]
    top = torch.zeros_like(scale).index_reduce_(0, s["page"], x.abs().amax(-1), "amax")[at]
    new = torch.where(s["fresh"], _power(top), torch.maximum(scale[at], _power(top)))
    held = _bytes(s[name])[at].view(E4M3).float()
    _bytes(s[name])[at] = _bytes((held * torch.where(s["fresh"], 1, scale[at] / new)[..., None, None]).to(E4M3))
    scale[at] = new
    return scale


def _pages(s, name):
    """The sequences' pages as f32, [seqs, width, nkv, ...]."""
    at = s["table"].long().clamp(min=0)
    if s["case"]["cache"] == "e4m3":
        return _bytes(s[name])[at].view(E4M3).float() * s[name + "_scale"][at][..., None, None]
    return s[name][at].float()


def _attention(s):
    c = s["case"]
    nq, nkv, hd, n = c["nq"], c["nkv"], c["hd"], c["seqs"]
    k = _pages(s, "k").permute(0, 2, 1, 3, 4).reshape(n, nkv, -1, hd)
    v = _pages(s, "v").permute(0, 2, 1, 4, 3).reshape(n, nkv, -1, hd)
    q = torch.zeros(n, s["max_rows"], nkv, nq // nkv, hd, device="cuda")
    q[s["seq"], s["row"]] = s["q"].view(-1, nkv, nq // nkv, hd).float()
    last = torch.full((n, s["max_rows"]), -1, dtype=torch.int64, device="cuda")
    last[s["seq"], s["row"]] = s["at"]
    q = q.permute(0, 2, 1, 3, 4).reshape(n, nkv, -1, hd)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(hd ** -0.5).view(n, nkv, s["max_rows"], nq // nkv, -1)
    score.masked_fill_((torch.arange(k.shape[2], device="cuda") > last[..., None])[:, None, :, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-30)).view(n, nkv, -1, k.shape[2])
    o = torch.matmul(p, v).view(n, nkv, s["max_rows"], nq // nkv, hd).permute(0, 2, 1, 3, 4)
    return {"out": o[s["seq"], s["row"]].reshape(-1, nq * hd).to(TYPE[c["dtype"]])}


# ---- what a pass cannot do without ----------------------------------------

def work(case):
    hd = case["hd"]
    if case["kind"] == "mrope":
        n = case["tokens"]
        return {"bytes": 4 * case["axes"] * n + 8 * n * hd, "flops": 40 * n * hd // 2}
    n, length = _batch(case)
    nq, nkv, tokens, each = case["nq"], case["nkv"], sum(n), 1 if case["cache"] == "e4m3" else 2
    if case["kind"] == "append":
        return {"bytes": tokens * hd * (2 * (nq + 2 * nkv) + 8 + 2 * nq + 2 * nkv * each), "flops": 12 * tokens * hd * (nq + nkv)}
    pairs = sum(k * (m - k) + k * (k + 1) // 2 for k, m in zip(n, length))
    return {"bytes": 4 * tokens * nq * hd + 2 * nkv * hd * each * sum(length), "flops": 4 * pairs * nq * hd}


# ---- the same in 64 bits --------------------------------------------------

def _round_e4m3(x):
    """Doubles to the nearest e4m3 value, ties to even, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    hd = case["hd"]
    if case["kind"] == "mrope":
        j, axes = np.arange(hd // 2), case["axes"]
        if case["inter"]:
            a = [i % axes if i < axes * s["sec"][i % axes] else 0 for i in j]
        else:
            a = [x for x in range(axes) for _ in range(s["sec"][x])]
        ang = s["pos"].cpu().numpy().astype(np.float64)[a].T / THETA ** (2.0 * j / hd)
        return {n: torch.from_numpy(np.tile(f(ang), 2)).float().to(TYPE[case["dtype"]]).double() for n, f in (("cos", np.cos), ("sin", np.sin))}
    nq, nkv, page = case["nq"], case["nkv"], case["page"]
    n, length = _batch(case)
    table, e4m3 = s["table"].tolist(), case["cache"] == "e4m3"
    first = 0
    if case["kind"] == "attention":
        out = []
        for i, (rows, keys) in enumerate(zip(n, length)):
            used = table[i][: -(-keys // page)]
            k, v = s["k"].view(torch.uint8)[used].view(s["k"].dtype).double(), s["v"].view(torch.uint8)[used].view(s["v"].dtype).double()
            if e4m3:
                k, v = k * s["k_scale"][used].double()[..., None, None], v * s["v_scale"][used].double()[..., None, None]
            k, v = k.transpose(0, 1).reshape(nkv, -1, hd)[:, :keys], v.permute(1, 0, 3, 2).reshape(nkv, -1, hd)[:, :keys]
            hidden = torch.arange(keys, device="cuda")[None] > keys - rows + torch.arange(rows, device="cuda")[:, None]
            q = s["q"][first:first + rows].double().view(rows, nq, hd)
            heads = [torch.softmax((q[:, h] @ k[h * nkv // nq].T / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1) @ v[h * nkv // nq] for h in range(nq)]
            out.append(torch.stack(heads, 1).view(rows, nq * hd))
            first += rows
        return {"out": torch.cat(out)}
    x = s["qkv"].double().view(-1, nq + 2 * nkv, hd)
    cos, sin = s["cos"].double()[:, None], s["sin"].double()[:, None]

    def turned(y, w):
        y = y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + EPS) * w.double()
        a, b = y.chunk(2, -1)
        return torch.cat([a * cos[..., : hd // 2] - b * sin[..., : hd // 2], b * cos[..., hd // 2:] + a * sin[..., hd // 2:]], -1)

    q, k, v = turned(x[:, :nq], s["qn"]), turned(x[:, nq:nq + nkv], s["kn"]), x[:, nq + nkv:]
    out = {"q": q.reshape(-1, nq * hd), "k": s["k"].double(), "v": s["v"].double()}
    if e4m3:
        out.update(k_scale=s["k_scale"].double(), v_scale=s["v_scale"].double())
    for i, (rows, keys) in enumerate(zip(n, length)):
        at = keys - rows
        while at < keys:  # the rows of one page
            to = min(keys, (at // page + 1) * page)
            p, slots, of = table[i][at // page], slice(at % page, to - (at // page) * page), slice(first, first + to - at)
            for name, y in (("k", k[of].transpose(0, 1)), ("v", v[of].permute(1, 2, 0))):  # [nkv, rows, hd], [nkv, hd, rows]
                if e4m3:
                    power = torch.exp2(torch.ceil(torch.log2(y.abs().amax((1, 2)) / 448)))
                    if at % page:  # the page held rows: they are rounded again if its scale grows
                        power, old = torch.maximum(out[name + "_scale"][p], power), out[name + "_scale"][p]
                        out[name][p] = _round_e4m3(out[name][p] * (old / power)[:, None, None])
                    out[name + "_scale"][p], y = power, _round_e4m3(y / power[:, None, None])
                out[name][p][(slice(None), slots) if name == "k" else (slice(None), slice(None), slots)] = y
            first += to - at
            at = to
    return out
