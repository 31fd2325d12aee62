"""Cases of the int8 KV cache (append, read back, decode) and of decode attention over a shared prefix.

Every case is one pass through a public entry point of ``sf37_b200.kv`` on data a serving loop holds:

- ``store``:  rows written to int8 caches (``kv.append_i8``) and the attended rows read back into f16 or f32
  caches (``kv.read_i8``), as a chunked prefill over int8 caches does before its attention;
- ``decode``: one decode step over int8 caches (``kv.decode_i8``), for the layers of a model or the sequences
  of a batch, optionally with the step's K/V rows quantised into the caches;
- ``shared``: one decode step of a batch whose sequences share a prefix (``kv.decode_shared``), each with rows
  of its own in an f16 or int8 cache.

An int8 cache of ``cap`` rows holds bytes c + 128 as [cap][kv_heads][128], then f32 scales [kv_heads][cap].
"""
import math

import numpy as np
import torch

own = False

D = 128  # head_dim
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token of 48 sliding-window layers (512-row window, 1024-row ring) as a decode loop stores it
        dict(name="store_step", op="store", n=48, kv_heads=8, cap=1024, pos0=5000, n_tok=1, first=5000, rows=1,
             io="f32", dst="f16"),
        # an odd chunk that wraps its ring, few heads, read back in full precision
        dict(name="store_wrap", op="store", n=6, kv_heads=4, cap=2000, pos0=1700, n_tok=1537, first=1237, rows=2000,
             io="f32", dst="f32"),
        # the 8192-token prefill chunk on a 24576-token prefix: all attended rows are read back for the attention
        dict(name="store_chunk", op="store", n=1, kv_heads=8, cap=32768, pos0=24576, n_tok=8192, first=0, rows=32768,
             io="bf16", dst="f16"),
        # a single layer of 2049 cached rows: the smallest step, where latency counts
        dict(name="decode_one", op="decode", n=1, q_heads=64, kv_heads=8, cap=2049, lo=2049, hi=2049, window=0,
             io="f32", append=False),
        # 48 layers at 32K context, the step's own rows quantised on the way
        dict(name="decode_layers", op="decode", n=48, q_heads=64, kv_heads=8, cap=32769, lo=32769, hi=32769, window=0,
             io="f32", append=True),
        # a ragged serving batch of one layer
        dict(name="decode_batch", op="decode", n=64, q_heads=64, kv_heads=8, cap=8192, lo=1, hi=8192, window=0,
             io="bf16", append=True),
        # a batch on a sliding-window layer (96 query heads, 12 for each KV head)
        dict(name="decode_sliding", op="decode", n=128, q_heads=96, kv_heads=8, cap=768, lo=40, hi=5000, window=512,
             io="bf16", append=True),
        # one sequence at 131072 tokens
        dict(name="decode_long", op="decode", n=1, q_heads=64, kv_heads=8, cap=131072, lo=131072, hi=131072, window=0,
             io="bf16", append=False),
        # a few requests with a short system prompt
        dict(name="shared_small", op="shared", n=4, q_heads=64, kv_heads=8, prefix=512, cap=64, lo=1, hi=64, window=0,
             io="bf16", cache="f16", append=False),
        # requests over one document, ragged answers
        dict(name="shared_chat", op="shared", n=32, q_heads=64, kv_heads=8, prefix=8192, cap=1024, lo=1, hi=1024,
             window=0, io="bf16", cache="f16", append=True),
        # a large batch over a long shared context, own rows in int8
        dict(name="shared_long", op="shared", n=64, q_heads=64, kv_heads=8, prefix=32768, cap=2048, lo=1, hi=2048,
             window=0, io="bf16", cache="i8", append=True),
        # full-precision queries and outputs, 12 heads a group, an odd prefix partly outside the window
        dict(name="shared_f32", op="shared", n=9, q_heads=96, kv_heads=8, prefix=4097, cap=700, lo=1, hi=700,
             window=4000, io="f32", cache="f16", append=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "decode", "decode", "shared", "shared"])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 8])
    group = rng.choice([1, 4, 5, 8, 8, 12, 16])
    io = rng.choice(["f32", "bf16", "bf16"])
    if op == "store":
        n, n_tok = rng.choice([1, 2, 7, 48]), _log(rng, 1, 4096)
        cap = max(n_tok, _log(rng, 16, 16384)) + rng.choice([0, 0, 1, 3])
        n = max(1, min(n, 60000 // cap))
        pos0 = _log(rng, 1, 40000) - 1
        end = pos0 + n_tok
        rows = min(cap, end, _log(rng, n_tok, max(n_tok, cap)))
        return dict(op=op, n=n, kv_heads=kv_heads, cap=cap, pos0=pos0, n_tok=n_tok, first=end - rows, rows=rows,
                    io=io, dst=rng.choice(["f16", "f32"]))
    if op == "decode":
        n, hi = _log(rng, 1, 160), _log(rng, 1, 40000)
        n = max(1, min(n, 1000000 // hi, 100000000 // (group * kv_heads * hi)))
        window = rng.choice([0, 0, 0, 512])
        cap = hi if not window else min(hi, window + rng.choice([0, 1, 256])) + rng.choice([0, 0, 5])
        return dict(op=op, n=n, q_heads=group * kv_heads, kv_heads=kv_heads, cap=cap, lo=rng.choice([1, hi]), hi=hi,
                    window=window, io=io, append=rng.choice([False, True]))
    n, prefix, hi = _log(rng, 1, 96), _log(rng, 16, 24000), _log(rng, 1, 1500)
    n = max(1, min(n, 130000000 // (group * kv_heads * (prefix + hi))))
    window = rng.choice([0, 0, 0, hi + prefix // 2])
    return dict(op=op, n=n, q_heads=group * kv_heads, kv_heads=kv_heads, prefix=prefix, cap=hi + rng.choice([0, 0, 7]),
                lo=rng.choice([1, hi]), hi=hi, window=window, io=io, cache=rng.choice(["f16", "f16", "i8"]),
                append=rng.choice([False, True]))


# ------------------------------------------------------------------ inputs

def _layout(cap, heads):
    """(bytes of the codes, bytes in all) of one int8 cache of K or V; caches lie 256 bytes apart."""
    codes = cap * heads * D
    return codes, (codes + 4 * heads * cap + 255) // 256 * 256


def _views(raw, cap, heads):
    """Codes [n, cap, heads, 128] and scales [n, heads, cap] of n int8 caches held as bytes [n, ...]."""
    codes = cap * heads * D
    return (raw[:, :codes].view(-1, cap, heads, D),
            raw[:, codes:codes + 4 * heads * cap].view(torch.float32).view(-1, heads, cap))


def _quantise(x):
    """Bytes c + 128 and scales of the heads of x [..., 128]."""
    x = x.float()
    a = x.abs().amax(-1)
    s = (a.double() / 127).float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    bad = ~torch.isfinite(x).all(-1)
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    live = (s > 0).unsqueeze(-1)
    c = torch.where(live, x.double() / s.double().unsqueeze(-1), 0.0).round().clamp(-127, 127)
    return (c + 128).to(torch.uint8), s


def _keys(g, *shape):
    """Rows with a few large channels, as keys have them."""
    x = torch.randn(*shape, D, device="cuda", generator=g)
    x[..., 5::32] *= 4
    return x


def _i8_caches(g, n, cap, heads):
    raw = []
    for make in (_keys, lambda g, *s: torch.randn(*s, D, device="cuda", generator=g)):
        r = torch.zeros(n, _layout(cap, heads)[1], dtype=torch.uint8, device="cuda")
        codes, scales = _views(r, cap, heads)
        for i in range(n):
            c, s = _quantise(make(g, cap, heads))
            codes[i], scales[i] = c, s.t()
        raw.append(r)
    return raw


def _tensors(case, seed):
    """The case's inputs by name, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, heads, cap, io = case["n"], case["kv_heads"], case["cap"], TYPES[case["io"]]
    s = {}
    if case["op"] == "store":
        s["k_cache"], s["v_cache"] = _i8_caches(g, n, cap, heads)
        s["k"] = _keys(g, n, case["n_tok"], heads).to(io)
        s["v"] = torch.randn(n, case["n_tok"], heads, D, device="cuda", generator=g).to(io)
        for name in ("dst_k", "dst_v"):
            s[name] = torch.zeros(n, case["rows"], heads, D, device="cuda", dtype=TYPES[case["dst"]])
        return s
    if case.get("cache", "i8") == "i8":
        s["k_cache"], s["v_cache"] = _i8_caches(g, n, cap, heads)
    else:
        s["k_cache"] = _keys(g, n, cap, heads).half()
        s["v_cache"] = torch.randn(n, cap, heads, D, device="cuda", generator=g).half()
    if case["op"] == "shared":
        s["prefix_k"] = _keys(g, case["prefix"], heads).half()
        s["prefix_v"] = torch.randn(case["prefix"], heads, D, device="cuda", generator=g).half()
    s["q"] = (1.5 * torch.randn(n, case["q_heads"], D, device="cuda", generator=g)).to(io)
    s["gate"] = torch.randn(n, case["q_heads"], device="cuda", generator=g)
    s["out"] = torch.empty_like(s["q"])
    if case["append"]:
        s["k_new"] = _keys(g, n, heads).to(io)
        s["v_new"] = torch.randn(n, heads, D, device="cuda", generator=g).to(io)
        for name in ("row_k", "row_v"):  # the appended rows, read back
            s[name] = torch.zeros(n, 1, heads, D, device="cuda")
    return s


def _positions(case, seed):
    """Every sequence's position: own lengths spread evenly over [lo, hi], in an order that the seed gives."""
    lens = np.linspace(case["lo"], case["hi"], case["n"]).round().astype(np.int64)
    lens[-1] = case["hi"]
    np.random.RandomState(seed % (1 << 31)).shuffle(lens)
    return lens - 1 + case.get("prefix", 0)


def prepare(case, seed):
    s = _tensors(case, seed)
    s["case"] = case
    if case["op"] != "store":
        s["pos_host"] = _positions(case, seed)
        s["pos"] = torch.from_numpy(s["pos_host"]).cuda()
        s["seq"] = torch.arange(case["n"], device="cuda")
    if own:
        _plan(s)
    return s


# ------------------------------------------------------------------ the framework's calls

def _plan(s):
    """The descriptor arrays and the workspace that a decode loop keeps from step to step."""
    from sf37_b200 import kv

    c = s["case"]
    if c["op"] == "store":
        s["append"] = kv.append_i8_desc(s["k_cache"], s["v_cache"], c["cap"], c["pos0"], s["k"], s["v"])
        s["read"] = kv.read_i8_desc(s["k_cache"], s["v_cache"], c["cap"], s["dst_k"], s["dst_v"], c["rows"],
                                    c["first"], c["rows"])
        return
    s["seqs"] = kv.decode_seqs_desc(s["k_cache"], s["v_cache"], c["cap"], s["pos_host"], s["q"], s["out"],
                                    gate=s["gate"], k_new=s.get("k_new"), v_new=s.get("v_new"),
                                    sliding=c["window"] > 0, window=c["window"])
    if c["append"] and c.get("cache", "i8") == "i8":
        s["read"] = kv.read_i8_desc(s["k_cache"], s["v_cache"], c["cap"], s["row_k"], s["row_v"], 1, s["pos_host"], 1)
    if c["op"] == "shared":
        s["groups"] = kv.shared_groups_desc([dict(k_cache=s["prefix_k"], v_cache=s["prefix_v"], prefix_len=c["prefix"],
                                                  seqs=s["seqs"])])
        size = kv.decode_shared_workspace(1, c["n"], c["q_heads"], c["kv_heads"])
    else:
        size = kv.decode_i8_workspace(c["n"], c["q_heads"], c["kv_heads"])
    s["workspace"] = torch.zeros(size, dtype=torch.uint8, device="cuda")


def _run_own(s):
    from sf37_b200 import kv

    c = s["case"]
    if c["op"] == "store":
        kv.append_i8(s["append"], c["kv_heads"], D, s["k"].dtype)
        kv.read_i8(s["read"], c["kv_heads"], D, s["dst_k"].dtype)
        return {"k": s["dst_k"], "v": s["dst_v"]}
    s["seqs"]["pos"] = s["pos_host"]  # a decode loop writes the step's positions
    if c["op"] == "shared":
        kv.decode_shared(s["groups"], c["q_heads"], c["kv_heads"], D, kv.I8 if c["cache"] == "i8" else kv.F16,
                         s["q"].dtype, s["workspace"])
    else:
        kv.decode_i8(s["seqs"], c["q_heads"], c["kv_heads"], D, s["q"].dtype, s["workspace"])
    if not c["append"]:
        return {"out": s["out"]}
    if c.get("cache", "i8") == "i8":
        kv.read_i8(s["read"], c["kv_heads"], D, torch.float32)
        return {"out": s["out"], "k": s["row_k"], "v": s["row_v"]}
    slot = s["pos"] % c["cap"]
    return {"out": s["out"], "k": s["k_cache"][s["seq"], slot], "v": s["v_cache"][s["seq"], slot]}


# ------------------------------------------------------------------ the plain form

def _values(raw, cap, heads):
    codes, scales = _views(raw, cap, heads)
    return (codes.float() - 128) * scales.transpose(1, 2).unsqueeze(-1)


def _store_plain(s):
    c = s["case"]
    at = torch.arange(c["n_tok"], device="cuda")[-c["cap"]:]
    slot = (c["pos0"] + at) % c["cap"]
    back = (c["first"] + torch.arange(c["rows"], device="cuda"))
    out = {}
    for name in ("k", "v"):
        codes, scales = _views(s[name + "_cache"], c["cap"], c["kv_heads"])
        q, sc = _quantise(s[name][:, at])
        codes[:, slot] = q
        scales[:, :, slot] = sc.transpose(1, 2)
        src, dst = back % c["cap"], s["dst_" + name]
        x = (codes[:, src].float() - 128) * scales[:, :, src].transpose(1, 2).unsqueeze(-1)
        dst[:, back % c["rows"]] = x.to(dst.dtype)
        out[name] = dst
    return out


def _attention_plain(s):
    c = s["case"]
    n, heads, cap = c["n"], c["kv_heads"], c["cap"]
    i8, pos, prefix = c.get("cache", "i8") == "i8", s["pos"], c.get("prefix", 0)
    slot, out = pos % cap, {}
    if c["append"]:
        for name in ("k", "v"):
            new = s[name + "_new"]
            if i8:
                codes, scales = _views(s[name + "_cache"], cap, heads)
                q, sc = _quantise(new)
                codes[s["seq"], slot], scales[s["seq"], :, slot] = q, sc
                out[name] = ((q.float() - 128) * sc.unsqueeze(-1)).unsqueeze(1)
            else:
                s[name + "_cache"][s["seq"], slot] = new.half()
                out[name] = s[name + "_cache"][s["seq"], slot]
    k, v = ((_values(s[x], cap, heads) if i8 else s[x].float()) for x in ("k_cache", "v_cache"))
    q = s["q"].float().view(n, heads, -1, D) / math.sqrt(D)
    held = pos[:, None] - (pos[:, None] - torch.arange(cap, device="cuda")) % cap  # the position in each slot
    first = torch.clamp(pos + 1 - c["window"], min=0) if c["window"] else torch.zeros_like(pos)
    live = (held >= torch.clamp(first, min=prefix)[:, None])[:, None, None]
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).masked_fill_(~live, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if prefix:
        pk, pv = s["prefix_k"].float().permute(1, 2, 0), s["prefix_v"].float().permute(1, 0, 2)
        rows = q.transpose(0, 1).reshape(heads, -1, D)
        ps = torch.matmul(rows, pk).view(heads, n, -1, prefix)
        seen = (torch.arange(prefix, device="cuda") >= first[:, None])[None, :, None]
        ps.masked_fill_(~seen, -math.inf)
        top = torch.maximum(top, ps.amax(-1).permute(1, 0, 2).unsqueeze(-1))
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.transpose(1, 2))
    if prefix:
        pp = torch.exp(ps - top.squeeze(-1).permute(1, 0, 2).unsqueeze(-1))
        total = total + pp.sum(-1).permute(1, 0, 2).unsqueeze(-1)
        o = o + torch.matmul(pp.view(heads, -1, prefix), pv).view(heads, n, -1, D).transpose(0, 1)
    gate = 1 / (1 + torch.exp(-s["gate"]))
    o = (o / total).view(n, -1, D) * gate.unsqueeze(-1)
    return {"out": o.to(s["q"].dtype), **out}


def run(state):
    if own:
        return _run_own(state)
    return _store_plain(state) if state["case"]["op"] == "store" else _attention_plain(state)


# ------------------------------------------------------------------ the work, and the values in 64 bits

def _rows(case):
    """Own rows attended to by each sequence, and prefix rows seen by each."""
    pos, prefix = _positions(case, 0), case.get("prefix", 0)
    first = np.maximum(pos + 1 - case["window"], 0) if case["window"] else np.zeros_like(pos)
    first = np.maximum(first, 0 if prefix else pos + 1 - case["cap"])
    return pos + 1 - np.maximum(first, prefix), np.maximum(prefix - first, 0)


def work(case):
    heads, size = case["kv_heads"], 4 if case["io"] == "f32" else 2
    i8_row = 2 * heads * (D + 4)
    if case["op"] == "store":
        dst = 4 if case["dst"] == "f32" else 2
        written = min(case["n_tok"], case["cap"])
        return {"bytes": case["n"] * (written * (2 * heads * D * size + i8_row) + case["rows"] * (i8_row + 2 * heads * D * dst)),
                "flops": case["n"] * 2 * heads * D * (4 * written + case["rows"])}
    rows, shared = _rows(case)
    row = i8_row if case.get("cache", "i8") == "i8" else 4 * heads * D
    total = int(rows.sum()) * row + int(shared.max()) * 4 * heads * D
    total += case["n"] * (2 * case["q_heads"] * D * size + 4 * case["q_heads"])
    if case["append"]:
        total += case["n"] * (2 * heads * D * size + row)
    return {"bytes": total, "flops": 4 * D * case["q_heads"] * int(rows.sum() + shared.sum())}


def _code_exact(x):
    """The values that a written head stands for: the scale is the f32 nearest max/127, the code the nearest integer."""
    x = x.double()
    s = (x.abs().amax(-1, keepdim=True) / 127).float().double()
    return torch.where(s >= 2.0 ** -126, torch.round(x / torch.where(s > 0, s, 1.0)) * s, 0.0)


def exact(case, seed):
    s = _tensors(case, seed)
    n, heads, cap = case["n"], case["kv_heads"], case["cap"]
    i8, out = case.get("cache", "i8") == "i8", {}

    def cached(name, i, slots):
        if not i8:
            return s[name + "_cache"][i][slots].double()
        codes, scales = _views(s[name + "_cache"][i:i + 1], cap, heads)
        return (codes[0][slots].double() - 128) * scales[0].t()[slots].double().unsqueeze(-1)

    if case["op"] == "store":
        for name in ("k", "v"):
            rows = torch.arange(case["first"], case["first"] + case["rows"], device="cuda")
            new = rows >= case["pos0"]
            new &= rows < case["pos0"] + case["n_tok"]
            got = torch.zeros(n, case["rows"], heads, D, dtype=torch.float64, device="cuda")
            for i in range(n):
                x = cached(name, i, rows % cap)
                x[new] = _code_exact(s[name][i, rows[new] - case["pos0"]])
                got[i, rows % case["rows"]] = x
            out[name] = got
        return out
    o = torch.zeros(n, case["q_heads"], D, dtype=torch.float64, device="cuda")
    back = {name: torch.zeros(n, 1, heads, D, dtype=torch.float64, device="cuda") for name in ("k", "v")}
    prefix = case.get("prefix", 0)
    for i, p in enumerate(_positions(case, seed).tolist()):
        first = max(0, p + 1 - case["window"]) if case["window"] else 0
        if not prefix:
            first = max(first, p + 1 - cap)
        rows = torch.arange(max(first, prefix), p + 1, device="cuda")
        kv = {}
        for name in ("k", "v"):
            x = cached(name, i, rows % cap)
            if case["append"]:
                new = s[name + "_new"][i]
                x[-1] = _code_exact(new) if i8 else new.half().double()
                back[name][i, 0] = x[-1]
            if first < prefix:
                x = torch.cat([s["prefix_" + name][first:].double(), x])
            kv[name] = x
        q = s["q"][i].double().view(heads, -1, D)
        w = torch.softmax(torch.einsum("hgd,rhd->hgr", q, kv["k"]) / math.sqrt(D), -1)
        gate = torch.sigmoid(s["gate"][i].double()).unsqueeze(-1)
        o[i] = torch.einsum("hgr,rhd->hgd", w, kv["v"]).reshape(-1, D) * gate
    out["out"] = o
    if case["append"]:
        for name in ("k", "v"):
            out[name] = back[name] if i8 else back[name][:, 0]
    return out
