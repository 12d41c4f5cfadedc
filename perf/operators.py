"""The operators of a decoding step over a paged key / value cache, as cases to be timed and checked.

Four operators that a decoder needs beside its projections: the rotation of queries and keys by their positions,
the write of new keys and values into a paged cache, attention of the new tokens over that cache, and the products of
a few rows with 4-bit weights.  With `own` false `run` computes them from elementary torch operations, with `own` true
through modules compiled by this package.  All lengths of a case follow from its numbers (`mix` seeds them), all
values from the seed."""
import functools
import math
import random

import torch

own = False

_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one new token of one conversation: the queries of a layer
        dict(name="rope_token", op="rope", tokens=1, heads=32, dim=128, rotary=128, interleaved=False, stretch=1.0, far=100000, dtype="f16"),
        # a prompt chunk at far positions, frequencies stretched for a longer context
        dict(name="rope_prompt", op="rope", tokens=8192, heads=32, dim=128, rotary=128, interleaved=False, stretch=8.0, far=1000000, dtype="bf16"),
        # odd token count, neighbouring pairs, a quarter of a 12-head decoder's head rotated, full precision
        dict(name="rope_partial", op="rope", tokens=997, heads=12, dim=64, rotary=16, interleaved=True, stretch=1.0, far=4096, dtype="f32"),
        # one token each of 48 conversations into pages of 16
        dict(name="append_tokens", op="append", seqs=48, new_min=1, new_max=1, ctx_max=4096, kv_heads=8, dim=128, page=16, rotate=True, dtype="f16", mix=11),
        # ragged prompts into pages of 64
        dict(name="append_prompts", op="append", seqs=9, new_min=333, new_max=2048, ctx_max=4096, kv_heads=8, dim=128, page=64, rotate=True, dtype="bf16", mix=12),
        # single-token decoding of a 12-head decoder, batch 4, up to 512 keys: latency
        dict(name="decode_small", op="attention", seqs=4, new_min=1, new_max=1, ctx_min=100, ctx_max=512, heads=12, kv_heads=12, dim=64, page=16, window=0, dtype="f16", mix=21),
        # single-token decoding of 32 conversations of uneven length, grouped heads
        dict(name="decode_batch", op="attention", seqs=32, new_min=1, new_max=1, ctx_min=200, ctx_max=8191, heads=32, kv_heads=8, dim=128, page=16, window=0, dtype="bf16", mix=22),
        # one long context, one token
        dict(name="decode_long", op="attention", seqs=1, new_min=1, new_max=1, ctx_min=131071, ctx_max=131071, heads=32, kv_heads=8, dim=128, page=32, window=0, dtype="f16", mix=23),
        # prompt chunks of five conversations over what is cached already
        dict(name="chunk_prompts", op="attention", seqs=5, new_min=515, new_max=2048, ctx_min=2048, ctx_max=12000, heads=32, kv_heads=8, dim=128, page=16, window=0, dtype="bf16", mix=24),
        # one layer's projection for one token, groups of 128, symmetric
        dict(name="w4_token", op="w4", rows=1, n=4096, k=4096, group=128, zeros=False, dtype="f16"),
        # the wide projection with zero points and small groups, odd column count
        dict(name="w4_wide", op="w4", rows=3, n=14337, k=4096, group=32, zeros=True, dtype="bf16"),
        # sixteen conversations at once through the narrow projection
        dict(name="w4_batch", op="w4", rows=16, n=4096, k=14336, group=64, zeros=True, dtype="f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention", "w4"])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128])
        return dict(op=op, tokens=_log_int(rng, 1, 8192), heads=rng.randint(1, 32), dim=dim, rotary=rng.choice([dim // 4 // 2 * 2, dim // 2, dim]), interleaved=rng.random() < 0.5,
                    stretch=rng.choice([1.0, 4.0, 8.0]), far=_log_int(rng, 64, 1000000), dtype=rng.choice(["f16", "bf16", "f32"]))
    if op == "append":
        single = rng.random() < 0.5
        new_max = 1 if single else _log_int(rng, 2, 2048)
        return dict(op=op, seqs=rng.randint(1, 64) if single else rng.randint(1, 9), new_min=0 if rng.random() < 0.3 else 1, new_max=new_max, ctx_max=new_max + _log_int(rng, 1, 4096),
                    kv_heads=rng.randint(1, 12), dim=rng.choice([64, 80, 96, 128]), page=rng.choice([8, 16, 32, 64]), rotate=rng.random() < 0.7,
                    dtype=rng.choice(["f16", "bf16", "f32"]), mix=rng.randrange(1 << 30))
    if op == "attention":
        kv_heads, ratio = rng.choice([(12, 1), (8, 4), (4, 8), (2, 7), (1, 16), (5, 3)])
        dim = rng.choice([64, 80, 96, 128])
        window = rng.choice([0, 0, 0, 100, 1024])
        if rng.random() < 0.5:
            ctx = _log_int(rng, 1, 16384)
            seqs = rng.randint(1, max(1, min(64, 262144 // ctx)))
            return dict(op=op, seqs=seqs, new_min=1, new_max=1, ctx_min=max(1, ctx // 8), ctx_max=ctx, heads=kv_heads * ratio, kv_heads=kv_heads, dim=dim,
                        page=rng.choice([8, 16, 32, 64]), window=window, dtype=rng.choice(["f16", "bf16"]), mix=rng.randrange(1 << 30))
        new = _log_int(rng, 2, 2048)
        return dict(op=op, seqs=rng.randint(1, 3), new_min=rng.choice([0, 1, new]), new_max=new, ctx_min=new, ctx_max=new + _log_int(rng, 1, 6144), heads=kv_heads * ratio,
                    kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 32, 64]), window=window, dtype=rng.choice(["f16", "bf16"]), mix=rng.randrange(1 << 30))
    group = rng.choice([32, 64, 128])
    return dict(op=op, rows=rng.choice([1, 1, 2, 3, 4, 7, 8, 16]), n=_log_int(rng, 100, 14336), k=128 * _log_int(rng, 1, 112), group=group, zeros=rng.random() < 0.5,
                dtype=rng.choice(["f16", "bf16"]))


def _lengths(case):
    """(new tokens, keys) of every sequence; the keys include the new tokens.  At least one token in all."""
    rng = random.Random(case["mix"])
    new = [rng.randint(case["new_min"], case["new_max"]) for _ in range(case["seqs"])]
    if sum(new) == 0:
        new[0] = 1
    low = case.get("ctx_min", 1)
    ctx = [rng.randint(max(n, min(low, case["ctx_max"])), case["ctx_max"]) for n in new]
    return new, ctx


def _pairs_seen(n, c, window):
    """Query / key pairs of n tokens that end a sequence of c keys."""
    if not window:
        return n * (c - n) + n * (n + 1) // 2
    return sum(min(window, p + 1) for p in range(c - n, c))


def work(case):
    es = _BYTES[case["dtype"]]
    if case["op"] == "rope":
        e = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * e * es + 4 * case["tokens"] + 2 * case["rotary"], "flops": 3 * case["tokens"] * case["heads"] * case["rotary"]}
    if case["op"] == "append":
        new, _ = _lengths(case)
        e = sum(new) * case["kv_heads"] * case["dim"]
        return {"bytes": 4 * e * es, "flops": 3 * e if case["rotate"] else 0}
    if case["op"] == "attention":
        new, ctx = _lengths(case)
        w = case["window"]
        keys = sum((min(c, n - 1 + w) if w else c) for n, c in zip(new, ctx) if n > 0)
        pairs = sum(_pairs_seen(n, c, w) for n, c in zip(new, ctx))
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * es + 2 * sum(new) * case["heads"] * case["dim"] * es, "flops": 4 * pairs * case["heads"] * case["dim"]}
    m, n, k = case["rows"], case["n"], case["k"]
    groups = k // case["group"]
    return {"bytes": n * k // 2 + n * groups * es + (n * groups if case["zeros"] else 0) + (m * k + m * n) * es, "flops": 2 * m * n * k}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _frequencies(rotary, stretch):
    """f32 angle per position of every rotated pair; a stretched context slows the low frequencies down, keeps the high ones and blends between."""
    i = torch.arange(0, rotary // 2, dtype=torch.float64)
    f = 10000.0 ** (-2.0 * i / rotary)
    turns = 4096.0 * f / (2.0 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return (f * (keep + (1.0 - keep) / stretch)).to(torch.float32)


def _amplitude(stretch):
    return 1.0 if stretch == 1.0 else 0.1 * math.log(stretch) + 1.0


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(1000003 * seed + 17)

    def normal(*dims):
        return torch.randn(dims, generator=g, device=dev, dtype=torch.float32).to(_TORCH[case["dtype"]])

    if case["op"] == "rope":
        pos = torch.randint(0, case["far"], (case["tokens"],), generator=g, device=dev, dtype=torch.int32)
        return dict(x=normal(case["tokens"], case["heads"], case["dim"]), positions=pos, inv_freq=_frequencies(case["rotary"], case["stretch"]).to(dev))
    if case["op"] == "w4":
        n, k, groups = case["n"], case["k"], case["k"] // case["group"]
        weight = torch.randint(0, 256, (n, k // 2), generator=g, device=dev, dtype=torch.uint8)
        scales = ((0.5 + torch.rand((n, groups), generator=g, device=dev)) * (0.2 / math.sqrt(k))).to(_TORCH[case["dtype"]])
        zeros = torch.randint(5, 11, (n, groups), generator=g, device=dev, dtype=torch.uint8) if case["zeros"] else None
        return dict(x=normal(case["rows"], k), weight=weight, scales=scales, zeros=zeros)
    new, ctx = _lengths(case)
    page = case["page"]
    width = max(1, (max(ctx) + page - 1) // page)
    used = [(c + page - 1) // page for c in ctx]
    pool = sum(used) + 3
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    start = torch.zeros(case["seqs"] + 1, dtype=torch.int32)
    start[1:] = torch.cumsum(torch.tensor(new), 0)
    s = dict(page_table=table, query_start=start.to(dev), context_len=torch.tensor(ctx, dtype=torch.int32, device=dev), new=new, ctx=ctx)
    s["k_cache"] = normal(pool, page, case["kv_heads"], case["dim"])
    s["v_cache"] = normal(pool, page, case["kv_heads"], case["dim"])
    if case["op"] == "append":
        s["k"] = normal(sum(new), case["kv_heads"], case["dim"])
        s["v"] = normal(sum(new), case["kv_heads"], case["dim"])
        s["inv_freq"] = _frequencies(case["dim"], 1.0).to(dev) if case["rotate"] else None
    else:
        s["q"] = normal(sum(new), case["heads"], case["dim"])
    return s


# ---- this package's operators ---------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _function(op, dtype, dims, options):
    """A loaded module that holds one operator: what a program compiles once for the shapes it serves."""
    from mononn_amd import MonoNNModule
    from mononn_amd.hlo.builder import HloModuleBuilder
    from mononn_amd.torch_op import MonoNNFunction
    mb = HloModuleBuilder("cluster_0__" + op)
    e = mb.entry
    o = dict(options)
    args = {name: e.parameter(t, d, name) for name, t, d in dims}
    if op == "rope":
        out = [e.rope(args["x"], args["positions"], args["inv_freq"], interleaved=o["interleaved"], amplitude=o["amplitude"])]
    elif op == "append":
        out = list(e.kv_append(args["k"], args["v"], args["k_cache"], args["v_cache"], args["page_table"], args["query_start"], args["context_len"], inv_freq=args.get("inv_freq")))
    elif op == "attention":
        out = [e.paged_attention(args["q"], args["k_cache"], args["v_cache"], args["page_table"], args["query_start"], args["context_len"], scale=o["scale"], window=o["window"])]
    else:
        out = [e.matvec_w4(args["x"], args["weight"], args["scales"], args.get("zeros"))]
    e.set_tuple_root(out)
    module = MonoNNModule.compile(mb.text())
    module.load(0)
    return MonoNNFunction(module, [{"dtype": v.dtype, "dims": list(v.dims)} for v in out])


_HLO = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32", torch.int32: "s32", torch.uint8: "u8"}
_ARGUMENTS = {"rope": ("x", "positions", "inv_freq"), "append": ("k", "v", "k_cache", "v_cache", "page_table", "query_start", "context_len", "inv_freq"),
              "attention": ("q", "k_cache", "v_cache", "page_table", "query_start", "context_len"), "w4": ("x", "weight", "scales", "zeros")}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        tensors = [(a, s[a]) for a in _ARGUMENTS[case["op"]] if s[a] is not None]
        options = {"rope": lambda: (("interleaved", case["interleaved"]), ("amplitude", _amplitude(case["stretch"]))), "append": lambda: (), "w4": lambda: (),
                   "attention": lambda: (("scale", 1.0 / math.sqrt(case["dim"])), ("window", case["window"]))}[case["op"]]()
        s["call"] = _function(case["op"], case["dtype"], tuple((a, _HLO[t.dtype], tuple(t.shape)) for a, t in tensors), options)
        s["args"] = [t for _, t in tensors]
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _rotate(x, positions, inv_freq, interleaved, amplitude):
    angle = positions.double()[:, None] * inv_freq.double()[None, :]      # 64 bits: far positions
    c, s = (torch.cos(angle) * amplitude).float()[:, None, :], (torch.sin(angle) * amplitude).float()[:, None, :]
    r = 2 * inv_freq.numel()
    x = x.float()
    head, rest = x[..., :r], x[..., r:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = head[..., :r // 2], head[..., r // 2:]
        turned = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_append(s):
    positions = torch.cat([torch.arange(c - n, c, device=s["k"].device) for n, c in zip(s["new"], s["ctx"])])
    seq = torch.repeat_interleave(torch.arange(len(s["new"]), device=positions.device), torch.tensor(s["new"], device=positions.device), output_size=len(positions))
    page = s["k_cache"].shape[1]
    where = (s["page_table"][seq, positions // page].long(), positions % page)
    k = s["k"] if s["inv_freq"] is None else _rotate(s["k"], positions, s["inv_freq"], False, 1.0).to(s["k"].dtype)
    s["k_cache"][where] = k
    s["v_cache"][where] = s["v"]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    case, out, at = s["case"], [], 0
    ratio = case["heads"] // case["kv_heads"]
    for b, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        if n == 0:
            continue
        pages = s["page_table"][b, :(c + case["page"] - 1) // case["page"]].long()
        k = s["k_cache"][pages].flatten(0, 1)[:c].float().permute(1, 2, 0).contiguous()       # kv head, dim, key
        v = s["v_cache"][pages].flatten(0, 1)[:c].float().permute(1, 0, 2).contiguous()       # kv head, key, dim
        q = s["q"][at:at + n].float().view(n, case["kv_heads"], ratio, case["dim"]).permute(1, 2, 0, 3).reshape(case["kv_heads"], ratio * n, case["dim"])
        score = torch.matmul(q, k).view(case["kv_heads"], ratio, n, c) * (1.0 / math.sqrt(case["dim"]))
        key, query = torch.arange(c, device=q.device), torch.arange(c - n, c, device=q.device)[:, None]
        hidden = key > query
        if case["window"]:
            hidden = hidden | (key <= query - case["window"])
        score = score.masked_fill(hidden, float("-inf"))
        weight = torch.exp(score - score.amax(-1, keepdim=True))
        o = torch.matmul((weight / weight.sum(-1, keepdim=True)).view(case["kv_heads"], ratio * n, c), v)
        out.append(o.view(case["heads"], n, case["dim"]).permute(1, 0, 2).to(s["q"].dtype))
        at += n
    return torch.cat(out)


def _unpack(weight):
    return torch.stack((weight & 15, weight >> 4), dim=-1).flatten(1)     # the low half of a byte is the lower column


def run(state):
    case = state["case"]
    if own:
        out = state["call"](*state["args"])
        return {"k_cache": out[0], "v_cache": out[1]} if case["op"] == "append" else out[0]
    if case["op"] == "rope":
        return _rotate(state["x"], state["positions"], state["inv_freq"], case["interleaved"], _amplitude(case["stretch"])).to(state["x"].dtype)
    if case["op"] == "append":
        return _plain_append(state)
    if case["op"] == "attention":
        return _plain_attention(state)
    n, k = case["n"], case["k"]
    q = _unpack(state["weight"]).float().view(n, -1, case["group"])
    zero = state["zeros"].float()[:, :, None] if state["zeros"] is not None else 8.0
    w = ((q - zero) * state["scales"].float()[:, :, None]).view(n, k)
    return torch.matmul(state["x"].float(), w.t()).to(state["x"].dtype)


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------
def _turn64(x, positions, inv_freq, interleaved, amplitude):
    y = x.double().clone()
    half = inv_freq.numel()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = positions.double() * inv_freq[i].double()
        c, s = amplitude * torch.cos(angle)[:, None], amplitude * torch.sin(angle)[:, None]
        y[:, :, a] = x[:, :, a].double() * c - x[:, :, b].double() * s
        y[:, :, b] = x[:, :, a].double() * s + x[:, :, b].double() * c
    return y


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rope":
        return _turn64(s["x"], s["positions"], s["inv_freq"], case["interleaved"], _amplitude(case["stretch"]))
    if case["op"] == "w4":
        x = s["x"].double()
        out = torch.zeros((case["rows"], case["n"]), dtype=torch.float64, device=x.device)
        for g in range(case["k"] // case["group"]):
            cols = slice(g * case["group"] // 2, (g + 1) * case["group"] // 2)
            zero = s["zeros"][:, g].double()[:, None] if s["zeros"] is not None else 8.0
            scale = s["scales"][:, g].double()
            xs = x[:, g * case["group"]:(g + 1) * case["group"]]
            low, high = (s["weight"][:, cols] & 15).double() - zero, (s["weight"][:, cols] >> 4).double() - zero
            out += (xs[:, 0::2] @ low.t().contiguous() + xs[:, 1::2] @ high.t().contiguous()) * scale
        return out
    page = case["page"]
    if case["op"] == "append":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        at = 0
        for b, (n, c) in enumerate(zip(s["new"], s["ctx"])):
            if n == 0:
                continue
            p = torch.arange(c - n, c, device=kc.device)
            k = s["k"][at:at + n]
            rows = s["page_table"][b].long()[p // page] * page + p % page
            kc.view(-1, case["kv_heads"], case["dim"])[rows] = _turn64(k, p, s["inv_freq"], False, 1.0) if case["rotate"] else k.double()
            vc.view(-1, case["kv_heads"], case["dim"])[rows] = s["v"][at:at + n].double()
            at += n
        return {"k_cache": kc, "v_cache": vc}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    at = 0
    for b, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        if n == 0:
            continue
        p = torch.arange(c, device=out.device)
        rows = s["page_table"][b].long()[p // page] * page + p % page
        behind = torch.arange(c - n, c, device=out.device)[:, None] - p        # how far a key lies behind the query
        seen = behind >= 0
        if case["window"]:
            seen &= behind < case["window"]
        for h in range(case["heads"]):
            kv = h * case["kv_heads"] // case["heads"]
            k = s["k_cache"].view(-1, case["kv_heads"], case["dim"])[rows, kv].double()
            v = s["v_cache"].view(-1, case["kv_heads"], case["dim"])[rows, kv].double()
            score = (s["q"][at:at + n, h].double() @ k.t().contiguous()) / math.sqrt(case["dim"])
            score = torch.where(seen, score, torch.full_like(score, -math.inf))
            e = torch.exp(score - score.max(dim=1, keepdim=True).values)
            out[at:at + n, h] = (e @ v) / e.sum(dim=1, keepdim=True)
        at += n
    return out
