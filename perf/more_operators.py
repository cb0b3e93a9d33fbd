"""Performance cases of a serving step around an 8-bit paged KV cache.

  rotary  Runtime.cache_append_rotary: new K and V rows into the 16-bit cache's
          pages, Q and K normalised per head and rotated on the way
  append  Runtime.cache8_append: the same into pages of 8-bit codes with a
          power-of-two scale for every 16 positions of a head
  attend  Runtime.tree_attention8: a token, or a tree of up to 64 drafted
          tokens, per sequence over the 8-bit pages
  keep    Runtime.cache8_keep: the accepted nodes of each draft to the front of
          the draft, in every layer, with the scales of the blocks they reach
  sample  Runtime.sample: the next token of every row from its logits by
          temperature, top-k, top-p and min-p, from a given random number

Head counts and sizes are those of the framework's qwen3 presets (16 query and
8 kv heads, 32 and 8, head size 128, 151936 tokens) and generic ones.

An 8-bit page holds kv_heads * page * d codes (e4m3), then kv_heads * page / 16
scale bytes (2 to the power byte - 127), and is padded to 128 bytes.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LAYERS = 28  # of the qwen3-0.6b preset
BLOCK = 16   # positions that share a scale
LEAST = 27   # the smallest scale byte, 2^-100
EPS = 1e-6
FP8 = torch.float8_e4m3fn


def listed():
    return [
        # a decode step's rows of a serving batch
        {"name": "rotary_step", "kind": "rotary", "dtype": "bf16", "heads": 32, "kv": 8, "d": 128, "page": 16,
         "seqs": 48, "nodes_low": 1, "nodes": 1, "low": 60, "high": 8000, "dims": 128, "adjacent": False,
         "gains": True, "pick": 1},
        # a serving step's new requests, of ragged lengths
        {"name": "rotary_prompt", "kind": "rotary", "dtype": "fp16", "heads": 32, "kv": 8, "d": 128, "page": 16,
         "seqs": 24, "nodes_low": 17, "nodes": 1500, "low": 0, "high": 0, "dims": 128, "adjacent": False,
         "gains": True, "pick": 2},
        # one token of one conversation
        {"name": "append8_token", "kind": "append", "dtype": "bf16", "heads": 16, "kv": 8, "d": 128, "page": 16,
         "seqs": 1, "nodes_low": 1, "nodes": 1, "low": 2103, "high": 2103, "dims": 128, "adjacent": False,
         "gains": True, "pick": 3},
        # the packed prompts' rows, a part of every head rotated in adjacent pairs
        {"name": "append8_prompt", "kind": "append", "dtype": "bf16", "heads": 32, "kv": 8, "d": 128, "page": 64,
         "seqs": 24, "nodes_low": 17, "nodes": 1500, "low": 1, "high": 90, "dims": 64, "adjacent": True,
         "gains": False, "pick": 4},
        # one token of one conversation: plain decoding
        {"name": "attend8_token", "kind": "attend", "dtype": "bf16", "heads": 16, "kv": 8, "d": 128, "page": 16,
         "seqs": 1, "nodes_low": 1, "nodes": 1, "low": 2100, "high": 2100, "pick": 5},
        # drafts of a serving batch, contexts of all lengths
        {"name": "attend8_batch", "kind": "attend", "dtype": "fp16", "heads": 32, "kv": 8, "d": 128, "page": 16,
         "seqs": 48, "nodes_low": 1, "nodes": 26, "low": 60, "high": 8000, "pick": 6},
        # a few long documents, large drafts
        {"name": "attend8_long", "kind": "attend", "dtype": "bf16", "heads": 16, "kv": 8, "d": 128, "page": 64,
         "seqs": 4, "nodes_low": 40, "nodes": 64, "low": 90000, "high": 131000, "pick": 7},
        # one conversation's accepted draft
        {"name": "keep8_one", "kind": "keep", "dtype": "bf16", "heads": 16, "kv": 8, "d": 128, "page": 16,
         "seqs": 1, "nodes_low": 60, "nodes": 60, "low": 403, "high": 403, "pick": 8},
        # a batch's accepted drafts
        {"name": "keep8_batch", "kind": "keep", "dtype": "fp16", "heads": 16, "kv": 8, "d": 128, "page": 16,
         "seqs": 48, "nodes_low": 8, "nodes": 26, "low": 60, "high": 400, "pick": 9},
        # one conversation's next token
        {"name": "sample_one", "kind": "sample", "dtype": "bf16", "rows": 1, "vocab": 151936, "t": 0.6, "k": 20,
         "p": 0.95, "m": 0.0, "mixed": False, "pick": 10},
        # a serving batch whose requests ask for different things
        {"name": "sample_mixed", "kind": "sample", "dtype": "bf16", "rows": 48, "vocab": 151936, "t": 0.8, "k": 50,
         "p": 0.9, "m": 0.05, "mixed": True, "pick": 11},
        # many samples of a task, by probability mass alone
        {"name": "sample_mass", "kind": "sample", "dtype": "fp32", "rows": 256, "vocab": 151936, "t": 1.0, "k": 0,
         "p": 0.95, "m": 0.0, "mixed": False, "pick": 12},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        have = top.setdefault(c["kind"], w)
        top[c["kind"]] = {n: max(have[n], w[n]) for n in w}
    kind = rng.choice(["rotary", "append", "attend", "attend", "keep", "sample", "sample"])
    case = {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), "pick": rng.randrange(1 << 20)}
    while True:
        if kind == "sample":
            case.update(dtype=rng.choice(["bf16", "fp16", "fp32"]), rows=_log(rng, 1, 256),
                        vocab=_log(rng, 1000, 155000), t=round(rng.uniform(0.3, 1.5), 2),
                        k=rng.choice([0, 0, 1, _log(rng, 2, 2000)]), p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                        m=rng.choice([0.0, round(rng.uniform(0.0, 0.2), 3)]), mixed=rng.random() < 0.4)
        else:
            heads, kv = rng.choice([(16, 8), (32, 8), (32, 8), (16, 16), (12, 2)])
            d, seqs = rng.choice([128, 128, 64]), _log(rng, 1, 64)
            case.update(heads=heads, kv=kv, d=d, seqs=seqs, page=rng.choice([16, 16, 32, 64, 128]))
            if kind in ("rotary", "append"):
                nodes, high = rng.choice([1, _log(rng, 1, 1500)]), _log(rng, 1, 8000 if kind == "rotary" else 500)
                case.update(dims=rng.choice([d, d, d // 2, 48]), adjacent=rng.random() < 0.3, gains=rng.random() < 0.5)
            else:
                nodes = rng.choice([1, _log(rng, 1, 64), 64])
                high = _log(rng, 1, 131072 if kind == "attend" else 400)
            case.update(nodes_low=_log(rng, 1, nodes), nodes=nodes, low=_log(rng, 1, high), high=high)
        w = work(case)
        if w["bytes"] <= top[kind]["bytes"] and w["flops"] <= max(top[kind]["flops"], 1) and _held(case) <= 3e10:
            return case


# ---------------------------------------------------------------- shapes of a case

def _between(rng, low, high):
    return low if low == high else int(round(math.exp(rng.uniform(math.log(max(low, 1)), math.log(high)))))


def _lengths(case):
    """Per sequence: (rows of the batch, positions before them)."""
    rng = random.Random(case["pick"])
    return [(_between(rng, case["nodes_low"], case["nodes"]), _between(rng, case["low"], case["high"]))
            for _ in range(case["seqs"])]


def _trees(case):
    """Per sequence: each node's parent (-1: the last cached token), and the accepted path's nodes."""
    rng, out = random.Random(case["pick"] + 1), []
    for n, _ in _lengths(case):
        parents = [rng.randint(max(-1, i - 5), i - 1) for i in range(n)]
        path, at = [], rng.randrange(n)
        while at >= 0:
            path.append(at)
            at = parents[at]
        out.append((parents, path[::-1]))
    return out


def _page_bytes(case):
    """Bytes of an 8-bit page."""
    return -(-(case["kv"] * case["page"] * case["d"] + case["kv"] * case["page"] // BLOCK) // 128) * 128


def _held(case):
    """Bytes of the plain form's largest tensor."""
    if case["kind"] == "sample":
        return 8 * case["rows"] * case["vocab"]
    n, c = max(n for n, _ in _lengths(case)), max(c for _, c in _lengths(case))
    pages = case["seqs"] * (-(-(n + c) // case["page"]) + 1) * (LAYERS if case["kind"] == "keep" else 1)
    pool = 4 * pages * case["page"] * case["kv"] * case["d"]
    return max(pool, 4 * case["seqs"] * (n + c) * case["heads"] * n if case["kind"] == "attend" else 0)


def work(case):
    if case["kind"] == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": 0}
    sizes, kv, d = _lengths(case), case["kv"], case["d"]
    rows, ends = sum(n for n, _ in sizes), sum(n + c for n, c in sizes)
    q = 2 * case["heads"] * d  # bytes of a row's queries
    if case["kind"] == "rotary":
        return {"bytes": rows * (2 * q + 8 * kv * d + 4 * case["dims"]), "flops": 0}
    if case["kind"] == "append":
        blocks = sum((c + n - 1) // BLOCK - c // BLOCK + 1 for n, c in sizes)
        return {"bytes": rows * (2 * q + 6 * kv * d + 4 * case["dims"]) + 2 * blocks * kv, "flops": 0}
    if case["kind"] == "keep":
        moved = sum(j != i for _, path in _trees(case) for j, i in enumerate(path))
        return {"bytes": max(4 * LAYERS * moved * kv * d, 4 * rows), "flops": 0}
    pairs = sum(n * c for n, c in sizes)
    for parents, _ in _trees(case):
        depth = []
        for p in parents:
            depth.append(1 + (depth[p] if p >= 0 else 0))
        pairs += sum(depth)
    return {"bytes": 2 * ends * kv * d + 2 * ends * kv // BLOCK + 2 * rows * q, "flops": 4 * d * case["heads"] * pairs}


# ---------------------------------------------------------------- inputs

def _generator(seed, which):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + which * 7919) % (1 << 62))
    return g


def _normal(shape, seed, which):
    return torch.randn(shape, generator=_generator(seed, which), device="cuda", dtype=torch.float32)


def _u32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sums(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def prepare(case, seed):
    s = {"case": case}
    if case["kind"] == "sample":
        _prepare_sample(s, case, seed)
    else:
        _prepare_batch(s, case, seed)
    if own:
        _handles(s, case)
    torch.cuda.synchronize()  # the runtime has its own stream
    return s


def _prepare_sample(s, case, seed):
    rows, vocab = case["rows"], case["vocab"]
    x = _normal((rows, vocab), seed, 1) * 2.5
    few = max(1, min(60, vocab // 20))  # the tokens that the context speaks for
    at = torch.randint(vocab, (rows, few), generator=_generator(seed, 2), device="cuda")
    x.scatter_add_(1, at, torch.rand((rows, few), generator=_generator(seed, 3), device="cuda") * 14)
    s["logits"] = x.to(DTYPES[case["dtype"]])
    t, k, p, m = ([case[n]] * rows for n in "tkpm")
    if case["mixed"]:  # greedy, everything, and each filter alone
        rng = random.Random(case["pick"])
        for i in range(rows):
            t[i], which = round(rng.uniform(0.4, 1.3), 2), rng.randrange(6)
            if which == 0:
                t[i] = 0.0
            k[i] = case["k"] if which in (2, 5) else 0
            p[i] = case["p"] if which in (3, 5) else 1.0
            m[i] = case["m"] if which in (4, 5) else 0.0
    s["t"], s["p"], s["m"] = (torch.tensor(v, dtype=torch.float32, device="cuda") for v in (t, p, m))
    s["k"] = _u32(k)
    s["u"] = torch.rand(rows, generator=_generator(seed, 4), device="cuda")
    s["tokens"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    s["probability"] = torch.zeros(rows, device="cuda")


def _codes(pool, case):
    """The codes of 8-bit pages, [layers, pages, kv, page, d]."""
    kv, page, d = case["kv"], case["page"], case["d"]
    return pool[:, :, : kv * page * d].unflatten(2, (kv, page, d))


def _scales(pool, case):
    """Their scale bytes, [layers, pages, kv, page / 16]."""
    kv, page, d = case["kv"], case["page"], case["d"]
    return pool[:, :, kv * page * d: kv * page * d + kv * page // BLOCK].unflatten(2, (kv, page // BLOCK))


def _pool8(case, layers, pages, seed, which):
    """Pages full of earlier rows, whose blocks' sizes differ."""
    kv, page, d = case["kv"], case["page"], case["d"]
    pool = torch.zeros((layers, pages, _page_bytes(case)), dtype=torch.uint8, device="cuda")
    for layer in range(layers):
        x = _normal((pages, kv, page // BLOCK, BLOCK, d), seed, which + 100 * layer)
        x *= torch.exp2(_normal((pages, kv, page // BLOCK, 1, 1), seed, which + 100 * layer + 50))
        m, e = torch.frexp(x.abs().amax((3, 4)))
        e = e - 9 + (m > 0.875)
        x *= torch.exp2(-e[..., None, None].float())
        _codes(pool, case)[layer] = x.reshape(pages, kv, page, d).to(FP8).view(torch.uint8)
        _scales(pool, case)[layer] = (e + 127).to(torch.uint8)
    return pool


def _prepare_batch(s, case, seed):
    """A cache whose sequences' pages lie scattered over the pool, and the batch's rows."""
    dtype, sizes, heads, kv, d, page = DTYPES[case["dtype"]], _lengths(case), case["heads"], case["kv"], case["d"], case["page"]
    held = [-(-(n + c) // page) for n, c in sizes]
    ids, tables = list(range(sum(held) + 3)), []
    random.Random(case["pick"] + 2).shuffle(ids)
    for first, count in zip(_sums(held), held):
        tables.append(ids[first: first + count] + [ids[0]] * (max(held) - count))
    layers = LAYERS if case["kind"] == "keep" else 1
    if case["kind"] == "rotary":
        s["k_pool"] = _normal((layers, len(ids), kv, page, d), seed, 1).to(dtype)
        s["v_pool"] = _normal((layers, len(ids), kv, page, d), seed, 2).to(dtype)
    else:
        s["k_pool"] = _pool8(case, layers, len(ids), seed, 1)
        s["v_pool"] = _pool8(case, layers, len(ids), seed, 2)
    s["tables"], s["starts"] = _u32(tables), _u32(_sums(n for n, _ in sizes))
    s["context"], s["rows"] = _u32([c for _, c in sizes]), sum(n for n, _ in sizes)
    s["longest"], s["end"] = max(n for n, _ in sizes), max(n + c for n, c in sizes)
    if case["kind"] in ("rotary", "append"):
        s["k"] = _normal((s["rows"], kv, d), seed, 3).to(dtype)
        s["v"] = _normal((s["rows"], kv, d), seed, 4).to(dtype)
        s["q"] = _normal((s["rows"], heads, d), seed, 5).to(dtype)
        s["q_out"] = torch.zeros_like(s["q"])
        if case["gains"]:
            s["q_gain"] = (1 + 0.2 * _normal((d,), seed, 6)).to(dtype)
            s["k_gain"] = (1 + 0.2 * _normal((d,), seed, 7)).to(dtype)
        pairs = case["dims"] // 2
        angle = torch.arange(s["end"], device="cuda", dtype=torch.float64)[:, None] * torch.pow(
            torch.tensor(1e6, device="cuda", dtype=torch.float64), -torch.arange(pairs, device="cuda") / pairs)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        return
    trees = _trees(case)
    if case["kind"] == "keep":
        kept = [path + [0] * (n - len(path)) for (n, _), (_, path) in zip(sizes, trees)]
        s["kept"], s["counts"] = _u32([i for k in kept for i in k]), _u32([len(path) for _, path in trees])
        s["new_context"] = torch.zeros_like(s["context"])
        return
    masks = []
    for parents, _ in trees:
        of = []
        for i, p in enumerate(parents):
            of.append((of[p] if p >= 0 else 0) | 1 << i)
        masks += of
    s["visible"] = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device="cuda")
    s["q"] = _normal((s["rows"], heads, d), seed, 3).to(dtype)
    s["out"] = torch.zeros_like(s["q"])


_rt = None


def _handles(s, case):
    """What a program keeps beside its tensors: the runtime, the shapes, the workspace."""
    global _rt
    import xpu_playground_amd as xpu

    if _rt is None:
        _rt = xpu.Runtime()
    s["rt"], code = _rt, {"bf16": xpu.BF16, "fp16": xpu.FP16, "fp32": xpu.FP32}[case["dtype"]]
    if case["kind"] == "sample":
        s["sampling"] = xpu.Sampling(code, case["rows"], case["vocab"], s["u"].data_ptr(), s["t"].data_ptr(),
                                     s["k"].data_ptr(), s["p"].data_ptr(), s["m"].data_ptr())
        size = _rt.sample_workspace(s["sampling"])
        s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        return
    layers, pool = s["k_pool"].shape[:2]
    shape = code, layers, case["kv"], case["d"], case["page"], pool, s["k_pool"].data_ptr(), s["v_pool"].data_ptr()
    if case["kind"] == "rotary":
        s["cache"] = xpu.Cache(*shape)
    else:
        s["cache"] = xpu.Cache8(*shape, layer_stride=pool * _page_bytes(case), page_stride=_page_bytes(case))
    s["batch"] = xpu.Batch(case["seqs"], s["rows"], s["tables"].shape[1], s["tables"].data_ptr(),
                           s["starts"].data_ptr(), s["context"].data_ptr())
    if case["kind"] in ("rotary", "append"):
        gains = {n: s[n].data_ptr() for n in ("q_gain", "k_gain") if n in s}
        s["rotary"] = xpu.Rotary(s["end"], case["dims"], s["cos"].data_ptr(), s["sin"].data_ptr(),
                                 pairs=xpu.ADJACENT if case["adjacent"] else xpu.HALVES, eps=EPS, **gains)
    if case["kind"] == "attend":
        size = _rt.tree_attention8_workspace(s["cache"], s["batch"], case["heads"])
        s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")


# ---------------------------------------------------------------- one pass

def run(state):
    kind, case = state["case"]["kind"], state["case"]
    if own:
        _run_own(state, kind)
    else:
        {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "keep": _plain_keep,
         "sample": _plain_sample}[kind](state)
    if kind == "sample":
        return {"tokens": state["tokens"], "probability": state["probability"]}
    if kind == "attend":
        return state["out"]
    if kind == "rotary":
        return {"k": state["k_pool"], "v": state["v_pool"], "q": state["q_out"]}
    out = {}
    for name in ("k", "v"):
        out[name] = _codes(state[name + "_pool"], case).view(FP8)
        out[name + "_scale"] = _scales(state[name + "_pool"], case).view(torch.float8_e8m0fnu)
    if kind == "append":
        return {**out, "q": state["q_out"]}
    return {**out, "context": state["new_context"]}


def _run_own(s, kind):
    rt = s["rt"]
    if kind == "sample":
        rt.sample(s["sampling"], s["logits"].data_ptr(), s["tokens"].data_ptr(), s["workspace"].data_ptr(),
                  s["workspace"].numel(), probability=s["probability"].data_ptr())
    elif kind == "attend":
        rt.tree_attention8(s["cache"], s["batch"], 0, s["case"]["heads"], s["q"].data_ptr(), s["out"].data_ptr(),
                           s["workspace"].data_ptr(), s["workspace"].numel(), visible=s["visible"].data_ptr())
    elif kind == "keep":
        rt.cache8_keep(s["cache"], s["batch"], s["kept"].data_ptr(), s["counts"].data_ptr(),
                       s["new_context"].data_ptr())
    else:
        call = rt.cache_append_rotary if kind == "rotary" else rt.cache8_append
        call(s["cache"], s["batch"], 0, s["k"].data_ptr(), s["v"].data_ptr(), rotary=s["rotary"],
             heads=s["case"]["heads"], q=s["q"].data_ptr(), q_out=s["q_out"].data_ptr())


def _places(starts, rows, longest):
    """The packed rows as [sequences, longest] row numbers, and which of them exist."""
    at = torch.arange(longest, device="cuda")
    lens = (starts[1:] - starts[:-1]).long()
    return torch.clamp(starts[:-1, None].long() + at, max=rows - 1), at < lens[:, None], lens


def _new_rows(s):
    """Of each of the batch's rows: its sequence and its position."""
    _, real, _ = _places(s["starts"], s["rows"], s["longest"])
    seq, i = real.nonzero(as_tuple=True)
    return seq, s["context"].long()[seq] + i


def _turned(x, s, gain, at):
    """Rows [rows, heads, d], normalised where there is a gain, rotated by their positions."""
    c = s["case"]
    x = x.float()
    if gain is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.float()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    a, rest = x[..., : c["dims"]], x[..., c["dims"]:]
    x, y = (a[..., 0::2], a[..., 1::2]) if c["adjacent"] else a.chunk(2, -1)
    x, y = x * cos - y * sin, y * cos + x * sin
    a = torch.stack((x, y), -1).flatten(-2) if c["adjacent"] else torch.cat((x, y), -1)
    return torch.cat((a, rest), -1)


def _plain_rotary(s):
    page = s["case"]["page"]
    seq, at = _new_rows(s)
    ids = s["tables"].long()[seq, at // page]
    s["k_pool"][0, ids, :, at % page] = _turned(s["k"], s, s.get("k_gain"), at).to(s["k"].dtype)
    s["v_pool"][0, ids, :, at % page] = s["v"]
    s["q_out"].copy_(_turned(s["q"], s, s.get("q_gain"), at))


def _exponent(top):
    """The scale byte with which values up to `top` are at most 448."""
    m, e = torch.frexp(top)
    return torch.where(top > 0, torch.clamp(e.long() - 9 + (m > 0.875) + 127, LEAST, 247), LEAST)


def _earlier(s, reached):
    """Positions before the batch's in a block that it reaches: their sequence and position."""
    context = s["context"].long()
    at = context[:, None] // BLOCK * BLOCK + torch.arange(BLOCK - 1, device="cuda")
    seq, i = ((at < context[:, None]) & reached[:, None]).nonzero(as_tuple=True)
    return seq, at[seq, i]


def _rescale(code, by):
    """Codes times 2^by, rounded."""
    return (code.view(FP8).float() * torch.exp2(by.float())[..., None]).to(FP8).view(torch.uint8)


def _plain_append(s):
    c = s["case"]
    page, per = c["page"], c["page"] // BLOCK
    tables, (seq, at) = s["tables"].long(), _new_rows(s)
    _, _, lens = _places(s["starts"], s["rows"], s["longest"])
    e_seq, e_at = _earlier(s, lens > 0)
    ids, e_ids = tables[seq, at // page], tables[e_seq, e_at // page]
    block, e_block = ids * per + at % page // BLOCK, e_ids * per + e_at % page // BLOCK
    k = _turned(s["k"], s, s.get("k_gain"), at)
    s["q_out"].copy_(_turned(s["q"], s, s.get("q_gain"), at))
    for pool, x in ((s["k_pool"], k), (s["v_pool"], s["v"].float())):
        codes, scales = _codes(pool, c)[0], _scales(pool, c)[0]
        old = scales.transpose(1, 2).reshape(-1, c["kv"]).long()
        new = torch.full_like(old, LEAST)
        new[e_block] = old[e_block]
        needed = _exponent(x.abs().amax(-1))
        new.scatter_reduce_(0, block[:, None].expand(-1, c["kv"]), needed, "amax")
        earlier = _rescale(codes[e_ids, :, e_at % page], old[e_block] - new[e_block])
        codes[e_ids, :, e_at % page] = earlier
        codes[ids, :, at % page] = (x * torch.exp2(127.0 - new[block])[..., None]).to(FP8).view(torch.uint8)
        scales[ids, :, at % page // BLOCK] = new[block].to(torch.uint8)


def _softmax(scores, seen):
    """Over the last axis, of the seen entries; 0 for a row that sees none."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _plain_attend(s):
    c = s["case"]
    seqs, kv, group, d = c["seqs"], c["kv"], c["heads"] // c["kv"], c["d"]
    qi, qv, n = _places(s["starts"], s["rows"], s["longest"])
    pages = s["tables"].long()

    def positions(pool):  # [seqs, kv, positions, d]
        codes = _codes(pool, c)[0][pages].view(FP8).float()
        scales = torch.exp2(_scales(pool, c)[0][pages].float() - 127)
        x = codes.unflatten(3, (-1, BLOCK)) * scales[..., None, None]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(seqs, kv, -1, d)[:, :, : s["end"]]

    at = torch.arange(s["end"], device="cuda")
    context = s["context"].long()[:, None, None]
    node = at[None, None, :] - context  # of a position: below 0 for the cached ones
    bit = s["visible"][qi][:, :, None] >> torch.clamp(node, 0, 63) & 1
    seen = (node < 0) | (node < n[:, None, None]) & (bit == 1)
    q = s["q"][qi].float().reshape(seqs, s["longest"], kv, group, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(seqs, kv, group * s["longest"], d)
    scores = q @ positions(s["k_pool"]).transpose(2, 3).contiguous() / math.sqrt(d)
    p = _softmax(scores.reshape(seqs, kv, group, s["longest"], -1), seen[:, None, None])
    o = p.reshape(seqs, kv, group * s["longest"], -1) @ torch.where(
        (at < context[:, 0] + n[:, None])[:, None, :, None], positions(s["v_pool"]), 0.0)
    o = o.reshape(seqs, kv, group, s["longest"], d).permute(0, 3, 1, 2, 4).reshape(seqs, s["longest"], kv * group, d)
    s["out"][qi[qv]] = o[qv].to(s["out"].dtype)


def _plain_keep(s):
    c = s["case"]
    page, per, kv = c["page"], c["page"] // BLOCK, c["kv"]
    rows, _, _ = _places(s["starts"], s["rows"], s["longest"])
    j = torch.arange(s["longest"], device="cuda")
    seq, j = (j < s["counts"].long()[:, None]).nonzero(as_tuple=True)
    context, tables = s["context"].long(), s["tables"].long()
    to, of = context[seq] + j, context[seq] + s["kept"].long()[rows[seq, j]]
    e_seq, e_at = _earlier(s, s["counts"] > 0)
    to_ids, of_ids, e_ids = tables[seq, to // page], tables[seq, of // page], tables[e_seq, e_at // page]
    to_block, of_block, e_block = (i * per + a % page // BLOCK for i, a in ((to_ids, to), (of_ids, of), (e_ids, e_at)))
    for pool in (s["k_pool"], s["v_pool"]):
        codes, scales = _codes(pool, c), _scales(pool, c)
        old = scales.transpose(2, 3).reshape(LAYERS, -1, kv).int()
        came = old[:, of_block]
        new = old.scatter_reduce(1, to_block[None, :, None].expand(LAYERS, -1, kv), came, "amax")
        moved = codes.permute(1, 3, 0, 2, 4)[of_ids, of % page]  # [rows, layers, kv, d]
        moved = _rescale(moved, (came - new[:, to_block]).transpose(0, 1))
        earlier = codes.permute(1, 3, 0, 2, 4)[e_ids, e_at % page]
        earlier = _rescale(earlier, (old[:, e_block] - new[:, e_block]).transpose(0, 1))
        codes.permute(1, 3, 0, 2, 4)[to_ids, to % page] = moved
        codes.permute(1, 3, 0, 2, 4)[e_ids, e_at % page] = earlier
        scales.permute(1, 3, 0, 2)[to_ids, to % page // BLOCK] = new[:, to_block].transpose(0, 1).to(torch.uint8)
    s["new_context"].copy_(s["context"] + s["counts"])


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    x, ids = x.sort(dim=1, descending=True, stable=True)
    t = s["t"].double()[:, None]
    rank = torch.arange(vocab, device="cuda")
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    k = s["k"].long()[:, None]
    w = torch.where((k == 0) | (rank < k), w, 0.0)
    w = torch.where((t > 0) | (rank == 0), w, 0.0)
    upto = w.cumsum(1)
    p = s["p"].double()[:, None]
    kept = (p >= 1) | (upto - w < p * upto[:, -1:]) | (rank == 0)
    w = torch.where(kept & (w >= s["m"].double()[:, None]), w, 0.0)
    upto = w.cumsum(1)
    past = upto > s["u"].double()[:, None] * upto[:, -1:]
    at = past.int().argmax(1, keepdim=True)
    s["tokens"].copy_(ids.gather(1, at)[:, 0])
    s["probability"].copy_((w.gather(1, at) / upto[:, -1:])[:, 0])


# ---------------------------------------------------------------- in 64 bits

def _attend(q, k, v, seen):
    """One head: rows of q against k and v, where seen says so."""
    s = (q @ k.T / math.sqrt(q.shape[1])).masked_fill(~seen, -math.inf)
    w = torch.where(seen, torch.exp(s - s.max(1, keepdim=True).values), 0.0)
    return w @ v / w.sum(1, keepdim=True)


def _exact_turned(x, s, gain, at):
    """The rotation as a product of complex numbers."""
    c, x = s["case"], x.double()
    if gain is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["d"] + EPS) * gain.double()
    half, turn = c["dims"] // 2, torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
    first = torch.arange(half, device="cuda") * (2 if c["adjacent"] else 1)
    second = first + (1 if c["adjacent"] else half)
    z = torch.complex(x[..., first], x[..., second]) * turn
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_sample(case, s):
    import numpy as np

    logits, t, p, m, u = (s[n].double().cpu().numpy() for n in ("logits", "t", "p", "m", "u"))
    k, tokens, probability = s["k"].cpu().numpy(), [], []
    for i in range(case["rows"]):
        order = np.lexsort((np.arange(case["vocab"]), -logits[i]))
        if t[i] == 0:
            order, w = order[:1], np.ones(1)
        else:
            order = order[: k[i]] if k[i] else order
            w = np.exp((logits[i][order] - logits[i][order[0]]) / t[i])
        if p[i] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), p[i] * w.sum()))
            order, w = order[:n], w[:n]
        order, w = order[w >= m[i]], w[w >= m[i]]
        at = int(np.searchsorted(np.cumsum(w), u[i] * w.sum(), side="right"))
        at = min(at, len(w) - 1)
        tokens.append(int(order[at]))
        probability.append(float(w[at] / w.sum()))
    return {"tokens": torch.tensor(tokens), "probability": torch.tensor(probability, dtype=torch.float64)}


def exact(case, seed):
    s = {"case": case}
    if case["kind"] == "sample":
        _prepare_sample(s, case, seed)
        return _exact_sample(case, s)
    _prepare_batch(s, case, seed)
    sizes, page, per, tables = _lengths(case), case["page"], case["page"] // BLOCK, s["tables"].tolist()
    group, kv, d, first = case["heads"] // case["kv"], case["kv"], case["d"], 0
    if case["kind"] == "attend":
        out, q, trees = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), s["q"].double(), _trees(case)
        for i, (n, c) in enumerate(sizes):
            parents, seen = trees[i][0], torch.zeros((n, n + c), dtype=torch.bool)
            seen[:, :c] = True
            for r, p in enumerate(parents):
                if p >= 0:
                    seen[r] = seen[p]
                seen[r, c + r] = True
            seen, held = seen.cuda(), tables[i][: -(-(n + c) // page)]
            for h in range(case["heads"]):
                k, v = (torch.ldexp(_codes(pool, case)[0, held, h // group].view(FP8).double().reshape(-1, BLOCK, d),
                                    _scales(pool, case)[0, held, h // group].reshape(-1, 1, 1).int() - 127)
                        .reshape(-1, d)[: n + c] for pool in (s["k_pool"], s["v_pool"]))
                out[first: first + n, h] = _attend(q[first: first + n, h], k, v, seen)
            first += n
        return out
    if case["kind"] == "keep":
        return _exact_keep(case, s)
    at = torch.cat([torch.arange(c, c + n, device="cuda") for n, c in sizes])
    rows = {"k": _exact_turned(s["k"], s, s.get("k_gain"), at), "v": s["v"].double()}
    out = {"q": _exact_turned(s["q"], s, s.get("q_gain"), at)}
    for name in ("k", "v"):
        if case["kind"] == "rotary":
            codes = s[name + "_pool"].double()
        else:
            codes = _codes(s[name + "_pool"], case).view(FP8).double()
            scales = torch.ldexp(torch.ones((), dtype=torch.float64, device="cuda"), _scales(s[name + "_pool"], case).int() - 127)
        first = 0
        for (n, c), table in zip(sizes, tables):
            for start in range(c // BLOCK * BLOCK, c + n, BLOCK):  # 16 positions are of one page
                low, high = max(start, c), min(start + BLOCK, c + n)
                x, id, slot = rows[name][first + low - c: first + high - c].transpose(0, 1), table[start // page], start % page
                if case["kind"] == "append":
                    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)) / 448)))
                    old = scales[0, id, :, slot // BLOCK]
                    if low > start:
                        scale = torch.maximum(scale, old)
                        codes[0, id, :, slot: slot + low - start] *= (old / scale)[:, None, None]
                    scales[0, id, :, slot // BLOCK] = scale
                    x = x / scale[:, None, None]
                codes[0, id, :, slot + low - start: slot + high - start] = x
            first += n
        out[name] = codes
        if case["kind"] == "append":
            out[name + "_scale"] = scales
    return out


def _exact_keep(case, s):
    page, tables, out = case["page"], s["tables"].tolist(), {"context": None}
    for name in ("k", "v"):
        codes = _codes(s[name + "_pool"], case).view(FP8).double()
        scales = torch.ldexp(torch.ones((), dtype=torch.float64, device="cuda"), _scales(s[name + "_pool"], case).int() - 127)
        for (n, c), table, (_, path) in zip(_lengths(case), tables, _trees(case)):
            def block(at):
                return slice(None), table[at // page], slice(None), at % page // BLOCK

            def row(at):
                return slice(None), table[at // page], slice(None), at % page

            old = {b: scales[block(b * BLOCK)].clone() for b in range(c // BLOCK, (c + n - 1) // BLOCK + 1)}
            held = [codes[row(c + i)] * old[(c + i) // BLOCK][..., None] for i in path]
            for j, i in enumerate(path):
                at = block(c + j)
                scales[at] = torch.maximum(scales[at], old[(c + i) // BLOCK])
            for at in range(c // BLOCK * BLOCK, c):
                codes[row(at)] *= (old[at // BLOCK] / scales[block(at)])[..., None]
            for j, x in enumerate(held):
                codes[row(c + j)] = x / scales[block(c + j)][..., None]
        out[name], out[name + "_scale"] = codes, scales
    return out
