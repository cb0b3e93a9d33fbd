"""Performance cases of the paged KV cache and the attention over it.

  prompt  Runtime.prompt_attention: causal attention of packed prompts of
          different lengths, grouped heads
  tree    Runtime.tree_attention: drafted tokens (a tree of up to 64 nodes
          per sequence, or one token each) over the paged cache
  append  Runtime.cache_append: new K and V rows into the cache's pages
  keep    Runtime.cache_keep: the accepted nodes of each draft move to the
          front of the draft, in every layer
  copy    Runtime.cache_copy: whole pages copied for forks, in every layer

Head counts and sizes are those of the framework's qwen3 presets (16 query and
8 kv heads, 32 and 8, head size 128) and the generic 64-wide heads.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
LAYERS = 28  # of the qwen3-0.6b preset


def listed():
    return [
        # one short question: launch latency counts
        {"name": "prompt_short", "kind": "prompt", "dtype": "bf16", "heads": 16, "kv": 8, "d": 128, "seqs": 1,
         "low": 128, "high": 128, "prior": 0, "pick": 1},
        # a serving step's new requests, of ragged lengths
        {"name": "prompt_packed", "kind": "prompt", "dtype": "fp16", "heads": 32, "kv": 8, "d": 128, "seqs": 24,
         "low": 17, "high": 1500, "prior": 0, "pick": 2},
        # a document in the prompt
        {"name": "prompt_long", "kind": "prompt", "dtype": "bf16", "heads": 32, "kv": 8, "d": 128, "seqs": 1,
         "low": 8192, "high": 8192, "prior": 0, "pick": 3},
        # one token of one conversation: plain decoding
        {"name": "tree_token", "kind": "tree", "dtype": "bf16", "heads": 16, "kv": 8, "d": 128, "page": 16,
         "seqs": 1, "nodes_low": 1, "nodes": 1, "low": 2100, "high": 2100, "pick": 4},
        # drafts of a serving batch, contexts of all lengths
        {"name": "tree_batch", "kind": "tree", "dtype": "fp16", "heads": 32, "kv": 8, "d": 128, "page": 16,
         "seqs": 48, "nodes_low": 1, "nodes": 26, "low": 60, "high": 8000, "pick": 5},
        # a few long documents, large drafts
        {"name": "tree_long", "kind": "tree", "dtype": "bf16", "heads": 16, "kv": 8, "d": 128, "page": 64,
         "seqs": 4, "nodes_low": 40, "nodes": 64, "low": 90000, "high": 131000, "pick": 6},
        # a decode step's rows of a serving batch
        {"name": "append_step", "kind": "append", "dtype": "bf16", "heads": 32, "kv": 8, "d": 128, "page": 16,
         "seqs": 48, "nodes_low": 1, "nodes": 1, "low": 60, "high": 500, "pick": 7},
        # the packed prompts' rows
        {"name": "append_prompt", "kind": "append", "dtype": "fp16", "heads": 32, "kv": 8, "d": 128, "page": 16,
         "seqs": 24, "nodes_low": 17, "nodes": 1500, "low": 0, "high": 0, "pick": 2},
        # one conversation's accepted draft
        {"name": "keep_one", "kind": "keep", "dtype": "bf16", "heads": 16, "kv": 8, "d": 128, "page": 16,
         "seqs": 1, "nodes_low": 60, "nodes": 60, "low": 403, "high": 403, "pick": 8},
        # a batch's accepted drafts
        {"name": "keep_batch", "kind": "keep", "dtype": "fp16", "heads": 16, "kv": 8, "d": 128, "page": 16,
         "seqs": 48, "nodes_low": 8, "nodes": 26, "low": 60, "high": 400, "pick": 9},
        # the last pages of a few forked conversations
        {"name": "copy_few", "kind": "copy", "dtype": "bf16", "heads": 16, "kv": 8, "d": 128, "page": 16,
         "pages": 4, "pool": 64, "pick": 10},
        # pages moved together to free the end of a pool
        {"name": "copy_many", "kind": "copy", "dtype": "fp16", "heads": 16, "kv": 8, "d": 128, "page": 64,
         "pages": 101, "pool": 256, "pick": 11},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    heads, kv = rng.choice([(16, 8), (32, 8), (32, 8), (16, 16), (12, 2)])
    case = {"kind": rng.choice(["prompt", "prompt", "tree", "tree", "append", "keep", "copy"]),
            "dtype": rng.choice(["bf16", "fp16"]), "heads": heads, "kv": kv, "d": rng.choice([128, 128, 64]),
            "pick": rng.randrange(1 << 20)}
    top = {c["kind"]: work(c) for c in listed()}  # the last listed case of a kind is its largest
    while True:
        if case["kind"] == "prompt":
            high = _log(rng, 2, 8192)
            case.update(seqs=_log(rng, 1, 32), low=_log(rng, 1, high), high=high,
                        prior=rng.choice([0, 0, _log(rng, 1, 4096)]))
        elif case["kind"] == "copy":
            pages = _log(rng, 1, 120)
            case.update(page=rng.choice([16, 32, 64]), pages=pages, pool=2 * pages + rng.randint(0, 60))
        else:
            seqs, page = _log(rng, 1, 64), rng.choice([16, 16, 32, 64, 128])
            if case["kind"] == "append":
                nodes, high = rng.choice([1, _log(rng, 1, 1500)]), _log(rng, 1, 500)
            else:
                nodes = rng.choice([1, _log(rng, 1, 64), 64])
                high = _log(rng, 1, 131072 if case["kind"] == "tree" else 400)
            case.update(seqs=seqs, page=page, nodes_low=_log(rng, 1, nodes), nodes=nodes, low=_log(rng, 1, high),
                        high=high)
        w, most = work(case), top[case["kind"]]
        if w["bytes"] <= most["bytes"] and w["flops"] <= max(most["flops"], 1) and _dense(case) <= 3e10:
            return case


# ---------------------------------------------------------------- shapes of a case

def _between(rng, low, high):
    return low if low == high else int(round(math.exp(rng.uniform(math.log(max(low, 1)), math.log(high)))))


def _lengths(case):
    """Per sequence: (rows of the batch, positions before them)."""
    rng = random.Random(case["pick"])
    if case["kind"] == "prompt":
        return [(_between(rng, case["low"], case["high"]), case["prior"]) for _ in range(case["seqs"])]
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


def _pairs(case):
    """Source and destination pages of a copy, all different."""
    ids = random.Random(case["pick"]).sample(range(case["pool"]), 2 * case["pages"])
    return ids[: case["pages"]], ids[case["pages"]:]


def _dense(case):
    """Bytes of the plain form's largest tensor."""
    if case["kind"] == "copy":
        return 0
    n, c = max(n for n, _ in _lengths(case)), max(c for _, c in _lengths(case))
    return 4 * case["seqs"] * (n + c) * max(case["heads"] * n if case["kind"] in ("prompt", "tree") else 1,
                                            case["kv"] * case["d"])


def work(case):
    row = 2 * case["kv"] * case["d"]  # bytes of one position's K
    if case["kind"] == "copy":
        return {"bytes": 4 * LAYERS * case["pages"] * case["page"] * row, "flops": 0}
    sizes = _lengths(case)
    rows, ends = sum(n for n, _ in sizes), sum(n + c for n, c in sizes)
    q = 2 * case["heads"] * case["d"]
    if case["kind"] == "append":
        return {"bytes": 4 * rows * row, "flops": 0}
    if case["kind"] == "keep":
        moved = sum(j != i for _, path in _trees(case) for j, i in enumerate(path))
        return {"bytes": max(4 * LAYERS * moved * row, 4 * rows), "flops": 0}
    if case["kind"] == "prompt":
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in sizes)
    else:
        pairs = sum(n * c for n, c in sizes)
        for parents, _ in _trees(case):
            depth = []
            for p in parents:
                depth.append(1 + (depth[p] if p >= 0 else 0))
            pairs += sum(depth)
    return {"bytes": 2 * ends * row + 2 * rows * q, "flops": 4 * case["d"] * case["heads"] * pairs}


# ---------------------------------------------------------------- inputs

def _normal(shape, dtype, seed, which):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + which * 7919) % (1 << 62))
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _u32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sums(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def prepare(case, seed):
    dtype, heads, kv, d = DTYPES[case["dtype"]], case["heads"], case["kv"], case["d"]
    s = {"case": case}
    if case["kind"] == "prompt":
        sizes = _lengths(case)
        s["q_starts"], s["k_starts"] = _u32(_sums(n for n, _ in sizes)), _u32(_sums(n + c for n, c in sizes))
        s["rows"], s["keys"] = sum(n for n, _ in sizes), sum(n + c for n, c in sizes)
        s["longest"], s["longest_keys"] = max(n for n, _ in sizes), max(n + c for n, c in sizes)
        s["q"] = _normal((s["rows"], heads, d), dtype, seed, 1)
        s["k"] = _normal((s["keys"], kv, d), dtype, seed, 2)
        s["v"] = _normal((s["keys"], kv, d), dtype, seed, 3)
        s["out"] = torch.zeros_like(s["q"])
    elif case["kind"] == "copy":
        s["src"], s["dst"] = _pairs(case)
        s["k_pool"] = _normal((LAYERS, case["pool"], kv, case["page"], d), dtype, seed, 1)
        s["v_pool"] = _normal((LAYERS, case["pool"], kv, case["page"], d), dtype, seed, 2)
    else:
        _prepare_batch(s, case, dtype, seed)
    if own:
        _handles(s, case)
    torch.cuda.synchronize()  # the runtime has its own stream
    return s


def _prepare_batch(s, case, dtype, seed):
    """A cache whose sequences' pages lie scattered over the pool, and the batch's rows."""
    sizes, heads, kv, d, page = _lengths(case), case["heads"], case["kv"], case["d"], case["page"]
    held = [-(-(n + c) // page) for n, c in sizes]
    ids, tables = list(range(sum(held) + 3)), []
    random.Random(case["pick"] + 2).shuffle(ids)
    for first, count in zip(_sums(held), held):
        tables.append(ids[first: first + count] + [ids[0]] * (max(held) - count))
    layers = LAYERS if case["kind"] == "keep" else 1
    s["k_pool"] = _normal((layers, len(ids), kv, page, d), dtype, seed, 1)
    s["v_pool"] = _normal((layers, len(ids), kv, page, d), dtype, seed, 2)
    s["tables"], s["starts"] = _u32(tables), _u32(_sums(n for n, _ in sizes))
    s["context"], s["rows"] = _u32([c for _, c in sizes]), sum(n for n, _ in sizes)
    s["longest"], s["end"] = max(n for n, _ in sizes), max(n + c for n, c in sizes)
    if case["kind"] == "append":
        s["k"] = _normal((s["rows"], kv, d), dtype, seed, 3)
        s["v"] = _normal((s["rows"], kv, d), dtype, seed, 4)
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
    s["q"] = _normal((s["rows"], heads, d), dtype, seed, 3)
    s["out"] = torch.zeros_like(s["q"])


_rt = None


def _handles(s, case):
    """What a program keeps beside its tensors: the runtime, the shapes, the workspace."""
    global _rt
    import numpy as np
    import xpu_playground_amd as xpu

    if _rt is None:
        _rt = xpu.Runtime()
    s["rt"], code = _rt, {"bf16": xpu.BF16, "fp16": xpu.FP16}[case["dtype"]]
    if case["kind"] == "prompt":
        s["packed"] = xpu.Packed(code, case["heads"], case["kv"], case["d"], case["seqs"], s["rows"],
                                 s["q_starts"].data_ptr(), s["keys"], s["k_starts"].data_ptr())
        return
    layers, pool = s["k_pool"].shape[:2]
    s["cache"] = xpu.Cache(code, layers, case["kv"], case["d"], case["page"], pool, s["k_pool"].data_ptr(),
                           s["v_pool"].data_ptr())
    if case["kind"] == "copy":
        s["pairs"] = np.array(s["src"], np.uint32), np.array(s["dst"], np.uint32)
        return
    s["batch"] = xpu.Batch(case["seqs"], s["rows"], s["tables"].shape[1], s["tables"].data_ptr(),
                           s["starts"].data_ptr(), s["context"].data_ptr())
    if case["kind"] == "tree":
        size = _rt.tree_attention_workspace(s["cache"], s["batch"], case["heads"])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")


# ---------------------------------------------------------------- one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        _run_own(state, kind)
    else:
        {"prompt": _plain_prompt, "tree": _plain_tree, "append": _plain_append, "keep": _plain_keep,
         "copy": _plain_copy}[kind](state)
    if kind in ("prompt", "tree"):
        return state["out"]
    if kind == "keep":
        return {"k": state["k_pool"], "v": state["v_pool"], "context": state["new_context"]}
    return {"k": state["k_pool"], "v": state["v_pool"]}


def _run_own(s, kind):
    rt = s["rt"]
    if kind == "prompt":
        rt.prompt_attention(s["packed"], s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr())
    elif kind == "tree":
        rt.tree_attention(s["cache"], s["batch"], 0, s["case"]["heads"], s["q"].data_ptr(), s["out"].data_ptr(),
                          s["workspace"].data_ptr(), s["workspace"].numel(), visible=s["visible"].data_ptr())
    elif kind == "append":
        rt.cache_append(s["cache"], s["batch"], 0, s["k"].data_ptr(), s["v"].data_ptr())
    elif kind == "keep":
        rt.cache_keep(s["cache"], s["batch"], s["kept"].data_ptr(), s["counts"].data_ptr(),
                      s["new_context"].data_ptr())
    else:
        rt.cache_copy(s["cache"], *s["pairs"])


def _softmax(scores, seen):
    """Over the last axis, of the seen entries; 0 for a row that sees none."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _places(starts, rows, longest):
    """The packed rows as [sequences, longest] row numbers, and which of them exist."""
    at = torch.arange(longest, device="cuda")
    lens = (starts[1:] - starts[:-1]).long()
    return torch.clamp(starts[:-1, None].long() + at, max=rows - 1), at < lens[:, None], lens


def _plain_prompt(s):
    c = s["case"]
    group = c["heads"] // c["kv"]
    qi, qv, lq = _places(s["q_starts"], s["rows"], s["longest"])
    ki, _, lk = _places(s["k_starts"], s["keys"], s["longest_keys"])
    q = s["q"][qi].float().permute(0, 2, 1, 3)  # [seqs, heads, rows, d]
    k = s["k"][ki].float().permute(0, 2, 3, 1).repeat_interleave(group, 1)
    v = s["v"][ki].float().permute(0, 2, 1, 3).repeat_interleave(group, 1)
    i, j = torch.arange(s["longest"], device="cuda"), torch.arange(s["longest_keys"], device="cuda")
    seen = j[None, None, :] <= i[None, :, None] + (lk - lq)[:, None, None]
    p = _softmax(q @ k / math.sqrt(c["d"]), seen[:, None])
    o = (p @ v).permute(0, 2, 1, 3)
    s["out"][qi[qv]] = o[qv].to(s["out"].dtype)


def _plain_tree(s):
    c = s["case"]
    seqs, kv, group, d = c["seqs"], c["kv"], c["heads"] // c["kv"], c["d"]
    qi, qv, n = _places(s["starts"], s["rows"], s["longest"])
    pages = s["tables"].long()

    def positions(pool):  # [seqs, kv, positions, d]
        x = pool[0][pages].permute(0, 2, 1, 3, 4)
        return x.reshape(seqs, kv, -1, d)[:, :, : s["end"]].float()

    at = torch.arange(s["end"], device="cuda")
    context = s["context"].long()[:, None, None]
    node = at[None, None, :] - context  # of a position: below 0 for the cached ones
    bit = s["visible"][qi][:, :, None] >> torch.clamp(node, 0, 63) & 1
    seen = (node < 0) | (node < n[:, None, None]) & (bit == 1)
    q = s["q"][qi].float().reshape(seqs, s["longest"], kv, group, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(seqs, kv, group * s["longest"], d)
    scores = q @ positions(s["k_pool"]).transpose(2, 3) / math.sqrt(d)
    p = _softmax(scores.reshape(seqs, kv, group, s["longest"], -1), seen[:, None, None])
    o = p.reshape(seqs, kv, group * s["longest"], -1) @ torch.where(
        (at < context[:, 0] + n[:, None])[:, None, :, None], positions(s["v_pool"]), 0.0)
    o = o.reshape(seqs, kv, group, s["longest"], d).permute(0, 3, 1, 2, 4).reshape(seqs, s["longest"], kv * group, d)
    s["out"][qi[qv]] = o[qv].to(s["out"].dtype)


def _plain_append(s):
    page = s["case"]["page"]
    _, real, _ = _places(s["starts"], s["rows"], s["longest"])
    seq, i = real.nonzero(as_tuple=True)
    at = s["context"].long()[seq] + i
    ids = s["tables"].long()[seq, at // page]
    s["k_pool"][0, ids, :, at % page] = s["k"]
    s["v_pool"][0, ids, :, at % page] = s["v"]


def _plain_keep(s):
    page = s["case"]["page"]
    rows, _, _ = _places(s["starts"], s["rows"], s["longest"])
    j = torch.arange(s["longest"], device="cuda")
    seq, j = (j < s["counts"].long()[:, None]).nonzero(as_tuple=True)
    new, old = s["context"].long()[seq] + j, s["context"].long()[seq] + s["kept"].long()[rows[seq, j]]
    tables = s["tables"].long()
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, tables[seq, new // page], :, new % page] = pool[:, tables[seq, old // page], :, old % page]
    s["new_context"].copy_(s["context"] + s["counts"])


def _plain_copy(s):
    src, dst = (torch.tensor(ids, device="cuda") for ids in (s["src"], s["dst"]))
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, dst] = pool[:, src]


# ---------------------------------------------------------------- in 64 bits

def _attend(q, k, v, seen):
    """One head: rows of q against k and v, where seen says so."""
    out = torch.zeros_like(q)
    for at in range(0, len(q), 2048):
        mask = seen[at: at + 2048]
        s = (q[at: at + 2048] @ k.T / math.sqrt(q.shape[1])).masked_fill(~mask, -math.inf)
        w = torch.where(mask, torch.exp(s - s.max(1, keepdim=True).values), 0.0)
        o = w @ v / w.sum(1, keepdim=True)
        out[at: at + 2048] = torch.where(mask.any(1, keepdim=True), o, 0.0)
    return out


def exact(case, seed):
    s, dtype = {}, DTYPES[case["dtype"]]
    group = case["heads"] // case["kv"]
    if case["kind"] == "prompt":
        sizes, d = _lengths(case), case["d"]
        rows, keys = sum(n for n, _ in sizes), sum(n + c for n, c in sizes)
        q = _normal((rows, case["heads"], d), dtype, seed, 1).double()
        k = _normal((keys, case["kv"], d), dtype, seed, 2).double()
        v = _normal((keys, case["kv"], d), dtype, seed, 3).double()
        out, a, b = torch.empty_like(q), 0, 0
        for n, c in sizes:
            seen = torch.ones((n, n + c), dtype=torch.bool, device="cuda").tril(c)
            for h in range(case["heads"]):
                out[a: a + n, h] = _attend(q[a: a + n, h], k[b: b + n + c, h // group], v[b: b + n + c, h // group],
                                           seen)
            a, b = a + n, b + n + c
        return out
    if case["kind"] == "copy":
        shape = (LAYERS, case["pool"], case["kv"], case["page"], case["d"])
        pools = [_normal(shape, dtype, seed, i).double() for i in (1, 2)]
        for pool in pools:
            for a, b in zip(*_pairs(case)):
                pool[:, b] = pool[:, a]
        return {"k": pools[0], "v": pools[1]}
    _prepare_batch(s, case, dtype, seed)
    pools, page, tables = [s["k_pool"].double(), s["v_pool"].double()], case["page"], s["tables"].tolist()
    sizes, at, out = _lengths(case), 0, None
    if case["kind"] == "tree":
        out, q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), s["q"].double()
    for i, ((n, c), table) in enumerate(zip(sizes, tables)):
        if case["kind"] == "append":
            for r in range(n):
                for pool, new in zip(pools, (s["k"], s["v"])):
                    pool[0, table[(c + r) // page], :, (c + r) % page] = new[at + r].double()
        elif case["kind"] == "keep":
            path = _trees(case)[i][1]
            for pool in pools:
                old = [pool[:, table[(c + r) // page], :, (c + r) % page].clone() for r in path]
                for j, row in enumerate(old):
                    pool[:, table[(c + j) // page], :, (c + j) % page] = row
        else:
            parents, seen = _trees(case)[i][0], torch.zeros((n, n + c), dtype=torch.bool)
            seen[:, :c] = True
            for r, p in enumerate(parents):
                if p >= 0:
                    seen[r] = seen[p]
                seen[r, c + r] = True
            seen = seen.cuda()
            held = table[: -(-(n + c) // page)]
            for h in range(case["heads"]):
                k, v = (pool[0, held, h // group].reshape(-1, case["d"])[: n + c] for pool in pools)
                out[at: at + n, h] = _attend(q[at: at + n, h], k, v, seen)
        at += n
    if case["kind"] == "tree":
        return out
    answer = {"k": pools[0], "v": pools[1]}
    return {**answer, "context": None} if case["kind"] == "keep" else answer
