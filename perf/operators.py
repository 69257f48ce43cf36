"""The operators of a pass over drafted tokens, as cases that can be measured.

A speculative step of the Qwen3 decoder runs a tree of drafted tokens a
conversation through the target model in one pass, keeps the path the target
agrees with and throws the rest away.  A case is a dict of plain values; `op`
names the operator and the rest its sizes:

  plan       parents -> positions, draft rows, ancestors' bits and the
             rotation rows of every node (gx_qwen_tree_plan): once a pass
  attention  every node against its conversation's cached prefix and its own
             ancestors' draft entries (gx_qwen_attention_tree): once a layer
  verify     the walk down each tree by the target's logits (gx_tree_verify):
             temperature 0 greedy; draft 1: the drafts were drawn from draft
             logits, 0: they are given tokens
  commit     the kept path's keys and values from the draft buffers into the
             caches, every layer (gx_qwen_cache_commit)
  fork       a conversation's first positions into other slots, every layer
             (gx_qwen_cache_fork)

n trees (conversations) have up to `nodes` nodes, the first that many and the
others fewer; prefixes are up to `prefix`, the first that long.  fanout 1 is a
chain of drafts, more a tree whose nodes have about that many children.
"""
import ctypes
import math

import torch

own = False

QWEN = {"heads": 32, "kv_heads": 8, "head_dim": 128}
VOCAB = 151936
LAYERS = 36
ROPE_BASE = 1e6


def listed():
    return [
        # one conversation's short chain: the least a pass plans
        {"name": "plan_chain", "op": "plan", "n": 1, "nodes": 6, "fanout": 1, "prefix": 300, "context": 640,
         "head_dim": 128},
        # a server's batch of slots, a large tree each
        {"name": "plan_slots", "op": "plan", "n": 16, "nodes": 63, "fanout": 3, "prefix": 4000, "context": 4096,
         "head_dim": 128},
        # five drafts after a chat turn: a layer's attention at its launch latency
        dict(QWEN, name="attention_chain", op="attention", n=1, nodes=5, fanout=1, prefix=500),
        # eight conversations' trees, ragged
        dict(QWEN, name="attention_slots", op="attention", n=8, nodes=33, fanout=3, prefix=1500),
        # a wide tree far into a document
        dict(QWEN, name="attention_long", op="attention", n=1, nodes=64, fanout=4, prefix=32000),
        # greedy decoding with a chain looked up in the prompt
        {"name": "verify_greedy", "op": "verify", "n": 1, "nodes": 8, "fanout": 1, "vocab": VOCAB, "temperature": 0.0,
         "draft": 0},
        # eight conversations sampling, chains from a draft model
        {"name": "verify_chains", "op": "verify", "n": 8, "nodes": 6, "fanout": 1, "vocab": VOCAB, "temperature": 0.8,
         "draft": 1},
        # a batch of trees from a draft model
        {"name": "verify_trees", "op": "verify", "n": 4, "nodes": 33, "fanout": 3, "vocab": VOCAB, "temperature": 1.0,
         "draft": 1},
        # one conversation keeps three nodes, in all 36 layers
        {"name": "commit_one", "op": "commit", "layers": LAYERS, "n": 1, "nodes": 8, "accepted": 3, "prefix": 600,
         "kv_heads": 8, "head_dim": 128},
        # sixteen conversations keep up to twelve
        {"name": "commit_slots", "op": "commit", "layers": LAYERS, "n": 16, "nodes": 33, "accepted": 12,
         "prefix": 500, "kv_heads": 8, "head_dim": 128},
        # a short common prompt given to a second conversation
        {"name": "fork_one", "op": "fork", "layers": LAYERS, "n": 1, "len": 301, "context": 640, "kv_heads": 8,
         "head_dim": 128},
        # a long one given to four
        {"name": "fork_four", "op": "fork", "layers": LAYERS, "n": 4, "len": 1999, "context": 2048, "kv_heads": 8,
         "head_dim": 128},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "attention", "attention", "attention", "verify", "verify", "commit", "fork"])
    fanout = rng.choice([1, 2, 3, 5])
    if op == "plan":
        prefix = _log(rng, 1, 4000)
        return {"op": op, "n": _log(rng, 1, 16), "nodes": _log(rng, 1, 63), "fanout": fanout, "prefix": prefix,
                "context": prefix + 64, "head_dim": rng.choice([64, 128])}
    if op == "attention":
        heads, kv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (16, 8, 128), (8, 2, 64), (4, 2, 32), (12, 4, 96)])
        n = _log(rng, 1, 12)
        return {"op": op, "heads": heads, "kv_heads": kv, "head_dim": hd, "n": n, "nodes": _log(rng, 1, 64),
                "fanout": fanout, "prefix": rng.choice([0] + 7 * [_log(rng, 1, 32000 // n)])}
    if op == "verify":
        n = _log(rng, 1, 8)
        return {"op": op, "n": n, "nodes": _log(rng, 1, 100 // n), "fanout": fanout,
                "vocab": _log(rng, 1024, VOCAB), "temperature": rng.choice([0.0, 0.6, 1.0, 1.3]),
                "draft": rng.choice([0, 1])}
    kv, hd = rng.choice([(8, 128), (2, 64), (4, 96)])
    if op == "commit":
        nodes = _log(rng, 2, 33)
        return {"op": op, "layers": rng.randint(1, LAYERS), "n": _log(rng, 1, 16), "nodes": nodes,
                "accepted": _log(rng, 1, min(nodes, 12)), "prefix": _log(rng, 1, 500), "kv_heads": kv, "head_dim": hd}
    length = _log(rng, 1, 1999)
    return {"op": op, "layers": rng.randint(1, LAYERS), "n": rng.randint(1, 4), "len": length,
            "context": (length + rng.randint(1, 48) + 7) // 8 * 8, "kv_heads": kv, "head_dim": hd}


def _sizes(case):
    t = case["nodes"]
    return [max(1, t - 5 * b % (t // 2 + 1)) for b in range(case["n"])]


def _prefixes(case):
    p = case["prefix"]
    return [p - 37 * b % (p // 2 + 1) for b in range(case["n"])]


def _accepted(case):
    return [max(1, min(case["accepted"] - b % (case["accepted"] // 2 + 1), t)) for b, t in enumerate(_sizes(case))]


# ---- inputs -------------------------------------------------------------------


def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) * 1000003 + 29)
    return g


def _dev(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _half(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)


def _parents(case, seed):
    """A parent (an earlier node of its tree) for every node, -1 for a root:
    each takes one of the nodes about nodes / fanout before it, so that a node
    has about `fanout` children; a chain where fanout is 1."""
    g = _gen(seed, "cpu")
    out = []
    for t in _sizes(case):
        i = torch.arange(1, t)
        if case["fanout"] == 1:
            p = i - 1
        else:
            p = ((i - 1) / case["fanout"] + torch.rand(len(i), generator=g)).long().clamp(max=t)
            p = torch.minimum(p, i - 1)
        out += [-1] + p.tolist()
    return out


def _offsets(sizes):
    at = [0]
    for t in sizes:
        at.append(at[-1] + t)
    return at


def _logits(g, rows, vocab):
    """Rows of logits as a model answers them: a broad floor, a few tokens far
    above it, differently peaked from row to row."""
    x = 1.5 * torch.randn((rows, vocab), generator=g, device="cuda")
    k = min(24, vocab)
    at = torch.randint(0, vocab, (rows, k), generator=g, device="cuda")
    peak = 8.0 + 10.0 * torch.rand((rows, k), generator=g, device="cuda")
    return x.scatter_(1, at, peak)


def _drafted(g, parents, first, logits, temperature, drawn):
    """Each node's token, from its parent's row of draft logits: siblings take
    different ones, drawn without replacement (the order of logits plus Gumbel
    noise) or the most likely in order."""
    if drawn:
        u = torch.rand(logits.shape, generator=g, device="cuda", dtype=torch.float64).clamp_(1e-300)
        order = logits.double() / temperature - (-u.log()).log()
    else:
        order = logits
    rank, seen, up = [], {}, []
    for b in range(len(first) - 1):
        for m in range(first[b], first[b + 1]):
            v = first[b] + parents[m] if parents[m] >= 0 else first[b]
            rank.append(seen.get(v, 0) if parents[m] >= 0 else 0)
            if parents[m] >= 0:
                seen[v] = seen.get(v, 0) + 1
            up.append(v)
    top = order.topk(min(max(seen.values(), default=1), logits.shape[1]), dim=1).indices
    at = _dev(rank, torch.int64).clamp(max=top.shape[1] - 1)
    return top[_dev(up, torch.int64), at].to(torch.int32), max(seen.values(), default=0)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = {"case": case}
    if op == "fork":
        l, n, kv, hd, ctx = case["layers"], case["n"], case["kv_heads"], case["head_dim"], case["context"]
        s["kc"], s["vc"] = _half(g, l, n + 1, kv, hd // 8, ctx, 8), _half(g, l, n + 1, kv, hd, ctx)
        # the conversation sits in the middle of the slots
        s["src"], s["dsts"] = n // 2, [i for i in range(n + 1) if i != n // 2]
        s["layers"] = [_pointers(s[k]) for k in ("kc", "vc")]
        s["slots"] = (ctypes.c_int32 * n)(*s["dsts"])
        return s
    sizes = _sizes(case)
    first, n, t = _offsets(sizes), case["n"], case["nodes"]
    m = first[-1]
    parents = _parents(case, seed) if "fanout" in case else None
    s["first"], s["m"] = _dev(first), m
    if parents:
        s["parents"] = _dev(parents)
    if "prefix" in case:
        s["prefix"] = _dev(_prefixes(case))
    if op == "plan":
        s["prefix"] -= (s["prefix"] * torch.rand(n, generator=g, device="cuda")).int()
        half = case["head_dim"] // 2
        freq = ROPE_BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        theta = torch.arange(case["context"], dtype=torch.float64, device="cuda")[:, None] * freq
        s["cos"], s["sin"] = theta.cos().float(), theta.sin().float()
        s["out"] = {"rows": torch.empty(m, dtype=torch.int32, device="cuda"),
                    "positions": torch.empty(m, dtype=torch.int32, device="cuda"),
                    "mask": torch.empty((m, (t + 31) // 32), dtype=torch.int32, device="cuda"),
                    "cos": torch.empty((m, half), device="cuda"), "sin": torch.empty((m, half), device="cuda")}
    elif op == "attention":
        h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        ctx, dctx = (case["prefix"] + t + 7) // 8 * 8, (m + 7) // 8 * 8
        s["context"], s["draft_context"] = ctx, dctx
        s["qh"] = (2.0 * _half(g, m, h * hd))
        s["kc"], s["vc"] = _half(g, n, kv, hd // 8, ctx, 8), _half(g, n, kv, hd, ctx)
        s["kd"], s["vd"] = _half(g, kv, hd // 8, dctx, 8), _half(g, kv, hd, dctx)
        s["mask"] = _dev(_mask_words(parents, first, t))
        # the trees' conversations, in an order of their own
        s["slots"] = torch.randperm(n, generator=_gen(seed, "cpu")).to(torch.int32).cuda()
        s["out"] = torch.empty((m, h * hd), device="cuda")
    elif op == "verify":
        v = case["vocab"]
        s["logits"] = _logits(g, m, v)
        draft = s["logits"] + 1.0 * torch.randn((m, v), generator=g, device="cuda")
        s["tokens"], s["kids"] = _drafted(g, parents, first, draft, max(case["temperature"], 0.1), case["draft"])
        s["draft"] = draft if case["draft"] else None
        s["uniforms"] = torch.rand(m, generator=g, device="cuda")
        s["path"] = torch.empty((n, t), dtype=torch.int32, device="cuda")
        s["counts"], s["next"] = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
    else:
        l, kv, hd = case["layers"], case["kv_heads"], case["head_dim"]
        ctx, dctx = (case["prefix"] + t + 7) // 8 * 8, (m + 7) // 8 * 8
        s["context"], s["draft_context"] = ctx, dctx
        s["kc"], s["vc"] = _half(g, l, n, kv, hd // 8, ctx, 8), _half(g, l, n, kv, hd, ctx)
        s["kd"], s["vd"] = _half(g, l, kv, hd // 8, dctx, 8), _half(g, l, kv, hd, dctx)
        s["layers"] = [_pointers(s[k]) for k in ("kc", "vc", "kd", "vd")]
        cg = _gen(seed, "cpu")
        counts, path = _accepted(case), torch.full((n, t), -1, dtype=torch.int32)
        for b in range(n):  # a root and later nodes, in order
            kept = 1 + torch.randperm(sizes[b] - 1, generator=cg)[:counts[b] - 1].sort().values
            path[b, :counts[b]] = torch.cat([torch.zeros(1, dtype=torch.int64), kept])
        s["path"], s["counts"] = path.cuda(), _dev(counts)
        s["slots"] = torch.randperm(n, generator=cg).to(torch.int32).cuda()
    return s


def _pointers(x):
    """The layers' device addresses, as an engine that holds a tensor a layer lists them."""
    return (ctypes.c_void_p * len(x))(*[t.data_ptr() for t in x])


def _mask_words(parents, first, t):
    """The plan's bits: bit j of a node's words is set where node j is itself or an ancestor."""
    words, out = (t + 31) // 32, []
    for b in range(len(first) - 1):
        bits = []
        for i, p in enumerate(parents[first[b]:first[b + 1]]):
            bits.append((1 << i) | (bits[p] if p >= 0 else 0))
        for x in bits:
            row = [(x >> 32 * w) & 0xFFFFFFFF for w in range(words)]
            out.append([w - (1 << 32) if w >> 31 else w for w in row])
    return out


# ---- the framework's calls ------------------------------------------------------

_kept = {}  # what a program holds as long as it runs: the context, and a workspace that grows


def _handle():
    from golem_amd import capi
    if "ctx" not in _kept:
        _kept["ctx"] = capi.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    return capi, _kept["ctx"].ptr


def _workspace(capi, *size):
    if size not in _kept:
        _kept[size] = (capi.size_out(*size) + 255) // 256 * 256
    need = _kept[size]
    if "ws" not in _kept or _kept["ws"].numel() < need:
        _kept["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    return _kept["ws"].data_ptr(), _kept["ws"].numel()


def _run_own(s):
    capi, ctx = _handle()
    case, call = s["case"], capi.call
    op, n = case["op"], case["n"]

    def p(k):
        return None if s[k] is None else s[k].data_ptr()

    if op == "plan":
        o = s["out"]
        call("gx_qwen_tree_plan", ctx, n, s["m"], case["nodes"], p("first"), p("parents"), p("prefix"), p("cos"),
             p("sin"), case["head_dim"] // 2, case["context"], o["rows"].data_ptr(), o["positions"].data_ptr(),
             o["mask"].data_ptr(), o["cos"].data_ptr(), o["sin"].data_ptr())
        return o
    if op == "attention":
        ws, size = _workspace(capi, "gx_qwen_attention_tree_workspace_bytes", n, s["m"], case["nodes"], case["heads"],
                              case["kv_heads"], case["head_dim"], case["prefix"])
        call("gx_qwen_attention_tree", ctx, p("qh"), n, s["m"], case["nodes"], p("first"), p("mask"), p("prefix"),
             case["prefix"], case["heads"], case["kv_heads"], case["head_dim"], p("kc"), p("vc"), s["context"],
             p("kd"), p("vd"), s["draft_context"], p("out"), None, None, None, ws, size, p("slots"), n)
        return s["out"]
    if op == "verify":
        ws, size = _workspace(capi, "gx_tree_verify_workspace_bytes", n, s["m"], case["vocab"])
        call("gx_tree_verify", ctx, p("logits"), case["vocab"], n, s["m"], case["nodes"], case["vocab"], p("first"),
             p("parents"), p("tokens"), p("draft"), case["vocab"], case["temperature"], case["temperature"],
             p("uniforms"), p("path"), p("counts"), p("next"), ws, size)
        return {k: s[k] for k in ("path", "counts", "next")}
    if op == "commit":
        call("gx_qwen_cache_commit", ctx, case["layers"], *s["layers"], n, s["m"], case["nodes"], p("first"),
             p("path"), p("counts"), p("prefix"), case["kv_heads"], case["head_dim"], s["context"],
             s["draft_context"], p("slots"), n)
    else:
        call("gx_qwen_cache_fork", ctx, case["layers"], *s["layers"], n + 1, case["kv_heads"], case["head_dim"],
             case["context"], s["src"], s["slots"], n, case["len"])
    return {"kc": s["kc"], "vc": s["vc"]}


# ---- the plain forms --------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    return {"plan": _plan, "attention": _attention, "verify": _verify, "commit": _commit, "fork": _fork}[
        s["case"]["op"]](s)


def _nodes(s):
    """Each token's tree and its index there."""
    m = torch.arange(s["m"], dtype=torch.int32, device="cuda")
    tree = torch.searchsorted(s["first"][1:].contiguous(), m, right=True)
    return m.long(), tree, (m - s["first"][tree]).long()


def _ancestors(s, tree, i):
    """(depth, [m][nodes] truth: node j is token m's self or ancestor), by
    doubling the step up the tree; a last row stands for what is above a root."""
    m, t = s["m"], s["case"]["nodes"]
    up = torch.where(s["parents"] < 0, torch.full_like(s["parents"], m), s["first"][tree] + s["parents"]).long()
    up = torch.cat([up, up.new_full((1,), m)])
    depth = (up < m).long()
    anc = torch.zeros((m + 1, t), dtype=torch.bool, device="cuda")
    anc[:m] = torch.arange(t, device="cuda") == i[:, None]
    for _ in range(max(t - 1, 1).bit_length()):
        anc, depth, up = anc | anc[up], depth + depth[up], up[up]
    return depth[:m], anc[:m]


def _plan(s):
    m, tree, i = _nodes(s)
    depth, anc = _ancestors(s, tree, i)
    pos = s["prefix"][tree].long() + depth
    words = (s["case"]["nodes"] + 31) // 32
    bits = torch.zeros((s["m"], words * 32), dtype=torch.int64, device="cuda")
    bits[:, :anc.shape[1]] = anc
    value = (bits.view(-1, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    return {"rows": m.int(), "positions": pos.int(), "mask": torch.where(value >= 1 << 31, value - (1 << 32), value).int(),
            "cos": s["cos"][pos], "sin": s["sin"][pos]}


def _attention(s):
    case = s["case"]
    n, t, h, kv, hd = (case[k] for k in ("n", "nodes", "heads", "kv_heads", "head_dim"))
    m, tree, i = _nodes(s)
    at = torch.zeros((n, t), dtype=torch.int64, device="cuda")
    at[tree, i] = m
    q = s["qh"].float()[at].view(n, t, kv, h // kv, hd).transpose(1, 2).reshape(n, kv, t * (h // kv), hd)
    slots, p = s["slots"].long(), case["prefix"]
    kd = s["kd"].permute(2, 0, 1, 3).reshape(-1, kv, hd)[at].transpose(1, 2)
    vd = s["vd"].permute(2, 0, 1)[at].transpose(1, 2)
    k = torch.cat([s["kc"][slots, :, :, :p].permute(0, 1, 3, 2, 4).reshape(n, kv, p, hd), kd], 2).float()
    v = torch.cat([s["vc"][slots, :, :, :p].transpose(2, 3), vd], 2).float()
    sees = torch.zeros((n, t, p + t), dtype=torch.bool, device="cuda")
    sees[:, :, :p] = (torch.arange(p, device="cuda") < s["prefix"][:, None])[:, None]
    bit = torch.arange(t, device="cuda")
    sees[tree, i, p:] = (s["mask"][:, bit // 32] >> (bit % 32) & 1).bool()
    sees = sees.repeat_interleave(h // kv, 1)[:, None]
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))
    score = torch.where(sees, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    e = torch.where(sees, (score - top).exp(), torch.zeros_like(score))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.view(n, kv, t, h // kv, hd).transpose(1, 2).reshape(n, t, h * hd)
    return o[tree, i]


def _softmax(x, temperature):
    x = x.double() / temperature
    e = (x - x.amax(-1, keepdim=True)).exp()
    return e / e.sum(-1, keepdim=True)


def _verify(s):
    case, (m, tree, i) = s["case"], _nodes(s)
    n, t, count = case["n"], case["nodes"], s["m"]
    parent = s["parents"].long()
    up = torch.where(parent < 0, torch.full_like(parent, count), s["first"][tree].long() + parent)
    rank = ((up[:, None] == up[None, :]) & (m[None, :] < m[:, None])).sum(1)
    # kid[v][r]: node v's child r, `count` where it has none
    kid = torch.full((count + 1, s["kids"] + 1), count, dtype=torch.int64, device="cuda")
    kid[up, rank.clamp(max=s["kids"])] = m
    kid = kid[:count, :s["kids"]]
    token = torch.cat([s["tokens"].long(), s["tokens"].new_zeros(1).long()])
    taken = torch.full((count,), -1, dtype=torch.int64, device="cuda")
    temperature = case["temperature"]
    if temperature == 0:
        x = s["logits"]
        col = torch.arange(x.shape[1], device="cuda")
        pick = torch.where(x == x.amax(1, keepdim=True), col, col.new_full((1,), x.shape[1])).amin(1)
        hit = (kid < count) & (token[kid] == pick[:, None])
        r = torch.arange(s["kids"], device="cuda").expand_as(hit)
        if s["kids"]:
            first = torch.where(hit, r, r + s["kids"]).amin(1)
            taken = torch.where(first < s["kids"], first, taken)
    else:
        p = _softmax(s["logits"], temperature)
        q = _softmax(s["draft"], temperature) if s["draft"] is not None else None
        u = torch.cat([s["uniforms"], s["uniforms"].new_zeros(1)]).double()
        c, tried = torch.zeros(count, dtype=torch.float64, device="cuda"), torch.zeros_like(u[:count])
        mass = torch.ones_like(c)
        before = torch.zeros((count, s["kids"]), dtype=torch.bool, device="cuda")  # children that were turned down
        for r in range(s["kids"]):
            has = (kid[:, r] < count) & (taken < 0)
            x = token[kid[:, r]]
            again = (before & (token[kid] == x[:, None])).any(1)
            px = p.gather(1, x[:, None])[:, 0]
            if q is None:
                px = torch.where(again, torch.zeros_like(px), px)
                yes = has & (u[kid[:, r]] * mass < px)
            else:
                qx, left = q.gather(1, x[:, None])[:, 0], 1.0 - tried
                px = torch.where(again, torch.zeros_like(px), (px - c * qx).clamp(min=0))
                can = has & (left > 0) & (mass > 0)
                yes = can & (u[kid[:, r]] * mass * qx < px * left)
                has = can
            no = has & ~yes
            taken = torch.where(yes, torch.full_like(taken, r), taken)
            before[:, r] = no
            if q is None:
                mass = torch.where(no, mass - px, mass)
            else:
                c = torch.where(no, c + mass / left, c)
                tried = torch.where(no, tried + qx, tried)
                mass = torch.where(no, (p - c[:, None] * q).clamp(min=0).sum(1), mass)
    taken = torch.cat([taken, taken.new_full((1,), -2)])
    chosen = (parent < 0) | (taken[up] == rank)
    _, anc = _ancestors(s, tree, i)
    # a node is kept where every ancestor and itself was chosen
    picked = torch.zeros((n, t), dtype=torch.bool, device="cuda")
    picked[tree, i] = chosen
    kept = ~(anc & ~picked[tree]).any(1)
    grid = torch.zeros((n, t), dtype=torch.int64, device="cuda")
    grid[tree, i] = kept.long()
    counts = grid.sum(1)
    order = torch.where(grid > 0, grid.cumsum(1) - 1, torch.full_like(grid, t))
    path = torch.full((n, t + 1), -1, dtype=torch.int64, device="cuda")
    path.scatter_(1, order, torch.arange(t, device="cuda").expand(n, t).contiguous())
    path = path[:, :t].scatter(1, counts[:, None].clamp(max=t - 1), torch.where(
        counts < t, torch.full_like(counts, -1), path[:, t - 1])[:, None])
    last = s["first"][:-1].long() + path.gather(1, counts[:, None] - 1)[:, 0]
    if temperature == 0:
        nxt = pick[last]
    else:
        w = p[last]
        if q is not None:
            rest = (w - c[last][:, None] * q[last]).clamp(min=0)
            w = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
        elif s["kids"]:
            rest = torch.ones_like(w)
            rest.scatter_reduce_(1, token[kid[last]], (~before[last]).double(), "amin")
            rest = w * rest
            w = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
        cum = w.cumsum(1)
        aim = s["uniforms"][s["first"][:-1].long()].double() * cum[:, -1]
        nxt = torch.searchsorted(cum, aim[:, None], right=True)[:, 0].clamp(max=w.shape[1] - 1)
    return {"path": path.int(), "counts": counts.int(), "next": nxt.int()}


def _commit(s):
    case = s["case"]
    n, t = case["n"], case["nodes"]
    j = torch.arange(t, device="cuda").expand(n, t)
    keep = (j < s["counts"][:, None]).reshape(-1)
    src = (s["first"][:-1, None] + s["path"].clamp(min=0)).long().reshape(-1)
    pos = (s["prefix"][:, None] + j).long().reshape(-1)
    slot = s["slots"].long()[:, None].expand(n, t).reshape(-1)
    k, v = s["kc"].permute(1, 4, 0, 2, 3, 5), s["vc"].permute(1, 4, 0, 2, 3)
    kd, vd = s["kd"].permute(3, 0, 1, 2, 4)[src], s["vd"].permute(3, 0, 1, 2)[src]
    k[slot, pos] = torch.where(keep.view(-1, 1, 1, 1, 1), kd, k[slot, pos])
    v[slot, pos] = torch.where(keep.view(-1, 1, 1, 1), vd, v[slot, pos])
    return {"kc": s["kc"], "vc": s["vc"]}


def _fork(s):
    src, length = s["src"], s["case"]["len"]
    dsts = torch.arange(s["case"]["n"], device="cuda")
    dsts = dsts + (dsts >= src)
    s["kc"][:, dsts, :, :, :length] = s["kc"][:, src:src + 1, :, :, :length]
    s["vc"][:, dsts, :, :, :length] = s["vc"][:, src:src + 1, :, :, :length]
    return {"kc": s["kc"], "vc": s["vc"]}


# ---- what one pass has to move and compute ----------------------------------------


def work(case):
    op, n = case["op"], case["n"]
    if op == "fork":
        one = case["layers"] * case["kv_heads"] * case["head_dim"] * case["len"] * 2 * 2
        return {"bytes": one * (1 + n), "flops": 0}
    sizes = _sizes(case)
    m, t = sum(sizes), case["nodes"]
    if op == "plan":
        half, words = case["head_dim"] // 2, (t + 31) // 32
        return {"bytes": m * (4 + 8 + 4 * words + 16 * half) + 8 * n, "flops": 0}
    if op == "attention":
        h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        pre = _prefixes(case)
        keys = sum(pre) + m
        return {"bytes": keys * kv * hd * 4 + m * h * hd * (2 + 4) + 4 * m * ((t + 31) // 32),
                "flops": 4 * h * hd * sum(x * (p + (x + 1) / 2) for x, p in zip(sizes, pre))}
    if op == "verify":
        rows = m * (2 if case["draft"] and case["temperature"] > 0 else 1)
        return {"bytes": rows * case["vocab"] * 4 + 4 * (3 * m + n * t), "flops": 2 * rows * case["vocab"]}
    return {"bytes": sum(_accepted(case)) * case["layers"] * case["kv_heads"] * case["head_dim"] * 2 * 2 * 2, "flops": 0}


# ---- the definitions in 64 bits ---------------------------------------------------


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "fork":
        kc, vc = s["kc"].clone(), s["vc"].clone()
        for d in s["dsts"]:
            for x in range(case["len"]):
                kc[:, d, :, :, x] = s["kc"][:, s["src"], :, :, x]
                vc[:, d, :, :, x] = s["vc"][:, s["src"], :, :, x]
        return {"kc": kc, "vc": vc}
    first = s["first"].tolist()
    pre = s["prefix"].tolist() if "prefix" in s else None  # (a plan's are drawn)
    if op == "commit":
        kc, vc = s["kc"].clone(), s["vc"].clone()
        for b, slot in enumerate(s["slots"].tolist()):
            for j in range(int(s["counts"][b])):
                row = first[b] + int(s["path"][b, j])
                kc[:, slot, :, :, pre[b] + j] = s["kd"][:, :, :, row]
                vc[:, slot, :, :, pre[b] + j] = s["vd"][:, :, :, row]
        return {"kc": kc, "vc": vc}
    if op == "attention":
        h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        out = torch.zeros((s["m"], h, hd), dtype=torch.float64, device="cuda")
        words = s["mask"].tolist()
        for b, slot in enumerate(s["slots"].tolist()):
            kp = s["kc"][slot, :, :, :pre[b]].double().transpose(1, 2).reshape(kv, pre[b], hd)
            vp = s["vc"][slot, :, :, :pre[b]].double().transpose(1, 2)
            for m in range(first[b], first[b + 1]):
                on = [first[b] + j for j in range(first[b + 1] - first[b]) if words[m][j // 32] >> (j % 32) & 1]
                k = torch.cat([kp, s["kd"][:, :, on].double().transpose(1, 2).reshape(kv, len(on), hd)], 1)
                v = torch.cat([vp, s["vd"][:, :, on].double().transpose(1, 2)], 1)
                q = s["qh"][m].double().view(kv, h // kv, 1, hd)
                w = torch.softmax((q * k[:, None]).sum(-1) / math.sqrt(hd), -1) if k.shape[1] < 4096 else torch.softmax(
                    torch.bmm(q[:, :, 0], k.transpose(1, 2).contiguous()) / math.sqrt(hd), -1)
                out[m] = torch.bmm(w, v.contiguous()).reshape(h, hd)
        return out.view(s["m"], h * hd)
    parents = s["parents"].tolist()
    if op == "plan":
        rows, positions, mask = [], [], _mask_words(parents, first, case["nodes"])
        for b in range(case["n"]):
            for i in range(first[b + 1] - first[b]):
                d, x = 0, i
                while parents[first[b] + x] >= 0:
                    d, x = d + 1, parents[first[b] + x]
                rows.append(first[b] + i)
                positions.append(pre[b] + d)
        return {"rows": _dev(rows), "positions": _dev(positions), "mask": _dev(mask),
                "cos": s["cos"].cpu().double()[positions], "sin": s["sin"].cpu().double()[positions]}
    return _exact_verify(case, s, first, parents)


def _exact_verify(case, s, first, parents):
    """The walk as it is defined, a node and a child at a time: the chance of
    each further child from what is left of the target's distribution."""
    n, t, temperature = case["n"], case["nodes"], case["temperature"]
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    path = torch.full((n, t), -1, dtype=torch.int32)
    counts, nxt = [], []

    def chances(x):
        return torch.softmax(x.cpu().double() / temperature, 0)

    for b in range(n):
        kept, v = [0], first[b]
        while True:
            kids = [m for m in range(first[b] + 1, first[b + 1]) if first[b] + parents[m] == v]
            go = None
            if temperature == 0:
                best = int(s["logits"][v].cpu().argmax())
                go = next((m for m in kids if tokens[m] == best), None)
            else:
                p = chances(s["logits"][v])
                left = p.clone()
                q = chances(s["draft"][v]) if s["draft"] is not None else None
                for m in kids:
                    x = tokens[m]
                    if q is None:
                        if u[m] * float(left.sum()) < float(left[x]):
                            go = m
                            break
                        left[x] = 0
                    else:
                        total = float(left.sum())
                        if float(q.sum()) <= 0 or total <= 0:
                            break
                        q = q / q.sum()
                        if u[m] * float(q[x]) * total < float(left[x]):
                            go = m
                            break
                        left = (left - total * q).clamp(min=0)
                        q[x] = 0
            if go is None:
                break
            kept.append(go - first[b])
            v = go
        if temperature == 0:
            nxt.append(best)
        else:
            if float(left.sum()) <= 0:
                left = p
            cum = left.cumsum(0)
            nxt.append(int((cum <= u[first[b]] * float(cum[-1])).sum().clamp(max=len(cum) - 1)))
        counts.append(len(kept))
        path[b, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
    return {"path": path, "counts": _dev(counts), "next": _dev(nxt)}
