"""Performance cases of the operators that a serving step with drafted tokens
takes beside attention over a cache: verification of the drafts against the
target's probabilities, the pages of a cache (forked, freed, copied, compacted),
rotary positions of several axes, and a cache in 8 bits with a scale for each
block of keys.

A case is one call, or the run of calls that belong together, as a serving
program makes it through `frisk_amd.runtime`.  `run` computes it with those
calls where `own` is true and from elementary torch operations where it is
false, in 32 bits, or in 64 where a choice hangs on it (probabilities next to
a random number, angles).

Fields of a case (all plain values):
  op "verify":  batch, tokens (nodes of a tree, the root among them), branch
                (children of a node, 1: a chain), vocab, dtype (logits), dense
                (draft probabilities given), greedy (temperature 0), ragged
  op "axes":    batch, seq, heads, kv_heads, head_dim, rot_dim, dtype, axes,
                interleaved, backward, dealt (axes in turn over the pairs)
  op "pages":   batch, max_pages, page, pages (of the cache), forks (sequences
                that continue another one), ended (sequences that end)
  op "copy":    pairs, kv_heads, page, head_dim, kind, block, part (filled rows only)
  op "compact": batch, tokens, taken, kv_heads, head_dim, kind, page, ctx
  op "cache":   batch, tokens, kv_heads, head_dim, dtype, kind, page, block
                (keys a scale), ctx, ragged
  op "attn":    batch, heads, kv_heads, tokens, head_dim, dtype, kind, page,
                block, ctx, ragged, tree; the new keys are appended first
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1, "i8": 1}
TOP = {"e4m3": 448.0, "i8": 127.0}
TINY = 2.0 ** -126
BASE = 10000.0


def _verify(name, batch, tokens, branch, vocab, dtype, dense=False, greedy=False, ragged=False):
    return {"name": name, "op": "verify", "batch": batch, "tokens": tokens, "branch": branch,
            "vocab": vocab, "dtype": dtype, "dense": dense, "greedy": greedy, "ragged": ragged}


def _axes(name, batch, seq, heads, kv_heads, head_dim, rot_dim, dtype, axes, interleaved=False,
          backward=False, dealt=False):
    return {"name": name, "op": "axes", "batch": batch, "seq": seq, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "rot_dim": rot_dim, "dtype": dtype,
            "axes": axes, "interleaved": interleaved, "backward": backward, "dealt": dealt}


def _pages(name, batch, max_pages, page, pages, forks, ended):
    return {"name": name, "op": "pages", "batch": batch, "max_pages": max_pages, "page": page,
            "pages": pages, "forks": forks, "ended": ended}


def _copy(name, pairs, kv_heads, page, head_dim, kind, block, part):
    return {"name": name, "op": "copy", "pairs": pairs, "kv_heads": kv_heads, "page": page,
            "head_dim": head_dim, "kind": kind, "block": block, "part": part}


def _compact(name, batch, tokens, taken, kv_heads, head_dim, kind, page, ctx):
    return {"name": name, "op": "compact", "batch": batch, "tokens": tokens, "taken": taken,
            "kv_heads": kv_heads, "head_dim": head_dim, "kind": kind, "page": page, "ctx": ctx}


def _cache(name, batch, tokens, kv_heads, head_dim, dtype, kind, page, block, ctx, ragged=False):
    return {"name": name, "op": "cache", "batch": batch, "tokens": tokens, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "kind": kind, "page": page, "block": block,
            "ctx": ctx, "ragged": ragged}


def _attn(name, batch, heads, kv_heads, tokens, head_dim, dtype, kind, page, block, ctx,
          ragged=False, tree=False):
    return {"name": name, "op": "attn", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "tokens": tokens, "head_dim": head_dim, "dtype": dtype, "kind": kind, "page": page,
            "block": block, "ctx": ctx, "ragged": ragged, "tree": tree}


def listed():
    return [
        # One sequence's next token drawn from its logits: latency.
        _verify("verify_token_bf16", 1, 1, 1, 32000, "bf16"),
        # Short chains of a draft model with its probabilities, in f32, an odd vocabulary.
        _verify("verify_chain_f32", 16, 6, 1, 50257, "f32", dense=True, ragged=True),
        # Drafted trees of a serving batch over a large vocabulary.
        _verify("verify_tree_bf16", 8, 64, 2, 131072, "bf16"),
        # A prompt with video: positions in time, height and width.
        _axes("axes_video_bf16", 1, 8192, 32, 8, 128, 128, "bf16", 3),
        # The gradient over images, part of an odd head rotated, in f32.
        _axes("axes_image_grad_f32", 3, 1111, 12, 3, 80, 48, "f32", 2, backward=True, dealt=True),
        # A step of a serving batch: some sequences fork, some end, all grow.
        _pages("pages_step", 64, 512, 16, 40000, 16, 8),
        # Forked sequences get their own last pages, a layer of an 8-bit cache.
        _copy("pages_copy_e4m3", 500, 8, 64, 128, "e4m3", 1, True),
        # The accepted branches of a batch's trees move behind their contexts.
        _compact("compact_tree_bf16", 32, 64, 6, 8, 128, "bf16", 64, 4000),
        # Prompts into int8 pages with a scale for 32 keys, from within a block on.
        _cache("block_prompt_i8", 4, 8192, 8, 128, "bf16", "i8", 64, 32, 77),
        # A decode step of a serving batch: one token appended, then attended.
        _attn("block_token_e4m3", 16, 32, 8, 1, 128, "bf16", "e4m3", 64, 64, 8191, ragged=True),
        # Drafted trees over long contexts.
        _attn("block_tree_e4m3", 8, 32, 8, 64, 128, "bf16", "e4m3", 128, 64, 16384, tree=True),
        # A ragged chunk of a prompt, f16 queries over int8, a scale for 16 keys.
        _attn("block_chunk_i8", 3, 8, 8, 311, 64, "f16", "i8", 16, 16, 5001, ragged=True),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo .. hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    op = rng.choice(["verify", "verify", "axes", "pages", "copy", "compact", "cache", "attn", "attn"])
    if op == "verify":
        dtype = rng.choice(["bf16", "f16", "f32"])
        vocab = _spread(rng, 500, 131072)
        dense = rng.random() < 0.4
        rows = max(1, int(1.3e8 / (vocab * (BYTES[dtype] + (4 if dense else 0)))))
        tokens = _spread(rng, 1, min(rows, 12 if dense else 64))
        return _verify(None, _spread(rng, 1, max(1, min(64, rows // tokens))), tokens,
                       rng.choice([1, 2, 3]), vocab, dtype, dense, rng.random() < 0.2,
                       rng.random() < 0.4)
    if op == "axes":
        dtype = rng.choice(["bf16", "f16", "f32"])
        head = rng.choice([64, 80, 96, 128])
        rot = head if rng.random() < 0.6 else 2 * rng.randint(6, head // 2)
        kv = rng.choice([1, 2, 3, 8])
        heads = kv * rng.choice([1, 2, 4, 7])
        rows = max(1, int(8.0e7 / ((heads + kv) * head * BYTES[dtype])))
        tokens = _spread(rng, 1, min(rows, 65536))
        batch = _spread(rng, 1, min(tokens, 64))
        return _axes(None, batch, max(1, tokens // batch), heads, kv, head, rot, dtype,
                     rng.choice([2, 3, 4]), rng.random() < 0.5, rng.random() < 0.3,
                     rng.random() < 0.5)
    if op == "pages":
        batch, most = _spread(rng, 1, 200), _spread(rng, 2, 600)
        return _pages(None, batch, most, rng.choice([1, 16, 64, 128]),
                      batch * most + _spread(rng, 1, 30000), rng.randint(0, batch // 2),
                      rng.randint(0, batch // 4))
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    page = rng.choice([16, 32, 64, 128])
    if op == "copy":
        kind, head = rng.choice(["bf16", "e4m3", "i8"]), rng.choice([32, 64, 80, 128, 256])
        most = max(1, int(6.0e7 / (kv * page * head * BYTES[kind])))
        return _copy(None, _spread(rng, 1, min(1000, most)), kv, page, head, kind,
                     1 if kind == "bf16" else rng.choice([1, 16]), rng.random() < 0.5)
    dtype = rng.choice(["bf16", "f16"])
    if op == "compact":
        tokens = _spread(rng, 4, 200)
        return _compact(None, _spread(rng, 1, 64), tokens, _spread(rng, 1, max(1, tokens // 4)), kv,
                        rng.choice([32, 64, 80, 128]), rng.choice([dtype, "e4m3", "i8"]), page,
                        rng.randint(0, 2000))
    kind, head = rng.choice(["e4m3", "i8"]), rng.choice([32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
    if op == "cache":
        tokens = _spread(rng, 1, min(int(3.0e7 / (kv * head)), 32768))
        batch = _spread(rng, 1, min(tokens, 64))
        return _cache(None, batch, max(1, tokens // batch), kv, head, dtype, kind, page, block,
                      rng.randint(0, 300), rng.random() < 0.5)
    group, tree = rng.choice([1, 2, 4, 5, 8]), rng.random() < 0.6
    tokens = _spread(rng, 1, 200 if tree else 600)
    most = min(6.0e8 / (kv * group * tokens), 4.0e8 / (kv * head))
    batch = _spread(rng, 1, max(1, min(32, int(most // 64))))
    ctx = _spread(rng, 1, max(1, min(65536, int(most / batch))))
    return _attn(None, batch, kv * group, kv, tokens, head, dtype, kind, page, block, ctx,
                 rng.random() < 0.5, tree)


# ---- sizes that follow from a case ------------------------------------------

def _lengths(case):
    """(keys before the call, new tokens) of each sequence."""
    n, ctx, tokens = case["batch"], case["ctx"], case["tokens"]
    if not case["ragged"]:
        return [ctx] * n, [tokens] * n
    return ([ctx - ctx * i // (2 * n) for i in range(n)],
            [tokens - tokens * i // (3 * n) for i in range(n)])


def _nodes(case):
    """Nodes of each tree."""
    n, t = case["batch"], case["tokens"]
    return [t - t * i // (2 * n) for i in range(n)] if case["ragged"] else [t] * n


def _frequencies(case):
    """Radians a position, a number for each pair."""
    rot = case["rot_dim"]
    return [BASE ** (-2.0 * i / rot) for i in range(rot // 2)]


def _table(freqs):
    """Turns a position in units of 2^-64, as 64-bit integers."""
    whole = [round(f / (2.0 * math.pi) * 2.0 ** 64) % 2 ** 64 for f in freqs]
    return [w - 2 ** 64 if w >= 2 ** 63 else w for w in whole]


def _axis_of(case):
    """The axis of each pair: a run of pairs for each axis, the first the
    shortest, or in turn."""
    pairs, axes = case["rot_dim"] // 2, case["axes"]
    if case["dealt"]:
        return [i % axes for i in range(pairs)]
    first = max(1, pairs // (axes + 1))
    rest = (pairs - first) / (axes - 1)
    return [0 if i < first else min(axes - 1, 1 + int((i - first) / rest)) for i in range(pairs)]


def _tree_of(case):
    """Each node's parent: the root (-1), then `branch` children of a node."""
    return [-1] + [(t - 1) // case["branch"] for t in range(1, case["tokens"])]


# ---- inputs ---------------------------------------------------------------------

def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _randn(shape, gen, dtype, spread=None):
    x = torch.randn(shape, generator=gen, device="cuda")
    if spread is not None:
        x.mul_(spread)
    return x.to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _channels(gen, head_dim):
    """Keys and values differ from channel to channel."""
    return torch.exp(0.5 * torch.randn(head_dim, generator=gen, device="cuda"))


def _quantised(x, kind, block):
    """(codes, scales) of [pages, kv_heads, page, head_dim] in 32 bits."""
    p, h, n, d = x.shape
    y = x.view(p, h, n // block, block, d)
    scale = torch.clamp(y.abs().amax((3, 4)) / TOP[kind], min=TINY)
    y = (y * (1.0 / scale)[..., None, None]).view(p, h, n, d)
    return y.to(torch.float8_e4m3fn) if kind == "e4m3" else torch.round(y).to(torch.int8), scale


def _cache_of(case, gen, pages, block):
    """A full cache: k, v [pages, kv_heads, page, head_dim] and, in 8 bits, a
    scale for each `block` keys."""
    shape, out = (pages, case["kv_heads"], case["page"], case["head_dim"]), {}
    for name in ("k", "v"):
        x = _randn(shape, gen, torch.float32, _channels(gen, shape[3]))
        if case["kind"] in TOP:
            out[name], out[name + "_scale"] = _quantised(x, case["kind"], block)
        else:
            out[name] = x.to(DTYPES[case["kind"]])
    return out


def _place(case, gen, state, most):
    """Pages in random order for `most` keys a sequence, and the cache."""
    per = -(-most // case["page"])
    pages = case["batch"] * per + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    state["table"] = order[:case["batch"] * per].view(case["batch"], per).contiguous()
    state["block"] = case.get("block", 1)
    state["cache"] = _cache_of(case, gen, pages, state["block"])


def _handle(s):
    """The cache as the framework's calls take it, made once with the tensors."""
    from frisk_amd import runtime as rt
    if "handle" not in s:
        c = s["cache"]
        s["handle"] = rt.KvCache(c["k"], c["v"], c.get("k_scale"), c.get("v_scale"), s.get("table"),
                                 scale_block=s["block"])
    return s["handle"]


def prepare(case, seed):
    return PREPARE[case["op"]](case, _gen(seed))


def _prepare_verify(case, gen):
    s = dict(case)
    b, t, v, dtype = case["batch"], case["tokens"], case["vocab"], DTYPES[case["dtype"]]
    # A few likely tokens above a wide floor, as a model's logits are.
    x = _randn((b, t, v), gen, torch.float32, 2.0)
    likely = torch.randint(0, v, (b, t, 8), generator=gen, device="cuda")
    x.scatter_add_(2, likely, torch.linspace(14.0, 6.0, 8, device="cuda").expand(b, t, 8).contiguous())
    s["logits"] = x.to(dtype)
    # The drafter sees them through noise.
    x.add_(_randn((b, t, v), gen, torch.float32, 0.5))
    if case["dense"]:
        s["draft_probs"] = torch.softmax(x, -1)
        kids = torch.multinomial(s["draft_probs"].view(b * t, v), case["branch"], replacement=True,
                                 generator=gen).view(b, t, case["branch"])
    else:
        s["draft_probs"] = None
        kids = torch.topk(x, case["branch"], -1).indices
    parents = _tree_of(case)
    s["parents"] = _ints([parents] * b).contiguous()
    s["drafts"] = torch.randint(0, v, (b, t), generator=gen, device="cuda").to(torch.int32)
    for i in range(1, t):
        s["drafts"][:, i] = kids[:, parents[i], (i - 1) % case["branch"]].to(torch.int32)
    s["new_len"] = _ints(_nodes(case)) if case["ragged"] else None
    s["uniform"] = torch.rand((b, t), generator=gen, device="cuda")
    s["final"] = torch.rand((b,), generator=gen, device="cuda")
    warm = 0.0 if case["greedy"] else 0.8
    s["temperature"] = torch.full((b,), warm, device="cuda")
    s["path"] = torch.zeros((b, t), dtype=torch.int32, device="cuda")
    s["count"], s["token"] = (torch.zeros((b,), dtype=torch.int32, device="cuda") for _ in range(2))
    s["probs"] = torch.zeros((b, t), device="cuda")
    return s


def _prepare_axes(case, gen):
    s = dict(case)
    b, n = case["batch"], case["seq"]
    freqs = _frequencies(case)
    s["freqs"] = torch.tensor(freqs, dtype=torch.float64, device="cuda")
    s["turns"] = _ints(_table(freqs), torch.int64)
    s["pair_axis"] = _ints(_axis_of(case), torch.uint8)
    # Frames of 24 x 32 patches, one after the other; a fourth axis counts tokens.
    at = torch.arange(n, device="cuda") + torch.randint(0, 100000, (b, 1), generator=gen, device="cuda")
    grid = [at // 768, at // 32 % 24, at % 32, at][:case["axes"]]
    s["positions"] = torch.stack(grid).to(torch.int32)
    for name, h in (("q", case["heads"]), ("k", case["kv_heads"])):
        # Heads next to each other in a token, as a projection leaves them.
        s[name] = _randn((b, n, h, case["head_dim"]), gen, DTYPES[case["dtype"]]).transpose(1, 2)
        s[name + "_out"] = torch.empty((b, n, h, case["head_dim"]), dtype=DTYPES[case["dtype"]],
                                       device="cuda").transpose(1, 2)
    return s


def _prepare_pages(case, gen):
    s = dict(case)
    b, most, page = case["batch"], case["max_pages"], case["page"]
    order = torch.randperm(case["pages"], generator=gen, device="cuda").to(torch.int32)
    room = torch.randint(1, most + 1, (b,), generator=gen, device="cuda")  # pages of each sequence
    s["table"] = torch.where(torch.arange(most, device="cuda") < room[:, None],
                             order[:b * most].view(b, most), -1).to(torch.int32).contiguous()
    # Forked sequences continue one of the others, ended ones nothing.
    parent = torch.arange(b, device="cuda")
    pick = torch.randperm(b, generator=gen, device="cuda")
    forks, ended = pick[:case["forks"]], pick[case["forks"]:case["forks"] + case["ended"]]
    stay = pick[case["forks"] + case["ended"]:]
    parent[forks] = stay[torch.randint(0, len(stay), (len(forks),), generator=gen, device="cuda")]
    parent[ended] = -1
    keys = room * page - torch.randint(0, page, (b,), generator=gen, device="cuda")
    s["parent"] = parent.to(torch.int32)
    s["keep"] = keys[parent.clamp(min=0)].to(torch.int32)
    s["want"] = s["keep"] + 8
    s["out"] = torch.empty_like(s["table"])
    for name in ("src", "dst", "rows"):
        s[name] = torch.empty((b,), dtype=torch.int32, device="cuda")
    s["lacking"] = torch.empty((1,), dtype=torch.int32, device="cuda")
    return s


def _prepare_copy(case, gen):
    s = dict(case)
    n = case["pairs"]
    s["cache"] = _cache_of(case, gen, 2 * n + 5, case["block"])
    order = torch.randperm(2 * n + 5, generator=gen, device="cuda").to(torch.int32)
    s["src"], s["dst"] = order[:n].contiguous(), order[n:2 * n].contiguous()
    s["rows"] = torch.randint(1, case["page"] + 1, (n,), generator=gen, device="cuda").to(torch.int32) \
        if case["part"] else None
    return s


def _prepare_compact(case, gen):
    s = dict(case)
    b, t, n = case["batch"], case["tokens"], case["taken"]
    _place(case, gen, s, case["ctx"] + t)
    s["ctx_len"] = _ints([case["ctx"] - i % 7 if case["ctx"] > 6 else case["ctx"] for i in range(b)])
    # A branch from the root on; its later nodes lie behind all that it moves to.
    pick = torch.argsort(torch.rand((b, t - n), generator=gen, device="cuda"), -1)[:, :n - 1] + n
    path = torch.full((b, t), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    path[:, 1:n] = torch.sort(pick, -1).values.to(torch.int32)
    s["path"] = path
    s["count"] = _ints([n - i % min(n, 3) for i in range(b)])
    return s


def _prepare_cache(case, gen):
    s = dict(case)
    ctx, new = _lengths(case)
    b, d, dtype = case["batch"], case["head_dim"], DTYPES[case["dtype"]]
    _place(case, gen, s, case["ctx"] + case["tokens"])
    s["ctx_len"], s["new_len"] = _ints(ctx), _ints(new) if case["ragged"] else None
    shape = (b, case["tokens"], case["kv_heads"], d)
    for name in ("k", "v"):
        s[name] = _randn(shape, gen, dtype, 1.1 * _channels(gen, d)).transpose(1, 2)
        s[name + "_out"] = torch.zeros((b, case["kv_heads"], case["tokens"], d), dtype=dtype,
                                       device="cuda")
    return s


def _prepare_attn(case, gen):
    s = _prepare_cache(case, gen)
    b, t, h, d = case["batch"], case["tokens"], case["heads"], case["head_dim"]
    s["q"] = _randn((b, t, h, d), gen, DTYPES[case["dtype"]]).transpose(1, 2)
    s["o"] = torch.zeros((b, t, h, d), dtype=DTYPES[case["dtype"]], device="cuda").transpose(1, 2)
    if case["tree"]:
        # Every drafted token continues an earlier one, or (-1) the context.
        at = torch.arange(t, device="cuda").expand(b, t)
        low = torch.clamp(at // 4 - 1, min=-1)
        pick = torch.rand((b, t), generator=gen, device="cuda") * (at - low)
        parents = torch.minimum(low + pick.long(), at - 1).to(torch.int32)
        s["seen"] = _ancestors(parents)
        # The mask's words, as the step that drafted them left them.
        bits = torch.nn.functional.pad(s["seen"].long(), (0, -t % 64)).view(b, t, -1, 64)
        s["mask"] = (bits << torch.arange(64, device="cuda")).sum(-1)
    return s


def _ancestors(parents):
    """bool [batch, t, t]: which drafted tokens each one continues, itself among them."""
    b, t = parents.shape
    up = torch.cat((parents.long(), torch.full((b, 1), -1, device="cuda")), 1)
    up = torch.where(up < 0, t, up)  # place t: the context, its own parent
    seen = torch.eye(t + 1, dtype=torch.bool, device="cuda").expand(b, -1, -1)
    for _ in range(max(1, t).bit_length()):
        seen = seen | seen.gather(1, up[:, :, None].expand(-1, -1, t + 1))
        up = up.gather(1, up)
    return seen[:, :t, :t]


PREPARE = {"verify": _prepare_verify, "axes": _prepare_axes, "pages": _prepare_pages,
           "copy": _prepare_copy, "compact": _prepare_compact, "cache": _prepare_cache,
           "attn": _prepare_attn}


# ---- one pass through the framework -----------------------------------------------

def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


def _own(s):
    from frisk_amd import runtime as rt
    op = s["op"]
    if op == "verify":
        rt.tree_verify(s["logits"], s["drafts"], s["parents"], s["uniform"], s["final"],
                       draft_probs=s["draft_probs"], temperature=s["temperature"],
                       new_len=s["new_len"], path=s["path"], count=s["count"], token=s["token"],
                       probs=s["probs"])
        return {name: s[name] for name in ("path", "count", "token", "probs")}
    if op == "axes":
        rt.rope(s["q"], s["q_out"], s["positions"], s["turns"], k=s["k"], k_out=s["k_out"],
                pair_axis=s["pair_axis"], interleaved=s["interleaved"], backward=s["backward"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if op == "pages":
        rt.kv_pages(s["table"], s["keep"], s["want"], s["page"], s["pages"], parent=s["parent"],
                    out=s["out"], src=s["src"], dst=s["dst"], rows=s["rows"], lacking=s["lacking"])
        return {name: s[name] for name in ("out", "src", "dst", "rows", "lacking")}
    cache = _handle(s)
    if op == "copy":
        rt.kv_copy_pages(cache, s["src"], s["dst"], rows=s["rows"])
        return _held(s)
    if op == "compact":
        rt.kv_compact(cache, s["path"], s["ctx_len"], s["count"])
        return _held(s)
    rt.kv_append(s["k"], s["v"], cache, s["ctx_len"], new_len=s["new_len"])
    if op == "cache":
        rt.kv_read(cache, s["k_out"], s["v_out"], s["ctx_len"], new_len=s["new_len"])
        return {"k": s["k_out"], "v": s["v_out"], "k_scale": cache.k_scale, "v_scale": cache.v_scale}
    rt.tree_attn(s["q"], cache, s["ctx_len"], s["o"], mask=s.get("mask"), new_len=s["new_len"])
    return {"o": s["o"], "k_scale": cache.k_scale, "v_scale": cache.v_scale}


def _held(s):
    """The cache's tensors."""
    return dict(s["cache"])


# ---- the same from elementary operations ----------------------------------------

def _plain_verify(s):
    """The whole batch node by node: `a` [batch, vocab] is what is left of the
    current node's probabilities."""
    b, t, v = s["logits"].shape
    warm = s["temperature"].double()[:, None]
    live = torch.full((b,), t, device="cuda") if s["new_len"] is None else s["new_len"].long()

    def row(i):
        x = s["logits"][:, i].double()
        hot = torch.zeros_like(x).scatter_(1, s["logits"][:, i].float().argmax(-1, keepdim=True), 1.0)
        y = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(warm > 0, warm, 1.0))
        return torch.where(warm > 0, y / y.sum(-1, keepdim=True), hot)

    a, at = row(0), torch.zeros((b,), dtype=torch.long, device="cuda")
    count = torch.ones((b,), dtype=torch.long, device="cuda")
    path = torch.full((b, t + 1), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    rows = [a]
    probs = torch.zeros((b, t), device="cuda")
    up = _tree_of(s)  # (the same tree in every sequence)
    for i in range(1, t):
        tried = (s["parents"][:, i] == at) & (i < live)
        token = s["drafts"][:, i:i + 1].long()
        probs[:, i] = torch.where(i < live, rows[up[i]].gather(1, token).squeeze(1), 0.0).float()
        if s["draft_probs"] is None:
            q = torch.zeros_like(a).scatter_(1, token, 1.0)
            rest = a * (1.0 - q)
        else:
            q = s["draft_probs"].gather(1, at[:, None, None].expand(b, 1, v)).squeeze(1).double()
            rest = torch.clamp(a - q, min=0.0)
        taken = tried & (s["uniform"][:, i].double() * q.gather(1, token).squeeze(1)
                         < a.gather(1, token).squeeze(1))
        mass = rest.sum(-1, keepdim=True)
        rest = torch.where(mass > 0, rest / mass, a)
        rows.append(row(i))
        a = torch.where(taken[:, None], rows[i], torch.where(tried[:, None], rest, a))
        path.scatter_(1, torch.where(taken, count, t)[:, None],
                      torch.full((b, 1), i, dtype=torch.int32, device="cuda"))
        at = torch.where(taken, i, at)
        count = count + taken.long()
    total = torch.cumsum(a, -1)
    past = total > s["final"].double()[:, None] * total[:, -1:]
    return {"path": path[:, :t].contiguous(), "count": count.to(torch.int32),
            "token": past.to(torch.uint8).argmax(-1).to(torch.int32), "probs": probs}


def _plain_axes(s):
    at = s["positions"].double()[s["pair_axis"].long()]  # [pairs, batch, seq]
    phase = at.permute(1, 2, 0)[:, None] * s["freqs"]
    cos, sin = torch.cos(phase).float(), torch.sin(phase).float()
    if s["backward"]:
        sin = -sin
    rot, half = s["rot_dim"], s["rot_dim"] // 2

    def turned(x):
        y = x.float()
        if s["interleaved"]:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            pair = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:rot]
            pair = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        return torch.cat((pair, y[..., rot:]), -1).to(x.dtype)

    return {"q": turned(s["q"]), "k": turned(s["k"])}


def _plain_pages(s):
    b, most, page, pages = s["batch"], s["max_pages"], s["page"], s["pages"]
    parent, keep = s["parent"].long(), s["keep"].long()
    live = parent >= 0
    keep = torch.where(live, keep.clamp(max=most * page), 0)
    want = torch.where(live, torch.maximum(s["want"].long().clamp(max=most * page), keep), 0)
    kept, wanted = -(-keep // page), -(-want // page)
    at = torch.arange(most, device="cuda")
    row = s["table"][parent.clamp(min=0)].long()
    row = torch.where((at < kept[:, None]) & (row >= 0) & (row < pages), row, -1)
    # The last page, where new keys go: its own if nobody else keeps it.
    last = row.gather(1, (kept - 1).clamp(min=0)[:, None]).squeeze(1)
    part = (kept > 0) & (keep % page > 0) & (last >= 0)
    ends = part[:, None] & (at == (kept - 1)[:, None])
    used = torch.zeros((pages + 1,), dtype=torch.int32, device="cuda")
    used.scatter_(0, torch.where((row >= 0) & ~ends, row, pages).flatten(), 1)
    first = torch.full((pages + 1,), b, device="cuda")
    spot = torch.where(part, last, pages)
    first.scatter_reduce_(0, spot, torch.arange(b, device="cuda"), "amin")
    stays = part & (used[spot] == 0) & (first[spot] == torch.arange(b, device="cuda"))
    used.scatter_(0, torch.where(part, last, pages), 1)
    moves = part & ~stays
    row = torch.where(ends & moves[:, None], -1, row)
    # Free pages by number to what lacks one, by sequence and place.
    free = torch.argsort(used[:pages], stable=True)
    lacks = ((row < 0) & (at < wanted[:, None])).flatten()
    rank = torch.cumsum(lacks.long(), 0) - 1
    have = pages - used[:pages].sum()
    given = torch.where(rank < have, free[rank.clamp(0, pages - 1)], -1)
    row = torch.where(lacks, given, row.flatten()).view(b, most)
    new = row.gather(1, (kept - 1).clamp(min=0)[:, None]).squeeze(1)
    moves = moves & (new >= 0)
    return {"out": row.to(torch.int32), "src": torch.where(moves, last, -1).to(torch.int32),
            "dst": torch.where(moves, new, -1).to(torch.int32),
            "rows": torch.where(moves, keep % page, 0).to(torch.int32),
            "lacking": (lacks.sum() - have).clamp(min=0).to(torch.int32)[None]}


def _bits(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for name, x in s["cache"].items():
        per = s["block"] if name.endswith("scale") else 1
        rows = x.shape[2]
        got = _bits(x)[src]
        if s["rows"] is not None:
            mine = torch.arange(rows, device="cuda") * per < s["rows"][:, None]
            mine = mine[:, None, :, None] if x.dim() == 4 else mine[:, None]
            got = torch.where(mine, got, _bits(x)[dst])
        _bits(x)[dst] = got
    return _held(s)


def _slots(s, at):
    """(page, row of the page) of each sequence's keys `at` ([batch, n])."""
    return s["table"].long().gather(1, at // s["page"]), at % s["page"]


def _plain_compact(s):
    n = s["taken"]
    ctx = s["ctx_len"].long()[:, None]
    path = s["path"][:, :n].long()
    live = torch.arange(n, device="cuda") < s["count"][:, None]
    page, row = _slots(s, ctx + path)
    to_page, to_row = _slots(s, ctx + torch.arange(n, device="cuda"))
    page, row, to_page, to_row = page[live], row[live], to_page[live], to_row[live]
    for x in s["cache"].values():
        _bits(x)[to_page, :, to_row] = _bits(x)[page, :, row]
    return _held(s)


def _plain_append(s):
    """New rows in blocks: [batch, blocks, keys of a block]."""
    size, kind = s["block"], s["kind"]
    b, t = s["batch"], s["tokens"]
    ctx = s["ctx_len"].long()
    new = torch.full_like(ctx, t) if s["new_len"] is None else s["new_len"].long()
    blocks = (t + size - 2) // size + 1
    key = (ctx // size * size)[:, None] + torch.arange(blocks * size, device="cuda")
    old, fresh = key < ctx[:, None], (key >= ctx[:, None]) & (key < (ctx + new)[:, None])
    page, row = _slots(s, key.clamp(max=s["table"].shape[1] * s["page"] - 1))
    part = old.view(b, blocks, size).any(-1)[..., None]
    some = fresh.view(b, blocks, size).any(-1)
    lead, slot = page.view(b, blocks, size)[..., 0], row.view(b, blocks, size)[..., 0] // size
    for name in ("k", "v"):
        codes, scales = s["cache"][name], s["cache"][name + "_scale"]
        x = s[name].transpose(1, 2).float()  # [batch, tokens, kv_heads, head_dim]
        x = x.gather(1, (key - ctx[:, None]).clamp(0, t - 1)[:, :, None, None].expand(-1, -1, *x.shape[2:]))
        x = torch.where(fresh[:, :, None, None], x, 0.0).view(b, blocks, size, *x.shape[2:])
        was = scales[lead, :, slot]  # [batch, blocks, kv_heads]
        scale = torch.clamp(x.abs().amax((2, 4)) / TOP[kind], min=TINY)
        scale = torch.where(part, torch.maximum(scale, was), scale)
        inv = 1.0 / scale
        y = x * inv[:, :, None, :, None]
        before = _values(codes, page, row).view(y.shape)
        again = before * (was * inv)[:, :, None, :, None]
        again = torch.where((scale > was)[:, :, None, :, None], again, before)
        y = torch.where(fresh.view(b, blocks, size)[..., None, None], y, again).view(b, blocks * size,
                                                                                     *y.shape[3:])
        y = y.to(torch.float8_e4m3fn).view(torch.uint8) if kind == "e4m3" else torch.round(y).to(torch.int8)
        put = (fresh | old) & some[:, :, None].expand(-1, -1, size).flatten(1)
        _bits(codes)[page[put], :, row[put]] = y[put]
        scales[lead[some], :, slot[some]] = scale[some]


def _values(codes, page, row):
    x = _bits(codes)[page, :, row]
    return x.view(torch.float8_e4m3fn).float() if codes.dtype == torch.float8_e4m3fn else x.float()


def _rows(s, name, at):
    """[batch, n, kv_heads, head_dim] of the cache's keys `at` in 32 bits."""
    page, row = _slots(s, at)
    x = _values(s["cache"][name], page, row)
    return x * s["cache"][name + "_scale"][page, :, row // s["block"]][..., None]


def _plain_cache(s):
    _plain_append(s)
    t = s["tokens"]
    at = s["ctx_len"].long()[:, None] + torch.arange(t, device="cuda")
    out = {}
    for name in ("k", "v"):
        back = _rows(s, name, at).transpose(1, 2)
        if s["new_len"] is not None:  # rows behind a sequence's last stay as they were
            live = torch.arange(t, device="cuda") < s["new_len"][:, None]
            back = torch.where(live[:, None, :, None], back, 0.0)
        out[name] = back.to(s[name].dtype).contiguous()
        out[name + "_scale"] = s["cache"][name + "_scale"]
    return out


def _seen_keys(s, n):
    """bool [batch, tokens, n]: which of n keys each new token sees."""
    b, t = s["batch"], s["tokens"]
    ctx = s["ctx_len"].long()
    new = torch.full_like(ctx, t) if s["new_len"] is None else s["new_len"].long()
    draft = torch.arange(n, device="cuda") - ctx[:, None]  # [batch, n]
    if s["tree"]:
        seen = s["seen"].gather(2, draft.clamp(0, t - 1)[:, None, :].expand(b, t, n))
    else:
        seen = draft[:, None, :] <= torch.arange(t, device="cuda")[:, None]
    return (seen & (draft < new[:, None])[:, None, :]) | (draft < 0)[:, None, :]


def _plain_attn(s):
    _plain_append(s)
    b, h, kv, t, d = s["batch"], s["heads"], s["kv_heads"], s["tokens"], s["head_dim"]
    n = s["ctx"] + t
    at = torch.arange(n, device="cuda").expand(b, n)
    seen = _seen_keys(s, n)
    k = _rows(s, "k", at).transpose(1, 2).contiguous()
    v = _rows(s, "v", at).transpose(1, 2).contiguous()
    q = s["q"].float().reshape(b, kv, (h // kv) * t, d)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(b, h, t, n)
    score.masked_fill_(~seen[:, None], -math.inf)
    weight = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = weight.sum(-1, keepdim=True)
    o = torch.matmul(weight.view(b, kv, (h // kv) * t, n), v).view(b, h, t, d) / total
    if s["new_len"] is not None:
        live = (torch.arange(t, device="cuda") < s["new_len"][:, None])[:, None, :]
        o = torch.where(live[..., None], o, 0.0)
    return {"o": o.to(s["q"].dtype), "k_scale": s["cache"]["k_scale"], "v_scale": s["cache"]["v_scale"]}


PLAIN = {"verify": _plain_verify, "axes": _plain_axes, "pages": _plain_pages, "copy": _plain_copy,
         "compact": _plain_compact, "cache": _plain_cache, "attn": _plain_attn}


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    op = case["op"]
    if op == "verify":
        # The rows of nodes that have children, and one that the last token comes from.
        rows = sum(1 + max(0, -(-(n - 1) // case["branch"]) - 1) for n in _nodes(case))
        dense = case["batch"] if case["dense"] and case["tokens"] > 1 else 0
        return {"bytes": case["vocab"] * (rows * BYTES[case["dtype"]] + 4 * dense) +
                16 * case["batch"] * case["tokens"], "flops": 40 * rows * case["vocab"]}
    if op == "axes":
        tokens, heads = case["batch"] * case["seq"], case["heads"] + case["kv_heads"]
        return {"bytes": 2 * tokens * heads * case["head_dim"] * BYTES[case["dtype"]] +
                4 * case["axes"] * tokens + 5 * case["rot_dim"] // 2,
                "flops": 3 * tokens * heads * case["rot_dim"]}
    if op == "pages":
        n = case["batch"] * case["max_pages"]
        return {"bytes": 8 * n + 24 * case["batch"], "flops": n}
    d = case["head_dim"]
    row = d * BYTES[case["kind"]] + (4.0 / case.get("block", 1) if case["kind"] in TOP else 0)  # key or value
    if op == "copy":
        rows = 2 * case["pairs"] * case["kv_heads"] * (case["page"] / 2 if case["part"] else case["page"])
        return {"bytes": int(2 * rows * row), "flops": 0}
    if op == "compact":
        rows = 2 * case["kv_heads"] * sum(case["taken"] - i % min(case["taken"], 3) - 1
                                          for i in range(case["batch"]))
        return {"bytes": int(2 * rows * row) + 8 * case["batch"], "flops": 0}
    e = BYTES[case["dtype"]]
    ctx, new = _lengths(case)
    fresh = 2 * sum(new) * case["kv_heads"]
    if op == "cache":  # read in, written to the cache, written out
        return {"bytes": int(fresh * (2 * d * e + row)), "flops": 4 * fresh * d}
    keys = sum(c + n for c, n in zip(ctx, new))
    seen = sum(n * (c + (min(n, n.bit_length()) if case["tree"] else (n + 1) / 2))
               for c, n in zip(ctx, new))
    return {"bytes": int(2 * keys * case["kv_heads"] * row + 2 * sum(new) * case["heads"] * d * e +
                         fresh * d * e),
            "flops": int(4 * d * case["heads"] * seen)}


# ---- in 64 bits, from the definitions -------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "axes":
        return _exact_axes(s)
    if case["op"] == "cache":
        return _exact_cache(s)
    if case["op"] == "attn":
        return _exact_attn(s)
    if case["op"] == "verify":
        return _exact_verify(s)
    return None  # copies and page numbers: no computed numbers


def _exact_verify(s):
    # log p(x) = x / T - log sum exp(x / T), a node at a time.
    b, t = s["uniform"].shape
    probs, up = torch.zeros((b, t), dtype=torch.float64, device="cuda"), _tree_of(s)
    for j, n in enumerate(_nodes(s)):
        for i in range(1, n):
            x = s["logits"][j, up[i]].double()
            token = int(s["drafts"][j, i])
            if s["greedy"]:
                probs[j, i] = float((x[token] == x.max()) & (x[:token] < x[token]).all())
            else:
                x = x / s["temperature"][j].double()
                probs[j, i] = torch.exp(x[token] - torch.logsumexp(x, 0))
    return {"path": None, "count": None, "token": None, "probs": probs}


def _exact_axes(s):
    # Pairs as complex numbers, turned by e^(i p f).
    at = s["positions"].double()
    phase = torch.stack([at[a] * f for a, f in zip(s["pair_axis"].tolist(), s["freqs"].tolist())], -1)[:, None]
    turn = torch.polar(torch.ones_like(phase), -phase if s["backward"] else phase)
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        rot, half = s["rot_dim"], s["rot_dim"] // 2
        y = x.clone()
        one, two = (slice(0, rot, 2), slice(1, rot, 2)) if s["interleaved"] else \
            (slice(0, half), slice(half, rot))
        z = torch.complex(x[..., one], x[..., two]) * turn
        y[..., one], y[..., two] = z.real, z.imag
        out[name] = y
    return out


def _rounded(y, kind):
    """y on the grid of `kind`, ties to the even neighbour."""
    if kind == "i8":
        return torch.round(y)
    power = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    power = torch.where(torch.ldexp(torch.ones_like(y), power) > y.abs().clamp(min=2.0 ** -6),
                        power - 1, power)
    step = torch.ldexp(torch.ones_like(y), power - 3)
    return torch.round(y / step) * step


def _exact_rows(s, name, j, ctx, new):
    """(values [kv_heads, ctx + new, head_dim], scales of its blocks) of sequence j after its append."""
    size = s["block"]
    at = torch.arange(-(-(ctx + new) // size) * size, device="cuda")
    page, row = s["table"][j].long()[at // s["page"]], at % s["page"]
    codes = s["cache"][name]
    x = codes[page, :, row].double() if codes.dtype == torch.int8 else \
        codes.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn).double()
    x = x.transpose(0, 1).clone()  # [kv_heads, keys, head_dim]
    scale = s["cache"][name + "_scale"].double()[page[::size], :, row[::size] // size].t().clone()
    for i in range(ctx // size, len(at) // size if new else 0):
        lo, hi = max(ctx, i * size), min(ctx + new, (i + 1) * size)
        mine = s[name][j, :, lo - ctx:hi - ctx].double()
        need = (mine.abs().amax((1, 2)) / TOP[s["kind"]]).clamp(min=TINY)
        if lo > i * size:
            was = scale[:, i].clone()
            grown = need > was
            need = torch.maximum(need, was)
            old = x[:, i * size:lo]
            moved = _rounded(old * (was / need)[:, None, None], s["kind"])
            x[:, i * size:lo] = torch.where(grown[:, None, None], moved, old)
        scale[:, i] = need
        x[:, lo:hi] = _rounded(mine / need[:, None, None], s["kind"])
    return x[:, :ctx + new] * scale.repeat_interleave(size, 1)[:, :ctx + new, None], scale


def _exact_cache(s):
    ctx, new = _lengths(s)
    out = {}
    for name in ("k", "v"):
        back = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
        scales = s["cache"][name + "_scale"].double()
        for j in range(s["batch"]):
            rows, scale = _exact_rows(s, name, j, ctx[j], new[j])
            back[j, :, :new[j]] = rows[:, ctx[j]:]
            first = torch.arange(scale.shape[1], device="cuda") * s["block"]
            scales[s["table"][j].long()[first // s["page"]], :, first % s["page"] // s["block"]] = scale.t()
        out[name], out[name + "_scale"] = back, scales
    return out


def _exact_attn(s):
    b, h, kv, t, d = s["batch"], s["heads"], s["kv_heads"], s["tokens"], s["head_dim"]
    ctx, new = _lengths(s)
    o = torch.zeros((b, h, t, d), dtype=torch.float64, device="cuda")
    out = {"o": o} | {n: s["cache"][n].double() for n in ("k_scale", "v_scale")}
    for j in range(b):
        hidden = torch.zeros((new[j], ctx[j] + new[j]), dtype=torch.bool, device="cuda")
        hidden[:, ctx[j]:] = ~(s["seen"][j, :new[j], :new[j]] if s["tree"] else
                               torch.ones((new[j], new[j]), dtype=torch.bool, device="cuda").tril())
        (kk, ks), (vv, vs) = (_exact_rows(s, name, j, ctx[j], new[j]) for name in ("k", "v"))
        first = torch.arange(ks.shape[1], device="cuda") * s["block"]
        for name, scale in (("k_scale", ks), ("v_scale", vs)):
            out[name][s["table"][j].long()[first // s["page"]], :, first % s["page"] // s["block"]] = scale.t()
        for head in range(h):
            g = head // (h // kv)
            score = (s["q"][j, head, :new[j]].double() @ kk[g].t()) / math.sqrt(d)
            weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            o[j, head, :new[j]] = weight @ vv[g]
    return out
