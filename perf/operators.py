"""Performance cases of the operators around attention over a cache: rotary
positions, a cache written in 16 or 8 bits and read back, and attention of
drafted tokens over it.

A case is one call, or the run of calls that belong together, as a serving or
training program makes it through `frisk_amd.runtime`.  `run` computes it with
those calls where `own` is true and from elementary torch operations in 32
bits (angles in 64) where it is false.

Fields of a case (all plain values):
  op "rope":  batch, seq, heads, kv_heads, head_dim, rot_dim, dtype,
              interleaved, backward, far (largest position), scaling
              ("none" or "ramp": low frequencies slowed down 8 times)
  op "cache": batch, tokens, kv_heads, head_dim, dtype, kind (what the cache
              holds: "e4m3", "i8", or the dtype itself), page (0: one page a
              sequence), ctx (keys already there), ragged
  op "attn":  batch, heads, kv_heads, tokens, head_dim, dtype, kind, page,
              ctx, ragged, tree (masks from drafted parents; else causal),
              lse
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1, "i8": 1}
TOP = {"e4m3": 448.0, "i8": 127.0}
TINY = 2.0 ** -126
BASE, SLOWED, TRAINED = 10000.0, 8.0, 8192


def _rope(name, batch, seq, heads, kv_heads, head_dim, rot_dim, dtype, interleaved=False,
          backward=False, far=8192, scaling="none"):
    return {"name": name, "op": "rope", "batch": batch, "seq": seq, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "rot_dim": rot_dim, "dtype": dtype,
            "interleaved": interleaved, "backward": backward, "far": far, "scaling": scaling}


def _cache(name, batch, tokens, kv_heads, head_dim, dtype, kind, page, ctx, ragged=False):
    return {"name": name, "op": "cache", "batch": batch, "tokens": tokens, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "kind": kind, "page": page, "ctx": ctx,
            "ragged": ragged}


def _attn(name, batch, heads, kv_heads, tokens, head_dim, dtype, kind, page, ctx, ragged=False,
          tree=False, lse=False):
    return {"name": name, "op": "attn", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "tokens": tokens, "head_dim": head_dim, "dtype": dtype, "kind": kind, "page": page,
            "ctx": ctx, "ragged": ragged, "tree": tree, "lse": lse}


def listed():
    return [
        # One decode step of a serving batch, far into long contexts.
        _rope("rope_token_bf16", 32, 1, 32, 8, 128, 128, "bf16", far=131072, scaling="ramp"),
        # A prompt.
        _rope("rope_prompt_bf16", 1, 8192, 32, 8, 128, 128, "bf16"),
        # A training step's gradient through the rotation, pairs interleaved.
        _rope("rope_grad_f16", 4, 4096, 32, 32, 128, 128, "f16", interleaved=True, backward=True),
        # Part of an odd head rotated, in f32, at odd sizes.
        _rope("rope_part_f32", 3, 1111, 12, 3, 80, 48, "f32", far=1000003),
        # One token of every sequence of a serving batch into 8-bit pages.
        _cache("cache_token_e4m3", 32, 1, 8, 128, "bf16", "e4m3", 64, 4095),
        # Prompts into 8-bit pages, and back as what later steps will see.
        _cache("cache_prompt_e4m3", 4, 8192, 8, 128, "bf16", "e4m3", 64, 0),
        # Ragged chunks into whole rows of int8, head size 64.
        _cache("cache_chunk_i8", 3, 1777, 5, 64, "f16", "i8", 0, 333, ragged=True),
        # One token against a short context: latency.
        _attn("attn_token_short", 1, 32, 8, 1, 128, "bf16", "bf16", 0, 1000),
        # A decode step of a serving batch over pages.
        _attn("attn_token_bf16", 16, 32, 8, 1, 128, "bf16", "bf16", 64, 8191, ragged=True),
        # Drafted trees over long contexts in 8-bit pages.
        _attn("attn_tree_e4m3", 8, 32, 8, 64, 128, "bf16", "e4m3", 16, 16384, tree=True),
        # Odd drafted trees, every head its own keys, int8, head size 64.
        _attn("attn_tree_i8", 4, 16, 16, 33, 64, "f16", "i8", 0, 5001, ragged=True, tree=True,
              lse=True),
        # A chunk of a long prompt over what came before it.
        _attn("attn_chunk_bf16", 2, 32, 8, 512, 128, "bf16", "bf16", 64, 32256),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo .. hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    op = rng.choice(["rope", "cache", "attn", "attn"])
    if op == "rope":
        dtype = rng.choice(["bf16", "f16", "f32"])
        head = rng.choice([32, 64, 80, 96, 128, 256])
        rot = head if rng.random() < 0.6 else 2 * rng.randint(4, head // 2)
        kv = rng.choice([1, 2, 3, 5, 8])
        heads = kv * rng.choice([1, 2, 4, 7])
        rows = max(1, int(1.2e8 / ((heads + kv) * head * BYTES[dtype])))
        tokens = _spread(rng, 1, min(rows, 65536))
        batch = _spread(rng, 1, min(tokens, 64))
        return _rope(None, batch, max(1, tokens // batch), heads, kv, head, rot, dtype,
                     rng.random() < 0.5, rng.random() < 0.3, _spread(rng, 100, 2000000),
                     rng.choice(["none", "ramp"]))
    dtype = rng.choice(["bf16", "f16"])
    kind = rng.choice([dtype, "e4m3", "i8"])
    page = rng.choice([0, 16, 32, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    head = rng.choice([32, 64, 128])
    if op == "cache":
        rows = int(3.0e7 / (kv * head))
        tokens = _spread(rng, 1, min(rows, 32768))
        batch = _spread(rng, 1, min(tokens, 64))
        return _cache(None, batch, max(1, tokens // batch), kv, head, dtype, kind, page,
                      rng.randint(0, 300), rng.random() < 0.5)
    group = rng.choice([1, 2, 4, 5, 8])
    tree = rng.random() < 0.6
    tokens = _spread(rng, 1, 200 if tree else 600)
    most = min(6.0e8 / (kv * group * tokens), 4.0e8 / (kv * head * BYTES[kind]))
    batch = _spread(rng, 1, max(1, min(32, int(most // 64))))
    ctx = _spread(rng, 1, max(1, min(65536, int(most / batch))))
    return _attn(None, batch, kv * group, kv, tokens, head, dtype, kind, page, ctx,
                 rng.random() < 0.5, tree, rng.random() < 0.4)


# ---- sizes that follow from a case ------------------------------------------

def _lengths(case):
    """(keys before the call, new tokens) of each sequence."""
    n, ctx, tokens = case["batch"], case["ctx"], case["tokens"]
    if not case["ragged"]:
        return [ctx] * n, [tokens] * n
    return ([ctx - ctx * i // (2 * n) for i in range(n)],
            [tokens - tokens * i // (3 * n) for i in range(n)])


def _frequencies(case):
    """Radians a position, a number for each pair."""
    rot, out = case["rot_dim"], []
    for i in range(rot // 2):
        f = BASE ** (-2.0 * i / rot)
        if case["scaling"] == "ramp":  # whole below 1 turn in the trained length, kept above 4
            keep = min(1.0, max(0.0, (TRAINED * f / (2.0 * math.pi) - 1.0) / 3.0))
            f = keep * f + (1.0 - keep) * f / SLOWED
        out.append(f)
    return out


def _table(freqs):
    """Turns a position in units of 2^-64, as 64-bit integers."""
    whole = [round(f / (2.0 * math.pi) * 2.0 ** 64) % 2 ** 64 for f in freqs]
    return [w - 2 ** 64 if w >= 2 ** 63 else w for w in whole]


# ---- inputs ---------------------------------------------------------------------

def _randn(shape, gen, dtype, spread=None):
    x = torch.randn(shape, generator=gen, device="cuda")
    if spread is not None:
        x.mul_(spread)
    return x.to(dtype)


def _channels(gen, head_dim):
    """Keys and values differ from channel to channel."""
    return torch.exp(0.5 * torch.randn(head_dim, generator=gen, device="cuda"))


def _pages(case, gen, most):
    """(pages, page size, block table or None) that hold `most` keys a sequence."""
    if case["page"] == 0:
        return case["batch"], most, None
    per = -(-most // case["page"])
    pages = case["batch"] * per + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    return pages, case["page"], order[:case["batch"] * per].view(case["batch"], per).contiguous()


def _quantised(x, kind):
    """(codes, scales) of the last dimension's rows of x, in 32 bits."""
    x = x.float()
    top = torch.clamp(x.abs().amax(-1, keepdim=True), min=TOP[kind] * TINY)
    y = x * TOP[kind] / top
    codes = y.to(torch.float8_e4m3fn) if kind == "e4m3" else torch.round(y).to(torch.int8)
    return codes, (top / TOP[kind]).squeeze(-1)


def _cache_of(case, gen, pages, size, full):
    """The cache's tensors: [pages, kv_heads, page size, head_dim] and, in 8
    bits, scales [pages, kv_heads, page size]; `full`: every row holds keys."""
    shape = (pages, case["kv_heads"], size, case["head_dim"])
    out = {}
    for name in ("k", "v"):
        if case["kind"] not in TOP:
            out[name] = _randn(shape, gen, DTYPES[case["dtype"]], _channels(gen, shape[3])) if full \
                else torch.zeros(shape, dtype=DTYPES[case["dtype"]], device="cuda")
        elif full:
            out[name], out[name + "_scale"] = _quantised(
                _randn(shape, gen, torch.float32, _channels(gen, shape[3])), case["kind"])
        else:
            out[name] = torch.zeros(shape, dtype=torch.uint8, device="cuda").view(
                torch.float8_e4m3fn if case["kind"] == "e4m3" else torch.int8)
            out[name + "_scale"] = torch.zeros(shape[:3], device="cuda")
    return out


def _handle(case, tensors, table):
    """The tensors as the framework's calls take them together."""
    return (tensors["k"], tensors["v"], tensors.get("k_scale"), tensors.get("v_scale"), table)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(case)
    dtype = DTYPES[case["dtype"]]
    b, d = case["batch"], case["head_dim"]
    if case["op"] == "rope":
        freqs = _frequencies(case)
        state["freqs"] = torch.tensor(freqs, dtype=torch.float64, device="cuda")
        state["table"] = torch.tensor(_table(freqs), dtype=torch.int64, device="cuda")
        first = torch.randint(0, max(1, case["far"] - case["seq"]), (b, 1), generator=gen, device="cuda")
        state["positions"] = first + torch.arange(case["seq"], device="cuda")
        for name, h in (("q", case["heads"]), ("k", case["kv_heads"])):
            # Heads next to each other in a token, as a projection leaves them.
            state[name] = _randn((b, case["seq"], h, d), gen, dtype).transpose(1, 2)
            state[name + "_out"] = torch.empty((b, case["seq"], h, d), dtype=dtype,
                                               device="cuda").transpose(1, 2)
        return state
    ctx, new = _lengths(case)
    state["ctx_len"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    state["new_len"] = torch.tensor(new, dtype=torch.int32, device="cuda") if case["ragged"] else None
    pages, size, table = _pages(case, gen, case["ctx"] + case["tokens"])
    state["table"] = table
    if case["op"] == "cache":
        state["cache"] = _handle(case, _cache_of(case, gen, pages, size, False), table)
        shape = (b, case["tokens"], case["kv_heads"], d)
        for name in ("k", "v"):
            state[name] = _randn(shape, gen, dtype, _channels(gen, d)).transpose(1, 2)
            state[name + "_out"] = torch.zeros((b, case["kv_heads"], case["tokens"], d), dtype=dtype,
                                               device="cuda")
        return state
    state["cache"] = _handle(case, _cache_of(case, gen, pages, size, True), table)
    t = case["tokens"]
    state["q"] = _randn((b, t, case["heads"], d), gen, dtype).transpose(1, 2)
    state["o"] = torch.zeros((b, t, case["heads"], d), dtype=dtype, device="cuda").transpose(1, 2)
    if case["lse"]:
        state["lse_out"] = torch.zeros((b, case["heads"], t), device="cuda")
    if case["tree"]:
        # Every drafted token continues an earlier one, or (-1) the context.
        at = torch.arange(t, device="cuda").expand(b, t)
        low = torch.clamp(at // 4 - 1, min=-1)
        pick = torch.rand((b, t), generator=gen, device="cuda") * (at - low)
        state["parents"] = torch.minimum(low + pick.long(), at - 1).to(torch.int32)
        state["mask"] = torch.empty((b, t, (t + 63) // 64), dtype=torch.int64, device="cuda")
        state["depth"] = torch.empty((b, t), dtype=torch.int32, device="cuda")
    return state


# ---- one pass -----------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    if state["op"] == "rope":
        return _plain_rope(state)
    if state["op"] == "cache":
        return _plain_cache(state)
    return _plain_attn(state)


def _own(s):
    from frisk_amd import runtime as rt
    if s["op"] == "rope":
        rt.rope(s["q"], s["q_out"], s["positions"], s["table"], k=s["k"], k_out=s["k_out"],
                interleaved=s["interleaved"], backward=s["backward"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if "handle" not in s:  # a program makes it once, with the tensors
        s["handle"] = rt.KvCache(*s["cache"])
    cache = s["handle"]
    if s["op"] == "cache":
        rt.kv_append(s["k"], s["v"], cache, s["ctx_len"], new_len=s["new_len"])
        rt.kv_read(cache, s["k_out"], s["v_out"], s["ctx_len"], new_len=s["new_len"])
        out = {"k": s["k_out"], "v": s["v_out"]}
        if cache.k_scale is not None:
            out |= {"k_scale": cache.k_scale, "v_scale": cache.v_scale}
        return out
    mask = None
    if s["tree"]:
        mask, _ = rt.tree_mask(s["parents"], s["mask"], s["depth"])
    lse = s.get("lse_out")
    rt.tree_attn(s["q"], cache, s["ctx_len"], s["o"], mask=mask, new_len=s["new_len"], lse=lse)
    out = {"o": s["o"]}
    if lse is not None:
        out["lse"] = lse
    if s["tree"]:
        out["depth"] = s["depth"]
    return out


def _plain_rope(s):
    phase = s["positions"].double()[:, None, :, None] * s["freqs"]
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


def _slots(s, at):
    """(page, row of the page) of each sequence's keys `at` ([batch, n])."""
    if s["table"] is None:
        return torch.arange(s["batch"], device="cuda")[:, None].expand_as(at), at
    return s["table"].long().gather(1, at // s["page"]), at % s["page"]


def _plain_cache(s):
    at = s["ctx_len"].long()[:, None] + torch.arange(s["tokens"], device="cuda")
    live = torch.ones_like(at, dtype=torch.bool) if s["new_len"] is None else \
        torch.arange(s["tokens"], device="cuda") < s["new_len"][:, None]
    page, row = _slots(s, at)
    page, row = page[live], row[live]
    ck, cv, ks, vs, _ = s["cache"]
    out = {}
    for name, cache, scales in (("k", ck, ks), ("v", cv, vs)):
        x = s[name].transpose(1, 2)  # [batch, tokens, kv_heads, head_dim]
        if s["kind"] in TOP:
            codes, scale = _quantised(x, s["kind"])
            cache.view(torch.uint8)[page, :, row] = codes.view(torch.uint8)[live]
            scales[page, :, row] = scale[live]
            out[name + "_scale"] = scales
            back = codes.float() * scale[..., None]
        else:
            cache[page, :, row] = x[live]
            back = x.float()
        back = torch.where(live[:, :, None, None], back, 0.0)
        out[name] = back.transpose(1, 2).to(s[name].dtype).contiguous()
    return out


def _ancestors(parents):
    """(bool [batch, t, t]: which drafted tokens each one continues, itself
    among them; how many came before it)."""
    b, t = parents.shape
    up = torch.cat((parents.long(), torch.full((b, 1), -1, device="cuda")), 1)
    up = torch.where(up < 0, t, up)  # place t: the context, its own parent
    seen = torch.eye(t + 1, dtype=torch.bool, device="cuda").expand(b, -1, -1)
    for _ in range(max(1, t).bit_length()):
        seen = seen | seen.gather(1, up[:, :, None].expand(-1, -1, t + 1))
        up = up.gather(1, up)
    seen = seen[:, :t, :t]
    return seen, (seen.sum(-1) - 1).to(torch.int32)


def _seen_keys(s, n):
    """bool [batch, tokens, n]: which of n keys each new token sees; depth."""
    b, t = s["batch"], s["tokens"]
    ctx = s["ctx_len"].long()
    new = torch.full_like(ctx, t) if s["new_len"] is None else s["new_len"].long()
    key = torch.arange(n, device="cuda")
    draft = key - ctx[:, None]  # [batch, n]
    depth = None
    if s["tree"]:
        tree, depth = _ancestors(s["parents"])
        seen = tree.gather(2, draft.clamp(0, t - 1)[:, None, :].expand(b, t, n))
    else:
        seen = draft[:, None, :] <= torch.arange(t, device="cuda")[:, None]
    seen = seen & (draft < new[:, None])[:, None, :]
    return seen | (draft < 0)[:, None, :], depth


def _rows(s, which, scale, n):
    """[batch, kv_heads, n, head_dim] of the cache in 32 bits."""
    at = torch.arange(n, device="cuda").expand(s["batch"], n)
    page, row = _slots(s, at)
    x = s["cache"][which]
    if x.dtype == torch.float8_e4m3fn:
        x = x.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn).float()
    else:
        x = x[page, :, row].float()
    if s["cache"][scale] is not None:
        x = x * s["cache"][scale][page, :, row][..., None]
    return x.transpose(1, 2).contiguous()


def _plain_attn(s):
    b, h, kv, t, d = s["batch"], s["heads"], s["kv_heads"], s["tokens"], s["head_dim"]
    n = s["ctx"] + t
    seen, depth = _seen_keys(s, n)
    k, v = _rows(s, 0, 2, n), _rows(s, 1, 3, n)
    q = s["q"].float().reshape(b, kv, (h // kv) * t, d)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(b, h, t, n)
    score.masked_fill_(~seen[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    o = torch.matmul(weight.view(b, kv, (h // kv) * t, n), v).view(b, h, t, d) / total
    lse = (top + torch.log(total)).squeeze(-1)
    if s["new_len"] is not None:  # rows behind a sequence's last stay as they were
        live = (torch.arange(t, device="cuda") < s["new_len"][:, None])[:, None, :]
        o, lse = torch.where(live[..., None], o, 0.0), torch.where(live, lse, 0.0)
    out = {"o": o.to(s["q"].dtype)}
    if s["lse"]:
        out["lse"] = lse
    if depth is not None:
        out["depth"] = depth
    return out


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    b, d = case["batch"], case["head_dim"]
    e = BYTES[case["dtype"]]
    if case["op"] == "rope":
        tokens = b * case["seq"]
        heads = case["heads"] + case["kv_heads"]
        return {"bytes": 2 * tokens * heads * d * e + 8 * tokens + 4 * case["rot_dim"],
                "flops": 3 * tokens * heads * case["rot_dim"]}
    ctx, new = _lengths(case)
    row = d * BYTES[case["kind"]] + (4 if case["kind"] in TOP else 0)  # one key or value
    if case["op"] == "cache":
        rows = 2 * sum(new) * case["kv_heads"]
        # Read in, written to the cache, written out.
        return {"bytes": rows * (2 * d * e + row), "flops": 4 * rows * d}
    keys = sum(c + n for c, n in zip(ctx, new))
    seen = sum(n * (c + (min(n, n.bit_length()) if case["tree"] else (n + 1) / 2))
               for c, n in zip(ctx, new))
    return {"bytes": int(2 * keys * case["kv_heads"] * row + 2 * sum(new) * case["heads"] * d * e),
            "flops": int(4 * d * case["heads"] * seen)}


# ---- in 64 bits, from the definitions -------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s)
    if case["op"] == "cache":
        return _exact_cache(s)
    return _exact_attn(s)


def _exact_rope(s):
    # Pairs as complex numbers, turned by e^(i p f).
    phase = s["positions"].double()[:, None, :, None] * s["freqs"]
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


def _exact_cache(s):
    b, t = s["batch"], s["tokens"]
    ctx, new = _lengths(s)
    out = {}
    for i, name in enumerate(("k", "v")):
        back = torch.zeros((b, s["kv_heads"], t, s["head_dim"]), dtype=torch.float64, device="cuda")
        scales = s["cache"][2 + i]
        scales = None if scales is None else scales.double()
        for j in range(b):
            x = s[name][j, :, :new[j]].double()  # [kv_heads, new, head_dim]
            if scales is not None:
                scale = (x.abs().amax(-1) / TOP[s["kind"]]).clamp(min=TINY)
                at = torch.arange(ctx[j], ctx[j] + new[j], device="cuda")
                if s["table"] is None:
                    scales[j, :, at] = scale
                else:
                    scales[s["table"][j].long()[at // s["page"]], :, at % s["page"]] = scale.t()
                # x / scale as x top / max, whose ties 64 bits keep.
                top = torch.clamp(x.abs().amax(-1, keepdim=True), min=TOP[s["kind"]] * TINY)
                x = _rounded(x * TOP[s["kind"]] / top, s["kind"]) * scale[..., None]
            back[j, :, :new[j]] = x
        out[name] = back
        if scales is not None:
            out[name + "_scale"] = scales
    return out


def _exact_attn(s):
    b, h, kv, t, d = s["batch"], s["heads"], s["kv_heads"], s["tokens"], s["head_dim"]
    ctx, new = _lengths(s)
    o = torch.zeros((b, h, t, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((b, h, t), dtype=torch.float64, device="cuda")
    parents = s["parents"].tolist() if s["tree"] else None
    for j in range(b):
        n = ctx[j] + new[j]
        at = torch.arange(n, device="cuda")
        page = torch.full_like(at, j) if s["table"] is None else s["table"][j].long()[at // s["page"]]
        row = at if s["table"] is None else at % s["page"]
        hidden = torch.zeros((new[j], n), dtype=torch.bool)
        hidden[:, ctx[j]:] = True
        for i in range(new[j]):
            if s["tree"]:
                up = i
                while up >= 0:
                    hidden[i, ctx[j] + up] = False
                    up = parents[j][up]
            else:
                hidden[i, ctx[j]:ctx[j] + i + 1] = False
        hidden = hidden.cuda()
        for g in range(kv):
            kk, vv = (s["cache"][i][:, g].view(torch.uint8)[page, row].view(torch.float8_e4m3fn).double()
                      if s["kind"] == "e4m3" else s["cache"][i][:, g][page, row].double()
                      for i in (0, 1))
            if s["kind"] in TOP:
                kk = kk * s["cache"][2][:, g][page, row].double()[:, None]
                vv = vv * s["cache"][3][:, g][page, row].double()[:, None]
            for head in range(g * (h // kv), (g + 1) * (h // kv)):
                score = (s["q"][j, head, :new[j]].double() @ kk.t()) / math.sqrt(d)
                score = score.masked_fill(hidden, -math.inf)
                lse[j, head, :new[j]] = torch.logsumexp(score, -1)
                o[j, head, :new[j]] = torch.exp(score - lse[j, head, :new[j], None]) @ vv
    out = {"o": o}
    if s["lse"]:
        out["lse"] = lse
    if s["tree"]:
        out["depth"] = None
    return out
