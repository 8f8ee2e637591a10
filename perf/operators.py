"""Cases and plain forms of the operators that serve a decoder from a paged key/value cache.

Four operators, reached through ``llm_kernels`` where ``own`` is true:

* ``rotary``  - rotary position embedding of queries and keys, positions with one or several
  axes (time, height, width), forward and gradient (``rotary_embed``);
* ``append``  - rotation of the new queries and keys and the write of the new keys and values
  into the pages of the cache (``paged_kv_append``);
* ``paged``   - attention of each sequence's newest tokens to its own pages
  (``paged_attention``);
* ``prefix``  - the same for a batch whose sequences share one long prefix, which is read and
  multiplied once for all of them (``shared_prefix_attention``).

Where ``own`` is false ``run`` computes them from elementary torch operations in 32 bits.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_TABLE_ROWS = 40000  # positions that the rotary tables of these cases cover


def _kernels():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attn-from-scratch_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import llm_kernels

    return llm_kernels


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # One short training sample of a small model, adjacent pairs rotated, fp16.
        {"name": "rotary short", "op": "rotary", "tokens": 60, "heads": 8, "kv_heads": 8, "dim": 64, "rotary_dim": 64,
         "dtype": "f16", "sections": "", "interleaved": True},
        # A training step's packed image and video tokens: (time, height, width) positions.
        {"name": "rotary video", "op": "rotary", "tokens": 16380, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary_dim": 128, "dtype": "bf16", "sections": "16-24-24", "interleaved": False},
        # One decode step of a batch of 16.
        {"name": "append decode", "op": "append", "tokens": 16, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary_dim": 128, "dtype": "bf16", "sections": "", "interleaved": False, "page": 16, "padding": 0},
        # A step that mixes prompts and single tokens, padded to a fixed count; rotation of half
        # of each head, adjacent pairs.
        {"name": "append mixed", "op": "append", "tokens": 1531, "heads": 24, "kv_heads": 6, "dim": 64,
         "rotary_dim": 32, "dtype": "f16", "sections": "", "interleaved": True, "page": 64, "padding": 37},
        # The prompts of a batch (4 x 4096 tokens, 32 heads as in the decoder layer).
        {"name": "append prompts", "op": "append", "tokens": 16384, "heads": 32, "kv_heads": 32, "dim": 128,
         "rotary_dim": 128, "dtype": "bf16", "sections": "", "interleaved": False, "page": 16, "padding": 0},
        # One user's next token.
        {"name": "paged one sequence", "op": "paged", "batch": 1, "new": 1, "min_len": 1000, "max_len": 1000, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 16, "lse": False},
        # A served batch with contexts of all lengths: the bulk of decode time.
        {"name": "paged batch", "op": "paged", "batch": 64, "new": 1, "min_len": 200, "max_len": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 16, "lse": False},
        # Four drafted tokens checked at once; one key/value head per query head, fp16.
        {"name": "paged drafted", "op": "paged", "batch": 16, "new": 4, "min_len": 4, "max_len": 2999, "heads": 16,
         "kv_heads": 16, "dim": 64, "dtype": "f16", "page": 32, "lse": True},
        # The next 500 prompt tokens of each of four long prompts.
        {"name": "paged prompt piece", "op": "paged", "batch": 4, "new": 500, "min_len": 500, "max_len": 9000, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "lse": False},
        # Five answers sampled from one question.
        {"name": "prefix few", "op": "prefix", "batch": 5, "new": 1, "prefix": 1111, "min_len": 0, "max_len": 60,
         "heads": 16, "kv_heads": 2, "dim": 64, "dtype": "f16", "page": 16},
        # A batch behind one system prompt.
        {"name": "prefix batch", "op": "prefix", "batch": 32, "new": 1, "prefix": 8192, "min_len": 1, "max_len": 512,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 16},
        # Many questions about one long document: the largest.
        {"name": "prefix document", "op": "prefix", "batch": 256, "new": 1, "prefix": 32768, "min_len": 16,
         "max_len": 1024, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 32},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "paged", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8])
    if op in ("rotary", "append"):
        half = dim // 2
        sections = rng.choice(["", "", "%d-%d" % (half // 4, half - half // 4),
                               "%d-%d-%d" % (half // 4, 3 * half // 8, 3 * half // 8)])
        case = {"op": op, "tokens": _log(rng, 1, 8000), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary_dim": dim if sections else rng.choice([dim, dim, half]), "dtype": dtype, "sections": sections,
                "interleaved": rng.random() < 0.3}
        if op == "append":
            case.update(page=rng.choice([8, 16, 16, 32, 64, 128]), padding=rng.choice([0, 0, case["tokens"] // 7]))
        return case
    new = rng.choice([1, 1, 1, 2, 3, 5, _log(rng, 8, 300)])
    batch = _log(rng, 1, 96)
    case = {"op": op, "batch": batch, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page": rng.choice([8, 16, 16, 32, 64, 128])}
    # The plain form holds every sequence's keys in 32 bits and the scores of every row.
    room = 400_000_000
    most = max(1, min(16384, room // (batch * kv_heads * dim), room // (batch * heads * new)))
    if op == "paged":
        case.update(max_len=_log(rng, 1, most), lse=rng.random() < 0.5)
        case["min_len"] = min(case["max_len"], rng.choice([0, 1, new, case["max_len"]]))
    else:
        case.update(prefix=_log(rng, 16, most), max_len=_log(rng, 1, min(most, 1024)))
        case["min_len"] = min(case["max_len"], rng.choice([0, 1, new]))
    return case


def _lengths(case):
    """Each sequence's count of keys: spread over the case's range, the same for every seed."""
    lo, hi = case["min_len"], case["max_len"]
    return [lo + int((hi - lo + 1) * (((b + 1) * 0.6180339887498949) % 1.0)) for b in range(case["batch"])]


def _sections(case):
    return tuple(int(s) for s in case["sections"].split("-")) if case["sections"] else None


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def _rotary_table(dim, device):
    freq = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    angle = torch.arange(_TABLE_ROWS, dtype=torch.float64, device=device)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float().contiguous()


def _positions(case, gen, device):
    T = case["tokens"]
    start = int(torch.randint(0, 1000, (1,), generator=gen, device=device))
    steps = torch.arange(T, device=device)
    axes = case["sections"].count("-") + 1 if case["sections"] else 1
    if axes == 1:
        return steps % 20000 + start
    # Frames of patches: time, then row, then column.
    width = max(1, min(48, math.isqrt(T)))
    per = width * width
    grid = [steps // per + start, steps % per // width + start, steps % width + start]
    return torch.stack(grid[:1] + grid[2:] if axes == 2 else grid)


def _pages(lengths, page, first, gen, device, rows):
    """Block table [rows, most pages], -1 where a sequence has none; page ids in random order."""
    counts = [-(-n // page) for n in lengths]
    width = max(1, max(counts, default=1))
    ids = torch.randperm(sum(counts), generator=gen, device=device).to(torch.int32) + first
    table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
    held = torch.arange(width, device=device)[None, :] < torch.tensor(counts, device=device)[:, None]
    table[held] = ids
    return table, sum(counts)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=device, dtype=torch.float32) * scale).to(dt)

    if case["op"] in ("rotary", "append"):
        T = case["tokens"]
        state = {"op": case["op"], "sections": _sections(case), "interleaved": case["interleaved"],
                 "positions": _positions(case, gen, device), "table": _rotary_table(case["rotary_dim"], device)}
        # Queries, keys and values as the one projection of a layer leaves them.
        qkv = normal(T, H + 2 * Hk, D)
        state["q"], state["k"], state["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        if case["op"] == "rotary":
            state["q"], state["k"] = state["q"].detach().requires_grad_(), state["k"].detach().requires_grad_()
            state["gq"], state["gk"] = normal(T, H, D), normal(T, Hk, D)
            return state
        page = case["page"]
        pages = -(-T // page) * 5 // 4 + 1
        # Sequences lie in whole pages; the tokens of a page are in order.
        order = torch.randperm(pages, generator=gen, device=device)[: -(-T // page)]
        slots = (order[:, None] * page + torch.arange(page, device=device)).reshape(-1)[:T].contiguous()
        if case["padding"]:
            slots[T - case["padding"]:] = -1
        state["slots"] = slots
        state["k_cache"], state["v_cache"] = normal(pages, page, Hk, D), normal(pages, page, Hk, D)
        return state

    B, page = case["batch"], case["page"]
    lengths = _lengths(case)
    state = {"op": case["op"], "lse": case.get("lse", False)}
    first = 0
    if case["op"] == "prefix":
        first = -(-case["prefix"] // page)
        state["prefix_pages"] = torch.randperm(first, generator=gen, device=device).to(torch.int32)
        state["prefix"] = case["prefix"]
    state["block_table"], count = _pages(lengths, page, first, gen, device, B)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    state["q"] = normal(B, case["new"], H, D, scale=1.5)
    state["k_cache"], state["v_cache"] = normal(first + count + 1, page, Hk, D), normal(first + count + 1, page, Hk, D)
    return state


# ---------------------------------------------------------------------------------------------
# The operators
# ---------------------------------------------------------------------------------------------
def _angles(positions, table, sections):
    """cos and sin of every token and pair, [T, 1, pairs]: pair i goes by its axis' position."""
    if sections is None:
        rows = table[positions]
    else:
        axis = torch.repeat_interleave(torch.arange(len(sections), device=table.device),
                                       torch.tensor(sections, device=table.device))
        rows = table[positions[axis].t(), torch.arange(table.shape[1], device=table.device)]
    return rows[..., 0].unsqueeze(1), rows[..., 1].unsqueeze(1)


def _rotate(x, cos, sin, interleaved):
    dim, pairs = x.shape[-1], cos.shape[-1]
    f = x.detach().float()
    if interleaved:
        a, b = f[..., 0:2 * pairs:2], f[..., 1:2 * pairs:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = f[..., :pairs], f[..., pairs:2 * pairs]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    if 2 * pairs < dim:
        turned = torch.cat((turned, f[..., 2 * pairs:]), -1)
    return turned.to(x.dtype)


def _keys(cache, pages):
    """The keys or values behind a block table, [rows, most keys, kv heads, dim], in 32 bits."""
    return cache[pages.clamp_min(0).long()].flatten(1, 2).float()


def _plain_rotary(s):
    cos, sin = _angles(s["positions"], s["table"], s["sections"])
    turn = lambda x, sn: _rotate(x, cos, sn, s["interleaved"])  # noqa: E731
    return {"q": turn(s["q"], sin), "k": turn(s["k"], sin), "dq": turn(s["gq"], -sin), "dk": turn(s["gk"], -sin)}


def _plain_append(s):
    cos, sin = _angles(s["positions"], s["table"], s["sections"])
    q, k = (_rotate(s[n], cos, sin, s["interleaved"]) for n in ("q", "k"))
    kept = s["slots"] >= 0
    at = s["slots"][kept]
    s["k_cache"].view(-1, *k.shape[1:])[at] = k[kept]
    s["v_cache"].view(-1, *k.shape[1:])[at] = s["v"][kept]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    q = s["q"]
    B, new, H, D = q.shape
    Hk = s["k_cache"].shape[2]
    qf = q.float().view(B, new, Hk, H // Hk, D) * D ** -0.5
    k, v = _keys(s["k_cache"], s["block_table"]), _keys(s["v_cache"], s["block_table"])
    at = torch.arange(k.shape[1], device=q.device)
    # Query i of a sequence's newest tokens sees its keys up to its own place among them.
    last = s["lengths"][:, None] - new + torch.arange(new, device=q.device) + 1
    seen = (at < last[..., None])[:, None, None]  # [B, 1, 1, new, keys]
    scores = torch.einsum("bnhgd,bkhd->bhgnk", qf, k).masked_fill(~seen, -math.inf)
    if "prefix" in s:
        pk = _keys(s["k_cache"], s["prefix_pages"][None])[0, : s["prefix"]]
        pv = _keys(s["v_cache"], s["prefix_pages"][None])[0, : s["prefix"]]
        before = torch.einsum("bnhgd,khd->bhgnk", qf, pk)
        top = torch.maximum(scores.amax(-1, keepdim=True), before.amax(-1, keepdim=True))
    else:
        top = scores.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    # What lies behind a sequence's end is not its own: no value of it is multiplied.
    own_keys = (at < s["lengths"][:, None])[..., None, None]
    out = torch.einsum("bhgnk,bkhd->bhgnd", p, v.masked_fill(~own_keys, 0.0))
    if "prefix" in s:
        e = (before - top).exp()
        total = total + e.sum(-1, keepdim=True)
        out = out + torch.einsum("bhgnk,khd->bhgnd", e, pv)
    out = out / total.masked_fill(total == 0, 1.0)
    answer = {"out": out.permute(0, 3, 1, 2, 4).reshape(B, new, H, D).to(q.dtype)}
    if s["lse"]:
        answer["lse"] = (top + total.log()).permute(0, 3, 1, 2, 4).reshape(B, new, H)
    return answer


def run(state):
    s = state
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append}.get(s["op"], _plain_attention)(s)
    lk = _kernels()
    if s["op"] == "rotary":
        q, k = lk.rotary_embed(s["q"], s["k"], s["positions"], s["table"], sections=s["sections"],
                               interleaved=s["interleaved"])
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if s["op"] == "append":
        q = lk.paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], q=s["q"],
                               positions=s["positions"], cos_sin=s["table"], sections=s["sections"],
                               interleaved=s["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if s["op"] == "paged":
        got = lk.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["lengths"],
                                 return_lse=s["lse"])
        return {"out": got[0], "lse": got[1]} if s["lse"] else {"out": got}
    return {"out": lk.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"], s["prefix"],
                                              s["block_table"], s["lengths"])}


def work(case):
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] in ("rotary", "append"):
        T, R = case["tokens"], case["rotary_dim"]
        axes = case["sections"].count("-") + 1 if case["sections"] else 1
        most = min(T * axes, _TABLE_ROWS) * R * 4  # rows of the table that the tokens can name
        turned = 3.0 * T * (H + Hk) * R  # two products and a sum for each rotated value
        if case["op"] == "rotary":
            return {"bytes": 2 * 2 * 2 * T * (H + Hk) * D + most + 8 * T * axes, "flops": 2 * turned}
        return {"bytes": 2 * 2 * T * (H + 2 * Hk) * D + most + 8 * T * axes + 8 * T, "flops": turned}
    B, new, lengths = case["batch"], case["new"], _lengths(case)
    keys = sum(lengths) + case.get("prefix", 0)
    pages = sum(-(-n // case["page"]) for n in lengths) + -(-case.get("prefix", 0) // case["page"])
    seen = sum(max(0, n - new + i + 1) for n in lengths for i in range(new)) + B * new * case.get("prefix", 0)
    moved = 2 * 2 * keys * Hk * D + 2 * 2 * B * new * H * D + 4 * pages + 4 * B
    return {"bytes": moved + (4 * B * new * H if case.get("lse") else 0), "flops": 4.0 * seen * H * D}


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_turn(x, positions, table, sections, interleaved, sign):
    """Each pair is a complex number, multiplied by that of its angle."""
    T, pairs = x.shape[0], table.shape[1]
    angle = torch.empty(T, pairs, dtype=torch.complex128, device=x.device)
    wide = torch.complex(table[..., 0].double(), sign * table[..., 1].double())
    begin = 0
    for axis, count in enumerate(sections or (pairs,)):
        where = positions[axis] if sections else positions
        angle[:, begin:begin + count] = wide[where][:, begin:begin + count]
        begin += count
    y = x.detach().double().clone()
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    z = torch.complex(y[..., first], y[..., second]) * angle[:, None, :]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rotary", "append"):
        turn = lambda x, sign: _exact_turn(x, s["positions"], s["table"], s["sections"], s["interleaved"], sign)  # noqa: E731
        if case["op"] == "rotary":
            return {"q": turn(s["q"], 1), "k": turn(s["k"], 1), "dq": turn(s["gq"], -1), "dk": turn(s["gk"], -1)}
        k_new, k_cache, v_cache = turn(s["k"], 1), s["k_cache"].double(), s["v_cache"].double()
        page = case["page"]
        kept = (s["slots"] >= 0).nonzero()[:, 0]
        where = s["slots"][kept]
        k_cache[where // page, where % page] = k_new[kept]
        v_cache[where // page, where % page] = s["v"].double()[kept]
        return {"q": turn(s["q"], 1), "k_cache": k_cache, "v_cache": v_cache}
    B, new, H, Hk, D, page = (case[n] for n in ("batch", "new", "heads", "kv_heads", "dim", "page"))
    out = torch.zeros(B, new, H, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((B, new, H), -math.inf, dtype=torch.float64, device=s["q"].device)

    def rows(cache, pages, count):
        return cache[pages[: -(-count // page)].long()].double().reshape(-1, Hk, D)[:count]

    prefix = case.get("prefix", 0)
    shared = [rows(s[n], s["prefix_pages"], prefix) if prefix else None for n in ("k_cache", "v_cache")]
    for b, n in enumerate(_lengths(case)):
        k, v = rows(s["k_cache"], s["block_table"][b], n), rows(s["v_cache"], s["block_table"][b], n)
        if prefix:
            k, v = torch.cat((shared[0], k)), torch.cat((shared[1], v))
        if not k.shape[0]:
            continue
        end = prefix + torch.arange(n - new + 1, n + 1, device=k.device).clamp_min(0)
        hidden = torch.arange(k.shape[0], device=k.device)[None, :] >= end[:, None]
        for h in range(Hk):
            heads = slice(h * (H // Hk), (h + 1) * (H // Hk))
            x = torch.matmul(s["q"][b, :, heads].double().transpose(0, 1), k[:, h].t()) / math.sqrt(D)
            x = x.masked_fill(hidden, -math.inf)
            norm = torch.logsumexp(x, -1, keepdim=True)
            p = torch.where(hidden, torch.zeros_like(x), (x - norm).exp())
            out[b, :, heads] = torch.matmul(p, v[:, h]).transpose(0, 1)
            lse[b, :, heads] = norm[..., 0].t()
    return {"out": out, "lse": lse} if case.get("lse") else {"out": out}
