"""Operators around a language model's attention, measured as its programs call them.

Four operators, used one after the other when a model trains or answers:

* ``rotary``  ``tg.nn.norm_rotary``: RMS norm of the queries and keys of each head and the rotation
  by their positions, forward, and with its gradients;
* ``append``  ``Graph.append``: the new tokens' keys and values into their slots of a paged cache,
  with the sums of the keys of every touched page;
* ``attend``  dot-product attention over ``Graph.paged``: one or a few new tokens of each sequence
  over its pages of the cache;
* ``sparse``  ``Graph.select_pages`` and the attention over what it selects: the newest page and the
  pages whose key sums score highest, for each token and key head.

``own`` false: the same operators in elementary Torch operations.  Inputs are synthetic, made on the
GPU from a seed.
"""

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def _tiga():
    """The framework (its folder is not importable by name)."""
    path = os.path.join(os.getcwd(), "tiga-lang_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import tiga

    return tiga


# ---------------------------------------------------------------------------
# Cases

def listed():
    return [
        # One sequence answered token by token: the smallest call, latency counts.
        dict(name="attend_one", op="attend", batch=1, low=1500, high=1500, short=False, tokens=1,
             heads=8, group=4, dim=128, page=16, dtype="bf16", lengths_seed=1),
        # A served batch of ragged sequences.
        dict(name="attend_batch", op="attend", batch=64, low=100, high=4000, short=False, tokens=1,
             heads=8, group=4, dim=128, page=16, dtype="bf16", lengths_seed=2),
        # A few very long sequences: the length has to be split.
        dict(name="attend_long", op="attend", batch=4, low=100000, high=131072, short=False,
             tokens=1, heads=8, group=4, dim=128, page=64, dtype="bf16", lengths_seed=3),
        # A few new tokens of each sequence at once (drafted tokens being checked), one head a
        # group, pages that end inside every tile, and sequences shorter than the tokens asked for.
        dict(name="attend_few", op="attend", batch=24, low=200, high=3000, short=True, tokens=4,
             heads=16, group=1, dim=64, page=24, dtype="f16", lengths_seed=4),
        # One long sequence answered over a small part of its pages.
        dict(name="sparse_one", op="sparse", batch=1, low=65500, high=65500, short=False, tokens=1,
             heads=8, group=4, dim=128, page=16, dtype="bf16", lengths_seed=5, count=64),
        # The same for a served batch.
        dict(name="sparse_batch", op="sparse", batch=32, low=2000, high=48000, short=False,
             tokens=1, heads=8, group=4, dim=128, page=64, dtype="bf16", lengths_seed=6, count=24),
        # The queries and keys of a decode step at far positions.
        dict(name="rotary_decode", op="rotary", tokens=48, q_heads=32, k_heads=8, dim=128,
             sections="64", far=1000000, interleaved=False, dtype="bf16", train=False),
        # A training step over a packed batch, forward and backward.
        dict(name="rotary_train", op="rotary", tokens=16384, q_heads=32, k_heads=8, dim=128,
             sections="64", far=8192, interleaved=False, dtype="bf16", train=True),
        # Video patches: time, height and width, adjacent pairs, in 32 bits, with gradients.
        dict(name="rotary_video", op="rotary", tokens=3137, q_heads=12, k_heads=12, dim=96,
             sections="16,16,16", far=300, interleaved=True, dtype="f32", train=True),
        # A long prompt, half of every head rotated.
        dict(name="rotary_prompt", op="rotary", tokens=40001, q_heads=16, k_heads=16, dim=64,
             sections="16", far=40001, interleaved=False, dtype="f16", train=False),
        # One new token of each sequence of a served batch.
        dict(name="append_step", op="append", batch=64, low=1, high=500, short=False, tokens=1,
             heads=8, group=1, dim=128, page=16, dtype="bf16", lengths_seed=7),
        # Prompts of 1500 tokens each, some behind an earlier part.
        dict(name="append_prompt", op="append", batch=8, low=1500, high=4000, short=False,
             tokens=1500, heads=16, group=1, dim=64, page=64, dtype="f16", lengths_seed=8),
    ]


def _log(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["attend", "sparse", "rotary", "append"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "rotary":
        interleaved = rng.random() < 0.5
        dim = rng.choice([32, 64, 80, 96, 128, 192, 256])
        half = rng.choice([dim // 2, dim // 4])
        axes = rng.choice([1, 1, 2, 3])
        first = half // axes // 2 * 2
        sections = ",".join(map(str, [half - first * (axes - 1)] + [first] * (axes - 1)))
        k_heads = rng.choice([1, 2, 4, 8, 12])
        q_heads = k_heads * rng.choice([1, 2, 3, 4])
        most = max(2, 16384 * 40 * 128 // ((q_heads + k_heads) * dim))
        return dict(op=op, tokens=_log(rng, 1, min(40000, most)), q_heads=q_heads, k_heads=k_heads,
                    dim=dim, sections=sections, far=_log(rng, 10, 1000000),
                    interleaved=interleaved, dtype=rng.choice(["f32", "bf16", "f16"]),
                    train=rng.random() < 0.5)
    dim = rng.choice([32, 64, 128])
    heads = rng.choice([1, 2, 4, 8, 16])
    page = rng.choice([8, 16, 24, 32, 48, 64, 100, 128])
    batch = _log(rng, 1, 64)
    if op == "append":
        tokens = 1 if rng.random() < 0.5 else _log(rng, 2, 2000)
        batch = max(1, min(batch, 16000 // tokens))
        high = tokens + _log(rng, 1, 500)
        return dict(op=op, batch=batch, low=rng.randint(1, high), high=high, short=False,
                    tokens=tokens, heads=heads, group=1, dim=dim, page=page, dtype=dtype,
                    lengths_seed=rng.randrange(1 << 30))
    # At most as many cached values as the longest listed cases hold.
    most = max(2, 400000 * 8 * 128 // (batch * heads * dim))
    high = _log(rng, 1, min(131072, most))
    case = dict(op=op, batch=batch, low=max(1, high // rng.choice([1, 2, 10])), high=high,
                short=rng.random() < 0.3, tokens=rng.choice([1, 1, 2, 3, 5]), heads=heads,
                group=rng.choice([1, 2, 4, 5, 8, 16]), dim=dim, page=page, dtype=dtype,
                lengths_seed=rng.randrange(1 << 30))
    if op == "sparse":
        rows = batch * case["tokens"] * heads * dim * page
        case["count"] = _log(rng, 1, max(1, min(64, 200_000_000 // rows)))
    return case


def _sections(case):
    """Frequencies of each axis of the positions."""
    return tuple(int(n) for n in case["sections"].split(","))


def _lengths(case):
    """Cached tokens of each sequence: the longest first; with `short` the last three hold 0, 1 and
    2 tokens."""
    rng = random.Random(case["lengths_seed"])
    lengths = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    lengths[0] = case["high"]
    if case["short"]:
        for k in range(min(3, case["batch"] - 1)):
            lengths[-1 - k] = k
    return lengths


def _visible(case):
    """Cached tokens that each query row sees, a list of `tokens` for each sequence."""
    t = case["tokens"]
    return [[max(0, n - t + 1 + j) for j in range(t)] for n in _lengths(case)]


# ---------------------------------------------------------------------------
# Work

def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        n, dim = case["tokens"], case["dim"]
        rows = n * (case["q_heads"] + case["k_heads"])
        fixed = 8 * n * len(_sections(case)) + 4 * sum(_sections(case)) + 2 * size * dim
        passes = 5 if case["train"] else 2   # x, y; and dy, dx with x again
        return {"bytes": passes * rows * dim * size + fixed,
                "flops": rows * dim * (22 if case["train"] else 7)}
    heads, dim, page, group = case["heads"], case["dim"], case["page"], case["group"]
    lengths, t = _lengths(case), case["tokens"]
    if case["op"] == "append":
        rows = sum(min(n, t) for n in lengths)
        older = sum((n - min(n, t)) % page for n in lengths)
        pages = sum((n + page - 1) // page - (n - min(n, t)) // page for n in lengths)
        return {"bytes": heads * dim * (4 * rows * size + older * size + 4 * pages) + 8 * rows,
                "flops": heads * dim * (rows + older)}
    rows = case["batch"] * t
    ends = 2 * rows * heads * group * dim * size
    seen = _visible(case)
    if case["op"] == "attend":
        keys = sum(lengths)
        table = 4 * sum((n + page - 1) // page for n in lengths)
        return {"bytes": 2 * keys * heads * dim * size + ends + table + 4 * len(lengths),
                "flops": 4 * heads * group * dim * sum(sum(s) for s in seen)}
    ranked = sum(max((n + page - 1) // page - 1, 0) for n in lengths)
    keys, flops = 0, 0
    for row in seen:
        for n in row:
            pages = (n + page - 1) // page
            kept = min(pages, case["count"])
            got = (kept - 1) * page + n - (pages - 1) * page if n else 0
            keys += got if row[-1] == n else min(got, page)   # the tokens of one sequence share pages
            flops += 4 * group * dim * got + 2 * dim * max(pages - 1, 0)
    return {"bytes": heads * (4 * dim * ranked + 2 * dim * size * keys + 4 * rows * case["count"])
            + ends, "flops": heads * flops}


# ---------------------------------------------------------------------------
# Inputs

def _cache_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    heads, dim, page, t = case["heads"], case["dim"], case["page"], case["tokens"]
    lengths = _lengths(case)
    used = [(n + page - 1) // page for n in lengths]
    width = max(used) + 2
    num_pages = sum(used) + 3
    order = torch.randperm(num_pages, device=DEV, generator=g).to(torch.int32).cpu()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    s = dict(case=case, page=page, num_pages=num_pages, table=table.to(DEV),
             lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV))
    make = lambda *shape: torch.randn(shape, device=DEV, dtype=dtype, generator=g)
    s["keys"] = make(num_pages * page, heads, dim)
    s["values"] = make(num_pages * page, heads, dim)
    rows = len(lengths) * t
    if case["op"] == "append":
        s["new_keys"], s["new_values"] = make(rows, heads, dim), make(rows, heads, dim)
        s["sums"] = torch.randn(num_pages, heads, dim, device=DEV, generator=g)
        return s
    s["query"] = make(rows, heads, case["group"], dim)
    s["scale"] = dim ** -0.5
    if case["op"] == "sparse":
        s["sums"] = torch.cat([part.float().sum(1) for part in
                               s["keys"].view(num_pages, page, heads, dim).split(256)])
    return s


def _rotary_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    n, hq, hk, dim = case["tokens"], case["q_heads"], case["k_heads"], case["dim"]
    # Queries, keys and values of one projection, as a model splits them.
    qkv = torch.randn(n, hq + 2 * hk, dim, device=DEV, dtype=dtype, generator=g)
    half = sum(_sections(case))
    base = torch.arange(half, device=DEV, dtype=torch.float64) / half
    s = dict(case=case, query=qkv[:, :hq], key=qkv[:, hq:hq + hk],
             frequencies=torch.pow(torch.tensor(10000.0, device=DEV, dtype=torch.float64),
                                   -base).float(),
             positions=torch.randint(0, case["far"], (n, len(_sections(case))), device=DEV,
                                     generator=g))
    weight = lambda: (1 + 0.2 * torch.randn(dim, device=DEV, generator=g)).to(dtype)
    s["q_weight"], s["k_weight"] = weight(), weight()
    if case["train"]:
        s["d_query"] = torch.randn(n, hq, dim, device=DEV, dtype=dtype, generator=g)
        s["d_key"] = torch.randn(n, hk, dim, device=DEV, dtype=dtype, generator=g)
        for name in ("query", "key", "q_weight", "k_weight"):
            s[name] = s[name].detach().requires_grad_(True)
    return s


def _inputs(case, seed):
    return (_rotary_inputs if case["op"] == "rotary" else _cache_inputs)(case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] != "rotary":
        tg = _tiga()

        class Attention(tg.MessagePassing):
            reducer = tg.online_softmax()

            def edge(self, src, dst, edge, scale):
                return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)

        s["graph"] = tg.Graph.paged(s["table"], s["lengths"], page_size=s["page"],
                                    num_pages=s["num_pages"], queries=case["tokens"])
        if case["op"] == "attend":
            s["attend"] = Attention().prepare(
                graph=s["graph"], src={"key": s["keys"][:, :, None], "value": s["values"][:, :, None]},
                dst={"query": s["query"]}, scale=s["scale"])
        if case["op"] == "sparse":
            # The selected relation counts a row for every (token, key head).
            flat = lambda t: t.view(-1, 1, case["dim"])
            s["chosen"] = s["graph"].select_pages(s["query"], s["sums"], case["count"])
            s["attend"] = Attention().prepare(
                graph=s["chosen"], src={"key": flat(s["keys"]), "value": flat(s["values"])},
                dst={"query": s["query"].view(-1, case["group"], case["dim"])}, scale=s["scale"])
    return s


# ---------------------------------------------------------------------------
# One pass

def run(state):
    op = state["case"]["op"]
    return (_own if own else _plain)[op](state)


def _own_attend(s):
    return s["attend"]()


def _own_sparse(s):
    chosen = s["graph"].select_pages(s["query"], s["sums"], s["case"]["count"], out=s["chosen"])
    out = s["attend"]()
    return chosen.page_table, chosen.lengths, out.view(s["query"].shape)


def _own_append(s):
    s["graph"].append(s["keys"], s["new_keys"], s["values"], s["new_values"], page_sums=s["sums"])
    return s["keys"], s["values"], s["sums"]


def _own_rotary(s):
    case = s["case"]
    out = _tiga().nn.norm_rotary(
        s["query"], s["key"], s["positions"], s["frequencies"], query_weight=s["q_weight"],
        key_weight=s["k_weight"], eps=EPS, sections=_sections(case),
        interleaved=case["interleaved"])
    return _with_gradients(s, out)


def _with_gradients(s, out):
    if not s["case"]["train"]:
        return out
    leaves = (s["query"], s["key"], s["q_weight"], s["k_weight"])
    grads = torch.autograd.grad(out, leaves, (s["d_query"], s["d_key"]))
    return tuple(o.detach() for o in out) + grads


# The plain forms.

def _slots(table, page, num_pages):
    """(slot, whether it exists) of every position the page tables reach."""
    at = torch.arange(table.shape[-1] * page, device=table.device)
    ids = table[..., at // page].long()
    ok = (ids >= 0) & (ids < num_pages)
    return torch.where(ok, ids, 0) * page + at % page, ok


def _limits(s):
    """Cached tokens that each query row sees, [sequences, tokens]."""
    t = s["case"]["tokens"]
    return s["lengths"].long()[:, None] - t + 1 + torch.arange(t, device=DEV)


def _softmax_sum(q, k, v, seen, scale):
    """q [..., rows, D], k and v [..., keys, D], seen [..., rows, keys]."""
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight / torch.where(total == 0, 1.0, total), v)


def _plain_attend(s):
    case = s["case"]
    t, group, heads, dim = case["tokens"], case["group"], case["heads"], case["dim"]
    slots, ok = _slots(s["table"], s["page"], s["num_pages"])            # [B, keys]
    batch, keys = slots.shape
    k = s["keys"][slots].float().permute(0, 2, 1, 3)                      # [B, heads, keys, D]
    v = torch.where(ok[:, None, :, None], s["values"][slots].float().permute(0, 2, 1, 3), 0.0)
    q = s["query"].float().view(batch, t, heads, group, dim).permute(0, 2, 1, 3, 4)
    seen = ok[:, None] & (torch.arange(keys, device=DEV) < _limits(s)[..., None])   # [B, t, keys]
    seen = seen[:, None, :, None].expand(batch, 1, t, group, keys).reshape(batch, 1, t * group, keys)
    out = _softmax_sum(q.reshape(batch, heads, t * group, dim), k, v, seen, s["scale"])
    out = out.view(batch, heads, t, group, dim).permute(0, 2, 1, 3, 4)
    return out.reshape(batch * t, heads, group, dim).to(s["query"].dtype)


def _plain_sparse(s):
    case = s["case"]
    t, page, count = case["tokens"], s["page"], case["count"]
    limit = _limits(s).clamp(min=0).reshape(-1)                           # [rows]
    rows, width = limit.numel(), s["table"].shape[1]
    pages = (limit + page - 1) // page
    ids = s["table"].long().repeat_interleave(t, 0)                       # [rows, width]
    ok = (ids >= 0) & (ids < s["num_pages"])
    # Scores in 64 bits: the choice turns on values next to each other.
    sums = s["sums"][torch.where(ok, ids, 0)].double()                    # [rows, width, heads, D]
    score = (s["query"].double().sum(2)[:, None] * sums).sum(-1)          # [rows, width, heads]
    score = torch.where(torch.isnan(score) | ~ok[..., None], -torch.inf, score).transpose(1, 2)
    at = torch.arange(width, device=DEV)
    last = (pages - 1)[:, None, None]
    # The newest page first, then by score, what is not there at the end; ties to the lowest.
    order = torch.argsort(score, dim=-1, descending=True, stable=True)
    rank = torch.where(order == last, 0, torch.where(order > last, 2, 1))
    order = order.gather(-1, torch.argsort(rank, dim=-1, stable=True))
    kept = pages.clamp(max=count)
    if width < count:
        order = torch.cat([order, order.new_full((*order.shape[:2], count - width), width)], -1)
    order = order[..., :count]
    there = torch.arange(count, device=DEV) < kept[:, None, None]
    order = torch.where(there, order, width).sort(-1).values
    got = ids[:, None].expand(rows, order.shape[1], width).gather(-1, order.clamp(max=width - 1))
    table = torch.where(there, got, -1)
    length = torch.where(limit > 0, (kept - 1) * page + limit - (pages - 1) * page, 0)
    # Attention over the selected pages, a table for each (row, key head).
    slots, ok = _slots(table, page, s["num_pages"])                       # [rows, heads, keys]
    head = torch.arange(slots.shape[1], device=DEV)[:, None]
    k = s["keys"][slots, head].float()                                    # [rows, heads, keys, D]
    v = torch.where(ok[..., None], s["values"][slots, head].float(), 0.0)
    seen = ok & (torch.arange(slots.shape[2], device=DEV) < length[:, None, None])
    out = _softmax_sum(s["query"].float(), k, v, seen[:, :, None], s["scale"])
    return table.to(torch.int32), length.to(torch.int32), out.to(s["query"].dtype)


def _plain_append(s):
    case = s["case"]
    t, page, batch = case["tokens"], s["page"], case["batch"]
    length = s["lengths"].long()
    at = length[:, None] - t + torch.arange(t, device=DEV)                # [B, t]
    there = at >= 0
    ids = s["table"].long().gather(1, at.clamp(min=0) // page)
    slots = (ids * page + at.clamp(min=0) % page)[there]
    s["keys"][slots] = s["new_keys"].view(batch, t, *s["keys"].shape[1:])[there]
    s["values"][slots] = s["new_values"].view(batch, t, *s["values"].shape[1:])[there]
    # Every touched page's keys, up to the newest token, summed.
    first = (length - t).clamp(min=0) // page
    touched = first[:, None] + torch.arange((t - 1) // page + 2, device=DEV)
    held = (length[:, None] - touched * page).clamp(min=0, max=page)
    ids = s["table"].long().gather(1, touched.clamp(max=s["table"].shape[1] - 1))[held > 0]
    held = held[held > 0]
    rows = s["keys"].view(s["num_pages"], page, *s["keys"].shape[1:])[ids].float()
    inside = torch.arange(page, device=DEV) < held[:, None]
    s["sums"][ids] = torch.where(inside[..., None, None], rows, 0.0).sum(1)
    return s["keys"], s["values"], s["sums"]


def _plain_rotary(s):
    case = s["case"]
    half, dim = sum(_sections(case)), case["dim"]
    axis = torch.tensor([a for a, n in enumerate(_sections(case)) for _ in range(n)], device=DEV)
    # Angles of far positions in 64 bits.
    angle = s["positions"].double()[:, axis] * s["frequencies"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def one(x, weight):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        turned, rest = x[..., :2 * half], x[..., 2 * half:]
        if case["interleaved"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = turned[..., :half], turned[..., half:]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, rest], -1)

    out = (one(s["query"], s["q_weight"]).to(s["query"].dtype),
           one(s["key"], s["k_weight"]).to(s["key"].dtype))
    return _with_gradients(s, out)


_plain = {"attend": _plain_attend, "sparse": _plain_sparse, "append": _plain_append,
          "rotary": _plain_rotary}
_own = {"attend": _own_attend, "sparse": _own_sparse, "append": _own_append,
        "rotary": _own_rotary}


# ---------------------------------------------------------------------------
# The definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    return {"attend": _exact_attend, "sparse": _exact_sparse, "append": _exact_append,
            "rotary": _exact_rotary}[case["op"]](case, s)


def _exact_rows(s, pages, length, head, q):
    """Softmax-weighted values of the first `length` keys on `pages` for the rows q [n, D]."""
    if length <= 0:
        return torch.zeros_like(q, dtype=torch.float64)
    slot = torch.cat([torch.arange(p * s["page"], (p + 1) * s["page"]) for p in pages])[:length]
    slot = slot.to(DEV)
    k, v = s["keys"][slot, head].double(), s["values"][slot, head].double()
    return torch.softmax(q.double() @ k.T * s["scale"], -1) @ v


def _exact_attend(case, s):
    t, page = case["tokens"], s["page"]
    table = s["table"].cpu().tolist()
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    for b, seen in enumerate(_visible(case)):
        whole = seen[-1]
        if whole <= 0:
            continue
        pages = torch.tensor(table[b][:-(-whole // page)])
        slot = (pages[:, None] * page + torch.arange(page)).reshape(-1)[:whole].to(DEV)
        k, v = s["keys"][slot].double(), s["values"][slot].double()
        for j, n in enumerate(seen):
            if n > 0:
                for h in range(case["heads"]):
                    q = s["query"][b * t + j, h].double()
                    out[b * t + j, h] = torch.softmax(q @ k[:n, h].T * s["scale"], -1) @ v[:n, h]
    return out


def _exact_sparse(case, s):
    t, page, count, heads = case["tokens"], s["page"], case["count"], case["heads"]
    ids = s["table"].cpu().tolist()
    rows = case["batch"] * t
    if rows * heads > 2000:
        return None
    table = torch.full((rows, heads, count), -1, dtype=torch.int32)
    length = torch.zeros(rows, dtype=torch.int32)
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    for b, seen in enumerate(_visible(case)):
        for j, n in enumerate(seen):
            if n <= 0:
                continue
            r, used = b * t + j, -(-n // page)
            full = torch.tensor(ids[b][:used - 1], dtype=torch.long, device=DEV)
            summed = s["query"][r].double().sum(1)
            score = torch.einsum("phd,hd->hp", s["sums"][full].double(), summed).cpu().tolist()
            kept = min(used, count)
            length[r] = (kept - 1) * page + n - (used - 1) * page
            for h in range(heads):
                best = sorted(range(used - 1), key=lambda p: (-score[h][p], p))[:kept - 1]
                pages = [ids[b][p] for p in sorted(best) + [used - 1]]
                table[r, h, :kept] = torch.tensor(pages, dtype=torch.int32)
                out[r, h] = _exact_rows(s, pages, int(length[r]), h, s["query"][r, h])
    return table.to(DEV), length.to(DEV), out


def _exact_append(case, s):
    t, page = case["tokens"], s["page"]
    ids = s["table"].cpu().tolist()
    keys, values, sums = s["keys"], s["values"], s["sums"].double()
    for b, n in enumerate(_lengths(case)):
        fresh = min(n, t)
        for first in range((n - fresh) // page * page, n, page):
            base = ids[b][first // page] * page
            low, high = max(first, n - fresh), min(first + page, n)
            new = slice(b * t + t - n + low, b * t + t - n + high)
            keys[base + low - first:base + high - first] = s["new_keys"][new]
            values[base + low - first:base + high - first] = s["new_values"][new]
            sums[ids[b][first // page]] = keys[base:base + high - first].double().sum(0)
    return keys, values, sums


def _exact_rotary(case, s):
    sections, half, dim = _sections(case), sum(_sections(case)), case["dim"]
    parts, at = [], 0
    for a, n in enumerate(sections):
        parts.append(s["positions"][:, a:a + 1].double() * s["frequencies"][at:at + n].double())
        at += n
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV).expand(len(parts[0]), half),
                       torch.cat(parts, 1))[:, None]

    def rotate(x, by):
        """Pairs as complex numbers, times `by`."""
        y = x.clone()
        if case["interleaved"]:
            first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        else:
            first, second = slice(0, half), slice(half, 2 * half)
        z = torch.complex(x[..., first], x[..., second]) * by
        y[..., first], y[..., second] = z.real, z.imag
        return y

    outs, grads, weights = [], [], []
    for x, w, d in (("query", "q_weight", "d_query"), ("key", "k_weight", "d_key")):
        x, w = s[x].detach().double(), s[w].detach().double()
        scale = 1 / torch.sqrt((x ** 2).sum(-1, keepdim=True) / dim + EPS)
        normed = x * scale
        outs.append(rotate(normed * w, turn))
        if case["train"]:
            back = rotate(s[d].double(), turn.conj())
            weights.append((back * normed).sum((0, 1)))
            back = back * w
            grads.append(scale * (back - normed * (back * normed).sum(-1, keepdim=True) / dim))
    return tuple(outs + grads + weights)
