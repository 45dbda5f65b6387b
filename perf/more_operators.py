"""Operators around a cache held in 8 bits and around attention that looks back over a window,
measured as a language model's programs call them.

* writing a cache in 8 bits and reading it back:
  ``store``   ``Graph.append`` into caches held in 8 bits (``tg.BlockScaled``: a scale for each
  block of tokens and head), the sums of the keys of every touched page, and ``Graph.read`` of the
  blocks that were written to;
  ``read``    ``Graph.read`` alone: the sequences' cached tokens back in 16 bits;
* ``attend``  dot-product attention of the newest tokens over the 8-bit cache;
* ``window``  the same over ``Graph.paged(window=, sinks=)``: each token sees the last `window`
  tokens and the first `sinks` of its sequence, in a 16-bit or an 8-bit cache;
* ``block``   dot-product attention over ``Graph.cu_seqlens(window=, sinks=)``: the whole sequences
  of a packed batch at once, forward, and with gradients.

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
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "int8": 1}
# The largest code: M; a block's scale is the smallest power of two s >= 2^-126 with amax <= M s.
# As frexp gives it, amax = f 2^n with f in [1/2, 1): s = 2^(n - shift), twice that where f is
# above M / 2^shift.
LARGEST = {"e4m3": (448.0, 9), "int8": (127.0, 7)}


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
             heads=8, group=4, dim=128, page=16, block=16, cache="e4m3", dtype="bf16",
             lengths_seed=1),
        # A served batch of ragged sequences.
        dict(name="attend_batch", op="attend", batch=64, low=100, high=4000, short=False, tokens=1,
             heads=8, group=4, dim=128, page=16, block=16, cache="e4m3", dtype="bf16",
             lengths_seed=2),
        # A few very long sequences: the length has to be split.
        dict(name="attend_long", op="attend", batch=4, low=100000, high=131072, short=False,
             tokens=1, heads=8, group=4, dim=128, page=64, block=64, cache="int8", dtype="bf16",
             lengths_seed=3),
        # A few new tokens of each sequence at once (drafted tokens being checked), one head a
        # group, pages that end inside every tile, and sequences shorter than the tokens asked for.
        dict(name="attend_few", op="attend", batch=24, low=200, high=3000, short=True, tokens=4,
             heads=16, group=1, dim=64, page=24, block=8, cache="int8", dtype="f16",
             lengths_seed=4),
        # A served batch of a model whose layers look back over 4096 tokens.
        dict(name="window_batch", op="window", batch=64, low=500, high=16000, short=False,
             tokens=1, heads=8, group=4, dim=128, page=64, cache="bf16", dtype="bf16",
             lengths_seed=5, window=4096, sinks=4),
        # A few conversations that have run far past a short window, the cache in 8 bits.
        dict(name="window_far", op="window", batch=8, low=90000, high=131072, short=False,
             tokens=1, heads=8, group=4, dim=128, page=16, block=16, cache="e4m3", dtype="bf16",
             lengths_seed=6, window=1024, sinks=64),
        # One new token of each sequence of a served batch.
        dict(name="store_step", op="store", batch=64, low=1, high=500, short=False, tokens=1,
             heads=8, group=1, dim=128, page=16, block=16, cache="e4m3", dtype="bf16",
             lengths_seed=7),
        # Prompts of 1500 tokens each, some behind an earlier part.
        dict(name="store_prompt", op="store", batch=8, low=1500, high=4000, short=False,
             tokens=1500, heads=16, group=1, dim=64, page=64, block=32, cache="int8", dtype="f16",
             lengths_seed=8),
        # Earlier turns of a batch of conversations back in 16 bits, for a pass over whole
        # sequences.
        dict(name="read_turns", op="read", batch=16, low=300, high=4000, short=False, tokens=4000,
             heads=8, group=1, dim=128, page=16, block=16, cache="e4m3", dtype="bf16",
             lengths_seed=9),
        # A training step over a packed batch, forward and backward, query heads grouped.
        dict(name="block_train", op="block", batch=8, low=500, high=4000, heads=4, group=4, dim=128,
             dtype="bf16", lengths_seed=10, window=1024, sinks=4, train=True),
        # A long prompt.
        dict(name="block_prompt", op="block", batch=1, low=32768, high=32768, heads=8, group=4,
             dim=128, dtype="bf16", lengths_seed=11, window=1024, sinks=16, train=False),
        # A small step of short sequences, one head a group, forward and backward.
        dict(name="block_small", op="block", batch=6, low=1, high=275, heads=12, group=1, dim=64,
             dtype="f16", lengths_seed=12, window=100, sinks=1, train=True),
    ]


def _log(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["attend", "window", "store", "read", "block"])
    dtype = rng.choice(["bf16", "f16"])
    dim = rng.choice([32, 64, 128])
    seed = rng.randrange(1 << 30)
    if op == "block":
        heads, group = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 1, 2, 4, 8])
        batch = _log(rng, 1, 32)
        # At most as many scores and queries as the long prompt has.
        most = max(2, min(32768 // batch, 32768 * 32 // (batch * heads * group)))
        high = _log(rng, 2, most)
        window = _log(rng, 2, max(2, min(4096, 32768 * 32 * 1024 // (batch * high * heads * group))))
        return dict(op=op, batch=batch, low=max(1, high // rng.choice([1, 2, 10])), high=high,
                    heads=heads, group=group, dim=dim, dtype=dtype, lengths_seed=seed,
                    window=window, sinks=rng.choice([0, 1, 4, 20, 100]),
                    train=high * batch * heads * group <= 32768 * 8 and rng.random() < 0.6)
    heads = rng.choice([1, 2, 4, 8, 16])
    page = rng.choice([8, 16, 24, 32, 48, 64, 100, 128])
    block = rng.choice([b for b in range(4, page + 1) if page % b == 0])
    cache = rng.choice(["e4m3", "int8"])
    batch = _log(rng, 1, 64)
    if op in ("store", "read"):
        tokens = 1 if op == "store" and rng.random() < 0.5 else _log(rng, 2, 4000)
        batch = max(1, min(batch, 16000 // tokens))
        high = tokens + _log(rng, 1, 500)
        return dict(op=op, batch=batch, low=rng.randint(1, high), high=high, short=False,
                    tokens=tokens, heads=heads, group=1, dim=dim, page=page, block=block,
                    cache=cache, dtype=dtype, lengths_seed=seed)
    # At most as many cached values as the longest listed cases hold.
    most = max(2, 400000 * 8 * 128 // (batch * heads * dim))
    high = _log(rng, 1, min(131072, most))
    case = dict(op=op, batch=batch, low=max(1, high // rng.choice([1, 2, 10])), high=high,
                short=rng.random() < 0.3, tokens=rng.choice([1, 1, 2, 3, 5]), heads=heads,
                group=rng.choice([1, 2, 4, 5, 8, 16]), dim=dim, page=page, dtype=dtype,
                cache=cache, block=block, lengths_seed=seed)
    if op == "window":
        case["window"], case["sinks"] = _log(rng, 1, 16384), rng.choice([0, 1, 4, 20, 100])
        if rng.random() < 0.5:
            case["cache"] = dtype
            del case["block"]
    return case


def _lengths(case):
    """Tokens of each sequence: the longest first; with `short` the last three hold 0, 1 and 2
    tokens."""
    rng = random.Random(case["lengths_seed"])
    lengths = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    lengths[0] = case["high"]
    if case.get("short"):
        for k in range(min(3, case["batch"] - 1)):
            lengths[-1 - k] = k
    return lengths


def _seen(case, n):
    """Tokens that the newest of n tokens sees."""
    if n <= 0:
        return 0
    window, sinks = case.get("window", n), case.get("sinks", 0)
    return n if n <= window + sinks else window + sinks


def _limits_of(case, n):
    """For each of the asking tokens of a sequence of n cached ones, how many there are up to it."""
    t = case["tokens"]
    return [max(0, n - t + 1 + j) for j in range(t)]


# ---------------------------------------------------------------------------
# Work

def work(case):
    size = BYTES[case["dtype"]]
    heads, dim, group, lengths = case["heads"], case["dim"], case["group"], _lengths(case)
    if case["op"] == "block":
        n = sum(lengths)
        # Pairs: the first window + sinks tokens see all before them, the others window + sinks.
        full = case["window"] + case["sinks"]
        pairs = sum(min(l, full) * (min(l, full) + 1) // 2 + max(0, l - full) * full
                    for l in lengths)
        ends = n * heads * dim * size * (2 * group + 2)   # q, out; k, v
        # Training: dout and dq, dk, dv as well; dP, dV, dQ and dK beside the scores and their sum.
        return {"bytes": ends * (2 if case["train"] else 1),
                "flops": 4 * dim * pairs * heads * group * (3 if case["train"] else 1)}
    cell = BYTES[case["cache"]]
    scales = lambda tokens: -(-tokens // case["block"]) * heads * 4 if "block" in case else 0
    if case["op"] == "read":
        rows = sum(min(n, case["tokens"]) for n in lengths)
        return {"bytes": 2 * (rows * heads * dim + scales(rows)) +
                2 * case["batch"] * case["tokens"] * heads * dim * size,
                "flops": 2 * rows * heads * dim}
    if case["op"] == "store":
        t, page, block = case["tokens"], case["page"], case["block"]
        rows = sum(min(n, t) for n in lengths)
        older = sum((n - min(n, t)) % page for n in lengths)
        again = sum((n - min(n, t)) % block for n in lengths)
        blocks = sum(-(-n // block) - (n - min(n, t)) // block for n in lengths)
        pages = sum(-(-n // page) - (n - min(n, t)) // page for n in lengths)
        back = case["batch"] * (t + block)
        return {"bytes": heads * dim * (2 * rows * (size + 1) + older + again + 4 * pages +
                                        2 * (rows + again) + 2 * back * size) +
                16 * heads * blocks,
                "flops": heads * dim * (6 * rows + 2 * older + 2 * back)}
    t = case["tokens"]
    rows = case["batch"] * t
    ends = 2 * rows * heads * group * dim * size
    keys, table, flops = 0, 0, 0
    for n in lengths:
        # (The asking tokens of one sequence share most of what they see.)
        got = min(n, case["window"] + t - 1 + case["sinks"]) if "window" in case else n
        keys += got
        table += 4 * -(-got // case["page"])
        flops += 4 * group * dim * heads * sum(_seen(case, m) for m in _limits_of(case, n))
    return {"bytes": 2 * (keys * heads * dim * cell + scales(keys)) + ends + table +
            4 * len(lengths), "flops": flops}


# ---------------------------------------------------------------------------
# Inputs

def _power(exponent):
    """2^exponent of whole numbers in [-126, 127], by its bits."""
    return ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale_of(amax, cache):
    """The power of two that a block of largest magnitude `amax` is stored by."""
    largest, shift = LARGEST[cache]
    part, exponent = torch.frexp(amax)
    exponent = torch.where(amax == 0, -126, exponent - shift + (part > largest / 2 ** shift))
    return _power(exponent.clamp(min=-126))


def _round_to(x, cache):
    """Values as 8-bit codes, to the nearest, ties to even."""
    return (torch.round(x) if cache == "int8" else x).to(CODES[cache])


def _stored(x, case):
    """Rows [slots, heads, dim] as (codes, scales [blocks, heads])."""
    cache = case["cache"]
    x = x.float().view(-1, case["block"], *x.shape[1:])
    scale = _scale_of(x.abs().amax((1, 3)), cache)
    return _round_to(x / scale[:, None, :, None], cache).flatten(0, 1), scale


def _inputs(case, seed):
    return (_block_inputs if case["op"] == "block" else _cache_inputs)(case, seed)


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
    # Channels of unlike size, as keys and values have them.
    channel = lambda: torch.exp(0.5 * torch.randn(heads, dim, device=DEV, generator=g))
    kc, vc = channel(), channel()
    make = lambda n, c: (torch.randn(n, heads, dim, device=DEV, generator=g) * c).to(dtype)
    rows = len(lengths) * t
    if "block" in case:
        for name, c in (("key", kc), ("value", vc)):
            codes, scales = [], []
            for first in range(0, num_pages, 1 << 20 >> (page - 1).bit_length()):
                count = min(num_pages - first, 1 << 20 >> (page - 1).bit_length())
                got = _stored(make(count * page, c), case)
                codes.append(got[0].view(torch.uint8))
                scales.append(got[1])
            s[name + "s"] = torch.cat(codes).view(CODES[case["cache"]])
            s[name + "_scales"] = torch.cat(scales)
    else:
        s["keys"], s["values"] = make(num_pages * page, kc), make(num_pages * page, vc)
    if case["op"] == "store":
        s["new_keys"], s["new_values"] = make(rows, kc), make(rows, vc)
        s["sums"] = torch.randn(num_pages, heads, dim, device=DEV, generator=g)
    if case["op"] in ("attend", "window"):
        s["query"] = torch.randn(rows, heads, case["group"], dim, device=DEV,
                                 generator=g).to(dtype)
        s["scale"] = dim ** -0.5
    return s


def _block_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    lengths = _lengths(case)
    n, heads, group, dim = sum(lengths), case["heads"], case["group"], case["dim"]
    starts = [0]
    for length in lengths:
        starts.append(starts[-1] + length)
    s = dict(case=case, scale=dim ** -0.5,
             cu_seqlens=torch.tensor(starts, dtype=torch.int32, device=DEV))
    make = lambda *shape: torch.randn(shape, device=DEV, generator=g).to(dtype)
    s["query"] = make(n, heads, group, dim)
    s["key"], s["value"] = make(n, heads, 1, dim), make(n, heads, 1, dim)
    if case["train"]:
        s["d_out"] = make(n, heads, group, dim)
        for name in ("query", "key", "value"):
            s[name].requires_grad_(True)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        tg = _tiga()

        class Attention(tg.MessagePassing):
            reducer = tg.online_softmax()

            def edge(self, src, dst, edge, scale):
                return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)

        if case["op"] == "block":
            s["graph"] = tg.Graph.cu_seqlens(s["cu_seqlens"], window=case["window"],
                                             sinks=case["sinks"])
            s["kernel"] = Attention()
            return s
        if "block" in case:
            s["cache"] = [tg.BlockScaled(s[name + "s"], s[name + "_scales"], block=case["block"])
                          for name in ("key", "value")]
        paged = lambda queries, **more: tg.Graph.paged(
            s["table"], s["lengths"], page_size=s["page"], num_pages=s["num_pages"],
            queries=queries, **more)
        if case["op"] == "store":
            s["graph"], s["back"] = paged(case["tokens"]), paged(case["tokens"] + case["block"])
        elif case["op"] == "read":
            s["graph"] = paged(case["tokens"])
        else:
            more = {k: case[k] for k in ("window", "sinks") if k in case}
            fields = [c.grouped() for c in s["cache"]] if "block" in case else \
                [s["keys"][:, :, None], s["values"][:, :, None]]
            s["attend"] = Attention().prepare(
                graph=paged(case["tokens"], **more), src=dict(zip(("key", "value"), fields)),
                dst={"query": s["query"]}, scale=s["scale"])
    return s


# ---------------------------------------------------------------------------
# One pass

def run(state):
    op = state["case"]["op"]
    return (_own if own else _plain)[op](state)


def _own_attend(s):
    return s["attend"]()


def _own_store(s):
    keys, values = s["cache"]
    s["graph"].append(keys, s["new_keys"], values, s["new_values"], page_sums=s["sums"])
    back = s["back"].read(keys, values, dtype=s["new_keys"].dtype)
    return (*back, s["key_scales"], s["value_scales"], s["sums"])


def _own_read(s):
    return s["graph"].read(*s["cache"], dtype=DTYPES[s["case"]["dtype"]])


def _own_block(s):
    out = s["kernel"](graph=s["graph"], src={"key": s["key"], "value": s["value"]},
                      dst={"query": s["query"]}, scale=s["scale"])
    return _with_gradients(s, out)


def _with_gradients(s, out):
    if not s["case"]["train"]:
        return out
    leaves = (s["query"], s["key"], s["value"])
    return (out.detach(), *torch.autograd.grad(out, leaves, s["d_out"]))


# The plain forms.

def _rows_of(s, name, slots, ok):
    """Cached rows [..., heads, D] at `slots` in 32 bits, zeros where they are not `ok`."""
    rows = s[name + "s"][slots] if "block" not in s["case"] else \
        s[name + "s"].view(torch.uint8)[slots].view(CODES[s["case"]["cache"]])
    rows = rows.float()
    if "block" in s["case"]:
        rows = rows * s[name + "_scales"][slots // s["case"]["block"]][..., None]
    return torch.where(ok[..., None, None], rows, 0.0)


def _slots(s, at):
    """(slot, whether it exists) of the positions `at` [sequences, n]."""
    ids = s["table"].long().gather(1, (at.clamp(min=0) // s["page"]).clamp(
        max=s["table"].shape[1] - 1))
    ok = (at >= 0) & (at < s["lengths"].long()[:, None]) & (ids >= 0) & (ids < s["num_pages"])
    return torch.where(ok, ids * s["page"] + at.clamp(min=0) % s["page"], 0), ok


def _softmax_sum(q, k, v, seen, scale):
    """q [..., rows, D], k and v [..., keys, D], seen [..., rows, keys]."""
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True).detach()
    weight = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight / torch.where(total == 0, 1.0, total), v)


def _plain_attend(s):
    case = s["case"]
    t, group, heads, dim = case["tokens"], case["group"], case["heads"], case["dim"]
    batch = case["batch"]
    if case["op"] == "window":
        # The first tokens, then those behind the newest that any asking token sees.
        first = torch.arange(min(case["sinks"], case["high"]), device=DEV)
        back = torch.arange(min(case["window"] + t - 1, case["high"]), 0, -1, device=DEV)
        near = s["lengths"].long()[:, None] - back
        at = torch.cat([first.expand(batch, -1),
                        torch.where(near >= case["sinks"], near, -1)], 1)     # [B, keys]
    else:
        at = torch.arange(case["high"], device=DEV).expand(batch, -1)
    slots, ok = _slots(s, at)
    keys = slots.shape[1]
    k = _rows_of(s, "key", slots, ok).permute(0, 2, 1, 3)                     # [B, heads, keys, D]
    v = _rows_of(s, "value", slots, ok).permute(0, 2, 1, 3)
    q = s["query"].float().view(batch, t, heads, group, dim).permute(0, 2, 1, 3, 4)
    newest = (s["lengths"].long()[:, None] - t + torch.arange(t, device=DEV))[..., None]
    seen = ok[:, None] & (at[:, None] <= newest)                              # [B, t, keys]
    if case["op"] == "window":
        seen = seen & ((at[:, None] > newest - case["window"]) | (at[:, None] < case["sinks"]))
    seen = seen[:, None, :, None].expand(batch, 1, t, group, keys).reshape(batch, 1, t * group, keys)
    out = _softmax_sum(q.reshape(batch, heads, t * group, dim), k, v, seen, s["scale"])
    out = out.view(batch, heads, t, group, dim).permute(0, 2, 1, 3, 4)
    return out.reshape(batch * t, heads, group, dim).to(s["query"].dtype)


def _newest(s, count):
    """(slot, whether it exists) of the newest `count` positions of each sequence."""
    return _slots(s, s["lengths"].long()[:, None] - count + torch.arange(count, device=DEV))


def _read(s, count):
    slots, ok = _newest(s, count)
    return tuple(_rows_of(s, name, slots, ok).flatten(0, 1).to(DTYPES[s["case"]["dtype"]])
                 for name in ("key", "value"))


def _plain_read(s):
    return _read(s, s["case"]["tokens"])


def _store_one(s, name, new):
    """The new rows of one cache: every touched block's scale, the older tokens of the block by it,
    and the new tokens."""
    case = s["case"]
    t, block, cache = case["tokens"], case["block"], case["cache"]
    length = s["lengths"].long()
    fresh = (length - t).clamp(min=0)                                  # the first new position
    at = ((fresh // block)[:, None] + torch.arange((t - 1) // block + 2, device=DEV)) * block
    at = at[..., None] + torch.arange(block, device=DEV)               # [B, blocks, block]
    slots, ok = (x.view(at.shape) for x in _slots(s, at.flatten(1)))
    row = at - length[:, None, None] + t + torch.arange(len(length), device=DEV)[:, None, None] * t
    is_new = ok & (at >= fresh[:, None, None])
    x = torch.where(is_new[..., None, None], new[torch.where(is_new, row, 0)].float(), 0.0)
    need = _scale_of(x.abs().amax((2, 4)), cache)                      # [B, blocks, heads]
    held = s[name + "_scales"][slots[:, :, 0] // block]
    older = ok[:, :, 0] & ~is_new[:, :, 0]                             # blocks begun before
    scale = torch.where(older[..., None], torch.maximum(need, held), need)
    codes = s[name + "s"].view(torch.uint8)[slots].view(CODES[cache]).float()
    kept = codes * torch.where(older[..., None], held / scale, 1.0)[:, :, None, :, None]
    got = _round_to(torch.where(is_new[..., None, None], x / scale[:, :, None, :, None], kept),
                    cache)
    s[name + "s"].view(torch.uint8)[slots[ok]] = got.view(torch.uint8)[ok]
    touched = is_new.any(-1)
    s[name + "_scales"][(slots[:, :, 0] // block)[touched]] = scale[touched]


def _plain_store(s):
    case = s["case"]
    t, page = case["tokens"], s["page"]
    _store_one(s, "key", s["new_keys"])
    _store_one(s, "value", s["new_values"])
    # Every touched page's keys, up to the newest token, summed.
    first = (s["lengths"].long() - t).clamp(min=0) // page
    at = (first[:, None] + torch.arange((t - 1) // page + 2, device=DEV)) * page
    at = at[..., None] + torch.arange(page, device=DEV)                # [B, pages, page]
    slots, ok = (x.view(at.shape) for x in _slots(s, at.flatten(1)))
    total = _rows_of(s, "key", slots, ok).sum(2)
    touched = ok[:, :, 0]
    s["sums"][(slots[:, :, 0] // page)[touched]] = total[touched]
    return (*_read(s, t + case["block"]), s["key_scales"], s["value_scales"], s["sums"])


def _plain_block(s):
    """The packed sequences as [sequences, longest], queries in chunks that see a band of keys and
    the first few."""
    case = s["case"]
    heads, group, dim = case["heads"], case["group"], case["dim"]
    window, sinks = min(case["window"], case["high"]), min(case["sinks"], case["high"])
    chunk = min(max(64, 1 << (window - 1).bit_length()), case["high"])
    count = -(-case["high"] // chunk)
    start = s["cu_seqlens"].long()[:-1]
    length = s["cu_seqlens"].long()[1:] - start
    batch, n = case["batch"], s["query"].shape[0]
    i = torch.arange(count * chunk, device=DEV).view(count, chunk)
    j = torch.arange(count, device=DEV)[:, None] * chunk + torch.arange(1 - window, chunk,
                                                                        device=DEV)
    j = torch.cat([torch.arange(sinks, device=DEV).expand(count, -1), j], 1)   # [count, keys]
    seen = (j[:, None] <= i[..., None]) & (j[:, None] >= 0)
    far = torch.arange(j.shape[1], device=DEV) < sinks                # the first tokens
    band = (j[:, None] > i[..., None] - window)
    seen = seen & torch.where(far, ~band, band)                               # [count, chunk, keys]
    seen = seen & (j[:, None] < length[:, None, None, None])                  # [B, ...]
    token = lambda p: (start.view(-1, *[1] * p.ndim) + p).clamp(min=0, max=n - 1)
    q = s["query"].float()[token(i)].permute(0, 1, 3, 2, 4, 5)     # [B, count, heads, chunk, g, D]
    k = s["key"].float()[token(j)][..., 0, :].transpose(2, 3)      # [B, count, heads, keys, D]
    v = s["value"].float()[token(j)][..., 0, :].transpose(2, 3)
    rows = q.reshape(batch, count, heads, chunk * group, dim)
    mask = seen[:, :, None, :, None].expand(-1, -1, 1, chunk, group, -1).flatten(3, 4)
    out = _softmax_sum(rows, k, v, mask, s["scale"])
    out = out.view(batch, count, heads, chunk, group, dim).permute(0, 1, 3, 2, 4, 5).flatten(1, 2)
    there = torch.arange(count * chunk, device=DEV) < length[:, None]
    return _with_gradients(s, out[there].to(s["query"].dtype))


_plain = {"attend": _plain_attend, "window": _plain_attend, "store": _plain_store,
          "read": _plain_read, "block": _plain_block}
_own = {"attend": _own_attend, "window": _own_attend, "store": _own_store, "read": _own_read,
        "block": _own_block}


# ---------------------------------------------------------------------------
# The definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    return {"attend": _exact_attend, "window": _exact_attend, "store": _exact_store,
            "read": _exact_read, "block": _exact_block}[case["op"]](case, s)


def _exact_slots(s, ids, low, high):
    """Slots of the positions low .. high - 1 of a sequence whose pages are `ids`."""
    page = s["page"]
    pages = torch.tensor(ids[low // page:-(-high // page)], dtype=torch.long)
    slot = (pages[:, None] * page + torch.arange(page)).reshape(-1)
    return slot[low - low // page * page:high - low // page * page].to(DEV)


def _exact_rows(case, s, name, slot):
    """Cached rows in 64 bits: a code times its block's scale."""
    rows = s[name + "s"].view(torch.uint8)[slot].view(CODES[case["cache"]]) if "block" in case \
        else s[name + "s"][slot]
    rows = rows.double()
    if "block" in case:
        rows *= s[name + "_scales"].double()[torch.div(slot, case["block"],
                                                       rounding_mode="floor")][:, :, None]
    return rows


def _exact_attend(case, s):
    t = case["tokens"]
    table = s["table"].cpu().tolist()
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lengths(case)):
        for j, m in enumerate(_limits_of(case, n)):
            if m == 0:
                continue
            far = max(0, m - case["window"]) if "window" in case else 0
            parts = [_exact_slots(s, table[b], far, m)]
            if far and case["sinks"]:
                parts.insert(0, _exact_slots(s, table[b], 0, min(far, case["sinks"])))
            slot = torch.cat(parts)
            k, v = _exact_rows(case, s, "key", slot), _exact_rows(case, s, "value", slot)
            for h in range(case["heads"]):
                q = s["query"][b * t + j, h].double()
                out[b * t + j, h] = torch.softmax(q @ k[:, h].T * s["scale"], -1) @ v[:, h]
    return out


def _exact_back(case, s, count):
    """The newest `count` tokens of each sequence."""
    got = []
    table = s["table"].cpu().tolist()
    for name in ("key", "value"):
        rows = torch.zeros(case["batch"] * count, case["heads"], case["dim"], dtype=torch.float64,
                           device=DEV)
        for b, n in enumerate(_lengths(case)):
            low = max(0, n - count)
            if n:
                rows[b * count + count - (n - low):(b + 1) * count] = _exact_rows(
                    case, s, name, _exact_slots(s, table[b], low, n))
        got.append(rows)
    return tuple(got)


def _exact_read(case, s):
    return _exact_back(case, s, case["tokens"])


def _exact_codes(x, cache):
    """Values in 64 bits to the nearest code, as numbers: steps of 1, or of 2^(e - 3) between 2^e
    and 2^(e + 1) and of 2^-9 below 2^-6."""
    if cache == "int8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_store(case, s):
    t, page, block, cache = case["tokens"], case["page"], case["block"], case["cache"]
    if case["batch"] * -(-t // block) > 4000:
        return None
    largest = LARGEST[cache][0]
    table = s["table"].cpu().tolist()
    sums = s["sums"].double()
    scales = {name: s[name + "_scales"].double() for name in ("key", "value")}
    for b, n in enumerate(_lengths(case)):
        fresh = max(0, n - t)
        for name, new in (("key", s["new_keys"]), ("value", s["new_values"])):
            for first in range(fresh // block * block, n, block):
                low, high = max(first, fresh), min(first + block, n)
                slot = _exact_slots(s, table[b], first, high)
                x = new[b * t + t - n + low:b * t + t - n + high].double()   # [new, heads, D]
                amax = x.abs().amax((0, 2))
                power = torch.ceil(torch.log2(amax / largest)).clamp(min=-126)
                power += (torch.exp2(power) * largest < amax).double()
                power -= (torch.exp2(power - 1) * largest >= amax).double()
                scale = torch.exp2(power.clamp(min=-126))
                at = int(slot[0]) // block
                if low > first:
                    scale = torch.maximum(scale, scales[name][at])
                    old = slot[:low - first]
                    codes = s[name + "s"].view(torch.uint8)[old].view(CODES[cache]).double()
                    codes = _exact_codes(codes * (scales[name][at] / scale)[:, None], cache)
                    s[name + "s"].view(torch.uint8)[old] = codes.to(CODES[cache]).view(torch.uint8)
                scales[name][at] = scale
                codes = _exact_codes(x / scale[:, None], cache).to(CODES[cache])
                s[name + "s"].view(torch.uint8)[slot[low - first:]] = codes.view(torch.uint8)
    for name in ("key", "value"):
        s[name + "_scales"] = scales[name]
    for b, n in enumerate(_lengths(case)):
        for first in range(max(0, n - t) // page * page, n, page):
            slot = _exact_slots(s, table[b], first, min(first + page, n))
            sums[table[b][first // page]] = _exact_rows(case, s, "key", slot).sum(0)
    return (*_exact_back(case, s, t + block), scales["key"], scales["value"], sums)


def _exact_block(case, s):
    window, sinks, scale = case["window"], case["sinks"], s["scale"]
    q, k, v = (s[name].detach() for name in ("query", "key", "value"))
    names = ("out", "dq", "dk", "dv") if case["train"] else ("out",)
    got = {name: torch.zeros((k if name in ("dk", "dv") else q).shape, dtype=torch.float64,
                             device=DEV) for name in names}
    lengths = _lengths(case)
    step = 1024
    if sum(-(-n // step) for n in lengths) * case["heads"] * case["group"] > 20000:
        return None
    start = 0
    for n in lengths:
        for first in range(0, n, step):
            last = min(first + step, n)
            low = max(0, first - window + 1)
            near = torch.arange(low, last, device=DEV)
            cols = torch.cat([torch.arange(min(low, sinks), device=DEV), near])
            i = torch.arange(first, last, device=DEV)[:, None]
            seen = (cols <= i) & ((i - cols < window) | (cols < sinks))
            rows, at = slice(start + first, start + last), start + cols
            for h in range(case["heads"]):
                kk, vv = k[at, h, 0].double(), v[at, h, 0].double()
                for g in range(case["group"]):
                    qq = q[rows, h, g].double()
                    p = torch.softmax((qq @ kk.T * scale).masked_fill(~seen, -torch.inf), -1)
                    out = p @ vv
                    got["out"][rows, h, g] = out
                    if case["train"]:
                        d = s["d_out"][rows, h, g].double()
                        ds = p * (d @ vv.T - (d * out).sum(-1, keepdim=True))
                        got["dq"][rows, h, g] = ds @ kk * scale
                        got["dk"][:, h, 0].index_add_(0, at, ds.T @ qq * scale)
                        got["dv"][:, h, 0].index_add_(0, at, p.T @ d)
        start += n
    return tuple(got.values()) if case["train"] else got["out"]
