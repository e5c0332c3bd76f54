"""Performance cases of the text model's attention whose cost does not grow with what a sequence shares or has left behind:
a sliding window with first tokens that stay visible, a prefix that several sequences share, and linear attention with
a state in the cache's place.

Kinds:

- spans       attention of each sequence's newest tokens over the 8-bit key/value cache (`ops.kv_attention`), of which a row sees
              the first `sinks` tokens and the last `window` (`sinks=`, `window=`); or all of it, the first tokens of which are the
              same blocks for all sequences of a group (`shared=`: computed once for the group); or both
- linear      linear attention with a decay for each head (`ops.lin_attention`): state = exp(-decay) state + k v^T, out = q state,
              token by token; the states of the sequences lie in a pool and are carried on

The cache holds blocks of 64 tokens: codes k [blocks, kv heads, 64, width] and v [blocks, kv heads, width, 64] (width: the
head size up to the next multiple of 64) and one float32 scale for each block and head. A sequence is a row of the
block table; blocks that no row can see any more are not kept (-1). States are float32 [slots, heads, dk, dv]. Sizes: the text
encoder's heads (64 over 8 of 128); others beside them are generic.

With `own` false, `run` computes the same in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one answered token behind a short window and a few first tokens: latency
        {"name": "sinks_one_700", "kind": "spans", "seqs": 1, "new": 1, "prefix": 0, "own": 700, "groups": 0, "window": 256, "sinks": 4,
         "kv": 8, "group": 8, "dim": 128, "dtype": "bf16"},
        # a step of 64 long conversations whose middles are no longer kept: the serving load of a window
        {"name": "sinks_step_64", "kind": "spans", "seqs": 64, "new": 1, "prefix": 0, "own": 32768, "groups": 0, "window": 4096, "sinks": 4,
         "kv": 8, "group": 8, "dim": 128, "dtype": "bf16"},
        # the second half of a long prompt, each row behind its own window: bound by products
        {"name": "sinks_prompt_4096", "kind": "spans", "seqs": 1, "new": 4096, "prefix": 0, "own": 8192, "groups": 0, "window": 1024,
         "sinks": 64, "kv": 8, "group": 8, "dim": 128, "dtype": "bf16"},
        # three ragged float32 prompts with first tokens that end inside a block, heads of 80, and the rows' log sums
        {"name": "sinks_prompts_f32", "kind": "spans", "seqs": 3, "new": 401, "prefix": 0, "own": 901, "groups": 0, "window": 300, "sinks": 70,
         "kv": 8, "group": 4, "dim": 80, "dtype": "f32", "lse": True},
        # four answers sampled from one short prompt: the smallest group
        {"name": "shared_4x512", "kind": "spans", "seqs": 4, "new": 1, "prefix": 512, "own": 100, "groups": 1, "window": 0, "sinks": 0,
         "kv": 8, "group": 8, "dim": 128, "dtype": "bf16"},
        # 64 conversations behind the same instructions: the serving load of a shared prefix
        {"name": "shared_64x8192", "kind": "spans", "seqs": 64, "new": 1, "prefix": 8192, "own": 1024, "groups": 1, "window": 0, "sinks": 0,
         "kv": 8, "group": 8, "dim": 128, "dtype": "bf16"},
        # six groups of eight, prefixes of their own, heads of 64 in groups of seven, with the rows' log sums
        {"name": "shared_groups_f16", "kind": "spans", "seqs": 48, "new": 1, "prefix": 4096, "own": 300, "groups": 6, "window": 0, "sinks": 0,
         "kv": 4, "group": 7, "dim": 64, "dtype": "f16", "lse": True},
        # eight questions of up to 256 tokens about one document
        {"name": "shared_prompts", "kind": "spans", "seqs": 8, "new": 256, "prefix": 4096, "own": 300, "groups": 1, "window": 0, "sinks": 0,
         "kv": 8, "group": 8, "dim": 128, "dtype": "bf16"},
        # one answered token of linear attention: the state read and written
        {"name": "linear_one", "kind": "linear", "seqs": 1, "new": 1, "heads": 64, "kv": 64, "dk": 128, "dv": 128, "begin": 0.0, "dtype": "bf16"},
        # a step of 64 sequences
        {"name": "linear_step_64", "kind": "linear", "seqs": 64, "new": 1, "heads": 64, "kv": 64, "dk": 128, "dv": 128, "begin": 0.0,
         "dtype": "bf16"},
        # a prompt from its beginning
        {"name": "linear_prompt_8192", "kind": "linear", "seqs": 1, "new": 8192, "heads": 64, "kv": 64, "dk": 128, "dv": 128, "begin": 1.0,
         "dtype": "bf16"},
        # four ragged float32 prompts, some of them carried on, keys and values shared by four heads, heads of 80 by 96
        {"name": "linear_prompts_f32", "kind": "linear", "seqs": 4, "new": 1500, "heads": 16, "kv": 4, "dk": 80, "dv": 96, "begin": 0.5,
         "dtype": "f32"},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if rng.random() < 0.4:
        heads = rng.choice([4, 8, 16, 32, 64])
        dk, dv = rng.choice([32, 64, 80, 128, 128, 192, 256]), rng.choice([32, 64, 96, 128, 128, 192, 256])
        case = {"kind": "linear", "heads": heads, "kv": heads // rng.choice([1, 1, 1, 4]), "dk": dk, "dv": dv,
                "begin": rng.choice([0.0, 0.5, 1.0]), "dtype": dtype}
        states = heads * dk * dv
        case["seqs"] = _between(rng, 1, max(1, min(64, (1 << 26) // states)))
        # at most the longest listed prompt's work and bytes
        most = min(32768, (1 << 33) // (states * case["seqs"]), (1 << 27) // (heads * (dk + dv) * case["seqs"] * (2 if dtype == "f32" else 1)))
        case["new"] = rng.choice([1, 1, 2, 5]) if rng.random() < 0.4 else _between(rng, 2, max(2, most))
        return case
    case = {"kind": "spans", "kv": rng.choice([1, 2, 4, 8, 16]), "dim": rng.choice([64, 80, 96, 128, 128, 256]), "group": rng.choice([1, 2, 4, 7, 8, 16]),
            "dtype": dtype, "seqs": _between(rng, 1, 64)}
    answers = rng.random() < 0.6
    if answers:
        case["dim"] = min(case["dim"], 128)
    heads = case["kv"] * case["group"] * case["dim"]
    case["new"] = rng.choice([1, 1, 1, 2, 5]) if answers else _between(rng, 2, max(2, min(2048 // case["seqs"], math.isqrt((1 << 35) // (heads * case["seqs"])))))
    # at most the longest listed cases' bytes and products
    most = max(64, min(32768, (1 << 28) // (case["kv"] * case["dim"] * max(case["seqs"], 4)), (1 << 35) // (heads * case["seqs"] * case["new"])))
    shared = rng.random() < 0.5
    case["groups"] = rng.randint(1, max(1, case["seqs"] // 3)) if shared else 0
    case["prefix"] = _between(rng, 64, max(64, min(most, 8192))) // BLOCK * BLOCK if shared else 0
    case["own"] = max(case["new"], _between(rng, 1, 1024 if shared else most))
    if not shared or rng.random() < 0.3:
        case["window"], case["sinks"] = _between(rng, 16, 4096), rng.choice([1, 4, 4, 16, 64, 70, 200])
    else:
        case["window"], case["sinks"] = 0, 0
    case["lse"] = rng.random() < 0.3
    case["mask"] = rng.random() < 0.2
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _spread(most, count, lowest, turn):
    """`count` whole numbers between lowest * most and most, the first of them `most`, in no order."""
    return [max(1, round(most * (1 - (1 - lowest) * ((i * turn) % count) / max(1, count - 1)))) if most else 0 for i in range(count)]


def _plan(case):
    """Of a spans case: each sequence's new tokens, its tokens in the cache after them, and the blocks that it shares; the first
    sequence of each group."""
    n = case["seqs"]
    new = _spread(case["new"], n, 0.4, 23)
    first = [g * n // case["groups"] for g in range(case["groups"] + 1)] if case["groups"] else []
    blocks = [p // BLOCK for p in _spread(case["prefix"], len(first) - 1, 0.5, 3)] if first else []
    shares = [0] * n
    for g, k in enumerate(blocks):
        shares[first[g]:first[g + 1]] = [k] * (first[g + 1] - first[g])
    lengths = [s * BLOCK + max(a, o) for s, a, o in zip(shares, new, _spread(case["own"], n, 0.3, 37))]
    return new, lengths, shares, first


def _lowest(case, new, length):
    """The first block that a row's window reaches into."""
    return max(0, length - new - case["window"] + 1) // BLOCK if case["window"] else 0


def _blocks(n):
    return -(-n // BLOCK)


class _Make:
    """The inputs of one case, from its seed alone."""

    def __init__(self, seed):
        self.seed = int(seed)
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(self.seed)

    def normal(self, *shape, sd=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=self.g, device="cuda") * sd).to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(mk, new):
    return mk.ints([sum(new[:i]) for i in range(len(new) + 1)])


def _table(case, plan, seed):
    """The block table, a group's shared blocks the same in all its rows, and the blocks of the pool. What no row sees is not kept."""
    new, lengths, shares, first = plan
    sinks, wide = _blocks(case["sinks"]), max(_blocks(x) for x in lengths)
    kept = np.zeros((case["seqs"], wide), bool)
    for b, (n, length) in enumerate(zip(new, lengths)):
        low = _lowest(case, n, length)
        kept[b, : min(sinks, _blocks(length))] = True
        kept[b, low:_blocks(length)] = True
    table = np.full((case["seqs"], wide), -1, np.int64)
    table[kept] = np.arange(kept.sum())
    for a, e in zip(first[:-1], first[1:]):
        k = shares[a]
        held = kept[a:e, :k].any(0)
        table[a:e, :k] = np.where(held, table[a:e, :k].max(0), -1)
    # the blocks lie anywhere in a pool that holds a few more
    names, table = np.unique(np.concatenate([[-1], table.ravel()]), return_inverse=True)
    order = np.concatenate([[-1], np.random.default_rng(seed).permutation(len(names) + 2)])
    return order[table[1:]].reshape(case["seqs"], wide).astype(np.int32), len(names) + 2


def _inputs(case, seed):
    """The case's tensors by name: what a user's program has in hand."""
    mk, dt = _Make(seed), TYPES[case["dtype"]]
    if case["kind"] == "linear":
        heads, kv, dk, dv, seqs = case["heads"], case["kv"], case["dk"], case["dv"], case["seqs"]
        new = _spread(case["new"], seqs, 0.4, 23)
        slots = torch.randperm(seqs + 2, generator=mk.g, device="cuda")[:seqs].to(torch.int32)
        old = torch.arange(seqs, device="cuda") >= round(case["begin"] * seqs)
        # one projection's rows: queries, keys and values side by side
        t = {"rows": mk.normal(sum(new), heads * dk + kv * (dk + dv), dtype=dt), "starts": _starts(mk, new),
             "source": torch.where(old, slots, torch.full_like(slots, -1)), "target": slots,
             "state": mk.normal(seqs + 2, heads, dk, dv, sd=4.0),
             # heads that forget within a few tokens to heads that hold hundreds
             "decay": 2.0 ** (-8 * torch.arange(1, heads + 1, device="cuda") / heads)}
        t["out"] = torch.zeros(sum(new), heads * dv, dtype=dt, device="cuda")
        return t
    plan = _plan(case)
    new, lengths, shares, first = plan
    kv, dim, seqs = case["kv"], case["dim"], case["seqs"]
    width, rows = -(-dim // 64) * 64, sum(new)
    table, pages = _table(case, plan, seed)
    t = {"table": mk.ints(table), "starts": _starts(mk, new), "lengths": mk.ints(lengths)}
    if first:
        t["first"], t["shared"] = mk.ints(first), mk.ints([shares[a] * BLOCK for a in first[:-1]])
    # keys with a few features larger than the rest, as rotated and normalized keys have them
    gain = torch.ones(width, device="cuda")
    gain[::16] = 3
    gain[dim:] = 0
    t["k"] = torch.empty(pages, kv, BLOCK, width, dtype=torch.int8, device="cuda")
    t["v"] = torch.empty(pages, kv, width, BLOCK, dtype=torch.int8, device="cuda")
    t["k_scale"], t["v_scale"] = (torch.empty(pages, kv, device="cuda") for _ in range(2))
    for p in range(0, pages, 256):
        x = mk.normal(min(256, pages - p), kv, BLOCK, width) * gain
        s = x.abs().amax((2, 3)) / 127
        t["k"][p:p + 256], t["k_scale"][p:p + 256] = (x / s[:, :, None, None]).round().to(torch.int8), s
        x = mk.normal(min(256, pages - p), kv, width, BLOCK)
        x[:, :, dim:] = 0
        s = x.abs().amax((2, 3)) / 127
        t["v"][p:p + 256], t["v_scale"][p:p + 256] = (x / s[:, :, None, None]).round().to(torch.int8), s
    t["q"] = mk.normal(rows, kv * case["group"] * dim, dtype=dt)
    t["out"] = torch.zeros(rows, kv * case["group"] * dim, dtype=dt, device="cuda")
    if case.get("lse"):
        t["lse"] = torch.zeros(rows, kv * case["group"], device="cuda")
    if case.get("mask"):
        t["mask"] = (mk.uniform(seqs, table.shape[1] * BLOCK) < 0.8).to(torch.uint8)
    return t


def prepare(case, seed):
    s = {"case": dict(case), "t": _inputs(case, seed)}
    if case["kind"] == "linear":
        return {**s, "new": _spread(case["new"], case["seqs"], 0.4, 23)}
    new, lengths, shares, _ = _plan(case)
    return {**s, "new": new, "lengths": lengths, "low": min(_lowest(case, n, x) for n, x in zip(new, lengths))}


# ---- the framework's calls ----------------------------------------------------------------------------------------------

_devices = {}


def _handles(s):
    """The framework's tensors over the state's, made once as a user's program makes them."""
    from sycl_minimax_h3_amd import Device, Tensor, ops

    stream = torch.cuda.current_stream().cuda_stream
    if stream not in _devices:
        _devices[stream] = Device.from_torch()
    dev, case = _devices[stream], s["case"]
    h = {k: Tensor.from_torch(v, dev=dev) for k, v in s["t"].items()}
    h["ops"], rows = ops, sum(s["new"])
    if case["kind"] == "linear":
        heads, kv, dk, dv = case["heads"], case["kv"], case["dk"], case["dv"]
        wide = heads * dk + kv * (dk + dv)
        h["q"] = ops.Rows(h["rows"], 0, wide, rows, heads, dk)
        h["k"] = ops.Rows(h["rows"], heads * dk, wide, rows, kv, dk)
        h["v"] = ops.Rows(h["rows"], (heads + kv) * dk, wide, rows, kv, dv)
        h["states"] = ops.LinState(h["state"])
    else:
        heads, dim = case["kv"] * case["group"], case["dim"]
        h["cache"] = ops.KvCache(h["k"], h["v"], h["k_scale"], h["v_scale"], dim)
        h["queries"] = ops.Rows(h["q"], 0, heads * dim, rows, heads, dim)
        h["groups"] = ops.KvShared(h["first"], h["shared"], case["prefix"]) if case["groups"] else None
    s["handles"] = h
    return h


def _run_own(s):
    h, t, case = s.get("handles") or _handles(s), s["t"], s["case"]
    if case["kind"] == "linear":
        h["ops"].lin_attention(h["states"], h["decay"], h["q"], h["k"], h["v"], h["starts"], h["source"], h["target"], max(s["new"]), h["out"])
        return t["out"], t["state"]
    h["ops"].kv_attention(h["cache"], h["table"], h["queries"], h["starts"], h["lengths"], max(s["new"]), h["out"], max_len=max(s["lengths"]),
                          window=case["window"], sinks=case["sinks"], shared=h["groups"], mask=h.get("mask"), lse=h.get("lse"))
    return (t["out"], t["lse"]) if "lse" in t else t["out"]


# ---- the plain form -----------------------------------------------------------------------------------------------------

def _row_index(starts, new):
    """For each sequence and each of its up to max(new) rows: the row, and whether it has one."""
    j = torch.arange(max(new), device=starts.device)[None, :]
    return (starts[:-1, None] + j).clamp_max(sum(new) - 1).long(), j < (starts[1:] - starts[:-1])[:, None]


def _plain_spans(s):
    t, case, new = s["t"], s["case"], s["new"]
    kv, dim, group, seqs, most = case["kv"], case["dim"], case["group"], case["seqs"], max(new)
    width, wide = t["k"].shape[3], _blocks(max(s["lengths"]))
    where = (t["lengths"] - t["starts"][1:] + t["starts"][:-1]).long()[:, None] + torch.arange(most, device="cuda")    # [seqs, new]
    # the blocks that a sequence's rows can see: the first tokens' and those that the windows reach into
    sinks = _blocks(case["sinks"]) if s["low"] else 0
    low = torch.div((where[:, 0] - case["window"] + 1).clamp_min(0), BLOCK, rounding_mode="floor") if s["low"] else torch.zeros_like(where[:, 0])
    count = min(wide, (case["window"] + most - 2) // BLOCK + 2) if s["low"] else wide
    at = torch.arange(sinks + count, device="cuda")[None, :].repeat(seqs, 1)
    at[:, sinks:] += (low - sinks)[:, None]
    once = (at < wide) & ((torch.arange(sinks + count, device="cuda") < sinks) | (at >= sinks))
    pages = torch.gather(t["table"].long(), 1, at.clamp(0, wide - 1))
    there = once & (pages >= 0)
    pages = pages.clamp_min(0)
    n = (sinks + count) * BLOCK
    k = t["k"][pages].float() * t["k_scale"][pages][..., None, None]                                  # [seqs, blocks, kv, 64, width]
    k = k.permute(0, 2, 1, 3, 4).reshape(seqs, kv, n, width)[..., :dim]
    v = t["v"][pages].float() * t["v_scale"][pages][..., None, None]                                  # [seqs, blocks, kv, width, 64]
    v = v.permute(0, 2, 1, 4, 3).reshape(seqs, kv, n, width)[..., :dim]
    row, real = _row_index(t["starts"], new)
    q = t["q"].float().reshape(-1, kv, group, dim)[row]                                               # [seqs, new, kv, group, dim]
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    x = torch.matmul(q, k.transpose(2, 3)).reshape(seqs, kv, group, most, n) * dim ** -0.5
    token = (at[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")).reshape(seqs, 1, n)
    seen = (token <= where[:, :, None]) & there.repeat_interleave(BLOCK, 1)[:, None, :]               # [seqs, new, keys]
    if case["window"]:
        seen &= (token > where[:, :, None] - case["window"]) | (token < case["sinks"])
    if case.get("mask"):
        seen &= torch.gather(t["mask"], 1, token[:, 0].clamp(0, t["mask"].shape[1] - 1))[:, None] != 0
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.reshape(seqs, kv, group * most, -1), v).reshape(seqs, kv, group, most, dim)
    y = torch.where(total > 0, y / total, torch.zeros_like(y))
    t["out"].copy_(y.permute(0, 3, 1, 2, 4)[real].reshape(-1, kv * group * dim))
    if "lse" in t:
        t["lse"].copy_((top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2)[real].reshape(-1, kv * group))
        return t["out"], t["lse"]
    return t["out"]


def _plain_linear(s):
    """In pieces of 128 tokens: within a piece by products of queries and keys, beyond it by the states at the pieces' beginnings, which a
    triangle of decays makes of the pieces' own sums."""
    t, case, new = s["t"], s["case"], s["new"]
    heads, kv, dk, dv, seqs = case["heads"], case["kv"], case["dk"], case["dv"], case["seqs"]
    piece = min(128, max(new))
    pieces = -(-max(new) // piece)
    n = pieces * piece
    j = torch.arange(n, device="cuda")
    count = (t["starts"][1:] - t["starts"][:-1]).long()
    row, real = (t["starts"][:-1, None] + j).clamp_max(sum(new) - 1).long(), j < count[:, None]
    x = t["rows"].float()[row] * real[:, :, None]                                                     # [seqs, n, features]
    parts = x.split([heads * dk, kv * dk, kv * dv], 2)
    q, k, v = (y.reshape(seqs, n, -1, d).transpose(1, 2) for y, d in zip(parts, (dk, dk, dv)))
    k, v = (y.repeat_interleave(heads // kv, 1) for y in (k, v))                                      # [seqs, heads, n, d]
    rate = t["decay"].double()
    fade = lambda steps: torch.exp(-rate.reshape(-1, *[1] * steps.dim()) * steps).float()  # noqa: E731  (angles of far tokens)
    s0 = torch.where((t["source"] >= 0)[:, None, None, None], t["state"][t["source"].clamp_min(0).long()], torch.zeros((), device="cuda"))
    # the state after the last token: token j fades for count - 1 - j steps
    last = torch.exp(-rate[None, :, None] * (count[:, None] - 1 - j).clamp_min(0)[:, None, :]).float() * real[:, None, :]
    end = s0 * torch.exp(-rate[None, :] * count[:, None]).float()[:, :, None, None] + torch.matmul((k * last[..., None]).transpose(2, 3), v)
    q, k, v = (y.reshape(seqs, heads, pieces, piece, y.shape[3]) for y in (q, k, v))
    i = torch.arange(piece, device="cuda")
    ahead = i[:, None] - i[None, :]
    inside = torch.matmul(q, k.transpose(3, 4)) * (fade(ahead.clamp_min(0)) * (ahead >= 0))[:, None]
    y = torch.matmul(inside, v)
    sums = torch.matmul((k * fade(piece - 1 - i)[:, None, :, None]).transpose(3, 4), v)               # [seqs, heads, pieces, dk, dv]
    m = torch.arange(pieces, device="cuda")
    behind = m[:, None] - m[None, :] - 1
    carry = fade(behind.clamp_min(0) * piece) * (behind >= 0)
    begin = torch.matmul(carry, sums.reshape(seqs, heads, pieces, dk * dv)).reshape(sums.shape) + s0[:, :, None] * fade(m * piece)[:, :, None, None]
    y = (y + torch.matmul(q, begin) * fade(i + 1)[:, None, :, None]) * dk ** -0.5
    t["out"].copy_(y.reshape(seqs, heads, n, dv).transpose(1, 2)[real].reshape(-1, heads * dv))
    t["state"][t["target"].long()] = end
    return t["out"], t["state"]


def run(state):
    if own:
        return _run_own(state)
    return _plain_linear(state) if state["case"]["kind"] == "linear" else _plain_spans(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "linear":
        heads, kv, dk, dv, seqs = case["heads"], case["kv"], case["dk"], case["dv"], case["seqs"]
        rows = sum(_spread(case["new"], seqs, 0.4, 23))
        states = 2 * seqs - round(case["begin"] * seqs)
        return {"bytes": size * rows * (heads * (dk + dv) + kv * (dk + dv)) + 4 * states * heads * dk * dv, "flops": 4 * rows * heads * dk * dv}
    new, lengths, shares, first = _plan(case)
    kv, dim, heads = case["kv"], case["dim"], case["kv"] * case["group"]
    window, sinks = case["window"] or 1 << 60, case["sinks"]
    pairs = sum(min(p, window + min(sinks, max(0, p - window))) for n, x in zip(new, lengths) for p in range(x - n + 1, x + 1))
    # the tokens that a sequence's rows see, without those that it shares, and those that any of a group sees
    spans = [(min(sinks, x), max(0, x - n + 1 - window), x) for n, x in zip(new, lengths)]
    read = sum(x - max(c * BLOCK, low) + max(0, min(top, low) - c * BLOCK) for (top, low, x), c in zip(spans, shares))
    for a, e in zip(first[:-1], first[1:]):
        end, low, top = shares[a] * BLOCK, min(s[1] for s in spans[a:e]), max(s[0] for s in spans[a:e])
        read += max(0, end - low) + min(top, low, end)
    return {"bytes": 2 * kv * dim * read + 2 * size * sum(new) * heads * dim, "flops": 4 * heads * dim * pairs}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------

def _exact_spans(t, case):
    """Sequence by sequence over the blocks that its row of the table names, head by head."""
    kv, dim, group = case["kv"], case["dim"], case["group"]
    out = torch.zeros(t["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(len(out), kv * group, dtype=torch.float64, device="cuda")
    lengths, starts = t["lengths"].tolist(), t["starts"].tolist()
    for b in range(case["seqs"]):
        a, e, length = starts[b], starts[b + 1], lengths[b]
        held = (t["table"][b, :_blocks(length)] >= 0).nonzero()[:, 0]
        pages = t["table"][b, held].long()
        at = (held[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).reshape(-1)
        where = torch.arange(length - e + a, length, device="cuda")[:, None]
        hide = at > where
        if case["window"]:
            hide |= (at <= where - case["window"]) & (at >= case["sinks"])
        if case.get("mask"):
            hide |= t["mask"][b, at.clamp_max(t["mask"].shape[1] - 1)] == 0
        for h in range(kv):
            k = (t["k"][pages, h, :, :dim].double() * t["k_scale"][pages, h].double()[:, None, None]).reshape(-1, dim)
            v = (t["v"][pages, h, :dim].double() * t["v_scale"][pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, dim)
            for g in range(h * group, (h + 1) * group):
                s = t["q"][a:e, g * dim:(g + 1) * dim].double() @ k.t().contiguous() / math.sqrt(dim)
                s[hide] = -math.inf
                lse[a:e, g] = torch.logsumexp(s, 1)
                out[a:e, g * dim:(g + 1) * dim] = torch.nan_to_num(torch.softmax(s, 1), nan=0.0) @ v
    return (out, lse) if "lse" in t else out


def _exact_linear(t, case):
    """Token by token, as the operator is defined."""
    heads, kv, dk, dv = case["heads"], case["kv"], case["dk"], case["dv"]
    starts, each = t["starts"].long(), heads // kv
    rows, fade = t["rows"].double(), torch.exp(-t["decay"].double())[None, :, None, None]
    state, out = t["state"].double(), torch.zeros(t["out"].shape, dtype=torch.float64, device="cuda")
    s = torch.stack([state[i] if i >= 0 else torch.zeros_like(state[0]) for i in t["source"].tolist()])
    count = starts[1:] - starts[:-1]
    head = torch.arange(heads, device="cuda") // each
    for i in range(int(count.max())):
        live = (count > i).nonzero()[:, 0]
        x = rows[starts[live] + i]
        q = x[:, : heads * dk].reshape(-1, heads, dk)
        k = x[:, heads * dk:(heads + kv) * dk].reshape(-1, kv, dk)[:, head]
        v = x[:, (heads + kv) * dk:].reshape(-1, kv, dv)[:, head]
        now = s[live] * fade + k[..., None] * v[..., None, :]
        s[live] = now
        out[starts[live] + i] = ((q[..., None] * now).sum(2) / math.sqrt(dk)).reshape(len(live), -1)
    state[t["target"].long()] = s
    return out, state


def exact(case, seed):
    t = _inputs(case, seed)
    return _exact_linear(t, case) if case["kind"] == "linear" else _exact_spans(t, case)
